"""The 8-bit linear layers' kernels against restatements in 64 bits.

Tolerances count roundings.  A code is off by at most half a step of e4m3 at its value (2^-4 of it, 2^-10 where the numbers are
subnormal) plus what the value itself was off before it was rounded; a scale is one float32 division of the block's maximum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                 # half a step of float32, relative
E4M3, F32, BF16 = torch.float8_e4m3fn, torch.float32, torch.bfloat16
LEAST = 2.0 ** -126


@pytest.fixture(scope="module")
def K():
    from aien_sovereign_core_mv_b200 import kernels
    kernels.lib()
    return kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape):
    return torch.randn(*shape, generator=gen(seed), device="cuda")


def per_number(scales_blocks_last, width):
    return scales_blocks_last.repeat_interleave(128, -1)[..., :width]


def padded_blocks(v):
    """[rows, K] float64 as [rows, blocks, 128], zeros behind the end."""
    rows, width = v.shape
    b = -(-width // 128)
    return torch.nn.functional.pad(v, (0, b * 128 - width)).view(rows, b, 128)


def check_codes(codes, scales, value, off):
    """codes [rows, K], scales [rows, blocks] (float64), value: what they stand for; off: how far the value may be off before rounding."""
    s = per_number(scales, value.shape[1])
    v = value / s
    step = torch.maximum(v.abs() / 16, torch.full_like(v, 2.0 ** -10))
    # x * (1 / s): two roundings beside the code's own
    far = (codes.double() - v.clamp(-448, 448)).abs() - step * (1 + 2.0 ** -20) - v.abs() * 4 * U - 1.0625 * off / s
    assert not bool((far > 0).any()), float(far.max())


def check_scales(scales, value, off):
    """A block's scale is max / 448, at least 2^-126: one division off, and what the values were off."""
    top, slack = padded_blocks(value.abs()).amax(-1), padded_blocks(off).amax(-1)
    want = torch.clamp(top / 448, min=LEAST)
    assert bool(((scales - want).abs() <= want * 2 * U + slack / 448 + 2.0 ** -149).all())


SIZES = [(1, 1), (1, 128), (2, 127), (3, 129), (17, 1001), (5, 4096), (300, 2064), (9, 2600), (1030, 136)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,width", SIZES)
@pytest.mark.parametrize("gap", [0, 3, 16])
def test_rows(K, dtype, T, width, gap):
    x = (randn(T + width, T, width + gap) * 3).to(dtype)[:, :width]
    codes = torch.zeros(T, width + gap, dtype=torch.uint8, device="cuda").view(E4M3)[:, :width]
    b = K.float8_blocks(width)
    whole = torch.full((b, T + gap), 7.0, device="cuda")
    K.quantize_rows_float8(x, codes, whole[:, :T])
    v = x.double()
    check_scales(whole[:, :T].double().t(), v, torch.zeros_like(v))
    check_codes(codes, whole[:, :T].double().t(), v, torch.zeros_like(v))
    assert bool((whole[:, T:] == 7.0).all())


def special_rows(width=300):
    """Blocks of zeros, of the smallest and largest numbers, and of what is not finite; the second block of every row is ordinary."""
    x = randn(5, 8, width)
    x[0, :128] = 0.0
    x[1, :128] = 1e-42
    x[2, :128] = 3.3e38
    x[3, 5] = math.inf
    x[4, 7] = math.nan
    x[5, :128] = -0.0
    x[6, 0:128] = torch.arange(128, device="cuda") * 2.0 ** -130
    x[7, 3] = -math.inf
    return x


def test_rows_of_zeros_extremes_and_numbers_that_are_none(K):
    x = special_rows()
    codes, scales = torch.empty(8, 300, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(3, 8, device="cuda")
    K.quantize_rows_float8(x, codes, scales)
    s, c = scales.t().double(), codes.double()
    assert bool((c[[0, 5], :128] == 0).all()) and bool((s[[0, 5], 0] == LEAST).all())
    for r in (3, 4, 7):
        assert bool(torch.isnan(c[r, :128]).all()) and math.isnan(float(s[r, 0]))
    rest = torch.tensor([0, 1, 2, 5, 6], device="cuda")
    v = x[rest].double()
    check_scales(s[rest], v, torch.zeros_like(v))
    check_codes(codes[rest], s[rest], v, torch.zeros_like(v))
    v = x[:, 128:].double()
    check_codes(codes[:, 128:], s[:, 1:], v, torch.zeros_like(v))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,width", [(1, 1), (128, 128), (130, 257), (1000, 2060), (77, 640), (640, 264)])
def test_blocks(K, dtype, N, width):
    w = (randn(N + width, N, width + 8) * 0.05).to(dtype)[:, :width]
    codes = torch.empty(N, width, dtype=torch.uint8, device="cuda").view(E4M3)
    nb, kb = K.float8_blocks(N), K.float8_blocks(width)
    scales = torch.empty(nb, kb, device="cuda")
    K.quantize_blocks_float8(w, codes, scales)
    v = w.double()
    top = torch.nn.functional.pad(v.abs(), (0, kb * 128 - width, 0, nb * 128 - N)).view(nb, 128, kb, 128).amax((1, 3))
    want = torch.clamp(top / 448, min=LEAST)
    assert bool(((scales.double() - want).abs() <= want * 2 * U).all())
    check_codes(codes, scales.double().repeat_interleave(128, 0)[:N], v, torch.zeros_like(v))


@pytest.mark.parametrize("delta", ["none", "bfloat16", "float32", "parts1", "parts5"])
@pytest.mark.parametrize("T,width", [(1, 1), (3, 129), (1, 4096), (40, 1000), (9, 2048), (5, 8192), (2, 16384), (2, 16400), (200, 4104)])
def test_norm(K, delta, T, width):
    x = randn(T + width, T, width) * 2
    if delta == "none":
        d, parts = None, []
    elif delta.startswith("parts"):
        d = randn(7, int(delta[5:]), T, width)
        parts = list(d)
    else:
        d = randn(7, T, width).to(getattr(torch, delta))
        parts = [d.float()]
    for w in ((0.5 + randn(8, width).abs()).to(BF16), 0.5 + randn(9, width).abs()):
        mine = x.clone()
        codes = torch.empty(T, width, dtype=torch.uint8, device="cuda").view(E4M3)
        scales = torch.empty(K.float8_blocks(width), T, device="cuda")
        K.add_rmsnorm_float8(mine, d, w, 1e-5, codes, scales)
        want = x.clone()
        for p in parts:
            want += p
        assert torch.equal(mine, want)                     # the same sums in the same order
        v = want.double()
        h = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-5) * w.double()
        # the sum of squares goes through at most 40 additions in a thread and 41 over the warps; its root halves the error; five more roundings
        off = h.abs() * 64 * U
        check_scales(scales.double().t(), h, off)
        check_codes(codes, scales.double().t(), h, off)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,width,group", [(1, 1, 0), (1, 128, 8), (3, 136, 8), (5, 129, 0), (7, 1000, 8), (7, 1000, 0), (130, 264, 4), (2, 12288, 8), (600, 96, 0)])
def test_gated(K, act, dtype, T, width, group):
    gu = (randn(T + width + group, T, 2 * width) * 3).to(dtype)
    codes = torch.empty(T, width, dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.empty(K.float8_blocks(width), T, device="cuda")
    K.swiglu_float8(gu, codes, scales, group=group, act=act)
    v = gu.double()
    if group:
        v = v.view(T, width // group, 2, group)
        g, u = v[:, :, 0].reshape(T, width), v[:, :, 1].reshape(T, width)
    else:
        g, u = v[:, :width], v[:, width:]
    z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    f = g * torch.sigmoid(g) if act == "silu" else 0.5 * g * (1 + torch.tanh(z))
    # silu: the exponential is off by 2 + 1.2 |g| units (|g| < 18 here: 24), the quotient by 2, two more roundings; gelu: z is off by 8 roundings,
    # which tanh passes on times z (1 - tanh^2) < 1, and 1 + tanh by 4 units of 1
    assert float(g.abs().max()) < 18
    off = (g * u).abs() * 64 * U
    check_scales(scales.double().t(), f * u, off)
    check_codes(codes, scales.double().t(), f * u, off)


def codes_of(seed, rows, width, gap=0):
    """Codes of all finite values and scales of uneven size, as a user would hold them."""
    c = torch.randint(0, 255, (rows, width + gap), generator=gen(seed), device="cuda", dtype=torch.uint8)
    c = torch.where((c & 0x7f) == 0x7f, torch.full_like(c, 0x3a), c)
    return c.view(E4M3)[:, :width]


def scales_of(seed, *shape):
    return torch.exp2(torch.randint(-6, 3, shape, generator=gen(seed), device="cuda").float()) * (1 + torch.rand(*shape, generator=gen(seed + 1), device="cuda"))


def product64(a, sa, w, sw):
    """(the product, the sum of its terms' magnitudes) in 64 bits."""
    N, width = w.shape
    x = a.double() * per_number(sa.t().double(), width)
    y = w.double() * per_number(sw.double().repeat_interleave(128, 0)[:N], width)
    return x @ y.t(), x.abs() @ y.abs().t()


def check_product(out, a, sa, w, sw):
    want, total = product64(a, sa, w, sw)
    b = sa.shape[0]
    # a block's 128 products added in float32, its two scales multiplied, b blocks added; then the result's own rounding
    off = total * (128 + b + 3) * U + want.abs() * (2.0 ** -8 if out.dtype == BF16 else U)
    far = (out.double() - want).abs() - off
    assert not bool((far > 0).any()), (float(far.max()), float(((out.double() - want).abs() / off).max()))


PRODUCTS = [(1, 1, 1), (1, 130, 127), (1, 1000, 1001), (1, 128, 128), (2, 1, 300), (1, 4096, 4096), (2, 130, 127), (3, 64, 129), (8, 1000, 2064), (16, 257, 4096), (17, 640, 256), (31, 129, 1000),
            (33, 520, 12288), (64, 300, 1008), (65, 384, 384), (100, 96, 144), (127, 1000, 512), (128, 128, 640), (129, 257, 272), (200, 1040, 1040),
            (256, 512, 2048), (300, 2000, 400), (513, 777, 1111), (1030, 1100, 1552), (2048, 1536, 512)]


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,width", PRODUCTS)
def test_product(K, out_dtype, M, N, width):
    a, w = codes_of(M + 1, M, width), codes_of(N + 2, N, width)
    sa, sw = scales_of(3, K.float8_blocks(width), M), scales_of(4, K.float8_blocks(N), K.float8_blocks(width))
    out = torch.full((M, N), math.nan, dtype=out_dtype, device="cuda")
    K.matmul_float8(a, sa, w, sw, out)
    check_product(out, a, sa, w, sw)
    assert K.read_wait_errors() == (0, 0, 0, 0)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,width", [(5, 200, 300), (16, 256, 1024), (70, 140, 260), (300, 520, 1001), (700, 1300, 640)])
@pytest.mark.parametrize("gap_a,gap_w,gap_out", [(16, 32, 8), (1, 0, 3), (0, 5, 0), (7, 9, 1)])
def test_product_of_rows_apart(K, out_dtype, M, N, width, gap_a, gap_w, gap_out):
    a, w = codes_of(M, M, width, gap_a), codes_of(N, N, width, gap_w)
    b = K.float8_blocks(width)
    sa, sw = scales_of(3, b, M + 5)[:, :M], scales_of(4, K.float8_blocks(N), b + 3)[:, :b]
    whole = torch.full((M, N + gap_out), 5.0, dtype=out_dtype, device="cuda")
    K.matmul_float8(a, sa, w, sw, whole[:, :N])
    check_product(whole[:, :N], a, sa, w, sw)
    assert bool((whole[:, N:] == 5.0).all())


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("width", [48, 55, 400])
@pytest.mark.parametrize("N", [1, 3, 7, 130, 257, 735, 1034])
@pytest.mark.parametrize("M", [1, 5, 40, 130, 400, 900])
def test_nothing_is_written_beyond_the_result(K, M, N, width, out_dtype):
    """Rows of the result that start on 16-byte borders and end inside a word, with others' numbers behind them."""
    a, w = codes_of(M, M, width), codes_of(N, N, width)
    b = K.float8_blocks(width)
    sa, sw = scales_of(3, b, M), scales_of(4, K.float8_blocks(N), b)
    for ld in ((N + 8) // 8 * 8, N + 1, N + 9):
        whole = torch.full((M + 2, ld), 5.0, dtype=out_dtype, device="cuda")
        K.matmul_float8(a, sa, w, sw, whole[1:M + 1, :N])
        check_product(whole[1:M + 1, :N], a, sa, w, sw)
        assert bool((whole[:, N:] == 5.0).all()) and bool((whole[0] == 5.0).all()) and bool((whole[M + 1] == 5.0).all())


@pytest.mark.parametrize("M", [4, 40, 200, 600])
def test_product_starts_anywhere(K, M):
    """Rows that begin off the 16-byte borders: a view of a larger tensor."""
    N, width = 260, 300
    a, w = codes_of(1, M, width + 40)[:, 13:13 + width], codes_of(2, N, width + 21)[:, 5:5 + width]
    sa, sw = scales_of(3, 3, M + 1)[:, 1:], scales_of(4, 3, 4)[:, 1:]
    out = torch.empty(M, N + 1, device="cuda")[:, 1:]
    K.matmul_float8(a, sa, w, sw, out)
    check_product(out, a, sa, w, sw)


@pytest.mark.parametrize("at,gap", [(0, 16), (16, 32), (1, 3), (15, 0), (5, 11), (0, "border"), (32, "border")])
@pytest.mark.parametrize("M,N,width", [(1, 130, 120), (20, 130, 129), (100, 200, 1000), (300, 260, 257), (600, 1030, 400)])
def test_what_lies_around_the_rows_is_not_looked_at(K, M, N, width, at, gap):
    """Codes that are not numbers before, between and behind the rows; scales that are not numbers beside the ones that count."""
    ld = width + at + gap if gap != "border" else (width + at + 16) // 16 * 16         # rows that start on 16-byte borders and end inside one
    def among_nan(seed, rows):
        whole = torch.full((rows + 2, ld), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
        part = whole[1:rows + 1, at:at + width]
        part.view(torch.uint8).copy_(codes_of(seed, rows, width).view(torch.uint8))
        return part
    a, w = among_nan(1, M), among_nan(2, N)
    b, nb = K.float8_blocks(width), K.float8_blocks(N)
    sa, sw = torch.full((b + 1, M + 3), math.nan, device="cuda"), torch.full((nb + 1, b + 2), math.nan, device="cuda")
    sa[:b, 2:2 + M], sw[:nb, 1:1 + b] = scales_of(3, b, M), scales_of(4, nb, b)
    sa, sw = sa[:b, 2:2 + M], sw[:nb, 1:1 + b]
    out = torch.empty(M, N, device="cuda")
    K.matmul_float8(a, sa, w, sw, out)
    check_product(out, a, sa, w, sw)


@pytest.mark.parametrize("M", [1, 20, 130, 400])
def test_one_bad_number_stays_in_its_row(K, M):
    N, width = 300, 520
    a, w = codes_of(1, M, width).clone(), codes_of(2, N, width)
    sa, sw = scales_of(3, 5, M), scales_of(4, 3, 5)
    want = torch.empty(M, N, device="cuda")
    K.matmul_float8(a, sa, w, sw, want)
    r = M - 1
    a.view(torch.uint8)[r, 200] = 0x7f
    got = torch.empty(M, N, device="cuda")
    K.matmul_float8(a, sa, w, sw, got)
    assert bool(torch.isnan(got[r]).all()) and torch.equal(got[:r], want[:r])
    sa[2, r] = math.nan
    a.view(torch.uint8)[r, 200] = 0x38
    K.matmul_float8(a, sa, w, sw, got)
    assert bool(torch.isnan(got[r]).all()) and torch.equal(got[:r], want[:r])


def gated64(y, width, act):
    """act(gate) * up of columns in runs of 8, and gate * up."""
    v = y.view(y.shape[0], width // 8, 2, 8)
    g, u = v[:, :, 0].reshape(-1, width), v[:, :, 1].reshape(-1, width)
    z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    return (g * torch.sigmoid(g) if act == "silu" else 0.5 * g * (1 + torch.tanh(z))) * u, g, u


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,I,width", [(1, 8, 16), (3, 136, 144), (130, 64, 128), (257, 264, 400), (300, 1000, 1040), (512, 1288, 640), (1500, 3200, 272)])
@pytest.mark.parametrize("gap", [0, 1, 16])
def test_gated_product(K, act, M, I, width, gap):
    pad = -width % 16
    a, w = codes_of(M, M, width, pad), codes_of(I, 2 * I, width, pad)
    b, nb, ob = K.float8_blocks(width), K.float8_blocks(2 * I), K.float8_blocks(I)
    # scales that bring the columns to about one: codes are 100 in the mean square, their products' sum 1e4 * sqrt(width)
    sa, sw = scales_of(3, b, M) * 2.0 ** -6, scales_of(4, nb, b) * (2.0 ** -7 / width ** 0.5)
    whole = torch.zeros(M, I + gap, dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.full((ob, M + gap), 7.0, device="cuda")
    K.matmul_swiglu_float8(a, sa, w, sw, whole[:, :I], scales[:, :M], act=act)
    want, total = product64(a, sa, w, sw)
    y, g, u = gated64(want, I, act)
    _, tg, tu = gated64(total, I, act)
    # the columns are off by their sums' roundings (check_product); the activation passes an error of its argument on times at most 1.13 (both
    # derivatives stay below that), its own value is off by 64 units of gate * up as in test_gated, or 1.2 |g| units more for |g| beyond 18
    e = (128 + b + 3) * U
    off = 1.13 * tg * e * (u.abs() + tu * e) + g.abs() * tu * e + (g * u).abs() * (64 + 1.2 * g.abs()) * U
    check_scales(scales[:, :M].double().t(), y, off)
    check_codes(whole[:, :I], scales[:, :M].double().t(), y, off)
    assert bool((whole.view(torch.uint8)[:, I:] == 0).all()) and bool((scales[:, M:] == 7.0).all())
    assert K.read_wait_errors() == (0, 0, 0, 0)


def test_gated_product_of_bad_rows(K):
    M, I, width = 300, 200, 256
    a, w = codes_of(1, M, width).clone(), codes_of(2, 2 * I, width)
    sa, sw = scales_of(3, 2, M) * 2.0 ** -12, scales_of(4, 4, 2) * 2.0 ** -8
    e = lambda: (torch.empty(M, I, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(2, M, device="cuda"))
    codes, scales = e()
    K.matmul_swiglu_float8(a, sa, w, sw, codes, scales)
    a.view(torch.uint8)[77, 3] = 0x7f
    a.view(torch.uint8)[78] = 0
    bad, bad_scales = e()
    K.matmul_swiglu_float8(a, sa, w, sw, bad, bad_scales)
    assert bool(torch.isnan(bad[77].float()).all()) and bool(torch.isnan(bad_scales[:, 77]).all())
    assert bool((bad[78].float() == 0).all()) and bool((bad_scales[:, 78] == LEAST).all())
    rest = [r for r in range(M) if r not in (77, 78)]
    assert torch.equal(bad.view(torch.uint8)[rest], codes.view(torch.uint8)[rest]) and torch.equal(bad_scales[:, rest], scales[:, rest])


def test_gated_product_refusals(K):
    a, sa = codes_of(1, 5, 256), scales_of(2, 2, 5)
    out = lambda I: (torch.empty(5, I, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(K.float8_blocks(I), 5, device="cuda"))
    with pytest.raises(K.KernelError, match="runs of 8"):
        K.matmul_swiglu_float8(a, sa, codes_of(3, 40, 256), scales_of(4, 1, 2), *out(20))
    with pytest.raises(K.KernelError, match="activation 'relu'"):
        K.matmul_swiglu_float8(a, sa, codes_of(3, 48, 256), scales_of(4, 1, 2), *out(24), act="relu")
    with pytest.raises(K.KernelError, match="w has shape"):
        K.matmul_swiglu_float8(a, sa, codes_of(3, 40, 256), scales_of(4, 1, 2), *out(24))
    with pytest.raises(K.KernelError, match="aligned"):
        K.matmul_swiglu_float8(codes_of(1, 5, 250), sa, codes_of(3, 48, 250), scales_of(4, 1, 2), *out(24))


def test_arguments_on_the_host_are_refused(K):
    x, codes, scales, w = randn(1, 3, 256), codes_of(2, 3, 256), scales_of(3, 2, 3), torch.ones(256, device="cuda")
    for bad in (dict(weight=w.cpu()), dict(x=x.cpu()), dict(scales=scales.cpu()), dict(delta=x.cpu())):
        args = {**dict(x=x, delta=None, weight=w, eps=1e-6, codes=codes, scales=scales), **bad}
        with pytest.raises(K.KernelError, match="CUDA device"):
            K.add_rmsnorm_float8(**args)
    with pytest.raises(K.KernelError, match="CUDA device"):
        K.quantize_rows_float8(x, codes.cpu(), scales)


def test_nothing_to_do(K):
    w, sw = codes_of(1, 5, 200), scales_of(2, 1, 2)
    e = lambda *s: torch.empty(*s, dtype=torch.uint8, device="cuda").view(E4M3)
    K.matmul_float8(e(0, 200), torch.empty(2, 0, device="cuda"), w, sw, torch.empty(0, 5, device="cuda"))
    K.quantize_rows_float8(torch.empty(0, 200, device="cuda"), e(0, 200), torch.empty(2, 0, device="cuda"))
    K.swiglu_float8(torch.empty(0, 400, device="cuda"), e(0, 200), torch.empty(2, 0, device="cuda"))
    K.add_rmsnorm_float8(torch.empty(0, 200, device="cuda"), None, torch.ones(200, device="cuda"), 1e-6, e(0, 200), torch.empty(2, 0, device="cuda"))
    torch.cuda.synchronize()


class Layer:
    """Norm, product, gated activation, product, added to the stream: the operators in the order that a decoder's layer has them."""

    def __init__(self, K, T, H, I, seed):
        self.K, self.T, self.H, self.I = K, T, H, I
        e = lambda *s: torch.empty(*s, dtype=torch.uint8, device="cuda").view(E4M3)
        f = lambda *s: torch.empty(*s, device="cuda")
        b = K.float8_blocks
        self.raw_up, self.raw_down = randn(seed, 2 * I, H) / H ** 0.5, (randn(seed + 1, H, I) / I ** 0.5).to(BF16)
        self.up, self.up_s, self.down, self.down_s = e(2 * I, H), f(b(2 * I), b(H)), e(H, I), f(b(H), b(I))
        self.norm = 1 + 0.1 * randn(seed + 2, H)
        self.h, self.h_s, self.act, self.act_s = e(T, H), f(b(H), T), e(T, I), f(b(I), T)
        self.gu, self.y = torch.empty(T, 2 * I, dtype=BF16, device="cuda"), torch.empty(T, H, dtype=BF16, device="cuda")

    def weights(self):
        self.K.quantize_blocks_float8(self.raw_up, self.up, self.up_s)
        self.K.quantize_blocks_float8(self.raw_down, self.down, self.down_s)

    def step(self, x, delta, w_ready=False):
        K = self.K
        K.add_rmsnorm_float8(x, delta, self.norm, 1e-6, self.h, self.h_s)
        K.matmul_float8(self.h, self.h_s, self.up, self.up_s, self.gu, w_ready=w_ready)
        K.swiglu_float8(self.gu, self.act, self.act_s, group=8)
        K.matmul_float8(self.act, self.act_s, self.down, self.down_s, self.y, w_ready=w_ready)
        return self.y


@pytest.mark.parametrize("T,H,I", [(1, 256, 384), (8, 1024, 1408), (33, 200, 264), (150, 512, 640), (600, 1024, 1536)])
def test_a_layer_of_them(K, T, H, I):
    """The operators in a row, with nothing waited for between them (weights quantised right before their first use among it): every stage against the
    definition on the stage's own inputs, then the same again many times and through a captured graph, to the same bits."""
    m = Layer(K, T, H, I, 3)
    x0, delta = randn(11, T, H), randn(12, T, H).to(BF16)
    x = x0.clone()
    m.weights()
    y = m.step(x, delta).clone()
    check_product(m.gu, m.h, m.h_s, m.up, m.up_s)
    check_product(m.y, m.act, m.act_s, m.down, m.down_s)
    g = m.gu.double().view(T, I // 8, 2, 8)
    f = (g[:, :, 0] * torch.sigmoid(g[:, :, 0]) * g[:, :, 1]).reshape(T, I)
    off = (g[:, :, 0] * g[:, :, 1]).abs().reshape(T, I) * 64 * U
    check_codes(m.act, m.act_s.double().t(), f, off)
    # against the same layer in 64 bits: what a product reads, its rows and its weight, is off by at most 2^-4 / sqrt(3) in the mean square (a step of e4m3 at
    # its worst), both together by 0.051 of the product's norm; the activation of gate and up, each off by that, at most doubles it; with the second
    # product's own 0.051 that is 0.114, and half as much again for the errors' spread over so few numbers
    v = (x0 + delta.float()).double()
    h = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * m.norm.double()
    g = (h @ m.raw_up.double().t()).view(T, I // 8, 2, 8)
    want = (g[:, :, 0] * torch.sigmoid(g[:, :, 0]) * g[:, :, 1]).reshape(T, I) @ m.raw_down.double().t()
    assert float((y.double() - want).norm() / want.norm()) < 1.5 * 0.114
    for i in range(20):
        if i < 10:
            m.weights()
        x.copy_(x0)
        m.step(x, delta, w_ready=i >= 10)                # the weights stay as they are from here on
    assert torch.equal(m.y, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.copy_(x0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            m.weights()
            m.step(x, delta)
        for _ in range(3):
            x.copy_(x0)
            m.y.zero_()
            graph.replay()
        assert torch.equal(m.y, y)
    torch.cuda.current_stream().wait_stream(side)
    assert K.read_wait_errors() == (0, 0, 0, 0)


def test_two_streams_at_once(K):
    """Two layers on two streams, which share nothing."""
    ms = [Layer(K, 40, 512, 768, 21), Layer(K, 300, 512, 768, 31)]
    xs = [randn(41, 40, 512), randn(42, 300, 512)]
    alone = []
    for m, x in zip(ms, xs):
        m.weights()
        alone.append(m.step(x.clone(), None).clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for s, m, x in zip(streams, ms, xs):
            with torch.cuda.stream(s):
                m.step(x, None)
    torch.cuda.synchronize()
    for m, y in zip(ms, alone):
        assert torch.equal(m.y, y)


def test_more_numbers_than_32_bits_count(K):
    """2.2 G numbers of a weight: rows beyond 2^31 bytes from the first."""
    N, width = 270_000, 8192
    w = torch.empty(N, width, dtype=torch.uint8, device="cuda")
    w.fill_(0x30)
    w[-1] = 0x38
    w = w.view(E4M3)
    sw = torch.full((K.float8_blocks(N), 64), 0.5, device="cuda")
    a, sa = torch.full((3, width), 0x38, dtype=torch.uint8, device="cuda").view(E4M3), torch.ones(64, 3, device="cuda")
    out = torch.empty(3, N, device="cuda")
    K.matmul_float8(a, sa, w, sw, out)
    assert bool((out[:, :-1] == 0.5 * 0.5 * width).all()) and bool((out[:, -1] == 0.5 * width).all())
