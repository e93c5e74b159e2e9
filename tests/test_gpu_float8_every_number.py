"""Every number of the 8-bit layers' results is one: comparisons that something that is not a number fails."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
E4M3, F32, BF16 = torch.float8_e4m3fn, torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def K():
    from aien_sovereign_core_mv_b200 import kernels
    kernels.lib()
    return kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def among(seed, rows, width, at, ld):
    """Codes of all finite values, [rows, width], with codes that are not numbers before, between and behind the rows."""
    whole = torch.full((rows + 2, ld), 0x7f, dtype=torch.uint8, device="cuda")
    c = torch.randint(0, 255, (rows, width), generator=gen(seed), device="cuda", dtype=torch.uint8)
    whole[1:rows + 1, at:at + width] = torch.where((c & 0x7f) == 0x7f, torch.full_like(c, 0x3a), c)
    return whole.view(E4M3)[1:rows + 1, at:at + width]


def scales_among(seed, rows, cols):
    whole = torch.full((rows + 1, cols + 3), math.nan, device="cuda")
    whole[:rows, 2:2 + cols] = torch.exp2(torch.randint(-6, 3, (rows, cols), generator=gen(seed), device="cuda").float()) \
        * (1 + torch.rand(rows, cols, generator=gen(seed + 1), device="cuda"))
    return whole[:rows, 2:2 + cols]


def product64(a, sa, w, sw):
    """(the product, the sum of its terms' magnitudes) in 64 bits."""
    N, width = w.shape
    x = a.double() * sa.t().double().repeat_interleave(128, 1)[:, :width]
    y = w.double() * sw.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :width]
    return x @ y.t(), x.abs() @ y.abs().t()


def layout(width, gap):
    """(where a row starts, bytes between rows) of rows that start on 16-byte borders and end inside a word ("border"), or that start anywhere."""
    return (16, (width + 32) // 16 * 16) if gap == "border" else (gap % 16, width + gap)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("gap", ["border", 0, 5, 19])
@pytest.mark.parametrize("M,N,width", [(1, 130, 120), (1, 1, 1), (7, 300, 1001), (20, 130, 129), (40, 257, 250), (64, 700, 2000), (100, 200, 1000), (130, 128, 128),
                                       (300, 260, 257), (600, 1030, 400), (1030, 1100, 130)])
def test_product(K, out_dtype, gap, M, N, width):
    """Nothing of what lies around codes and scales, and every number of the result, whose room held what is not a number."""
    at, ld = layout(width, gap)
    a, w = among(1, M, width, at, ld), among(2, N, width, at, ld)
    b, nb = K.float8_blocks(width), K.float8_blocks(N)
    sa, sw = scales_among(3, b, M), scales_among(5, nb, b)
    out = torch.full((M, N), math.nan, dtype=out_dtype, device="cuda")
    K.matmul_float8(a, sa, w, sw, out)
    want, total = product64(a, sa, w, sw)
    # a block's 128 products added in float32, its two scales multiplied, b blocks added; then the result's own rounding
    off = total * (128 + b + 3) * U + want.abs() * (2.0 ** -8 if out_dtype == BF16 else U)
    assert bool(((out.double() - want).abs() <= off).all())
    assert K.read_wait_errors() == (0, 0, 0, 0)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,I,width", [(1, 8, 1), (3, 136, 129), (130, 64, 250), (300, 1000, 1001), (257, 264, 400)])
def test_gated_product(K, act, M, I, width):
    """K that ends inside a 16-byte word, as the engine's rows and weights have it, what lies behind it not numbers."""
    at, ld = layout(width, "border")
    a, w = among(1, M, width, at, ld), among(2, 2 * I, width, at, ld)
    b, nb, ob = K.float8_blocks(width), K.float8_blocks(2 * I), K.float8_blocks(I)
    # scales that bring the columns to about one: codes are 100 in the mean square, their products' sum 1e4 * sqrt(width)
    sa, sw = scales_among(3, b, M).mul_(2.0 ** -6), scales_among(5, nb, b).mul_(2.0 ** -7 / width ** 0.5)
    codes = torch.full((M, I), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.full((ob, M), math.nan, device="cuda")
    K.matmul_swiglu_float8(a, sa, w, sw, codes, scales, act=act)
    want, total = product64(a, sa, w, sw)
    g, u = (want.view(M, I // 8, 2, 8)[:, :, i].reshape(M, I) for i in (0, 1))
    tg, tu = (total.view(M, I // 8, 2, 8)[:, :, i].reshape(M, I) for i in (0, 1))
    z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    f = g / (1 + torch.exp(-(g if act == "silu" else 2 * z)))
    # columns off by their sums' roundings, which the activation passes on times at most 1.13; its own error: 12 half steps of f (silu), 14 |z| + 12 (gelu)
    e = (128 + b + 3) * U
    own = 12 if act == "silu" else 14 * z.abs() + 12
    off = 1.13 * tg * e * (u.abs() + tu * e) + (f.abs() + 1.13 * tg * e) * tu * e + (f * u).abs() * own * U
    y = f * u
    pad = lambda v: torch.nn.functional.pad(v, (0, ob * 128 - I)).view(M, ob, 128).amax(2)
    s, top, slack = scales.t().double(), pad(y.abs()), pad(off)
    assert bool(((s - torch.clamp(top / 448, min=2.0 ** -126)).abs() <= top / 448 * 2 * U + slack / 448 + 2.0 ** -149).all())
    s = s.repeat_interleave(128, 1)[:, :I]
    # half a step of e4m3 (2^-4 of the number, 2^-10 where it is subnormal); the largest may be cut at 448 by as much as the scale is off
    far = (codes.double() * s - y).abs() - torch.maximum(y.abs() / 16, s * 2.0 ** -10) * (1 + 2.0 ** -18) - 1.0625 * off - y.abs() * 8 * U
    assert bool((far <= 0).all()), float(far.max())
    assert K.read_wait_errors() == (0, 0, 0, 0)
