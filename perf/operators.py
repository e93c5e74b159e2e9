"""What is timed when the 8-bit linear layers are looked at: the operators that take a decoder's matrix products to e4m3 codes
with one float32 scale for each block of 128, each on its own.

A case is a dict of plain values.  ``kind`` says which operator it is:

  product   y = a . w^T of codes, every block's sum times the row's scale and the weight block's     (``M``, ``N``, ``K``, ``out``)
  norm      x += delta, then the RMS norm of x in 8 bits                                             (``T``, ``K``, ``delta``, ``parts``)
  gated     act(gate) * up in 8 bits                                                                 (``T``, ``K``, ``type``, ``group``, ``act``)
  rows      rows of numbers in 8 bits, a scale for 128 numbers of a row                              (``T``, ``K``, ``type``)
  blocks    a weight in 8 bits, a scale for 128 x 128 numbers                                        (``N``, ``K``, ``type``)

A block's scale is max|x| / 448 (2^-126 at least; not a number where the block holds something that is not finite), a code is
x / scale in e4m3, to the nearest and at most 448.  Scales of rows are kept as [blocks, rows], scales of a weight as
[blocks of rows, blocks of columns]; the last block of a row may be short.  Codes come back in e4m3, the values they stand for
are those times the scales that come back beside them.
"""
import math

import torch

own = False

BLOCK = 128
TOP = 448.0
LEAST = 2.0 ** -126
EPS = 1e-6
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # one user's token through the output projection of a decoder of width 4096: latency
        dict(name="product_1", kind="product", M=1, N=4096, K=4096, out="bfloat16"),
        # eight generating users through the stacked gate and up projections: the weight's bytes
        dict(name="product_8", kind="product", M=8, N=24576, K=4096, out="bfloat16"),
        # a small batch through sizes that end inside blocks and tiles, result in 32 bits
        dict(name="product_odd", kind="product", M=67, N=1000, K=2064, out="float32"),
        # a prompt of 2,048 tokens through the stacked gate and up projections: the tensor cores' rate
        dict(name="product_prompt", kind="product", M=2048, N=24576, K=4096, out="bfloat16"),
        # the norm ahead of a sublayer: eight users (the sum before it in two parts), and a prompt
        dict(name="norm_8", kind="norm", T=8, K=4096, delta="float32", parts=2),
        dict(name="norm_prompt", kind="norm", T=2048, K=4096, delta="bfloat16", parts=1),
        # between the feed-forward's two products: eight users, and a prompt
        dict(name="gated_8", kind="gated", T=8, K=12288, type="bfloat16", group=8, act="silu"),
        dict(name="gated_prompt", kind="gated", T=2048, K=12288, type="bfloat16", group=8, act="silu"),
        # the attention's output ahead of its projection: a prompt; and rows that end inside a block
        dict(name="rows_prompt", kind="rows", T=2048, K=4096, type="bfloat16"),
        dict(name="rows_odd", kind="rows", T=77, K=1001, type="float32"),
        # weights as a model is loaded: the stacked q, k, v projections; and one that ends inside its blocks
        dict(name="blocks_qkv", kind="blocks", N=6144, K=4096, type="bfloat16"),
        dict(name="blocks_odd", kind="blocks", N=1000, K=2060, type="float32"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("product", "product", "product", "norm", "gated", "rows", "blocks"))
    wide = rng.random() < 0.7                            # widths of models are whole blocks; the others end anywhere
    size = lambda lo, hi: BLOCK * _spread(rng, max(1, lo // BLOCK), hi // BLOCK) if wide else _spread(rng, lo, hi)
    if kind == "product":
        case = dict(kind=kind, M=_spread(rng, 1, 2048), N=size(64, 24576), K=size(32, 12288), out=rng.choice(("bfloat16", "bfloat16", "float32")))
        while case["M"] * case["N"] * case["K"] > 2048 * 24576 * 4096 or case["N"] * case["K"] > 24576 * 4096:
            case.update(M=max(1, case["M"] // 2), N=max(64, case["N"] // 2))
        return case
    if kind == "norm":
        delta = rng.choice(("none", "bfloat16", "float32"))
        return dict(kind=kind, T=_spread(rng, 1, 2048), K=size(32, 8192), delta=delta, parts=rng.choice((1, 2, 4)) if delta == "float32" else 1)
    if kind == "gated":
        k = size(32, 12288)
        return dict(kind=kind, T=_spread(rng, 1, 2048), K=k, type=rng.choice(("bfloat16", "float32")), group=8 if k % 8 == 0 and rng.random() < 0.5 else 0,
                    act=rng.choice(("silu", "silu", "gelu_tanh")))
    if kind == "rows":
        return dict(kind=kind, T=_spread(rng, 1, 2048), K=size(32, 12288), type=rng.choice(("bfloat16", "float32")))
    return dict(kind=kind, N=size(64, 12288), K=size(32, 4096), type=rng.choice(("bfloat16", "float32")))


# ------------------------------------------------------------------ inputs
def _blocks(n):
    return -(-n // BLOCK)


def _stream(g, rows, cols):
    """Activations: rows of uneven size, a few columns far above the rest."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    loud = torch.randint(0, cols, (max(1, cols // 256),), generator=g, device="cuda")
    x[:, loud] *= 16.0
    return x


def _weight(g, rows, cols):
    """A projection: columns keep a vector's length, rows of uneven size."""
    return torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(0.3 * torch.randn(rows, 1, generator=g, device="cuda")) / math.sqrt(cols)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, K = case["kind"], case["K"]
    codes = lambda rows: torch.empty(rows, K, dtype=torch.float8_e4m3fn, device="cuda")
    f32 = lambda *shape: torch.empty(*shape, dtype=torch.float32, device="cuda")
    if kind == "product":
        a, a_scales = _rows_in_8_bits(_stream(g, case["M"], K))
        w, w_scales = _weight_in_8_bits(_weight(g, case["N"], K))
        return dict(case=case, a=a, a_scales=a_scales, w=w, w_scales=w_scales, out=torch.empty(case["M"], case["N"], dtype=TYPES[case["out"]], device="cuda"))
    if kind == "blocks":
        return dict(case=case, w=_weight(g, case["N"], K).to(TYPES[case["type"]]), codes=codes(case["N"]), scales=f32(_blocks(case["N"]), _blocks(K)))
    T = case["T"]
    state = dict(case=case, codes=codes(T), scales=f32(_blocks(K), T))
    if kind == "norm":
        state.update(x=_stream(g, T, K), weight=(0.8 + 0.4 * torch.rand(K, generator=g, device="cuda")).to(torch.bfloat16))
        if case["delta"] == "none":
            state["delta"] = None
        elif case["parts"] > 1:
            state["delta"] = 0.3 * torch.randn(case["parts"], T, K, generator=g, device="cuda")
        else:
            state["delta"] = (0.3 * torch.randn(T, K, generator=g, device="cuda")).to(TYPES[case["delta"]])
    elif kind == "gated":
        state["gate_up"] = _stream(g, T, 2 * K).to(TYPES[case["type"]])
    else:
        state["x"] = _stream(g, T, K).to(TYPES[case["type"]])
    return state


# ------------------------------------------------------------------ the plain forms, in 32 bits
def _scale_of(top):
    s = torch.clamp(top / TOP, min=LEAST)
    return torch.where(torch.isfinite(top), s, torch.full_like(s, math.nan))


def _code(x, scale):
    return torch.clamp(x * (1.0 / scale), -TOP, TOP).to(torch.float8_e4m3fn)


def _rows_in_8_bits(x):
    """(codes [T, K], scales [blocks, T]) of float32 rows."""
    T, K = x.shape
    b = _blocks(K)
    p = torch.nn.functional.pad(x, (0, b * BLOCK - K)).view(T, b, BLOCK)
    s = _scale_of(p.abs().amax(-1))
    return _code(p, s[:, :, None]).view(T, b * BLOCK)[:, :K].contiguous(), s.t().contiguous()


def _weight_in_8_bits(w):
    """(codes [N, K], scales [blocks of rows, blocks of columns]) of a float32 weight."""
    N, K = w.shape
    n, b = _blocks(N), _blocks(K)
    p = torch.nn.functional.pad(w, (0, b * BLOCK - K, 0, n * BLOCK - N)).view(n, BLOCK, b, BLOCK)
    s = _scale_of(p.abs().amax(3).amax(1))
    return _code(p, s[:, None, :, None]).view(n * BLOCK, b * BLOCK)[:N, :K].contiguous(), s


def _per_number(scales, n, k, rows):
    """A weight's scales, one for each of its numbers ([n, k]); with ``rows`` the scales of rows, [blocks, n]."""
    if rows:
        return scales.t().repeat_interleave(BLOCK, 1)[:, :k]
    return scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _gate_and_up(gu, group):
    T, K = gu.shape[0], gu.shape[1] // 2
    if group == 0:
        return gu[:, :K], gu[:, K:]
    v = gu.view(T, K // group, 2, group)
    return v[:, :, 0].reshape(T, K), v[:, :, 1].reshape(T, K)


def _act(g, act):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from aien_sovereign_core_mv_b200 import kernels
        if kind == "product":
            kernels.matmul_float8(state["a"], state["a_scales"], state["w"], state["w_scales"], state["out"])
            return [state["out"]]
        if kind == "blocks":
            kernels.quantize_blocks_float8(state["w"], state["codes"], state["scales"])
        elif kind == "norm":
            kernels.add_rmsnorm_float8(state["x"], state["delta"], state["weight"], EPS, state["codes"], state["scales"])
            return [state["x"], state["codes"], state["scales"]]
        elif kind == "gated":
            kernels.swiglu_float8(state["gate_up"], state["codes"], state["scales"], group=case["group"], act=case["act"])
        else:
            kernels.quantize_rows_float8(state["x"], state["codes"], state["scales"])
        return [state["codes"], state["scales"]]
    if kind == "product":
        a = state["a"].float() * _per_number(state["a_scales"], case["M"], case["K"], True)
        w = state["w"].float() * _per_number(state["w_scales"], case["N"], case["K"], False)
        return [(a @ w.t()).to(TYPES[case["out"]])]
    if kind == "blocks":
        return list(_weight_in_8_bits(state["w"].float()))
    if kind == "norm":
        x, d = state["x"], state["delta"]
        if d is not None:
            x += d.sum(0) if d.dim() == 3 else d.float()
        h = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * state["weight"].float()
        return [x] + list(_rows_in_8_bits(h))
    if kind == "gated":
        g, u = _gate_and_up(state["gate_up"].float(), case["group"])
        return list(_rows_in_8_bits(_act(g, case["act"]) * u))
    return list(_rows_in_8_bits(state["x"].float()))


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, K = case["kind"], case["K"]
    if kind == "product":
        M, N = case["M"], case["N"]
        scales = 4 * _blocks(K) * (M + _blocks(N))
        return {"bytes": (M + N) * K + scales + M * N * TYPES[case["out"]].itemsize, "flops": 2 * M * N * K}
    if kind == "blocks":
        n = case["N"] * K
        return {"bytes": n * (TYPES[case["type"]].itemsize + 1) + 4 * _blocks(case["N"]) * _blocks(K), "flops": 2 * n}
    T = case["T"]
    n, scales = T * K, 4 * _blocks(K) * T
    if kind == "norm":
        if case["delta"] == "none":
            return {"bytes": n * 5 + 2 * K + scales, "flops": 6 * n}
        return {"bytes": n * (9 + TYPES[case["delta"]].itemsize * case["parts"]) + 2 * K + scales, "flops": (6 + case["parts"]) * n}
    size = TYPES[case["type"]].itemsize
    if kind == "gated":
        return {"bytes": n * (2 * size + 1) + scales, "flops": 8 * n}
    return {"bytes": n * (size + 1) + scales, "flops": 2 * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def _cut(v, axis):
    """The blocks of 128 along an axis, as a list of views."""
    return torch.split(v, BLOCK, axis)


def _scale64(top):
    return torch.maximum(top / TOP, torch.full_like(top, LEAST))


def _rows64(h):
    """Codes before their rounding to e4m3, and scales, of float64 rows."""
    codes, scales = [], []
    for part in _cut(h, 1):
        s = _scale64(part.abs().max(1).values)
        codes.append(part / s[:, None])
        scales.append(s)
    return [torch.cat(codes, 1), torch.stack(scales)]


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "product":
        a, w = state["a"].double(), state["w"].double()
        y = torch.zeros(case["M"], case["N"], dtype=torch.float64, device="cuda")
        for b, (ak, wk) in enumerate(zip(_cut(a, 1), _cut(w, 1))):
            sw = state["w_scales"][:, b].double().repeat_interleave(BLOCK)[:case["N"]]
            y += (ak @ wk.t()) * state["a_scales"][b].double()[:, None] * sw[None, :]
        return [y]
    if kind == "blocks":
        codes, scales = [], []
        for strip in _cut(state["w"].double(), 0):
            s = torch.stack([_scale64(part.abs().max()) for part in _cut(strip, 1)])
            codes.append(torch.cat([part / v for part, v in zip(_cut(strip, 1), s)], 1))
            scales.append(s)
        return [torch.cat(codes, 0), torch.stack(scales)]
    if kind == "norm":
        x, d = state["x"].double(), state["delta"]
        if d is not None:
            x = x + (d.double().sum(0) if d.dim() == 3 else d.double())
        r = (x.square().sum(1) / case["K"] + EPS).rsqrt()
        return [x] + _rows64(x * r[:, None] * state["weight"].double())
    if kind == "gated":
        gu, K = state["gate_up"].double(), case["K"]
        if case["group"]:
            at = torch.arange(K, device="cuda")
            at = at // case["group"] * 2 * case["group"] + at % case["group"]
            g, u = gu[:, at], gu[:, at + case["group"]]
        else:
            g, u = gu[:, :K], gu[:, K:]
        if case["act"] == "silu":
            f = g * torch.sigmoid(g)
        else:
            f = g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))
        return _rows64(f * u)
    return _rows64(state["x"].double())
