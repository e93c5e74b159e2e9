"""The gated activations of the 8-bit layers, number by number.

A block that holds one number (or one number eight times) has the scale |number| / 448, so that its scale shows the activation to the last
bits, where codes would hide all but four.  An error is counted in U = 2^-24, half a step of float32, relative to the number:
  silu(g) * u    the exponential 5 (four of the instruction's 2^-22, one of a correction), g e, 1 + e, the quotient and times u one each, the scale 2: 11, and one
                 more for what errors make of each other
  gelu(g) * u    as g / (1 + exp(-2 z)) * u; z = c (g + d g^3) is off by at most 7 (two rounded constants, five operations), which the exponential passes on
                 times |2 z|: 14 |z| + 12
Beside that a float32 number below 2^-126 is off by 2^-150 wherever it stands: of e, of g e and of a scale, when gates are below -87."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def K():
    from aien_sovereign_core_mv_b200 import kernels
    kernels.lib()
    return kernels


def gates(act):
    """The whole range in which the activation is an ordinary float32 number, and its middle more closely.  (Below -88.7 the exponential of silu is beyond float32, and the
    result 0; the exponential of the gelu below -10.05.)"""
    low, high = (-88.7, 88.0) if act == "silu" else (-10.0, 10.0)
    g = torch.cat([torch.linspace(low, high, 6000, dtype=torch.float64), torch.linspace(-6, 6, 2000, dtype=torch.float64)])
    return g.float().cuda()


def activation64(g, act):
    """(f(g), how many U it times something may be off)"""
    g = g.double()
    if act == "silu":
        return g / (1 + torch.exp(-g)), torch.full_like(g, 12)
    z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    return g / (1 + torch.exp(-2 * z)), 14 * z.abs() + 12


def check(scales, want, units):
    want = want.abs()
    far = ((scales.double() * 448 - want).abs() - want * units * U) / (want * U + 2.0 ** -149)
    assert bool((far <= 0).all()), f"{float(far.max())} units beyond"


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_one_number_a_row(K, act):
    """Every gate in a row of its own, times 2^24, so that no scale is the least one."""
    g = gates(act)
    gu = torch.stack([g, torch.full_like(g, 2.0 ** 24)], 1)
    codes, scales = torch.empty(len(g), 1, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(1, len(g), device="cuda")
    K.swiglu_float8(gu, codes, scales, act=act)
    f, units = activation64(g, act)
    check(scales[0], f * 2.0 ** 24, units)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_one_number_a_row_of_a_gated_product(K, act):
    """gate = the row's scale times its sign, up = 256 times that: one k whose codes are 1 and 256, eight columns that are the same."""
    g = gates(act)
    g = g[g.abs() > 1e-2].contiguous()
    M = len(g)
    a = torch.zeros(M, 16, device="cuda")
    a[:, 0] = torch.sign(g)
    w = torch.zeros(16, 16, device="cuda")
    w[:8, 0], w[8:, 0] = 1.0, 256.0
    codes, scales = torch.empty(M, 8, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(1, M, device="cuda")
    K.matmul_swiglu_float8(a.to(E4M3), g.abs().view(1, M).contiguous(), w.to(E4M3), torch.ones(1, 1, device="cuda"), codes, scales, act=act)
    f, units = activation64(g, act)
    check(scales[0], f * 256 * g.double(), units)
    assert K.read_wait_errors() == (0, 0, 0, 0)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("width", [1, 8])
def test_gates_of_any_size(K, act, width):
    """Up to the largest float32 number the activation is the gate, or 0; one that is not finite leaves a block that is none."""
    sizes = [1e2, 1e4, 1e13, 1e20, 2e38, 3.4e38]
    g = torch.tensor(sizes + [-v for v in sizes] + [math.inf, -math.inf, math.nan], device="cuda").view(-1, 1).repeat(1, width)
    gu = torch.cat([g, torch.full_like(g, 2.0 ** -20)], 1)
    codes, scales = torch.empty(len(g), width, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(1, len(g), device="cuda")
    K.swiglu_float8(gu, codes, scales, act=act)
    n = len(sizes)
    check(scales[0, :n], g[:n, 0].double() * 2.0 ** -20, 12)
    assert bool((codes[:n].float() == 448).all()) and bool((codes[n:2 * n].float() == 0).all()) and bool((scales[0, n:2 * n] == 2.0 ** -126).all())
    assert bool(torch.isnan(codes[2 * n:].float()).all()) and bool(torch.isnan(scales[0, 2 * n:]).all())


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("group", [0, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_blocks_of_small_activations(K, act, group, dtype):
    """Gates of -9 to -4 alone in a block (rows of 136: the last eight numbers of each), beside a block of ordinary ones: codes stand for the
    small numbers as well as for any others."""
    T, width = 64, 136
    gen = torch.Generator(device="cuda").manual_seed(3)
    g = torch.randn(T, width, generator=gen, device="cuda")
    g[:, 128:] = -4 - 5 * torch.rand(T, 8, generator=gen, device="cuda")
    u = 1 + torch.rand(T, width, generator=gen, device="cuda")
    g, u = g.to(dtype), u.to(dtype)
    gu = torch.stack([g.view(T, -1, 8), u.view(T, -1, 8)], 2).reshape(T, -1).contiguous() if group else torch.cat([g, u], 1)
    codes, scales = torch.empty(T, width, dtype=torch.uint8, device="cuda").view(E4M3), torch.empty(2, T, device="cuda")
    K.swiglu_float8(gu, codes, scales, group=group, act=act)
    f, units = activation64(g, act)
    y, off = f * u.double(), (f * u.double()).abs() * units * U
    s = scales.t().double().repeat_interleave(128, 1)[:, :width]
    # half a step of e4m3 (2^-4 of the number, 2^-10 where it is subnormal), at most what the number and its scale were off
    far = (codes.double() * s - y).abs() - torch.maximum(y.abs() / 16, s * 2.0 ** -10) * (1 + 2.0 ** -18) - off - y.abs() * 8 * U
    assert bool((far <= 0).all()), float(far.max())
    assert bool((codes.double().abs().view(T, -1)[:, 128:].amax(1) == 448).all())
