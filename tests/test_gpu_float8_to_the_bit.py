"""Scales and codes of the 8-bit layers to the bit: s = m * (1 / 448) of a block's largest magnitude m, and e4m3(x * (1 / s)), each reciprocal and
each product rounded to float32, at most 448."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3, F32, BF16 = torch.float8_e4m3fn, torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def K():
    from aien_sovereign_core_mv_b200 import kernels
    kernels.lib()
    return kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def padded(v, rows):
    """The largest magnitude of each block of 128 numbers of a row (``rows``), or of 128 x 128."""
    v = v.abs()
    n, k = v.shape
    nb, kb = -(-n // 128), -(-k // 128)
    if rows:
        return torch.nn.functional.pad(v, (0, kb * 128 - k)).view(n, kb, 128).amax(2)
    return torch.nn.functional.pad(v, (0, kb * 128 - k, 0, nb * 128 - n)).view(nb, 128, kb, 128).amax((1, 3))


def scale_by_definition(top):
    return top * torch.tensor(1 / 448, dtype=F32, device="cuda")


def codes_by_definition(x, scale):
        return (x.float() * (1.0 / scale.double()).float()).clamp(-448.0, 448.0).to(E4M3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,width", [(1, 1), (300, 1001), (300, 1000), (2048, 4096)])
def test_rows_to_the_bit(K, dtype, T, width):
    x = (torch.randn(T, width, generator=gen(T + width), device="cuda") * 3).to(dtype)
    codes = torch.full((T, width), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.full((K.float8_blocks(width), T), math.nan, device="cuda")
    K.quantize_rows_float8(x, codes, scales)
    assert torch.equal(scales.t(), scale_by_definition(padded(x.float(), True)))
    want = codes_by_definition(x, scales.t().repeat_interleave(128, 1)[:, :width])
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,width", [(1, 1), (1000, 2060), (640, 264), (1024, 4096)])
def test_blocks_to_the_bit(K, dtype, N, width):
    w = (torch.randn(N, width, generator=gen(N + width), device="cuda") * 0.05).to(dtype)
    codes = torch.full((N, width), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.full((K.float8_blocks(N), K.float8_blocks(width)), math.nan, device="cuda")
    K.quantize_blocks_float8(w, codes, scales)
    assert torch.equal(scales, scale_by_definition(padded(w.float(), False)))
    want = codes_by_definition(w, scales.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :width])
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
