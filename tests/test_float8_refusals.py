"""What the 8-bit linear layers' entry points refuse, on the CPU: every refusal comes before a launch."""
import pytest
import torch

from aien_sovereign_core_mv_b200 import kernels as K

E4M3 = torch.float8_e4m3fn


def e4m3(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(E4M3)


def product(M=3, N=5, width=200, **put):
    b = K.float8_blocks(width)
    args = dict(a=e4m3(M, width), a_scales=torch.ones(b, M), w=e4m3(N, width), w_scales=torch.ones(K.float8_blocks(N), b), out=torch.empty(M, N))
    args.update(put)
    return K.matmul_float8(**args)


@pytest.mark.parametrize("put,why", [
    (dict(a=torch.zeros(3, 200)), "a is torch.float32"),
    (dict(a=e4m3(4, 200)), "a has shape"),
    (dict(w=e4m3(5, 201)), "w has shape"),
    (dict(w=torch.zeros(5, 200, dtype=torch.uint8).view(torch.float8_e5m2)), "w is torch.float8_e5m2"),
    (dict(a_scales=torch.ones(3, 2)), "a_scales has shape"),
    (dict(a_scales=torch.ones(2, 3, dtype=torch.bfloat16)), "a_scales is"),
    (dict(w_scales=torch.ones(1, 1)), "w_scales has shape"),
    (dict(out=torch.empty(3, 5, dtype=torch.float16)), "out is"),
    (dict(out=torch.empty(5, 3).t()), "out has strides"),
    (dict(a=e4m3(1, 200).expand(3, 200)), "a has strides"),
    (dict(a_scales=torch.ones(3, 2).t()), "a_scales has strides"),
    (dict(a=e4m3(3, 0), w=e4m3(5, 0), a_scales=torch.ones(0, 3), w_scales=torch.ones(1, 0)), "rows of no numbers"),
    (dict(), "CUDA device"),
])
def test_product(put, why):
    with pytest.raises(K.KernelError, match=why):
        product(**put)


@pytest.mark.parametrize("call,why", [
    (lambda: K.quantize_rows_float8(torch.zeros(3, 200, dtype=torch.float16), e4m3(3, 200), torch.ones(2, 3)), "x is torch.float16"),
    (lambda: K.quantize_rows_float8(torch.zeros(3, 201), e4m3(3, 200), torch.ones(2, 3)), "x has shape"),
    (lambda: K.quantize_rows_float8(torch.zeros(3, 400)[:, ::2], e4m3(3, 200), torch.ones(2, 3)), "x has strides"),
    (lambda: K.quantize_rows_float8(torch.zeros(3, 200), e4m3(3, 200), torch.ones(2, 3)), "CUDA device"),
    (lambda: K.swiglu_float8(torch.zeros(3, 200), e4m3(3, 200), torch.ones(2, 3)), "gate_up has shape"),
    (lambda: K.swiglu_float8(torch.zeros(3, 400), e4m3(3, 200), torch.ones(2, 3), act="relu"), "activation 'relu'"),
    (lambda: K.swiglu_float8(torch.zeros(3, 400), e4m3(3, 200), torch.ones(2, 3), group=7), "runs of 7"),
    (lambda: K.swiglu_float8(torch.zeros(3, 401)[:, :400], e4m3(3, 200), torch.ones(2, 3)), "contiguous"),
    (lambda: K.add_rmsnorm_float8(torch.zeros(3, 200, dtype=torch.bfloat16), None, torch.ones(200), 1e-6, e4m3(3, 200), torch.ones(2, 3)), "x is torch.bfloat16"),
    (lambda: K.add_rmsnorm_float8(torch.zeros(3, 201)[:, :200], None, torch.ones(200), 1e-6, e4m3(3, 200), torch.ones(2, 3)), "x must be contiguous"),
    (lambda: K.quantize_blocks_float8(torch.zeros(130, 200), e4m3(130, 200), torch.ones(1, 2)), "scales has shape"),
])
def test_rows_and_blocks(call, why):
    with pytest.raises(K.KernelError, match=why):
        call()


def test_blocks_of():
    assert [K.float8_blocks(n) for n in (0, 1, 128, 129, 4096)] == [0, 1, 1, 2, 32]
