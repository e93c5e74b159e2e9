"""The tensor-core product into rows that lie apart: what is behind a row's end is left as it was."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K_", [(2000, 8167, 1032), (2048, 3050, 712), (512, 4099, 2048), (300, 1001, 512), (40, 130, 512)])
def test_nothing_is_written_behind_a_row(M, N, K_, out_dtype):
    from aien_sovereign_core_mv_b200 import kernels as K
    g = torch.Generator(device="cuda").manual_seed(M)
    a = torch.randn(M, K_, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(N, K_, generator=g, device="cuda").to(torch.bfloat16)
    want = a.double() @ w.double().t()
    for ld in ((N + 8) // 8 * 8, N + 1, N):
        whole = torch.full((M, ld), 5.0, dtype=out_dtype, device="cuda")
        K.gemm_tc(a, w, whole[:, :N])
        assert bool((whole[:, N:] == 5.0).all())
        # K products added in float32, then the result's own rounding
        off = (a.double().abs() @ w.double().abs().t()) * K_ * 2.0 ** -24 + want.abs() * (2.0 ** -8 if out_dtype == torch.bfloat16 else 2.0 ** -24)
        assert bool(((whole[:, :N].double() - want).abs() <= off).all())
