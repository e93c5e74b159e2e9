"""Results of products whose rows start on 16-byte borders and end inside a 16-byte word: whole boxes of columns leave by a copy engine that
writes whole words, the last one does not."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
# tiles of one CTA and of pairs, one to a CTA and several
SIZES = [(130, 33), (300, 31), (300, 97), (520, 258), (700, 1301), (2048, 129), (2050, 6151)]


@pytest.fixture(scope="module")
def K():
    from aien_sovereign_core_mv_b200 import kernels
    kernels.lib()
    return kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def into_padded_rows(run, M, N, dtype):
    """The same numbers as in rows that lie close together, and what lies behind them as it was."""
    close = torch.empty(M, N, dtype=dtype, device="cuda")
    run(close)
    for ld in ((N + 8) // 8 * 8, (N + 16) // 8 * 8 + 8):
        whole = torch.full((M + 1, ld), 5.0, dtype=dtype, device="cuda")
        run(whole[:M, :N])
        assert torch.equal(whole[:M, :N], close)
        assert bool((whole[:, N:] == 5.0).all()) and bool((whole[M] == 5.0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N", SIZES)
def test_product_of_codes(K, M, N, dtype):
    width = 400
    code = lambda rows: (torch.randn(rows, width, generator=gen(rows), device="cuda") * 50).clamp(-448, 448).to(E4M3)
    a, w = code(M), code(N)
    sa, sw = 0.5 + torch.rand(4, M, generator=gen(1), device="cuda"), 0.5 + torch.rand(K.float8_blocks(N), 4, generator=gen(2), device="cuda")
    into_padded_rows(lambda out: K.matmul_float8(a, sa, w, sw, out), M, N, dtype)
    assert K.read_wait_errors() == (0, 0, 0, 0)


@pytest.mark.parametrize("M,N", SIZES)
def test_product_in_16_bits(K, M, N):
    a, w = (torch.randn(rows, 456, generator=gen(rows), device="cuda").to(torch.bfloat16) for rows in (M, N))
    into_padded_rows(lambda out: K.gemm_tc(a, w, out), M, N, torch.float32)
    assert K.read_wait_errors() == (0, 0, 0, 0)
