"""The product of 8-bit integer rows (mllm_i8_gemm) at the ends of the sizes that it is documented for."""
import pytest
import torch

from mojollama_amd import kernels as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return K.DeviceOps()


@pytest.mark.parametrize("T,R", [(4096, 1 << 22), (4097, (1 << 22) + 33)])
def test_many_results_of_far_rows(dev, T, R):
    """Rows of x at 4 MB (addresses of 64 bits), 1.7 10^10 results: more workgroups than 2^24."""
    C, ld = 16, 1 << 22
    g = torch.Generator(device="cuda").manual_seed(T)
    w = torch.randint(-128, 128, (R, C), dtype=torch.int8, device="cuda", generator=g)
    q = torch.empty(T * ld, dtype=torch.int8, device="cuda").view(T, ld)[:, :C]
    q.copy_(torch.randint(-128, 128, (T, C), dtype=torch.int8, device="cuda", generator=g))
    out = torch.full((T, R), 7.0, dtype=torch.bfloat16, device="cuda")
    dev.i8_gemm(dev.i8_weights(w, torch.ones(R, device="cuda")), q, torch.ones(T, device="cuda"), out=out)
    rows = torch.tensor([0, 1, 31, 32, 2047, 2048, T - 2, T - 1], device="cuda")
    for cols in (slice(0, 4096), slice(R // 2 - 100, R // 2 + 100), slice(R - 4096, R)):
        want = (q[rows].double() @ w[cols].double().T.contiguous()).float().bfloat16()
        assert torch.equal(out[rows, cols], want)
    # every result is written: sums of these products are whole, and 7.0 in a column of a whole tile is none of them all
    assert not (out[:, ::31] == 7.0).all(0).any() and not (out[::31] == 7.0).all(1).any()
    del out, q, w
    torch.cuda.empty_cache()
