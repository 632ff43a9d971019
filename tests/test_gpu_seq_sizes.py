"""The sequence operators at sizes and plans that small cases do not reach: many sequences, many rows, many channels, many blocks of time."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope='module')
def h():
    from rgp_amd.capi import Handle
    return Handle()


def _randn(seed, *shape, dtype=F32):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randn(*shape, device='cuda', generator=g, dtype=F32).to(dtype)


def test_many_sequences_of_many_channels(h):
    """65536 sequences of two steps in 1024 channels, forward and backward: the first and the last ones give what they give alone, to the bit."""
    from rgp_amd import seq_ops
    T, n, D, N, k = 2, 65536, 1024, 16, 50
    acts = [_randn(i, T, n, w, dtype=BF16) for i, w in enumerate((D, D, N, N, D, D))]                # u, delta, B, C, z, gy
    A, skip = -torch.exp(_randn(7, D, N)), _randn(8, D)

    def run(ts):
        leaves = [t.detach().requires_grad_(True) for t in ts[:5]]
        u, delta, B, Cm, z = leaves
        y, last = seq_ops.ssm_scan(h, u, delta, A, B, Cm, D=skip, z=z, return_state=True)
        return [last, y.detach()] + list(torch.autograd.grad(y, leaves, ts[5]))
    big = run(acts)
    for s in (slice(0, k), slice(n - k, n)):
        small = run([t[:, s] for t in acts])
        assert torch.equal(big[0][s], small[0])
        assert all(torch.equal(a[:, s], b) for a, b in zip(big[1:], small[1:]))
    torch.cuda.empty_cache()
