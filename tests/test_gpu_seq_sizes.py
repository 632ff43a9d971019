"""The sequence operators at sizes and plans that small cases do not reach: many sequences, many rows, many channels, many blocks of time."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import seq_batched
import seq_reference as ref

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


def _compare(h, acts, par, init, reverse=False, size=None, spare=0):
    """Scan of (T, n, ..) activations forward and backward against the batched 64-bit form."""
    from rgp_amd import seq_ops
    names = [('gu', 'u'), ('gdelta', 'delta'), ('gB', 'B'), ('gC', 'Cm'), ('gz', 'z'), ('gA', 'A'), ('gD', 'D'), ('gbias', 'bias')]
    leaf = {k: v.detach().requires_grad_(True) for k, v in list(acts.items()) + list(par.items()) if k != 'gy' and v is not None}
    y, last = seq_ops.ssm_scan(h, leaf['u'], leaf['delta'], leaf['A'], leaf['B'], leaf['Cm'], D=leaf.get('D'), z=leaf.get('z'), delta_bias=leaf.get('bias'),
                               init=init, reverse=reverse, return_state=True)
    names = [(g, k) for g, k in names if k in leaf]
    got = dict(zip([g for g, _ in names], torch.autograd.grad(y, [leaf[k] for _, k in names], acts['gy'])))
    got.update(y=y, last=last)
    T, n, Dn = acts['u'].shape
    G, N = acts['B'].shape[2:]
    want = seq_batched.scan_in_chunks(size or n, **acts, **par, init=init, reverse=reverse)
    acc = ref.acc_of(acts['u'].dtype)
    for k, t in got.items():                       # 8 roundings a step, the additions over states, channels and (parameters only) rows, 64 elementwise
        ref.check(k, t, *want[k], ops=8 * T + N + Dn // G + 64 + (T * n if k in ('gA', 'gD', 'gbias') else 0), acc=acc)


def _inputs(seed, T, n, D, N, G=1, dtype=F32, z=True, carry=True):
    acc = ref.acc_of(dtype)
    acts = dict(u=_randn(seed, T, n, D, dtype=dtype), delta=_randn(seed + 1, T, n, D, dtype=dtype), B=_randn(seed + 2, T, n, G, N, dtype=dtype),
                Cm=_randn(seed + 3, T, n, G, N, dtype=dtype), z=_randn(seed + 4, T, n, D, dtype=dtype) if z else None, gy=_randn(seed + 5, T, n, D, dtype=dtype))
    par = dict(A=-torch.exp(_randn(seed + 6, D, N)).to(acc), D=_randn(seed + 7, D).to(acc), bias=_randn(seed + 8, D).to(acc) - 2)
    return acts, par, _randn(seed + 9, n, D, N).to(acc) if carry else None


def test_more_sums_over_channels_than_a_launch_has_workgroups(h):
    """gB and gC of 65544 rows, 64 states and 33 workgroups of channels: 131082 workgroups' worth of sums, twice what a launch takes at once."""
    acts, par, init = _inputs(20, 8, 8193, 520, 64)
    _compare(h, acts, par, init, size=1024)
    torch.cuda.empty_cache()


@pytest.mark.parametrize('rows,C', [((1 << 24) + 5, 2), ((1 << 24) + 5, 9), (5000, 16400)])
def test_norms_of_many_rows(h, rows, C):
    """More rows than 2^24: the values and gradients of the rows' own formula."""
    from rgp_amd import seq_ops
    x, r, gy, gh = (_randn(i, rows, C, dtype=BF16) for i in range(4))
    w = _randn(5, C)
    leaf = [t.detach().requires_grad_(True) for t in (x, r, w)]
    y, hid = seq_ops.rms_norm(h, leaf[0], leaf[2], residual=leaf[1])
    gx, gr, gw = torch.autograd.grad((y, hid), leaf, (gy, gh))
    assert torch.equal(gx, gr)
    gw64, gwm = torch.zeros(C, dtype=F64), torch.zeros(C, dtype=F64)
    ops = C + 64                                                  # the additions over a row
    for c in seq_batched.chunks(rows, max(1, (1 << 23) // C)):
        want = ref.rms(x[c].double(), r[c].double(), w.double(), 1e-6, gy[c].double(), gh[c].double())
        for k, t in (('y', y), ('hid', hid), ('gx', gx)):
            ref.check(k, t[c], *(v.cpu() for v in want[k]), ops=ops, acc=F32)
        gw64 += want['gw'][0].cpu()
        gwm += want['gw'][1].cpu()
    ref.check('gw', gw, gw64, gwm, ops=ops + rows, acc=F32)
    torch.cuda.empty_cache()


def test_clipping_by_a_factor_below_the_normal_numbers(h):
    """Gradients near the end of the 32-bit range, and 32-bit gradients beside fp64 ones that are larger still: the factor is not one of 32 bits."""
    from rgp_amd import seq_ops
    for big, most in ((3e38, 1e-3), (1e39, 1.0), (1e70, 1e30)):
        f32, b16 = (torch.linspace(lo, 3e38, n, device='cuda', dtype=F64).to(t) for lo, n, t in ((-3e38, 1003, F32), (1e36, 777, BF16)))
        f64 = torch.full((33,), big, device='cuda', dtype=F64)
        grads = [f32, b16, f64]
        before = [t.double().clone() for t in grads]
        norm = torch.sqrt(sum((t * t).sum() for t in before))
        c = most / (float(norm) + 1e-6)
        assert c < 2.0 ** -126
        got = seq_ops.clip_grad_norm(h, grads, most)
        assert abs(float(got) - float(norm)) <= 1e-12 * float(norm)
        for t, b in zip(grads, before):              # the product's roundings, one in 32 bits and one to the type (half a step of the smallest numbers below the normal ones)
            assert bool(((t.double() - b * c).abs() <= (ref.half(t.dtype) + ref.half(ref.acc_of(t.dtype)) + 1e-12) * (b * c).abs() +
                         (2.0 ** -134 if t.dtype == BF16 else 2.0 ** -150)).all())
