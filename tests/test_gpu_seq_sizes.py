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


@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('dtype', [F64, F32, BF16], ids=str)
def test_long_sequences_of_few_channels(h, dtype, reverse):
    """512 blocks of 8 steps: the join with 16 threads a state, states carried in."""
    acts, par, init = _inputs(30, 4096, 1, 8, 16, dtype=dtype)
    _compare(h, acts, par, init, reverse=reverse)


@pytest.mark.parametrize('dtype', [F64, F32, BF16], ids=str)
def test_many_states_in_many_blocks(h, dtype):
    """131072 states and 14 blocks of 64 steps (a ragged last one): the join with one thread a state, states carried in."""
    acts, par, init = _inputs(40, 840, 4, 2048, 16, dtype=dtype)
    _compare(h, acts, par, init, reverse=dtype == F32)
    torch.cuda.empty_cache()


@pytest.mark.parametrize('dtype', [F16, BF16], ids=str)
def test_packed_rows_of_many_channel_workgroups_with_rows_behind(h, dtype):
    """33 workgroups of channels: gB and gC are sums of 33 partials, of which the rows behind the last sequence have none and stay as they are."""
    import ctypes as C
    from rgp_amd import _lib
    D, N, spare, lengths, fill = 2112, 16, 9, [70, 0, 5, 130], 7.0
    rows, n = sum(lengths), len(lengths)
    off = torch.tensor([0, 70, 70, 75, 205], device='cuda')
    code = _lib.DT_F16 if dtype == F16 else _lib.DT_BF16
    acts, par, init = _inputs(50, rows, 1, D, N, dtype=dtype)
    init = _randn(60, n, D, N)
    behind = lambda t, v: torch.cat([t[:, 0], torch.full((spare,) + t.shape[2:], v, device='cuda', dtype=t.dtype)]).contiguous()      # noqa: E731
    got = None
    for v in (float('nan'), 3.0):
        t = {k: behind(x, v) for k, x in acts.items()}
        o = lambda *s, dt=dtype: torch.full(s, fill, device='cuda', dtype=dt)                                                       # noqa: E731
        out = dict(y=o(rows + spare, D), gu=o(rows + spare, D), gdelta=o(rows + spare, D), gz=o(rows + spare, D), gB=o(rows + spare, 1, N), gC=o(rows + spare, 1, N),
                   gA=o(D, N, dt=F32), gskip=o(D, dt=F32), gbias=o(D, dt=F32), last=o(n, D, N, dt=F32))
        a = _lib.SsmScan()
        a.dtype, a.n_seq, a.D, a.N, a.G, a.rows, a.max_len, a.off = code, n, D, N, 1, rows + spare, 130, off.data_ptr()
        for k, x in dict(out, A=par['A'], skip=par['D'], bias=par['bias'], init=init, u=t['u'], delta=t['delta'], z=t['z'], gy=t['gy'], B=t['B'], C=t['Cm']).items():
            setattr(a, k, x.data_ptr())
        a.u_st = a.delta_st = a.z_st = a.gy_st = D
        a.B_st = a.C_st = N
        states = torch.empty(h.lib.rgp_ssm_scan_states_bytes(C.byref(a)), dtype=torch.uint8, device='cuda')
        a.states = states.data_ptr()
        for back, fn in ((0, h.lib.rgp_ssm_scan_forward), (1, h.lib.rgp_ssm_scan_backward)):
            work = torch.full(((h.lib.rgp_ssm_scan_workspace(C.byref(a), back) + 3) // 4,), v, device='cuda')
            a.work, a.work_bytes = work.data_ptr(), work.numel() * 4
            assert fn(h.h, torch.cuda.current_stream().cuda_stream, C.byref(a)) == 0
        torch.cuda.synchronize()
        if got is not None:
            assert all(torch.equal(got[k], out[k]) for k in out)
        got = out
    assert all(bool((got[k][rows:] == fill).all()) for k in ('y', 'gu', 'gdelta', 'gz', 'gB', 'gC'))
    sums, start = {k: [0, 0] for k in ('gA', 'gD', 'gbias')}, 0
    for i, L in enumerate(lengths):
        cut = slice(start, start + L)
        start += L
        if L == 0:
            assert torch.equal(got['last'][i], init[i])
            continue
        want = seq_batched.scan(**{k: x[cut] for k, x in acts.items()}, **par, init=init[i:i + 1])
        ops = 8 * L + N + D + 64
        for k in ('y', 'gu', 'gdelta', 'gz', 'gB', 'gC'):
            ref.check(k, got[k][cut].unsqueeze(1), *want[k], ops=ops, acc=F32)
        ref.check('last', got['last'][i:i + 1], *want['last'], ops=ops, acc=F32)
        for k in sums:
            sums[k] = [s + w for s, w in zip(sums[k], want[k])]
    for k, t in (('gA', got['gA']), ('gD', got['gskip']), ('gbias', got['gbias'])):
        ref.check(k, t, *sums[k], ops=8 * 130 + N + rows + 64, acc=F32)


def test_clipping_of_many_large_tensors(h):
    """130 MB of all types in 2000 pieces of 64 KB: more pieces than every workgroup adds for itself."""
    from rgp_amd import seq_ops
    sizes = [(20000003, F32), (9999999, BF16), (1500001, F64), (5000000, F16), (1, F64), (0, F32), (32769, F32)]
    grads = [_randn(i, n).to(t) for i, (n, t) in enumerate(sizes)]
    before = [t.double().clone() for t in grads]
    norm = torch.sqrt(sum((t * t).sum() for t in before))
    got = seq_ops.clip_grad_norm(h, grads, 2.5)
    assert abs(float(got) - float(norm)) <= 1e-12 * float(norm)            # 4e7 additions of positive terms in pairs or chains of at most 1e4: below 1e4 half steps
    c = 2.5 / (float(norm) + 1e-6)
    for t, b in zip(grads, before):
        acc, want = ref.acc_of(t.dtype), b * c
        assert bool(((t.double() - want).abs() <= (ref.half(t.dtype) * 1.001 + 2 * ref.half(acc) + 1e-12) * want.abs() + (2.0 ** -25 if t.dtype == F16 else 0)).all())
    torch.cuda.empty_cache()


@pytest.mark.parametrize('n', [20, 300, 3000, 9001])
def test_sums_over_sequences(h, n):
    """The gradient of D is a sum over sequences, by every way the sums have (one thread an output, 16 or 64, rows gathered first).  Where every
    term and partial sum is a number of 32 bits -- multiples of 2^-8 up to 18002 -- it is exact; of positive terms it is off by the additions that
    one of them passes: at most 20 in a chain, or 6 + 7 + 6 and 9 + 14 behind rows gathered by 6, and the 2 steps: below 32 half steps."""
    from rgp_amd import seq_ops
    T, D, N = 2, 70, 4
    delta, B, Cm, A = _randn(1, T, n, D), _randn(2, T, n, N), _randn(3, T, n, N), -torch.ones(D, N, device='cuda')

    def gD(u, gy):
        skip = torch.ones(D, device='cuda', requires_grad=True)
        y = seq_ops.ssm_scan(h, u, delta, A, B, Cm, D=skip)
        g, = torch.autograd.grad(y, skip, gy)
        return g.double(), (u.double() * gy.double()).sum((0, 1))
    got, want = gD(*((torch.round(_randn(i, T, n, D) * 6).clamp(-16, 16) / 16) for i in (4, 5)))
    assert torch.equal(got, want)
    got, want = gD(*(0.5 + 0.5 * torch.rand(T, n, D, device='cuda', generator=torch.Generator(device='cuda').manual_seed(i)) for i in (6, 7)))
    assert bool(((got - want).abs() <= 32 * 2.0 ** -24 * want).all())


@pytest.mark.parametrize('T', [60, 96, 200, 1500])
@pytest.mark.parametrize('dtype', [F64, F32], ids=str)
def test_growing_states_that_begin_late(h, dtype, T):
    """A positive A: a block's decays multiply beyond the type's range, and what enters the blocks is zero -- inputs in the last three steps, gradients
    of the first three -- so states and adjoints are finite wherever the steps one after the other make them so."""
    acts, par, _ = _inputs(70, T, 2, 20, 16, dtype=dtype, carry=False)
    acts['u'][:-3] = 0
    acts['gy'][3:] = 0
    acts['delta'].zero_()
    par = dict(A=torch.full_like(par['A'], 20.0 if dtype == F32 else 160.0), D=par['D'], bias=torch.zeros_like(par['bias']))
    _compare(h, acts, par, None)
    _compare(h, {k: v.flip(0) for k, v in acts.items()}, par, None, reverse=True)


def test_packed_sequences_without_rows_in_many_channels(h):
    """No rows at all, three workgroups of channels: states are handed on and every gradient of a parameter is zero."""
    from rgp_amd import seq_ops
    D, N, seqs = 130, 16, seq_ops.SeqTable(h, [0, 0, 0])
    e = lambda *s: torch.zeros(*s, device='cuda', requires_grad=True)                               # noqa: E731
    A, skip, bias, w = (-_randn(1, D, N).abs()).requires_grad_(True), e(D), e(D), e(D, 4)
    init, cinit = _randn(2, 3, D, N), _randn(3, 3, 3, D)
    u, delta, B, Cm, z = e(0, D), e(0, D), e(0, 1, N), e(0, 1, N), e(0, D)
    y, last = seq_ops.ssm_scan(h, u, delta, A, B, Cm, D=skip, z=z, delta_bias=bias, seqs=seqs, init=init, return_state=True)
    v, clast = seq_ops.ssm_conv(h, u, w, bias, seqs=seqs, init=cinit, return_state=True)
    assert y.shape == v.shape == (0, D) and torch.equal(last, init) and torch.equal(clast, cinit)
    for g in torch.autograd.grad((y, v), (u, delta, A, B, Cm, skip, z, bias, w), (torch.zeros_like(y), torch.zeros_like(v))):
        assert bool((g == 0).all())


def test_a_step_of_very_many_sequences(h):
    """131073 sequences of 2048 channels in one step: the first and the last ones give what they give alone, to the bit."""
    from rgp_amd import seq_ops
    n, D, N, k = 131073, 2048, 4, 40
    ops = [_randn(i, n, w, dtype=BF16) for i, w in enumerate((D, D, N, N))]                       # u, delta, B, C
    A, state = -torch.exp(_randn(7, D, N)), _randn(8, n, D, N)
    parts = [(s, [t[s].clone() for t in ops], state[s].clone()) for s in (slice(0, k), slice(n - k, n))]
    y = seq_ops.ssm_scan_step(h, ops[0], ops[1], A, ops[2], ops[3], None, state)
    for s, (u, delta, B, Cm), st in parts:
        assert torch.equal(y[s], seq_ops.ssm_scan_step(h, u, delta, A, B, Cm, None, st)) and torch.equal(state[s], st)
    del ops, state, y
    torch.cuda.empty_cache()
