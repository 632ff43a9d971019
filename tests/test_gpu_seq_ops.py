"""The sequence operators on the GPU against the plain 64-bit forms of seq_reference.py, at the sizes, layouts and values where they can go
wrong.  Tolerances are counted there; ``ops`` below is what a product passes through: 8 roundings a step of the longest sequence (forward and
backward chain), the additions over states, over the channels of a group and over all rows, and 64 for the elementwise parts."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

import seq_reference as ref

F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16
ALL = [F64, F32, BF16, F16]


@pytest.fixture(scope='module')
def h():
    from rgp_amd.capi import Handle
    return Handle()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=F64, scale=1.0):
    return (torch.randn(*shape, generator=g, dtype=F64) * scale).to(dtype)


class Problem(object):
    """Inputs on the CPU in their storage types, and the same on the GPU."""

    def __init__(self, dtype, D, N=16, G=1, W=4, T=0, n=1, lengths=None, z=True, skip=True, bias=True, carry=False, reverse=False, seed=0):
        g = _gen(seed)
        acc = ref.acc_of(dtype)
        self.dtype, self.packed, self.reverse, self.carry = dtype, lengths is not None, reverse, carry
        self.lengths = list(lengths) if lengths is not None else [T] * n
        lead = (sum(self.lengths),) if self.packed else (T, n)
        n = len(self.lengths)
        self.acts = dict(x=_randn(g, *lead, D, dtype=dtype), u=_randn(g, *lead, D, dtype=dtype), delta=_randn(g, *lead, D, dtype=dtype),
                         B=_randn(g, *lead, G, N, dtype=dtype), C=_randn(g, *lead, G, N, dtype=dtype), z=_randn(g, *lead, D, dtype=dtype) if z else None,
                         gy=_randn(g, *lead, D, dtype=dtype), gv=_randn(g, *lead, D, dtype=dtype))
        self.par = dict(w=_randn(g, D, W, dtype=acc, scale=0.5), b=_randn(g, D, dtype=acc, scale=0.5) if bias else None,
                        A=-torch.exp(_randn(g, D, N)).to(acc), D=_randn(g, D, dtype=acc) if skip else None,
                        bias=_randn(g, D, dtype=acc) - 2 if bias else None)
        self.cstate = _randn(g, n, W - 1, D, dtype=dtype) if carry else None
        self.state = _randn(g, n, D, N, dtype=acc) if carry else None
        self.ops = 8 * max(self.lengths + [1]) + N + D // G + sum(self.lengths) + 64

    def dev(self, t, grad=False):
        if t is None:
            return None
        t = t.cuda()
        return t.requires_grad_(True) if grad else t

    def seqs(self, h):
        from rgp_amd import seq_ops
        return seq_ops.SeqTable(h, self.lengths) if self.packed else None

    def reference(self):
        d = lambda t: None if t is None else t.double()                       # noqa: E731
        a, p = self.acts, self.par
        conv = ref.by_sequence(ref.conv_one, dict(x=d(a['x']), gv=d(a['gv'])), dict(init=d(self.cstate)), self.lengths, self.packed, self.reverse,
                               ('v', 'gx'), ('gw', 'gb'), dict(w=d(p['w']), bias=d(p['b'])))
        scan = ref.by_sequence(ref.scan_one, dict(u=d(a['u']), delta=d(a['delta']), B=d(a['B']), Cm=d(a['C']), z=d(a['z']), gy=d(a['gy'])),
                               dict(init=d(self.state)), self.lengths, self.packed, self.reverse, ('y', 'gu', 'gdelta', 'gz', 'gB', 'gC'),
                               ('gA', 'gD', 'gbias'), dict(A=d(p['A']), D=d(p['D']), bias=d(p['bias'])))
        return conv, scan

    def run(self, h, spread=None):
        """All outputs of both operators and their gradients; ``spread`` lays an activation out another way."""
        from rgp_amd import seq_ops
        seqs = self.seqs(h)
        lay = spread or (lambda t: t)
        a = {k: None if v is None else lay(v.cuda()).requires_grad_(k[0] != 'g') for k, v in self.acts.items()}
        p = {k: self.dev(v, True) for k, v in self.par.items()}
        cst, st = self.dev(self.cstate), self.dev(self.state)
        v, clast = seq_ops.ssm_conv(h, a['x'], p['w'], p['b'], seqs=seqs, init=cst, reverse=self.reverse, return_state=True)
        y, last = seq_ops.ssm_scan(h, a['u'], a['delta'], p['A'], a['B'], a['C'], D=p['D'], z=a['z'], delta_bias=p['bias'], seqs=seqs, init=st,
                                   reverse=self.reverse, return_state=True)
        conv, scan = dict(v=v, last=clast), dict(y=y, last=last)
        names = [('gx', a['x']), ('gw', p['w']), ('gb', p['b'])]
        names = [(k, t) for k, t in names if t is not None]
        conv.update(zip([k for k, _ in names], torch.autograd.grad(v, [t for _, t in names], a['gv'])))
        names = [('gu', a['u']), ('gdelta', a['delta']), ('gA', p['A']), ('gB', a['B']), ('gC', a['C']), ('gD', p['D']), ('gz', a['z']), ('gbias', p['bias'])]
        names = [(k, t) for k, t in names if t is not None]
        scan.update(zip([k for k, _ in names], torch.autograd.grad(y, [t for _, t in names], a['gy'])))
        return conv, scan

    def compare(self, got, want):
        acc = ref.acc_of(self.dtype)
        for g, w in zip(got, want):
            for k, t in g.items():
                ref.check(k, t, *w[k], ops=self.ops, acc=acc)


CASES = [
    dict(D=5, N=3, T=1, n=1), dict(D=1, N=1, T=2, n=3, W=2), dict(D=16, N=16, T=17, n=2, carry=True), dict(D=70, N=16, T=33, n=2, reverse=True, carry=True),
    dict(D=24, N=4, G=3, T=40, n=2, W=3, z=False), dict(D=130, N=8, T=9, n=2, skip=False, bias=False), dict(D=66, N=5, G=2, T=21, n=3, carry=True, W=8),
    dict(D=40, N=17, T=19, n=2), dict(D=33, N=32, T=35, n=1, carry=True, z=False), dict(D=20, N=64, G=4, T=18, n=2, carry=True), dict(D=17, N=33, T=5, n=2, reverse=True),
    dict(D=40, N=16, lengths=[3, 0, 1, 37, 16, 0], carry=True), dict(D=72, N=12, G=2, lengths=[1, 1, 1, 50], reverse=True, W=5), dict(D=8, N=2, lengths=[0, 31], carry=True, W=7),
    dict(D=9, N=7, T=300, n=1, carry=True), dict(D=6, N=16, G=2, lengths=[290, 5, 64, 0, 130], carry=True, reverse=True), dict(D=130, N=6, T=260, n=1, W=6),
    dict(D=12, N=16, lengths=[0, 0], carry=True),
]


@pytest.mark.parametrize('dtype', ALL, ids=str)
@pytest.mark.parametrize('i', range(len(CASES)))
def test_conv_and_scan_forward_backward(h, i, dtype):
    p = Problem(dtype, seed=100 + i, **CASES[i])
    p.compare(p.run(h), p.reference())


@pytest.mark.parametrize('dtype', [F64, BF16], ids=str)
def test_strided_operands(h, dtype):
    """Column slices of wider rows at an odd offset, batch-first memory, and features that are not contiguous (copied)."""
    p = Problem(dtype, D=24, N=16, G=2, T=21, n=3, carry=True, seed=5)
    want = p.reference()

    def wide(t):
        buf = torch.full(t.shape[:-1] + (t.shape[-1] + 7,), float('nan'), dtype=t.dtype, device=t.device)
        o = buf[..., 3:3 + t.shape[-1]]
        o.copy_(t)
        return o.detach()
    p.compare(p.run(h, lambda t: wide(t) if t.dim() == 3 else t.detach()), want)
    p.compare(p.run(h, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1).detach()), want)
    p.compare(p.run(h, lambda t: t.transpose(0, 2).contiguous().transpose(0, 2).detach()), want)
    q = Problem(dtype, D=24, N=16, lengths=[7, 0, 30], carry=True, seed=6)
    q.compare(q.run(h, lambda t: wide(t) if t.dim() == 2 else t.detach()), q.reference())


@pytest.mark.parametrize('dtype', [F64, F32, BF16], ids=str)
def test_steps_continue_a_prompt(h, dtype):
    """A prompt, then single steps from its states: every step is the prompt's own next row, and the states end as the whole prompt's."""
    from rgp_amd import seq_ops
    T, n, D, N, G, W, T0 = 12, 3, 18, 16, 2, 4, 7
    p = Problem(dtype, D=D, N=N, G=G, T=T, n=n, W=W, seed=3)
    a = {k: None if v is None else v.cuda() for k, v in p.acts.items()}
    q = {k: p.dev(v) for k, v in p.par.items()}
    scan = lambda s, **k: seq_ops.ssm_scan(h, a['u'][s], a['delta'][s], q['A'], a['B'][s], a['C'][s], D=q['D'], z=a['z'][s], delta_bias=q['bias'], return_state=True, **k)    # noqa: E731
    want = p.reference()
    v0, cst = seq_ops.ssm_conv(h, a['x'][:T0], q['w'], q['b'], return_state=True)
    y0, st = scan(slice(0, T0))
    vs, ys = [v0], [y0]
    for t in range(T0, T - 2):
        vs.append(seq_ops.ssm_conv_step(h, a['x'][t], q['w'], q['b'], cst).unsqueeze(0))
        ys.append(seq_ops.ssm_scan_step(h, a['u'][t], a['delta'][t], q['A'], a['B'][t], a['C'][t], q['D'], st, z=a['z'][t], delta_bias=q['bias']).unsqueeze(0))
    v1, cst = seq_ops.ssm_conv(h, a['x'][T - 2:], q['w'], q['b'], init=cst, return_state=True)        # and a chunk again behind the steps
    y1, st = scan(slice(T - 2, T), init=st)
    p.compare((dict(v=torch.cat(vs + [v1]), last=cst), dict(y=torch.cat(ys + [y1]), last=st)), want)
    for N2 in (1, 4, 7, 20, 40, 64):                                                                  # every width of the step kernel
        r = Problem(dtype, D=10, N=N2, T=1, n=2, carry=True, z=N2 != 7, skip=N2 != 4, bias=N2 != 1, seed=N2)
        b = {k: None if v is None else v.cuda()[0] for k, v in r.acts.items()}
        q2, c2, s2 = {k: r.dev(v) for k, v in r.par.items()}, r.dev(r.cstate), r.dev(r.state)
        v = seq_ops.ssm_conv_step(h, b['x'], q2['w'], q2['b'], c2)
        y = seq_ops.ssm_scan_step(h, b['u'], b['delta'], q2['A'], b['B'], b['C'], q2['D'], s2, z=b['z'], delta_bias=q2['bias'])
        r.compare((dict(v=v.unsqueeze(0), last=c2), dict(y=y.unsqueeze(0), last=s2)), r.reference())


def test_same_bits_every_time_and_no_shared_buffers(h):
    """Two problems interleaved on two streams, the second run of each equal to the first to the last bit."""
    a, b = Problem(BF16, D=96, N=16, T=300, n=2, seed=1), Problem(F32, D=20, N=9, lengths=[280, 3], carry=True, seed=2)
    flat = lambda r: [t.detach().clone() for o in r for t in o.values()]          # noqa: E731
    first = flat(a.run(h)), flat(b.run(h))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        ra = flat(a.run(h))
    with torch.cuda.stream(s2):
        rb = flat(b.run(h))
    torch.cuda.synchronize()
    for x, y in zip(first[0] + first[1], ra + rb):
        assert torch.equal(x, y)


def test_nan_and_infinities_stay_where_they_belong(h):
    """A NaN in one channel of one sequence leaves the other sequences and, forward, the other channels as they were; a step of minus
    infinity (dt = 0) keeps the state; A of minus infinity forgets it."""
    from rgp_amd import seq_ops
    p = Problem(F32, D=20, N=16, lengths=[40, 33, 21], seed=8)
    clean = p.run(h)
    p.acts['u'][45, 3] = float('nan')
    p.acts['x'][45, 3] = float('nan')
    dirty = p.run(h)
    for k, o, d in (('v', clean[0], dirty[0]), ('y', clean[1], dirty[1])):
        bad = torch.isnan(d[k])
        assert bool(bad[45, 3]) and not bool(bad[:45].any()) and not bool(bad[73:].any()) and not bool(bad[:, :3].any()) and not bool(bad[:, 4:].any())
        assert torch.equal(o[k][~bad], d[k][~bad])
    for k in ('gu', 'gdelta', 'gz', 'gB', 'gC'):
        assert torch.equal(clean[1][k][:40], dirty[1][k][:40]) and torch.equal(clean[1][k][73:], dirty[1][k][73:])
    T, D, N = 37, 5, 3
    g = _gen(1)
    u, B, Cm = (_randn(g, T, 1, m, dtype=F32).cuda() for m in (D, N, N))
    delta = torch.zeros(T, 1, D, device='cuda')
    delta[10:20] = float('-inf')
    A = -torch.ones(D, N, device='cuda')
    A[2] = float('-inf')
    st = _randn(g, 1, D, N, dtype=F32).cuda()
    _, at10 = seq_ops.ssm_scan(h, u[:10], delta[:10], A, B[:10], Cm[:10], init=st, return_state=True)
    _, at20 = seq_ops.ssm_scan(h, u[:20], delta[:20], A, B[:20], Cm[:20], init=st, return_state=True)
    live = [d for d in range(D) if d != 2]                       # 0 times minus infinity has no value
    assert torch.equal(at10[:, live], at20[:, live])
    y, end = seq_ops.ssm_scan(h, u[:9], delta[:9], A, B[:9], Cm[:9], init=st, return_state=True)
    own = torch.log1p(torch.exp(torch.zeros((), dtype=F64))) * u[8, 0, 2].double().cpu() * B[8, 0].double().cpu()
    assert torch.allclose(end[0, 2].double().cpu(), own, rtol=1e-6, atol=0)
    big = torch.full((3, 1, D), 88.0, device='cuda')              # large steps: softplus is the identity, the decay is 0, nothing overflows
    y, end = seq_ops.ssm_scan(h, u[:3], big, A, B[:3], Cm[:3], return_state=True)
    assert torch.allclose(end[0, 0].cpu(), (88.0 * u[2, 0, 0] * B[2, 0]).cpu(), rtol=1e-6)


def test_scan_gradients_match_differences(h):
    from rgp_amd import seq_ops
    p = Problem(F64, D=6, N=5, G=2, T=20, n=2, carry=True, seed=4)
    conv, scan = p.run(h)
    a = {k: v.cuda() for k, v in p.acts.items()}
    q = {k: p.dev(v) for k, v in p.par.items()}

    def f(**kw):
        o = {**{k: a[k] for k in ('u', 'delta', 'B', 'C', 'z')}, **{k: q[k] for k in ('A', 'D', 'bias')}, **kw}
        y = seq_ops.ssm_scan(h, o['u'], o['delta'], o['A'], o['B'], o['C'], D=o['D'], z=o['z'], delta_bias=o['bias'], init=p.state.cuda())
        return float((y * a['gy']).sum())
    for k, g in (('u', 'gu'), ('delta', 'gdelta'), ('B', 'gB'), ('C', 'gC'), ('z', 'gz'), ('A', 'gA'), ('D', 'gD'), ('bias', 'gbias')):
        t = {**a, **q}[k]
        d = _randn(_gen(7), *t.shape).cuda()
        e = 1e-5
        num = (f(**{k: t + e * d}) - f(**{k: t - e * d})) / (2 * e)
        assert abs(num - float((scan[g] * d).sum())) <= 1e-6 * max(1.0, abs(num)), (k, num)       # e^2 = 1e-10 of the third derivative, 1e-16 / e of rounding


def test_broadcast_and_shared_operands(h):
    """Operands with stride 0, one tensor as two operands, and gradients summed over what was broadcast."""
    from rgp_amd import seq_ops
    T, n, D, N = 19, 3, 8, 16
    g = _gen(0)
    u, delta = _randn(g, T, n, D).cuda().requires_grad_(True), _randn(g, T, 1, D).cuda().requires_grad_(True)
    B, A = _randn(g, T, 1, 1, N).cuda().requires_grad_(True), -torch.rand(D, N, generator=g, dtype=F64).cuda()
    gy = _randn(g, T, n, D).cuda()
    Bx = B.expand(T, n, 2, N)
    y = seq_ops.ssm_scan(h, u, delta.expand(T, n, D), A, Bx, Bx, z=u)
    got = torch.autograd.grad(y, (u, delta, B), gy)
    u2, d2, b2 = (t.detach().clone().requires_grad_(True) for t in (u, delta, B))
    full = lambda t, *s: t.expand(*s).contiguous()                        # noqa: E731
    y2 = seq_ops.ssm_scan(h, u2, full(d2, T, n, D), A, full(b2, T, n, 2, N), full(b2, T, n, 2, N), z=u2.clone())
    want = torch.autograd.grad(y2, (u2, d2, b2), gy)
    assert torch.equal(y, y2)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-12)


def test_states_updated_in_place_are_noticed(h):
    """A graph that saved a state refuses its backward pass once a step has changed it; steps refuse operands that want gradients."""
    from rgp_amd import seq_ops
    from rgp_amd._lib import RgpError
    w = torch.randn(6, 4, device='cuda', requires_grad=True)
    x, st = torch.randn(5, 2, 6, device='cuda'), torch.randn(2, 3, 6, device='cuda')
    v = seq_ops.ssm_conv(h, x, w, init=st)
    with pytest.raises(RgpError, match='no gradients'):
        seq_ops.ssm_conv_step(h, x[0], w, None, st)
    seq_ops.ssm_conv_step(h, x[0], w.detach(), None, st)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        v.sum().backward()


def test_rows_beyond_2_31_elements(h):
    """Packed rows whose last sequence lies behind 2^31 elements, forward and backward: it gives what it gives alone."""
    from rgp_amd import seq_ops
    D, N, tail = 2048, 2, 70
    rows = (1 << 31) // D + 4000
    g = torch.Generator(device='cuda').manual_seed(0)
    f = lambda *s: torch.randn(*s, device='cuda', generator=g, dtype=F32).to(BF16)          # noqa: E731
    big = {k: torch.zeros(rows, w, device='cuda', dtype=BF16) for k, w in (('x', D), ('u', D), ('delta', D), ('B', N), ('C', N), ('gy', D))}
    for t in big.values():
        t[-3 * tail:] = f(3 * tail, t.shape[1])
    A, w, ws = -torch.rand(D, N, device='cuda') - 0.1, torch.randn(D, 4, device='cuda'), torch.rand(D, device='cuda')

    def run(t, lengths):
        s = seq_ops.SeqTable(h, lengths)
        leaves = [t[k].detach().requires_grad_(True) for k in ('x', 'u', 'delta', 'B', 'C')]
        x, u, delta, B, Cm = leaves
        v = seq_ops.ssm_conv(h, x, w, seqs=s)
        y = seq_ops.ssm_scan(h, u, delta, A, B, Cm, z=v, seqs=s)
        n, hid = seq_ops.rms_norm(h, y, ws, residual=v)
        return [o.detach()[-tail:].float() for o in (v, y, n, hid)] + [o[-tail:].float() for o in torch.autograd.grad((n, hid), leaves, (t['gy'], t['gy']))]
    got = run(big, [rows - 3 * tail, 2 * tail, tail])
    want = run({k: t[-tail:].clone() for k, t in big.items()}, [tail])
    for a, b in zip(got, want):                                              # the same roundings except for the order of sums over channels
        assert float((a - b).norm()) <= 1e-2 * float(b.norm())
    del big
    torch.cuda.empty_cache()


def test_graph_capture_of_forward_and_backward(h):
    """Forward and backward in one captured region, replayed with new inputs and with eager work between the replays."""
    from rgp_amd import seq_ops
    probs = [Problem(BF16, D=72, N=16, T=270, n=2, seed=s) for s in (1, 2, 3)]
    st = {k: v.cuda().requires_grad_(k[0] != 'g') for k, v in probs[0].acts.items()}
    pa = {k: v.cuda().requires_grad_(True) for k, v in probs[0].par.items()}

    def region():
        v = seq_ops.ssm_conv(h, st['x'], pa['w'], pa['b'])
        y = seq_ops.ssm_scan(h, st['u'], st['delta'], pa['A'], st['B'], st['C'], D=pa['D'], z=st['z'], delta_bias=pa['bias'])
        n, hid = seq_ops.rms_norm(h, y, pa['D'], residual=v)
        g = torch.autograd.grad((n, hid), [st[k] for k in ('x', 'u', 'delta', 'B', 'C', 'z')] + list(pa.values()), (st['gy'], st['gv']))
        grads = [t.clone() for t in g]
        norm = seq_ops.clip_grad_norm(h, grads, 0.5)
        return [v.detach(), y.detach(), n.detach(), hid.detach(), norm] + grads
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        region()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = region()
    for p in (probs[1], probs[2], probs[0], probs[1]):
        with torch.no_grad():
            for k, v in p.acts.items():
                st[k].copy_(v)
            for k, v in p.par.items():
                pa[k].copy_(v)
        graph.replay()
        got = [t.clone() for t in out]
        want = region()                                             # eager work between the replays, same inputs
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


# ---------------------------------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize('dtype', ALL, ids=str)
@pytest.mark.parametrize('rows,C', [(1, 1), (3, 7), (130, 40), (9, 64), (5, 513), (7, 2048), (3, 2050), (2, 9001), (3, 20011), (2500, 16)])
@pytest.mark.parametrize('residual', [True, False])
def test_rms_norm(h, dtype, rows, C, residual):
    from rgp_amd import seq_ops
    g = _gen(rows * C)
    x, r, gy, gh = (_randn(g, rows, C, dtype=dtype) for _ in range(4))
    w = _randn(g, C, dtype=ref.acc_of(dtype))
    x[0] = 0
    r[0] = 0                                                       # a row of zeros
    lx, lr, lw = x.cuda().requires_grad_(True), r.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    d = lambda t: t.double()                                      # noqa: E731
    want = ref.rms(d(x), d(r) if residual else None, d(w), 1e-6, d(gy), d(gh) if residual else None)
    ops = C + rows + 64                                           # the additions over a row and over the rows
    if residual:
        y, hid = seq_ops.rms_norm(h, lx, lw, residual=lr)
        gx, gr, gw = torch.autograd.grad((y, hid), (lx, lr, lw), (gy.cuda(), gh.cuda()))
        ref.check('hid', hid, *want['hid'], ops=ops)
        assert torch.equal(gx, gr)
    else:
        y = seq_ops.rms_norm(h, lx, lw)
        gx, gw = torch.autograd.grad(y, (lx, lw), gy.cuda())
    ref.check('y', y, *want['y'], ops=ops)
    ref.check('gx', gx, *want['gx'], ops=ops, acc=ref.acc_of(dtype))
    ref.check('gw', gw, *want['gw'], ops=ops, acc=ref.acc_of(dtype))


def test_rms_norm_layouts_and_partial_gradients(h):
    from rgp_amd import seq_ops
    g = _gen(3)
    w = _randn(g, 24, dtype=F32).cuda().requires_grad_(True)
    big = _randn(g, 6, 5, 60, dtype=F32).cuda()
    x, r = big[..., 1:25].detach().requires_grad_(True), big.transpose(0, 1)[..., 30:54].transpose(0, 1).detach().requires_grad_(True)
    y, hid = seq_ops.rms_norm(h, x, w, residual=r, eps=1e-3)
    yc, hc = seq_ops.rms_norm(h, x.contiguous(), w, residual=r.contiguous(), eps=1e-3)
    assert torch.equal(y, yc) and torch.equal(hid, hc) and y.shape == x.shape
    gy = _randn(g, 6, 5, 24, dtype=F32).cuda()
    only_h = torch.autograd.grad(hid, (x, r), gy, retain_graph=True)
    assert torch.equal(only_h[0], gy) and torch.equal(only_h[1], gy)
    only_y = torch.autograd.grad(y, (x, w), gy, retain_graph=True)
    both = torch.autograd.grad((y, hid), (x, w), (gy, torch.zeros_like(gy)))
    assert torch.equal(only_y[0], both[0]) and torch.equal(only_y[1], both[1])
    e = torch.zeros(0, 24, device='cuda', requires_grad=True)
    ye, he = seq_ops.rms_norm(h, e, w, residual=e)
    ge, gwe = torch.autograd.grad((ye, he), (e, w), (torch.zeros_like(ye), torch.zeros_like(he)))
    assert ye.shape == (0, 24) and bool((gwe == 0).all())
    n = torch.full((2, 24), float('nan'), device='cuda')
    n[1] = 1
    yn = seq_ops.rms_norm(h, n, w.detach())
    assert bool(torch.isnan(yn[0]).all()) and bool(torch.isfinite(yn[1]).all())


# ---------------------------------------------------------------------------------------------------------------------- gradient norm
def test_clip_many_tensors_of_all_types(h):
    from rgp_amd import seq_ops
    g = _gen(0)
    sizes = [0, 1, 3, 7, 64, 100003, 40000, 33, 8, 0, 65536, 2] + [(i * 37) % 211 for i in range(300)]
    flat = {t: _randn(g, sum(sizes) + 64, dtype=t).cuda() for t in ALL}
    grads, off = [], 1
    for i, n in enumerate(sizes):                                  # views at odd offsets of four buffers
        grads.append(flat[ALL[i % 4]][off:off + n])
        off += n
    grads.append(torch.ones(5, 7, device='cuda').t())              # dense in another order
    before = [x.clone() for x in grads]
    keep = {t: f.clone() for t, f in flat.items()}
    norm64 = torch.sqrt(sum(x.double().square().sum() for x in before))
    norm = seq_ops.clip_grad_norm(h, grads, 1.5)
    assert norm.dtype == F64 and norm.dim() == 0
    assert abs(float(norm) - float(norm64)) <= 1e-12 * float(norm64)          # 1e6 additions of positive terms in pairs: below 1e4 half steps
    c = 1.5 / (float(norm64) + 1e-6)
    for b, x in zip(before, grads):
        acc = ref.acc_of(x.dtype)
        want = b.double() * c
        assert bool(((x.double() - want).abs() <= ref.half(x.dtype) * want.abs() * 1.001 + 4 * ref.half(acc) * want.abs() + (2.0 ** -25 if x.dtype == F16 else 0)).all())
    touched = {t: torch.zeros_like(f, dtype=torch.bool) for t, f in flat.items()}
    off = 1
    for i, n in enumerate(sizes):
        touched[ALL[i % 4]][off:off + n] = True
        off += n
    for t in ALL:
        assert torch.equal(flat[t][~touched[t]], keep[t][~touched[t]])         # nothing beside the tensors moved


def test_clip_below_the_threshold_and_without_a_finite_norm(h):
    from rgp_amd import seq_ops
    for t in ALL:
        x = torch.linspace(-1, 1, 1001, device='cuda').to(t)
        k = x.clone()
        norm = seq_ops.clip_grad_norm(h, [x], 1e6)
        assert torch.equal(x, k) and abs(float(norm) - float(k.double().norm())) < 1e-9
        for bad in (float('nan'), float('inf')):
            x[500] = bad
            k = x.clone()
            norm = seq_ops.clip_grad_norm(h, [x], 1e-3)
            assert torch.equal(x.nan_to_num(7.0), k.nan_to_num(7.0)) and not bool(torch.isfinite(norm))
    x = torch.full((3, 5), 1e30, device='cuda')                    # squares that 32 bits do not hold
    assert abs(float(seq_ops.clip_grad_norm(h, [x], 1.0)) / (1e30 * 15 ** 0.5) - 1) < 1e-6
    assert torch.allclose(x, torch.full_like(x, 15 ** -0.5), rtol=1e-6)
    z = torch.zeros(9, device='cuda')
    assert float(seq_ops.clip_grad_norm(h, [z], 1.0)) == 0.0 and float(seq_ops.clip_grad_norm(h, [], 1.0)) == 0.0
    y = torch.ones(16, device='cuda')                              # sums of squares of other ranks
    total = seq_ops.grad_sumsq(h, [y]) * 4
    assert float(seq_ops.clip_grad_norm(h, [y], 4.0, sumsq=total)) == 8.0 and torch.allclose(y, torch.full_like(y, 0.5), rtol=1e-6)


def test_second_derivatives_are_refused(h):
    from rgp_amd import seq_ops
    x = torch.randn(3, 4, device='cuda', requires_grad=True)
    with pytest.raises(RuntimeError, match='second derivatives'):
        torch.autograd.grad(seq_ops.rms_norm(h, x, torch.ones(4, device='cuda')).sum(), x, create_graph=True)


def test_library_refuses_what_python_would_not_send(h):
    """The C entries check by themselves: sizes, missing buffers, a work buffer that is too small."""
    from rgp_amd import _lib
    a = _lib.SsmScan()
    a.dtype, a.n_seq, a.D, a.N, a.G, a.T, a.rows, a.max_len = _lib.DT_F32, 1, 4, 4, 1, 3, 3, 3
    t = torch.zeros(64, device='cuda')
    assert h.lib.rgp_ssm_scan_forward(h.h, None, C.byref(a)) == _lib.RGP_ERR_BAD_ARG
    for f in ('u', 'delta', 'B', 'C', 'A', 'y', 'gy', 'states', 'gu', 'gdelta', 'gB', 'gC', 'gA'):
        setattr(a, f, t.data_ptr())
    assert h.lib.rgp_ssm_scan_backward(h.h, None, C.byref(a)) == _lib.RGP_ERR_WORKSPACE
    a.rows = 4
    assert h.lib.rgp_ssm_scan_forward(h.h, None, C.byref(a)) == _lib.RGP_ERR_BAD_ARG and b'rows' in h.lib.rgp_last_error(h.h)
    c = _lib.SsmConv()
    c.dtype, c.n_seq, c.D, c.W, c.T, c.rows = _lib.DT_F32, 1, 4, 4, 3, 3
    c.x = c.w = c.v = t.data_ptr()
    c.init = c.last = t.data_ptr()
    assert h.lib.rgp_ssm_conv_forward(h.h, None, C.byref(c)) == _lib.RGP_ERR_BAD_ARG
    assert h.lib.rgp_grad_clip(h.h, None, 0, None, None, None, t.data_ptr(), 0.0, t.data_ptr() + 8, None, 0) == _lib.RGP_ERR_BAD_ARG


@pytest.mark.parametrize('D,reverse', [(130, False), (16, True)])
def test_rows_behind_the_last_sequence_stay_as_they_are(h, D, reverse):
    """Packed rows may have capacity behind off[n_seq] (a table that is refilled between replays): nothing of it is read or written, also by
    the sums over the channels' workgroups, and the rows of the sequences are right."""
    from rgp_amd import _lib
    N, spare = 16, 77
    p = Problem(F32, D=D, N=N, lengths=[70, 0, 5, 130], skip=False, bias=False, reverse=reverse, seed=11)
    rows, n = sum(p.lengths), len(p.lengths)
    off = torch.tensor([0, 70, 70, 75, 205], device='cuda')
    A, w = p.par['A'].cuda(), p.par['w'].cuda()
    st = torch.cuda.current_stream().cuda_stream

    def run(behind):
        acts = {k: torch.cat([t.cuda(), torch.full((spare,) + t.shape[1:], behind, device='cuda')]) for k, t in p.acts.items()}
        out = lambda *s: torch.full(s, 7.0, device='cuda')                                                   # noqa: E731
        scan = dict(y=out(rows + spare, D), gu=out(rows + spare, D), gdelta=out(rows + spare, D), gz=out(rows + spare, D), gB=out(rows + spare, 1, N),
                    gC=out(rows + spare, 1, N), gA=out(D, N))
        a = _lib.SsmScan()
        a.dtype, a.n_seq, a.D, a.N, a.G, a.reverse, a.rows, a.max_len, a.off = _lib.DT_F32, n, D, N, 1, int(reverse), rows + spare, 130, off.data_ptr()
        for k, t in dict(scan, A=A, **{k: acts[k] for k in ('u', 'delta', 'z', 'gy', 'B', 'C')}).items():
            setattr(a, k, t.data_ptr())
        a.u_st = a.delta_st = a.z_st = a.gy_st = D
        a.B_st = a.C_st = N
        states = torch.empty(h.lib.rgp_ssm_scan_states_bytes(C.byref(a)), dtype=torch.uint8, device='cuda')
        a.states = states.data_ptr()
        for back, fn in ((0, h.lib.rgp_ssm_scan_forward), (1, h.lib.rgp_ssm_scan_backward)):
            work = torch.full((h.lib.rgp_ssm_scan_workspace(C.byref(a), back) // 4,), behind, device='cuda')
            a.work, a.work_bytes = work.data_ptr(), work.numel() * 4
            assert fn(h.h, st, C.byref(a)) == 0
        conv = dict(v=out(rows + spare, D), gx=out(rows + spare, D), gw=out(D, 4))
        c = _lib.SsmConv()
        c.dtype, c.n_seq, c.D, c.W, c.reverse, c.rows, c.max_len, c.off = _lib.DT_F32, n, D, 4, int(reverse), rows + spare, 130, off.data_ptr()
        for k, t in dict(conv, x=acts['x'], gv=acts['gv'], w=w).items():
            setattr(c, k, t.data_ptr())
        c.x_st = c.gv_st = D
        assert h.lib.rgp_ssm_conv_forward(h.h, st, C.byref(c)) == 0
        work = torch.full((h.lib.rgp_ssm_conv_workspace(C.byref(c), 1) // 4,), behind, device='cuda')
        c.work, c.work_bytes = work.data_ptr(), work.numel() * 4
        assert h.lib.rgp_ssm_conv_backward(h.h, st, C.byref(c)) == 0
        torch.cuda.synchronize()
        return conv, scan

    got, other = run(float('nan')), run(3.0)
    for g, o in zip(got, other):
        for k in g:
            assert torch.equal(g[k], o[k]), k
            if g[k].shape[0] == rows + spare:
                assert (g[k][rows:] == 7.0).all(), k
    p.compare([{k: t[:rows] if t.shape[0] == rows + spare else t for k, t in g.items()} for g in got], p.reference())


def test_steps_with_infinite_decay(h):
    """A = -inf forgets the state, also where a step's dt underflows to zero (then nothing decays), as over whole sequences."""
    from rgp_amd import seq_ops
    g, D, N = _gen(12), 6, 4
    u, B, Cm = _randn(g, 2, D, dtype=F32).cuda(), _randn(g, 2, N, dtype=F32).cuda(), _randn(g, 2, N, dtype=F32).cuda()
    A = torch.full((D, N), -float('inf'), device='cuda')
    s0 = _randn(g, 2, D, N, dtype=F32).cuda()
    for value in (0.5, -300.0):
        delta = torch.full((2, D), value, device='cuda')
        st = s0.clone()
        y = seq_ops.ssm_scan_step(h, u, delta, A, B, Cm, None, st)
        y1, last = seq_ops.ssm_scan(h, u[None], delta[None], A, B[None], Cm[None], init=s0, return_state=True)
        assert torch.isfinite(st).all() and torch.isfinite(y).all()
        if value < 0:
            assert torch.equal(st, s0)
        torch.testing.assert_close(st, last, rtol=1e-6, atol=1e-6)
        torch.testing.assert_close(y, y1[0], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize('dtype', ALL, ids=str)
@pytest.mark.parametrize('D', [2, 9, 65, 67, 79, 127])
def test_widths_that_are_not_whole_vectors(h, dtype, D):
    """Channels that end inside a 16-byte vector or with fewer than one vector in a tile (65), rows at any element's address: the moved-back
    last vector counts no channel twice and writes nothing behind the row."""
    p = Problem(dtype, D=D, N=16, T=37, n=2, W=4, seed=D)
    want = p.reference()
    p.compare(p.run(h), want)

    def odd(t):
        buf = torch.full((t.numel() + 1,), float('nan'), dtype=t.dtype, device=t.device)[1:].view(t.shape)
        return buf.copy_(t).detach()
    p.compare(p.run(h, odd), want)
    q = Problem(dtype, D=D, N=5, lengths=[9, 0, 70], seed=D + 1, carry=True, z=False)
    q.compare(q.run(h, odd), q.reference())


@pytest.mark.parametrize('dtype', ALL, ids=str)
@pytest.mark.parametrize('rows,C', [(70, 2), (700, 9), (4000, 15), (50, 33), (20000, 17), (300, 301), (11, 1027), (1300, 127), (6, 4099), (600, 8195), (90, 600), (41, 611), (60, 151)])
def test_rms_norm_rows_that_are_not_whole_vectors(h, dtype, rows, C):
    """Odd widths through every shape of the kernels, at an odd address, with no element of a neighbouring row touched."""
    from rgp_amd import seq_ops
    g = _gen(rows + C)
    odd = lambda t: torch.full((rows, C + 1), float('nan'), dtype=dtype, device='cuda')[:, 1:].copy_(t)           # noqa: E731
    x, r, gy, gh = (_randn(g, rows, C, dtype=dtype) for _ in range(4))
    w = _randn(g, C, dtype=ref.acc_of(dtype))
    lx, lr, lw = odd(x).requires_grad_(True), odd(r).requires_grad_(True), w.cuda().requires_grad_(True)
    y, hid = seq_ops.rms_norm(h, lx, lw, residual=lr)
    gx, gr, gw = torch.autograd.grad((y, hid), (lx, lr, lw), (odd(gy), odd(gh)))
    d = lambda t: t.double()                                      # noqa: E731
    want = ref.rms(d(x), d(r), d(w), 1e-6, d(gy), d(gh))
    ops = C + rows + 64                                           # the additions over a row and over the rows
    ref.check('y', y, *want['y'], ops=ops)
    ref.check('hid', hid, *want['hid'], ops=ops)
    ref.check('gx', gx, *want['gx'], ops=ops, acc=ref.acc_of(dtype))
    ref.check('gw', gw, *want['gw'], ops=ops, acc=ref.acc_of(dtype))


def test_graphs_keep_what_they_need_and_end_like_others(h):
    """A backward pass twice without retain_graph is refused, with it gives the same bits; gradients of x and residual that accumulate into
    leaves share no memory; a graph keeps its handle; a closed handle refuses."""
    from rgp_amd import seq_ops
    from rgp_amd._lib import RgpError
    from rgp_amd.capi import Handle
    g = _gen(21)
    t = {k: _randn(g, *s, dtype=F32).cuda().requires_grad_(True) for k, s in
         dict(u=(9, 2, 6), delta=(9, 2, 6), A=(6, 3), B=(9, 2, 3), C=(9, 2, 3), w=(6, 4), x=(5, 8), r=(5, 8), n=(8,)).items()}
    other = Handle()
    y = seq_ops.ssm_scan(other, t['u'], t['delta'], t['A'], t['B'], t['C'])
    v = seq_ops.ssm_conv(other, t['u'], t['w'])
    n, hid = seq_ops.rms_norm(other, t['x'], t['n'], residual=t['r'])
    del other
    for out, ins in ((y, 'u delta A B C'), (v, 'u w'), (n, 'x r n')):
        ins = [t[k] for k in ins.split()]
        one = torch.autograd.grad(out.sum(), ins, retain_graph=True)
        two = torch.autograd.grad(out.sum(), ins)
        assert all(torch.equal(a, b) for a, b in zip(one, two))
        with pytest.raises(RuntimeError, match='second time'):
            torch.autograd.grad(out.sum(), ins)
    n, hid = seq_ops.rms_norm(h, t['x'], t['n'], residual=t['r'])
    (n.sum() + 2 * hid.sum()).backward()
    assert torch.equal(t['x'].grad, t['r'].grad) and t['x'].grad.data_ptr() != t['r'].grad.data_ptr()
    before = t['r'].grad.clone()
    t['x'].grad.zero_()
    assert torch.equal(t['r'].grad, before)
    n, hid = seq_ops.rms_norm(h, t['x'], t['n'], residual=t['x'])                # the same leaf twice
    gx, = torch.autograd.grad(n.sum(), t['x'])
    n2, _ = seq_ops.rms_norm(h, t['x'], t['n'], residual=t['x'].detach().clone().requires_grad_(True))
    g2, = torch.autograd.grad(n2.sum(), t['x'])
    torch.testing.assert_close(gx, 2 * g2)
    closed = Handle()
    closed.close()
    with pytest.raises(RgpError):
        seq_ops.rms_norm(closed, t['x'].detach(), t['n'].detach())


def test_threads_with_streams_of_their_own_share_a_handle(h):
    """Four threads at once on one handle, each on its own stream, forward and backward: everybody gets the bits that a lone caller gets."""
    import threading
    from rgp_amd import seq_ops
    g = _gen(22)
    inputs = [[_randn(g, 300, 3, n, dtype=F32).cuda() for n in (20, 20, 16, 16)] + [-torch.exp(_randn(g, 20, 16)).float().cuda(), _randn(g, 20, dtype=F32).cuda()]
              for _ in range(4)]

    def work(ops):
        u, delta, B, Cm, A, w = [t.clone().requires_grad_(True) for t in ops]
        y = seq_ops.ssm_scan(h, u, delta, A, B, Cm)
        n, hid = seq_ops.rms_norm(h, y, w, residual=u)
        grads = torch.autograd.grad(n.square().sum() + hid.sum(), (u, delta, A, B, Cm, w))
        return [t.detach() for t in (y, n, hid) + grads]

    want = [work(ops) for ops in inputs]
    torch.cuda.synchronize()
    got, failed = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = work(inputs[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                      # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('dtype', [F64, F32, BF16], ids=str)
@pytest.mark.parametrize('T', [72, 96, 97, 104, 105, 200])
def test_few_and_many_blocks_of_time(h, dtype, T):
    """Lengths on both sides of where the blocks of the time split are joined by a launch of their own, states carried in, both directions; and
    a packed batch whose longest sequence decides."""
    for reverse in (False, True):
        p = Problem(dtype, D=20, N=16, T=T, n=2, carry=True, reverse=reverse, seed=T)
        p.compare(p.run(h), p.reference())
    q = Problem(dtype, D=33, N=6, lengths=[T, 0, 1, T // 2, 9], carry=True, seed=T + 1)
    q.compare(q.run(h), q.reference())


def test_steps_in_a_graph(h):
    """Single steps captured once and replayed: the states move on with every replay as with eager calls, with other work in between."""
    from rgp_amd import seq_ops
    g, n, D, N = _gen(31), 3, 24, 16
    w, b, A, D0 = _randn(g, D, 4, dtype=F32).cuda(), _randn(g, D, dtype=F32).cuda(), -torch.exp(_randn(g, D, N)).float().cuda(), _randn(g, D, dtype=F32).cuda()
    xs = [[_randn(g, n, k, dtype=BF16).cuda() for k in (D, D, N, N)] for _ in range(6)]
    inp = [t.clone() for t in xs[0]]
    cst, sst = torch.zeros(n, 3, D, device='cuda', dtype=BF16), torch.zeros(n, D, N, device='cuda')

    def step(x, delta, B, Cm, c, s):
        u = seq_ops.ssm_conv_step(h, x, w, b, c)
        y = seq_ops.ssm_scan_step(h, u, delta, A, B, Cm, D0, s, delta_bias=b)
        return seq_ops.rms_norm(h, y, D0, residual=u)[0]
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*inp, cst, sst)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*inp, cst, sst)
        cst.zero_(), sst.zero_()
        ce, se = torch.zeros_like(cst), torch.zeros_like(sst)
        for x in xs:
            for t, v in zip(inp, x):
                t.copy_(v)
            graph.replay()
            want = step(*x, ce, se)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(cst, ce) and torch.equal(sst, se)


def test_captured_backward_refuses_leaves_of_an_eager_graph(h):
    """While a graph made outside holds the leaf, the captured backward pass raises before anything crosses the streams; without it, it works."""
    from rgp_amd import seq_ops
    x, w = torch.randn(6, 8, device='cuda', requires_grad=True), torch.ones(8, device='cuda', requires_grad=True)
    gy = torch.randn(6, 8, device='cuda')

    def region():
        return torch.autograd.grad(seq_ops.rms_norm(h, x, w), (x, w), gy)
    region()
    torch.cuda.synchronize()
    eager = seq_ops.rms_norm(h, x, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='outside the capture'):
        with torch.cuda.graph(graph):
            region()
    torch.cuda.synchronize()
    want = torch.autograd.grad(eager, (x, w), gy)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = region()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('dtype', [F64, F32], ids=str)
def test_very_many_short_sequences(h, dtype):
    """More blocks than the sums over them take at once (8192): gradients of the parameters are sums over all sequences."""
    from rgp_amd import seq_ops
    g, T, n, D, N = _gen(41), 2, 9001, 3, 2
    acc = ref.acc_of(dtype)
    acts = [_randn(g, T, n, k, dtype=dtype) for k in (D, D, N, N, D)]                            # u, delta, B, C, gy
    par = [-torch.exp(_randn(g, D, N)).to(acc), _randn(g, D, dtype=acc), _randn(g, D, dtype=acc)]     # A, D, bias
    leaves = [t.cuda().requires_grad_(True) for t in acts[:4] + par]
    u, delta, B, Cm, A, skip, bias = leaves
    y = seq_ops.ssm_scan(h, u, delta, A, B, Cm, D=skip, delta_bias=bias)
    got = torch.autograd.grad(y, leaves, acts[4].cuda())
    w = [t.double().requires_grad_(True) for t in acts[:4] + par]
    u, delta, B, Cm, A, skip, bias = w
    s, ys = torch.zeros(n, D, N, dtype=F64), []
    for t in range(T):
        dt = torch.nn.functional.softplus(delta[t] + bias)
        s = torch.exp(dt[..., None] * A) * s + (dt * u[t])[..., None] * B[t][:, None]
        ys.append((s * Cm[t][:, None]).sum(-1) + skip * u[t])
    want = torch.autograd.grad(torch.stack(ys), w, acts[4].double())
    # relative to the largest: rounding of the operands of each product (64 operations a term), and of adding T n terms of either sign, whose
    # absolute values sum to at most T n times the largest term
    half = torch.finfo(acc).eps / 2
    for a, b in zip(got[:4], want[:4]):
        assert float((a.cpu().double() - b).abs().max()) <= 64 * half * float(b.abs().max())
    terms = T * n * 64 * half
    for a, b in zip(got[4:], want[4:]):
        assert float((a.cpu().double() - b).abs().max()) <= terms * max(1.0, float(b.abs().max()) / (T * n) ** 0.5)
