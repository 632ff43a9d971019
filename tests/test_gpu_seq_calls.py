"""Calls of the sequence operators from places where they can be given what no kernel may see: a graph whose handle is gone, the framework's
other ways to run a function, tensors whose memory does not hold their values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F64, F32, BF16 = torch.float64, torch.float32, torch.bfloat16


@pytest.fixture(scope='module')
def h():
    from rgp_amd.capi import Handle
    return Handle()


def _leaves(*names, seed=0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    shapes = dict(u=(9, 2, 6), delta=(9, 2, 6), A=(6, 3), B=(9, 2, 3), C=(9, 2, 3), w=(6, 4), x=(5, 8), r=(5, 8), n=(8,))
    return [torch.randn(*shapes[k], generator=g, dtype=F64).to(dtype).cuda().requires_grad_(True) for k in names]


def _three(h, ops):
    """One result of each differentiable operator."""
    from rgp_amd import seq_ops
    u, delta, A, B, Cm, w, x, r, n = ops
    return seq_ops.ssm_scan(h, u, delta, A, B, Cm), seq_ops.ssm_conv(h, u, w), seq_ops.rms_norm(h, x, n, residual=r)[0]


ALL_LEAVES = ('u', 'delta', 'A', 'B', 'C', 'w', 'x', 'r', 'n')


def test_backward_pass_after_the_handle_is_closed_is_refused(h):
    """close() under graphs that are still alive: their backward passes raise, another handle's go on, and so do those of a handle that is only
    out of scope."""
    from rgp_amd.capi import Handle
    ops = _leaves(*ALL_LEAVES)
    other = Handle()
    closed, mine = _three(other, ops), _three(h, ops)
    other.close()
    assert not other.h
    for out in closed:
        for _ in range(2):                                          # the refused pass takes nothing with it
            with pytest.raises(RuntimeError, match='handle of this graph is closed'):
                out.sum().backward(retain_graph=True)
    assert all(t.grad is None for t in ops)
    dropped = Handle()
    still = _three(dropped, ops)
    del dropped
    for a, b in zip(mine, still):
        for x, y in zip(torch.autograd.grad(a.sum(), ops, allow_unused=True), torch.autograd.grad(b.sum(), ops, allow_unused=True)):
            assert (x is None and y is None) or torch.equal(x, y)
    other.close()                                                   # once more is nothing


def test_tangents_are_refused_in_both_directions(h):
    """Forward-mode derivatives never come back as nothing: a dual operand, a dual gradient and a dual tensor to clip raise; inside a dual level
    the operators work on tensors without tangents."""
    import torch.autograd.forward_ad as fwad
    from rgp_amd import seq_ops
    from rgp_amd._lib import RgpError
    ops = _leaves(*ALL_LEAVES)
    plain = [t.detach() for t in _three(h, ops)]
    with fwad.dual_level():
        for i, t in enumerate(ops):
            dual = list(ops)
            dual[i] = fwad.make_dual(t.detach(), torch.ones_like(t))
            with pytest.raises(RgpError, match='forward-mode'):
                _three(h, dual)
        outs = _three(h, ops)
        assert all(torch.equal(a, b) for a, b in zip(outs, plain))
        for out in outs:
            with pytest.raises(RuntimeError, match='forward-mode tangent'):
                torch.autograd.grad(out, ops, fwad.make_dual(torch.ones_like(out), torch.ones_like(out)), allow_unused=True, retain_graph=True)
            torch.autograd.grad(out, ops, torch.ones_like(out), allow_unused=True)
        g = torch.randn(40, device='cuda')
        keep = g.clone()
        with pytest.raises(RgpError, match='forward-mode'):
            seq_ops.clip_grad_norm(h, [fwad.make_dual(g, g)], 1e-3)
        assert torch.equal(g, keep)


def test_recording_a_function_is_refused(h):
    """torch.jit.trace and make_fx raise, the latter for a backward pass too; afterwards the calls are as before."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from rgp_amd import seq_ops
    from rgp_amd._lib import RgpError
    ops = [t.detach() for t in _leaves(*ALL_LEAVES)]
    plain = _three(h, ops)
    for record in (lambda f, x: torch.jit.trace(f, x, check_trace=False), lambda f, x: make_fx(f)(x)):
        with pytest.raises(RgpError, match='cannot be recorded'):
            record(lambda x: seq_ops.rms_norm(h, x, ops[8]), ops[6])
    leaf = ops[6].clone().requires_grad_(True)
    out = seq_ops.rms_norm(h, leaf, ops[8])
    with pytest.raises(RuntimeError, match='cannot be recorded'):
        make_fx(lambda g: torch.autograd.grad(out, leaf, g, retain_graph=True)[0])(torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(_three(h, ops), plain))


@pytest.mark.parametrize('D', [1, 5])
def test_operands_with_a_pending_negation(h, D):
    """The imaginary part of a conjugate is a view whose memory holds the negated values (one feature: also one that looks contiguous): operands
    and gradients of that kind count by their values."""
    from rgp_amd import seq_ops
    g = torch.Generator().manual_seed(D)
    f = lambda *s: torch.randn(*s, generator=g).cuda()                                          # noqa: E731
    ops = dict(u=f(7, 2, D), delta=f(7, 2, D), A=-f(D, 1).abs(), B=f(7, 2, 1), C=f(7, 2, 1), D=f(D), z=f(7, 2, D), bias=f(D), init=f(2, D, 1), w=f(D, 4),
               cinit=f(2, 3, D), n=f(D), r=f(7, 2, D), gy=f(7, 2, D))

    def negated(t):
        v = torch.complex(torch.zeros_like(t), -t).conj().imag
        assert v.is_neg()
        return v

    def run(t):
        leaf = {k: v if k in ('init', 'cinit', 'gy') else v.detach().requires_grad_(True) for k, v in t.items()}
        y = seq_ops.ssm_scan(h, leaf['u'], leaf['delta'], leaf['A'], leaf['B'], leaf['C'], D=leaf['D'], z=leaf['z'], delta_bias=leaf['bias'], init=leaf['init'])
        v = seq_ops.ssm_conv(h, leaf['u'], leaf['w'], leaf['bias'], init=leaf['cinit'])
        n, hid = seq_ops.rms_norm(h, leaf['u'], leaf['n'], residual=leaf['r'])
        grads = torch.autograd.grad((y, v, n, hid), [leaf[k] for k in ('u', 'delta', 'A', 'B', 'C', 'D', 'z', 'bias', 'w', 'n', 'r')], [leaf['gy']] * 4)
        return [y, v, n, hid] + list(grads)

    want = run(ops)
    for k in list(ops) + ['all']:
        got = run({q: negated(t) if k in (q, 'all') else t for q, t in ops.items()})
        assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(got, want)), k
    two = torch.full((D,), 2.0, device='cuda')
    total = negated(torch.full((1,), 16.0, device='cuda', dtype=F64))
    assert float(seq_ops.clip_grad_norm(h, [two], 2.0, sumsq=total)) == 4.0 and torch.allclose(two, torch.ones_like(two), rtol=1e-6)


@pytest.mark.parametrize('dtype', [F32, BF16], ids=str)
def test_saved_operands_that_come_back_through_hooks(h, dtype):
    """torch.autograd.graph's hooks may keep saved operands elsewhere: on the host, in another memory order -- the gradients are the same bits; as
    another type or shape they are refused."""
    from rgp_amd import seq_ops
    g = torch.Generator().manual_seed(4)
    acc = F32
    f = lambda *s, t=dtype: torch.randn(*s, generator=g).to(t).cuda()                                   # noqa: E731
    ops = dict(u=f(9, 2, 6), delta=f(9, 2, 6), A=-f(6, 3, t=acc).abs(), B=f(9, 2, 2, 3), C=f(9, 2, 2, 3), D=f(6, t=acc), z=f(9, 2, 6), bias=f(6, t=acc), w=f(6, 4, t=acc),
               n=f(6, t=acc), x=f(5, 6), r=f(5, 6))
    leaf = {k: v.requires_grad_(True) for k, v in ops.items()}
    cinit, init, gy = f(2, 3, 6), f(2, 6, 3, t=acc), f(9, 2, 6)

    def forward():
        y = seq_ops.ssm_scan(h, leaf['u'], leaf['delta'], leaf['A'], leaf['B'], leaf['C'], D=leaf['D'], z=leaf['z'], delta_bias=leaf['bias'], init=init)
        return y, seq_ops.ssm_conv(h, leaf['u'], leaf['w'], leaf['bias'], init=cinit), seq_ops.rms_norm(h, leaf['x'], leaf['n'], residual=leaf['r'])[0]

    def backward(outs):
        return torch.autograd.grad(outs, list(leaf.values()), [gy, gy, gy[:5, 0].contiguous()])
    want = backward(forward())
    turned = lambda t: t.transpose(0, -1).contiguous().transpose(0, -1)                                 # noqa: E731
    for pack, unpack in ((lambda t: t.cpu(), lambda t: t.cuda()), (lambda t: t, turned), (lambda t: t, lambda t: torch._neg_view(-t))):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            outs = forward()
        assert all(torch.equal(a, b) for a, b in zip(backward(outs), want))
    with torch.autograd.graph.save_on_cpu():
        outs = forward()
    assert all(torch.equal(a, b) for a, b in zip(backward(outs), want))
    for unpack in (lambda t: t.double(), lambda t: t[:1], lambda t: t[..., :2], lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            outs = forward()
        for o in outs:
            with pytest.raises(RuntimeError, match='came back'):
                torch.autograd.grad(o.sum(), list(leaf.values()), allow_unused=True)


def test_threads_that_fail_at_once_read_their_own_messages(h):
    """Refusals from several threads on one handle (the library is entered without the interpreter's lock): every thread finds the message of
    its own call, and a thread without a failure a whole one."""
    import ctypes as C
    import threading
    from rgp_amd import _lib
    from rgp_amd.capi import Handle
    other = Handle()
    calls = []
    for entry, struct in (('rgp_ssm_scan_forward', _lib.SsmScan), ('rgp_ssm_scan_step', _lib.SsmScan), ('rgp_ssm_conv_forward', _lib.SsmConv),
                          ('rgp_ssm_conv_step', _lib.SsmConv), ('rgp_rms_norm_forward', _lib.RmsNorm), ('rgp_rms_norm_backward', _lib.RmsNorm)):
        for dtype in (-1, 0):                                       # an unknown type, an empty problem
            a = struct()
            a.dtype = dtype
            if struct is _lib.RmsNorm:
                a.rows = -1 if dtype == 0 else 0
            fn = getattr(h.lib, entry)
            assert fn(other.h, None, C.byref(a)) == _lib.RGP_ERR_BAD_ARG
            calls.append((fn, a, other.lib.rgp_last_error(other.h)))
    assert len({m for _, _, m in calls}) == len(calls) and all(len(m) > 16 for _, _, m in calls)         # longer than a string holds in place
    wrong, start = [], threading.Barrier(len(calls) + 1)

    def run(fn, a, want):
        start.wait()
        for _ in range(2000):
            if fn(h.h, None, C.byref(a)) != _lib.RGP_ERR_BAD_ARG or h.lib.rgp_last_error(h.h) != want:
                wrong.append(want)

    def read():
        start.wait()
        for _ in range(2000):
            if h.lib.rgp_last_error(h.h) not in messages:
                wrong.append(b'reader')
    first = calls[0]
    assert first[0](h.h, None, C.byref(first[1])) == _lib.RGP_ERR_BAD_ARG
    messages = {m for _, _, m in calls}
    threads = [threading.Thread(target=run, args=c) for c in calls] + [threading.Thread(target=read)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]
    fresh = Handle()
    assert fresh.lib.rgp_last_error(fresh.h) == b''                 # whatever address it has


def test_states_of_whole_sequences_must_not_share_memory(h):
    """The C entries for whole sequences refuse a final state that overlaps the initial one (blocks of time run at once); buffers side by side
    are taken, and give what two allocations give."""
    import ctypes as C
    from rgp_amd import _lib
    T, n, D, N, W = 200, 2, 6, 3, 4
    g = torch.Generator().manual_seed(5)
    f = lambda *s: torch.randn(*s, generator=g).cuda()                                         # noqa: E731
    x, delta, B, Cm, A, w = f(T, n, D), f(T, n, D), f(T, n, N), f(T, n, N), -f(D, N).abs(), f(D, W)
    st = torch.cuda.current_stream().cuda_stream

    def scan(buf, init, last):
        a = _lib.SsmScan()
        a.dtype, a.n_seq, a.D, a.N, a.G, a.T, a.rows, a.max_len = _lib.DT_F32, n, D, N, 1, T, T * n, T
        y = torch.empty_like(x)
        for k, t in dict(u=x, delta=delta, B=B, C=Cm, A=A, y=y).items():
            setattr(a, k, t.data_ptr())
        a.u_st = a.delta_st = n * D
        a.u_sb = a.delta_sb = D
        a.B_st = a.C_st = n * N
        a.B_sb = a.C_sb = N
        work = torch.empty(h.lib.rgp_ssm_scan_workspace(C.byref(a), 0), dtype=torch.uint8, device='cuda')
        assert work.numel() > 0                                     # split over time: the case in which blocks read init while another writes last
        a.work, a.work_bytes = work.data_ptr(), work.numel()
        a.init, a.last = buf.data_ptr() + 4 * init, buf.data_ptr() + 4 * last
        r = h.lib.rgp_ssm_scan_forward(h.h, st, C.byref(a))
        torch.cuda.synchronize()
        return r

    def conv(buf, init, last):
        c = _lib.SsmConv()
        c.dtype, c.n_seq, c.D, c.W, c.T, c.rows, c.max_len = _lib.DT_F32, n, D, W, T, T * n, T
        v = torch.empty_like(x)
        for k, t in dict(x=x, w=w, v=v).items():
            setattr(c, k, t.data_ptr())
        c.x_st, c.x_sb = n * D, D
        c.init, c.last = buf.data_ptr() + 4 * init, buf.data_ptr() + 4 * last
        r = h.lib.rgp_ssm_conv_forward(h.h, st, C.byref(c))
        torch.cuda.synchronize()
        return r
    for call, size in ((scan, n * D * N), (conv, n * (W - 1) * D)):
        start = f(size)
        for init, last in ((0, 0), (0, 1), (1, 0), (0, size - 1), (size - 1, 0)):
            buf = torch.cat((start, start))
            keep = buf.clone()
            assert call(buf, init, last) == _lib.RGP_ERR_BAD_ARG and b'share memory' in h.lib.rgp_last_error(h.h)
            assert torch.equal(buf, keep)
        one, two = torch.cat((start, start)), torch.cat((start, start, start))
        assert call(one, 0, size) == 0 and call(two, 0, 2 * size) == 0
        assert torch.equal(one[size:], two[2 * size:]) and torch.equal(one[:size], start) and not torch.equal(one[size:], start)


@pytest.mark.parametrize('dtype', [F64, BF16], ids=str)
@pytest.mark.parametrize('reentrant', [False, True])
def test_checkpointed_regions(h, dtype, reentrant):
    """torch.utils.checkpoint runs the region again in the backward pass: the same bits, whichever way it saves."""
    from torch.utils.checkpoint import checkpoint
    from rgp_amd import seq_ops
    g = torch.Generator().manual_seed(6)
    acc = F64 if dtype == F64 else F32
    f = lambda *s, t=dtype: torch.randn(*s, generator=g, dtype=F64).to(t).cuda().requires_grad_(True)           # noqa: E731
    x, delta, B, Cm, z = f(40, 2, 12), f(40, 2, 12), f(40, 2, 16), f(40, 2, 16), f(40, 2, 12)
    A, w, b, n = f(12, 16, t=acc), f(12, 4, t=acc), f(12, t=acc), f(12, t=acc)

    def region(x, delta, B, Cm, z, A, w, b, n):
        v = seq_ops.ssm_conv(h, x, w, b)
        y = seq_ops.ssm_scan(h, v, delta, -A.abs(), B, Cm, D=b, z=z, delta_bias=b)
        return seq_ops.rms_norm(h, y, n, residual=x)
    ops = (x, delta, B, Cm, z, A, w, b, n)
    gy, gh = (torch.randn(40, 2, 12, generator=g, dtype=F64).to(dtype).cuda() for _ in range(2))
    want = torch.autograd.grad(region(*ops), ops, (gy, gh))
    outs = checkpoint(region, *ops, use_reentrant=reentrant)
    torch.autograd.backward(outs, (gy, gh))
    for t, e in zip(ops, want):
        assert torch.equal(t.grad, e)


def test_some_operands_without_gradients_and_other_modes(h):
    """Each leaf alone gives the gradient that it has among all; inference mode and anomaly detection change nothing."""
    ops = _leaves(*ALL_LEAVES)
    outs = _three(h, ops)
    want = torch.autograd.grad([o.square().sum() for o in outs], ops)
    for i, e in enumerate(want):
        one = [t.detach().requires_grad_(i == j) for j, t in enumerate(ops)]
        loss = sum(o.square().sum() for o in _three(h, one))
        assert torch.equal(torch.autograd.grad(loss, one[i])[0], e)
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(_three(h, ops), outs))
    with torch.autograd.detect_anomaly(check_nan=True):
        got = torch.autograd.grad([o.square().sum() for o in _three(h, ops)], ops)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
