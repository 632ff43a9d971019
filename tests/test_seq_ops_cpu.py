"""CPU checks of the sequence operators: the plain 64-bit forms the GPU tests compare with (their gradients against autograd and against
differences), the refusals -- raised before the library is entered -- and the argument checks of the library's size queries."""
import ctypes as C

import pytest
import torch

import seq_reference as ref


class _Nothing(object):
    """A handle whose library must not be entered."""
    device = torch.device('cpu')
    h = None

    class lib(object):
        def __getattr__(self, name):
            raise AssertionError('the library was entered: ' + name)
    lib = lib()


H = _Nothing()


def _leaf(*shape, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).requires_grad_(True)


def test_reference_scan_gradients_are_autograds_and_differences():
    L, Dn, G, N = 5, 4, 2, 3
    t = dict(u=_leaf(L, Dn, seed=1), delta=_leaf(L, Dn, seed=2), A=_leaf(Dn, N, seed=3), B=_leaf(L, G, N, seed=4), Cm=_leaf(L, G, N, seed=5),
             D=_leaf(Dn, seed=6), z=_leaf(L, Dn, seed=7), bias=_leaf(Dn, seed=8))
    init, gy = _leaf(Dn, N, seed=9).detach(), _leaf(L, Dn, seed=10).detach()
    f = lambda **k: ref.scan_one(init=init, gy=None, **k)['y'][0]              # noqa: E731
    grads = torch.autograd.grad(f(**t), list(t.values()), gy)
    o = ref.scan_one(init=init, gy=gy, **{k: v.detach() for k, v in t.items()})
    names = dict(u='gu', delta='gdelta', A='gA', B='gB', Cm='gC', D='gD', z='gz', bias='gbias')
    for (k, v), g in zip(t.items(), grads):
        torch.testing.assert_close(o[names[k]][0], g, rtol=1e-12, atol=1e-12)
        d = v.detach().clone()
        i = tuple(0 if n == 1 else 1 for n in d.shape)
        vals = []
        for e in (1e-6, -1e-6):
            d2 = d.clone()
            d2[i] += e
            vals.append((f(**{**{q: w.detach() for q, w in t.items()}, k: d2}) * gy).sum())
        assert abs(float((vals[0] - vals[1]) / 2e-6) - float(g[i])) < 1e-7 * max(1.0, abs(float(g[i])))


def test_reference_conv_and_rms_gradients_are_autograds():
    L, D, W = 6, 3, 4
    x, w, b = _leaf(L, D, seed=1), _leaf(D, W, seed=2), _leaf(D, seed=3)
    init, gv = _leaf(W - 1, D, seed=4).detach(), _leaf(L, D, seed=5).detach()
    g = torch.autograd.grad(ref.conv_one(x, w, b, init, None)['v'][0], (x, w, b), gv)
    o = ref.conv_one(x.detach(), w.detach(), b.detach(), init, gv)
    for k, q in zip(('gx', 'gw', 'gb'), g):
        torch.testing.assert_close(o[k][0], q, rtol=1e-12, atol=1e-12)
    x, r, w = _leaf(4, 5, seed=1), _leaf(4, 5, seed=2), _leaf(5, seed=3)
    gy, gh = _leaf(4, 5, seed=4).detach(), _leaf(4, 5, seed=5).detach()
    f = ref.rms(x, r, w, 1e-6, None, None)
    g = torch.autograd.grad((f['y'][0], f['hid'][0]), (x, w), (gy, gh))
    o = ref.rms(x.detach(), r.detach(), w.detach(), 1e-6, gy, gh)
    torch.testing.assert_close(o['gx'][0], g[0], rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(o['gw'][0], g[1], rtol=1e-12, atol=1e-12)


def _conv(**k):
    from rgp_amd import seq_ops
    a = dict(x=torch.zeros(5, 2, 6), weight=torch.zeros(6, 4), bias=torch.zeros(6))
    a.update(k)
    return seq_ops.ssm_conv(H, **a)


def _scan(**k):
    from rgp_amd import seq_ops
    a = dict(u=torch.zeros(5, 2, 6), delta=torch.zeros(5, 2, 6), A=torch.zeros(6, 3), B=torch.zeros(5, 2, 3), Cm=torch.zeros(5, 2, 3), D=torch.zeros(6),
             z=torch.zeros(5, 2, 6), delta_bias=torch.zeros(6))
    a.update(k)
    return seq_ops.ssm_scan(H, **a)


def _refused(fn, match, **k):
    from rgp_amd._lib import RgpError, RGP_ERR_BAD_ARG
    with pytest.raises(RgpError, match=match) as e:
        fn(**k)
    assert e.value.code == RGP_ERR_BAD_ARG


def test_conv_refusals():
    from rgp_amd import seq_ops
    t3 = seq_ops.SeqTable(H, [3, 0, 2])
    _refused(_conv, 'T, batch', x=torch.zeros(5, 6))
    _refused(_conv, 'packed rows', x=torch.zeros(5, 2, 6), seqs=t3)
    _refused(_conv, 'sequence table 5', x=torch.zeros(7, 6), seqs=t3)
    _refused(_conv, 'empty', x=torch.zeros(0, 2, 6))
    _refused(_conv, 'float64, float32', x=torch.zeros(5, 2, 6, dtype=torch.int32))
    _refused(_conv, '2 to 8 taps', weight=torch.zeros(6, 9))
    _refused(_conv, '2 to 8 taps', weight=torch.zeros(6, 1))
    _refused(_conv, 'weight has shape', weight=torch.zeros(5, 4))
    _refused(_conv, 'bias has shape', bias=torch.zeros(5))
    _refused(_conv, 'parameters and states', x=torch.zeros(5, 2, 6, dtype=torch.float64))
    _refused(_conv, 'parameters and states', weight=torch.zeros(6, 4, dtype=torch.bfloat16))
    _refused(_conv, 'init must be', init=torch.zeros(2, 4, 6))
    _refused(_conv, 'init must be', init=torch.zeros(2, 3, 6, dtype=torch.float64))
    _refused(_conv, 'no gradient', init=torch.zeros(2, 3, 6, requires_grad=True))
    _refused(_conv, 'device tensor', x=None)
    _refused(_conv, 'on meta', x=torch.zeros(5, 2, 6, device='meta'))
    step = lambda **k: seq_ops.ssm_conv_step(H, **{**dict(x=torch.zeros(2, 6), weight=torch.zeros(6, 4), bias=None, state=torch.zeros(2, 3, 6)), **k})     # noqa: E731
    _refused(step, 'batch, D', x=torch.zeros(1, 2, 6))
    _refused(step, 'state must be', state=torch.zeros(2, 4, 6))
    _refused(step, 'state must be', state=torch.zeros(3, 2, 6).transpose(0, 1))
    _refused(step, 'in place', state=torch.zeros(2, 3, 6, requires_grad=True))


def test_scan_refusals():
    from rgp_amd import seq_ops
    _refused(_scan, 'delta has shape', delta=torch.zeros(5, 2, 7))
    _refused(_scan, 'leading dimensions', delta=torch.zeros(5, 3, 6))
    _refused(_scan, 'delta is', delta=torch.zeros(5, 2, 6, dtype=torch.float64))
    _refused(_scan, 'z has shape', z=torch.zeros(5, 2, 1))
    _refused(_scan, 'divisor', B=torch.zeros(5, 2, 4, 3), Cm=torch.zeros(5, 2, 4, 3))
    _refused(_scan, 'groups', B=torch.zeros(5, 2, 2, 3))
    _refused(_scan, 'N = 3', B=torch.zeros(5, 2, 4))
    _refused(_scan, '1 to 64 states', A=torch.zeros(6, 65))
    _refused(_scan, '1 to 64 states', A=torch.zeros(6))
    _refused(_scan, 'A has shape', A=torch.zeros(5, 3))
    _refused(_scan, 'D has shape', D=torch.zeros(1))
    _refused(_scan, 'parameters and states', A=torch.zeros(6, 3, dtype=torch.float64))
    _refused(_scan, 'init has shape', init=torch.zeros(1, 6, 3))
    _refused(_scan, 'no gradient', init=torch.zeros(2, 6, 3, requires_grad=True))
    _refused(_scan, 'delta is required', delta=None)
    step = lambda **k: seq_ops.ssm_scan_step(H, **{**dict(u=torch.zeros(2, 6), delta=torch.zeros(2, 6), A=torch.zeros(6, 3), B=torch.zeros(2, 3), Cm=torch.zeros(2, 3), D=None, state=torch.zeros(2, 6, 3)), **k})     # noqa: E731
    _refused(step, 'batch, D', u=torch.zeros(2, 6, 1))
    _refused(step, 'state must be', state=torch.zeros(2, 6, 4))
    _refused(step, 'state must be', state=torch.zeros(2, 6, 3, dtype=torch.float64))
    _refused(step, 'leading dimensions', B=torch.zeros(3, 3))
    for bad in ([], [3, -1]):
        _refused(lambda: seq_ops.SeqTable(H, bad), 'at least one length')
    t = seq_ops.SeqTable(H, [3, 0, 2])
    assert t.off.tolist() == [0, 3, 3, 5] and t.max_len == 3 and t.rows == 5


def test_rms_and_clip_refusals():
    from rgp_amd import seq_ops
    rms = lambda **k: seq_ops.rms_norm(H, **{**dict(x=torch.zeros(3, 4), weight=torch.zeros(4)), **k})             # noqa: E731
    _refused(rms, 'eps', eps=0.0)
    _refused(rms, 'eps', eps=float('nan'))
    _refused(rms, 'weight has shape', weight=torch.zeros(3))
    _refused(rms, 'parameters and states', weight=torch.zeros(4, dtype=torch.float64))
    _refused(rms, 'residual', residual=torch.zeros(3, 5))
    _refused(rms, 'residual', residual=torch.zeros(3, 4, dtype=torch.float64))
    _refused(rms, 'x must be', x=torch.zeros(3, 4, dtype=torch.int8))
    clip = lambda g, m=1.0: seq_ops.clip_grad_norm(H, g, m)                                                        # noqa: E731
    g = torch.zeros(10)
    for m in (0.0, -1.0, float('nan')):
        _refused(lambda: clip([g], m), 'positive')
    _refused(lambda: clip([g, g]), 'share memory')
    _refused(lambda: clip([g[:6], g[5:]]), 'share memory')
    _refused(lambda: clip([torch.zeros(3, 8)[:, :5]]), 'gaps')
    _refused(lambda: clip([torch.zeros(1).expand(4)]), 'gaps')
    _refused(lambda: clip([torch.zeros(4, dtype=torch.int64)]), 'gradient 0')
    _refused(lambda: clip([None]), 'gradient 0')


def test_size_queries_refuse_and_count():
    from rgp_amd import _lib
    lib = _lib.load()
    a = _lib.SsmScan()
    a.dtype, a.n_seq, a.D, a.N, a.G, a.T, a.rows, a.max_len = _lib.DT_F32, 2, 6, 3, 2, 5, 10, 5
    assert lib.rgp_ssm_scan_states_bytes(C.byref(a)) == 2 * 1 * 6 * 3 * 4          # one state every 8 steps of each sequence
    for T, rows, off in ((5, 10, 0), (8, 16, 0), (17, 34, 0), (0, 0, 1), (0, 7, 1), (0, 8, 1), (0, 1001, 1)):      # the count that seq_ops allocates by
        b = _lib.SsmScan.from_buffer_copy(a)
        b.T, b.rows, b.off = T, rows, off
        blocks = (rows >> 3) + 2 if off else 2 * ((T + 7) >> 3)
        assert lib.rgp_ssm_scan_states_bytes(C.byref(b)) == blocks * 6 * 3 * 4
    assert lib.rgp_ssm_scan_workspace(C.byref(a), 0) == 0 and lib.rgp_ssm_scan_workspace(C.byref(a), 1) > 0
    for f, v in (('dtype', 4), ('n_seq', 0), ('N', 65), ('N', 0), ('G', 4), ('rows', 9), ('T', 0)):
        b = _lib.SsmScan.from_buffer_copy(a)
        setattr(b, f, v)
        assert lib.rgp_ssm_scan_workspace(C.byref(b), 1) == -1, f
    c = _lib.SsmConv()
    c.dtype, c.n_seq, c.D, c.W, c.T, c.rows = _lib.DT_BF16, 2, 6, 4, 5, 10
    assert lib.rgp_ssm_conv_workspace(C.byref(c), 0) == 0 and lib.rgp_ssm_conv_workspace(C.byref(c), 1) >= 5 * 6 * 4
    c.W = 9
    assert lib.rgp_ssm_conv_workspace(C.byref(c), 1) == -1
    r = _lib.RmsNorm()
    r.dtype, r.rows, r.C, r.eps = _lib.DT_F64, 3, 7, 1e-6
    assert lib.rgp_rms_norm_workspace(C.byref(r), 1) >= 7 * 8
    r.eps = 0.0
    assert lib.rgp_rms_norm_workspace(C.byref(r), 1) == -1
    n = (C.c_int64 * 2)(10, -1)
    d = (C.c_int32 * 2)(0, 1)
    assert lib.rgp_grad_workspace(1, n, d) == 8 and lib.rgp_grad_workspace(2, n, d) == -1 and lib.rgp_grad_workspace(0, None, None) == 8
    for call in (lib.rgp_ssm_scan_forward, lib.rgp_ssm_scan_backward, lib.rgp_ssm_scan_step):
        assert call(None, None, C.byref(a)) == _lib.RGP_ERR_BAD_ARG
    assert C.sizeof(_lib.SsmScan) == 6 * 4 + 3 * 8 + 6 * 8 + 12 * 8 + 17 * 8 + 8
    assert C.sizeof(_lib.SsmConv) == 6 * 4 + 3 * 8 + 2 * 8 + 4 * 8 + 10 * 8 + 8
    assert C.sizeof(_lib.RmsNorm) == 2 * 4 + 2 * 8 + 8 + 2 * 8 + 4 * 8 + 9 * 8 + 8


def test_sizes_beyond_the_library_are_refused():
    from rgp_amd import _lib
    lib = _lib.load()
    a = _lib.SsmScan()
    a.dtype, a.n_seq, a.D, a.N, a.G, a.off = _lib.DT_F32, 2, 6, 3, 2, 1
    a.rows = 1 << 40
    assert lib.rgp_ssm_scan_workspace(C.byref(a), 1) > 0
    a.rows += 1
    assert lib.rgp_ssm_scan_workspace(C.byref(a), 1) == -1
    c = _lib.SsmConv()
    c.dtype, c.n_seq, c.D, c.W, c.T, c.rows = _lib.DT_BF16, 1, 6, 4, (1 << 40) + 1, (1 << 40) + 1
    assert lib.rgp_ssm_conv_workspace(C.byref(c), 1) == -1
    r = _lib.RmsNorm()
    r.dtype, r.rows, r.C, r.eps = _lib.DT_F64, 3, 7, 1e-60
    assert lib.rgp_rms_norm_workspace(C.byref(r), 1) >= 7 * 8
    r.dtype = _lib.DT_BF16                                  # zero in 32 bits: a row of zeros would have no norm
    assert lib.rgp_rms_norm_workspace(C.byref(r), 1) == -1
