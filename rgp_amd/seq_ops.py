"""Sequence operators of the state-space encoder cell and the gradient clipping of the training step, on the C ABI's sequence section
(include/rgp_hip.h): differentiable torch functions over device tensors.

  ssm_conv / ssm_conv_step      short causal convolution with silu, over whole sequences / for one step with a state
  ssm_scan / ssm_scan_step      selective state-space scan, likewise
  rms_norm                      root-mean-square norm of x + residual
  clip_grad_norm                global norm of many gradient tensors, clipped in place

Activations are float64, float32, bfloat16 or float16; parameters (filters, A, D, biases, norm weights) and states are float64 for float64
activations and float32 for the others.  Sequences of equal length are (T, batch, features) tensors, in any memory order with contiguous
features; sequences of different lengths are packed rows (rows, features) with a SeqTable.  Every call is enqueued on the current torch
stream of the handle's device, allocates through torch (so it can be captured into a graph together with its backward pass) and gives the
same bits every time.  Wrong arguments raise RgpError (RGP_ERR_BAD_ARG) before anything is launched.

A captured backward pass needs leaves that no eager graph holds at that time: take the gradients with torch.autograd.grad inside the
captured region, on a forward pass of the same region."""
import ctypes as C
import math

import torch

from . import _lib
from ._lib import RgpError

_DTYPES = {torch.float64: _lib.DT_F64, torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


def _bad(msg):
    raise RgpError(_lib.RGP_ERR_BAD_ARG, msg)


def _acc(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _stream(handle):
    return C.c_void_p(torch.cuda.current_stream(handle.device).cuda_stream)


def _call(handle, fn, a):
    st = fn(handle.h, _stream(handle), C.byref(a))
    if st != 0:
        handle._check(st)


def _work(handle, nbytes):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=handle.device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _overlaps(t):
    """True if two elements of the tensor may share memory (strides that do not nest)."""
    dims = sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1)
    reach = 1
    for s, n in dims:
        if s < reach:
            return True
        reach = s * n
    return False


class SeqTable(object):
    """Lengths of packed sequences: rows off[s] .. off[s + 1] of a packed tensor are sequence s.  ``lengths`` is a list (or a CPU tensor)
    of whole numbers >= 0; it is checked here, once, and its offsets are kept on the handle's device."""

    def __init__(self, handle, lengths):
        lengths = [int(v) for v in (lengths.tolist() if hasattr(lengths, 'tolist') else lengths)]
        if not lengths or min(lengths) < 0:
            _bad('a sequence table needs at least one length, none of them negative')
        off = [0]
        for v in lengths:
            off.append(off[-1] + v)
        self.lengths, self.n_seq, self.rows, self.max_len = lengths, len(lengths), off[-1], max(lengths)
        self.device = handle.device
        self.off = torch.tensor(off, dtype=torch.int64).to(handle.device)


def _rows(name, t, like=None, lead=None, tail=1):
    """Leading shape of an activation after its checks."""
    if not isinstance(t, torch.Tensor):
        _bad('%s must be a device tensor' % name)
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        _bad('%s is %s on %s, %s on %s expected' % (name, t.dtype, t.device, like.dtype, like.device))
    if lead is not None and tuple(t.shape[:len(lead)]) != tuple(lead):
        _bad('%s has shape %s, leading dimensions %s expected' % (name, tuple(t.shape), tuple(lead)))
    return t


def _inner(t, dims):
    """The tensor with its last ``dims`` dimensions contiguous (a copy only where they are not)."""
    want = 1
    for i in range(1, dims + 1):
        if t.shape[-i] > 1 and t.stride(-i) != want:
            return t.contiguous()
        want *= t.shape[-i]
    return t


def _geometry(handle, x, seqs, what):
    """(lead, n_seq, T, rows, max_len, off) of a (T, batch, D) or packed (rows, D) activation."""
    if not isinstance(x, torch.Tensor):
        _bad('%s must be a device tensor' % what)
    if x.dtype not in _DTYPES:
        _bad('%s must be float64, float32, bfloat16 or float16, not %s' % (what, x.dtype))
    if x.device != handle.device:
        _bad('%s is on %s, the handle on %s' % (what, x.device, handle.device))
    if seqs is None:
        if x.dim() != 3:
            _bad('%s must be (T, batch, features); packed rows need a SeqTable' % what)
        T, n = x.shape[0], x.shape[1]
        if T < 1 or n < 1 or x.shape[2] < 1:
            _bad('%s is empty: shape %s' % (what, tuple(x.shape)))
        return (T, n), n, T, T * n, T, None
    if x.dim() != 2 or x.shape[1] < 1:
        _bad('%s must be packed rows (rows, features) with a SeqTable' % what)
    if seqs.device != x.device:
        _bad('the sequence table is on %s, %s on %s' % (seqs.device, what, x.device))
    if seqs.rows != x.shape[0]:
        _bad('%s has %d rows, the sequence table %d' % (what, x.shape[0], seqs.rows))
    return (x.shape[0],), seqs.n_seq, 0, seqs.rows, seqs.max_len, seqs.off


def _strides(t, packed):
    """Element strides of (step, sequence)."""
    return (t.stride(0), 0) if packed else (t.stride(0), t.stride(1))


def _param(name, t, shape, x, optional=False):
    if t is None:
        if optional:
            return None
        _bad('%s is required' % name)
    if not isinstance(t, torch.Tensor) or t.device != x.device:
        _bad('%s must be a tensor on %s' % (name, x.device))
    if tuple(t.shape) != tuple(shape):
        _bad('%s has shape %s, %s expected' % (name, tuple(t.shape), tuple(shape)))
    if t.dtype != _acc(x.dtype):
        _bad('%s is %s: parameters and states are %s for %s activations' % (name, t.dtype, _acc(x.dtype), x.dtype))
    return t if t.is_contiguous() else t.contiguous()


def _state(name, t, shape, dtype, x):
    """A state that is updated in place."""
    if not isinstance(t, torch.Tensor) or t.device != x.device or tuple(t.shape) != tuple(shape) or t.dtype != dtype or not t.is_contiguous():
        _bad('%s must be a contiguous %s tensor of shape %s on %s' % (name, dtype, tuple(shape), x.device))
    if t.requires_grad:
        _bad('%s is updated in place and takes no gradient' % name)
    return t


def _no_grad_state(name, t):
    if t is not None and t.requires_grad:
        _bad('%s takes no gradient: detach it' % name)


# ---------------------------------------------------------------------------------------------------------------------- convolution
def _conv_args(x, w, bias, geo, reverse):
    lead, n_seq, T, rows, max_len, off = geo
    a = _lib.SsmConv()
    a.dtype, a.n_seq, a.D, a.W, a.reverse = _DTYPES[x.dtype], n_seq, x.shape[-1], w.shape[1], 1 if reverse else 0
    a.T, a.rows, a.max_len, a.off = T, rows, max_len, _ptr(off)
    a.x, a.w, a.bias = x.data_ptr(), w.data_ptr(), _ptr(bias)
    a.x_st, a.x_sb = _strides(x, off is not None)
    return a


class _ConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, handle, x, w, bias, init, geo, reverse, want_last):
        v = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        last = torch.empty(geo[1], w.shape[1] - 1, x.shape[-1], dtype=x.dtype, device=x.device) if want_last else None
        a = _conv_args(x, w, bias, geo, reverse)
        a.init, a.v, a.last = _ptr(init), v.data_ptr(), _ptr(last)
        _call(handle, handle.lib.rgp_ssm_conv_forward, a)
        ctx.handle, ctx.geo, ctx.reverse = handle, geo, reverse
        ctx.save_for_backward(x, w, bias, init)
        ctx.set_materialize_grads(False)
        if want_last:
            ctx.mark_non_differentiable(last)
        return v, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gv, _):
        if gv is None:
            return (None,) * 8
        x, w, bias, init = ctx.saved_tensors
        handle = ctx.handle
        gv = _inner(gv, 1)
        a = _conv_args(x, w, bias, ctx.geo, ctx.reverse)
        a.gv_st, a.gv_sb = _strides(gv, ctx.geo[5] is not None)
        gx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        gw = torch.empty_like(w)
        gb = torch.empty_like(bias) if bias is not None else None
        work = _work(handle, handle.lib.rgp_ssm_conv_workspace(C.byref(a), 1))
        a.init, a.gv, a.gx, a.gw, a.gbias, a.work, a.work_bytes = _ptr(init), gv.data_ptr(), gx.data_ptr(), gw.data_ptr(), _ptr(gb), work.data_ptr(), work.numel()
        _call(handle, handle.lib.rgp_ssm_conv_backward, a)
        return None, gx, gw, gb, None, None, None, None


def ssm_conv(handle, x, weight, bias=None, seqs=None, init=None, reverse=False, return_state=False):
    """silu(bias + causal convolution of x with one filter per channel): v_t uses x_{t-W+1} .. x_t of its own sequence.

    x: (T, batch, D), or packed (rows, D) with ``seqs``; weight (D, W), 2 <= W <= 8; bias (D,).  init: (n_seq, W - 1, D), the inputs before
    the first step, oldest first (zeros without it); return_state=True also returns them for the step behind the last one.  reverse=True
    walks every sequence from its last step.  Gradients: x, weight, bias (states take none)."""
    geo = _geometry(handle, x, seqs, 'x')
    D = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[1] <= 8:
        _bad('weight must be (D, W) with 2 to 8 taps')
    w = _param('weight', weight, (D, weight.shape[1]), x)
    b = _param('bias', bias, (D,), x, optional=True)
    if init is not None:
        _no_grad_state('init', init)
        if tuple(init.shape) != (geo[1], w.shape[1] - 1, D) or init.dtype != x.dtype or init.device != x.device:
            _bad('init must be %s of shape %s on %s' % (x.dtype, (geo[1], w.shape[1] - 1, D), x.device))
        init = init.contiguous()
    v, last = _ConvFn.apply(handle, _inner(x, 1), w, b, init, geo, bool(reverse), bool(return_state))
    return (v, last) if return_state else v


def ssm_conv_step(handle, x, weight, bias, state):
    """One step of ``ssm_conv``: x (batch, D), state (batch, W - 1, D) of x's type, updated in place.  No gradients."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        _bad('x must be (batch, D)')
    x3 = x.detach().unsqueeze(0)
    geo = _geometry(handle, x3, None, 'x')
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[1] <= 8:
        _bad('weight must be (D, W) with 2 to 8 taps')
    D = x.shape[1]
    w, b = _param('weight', weight, (D, weight.shape[1]), x), _param('bias', bias, (D,), x, optional=True)
    _state('state', state, (x.shape[0], weight.shape[1] - 1, D), x.dtype, x)
    x3 = _inner(x3, 1)
    v = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = _conv_args(x3, w, b, geo, False)
    a.init = a.last = state.data_ptr()
    a.v = v.data_ptr()
    _call(handle, handle.lib.rgp_ssm_conv_step, a)
    return v


# ---------------------------------------------------------------------------------------------------------------------- scan
def _scan_args(u, delta, A, B, Cm, skip, z, bias, geo, reverse):
    lead, n_seq, T, rows, max_len, off = geo
    packed = off is not None
    a = _lib.SsmScan()
    a.dtype, a.n_seq, a.D, a.N, a.G, a.reverse = _DTYPES[u.dtype], n_seq, u.shape[-1], B.shape[-1], B.shape[-2], 1 if reverse else 0
    a.T, a.rows, a.max_len, a.off = T, rows, max_len, _ptr(off)
    a.u, a.delta, a.z, a.B, a.C = u.data_ptr(), delta.data_ptr(), _ptr(z), B.data_ptr(), Cm.data_ptr()
    a.u_st, a.u_sb = _strides(u, packed)
    a.delta_st, a.delta_sb = _strides(delta, packed)
    if z is not None:
        a.z_st, a.z_sb = _strides(z, packed)
    a.B_st, a.B_sb = _strides(B, packed)
    a.C_st, a.C_sb = _strides(Cm, packed)
    a.A, a.skip, a.bias = A.data_ptr(), _ptr(skip), _ptr(bias)
    return a


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, handle, u, delta, A, B, Cm, skip, z, bias, init, geo, reverse, want_last, train):
        y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
        last = torch.empty(geo[1], u.shape[-1], A.shape[1], dtype=A.dtype, device=u.device) if want_last else None
        a = _scan_args(u, delta, A, B, Cm, skip, z, bias, geo, reverse)
        states = _work(handle, handle.lib.rgp_ssm_scan_states_bytes(C.byref(a))) if train else None
        work = _work(handle, handle.lib.rgp_ssm_scan_workspace(C.byref(a), 0))
        a.init, a.y, a.last, a.states, a.work, a.work_bytes = _ptr(init), y.data_ptr(), _ptr(last), _ptr(states), work.data_ptr(), work.numel()
        _call(handle, handle.lib.rgp_ssm_scan_forward, a)
        ctx.handle, ctx.geo, ctx.reverse = handle, geo, reverse
        ctx.save_for_backward(u, delta, A, B, Cm, skip, z, bias, states)
        ctx.set_materialize_grads(False)
        if want_last:
            ctx.mark_non_differentiable(last)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, _):
        if gy is None:
            return (None,) * 14
        u, delta, A, B, Cm, skip, z, bias, states = ctx.saved_tensors
        handle = ctx.handle
        gy = _inner(gy, 1)
        new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)      # noqa: E731
        gu, gdelta, gA, gB, gC, gskip, gz, gbias = (new(t) for t in (u, delta, A, B, Cm, skip, z, bias))
        a = _scan_args(u, delta, A, B, Cm, skip, z, bias, ctx.geo, ctx.reverse)
        a.gy_st, a.gy_sb = _strides(gy, ctx.geo[5] is not None)
        work = _work(handle, handle.lib.rgp_ssm_scan_workspace(C.byref(a), 1))
        a.states, a.gy, a.gu, a.gdelta, a.gz, a.gB, a.gC = states.data_ptr(), gy.data_ptr(), gu.data_ptr(), gdelta.data_ptr(), _ptr(gz), gB.data_ptr(), gC.data_ptr()
        a.gA, a.gskip, a.gbias, a.work, a.work_bytes = gA.data_ptr(), _ptr(gskip), _ptr(gbias), work.data_ptr(), work.numel()
        _call(handle, handle.lib.rgp_ssm_scan_backward, a)
        return None, gu, gdelta, gA, gB, gC, gskip, gz, gbias, None, None, None, None, None


def _scan_check(u, delta, A, B, Cm, D, z, delta_bias, lead):
    """Operands in the form the library takes: (.., D) activations with contiguous features, (.., G, N) maps, contiguous parameters."""
    nd, n = len(lead), u.shape[-1]
    for name, t in (('delta', delta), ('z', z)):
        if t is not None:
            _rows(name, t, u, lead)
            if t.dim() != nd + 1 or t.shape[-1] != n:
                _bad('%s has shape %s, %s expected' % (name, tuple(t.shape), tuple(u.shape)))
    if delta is None:
        _bad('delta is required')
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= 64:
        _bad('A must be (D, N) with 1 to 64 states')
    N = A.shape[1]
    maps = []
    for name, t in (('B', B), ('C', Cm)):
        _rows(name, t, u, lead)
        if t.dim() == nd + 1:
            t = t.unsqueeze(-2)
        if t.dim() != nd + 2 or t.shape[-1] != N or t.shape[-2] < 1 or n % t.shape[-2]:
            _bad('%s has shape %s: (.., N) or (.., G, N) with N = %d and G a divisor of D = %d expected' % (name, tuple(t.shape), N, n))
        maps.append(_inner(t, 2))
    if maps[0].shape[-2] != maps[1].shape[-2]:
        _bad('B has %d groups, C %d' % (maps[0].shape[-2], maps[1].shape[-2]))
    return (_inner(u, 1), _inner(delta, 1), _param('A', A, (n, N), u), maps[0], maps[1], _param('D', D, (n,), u, optional=True),
            None if z is None else _inner(z, 1), _param('delta_bias', delta_bias, (n,), u, optional=True))


def ssm_scan(handle, u, delta, A, B, Cm, D=None, z=None, delta_bias=None, seqs=None, init=None, reverse=False, return_state=False):
    """Selective state-space scan.  Per step, channel d and its group g of B / C:
        dt = softplus(delta + delta_bias);  s[n] = exp(dt A[d, n]) s[n] + dt u B[g, n];  y = (sum_n C[g, n] s[n] + D[d] u) z sigmoid(z)
    u, delta, z: (T, batch, Dn), or packed (rows, Dn) with ``seqs``; B, C: the same leading dimensions and (N,) or (G, N); A (Dn, N),
    N <= 64; D, delta_bias (Dn,).  init: (n_seq, Dn, N), the state before the first step (zeros without it); return_state=True also returns
    the state behind the last step.  reverse=True walks every sequence from its last step.  Gradients: u, delta, A, B, C, D, z, delta_bias
    (states take none)."""
    geo = _geometry(handle, u, seqs, 'u')
    ops = _scan_check(u, delta, A, B, Cm, D, z, delta_bias, geo[0])
    if init is not None:
        _no_grad_state('init', init)
        init = _param('init', init, (geo[1], u.shape[-1], A.shape[1]), u)
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ops)
    y, last = _ScanFn.apply(handle, *ops, init, geo, bool(reverse), bool(return_state), train)
    return (y, last) if return_state else y


def ssm_scan_step(handle, u, delta, A, B, Cm, D, state, z=None, delta_bias=None):
    """One step of ``ssm_scan``: u, delta, z (batch, Dn); B, C (batch, N) or (batch, G, N); state (batch, Dn, N), updated in place.  No
    gradients."""
    if not isinstance(u, torch.Tensor) or u.dim() != 2:
        _bad('u must be (batch, D)')
    with torch.no_grad():
        u3 = u.unsqueeze(0)
        geo = _geometry(handle, u3, None, 'u')
        ops = _scan_check(u, delta, A, B, Cm, D, z, delta_bias, (u.shape[0],))
        _state('state', state, (u.shape[0], u.shape[1], A.shape[1]), _acc(u.dtype), u)
        y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
        a = _scan_args(*(t if i in (2, 5, 7) or t is None else t.unsqueeze(0) for i, t in enumerate(ops)), geo, False)
        a.init = a.last = state.data_ptr()
        a.y = y.data_ptr()
        _call(handle, handle.lib.rgp_ssm_scan_step, a)
    return y


# ---------------------------------------------------------------------------------------------------------------------- norm
def _rms_args(x, w, eps):
    a = _lib.RmsNorm()
    a.dtype, a.rows, a.C, a.eps = _DTYPES[x.dtype], x.shape[0], x.shape[1], eps
    a.x, a.x_st, a.w = x.data_ptr(), x.stride(0), w.data_ptr()
    return a


class _RmsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, handle, x, w, residual, eps, train):
        a = _rms_args(x, w, eps)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        hid = torch.empty_like(y) if residual is not None else None
        rstd = torch.empty(x.shape[0], dtype=w.dtype, device=x.device) if train else None
        if residual is not None:
            a.residual, a.residual_st, a.hid = residual.data_ptr(), residual.stride(0), hid.data_ptr()
        a.y, a.rstd = y.data_ptr(), _ptr(rstd)
        _call(handle, handle.lib.rgp_rms_norm_forward, a)
        ctx.handle, ctx.eps, ctx.two = handle, eps, residual is not None
        # 16-bit: the backward pass adds x and residual again, hid's rounding would show in the weight's gradient; 32 and 64 bits: hid is that sum
        again = residual is not None and x.element_size() == 2
        ctx.save_for_backward(x if again or residual is None else hid, residual if again else None, w, rstd)
        ctx.set_materialize_grads(False)
        return (y, hid) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gh=None):
        hid, residual, w, rstd = ctx.saved_tensors
        if gy is None:                                    # only the sum was used further on
            return None, gh, None, gh if ctx.two else None, None, None
        handle = ctx.handle
        a = _rms_args(hid, w, ctx.eps)
        gy = _inner(gy, 1)
        gx, gw = torch.empty(hid.shape, dtype=hid.dtype, device=hid.device), torch.empty_like(w)
        work = _work(handle, handle.lib.rgp_rms_norm_workspace(C.byref(a), 1))
        if residual is not None:
            a.residual, a.residual_st = residual.data_ptr(), residual.stride(0)
        if gh is not None:
            gh = _inner(gh, 1)
            a.ghid, a.ghid_st = gh.data_ptr(), gh.stride(0)
        a.rstd, a.gy, a.gy_st, a.gx, a.gw, a.work, a.work_bytes = rstd.data_ptr(), gy.data_ptr(), gy.stride(0), gx.data_ptr(), gw.data_ptr(), work.data_ptr(), work.numel()
        _call(handle, handle.lib.rgp_rms_norm_backward, a)
        return None, gx, gw, gx if ctx.two else None, None, None


def rms_norm(handle, x, weight, residual=None, eps=1e-6):
    """weight * hid / sqrt(mean(hid^2) + eps) over the last dimension, hid = x + residual.  Returns the norm, or (norm, hid) where a residual
    is given.  x, residual: any leading shape; weight (C,).  Gradients: x, residual, weight."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES or x.dim() < 1 or x.shape[-1] < 1:
        _bad('x must be a device tensor of float64, float32, bfloat16 or float16 with a last dimension')
    if x.device != handle.device:
        _bad('x is on %s, the handle on %s' % (x.device, handle.device))
    eps = float(eps)
    if not eps > 0.0 or math.isinf(eps):
        _bad('eps must be positive')
    w = _param('weight', weight, (x.shape[-1],), x)
    flat = lambda t: _inner(t.reshape(-1, t.shape[-1]), 1)                   # noqa: E731
    if residual is not None:
        _rows('residual', residual, x, x.shape)
        if residual.dim() != x.dim():
            _bad('residual has shape %s, x %s' % (tuple(residual.shape), tuple(x.shape)))
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight))
    r = _RmsFn.apply(handle, flat(x), w, None if residual is None else flat(residual), eps, train)
    return r.view(x.shape) if residual is None else (r[0].view(x.shape), r[1].view(x.shape))


# ---------------------------------------------------------------------------------------------------------------------- gradient norm
class _GradList(object):
    """Checked pointer table of one call."""

    def __init__(self, handle, grads):
        grads = list(grads)
        n = len(grads)
        spans = []
        self.ptr, self.numel, self.dtype = (C.c_void_p * max(n, 1))(), (C.c_int64 * max(n, 1))(), (C.c_int32 * max(n, 1))()
        for i, g in enumerate(grads):
            if not isinstance(g, torch.Tensor) or g.device != handle.device or g.dtype not in _DTYPES or g.layout != torch.strided:
                _bad('gradient %d must be a float64, float32, bfloat16 or float16 tensor on %s' % (i, handle.device))
            k = g.numel()
            if k and not g.is_contiguous() and (_overlaps(g) or sum((m - 1) * s for m, s in zip(g.shape, g.stride())) + 1 != k):
                _bad('gradient %d has gaps or repeats in memory: it cannot be clipped in place as one range' % i)
            p = g.data_ptr()
            self.ptr[i], self.numel[i], self.dtype[i] = p, k, _DTYPES[g.dtype]
            if k:
                spans.append((p, p + k * g.element_size()))
        spans.sort()
        for (_, e), (s, _) in zip(spans, spans[1:]):
            if s < e:
                _bad('two gradients share memory: each element may be clipped once')
        self.n = n


def grad_sumsq(handle, grads):
    """Sum of the squares of all elements of ``grads`` as a float64 device scalar (a data-parallel caller adds the ranks' sums)."""
    t = _GradList(handle, grads)
    out = torch.empty((), dtype=torch.float64, device=handle.device)
    work = _work(handle, handle.lib.rgp_grad_workspace(t.n, t.numel, t.dtype))
    handle._check(handle.lib.rgp_grad_sumsq(handle.h, _stream(handle), t.n, t.ptr, t.numel, t.dtype, out.data_ptr(), work.data_ptr(), work.numel()))
    return out


def clip_grad_norm(handle, grads, max_norm, sumsq=None):
    """Multiplies every tensor of ``grads`` in place by max_norm / (norm + 1e-6) where that is below 1; norm = the square root of the sum of
    all squares (taken in float64).  A norm that is not finite leaves the gradients as they are.  Returns the norm, a float64 device scalar;
    nothing is synchronised.  grads: dense tensors that share no memory, of any mix of types.  sumsq: the sum of squares to use instead of
    these tensors' own (grad_sumsq of several ranks, added up)."""
    max_norm = float(max_norm)
    if not max_norm > 0.0:
        _bad('max_norm must be positive')
    t = _GradList(handle, grads)
    norm = torch.empty((), dtype=torch.float64, device=handle.device)
    s = _stream(handle)
    if sumsq is None:
        work = _work(handle, handle.lib.rgp_grad_workspace(t.n, t.numel, t.dtype))
        handle._check(handle.lib.rgp_grad_sumsq(handle.h, s, t.n, t.ptr, t.numel, t.dtype, norm.data_ptr(), work.data_ptr(), work.numel()))
        src = norm
    else:
        if not isinstance(sumsq, torch.Tensor) or sumsq.dtype != torch.float64 or sumsq.numel() != 1 or sumsq.device != handle.device:
            _bad('sumsq must be one float64 value on %s' % handle.device)
        src = sumsq
    handle._check(handle.lib.rgp_grad_clip(handle.h, s, t.n, t.ptr, t.numel, t.dtype, src.data_ptr(), max_norm, norm.data_ptr()))
    return norm
