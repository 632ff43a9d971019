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
captured region, on a forward pass of the same region.  There are no second derivatives: a backward pass with create_graph=True is refused."""
import math
import struct

import torch

from . import _lib
from ._lib import RgpError

_DTYPES = {torch.float64: _lib.DT_F64, torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


def _bad(msg):
    raise RgpError(_lib.RGP_ERR_BAD_ARG, msg)


def _acc(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _stream(handle):
    return torch._C._cuda_getCurrentRawStream(handle.device.index)


# The argument structs of include/rgp_hip.h as one pack each (a ctypes struct costs several microseconds to fill, as much as a short kernel
# runs); the last two fields, work and work_bytes, are packed apart because their size is asked for with the others.
_SCAN, _CONV, _RMS = struct.Struct('@6i3q6Q12q16Q'), struct.Struct('@6i3q2Q4q9Q'), struct.Struct('@2i2qd2Q4q8Q')
_WORK, _NO_WORK = struct.Struct('@Qq'), b'\0' * 16


def _call(handle, fn, head, tail=_NO_WORK):
    st = fn(handle.h, _stream(handle), head + tail)
    if st != 0:
        handle._check(st)


def _new_work(handle, query, head, backward):
    """The work buffer of a call and its fields of the struct."""
    n = query(head + _NO_WORK, backward)
    if n <= 0:
        return None, _NO_WORK
    w = torch.empty(n, dtype=torch.uint8, device=handle.device)
    return w, _WORK.pack(w.data_ptr(), n)


def _new_like(t):
    return None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _wants_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _once():
    if torch.is_grad_enabled():
        raise RuntimeError('the sequence operators have no second derivatives (create_graph=True)')


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
        if self.device.type == 'cuda':                     # there for every stream from now on
            torch.cuda.current_stream(self.device).synchronize()


def _rows(name, t, like, lead):
    """Checks an activation's type, place and leading shape."""
    if not isinstance(t, torch.Tensor):
        _bad('%s must be a device tensor' % name)
    if t.dtype is not like.dtype or t.device != like.device:
        _bad('%s is %s on %s, %s on %s expected' % (name, t.dtype, t.device, like.dtype, like.device))
    if t.shape[:len(lead)] != lead:
        _bad('%s has shape %s, leading dimensions %s expected' % (name, tuple(t.shape), tuple(lead)))


def _all_plain(x, acts, params):
    """True for contiguous activations of x's type and parameters of its arithmetic type (or None), all on x's device: the common case, found
    in one pass.  Anything else goes through the checks that name what is wrong."""
    dt, dev = x.dtype, x.device
    acc = torch.float64 if dt is torch.float64 else torch.float32
    try:
        for t in acts:
            if t.dtype is not dt or t.device != dev or not t.is_contiguous():
                return False
        for t in params:
            if t is not None and (t.dtype is not acc or t.device != dev or not t.is_contiguous()):
                return False
    except AttributeError:
        return False
    return True


def _inner(t, dims):
    """The tensor with its last ``dims`` dimensions contiguous (a copy only where they are not)."""
    if t.is_contiguous():
        return t
    shape, stride, want = t.shape, t.stride(), 1
    for i in range(1, dims + 1):
        if stride[-i] != want and shape[-i] > 1:
            return t.contiguous()
        want *= shape[-i]
    return t


def _geometry(handle, x, seqs, what, step=False):
    """(lead, n_seq, T, rows, max_len, off) of a (T, batch, D) or packed (rows, D) activation."""
    if not isinstance(x, torch.Tensor):
        _bad('%s must be a device tensor' % what)
    if x.dtype not in _DTYPES:
        _bad('%s must be float64, float32, bfloat16 or float16, not %s' % (what, x.dtype))
    if x.device != handle.device:
        _bad('%s is on %s, the handle on %s' % (what, x.device, handle.device))
    if step:                                     # (batch, D): one row of every sequence
        if x.numel() == 0:
            _bad('%s is empty: shape %s' % (what, tuple(x.shape)))
        return x.shape[:1], x.shape[0], 1, x.shape[0], 1, None
    if seqs is None:
        if x.dim() != 3:
            _bad('%s must be (T, batch, features); packed rows need a SeqTable' % what)
        T, n = x.shape[0], x.shape[1]
        if T < 1 or n < 1 or x.shape[2] < 1:
            _bad('%s is empty: shape %s' % (what, tuple(x.shape)))
        return x.shape[:2], n, T, T * n, T, None
    if x.dim() != 2 or x.shape[1] < 1:
        _bad('%s must be packed rows (rows, features) with a SeqTable' % what)
    if seqs.device != x.device:
        _bad('the sequence table is on %s, %s on %s' % (seqs.device, what, x.device))
    if seqs.rows != x.shape[0]:
        _bad('%s has %d rows, the sequence table %d' % (what, x.shape[0], seqs.rows))
    return x.shape[:1], seqs.n_seq, 0, seqs.rows, seqs.max_len, seqs.off


def _strides(t, packed):
    """Element strides of (step, sequence)."""
    st = t.stride()
    return (st[0], 0) if packed else (st[0], st[1])


def _param(name, t, shape, x, optional=False):
    if t is None:
        if optional:
            return None
        _bad('%s is required' % name)
    if not isinstance(t, torch.Tensor) or t.device != x.device:
        _bad('%s must be a tensor on %s' % (name, x.device))
    if t.shape != shape:
        _bad('%s has shape %s, %s expected' % (name, tuple(t.shape), tuple(shape)))
    if t.dtype is not _acc(x.dtype):
        _bad('%s is %s: parameters and states are %s for %s activations' % (name, t.dtype, _acc(x.dtype), x.dtype))
    return t if t.is_contiguous() else t.contiguous()


def _state(name, t, shape, dtype, x):
    """A state that is updated in place."""
    if not isinstance(t, torch.Tensor) or t.device != x.device or t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
        _bad('%s must be a contiguous %s tensor of shape %s on %s' % (name, dtype, tuple(shape), x.device))
    if t.requires_grad:
        _bad('%s is updated in place and takes no gradient' % name)
    torch.autograd.graph.increment_version(t)       # a graph that saved the state notices the update
    return t


def _no_step_grad(*ts):
    if _wants_grad(*ts):
        _bad('a single step takes no gradients: call it under torch.no_grad()')


def _no_grad_state(name, t):
    if t is not None and t.requires_grad:
        _bad('%s takes no gradient: detach it' % name)


# ---------------------------------------------------------------------------------------------------------------------- convolution
def _conv_head(x, w, bias, geo, reverse, init=0, v=0, last=0, gv=0, gv_st=(0, 0), gx=0, gw=0, gb=0):
    _, n_seq, T, rows, max_len, off = geo
    st = _strides(x, off is not None)
    return _CONV.pack(_DTYPES[x.dtype], n_seq, x.shape[-1], w.shape[1], reverse, 0, T, rows, max_len, _ptr(off), x.data_ptr(), st[0], st[1], gv_st[0],
                      gv_st[1], w.data_ptr(), _ptr(bias), init, v, last, gv, gx, gw, gb)


def _conv_forward(handle, x, w, bias, init, geo, reverse, want_last):
    v = _new_like(x)
    last = torch.empty(geo[1], w.shape[1] - 1, x.shape[-1], dtype=x.dtype, device=x.device) if want_last else None
    _call(handle, handle.lib.rgp_ssm_conv_forward, _conv_head(x, w, bias, geo, reverse, _ptr(init), v.data_ptr(), _ptr(last)))
    return v, last


class _ConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, handle, x, w, bias, init, geo, reverse, want_last):
        v, last = _conv_forward(handle, x, w, bias, init, geo, reverse, want_last)
        ctx.handle, ctx.geo, ctx.reverse = handle, geo, reverse
        ctx.save_for_backward(x, w, bias, init)
        ctx.set_materialize_grads(False)
        if want_last:
            ctx.mark_non_differentiable(last)
        return v, last

    @staticmethod
    def backward(ctx, gv, _):
        _once()
        if gv is None:
            return (None,) * 8
        x, w, bias, init = ctx.saved_tensors
        handle = ctx.handle
        gv = _inner(gv, 1)
        gx, gw, gb = _new_like(x), _new_like(w), _new_like(bias)
        head = _conv_head(x, w, bias, ctx.geo, ctx.reverse, _ptr(init), 0, 0, gv.data_ptr(), _strides(gv, ctx.geo[5] is not None), gx.data_ptr(),
                          gw.data_ptr(), _ptr(gb))
        work, tail = _new_work(handle, handle.lib.rgp_ssm_conv_workspace, head, 1)
        _call(handle, handle.lib.rgp_ssm_conv_backward, head, tail)
        return None, gx, gw, gb, None, None, None, None


def _conv_check(x, weight, bias):
    """x, filters and bias in the form the library takes."""
    D = x.shape[-1]
    if _all_plain(x, (x,), (weight, bias)):
        sw = weight.shape
        if len(sw) == 2 and sw[0] == D and 2 <= sw[1] <= 8 and (bias is None or bias.shape == (D,)):
            return x, weight, bias
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[1] <= 8:
        _bad('weight must be (D, W) with 2 to 8 taps')
    return _inner(x, 1), _param('weight', weight, (D, weight.shape[1]), x), _param('bias', bias, (D,), x, optional=True)


def ssm_conv(handle, x, weight, bias=None, seqs=None, init=None, reverse=False, return_state=False):
    """silu(bias + causal convolution of x with one filter per channel): v_t uses x_{t-W+1} .. x_t of its own sequence.

    x: (T, batch, D), or packed (rows, D) with ``seqs``; weight (D, W), 2 <= W <= 8; bias (D,).  init: (n_seq, W - 1, D), the inputs before
    the first step, oldest first (zeros without it); return_state=True also returns them for the step behind the last one.  reverse=True
    walks every sequence from its last step (init and the returned state are then those of that walk).  Gradients: x, weight, bias (states
    take none)."""
    geo = _geometry(handle, x, seqs, 'x')
    D = x.shape[-1]
    x, w, b = _conv_check(x, weight, bias)
    if init is not None:
        _no_grad_state('init', init)
        if init.shape != (geo[1], w.shape[1] - 1, D) or init.dtype is not x.dtype or init.device != x.device:
            _bad('init must be %s of shape %s on %s' % (x.dtype, (geo[1], w.shape[1] - 1, D), x.device))
        init = init.contiguous()
    run = _ConvFn.apply if _wants_grad(x, w, b) else _conv_forward
    v, last = run(handle, x, w, b, init, geo, bool(reverse), bool(return_state))
    return (v, last) if return_state else v


def ssm_conv_step(handle, x, weight, bias, state):
    """One step of ``ssm_conv``: x (batch, D), state (batch, W - 1, D) of x's type, updated in place.  It takes no
    gradients: operands that require them are refused outside torch.no_grad()."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        _bad('x must be (batch, D)')
    geo = _geometry(handle, x, None, 'x', step=True)
    D = x.shape[1]
    x, w, b = _conv_check(x, weight, bias)
    _no_step_grad(x, w, b)
    _state('state', state, (x.shape[0], w.shape[1] - 1, D), x.dtype, x)
    v, st = _new_like(x), state.data_ptr()
    _call(handle, handle.lib.rgp_ssm_conv_step, _CONV.pack(_DTYPES[x.dtype], x.shape[0], D, w.shape[1], 0, 0, 1, x.shape[0], 1, 0, x.data_ptr(), 0,
                                                          x.stride(0), 0, 0, w.data_ptr(), _ptr(b), st, v.data_ptr(), st, 0, 0, 0, 0))
    return v


# ---------------------------------------------------------------------------------------------------------------------- scan
def _scan_head(ops, geo, G, reverse, init=0, y=0, last=0, states=0, gy=0, gy_st=(0, 0), grads=(0,) * 8):
    u, delta, A, B, Cm, skip, z, bias = ops
    _, n_seq, T, rows, max_len, off = geo
    packed = off is not None
    su, sd, sB, sC = _strides(u, packed), _strides(delta, packed), _strides(B, packed), _strides(Cm, packed)
    sz = _strides(z, packed) if z is not None else (0, 0)
    gu, gdelta, gA, gB, gC, gskip, gz, gbias = grads
    return _SCAN.pack(_DTYPES[u.dtype], n_seq, u.shape[-1], A.shape[1], G, reverse, T, rows, max_len, _ptr(off), u.data_ptr(),
                      delta.data_ptr(), _ptr(z), B.data_ptr(), Cm.data_ptr(), su[0], su[1], sd[0], sd[1], sz[0], sz[1], sB[0], sB[1], sC[0], sC[1],
                      gy_st[0], gy_st[1], A.data_ptr(), _ptr(skip), _ptr(bias), init, y, last, states, gy, gu, gdelta, gz, gB, gC, gA, gskip, gbias)


def _scan_forward(handle, u, delta, A, B, Cm, skip, z, bias, init, geo, G, reverse, want_last, train=False):
    ops = (u, delta, A, B, Cm, skip, z, bias)
    y = _new_like(u)
    last = torch.empty(geo[1], u.shape[-1], A.shape[1], dtype=A.dtype, device=u.device) if want_last else None
    states = None
    if train:
        # a state of N every 8 steps of every sequence: (blocks of 8) D N values (rgp_ssm_scan_states_bytes)
        blocks = (geo[3] >> 3) + geo[1] if geo[5] is not None else geo[1] * ((geo[2] + 7) >> 3)
        states = torch.empty(blocks * A.numel(), dtype=A.dtype, device=u.device)
    head = _scan_head(ops, geo, G, reverse, _ptr(init), y.data_ptr(), _ptr(last), _ptr(states))
    work, tail = _new_work(handle, handle.lib.rgp_ssm_scan_workspace, head, 0)
    _call(handle, handle.lib.rgp_ssm_scan_forward, head, tail)
    return (y, last, states) if train else (y, last)


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, handle, u, delta, A, B, Cm, skip, z, bias, init, geo, G, reverse, want_last):
        y, last, states = _scan_forward(handle, u, delta, A, B, Cm, skip, z, bias, init, geo, G, reverse, want_last, True)
        ctx.handle, ctx.geo, ctx.G, ctx.reverse = handle, geo, G, reverse
        ctx.save_for_backward(u, delta, A, B, Cm, skip, z, bias, states)
        ctx.set_materialize_grads(False)
        if want_last:
            ctx.mark_non_differentiable(last)
        return y, last

    @staticmethod
    def backward(ctx, gy, _):
        _once()
        if gy is None:
            return (None,) * 14
        saved = ctx.saved_tensors
        ops, states, handle = saved[:8], saved[8], ctx.handle
        gy = _inner(gy, 1)
        grads = [_new_like(t) for t in ops]
        head = _scan_head(ops, ctx.geo, ctx.G, ctx.reverse, states=states.data_ptr(), gy=gy.data_ptr(), gy_st=_strides(gy, ctx.geo[5] is not None),
                          grads=[_ptr(t) for t in grads])
        work, tail = _new_work(handle, handle.lib.rgp_ssm_scan_workspace, head, 1)
        _call(handle, handle.lib.rgp_ssm_scan_backward, head, tail)
        return (None, *grads, None, None, None, None, None)


def _scan_check(u, delta, A, B, Cm, D, z, delta_bias, lead):
    """Operands in the form the library takes: (.., D) activations with contiguous features, (.., N) or (.., G, N) maps, contiguous
    parameters."""
    nd, n = len(lead), u.shape[-1]
    if _all_plain(u, (u, delta, B, Cm) if z is None else (u, delta, B, Cm, z), (A, D, delta_bias)):      # then only the shapes are left to check
        sh, sb, N = u.shape, B.shape, A.shape[-1]
        G = 1 if len(sb) == nd + 1 else sb[-2] if len(sb) == nd + 2 else 0
        if delta.shape == sh and (z is None or z.shape == sh) and Cm.shape == sb and sb[:nd] == lead and sb[-1] == N and G and not n % G and 1 <= N <= 64 \
                and A.shape == (n, N) and (D is None or D.shape == (n,)) and (delta_bias is None or delta_bias.shape == (n,)):
            return (u, delta, A, B, Cm, D, z, delta_bias), G
    for name, t in (('delta', delta), ('z', z)):
        if t is not None:
            _rows(name, t, u, lead)
            if t.shape != u.shape:
                _bad('%s has shape %s, %s expected' % (name, tuple(t.shape), tuple(u.shape)))
    if delta is None:
        _bad('delta is required')
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= 64:
        _bad('A must be (D, N) with 1 to 64 states')
    N = A.shape[1]
    maps, groups = [], []
    for name, t in (('B', B), ('C', Cm)):
        _rows(name, t, u, lead)
        G = 1 if t.dim() == nd + 1 else t.shape[-2] if t.dim() == nd + 2 else 0
        if t.shape[-1] != N or G < 1 or n % G:
            _bad('%s has shape %s: (.., N) or (.., G, N) with N = %d and G a divisor of D = %d expected' % (name, tuple(t.shape), N, n))
        groups.append(G)
        maps.append(_inner(t, t.dim() - nd))
    if groups[0] != groups[1]:
        _bad('B has %d groups, C %d' % tuple(groups))
    return (_inner(u, 1), _inner(delta, 1), _param('A', A, (n, N), u), maps[0], maps[1], _param('D', D, (n,), u, optional=True),
            None if z is None else _inner(z, 1), _param('delta_bias', delta_bias, (n,), u, optional=True)), groups[0]


def ssm_scan(handle, u, delta, A, B, Cm, D=None, z=None, delta_bias=None, seqs=None, init=None, reverse=False, return_state=False):
    """Selective state-space scan.  Per step, channel d and its group g of B / C:
        dt = softplus(delta + delta_bias);  s[n] = exp(dt A[d, n]) s[n] + dt u B[g, n];  y = (sum_n C[g, n] s[n] + D[d] u) z sigmoid(z)
    u, delta, z: (T, batch, Dn), or packed (rows, Dn) with ``seqs``; B, C: the same leading dimensions and (N,) or (G, N); A (Dn, N),
    N <= 64; D, delta_bias (Dn,).  init: (n_seq, Dn, N), the state before the first step (zeros without it); return_state=True also returns
    the state behind the last step.  reverse=True walks every sequence from its last step.  Gradients: u, delta, A, B, C, D, z, delta_bias
    (states take none)."""
    geo = _geometry(handle, u, seqs, 'u')
    ops, G = _scan_check(u, delta, A, B, Cm, D, z, delta_bias, geo[0])
    if init is not None:
        _no_grad_state('init', init)
        init = _param('init', init, (geo[1], u.shape[-1], A.shape[1]), u)
    run = _ScanFn.apply if _wants_grad(*ops) else _scan_forward
    y, last = run(handle, *ops, init, geo, G, bool(reverse), bool(return_state))
    return (y, last) if return_state else y


def ssm_scan_step(handle, u, delta, A, B, Cm, D, state, z=None, delta_bias=None):
    """One step of ``ssm_scan``: u, delta, z (batch, Dn); B, C (batch, N) or (batch, G, N); state (batch, Dn, N), updated in place.  It
    takes no gradients: operands that require them are refused outside torch.no_grad()."""
    if not isinstance(u, torch.Tensor) or u.dim() != 2:
        _bad('u must be (batch, D)')
    geo = _geometry(handle, u, None, 'u', step=True)
    _no_step_grad(u, delta, A, B, Cm, D, z, delta_bias)
    (u, delta, A, B, Cm, skip, z, bias), G = _scan_check(u, delta, A, B, Cm, D, z, delta_bias, geo[0])
    n, Dn = u.shape
    N = A.shape[1]
    _state('state', state, (n, Dn, N), A.dtype, u)
    y, st = _new_like(u), state.data_ptr()
    _call(handle, handle.lib.rgp_ssm_scan_step, _SCAN.pack(
        _DTYPES[u.dtype], n, Dn, N, G, 0, 1, n, 1, 0, u.data_ptr(), delta.data_ptr(), _ptr(z), B.data_ptr(), Cm.data_ptr(), 0, u.stride(0), 0,
        delta.stride(0), 0, 0 if z is None else z.stride(0), 0, B.stride(0), 0, Cm.stride(0), 0, 0, A.data_ptr(), _ptr(skip), _ptr(bias), st,
        y.data_ptr(), st, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0))
    return y


# ---------------------------------------------------------------------------------------------------------------------- norm
def _rms_head(x, w, residual, eps, y=0, hid=0, rstd=0, gy=None, gh=None, gx=0, gw=0):
    st = lambda t: 0 if t is None else t.stride(0)                           # noqa: E731
    return _RMS.pack(_DTYPES[x.dtype], 0, x.shape[0], x.shape[1], eps, x.data_ptr(), _ptr(residual), x.stride(0), st(residual), st(gy), st(gh),
                     w.data_ptr(), y, hid, rstd, _ptr(gy), _ptr(gh), gx, gw)


def _rms_forward(handle, x, w, residual, eps, train=False):
    y = _new_like(x)
    hid = _new_like(x) if residual is not None else None
    rstd = torch.empty(x.shape[0], dtype=w.dtype, device=x.device) if train else None
    _call(handle, handle.lib.rgp_rms_norm_forward, _rms_head(x, w, residual, eps, y.data_ptr(), _ptr(hid), _ptr(rstd)))
    return (y, hid, rstd) if train else (y, hid)


class _RmsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, handle, x, w, residual, eps):
        y, hid, rstd = _rms_forward(handle, x, w, residual, eps, True)
        ctx.handle, ctx.eps, ctx.two = handle, eps, residual is not None
        # 16-bit: the backward pass adds x and residual again, hid's rounding would show in the weight's gradient; 32 and 64 bits: hid is that sum
        again = residual is not None and x.element_size() == 2
        ctx.save_for_backward(x if again or residual is None else hid, residual if again else None, w, rstd)
        ctx.set_materialize_grads(False)
        return y, hid

    @staticmethod
    def backward(ctx, gy, gh):
        _once()
        hid, residual, w, rstd = ctx.saved_tensors
        if gy is None:                                    # only the sum was used further on
            return None, gh, None, gh if ctx.two else None, None
        handle = ctx.handle
        gy, gh = _inner(gy, 1), None if gh is None else _inner(gh, 1)
        gx, gw = _new_like(hid), _new_like(w)
        head = _rms_head(hid, w, residual, ctx.eps, rstd=rstd.data_ptr(), gy=gy, gh=gh, gx=gx.data_ptr(), gw=gw.data_ptr())
        work, tail = _new_work(handle, handle.lib.rgp_rms_norm_workspace, head, 1)
        _call(handle, handle.lib.rgp_rms_norm_backward, head, tail)
        return None, gx, gw, gx if ctx.two else None, None


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
    shape, two = x.shape, x.dim() == 2
    if two and _all_plain(x, (x,) if residual is None else (x, residual), (weight,)) and weight.shape == shape[1:] and (residual is None or residual.shape == shape):
        x2, r2, w = x, residual, weight
    else:
        w = _param('weight', weight, shape[-1:], x)
        if residual is not None:
            _rows('residual', residual, x, shape)
            if residual.dim() != x.dim():
                _bad('residual has shape %s, x %s' % (tuple(residual.shape), tuple(shape)))
        x2 = _inner(x if two else x.reshape(-1, shape[-1]), 1)
        r2 = None if residual is None else _inner(residual if two else residual.reshape(-1, shape[-1]), 1)
    y, hid = (_RmsFn.apply if _wants_grad(x2, r2, w) else _rms_forward)(handle, x2, w, r2, eps)
    if not two:
        y, hid = y.view(shape), None if hid is None else hid.view(shape)
    return y if residual is None else (y, hid)


# ---------------------------------------------------------------------------------------------------------------------- gradient norm
def _grad_list(handle, grads):
    """(n, addresses, element counts, types) of one call's tensors, checked; the arrays live as long as the tuple."""
    n, dev = len(grads), handle.device
    try:
        plain = all([g.device == dev and g.is_contiguous() for g in grads])
        dtype = [_DTYPES[g.dtype] for g in grads]
    except (AttributeError, KeyError, RuntimeError):
        plain = False
    if not plain:
        for i, g in enumerate(grads):
            if not isinstance(g, torch.Tensor) or g.dtype not in _DTYPES or g.device != dev or g.layout is not torch.strided:
                _bad('gradient %d must be a float64, float32, bfloat16 or float16 tensor on %s' % (i, dev))
            if not g.is_contiguous() and g.numel() and (_overlaps(g) or sum((m - 1) * s for m, s in zip(g.shape, g.stride())) + 1 != g.numel()):
                _bad('gradient %d has gaps or repeats in memory: it cannot be clipped in place as one range' % i)
    ptr, numel = [g.data_ptr() for g in grads], [g.numel() for g in grads]
    end = 0
    for p, k, d in sorted(zip(ptr, numel, dtype)):
        if p < end and k:
            _bad('two gradients share memory: each element may be clipped once')
        end = max(end, p + k * _BYTES[d])
    return n, struct.pack('%dQ' % n, *ptr), struct.pack('%dq' % n, *numel), struct.pack('%di' % n, *dtype)


_BYTES = {_lib.DT_F64: 8, _lib.DT_F32: 4, _lib.DT_BF16: 2, _lib.DT_F16: 2}


def grad_sumsq(handle, grads):
    """Sum of the squares of all elements of ``grads`` as a float64 device scalar (a data-parallel caller adds the ranks' sums)."""
    n, ptr, numel, dtype = _grad_list(handle, list(grads))
    nbytes = handle.lib.rgp_grad_workspace(n, numel, dtype)
    buf = torch.empty(1 + nbytes // 8, dtype=torch.float64, device=handle.device)
    p = buf.data_ptr()
    handle._check(handle.lib.rgp_grad_sumsq(handle.h, _stream(handle), n, ptr, numel, dtype, p, p + 8, nbytes))
    return buf[0]


def clip_grad_norm(handle, grads, max_norm, sumsq=None):
    """Multiplies every tensor of ``grads`` in place by max_norm / (norm + 1e-6) where that is below 1; norm = the square root of the sum of
    all squares (taken in float64).  A norm that is not finite leaves the gradients as they are.  Returns the norm, a float64 device scalar;
    nothing is synchronised.  grads: dense tensors that share no memory, of any mix of types.  sumsq: the sum of squares to use instead of
    these tensors' own (grad_sumsq of several ranks, added up)."""
    max_norm = float(max_norm)
    if not max_norm > 0.0:
        _bad('max_norm must be positive')
    grads = list(grads)
    n, ptr, numel, dtype = _grad_list(handle, grads)
    nbytes = 0
    if sumsq is None:
        nbytes = handle.lib.rgp_grad_workspace(n, numel, dtype)
    elif not isinstance(sumsq, torch.Tensor) or sumsq.dtype is not torch.float64 or sumsq.numel() != 1 or sumsq.device != handle.device:
        _bad('sumsq must be one float64 value on %s' % handle.device)
    buf = torch.empty(1 + nbytes // 8, dtype=torch.float64, device=handle.device)
    p = buf.data_ptr()
    torch.autograd.graph.increment_version(grads)
    handle._check(handle.lib.rgp_grad_clip(handle.h, _stream(handle), n, ptr, numel, dtype, _ptr(sumsq), max_norm, p, p + 8 if nbytes else 0, nbytes))
    return buf[0]
