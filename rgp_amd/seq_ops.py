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

A captured backward pass needs leaves that no eager graph holds at that time (it is refused): take the gradients with torch.autograd.grad
inside the captured region, on a forward pass of the same region.  There are no second derivatives (a backward pass with
create_graph=True is refused) and no forward-mode ones (operands and gradients that carry a tangent are refused).  A
function that torch records (torch.jit.trace, make_fx) cannot hold these operators: refused too.  So is the backward pass of a graph whose handle
has been closed in between."""
import ctypes as C
import math

import torch

from . import _lib
from . import _seq                            # csrc/rgp_torch.cpp: checks, allocation and autograd nodes around the C entries
from ._lib import RgpError

_DTYPES = (torch.float64, torch.float32, torch.bfloat16, torch.float16)


def _bind():
    lib = _lib.load()
    _seq.bind(RgpError, {name: C.cast(getattr(lib, name), C.c_void_p).value for name in _lib.SYMBOLS if name.startswith(('rgp_ssm_', 'rgp_rms_', 'rgp_grad_'))
                         or name == 'rgp_last_error'})


_bind()


def _bad(msg):
    raise RgpError(_lib.RGP_ERR_BAD_ARG, msg)


def _acc(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _again(r, what):
    """The result of a call whose operands have been looked over (and made contiguous where that was all)."""
    if r is None:
        _bad('%s: operands that the library does not take' % what)
    return r


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


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
        given = lengths.tolist() if hasattr(lengths, 'tolist') else lengths
        try:
            given = list(given)
            lengths = [int(v) for v in given]
        except (TypeError, ValueError, OverflowError):
            lengths = None
        if lengths is None or any(v != g for v, g in zip(lengths, given)):
            _bad('the lengths of a sequence table must be a list of whole numbers, not %.200r' % (given,))
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


def _inner(t, dims):
    """The tensor with its last ``dims`` dimensions contiguous (a copy only where they are not, or where its memory holds the negated values)."""
    if t.is_neg():
        t = t.resolve_neg()
    if t.is_contiguous():
        return t
    shape, stride, want = t.shape, t.stride(), 1
    for i in range(1, dims + 1):
        if stride[-i] != want and shape[-i] > 1:
            return t.contiguous()
        want *= shape[-i]
    return t


def _geometry(handle, x, seqs, what, step=False):
    """(leading dimensions, sequences) of a (T, batch, D) or packed (rows, D) activation."""
    if not isinstance(x, torch.Tensor):
        _bad('%s must be a device tensor' % what)
    if x.dtype not in _DTYPES:
        _bad('%s must be float64, float32, bfloat16 or float16, not %s' % (what, x.dtype))
    if x.device != handle.device:
        _bad('%s is on %s, the handle on %s' % (what, x.device, handle.device))
    if step:                                     # (batch, D): one row of every sequence
        if x.numel() == 0:
            _bad('%s is empty: shape %s' % (what, tuple(x.shape)))
        return x.shape[:1], x.shape[0]
    if seqs is None:
        if x.dim() != 3:
            _bad('%s must be (T, batch, features); packed rows need a SeqTable' % what)
        T, n = x.shape[0], x.shape[1]
        if T < 1 or n < 1 or x.shape[2] < 1:
            _bad('%s is empty: shape %s' % (what, tuple(x.shape)))
        return x.shape[:2], n
    if x.dim() != 2 or x.shape[1] < 1:
        _bad('%s must be packed rows (rows, features) with a SeqTable' % what)
    if seqs.device != x.device:
        _bad('the sequence table is on %s, %s on %s' % (seqs.device, what, x.device))
    if seqs.rows != x.shape[0]:
        _bad('%s has %d rows, the sequence table %d' % (what, x.shape[0], seqs.rows))
    return x.shape[:1], seqs.n_seq


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
    return t if t.is_contiguous() and not t.is_neg() else t.resolve_neg().contiguous()


def _state(name, t, shape, dtype, x):
    """A state that is updated in place."""
    if not isinstance(t, torch.Tensor) or t.device != x.device or t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
        _bad('%s must be a contiguous %s tensor of shape %s on %s' % (name, dtype, tuple(shape), x.device))
    if t.is_neg():
        _bad('%s is updated in place: its memory must hold its values (resolve_neg)' % name)
    if t.requires_grad:
        _bad('%s is updated in place and takes no gradient' % name)


def _no_step_grad(*ts):
    if _wants_grad(*ts):
        _bad('a single step takes no gradients: call it under torch.no_grad()')


def _no_grad_state(name, t):
    if not isinstance(t, torch.Tensor):
        _bad('%s must be a tensor' % name)
    if t.requires_grad:
        _bad('%s takes no gradient: detach it' % name)


# ---------------------------------------------------------------------------------------------------------------------- convolution
def _conv_check(x, weight, bias):
    """x, filters and bias in the form the library takes."""
    D = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[1] <= 8:
        _bad('weight must be (D, W) with 2 to 8 taps')
    return _inner(x, 1), _param('weight', weight, (D, weight.shape[1]), x), _param('bias', bias, (D,), x, optional=True)


def ssm_conv(handle, x, weight, bias=None, seqs=None, init=None, reverse=False, return_state=False):
    """silu(bias + causal convolution of x with one filter per channel): v_t uses x_{t-W+1} .. x_t of its own sequence.

    x: (T, batch, D), or packed (rows, D) with ``seqs``; weight (D, W), 2 <= W <= 8; bias (D,).  init: (n_seq, W - 1, D), the inputs before
    the first step, oldest first (zeros without it); return_state=True also returns them for the step behind the last one.  reverse=True
    walks every sequence from its last step (init and the returned state are then those of that walk).  Gradients: x, weight, bias (states
    take none)."""
    r = _seq.conv(handle, x, weight, bias, seqs, init, bool(reverse), bool(return_state))
    if r is None:
        _, n_seq = _geometry(handle, x, seqs, 'x')
        x, w, b = _conv_check(x, weight, bias)
        if init is not None:
            _no_grad_state('init', init)
            shape = (n_seq, w.shape[1] - 1, x.shape[-1])
            if init.shape != shape or init.dtype is not x.dtype or init.device != x.device:
                _bad('init must be %s of shape %s on %s' % (x.dtype, shape, x.device))
            init = init.resolve_neg().contiguous()
        r = _again(_seq.conv(handle, x, w, b, seqs, init, bool(reverse), bool(return_state)), 'ssm_conv')
    return r if return_state else r[0]


def ssm_conv_step(handle, x, weight, bias, state):
    """One step of ``ssm_conv``: x (batch, D), state (batch, W - 1, D) of x's type, updated in place.  It takes no
    gradients: operands that require them are refused outside torch.no_grad()."""
    v = _seq.conv_step(handle, x, weight, bias, state)
    if v is None:
        if not isinstance(x, torch.Tensor) or x.dim() != 2:
            _bad('x must be (batch, D)')
        _geometry(handle, x, None, 'x', step=True)
        x, w, b = _conv_check(x, weight, bias)
        _no_step_grad(x, w, b)
        _state('state', state, (x.shape[0], w.shape[1] - 1, x.shape[1]), x.dtype, x)
        v = _again(_seq.conv_step(handle, x, w, b, state), 'ssm_conv_step')
    return v


# ---------------------------------------------------------------------------------------------------------------------- scan
def _scan_check(u, delta, A, B, Cm, D, z, delta_bias, lead):
    """Operands in the form the library takes: (.., D) activations with contiguous features, (.., N) or (.., G, N) maps, contiguous
    parameters."""
    nd, n = len(lead), u.shape[-1]
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
            None if z is None else _inner(z, 1), _param('delta_bias', delta_bias, (n,), u, optional=True))


def ssm_scan(handle, u, delta, A, B, Cm, D=None, z=None, delta_bias=None, seqs=None, init=None, reverse=False, return_state=False):
    """Selective state-space scan.  Per step, channel d and its group g of B / C:
        dt = softplus(delta + delta_bias);  s[n] = exp(dt A[d, n]) s[n] + dt u B[g, n];  y = (sum_n C[g, n] s[n] + D[d] u) z sigmoid(z)
    u, delta, z: (T, batch, Dn), or packed (rows, Dn) with ``seqs``; B, C: the same leading dimensions and (N,) or (G, N); A (Dn, N),
    N <= 64; D, delta_bias (Dn,).  init: (n_seq, Dn, N), the state before the first step (zeros without it); return_state=True also returns
    the state behind the last step.  reverse=True walks every sequence from its last step.  Gradients: u, delta, A, B, C, D, z, delta_bias
    (states take none).  A is meant to be negative: long sequences are walked in blocks of time, and where A is positive and exp(sum of dt A)
    over a block leaves the range of the arithmetic type, so does what the block makes of a state that is not zero."""
    r = _seq.scan(handle, u, delta, A, B, Cm, D, z, delta_bias, seqs, init, bool(reverse), bool(return_state))
    if r is None:
        lead, n_seq = _geometry(handle, u, seqs, 'u')
        ops = _scan_check(u, delta, A, B, Cm, D, z, delta_bias, lead)
        if init is not None:
            _no_grad_state('init', init)
            init = _param('init', init, (n_seq, u.shape[-1], A.shape[1]), u)
        r = _again(_seq.scan(handle, *ops, seqs, init, bool(reverse), bool(return_state)), 'ssm_scan')
    return r if return_state else r[0]


def ssm_scan_step(handle, u, delta, A, B, Cm, D, state, z=None, delta_bias=None):
    """One step of ``ssm_scan``: u, delta, z (batch, Dn); B, C (batch, N) or (batch, G, N); state (batch, Dn, N), updated in place.  It
    takes no gradients: operands that require them are refused outside torch.no_grad()."""
    y = _seq.scan_step(handle, u, delta, A, B, Cm, D, z, delta_bias, state)
    if y is None:
        if not isinstance(u, torch.Tensor) or u.dim() != 2:
            _bad('u must be (batch, D)')
        lead, n = _geometry(handle, u, None, 'u', step=True)
        _no_step_grad(u, delta, A, B, Cm, D, z, delta_bias)
        ops = _scan_check(u, delta, A, B, Cm, D, z, delta_bias, lead)
        _state('state', state, (n, u.shape[1], A.shape[1]), _acc(u.dtype), u)
        y = _again(_seq.scan_step(handle, *ops, state), 'ssm_scan_step')
    return y


# ---------------------------------------------------------------------------------------------------------------------- norm
def rms_norm(handle, x, weight, residual=None, eps=1e-6):
    """weight * hid / sqrt(mean(hid^2) + eps) over the last dimension, hid = x + residual.  Returns the norm, or (norm, hid) where a residual
    is given.  x, residual: any leading shape; weight (C,).  Gradients: x, residual, weight."""
    eps = float(eps)
    r = _seq.rms(handle, x, weight, residual, eps)
    if r is None:
        if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES or x.dim() < 1 or x.shape[-1] < 1:
            _bad('x must be a device tensor of float64, float32, bfloat16 or float16 with a last dimension')
        if x.device != handle.device:
            _bad('x is on %s, the handle on %s' % (x.device, handle.device))
        if not eps > 0.0 or math.isinf(eps):
            _bad('eps must be positive')
        shape = x.shape
        w = _param('weight', weight, shape[-1:], x)
        rows = lambda t: _inner(t if t.dim() == 2 else t.reshape(-1, shape[-1]), 1)                          # noqa: E731
        if residual is not None:
            _rows('residual', residual, x, shape)
            if residual.dim() != x.dim():
                _bad('residual has shape %s, x %s' % (tuple(residual.shape), tuple(shape)))
            residual = rows(residual)
        y, hid = _again(_seq.rms(handle, rows(x), w, residual, eps), 'rms_norm')
        r = y.view(shape), None if hid is None else hid.view(shape)
    return r[0] if residual is None else r


# ---------------------------------------------------------------------------------------------------------------------- gradient norm
def _bad_grads(handle, grads):
    """Names what is wrong with a list of gradients."""
    for i, g in enumerate(grads):
        if not isinstance(g, torch.Tensor) or g.dtype not in _DTYPES or g.device != handle.device or g.layout is not torch.strided:
            _bad('gradient %d must be a float64, float32, bfloat16 or float16 tensor on %s' % (i, handle.device))
        if g.is_neg():
            _bad('gradient %d is clipped in place: its memory must hold its values (resolve_neg)' % i)
        if not g.is_contiguous() and g.numel() and (_overlaps(g) or sum((m - 1) * s for m, s in zip(g.shape, g.stride())) + 1 != g.numel()):
            _bad('gradient %d has gaps or repeats in memory: it cannot be clipped in place as one range' % i)
    _bad('two gradients share memory: each element may be clipped once')


def grad_sumsq(handle, grads):
    """Sum of the squares of all elements of ``grads`` as a float64 device scalar (a data-parallel caller adds the ranks' sums)."""
    grads = list(grads)
    r = _seq.sumsq(handle, grads)
    return _bad_grads(handle, grads) if r is None else r


def clip_grad_norm(handle, grads, max_norm, sumsq=None):
    """Multiplies every tensor of ``grads`` in place by max_norm / (norm + 1e-6) where that is below 1; norm = the square root of the sum of
    all squares (taken in float64).  A norm that is not finite leaves the gradients as they are.  Returns the norm, a float64 device scalar;
    nothing is synchronised.  grads: dense tensors that share no memory, of any mix of types.  sumsq: the sum of squares to use instead of
    these tensors' own (grad_sumsq of several ranks, added up)."""
    max_norm = float(max_norm)
    if not max_norm > 0.0:
        _bad('max_norm must be positive')
    grads = list(grads)
    r = _seq.clip(handle, grads, max_norm, sumsq)
    if r is None:
        if sumsq is not None and (not isinstance(sumsq, torch.Tensor) or sumsq.dtype is not torch.float64 or sumsq.numel() != 1 or
                                  sumsq.device != handle.device):
            _bad('sumsq must be one float64 value on %s' % handle.device)
        if sumsq is not None and sumsq.is_neg():
            return clip_grad_norm(handle, grads, max_norm, sumsq.resolve_neg())
        _bad_grads(handle, grads)
    return r
