"""Calls of the sequence operators that are refused before the library is entered, whatever the device."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from test_seq_ops_cpu import H, _refused


def _calls():
    """{name: (function of its operands, operands)} for every entry point that takes tensors."""
    from rgp_amd import seq_ops
    z = torch.zeros
    return {
        'conv': (lambda x, w, b, init: seq_ops.ssm_conv(H, x, w, b, init=init), [z(5, 2, 6), z(6, 4), z(6), z(2, 3, 6)]),
        'conv_step': (lambda x, w, b, st: seq_ops.ssm_conv_step(H, x, w, b, st), [z(2, 6), z(6, 4), z(6), z(2, 3, 6)]),
        'scan': (lambda u, d, A, B, Cm, D, zz, b, init: seq_ops.ssm_scan(H, u, d, A, B, Cm, D=D, z=zz, delta_bias=b, init=init),
                 [z(5, 2, 6), z(5, 2, 6), z(6, 3), z(5, 2, 3), z(5, 2, 3), z(6), z(5, 2, 6), z(6), z(2, 6, 3)]),
        'scan_step': (lambda u, d, A, B, Cm, D, st, zz, b: seq_ops.ssm_scan_step(H, u, d, A, B, Cm, D, st, z=zz, delta_bias=b),
                      [z(2, 6), z(2, 6), z(6, 3), z(2, 3), z(2, 3), z(6), z(2, 6, 3), z(2, 6), z(6)]),
        'rms': (lambda x, w, r: seq_ops.rms_norm(H, x, w, residual=r), [z(3, 4), z(4), z(3, 4)]),
        'rms of three dimensions': (lambda x, w, r: seq_ops.rms_norm(H, x, w, residual=r), [z(2, 3, 4), z(4), z(2, 3, 4)]),
        'sumsq': (lambda a, b: seq_ops.grad_sumsq(H, [a, b]), [z(3), z(4)]),
        'clip': (lambda a, b, s: seq_ops.clip_grad_norm(H, [a, b], 1.0, sumsq=s), [z(3), z(4), z(1, dtype=torch.float64)]),
    }


@pytest.mark.parametrize('name', list(_calls()))
def test_operands_with_a_tangent_are_refused(name):
    """Forward-mode derivatives: every operand that carries a tangent, one at a time; inside a dual level, tensors without one are as ever."""
    f, ops = _calls()[name]
    with fwad.dual_level():
        for i, t in enumerate(ops):
            with torch.no_grad():                                   # a step refuses gradients first
                dual = list(ops)
                dual[i] = fwad.make_dual(t, torch.ones_like(t))
                _refused(lambda: f(*dual), 'forward-mode')
        _refused(lambda: f(*ops), '^(?!.*forward-mode)')


@pytest.mark.parametrize('name', list(_calls()))
def test_recording_a_function_is_refused(name):
    """torch.jit.trace and make_fx see allocations only: a recorded function would return memory that nothing has written."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, ops = _calls()[name]
    with torch.no_grad():
        _refused(lambda: torch.jit.trace(lambda x: f(x, *ops[1:]), ops[0], check_trace=False), 'cannot be recorded')
        _refused(lambda: make_fx(lambda x: f(x, *ops[1:]))(ops[0]), 'cannot be recorded')


def _negated(t):
    """The values of ``t`` as the imaginary part of a conjugate: memory that holds them negated."""
    v = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert v.is_neg() and torch.equal(v, t)
    return v


def test_in_place_operands_with_a_pending_negation_are_refused():
    from rgp_amd import seq_ops
    z = lambda *s: torch._neg_view(torch.zeros(*s))                         # noqa: E731
    _refused(lambda: seq_ops.ssm_conv_step(H, torch.zeros(2, 6), torch.zeros(6, 4), None, z(2, 3, 6)), 'resolve_neg')
    _refused(lambda: seq_ops.ssm_scan_step(H, torch.zeros(2, 6), torch.zeros(2, 6), torch.zeros(6, 3), torch.zeros(2, 3), torch.zeros(2, 3), None, z(2, 6, 3)),
             'resolve_neg')
    _refused(lambda: seq_ops.clip_grad_norm(H, [z(5)], 1.0), 'gradient 0 is clipped in place')
    _refused(lambda: seq_ops.clip_grad_norm(H, [_negated(torch.ones(1))], 1.0), 'gradient 0 is clipped in place')


def test_the_norm_takes_as_many_rows_as_the_scan():
    import ctypes as C
    from rgp_amd import _lib
    r = _lib.RmsNorm()
    r.dtype, r.C, r.eps = _lib.DT_BF16, 40, 1e-6
    for rows, ok in ((1 << 24, True), (1 << 40, True), ((1 << 40) + 1, False)):
        r.rows = rows
        assert (_lib.load().rgp_rms_norm_workspace(C.byref(r), 1) > 0) == ok


@pytest.mark.parametrize('lengths', [[2.7, 1], [3, 0.5], torch.tensor([1.5, 2.5]), [float('nan')], [float('inf'), 2], [[1, 2]], ['3'], [None], torch.tensor(3), 3])
def test_lengths_that_are_not_whole_numbers_are_refused(lengths):
    from rgp_amd import seq_ops
    _refused(lambda: seq_ops.SeqTable(H, lengths), 'whole numbers')


def test_whole_numbers_of_any_type_are_lengths():
    import numpy as np
    from rgp_amd import seq_ops
    for lengths in ([3, 0, 2], (3, 0, 2), torch.tensor([3, 0, 2]), np.array([3, 0, 2]), [3.0, np.int64(0), torch.tensor(2)], iter([3, 0, 2])):
        assert seq_ops.SeqTable(H, lengths).off.tolist() == [0, 3, 3, 5]
