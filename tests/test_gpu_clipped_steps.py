"""What an SVI step makes of its own gradients, to the rounding: the stored (clipped) gradients of a step go into Adam's formula, written out in
torch, and the parameters behind the step have to be its result.  No second gradient is computed, so nothing is left to the order of sums."""
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_ssm_encoder import _gp, _mlp, build


def _adam(x, p, g, m, v, positive, lr, t):
    import torch
    g = torch.where(positive, g * -torch.expm1(-p), g)
    m.mul_(0.9).add_(0.1 * g)
    v.mul_(0.999).add_(0.001 * g * g)
    x.add_(lr * (m / (1 - 0.9 ** t)) / (torch.sqrt(v / (1 - 0.999 ** t)) + 1e-8))
    p.copy_(torch.where(positive, torch.nn.functional.softplus(x, threshold=36.0), x))


def _close(a, b, scale):
    assert float((a - b).abs().max()) <= scale * max(1.0, float(b.abs().max()))


@pytest.mark.parametrize('seqs', [slice(0, 4), [2, 0], [1, 1, 3], None])
@pytest.mark.parametrize('clips', [(0.5, 0.5), (1e12, 0.25), (None, 0.5, None)])
def test_parameters_behind_a_step_are_adams_of_the_stored_gradients(seqs, clips):
    """Also of plain (pipelined) steps between clipped ones.  32 roundings of values up to the parameters' size a step, and of the update's quotient,
    which is at most 10."""
    import torch
    a = _gp()
    a.svi_step(seqs, lr=1e-2, max_grad_norm=1.0)                     # moments that are not zero
    ids = [0, 1, 2, 3] if seqs is None or isinstance(seqs, slice) else seqs
    for c in clips:
        a.handle.sync()
        x, p, m, v = (t.clone() for t in (a.opt_array, a.param_array, a._adam['m'], a._adam['v']))
        t_glob, t_loc = a._adam['t_glob'], a._adam['t_loc'].copy()
        a.svi_step(seqs, lr=1e-2, max_grad_norm=c)
        a.handle.sync()
        g, pos, G = a.grad_array, a.positive.bool(), a.n_global
        if c is not None:
            mine = torch.cat([g[:G]] + [g[b + int(a.seq_loc_off[s]):b + int(a.seq_loc_off[s + 1])] for s in sorted(set(ids)) for b in (a.loc0, a.loc0 + a.n_local)])
            want = min(float(a.last_grad_norm), c * float(a.last_grad_norm) / (float(a.last_grad_norm) + 1e-6))
            assert abs(float(mine.norm()) - want) <= 1e-12 * want     # the stored gradients have the norm that was asked for
        _adam(x[:G], p[:G], g[:G], m[:G], v[:G], pos[:G], 1e-2, t_glob + 1)
        for s in ids:
            t_loc[s] += 1
            for b in (a.loc0, a.loc0 + a.n_local):
                k = slice(b + int(a.seq_loc_off[s]), b + int(a.seq_loc_off[s + 1]))
                _adam(x[k], p[k], g[k], m[k], v[k], pos[k], 1e-2, int(t_loc[s]))
        for have, want in ((a.opt_array, x), (a.param_array, p), (a._adam['m'], m), (a._adam['v'], v)):
            _close(have, want, 32 * 2.0 ** -53 * 10)


@pytest.mark.parametrize('make', [_mlp, lambda: build(n_seq=4, n_total=4)[0]], ids=['mlp', 'ssm'])
def test_encoder_models_update_by_the_clipped_gradients(make):
    """GP globals by the formula, the encoder's weights by torch's Adam on a copy of them with the stored gradients."""
    import torch
    a = make()
    for c in (0.5, 1e12):
        a.handle.sync()
        weights = [q for q in a.encoder.parameters()]
        old = [q.detach().clone() for q in weights]
        fresh = a._adam is None
        if not fresh:
            x, p, m, v = (t.clone() for t in (a.opt_array, a.param_array, a._adam['m'], a._adam['v']))
            t = a._adam['t_glob']
        a.svi_step(slice(0, 4), lr=1e-2, max_grad_norm=c)
        a.handle.sync()
        have = [q.grad for q in weights if q.grad is not None]
        total = float(torch.sqrt(sum((q * q).sum() for q in [a.grad_array[:a.n_global]] + have)))
        norm = float(a.last_grad_norm)
        want = min(norm, c * norm / (norm + 1e-6))
        assert abs(total - want) <= 1e-12 * want
        if not fresh:
            G, pos = a.n_global, a.positive.bool()
            _adam(x[:G], p[:G], a.grad_array[:G], m[:G], v[:G], pos[:G], 1e-2, t + 1)
            for got, exp in ((a.opt_array, x), (a.param_array, p), (a._adam['m'], m), (a._adam['v'], v)):
                _close(got[:G], exp[:G], 32 * 2.0 ** -53 * 10)
        else:                                                          # the first update of a weight is lr g / (|g| + eps)
            for q, o in zip(weights, old):
                if q.grad is not None:
                    _close(q.detach(), o + 1e-2 * q.grad / (q.grad.abs() + 1e-8), 32 * 2.0 ** -53 * 10)
