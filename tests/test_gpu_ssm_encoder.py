"""The operators together, as the models run them: the state-space encoder of DeepAutoreg_rnn (whole sequences, training, one observation at
a time, types) and gradient clipping inside the SVI steps."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_model import make_data


def build(n_seq=3, T=12, n_total=None, **kw):
    from rgp_amd.model import DeepAutoreg_rnn
    U, Y = make_data(n_seq, T, seed=4)
    m = DeepAutoreg_rnn([0, 3, 3], Y, U=U, U_win=2, nDims=[3, 2, 3], num_inducing=4, rnn_type='ssm', rnn_hidden_dims=[6],
                        inference_method='svi', mb_inf_tot_data_size=n_total, seed=1, **kw)
    rng = np.random.default_rng(2)
    for L in m.layers:
        m.set_param(L, 'inv_l', 0.3 + rng.random(L.Q))
        m.set_param(L, 'noise', 0.2 + 0.1 * rng.random())
        m.set_param(L, 'qU_W', rng.standard_normal((L.M, L.M)) * 0.2)
        m.set_param(L, 'qU_a', 0.3)
    return m, U, Y


def plain_block(blk, x):
    """The block's formulas step by step in elementary torch operations."""
    import torch
    xs = x.flip(0) if blk.reverse else x
    rms = lambda v, w: v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w           # noqa: E731
    h = xs @ blk.inp.weight.t() + blk.inp.bias
    c, z = (rms(h, blk.norm_in) @ blk.uz.weight.t()).split(blk.E, dim=-1)
    pad = torch.cat((torch.zeros_like(c[:1]).expand(blk.W - 1, -1, -1), c), 0)
    pre = blk.conv_bias + sum(pad[j:j + c.shape[0]] * blk.conv_weight[:, j] for j in range(blk.W))
    u = pre * torch.sigmoid(pre)
    r, B, Cm = (u @ blk.maps.weight.t()).split((blk.R, blk.N, blk.N), dim=-1)
    dt = torch.nn.functional.softplus(r @ blk.dt.t() + blk.dt_bias)
    A, s, ys = -torch.exp(blk.A_log), 0.0, []
    for t in range(u.shape[0]):
        s = torch.exp(dt[t].unsqueeze(-1) * A) * s + (dt[t] * u[t]).unsqueeze(-1) * B[t].unsqueeze(-2)
        ys.append((s * Cm[t].unsqueeze(-2)).sum(-1) + blk.skip * u[t])
    y = torch.stack(ys) * z * torch.sigmoid(z)
    n = rms(y @ blk.out.weight.t() + h, blk.norm_out)
    return n.flip(0) if blk.reverse else n


@pytest.mark.parametrize('T,B,H,bi', [(1, 2, 5, False), (37, 3, 20, True), (400, 4, 12, False)])
def test_block_matches_its_formulas(T, B, H, bi):
    """Means, variances and the gradients of every parameter and of the input against the formulas in fp64 (400 x 4 rows: the split over
    time and the split-K weight gradients run).  Both sides are fp64: 8 T + 100 roundings of values up to the output's own size."""
    import torch
    from rgp_amd.capi import Handle
    from rgp_amd.rnn_encoder import MeanVarSSM
    Hd = Handle()
    torch.manual_seed(3)
    lay = MeanVarSSM(4, 3, H, bi).double().to(Hd.device)
    lay.handle = Hd
    x = torch.randn(T, B, 4, dtype=torch.float64, device=Hd.device, requires_grad=True)
    wm, wv = (torch.randn(T, B, 3, dtype=torch.float64, device=Hd.device) for _ in range(2))
    par = list(lay.parameters())
    mean, var = lay(x)
    got = torch.autograd.grad((mean * wm).sum() + (var * wv).sum(), [x] + par)
    n = torch.cat([plain_block(b, x) for b in lay.blocks], dim=2)
    m2, v2 = lay.linear_mean(n), lay.soft_plus(lay.linear_var(n))
    want = torch.autograd.grad((m2 * wm).sum() + (v2 * wv).sum(), [x] + par)
    tol = (8 * T + 100) * 1.2e-16 * 100
    for a, b in zip((mean, var) + got, (m2, v2) + want):
        assert float((a - b).abs().max()) <= tol * max(1.0, float(b.abs().max())) * max(1.0, (T * B) ** 0.5), (a.shape, float((a - b).abs().max()))


@pytest.mark.parametrize('bi', [False, True])
def test_encoder_weight_gradients_of_the_bound(bi):
    """dELBO/d(encoder weight) against central differences of the ELBO, one element of every parameter."""
    import torch
    m, U, Y = build(rnn_bidirectional=bi)
    m.evaluate()
    m.handle.sync()
    rng, eps = np.random.default_rng(7), 1e-6
    grads = [p.grad.clone() for p in m.encoder.parameters()]
    for p, g in zip(m.encoder.parameters(), grads):
        j = int(rng.integers(p.numel()))
        old = float(p.view(-1)[j].item())
        es = []
        for v in (old + eps, old - eps, old):
            with torch.no_grad():
                p.view(-1)[j] = v
            es.append(float(m.evaluate().item()))
        num = (es[0] - es[1]) / (2 * eps)
        assert abs(num - float(g.view(-1)[j])) <= 2e-5 * max(1.0, abs(num)), (tuple(p.shape), j, num, float(g.view(-1)[j]))


def test_steps_and_minibatches_and_checkpoint(tmp_path):
    """SVI steps run and move every parameter, minibatch sums are additive, save / load keeps the encoder."""
    m, U, Y = build(n_seq=4, n_total=4)
    e = float(m.evaluate().item()); g = m.grad_array[:m.n_global].cpu().numpy().copy(); ge = m.encoder_grad_vector().cpu().numpy().copy()
    e1 = float(m.evaluate(slice(0, 2)).item()); g1 = m.grad_array[:m.n_global].cpu().numpy().copy(); ge1 = m.encoder_grad_vector().cpu().numpy().copy()
    e2 = float(m.evaluate([2, 3]).item()); g2 = m.grad_array[:m.n_global].cpu().numpy().copy(); ge2 = m.encoder_grad_vector().cpu().numpy().copy()
    m.handle.sync()
    assert abs(e1 + e2 - e) <= 1e-12 * abs(e)
    np.testing.assert_allclose(g1 + g2, g, rtol=1e-9, atol=1e-10)
    np.testing.assert_allclose(ge1 + ge2, ge, rtol=1e-8, atol=1e-10)
    before = [p.detach().clone() for p in m.encoder.parameters()]
    for _ in range(3):
        m.svi_step(slice(0, 4), lr=1e-3)
    assert all(not bool((a == b).all()) for a, b in zip(before, m.encoder.parameters()))
    e0 = float(m.evaluate().item()); m.handle.sync()
    m.save(str(tmp_path / 'ck'))
    m2, _, _ = build(n_seq=4, n_total=4)
    m2.load(str(tmp_path / 'ck'))
    assert float(m2.evaluate().item()) == e0


def test_online_encoding_is_the_whole_sequences():
    """Observations one at a time from the empty state, and from the state behind a history, give the rows of the whole-sequence encoding."""
    import torch
    m, U, Y = build(n_seq=3, T=15)
    x = m.enc_input
    means, variances = m.encoder(x)
    st = m.encoder.initial_state(3)
    for t in range(15):
        ms, vs = m.encode_online(x[t], st)
        for a, b in zip(list(ms) + list(vs), means + variances):
            assert float((a - b[t]).detach().abs().max()) <= 1e-12
    _, _, st = m.encoder(x[:9], return_state=True)
    tail = m.encoder(x[9:12], state=st)                                      # a chunk of new rows
    for a, b in zip(tail[0] + tail[1], means + variances):
        assert float((a - b[9:12]).detach().abs().max()) <= 1e-12
    st = m.online_state([0, 2])
    new = torch.cat((x[:, [0, 2]], x[:1, [0, 2]] * 0.5), 0)
    want = m.encoder(new)
    ms, vs = m.encode_online((x[0, [0, 2]] * 0.5).cpu().numpy(), st)
    for a, b in zip(list(ms) + list(vs), want[0] + want[1]):
        assert float((a - b[-1]).detach().abs().max()) <= 1e-12


@pytest.mark.parametrize('name,rel', [('float32', 1e-4), ('bfloat16', 0.15), ('float16', 0.03)])
def test_compute_types(name, rel):
    """The same weights in narrower activations: q(X) moves by the type's roundings (about thirty products deep: 30 half steps, with a factor
    for cancellations), parameters and q(X) stay fp64, and steps with gradients in every parameter run."""
    import torch
    a, _, _ = build(T=40)
    b, _, _ = build(T=40, rnn_compute_dtype=getattr(torch, name))
    ma, va = a.encoder(a.enc_input)
    mb, vb = b.encoder(b.enc_input)
    for p, q in zip(ma + va, mb + vb):
        assert q.dtype == torch.float64 and float((p - q).norm()) <= rel * float(p.norm())
    b.svi_step(slice(0, 3), lr=1e-3, max_grad_norm=1.0)
    assert all(p.dtype == torch.float64 and bool(torch.isfinite(p.grad).all()) for p in b.encoder.parameters())
    st = b.online_state()
    b.encode_online(b.enc_input[0], st)


def test_refusals():
    import torch
    from rgp_amd.rnn_encoder import MeanVarSSM, SeqEncoder
    with pytest.raises(ValueError, match='rnn_compute_dtype'):
        SeqEncoder([3], [2], 4, 'gru', False, torch.float32)
    with pytest.raises(ValueError, match='rnn_compute_dtype'):
        MeanVarSSM(3, 2, 4, False, torch.int8)
    with pytest.raises(ValueError, match='Unknown rnn type'):
        SeqEncoder([3], [2], 4, 'other')
    with pytest.raises(ValueError, match='go on from a state'):
        SeqEncoder([3], [2], 4, 'gru').initial_state(2)
    with pytest.raises(RuntimeError, match='handle'):
        SeqEncoder([3], [2], 4, 'ssm')(torch.zeros(3, 1, 3, dtype=torch.float64))
    m, _, _ = build(rnn_bidirectional=True)
    with pytest.raises(ValueError, match='bidirectional'):
        m.online_state()


# ---------------------------------------------------------------------------------------------------------------------- clipping in the steps
def _gp(**kw):
    from rgp_amd.model import DeepAutoreg
    U, Y = make_data(4, 14, seed=0)
    return DeepAutoreg([0, 3, 3], Y, U=U, U_win=2, nDims=[3, 2, 3], X_variance=0.05, num_inducing=4, init='Y', inference_method='svi',
                       mb_inf_tot_data_size=4, seed=3, **kw)


def _mlp():
    from rgp_amd.model import DeepAutoreg_mlp
    U, Y = make_data(4, 14, seed=0)
    return DeepAutoreg_mlp([0, 3, 3], Y, U=U, U_win=2, nDims=[3, 2, 3], num_inducing=4, MLP_dims=[3, 2], inference_method='svi', mb_inf_tot_data_size=4, seed=3)


def _same_step(a, b, lr, updates=1, n=None):
    """One step of two models from the same parameters: gradients to the order of their sums (kernels with atomic additions differ there from run
    to run, 1e-9 of the largest), parameters to what Adam makes of that.  Its update is lr m / (sqrt(v) + eps), eps = 1e-8, with both moments
    corrected for the step number.  One gradient enters m with a weight of at most 1 and sqrt(v) with a slope of at most 1, and |m| <= 8 sqrt(v)
    (Cauchy-Schwarz over the two weightings, 0.9 and 0.999), so a change dg of the gradient moves the update by at most (1 + 8) lr dg / eps
    wherever sqrt(v) is; plus 32 roundings of the parameter."""
    a.handle.sync(); b.handle.sync()
    dg, dp = (a.grad_array[:n] - b.grad_array[:n]).abs(), (a.param_array[:n] - b.param_array[:n]).abs()
    assert float(dg.max()) <= 1e-9 * float(b.grad_array[:n].abs().max())
    assert bool((dp <= updates * 9 * lr / 1e-8 * dg + 32 * 2.0 ** -53 * b.param_array[:n].abs().max()).all())


@pytest.mark.parametrize('seqs', [slice(0, 4), [2, 0], [1, 1, 3], None])
def test_clipped_step_is_an_adam_step_on_the_scaled_gradient(seqs):
    """The norm is that of the stored gradients, the gradients are scaled by it, and with a threshold far above the norm a step is the plain
    step."""
    import torch
    a, b = _gp(), _gp()
    b.pipeline = False
    a.svi_step(seqs, lr=1e-2, max_grad_norm=1e12)
    b.svi_step(seqs, lr=1e-2)
    _same_step(a, b, 1e-2, updates=2)                               # a sequence that is named twice is updated twice
    a, b = _gp(), _gp()
    b.evaluate(seqs)
    b.handle.sync()
    ids = range(4) if seqs is None or isinstance(seqs, slice) else sorted(set(seqs))
    idx = b._index_set(ids)
    g = b.grad_array[idx]
    a.svi_step(seqs, max_grad_norm=0.5)
    a.handle.sync()
    norm = float(g.norm())
    assert abs(float(a.last_grad_norm) - norm) <= 1e-9 * norm
    want = g * min(1.0, 0.5 / (norm + 1e-6))
    assert float((a.grad_array[idx] - want).abs().max()) <= 1e-9 * float(want.abs().max())
    assert float((a.param_array - b.param_array).abs().max()) > 0


def test_clipped_steps_of_the_encoder_models_and_mixed_with_pipelined_ones():
    import torch
    for make in (_mlp, lambda: build(n_seq=4, n_total=4)[0]):
        m, r = make(), make()
        r.evaluate(slice(0, 4)); r.handle.sync()
        gs = [r.grad_array[:r.n_global]] + [p.grad for p in r.encoder.parameters() if p.grad is not None]
        norm = float(torch.sqrt(sum((g * g).sum() for g in gs)))
        m.svi_step(slice(0, 4), max_grad_norm=0.25 * norm)
        m.handle.sync()
        assert abs(float(m.last_grad_norm) - norm) <= 1e-9 * norm
        after = [m.grad_array[:m.n_global]] + [p.grad for p in m.encoder.parameters() if p.grad is not None]
        for x, y in zip(after, gs):
            assert float((x - 0.25 * y).abs().max()) <= 1e-6 * norm
    a, b = _gp(), _gp()
    b.pipeline = False
    for k, c in enumerate((None, 1e9, None, None, 1e9, None)):       # pipelined and clipped steps in turn equal plain steps
        a.svi_step(slice(0, 4), lr=1e-2, max_grad_norm=c)
        b.svi_step(slice(0, 4), lr=1e-2)
        _same_step(a, b, 1e-2)
        for x, y in ((a.param_array, b.param_array), (a.opt_array, b.opt_array), (a._adam['m'], b._adam['m']), (a._adam['v'], b._adam['v'])):
            y.copy_(x)                                              # the next step from the same place


def test_two_ranks_clip_like_one_process():
    """Two halves of the data in two models of this process, their exchange done by hand: the same norm, the same global update."""
    import torch
    from rgp_amd.model import DeepAutoreg
    U, Y = make_data(4, 14, seed=0)
    kw = dict(U_win=2, nDims=[3, 2, 3], X_variance=0.05, num_inducing=4, init='Y', inference_method='svi', mb_inf_tot_data_size=4, seed=3)
    one = DeepAutoreg([0, 3, 3], Y, U=U, **kw)
    halves = [DeepAutoreg([0, 3, 3], Y[i:i + 2], U=U[i:i + 2], **kw) for i in (0, 2)]
    for m in halves:
        m.param_array[:m.n_global].copy_(one.param_array[:one.n_global])
        m.params_changed()
    for i, m in enumerate(halves):                                  # the latents of one are the two halves' latents
        for l in (1, 2):
            for s in (0, 1):
                m.latent(l, s).copy_(one.latent(l, 2 * i + s)); m.latent(l, s, var=True).copy_(one.latent(l, 2 * i + s, var=True))
    # what each half sends: recorded in a first run that exchanges nothing, then summed
    sent = []
    for m in halves:
        mine = []
        m.evaluate(slice(0, 2), qU_ratio=0.5)
        mine.append(m.grad_array[:m.n_global + 1].clone())
        mine.append((m.grad_array[m.loc0:] ** 2).sum().view(1))
        m.handle.sync()
        sent.append(mine)
    total = [x + y for x, y in zip(*sent)]
    for m in halves:
        left = list(total)
        m.svi_step(slice(0, 2), lr=1e-2, qU_ratio=0.5, max_grad_norm=0.5, allreduce=lambda t: t.copy_(left.pop(0)))
        assert not left
    one.svi_step(slice(0, 4), lr=1e-2, max_grad_norm=0.5)
    for m in halves:
        m.handle.sync()
        assert abs(float(m.last_grad_norm) - float(one.last_grad_norm)) <= 1e-9 * float(one.last_grad_norm)
        _same_step(m, one, 1e-2, n=one.n_global)
