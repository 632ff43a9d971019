"""The 64-bit forms of seq_reference.py over all sequences of a batch at once, on any device: for sizes at which one sequence after the other
would take minutes.  The same values and magnitudes (tests/test_seq_batched_cpu.py compares them)."""
import torch

import seq_reference as ref


def scan(u, delta, A, B, Cm, D=None, z=None, bias=None, init=None, gy=None, reverse=False):
    """u, delta, z, gy (T, n, Dn); B, Cm (T, n, G, N); init (n, Dn, N): {name: (value, magnitude)} on the CPU, sums over the sequences in gA, gD
    and gbias."""
    d = lambda t: None if t is None else t.detach().double()                                # noqa: E731
    u, delta, A, B, Cm, D, z, bias, init, gy = map(d, (u, delta, A, B, Cm, D, z, bias, init, gy))
    T, n, Dn = u.shape
    N, G = A.shape[1], B.shape[2]
    order = range(T - 1, -1, -1) if reverse else range(T)
    full = lambda v: v.repeat_interleave(Dn // G, dim=1)                                    # noqa: E731  (n, G, N) -> (n, Dn, N)
    group = lambda v: v.reshape(n, G, Dn // G, N).sum(2)                                    # noqa: E731
    Dk = D if D is not None else torch.zeros(Dn, dtype=u.dtype, device=u.device)
    s = init if init is not None else torch.zeros(n, Dn, N, dtype=u.dtype, device=u.device)
    m = s.abs()
    states, mags, dts, sgs, ps, pms = {}, {}, {}, {}, {}, {}
    y, ym = torch.empty_like(u), torch.empty_like(u)
    f = lambda t: (ref.silu(z[t]), ref.dsilu(z[t])) if z is not None else (torch.ones_like(u[t]), torch.zeros_like(u[t]))     # noqa: E731

    def decay(t):
        x = dts[t].unsqueeze(-1) * A
        a = torch.exp(x)
        return a, a * (1 + x.abs())
    for t in order:
        raw = delta[t] + bias if bias is not None else delta[t]
        dts[t], sgs[t] = ref.softplus(raw), torch.sigmoid(raw)
        a, grow = decay(t)
        inc = (dts[t] * u[t]).unsqueeze(-1) * full(B[t])
        if gy is not None:
            states[t], mags[t] = s, m                                                       # before the step
        s, m = a * s + inc, grow * m + inc.abs()
        Cw = full(Cm[t])
        ps[t], pms[t] = (s * Cw).sum(-1) + Dk * u[t], (m * Cw.abs()).sum(-1) + (Dk * u[t]).abs()
        y[t], ym[t] = ps[t] * f(t)[0], pms[t] * f(t)[0].abs()
    out = {'y': (y, ym), 'last': (s, m)}
    if gy is not None:
        names = ('gu', 'gdelta', 'gz')
        g = {k: (torch.empty_like(u), torch.empty_like(u)) for k in names}
        g.update({k: (torch.empty_like(B), torch.empty_like(B)) for k in ('gB', 'gC')})
        g.update({k: [torch.zeros_like(v), torch.zeros_like(v)] for k, v in (('gA', A), ('gD', Dk), ('gbias', Dk))})
        carry, cm = torch.zeros_like(s), torch.zeros_like(s)

        def put(k, t, value, magnitude):
            g[k][0][t], g[k][1][t] = value, magnitude

        def add(k, value, magnitude):
            g[k][0] += value.sum(0)
            g[k][1] += magnitude.sum(0)
        for t in list(order)[::-1]:
            a, grow = decay(t)
            Bw, Cw, dt, sg, (ft, fd) = full(B[t]), full(Cm[t]), dts[t], sgs[t], f(t)
            gp, gpm = gy[t] * ft, gy[t].abs() * ft.abs()
            inc = (dt * u[t]).unsqueeze(-1)
            after, am = a * states[t] + inc * Bw, grow * mags[t] + (inc * Bw).abs()
            lam, lm = Cw * gp.unsqueeze(-1) + carry, Cw.abs() * gpm.unsqueeze(-1) + cm
            carry, cm = a * lam, grow * lm
            q, qm = carry * states[t], cm * mags[t]
            lb, lbm = (lam * Bw).sum(-1), (lm * Bw.abs()).sum(-1)
            graw, grm = (u[t] * lb + (q * A).sum(-1)) * sg, (u[t].abs() * lbm + (qm * A.abs()).sum(-1)) * sg
            put('gu', t, dt * lb + Dk * gp, dt * lbm + Dk.abs() * gpm)
            put('gdelta', t, graw, grm)
            put('gz', t, gy[t] * ps[t] * fd, gy[t].abs() * pms[t] * (fd.abs() + 0.5))
            put('gB', t, group(lam * inc), group(lm * inc.abs()))
            put('gC', t, group(gp.unsqueeze(-1) * after), group(gpm.unsqueeze(-1) * am))
            add('gA', q * dt.unsqueeze(-1), qm * dt.unsqueeze(-1))
            add('gD', gp * u[t], gpm * u[t].abs())
            add('gbias', graw, grm)
            del states[t], mags[t]
        out.update(g)
    return {k: (v[0].cpu(), v[1].cpu()) for k, v in out.items()}


def chunks(n, size):
    return [slice(i, min(i + size, n)) for i in range(0, n, size)]


def scan_in_chunks(size, u, delta, A, B, Cm, D=None, z=None, bias=None, init=None, gy=None, reverse=False):
    """``scan`` over ``size`` sequences at a time."""
    outs = []
    for c in chunks(u.shape[1], size):
        cut = lambda t: None if t is None else t[:, c]                                      # noqa: E731
        outs.append(scan(u[:, c], delta[:, c], A, B[:, c], Cm[:, c], D, cut(z), bias, None if init is None else init[c], cut(gy), reverse))
    join = lambda k, j: (sum(o[k][j] for o in outs) if k in ('gA', 'gD', 'gbias') else torch.cat([o[k][j] for o in outs], 0 if k == 'last' else 1))    # noqa: E731
    return {k: (join(k, 0), join(k, 1)) for k in outs[0]}
