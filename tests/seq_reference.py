"""Plain 64-bit forms of the sequence operators on the CPU, one sequence at a time and one step after the other, with a magnitude beside each
value: the same sums over absolute values.  An output's tolerance is then counted, not chosen:

    half a step of its storage type  *  |value|        (its one rounding: finfo.eps / 2 relative to the value)
  + ops * half a step of the arithmetic type * magnitude

where ``ops`` bounds the roundings that any product in the sum passes through: per step of the recurrence the exponential, its argument,
the product and the addition (at most 8 counting forward and backward chains), plus the additions of the sums over states, channels and
rows, plus a constant for softplus, silu and the final products."""
import numpy as np
import torch


def half(dtype):
    return torch.finfo(dtype).eps / 2


def acc_of(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def tolerance(dtype, value, magnitude, ops, acc=None):
    acc = acc or acc_of(dtype)
    tiny = {torch.float16: 2.0 ** -25}.get(dtype, 0.0)                 # half a step below the smallest normal number
    return half(dtype) * value.abs() * 1.001 + ops * half(acc) * magnitude + tiny


def check(name, got, value, magnitude, ops, acc=None):
    got64 = got.detach().double().cpu()
    assert got64.shape == value.shape, (name, got64.shape, value.shape)
    tol = tolerance(got.dtype, value, magnitude, ops, acc)
    err = (got64 - value).abs()
    bad = ~(err <= tol)
    if bool(bad.any()):
        i = int(torch.argmax(torch.where(bad, err / tol.clamp(min=1e-300), torch.zeros_like(err)).reshape(-1)))
        raise AssertionError('%s: %d of %d values off, worst at %s: got %r, want %r, tolerance %r' % (
            name, int(bad.sum()), bad.numel(), np.unravel_index(i, tuple(err.shape)), float(got64.reshape(-1)[i]), float(value.reshape(-1)[i]),
            float(tol.reshape(-1)[i])))


def silu(x):
    return x * torch.sigmoid(x)


def dsilu(x):
    s = torch.sigmoid(x)
    return s + x * s * (1 - s)


def softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def conv_one(x, w, bias, init, gv):
    """One sequence (L, D): {name: (value, magnitude)}."""
    L, D = x.shape
    W = w.shape[1]
    full = torch.cat((init if init is not None else torch.zeros(W - 1, D, dtype=x.dtype), x), 0)
    b = bias if bias is not None else torch.zeros(D, dtype=x.dtype)
    pre, mag = torch.zeros(L, D, dtype=x.dtype), torch.zeros(L, D, dtype=x.dtype)
    for t in range(L):
        pre[t], mag[t] = b, b.abs()
        for j in range(W):
            pre[t] += w[:, j] * full[t + j]
            mag[t] += (w[:, j] * full[t + j]).abs()
    # an error e of pre moves silu by at most 1.1 e
    out = {'v': (silu(pre), 1.1 * mag + silu(pre).abs()), 'last': (full[L:], full[L:].abs() * 0)}
    if gv is not None:
        gp = gv * dsilu(pre)
        gpm = gv.abs() * (dsilu(pre).abs() + 0.5 * mag + 1.0)             # |silu''| <= 1/2; the factor itself is a sum of terms up to 1
        gx, gxm = torch.zeros_like(full), torch.zeros_like(full)
        gw, gwm = torch.zeros_like(w), torch.zeros_like(w)
        for t in range(L):
            for j in range(W):
                gx[t + j] += w[:, j] * gp[t]
                gxm[t + j] += (w[:, j]).abs() * gpm[t]
                gw[:, j] += gp[t] * full[t + j]
                gwm[:, j] += gpm[t] * full[t + j].abs()
        out['gx'], out['gw'], out['gb'] = (gx[W - 1:], gxm[W - 1:]), (gw, gwm), (gp.sum(0), gpm.sum(0))
    return out


def scan_one(u, delta, A, B, Cm, D, z, bias, init, gy):
    """One sequence: u, delta, z, gy (L, Dn), B, C (L, G, N): {name: (value, magnitude)}."""
    L, Dn = u.shape
    N, G = A.shape[1], B.shape[1]
    ch = torch.arange(Dn) // (Dn // G)
    raw = delta + (bias if bias is not None else 0.0)
    dt, sg = softplus(raw), torch.sigmoid(raw)
    Bw, Cw = B[:, ch], Cm[:, ch]
    a = torch.exp(dt.unsqueeze(-1) * A)
    inc = (dt * u).unsqueeze(-1) * Bw
    s = [init if init is not None else torch.zeros(Dn, N, dtype=u.dtype)]
    m = [s[0].abs()]
    # an exponential's argument x = dt A is off by a few half steps of |x|: the factor 1 + |x| carries that into the magnitude
    grow = a * (1 + (dt.unsqueeze(-1) * A).abs())
    for t in range(L):
        s.append(a[t] * s[t] + inc[t])
        m.append(grow[t] * m[t] + inc[t].abs())
    s, m = torch.stack(s), torch.stack(m)
    Dk = D if D is not None else torch.zeros(Dn, dtype=u.dtype)
    p = (s[1:] * Cw).sum(-1) + Dk * u
    pm = (m[1:] * Cw.abs()).sum(-1) + (Dk * u).abs()
    f, fd = (silu(z), dsilu(z)) if z is not None else (torch.ones_like(u), torch.zeros_like(u))
    out = {'y': (p * f, pm * f.abs()), 'last': (s[L], m[L])}
    if gy is None:
        return out
    gp, gpm = gy * f, gy.abs() * f.abs()
    lam, lm = torch.zeros(L + 1, Dn, N, dtype=u.dtype), torch.zeros(L + 1, Dn, N, dtype=u.dtype)
    carry, cm = torch.zeros(Dn, N, dtype=u.dtype), torch.zeros(Dn, N, dtype=u.dtype)
    for t in range(L - 1, -1, -1):
        lam[t] = Cw[t] * gp[t].unsqueeze(-1) + carry
        lm[t] = Cw[t].abs() * gpm[t].unsqueeze(-1) + cm
        carry, cm = a[t] * lam[t], grow[t] * lm[t]
    lam, lm = lam[:L], lm[:L]
    lb, lbm = (lam * Bw).sum(-1), (lm * Bw.abs()).sum(-1)
    q, qm = lam * a * s[:L], lm * grow * m[:L]
    la, lam_ = (q * A).sum(-1), (qm * A.abs()).sum(-1)
    graw, grm = (u * lb + la) * sg, (u.abs() * lbm + lam_) * sg
    out['gu'] = (dt * lb + Dk * gp, dt * lbm + Dk.abs() * gpm)
    out['gdelta'] = (graw, grm)
    out['gz'] = (gy * p * fd, gy.abs() * pm * (fd.abs() + 0.5))
    group = lambda v: v.reshape(L, G, Dn // G, N).sum(2)                   # noqa: E731
    out['gB'] = (group(lam * (dt * u).unsqueeze(-1)), group(lm * (dt * u).abs().unsqueeze(-1)))
    out['gC'] = (group(gp.unsqueeze(-1) * s[1:]), group(gpm.unsqueeze(-1) * m[1:]))
    out['gA'] = ((q * dt.unsqueeze(-1)).sum(0), (qm * dt.unsqueeze(-1)).sum(0))
    out['gD'] = ((gp * u).sum(0), (gpm * u.abs()).sum(0))
    out['gbias'] = (graw.sum(0), grm.sum(0))
    return out


def by_sequence(one, acts, states, lengths, packed, reverse, shared, sums, kw):
    """Runs ``one`` over the sequences of a (T, batch, ..) or packed batch.  acts / states: {argument: tensor or None}; shared: outputs laid
    out like the activations, sums: outputs added over the sequences; everything else is stacked per sequence."""
    rows, stacked, total = [], {}, {}
    off = np.concatenate(([0], np.cumsum(lengths)))
    for i, L in enumerate(lengths):
        pick = (lambda v: v[off[i]:off[i + 1]]) if packed else (lambda v: v[:, i])
        turn = (lambda v: v.flip(0)) if reverse else (lambda v: v)
        a = {k: None if v is None else turn(pick(v)) for k, v in acts.items()}
        s = {k: None if v is None else v[i] for k, v in states.items()}
        o = one(**a, **s, **kw)
        rows.append({k: tuple(turn(x) for x in o[k]) for k in shared if k in o})
        for k, v in o.items():
            if k in sums:
                total[k] = v if k not in total else tuple(p + q for p, q in zip(total[k], v))
            elif k not in shared:
                stacked.setdefault(k, []).append(v)
    out = {k: tuple(torch.stack([v[j] for v in vs]) for j in (0, 1)) for k, vs in stacked.items()}
    out.update(total)
    for k in rows[0]:
        out[k] = tuple(torch.cat([r[k][j] for r in rows], 0) if packed else torch.stack([r[k][j] for r in rows], 1) for j in (0, 1))
    return out


def rms(x, r, w, eps, gy, gh):
    h = x if r is None else x + r
    C = h.shape[-1]
    rs = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    hm = x.abs() if r is None else x.abs() + r.abs()
    out = {'hid': (h, hm), 'y': (h * rs * w, hm * rs * w.abs() * 2)}
    if gy is not None:
        dot, dotm = (gy * w * h).mean(-1, keepdim=True), (gy * w * hm).abs().mean(-1, keepdim=True)
        g, gm = rs * (gy * w - h * rs * rs * dot), rs * ((gy * w).abs() + hm * rs * rs * dotm * 3)
        if gh is not None:
            g, gm = g + gh, gm + gh.abs()
        out['gx'] = (g, gm)
        out['gw'] = ((gy * h * rs).reshape(-1, C).sum(0), (gy.abs() * hm * rs).reshape(-1, C).sum(0) * 2)
    return out
