"""Plain float64 restatements of the token-sequence operators, one step at a time (CPU).  Every function also runs on
magnitudes (``mag=True``: every term by its absolute value): the scale that rounding errors are measured on."""
import torch


def f64(t):
    return None if t is None else t.detach().double().cpu()


def embedding(idx, weight, dout, scale, pad):
    w, idx = f64(weight), idx.cpu().reshape(-1)
    out = w[idx.clamp(0, w.shape[0] - 1)] * scale
    out[(idx < 0) | (idx >= w.shape[0])] = float("nan")
    dw, mag, count = torch.zeros_like(w), torch.zeros_like(w), torch.zeros(w.shape[0])
    if dout is not None:
        g = f64(dout).reshape(idx.numel(), w.shape[1])
        for r, v in enumerate(idx.tolist()):
            if 0 <= v < w.shape[0] and v != pad:
                dw[v] += scale * g[r]
                mag[v] += abs(scale) * g[r].abs()
                count[v] += 1
    return out, dw, mag, count


def conv(x, weight, bias, silu, lengths, state, dy=None, dstate_out=None, mag=False):
    """-> y, final state, and with dy: dx, dweight, dbias, dstate.  mag: sums of |terms| of the linear parts."""
    x, w, b, st, dy, dso = (f64(v) for v in (x, weight, bias, state, dy, dstate_out))
    t, n, d = x.shape
    k = w.shape[1]
    ab = (lambda v: v.abs()) if mag else (lambda v: v)
    lens = [t] * n if lengths is None else [min(max(int(v), 0), t) for v in lengths.tolist()]
    y, fin = torch.zeros_like(x), torch.zeros(k - 1, n, d, dtype=torch.float64)
    dx, dst = torch.zeros_like(x), torch.zeros(k - 1, n, d, dtype=torch.float64)
    dw, db = torch.zeros_like(w), torch.zeros(d, dtype=torch.float64)
    for i in range(n):
        m = lens[i]
        front = torch.zeros(k - 1, d, dtype=torch.float64) if st is None else st[:, i]
        full = torch.cat([front, x[:m, i]])
        gfull = torch.zeros_like(full)
        fin[:, i] = full[full.shape[0] - (k - 1):]
        if dso is not None:
            gfull[full.shape[0] - (k - 1):] += ab(dso[:, i])
        for s in range(m):
            win = full[s:s + k]
            p = (win * w.t()).sum(0) + (0 if b is None else b)
            sg = torch.sigmoid(p)
            y[s, i] = (ab(win) * ab(w.t())).sum(0) + (0 if b is None else ab(b)) if mag else (p * sg if silu else p)
            if dy is not None:
                dp = dy[s, i] * (sg * (1 + p * (1 - sg)) if silu else 1.0)
                if mag:                                  # |slope| <= 1.1, and an error of p moves it by at most |dp|/2
                    dp = 1.1 * dy[s, i].abs() * (1 + y[s, i]) if silu else dy[s, i].abs()
                gfull[s:s + k] += ab(w.t()) * dp
                dw += (ab(win) * dp).t()
                db += dp
        dx[:m, i] = gfull[k - 1:]
        dst[:, i] = gfull[:k - 1]
    return (y, fin) if dy is None and dso is None else (y, fin, dx, dw, db, dst)


def scan(x, dt, A, B, C, D, z, bias, softplus, lengths, state, dy=None, dh=None, mag=False):
    """-> y, final state, and with dy: dict of gradients.  B, C [steps, batch, groups, n]."""
    x, dt, A, B, C, D, z, bias, state, dy, dh = (f64(v) for v in (x, dt, A, B, C, D, z, bias, state, dy, dh))
    (t, nb, d), n, g = x.shape, A.shape[1], B.shape[2]
    ab = (lambda v: v.abs()) if mag else (lambda v: v)
    of = torch.arange(d) // (d // g)
    raw = dt if bias is None else dt + bias
    e = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    lens = torch.full((nb,), t) if lengths is None else lengths.cpu().long().clamp(0, t)
    h = torch.zeros(nb, d, n, dtype=torch.float64) if state is None else ab(state).clone()
    D_ = torch.zeros(d, dtype=torch.float64) if D is None else ab(D)
    y, olds = torch.zeros_like(x), []
    zero = torch.zeros((), dtype=torch.float64)
    for i in range(t):
        live = (lens > i)[:, None]
        olds.append(h)
        new = torch.exp(e[i][..., None] * A) * h + ab(e[i] * x[i])[..., None] * ab(B[i][:, of])
        h = torch.where(live[..., None], new, h)
        o = (ab(C[i][:, of]) * h).sum(-1) + D_ * ab(x[i])
        if z is not None:
            o = o * ab(z[i] * torch.sigmoid(z[i]))
        y[i] = torch.where(live, o, zero)
    if dy is None and dh is None:
        return y, h
    dy = torch.zeros_like(x) if dy is None else dy
    out = {k: torch.zeros_like(v) for k, v in (("x", x), ("dt", x), ("z", x), ("A", A), ("B", B), ("C", B), ("D", x[0, 0] if t and nb else D_),
                                               ("bias", D_))}
    q = torch.zeros_like(h) if dh is None else ab(dh).clone()
    for i in reversed(range(t)):
        live, old = (lens > i)[:, None], olds[i]
        a, Bi, Ci = torch.exp(e[i][..., None] * A), ab(B[i][:, of]), ab(C[i][:, of])
        u = ab(e[i] * x[i])
        now = a * old + u[..., None] * Bi
        gy = torch.where(live, ab(dy[i]), zero)
        if z is not None:
            s = torch.sigmoid(z[i])
            pre = (Ci * now).sum(-1) + D_ * ab(x[i])
            out["z"][i] = torch.where(live, gy * pre * ab(s * (1 + z[i] * (1 - s))) if not mag else gy * pre * 1.1, zero)
            gy = torch.where(live, gy * ab(z[i] * s), zero)
        q = q + torch.where(live[..., None], Ci * gy[..., None], zero)
        m = torch.where(live[..., None], q, zero)
        out["C"][i].index_add_(1, of, torch.where(live[..., None], now * gy[..., None], zero))
        out["B"][i].index_add_(1, of, m * u[..., None])
        out["D"] += torch.where(live, gy * ab(x[i]), zero).sum(0)
        thr = m * a * old
        out["A"] += (thr * ab(e[i])[..., None]).sum(0)
        mb = (m * Bi).sum(-1)
        de = (thr * ab(A)).sum(-1) + mb * ab(x[i])
        if softplus:
            de = de * torch.sigmoid(raw[i])
        out["dt"][i] = torch.where(live, de, zero)
        out["bias"] += out["dt"][i].sum(0)
        out["x"][i] = torch.where(live, gy * D_ + mb * ab(e[i]), zero)
        q = torch.where(live[..., None], a * q, q)
    out["state"] = q
    return y, h, out
