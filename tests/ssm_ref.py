"""The state-space operators and their gradients written out in 64 bits, step by step, from the formulas - and the same with
every term taken by its magnitude, which is what rounding errors are measured against: a computed sum is off by at most
(number of roundings on the way) x (half a step) x (sum of the terms' magnitudes)."""
import torch


def f64(v):
    return {k: (x.detach().cpu().double() if torch.is_tensor(x) and x.is_floating_point() else x.cpu() if torch.is_tensor(x) else x)
            for k, x in v.items()}


def close(got, ref, mag, roundings, name=""):
    """|got - ref| <= roundings 2^-24 mag + half a step of got's type: fp32 arithmetic, then one rounding to the type."""
    half = torch.finfo(got.dtype).eps / 2
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    mag = mag.abs()                              # copies (a carried state) stand in the magnitudes with their sign
    tol = roundings * 2.0 ** -24 * mag + half * (ref.abs() + roundings * 2.0 ** -24 * mag) + 1e-37
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of its tolerance" % (
        name, int(bad.sum()), bad.numel(), float(((got - ref).abs() / tol)[bad].max()))


def scan_roundings(v, grads, softplus=True):
    """Roundings on the way to an output of the scan, counted from above. The step size is off by (14 + |dt + bias|) half
    steps of itself (the sum, exp, log1p), a decay by that times its exponent and 4 of its own, per step of a chain that the
    forward walks once and a gradient twice; sums over states, channels, rows and steps come on top."""
    T, B, D = v["u"].shape
    ok = torch.ones(T, B, 1, dtype=torch.bool) if v.get("lengths") is None else (torch.arange(T)[:, None] < v["lengths"][None])[..., None]
    pre = torch.where(ok, v["dt"], 0.0) + (v["dt_bias"] if v.get("dt_bias") is not None else 0.0)
    s = torch.nn.functional.softplus(pre) if softplus else pre
    pmax = float(pre.abs().max())
    xmax = float((s[..., None] * v["A"]).abs().max())
    step = 4 + (1 + xmax) * (14 + pmax)
    N = v["A"].shape[1]
    return T * step + N + 16 if not grads else 2 * T * step + N + D + T * B + 64


def scan(v, softplus=True, mag=False):
    """v: u, dt, A, Bm, Cm and optionally D, z, dt_bias, h0, reset, lengths, dy, dhT -> dict of outputs and gradients.
    mag: the sums of the terms' magnitudes instead."""
    m = (lambda x: x.abs()) if mag else (lambda x: x)
    T, B, Dc = v["u"].shape
    A = v["A"]
    N = A.shape[1]
    zero = torch.zeros(Dc, dtype=torch.float64)
    Dp, bias = v.get("D"), v.get("dt_bias")
    Dp = zero if Dp is None else Dp
    bias = zero if bias is None else bias
    end = v["lengths"].clamp(0, T) if v.get("lengths") is not None else torch.full((B,), T)
    h = m(v["h0"]) if v.get("h0") is not None else torch.zeros(B, Dc, N, dtype=torch.float64)
    live = torch.arange(T)[:, None] < end[None]
    lv = lambda x: torch.where(live[..., None], x, 0.0)                       # noqa: E731
    u, Bm, Cm, dtv = (lv(v[k]) for k in ("u", "Bm", "Cm", "dt"))
    pre = dtv + bias
    if softplus:
        s, sg = pre.clamp(min=0) + torch.log1p(torch.exp(-pre.abs())), torch.sigmoid(pre)
    else:
        s, sg = pre, torch.ones_like(pre)
    s, sg = lv(s), lv(sg)
    if v.get("z") is not None:
        z = lv(v["z"])
        gate, dgate = z * torch.sigmoid(z), torch.sigmoid(z) * (1 + m(z) * (1 - torch.sigmoid(z)))
    else:
        gate, dgate = torch.ones_like(u), torch.zeros_like(u)
    keep = torch.ones(T, B) if v.get("reset") is None else (v["reset"] == 0).double()
    a = torch.exp(s[..., None] * A)
    hs, olds, q = [], [], []
    for t in range(T):
        old = h * keep[t][:, None, None]
        new = a[t] * old + m((s[t] * u[t])[..., None] * Bm[t][:, None])
        old = torch.where(live[t][:, None, None], old, 0.0)
        h = torch.where(live[t][:, None, None], new, h)
        hs.append(h)
        olds.append(old)
        q.append(m(h * Cm[t][:, None]).sum(-1) + m(Dp * u[t]))
    q = torch.stack(q)
    out = {"y": lv(m(q * gate)), "hT": h}
    if v.get("dy") is None:
        return out
    dy = lv(v["dy"])
    ds = dy * gate
    dh = m(v["dhT"]) if v.get("dhT") is not None else torch.zeros_like(h)
    r = {k: [None] * T for k in ("du", "ddt", "dB", "dC")}
    dA = torch.zeros_like(A)
    for t in range(T - 1, -1, -1):
        g = dh + m(ds[t][..., None] * Cm[t][:, None])
        gB = m(g * Bm[t][:, None]).sum(-1)
        w = g * a[t] * olds[t]
        r["du"][t] = m(Dp * ds[t]) + m(s[t]) * gB
        r["ddt"][t] = (m(w * A).sum(-1) + m(u[t]) * gB) * sg[t]
        r["dB"][t] = m(g * (s[t] * u[t])[..., None]).sum(1)
        r["dC"][t] = m(hs[t] * ds[t][..., None]).sum(1)
        dA = dA + m(w * s[t][..., None]).sum(0)
        dh = torch.where(live[t][:, None, None], g * a[t] * keep[t][:, None, None], dh)
    out.update({k: torch.stack(x) for k, x in r.items()})
    out.update(dz=m(dy * q * dgate), dA=dA, dD=m(ds * u).sum((0, 1)), ddt_bias=out["ddt"].sum((0, 1)), dh0=dh)
    return out


def conv(v, silu=True, mag=False):
    """v: x, w and optionally bias, state_in, reset, lengths, dy, dstate_out -> outputs and gradients."""
    m = (lambda x: x.abs()) if mag else (lambda x: x)
    T, B, D = v["x"].shape
    W = v["w"].shape[1]
    end = v["lengths"].clamp(0, T) if v.get("lengths") is not None else torch.full((B,), T)
    st = v["state_in"] if v.get("state_in") is not None else torch.zeros(B, W - 1, D, dtype=torch.float64)
    rows = torch.cat([st.transpose(0, 1), v["x"]])                              # row i is the input of time i - (W - 1)
    y, state = torch.zeros(T, B, D, dtype=torch.float64), st.clone()
    out = {"y": y, "state_out": state, "dx": torch.zeros_like(y), "dw": torch.zeros_like(v["w"]), "db": torch.zeros(D, dtype=torch.float64),
           "dstate_in": torch.zeros_like(st)}
    drow = torch.zeros(T + W - 1, B, D, dtype=torch.float64)
    for b in range(B):
        n, first = int(end[b]), 0                                               # first usable row
        for t in range(n):
            if v.get("reset") is not None and v["reset"][t, b] != 0:
                first = t + W - 1
            use = [k for k in range(W) if t + k >= first]
            exact = sum(v["w"][:, k] * rows[t + k, b] for k in use) + (v["bias"] if v.get("bias") is not None else 0.0)
            pre = sum(m(v["w"][:, k] * rows[t + k, b]) for k in use) + (m(v["bias"]) if v.get("bias") is not None else 0.0)
            sg = torch.sigmoid(exact)
            slope = sg * (1 + exact * (1 - sg))
            if mag:                              # an error of pre enters silu by its slope and silu' by the slope's slope
                slope = sg * (1 + exact.abs()) + pre * sg * (2 + exact.abs())
            y[t, b] = (pre * sg * (1 + exact.abs()) if mag else pre * sg) if silu else pre
            if v.get("dy") is not None:
                g = v["dy"][t, b] * (slope if silu else 1.0)
                for k in use:
                    drow[t + k, b] += m(g * v["w"][:, k])
                    out["dw"][:, k] += m(g * rows[t + k, b])
                out["db"] += m(g)
        for k in range(W - 1):
            i = n + k
            state[b, k] = rows[i, b] if i >= first else 0.0
            if i >= first and v.get("dstate_out") is not None:
                drow[i, b] += m(v["dstate_out"][b, k])
    out["dx"], out["dstate_in"] = drow[W - 1:], drow[:W - 1].transpose(0, 1)
    return out


def norm(v, eps=1e-5, mag=False):
    """v: x [rows, D], w and optionally b, dy."""
    m = (lambda x: x.abs()) if mag else (lambda x: x)
    x, w = v["x"], v["w"]
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    n = (x - mean) * rstd
    if mag:                                     # x - mean is computed from both: their magnitudes count
        n = (x.abs() + x.abs().mean(-1, keepdim=True)) * rstd
    out = {"y": m(n * w) + (m(v["b"]) if v.get("b") is not None else 0.0), "mean": m(x).mean(-1), "rstd": rstd[:, 0] * (1 + (n.amax(-1) if mag else 0.0))}
    if v.get("dy") is not None:
        dy = m(v["dy"])
        dn = dy * m(w)
        a, c = dn.mean(-1, keepdim=True), n * (dn * n).mean(-1, keepdim=True)
        out.update(dx=(dn + a + c if mag else dn - a - c) * rstd, dw=(dy * n).sum(0), db=dy.sum(0))
    return out


def scan_bounds(v, softplus=True, cut=False):
    """How far each output of the scan may be off before it is rounded to its type, counted along the recurrences, so that what
    has decayed no longer counts: beside the magnitude M of a state or of its gradient runs its error E, and both fade by the
    same decay. In half steps e = 2^-24: a step size is off by 14 + |pre| of itself (sum, exp, log1p), a decay by 4 (exp, its
    product) and by its exponent times the 17 + |pre| of that (A log2(e), its product), a gate by 8 + 3 |z|, a product by 1 and a
    sum of n terms by n + 6. ``cut``: the time may be cut into joined segments, whose summed step sizes take up to T / 4 + 3 more."""
    e = 2.0 ** -24
    T, B, Dc = v["u"].shape
    A, N = v["A"], v["A"].shape[1]
    zero = torch.zeros(Dc, dtype=torch.float64)
    Dp, bias = (zero if v.get(k) is None else v[k] for k in ("D", "dt_bias"))
    end = v["lengths"].clamp(0, T) if v.get("lengths") is not None else torch.full((B,), T)
    live = torch.arange(T)[:, None] < end[None]
    lv = lambda x: torch.where(live[..., None], x, 0.0)                       # noqa: E731
    u, Bm, Cm, dtv = (lv(v[k]) for k in ("u", "Bm", "Cm", "dt"))
    u, Bm, Cm = u.abs(), Bm.abs(), Cm.abs()
    pre = dtv + bias
    if softplus:
        s, sg = pre.clamp(min=0) + torch.log1p(torch.exp(-pre.abs())), torch.sigmoid(pre)
    else:
        s, sg = pre, torch.ones_like(pre)
    s, sg = lv(s), lv(sg)
    ap = pre.abs().clamp(max=200.0)                           # beyond, a softplus is 0 or the sum itself
    rs = (14 + ap) * e
    x = s[..., None] * A
    a = torch.exp(x)
    ra = (4 + x.abs() * (17 + ap + (T / 4 + 3 if cut else 0))[..., None]) * e
    s = s.abs()
    keep = torch.ones(T, B) if v.get("reset") is None else (v["reset"] == 0).double()
    if v.get("z") is not None:
        z = lv(v["z"])
        sz = torch.sigmoid(z)
        gate, dgate = (z * sz).abs(), sz * (1 + z.abs() * (1 - sz))
        rg = (8 + 3 * z.abs()) * e
        e_dgate = (rg + 6 * e) * dgate + z.abs() * sz * sz * rg
    else:
        gate, dgate, rg, e_dgate = torch.ones_like(u), torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(u)
    h = v["h0"].abs() if v.get("h0") is not None else torch.zeros(B, Dc, N, dtype=torch.float64)
    eh = torch.zeros_like(h)
    hs, ehs, olds, eolds, qs, eqs = [], [], [], [], [], []
    for t in range(T):
        ok, k = live[t][:, None, None], keep[t][:, None, None]
        old, eold = h * k, eh * k
        add = (s[t] * u[t])[..., None] * Bm[t][:, None]
        new = a[t] * old + add
        enew = a[t] * (eold + ra[t] * old) + (rs[t] + 3 * e)[..., None] * add + e * new
        h, eh = torch.where(ok, new, h), torch.where(ok, enew, eh)
        hs.append(h), ehs.append(eh)
        olds.append(torch.where(ok, old, 0.0)), eolds.append(torch.where(ok, eold, 0.0))
        q = (h * Cm[t][:, None]).sum(-1) + (Dp * u[t]).abs()
        qs.append(q), eqs.append((eh * Cm[t][:, None]).sum(-1) + (N + 6) * e * q)
    q, eq = torch.stack(qs), torch.stack(eqs)
    out = {"y": lv(gate * eq + (rg + 3 * e) * gate * q), "hT": eh}
    if v.get("dy") is None:
        return {k: 1.01 * x for k, x in out.items()}          # products of two errors
    dy = lv(v["dy"]).abs()
    ds, rds = dy * gate, rg + 2 * e
    G = v["dhT"].abs() if v.get("dhT") is not None else torch.zeros_like(h)
    eG = torch.zeros_like(G)
    r = {k: [None] * T for k in ("du", "ddt", "dB", "dC")}
    dA, mA = torch.zeros_like(A), torch.zeros_like(A)
    mdt = []
    for t in range(T - 1, -1, -1):
        ok, k = live[t][:, None, None], keep[t][:, None, None]
        cds = ds[t][..., None] * Cm[t][:, None]
        g = G + cds
        eg = eG + rds[t][..., None] * cds + e * g
        gB = (g * Bm[t][:, None]).sum(-1)
        egB = (eg * Bm[t][:, None]).sum(-1) + (N + 6) * e * gB
        r["du"][t] = (Dp * ds[t]).abs() * (rds[t] + 2 * e) + s[t] * (egB + (rs[t] + 3 * e) * gB)
        w = g * a[t] * olds[t]
        ew = a[t] * (eg * olds[t] + g * eolds[t] + (ra[t] + 2 * e) * g * olds[t])
        wA = (w * A.abs()).sum(-1)
        ewA = (ew * A.abs()).sum(-1) + (N + 6) * e * wA
        m = wA + u[t] * gB
        r["ddt"][t] = sg[t] * (ewA + u[t] * egB + (11 + ap[t]) * e * m)
        mdt.append(sg[t] * m)
        su = s[t] * u[t]
        r["dB"][t] = (eg * su[..., None] + g * ((rs[t] + 2 * e) * su)[..., None] + (Dc + 8) * e * g * su[..., None]).sum(1)
        r["dC"][t] = (ehs[t] * ds[t][..., None] + hs[t] * ((rds[t] + (Dc + 9) * e) * ds[t])[..., None]).sum(1)
        dA = dA + (ew * s[t][..., None] + w * ((rs[t] + 2 * e) * s[t])[..., None]).sum(0)
        mA = mA + (w * s[t][..., None]).sum(0)
        G, eG = torch.where(ok, g * a[t] * k, G), torch.where(ok, a[t] * (eg + (ra[t] + e) * g) * k, eG)
    out.update({k: torch.stack(x) for k, x in r.items()})
    n = (T + B + 80) * e                                      # sums over the steps of a row, then over rows and segments
    out.update(dz=dy * (eq * dgate + q * e_dgate + 3 * e * q * dgate), dA=dA + n * mA,
               dD=((rds + 2 * e + n) * ds * u).sum((0, 1)), ddt_bias=out["ddt"].sum((0, 1)) + n * torch.stack(mdt).sum((0, 1)), dh0=eG)
    return {k: 1.01 * x for k, x in out.items()}


def within(got, ref, bound, name=""):
    """|got - ref| <= bound + half a step of got's type."""
    half = torch.finfo(got.dtype).eps / 2
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    tol = bound + half * (ref.abs() + bound) + 1e-37
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of its tolerance" % (
        name, int(bad.sum()), bad.numel(), float(((got - ref).abs() / tol)[bad].max()))
