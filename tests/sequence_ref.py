"""The sequence operators in 64 bits, and how far a float32 result may be from them.

Every bound is first-order rounding analysis with u = 2^-24 (half a step of float32):
each float32 operation multiplies its result by (1 + d), |d| <= u.  An exponential is
formed as 2^(d * log2 e): ex2.approx is documented to 2^-22.5, that is 2.83u relative, and
its argument is off by u |d| each for the difference d = x - m and the product, and by
0.23u |d| for the constant in float32 (1.3e-8 relative), all in units of the exponent.
"""

import numpy as np

U = 2.0 ** -24
EXP, ARG = 4 * U, 2.25 * U  # of the exponential itself, and per |d|
TINY = 2.0 ** -120  # results so small that float32 holds them as subnormals or zero


def _lanes(x, axis):
    return np.moveaxis(x, axis, 0)


def scan(gate, x, init, axis):
    """(h, its bound).  Of h[t] = sum_s gate[s+1..t] x[s], a term meets at most two roundings
    a step (of the state, and of the gates' product where the axis is cut in pieces that
    are joined) and a few where pieces join: u * (2 w + 16 m), m the magnitude scan and w
    the same scan with each term counted once per step it has passed."""
    a, v = (_lanes(np.broadcast_to(np.asarray(q, np.float64), np.broadcast_shapes(gate.shape, x.shape)), axis)
            for q in (gate, x))
    h, tol = np.zeros(v.shape), np.zeros(v.shape)
    s = np.zeros(v.shape[1:]) if init is None else np.broadcast_to(np.asarray(init, np.float64), v.shape[1:]).copy()
    m, w = np.abs(s), np.zeros_like(s)
    with np.errstate(all="ignore"):
        for t in range(v.shape[0]):
            s = a[t] * s + v[t]
            m = np.abs(a[t]) * m + np.abs(v[t])
            w = np.abs(a[t]) * w + m
            h[t], tol[t] = s, U * (2 * w + 16 * m) + TINY
    last = (s, U * (2 * w + 16 * m) + TINY)
    return (np.moveaxis(h, 0, axis), np.moveaxis(tol, 0, axis)), last


def scan_grad(gate, x, init, axis, g, glast):
    """[(value, bound)] of dgate, dx, dinit at full shape.  The reverse scan is a scan of
    c[t] = gate[t] (g[t] + c[t+1]): a product and a sum a step, so one rounding more."""
    (h, htol), _ = scan(gate, x, init, axis)
    a = _lanes(np.broadcast_to(np.asarray(gate, np.float64), h.shape), axis)
    h, htol = _lanes(h, axis), _lanes(htol, axis)
    T = h.shape[0]
    first = np.zeros(h.shape[1:]) if init is None else np.broadcast_to(np.asarray(init, np.float64), h.shape[1:])
    c = np.zeros(h.shape[1:]) if glast is None else np.asarray(glast, np.float64).copy()
    m, w = np.abs(c), np.zeros_like(c)
    gv = np.zeros(h.shape) if g is None else _lanes(np.asarray(g, np.float64), axis)
    da, dx, tda, tdx = (np.zeros(h.shape) for _ in range(4))
    for t in range(T - 1, -1, -1):
        u = gv[t] + c
        m = m + np.abs(gv[t])
        w = w + m
        ut = U * (4 * w + 16 * m) + TINY
        before, bt = (h[t - 1], htol[t - 1]) if t > 0 else (first, 0.0)
        dx[t], tdx[t] = u, ut
        da[t] = u * before
        tda[t] = ut * np.abs(before) + (np.abs(u) + ut) * bt + U * np.abs(da[t]) + TINY
        c = a[t] * u
        m, w = np.abs(a[t]) * m, np.abs(a[t]) * w
    cl = U * (4 * w + 18 * m) + TINY
    return [(np.moveaxis(da, 0, axis), np.moveaxis(tda, 0, axis)), (np.moveaxis(dx, 0, axis), np.moveaxis(tdx, 0, axis)),
            (c, cl)]


def _rows(logits, tokens):
    """Per row: p (the token's log-probability) and its bound, softmax and its relative bound."""
    x = np.asarray(logits, np.float64)
    with np.errstate(all="ignore"):
        m = x.max(-1, keepdims=True)
        d = x - m
        e = np.exp(d)
        s = e.sum(-1, keepdims=True)
        soft = e / s
        dist = np.where(soft > 0, np.abs(d), 0.0)
        V = x.shape[-1]
        # a sum of V terms in which no term passes more than V/256 + 48 additions
        rel = EXP + U * (V / 256 + 48) + ARG * (soft * dist).sum(-1, keepdims=True)
        k = np.maximum(tokens, 0)[..., None]
        p = np.take_along_axis(d, k, -1)[..., 0] - np.log(s)[..., 0]
        ptol = rel[..., 0] + U * np.abs(p)
        soft_rel = EXP + ARG * dist + rel + 8 * U
    return p, ptol, soft, soft_rel


def _logits_grad(tokens, soft, soft_rel, slope, stol):
    """slope * (onehot - softmax), zero in padded rows."""
    hot = np.zeros(soft.shape)
    np.put_along_axis(hot, np.maximum(tokens, 0)[..., None], 1.0, -1)
    live = (tokens >= 0)[..., None]
    with np.errstate(all="ignore"):
        v = slope[..., None] * (hot - soft)
        tol = (stol[..., None] + U * np.abs(slope[..., None])) * (hot + soft) + np.abs(slope)[..., None] * soft * soft_rel
        tol = tol + U * np.abs(v) + TINY
    return np.where(live, v, 0.0), np.where(live, tol, 0.0)


def logprob(logits, tokens, g=None):
    p, ptol, soft, rel = _rows(logits, tokens)
    live = tokens >= 0
    y = (np.where(live, p, 0.0), np.where(live, ptol, 0.0))
    if g is None:
        return [y]
    slope = np.broadcast_to(np.asarray(g, np.float64), tokens.shape)
    return [y, _logits_grad(tokens, soft, rel, slope, np.zeros(tokens.shape))]


def policy(logits, tokens, old, adv, ref, clip, kl, g=None):
    """The bound follows p's own: d value / d p and d slope / d p are at most |A| r + kl |1 - e|
    and |A| r + kl e."""
    p, ptol, soft, rel = _rows(logits, tokens)
    old, adv = (np.broadcast_to(np.asarray(q, np.float64), tokens.shape) for q in (old, adv))
    lo, hi = 1.0 - np.float64(np.float32(clip[0])), 1.0 + np.float64(np.float32(clip[1]))
    with np.errstate(all="ignore"):
        r = np.exp(p - old)
        plain, held = r * adv, np.clip(r, lo, hi) * adv
        value = -np.minimum(plain, held)
        slope = np.where(plain <= held, -plain, 0.0)
        vt = st = np.abs(adv) * r * ptol
        if ref is not None:
            kl = np.float64(np.float32(kl))
            k = np.broadcast_to(np.asarray(ref, np.float64), tokens.shape) - p
            e = np.exp(k)
            value = value + kl * (e - k - 1.0)
            slope = slope + kl * (1.0 - e)
            vt, st = vt + kl * np.abs(1 - e) * ptol + kl * e * ptol ** 2, st + kl * e * ptol
        vt, st = 1.01 * vt + U * np.abs(value) + TINY, 1.01 * st + U * np.abs(slope)
    live = tokens >= 0
    y = (np.where(live, value, 0.0), np.where(live, vt, 0.0))
    if g is None:
        return [y]
    g = np.broadcast_to(np.asarray(g, np.float64), tokens.shape)
    return [y, _logits_grad(tokens, soft, rel, g * slope, np.abs(g) * st)]


def preference(logits, tokens, ref, beta, smoothing, g=None):
    p, ptol, soft, rel = _rows(logits, tokens)
    live = tokens >= 0
    ref = np.broadcast_to(np.asarray(ref, np.float64), tokens.shape)
    beta, eps = np.float64(np.float32(beta)), np.float64(np.float32(smoothing))
    with np.errstate(all="ignore"):
        d = np.where(live, p - ref, 0.0)
        dt = np.where(live, ptol + U * np.abs(d), 0.0).sum((1, 2))
        S = d.sum(-1)
        z = beta * (S[:, 0] - S[:, 1])
        zt = beta * dt
        logsig = lambda v: -(np.log1p(np.exp(-np.abs(v))) + np.maximum(-v, 0))  # noqa: E731
        pos = np.where(z >= 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))
        value = -(1 - eps) * logsig(z) - (eps * logsig(-z) if eps > 0 else 0.0)
        dz = eps * pos - (1 - eps) * (1 - pos)
    y = (value, zt + U * np.abs(value) + TINY)
    if g is None:
        return [y]
    k = np.broadcast_to(np.asarray(g, np.float64), value.shape) * beta
    slope = (np.stack([k * dz, -k * dz], 1)[..., None]) * np.ones(tokens.shape)
    stol = (np.stack([np.abs(k) * zt * 0.25] * 2, 1)[..., None]) * np.ones(tokens.shape)
    return [y, _logits_grad(tokens, soft, rel, slope, stol + U * np.abs(slope))]


def assert_within(got, ref):
    """got against (value, bound): NaN where the value is NaN, equal infinities, the rest
    within the bound (0 means equal)."""
    value, tol = ref
    got, value = np.asarray(got, np.float64), np.asarray(value, np.float64)
    tol = np.broadcast_to(tol, value.shape)
    assert got.shape == value.shape, (got.shape, value.shape)
    assert np.array_equal(np.isnan(got), np.isnan(value)), "NaN pattern differs"
    inf = np.isinf(value)
    assert np.array_equal(got[inf], value[inf]), "infinities differ"
    ok = ~(inf | np.isnan(value))
    err = np.abs(got - np.where(ok, value, 0.0))[ok]
    bad = err > tol[ok]
    assert not bad.any(), (
        f"{int(bad.sum())} of {bad.size} outside their bound; worst {np.max(err[bad] / np.maximum(tol[ok][bad], 1e-300)):.3g} "
        f"times it, error {np.max(err[bad]):.3e}")
