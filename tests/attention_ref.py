"""Rotary positions, the per-head norm and attention in 64 bits, with numpy, and how far 32-bit results may be from them.

The bounds count roundings, each at most half a step: U = 2^-24 relative in fp32.
"""
import numpy as np

U = 2.0 ** -24


def rope64(x, pos, dims, base, interleaved, sign=1.0):
    """x [B, L, H, D]; pos [L, A] or [B, L, A].  Returns (y, |first| + |second| of each column's pair)."""
    x = np.asarray(x, np.float64)
    y, mag, at = x.copy(), np.abs(x), 0
    pos = np.asarray(pos, np.float64)
    pos = pos if pos.ndim == 3 else pos[None]
    for a, d in enumerate(dims):
        ang = pos[:, :, a, None] * float(np.float32(base)) ** (-2.0 * np.arange(d // 2) / d)
        c, s = np.cos(ang)[:, :, None], sign * np.sin(ang)[:, :, None]
        i1 = at + (2 * np.arange(d // 2) if interleaved else np.arange(d // 2))
        i2 = i1 + 1 if interleaved else i1 + d // 2
        y[..., i1], y[..., i2] = x[..., i1] * c - x[..., i2] * s, x[..., i2] * c + x[..., i1] * s
        mag[..., i1] = mag[..., i2] = np.abs(x[..., i1]) + np.abs(x[..., i2])
        at += d
    return y, mag


# cosine and sine: the angle's rounding (0.8 U), at most 4 units in the last place of the function (4 U); the product's and the
# fused multiply-add's own roundings: 2 U.  All relative to the pair's magnitudes.
ROPE_TOL = 7 * U


def qk_norm_rope64(x, q_heads, wq, wk, eps, pos, dims, base, interleaved):
    """(y, bound)"""
    x = np.asarray(x, np.float64)
    h = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * head_weights(x, q_heads, wq, wk)
    y, mag = rope64(h, pos, dims, base, interleaved)
    # the sum of squares: at most 16 sequential and 6 tree additions; its division, eps, root and inverse; two products
    return y, (ROPE_TOL + (22 / 2 + 1 + 1 + 1 + 1 + 2) * U) * mag + 1e-44


def head_weights(x, q_heads, wq, wk):
    H, D = x.shape[2:]
    one = np.ones(D)
    return np.stack([np.asarray(w if w is not None else one, np.float64)
                     for w in [wq] * q_heads + [wk] * (H - q_heads)] or [one])[:H]


def qk_norm_rope_bwd64(x, q_heads, wq, wk, eps, pos, dims, base, interleaved, gy):
    """{gx, gwq, gwk}: (value, bound)"""
    x = np.asarray(x, np.float64)
    w = head_weights(x, q_heads, wq, wk)
    g, mag = rope64(gy, pos, dims, base, interleaved, -1.0)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps)))
    n, h, hm = x * r, g * w, mag * np.abs(w)
    m = (h * n).mean(-1, keepdims=True)
    gx = r * (h - n * m)
    a = (hm * np.abs(n)).mean(-1, keepdims=True)  # what the mean adds up, in magnitude
    # h: 8 U of hm; n: 16 U; the mean: its terms' 24 U, 22 additions, a division and two products; then r and two roundings
    out = {"gx": (gx, U * r * ((8 + 17) * hm + np.abs(n) * a * (24 + 25 + 16 + 17)) + 1e-44)}
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    for name, sl in (("gwq", slice(0, q_heads)), ("gwk", slice(q_heads, None))):
        t, tm = (g * n)[:, :, sl], (mag * np.abs(n))[:, :, sl]
        # the terms' 7 + 16 + 1 U and at most one addition for each row
        out[name] = (t.sum((0, 1, 2)), U * (24 + 2 + rows) * tm.sum((0, 1, 2)) + 1e-44)
    return out


def attention64(q, k, v, lens, scale, go=None):
    """Forward, and backward where go is given: {o, lse, gq, gk, gv}: (value, bound).

    eps(n) = 2^-20 + n U bounds a product of n terms relative to the sum of their magnitudes: the operands' own roundings where
    they are held in pieces (at most 2^-22 each, and 2^-22 for the product that is left out) and n additions.  Pieces also have a
    smallest step: probabilities 2^-35 of the row's largest, values 2^-40 of their tile's largest, their products' gradients 2^-36
    (2^-25 against a largest of 2^11 at least)."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    G = Hq // Hkv
    sc = float(np.float32(scale))
    names = ("o", "gq", "gk", "gv") if go is not None else ("o",)
    like = {"o": q, "gq": q, "gk": k, "gv": v}
    out = {i: (np.zeros_like(like[i]), np.full(like[i].shape, 1e-37)) for i in names}
    out["lse"] = (np.full((B, Hq, Lq), -np.inf), np.zeros((B, Hq, Lq)))

    def eps(n):
        return 2.0 ** -20 + n * U

    def add(name, at, value, bound):
        out[name][0][at] += value
        out[name][1][at] += bound

    for b in range(B):
        n = Lk if lens is None else int(np.clip(lens[b], 0, Lk))
        if n == 0:
            continue
        for h in range(Hq):
            u = h // G
            Q, K, V = q[b, :, h], k[b, :n, u], v[b, :n, u]
            s = sc * (Q @ K.T)
            es = (eps(D) + 4 * U) * abs(sc) * (np.abs(Q) @ np.abs(K).T) + 1e-37
            m = s.max(1, keepdims=True)
            e = np.exp(s - m)
            l = e.sum(1, keepdims=True)
            p = e / l
            # exp's own error: 4 U, and the argument's rounding relative to the largest magnitudes in the row
            ep = es + es.max(1, keepdims=True) + U * (8 + 2 * np.abs(s) + 2 * np.abs(m))
            o = p @ V
            eo = (p * (2 * ep.max(1, keepdims=True) + eps(n) + n * U)) @ np.abs(V) + 2.0 ** -35 * np.abs(V).max() * n
            add("o", (b, slice(None), h), o, eo)
            lse = (m + np.log(l))[:, 0]
            out["lse"][0][b, h] = lse
            out["lse"][1][b, h] = ep.max(1) + (n + 8) * U * (1 + np.abs(lse))
            if go is None:
                continue
            g = np.asarray(go[b, :, h], np.float64)
            dp, dpm = g @ V.T, np.abs(g) @ np.abs(V).T
            delta, dm = (g * o).sum(1, keepdims=True), (np.abs(g) * np.abs(o)).sum(1, keepdims=True)
            ep = ep + out["lse"][1][b, h][:, None]  # p is taken again from the row's log-sum-exp
            ds = p * (dp - delta) * sc
            eds = abs(sc) * p * (eps(D) * (dpm + dm) + (np.abs(g) * eo).sum(1, keepdims=True)
                                 + np.abs(dp - delta) * (2 * ep + 4 * U)) + 2.0 ** -36 * np.abs(ds).max()
            add("gq", (b, slice(None), h), ds @ K, eds @ np.abs(K) + eps(n) * np.abs(ds) @ np.abs(K))
            add("gk", (b, slice(0, n), u), ds.T @ Q, eds.T @ np.abs(Q) + eps(Lq * G) * np.abs(ds).T @ np.abs(Q))
            add("gv", (b, slice(0, n), u), p.T @ g,
                (p * (2 * ep + eps(Lq * G))).T @ np.abs(g) + 2.0 ** -38 * np.abs(g).max())
    return out


def within(got, want, bound, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    inf = np.isinf(want)
    assert (got[inf] == want[inf]).all(), f"{what}: infinities differ"
    assert np.isfinite(got[~inf]).all(), f"{what}: {int((~np.isfinite(got[~inf])).sum())} values are not finite"
    err, bound = np.abs(got[~inf] - want[~inf]), np.broadcast_to(bound, want.shape)[~inf]
    if not (err <= bound).all():
        i = int(np.argmax(err - bound))
        raise AssertionError(f"{what}: {int((err > bound).sum())} of {err.size} off; worst: got {got[~inf][i]!r}, want "
                             f"{want[~inf][i]!r}, bound {bound[i]:.3g}")
