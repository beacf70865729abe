"""How near fp32 attention comes to 64 bits: tight enough that one operand held in 11 bits shows, and each row on its own scale.

A product's operands are held in two fp16 pieces, |x - hi - lo| <= 2^-22 |x|, and the product of the two low pieces, at most 2^-22 of
the whole, is left out; roundings of sums and of exp2's argument are fp32's.  Taken as independent, with scores of a few units:
  a score: sqrt(2) * 2^-22 / sqrt(3) for the operands and 2^-22 / 3 for what is left out, of the root of the sum of its squared
  terms (about 2.3 for rows of deviation 1.5 and a scale of D^-1/2), and sqrt(D) roundings of U / sqrt(3) of the score:
  5e-7 .. 9e-7 absolute;
  a probability: that, exp2's argument at up to 16 (2^-21 ln 2 / sqrt(3) = 2e-7) and its sum's: 1e-6 relative;
  an output or a gradient: a probability's, the other factor's 2^-22 and its sum's: 1.2e-6 of its norm, less where many keys share it.
WHOLE, of a tensor's norm, allows three times that; an operand that lost its low piece is off by 2^-11 / sqrt(12) = 1.4e-4.
ROW is for every row by itself, of the norm of the magnitudes that it adds up: p |v|, p |go|, and p (|go . v| + |go . o| + the roots of
the sums of go . v's squared terms and of go . o's, with p |v| for o) |k| or |q| -- a row's gradient may cancel far below them
(one key that takes nearly all; go . o of values that cancel), in any arithmetic.  It allows twice WHOLE: a row has no other rows to average with, and its scores go to ten units.
"""
import numpy as np

from newch_amd.hipmem import DeviceBuffer, synchronize

WHOLE = 2.0 ** -18
ROW = 2.0 ** -17


def forward_backward(q, k, v, lens, scale, go, cut=None):
    """{o, lse, gq, gk, gv} in 64 bits, and mag: the magnitudes that o and the gradients add up.  cut = (gradient or "o", operand): that product takes the operand rounded to fp16."""
    q, k, v, go = (np.asarray(t, np.float64) for t in (q, k, v, go))

    def part(name, operand, x):
        if cut != (name, operand):
            return x
        top = np.abs(x).max()
        e = np.exp2(np.floor(np.log2(top)) - 14) if top else 1.0
        return (x / e).astype(np.float16).astype(np.float64) * e

    B, Lq, Hq, _ = q.shape
    Lk, Hkv = k.shape[1:3]
    out = {"o": np.zeros_like(q), "lse": np.full((B, Hq, Lq), -np.inf), "gq": np.zeros_like(q), "gk": np.zeros_like(k),
           "gv": np.zeros_like(v)}
    mag = out["mag"] = {i: np.zeros_like(out[i]) for i in ("o", "gq", "gk", "gv")}
    for b in range(B):
        n = Lk if lens is None else int(np.clip(lens[b], 0, Lk))
        if n == 0:
            continue
        for h in range(Hq):
            u = h // (Hq // Hkv)
            Q, K, V, G = q[b, :, h], k[b, :n, u], v[b, :n, u], go[b, :, h]
            s = float(np.float32(scale)) * (part("s", "q", Q) @ part("s", "k", K).T)
            m = s.max(1, keepdims=True)
            e = np.exp(s - m)
            total = e.sum(1, keepdims=True)
            p = e / total
            out["o"][b, :, h] = o = part("o", "p", p) @ part("o", "v", V)
            out["lse"][b, h] = (m + np.log(total))[:, 0]
            dp, delta = part("dp", "go", G) @ part("dp", "v", V).T, (G * o).sum(1, keepdims=True)
            ds = p * (dp - delta) * float(np.float32(scale))
            out["gq"][b, :, h] = part("gq", "ds", ds) @ part("gq", "k", K)
            out["gk"][b, :n, u] += part("gk", "ds", ds).T @ part("gk", "q", Q)
            out["gv"][b, :n, u] += part("gv", "p", p).T @ part("gv", "go", G)
            mag["o"][b, :, h] = mo = p @ np.abs(V)
            rough = np.sqrt((G * G) @ (V * V).T) + np.sqrt((G * G * mo * mo).sum(1, keepdims=True))
            mds = p * (np.abs(dp) + np.abs(delta) + rough) * abs(float(np.float32(scale)))
            mag["gq"][b, :, h] = mds @ np.abs(K)
            mag["gk"][b, :n, u] += mds.T @ np.abs(Q)
            mag["gv"][b, :n, u] += p.T @ np.abs(G)
    return out


def check(got, want, what="", names=("o", "gq", "gk", "gv"), pick=None, skip=0, whole=True):
    """Every tensor within WHOLE and each of its rows within ROW.  pick: which tokens of each count; skip: the first columns of gq and
    gk, which do not (two_groups)."""
    for name in names:
        g, w, m = np.asarray(got[name], np.float64), want[name], want["mag"][name]
        assert g.shape == w.shape, (what, name)
        if pick is not None:
            g, w, m = g[:, pick[name]], w[:, pick[name]], m[:, pick[name]]
        if name in ("gq", "gk"):
            g, w, m = g[..., skip:], w[..., skip:], m[..., skip:]
        assert np.isfinite(g).all(), f"{what} {name}: {int((~np.isfinite(g)).sum())} values are not finite"
        if whole and w.any():
            r = np.linalg.norm(g - w) / np.linalg.norm(w)
            assert r <= WHOLE, f"{what} {name}: off by {r:.3g} of its norm, {WHOLE:.3g} allowed"
        err, top = np.linalg.norm(g - w, axis=-1), np.linalg.norm(m, axis=-1)
        over = err > ROW * top + 2.0 ** -120  # what a float can hold at all
        if over.any():
            i = np.unravel_index(int(np.argmax(err - ROW * top)), err.shape)
            raise AssertionError(f"{what} {name}: {int(over.sum())} rows of {err.size} off; row {tuple(int(x) for x in i)} off by "
                                 f"{err[i] / top[i] if top[i] else np.inf:.3g} of its magnitudes, {ROW:.3g} allowed")


def random_inputs(shape, seed, std=1.5):
    """q, k, v, go and lengths of shape (B, Lq, Lk, Hq, Hkv, D, lengths)"""
    B, Lq, Lk, Hq, Hkv, D, lens = shape
    rng = np.random.default_rng(seed)
    q, g = (rng.standard_normal((B, Lq, Hq, D)).astype(np.float32) for _ in range(2))
    k, v = (rng.standard_normal((B, Lk, Hkv, D)).astype(np.float32) for _ in range(2))
    return q * np.float32(std), k * np.float32(std), v, g, None if lens is None else np.array(lens, np.int32)


def two_groups(shape, seed, far_queries, far_keys, apart=200.0):
    """Inputs whose queries and keys fall into two groups that do not see each other: scores across are `apart` lower, so that their
    probabilities are zero in fp32.  far_queries [Lq], far_keys [Lk]: who is in the second group.  Two columns carry it, which the
    members' own scores multiply by zero; gradients in them are the groups', not the scores'."""
    q, k, v, g, _ = random_inputs(shape, seed)
    D = q.shape[-1]
    a = np.float32(np.sqrt(apart * np.sqrt(D)))
    q[..., :2] = 0
    k[..., :2] = 0
    q[:, far_queries, :, 0] = a
    q[:, ~far_queries, :, 1] = a
    k[:, far_keys, :, 1] = -a
    k[:, ~far_keys, :, 0] = -a
    return q, k, v, g


# ---- on the device ----------------------------------------------------------------------------------------------------------
def up(a):
    return None if a is None else DeviceBuffer.from_numpy(np.asarray(a))


def run(K, q, k, v, g, lens, scale, backward=True, old=None):
    """Forward, and backward, on contiguous buffers; outputs begin as NaN, or, old, gradients as that and are added to."""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    sizes, sq, sk = (B, Lq, Lk, Hq, Hkv, D), (Lq * Hq * D, Hq * D, D), (Lk * Hkv * D, Hkv * D, D)
    Q, K_, V, G, N = up(q), up(k), up(v), up(g), up(lens)
    new = lambda *shape: DeviceBuffer.from_numpy(np.full(shape, np.nan, np.float32))
    out = {"o": new(*q.shape), "lse": new(B, Hq, Lq)}
    src = (Q.ptr, sq, K_.ptr, sk, V.ptr, sk, None if N is None else N.ptr)
    n1, n2 = K.cross_attention_fwd_workspace(*sizes), K.cross_attention_bwd_workspace(*sizes)
    ws = DeviceBuffer.from_numpy(np.full(max(n1, n2, 16), 0xFF, np.uint8))
    K.cross_attention_fwd(*sizes, scale, *src, out["o"].ptr, out["lse"].ptr, ws.ptr, n1)
    if backward:
        begin = new if old is None else lambda *shape: DeviceBuffer.from_numpy(np.full(shape, old, np.float32))
        out.update(gq=begin(*q.shape), gk=begin(*k.shape), gv=begin(*v.shape))
        K.cross_attention_bwd(*sizes, scale, *src, out["o"].ptr, out["lse"].ptr, G.ptr, *(out["g" + c].ptr for c in "qkv"), ws.ptr, n2,
                              accumulate=old is not None)
    synchronize()
    like = {"o": q, "gq": q, "gk": k, "gv": v}
    return {i: t.to_numpy(np.float32, like[i].shape if i in like else (B, Hq, Lq)) for i, t in out.items()}
