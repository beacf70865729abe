"""Bounds of the vocabulary loss's outputs entry by entry, for tests that look at single rows and columns of gx and gW, and the scheme of
operands in two fp16 pieces in numpy, so that the bounds can be seen to tell a good choice of powers of two from a bad one.

Where an operand a is a = 2^e (hi + 2^-11 lo) with its row's largest finite value in [2^14, 2^15) after the scaling, hi is off by half a step
of fp16 and lo holds what is left in another 11 bits: 22 bits together, down to values whose lo is below fp16's smallest normal, 2^-14.
From there on the error is absolute, half of fp16's smallest step, 2^-25."""
import numpy as np

from tests.language_ref import HALF

# The absolute errors, of the row's largest value, which is at least 2^14 in those units, counted twice for the other operand's hi that is
# scaled on the way.  z: lo is brought to 2^5, so 2^-30 of 2^14; gx and gW: 2^-36 of 2^14.
Z_FLOOR = 2.0 ** -43
SUM_FLOOR = 2.0 ** -49
# G's own: 2^-25 and as much again for its hi that is scaled, of the largest term's power (2^14; one less where the logarithm that gives it
# is rounded up), and a factor of 2 between a row's largest and its power
G_FLOOR = 2.0 ** -36


def largest(a):
    return np.abs(a).max(-1)


def bounds(x, w, ref, gout=1.0):
    """{gx [N, D], gw [V, D], rows [N]}: what each entry's error may be in the root mean square over any row or column.  The terms are
    those of language_ref.vocab_loss_tol, taken entry by entry, and the floors above."""
    on, G, N, V, D = ref["on"], ref["G"], len(x), len(w), x.shape[1]
    rel = lambda K: HALF * (7 + np.sqrt(K))
    x64, w64 = np.where(on[:, None], x, 0).astype(np.float64), w.astype(np.float64)
    size = np.sqrt((x64 ** 2) @ (w64 ** 2).T)
    z = np.where(np.isfinite(ref["z"]), np.abs(ref["z"]), 0)
    lx, lw = largest(x64), largest(w64)
    l2 = lambda a: np.sqrt((a ** 2).sum(-1))
    dz = rel(D) * size + 3 * HALF * z + Z_FLOOR * (np.outer(lx, l2(w64)) + np.outer(l2(x64), lw))
    # a word without probability moves nothing
    worst = np.where(G != 0, dz, 0).max(-1, keepdims=True)
    dG = np.abs(G) * (2 * worst + 10 * HALF)
    aG, safe = np.abs(G), lambda a: np.where(a > 0, a, 1)

    def product(dA, A, B, lB, K):
        """A B summed over K: A's error, the products' roundings, B's floor and A's"""
        term = (A * lB).max(-1, keepdims=True)
        return (dA @ np.abs(B) + rel(K) * np.sqrt((A ** 2) @ (B ** 2)) + SUM_FLOOR * np.sqrt(((A * lB) ** 2).sum(-1, keepdims=True))
                + G_FLOOR * term * l2((B / safe(lB)[:, None]).T)
                + 2 * K * 2.0 ** -150)  # where terms are below a float's normal range each product and each addition rounds to steps of 2^-149

    rows = (2 * worst + 4 * HALF)[:, 0] * on + 4 * HALF * np.abs(ref["rows"])
    return {"gx": product(dG, aG, w64, lw, V), "gw": product(dG.T, aG.T, x64, lx, N), "rows": rows}


def rms(a, axis):
    return np.sqrt(np.mean(np.square(np.asarray(a, np.float64)), axis))


def beyond(got, ref, tol, old=None):
    """The outputs' rows and columns (gx, gW) and entries (rows) that are off by more than their bounds, as texts"""
    wrong = []
    for k in ("gx", "gw"):
        if k not in got:
            continue
        want = ref[k] + (0 if old is None else old[k])
        # one rounding of the result, one more where it is added to what was there; the smallest float's step
        allowed = tol[k] + 2 * HALF * np.abs(want) + 2.0 ** -148
        err = got[k].astype(np.float64) - want
        for axis, what in ((1, "row"), (0, "column")):
            e, a = rms(err, axis), rms(allowed, axis)
            bad = np.flatnonzero(~(e <= a))
            wrong += [f"{k} {what} {i}: {e[i]:.3g} off, {a[i]:.3g} allowed, {rms(want, axis)[i]:.3g} large" for i in bad[:3]]
    if "rows" in got:
        err = np.abs(got["rows"].astype(np.float64) - ref["rows"])
        bad = np.flatnonzero(~(err <= tol["rows"] + HALF * np.abs(ref["rows"])))
        wrong += [f"loss of row {i}: {err[i]:.3g} off, {tol['rows'][i]:.3g} allowed" for i in bad[:3]]
    return wrong


# ---- inputs ------------------------------------------------------------------------------------------------------------
def columns_of_unlike_sizes(N, D, V, seed, what):
    """Columns whose sizes lie far apart: in w alone (gx), in x alone (gW), or in both the other way round (z, and all that follows)."""
    rng = np.random.default_rng(seed)
    x, w = rng.standard_normal((N, D)), rng.standard_normal((V, D)) * 2 / np.sqrt(D)
    # the columns between are there twice each, so that their sizes, not one entry, are what a row's power comes from
    size = np.zeros(D)
    size[1::7], size[3::7], size[5::7] = -20, -24, -28
    if what == "w":
        w *= np.exp2(size)
    elif what == "x":
        x *= np.exp2(size)
    else:
        x, w = x * np.exp2(-size / 1.25), w * np.exp2(size / 1.25)  # up to 2^22.4
    return x.astype(np.float32), w.astype(np.float32), None, rng.integers(0, V, N).astype(np.int32)


def rows_of_unlike_sizes(N, D, V, seed, what):
    """Rows 2^40 times the others' that a result does not count, since their words have next to no probability there: every result is
    the sum of small rows."""
    rng = np.random.default_rng(seed)
    x, w = rng.standard_normal((N, D)), rng.standard_normal((V, D)) * 2 / np.sqrt(D)
    labels = rng.integers(0, V // 2, N) * 2 + 1
    if what == "w":  # even words are large and out of the way by their bias: e^-60 of 1 is 2^-86, the others' terms are 2^-50
        w[1::2] *= 2.0 ** -40
        b = np.where(np.arange(V) % 2 == 0, -60.0, 0.0).astype(np.float32)
        x /= np.sqrt(D)  # so that no product of theirs makes up for it
        return x.astype(np.float32), w.astype(np.float32), b, labels.astype(np.int32)
    # even rows of x are large, and column 0 takes the even words out for them: gW of an even word is the sum of the small rows
    x[1::2] *= 2.0 ** -40
    x[:, 1:] /= np.sqrt(D)
    x[0::2, 0] = 1.0
    w[:, 0] = np.where(np.arange(V) % 2 == 0, -80.0, 0.0)
    return x.astype(np.float32), w.astype(np.float32), None, labels.astype(np.int32)


# ---- the scheme ------------------------------------------------------------------------------------------------------------
def power_of(most):
    """the exponent that puts `most` into [2^14, 2^15)"""
    return np.floor(np.log2(np.where(most > 0, most, 1.0))) - 14


def pieces(a, e, low):
    """(hi, lo 2^-low) of a / 2^e, with lo held as lo 2^low in fp16; e one exponent for each row"""
    v = a * np.exp2(-np.asarray(e, np.float64))[..., None]
    hi = v.astype(np.float16).astype(np.float64)
    return hi, ((v - hi) * 2.0 ** low).astype(np.float16).astype(np.float64) * 2.0 ** -low


def product_of_pieces(a, b):
    """A B^T of two operands' pieces, summed in 64 bits"""
    return a[0] @ b[0].T + a[0] @ b[1].T + a[1] @ b[0].T


def loss_in_pieces(x, w, bias, ref, low=11, by_row=True, by_term=True):
    """{gx, gw, rows} with operands in two pieces, everything else in 64 bits.  by_row: a power of two for each row of x and of w,
    else one for all; by_term: G's powers by its results' largest terms, else by its largest entries."""
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    powers = lambda a: power_of(largest(a)) if by_row else np.full(len(a), power_of(np.abs(a).max()))
    ex, ew = powers(x64), powers(w64)
    px, pw = pieces(x64, ex, low), pieces(w64, ew, low)
    z = product_of_pieces(px, pw) * np.exp2(ex[:, None] + ew)
    if bias is not None:
        z = z + bias.astype(np.float64)
    m = z.max(-1, keepdims=True)
    lse = np.log(np.exp(z - m).sum(-1, keepdims=True)) + m
    at = np.flatnonzero(ref["on"])
    label = ref["labels"]
    p = np.exp(z - lse)
    p[at, label[at]] = 0
    p[at, label[at]] = -p.sum(-1)[at]
    rows = (lse[:, 0] - z[np.arange(len(z)), np.where(ref["on"], label, 0)]) * ref["on"]
    p *= (ref["on"] / max(1, ref["on"].sum()))[:, None]

    def gradient(g, e_sum, b):
        scaled = g * np.exp2(e_sum)
        e = power_of(largest(scaled)) if by_term else power_of(largest(g)) + e_sum.max()
        turned = tuple(t.T for t in b)
        return product_of_pieces(pieces(scaled, e, 0), turned) * np.exp2(e)[:, None]

    return {"gx": gradient(p, ew, pw), "gw": gradient(p.T, ex, px), "rows": rows}
