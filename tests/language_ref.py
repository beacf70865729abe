"""64-bit references of a language model's two ends: embedding rows and their gradient, the counter-based dropout mask, the cross
entropy of a product; and the tolerances that fp32 kernels owe them, counted in roundings."""
import numpy as np

HALF = 2.0 ** -24  # the most that one rounding to fp32 is off by, of the value


def embedding(w, tokens, scale):
    ok = (tokens >= 0) & (tokens < len(w))
    y = np.zeros(tokens.shape + (w.shape[1],))
    y[ok] = w[tokens[ok]].astype(np.float64) * scale
    return y


def embedding_grad(tokens, g, V, scale, padding=-1):
    """(gradient, sum of the terms' sizes)"""
    t, g = tokens.reshape(-1), g.reshape(-1, g.shape[-1]).astype(np.float64) * scale
    ok = (t >= 0) & (t < V) & (t != padding)
    gw, size = np.zeros((V, g.shape[1])), np.zeros((V, g.shape[1]))
    np.add.at(gw, t[ok], g[ok])
    np.add.at(size, t[ok], np.abs(g[ok]))
    return gw, size


def embedding_grad_tol(size, old=0.0):
    """Blocks of at most 64 terms are summed one after the other in fp32 (63 roundings of partial sums no larger than the terms'
    sizes together), the blocks in fp64; one rounding of that, one with the scale and one where it is added to what was there."""
    return HALF * (66 * size + np.abs(old)) + 1e-44


def philox(counter, key):
    """Philox 4x32-10 of four counter words and two key words (arrays or numbers) as four uint64 arrays below 2^32."""
    low = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def kept(n, p, seed, offset, first=0):
    """Which of n values (from value `first`, a multiple of 4, on) stay."""
    block = np.arange(first // 4, first // 4 + (n + 3) // 4, dtype=np.uint64)
    zero = np.zeros_like(block)
    low = np.uint64(0xFFFFFFFF)
    words = philox((block & low, block >> np.uint64(32), zero + np.uint64(offset % 2 ** 32), zero + np.uint64(offset >> 32)),
                   (seed % 2 ** 32, seed >> 32))
    return np.stack(words, -1).reshape(-1)[:n] >= np.uint64(round(p * 2.0 ** 32))


def dropout(x, p, seed, offset, residual=None):
    """The kernel's own fp32 roundings: one of the product, or one of the product and the sum together."""
    keep = kept(x.size, p, seed, offset).reshape(x.shape)
    scale = np.float32(1.0 / (1.0 - p)) if p < 1 else np.float32(0)
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.where(keep, x * scale, np.float32(0))
        if residual is not None:
            wide = residual.astype(np.float64) + x.astype(np.float64) * np.float64(scale)
            y = np.where(keep, wide.astype(np.float32), residual)
    return y


def vocab_loss(x, w, bias, labels, ignore=-100, sum=False, gout=1.0):
    """{loss, rows, gx, gw, gb} in 64 bits, and the products z with the probabilities p of the rows that count."""
    N, V = len(x), len(w)
    on = (labels != ignore) & (labels >= 0) & (labels < V)
    x64, w64 = np.where(on[:, None], x, 0).astype(np.float64), w.astype(np.float64)
    z = x64 @ w64.T + (0 if bias is None else bias.astype(np.float64))
    at = np.where(on, labels, 0)
    rows_at = np.arange(N)
    m = z.max(-1, keepdims=True) if N else np.zeros((0, 1))
    e = np.exp(z - m)
    total = e.sum(-1, keepdims=True)
    rows = np.where(on, np.log(total[:, 0]) + m[:, 0] - z[rows_at, at], 0.0)
    p = e / total
    G = p.copy()
    others = e.copy()
    others[rows_at, at] = 0
    G[rows_at, at] = -others.sum(-1) / total[:, 0]
    count = on.sum()
    c = gout if sum else gout / count if count else 0.0
    G = G * (on * c)[:, None]
    loss = rows.sum() if sum else rows.sum() / count if count else np.nan
    return {"loss": loss, "rows": rows, "gx": G @ w64, "gw": G.T @ x64, "gb": G.sum(0), "z": z, "G": G, "on": on}


def vocab_loss_tol(x, w, ref):
    """Bounds of each output's root mean square error, by the roundings.

    A product of K terms: each operand is held to 2^-22 (two pieces of 11 bits) and the parts left out are at most 2^-22 more, so a
    term is off by at most 3 2^-22 of it, independently: sqrt(3) 2^-22 of the sum's size in the root mean square counts as 7 HALF.  K
    additions in turn, each off by at most HALF of a partial sum that grows as sqrt(k): at most HALF sqrt(K / 2) of the terms' size
    together.  So: rel(K) = HALF (7 + sqrt(K)) times the root of the sum of the terms' squares.  The exponential is off by 8 HALF and the
    difference z - lse by HALF of the largest |z| in both."""
    on, G, N, V, D = ref["on"], ref["G"], len(x), len(w), x.shape[1]
    if not on.any():
        return {k: 0.0 for k in ("gx", "gw", "gb", "rows", "loss")}
    rel = lambda K: HALF * (7 + np.sqrt(K))
    x64, w64 = np.where(on[:, None], x, 0).astype(np.float64), w.astype(np.float64)
    size = np.sqrt((x64 ** 2) @ (w64 ** 2).T)  # of each z's terms
    finite = np.isfinite(ref["z"])
    dz = rel(D) * size + 3 * HALF * np.where(finite, np.abs(np.where(finite, ref["z"], 0)), 0)
    # p moves by p (dz + the row's own dlse); the row's by the mean of dz under p at most
    worst = dz.max(-1, keepdims=True)
    dG = np.abs(G) * (2 * worst + 10 * HALF)
    rms = lambda a: float(np.sqrt(np.mean(np.square(a))))
    per_row = (2 * worst + 4 * HALF)[:, 0] * on + 4 * HALF * np.abs(ref["rows"])
    return {
        # the errors of a row's G are shared by its entries through lse: they add up as G W itself does, at worst as sums of sizes
        "gx": rms(dG @ np.abs(w64)) + rel(V) * rms(np.sqrt((G ** 2) @ (w64 ** 2))),
        "gw": rms(dG.T @ np.abs(x64)) + rel(N) * rms(np.sqrt((G ** 2).T @ (x64 ** 2))),
        "gb": rms(dG.sum(0)) + 2 * HALF * rms(np.abs(G).sum(0)),
        "rows": rms(per_row), "loss": float(np.abs(per_row).max()) + 2 * HALF * abs(ref["loss"]) if np.isfinite(ref["loss"]) else 0.0,
    }
