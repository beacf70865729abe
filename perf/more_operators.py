"""Performance cases of a language model's two ends and the regulariser between them: rows of an embedding table looked up and
scaled, dropout whose mask is made anew from a counter wherever it is needed, and the cross entropy of a product with a vocabulary's
weights, whose logits are not kept.

The plain forms are elementary torch operations in 32 bits; the framework's operators are called through its kernel layer on the
program's own buffers.
"""
import math

import torch

DEV = "cuda"
IGNORED = -100
own = False


def listed():
    return [
        # the next tokens of 16 sequences, served: one row of the table each
        {"name": "embed_token", "op": "embedding", "train": False, "b": 16, "l": 1, "v": 32000, "d": 2048, "padded": False},
        # a training step's batch of texts: the lookup and the table's gradient
        {"name": "embed_train", "op": "embedding", "train": True, "b": 16, "l": 512, "v": 32000, "d": 1024, "padded": False},
        # texts of unlike lengths, padded, over a small table with odd sizes
        {"name": "embed_odd_train", "op": "embedding", "train": True, "b": 3, "l": 777, "v": 10007, "d": 250, "padded": True},
        # a large table and many tokens, padded
        {"name": "embed_large_train", "op": "embedding", "train": True, "b": 32, "l": 2048, "v": 128000, "d": 2048,
         "padded": True},
        # a classifier's hidden layer at batch 64, in training
        {"name": "dropout_small_train", "op": "dropout", "train": True, "rows": 64, "d": 128, "p": 0.5, "residual": False},
        # a block's output dropped and added to what it was given, in training
        {"name": "dropout_residual_train", "op": "dropout", "train": True, "rows": 8192, "d": 1024, "p": 0.1, "residual": True},
        # an odd number of values, drawn anew without a gradient (an estimate's repeated passes)
        {"name": "dropout_odd", "op": "dropout", "train": False, "rows": 2331, "d": 1001, "p": 0.25, "residual": False},
        # the wide layer of a large batch, in training
        {"name": "dropout_large_train", "op": "dropout", "train": True, "rows": 32768, "d": 8192, "p": 0.1, "residual": False},
        # a few texts' last tokens over a small vocabulary, in training
        {"name": "loss_small_train", "op": "loss", "train": True, "n": 64, "d": 512, "v": 1000, "bias": True, "ignored": 0.0},
        # texts scored: the loss of every token, no gradient
        {"name": "loss_score", "op": "loss", "train": False, "n": 2048, "d": 1024, "v": 32000, "bias": False, "ignored": 0.0},
        # a padded batch with an odd number of tokens, words and columns, in training
        {"name": "loss_odd_train", "op": "loss", "train": True, "n": 999, "d": 770, "v": 50021, "bias": True, "ignored": 0.3},
        # a training step's tokens over a large vocabulary
        {"name": "loss_large_train", "op": "loss", "train": True, "n": 8192, "d": 2048, "v": 128000, "bias": False,
         "ignored": 0.1},
    ]


def _log_int(rng, lo, hi):
    """lo .. hi, spread over the logarithm; as often as not rounded down to a multiple of 16 where it is large."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.5:
        v -= v % 16
    return max(lo, min(hi, v))


def draw(rng):
    L = _log_int
    op = rng.choice(("embedding", "dropout", "loss", "loss"))
    while True:
        if op == "embedding":
            train = rng.random() < 0.75
            c = {"op": op, "train": train, "b": L(rng, 1, 32), "l": L(rng, 1, 4096), "v": L(rng, 256, 128000),
                 "d": L(rng, 16, 4096), "padded": rng.random() < 0.5}
            if c["b"] * c["l"] <= 65536 and max(c["b"] * c["l"], c["v"]) * c["d"] <= 128000 * 2048:
                return c
        elif op == "dropout":
            c = {"op": op, "train": rng.random() < 0.75, "rows": L(rng, 1, 32768), "d": L(rng, 16, 16384),
                 "p": round(rng.uniform(0.05, 0.6), 3), "residual": rng.random() < 0.5}
            if c["rows"] * c["d"] <= 1 << 28:
                return c
        else:
            c = {"op": op, "train": rng.random() < 0.75, "n": L(rng, 1, 8192), "d": L(rng, 32, 4096), "v": L(rng, 100, 128000),
                 "bias": rng.random() < 0.5, "ignored": rng.choice((0.0, 0.1, 0.5)) if rng.random() < 0.7 else 0.0}
            if c["n"] * c["d"] * c["v"] <= 8192 * 2048 * 128000:
                return c


# ---- inputs: plain torch, from the seed alone ---------------------------------------------------------
def _words(g, n, v):
    """n tokens whose frequencies fall about as one over their rank."""
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    return (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))

    def normal(*shape, std=1.0):
        t = torch.randn(shape, generator=g, device=DEV)
        return t.mul_(std) if std != 1.0 else t

    if case["op"] == "embedding":
        b, l, v, d = (case[k] for k in ("b", "l", "v", "d"))
        tokens = _words(g, b * l, v).view(b, l)
        if case["padded"]:  # token 0 behind each text's end
            end = l - torch.arange(b, device=DEV) * l // (2 * b)
            tokens = torch.where(torch.arange(l, device=DEV)[None] < end[:, None], tokens, 0)
        ins = {"w": normal(v, d, std=0.02), "tokens": tokens.to(torch.int32).contiguous(), "scale": math.sqrt(d)}
        if case["train"]:
            ins["g"] = normal(b, l, d)
        return ins
    if case["op"] == "dropout":
        ins = {"x": normal(case["rows"], case["d"]), "seed": (int(seed) * 0x9E3779B9 + 12345) % 2 ** 63, "offset": 7 + int(seed) % 1000}
        if case["residual"]:
            ins["r"] = normal(case["rows"], case["d"])
        if case["train"]:
            ins["g"] = normal(case["rows"], case["d"])
        return ins
    n, d, v = (case[k] for k in ("n", "d", "v"))
    labels = _words(g, n, v)
    w = normal(v, d, std=2.0 / math.sqrt(d))
    # states that lean towards their words, some of them far: probabilities from even ones to near certainty
    x = normal(n, d)
    x += w[labels] * (4.0 * torch.rand((n, 1), generator=g, device=DEV) ** 2)
    labels = torch.where(torch.rand(n, generator=g, device=DEV) < case["ignored"], IGNORED, labels)
    labels[0] = min(v - 1, 1)  # one counts at least
    ins = {"x": x, "w": w, "labels": labels.to(torch.int32)}
    if case["bias"]:
        ins["bias"] = normal(v, std=0.5)
    return ins


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    torch.cuda.synchronize()
    return state


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state, state["case"])
    return _PLAIN[state["case"]["op"]](state, state["case"])


# ---- the plain forms ---------------------------------------------------------------------------------------
def _plain_embedding(state, case):
    tokens, scale = state["tokens"].long(), state["scale"]
    y = state["w"][tokens] * scale
    if not case["train"]:
        return {"y": y}
    g = state["g"] * scale
    if case["padded"]:
        g = g * (tokens != 0)[..., None]
    gw = torch.zeros_like(state["w"])
    return {"y": y, "gw": gw.index_add_(0, tokens.view(-1), g.view(-1, case["d"]))}


_LOW = 0xFFFFFFFF


def _kept(n, p, seed, offset):
    """Which of n values stay: the generator Philox 4x32 of 10 rounds, key `seed`, counter (i / 4, offset), gives value i its word
    i % 4; it stays where that is at least p 2^32."""
    at = torch.arange((n + 3) // 4, device=DEV)
    c0, c1 = at & _LOW, at >> 32
    c2, c3 = torch.full_like(at, offset & _LOW), torch.full_like(at, offset >> 32)
    k0, k1 = seed & _LOW, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the 64 bits of the products, whatever the sign they are given
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack((c0, c1, c2, c3), -1).view(-1)[:n] >= int(round(p * 2.0 ** 32))


def _plain_dropout(state, case):
    x = state["x"]
    keep = _kept(x.numel(), case["p"], state["seed"], state["offset"]).view(x.shape)
    scale = 1.0 / (1.0 - case["p"])
    y = torch.where(keep, x * scale, 0.0)
    if case["residual"]:
        y = state["r"] + y
    if not case["train"]:
        return {"y": y}
    return {"y": y, "gx": torch.where(keep, state["g"] * scale, 0.0)}


def _plain_loss(state, case):
    x, w, labels = state["x"], state["w"], state["labels"].long()
    counts = labels != IGNORED
    at = torch.where(counts, labels, 0)[:, None]
    z = x @ w.t()
    if case["bias"]:
        z = z + state["bias"]
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True)
    rows = (torch.log(total) + m - z.gather(1, at))[:, 0] * counts
    number = counts.sum()
    loss = (rows.sum() / number).view(1)
    if not case["train"]:
        return {"loss": loss, "rows": rows}
    p = e / total
    p.scatter_add_(1, at, torch.full_like(m, -1.0))
    p = p * (counts / number)[:, None]
    res = {"loss": loss, "gx": p @ w, "gw": p.t() @ x}
    if case["bias"]:
        res["gb"] = p.sum(0)
    return res


_PLAIN = {"embedding": _plain_embedding, "dropout": _plain_dropout, "loss": _plain_loss}


# ---- the framework's operators -------------------------------------------------------------------------------
_shared = {}


def _kernels():
    if not _shared:
        from newch_amd import hip
        _shared["k"] = hip.Kernels()
    return _shared["k"]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _buffers(state, make):
    """The program's outputs and workspaces, allocated with its first pass and kept."""
    if "buffers" not in state:
        state["buffers"] = make()
    return state["buffers"]


def _workspace(n):
    return torch.empty(max(int(n), 256), device=DEV, dtype=torch.uint8)


def _own_embedding(state, case):
    K, st, w, tokens = _kernels(), _stream(), state["w"], state["tokens"]
    n, v, d = tokens.numel(), case["v"], case["d"]

    def make():
        m = {"y": torch.empty(case["b"], case["l"], d, device=DEV)}
        if case["train"]:
            m.update(gw=torch.empty(v, d, device=DEV), ws=_workspace(K.embedding_bwd_workspace(n, v, d)))
        return m

    m = _buffers(state, make)
    K.embedding_fwd(n, v, d, w.data_ptr(), w.stride(0), tokens.data_ptr(), state["scale"], m["y"].data_ptr(), stream=st)
    if not case["train"]:
        return {"y": m["y"]}
    K.embedding_bwd(n, v, d, tokens.data_ptr(), 0 if case["padded"] else -1, state["scale"], state["g"].data_ptr(),
                    m["gw"].data_ptr(), m["ws"].data_ptr(), m["ws"].numel(), accumulate=False, stream=st)
    return {"y": m["y"], "gw": m["gw"]}


def _own_dropout(state, case):
    K, st, x = _kernels(), _stream(), state["x"]
    m = _buffers(state, lambda: {k: torch.empty_like(x) for k in (("y", "gx") if case["train"] else ("y",))})
    K.dropout_fwd(x.numel(), case["p"], state["seed"], state["offset"], x.data_ptr(), _ptr(state.get("r")), m["y"].data_ptr(),
                  stream=st)
    if not case["train"]:
        return {"y": m["y"]}
    K.dropout_bwd(x.numel(), case["p"], state["seed"], state["offset"], state["g"].data_ptr(), m["gx"].data_ptr(),
                  accumulate=False, stream=st)
    return {"y": m["y"], "gx": m["gx"]}


def _own_loss(state, case):
    K, st, x, w, bias = _kernels(), _stream(), state["x"], state["w"], state.get("bias")
    n, d, v, train = case["n"], case["d"], case["v"], case["train"]

    def make():
        m = {"loss": torch.empty(1, device=DEV)}
        if train:
            m.update(gx=torch.empty_like(x), gw=torch.empty_like(w))
            if case["bias"]:
                m["gb"] = torch.empty_like(bias)
        else:
            m["rows"] = torch.empty(n, device=DEV)
        m["ws"] = _workspace(K.linear_cross_entropy_workspace(n, d, v, gx=train, gw=train, gb=train and case["bias"]))
        return m

    m = _buffers(state, make)
    K.linear_cross_entropy(n, d, v, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), _ptr(bias), state["labels"].data_ptr(),
                           m["loss"].data_ptr(), m["ws"].data_ptr(), m["ws"].numel(), ignore=IGNORED, rows=_ptr(m.get("rows")),
                           gx=_ptr(m.get("gx")), gw=_ptr(m.get("gw")), gb=_ptr(m.get("gb")), accumulate=False, stream=st)
    return {k: m[k] for k in ("loss", "rows", "gx", "gw", "gb") if k in m}


_OWN = {"embedding": _own_embedding, "dropout": _own_dropout, "loss": _own_loss}


# ---- what a pass cannot do without --------------------------------------------------------------------------
def work(case):
    """Bytes: inputs read once, results written once; flops: the products' multiply-adds, a few a value elsewhere."""
    if case["op"] == "embedding":
        n, v, d = case["b"] * case["l"], case["v"], case["d"]
        looked_up = v * -math.expm1(-n / v) if n < v else min(n, v) * 0.6  # rows of the table that occur, about
        b = 4 * (n * d + looked_up * d + n)
        if case["train"]:
            b += 4 * (n * d + v * d + n)
        return {"bytes": int(b), "flops": (2 if case["train"] else 1) * n * d}
    if case["op"] == "dropout":
        n = case["rows"] * case["d"]
        return {"bytes": 4 * n * ((3 if case["residual"] else 2) + (2 if case["train"] else 0)), "flops": 2 * n}
    n, d, v = (case[k] for k in ("n", "d", "v"))
    once = n * d + v * d + (v if case["bias"] else 0)
    return {"bytes": 4 * (once * (2 if case["train"] else 1) + n), "flops": (6 if case["train"] else 2) * n * d * v}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------
def _mask_exactly(n, p, seed, offset):
    """The generator again, its products put together from halves of 16 bits."""
    def product(a, m):
        hi16, lo16 = m >> 16, m & 0xFFFF
        low = a * lo16
        mid = a * hi16 + (low >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)

    block = torch.arange(-(-n // 4), dtype=torch.int64, device=DEV)
    word = [block % 2 ** 32, block // 2 ** 32, torch.zeros_like(block) + offset % 2 ** 32, torch.zeros_like(block) + offset // 2 ** 32]
    for turn in range(10):
        key = ((seed % 2 ** 32 + turn * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + turn * 0xBB67AE85) % 2 ** 32)
        h0, l0 = product(word[0], 0xD2511F53)
        h1, l1 = product(word[2], 0xCD9E8D57)
        word = [h1 ^ word[1] ^ key[0], l1, h0 ^ word[3] ^ key[1], l0]
    drawn = torch.empty(4 * block.numel(), dtype=torch.int64, device=DEV)
    for i in range(4):
        drawn[i::4] = word[i]
    return drawn[:n] >= round(p * 2 ** 32)


def exact(case, seed):
    ins = _inputs(case, seed)
    if case["op"] == "embedding":
        t, s, d = ins["tokens"].long(), ins["scale"], case["d"]
        y = torch.nn.functional.embedding(t, ins["w"].double()) * s
        if not case["train"]:
            return {"y": y}
        g = ins["g"].double().view(-1, d)
        flat = t.view(-1)
        if case["padded"]:
            g, flat = g[flat != 0], flat[flat != 0]
        order = torch.argsort(flat, stable=True)
        gw = torch.zeros(case["v"], d, dtype=torch.float64, device=DEV)
        gw.index_put_((flat[order],), g[order] * s, accumulate=True)
        return {"y": y, "gw": gw}
    if case["op"] == "dropout":
        x = ins["x"].double()
        m = _mask_exactly(x.numel(), case["p"], ins["seed"], ins["offset"]).view(x.shape).double() / (1.0 - case["p"])
        res = {"y": x * m + (ins["r"].double() if case["residual"] else 0.0)}
        if case["train"]:
            res["gx"] = ins["g"].double() * m
        return res
    n, v = case["n"], case["v"]
    w, labels = ins["w"].double(), ins["labels"].long()
    number = int((labels != IGNORED).sum())
    rows = torch.zeros(n, dtype=torch.float64, device=DEV)
    res = {"gx": torch.zeros(n, case["d"], dtype=torch.float64, device=DEV), "gw": torch.zeros_like(w),
           "gb": torch.zeros(v, dtype=torch.float64, device=DEV)} if case["train"] else {}
    step = max(1, min(n, (1 << 27) // v))
    for i in range(0, n, step):
        part = torch.arange(i, min(n, i + step), device=DEV)
        part = part[labels[part] != IGNORED]
        if part.numel() == 0:
            continue
        x, at = ins["x"][part].double(), labels[part]
        logp = x @ w.T
        if case["bias"]:
            logp += ins["bias"].double()
        logp = torch.log_softmax(logp, -1)
        here = torch.arange(part.numel(), device=DEV)
        rows[part] = -logp[here, at]
        if case["train"]:
            p = logp.exp_()
            p[here, at] = torch.expm1(-rows[part])
            p /= number
            res["gx"][part] = p @ w
            res["gw"] += p.T @ x
            res["gb"] += p.sum(0)
    out = {"loss": rows.sum().view(1) / number}
    if not case["train"]:
        return dict(out, rows=rows)
    if not case["bias"]:
        del res["gb"]
    return dict(out, **res)
