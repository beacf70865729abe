"""Performance cases of the attention block's operators: rotary positions of several axes, the per-head norm of queries and
keys with the rotation in the same pass, and attention of queries to keys and values of another length.

Tensors are [batch, tokens, heads, head dim], as a projection leaves them.  The plain forms are elementary torch operations in
32 bits (angles in 64); the framework's operators are called through its kernel layer on the program's own buffers.
"""
import math

import torch

DEV = "cuda"
EPS = 1e-6
BASE = 10000.0
own = False


def listed():
    return [
        # positions of 32 x 32 image patches, in training: the rotation and its gradient
        {"name": "rope_image_train", "op": "rope", "train": True, "b": 8, "l": 1024, "h": 16, "d": 64, "axes": "32+32",
         "interleaved": False},
        # positions of a clip's frames, rows and columns, served; pairs side by side
        {"name": "rope_video", "op": "rope", "train": False, "b": 1, "l": 16384, "h": 32, "d": 128, "axes": "32+48+48",
         "interleaved": True},
        # queries and keys of one new token for each of 16 sequences, far into their texts
        {"name": "qk_norm_token", "op": "qk_norm_rope", "train": False, "b": 16, "l": 1, "hq": 32, "hk": 8, "d": 128,
         "axes": "128", "interleaved": False, "far": True},
        # queries and keys of a fused projection in training, keys' heads shared
        {"name": "qk_norm_train", "op": "qk_norm_rope", "train": True, "b": 4, "l": 2048, "hq": 16, "hk": 4, "d": 128,
         "axes": "128", "interleaved": False, "far": False},
        # a small video model in training: three axes in a head of 80, an odd number of tokens
        {"name": "qk_norm_odd_train", "op": "qk_norm_rope", "train": True, "b": 3, "l": 777, "hq": 5, "hk": 5, "d": 80,
         "axes": "20+30+30", "interleaved": False, "far": False},
        # one new token against an encoder's 1500 states
        {"name": "attention_token", "op": "attention", "train": False, "b": 8, "lq": 1, "lk": 1500, "hq": 12, "hkv": 12,
         "d": 64, "lengths": "full"},
        # one new token of 16 sequences against long caches of unlike lengths, keys' heads shared by four
        {"name": "attention_token_long", "op": "attention", "train": False, "b": 16, "lq": 1, "lk": 16384, "hq": 32,
         "hkv": 8, "d": 128, "lengths": "ragged"},
        # 14 x 14 patches and a class token, 8 images of 12 heads, in training
        {"name": "attention_patches_train", "op": "attention", "train": True, "b": 8, "lq": 197, "lk": 197, "hq": 12,
         "hkv": 12, "d": 64, "lengths": "full"},
        # image patches against a padded text of at most 77 tokens, in training
        {"name": "attention_text_train", "op": "attention", "train": True, "b": 4, "lq": 4096, "lk": 77, "hq": 16,
         "hkv": 16, "d": 64, "lengths": "ragged"},
        # odd sizes all over, shared heads, one sequence of the batch without any state to look at, in training
        {"name": "attention_odd_train", "op": "attention", "train": True, "b": 3, "lq": 1001, "lk": 333, "hq": 8, "hkv": 2,
         "d": 80, "lengths": "empty"},
        # a long prompt against as long a document, served
        {"name": "attention_long", "op": "attention", "train": False, "b": 1, "lq": 8192, "lk": 8192, "hq": 16, "hkv": 16,
         "d": 128, "lengths": "full"},
        # decoder states against encoder states of twice the length, keys' heads shared by four, in training
        {"name": "attention_wide_train", "op": "attention", "train": True, "b": 2, "lq": 2048, "lk": 4096, "hq": 16,
         "hkv": 4, "d": 128, "lengths": "full"},
    ]


def _log_int(rng, lo, hi):
    """lo .. hi, spread over the logarithm; as often as not rounded down to a multiple of 16 where it is large."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.5:
        v -= v % 16
    return max(lo, min(hi, v))


def _axes(rng, d):
    """One to three even sections that fill the head, or leave some of its columns as they are."""
    n = rng.choice((1, 1, 2, 3))
    if n == 1:
        return str(rng.choice((d, d // 4 * 2)))
    each = d // n // 2 * 2
    return "+".join(map(str, [d - each * (n - 1)] + [each] * (n - 1) if d % 2 == 0 else [each] * n))


def draw(rng):
    L = _log_int
    op = rng.choice(("rope", "qk_norm_rope", "attention", "attention"))
    while True:
        if op != "attention":
            c = {"op": op, "train": rng.random() < 0.5, "b": L(rng, 1, 32), "l": L(rng, 1, 16384),
                 "d": rng.choice((32, 40, 64, 80, 96, 128, 256))}
            c.update(axes=_axes(rng, c["d"]), interleaved=rng.random() < 0.5)
            if op == "rope":
                c["h"] = heads = L(rng, 1, 40)
            else:
                c["hk"] = L(rng, 1, 16)
                c.update(hq=c["hk"] * rng.choice((1, 1, 2, 4, 8)), far=rng.random() < 0.5)
                heads = c["hq"] + c["hk"]
            if c["b"] * c["l"] * heads * c["d"] <= 1 << 26:
                return c
            continue
        form = rng.choice(("token", "prompt", "train", "train"))
        c = {"op": op, "train": form == "train", "b": L(rng, 1, 16), "lq": 1 if form == "token" else L(rng, 2, 8192),
             "lk": L(rng, 1, 16384), "hkv": L(rng, 1, 16)}
        c.update(hq=c["hkv"] * rng.choice((1, 1, 2, 4, 8)), d=rng.choice((32, 40, 64, 64, 80, 96, 128, 128)),
                 lengths=rng.choice(("full", "ragged", "ragged", "empty")))
        scores = c["b"] * c["hq"] * c["lq"] * c["lk"]
        if scores * c["d"] * (3 if c["train"] else 1) <= 1 << 37 and c["b"] * c["lk"] * c["hkv"] * c["d"] <= 1 << 28:
            return c


# ---- inputs: plain torch, from the seed alone ---------------------------------------------------------
def _sections(case):
    return [int(n) for n in case["axes"].split("+")]


def _key_lengths(case, g):
    """None, or how many of each sequence's states count: unlike parts of lk, the same ones for every seed in another order."""
    b, lk = case["b"], case["lk"]
    if case["lengths"] == "full":
        return None
    n = [max(1, lk * (i + 1) // b) for i in range(b)]
    if case["lengths"] == "empty" and b > 1:
        n[0] = 0
    return torch.tensor(n, dtype=torch.int32)[torch.randperm(b, generator=g)]


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    host = torch.Generator()
    host.manual_seed(int(seed))

    def normal(*shape, std=1.0, mean=0.0):
        t = torch.randn(shape, generator=g, device=DEV)
        if std != 1.0:
            t.mul_(std)
        return t.add_(mean) if mean else t

    if case["op"] == "attention":
        b, lq, lk, hq, hkv, d = (case[k] for k in ("b", "lq", "lk", "hq", "hkv", "d"))
        ins = {"q": normal(b, lq, hq, d, std=1.5), "k": normal(b, lk, hkv, d, std=1.5), "v": normal(b, lk, hkv, d)}
        n = _key_lengths(case, host)
        ins["n"] = None if n is None else n.to(DEV)
        if case["train"]:
            ins["g"] = normal(b, lq, hq, d)
        return ins
    b, l, d, axes = case["b"], case["l"], case["d"], _sections(case)
    if case["op"] == "rope":
        x = normal(b, l, case["h"], d)
        # patches in order: the first axis outermost, each grid about as wide as its neighbour
        side = max(1, math.ceil(l ** (1 / len(axes))))
        at, pos = torch.arange(l, device=DEV), []
        for _ in axes:
            pos.insert(0, at % side)
            at = at // side
        pos = torch.stack(pos, -1)
    else:
        # queries and keys as the first columns of one projection that holds the values behind them
        hq, hk = case["hq"], case["hk"]
        x = normal(b, l, (hq + 2 * hk) * d, std=2.0)[:, :, : (hq + hk) * d].unflatten(2, (hq + hk, d))
        start = torch.randint(0, 200_000 if case["far"] else 64, (b, 1, len(axes)), generator=g, device=DEV)
        pos = start + torch.arange(l, device=DEV)[None, :, None]
    ins = {"x": x, "pos": pos.to(torch.int32).contiguous()}
    if case["op"] == "qk_norm_rope":
        ins.update(wq=normal(d, std=0.2, mean=1.0), wk=normal(d, std=0.2, mean=1.0))
    if case["train"]:
        ins["g"] = normal(b, l, x.shape[2], d)
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
def _turned(x, pos, case, sign):
    """x with the pairs of each axis's section turned by their angles, which are taken in 64 bits."""
    out, at = [], 0
    for a, d in enumerate(_sections(case)):
        freq = BASE ** (torch.arange(0, d, 2, device=x.device, dtype=torch.float64) / -d)
        angle = (pos[..., a, None].double() * freq)[..., None, :]
        c, s = torch.cos(angle).float(), (sign * torch.sin(angle)).float()
        part = x[..., at: at + d]
        if case["interleaved"]:
            x1, x2 = part[..., 0::2], part[..., 1::2]
            out.append(torch.stack((x1 * c - x2 * s, x2 * c + x1 * s), -1).flatten(-2))
        else:
            x1, x2 = part[..., : d // 2], part[..., d // 2:]
            out += [x1 * c - x2 * s, x2 * c + x1 * s]
        at += d
    return torch.cat(out + [x[..., at:]], -1)


def _plain_rope(state, case):
    y = _turned(state["x"], state["pos"], case, 1.0)
    if not case["train"]:
        return {"y": y}
    return {"y": y, "gx": _turned(state["g"], state["pos"], case, -1.0)}


def _plain_qk_norm_rope(state, case):
    x, hq, hk, d = state["x"], case["hq"], case["hk"], case["d"]
    w = torch.cat((state["wq"].expand(hq, d), state["wk"].expand(hk, d)))
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * r
    y = _turned(n * w, state["pos"], case, 1.0)
    if not case["train"]:
        return {"y": y}
    g = _turned(state["g"], state["pos"], case, -1.0)
    gw = (g * n).sum((0, 1))
    h = g * w
    gx = r * (h - n * (h * n).mean(-1, keepdim=True))
    return {"y": y, "gx": gx, "gwq": gw[:hq].sum(0), "gwk": gw[hq:].sum(0)}


def _plain_attention(state, case):
    b, lq, lk, hq, hkv, d = (case[k] for k in ("b", "lq", "lk", "hq", "hkv", "d"))
    group, scale = hq // hkv, d ** -0.5

    def rows(t):  # [b, lq, hq, d] -> [b * hkv, group * lq, d]: the queries that share a head of keys
        return t.view(b, lq, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b * hkv, group * lq, d)

    def back(t):
        return t.view(b, hkv, group, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, hq, d)

    def states(t):  # [b, lk, hkv, d] -> [b * hkv, lk, d]
        return t.permute(0, 2, 1, 3).reshape(b * hkv, lk, d)

    def back_states(t):
        return t.view(b, hkv, lk, d).permute(0, 2, 1, 3).contiguous()

    q, k, v = rows(state["q"]), states(state["k"]), states(state["v"])
    s = torch.bmm(q, k.transpose(1, 2).contiguous()) * scale
    if state["n"] is not None:
        out = torch.arange(lk, device=q.device)[None, :] >= state["n"][:, None]
        out = out[:, None, None, :].expand(b, hkv, 1, lk).reshape(b * hkv, 1, lk)
        s = s.masked_fill(out, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True)).masked_fill(out, 0.0)
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
    else:
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    o = torch.bmm(p, v)
    if not case["train"]:
        return {"o": back(o)}
    g = rows(state["g"])
    gv = torch.bmm(p.transpose(1, 2).contiguous(), g)
    ds = torch.bmm(g, v.transpose(1, 2).contiguous())
    ds = p * (ds - (g * o).sum(-1, keepdim=True)) * scale
    gq = torch.bmm(ds, k)
    gk = torch.bmm(ds.transpose(1, 2).contiguous(), q)
    return {"o": back(o), "gq": back(gq), "gk": back_states(gk), "gv": back_states(gv)}


_PLAIN = {"rope": _plain_rope, "qk_norm_rope": _plain_qk_norm_rope, "attention": _plain_attention}


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


def _rotation(state, case):
    pos = state["pos"]
    return pos.data_ptr(), pos.dim() == 3, _sections(case), BASE, case["interleaved"]


def _own_rope(state, case):
    K, x, st = _kernels(), state["x"], _stream()
    shape, turn = tuple(x.shape), _rotation(state, case)
    m = _buffers(state, lambda: {"y": torch.empty(shape, device=DEV),
                                 "gx": torch.empty(shape, device=DEV) if case["train"] else None})
    K.rope_fwd(*shape, x.data_ptr(), x.stride()[:3], *turn, m["y"].data_ptr(), stream=st)
    if not case["train"]:
        return {"y": m["y"]}
    K.rope_bwd(*shape, state["g"].data_ptr(), *turn, m["gx"].data_ptr(), accumulate=False, stream=st)
    return {"y": m["y"], "gx": m["gx"]}


def _own_qk_norm_rope(state, case):
    K, x, st = _kernels(), state["x"], _stream()
    shape, turn = tuple(x.shape), _rotation(state, case)

    def make():
        m = {"y": torch.empty(shape, device=DEV)}
        if case["train"]:
            m.update(gx=torch.empty(shape, device=DEV), gwq=torch.empty(case["d"], device=DEV),
                     gwk=torch.empty(case["d"], device=DEV), ws=_workspace(K.qk_norm_rope_bwd_workspace(*shape)))
        return m

    m = _buffers(state, make)
    src = (x.data_ptr(), x.stride()[:3], state["wq"].data_ptr(), state["wk"].data_ptr(), EPS)
    K.qk_norm_rope_fwd(*shape, case["hq"], *src, *turn, m["y"].data_ptr(), stream=st)
    if not case["train"]:
        return {"y": m["y"]}
    K.qk_norm_rope_bwd(*shape, case["hq"], *src, *turn, state["g"].data_ptr(), m["gx"].data_ptr(), m["gwq"].data_ptr(),
                       m["gwk"].data_ptr(), m["ws"].data_ptr(), m["ws"].numel(), accumulate=False, stream=st)
    return {k: m[k] for k in ("y", "gx", "gwq", "gwk")}


def _own_attention(state, case):
    K, st = _kernels(), _stream()
    sizes = tuple(case[k] for k in ("b", "lq", "lk", "hq", "hkv", "d"))
    q, k, v, train = state["q"], state["k"], state["v"], case["train"]

    def make():
        m = {"o": torch.empty_like(q), "ws": _workspace(K.cross_attention_fwd_workspace(*sizes)), "lse": None}
        if train:
            m.update(lse=torch.empty(case["b"], case["hq"], case["lq"], device=DEV), gq=torch.empty_like(q),
                     gk=torch.empty_like(k), gv=torch.empty_like(v),
                     ws2=_workspace(K.cross_attention_bwd_workspace(*sizes)))
        return m

    m = _buffers(state, make)
    src = sum(((t.data_ptr(), t.stride()[:3]) for t in (q, k, v)), ()) + (_ptr(state["n"]),)
    K.cross_attention_fwd(*sizes, case["d"] ** -0.5, *src, m["o"].data_ptr(), _ptr(m["lse"]), m["ws"].data_ptr(),
                          m["ws"].numel(), stream=st)
    if not train:
        return {"o": m["o"]}
    K.cross_attention_bwd(*sizes, case["d"] ** -0.5, *src, m["o"].data_ptr(), m["lse"].data_ptr(), state["g"].data_ptr(),
                          m["gq"].data_ptr(), m["gk"].data_ptr(), m["gv"].data_ptr(), m["ws2"].data_ptr(),
                          m["ws2"].numel(), stream=st)
    return {i: m[i] for i in ("o", "gq", "gk", "gv")}


_OWN = {"rope": _own_rope, "qk_norm_rope": _own_qk_norm_rope, "attention": _own_attention}


# ---- what a pass cannot do without --------------------------------------------------------------------------
def work(case):
    """Bytes: inputs read once, results written once; flops: the products' multiply-adds, a few a value elsewhere."""
    if case["op"] == "attention":
        b, lq, lk, hq, hkv, d = (case[k] for k in ("b", "lq", "lk", "hq", "hkv", "d"))
        n = _key_lengths(case, torch.Generator())
        keys = b * lk if n is None else int(n.sum())
        queries, scores = b * lq * hq * d, lq * hq * keys
        if not case["train"]:
            return {"bytes": 4 * (2 * queries + 2 * keys * hkv * d), "flops": 4 * scores * d}
        return {"bytes": 4 * (4 * queries + 2 * keys * hkv * d + 2 * b * lk * hkv * d), "flops": 14 * scores * d}
    n = case["b"] * case["l"] * case["d"] * (case["h"] if case["op"] == "rope" else case["hq"] + case["hk"])
    if case["op"] == "rope":
        return {"bytes": (16 if case["train"] else 8) * n, "flops": (6 if case["train"] else 3) * n}
    return {"bytes": (16 if case["train"] else 8) * n, "flops": (22 if case["train"] else 7) * n}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------
def _turned_exactly(x, pos, case):
    """The rotation as a product of complex numbers."""
    out, at = x.clone(), 0
    for a, d in enumerate(_sections(case)):
        cols = torch.arange(at, at + d, device=x.device)
        first, second = (cols[0::2], cols[1::2]) if case["interleaved"] else cols.chunk(2)
        j = torch.arange(d // 2, device=x.device, dtype=torch.float64)
        angle = pos[..., a].double()[..., None] * torch.exp(j * (-2.0 * math.log(BASE) / d))
        z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)[..., None, :]
        out = out.index_copy(-1, first, z.real).index_copy(-1, second, z.imag)
        at += d
    return out


def exact(case, seed):
    ins = _inputs(case, seed)
    x64 = {k: ins[k].double() for k in ("x", "wq", "wk", "g", "q", "k", "v") if k in ins}
    if case["op"] != "attention":
        leaves = {k: x64[k].requires_grad_(case["train"]) for k in ("x", "wq", "wk") if k in x64}
        n = leaves["x"]
        if case["op"] == "qk_norm_rope":
            n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + EPS)
            n = torch.cat((n[:, :, : case["hq"]] * leaves["wq"], n[:, :, case["hq"]:] * leaves["wk"]), 2)
        y = _turned_exactly(n, ins["pos"], case)
        res = {"y": y.detach()}
        if case["train"]:
            y.backward(x64["g"])
            res.update({"g" + k: v.grad for k, v in leaves.items()})
        return res
    b, hq, hkv, d = (case[k] for k in ("b", "hq", "hkv", "d"))
    res = {"o": torch.zeros_like(x64["q"])}
    if case["train"]:
        res.update({"g" + k: torch.zeros_like(x64[k]) for k in "qkv"})
    for i in range(b):
        n = case["lk"] if ins["n"] is None else int(ins["n"][i])
        if n == 0:
            continue
        for h in range(hq):
            u = h // (hq // hkv)
            q, k, v = x64["q"][i, :, h], x64["k"][i, :n, u], x64["v"][i, :n, u]
            p = torch.softmax(q @ k.T * d ** -0.5, -1)
            res["o"][i, :, h] = p @ v
            if case["train"]:
                g = x64["g"][i, :, h]
                t = g @ v.T
                t = p * (t - (p * t).sum(-1, keepdim=True)) * d ** -0.5
                res["gq"][i, :, h] = t @ k
                res["gk"][i, :n, u] += t.T @ q
                res["gv"][i, :n, u] += p.T @ g
    return res
