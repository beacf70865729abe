// The attention block: rotary positions, the per-head norm of queries and keys with the rotation, and cross attention.  No
// counterpart in the reference, whose Python layer composes attention of matmul, masked_fill and softmax.
//
// Tensors are [B, L, H, D].  The backwards read the forward's inputs again (and, for attention, its output and the rows'
// log-sum-exps): they refuse inputs that were written since.
#include <math.h>

#include "engine.hpp"

namespace nce {

constexpr int kMaxAxes = 4;
constexpr int64_t kMaxHeadDim = 256;

// a [B, L, H, D] tensor as the kernels read it: element 0 and the strides of batch, token and head
struct Heads {
    const float *p;
    int64_t s[3];
};

static bool heads_of(nc_tensor *t, Heads &h) {
    const bool in_place = t->stride[3] == 1 || t->shape[3] == 1;
    h.p = in_place ? fptr(t) : contig_f32(t);
    h.s[2] = in_place ? t->stride[2] : t->shape[3];
    h.s[1] = in_place ? t->stride[1] : h.s[2] * t->shape[2];
    h.s[0] = in_place ? t->stride[0] : h.s[1] * t->shape[1];
    return h.p != nullptr;
}

// i32 tensor, contiguous on the device (itself, or a copy that lives as long as the call)
static const int32_t *contig_i32(nc_tensor *t) {
    char *p = dptr(t);
    if (!p || nc_is_contiguous(t)) return (const int32_t *)p;
    char *c = arena_alloc(t->ctx, (size_t)nc_numel(t) * sizeof(int32_t));
    if (!c || !hip_layer_ok(t->ctx, nc_hip_copy_strided(4, t->ndim, t->shape, p, t->stride, c, stream(t->ctx)), "copy"))
        return nullptr;
    return (const int32_t *)c;
}

// counts every write to the storage of the inputs from `first` on: the same number means that none was written
static int64_t generations(const nc_node *n, int first = 0) {
    uint64_t g = 0;
    for (int i = first; i < n->n_in; i++) g += owner_of(n->in[i])->wgen;
    return (int64_t)g;
}

static bool unwritten(const nc_node *n, int64_t then, int first = 0) {
    if (generations(n, first) == then) return true;
    error(n->in[0]->ctx, NC_ERR_STATE, "%s: an input was written after the forward (the backward reads it again)", n->op->name);
    return false;
}

// ---- rotary positions, with or without the norm ------------------------------------------------------
// inputs: x, then positions, q_weight, k_weight as the flags say.  p.i: axes, their columns [4], flags, q_heads, generations;
// p.f: base, eps
enum { ROPE_PLAIN = 0, ROPE_NORM = 1 };
enum { RF_INTERLEAVED = 1, RF_POS = 2, RF_WQ = 4, RF_WK = 8 };

struct RopeCall {
    nc_tensor *x, *pos = nullptr, *wq = nullptr, *wk = nullptr;
    int axes, flags;
    const int64_t *dims;
    int64_t q_heads, B, L, H, D;

    explicit RopeCall(const nc_node *n) : x(n->in[0]), axes((int)n->p.i[0]), flags((int)n->p.i[5]), dims(n->p.i + 1), q_heads(n->p.i[6]) {
        int k = 1;
        if (flags & RF_POS) pos = n->in[k++];
        if (flags & RF_WQ) wq = n->in[k++];
        if (flags & RF_WK) wk = n->in[k++];
        B = x->shape[0], L = x->shape[1], H = x->shape[2], D = x->shape[3];
    }
    bool batched() const { return pos && pos->ndim == 3; }
    bool interleaved() const { return (flags & RF_INTERLEAVED) != 0; }
};

static nc_status rope_shape(nc_node *n, OutSpec &out) {
    const char *name = n->op->name;
    const RopeCall c(n);
    const nc_tensor *floats[3] = {c.x, c.wq, c.wk};
    for (const nc_tensor *t : floats)
        if (t && t->dtype != NC_F32) return reject(n, NC_ERR_DTYPE, "%s: x and weights must be f32", name);
    if (c.pos && c.pos->dtype != NC_I32) return reject(n, NC_ERR_DTYPE, "%s: positions must be i32", name);
    out.dims = Dims::of(c.x);
    char tx[96], tp[96];
    if (out.dims.rank != 4 || c.D < 1 || c.D > kMaxHeadDim)
        return reject(n, NC_ERR_SHAPE, "%s: expected x [batch, tokens, heads, 1 to %d columns], got %s", name,
                      (int)kMaxHeadDim, out.dims.text(tx, sizeof tx));
    int64_t cols = 0;
    for (int a = 0; a < c.axes; a++) {
        if (c.dims[a] < 2 || c.dims[a] % 2 || c.dims[a] > c.D - cols)
            return reject(n, NC_ERR_SHAPE, "%s: axis %d has %lld columns (even, at least 2, %lld left in the head)", name, a,
                          (long long)c.dims[a], (long long)(c.D - cols));
        cols += c.dims[a];
    }
    if (c.pos) {
        const Dims p = Dims::of(c.pos);
        const bool ok = (p.rank == 2 || (p.rank == 3 && p.e[0] == c.B)) && p.back(0) == c.axes && p.back(1) == c.L;
        if (!ok)
            return reject(n, NC_ERR_SHAPE, "%s: expected positions [tokens, axes] or [batch, tokens, axes] for %d axes of x %s, got %s",
                          name, c.axes, out.dims.text(tx, sizeof tx), p.text(tp, sizeof tp));
    }
    if (c.q_heads < 0 || c.q_heads > c.H)
        return reject(n, NC_ERR_ARG, "%s: %lld query heads of %lld", name, (long long)c.q_heads, (long long)c.H);
    for (int i = 1; i < 3; i++)
        if (floats[i] && (floats[i]->ndim != 1 || floats[i]->shape[0] != c.D))
            return reject(n, NC_ERR_SHAPE, "%s: weights need %lld elements", name, (long long)c.D);
    const float base = n->p.f[0], eps = n->p.f[1];
    if (c.axes && !(base > 0.0f && isfinite(base))) return reject(n, NC_ERR_ARG, "%s: the base must be positive and finite", name);
    if (!(eps >= 0.0f && isfinite(eps))) return reject(n, NC_ERR_ARG, "%s: eps must be finite and not negative", name);
    return NC_OK;
}

static nc_status rope_fwd(nc_node *n) {
    const RopeCall c(n);
    nc_ctx *ctx = c.x->ctx;
    Heads x;
    float *y = fptr(n->out);
    if (!y || !heads_of(c.x, x)) return NC_ERR_STATE;
    const int32_t *pos = c.pos ? contig_i32(c.pos) : nullptr;
    const float *wq = c.wq ? contig_f32(c.wq) : nullptr, *wk = c.wk ? contig_f32(c.wk) : nullptr;
    if ((c.pos && !pos) || (c.wq && !wq) || (c.wk && !wk)) return NC_ERR_STATE;
    const int rc = n->op->kind == ROPE_PLAIN
                       ? nc_hip_rope_fwd(c.B, c.L, c.H, c.D, x.p, x.s, pos, c.batched(), c.axes, c.dims, n->p.f[0], c.interleaved(), y, stream(ctx))
                       : nc_hip_qk_norm_rope_fwd(c.B, c.L, c.H, c.D, c.q_heads, x.p, x.s, wq, wk, n->p.f[1], pos, c.batched(), c.axes, c.dims,
                                                 n->p.f[0], c.interleaved(), y, stream(ctx));
    if (!hip_layer_ok(ctx, rc, n->op->name)) return NC_ERR_STATE;
    wrote_dev(n->out);
    n->p.i[7] = generations(n, n->op->kind == ROPE_PLAIN);
    return NC_OK;
}

static void rope_bwd(nc_node *n) {
    const RopeCall c(n);
    nc_ctx *ctx = c.x->ctx;
    if (!unwritten(n, n->p.i[7], n->op->kind == ROPE_PLAIN)) return;  // the rotation alone does not read x again
    const float *g = fptr(n->out->grad);
    const int32_t *pos = c.pos ? contig_i32(c.pos) : nullptr;
    if (!g || (c.pos && !pos)) return;
    const bool want_x = needs_grad(c.x), want_q = c.wq && needs_grad(c.wq), want_k = c.wk && needs_grad(c.wk);
    if (want_x && !grad_buf(c.x)) return;
    if (n->op->kind == ROPE_PLAIN) {
        if (!want_x) return;
        const int acc = grad_acc(c.x);
        float *gx = fptr(c.x->grad);
        if (gx && hip_layer_ok(ctx, nc_hip_rope_bwd(c.B, c.L, c.H, c.D, g, pos, c.batched(), c.axes, c.dims, n->p.f[0], c.interleaved(), gx, acc, stream(ctx)), n->op->name))
            wrote_dev(c.x->grad);
        return;
    }
    Heads x;
    if (!heads_of(c.x, x)) return;
    const float *wq = c.wq ? contig_f32(c.wq) : nullptr, *wk = c.wk ? contig_f32(c.wk) : nullptr;
    if ((c.wq && !wq) || (c.wk && !wk) || (want_q && !grad_buf(c.wq)) || (want_k && !grad_buf(c.wk))) return;
    // the kernel writes every row's gradient: into scratch where x wants none
    const size_t bytes = (size_t)nc_numel(c.x) * sizeof(float);
    const int acc_x = want_x ? grad_acc(c.x) : 0;
    float *gx = want_x ? fptr(c.x->grad) : (float *)arena_alloc(ctx, bytes ? bytes : 1);
    // one weight for queries and keys: the keys' part is added afterwards
    const bool shared = want_q && want_k && c.wq == c.wk;
    const int acc_q = want_q ? grad_acc(c.wq) : 0, acc_k = want_k && !shared ? grad_acc(c.wk) : 0;
    float *gwq = want_q ? fptr(c.wq->grad) : nullptr;
    float *gwk = shared ? (float *)arena_alloc(ctx, (size_t)c.D * sizeof(float)) : want_k ? fptr(c.wk->grad) : nullptr;
    const size_t ws_bytes = want_q || want_k ? nc_hip_qk_norm_rope_bwd_workspace(c.B, c.L, c.H, c.D) : 0;
    char *ws = ws_bytes ? arena_alloc(ctx, ws_bytes) : nullptr;
    if (!gx || (want_q && !gwq) || (want_k && !gwk) || (ws_bytes && !ws)) return;
    if (!hip_layer_ok(ctx,
                      nc_hip_qk_norm_rope_bwd(c.B, c.L, c.H, c.D, c.q_heads, x.p, x.s, wq, wk, n->p.f[1], pos, c.batched(), c.axes, c.dims,
                                              n->p.f[0], c.interleaved(), g, gx, gwq, gwk, acc_x, acc_q, acc_k, ws, ws_bytes,
                                              stream(ctx)),
                      n->op->name))
        return;
    if (shared && !hip_layer_ok(ctx, nc_hip_axpy(c.D, 1.0f, gwk, gwq, stream(ctx)), n->op->name)) return;
    if (want_x) wrote_dev(c.x->grad);
    if (want_q) wrote_dev(c.wq->grad);
    if (want_k) wrote_dev(c.wk->grad);
}

static const OpDef op_rope = {"rope", 0, ROPE_PLAIN, rope_shape, nullptr, rope_fwd, rope_bwd};
static const OpDef op_qk_norm_rope = {"qk_norm_rope", 0, ROPE_NORM, rope_shape, nullptr, rope_fwd, rope_bwd};

static nc_tensor *rope_call(const OpDef *op, nc_tensor *x, int64_t q_heads, nc_tensor *wq, nc_tensor *wk, float eps,
                            nc_tensor *pos, int n_axes, const int64_t *dims, float base, int interleaved) {
    if (!x) return nullptr;
    const int least = op->kind == ROPE_PLAIN ? 1 : 0;
    if (n_axes < least || n_axes > kMaxAxes || (n_axes > 0 && (!dims || !pos)) || (n_axes == 0 && pos)) {
        error(x->ctx, NC_ERR_ARG, "%s: %d to %d axes, with their columns and positions", op->name, least, kMaxAxes);
        return nullptr;
    }
    Params p{};
    nc_tensor *in[4] = {x, nullptr, nullptr, nullptr};
    int k = 1;
    p.i[0] = n_axes;
    for (int a = 0; a < n_axes; a++) p.i[1 + a] = dims[a];
    p.i[5] = interleaved ? RF_INTERLEAVED : 0;
    if (pos) in[k++] = pos, p.i[5] |= RF_POS;
    if (wq) in[k++] = wq, p.i[5] |= RF_WQ;
    if (wk) in[k++] = wk, p.i[5] |= RF_WK;
    p.i[6] = q_heads;
    p.f[0] = base;
    p.f[1] = eps;
    return apply(op, in, k, &p);
}

// ---- cross attention -----------------------------------------------------------------------------------
// inputs: q, k, v, then the key lengths where given.  saved: the rows' log-sum-exps [B, Hq, Lq]
struct AttnCall {
    nc_tensor *q, *k, *v, *len;
    int64_t B, Lq, Lk, Hq, Hkv, D;

    explicit AttnCall(const nc_node *n) : q(n->in[0]), k(n->in[1]), v(n->in[2]), len(n->n_in > 3 ? n->in[3] : nullptr) {
        B = q->shape[0], Lq = q->shape[1], Hq = q->shape[2], D = q->shape[3];
        Lk = k->shape[1], Hkv = k->shape[2];
    }
};

static nc_status attn_shape(nc_node *n, OutSpec &out) {
    const char *name = n->op->name;
    if (!inputs_f32(n, 0, 3)) return NC_ERR_DTYPE;
    if (n->n_in > 3 && n->in[3]->dtype != NC_I32) return reject(n, NC_ERR_DTYPE, "%s: key lengths must be i32", name);
    const Dims q = Dims::of(n->in[0]), k = Dims::of(n->in[1]), v = Dims::of(n->in[2]);
    bool ok = q.rank == 4 && k.rank == 4 && v.rank == 4 && q.e[0] == k.e[0] && q.e[3] == k.e[3] && q.e[3] >= 1 &&
              q.e[3] <= kMaxHeadDim && q.e[2] >= 1 && k.e[2] >= 1;
    for (int i = 0; ok && i < 4; i++) ok = k.e[i] == v.e[i];
    char tq[96], tk[96], tv[96];
    if (!ok)
        return reject(n, NC_ERR_SHAPE, "%s: expected q [batch, queries, heads, 1 to %d columns] and k, v [batch, keys, heads, columns], got %s, %s, %s",
                      name, (int)kMaxHeadDim, q.text(tq, sizeof tq), k.text(tk, sizeof tk), v.text(tv, sizeof tv));
    if (q.e[2] % k.e[2])
        return reject(n, NC_ERR_SHAPE, "%s: %lld query heads cannot share %lld heads of keys", name, (long long)q.e[2], (long long)k.e[2]);
    if (n->n_in > 3 && (n->in[3]->ndim != 1 || n->in[3]->shape[0] != q.e[0]))
        return reject(n, NC_ERR_SHAPE, "%s: expected a key length for each of %lld sequences", name, (long long)q.e[0]);
    if (!isfinite(n->p.f[0])) return reject(n, NC_ERR_ARG, "%s: the scale must be finite", name);
    out.dims = q;
    return NC_OK;
}

static nc_status attn_fwd(nc_node *n) {
    const AttnCall c(n);
    nc_ctx *ctx = c.q->ctx;
    Heads q, k, v;
    float *o = fptr(n->out);
    if (!o || !heads_of(c.q, q) || !heads_of(c.k, k) || !heads_of(c.v, v)) return NC_ERR_STATE;
    const int32_t *len = c.len ? contig_i32(c.len) : nullptr;
    float *lse = (float *)save_state(n, (size_t)(c.B * c.Hq * c.Lq) * sizeof(float));
    const size_t ws_bytes = nc_hip_cross_attention_fwd_workspace(c.B, c.Lq, c.Lk, c.Hq, c.Hkv, c.D);
    char *ws = ws_bytes ? arena_alloc(ctx, ws_bytes) : nullptr;
    if ((c.len && !len) || !lse || (ws_bytes && !ws)) return NC_ERR_STATE;
    if (!hip_layer_ok(ctx,
                      nc_hip_cross_attention_fwd(c.B, c.Lq, c.Lk, c.Hq, c.Hkv, c.D, n->p.f[0], q.p, q.s, k.p, k.s, v.p, v.s, len, o, lse,
                                                 ws, ws_bytes, stream(ctx)),
                      n->op->name))
        return NC_ERR_STATE;
    wrote_dev(n->out);
    const nc_tensor *out = owner_of(n->out);
    n->p.i[0] = generations(n);
    n->p.i[1] = (int64_t)out->wgen, n->p.i[2] = (int64_t)out->hgen;
    return NC_OK;
}

// The output as the forward left it: its own storage, or, where the caller had a host pointer to it since (and may have written
// through that), the forward once more into scratch.  An output that a call wrote is refused.
static const float *output_of(const nc_node *n, const AttnCall &c, const Heads &q, const Heads &k, const Heads &v, const int32_t *len) {
    nc_ctx *ctx = c.q->ctx;
    const nc_tensor *out = owner_of(n->out);
    const uint64_t writes = out->wgen - (uint64_t)n->p.i[1], pointers = out->hgen - (uint64_t)n->p.i[2];
    if (writes == 0) return fptr(n->out);
    if (writes != pointers) {
        error(ctx, NC_ERR_STATE, "%s: the output was written after the forward (the backward reads it again)", n->op->name);
        return nullptr;
    }
    const size_t bytes = (size_t)nc_numel(n->out) * sizeof(float), ws_bytes = nc_hip_cross_attention_fwd_workspace(c.B, c.Lq, c.Lk, c.Hq, c.Hkv, c.D);
    float *o = (float *)arena_alloc(ctx, bytes ? bytes : 1);
    char *ws = ws_bytes ? arena_alloc(ctx, ws_bytes) : nullptr;
    if (!o || (ws_bytes && !ws)) return nullptr;
    return hip_layer_ok(ctx,
                        nc_hip_cross_attention_fwd(c.B, c.Lq, c.Lk, c.Hq, c.Hkv, c.D, n->p.f[0], q.p, q.s, k.p, k.s, v.p, v.s, len, o, nullptr,
                                                   ws, ws_bytes, stream(ctx)),
                        n->op->name)
               ? o
               : nullptr;
}

static void attn_bwd(nc_node *n) {
    const AttnCall c(n);
    nc_ctx *ctx = c.q->ctx;
    if (!unwritten(n, n->p.i[0])) return;
    Heads q, k, v;
    const float *go = fptr(n->out->grad);
    if (!go || !heads_of(c.q, q) || !heads_of(c.k, k) || !heads_of(c.v, v)) return;
    const int32_t *len = c.len ? contig_i32(c.len) : nullptr;
    if (c.len && !len) return;
    const float *o = output_of(n, c, q, k, v, len);
    if (!o) return;
    const bool want_q = needs_grad(c.q), want_k = needs_grad(c.k), want_v = needs_grad(c.v);
    if ((want_q && !grad_buf(c.q)) || (want_k && !grad_buf(c.k)) || (want_v && !grad_buf(c.v))) return;
    // One tensor as several of the three has one gradient, and the kernels' must not overlap: its later parts go through scratch.
    nc_tensor *const in[3] = {c.q, c.k, c.v};
    const bool want[3] = {want_q, want_k, want_v};
    int first[3], acc[3];
    float *g[3] = {};
    for (int i = 0; i < 3; i++) {
        first[i] = 0;
        while (in[first[i]] != in[i]) first[i]++;
        const size_t bytes = (size_t)nc_numel(in[i]) * sizeof(float);
        acc[i] = want[i] && first[i] == i ? grad_acc(in[i]) : 0;
        if (want[i]) g[i] = first[i] == i ? fptr(in[i]->grad) : (float *)arena_alloc(ctx, bytes ? bytes : 1);
        if (want[i] && !g[i]) return;
    }
    const size_t ws_bytes = nc_hip_cross_attention_bwd_workspace(c.B, c.Lq, c.Lk, c.Hq, c.Hkv, c.D);
    char *ws = ws_bytes ? arena_alloc(ctx, ws_bytes) : nullptr;
    if (ws_bytes && !ws) return;
    if (!hip_layer_ok(ctx,
                      nc_hip_cross_attention_bwd(c.B, c.Lq, c.Lk, c.Hq, c.Hkv, c.D, n->p.f[0], q.p, q.s, k.p, k.s, v.p, v.s, len, o,
                                                 (const float *)n->saved, go, g[0], g[1], g[2], acc[0], acc[1], acc[2], ws, ws_bytes,
                                                 stream(ctx)),
                      n->op->name))
        return;
    for (int i = 1; i < 3; i++)
        if (want[i] && first[i] != i &&
            !hip_layer_ok(ctx, nc_hip_axpy(nc_numel(in[i]), 1.0f, g[i], g[first[i]], stream(ctx)), n->op->name))
            return;
    for (int i = 0; i < 3; i++)
        if (want[i] && first[i] == i) wrote_dev(in[i]->grad);
}

static const OpDef op_cross_attention = {"cross_attention", 0, 0, attn_shape, nullptr, attn_fwd, attn_bwd};

}  // namespace nce

using namespace nce;

extern "C" {
nc_tensor *nc_rope(nc_tensor *x, nc_tensor *positions, int n_axes, const int64_t *axis_dims, float base, int interleaved) {
    return rope_call(&op_rope, x, 0, nullptr, nullptr, 0.0f, positions, n_axes, axis_dims, base, interleaved);
}

nc_tensor *nc_qk_norm_rope(nc_tensor *x, int64_t q_heads, nc_tensor *q_weight, nc_tensor *k_weight, float eps,
                           nc_tensor *positions, int n_axes, const int64_t *axis_dims, float base, int interleaved) {
    return rope_call(&op_qk_norm_rope, x, q_heads, q_weight, k_weight, eps, positions, n_axes, axis_dims, base, interleaved);
}

nc_tensor *nc_cross_attention(nc_tensor *q, nc_tensor *k, nc_tensor *v, nc_tensor *key_lengths, float scale) {
    nc_tensor *in[4] = {q, k, v, key_lengths};
    Params p{};
    p.f[0] = scale;
    return apply(&op_cross_attention, in, key_lengths ? 4 : 3, &p);
}
}
