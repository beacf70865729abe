// A language model's two ends and the regulariser between them: rows of an embedding table, dropout from a counter, the cross entropy of
// a product whose logits are not kept.  The reference has index_select, dropout and cross_entropy (ops_shape.c, ops_nn.c:168-213, 83-156),
// which copy rows without a gradient by token, keep the mask, and read stored logits.
#include <math.h>

#include "engine.hpp"

namespace nce {

// an i32 tensor's values in `to`, contiguous
static bool copy_i32(nc_tensor *t, int32_t *to, const char *what) {
    const char *from = dptr(t);
    if (!from) return false;
    return nc_numel(t) == 0 || hip_layer_ok(t->ctx, nc_hip_copy_strided(4, t->ndim, t->shape, from, t->stride, to, stream(t->ctx)), what);
}

// a matrix as the kernels read it: element 0 and the distance of its rows
struct Rows {
    const float *p;
    int64_t ld;
};

static bool rows_of(nc_tensor *t, Rows &r) {
    const int64_t cols = t->shape[t->ndim - 1];
    const bool in_place = t->ndim == 2 && t->stride[1] == 1 && t->stride[0] >= cols;
    r.p = in_place ? fptr(t) : contig_f32(t);
    r.ld = in_place ? t->stride[0] : cols;
    return r.p != nullptr;
}

// ---- embedding ---------------------------------------------------------------------------------------------------
// inputs: weight [V, D], tokens.  p.f: scale; p.i: padding.  saved: the tokens
static nc_status embedding_shape(nc_node *n, OutSpec &out) {
    const char *name = n->op->name;
    if (!inputs_f32(n, 0, 1)) return NC_ERR_DTYPE;
    if (n->in[1]->dtype != NC_I32) return reject(n, NC_ERR_DTYPE, "%s: tokens must be i32", name);
    const Dims w = Dims::of(n->in[0]), t = Dims::of(n->in[1]);
    char tw[96], tt[96];
    if (w.rank != 2 || w.e[1] < 1 || t.rank >= NC_MAX_DIMS)
        return reject(n, NC_ERR_SHAPE, "%s: expected weight [words, columns] and tokens of at most %d dims, got %s and %s", name,
                      NC_MAX_DIMS - 1, w.text(tw, sizeof tw), t.text(tt, sizeof tt));
    if (!isfinite(n->p.f[0])) return reject(n, NC_ERR_ARG, "%s: the scale must be finite", name);
    out.dims = t;
    out.dims.push(w.e[1]);
    return NC_OK;
}

static nc_status embedding_fwd(nc_node *n) {
    nc_tensor *w = n->in[0], *t = n->in[1];
    nc_ctx *ctx = w->ctx;
    const int64_t N = nc_numel(t), V = w->shape[0], D = w->shape[1];
    Rows table;
    float *y = fptr(n->out);
    int32_t *tokens = (int32_t *)save_state(n, (size_t)N * sizeof(int32_t));
    IndexCheck check;
    if (!y || !tokens || !rows_of(w, table) || !copy_i32(t, tokens, n->op->name) || !check.begin(ctx)) return NC_ERR_STATE;
    if (!hip_layer_ok(ctx, nc_hip_embedding_fwd(N, V, D, table.p, table.ld, tokens, n->p.f[0], y, check.bad, stream(ctx)), n->op->name) ||
        !check.read(ctx, n->op->name))
        return NC_ERR_STATE;
    if (!check.ok()) {
        error(ctx, NC_ERR_ARG, "%s: token %d at position %lld outside [0, %lld)", n->op->name, check.value(), check.at(), (long long)V);
        return NC_ERR_ARG;
    }
    wrote_dev(n->out);
    return NC_OK;
}

static void embedding_bwd(nc_node *n) {
    nc_tensor *w = n->in[0];
    nc_ctx *ctx = w->ctx;
    const int64_t N = nc_numel(n->in[1]), V = w->shape[0], D = w->shape[1];
    const float *g = fptr(n->out->grad);
    if (!g || !grad_buf(w)) return;
    const size_t ws_bytes = nc_hip_embedding_bwd_workspace(N, V, D);
    char *ws = ws_bytes ? arena_alloc(ctx, ws_bytes) : nullptr;
    if (ws_bytes && !ws) return;
    const int acc = grad_acc(w);
    float *gw = fptr(w->grad);
    if (gw && hip_layer_ok(ctx,
                           nc_hip_embedding_bwd(N, V, D, (const int32_t *)n->saved, (int32_t)n->p.i[0], n->p.f[0], g, gw, acc, ws, ws_bytes,
                                                stream(ctx)),
                           n->op->name))
        wrote_dev(w->grad);
}

static const OpDef op_embedding = {"embedding", 0, 0, embedding_shape, nullptr, embedding_fwd, embedding_bwd};

// ---- dropout -------------------------------------------------------------------------------------------------------
// inputs: x, then the residual where given.  p.i: seed, offset, the bits of p
static double dropout_p(const nc_node *n) {
    double p;
    memcpy(&p, &n->p.i[2], sizeof p);
    return p;
}

static nc_status dropout_shape(nc_node *n, OutSpec &out) {
    if (!inputs_f32(n, 0, n->n_in)) return NC_ERR_DTYPE;
    const double p = dropout_p(n);
    if (!(p >= 0.0 && p <= 1.0)) return reject(n, NC_ERR_ARG, "%s: p must be in [0, 1], got %g", n->op->name, p);
    out.dims = Dims::of(n->in[0]);
    if (n->n_in > 1 && !same_shape(n->in[0], n->in[1])) {
        char tx[96], tr[96];
        return reject(n, NC_ERR_SHAPE, "%s: x %s and the residual %s differ", n->op->name, out.dims.text(tx, sizeof tx),
                      Dims::of(n->in[1]).text(tr, sizeof tr));
    }
    return NC_OK;
}

static nc_status dropout_fwd(nc_node *n) {
    nc_ctx *ctx = n->in[0]->ctx;
    const float *x = contig_f32(n->in[0]), *r = n->n_in > 1 ? contig_f32(n->in[1]) : nullptr;
    float *y = fptr(n->out);
    if (!x || !y || (n->n_in > 1 && !r)) return NC_ERR_STATE;
    if (!hip_layer_ok(ctx,
                      nc_hip_dropout_fwd(nc_numel(n->out), dropout_p(n), (uint64_t)n->p.i[0], (uint64_t)n->p.i[1], nullptr, x, r, y, stream(ctx)),
                      n->op->name))
        return NC_ERR_STATE;
    wrote_dev(n->out);
    return NC_OK;
}

static void dropout_bwd(nc_node *n) {
    nc_ctx *ctx = n->in[0]->ctx;
    const int64_t count = nc_numel(n->out);
    const float *g = fptr(n->out->grad);
    if (!g) return;
    for (int i = 0; i < n->n_in; i++) {
        nc_tensor *t = n->in[i];
        if (!needs_grad(t)) continue;
        if (!grad_buf(t)) return;
        const int acc = grad_acc(t);
        float *gt = fptr(t->grad);
        if (!gt) return;
        const int rc = i == 0 ? nc_hip_dropout_bwd(count, dropout_p(n), (uint64_t)n->p.i[0], (uint64_t)n->p.i[1], nullptr, g, gt, acc, stream(ctx))
                              : nc_hip_unary_bwd(NC_HIP_UN_ADD_SCALAR, 0.0f, nullptr, nullptr, g, gt, count, acc, stream(ctx));
        if (!hip_layer_ok(ctx, rc, n->op->name)) return;
        wrote_dev(t->grad);
    }
}

static const OpDef op_dropout_seeded = {"dropout_seeded", 0, 0, dropout_shape, nullptr, dropout_fwd, dropout_bwd};

// ---- cross entropy of a product --------------------------------------------------------------------------------------
// inputs: x [.., D], weight [V, D], labels, then the bias where given.  p.i: the ignored label, sum, which gradients are saved (a bit
// each of x, weight, bias).  saved: those gradients of the loss, which the backward scales: 6 N V D operations in all, where a backward
// that took the products again would make it 8
struct VocabLoss {
    nc_tensor *t[3];  // x, weight, bias
    int64_t N, D, V;
    size_t at[3], bytes;  // of the saved gradients

    explicit VocabLoss(const nc_node *n) : t{n->in[0], n->in[1], n->n_in > 3 ? n->in[3] : nullptr}, at{}, bytes(0) {
        D = t[0]->shape[t[0]->ndim - 1], N = D ? nc_numel(t[0]) / D : 0, V = t[1]->shape[0];
        for (int i = 0; i < 3; i++) {
            at[i] = bytes;
            if (n->p.i[2] & (1 << i)) bytes += ((size_t)nc_numel(t[i]) * sizeof(float) + kDevAlign - 1) / kDevAlign * kDevAlign;
        }
    }
};

static nc_status vocab_loss_shape(nc_node *n, OutSpec &out) {
    const char *name = n->op->name;
    if (!inputs_f32(n, 0, 2) || (n->n_in > 3 && !inputs_f32(n, 3, 1))) return NC_ERR_DTYPE;
    if (n->in[2]->dtype != NC_I32) return reject(n, NC_ERR_DTYPE, "%s: labels must be i32", name);
    const Dims x = Dims::of(n->in[0]), w = Dims::of(n->in[1]), l = Dims::of(n->in[2]);
    bool ok = x.rank >= 1 && w.rank == 2 && x.back(0) == w.e[1] && w.e[0] >= 1 && w.e[1] >= 1 && l.rank == x.rank - 1;
    for (int i = 0; ok && i < l.rank; i++) ok = l.e[i] == x.e[i];
    char tx[96], tw[96], tl[96];
    if (!ok)
        return reject(n, NC_ERR_SHAPE, "%s: expected x [.., columns], weight [words, columns] and a label for each row of x, got %s, %s and %s",
                      name, x.text(tx, sizeof tx), w.text(tw, sizeof tw), l.text(tl, sizeof tl));
    if (n->n_in > 3 && (n->in[3]->ndim != 1 || n->in[3]->shape[0] != w.e[0]))
        return reject(n, NC_ERR_SHAPE, "%s: the bias needs %lld elements", name, (long long)w.e[0]);
    out.dims = Dims{};  // a 0-d loss
    return NC_OK;
}

static nc_status vocab_loss_fwd(nc_node *n) {
    nc_ctx *ctx = n->in[0]->ctx;
    n->p.i[2] = 0;
    if (ctx->grad_enabled && !persistent_mode(ctx))
        for (int i = 0; i < 3; i++) {
            const nc_tensor *t = i < 2 ? n->in[i] : n->n_in > 3 ? n->in[3] : nullptr;
            if (t && needs_grad(t)) n->p.i[2] |= 1 << i;
        }
    const VocabLoss c(n);
    Rows x, w;
    float *loss = fptr(n->out);
    if (!loss || !rows_of(c.t[0], x) || !rows_of(c.t[1], w)) return NC_ERR_STATE;
    const float *bias = c.t[2] ? contig_f32(c.t[2]) : nullptr;
    int32_t *labels = (int32_t *)arena_alloc(ctx, (size_t)(c.N ? c.N : 1) * sizeof(int32_t));
    if ((c.t[2] && !bias) || !labels || !copy_i32(n->in[2], labels, n->op->name)) return NC_ERR_STATE;
    float *g[3] = {};
    if (n->p.i[2]) {
        char *saved = (char *)save_state(n, c.bytes);
        if (!saved) return NC_ERR_STATE;
        for (int i = 0; i < 3; i++)
            if (n->p.i[2] & (1 << i)) g[i] = (float *)(saved + c.at[i]);
    }
    const size_t ws_bytes = nc_hip_linear_cross_entropy_workspace(c.N, c.D, c.V, g[0] != nullptr, g[1] != nullptr, g[2] != nullptr);
    char *ws = arena_alloc(ctx, ws_bytes ? ws_bytes : 1);
    IndexCheck check;
    if (!ws || !check.begin(ctx)) return NC_ERR_STATE;
    if (!hip_layer_ok(ctx,
                      nc_hip_linear_cross_entropy(c.N, c.D, c.V, x.p, x.ld, w.p, w.ld, bias, labels, (int32_t)n->p.i[0], (int)n->p.i[1],
                                                  nullptr, loss, nullptr, check.bad, g[0], g[1], g[2], 0, 0, 0, ws, ws_bytes, stream(ctx)),
                      n->op->name) ||
        !check.read(ctx, n->op->name))
        return NC_ERR_STATE;
    if (!check.ok()) {
        error(ctx, NC_ERR_ARG, "%s: label %d at row %lld outside [0, %lld)", n->op->name, check.value(), check.at(), (long long)c.V);
        return NC_ERR_ARG;
    }
    wrote_dev(n->out);
    return NC_OK;
}

static void vocab_loss_bwd(nc_node *n) {
    const VocabLoss c(n);
    nc_ctx *ctx = n->in[0]->ctx;
    const float *gout = fptr(n->out->grad);
    if (!gout) return;
    for (int i = 0; i < 3; i++) {
        nc_tensor *t = c.t[i];
        if (!t || !needs_grad(t)) continue;
        if (!(n->p.i[2] & (1 << i))) {
            error(ctx, NC_ERR_STATE, "%s: an input came to need a gradient after the forward (which takes the gradients)", n->op->name);
            return;
        }
        const int64_t count = nc_numel(t);
        if (!grad_buf(t)) return;
        if (count == 0) continue;
        const int acc = grad_acc(t);
        float *gt = fptr(t->grad);
        const float *saved = (const float *)((const char *)n->saved + c.at[i]);
        const int64_t one = 1, none = 0;
        if (!gt || !hip_layer_ok(ctx,
                                 nc_hip_binary_bwd(NC_HIP_BIN_MUL, 0, 1, &count, saved, &one, saved, &one, gout, &none, gt, &one, acc, nullptr, 0,
                                                   stream(ctx)),
                                 n->op->name))
            return;
        wrote_dev(t->grad);
    }
}

static const OpDef op_linear_cross_entropy = {"linear_cross_entropy", 0, 0, vocab_loss_shape, nullptr, vocab_loss_fwd, vocab_loss_bwd};

}  // namespace nce

using namespace nce;

extern "C" {
nc_tensor *nc_embedding(nc_tensor *weight, nc_tensor *tokens, float scale, int32_t padding) {
    nc_tensor *in[2] = {weight, tokens};
    Params p{};
    p.f[0] = scale;
    p.i[0] = padding;
    return apply(&op_embedding, in, 2, &p);
}

nc_tensor *nc_dropout_seeded(nc_tensor *x, nc_tensor *residual, double p, uint64_t seed, uint64_t offset) {
    nc_tensor *in[2] = {x, residual};
    Params q{};
    q.i[0] = (int64_t)seed, q.i[1] = (int64_t)offset;
    memcpy(&q.i[2], &p, sizeof p);
    return apply(&op_dropout_seeded, in, residual ? 2 : 1, &q);
}

nc_tensor *nc_linear_cross_entropy(nc_tensor *x, nc_tensor *weight, nc_tensor *bias, nc_tensor *labels, int32_t ignore, int sum) {
    nc_tensor *in[4] = {x, weight, labels, bias};
    Params p{};
    p.i[0] = ignore;
    p.i[1] = sum ? 1 : 0;
    return apply(&op_linear_cross_entropy, in, bias ? 4 : 3, &p);
}
}
