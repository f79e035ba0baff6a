// C ABI of the paged cache and the drafted trees: argument checks and
// dispatch.  See include/affon_b200.h.
#include <cstdarg>
#include <cstdio>

#include "../../include/affon_b200.h"
#include "internal.h"

namespace {

int fail(int status, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int status, const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return afb::set_error(status, buf);
}

bool al16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_desc(const affon_b200_paged_desc *d, afb::PagedShape *s) {
    if (!d || d->struct_size != sizeof(affon_b200_paged_desc))
        return fail(AFFON_B200_INVALID_ARG, "paged: null or bad descriptor");
    if (d->seqs < 1 || d->seqs > 65536) return fail(AFFON_B200_INVALID_SHAPE, "paged: seqs must be 1 to 65536");
    if (d->rows < 0) return fail(AFFON_B200_INVALID_SHAPE, "paged: rows must not be negative");
    if (d->max_nodes < 1 || d->max_nodes > afb::kMaxTreeNodes)
        return fail(AFFON_B200_INVALID_SHAPE, "paged: max_nodes must be 1 to %d", afb::kMaxTreeNodes);
    if (d->kv_heads < 1 || d->kv_heads > 1024) return fail(AFFON_B200_INVALID_SHAPE, "paged: kv_heads must be 1 to 1024");
    if (d->head_dim != 64 && d->head_dim != 128)
        return fail(AFFON_B200_UNSUPPORTED, "paged: head_dim must be 64 or 128");
    int shift = 4;
    while (shift <= 8 && (1 << shift) != d->page_size) ++shift;
    if (shift > 8) return fail(AFFON_B200_UNSUPPORTED, "paged: page_size must be 16, 32, 64, 128 or 256");
    if (d->mask_words > 8 || d->mask_words * 32 < d->max_nodes)
        return fail(AFFON_B200_INVALID_SHAPE, "paged: mask_words must cover max_nodes bits, at most 8");
    const int64_t lim = int64_t(1) << 31;
    if (d->pages < 1 || d->pages > (lim - 1) / d->page_size)
        return fail(AFFON_B200_INVALID_SHAPE, "paged: pages must be positive, pages * page_size below 2^31");
    if (d->ld_table < 1 || d->ld_table > (lim / 2 - 1) / d->page_size)
        return fail(AFFON_B200_INVALID_SHAPE, "paged: ld_table must be positive, ld_table * page_size below 2^30");
    // A stride of a one-element axis is never used.
    *s = afb::PagedShape{d->seqs,  d->rows,        d->max_nodes,   d->kv_heads,     d->head_dim, shift, d->mask_words,
                         d->pages, d->page_stride, d->head_stride, d->token_stride, d->ld_table};
    if (d->kv_heads == 1) s->head_stride = d->head_dim;
    if (d->pages == 1) s->page_stride = d->head_dim;
    const int64_t st[3] = {s->page_stride, s->head_stride, s->token_stride};
    for (int64_t v : st)
        if (v < d->head_dim || v % 8 || v >= (int64_t(1) << 39))
            return fail(AFFON_B200_INVALID_SHAPE, "paged: cache strides must be multiples of 8 elements, at least "
                                                  "head_dim and below 2^39");
    return AFFON_B200_OK;
}

int check_launch(affon_b200_ctx *ctx, const char *what, const afb::DeviceGuard &guard) {
    if (!ctx->workspace)  // its growth failed: the status word and the counters have no place
        return fail(AFFON_B200_UNSUPPORTED, "%s: the context has no workspace", what);
    if (!guard.ok) return fail(AFFON_B200_CUDA_ERROR, "%s: cudaSetDevice(%d) failed", what, ctx->device);
    return AFFON_B200_OK;
}

}  // namespace

extern "C" {

int affon_b200_paged_validate(const affon_b200_paged_desc *desc) {
    afb::clear_error();
    afb::PagedShape s;
    return check_desc(desc, &s);
}

int affon_b200_paged_plan(affon_b200_ctx *ctx, const affon_b200_paged_desc *desc, const int *cu_nodes,
                          const int *parents, const int *ctx_lens, const int *page_table, int *positions, int *slots,
                          uint32_t *mask) {
    afb::clear_error();
    afb::PagedShape s;
    if (int rc = check_desc(desc, &s)) return rc;
    if (!ctx) return fail(AFFON_B200_INVALID_ARG, "paged_plan: null context");
    if (s.rows == 0) return AFFON_B200_OK;
    if (!cu_nodes || !ctx_lens || !page_table || !positions || !slots || !mask)
        return fail(AFFON_B200_INVALID_ARG, "paged_plan: null buffer");
    afb::DeviceGuard guard(ctx->device);
    if (int rc = check_launch(ctx, "paged_plan", guard)) return rc;
    const cudaError_t e = afb::launch_paged_plan(s, {cu_nodes, parents, ctx_lens, page_table}, positions, slots, mask,
                                                 ctx->workspace, ctx->stream, ctx->overlap);
    return e == cudaSuccess ? AFFON_B200_OK : afb::set_cuda_error(e, "paged_plan launch");
}

int affon_b200_paged_append(affon_b200_ctx *ctx, const affon_b200_paged_desc *desc, const affon_b200_append_desc *d,
                            const void *qkv, const float *rope_cos, const float *rope_sin, const int *positions,
                            const int *slots, void *q_out, void *k_cache, void *v_cache) {
    afb::clear_error();
    afb::PagedShape s;
    if (int rc = check_desc(desc, &s)) return rc;
    if (!ctx || !d || d->struct_size != sizeof(affon_b200_append_desc))
        return fail(AFFON_B200_INVALID_ARG, "paged_append: null context or bad descriptor");
    if (d->x_dtype != AFFON_B200_F32 && d->x_dtype != AFFON_B200_BF16)
        return fail(AFFON_B200_INVALID_DTYPE, "paged_append: qkv must be f32 or bf16");
    if (d->rope < 0 || d->rope > 2) return fail(AFFON_B200_INVALID_ARG, "paged_append: unknown rotation %d", d->rope);
    if (d->q_heads < 0 || d->q_heads > 65536) return fail(AFFON_B200_INVALID_SHAPE, "paged_append: bad q_heads");
    const int64_t q_cols = int64_t(d->q_heads) * s.head_dim, kv_cols = int64_t(s.kv_heads) * s.head_dim;
    const int64_t per = d->x_dtype == AFFON_B200_F32 ? 4 : 8;  // elements of 16 bytes
    const int64_t begin[3] = {d->q_offset, d->k_offset, d->v_offset}, cols[3] = {q_cols, kv_cols, kv_cols};
    for (int i = d->q_heads ? 0 : 1; i < 3; ++i)
        if (begin[i] < 0 || begin[i] % per || begin[i] + cols[i] > d->ld_qkv || begin[i] + cols[i] > 0x7FFFFFFF)
            return fail(AFFON_B200_INVALID_SHAPE, "paged_append: query, key and value columns must be 16-byte aligned "
                                                  "and lie inside a row of qkv, before its column 2^31");
    if (d->ld_qkv % per) return fail(AFFON_B200_INVALID_SHAPE, "paged_append: rows of qkv must be 16-byte aligned");
    if (d->q_heads && (d->ld_q < q_cols || d->ld_q % 8))
        return fail(AFFON_B200_INVALID_SHAPE, "paged_append: ld_q must be a multiple of 8 and hold q_heads heads");
    if (d->rope && d->table_rows < 1) return fail(AFFON_B200_INVALID_SHAPE, "paged_append: empty rotation tables");
    if (s.rows == 0) return AFFON_B200_OK;
    if (!qkv || !slots || !k_cache || !v_cache || (d->q_heads && !q_out) ||
        (d->rope && (!rope_cos || !rope_sin || !positions)))
        return fail(AFFON_B200_INVALID_ARG, "paged_append: null buffer");
    if (!al16(qkv) || !al16(q_out) || !al16(k_cache) || !al16(v_cache) || !al16(rope_cos) || !al16(rope_sin))
        return fail(AFFON_B200_INVALID_ARG, "paged_append: buffers must be 16-byte aligned");
    afb::AppendArgs a{};
    a.qkv = qkv;
    a.cos_t = rope_cos;
    a.sin_t = rope_sin;
    a.positions = positions;
    a.slots = slots;
    a.q_out = static_cast<uint16_t *>(q_out);
    a.k_cache = static_cast<uint16_t *>(k_cache);
    a.v_cache = static_cast<uint16_t *>(v_cache);
    a.x_f32 = d->x_dtype == AFFON_B200_F32;
    a.rope = d->rope;
    a.q_heads = d->q_heads;
    a.q_off = d->q_offset;
    a.k_off = d->k_offset;
    a.v_off = d->v_offset;
    a.table_rows = d->table_rows;
    a.ld_qkv = d->ld_qkv;
    a.ld_q = d->ld_q;
    afb::DeviceGuard guard(ctx->device);
    if (int rc = check_launch(ctx, "paged_append", guard)) return rc;
    const cudaError_t e = afb::launch_paged_append(s, a, ctx->workspace, ctx->stream, ctx->overlap);
    return e == cudaSuccess ? AFFON_B200_OK : afb::set_cuda_error(e, "paged_append launch");
}

int affon_b200_tree_attention(affon_b200_ctx *ctx, const affon_b200_paged_desc *desc,
                              const affon_b200_tree_attn_desc *d, const void *q, const int *cu_nodes,
                              const int *ctx_lens, const int *page_table, const uint32_t *mask, const void *k_cache,
                              const void *v_cache, void *out) {
    afb::clear_error();
    afb::PagedShape s;
    if (int rc = check_desc(desc, &s)) return rc;
    if (!ctx || !d || d->struct_size != sizeof(affon_b200_tree_attn_desc))
        return fail(AFFON_B200_INVALID_ARG, "tree_attention: null context or bad descriptor");
    if (d->q_heads < 1 || d->q_heads > 65536 || d->q_heads % s.kv_heads)
        return fail(AFFON_B200_INVALID_SHAPE, "tree_attention: q_heads must be a multiple of kv_heads, at most 65536");
    if (!(d->scale > -2.0e38f && d->scale < 2.0e38f) || d->scale == 0.0f)  // scale * log2(e) is finite, too
        return fail(AFFON_B200_INVALID_ARG, "tree_attention: scale must be below 2e38 in magnitude and not zero");
    const int64_t cols = int64_t(d->q_heads) * s.head_dim;
    if (d->ld_q < cols || d->ld_out < cols || d->ld_q % 8 || d->ld_out % 8)
        return fail(AFFON_B200_INVALID_SHAPE, "tree_attention: ld_q and ld_out must be multiples of 8 and hold q_heads "
                                              "heads");
    if (s.rows == 0) return AFFON_B200_OK;
    if (!q || !cu_nodes || !ctx_lens || !page_table || !k_cache || !v_cache || !out)
        return fail(AFFON_B200_INVALID_ARG, "tree_attention: null buffer");
    if (!al16(q) || !al16(k_cache) || !al16(v_cache) || !al16(out))
        return fail(AFFON_B200_INVALID_ARG, "tree_attention: buffers must be 16-byte aligned");
    if (afb::tree_attention_workspace_bytes(s.head_dim, ctx->num_sms) > ctx->workspace_bytes)
        return fail(AFFON_B200_UNSUPPORTED, "tree_attention: partial results exceed the context workspace");
    afb::TreeAttnArgs a{};
    a.q = static_cast<const uint16_t *>(q);
    a.k_cache = static_cast<const uint16_t *>(k_cache);
    a.v_cache = static_cast<const uint16_t *>(v_cache);
    a.out = static_cast<uint16_t *>(out);
    a.mask = mask;
    a.q_heads = d->q_heads;
    a.out_pair_order = d->out_pair_order;
    a.scale = d->scale;
    a.ld_q = d->ld_q;
    a.ld_out = d->ld_out;
    afb::DeviceGuard guard(ctx->device);
    if (int rc = check_launch(ctx, "tree_attention", guard)) return rc;
    const cudaError_t e = afb::launch_tree_attention(s, {cu_nodes, nullptr, ctx_lens, page_table}, a, ctx->workspace,
                                                     ctx->num_sms, ctx->stream, ctx->overlap);
    return e == cudaSuccess ? AFFON_B200_OK : afb::set_cuda_error(e, "tree_attention launch");
}

int affon_b200_tree_accept(affon_b200_ctx *ctx, const affon_b200_paged_desc *desc, int layers, int64_t layer_stride,
                           const int *cu_nodes, const int *parents, const int *tokens, const int *predicted,
                           const int *page_table, const int *ctx_lens, void *k_cache, void *v_cache, int *counts,
                           int *path, int64_t ld_path, int *next_tokens, int *lens_out) {
    afb::clear_error();
    afb::PagedShape s;
    if (int rc = check_desc(desc, &s)) return rc;
    if (!ctx) return fail(AFFON_B200_INVALID_ARG, "tree_accept: null context");
    if (layers < 0 || layers > 65536 || (layers > 1 && (layer_stride < s.head_dim || layer_stride % 8)))
        return fail(AFFON_B200_INVALID_SHAPE, "tree_accept: layers must be 0 to 65536, layer_stride a multiple of 8 "
                                              "elements and at least head_dim");
    if (ld_path < s.max_nodes) return fail(AFFON_B200_INVALID_SHAPE, "tree_accept: ld_path must hold max_nodes entries");
    if (!cu_nodes || !page_table || !ctx_lens || !counts || !path || !next_tokens || !lens_out ||
        (s.rows && (!tokens || !predicted)) || (layers && (!k_cache || !v_cache)))
        return fail(AFFON_B200_INVALID_ARG, "tree_accept: null buffer");
    if (layers && (!al16(k_cache) || !al16(v_cache)))
        return fail(AFFON_B200_INVALID_ARG, "tree_accept: caches must be 16-byte aligned");
    const afb::AcceptArgs a{tokens,  predicted, static_cast<uint16_t *>(k_cache), static_cast<uint16_t *>(v_cache),
                            layers,  layer_stride, ld_path, counts, path, next_tokens, lens_out};
    afb::DeviceGuard guard(ctx->device);
    if (int rc = check_launch(ctx, "tree_accept", guard)) return rc;
    const cudaError_t e = afb::launch_tree_accept(s, {cu_nodes, parents, ctx_lens, page_table}, a, ctx->workspace,
                                                  ctx->stream, ctx->overlap);
    return e == cudaSuccess ? AFFON_B200_OK : afb::set_cuda_error(e, "tree_accept launch");
}

}  // extern "C"
