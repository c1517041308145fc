/*
 * md_paged.c — the entry points of the paged K/V cache (mdx_ext.h): checks of
 * the arguments, then the launch.  Nothing here touches the device before every
 * argument has been checked.
 */
#include <math.h>
#include <stdio.h>

#include "md_internal.h"
#include "mdx_paged.h"

static int refuse(int rc, const char* fn, const char* what) {
    char msg[200];
    snprintf(msg, sizeof msg, "%s: %s", fn, what);
    return mdxrt_refuse(rc, msg);
}
#define REFUSE_IF(cond, what) \
    if (cond) return refuse(MATMUL_DECODER_ERR_INVALID_ARG, fn, what)

static int misaligned(const void* p, size_t n) { return (uintptr_t)p % n != 0; }

static int check_cache(const MdxPagedCache* c, const char* fn) {
    REFUSE_IF(!c, "no cache");
    REFUSE_IF(c->type != MDX_TYPE_F16 && c->type != MDX_TYPE_BF16, "unknown type");
    REFUSE_IF(c->num_kv_heads < 1 || c->num_q_heads < 1 || c->num_q_heads % c->num_kv_heads,
              "num_q_heads has to be a multiple of num_kv_heads");
    REFUSE_IF(c->num_q_heads > 16384, "too many heads");
    REFUSE_IF(c->n_pages < 1 || !c->k_pages || !c->v_pages, "no pages");
    REFUSE_IF(misaligned(c->k_pages, 16) || misaligned(c->v_pages, 16), "pages have to be 16-byte aligned");
    REFUSE_IF(misaligned(c->mass, 16) || misaligned(c->pos, 16), "mass and pos have to be 16-byte aligned");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return refuse(MATMUL_DECODER_ERR_UNSUPPORTED, fn, "head_dim has to be 64, 128 or 256");
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return refuse(MATMUL_DECODER_ERR_UNSUPPORTED, fn, "page_size has to be a power of two from 16 to 1024");
    return 0;
}

/* `rows`: the call reads the new rows (q_start, n_tokens, max_q_len).  Kernels count a
 * request's cache rows, rounded up to whole tiles, in 32 bits. */
static int check_batch(const MdxPagedCache* c, const MdxPagedBatch* b, int rows, const char* fn) {
    REFUSE_IF(!b, "no batch");
    REFUSE_IF(b->n_req < 0 || b->n_req > 65535, "n_req has to be 0 to 65535");
    if (b->n_req == 0) return 0;
    REFUSE_IF(b->max_kv_len < 0 || b->max_pages < 0, "negative max_kv_len or max_pages");
    REFUSE_IF(b->max_kv_len > 1 << 29 && (long long)b->max_pages * c->page_size > 1 << 29,
              "a request has 2^29 cache rows at most");
    REFUSE_IF(!b->kv_len || !b->block_table, "no kv_len or block_table");
    REFUSE_IF(misaligned(b->kv_len, 4) || misaligned(b->block_table, 4) || misaligned(b->q_start, 4),
              "lengths and tables have to be 4-byte aligned");
    if (!rows) return 0;
    REFUSE_IF(b->n_tokens < 0 || b->max_q_len < 0, "negative n_tokens or max_q_len");
    REFUSE_IF(!b->q_start, "no q_start");
    return 0;
}

static int check_rows(const MdxPagedCache* c, const void* p, long long stride, const char* fn, const char* what) {
    REFUSE_IF(!p, what);
    REFUSE_IF(misaligned(p, 16), "rows have to be 16-byte aligned");
    REFUSE_IF(stride < (long long)c->num_q_heads * c->head_dim || stride % 8,
              "a row's stride has to hold its heads and be a multiple of 8 values");
    return 0;
}

/* a scale of 0 is 1 / sqrt(head_dim) */
static int check_scale(float scale, const char* fn) {
    REFUSE_IF(scale != 0.0f && !(scale >= 1.2e-38f && scale <= 1e30f),
              "scale has to be 1.2e-38 to 1e30, or 0 for 1 / sqrt(head_dim)");
    return 0;
}
static float scale_of(const MdxPagedCache* c, float scale) {
    return scale > 0.0f ? scale : 1.0f / sqrtf((float)c->head_dim);
}

static int check_workspace(const void* ws, size_t have, size_t need, const char* fn) {
    REFUSE_IF(have < need || (need && !ws), "the workspace is too small");
    REFUSE_IF(need && misaligned(ws, 16), "the workspace has to be 16-byte aligned");
    return 0;
}

int mdx_paged_append(const MdxPagedCache* c, const MdxPagedBatch* b, const float* qkv, long long qkv_stride,
                     const int* positions, const float* q_norm, const float* k_norm, float eps,
                     const float* cos_t, const float* sin_t, int max_pos, int rope_style, void* q_out,
                     long long q_stride, void* stream) {
    static const char fn[] = "mdx_paged_append";
    int rc = check_cache(c, fn);
    if (!rc) rc = check_batch(c, b, 1, fn);
    if (rc || b->n_req == 0 || b->n_tokens == 0) return rc;
    REFUSE_IF(!qkv || misaligned(qkv, 16), "qkv has to be there and 16-byte aligned");
    REFUSE_IF(qkv_stride < ((long long)c->num_q_heads + 2LL * c->num_kv_heads) * c->head_dim || qkv_stride % 4,
              "qkv_stride has to hold the heads and be a multiple of 4 floats");
    REFUSE_IF(!positions || misaligned(positions, 4), "no positions");
    REFUSE_IF(!cos_t || !sin_t || misaligned(cos_t, 16) || misaligned(sin_t, 16),
              "the tables have to be there and 16-byte aligned");
    REFUSE_IF(misaligned(q_norm, 16) || misaligned(k_norm, 16), "norms have to be 16-byte aligned");
    REFUSE_IF(max_pos < 1, "max_pos has to be positive");
    REFUSE_IF(rope_style != 0 && rope_style != 1, "rope_style has to be 0 or 1");
    REFUSE_IF(!(eps >= 0.0f) || isinf(eps), "eps has to be finite and not negative");
    rc = check_rows(c, q_out, q_stride, fn, "no q_out");
    if (rc) return rc;
    return mdx_launch_paged_append(c, b, qkv, qkv_stride, positions, q_norm, k_norm, eps, cos_t, sin_t, max_pos,
                                   rope_style, q_out, q_stride, stream);
}

size_t mdx_paged_attention_workspace(const MdxPagedCache* c, const MdxPagedBatch* b) {
    static const char fn[] = "mdx_paged_attention_workspace";
    if (check_cache(c, fn) || check_batch(c, b, 1, fn) || b->n_req == 0 || b->n_tokens == 0) return 0;
    return mdx_paged_attn_scratch(c, b);
}

int mdx_paged_attention(const MdxPagedCache* c, const MdxPagedBatch* b, const void* q, long long q_stride,
                        float scale, void* out, long long out_stride, float* lse, void* workspace,
                        size_t workspace_bytes, void* stream) {
    static const char fn[] = "mdx_paged_attention";
    int rc = check_cache(c, fn);
    if (!rc) rc = check_batch(c, b, 1, fn);
    if (!rc) rc = check_scale(scale, fn);
    if (rc || b->n_req == 0 || b->n_tokens == 0) return rc;
    rc = check_rows(c, q, q_stride, fn, "no q");
    if (!rc) rc = check_rows(c, out, out_stride, fn, "no out");
    if (!rc) rc = check_workspace(workspace, workspace_bytes, mdx_paged_attn_scratch(c, b), fn);
    if (rc) return rc;
    REFUSE_IF(q == out, "out has to be apart from q");
    REFUSE_IF(misaligned(lse, 4), "lse has to be 4-byte aligned");
    return mdx_launch_paged_attn(c, b, q, q_stride, scale_of(c, scale), out, out_stride, lse, workspace, stream);
}

size_t mdx_paged_mass_workspace(const MdxPagedCache* c, const MdxPagedBatch* b) {
    static const char fn[] = "mdx_paged_mass_workspace";
    if (check_cache(c, fn) || check_batch(c, b, 1, fn) || b->n_req == 0 || b->n_tokens == 0) return 0;
    return mdx_paged_mass_scratch(c, b);
}

int mdx_paged_mass(const MdxPagedCache* c, const MdxPagedBatch* b, const void* q, long long q_stride, float scale,
                   const float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    static const char fn[] = "mdx_paged_mass";
    int rc = check_cache(c, fn);
    if (!rc) rc = check_batch(c, b, 1, fn);
    if (!rc) rc = check_scale(scale, fn);
    if (rc) return rc;
    REFUSE_IF(!c->mass, "the cache keeps no mass");
    if (b->n_req == 0 || b->n_tokens == 0) return 0;
    rc = check_rows(c, q, q_stride, fn, "no q");
    if (!rc) rc = check_workspace(workspace, workspace_bytes, mdx_paged_mass_scratch(c, b), fn);
    if (rc) return rc;
    REFUSE_IF(!lse || misaligned(lse, 4), "lse has to be there and 4-byte aligned");
    return mdx_launch_paged_mass(c, b, q, q_stride, scale_of(c, scale), lse, workspace, stream);
}

size_t mdx_paged_evict_workspace(const MdxPagedCache* c, const MdxPagedBatch* b, int budget) {
    static const char fn[] = "mdx_paged_evict_workspace";
    if (check_cache(c, fn) || check_batch(c, b, 0, fn) || b->n_req == 0 || budget < 0) return 0;
    return mdx_paged_evict_scratch(c, b, budget);
}

int mdx_paged_evict(const MdxPagedCache* c, const MdxPagedBatch* b, int budget, int sink, int recent,
                    float* mass_out, int* pos_out, void* workspace, size_t workspace_bytes, void* stream) {
    static const char fn[] = "mdx_paged_evict";
    int rc = check_cache(c, fn);
    if (!rc) rc = check_batch(c, b, 0, fn);
    if (rc) return rc;
    REFUSE_IF(!c->mass || !c->pos, "the cache keeps no mass or no pos");
    REFUSE_IF(budget < 0 || sink < 0 || recent < 0 || (long long)sink + recent > budget,
              "sink + recent have to fit the budget");
    REFUSE_IF(!mass_out || !pos_out || misaligned(mass_out, 4) || misaligned(pos_out, 4),
              "mass_out and pos_out have to be there and 4-byte aligned");
    if (b->n_req == 0) return 0;
    rc = check_workspace(workspace, workspace_bytes, mdx_paged_evict_scratch(c, b, budget), fn);
    if (rc) return rc;
    return mdx_launch_paged_evict(c, b, budget, sink, recent, mass_out, pos_out, workspace, stream);
}
