/*
 * mdx_paged.h — launchers of the paged cache's kernels (mdx_paged.hip).  The
 * arguments have been checked by the entry points of md_paged.c; pointers are
 * device pointers.  Every launcher returns 0 or a negative MatmulDecoderError
 * and never synchronises.
 */
#ifndef MDX_PAGED_H
#define MDX_PAGED_H

#include "mdx_ext.h"

#ifdef __cplusplus
extern "C" {
#endif

int mdx_launch_paged_append(const MdxPagedCache* c, const MdxPagedBatch* b, const float* qkv, long long qkv_stride,
                            const int* positions, const float* q_norm, const float* k_norm, float eps,
                            const float* cos_t, const float* sin_t, int max_pos, int rope_style, void* q_out,
                            long long q_stride, void* stream);

/* Bytes of the splits' partial results (0: no split). */
size_t mdx_paged_attn_scratch(const MdxPagedCache* c, const MdxPagedBatch* b);
int mdx_launch_paged_attn(const MdxPagedCache* c, const MdxPagedBatch* b, const void* q, long long q_stride,
                          float scale, void* out, long long out_stride, float* lse, void* scratch, void* stream);

size_t mdx_paged_mass_scratch(const MdxPagedCache* c, const MdxPagedBatch* b);
int mdx_launch_paged_mass(const MdxPagedCache* c, const MdxPagedBatch* b, const void* q, long long q_stride,
                          float scale, const float* lse, void* scratch, void* stream);

size_t mdx_paged_evict_scratch(const MdxPagedCache* c, const MdxPagedBatch* b, int budget);
int mdx_launch_paged_evict(const MdxPagedCache* c, const MdxPagedBatch* b, int budget, int sink, int recent,
                           float* mass_out, int* pos_out, void* scratch, void* stream);

#ifdef __cplusplus
}
#endif

#endif
