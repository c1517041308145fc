// mdx_paged.hip — a K/V cache in pages that many requests share: append of the
// new rows (QK-norm + RoPE), attention over the pages, the weight that cached
// rows receive, and eviction by it; gfx950.
//
// Pages are [n_pages][nkv][page][hd], so that a KV head's rows within a page
// are contiguous.  Row i of a request's n new rows is cache row L - n + i.
#include <hip/hip_runtime.h>

#include <cmath>

#include "mdx_common.h"
#include "mdx_device.h"
#include "mdx_paged.h"

using namespace mdx;

namespace {

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }
// a / b up to a multiple of 4
__device__ __forceinline__ int cdiv4(int a, int b) { return ((a - 1) / b / 4 + 1) * 4; }

// The cache and the batch as the kernels take them.
struct Paged {
    uint16_t* kp;
    uint16_t* vp;
    float* mass;
    int* pos;
    const int* q_start;
    const int* kv_len;
    const int* table;
    int n_req, n_tokens, max_q, max_pages, n_pages;
    int nq, nkv, G, shift;     // page size 1 << shift
    int limit;                 // cache rows that exist: min(max_kv_len, max_pages * page)
};

Paged paged(const MdxPagedCache* c, const MdxPagedBatch* b) {
    Paged p = {};
    p.kp = (uint16_t*)c->k_pages;
    p.vp = (uint16_t*)c->v_pages;
    p.mass = c->mass;
    p.pos = c->pos;
    p.q_start = b->q_start;
    p.kv_len = b->kv_len;
    p.table = b->block_table;
    p.n_req = b->n_req;
    p.n_tokens = b->n_tokens;
    p.max_q = b->max_q_len;
    p.max_pages = b->max_pages;
    p.n_pages = c->n_pages;
    p.nq = c->num_q_heads;
    p.nkv = c->num_kv_heads;
    p.G = c->num_q_heads / c->num_kv_heads;
    p.shift = __builtin_ctz((unsigned)c->page_size);
    const long long rows = (long long)b->max_pages * c->page_size;
    p.limit = rows < b->max_kv_len ? (int)rows : b->max_kv_len;
    return p;
}

// A value of the batch's arrays, which no kernel writes, by a scalar load (the
// compiler takes a vector load where the address is one that could be stored to).
__device__ __forceinline__ int fixed(const int* a, size_t i) {
    typedef __attribute__((address_space(4))) const int c_int;
    return ((c_int*)a)[i];
}

// A request's new rows: [start, start + n) of the batch; base: the cache row of
// the first (negative if the cache is shorter than they are).
struct Req {
    int start, n, base;
};
__device__ __forceinline__ Req req_of(const Paged& p, int r) {
    Req q;
    q.start = min(max(fixed(p.q_start, r), 0), p.n_tokens);
    q.n = max(min(fixed(p.q_start, r + 1), p.n_tokens) - q.start, 0);
    q.base = max(fixed(p.kv_len, r), 0) - q.n;
    return q;
}

// Sum over the wave, the same in a scalar register.
__device__ __forceinline__ int wave_total(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return __builtin_amdgcn_readfirstlane(v);
}

// The request of batch row t, by a whole wave: how many requests end at or
// before it (n_req: the row is behind the last one).
__device__ __forceinline__ int find_req(const Paged& p, int t, int lane) {
    int r = 0;
    for (int j = 0; j < p.n_req; j += 64)
        r += __popcll(__ballot(j + lane < p.n_req && p.q_start[min(j + lane, p.n_req - 1) + 1] <= t));
    return r;
}

// Row number (of the pool, for one head) of cache row j, or -1.
__device__ __forceinline__ long long pool_row(const Paged& p, int r, int h, int j) {
    const int pg = p.table[(size_t)r * p.max_pages + (j >> p.shift)];
    if ((unsigned)pg >= (unsigned)p.n_pages) return -1;
    return ((((long long)pg * p.nkv + h) << p.shift)) + (j & ((1 << p.shift) - 1));
}

template <class T>
__device__ __forceinline__ uint16_t bits16(float f) {
    return __builtin_bit_cast(uint16_t, (T)f);
}
template <class T>
__device__ __forceinline__ float widen16(uint16_t b) {
    return (float)__builtin_bit_cast(T, b);
}
template <class T>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    typedef T t2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t{a, b}), t2_t));
}

__device__ __forceinline__ float4_t mfma16(_Float16, u32x4_t a, u32x4_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                  0, 0);
}
__device__ __forceinline__ float4_t mfma16(__bf16, u32x4_t a, u32x4_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0,
                                                   0);
}

// ---- append -----------------------------------------------------------------------
//
// One workgroup per new row; HD/4 lanes per head, four values each, so that a
// head is read with 16-byte loads, its sum of squares is a few cross-lane adds
// and a rotation's partner is in this lane (pairs) or HD/8 lanes away (halves).
// Reads and writes are all it does: 4 + 2 bytes per value; four rounds of loads are
// issued before the request is looked up (4096 rows of 16 + 2 x 8 heads of 128: 24.0
// us, 4.3 TB/s, where a large copy reaches 4.7; looked up first 25.5).  One row is the
// latency of two loads and a launch: 7.9 us with the host's part.
struct AppendArgs {
    Paged p;
    const float* qkv;
    long long qkv_stride;
    const int* positions;
    const float* q_norm;
    const float* k_norm;
    float eps;
    const float* cos_t;
    const float* sin_t;
    int max_pos, style;
    uint16_t* q_out;
    long long q_stride;
};

template <int HD, class T>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
    constexpr int LPH = HD / 4, HPB = 256 / LPH;   // lanes per head, heads per round
    constexpr int AHEAD = 4;                        // rounds whose loads are issued together
    const Paged& p = a.p;
    const int t = blockIdx.x, lane = threadIdx.x & 63;
    const int l = threadIdx.x % LPH, heads = p.nq + 2 * p.nkv;
    const float* row = a.qkv + (size_t)t * a.qkv_stride;
    float4 v[AHEAD];
    auto load = [&](int h0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            v[i] = *reinterpret_cast<const float4*>(row + (size_t)min(h0 + HPB * i + (int)threadIdx.x / LPH, heads - 1) * HD + 4 * l);
    };
    // the row itself depends on nothing that has to be looked up first
    load(0);
    const int pos = fixed(a.positions, t);
    const int r = find_req(p, t, lane);
    if (r >= p.n_req) return;
    const Req q = req_of(p, r);
    const int i = t - q.start;
    if (i < 0 || i >= min(q.n, p.max_q) || pos < 0 || pos >= a.max_pos) return;
    const int j = q.base + i;              // cache row
    const long long slot = j >= 0 && j < p.limit ? pool_row(p, r, 0, j) : -1;
    // this lane's part of the tables: for pairs its two, for halves the four it shares
    const size_t at = (size_t)pos * (HD / 2) + (a.style == 0 ? 2 * l : 4 * (l % (LPH / 2)));
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f), s = c;
    if (a.style == 0) {
        const float2 c2 = *reinterpret_cast<const float2*>(a.cos_t + at), s2 = *reinterpret_cast<const float2*>(a.sin_t + at);
        c.x = c2.x;
        c.y = c2.y;
        s.x = s2.x;
        s.y = s2.y;
    } else {
        c = *reinterpret_cast<const float4*>(a.cos_t + at);
        s = *reinterpret_cast<const float4*>(a.sin_t + at);
        if (l < LPH / 2) s = make_float4(-s.x, -s.y, -s.z, -s.w);
    }
    for (int h0 = 0; h0 < heads; h0 += HPB * AHEAD) {
        if (h0 > 0) load(h0);
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int h = h0 + HPB * i + threadIdx.x / LPH;
            if (h0 + HPB * i >= heads) break;
            float4 x = v[i];
            const float* nw = h < p.nq ? a.q_norm : a.k_norm;
            const bool turn = h < p.nq + p.nkv;
            float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
            ss = group_sum(ss, LPH);
            if (turn && nw) {
                const float rms = 1.0f / sqrtf(ss / (float)HD + a.eps);
                const float4 w = *reinterpret_cast<const float4*>(nw + 4 * l);
                x.x = (x.x * rms) * w.x;
                x.y = (x.y * rms) * w.y;
                x.z = (x.z * rms) * w.z;
                x.w = (x.w * rms) * w.w;
            }
            if (a.style == 0) {
                if (turn)
                    x = make_float4(x.x * c.x - x.y * s.x, x.y * c.x + x.x * s.x, x.z * c.y - x.w * s.y,
                                    x.w * c.y + x.z * s.y);
            } else {
                float4 y;
                y.x = __shfl_xor(x.x, LPH / 2, kWave);
                y.y = __shfl_xor(x.y, LPH / 2, kWave);
                y.z = __shfl_xor(x.z, LPH / 2, kWave);
                y.w = __shfl_xor(x.w, LPH / 2, kWave);
                if (turn)
                    x = make_float4(x.x * c.x + y.x * s.x, x.y * c.y + y.y * s.y, x.z * c.z + y.z * s.z,
                                    x.w * c.w + y.w * s.w);
            }
            if (h >= heads) continue;
            const uint2 o = make_uint2(pack16<T>(x.x, x.y), pack16<T>(x.z, x.w));
            if (h < p.nq) {
                *reinterpret_cast<uint2*>(a.q_out + (size_t)t * a.q_stride + (size_t)h * HD + 4 * l) = o;
            } else if (slot >= 0) {
                const bool is_k = h < p.nq + p.nkv;
                const long long to = slot + ((long long)(is_k ? h - p.nq : h - p.nq - p.nkv) << p.shift);
                *reinterpret_cast<uint2*>((is_k ? p.kp : p.vp) + to * HD + 4 * l) = o;
                if (is_k && l == 0) {
                    if (p.mass) p.mass[to] = 0.0f;
                    if (p.pos) p.pos[to] = pos;
                }
            }
        }
    }
}

// ---- attention ----------------------------------------------------------------------
//
// A workgroup takes 16 query rows (new rows x the heads of one KV head's group)
// and a split of the keys; its waves take alternate tiles of 32 keys, each with
// a running maximum and sum of its own, and are joined through LDS; splits are
// joined by a second kernel.  K and V go from the pages into registers as the
// matrix operands, without LDS:
//   S^T = K . Q^T      lane (g, c): key row c of 16, dims 32s + 8g ..
//   O^T = V^T . P^T    lane (g, c): 8 keys x the dims (HD/16) c .., transposed
//                      in registers by v_perm; the k order is that in which S^T
//                      leaves a lane's keys (4g + i, 16 + 4g + i), and product
//                      j has the dims (HD/16) m + j, so a lane's outputs of all
//                      products are contiguous.
// Probabilities enter as the sum of two 16-bit values (22 bits in fp16, 16 in
// bf16): the keys' bytes bound this kernel, not its products.  64 requests of 4096
// rows, 8 heads of 128: 140 us, 5.0 TB/s; one of 131072: 101 us, 5.3 TB/s, with the
// join.  (A wave that requests its next tile ahead gains nothing: 138.0 us for 137.4,
// and 9.2 for 8.8 over 512 rows.)
//
// Rows and their order: masks are -inf scores; V rows that no row of the tile
// sees are zeroed as they are loaded.  What is left of a non-finite V value at a
// masked place would be 0 * inf; outputs that are not finite therefore make the
// wave run again with every tile checked, and tiles that hold such values take
// the products of visible keys alone, in fp32.
constexpr int kShort = 32;             // query rows up to which k_paged_attn takes a request
constexpr int kRows = 128;             // query rows per block of k_paged_chunk

struct AttnArgs {
    Paged p;
    const uint16_t* q;
    long long q_stride;
    float scale, c;            // c: scale * log2 e
    uint16_t* out;
    long long out_stride;
    float* lse;
    // partial results of splits: unnormalised outputs; reference score and sum
    float* short_o;            // k_paged_attn: [splits][n_req][nkv][short_rows][hd]
    float2* short_ml;
    int splits, split_keys, short_rows;
    int short_max;             // the most query rows of a request that is k_paged_attn's
    float* part_o;             // k_paged_chunk: [chunk_splits][n_tokens][nq][hd]
    float2* part_ml;
    int chunk_splits, chunk_keys;
};

// Probabilities are 2^(c (s - ref) + lift).  The difference comes first, so that it
// is exact near the maximum however large the scores are (k_paged_chunk does that
// where c ref is large).  The reference only moves when a row's maximum has outgrown
// it by 2^8; the lift takes fp16 values away from the subnormal ones.
template <class T> constexpr float kLift = 0.0f;
template <> constexpr float kLift<_Float16> = 7.0f;

// The result of a row from its unnormalised sum.  top: the reference; l: the sum,
// or for a reference of -inf a mark: 0 when no key was seen, else more (all at
// -inf) or NaN.
__device__ __forceinline__ float row_result(float o, float top, float l) {
    return top == -INFINITY ? (l == 0.0f ? 0.0f : NAN) : o / l;
}
template <class T>
__device__ __forceinline__ float row_lse(float top, float l, float scale) {
    return top == -INFINITY ? (l != l ? l : -INFINITY) : __builtin_fmaf(top, scale, (__log2f(l) - kLift<T>) * kLn2);
}
// What sums relative to `ref` weigh in ones relative to `top` >= ref.
__device__ __forceinline__ float ref_weight(float ref, float top, float c) {
    return ref == top ? 1.0f : __builtin_amdgcn_exp2f((ref - top) * c);
}

template <int HD, class T, int W>
__global__ __launch_bounds__(64 * W, 2) void k_paged_attn(AttnArgs a) {
    constexpr int DS = HD / 32, DJ = HD / 16;
    constexpr int OS = HD + 4;                       // floats per row of the joined sums
    __shared__ float osh[W * 16 * OS];
    __shared__ float msh[W][16], lsh[W][16];
    const Paged& p = a.p;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int g = lane >> 4, c16 = lane & 15;
    const int r = blockIdx.z, kvh = blockIdx.y % p.nkv, tile = blockIdx.y / p.nkv, split = blockIdx.x;
    const Req q = req_of(p, r);
    const int rows = min(q.n, p.max_q) * p.G;
    if (tile * 16 >= rows || rows > a.short_max) return;
    const int R = min(tile * 16 + c16, rows - 1);    // this lane's query row (the last one repeated)
    const int tok = q.start + R / p.G, hq = kvh * p.G + R % p.G;
    const int vis = min(q.base + R / p.G + 1, p.limit);
    const int vmin = min(q.base + tile * 16 / p.G + 1, p.limit);
    const int kend = min(q.base + min(tile * 16 + 15, rows - 1) / p.G + 1, p.limit);
    const int k0 = split * a.split_keys, k1 = min(kend, k0 + a.split_keys);
    if (k0 >= k1 && split > 0) return;

    u32x4_t qf[DS];
    {
        const uint16_t* qr = a.q + (size_t)tok * a.q_stride + (size_t)hq * HD + 8 * g;
#pragma unroll
        for (int s = 0; s < DS; s++) qf[s] = *reinterpret_cast<const u32x4_t*>(qr + 32 * s);
    }
    const int* table = p.table + (size_t)r * p.max_pages;
    const int pmask = (1 << p.shift) - 1;

    float4_t o[DJ];
    float ref, l;
    bool seen;
    for (int careful = 0;; careful = 1) {
#pragma unroll
        for (int j = 0; j < DJ; j++) o[j] = float4_t{0.f, 0.f, 0.f, 0.f};
        ref = -INFINITY;
        l = 0.0f;
        seen = false;
        for (int kb = k0 + 32 * wave; kb < k1; kb += 32 * W) {
            u32x4_t kf[2][DS];
            uint32_t vr[8][DJ / 2];
            size_t vrow[2];
            bool ok[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int kk = kb + 16 * u;
                const int pg = kk < k1 ? table[kk >> p.shift] : -1;
                ok[u] = (unsigned)pg < (unsigned)p.n_pages;
                const size_t row = (((size_t)(ok[u] ? pg : 0) * p.nkv + kvh) << p.shift) + (kk & pmask);
                vrow[u] = row * HD;
                const uint16_t* kp = p.kp + (row + c16) * HD + 8 * g;
#pragma unroll
                for (int s = 0; s < DS; s++) kf[u][s] = *reinterpret_cast<const u32x4_t*>(kp + 32 * s);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint16_t* vp = p.vp + (row + 4 * g + e) * HD + DJ * c16;
                    if constexpr (DJ == 4) {
                        const uint2 v = *reinterpret_cast<const uint2*>(vp);
                        vr[4 * u + e][0] = v.x;
                        vr[4 * u + e][1] = v.y;
                    } else {
#pragma unroll
                        for (int d = 0; d < DJ / 8; d++) {
                            const u32x4_t v = *reinterpret_cast<const u32x4_t*>(vp + 8 * d);
#pragma unroll
                            for (int w = 0; w < 4; w++) vr[4 * u + e][4 * d + w] = v[w];
                        }
                    }
                }
            }
            const bool edge = kb + 32 > vmin || !ok[0] || !ok[1];
            if (kb + 32 > kend || !ok[0] || !ok[1]) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (!ok[e >> 2] || kb + 16 * (e >> 2) + 4 * g + (e & 3) >= kend)
#pragma unroll
                        for (int d = 0; d < DJ / 2; d++) vr[e][d] = 0;
            }
            float4_t s[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                s[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int d = 0; d < DS; d++) s[u] = mfma16(T(), kf[u][d], qf[d], s[u]);
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!ok[u] || kb + 16 * u + 4 * g + i >= vis) s[u][i] = -INFINITY;
                }
                seen |= ok[u] && kb + 16 * u < vis;
            }
            float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                             fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            mx = rows_max4(mx);
            const float next = (mx - ref) * a.c > 8.0f ? mx : ref;
            const float off = next == -INFINITY ? 0.0f : next;
            if (__any(next != ref)) {
                const float alpha = ref_weight(ref, next, a.c);
                l = l * alpha;
#pragma unroll
                for (int j = 0; j < DJ; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[j][i] = o[j][i] * alpha;
                ref = next;
            }
            u32x4_t ph, pl;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                float lo[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i] - off, a.c, kLift<T>));
                    l = l + s[u][i];
                    lo[i] = s[u][i] - (float)(T)s[u][i];
                }
                ph[2 * u] = pack16<T>(s[u][0], s[u][1]);
                ph[2 * u + 1] = pack16<T>(s[u][2], s[u][3]);
                pl[2 * u] = pack16<T>(lo[0], lo[1]);
                pl[2 * u + 1] = pack16<T>(lo[2], lo[3]);
            }
            bool slow = false;
            if (careful) {
                constexpr uint32_t ex = sizeof(T) == 2 && kLift<T> != 0.0f ? 0x7c00u : 0x7f80u;
#pragma unroll
                for (int e = 0; e < 8; e++)
#pragma unroll
                    for (int d = 0; d < DJ / 2; d++)
                        slow |= (vr[e][d] & ex) == ex || ((vr[e][d] >> 16) & ex) == ex;
                slow = __any(slow);
            }
            if (!slow) {
#pragma unroll
                for (int j = 0; j < DJ; j++) {
                    const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
                    u32x4_t vf;
#pragma unroll
                    for (int w = 0; w < 4; w++)
                        vf[w] = __builtin_amdgcn_perm(vr[2 * w + 1][j / 2], vr[2 * w][j / 2], sel);
                    o[j] = mfma16(T(), vf, pl, o[j]);
                    o[j] = mfma16(T(), vf, ph, o[j]);
                }
            } else {
                float* ps = osh + wave * 16 * OS;            // [32 keys][16 rows]
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) ps[(16 * u + 4 * g + i) * 16 + c16] = s[u][i];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                for (int key = 0; key < 32; key++) {
                    if (!ok[key >> 4] || kb + key >= vis) continue;
                    const float pk = ps[key * 16 + c16];
                    const uint16_t* vp = p.vp + vrow[key >> 4] + (size_t)(key & 15) * HD;
#pragma unroll
                    for (int j = 0; j < DJ; j++)
#pragma unroll
                        for (int i = 0; i < 4; i++) o[j][i] = o[j][i] + pk * widen16<T>(vp[DJ * (4 * g + i) + j]);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
        if (careful) break;
        float any = 0.0f;                            // NaN when an output is not finite
#pragma unroll
        for (int j = 0; j < DJ; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) any = any + o[j][i] * 0.0f;
        if (!__any(any != any && l == l)) break;     // (a sum that is none is one of scores)
    }

    l = rows_sum4(l);
    if (ref == -INFINITY && l == l) l = seen ? 1.0f : 0.0f;
    if (g == 0) {
        msh[wave][c16] = ref;
        lsh[wave][c16] = l;
    }
    __syncthreads();
    {
        float top = msh[0][c16];
#pragma unroll
        for (int x = 1; x < W; x++) top = fmaxf(top, msh[x][c16]);
        const float w = ref_weight(ref, top, a.c);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < DJ; j += 4)
                *reinterpret_cast<float4*>(osh + (wave * 16 + c16) * OS + DJ * (4 * g + i) + j) =
                    make_float4(o[j][i] * w, o[j + 1][i] * w, o[j + 2][i] * w, o[j + 3][i] * w);
    }
    __syncthreads();
    // 4 W threads per row, DV values each
    constexpr int DV = HD / (4 * W);
    const int row = threadIdx.x / (4 * W), d0 = DV * (threadIdx.x % (4 * W));
    if (tile * 16 + row >= rows) return;
    float top = msh[0][row];
#pragma unroll
    for (int x = 1; x < W; x++) top = fmaxf(top, msh[x][row]);
    float sum = 0.0f, v[DV];
#pragma unroll
    for (int j = 0; j < DV; j++) v[j] = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) {
        sum = sum + lsh[w][row] * ref_weight(msh[w][row], top, a.c);
#pragma unroll
        for (int j = 0; j < DV; j += 2) {
            const float2 x = *reinterpret_cast<const float2*>(osh + (w * 16 + row) * OS + d0 + j);
            v[j] += x.x;
            v[j + 1] += x.y;
        }
    }
    const int orow = tile * 16 + row, otok = q.start + orow / p.G, oh = kvh * p.G + orow % p.G;
    if (a.splits > 1) {
        const size_t at = (((size_t)split * p.n_req + r) * p.nkv + kvh) * a.short_rows + orow;
        float* po = a.short_o + at * HD + d0;
#pragma unroll
        for (int j = 0; j < DV; j += 2) *reinterpret_cast<float2*>(po + j) = make_float2(v[j], v[j + 1]);
        if (d0 == 0) a.short_ml[at] = make_float2(top, sum);
        return;
    }
    uint16_t* dst = a.out + (size_t)otok * a.out_stride + (size_t)oh * HD + d0;
#pragma unroll
    for (int j = 0; j < DV; j += 2)
        *reinterpret_cast<uint32_t*>(dst + j) = pack16<T>(row_result(v[j], top, sum), row_result(v[j + 1], top, sum));
    if (a.lse && d0 == 0) a.lse[(size_t)otok * p.nq + oh] = row_lse<T>(top, sum, a.scale);
}

// ---- attention: many query rows -----------------------------------------------------
//
// Requests with more than kShort query rows: a block takes 128 of them (new rows
// x the group's heads) of one KV head against tiles of KB keys, 32 rows a wave, so
// that a K or V fragment read from LDS feeds 32 rows.  Two groups of four waves
// (one at 256 dimensions, for its registers) take alternate tiles and are joined
// in LDS at the end: a CU holds one block, and two waves per SIMD let one's
// exponentials run beside the other's products.
//   S^T = K . Q^T    v_mfma_32x32x16: a lane holds half of its row's scores, the
//                    lane 32 away the other half
//   O^T = V^T . P^T  the scores' order in a lane is the k order of this product;
//                    V^T comes out of row-major LDS by ds_read_b64_tr_b16
// LDS rows have their 16-byte chunks permuted by the row number, so that neither
// kind of read meets its own banks.
// Probabilities go in rounded to the type once (the output's own rounding is as
// large, and a second part would cost half as many products again); the sums are
// of the unrounded ones.
// What bounds it: 2048 rows over 8192, 16 heads of 128 over 8, 148 us, 810 TFLOP/s (a
// large library product: 1108).  Softmax and barriers alone take 96 us of it, with
// the products beside them 105; the rest is the tiles' way into LDS.  64 rows a wave
// would halve what is read from there, but need 416 registers besides addresses,
// with one wave per SIMD, and did not fit without spills.
//
// Masked places have probability 0, but K and V values there that are not finite
// leave 0 * inf behind: rows whose sum of weights is a number and whose output is
// not are computed again by row_again, key by key in fp32.
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float16_t mfma32(_Float16, u32x4_t a, u32x4_t b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                  0, 0);
}
__device__ __forceinline__ float16_t mfma32(__bf16, u32x4_t a, u32x4_t b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0,
                                                   0);
}
// Four rows of an LDS matrix, transposed: lane t of each 16 gives the address of
// values 4 (t % 4) .. of row t / 4 and gets value t of the four rows.
__device__ __forceinline__ uint2 lds_read_tr(const uint16_t* p) {
    typedef __attribute__((address_space(3))) s16x4_t lds_t;
    const s16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)p);
    return __builtin_bit_cast(uint2, v);
}
// What a row's 16-byte chunk numbers are XORed with in LDS, by the row number
// mod 16.  A read of K takes one chunk of each of 32 rows: all values occur.  A
// transposing read of V takes four neighbouring chunks of rows 0-3 and 4-7 (or 8-11
// and 12-15): consecutive rows differ in the bits above the lowest two.
template <int HD>
__device__ __forceinline__ int lds_swap(int row) {
    return HD == 64 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
}
// The other 32 lanes' value.
__device__ __forceinline__ float half_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// One query row over keys [k0, k1) by a wave, in fp32 and without matrix products:
// the unnormalised outputs of dims (HD/64) lane .., their reference and sum.
template <int HD, class T>
__device__ __forceinline__ void row_again(const Paged& p, int r, int kvh, const uint16_t* qr, float c, int k0, int k1,
                                       float* o, float* top, float* sum) {
    constexpr int DL = HD / 64;
    const int lane = threadIdx.x & 63;
    float ref = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < DL; d++) o[d] = 0.0f;
    for (int kb = k0; kb < k1; kb += 64) {
        const int j = kb + lane;
        const long long at = j < k1 ? pool_row(p, r, kvh, j) : -1;
        float s = -INFINITY;
        if (at >= 0) {
            s = 0.0f;
            for (int d = 0; d < HD; d += 8) {
                const u32x4_t k = *reinterpret_cast<const u32x4_t*>(p.kp + at * HD + d);
                const u32x4_t q = *reinterpret_cast<const u32x4_t*>(qr + d);
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    s = s + widen16<T>((uint16_t)k[w]) * widen16<T>((uint16_t)q[w]);
                    s = s + widen16<T>((uint16_t)(k[w] >> 16)) * widen16<T>((uint16_t)(q[w] >> 16));
                }
            }
        }
        const float mx = fmaxf(wave_max(s), ref);
        if (mx == -INFINITY) continue;
        const float alpha = ref_weight(ref, mx, c);
        const float w = at >= 0 ? __builtin_amdgcn_exp2f(__builtin_fmaf(s - mx, c, kLift<T>)) : 0.0f;
        ref = mx;
        l = l * alpha + wave_sum(w);
#pragma unroll
        for (int d = 0; d < DL; d++) o[d] = o[d] * alpha;
        for (int i = 0; i < 64; i++) {
            const long long v = __shfl(at, i, kWave);
            if (v < 0) continue;
            const float wi = __shfl(w, i, kWave);
#pragma unroll
            for (int d = 0; d < DL; d++) o[d] = o[d] + wi * widen16<T>(p.vp[v * HD + DL * lane + d]);
        }
    }
    *top = ref;
    *sum = l;
}

template <int HD>
constexpr int kTileKeys = HD == 256 ? 32 : 64;

template <int HD, class T, bool WHOLE>
__global__ __launch_bounds__(HD == 256 ? 256 : 512, HD == 256 ? 1 : 2) void k_paged_chunk(AttnArgs a) {
    constexpr int GR = HD == 256 ? 1 : 2;           // groups of four waves
    constexpr int KB = kTileKeys<HD>;               // keys per tile
    constexpr int CH = HD / 8;                      // 16-byte chunks per row
    constexpr int DS = HD / 16, DT = HD / 32, KT = KB / 32;
    constexpr int U = KB * CH / 256;                // 16-byte loads per thread and tile
    constexpr int RPU = 256 / CH, RPW = 64 / CH;    // rows per round of loads, of a group and of a wave
    constexpr int TN = KB * HD;                     // values per tile
    // tiles of even and odd numbers apart: the compiler then knows that a tile on
    // its way to LDS is not the one that is read
    __shared__ __attribute__((aligned(16))) uint16_t k_even[GR * TN], k_odd[GR * TN], v_even[GR * TN], v_odd[GR * TN];
    __shared__ float mg_ref[GR * kRows], mg_sum[GR * kRows];
    __shared__ int again, redo[kRows];

    const Paged& p = a.p;
    const int grp = GR == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int tid = threadIdx.x & 255, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int hi = lane >> 5, c32 = lane & 31;
    const int kvh = blockIdx.x % p.nkv;

    // the request and the block of rows in it: the last ones (the longest) first
    auto blocks_of = [&](const Req& q) __attribute__((always_inline)) -> int {
        const int rows = min(q.n, p.max_q) * p.G;
        return rows > a.short_max ? (rows + kRows - 1) / kRows : 0;
    };
    Req q = {0, 0, 0};
    int r = -1, tile = 0, total = 0;
    for (int j0 = 0; j0 < p.n_req; j0 += 64) total += wave_total(j0 + lane < p.n_req ? blocks_of(req_of(p, j0 + lane)) : 0);
    int want = total - 1 - (int)(blockIdx.x / p.nkv);
    if (want < 0) return;
    for (int j0 = 0; j0 < p.n_req && r < 0; j0 += 64) {
        const Req mine = j0 + lane < p.n_req ? req_of(p, j0 + lane) : Req{0, 0, 0};
        const int t = blocks_of(mine);
        int upto = t;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(upto, o, kWave);
            if (lane >= o) upto += y;
        }
        const unsigned long long hit = __ballot(upto > want);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            r = j0 + src;
            tile = want - __builtin_amdgcn_readlane(upto - t, src);
            q.start = __builtin_amdgcn_readlane(mine.start, src);
            q.n = __builtin_amdgcn_readlane(mine.n, src);
            q.base = __builtin_amdgcn_readlane(mine.base, src);
        } else {
            want -= __builtin_amdgcn_readlane(upto, 63);
        }
    }
    const int rows = min(q.n, p.max_q) * p.G, row0 = tile * kRows;
    const int R = min(row0 + 32 * wave + c32, rows - 1);
    const int tok = q.start + R / p.G, hq = kvh * p.G + R % p.G;
    const int vis = min(q.base + R / p.G + 1, p.limit);
    const int vmin = min(q.base + row0 / p.G + 1, p.limit);
    const int kend = min(q.base + min(row0 + kRows - 1, rows - 1) / p.G + 1, p.limit);
    const int split = blockIdx.y;
    const int k0 = split * a.chunk_keys, k1 = min(kend, k0 + a.chunk_keys);
    if (k0 >= k1 && split > 0) return;

    u32x4_t qf[DS];
    {
        const uint16_t* qr = a.q + (size_t)tok * a.q_stride + (size_t)hq * HD + 8 * hi;
#pragma unroll
        for (int s = 0; s < DS; s++) qf[s] = *reinterpret_cast<const u32x4_t*>(qr + 16 * s);
    }

    // Tiles go from the pages straight into LDS.  Round i of a wave is RPW rows of
    // it, which lie in 16 keys and so in one page; LDS takes the lanes' chunks in
    // order, so a lane asks for the chunk that belongs in its place.  Keys past the
    // last one that the block sees repeat it; keys on pages that do not exist are
    // rows of page 0.  Both are masked.
    const int* table = p.table + (size_t)r * p.max_pages;
    const int pmask = (1 << p.shift) - 1;
    const int srow = tid / CH, sch = tid % CH;
    constexpr int NG = KB / 16;                     // 16-key groups of a tile
    typedef int i4_t __attribute__((ext_vector_type(4)));
    i4_t pgv, pgk, pgn;                             // page numbers of the next V and K tiles, and of one more
    auto pages = [&](int kb) __attribute__((always_inline)) {
        pgn = i4_t(fixed(table, min(kb, kend - 1) >> p.shift));
        if (!WHOLE) {
            pgn.y = fixed(table, min(kb + 16, kend - 1) >> p.shift);
            if constexpr (NG == 4) {
                pgn.z = fixed(table, min(kb + 32, kend - 1) >> p.shift);
                pgn.w = fixed(table, min(kb + 48, kend - 1) >> p.shift);
            }
        }
    };
    auto turn_pages = [&]() __attribute__((always_inline)) {
        pgv = pgk;
        pgk = pgn;
    };
    auto there = [&](int page) __attribute__((always_inline)) -> bool { return (unsigned)page < (unsigned)p.n_pages; };
    auto exist = [&]() __attribute__((always_inline)) -> int {  // which of the K tile's groups do
        const int bits = (there(pgk.x) ? 1 : 0) | (there(pgk.y) ? 2 : 0);
        return NG == 4 ? bits | (there(pgk.z) ? 4 : 0) | (there(pgk.w) ? 8 : 0) : bits;
    };
    // byte offset of this lane's chunk in a whole tile; rounds V apart have the
    // same chunks, V RPU rows on
    constexpr int V = RPU % 16 ? 2 : 1;
    unsigned goes[V];
#pragma unroll
    for (int i = 0; i < V; i++) goes[i] = 2 * ((srow + i * RPU) * HD + 8 * (sch ^ lds_swap<HD>(srow + i * RPU)));
    auto base = [&](const uint16_t* src, int page, int key) __attribute__((always_inline)) -> const char* {
        return reinterpret_cast<const char*>(src + ((((size_t)(there(page) ? page : 0) * p.nkv + kvh) << p.shift) + (key & pmask)) * HD);
    };
    auto go = [&](const char* from, uint16_t* dst, int i) __attribute__((always_inline)) {
        typedef __attribute__((address_space(1))) const void gptr_t;
        typedef __attribute__((address_space(3))) void lptr_t;
        __builtin_amdgcn_global_load_lds((gptr_t*)from, (lptr_t*)(dst + (grp * KB + i * RPU + wave * RPW) * HD), 16, 0, 0);
    };
    // round i of a whole tile at `at`
    auto go_whole = [&](const char* at, uint16_t* dst, int i) __attribute__((always_inline)) {
        go(at + i / V * (V * RPU * HD * 2) + goes[i % V], dst, i);
    };
    auto load = [&](const uint16_t* src, i4_t pg, uint16_t* dst, int kb) __attribute__((always_inline)) {
        if (kb >= k1) return;
#pragma unroll
        for (int i = 0; i < U; i++) {
            // this round's 16 keys: 2 i + wave / 2, i or i / 2
            const int even = CH == 8 ? 2 * i : (CH == 16 ? i : i >> 1);
            const int page = CH == 8 && (wave >> 1) ? pg[(even + 1) & 3] : pg[even];
            const int key = min(kb + 16 * (even + (CH == 8 ? wave >> 1 : 0)), (kend - 1) & ~15);
            const unsigned row = min((srow + i * RPU) & 15, kend - 1 - key);
            go(base(src, page, key) + 2 * (row * HD + 8 * (sch ^ lds_swap<HD>(srow + i * RPU))), dst, i);
        }
    };
    // where this lane reads: K rows c32 (+ 32 kt), chunk 2 d + hi; V rows 4 hi + ..
    // (+ 16 kk, + 8), four values of column 32 d + ..
    int kat[DS], vat[DT][2];
#pragma unroll
    for (int d = 0; d < DS; d++) kat[d] = grp * TN + c32 * HD + 8 * ((2 * d + hi) ^ lds_swap<HD>(c32));
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int key = 8 * e + 4 * hi + ((lane & 15) >> 2), col = 32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            vat[d][e] = grp * TN + key * HD + 8 * ((col >> 3) ^ lds_swap<HD>(key)) + (col & 7);
        }

    float16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float ref = -INFINITY, l = 0.0f;
    bool seen = false;
    float16_t s[KT];
    u32x4_t pf[KB / 16];

    // The products read their fragments from LDS ahead: the first ones before the
    // phase begins, the others one product set before they are needed.
    u32x4_t kf[DS];
    uint2 vf[2][DT][2];
    auto kload = [&](const uint16_t* ks, int kt, int d) __attribute__((always_inline)) {
        kf[d] = *reinterpret_cast<const u32x4_t*>(ks + kat[d] + 32 * kt * HD);
    };
    auto vload = [&](const uint16_t* vs, int kk, int d) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 2; e++) vf[kk & 1][d][e] = lds_read_tr(vs + vat[d][e] + 16 * kk * HD);
    };
    // s = scores of the K tile (its first fragments are in kf); issue(i) requests what
    // goes beside product i of a phase
    constexpr int NM = KB / 16 * DT;                // products with V of a tile, and as many with K
    auto scores = [&](const uint16_t* ks, auto issue) __attribute__((always_inline)) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[kt][i] = 0.0f;
#pragma unroll
            for (int d = 0; d < DS; d++) {
                s[kt] = mfma32(T(), kf[d], qf[d], s[kt]);
                if (kt + 1 < KT) kload(ks, kt + 1, d);
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                if (kt + 1 < KT) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                issue(NM + kt * DS + d);
            }
        }
    };
    // pf = probabilities of s (keys kb ..), and what becomes of the sums so far
    auto softmax = [&](int kb, int bits) __attribute__((always_inline)) {
        if (kb + KB > vmin || bits != (1 << NG) - 1) {
            // keys that some row does not see, and pages that do not exist
            const int end = vis - kb - 4 * hi;
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[kt][i] = 32 * kt + 8 * (i >> 2) + (i & 3) < end ? s[kt][i] : -INFINITY;
#pragma unroll
            for (int u = 0; u < NG; u++) {
                if ((bits >> u) & 1) {
                    seen |= kb + 16 * u < vis;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) s[u >> 1][8 * (u & 1) + i] = -INFINITY;
                }
            }
        } else {
            seen = true;
        }
        float m4[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            m4[e] = s[0][e];
#pragma unroll
            for (int i = 4 + e; i < 16 * KT; i += 4) m4[e] = fmaxf(m4[e], s[i >> 4][i & 15]);
        }
        const float mx = half_max(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
        const float next = (mx - ref) * a.c > 8.0f ? mx : ref;
        if (__any(next != ref)) {
            const float alpha = ref_weight(ref, next, a.c);
            l = l * alpha;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] = o[d][i] * alpha;
            ref = next;
        }
        // the reference's exponent, rounded, is one factor of all probabilities
        // of the row; where a step of it is no longer small, the scores are taken
        // relative to the reference first
        float off = ref == -INFINITY ? 0.0f : __builtin_fmaf(-ref, a.c, kLift<T>);
        if (__any(fabsf(off) > 0x1p20f)) {
            const float base = ref == -INFINITY ? 0.0f : ref;
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[kt][i] = s[kt][i] - base;
            off = kLift<T>;
        }
        float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KB / 16; kk++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                float x[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk >> 1][8 * (kk & 1) + 2 * w + e], a.c, off));
                    l4[2 * (w & 1) + e] = l4[2 * (w & 1) + e] + x[e];
                }
                pf[kk][w] = pack16<T>(x[0], x[1]);
            }
        l = l + ((l4[0] + l4[1]) + (l4[2] + l4[3]));
    };
    // o += V tile . pf (its first fragments are in vf[0]); then the first of ks
    auto values = [&](const uint16_t* vs, const uint16_t* ks, auto issue) __attribute__((always_inline)) {
        constexpr int KK = KB / 16, KPD = (DS + DT - 1) / DT;
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const uint2 v0 = vf[kk & 1][d][0], v1 = vf[kk & 1][d][1];
                o[d] = mfma32(T(), u32x4_t{v0.x, v0.y, v1.x, v1.y}, pf[kk], o[d]);
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                if (kk + 1 < KK) {
                    vload(vs, kk + 1, d);
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                } else {
#pragma unroll
                    for (int x = KPD * d; x < KPD * (d + 1) && x < DS; x++) kload(ks, 0, x);
                    __builtin_amdgcn_sched_group_barrier(0x100, KPD, 0);
                }
                issue(kk * DT + d);
            }
    };

    // A group's phases: the softmax of tile t; then the products V of t and K of
    // t + 1.  The other group is one phase off, so that the SIMDs' matrix and
    // vector units are asked for by one of the two at a time.  Rows of t + 1 (V)
    // and t + 2 (K) are requested a few products apart in the second phase and are
    // waited for before the next one.  (All at once at the beginning of the first phase
    // they hold up the wave that asks: 2048 rows over 8192, 16 heads of 128 over 8, 156
    // us for 148; 8 of 256 over 4, 257 for 225; 1024 rows, 32 of 64 over 8, 112 for 99.)
    // Where a tile is of several pages or is not whole, they are requested at the
    // beginning of the first phase and waited for at the end of the second.
    const int nt = (k1 - k0 + KB - 1) / KB, steps = (nt + GR - 1) / GR;
    int kb = k0 + grp * KB;                         // this group's tile
    if (threadIdx.x == 0) again = 0;
    int bits = 0, bits1 = 0, bits2;                 // groups of 16 keys that exist: this tile, the next ones
    // what a wave has requested is in LDS once it has waited for it
    auto arrived = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    auto barrier = [&]() __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto none = [](int) __attribute__((always_inline)) {};
    if (nt > 0) {
        pages(kb);
        turn_pages();
        pages(kb + GR * KB);
        bits = exist();
        load(p.kp, pgk, k_even, kb);
        load(p.vp, pgk, v_even, kb);
        turn_pages();
        pages(kb + 2 * GR * KB);
        bits1 = exist();
        load(p.kp, pgk, k_odd, kb + GR * KB);
        turn_pages();
        arrived();
        if (grp < nt) {
#pragma unroll
            for (int d = 0; d < DS; d++) kload(k_even, 0, d);
            scores(k_even, none);
        }
        if (grp == 1) __syncthreads();
    }
    bool pending = false;
    auto first = [&](const uint16_t* vs) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < DT; d++) vload(vs, 0, d);
    };
    for (int t0 = 0; t0 < steps; t0 += 2) {
#pragma unroll
        for (int odd = 0; odd < 2; odd++) {
            const int t = (t0 + odd) * GR + grp;
            if (t0 + odd >= steps) break;
            uint16_t* const vn = odd ? v_even : v_odd;
            uint16_t* const kn = odd ? k_odd : k_even;
            const bool fast = WHOLE && kb + 2 * GR * KB + KB <= k1;
            // (the wait for a page number goes where it delays less: 148 for 158 us, and
            // with pages of 16 rows 44.4 for 48.9)
            if (WHOLE) {
                bits2 = exist();
                pages(kb + 3 * GR * KB);
            }
            if (!fast) {
                load(p.vp, pgv, vn, kb + GR * KB);
                load(p.kp, pgk, kn, kb + 2 * GR * KB);
            }
            if (!WHOLE) {
                bits2 = exist();
                pages(kb + 3 * GR * KB);
            }
            if (t < nt) softmax(kb, bits);
            if (pending) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                barrier();
                first(odd ? v_odd : v_even);
            } else {
                first(odd ? v_odd : v_even);
                barrier();
            }
            // (after the last tile: the scores of one that nobody asks for)
            if (t < nt) {
                const char* const va = base(p.vp, pgv.x, kb + GR * KB);
                const char* const ka = base(p.kp, pgk.x, kb + 2 * GR * KB);
                auto issue = [&](int i) __attribute__((always_inline)) {
                    if (i % (NM / U) != 0) return;
                    i /= NM / U;
                    if (!fast) return;
                    if (i < U) go_whole(va, vn, i);
                    else go_whole(ka, kn, i - U);
                };
                values(odd ? v_odd : v_even, odd ? k_even : k_odd, issue);
                scores(odd ? k_even : k_odd, issue);
            }
            turn_pages();
            bits = bits1;
            bits1 = bits2;
            kb += GR * KB;
            if (!fast) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            pending = fast;
            barrier();
        }
    }
    if (GR == 2 && grp == 0 && nt > 0) __syncthreads();
    __syncthreads();

    // The groups' sums, brought to a common reference: each group finishes half of
    // the dims (at 256 dimensions the one group all) and leaves the other half in
    // LDS for the other.
    l = half_sum(l);
    if (ref == -INFINITY && l == l) l = seen ? 1.0f : 0.0f;
    constexpr int DH = DT / GR;
    static_assert(GR == 1 || DH * 16 * 256 * 4 <= (int)sizeof k_even, "the halves fit the tiles");
    const int row = 32 * wave + c32;                // of the block
    if (GR == 2) {
        if (grp == 1) {
#pragma unroll
            for (int d = 0; d < DH; d++) {
                const float16_t x = o[d];
                o[d] = o[d + DH];
                o[d + DH] = x;
            }
        }
        float4* const give = reinterpret_cast<float4*>(grp == 0 ? k_odd : k_even);
#pragma unroll
        for (int d = 0; d < DH; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                give[(4 * d + i / 4) * 256 + tid] =
                    make_float4(o[d + DH][i], o[d + DH][i + 1], o[d + DH][i + 2], o[d + DH][i + 3]);
        if (hi == 0) {
            mg_ref[grp * kRows + row] = ref;
            mg_sum[grp * kRows + row] = l;
        }
        if (threadIdx.x < kRows) redo[threadIdx.x] = 0;
        __syncthreads();
        const float ref1 = mg_ref[(grp ^ 1) * kRows + row], l1 = mg_sum[(grp ^ 1) * kRows + row], top = fmaxf(ref, ref1);
        const float w0 = ref_weight(ref, top, a.c), w1 = ref_weight(ref1, top, a.c);
        const float4* const take = reinterpret_cast<const float4*>(grp == 0 ? k_even : k_odd);
#pragma unroll
        for (int d = 0; d < DH; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 x = take[(4 * d + i / 4) * 256 + tid];
                o[d][i] = o[d][i] * w0 + x.x * w1;
                o[d][i + 1] = o[d][i + 1] * w0 + x.y * w1;
                o[d][i + 2] = o[d][i + 2] * w0 + x.z * w1;
                o[d][i + 3] = o[d][i + 3] * w0 + x.w * w1;
            }
        l = l * w0 + l1 * w1;
        ref = top;
    } else {
        if (threadIdx.x < kRows) redo[threadIdx.x] = 0;
        __syncthreads();
    }
    const bool rv = row0 + row < rows;
    const size_t orow = (size_t)tok * p.nq + hq;
    {
        float any = 0.0f;                  // NaN when an output is not finite
#pragma unroll
        for (int d = 0; d < DH; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) any = __builtin_fmaf(o[d][i], 0.0f, any);
        if (rv && any != any && l == l) {
            redo[row] = 1;
            again = 1;
        }
        const int col = 32 * DH * grp;
        if (a.chunk_splits > 1) {
            const size_t at = (size_t)split * p.n_tokens * p.nq + orow;
            float* po = a.part_o + at * HD + col + 4 * hi;
            if (rv) {
#pragma unroll
                for (int d = 0; d < DH; d++)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<float4*>(po + 32 * d + 2 * i) = make_float4(o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
                if (hi == 0 && grp == 0) a.part_ml[at] = make_float2(ref, l);
            }
        } else {
            // eight dims a lane: the halves of a wave exchange every other four
            uint16_t* dst = a.out + (size_t)tok * a.out_stride + (size_t)hq * HD + col + 8 * hi;
            const float inv = ref == -INFINITY ? 0.0f : 1.0f / l;
            const float none = row_result(0.0f, ref, l);
#pragma unroll
            for (int d = 0; d < DH; d++)
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x = o[d][i + 2 * e] * inv, y = o[d][i + 2 * e + 1] * inv;
                        w[e] = ref == -INFINITY ? pack16<T>(none, none) : pack16<T>(x, y);
                    }
                    const auto a0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
                    const auto a1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                    if (rv) *reinterpret_cast<uint4*>(dst + 32 * d + 2 * i) = make_uint4(a0[0], a1[0], a0[1], a1[1]);
                }
            if (rv && a.lse && hi == 0 && grp == 0) a.lse[orow] = row_lse<T>(ref, l, a.scale);
        }
    }
    __syncthreads();
    if (!again || grp != 0) return;
    unsigned long long todo = __ballot(redo[row] != 0) & 0xffffffffull;
    while (todo) {
        const int c = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int R2 = row0 + 32 * wave + c, t2 = q.start + R2 / p.G, h2 = kvh * p.G + R2 % p.G;
        float x[HD / 64], top, sum;
        row_again<HD, T>(p, r, kvh, a.q + (size_t)t2 * a.q_stride + (size_t)h2 * HD, a.c, k0,
                         min(k1, min(q.base + R2 / p.G + 1, p.limit)), x, &top, &sum);
        const size_t row2 = (size_t)t2 * p.nq + h2;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) {
            const int at = HD / 64 * lane + d;
            if (a.chunk_splits > 1) a.part_o[((size_t)split * p.n_tokens * p.nq + row2) * HD + at] = x[d];
            else a.out[(size_t)t2 * a.out_stride + (size_t)h2 * HD + at] = bits16<T>(row_result(x[d], top, sum));
        }
        if (a.chunk_splits > 1 && lane == 0) a.part_ml[(size_t)split * p.n_tokens * p.nq + row2] = make_float2(top, sum);
    }
}

// Joins the splits of a row: W waves per row.  Rows of a short request lie at
// ((split * n_req + r) * nkv + KV head) * short_rows + row of the short partials,
// the others at split * n_tokens * nq + token * nq + head.
template <int HD, class T, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void k_paged_join(AttnArgs a) {
    constexpr int DL = HD / 64;
    __shared__ float osh[W][HD + 4];
    const Paged& p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = W == 1 ? 0 : wave;
    const float* part_o;
    const float2* part_ml;
    size_t step;
    int t, h, kend, keys;
    if (W > 1) {
        // a block per short row
        const int r = blockIdx.z, kvh = blockIdx.y, R = blockIdx.x;
        const Req q = req_of(p, r);
        const int rows = min(q.n, p.max_q) * p.G;
        if (R >= rows || rows > a.short_max) return;
        const int tile = R / 16;
        t = q.start + R / p.G;
        h = kvh * p.G + R % p.G;
        kend = min(q.base + min(tile * 16 + 15, rows - 1) / p.G + 1, p.limit);
        keys = a.split_keys;
        step = (size_t)p.n_req * p.nkv * a.short_rows;
        const size_t row = ((size_t)r * p.nkv + kvh) * a.short_rows + R;
        part_o = a.short_o + row * HD;
        part_ml = a.short_ml + row;
    } else {
        const long long row = (long long)blockIdx.x * 4 + wave;
        if (row >= (long long)p.n_tokens * p.nq) return;
        t = (int)(row / p.nq);
        h = (int)(row % p.nq);
        const int r = find_req(p, t, lane);
        if (r >= p.n_req) return;
        const Req q = req_of(p, r);
        const int i = t - q.start, rows = min(q.n, p.max_q) * p.G, R = i * p.G + h % p.G;
        if (i < 0 || R >= rows || rows <= a.short_max) return;
        kend = min(q.base + min(R / kRows * kRows + kRows - 1, rows - 1) / p.G + 1, p.limit);
        keys = a.chunk_keys;
        step = (size_t)p.n_tokens * p.nq;
        part_o = a.part_o + row * HD;
        part_ml = a.part_ml + row;
    }
    const int ns = max((kend + keys - 1) / keys, 1);
    float top = -INFINITY;
    for (int s = lane; s < ns; s += 64) top = fmaxf(top, part_ml[s * step].x);
    top = wave_max(top);
    float sum = 0.0f, v[DL];
#pragma unroll
    for (int d = 0; d < DL; d++) v[d] = 0.0f;
#pragma unroll 4
    for (int s = sub; s < ns; s += W) {
        const float2 ml = part_ml[s * step];
        const float w = ref_weight(ml.x, top, a.c);
        sum = sum + ml.y * w;
        const float* po = part_o + s * step * HD + DL * lane;
#pragma unroll
        for (int d = 0; d < DL; d++) v[d] = v[d] + po[d] * w;
    }
    if (W > 1) {
#pragma unroll
        for (int d = 0; d < DL; d++) osh[wave][DL * lane + d] = v[d];
        if (lane == 0) osh[wave][HD] = sum;
        __syncthreads();
        if (sub != 0) return;
#pragma unroll
        for (int w = 1; w < W; w++) {
#pragma unroll
            for (int d = 0; d < DL; d++) v[d] = v[d] + osh[w][DL * lane + d];
            sum = sum + osh[w][HD];
        }
    }
    uint16_t* dst = a.out + (size_t)t * a.out_stride + (size_t)h * HD + DL * lane;
#pragma unroll
    for (int d = 0; d < DL; d++) dst[d] = bits16<T>(row_result(v[d], top, sum));
    if (a.lse && lane == 0) a.lse[(size_t)t * p.nq + h] = row_lse<T>(top, sum, a.scale);
}

// ---- received weight ---------------------------------------------------------------
//
// The keys are what is owned: nobody else adds to a workgroup's keys, so their sums
// have one order and need no atomics.  K rows stay in registers as the matrix
// operand, query rows pass by.
//   few query rows (a decoding step): a wave owns 16 keys and goes over all rows.
//     Reading K is all there is to it: 32 requests of 2049 rows, 8 heads of 128, 18
//     us, 4.7 TB/s.
//   many (a chunk): a workgroup owns 64 keys (32 at 256 dimensions), its four
//     waves take every fourth tile of 32 rows, the next tile's rows on their way
//     during the products of this one, and their sums are added in LDS in order.
//     515 rows over 4000, 8 heads over 4 of 64, two requests: 12.5 us, where the
//     other form, which waits for each tile's rows, takes 34.5.  Half of it are the
//     exponentials, of which there are as many as scores.  (Of 1, 2, 4, 8 and 16
//     waves: 15.5, 19.6, 12.5, 17.9 and 29.5 us.)
struct MassArgs {
    Paged p;
    const uint16_t* q;
    long long q_stride;
    float scale;
    const float* lse;
};

// The weight of score s.
__device__ __forceinline__ float weight(float s, float scale, float lse) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(s, scale, -lse) * kLog2e);
}

template <int HD, class T>
__global__ __launch_bounds__(256) void k_paged_mass(MassArgs a) {
    constexpr int DS = HD / 32;
    const Paged& p = a.p;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int g = lane >> 4, c16 = lane & 15;
    const int r = blockIdx.z, kvh = blockIdx.y;
    const Req q = req_of(p, r);
    const int n = min(q.n, p.max_q), rows = n * p.G;
    const int kend = min(q.base + n, p.limit);
    const int kb = 64 * blockIdx.x + 16 * wave;
    if (rows == 0 || kb >= kend) return;
    const int pg = fixed(p.table, (size_t)r * p.max_pages + (kb >> p.shift));
    if ((unsigned)pg >= (unsigned)p.n_pages) return;
    const size_t row = (((size_t)pg * p.nkv + kvh) << p.shift) + (kb & ((1 << p.shift) - 1));
    u32x4_t kf[DS];
#pragma unroll
    for (int s = 0; s < DS; s++) kf[s] = *reinterpret_cast<const u32x4_t*>(p.kp + (row + c16) * HD + 32 * s + 8 * g);
    float4_t sum = float4_t{0.f, 0.f, 0.f, 0.f};
    const int r0 = max(kb - q.base, 0) * p.G;              // the first row that sees key kb
    for (int t0 = r0 & ~15; t0 < rows; t0 += 16) {
        const int R = t0 + c16, Rc = min(R, rows - 1), i = Rc / p.G;
        const int tok = q.start + i, h = kvh * p.G + Rc % p.G;
        const uint16_t* qr = a.q + (size_t)tok * a.q_stride + (size_t)h * HD + 8 * g;
        float4_t s = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DS; d++) s = mfma16(T(), kf[d], *reinterpret_cast<const u32x4_t*>(qr + 32 * d), s);
        const float ls = a.lse[(size_t)tok * p.nq + h];
        const int vis = R < rows && ls != -INFINITY ? min(q.base + i + 1, p.limit) : 0;
#pragma unroll
        for (int e = 0; e < 4; e++) sum[e] = sum[e] + (kb + 4 * g + e < vis ? weight(s[e], a.scale, ls) : 0.0f);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) sum[e] = row_sum16(sum[e]);
    if (c16 < 4 && kb + 4 * g + c16 < kend) {
        const float add = c16 == 0 ? sum[0] : c16 == 1 ? sum[1] : c16 == 2 ? sum[2] : sum[3];
        p.mass[row + 4 * g + c16] += add;
    }
}

constexpr int kMassRows = 32;          // query rows up to which the first form is taken
constexpr int kMassWaves = 4;

template <int HD, class T>
__global__ __launch_bounds__(64 * kMassWaves, 2) void k_paged_mass_chunk(MassArgs a) {
    constexpr int DS = HD / 16, KT = HD == 256 ? 1 : 2, KB = 32 * KT;
    __shared__ float part[kMassWaves][KB];
    const Paged& p = a.p;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int hi = lane >> 5, c32 = lane & 31;
    const int r = blockIdx.z, kvh = blockIdx.y, kb = KB * blockIdx.x;
    const Req q = req_of(p, r);
    const int n = min(q.n, p.max_q), rows = n * p.G;
    const int kend = min(q.base + n, p.limit);
    if (rows == 0 || kb >= kend) return;

    // K rows (of page 0 where a page does not exist: not written below)
    u32x4_t kf[KT][DS];
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
        const long long at = pool_row(p, r, kvh, min(kb + 32 * kt + c32, kend - 1));
        const uint16_t* kp = p.kp + (at < 0 ? 0 : at) * HD + 8 * hi;
#pragma unroll
        for (int d = 0; d < DS; d++) kf[kt][d] = *reinterpret_cast<const u32x4_t*>(kp + 16 * d);
    }
    float16_t sum[KT];
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
        for (int i = 0; i < 16; i++) sum[kt][i] = 0.0f;

    u32x4_t qn[DS];
    float ln;
    int vn;                                         // keys that this lane's row of the next tile sees
    auto load = [&](int t0) __attribute__((always_inline)) {
        const int R = t0 + c32, Rc = min(R, rows - 1), i = Rc / p.G;
        const int tok = q.start + i, h = kvh * p.G + Rc % p.G;
        const uint16_t* qr = a.q + (size_t)tok * a.q_stride + (size_t)h * HD + 8 * hi;
#pragma unroll
        for (int d = 0; d < DS; d++) qn[d] = *reinterpret_cast<const u32x4_t*>(qr + 16 * d);
        ln = a.lse[(size_t)tok * p.nq + h];
        vn = R < rows ? min(q.base + i + 1, p.limit) : 0;
    };
    const int first = max(kb - q.base, 0) * p.G / 32;     // the first tile with a row that sees key kb
    int t0 = 32 * (first + wave);
    load(t0);
    for (; t0 < rows; t0 += 32 * kMassWaves) {
        u32x4_t qf[DS];
#pragma unroll
        for (int d = 0; d < DS; d++) qf[d] = qn[d];
        const float ls = ln;
        const int vis = ls == -INFINITY ? 0 : vn;
        load(t0 + 32 * kMassWaves);
        float16_t s[KT];
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[kt][i] = 0.0f;
#pragma unroll
            for (int d = 0; d < DS; d++) s[kt] = mfma32(T(), kf[kt][d], qf[d], s[kt]);
        }
        const bool edge = __any(vis < kb + KB);
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[kt][i] = weight(s[kt][i], a.scale, ls);
        if (edge) {
            const int end = vis - kb - 4 * hi;
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (32 * kt + 8 * (i >> 2) + (i & 3) >= end) s[kt][i] = 0.0f;
        }
#pragma unroll
        for (int kt = 0; kt < KT; kt++) sum[kt] += s[kt];
    }
#pragma unroll
    for (int kt = 0; kt < KT; kt++) {
        // over the 32 lanes of a half: lane l is left with value l / 2 of 16
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = sum[kt][i];
        const float total = reduce_scatter<16, 32>(v, lane);
        const int i = c32 >> 1;
        if (!(lane & 1)) part[wave][32 * kt + 8 * (i >> 2) + 4 * hi + (i & 3)] = total;
    }
    __syncthreads();
    const int key = threadIdx.x;
    if (key >= KB || kb + key >= kend) return;
    const long long at = pool_row(p, r, kvh, kb + key);
    if (at < 0) return;
    float add = 0.0f;
#pragma unroll
    for (int w = 0; w < kMassWaves; w++) add = add + part[w][key];
    p.mass[at] += add;
}

// ---- eviction -------------------------------------------------------------------------

struct EvictArgs {
    Paged p;
    int budget, sink, recent;
    float* mass_out;
    int* pos_out;
    int* count;                // [n_req * nkv]: rows that move
    int* from;                 // [n_req * nkv][most]: cache rows, in pairs
    int* to;
    int most, hd;
    int move_here;             // the selecting workgroup also moves the rows
};

// Order of a mass: larger is larger, zeros alike, a NaN the least number.
__device__ __forceinline__ uint32_t mass_key(float m) {
    if (m != m) return 0u;
    const uint32_t u = __float_as_uint(m == 0.0f ? 0.0f : m);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t kProtected = 0xffffffffu;      // above the key of any mass

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kSelBins = 2048;
constexpr int kSelMoves = 64;      // moves that the selecting workgroup makes itself

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1, 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2, 3
    return v;
}

// Sums of two values over the threads before this one; `sums` is scratch that is
// not in use.
__device__ __forceinline__ int2 sel_scan(int x, int y, int2* sums, int lane, int wave) {
    const int ix = wave_scan(x), iy = wave_scan(y);
    if (lane == 63) sums[wave] = make_int2(ix, iy);
    __syncthreads();
    int2 before = make_int2(ix - x, iy - y);
#pragma unroll
    for (int w = 0; w < kSelWaves; w++) {
        const int2 s = sums[w];
        before.x += w < wave ? s.x : 0;
        before.y += w < wave ? s.y : 0;
    }
    return before;
}

// Row moves by a workgroup; sources lie behind the budget and targets before it,
// so no order is needed.  16 bytes per thread, hd / 8 threads per row.
__device__ __forceinline__ void move_rows(const EvictArgs& a, int r, int h, const int* from, const int* to, int count,
                                          int first, int step) {
    const Paged& p = a.p;
    const int per = a.hd / 8, c = threadIdx.x % per;
    for (int m = first + threadIdx.x / per; m < count; m += step) {
        const long long src = pool_row(p, r, h, from[m]), dst = pool_row(p, r, h, to[m]);
        if (src < 0 || dst < 0) continue;
        const uint4 k = *reinterpret_cast<const uint4*>(p.kp + src * a.hd + 8 * c);
        const uint4 v = *reinterpret_cast<const uint4*>(p.vp + src * a.hd + 8 * c);
        *reinterpret_cast<uint4*>(p.kp + dst * a.hd + 8 * c) = k;
        *reinterpret_cast<uint4*>(p.vp + dst * a.hd + 8 * c) = v;
        if (c == 0) {
            a.mass_out[dst] = p.mass[src];
            a.pos_out[dst] = p.pos[src];
        }
    }
}

// One workgroup per (request, KV head).  A thread owns C consecutive rows (a
// multiple of 4, so that four masses or positions are one load), whose keys it
// keeps in registers; C = 0: as many rows as it takes, read again in each pass.
// The key of the last row that stays comes from a radix selection of 11, 11 and
// 10 bits with histograms in LDS (the first digit is a mass's exponent and two
// bits: 8 bits would put most rows into a few counters; four copies of a counter,
// by lane; protected rows are counted per thread).  One scan over the threads then tells each how many rows before its
// own stay, and with that which gaps and fillers its rows are.
// What bounds it is latency: the chain of loads (length, page, mass) and five
// scans with their barriers.  4 requests x 8 heads of 16384 rows 18 us (and 12 for
// the moves), 32 x 8 of 2049, moves included, 9.2 us.
template <int C>
__global__ __launch_bounds__(kSelThreads) void k_evict_select(EvictArgs a) {
    __shared__ int4 hist[kSelBins];
    __shared__ int2 sums[4][kSelWaves];
    __shared__ int lds_from[kSelMoves], lds_to[kSelMoves];
    __shared__ int s_newest, s_digit, s_left, s_first;
    const Paged& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.x, r = blockIdx.y, item = r * p.nkv + h;
    const int n = min(max(fixed(p.kv_len, r), 0), p.limit);
    const bool over = n > a.budget;
    // a row that stays keeps its place: all rows before the budget are copied, and
    // what is moved into gaps then overwrites them
    if (a.mass_out != p.mass || a.pos_out != p.pos)
        for (int j = tid; j < min(n, a.budget); j += kSelThreads) {
            const long long at = pool_row(p, r, h, j);
            if (at < 0) continue;
            a.mass_out[at] = p.mass[at];
            a.pos_out[at] = p.pos[at];
        }
    if (!over) {
        if (tid == 0) a.count[item] = 0;
        return;
    }
    const int per = C ? C : cdiv4(n, kSelThreads);
    const int j0 = min(tid * per, n), j1 = min(n, j0 + per);

    // four rows from j (a multiple of 4): positions (-1 where there is no row), masses
    auto rows4 = [&](int j, int4& q, float4& m) __attribute__((always_inline)) {
        q = make_int4(-1, -1, -1, -1);
        m = make_float4(0.f, 0.f, 0.f, 0.f);
        const long long at = j < j1 ? pool_row(p, r, h, j) : -1;
        if (at < 0) return;
        q = *reinterpret_cast<const int4*>(p.pos + at);
        m = *reinterpret_cast<const float4*>(p.mass + at);
        if (j + 1 >= j1) q.y = -1;
        if (j + 2 >= j1) q.z = -1;
        if (j + 3 >= j1) q.w = -1;
    };
    if (tid == 0) s_newest = -1;
    for (int b = tid; b < kSelBins; b += kSelThreads) hist[b] = make_int4(0, 0, 0, 0);
    int4 q[C ? C / 4 : 1];
    float4 m[C ? C / 4 : 1];
    int newest = -1;
    if constexpr (C != 0) {
#pragma unroll
        for (int c = 0; c < C / 4; c++) rows4(j0 + 4 * c, q[c], m[c]);
#pragma unroll
        for (int c = 0; c < C / 4; c++) newest = max(newest, max(max(q[c].x, q[c].y), max(q[c].z, q[c].w)));
    } else {
        for (int j = j0; j < j1; j += 4) {
            rows4(j, q[0], m[0]);
            newest = max(newest, max(max(q[0].x, q[0].y), max(q[0].z, q[0].w)));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) newest = max(newest, __shfl_xor(newest, o, kWave));
    __syncthreads();
    if (lane == 0) atomicMax(&s_newest, newest);
    __syncthreads();
    const long long recent = (long long)s_newest - a.recent;
    // (a row on a page that does not exist has the least key; its position is -1)
    auto key_of = [&](int pos, float mass) __attribute__((always_inline)) -> uint32_t {
        if (pos < 0) return 0u;
        return pos < a.sink || pos > recent ? kProtected : mass_key(mass);
    };
    uint32_t key[C ? C : 1];
    if constexpr (C != 0) {
#pragma unroll
        for (int c = 0; c < C / 4; c++) {
            key[4 * c] = key_of(q[c].x, m[c].x);
            key[4 * c + 1] = key_of(q[c].y, m[c].y);
            key[4 * c + 2] = key_of(q[c].z, m[c].z);
            key[4 * c + 3] = key_of(q[c].w, m[c].w);
        }
    }
    // f(row, key) for this thread's rows in order
    auto each = [&](auto f) __attribute__((always_inline)) {
        if constexpr (C != 0) {
#pragma unroll
            for (int c = 0; c < C; c++)
                if (j0 + c < j1) f(j0 + c, key[c]);
        } else {
            for (int j = j0; j < j1; j += 4) {
                rows4(j, q[0], m[0]);
                f(j, key_of(q[0].x, m[0].x));
                if (j + 1 < j1) f(j + 1, key_of(q[0].y, m[0].y));
                if (j + 2 < j1) f(j + 2, key_of(q[0].z, m[0].z));
                if (j + 3 < j1) f(j + 3, key_of(q[0].w, m[0].w));
            }
        }
    };

    // kth: the least key that stays; left: how many rows of that key stay
    uint32_t kth = 0;
    int left = a.budget;
    int* const mine = reinterpret_cast<int*>(hist) + (lane & 3);
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
        const int top = 32 - 11 * pass, bits = pass < 2 ? 11 : 10, shift = top - bits, last = (1 << bits) - 1;
        int safe = 0;
        each([&](int, uint32_t k) {
            if (pass > 0 && (k >> (top & 31)) != (kth >> (top & 31))) return;
            if (k == kProtected) safe++;
            else atomicAdd(mine + 4 * ((k >> shift) & last), 1);
        });
        if (safe) atomicAdd(mine + 4 * last, safe);
        __syncthreads();
        // bins from the largest digit down, two per thread
        const int b1 = kSelBins - 1 - 2 * tid;
        const int4 n1 = hist[b1], n0 = hist[b1 - 1];
        const int c1 = (n1.x + n1.y) + (n1.z + n1.w), c0 = (n0.x + n0.y) + (n0.z + n0.w);
        hist[b1] = hist[b1 - 1] = make_int4(0, 0, 0, 0);
        const int above = sel_scan(c1 + c0, 0, sums[pass], lane, wave).x;
        if (above < left && above + c1 + c0 >= left) {
            const bool second = above + c1 < left;
            s_digit = second ? b1 - 1 : b1;
            s_left = left - above - (second ? c1 : 0);
        }
        __syncthreads();
        kth |= (uint32_t)s_digit << shift;
        left = s_left;
    }
    if (a.budget == 0) kth = kProtected, left = 0;  // (no digit was found: nothing stays)
    int greater = 0, ties = 0;
    each([&](int, uint32_t k) {
        greater += k > kth;
        ties += k == kth;
    });
    const int2 before = sel_scan(ties, greater, sums[3], lane, wave);
    int tie = before.x;
    const int stay0 = before.y + min(tie, left);    // rows before j0 that stay
    // rows before the budget that stay: its thread knows
    {
        int st = stay0, t = tie;
        if (j0 <= a.budget && a.budget < j0 + per) {
            each([&](int j, uint32_t k) { st += j < a.budget && (k > kth || (k == kth && t++ < left)); });
            s_first = st;
        }
    }
    __syncthreads();
    const int first = s_first;
    const size_t list = (size_t)item * a.most;
    int* const from = a.move_here ? lds_from : a.from + list;
    int* const to = a.move_here ? lds_to : a.to + list;
    int st = stay0;
    each([&](int j, uint32_t k) {
        const bool stay = k > kth || (k == kth && tie++ < left);
        if (j < a.budget) {
            if (!stay) to[j - st] = j;
        } else if (stay) {
            from[st - first] = j;
        }
        st += stay;
    });
    const int moves = a.budget - first;
    if (!a.move_here) {
        if (tid == 0) a.count[item] = moves;
        return;
    }
    // the copies above are there before a row is moved
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    move_rows(a, r, h, lds_from, lds_to, moves, 0, kSelThreads / (a.hd / 8));
}

__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a) {
    const int h = blockIdx.y, r = blockIdx.z, rows = 256 / (a.hd / 8);
    const size_t item = (size_t)r * a.p.nkv + h;
    move_rows(a, r, h, a.from + item * a.most, a.to + item * a.most, a.count[item], blockIdx.x * rows, gridDim.x * rows);
}

// ---- shapes -----------------------------------------------------------------------------

// How a batch is cut up.  Short requests: enough workgroups for the chip, but
// splits of at least 256 keys; the others: splits only while there are fewer
// blocks than CUs.
constexpr int kCus = 256;
constexpr int kOneSplit = 512;         // keys that one workgroup of eight waves takes, without a split
constexpr int kSplitBlocks = 1024;
constexpr int kWideJoin = 16;
struct Plan {
    int short_max;
    int tiles, waves, splits, split_keys, short_rows;    // k_paged_attn (tiles 0: not launched)
    long long blocks;
    int chunk_splits, chunk_keys;                        // k_paged_chunk (blocks 0: not launched)
};
Plan attn_plan(const Paged& p) {
    Plan s = {};
    const int limit = p.limit > 0 ? p.limit : 1;
    const long long rows = (long long)p.max_q * p.G;
    s.short_rows = rows < kShort ? (int)rows : kShort;
    // A batch with chunks whose blocks leave CUs free takes its short requests along
    // in them: 67 -> 48 us (now 44) for 24 requests, ten of them with chunks.
    const long long chunk_blocks = (long long)p.n_tokens * p.G / kRows + p.n_req;
    s.short_max = rows > kShort && chunk_blocks * p.nkv <= kCus ? 0 : kShort;
    // With as many rows as all requests can have, none is expected to be short (one
    // that is all the same is taken along).
    if (rows > kShort && (long long)p.n_req * p.max_q <= p.n_tokens) s.short_max = 0;
    if (s.short_max) {
        s.tiles = cdiv(s.short_rows, 16);
        s.waves = limit <= kOneSplit ? 8 : 4;
        long long want = cdiv(kSplitBlocks, (long long)p.n_req * p.nkv * s.tiles);
        const long long most = s.waves == 8 ? 1 : cdiv(limit, 256);
        if (want > most) want = most;
        s.split_keys = cdiv(cdiv(limit, want), 128) * 128;
        s.splits = cdiv(limit, s.split_keys);
    }
    if (rows > kShort) {
        long long n = chunk_blocks;
        const long long each = (long long)p.n_req * cdiv(rows, kRows);
        if (n > each) n = each;
        s.blocks = n;
        long long want = kCus / (n * p.nkv);
        const long long most = cdiv(limit, 512);
        want = want < 1 ? 1 : (want > most ? most : want);
        s.chunk_keys = cdiv(cdiv(limit, want), 128) * 128;
        s.chunk_splits = cdiv(limit, s.chunk_keys);
    }
    return s;
}
size_t short_parts(const Paged& p, const Plan& s) {
    return s.tiles && s.splits > 1 ? (size_t)s.splits * p.n_req * p.nkv * s.short_rows : 0;
}
size_t chunk_parts(const Paged& p, const Plan& s) {
    return s.blocks && s.chunk_splits > 1 ? (size_t)s.chunk_splits * p.n_tokens * p.nq : 0;
}

}  // namespace

#define MDX_PAGED_HD(FN, ...)                                                                     \
    (c->type == MDX_TYPE_F16                                                                      \
         ? (c->head_dim == 64 ? FN<64, _Float16>(__VA_ARGS__)                                     \
                              : c->head_dim == 128 ? FN<128, _Float16>(__VA_ARGS__) : FN<256, _Float16>(__VA_ARGS__)) \
         : (c->head_dim == 64 ? FN<64, __bf16>(__VA_ARGS__)                                       \
                              : c->head_dim == 128 ? FN<128, __bf16>(__VA_ARGS__) : FN<256, __bf16>(__VA_ARGS__)))

namespace {

template <int HD, class T>
void append_launch(const AppendArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((k_paged_append<HD, T>), dim3(a.p.n_tokens), dim3(256), 0, s, a);
}

template <int HD, class T>
void attn_launch(const AttnArgs& a, const Plan& s, hipStream_t st) {
    if (s.blocks) {
        const dim3 blocks((unsigned)(s.blocks * a.p.nkv), s.chunk_splits), threads(HD == 256 ? 256 : 512);
        if (1 << a.p.shift >= kTileKeys<HD>) hipLaunchKernelGGL((k_paged_chunk<HD, T, true>), blocks, threads, 0, st, a);
        else hipLaunchKernelGGL((k_paged_chunk<HD, T, false>), blocks, threads, 0, st, a);
    }
    const dim3 grid(s.splits, a.p.nkv * s.tiles, a.p.n_req);
    if (s.tiles && s.waves == 8) hipLaunchKernelGGL((k_paged_attn<HD, T, 8>), grid, dim3(512), 0, st, a);
    else if (s.tiles) hipLaunchKernelGGL((k_paged_attn<HD, T, 4>), grid, dim3(256), 0, st, a);
    if (chunk_parts(a.p, s))
        hipLaunchKernelGGL((k_paged_join<HD, T, 1>), dim3(cdiv((long long)a.p.n_tokens * a.p.nq, 4)), dim3(256), 0, st, a);
    if (short_parts(a.p, s)) {
        const dim3 rows(s.short_rows, a.p.nkv, a.p.n_req);
        if (s.splits > kWideJoin) hipLaunchKernelGGL((k_paged_join<HD, T, 16>), rows, dim3(1024), 0, st, a);
        else hipLaunchKernelGGL((k_paged_join<HD, T, 4>), rows, dim3(256), 0, st, a);
    }
}

template <int HD, class T>
void mass_launch(const MassArgs& a, hipStream_t s) {
    if ((long long)a.p.max_q * a.p.G <= kMassRows)
        hipLaunchKernelGGL((k_paged_mass<HD, T>), dim3(cdiv(a.p.limit, 64), a.p.nkv, a.p.n_req), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((k_paged_mass_chunk<HD, T>), dim3(cdiv(a.p.limit, HD == 256 ? 32 : 64), a.p.nkv, a.p.n_req),
                           dim3(64 * kMassWaves), 0, s, a);
}

}  // namespace

extern "C" {

int mdx_launch_paged_append(const MdxPagedCache* c, const MdxPagedBatch* b, const float* qkv, long long qkv_stride,
                            const int* positions, const float* q_norm, const float* k_norm, float eps,
                            const float* cos_t, const float* sin_t, int max_pos, int rope_style, void* q_out,
                            long long q_stride, void* stream) {
    AppendArgs a = {};
    a.p = paged(c, b);
    a.qkv = qkv;
    a.qkv_stride = qkv_stride;
    a.positions = positions;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.max_pos = max_pos;
    a.style = rope_style;
    a.q_out = (uint16_t*)q_out;
    a.q_stride = q_stride;
    MDX_PAGED_HD(append_launch, a, (hipStream_t)stream);
    return mdxrt_launched("mdx_paged_append");
}

size_t mdx_paged_attn_scratch(const MdxPagedCache* c, const MdxPagedBatch* b) {
    const Paged p = paged(c, b);
    if (p.max_q == 0) return 0;
    const Plan s = attn_plan(p);
    return (short_parts(p, s) + chunk_parts(p, s)) * ((size_t)c->head_dim * 4 + 8);
}

int mdx_launch_paged_attn(const MdxPagedCache* c, const MdxPagedBatch* b, const void* q, long long q_stride,
                          float scale, void* out, long long out_stride, float* lse, void* scratch, void* stream) {
    AttnArgs a = {};
    a.p = paged(c, b);
    if (a.p.max_q == 0) return 0;
    const Plan s = attn_plan(a.p);
    a.q = (const uint16_t*)q;
    a.q_stride = q_stride;
    a.scale = scale;
    a.c = scale * kLog2e;
    a.out = (uint16_t*)out;
    a.out_stride = out_stride;
    a.lse = lse;
    const size_t ns = short_parts(a.p, s), nc = chunk_parts(a.p, s), hd = c->head_dim;
    a.splits = s.splits;
    a.split_keys = s.split_keys;
    a.short_rows = s.short_rows;
    a.short_max = s.short_max;
    a.chunk_splits = s.chunk_splits;
    a.chunk_keys = s.chunk_keys;
    a.short_o = (float*)scratch;
    a.part_o = a.short_o + ns * hd;
    a.short_ml = (float2*)(a.part_o + nc * hd);
    a.part_ml = a.short_ml + ns;
    if (s.blocks * a.p.nkv > 0x7fffffLL) return mdxrt_refuse(-1, "mdx_paged_attention: too many rows");
    MDX_PAGED_HD(attn_launch, a, s, (hipStream_t)stream);
    return mdxrt_launched("mdx_paged_attention");
}

size_t mdx_paged_mass_scratch(const MdxPagedCache* c, const MdxPagedBatch* b) {
    (void)c;
    (void)b;
    return 0;
}

int mdx_launch_paged_mass(const MdxPagedCache* c, const MdxPagedBatch* b, const void* q, long long q_stride,
                          float scale, const float* lse, void* scratch, void* stream) {
    (void)scratch;
    MassArgs a = {};
    a.p = paged(c, b);
    if (a.p.max_q == 0 || a.p.limit == 0) return 0;
    a.q = (const uint16_t*)q;
    a.q_stride = q_stride;
    a.scale = scale;
    a.lse = lse;
    MDX_PAGED_HD(mass_launch, a, (hipStream_t)stream);
    return mdxrt_launched("mdx_paged_mass");
}

static int evict_most(const Paged& p, int budget) {
    return p.limit <= budget ? 0 : (p.limit - budget < budget ? p.limit - budget : budget);
}

size_t mdx_paged_evict_scratch(const MdxPagedCache* c, const MdxPagedBatch* b, int budget) {
    const Paged p = paged(c, b);
    return (size_t)p.n_req * p.nkv * 4 * (1 + 2 * (size_t)evict_most(p, budget));
}

int mdx_launch_paged_evict(const MdxPagedCache* c, const MdxPagedBatch* b, int budget, int sink, int recent,
                           float* mass_out, int* pos_out, void* scratch, void* stream) {
    EvictArgs a = {};
    a.p = paged(c, b);
    a.budget = budget;
    a.sink = sink;
    a.recent = recent;
    a.mass_out = mass_out;
    a.pos_out = pos_out;
    a.most = evict_most(a.p, budget);
    a.hd = c->head_dim;
    const size_t items = (size_t)a.p.n_req * a.p.nkv;
    a.count = (int*)scratch;
    a.from = a.count + items;
    a.to = a.from + items * a.most;
    hipStream_t s = (hipStream_t)stream;
    a.move_here = a.most <= kSelMoves;
    const dim3 grid(a.p.nkv, a.p.n_req), block(kSelThreads);
    const int per = cdiv(a.p.limit, kSelThreads);
    if (per <= 4) hipLaunchKernelGGL(k_evict_select<4>, grid, block, 0, s, a);
    else if (per <= 16) hipLaunchKernelGGL(k_evict_select<16>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(k_evict_select<0>, grid, block, 0, s, a);
    if (!a.move_here) {
        const int rows = 256 / (a.hd / 8), need = cdiv(a.most, rows);
        hipLaunchKernelGGL(k_evict_move, dim3(need < 64 ? need : 64, a.p.nkv, a.p.n_req), dim3(256), 0, s, a);
    }
    return mdxrt_launched("mdx_paged_evict");
}

}  // extern "C"
