/*
 * paged_q4.hip -- rows into and out of the paged 4-bit K/V cache (layout:
 * paged_q4.h).
 *
 * Append, per row and head (k and q; v is only quantized):
 *   y = x / sqrt(mean(x^2) + eps) * w,
 *   (y_i, y_{i+D/2}) -> (y_i c - y_{i+D/2} s, y_{i+D/2} c + y_i s)
 * in 64 bits, rounded once to fp32; then per group of 32 dims, with m the
 * value of largest magnitude (the positive one of two),
 *   d = fp16(-m / 8),  code = clamp(floor(x / d + 8.5), 0, 15)
 * with the fp32 quotient and sum.  So the codes do not depend on the order
 * in which the squares are added.  A group with a value that is not finite
 * keeps a NaN scale: it reads back as NaN, and as nothing where it is masked.
 *
 * One workgroup per (sequence, block of 32 positions, KV head): keys are
 * whole words of their own; a value word holds 8 positions of one dim, so the
 * codes meet in LDS and the positions that this call does not store keep
 * their nibbles (read, merge, write by one thread).  Further workgroups rotate
 * the queries; 8 * D / 64 lanes work on a head.  HBM-bound: 2 x 3001 rows, 16
 * query and 4 KV heads of 128 dims, 142 MB in 26 us, 5.4 TB/s (a large copy
 * reaches 5.1); 64 single rows of 32 and 8 heads of 64 take 6 us, a launch and
 * three dependent trips to memory (position, page id, block).
 *
 * Gather: one workgroup per (sequence, block, KV head) stages the block in LDS,
 * so that it is read in whole lines and written as rows.  32 ragged sequences of
 * up to 4100 positions, 4 KV heads of 128: 196 MB in 31 us, 6.3 TB/s.
 */
#include <hip/hip_runtime.h>

#include "kernels.h"
#include "lfm_attn.h"
#include "paged_q4.h"

namespace lfm {
namespace {

struct AppendParams {
    PagedQ4 c;
    const float *q, *k, *v;
    float *q_out;
    const float *qw, *kw, *cos_lut, *sin_lut;
    double eps;
    uint32_t reach;   /* positions that table and rotation table both reach */
    uint32_t n_blk;   /* blocks that n_rows consecutive positions can meet  */
    uint32_t n_head_q;
    uint32_t n_kv_wg; /* workgroups of the K/V part                         */
};

__device__ __forceinline__ uint32_t seq_rows(const PagedQ4 &c, uint32_t s, uint32_t pos0, uint32_t reach) {
    return lfm_q4_rows(pos0, c.rows_seq ? c.rows_seq[s] : c.n_rows, c.n_rows, reach);
}

/* Block `blk` of KV head h of sequence s, or null where the table has no page. */
__device__ __forceinline__ uint8_t *block_at(const PagedQ4 &c, uint32_t s, uint32_t blk, uint32_t h) {
    const int32_t id = c.table[(size_t)s * c.table_stride + (blk >> c.blk_shift)];
    if ((uint32_t)id >= c.n_pages) return nullptr;
    const uint32_t in = blk & ((1u << c.blk_shift) - 1u);
    return c.pages + (uint64_t)(uint32_t)id * c.page_bytes +
           (uint64_t)((h << c.blk_shift) + in) * lfm_q4_block_bytes(c.head_dim);
}

struct Dims8 { /* 4 dims and their rotation partners, D / 2 further */
    float lo[4], hi[4];
};

template <int HD> __device__ __forceinline__ Dims8 load8(const float *head, uint32_t i) {
    Dims8 r;
    const float4 a = reinterpret_cast<const float4 *>(head)[i], b = reinterpret_cast<const float4 *>(head + HD / 2)[i];
    r.lo[0] = a.x; r.lo[1] = a.y; r.lo[2] = a.z; r.lo[3] = a.w;
    r.hi[0] = b.x; r.hi[1] = b.y; r.hi[2] = b.z; r.hi[3] = b.w;
    return r;
}

/* Norm (w null: none) and rotation of a head held by HD / 8 adjacent lanes. */
template <int HD>
__device__ __forceinline__ void norm_rope(Dims8 &x, const float *w, double eps, const float *cos_row,
                                          const float *sin_row, uint32_t i) {
    double lo[4], hi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) lo[j] = (double)x.lo[j], hi[j] = (double)x.hi[j];
    if (w) {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) s = fma(lo[j], lo[j], fma(hi[j], hi[j], s));
#pragma unroll
        for (int o = HD / 16; o > 0; o >>= 1) s += __shfl_xor(s, o);
        const double r   = 1.0 / sqrt(s / (double)HD + eps);
        const Dims8 norm = load8<HD>(w, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = lo[j] * r * (double)norm.lo[j], hi[j] = hi[j] * r * (double)norm.hi[j];
    }
    const float4 c4 = reinterpret_cast<const float4 *>(cos_row)[i], s4 = reinterpret_cast<const float4 *>(sin_row)[i];
    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x.lo[j] = (float)(lo[j] * (double)c[j] - hi[j] * (double)s[j]);
        x.hi[j] = (float)(hi[j] * (double)c[j] + lo[j] * (double)s[j]);
    }
}

/* Codes (4 dims per lane) and the fp16 scale of a group of 32 dims held by 8
 * adjacent lanes. */
__device__ __forceinline__ uint16_t quant_group(const float x[4], uint32_t code[4]) {
    float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    float low = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
    uint32_t mag = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) mag = max(mag, __float_as_uint(x[j]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor(top, o));
        low = fminf(low, __shfl_xor(low, o));
        mag = max(mag, (uint32_t)__shfl_xor((int)mag, o));
    }
    const _Float16 d16 = (_Float16)((top >= -low ? top : low) / -8.0f);
    const float d      = (float)d16;
    const bool finite  = mag < 0x7F800000u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float t = x[j] / d + 8.5f;
        code[j]       = finite && d != 0.0f ? (uint32_t)fminf(fmaxf(floorf(t), 0.0f), 15.0f) : 8u;
    }
    return !finite ? (uint16_t)0x7E00u : d == 0.0f ? (uint16_t)0u : __builtin_bit_cast(uint16_t, d16);
}

/* The word of 8 dims: this lane holds dims 0-3 (even lane) or 4-7 (odd). */
__device__ __forceinline__ uint32_t pack_word(const uint32_t code[4], uint32_t lane) {
    uint32_t w = 0u;
#pragma unroll
    for (uint32_t j = 0; j < 4u; ++j) w |= code[j] << (4u * lfm_q4_nibble(j));
    w <<= (lane & 1u) * 8u; /* nibble of element e + 4 is nibble of e, plus 2 */
    return w | (uint32_t)__shfl_xor((int)w, 1);
}

template <int HD> __device__ void append_kv(const AppendParams &p, uint8_t *codes) {
    constexpr uint32_t L = HD / 8, TPP = 256u / L; /* lanes per head, positions per pass of the workgroup */
    const PagedQ4 &c = p.c;
    const uint32_t h = blockIdx.x % c.n_head_kv, rest = blockIdx.x / c.n_head_kv;
    const uint32_t s = rest / p.n_blk, bi = rest - s * p.n_blk;
    const uint32_t pos0 = c.pos0[s], rows = seq_rows(c, s, pos0, p.reach);
    if (rows == 0u) return;
    const uint32_t blk = pos0 / 32u + bi;
    if (blk > (pos0 + rows - 1u) / 32u) return;
    uint8_t *base = block_at(c, s, blk, h);
    if (!base) return;
    /* positions [t0, t1) of the block */
    const uint32_t t0 = bi == 0u ? pos0 % 32u : 0u;
    const uint32_t t1 = min(32u, pos0 + rows - blk * 32u);
    const uint32_t i = threadIdx.x % L, lane = threadIdx.x & 63u;
    for (uint32_t t = t0 + threadIdx.x / L; t < t1; t += TPP) {
        const uint32_t pos = blk * 32u + t;
        const size_t head  = (((size_t)s * c.n_rows + (pos - pos0)) * c.n_head_kv + h) * HD;
        Dims8 x            = load8<HD>(p.k + head, i);
        const Dims8 y      = load8<HD>(p.v + head, i);
        norm_rope<HD>(x, p.kw, p.eps, p.cos_lut + (size_t)pos * (HD / 2), p.sin_lut + (size_t)pos * (HD / 2), i);
#pragma unroll
        for (uint32_t hi = 0; hi < 2u; ++hi) {
            uint32_t code[4];
            const uint32_t g  = hi * (HD / 64) + i / 8u;
            const uint16_t kd = quant_group(hi ? x.hi : x.lo, code);
            const uint32_t w  = pack_word(code, lane);
            if ((lane & 1u) == hi)
                *reinterpret_cast<uint32_t *>(base + lfm_q4_k_word(HD, t, g, (i & 7u) >> 1)) = w;
            const uint16_t vd = quant_group(hi ? y.hi : y.lo, code);
            if ((i & 7u) == 0u) {
                *reinterpret_cast<uint16_t *>(base + lfm_q4_scale(HD, 0u, t, g)) = kd;
                *reinterpret_cast<uint16_t *>(base + lfm_q4_scale(HD, 1u, t, g)) = vd;
            }
            *reinterpret_cast<uint32_t *>(codes + t * HD + hi * (HD / 2) + 4u * i) =
                code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
        }
    }
    __syncthreads();
    for (uint32_t w = threadIdx.x; w < 4u * HD; w += 256u) {
        const uint32_t kg = w / HD, x = w % HD;
        uint32_t word = 0u, mine = 0u;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
            const uint32_t t = 4u * kg + (e & 3u) + 16u * (e >> 2);
            if (t >= t0 && t < t1) {
                word |= (uint32_t)codes[t * HD + x] << (4u * lfm_q4_nibble(e));
                mine |= 15u << (4u * lfm_q4_nibble(e));
            }
        }
        if (mine == 0u) continue;
        uint32_t *at = reinterpret_cast<uint32_t *>(base + lfm_q4_v_word(HD, kg, x));
        *at          = mine == 0xFFFFFFFFu ? word : (*at & ~mine) | word;
    }
}

template <int HD> __device__ void rotate_q(const AppendParams &p) {
    constexpr uint32_t L = HD / 8;
    const PagedQ4 &c = p.c;
    const uint64_t head = (uint64_t)(blockIdx.x - p.n_kv_wg) * (256u / L) + threadIdx.x / L;
    const uint64_t row = head / p.n_head_q;
    const uint32_t s = (uint32_t)(row / c.n_rows), r = (uint32_t)(row % c.n_rows);
    if (s >= c.n_seq) return; /* whole groups of L lanes leave together */
    const uint32_t pos0 = c.pos0[s];
    if (r >= seq_rows(c, s, pos0, p.reach)) return;
    const uint32_t i = threadIdx.x % L;
    const size_t pos = (size_t)pos0 + r;
    Dims8 x = load8<HD>(p.q + head * HD, i);
    norm_rope<HD>(x, p.qw, p.eps, p.cos_lut + pos * (HD / 2), p.sin_lut + pos * (HD / 2), i);
    float4 *out     = reinterpret_cast<float4 *>(p.q_out + head * HD);
    out[i]          = make_float4(x.lo[0], x.lo[1], x.lo[2], x.lo[3]);
    out[HD / 8 + i] = make_float4(x.hi[0], x.hi[1], x.hi[2], x.hi[3]);
}

template <int HD> __global__ __launch_bounds__(256) void k_paged_append(const AppendParams p) {
    __shared__ __align__(16) uint8_t codes[32 * HD];
    if (blockIdx.x < p.n_kv_wg)
        append_kv<HD>(p, codes);
    else
        rotate_q<HD>(p);
}

struct GatherParams {
    PagedQ4 c;
    uint16_t *k_out, *v_out;
    uint32_t capacity, n_blk;
};

__device__ __forceinline__ uint32_t half_of(uint32_t code, float d) {
    return __builtin_bit_cast(uint16_t, (_Float16)(d * ((float)code - 8.0f)));
}

/* One workgroup per (sequence, block, KV head).  The block comes to LDS whole, in
 * 16-byte loads; a thread then unpacks 8 dims of a position: of the keys one
 * word, of the values a nibble of each of 8 words. */
template <int HD> __global__ __launch_bounds__(256) void k_paged_gather(const GatherParams p) {
    __shared__ __align__(16) uint8_t blk_lds[36 * HD];
    const PagedQ4 &c = p.c;
    const uint32_t h = blockIdx.x % c.n_head_kv, rest = blockIdx.x / c.n_head_kv;
    const uint32_t s = rest / p.n_blk, bi = rest - s * p.n_blk;
    const uint32_t pos0 = c.pos0[s], rows = seq_rows(c, s, pos0, p.capacity);
    if (rows == 0u) return;
    const uint32_t blk = pos0 / 32u + bi;
    if (blk > (pos0 + rows - 1u) / 32u) return;
    const uint8_t *base = block_at(c, s, blk, h);
    for (uint32_t i = threadIdx.x; i < 36u * HD / 16u; i += 256u)
        reinterpret_cast<uint4 *>(blk_lds)[i] = base ? reinterpret_cast<const uint4 *>(base)[i] : make_uint4(0u, 0u, 0u, 0u);
    __syncthreads(); /* without a page: scales 0, so zeros */
    const uint32_t t0 = bi == 0u ? pos0 % 32u : 0u;
    const uint32_t t1 = min(32u, pos0 + rows - blk * 32u);
    for (uint32_t w = threadIdx.x; w < 4u * HD; w += 256u) {
        const uint32_t t = w / (HD / 8), part = w % (HD / 8), g = part / 4u;
        if (t < t0 || t >= t1) continue;
        const uint32_t kw = *reinterpret_cast<const uint32_t *>(blk_lds + lfm_q4_k_word(HD, t, g, part & 3u));
        const float kd = (float)*reinterpret_cast<const _Float16 *>(blk_lds + lfm_q4_scale(HD, 0u, t, g));
        const float vd = (float)*reinterpret_cast<const _Float16 *>(blk_lds + lfm_q4_scale(HD, 1u, t, g));
        const uint32_t vs = 4u * lfm_q4_nibble(lfm_q4_elem(t));
        uint32_t k[4], v[4];
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
            const uint32_t vw =
                *reinterpret_cast<const uint32_t *>(blk_lds + lfm_q4_v_word(HD, lfm_q4_kg(t), 8u * part + e));
            const uint32_t a = half_of((kw >> (4u * lfm_q4_nibble(e))) & 15u, kd);
            const uint32_t b = half_of((vw >> vs) & 15u, vd);
            k[e / 2u] = e & 1u ? k[e / 2u] | a << 16 : a;
            v[e / 2u] = e & 1u ? v[e / 2u] | b << 16 : b;
        }
        const size_t at = (((size_t)s * c.n_rows + (blk * 32u + t - pos0)) * c.n_head_kv + h) * (HD / 8) + part;
        reinterpret_cast<uint4 *>(p.k_out)[at] = make_uint4(k[0], k[1], k[2], k[3]);
        reinterpret_cast<uint4 *>(p.v_out)[at] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

uint32_t blocks_met(uint32_t n_rows) { return (n_rows + 30u) / 32u + 1u; }

} // namespace

bool paged_q4_append_fits(const PagedQ4 &c, uint32_t n_head_q) {
    /* of 256 threads each: a launch's threads are 32 bits */
    const uint64_t limit = 1ull << 24, heads = 256u / (c.head_dim / 8u);
    uint64_t kv, q;
    if (__builtin_mul_overflow((uint64_t)c.n_seq * blocks_met(c.n_rows), (uint64_t)c.n_head_kv, &kv) ||
        __builtin_mul_overflow((uint64_t)c.n_seq * c.n_rows, (uint64_t)n_head_q, &q))
        return false;
    return kv < limit && q < limit * heads && kv + (q + heads - 1u) / heads < limit;
}

int launch_paged_q4_append(const PagedQ4 &c, const float *q, const float *k, const float *v, float *q_out,
                           uint32_t n_head_q, const float *q_norm_w, const float *k_norm_w, float eps,
                           const float *cos_lut, const float *sin_lut, uint32_t lut_rows, hipStream_t stream) {
    AppendParams p;
    p.c        = c;
    p.q        = q;
    p.k        = k;
    p.v        = v;
    p.q_out    = q_out;
    p.qw       = q_norm_w;
    p.kw       = k_norm_w;
    p.cos_lut  = cos_lut;
    p.sin_lut  = sin_lut;
    p.eps      = (double)eps;
    p.reach    = lut_rows < c.capacity ? lut_rows : c.capacity;
    p.n_blk    = blocks_met(c.n_rows);
    p.n_head_q = n_head_q;
    p.n_kv_wg  = c.n_seq * p.n_blk * c.n_head_kv;
    const uint32_t per_wg = 256u / (c.head_dim / 8u);
    const uint32_t q_wg =
        q ? (uint32_t)(((uint64_t)c.n_seq * c.n_rows * n_head_q + per_wg - 1u) / per_wg) : 0u;
    const dim3 grid(p.n_kv_wg + q_wg);
    if (c.head_dim == 64u)
        hipLaunchKernelGGL(k_paged_append<64>, grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL(k_paged_append<128>, grid, dim3(256), 0, stream, p);
    return hip_status(hipGetLastError());
}

int launch_paged_q4_gather(const PagedQ4 &c, uint16_t *k_out, uint16_t *v_out, hipStream_t stream) {
    GatherParams p;
    p.c        = c;
    p.k_out    = k_out;
    p.v_out    = v_out;
    p.capacity = c.capacity;
    p.n_blk    = blocks_met(c.n_rows);
    const dim3 grid(c.n_seq * p.n_blk * c.n_head_kv);
    if (c.head_dim == 64u)
        hipLaunchKernelGGL(k_paged_gather<64>, grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL(k_paged_gather<128>, grid, dim3(256), 0, stream, p);
    return hip_status(hipGetLastError());
}

} // namespace lfm
