/*
 * paged_q4_attn.hip -- attention over the paged 4-bit K/V cache (layout:
 * paged_q4.h).
 *
 *   s_t = scale * q . k_t,  k_t = d * (code - 8) per group of 32 dims
 *   o   = sum_t exp(s_t) v_t / sum_t exp(s_t)   (times the gate)
 *
 * A wave takes a tile of query columns (rows x heads of one KV head) and walks
 * the keys in steps.  Both products run on v_mfma_f32_16x16x32_f16 with the
 * codes as exact fp16 integers; the scales never meet the codes:
 *   S[g] = K codes . q over the 32 dims of group g,  s = sum_g d_g S[g]
 *   O[dims of g] += V codes . (p * dv_g)
 * so unpacking is and / or / add on packed pairs, and the products are exact.
 * q (normalised by a power of two per column) and p * dv enter as fp16 hi + lo,
 * which keeps ~22 bits: outputs have fp32 accuracy.
 *
 * Running reference per column: p = exp2(s - m), m = top + E - 7 with top a
 * maximum of s (raised when a score passes it by more than 2^8) and 2^E a bound
 * of the V scales met so far: p * dv stays below 2^15 whatever the values' size,
 * and what counts stays far above fp16's smallest numbers.
 */
#include <hip/hip_runtime.h>

#include "kernels.h"
#include "lfm_attn.h"
#include "paged_q4.h"

namespace lfm {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr float kNoScore = -1e30f; /* top before any key: finite, so masked scores (-inf) give p = 0 */
constexpr float kSlack   = 8.0f;   /* log2 by which a score may pass top */
constexpr float kLift    = 7.0f;   /* p * dv < 2^(kSlack + kLift) */

struct GqaParams {
    PagedQ4 c;
    lfm_q4_plan plan;
    const float *q, *gate;
    float *out;
    int gate_is_logit;
    float scale;
};

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

/* The 8 codes of a word as the A operand of one MFMA, exact: code - 8. */
__device__ __forceinline__ half8v unpack(uint32_t w) {
    union {
        uint32_t u[4];
        half2v h[4];
        half8v v;
    } r;
    const half2v b0 = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    const half2v s1 = {(_Float16)0.0625f, (_Float16)0.0625f}, b1 = {(_Float16)-72.0f, (_Float16)-72.0f};
    const uint32_t x = w >> 8;
    r.u[0] = (w & 0x000F000Fu) | 0x64006400u; /* 1024 + code      */
    r.u[1] = (w & 0x00F000F0u) | 0x64006400u; /* 1024 + 16 * code */
    r.u[2] = (x & 0x000F000Fu) | 0x64006400u;
    r.u[3] = (x & 0x00F000F0u) | 0x64006400u;
    r.h[0] = r.h[0] + b0;
    r.h[1] = __builtin_elementwise_fma(r.h[1], s1, b1);
    r.h[2] = r.h[2] + b0;
    r.h[3] = __builtin_elementwise_fma(r.h[3], s1, b1);
    return r.v;
}

__device__ __forceinline__ uint32_t pk_rtz(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}

__device__ __forceinline__ float half_lo(uint32_t w) { return (float)__builtin_bit_cast(half2v, w)[0]; }
__device__ __forceinline__ float half_hi(uint32_t w) { return (float)__builtin_bit_cast(half2v, w)[1]; }

template <int HD> struct Block { /* one lane's share of a block of 32 positions */
    uint4 k[HD / 64], v[HD / 64], ks[HD / 32], vs[HD / 32];
};

template <int HD> __device__ __forceinline__ void load_block(Block<HD> &b, const uint8_t *base, uint32_t lane) {
    const uint32_t kg = lane >> 4;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i) {
        b.k[i] = *reinterpret_cast<const uint4 *>(base + i * 1024 + lane * 16u);
        b.v[i] = *reinterpret_cast<const uint4 *>(base + 16 * HD + i * 1024 + lane * 16u);
    }
#pragma unroll
    for (int g = 0; g < HD / 32; ++g) {
        b.ks[g] = *reinterpret_cast<const uint4 *>(base + 32 * HD + g * 64 + kg * 16u);
        b.vs[g] = *reinterpret_cast<const uint4 *>(base + 34 * HD + g * 64 + kg * 16u);
    }
}

__device__ __forceinline__ uint32_t word_of(const uint4 &v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

/* One wave: columns of one tile over all its keys. */
template <int HD> __global__ __launch_bounds__(256) void k_paged_gqa(const GqaParams p) {
    constexpr int G = HD / 32, DT = HD / 16;
    const PagedQ4 &c     = p.c;
    const uint32_t lane  = threadIdx.x & 63u, col = lane & 15u, kg = lane >> 4;
    const uint32_t unit  = uniform(blockIdx.x * 4u + (threadIdx.x >> 6));
    const uint32_t h     = unit % c.n_head_kv, sc = unit / c.n_head_kv;
    const uint32_t s     = sc / p.plan.n_ct, ct = sc - s * p.plan.n_ct;
    if (s >= c.n_seq) return;
    const uint32_t pos0 = uniform(c.pos0[s]);
    const uint32_t rows = lfm_q4_rows(pos0, c.rows_seq ? uniform(c.rows_seq[s]) : c.n_rows, c.n_rows, c.capacity);
    const lfm_q4_tile t = lfm_q4_tile_of(&p.plan, pos0, rows, ct);
    if (t.n_steps == 0u) return;

    /* this lane's column */
    const uint32_t mul = p.plan.kv_mul, n_q = c.n_head_kv * mul;
    const uint32_t ci = ct * p.plan.cols + col, row = ci / mul;
    const bool live   = ci < rows * mul;
    const size_t head = ((size_t)s * c.n_rows + row) * n_q + h * mul + (ci - row * mul);
    const uint32_t lo = live ? lfm_q4_row_lo(pos0 + row, p.plan.window) : 0u, hi = live ? pos0 + row + 1u : 0u;

    half8v qh[G], ql[G];
    float cs;
    {
        float x[G][8];
        float big = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (live) a = reinterpret_cast<const float4 *>(p.q + head * HD)[g * 8 + kg * 2u + i];
                x[g][4 * i] = a.x; x[g][4 * i + 1] = a.y; x[g][4 * i + 2] = a.z; x[g][4 * i + 3] = a.w;
                big = fmaxf(big, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))));
            }
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        const int e = big > 0.0f && big < __builtin_inff() ? __builtin_amdgcn_frexp_expf(big) : 0;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = ldexpf(x[g][i], -e);
                qh[g][i]      = (_Float16)y;
                ql[g][i]      = (_Float16)(y - (float)qh[g][i]);
            }
        cs = ldexpf(p.scale * 1.4426950408889634f, e);
    }

    float4v o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    float top = kNoScore, m = kNoScore, l = 0.0f;
    uint32_t vmax = 0u; /* magnitude (fp16 bits) of the V scales that m covers */

    const int32_t *table = c.table + (size_t)s * c.table_stride;
    for (uint32_t step = t.step0; step < t.step0 + t.n_steps; ++step) {
        const int32_t id  = table[step >> c.blk_shift];
        const uint32_t in = step & ((1u << c.blk_shift) - 1u);
        if ((uint32_t)id >= c.n_pages) continue; /* no page: nothing to attend */
        const uint8_t *base = c.pages + (uint64_t)(uint32_t)id * c.page_bytes +
                              (uint64_t)((h << c.blk_shift) + in) * lfm_q4_block_bytes(HD);
        Block<HD> b;
        load_block<HD>(b, base, lane);

        float sv[8]; /* keys 32 step + 4 kg + i (i < 4) and 16 further */
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float4v acc[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t w = HD == 64 ? word_of(b.k[0], half * 2 + g) : word_of(b.k[half % (HD / 64)], g);
                const half8v a   = unpack(w);
                acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[g], float4v{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
                acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[g], acc[g], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = 0.0f;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t d = word_of(b.ks[g], half * 2 + i / 2);
                    x                = fmaf(i & 1 ? half_hi(d) : half_lo(d), acc[g][i], x);
                }
                const uint32_t key = step * 32u + half * 16u + kg * 4u + i;
                sv[half * 4 + i]   = key >= lo && key < hi ? x * cs : -__builtin_inff();
            }
        }
        float best = sv[0];
        uint32_t dv = 0u;
#pragma unroll
        for (int i = 1; i < 8; ++i) best = fmaxf(best, sv[i]);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t d = (word_of(b.vs[g], i / 2) >> (16 * (i & 1))) & 0x7FFFu;
                dv               = max(dv, sv[i] > -__builtin_inff() && d < 0x7C00u ? d : 0u);
            }
        if (__any(best > top + kSlack || dv > vmax)) {
            best = fmaxf(best, __shfl_xor(best, 16));
            best = fmaxf(best, __shfl_xor(best, 32));
            dv   = max(dv, (uint32_t)__shfl_xor((int)dv, 16));
            dv   = max(dv, (uint32_t)__shfl_xor((int)dv, 32));
            vmax = max(dv, vmax);
            top  = fmaxf(top, best);
            const float d = (float)__builtin_bit_cast(_Float16, (uint16_t)vmax);
            const float n = top + (d > 0.0f ? (float)__builtin_amdgcn_frexp_expf(d) : 0.0f) - kLift;
            const float a = __builtin_amdgcn_exp2f(m - n);
            l *= a;
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= a;
            m = n;
        }
        float pr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            pr[i] = __builtin_amdgcn_exp2f(sv[i] - m);
            l += pr[i];
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            union {
                uint32_t u[4];
                half8v v;
            } wh, wl;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t d = word_of(b.vs[g], i);
                const float a = sv[2 * i] > -__builtin_inff() ? pr[2 * i] * half_lo(d) : 0.0f;
                const float z = sv[2 * i + 1] > -__builtin_inff() ? pr[2 * i + 1] * half_hi(d) : 0.0f;
                wh.u[i]       = pk_rtz(a, z);
                wl.u[i]       = pk_rtz(a - half_lo(wh.u[i]), z - half_hi(wh.u[i]));
            }
#pragma unroll
            for (int i = 2 * g; i < 2 * g + 2; ++i) {
                const half8v a = unpack(word_of(b.v[i / 4], i & 3));
                o[i]           = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wl.v, o[i], 0, 0, 0);
                o[i]           = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wh.v, o[i], 0, 0, 0);
            }
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (!live) return;
    float f = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l); /* no key: 0; NaN stays */
    if (p.gate) {
        const float x = p.gate[head];
        f *= p.gate_is_logit ? 1.0f / (1.0f + expf(-x)) : x;
    }
#pragma unroll
    for (int i = 0; i < DT; ++i)
        reinterpret_cast<float4 *>(p.out + head * HD)[i * 4 + kg] =
            make_float4(o[i][0] * f, o[i][1] * f, o[i][2] * f, o[i][3] * f);
}

} // namespace

int paged_q4_gqa_workspace(uint32_t n_seq, uint32_t n_rows, uint32_t keys_hint, uint32_t n_head_q, uint32_t n_head_kv,
                           uint32_t head_dim, uint32_t capacity, uint32_t window, size_t *bytes) {
    (void)keys_hint, (void)head_dim, (void)capacity, (void)window;
    const uint64_t cols = (uint64_t)n_rows * (n_head_q / n_head_kv);
    if (cols > 0x7FFFFFFFull || (cols + 15u) / 16u * n_seq > 0x7FFFFFFFull / n_head_kv) return LFM_ATTN_E_UNSUPPORTED;
    *bytes = 0;
    return LFM_ATTN_OK;
}

int launch_paged_q4_gqa(const PagedQ4 &c, const float *q, const float *gate, int gate_is_logit, float *out,
                        uint32_t n_head_q, uint32_t keys_hint, uint32_t window, float scale, void *workspace,
                        hipStream_t stream) {
    (void)keys_hint, (void)workspace;
    GqaParams p;
    p.c              = c;
    p.plan.n_seq     = c.n_seq;
    p.plan.n_rows    = c.n_rows;
    p.plan.kv_mul    = n_head_q / c.n_head_kv;
    p.plan.n_head_kv = c.n_head_kv;
    p.plan.window    = window;
    p.plan.capacity  = c.capacity;
    p.plan.cols      = 16u;
    p.plan.step      = 32u;
    p.plan.n_ct      = (c.n_rows * p.plan.kv_mul + 15u) / 16u;
    p.plan.min_steps = 1u;
    p.plan.n_waves   = 0u;
    p.q              = q;
    p.gate           = gate;
    p.out            = out;
    p.gate_is_logit  = gate_is_logit;
    p.scale          = scale;
    const uint64_t units = (uint64_t)c.n_seq * p.plan.n_ct * c.n_head_kv;
    const dim3 grid((uint32_t)((units + 3u) / 4u));
    if (c.head_dim == 64u)
        hipLaunchKernelGGL(k_paged_gqa<64>, grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL(k_paged_gqa<128>, grid, dim3(256), 0, stream, p);
    return hip_status(hipGetLastError());
}

} // namespace lfm
