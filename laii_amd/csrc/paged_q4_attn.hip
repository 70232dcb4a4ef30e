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
 *
 * What bounds it.  A position and KV head is 1.125 HD bytes, so long decodes are
 * close to the memory: 32 sequences of 32768 keys, head_dim 128, 604 MB in 118 us,
 * 5.1 TB/s (a large copy reaches 5.1, reading alone 7.0); 64 ragged ones of up to
 * 8192, head_dim 64, 171 MB in 43 us, of which 4.6 us are the merge and about 7 the
 * first loads.  There loads alone take 94 us of 604 MB and the arithmetic alone 91.
 * With more columns it is the vector unit: a step of 32 keys and 32 columns is 178
 * vector instructions beside 32 MFMAs, and the prompts (4 ragged of 1999 rows from
 * position 1023, 80.7 GFLOP in 348 us) reach 232 TFLOP/s of the formula's work, 464
 * with the lo products, where a large matrix product reaches 1176.  Tried and no
 * faster: 3 waves per SIMD, other orders of the MFMAs and a schedule that spreads
 * them, loads further ahead, workgroups of 8 waves in a split, weights formed in
 * packed fp16.
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
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));

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
    /* split: first and last workgroup of each unit, partial outputs
     * [slot][cols][HD], their (m, l) [slot][cols] */
    uint2 *range;
    float *part_o;
    float2 *part_ml;
};

/* Sum and maximum over the 4 lanes 16 apart, which share a column: the swaps
 * give both halves' values to every lane, in whatever order. */
__device__ __forceinline__ float kg_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x      = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r      = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float kg_max(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x      = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r      = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ uint32_t kg_max(uint32_t x) {
    auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x      = max((uint32_t)r[0], (uint32_t)r[1]);
    r      = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return max((uint32_t)r[0], (uint32_t)r[1]);
}

/* The same over the two lanes 32 apart. */
__device__ __forceinline__ float pair_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float pair_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

/* x of the lane N further round its row of 16. */
template <int N> __device__ __forceinline__ float row_ror(float x) {
    return __uint_as_float(
        (uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), 0x120 + N, 0xF, 0xF, true));
}
/* Sum and maximum over the R copies of a column, 16 / R lanes apart in a row. */
template <int R> __device__ __forceinline__ float copies_sum(float x) {
    static_assert(R == 2 || R == 4, "copies");
    if (R == 4) x += row_ror<4>(x);
    return x + row_ror<8>(x);
}
template <int R> __device__ __forceinline__ float copies_max(float x) {
    static_assert(R == 2 || R == 4, "copies");
    if (R == 4) x = fmaxf(x, row_ror<4>(x));
    return fmaxf(x, row_ror<8>(x));
}

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

/* Constants of the unpacking.  In vector registers: an AND of two vector
 * registers takes 2.6 cycles of a SIMD with two waves, with a scalar one 4.4. */
struct Magic {
    uint32_t low, high; /* nibble 0 and nibble 1 of both halves */
    half2v up0, up1, less8;
    float zero; /* keeps p * d one mixed-precision fma */
};
__device__ __forceinline__ uint32_t in_vgpr(uint32_t x) {
    uint32_t r;
    asm("v_mov_b32 %0, %1" : "=v"(r) : "s"(x));
    return r;
}
__device__ __forceinline__ Magic magic() {
    Magic m;
    m.low   = in_vgpr(0x000F000Fu);
    m.high  = in_vgpr(0x00F000F0u);
    m.up0   = __builtin_bit_cast(half2v, in_vgpr(0x78007800u)); /* 2^15  */
    m.up1   = __builtin_bit_cast(half2v, in_vgpr(0x68006800u)); /* 2^11  */
    m.less8 = __builtin_bit_cast(half2v, in_vgpr(0xA400A400u)); /* -2^-6 */
    m.zero  = __uint_as_float(in_vgpr(0u));
    return m;
}

union Words {
    uint32_t u[4];
    half2v h[4];
    half8v v;
};

/* The 8 codes of a V word as the A operand of one MFMA: 2^-9 (code - 8), exact.
 * A nibble alone is the fp16 subnormal code * 2^-24 (or 2^-20), so an AND and a
 * packed fma do: 7.2 cycles a pair where setting an exponent by and-or and
 * subtracting it takes 9.1. */
constexpr float kVUp = 512.0f;
__device__ __forceinline__ half8v unpack_v(uint32_t w, const Magic &k) {
    Words r;
    const uint32_t x = w >> 8;
    r.u[0] = w & k.low;
    r.u[1] = w & k.high;
    r.u[2] = x & k.low;
    r.u[3] = x & k.high;
    r.h[0] = __builtin_elementwise_fma(r.h[0], k.up0, k.less8);
    r.h[1] = __builtin_elementwise_fma(r.h[1], k.up1, k.less8);
    r.h[2] = __builtin_elementwise_fma(r.h[2], k.up0, k.less8);
    r.h[3] = __builtin_elementwise_fma(r.h[3], k.up1, k.less8);
    return r.v;
}

/* A K word as 2^-20 code: subnormals, as they stand.  The product with q starts
 * from -8 times the sum of q, so it is that of code - 8; the values' long sums
 * would lose bits to such an offset, these of 32 terms do not.  (rms error of a
 * group's product on the matrix unit, of its rms: 7.6e-8 with code - 8, 1.8e-7
 * with subnormals in bits 6-9, 1.0e-6 with half the codes as code + 64, 4e-6
 * with subnormals that leave up to 9 bits of the mantissa empty.) */
constexpr int kKDown = 20;
__device__ __forceinline__ half8v unpack_k(uint32_t w, const Magic &k) {
    Words r;
    r.u[0] = (w << 4) & k.high;
    r.u[1] = w & k.high;
    r.u[2] = (w >> 4) & k.high;
    r.u[3] = (w >> 8) & k.high;
    return r.v;
}

__device__ __forceinline__ float half_lo(uint32_t w) { return (float)__builtin_bit_cast(half2v, w)[0]; }
__device__ __forceinline__ float half_hi(uint32_t w) { return (float)__builtin_bit_cast(half2v, w)[1]; }

/* Two weights p * d as fp16 hi + lo: hi is the product truncated, lo what is
 * left of it, truncated.  (v_fma_mixlo_f16 would round in one instruction, but
 * takes 8.5 cycles; this takes 28 a pair, that 34.) */
__device__ __forceinline__ void split_weights(float p0, float p1, uint32_t d, uint32_t *hi, uint32_t *lo,
                                              const Magic &k) {
    const float w0 = fmaf(p0, half_lo(d), k.zero), w1 = fmaf(p1, half_hi(d), k.zero);
    *hi            = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(w0, w1));
    const float l0 = fmaf(p0, half_lo(d), -half_lo(*hi)), l1 = fmaf(p1, half_hi(d), -half_hi(*hi));
    *lo            = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(l0, l1));
}

/* What one wave computes with.  HD: head_dim.  NT: tiles of 16 query columns.
 * R: with at most 16 / R columns (NT 1), each is held R times, and copy u of it
 * takes every R-th 16-key tile of a step: softmax work shrinks by R.  The query
 * operand is kept R times, zero outside copy r's columns, so that the S product of
 * tile t with copy t % R leaves each column the tile that it takes, with no
 * selection.  NB: blocks of 32 keys per step.  Registers are cut for two waves
 * per SIMD. */
template <int HD_, int NT_, int R_, int NB_> struct Form {
    static constexpr int HD = HD_, NT = NT_, R = R_, NB = NB_;
    static constexpr int G = HD / 32, DT = HD / 16, TILES = 2 * NB, J = TILES / R;
    static constexpr int COLS = R > 1 ? 16 / R : 16 * NT, STEP = 32 * NB;
    static constexpr int SB = J > 1 ? NB : 1; /* scales: 8 per block and group, or the 4 of this lane's tile */
    static constexpr int SW = J > 1 ? 4 : 2;
    static_assert(R == 1 || (NT == 1 && J == 1), "a copy takes one tile per step");
};

/* One lane's share of a step's codes and scales, keys or values.  Native
 * vectors: a load in flight stays one value through the loop (as four, the
 * compiler moved some at the loop's end, and waited for them to do so). */
template <class F> struct Half {
    uint4v c[F::NB][F::HD / 64];
    uint4v s[F::SB][F::G * F::SW / 4];
    /* words i < SW (two fp16 each) of group g of block b */
    __device__ __forceinline__ uint32_t scales(int b, int g, int i) const { return s[b][(g * F::SW + i) / 4][(g * F::SW + i) % 4]; }
};

/* Wave-uniform values through the scalar cache: no kernel that runs beside this one writes them. */
typedef const __attribute__((address_space(4))) int32_t *TableRow;
__device__ __forceinline__ uint32_t scalar_at(const uint32_t *a, uint32_t i) {
    return ((const __attribute__((address_space(4))) uint32_t *)(uintptr_t)a)[i];
}

/* Page ids of a step's one or two blocks, wave-uniform. */
struct Ids {
    uint32_t a, b;
};

template <class F> __device__ __forceinline__ Ids ids_of(const PagedQ4 &c, TableRow table, uint32_t step) {
    Ids r;
    r.a = r.b = (uint32_t)table[(step * F::NB) >> c.blk_shift];
    if (F::NB > 1) { /* a step's last block may lie behind the table: its keys are masked, read the first twice */
        const uint32_t blk = step * F::NB + 1u;
        r.b = (uint32_t)table[(blk * 32u < c.capacity ? blk : blk - 1u) >> c.blk_shift];
    }
    return r;
}

__device__ __forceinline__ const uint8_t *block_base(const PagedQ4 &c, uint32_t id, uint32_t h, uint32_t blk,
                                                     uint32_t block_bytes) {
    const uint32_t in = blk & ((1u << c.blk_shift) - 1u);
    return c.pages + (uint64_t)(id < c.n_pages ? id : 0u) * c.page_bytes +
           (uint64_t)(((h << c.blk_shift) + in) * block_bytes);
}

/* 16 bytes of codes.  ONCE: a single wave reads them, past the caches (loads
 * alone, B64 x 16384: 108 -> 94 us). */
template <bool ONCE> __device__ __forceinline__ uint4v load_codes(const uint8_t *p) {
    const uint4v *q = reinterpret_cast<const uint4v *>(p);
    return ONCE ? __builtin_nontemporal_load(q) : *q;
}

/* V 0: keys, 1: values. */
template <class F, int V>
__device__ __forceinline__ void load_half(Half<F> &d, const PagedQ4 &c, const Ids &ids, uint32_t h, uint32_t step,
                                          uint32_t lane) {
    constexpr int HD = F::HD;
    const uint32_t kg = lane >> 4, blk = step * F::NB;
    const uint8_t *base0 = block_base(c, ids.a, h, blk, 36u * HD), *base1 = base0;
    if (F::NB > 1) base1 = block_base(c, ids.b, h, (blk + 1u) * 32u < c.capacity ? blk + 1u : blk, 36u * HD);
#pragma unroll
    for (int b = 0; b < F::NB; ++b)
#pragma unroll
        for (int i = 0; i < HD / 64; ++i)
            d.c[b][i] = load_codes<(F::R > 1)>((b ? base1 : base0) + V * 16 * HD + i * 1024 + lane * 16u);
    if constexpr (F::J > 1) {
#pragma unroll
        for (int b = 0; b < F::NB; ++b)
#pragma unroll
            for (int g = 0; g < F::G; ++g)
                d.s[b][g] = *reinterpret_cast<const uint4v *>((b ? base1 : base0) + (32 + 2 * V) * HD + g * 64 +
                                                              kg * 16u);
    } else { /* the 4 keys of this lane's tile */
        const uint32_t u    = (lane & 15u) / (16u / F::R);
        const int64_t other = F::NB > 1 ? -(int64_t)(u >> 1) & (base1 - base0) : 0;
        const uint8_t *base = base0 + other + ((32 + 2 * V) * HD + kg * 16u + (u & 1u) * 8u);
#pragma unroll
        for (int g = 0; g < F::G; g += 2) {
            const uint2v a = __builtin_nontemporal_load(reinterpret_cast<const uint2v *>(base + g * 64));
            const uint2v z = __builtin_nontemporal_load(reinterpret_cast<const uint2v *>(base + g * 64 + 64));
            d.s[0][g / 2]  = __builtin_shufflevector(a, z, 0, 1, 2, 3);
        }
    }
}

/* Queries and running state of a unit's columns. */
template <class F> struct State {
    half8v qh[F::NT][F::R][F::G], ql[F::NT][F::R][F::G];
    float4v o[F::NT][F::DT];
    float c0[F::NT][F::G];           /* start of the S product: minus 8 sum q (unpack_k) */
    float cs[F::NT], top[F::NT], m[F::NT], l[F::NT];
    uint32_t vmax;                   /* magnitude (fp16 bits) of the V scales that m covers */
    uint32_t lo[F::NT], hi[F::NT];   /* keys [lo, hi) of the column's row */
};

/* Index of the column's (row, head) in q, out and gate; ~0: none. */
template <class F>
__device__ __forceinline__ size_t head_of(const GqaParams &p, uint32_t s, uint32_t h, uint32_t rows, uint32_t ci) {
    const uint32_t mul = p.plan.kv_mul, row = ci / mul;
    if (row >= rows) return ~(size_t)0;
    return ((size_t)s * p.c.n_rows + row) * (p.c.n_head_kv * mul) + h * mul + (ci - row * mul);
}

template <class F>
__device__ __forceinline__ void start(State<F> &st, const GqaParams &p, uint32_t s, uint32_t ct, uint32_t h,
                                      uint32_t pos0, uint32_t rows, uint32_t lane) {
    const uint32_t col = lane & 15u, kg = lane >> 4, u = col / (16u / F::R);
#pragma unroll
    for (int n = 0; n < F::NT; ++n) {
        const uint32_t ci = ct * F::COLS + n * 16u + (F::R > 1 ? col % (16u / F::R) : col);
        const size_t head = head_of<F>(p, s, h, rows, ci);
        const bool live   = head != ~(size_t)0;
        const uint32_t ps = pos0 + ci / p.plan.kv_mul;
        st.lo[n]          = live ? lfm_q4_row_lo(ps, p.plan.window) : 0u;
        st.hi[n]          = live ? ps + 1u : 0u;
        float x[F::G][8], big = 0.0f;
#pragma unroll
        for (int g = 0; g < F::G; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (live) a = reinterpret_cast<const float4 *>(p.q + head * F::HD)[g * 8 + kg * 2u + i];
                x[g][4 * i] = a.x; x[g][4 * i + 1] = a.y; x[g][4 * i + 2] = a.z; x[g][4 * i + 3] = a.w;
                big = fmaxf(big, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))));
            }
        big = kg_max(big);
        int e = big > 0.0f && big < __builtin_inff() ? __builtin_amdgcn_frexp_expf(big) : 0;
        if (e < -100) e = -100; /* 2^-e stays finite; such scores are 0 in fp32 */
        const float unit = ldexpf(p.scale < 0.0f ? -1.0f : 1.0f, -e);
#pragma unroll
        for (int g = 0; g < F::G; ++g) {
            float sum = 0.0f;
            Words yh, yl;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[g][i] * unit;
                yh.v[i]       = (_Float16)y;
                yl.v[i]       = (_Float16)(y - (float)yh.v[i]);
                sum += (float)yh.v[i] + (float)yl.v[i];
            }
#pragma unroll
            for (int r = 0; r < F::R; ++r) {
                const uint32_t mine = F::R == 1 || u == (uint32_t)r ? 0xFFFFFFFFu : 0u;
                Words a, z;
#pragma unroll
                for (int i = 0; i < 4; ++i) a.u[i] = yh.u[i] & mine, z.u[i] = yl.u[i] & mine;
                st.qh[n][r][g] = a.v;
                st.ql[n][r][g] = z.v;
            }
            st.c0[n][g] = ldexpf(-8.0f * kg_sum(sum), -kKDown);
        }
        /* Never 0: a masked score is cs * -inf.  At most 2^80: scores stay below 2^96, far from kNoScore, and where
         * that cuts, different scores (by 2^-68 before the factor, or more) are still 2^12 apart, so one weight is 1
         * and the others 0 as they should be. */
        st.cs[n]  = fminf(fmaxf(ldexpf(fabsf(p.scale) * 1.4426950408889634f, e + kKDown), 1e-37f), 0x1p80f);
        st.top[n] = st.m[n] = kNoScore;
        st.l[n] = 0.0f;
        st.vmax = 0u;
#pragma unroll
        for (int i = 0; i < F::DT; ++i) st.o[n][i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max_u16(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, a),
                                                                  __builtin_bit_cast(ushort2v, b)));
}

/* Two fp16 magnitudes in order, as 2 bits + 0x800: wraps for those that are not finite, which come before 0. */
__device__ __forceinline__ uint32_t finite_rank(uint32_t w) {
    const ushort2v a = __builtin_bit_cast(ushort2v, w);
    return __builtin_bit_cast(uint32_t, (ushort2v)(a * (ushort2v){2, 2} + (ushort2v){0x800, 0x800}));
}

/* Scores of a step before the factor cs: sum over groups of scale * (codes . q). */
template <class F>
__device__ __forceinline__ void scores(float (&x)[F::NT][4 * F::J], const State<F> &st, const Half<F> &k,
                                       const Magic &mg) {
    constexpr int NT = F::NT, G = F::G, J = F::J, R = F::R;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        float4v acc[NT][G];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int g = 0; g < G; ++g)
                acc[n][g] = float4v{st.c0[n][g], st.c0[n][g], st.c0[n][g], st.c0[n][g]};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int t = j * R + r, b = t / 2, half = t & 1;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t w =
                    F::HD == 64 ? k.c[b][0][half * 2 + g % 2] : k.c[b][half % (F::HD / 64)][g];
                const half8v a = unpack_k(w, mg);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    acc[n][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, st.ql[n][r][g], acc[n][g], 0, 0, 0);
                    acc[n][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, st.qh[n][r][g], acc[n][g], 0, 0, 0);
                }
            }
        }
        const int b = J > 1 ? j / 2 : 0, w0 = J > 1 ? (j & 1) * 2 : 0;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float y = 0.0f;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint32_t z = k.scales(b, g, w0 + i / 2);
                    y                = fmaf(i & 1 ? half_hi(z) : half_lo(z), acc[n][g][i], y);
                }
                x[n][4 * j + i] = y;
            }
    }
}

__device__ __forceinline__ uint32_t not_finite(uint32_t w) { /* halves of two fp16 */
    return ((w & 0x7C00u) == 0x7C00u ? 0x0000FFFFu : 0u) | ((w & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u);
}

/* A step that some row does not attend whole, or with a block that has no
 * page: masked scores become -inf, V scales that no column of the lane needs
 * 0 (weights of masked keys are then 0 whatever was stored).  A scale that is not
 * finite, of a key that one of the lane's columns attends and another does not,
 * is taken out too; the columns that attend it get their NaN here. */
template <class F>
__device__ __forceinline__ void mask_step(float (&x)[F::NT][4 * F::J], Half<F> &v, State<F> &st, bool there_a,
                                          bool there_b, uint32_t key0, uint32_t lane) {
    constexpr int NT = F::NT, G = F::G, J = F::J;
    const uint32_t kg = lane >> 4, u = (lane & 15u) / (16u / F::R);
    uint32_t bad = 0u;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const uint32_t t = J > 1 ? (uint32_t)j : u;
        const bool page  = (there_a || t >= 2u) && (there_b || t < 2u);
        uint32_t keep[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t key = key0 + 16u * t + 4u * kg + i;
            bool any           = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const bool see = page && key >= st.lo[n] && key < st.hi[n];
                if (!see) x[n][4 * j + i] = -__builtin_inff();
                any |= see;
            }
            if (any) keep[i / 2] |= i & 1 ? 0xFFFF0000u : 0x0000FFFFu;
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = g * F::SW + (J > 1 ? (j & 1) * 2 : 0) + i;
                v.s[J > 1 ? j / 2 : 0][at / 4][at % 4] &= keep[i];
                if (NT > 1) bad |= not_finite(v.s[J > 1 ? j / 2 : 0][at / 4][at % 4]);
            }
    }
    if (NT > 1 && __any(bad != 0u)) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            uint32_t hit[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) hit[n] = 0u;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int at = g * F::SW + (J > 1 ? (j & 1) * 2 : 0) + i;
                    uint32_t w   = v.s[J > 1 ? j / 2 : 0][at / 4][at % 4];
                    asm volatile("" : "+v"(w)); /* worked out here anew: the masks above are not held for this */
                    const uint32_t m = not_finite(w);
                    /* x is -inf exactly where the column does not attend */
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (x[n][4 * j + 2 * i] != -__builtin_inff()) hit[n] |= m & 0xFFFFu;
                        if (x[n][4 * j + 2 * i + 1] != -__builtin_inff()) hit[n] |= m >> 16;
                    }
                    v.s[J > 1 ? j / 2 : 0][at / 4][at % 4] = w & ~m;
                }
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (kg_max(hit[n]))
#pragma unroll
                    for (int i = 2 * g; i < 2 * g + 2; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k) st.o[n][i][k] = __builtin_nanf("");
        }
    }
}

/* Raises top and the bound of the V scales where a step passes them. */
template <class F>
__device__ __forceinline__ void check_step(State<F> &st, const float (&x)[F::NT][4 * F::J], const Half<F> &v) {
    constexpr int NT = F::NT, G = F::G, J = F::J;
    float best[NT];
    uint32_t dv = 0u;
    bool raise  = false;
#pragma unroll
    for (int b = 0; b < F::SB; ++b)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < F::SW; ++i) dv = pk_max_u16(dv, v.scales(b, g, i) & 0x7FFF7FFFu);
    dv = max(dv & 0xFFFFu, dv >> 16);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        best[n] = x[n][0];
#pragma unroll
        for (int i = 1; i < 4 * J; ++i) best[n] = fmaxf(best[n], x[n][i]);
        best[n] *= st.cs[n];
        raise |= best[n] > st.top[n] + kSlack;
    }
    raise |= dv > st.vmax;
    if (__any(raise)) {
        if (__any(dv >= 0x7C00u)) { /* a scale that is not finite gives NaN in its own dims alone */
            dv = 0u;
#pragma unroll
            for (int b = 0; b < F::SB; ++b)
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int i = 0; i < F::SW; ++i) dv = pk_max_u16(dv, finite_rank(v.scales(b, g, i)));
            dv = max(dv & 0xFFFFu, dv >> 16);
            dv = dv > 0x800u ? (dv - 0x800u) >> 1 : 0u;
        }
        st.vmax       = max(kg_max(dv), st.vmax);
        const float z = (float)__builtin_bit_cast(_Float16, (uint16_t)st.vmax);
        const float e = (z > 0.0f ? (float)__builtin_amdgcn_frexp_expf(z) : 0.0f) - kLift;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            st.top[n]     = fmaxf(st.top[n], kg_max(best[n]));
            const float m = st.top[n] + e;
            const float a = __builtin_amdgcn_exp2f(st.m[n] - m);
            st.l[n] *= a;
#pragma unroll
            for (int i = 0; i < F::DT; ++i) st.o[n][i] *= a;
            st.m[n] = m;
        }
    }
}

/* p = exp2(cs x - m), O += codes . (p * scale) per block and group of dims. */
template <class F>
__device__ __forceinline__ void accumulate(State<F> &st, float (&x)[F::NT][4 * F::J], const Half<F> &v,
                                           uint32_t lane, const Magic &mg) {
    constexpr int NT = F::NT, G = F::G, J = F::J, R = F::R;
    uint32_t mine[R]; /* all bits in the lanes of copy r */
#pragma unroll
    for (int r = 0; r < R; ++r) {
        mine[r] = (lane & 15u) / (16u / R) == (uint32_t)r ? ~0u : 0u;
        if (R > 1) asm("" : "+v"(mine[r])); /* an AND (2.6 cycles), not a select (4.5) */
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4 * J; ++i) {
            x[n][i] = __builtin_amdgcn_exp2f(fmaf(x[n][i], st.cs[n], -st.m[n]));
            st.l[n] += x[n][i];
        }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        uint32_t ch[2], cl[2]; /* R > 1: this lane's 4 keys */
        if constexpr (R > 1) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                split_weights(x[0][2 * i], x[0][2 * i + 1], v.scales(0, g, i), &ch[i], &cl[i], mg);
        }
#pragma unroll
        for (int b = 0; b < F::NB; ++b) {
            Words wh[NT], wl[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (R > 1) {
                        wh[n].u[i] = ch[i & 1] & mine[(2 * b + i / 2) % R];
                        wl[n].u[i] = cl[i & 1] & mine[(2 * b + i / 2) % R];
                    } else {
                        split_weights(x[n][8 * b + 2 * i], x[n][8 * b + 2 * i + 1], v.scales(b, g, i),
                                      &wh[n].u[i], &wl[n].u[i], mg);
                    }
                }
#pragma unroll
            for (int i = 2 * g; i < 2 * g + 2; ++i) {
                const half8v a = unpack_v(v.c[b][i / 4][i & 3], mg);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    st.o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wl[n].v, st.o[n][i], 0, 0, 0);
                    st.o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, wh[n].v, st.o[n][i], 0, 0, 0);
                }
            }
        }
    }
}

/* Where a piece stands, wave-uniform. */
struct Walk {
    TableRow table;
    uint32_t h, step, last; /* last: the piece's last step */
    uint32_t in0, in1;      /* keys that every row of the tile attends */
    Ids ids[4];             /* of steps step .. step + 3, as far as there are any */
};

/* One step: its P.V product beside the S product of the next step, neither
 * waiting for the other.  LOAD: while the next values and the keys behind the
 * next ones are loaded; the page ids come one step before that.  (Loads one step
 * further ahead were no faster.) */
template <class F, bool LOAD>
__device__ __forceinline__ void step_once(State<F> &st, const GqaParams &p, Walk &w, float (&x)[F::NT][4 * F::J],
                                          Half<F> &v, Half<F> &v_new, const Half<F> &k_next, Half<F> &k_new,
                                          uint32_t lane, const Magic &mg) {
    if constexpr (LOAD) {
        load_half<F, 1>(v_new, p.c, w.ids[1], w.h, w.step + 1u < w.last ? w.step + 1u : w.last, lane);
        load_half<F, 0>(k_new, p.c, w.ids[2], w.h, w.step + 2u < w.last ? w.step + 2u : w.last, lane);
        w.ids[3] = ids_of<F>(p.c, w.table, w.step + 3u < w.last ? w.step + 3u : w.last);
    }
    const uint32_t key0 = w.step * F::STEP;
    const bool there_a = w.ids[0].a < p.c.n_pages, there_b = w.ids[0].b < p.c.n_pages;
    if (!(key0 >= w.in0 && key0 + F::STEP <= w.in1 && there_a && there_b))
        mask_step<F>(x, v, st, there_a, there_b, key0, lane);
    check_step<F>(st, x, v);
    float y[F::NT][4 * F::J];
    scores<F>(y, st, k_next, mg);
    accumulate<F>(st, x, v, lane, mg);
#pragma unroll
    for (int n = 0; n < F::NT; ++n)
#pragma unroll
        for (int i = 0; i < 4 * F::J; ++i) x[n][i] = y[n][i];
#pragma unroll
    for (uint32_t i = 0; i < 3u; ++i) w.ids[i] = w.ids[i + 1u];
    ++w.step;
}

/* Steps [a, b) of unit (s, ct, h) into a fresh state.  Buffers change roles every
 * step, so two steps make a turn without copies; an odd last step comes after
 * the loop, which so has one way out (with one per step, values met there in new
 * registers, and every turn waited for its last loads).  The first loads go out
 * before the queries are read and split. */
template <class F>
__device__ __forceinline__ void run_piece(State<F> &st, const GqaParams &p, uint32_t s, uint32_t ct, uint32_t h,
                                          const lfm_q4_tile &t, uint32_t pos0, uint32_t rows, uint32_t a, uint32_t b,
                                          uint32_t lane) {
    const Magic mg = magic();
    Walk w;
    w.table = (TableRow)(uintptr_t)(p.c.table + (size_t)s * p.c.table_stride);
    w.h     = h;
    w.step  = a;
    w.last  = b - 1u;
    w.in0   = lfm_q4_row_lo(pos0 + t.r1 - 1u, p.plan.window);
    w.in1   = pos0 + t.r0 + 1u;
    Half<F> k0, k1, v0, v1;
#pragma unroll
    for (uint32_t i = 0; i < 3u; ++i) w.ids[i] = ids_of<F>(p.c, w.table, a + i < w.last ? a + i : w.last);
    load_half<F, 0>(k0, p.c, w.ids[0], h, a, lane);
    load_half<F, 1>(v0, p.c, w.ids[0], h, a, lane);
    load_half<F, 0>(k1, p.c, w.ids[1], h, a + 1u < w.last ? a + 1u : w.last, lane);
    start<F>(st, p, s, ct, h, pos0, rows, lane);
    float x[F::NT][4 * F::J];
    scores<F>(x, st, k0, mg);
    while (w.step + 2u <= b) {
        step_once<F, true>(st, p, w, x, v0, v1, k1, k0, lane, mg);
        step_once<F, true>(st, p, w, x, v1, v0, k0, k1, lane, mg);
    }
    if (w.step < b) step_once<F, false>(st, p, w, x, v0, v1, k1, k0, lane, mg);
}

/* Sums over the lanes that share a column; with R > 1 its copies too. */
template <class F> __device__ __forceinline__ void join_lanes(State<F> &st) {
#pragma unroll
    for (int n = 0; n < F::NT; ++n) st.l[n] = kg_sum(st.l[n]);
    if constexpr (F::R > 1) {
        const float m = copies_max<F::R>(st.m[0]), a = __builtin_amdgcn_exp2f(st.m[0] - m);
        st.l[0]       = copies_sum<F::R>(st.l[0] * a);
#pragma unroll
        for (int i = 0; i < F::DT; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) st.o[0][i][k] = copies_sum<F::R>(st.o[0][i][k] * a);
        st.m[0] = m;
    }
}

/* 1 / l (0 where no key was attended, NaN where a score was) times the gate,
 * and what unpack_v left out. */
__device__ __forceinline__ float out_factor(const GqaParams &p, float l, size_t head) {
    float f = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    if (p.gate) {
        const float x = p.gate[head];
        f *= p.gate_is_logit ? 1.0f / (1.0f + expf(-x)) : x;
    }
    return f * kVUp;
}

template <class F>
__device__ __forceinline__ void write_out(const State<F> &st, const GqaParams &p, uint32_t s, uint32_t ct, uint32_t h,
                                          uint32_t rows, uint32_t lane) {
    const uint32_t col = lane & 15u, kg = lane >> 4;
#pragma unroll
    for (int n = 0; n < F::NT; ++n) {
        if (F::R > 1 && col >= 16u / F::R) continue;
        const size_t head = head_of<F>(p, s, h, rows, ct * F::COLS + n * 16u + col);
        if (head == ~(size_t)0) continue;
        const float f = out_factor(p, st.l[n], head);
#pragma unroll
        for (int i = 0; i < F::DT; ++i)
            reinterpret_cast<float4 *>(p.out + head * F::HD)[i * 4 + kg] =
                make_float4(st.o[n][i][0] * f, st.o[n][i][1] * f, st.o[n][i][2] * f, st.o[n][i][3] * f);
    }
}

/* A piece's columns as they stand: outputs [col][HD], (m, l) [col]. */
template <class F>
__device__ __forceinline__ void put_part(const State<F> &st, float *o, float2 *ml, uint32_t lane) {
    const uint32_t col = lane & 15u, kg = lane >> 4;
#pragma unroll
    for (int n = 0; n < F::NT; ++n) {
        if (F::R > 1 && col >= 16u / F::R) continue;
        const uint32_t c = n * 16u + col;
        if (kg == 0u) ml[c] = make_float2(st.m[n], st.l[n]);
#pragma unroll
        for (int i = 0; i < F::DT; ++i)
            reinterpret_cast<float4 *>(o + c * F::HD)[i * 4 + kg] =
                make_float4(st.o[n][i][0], st.o[n][i][1], st.o[n][i][2], st.o[n][i][3]);
    }
}

/* The same for a wave-uniform s. */
__device__ __forceinline__ uint32_t rows_at(const PagedQ4 &c, uint32_t s, uint32_t pos0) {
    return lfm_q4_rows(pos0, c.rows_seq ? scalar_at(c.rows_seq, s) : c.n_rows, c.n_rows, c.capacity);
}

__device__ __forceinline__ uint32_t rows_of(const PagedQ4 &c, uint32_t s, uint32_t pos0) {
    return lfm_q4_rows(pos0, c.rows_seq ? c.rows_seq[s] : c.n_rows, c.n_rows, c.capacity);
}

/* Every wave one unit, all its keys: 4 adjacent tiles of a (sequence, KV head)
 * per workgroup, which read the same pages at about the same time.  The last
 * tiles, with the most keys, are dispatched first; consecutive workgroups, which
 * go to the 8 XCDs in turn, differ in KV head, so a head's pages mostly stay in
 * one XCD's L2. */
template <class F> __global__ __launch_bounds__(256, 2) void k_paged_gqa(const GqaParams p) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t pairs = p.c.n_seq * p.c.n_head_kv, quad = blockIdx.x / pairs, pair = blockIdx.x - quad * pairs;
    const uint32_t s = pair / p.c.n_head_kv, h = pair - s * p.c.n_head_kv;
    const uint32_t back = quad * 4u + uniform(threadIdx.x >> 6);
    if (back >= p.plan.n_ct) return;
    const uint32_t ct   = p.plan.n_ct - 1u - back;
    const uint32_t pos0 = scalar_at(p.c.pos0, s), rows = rows_at(p.c, s, pos0);
    const lfm_q4_tile t = lfm_q4_tile_of(&p.plan, pos0, rows, ct);
    if (t.n_steps == 0u) return;
    State<F> st;
    run_piece<F>(st, p, s, ct, h, t, pos0, rows, t.step0, t.step0 + t.n_steps, lane);
    join_lanes<F>(st);
    write_out<F>(st, p, s, ct, h, rows, lane);
}

/* Column col, dims 4 d .. of the pieces at the places in `run` (8 at most). */
struct Merged {
    float m, l;
    float4 o;
};
template <class F>
__device__ __forceinline__ Merged merge_run(const float *so, const float2 *sml, uint32_t run, uint32_t col, uint32_t d) {
    Merged r = {kNoScore, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
    float2 ml[8];
#pragma unroll
    for (uint32_t w = 0; w < 8u; ++w) {
        ml[w] = make_float2(kNoScore, 0.0f);
        if (run >> w & 1u) ml[w] = sml[w * F::COLS + col];
        r.m = fmaxf(r.m, ml[w].x);
    }
#pragma unroll
    for (uint32_t w = 0; w < 8u; ++w) {
        if (!(run >> w & 1u)) continue; /* wave-uniform */
        const float f  = __builtin_amdgcn_exp2f(ml[w].x - r.m);
        const float4 x = reinterpret_cast<const float4 *>(so + (w * F::COLS + col) * F::HD)[d];
        r.l += ml[w].y * f;
        r.o = make_float4(r.o.x + x.x * f, r.o.y + x.y * f, r.o.z + x.z * f, r.o.w + x.w * f);
    }
    return r;
}

/* One workgroup of W waves per unit: its waves share the steps and join in
 * LDS.  For short units: one launch, no partials. */
template <class F, int W> __global__ __launch_bounds__(64 * W, 2) void k_paged_gqa_wg(const GqaParams p) {
    static_assert(W <= 8, "merge_run takes 8 pieces");
    __shared__ __align__(16) float so[W][F::COLS][F::HD];
    __shared__ float2 sml[W][F::COLS];
    const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6);
    const uint32_t unit = blockIdx.x, h = unit % p.c.n_head_kv, sc = unit / p.c.n_head_kv;
    const uint32_t s = sc / p.plan.n_ct, ct = sc - s * p.plan.n_ct;
    const uint32_t pos0 = scalar_at(p.c.pos0, s), rows = rows_at(p.c, s, pos0);
    const lfm_q4_tile t = lfm_q4_tile_of(&p.plan, pos0, rows, ct);
    if (t.n_steps == 0u) return;
    /* the first shares are the longer ones */
    const uint32_t more = t.n_steps % W, parts = t.n_steps < W ? t.n_steps : W;
    uint32_t a = wave * (t.n_steps / W) + (wave < more ? wave : more), b = a + t.n_steps / W + (wave < more ? 1u : 0u);
    a = uniform(a), b = uniform(b);
    if (a < b) {
        State<F> st;
        run_piece<F>(st, p, s, ct, h, t, pos0, rows, t.step0 + a, t.step0 + b, lane);
        join_lanes<F>(st);
        put_part<F>(st, &so[wave][0][0], &sml[wave][0], lane);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < F::COLS * F::HD / 4u; i += 64u * W) {
        const uint32_t col = i / (F::HD / 4u), d = i % (F::HD / 4u);
        const size_t head  = head_of<F>(p, s, h, rows, ct * F::COLS + col);
        if (head == ~(size_t)0) continue;
        const Merged r = merge_run<F>(&so[0][0][0], &sml[0][0], (1u << parts) - 1u, col, d);
        const float f  = out_factor(p, r.l, head);
        reinterpret_cast<float4 *>(p.out + head * F::HD)[d] = make_float4(r.o.x * f, r.o.y * f, r.o.z * f, r.o.w * f);
    }
}

/* Steps of entry e (sequence, tile), none past the last. */
__device__ __forceinline__ uint32_t steps_of(const GqaParams &p, uint32_t e, uint32_t n_entries) {
    if (e >= n_entries) return 0u;
    const uint32_t s = p.plan.n_ct == 1u ? e : e / p.plan.n_ct, pos0 = p.c.pos0[s];
    return lfm_q4_tile_of(&p.plan, pos0, rows_of(p.c, s, pos0), e - s * p.plan.n_ct).n_steps;
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t x, uint32_t lane) { /* inclusive */
#pragma unroll
    for (uint32_t o = 1; o < 64u; o *= 2u) {
        const uint32_t y = (uint32_t)__shfl_up((int)x, o);
        if (lane >= o) x += y;
    }
    return x;
}

__device__ __forceinline__ uint32_t lane_of(uint32_t x, uint32_t i) {
    return (uint32_t)__builtin_amdgcn_readlane((int)x, (int)i);
}

/* Equal shares of the batch's steps per wave.  A wave's first and last piece
 * may be parts of units; those of the 4 waves of a workgroup join in LDS, and
 * what is still part of a unit goes to the workspace. */
template <class F> __global__ __launch_bounds__(256, 2) void k_paged_gqa_split(const GqaParams p) {
    __shared__ __align__(16) float so[8][F::COLS][F::HD]; /* first and last piece of each wave */
    __shared__ float2 sml[8][F::COLS];
    __shared__ struct {
        uint32_t unit, s, ct, h, rows, whole; /* unit ~0: none; whole: 1 has the unit's first step, 2 its last */
    } meta[8];
    const uint32_t lane = threadIdx.x & 63u, nh = p.c.n_head_kv;
    const uint32_t in_wg = uniform(threadIdx.x >> 6), wave = blockIdx.x * 4u + in_wg;
    const uint32_t n_e = p.c.n_seq * p.plan.n_ct;
    if (lane < 2u) meta[in_wg * 2u + lane].unit = ~0u;
    /* a window of 64 entries, one per lane; batches of up to 64 keep it */
    uint32_t inc   = wave_scan(steps_of(p, lane, n_e), lane);
    uint32_t total = lane_of(inc, 63u);
    for (uint32_t e0 = 64u; e0 < n_e; e0 += 64u)
        total += lane_of(wave_scan(steps_of(p, e0 + lane, n_e), lane), 63u);
    const uint32_t N = total * nh, G = lfm_q4_waves(&p.plan, N);
    uint32_t t = 0u, t1 = 0u;
    if (wave < G) {
        lfm_q4_share(wave, N, G, &t, &t1);
        t  = uniform(t);
        t1 = uniform(t1);
    }
    const uint32_t t0 = t;
    uint32_t e0 = 0u, base = 0u; /* the window's first entry, steps before it */
    while (t < t1) {
        const uint32_t want = uniform(t / nh);
        uint64_t hit        = __ballot(base + inc > want);
        while (!hit) { /* ends: want is below the total */
            base += lane_of(inc, 63u);
            e0 += 64u;
            inc = wave_scan(steps_of(p, e0 + lane, n_e), lane);
            hit = __ballot(base + inc > want);
        }
        const uint32_t i = (uint32_t)__builtin_ctzll(hit), e = e0 + i;
        const uint32_t s = p.plan.n_ct == 1u ? e : uniform(e / p.plan.n_ct), ct = e - s * p.plan.n_ct;
        const uint32_t pos0 = scalar_at(p.c.pos0, s), rows = rows_at(p.c, s, pos0);
        const lfm_q4_tile tile = lfm_q4_tile_of(&p.plan, pos0, rows, ct);
        const uint32_t n = uniform(tile.n_steps), first = (base + lane_of(inc, i) - n) * nh;
        uint32_t h = uniform((t - first) / n);
        uint32_t a = t - first - h * n;
        for (; t < t1 && h < nh; ++h, a = 0u) {
            const uint32_t b = n - a < t1 - t ? n : a + (t1 - t);
            uint32_t ln = lane;
            /* of its own in every turn, so that what hangs on it is not held in registers across pieces: 35.9 ->
             * 33.7 us for 16 x 8 rows at 4096 keys of head_dim 128, 33.1 -> 32.4 of 64.  Forms with registers to
             * spare lose 1 % by it. */
            if (F::HD == 128 || F::NT > 1) asm volatile("" : "+v"(ln));
            State<F> st;
            run_piece<F>(st, p, s, ct, h, tile, pos0, rows, tile.step0 + a, tile.step0 + b, ln);
            join_lanes<F>(st);
            if (a == 0u && b == n) {
                write_out<F>(st, p, s, ct, h, rows, ln);
                if (lane == 0u) p.range[e * nh + h] = make_uint2(blockIdx.x, blockIdx.x);
            } else { /* the first piece of the share, or its last */
                const uint32_t at = in_wg * 2u + (t == t0 ? 0u : 1u);
                put_part<F>(st, &so[at][0][0], &sml[at][0], ln);
                if (lane == 0u) {
                    meta[at].unit = e * nh + h;
                    meta[at].s = s, meta[at].ct = ct, meta[at].h = h, meta[at].rows = rows;
                    meta[at].whole = (a == 0u ? 1u : 0u) | (b == n ? 2u : 0u);
                }
            }
            t += b - a;
        }
    }
    __syncthreads();
    /* runs of pieces of one unit, with empty places between them */
    uint32_t units[8], have = 0u;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        units[i] = uniform(meta[i].unit);
        have |= units[i] != ~0u ? 1u << i : 0u;
    }
    while (have) {
        const uint32_t i = (uint32_t)__builtin_ctz(have), unit = uniform(meta[i].unit);
        uint32_t run = 0u, whole = 0u;
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k)
            if ((have >> k & 1u) && units[k] == unit) run |= 1u << k;
        have &= ~run;
        whole = uniform(meta[i].whole | meta[31 - __builtin_clz(run)].whole);
        if (threadIdx.x == 0u) {
            if (whole & 1u) p.range[unit].x = blockIdx.x;
            if (whole & 2u) p.range[unit].y = blockIdx.x;
        }
        const uint32_t s = meta[i].s, ct = meta[i].ct, h = meta[i].h, rows = meta[i].rows;
        for (uint32_t x = threadIdx.x; x < F::COLS * F::HD / 4u; x += 256u) {
            const uint32_t col = x / (F::HD / 4u), d = x % (F::HD / 4u);
            const Merged r     = merge_run<F>(&so[0][0][0], &sml[0][0], run, col, d);
            if (whole == 3u) {
                const size_t head = head_of<F>(p, s, h, rows, ct * F::COLS + col);
                if (head == ~(size_t)0) continue;
                const float f = out_factor(p, r.l, head);
                reinterpret_cast<float4 *>(p.out + head * F::HD)[d] =
                    make_float4(r.o.x * f, r.o.y * f, r.o.z * f, r.o.w * f);
            } else {
                const size_t at = ((size_t)blockIdx.x + unit) * F::COLS + col;
                if (d == 0u) p.part_ml[at] = make_float2(r.m, r.l);
                reinterpret_cast<float4 *>(p.part_o + at * F::HD)[d] = r.o;
            }
        }
    }
}

/* The pieces of the units that more than one workgroup holds: an item is a
 * (unit, column), HD / 4 threads take a piece.  T 64: a wave per item, 4 in a
 * workgroup, which meet in registers: for few pieces.  Else T threads per item,
 * which meet in LDS.  Per piece and column (m, l) and HD floats are read. */
template <int HD, int T> __global__ __launch_bounds__(T < 256 ? 256 : T) void k_paged_merge(const GqaParams p) {
    constexpr uint32_t L = HD / 4, P = T / L;
    const uint32_t nh = p.c.n_head_kv, cols = p.plan.cols;
    const uint32_t item = T < 256 ? blockIdx.x * 4u + uniform(threadIdx.x >> 6) : blockIdx.x;
    const uint32_t unit = item / cols, col = item - unit * cols;
    const uint32_t e = unit / nh, h = unit - e * nh;
    const uint32_t s = e / p.plan.n_ct, ct = e - s * p.plan.n_ct;
    if (s >= p.c.n_seq) return;
    /* not written, and not used, where the column has no row; what is used is
     * checked against the launch all the same */
    const uint2 g       = p.range[unit];
    const uint32_t rows = rows_of(p.c, s, p.c.pos0[s]);
    const uint32_t mul = p.plan.kv_mul, ci = ct * cols + col, row = ci / mul;
    if (row >= rows || g.x >= g.y || g.y >= p.plan.n_waves / 4u) return;
    const uint32_t g0 = g.x, g1 = g.y;
    const size_t head = ((size_t)s * p.c.n_rows + row) * (nh * mul) + h * mul + (ci - row * mul);
    const uint32_t t = T < 256 ? threadIdx.x & 63u : threadIdx.x, i = t % L, k = t / L;
    float m = kNoScore, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t w = g0 + k; w <= g1; w += P) {
        const size_t at = ((size_t)w + unit) * cols + col;
        const float2 ml = p.part_ml[at];
        const float4 x  = reinterpret_cast<const float4 *>(p.part_o + at * HD)[i];
        const float mn = fmaxf(m, ml.x), a = __builtin_amdgcn_exp2f(m - mn), b = __builtin_amdgcn_exp2f(ml.x - mn);
        m = mn;
        l = l * a + ml.y * b;
        o = make_float4(o.x * a + x.x * b, o.y * a + x.y * b, o.z * a + x.z * b, o.w * a + x.w * b);
    }
    if constexpr (T < 256) { /* P is 4 or 2: the lanes 16 or 32 apart */
        const float mm = P == 4 ? kg_max(m) : pair_max(m), f = __builtin_amdgcn_exp2f(m - mm);
        l              = P == 4 ? kg_sum(l * f) : pair_sum(l * f);
        o.x            = P == 4 ? kg_sum(o.x * f) : pair_sum(o.x * f);
        o.y            = P == 4 ? kg_sum(o.y * f) : pair_sum(o.y * f);
        o.z            = P == 4 ? kg_sum(o.z * f) : pair_sum(o.z * f);
        o.w            = P == 4 ? kg_sum(o.w * f) : pair_sum(o.w * f);
    } else {
        __shared__ float sm[P], sl[P];
        __shared__ float4 so[P][L];
        so[k][i] = o;
        if (i == 0u) sm[k] = m, sl[k] = l;
        __syncthreads();
        if (k != 0u) return;
        float mm = m;
#pragma unroll
        for (uint32_t j = 1; j < P; ++j) mm = fmaxf(mm, sm[j]);
        l = 0.0f;
        o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t j = 0; j < P; ++j) {
            const float b  = __builtin_amdgcn_exp2f(sm[j] - mm);
            const float4 x = so[j][i];
            l += sl[j] * b;
            o = make_float4(o.x + x.x * b, o.y + x.y * b, o.z + x.z * b, o.w + x.w * b);
        }
    }
    const float f = out_factor(p, l, head);
    if (k == 0u)
        reinterpret_cast<float4 *>(p.out + head * HD)[i] = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
}

/* ---- host: forms, split, scratch ------------------------------------------------ */
constexpr uint32_t kCus        = 256u;
constexpr uint32_t kWaves      = 8u * kCus; /* two per SIMD */
constexpr uint32_t kGroupSteps = 128u;

struct Launch {
    lfm_q4_plan plan;
    uint32_t copies, tiles; /* R and NT of the form */
    enum { kDirect, kSplit, kGroup } how;
    size_t o_bytes, ml_bytes, range_bytes;
};

int plan_launch(Launch *L, uint32_t n_seq, uint32_t n_rows, uint32_t keys_hint, uint32_t n_head_q, uint32_t n_head_kv,
                uint32_t head_dim, uint32_t capacity, uint32_t window) {
    lfm_q4_plan &p      = L->plan;
    const uint32_t mul  = n_head_q / n_head_kv;
    const uint64_t cols = (uint64_t)n_rows * mul;
    if (cols > 0x7FFFFFFFull) return LFM_ATTN_E_UNSUPPORTED;
    p.n_seq     = n_seq;
    p.n_rows    = n_rows;
    p.kv_mul    = mul;
    p.n_head_kv = n_head_kv;
    p.window    = window;
    p.capacity  = capacity;
    L->tiles    = 1u;
    L->copies   = 1u;
    if (head_dim == 64u) {
        if (cols <= 4u) L->copies = 4u;
        if (cols > 16u) L->tiles = 2u;
    } else {
        if (cols <= 8u) L->copies = 2u;
    }
    p.cols = L->copies > 1u ? 16u / L->copies : 16u * L->tiles;
    p.step_shift = L->copies == 4u ? 6u : 5u;
    p.n_ct = (uint32_t)((cols + p.cols - 1u) / p.cols);
    /* the threads of a launch are 32 bits: 256 per 4 tiles, and 64 per column in a merge (below) */
    const uint64_t pairs = (uint64_t)n_seq * n_head_kv;
    if (pairs >= 1ull << 24 || pairs * ((p.n_ct + 3u) / 4u) >= 1ull << 24) return LFM_ATTN_E_UNSUPPORTED;
    const uint64_t units = pairs * p.n_ct;
    uint64_t keys = keys_hint && keys_hint < capacity ? keys_hint : capacity;
    const uint64_t span = p.n_ct > 1u ? p.cols / mul + 2u : n_rows; /* rows that a tile may meet */
    if (window && window + span < keys) keys = window + span;
    const uint64_t steps = (keys >> p.step_shift) + 1u + (window ? 1u : 0u); /* of the longest unit */
    /* A wave per unit, or equal shares of all steps (whose counts, and whose merge's threads, are 32 bits).  In
     * 1 / 1450 us: a wave takes its unit's steps one after the other, 1340 each alone on a SIMD, 2060 beside a second
     * one, and decodes that fill the card are bound by memory, which units of one length each use worse; a split
     * takes the mean, and a start, pieces and merge by the unit.  Us, wave per unit | split: prompts, head_dim 64:
     * 4 x 600 rows 30 | 93, 1 x 4000 rows 176 | 399, 4 x 500 rows from position 2000 112 | 140, 1 x 700 from 1000
     * 52 | 49, 1 x 300 from 8000 222 | 75; single rows: 96 x 250 keys 8.6 | 16.7, 96 x 2000 31.1 | 32.3, 256 x 500
     * 28.7 | 25.2, 256 x up to 500 24.4 | 31.4, 256 x 2000 83.5 | 60.8; head_dim 128: 160 x 500 19.5 | 25.9,
     * 160 x 2000 57.3 | 49.6. */
    const uint64_t early = (n_rows >> p.step_shift) / 2u, mean = window || steps <= early ? steps : steps - early;
    uint64_t apart       = steps * (units > kWaves / 2u ? 2060u : 1340u);
    if (p.n_ct == 1u && units > kWaves / 2u && 2u * units * steps > apart) apart = 2u * units * steps;
    const uint64_t even_cost = units * mean + (L->copies > 1u ? 10u : 32u) * units + 10000u;
    const bool can_split     = units * (capacity / 32u) < 1ull << 31 && units * p.cols < 1ull << 26;
    L->how = can_split && apart > even_cost ? Launch::kSplit : Launch::kDirect;
    /* A workgroup per unit has no second launch and no partials, 2 to 8 us (the more units, the more), but only
     * `units` of the 256 CUs work: it is ahead while steps * (256 - units) is small.  Us, group | split, at
     * 16 x 8 rows of head_dim 64 (128 units): 2000 keys 19.8 | 21.1, 4000 keys 31.1 | 26.8; 4 rows (16 columns,
     * half the work a step): 2000 keys 13.8 | 15.1, 4000 keys 21.2 | 19.0; 1 row of 8 sequences: 2000 keys
     * 12.2 | 12.6, 4000 keys 17.4 | 14.6.  Up to 128 steps, so that a long sequence among short ones is split. */
    const uint64_t wait = head_dim == 128u || L->copies > 1u ? 7168u : L->tiles > 1u ? 9216u : 12288u;
    if (units <= kCus && steps <= kGroupSteps && steps * (kCus - units) <= wait) L->how = Launch::kGroup;
    uint64_t waves = units * steps;
    if (waves > kWaves) waves = kWaves;
    p.n_waves = (uint32_t)((waves + 3u) / 4u * 4u);
    /* whole workgroups per unit, where that leaves few waves out */
    const uint32_t even = (uint32_t)(p.n_waves / (4u * units) * (4u * units));
    if (even >= p.n_waves - p.n_waves / 16u) p.n_waves = even;
    const uint64_t slots = L->how == Launch::kSplit ? p.n_waves / 4u + units : 0u;
    L->o_bytes     = slots * p.cols * head_dim * 4u;
    L->ml_bytes    = slots * p.cols * 8u;
    L->range_bytes = L->how == Launch::kSplit ? units * 8u : 0u;
    return LFM_ATTN_OK;
}

template <class F> void launch_form(const GqaParams &p, const Launch &L, hipStream_t stream) {
    const uint32_t pairs = p.c.n_seq * p.c.n_head_kv, units = pairs * p.plan.n_ct, cols = units * p.plan.cols;
    if (L.how == Launch::kDirect) {
        hipLaunchKernelGGL(k_paged_gqa<F>, dim3(pairs * ((p.plan.n_ct + 3u) / 4u)), dim3(256), 0, stream, p);
        return;
    }
    if (L.how == Launch::kGroup) {
        hipLaunchKernelGGL((k_paged_gqa_wg<F, 8>), dim3(units), dim3(512), 0, stream, p);
        return;
    }
    hipLaunchKernelGGL(k_paged_gqa_split<F>, dim3(p.plan.n_waves / 4u), dim3(256), 0, stream, p);
    /* A unit's pieces: a wave takes 256 / HD at a time, a workgroup 8 times that.  Up to 4 turns of a wave; us, wave |
     * workgroup: head_dim 64, 16 pieces, 4 x 8 rows: 16.1 | 19.3; head_dim 128, 16 pieces, 8 x 1 rows of 5000 keys:
     * 19.0 | 17.4. */
    if (p.plan.n_waves / 4u * F::HD <= 1024u * units)
        hipLaunchKernelGGL((k_paged_merge<F::HD, 64>), dim3((cols + 3u) / 4u), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((k_paged_merge<F::HD, 512>), dim3(cols), dim3(512), 0, stream, p);
}

} // namespace

int paged_q4_gqa_workspace(uint32_t n_seq, uint32_t n_rows, uint32_t keys_hint, uint32_t n_head_q, uint32_t n_head_kv,
                           uint32_t head_dim, uint32_t capacity, uint32_t window, size_t *bytes) {
    Launch L;
    const int st = plan_launch(&L, n_seq, n_rows, keys_hint, n_head_q, n_head_kv, head_dim, capacity, window);
    if (st != LFM_ATTN_OK) return st;
    *bytes = L.o_bytes + L.ml_bytes + L.range_bytes;
    return LFM_ATTN_OK;
}

int launch_paged_q4_gqa(const PagedQ4 &c, const float *q, const float *gate, int gate_is_logit, float *out,
                        uint32_t n_head_q, uint32_t keys_hint, uint32_t window, float scale, void *workspace,
                        hipStream_t stream) {
    Launch L;
    const int st =
        plan_launch(&L, c.n_seq, c.n_rows, keys_hint, n_head_q, c.n_head_kv, c.head_dim, c.capacity, window);
    if (st != LFM_ATTN_OK) return st;
    GqaParams p;
    p.c             = c;
    p.plan          = L.plan;
    p.q             = q;
    p.gate          = gate;
    p.out           = out;
    p.gate_is_logit = gate_is_logit;
    p.scale         = scale;
    uint8_t *w      = static_cast<uint8_t *>(workspace);
    p.part_o        = reinterpret_cast<float *>(w);
    p.part_ml       = reinterpret_cast<float2 *>(w + L.o_bytes);
    p.range         = reinterpret_cast<uint2 *>(w + L.o_bytes + L.ml_bytes);
    if (c.head_dim == 64u) {
        if (L.copies == 4u)
            launch_form<Form<64, 1, 4, 2>>(p, L, stream);
        else if (L.tiles == 1u)
            launch_form<Form<64, 1, 1, 1>>(p, L, stream);
        else
            launch_form<Form<64, 2, 1, 1>>(p, L, stream);
    } else {
        if (L.copies == 2u)
            launch_form<Form<128, 1, 2, 1>>(p, L, stream);
        else
            launch_form<Form<128, 1, 1, 1>>(p, L, stream);
    }
    return hip_status(hipGetLastError());
}

} // namespace lfm
