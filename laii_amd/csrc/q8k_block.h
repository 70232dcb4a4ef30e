/*
 * q8k_block.h -- one 256-value Q8_K block quantized by one wave, shared by the
 * quantizer (quant_matmul.hip) and the norm that feeds it (norm_quant.hip).
 */
#ifndef LFM_Q8K_BLOCK_H
#define LFM_Q8K_BLOCK_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lfm {

constexpr uint32_t kQ8K = 292u; /* float d, int8 qs[256], int16 bsums[16] */

/* Lane l holds values 4 l .. 4 l + 3 of the block at `out` (4-byte aligned). */
__device__ __forceinline__ void quant_q8k_block(const float v[4], uint8_t *out, uint32_t lane) {
    float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if (amax == 0.0f) {
        *reinterpret_cast<uint32_t *>(out + 4u + 4u * lane) = 0u;
        if (lane < 16u) *reinterpret_cast<int16_t *>(out + 260u + 2u * lane) = 0;
        if (lane == 0u) *reinterpret_cast<float *>(out) = 0.0f;
        return;
    }
    const float d      = amax / 127.0f;  /* correctly rounded (HIP default) */
    const float iscale = 127.0f / amax;
    int32_t q[4], part = 0;
    uint32_t packed = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        q[i] = (int32_t)__builtin_rintf(v[i] * iscale); /* one rounding, then half-even */
        part += q[i];
        const int32_t s = q[i] > 127 ? 127 : (q[i] < -128 ? -128 : q[i]);
        packed |= (uint32_t)(uint8_t)(int8_t)s << (8 * i);
    }
    *reinterpret_cast<uint32_t *>(out + 4u + 4u * lane) = packed;
    part += __shfl_xor(part, 1);
    part += __shfl_xor(part, 2);
    if ((lane & 3u) == 0u) *reinterpret_cast<int16_t *>(out + 260u + (lane >> 1)) = (int16_t)part;
    if (lane == 0u) *reinterpret_cast<float *>(out) = d;
}

} // namespace lfm

#endif
