/*
 * paged_q4.h -- layout of the paged 4-bit K/V cache and the integer plan of
 * the attention over it.  Compiled into the kernels and into the host launch
 * code, so the index math the tests check is the math the device runs.
 *
 * A page holds page_size positions (a power of two, at least 32) as
 * [KV head][block of 32 positions].  A block of head_dim D is 36 D bytes:
 *   K codes   16 D   a word holds 8 dims of one position: the lane that needs it
 *                    as an MFMA A operand (row = key, 8 consecutive k) loads
 *                    16 bytes at 16 * lane and has all its words
 *   V codes   16 D   a word holds 8 positions of one dim: the transpose that the
 *                    P.V product needs is made once, when a row is stored
 *   K scales   2 D   fp16 [group of 32 dims][position], positions in V's order
 *   V scales   2 D   the same
 * Value of code c under scale d: d * (c - 8).
 */
#ifndef LFM_PAGED_Q4_H
#define LFM_PAGED_Q4_H

#include <stddef.h>
#include <stdint.h>

#include "attn_index.h"

#define LFM_Q4_BLOCK 32u

LFM_IDX_FN uint32_t lfm_q4_block_bytes(uint32_t head_dim) { return 36u * head_dim; }

/* Nibble of a word that holds its element e = 0..7: elements 2i and 2i + 1 are
 * the two 16-bit halves' nibble i, so one AND gives both as a packed pair. */
LFM_IDX_FN uint32_t lfm_q4_nibble(uint32_t e) { return (e >> 1) + 4u * (e & 1u); }

/* Byte of the K word holding dims 32 g + 8 part .. + 7 of position t < 32. */
LFM_IDX_FN uint32_t lfm_q4_k_word(uint32_t head_dim, uint32_t t, uint32_t g, uint32_t part) {
    const uint32_t half = t >> 4, lane = part * 16u + (t & 15u);
    return head_dim == 64u ? lane * 16u + half * 8u + g * 4u : half * 1024u + lane * 16u + g * 4u;
}

/* V words hold positions 4 kg .. 4 kg + 3 and 16 + the same: the keys a lane
 * group has after the S product.  kg and element of position t < 32: */
LFM_IDX_FN uint32_t lfm_q4_kg(uint32_t t) { return (t >> 2) & 3u; }
LFM_IDX_FN uint32_t lfm_q4_elem(uint32_t t) { return (t & 3u) + 4u * (t >> 4); }

/* Byte (from the block) of the V word of key group kg and dim x. */
LFM_IDX_FN uint32_t lfm_q4_v_word(uint32_t head_dim, uint32_t kg, uint32_t x) {
    return 16u * head_dim + (x >> 6) * 1024u + (kg * 16u + (x & 15u)) * 16u + ((x >> 4) & 3u) * 4u;
}

/* Byte of the K (v = 0) or V (v = 1) scale of position t and dim group g. */
LFM_IDX_FN uint32_t lfm_q4_scale(uint32_t head_dim, uint32_t v, uint32_t t, uint32_t g) {
    return (32u + 2u * v) * head_dim + g * 64u + lfm_q4_kg(t) * 16u + lfm_q4_elem(t) * 2u;
}

/* ---- attention: units, steps, shares -------------------------------------------
 * The query columns of a (sequence, KV head) are its rows x kv_mul query heads,
 * row major, cut into tiles of `cols`.  A unit is (sequence, tile, KV head),
 * numbered in that order; its work is the steps of 2^step_shift keys that cover
 * the keys its rows attend.  The batch's N < 2^32 steps, in unit order, go to G
 * waves in shares equal to within one step, cut at units.  The pieces
 * of a workgroup's waves join in LDS; what workgroup g then holds of unit v, if
 * not all of it, has partial slot g + v: along the walk g or v grows, so slots
 * are unique and below workgroups + units.  Everything here is 32-bit: a 64-bit division costs a wave more than
 * a step of keys. */
typedef struct {
    uint32_t n_seq, n_rows, kv_mul, n_head_kv;
    uint32_t window;     /* 0: none                                      */
    uint32_t capacity;   /* positions a sequence's table reaches, <= 2^31 */
    uint32_t cols;       /* query columns per tile                       */
    uint32_t step_shift; /* log2 of the keys per step, at least 5        */
    uint32_t n_ct;       /* tiles per sequence                           */
    uint32_t n_waves;    /* waves launched                               */
} lfm_q4_plan;

/* Rows of a sequence that count: of its n_rows_seq (or all n_rows) those whose
 * positions the table reaches.  No position of such a row exceeds 2^31. */
LFM_IDX_FN uint32_t lfm_q4_rows(uint32_t pos0, uint32_t rows, uint32_t n_rows, uint32_t capacity) {
    const uint32_t room = pos0 < capacity ? capacity - pos0 : 0u;
    if (rows > n_rows) rows = n_rows;
    return rows < room ? rows : room;
}

/* Rows and steps of tile ct of a sequence whose `rows` rows that count start
 * at position pos0.  n_steps 0: the tile has no rows. */
typedef struct {
    uint32_t r0, r1; /* rows [r0, r1) */
    uint32_t step0, n_steps;
} lfm_q4_tile;

LFM_IDX_FN uint32_t lfm_q4_row_lo(uint32_t pos, uint32_t window) {
    return window > 0u && pos >= window ? pos - window + 1u : 0u;
}

LFM_IDX_FN lfm_q4_tile lfm_q4_tile_of(const lfm_q4_plan *p, uint32_t pos0, uint32_t rows, uint32_t ct) {
    lfm_q4_tile t;
    t.r0 = t.r1 = t.step0 = t.n_steps = 0u;
    if (p->n_ct == 1u) { /* one tile holds every row */
        t.r1 = rows;
    } else {
        const uint32_t cols = rows * p->kv_mul, c0 = ct * p->cols;
        if (c0 >= cols) return t;
        const uint32_t c1 = cols - c0 < p->cols ? cols : c0 + p->cols;
        t.r0              = c0 / p->kv_mul;
        t.r1              = (c1 - 1u) / p->kv_mul + 1u;
    }
    if (t.r1 == 0u) return t;
    t.step0   = lfm_q4_row_lo(pos0 + t.r0, p->window) >> p->step_shift;
    t.n_steps = ((pos0 + t.r1 - 1u) >> p->step_shift) + 1u - t.step0;
    return t;
}

/* Waves taking part, for N steps in all. */
LFM_IDX_FN uint32_t lfm_q4_waves(const lfm_q4_plan *p, uint32_t n_steps) {
    return n_steps < p->n_waves ? n_steps : p->n_waves;
}

/* Steps [*t0, *t1) of wave g < G <= 2048: from floor(g N / G), so that a batch of
 * equal units is cut at every unit when G is a multiple of their number (a wave
 * with the end of one and the start of the next has two beginnings to wait for). */
LFM_IDX_FN void lfm_q4_share(uint32_t g, uint32_t n_steps, uint32_t G, uint32_t *t0, uint32_t *t1) {
    const uint32_t q = n_steps / G, r = n_steps - q * G;
    *t0 = g * q + g * r / G;
    *t1 = (g + 1u) * q + (g + 1u) * r / G;
}

#endif
