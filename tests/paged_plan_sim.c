/*
 * paged_plan_sim.c -- CPU simulation of the split of the paged attention
 * (k_paged_gqa_split / k_paged_merge), built on the header the kernels use
 * (laii_amd/csrc/paged_q4.h).  Test infrastructure: compiled by
 * tests/test_paged_q4_plan.py with gcc and called through ctypes.
 *
 * plan_check() runs every wave's walk as the kernel does, joins the pieces of
 * a workgroup's waves, records every direct output and partial slot, and runs
 * the merge's slot range for every unit.  It checks:
 *   - every (row, head, key) that the formula attends is covered by exactly one
 *     piece, and every query column that counts lies in one tile;
 *   - shares differ by one step at most, and are contiguous;
 *   - partial slots are unique and below workgroups + units;
 *   - a unit has one direct output and no partials, or the merge reads exactly
 *     the slots written for it.
 * Returns 0, or a negative code with a message in msg.
 *
 * mutant != 0 plants a mistake in the simulated walk (1: slots without the
 * workgroup; 2: the range's end one early; 3: a tile's last row left out),
 * which the checks must reject.
 */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "paged_q4.h"

typedef struct {
    uint32_t unit, a, b, n; /* steps [a, b) of the unit's n; unit ~0: none */
} piece;

#define FAIL(code, ...)                                                                                               \
    do {                                                                                                              \
        snprintf(msg, msg_len, __VA_ARGS__);                                                                          \
        rc = code;                                                                                                    \
        goto out;                                                                                                     \
    } while (0)

void share(uint32_t g, uint32_t n_steps, uint32_t G, uint32_t *t0, uint32_t *t1) { lfm_q4_share(g, n_steps, G, t0, t1); }

int plan_check(uint32_t n_seq, const uint32_t *pos0, const uint32_t *rows_seq, uint32_t n_rows, uint32_t kv_mul,
               uint32_t n_head_kv, uint32_t window, uint32_t capacity, uint32_t cols, uint32_t step_shift,
               uint32_t n_waves, int mutant, char *msg, size_t msg_len) {
    int rc              = 0;
    const uint32_t n_ct = (n_rows * kv_mul + cols - 1u) / cols;
    const lfm_q4_plan p = {n_seq, n_rows, kv_mul, n_head_kv, window, capacity, cols, step_shift, n_ct, n_waves};
    const uint32_t n_e = n_seq * n_ct, units = n_e * n_head_kv, n_wg = n_waves / 4u, n_slots = n_wg + units;
    uint32_t *steps = calloc(n_e, 4), *rows = calloc(n_seq, 4);
    uint32_t *done  = calloc(units, 4);    /* steps covered, in order */
    uint32_t *first = calloc(units, 4), *last = calloc(units, 4);
    int *direct = calloc(units, sizeof(int)), *written = calloc(units, sizeof(int));
    uint32_t *owner = malloc(n_slots * 4ull);
    memset(owner, 0xFF, n_slots * 4ull);
    uint64_t total = 0;

    for (uint32_t s = 0; s < n_seq; ++s) {
        rows[s]       = lfm_q4_rows(pos0[s], rows_seq ? rows_seq[s] : n_rows, n_rows, capacity);
        uint64_t want = pos0[s] < capacity ? capacity - pos0[s] : 0;
        if (rows_seq ? want > rows_seq[s] : 0) want = rows_seq[s];
        if (want > n_rows) want = n_rows;
        if (rows[s] != want) FAIL(-1, "seq %u: %u rows", s, rows[s]);
        /* columns: tile ct holds row * kv_mul + head in [ct cols, (ct + 1) cols) */
        for (uint32_t ct = 0; ct < n_ct; ++ct) {
            lfm_q4_tile t = lfm_q4_tile_of(&p, pos0[s], rows[s], ct);
            if (mutant == 3 && t.n_steps > 1u) t.n_steps -= 1u;
            steps[s * n_ct + ct] = t.n_steps;
            total += t.n_steps;
            const uint64_t c0 = (uint64_t)ct * cols, c1 = c0 + cols < (uint64_t)rows[s] * kv_mul ? c0 + cols : (uint64_t)rows[s] * kv_mul;
            if ((t.n_steps == 0u) != (c0 >= c1)) FAIL(-2, "seq %u tile %u: %u steps", s, ct, t.n_steps);
            for (uint64_t c = c0; c < c1; ++c) {
                const uint32_t r = (uint32_t)(c / kv_mul), pos = pos0[s] + r;
                const uint32_t lo = window && pos + 1u > window ? pos + 1u - window : 0u;
                if (r < t.r0 || r >= t.r1) FAIL(-3, "seq %u tile %u: row %u", s, ct, r);
                if (lfm_q4_row_lo(pos, window) != lo) FAIL(-4, "row_lo");
                const uint64_t end = (uint64_t)(t.step0 + t.n_steps) << step_shift;
                if (((uint64_t)t.step0 << step_shift) > lo || end <= pos)
                    FAIL(-5, "seq %u tile %u row %u: keys [%u, %u] in steps %u + %u", s, ct, r, lo, pos, t.step0, t.n_steps);
                if ((((uint64_t)t.step0 + t.n_steps - 1u) << step_shift) >= capacity) FAIL(-6, "a step behind the table");
            }
        }
    }
    total *= n_head_kv;
    if (total >= 0x80000000ull) FAIL(-7, "case too large");
    const uint32_t N = (uint32_t)total, G = lfm_q4_waves(&p, N);
    uint32_t at = 0, e = 0, base = 0; /* the walk's place: entry e, steps before it */
    for (uint32_t g = 0; g < n_wg; ++g) {
        piece ps[8];
        for (int i = 0; i < 8; ++i) ps[i].unit = ~0u;
        for (uint32_t w = 0; w < 4u; ++w) {
            const uint32_t wave = g * 4u + w;
            uint32_t t = 0, t1 = 0;
            if (wave < G) {
                lfm_q4_share(wave, N, G, &t, &t1);
                if (t != at || t1 <= t || t1 - t > N / G + 1u) FAIL(-8, "share of wave %u: [%u, %u)", wave, t, t1);
                at = t1;
            }
            const uint32_t t0 = t;
            while (t < t1) {
                while ((base + steps[e]) * n_head_kv <= t) base += steps[e++];
                const uint32_t n = steps[e];
                uint32_t h = (t - base * n_head_kv) / n, a = t - base * n_head_kv - h * n;
                for (; t < t1 && h < n_head_kv; ++h, a = 0u) {
                    const uint32_t b = n - a < t1 - t ? n : a + (t1 - t), unit = e * n_head_kv + h;
                    if (done[unit] != a) FAIL(-9, "unit %u: step %u after %u", unit, a, done[unit]);
                    done[unit] = b;
                    if (a == 0u && b == n) {
                        direct[unit] += 1;
                        first[unit] = last[unit] = g;
                    } else {
                        piece *q = &ps[w * 2u + (t == t0 ? 0u : 1u)];
                        if (q->unit != ~0u) FAIL(-10, "wave %u: a third part", wave);
                        *q = (piece){unit, a, b, n};
                    }
                    t += b - a;
                }
            }
        }
        for (int i = 0; i < 8; ++i) {
            if (ps[i].unit == ~0u) continue;
            const uint32_t unit = ps[i].unit, n = ps[i].n, a = ps[i].a;
            uint32_t b = ps[i].b;
            for (int k = i + 1; k < 8; ++k)
                if (ps[k].unit == unit) {
                    if (ps[k].a != b) FAIL(-11, "unit %u: pieces of a workgroup", unit);
                    b          = ps[k].b;
                    ps[k].unit = ~0u;
                }
            if (a == 0u) first[unit] = g;
            if (b == n) last[unit] = g;
            if (a == 0u && b == n) {
                direct[unit] += 1;
            } else {
                const uint32_t slot = (mutant == 1 ? 0u : g) + unit;
                if (slot >= n_slots || owner[slot] != ~0u) FAIL(-12, "slot %u of unit %u", slot, unit);
                owner[slot] = unit;
                written[unit] += 1;
            }
        }
    }
    if (at != N) FAIL(-13, "%u of %u steps", at, N);
    for (uint32_t u = 0; u < units; ++u) {
        const uint32_t n = steps[u / n_head_kv];
        if (done[u] != n) FAIL(-14, "unit %u: %u of %u steps", u, done[u], n);
        if (n == 0u) continue;
        if (direct[u] + (written[u] > 0) != 1) FAIL(-15, "unit %u: %d direct, %d partials", u, direct[u], written[u]);
        const uint32_t g0 = first[u], g1 = last[u] - (mutant == 2 && last[u] ? 1u : 0u);
        if (direct[u] ? g0 < g1 : g0 >= g1) FAIL(-16, "unit %u: range [%u, %u]", u, g0, g1);
        if (g1 >= n_wg) FAIL(-17, "unit %u: range past the launch", u);
        int met = 0;
        for (uint32_t g = g0; !direct[u] && g <= g1; ++g) {
            if (owner[g + u] != u) FAIL(-18, "unit %u: slot %u", u, g + u);
            ++met;
        }
        if (met != written[u]) FAIL(-19, "unit %u: %d of %d partials", u, met, written[u]);
    }
out:
    free(steps), free(rows), free(done), free(first), free(last), free(direct), free(written), free(owner);
    return rc;
}
