/*
 * Exhaustive check of the 4-bit quantizer's divisions (TEST INFRASTRUCTURE ONLY), against C's IEEE division.
 *
 *  reciprocal  y1 = RN(y0 + y0 RN(1 - s y0)), one step of Newton's iteration, for a block scale s of four significant
 *              bits and an approximation y0 up to two units in the last place off (rcp.approx.ftz is documented to
 *              be within one): y1 = RN(1 / s).
 *  quotient    q0 = RN(v y), r = RN(v - q0 s) (exact), q = RN(q0 + r y) with y = RN(1 / s), the correction step of
 *              Markstein's division (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000
 *              processor", IBM J. Res. Dev. 34(1), 1990): q = RN(v / s), for every significand of v.
 *  sixth       the same step with y = RN(1 / 6): t / 6.
 *
 * Scales are 2^-9 to 448 and quotients matter from the code grid's first border on, 0.25: v and t are 2^-11 or more where
 * a code or a scale can hang on them, 2^100 above where a residue loses bits, so each result scales exactly with the
 * exponents of v, t and s, and one binade of each stands for all.  Prints checks and mismatches of the three.
 */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

static float from_bits(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static uint32_t to_bits(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }

int main(void) {
    long long checked[3] = {0, 0, 0}, wrong[3] = {0, 0, 0};
    for (int m = 8; m < 16; ++m) {
        const float s = (float)m / 8.0f, exact = 1.0f / s;
        for (int off = -2; off <= 2; ++off) {
            const float y0 = from_bits(to_bits(exact) + (uint32_t)off);
            const float y1 = fmaf(y0, fmaf(-s, y0, 1.0f), y0);
            ++checked[0];
            wrong[0] += to_bits(y1) != to_bits(exact);
        }
        for (uint32_t i = 0; i < (2u << 23); ++i) {
            const float v = from_bits((i >> 23 << 31) | (127u << 23) | (i & 0x7fffffu));
            const float q0 = -v * -exact;
            const float q = fmaf(fmaf(q0, s, -v), -exact, q0); /* the kernel's signs */
            ++checked[1];
            wrong[1] += to_bits(q) != to_bits(v / s);
        }
    }
    for (uint32_t i = 0; i < (1u << 23); ++i) {
        const float t = from_bits((127u << 23) | i), c = 1.0f / 6.0f;
        const float q = t * c;
        ++checked[2];
        wrong[2] += to_bits(fmaf(fmaf(q, -6.0f, t), c, q)) != to_bits(t / 6.0f);
    }
    for (int i = 0; i < 3; ++i) printf("%lld %lld\n", checked[i], wrong[i]);
    return wrong[0] || wrong[1] || wrong[2];
}
