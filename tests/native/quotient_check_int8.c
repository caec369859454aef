/* Every (max|x|, x) pair of non-negative BF16 values with x <= max|x| and max|x| = 0 or in [2^-60,
 * largest finite]: the int8 code of the two-FMA quotient that the 8-bit cache's write forms equals
 * the code of the IEEE quotient, s = max|x| / 127.  Both are rounded as the kernel does, by adding
 * 1.5 * 2^23.  Prints the number of differences. */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

static float from_bits(uint32_t u) {
    float f;
    memcpy(&f, &u, 4);
    return f;
}

static int32_t code(float q) {
    volatile float r = q + 12582912.0f;
    float f = r;
    int32_t u;
    memcpy(&u, &f, 4);
    return (int8_t)(u & 0xFF);
}

int main(void) {
    long long bad = 0, pairs = 0;
#pragma omp parallel for schedule(dynamic, 64) reduction(+ : bad, pairs)
    for (uint32_t a = 0; a < 0x7F80u; ++a) {
        const uint32_t bits = a << 16;
        if (a != 0 && bits < 0x21800000u) continue;
        const float amax = from_bits(bits);
        float s = amax / 127.0f;
        if (s == 0.0f) s = 1.0f;
        const float r = 1.0f / s;
        for (uint32_t x = 0; x <= a; ++x) {
            const float v = from_bits(x << 16);
            const float q0 = v * r;
            const float e = fmaf(-q0, s, v);
            const float q = fmaf(e, r, q0);
            const int32_t want = (int32_t)nearbyintf(v / s);
            if (code(q) != want || code(-q) != -want || want > 127) ++bad;
            ++pairs;
        }
    }
    printf("%lld pairs, %lld differences\n", pairs, bad);
    return bad != 0;
}
