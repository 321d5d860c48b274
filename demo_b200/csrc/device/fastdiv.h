/* Unsigned 32-bit division by a run-time constant: q = (umulhi(n, m) + n) >> s
 * with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1 (Granlund and
 * Montgomery, "Division by invariant integers using multiplication", 1994). */
#ifndef FASTDIV_H
#define FASTDIV_H

#include <cstdint>

struct FastDiv {
    uint32_t d, m, s;
};

static inline FastDiv make_fastdiv(uint32_t d)
{
    FastDiv f;
    uint32_t s = 0;
    while ((1ull << s) < d)
        s++;
    f.d = d;
    f.s = s;
    f.m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
    return f;
}

static __device__ __forceinline__ uint32_t fdiv(uint32_t n, const FastDiv &f)
{
    return (uint32_t)(((uint64_t)__umulhi(n, f.m) + n) >> f.s);
}

#endif
