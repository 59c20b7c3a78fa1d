// attend.cuh -- what the attention kernels on tensor cores share.
//
// Scores are in powers of two: s = S log2(e).  The weights of the values are e^(S - m) s_v; with s_v = f 2^e, 1/2 <= f < 1, they are held as 2^(s + e - M) f, M the
// largest s + e of the row so far (not of s: pages whose s_v are far apart would lose the weights that count), which are at most 1 and f16 numbers for the product with the
// codes.  The sum below the line is 2^(s - m) with the row's largest s, in f32.  y = (sum of weights times codes) / (sum) 2^(M - m).
//
// Queries are f16 numbers: each row times the power of two that brings its largest magnitude to 2^14 .. 2^15.  f16 and bf16 values are those numbers exactly, but for those
// below 2^-28 of the row's largest, which are off by at most 2^-39 of it.
#pragma once
#include "cache.cuh"

namespace vqb {

constexpr float LOG2_E = 1.44269504088896341f;

// 2^x, x <= 0 or NaN (what is below 2^-126 is 0)
__device__ __forceinline__ float power_of_two(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two largest numbers so far, from a to b: what is relative to a times this is relative to b (nothing is relative to -infinity)
__device__ __forceinline__ float relative(float a, float b) { return a == -INFINITY ? 0.0f : power_of_two(a - b); }

// Four bytes of the cache as f16 numbers: 1024 + byte is the f16 number 0x6400 | byte, 1152 less is the code.
__device__ __forceinline__ void codes_to_halves(uint32_t four, uint32_t &low, uint32_t &high)
{
    const uint32_t exponent = 0x64646464u, minus = 0xE480E480u; // -1152 twice
    low = __byte_perm(four, exponent, 0x4140), high = __byte_perm(four, exponent, 0x4342);
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(low) : "r"(minus));
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(high) : "r"(minus));
}
__device__ __forceinline__ uint32_t halves_of_floats(float a, float b)
{
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(a), "f"(b));
    return d;
}

// What a row of queries with this largest magnitude (its bits) is multiplied by, and what its products with codes are multiplied by for the score (but for s_k).
struct QueryScale {
    float up, down;
    __device__ __forceinline__ QueryScale(uint32_t largest, float scale)
    {
        const int exponent = (int)(largest >> 23) - 127, k = min(14 - exponent, 126); // (f32 numbers below 2^-112 stay below 2^14: 2^126 is enough for bf16's smallest)
        const float factor = scale * LOG2_E;
        up = __int_as_float((k + 127) << 23);
        down = k <= 126 - 1 && k >= -126 ? factor * __int_as_float((127 - k) << 23) : ldexpf(factor, -k);
        if (largest == 0) up = 1.0f, down = factor;
        if (largest >= 0x7F800000u) up = 0.0f, down = __int_as_float(0x7FC00000);
    }
};

// s_k and s_v of a page and head as the kernels take them
struct PageScales {
    float k;
    float f; // s_v = f 2^e; 0 and NaN have e = 0
    float e;
    __device__ __forceinline__ PageScales(float2 s)
    {
        k = s.x;
        const uint32_t bits = __float_as_uint(s.y);
        const int exponent = (int)(bits >> 23);
        if (exponent == 0 || exponent == 255) { // (subnormal ones exactly: 2^24 times that, and back)
            const float big = s.y * 16777216.0f;
            const bool small = exponent == 0 && big > 0.0f;
            f = small ? __uint_as_float((__float_as_uint(big) & 0x7FFFFFu) | 0x3F000000u) : s.y;
            e = small ? (float)((int)(__float_as_uint(big) >> 23) - 126 - 24) : 0.0f;
        } else {
            f = __uint_as_float((bits & 0x7FFFFFu) | 0x3F000000u);
            e = (float)(exponent - 126);
        }
    }
};
// down s_k: what a row's products with a page's codes are multiplied by.  (Infinite only where any score but 0 is: 0 times that is to stay 0.)
__device__ __forceinline__ float score_factor(float down, float k)
{
    const float t = down * k;
    return fabsf(t) == INFINITY ? copysignf(3.4e38f, t) : t;
}

// The pages that rows at positions p0 .. p1 of a sequence see some of: the first sink_pages of its table, then those from column `begin` on.
struct Pages {
    int sink_pages, begin, count;
    __device__ __forceinline__ Pages(int p0, int p1, int keys, int window, int sinks)
    {
        const int last = min(p1, keys - 1), last_page = last < 0 ? -1 : last >> 6; // (column of the last token)
        begin = window ? max(max(p0, 0) - window + 1, 0) >> 6 : 0;
        sink_pages = min(min((int)(((unsigned)sinks + 63u) >> 6), begin), last_page + 1);
        count = sink_pages + max(last_page - begin + 1, 0);
    }
    __device__ __forceinline__ int column(int i) const { return i < sink_pages ? i : begin + i - sink_pages; }
};

// Whether all rows at positions p0 .. p1 see all of the tokens of a column.
__device__ __forceinline__ bool all_seen(int column, int p0, int p1, int keys, int window, int sinks)
{
    const int first = column * CACHE_PAGE, last = first + CACHE_PAGE - 1;
    return last <= p0 && last < keys && (!window || first > p1 - window || last < sinks);
}
__device__ __forceinline__ bool seen(int token, int position, int keys, int window, int sinks)
{
    return token <= position && token < keys && (!window || token > position - window || token < sinks);
}

} // namespace vqb
