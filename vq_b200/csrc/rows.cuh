// rows.cuh -- the arithmetic of rows.cu: pieces of a row, its scale, its codes.
//
// The code is the nearest whole number to the REAL quotient x / s (halves to even), so that it depends on nothing but x and the
// row's largest magnitude.  1 / s lies between two neighbouring f32 numbers; where x times either rounds to the same whole number, that is
// the code, and elsewhere (the quotient is next to a half h) the sign of x - h s decides, which one fused multiply-add gives exactly.
#pragma once
#include <type_traits>

#include "qmat.cuh"

namespace vqb {

constexpr float MAGIC = 12582912.0f; // 1.5 2^23: adding it rounds to a whole number, whose two's complement is then in the low bits
constexpr float LARGEST_8 = 127.0f, LARGEST_24 = 127.0f * 65536.0f; // the first of three digits stays within 127 (127.5 would)

template <typename T> struct Piece; // 16 bytes of a row
template <> struct Piece<float> {
    static constexpr int N = 4;
    uint4 w;
    __device__ __forceinline__ float at(int i) const { return __uint_as_float((&w.x)[i]); }
};
template <> struct Piece<__half> {
    static constexpr int N = 8;
    uint4 w;
    __device__ __forceinline__ float at(int i) const { return __half2float(__ushort_as_half((unsigned short)((&w.x)[i >> 1] >> (16 * (i & 1))))); }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr int N = 8;
    uint4 w;
    __device__ __forceinline__ float at(int i) const { return __uint_as_float((i & 1) ? ((&w.x)[i >> 1] & 0xFFFF0000u) : ((&w.x)[i >> 1] << 16)); }
};

// Which columns a lane has.  Where rows and codes are aligned: N neighbouring ones a piece, 16 bytes loaded and N stored at once.  Elsewhere
// every LANESth column: 4 or 2 bytes a lane, but a warp's are next to each other.
template <int N, int LANES, bool ALIGNED> __device__ __forceinline__ uint32_t column(uint32_t piece, int lane, int i)
{
    return ALIGNED ? (piece * LANES + lane) * N + i : (piece * N + i) * LANES + lane;
}

// a piece of a row, 0 behind its end
template <typename T, int LANES, bool ALIGNED> __device__ __forceinline__ Piece<T> load_values(const T *row, uint32_t piece, int lane, uint32_t width)
{
    constexpr int N = Piece<T>::N;
    Piece<T> p;
    p.w = make_uint4(0, 0, 0, 0);
    const uint32_t k = column<N, LANES, ALIGNED>(piece, lane, 0);
    if (ALIGNED && k + N <= width) {
        p.w = *reinterpret_cast<const uint4 *>(row + k);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t at = column<N, LANES, ALIGNED>(piece, lane, i);
            if (at < width) {
                if (sizeof(T) == 4) (&p.w.x)[i] = reinterpret_cast<const uint32_t *>(row)[at];
                else (&p.w.x)[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t *>(row)[at] << (16 * (i & 1));
            }
        }
    }
    return p;
}

// two f32 at a time
__device__ __forceinline__ uint64_t pair_of(float a, float b)
{
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void halves_of(uint64_t d, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// max(|a|, |b|) of two 16-bit floats each, with whatever sign; NaN wins
template <typename T> __device__ __forceinline__ uint32_t larger_pair(uint32_t a, uint32_t b)
{
    uint32_t d;
    if (std::is_same<T, __half>::value) asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ float larger(float a, float b)
{
    float d;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// whole numbers of magnitudes up to 127 as bytes
template <int N> struct Packed {
    uint32_t w[N / 4];
};

// What a row's values are multiplied by: the f32 numbers on both sides of 1 / scale.
struct Inverse {
    float scale, nearest;
    uint64_t up, down;
    __device__ __forceinline__ explicit Inverse(float s) : scale(s)
    {
        nearest = __frcp_rn(s);
        const float u = __uint_as_float(__float_as_uint(nearest) + 1), d = __uint_as_float(__float_as_uint(nearest) - 1);
        up = pair_of(u, u), down = pair_of(d, d);
    }
};

template <int N> __device__ __forceinline__ Packed<N> low_bytes(const float (&m)[N])
{
    Packed<N> out;
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
        out.w[i] = __byte_perm(__byte_perm(__float_as_uint(m[4 * i]), __float_as_uint(m[4 * i + 1]), 0x0040),
                               __byte_perm(__float_as_uint(m[4 * i + 2]), __float_as_uint(m[4 * i + 3]), 0x0040), 0x5410);
    return out;
}

// The codes, unless some quotient is next to a half: then a half of `unlike` becomes positive.
template <int N> __device__ __forceinline__ Packed<N> pack_most(const float (&v)[N], const Inverse &inverse, uint64_t &unlike)
{
    const uint64_t magic = pair_of(MAGIC, MAGIC), minus = pair_of(-1.0f, -1.0f);
    float m[N];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const uint64_t pair = pair_of(v[i], v[i + 1]), u = fma_pair(pair, inverse.up, magic), d = fma_pair(pair, inverse.down, magic);
        const uint64_t off = fma_pair(d, minus, u);
        unlike = fma_pair(off, off, unlike);
        halves_of(u, m[i], m[i + 1]);
    }
    return low_bytes<N>(m);
}
__device__ __forceinline__ bool any_unlike(uint64_t unlike)
{
    float a, b;
    halves_of(unlike, a, b);
    return a + b > 0.0f;
}

// The codes, whatever the quotients.  r = v times a neighbour of 1 / s, to a whole number, is right or one off; e = v - r s is exact (a multiple of half the last place
// of s, and not above 1.5 s) and says which: beyond s / 2, or s / 2 itself with r odd, r moves towards v.  In 16-bit rows halves are not rare (v and the row's largest are
// eight-bit numbers): this is taken for one piece in some ten.
template <int N> __device__ __forceinline__ Packed<N> pack_all(const float (&v)[N], const Inverse &inverse)
{
    float up, unused;
    halves_of(inverse.up, up, unused);
    // twice the values where e could be below what f32 holds
    const float twice = inverse.scale < 1.0f ? 2.0f : 1.0f, s = inverse.scale * twice;
    const uint32_t half = __float_as_uint(0.5f * s);
    float m[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = __fmaf_rn(v[i], up, MAGIC), e = __fmaf_rn(-__fsub_rn(t, MAGIC), s, v[i] * twice);
        const float border = __uint_as_float(half - (__float_as_uint(t) & 1u)); // (odd: the next number below)
        uint32_t bits = __float_as_uint(t);
        if (e > border) ++bits;
        if (e < -border) --bits;
        m[i] = __uint_as_float(bits);
    }
    return low_bytes<N>(m);
}

template <int N> __device__ __forceinline__ Packed<N> pack_codes(const float (&v)[N], const Inverse &inverse)
{
    uint64_t unlike = 0;
    const Packed<N> out = pack_most<N>(v, inverse, unlike);
    return __builtin_expect(any_unlike(unlike), 0) ? pack_all<N>(v, inverse) : out;
}

// The three digits of the whole number v next to u / t, |v| <= 127 * 65536: v = 65536 d0 + 256 d1 + d2, each in -128 .. 127.  They are the bytes of
// v + 0x808080, which is positive and below 2^24, less 128 each.  (v is off by at most half a step, and 2^-24 of v for the reciprocal and 2^-25 for the product.)
template <int N> __device__ __forceinline__ void pack_digits(const float (&u)[N], const Inverse &inverse, Packed<N> (&digits)[3])
{
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (uint32_t)(__float2int_rn(__fmul_rn(u[4 * i + j], inverse.nearest)) + 0x808080);
        const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140); // the last and the middle digits of two
        digits[2].w[i] = __byte_perm(a, b, 0x5410) ^ 0x80808080u;
        digits[1].w[i] = __byte_perm(a, b, 0x7632) ^ 0x80808080u;
        digits[0].w[i] = __byte_perm(__byte_perm(w[0], w[1], 0x0062), __byte_perm(w[2], w[3], 0x0062), 0x5410) ^ 0x80808080u;
    }
}

template <int N, int LANES, bool ALIGNED> __device__ __forceinline__ void store_codes(int8_t *row, uint32_t piece, int lane, uint32_t width, const Packed<N> &c)
{
    const uint32_t k = column<N, LANES, ALIGNED>(piece, lane, 0);
    if (ALIGNED && k + N <= width) {
        if (N == 8) *reinterpret_cast<uint2 *>(row + k) = make_uint2(c.w[0], c.w[N / 4 - 1]);
        else *reinterpret_cast<uint32_t *>(row + k) = c.w[0];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t at = column<N, LANES, ALIGNED>(piece, lane, i);
            if (at < width) row[at] = (int8_t)(c.w[i >> 2] >> (8 * (i & 3)));
        }
    }
}

struct RowParams {
    const void *x;
    size_t n, ld;
    uint32_t width;
    int8_t *codes;
    size_t ld_codes, plane; // plane: bytes from a digit's rows to the next digit's (three digits)
    float *scales;
    const float *column_scales; // groups x width (three digits)
    const long long *offsets;
    int groups;
    bool product_follows; // the next kernel of the stream is a product of this call
};

// One row's arithmetic on pieces of it.
template <typename T, int DIGITS, int LANES, bool ALIGNED> struct RowOf {
    static constexpr int N = Piece<T>::N;
    const RowParams &P;
    size_t r;
    int lane;
    const float *columns;
    bool columns4; // N neighbouring columns' scales are 16-byte aligned
    uint32_t most = 0;

    __device__ __forceinline__ RowOf(const RowParams &p, size_t row, int l, const float *c) : P(p), r(row), lane(l), columns(c), columns4(DIGITS == 3 && ALIGNED && p.width % 4 == 0) {}

    __device__ __forceinline__ void values(const Piece<T> &p, uint32_t piece, float (&v)[N]) const
    {
        float c[N];
        if (DIGITS == 3) {
            const uint32_t k = column<N, LANES, ALIGNED>(piece, lane, 0);
            if (columns4 && k + N <= P.width) {
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(columns + k + i);
                    c[i] = f.x, c[i + 1] = f.y, c[i + 2] = f.z, c[i + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint32_t at = column<N, LANES, ALIGNED>(piece, lane, i);
                    c[i] = at < P.width ? columns[at] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = DIGITS == 3 ? p.at(i) * c[i] : p.at(i);
    }
    // the largest magnitude so far (two 16-bit ones at a time); its sign means nothing, NaN wins
    __device__ __forceinline__ void look(const Piece<T> &p, uint32_t piece)
    {
        if (DIGITS == 1 && sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) most = larger_pair<T>(most, (&p.w.x)[i]);
        } else {
            float v[N];
            values(p, piece, v);
            look(v);
        }
    }
    __device__ __forceinline__ void look(const float (&v)[N])
    {
#pragma unroll
        for (int i = 0; i < N; ++i) most = __float_as_uint(larger(__uint_as_float(most), v[i]));
    }
    // the largest magnitude's bits, of the whole warp (their order is that of the magnitudes, infinities and NaN on top)
    __device__ __forceinline__ uint32_t largest() const
    {
        uint32_t m = most & 0x7FFFFFFFu;
        if (DIGITS == 1 && sizeof(T) == 2) {
            Piece<T> one;
            one.w = make_uint4(max(most & 0x7FFFu, (most >> 16) & 0x7FFFu), 0, 0, 0);
            m = __float_as_uint(one.at(0)); // (a NaN stays one)
        }
        return __reduce_max_sync(~0u, m);
    }
    static __device__ __forceinline__ bool no_codes(uint32_t largest) { return largest == 0 || largest >= 0x7F800000u; }
    static __device__ __forceinline__ float scale_of(uint32_t largest)
    {
        if (largest >= 0x7F800000u) return __int_as_float(0x7FC00000);
        return largest == 0 ? 0.0f : fmaxf(__fdiv_rn(__uint_as_float(largest), DIGITS == 1 ? LARGEST_8 : LARGEST_24), 0x1p-126f);
    }
    __device__ __forceinline__ void pack(const Piece<T> &p, uint32_t piece, const Inverse &inverse, Packed<N> (&digits)[DIGITS]) const
    {
        float v[N];
        values(p, piece, v);
        if constexpr (DIGITS == 1) digits[0] = pack_codes<N>(v, inverse);
        else pack_digits<N>(v, inverse, digits);
    }
    __device__ __forceinline__ void write(const Piece<T> &p, uint32_t piece, bool none, const Inverse &inverse) const
    {
        Packed<N> digits[DIGITS] = {};
        if (!none) pack(p, piece, inverse, digits);
        store(piece, digits);
    }
    // a whole piece, aligned
    __device__ __forceinline__ void put(uint32_t piece, const Packed<N> (&digits)[DIGITS]) const
    {
        int8_t *to = P.codes + r * P.ld_codes + column<N, LANES, true>(piece, lane, 0);
#pragma unroll
        for (int d = 0; d < DIGITS; ++d, to += P.plane) {
            if (N == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(digits[d].w[0], digits[d].w[N / 4 - 1]);
            else *reinterpret_cast<uint32_t *>(to) = digits[d].w[0];
        }
    }
    __device__ __forceinline__ void store(uint32_t piece, const Packed<N> (&digits)[DIGITS]) const
    {
#pragma unroll
        for (int d = 0; d < DIGITS; ++d) store_codes<N, LANES, ALIGNED>(P.codes + d * P.plane + r * P.ld_codes, piece, lane, P.width, digits[d]);
    }
};

} // namespace vqb
