// cache.cu -- tokens into the pages of a cache of 8-bit codes, and back.
//
//   scale s of a page and head = max(s_old, max |x| / 127, 2^-126), code = x / s to the nearest whole number, codes that stay: code s_old / s to the nearest
//
// One block for each page that the call touches, head, and of keys and values: nobody else writes there, and the largest magnitude of all its new tokens is
// known before the first code.  The floor is memory, size + 1 bytes a value; writing and reading take two to three times that (16,558 tokens of 8 heads x 128 in bf16: written in 50 us,
// read in 28, for 15 and 15).  What bounds them is the values' turn through shared memory, a byte at a time, and the instructions for it: 64 to 66 % of the issue slots, memory 18 % of its peak.
#include <algorithm>

#include "cache.cuh"
#include "cuda_device.hpp"
#include "rows.cuh"

namespace vqb {

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int PITCH = CACHE_PAGE + 4; // of a dimension's row in shared memory: 17 banks

struct CacheRows {
    Cache c;
    Sequences s;
    HeadRows x[2]; // keys, values
};

// The part of a page that a block has: tokens a .. b - 1 are rows row .. of the call, for head blockIdx.y of keys or values (blockIdx.z).
struct Part {
    int page, a, b, row;
    __device__ __forceinline__ bool find(const Cache &c, const Sequences &s)
    {
        const int i = sequence_of(s, blockIdx.x, CACHE_PAGE, 2), m = (int)blockIdx.x - offset_of(s, i) / CACHE_PAGE - 2 * i;
        const Span span(s, i);
        const int column = floor_page(span.first) + m, from = column * CACHE_PAGE - span.first; // (row of the page's first token)
        if (m < 0 || span.count == 0 || from >= span.count) return false;
        a = max(-from, 0), b = min(span.count - from, CACHE_PAGE), row = span.row + from + a;
        page = page_of(s, c.pages, i, column);
        return true;
    }
};
__device__ __forceinline__ uint8_t *codes_of(const Cache &c, int page, int head, int which)
{
    return c.codes + (((size_t)page * c.heads + head) * 2 + which) * CACHE_PAGE * c.padded;
}
__device__ __forceinline__ float *scale_of(const Cache &c, int page, int head, int which) { return c.scales + ((size_t)page * c.heads + head) * 2 + which; }

// blocks that are enough for the pages of n rows of so many sequences (sequence_of)
inline unsigned parts_of(const Sequences &s) { return (unsigned)(s.n / CACHE_PAGE + 2 * s.sequences); }

constexpr uint32_t ZEROS = 0x01010101u * Cache::ZERO; // four bytes that stand for 0; a byte is the code with its first bit turned

// Four codes' bytes of scale `old` in the new one; the quotient's nearest whole number in 64 bits is the real quotient's (|code old / scale - (k + 1/2)| is 0 or more than 2^-31).
__device__ __forceinline__ uint32_t codes_again(uint32_t four, float old, float scale)
{
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int q = (int)(four >> (8 * i) & 255u) - 128;
        out |= (uint32_t)(__double2int_rn((double)q * old / scale) + 128) << (8 * i);
    }
    return out;
}

// Numbers below 64 x 256 in rows of `length`: division by multiplication with the reciprocal, half a step up (exact: i / length + 1 / (2 length) is 2^-9 or more from the next whole number).
struct Rows {
    int length;
    float inverse;
    __device__ __forceinline__ explicit Rows(int l) : length(l), inverse(1.0f / (float)l) {}
    __device__ __forceinline__ int of(int i) const { return (int)(((float)i + 0.5f) * inverse); }
};

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __global__ void __launch_bounds__(THREADS) cache_write_kernel(const CacheRows P)
{
    __shared__ uint32_t tile[CACHE_MOST_WIDTH * PITCH / 4];
    __shared__ uint32_t parts[WARPS];
    __shared__ float old_scale;
    cache_is_there();
    const Cache &c = P.c;
    Part part;
    if (!part.find(c, P.s) || part.page < 0) return; // (the same for all threads)
    const int head = blockIdx.y, which = blockIdx.z, width = (int)c.width, padded = (int)c.padded;
    const HeadRows &in = P.x[which];
    const T *x = static_cast<const T *>(in.x) + (size_t)part.row * in.ld + (size_t)head * in.head_ld;
    const int a = part.a, b = part.b, count = b - a;
    if (threadIdx.x == 0) old_scale = a == 0 ? 0.0f : *scale_of(c, part.page, head, which); // (a page that begins anew)
    // eight or four values at a time where rows begin at multiples of 16 bytes; the second time three of four come from L1, the others from L2
    constexpr int N = Piece<T>::N;
    const bool aligned = width % N == 0 && in.ld % N == 0 && in.head_ld % N == 0 && (reinterpret_cast<uintptr_t>(in.x) & 15) == 0;
    const Rows rows(aligned ? width / N : width);
    uint32_t most = 0;
    if (aligned) {
#pragma unroll 4
        for (int i = threadIdx.x; i < count * rows.length; i += THREADS) {
            const int t = rows.of(i);
            Piece<T> piece;
            piece.w = *reinterpret_cast<const uint4 *>(x + t * in.ld + (i - t * rows.length) * N);
#pragma unroll
            for (int j = 0; j < N; ++j) most = max(most, __float_as_uint(piece.at(j)) & 0x7FFFFFFFu);
        }
    } else {
        for (int i = threadIdx.x; i < count * width; i += THREADS) {
            const int t = rows.of(i);
            most = max(most, __float_as_uint(to_float(x[t * in.ld + (i - t * width)])) & 0x7FFFFFFFu);
        }
    }
    most = __reduce_max_sync(~0u, most);
    if (threadIdx.x % 32 == 0) parts[threadIdx.x / 32] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) most = max(most, parts[w]);
    const float old = old_scale, mine = RowOf<float, 1, 1, false>::scale_of(most);
    const float scale = old != old || mine != mine ? __int_as_float(0x7FC00000) : fmaxf(old, mine);
    const bool none = !(scale > 0.0f), grown = a > 0 && scale > old;
    const Inverse inverse(none ? 1.0f : scale);
    if (threadIdx.x == 0) *scale_of(c, part.page, head, which) = scale;
    uint32_t *codes = reinterpret_cast<uint32_t *>(codes_of(c, part.page, head, which));
    const int words = padded / 4;
    if (which == 0 && grown)
        for (int i = threadIdx.x; i < a * words; i += THREADS) codes[i] = codes_again(codes[i], old, scale);
    // keys to their places, values (turned) to shared memory
    uint8_t *bytes = reinterpret_cast<uint8_t *>(tile);
    if (aligned) {
#pragma unroll 4
        for (int i = threadIdx.x; i < count * rows.length; i += THREADS) {
            const int t = rows.of(i), d = (i - t * rows.length) * N;
            Piece<T> piece;
            piece.w = *reinterpret_cast<const uint4 *>(x + t * in.ld + d);
            Packed<N> four = {};
            if (!none) {
                float v[N];
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = piece.at(j);
                four = pack_codes<N>(v, inverse);
            }
            if (which == 0) {
                uint32_t *to = codes + key_at(padded, a + t, d) / 4;
                if (N == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(four.w[0] ^ ZEROS, four.w[N / 4 - 1] ^ ZEROS);
                else *to = four.w[0] ^ ZEROS;
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) bytes[(d + j) * PITCH + a + t] = (uint8_t)((four.w[j / 4] ^ ZEROS) >> (8 * (j % 4)));
            }
        }
    } else {
        const Rows fours((width + 3) / 4);
        for (int i = threadIdx.x; i < count * fours.length; i += THREADS) {
            const int t = fours.of(i), d = 4 * (i - t * fours.length);
            uint32_t w = ZEROS;
            if (!none) {
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = d + j < width ? to_float(x[t * in.ld + d + j]) : 0.0f;
                w = pack_codes<4>(v, inverse).w[0] ^ ZEROS;
            }
            if (which == 0) {
                codes[key_at(padded, a + t, d) / 4] = w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) bytes[(d + j) * PITCH + a + t] = (uint8_t)(w >> (8 * j));
            }
        }
    }
    if (which == 0) return;
    __syncthreads();
    if (count == CACHE_PAGE) {
        for (int i = threadIdx.x; i < 4 * width; i += THREADS) {
            const uint32_t *from = tile + i / 4 * (PITCH / 4) + i % 4 * 4;
            reinterpret_cast<uint4 *>(codes)[i] = make_uint4(from[0], from[1], from[2], from[3]);
        }
        return;
    }
    const int first = grown ? 0 : a / 4; // words of a dimension
    const Rows dims((b + 3) / 4 - first);
    for (int i = threadIdx.x; i < dims.length * width; i += THREADS) {
        const int d = dims.of(i), at = first + i - d * dims.length, t = 4 * at;
        uint32_t *to = codes + d * (CACHE_PAGE / 4) + at, w = tile[d * (PITCH / 4) + at];
        if (t < a || t + 4 > b) { // bytes of tokens a .. b - 1 among others
            uint32_t others = *to;
            if (t < a && grown) others = codes_again(others, old, scale); // (what is behind b is nobody's)
            uint32_t mask = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) mask |= t + j >= a && t + j < b ? 255u << (8 * j) : 0u;
            w = (w & mask) | (others & ~mask);
        }
        *to = w;
    }
}

template <typename T> __global__ void __launch_bounds__(THREADS) cache_read_kernel(const CacheRows P, unsigned blocks)
{
    __shared__ uint32_t tile[CACHE_MOST_WIDTH * PITCH / 4];
    cache_is_there();
    const Cache &c = P.c;
    const int head = blockIdx.y, which = blockIdx.z, width = (int)c.width;
    const HeadRows &out = P.x[which];
    T *y = static_cast<T *>(out.x) + (size_t)head * out.head_ld;
    if (blockIdx.x >= blocks) { // rows of no sequence
        const int before = offset_of(P.s, 0), behind = max(offset_of(P.s, P.s.sequences), before), rest = before + P.s.n - behind;
        for (size_t i = threadIdx.x; i < (size_t)rest * width; i += THREADS) {
            const size_t r = i / width;
            y[(r < (size_t)before ? r : r - before + behind) * out.ld + i % width] = from_float<T>(0.0f);
        }
        return;
    }
    Part part;
    if (!part.find(c, P.s)) return;
    const int a = part.a, count = part.b - a;
    y += (size_t)part.row * out.ld;
    if (part.page < 0) {
        for (int i = threadIdx.x; i < count * width; i += THREADS) y[(i / width) * out.ld + i % width] = from_float<T>(0.0f);
        return;
    }
    const uint32_t *codes = reinterpret_cast<const uint32_t *>(codes_of(c, part.page, head, which));
    const float scale = *scale_of(c, part.page, head, which);
    const uint8_t *bytes = reinterpret_cast<const uint8_t *>(tile);
    if (which) {
#pragma unroll 4
        for (int i = threadIdx.x; i < 4 * width; i += THREADS) {
            const uint4 w = reinterpret_cast<const uint4 *>(codes)[i];
            uint32_t *to = tile + i / 4 * (PITCH / 4) + i % 4 * 4;
            to[0] = w.x, to[1] = w.y, to[2] = w.z, to[3] = w.w;
        }
        __syncthreads();
    }
    // eight values at a time where rows begin at multiples of 16 bytes
    const bool aligned = width % 8 == 0 && out.ld % 8 == 0 && out.head_ld % 8 == 0 && (reinterpret_cast<uintptr_t>(out.x) & 15) == 0;
    const Rows rows(aligned ? width / 8 : (width + 3) / 4);
    if (aligned) {
#pragma unroll 2
        for (int i = threadIdx.x; i < count * rows.length; i += THREADS) {
            const int t = rows.of(i), d = 8 * (i - t * rows.length);
            uint2 w = make_uint2(0, 0);
            if (!which) w = *reinterpret_cast<const uint2 *>(codes + key_at((int)c.padded, a + t, d) / 4);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (float)((which ? (int)bytes[(d + j) * PITCH + a + t] : (int)((&w.x)[j / 4] >> (8 * (j % 4)) & 255u)) - 128) * scale;
            T *to = y + t * out.ld + d;
            if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4 *>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                uint4 o;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    T two[2] = {from_float<T>(v[2 * j]), from_float<T>(v[2 * j + 1])};
                    (&o.x)[j] = *reinterpret_cast<const uint32_t *>(two);
                }
                *reinterpret_cast<uint4 *>(to) = o;
            }
        }
        return;
    }
    for (int i = threadIdx.x; i < count * rows.length; i += THREADS) {
        const int t = rows.of(i), d = 4 * (i - t * rows.length);
        const uint32_t w = which ? 0 : codes[key_at((int)c.padded, a + t, d) / 4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int q = (which ? (int)bytes[(d + j) * PITCH + a + t] : (int)(w >> (8 * j) & 255u)) - 128;
            if (d + j < width) y[t * out.ld + d + j] = from_float<T>((float)q * scale);
        }
    }
}

// A page and head between its natural order (64 x width) and the cache's.
template <bool IN> __global__ void __launch_bounds__(THREADS) cache_pages_kernel(const Cache c, int which, int8_t *natural, float *scales)
{
    cache_is_there();
    const size_t at = blockIdx.x;
    const int page = (int)(at / c.heads), head = (int)(at % c.heads), width = (int)c.width, padded = (int)c.padded;
    if (threadIdx.x == 0 && scales) {
        float *scale = scale_of(c, page, head, which);
        if (!IN) scales[at] = *scale;
        else *scale = scales[at] >= 0.0f && scales[at] < INFINITY ? scales[at] : __int_as_float(0x7FC00000);
    }
    if (!natural) return;
    natural += at * CACHE_PAGE * width;
    uint8_t *codes = codes_of(c, page, head, which);
    for (int i = threadIdx.x; i < CACHE_PAGE * padded; i += THREADS) {
        const int t = which ? i % CACHE_PAGE : i / padded, d = which ? i / CACHE_PAGE : i % padded;
        uint8_t *code = codes + (which ? i : key_at(padded, t, d));
        if (IN) *code = (uint8_t)((d < width ? natural[t * width + d] : 0) ^ Cache::ZERO);
        else if (d < width) natural[t * width + d] = (int8_t)(*code ^ Cache::ZERO);
    }
}

template <typename T> void write_typed(CudaDevice &dev, const CacheRows &P)
{
    launch_following(cache_write_kernel<T>, dim3(parts_of(P.s), (unsigned)P.c.heads, 2), dim3(THREADS), 0, dev.stream(), P);
}
template <typename T> void read_typed(CudaDevice &dev, const CacheRows &P)
{
    const unsigned blocks = parts_of(P.s);
    launch_following(cache_read_kernel<T>, dim3(blocks + (P.s.offsets ? 1 : 0), (unsigned)P.c.heads, 2), dim3(THREADS), 0, dev.stream(), P, blocks);
}

} // namespace

void launch_cache_write(CudaDevice &dev, const Cache &c, const Sequences &s, const HeadRows &keys, const HeadRows &values)
{
    const CacheRows P{c, s, {keys, values}};
    KernelScope ks(dev, "cache_write");
    if (keys.type == VALUE_F32) write_typed<float>(dev, P);
    else if (keys.type == VALUE_F16) write_typed<__half>(dev, P);
    else write_typed<__nv_bfloat16>(dev, P);
    dev.count_launch();
}

void launch_cache_read(CudaDevice &dev, const Cache &c, const Sequences &s, const HeadRows &keys, const HeadRows &values)
{
    const CacheRows P{c, s, {keys, values}};
    KernelScope ks(dev, "cache_read");
    if (keys.type == VALUE_F32) read_typed<float>(dev, P);
    else if (keys.type == VALUE_F16) read_typed<__half>(dev, P);
    else read_typed<__nv_bfloat16>(dev, P);
    dev.count_launch();
}

void launch_cache_pages_in(CudaDevice &dev, const Cache &c, int which, const int8_t *natural, const float *scales)
{
    KernelScope ks(dev, "cache_pages_in");
    launch_following(cache_pages_kernel<true>, dim3((unsigned)(c.pages * c.heads)), dim3(THREADS), 0, dev.stream(), c, which, const_cast<int8_t *>(natural), const_cast<float *>(scales));
    dev.count_launch();
}

void launch_cache_pages_out(CudaDevice &dev, const Cache &c, int which, int8_t *natural, float *scales)
{
    KernelScope ks(dev, "cache_pages_out");
    launch_following(cache_pages_kernel<false>, dim3((unsigned)(c.pages * c.heads)), dim3(THREADS), 0, dev.stream(), c, which, natural, scales);
    dev.count_launch();
}

} // namespace vqb
