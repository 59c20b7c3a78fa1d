// cache.cu -- tokens into the pages of a cache of 8-bit codes, and back.
//
//   scale s of a page and head = max(s_old, max |x| / 127, 2^-126), code = x / s to the nearest whole number, codes that stay: code s_old / s to the nearest
//
// One block for each page that the call touches, head, and of keys and values: nobody else writes there, and the largest magnitude of all its new tokens is
// known before the first code.  What bounds it is memory: s + 1 bytes a value.
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
    uint32_t most = 0;
    for (int i = threadIdx.x; i < count * width; i += THREADS) {
        const int t = i / width;
        most = max(most, __float_as_uint(to_float(x[t * in.ld + (i - t * width)])) & 0x7FFFFFFFu);
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
    if (which == 0) { // a token's key: words of four dimensions
        for (int i = threadIdx.x; i < (grown ? b : count) * words; i += THREADS) {
            const int k = i / words, d = 4 * (i - k * words), t = (grown ? 0 : a) + k;
            uint32_t w = ZEROS, *to = codes + key_at(padded, t, d) / 4;
            if (t < a) {
                w = codes_again(*to, old, scale);
            } else if (!none) {
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = d + j < width ? to_float(x[(t - a) * in.ld + d + j]) : 0.0f;
                w = pack_codes<4>(v, inverse).w[0] ^ ZEROS;
            }
            *to = w;
        }
        return;
    }
    // values: turned in shared memory, a dimension's words of four tokens
    for (int i = threadIdx.x; i < count * words; i += THREADS) {
        const int k = i / words, d = 4 * (i - k * words);
        uint32_t w = ZEROS;
        if (!none) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = d + j < width ? to_float(x[k * in.ld + d + j]) : 0.0f;
            w = pack_codes<4>(v, inverse).w[0] ^ ZEROS;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) reinterpret_cast<uint8_t *>(tile)[(d + j) * PITCH + a + k] = (uint8_t)(w >> (8 * j));
    }
    __syncthreads();
    const int first = grown ? 0 : a / 4, many = (b + 3) / 4 - first; // words of a dimension
    for (int i = threadIdx.x; i < many * padded; i += THREADS) {
        const int d = i / many, at = first + i - d * many, t = 4 * at;
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
    const int head = blockIdx.y, which = blockIdx.z, width = (int)c.width, words = (int)c.padded / 4;
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
    if (which) {
        for (int i = threadIdx.x; i < (int)c.padded * (CACHE_PAGE / 4); i += THREADS) tile[i / (CACHE_PAGE / 4) * (PITCH / 4) + i % (CACHE_PAGE / 4)] = codes[i];
        __syncthreads();
    }
    for (int i = threadIdx.x; i < count * words; i += THREADS) {
        const int k = i / words, d = 4 * (i - k * words);
        const uint32_t w = which ? 0 : codes[key_at((int)c.padded, a + k, d) / 4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int q = (which ? reinterpret_cast<const uint8_t *>(tile)[(d + j) * PITCH + a + k] : (int)(w >> (8 * j) & 255u)) - 128;
            if (d + j < width) y[k * out.ld + d + j] = from_float<T>((float)q * scale);
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
