// rows.cu -- rows of floats to 8-bit codes with a scale for each row, and the layouts of codes that the products read.
//
// One pass over the data: the lanes of a row keep it in registers, agree on its largest magnitude, and write the codes.  What bounds
// it is memory: s + 1 bytes a value.
//
// The code is the nearest whole number to the REAL quotient x / s (halves to even), so that it depends on nothing but x and the
// row's largest magnitude.  x (1 / s) in f32 is off by less than 128 2^-23 = 2^-16; only where its distance from a half is below that
// does the quotient in f64 decide (two f32 numbers' quotient is either a half or further from it than f64 rounds by).
#include <algorithm>

#include "cuda_device.hpp"
#include "qmat.cuh"

namespace vqb {

namespace {

constexpr float MAGIC = 12582912.0f; // 1.5 2^23: adding it rounds to a whole number, whose two's complement is then in the low bits
constexpr float LARGEST_8 = 127.0f, LARGEST_15 = 16256.0f; // 16256 = 127 * 128: the high digit stays within 127

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

// N values of a row from column k on, 0 behind its end
template <typename T, bool ALIGNED> __device__ __forceinline__ Piece<T> load_values(const T *row, size_t k, size_t width)
{
    constexpr int N = Piece<T>::N;
    Piece<T> p;
    p.w = make_uint4(0, 0, 0, 0);
    if (ALIGNED && k + N <= width) {
        p.w = *reinterpret_cast<const uint4 *>(row + k);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (k + i < width) {
                if (sizeof(T) == 4) (&p.w.x)[i] = reinterpret_cast<const uint32_t *>(row)[k + i];
                else (&p.w.x)[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t *>(row)[k + i] << (16 * (i & 1));
            }
    }
    return p;
}

// whole numbers of magnitudes up to 127 as bytes; `far`: no quotient was near a half
template <int N> struct Packed {
    uint32_t w[N / 4];
};
template <int N> __device__ __forceinline__ Packed<N> pack_codes(const float (&v)[N], float scale, float inverse)
{
    uint32_t m[N];
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = __fmaf_rn(v[i], inverse, MAGIC);
        m[i] = __float_as_uint(t);
        off = fmaxf(off, fabsf(__fmaf_rn(v[i], inverse, __fsub_rn(MAGIC, t))));
    }
    if (off > 0.5f - 0x1p-15f) { // some quotient may be nearer to the other neighbour
#pragma unroll 1
        for (int i = 0; i < N; ++i) m[i] = (uint32_t)__double2int_rn((double)v[i] / (double)scale);
    }
    Packed<N> out;
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
        out.w[i] = __byte_perm(__byte_perm(m[4 * i], m[4 * i + 1], 0x0040), __byte_perm(m[4 * i + 2], m[4 * i + 3], 0x0040), 0x5410);
    return out;
}

// The two digits of u / t, |u / t| <= 16256: the high one is the whole number nearest to a 128th of it.
template <int N> __device__ __forceinline__ void pack_digits(const float (&u)[N], float inverse, Packed<N> &high, Packed<N> &low)
{
    uint32_t h[N], l[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int v = (int)__float_as_uint(__fmaf_rn(u[i], inverse, MAGIC)) - (int)__float_as_uint(MAGIC);
        const int top = (v + 64) >> 7; // -127 .. 127
        h[i] = (uint32_t)top, l[i] = (uint32_t)(v - (top << 7)); // -64 .. 63
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        high.w[i] = __byte_perm(__byte_perm(h[4 * i], h[4 * i + 1], 0x0040), __byte_perm(h[4 * i + 2], h[4 * i + 3], 0x0040), 0x5410);
        low.w[i] = __byte_perm(__byte_perm(l[4 * i], l[4 * i + 1], 0x0040), __byte_perm(l[4 * i + 2], l[4 * i + 3], 0x0040), 0x5410);
    }
}

template <int N, bool ALIGNED> __device__ __forceinline__ void store_codes(int8_t *row, size_t k, size_t width, const Packed<N> &c)
{
    if (ALIGNED && k + N <= width) {
        if (N == 8) *reinterpret_cast<uint2 *>(row + k) = make_uint2(c.w[0], c.w[N / 4 - 1]);
        else *reinterpret_cast<uint32_t *>(row + k) = c.w[0];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (k + i < width) row[k + i] = (int8_t)(c.w[i >> 2] >> (8 * (i & 3)));
    }
}

struct RowParams {
    const void *x;
    size_t n, width, ld;
    int8_t *codes, *low; // low: the low digits' plane (two digits)
    size_t ld_codes;
    float *scales;
    const float *column_scales; // groups x width (two digits)
    const long long *offsets;
    int groups;
};

// Row r's column scales; null: the row belongs to no group.
__device__ __forceinline__ const float *columns_of(const RowParams &P, size_t r)
{
    if (!P.offsets) return P.column_scales;
    const long long row = (long long)r;
    if (row < P.offsets[0] || row >= P.offsets[P.groups]) return nullptr;
    int lo = 0, hi = P.groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (P.offsets[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return P.column_scales + (size_t)lo * P.width;
}

// LANES threads a row, HELD pieces a thread in registers; what is behind them is read a second time.
template <typename T, int DIGITS, int LANES, int HELD, bool ALIGNED_X, bool ALIGNED_CODES>
__global__ void __launch_bounds__(LANES < 128 ? 128 : LANES) quantize_rows_kernel(const RowParams P)
{
    constexpr int N = Piece<T>::N, THREADS = LANES < 128 ? 128 : LANES, WARPS = LANES / 32;
    __shared__ uint32_t parts[WARPS > 1 ? WARPS : 1];
    rows_are_there();
    product_may_start();
    const size_t r = (size_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    if (r >= P.n) return; // (whole warps; where a block barrier follows, a block is one row)
    const T *row = static_cast<const T *>(P.x) + r * P.ld;
    const float *columns = DIGITS == 2 ? columns_of(P, r) : nullptr;
    if (DIGITS == 2 && !columns) return;

    auto values = [&](const Piece<T> &p, size_t k, float(&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = p.at(i);
            if (DIGITS == 2) v[i] = k + i < P.width ? v[i] * columns[k + i] : 0.0f;
        }
    };
    // magnitudes as whole numbers: their order is that of the bits, infinities and NaN on top
    uint32_t most = 0;
    auto look = [&](const Piece<T> &p, size_t k) {
        float v[N];
        values(p, k, v);
#pragma unroll
        for (int i = 0; i < N; ++i) most = max(most, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    };
    Piece<T> held[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) held[h] = load_values<T, ALIGNED_X>(row, (size_t)(h * LANES + lane) * N, P.width);
#pragma unroll
    for (int h = 0; h < HELD; ++h) look(held[h], (size_t)(h * LANES + lane) * N);
    for (size_t k = (size_t)(HELD * LANES + lane) * N; k < P.width; k += (size_t)LANES * N) look(load_values<T, ALIGNED_X>(row, k, P.width), k);
    most = __reduce_max_sync(~0u, most);
    if (WARPS > 1) {
        if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; ++w) most = max(most, parts[w]);
    }
    const bool finite = most < 0x7F800000u;
    const float a = __uint_as_float(most);
    const float scale = !finite ? __int_as_float(0x7FC00000) : most == 0 ? 0.0f : fmaxf(__fdiv_rn(a, DIGITS == 1 ? LARGEST_8 : LARGEST_15), 0x1p-126f);
    if (lane == 0) P.scales[r] = scale;
    const bool none = !finite || most == 0; // all codes 0
    const float inverse = none ? 0.0f : __frcp_rn(scale);
    int8_t *codes = P.codes + r * P.ld_codes;
    auto write = [&](const Piece<T> &p, size_t k) {
        float v[N];
        values(p, k, v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = none ? 0.0f : v[i];
        if (DIGITS == 1) {
            store_codes<N, ALIGNED_CODES>(codes, k, P.width, pack_codes<N>(v, none ? 1.0f : scale, inverse));
        } else {
            Packed<N> high, low;
            pack_digits<N>(v, inverse, high, low);
            store_codes<N, ALIGNED_CODES>(codes, k, P.width, high);
            store_codes<N, ALIGNED_CODES>(P.low + r * P.ld_codes, k, P.width, low);
        }
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const size_t k = (size_t)(h * LANES + lane) * N;
        if (k < P.width) write(held[h], k);
    }
    for (size_t k = (size_t)(HELD * LANES + lane) * N; k < P.width; k += (size_t)LANES * N) write(load_values<T, ALIGNED_X>(row, k, P.width), k);
}

template <typename T, int DIGITS, int LANES, int HELD> void quantize_rows_with(CudaDevice &dev, const RowParams &P, bool aligned_x, bool aligned_codes)
{
    constexpr int THREADS = LANES < 128 ? 128 : LANES, ROWS = THREADS / LANES;
    const dim3 grid((unsigned)((P.n + ROWS - 1) / ROWS));
    if (aligned_x && aligned_codes) launch_following(quantize_rows_kernel<T, DIGITS, LANES, HELD, true, true>, grid, dim3(THREADS), 0, dev.stream(), P);
    else if (aligned_codes) launch_following(quantize_rows_kernel<T, DIGITS, LANES, HELD, false, true>, grid, dim3(THREADS), 0, dev.stream(), P);
    else launch_following(quantize_rows_kernel<T, DIGITS, LANES, HELD, false, false>, grid, dim3(THREADS), 0, dev.stream(), P);
}

template <typename T, int DIGITS> void quantize_rows_typed(CudaDevice &dev, const RowParams &P)
{
    const bool aligned_x = (reinterpret_cast<uintptr_t>(P.x) | (P.ld * sizeof(T))) % 16 == 0;
    const bool aligned_codes = (reinterpret_cast<uintptr_t>(P.codes) | P.ld_codes | reinterpret_cast<uintptr_t>(P.low)) % 8 == 0;
    const size_t pieces = (P.width + Piece<T>::N - 1) / Piece<T>::N;
    if (pieces <= 32 * 4) quantize_rows_with<T, DIGITS, 32, 4>(dev, P, aligned_x, aligned_codes);
    else quantize_rows_with<T, DIGITS, 256, 4>(dev, P, aligned_x, aligned_codes);
}

template <int DIGITS> void quantize_rows_any(CudaDevice &dev, const char *name, const RowParams &P, int type)
{
    if (P.n == 0) return;
    KernelScope ks(dev, name);
    if (type == VALUE_F32) quantize_rows_typed<float, DIGITS>(dev, P);
    else if (type == VALUE_F16) quantize_rows_typed<__half, DIGITS>(dev, P);
    else quantize_rows_typed<__nv_bfloat16, DIGITS>(dev, P);
    dev.count_launch();
}

// Transposes 64 x 64 bytes at a time through shared memory; used once for a matrix.
__global__ void turn_codes_kernel(const int8_t *codes, size_t rows, size_t width, size_t ld, int8_t *turned, size_t turned_ld)
{
    __shared__ int8_t tile[64][65];
    const size_t g = blockIdx.z;
    codes += g * rows * ld, turned += g * width * turned_ld;
    const size_t k0 = (size_t)blockIdx.x * 64;
    for (size_t j0 = (size_t)blockIdx.y * 64; j0 < rows; j0 += (size_t)gridDim.y * 64) {
        for (int i = threadIdx.x; i < 64 * 64; i += blockDim.x) {
            const size_t j = j0 + i / 64, k = k0 + i % 64;
            if (j < rows && k < width) tile[i / 64][i % 64] = codes[j * ld + k];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * 64; i += blockDim.x) {
            const size_t k = k0 + i / 64, j = j0 + i % 64;
            if (j < rows && k < width) turned[k * turned_ld + j] = tile[i % 64][i / 64];
        }
        __syncthreads();
    }
}

__global__ void align_codes_kernel(const int8_t *codes, size_t n, size_t width, size_t ld, int8_t *aligned, size_t aligned_ld)
{
    for (size_t r = blockIdx.x; r < n; r += gridDim.x)
        for (size_t k = threadIdx.x; k < width; k += blockDim.x) aligned[r * aligned_ld + k] = codes[r * ld + k];
}

} // namespace

void launch_quantize_rows(CudaDevice &dev, const void *x, int type, size_t n, size_t width, size_t ld, int8_t *codes, size_t ld_codes, float *scales)
{
    RowParams P{x, n, width, ld, codes, nullptr, ld_codes, scales, nullptr, nullptr, 0};
    quantize_rows_any<1>(dev, "quantize_rows", P, type);
}

void launch_digit_rows(CudaDevice &dev, const void *x, int type, size_t n, size_t width, size_t ld, const float *column_scales, size_t groups, const int64_t *offsets,
                       int8_t *digits, size_t ld_codes, float *scales)
{
    RowParams P{x, n, width, ld, digits, digits + n * ld_codes, ld_codes, scales, column_scales, reinterpret_cast<const long long *>(offsets), (int)groups};
    quantize_rows_any<2>(dev, "digit_rows", P, type);
}

void launch_turn_codes(CudaDevice &dev, const int8_t *codes, size_t groups, size_t rows, size_t width, int8_t *turned)
{
    KernelScope ks(dev, "turn_codes");
    const dim3 grid((unsigned)((width + 63) / 64), (unsigned)std::min<size_t>((rows + 63) / 64, 65535), (unsigned)groups);
    turn_codes_kernel<<<grid, 256, 0, dev.stream()>>>(codes, rows, width, codes_ld(width), turned, codes_ld(rows));
    VQB_CUDA_CHECK(cudaGetLastError());
    dev.count_launch();
}

void launch_align_codes(CudaDevice &dev, const int8_t *codes, size_t n, size_t width, size_t ld, int8_t *aligned)
{
    KernelScope ks(dev, "align_codes");
    align_codes_kernel<<<(unsigned)std::min<size_t>(n, (size_t)dev.sm_count() * 16), 256, 0, dev.stream()>>>(codes, n, width, ld, aligned, codes_ld(width));
    VQB_CUDA_CHECK(cudaGetLastError());
    dev.count_launch();
}

} // namespace vqb
