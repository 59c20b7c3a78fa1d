// rows.cu -- rows of floats to 8-bit codes with a scale for each row, and the layouts of codes that the products read.
//
// One pass over the data: the threads of a row keep it in registers, agree on its largest magnitude, and write the codes.  What bounds
// it is memory: s + 1 bytes a value.
#include <algorithm>

#include "cuda_device.hpp"
#include "rows.cuh"

namespace vqb {

namespace {

// Row r's column scales, by a whole warp; null: the row belongs to no group.
__device__ __forceinline__ const float *columns_of(const RowParams &P, size_t r)
{
    if (!P.offsets) return P.column_scales;
    int begun = 0; // offsets that are not behind the row
    for (int g0 = 0; g0 <= P.groups; g0 += 32) {
        const int g = g0 + (threadIdx.x & 31);
        begun += __popc(__ballot_sync(~0u, g <= P.groups && P.offsets[g] <= (long long)r));
    }
    return begun == 0 || begun > P.groups ? nullptr : P.column_scales + (size_t)(begun - 1) * P.width;
}

// threads of a block: a row's, or four rows' warps
template <int LANES> constexpr int THREADS_OF = LANES < 64 ? 128 : LANES;

// LANES threads a row, HELD pieces a thread in registers; what is behind them is read a second time.  (256 threads: five blocks an SM, 8192 x 8192 bf16 in 39 us; 44 with
// the registers that four leave.  Blocks of 128 take 35 instead of 32 for 16384 x 4096 when they are held to fewer.)
template <typename T, int DIGITS, int LANES, int HELD, bool ALIGNED>
__global__ void __launch_bounds__(THREADS_OF<LANES>, DIGITS == 1 && LANES == 256 ? 5 : 0) quantize_rows_kernel(const RowParams P)
{
    constexpr int N = Piece<T>::N, THREADS = THREADS_OF<LANES>, WARPS = LANES / 32;
    __shared__ uint32_t parts[WARPS > 1 ? WARPS : 1];
    rows_are_there();
    if (P.product_follows) product_may_start();
    const size_t r = (size_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    if (r >= P.n) return; // (whole warps; where a block barrier follows, a block is one row)
    const T *row = static_cast<const T *>(P.x) + r * P.ld;
    const uint32_t pieces = (P.width + LANES * N - 1) / (LANES * N);
    const bool full = ALIGNED && HELD * LANES * N <= P.width; // all of the held pieces are whole
    Piece<T> held[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        if (full) held[h].w = *reinterpret_cast<const uint4 *>(row + column<N, LANES, true>(h, lane, 0));
        else held[h] = load_values<T, LANES, ALIGNED>(row, h, lane, P.width);
    }
    const float *columns = DIGITS == 3 ? columns_of(P, r) : nullptr; // (its loads beside the row's)
    if (DIGITS == 3 && !columns) return;
    RowOf<T, DIGITS, LANES, ALIGNED> it(P, r, lane, columns);
    float u[DIGITS == 3 ? HELD : 1][N]; // three digits: what the columns' scales make of the row is kept instead
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        if (DIGITS == 3) it.values(held[h], h, u[DIGITS == 3 ? h : 0]), it.look(u[DIGITS == 3 ? h : 0]);
        else it.look(held[h], h);
    }
    for (uint32_t h = HELD; h < pieces; ++h) it.look(load_values<T, LANES, ALIGNED>(row, h, lane, P.width), h);
    uint32_t most = it.largest();
    if (WARPS > 1) {
        if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; ++w) most = max(most, parts[w]);
    }
    const float scale = it.scale_of(most);
    const bool none = it.no_codes(most);
    if (lane == 0) P.scales[r] = scale;
    const Inverse inverse(none ? 1.0f : scale);
    Packed<N> packed[HELD][DIGITS] = {};
    if (!none) {
        uint64_t unlike[HELD] = {};
        bool some = false;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            if constexpr (DIGITS == 3) {
                pack_digits<N>(u[h], inverse, packed[h]);
            } else {
                it.values(held[h], h, u[0]);
                packed[h][0] = pack_most<N>(u[0], inverse, unlike[h]);
                some |= any_unlike(unlike[h]);
            }
        }
        if (DIGITS == 1 && some) {
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
                if (!any_unlike(unlike[h])) continue;
                it.values(held[h], h, u[0]);
                packed[h][0] = pack_all<N>(u[0], inverse);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        if (full) it.put(h, packed[h]);
        else if (column<N, LANES, ALIGNED>(h, lane, 0) < P.width) it.store(h, packed[h]);
    }
    for (uint32_t h = HELD; h < pieces; ++h) it.write(load_values<T, LANES, ALIGNED>(row, h, lane, P.width), h, none, inverse);
}

template <typename T, int DIGITS, int LANES, int HELD> void quantize_rows_with(CudaDevice &dev, const RowParams &P, bool aligned)
{
    constexpr int THREADS = THREADS_OF<LANES>, ROWS = THREADS / LANES;
    const dim3 grid((unsigned)((P.n + ROWS - 1) / ROWS));
    if (aligned) launch_following(quantize_rows_kernel<T, DIGITS, LANES, HELD, true>, grid, dim3(THREADS), 0, dev.stream(), P);
    else launch_following(quantize_rows_kernel<T, DIGITS, LANES, HELD, false>, grid, dim3(THREADS), 0, dev.stream(), P);
}

// As many threads a row as have four pieces of it each: bytes under way and not threads are what it takes (us with two and four pieces: 1024 x 1024 bf16 2.6 and
// 2.5, 16384 x 1024 18.0 and 10.6, 4096 x 4096 12.9 and 10.8, 8192 x 4096 24.6 and 19.5); two where a warp has them all.
template <typename T, int DIGITS> void quantize_rows_typed(CudaDevice &dev, const RowParams &P)
{
    const size_t apart = P.n == 1 ? 0 : P.ld * sizeof(T), codes_apart = P.n == 1 ? 0 : P.ld_codes; // (one row has no next one)
    const bool aligned = (reinterpret_cast<uintptr_t>(P.x) | apart) % 16 == 0 && (reinterpret_cast<uintptr_t>(P.codes) | codes_apart | P.plane) % 8 == 0;
    const size_t pieces = (P.width + Piece<T>::N - 1) / Piece<T>::N;
    if (pieces <= 64) quantize_rows_with<T, DIGITS, 32, 2>(dev, P, aligned);
    else if (pieces <= 128) quantize_rows_with<T, DIGITS, 32, 4>(dev, P, aligned);
    else if (pieces <= 256) quantize_rows_with<T, DIGITS, 64, 4>(dev, P, aligned);
    else if (pieces <= 512) quantize_rows_with<T, DIGITS, 128, 4>(dev, P, aligned);
    else if (pieces <= 1024) quantize_rows_with<T, DIGITS, 256, 4>(dev, P, aligned);
    else quantize_rows_with<T, DIGITS, 512, 4>(dev, P, aligned);
}

template <int DIGITS> void quantize_rows_any(CudaDevice &dev, const char *name, const RowParams &P, int type)
{
    if (P.n == 0) return;
    KernelScope ks(dev, name);
    if (type == VALUE_F16) quantize_rows_typed<__half, DIGITS>(dev, P);
    else if (type == VALUE_BF16) quantize_rows_typed<__nv_bfloat16, DIGITS>(dev, P);
    else if (DIGITS == 1) quantize_rows_typed<float, 1>(dev, P); // (three digits are 16-bit rows')
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

void launch_quantize_rows(CudaDevice &dev, const void *x, int type, size_t n, size_t width, size_t ld, int8_t *codes, size_t ld_codes, float *scales,
                          bool product_follows)
{
    RowParams P{x, n, ld, (uint32_t)width, codes, ld_codes, 0, scales, nullptr, nullptr, 0, product_follows};
    quantize_rows_any<1>(dev, "quantize_rows", P, type);
}

void launch_digit_rows(CudaDevice &dev, const void *x, int type, size_t n, size_t width, size_t ld, const float *column_scales, size_t groups, const int64_t *offsets,
                       int8_t *digits, size_t ld_codes, float *scales)
{
    RowParams P{x, n, ld, (uint32_t)width, digits, ld_codes, n * ld_codes, scales, column_scales, reinterpret_cast<const long long *>(offsets), (int)groups, true};
    quantize_rows_any<3>(dev, "digit_rows", P, type);
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
