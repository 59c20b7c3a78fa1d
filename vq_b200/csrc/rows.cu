// rows.cu -- rows of floats to 8-bit codes with a scale for each row, and the layouts of codes that the products read.
//
// One pass over the data: the threads of a row keep it in registers, agree on its largest magnitude, and write the codes.  What bounds
// it is memory: s + 1 bytes a value.
#include <algorithm>

#include "cuda_device.hpp"
#include "rows.cuh"
#include "umma.cuh"

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

// LANES threads a row, HELD pieces a thread in registers; what is behind them is read a second time.
template <typename T, int DIGITS, int LANES, int HELD, bool ALIGNED>
__global__ void __launch_bounds__(THREADS_OF<LANES>) quantize_rows_kernel(const RowParams P)
{
    constexpr int N = Piece<T>::N, THREADS = THREADS_OF<LANES>, WARPS = LANES / 32;
    __shared__ uint32_t parts[WARPS > 1 ? WARPS : 1];
    rows_are_there();
    product_may_start();
    const size_t r = (size_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES;
    if (r >= P.n) return; // (whole warps; where a block barrier follows, a block is one row)
    const T *row = static_cast<const T *>(P.x) + r * P.ld;
    const float *columns = DIGITS == 2 ? columns_of(P, r) : nullptr;
    if (DIGITS == 2 && !columns) return;
    const size_t pieces = (P.width + (size_t)LANES * N - 1) / ((size_t)LANES * N);
    RowOf<T, DIGITS, LANES, ALIGNED> it(P, r, lane, columns);
    Piece<T> held[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) held[h] = load_values<T, LANES, ALIGNED>(row, h, lane, P.width);
#pragma unroll
    for (int h = 0; h < HELD; ++h) it.look(held[h], h);
    for (size_t h = HELD; h < pieces; ++h) it.look(load_values<T, LANES, ALIGNED>(row, h, lane, P.width), h);
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
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (column<N, LANES, ALIGNED>(h, lane, 0) < P.width) it.write(held[h], h, none, inverse);
    for (size_t h = HELD; h < pieces; ++h) it.write(load_values<T, LANES, ALIGNED>(row, h, lane, P.width), h, none, inverse);
}

// Many aligned rows: a block stays on its SM and has `ring` rows in shared memory, on their way (bulk copies) or worked on; a team of warps takes every
// `teams`th of them and reads it twice from there.
constexpr int STREAM_WARPS = 24;
constexpr size_t STREAM_BYTES = 192 << 10;
constexpr int STREAM_ROWS = STREAM_WARPS; // in the ring, at most

template <typename T, int DIGITS> __global__ void __launch_bounds__(32 * STREAM_WARPS) stream_rows_kernel(const RowParams P, int teams, int slots, int *error)
{
    constexpr int N = Piece<T>::N;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ unsigned long long full[STREAM_ROWS];
    __shared__ uint32_t parts[2][STREAM_WARPS];
    __shared__ int abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, size = STREAM_WARPS / teams, team = warp / size, threads = 32 * size, t = threadIdx.x - team * threads;
    const uint32_t bytes = (uint32_t)(P.width * sizeof(T));
    if (threadIdx.x == 0) {
        for (int i = 0; i < teams * slots; ++i) mbar_init(&full[i], 1);
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    rows_are_there();
    product_may_start();
    auto together = [&] { // the team's warps
        if (size == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(threads) : "memory");
    };
    const size_t first = (size_t)blockIdx.x * teams + team, step = (size_t)gridDim.x * teams;
    unsigned char *mine = ring + (size_t)team * slots * bytes;
    unsigned long long *bars = full + team * slots;
    auto fetch = [&](size_t r, int slot) {
        mbar_expect_tx(&bars[slot], bytes);
        bulk_load_1d(mine + (size_t)slot * bytes, static_cast<const T *>(P.x) + r * P.ld, bytes, &bars[slot]);
    };
    if (t == 0)
        for (int i = 0; i < slots && first + i * step < P.n; ++i) fetch(first + i * step, i);
    const int last = (int)(bytes / 16); // 16-byte pieces of the row
    int slot = 0, turn = 0;
    uint32_t parity = 0;
    for (size_t r = first; r < P.n; r += step, turn ^= 1) {
        // A wait that is given up ends the row, not the loop: the team's other warps count on this one at their barriers, and every later wait ends at
        // once.
        const bool there = __all_sync(~0u, *(volatile int *)&abort_word == 0 && mbar_wait(&bars[slot], parity, &abort_word, error, 71));
        const float *columns = DIGITS == 2 ? columns_of(P, r) : nullptr;
        if (DIGITS == 1 || columns) { // (the same for the whole team)
            RowOf<T, DIGITS, 1, true> it(P, r, 0, columns); // (piece i: 16 bytes at 16 i)
            const uint4 *row = reinterpret_cast<const uint4 *>(mine + (size_t)slot * bytes);
#pragma unroll 4
            for (int i = t; i < last; i += threads) it.look(Piece<T>{row[i]}, i);
            uint32_t most = it.largest();
            if (size > 1) {
                if (lane == 0) parts[turn][warp] = most;
                together();
                for (int w = 0; w < size; ++w) most = max(most, parts[turn][team * size + w]);
            }
            const float scale = it.scale_of(most);
            if (t == 0 && there) P.scales[r] = scale;
            int8_t *codes = P.codes + r * P.ld_codes, *lows = DIGITS == 2 ? P.low + r * P.ld_codes : nullptr;
            auto put = [&](int8_t *to, int i, const Packed<N> &c) {
                if (N == 8) reinterpret_cast<uint2 *>(to)[i] = make_uint2(c.w[0], c.w[N / 4 - 1]);
                else reinterpret_cast<uint32_t *>(to)[i] = c.w[0];
            };
            if (it.no_codes(most)) {
                for (int i = t; i < last; i += threads) {
                    put(codes, i, Packed<N>{});
                    if (DIGITS == 2) put(lows, i, Packed<N>{});
                }
            } else {
                const Inverse inverse(scale);
#pragma unroll 4
                for (int i = t; i < last; i += threads) {
                    Packed<N> high, low;
                    it.pack(Piece<T>{row[i]}, i, inverse, high, low);
                    put(codes, i, high);
                    if (DIGITS == 2) put(lows, i, low);
                }
            }
        }
        together();
        if (t == 0 && r + slots * step < P.n && there) fetch(r + slots * step, slot);
        if (++slot == slots) slot = 0, parity ^= 1u;
    }
    if (*(volatile int *)&abort_word) // what has been asked for lands before the block leaves
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

template <typename T, int DIGITS, int LANES, int HELD> void quantize_rows_with(CudaDevice &dev, const RowParams &P, bool aligned)
{
    constexpr int THREADS = THREADS_OF<LANES>, ROWS = THREADS / LANES;
    const dim3 grid((unsigned)((P.n + ROWS - 1) / ROWS));
    if (aligned) launch_following(quantize_rows_kernel<T, DIGITS, LANES, HELD, true>, grid, dim3(THREADS), 0, dev.stream(), P);
    else launch_following(quantize_rows_kernel<T, DIGITS, LANES, HELD, false>, grid, dim3(THREADS), 0, dev.stream(), P);
}

// As many threads a row as have two pieces of it each; many wide rows are streamed.
template <typename T, int DIGITS> void quantize_rows_typed(CudaDevice &dev, const RowParams &P)
{
    const size_t apart = P.n == 1 ? 0 : P.ld * sizeof(T), codes_apart = P.n == 1 ? 0 : P.ld_codes; // (one row has no next one)
    const bool aligned = (reinterpret_cast<uintptr_t>(P.x) | apart) % 16 == 0 && (reinterpret_cast<uintptr_t>(P.codes) | codes_apart | reinterpret_cast<uintptr_t>(P.low)) % 8 == 0;
    const size_t pieces = (P.width + Piece<T>::N - 1) / Piece<T>::N, bytes = P.width * sizeof(T);
    // Measured (us, streamed and not): 16384 x 4096 bf16 34 and 41, 8192 x 8192 44 and 52; but 8192 x 4096 26 and 25, 16384 x 2048 25 and 23.
    if (aligned && bytes % 16 == 0 && bytes >= 8192 && bytes <= STREAM_BYTES / 4 && dev.error_word()) {
        size_t teams = STREAM_WARPS; // two rows for each in the ring
        while (2 * teams * bytes > STREAM_BYTES) teams /= 2;
        if (P.n >= 8 * teams * (size_t)dev.sm_count()) {
            const size_t slots = std::min<size_t>(STREAM_BYTES / (teams * bytes), STREAM_ROWS / teams);
            allow_shared_memory(dev, stream_rows_kernel<T, DIGITS>);
            launch_following(stream_rows_kernel<T, DIGITS>, dim3((unsigned)dev.sm_count()), dim3(32 * STREAM_WARPS), slots * bytes * teams, dev.stream(), P, (int)teams, (int)slots, dev.error_word());
            return;
        }
    }
    if (pieces <= 64) quantize_rows_with<T, DIGITS, 32, 2>(dev, P, aligned);
    else if (pieces <= 128) quantize_rows_with<T, DIGITS, 64, 2>(dev, P, aligned);
    else if (pieces <= 256) quantize_rows_with<T, DIGITS, 128, 2>(dev, P, aligned);
    else if (pieces <= 512) quantize_rows_with<T, DIGITS, 256, 2>(dev, P, aligned);
    else if (pieces <= 1024) quantize_rows_with<T, DIGITS, 512, 2>(dev, P, aligned);
    else quantize_rows_with<T, DIGITS, 512, 4>(dev, P, aligned);
}

template <int DIGITS> void quantize_rows_any(CudaDevice &dev, const char *name, const RowParams &P, int type)
{
    if (P.n == 0) return;
    KernelScope ks(dev, name);
    if (type == VALUE_F16) quantize_rows_typed<__half, DIGITS>(dev, P);
    else if (type == VALUE_BF16) quantize_rows_typed<__nv_bfloat16, DIGITS>(dev, P);
    else if (DIGITS == 1) quantize_rows_typed<float, 1>(dev, P); // (two digits are 16-bit rows')
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
