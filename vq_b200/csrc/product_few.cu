// product_few.cu -- products of up to sixteen rows with one matrix.
//
// Nothing counts here but the matrix's bytes, which are read once, and the time until the first of them arrive.  Every block has a slice of
// the channels.  One warp keeps them coming into a ring in shared memory, 128 bytes of up to 128 channels a stage or 512 of up to 32 (TMA boxes of 128
// bytes, swizzled; a plain bulk copy for each channel's 512 bytes takes 43 ns of an SM's copy unit, four times too long), from the kernel's first moment
// on: a matrix is complete before any product of it is launched, so that there is nothing to wait for.
// Meanwhile the other twenty warps bring the rows' codes into shared memory; one row or two are quantized right there, by every block for
// itself, which takes less than another launch.  Then two warps for each place in the ring take what comes there (mma.sync m16n8k32: 16 channels, 8 rows) and add their
// sums to the block's in shared memory when the channels change; they are whole numbers, so their order does not matter.  (With all warps
// at work on one stage, each had two instructions a stage and 0.3 us of waiting; and dp4a, which did this first, runs at some ten lanes an SM and cycle
// here: 8 rows of 8192 took 46 us.)
//
// The order of the bytes along K is free as long as channels and rows have the same: a lane takes 16 neighbouring bytes and feeds two
// instructions with them.
#include <algorithm>

#include "cuda_device.hpp"
#include "rows.cuh"
#include "tma_host.hpp"
#include "umma.cuh"

namespace vqb {

namespace {

constexpr int MOST_STAGES = 10, WARPS = 2 * MOST_STAGES, THREADS = 32 * (WARPS + 1);
constexpr int BOX_K = 128, MOST_CHANNELS = 128; // bytes and channels of a box
constexpr uint32_t STAGE_BYTES = MOST_CHANNELS * BOX_K;
constexpr size_t SMEM_BYTES = 216 << 10;

struct FewParams {
    RowParams rows;      // x, n, width, ld (values)
    const int8_t *given; // codes instead
    size_t given_ld;
    const float *given_scales;
    int ld, pitch;   // of the matrix; of the rows' codes in shared memory
    int box_channels;
    int channels;
    const float *channel_scales, *bias;
    void *y;
    int y_type;
    size_t y_ld;
    int stages;
    int *error;
};

__device__ __forceinline__ void all_but_one() { asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory"); }

__device__ __forceinline__ void store_value(void *y, size_t at, int type, float v)
{
    if (type == VALUE_F32) static_cast<float *>(y)[at] = v;
    else if (type == VALUE_F16) static_cast<__half *>(y)[at] = from_float<__half>(v);
    else static_cast<__nv_bfloat16 *>(y)[at] = from_float<__nv_bfloat16>(v);
}

// sums += 16 channels x 32 bytes times 32 bytes x 8 rows
__device__ __forceinline__ void mma_i8(int (&sums)[4], int a0, int a1, int a2, int a3, int b0, int b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(sums[0]), "+r"(sums[1]), "+r"(sums[2]), "+r"(sums[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// T: the rows' type, int8_t for codes; EIGHTS: eights of rows; PAIRS: pairs of sixteen channels a box has room for (4 / PAIRS boxes a stage)
template <typename T, int EIGHTS, int PAIRS> __global__ void __launch_bounds__(THREADS, 1) product_few_kernel(const __grid_constant__ CUtensorMap map_codes, const FewParams P)
{
    constexpr int NT = 8 * EIGHTS;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ unsigned long long full[MOST_STAGES], empty[MOST_STAGES];
    __shared__ uint32_t parts[WARPS];
    __shared__ float row_scales[NT];
    __shared__ int abort_word;
    int8_t *ring = reinterpret_cast<int8_t *>(smem), *rows = ring + P.stages * STAGE_BYTES; // NT x pitch
    int *sums = reinterpret_cast<int *>(rows + NT * P.pitch);                                             // NT x the slice's channels
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = (int)((long long)blockIdx.x * P.channels / gridDim.x), count = (int)((long long)(blockIdx.x + 1) * P.channels / gridDim.x) - first;
    const int per_part = P.box_channels, stage_k = 4 / PAIRS * BOX_K, steps = (P.ld + stage_k - 1) / stage_k; // the slice is taken in parts of so many channels
    const uint32_t box_bytes = (uint32_t)((P.box_channels + 7) / 8 * 8 * BOX_K);
    const int all = (count + per_part - 1) / per_part * steps; // stages

    if (warp == WARPS) {
        if (lane < P.stages) {
            mbar_init(&full[lane], 1);
            mbar_init(&empty[lane], 2);
        }
        if (lane == 0) abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        int channel = first, k = 0; // of the next stage
        auto fetch = [&](int st) {
            const int boxes = min(4 / PAIRS, (P.ld - k + BOX_K - 1) / BOX_K);
            mbar_expect_tx(&full[st], (uint32_t)(boxes * per_part * BOX_K));
            for (int b = 0; b < boxes; ++b) tma_load_2d(ring + st * STAGE_BYTES + b * box_bytes, &map_codes, k + b * BOX_K, channel, &full[st]);
            if ((k += stage_k) >= P.ld) k = 0, channel += per_part;
        };
        if (lane == 0)
            for (int i = 0; i < min(all, P.stages); ++i) fetch(i);
        __syncthreads(); // the others may look at the barriers
        rows_are_there();
        if (lane == 0) {
            int st = 0;
            uint32_t parity = 0;
            for (int i = P.stages; i < all; ++i) {
                if (!mbar_wait(&empty[st], parity, &abort_word, P.error, 81)) { // what has been asked for lands before the block leaves
                    for (int w = 0; w < 1000; ++w) __nanosleep(1000);
                    break;
                }
                fetch(st);
                if (++st == P.stages) st = 0, parity ^= 1u;
            }
        }
        return;
    }

    for (int i = threadIdx.x; i < NT * count; i += 32 * WARPS) sums[i] = 0;
    const int n = (int)P.rows.n;
    rows_are_there();
    if constexpr (std::is_same<T, int8_t>::value) {
        const int pieces = P.pitch / 16, width = (int)P.rows.width;
        for (int i = threadIdx.x; i < NT * pieces; i += 32 * WARPS) { // (zeros behind the width)
            const int t = i / pieces, k = 16 * (i - t * pieces);
            const int8_t *from = P.given + t * P.given_ld + k;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (t < n && k + 16 <= width) {
                v = *reinterpret_cast<const uint4 *>(from);
            } else if (t < n && k < width) {
#pragma unroll 1
                for (int b = 0; k + b < width; ++b) {
                    const uint32_t byte = (uint32_t)(uint8_t)from[b] << (8 * (b & 3));
                    if (b < 4) v.x |= byte;
                    else if (b < 8) v.y |= byte;
                    else if (b < 12) v.z |= byte;
                    else v.w |= byte;
                }
            }
            reinterpret_cast<uint4 *>(rows)[i] = v;
        }
        if (threadIdx.x < NT) row_scales[threadIdx.x] = threadIdx.x < n ? P.given_scales[threadIdx.x] : 0.0f;
    } else {
        constexpr int N = Piece<T>::N;
        const int team = WARPS / n, t = min(warp / team, n - 1), l = threadIdx.x - 32 * team * t, step = 32 * team, pieces = P.pitch / N; // (n: 1 or 2)
        const T *row = static_cast<const T *>(P.rows.x) + t * P.rows.ld;
        RowOf<T, 1, 1, true> it(P.rows, t, 0, nullptr); // (piece i: 16 bytes at 16 i)
        const int last = (int)((P.rows.width + N - 1) / N);
        const Piece<T> held = load_values<T, 1, true>(row, l, 0, P.rows.width); // (up to `step` pieces a row, 640 or of two rows 320 each, there are no others)
        it.look(held, l);
#pragma unroll 4
        for (int i = l + step; i < last; i += step) it.look(load_values<T, 1, true>(row, i, 0, P.rows.width), i);
        uint32_t most = it.largest();
        if (lane == 0) parts[warp] = most;
        all_but_one();
        most = __reduce_max_sync(~0u, parts[t * team + lane % team]);
        const float scale = it.scale_of(most);
        const bool none = it.no_codes(most);
        if (l == 0) row_scales[t] = scale;
        const Inverse inverse(none ? 1.0f : scale);
        auto put = [&](int r, int i, const Packed<N> &c) {
            if (N == 8) reinterpret_cast<uint2 *>(rows + r * P.pitch)[i] = make_uint2(c.w[0], c.w[N / 4 - 1]);
            else reinterpret_cast<uint32_t *>(rows + r * P.pitch)[i] = c.w[0];
        };
#pragma unroll 2
        for (int i = l; i < pieces; i += step) { // (zeros behind the width)
            Packed<N> c[1] = {};
            if (!none && i < last) it.pack(i == l ? held : load_values<T, 1, true>(row, i, 0, P.rows.width), i, inverse, c);
            put(t, i, c[0]);
        }
        for (int i = threadIdx.x; i < (NT - n) * pieces; i += 32 * WARPS) put(n + i / pieces, i % pieces, Packed<N>{});
    }
    __syncthreads();

    // This lane's channels are c and c + 8 of every sixteen of its warp's, its bytes 16 of each 64.  Lanes next to each other take channels whose swizzled
    // places are in different halves of the banks.
    const int g = lane >> 2, q = lane & 3, c = (g >> 1) | (g & 1) << 2;
    // Two warps for each place in the ring, for every other sixteen of the channels each, so that whoever waits for a place's next contents has seen the
    // ones before them (a barrier tells only two rounds apart).
    const int st = warp >> 1, half = warp & 1;
    int sum[PAIRS][EIGHTS][4] = {};
    for (int i = st; st < P.stages && i < all; i += P.stages) {
        const int part = i / steps, k0 = (i - part * steps) * stage_k, here = min(per_part, count - part * per_part), mine = (here + 31 - 16 * half) / 32; // sixteens
        if (!__all_sync(~0u, mbar_wait(&full[st], (uint32_t)(i / P.stages) & 1u, &abort_word, P.error, 82))) break;
        const int8_t *stage = ring + st * STAGE_BYTES + (16 * half + c) * BOX_K;
        const int units = min(stage_k, P.ld - k0 + 63) / 64; // 64 bytes
#pragma unroll 2
        for (int u = 0; u < units; ++u) {
            const int8_t *w = stage + (u >> 1) * box_bytes + 16 * ((4 * (u & 1) + q) ^ c), *r = rows + g * P.pitch + k0 + 64 * u + 16 * q;
            int4 x[EIGHTS];
#pragma unroll
            for (int e = 0; e < EIGHTS; ++e) x[e] = *reinterpret_cast<const int4 *>(r + 8 * e * P.pitch);
#pragma unroll
            for (int m = 0; m < PAIRS; ++m) {
                if (m >= mine) continue;
                const int4 a = *reinterpret_cast<const int4 *>(w + 32 * m * BOX_K), b = *reinterpret_cast<const int4 *>(w + (32 * m + 8) * BOX_K);
#pragma unroll
                for (int e = 0; e < EIGHTS; ++e) {
                    mma_i8(sum[m][e], a.x, b.x, a.y, b.y, x[e].x, x[e].y);
                    mma_i8(sum[m][e], a.z, b.z, a.w, b.w, x[e].z, x[e].w);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]); // (a release: the reads of this place are before whatever the copy that waits for it writes there)
        if ((i + P.stages) / steps == part && i + P.stages < all) continue;
        // (the next stage has other channels)
#pragma unroll
        for (int m = 0; m < PAIRS; ++m)
#pragma unroll
            for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int channel = 32 * m + 16 * half + c + 8 * (j >> 1);
                    if (channel < here) atomicAdd(&sums[(8 * e + 2 * q + (j & 1)) * count + part * per_part + channel], sum[m][e][j]);
                    sum[m][e][j] = 0;
                }
    }
    all_but_one();
    if (*(volatile int *)&abort_word) // what has been asked for lands before the block leaves
        for (int w = 0; w < 1000; ++w) __nanosleep(1000);
    for (int i = threadIdx.x; i < n * count; i += 32 * WARPS) {
        const int t = i / count, channel = first + i - t * count;
        store_value(P.y, (size_t)t * P.y_ld + channel, P.y_type, finish_sum((float)sums[i], row_scales[t], P.channel_scales[channel], P.bias ? P.bias[channel] : 0.0f));
    }
}

template <typename T, int EIGHTS, int PAIRS> void product_few_with(CudaDevice &dev, const CUtensorMap &map, const FewParams &P, unsigned grid, size_t smem)
{
    allow_shared_memory(dev, product_few_kernel<T, EIGHTS, PAIRS>);
    launch_following(product_few_kernel<T, EIGHTS, PAIRS>, dim3(grid), dim3(THREADS), smem, dev.stream(), map, P);
}

template <typename T, int EIGHTS> void product_few_pairs(CudaDevice &dev, const CUtensorMap &map, const FewParams &P, unsigned grid, size_t smem)
{
    if (P.box_channels <= 32) product_few_with<T, EIGHTS, 1>(dev, map, P, grid, smem);
    else if (P.box_channels <= 64) product_few_with<T, EIGHTS, EIGHTS == 1 ? 2 : 1>(dev, map, P, grid, smem);
    else product_few_with<T, EIGHTS, EIGHTS == 1 ? 4 : 1>(dev, map, P, grid, smem);
}

} // namespace

bool launch_product_few(CudaDevice &dev, const Product &p, const void *x, int type, size_t ld)
{
    if (!dev.error_word() || p.offsets || p.digits != 1 || p.n > 16) return false;
    // every block quantizes the rows: with more than 25 values a thread (16384 over 20 warps) that takes longer than a kernel before this one
    if (x && (p.n > 2 || p.n * p.width > 16384 || (reinterpret_cast<uintptr_t>(x) | (p.n == 1 ? 0 : ld * value_bytes(type))) % 16)) return false;
    const size_t eights = (p.n + 7) / 8;
    FewParams P{};
    P.rows.x = x, P.rows.n = p.n, P.rows.width = (uint32_t)p.width, P.rows.ld = ld;
    P.given = p.rows, P.given_ld = p.rows_ld, P.given_scales = p.row_scales;
    P.ld = (int)codes_ld(p.width), P.pitch = (P.ld + 127) / 128 * 128 + 64, P.channels = (int)p.channels;
    P.channel_scales = p.channel_scales, P.bias = p.bias, P.y = p.y, P.y_type = p.y_type, P.y_ld = p.y_ld, P.error = dev.error_word();
    // a block for every SM, but none for less than 8 KB
    const unsigned grid = (unsigned)std::max<size_t>(1, std::min<size_t>({(size_t)dev.sm_count(), p.channels, p.channels * P.ld / 8192}));
    const size_t slice = (p.channels + grid - 1) / grid, held = 8 * eights * (P.pitch + slice * sizeof(int));
    if (held + 4 * STAGE_BYTES > SMEM_BYTES) return false;
    if (eights == 2 && slice > 32) return false;
    P.stages = (int)std::min<size_t>(MOST_STAGES, (SMEM_BYTES - held) / STAGE_BYTES);
    const size_t parts = (slice + MOST_CHANNELS - 1) / MOST_CHANNELS; // as few parts as there can be, of the same size
    P.box_channels = (int)((slice + parts - 1) / parts);
    const CUtensorMap map = make_tensor_map_2d<int8_t>(p.codes, P.ld, p.channels, BOX_K, (unsigned)P.box_channels, CU_TENSOR_MAP_SWIZZLE_128B, P.ld);
    const size_t smem = 1024 + P.stages * STAGE_BYTES + held;
    KernelScope ks(dev, "product_few");
    if (!x) eights == 2 ? product_few_pairs<int8_t, 2>(dev, map, P, grid, smem) : product_few_pairs<int8_t, 1>(dev, map, P, grid, smem);
    else if (type == VALUE_F32) product_few_pairs<float, 1>(dev, map, P, grid, smem);
    else if (type == VALUE_F16) product_few_pairs<__half, 1>(dev, map, P, grid, smem);
    else product_few_pairs<__nv_bfloat16, 1>(dev, map, P, grid, smem);
    dev.count_launch();
    return true;
}

} // namespace vqb
