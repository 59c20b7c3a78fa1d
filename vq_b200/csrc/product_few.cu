// product_few.cu -- products of up to eight rows with one matrix, the rows quantized in the same kernel.
//
// Nothing counts here but the matrix's bytes, which are read once, and the time until the first of them arrive.  Every block has a slice of
// the channels, which is one piece of memory: a warp keeps it coming into a ring in shared memory (bulk copies of up to 16 KB) from
// the kernel's first moment on, while the other sixteen quantize the rows; a matrix is complete before any product of it is launched, so
// nothing has to be waited for.  Then each warp takes 512 bytes of a channel at a time, adds four products an instruction (dp4a) for each
// row, and the block's sums meet in shared memory; they are whole numbers, so their order does not matter.  At eight rows the dp4a's
// take about as long as the bytes.
#include <algorithm>

#include "cuda_device.hpp"
#include "rows.cuh"
#include "umma.cuh"

namespace vqb {

namespace {

constexpr int WARPS = 16, THREADS = 32 * (WARPS + 1);
constexpr int MOST_STAGES = 12;
constexpr uint32_t STAGE_BYTES = 16384;
constexpr size_t SMEM_BYTES = 216 << 10;

struct FewParams {
    RowParams rows; // x, n, width, ld (values)
    const int8_t *given; // codes instead
    size_t given_ld;
    const float *given_scales;
    const int8_t *codes;
    size_t ld;
    int channels;
    const float *channel_scales, *bias;
    void *y;
    int y_type;
    size_t y_ld;
    int stages, stage_rows, parts; // a stage: stage_rows whole channels, or one of `parts` parts of a channel
    int *error;
};

__device__ __forceinline__ void sixteen_warps() { asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory"); }

__device__ __forceinline__ void store_value(void *y, size_t at, int type, float v)
{
    if (type == VALUE_F32) static_cast<float *>(y)[at] = v;
    else if (type == VALUE_F16) static_cast<__half *>(y)[at] = from_float<__half>(v);
    else static_cast<__nv_bfloat16 *>(y)[at] = from_float<__nv_bfloat16>(v);
}

// T: the rows' type, int8_t for codes; NT: rows, rounded up
template <typename T, int NT> __global__ void __launch_bounds__(THREADS, 1) product_few_kernel(const FewParams P)
{
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned long long full[MOST_STAGES], empty[MOST_STAGES];
    __shared__ uint32_t parts[WARPS];
    __shared__ float row_scales[NT];
    __shared__ int abort_word;
    const uint32_t stage_bytes = P.parts > 1 ? STAGE_BYTES : (uint32_t)(P.stage_rows * P.ld);
    unsigned char *ring = smem;
    int8_t *rows = reinterpret_cast<int8_t *>(smem + (size_t)P.stages * stage_bytes); // NT x ld
    int *sums = reinterpret_cast<int *>(rows + NT * P.ld);                            // channels x NT
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = (int)((long long)blockIdx.x * P.channels / gridDim.x), count = (int)((long long)(blockIdx.x + 1) * P.channels / gridDim.x) - first;
    const int all = P.parts > 1 ? count * P.parts : (count + P.stage_rows - 1) / P.stage_rows;
    if (threadIdx.x == 32 * WARPS) {
        for (int s = 0; s < P.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], WARPS);
        }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();

    if (warp == WARPS) {
        if (lane == 0) {
            bool ok = true;
            int st = 0;
            uint32_t parity = 0;
            for (int s = 0; s < all; ++s) {
                if (s == P.stages) rows_are_there();
                if (!mbar_wait(&empty[st], parity ^ 1u, &abort_word, P.error, 81)) {
                    ok = false;
                    break;
                }
                const int channel = P.parts > 1 ? s / P.parts : s * P.stage_rows;
                const size_t from = P.parts > 1 ? (size_t)(s % P.parts) * STAGE_BYTES : 0;
                const uint32_t bytes = P.parts > 1 ? (uint32_t)min((size_t)STAGE_BYTES, P.ld - from) : (uint32_t)(min(P.stage_rows, count - channel) * P.ld);
                mbar_expect_tx(&full[st], bytes);
                bulk_load_1d(ring + (size_t)st * stage_bytes, P.codes + (size_t)(first + channel) * P.ld + from, bytes, &full[st]);
                if (++st == P.stages) st = 0, parity ^= 1u;
            }
            if (!ok) // what has been asked for lands before the block leaves
                for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        }
        rows_are_there();
    } else {
        for (int i = threadIdx.x; i < count * NT; i += 32 * WARPS) sums[i] = 0;
        rows_are_there();
        if constexpr (std::is_same<T, int8_t>::value) {
            const int pieces = (int)(P.ld / 16);
            for (int i = threadIdx.x; i < NT * pieces; i += 32 * WARPS) {
                const int t = i / pieces, k = i - t * pieces;
                reinterpret_cast<uint4 *>(rows)[i] = t < P.rows.n ? *reinterpret_cast<const uint4 *>(P.given + t * P.given_ld + 16 * k) : make_uint4(0, 0, 0, 0);
            }
            if (threadIdx.x < NT) row_scales[threadIdx.x] = threadIdx.x < P.rows.n ? P.given_scales[threadIdx.x] : 0.0f;
        } else {
            constexpr int N = Piece<T>::N, LANES = 32 * WARPS / NT;
            const int t = threadIdx.x / LANES, l = threadIdx.x % LANES, pieces = (int)(P.ld / N);
            const bool there = t < P.rows.n;
            const T *row = static_cast<const T *>(P.rows.x) + (there ? t : 0) * P.rows.ld;
            RowOf<T, 1, LANES, true> it(P.rows, t, l, nullptr);
            if (there)
#pragma unroll 4
                for (int i = l; i < pieces; i += LANES) it.look(load_values<T, LANES, true>(row, i / LANES, l, P.rows.width), i / LANES);
            uint32_t most = it.largest();
            if (lane == 0) parts[warp] = most;
            sixteen_warps();
#pragma unroll
            for (int w = 0; w < LANES / 32; ++w) most = max(most, parts[t * (LANES / 32) + w]);
            const float scale = it.scale_of(most);
            const bool none = !there || it.no_codes(most);
            if (l == 0) row_scales[t] = scale;
            const Inverse inverse(none ? 1.0f : scale);
#pragma unroll 2
            for (int i = l; i < pieces; i += LANES) { // (up to ld: zeros behind the width)
                Packed<N> c = {}, unused;
                if (!none) it.pack(load_values<T, LANES, true>(row, i / LANES, l, P.rows.width), i / LANES, inverse, c, unused);
                if (N == 8) reinterpret_cast<uint2 *>(rows + t * P.ld)[i] = make_uint2(c.w[0], c.w[N / 4 - 1]);
                else reinterpret_cast<uint32_t *>(rows + t * P.ld)[i] = c.w[0];
            }
        }
        sixteen_warps();

        int st = 0;
        uint32_t parity = 0;
        for (int s = 0; s < all; ++s) {
            if (!__all_sync(~0u, mbar_wait(&full[st], parity, &abort_word, P.error, 82))) break;
            const int channel = P.parts > 1 ? s / P.parts : s * P.stage_rows, here = P.parts > 1 ? 1 : min(P.stage_rows, count - channel);
            const int from = P.parts > 1 ? (s % P.parts) * (int)STAGE_BYTES : 0, bytes = P.parts > 1 ? min((int)STAGE_BYTES, (int)P.ld - from) : (int)P.ld;
            // 512 bytes a unit; this warp's are neighbours, of one channel for the most part
            const int a_channel = (bytes + 511) / 512, units = here * a_channel, each = (units + WARPS - 1) / WARPS;
            int u = warp * each, c = u / a_channel, i = u - c * a_channel;
            const int end = min(u + each, units);
            while (u < end) {
                int sum[NT] = {};
                const unsigned char *w = ring + (size_t)st * stage_bytes + (size_t)c * P.ld;
                for (; u < end && i < a_channel; ++u, ++i) {
                    const int k = 512 * i + 16 * lane;
                    if (k < bytes) {
                        const int4 a = *reinterpret_cast<const int4 *>(w + k);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const int4 r = *reinterpret_cast<const int4 *>(rows + t * P.ld + from + k);
                            sum[t] = __dp4a(a.x, r.x, sum[t]);
                            sum[t] = __dp4a(a.y, r.y, sum[t]);
                            sum[t] = __dp4a(a.z, r.z, sum[t]);
                            sum[t] = __dp4a(a.w, r.w, sum[t]);
                        }
                    }
                }
                int mine = 0;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int whole = __reduce_add_sync(~0u, sum[t]);
                    if (lane == t) mine = whole;
                }
                if (lane < NT) atomicAdd(&sums[(channel + c) * NT + lane], mine);
                if (i == a_channel) i = 0, ++c;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_relaxed(&empty[st]);
            if (++st == P.stages) st = 0, parity ^= 1u;
        }
        sixteen_warps();
        for (int i = threadIdx.x; i < count * (int)P.rows.n; i += 32 * WARPS) {
            const int t = i / count, c = i - t * count, channel = first + c;
            store_value(P.y, (size_t)t * P.y_ld + channel, P.y_type, finish_sum((float)sums[c * NT + t], row_scales[t], P.channel_scales[channel], P.bias ? P.bias[channel] : 0.0f));
        }
    }
}

template <typename T, int NT> void product_few_with(CudaDevice &dev, const FewParams &P, unsigned grid, size_t smem)
{
    allow_shared_memory(dev, product_few_kernel<T, NT>);
    launch_following(product_few_kernel<T, NT>, dim3(grid), dim3(THREADS), smem, dev.stream(), P);
}

template <typename T> void product_few_rows(CudaDevice &dev, const FewParams &P, int nt, unsigned grid, size_t smem)
{
    if (nt == 1) product_few_with<T, 1>(dev, P, grid, smem);
    else if (nt == 2) product_few_with<T, 2>(dev, P, grid, smem);
    else if (nt == 4) product_few_with<T, 4>(dev, P, grid, smem);
    else product_few_with<T, 8>(dev, P, grid, smem);
}

} // namespace

bool launch_product_few(CudaDevice &dev, const Product &p, const void *x, int type, size_t ld)
{
    if (!dev.error_word() || p.offsets || p.digits != 1 || p.n > 8) return false;
    if (x && (reinterpret_cast<uintptr_t>(x) | (ld * value_bytes(type))) % 16) return false;
    const int nt = p.n <= 1 ? 1 : p.n <= 2 ? 2 : p.n <= 4 ? 4 : 8;
    FewParams P{};
    P.rows.x = x, P.rows.n = p.n, P.rows.width = p.width, P.rows.ld = ld;
    P.given = p.rows, P.given_ld = p.rows_ld, P.given_scales = p.row_scales;
    P.codes = p.codes, P.ld = codes_ld(p.width), P.channels = (int)p.channels;
    P.channel_scales = p.channel_scales, P.bias = p.bias, P.y = p.y, P.y_type = p.y_type, P.y_ld = p.y_ld, P.error = dev.error_word();
    // a block for every SM, but no block for less than 8 KB
    const size_t grid = std::max<size_t>(1, std::min<size_t>({(size_t)dev.sm_count(), p.channels, p.channels * P.ld / 8192}));
    const size_t most_channels = (p.channels + grid - 1) / grid; // of a block
    P.parts = (int)((P.ld + STAGE_BYTES - 1) / STAGE_BYTES);
    P.stage_rows = P.parts > 1 ? 1 : (int)std::min<size_t>(STAGE_BYTES / P.ld, most_channels);
    const size_t stage = P.parts > 1 ? STAGE_BYTES : P.stage_rows * P.ld, held = nt * P.ld + most_channels * nt * sizeof(int);
    if (held + 4 * stage > SMEM_BYTES) return false;
    P.stages = (int)std::min<size_t>(MOST_STAGES, (SMEM_BYTES - held) / stage);
    const size_t smem = P.stages * stage + held;
    KernelScope ks(dev, "product_few");
    if (!x) product_few_rows<int8_t>(dev, P, nt, (unsigned)grid, smem);
    else if (type == VALUE_F32) product_few_rows<float>(dev, P, nt, (unsigned)grid, smem);
    else if (type == VALUE_F16) product_few_rows<__half>(dev, P, nt, (unsigned)grid, smem);
    else product_few_rows<__nv_bfloat16>(dev, P, nt, (unsigned)grid, smem);
    dev.count_launch();
    return true;
}

} // namespace vqb
