// qmat.cuh -- what the kernels on 8-bit codes share: which rows a tile has, how a result leaves, when the rows are there.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "qmat.hpp"

namespace vqb {

// Kernels of a product may start before the kernel in front of them ends.  All earlier work of the stream is complete and visible
// from here on; every thread calls it before it reads what that kernel may have written, or leaves.  (What is read before: codes of a matrix,
// which is complete when the call that made it returns.)
__device__ __forceinline__ void rows_are_there() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Only where a product of the same call comes next: a kernel of another call may take this one's results for memory that stays the same.
__device__ __forceinline__ void product_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A sum of products of codes to the value it stands for.  Sums above 2^24 round to f32 here, as each step behind does.
__device__ __forceinline__ float finish_sum(float sum, float row_scale, float channel_scale, float bias)
{
    return __fmaf_rn(__fmul_rn(sum, row_scale), channel_scale, bias);
}

// What the sums of three digits stand for.
__device__ __forceinline__ float join_digits(int first, int middle, int last) { return __fmaf_rn(65536.0f, (float)first, __fmaf_rn(256.0f, (float)middle, (float)last)); }

// How the rows of all groups fall into tiles of at most `rows` rows: tile u belongs to the last group g with before[g] <= u, and starts at row
// first[g] + (u - before[g]) * rows.  In shared memory.  Offsets come from the device unchecked: whatever they are, every group has some of the n
// rows that there are, and no row has two groups.
struct RowTiles {
    int *before; // groups + 1
    int *first;  // groups + 1: group g has rows first[g] .. first[g + 1] - 1
    static __host__ __device__ constexpr size_t bytes(size_t groups) { return 2 * (groups + 1) * sizeof(int); }
    __device__ __forceinline__ RowTiles(void *smem, int groups) : before(static_cast<int *>(smem)), first(before + groups + 1) {}
    __device__ __forceinline__ int end(int g) const { return first[g + 1]; }

    // by all threads of the block; ends with a block barrier
    __device__ __forceinline__ void build(const long long *offsets, int groups, int n, int rows)
    {
        for (int g = threadIdx.x; g <= groups; g += blockDim.x) {
            const long long a = offsets ? offsets[g] : g ? n : 0;
            first[g] = (int)(a < 0 ? 0 : a > n ? n : a);
        }
        __syncthreads();
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x;
            int most = 0, tiles = 0;
            for (int g0 = 0; g0 <= groups; g0 += 32) { // ascending
                int v = g0 + lane <= groups ? first[g0 + lane] : 0;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int up = __shfl_up_sync(~0u, v, d);
                    if (lane >= d) v = max(v, up);
                }
                v = max(v, most);
                if (g0 + lane <= groups) first[g0 + lane] = v;
                most = __shfl_sync(~0u, v, 31);
            }
            __syncwarp();
            if (lane == 0) before[0] = 0;
            for (int g0 = 0; g0 < groups; g0 += 32) {
                const int g = g0 + lane;
                int v = g < groups ? (first[g + 1] - first[g] + rows - 1) / rows : 0;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int up = __shfl_up_sync(~0u, v, d);
                    if (lane >= d) v += up;
                }
                if (g < groups) before[g + 1] = tiles + v;
                tiles += __shfl_sync(~0u, v, 31);
            }
        }
        __syncthreads();
    }
    __device__ __forceinline__ int group_of(int u, int groups) const
    {
        int lo = 0, hi = groups - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before[mid] <= u) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
};

// Rows in front of the first group and behind the last one become 0, by `threads` threads of which this is number t.
template <typename T> __device__ void zero_rest(T *y, size_t ld, int channels, int n, int head, int tail, size_t t, size_t threads)
{
    const size_t rest = (size_t)head + (size_t)(n - tail);
    for (size_t i = t; i < rest * channels; i += threads) {
        const size_t r = i / channels;
        y[(r < (size_t)head ? r : r - head + tail) * ld + i % channels] = from_float<T>(0.0f);
    }
}

} // namespace vqb
