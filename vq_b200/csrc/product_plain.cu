// product_plain.cu -- the products of codes on the CUDA cores: what VQB_NO_TENSOR=1 runs, and what product_tc.cu is compared with.
//
// A block takes 64 channels x 64 rows; 64 bytes of both at a time go through shared memory, a thread keeps 4 x 4 sums and adds four
// products an instruction (dp4a).  What bounds it is that instruction, which runs at some ten lanes an SM and cycle here.
#include <algorithm>

#include "cuda_device.hpp"
#include "qmat.cuh"

namespace vqb {

namespace {

constexpr int TILE = 64, BYTES = 64, PITCH = BYTES / 4 + 1;

struct PlainParams {
    const int8_t *codes, *rows;
    size_t ld, rows_ld, plane; // plane: bytes from digit to digit
    const float *channel_scales, *row_scales, *bias;
    const long long *offsets;
    int groups, channels, width, n;
    void *y;
    size_t y_ld;
    int zero_rest;
};

// 64 rows of 64 bytes to shared memory, zeros outside; rows and their bytes as they come (any alignment)
__device__ __forceinline__ void stage(const int8_t *from, size_t ld, int rows, int k0, int width, int (*to)[PITCH])
{
    for (int i = threadIdx.x; i < TILE * (BYTES / 4); i += blockDim.x) {
        const int r = i / (BYTES / 4), k = k0 + 4 * (i % (BYTES / 4));
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if (r < rows && k + b < width) w |= (uint32_t)(uint8_t)from[(size_t)r * ld + k + b] << (8 * b);
        to[r][i % (BYTES / 4)] = (int)w;
    }
}

template <typename T, int DIGITS> __global__ void __launch_bounds__(256) product_plain_kernel(const PlainParams P)
{
    extern __shared__ int walk[];
    __shared__ int cs[TILE][PITCH], rs[DIGITS][TILE][PITCH];
    RowTiles tiles(walk, P.groups);
    tiles.build(P.offsets, P.groups, P.n, TILE);
    const int per_row_tile = (P.channels + TILE - 1) / TILE;
    const long long total = (long long)tiles.before[P.groups] * per_row_tile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    T *y = static_cast<T *>(P.y);
    if (P.zero_rest)
        zero_rest<T>(y, P.y_ld, P.channels, P.n, tiles.first[0], tiles.end(P.groups - 1), (size_t)blockIdx.x * blockDim.x + threadIdx.x, (size_t)gridDim.x * blockDim.x);
    for (long long tile = blockIdx.x; tile < total; tile += gridDim.x) {
        const int u = (int)(tile / per_row_tile), j0 = (int)(tile % per_row_tile) * TILE;
        const int g = tiles.group_of(u, P.groups);
        const int r0 = tiles.first[g] + (u - tiles.before[g]) * TILE, rows = min(TILE, tiles.end(g) - r0), channels = min(TILE, P.channels - j0);
        int sum[DIGITS][4][4] = {};
        for (int k0 = 0; k0 < P.width; k0 += BYTES) {
            __syncthreads();
            stage(P.codes + ((size_t)g * P.channels + j0) * P.ld, P.ld, channels, k0, P.width, cs);
#pragma unroll
            for (int d = 0; d < DIGITS; ++d) stage(P.rows + d * P.plane + (size_t)r0 * P.rows_ld, P.rows_ld, rows, k0, P.width, rs[d]);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < BYTES / 4; ++k)
#pragma unroll
                for (int d = 0; d < DIGITS; ++d)
#pragma unroll
                    for (int a = 0; a < 4; ++a)
#pragma unroll
                        for (int b = 0; b < 4; ++b) sum[d][a][b] = __dp4a(rs[d][ty + 16 * a][k], cs[tx + 16 * b][k], sum[d][a][b]);
        }
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int r = ty + 16 * a, j = tx + 16 * b;
                if (r >= rows || j >= channels) continue;
                const size_t channel = (size_t)g * P.channels + j0 + j;
                const float s = DIGITS == 3 ? join_digits(sum[0][a][b], sum[DIGITS / 2][a][b], sum[DIGITS - 1][a][b]) : (float)sum[0][a][b];
                y[(size_t)(r0 + r) * P.y_ld + j0 + j] = from_float<T>(finish_sum(s, P.row_scales[r0 + r], P.channel_scales ? P.channel_scales[channel] : 1.0f, P.bias ? P.bias[channel] : 0.0f));
            }
    }
}

template <typename T> void product_plain_typed(CudaDevice &dev, const PlainParams &P, int digits)
{
    const size_t tiles = ((size_t)P.n / TILE + P.groups) * ((P.channels + TILE - 1) / TILE);
    const dim3 grid((unsigned)std::min<size_t>(tiles, (size_t)dev.sm_count() * 8));
    const size_t smem = RowTiles::bytes(P.groups);
    if (digits == 3) product_plain_kernel<T, 3><<<grid, 256, smem, dev.stream()>>>(P);
    else product_plain_kernel<T, 1><<<grid, 256, smem, dev.stream()>>>(P);
    VQB_CUDA_CHECK(cudaGetLastError());
}

} // namespace

void launch_product_plain(CudaDevice &dev, const Product &p)
{
    PlainParams P{p.codes, p.rows, codes_ld(p.width), p.rows_ld, p.n * p.rows_ld, p.channel_scales, p.row_scales, p.bias, reinterpret_cast<const long long *>(p.offsets),
                  (int)p.groups, (int)p.channels, (int)p.width, (int)p.n, p.y, p.y_ld, p.zero_rest};
    KernelScope ks(dev, "product_plain");
    if (p.y_type == VALUE_F32) product_plain_typed<float>(dev, P, p.digits);
    else if (p.y_type == VALUE_F16) product_plain_typed<__half>(dev, P, p.digits);
    else product_plain_typed<__nv_bfloat16>(dev, P, p.digits);
    dev.count_launch();
}

} // namespace vqb
