// product_tc.cu -- the products of codes on the tensor cores (tcgen05, kind::i8, whole-number sums in tensor memory).
//
// Channels are the accumulator's lanes and rows of codes its columns, so that a tile can have any number of rows (a group's last
// ones, a few tokens) at the cost of 32 each, and the result of one row leaves in pieces of 32 neighbouring channels.  A CTA keeps
// taking tiles of 128 channels x up to 256 rows:
//
//   warp 0      TMA: 128 bytes of 128 channels and of the tile's rows a stage, four stages
//   warp 1      one thread issues tcgen05.mma, 4 x 32 bytes a stage; two accumulators of 256 columns, so that the next tile's sums
//               begin while the last one's leave
//   warps 2-5   epilogue: scales, bias, rounding, stores
//
// Two digits (gradients): the columns' first half are the rows' high digits, the second half the low ones; the epilogue joins them.
#include <algorithm>

#include "cuda_device.hpp"
#include "qmat.cuh"
#include "tma_host.hpp"
#include "umma.cuh"

namespace vqb {

namespace {

constexpr int BM = 128;        // channels a tile
constexpr int MOST_COLS = 256; // accumulator columns a tile
constexpr int KB = 128;        // bytes of K a stage: one swizzled row
constexpr int NST = 4;
constexpr int THREADS = 192;
constexpr uint32_t A_BYTES = BM * KB, B_BYTES = MOST_COLS * KB;

struct alignas(8) Barriers {
    unsigned long long full[NST], empty[NST], tfull[2], tempty[2], drained;
    uint32_t tmem_base;
    int abort_flag;
};

struct TcParams {
    int groups, channels, width, n;
    const long long *offsets;
    const float *channel_scales, *row_scales, *bias;
    void *y;
    size_t y_ld;
    int tile_rows; // rows a tile, a multiple of 32; times DIGITS at most 256
    int box_rows;  // rows a token load brings
    int band;      // tiles of rows that are taken together for one tile of channels
    int zero_rest, rows_follow;
    int *error;
};

// kind::i8: signed operands, 32-bit sums, both K-major, M = 128, N = n
__device__ __forceinline__ uint32_t idesc_i8(int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24); }

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(tmem_d),
                 "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u)
                 : "memory");
}

struct Tile {
    int group, channel0, row0, rows;
};

// Tile number id: `band` tiles of rows for one tile of channels, then the next channels, then the next band.  What a wave of CTAs reads is
// then some channels and some rows, instead of all channels for each tile of rows.
__device__ __forceinline__ Tile tile_at(const TcParams &P, const RowTiles &tiles, long long id, int channel_tiles)
{
    const int all = tiles.before[P.groups];
    const long long per_band = (long long)P.band * channel_tiles;
    const int b = (int)(id / per_band), in = (int)(id % per_band), here = min(P.band, all - b * P.band);
    const int u = b * P.band + in % here;
    Tile t;
    t.group = tiles.group_of(u, P.groups);
    t.channel0 = in / here * BM;
    t.row0 = tiles.first[t.group] + (u - tiles.before[t.group]) * P.tile_rows;
    t.rows = min(P.tile_rows, tiles.end[t.group] - t.row0);
    return t;
}

// Accumulator columns of one digit: rows in steps of 32.  The low digits' rows begin where the loads of the high ones end.
template <int DIGITS> __device__ __forceinline__ int columns_of(const TcParams &P, int rows)
{
    const int step = DIGITS == 2 ? P.box_rows : 32;
    return (rows + step - 1) / step * step;
}

template <typename T, int DIGITS>
__global__ void __launch_bounds__(THREADS, 1) product_tc_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_rows, const TcParams P)
{
    extern __shared__ unsigned char smem_raw[];
    unsigned char *base = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *a_smem = base, *b_smem = base + NST * A_BYTES;
    float *scales_smem = reinterpret_cast<float *>(b_smem + NST * B_BYTES); // 4 warps x 256
    Barriers *bars = reinterpret_cast<Barriers *>(scales_smem + 4 * MOST_COLS);
    RowTiles tiles(bars + 1, P.groups);
    volatile int *abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bars->tfull[b], 1);
            mbar_init(&bars->tempty[b], 4);
        }
        mbar_init(&bars->drained, 1);
        bars->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // Codes of the matrix may be fetched before the rows' are there, where only those are new.
    const bool codes_first = P.rows_follow && !P.offsets;
    if (!codes_first) rows_are_there();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    tiles.build(P.offsets, P.groups, P.n, P.tile_rows); // (block barriers)
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = bars->tmem_base;
    const int channel_tiles = (P.channels + BM - 1) / BM, chunks = (P.width + KB - 1) / KB;
    const long long total = (long long)tiles.before[P.groups] * channel_tiles;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true, waited = !codes_first;
            auto load_rows = [&](const Tile &t, int columns, int c, int st) {
                unsigned char *to = b_smem + st * B_BYTES;
                for (int d = 0; d < DIGITS; ++d, to += columns * KB)
                    for (int i = 0; i < columns; i += P.box_rows) tma_load_2d(to + i * KB, &map_rows, c * KB, d * P.n + t.row0 + i, &bars->full[st]);
            };
            for (long long id = blockIdx.x; ok && id < total; id += gridDim.x) {
                const Tile t = tile_at(P, tiles, id, channel_tiles);
                const int columns = columns_of<DIGITS>(P, t.rows);
                const uint32_t bytes = A_BYTES + (uint32_t)(DIGITS * ((columns + P.box_rows - 1) / P.box_rows) * P.box_rows * KB);
                const int ahead = waited ? 0 : min(NST, chunks);
                for (int c = 0; c < chunks; ++c, ++it) {
                    const int st = it % NST;
                    if (!mbar_wait(&bars->empty[st], ((it / NST) & 1u) ^ 1u, abort_flag, P.error, 61)) {
                        ok = false;
                        break;
                    }
                    mbar_expect_tx(&bars->full[st], bytes);
                    tma_load_2d(a_smem + st * A_BYTES, &map_codes, c * KB, t.group * P.channels + t.channel0, &bars->full[st]);
                    if (c + 1 < ahead) continue;
                    if (!waited) {
                        rows_are_there();
                        waited = true;
                        for (int e = 0; e < ahead; ++e) load_rows(t, columns, e, e);
                    } else {
                        load_rows(t, columns, c, st);
                    }
                }
            }
            if (!waited) rows_are_there();
            // what has been asked for has landed before the block leaves (a tile that is finished has been waited for)
            if (!ok)
                for (uint32_t i = it > NST ? it - NST : 0; i < it; ++i) mbar_wait(&bars->full[i % NST], (i / NST) & 1u, abort_flag, P.error, 62);
        } else if (codes_first) {
            rows_are_there();
        }
    } else if (warp == 1) {
        if (codes_first) rows_are_there();
        if (lane == 0) {
            uint32_t it = 0, local = 0;
            bool ok = true;
            for (long long id = blockIdx.x; ok && id < total; id += gridDim.x, ++local) {
                const Tile t = tile_at(P, tiles, id, channel_tiles);
                const uint32_t b = local & 1u, idesc = idesc_i8(DIGITS * columns_of<DIGITS>(P, t.rows)), d_tmem = tmem_base + b * MOST_COLS;
                if (!mbar_wait(&bars->tempty[b], ((local >> 1) & 1u) ^ 1u, abort_flag, P.error, 63)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int c = 0; c < chunks; ++c, ++it) {
                    const int st = it % NST;
                    if (!mbar_wait(&bars->full[st], (it / NST) & 1u, abort_flag, P.error, 64)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t a = smem_desc_sw128(smem_u32(a_smem + st * A_BYTES)), r = smem_desc_sw128(smem_u32(b_smem + st * B_BYTES));
                    const int steps = min(KB / 32, (P.width - c * KB + 31) / 32);
                    for (int s = 0; s < steps; ++s) umma_i8(d_tmem, a + (uint64_t)(2 * s), r + (uint64_t)(2 * s), idesc, (c | s) ? 1u : 0u);
                    umma_commit(&bars->empty[st]);
                }
                if (ok) umma_commit(&bars->tfull[b]);
            }
            if (*abort_flag) { // nothing of the tensor core's is under way when the block leaves
                umma_commit(&bars->drained);
                mbar_wait(&bars->drained, 0, abort_flag, P.error, 65);
            }
        }
    } else {
        if (codes_first) rows_are_there();
        const int q = warp & 3; // the quarter of the lanes that this warp may read
        float *mine = scales_smem + q * MOST_COLS;
        T *y = static_cast<T *>(P.y);
        uint32_t local = 0;
        for (long long id = blockIdx.x; id < total; id += gridDim.x, ++local) {
            const Tile t = tile_at(P, tiles, id, channel_tiles);
            const uint32_t b = local & 1u;
            const int channel = t.channel0 + 32 * q + lane, columns = columns_of<DIGITS>(P, t.rows);
            const bool there = channel < P.channels;
            const size_t at = (size_t)t.group * P.channels + channel;
            const float channel_scale = !there ? 0.0f : P.channel_scales ? P.channel_scales[at] : 1.0f, bias = there && P.bias ? P.bias[at] : 0.0f;
            __syncwarp();
            for (int i = lane; i < columns; i += 32) mine[i] = i < t.rows ? P.row_scales[t.row0 + i] : 0.0f;
            __syncwarp();
            if (!__all_sync(~0u, mbar_wait(&bars->tfull[b], (local >> 1) & 1u, abort_flag, P.error, 66))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem_base + ((uint32_t)(32 * q) << 16) + b * MOST_COLS;
            for (int c0 = 0; c0 < columns; c0 += 32) {
                uint32_t acc[32], low[32];
                tmem_ld32_issue(taddr + c0, acc);
                if (DIGITS == 2) tmem_ld32_issue(taddr + columns + c0, low);
                tmem_wait();
                T *to = y + (size_t)(t.row0 + c0) * P.y_ld + channel;
                const int left = there ? t.rows - c0 : 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float sum = DIGITS == 2 ? __fmaf_rn(128.0f, (float)(int)acc[i], (float)(int)low[i]) : (float)(int)acc[i];
                    if (i < left) to[(size_t)i * P.y_ld] = from_float<T>(finish_sum(sum, mine[c0 + i], channel_scale, bias));
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->tempty[b]);
        }
        if (P.zero_rest)
            zero_rest<T>(y, P.y_ld, P.channels, P.n, tiles.first[0], tiles.end[P.groups - 1], (size_t)blockIdx.x * 128 + (threadIdx.x - 64), (size_t)gridDim.x * 128);
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

template <typename T, int DIGITS> void product_tc_typed(CudaDevice &dev, const Product &p, TcParams &P, const CUtensorMap &map_codes, const CUtensorMap &map_rows, unsigned grid)
{
    const size_t smem = 1024 + NST * (A_BYTES + B_BYTES) + 4 * MOST_COLS * sizeof(float) + sizeof(Barriers) + RowTiles::bytes(p.groups);
    allow_shared_memory(dev, product_tc_kernel<T, DIGITS>);
    launch_following(product_tc_kernel<T, DIGITS>, dim3(grid), dim3(THREADS), smem, dev.stream(), map_codes, map_rows, P);
}

template <typename T> void product_tc_digits(CudaDevice &dev, const Product &p, TcParams &P, const CUtensorMap &mc, const CUtensorMap &mr, unsigned grid)
{
    if (p.digits == 2) product_tc_typed<T, 2>(dev, p, P, mc, mr, grid);
    else product_tc_typed<T, 1>(dev, p, P, mc, mr, grid);
}

} // namespace

void launch_product(CudaDevice &dev, const Product &p)
{
    if (!dev.error_word()) return launch_product_plain(dev, p); // VQB_NO_TENSOR=1
    TcParams P{};
    P.groups = (int)p.groups, P.channels = (int)p.channels, P.width = (int)p.width, P.n = (int)p.n;
    P.offsets = reinterpret_cast<const long long *>(p.offsets);
    P.channel_scales = p.channel_scales, P.row_scales = p.row_scales, P.bias = p.bias;
    P.y = p.y, P.y_ld = p.y_ld, P.zero_rest = p.zero_rest, P.rows_follow = p.rows_follow, P.error = dev.error_word();
    const size_t most = MOST_COLS / p.digits;
    if (p.offsets) {
        P.tile_rows = (int)most;
        P.box_rows = p.n / p.groups >= 64 ? 64 : 32;
    } else { // as few tiles as there can be, of the same size
        const size_t tiles = (p.n + most - 1) / most;
        P.tile_rows = (int)(((p.n + tiles - 1) / tiles + 31) / 32 * 32);
        P.box_rows = P.tile_rows;
    }
    P.band = 8;
    const CUtensorMap map_codes = make_tensor_map_2d<int8_t>(p.codes, p.width, p.groups * p.channels, KB, BM, CU_TENSOR_MAP_SWIZZLE_128B, codes_ld(p.width));
    const CUtensorMap map_rows = make_tensor_map_2d<int8_t>(p.rows, p.width, p.digits * p.n, KB, (unsigned)P.box_rows, CU_TENSOR_MAP_SWIZZLE_128B, p.rows_ld);
    const size_t row_tiles = p.offsets ? p.n / P.tile_rows + p.groups : (p.n + P.tile_rows - 1) / P.tile_rows;
    const unsigned grid = (unsigned)std::min<size_t>((size_t)dev.sm_count(), row_tiles * ((p.channels + BM - 1) / BM));
    KernelScope ks(dev, "product_tc");
    if (p.y_type == VALUE_F32) product_tc_digits<float>(dev, p, P, map_codes, map_rows, grid);
    else if (p.y_type == VALUE_F16) product_tc_digits<__half>(dev, p, P, map_codes, map_rows, grid);
    else product_tc_digits<__nv_bfloat16>(dev, p, P, map_codes, map_rows, grid);
    dev.count_launch();
}

} // namespace vqb
