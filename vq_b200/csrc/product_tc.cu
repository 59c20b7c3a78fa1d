// product_tc.cu -- the products of codes on the tensor cores (tcgen05, kind::i8, whole-number sums in tensor memory).
//
// Channels are the accumulator's lanes and rows of codes its columns, so that a tile can have any number of rows (a group's last
// ones, a few tokens) at the cost of 32 each, and the result of one row leaves in pieces of 32 neighbouring channels.  Two CTAs of a
// cluster (one pair of SMs, cta_group::2) keep taking tiles of 256 channels x up to 256 rows: each fetches its 128 channels and one half of
// the rows, both halves are multiplied with both CTAs' channels, and each has its channels' sums in its own tensor memory.
//
//   warp 0      TMA: 128 bytes of 128 channels and of half the tile's rows a stage, six stages
//   warp 1      in the first CTA one thread issues tcgen05.mma for both, 4 x 32 bytes a stage; two accumulators of 256 columns,
//               so that the next tile's sums begin while the last one's leave
//   warps 2-9   epilogue: scales, bias, rounding, stores; two warps share the lanes that either may read and take turns at 32 columns each.
//               16-bit results go through shared memory, two rows' values of a channel in a word, and leave 16 bytes at a time
//
// Where there are too few tiles for the SMs, two or four pairs of a larger cluster take a part of the width each, one tile a cluster.  Their sums stay in
// their shared memory (the ring is free by then), and every pair finishes some of the rows, adding up what the others have there: whole
// numbers, so that nothing depends on their order, and no memory outside the SMs that would have to be zero.
//
// Three digits (gradients): the first CTA fetches the rows' first digits and the second one their middle digits, each half of the last ones; two instructions a step, the
// first one's columns' halves are the first and the middle sums, the second one's the last sums.  A tile of 128 rows has 384 columns, for which there is room once: its sums
// are joined in registers, and the next tile's begin, before they leave.  (Tiles of 64 rows, two at a time, read 1.9 GB of L2 for 4096 x 4096 x 4096 and take 170 us for that, not 120.)
#include <algorithm>
#include <map>
#include <mutex>

#include "cuda_device.hpp"
#include "qmat.cuh"
#include "tma_host.hpp"
#include "umma.cuh"

namespace vqb {

namespace {

constexpr int BM = 128;        // channels a CTA and tile
constexpr int MOST_COLS = 256; // accumulator columns a tile
constexpr int KB = 128;        // bytes of K a stage: one swizzled row
constexpr int MOST_STAGES = 6;
constexpr int EPILOGUE_WARPS = 8, THREADS = 64 + 32 * EPILOGUE_WARPS;
constexpr int STAGE_WORDS = 36; // 32 channels' words and 16 bytes, so that rows start in different banks
constexpr uint32_t A_BYTES = BM * KB, B_BYTES = MOST_COLS / 2 * KB; // with three digits another half of B_BYTES follows
template <int DIGITS> constexpr uint32_t STAGE_BYTES = A_BYTES + (DIGITS == 3 ? B_BYTES * 3 / 2 : B_BYTES);

struct alignas(8) Barriers {
    unsigned long long full[MOST_STAGES], empty[MOST_STAGES], tfull[2], tempty[2], drained; // full, tempty, drained: the first CTA's count for both
    uint32_t tmem_base;
    int abort_flag;
};

struct TcParams {
    int groups, channels, width, n;
    const long long *offsets;
    const float *channel_scales, *row_scales, *bias;
    void *y;
    size_t y_ld;
    int tile_rows; // rows a tile, a multiple of 32, at most 256; 128 with three digits
    int stages;    // 6; with three digits 5, or 4 beside many groups' offsets
    int band;      // tiles of rows that are taken together for one tile of channels
    int zero_rest, rows_follow;
    int parts; // of the width, a pair each
    int wide; // results can be stored 16 bytes at a time
    int *error;
};

// kind::i8: signed operands, 32-bit sums, both K-major, M = 256 (two CTAs), N = n
__device__ __forceinline__ uint32_t idesc_i8(int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(2 * BM >> 4) << 24); }

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
                 "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
                 : "memory");
}

// Arrives at the same barrier of both CTAs once all that this thread has issued is done.
__device__ __forceinline__ void commit_both(void *bar, uint32_t leader)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)(3u << leader)) : "memory");
}
__device__ __forceinline__ void commit_here(void *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// The address of another CTA's copy of a shared-memory object.
__device__ __forceinline__ uint32_t in_cta(const void *p, uint32_t rank)
{
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ int4 load_cluster(uint32_t addr)
{
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
// A load into this CTA that counts at a barrier of the first one (no multicast).
__device__ __forceinline__ void tma_load_counted(void *dst, const CUtensorMap *map, int c0, int c1, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)), "l"(map),
                 "r"(bar), "r"(c0), "r"(c1)
                 : "memory");
}
// The same of a map with planes.
__device__ __forceinline__ void tma_load_plane_counted(void *dst, const CUtensorMap *map, int c0, int c1, int c2, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)), "l"(map),
                 "r"(bar), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
// Hands an accumulator back.  Nothing but tensor memory is handed over, and what orders that is the pair of tcgen05 fences around the barrier: PTX has tcgen05.ld of one thread before
// tcgen05.mma of another as tcgen05.wait::ld, tcgen05.fence::before_thread_sync and a relaxed arrival, then the wait and tcgen05.fence::after_thread_sync.  (The other lanes' loads
// and fences are before the arrival by __syncwarp.)  A release would wait for the results' stores, too, 1 us a tile.
__device__ __forceinline__ void arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// two results of one channel, of the rows 2 i (low half) and 2 i + 1
template <typename T> __device__ __forceinline__ uint32_t two_values(float a, float b);
template <> __device__ __forceinline__ uint32_t two_values<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t two_values<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t two_values<float>(float, float) { return 0; } // (f32 leaves as it is)

struct Tile {
    int group, channel0, row0, rows;
};

// Tile number id: `band` tiles of rows for one tile of channels, then the next channels, then the next band.  What a wave of CTAs reads is
// then some channels and some rows, instead of all channels for each tile of rows.
__device__ __forceinline__ Tile tile_at(const TcParams &P, const RowTiles &tiles, int id, int channel_tiles)
{
    const int per_band = P.band * channel_tiles, b = id / per_band, in = id - b * per_band, here = min(P.band, tiles.before[P.groups] - b * P.band);
    const int c = in / here, u = b * P.band + in - c * here;
    Tile t;
    t.group = tiles.group_of(u, P.groups);
    t.channel0 = c * (2 * BM);
    t.row0 = tiles.first[t.group] + (u - tiles.before[t.group]) * P.tile_rows;
    t.rows = min(P.tile_rows, tiles.end(t.group) - t.row0);
    return t;
}

// Accumulator columns of one digit: rows in steps of 32 (16 for each box).
__device__ __forceinline__ int columns_of(int rows) { return (rows + 31) / 32 * 32; }

template <typename T, int DIGITS, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) product_tc_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_rows,
                                                                const __grid_constant__ CUtensorMap map_half, const TcParams P)
{
    extern __shared__ unsigned char smem_raw[];
    unsigned char *base = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int nst = DIGITS == 3 ? P.stages : MOST_STAGES;
    constexpr uint32_t B_STAGE = STAGE_BYTES<DIGITS> - A_BYTES;
    unsigned char *a_smem = base, *b_smem = base + nst * A_BYTES;
    float *scales_smem = reinterpret_cast<float *>(b_smem + nst * B_STAGE);                                 // 8 warps x 128
    uint32_t *out_smem = reinterpret_cast<uint32_t *>(scales_smem + EPILOGUE_WARPS * MOST_COLS / 2);        // 8 warps x 16 x STAGE_WORDS
    Barriers *bars = reinterpret_cast<Barriers *>(out_smem + EPILOGUE_WARPS * 16 * STAGE_WORDS);
    RowTiles tiles(bars + 1, P.groups);
    volatile int *abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = SPLIT ? P.parts : 1, rank = blockIdx.x % (2 * parts), half = rank & 1, part = rank >> 1; // this CTA's place in its cluster
    const uint32_t leader = rank & ~1;                                                                          // the first one of its pair

    if (threadIdx.x == 0) {
        for (int s = 0; s < nst; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bars->tfull[b], 1);
            mbar_init(&bars->tempty[b], 2 * EPILOGUE_WARPS);
        }
        mbar_init(&bars->drained, 1);
        bars->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    // Codes of the matrix may be fetched before the rows' are there; which of them, offsets say, where there are some.
    const bool codes_first = !P.offsets || P.rows_follow;
    if (!codes_first) rows_are_there();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    tiles.build(P.offsets, P.groups, P.n, P.tile_rows); // (block barriers)
    cluster_sync();                                     // both CTAs' barriers are there
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = bars->tmem_base;
    const int twice = DIGITS == 1 || 3 * P.tile_rows <= MOST_COLS; // room for two tiles' sums
    const int channel_tiles = (P.channels + 2 * BM - 1) / (2 * BM), chunks = (P.width + KB - 1) / KB;
    const int c_begin = chunks * part / parts, c_end = chunks * (part + 1) / parts;
    const int total = tiles.before[P.groups] * channel_tiles, first = blockIdx.x / (2 * parts), step = gridDim.x / (2 * parts);

    if (warp == 0) {
        if (lane == 0) {
            int st = 0;
            uint32_t parity = 0; // of the stages' current round
            bool ok = true, waited = !codes_first;
            const uint32_t bytes = 2 * (A_BYTES + (uint32_t)(DIGITS == 3 ? 3 : 1) * P.tile_rows / 2 * KB), full0 = in_cta(&bars->full[0], leader);
            unsigned long long loads = 0;
            for (int id = first; ok && id < total; id += step) {
                const Tile t = tile_at(P, tiles, id, channel_tiles);
                // This CTA's rows: one half of the columns, or one digit of all and half of the last one's.  Boxes are those of a whole tile: what is behind the tile's rows is
                // not multiplied.
                const int mid = t.row0 + half * (columns_of(t.rows) / 2);
                const int channel = t.group * P.channels + t.channel0 + half * BM;
                auto load_rows = [&](int stage, int c) {
                    unsigned char *to = b_smem + stage * B_STAGE;
                    if (DIGITS == 1) {
                        tma_load_counted(to, &map_rows, c * KB, mid, full0 + 8u * stage);
                    } else {
                        tma_load_plane_counted(to, &map_rows, c * KB, t.row0, half, full0 + 8u * stage);
                        tma_load_plane_counted(to + B_BYTES, &map_half, c * KB, mid, 2, full0 + 8u * stage);
                    }
                };
                const int ahead = waited ? 0 : min(nst, c_end - c_begin);
                for (int c = c_begin; c < c_end; ++c) {
                    if (!mbar_wait(&bars->empty[st], parity ^ 1u, abort_flag, P.error, 61)) {
                        ok = false;
                        break;
                    }
                    if (half == 0) mbar_expect_tx(&bars->full[st], bytes);
                    tma_load_counted(a_smem + st * A_BYTES, &map_codes, c * KB, channel, full0 + 8u * st);
                    ++loads;
                    if (c - c_begin + 1 >= ahead) {
                        if (!waited) {
                            rows_are_there();
                            waited = true;
                            for (int e = 0; e < ahead; ++e) load_rows(e, c_begin + e);
                        } else {
                            load_rows(st, c);
                        }
                    }
                    if (++st == nst) st = 0, parity ^= 1u;
                }
            }
            if (!waited) rows_are_there();
            if (ok) { // the tensor core's arrivals here have come before the block leaves
                for (int i = 0; i < nst; ++i) {
                    if (loads + i >= nst) mbar_wait(&bars->empty[st], parity ^ 1u, abort_flag, P.error, 62);
                    if (++st == nst) st = 0, parity ^= 1u;
                }
            } else { // what has been asked for lands
                for (int i = 0; i < 1000; ++i) __nanosleep(1000);
            }
        } else if (codes_first) {
            rows_are_there();
        }
    } else if (warp == 1) {
        if (codes_first) rows_are_there();
        if (half == 0 && elect_one()) {
            int st = 0;
            uint32_t parity = 0, local = 0;
            bool ok = true;
            const uint64_t a0 = smem_desc_sw128(smem_u32(a_smem)), r0 = smem_desc_sw128(smem_u32(b_smem));
            for (int id = first; ok && id < total; id += step, ++local) {
                const Tile t = tile_at(P, tiles, id, channel_tiles);
                const int columns = columns_of(t.rows);
                const uint32_t b = twice ? local & 1u : 0u, idesc = idesc_i8(DIGITS == 3 ? 2 * columns : columns), d_tmem = tmem_base + b * MOST_COLS;
                const uint32_t idesc_last = idesc_i8(columns), last_tmem = d_tmem + 2 * columns; // (three digits)
                if (!mbar_wait(&bars->tempty[b], ((twice ? local >> 1 : local) & 1u) ^ 1u, abort_flag, P.error, 63)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int c = c_begin; c < c_end; ++c) {
                    if (!mbar_wait(&bars->full[st], parity, abort_flag, P.error, 64)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t a = a0 + (uint32_t)(st * (int)(A_BYTES >> 4)), r = r0 + (uint32_t)(st * (int)(B_STAGE >> 4));
                    // Always four: behind the width there are zeros.  (Rolled up, with a count, one such instruction took 54 ns to issue, as long
                    // as the tensor core needs for 200 columns; a stage 0.42 instead of 0.27 us.)
                    umma_i8(d_tmem, a, r, idesc, (uint32_t)(c - c_begin));
                    if (DIGITS == 3) umma_i8(last_tmem, a, r + (B_BYTES >> 4), idesc_last, (uint32_t)(c - c_begin));
                    umma_i8(d_tmem, a + 2, r + 2, idesc, 1u);
                    if (DIGITS == 3) umma_i8(last_tmem, a + 2, r + (B_BYTES >> 4) + 2, idesc_last, 1u);
                    umma_i8(d_tmem, a + 4, r + 4, idesc, 1u);
                    if (DIGITS == 3) umma_i8(last_tmem, a + 4, r + (B_BYTES >> 4) + 4, idesc_last, 1u);
                    umma_i8(d_tmem, a + 6, r + 6, idesc, 1u);
                    if (DIGITS == 3) umma_i8(last_tmem, a + 6, r + (B_BYTES >> 4) + 6, idesc_last, 1u);
                    commit_both(&bars->empty[st], leader);
                    if (++st == nst) st = 0, parity ^= 1u;
                }
                if (ok) commit_both(&bars->tfull[b], leader);
            }
            if (*abort_flag) { // nothing of the tensor core's is under way when the blocks leave
                commit_here(&bars->drained);
                mbar_wait(&bars->drained, 0, abort_flag, P.error, 65);
            }
        }
    } else {
        if (codes_first) rows_are_there();
        const int q = warp & 3, turn = (warp - 2) >> 2; // the quarter of the lanes that this warp may read, and which of its two warps it is
        float *mine = scales_smem + (warp - 2) * (MOST_COLS / 2);
        uint32_t *stage = out_smem + (warp - 2) * 16 * STAGE_WORDS;
        T *y = static_cast<T *>(P.y);
        // what the next tile's results are multiplied by, on its way while this one's leave
        constexpr int TURNS = DIGITS == 3 ? 2 : MOST_COLS / 64;
        struct Scales {
            Tile t;
            float rows[TURNS], channel, bias; // of this lane's rows (one in each of the warp's turns) and channel
        };
        auto scales_of = [&](int id) {
            Scales n;
            n.t = tile_at(P, tiles, id, channel_tiles);
#pragma unroll
            for (int i = 0; i < TURNS; ++i) {
                const int r = 64 * i + 32 * turn + lane;
                n.rows[i] = r < n.t.rows ? P.row_scales[n.t.row0 + r] : 0.0f;
            }
            const int channel = n.t.channel0 + half * BM + 32 * q + lane;
            const size_t at = (size_t)n.t.group * P.channels + channel;
            n.channel = channel >= P.channels ? 0.0f : P.channel_scales ? P.channel_scales[at] : 1.0f;
            n.bias = channel < P.channels && P.bias ? P.bias[at] : 0.0f;
            return n;
        };
        uint32_t local = 0;
        Scales next;
        if (first < total) next = scales_of(first);
        for (int id = first; id < total; id += step, ++local) {
            const Tile t = next.t;
            const uint32_t b = twice ? local & 1u : 0u;
            const int channel0 = t.channel0 + half * BM + 32 * q, channel = channel0 + lane, columns = columns_of(t.rows);
            const bool there = channel < P.channels;
            const float channel_scale = next.channel, bias = next.bias;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < TURNS; ++i) mine[32 * i + lane] = next.rows[i];
            __syncwarp();
            if (id + step < total) next = scales_of(id + step);
            if (!__all_sync(~0u, mbar_wait(&bars->tfull[b], (twice ? local >> 1 : local) & 1u, abort_flag, P.error, 66))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem_base + ((uint32_t)(32 * q) << 16) + b * MOST_COLS;
            if (SPLIT) { // this part's sums to the ring, a channel's next to each other
                uint32_t *dump = reinterpret_cast<uint32_t *>(base);
                for (int c0 = 32 * turn; c0 < DIGITS * columns; c0 += 64) {
                    uint32_t acc[32];
                    tmem_ld32_issue(taddr + c0, acc);
                    tmem_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) dump[(c0 + i) * BM + 32 * q + lane] = acc[i];
                }
                continue;
            }
            // 32 rows' results, from column c0 on, of their sums
            auto leave = [&](int c0, auto sum_of) {
                const float4 *row_scales = reinterpret_cast<const float4 *>(mine + c0 / 2 - 16 * turn);
                const int left = t.rows - c0;
                auto value = [&](int i) {
                    const float4 s4 = row_scales[i >> 2];
                    const float row_scale = (i & 3) == 0 ? s4.x : (i & 3) == 1 ? s4.y : (i & 3) == 2 ? s4.z : s4.w;
                    return finish_sum(sum_of(i), row_scale, channel_scale, bias);
                };
                if (sizeof(T) == 2 && P.wide) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) stage[i * STAGE_WORDS + lane] = two_values<T>(value(2 * i), value(2 * i + 1));
                    __syncwarp();
                    const int piece = lane & 3, here = P.channels - channel0 - 8 * piece; // 8 channels a lane
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int pair = 8 * i + (lane >> 2);
                        const uint4 u = *reinterpret_cast<const uint4 *>(stage + pair * STAGE_WORDS + 8 * piece), v = *reinterpret_cast<const uint4 *>(stage + pair * STAGE_WORDS + 8 * piece + 4);
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            const uint32_t pick = d ? 0x7632u : 0x5410u;
                            const uint4 w = make_uint4(__byte_perm(u.x, u.y, pick), __byte_perm(u.z, u.w, pick), __byte_perm(v.x, v.y, pick), __byte_perm(v.z, v.w, pick));
                            if (2 * pair + d >= left) continue;
                            T *to = y + (size_t)(t.row0 + c0 + 2 * pair + d) * P.y_ld + channel0 + 8 * piece;
                            if (here >= 8) {
                                *reinterpret_cast<uint4 *>(to) = w;
                            } else {
#pragma unroll
                                for (int k = 0; k < 7; ++k)
                                    if (k < here) reinterpret_cast<unsigned short *>(to)[k] = (unsigned short)((&w.x)[k >> 1] >> (16 * (k & 1)));
                            }
                        }
                    }
                    __syncwarp();
                } else {
                    T *to = y + (size_t)(t.row0 + c0) * P.y_ld + channel;
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (there && i < left) to[(size_t)i * P.y_ld] = from_float<T>(value(i));
                }
            };
            auto has_been_read = [&] {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive_at(in_cta(&bars->tempty[b], leader));
            };
            if (DIGITS == 3) {
                float held[2][32]; // both of the warp's turns, so that the accumulator is free before either leaves
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int c0 = 32 * turn + 64 * k;
                    if (c0 >= columns) break;
                    uint32_t acc[32], last[32];
                    tmem_ld32_issue(taddr + columns + c0, acc);
                    tmem_ld32_issue(taddr + 2 * columns + c0, last);
                    tmem_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) held[k][i] = __fmaf_rn(256.0f, (float)(int)acc[i], (float)(int)last[i]); // (join_digits, in two steps)
                    tmem_ld32_issue(taddr + c0, acc);
                    tmem_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) held[k][i] = __fmaf_rn(65536.0f, (float)(int)acc[i], held[k][i]);
                }
                has_been_read();
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (32 * turn + 64 * k < columns) leave(32 * turn + 64 * k, [&](int i) { return held[k][i]; });
            } else {
                if (32 * turn >= columns) has_been_read(); // (nothing of it is this warp's)
                for (int c0 = 32 * turn; c0 < columns; c0 += 64) {
                    uint32_t acc[32];
                    tmem_ld32_issue(taddr + c0, acc);
                    tmem_wait();
                    if (c0 + 64 >= columns) has_been_read();
                    leave(c0, [&](int i) { return (float)(int)acc[i]; });
                }
            }
        }
        if (P.zero_rest)
            zero_rest<T>(y, P.y_ld, P.channels, P.n, tiles.first[0], tiles.end(P.groups - 1), (size_t)blockIdx.x * (THREADS - 64) + (threadIdx.x - 64),
                         (size_t)gridDim.x * (THREADS - 64));
    }

    __syncwarp();
    if (SPLIT) {
        cluster_sync(); // all parts' sums are there
        const Tile t = tile_at(P, tiles, first, channel_tiles);
        const int columns = columns_of(t.rows), channel = t.channel0 + half * BM + 4 * lane; // a warp a row, four channels a lane
        if (warp >= 2 && channel < P.channels) {
            const size_t at = (size_t)t.group * P.channels + channel;
            const int here = min(4, P.channels - channel);
            float channel_scale[4], bias[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                channel_scale[k] = k < here && P.channel_scales ? P.channel_scales[at + k] : 1.0f;
                bias[k] = k < here && P.bias ? P.bias[at + k] : 0.0f;
            }
            const uint32_t *mine = reinterpret_cast<const uint32_t *>(base) + 4 * lane;
            T *y = static_cast<T *>(P.y) + (size_t)t.row0 * P.y_ld + channel;
#pragma unroll 4
            for (int r = EPILOGUE_WARPS * part + warp - 2; r < t.rows; r += EPILOGUE_WARPS * parts) {
                int4 sums[DIGITS] = {};
                for (int s = 0; s < parts; ++s)
#pragma unroll
                    for (int d = 0; d < DIGITS; ++d) {
                        const int4 v = load_cluster(in_cta(mine + (d * columns + r) * BM, 2 * s + half));
                        sums[d].x += v.x, sums[d].y += v.y, sums[d].z += v.z, sums[d].w += v.w;
                    }
                const float row_scale = P.row_scales[t.row0 + r];
                alignas(16) T out[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float sum = DIGITS == 3 ? join_digits((&sums[0].x)[k], (&sums[DIGITS / 2].x)[k], (&sums[DIGITS - 1].x)[k]) : (float)(&sums[0].x)[k];
                    out[k] = from_float<T>(finish_sum(sum, row_scale, channel_scale[k], bias[k]));
                }
                T *to = y + (size_t)r * P.y_ld;
                if (P.wide && here == 4) {
                    if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(out);
                    else *reinterpret_cast<uint2 *>(to) = *reinterpret_cast<const uint2 *>(out);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k < here) to[k] = out[k];
                }
            }
        }
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync(); // neither CTA's shared memory and barriers are needed any more
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

static_assert(3 * MOST_COLS / 2 * BM * sizeof(int) <= 5 * STAGE_BYTES<3>, "three digits' sums, where the width is parted, lie in the ring");
size_t smem_bytes(size_t groups, size_t ring) { return 1024 + ring + EPILOGUE_WARPS * (MOST_COLS / 2 + 16 * STAGE_WORDS) * 4 + sizeof(Barriers) + RowTiles::bytes(groups); }

template <typename T, int DIGITS>
void product_tc_typed(CudaDevice &dev, const Product &p, const TcParams &P, const CUtensorMap &map_codes, const CUtensorMap &map_rows, const CUtensorMap &map_half, unsigned clusters)
{
    const size_t smem = smem_bytes(p.groups, P.stages * STAGE_BYTES<DIGITS>);
    if (P.parts == 1) {
        allow_shared_memory(dev, product_tc_kernel<T, DIGITS, false>);
        launch_following_clusters(product_tc_kernel<T, DIGITS, false>, dim3(2 * clusters), dim3(THREADS), smem, 2, dev.stream(), map_codes, map_rows, map_half,
                                  P);
    } else {
        allow_shared_memory(dev, product_tc_kernel<T, DIGITS, true>);
        launch_following_clusters(product_tc_kernel<T, DIGITS, true>, dim3(2 * P.parts * clusters), dim3(THREADS), smem, 2 * P.parts, dev.stream(), map_codes,
                                  map_rows, map_half, P);
    }
}

// How many clusters of so many CTAs there is room for at a time (a cluster stays within a part of the GPU whose SMs need not be a multiple of it).
size_t room_for_clusters(CudaDevice &dev, int ctas)
{
    static std::mutex mu;
    static std::map<std::pair<int, int>, int> known;
    std::lock_guard<std::mutex> lk(mu);
    auto found = known.find({dev.device(), ctas});
    if (found == known.end()) {
        auto kernel = product_tc_kernel<float, 1, true>;
        allow_shared_memory(dev, kernel);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(THREADS), cfg.dynamicSmemBytes = smem_bytes(1, MOST_STAGES * STAGE_BYTES<1>);
        cudaLaunchAttribute attr = {};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = ctas, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr, cfg.numAttrs = 1;
        int room = 0;
        if (cudaOccupancyMaxActiveClusters(&room, kernel, &cfg) != cudaSuccess) { // none, then
            cudaGetLastError();
            room = 0;
        }
        found = known.insert({{dev.device(), ctas}, room}).first;
    }
    return (size_t)found->second;
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
    const size_t pairs = (size_t)dev.sm_count() / 2, channel_tiles = (p.channels + 2 * BM - 1) / (2 * BM);
    const size_t a_group = (p.n + p.groups - 1) / p.groups; // rows
    // The tile's rows, and among how many pairs its width is parted: whatever makes the rounds of all SM pairs last the shortest.  Measured, in units of one
    // column's time in one stage (1.15 ns): a stage takes as long as its columns, but 160 and an eighth of them at least (0.20 us at 64 or 128 columns,
    // 0.22 at 160, 0.30 at 256); a tile's change 400; its results leave at 10 a column, behind the next tile's stages or, at the end, behind
    // nothing.  (Three digits have three columns a row; the rule held there: within 10 % of the best height for ten of twelve sizes, 18 % for 192 to 5184 of 4057 rows.)  Joining parts takes 700 and 52 a column, shared by the pairs (us for 1, 2 and 4 parts: 128 rows of 8192 with 2048 channels 17.4, 13.4, 11.7; 100 of
    // 1024 with 1024 6.3, 7.2, 7.1).
    const size_t chunks = (p.width + KB - 1) / KB;
    size_t least = ~size_t(0);
    P.parts = 1;
    const size_t most_rows = p.digits == 3 ? MOST_COLS / 2 : MOST_COLS;
    for (size_t rows = 32; rows <= most_rows; rows += 32) {
        const size_t columns = rows * p.digits, a_stage = std::max(columns, 160 + columns / 8), tiles = p.groups * ((a_group + rows - 1) / rows) * channel_tiles;
        const size_t stages = chunks * a_stage + 400, leaves = 10 * rows;
        const size_t cost = (tiles + pairs - 1) / pairs * std::max(stages, leaves) + leaves;
        if (cost < least) P.tile_rows = (int)rows, P.parts = 1, least = cost;
        for (size_t parts = 2; parts <= 4 && !p.offsets && parts <= chunks && tiles * parts <= pairs; parts *= 2) {
            const size_t split = (chunks + parts - 1) / parts * a_stage + 400 + 700 + 52 * columns / parts;
            if (split < least && tiles <= room_for_clusters(dev, (int)(2 * parts))) P.tile_rows = (int)rows, P.parts = (int)parts, least = split;
        }
    }
    P.wide = (reinterpret_cast<uintptr_t>(p.y) | (p.y_ld * 2)) % 16 == 0;
    P.band = 8;
    const CUtensorMap map_codes = make_tensor_map_2d<int8_t>(p.codes, p.width, p.groups * p.channels, KB, BM, CU_TENSOR_MAP_SWIZZLE_128B, codes_ld(p.width));
    // a box: half a tile of one digit's rows; with three digits a whole one of each CTA's and half of the last one's
    auto rows_map = [&](int rows) {
        return make_tensor_map<int8_t>(p.rows, p.width, p.n, KB, (unsigned)rows, CU_TENSOR_MAP_SWIZZLE_128B, p.rows_ld, (unsigned)p.digits, p.n * p.rows_ld);
    };
    const CUtensorMap map_half = rows_map(P.tile_rows / 2), map_rows = p.digits == 3 ? rows_map(P.tile_rows) : map_half;
    P.stages = p.digits == 1 ? MOST_STAGES : smem_bytes(p.groups, 5 * STAGE_BYTES<3>) <= dev.smem_limit() ? 5 : 4;
    const size_t row_tiles = p.offsets ? p.n / P.tile_rows + p.groups : (p.n + P.tile_rows - 1) / P.tile_rows;
    const unsigned clusters = (unsigned)(P.parts > 1 ? row_tiles * channel_tiles : std::min<size_t>(pairs, row_tiles * channel_tiles));
    KernelScope ks(dev, "product_tc");
    if (p.digits == 3) { // (gradients are 16-bit)
        if (p.y_type == VALUE_F16) product_tc_typed<__half, 3>(dev, p, P, map_codes, map_rows, map_half, clusters);
        else product_tc_typed<__nv_bfloat16, 3>(dev, p, P, map_codes, map_rows, map_half, clusters);
    } else if (p.y_type == VALUE_F32) product_tc_typed<float, 1>(dev, p, P, map_codes, map_rows, map_half, clusters);
    else if (p.y_type == VALUE_F16) product_tc_typed<__half, 1>(dev, p, P, map_codes, map_rows, map_half, clusters);
    else product_tc_typed<__nv_bfloat16, 1>(dev, p, P, map_codes, map_rows, map_half, clusters);
    dev.count_launch();
}

} // namespace vqb
