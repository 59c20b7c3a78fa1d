// attend_many.cu -- attention of many rows of a sequence (prompts) over a cache of 8-bit codes, on the tensor cores (tcgen05, kind::f16).
//
// Rows that share a cached head (query heads of a token, then those of the next one) are taken 256 at a time (128 for heads of more than 128 values), over one page of 64 tokens
// a step.  The codes become f16 numbers on their way into shared memory; scores and sums of values are in tensor memory, and so are the weights between the two products.
//
//   warp 0          issues the products: for each half of the rows weights times values of a step, then queries times keys of the step after the next one, so that the next
//                   scores are there when a half's weights are done.  (With 128 tokens a step and room for one step's scores, each half waited for its products after every
//                   step: 8192 tokens x 32 heads x 128 took 1.05 ms.)
//   warp 1          finds what the block takes next, and tells the others ahead of time
//   warp 2          fetches pages' codes (bulk copies)
//   warps 4 .. 7    codes of a page's keys, or values, to operand tiles (128-byte rows, 128-byte swizzle).  (With the codes on their way to registers instead, the fence between
//                   these stores and the products waited for them, a memory's latency every half step.)
//   warps 8 .. 15   four for each half of the rows, a row a thread: scores to weights, largest score and sum; queries in, results out.  They take most of the registers
//                   (setmaxnreg: 2 x 96 + 2 x 160 a thread of each four warps, of 4 x 128)
//
// The floor is the tensor cores' rate (4 x width operations for each row and token); the exponentials, 16 an SM and cycle, take nearly as long.  What bounds it is neither: a step of 256 rows
// of 128 takes some 2600 cycles, the tensor core 1280 of them (alone) and the exponentials 1024.  Two warps a scheduler make weights, each of them a chain of waits, loads, exponentials
// and stores (2048 tokens behind 6144, 32 heads on 8: issue slots 54 %, tensor cores 35 to 44 %, the exponentials' unit 36 %).
// Widths above 128 have one half, whose products and weights cannot take turns: 8192 tokens, 16 heads on 4 of 128 values in 400 us, of 160 in 831, of 256 in 1016 (687, 414 and 541 TFLOP/s).
//
// The largest score that weights are relative to stays as it is until a row has one 2^8 times as large; then the row's sums in tensor memory are brought down, once the product
// that adds to them is done.  Weights are up to 2^8 until then, and f16 numbers all the same.
//
// Blocks share out all tiles' steps as those of attend_few.cu do their pages.
#include <algorithm>

#include "attend.cuh"
#include "cuda_device.hpp"
#include "kernels_common.cuh"
#include "rows.cuh"
#include "umma.cuh"

namespace vqb {

namespace {

constexpr int THREADS = 512, STEP = CACHE_PAGE; // tokens of a step
constexpr float LATE = 8.0f;                    // a row's largest is followed when it is 2^LATE times as large
constexpr int CONVERTERS = 4;                   // warps

template <int PADDED> struct ManyShape {
    static constexpr int HALVES = PADDED <= 128 ? 2 : 1, ROWS = 128 * HALVES;
    static constexpr int BLOCKS = (PADDED + 63) / 64;       // of 64 dimensions: a swizzled row of an operand tile
    static constexpr uint32_t QUERIES = BLOCKS * 128 * 128; // bytes of one half's queries
    static constexpr uint32_t STAGE = BLOCKS * STEP * 128;  // of a page's keys; of its values (PADDED rows of 128 bytes) as much or less
    static constexpr int STAGES = PADDED <= 128 ? 6 : 3;
    static constexpr uint32_t CODES = STEP * PADDED; // bytes of a page's keys, or values
    static constexpr int CODE_STAGES = PADDED <= 128 ? 4 : 2;
    static constexpr size_t SMEM = HALVES * QUERIES + STAGES * STAGE + CODE_STAGES * CODES + 1024;
    static constexpr uint32_t SUMS = 256; // columns of tensor memory: half h's scores of step i from 128 h + 64 (i % 2), sums from 256 + 128 h
};

struct alignas(8) ManyBarriers {
    unsigned long long full[6], empty[6], codes_full[4], codes_empty[4], queries[2], scores[2][2], weights[2][2], added[2], sums[2], told[2], heard[2];
    uint32_t tmem_base;
    int abort_flag;
    int missing[4]; // codes that are not there
};

// kind::f16, binary16 operands, f32 sums, both K-major, M = 128, N = n
__host__ __device__ constexpr uint32_t idesc_f16(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }

template <uint32_t IDESC> __device__ __forceinline__ void umma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "n"(IDESC),
                 "r"(accumulate)
                 : "memory");
}
template <uint32_t IDESC> __device__ __forceinline__ void umma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "n"(IDESC),
                 "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A part of a tile that the block takes, as one warp tells the others ahead of time.  (Aligned to be copied 16 bytes at a time: a prompt of 16,384 tokens through a window of 1024 takes 455 us,
// and 463 without.)
struct alignas(16) Work {
    int row, rows, p0, p1, keys;    // first row of the sequence, rows, positions of the first and last, tokens
    int first_row, head, b;         // as of Tile
    int sink_pages, begin, pages;   // as of Pages
    int from, steps;                // first page (of the tile's list), steps; -1: there are no more parts
    int begins, whole;              // the share begins here; the tile is all here
    // page i of this part, -1 where there is none
    __device__ __forceinline__ int column(int i) const { return from + i < sink_pages ? from + i : begin + from + i - sink_pages; }
    __device__ __forceinline__ int page(const Attend &a, int i) const { return from + i < pages ? page_of(a.seq, a.cache.pages, b, column(i)) : -1; }
};
struct WorkRoom {
    Work work[2];
};

// The parts of the block's share, one after the other, as a role hears of them.
struct Listener {
    const WorkRoom &room;
    ManyBarriers &bars;
    int *error;
    uint32_t number = 0;
    // by a whole warp; false: there are no more
    __device__ __forceinline__ bool next(Work &work)
    {
        const uint32_t at = number & 1u;
        if (!__all_sync(~0u, mbar_wait(&bars.told[at], (number >> 1) & 1u, &bars.abort_flag, error, 110))) return false;
        work = room.work[at];
        __syncwarp();
        if (threadIdx.x % 32 == 0) mbar_arrive(&bars.heard[at]);
        ++number;
        return work.steps >= 0;
    }
};

// The order in which a part's codes are multiplied: keys 0, keys 1, values 0, keys 2, values 1, .. values steps - 1; the n-th one of 2 x steps.
struct HalfStep {
    int step, which; // 0: keys, 1: values
    __device__ __forceinline__ HalfStep(int n, int steps)
    {
        which = n > 0 && (n % 2 == 0 || n == 2 * steps - 1);
        step = n == 0 ? 0 : which == 0 ? (n + 1) / 2 : n == 2 * steps - 1 ? steps - 1 : n / 2 - 1;
    }
};

template <int PADDED>
__device__ __forceinline__ void tell_parts(const ShareParams &P, const Plan<ManyShape<PADDED>::ROWS, THREADS> &plan, ManyBarriers &bars, WorkRoom &room, long long start, long long end)
{
    constexpr int ROWS = ManyShape<PADDED>::ROWS;
    const int lane = threadIdx.x % 32;
    const Attend &a = P.a;
    long long x = start;
    for (uint32_t number = 0;; ++number) {
        const uint32_t at = number & 1u;
        Work work = {};
        Tile<ROWS> tile;
        work.steps = -1;
        if (x < end && plan.find(x, tile)) {
            const Span span(a.seq, tile.b);
            work.rows = min(span.count * a.group - tile.first_row, ROWS);
            work.row = span.row, work.keys = span.keys, work.first_row = tile.first_row, work.head = tile.head, work.b = tile.b;
            work.p0 = span.first + tile.first_row / a.group, work.p1 = span.first + (tile.first_row + work.rows - 1) / a.group;
            const Pages pages(work.p0, work.p1, work.keys, a.window, a.sinks);
            work.sink_pages = pages.sink_pages, work.begin = pages.begin, work.pages = pages.count;
            // the first P.extra units stand for what a tile takes beside its steps
            const int first = (int)(x - tile.begin), behind = (int)(min(end, tile.begin + tile.units) - tile.begin);
            work.from = 2 * max(first - P.extra, 0);
            work.steps = max(min(2 * max(behind - P.extra, 0), pages.count) - work.from, 0);
            work.begins = x == start, work.whole = first == 0 && behind == tile.units;
            if (x == start && lane == 0) plan.tell(&tile, span.row, work.rows);
            x = tile.begin + behind;
        }
        if (!__all_sync(~0u, mbar_wait(&bars.heard[at], ((number >> 1) & 1u) ^ 1u, &bars.abort_flag, P.error, 111))) return;
        if (lane == 0) {
            room.work[at] = work;
            mbar_arrive(&bars.told[at]);
        }
        if (work.steps < 0) return;
    }
}

template <int PADDED> __device__ __forceinline__ void fetch_codes(const ShareParams &P, ManyBarriers &bars, const WorkRoom &room, uint8_t *codes)
{
    using Shape = ManyShape<PADDED>;
    const int lane = threadIdx.x % 32;
    const Attend &a = P.a;
    int slot = 0;
    uint32_t parity = 0;
    Listener listener{room, bars, P.error};
    for (Work work; listener.next(work);) {
        // the pages of 32 steps, and the 32 behind them, a lane each
        int look_now = work.page(a, lane), look_next = work.steps > 32 ? work.page(a, 32 + lane) : -1, looked = 0;
#pragma unroll 1
        for (int n = 0; n < 2 * work.steps; ++n) {
            const HalfStep half(n, work.steps);
            if (half.which == 1 && half.step - looked == 32) { // (everything before has been asked for)
                looked += 32, look_now = look_next;
                look_next = work.page(a, looked + 32 + lane);
            }
            const int page = __shfl_sync(~0u, half.step - looked >= 32 ? look_next : look_now, half.step % 32);
            if (!__all_sync(~0u, mbar_wait(&bars.codes_empty[slot], parity ^ 1u, &bars.abort_flag, P.error, 112))) return;
            if (lane == 0) {
                bars.missing[slot] = page < 0;
                if (page >= 0) {
                    mbar_expect_tx(&bars.codes_full[slot], Shape::CODES);
                    bulk_load_1d(codes + slot * Shape::CODES, a.cache.codes + (((size_t)page * a.cache.heads + work.head) * 2 + half.which) * Shape::CODES, Shape::CODES, &bars.codes_full[slot]);
                } else {
                    mbar_arrive(&bars.codes_full[slot]);
                }
            }
            if (++slot == Shape::CODE_STAGES) slot = 0, parity ^= 1u;
        }
    }
}

template <int N> __host__ __device__ constexpr int power_above() { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : 32; }

// The 32 rows of queries of a warp to their places in the operand tile, 0 behind their width; their factors of scores to `down`.  Lanes next to
// each other have eight values of a row each.  Factors are not negative: the largest product is the largest score.
template <int PADDED> struct Bringer {
    static constexpr int LANES = power_above<PADDED / 8>(), ROWS_AT_ONCE = 32 / LANES; // lanes of a row
    const Attend &a;
    const Work &work;
    const int r0, tile_row; // first of the warp's rows, of the tile and of its half
    uint8_t *tile;
    float *down;
    const int token0, head0; // of the tile's first row
    const float inverse;     // 1 / group: numbers of rows are small enough for that
    const int lane, piece, d, width;
    const bool f16;
    __device__ __forceinline__ Bringer(const Attend &a_, const Work &work_, int r0_, uint8_t *tile_, int tile_row_, float *down_)
        : a(a_), work(work_), r0(r0_), tile_row(tile_row_), tile(tile_), down(down_), token0(work_.first_row / a_.group), head0(work_.first_row % a_.group), inverse(1.0f / (float)a_.group),
          lane(threadIdx.x % 32), piece(lane % LANES), d(8 * piece), width((int)a_.cache.width), f16(a_.queries.type == VALUE_F16)
    {
    }
    __device__ __forceinline__ const uint16_t *row_at(int i) const // (of rows behind the tile's: its last one)
    {
        const int x = head0 + min(r0 + i * ROWS_AT_ONCE + lane / LANES, work.rows - 1), t = (int)(((float)x + 0.5f) * inverse);
        return static_cast<const uint16_t *>(a.queries.x) + (size_t)(work.row + token0 + t) * a.queries.ld + (size_t)(work.head * a.group + x - t * a.group) * a.queries.head_ld;
    }
    // Rows i0 .. of the warp's turns.  All rows' steps next to each other: one row's take a thousand cycles.
    template <int N> __device__ __forceinline__ void convert(int i0, uint4 (&w)[N]) const
    {
        uint32_t most[N]; // magnitudes' order is that of their bits in either type
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (d + 8 > width) { // 0 behind the width
#pragma unroll
                for (int j = 0; j < 4; ++j) (&w[i].x)[j] &= (d + 2 * j < width ? 0xFFFFu : 0u) | (d + 2 * j + 1 < width ? 0xFFFF0000u : 0u);
            }
            most[i] = __vmaxu2(__vmaxu2(w[i].x & 0x7FFF7FFFu, w[i].y & 0x7FFF7FFFu), __vmaxu2(w[i].z & 0x7FFF7FFFu, w[i].w & 0x7FFF7FFFu));
        }
#pragma unroll
        for (int o = LANES / 2; o; o /= 2)
#pragma unroll
            for (int i = 0; i < N; ++i) most[i] = __vmaxu2(most[i], __shfl_xor_sync(~0u, most[i], o));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = (i0 + i) * ROWS_AT_ONCE + lane / LANES; // of the warp's
            const uint32_t half = max(most[i] & 0xFFFFu, most[i] >> 16);
            const QueryScale scale(f16 ? __float_as_uint(__half2float(__ushort_as_half((unsigned short)half))) : half << 16, fabsf(a.scale));
            const float up = a.scale < 0.0f ? -scale.up : scale.up;
            uint4 h;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t two = (&w[i].x)[j];
                const float low = f16 ? __half2float(__ushort_as_half((unsigned short)(two & 0xFFFFu))) : __uint_as_float(two << 16);
                const float high = f16 ? __half2float(__ushort_as_half((unsigned short)(two >> 16))) : __uint_as_float(two & 0xFFFF0000u);
                (&h.x)[j] = scale.up == 0.0f ? 0u : halves_of_floats(low * up, high * up); // (an infinity or a NaN: 0 times that is none)
            }
            if (d < PADDED) *reinterpret_cast<uint4 *>(tile + d / 64 * 16384 + (tile_row + r) * 128 + ((piece % 8) ^ (r & 7)) * 16) = h;
            if (piece == 0) down[tile_row + r] = scale.down;
        }
    }
    __device__ __forceinline__ void all() const
    {
        if (width % 8 == 0 && a.queries.ld % 8 == 0 && a.queries.head_ld % 8 == 0 && (reinterpret_cast<uintptr_t>(a.queries.x) & 15) == 0) {
            constexpr int N = 4;
#pragma unroll 1
            for (int i = 0; i < LANES; i += N) {
                uint4 w[N];
#pragma unroll
                for (int k = 0; k < N; ++k) w[k] = *reinterpret_cast<const uint4 *>(row_at(i + k) + min(d, width - 8));
                convert<N>(i, w);
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < LANES; ++i) {
                const uint16_t *x = row_at(i);
                uint4 w[1] = {make_uint4(0, 0, 0, 0)};
#pragma unroll
                for (int j = 0; j < 8; ++j) (&w[0].x)[j / 2] |= (uint32_t)x[min(d + j, width - 1)] << (16 * (j % 2));
                convert<1>(i, w);
            }
        }
    }
};

// Bits of a page's tokens that a row sees.
__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
__device__ __forceinline__ uint64_t seen_bits(int column, int position, int keys, int window, int sinks)
{
    const int first = column * CACHE_PAGE;
    uint64_t bits = bits_below(min(position + 1, keys) - first);
    if (window) bits &= ~(bits_below(max(max(position, 0) - window + 1, 0) - first) & ~bits_below(min(sinks, keys) - first));
    return position < 0 ? 0 : bits;
}

template <int PADDED>
__device__ __forceinline__ void issue_products(const ShareParams &P, ManyBarriers &bars, const WorkRoom &room, uint8_t *queries, uint8_t *ring, uint32_t tmem)
{
    using Shape = ManyShape<PADDED>;
    constexpr int STAGES = Shape::STAGES;
    volatile int *abort_flag = &bars.abort_flag;
    const bool leader = elect_one(); // the one lane that knows the following
    int st = 0;
    uint32_t parity = 0, weights_parity[2] = {0, 0}, queries_parity[2] = {0, 0}; // parity: of the ring's round; bit b of weights_parity[h]: of the next weights in buffer b
    bool ok = true;
    Listener listener{room, bars, P.error};
    for (Work work; listener.next(work);) {
        if (work.steps == 0) continue;
        const int halves = work.rows > 128 ? 2 : 1;
        if (leader) {
            auto next_stage = [&] {
                if (++st == STAGES) st = 0, parity ^= 1u;
            };
            auto stage_there = [&] { return mbar_wait(&bars.full[st], parity, abort_flag, P.error, 101); };
            auto keys_times = [&](int h, int buffer) {
                const uint64_t q = smem_desc_sw128(smem_u32(queries + h * Shape::QUERIES)), k = smem_desc_sw128(smem_u32(ring + st * Shape::STAGE));
                const uint32_t to = tmem + 128 * h + 64 * buffer;
#pragma unroll
                for (int i = 0; i < PADDED / 16; ++i) umma_smem<idesc_f16(STEP)>(to, q + (i / 4) * 1024 + (i % 4) * 2, k + (i / 4) * (STEP * 128 / 16) + (i % 4) * 2, i > 0);
                umma_commit(&bars.scores[h][buffer]);
            };
            auto values_times = [&](int h, int buffer, bool add) {
                const uint64_t v = smem_desc_sw128(smem_u32(ring + st * Shape::STAGE));
                const uint32_t from = tmem + 128 * h + 64 * buffer;
#pragma unroll
                for (int k = 0; k < STEP / 16; ++k) umma_tmem<idesc_f16(PADDED)>(tmem + Shape::SUMS + 128 * h, from + 8 * k, v + k * 2, add || k > 0);
                umma_commit(&bars.added[h]);
            };
            // the first two steps' scores
#pragma unroll 1
            for (int i = 0; ok && i < min(work.steps, 2); ++i) {
                ok = stage_there();
#pragma unroll 1
                for (int h = 0; ok && h < halves; ++h) {
                    if (i == 0) {
                        ok = mbar_wait(&bars.queries[h], queries_parity[h], abort_flag, P.error, 102);
                        queries_parity[h] ^= 1u;
                        if (!ok) break;
                    }
                    tmem_after();
                    keys_times(h, i);
                }
                if (ok) umma_commit(&bars.empty[st]);
                next_stage();
            }
#pragma unroll 1
            for (int i = 0; ok && i < work.steps; ++i) {
                const int buffer = i & 1, values_at = st;
                const bool more = i + 2 < work.steps;
                ok = stage_there();
                if (ok && more) { // (the keys are behind the values in the ring)
                    next_stage();
                    ok = stage_there();
                    if (--st < 0) st = STAGES - 1, parity ^= 1u;
                }
#pragma unroll 1
                for (int h = 0; ok && h < halves; ++h) {
                    ok = mbar_wait(&bars.weights[h][buffer], weights_parity[h] >> buffer & 1u, abort_flag, P.error, 103);
                    if (!ok) break;
                    weights_parity[h] ^= 1u << buffer;
                    tmem_after();
                    values_times(h, buffer, i > 0);
                    if (i + 1 == work.steps) umma_commit(&bars.sums[h]);
                    // (instructions of one thread run in the order they were issued: the scores do not overtake the weights that they take the place of)
                    if (more) {
                        next_stage();
                        keys_times(h, buffer);
                        if (--st < 0) st = STAGES - 1, parity ^= 1u;
                    }
                }
                if (!ok) break;
                umma_commit(&bars.empty[values_at]);
                next_stage();
                if (more) {
                    umma_commit(&bars.empty[st]);
                    next_stage();
                }
            }
        }
        if (!__all_sync(~0u, ok)) break;
    }
    if (leader && ok) // the tensor core's arrivals have come before the block leaves
        for (int j = 0; j < STAGES; ++j) mbar_wait(&bars.empty[j], j < st ? parity : parity ^ 1u, abort_flag, P.error, 109);
    __syncwarp();
}

template <int PADDED>
__device__ __forceinline__ void convert_codes(const ShareParams &P, ManyBarriers &bars, const WorkRoom &room, const uint8_t *codes, uint8_t *ring)
{
    using Shape = ManyShape<PADDED>;
    constexpr int STAGES = Shape::STAGES;
    const int lane = threadIdx.x % 32;
    volatile int *abort_flag = &bars.abort_flag;
    const int t = threadIdx.x - 128; // of the converters' threads
    constexpr int THREADS_HERE = 32 * CONVERTERS, ALL = STEP * PADDED / 16, PIECES = (ALL + THREADS_HERE - 1) / THREADS_HERE; // pieces of 16 codes of a page, and a thread's
    constexpr int PER_ROW = PADDED / 16;                                                                                     // of a token's key
    int st = 0, slot = 0;
    uint32_t parity = 0, codes_parity = 0;
    bool ok = true;
    Listener listener{room, bars, P.error};
    for (Work work; ok && listener.next(work);) {
#pragma unroll 1
        for (int n = 0; n < 2 * work.steps; ++n) {
            const int which = HalfStep(n, work.steps).which;
            if (!(ok = __all_sync(~0u, mbar_wait(&bars.codes_full[slot], codes_parity, abort_flag, P.error, 105)))) break;
            uint4 piece[PIECES];
            if (bars.missing[slot]) {
#pragma unroll
                for (int k = 0; k < PIECES; ++k) piece[k] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
            } else {
#pragma unroll
                for (int k = 0; k < PIECES; ++k)
                    if (ALL % THREADS_HERE == 0 || t + THREADS_HERE * k < ALL) piece[k] = reinterpret_cast<const uint4 *>(codes + slot * Shape::CODES)[t + THREADS_HERE * k];
            }
            if (!(ok = __all_sync(~0u, mbar_wait(&bars.empty[st], parity ^ 1u, abort_flag, P.error, 106)))) break;
            uint8_t *to = ring + st * Shape::STAGE;
#pragma unroll
            for (int k = 0; k < PIECES; ++k) {
                const int at = t + THREADS_HERE * k;
                if (ALL % THREADS_HERE && at >= ALL) continue;
                int row, chunk; // of 128 bytes; the first of two pieces of 16 bytes
                uint8_t *part = to;
                bool turned = false; // second piece first: lanes that write at once find different banks
                if (which == 0) {
                    row = at / PER_ROW; // token
                    int p = at % PER_ROW;
                    if (PADDED % 128 == 0) p ^= (row & 1) * 4;
                    part += p / 4 * (STEP * 128), chunk = 2 * (p % 4), turned = p / 4 % 2;
                } else {
                    row = at / 4, chunk = 2 * (at % 4); // dimension
                }
                uint4 first, second;
                codes_to_halves(piece[k].x, first.x, first.y);
                codes_to_halves(piece[k].y, first.z, first.w);
                codes_to_halves(piece[k].z, second.x, second.y);
                codes_to_halves(piece[k].w, second.z, second.w);
                uint8_t *at_row = part + row * 128;
                *reinterpret_cast<uint4 *>(at_row + ((chunk + turned) ^ (row & 7)) * 16) = turned ? second : first;
                *reinterpret_cast<uint4 *>(at_row + ((chunk + !turned) ^ (row & 7)) * 16) = turned ? first : second;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&bars.full[st]);
                mbar_arrive(&bars.codes_empty[slot]);
            }
            if (++st == STAGES) st = 0, parity ^= 1u;
            if (++slot == Shape::CODE_STAGES) slot = 0, codes_parity ^= 1u;
        }
    }
}

template <int PADDED>
__device__ __forceinline__ void weigh_rows(const ShareParams &P, ManyBarriers &bars, const WorkRoom &room, uint8_t *queries, float *down_room, uint32_t tmem)
{
    using Shape = ManyShape<PADDED>;
    constexpr int ROWS = Shape::ROWS, HALVES = Shape::HALVES;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    volatile int *abort_flag = &bars.abort_flag;
    const Attend &a = P.a;
    const Cache &c = a.cache;
    const int h = (warp - 8) / 4, r = (warp % 4) * 32 + lane; // half, row of it
    const uint32_t lanes = (uint32_t)(warp % 4) << 21, sums = tmem + lanes + Shape::SUMS + 128 * h; // (lane 32 q: bits 16 ..)
    uint32_t scores_parity = 0, added_parity = 0, sums_parity = 0; // scores_parity: bit b of the next scores in buffer b; added_parity: of this step's product
    if (h >= HALVES) return;
    bool ok = true;
    Listener listener{room, bars, P.error};
    for (Work work; ok && listener.next(work);) {
        const int in_tile = 128 * h + r, at = work.first_row + min(in_tile, work.rows - 1);
        const bool there = in_tile < work.rows;
        const int token = at / a.group, position = work.p0 + token - work.first_row / a.group;
        float m = -INFINITY, top = -INFINITY, l = 0.0f;
        const bool taken = work.steps > 0 && 128 * h < work.rows;
        if (taken) {
            // the pages of 32 steps with s_k and log2(s_v) (-infinity: values of 0), a lane each, and the 32 behind them
            auto look = [&](int i, int &page, float2 &scale) {
                page = work.page(a, i + lane);
                scale = page >= 0 ? *reinterpret_cast<const float2 *>(c.scales + ((size_t)page * c.heads + work.head) * 2) : make_float2(0.0f, 0.0f);
                scale.y = log2f(scale.y);
            };
            int page_now, page_next = -1;
            float2 scale_now, scale_next = make_float2(0.0f, 0.0f);
            look(0, page_now, scale_now);
            if (work.steps > 32) look(32, page_next, scale_next);
            Bringer<PADDED>(a, work, 128 * h + warp % 4 * 32, queries + h * Shape::QUERIES, warp % 4 * 32, down_room + 128 * h).all();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tmem_before(); // (the last tile's sums have been read)
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.queries[h]);
            const float down = down_room[in_tile];
            uint32_t v[2][32]; // a step's scores; the next ones are on their way to where weights have been made of these
            auto scores_there = [&](int i) {
                const uint32_t buffer = i & 1;
                ok = __all_sync(~0u, mbar_wait(&bars.scores[h][buffer], scores_parity >> buffer & 1u, abort_flag, P.error, 107));
                scores_parity ^= 1u << buffer;
                tmem_after();
                return ok;
            };
            if (!scores_there(0)) break;
            tmem_ld32_issue(tmem + lanes + 128 * h, v[0]);
            tmem_ld32_issue(tmem + lanes + 128 * h + 32, v[1]);
            for (int i = 0; i < work.steps; ++i) {
                const uint32_t buffer = i & 1, scores = tmem + lanes + 128 * h + 64 * buffer, scores_next = tmem + lanes + 128 * h + 64 * (buffer ^ 1);
                const bool more = i + 1 < work.steps;
                const int column = work.column(i);
                const bool is_there = __shfl_sync(~0u, page_now, i % 32) >= 0;
                const float factor = score_factor(down, __shfl_sync(~0u, scale_now.x, i % 32));
                const float log_v = __shfl_sync(~0u, scale_now.y, i % 32);
                uint64_t bits = is_there ? ~0ull : 0;
                if (is_there && !all_seen(column, work.p0, work.p1, work.keys, a.window, a.sinks)) bits = seen_bits(column, position, work.keys, a.window, a.sinks);
                const bool masked = __any_sync(~0u, bits != ~0ull);
                if (i % 32 == 31) {
                    page_now = page_next, scale_now = scale_next;
                    look(i + 33, page_next, scale_next);
                }
                tmem_wait();
                if (masked) {
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (!((uint32_t)(bits >> (32 * q)) >> j & 1u)) v[q][j] = 0xFF800000u;
                }
                float most[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) most[e] = fmaxf(__uint_as_float(v[e / 2][e % 2 * 16]), __uint_as_float(v[e / 2][e % 2 * 16 + 1]));
#pragma unroll
                for (int j = 2; j < 16; j += 2)
#pragma unroll
                    for (int e = 0; e < 4; ++e) most[e] = max3f(most[e], __uint_as_float(v[e / 2][e % 2 * 16 + j]), __uint_as_float(v[e / 2][e % 2 * 16 + j + 1]));
                const float raw = fmaxf(max3f(most[0], most[1], most[2]), most[3]), higher_m = raw == -INFINITY ? raw : raw * factor;
                const float higher_top = higher_m + (log_v == log_v ? log_v : 0.0f);
                const bool rise = higher_top > top + LATE;
                if (__any_sync(~0u, rise || higher_m > m + LATE)) {
                    if (higher_m > m + LATE) l *= relative(m, higher_m), m = higher_m;
                    const float by = rise ? relative(top, higher_top) : 1.0f;
                    if (rise) top = higher_top;
                    if (i > 0) {
                        // the last step's product; the one before it is done (these scores came behind it), so that its turn is not taken for this one
                        if (!__all_sync(~0u, mbar_wait(&bars.added[h], added_parity ^ 1u, abort_flag, P.error, 104))) {
                            ok = false;
                            break;
                        }
                        tmem_after();
#pragma unroll 1
                        for (int d = 0; d < PADDED; d += 16) {
                            uint32_t y[16];
                            tmem_ld16_issue(sums + d, y);
                            tmem_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * by);
                            tmem_st16(sums + d, y);
                        }
                    }
                }
                added_parity ^= 1u;
                const float from_m = m == -INFINITY ? 0.0f : m, from_top = top == -INFINITY ? 0.0f : top;
                const float shift = log_v + from_m - from_top, plus = log_v - from_top; // a weight is 2^(s - m) 2^shift (values of 0: shift is -infinity, weights are 0)
                // (a factor of 0 or NaN, or NaN for s_v, would make NaN of what is hidden)
                if (__any_sync(~0u, fabsf(shift) > 60.0f || (masked && !(factor > 0.0f && shift == shift)))) {
#pragma unroll 1
                    for (int q = 0; q < 4; ++q) {
                        uint32_t some[16], out[8];
                        tmem_ld16_issue(scores + 16 * q, some);
                        tmem_wait();
                        const uint32_t shown = (uint32_t)(bits >> (16 * q));
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float w[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float s = __uint_as_float(some[j + e]);
                                w[e] = shown >> (j + e) & 1u ? power_of_two(fmaf(s, factor, plus)) : 0.0f;
                                l += shown >> (j + e) & 1u ? power_of_two(fmaf(s, factor, -from_m)) : 0.0f; // (either may be 0 where the other is not)
                            }
                            out[j / 2] = halves_of_floats(w[0], w[1]);
                        }
                        tmem_st8(scores + 8 * q, out);
                    }
                    if (more) {
                        if (!scores_there(i + 1)) break;
                        tmem_ld32_issue(scores_next, v[0]);
                        tmem_ld32_issue(scores_next + 32, v[1]);
                    }
                } else {
                    const uint64_t by = pair_of(factor, factor), and_plus = pair_of(plus, plus);
                    uint64_t sum[2] = {0, 0};
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t out[16];
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            float w0, w1;
                            halves_of(fma_pair(pair_of(__uint_as_float(v[q][j]), __uint_as_float(v[q][j + 1])), by, and_plus), w0, w1);
                            w0 = power_of_two(w0), w1 = power_of_two(w1);
                            sum[j / 2 % 2] = add_pair(sum[j / 2 % 2], pair_of(w0, w1));
                            out[j / 2] = halves_of_floats(w0, w1);
                        }
                        tmem_st16(scores + 16 * q, out);
                        if (more) {
                            if (q == 0 && !scores_there(i + 1)) break;
                            tmem_ld32_issue(scores_next + 32 * q, v[q]);
                        }
                    }
                    if (!ok) break;
                    float a0, a1;
                    halves_of(add_pair(sum[0], sum[1]), a0, a1);
                    l += (a0 + a1) * exp2f(-shift);
                }
                tmem_stored();
                tmem_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.weights[h][buffer]);
            }
            if (!ok) break;
            if (!__all_sync(~0u, mbar_wait(&bars.sums[h], sums_parity, abort_flag, P.error, 108))) {
                ok = false;
                break;
            }
            sums_parity ^= 1u;
            tmem_after();
        }
        // results
        float *part = work.whole ? nullptr : P.parts + (2 * (size_t)blockIdx.x + !work.begins) * part_floats<ROWS>(PADDED);
        if (part) {
            float *f = part + ROWS * PADDED + in_tile;
            f[0] = m, f[ROWS] = top, f[2 * ROWS] = l;
            if (!taken) continue; // (a part without weight: nobody reads its sums)
        }
        const size_t to = (size_t)(work.row + token) * a.y.ld + (size_t)(work.head * a.group + at % a.group) * a.y.head_ld;
        const RowEnd row_end(m, top, l);
        const bool wide = !part && (reinterpret_cast<uintptr_t>(static_cast<uint16_t *>(a.y.x) + to) & 15) == 0;
#pragma unroll 1
        for (int d = 0; d < PADDED; d += 16) {
            uint32_t v[16];
            __syncwarp();
            if (taken) {
                tmem_ld16_issue(sums + d, v);
                tmem_wait();
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = 0;
            }
            if (!there) continue;
            if (part) {
#pragma unroll
                for (int j = 0; j < 16; j += 4) *reinterpret_cast<uint4 *>(part + (size_t)in_tile * PADDED + d + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                continue;
            }
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y0 = row_end.of(__uint_as_float(v[2 * j])), y1 = row_end.of(__uint_as_float(v[2 * j + 1]));
                const __nv_bfloat162 b = __floats2bfloat162_rn(y0, y1);
                o[j] = a.y.type == VALUE_F16 ? halves_of_floats(y0, y1) : *reinterpret_cast<const uint32_t *>(&b);
            }
            uint16_t *y = static_cast<uint16_t *>(a.y.x) + to + d;
            if (wide && d + 16 <= (int)c.width) {
                *reinterpret_cast<uint4 *>(y) = make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4 *>(y + 8) = make_uint4(o[4], o[5], o[6], o[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (d + j < (int)c.width) y[j] = (uint16_t)(o[j / 2] >> (16 * (j % 2)));
            }
        }
    }
}

template <int PADDED> __global__ void __launch_bounds__(THREADS, 1) attend_many_kernel(const __grid_constant__ ShareParams P)
{
    using Shape = ManyShape<PADDED>;
    constexpr int ROWS = Shape::ROWS, HALVES = Shape::HALVES;
    extern __shared__ unsigned char smem_raw[];
    __shared__ typename Plan<ROWS, THREADS>::Room room;
    __shared__ ManyBarriers bars;
    __shared__ WorkRoom work_room;
    __shared__ float down_room[ROWS];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *queries = base, *ring = base + HALVES * Shape::QUERIES, *codes = ring + Shape::STAGES * Shape::STAGE;
    const int warp = threadIdx.x / 32;
    volatile int *abort_flag = &bars.abort_flag;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 6; ++i) mbar_init(&bars.full[i], CONVERTERS), mbar_init(&bars.empty[i], 1);
        for (int i = 0; i < 4; ++i) mbar_init(&bars.codes_full[i], 1), mbar_init(&bars.codes_empty[i], CONVERTERS);
        for (int h = 0; h < 2; ++h) {
            mbar_init(&bars.queries[h], 4), mbar_init(&bars.added[h], 1), mbar_init(&bars.sums[h], 1);
            for (int i = 0; i < 2; ++i) mbar_init(&bars.scores[h][i], 1), mbar_init(&bars.weights[h][i], 4);
        }
        for (int i = 0; i < 2; ++i) mbar_init(&bars.told[i], 1), mbar_init(&bars.heard[i], 2 + CONVERTERS + 4 * HALVES);
        bars.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    cache_is_there();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // (attend_join_kernel of the same call)
    tmem_before();
    const Plan<ROWS, THREADS> plan(P, room); // (block barriers)
    tmem_after();
    const uint32_t tmem = bars.tmem_base;
    const long long start = plan.share * blockIdx.x, end = min(start + plan.share, plan.total);

    if (start >= end && threadIdx.x == 0) plan.tell(nullptr, 0, 0);

    // (each in its role's own branch: the compiler counts a role's registers from there)
    if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (warp == 0) issue_products<PADDED>(P, bars, work_room, queries, ring, tmem);
        else if (warp == 1) tell_parts<PADDED>(P, plan, bars, work_room, start, end);
        else if (warp == 2) fetch_codes<PADDED>(P, bars, work_room, codes);
        else if (warp >= 4) convert_codes<PADDED>(P, bars, work_room, codes, ring);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;");
        weigh_rows<PADDED>(P, bars, work_room, queries, down_room, tmem);
    }
    tmem_before();
    __syncthreads();
    if (*abort_flag) // what the tensor cores have been given is done before the block leaves
        for (int w = 0; w < 1000; ++w) __nanosleep(1000);
    if (warp == 0) {
        tmem_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int PADDED> void attend_many_with(CudaDevice &dev, ShareParams &P, const Attend &a)
{
    constexpr int ROWS = ManyShape<PADDED>::ROWS;
    P.slots = (int)slots_of<ROWS>(a);
    size_t pages = std::max(a.seq.columns, 1); // of a tile at most
    if (a.window) pages = std::min(pages, ((size_t)a.sinks + 63) / 64 + ((size_t)a.window + ROWS + 62) / CACHE_PAGE + 1);
    const size_t steps = (pages + 1) / 2;
    const bool join = steps > 1;
    const size_t places = dev.sm_count(), tiles = (size_t)P.slots * a.cache.heads;
    P.unit = 2, P.extra = join && tiles > places ? 4 : 0; // (what a tile takes beside its steps, in units; where nothing is joined a tile is one unit, which no share's end cuts)
    P.blocks = (int)std::min(tiles * (steps + P.extra), places);
    Parts parts(dev);
    if (join) parts.make<ROWS>(P, PADDED);
    allow_shared_memory(dev, attend_many_kernel<PADDED>);
    {
        KernelScope ks(dev, "attend_many");
        launch_following(attend_many_kernel<PADDED>, dim3((unsigned)P.blocks), dim3(THREADS), ManyShape<PADDED>::SMEM, dev.stream(), P);
        dev.count_launch();
    }
    launch_join<PADDED, ROWS>(dev, P);
}

} // namespace

void launch_attend_many(CudaDevice &dev, const Attend &a)
{
    ShareParams P{};
    P.a = a, P.error = dev.error_word(), P.least = ATTEND_FEW, P.most = 0x7FFFFFFF;
    switch (a.cache.padded / 32) {
    case 1: return attend_many_with<32>(dev, P, a);
    case 2: return attend_many_with<64>(dev, P, a);
    case 3: return attend_many_with<96>(dev, P, a);
    case 4: return attend_many_with<128>(dev, P, a);
    case 5: return attend_many_with<160>(dev, P, a);
    case 6: return attend_many_with<192>(dev, P, a);
    case 7: return attend_many_with<224>(dev, P, a);
    default: return attend_many_with<256>(dev, P, a);
    }
}

} // namespace vqb
