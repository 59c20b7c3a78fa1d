// attend_many.cu -- attention of many rows of a sequence (prompts) over a cache of 8-bit codes, on the tensor cores (tcgen05, kind::f16).
//
// Rows that share a cached head (query heads of a token, then those of the next one) are taken 256 at a time (128 for heads of more than 128 values), over 128 tokens, two pages,
// a step.  The codes become f16 numbers on their way into shared memory; scores and sums of values are in tensor memory, and so are the weights between the two products.
//
//   warp 1               issues the products: for each half of the rows weights times values of a step, then the next step's queries times keys, so that one half's
//                        products run while the other half's scores become weights
//   warps 2, 3, 12, 13   codes of a step's keys, then of its values, to operand tiles (128-byte rows, 128-byte swizzle); the next ones are on their way from memory meanwhile
//   warps 4 .. 7, 8 .. 11  a half of the rows each, a row a thread: scores to weights, largest score and sum; queries in, results out
//
// What bounds it is the tensor cores' rate (4 x width operations for each row and token) and, as much, the exponentials: 16 an SM and cycle.
//
// The largest score that weights are relative to stays as it is until a row has one 2^8 times as large; then the row's sums in tensor memory, which nobody
// is adding to at that time, are brought down.  Weights are up to 2^8 until then, and f16 numbers all the same.
//
// Blocks share out all tiles' steps as those of attend_few.cu do their pages.
#include <algorithm>

#include "attend.cuh"
#include "cuda_device.hpp"
#include "umma.cuh"

namespace vqb {

namespace {

constexpr int THREADS = 448, STEP = 2 * CACHE_PAGE; // tokens of a step
constexpr float LATE = 8.0f;                        // a row's largest is followed when it is 2^LATE times as large

template <int PADDED> struct ManyShape {
    static constexpr int HALVES = PADDED <= 128 ? 2 : 1, ROWS = 128 * HALVES;
    static constexpr int BLOCKS = (PADDED + 63) / 64;             // of 64 dimensions: a swizzled row of an operand tile
    static constexpr uint32_t QUERIES = BLOCKS * 128 * 128;       // bytes of one half's queries
    static constexpr uint32_t STAGE = BLOCKS * 128 * 128;         // of a step's keys; of its values (2 x PADDED rows of 128 bytes) as much or less
    static constexpr int STAGES = PADDED <= 128 ? 4 : 2;
    static constexpr size_t SMEM = HALVES * QUERIES + STAGES * STAGE + 1024;
    static constexpr uint32_t SCORES = 128, SUMS = 256; // columns of tensor memory: half h's scores from 128 h, sums from 256 + 128 h
};

struct alignas(8) ManyBarriers {
    unsigned long long full[4], empty[4], queries[2], scores[2], weights[2], sums[2];
    uint32_t tmem_base;
    int abort_flag;
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
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, "
                 "%27, %28, %29, %30, %31, %32};" ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
                 "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
                 "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// What all roles know of the part of a tile that the block takes next.
template <int ROWS> struct Work {
    Tile<ROWS> tile;
    int row, rows, p0, p1, keys; // first row of the call, rows, positions of the first and last, tokens
    int from, steps;             // first page (of the tile's list), steps
    int behind;                  // units
    bool begins, whole;          // the share begins here; the tile is all here
    Pages pages;
    __device__ __forceinline__ Work(const ShareParams &P, const Plan<ROWS, THREADS> &plan, long long x, long long start, long long end, bool &ok) : pages(0, 0, 0, 0, 0)
    {
        ok = plan.find(x, tile);
        if (!ok) return;
        const Attend &a = P.a;
        const Span span(a.seq, tile.b);
        rows = min(span.count * a.group - tile.first_row, ROWS);
        row = span.row, keys = span.keys;
        p0 = span.first + tile.first_row / a.group, p1 = span.first + (tile.first_row + rows - 1) / a.group;
        pages = Pages(p0, p1, keys, a.window, a.sinks);
        const int first = (int)(x - tile.begin);
        behind = (int)(min(end, tile.begin + tile.units) - tile.begin);
        from = first * 2;
        steps = (max(min(behind * 2, pages.count) - from, 0) + 1) / 2;
        begins = x == start, whole = first == 0 && behind == tile.units;
    }
    // page i of this part, -1 where there is none
    __device__ __forceinline__ int page(const Attend &a, int i) const { return from + i < pages.count ? page_of(a.seq, a.cache.pages, tile.b, pages.column(from + i)) : -1; }
};

// A row of queries to its place in the operand tile, 0 behind its width; its factor of scores.
template <int PADDED> __device__ __forceinline__ float bring_row(const Attend &a, const void *from, bool there, uint8_t *tile, int r)
{
    const uint16_t *x = static_cast<const uint16_t *>(from);
    const int width = (int)a.cache.width;
    const bool f16 = a.queries.type == VALUE_F16, aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    auto eight = [&](int d) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (there && aligned && d + 8 <= width) {
            w = *reinterpret_cast<const uint4 *>(x + d);
        } else if (there) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (d + j < width) (&w.x)[j / 2] |= (uint32_t)x[d + j] << (16 * (j % 2));
        }
        return w;
    };
    auto value = [&](const uint4 &w, int j) {
        const uint32_t half = j % 2 ? (&w.x)[j / 2] >> 16 : (&w.x)[j / 2] & 0xFFFFu;
        return f16 ? __half2float(__ushort_as_half((unsigned short)half)) : __uint_as_float(half << 16);
    };
    uint32_t most = 0;
#pragma unroll 4
    for (int d = 0; d < PADDED; d += 8) {
        const uint4 w = eight(d);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(value(w, j)) & 0x7FFFFFFFu);
    }
    const QueryScale scale(most, fabsf(a.scale));
    const float up = a.scale < 0.0f ? -scale.up : scale.up; // (factors of scores are not negative: the largest product is the largest score)
#pragma unroll 4
    for (int d = 0; d < PADDED; d += 8) {
        const uint4 w = eight(d);
        uint4 h = make_uint4(0, 0, 0, 0);
        if (scale.up != 0.0f) {
#pragma unroll
            for (int j = 0; j < 4; ++j) (&h.x)[j] = halves_of_floats(value(w, 2 * j) * up, value(w, 2 * j + 1) * up);
        }
        *reinterpret_cast<uint4 *>(tile + d / 64 * 16384 + r * 128 + ((d / 8 % 8) ^ (r & 7)) * 16) = h;
    }
    return scale.down;
}

// Bits of a page's tokens that a row sees.
__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
__device__ __forceinline__ uint64_t seen_bits(int column, int position, int keys, int window, int sinks)
{
    const int first = column * CACHE_PAGE;
    uint64_t bits = bits_below(min(position + 1, keys) - first);
    if (window) bits &= ~(bits_below(max(position - window + 1, 0) - first) & ~bits_below(min(sinks, keys) - first));
    return position < 0 ? 0 : bits;
}

template <int PADDED> __global__ void __launch_bounds__(THREADS, 1) attend_many_kernel(const __grid_constant__ ShareParams P)
{
    using Shape = ManyShape<PADDED>;
    constexpr int ROWS = Shape::ROWS, HALVES = Shape::HALVES, STAGES = Shape::STAGES;
    extern __shared__ unsigned char smem_raw[];
    __shared__ typename Plan<ROWS, THREADS>::Room room;
    __shared__ ManyBarriers bars;
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *queries = base, *ring = base + HALVES * Shape::QUERIES;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    volatile int *abort_flag = &bars.abort_flag;
    const Attend &a = P.a;
    const Cache &c = a.cache;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 4; ++i) mbar_init(&bars.full[i], 4), mbar_init(&bars.empty[i], 1);
        for (int h = 0; h < 2; ++h) mbar_init(&bars.queries[h], 4), mbar_init(&bars.scores[h], 1), mbar_init(&bars.weights[h], 4), mbar_init(&bars.sums[h], 1);
        bars.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
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

    if (warp == 1) {
        const bool leader = elect_one(); // the one lane that knows the following
        int st = 0;
        uint32_t parity = 0, weights_parity[2] = {0, 0}, queries_parity[2] = {0, 0}; // parity: of the ring's round
        bool ok = true;
        for (long long x = start; x < end;) {
            bool found;
            const Work<ROWS> work(P, plan, x, start, end, found);
            if (!found) break;
            x = work.tile.begin + work.behind;
            if (work.steps == 0) continue;
            const int halves = work.rows > 128 ? 2 : 1;
            if (leader) {
                auto keys_times = [&](int h) {
                    const uint64_t q = smem_desc_sw128(smem_u32(queries + h * Shape::QUERIES)), k = smem_desc_sw128(smem_u32(ring + st * Shape::STAGE));
#pragma unroll
                    for (int i = 0; i < PADDED / 16; ++i)
                        umma_smem<idesc_f16(STEP)>(tmem + Shape::SCORES * h, q + (i / 4) * 1024 + (i % 4) * 2, k + (i / 4) * 1024 + (i % 4) * 2, i > 0);
                    umma_commit(&bars.scores[h]);
                };
                auto next_stage = [&] {
                    if (++st == STAGES) st = 0, parity ^= 1u;
                };
                ok = mbar_wait(&bars.full[st], parity, abort_flag, P.error, 101);
                for (int h = 0; ok && h < halves; ++h) {
                    ok = mbar_wait(&bars.queries[h], queries_parity[h], abort_flag, P.error, 102);
                    queries_parity[h] ^= 1u;
                    tmem_after();
                    if (ok) keys_times(h);
                }
                if (ok) umma_commit(&bars.empty[st]);
                next_stage();
                for (int i = 0; ok && i < work.steps; ++i) {
                    const bool more = i + 1 < work.steps;
                    const int values_at = st;
                    ok = mbar_wait(&bars.full[st], parity, abort_flag, P.error, 103);
                    next_stage();
                    if (ok && more) ok = mbar_wait(&bars.full[st], parity, abort_flag, P.error, 104);
                    for (int h = 0; ok && h < halves; ++h) {
                        ok = mbar_wait(&bars.weights[h], weights_parity[h], abort_flag, P.error, 105);
                        if (!ok) break;
                        weights_parity[h] ^= 1u;
                        tmem_after();
                        const uint64_t v = smem_desc_sw128(smem_u32(ring + values_at * Shape::STAGE));
#pragma unroll
                        for (int k = 0; k < STEP / 16; ++k)
                            umma_tmem<idesc_f16(PADDED)>(tmem + Shape::SUMS + 128 * h, tmem + Shape::SCORES * h + 8 * k, v + (k / 4) * (PADDED * 128 / 16) + (k % 4) * 2, i + k > 0);
                        // (instructions of one thread run in the order they were issued: the next scores do not overtake the weights that they take the place of)
                        if (more) keys_times(h);
                        else umma_commit(&bars.sums[h]);
                    }
                    if (!ok) break;
                    umma_commit(&bars.empty[values_at]);
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
    } else if (warp == 2 || warp == 3 || warp >= 12) {
        // codes to operand tiles
        const int t = (warp < 4 ? warp - 2 : warp - 10) * 32 + lane; // of 128
        constexpr int PIECES = STEP * PADDED / 16 / 128, PER_ROW = PADDED / 16; // of 16 codes; a thread's, and those of a token's key
        int st = 0;
        uint32_t parity = 0;
        bool ok = true;
        constexpr int DEPTH = PADDED <= 128 ? 2 : 1; // half steps whose codes are on their way
        uint4 piece[DEPTH][PIECES];
        const uint4 zeros = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        for (long long x = start; ok && x < end;) {
            const Work<ROWS> work(P, plan, x, start, end, ok);
            if (!ok) break;
            x = work.tile.begin + work.behind;
            if (work.steps == 0) continue;
            int now[2] = {work.page(a, 0), work.page(a, 1)}, next[2] = {work.page(a, 2), work.page(a, 3)}; // of this step and the next one
            auto load = [&](uint4 (&to)[PIECES], const int (&pages)[2], int which) {
#pragma unroll
                for (int k = 0; k < PIECES; ++k) {
                    const int at = t + 128 * k, half = at / (STEP * PADDED / 32); // (pieces of a page: 64 PADDED / 16)
                    const int page = half ? pages[1] : pages[0];
                    to[k] = page < 0 ? zeros
                                     : *reinterpret_cast<const uint4 *>(c.codes + (((size_t)page * c.heads + work.tile.head) * 2 + which) * CACHE_PAGE * PADDED +
                                                                        (size_t)(at - half * (STEP * PADDED / 32)) * 16);
                }
            };
            load(piece[0], now, 0);
            if (DEPTH == 2) load(piece[DEPTH - 1], now, 1);
            for (int i = 0; ok && i < work.steps; ++i) {
#pragma unroll
                for (int which = 0; which < 2; ++which) { // keys, values
                    if (!__all_sync(~0u, mbar_wait(&bars.empty[st], parity ^ 1u, abort_flag, P.error, 106))) {
                        ok = false;
                        break;
                    }
                    uint4(&mine)[PIECES] = piece[which % DEPTH];
                    uint8_t *to = ring + st * Shape::STAGE;
#pragma unroll
                    for (int k = 0; k < PIECES; ++k) {
                        const int at = t + 128 * k;
                        int row, chunk; // of 128 bytes; the first of two pieces of 16 bytes
                        uint8_t *part = to;
                        bool turned = false; // second piece first: lanes that write at once find different banks
                        if (which == 0) {
                            row = at / PER_ROW; // token of the step
                            int p = at % PER_ROW;
                            if (PADDED % 128 == 0) p ^= (row & 1) * 4;
                            part += p / 4 * 16384, chunk = 2 * (p % 4), turned = p / 4 % 2;
                        } else {
                            row = at / 4, chunk = 2 * (at % 4); // dimension; the second page's behind the first one's
                        }
                        uint4 first, second;
                        codes_to_halves(mine[k].x, first.x, first.y);
                        codes_to_halves(mine[k].y, first.z, first.w);
                        codes_to_halves(mine[k].z, second.x, second.y);
                        codes_to_halves(mine[k].w, second.z, second.w);
                        uint8_t *at_row = part + row * 128;
                        *reinterpret_cast<uint4 *>(at_row + ((chunk + turned) ^ (row & 7)) * 16) = turned ? second : first;
                        *reinterpret_cast<uint4 *>(at_row + ((chunk + !turned) ^ (row & 7)) * 16) = turned ? first : second;
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.full[st]);
                    if (++st == STAGES) st = 0, parity ^= 1u;
                    if (DEPTH == 2) {
                        if (i + 1 < work.steps) load(mine, next, which);
                    } else if (which == 0) {
                        load(mine, now, 1);
                    } else if (i + 1 < work.steps) {
                        load(mine, next, 0);
                    }
                }
                now[0] = next[0], now[1] = next[1];
                next[0] = work.page(a, 2 * i + 4), next[1] = work.page(a, 2 * i + 5);
            }
        }
    } else if (warp >= 4) {
        const int h = (warp - 4) / 4, r = (warp % 4) * 32 + lane; // half, row of it
        const uint32_t lanes = (uint32_t)(warp % 4) << 21, scores = tmem + lanes + Shape::SCORES * h, sums = tmem + lanes + Shape::SUMS + 128 * h; // (lane 32 q: bits 16 ..)
        uint32_t step_parity = 0, sums_parity = 0;
        bool ok = h < HALVES;
        for (long long x = start; ok && x < end;) {
            const Work<ROWS> work(P, plan, x, start, end, ok);
            if (!ok) break;
            x = work.tile.begin + work.behind;
            const int in_tile = 128 * h + r, at = work.tile.first_row + min(in_tile, work.rows - 1);
            const bool there = in_tile < work.rows;
            const int token = at / a.group, head = work.tile.head * a.group + at % a.group, position = work.p0 + token - work.tile.first_row / a.group;
            const size_t row = (size_t)(work.row + token);
            float m = -INFINITY, top = -INFINITY, l = 0.0f;
            const bool taken = work.steps > 0 && 128 * h < work.rows;
            if (taken) {
                const uint16_t *q = static_cast<const uint16_t *>(a.queries.x) + row * a.queries.ld + (size_t)head * a.queries.head_ld;
                const float down = bring_row<PADDED>(a, q, there, queries + h * Shape::QUERIES, r);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tmem_before(); // (the last tile's sums have been read)
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.queries[h]);
                auto scales_of = [&](int page) {
                    return page < 0 ? make_float2(0.0f, 0.0f) : *reinterpret_cast<const float2 *>(c.scales + ((size_t)page * c.heads + work.tile.head) * 2);
                };
                int page[2] = {work.page(a, 0), work.page(a, 1)}, page_next[2] = {work.page(a, 2), work.page(a, 3)};
                float2 scale[2] = {scales_of(page[0]), scales_of(page[1])}, scale_next[2];
                for (int i = 0; i < work.steps; ++i) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) scale_next[k] = scales_of(page_next[k]);
                    uint64_t bits[2];
                    bool masked = false;
                    float factor[2], log_v[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int number = work.from + 2 * i + k, column = number < work.pages.count ? work.pages.column(number) : 0;
                        bits[k] = page[k] < 0 ? 0 : ~0ull;
                        if (page[k] >= 0 && !all_seen(column, work.p0, work.p1, work.keys, a.window, a.sinks)) bits[k] = seen_bits(column, position, work.keys, a.window, a.sinks);
                        masked |= bits[k] != ~0ull;
                        factor[k] = score_factor(down, scale[k].x);
                        log_v[k] = log2f(scale[k].y); // (-infinity: values of 0)
                    }
                    masked = __any_sync(~0u, masked);
                    if (!__all_sync(~0u, mbar_wait(&bars.scores[h], step_parity, abort_flag, P.error, 107))) {
                        ok = false;
                        break;
                    }
                    step_parity ^= 1u;
                    tmem_after();
                    // the largest score
                    float higher_m = -INFINITY, higher_top = -INFINITY;
                    uint32_t v[2][32];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        tmem_ld32_issue(scores + 64 * k, v[0]);
                        tmem_ld32_issue(scores + 64 * k + 32, v[1]);
                        tmem_wait();
                        if (masked) {
#pragma unroll
                            for (int j = 0; j < 64; ++j)
                                if (!(bits[k] >> j & 1)) v[j / 32][j % 32] = 0xFF800000u;
                        }
                        float most[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) most[e] = __uint_as_float(v[e / 2][e % 2 * 16]);
#pragma unroll
                        for (int j = 1; j < 15; j += 2)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int from = e % 2 * 16 + j;
                                most[e] = fmaxf(fmaxf(most[e], __uint_as_float(v[e / 2][from])), __uint_as_float(v[e / 2][from + 1]));
                            }
#pragma unroll
                        for (int e = 0; e < 4; ++e) most[e] = fmaxf(most[e], __uint_as_float(v[e / 2][e % 2 * 16 + 15]));
                        const float raw = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])), s = raw == -INFINITY ? raw : raw * factor[k];
                        higher_m = fmaxf(higher_m, s);
                        if (scale[k].y != 0.0f) higher_top = fmaxf(higher_top, s + (scale[k].y == scale[k].y ? log_v[k] : 0.0f));
                    }
                    if (higher_m > m + LATE || (m == -INFINITY && higher_m > m)) l *= relative(m, higher_m), m = higher_m;
                    const bool rise = higher_top > top + LATE || (top == -INFINITY && higher_top > top);
                    if (__any_sync(~0u, rise)) {
                        const float by = rise ? relative(top, higher_top) : 1.0f;
                        if (rise) top = higher_top;
                        if (i > 0) { // (the products that add to the sums are done: this step's scores came behind them)
#pragma unroll 1
                            for (int d = 0; d < PADDED; d += 32) {
                                tmem_ld32_issue(sums + d, v[0]);
                                tmem_wait();
#pragma unroll
                                for (int j = 0; j < 32; ++j) v[0][j] = __float_as_uint(__uint_as_float(v[0][j]) * by);
                                tmem_st32(sums + d, v[0]);
                            }
                        }
                    }
                    const float from_m = m == -INFINITY ? 0.0f : m, from_top = top == -INFINITY ? 0.0f : top;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (scale[k].y == 0.0f) log_v[k] = from_top - from_m;
                        const float shift = log_v[k] + from_m - from_top; // a weight is 2^(s - m) 2^shift
                        const bool far = __any_sync(~0u, fabsf(shift) > 60.0f);
                        const float plus = log_v[k] - from_top;
                        float sum[4] = {};
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            tmem_ld32_issue(scores + 64 * k + 32 * q, v[q]);
                            tmem_wait();
                            uint32_t out[16];
                            const uint32_t some = (uint32_t)(bits[k] >> (32 * q));
#pragma unroll
                            for (int j = 0; j < 32; j += 2) {
                                float w[2];
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    float s = __uint_as_float(v[q][j + e]);
                                    float y = fmaf(s, factor[k], plus);
                                    const bool hidden = masked && !(some >> (j + e) & 1);
                                    if (hidden) y = -INFINITY;
                                    w[e] = power_of_two(y);
                                    if (far) sum[j / 2 % 4] += hidden ? 0.0f : power_of_two(fmaf(s, factor[k], -from_m)); // (either may be 0 where the other is not)
                                    else sum[j / 2 % 4] += w[e];
                                }
                                out[j / 2] = halves_of_floats(w[0], w[1]);
                            }
                            tmem_st16(scores + 32 * k + 16 * q, out);
                        }
                        const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                        if (all != 0.0f) l += far ? all : all * exp2f(-shift);
                    }
                    tmem_stored();
                    tmem_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.weights[h]);
#pragma unroll
                    for (int k = 0; k < 2; ++k) page[k] = page_next[k], scale[k] = scale_next[k], page_next[k] = work.page(a, 2 * i + 4 + k);
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
            float *part = work.whole ? nullptr : plan.part(blockIdx.x, work.begins, PADDED);
            if (part) {
                float *f = part + ROWS * PADDED + in_tile;
                f[0] = m, f[ROWS] = top, f[2 * ROWS] = l;
            }
            const size_t to = row * a.y.ld + (size_t)head * a.y.head_ld;
            const RowEnd row_end(m, top, l);
            const bool wide = !part && (reinterpret_cast<uintptr_t>(static_cast<uint16_t *>(a.y.x) + to) & 15) == 0;
#pragma unroll 1
            for (int d = 0; d < PADDED; d += 32) {
                uint32_t v[32];
                __syncwarp();
                if (taken) {
                    tmem_ld32_issue(sums + d, v);
                    tmem_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0;
                }
                if (!there) continue;
                if (part) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4 *>(part + (size_t)in_tile * PADDED + d + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = row_end.of(__uint_as_float(v[j + e]));
                        if (wide && d + j + 8 <= (int)c.width) {
                            uint4 o;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if (a.y.type == VALUE_F16) {
                                    (&o.x)[e] = halves_of_floats(y[2 * e], y[2 * e + 1]);
                                } else {
                                    const __nv_bfloat162 b = __floats2bfloat162_rn(y[2 * e], y[2 * e + 1]);
                                    (&o.x)[e] = *reinterpret_cast<const uint32_t *>(&b);
                                }
                            }
                            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.y.x) + to + d + j) = o;
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (d + j + e < (int)c.width) put_value(a.y, to + d + j + e, y[e]);
                        }
                    }
                }
            }
        }
    }
    tmem_before();
    __syncthreads();
    if (*abort_flag) // what the tensor cores have been given is done before the block leaves
        for (int w = 0; w < 1000; ++w) __nanosleep(1000);
    if (warp == 1) {
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
    P.unit = 2;
    P.blocks = (int)std::min((size_t)P.slots * a.cache.heads * steps, (size_t)dev.sm_count());
    struct Parts {
        CudaDevice &dev;
        void *p;
        ~Parts() { dev.release(p); }
    } parts{dev, join ? dev.alloc(2 * (size_t)P.blocks * part_floats<ROWS>(PADDED) * sizeof(float)) : nullptr};
    P.parts = static_cast<float *>(parts.p);
    allow_shared_memory(dev, attend_many_kernel<PADDED>);
    {
        KernelScope ks(dev, "attend_many");
        launch_following(attend_many_kernel<PADDED>, dim3((unsigned)P.blocks), dim3(THREADS), ManyShape<PADDED>::SMEM, dev.stream(), P);
        dev.count_launch();
    }
    if (!join) return;
    KernelScope ks(dev, "attend_join");
    launch_following(attend_join_kernel<PADDED, ROWS>, dim3((unsigned)std::min(P.blocks * ROWS / 4, 8 * dev.sm_count())), dim3(128), 0, dev.stream(), P);
    dev.count_launch();
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
