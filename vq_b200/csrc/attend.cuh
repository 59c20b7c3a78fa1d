// attend.cuh -- what the attention kernels on tensor cores share.
//
// Scores are in powers of two: s = S log2(e).  The weights of the values are e^(S - m) s_v; they are held as 2^(s + log2(s_v) - M), M the largest s + log2(s_v) of the
// row so far (not of s: pages whose s_v are far apart would lose the weights that count), f16 numbers for the product with the codes.  M is followed when it is left behind by
// 2^8: weights are up to 2^8 until then.  Values of scale 0 have weights of 0, whatever their codes.  The sum below the line is 2^(s - m) with the row's largest s (followed
// likewise), in f32.  y = (sum of weights times codes) / (sum) 2^(M - m).
//
// Queries are f16 numbers: each row times the power of two that brings its largest magnitude to 2^14 .. 2^15.  f16 and bf16 values are those numbers exactly, but for those
// below 2^-28 of the row's largest, which are off by at most 2^-39 of it.
#pragma once
#include "cache.cuh"
#include "cuda_device.hpp"

namespace vqb {

constexpr float LOG2_E = 1.44269504088896341f;

// 2^x, x <= 0 or NaN (what is below 2^-126 is 0)
__device__ __forceinline__ float power_of_two(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two largest numbers so far, from a to b: what is relative to a times this is relative to b (nothing is relative to -infinity)
__device__ __forceinline__ float relative(float a, float b) { return a == -INFINITY ? 0.0f : power_of_two(a - b); }

// Four bytes of the cache as f16 numbers: 1024 + byte is the f16 number 0x6400 | byte, 1152 less is the code.
__device__ __forceinline__ void codes_to_halves(uint32_t four, uint32_t &low, uint32_t &high)
{
    const uint32_t exponent = 0x64646464u, minus = 0xE480E480u; // -1152 twice
    low = __byte_perm(four, exponent, 0x4140), high = __byte_perm(four, exponent, 0x4342);
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(low) : "r"(minus));
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(high) : "r"(minus));
}
__device__ __forceinline__ uint32_t halves_of_floats(float a, float b)
{
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(a), "f"(b));
    return d;
}

// What a row of queries with this largest magnitude (its bits) is multiplied by, and what its products with codes are multiplied by for the score (but for s_k).
struct QueryScale {
    float up, down;
    __device__ __forceinline__ QueryScale(uint32_t largest, float scale)
    {
        const int exponent = (int)(largest >> 23) - 127, k = min(14 - exponent, 126); // (f32 numbers below 2^-112 stay below 2^14: 2^126 is enough for bf16's smallest)
        const float factor = scale * LOG2_E;
        up = __int_as_float((k + 127) << 23);
        down = factor * __int_as_float((127 - k) << 23); // (-113 <= k <= 126)
        if (largest == 0) up = 1.0f, down = factor;
        if (largest >= 0x7F800000u) up = 0.0f, down = __int_as_float(0x7FC00000);
    }
};

// down s_k: what a row's products with a page's codes are multiplied by.  (Infinite only where any score but 0 is: 0 times that is to stay 0.)
__device__ __forceinline__ float score_factor(float down, float k)
{
    const float t = down * k;
    return fabsf(t) == INFINITY ? copysignf(3.4e38f, t) : t;
}

// The pages that rows at positions p0 .. p1 of a sequence see some of: the first sink_pages of its table, then those from column `begin` on.
struct Pages {
    int sink_pages, begin, count;
    __device__ __forceinline__ Pages(int p0, int p1, int keys, int window, int sinks)
    {
        const int last = min(p1, keys - 1), last_page = last < 0 ? -1 : last >> 6; // (column of the last token)
        begin = window ? max(max(p0, 0) - window + 1, 0) >> 6 : 0;
        sink_pages = min(min((int)(((unsigned)sinks + 63u) >> 6), begin), last_page + 1);
        count = sink_pages + max(last_page - begin + 1, 0);
    }
    __device__ __forceinline__ int column(int i) const { return i < sink_pages ? i : begin + i - sink_pages; }
};

// Whether all rows at positions p0 .. p1 see all of the tokens of a column.
__device__ __forceinline__ bool all_seen(int column, int p0, int p1, int keys, int window, int sinks)
{
    const int first = column * CACHE_PAGE, last = first + CACHE_PAGE - 1;
    return last <= p0 && last < keys && (!window || first > p1 - window || last < sinks);
}
__device__ __forceinline__ bool seen(int token, int position, int keys, int window, int sinks)
{
    return token <= position && token < keys && (!window || token > position - window || token < sinks);
}

// What a kernel that shares tiles out is given.
struct ShareParams {
    Attend a;
    int least, most; // rows (counting query heads) of the sequences that it takes: above least, at most `most`
    int slots;       // numbers of tiles (slots_of)
    int blocks;      // that share the pages
    int unit;        // pages that are not shared out
    int extra;       // units that a tile counts for beside its pages
    float *parts;    // 2 x blocks parts; null where no share's end cuts a tile
    struct Cut *cuts; // what each block's begin cuts
    int *error;
};

// A tile that the end of a share, in front of a block, cuts, if it is the first such end: the tile has parts in blocks first .. last.
struct Cut {
    int row, rows;       // first row of the sequence, rows of the tile (0: nothing is cut here first)
    int first_row, head; // as of Tile
    int first, last;
    int begins; // the tile begins with the first block's share
};

// A part of a tile: ROWS x padded sums, and ROWS each of m, M and the sum below the line.
template <int ROWS> __host__ __device__ constexpr size_t part_floats(int padded) { return (size_t)ROWS * (padded + 3); }

// A row's result from the sums of its values' weights times codes, by the figures that these are relative to.  0 for a row that saw nothing (or only values of 0).
struct RowEnd {
    float first, second; // (in two steps: 2^(top - m) may leave f32 where the result does not)
    __device__ __forceinline__ RowEnd(float m, float top, float l)
    {
        second = exp2f(0.5f * (top - m)), first = second / l;
        if (l == 0.0f || (top == -INFINITY && l == l)) first = second = 0.0f;
    }
    __device__ __forceinline__ float of(float sum) const { return sum * first * second; }
};

// Tiles that there may be of all sequences, whatever their rows: sequence b's are numbered from offsets[b] group / ROWS + b on.
template <int ROWS> inline size_t slots_of(const Attend &a)
{
    const size_t rows = (size_t)a.seq.n * a.group, sequences = a.seq.sequences;
    return a.seq.offsets ? rows / ROWS + sequences : sequences * ((rows / sequences + ROWS - 1) / ROWS);
}

// One tile of one head.
template <int ROWS> struct Tile {
    int b, head, first_row; // first_row: of the sequence's rows, counting query heads
    int units;              // numbered for it
    long long begin;        // number of its first unit
};

// Units of all tiles and heads in a row; every block has an equal share of them.  Block barriers: THREADS threads.
template <int ROWS, int THREADS> struct Plan {
    static constexpr int MOST_GROUPS = 512, WARPS = THREADS / 32;
    struct Room {
        long long before[MOST_GROUPS + 1]; // of a group of `per` slots
        long long sums[WARPS];
    };
    const ShareParams &P;
    long long *before;
    int per, groups;
    long long total, share;

    // units of a slot's tile, 0 where it has none
    __device__ __forceinline__ int of_slot(int u, int &b, int &first_row) const
    {
        const Attend &a = P.a;
        if (!a.seq.offsets) {
            const int each = P.slots / a.seq.sequences;
            b = u / each, first_row = (u - b * each) * ROWS;
        } else {
            int lo = 0, hi = a.seq.sequences - 1; // the last one that begins at or before u
#pragma unroll 1
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if ((int)((long long)offset_of(a.seq, mid) * a.group / ROWS) + mid <= u) lo = mid;
                else hi = mid - 1;
            }
            b = lo;
            const int r = u - (int)((long long)offset_of(a.seq, b) * a.group / ROWS) - b;
            if (r < 0) return 0;
            first_row = r * ROWS;
        }
        const Span span(a.seq, b);
        const long long rows = (long long)span.count * a.group;
        if (first_row >= rows || rows <= P.least || rows > P.most) return 0;
        const int last_row = (int)min((long long)first_row + ROWS, rows) - 1;
        const Pages pages(span.first + first_row / a.group, span.first + last_row / a.group, span.keys, a.window, a.sinks);
        return max((pages.count + P.unit - 1) / P.unit, 1) + P.extra; // (at least one: somebody writes its rows)
    }
    // by all threads; ends with a block barrier
    __device__ __forceinline__ Plan(const ShareParams &params, Room &room) : P(params), before(room.before)
    {
        const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
        per = (P.slots + MOST_GROUPS - 1) / MOST_GROUPS, groups = (P.slots + per - 1) / per;
        long long base = 0;
#pragma unroll 1
        for (int g0 = 0; g0 < groups; g0 += THREADS) {
            long long mine = 0;
#pragma unroll 1
            for (int u = (g0 + (int)threadIdx.x) * per; u < min((g0 + (int)threadIdx.x + 1) * per, P.slots); ++u) {
                int b, row;
                mine += of_slot(u, b, row);
            }
            long long up = mine;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const long long other = __shfl_up_sync(~0u, up, d);
                if (lane >= d) up += other;
            }
            if (lane == 31) room.sums[warp] = up;
            __syncthreads();
            long long all = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                if (w < warp) up += room.sums[w];
                all += room.sums[w];
            }
            if (g0 + (int)threadIdx.x < groups) before[g0 + threadIdx.x + 1] = (base + up) * (long long)P.a.cache.heads;
            base += all;
            __syncthreads();
        }
        if (threadIdx.x == 0) before[0] = 0;
        __syncthreads();
        total = before[groups];
        share = max((total + P.blocks - 1) / P.blocks, 1ll);
    }
    // By a whole warp: the tile that unit x (below total) is of.
    __device__ __forceinline__ bool find(long long x, Tile<ROWS> &tile) const
    {
        const int lane = threadIdx.x % 32, heads = (int)P.a.cache.heads;
        int lo = 0, hi = groups - 1;
#pragma unroll 1
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before[mid] <= x) lo = mid;
            else hi = mid - 1;
        }
        long long rest = x - before[lo];
#pragma unroll 1
        for (int u = lo * per, end = min(u + per, P.slots); u < end; u += 32) {
            int b = 0, row = 0;
            const int units = u + lane < end ? of_slot(u + lane, b, row) : 0;
            const long long mine = (long long)units * heads;
            long long up = mine;
            if (per > 1) {
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const long long other = __shfl_up_sync(~0u, up, d);
                    if (lane >= d) up += other;
                }
            }
            const unsigned behind = __ballot_sync(~0u, up > rest);
            if (behind) {
                const int k = __ffs(behind) - 1;
                rest -= __shfl_sync(~0u, up - mine, k);
                tile.units = __shfl_sync(~0u, units, k), tile.b = __shfl_sync(~0u, b, k), tile.first_row = __shfl_sync(~0u, row, k);
                const int i = (int)(rest / tile.units);
                tile.head = i, tile.begin = x - rest + (long long)i * tile.units;
                return true;
            }
            rest -= __shfl_sync(~0u, up, 31);
        }
        return false;
    }
    // The part that a block's share of a tile leaves: what begins with the share is its first one.
    __device__ __forceinline__ float *part(int block, bool begins_share, int padded) const { return P.parts + (2 * (size_t)block + !begins_share) * part_floats<ROWS>(padded); }
    // The first tile that this block has some of; null: it has none.  By one thread.
    __device__ __forceinline__ void tell(const Tile<ROWS> *tile, int row, int rows) const
    {
        if (!P.parts) return;
        Cut cut = {};
        const long long start = share * blockIdx.x;
        if (tile && tile->begin < start && tile->begin >= start - share)
            cut = Cut{row, rows, tile->first_row, tile->head, (int)blockIdx.x - 1, (int)((tile->begin + tile->units - 1) / share), tile->begin == start - share};
        P.cuts[blockIdx.x] = cut;
    }
};

// The parts of tiles that more than one block had a share of: a warp for each row.
template <int PADDED, int ROWS> __global__ void __launch_bounds__(128) attend_join_kernel(const __grid_constant__ ShareParams P)
{
    cache_is_there();
    const Attend &a = P.a;
    const int lane = threadIdx.x % 32, at = blockIdx.x * 4 + threadIdx.x / 32, r = at % ROWS;
    if (at / ROWS + 1 >= P.blocks) return;
    const Cut cut = P.cuts[at / ROWS + 1];
    if (r >= cut.rows) return;
    const auto part_of = [&](int block) { return P.parts + (2 * (size_t)block + (block == cut.first && !cut.begins)) * part_floats<ROWS>(PADDED); };
    float m = -INFINITY, top = -INFINITY, l = 0.0f;
    float y[PADDED / 32] = {};
    for (int s0 = cut.first; s0 <= cut.last; s0 += 32) { // (usually once)
        const int s = s0 + lane, many = min(cut.last - s0 + 1, 32);
        const float *f = part_of(min(s, cut.last)) + ROWS * PADDED + r;
        const float part_m = s <= cut.last ? f[0] : -INFINITY, part_top = s <= cut.last ? f[ROWS] : -INFINITY, part_l = s <= cut.last ? f[2 * ROWS] : 0.0f;
        float new_m = fmaxf(m, part_m), new_top = fmaxf(top, part_top);
#pragma unroll
        for (int o = 16; o; o /= 2) new_m = fmaxf(new_m, __shfl_xor_sync(~0u, new_m, o)), new_top = fmaxf(new_top, __shfl_xor_sync(~0u, new_top, o));
        float sum = part_l * relative(part_m, new_m);
        const float by = relative(part_top, new_top);
#pragma unroll
        for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(~0u, sum, o);
        l = l * relative(m, new_m) + sum;
        const float old = relative(top, new_top);
#pragma unroll
        for (int d = 0; d < PADDED / 32; ++d) y[d] *= old;
        m = new_m, top = new_top;
#pragma unroll 8
        for (int k = 0; k < many; ++k) {
            const float *part = part_of(s0 + k) + r * PADDED + lane;
            const float w = __shfl_sync(~0u, by, k);
#pragma unroll
            for (int d = 0; d < PADDED / 32; ++d) {
                const float v = part[32 * d];
                y[d] += w != 0.0f ? v * w : 0.0f; // (a part that saw nothing may have no sums)
            }
        }
    }
    const RowEnd row_end(m, top, l);
    const int row = cut.first_row + r;
    const size_t to = (size_t)(cut.row + row / a.group) * a.y.ld + (size_t)(cut.head * a.group + row % a.group) * a.y.head_ld;
#pragma unroll
    for (int d = 0; d < PADDED / 32; ++d)
        if (32 * d + lane < (int)a.cache.width) put_value(a.y, to + 32 * d + lane, row_end.of(y[d]));
}

// Memory for what is left to join, for the time of a call.
struct Parts {
    CudaDevice &dev;
    unsigned char *p = nullptr;
    template <int ROWS> static size_t cuts_at(const ShareParams &P, int padded) { return 2 * (size_t)P.blocks * part_floats<ROWS>(padded) * sizeof(float); }
    explicit Parts(CudaDevice &d) : dev(d) {}
    template <int ROWS> void make(ShareParams &P, int padded)
    {
        p = static_cast<unsigned char *>(dev.alloc(cuts_at<ROWS>(P, padded) + P.blocks * sizeof(Cut)));
        P.parts = reinterpret_cast<float *>(p), P.cuts = reinterpret_cast<Cut *>(p + cuts_at<ROWS>(P, padded));
    }
    ~Parts() { dev.release(p); }
    Parts(const Parts &) = delete;
    Parts &operator=(const Parts &) = delete;
};
template <int PADDED, int ROWS> void launch_join(CudaDevice &dev, const ShareParams &P)
{
    if (!P.parts || P.blocks < 2) return;
    KernelScope ks(dev, "attend_join");
    launch_following(attend_join_kernel<PADDED, ROWS>, dim3((unsigned)(((size_t)(P.blocks - 1) * ROWS + 3) / 4)), dim3(128), 0, dev.stream(), P);
    dev.count_launch();
}

} // namespace vqb
