// attend_few.cu -- attention of a few rows of each sequence (single tokens above all) over a cache of 8-bit codes.
//
// Eight or sixteen rows that share a cached head (query heads of a token, then those of the next one) are a tile.  The floor is the cache's bytes, 2 x 64 x width of them a page and head, read
// once for a tile: of a sequence with 17 to 32 rows twice, by different blocks (16 sequences of up to 8192 tokens, 8 heads x 128: 47 us for one token of eight query heads a cached one, 61 for two, 98 for four;
// the bytes once are 26).  What bounds it is less the bytes (76 % of the copy rate for 64 sequences, 59 % for two of 131,072) than fixed latencies with three warps a scheduler.  Every warp fetches pages for itself (one bulk copy for a page's keys, one for its values) into a ring of its own,
// turns the codes to f16 numbers in registers and multiplies: mma.sync m16n8k16 with sixteen tokens by eight rows, then sixteen dimensions by eight rows.  (The tensor
// cores' larger instructions have 128 rows where there are eight.)  A lane's 16 bytes of a key serve four instructions: which of its dimensions go into
// which is free as long as the queries have the same.  So is which tokens are a score tile's rows; they are chosen so that the tile, transposed (movmatrix), is the operand
// of the product with the values, of which a lane has four tokens side by side.
//
// All tiles' pages are numbered in a row, and each block takes an equal share of that, whatever the sequences' lengths are (nobody on the host knows them).  What
// a share's end cuts off a tile leaves as a part (its largest scores, sum, and sums of values), and a second kernel joins parts, in the order of their pages.
#include <algorithm>

#include "attend.cuh"
#include "cuda_device.hpp"
#include "umma.cuh"

namespace vqb {

namespace {

constexpr int STAGES = 2;
constexpr float LATE = 8.0f; // a row's largest score is followed when it is 2^LATE times as large

__device__ __forceinline__ void mma_f16(float (&sums)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(sums[0]), "+f"(sums[1]), "+f"(sums[2]), "+f"(sums[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}
// 8 x 8 16-bit values, two of a row a lane, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v)
{
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

template <int BYTES> struct Words;
template <> struct Words<16> {
    uint4 v;
    __device__ __forceinline__ uint32_t operator[](int i) const { return (&v.x)[i]; }
};
template <> struct Words<8> {
    uint2 v;
    __device__ __forceinline__ uint32_t operator[](int i) const { return (&v.x)[i]; }
};
template <int BYTES> __device__ __forceinline__ Words<BYTES> words_at(const uint8_t *p) { return *reinterpret_cast<const Words<BYTES> *>(p); }

// EIGHTS: of rows a tile has; WARPS: of a block
template <int PADDED, int EIGHTS, int WARPS> struct FewShape {
    static constexpr int ROWS = 8 * EIGHTS, THREADS = 32 * WARPS;
    static constexpr int PIECE = PADDED % 64 == 0 ? 16 : 8;                // bytes of a key that a lane reads at once
    static constexpr int CHUNKS = PADDED / (4 * PIECE), STEPS = PIECE / 4; // a chunk: four lanes' pieces, STEPS instructions
    static constexpr uint32_t HALF = CACHE_PAGE * PADDED;                  // a page's keys, or its values
    static constexpr size_t QUERIES = (size_t)ROWS * PADDED * 2;           // operand fragments
    static constexpr bool HELD = PADDED * EIGHTS <= 256;                   // in registers
    static constexpr size_t RING = WARPS * STAGES * HALF;
    static_assert(ROWS * PADDED * 4 <= STAGES * HALF, "the ring takes the warps' sums");
    static constexpr size_t SMEM = RING + QUERIES;
    static constexpr int BLOCKS = WARPS == 8 ? 1 : PADDED <= 128 ? EIGHTS == 1 ? 3 : 2 : PADDED <= 192 ? 2 : 1; // an SM's
    using Sharing = Plan<ROWS, THREADS>;
};

// Lane 4 g + t: sums of values of dimensions 16 i + g (first two) and 16 i + 8 + g, for rows 2 t and 2 t + 1 (of each eight); these rows' figures.
template <int PADDED, int EIGHTS> struct Running {
    float y[EIGHTS][PADDED / 16][4];
    float m[EIGHTS][2], top[EIGHTS][2], l[EIGHTS][2];
};

// Products of a page's keys with the rows.  Tile i: row g of it is token 16 (g / 2) + 4 i + g % 2, row 8 + g the token two behind that.
template <int PADDED, int EIGHTS, int WARPS> __device__ __forceinline__ void take_keys(const uint8_t *keys, const uint2 *queries, const uint2 (&held)[EIGHTS][PADDED / 16], float (&s)[EIGHTS][4][4])
{
    using Shape = FewShape<PADDED, EIGHTS, WARPS>;
    const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[e][i][0] = s[e][i][1] = s[e][i][2] = s[e][i][3] = 0.0f;
    const uint8_t *mine = keys + (16 * (g >> 1) + (g & 1)) * PADDED;
    const int turned = PADDED % 128 == 0 ? 64 * (g & 1) : 0;
#pragma unroll
    for (int c = 0; c < Shape::CHUNKS; ++c) {
        uint2 b[EIGHTS][Shape::STEPS];
#pragma unroll
        for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
            for (int k = 0; k < Shape::STEPS; ++k) b[e][k] = Shape::HELD ? held[e][c * Shape::STEPS + k] : queries[(e * PADDED / 16 + c * Shape::STEPS + k) * 32 + lane];
        const int at = (c * 4 * Shape::PIECE + t * Shape::PIECE) ^ turned;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Words<Shape::PIECE> w0 = words_at<Shape::PIECE>(mine + 4 * i * PADDED + at), w1 = words_at<Shape::PIECE>(mine + (4 * i + 2) * PADDED + at);
#pragma unroll
            for (int k = 0; k < Shape::STEPS; ++k) {
                uint32_t a0, a1, a2, a3;
                codes_to_halves(w0[k], a0, a2);
                codes_to_halves(w1[k], a1, a3);
#pragma unroll
                for (int e = 0; e < EIGHTS; ++e) mma_f16(s[e][i], a0, a1, a2, a3, b[e][k]);
            }
        }
    }
}

template <int PADDED, int EIGHTS> __device__ __forceinline__ void take_values(const uint8_t *values, const uint2 (&weights)[EIGHTS][4], float (&y)[EIGHTS][PADDED / 16][4])
{
    const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const uint8_t *mine = values + g * CACHE_PAGE + 16 * t;
#pragma unroll
    for (int d = 0; d < PADDED / 16; ++d) {
        const Words<16> w0 = words_at<16>(mine + 16 * d * CACHE_PAGE), w1 = words_at<16>(mine + (16 * d + 8) * CACHE_PAGE);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t a0, a1, a2, a3;
            codes_to_halves(w0[k], a0, a2);
            codes_to_halves(w1[k], a1, a3);
#pragma unroll
            for (int e = 0; e < EIGHTS; ++e) mma_f16(y[e][d], a0, a1, a2, a3, weights[e][k]);
        }
    }
}

// A page's scores to weights of its values; the running figures go along.  hidden[e][h]: bit 2 i + j for token j of tile i (the lane's two) where row 2 t + h does not see it.
template <int PADDED, int EIGHTS, bool MASKED>
__device__ __forceinline__ void weigh(float (&s)[EIGHTS][4][4], const float (&down)[EIGHTS][2], float scale_k, float scale_v, const uint32_t (&hidden)[EIGHTS][2],
                                      Running<PADDED, EIGHTS> &run, uint2 (&weights)[EIGHTS][4])
{
    const bool none = scale_v == 0.0f, is_nan = scale_v != scale_v;
    const float log_v = log2f(scale_v);
    float factor[EIGHTS][2], higher[EIGHTS][2];
    bool rise = false;
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (MASKED) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (hidden[e][h] >> (2 * i + j) & 1u) s[e][i][2 * j + h] = -INFINITY;
            }
            factor[e][h] = score_factor(down[e][h], scale_k);
            float most = fmaxf(s[e][0][h], s[e][0][2 + h]);
#pragma unroll
            for (int i = 1; i < 4; ++i) most = fmaxf(fmaxf(most, s[e][i][h]), s[e][i][2 + h]);
            higher[e][h] = most == -INFINITY ? most : most * factor[e][h];
            rise |= higher[e][h] > run.m[e][h] + LATE || (!none && higher[e][h] + (is_nan ? 0.0f : log_v) > run.top[e][h] + LATE);
        }
    if (__any_sync(~0u, rise)) {
#pragma unroll
        for (int e = 0; e < EIGHTS; ++e) {
            float old[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float m = higher[e][h];
#pragma unroll
                for (int o = 4; o < 32; o *= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, o)); // (NaN is passed over)
                const float top = none ? -INFINITY : m + (is_nan ? 0.0f : log_v), new_m = fmaxf(run.m[e][h], m), new_top = fmaxf(run.top[e][h], top);
                run.l[e][h] *= relative(run.m[e][h], new_m);
                old[h] = relative(run.top[e][h], new_top);
                run.m[e][h] = new_m, run.top[e][h] = new_top;
            }
#pragma unroll
            for (int d = 0; d < PADDED / 16; ++d) run.y[e][d][0] *= old[0], run.y[e][d][1] *= old[1], run.y[e][d][2] *= old[0], run.y[e][d][3] *= old[1];
        }
    }
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e) {
        float shift[2], plus[2], from[2];
        bool far = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            from[h] = run.m[e][h] == -INFINITY ? 0.0f : run.m[e][h];
            const float from_top = run.top[e][h] == -INFINITY ? 0.0f : run.top[e][h];
            shift[h] = log_v + from[h] - from_top; // a weight is 2^(s - m) 2^shift (values of 0: shift is -infinity, weights are 0)
            plus[h] = log_v - from_top;
            far |= fabsf(shift[h]) > 60.0f;
        }
        far = __any_sync(~0u, far);
        float w[4][4], sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int h = j % 2;
                w[i][j] = power_of_two(fmaf(s[e][i][j], factor[e][h], plus[h]));
                if (MASKED && (hidden[e][h] >> (2 * i + j / 2) & 1u)) w[i][j] = 0.0f; // (NaN where a factor is 0 or NaN)
                sum[h] += w[i][j];
            }
        if (far) { // either of 2^(s - m) and the weight may be 0 where the other is not
            sum[0] = sum[1] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int h = j % 2;
                    const float p = power_of_two(fmaf(s[e][i][j], factor[e][h], -from[h]));
                    sum[h] += MASKED && (hidden[e][h] >> (2 * i + j / 2) & 1u) ? 0.0f : p;
                }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (sum[h] != 0.0f) run.l[e][h] += far ? sum[h] : sum[h] * exp2f(-shift[h]);
#pragma unroll
        for (int i = 0; i < 4; ++i) weights[e][i] = make_uint2(transposed(halves_of_floats(w[i][0], w[i][1])), transposed(halves_of_floats(w[i][2], w[i][3])));
    }
}

// A tile's queries as operand fragments, and each row's factor of scores: lane 4 g + t of step k of chunk c has dimensions d .. d + 3, d = (4 c + t) PIECE + 4 k, of row g of
// each eight.  By the block: eight threads a row.  A negative scale turns the queries' signs: factors are not negative, and the largest product is the largest score.
template <int PADDED, int EIGHTS, int WARPS>
__device__ __forceinline__ void bring_queries(const Attend &a, const Span &span, const Tile<8 * EIGHTS> &tile, int rows, uint2 *queries, float *down)
{
    using Shape = FewShape<PADDED, EIGHTS, WARPS>;
    const int part = threadIdx.x % 8, width = (int)a.cache.width;
    const bool f16 = a.queries.type == VALUE_F16;
    const bool aligned = width % 4 == 0 && a.queries.ld % 4 == 0 && a.queries.head_ld % 4 == 0 && (reinterpret_cast<uintptr_t>(a.queries.x) & 7) == 0;
    for (int r = threadIdx.x / 8; r < Shape::ROWS; r += Shape::THREADS / 8) {
        const int at = tile.first_row + min(r, rows - 1); // (rows behind the tile's: its last one)
        const uint16_t *x = static_cast<const uint16_t *>(a.queries.x) + (size_t)(span.row + at / a.group) * a.queries.ld + (size_t)(tile.head * a.group + at % a.group) * a.queries.head_ld;
        constexpr int FOURS = PADDED / 32; // four dimensions at a time: 4 (8 i + part)
        uint2 four[FOURS];
        float v[FOURS][4];
        uint32_t most = 0;
        if (aligned) { // (no branch for each load, at whose end it would be waited for)
#pragma unroll
            for (int i = 0; i < FOURS; ++i) four[i] = *reinterpret_cast<const uint2 *>(x + min(4 * (8 * i + part), width - 4));
        } else {
#pragma unroll
            for (int i = 0; i < FOURS; ++i) {
                const int d = 4 * (8 * i + part);
                four[i] = make_uint2(x[min(d, width - 1)] | (uint32_t)x[min(d + 1, width - 1)] << 16, x[min(d + 2, width - 1)] | (uint32_t)x[min(d + 3, width - 1)] << 16);
            }
        }
#pragma unroll
        for (int i = 0; i < FOURS; ++i) {
            const int d = 4 * (8 * i + part);
            const uint32_t w[2] = {four[i].x & ((d < width ? 0xFFFFu : 0u) | (d + 1 < width ? 0xFFFF0000u : 0u)), four[i].y & ((d + 2 < width ? 0xFFFFu : 0u) | (d + 3 < width ? 0xFFFF0000u : 0u))};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t half = j % 2 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu;
                v[i][j] = f16 ? __half2float(__ushort_as_half((unsigned short)half)) : __uint_as_float(half << 16);
                most = max(most, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
            }
        }
#pragma unroll
        for (int o = 4; o; o /= 2) most = max(most, __shfl_xor_sync(~0u, most, o));
        const QueryScale scale(most, fabsf(a.scale));
        const float up = a.scale < 0.0f ? -scale.up : scale.up;
        if (part == 0) down[r] = scale.down;
#pragma unroll
        for (int i = 0; i < FOURS; ++i) {
            const int d = 4 * (8 * i + part), c = d / (4 * Shape::PIECE), t = d / Shape::PIECE % 4, step = d % Shape::PIECE / 4;
            const bool none = scale.up == 0.0f; // (an infinity or a NaN: 0 times that is none)
            queries[(r / 8 * PADDED / 16 + c * Shape::STEPS + step) * 32 + 4 * (r % 8) + t] =
                none ? make_uint2(0, 0) : make_uint2(halves_of_floats(v[i][0] * up, v[i][1] * up), halves_of_floats(v[i][2] * up, v[i][3] * up));
        }
    }
}

template <int PADDED, int EIGHTS, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, FewShape<PADDED, EIGHTS, WARPS>::BLOCKS) attend_few_kernel(const __grid_constant__ ShareParams P)
{
    using Shape = FewShape<PADDED, EIGHTS, WARPS>;
    constexpr int ROWS = Shape::ROWS, THREADS = Shape::THREADS;
    extern __shared__ unsigned char smem_raw[];
    __shared__ typename Shape::Sharing::Room room;
    __shared__ unsigned long long full[WARPS][STAGES];
    __shared__ float down[ROWS], figures[WARPS][3][ROWS], final_figures[3][ROWS];
    __shared__ int abort_word;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~(uintptr_t)127);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    uint8_t *ring = smem + (size_t)warp * STAGES * Shape::HALF;
    uint2 *queries = reinterpret_cast<uint2 *>(smem + Shape::RING);
    if (threadIdx.x == 0) abort_word = 0;
    if (lane < STAGES) mbar_init(&full[warp][lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    cache_is_there();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // (attend_join_kernel of the same call)
    const Attend &a = P.a;
    const Cache &c = a.cache;
    if (a.zero_rest && a.seq.offsets) {
        const int front = offset_of(a.seq, 0), behind = max(offset_of(a.seq, a.seq.sequences), front), heads = (int)c.heads * a.group, width = (int)c.width;
        const size_t many = (size_t)(front + a.seq.n - behind) * heads * width;
        for (size_t i = (size_t)blockIdx.x * THREADS + threadIdx.x; i < many; i += (size_t)gridDim.x * THREADS) {
            const size_t r = i / ((size_t)heads * width), rest = i % ((size_t)heads * width);
            put_value(a.y, (r < (size_t)front ? r : r - front + behind) * a.y.ld + rest / width * a.y.head_ld + rest % width, 0.0f);
        }
    }
    const typename Shape::Sharing plan(P, room);
    const long long start = plan.share * blockIdx.x, end = min(start + plan.share, plan.total);
    if (start >= end && threadIdx.x == 0) plan.tell(nullptr, 0, 0);
    int st = 0; // of the ring, and how often it went round
    uint32_t parity = 0;
    for (long long x = start; x < end;) {
        Tile<ROWS> tile;
        if (!plan.find(x, tile)) break;
        const Span span(a.seq, tile.b);
        const int rows = min(span.count * a.group - tile.first_row, ROWS);
        if (x == start && threadIdx.x == 0) plan.tell(&tile, span.row, rows);
        const int p0 = span.first + tile.first_row / a.group, p1 = span.first + (tile.first_row + rows - 1) / a.group;
        const Pages pages(p0, p1, span.keys, a.window, a.sinks);
        const int first = (int)(x - tile.begin), behind = (int)(min(end, tile.begin + tile.units) - tile.begin); // units
        const int from = first * P.unit, last = (int)min((long long)behind * P.unit, (long long)pages.count);
        const int many = last > from + warp ? (last - from - warp + WARPS - 1) / WARPS : 0; // pages of this warp: from + warp + WARPS i

        // where the next 32 pages are, a lane each, and the 32 behind them
        int page_now, page_next = -1;
        float2 scales_now, scales_next = make_float2(0.0f, 0.0f);
        auto look = [&](int i0, int &page, float2 &scales) {
            const int i = i0 + lane;
            page = i < many ? page_of(a.seq, c.pages, tile.b, pages.column(from + warp + WARPS * i)) : -1;
            scales = page >= 0 ? *reinterpret_cast<const float2 *>(c.scales + ((size_t)page * c.heads + tile.head) * 2) : make_float2(0.0f, 0.0f);
        };
        look(0, page_now, scales_now);
        if (many > 32) look(32, page_next, scales_next);
        // half 2 i: keys of page i, 2 i + 1: its values; block: i / 32 of page_now
        auto fetch = [&](int half, int stage, int block) {
            const int i = half / 2, page = __shfl_sync(~0u, i / 32 == block ? page_now : page_next, i % 32);
            if (lane == 0 && i < many) {
                if (page >= 0) {
                    mbar_expect_tx(&full[warp][stage], Shape::HALF);
                    bulk_load_1d(ring + stage * Shape::HALF, c.codes + (((size_t)page * c.heads + tile.head) * 2 + (half & 1)) * Shape::HALF, Shape::HALF, &full[warp][stage]);
                } else {
                    mbar_arrive(&full[warp][stage]);
                }
            }
        };
        for (int k = 0, stage = st; k < STAGES; ++k) {
            fetch(k, stage, 0);
            if (++stage == STAGES) stage = 0;
        }
        bring_queries<PADDED, EIGHTS, WARPS>(a, span, tile, rows, queries, down);
        __syncthreads();
        Running<PADDED, EIGHTS> run;
        float mine[EIGHTS][2];
        int position[EIGHTS][2];
        uint2 held[EIGHTS][PADDED / 16];
#pragma unroll
        for (int e = 0; e < EIGHTS; ++e) {
#pragma unroll
            for (int d = 0; d < PADDED / 16; ++d) run.y[e][d][0] = run.y[e][d][1] = run.y[e][d][2] = run.y[e][d][3] = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = 8 * e + 2 * t + h;
                run.m[e][h] = run.top[e][h] = -INFINITY, run.l[e][h] = 0.0f;
                mine[e][h] = down[r], position[e][h] = span.first + (tile.first_row + min(r, rows - 1)) / a.group;
            }
            if (Shape::HELD) {
#pragma unroll
                for (int k = 0; k < PADDED / 16; ++k) held[e][k] = queries[(e * PADDED / 16 + k) * 32 + lane];
            }
        }
        for (int i = 0; i < many; ++i) {
            const int page = __shfl_sync(~0u, page_now, i % 32);
            const float scale_k = __shfl_sync(~0u, scales_now.x, i % 32), scale_v = __shfl_sync(~0u, scales_now.y, i % 32);
            uint2 weights[EIGHTS][4];
            if (!__all_sync(~0u, mbar_wait(&full[warp][st], parity, &abort_word, P.error, 91))) break;
            float s[EIGHTS][4][4];
            if (page >= 0) take_keys<PADDED, EIGHTS, WARPS>(ring + st * Shape::HALF, queries, held, s);
            __syncwarp();
            fetch(2 * i + STAGES, st, i / 32);
            if (++st == STAGES) st = 0, parity ^= 1u;
            if (page >= 0) {
                const int column = pages.column(from + warp + WARPS * i);
                uint32_t hidden[EIGHTS][2] = {};
                if (all_seen(column, p0, p1, span.keys, a.window, a.sinks)) {
                    weigh<PADDED, EIGHTS, false>(s, mine, scale_k, scale_v, hidden, run, weights);
                } else {
#pragma unroll
                    for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (!seen(column * CACHE_PAGE + 16 * (g >> 1) + (g & 1) + 2 * j, position[e][h], span.keys, a.window, a.sinks)) hidden[e][h] |= 1u << j;
                    weigh<PADDED, EIGHTS, true>(s, mine, scale_k, scale_v, hidden, run, weights);
                }
            }
            if (!__all_sync(~0u, mbar_wait(&full[warp][st], parity, &abort_word, P.error, 92))) break;
            if (page >= 0) take_values<PADDED, EIGHTS>(ring + st * Shape::HALF, weights, run.y);
            __syncwarp();
            fetch(2 * i + 1 + STAGES, st, i / 32);
            if (++st == STAGES) st = 0, parity ^= 1u;
            if (i % 32 == 31) {
                page_now = page_next, scales_now = scales_next;
                look(i + 33, page_next, scales_next);
            }
        }
        // the warps' figures together, in the place of the ring (all that was asked for has come)
#pragma unroll
        for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int o = 4; o < 32; o *= 2) run.l[e][h] += __shfl_xor_sync(~0u, run.l[e][h], o);
                const int r = 8 * e + 2 * t + h;
                if (g == 0) figures[warp][0][r] = run.m[e][h], figures[warp][1][r] = run.top[e][h], figures[warp][2][r] = run.l[e][h];
            }
        __syncthreads();
        float *sum = reinterpret_cast<float *>(ring); // ROWS x PADDED, of this warp
#pragma unroll
        for (int e = 0; e < EIGHTS; ++e)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = 8 * e + 2 * t + h;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) top = fmaxf(top, figures[w][1][r]);
                const float by = relative(run.top[e][h], top);
#pragma unroll
                for (int d = 0; d < PADDED / 16; ++d) sum[r * PADDED + 16 * d + g] = run.y[e][d][h] * by, sum[r * PADDED + 16 * d + 8 + g] = run.y[e][d][2 + h] * by;
            }
        if (threadIdx.x < ROWS) {
            float m = -INFINITY, top = -INFINITY, l = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) m = fmaxf(m, figures[w][0][threadIdx.x]), top = fmaxf(top, figures[w][1][threadIdx.x]);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) l += figures[w][2][threadIdx.x] * relative(figures[w][0][threadIdx.x], m);
            final_figures[0][threadIdx.x] = m, final_figures[1][threadIdx.x] = top, final_figures[2][threadIdx.x] = l;
        }
        __syncthreads();
        const bool whole = first == 0 && behind == tile.units;
        float *part = whole ? nullptr : plan.part(blockIdx.x, x == start, PADDED);
        if (!whole && threadIdx.x < 3 * ROWS) part[ROWS * PADDED + threadIdx.x] = (&final_figures[0][0])[threadIdx.x];
        for (int i = threadIdx.x; i < rows * PADDED; i += THREADS) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v += reinterpret_cast<const float *>(smem + (size_t)w * STAGES * Shape::HALF)[i];
            const int r = i / PADDED, d = i % PADDED, at = tile.first_row + r;
            if (!whole) part[i] = v;
            else if (d < (int)c.width)
                put_value(a.y, (size_t)(span.row + at / a.group) * a.y.ld + (size_t)(tile.head * a.group + at % a.group) * a.y.head_ld + d,
                          RowEnd(final_figures[0][r], final_figures[1][r], final_figures[2][r]).of(v));
        }
        x = tile.begin + behind;
        if (*(volatile int *)&abort_word) break; // (set before the barriers above if at all)
        if (x < end) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // (the ring is written by copies next)
            __syncthreads();
        }
    }
    if (*(volatile int *)&abort_word) // what has been asked for lands before the block leaves
        for (int w = 0; w < 1000; ++w) __nanosleep(1000);
}

// Pages of a tile at most, as far as the host knows.
template <int ROWS> size_t most_pages(const Attend &a)
{
    const size_t pages = std::max(a.seq.columns, 1);
    return a.window ? std::min(pages, ((size_t)a.sinks + 63) / 64 + ((size_t)a.window + ROWS + 62) / CACHE_PAGE + 1) : pages;
}

template <int PADDED, int EIGHTS, int WARPS> void attend_few_with(CudaDevice &dev, ShareParams &P)
{
    using Shape = FewShape<PADDED, EIGHTS, WARPS>;
    constexpr int ROWS = Shape::ROWS;
    P.slots = (int)slots_of<ROWS>(P.a);
    const size_t rounds = (most_pages<ROWS>(P.a) + WARPS - 1) / WARPS;
    const bool join = rounds > 16 / WARPS; // (up to sixteen pages are not shared out: one token behind 1000 in 14 us, 12 and another launch where they are)
    P.unit = (int)(join ? WARPS : rounds * WARPS);
    const size_t units = (size_t)P.slots * P.a.cache.heads * (join ? rounds : 1), places = (size_t)dev.sm_count() * Shape::BLOCKS;
    P.blocks = (int)std::min(units, places);
    Parts parts(dev);
    if (join) parts.make<ROWS>(P, PADDED);
    allow_shared_memory(dev, attend_few_kernel<PADDED, EIGHTS, WARPS>);
    {
        KernelScope ks(dev, "attend_few");
        launch_following(attend_few_kernel<PADDED, EIGHTS, WARPS>, dim3((unsigned)P.blocks), dim3(Shape::THREADS), Shape::SMEM + 128, dev.stream(), P);
        dev.count_launch();
    }
    launch_join<PADDED, ROWS>(dev, P);
}

// Eight warps a block where every tile has an SM to itself and as few pages as are not shared out: one token behind 1000 in 11.8 us instead of 14.  (The table's columns say how many pages there may
// be, for the lengths are not known here: in a table of more than 16 columns the same token takes 14 us, whatever its length.)  (Elsewhere four are better
// used: 64 sequences of up to 8192 tokens take 101 us and not 118.)
template <int PADDED, int EIGHTS> void attend_few_rows(CudaDevice &dev, ShareParams &P)
{
    if constexpr (PADDED <= 160) {
        const size_t pages = most_pages<8 * EIGHTS>(P.a);
        if (pages > 4 && pages <= 16 && slots_of<8 * EIGHTS>(P.a) * P.a.cache.heads <= (size_t)dev.sm_count()) return attend_few_with<PADDED, EIGHTS, 8>(dev, P);
    }
    attend_few_with<PADDED, EIGHTS, 4>(dev, P);
}

template <int PADDED> void attend_few_width(CudaDevice &dev, ShareParams &P)
{
    const size_t rows = (size_t)P.a.seq.n * P.a.group;
    if (!P.a.seq.offsets && rows / P.a.seq.sequences <= 8) attend_few_rows<PADDED, 1>(dev, P);
    else attend_few_rows<PADDED, 2>(dev, P);
}

} // namespace

void launch_attend_few(CudaDevice &dev, const Attend &a)
{
    ShareParams P{};
    P.a = a, P.error = dev.error_word(), P.least = 0, P.most = ATTEND_FEW;
    switch (a.cache.padded / 32) {
    case 1: return attend_few_width<32>(dev, P);
    case 2: return attend_few_width<64>(dev, P);
    case 3: return attend_few_width<96>(dev, P);
    case 4: return attend_few_width<128>(dev, P);
    case 5: return attend_few_width<160>(dev, P);
    case 6: return attend_few_width<192>(dev, P);
    case 7: return attend_few_width<224>(dev, P);
    default: return attend_few_width<256>(dev, P);
    }
}

void launch_attend(CudaDevice &dev, const Attend &a)
{
    if (!dev.error_word()) return launch_attend_plain(dev, a);
    // sequences of many rows, if there can be any, go to the one kernel, the others to the other
    const size_t rows = (size_t)a.seq.n * a.group, most = a.seq.offsets ? rows : rows / a.seq.sequences;
    const bool few = a.seq.offsets || most <= ATTEND_FEW, many = most > ATTEND_FEW;
    if (few) launch_attend_few(dev, a);
    if (many) launch_attend_many(dev, a);
}

} // namespace vqb
