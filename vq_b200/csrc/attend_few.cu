// attend_few.cu -- attention of a few rows of each sequence (single tokens above all) over a cache of 8-bit codes.
//
// Sixteen rows that share a cached head (query heads of a token, then those of the next one) are a tile.  What bounds it is the cache's bytes, read once for a tile: 2 x 64 x
// width of them a page and head.  Every warp fetches pages for itself (one bulk copy for a page's keys, one for its values) into a ring of its own, some 90 KB of an SM's on their
// way at any time, turns the codes to f16 numbers in registers and multiplies (mma.sync m16n8k16: with sixteen rows the tensor cores' larger instructions would
// be seven eighths empty).  Scores never leave registers: columns of a page's score tile stand for tokens in such an order that a lane's scores are
// the operand of the product with the values, whose tokens lie side by side.
//
// All tiles' pages are numbered in a row, and each block takes an equal share of that, whatever the sequences' lengths are (nobody on the host knows them).  What
// a share's end cuts off a tile leaves as a part (its largest scores, sum, and sums of values), and a second kernel joins parts, in the order of their pages.
#include <algorithm>

#include "attend.cuh"
#include "cuda_device.hpp"
#include "umma.cuh"

namespace vqb {

namespace {

constexpr int WARPS = 4, THREADS = 32 * WARPS, ROWS = 16, STAGES = 3;

using FewPlan = Plan<ROWS, THREADS>;
using FewTile = Tile<ROWS>;

__device__ __forceinline__ void mma_f16(float (&sums)[4], const uint4 &a, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(sums[0]), "+f"(sums[1]), "+f"(sums[2]), "+f"(sums[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
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

template <int PADDED> struct FewShape {
    static constexpr int PIECE = PADDED % 64 == 0 ? 16 : 8;     // bytes of a key that a lane reads at once
    static constexpr int CHUNKS = PADDED / (4 * PIECE), STEPS = PIECE / 4; // a chunk: four lanes' pieces, STEPS instructions
    static constexpr uint32_t HALF = CACHE_PAGE * PADDED;       // a page's keys, or its values
    static constexpr size_t QUERIES = (size_t)ROWS * PADDED * 2; // operand fragments
    static constexpr size_t SMEM = WARPS * STAGES * HALF + QUERIES;
};

// the rows' largest scores, the sum below the line and the sums of values, of one warp's pages
template <int PADDED> struct Running {
    float y[PADDED / 8][4]; // rows g, g, g + 8, g + 8; dimensions 2 t, 2 t + 1 of each eight (lane = 4 g + t)
    float m[2], top[2], l[2];
};

// products of the rows with a page's keys
template <int PADDED> __device__ __forceinline__ void take_keys(const uint8_t *keys, const uint4 *queries, float (&s)[8][4])
{
    using Shape = FewShape<PADDED>;
    const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
    const uint8_t *mine = keys + (16 * (g >> 1) + (g & 1)) * PADDED; // tile j's column g is token 16 (g / 2) + 2 j + g % 2
    const int turned = PADDED % 128 == 0 ? 64 * (g & 1) : 0;
#pragma unroll
    for (int c = 0; c < Shape::CHUNKS; ++c) {
        uint4 a[Shape::STEPS];
#pragma unroll
        for (int i = 0; i < Shape::STEPS; ++i) a[i] = queries[(c * Shape::STEPS + i) * 32 + lane];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const Words<Shape::PIECE> w = words_at<Shape::PIECE>(mine + 2 * j * PADDED + ((c * 4 * Shape::PIECE + t * Shape::PIECE) ^ turned));
#pragma unroll
            for (int i = 0; i < Shape::STEPS; ++i) {
                uint32_t b0, b1;
                codes_to_halves(w[i], b0, b1);
                mma_f16(s[j], a[i], b0, b1);
            }
        }
    }
}

template <int PADDED> __device__ __forceinline__ void take_values(const uint8_t *values, const uint4 (&weights)[4], float (&y)[PADDED / 8][4])
{
    const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const uint8_t *mine = values + g * CACHE_PAGE + 16 * t;
#pragma unroll
    for (int d = 0; d < PADDED / 8; ++d) {
        const Words<16> w = words_at<16>(mine + 8 * d * CACHE_PAGE);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t b0, b1;
            codes_to_halves(w[i], b0, b1);
            mma_f16(y[d], weights[i], b0, b1);
        }
    }
}

// The scores of a page to weights of its values; the running figures go along.  hidden: bit 2 j + e for what row h (0, 1) does not see.
template <int PADDED, bool MASKED>
__device__ __forceinline__ void weigh(float (&s)[8][4], const float (&factor)[2], const PageScales &page, const uint32_t (&hidden)[2], Running<PADDED> &run, uint4 (&weights)[4])
{
    float largest[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int h = i / 2;
            s[j][i] *= factor[h];
            if (MASKED && (hidden[h] >> (2 * j + i % 2) & 1u)) s[j][i] = -INFINITY;
            largest[h] = fmaxf(largest[h], s[j][i]);
        }
    float base[2], shift[2], old[2];
    bool far = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        largest[h] = fmaxf(largest[h], __shfl_xor_sync(~0u, largest[h], 1));
        largest[h] = fmaxf(largest[h], __shfl_xor_sync(~0u, largest[h], 2));
        const float m = fmaxf(run.m[h], largest[h]), top = page.f == 0.0f ? run.top[h] : fmaxf(run.top[h], largest[h] + page.e);
        run.l[h] *= relative(run.m[h], m);
        old[h] = relative(run.top[h], top);
        run.m[h] = m, run.top[h] = top;
        base[h] = m == -INFINITY ? 0.0f : m;
        const float from = top == -INFINITY ? 0.0f : top;
        shift[h] = page.f == 0.0f ? -1e30f : base[h] + page.e - from; // weights: 2^(s - base) 2^shift f
        far |= shift[h] > 60.0f;
    }
    if (__any_sync(~0u, old[0] != 1.0f || old[1] != 1.0f)) {
#pragma unroll
        for (int d = 0; d < PADDED / 8; ++d) run.y[d][0] *= old[0], run.y[d][1] *= old[0], run.y[d][2] *= old[1], run.y[d][3] *= old[1];
    }
    float w[8][4];
    if (__any_sync(~0u, far)) { // 2^(s - base) may be 0 where the weight is not
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int h = i / 2;
                run.l[h] += power_of_two(s[j][i] - base[h]);
                w[j][i] = power_of_two(s[j][i] - (base[h] - shift[h])) * page.f;
            }
    } else {
        float scale[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) scale[h] = exp2f(shift[h]) * page.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int h = i / 2;
                const float p = power_of_two(s[j][i] - base[h]);
                run.l[h] += p;
                w[j][i] = p * scale[h];
            }
    }
    if (MASKED) { // (0 times NaN)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (hidden[i / 2] >> (2 * j + i % 2) & 1u) w[j][i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        weights[i] = make_uint4(halves_of_floats(w[2 * i][0], w[2 * i][1]), halves_of_floats(w[2 * i][2], w[2 * i][3]), halves_of_floats(w[2 * i + 1][0], w[2 * i + 1][1]),
                                halves_of_floats(w[2 * i + 1][2], w[2 * i + 1][3]));
}

// A tile's queries as operand fragments, and each row's factor of scores: lane 4 g + t of step i of chunk c has dimensions d .. d + 3, d = (4 c + t) PIECE + 4 i, of
// rows g and g + 8.  By the block: eight threads a row.
template <int PADDED> __device__ __forceinline__ void bring_queries(const Attend &a, const Span &span, const FewTile &tile, int rows, uint32_t *queries, float *down)
{
    using Shape = FewShape<PADDED>;
    const int r = threadIdx.x / 8, part = threadIdx.x % 8, at = tile.first_row + r, width = (int)a.cache.width;
    const bool there = r < rows;
    const size_t from = there ? (size_t)(span.row + at / a.group) * a.queries.ld + (size_t)(tile.head * a.group + at % a.group) * a.queries.head_ld : 0;
    const uint16_t *x = static_cast<const uint16_t *>(a.queries.x) + from;
    const bool f16 = a.queries.type == VALUE_F16, aligned = (reinterpret_cast<uintptr_t>(x) & 7) == 0;
    constexpr int FOURS = PADDED / 32; // four dimensions at a time: 4 (8 i + part)
    float v[FOURS][4];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
        const int d = 4 * (8 * i + part);
        uint32_t w[2] = {0, 0};
        if (there && aligned && d + 4 <= width) {
            const uint2 q = *reinterpret_cast<const uint2 *>(x + d);
            w[0] = q.x, w[1] = q.y;
        } else if (there) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < width) w[j / 2] |= (uint32_t)x[d + j] << (16 * (j % 2));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t half = j % 2 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu;
            v[i][j] = f16 ? __half2float(__ushort_as_half((unsigned short)half)) : __uint_as_float(half << 16);
            most = max(most, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
        }
    }
#pragma unroll
    for (int o = 4; o; o /= 2) most = max(most, __shfl_xor_sync(~0u, most, o));
    const QueryScale scale(most, a.scale);
    if (part == 0) down[r] = scale.down;
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
        const int d = 4 * (8 * i + part), c = d / (4 * Shape::PIECE), t = d / Shape::PIECE % 4, step = d % Shape::PIECE / 4;
        uint32_t *to = queries + (((c * Shape::STEPS + step) * 32 + 4 * (r % 8) + t) * 4 + r / 8);
        const bool none = scale.up == 0.0f; // (an infinity or a NaN: 0 times that is none)
        to[0] = none ? 0u : halves_of_floats(v[i][0] * scale.up, v[i][1] * scale.up);
        to[2] = none ? 0u : halves_of_floats(v[i][2] * scale.up, v[i][3] * scale.up);
    }
}

template <int PADDED> __global__ void __launch_bounds__(THREADS, PADDED <= 128 ? 2 : 1) attend_few_kernel(const __grid_constant__ ShareParams P)
{
    using Shape = FewShape<PADDED>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ FewPlan::Room room;
    __shared__ unsigned long long full[WARPS][STAGES];
    __shared__ float down[ROWS], figures[WARPS][3][ROWS], final_figures[3][ROWS];
    __shared__ int abort_word;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~(uintptr_t)127);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    uint8_t *ring = smem + (size_t)warp * STAGES * Shape::HALF;
    uint32_t *queries = reinterpret_cast<uint32_t *>(smem + (size_t)WARPS * STAGES * Shape::HALF);
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
    const FewPlan plan(P, room);
    const long long start = plan.share * blockIdx.x, end = min(start + plan.share, plan.total);
    int st = 0;          // of the ring, and how often it went round
    uint32_t parity = 0;
    for (long long x = start; x < end;) {
        FewTile tile;
        if (!plan.find(x, tile)) break;
        const Span span(a.seq, tile.b);
        const int rows = min(span.count * a.group - tile.first_row, ROWS);
        const int p0 = span.first + tile.first_row / a.group, p1 = span.first + (tile.first_row + rows - 1) / a.group;
        const Pages pages(p0, p1, span.keys, a.window, a.sinks);
        const int first = (int)(x - tile.begin), behind = (int)(min(end, tile.begin + tile.units) - tile.begin); // units
        const int from = first * P.unit, last = (int)min((long long)behind * P.unit, (long long)pages.count);
        const int many = last > from + warp ? (last - from - warp + WARPS - 1) / WARPS : 0; // pages of this warp: from + warp + WARPS i

        // where the next 32 pages are, a lane each, and the 32 behind them
        int page_now, page_next;
        float2 scales_now, scales_next;
        auto look = [&](int i0, int &page, float2 &scales) {
            const int i = i0 + lane;
            page = i < many ? page_of(a.seq, c.pages, tile.b, pages.column(from + warp + WARPS * i)) : -1;
            scales = page >= 0 ? *reinterpret_cast<const float2 *>(c.scales + ((size_t)page * c.heads + tile.head) * 2) : make_float2(0.0f, 0.0f);
        };
        look(0, page_now, scales_now);
        page_next = -1, scales_next = scales_now;
        if (many > 32) look(32, page_next, scales_next);
        // half 2 i: keys of page i, 2 i + 1: its values
        auto fetch = [&](int half, int stage, int block) { // block: i / 32 of page_now
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
        bring_queries<PADDED>(a, span, tile, rows, queries, down);
        __syncthreads();
        Running<PADDED> run;
#pragma unroll
        for (int d = 0; d < PADDED / 8; ++d) run.y[d][0] = run.y[d][1] = run.y[d][2] = run.y[d][3] = 0.0f;
        run.m[0] = run.m[1] = run.top[0] = run.top[1] = -INFINITY, run.l[0] = run.l[1] = 0.0f;
        const float mine[2] = {down[g], down[g + 8]};
        const int position[2] = {span.first + (tile.first_row + min(g, rows - 1)) / a.group, span.first + (tile.first_row + min(g + 8, rows - 1)) / a.group};
        for (int i = 0; i < many; ++i) {
            const int page = __shfl_sync(~0u, page_now, i % 32);
            const float2 both = make_float2(__shfl_sync(~0u, scales_now.x, i % 32), __shfl_sync(~0u, scales_now.y, i % 32));
            uint4 weights[4];
            if (!__all_sync(~0u, mbar_wait(&full[warp][st], parity, &abort_word, P.error, 91))) break;
            if (page >= 0) {
                float s[8][4];
                take_keys<PADDED>(ring + st * Shape::HALF, reinterpret_cast<const uint4 *>(queries), s);
                const PageScales scales(both);
                const float factor[2] = {score_factor(mine[0], scales.k), score_factor(mine[1], scales.k)};
                const int column = pages.column(from + warp + WARPS * i);
                uint32_t hidden[2] = {0, 0};
                if (all_seen(column, p0, p1, span.keys, a.window, a.sinks)) {
                    weigh<PADDED, false>(s, factor, scales, hidden, run, weights);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            if (!seen(column * CACHE_PAGE + 16 * t + j, position[h], span.keys, a.window, a.sinks)) hidden[h] |= 1u << j;
                    weigh<PADDED, true>(s, factor, scales, hidden, run, weights);
                }
            }
            __syncwarp();
            fetch(2 * i + STAGES, st, i / 32);
            if (++st == STAGES) st = 0, parity ^= 1u;
            if (!__all_sync(~0u, mbar_wait(&full[warp][st], parity, &abort_word, P.error, 92))) break;
            if (page >= 0) take_values<PADDED>(ring + st * Shape::HALF, weights, run.y);
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
        for (int h = 0; h < 2; ++h) {
            run.l[h] += __shfl_xor_sync(~0u, run.l[h], 1);
            run.l[h] += __shfl_xor_sync(~0u, run.l[h], 2);
            if (t == 0) figures[warp][0][g + 8 * h] = run.m[h], figures[warp][1][g + 8 * h] = run.top[h], figures[warp][2][g + 8 * h] = run.l[h];
        }
        __syncthreads();
        float *sum = reinterpret_cast<float *>(ring); // ROWS x PADDED, of this warp: as many bytes as a stage
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, figures[w][1][g + 8 * h]);
            const float by = relative(run.top[h], top);
#pragma unroll
            for (int d = 0; d < PADDED / 8; ++d)
                *reinterpret_cast<float2 *>(sum + (g + 8 * h) * PADDED + 8 * d + 2 * t) = make_float2(run.y[d][2 * h] * by, run.y[d][2 * h + 1] * by);
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

template <int PADDED> void attend_few_with(CudaDevice &dev, const ShareParams &P, bool join)
{
    const size_t smem = FewShape<PADDED>::SMEM + 128;
    allow_shared_memory(dev, attend_few_kernel<PADDED>);
    {
        KernelScope ks(dev, "attend_few");
        launch_following(attend_few_kernel<PADDED>, dim3((unsigned)P.blocks), dim3(THREADS), smem, dev.stream(), P);
        dev.count_launch();
    }
    if (!join) return;
    KernelScope ks(dev, "attend_join");
    launch_following(attend_join_kernel<PADDED, ROWS>, dim3((unsigned)std::min(P.blocks * ROWS / 4, 4 * dev.sm_count())), dim3(128), 0, dev.stream(), P);
    dev.count_launch();
}

} // namespace

void launch_attend_few(CudaDevice &dev, const Attend &a)
{
    ShareParams P{};
    P.a = a, P.error = dev.error_word();
    P.least = 0, P.most = ATTEND_FEW, P.slots = (int)slots_of<ROWS>(a);
    const size_t padded = a.cache.padded;
    size_t pages = std::max(a.seq.columns, 1); // of a tile at most
    if (a.window) pages = std::min(pages, ((size_t)a.sinks + 63) / 64 + ((size_t)a.window + ROWS + 62) / CACHE_PAGE + 1);
    const size_t rounds = (pages + WARPS - 1) / WARPS;
    const bool join = rounds > 4;
    P.unit = (int)(join ? WARPS : rounds * WARPS);
    const size_t units = (size_t)P.slots * a.cache.heads * (join ? rounds : 1), places = (size_t)dev.sm_count() * (padded <= 128 ? 2 : 1);
    P.blocks = (int)std::min(units, places);
    struct Parts {
        CudaDevice &dev;
        void *p;
        ~Parts() { dev.release(p); }
    } parts{dev, join ? dev.alloc(2 * (size_t)P.blocks * part_floats<ROWS>((int)padded) * sizeof(float)) : nullptr};
    P.parts = static_cast<float *>(parts.p);
    switch (padded / 32) {
    case 1: return attend_few_with<32>(dev, P, join);
    case 2: return attend_few_with<64>(dev, P, join);
    case 3: return attend_few_with<96>(dev, P, join);
    case 4: return attend_few_with<128>(dev, P, join);
    case 5: return attend_few_with<160>(dev, P, join);
    case 6: return attend_few_with<192>(dev, P, join);
    case 7: return attend_few_with<224>(dev, P, join);
    default: return attend_few_with<256>(dev, P, join);
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
