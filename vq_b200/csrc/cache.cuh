// cache.cuh -- what the kernels on a cache's pages share.
#pragma once
#include "cache.hpp"
#include "qmat.cuh"

namespace vqb {

// All earlier work of the stream is complete and visible from here on.  Every thread calls it before it touches global memory or leaves.
__device__ __forceinline__ void cache_is_there() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ int offset_of(const Sequences &s, int b)
{
    if (!s.offsets) return s.each * b;
    const long long o = s.offsets[b];
    return (int)(o < 0 ? 0 : o > s.n ? s.n : o);
}

struct Span {
    int row, count; // first row, rows
    int first;      // position of the first row's token
    int keys;       // tokens of the sequence that the table has columns for
    __device__ __forceinline__ Span(const Sequences &s, int b)
    {
        row = offset_of(s, b);
        const int end = offset_of(s, b + 1), length = max(s.lengths[b], 0);
        count = max(end - row, 0);
        first = length - count;
        keys = (int)min((long long)length, (long long)s.columns * CACHE_PAGE);
    }
};

// The last sequence b with offset / per + extra * b <= u, by a whole warp (32 at a time).  So many pieces of `per` rows, `extra` more for each sequence, are enough
// for all sequences whatever their rows: a sequence's pieces are numbered from offset / per + extra * b on.
__device__ __forceinline__ int sequence_of(const Sequences &s, int u, int per, int extra)
{
    const int lane = threadIdx.x & 31;
    int low = 0, many = s.sequences;
    while (many > 1) {
        const int step = (many + 31) / 32, b = low + lane * step;
        const bool begun = lane * step < many && offset_of(s, b) / per + extra * b <= u;
        const int k = max(__popc(__ballot_sync(~0u, begun)) - 1, 0);
        low += k * step;
        many = min(step, many - k * step);
    }
    return low;
}
__device__ __forceinline__ int floor_page(int position) { return position >> 6; } // (also of negative positions)
static_assert(CACHE_PAGE == 64, "");

// The page of a column, -1 where there is none.
__device__ __forceinline__ int page_of(const Sequences &s, size_t pages, int b, int column)
{
    if (column < 0 || column >= s.columns) return -1;
    const int p = s.table[b * s.table_ld + column];
    return p < 0 || (size_t)p >= pages ? -1 : p;
}

// Where byte d of token t's key is in its page's keys.
__device__ __forceinline__ int key_at(int padded, int t, int d) { return t * padded + (padded % 128 == 0 ? d ^ ((t & 1) * 64) : d); }

__device__ __forceinline__ float value_at(const HeadRows &r, size_t at)
{
    if (r.type == VALUE_F32) return static_cast<const float *>(r.x)[at];
    if (r.type == VALUE_F16) return __half2float(static_cast<const __half *>(r.x)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(r.x)[at]);
}
__device__ __forceinline__ void put_value(const HeadRows &r, size_t at, float v)
{
    if (r.type == VALUE_F32) static_cast<float *>(r.x)[at] = v;
    else if (r.type == VALUE_F16) static_cast<__half *>(r.x)[at] = from_float<__half>(v);
    else static_cast<__nv_bfloat16 *>(r.x)[at] = from_float<__nv_bfloat16>(v);
}

} // namespace vqb
