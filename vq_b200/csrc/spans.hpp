// spans.hpp -- how far the caller's rows reach in memory, from the distances that it gives.
#pragma once
#include <cstddef>

namespace vqb {

// Values: more than any memory has, and few enough that twice as many, in bytes, are a number of 64 bits.
constexpr size_t MOST_SPAN = size_t(1) << 58;

// Whether `many` things, `step` values from each to the next, reach further than that.
constexpr bool too_far(size_t many, size_t step) { return many > 1 && step > MOST_SPAN / (many - 1); }

// What is wrong with the distances of n rows of heads, null where nothing is: neither rows nor heads overlap, whichever of the two is the outer one.
inline const char *heads_fault(size_t n, size_t heads, size_t width, size_t ld, size_t head_ld)
{
    if (too_far(n, ld) || too_far(heads, head_ld)) return "rows are too far apart";
    const bool heads_inside = (heads == 1 || head_ld >= width) && (n == 1 || ld >= (heads - 1) * head_ld + width);
    const bool rows_inside = (n == 1 || ld >= width) && (heads == 1 || head_ld >= (n - 1) * ld + width);
    return heads_inside || rows_inside ? nullptr : "rows or heads overlap";
}

// Values from the first one to the last one (of distances that have no fault).
constexpr size_t heads_values(size_t n, size_t heads, size_t width, size_t ld, size_t head_ld) { return n ? (n - 1) * ld + (heads - 1) * head_ld + width : 0; }

} // namespace vqb
