// cache.hpp -- keys and values of attention as 8-bit codes: pages of 64 tokens, one scale for each page and head.
//
// cache.cu writes tokens into pages, reads them back and lays pages out; attend_few.cu, attend_many.cu and attend_plain.cu compute attention over them.
#pragma once
#include <cstddef>
#include <cstdint>

#include "qmat.hpp"

namespace vqb {

constexpr int CACHE_PAGE = 64;
constexpr size_t CACHE_MOST_WIDTH = 256;
constexpr size_t CACHE_MOST_HEADS = 4096, CACHE_MOST_SEQUENCES = 65535;
constexpr size_t CACHE_MOST_PAGES = (size_t(1) << 31) - 1;
constexpr size_t CACHE_MOST_COLUMNS = (size_t(1) << 25) - 1; // (positions of tokens are 32-bit numbers)

// Of page p and head h: 64 rows of `padded` bytes, a token's key each, and behind them `padded` rows of 64 bytes, a dimension's value in each token.  (Both as
// the tensor cores' operands want them: what is summed over lies side by side.)  A byte is the code + 128 (three instructions make two f16 numbers of two such bytes, four
// of two codes); those of the dimensions behind `width` stand for 0.  Where a key's row is a multiple of 128 bytes, the halves of each 128 of an odd token's change places, so that
// lanes that read the same 64 bytes of two neighbouring tokens find them in different banks.
struct Cache {
    size_t pages = 0, heads = 0, width = 0;
    size_t padded = 0;         // width to the next multiple of 32
    uint8_t *codes = nullptr;  // pages x heads x 2 x 64 x padded
    float *scales = nullptr;   // pages x heads x 2
    static constexpr int ZERO = 0x80; // a byte that stands for 0
    size_t code_bytes() const { return pages * heads * 2 * CACHE_PAGE * padded; }
    size_t scale_bytes() const { return pages * heads * 2 * sizeof(float); }
};

// Which tokens of which pages the rows of a call are.  Sequence b has rows offsets[b] .. offsets[b + 1] - 1 of the n (n / sequences each where offsets is null), and they
// are its last tokens: the last one has position lengths[b] - 1.  Position j is token j % 64 of page table[b][j / 64].  Tokens at negative positions, of columns that the table does
// not have, or of pages that the cache does not have are not there.
struct Sequences {
    const int32_t *table = nullptr; // sequences x table_ld
    size_t table_ld = 0;
    int sequences = 0, columns = 0;
    const int32_t *lengths = nullptr;
    const long long *offsets = nullptr;
    int n = 0, each = 0; // each: n / sequences, where offsets is null
};

// Values of n rows x heads x width, each head's next to each other.
struct HeadRows {
    void *x = nullptr;
    int type = VALUE_F32;
    size_t ld = 0, head_ld = 0; // values from row to row, from head to head
};

void launch_cache_write(CudaDevice &dev, const Cache &c, const Sequences &s, const HeadRows &keys, const HeadRows &values);
void launch_cache_read(CudaDevice &dev, const Cache &c, const Sequences &s, const HeadRows &keys, const HeadRows &values);
// natural: pages x heads x 64 x width, of keys (which = 0) or values (1); scales: pages x heads
void launch_cache_pages_in(CudaDevice &dev, const Cache &c, int which, const int8_t *natural, const float *scales);
void launch_cache_pages_out(CudaDevice &dev, const Cache &c, int which, int8_t *natural, float *scales);

struct Attend {
    Cache cache;
    Sequences seq;
    HeadRows queries, y;
    int group = 1;      // query heads to a key head
    float scale = 1.0f; // of the scores
    int window = 0;     // 0: none
    int sinks = 0;
    bool zero_rest = false; // rows of no sequence become 0
};
// Rows of a sequence are taken together where they have the same cached head: `group` query heads of one token, then those of the next.  A sequence of up to ATTEND_FEW of
// them is taken eight or sixteen at a time, by tensor-core instructions of a warp on pages that the warp fetches for itself (from 17 rows on, every page twice).
// Others are taken 256 or 128 at a time by tcgen05 instructions.  (us by the one and by the other: 16 sequences of up to 8192 tokens with 32 rows each 107 and 167, with 64 rows 203 and 167; 64 of
// up to 1000 with 64 rows 167 and 134.)
constexpr int ATTEND_FEW = 32;
void launch_attend(CudaDevice &dev, const Attend &a);
void launch_attend_few(CudaDevice &dev, const Attend &a);  // sequences of up to ATTEND_FEW rows, and rows of no sequence
void launch_attend_many(CudaDevice &dev, const Attend &a); // the other sequences
void launch_attend_plain(CudaDevice &dev, const Attend &a); // CUDA cores

} // namespace vqb
