// Which rows, tokens and blocks of tokens a call over the paged cache deals with.  Plain C++ besides the kernels' use of it.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define B200FC_HD __host__ __device__ __forceinline__
#else
#define B200FC_HD inline
#endif

namespace b200fc {

constexpr int kMaxTokens = 0x7fffff00;     // of a sequence: sums with a block size stay in 32 bits

// Rows [row0, row0 + rows) of a sequence with `len` tokens; row r stands at place len - rows + (r - row0).
struct SeqRows { int row0, rows, len; };
// false (and no rows): the numbers lie outside their buffers
B200FC_HD bool seq_rows(int r0, int r1, int len, int T, int max_rows, long long capacity, SeqRows* s) {
    const bool ok = r0 >= 0 && r0 <= r1 && r1 <= T && r1 - r0 <= max_rows && len >= 0 && len <= kMaxTokens && (long long)len <= capacity;
    *s = ok ? SeqRows{r0, r1 - r0, len} : SeqRows{0, 0, 0};
    return ok;
}
B200FC_HD int first_token(const SeqRows& s) { return s.len > s.rows ? s.len - s.rows : 0; }      // the first that a row stands for
B200FC_HD int touched_pages(const SeqRows& s, int page_shift) {
    const int first = first_token(s);
    return s.rows > 0 && first < s.len ? ((s.len - 1) >> page_shift) - (first >> page_shift) + 1 : 0;
}

B200FC_HD bool key_visible(int j, int p, int window, int sinks) { return j <= p && (window == 0 || j > p - window || j < sinks); }

// The blocks of 1 << shift tokens that hold what rows at places [p_lo, p_hi] see: tokens [0, sink_end) and [begin, end), as blocks [0, sink_blocks) and
// [first, ...), `count` in all.
struct KeyBlocks { int sink_end, begin, end, sink_blocks, first, count; };
B200FC_HD KeyBlocks key_blocks(int p_lo, int p_hi, int window, int sinks, int shift) {
    KeyBlocks k;
    k.end = p_hi + 1;
    if (k.end <= 0) return KeyBlocks{0, 0, 0, 0, 0, 0};
    k.begin = window > 0 && p_lo >= window ? p_lo - window + 1 : 0;
    k.sink_end = sinks < k.begin ? sinks : k.begin;
    k.sink_blocks = (k.sink_end + (1 << shift) - 1) >> shift;
    k.first = k.begin >> shift;
    if (k.sink_blocks >= k.first) k.sink_blocks = k.first = 0;        // one run
    k.count = ((k.end + (1 << shift) - 1) >> shift) - k.first + k.sink_blocks;
    return k;
}
B200FC_HD int key_block(const KeyBlocks& k, int i) { return i < k.sink_blocks ? i : i - k.sink_blocks + k.first; }

}  // namespace b200fc
