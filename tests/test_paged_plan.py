"""CPU: which rows, pages and blocks of tokens a call over the paged cache touches (csrc/paged.h), against counting token by token."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <climits>
#include <cstdio>
#include <set>
#include "paged.h"
using namespace b200fc;
static int bad;
#define EXPECT(ok, ...) do { if (!(ok) && bad++ < 20) std::printf(__VA_ARGS__); } while (0)
int main() {
    const int windows[] = {0, 1, 2, 7, 16, 33, 64, 1000, INT_MAX}, sinks[] = {0, 1, 5, 16, 17, 70, INT_MAX};
    for (int shift = 4; shift <= 7; shift += 3)
        for (int w : windows)
            for (int sk : sinks)
                for (int lo = 0; lo < 300; lo += 13)
                    for (int n : {1, 2, 40, 150}) {
                        const int hi = lo + n - 1;
                        std::set<int> want, got;
                        for (int p = lo; p <= hi; p++)
                            for (int j = 0; j <= p; j++)
                                if (j <= p && (w == 0 || (long long)j > (long long)p - w || j < sk)) {
                                    want.insert(j >> shift);
                                    EXPECT(key_visible(j, p, w, sk), "visible %d %d %d %d\n", j, p, w, sk);
                                } else {
                                    EXPECT(!key_visible(j, p, w, sk), "invisible %d %d %d %d\n", j, p, w, sk);
                                }
                        const KeyBlocks k = key_blocks(lo, hi, w, sk, shift);
                        int last = -1;
                        for (int i = 0; i < k.count; i++) {
                            const int b = key_block(k, i);
                            EXPECT(b > last, "blocks out of order\n");
                            last = b;
                            got.insert(b);
                        }
                        for (int b : want) EXPECT(got.count(b), "block %d missing: places %d..%d window %d sinks %d\n", b, lo, hi, w, sk);
                        // nothing else, but blocks between the sinks and the window of the lowest place, which later places may leave behind
                        for (int b : got) EXPECT(want.count(b), "block %d not needed: places %d..%d window %d sinks %d\n", b, lo, hi, w, sk);
                        EXPECT(k.end == hi + 1 && k.begin >= 0 && k.sink_end >= 0 && k.sink_end <= k.begin, "ranges\n");
                    }
    EXPECT(key_blocks(-5, -1, 0, 0, 4).count == 0, "rows without tokens\n");
    EXPECT(key_blocks(-5, 3, 2, 1, 4).count == 1, "rows of which some have tokens\n");
    EXPECT(key_blocks(kMaxTokens - 1, kMaxTokens - 1, 0, 0, 7).count == kMaxTokens / 128, "the longest sequence\n");
    EXPECT(key_blocks(kMaxTokens - 1, kMaxTokens - 1, INT_MAX, INT_MAX, 7).count == kMaxTokens / 128, "the longest sequence, everything in the window\n");
    SeqRows s;
    const int ints[] = {INT_MIN, -1, 0, 1, 5, 16, 17, 100, INT_MAX};
    for (int r0 : ints)
        for (int r1 : ints)
            for (int len : ints)
                for (long long cap : {0LL, 16LL, 1LL << 34}) {
                    const bool ok = seq_rows(r0, r1, len, 17, 16, cap, &s);
                    const bool want = r0 >= 0 && r1 >= r0 && r1 <= 17 && (long long)r1 - r0 <= 16 && len >= 0 && len <= cap && len <= kMaxTokens;
                    EXPECT(ok == want, "rows %d..%d len %d cap %lld: %d\n", r0, r1, len, cap, ok);
                    EXPECT(ok || (s.rows == 0 && s.len == 0), "rows of a refused sequence\n");
                }
    for (int rows = 0; rows < 70; rows++)
        for (int len = 0; len < 140; len++) {
            seq_rows(3, 3 + rows, len, 200, 200, 1 << 20, &s);
            std::set<int> pages;
            for (int r = 0; r < rows; r++)
                if (len - rows + r >= 0) pages.insert((len - rows + r) >> 4);
            EXPECT(touched_pages(s, 4) == (int)pages.size(), "pages of %d rows, %d tokens\n", rows, len);
            EXPECT(touched_pages(s, 4) <= rows && touched_pages(s, 4) <= rows / 16 + 2, "the launch's bound\n");
        }
    return bad != 0;
}
"""


def test_rows_pages_and_blocks(tmp_path):
    src, exe = tmp_path / "paged.cpp", str(tmp_path / "paged")
    src.write_text(PROGRAM)
    subprocess.check_call(["/usr/bin/g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I" + os.path.join(ROOT, "mm_amx_b200", "csrc"),
                           str(src), "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
