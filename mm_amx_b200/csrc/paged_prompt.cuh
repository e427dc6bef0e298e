// Paged attention for more than 16 packed rows (query rows x heads of a group) per sequence and kv head: prompts, chunks of prompts, longer drafts.
// On the tensor cores (tcgen05), bound by them and by the exponentials beside them.
//
// A CTA takes 256 packed rows of one (sequence, kv head), as two tiles of 128 rows, over all 128-token blocks that they see, or over a share of those
// where the call has too few tiles for the GPU.  Packing the heads of a group into the rows keeps K and V of a block in shared memory for all of them.
// With heads of 64 in bf16 a CTA takes one tile, and an SM two CTAs: what a CTA does before its first block and after its last (7 us) then runs under the
// other's blocks, and the last tiles are shorter (6000 rows, window 1000, 16 heads: 94 us with two tiles, 83 with one; 2 x up to 2048 rows, 4096 tokens, 16
// heads: 78 / 60).  Heads of 128 have room for that only with a ring of
// 64-token slots (3 sequences of up to 2048 rows: 246 us, and 200 without any loads, where two tiles then took 182).  With 8 bits every CTA widens its blocks itself, so two
// CTAs would widen each block twice; that form was not built.
//   warps 0-3, 4-7   softmax of tile 0, 1: a thread has one row.  S comes from tensor memory 64 tokens at a time, exp2(S - max) goes back over it as bf16.  The
//                    maximum that is subtracted follows the true one only when that is 2^8 ahead, so that O in tensor memory is rescaled hardly ever (the
//                    probabilities' rounding is relative; sums of p v are fp32 and reach 2^8 * tokens * |v|, which bounds v.  A smaller scale would end that
//                    bound, but lose probabilities near 2^-126, which sharply peaked rows with zeros in v at their peak show).
//   2, 4 or 8 more   fetch K and V blocks into a ring of 128-token slots (128-byte swizzle): bf16 by TMA, or in blocks that not every row sees by cp.async with zeros
//                    for tokens that nobody sees (which may hold anything), 8 bits widened on the way to bf16 of (value / 64), exactly; the page's factors go to the softmax.
//   one a tile       issues its products: S_w = Q_w K^T (Q, K in shared memory), O_w += P_w V (P in tensor memory, V as it lies: N-major).  One
//                    tile's products run under the other tile's softmax.  (One warp for both tiles was the bottleneck: 3900 clocks a block.)
// Tensor memory: S_0 S_1 (128 columns each; P over the first half of either 64) O_0 O_1 (D columns each).
// A value that is no number in a block that some rows do not see would reach them as 0 * NaN: the fetching warps look for one in such blocks, and a CTA that
// met one does its rows again one by one (row_state).
#pragma once
#include "paged_common.cuh"

namespace b200fc {

namespace {

constexpr int PR_BLOCK = 128;                      // tokens of a block
constexpr int PR_FIND_BYTES = 1024;
constexpr int PR_META = 8;                         // blocks whose facts are kept; more than the ring holds

// Warps and registers.  8 bits are widened by eight warps (with four they were the bottleneck: 185 us where this takes 155), bf16 needs two a tile.  The last
// warps only fill their group of four.  (bf16, one tile: with 152 and 104 registers some are spilled, 90 us where this takes 83.)
template <int D, bool S8> struct PromptShape {
    static constexpr int TILES = D == 64 && !S8 ? 1 : 2, ROWS = 128 * TILES, CTAS = 3 - TILES;      // CTAs: per SM
    static constexpr int LOADER = 4 * TILES, MMA = LOADER + (S8 ? 8 : 2 * TILES), THREADS = (MMA + 2 * TILES) * 32;      // first of the warps that fetch, that multiply
    static constexpr int REGS = S8 ? 96 : 128, REGS_SOFTMAX = S8 ? 152 : 160, REGS_OTHER = S8 ? 56 : 96;      // a thread, at launch and in the roles
    static constexpr int COLUMNS = 256 * TILES, O_AT = 128 * TILES;                                 // of tensor memory
    static_assert(REGS_SOFTMAX * LOADER * 32 + REGS_OTHER * (THREADS - LOADER * 32) <= REGS * THREADS && REGS * THREADS * CTAS <= 65536,
                  "the split must not ask for more than the launch has");
    static_assert(LOADER % 4 == 0 && (THREADS / 32) % 4 == 0, "registers are split between groups of four warps");
};

template <int D, bool S8> struct PromptSmem {
    static constexpr int TILES = PromptShape<D, S8>::TILES;
    static constexpr int HALF = PR_BLOCK * 128;                       // 128 rows of 64 components
    static constexpr int TILE = HALF * (D / 64);                      // a tile of Q, a block of K or V
    static constexpr int SLOTS = D == 128 || TILES == 1 ? 5 : 8;
    static constexpr int AHEAD = 2;                                   // fills by cp.async whose arrival is waited for later
    static constexpr int RING = TILES * TILE, BARS = RING + SLOTS * TILE;
    static constexpr int META = BARS + 384;
    static constexpr int FIND = META + PR_META * 80;                  // for the search for the tile
    static constexpr int BYTES = FIND + PR_FIND_BYTES;
    static_assert(PromptShape<D, S8>::CTAS * (BYTES + 1024) <= 233472, "shared memory of the CTAs of an SM (1 KB of each is the system's)");
    static_assert(BYTES % 1024 == 0 || PromptShape<D, S8>::CTAS == 1, "the swizzle goes by addresses: each CTA begins at a multiple of 1024");
};
// Of a block: its first token; granules of 16 tokens that lie in no page of the pool (bits 0-7), whether tile w sees any of it (bit 8 + w) and all rows of the
// tile all of half h (bit 16 + 2 w + h); factors times 64.  Worked out once, by the warps that fetch it.
struct PromptMeta { int tok0; unsigned facts; float k[8], v[8]; float pad[2]; };
static_assert(sizeof(PromptMeta) == 80, "");

struct PromptParams {
    PagedAttn a;                  // (scale_log2e: its absolute value, not zero)
    unsigned group_inverse;       // ceil(2^32 / G)
    unsigned flip;                // sign bits of two bf16: the scale's sign, carried by Q
    int splits;                   // CTAs that share a tile's blocks at most
    float* ws_o;                  // [CTA][ROWS][D]
    float* ws_ml;                 // [CTA][ROWS][2]
    int tma;                      // the tensor maps are there
    unsigned long long wait_limit_ns;
};

// operand of which the rows (K dimension, 128 bytes of 64 components each, 128-byte swizzle) lie one behind another: N-major; HALF bytes between 64 components
__device__ __forceinline__ unsigned long long make_smem_desc_nmajor(unsigned smem_addr, unsigned half) {
    unsigned long long d = 0;
    d |= (unsigned long long)((smem_addr & 0x3FFFFu) >> 4);
    d |= (unsigned long long)(half >> 4) << 16;
    d |= (unsigned long long)(1024 >> 4) << 32;
    d |= (unsigned long long)1 << 46;
    d |= (unsigned long long)2 << 61;
    return d;
}
// instruction descriptor of a 128-row bf16 product with fp32 sums, B K-major or N-major
__device__ __forceinline__ unsigned make_idesc_bf16(int columns, bool b_nmajor) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (b_nmajor ? 1u << 16 : 0u) | (unsigned)(columns >> 3) << 17 | (unsigned)(BM >> 4) << 24;
}
__device__ __forceinline__ void tc_st16(unsigned taddr, const unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(unsigned dst, const CUtensorMap* map, unsigned bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// the lowest n bits, none or all of them beyond 0 .. 32
__device__ __forceinline__ unsigned first_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// n / G for n < 2^31: the product with ceil(2^32 / G) is at most one too large
__device__ __forceinline__ int over_group(const PromptParams& p, int n) {
    if (p.a.G == 1) return n;
    const int q = (int)__umulhi((unsigned)n, p.group_inverse);
    return q - (q * p.a.G > n);
}

// A CTA's work: a tile of a (sequence, kv head) and a share of its blocks.
struct PromptItem {
    int b, hk, row0;              // row0: first packed row
    SeqRows s;
    KeyBlocks kb;                 // of all its rows, 128 tokens a block
    int rows;                     // packed rows of the tile
    int splits, n0, n1;           // shares of the blocks, this one's
};
__device__ __forceinline__ int prompt_splits(int count, int splits) { return max(1, min(splits, count >> 1)); }
// item-th tile: of each sequence the last rows first (they see most), and of up to PR_RANKED sequences those whose last tile sees most first, so that no long
// tile is left for the end (3 sequences of up to 2048 rows and 4096 tokens: 209 us in the order given, 193 so).  By all threads of a block.
constexpr int PR_RANKED = 64;
struct FindSpace {
    PromptItem item;
    int warp_sum[PromptShape<128, true>::THREADS / 32], keys[PR_RANKED], order[PR_RANKED];
};
static_assert(sizeof(FindSpace) <= PR_FIND_BYTES, "");
template <int ROWS, int THREADS>
__device__ __forceinline__ bool find_prompt_item(const PagedAttn& a, int item, int split, int splits, bool report, PromptItem* it, FindSpace* space) {
    PromptItem* shared = &space->item;
    int *warp_sum = space->warp_sum, *keys = space->keys, *order = space->order;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto sequence = [&](int b, SeqRows* s, int* tiles) {
        *s = SeqRows{0, 0, 0};
        const bool ok = load_seq(a.c, b, s);
        *tiles = (s->rows * a.G + ROWS - 1) / ROWS;
        return ok;
    };
    auto found = [&](int b, const SeqRows& s, int tiles, int at) {
        const int rt = tiles - 1 - at / a.c.Hkv, first = s.len - s.rows;
        PromptItem x;
        x.b = b; x.hk = at % a.c.Hkv; x.row0 = rt * ROWS; x.s = s;
        x.rows = min(ROWS, s.rows * a.G - x.row0);
        x.kb = key_blocks(max(first + x.row0 / a.G, 0), first + (x.row0 + x.rows - 1) / a.G, a.window, a.sinks, 7);
        x.splits = prompt_splits(x.kb.count, splits);
        x.n0 = split < x.splits ? (int)((long long)x.kb.count * split / x.splits) : 0;
        x.n1 = split < x.splits ? (int)((long long)x.kb.count * (split + 1) / x.splits) : 0;
        *shared = x;
    };
    if (threadIdx.x == 0) shared->b = -1;
    if (a.c.B <= PR_RANKED) {
        const int b = threadIdx.x;
        SeqRows s;
        int tiles = 0, key = 0, n = 0;
        if (b < a.c.B) {
            if (!sequence(b, &s, &tiles) && report) report_paged(a.c);
            n = tiles * a.c.Hkv;
            const KeyBlocks kb = key_blocks(max(s.len - 1 - (ROWS - 1) / a.G, 0), s.len - 1, a.window, a.sinks, 7);
            key = n ? kb.count : -1;
            keys[b] = key;
        }
        __syncthreads();
        if (b < a.c.B) {
            int rank = 0;
            for (int o = 0; o < a.c.B; o++) rank += keys[o] > key || (keys[o] == key && o < b);
            order[rank] = n;
            n = rank;                                        // (from here on the sequence's place in the order)
        }
        __syncthreads();
        if (b < a.c.B && tiles) {
            long long before = 0;
            for (int o = 0; o < n; o++) before += order[o];
            if (item >= before && item < before + tiles * a.c.Hkv) found(b, s, tiles, (int)(item - before));
        }
        __syncthreads();
    } else {
        long long seen = 0;
        for (int b0 = 0; b0 < a.c.B && (seen <= item || report); b0 += THREADS) {      // (who reports looks at all of them)
            const int b = b0 + threadIdx.x;
            SeqRows s;
            int tiles = 0;
            if (b < a.c.B && !sequence(b, &s, &tiles) && report) report_paged(a.c);
            const int n = tiles * a.c.Hkv;
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += u;
            }
            __syncthreads();
            if (lane == 31) warp_sum[warp] = upto;
            __syncthreads();
            long long before = 0, all = 0;
#pragma unroll
            for (int w = 0; w < THREADS / 32; w++) { before += w < warp ? warp_sum[w] : 0; all += warp_sum[w]; }
            const long long lo = seen + before + upto - n;
            if (item >= lo && item < lo + n) found(b, s, tiles, (int)(item - lo));
            seen += all;
        }
        __syncthreads();
    }
    const bool hit = shared->b >= 0;
    if (hit) *it = *shared;
    return hit;
}

template <int D, bool S8>
__global__ void __launch_bounds__(PromptShape<D, S8>::THREADS, PromptShape<D, S8>::CTAS) paged_prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PromptParams p) {
    using SM = PromptSmem<D, S8>;
    using SH = PromptShape<D, S8>;
    constexpr int SLOTS = SM::SLOTS, HALF = SM::HALF, PR_ROWS = SH::ROWS, PR_LOADER = SH::LOADER, PR_MMA = SH::MMA, PR_THREADS = SH::THREADS;
    // no static shared memory: the dynamic part then begins at a multiple of 1024, as the swizzle wants it
    extern __shared__ __align__(1024) unsigned char smem[];
    int& odd_value = *(int*)(smem + SM::BARS + 368);
    int& abort_flag_word = *(int*)(smem + SM::BARS + 372);
    unsigned& tmem_holder = *(unsigned*)(smem + SM::BARS + 376);
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) atomicExch(p.a.c.status, 4);
        return;
    }
    unsigned char* ring = smem + SM::RING;
    const unsigned bars = smem_u32(smem + SM::BARS);
    const unsigned bar_full = bars, bar_empty = bars + 8 * SLOTS, bar_s = bar_empty + 8 * SLOTS, bar_p = bar_s + 32, bar_v = bar_p + 32, bar_o = bar_v + 16, bar_q = bar_o + 16, bar_turn = bar_q + 16;   // bar_s, bar_p: [half of the block][tile]
    volatile PromptMeta* meta = (volatile PromptMeta*)(smem + SM::META);
    volatile int* abort_flag = &abort_flag_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PagedAttn& a = p.a;
    const unsigned long long limit = p.wait_limit_ns;

    if (threadIdx.x == 0) {
        for (int i = 0; i < SLOTS; i++) { mbar_init(bar_full + 8 * i, PR_MMA - PR_LOADER); mbar_init(bar_empty + 8 * i, SH::TILES); }
        for (int w = 0; w < 2; w++) {
            mbar_init(bar_s + 8 * w, 1); mbar_init(bar_s + 16 + 8 * w, 1);
            mbar_init(bar_p + 8 * w, 4); mbar_init(bar_p + 16 + 8 * w, 4);
            mbar_init(bar_v + 8 * w, 1); mbar_init(bar_o + 8 * w, 1); mbar_init(bar_q + 8 * w, 4); mbar_init(bar_turn + 8 * w, 4);
        }
        abort_flag_word = 0;
        odd_value = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == PR_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_holder)), "r"((unsigned)SH::COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    PromptItem it;
    const bool has_item = find_prompt_item<PR_ROWS, PR_THREADS>(a, (int)(blockIdx.x / p.splits), (int)(blockIdx.x % p.splits), p.splits, blockIdx.x == 0, &it, (FindSpace*)(smem + SM::FIND));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = tmem_holder;
    const int tiles = has_item ? (it.rows > 128 ? 2 : 1) : 0, n = has_item ? it.n1 - it.n0 : 0;
    const bool split = has_item && it.splits > 1;
    const bool work = has_item && (n > 0 || (it.kb.count == 0 && blockIdx.x % p.splits == 0));
    // places of a tile's first and last row, and which blocks it sees any of
    const int first_place = has_item ? it.s.len - it.s.rows : 0;
    auto place_lo = [&](int w) { return max(first_place + over_group(p, it.row0 + 128 * w), 0); };      // (rows in front of the first token see nothing)
    auto place_hi = [&](int w) { return first_place + over_group(p, it.row0 + min(128 * w + 127, it.rows - 1)); };
    auto block_token = [&](int j) { return key_block(it.kb, it.n0 + j) << 7; };

    if (warp < PR_LOADER) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SH::REGS_SOFTMAX));
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SH::REGS_OTHER));
    }
    // (each role ends by itself: behind the branches the roles' numbers of registers would differ)
    auto all_done = [] { asm volatile("bar.sync 1, %0;" ::"n"(PR_THREADS) : "memory"); };
    if (warp < PR_LOADER) {
        if (!work) { all_done(); return; }
        const int w = warp >> 2, tid = threadIdx.x & 127;
        if (w < tiles) {
            // ---- Q tile: rows of 64 components, 128-byte swizzle; zeros behind the last row ----
            constexpr int CH = D / 8, AT_ONCE = 128 / CH;
            const int r0 = tid / CH, ch = tid % CH;
            unsigned char* qt = smem + w * SM::TILE + (ch >> 3) * HALF;
#pragma unroll
            for (int k = 0; k < CH; k++) {
                const int r = k * AT_ONCE + r0, i = it.row0 + 128 * w + r, row = over_group(p, i);
                const bool ok = 128 * w + r < it.rows;
                cp_async16_or_zero(smem_u32(qt + r * 128 + (((ch & 7) ^ (r & 7)) << 4)),
                                   ok ? a.q + (long long)(it.s.row0 + row) * a.q_rs + (long long)(it.hk * a.G + i - row * a.G) * a.q_hs + ch * 16 : a.q, ok);
            }
            cp_async_commit();
            cp_async_wait<0>();
            if (p.flip) {
                for (int k = 0; k < CH; k++) {
                    const int r = k * AT_ONCE + r0;
                    uint4* x = (uint4*)(qt + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                    *x = make_uint4(x->x ^ p.flip, x->y ^ p.flip, x->z ^ p.flip, x->w ^ p.flip);
                }
            }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_q + 8 * w);

        // ---- softmax: a row per thread, 64 tokens at a time ----
        const int i = 128 * w + tid;
        const bool mine = w < tiles && i < it.rows;
        const int packed = it.row0 + i, row = over_group(p, packed), place = first_place + row;
        const unsigned lanes = (unsigned)(warp & 3) << 21;              // lane quarter of tensor memory
        const unsigned to = tmem + SH::O_AT + w * D + lanes;
        const float c = a.scale_log2e;
        float m_used = -INFINITY, l = 0.0f;
        unsigned phase = 0, v_phase = 1;                                // v_phase: of the products with V that have been asked for
        bool alive = true, any = false;
        auto wait = [&](unsigned bar, unsigned parity) {
            if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) alive = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, limit));
        };
        // Heads of 128: the two tiles begin their exponentials in turns (tile 0, tile 1, tile 0, ...); side by side, the unit that computes them would be busy
        // while both need it and idle while both do the rest (3 sequences of up to 2048 rows: 194.4 us without, 185.4 with, medians of runs in turn; 512 rows over 30000 tokens
        // 309 / 290; with turns that are passed on at the end a quarter of that is left).  One turn for each half of a block, seen or not.  Not for 8 bits, whose
        // widening takes as long: no difference.
        constexpr bool TURNS = D == 128 && !S8;
        unsigned turn_phase = w == 1 ? 0 : 1;
        auto take_turn = [&] {
            if (TURNS && tiles == 2) wait(bar_turn + 8 * w, turn_phase);
            turn_phase ^= 1;
        };
        auto pass_turn = [&] {
            if (TURNS && tiles == 2) {
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_turn + 8 * (1 - w));
            }
        };
        for (int j = 0; j < n && w < tiles && alive; j++) {
            const volatile PromptMeta& mt = meta[j % PR_META];
#pragma unroll 1
            for (int h = 0; h < 2; h++) {
                const unsigned bp = bar_p + 16 * h + 8 * w, ts = tmem + w * 128 + 64 * h + lanes;
                wait(bar_s + 16 * h + 8 * w, phase);
                if (!alive) break;
                tc_fence_after();
                const unsigned facts = mt.facts;
                if (!(facts & 256u << w)) {
                    if (lane == 0) mbar_arrive(bp);
                    take_turn();
                    if (!alive) break;
                    pass_turn();
                    continue;
                }
                unsigned xa[32], xb[32];
                tc_ld32(ts, xa);
                tc_ld32(ts + 32, xb);
                const bool whole = facts & 65536u << (2 * w + h);
                // bit e of seen[q]: token tok0 + 64 h + 32 q + e is seen
                unsigned seen[2] = {0xffffffffu, 0xffffffffu};
                if (!whole) {
                    const int at = mt.tok0 + 64 * h, to_hi = place - at, from = a.window ? place - a.window - at : -1, sink = a.sinks > at ? a.sinks - at : 0;
                    const unsigned bad = facts >> (4 * h);
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        seen[q] = first_bits(to_hi + 1 - 32 * q) & (~first_bits(from + 1 - 32 * q) | first_bits(sink - 32 * q));
                        seen[q] &= ((bad >> (2 * q)) & 1 ? 0u : 0x0000ffffu) | ((bad >> (2 * q + 1)) & 1 ? 0u : 0xffff0000u);
                    }
                }
                tc_wait_ld();
                // ---- the largest score ----
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                auto largest = [&](unsigned (&x)[32], int q) {
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (!(seen[q] & (1u << e))) x[e] = 0xff800000u;
                    }
                    if constexpr (S8) {
#pragma unroll
                        for (int g = 0; g < 2; g++) {               // (factors are not negative; none seen stays -inf beside a factor of 0)
                            float t0 = max3(__uint_as_float(x[16 * g]), __uint_as_float(x[16 * g + 1]), __uint_as_float(x[16 * g + 2]));
                            float t1 = max3(__uint_as_float(x[16 * g + 3]), __uint_as_float(x[16 * g + 4]), __uint_as_float(x[16 * g + 5]));
#pragma unroll
                            for (int e = 6; e < 16; e += 4) {
                                t0 = max3(t0, __uint_as_float(x[16 * g + e]), __uint_as_float(x[16 * g + e + 1]));
                                if (e + 2 < 16) t1 = max3(t1, __uint_as_float(x[16 * g + e + 2]), __uint_as_float(x[16 * g + e + 3]));
                            }
                            t0 = max3(t0, t1, t1);
                            top[2 * q + g] = t0 == -INFINITY ? t0 : t0 * mt.k[4 * h + 2 * q + g];
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
#pragma unroll
                            for (int u = 0; u < 4; u++) top[u] = max3(top[u], __uint_as_float(x[e + 2 * u]), __uint_as_float(x[e + 2 * u + 1]));
                    }
                };
                largest(xa, 0);
                largest(xb, 1);
                const float m_new = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * c;      // (c > 0)
                const bool far = m_new > m_used + 8.0f;
                if (__any_sync(0xffffffffu, far)) {
                    float f = 1.0f;
                    if (far) { f = exp2_approx(m_used - m_new); m_used = m_new; }
                    l *= f;
                    if (any) {
                        wait(bar_v + 8 * w, v_phase);              // every product into O that has been asked for
                        if (!alive) break;
                        tc_fence_after();
#pragma unroll
                        for (int q = 0; q < D / 16; q++) {
                            unsigned y[16];
                            tc_ld16(to + 16 * q, y);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) y[e] = __float_as_uint(__uint_as_float(y[e]) * f);
                            tc_st16(to + 16 * q, y);
                        }
                    }
                }
                any = true;
                v_phase ^= 1;
                const float shift = m_used == -INFINITY ? 0.0f : -m_used;
                const f32x2 c2 = pack2(c, c), s2 = pack2(shift, shift);
                f32x2 sum[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
                // ---- probabilities of 32 columns, over columns of S that have been read ----
                auto weigh = [&](const unsigned (&x)[32], int q, auto all) {
                    constexpr bool ALL = decltype(all)::value != 0;
                    unsigned pk[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        f32x2 f2 = c2;
                        if constexpr (S8) {
                            const float f = mt.k[4 * h + 2 * q + (e >> 4)] * c;
                            f2 = pack2(f, f);
                        }
                        float y0, y1;
                        unpack2(fma2(pack2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f2, s2), y0, y1);
                        y0 = exp2_approx(y0); y1 = exp2_approx(y1);
                        if (!ALL) {
                            if (!(seen[q] & (1u << e))) y0 = 0.0f;
                            if (!(seen[q] & (2u << e))) y1 = 0.0f;
                        }
                        sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pack2(y0, y1));
                        if constexpr (S8) {
                            const float f = mt.v[4 * h + 2 * q + (e >> 4)];
                            unpack2(mul2(pack2(y0, y1), pack2(f, f)), y0, y1);
                            if (!ALL) {                              // (a masked token has no part in its page's factor, which may be NaN)
                                if (!(seen[q] & (1u << e))) y0 = 0.0f;
                                if (!(seen[q] & (2u << e))) y1 = 0.0f;
                            }
                        }
                        pk[e >> 1] = pack_bf16x2(y0, y1);
                    }
                    tc_st16(ts + 16 * q, pk);
                };
                take_turn();
                if (!alive) break;
                if (whole) {
                    weigh(xa, 0, IntConst<1>());
                    pass_turn();
                    weigh(xb, 1, IntConst<1>());
                } else {
                    weigh(xa, 0, IntConst<0>());
                    pass_turn();
                    weigh(xb, 1, IntConst<0>());
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bp);
                float a0, a1, b0, b1;
                unpack2(sum[0], a0, a1); unpack2(sum[1], b0, b1);
                l += (a0 + a1) + (b0 + b1);
            }
            phase ^= 1;
        }
        // ---- O ----
        if (any && alive) wait(bar_o + 8 * w, 0);
        tc_fence_after();
        if (alive && w < tiles && !*(volatile int*)&odd_value) {
            const float inv = split ? 1.0f : (l != 0.0f ? 1.0f / l : 0.0f);
            float* wo = p.ws_o + ((size_t)blockIdx.x * PR_ROWS + i) * D;
            // rows leave by way of the warp's quarter of the Q tile (all products with it are complete), so that they are stored in whole
            constexpr int CH = D / 8, AT_ONCE = 32 / CH;
            unsigned char* own = smem + w * SM::TILE + (warp & 3) * 32 * D * 2;
#pragma unroll
            for (int q = 0; q < D / 32; q++) {
                unsigned y[32];
                if (any) {
                    tc_ld32(to + 32 * q, y);
                    tc_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) y[e] = 0;
                }
                if (split) {
                    if (mine)
#pragma unroll
                        for (int e = 0; e < 32; e += 4) *(uint4*)(wo + 32 * q + e) = make_uint4(y[e], y[e + 1], y[e + 2], y[e + 3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        unsigned o[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) o[u] = pack_bf16x2(__uint_as_float(y[e + 2 * u]) * inv, __uint_as_float(y[e + 2 * u + 1]) * inv);
                        *(uint4*)(own + lane * D * 2 + (((4 * q + (e >> 3)) ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
            if (!split) {
                __syncwarp();
#pragma unroll
                for (int k = 0; k < CH; k++) {
                    const int r = k * AT_ONCE + lane / CH, ch = lane % CH, i2 = 128 * w + (warp & 3) * 32 + r, row2 = over_group(p, it.row0 + i2);
                    if (i2 < it.rows)
                        *(uint4*)(a.out + (long long)(it.s.row0 + row2) * a.o_rs + (long long)(it.hk * a.G + it.row0 + i2 - row2 * a.G) * a.o_hs + ch * 16) =
                            *(const uint4*)(own + r * D * 2 + ((ch ^ (r & 7)) << 4));
                }
            }
            if (split && mine) *(float2*)(p.ws_ml + ((size_t)blockIdx.x * PR_ROWS + i) * 2) = make_float2(m_used, l);
        }
        tc_fence_before();
        all_done();
        if (odd_value && !abort_flag_word) {
            for (int r = warp; r < it.rows; r += PR_LOADER) {
                const int at = it.row0 + r, token = at / a.G;
                row_state<D, S8>(a, it.b, it.s, token, it.hk * a.G + at - token * a.G, it.kb, 7, it.n0, it.n1,
                                 split ? p.ws_o + ((size_t)blockIdx.x * PR_ROWS + r) * D : nullptr, split ? p.ws_ml + ((size_t)blockIdx.x * PR_ROWS + r) * 2 : nullptr, p.flip);
            }
        }
    } else if (warp < PR_MMA) {
        if (!work) { all_done(); return; }
        // ---- K and V: fill f = 2 j + (0 for K, 1 for V) goes to slot f % SLOTS ----
        const int tid = threadIdx.x - PR_LOADER * 32;
        constexpr int CH = S8 ? D / 16 : D / 8, AT_ONCE = (PR_MMA - PR_LOADER) * 32 / CH, STEPS = 128 / AT_ONCE;    // 16-byte chunks of a token; tokens that the warps take at once
        const int r0 = tid / CH, ch = tid % CH, psh = a.c.page_shift;
        const int lo = place_lo(0), hi = place_hi(tiles - 1);
        int next_page = -1;
        const int lo_of[2] = {lo, place_lo(1)}, hi_of[2] = {place_hi(0), hi};
        auto facts = [&](int tok0, unsigned bad) {
            unsigned f = bad;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                if (w >= tiles) continue;
                if (tok0 <= hi_of[w] && (a.window == 0 || tok0 + 127 > lo_of[w] - a.window || tok0 < a.sinks)) f |= 256u << w;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int at = tok0 + 64 * h;
                    if ((bad >> (4 * h) & 15u) == 0 && at + 63 <= lo_of[w] && (a.window == 0 || at > hi_of[w] - a.window || at + 63 < a.sinks)) f |= 65536u << (2 * w + h);
                }
            }
            return f;
        };
        auto look_up = [&](int j) {                        // lane g < 8: page of granule g of block j
            next_page = -1;
            if (j < n && lane < 8) {
                const int tok = block_token(j) + 16 * lane;
                if (tok < it.kb.end && (tok + 15 >= it.kb.begin || tok < it.kb.sink_end)) {
                    next_page = table_page(a.c, it.b, tok >> psh);
                    if (next_page < 0) report_paged(a.c);
                }
            }
        };
        auto seen = [&](int tok) { return tok < it.kb.end && (tok >= it.kb.begin || tok < it.kb.sink_end); };
        bool alive = true;
        look_up(0);
        if constexpr (!S8) {
            auto arrived = [&](int f) {                    // the thread's part of fill f lies in shared memory
                const int tok0 = block_token(f >> 1);
                unsigned char* dst = ring + f % SLOTS * SM::TILE;
                if ((f & 1) && !(tok0 + 127 <= lo && (a.window == 0 || tok0 > hi - a.window || tok0 + 127 < a.sinks))) {
                    unsigned odd = 0;
#pragma unroll 4
                    for (int k = 0; k < STEPS; k++) {
                        const int r = k * AT_ONCE + r0;
                        const uint4 x = *(const uint4*)(dst + (ch >> 3) * HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                        odd |= not_finite2(x.x) | not_finite2(x.y) | not_finite2(x.z) | not_finite2(x.w);
                    }
                    if (odd) odd_value = 1;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_full + 8 * (f % SLOTS));
            };
            const long long ts = a.c.token_stride, thread_off = r0 * ts + ch * 16;
            int pending = 0;                               // fills f - pending .. f - 1 are on their way by cp.async
            const unsigned thread_dst = smem_u32(ring) + (ch >> 3) * HALF + r0 * 128 + (((ch & 7) ^ (r0 & 7)) << 4);
            for (int j = 0; j < n && alive; j++) {
                const int tok0 = block_token(j), page = next_page;
                const unsigned bad = __ballot_sync(0xffffffffu, lane < 8 && page < 0) & 255u;
                if (tid == 0) {
                    meta[j % PR_META].tok0 = tok0;
                    meta[j % PR_META].facts = facts(tok0, bad);
                }
                __syncwarp();                              // (another lane may be the one that announces the block)
                look_up(j + 1);
                // blocks that all rows see come by TMA, the others token by token with zeros for those that nobody sees
                const bool plain = p.tma && bad == 0 && tok0 + 127 <= lo && (a.window == 0 || tok0 > hi - a.window || tok0 + 127 < a.sinks);
#pragma unroll 1
                for (int kv = 0; kv < 2; kv++) {
                    const int f = 2 * j + kv, slot = f % SLOTS;
                    alive = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * slot, ((f / SLOTS) & 1) ^ 1, abort_flag, limit));
                    if (!alive) break;
                    if (plain) {
                        if (pending) {
                            cp_async_wait<0>();
                            for (; pending; pending--) arrived(f - pending);
                        }
                        if (warp == PR_LOADER) {
                            const unsigned full = bar_full + 8 * slot, dst = smem_u32(ring + slot * SM::TILE);
                            const bool one = elect_one();
                            if (one) mbar_expect_tx(full, SM::TILE);
                            const int per = 16 >> (psh - 3);            // pages of a block
#pragma unroll
                            for (int q = 0; q < 8; q++) {
                                const int pg = __shfl_sync(0xffffffffu, page, (q << (psh - 4)) & 7);
                                if (q < per && one) {
#pragma unroll
                                    for (int h = 0; h < D / 64; h++) tma_load_4d(dst + h * HALF + (q << (psh + 7)), kv ? &map_v : &map_k, full, 64 * h, 0, it.hk, pg);
                                }
                            }
                            __syncwarp();
                        } else if (lane == 0) {
                            mbar_arrive(bar_full + 8 * slot);
                        }
                        continue;
                    }
                    const unsigned char* base = (kv ? a.c.v : a.c.k) + (long long)it.hk * a.c.head_stride;
                    const unsigned dst = thread_dst + slot * SM::TILE;
#pragma unroll
                    for (int g = 0; g < 8; g++) {
                        const int pg = __shfl_sync(0xffffffffu, page, g);
                        const unsigned char* src = base + (long long)max(pg, 0) * a.c.page_stride + ((tok0 + 16 * g) & ((1 << psh) - 1)) * ts + thread_off;
#pragma unroll
                        for (int k = 0; k < 16 / AT_ONCE; k++) {
                            const bool ok = pg >= 0 && seen(tok0 + 16 * g + k * AT_ONCE + r0);
                            cp_async16_or_zero(dst + (16 * g + k * AT_ONCE) * 128, ok ? src + k * AT_ONCE * ts : base, ok);
                        }
                    }
                    cp_async_commit();
                    if (++pending > SM::AHEAD) { cp_async_wait<SM::AHEAD>(); arrived(f - SM::AHEAD); pending--; }
                }
            }
            cp_async_wait<0>();
            if (alive)
                for (; pending; pending--) arrived(2 * n - pending);
        } else {
            uint4 data[STEPS];
            auto fetch = [&](int tok0, int page, int kv) {
                const unsigned char* base = (kv ? a.c.v : a.c.k) + (long long)it.hk * a.c.head_stride;
#pragma unroll
                for (int k = 0; k < STEPS; k++) {
                    const int r = k * AT_ONCE + r0, tok = tok0 + r;
                    const int pg = __shfl_sync(0xffffffffu, page, r >> 4);
                    data[k] = make_uint4(0, 0, 0, 0);
                    if (pg >= 0 && seen(tok))
                        data[k] = __ldg((const uint4*)(base + (long long)pg * a.c.page_stride + (long long)(tok & ((1 << psh) - 1)) * a.c.token_stride) + ch);
                }
            };
            int page = next_page;
            if (n > 0) fetch(block_token(0), page, 0);
            for (int j = 0; j < n && alive; j++) {
                if (tid < 32) {
                    const unsigned bad = __ballot_sync(0xffffffffu, lane < 8 && page < 0) & 255u;
                    if (lane < 8) {
                        const long long at = (long long)max(page, 0) * a.c.scale_stride + it.hk;
                        meta[j % PR_META].k[lane] = page < 0 ? 0.0f : 64.0f * __ldg(a.c.k_scale + at);
                        meta[j % PR_META].v[lane] = page < 0 ? 0.0f : 64.0f * __ldg(a.c.v_scale + at);
                    }
                    if (lane == 0) {
                        meta[j % PR_META].tok0 = block_token(j);
                        meta[j % PR_META].facts = facts(block_token(j), bad);
                    }
                }
                const int tok0 = block_token(j);
                look_up(j + 1);
#pragma unroll 1
                for (int kv = 0; kv < 2; kv++) {
                    const int f = 2 * j + kv, slot = f % SLOTS;
                    alive = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * slot, ((f / SLOTS) & 1) ^ 1, abort_flag, limit));
                    if (!alive) break;
                    unsigned char* dst = ring + slot * SM::TILE;
#pragma unroll
                    for (int k = 0; k < STEPS; k++) {
                        const int r = k * AT_ONCE + r0;
                        const unsigned q4[4] = {data[k].x, data[k].y, data[k].z, data[k].w};
                        unsigned o[8];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const unsigned u = q4[e] ^ 0x80808080u;
                            o[2 * e] = u8x2_to_bf16x2_64th(u, 0x4140);
                            o[2 * e + 1] = u8x2_to_bf16x2_64th(u, 0x4342);
                        }
                        unsigned char* d = dst + (ch >> 2) * HALF + r * 128;
                        // (threads of the second 64 components store their second chunk first: the two halves' banks are the same)
                        const int first = ch >> 2 & 1;
                        *(uint4*)(d + ((((2 * ch + first) & 7) ^ (r & 7)) << 4)) = first ? make_uint4(o[4], o[5], o[6], o[7]) : make_uint4(o[0], o[1], o[2], o[3]);
                        *(uint4*)(d + ((((2 * ch + 1 - first) & 7) ^ (r & 7)) << 4)) = first ? make_uint4(o[0], o[1], o[2], o[3]) : make_uint4(o[4], o[5], o[6], o[7]);
                    }
                    // the next fill's bytes travel while this one is used
                    if (kv == 0) fetch(tok0, page, 1);
                    else if (j + 1 < n) { page = next_page; fetch(block_token(j + 1), page, 0); }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_full + 8 * slot);
                }
            }
        }
        all_done();
    } else if (warp < PR_MMA + SH::TILES) {
        // ---- products of tile w ----
        const int w = warp - PR_MMA;
        const unsigned idesc_s = make_idesc_bf16(PR_BLOCK / 2, false), idesc_o = make_idesc_bf16(D, true);
        auto needed = [&](int j) { return (meta[j % PR_META].facts & 256u << w) != 0; };       // (of a block whose K has arrived)
        const int frees = SH::TILES == 2 && tiles == 1 ? 2 : 1;               // arrivals of this tile on a slot's barrier (a lone tile's for both)
        bool alive = work && n > 0 && w < tiles, begun = false;
        unsigned p_phase = 0, phase = 0;                     // phase: of the ring, at slot `slot`
        int slot = 0;
        const unsigned ts = tmem + w * 128, to = tmem + SH::O_AT + w * D, bs = bar_s + 8 * w, bp = bar_p + 8 * w, bv = bar_v + 8 * w;
        const unsigned long long q_desc = make_smem_desc(smem_u32(smem + w * SM::TILE)), k_desc = make_smem_desc(smem_u32(ring)),
                                 v_desc = make_smem_desc_nmajor(smem_u32(ring), HALF);
        auto wait = [&](unsigned bar, unsigned parity) { alive = alive && __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, limit)); };
        auto free_slot = [&](int at, bool used) {
            if (elect_one()) {
                for (int i = 0; i < frees; i++) {
                    if (used) tc_commit(bar_empty + 8 * at);
                    else mbar_arrive(bar_empty + 8 * at);
                }
            }
        };
        auto step = [&](int& at, unsigned& ph) { if (++at == SLOTS) { at = 0; ph ^= 1; } };
        // by one lane: S of half h of a block's tokens; and the product of its probabilities with V
        // (every half of every block is handed back and forth, seen or not: so no side can be two steps ahead on a barrier)
        auto scores = [&](unsigned long long kd, int h, bool some) {
            if (!some) {
                mbar_arrive(bs + 16 * h);
                return;
            }
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                const unsigned long long off = (unsigned long long)((k >> 2) * (HALF >> 4) + (k & 3) * 2);
                tc_mma<false>(ts + 64 * h, q_desc + off, kd + off + (unsigned long long)(h * (64 * 128 >> 4)), idesc_s, (unsigned)(k != 0));
            }
            tc_commit(bs + 16 * h);
        };
        auto weighted = [&](unsigned long long vd, int h) {
#pragma unroll
            for (int k = 0; k < 4; k++)
                tc_mma_ts(to, ts + 64 * h + k * 8, vd + (unsigned long long)((4 * h + k) * (2048 >> 4)), idesc_o, (unsigned)(begun || h != 0 || k != 0));
            tc_commit(bv);
        };
        wait(bar_q + 8 * w, 0);
        wait(bar_full, 0);
        bool need = alive && needed(0);
        if (alive) {
            tc_fence_after();
            if (elect_one()) {
                scores(k_desc, 0, need);
                scores(k_desc, 1, need);
            }
            free_slot(0, need);
            step(slot, phase);
        }
        for (int j = 0; j < n && alive; j++) {
            // fills 2 j + 1 (V of this block) and 2 j + 2 (K of the next).  Everything that can be known is known before the probabilities come: between them
            // and the next scores in their place there is nothing but products
            const int vs = slot;
            wait(bar_full + 8 * slot, phase);
            step(slot, phase);
            const unsigned long long vd = v_desc + (unsigned long long)(vs * (SM::TILE >> 4)), kd = k_desc + (unsigned long long)(slot * (SM::TILE >> 4));
            const bool last = j + 1 == n;
            if (!last) wait(bar_full + 8 * slot, phase);
            const bool next = !last && alive && needed(j + 1);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                wait(bp + 16 * h, p_phase);
                if (!alive) break;
                tc_fence_after();
                if (elect_one()) {
                    if (need) weighted(vd, h);
                    if (!last) scores(kd, h, next);
                }
            }
            if (!alive) break;
            p_phase ^= 1;
            begun = begun || need;
            free_slot(vs, need);
            if (!last) {
                free_slot(slot, next);
                step(slot, phase);
            }
            need = next;
        }
        if (alive && elect_one()) tc_commit(bar_o + 8 * w);
        __syncwarp();
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        tc_fence_before();
        all_done();
        if (w != 0) return;
        if (lane == 0 && abort_flag_word) atomicExch(a.c.status, 4);
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)SH::COLUMNS) : "memory");
    } else {
        all_done();
    }
}

// Merges the sub-states of tiles whose blocks several CTAs shared: a warp per packed row.
constexpr int PRC_CTAS = 16;      // CTAs of a tile: 16 rows each, 8 where a tile has 128
template <int D, bool S8>
__global__ void __launch_bounds__(128) paged_prompt_combine_kernel(const PromptParams p) {
    constexpr int PR_ROWS = PromptShape<D, S8>::ROWS;
    __shared__ FindSpace space;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const PagedAttn& a = p.a;
    PromptItem it;
    if (!find_prompt_item<PR_ROWS, 128>(a, (int)(blockIdx.x / PRC_CTAS), 0, p.splits, false, &it, &space) || it.splits < 2) return;
    const int lane = threadIdx.x & 31;
    constexpr int N = D / 32;
    for (int i = blockIdx.x % PRC_CTAS * 4 + (threadIdx.x >> 5); i < it.rows; i += PRC_CTAS * 4) {
        const size_t first = ((size_t)(blockIdx.x / PRC_CTAS) * p.splits * PR_ROWS + i);
        float m = -INFINITY, l = 0.0f, acc[N];
#pragma unroll
        for (int e = 0; e < N; e++) acc[e] = 0.0f;
        for (int q = 0; q < it.splits; q++) {
            const size_t at = first + (size_t)q * PR_ROWS;
            const float2 ml = *(const float2*)(p.ws_ml + at * 2);
            float v[N];
#pragma unroll
            for (int e = 0; e < N; e += 2) { const float2 y = *(const float2*)(p.ws_o + at * D + lane * N + e); v[e] = y.x; v[e + 1] = y.y; }
            const float m_new = fmaxf(m, ml.x), f = m == -INFINITY ? 0.0f : exp2_approx(m - m_new), w = ml.x == -INFINITY ? 0.0f : exp2_approx(ml.x - m_new);
            l = l * f + ml.y * w;
#pragma unroll
            for (int e = 0; e < N; e++) acc[e] = acc[e] * f + v[e] * w;
            m = m_new;
        }
        const int packed = it.row0 + i, row = packed / a.G;
        unsigned char* out = a.out + (long long)(it.s.row0 + row) * a.o_rs + (long long)(it.hk * a.G + packed - row * a.G) * a.o_hs;
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int e = 0; e < N; e += 2) *(unsigned*)(out + 2 * (lane * N + e)) = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
    }
}

// A page of one head per box: {64 components, tokens of a page}, 128-byte swizzle.  False where the strides have no tensor map (blocks then come by
// cp.async, all of them).
inline bool make_page_map(CUtensorMap* map, const void* base, int D, const PagedView& c) {
    EncodeTiledFn fn = encode_fn();
    const uint64_t tokens = 1ull << c.page_shift;
    const cuuint64_t dims[4] = {(cuuint64_t)D, tokens, (cuuint64_t)c.Hkv, (cuuint64_t)std::max(c.pages, 1)};
    // (an extent of one is never stepped along)
    const cuuint64_t strides[3] = {(cuuint64_t)c.token_stride, (cuuint64_t)(c.Hkv > 1 ? c.head_stride : 16), (cuuint64_t)(c.pages > 1 ? c.page_stride : 16)};
    const cuuint32_t box[4] = {64, (cuuint32_t)tokens, 1, 1}, ones[4] = {1, 1, 1, 1};
    for (const cuuint64_t st : strides) if (st == 0 || st >= 1ull << 40) return false;
    return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, (void*)base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool S8>
int launch_paged_prompt(PagedAttn a, float scale, cudaStream_t s) {
    using SM = PromptSmem<D, S8>;
    using SH = PromptShape<D, S8>;
    static std::atomic<unsigned long long> attr_devices{0};
    const int arc = once_per_device(attr_devices, [] {
        B200FC_CUDA(cudaFuncSetAttribute(paged_prompt_kernel<D, S8>, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::BYTES));
        B200FC_CUDA(cudaFuncSetAttribute(paged_prompt_kernel<D, S8>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        return (int)B200FC_OK;
    });
    if (arc) return arc;
    PromptParams p;
    p.group_inverse = a.G > 1 ? (unsigned)(((1ULL << 32) + a.G - 1) / a.G) : 0;
    // masked scores are -inf whatever the scale: its sign goes into Q, and zero becomes the smallest number
    p.flip = scale < 0.0f ? 0x80008000u : 0u;
    a.scale_log2e = fmaxf(fabsf(a.scale_log2e), FLT_MIN);
    p.a = a;
    p.wait_limit_ns = wait_limit_ns();
    // tiles: full ones, and one more of each sequence
    const long long bound = ((long long)a.c.T * a.G / SH::ROWS + std::min(a.c.B, a.c.T)) * a.c.Hkv;
    const long long by_rows = (long long)a.c.B * (((long long)a.c.max_rows * a.G + SH::ROWS - 1) / SH::ROWS) * a.c.Hkv;
    const long long items = std::min(bound, by_rows);
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    p.splits = (int)std::max(1LL, std::min<long long>(std::min<long long>(16, sms * SH::CTAS / items), (a.c.capacity / PR_BLOCK + 1) / 2));
    if (items * p.splits > 1 << 25) { set_error("paged_attention: too many rows and heads for one call"); return B200FC_ERR_INVALID; }
    CUtensorMap maps[2] = {};
    p.tma = !S8 && make_page_map(&maps[0], a.c.k, D, a.c) && make_page_map(&maps[1], a.c.v, D, a.c);
    void* ws = nullptr;
    bool own = false;
    p.ws_o = p.ws_ml = nullptr;
    if (p.splits > 1) {
        const size_t states = (size_t)items * p.splits * SH::ROWS;
        const int rc = get_stream_scratch(states * (D + 2) * sizeof(float), s, 8, &ws, &own);
        if (rc) return rc;
        p.ws_o = (float*)ws;
        p.ws_ml = p.ws_o + states * D;
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * p.splits));
    cfg.blockDim = dim3(SH::THREADS);
    cfg.dynamicSmemBytes = SM::BYTES;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, paged_prompt_kernel<D, S8>, (const CUtensorMap)maps[0], (const CUtensorMap)maps[1], (const PromptParams)p);
    if (e == cudaSuccess) {
        count_launch();
        if (p.splits > 1) {
            cfg.gridDim = dim3((unsigned)(items * PRC_CTAS));
            cfg.blockDim = dim3(128);
            cfg.dynamicSmemBytes = 0;
            e = cudaLaunchKernelEx(&cfg, paged_prompt_combine_kernel<D, S8>, (const PromptParams)p);
            if (e == cudaSuccess) count_launch();
        }
    }
    if (own) {
        const cudaError_t f = cudaFreeAsync(ws, s);
        if (e == cudaSuccess) e = f;
    }
    return e == cudaSuccess ? (int)B200FC_OK : cuda_fail(e, "paged prompt attention");
}

}  // namespace

}  // namespace b200fc
