// Paged attention for few rows: at most 16 packed rows (query rows x heads of a group) per sequence and kv head, i.e. single tokens and short drafts.  A
// stream of K and V from HBM.
//
// The visible blocks of all (sequence, kv head) pairs, one behind the other in units of 64 tokens, form one sequence of work that is cut into equal
// pieces, one per CTA, whatever the lengths: with a piece per pair the longest sequence would decide.  A CTA walks its piece pair by pair; a pair that
// lies in several pieces leaves a sub-state (maximum, sum, unnormalised values) per piece, which paged_combine_kernel merges.
// Inside a CTA four warps take 16-token blocks of a unit each, with rings of their own filled by cp.async, and meet at the end of a pair.  The
// next pair's first blocks are on their way before that.  Scores and values go through mma.sync.m16n8k16 with tokens (then components) as the 16 rows and
// the packed rows as one or two operands of 8 columns (with the packed rows as the 16 rows, most groups leave half of every product empty); the
// probabilities turn from one form into the other by movmatrix.  (tcgen05 would work on 128 rows; bytes bound this: 23 per clock and SM at HBM speed.)
// 8 bits: bytes become bf16 of (value / 64), exactly, in two instructions a pair; the page's factors go into the scores and into the probabilities.
#pragma once
#include <cfloat>
#include "paged_common.cuh"

namespace b200fc {

namespace {

constexpr int DEC_WARPS = 4, DEC_THREADS = 128;
constexpr int DEC_UNIT = 64;                       // tokens of a unit: 16 per warp

template <int D, bool S8, int NT> struct DecSmem {
    static constexpr int ROW = D * (S8 ? 1 : 2), CHUNKS = ROW / 16;
    static constexpr int BLOCK = 16 * ROW;                              // 16 tokens of K (or V)
    static constexpr int CTAS = D == 128 ? (S8 ? 3 : 2) : (S8 ? 4 : 3);  // per SM
    static constexpr int STAGES = D == 128 ? 3 : 4;
    static constexpr int STAGE = 2 * BLOCK, RING = DEC_WARPS * STAGES * STAGE;
    static constexpr int ROW_STATE = D + (NT == 1 ? 8 : 0), WARP_STATE = 8 * NT * ROW_STATE;   // floats: a packed row's values, a warp's
    static constexpr int STATE = 2 * WARP_STATE * 4;
    static constexpr int BYTES = RING + STATE + DEC_WARPS * (16 * 8 + STAGES * 8) + 128;
    static_assert(CTAS * (BYTES + 1024 + 256) <= 233472, "resident together (1 KB of each CTA is the system's)");
};
// byte offset of 16-byte chunk c of token row r inside a block: eight rows of one chunk lie in eight different bank groups
template <int CHUNKS> __device__ __forceinline__ int dec_place(int r, int c) {
    if constexpr (CHUNKS == 4) return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ ((r >> 1) & 3)) << 4);
    else return r * CHUNKS * 16 + ((c ^ (r & 7)) << 4);
}

struct DecParams {
    PagedAttn a;
    int ctas;                     // pieces at most
    int min_units;                // units of a piece at least
    long long* prefix;            // [B + 1] units in front of sequence b's
    float* ws_o;                  // [ctas][2][16][D]: sub-states of a piece's first pair (if it begins in front) and of its last one (if it goes on behind)
    float* ws_ml;                 // [ctas][2][16][2]
};

__device__ __forceinline__ int dec_pieces(long long total, int ctas, int min_units) {
    const long long n = (total + min_units - 1) / min_units;
    return n < ctas ? (int)n : ctas;
}
// what a sequence has for the call: its packed rows' places and the blocks of 16 tokens that they see
struct DecSeq { SeqRows s; KeyBlocks kb; int units; };
__device__ __forceinline__ bool dec_seq(const PagedAttn& p, int b, DecSeq* q) {
    const bool ok = load_seq(p.c, b, &q->s);
    const int n = q->s.rows;
    q->kb = n > 0 ? key_blocks(max(q->s.len - n, 0), q->s.len - 1, p.window, p.sinks, 4) : KeyBlocks{0, 0, 0, 0, 0, 0};
    q->units = (q->kb.count + 3) >> 2;
    return ok;
}

template <int D, bool S8, int NT>
__global__ void __launch_bounds__(DEC_THREADS, DecSmem<D, S8, NT>::CTAS) paged_decode_kernel(const DecParams p) {
    using SM = DecSmem<D, S8, NT>;
    constexpr int CHUNKS = SM::CHUNKS, KSTEPS = D / 16, DEC_STAGES = SM::STAGES;
    extern __shared__ unsigned char dec_smem_raw[];
    __shared__ int warp_sum[DEC_WARPS];
    __shared__ struct { DecSeq seq; int b, hk, j; } first;
    unsigned char* smem = dec_smem_raw + (((smem_u32(dec_smem_raw) + 127u) & ~127u) - smem_u32(dec_smem_raw));
    float* st_o = (float*)(smem + SM::RING);                  // states of two warps
    float* st_ml = st_o + 2 * SM::WARP_STATE;                         // [warp][16][2]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const PagedAttn& a = p.a;
    const int Hkv = a.c.Hkv, B = a.c.B;

    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- units of all sequences, 128 at a time; CTA 0 leaves their running sum for the combining kernel ----
    DecSeq mine;                                              // of the thread's sequence of the round at hand
    int units_of_mine = 0, in_front = 0, round_units = 0;     // in_front: units of the round's sequences before the thread's
    auto scan_round = [&](int b0) {
        const int b = b0 + threadIdx.x;
        units_of_mine = 0;
        bool ok = true;
        if (b < B) {
            ok = dec_seq(a, b, &mine);
            units_of_mine = mine.units;
        }
        int upto = units_of_mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        __syncthreads();
        if (lane == 31) warp_sum[warp] = upto;
        __syncthreads();
        in_front = upto - units_of_mine;
        round_units = 0;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; w++) { in_front += w < warp ? warp_sum[w] : 0; round_units += warp_sum[w]; }
        return ok;
    };
    long long total = 0;
    for (int b0 = 0; b0 < B; b0 += DEC_THREADS) {
        const int b = b0 + threadIdx.x;
        if (!scan_round(b0) && blockIdx.x == 0) report_paged(a.c);
        if (b < B) {
            if (units_of_mine == 0 && mine.s.rows > 0 && b % gridDim.x == blockIdx.x) zero_rows<D>(a, mine.s);
            if (blockIdx.x == 0) p.prefix[b] = total + in_front;
        }
        total += round_units;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.prefix[B] = total;
    total *= Hkv;
    const int pieces = dec_pieces(total, p.ctas, p.min_units);
    if ((int)blockIdx.x >= pieces) return;
    const long long u0 = total * blockIdx.x / pieces, u1 = total * (blockIdx.x + 1) / pieces;

    // ---- the sequence that unit u0 belongs to ----
    for (long long b0 = 0, seen = 0; b0 < B; b0 += DEC_THREADS) {
        if (B > DEC_THREADS) scan_round((int)b0);             // (else the one round's numbers are still there)
        const long long lo = (seen + in_front) * Hkv;
        if (units_of_mine && u0 >= lo && u0 < lo + (long long)units_of_mine * Hkv) {
            first.seq = mine;
            first.b = (int)b0 + threadIdx.x; first.hk = (int)((u0 - lo) / units_of_mine); first.j = (int)((u0 - lo) % units_of_mine);
        }
        seen += round_units;
        if (u0 < seen * Hkv) break;
    }
    __syncthreads();
    int b = first.b, hk = first.hk, j0 = first.j;
    long long left = u1 - u0;
    DecSeq cur = first.seq;
    unsigned char* ring = smem + warp * DEC_STAGES * SM::STAGE;

    // One run of units [j0, j1) of a pair.  A warp's blocks are 4 j + warp.
    int j1 = (int)min((long long)cur.units, j0 + left);
    int next_page = -1;
    unsigned have = 0;                                     // slots of the ring whose block lies in a page of the pool
    float* factors = (float*)(st_ml + DEC_WARPS * 16 * 2) + warp * DEC_STAGES * 2;     // 8 bits: of the blocks in the ring, k's and v's
    const float* factor_src = lane == 0 ? a.c.k_scale : a.c.v_scale;
    const unsigned char *kbase, *vbase;
    auto look_up = [&](int j) {                            // page of the warp's block of unit j
        const int i = 4 * j + warp;
        next_page = -1;
        if (j < j1 && i < cur.kb.count) {
            const int tok = key_block(cur.kb, i) << 4;
            next_page = table_page(a.c, b, tok >> a.c.page_shift);
            if (next_page < 0) report_paged(a.c);
        }
    };
    auto begin_pair = [&]() {
        kbase = a.c.k + (long long)hk * a.c.head_stride;
        vbase = a.c.v + (long long)hk * a.c.head_stride;
    };
    const int lane_row = lane / CHUNKS, lane_chunk = lane % CHUNKS;
    constexpr int ROWS_AT_ONCE = 32 / CHUNKS;               // token rows of one copy instruction of the warp
    const long long lane_off = (long long)lane_row * a.c.token_stride + lane_chunk * 16, step = (long long)ROWS_AT_ONCE * a.c.token_stride;
    int slot = 0;                                           // of the ring, that the next block goes to
    auto issue = [&](int j) {
        const int i = 4 * j + warp, page = next_page;
        if (j < j1) {
            const int tok0 = key_block(cur.kb, i) << 4;
            const unsigned st = smem_u32(ring) + slot * SM::STAGE;
            const long long at = (long long)max(page, 0) * a.c.page_stride + (long long)(tok0 & ((1 << a.c.page_shift) - 1)) * a.c.token_stride + lane_off;
            const unsigned char *ks = kbase + at, *vs = vbase + at;
            const bool all = page >= 0 && tok0 + 16 <= cur.kb.end && (tok0 >= cur.kb.begin || tok0 + 16 <= cur.kb.sink_end);
#pragma unroll
            for (int n = 0; n < 16 / ROWS_AT_ONCE; n++) {
                const int row = n * ROWS_AT_ONCE + lane_row, tok = tok0 + row;
                const bool ok = all || (page >= 0 && tok < cur.kb.end && (tok >= cur.kb.begin || tok < cur.kb.sink_end));
                const unsigned dst = st + dec_place<CHUNKS>(row, lane_chunk);
                cp_async16_or_zero(dst, ok ? ks : kbase, ok);
                cp_async16_or_zero(dst + SM::BLOCK, ok ? vs : vbase, ok);
                ks += step; vs += step;
            }
        }
        have = page >= 0 ? have | 1u << slot : have & ~(1u << slot);
        if (S8 && lane < 2 && page >= 0) cp_async4(smem_u32(factors + 2 * slot + lane), factor_src + page * a.c.scale_stride + hk);
        slot = slot + 1 == DEC_STAGES ? 0 : slot + 1;
        cp_async_commit();
        look_up(j + 1);
    };
    begin_pair();
    look_up(j0);
    for (int j = j0; j < j0 + DEC_STAGES - 1; j++) issue(j);

    while (true) {
        const SeqRows s = cur.s;
        const KeyBlocks kb = cur.kb;
        const int rows = s.rows * a.G, units = cur.units, run0 = j0, run1 = j1, at_b = b, at_hk = hk;
        // ---- Q as the 8-column operand: column n of tile nt = packed row 8 nt + n = (row / G, head % G of the group); zeros past the last one ----
        unsigned qb[NT][KSTEPS][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int i = 8 * nt + g, row = i / a.G;
            const bool ok = i < rows;
            const unsigned char* qp = a.q + (long long)(s.row0 + (ok ? row : 0)) * a.q_rs + (long long)(hk * a.G + (ok ? i - row * a.G : 0)) * a.q_hs;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ks++) {
                // (8 bits: the components of a k-step are permuted as the bytes of a chunk come out of ldmatrix)
                const int d0 = ks * 16 + (S8 ? 4 * t : 2 * t), d1 = d0 + (S8 ? 2 : 8);
                qb[nt][ks][0] = ok ? __ldg((const unsigned*)(qp + d0 * 2)) : 0u;
                qb[nt][ks][1] = ok ? __ldg((const unsigned*)(qp + d1 * 2)) : 0u;
            }
        }
        // a lane's scores and values belong to packed rows 8 nt + 2 t + r
        int place[NT][2];
        float o[NT][D / 16][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int i = 0; i < D / 16; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                place[nt][r] = s.len - s.rows + (8 * nt + 2 * t + r) / a.G;
                m_run[nt][r] = -FLT_MAX;                          // (not -inf: scores of -inf, masked or not, then weigh 0 without a look at them)
                l_run[nt][r] = 0.0f;
            }
        }
        const int place_lo = s.len - s.rows, place_hi = s.len - 1;
        bool odd = false;

#pragma unroll 1
        for (int j = run0; j < run1; j++) {
            issue(j + DEC_STAGES - 1);
            cp_async_wait<DEC_STAGES - 1>();
            __syncwarp();
            const int at = slot, i = 4 * j + warp, mi = lane >> 3;     // (the ring has gone round: the oldest block is where the next one goes)
            const unsigned kst = smem_u32(ring) + at * SM::STAGE, vst = kst + SM::BLOCK;
            const int tok0 = key_block(kb, i) << 4;
            float fk = a.scale_log2e, fv = 1.0f;
            if (S8) {
                const float2 f = *(const float2*)(factors + 2 * at);
                fk *= 64.0f * f.x;
                fv = 64.0f * f.y;
            }
            // ---- S = K Q^T: 16 tokens x 8 rows; two chains of products ----
            float sc[NT][4];
            {
                float part[NT][2][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 8; e++) part[nt][e >> 2][e & 3] = 0.0f;
                const int tok = (mi & 1) * 8 + (lane & 7);
                if constexpr (!S8) {
#pragma unroll
                    for (int ks = 0; ks < KSTEPS; ks++) {
                        unsigned kr[4];                       // tokens 0-7, 8-15 of the first 8 components, then of the second
                        ldsm_x4(kr, kst + dec_place<CHUNKS>(tok, 2 * ks + (mi >> 1)));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma_bf16_16816(part[nt][ks & 1], kr[0], kr[1], kr[2], kr[3], qb[nt][ks][0], qb[nt][ks][1]);
                    }
                } else {
#pragma unroll
                    for (int k2 = 0; k2 < KSTEPS / 2; k2++) {
                        unsigned kr[4];                       // tokens 0-7, 8-15 of one chunk of 16 components, then of the next
                        ldsm_x4(kr, kst + dec_place<CHUNKS>(tok, 2 * k2 + (mi >> 1)));
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const unsigned w0 = kr[2 * e] ^ 0x80808080u, w1 = kr[2 * e + 1] ^ 0x80808080u;
                            const unsigned a0 = u8x2_to_bf16x2_64th(w0, 0x4140), a1 = u8x2_to_bf16x2_64th(w1, 0x4140);
                            const unsigned a2 = u8x2_to_bf16x2_64th(w0, 0x4342), a3 = u8x2_to_bf16x2_64th(w1, 0x4342);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma_bf16_16816(part[nt][e], a0, a1, a2, a3, qb[nt][2 * k2 + e][0], qb[nt][2 * k2 + e][1]);
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++) sc[nt][c] = (part[nt][0][c] + part[nt][1][c]) * fk;
            }
            // ---- online softmax (exp2 domain): a lane's tokens are tok0 + g and tok0 + g + 8 ----
            const bool there = have >> at & 1;
            const bool whole = there && tok0 + 15 <= place_lo && (tok0 + 15 < a.sinks || a.window == 0 || tok0 > place_hi - a.window);
            if (!whole) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (!(there && key_visible(tok0 + g + (c >> 1) * 8, place[nt][c & 1], a.window, a.sinks))) sc[nt][c] = -INFINITY;
            }
            float top[NT][2];
            bool rose = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    float x = fmaxf(sc[nt][r], sc[nt][2 + r]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    top[nt][r] = fmaxf(m_run[nt][r], x);
                    rose = rose || top[nt][r] > m_run[nt][r];
                }
            if (__any_sync(0xffffffffu, rose)) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float f[2];
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        f[r] = exp2_approx(m_run[nt][r] - top[nt][r]);
                        m_run[nt][r] = top[nt][r];
                        l_run[nt][r] *= f[r];
                    }
#pragma unroll
                    for (int n = 0; n < D / 16; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++) o[nt][n][c] *= f[c & 1];
                }
            }
            unsigned pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float e[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float x = sc[nt][c];
                    e[c] = exp2_approx(x - m_run[nt][c & 1]);
                    l_run[nt][c & 1] += e[c];
                    if (S8 && (whole || x != -INFINITY)) e[c] *= fv;          // (a masked token has no part in its page's factor, which may be NaN)
                }
                // (token g, rows 2 t, 2 t + 1) -> (row g, tokens 2 t, 2 t + 1)
                pb[nt][0] = transpose8x8(pack_bf16x2(e[0], e[1]));
                pb[nt][1] = transpose8x8(pack_bf16x2(e[2], e[3]));
            }
            // ---- O^T += V^T P^T: 16 components x 8 rows ----
            if constexpr (!S8) {
                const int tok = (mi >> 1) * 8 + (lane & 7);
                unsigned worst = 0;
#pragma unroll
                for (int n = 0; n < D / 16; n++) {
                    unsigned vr[4];                           // components 0-7, 8-15 of tokens 0-7, then of tokens 8-15
                    ldsm_x4_trans(vr, vst + dec_place<CHUNKS>(tok, 2 * n + (mi & 1)));
                    if (!whole) worst |= not_finite2(vr[0]) | not_finite2(vr[1]) | not_finite2(vr[2]) | not_finite2(vr[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma_bf16_16816(o[nt][n], vr[0], vr[1], vr[2], vr[3], pb[nt][0], pb[nt][1]);
                }
                odd = odd || worst != 0;
            } else {
                const int tok = (mi & 1) * 8 + (lane & 7);
#pragma unroll
                for (int n2 = 0; n2 < D / 32; n2++) {
                    unsigned vr[4];                           // two chunks of (tokens 0-7, 8-15); a register holds components 2 g, 2 g + 1 of two tokens
                    ldsm_x4_trans(vr, vst + dec_place<CHUNKS>(tok, 2 * n2 + (mi >> 1)));
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const unsigned w0 = vr[2 * e] ^ 0x80808080u, w1 = vr[2 * e + 1] ^ 0x80808080u;
                        const unsigned a0 = u8x2_to_bf16x2_64th(w0, 0x4240), a1 = u8x2_to_bf16x2_64th(w0, 0x4341);
                        const unsigned a2 = u8x2_to_bf16x2_64th(w1, 0x4240), a3 = u8x2_to_bf16x2_64th(w1, 0x4341);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) mma_bf16_16816(o[nt][2 * n2 + e], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                    }
                }
            }
            __syncwarp();
        }

        // ---- on to the next pair: its first blocks travel while this one is finished ----
        left -= run1 - run0;
        const bool more = left > 0;
        if (more) {
            j0 = 0;
            if (++hk == Hkv) {
                hk = 0;
                do dec_seq(a, ++b, &cur); while (cur.units == 0);
            }
            j1 = (int)min((long long)cur.units, left);
            slot = 0;
            begin_pair();
            look_up(0);
            for (int j = 0; j < DEC_STAGES - 1; j++) issue(j);
        }

        // (the combining kernel may come up now: earlier its CTAs would only take places)
        else asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

        // ---- the four warps' states: values by lane (each warp's lanes hold the same places), maxima and sums by row ----
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int x = 4; x < 32; x *= 2) l_run[nt][r] += __shfl_xor_sync(0xffffffffu, l_run[nt][r], x);
        auto put_state = [&](float* dst) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int n = 0; n < D / 16; n++) ((float4*)dst)[(nt * (D / 16) + n) * 32 + lane] = make_float4(o[nt][n][0], o[nt][n][1], o[nt][n][2], o[nt][n][3]);
        };
        auto put_ml = [&](int w) {
            if (g == 0)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int r = 0; r < 2; r++) *(float2*)(st_ml + (w * 16 + 8 * nt + 2 * t + r) * 2) = make_float2(m_run[nt][r], l_run[nt][r]);
        };
        auto take_state = [&](const float* src, int w) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float f[2], e[2];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const float2 ml = *(const float2*)(st_ml + (w * 16 + 8 * nt + 2 * t + r) * 2);
                    const float m = fmaxf(m_run[nt][r], ml.x);
                    f[r] = exp2_approx(m_run[nt][r] - m);
                    e[r] = exp2_approx(ml.x - m);
                    l_run[nt][r] = l_run[nt][r] * f[r] + ml.y * e[r];
                    m_run[nt][r] = m;
                }
#pragma unroll
                for (int n = 0; n < D / 16; n++) {
                    const float4 x = ((const float4*)src)[(nt * (D / 16) + n) * 32 + lane];
                    o[nt][n][0] = o[nt][n][0] * f[0] + x.x * e[0]; o[nt][n][1] = o[nt][n][1] * f[1] + x.y * e[1];
                    o[nt][n][2] = o[nt][n][2] * f[0] + x.z * e[0]; o[nt][n][3] = o[nt][n][3] * f[1] + x.w * e[1];
                }
            }
        };
        __syncthreads();                                  // (the previous pair's states have been read)
        put_ml(warp);
        if (warp >= 2) put_state(st_o + (warp - 2) * SM::WARP_STATE);
        // has any warp met a value that is no number?  (Every thread gets the answer from the barrier: a shared word would have to be cleared for the next pair while
        // late warps still read it.)
        bool any_odd = false;                             // (8 bits hold none)
        if constexpr (S8) __syncthreads();
        else any_odd = __syncthreads_or(odd);
        if (warp < 2) take_state(st_o + warp * SM::WARP_STATE, warp + 2);
        __syncwarp();
        if (warp == 1) { put_ml(1); put_state(st_o + SM::WARP_STATE); }
        __syncthreads();
        const bool split = run0 > 0 || run1 < units;
        const size_t sub = ((size_t)blockIdx.x * 2 + (run0 > 0 ? 0 : 1)) * 16;
        if (any_odd && s.rows > 1) {
            // a value that is no number stands in a block that some rows do not see: row by row, each over what it sees
            for (int i = warp; i < rows; i += DEC_WARPS)
                row_state<D, S8>(a, at_b, s, i / a.G, at_hk * a.G + i % a.G, kb, 4, 4 * run0, min(4 * run1, kb.count), split ? p.ws_o + (sub + i) * D : nullptr,
                                 split ? p.ws_ml + (sub + i) * 2 : nullptr, 0);
        } else if (warp == 0) {
            take_state(st_o + SM::WARP_STATE, 1);
            // through shared memory once more (where warp 0's state would have been), so that rows are stored in whole
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    float* dst = st_o + (8 * nt + 2 * t + r) * SM::ROW_STATE;
#pragma unroll
                    for (int n = 0; n < D / 16; n++) {
                        dst[16 * n + (S8 ? 2 * g : g)] = o[nt][n][r];
                        dst[16 * n + (S8 ? 2 * g + 1 : g + 8)] = o[nt][n][2 + r];
                    }
                    if (g == 0) *(float2*)(st_ml + (8 * nt + 2 * t + r) * 2) = make_float2(m_run[nt][r], l_run[nt][r]);
                }
            __syncwarp();
            for (int i = 0; i < rows; i++) {
                const float2 ml = *(const float2*)(st_ml + i * 2);
                const int row = i / a.G;
#pragma unroll
                for (int d = lane * 2; d < D; d += 64) {
                    const float2 x = *(const float2*)(st_o + i * SM::ROW_STATE + d);
                    if (split) *(float2*)(p.ws_o + (sub + i) * D + d) = x;
                    else {
                        const float inv = ml.y != 0.0f ? 1.0f / ml.y : 0.0f;
                        *(unsigned*)(a.out + (long long)(s.row0 + row) * a.o_rs + (long long)(at_hk * a.G + i - row * a.G) * a.o_hs + 2 * d) = pack_bf16x2(x.x * inv, x.y * inv);
                    }
                }
                if (split && lane == 0) *(float2*)(p.ws_ml + (sub + i) * 2) = ml;
            }
        }
        if (!more) break;
    }
    cp_async_wait<0>();
}

// Merges the sub-states of the pairs that lie in several pieces: a warp per packed row, CTAs of (pair, four rows).
template <int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const DecParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const PagedAttn& a = p.a;
    const int b = blockIdx.x / a.c.Hkv, hk = blockIdx.x % a.c.Hkv, i = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    SeqRows s;
    load_seq(a.c, b, &s);
    const long long before = p.prefix[b], n = p.prefix[b + 1] - before;
    if (n == 0) return;
    const long long total = p.prefix[a.c.B] * a.c.Hkv, x = before * a.c.Hkv + hk * n;
    const int pieces = dec_pieces(total, p.ctas, p.min_units);
    // the pieces of the pair's first and last unit
    const int c0 = (int)(((x + 1) * pieces - 1) / total), c1 = (int)(((x + n) * pieces - 1) / total);
    if (c0 == c1 || i >= s.rows * a.G) return;
    // the first piece holds the pair's beginning unless it begins exactly there, in which case too it is a sub-state that goes on behind
    auto slot = [&](int c) { return ((size_t)c * 2 + (c == c0 ? 1 : 0)) * 16 + i; };
    constexpr int N = D / 32;
    float m = -INFINITY, l = 0.0f, acc[N];
#pragma unroll
    for (int e = 0; e < N; e++) acc[e] = 0.0f;
    for (int cb = c0; cb <= c1; cb += 32) {
        const int c = cb + lane;
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (c <= c1) ml = *(const float2*)(p.ws_ml + slot(c) * 2);
        float top = ml.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m, top);
        const float f = m == -INFINITY ? 0.0f : exp2_approx(m - m_new), w = ml.x == -INFINITY ? 0.0f : exp2_approx(ml.x - m_new);
        float sum = w * ml.y;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = l * f + sum;
        m = m_new;
#pragma unroll
        for (int e = 0; e < N; e++) acc[e] *= f;
        const int count = min(32, c1 - cb + 1);
        for (int q0 = 0; q0 < count; q0 += 8) {
            float v[8][N];
#pragma unroll
            for (int q = 0; q < 8; q++)
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const float2 y = q0 + q < count ? *(const float2*)(p.ws_o + slot(cb + q0 + q) * D + lane * N + e) : make_float2(0.0f, 0.0f);
                    v[q][e] = y.x; v[q][e + 1] = y.y;
                }
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const float wq = __shfl_sync(0xffffffffu, w, (q0 + q) & 31);
#pragma unroll
                for (int e = 0; e < N; e++) if (q0 + q < count) acc[e] = fmaf(v[q][e], wq, acc[e]);
            }
        }
    }
    const int row = i / a.G;
    unsigned char* out = a.out + (long long)(s.row0 + row) * a.o_rs + (long long)(hk * a.G + i - row * a.G) * a.o_hs;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int e = 0; e < N; e += 2) *(unsigned*)(out + 2 * (lane * N + e)) = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
}

template <int D, bool S8, int NT>
int launch_paged_decode_as(DecParams& p, cudaStream_t s) {
    using SM = DecSmem<D, S8, NT>;
    static std::atomic<unsigned long long> attr_devices{0};
    const int arc = once_per_device(attr_devices, [] {
        B200FC_CUDA(cudaFuncSetAttribute(paged_decode_kernel<D, S8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::BYTES));
        return (int)B200FC_OK;
    });
    if (arc) return arc;
    const PagedView& c = p.a.c;
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    // as many pieces as are resident together, if the cache can hold that many
    const long long units = (c.capacity + DEC_UNIT - 1) / DEC_UNIT * c.B * c.Hkv;
    p.min_units = 2;
    p.ctas = (int)std::max(1LL, std::min<long long>((long long)sms * SM::CTAS, (units + p.min_units - 1) / p.min_units));
    void* ws = nullptr;
    bool own = false;
    const size_t states = (size_t)p.ctas * 2 * 16;
    const int rc = get_stream_scratch(states * (D + 2) * sizeof(float) + ((size_t)c.B + 1) * sizeof(long long), s, 7, &ws, &own);
    if (rc) return rc;
    p.ws_o = (float*)ws;
    p.ws_ml = p.ws_o + states * D;
    p.prefix = (long long*)(p.ws_ml + states * 2);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.ctas);
    cfg.blockDim = dim3(DEC_THREADS);
    cfg.dynamicSmemBytes = SM::BYTES;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, paged_decode_kernel<D, S8, NT>, (const DecParams)p);
    if (e == cudaSuccess) {
        count_launch();
        if (p.ctas > 1) {
            cfg.gridDim = dim3((unsigned)(c.B * c.Hkv), (unsigned)((std::min<long long>(16, (long long)c.max_rows * p.a.G) + 3) / 4));
            cfg.dynamicSmemBytes = 0;
            e = cudaLaunchKernelEx(&cfg, paged_combine_kernel<D>, (const DecParams)p);
            if (e == cudaSuccess) count_launch();
        }
    }
    if (own) {
        const cudaError_t f = cudaFreeAsync(ws, s);
        if (e == cudaSuccess) e = f;
    }
    return e == cudaSuccess ? (int)B200FC_OK : cuda_fail(e, "paged decode attention");
}

}  // namespace

}  // namespace b200fc
