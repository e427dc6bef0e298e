// Paged attention for few rows: at most 16 packed rows (query rows x heads of a group) per sequence and kv head, i.e. single tokens and short drafts.  A
// stream of K and V from HBM.
//
// The visible blocks of all (sequence, kv head) pairs, one behind the other in units of 64 tokens, form one sequence of work that is cut into equal
// pieces, one per CTA, whatever the lengths: with a piece per pair the longest sequence would decide.  A CTA walks its piece pair by pair; a pair that
// lies in several pieces leaves a sub-state (maximum, sum, unnormalised values) per piece, which paged_combine_kernel merges.
// Inside a CTA four warps take 16-token blocks of a unit each, with rings of their own filled by cp.async, and meet at the end of a pair.  The
// next pair's first blocks are on their way before that.  Scores and values go through mma.sync.m16n8k16: the packed rows are the 16 rows, so K and V
// cross shared memory once for all of them (bytes bound it: 23 per clock and SM at HBM speed; tcgen05 would work on 128 rows).
// 8 bits: bytes become bf16 of (value / 64), exactly, in two instructions a pair; the page's factors go into the scores and into the probabilities.
#pragma once
#include "paged_common.cuh"

namespace b200fc {

namespace {

constexpr int DEC_WARPS = 4, DEC_THREADS = 128, DEC_STAGES = 3;
constexpr int DEC_UNIT = 64;                       // tokens of a unit: 16 per warp

template <int D, bool S8> struct DecSmem {
    static constexpr int ROW = D * (S8 ? 1 : 2), CHUNKS = ROW / 16;
    static constexpr int BLOCK = 16 * ROW;                              // 16 tokens of K (or V)
    static constexpr int STAGE = 2 * BLOCK, RING = DEC_WARPS * DEC_STAGES * STAGE;
    static constexpr int STATE = 2 * 16 * D * 4;                        // values of two warps
    static constexpr int BYTES = RING + STATE + DEC_WARPS * 16 * 8 + 128;
    static constexpr int CTAS = D == 128 ? (S8 ? 3 : 2) : 4;            // per SM
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

template <int D, bool S8>
__global__ void __launch_bounds__(DEC_THREADS, DecSmem<D, S8>::CTAS) paged_decode_kernel(const DecParams p) {
    using SM = DecSmem<D, S8>;
    constexpr int CHUNKS = SM::CHUNKS, KSTEPS = D / 16;
    extern __shared__ unsigned char dec_smem_raw[];
    __shared__ int warp_sum[DEC_WARPS], found[4], odd_value;
    unsigned char* smem = dec_smem_raw + (((smem_u32(dec_smem_raw) + 127u) & ~127u) - smem_u32(dec_smem_raw));
    float* st_o = (float*)(smem + SM::RING);                  // [2][16][D]
    float* st_ml = st_o + 2 * 16 * D;                         // [warp][16][2]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const PagedAttn& a = p.a;
    const int Hkv = a.c.Hkv, B = a.c.B;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- units of all sequences; CTA 0 leaves their running sum for the combining kernel ----
    long long total = 0;
    for (int b0 = 0; b0 < B; b0 += DEC_THREADS) {
        const int b = b0 + threadIdx.x;
        DecSeq q;
        int n = 0;
        if (b < B) {
            if (!dec_seq(a, b, &q) && blockIdx.x == 0) report_paged(a.c);
            n = q.units;
            if (n == 0 && q.s.rows > 0 && b % gridDim.x == blockIdx.x) zero_rows<D>(a, q.s);
        }
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        if (lane == 31) warp_sum[warp] = upto;
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; w++) { before += w < warp ? warp_sum[w] : 0; all += warp_sum[w]; }
        if (blockIdx.x == 0 && b < B) p.prefix[b] = total + before + upto - n;
        total += all;
        __syncthreads();
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.prefix[B] = total;
    total *= Hkv;
    const int pieces = dec_pieces(total, p.ctas, p.min_units);
    if ((int)blockIdx.x >= pieces) return;
    const long long u0 = total * blockIdx.x / pieces, u1 = total * (blockIdx.x + 1) / pieces;

    // ---- the sequence that unit u0 belongs to ----
    long long seen = 0;
    for (int b0 = 0; b0 < B; b0 += DEC_THREADS) {
        const int b = b0 + threadIdx.x;
        DecSeq q;
        int n = 0;
        if (b < B) { dec_seq(a, b, &q); n = q.units; }
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        if (lane == 31) warp_sum[warp] = upto;
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < DEC_WARPS; w++) { before += w < warp ? warp_sum[w] : 0; all += warp_sum[w]; }
        const long long lo = (seen + before + upto - n) * Hkv, hi = lo + (long long)n * Hkv;
        if (n && u0 >= lo && u0 < hi) { found[0] = b; found[1] = (int)((u0 - lo) / n); found[2] = (int)((u0 - lo) % n); }
        seen += all;
        __syncthreads();
        if (u0 < seen * Hkv) break;
    }
    int b = found[0], hk = found[1], j0 = found[2];
    long long left = u1 - u0;
    DecSeq cur;
    dec_seq(a, b, &cur);
    unsigned char* ring = smem + warp * DEC_STAGES * SM::STAGE;

    // One run of units [j0, j1) of a pair.  A warp's blocks are 4 j + warp.
    int j1 = (int)min((long long)cur.units, j0 + left);
    int next_page = -1;
    unsigned have = 0;                                     // slots of the ring whose block lies in a page of the pool
    float kf[DEC_STAGES], vf[DEC_STAGES];                  // 8 bits: factors of the blocks in the ring
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
    auto issue = [&](int j) {
        const int i = 4 * j + warp, page = next_page, slot = (j - j0) % DEC_STAGES;
        if (j < j1) {
            const int tok0 = key_block(cur.kb, i) << 4;
            unsigned char* st = ring + slot * SM::STAGE;
            const long long at = (long long)max(page, 0) * a.c.page_stride + (long long)(tok0 & ((1 << a.c.page_shift) - 1)) * a.c.token_stride;
#pragma unroll
            for (int n = 0; n < 16 * CHUNKS / 32; n++) {
                const int u = n * 32 + lane, row = u / CHUNKS, c = u % CHUNKS, tok = tok0 + row;
                const bool ok = page >= 0 && tok < cur.kb.end && (tok >= cur.kb.begin || tok < cur.kb.sink_end);
                const unsigned dst = smem_u32(st) + dec_place<CHUNKS>(row, c);
                const long long off = ok ? at + (long long)row * a.c.token_stride + c * 16 : 0;
                cp_async16_or_zero(dst, kbase + off, ok);
                cp_async16_or_zero(dst + SM::BLOCK, vbase + off, ok);
            }
        }
        have = page >= 0 ? have | 1u << slot : have & ~(1u << slot);
        if (S8) {
            float fk = 0.0f, fv = 0.0f;
            if (page >= 0) {
                fk = __ldg(a.c.k_scale + page * a.c.scale_stride + hk);
                fv = __ldg(a.c.v_scale + page * a.c.scale_stride + hk);
            }
#pragma unroll
            for (int q = 0; q < DEC_STAGES; q++) if (q == slot) { kf[q] = fk; vf[q] = fv; }
        }
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
        // ---- Q: packed row i = (row i / G, head i % G of the group); rows past the last one are zeros ----
        unsigned qa[KSTEPS][4];
        int place[2];
        {
            const unsigned char* qp[2];
            bool ok[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int i = g + 8 * r, row = i / a.G;
                ok[r] = i < rows;
                place[r] = s.len - s.rows + row;
                qp[r] = a.q + (long long)(s.row0 + row) * a.q_rs + (long long)(hk * a.G + i - row * a.G) * a.q_hs;
            }
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ks++) {
                // (8 bits: a k-step's columns are permuted as the bytes of a chunk come out of ldmatrix)
                const int d0 = ks * 16 + (S8 ? 4 * t : 2 * t), d1 = d0 + (S8 ? 2 : 8);
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    qa[ks][r] = ok[r] ? __ldg((const unsigned*)(qp[r] + d0 * 2)) : 0u;
                    qa[ks][2 + r] = ok[r] ? __ldg((const unsigned*)(qp[r] + d1 * 2)) : 0u;
                }
            }
        }
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
        const int place_lo = s.len - s.rows, place_hi = s.len - 1;
        bool odd = false;

#pragma unroll 1
        for (int j = run0; j < run1; j++) {
            issue(j + DEC_STAGES - 1);
            cp_async_wait<DEC_STAGES - 1>();
            __syncwarp();
            const int slot = (j - run0) % DEC_STAGES, i = 4 * j + warp;
            const unsigned kst = smem_u32(ring) + slot * SM::STAGE, vst = kst + SM::BLOCK;
            const int tok0 = key_block(kb, i) << 4;
            float fk = a.scale_log2e, fv = 1.0f;
            if (S8) {
#pragma unroll
                for (int q = 0; q < DEC_STAGES; q++) if (q == slot) { fk = kf[q]; fv = vf[q]; }
                fk *= 64.0f * a.scale_log2e;
                fv *= 64.0f;
            }
            float sc[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
            if constexpr (!S8) {
                const int mi = lane >> 3, tok = (mi >> 1) * 8 + (lane & 7);
#pragma unroll
                for (int ks = 0; ks < KSTEPS; ks++) {
                    unsigned kr[4];
                    ldsm_x4(kr, kst + dec_place<CHUNKS>(tok, 2 * ks + (mi & 1)));
                    mma_bf16_16816(sc[0], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kr[0], kr[1]);
                    mma_bf16_16816(sc[1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kr[2], kr[3]);
                }
            } else {
                const int mi = lane >> 3, tok = (mi >> 1) * 8 + (lane & 7);
#pragma unroll
                for (int k2 = 0; k2 < KSTEPS / 2; k2++) {
                    unsigned kr[4];                       // [tokens 0-7, 8-15][two chunks of 16 components]
                    ldsm_x4(kr, kst + dec_place<CHUNKS>(tok, 2 * k2 + (mi & 1)));
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const unsigned w = kr[2 * h + e] ^ 0x80808080u;
                            mma_bf16_16816(sc[h], qa[2 * k2 + e][0], qa[2 * k2 + e][1], qa[2 * k2 + e][2], qa[2 * k2 + e][3],
                                           u8x2_to_bf16x2_64th(w, 0x4140), u8x2_to_bf16x2_64th(w, 0x4342));
                        }
                }
            }
            // ---- online softmax (exp2 domain) ----
            const bool there = have >> slot & 1;
            const bool whole = there && tok0 + 15 <= place_lo && (tok0 + 15 < a.sinks || a.window == 0 || tok0 > place_hi - a.window);
            float bm[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int tt = 0; tt < 2; tt++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int tok = tok0 + tt * 8 + 2 * t + (c & 1);
                    float x = sc[tt][c] * fk;
                    if (!whole && !(there && key_visible(tok, place[c >> 1], a.window, a.sinks))) x = -INFINITY;
                    sc[tt][c] = x;
                    bm[c >> 1] = fmaxf(bm[c >> 1], x);
                }
#pragma unroll
            for (int r = 0; r < 2; r++) {
                bm[r] = fmaxf(bm[r], __shfl_xor_sync(0xffffffffu, bm[r], 1));
                bm[r] = fmaxf(bm[r], __shfl_xor_sync(0xffffffffu, bm[r], 2));
            }
            float corr[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const float m_new = fmaxf(m_run[r], bm[r]);
                corr[r] = m_new == -INFINITY ? 1.0f : exp2_approx(m_run[r] - m_new);
                m_run[r] = m_new;
                l_run[r] *= corr[r];
            }
#pragma unroll
            for (int tt = 0; tt < 2; tt++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float x = sc[tt][c];
                    const float e = whole || x != -INFINITY ? exp2_approx(x - m_run[c >> 1]) : 0.0f;
                    l_run[c >> 1] += e;
                    sc[tt][c] = S8 ? (whole || x != -INFINITY ? e * fv : 0.0f) : e;
                }
            const unsigned pa0 = pack2_bf16(sc[0][0], sc[0][1]), pa1 = pack2_bf16(sc[0][2], sc[0][3]);
            const unsigned pa2 = pack2_bf16(sc[1][0], sc[1][1]), pa3 = pack2_bf16(sc[1][2], sc[1][3]);
            // ---- O = O * corr + P V ----
            const int mi = lane >> 3;
            if constexpr (!S8) {
                const int tok = (mi & 1) * 8 + (lane & 7);
                unsigned worst = 0;
#pragma unroll
                for (int c2 = 0; c2 < CHUNKS / 2; c2++) {
                    unsigned vr[4];
                    ldsm_x4_trans(vr, vst + dec_place<CHUNKS>(tok, 2 * c2 + (mi >> 1)));
                    if (!whole) {
#pragma unroll
                        for (int q = 0; q < 4; q++) worst |= not_finite2(vr[q]);
                    }
#pragma unroll
                    for (int h2 = 0; h2 < 2; h2++) {
                        float (&acc)[4] = o[2 * c2 + h2];
                        acc[0] *= corr[0]; acc[1] *= corr[0]; acc[2] *= corr[1]; acc[3] *= corr[1];
                        mma_bf16_16816(acc, pa0, pa1, pa2, pa3, vr[2 * h2], vr[2 * h2 + 1]);
                    }
                }
                odd = odd || worst != 0;
            } else {
                const int tok = (mi & 1) * 8 + (lane & 7);
#pragma unroll
                for (int c2 = 0; c2 < CHUNKS / 2; c2++) {
                    unsigned vr[4];                       // [two chunks][tokens 0-7, 8-15]: a register holds components 2 g, 2 g + 1 of two tokens
                    ldsm_x4_trans(vr, vst + dec_place<CHUNKS>(tok, 2 * c2 + (mi >> 1)));
#pragma unroll
                    for (int h2 = 0; h2 < 2; h2++) {
                        const unsigned w0 = vr[2 * h2] ^ 0x80808080u, w1 = vr[2 * h2 + 1] ^ 0x80808080u;
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float (&acc)[4] = o[2 * (2 * c2 + h2) + e];
                            acc[0] *= corr[0]; acc[1] *= corr[0]; acc[2] *= corr[1]; acc[3] *= corr[1];
                            mma_bf16_16816(acc, pa0, pa1, pa2, pa3, u8x2_to_bf16x2_64th(w0, e ? 0x4341 : 0x4240), u8x2_to_bf16x2_64th(w1, e ? 0x4341 : 0x4240));
                        }
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
            begin_pair();
            look_up(0);
            for (int j = 0; j < DEC_STAGES - 1; j++) issue(j);
        }

        // ---- the four warps' states ----
#pragma unroll
        for (int r = 0; r < 2; r++) {
            l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
            l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
        }
        auto put_state = [&](float* dst) {
#pragma unroll
            for (int i = 0; i < D / 8; i++) {
                *(float2*)(dst + g * D + i * 8 + 2 * t) = make_float2(o[i][0], o[i][1]);
                *(float2*)(dst + (g + 8) * D + i * 8 + 2 * t) = make_float2(o[i][2], o[i][3]);
            }
        };
        auto put_ml = [&](int w) {
            if (t == 0) {
                *(float2*)(st_ml + (w * 16 + g) * 2) = make_float2(m_run[0], l_run[0]);
                *(float2*)(st_ml + (w * 16 + g + 8) * 2) = make_float2(m_run[1], l_run[1]);
            }
        };
        auto take_state = [&](const float* src, int w) {
            float f[2], e[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const float2 ml = *(const float2*)(st_ml + (w * 16 + g + 8 * r) * 2);
                const float m = fmaxf(m_run[r], ml.x);
                f[r] = m_run[r] == -INFINITY ? 0.0f : exp2_approx(m_run[r] - m);
                e[r] = ml.x == -INFINITY ? 0.0f : exp2_approx(ml.x - m);
                l_run[r] = l_run[r] * f[r] + ml.y * e[r];
                m_run[r] = m;
            }
#pragma unroll
            for (int i = 0; i < D / 8; i++) {
                const float2 x = *(const float2*)(src + g * D + i * 8 + 2 * t), y = *(const float2*)(src + (g + 8) * D + i * 8 + 2 * t);
                o[i][0] = o[i][0] * f[0] + x.x * e[0]; o[i][1] = o[i][1] * f[0] + x.y * e[0];
                o[i][2] = o[i][2] * f[1] + y.x * e[1]; o[i][3] = o[i][3] * f[1] + y.y * e[1];
            }
        };
        if (threadIdx.x == 0) odd_value = 0;
        __syncthreads();                                  // (the previous pair's states have been read)
        if (odd) odd_value = 1;
        put_ml(warp);
        if (warp >= 2) put_state(st_o + (warp - 2) * 16 * D);
        __syncthreads();
        if (warp < 2) take_state(st_o + warp * 16 * D, warp + 2);
        __syncwarp();
        if (warp == 1) { put_ml(1); put_state(st_o + 16 * D); }
        __syncthreads();
        const bool split = run0 > 0 || run1 < units;
        const size_t sub = ((size_t)blockIdx.x * 2 + (run0 > 0 ? 0 : 1)) * 16;
        if (odd_value && s.rows > 1) {
            // a value that is no number stands in a block that some rows do not see: row by row, each over what it sees
            for (int i = warp; i < rows; i += DEC_WARPS)
                row_state<D, S8>(a, at_b, s, i / a.G, at_hk * a.G + i % a.G, kb, 4 * run0, min(4 * run1, kb.count), split ? p.ws_o + (sub + i) * D : nullptr,
                                 split ? p.ws_ml + (sub + i) * 2 : nullptr);
        } else if (warp == 0) {
            take_state(st_o + 16 * D, 1);
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int i = g + 8 * r, row = i / a.G;
                if (i >= rows) continue;
                float* wo = p.ws_o + (sub + i) * D;
                unsigned char* out = a.out + (long long)(s.row0 + row) * a.o_rs + (long long)(at_hk * a.G + i - row * a.G) * a.o_hs;
                const float inv = l_run[r] != 0.0f ? 1.0f / l_run[r] : 0.0f;
                if (split && t == 0) *(float2*)(p.ws_ml + (sub + i) * 2) = make_float2(m_run[r], l_run[r]);
#pragma unroll
                for (int n = 0; n < D / 8; n += 2) {
                    // two runs of two neighbours, or (8 bits) four neighbours
                    float x[4] = {o[n][2 * r], o[n][2 * r + 1], o[n + 1][2 * r], o[n + 1][2 * r + 1]};
                    if (S8) { const float y = x[1]; x[1] = x[2]; x[2] = y; }
                    const int d0 = S8 ? 8 * n + 4 * t : 8 * n + 2 * t, d1 = S8 ? d0 + 2 : d0 + 8;
                    if (split) {
                        *(float2*)(wo + d0) = make_float2(x[0], x[1]);
                        *(float2*)(wo + d1) = make_float2(x[2], x[3]);
                    } else {
                        *(unsigned*)(out + 2 * d0) = pack2_bf16(x[0] * inv, x[1] * inv);
                        *(unsigned*)(out + 2 * d1) = pack2_bf16(x[2] * inv, x[3] * inv);
                    }
                }
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
    const long long before = p.prefix[b], n = p.prefix[b + 1] - before;
    if (n == 0) return;
    const long long total = p.prefix[a.c.B] * a.c.Hkv, x = before * a.c.Hkv + hk * n;
    const int pieces = dec_pieces(total, p.ctas, p.min_units);
    // the pieces of the pair's first and last unit
    const int c0 = (int)(((x + 1) * pieces - 1) / total), c1 = (int)(((x + n) * pieces - 1) / total);
    if (c0 == c1) return;
    SeqRows s;
    load_seq(a.c, b, &s);
    if (i >= s.rows * a.G) return;
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
    for (int e = 0; e < N; e += 2) *(unsigned*)(out + 2 * (lane * N + e)) = pack2_bf16(acc[e] * inv, acc[e + 1] * inv);
}

template <int D, bool S8>
int launch_paged_decode_as(DecParams& p, cudaStream_t s) {
    using SM = DecSmem<D, S8>;
    static std::atomic<unsigned long long> attr_devices{0};
    const int arc = once_per_device(attr_devices, [] {
        B200FC_CUDA(cudaFuncSetAttribute(paged_decode_kernel<D, S8>, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::BYTES));
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
    cudaError_t e = cudaLaunchKernelEx(&cfg, paged_decode_kernel<D, S8>, (const DecParams)p);
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
