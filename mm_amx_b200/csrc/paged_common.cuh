// What the kernels of the paged attention share: the call's parameters, instructions, and the attention of one row by one warp.
#pragma once
#include "paged.cuh"
#include "tc_common.cuh"
#include "warp_mma.cuh"

namespace b200fc {

namespace {

struct PagedAttn {
    PagedView c;
    const unsigned char* q; long long q_rs, q_hs;      // bytes
    unsigned char* out; long long o_rs, o_hs;
    int H, G, window, sinks;
    float scale_log2e;                                 // scale * log2(e)
};

// 16 bytes, or zeros
__device__ __forceinline__ void cp_async16_or_zero(unsigned dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(unsigned dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// an 8 x 8 matrix of 16-bit values, two neighbours of row lane / 4 in each lane -> its transpose in the same form
__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// non-zero where one of two bf16 is an infinity or a NaN (all bits of its exponent set)
__device__ __forceinline__ unsigned not_finite2(unsigned w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

// rows of a sequence that sees nothing
template <int D>
__device__ __forceinline__ void zero_rows(const PagedAttn& p, const SeqRows& s) {
    for (int r = s.row0; r < s.row0 + s.rows; r++)
        for (int h = 0; h < p.H; h++) {
            uint4* out = (uint4*)(p.out + (long long)r * p.o_rs + (long long)h * p.o_hs);
#pragma unroll
            for (int i = 0; i < D / 8; i++) out[i] = make_uint4(0, 0, 0, 0);
        }
}

// 8 cached components at p as fp32
template <bool S8>
__device__ __forceinline__ void load8(const unsigned char* p, float (&x)[8]) {
    if constexpr (S8) {
        const uint2 u = *(const uint2*)p;
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = (float)(signed char)((j < 4 ? u.x : u.y) >> (8 * (j & 3)));
    } else {
        const uint4 u = *(const uint4*)p;
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; j++) { x[2 * j] = __uint_as_float(w[j] << 16); x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
    }
}

// The attention of one row (the row-th of sequence b) and query head over blocks [i0, i1) of kb (1 << shift tokens each), by one warp that reads nothing its row does not
// see: a lane scores one token of 32, then every lane sums D / 32 components of the values.  Into out, or (state given) as a sub-state.  flip: the scale's sign has been
// taken off it.  Slow; the
// kernels take it where a value that is no number would reach rows that do not see it through a product of zero.
template <int D, bool S8>
__device__ __noinline__ void row_state(const PagedAttn& p, int b, SeqRows s, int row, int head, KeyBlocks kb, int shift, int i0, int i1, float* state_o, float* state_ml,
                                       unsigned flip) {
    const int lane = threadIdx.x & 31, place = s.len - s.rows + row, hk = head / p.G;
    const unsigned char* q = p.q + (long long)(s.row0 + row) * p.q_rs + (long long)head * p.q_hs;
    constexpr int N = D / 32;
    float acc[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e++) acc[e] = 0.0f;
    for (int x0 = 0; x0 < (i1 - i0) << shift; x0 += 32) {
        const int x = x0 + lane, block = i0 + (x >> shift), tok = (key_block(kb, block) << shift) + (x & ((1 << shift) - 1));
        int page = -1;
        if (block < i1 && key_visible(tok, place, p.window, p.sinks)) {
            page = table_page(p.c, b, tok >> p.c.page_shift);
            if (page < 0) report_paged(p.c);
        }
        const long long at = (long long)page * p.c.page_stride + (long long)hk * p.c.head_stride + (long long)(tok & ((1 << p.c.page_shift) - 1)) * p.c.token_stride;
        float score = -INFINITY, vs = 1.0f;
        if (page >= 0) {
            float dot = 0.0f;
#pragma unroll 4
            for (int d = 0; d < D; d += 8) {
                float k[8], y[8];
                load8<S8>(p.c.k + at + d * (S8 ? 1 : 2), k);
                load8<false>(q + 2 * d, y);
#pragma unroll
                for (int e = 0; e < 8; e++) dot = fmaf(y[e], k[e], dot);
            }
            if (flip) dot = -dot;
            if (S8) { dot *= p.c.k_scale[page * p.c.scale_stride + hk]; vs = p.c.v_scale[page * p.c.scale_stride + hk]; }
            score = dot * p.scale_log2e;
        }
        float top = score;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m, top);
        if (m_new == -INFINITY && !__any_sync(0xffffffffu, score != score)) continue;
        const float f = exp2_approx(m - m_new), w = page >= 0 ? exp2_approx(score - m_new) : 0.0f;
        float sum = w;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = fmaf(l, f, sum);
        m = m_new;
#pragma unroll
        for (int e = 0; e < N; e++) acc[e] *= f;
        for (int t = 0; t < 32; t++) {
            if (__shfl_sync(0xffffffffu, page, t) < 0) continue;
            const float wt = __shfl_sync(0xffffffffu, w * vs, t);
            const long long vt = __shfl_sync(0xffffffffu, at, t);
#pragma unroll
            for (int e = 0; e < N; e++) {
                const int d = lane * N + e;
                const float v = S8 ? (float)(signed char)p.c.v[vt + d] : __uint_as_float((unsigned)*(const unsigned short*)(p.c.v + vt + 2 * d) << 16);
                acc[e] = fmaf(wt, v, acc[e]);
            }
        }
    }
    if (state_o) {
#pragma unroll
        for (int e = 0; e < N; e++) state_o[lane * N + e] = acc[e];
        if (lane == 0) *(float2*)state_ml = make_float2(m, l);
    } else {
        unsigned short* out = (unsigned short*)(p.out + (long long)(s.row0 + row) * p.o_rs + (long long)head * p.o_hs);
#pragma unroll
        for (int e = 0; e < N; e++) out[lane * N + e] = f32_to_bf16_bits(l != 0.0f ? acc[e] / l : 0.0f);
    }
}

}  // namespace

}  // namespace b200fc
