// Attention over the paged cache.
#include "paged.cuh"

namespace b200fc {

namespace {

struct PagedAttnParams {
    PagedView c;
    const unsigned char* q; long long q_rs, q_hs;      // bytes
    unsigned char* out; long long o_rs, o_hs;
    int H, G, window, sinks;
    float scale_log2e;
};

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

// One warp per row and query head: 32 tokens at a time, a lane scores one token, then every lane sums D / 32 components of the values.
template <int D, bool S8>
__global__ void __launch_bounds__(128) paged_rows_kernel(const PagedAttnParams p) {
    __shared__ float q_s[4][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.y * 4 + warp, r = blockIdx.x;
    const int b = find_sequence(p.c, r);
    if (b < 0) return;
    SeqRows s;
    if (!load_seq(p.c, b, &s)) {
        if (threadIdx.x == 0) report_paged(p.c);
        return;
    }
    if (r < s.row0 || r >= s.row0 + s.rows || head >= p.H) return;
    const int place = s.len - s.rows + (r - s.row0), hk = head / p.G;
    const unsigned short* q = (const unsigned short*)(p.q + (long long)r * p.q_rs + (long long)head * p.q_hs);
    for (int d = lane; d < D; d += 32) q_s[warp][d] = __uint_as_float((unsigned)q[d] << 16);
    __syncwarp();
    constexpr int N = D / 32;
    float acc[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e++) acc[e] = 0.0f;
    const KeyBlocks kb = key_blocks(place, place, p.window, p.sinks, 4);
    for (int i = 0; i < kb.count; i += 2) {
        const int block = i + (lane >> 4), tok = key_block(kb, block) * 16 + (lane & 15);
        int page = -1;
        const bool seen = block < kb.count && key_visible(tok, place, p.window, p.sinks);
        if (seen) {
            page = table_page(p.c, b, tok >> p.c.page_shift);
            if (page < 0) report_paged(p.c);
        }
        const long long at = (long long)page * p.c.page_stride + (long long)hk * p.c.head_stride + (long long)(tok & ((1 << p.c.page_shift) - 1)) * p.c.token_stride;
        float score = -INFINITY, vs = 1.0f;
        if (page >= 0) {
            float dot = 0.0f;
            for (int d = 0; d < D; d += 8) {
                float k[8];
                load8<S8>(p.c.k + at + d * (S8 ? 1 : 2), k);
#pragma unroll
                for (int e = 0; e < 8; e++) dot = fmaf(q_s[warp][d + e], k[e], dot);
            }
            if (S8) { dot *= p.c.k_scale[page * p.c.scale_stride + hk]; vs = p.c.v_scale[page * p.c.scale_stride + hk]; }
            score = dot * p.scale_log2e;
        }
        float top = score;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m, top);
        if (m_new == -INFINITY) continue;
        const float f = exp2f(m - m_new), w = page >= 0 ? exp2f(score - m_new) : 0.0f;
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
    unsigned short* out = (unsigned short*)(p.out + (long long)r * p.o_rs + (long long)head * p.o_hs);
#pragma unroll
    for (int e = 0; e < N; e++) out[lane * N + e] = f32_to_bf16_bits(l != 0.0f ? acc[e] / l : 0.0f);
}

}  // namespace

int launch_paged_attention(const b200fc_paged_attention_t& a, cudaStream_t s) {
    PagedAttnParams p;
    int rc = paged_view(a.cache, "paged_attention", a.T, a.max_rows, a.row_start, &p.c);
    if (rc) return rc;
    const b200fc_paged_cache_t& c = *a.cache;
    if (!a.q || !a.out) { set_error("paged_attention: null pointer"); return B200FC_ERR_INVALID; }
    if (a.H <= 0 || a.H > 65535 || a.H % c.Hkv) { set_error("paged_attention: need H %% Hkv == 0 and at most 65535 query heads"); return B200FC_ERR_INVALID; }
    if (unaligned16(a.q, a.q_row_stride, a.q_head_stride) || unaligned16(a.out, a.out_row_stride, a.out_head_stride)) {
        set_error("paged_attention: q, out and their strides need 16-byte alignment");
        return B200FC_ERR_INVALID;
    }
    if (a.window < 0 || a.sinks < 0) { set_error("paged_attention: negative window or sinks"); return B200FC_ERR_INVALID; }
    if (!a.row_start && a.max_rows < 1) { set_error("paged_attention: max_rows must be at least 1"); return B200FC_ERR_INVALID; }
    if (a.T == 0 || c.B == 0) return B200FC_OK;
    if ((rc = paged_status("paged_attention", &p.c))) return rc;
    p.q = (const unsigned char*)a.q; p.q_rs = a.q_row_stride; p.q_hs = a.q_head_stride;
    p.out = (unsigned char*)a.out; p.o_rs = a.out_row_stride; p.o_hs = a.out_head_stride;
    p.H = a.H; p.G = a.H / c.Hkv;
    p.window = a.window; p.sinks = a.sinks;
    p.scale_log2e = a.scale * 1.4426950408889634f;
    const dim3 grid((unsigned)a.T, (unsigned)((a.H + 3) / 4));
    const bool s8 = c.dtype == B200FC_S8;
    if (c.D == 128) s8 ? paged_rows_kernel<128, true><<<grid, 128, 0, s>>>(p) : paged_rows_kernel<128, false><<<grid, 128, 0, s>>>(p);
    else s8 ? paged_rows_kernel<64, true><<<grid, 128, 0, s>>>(p) : paged_rows_kernel<64, false><<<grid, 128, 0, s>>>(p);
    B200FC_CUDA(cudaGetLastError());
    count_launch();
    return B200FC_OK;
}

}  // namespace b200fc
