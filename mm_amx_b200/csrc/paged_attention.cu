// Attention over the paged cache: checks of the call and the choice of its kernel.
#include <algorithm>
#include "paged_common.cuh"
#include "paged_decode.cuh"

namespace b200fc {

namespace {

// a warp per row and head
template <int D, bool S8>
__global__ void __launch_bounds__(128) paged_rows_kernel(const PagedAttn p) {
    const int head = blockIdx.y * 4 + (threadIdx.x >> 5), r = blockIdx.x;
    const int b = find_sequence(p.c, r);
    if (b < 0) return;
    SeqRows s;
    if (!load_seq(p.c, b, &s)) {
        if (threadIdx.x == 0) report_paged(p.c);
        return;
    }
    if (r < s.row0 || r >= s.row0 + s.rows || head >= p.H) return;
    const int place = s.len - s.rows + (r - s.row0);
    const KeyBlocks kb = key_blocks(place, place, p.window, p.sinks, 4);
    row_state<D, S8>(p, b, s, r - s.row0, head, kb, 0, kb.count, nullptr, nullptr);
}

}  // namespace

int launch_paged_attention(const b200fc_paged_attention_t& a, cudaStream_t s) {
    PagedAttn p;
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
    const bool s8 = c.dtype == B200FC_S8;
    if (!a.row_start) p.c.max_rows = 1;
    if ((long long)p.c.max_rows * p.G <= 16 && (long long)c.B * c.Hkv < (1LL << 31)) {
        DecParams d;
        d.a = p;
        const bool two = (long long)p.c.max_rows * p.G > 8;
        if (c.D == 128) {
            if (s8) return two ? launch_paged_decode_as<128, true, 2>(d, s) : launch_paged_decode_as<128, true, 1>(d, s);
            return two ? launch_paged_decode_as<128, false, 2>(d, s) : launch_paged_decode_as<128, false, 1>(d, s);
        }
        if (s8) return two ? launch_paged_decode_as<64, true, 2>(d, s) : launch_paged_decode_as<64, true, 1>(d, s);
        return two ? launch_paged_decode_as<64, false, 2>(d, s) : launch_paged_decode_as<64, false, 1>(d, s);
    }
    const dim3 grid((unsigned)a.T, (unsigned)((a.H + 3) / 4));
    if (c.D == 128) s8 ? paged_rows_kernel<128, true><<<grid, 128, 0, s>>>(p) : paged_rows_kernel<128, false><<<grid, 128, 0, s>>>(p);
    else s8 ? paged_rows_kernel<64, true><<<grid, 128, 0, s>>>(p) : paged_rows_kernel<64, false><<<grid, 128, 0, s>>>(p);
    B200FC_CUDA(cudaGetLastError());
    count_launch();
    return B200FC_OK;
}

}  // namespace b200fc
