// Attention over the paged cache: checks of the call and the choice of its kernel.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include "paged_common.cuh"
#include "paged_decode.cuh"
#include "paged_prompt.cuh"

namespace b200fc {

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
    // (rows that met a value that is no number are done again from q, when some of out is written)
    if (a.out == a.q) { set_error("paged_attention: out must not be q"); return B200FC_ERR_INVALID; }
    p.scale_log2e = a.scale * 1.4426950408889634f;
    if (!std::isfinite(p.scale_log2e)) { set_error("paged_attention: scale is no number, or 2^127 and more"); return B200FC_ERR_INVALID; }
    if (a.window < 0 || a.sinks < 0) { set_error("paged_attention: negative window or sinks"); return B200FC_ERR_INVALID; }
    if (a.T == 0 || c.B == 0) return B200FC_OK;
    if (a.max_rows < 1) { set_error("paged_attention: max_rows must be at least 1"); return B200FC_ERR_INVALID; }
    if ((long long)a.T * (a.H / c.Hkv) > 1 << 30) { set_error("paged_attention: too many rows and heads for one call"); return B200FC_ERR_INVALID; }
    if ((rc = paged_status("paged_attention", &p.c))) return rc;
    p.q = (const unsigned char*)a.q; p.q_rs = a.q_row_stride; p.q_hs = a.q_head_stride;
    p.out = (unsigned char*)a.out; p.o_rs = a.out_row_stride; p.o_hs = a.out_head_stride;
    p.H = a.H; p.G = a.H / c.Hkv;
    p.window = a.window < p.c.capacity ? a.window : 0;        // (a window as long as the cache is none)
    p.sinks = a.sinks;
    const bool s8 = c.dtype == B200FC_S8;
    p.c.max_rows = a.row_start ? std::min(a.max_rows, a.T) : 1;
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
    if (c.D == 128) return s8 ? launch_paged_prompt<128, true>(p, a.scale, s) : launch_paged_prompt<128, false>(p, a.scale, s);
    return s8 ? launch_paged_prompt<64, true>(p, a.scale, s) : launch_paged_prompt<64, false>(p, a.scale, s);
}

}  // namespace b200fc
