// Appending to the paged cache: rows of k and v enter their sequences' pages, k rotated by its position on the way, and q rotated beside it.  Bound
// by the bytes of the rows (read once, written once); for a few rows by the chain of dependent loads (row -> sequence -> page -> store).
//
// A head's D components are D / 16 items of 16 components that one thread turns by itself: with pairs (i, i + rot / 2) the item holds 8 neighbours of
// either half, with pairs (2 i, 2 i + 1) 16 neighbours; what is not rotated comes in items of 16 neighbours as well.  So every access is 16 bytes
// wide, and q may be turned in place.  A thread keeps its item for all heads of a row: cos and sin are loaded once per row.
// An 8-bit page shares one factor among its tokens, so there a CTA owns all new tokens of a (page, kv head, k or v): it finds their largest
// value, then quantises them, and the page's older tokens anew where the factor grew.
#include <algorithm>
#include <cfloat>
#include "paged.cuh"

namespace b200fc {

namespace {

constexpr int APP_THREADS = 128;

struct AppendParams {
    PagedView c;
    const unsigned char* k; long long k_rs, k_hs;      // bytes
    const unsigned char* v; long long v_rs, v_hs;
    const unsigned char* q; long long q_rs, q_hs;
    unsigned char* q_out; long long qo_rs, qo_hs;
    int H;                                             // query heads, 0 without q
    int rot, interleaved, rot_positions;
    const float* cos; const float* sin; long long rot_stride;   // floats
    const int* positions; long long position_stride;            // entries
    int axes, sec0, sec01;                             // pairs below sec0 take axis 0, below sec01 axis 1
    int check_ctas, page_ctas;                         // the first CTAs look the sequences over, the next (8-bit cache) take pages, the others rows
};

__device__ __forceinline__ float bf_lo(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(unsigned w) { return __uint_as_float(w & 0xffff0000u); }

// where an item's two runs of 8 components begin, and whether it is rotated
struct Item { int lo, hi; bool turned; };
__device__ __forceinline__ Item item_of(const AppendParams& p, int i) {
    const bool turned = 16 * i < p.rot;
    if (turned && !p.interleaved) return {8 * i, p.rot / 2 + 8 * i, true};
    return {16 * i, 16 * i + 8, turned};
}
// cos and sin of the item's 8 pairs for row r at place `place`; false: a position outside the table
__device__ __forceinline__ bool load_turn(const AppendParams& p, int i, int r, int place, float (&cs)[8], float (&sn)[8]) {
    const int pair0 = 8 * i;
    if (p.axes == 1) {
        const int pos = p.positions ? __ldg(p.positions + r) : place;
        const bool ok = (unsigned)pos < (unsigned)p.rot_positions;
        const long long at = (ok ? pos : 0) * p.rot_stride + pair0;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float4 c4 = ok ? __ldg((const float4*)(p.cos + at) + h) : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
            const float4 s4 = ok ? __ldg((const float4*)(p.sin + at) + h) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            cs[4 * h] = c4.x; cs[4 * h + 1] = c4.y; cs[4 * h + 2] = c4.z; cs[4 * h + 3] = c4.w;
            sn[4 * h] = s4.x; sn[4 * h + 1] = s4.y; sn[4 * h + 2] = s4.z; sn[4 * h + 3] = s4.w;
        }
        return ok;
    }
    bool all = true;
    int pos[3];
#pragma unroll
    for (int a = 0; a < 3; a++) pos[a] = p.positions ? __ldg(p.positions + a * p.position_stride + r) : place;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int pair = pair0 + j, at = pair < p.sec0 ? pos[0] : (pair < p.sec01 ? pos[1] : pos[2]);
        const bool ok = (unsigned)at < (unsigned)p.rot_positions;
        cs[j] = ok ? __ldg(p.cos + at * p.rot_stride + pair) : 1.0f;
        sn[j] = ok ? __ldg(p.sin + at * p.rot_stride + pair) : 0.0f;
        all = all && ok;
    }
    return all;
}
// the item's 16 components in fp32: products and sums rounded one by one, so that every way to the same value gives the same bits
__device__ __forceinline__ void turn(const uint4 lo, const uint4 hi, bool turned, bool interleaved, const float (&cs)[8], const float (&sn)[8], float (&y)[16]) {
    const unsigned w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int j = 0; j < 8; j++) { y[2 * j] = bf_lo(w[j]); y[2 * j + 1] = bf_hi(w[j]); }
    if (!turned) return;
    if (interleaved) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float a = y[2 * j], b = y[2 * j + 1];
            y[2 * j] = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(b, sn[j]));
            y[2 * j + 1] = __fadd_rn(__fmul_rn(b, cs[j]), __fmul_rn(a, sn[j]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float a = y[j], b = y[8 + j];
            y[j] = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(b, sn[j]));
            y[8 + j] = __fadd_rn(__fmul_rn(b, cs[j]), __fmul_rn(a, sn[j]));
        }
    }
}
__device__ __forceinline__ void store_bf16(unsigned char* dst, const Item& it, const float (&y)[16]) {
    *(uint4*)(dst + 2 * it.lo) = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
    *(uint4*)(dst + 2 * it.hi) = make_uint4(pack_bf16x2(y[8], y[9]), pack_bf16x2(y[10], y[11]), pack_bf16x2(y[12], y[13]), pack_bf16x2(y[14], y[15]));
}

// Heads of one row: q, and with a bf16 cache k and v.
template <int D, bool S8>
__device__ __forceinline__ void append_row(const AppendParams& p, int r) {
    constexpr int ITEMS = D / 16, SLOTS = APP_THREADS / ITEMS;
    const int i = threadIdx.x % ITEMS, slot = threadIdx.x / ITEMS;
    const Item it = item_of(p, i);
    const int heads = p.H + (S8 ? 0 : 2 * p.c.Hkv);
    auto source = [&](int h) {
        if (h < p.H) return p.q + (long long)r * p.q_rs + (long long)h * p.q_hs;
        const int hk = h - p.H;
        return hk < p.c.Hkv ? p.k + (long long)r * p.k_rs + (long long)hk * p.k_hs : p.v + (long long)r * p.v_rs + (long long)(hk - p.c.Hkv) * p.v_hs;
    };
    // two heads at a time; the first two travel while the row's sequence, page and angles are looked up (5120 rows of 32 + 16 heads: 28.0 us without, 27.3 with)
    uint4 x[2][2];
    auto load = [&](int h) {
#pragma unroll
        for (int u = 0; u < 2; u++)
            if (h + u * SLOTS < heads) {
                const unsigned char* src = source(h + u * SLOTS);
                x[u][0] = *(const uint4*)(src + 2 * it.lo);
                x[u][1] = *(const uint4*)(src + 2 * it.hi);
            }
    };
    int h = slot;
    load(h);
    const int b = find_sequence(p.c, r);
    if (b < 0) return;
    SeqRows s;
    load_seq(p.c, b, &s);
    if (r < s.row0 || r >= s.row0 + s.rows) return;
    const int place = s.len - s.rows + (r - s.row0);
    if (place < 0) return;
    const int page = S8 ? 0 : table_page(p.c, b, place >> p.c.page_shift);
    float cs[8], sn[8];
    bool ok = page >= 0;
    if (it.turned) ok = load_turn(p, i, r, place, cs, sn) && ok;
    if (!ok) report_paged(p.c);
    const long long token = (long long)(place & ((1 << p.c.page_shift) - 1)) * p.c.token_stride + (long long)page * p.c.page_stride;
    for (; h < heads; h += 2 * SLOTS, load(h))
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int hh = h + u * SLOTS;
            if (hh >= heads) break;
            unsigned char* dst;
            bool turned = it.turned;
            if (hh < p.H) {
                dst = p.q_out + (long long)r * p.qo_rs + (long long)hh * p.qo_hs;
            } else {
                if (page < 0) break;
                const int hk = hh - p.H;
                const bool is_v = hk >= p.c.Hkv;
                dst = (is_v ? p.c.v : p.c.k) + token + (long long)(is_v ? hk - p.c.Hkv : hk) * p.c.head_stride;
                turned = turned && !is_v;
            }
            float y[16];
            turn(x[u][0], x[u][1], turned, p.interleaved, cs, sn, y);
            store_bf16(dst, it, y);
        }
}

// four values -> int8, by the factor's reciprocal
__device__ __forceinline__ unsigned quant4(float a, float b, float c, float d, float inv) {
    const unsigned x = (unsigned)f32_to_s8(__fmul_rn(a, inv)) & 255u, y = (unsigned)f32_to_s8(__fmul_rn(b, inv)) & 255u;
    const unsigned z = (unsigned)f32_to_s8(__fmul_rn(c, inv)) & 255u, w = (unsigned)f32_to_s8(__fmul_rn(d, inv)) & 255u;
    return x | y << 8 | z << 16 | w << 24;
}

template <int N> struct Rounds { static constexpr int value = N; };
// All new tokens of one page for a kv head, of k or of v.  segment: the how-manieth page that the call touches, over the sequences in order.
template <int D>
__device__ __forceinline__ void append_page(const AppendParams& p, int segment, int h, bool is_v) {
    constexpr int ITEMS = D / 16, SLOTS = APP_THREADS / ITEMS;
    __shared__ unsigned warp_max[APP_THREADS / 32];
    const int lane = threadIdx.x & 31, shift = p.c.page_shift;
    // ---- which page: every warp counts the touched pages of 32 sequences at a time ----
    SeqRows s{0, 0, 0};
    int b = -1, index = 0;
    for (int b0 = 0; b0 < p.c.B; b0 += 32) {
        SeqRows mine{0, 0, 0};
        if (b0 + lane < p.c.B) load_seq(p.c, b0 + lane, &mine);
        const int n = touched_pages(mine, shift);
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        const unsigned m = __ballot_sync(0xffffffffu, upto > segment);
        if (m) {
            const int src = __ffs(m) - 1;
            s.row0 = __shfl_sync(0xffffffffu, mine.row0, src); s.rows = __shfl_sync(0xffffffffu, mine.rows, src); s.len = __shfl_sync(0xffffffffu, mine.len, src);
            index = (first_token(s) >> shift) + segment - __shfl_sync(0xffffffffu, upto - n, src);
            b = b0 + src;
            break;
        }
        segment -= __shfl_sync(0xffffffffu, upto, 31);
    }
    if (b < 0) return;
    const int page = table_page(p.c, b, index);
    if (page < 0) {
        if (threadIdx.x == 0) report_paged(p.c);
        return;
    }
    const int begin = index << shift, lo = max(first_token(s), begin), hi = min(s.len, begin + (1 << shift));
    float* factor = (is_v ? p.c.v_scale : p.c.k_scale) + (long long)page * p.c.scale_stride + h;
    const bool has_old = lo > begin;
    const float before = has_old ? *factor : 0.0f;
    const unsigned char* src = is_v ? p.v + (long long)h * p.v_hs : p.k + (long long)h * p.k_hs;
    const long long rs = is_v ? p.v_rs : p.k_rs;
    unsigned char* dst = (is_v ? p.c.v : p.c.k) + (long long)page * p.c.page_stride + (long long)h * p.c.head_stride;
    const int i = threadIdx.x % ITEMS, slot = threadIdx.x / ITEMS;
    Item it = item_of(p, i);
    it.turned = it.turned && !is_v;
    // the rotated values of R of the thread's tokens, t0 and every SLOTS-th from there on; behind the last one the last one again, so that all loads travel
    // together
    auto values = [&](auto rounds, int t0, auto& y) {
        constexpr int R = decltype(rounds)::value;
        uint4 x[R][2];
#pragma unroll
        for (int n = 0; n < R; n++) {
            const int t = min(t0 + n * SLOTS, hi - 1);
            const unsigned char* row = src + (long long)(s.row0 + (t - (s.len - s.rows))) * rs;
            x[n][0] = *(const uint4*)(row + 2 * it.lo);
            x[n][1] = *(const uint4*)(row + 2 * it.hi);
        }
#pragma unroll
        for (int n = 0; n < R; n++) {
            const int t = min(t0 + n * SLOTS, hi - 1);
            float cs[8], sn[8];
            if (it.turned && !load_turn(p, i, s.row0 + (t - (s.len - s.rows)), t, cs, sn)) report_paged(p.c);
            turn(x[n][0], x[n][1], it.turned, p.interleaved, cs, sn, y[n]);
        }
    };
    unsigned most = 0;                                               // as bits: infinities and NaN are larger than any number
    float after = 0.0f, inv = 0.0f;
    auto largest = [&](auto rounds, const auto& y) {
#pragma unroll
        for (int n = 0; n < decltype(rounds)::value; n++)
#pragma unroll
            for (int j = 0; j < 16; j++) most = max(most, __float_as_uint(y[n][j]) & 0x7fffffffu);
    };
    auto settle = [&] {                                              // the page's factor, once the whole CTA knows its largest value
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) warp_max[threadIdx.x >> 5] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < APP_THREADS / 32; w++) most = max(most, warp_max[w]);
        after = fmaxf(before, __fdiv_rn(__uint_as_float(most), 127.0f));
        if (after < FLT_MIN) after = 0.0f;                           // (its reciprocal would not be a number of fp32)
        if (most >= 0x7f800000u || before != before) after = __uint_as_float(0x7fc00000u);
        inv = after >= FLT_MIN ? __fdiv_rn(1.0f, after) : 0.0f;
        if (threadIdx.x == 0) *factor = after;
    };
    auto store = [&](auto rounds, int t0, const auto& y) {
#pragma unroll
        for (int n = 0; n < decltype(rounds)::value; n++) {
            const int t = t0 + n * SLOTS;
            if (t >= hi) break;
            unsigned char* d = dst + (long long)(t - begin) * p.c.token_stride;
            *(uint2*)(d + it.lo) = make_uint2(quant4(y[n][0], y[n][1], y[n][2], y[n][3], inv), quant4(y[n][4], y[n][5], y[n][6], y[n][7], inv));
            *(uint2*)(d + it.hi) = make_uint2(quant4(y[n][8], y[n][9], y[n][10], y[n][11], inv), quant4(y[n][12], y[n][13], y[n][14], y[n][15], inv));
        }
    };
    constexpr int R = 4;
    if (hi - lo <= SLOTS) {                                          // a few tokens: one each
        float y[1][16];
        values(Rounds<1>(), lo + slot, y);
        largest(Rounds<1>(), y);
        settle();
        store(Rounds<1>(), lo + slot, y);
    } else if (hi - lo <= R * SLOTS) {                               // the values stay in registers
        float y[R][16];
        values(Rounds<R>(), lo + slot, y);
        largest(Rounds<R>(), y);
        settle();
        store(Rounds<R>(), lo + slot, y);
    } else {                                                         // (pages of 128 tokens of 128 components: everything twice)
        for (int t0 = lo + slot; t0 - slot < hi; t0 += R * SLOTS) {
            float y[R][16];
            values(Rounds<R>(), t0, y);
            largest(Rounds<R>(), y);
        }
        settle();
        for (int t0 = lo + slot; t0 - slot < hi; t0 += R * SLOTS) {
            float y[R][16];
            values(Rounds<R>(), t0, y);
            store(Rounds<R>(), t0, y);
        }
    }
    if (!(after > before) || !has_old) return;
    for (int t = slot; t < lo - begin; t += SLOTS) {
        uint4* d = (uint4*)(dst + (long long)t * p.c.token_stride + 16 * i);
        const uint4 q = *d;
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
        unsigned o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = __fmul_rn((float)(signed char)(w[j] >> (8 * e)), before);
            o[j] = quant4(f[0], f[1], f[2], f[3], inv);
        }
        *d = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// CTAs per SM: 8 bits have as many CTAs as pages, kv heads and k and v, so that those of a step over some 30 sequences are resident together (one row each of 32
// sequences, 8 kv heads: with 4 per SM 5.2 us, 3 per SM 6.3, 5 per SM 4.8, although 88 bytes are spilled); rows have 74 registers.
template <int D, bool S8>
__global__ void __launch_bounds__(APP_THREADS, S8 ? 5 : 6) kv_append_kernel(const AppendParams p) {
    const int cta = (int)blockIdx.x - p.check_ctas;
    if (cta < 0) {                                     // reports sequences whose numbers lie outside their buffers, whether they have rows or not
        const int b = blockIdx.x * APP_THREADS + threadIdx.x;
        SeqRows s;
        if (b < p.c.B && !load_seq(p.c, b, &s)) report_paged(p.c);
        return;
    }
    if (S8 && cta < p.page_ctas) {
        const int part = cta % (2 * p.c.Hkv);
        append_page<D>(p, cta / (2 * p.c.Hkv), part >> 1, part & 1);
        return;
    }
    append_row<D, S8>(p, cta - p.page_ctas);
}

}  // namespace

int launch_kv_append(const b200fc_kv_append_t& a, cudaStream_t s) {
    AppendParams p;
    int rc = paged_view(a.cache, "kv_append", a.T, a.T, a.row_start, &p.c);
    if (rc) return rc;
    const b200fc_paged_cache_t& c = *a.cache;
    if (!a.k || !a.v || (a.q && !a.q_out)) { set_error("kv_append: null pointer"); return B200FC_ERR_INVALID; }
    if (a.q && (a.H <= 0 || a.H > 65535)) { set_error("kv_append: query heads outside 1..65535"); return B200FC_ERR_INVALID; }
    if (unaligned16(a.k, a.k_row_stride, a.k_head_stride) || unaligned16(a.v, a.v_row_stride, a.v_head_stride) ||
        (a.q && (unaligned16(a.q, a.q_row_stride, a.q_head_stride) || unaligned16(a.q_out, a.q_out_row_stride, a.q_out_head_stride)))) {
        set_error("kv_append: q, k, v, q_out and their strides need 16-byte alignment");
        return B200FC_ERR_INVALID;
    }
    if (a.q == a.q_out && a.q && (a.q_row_stride != a.q_out_row_stride || a.q_head_stride != a.q_out_head_stride)) {
        set_error("kv_append: q is rotated in place only with the same strides");
        return B200FC_ERR_INVALID;
    }
    if (a.rot_dim < 0 || a.rot_dim > c.D || a.rot_dim % 16) { set_error("kv_append: rot_dim must be a multiple of 16, at most D"); return B200FC_ERR_INVALID; }
    if (a.rot_dim) {
        if (!a.rot_cos || !a.rot_sin || a.rot_positions <= 0 || unaligned16(a.rot_cos, a.rot_stride, 0) || unaligned16(a.rot_sin, 0, 0) ||
            a.rot_stride < (int64_t)a.rot_dim * 2) {
            set_error("kv_append: the rotation needs 16-byte aligned tables of cos and sin with a row for each position");
            return B200FC_ERR_INVALID;
        }
        if (a.axes != 1 && a.axes != 3) { set_error("kv_append: positions have 1 or 3 axes"); return B200FC_ERR_INVALID; }
        if (a.axes == 3 && (a.section[0] < 0 || a.section[1] < 0 || a.section[2] < 0 || a.section[0] > a.rot_dim || a.section[1] > a.rot_dim ||
                            a.section[2] > a.rot_dim || a.section[0] + a.section[1] + a.section[2] != a.rot_dim / 2)) {
            set_error("kv_append: the sections of three axes must add up to rot_dim / 2 pairs");
            return B200FC_ERR_INVALID;
        }
        if (((uintptr_t)a.positions & 3) || (a.positions && a.axes == 3 && ((a.position_stride & 3) || a.position_stride < (int64_t)a.T * 4))) {
            set_error("kv_append: positions need 4-byte alignment and room for T rows between axes");
            return B200FC_ERR_INVALID;
        }
    }
    if (a.T == 0 || c.B == 0) return B200FC_OK;
    if ((rc = paged_status("kv_append", &p.c))) return rc;
    p.k = (const unsigned char*)a.k; p.k_rs = a.k_row_stride; p.k_hs = a.k_head_stride;
    p.v = (const unsigned char*)a.v; p.v_rs = a.v_row_stride; p.v_hs = a.v_head_stride;
    p.q = (const unsigned char*)a.q; p.q_rs = a.q_row_stride; p.q_hs = a.q_head_stride;
    p.q_out = (unsigned char*)a.q_out; p.qo_rs = a.q_out_row_stride; p.qo_hs = a.q_out_head_stride;
    p.H = a.q ? a.H : 0;
    p.rot = a.rot_dim; p.interleaved = a.interleaved != 0; p.rot_positions = a.rot_positions;
    p.cos = a.rot_cos; p.sin = a.rot_sin; p.rot_stride = a.rot_stride / 4;
    p.positions = a.positions; p.position_stride = a.position_stride / 4;
    p.axes = a.axes; p.sec0 = a.section[0]; p.sec01 = a.section[0] + a.section[1];
    const bool s8 = c.dtype == B200FC_S8;
    // pages that the call can touch: (rows - 1) / page_tokens + 2 of each sequence, and no more than rows
    const long long segments = std::min<long long>(a.T, a.T / c.page_tokens + 2LL * c.B);
    const long long page_ctas = s8 ? segments * 2 * c.Hkv : 0;
    const long long row_ctas = s8 && !p.H ? 0 : (long long)a.T;
    const long long check_ctas = (c.B + APP_THREADS - 1) / APP_THREADS;
    if (page_ctas + row_ctas + check_ctas > 0x7fffffffLL) { set_error("kv_append: too many rows and heads for one call"); return B200FC_ERR_INVALID; }
    p.check_ctas = (int)check_ctas; p.page_ctas = (int)page_ctas;
    const dim3 grid((unsigned)(page_ctas + row_ctas + check_ctas));
    if (c.D == 128) s8 ? kv_append_kernel<128, true><<<grid, APP_THREADS, 0, s>>>(p) : kv_append_kernel<128, false><<<grid, APP_THREADS, 0, s>>>(p);
    else s8 ? kv_append_kernel<64, true><<<grid, APP_THREADS, 0, s>>>(p) : kv_append_kernel<64, false><<<grid, APP_THREADS, 0, s>>>(p);
    B200FC_CUDA(cudaGetLastError());
    count_launch();
    return B200FC_OK;
}

}  // namespace b200fc
