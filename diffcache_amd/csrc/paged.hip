// Keys and values in pages: writing new tokens' rows, K and the queries rotated by their positions on the way.
//
// A head's numbers are turned in pairs (x_a, x_b) -> (x_a cos t - x_b sin t, x_b cos t + x_a sin t), t = position times the pair's
// frequency.  The product is taken in 64 bits in turns, whole turns dropped, and only then rounded to 32: a position of a
// million times a frequency of 1 has 6e-2 radians of error in 32 bits.  Sine and cosine are the hardware's, which take turns and
// are off by 1.2e-7 at most (100001 places of a turn against 64 bits), far below the 2^-8 of the bf16 result's own
// rounding; the rotation is in fp32 and rounded once.
#include "dc_paged.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMany = 1024;  // tokens, from which a block takes several
// Bytes read and written that no cache holds: beyond the last one's 256 MB the hints save (801 MB 157 -> 143 us, 604 MB 122 -> 109), below they cost
// what the caches would keep (151 MB 27 -> 36 us).
constexpr int64_t kStream = 256ll << 20;

struct AppendArgs {
    DcPages p;
    DcNew t;
    const uint16_t *k, *v, *q;
    uint16_t *q_out;
    const float *inv_freq;
    const int32_t *pos;
    DcTokenStrides ks, vs, qs;
    int n_h, n_q, rot16, n_axes, bound[3];  // rotated columns / 16; the first frequencies of axes 1, 2, 3
    int table_pages, chunks, side;          // blocks of a sequence; heads that a block takes side by side
};

// A block has 256 / (HD / 16) places for heads: `side` of one token, the rest for more tokens.  A thread has 16 numbers of a head, the
// two eights that are turned with each other, and takes the same of every side-th head, so that it needs eight angles in
// all.  ADJACENT: pairs of adjacent columns.  STREAM: what is read and written passes through the caches.
//
// What bounds it: HBM, from some 1000 tokens on.  32601 tokens of 32 + 2 x 8 heads x 128, 801 MB: 143 us = 5.6 TB/s (a large copy 4.9);
// without the hints of STREAM 157, and then with four heads at a time for three 158 and eight heads or more to a thread for four 163.  Eight tokens of as many sequences:
// 4.1 us, a kernel's start and the chain of start, page and row; the host takes 8 us more.
template <int HD, bool ADJACENT, bool STREAM>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(AppendArgs a) {
    constexpr int J = HD / 16, kPlaces = kThreads / J, kBatch = 3;
    const int b = (int)(blockIdx.x / (unsigned)a.chunks), chunk = (int)(blockIdx.x % (unsigned)a.chunks);
    const int j = threadIdx.x % J, place = threadIdx.x / J;
    const DcSpan span = dc_span(a.t, b);
    const int i = chunk * (kPlaces / a.side) + place / a.side, h0 = place % a.side;
    if (i >= span.count) return;
    const bool turned = j < a.rot16;
    const int c0 = ADJACENT || !turned ? 16 * j : 8 * j, c1 = ADJACENT || !turned ? 16 * j + 8 : 8 * (a.rot16 + j);
    const int heads = a.n_q + 2 * a.n_h;
    const uint16_t *q_src = a.q + dc_token_at(a.t, a.qs, span, b, i);
    const uint16_t *k_src = a.k + dc_token_at(a.t, a.ks, span, b, i);
    const uint16_t *v_src = a.v + dc_token_at(a.t, a.vs, span, b, i);
    uint4 x[kBatch][2];
    auto load = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
            int at = h + n * a.side;
            if (at >= heads) continue;
            const uint16_t *src = at < a.n_q ? q_src + at * a.qs.h : at < a.n_q + a.n_h ? k_src + (at - a.n_q) * a.ks.h : v_src + (at - a.n_q - a.n_h) * a.vs.h;
            if constexpr (STREAM) x[n][0] = dc_load_stream16(src + c0), x[n][1] = dc_load_stream16(src + c1);
            else x[n][0] = *reinterpret_cast<const uint4 *>(src + c0), x[n][1] = *reinterpret_cast<const uint4 *>(src + c1);
        }
    };
    load(h0);
    // the token's row; none where the sequence's table has no page of the store there
    const int row = span.start + i, index = row >> a.p.shift;
    int id = -1;
    if (index < a.table_pages) id = a.p.table[(int64_t)b * a.p.table_stride + index];
    const bool held = (unsigned)id < (unsigned)a.p.n_pages;
    const int64_t slot = (int64_t)(row & ((1 << a.p.shift) - 1)) * HD;
    uint16_t *k_dst = a.p.k + (held ? id * a.p.kp : 0) + slot, *v_dst = a.p.v + (held ? id * a.p.vp : 0) + slot;
    uint16_t *q_dst = a.q_out + (int64_t)(span.first + i) * a.n_q * HD;
    float cs[8], sn[8];
    if (turned) {
        int pos[4] = {row, 0, 0, 0};
        if (a.pos) {
            const int32_t *p = a.pos + (int64_t)(span.first + i) * a.n_axes;
#pragma unroll
            for (int n = 0; n < 4; ++n) pos[n] = n < a.n_axes ? p[n] : 0;
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int f = 8 * j + n;
            const int at = f >= a.bound[2] ? pos[3] : f >= a.bound[1] ? pos[2] : f >= a.bound[0] ? pos[1] : pos[0];
            const double t = (double)at * ((double)a.inv_freq[f] * 0.15915494309189533577);
            const float turn = (float)(t - __builtin_rint(t));
            sn[n] = __builtin_amdgcn_sinf(turn), cs[n] = __builtin_amdgcn_cosf(turn);
        }
    }
    auto turn = [&](uint32_t &w0, uint32_t &w1, int n) __attribute__((always_inline)) {
        // ADJACENT: a word is a pair; otherwise two words are two pairs
        if constexpr (ADJACENT) {
            const float a0 = dc_bf16_lo(w0), b0 = dc_bf16_hi(w0), a1 = dc_bf16_lo(w1), b1 = dc_bf16_hi(w1);
            w0 = dc_pack_bf16(a0 * cs[n] - b0 * sn[n], b0 * cs[n] + a0 * sn[n]);
            w1 = dc_pack_bf16(a1 * cs[n + 4] - b1 * sn[n + 4], b1 * cs[n + 4] + a1 * sn[n + 4]);
        } else {
            const float a0 = dc_bf16_lo(w0), a1 = dc_bf16_hi(w0), b0 = dc_bf16_lo(w1), b1 = dc_bf16_hi(w1);
            w0 = dc_pack_bf16(a0 * cs[2 * n] - b0 * sn[2 * n], a1 * cs[2 * n + 1] - b1 * sn[2 * n + 1]);
            w1 = dc_pack_bf16(b0 * cs[2 * n] + a0 * sn[2 * n], b1 * cs[2 * n + 1] + a1 * sn[2 * n + 1]);
        }
    };
    for (int h = h0; h < heads; h += kBatch * a.side) {
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
            const int at = h + n * a.side;
            if (at >= heads) continue;
            if (turned && at < a.n_q + a.n_h) {
                turn(x[n][0].x, x[n][1].x, 0), turn(x[n][0].y, x[n][1].y, 1);
                turn(x[n][0].z, x[n][1].z, 2), turn(x[n][0].w, x[n][1].w, 3);
            }
            uint16_t *dst = at < a.n_q ? q_dst + at * HD : at < a.n_q + a.n_h ? k_dst + (at - a.n_q) * a.p.kh : v_dst + (at - a.n_q - a.n_h) * a.p.vh;
            if (at >= a.n_q && !held) continue;
            if constexpr (STREAM) dc_store_stream16(dst + c0, x[n][0]), dc_store_stream16(dst + c1, x[n][1]);
            else *reinterpret_cast<uint4 *>(dst + c0) = x[n][0], *reinterpret_cast<uint4 *>(dst + c1) = x[n][1];
        }
        load(h + kBatch * a.side);
    }
}

}  // namespace

int dc_check_paged(const char *who, const dc_paged_store &s, const dc_paged_tokens &t, int n_h, int hd, bool written) {
    DC_REQUIRE(hd == 64 || hd == 128 || hd == 256, "%s: head_dim %d unsupported", who, hd);
    DC_REQUIRE(n_h >= 1 && n_h < (1 << 16) && (int64_t)t.n_b * n_h < (1 << 24), "%s: bad sizes or too many units", who);
    DC_REQUIRE(s.page >= 16 && s.page <= (1 << 16) && (s.page & (s.page - 1)) == 0, "%s: a page of %d rows is not a power of two from 16 to 65536", who, s.page);
    DC_REQUIRE(s.n_pages >= 1, "%s: a store needs a page", who);
    DC_REQUIRE(s.k && s.v, "%s: null pointer in the store", who);
    DC_REQUIRE(dc_aligned16(s.k) && dc_aligned16(s.v), "%s: pages must be 16-byte aligned", who);
    DC_REQUIRE(s.k_page_stride % 8 == 0 && s.k_head_stride % 8 == 0 && s.v_page_stride % 8 == 0 && s.v_head_stride % 8 == 0,
               "%s: strides must be multiples of 8 elements", who);
    DC_REQUIRE(s.k_page_stride >= 0 && s.k_head_stride >= 0 && s.v_page_stride >= 0 && s.v_head_stride >= 0, "%s: negative stride in the store", who);
    DC_REQUIRE(t.table && t.table_pages >= 1 && t.table_stride >= t.table_pages, "%s: bad table", who);
    DC_REQUIRE((int64_t)t.table_pages * s.page <= kMostRows, "%s: a table of more than 2^30 rows", who);
    DC_REQUIRE(!(t.cu && t.counts), "%s: cu and counts are for tokens laid out in different ways", who);
    DC_REQUIRE(t.max_new < kMostRows && (t.cu || (int64_t)t.n_b * t.max_new < (1ll << 31)), "%s: too many tokens", who);
    if (written) {
        // a page's heads, and all pages of a head, each with its rows alone
        const int64_t rows = (int64_t)s.page * hd;
        auto apart = [&](int64_t ps, int64_t hs) {
            const bool heads_inside = (n_h == 1 || hs >= rows) && (s.n_pages == 1 || ps >= (n_h - 1) * hs + rows);
            const bool pages_inside = (s.n_pages == 1 || ps >= rows) && (n_h == 1 || hs >= (s.n_pages - 1) * ps + rows);
            return heads_inside || pages_inside;
        };
        DC_REQUIRE(apart(s.k_page_stride, s.k_head_stride) && apart(s.v_page_stride, s.v_head_stride), "%s: pages or heads of the store share their rows", who);
    }
    return DC_OK;
}

extern "C" int dc_paged_append_bf16(const dc_paged_append_args *x, void *stream) {
    const char *who = "dc_paged_append_bf16";
    DC_REQUIRE(x, "%s: null pointer", who);
    const dc_paged_tokens &t = x->tokens;
    DC_REQUIRE(t.n_b >= 0 && t.max_new >= 0 && t.n_tokens >= 0, "%s: bad sizes", who);
    if (t.n_b == 0 || t.max_new == 0) return DC_OK;
    if (const int rc = dc_check_paged(who, x->store, t, x->n_h, x->hd, true)) return rc;
    DC_REQUIRE(x->k_src && x->v_src, "%s: null pointer", who);
    DC_REQUIRE((x->q_src == nullptr) == (x->q_out == nullptr), "%s: q_src and q_out must both be set or both be null", who);
    DC_REQUIRE(x->n_q >= (x->q_src ? 1 : 0) && x->n_q < (1 << 20) && (x->q_src || x->n_q == 0), "%s: n_q does not fit q_src", who);
    DC_REQUIRE(dc_aligned16(x->k_src) && dc_aligned16(x->v_src) && dc_aligned16(x->q_src) && dc_aligned16(x->q_out), "%s: pointers must be 16-byte aligned", who);
    const int64_t strides[9] = {x->k_batch_stride, x->k_token_stride, x->k_head_stride, x->v_batch_stride, x->v_token_stride, x->v_head_stride,
                                x->q_batch_stride, x->q_token_stride, x->q_head_stride};
    for (int64_t s : strides) DC_REQUIRE(s % 8 == 0, "%s: strides must be multiples of 8 elements", who);
    DC_REQUIRE(x->rot >= 0 && x->rot <= x->hd && x->rot % 16 == 0, "%s: %d rotated columns of %d (a multiple of 16)", who, x->rot, x->hd);
    DC_REQUIRE(x->rot == 0 || x->inv_freq, "%s: null pointer", who);
    DC_REQUIRE(x->rot > 0 || !x->q_src, "%s: queries are given, and nothing is rotated", who);
    DC_REQUIRE(x->n_axes >= 1 && x->n_axes <= 4, "%s: %d axes (1 to 4)", who, x->n_axes);
    DC_REQUIRE(x->pos || x->n_axes == 1, "%s: several axes need positions", who);
    AppendArgs a;
    int upto = 0;
    for (int i = 0; i < 4; ++i) {
        if (i < x->n_axes) {
            DC_REQUIRE(x->section[i] >= 0 && x->section[i] <= x->rot / 2, "%s: bad section", who);
            upto += x->section[i];
        }
        if (i < 3) a.bound[i] = i + 1 < x->n_axes ? upto : x->hd;
    }
    DC_REQUIRE((x->n_axes == 1 && upto == 0) || upto == x->rot / 2, "%s: the sections hold %d frequencies, not %d", who, upto, x->rot / 2);
    a.p = dc_pages_of(x->store, t);
    a.t = dc_new_of(t);
    a.k = (const uint16_t *)x->k_src, a.v = (const uint16_t *)x->v_src, a.q = (const uint16_t *)x->q_src, a.q_out = (uint16_t *)x->q_out;
    a.inv_freq = x->inv_freq, a.pos = x->pos;
    a.ks = {strides[0], strides[1], strides[2]}, a.vs = {strides[3], strides[4], strides[5]}, a.qs = {strides[6], strides[7], strides[8]};
    a.n_h = x->n_h, a.n_q = x->n_q, a.rot16 = x->rot / 16, a.n_axes = x->n_axes, a.table_pages = t.table_pages;
    // few tokens: a block each; many: as many to a block as give a thread four heads or more
    const int places = kThreads / (x->hd / 16), heads = x->n_q + 2 * x->n_h;
    const int64_t tokens = t.cu ? t.n_tokens : (int64_t)t.n_b * t.max_new;
    a.side = places;
    if (tokens > kMany)
        while (a.side > 2 && heads < 4 * a.side) a.side /= 2;
    const bool through = tokens * heads * x->hd * 4 > kStream;
    const int per = places / a.side;
    const int64_t chunks = ((int64_t)t.max_new + per - 1) / per;
    DC_REQUIRE(dc_grid_fits((int64_t)t.n_b * chunks, kThreads), "%s: grid too large", who);
    a.chunks = (int)chunks;
    const dim3 grid((unsigned)(t.n_b * chunks)), block(kThreads);
    hipStream_t st = (hipStream_t)stream;
#define DC_APPEND(HD)                                                                                             \
    do {                                                                                                          \
        if (x->interleaved && through) hipLaunchKernelGGL((paged_append_kernel<HD, true, true>), grid, block, 0, st, a); \
        else if (x->interleaved) hipLaunchKernelGGL((paged_append_kernel<HD, true, false>), grid, block, 0, st, a);   \
        else if (through) hipLaunchKernelGGL((paged_append_kernel<HD, false, true>), grid, block, 0, st, a);             \
        else hipLaunchKernelGGL((paged_append_kernel<HD, false, false>), grid, block, 0, st, a);                      \
    } while (0)
    if (x->hd == 64) DC_APPEND(64);
    else if (x->hd == 128) DC_APPEND(128);
    else DC_APPEND(256);
#undef DC_APPEND
    DC_CHECK_LAUNCH(who);
    return DC_OK;
}
