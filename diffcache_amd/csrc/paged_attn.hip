// Attention over keys and values in pages: the entry point, the kernel for up to 16 rows of queries of a KV head (one token, or
// a few drafted ones), and the join of the parts of a long axis.
#include "dc_paged.h"
#include <math.h>

namespace {

constexpr int kThreads = 256, kWaves = 4, kMostWaves = 8, kRows = 16;

// out = sum_r p_r v_r / sum_r p_r with p_r = exp(scale q k_r - m), over the rows that a token attends to.  A unit's (one sequence's, one KV
// head's) rows are cut into steps of 16 TILES, its steps into parts, a block each, whose waves take them in turn; a wave
// keeps its running maximum, sum and weighted rows in registers, so K and V are read once and nothing is written but the parts' results.
//
//   S = K Q^T   v_mfma_f32_16x16x32_bf16 over 16 rows (M), 16 (token, head) pairs (N) and 32 columns.  Lane (q, c) = (lane / 16, lane % 16)
//               loads 16 bytes of one row, its four lanes side by side.
//   softmax     in powers of two, fp32.  Lane c keeps pair c's maximum, which moves only where a logit passes it by more than 8: nothing
//               crosses lanes from step to step, and a weight is at most 2^8 of fp32 sums.
//   O = P V     M = 16 pairs, N = 16 of the hd columns, K = 32 rows of two tiles, P as it stands in the lanes.  P is the sum of two bf16
//               numbers: 2^-16 of a weight is lost at most, far below the output's own 2^-8; the matrix unit has the time.  Lane (q, c) loads
//               adjacent columns of its own rows; byte permutes put the rows of a column together.
//
// Which row of a tile is which row of M is free as long as K and V agree: M row 4 q + i is the tile's row 4 i + q, so that every
// load takes whole lines.  A tile of 16 rows lies in one page, so its address is the scalar unit's; page ids are read a step ahead.
//
// What bounds it: HBM from some 300 MB on.  8 x 131072 rows of 8 heads x 128 with groups of 4, 4.29 GB: 626 us = 6.9 TB/s (pages of 16 rows 647);
// 8 x 65536 of 4 heads x 256 321 us = 6.7 TB/s; 16 x 65536 of 8 heads x 64 343 us = 6.3; four drafted tokens of 8 x 32601 rows 171 us = 6.2.  A step of
// 32 rows x 128 columns is 50 vector, 6 matrix and 4 load instructions for each 4 KB; the vector unit issues a fifth of the time.  Below, the chain of start,
// page ids, rows, products and the join: 32601 rows of 8 units 23.9 + 4.0 us (the bytes 19), 517 rows in one kernel 9.7 us, 64 rows 5.
// Steps of 64 rows at 128 columns (two blocks to a CU) took 10.8 us for 517 rows and 279 for 48 x 8192 (242 now), the large ones the same.
// At 256 columns 25 registers spilled cost 447 us for 321.
template <int HD, int TILES>
struct Rows {
    static constexpr int STEP = 16 * TILES, CH = HD / 32, EPL = HD / 16, VW = EPL / 2;

    static constexpr bool kQueryInLds = HD == 256;  // (its registers are 25 too many there)
    dc_u32x4 bq[kQueryInLds ? 1 : CH];
    dc_u32x4 kw[TILES][CH];
    uint32_t vw[TILES * 4][VW];
    dc_f32x4 acc[EPL];
    float m, l;
    int q, c;

    __device__ __forceinline__ void start(int lane) {
        q = lane >> 4, c = lane & 15;
#pragma unroll
        for (int j = 0; j < EPL; ++j) acc[j] = dc_f32x4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY, l = 0.f;
    }
    // columns 32 s + 8 q .. of the queries of pair c: src its column 0, lds 16 HD numbers for all waves
    __device__ __forceinline__ void load_q(const uint16_t *src, dc_u32x4 *lds, int wave) {
        if constexpr (kQueryInLds) {
            if (wave == 0) {
#pragma unroll
                for (int s = 0; s < CH; ++s) lds[place(s)] = *reinterpret_cast<const dc_u32x4 *>(src + 32 * s + 8 * q);
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int s = 0; s < CH; ++s) bq[s] = *reinterpret_cast<const dc_u32x4 *>(src + 32 * s + 8 * q);
        }
    }
    __device__ __forceinline__ int place(int s) const { return c * (HD / 8) + ((4 * s + q) ^ c); }  // (16 pairs' same chunk in 16 places)
    __device__ __forceinline__ dc_u32x4 query(const dc_u32x4 *lds, int s) const {
        if constexpr (kQueryInLds) return lds[place(s)];  // (every step anew, for what the barrier in logits() tells the compiler)
        else return bq[s];
    }
    // lane (q, c) has columns 32 s + 8 q .. of row 4 (c % 4) + c / 4 of every tile
    __device__ __forceinline__ void load_k(const uint16_t *const (&tile)[TILES]) {
        const int off = (4 * (c & 3) + (c >> 2)) * HD + 8 * q;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int s = 0; s < CH; ++s) kw[t][s] = __builtin_nontemporal_load(reinterpret_cast<const dc_u32x4 *>(tile[t] + off + 32 * s));
    }
    // column j of lane c's
    static __device__ __forceinline__ int column(int c, int j) { return HD == 64 ? 4 * c + j : 128 * (j / 8) + 8 * c + j % 8; }
    // lane (q, c) has its columns of the rows 4 i + q of every tile
    __device__ __forceinline__ void load_v(const uint16_t *const (&tile)[TILES]) {
        const int off = q * HD + column(c, 0);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t *src = tile[t] + off + 4 * i * HD;
                if constexpr (HD == 64) {
                    const dc_u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const dc_u32x2 *>(src));
                    vw[4 * t + i][0] = w.x, vw[4 * t + i][1] = w.y;
                } else {
#pragma unroll
                    for (int u = 0; u < HD / 128; ++u) {
                        const dc_u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const dc_u32x4 *>(src + 128 * u));
#pragma unroll
                        for (int e = 0; e < 4; ++e) vw[4 * t + i][4 * u + e] = w[e];
                    }
                }
            }
    }

    // x[t][i]: tile t, row 4 i + q, pair c
    __device__ __forceinline__ void logits(float scale, const dc_u32x4 *lds, float (&x)[TILES][4]) const {
        if constexpr (kQueryInLds) asm volatile("" ::: "memory");
        dc_f32x4 s[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) s[t] = dc_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const dc_bf16x8 w = __builtin_bit_cast(dc_bf16x8, query(lds, j));
#pragma unroll
            for (int t = 0; t < TILES; ++t) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dc_bf16x8, kw[t][j]), w, s[t], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[t][i] = s[t][i] * scale;
    }

    // a new maximum for every pair, and what was summed so far brought to it
    __device__ __forceinline__ void raise(float most) {
        const float to = fmaxf(m, dc_over16(most, [](float a, float b) { return fmaxf(a, b); }));
        if (__any(m > kNoLogit)) {
            const float f = m > kNoLogit ? __builtin_amdgcn_exp2f(m - to) : 1.f;  // (nothing was summed, or what is no number)
            l *= f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float g = __shfl(f, 4 * q + i, 64);
#pragma unroll
                for (int j = 0; j < EPL; ++j) acc[j][i] *= g;
            }
        }
        m = to;
    }
    __device__ __forceinline__ void weigh(float (&x)[TILES][4]) {
        float most = -INFINITY;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, x[t][i]);
        if (__any(most > m + 8.f)) raise(most);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[t][i] = __builtin_amdgcn_exp2f(dc_less(x[t][i], m));
                l += x[t][i];
            }
    }

    // whether a number of the step that load_v brought is not finite
    __device__ __forceinline__ bool unbounded() const {
        DcUnbounded u;
#pragma unroll
        for (int t = 0; t < TILES * 4; ++t)
#pragma unroll
            for (int i = 0; i < VW; ++i) u.look(vw[t][i]);
        return u.any();
    }

    __device__ __forceinline__ void bound() {
#pragma unroll
        for (int t = 0; t < TILES * 4; ++t)
#pragma unroll
            for (int i = 0; i < VW; ++i) vw[t][i] = dc_finite(vw[t][i]);
    }
    // acc += what is not finite of one row of V (src, the row's column 0), for the pairs that attend to it
    __device__ __forceinline__ void add_unbounded(const uint16_t *src, const bool (&in)[4]) {
#pragma unroll
        for (int j = 0; j < EPL; j += 4) {
            const uint2 w = *reinterpret_cast<const uint2 *>(src + column(c, j));
            const float x[4] = {dc_only_unbounded(dc_bf16_lo(w.x)), dc_only_unbounded(dc_bf16_hi(w.x)), dc_only_unbounded(dc_bf16_lo(w.y)),
                                dc_only_unbounded(dc_bf16_hi(w.y))};
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j + e][i] += in[i] ? x[e] : 0.f;
        }
    }

    // acc += P V over the step that load_v brought
    __device__ __forceinline__ void add(const float (&x)[TILES][4]) {
#pragma unroll
        for (int u = 0; u < TILES / 2; ++u) {
            dc_u32x4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x0 = x[2 * u + i / 2][2 * (i % 2)], x1 = x[2 * u + i / 2][2 * (i % 2) + 1];
                hi[i] = dc_pack_bf16(x0, x1);
                lo[i] = dc_pack_bf16(x0 - dc_bf16_lo(hi[i]), x1 - dc_bf16_hi(hi[i]));
            }
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                const uint32_t sel = j % 2 ? 0x07060302u : 0x05040100u;  // the high or the low halves of two words
                dc_u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(vw[8 * u + 2 * i + 1][j / 2], vw[8 * u + 2 * i][j / 2], sel);
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dc_bf16x8, lo), __builtin_bit_cast(dc_bf16x8, w), acc[j], 0, 0, 0);
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dc_bf16x8, hi), __builtin_bit_cast(dc_bf16x8, w), acc[j], 0, 0, 0);
            }
        }
    }

    // dst[pair][column] = the wave's sums
    __device__ __forceinline__ void finish(float *dst, int pairs) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (4 * q + i < pairs) {
#pragma unroll
                for (int j = 0; j < EPL; j += 4)
                    *reinterpret_cast<float4 *>(dst + (4 * q + i) * HD + column(c, j)) = make_float4(acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]);
            }
        }
    }
};

template <int HD, int TILES>
__global__ __launch_bounds__(kMostWaves * 64, HD == 128 ? 3 : 2) void paged_rows_kernel(DcPagedAttn a) {
    using T = Rows<HD, TILES>;
    constexpr int STEP = T::STEP;
    extern __shared__ float s_dyn[];
    const int waves = a.waves;
    __shared__ dc_u32x4 s_q[T::kQueryInLds ? kRows * HD / 8 : 1];
    float *s_m = s_dyn, *s_l = s_dyn + waves * kRows, *s_acc = s_dyn + 2 * waves * kRows;  // [wave][16], [wave][16], [wave][pairs * HD]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), G = a.group;
    int b = blockIdx.x, h = blockIdx.y, part_ = 0, parts = 1;
    int64_t slot = 0;
    if (a.at_once) {
        const int x = (int)(blockIdx.x / (unsigned)a.n_h);
        const DcItem d = dc_deal<STEP, false>(a, x, lane);
        if (d.part >= d.parts) return;
        b = d.b, h = (int)(blockIdx.x % (unsigned)a.n_h), part_ = d.part, parts = d.parts, slot = d.slot + (int64_t)part_ * a.n_h + h;
    }
    const DcSpan span = dc_span(a.t, b);
    if (span.count == 0) return;
    const int pairs = span.count * G, p_lo = span.start, p_hi = span.start + span.count - 1;
    const DcSteps st = dc_steps<STEP>(a, p_lo, p_hi);
    const int per = (st.steps + parts - 1) / parts, begin = part_ * per, end = begin + per < st.steps ? begin + per : st.steps;
    if (begin >= end && parts > 1) {  // a part without rows: the join takes nothing of it
        if (tid < pairs) reinterpret_cast<float2 *>(a.ws_ml)[slot * a.tile_rows + tid] = make_float2(-INFINITY, 0.f);
        return;
    }
    T w;
    w.start(lane);
    const int pair = w.c < pairs ? w.c : pairs - 1, token = pair / G;  // (the last pair again in the place of one that does not exist)
    w.load_q(a.q + dc_token_at(a.t, a.qs, span, b, token) + (int64_t)(h * G + pair % G) * a.qs.h, s_q, wave);
    const DcReach reach = dc_reach(a, span.start + token);

    const uint16_t *kh = a.p.k + h * a.p.kh, *vh = a.p.v + h * a.p.vh;
    const int32_t *table = a.p.table + (int64_t)b * a.p.table_stride;
    const int last_page = (a.n_rows - 1) >> a.p.shift, mask = (1 << a.p.shift) - 1;
    // a wave's steps are every waves-th of the block's, from a start of its block's own on
    const int mine = end > begin + wave ? (end - begin - wave + waves - 1) / waves : 0;
    int at = (int)(((uint64_t)((uint32_t)blockIdx.x * 0x9e3779b9u) * (uint32_t)mine) >> 32);
    int id[TILES], row = 0;
    auto look = [&]() __attribute__((always_inline)) {
        row = st.row(begin + wave + at * waves, STEP);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int page = (row + 16 * t) >> a.p.shift;
            id[t] = dc_page_id(a.p, table, page < last_page ? page : last_page);
        }
    };
    const uint16_t *kt[TILES], *vt[TILES];
    int held_row = 0, live = 0;  // of the step in the registers: its first row, and a bit for each tile that has a page
    auto place = [&]() __attribute__((always_inline)) {
        held_row = row, live = 0;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int64_t page = id[t] < 0 ? 0 : id[t];
            live |= id[t] < 0 ? 0 : 1 << t;
            const int64_t in = (int64_t)((row + 16 * t) & mask) * HD;
            kt[t] = kh + page * a.p.kp + in, vt[t] = vh + page * a.p.vp + in;
        }
    };
    if (mine > 0) {
        w.m = kNoLogit;
        look();
        place();
        w.load_k(kt);
        w.load_v(vt);
        at = at + 1 < mine ? at + 1 : 0;
        look();
    }
    for (int n = 0; n < mine; ++n) {
        float x[TILES][4];
        w.logits(a.scale, s_q, x);
        const bool more = n + 1 < mine;
        const int r0 = held_row, have = live;
        if (more) {
            place();
            w.load_k(kt);
            at = at + 1 < mine ? at + 1 : 0;
            look();
        }
        const bool whole = have == (1 << TILES) - 1 && dc_whole(a, p_lo, p_hi, r0, STEP);  // every row for every pair
        if (!whole) {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!((have >> t) & 1) | !reach.has(r0 + 16 * t + 4 * i + w.q)) x[t][i] = -INFINITY;
        }
        // (in every step, for P's second part may be negative: the sum of its products with an infinity would be NaN)
        const bool odd = w.unbounded();
        if (odd) w.bound();
        w.weigh(x);
        w.add(x);
        if (odd) {
            DcReach of[4];  // of the pairs whose sums the lane has
#pragma unroll
            for (int i = 0; i < 4; ++i) of[i] = dc_reach(a, span.start + (4 * w.q + i < pairs ? 4 * w.q + i : pairs - 1) / G);
            for (int r = 0; r < STEP; ++r) {
                const int page = (r0 + r) >> a.p.shift, at_id = dc_page_id(a.p, table, page < last_page ? page : last_page);
                if (at_id < 0) continue;
                bool in[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) in[i] = of[i].has(r0 + r);
                w.add_unbounded(vh + at_id * a.p.vp + (int64_t)((r0 + r) & mask) * HD, in);
            }
        }
        if (more) w.load_v(vt);
    }

    // the pairs' statistics and sums over the block's waves
    const float l = dc_over16(w.l, [](float a, float b) { return a + b; });
    if (lane < kRows) s_m[wave * kRows + lane] = w.m, s_l[wave * kRows + lane] = l;
    w.finish(s_acc + wave * pairs * HD, pairs);
    __syncthreads();
    // (four columns at a time: the weights are made again for every one of a thread's pieces, 16 heads of 256 columns 16.1 us by single numbers, 8.5 so)
    constexpr int kLanes = HD / 4;
    for (int o = tid; o < pairs * kLanes; o += waves * 64) {
        const int r = o / kLanes, column = 4 * (o % kLanes);
        // (without a branch to a wave: the first one again in the place of those that a block of four does not have)
        float m[kMostWaves], ls[kMostWaves];
        float4 part[kMostWaves];
#pragma unroll
        for (int i = 0; i < kMostWaves; ++i) {
            const int x = i < waves ? i : 0;
            m[i] = s_m[x * kRows + r], ls[i] = s_l[x * kRows + r], part[i] = reinterpret_cast<const float4 *>(s_acc)[x * pairs * kLanes + o];
        }
        float top = m[0];
#pragma unroll
        for (int i = 1; i < kMostWaves; ++i) top = fmaxf(top, m[i]);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < kMostWaves; ++i) {
            const bool is = i < waves;
            const float f = is ? dc_weight(m[i], top) : 0.f;
            sum.x = fmaf(f, is ? part[i].x : 0.f, sum.x), sum.y = fmaf(f, is ? part[i].y : 0.f, sum.y);
            sum.z = fmaf(f, is ? part[i].z : 0.f, sum.z), sum.w = fmaf(f, is ? part[i].w : 0.f, sum.w);
            total += is ? dc_share(m[i], ls[i], top) : 0.f;
        }
        if (parts > 1) {
            *reinterpret_cast<float4 *>(a.ws_acc + (slot * a.tile_rows + r) * HD + column) = sum;
            if (column == 0) reinterpret_cast<float2 *>(a.ws_ml)[slot * a.tile_rows + r] = make_float2(top, total);
        } else {
            const int64_t dst = (int64_t)(span.first + r / G) * a.n_h * G + h * G + r % G;
            const float by = total == 0.f ? 1.f : total;
            *reinterpret_cast<uint2 *>(a.out + dst * HD + column) = make_uint2(dc_pack_bf16(sum.x / by, sum.y / by), dc_pack_bf16(sum.z / by, sum.w / by));
            if (a.lse && column == 0) a.lse[dst] = dc_log_sum(top, total);
        }
    }
}

// The parts of one row joined by a block: HD / 4 threads to a part, all of a round's parts asked for before any weight is known.
template <int HD, int STEP>
__global__ __launch_bounds__(kThreads) void paged_join_kernel(DcPagedAttn a) {
    constexpr int kLanes = HD / 4, kParts = kThreads / kLanes, kBatch = HD == 256 ? 8 : 4;
    __shared__ float4 s_acc[kThreads];
    const int tid = threadIdx.x, lane = tid & 63, h = (int)(blockIdx.x % (unsigned)a.n_h), r = blockIdx.y;
    const DcItem d = dc_deal<STEP, false, true>(a, (int)(blockIdx.x / (unsigned)a.n_h), lane);
    if (d.parts < 2) return;
    const DcSpan span = dc_span(a.t, d.b);
    const int token = r / a.group, n = d.parts;
    if (token >= span.count) return;
    const int64_t dst = (int64_t)(span.first + token) * a.n_h * a.group + h * a.group + r % a.group;
    const int64_t slot0 = (d.slot + h) * a.tile_rows + r, step = (int64_t)a.n_h * a.tile_rows;
    const float2 *ml = reinterpret_cast<const float2 *>(a.ws_ml) + slot0;
    const float4 *pa = reinterpret_cast<const float4 *>(a.ws_acc) + slot0 * kLanes + tid % kLanes;
    float4 v[kBatch];
    float2 o[kBatch];
    auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {  // (the last part again where there are no more)
            const int s = s0 + i * kParts;
            const int64_t at = (s < n ? s : n - 1) * step;
            o[i] = ml[at], v[i] = pa[at * kLanes];
        }
    };
    const float2 own = lane < n ? ml[lane * step] : make_float2(-INFINITY, 0.f);
    load(tid / kLanes);
    auto all = [&](float x, auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) x = f(x, __shfl_xor(x, d, 64));
        return dc_over16(x, f);
    };
    float top = own.x;
    for (int s = lane + 64; s < n; s += 64) top = fmaxf(top, ml[s * step].x);
    top = all(top, [](float x, float y) { return fmaxf(x, y); });
    float total = dc_share(own.x, own.y, top);
    for (int s = lane + 64; s < n; s += 64) total += dc_share(ml[s * step].x, ml[s * step].y, top);
    total = all(total, [](float x, float y) { return x + y; });
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = tid / kLanes;;) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            // (a part without rows has no sums in the workspace)
            const bool in = s0 + i * kParts < n && o[i].x > -INFINITY;
            const float f = in ? dc_weight(o[i].x, top) : 0.f;
            acc.x = fmaf(f, in ? v[i].x : 0.f, acc.x), acc.y = fmaf(f, in ? v[i].y : 0.f, acc.y);
            acc.z = fmaf(f, in ? v[i].z : 0.f, acc.z), acc.w = fmaf(f, in ? v[i].w : 0.f, acc.w);
        }
        s0 += kBatch * kParts;
        if (s0 - tid / kLanes >= n) break;
        load(s0);
    }
    s_acc[tid] = acc;
    __syncthreads();
    if (tid < HD) {
        const float *x = reinterpret_cast<const float *>(s_acc) + tid;
        float sum = x[0];
#pragma unroll
        for (int i = 1; i < kParts; ++i) sum += x[i * HD];
        a.out[dst * HD + tid] = dc_f32_to_bf16(sum / (total == 0.f ? 1.f : total));
    }
    if (a.lse && tid == 0) a.lse[dst] = dc_log_sum(top, total);
}

// ---- host -----------------------------------------------------------------------------------------------------------

constexpr int row_tiles(int hd) { return hd == 64 ? 4 : 2; }
constexpr int rows_at_once(int hd) { return hd == 256 ? 512 : 768; }  // two or three blocks to a CU
// Rows times columns up to which a unit is one block of eight waves, which writes the output itself: 384 KB of K and V, some 2 us of what a CU
// can read more, but less than a second kernel that joins parts where the host waits for its launches (one sequence of 8 heads x
// 128: 700 rows 10.7 us, in parts 8.9, called one after another 11.0 and 15.4; 32 sequences 17.2 and 22.7 us).
constexpr int64_t kAlone = 768 * 128;

struct Cut {
    bool chunk, deal, join;   // deal: blocks find their items; join: some may be parts
    int waves, tiles, tile_rows, at_once, least, fewest;
    unsigned sharers;         // blocks of the chunks' join to each part
    int64_t blocks, places;   // places: of parts, in the workspace
};
// tokens: of all sequences together, where they are packed; else 0
Cut cut_of(int64_t n_b, int n_h, int group, int hd, int64_t rows, int max_new, int64_t tokens) {
    Cut c;
    const int64_t n_units = n_b * n_h;
    c.chunk = (int64_t)max_new * group > kRows;
    if (c.chunk) {
        c.tile_rows = kChunkRows, c.waves = 4, c.at_once = dc_chunk_at_once(hd);
        c.tiles = (int)(((int64_t)max_new * group + kChunkRows - 1) / kChunkRows);
        const int64_t places = tokens * group / kChunkRows + n_b;  // of packed tokens' tiles (dc_packed)
        int64_t all = n_b * c.tiles;
        if (tokens && places < all) all = places;
        // Short parts where the tiles alone leave most CUs idle: three steps at least, four of the smaller ones of 256 columns, and up to seven as
        // long as CUs are left without a block (38 tokens of 12 units of 128 columns over 700 rows 20.2 us in parts of seven steps, 15.4 of
        // three; over 8195 rows 29.0 and 33.6, as few as CUs 27), and none of ten steps or fewer (a prompt of 517 of one head in groups of 8: 17.6
        // and 19.3).  Where they do not, a part has to save more than the join takes (a prompt of 517 tokens of 8 heads, 136 tiles: 19.6 us, in two
        // parts 26.7; of 2048, 512 tiles: 63 us, the longer half of them in two parts of 16 steps 84).
        const int64_t steps = (rows + dc_chunk_step(hd) - 1) / dc_chunk_step(hd);
        c.least = all * n_h <= 128 ? 7 : 24, c.fewest = all * n_h > 128 ? 24 : hd == 256 ? 4 : 3;
        // Of more tiles than that, where tokens have rows before them and there are few rounds, the last round's are cut if they are at most half of
        // what runs at once, or two thirds where they are all (dc_deal; 2048 tokens of 8 heads x 128 behind some 30000 rows, 512 tiles: 1036 us; 2100
        // 1697 and 1081, 2600 1688 and 1340, 1100 873 and 658).  At 64 columns, four blocks to a CU, the others of a CU gain more by one that ends.
        const bool few = all * n_h <= (n_b == 1 ? c.at_once / 2 : 2 * c.at_once);
        const int64_t left = all * n_h % c.at_once, cut = all * n_h < c.at_once ? c.at_once * 2 / 3 : hd == 64 ? c.at_once * 3 / 10 : c.at_once / 2;
        const bool tail = all * n_h <= 4 * c.at_once && n_b <= 64 && rows >= 2 * (int64_t)max_new && left > 0 && left <= cut;
        c.join = (few || tail) && 2 * steps >= 3 * c.least;
        c.deal = c.join;
        if (c.tiles > all) c.tiles = (int)all;  // (one sequence of fewer packed tokens than max_new)
        if (!c.join && tokens && n_b > 1) all = places;
        // (items: see dc_deal; and no tile has more parts than its steps allow.  A thousand blocks that find none cost 1-2 us in each kernel)
        const int64_t parts = c.join ? 2 * c.at_once / n_h + 1 : 0, most = all * (c.join ? steps / c.fewest + 1 : 1);
        c.blocks = n_h * (all + parts < most ? all + parts : most), c.places = n_h * ((all < parts ? all : parts) + parts);
        if (c.places > c.blocks) c.places = c.blocks;
        c.sharers = c.blocks <= 128 ? 4 : c.blocks <= 512 ? 2 : 1;  // (38 tokens of 12 units over 1575 rows of 256 columns, 96 blocks: 36 us, four times as many to join 31)
        return c;
    }
    c.tiles = 1, c.tile_rows = max_new * group, c.at_once = rows_at_once(hd), c.least = c.fewest = kWaves;
    const int64_t step = 16 * row_tiles(hd), steps = (rows + step - 1) / step;
    c.deal = c.join = steps * step * hd > kAlone && n_units <= 2 * c.at_once;
    c.waves = steps * step * hd > kAlone || steps <= kWaves ? kWaves : kMostWaves;
    const int64_t items = n_b + c.at_once / n_h + 1, most = n_b * (steps / c.least + 1);
    c.blocks = c.places = c.deal ? n_h * (items < most ? items : most) : n_units;
    return c;
}
size_t acc_bytes(int64_t slots, int rows, int hd) { return dc_align_up((size_t)slots * rows * hd * 4, 256); }
size_t ml_bytes(int64_t slots, int rows) { return dc_align_up((size_t)slots * rows * 8, 256); }

template <int HD>
void launch_rows(const DcPagedAttn &a, const Cut &c, hipStream_t st) {
    constexpr int TILES = row_tiles(HD);
    const size_t lds = (size_t)a.waves * (2 * kRows + a.tile_rows * HD) * sizeof(float);
    const dim3 grid = c.deal ? dim3((unsigned)c.blocks) : dim3((unsigned)a.n_b, (unsigned)a.n_h);
    hipLaunchKernelGGL((paged_rows_kernel<HD, TILES>), grid, dim3(a.waves * 64), lds, st, a);
    if (c.join) hipLaunchKernelGGL((paged_join_kernel<HD, 16 * TILES>), dim3((unsigned)(a.n_b * a.n_h), (unsigned)a.tile_rows), dim3(kThreads), 0, st, a);
}

}  // namespace

extern "C" size_t dc_paged_attn_workspace_bytes(int n_b, int n_h, int group, int hd, int n_rows, int max_new, int n_tokens) {
    if (n_b <= 0 || n_h <= 0 || (int64_t)n_b * n_h >= (1 << 24) || group <= 0 || group > 16 || hd < 64 || n_rows < 0 || max_new <= 0 || n_tokens < 0) return 0;
    // (so many sequences that nothing is dealt out: enough for fewer, where it is)
    const int64_t most = 2 * rows_at_once(hd) / n_h;
    const bool few = (int64_t)max_new * group <= kRows;
    const Cut c = cut_of(few && most > 0 && n_b > most ? most : n_b, n_h, group, hd, n_rows, max_new, n_tokens);
    return c.join ? acc_bytes(c.places, c.tile_rows, hd) + ml_bytes(c.places, c.tile_rows) : 0;
}

extern "C" int dc_paged_attn_bf16(const dc_paged_attn_args *x, void *stream) {
    const char *who = "dc_paged_attn_bf16";
    DC_REQUIRE(x, "%s: null pointer", who);
    const dc_paged_tokens &t = x->tokens;
    DC_REQUIRE(t.n_b >= 0 && t.max_new >= 0 && t.n_tokens >= 0, "%s: bad sizes", who);
    if (t.n_b == 0 || t.max_new == 0) return DC_OK;
    if (const int rc = dc_check_paged(who, x->store, t, x->n_h, x->hd, false)) return rc;
    DC_REQUIRE(x->q && x->out, "%s: null pointer", who);
    DC_REQUIRE(dc_aligned16(x->q) && dc_aligned16(x->out) && x->q_batch_stride % 8 == 0 && x->q_token_stride % 8 == 0 && x->q_head_stride % 8 == 0,
               "%s: pointers must be 16-byte aligned, strides multiples of 8 elements", who);
    DC_REQUIRE(x->group >= 1 && x->group <= 16, "%s: group %d not in [1,16]", who, x->group);
    DC_REQUIRE(x->n_rows >= 1 && x->n_rows <= (int64_t)t.table_pages * x->store.page, "%s: %d rows outside the table", who, x->n_rows);
    DC_REQUIRE(x->n_sink >= 0 && x->window >= 0, "%s: negative n_sink or window", who);
    const float scale = x->scale * 1.44269504088896341f;  // in powers of two
    DC_REQUIRE(x->scale > 0.f && scale < INFINITY, "%s: scale must be positive and at most 2.35e38", who);
    DC_REQUIRE((int64_t)t.max_new * x->group < (1ll << 30) && (int64_t)t.n_tokens * x->group < (1ll << 31), "%s: too many tokens", who);
    // rows that a window's tokens, or those of a tile, can need at most, and a step more at its two ends
    const int64_t of_tile = (int64_t)t.max_new * x->group > kRows ? kChunkRows / x->group + 2 : t.max_new;
    const int64_t in_window = (int64_t)x->n_sink + x->window + (of_tile < t.max_new ? of_tile : t.max_new) + 256;
    const int64_t rows = x->window && in_window < x->n_rows ? in_window : x->n_rows;
    const Cut c = cut_of(t.n_b, x->n_h, x->group, x->hd, rows, t.max_new, t.cu ? t.n_tokens : 0);
    DC_REQUIRE(dc_grid_fits(c.chunk || c.deal ? c.blocks : t.n_b, c.waves * 64), "%s: grid too large", who);
    DcPagedAttn a;
    a.ws_acc = a.ws_ml = nullptr;
    if (c.join) {
        const size_t acc = acc_bytes(c.places, c.tile_rows, x->hd), need = acc + ml_bytes(c.places, c.tile_rows);
        DC_REQUIRE(x->workspace && ((uintptr_t)x->workspace & 255u) == 0, "%s: workspace must be non-null and 256-byte aligned", who);
        if (x->workspace_bytes < need) {
            dc_set_error("%s: workspace %zu bytes < %zu needed", who, x->workspace_bytes, need);
            return DC_ENOMEM;
        }
        a.ws_acc = (float *)x->workspace, a.ws_ml = (float *)((char *)x->workspace + acc);
    }
    a.q = (const uint16_t *)x->q, a.out = (uint16_t *)x->out, a.lse = x->lse;
    a.p = dc_pages_of(x->store, t), a.t = dc_new_of(t);
    a.qs = {x->q_batch_stride, x->q_token_stride, x->q_head_stride};
    a.n_h = x->n_h, a.group = x->group, a.n_rows = x->n_rows, a.n_sink = x->n_sink, a.window = x->window;
    a.n_b = t.n_b, a.waves = c.waves, a.tiles = c.tiles, a.tile_rows = c.tile_rows;
    a.at_once = c.deal ? c.at_once : 0, a.round = c.at_once > x->n_h ? c.at_once / x->n_h : 1, a.least = c.least, a.fewest = c.fewest, a.places = (int)(c.places / x->n_h), a.of_all = 1.0001f / (float)c.at_once;
    a.scale = scale;
    hipStream_t st = (hipStream_t)stream;
    if (c.chunk) return dc_paged_chunk_launch(a, x->hd, (unsigned)c.blocks, c.join ? c.sharers : 0, st);
    if (x->hd == 64) launch_rows<64>(a, c, st);
    else if (x->hd == 128) launch_rows<128>(a, c, st);
    else launch_rows<256>(a, c, st);
    DC_CHECK_LAUNCH(who);
    return DC_OK;
}
