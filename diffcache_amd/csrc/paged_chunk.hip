// Attention of many new tokens over keys and values in pages, each over the rows up to its own.
//
// A unit (one sequence, one KV head) has count * group (token, head) pairs, its heads side by side so that they share K and V.  A block
// of four waves takes 128 of them and goes over the rows that they attend to in steps of KT, staged through LDS; a wave has 32 pairs.
//
//   S^T = K Q^T   v_mfma_f32_32x32x16_bf16, M = 32 rows, N = the wave's 32 pairs.  A lane then has one pair's logits of half the rows, so that
//                 maximum and sum stay inside it but for one exchange between the wave's halves where the maximum moves.
//   O^T = V^T P^T M = 32 of the hd columns, N = the pairs, K = 16 rows: P^T stands in the lanes as the operand wants it, and V^T comes out of
//                 LDS by the transposing reads, rows in the order that P^T has them.  Rescaling O is a factor of the lane's own.
//
// P is rounded to bf16 (2^-8 of a weight at most; the sum is that of the weights before): a second product for the rest would be half as
// much matrix work again, for an error no larger than that of the output's own rounding (against 64 bits 2.1e-3 of the result with both,
// 1.7e-3 is the output's alone).  Softmax in powers of two, fp32; the maximum moves where a
// logit passes it by more than 8.
//
// What bounds it: the power that the products take, and the matrix and the vector unit side by side only in part.  2048 tokens of 32 heads x
// 128 behind 30553 rows: 1017-1066 us = 990-1040 TFLOP/s, by the card (a large library product: 1160); on Q, K and V of one value, where the
// clock stays up, 881 us.  A prompt of 8195 tokens 551-581 us = 950-1000 TFLOP/s; 1024 tokens at 256 columns 1050-1095 us = 980-1030; at 64
// columns, where a row has half the products for the same exponentials, 325-330 us for 224 GFLOP = 690.  A prompt of 517 tokens (nine steps)
// 18 us, of 1024 29: there a step is a chain that nothing else fills, 1.26 us where a CU has one block.
// Kept: K and V straight to LDS instead of through registers (1163 -> 1060), page ids a step ahead and masks without branches (1348 -> 1163),
// at 256 columns two blocks to a CU (1781 -> 1068); a wave that is at S ahead of the one it shares its SIMD with, so that the two do not stand
// at the same unit at once (1125 -> 1073 on one card; at 64 columns to the step's end, 337 -> 328, which is slower at 128, 1017 -> 1035), and K
// read from LDS three products ahead at 128 columns (1026 -> 1017 on another); the loads' addresses made by lanes, and steps without masks known
// as such by the block (517 tokens 19.0 -> 17.7).
// Tried and dropped: S of a step beside the exponentials of the one before (1105 -> 1145, and slower on equal values too), the weights'
// products ahead as well (1073 -> 1149), the next step's loads between this one's products or V's behind them (one block alone 1.26 -> 1.34 a
// step; 1049 -> 1037 and 1084), blocks started half a step apart (the same), three blocks of 32-row steps to a CU at 128 columns (1293 for
// 1116), a zero operand kept for the first product (1222 for 1172).
#include "dc_paged.h"

namespace {

constexpr int kThreads = 256, kRowsOfWave = 32;
constexpr int kLoaded = 0x0f70;  // s_waitcnt vmcnt(0)
constexpr int kMatrix = 0x008, kLdsRead = 0x100;  // (kinds of instruction, to the scheduler)
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) uint32_t lds_u32;
typedef __attribute__((address_space(1))) uint32_t glb_u32;

template <int HD, int KT>
struct Tile {
    static constexpr int ROW = HD * 2, CHUNKS = HD / 8;          // bytes and 16-byte chunks of a row
    static constexpr int PER = 64 / CHUNKS;                      // rows of a wave's load
    static constexpr int LOADS = KT / PER / 4;                   // loads of a wave for K, and for V
    static constexpr int BYTES = KT * ROW;
    // Where chunk c of a row lies in LDS: chunk c ^ k_turn(row) for K, so that 16 rows' same chunk are 16 different banks' groups; whole groups
    // of four chunks (what a transposing read takes of a row) changed about for V.
    static __device__ __forceinline__ int k_turn(int row) { return HD == 64 ? (row >> 1) & 7 : row & 15; }
    static __device__ __forceinline__ int v_turn(int row) { return HD == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }
};

template <int HD, int KT>
__global__ __launch_bounds__(kThreads, 2) void paged_chunk_kernel(DcPagedAttn a) {
    using T = Tile<HD, KT>;
    constexpr int KS = HD / 16, DT = HD / 32, ST = KT / 32, TILES = KT / 16;  // products of a tile's S; tiles of O, of S, and of what a page holds whole
    // (four arrays, not one of four: the reads of one are then known not to wait for the loads into another)
    __shared__ __attribute__((aligned(1024))) uint8_t s_k0[T::BYTES], s_v0[T::BYTES], s_k1[T::BYTES], s_v1[T::BYTES];
    __shared__ __attribute__((aligned(16))) uint32_t s_odd[2][4];  // [buffer][wave]: whether the wave left out numbers of V that are not finite
    // (at 256 columns three of a lane's sixteen pieces of Q stand in LDS: with them its registers would be 16 too many for two blocks to a CU)
    constexpr int QL = HD == 256 ? 3 : 0;
    __shared__ dc_u32x4 s_q[QL ? QL : 1][QL ? kThreads : 1];
    // heads first, so that a sequence's blocks of one head are on one XCD where their number divides by eight; late tokens first
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int h = (int)(blockIdx.x % (unsigned)a.n_h), x_ = (int)(blockIdx.x / (unsigned)a.n_h), G = a.group;
    DcItem d = {x_ % a.n_b, a.tiles - 1 - x_ / a.n_b, 0, 1, 0};
    if (a.at_once) d = dc_deal<KT, true>(a, x_, lane);
    else if (a.t.cu && a.n_b > 1) d = dc_packed(a, x_, lane);
    if (d.part >= d.parts) return;  // (its tile has fewer parts than the sequence's last one)
    const int b = d.b;
    const DcSpan span = dc_span(a.t, b);
    const int pairs = span.count * G, pair0 = d.tile * kChunkRows;
    if (pair0 >= pairs) return;
    const int t_lo = pair0 / G, t_hi = (pair0 + kChunkRows < pairs ? pair0 + kChunkRows : pairs) - 1;
    const DcSteps steps = dc_steps<KT>(a, span.start + t_lo, span.start + t_hi / G);
    const int per = (steps.steps + d.parts - 1) / d.parts;
    const int begin = d.part * per, end = begin + per < steps.steps ? begin + per : steps.steps;

    // the wave's pairs: lane's own, and the least and the largest row
    const int first = pair0 + wave * kRowsOfWave;
    const bool live = first < pairs;
    const int own = first + (lane & 31), pair = own < pairs ? own : pairs - 1, token = pair / G;
    const int p = span.start + token;
    const int p_lo = span.start + (live ? first : pairs - 1) / G;
    const int p_hi = span.start + (first + kRowsOfWave - 1 < pairs ? first + kRowsOfWave - 1 : pairs - 1) / G;
    dc_u32x4 bq[KS - QL];
    {
        const uint16_t *src = a.q + dc_token_at(a.t, a.qs, span, b, token) + (int64_t)(h * G + pair % G) * a.qs.h + 8 * half;
#pragma unroll
        for (int s = 0; s < KS - QL; ++s) bq[s] = *reinterpret_cast<const dc_u32x4 *>(src + 16 * s);
#pragma unroll
        for (int s = KS - QL; s < KS; ++s) s_q[s - KS + QL][tid] = *reinterpret_cast<const dc_u32x4 *>(src + 16 * s);
    }
    dc_f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = begin < end ? kNoLogit : -INFINITY, l = 0.f;

    // staging: a wave's load n has rows (wave + 4 n) PER .., of one tile of 16 and so of one page, and goes straight to LDS: lane i's 16 bytes to
    // place i, so that which chunk it asks for is what turns the rows.  The step's page ids are one load of as many lanes, made a
    // step before they are needed.
    const uint16_t *kh = a.p.k + h * a.p.kh, *vh = a.p.v + h * a.p.vh;
    const int32_t *table = a.p.table + (int64_t)b * a.p.table_stride;
    const int last_page = (a.n_rows - 1) >> a.p.shift, mask = (1 << a.p.shift) - 1;
    const int in_row = lane / T::CHUNKS, chunk = lane % T::CHUNKS;
    auto ids_of = [&](int s) __attribute__((always_inline)) {
        const int page = (steps.row(s, KT) + 16 * (lane % TILES)) >> a.p.shift;
        return table[page < last_page ? page : last_page];
    };
    const uint32_t in_tile = (uint32_t)(wave * T::PER % 16 + in_row);  // of a load's rows, for those n that begin a tile
    auto fetch = [&](uint8_t *k_lds, uint8_t *v_lds, int s, int ids) __attribute__((always_inline)) {  // returns a bit for each tile of 16 rows that has a page
        // (lane t makes tile t's addresses, page 0's in the place of one that there is not: some 30 vector instructions for 150 of the scalar unit)
        const bool is = (unsigned)ids < (unsigned)a.p.n_pages;
        const int64_t id = is ? ids : 0;
        const int first = ((steps.row(s, KT) + 16 * (lane % TILES)) & mask) * HD;
        const uint64_t kb = (uint64_t)(kh + (id * a.p.kp + first)), vb = (uint64_t)(vh + (id * a.p.vp + first));
        auto of_tile = [](uint64_t x, int t) __attribute__((always_inline)) {
            return (uint64_t)dc_of_lane((uint32_t)(x >> 32), t) << 32 | dc_of_lane((uint32_t)x, t);
        };
#pragma unroll
        for (int n = 0; n < T::LOADS; ++n) {
            const int row = (wave + 4 * n) * T::PER, tile = T::PER == 8 ? 2 * n + (wave >> 1) : 4 * n * T::PER / 16;
            const uint32_t mine = in_tile + 4 * n * T::PER % 16;
            const uint32_t k_at = mine * T::ROW + ((chunk ^ T::k_turn(mine)) << 4), v_at = mine * T::ROW + ((chunk ^ T::v_turn(mine)) << 4);
            __builtin_amdgcn_global_load_lds((const glb_u32 *)(of_tile(kb, tile) + k_at), (lds_u32 *)(k_lds + row * T::ROW), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((const glb_u32 *)(of_tile(vb, tile) + v_at), (lds_u32 *)(v_lds + row * T::ROW), 16, 0, 0);
        }
        return (int)__ballot(is) & ((1 << TILES) - 1);
    };
    // what fetch brought is there, for the wave that asked for it; returns whether all of the rows have pages and all of the block's pairs attend to
    // them (as every wave finds: then no one has to look for numbers that are not finite, nor at masks)
    auto stage = [&](uint8_t *v_lds, int buf, int s, int have) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(kLoaded);
        const bool plain = have == (1 << TILES) - 1 && dc_whole(a, span.start + t_lo, span.start + t_hi / G, steps.row(s, KT), KT);
        if (!plain) {
            uint32_t odd = 0;
            DcUnbounded u;
            dc_u32x4 w[T::LOADS];
#pragma unroll
            for (int n = 0; n < T::LOADS; ++n) {
                w[n] = *reinterpret_cast<const dc_u32x4 *>(v_lds + (wave + 4 * n) * T::PER * T::ROW + lane * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) u.look(w[n][i]);
            }
            if (u.any()) {
                odd = 1;
#pragma unroll
                for (int n = 0; n < T::LOADS; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[n][i] = dc_finite(w[n][i]);
                    *reinterpret_cast<dc_u32x4 *>(v_lds + (wave + 4 * n) * T::PER * T::ROW + lane * 16) = w[n];
                }
            }
            if (lane == 0) s_odd[buf][wave] = odd;
        }
        return plain;
    };

    auto any_odd = [&](int buf) __attribute__((always_inline)) {
        const uint4 odd = *reinterpret_cast<const uint4 *>(s_odd[buf]);
        return __builtin_amdgcn_readfirstlane(odd.x | odd.y | odd.z | odd.w) != 0;
    };
    bool huge = true;  // (as kNoLogit is)
    int have = 0, next = 0, ids = 0;
    bool plain = true;  // a step whose rows are there and attended to by all of the block's pairs
    if (begin < end) {
        have = fetch(s_k0, s_v0, begin, ids_of(begin));
        if (begin + 1 < end) ids = ids_of(begin + 1);
        plain = stage(s_v0, 0, begin, have);
    }
    __builtin_amdgcn_s_waitcnt(kLoaded);  // (Q too, on every way here: the loop would wait for it, and for all loads, in every step)
    __syncthreads();
    auto step = [&](int s, int buf, const uint8_t *k_now, const uint8_t *v_now, uint8_t *k_next, uint8_t *v_next) __attribute__((always_inline)) {
        const int row0 = steps.row(s, KT);
        if (s + 1 < end) {
            next = fetch(k_next, v_next, s + 1, ids);
            if (s + 2 < end) ids = ids_of(s + 2);
        }
        // rows that the wave has no use for: behind all its pairs, or between the sinks and all windows
        const bool use = live && (plain || (row0 <= p_hi && (a.window == 0 || row0 + KT - 1 > p_lo - a.window || row0 < a.n_sink)));
        if (use) {
            __builtin_amdgcn_s_setprio(1);  // (among waves of the SIMD)
            // S^T: x[t][i] is row 32 t + 8 (i / 4) + 4 half + i % 4
            dc_f32x16 x[ST];
            const uint8_t *ks = k_now + (lane & 31) * T::ROW;
            const int turn = (half ^ T::k_turn(lane & 31)) << 4;
#pragma unroll
            for (int t = 0; t < ST; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[t][i] = 0.f;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const dc_u32x4 qw = j < KS - QL ? bq[j < KS - QL ? j : 0] : s_q[j < KS - QL ? 0 : j - KS + QL][QL ? tid : 0];
#pragma unroll
                for (int t = 0; t < ST; ++t) {
                    const dc_u32x4 w = *reinterpret_cast<const dc_u32x4 *>(ks + 32 * t * T::ROW + (turn ^ (j << 5)));
                    x[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(dc_bf16x8, w), __builtin_bit_cast(dc_bf16x8, qw), x[t], 0, 0, 0);
                }
            }
            if constexpr (HD == 128) {  // K's reads three products' ahead
                __builtin_amdgcn_sched_group_barrier(kLdsRead, 6, 0);
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    __builtin_amdgcn_sched_group_barrier(kMatrix, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(kLdsRead, 2, 0);
                }
            }
            if constexpr (HD > 64) __builtin_amdgcn_s_setprio(0);
            if (!plain && (have != (1 << TILES) - 1 || !dc_whole(a, p_lo, p_hi, row0, KT))) {
                const DcReach reach = dc_reach(a, p);
#pragma unroll
                for (int t = 0; t < ST; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!((have >> (2 * t + i / 8)) & 1) | !reach.has(row0 + 32 * t + 8 * (i / 4) + 4 * half + i % 4)) x[t][i] = -INFINITY;
            }
            float most = -INFINITY;
#pragma unroll
            for (int t = 0; t < ST; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) most = fmaxf(most, x[t][i]);
            most *= a.scale;
            if (__builtin_expect(__any(most > m + 8.f), 0)) {
                const float to = fmaxf(m, dc_over32(most, [](float u, float v) { return fmaxf(u, v); }));
                const float f = m > kNoLogit ? __builtin_amdgcn_exp2f(m - to) : 1.f;  // (nothing was summed, or what is no number)
                l *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= f;
                m = to;
                huge = __any(fabsf(m) > 0x1p24f);
            }
            // The product below is exact and m is not: of logits so large that would be more than a weight can grow.
            if (__builtin_expect(huge, 0)) {
#pragma unroll
                for (int t = 0; t < ST; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[t][i] = dc_less(x[t][i] * a.scale, m);
            }
            const float by = huge ? 1.f : a.scale, less = huge ? 0.f : -m;
#pragma unroll
            for (int t = 0; t < ST; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    x[t][i] = __builtin_amdgcn_exp2f(fmaf(x[t][i], by, less));
                    l += x[t][i];
                }
            // O^T: rows 16 j + {0 .. 3, 8 .. 11} + 4 half at a time
            const int in = (lane >> 2) & 3;  // a transposing read's row of four
            const uint8_t *vs = v_now + (4 * half + in) * T::ROW + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
            const int vturn = T::v_turn(4 * half + in) << 4;
#pragma unroll
            for (int j = 0; j < KT / 16; ++j) {
                dc_u32x4 pw;
#pragma unroll
                for (int i = 0; i < 4; ++i) pw[i] = dc_pack_bf16(x[j / 2][8 * (j % 2) + 2 * i], x[j / 2][8 * (j % 2) + 2 * i + 1]);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const uint8_t *at = vs + 16 * j * T::ROW + (vturn ^ (d << 6));
                    const dc_u32x2 lo = __builtin_bit_cast(dc_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(s16x4 *)(at)));
                    const dc_u32x2 hi = __builtin_bit_cast(dc_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(s16x4 *)(at + 8 * T::ROW)));
                    const dc_u32x4 w = {lo.x, lo.y, hi.x, hi.y};
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(dc_bf16x8, w), __builtin_bit_cast(dc_bf16x8, pw), o[d], 0, 0, 0);
                }
            }
            if (!plain && any_odd(buf)) {
                for (int r = 0; r < KT; ++r) {
                    const int page = (row0 + r) >> a.p.shift, id = dc_page_id(a.p, table, page < last_page ? page : last_page);
                    if (id < 0) continue;
                    const uint16_t *src = vh + id * a.p.vp + (int64_t)((row0 + r) & mask) * HD + 4 * half;
                    const bool in = dc_reach(a, p).has(row0 + r);
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const uint2 w = *reinterpret_cast<const uint2 *>(src + 32 * d + 2 * i);
                            o[d][i] += in ? dc_only_unbounded(dc_bf16_lo(w.x)) : 0.f, o[d][i + 1] += in ? dc_only_unbounded(dc_bf16_hi(w.x)) : 0.f;
                            o[d][i + 2] += in ? dc_only_unbounded(dc_bf16_lo(w.y)) : 0.f, o[d][i + 3] += in ? dc_only_unbounded(dc_bf16_hi(w.y)) : 0.f;
                        }
                }
            }
        }
        if constexpr (HD == 64) __builtin_amdgcn_s_setprio(0);
        if (s + 1 < end) plain = stage(v_next, buf ^ 1, s + 1, next);
        have = next;
        __syncthreads();
    };
    for (int s = begin; s < end; s += 2) {
        step(s, 0, s_k0, s_v0, s_k1, s_v1);
        if (s + 1 < end) step(s + 1, 1, s_k1, s_v1, s_k0, s_v0);
    }

    l = dc_over32(l, [](float u, float v) { return u + v; });
    // (the lane's number and its pair again, from nothing: no register has to keep them through the loop)
    const int lane_ = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), half_ = lane_ >> 5, mine = first + (lane_ & 31);
    if (mine >= pairs) return;
    const int64_t dst = (int64_t)(span.first + mine / G) * a.n_h * G + h * G + mine % G;
    if (d.parts > 1) {
        const int64_t slot = (d.slot + (int64_t)d.part * a.n_h + h) * kChunkRows + wave * kRowsOfWave + (lane_ & 31);
        float *acc = a.ws_acc + slot * HD + 4 * half_;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4 *>(acc + 32 * d + 2 * i) = make_float4(o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
        if (half_ == 0) reinterpret_cast<float2 *>(a.ws_ml)[slot] = make_float2(m, l);
        return;
    }
    const float inv = l == 0.f ? 1.f : l;
    uint16_t *out = a.out + dst * HD + 4 * half_;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<uint2 *>(out + 32 * d + 2 * i) =
                make_uint2(dc_pack_bf16(o[d][i] / inv, o[d][i + 1] / inv), dc_pack_bf16(o[d][i + 2] / inv, o[d][i + 3] / inv));
    if (a.lse && half_ == 0) a.lse[dst] = dc_log_sum(m, l);
}

// The parts of a tile joined: as many blocks as it has parts, times the grid's y, share its rows, every so many-th of them each, HD / 4 threads to a row, four
// parts asked for at once.
template <int HD, int KT>
__global__ __launch_bounds__(kThreads) void paged_chunk_join_kernel(DcPagedAttn a) {
    constexpr int kLanes = HD / 4, kPer = kThreads / kLanes, kBatch = 4;
    const int tid = threadIdx.x, c = tid % kLanes, h = (int)(blockIdx.x % (unsigned)a.n_h), G = a.group;
    const DcItem d = dc_deal<KT, true>(a, (int)(blockIdx.x / (unsigned)a.n_h), tid & 63);
    if (d.parts < 2 || d.part >= d.parts) return;
    const DcSpan span = dc_span(a.t, d.b);
    const int n = d.parts, pair0 = d.tile * kChunkRows, left = span.count * G - pair0, rows = left < kChunkRows ? left : kChunkRows;
    const int sharers = n * (int)gridDim.y;
    const int64_t step = (int64_t)a.n_h * kChunkRows;
    for (int r = d.part + n * (int)blockIdx.y + tid / kLanes * sharers; r < rows; r += kPer * sharers) {
        const int64_t slot0 = (d.slot + h) * kChunkRows + r;
        const float2 *ml = reinterpret_cast<const float2 *>(a.ws_ml) + slot0;
        const float4 *pa = reinterpret_cast<const float4 *>(a.ws_acc) + slot0 * kLanes + c;
        float top = -INFINITY, total = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < n; s0 += kBatch) {
            float2 o[kBatch];
            float4 v[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {  // (the last part again where there are no more)
                const int64_t s = (int64_t)(s0 + i < n ? s0 + i : n - 1) * step;
                o[i] = ml[s], v[i] = pa[s * kLanes];
            }
            float to = top;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) to = fmaxf(to, o[i].x);
            const float f = dc_weight(top, to);
            acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
            total = dc_share(top, total, to);
            top = to;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                // (a part without rows has nothing to add)
                const bool in = s0 + i < n && o[i].x > -INFINITY;
                const float g = in ? dc_weight(o[i].x, top) : 0.f;
                total += in ? dc_share(o[i].x, o[i].y, top) : 0.f;
                acc.x = fmaf(g, in ? v[i].x : 0.f, acc.x), acc.y = fmaf(g, in ? v[i].y : 0.f, acc.y);
                acc.z = fmaf(g, in ? v[i].z : 0.f, acc.z), acc.w = fmaf(g, in ? v[i].w : 0.f, acc.w);
            }
        }
        const int pair = pair0 + r;
        const int64_t dst = (int64_t)(span.first + pair / G) * a.n_h * G + h * G + pair % G;
        const float by = total == 0.f ? 1.f : total;
        *reinterpret_cast<uint2 *>(a.out + dst * HD + 4 * c) = make_uint2(dc_pack_bf16(acc.x / by, acc.y / by), dc_pack_bf16(acc.z / by, acc.w / by));
        if (a.lse && c == 0) a.lse[dst] = dc_log_sum(top, total);
    }
}

template <int HD>
void launch(const DcPagedAttn &a, unsigned blocks, unsigned join, hipStream_t st) {
    constexpr int KT = dc_chunk_step(HD);
    hipLaunchKernelGGL((paged_chunk_kernel<HD, KT>), dim3(blocks), dim3(kThreads), 0, st, a);
    if (join) hipLaunchKernelGGL((paged_chunk_join_kernel<HD, KT>), dim3(blocks, join), dim3(kThreads), 0, st, a);
}

}  // namespace

int dc_paged_chunk_launch(const DcPagedAttn &a, int hd, unsigned blocks, unsigned join, hipStream_t st) {
    if (hd == 64) launch<64>(a, blocks, join, st);
    else if (hd == 128) launch<128>(a, blocks, join, st);
    else launch<256>(a, blocks, join, st);
    DC_CHECK_LAUNCH("dc_paged_attn_bf16");
    return DC_OK;
}
