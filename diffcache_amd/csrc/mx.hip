// A cache held in blocks of 32 numbers: 4-bit (E2M1) or 8-bit (E4M3) codes and one power of two for a block.
// Writing it (prompts, tokens), reading rows back, and one token's attention over what it holds.
//
// A block of numbers x_0 .. x_31 is held as round(x_i / 2^e), rounded to the nearest number of the format, ties to the
// even code, and the byte e + 127.  e is the least exponent at which the largest |x_i| does not round past the last
// number of the format (6 in 4 bits, 448 in 8): |x_i - held| <= 2^e in 4 bits, 16 2^e in 8, wherever e is not at its
// limits.  The limits keep every number that is held a normal bf16 number or zero, so reading back into bf16 is exact.  A
// block with an infinity or a NaN in it is held as NaN (byte 255).
//
// Columns 2 i and 2 i + 1 of a 4-bit row are the low and the high half of byte i.
#include "dc_common.h"
#include <math.h>
#include <type_traits>
#include <utility>

namespace {

typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf16x8 __attribute__((ext_vector_type(8)));
typedef short mx_s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short mx_u16x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mx_u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMostWaves = 8;  // of a block of the attention

// A store as the kernels see it; strides in bytes.
struct View {
    uint8_t *codes, *scale;
    int64_t cb, ch, sb, sh;
};
inline View view_of(const dc_mx_store &s) {
    return {(uint8_t *)s.codes, (uint8_t *)s.scale, s.code_batch_stride, s.code_head_stride, s.scale_batch_stride, s.scale_head_stride};
}

// ---- the format -----------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t mx_bits(mx_bf16x2 v) { return __builtin_bit_cast(uint32_t, v); }

// 2^(byte - 127) as the conversions want it: they read the exponent of a float.  Byte 255 gives an infinity, at which
// they return NaN, and byte 0 zero, at which the codes 0 of a row that is not there give 0.
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// numbers 2 PAIR and 2 PAIR + 1 of the words w, as two bf16 numbers
template <int BITS, int PAIR>
__device__ __forceinline__ uint32_t mx_pair(const uint32_t *w, float scale) {
    if constexpr (BITS == 4)
        return mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[PAIR / 4], scale, PAIR % 4));
    else
        return mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[PAIR / 2], scale, PAIR % 2 != 0));
}

template <int BITS>
struct Coded {
    uint32_t w[BITS / 4];  // the codes of 8 numbers
    uint32_t scale;        // the block's byte
};

// Eight numbers of a block whose others are with the three lanes of the same quad.  On the bits of bf16 numbers, whose
// magnitudes are ordered as whole numbers.
template <int BITS>
__device__ __forceinline__ Coded<BITS> mx_quantise(const uint4 &x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    mx_u16x2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        top = __builtin_elementwise_max(top, __builtin_bit_cast(mx_u16x2, w[i] & 0x7fff7fffu));
    uint32_t most = top.x > top.y ? top.x : top.y;
    auto other = [](uint32_t v, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, true);
    };
    const uint32_t a = other(most, std::integral_constant<int, 0xB1>{});  // quad_perm [1,0,3,2]
    most = most > a ? most : a;
    const uint32_t b = other(most, std::integral_constant<int, 0x4E>{});  // quad_perm [2,3,0,1]
    most = most > b ? most : b;
    // the exponent, one more where the fraction would round past the last code: from 7 / 4 on in 4 bits (that tie goes
    // to the even code, beyond the last), above 29 / 16 in 8 (that one goes down)
    constexpr int kBump = BITS == 4 ? 0x20 : 0x17, kTop = BITS == 4 ? 2 : 8;
    constexpr int kLo = BITS == 4 ? 2 : 10, kHi = BITS == 4 ? 252 : 246;
    int e = (int)((most + kBump) >> 7) - kTop;
    e = e < kLo ? kLo : (e > kHi ? kHi : e);
    const bool fine = most < 0x7f80u;
    const float s = mx_scale((uint32_t)e);
    Coded<BITS> c;
    c.scale = fine ? (uint32_t)e : 255u;
    if constexpr (BITS == 4) {  // (beyond the last code the conversion gives the last one)
        uint32_t r = 0;
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_bf16x2, w[0]), s, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_bf16x2, w[1]), s, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_bf16x2, w[2]), s, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(mx_bf16x2, w[3]), s, 3);
        c.w[0] = fine ? r : 0u;
    } else {  // (here it gives NaN: numbers beyond 448 2^119, which only the largest scale leaves, are brought back first)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx_s16x2 r = {0, 0};
            auto held = [](uint32_t v) {
                const mx_u16x2 mag = __builtin_elementwise_min(__builtin_bit_cast(mx_u16x2, v & 0x7fff7fffu), mx_u16x2{0x7f60, 0x7f60});
                return __builtin_bit_cast(mx_bf16x2, __builtin_bit_cast(uint32_t, mag) | (v & 0x80008000u));
            };
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, held(w[2 * i]), s, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, held(w[2 * i + 1]), s, true);
            c.w[i] = fine ? __builtin_bit_cast(uint32_t, r) : 0u;
        }
    }
    return c;
}

// piece p (8 columns) of a row; the scale by the lane with the first piece of a block
template <int BITS>
__device__ __forceinline__ void mx_store_piece(uint8_t *codes, uint8_t *scale, int p, const Coded<BITS> &c) {
    if constexpr (BITS == 4)
        *reinterpret_cast<uint32_t *>(codes + p * 4) = c.w[0];
    else
        *reinterpret_cast<uint2 *>(codes + p * 8) = make_uint2(c.w[0], c.w[1]);
    if (p % 4 == 0) scale[p / 4] = (uint8_t)c.scale;
}

// ---- writing --------------------------------------------------------------------------------------------------------

struct IngestArgs {
    View k, v;
    const uint16_t *src_k, *src_v;
    int64_t ksb, kss, ksh, vsb, vss, vsh;  // element strides of the sources: batch, token, head
    const int32_t *lens;
    int n_h, seq, dst_pos, chunks;         // chunks: blocks of a unit
};

// Rows of a prompt.  A thread takes 8 columns (16 bytes), a quad a block of 32, so a wave's piece is 512 / hd whole rows of
// one unit: it reads segments of 2 hd bytes and writes one contiguous run.  The largest number of a block is two DPP steps
// away and the conversions do the rounding, so what bounds it is HBM: 2 + 17/32 bytes a number in 4 bits (K and V of 8 x
// 32768 tokens of 8 heads x 128: 208 us = 6.5 TB/s; of 32601 of one sequence 28 us = 6.0).  Four pieces to a thread,
// requested together: 208 us, with eight 208, with two 214, with one 290.
constexpr int kIngestBatch = 4;
template <int BITS>
__device__ __forceinline__ void mx_ingest_rows(const View &st, const uint16_t *src, int64_t ss, const IngestArgs &a, int hd,
                                               int b, int h, int chunk, int live) {
    const int ppr = hd / 8, rows_per = kThreads / ppr;  // pieces of a row, rows a block takes at once
    const int p = threadIdx.x % ppr, r0 = chunk * rows_per * kIngestBatch + threadIdx.x / ppr;
    uint4 x[kIngestBatch];
#pragma unroll
    for (int i = 0; i < kIngestBatch; ++i) {
        const int r = r0 + i * rows_per;
        x[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < live) x[i] = dc_load_stream16(src + (int64_t)r * ss + p * 8);
    }
    uint8_t *codes = st.codes + b * st.cb + h * st.ch, *scale = st.scale + b * st.sb + h * st.sh;
#pragma unroll
    for (int i = 0; i < kIngestBatch; ++i) {
        const int r = r0 + i * rows_per;
        const Coded<BITS> c = mx_quantise<BITS>(x[i]);  // (the four lanes of a quad hold one row's: all or none store)
        const int64_t at = (int64_t)a.dst_pos + r;
        if (r < live) mx_store_piece<BITS>(codes + at * (ppr * BITS), scale + at * (ppr / 4), p, c);
    }
}

template <int KB, int VB>
__global__ __launch_bounds__(kThreads) void mx_ingest_kernel(IngestArgs a, int hd) {
    const int unit = (int)(blockIdx.x / (unsigned)a.chunks), chunk = (int)(blockIdx.x % (unsigned)a.chunks);
    const int b = unit / a.n_h, h = unit % a.n_h;
    int live = a.seq;
    if (a.lens) {
        const int n = dc_step_word(a.lens + b);
        live = n < live ? n : live;
    }
    if (blockIdx.y == 0)
        mx_ingest_rows<KB>(a.k, a.src_k + b * a.ksb + h * a.ksh, a.kss, a, hd, b, h, chunk, live);
    else
        mx_ingest_rows<VB>(a.v, a.src_v + b * a.vsb + h * a.vsh, a.vss, a, hd, b, h, chunk, live);
}

// A token's row of one unit, by hd / 4 lanes: the first half of them K's pieces, the second V's.
template <int KB, int VB>
__device__ __forceinline__ void mx_write_token(const View &k, const View &v, const uint16_t *new_k, const uint16_t *new_v, int hd,
                                               int unit, int b, int h, int64_t at, int lane) {
    const int ppr = hd / 8;
    if (lane < ppr) {
        const Coded<KB> c = mx_quantise<KB>(*reinterpret_cast<const uint4 *>(new_k + (int64_t)unit * hd + lane * 8));
        mx_store_piece<KB>(k.codes + b * k.cb + h * k.ch + at * (ppr * KB), k.scale + b * k.sb + h * k.sh + at * (ppr / 4), lane, c);
    } else if (lane < 2 * ppr) {
        const int p = lane - ppr;
        const Coded<VB> c = mx_quantise<VB>(*reinterpret_cast<const uint4 *>(new_v + (int64_t)unit * hd + p * 8));
        mx_store_piece<VB>(v.codes + b * v.cb + h * v.ch + at * (ppr * VB), v.scale + b * v.sb + h * v.sh + at * (ppr / 4), p, c);
    }
}

// A token's rows alone, a wave to a unit: one round trip to the length, one to the numbers, and the launch: 2.3 us for 8 units of 128
// columns, 3.5 for 4096.
template <int KB, int VB>
__global__ __launch_bounds__(kThreads) void mx_append_kernel(View k, View v, const uint16_t *new_k, const uint16_t *new_v,
                                                             const int32_t *lens, int n_units, int n_h, int hd, int cap) {
    const int unit = (int)blockIdx.x * kWaves + (int)(threadIdx.x >> 6);
    if (unit >= n_units) return;
    const int b = unit / n_h, at = lens[b];
    if (at < 0 || at >= cap) return;
    mx_write_token<KB, VB>(k, v, new_k, new_v, hd, unit, b, unit % n_h, at, threadIdx.x & 63);
}

// ---- reading back ---------------------------------------------------------------------------------------------------

struct GatherArgs {
    View k, v;
    const uint32_t *idx;
    int64_t idx_stride, row_offset;
    uint16_t *out_k, *out_v;
    int64_t db, dh, dr;  // element strides of the outputs
    int n_h, n_idx, k_rows, v_rows, chunks;
};

// Rows back into bf16: a thread makes 8 columns of a row, 4 or 8 bytes of codes and one of scales into 16.  All rows of K and V
// of 32601 tokens of 8 heads x 128: 26 us = 6.5 TB/s, written mostly.  Rows in any order touch a line for their codes and one
// for their scales and are bound by that and by the id in front: 2117 of 131072 rows of 64 units 25 us, 1092 of 8 units 4.1 us.
// Two rows to a thread; with four 29 and 5.1 us, with one 28 and 4.2 (and all rows 37).
constexpr int kGatherBatch = 2;

template <int BITS>
__device__ __forceinline__ void mx_gather(const View &st, uint16_t *out, int n_rows, const GatherArgs &a, int hd, int unit, int chunk) {
    const int ppr = hd / 8, rows_per = kThreads / ppr, b = unit / a.n_h, h = unit % a.n_h;
    const int p = threadIdx.x % ppr, j0 = chunk * rows_per * kGatherBatch + threadIdx.x / ppr;
    const uint8_t *codes = st.codes + b * st.cb + h * st.ch, *scale = st.scale + b * st.sb + h * st.sh;
    int64_t row[kGatherBatch];
#pragma unroll
    for (int i = 0; i < kGatherBatch; ++i) {
        const int j = j0 + i * rows_per;
        row[i] = -1;
        if (j < a.n_idx) row[i] = a.row_offset + (a.idx ? (int64_t)a.idx[(int64_t)unit * a.idx_stride + j] : (int64_t)j);
        if (row[i] >= n_rows) row[i] = -1;  // (a row that the store does not have reads as zeros)
    }
    uint32_t w[kGatherBatch][BITS / 4], s[kGatherBatch];
#pragma unroll
    for (int i = 0; i < kGatherBatch; ++i) {
        s[i] = 0u;
#pragma unroll
        for (int t = 0; t < BITS / 4; ++t) w[i][t] = 0u;
        if (row[i] >= 0) {
            const uint8_t *src = codes + row[i] * (ppr * BITS) + p * BITS;
            if constexpr (BITS == 4) {
                w[i][0] = *reinterpret_cast<const uint32_t *>(src);
            } else {
                const uint2 t = *reinterpret_cast<const uint2 *>(src);
                w[i][0] = t.x, w[i][1] = t.y;
            }
            s[i] = scale[row[i] * (ppr / 4) + p / 4];
        }
    }
    uint16_t *dst = out + b * a.db + h * a.dh + p * 8;
#pragma unroll
    for (int i = 0; i < kGatherBatch; ++i) {
        const int j = j0 + i * rows_per;
        const float f = mx_scale(s[i]);
        const uint4 x = make_uint4(mx_pair<BITS, 0>(w[i], f), mx_pair<BITS, 1>(w[i], f), mx_pair<BITS, 2>(w[i], f), mx_pair<BITS, 3>(w[i], f));
        if (j < a.n_idx) dc_store_stream16(dst + (int64_t)j * a.dr, x);
    }
}

template <int KB, int VB>
__global__ __launch_bounds__(kThreads) void mx_gather_kernel(GatherArgs a, int hd, int first) {
    const int unit = (int)(blockIdx.x / (unsigned)a.chunks), chunk = (int)(blockIdx.x % (unsigned)a.chunks);
    if ((int)blockIdx.y + first == 0)
        mx_gather<KB>(a.k, a.out_k, a.k_rows, a, hd, unit, chunk);
    else
        mx_gather<VB>(a.v, a.out_v, a.v_rows, a, hd, unit, chunk);
}

// ---- attention ------------------------------------------------------------------------------------------------------
//
// One token's attention, out = sum_r p_r v_r / sum_r p_r with p_r = exp(scale q k_r - m), over the rows of every sequence
// (all of them, or its first n_sink and its last window).  A unit's rows are cut into steps of 16 TILES rows and its steps
// into n_splits equal parts, a block each, whose waves take them in turn; a wave keeps its running maximum, sum and
// weighted rows in registers, so the codes are read once and nothing is written but the parts' results.
//
//   S = K Q^T   v_mfma_f32_16x16x32_bf16 over 16 rows (M), 16 query heads (N) and 32 columns.  The codes become bf16 numbers, their
//               scale included, exactly (one conversion for two numbers), and are operands as they come: which columns an
//               instruction takes is free as long as Q's are the same, so lane (q, c) = (lane / 16, lane % 16) has 16 bytes (8
//               of 64 columns in 4 bits) of one row, the row's four lanes side by side.  (The instructions that multiply
//               4-bit and 8-bit numbers as they are gave sums off by up to 2^-13 of that of the products' magnitudes: not
//               enough for logits of a few tens.)
//   softmax     The heads of a group of up to GP stand in the columns again and again, and lane c keeps the result of tile
//               c / GP only: 64 rows of 4 heads are then 4 numbers a lane, none of them idle.  In powers of two.  The maximum
//               moves only where a logit passes it by more than 8: rare, so nothing crosses lanes from step to step, and a
//               weight is at most 2^8 of fp32 sums.
//   O = P V     M = (tile, head) as the lanes have them, N = 16 of the hd columns, K = 32 rows of two tiles; P of the tiles that are not
//               a lane's is zero.  P is the sum of two bf16 numbers: 2^-16 of a weight is lost at most, far below the output's own
//               2^-8.  Column n of instruction j is hd / 16 n + j,
//               so that a lane loads adjacent codes of its own rows and pairs of rows are put together by byte permutes.
//
// Which row of a tile is which row of M is free as long as K and V agree: M row 4 q + i is the tile's row 4 i + q, so that
// every load takes whole lines (with row 4 q + i they are asked for in pieces, which non-temporal loads do not find in the
// nearest cache: 2.4 times the requests of the next, 183 us for 174 at 8 x 131072 tokens).
// Rows behind the end are not asked for: a step's buffers end at its last row, and what a load asks of the words past a buffer's
// end is zero.  Offsets inside a step are constants of the load up to its 4095; the later rows of a step of 8 bits a number lie past that at 128
// columns and at 256, and add to a register.
//
// What bounds it: HBM from some 100 MB on.  8 x 131072 tokens of 8 heads x 128 with groups of 4, in 4 bits, 1.14 GB: 173-181 us =
// 6.3-6.6 TB/s (medians of seven runs of 20 launches); a million of one sequence 170-180 us; 8 x 65536 of 4 heads x 256 97 us = 5.9 TB/s;
// 8 x 131072 of 8 heads x 64 98 us = 5.8 TB/s.  64
// rows of 128 columns are some 370 vector, 48 matrix and 22 load instructions of a wave, 55 % of the time the bytes take.
// Below, the chain of length, rows, products and the join: 32601 tokens of 8 units 12.1 + 3.9 us (the bytes 5.4), 517 tokens
// 7.5 us in one kernel.  Starts of their own for the blocks' steps: without them a million tokens take 200 us for 177, the
// blocks' places being a power of two apart.  Loads without the non-temporal hint: 198 us for 180.
struct AttnArgs {
    const uint16_t *q, *new_k, *new_v;
    uint16_t *out;
    float *lse, *ws_acc, *ws_ml;
    const int32_t *lens;
    View k, v;
    int n_h, group, cap, n_sink, window, n_splits, waves;  // waves of a block
    uint32_t per_split;  // 2^32 / n_splits, rounded up
    float scale;  // times log2(e)
};

// What a unit's lengths come to.
struct Plan {
    int len, rows;            // rows before the token, and with it
    int sink, lo;             // rows [0, sink) and [lo, rows) are attended
    int sink_steps, steps, per;
};
template <int STEP>
__device__ __forceinline__ Plan mx_plan(const AttnArgs &a, int b) {
    Plan p;
    const int has_new = a.new_k != nullptr;
    int len = a.lens ? dc_step_word(a.lens + b) : a.cap - has_new;
    len = len < 0 ? 0 : (len < a.cap ? len : a.cap);
    p.len = len;
    p.rows = len + (has_new && len < a.cap ? 1 : 0);
    p.sink = 0, p.lo = 0;
    if (a.window > 0 && (int64_t)a.n_sink + a.window < p.rows) p.sink = a.n_sink, p.lo = p.rows - a.window;
    p.sink_steps = (int)(((uint32_t)p.sink + STEP - 1) / STEP);
    p.steps = p.sink_steps + (int)(((int64_t)p.rows - p.lo + STEP - 1) / STEP);
    // steps / n_splits, rounded up; now and then one more, which leaves a last part shorter
    p.per = a.n_splits == 1 ? p.steps : (int)__umulhi((uint32_t)(p.steps + a.n_splits - 1), a.per_split);
    p.per = p.per < a.waves ? a.waves : p.per;
    return p;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_rsrc(const uint8_t *base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, (int)bytes, 0x00020000);
}

// An offset whose bits the compiler does not know: it would make an or of a constant added to it, which the loads cannot take
// into their own constant, and spend a register and an instruction on every one of them.
__device__ __forceinline__ uint32_t mx_opaque(int x) {
    asm("" : "+v"(x));
    return (uint32_t)x;
}

// BYTES adjacent bytes at offset off.  AUX 2: read once (non-temporal)
constexpr int kOnce = 2;
template <int BYTES, int AUX>
__device__ __forceinline__ void mx_load(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t *dst) {
    if constexpr (BYTES == 1) {
        dst[0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(r, (int)off, 0, AUX);
    } else if constexpr (BYTES == 2) {
        dst[0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)off, 0, AUX);
    } else if constexpr (BYTES == 4) {
        dst[0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, AUX);
    } else if constexpr (BYTES == 8) {
        const mx_u32x2 t = __builtin_bit_cast(mx_u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, AUX));
        dst[0] = t.x, dst[1] = t.y;
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const mx_u32x4 t = __builtin_bit_cast(mx_u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(off + 16 * i), 0, AUX));
            dst[4 * i] = t.x, dst[4 * i + 1] = t.y, dst[4 * i + 2] = t.z, dst[4 * i + 3] = t.w;
        }
    }
}

__device__ __forceinline__ uint32_t mx_pack_bf16(float lo, float hi) { return mx_bits(mx_bf16x2{(__bf16)lo, (__bf16)hi}); }

// a over the lanes' halves in the low half, b over them in the high one
__device__ __forceinline__ float mx_fold32(float a, float b) {
    const mx_u32x2 r = __builtin_bit_cast(mx_u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false));
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}
// a over the rows 0 and 1 (2 and 3) of 16 lanes in row 0 (2), b over them in row 1 (3)
__device__ __forceinline__ float mx_fold16(float a, float b) {
    const mx_u32x2 r = __builtin_bit_cast(mx_u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false));
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}

// f over the lanes whose number is the same modulo GP (4, 8 or 16), in every one of them
template <int GP, typename F>
__device__ __forceinline__ float mx_over_lanes(float x, F f) {
    auto turned = [](float v, auto ctrl) __attribute__((always_inline)) {  // by 4 or 8 lanes of 16
        return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if constexpr (GP <= 4) x = f(x, turned(x, std::integral_constant<int, 0x124>{}));  // row_ror:4
    if constexpr (GP <= 8) x = f(x, turned(x, std::integral_constant<int, 0x128>{}));  // row_ror:8
    const uint32_t u = __float_as_uint(x);
    const mx_u32x2 r = __builtin_bit_cast(mx_u32x2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    x = f(__uint_as_float(r.x), __uint_as_float(r.y));
    const uint32_t w = __float_as_uint(x);
    const mx_u32x2 s = __builtin_bit_cast(mx_u32x2, __builtin_amdgcn_permlane32_swap(w, w, false, false));
    return f(__uint_as_float(s.x), __uint_as_float(s.y));
}

template <int HD, int KB, int VB, int GP, int TILES>
struct Attn {
    static constexpr int STEP = 16 * TILES;
    static constexpr int CH = HD / 32;          // products of a tile's S; blocks of a row
    static constexpr int EPL = HD / 16;         // columns of V of a lane
    // K: KN loads of KBYTES, KCOLS columns of one block each, those of a row's four lanes side by side
    static constexpr int KCOLS = HD == 64 ? 16 : 128 / KB, KN = HD / 4 / KCOLS, KBYTES = KCOLS * KB / 8, KW = KN * KBYTES / 4;
    static constexpr int kcol(int j) { return j * 8 / KCOLS * 4 * KCOLS + j * 8 % KCOLS; }  // first column of chunk j, of lanes q = 0
    static constexpr int VBYTES = EPL * VB / 8, VW = VBYTES < 4 ? 1 : VBYTES / 4;
    static constexpr int KROW = HD * KB / 8, VROW = HD * VB / 8;
    static constexpr int SBYTES = STEP * CH;    // a step's scales
    static constexpr int SETS = 16 / GP < TILES ? 16 / GP : TILES;  // tiles whose logits share a register
    static constexpr int REGS = TILES / SETS;   // logit registers of a lane (times 4)

    // A head's maximum before any logit passed it, in a wave with rows (-inf stands for no rows): finite, so that a row whose logit is
    // -inf has the weight 0 then too, where -inf - -inf would be NaN.
    static constexpr float kLowest = -3.402823466e+38f;

    mx_u32x4 bq[CH];
    uint32_t kw[TILES][KW], ks[CH > 4 ? 2 : 1];
    uint32_t vw[TILES * 4][VW], vs[CH > 4 ? 2 : 1];
    mx_f32x4 acc[EPL];
    float m, l;
    int q, c;

    __device__ __forceinline__ void start(const AttnArgs &a, int unit, int lane) {
        q = lane >> 4, c = lane & 15;
        const int head = c % GP < a.group ? c % GP : a.group - 1;  // (the last head again in the place of one that does not exist)
        const uint16_t *src = a.q + ((int64_t)unit * a.group + head) * HD + q * KCOLS;
#pragma unroll
        for (int j = 0; j < CH; ++j) bq[j] = *reinterpret_cast<const mx_u32x4 *>(src + kcol(j));
#pragma unroll
        for (int j = 0; j < EPL; ++j) acc[j] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY, l = 0.f;
    }

    // Codes and scales of the rows [row, row + live) of a unit, live <= STEP; lane (q, c) has row 4 (c % 4) + c / 4 of every tile.
    // The scales of the whole step are one load: lane l has row l's.
    __device__ __forceinline__ void load_k(const uint8_t *codes, const uint8_t *scale, int64_t row, int live) {
        const __amdgpu_buffer_rsrc_t rc = mx_rsrc(codes + row * KROW, (uint32_t)live * KROW), rs = mx_rsrc(scale + row * CH, (uint32_t)live * CH);
        const uint32_t oc = mx_opaque((4 * (c & 3) + (c >> 2)) * KROW + q * KBYTES);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int n = 0; n < KN; ++n) mx_load<KBYTES, kOnce>(rc, oc + 16 * KROW * t + 4 * KBYTES * n, &kw[t][KBYTES / 4 * n]);
        mx_load<CH, 0>(rs, (uint32_t)(16 * q + c) * CH, ks);
    }
    // lane (q, c) has columns EPL c .. of the rows 4 i + q of every tile
    __device__ __forceinline__ void load_v(const uint8_t *codes, const uint8_t *scale, int64_t row, int live) {
        const __amdgpu_buffer_rsrc_t rc = mx_rsrc(codes + row * VROW, (uint32_t)live * VROW), rs = mx_rsrc(scale + row * CH, (uint32_t)live * CH);
        const uint32_t oc = mx_opaque(q * VROW + c * VBYTES);
#pragma unroll
        for (int t = 0; t < TILES * 4; ++t) mx_load<VBYTES, kOnce>(rc, oc + 4 * VROW * t, vw[t]);
        mx_load<CH, 0>(rs, (uint32_t)(16 * q + c) * CH, vs);
    }

    // A step's scales go through the wave's own bytes of LDS, from a row to a lane to what the lanes use: block by block, the rows
    // in the order of the lanes that have them.  (Byte by byte from memory they are 20 of a step's 40 loads.)
    __device__ __forceinline__ void spread(uint8_t *lds, const uint32_t *w, int slot) const {
        if (16 * q + c < STEP) {
#pragma unroll
            for (int j = 0; j < CH; ++j) lds[j * STEP + slot] = (uint8_t)(w[j / 4] >> (8 * (j % 4)));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (what is read back is other lanes')
        __builtin_amdgcn_wave_barrier();
    }
    __device__ __forceinline__ void spread_k(uint8_t *lds, uint32_t (&f)[KN]) const {
        spread(lds, ks, (4 * (c & 3) + (c >> 2)) * TILES + q);  // row 16 q + c of the step is tile q's, of the lanes 4 (c % 4) + c / 4
#pragma unroll
        for (int n = 0; n < KN; ++n) {
            const uint8_t *src = lds + (4 * KCOLS * n + q * KCOLS) / 32 * STEP + c * TILES;
            if constexpr (TILES == 4) f[n] = *reinterpret_cast<const uint32_t *>(src);
            else f[n] = *reinterpret_cast<const uint16_t *>(src);
        }
    }
    __device__ __forceinline__ void spread_v(uint8_t *lds, uint32_t (&f)[TILES]) const {
        spread(lds, vs, (c & 3) * 4 * TILES + 4 * q + (c >> 2));  // row 16 q + c is row 4 i + c % 4 of tile q, i = c / 4
        const uint8_t *src = lds + c * EPL / 32 * STEP + q * 4 * TILES;
        if constexpr (TILES == 4) {
            const uint4 t = *reinterpret_cast<const uint4 *>(src);
            f[0] = t.x, f[1] = t.y, f[2] = t.z, f[3] = t.w;
        } else {
            const uint2 t = *reinterpret_cast<const uint2 *>(src);
            f[0] = t.x, f[1] = t.y;
        }
    }

    template <int T>
    __device__ __forceinline__ mx_f32x4 logits_of(const uint32_t (&ksc)[KN]) const {
        mx_f32x4 s = {0.f, 0.f, 0.f, 0.f};
        auto chunk = [&](auto jj) __attribute__((always_inline)) {
            constexpr int J = decltype(jj)::value;
            const float f = mx_scale((ksc[J * 8 / KCOLS] >> (8 * T)) & 0xffu);
            const mx_u32x4 x = {mx_pair<KB, 4 * J>(kw[T], f), mx_pair<KB, 4 * J + 1>(kw[T], f), mx_pair<KB, 4 * J + 2>(kw[T], f),
                                mx_pair<KB, 4 * J + 3>(kw[T], f)};
            s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx_bf16x8, x), __builtin_bit_cast(mx_bf16x8, bq[J]), s, 0, 0, 0);
        };
        each<CH>(chunk);
        return s;
    }

    template <int N, typename F>
    static __device__ __forceinline__ void each(F f) {
        each_of(f, std::make_integer_sequence<int, N>{});
    }
    template <typename F, int... I>
    static __device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
        (f(std::integral_constant<int, I>{}), ...);
    }

    // the logits of the step that load_k brought, by lane and register: x[r][i] = tile r SETS + c / GP, row 4 i + q, head c % GP
    __device__ __forceinline__ void logits(uint8_t *lds, float scale, float (&x)[REGS][4]) const {
        const int set = c / GP;
        uint32_t ksc[KN];
        spread_k(lds, ksc);
        each<TILES>([&](auto tt) __attribute__((always_inline)) {
            constexpr int T = decltype(tt)::value;
            const mx_f32x4 s = logits_of<T>(ksc);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (T % SETS == 0)
                    x[T / SETS][i] = s[i];
                else
                    x[T / SETS][i] = set >= T % SETS ? s[i] : x[T / SETS][i];
            }
        });
#pragma unroll
        for (int r = 0; r < REGS; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[r][i] *= scale;
    }

    // a new maximum for every head, and what was summed so far brought to it
    __device__ __forceinline__ void raise(float most) {
        const float to = fmaxf(m, mx_over_lanes<GP>(most, [](float a, float b) { return fmaxf(a, b); }));
        if (__any(m > kLowest)) {
            const float f = m > kLowest ? __builtin_amdgcn_exp2f(m - to) : 1.f;  // (nothing was summed, or what is no number)
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

    // weights of the step: p from x; live < STEP where rows are missing
    __device__ __forceinline__ void weigh(float (&x)[REGS][4], int live) {
        if (live < STEP) {
#pragma unroll
            for (int r = 0; r < REGS; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if ((r * SETS + c / GP) * 16 + 4 * i + q >= live) x[r][i] = -INFINITY;
        }
        float most = -INFINITY;
#pragma unroll
        for (int r = 0; r < REGS; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, x[r][i]);
        if (__any(most > m + 8.f)) raise(most);
#pragma unroll
        for (int r = 0; r < REGS; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[r][i] = __builtin_amdgcn_exp2f(x[r][i] - m);
        if (live < STEP) {
#pragma unroll
            for (int r = 0; r < REGS; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if ((r * SETS + c / GP) * 16 + 4 * i + q >= live) x[r][i] = 0.f;
        }
#pragma unroll
        for (int r = 0; r < REGS; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) l += x[r][i];
    }

    // dst[head][column] = the wave's sums over all tiles: M row 4 q + i is head (4 q + i) % GP of a tile.  Rows of 16 lanes trade
    // halves of what they hold, so that each ends with the sums of its own heads.
    __device__ __forceinline__ void finish(float *dst, int G) const {
        float o[GP / 4][EPL];  // the heads of this row of lanes
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            if constexpr (GP == 4) {
                o[0][j] = mx_fold16(mx_fold32(acc[j][0], acc[j][2]), mx_fold32(acc[j][1], acc[j][3]));
            } else if constexpr (GP == 8) {
                o[0][j] = mx_fold32(acc[j][0], acc[j][2]), o[1][j] = mx_fold32(acc[j][1], acc[j][3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i][j] = acc[j][i];
            }
        }
#pragma unroll
        for (int r = 0; r < GP / 4; ++r) {
            const int head = GP == 4 ? q : GP == 8 ? 4 * (q & 1) + (q >> 1) * 2 + r : 4 * q + r;
            if (head < G) {
#pragma unroll
                for (int j = 0; j < EPL; j += 4)
                    *reinterpret_cast<float4 *>(dst + head * HD + c * EPL + j) = make_float4(o[r][j], o[r][j + 1], o[r][j + 2], o[r][j + 3]);
            }
        }
    }

    // acc += P V over the step that load_v brought
    __device__ __forceinline__ void add(uint8_t *lds, const float (&x)[REGS][4]) {
        uint32_t vsc[TILES];
        spread_v(lds, vsc);
        uint32_t hi[REGS][2], lo[REGS][2];
#pragma unroll
        for (int r = 0; r < REGS; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                hi[r][i] = mx_pack_bf16(x[r][2 * i], x[r][2 * i + 1]);
                lo[r][i] = mx_pack_bf16(x[r][2 * i] - dc_bf16_lo(hi[r][i]), x[r][2 * i + 1] - dc_bf16_hi(hi[r][i]));
            }
        const int set = c / GP;
        each<TILES / 2>([&](auto uu) __attribute__((always_inline)) {
            constexpr int U = decltype(uu)::value, T0 = 2 * U, T1 = 2 * U + 1;
            auto of = [&](const uint32_t(&w)[REGS][2], int tile, int i) __attribute__((always_inline)) {
                return set == tile % SETS ? w[tile / SETS][i] : 0u;
            };
            const mx_u32x4 ah = {of(hi, T0, 0), of(hi, T0, 1), of(hi, T1, 0), of(hi, T1, 1)};
            const mx_u32x4 al = {of(lo, T0, 0), of(lo, T0, 1), of(lo, T1, 0), of(lo, T1, 1)};
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = mx_scale((vsc[2 * U + i / 4] >> (8 * (i % 4))) & 0xffu);
            each<EPL / 2>([&](auto jj) __attribute__((always_inline)) {
                constexpr int J = decltype(jj)::value;
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = mx_pair<VB, J>(vw[8 * U + i], f[i]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t sel = half ? 0x07060302u : 0x05040100u;  // the high or the low halves of two words
                    const mx_u32x4 b = {__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel),
                                        __builtin_amdgcn_perm(w[5], w[4], sel), __builtin_amdgcn_perm(w[7], w[6], sel)};
                    mx_f32x4 &o = acc[2 * J + half];
                    o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx_bf16x8, al), __builtin_bit_cast(mx_bf16x8, b), o, 0, 0, 0);
                    o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx_bf16x8, ah), __builtin_bit_cast(mx_bf16x8, b), o, 0, 0, 0);
                }
            });
        });
    }
};

inline size_t attn_shared_bytes(int hd, int group, int waves) {
    const size_t sums = (size_t)group * hd * sizeof(float), scales = 2 * (hd == 256 ? 32 : 64) * (hd / 32);
    return waves * (32 * sizeof(float) + (sums > scales ? sums : scales));
}

template <int HD, int KB, int VB, int GP, int TILES>
__global__ __launch_bounds__(kMostWaves * 64, 2) void mx_attn_kernel(AttnArgs a) {
    using T = Attn<HD, KB, VB, GP, TILES>;
    constexpr int STEP = T::STEP;
    extern __shared__ float s_dyn[];
    // (all arguments at once: read where they are first used, they are half a dozen round trips in a row)
    asm volatile("" ::"s"(a.q), "s"(a.new_k), "s"(a.lens), "s"(a.k.codes), "s"(a.k.scale), "s"(a.k.cb), "s"(a.k.ch), "s"(a.k.sb),
                 "s"(a.k.sh), "s"(a.v.codes), "s"(a.v.scale), "s"(a.v.cb), "s"(a.v.ch), "s"(a.v.sb), "s"(a.v.sh),
                 "s"(a.n_h), "s"(a.group), "s"(a.cap), "s"(a.n_sink), "s"(a.window), "s"(a.n_splits), "s"(a.waves));
    const int waves = a.waves;
    float *s_m = s_dyn, *s_l = s_dyn + waves * 16, *s_acc = s_dyn + 2 * waves * 16;  // [wave][16], [wave][16], [wave][group * HD]
    const int b = blockIdx.x, h = blockIdx.y, split = blockIdx.z, unit = b * a.n_h + h, G = a.group;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    T w;
    w.start(a, unit, lane);
    uint8_t *lds = reinterpret_cast<uint8_t *>(s_acc) + wave * 2 * T::SBYTES;  // (the sums come when all scales were used)
    const Plan p = mx_plan<STEP>(a, b);
    const int begin = split * p.per, end = begin + p.per < p.steps ? begin + p.per : p.steps;
    if (begin >= end && a.n_splits > 1) {  // a part without rows: the merge takes nothing of it
        if (tid < G) reinterpret_cast<float2 *>(a.ws_ml)[((int64_t)unit * a.n_splits + split) * G + tid] = make_float2(-INFINITY, 0.f);
        return;
    }
    const uint8_t *kc = a.k.codes + b * a.k.cb + h * a.k.ch, *ksc = a.k.scale + b * a.k.sb + h * a.k.sh;
    const uint8_t *vc = a.v.codes + b * a.v.cb + h * a.v.ch, *vsc = a.v.scale + b * a.v.sb + h * a.v.sh;

    // step s: rows [row, row + live)
    auto place = [&](int s, int64_t &row, int &live) __attribute__((always_inline)) {
        const bool in_sink = s < p.sink_steps;
        row = in_sink ? (int64_t)s * STEP : p.lo + (int64_t)(s - p.sink_steps) * STEP;
        const int64_t left = (in_sink ? p.sink : p.rows) - row;
        live = left < STEP ? (int)left : STEP;
    };
    // a wave's steps are every waves-th of the block's, from a start of its block's own on
    const int mine = end > begin + wave ? (end - begin - wave + waves - 1) / waves : 0;
    const uint32_t turn = (uint32_t)(unit * a.n_splits + split) * 0x9e3779b9u;
    // The token's row is the unit's last: the wave with the last step writes it first and takes that step last, token or not (so
    // that a row written beforehand gives the same sums).
    const bool last = mine > 0 && begin + wave + (mine - 1) * waves == p.steps - 1, writes = last && p.rows > p.len;
    if (mine > 0) w.m = T::kLowest;
    int at = last ? 0 : (int)(((uint64_t)turn * (uint32_t)mine) >> 32);
    if (writes) mx_write_token<KB, VB>(a.k, a.v, a.new_k, a.new_v, HD, unit, b, h, p.len, lane);
    int64_t row;
    int live = 0;
    auto load_k = [&]() __attribute__((always_inline)) {
        if (writes && at == mine - 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // (its lanes see each other's stores)
        place(begin + wave + at * waves, row, live);
        w.load_k(kc, ksc, row, live);
    };
    if (mine > 0) {
        load_k();
        w.load_v(vc, vsc, row, live);
    }
    for (int i = 0; i < mine; ++i) {
        float x[T::REGS][4];
        w.logits(lds, a.scale, x);
        const int now = live;
        const bool more = i + 1 < mine;
        if (more) {
            at = at + 1 < mine ? at + 1 : 0;
            load_k();
        }
        w.weigh(x, now);
        w.add(lds + T::SBYTES, x);
        if (more) w.load_v(vc, vsc, row, live);
    }

    // the wave's heads: over the lanes that had other rows, and over the tiles
    __syncthreads();
    const float l = mx_over_lanes<GP>(w.l, [](float a, float b) { return a + b; });
    if (lane < GP) s_m[wave * 16 + lane] = w.m, s_l[wave * 16 + lane] = l;
    w.finish(s_acc + wave * G * HD, G);
    __syncthreads();
    auto weight = [](float m, float top) __attribute__((always_inline)) { return m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 0.f; };
    const int64_t slot = (int64_t)unit * a.n_splits + split;
    for (int o = tid; o < G * HD; o += waves * 64) {
        const int head = o / HD;
        // (without a branch to a wave: the first one again in the place of those that a block of four does not have)
        float m[kMostWaves], l[kMostWaves], part[kMostWaves];
#pragma unroll
        for (int i = 0; i < kMostWaves; ++i) {
            const int at = i < waves ? i : 0;
            m[i] = s_m[at * 16 + head], l[i] = s_l[at * 16 + head], part[i] = s_acc[at * G * HD + o];
        }
        float top = m[0];
#pragma unroll
        for (int i = 1; i < kMostWaves; ++i) top = fmaxf(top, m[i]);
        float sum = 0.f, total = 0.f;
#pragma unroll
        for (int i = 0; i < kMostWaves; ++i) {
            const float f = i < waves ? weight(m[i], top) : 0.f;
            sum = fmaf(f, i < waves ? part[i] : 0.f, sum);
            total += i >= waves ? 0.f : l[i] == l[i] ? f * l[i] : l[i];  // (a sum that is no number stays none, whatever its maximum)
        }
        if (a.n_splits > 1) {
            a.ws_acc[slot * (G * HD) + o] = sum;
            if (o % HD == 0) {
                float *ml = a.ws_ml + (slot * G + head) * 2;
                ml[0] = top, ml[1] = total;
            }
        } else {
            a.out[(int64_t)unit * G * HD + o] = dc_f32_to_bf16(sum / (total == 0.f ? 1.f : total));
            if (a.lse && o % HD == 0) a.lse[(int64_t)unit * G + head] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.693147180559945309f;
        }
    }
}

// The parts of one query head joined: one block per (unit, head).  What it reads is asked for at once, before any weight is
// known: rounds of kBatch kParts parts (32 at 128 and at 256 columns, 64 at 64), HD / 4 threads to a part.  A kernel's start and two round trips: 64
// parts of 32 heads 3.9 us (5.5 part by part), 8 parts of 256 heads 4.8, 128 parts of 16 heads of 256 columns 5.0 (6.2 in rounds of 16).
// A unit alone has its rounds one after the other: 512 parts of 4 heads of 128 columns 13.4, 1024 of 64 columns 17.7.
template <int HD>
__global__ __launch_bounds__(kThreads) void mx_merge_kernel(AttnArgs a) {
    constexpr int kLanes = HD / 4, kParts = kThreads / kLanes, kBatch = HD == 256 ? 8 : 4;
    __shared__ float4 s_acc[kThreads];
    const int unit = blockIdx.x / a.group, g = blockIdx.x % a.group, tid = threadIdx.x, lane = tid & 63, n = a.n_splits;
    const int64_t slot0 = (int64_t)unit * n * a.group + g;
    const float2 *ml = reinterpret_cast<const float2 *>(a.ws_ml) + slot0;
    const float4 *pa = reinterpret_cast<const float4 *>(a.ws_acc) + slot0 * kLanes + tid % kLanes;
    float4 v[kBatch];
    float2 o[kBatch];
    auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {  // (the last part again where there are no more)
            const int s = s0 + i * kParts, at = (s < n ? s : n - 1) * a.group;
            o[i] = ml[at], v[i] = pa[(int64_t)at * kLanes];
        }
    };
    const float2 own = lane < n ? ml[lane * a.group] : make_float2(-INFINITY, 0.f);
    load(tid / kLanes);
    float top = own.x;
    for (int s = lane + 64; s < n; s += 64) top = fmaxf(top, ml[s * a.group].x);
    top = mx_over_lanes<4>(top, [](float x, float y) { return fmaxf(x, y); });
#pragma unroll
    for (int d = 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    auto weight = [&](float m) __attribute__((always_inline)) { return m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 0.f; };
    auto share = [&](float2 x) __attribute__((always_inline)) { return x.y == x.y ? weight(x.x) * x.y : x.y; };
    float total = share(own);
    for (int s = lane + 64; s < n; s += 64) total += share(ml[s * a.group]);
    total = mx_over_lanes<4>(total, [](float x, float y) { return x + y; });
#pragma unroll
    for (int d = 2; d > 0; d >>= 1) total += __shfl_xor(total, d, 64);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = tid / kLanes;;) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            // (a part without rows has no sums in the workspace)
            const bool in = s0 + i * kParts < n && o[i].x > -INFINITY;
            const float f = in ? weight(o[i].x) : 0.f;
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
        a.out[(int64_t)blockIdx.x * HD + tid] = dc_f32_to_bf16(sum / (total == 0.f ? 1.f : total));
    }
    if (a.lse && tid == 0) a.lse[blockIdx.x] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.693147180559945309f;
}

// ---- host -----------------------------------------------------------------------------------------------------------

// Whether no two of n_b x n_h units, size bytes each, have a byte in common: every pair is an offset of i sb and one of j sh apart.
bool units_apart(int64_t n_b, int64_t n_h, uint64_t sb, uint64_t sh, uint64_t size) {
    if ((n_h <= 1 || sh >= size) && (n_b <= 1 || sb >= (uint64_t)(n_h - 1) * sh + size)) return true;  // (a sequence behind the other)
    if (n_b > n_h) {
        const int64_t n = n_b;
        const uint64_t s = sb;
        n_b = n_h, sb = sh, n_h = n, sh = s;
    }
    // n_b is the smaller count: for every i sb the multiples of sh next to it
    for (int64_t i = 0; i < n_b; ++i) {
        const uint64_t x = (uint64_t)i * sb;
        uint64_t j = sh ? x / sh : 0;
        if (j > (uint64_t)(n_h - 1)) j = (uint64_t)(n_h - 1);
        if ((i || j) && x - j * sh < size) return false;
        if (j + 1 < (uint64_t)n_h && (j + 1) * sh - x < size) return false;
    }
    return true;
}

int check_store(const char *who, const char *which, const dc_mx_store &s, int n_b, int n_h, int hd, bool written) {
    DC_REQUIRE(s.bits == 4 || s.bits == 8, "%s: %s holds %d bits, not 4 or 8", who, which, s.bits);
    DC_REQUIRE(s.n_rows >= 0, "%s: %s has a negative number of rows", who, which);
    DC_REQUIRE((s.codes && s.scale) || s.n_rows == 0, "%s: null pointer in %s", who, which);
    const int64_t blocks = hd / 32;
    DC_REQUIRE(dc_aligned16(s.codes) && s.code_batch_stride % 16 == 0 && s.code_head_stride % 16 == 0,
               "%s: %s's codes must be 16-byte aligned, their strides multiples of 16 bytes", who, which);
    DC_REQUIRE((uintptr_t)s.scale % blocks == 0 && s.scale_batch_stride % blocks == 0 && s.scale_head_stride % blocks == 0,
               "%s: %s's scales and their strides must be multiples of %lld bytes", who, which, (long long)blocks);
    DC_REQUIRE(s.code_batch_stride >= 0 && s.code_head_stride >= 0 && s.scale_batch_stride >= 0 && s.scale_head_stride >= 0,
               "%s: negative stride in %s", who, which);
    if (written) {
        DC_REQUIRE(units_apart(n_b, n_h, (uint64_t)s.code_batch_stride, (uint64_t)s.code_head_stride, (uint64_t)s.n_rows * (hd * s.bits / 8)) &&
                       units_apart(n_b, n_h, (uint64_t)s.scale_batch_stride, (uint64_t)s.scale_head_stride, (uint64_t)s.n_rows * blocks),
                   "%s: units of %s share their rows", who, which);
    }
    return DC_OK;
}

int check_units(const char *who, int n_b, int n_h, int hd) {
    DC_REQUIRE(n_b >= 0 && n_h >= 1, "%s: bad sizes", who);
    DC_REQUIRE((int64_t)n_b * n_h < (1 << 24), "%s: too many units", who);
    DC_REQUIRE(hd == 64 || hd == 128 || hd == 256, "%s: head_dim %d unsupported", who, hd);
    return DC_OK;
}

// A launch has less than 2^32 threads in a dimension.
bool grid_fits(int64_t blocks, int threads) { return blocks * threads < (1ll << 32); }

// chunks: blocks of a unit in a grid of (unit, chunk) in one dimension; the last one's rows, those beyond the end too, are ints
int check_grid(const char *who, int64_t n_units, int64_t chunks, int rows_per) {
    DC_REQUIRE(grid_fits(n_units * chunks, kThreads) && chunks * rows_per < (1ll << 31), "%s: grid too large", who);
    return DC_OK;
}

#define DC_TRY(x)                 \
    do {                          \
        const int rc_ = (x);      \
        if (rc_ != DC_OK) return rc_; \
    } while (0)

#define DC_MX_BY_BITS(KERNEL, KBITS, VBITS, ...)                                              \
    do {                                                                                      \
        if ((KBITS) == 4 && (VBITS) == 4) hipLaunchKernelGGL((KERNEL<4, 4>), __VA_ARGS__);    \
        else if ((KBITS) == 4) hipLaunchKernelGGL((KERNEL<4, 8>), __VA_ARGS__);               \
        else if ((VBITS) == 4) hipLaunchKernelGGL((KERNEL<8, 4>), __VA_ARGS__);               \
        else hipLaunchKernelGGL((KERNEL<8, 8>), __VA_ARGS__);                                 \
    } while (0)

constexpr int attn_tiles(int hd) { return hd == 256 ? 2 : 4; }

// How a unit's rows are dealt out.
struct AttnCut {
    int n_splits, waves;
};
// Blocks of four waves: two to a CU, which the loads in flight of 64 rows to a wave keep busy (8 x 131072 tokens of 8 heads x
// 128 in 4 bits: 174 us, with 768 blocks 176, with 1024 183; a document of 32601 12.5 / 13.7 / 14.0).  Rows of 32 bytes are half
// of that in flight: four to a CU once every wave has six steps or more (64 columns, 4 bits: 16 x 32000 tokens 60.6 -> 50.8 us, a
// million of one 112 -> 92.5, but 2 x 32000 12.3 -> 12.6).  Every unit gets the same number of blocks, rounded down: with 8192 rows of 128
// columns 256 units take 47 us, 384 79, 512 89, 640 121; of 64 units whose lengths differ the longest's blocks end last (8 of 131072
// rows and 56 of 8192: 152 us, 64 of their mean length 36).
constexpr int kBlocks = 512, kLeanBlocks = 2 * kBlocks, kLeanSteps = 6 * kWaves;
// Steps of a wave up to which a unit is one block of eight waves, which writes the output itself: less than a second kernel
// that joins parts (1024 tokens: 9.3 us, in parts 6.5 + 2.7 and a launch; 1500: 11.5, 8.7 + 2.9; 2048: 13.6, 7.5 + 2.8).
constexpr int kAlone = 3, kWide = 8;
AttnCut attn_cut(int64_t n_units, int hd, int64_t n_rows, int n_sink, int bits) {
    const int64_t step = 16 * attn_tiles(hd);
    const int64_t steps = (n_rows + step - 1) / step + (n_sink + step - 1) / step;
    if (steps <= kAlone * kWide) return {1, steps <= kWaves ? kWaves : kWide};
    const bool lean = hd == 64 && bits == 8 && n_units * steps >= (int64_t)kLeanSteps * kBlocks;
    const int64_t parts = (steps + kWaves - 1) / kWaves, blocks = lean ? kLeanBlocks : kBlocks, most = blocks / n_units > 1 ? blocks / n_units : 1;
    return {(int)(parts < most ? parts : most), kWaves};
}

template <int HD, int KB, int VB>
void launch_attn(const AttnArgs &a, int n_units, hipStream_t st) {
    constexpr int TILES = attn_tiles(HD);
    const dim3 grid((unsigned)(n_units / a.n_h), (unsigned)a.n_h, (unsigned)a.n_splits);
    const size_t lds = attn_shared_bytes(HD, a.group, a.waves);
#define DC_LAUNCH_MX(GP) hipLaunchKernelGGL((mx_attn_kernel<HD, KB, VB, GP, TILES>), grid, dim3(a.waves * 64), lds, st, a)
    if (a.group > 8) DC_LAUNCH_MX(16);
    else if (a.group > 4 || TILES == 2) DC_LAUNCH_MX(8);
    else if constexpr (TILES == 4) DC_LAUNCH_MX(4);
#undef DC_LAUNCH_MX
    if (a.n_splits > 1)
        hipLaunchKernelGGL(mx_merge_kernel<HD>, dim3((unsigned)(n_units * a.group)), dim3(kThreads), 0, st, a);
}

template <int HD>
void launch_attn_bits(int kbits, int vbits, const AttnArgs &a, int n_units, hipStream_t st) {
    if (kbits == 4 && vbits == 4) launch_attn<HD, 4, 4>(a, n_units, st);
    else if (kbits == 4) launch_attn<HD, 4, 8>(a, n_units, st);
    else if (vbits == 4) launch_attn<HD, 8, 4>(a, n_units, st);
    else launch_attn<HD, 8, 8>(a, n_units, st);
}

}  // namespace

extern "C" int dc_mx_ingest_bf16(const dc_mx_store *k, const dc_mx_store *v, const void *k_src, const void *v_src,
                                 const int32_t *lens, int n_b, int seq, int n_h, int hd, int dst_pos, int64_t ksb, int64_t kss,
                                 int64_t ksh, int64_t vsb, int64_t vss, int64_t vsh, void *stream) {
    const char *who = "dc_mx_ingest_bf16";
    DC_TRY(check_units(who, n_b, n_h, hd));
    DC_REQUIRE(seq >= 0 && dst_pos >= 0, "%s: bad sizes", who);
    const int64_t n_units = (int64_t)n_b * n_h;
    if (n_units == 0 || seq == 0) return DC_OK;
    DC_REQUIRE(k && v && k_src && v_src, "%s: null pointer", who);
    DC_TRY(check_store(who, "k", *k, n_b, n_h, hd, true));
    DC_TRY(check_store(who, "v", *v, n_b, n_h, hd, true));
    DC_REQUIRE((int64_t)dst_pos + seq <= k->n_rows && (int64_t)dst_pos + seq <= v->n_rows,
               "%s: rows [%d, %lld) outside the store", who, dst_pos, (long long)dst_pos + seq);
    DC_REQUIRE(dc_aligned16(k_src) && dc_aligned16(v_src), "%s: pointers must be 16-byte aligned", who);
    DC_REQUIRE(ksb % 8 == 0 && kss % 8 == 0 && ksh % 8 == 0 && vsb % 8 == 0 && vss % 8 == 0 && vsh % 8 == 0,
               "%s: strides must be multiples of 8 elements", who);
    const int rows_per = kThreads / (hd / 8) * kIngestBatch;
    const int64_t chunks = ((int64_t)seq + rows_per - 1) / rows_per;
    DC_TRY(check_grid(who, n_units, chunks, rows_per));
    IngestArgs a = {view_of(*k), view_of(*v), (const uint16_t *)k_src, (const uint16_t *)v_src, ksb, kss, ksh, vsb, vss, vsh,
                    lens, n_h, seq, dst_pos, (int)chunks};
    DC_MX_BY_BITS(mx_ingest_kernel, k->bits, v->bits, dim3((unsigned)(n_units * chunks), 2), dim3(kThreads), 0, (hipStream_t)stream, a, hd);
    DC_CHECK_LAUNCH(who);
    return DC_OK;
}

extern "C" int dc_mx_append_bf16(const dc_mx_store *k, const dc_mx_store *v, const void *new_k, const void *new_v, const int32_t *lens,
                                 int n_b, int n_h, int hd, void *stream) {
    const char *who = "dc_mx_append_bf16";
    DC_TRY(check_units(who, n_b, n_h, hd));
    const int n_units = n_b * n_h;
    if (n_units == 0) return DC_OK;
    DC_REQUIRE(k && v && new_k && new_v && lens, "%s: null pointer", who);
    DC_TRY(check_store(who, "k", *k, n_b, n_h, hd, true));
    DC_TRY(check_store(who, "v", *v, n_b, n_h, hd, true));
    DC_REQUIRE(dc_aligned16(new_k) && dc_aligned16(new_v), "%s: pointers must be 16-byte aligned", who);
    const int cap = k->n_rows < v->n_rows ? k->n_rows : v->n_rows;
    DC_MX_BY_BITS(mx_append_kernel, k->bits, v->bits, dim3((unsigned)((n_units + kWaves - 1) / kWaves)), dim3(kThreads), 0,
                  (hipStream_t)stream, view_of(*k), view_of(*v), (const uint16_t *)new_k, (const uint16_t *)new_v, lens, n_units, n_h, hd, cap);
    DC_CHECK_LAUNCH(who);
    return DC_OK;
}

extern "C" int dc_mx_gather_rows_bf16(const dc_mx_store *k, const dc_mx_store *v, const uint32_t *idx, void *out_k, void *out_v, int n_b,
                                      int n_h, int n_idx, int64_t idx_unit_stride, int hd, int64_t row_offset, int64_t dsb, int64_t dsh,
                                      int64_t dsr, void *stream) {
    const char *who = "dc_mx_gather_rows_bf16";
    DC_TRY(check_units(who, n_b, n_h, hd));
    DC_REQUIRE(n_idx >= 0 && row_offset >= 0 && row_offset < (1ll << 62), "%s: bad sizes", who);  // (an id is added to it)
    const int64_t n_units = (int64_t)n_b * n_h;
    if (n_units == 0 || n_idx == 0) return DC_OK;
    DC_REQUIRE(out_k || out_v, "%s: null pointer", who);
    DC_REQUIRE((!out_k || k) && (!out_v || v), "%s: source missing for an output", who);
    if (out_k) DC_TRY(check_store(who, "k", *k, n_b, n_h, hd, false));
    if (out_v) DC_TRY(check_store(who, "v", *v, n_b, n_h, hd, false));
    DC_REQUIRE(!idx || idx_unit_stride >= n_idx, "%s: idx_unit_stride < n_idx", who);
    DC_REQUIRE((!out_k || dc_aligned16(out_k)) && (!out_v || dc_aligned16(out_v)), "%s: pointers must be 16-byte aligned", who);
    DC_REQUIRE(dsb % 8 == 0 && dsh % 8 == 0 && dsr % 8 == 0, "%s: strides must be multiples of 8 elements", who);
    const int rows_per = kThreads / (hd / 8) * kGatherBatch;
    const int64_t chunks = ((int64_t)n_idx + rows_per - 1) / rows_per;
    DC_TRY(check_grid(who, n_units, chunks, rows_per));
    const dc_mx_store &ks = out_k ? *k : *v, &vs = out_v ? *v : *k;
    GatherArgs a = {view_of(ks), view_of(vs), idx, idx_unit_stride, row_offset, (uint16_t *)out_k, (uint16_t *)out_v, dsb, dsh, dsr,
                    n_h, n_idx, ks.n_rows, vs.n_rows, (int)chunks};
    DC_MX_BY_BITS(mx_gather_kernel, ks.bits, vs.bits, dim3((unsigned)(n_units * chunks), out_k && out_v ? 2 : 1), dim3(kThreads), 0,
                  (hipStream_t)stream, a, hd, out_k ? 0 : 1);
    DC_CHECK_LAUNCH(who);
    return DC_OK;
}

extern "C" size_t dc_mx_attn_workspace_bytes(int n_units, int group, int hd, int n_rows) {
    if (n_units <= 0 || group <= 0 || hd < 64 || n_rows < 0) return 0;
    // none where every unit is one block; else as many parts as the grid has blocks, or as there are: never less for more
    // units or rows.  (Sinks may make one step more of the rows.)
    const int64_t step = 16 * attn_tiles(hd), steps = (n_rows + step - 1) / step + 1;
    if (steps <= kAlone * kWide) return 0;
    const int64_t parts = n_units * ((steps + kWaves - 1) / kWaves);
    const int64_t blocks = hd == 64 ? kLeanBlocks : kBlocks;
    const size_t slots = (size_t)(parts < blocks ? parts : blocks);
    return dc_align_up(slots * group * hd * 4, 256) + dc_align_up(slots * group * 2 * 4, 256);
}

extern "C" int dc_mx_attn_bf16(const dc_mx_attn_args *x, void *stream) {
    const char *who = "dc_mx_attn_bf16";
    DC_REQUIRE(x, "%s: null pointer", who);
    DC_TRY(check_units(who, x->n_b, x->n_h, x->hd));
    const int n_units = x->n_b * x->n_h;
    if (n_units == 0) return DC_OK;
    DC_REQUIRE(x->q && x->out, "%s: null pointer", who);
    DC_REQUIRE((x->new_k == nullptr) == (x->new_v == nullptr), "%s: new_k and new_v must both be set or both be null", who);
    DC_TRY(check_store(who, "k", x->k, x->n_b, x->n_h, x->hd, x->new_k != nullptr));
    DC_TRY(check_store(who, "v", x->v, x->n_b, x->n_h, x->hd, x->new_k != nullptr));
    DC_REQUIRE(x->group >= 1 && x->group <= 16, "%s: group %d not in [1,16]", who, x->group);
    DC_REQUIRE(x->n_rows >= 0 && x->n_rows <= x->k.n_rows && x->n_rows <= x->v.n_rows, "%s: %d rows outside the store", who, x->n_rows);
    DC_REQUIRE(x->n_sink >= 0 && x->window >= 0, "%s: negative n_sink or window", who);
    DC_REQUIRE(dc_aligned16(x->q) && (!x->new_k || (dc_aligned16(x->new_k) && dc_aligned16(x->new_v))),
               "%s: pointers must be 16-byte aligned", who);
    DC_REQUIRE(x->n_h < (1 << 16), "%s: too many heads", who);
    const int64_t attended = x->window > 0 && (int64_t)x->n_sink + x->window < x->n_rows ? x->window : x->n_rows;
    AttnCut cut = attn_cut(n_units, x->hd, attended, attended < x->n_rows ? x->n_sink : 0, x->k.bits + x->v.bits);
    if (!grid_fits(x->n_b, cut.waves * 64)) cut.waves = kWaves;  // (of four waves all units fit that check_units lets through)
    AttnArgs a;
    a.n_splits = cut.n_splits, a.waves = cut.waves;
    a.per_split = (uint32_t)((0xffffffffull + a.n_splits) / a.n_splits);
    if (a.n_splits > 1) {
        const size_t slots = (size_t)n_units * a.n_splits;
        const size_t acc_bytes = dc_align_up(slots * x->group * x->hd * 4, 256), need = acc_bytes + dc_align_up(slots * x->group * 2 * 4, 256);
        DC_REQUIRE(x->workspace && ((uintptr_t)x->workspace & 255u) == 0, "%s: workspace must be non-null and 256-byte aligned", who);
        if (x->workspace_bytes < need) {
            dc_set_error("%s: workspace %zu bytes < %zu needed", who, x->workspace_bytes, need);
            return DC_ENOMEM;
        }
        a.ws_acc = (float *)x->workspace;
        a.ws_ml = (float *)((char *)x->workspace + acc_bytes);
    } else {
        a.ws_acc = a.ws_ml = nullptr;
    }
    a.q = (const uint16_t *)x->q, a.new_k = (const uint16_t *)x->new_k, a.new_v = (const uint16_t *)x->new_v;
    a.out = (uint16_t *)x->out, a.lse = x->lse, a.lens = x->lens;
    a.k = view_of(x->k), a.v = view_of(x->v);
    a.n_h = x->n_h, a.group = x->group, a.cap = x->n_rows, a.n_sink = x->n_sink, a.window = x->window;
    a.scale = x->scale * 1.44269504088896341f;
    hipStream_t st = (hipStream_t)stream;
    if (x->hd == 64) launch_attn_bits<64>(x->k.bits, x->v.bits, a, n_units, st);
    else if (x->hd == 128) launch_attn_bits<128>(x->k.bits, x->v.bits, a, n_units, st);
    else launch_attn_bits<256>(x->k.bits, x->v.bits, a, n_units, st);
    DC_CHECK_LAUNCH(who);
    return DC_OK;
}
