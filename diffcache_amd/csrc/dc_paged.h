// What the kernels of the paged cache share (paged.hip, paged_attn.hip, paged_chunk.hip): where a sequence's rows and its new tokens lie.
#pragma once
#include "dc_common.h"

// K and V in pages, as the kernels see them: row r of sequence b is row r % page of page table[b * table_stride + r / page].
struct DcPages {
    uint16_t *k, *v;
    int64_t kp, kh, vp, vh;  // strides of a page and of a head, in elements
    const int32_t *table;
    int64_t table_stride;
    int n_pages, shift;      // page = 1 << shift
};

// The new tokens of the sequences (dc_paged_tokens of the header).
struct DcNew {
    const int32_t *start, *cu, *counts;
    int max_new, n_tokens;
};

// One sequence's: token i < count stands at place first + i of the packed tensors and is the sequence's row start + i.
struct DcSpan {
    int first, count, start;
};
// Rows are 32-bit numbers: no sequence has more than this, and a longer start counts as this.
constexpr int kMostRows = 1 << 30;

__device__ __forceinline__ int dc_clamp(int x, int lo, int hi) { return x < lo ? lo : (x < hi ? x : hi); }
__device__ __forceinline__ DcSpan dc_span(const DcNew &t, int b) {
    DcSpan s;
    if (t.cu) {  // (whatever cu holds, no token lies outside the tensors)
        s.first = dc_clamp(dc_step_word(t.cu + b), 0, t.n_tokens);
        s.count = dc_clamp(dc_step_word(t.cu + b + 1), s.first, t.n_tokens) - s.first;
        s.count = s.count < t.max_new ? s.count : t.max_new;
    } else {
        s.first = b * t.max_new;
        s.count = t.counts ? dc_clamp(dc_step_word(t.counts + b), 0, t.max_new) : t.max_new;
    }
    s.start = t.start ? dc_clamp(dc_step_word(t.start + b), 0, kMostRows) : 0;
    return s;
}

// Tensors of tokens by strides (batch, token, head); the batch's is not used where tokens are packed.
struct DcTokenStrides {
    int64_t b, t, h;
};
__device__ __forceinline__ int64_t dc_token_at(const DcNew &t, const DcTokenStrides &s, const DcSpan &span, int b, int i) {
    return t.cu ? (int64_t)(span.first + i) * s.t : (int64_t)b * s.b + (int64_t)i * s.t;
}

// paged.hip: the checks that every entry makes of its pages and tokens
int dc_check_paged(const char *who, const dc_paged_store &s, const dc_paged_tokens &t, int n_h, int hd, bool written);
inline DcPages dc_pages_of(const dc_paged_store &s, const dc_paged_tokens &t) {
    return {(uint16_t *)s.k, (uint16_t *)s.v, s.k_page_stride, s.k_head_stride, s.v_page_stride, s.v_head_stride, t.table, t.table_stride,
            s.n_pages, __builtin_ctz((unsigned)s.page)};
}
inline DcNew dc_new_of(const dc_paged_tokens &t) { return {t.start, t.cu, t.counts, t.max_new, t.n_tokens}; }

// A launch has less than 2^32 threads in a dimension.
inline bool dc_grid_fits(int64_t blocks, int threads) { return blocks * threads < (1ll << 32); }

// ---- attention (paged_attn.hip, paged_chunk.hip) --------------------------------------------------------------------
struct DcPagedAttn {
    const uint16_t *q;
    uint16_t *out;
    float *lse, *ws_acc, *ws_ml;
    DcPages p;
    DcNew t;
    DcTokenStrides qs;
    int n_h, group, n_rows, n_sink, window;
    int n_splits, waves;     // parts of a unit's steps; waves of a block (paged_attn.hip)
    int tiles, tile_rows;    // of a unit's (token, head) rows: blocks, and rows of one
    float scale;             // times log2(e)
};

// Which rows a token attends to: [0, hi] without those in [sink, lo].
struct DcReach {
    int hi, lo, sink;
    __device__ __forceinline__ bool has(int row) const { return (row <= hi) & ((row > lo) | (row < sink)); }
};
__device__ __forceinline__ DcReach dc_reach(const DcPagedAttn &a, int p) {
    return {p < a.n_rows ? p : a.n_rows - 1, a.window ? p - a.window : -1, a.window ? a.n_sink : 0};
}
// Whether tokens at rows p_lo .. p_hi attend to all of rows [row, row + n)
__device__ __forceinline__ bool dc_whole(const DcPagedAttn &a, int p_lo, int p_hi, int row, int n) {
    return row + n - 1 <= p_lo && row + n <= a.n_rows && (a.window == 0 || row > p_hi - a.window || row + n <= a.n_sink);
}

// The steps of STEP rows that tokens at rows [p_lo, p_hi] need: the first `sinks` of a sequence's, then those from `first` on.
struct DcSteps {
    int sinks, first, steps;
    __device__ __forceinline__ int row(int s, int step) const { return (s < sinks ? s : first + s - sinks) * step; }
};
template <int STEP>
__device__ __forceinline__ DcSteps dc_steps(const DcPagedAttn &a, int p_lo, int p_hi) {
    DcSteps s;
    const int last = p_hi < a.n_rows ? p_hi : a.n_rows - 1;
    const int lo = a.window && p_lo >= a.window ? p_lo - a.window + 1 : 0;
    s.first = lo / STEP;
    const int sinks = (int)(((uint32_t)a.n_sink + STEP - 1) / STEP);
    s.sinks = sinks < s.first ? sinks : s.first;
    int to = last < 0 ? 0 : last / STEP + 1;
    // (a window behind the rows that there are: sinks alone)
    if (s.sinks > to) s.sinks = to;
    s.steps = s.sinks + (to > s.first ? to - s.first : 0);
    return s;
}

// A page's id, or -1 where the table names none that there is.
__device__ __forceinline__ int dc_page_id(const DcPages &p, const int32_t *table, int index) {
    const int id = dc_step_word(table + index);
    return (unsigned)id < (unsigned)p.n_pages ? id : -1;
}

int dc_paged_chunk_launch(const DcPagedAttn &a, int hd, int n_units, hipStream_t st);
// Parts that a chunk's blocks are cut into.
int dc_paged_chunk_splits(int64_t n_units, int64_t tiles, int hd, int64_t rows);
constexpr int kChunkRows = 128;

typedef __bf16 dc_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 dc_bf16x8 __attribute__((ext_vector_type(8)));
typedef float dc_f32x4 __attribute__((ext_vector_type(4)));
typedef float dc_f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t dc_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t dc_u32x2 __attribute__((ext_vector_type(2)));

// A head's maximum before any logit passed it: finite, so that a logit of -inf has the weight 0 then too, where -inf - -inf
// would be NaN.  -inf stands for no rows.
constexpr float kNoLogit = -3.402823466e+38f;

__device__ __forceinline__ uint32_t dc_pack_bf16(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, dc_bf16x2{(__bf16)lo, (__bf16)hi});
}

// f over the two lanes whose numbers differ by 32, in both
template <typename F>
__device__ __forceinline__ float dc_over32(float x, F f) {
    const uint32_t u = __float_as_uint(x);
    const dc_u32x2 r = __builtin_bit_cast(dc_u32x2, __builtin_amdgcn_permlane32_swap(u, u, false, false));
    return f(__uint_as_float(r.x), __uint_as_float(r.y));
}
// f over the four lanes whose numbers are the same modulo 16, in every one of them
template <typename F>
__device__ __forceinline__ float dc_over16(float x, F f) {
    const uint32_t u = __float_as_uint(x);
    const dc_u32x2 r = __builtin_bit_cast(dc_u32x2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    return dc_over32(f(__uint_as_float(r.x), __uint_as_float(r.y)), f);
}

// Rows that some of a step's pairs attend to and others do not are multiplied by 0 for those: where V is not finite the product would be
// NaN.  A step that is not attended to as a whole is looked over for such numbers; where there are any, the product takes zeros in their
// places, and they are added to the outputs of the pairs that attend to them afterwards, as they are.
typedef unsigned short dc_u16x2 __attribute__((ext_vector_type(2)));
struct DcUnbounded {
    dc_u16x2 most = {0, 0};
    __device__ __forceinline__ void look(uint32_t w) {
        most = __builtin_elementwise_max(most, __builtin_bit_cast(dc_u16x2, w & 0x7f807f80u));
    }
    __device__ __forceinline__ bool any() const { return __any(most.x == 0x7f80 || most.y == 0x7f80); }
};
__device__ __forceinline__ uint32_t dc_finite(uint32_t w) {  // 0 in the halves that are not
    const uint32_t lo = (w & 0x7f80u) == 0x7f80u ? 0u : 0xffffu, hi = (w & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u;
    return w & (lo | hi);
}
__device__ __forceinline__ float dc_only_unbounded(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? x : 0.f; }
