// What the kernels of the paged cache share (paged.hip, paged_attn.hip, paged_chunk.hip): where a sequence's rows and its new tokens lie.
#pragma once
#include "dc_common.h"
#include <type_traits>

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
// word(p): the number at p, which no block changes
template <typename F>
__device__ __forceinline__ DcSpan dc_span_by(const DcNew &t, int b, F word) {
    DcSpan s;
    if (t.cu) {  // (whatever cu holds, no token lies outside the tensors)
        s.first = dc_clamp(word(t.cu + b), 0, t.n_tokens);
        s.count = dc_clamp(word(t.cu + b + 1), s.first, t.n_tokens) - s.first;
        s.count = s.count < t.max_new ? s.count : t.max_new;
    } else {
        s.first = b * t.max_new;
        s.count = t.counts ? dc_clamp(word(t.counts + b), 0, t.max_new) : t.max_new;
    }
    s.start = t.start ? dc_clamp(word(t.start + b), 0, kMostRows) : 0;
    return s;
}
__device__ __forceinline__ DcSpan dc_span(const DcNew &t, int b) {  // the same b in the whole wave
    return dc_span_by(t, b, [](const int32_t *p) { return dc_step_word(p); });
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
    int n_b, waves;          // waves of a block (paged_attn.hip)
    int tiles, tile_rows;    // of a unit's (token, head) pairs: at most so many tiles of so many
    int at_once, round;      // blocks that the GPU runs at once, and those of a KV head among them; at_once 0: nothing is dealt out
    int least, fewest;       // steps of a part, at least; down to the fewest as long as there is no more than one block to a CU
    int places;              // the cut tiles' parts that there is room for
    float of_all;            // 1.0001 / at_once: a little more steps to a part than come of the division, so that rounding makes no more of them
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

// ---- how the steps are dealt out ------------------------------------------------------------------------------------
//
// Sequences differ in length, and the host does not know by how much: with as many blocks to each, the longest one's end last (8 x 131072
// rows of 8 heads x 128 attended to by one token 625 us; one such sequence and seven of 8192 would take as long).  So the blocks count the steps of all
// sequences themselves, divide them by the blocks that run at once, and cut every tile of a sequence's pairs by that: to the nearest number of parts, or
// rounded up with a share so large that all items run at once, if up to a fifth more does for that; or else, of tiles, that they run in two rounds.
// Of more tiles than run at once, none much longer than a share, whole rounds stay uncut, and the rest is cut for one round more.
// To the nearest alone a last few blocks often run by themselves (up to 512 tokens of 4 sequences of up to 32601 rows, 8 heads x 128: 528 items
// for 512 places took 712 us, 984 take 508; 1021 tokens of 5 sequences, 4 heads x 64: 319 and 262; a token of 7 sequences of 32601 rows 176
// and 154).  Block x of the grid takes item x / n_h of KV head x % n_h; the items are those of sequence 0, then those of sequence 1, ...; a sequence
// has for each of its tiles the parts of its last one, which has the most steps (others may leave some of them empty).  A part's results stand in
// the workspace at the item's own place; a tile of one part goes to the outputs at once.
//
// Rounded to the nearest, a part has at least half of steps / at_once steps or is a tile's only one, and a sequence's tiles have at most twice the steps
// that the mean of its first and last suggests: there are never more items than 2 at_once / n_h and one for each tile (at_once / n_h and one for each
// sequence where those have one tile); rounded up, the items are counted first.
struct DcItem {
    int b, tile, part, parts;  // parts of this tile; 0: nothing to do
    int64_t slot;              // of part 0; the next part is n_h slots on
};

// the sum over the wave's lanes up to each lane's own
template <typename T>
__device__ __forceinline__ T dc_lane_sums(T x) {
    auto moved = [](T v, auto ctrl, auto rows) __attribute__((always_inline)) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
    };
    using std::integral_constant;
    const integral_constant<int, 0xf> all;
    x += moved(x, integral_constant<int, 0x111>{}, all);                               // row_shr:1
    x += moved(x, integral_constant<int, 0x112>{}, all);                               // row_shr:2
    x += moved(x, integral_constant<int, 0x114>{}, all);                               // row_shr:4
    x += moved(x, integral_constant<int, 0x118>{}, all);                               // row_shr:8
    x += moved(x, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});     // row_bcast:15
    x += moved(x, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});     // row_bcast:31
    return x;
}
template <typename T>
__device__ __forceinline__ T dc_of_lane(T x, int lane) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}

struct DcTiles {
    int tiles, first, last;  // of a sequence: how many, and the steps of the first and of the last
};
// TILED: a sequence's pairs may be several tiles
template <int STEP, bool TILED>
__device__ __forceinline__ DcTiles dc_tiles_of(const DcPagedAttn &a, const DcSpan &s) {
    if (s.count == 0) return {0, 0, 0};
    if constexpr (!TILED) {
        const int steps = dc_steps<STEP>(a, s.start, s.start + s.count - 1).steps;
        return {1, steps, steps};
    }
    const int pairs = s.count * a.group, tiles = (int)((unsigned)(pairs + a.tile_rows - 1) / (unsigned)a.tile_rows);
    const int hi = (int)((unsigned)((a.tile_rows < pairs ? a.tile_rows : pairs) - 1) / (unsigned)a.group), lo = (int)((unsigned)((tiles - 1) * a.tile_rows) / (unsigned)a.group);
    return {tiles, dc_steps<STEP>(a, s.start, s.start + hi).steps, dc_steps<STEP>(a, s.start + lo, s.start + s.count - 1).steps};
}
// A tile's parts: its steps times by (1 / those of a part), up added and the fraction dropped, 1 at least.  (In fp32: what it loses, 1e-7 of the
// number, is little beside the 1e-4 below.)
struct DcParts {
    float by, up;
    int most;
    __device__ __forceinline__ int of(int steps) const {
        const int n = (int)fmaf((float)steps, by, up);
        return n <= 1 ? 1 : n < most ? n : most;
    }
};

// Item x, or with OF_SEQUENCE the first one of sequence x (x is the same in the whole wave, all of whose lanes are here).
template <int STEP, bool TILED, bool OF_SEQUENCE = false>
__device__ __forceinline__ DcItem dc_deal(const DcPagedAttn &a, int x, int lane) {
    DcItem d = {0, 0, 0, 0, 0};
    DcParts cut = {0.f, 0.5f, INT32_MAX};
    int whole = 0;  // so many tiles, from the first sequence's last tile on, are not cut
    // x is item `in` of sequence b, whose first is at; `uncut` of its tiles are, and its last tile would have `most` parts
    auto found = [&](const DcSpan &s, int b, int at, int in, int tiles, int uncut, int most) __attribute__((always_inline)) {
        d.b = b;
        if constexpr (TILED) {
            // (late tokens first: they have the most rows)
            if (in < uncut) {
                d.tile = tiles - 1 - in, d.parts = 1;
                return;
            }
            const unsigned of_cut = (unsigned)(in - uncut);
            d.tile = tiles - uncut - 1 - (int)(of_cut / (unsigned)most), d.part = (int)(of_cut % (unsigned)most);
            const int pairs = s.count * a.group, lo = d.tile * a.tile_rows, hi = (lo + a.tile_rows < pairs ? lo + a.tile_rows : pairs) - 1;
            const int own = cut.of(dc_steps<STEP>(a, s.start + (int)((unsigned)lo / (unsigned)a.group), s.start + (int)((unsigned)hi / (unsigned)a.group)).steps);
            d.parts = own < most ? own : most;
        } else {
            d.part = in, d.parts = most;
        }
        const int first = at + in - d.part - whole;  // (places of uncut tiles are not kept)
        if (first + most > a.places) d.parts = 1;    // (never, but for numbers of tokens that say more than there are)
        d.slot = (int64_t)first * a.n_h;
    };
    // How the tiles are cut, for the work of all sequences.
    auto plan = [&](float work, auto &&each) __attribute__((always_inline)) {
        const float even = work * (float)a.n_h * a.of_all;  // (of_all is 1.0001 / at_once)
        const float least = fminf(fmaxf(even * (float)a.at_once * (1.f / 256), (float)a.fewest), (float)a.least);
        cut.by = __builtin_amdgcn_rcpf(even > least ? even : least);
        // (a part's least steps are what counts, or so many sequences that it all evens out and counting takes longer than it saves: 60 of one
        // tile 697 us and 706)
        if (!(even > least) || a.n_b > (TILED ? 64 : 16)) return;
        // Each lane counts the items of a share of its own: lanes 0 .. 31 one part's work for each block that runs at once and up to a fifth
        // more, the others half of it and up to all of it.
        const float base = lane < 32 ? even : fmaxf(0.5f * even, least), rise = lane < 32 ? 0.2f / 32 : 1.f / 32;
        const DcParts mine = {__builtin_amdgcn_rcpf(fmaf(base * rise, (float)(lane & 31), base)), 0.999f, INT32_MAX};
        float n = 0.f, all = 0.f, longest = 0.f;
        each([&](float tiles, float last) __attribute__((always_inline)) {
            n = fmaf(tiles, fmaxf(floorf(fmaf(last, mine.by, mine.up)), 1.f), n);
            if constexpr (TILED) all += tiles, longest = fmaxf(longest, last);
        });
        if constexpr (TILED) {
            const int tiles = (int)dc_of_lane(all, 0), over = tiles * a.n_h - a.at_once;
            if (over > 0 && dc_of_lane(longest, 0) <= 1.3f * even) {
                // whole rounds, and what is left cut for one more
                const unsigned left = (unsigned)tiles % (unsigned)a.round;
                const int parts = left ? (int)((unsigned)a.round / left) : 1;
                if (parts > 1) whole = tiles - (int)left, cut = {__builtin_amdgcn_rcpf(least), 0.f, parts};
                else whole = INT32_MAX;
                return;
            }
            if (over > a.at_once) {
                whole = INT32_MAX;
                return;
            }
        }
        const uint64_t fits = __ballot(n * (float)a.n_h <= (float)(lane < 32 ? a.at_once : TILED ? 2 * a.at_once : 0));
        if (!fits) return;
        const int k = __builtin_ctzll(fits);  // (the least share that does)
        cut = {dc_of_lane(mine.by, k), 0.999f, INT32_MAX};
        // (two rounds that are not shorter than the longest tile)
        if constexpr (TILED)
            if (k >= 32 && dc_of_lane(longest, 0) * cut.by < 2.1f) whole = INT32_MAX;
    };
    if (a.n_b == 1) {
        const DcSpan s = dc_span(a.t, 0);
        const DcTiles t = dc_tiles_of<STEP, TILED>(a, s);
        plan(0.5f * (float)t.tiles * (float)(t.first + t.last), [&](auto &&f) { f((float)t.tiles, (float)t.last); });
        const int most = cut.of(t.last), uncut = whole < t.tiles ? whole : t.tiles;
        if (x < uncut + (t.tiles - uncut) * most) found(s, 0, 0, x, t.tiles, uncut, most);
        return d;
    }
    auto tiles_of = [&](int b) __attribute__((always_inline)) {
        if (b >= a.n_b) return DcTiles{0, 0, 0};
        return dc_tiles_of<STEP, TILED>(a, dc_span_by(a.t, b, [](const int32_t *p) { return *p; }));
    };
    const DcTiles mine = tiles_of(lane);  // of sequence lane; those from 64 on are read again when it is their turn
    float work = 0.f;
    for (int b0 = 0; b0 < a.n_b; b0 += 64) {
        const DcTiles t = b0 == 0 ? mine : tiles_of(b0 + lane);
        work += dc_of_lane(dc_lane_sums(0.5f * (float)t.tiles * (float)(t.first + t.last)), 63);
    }
    const float tiles_f = (float)mine.tiles, last_f = (float)mine.last;
    plan(work, [&](auto &&f) {
#pragma unroll 4
        for (int b = 0; b < a.n_b; ++b) f(dc_of_lane(tiles_f, b), dc_of_lane(last_f, b));
    });
    int base = 0;
    for (int b0 = 0; b0 < a.n_b; b0 += 64) {
        const DcTiles t = b0 == 0 ? mine : tiles_of(b0 + lane);
        const int parts = cut.of(t.last);
        int uncut = whole == 0 ? 0 : t.tiles;
        if (TILED && whole > 0 && whole < INT32_MAX) {  // (of 64 sequences at most)
            uncut = whole - (dc_lane_sums(t.tiles) - t.tiles);
            uncut = uncut < 0 ? 0 : uncut < t.tiles ? uncut : t.tiles;
        }
        const int items = uncut + (t.tiles - uncut) * parts, upto = dc_lane_sums(items);
        const uint64_t past = OF_SEQUENCE ? (x < b0 + 64 ? 1ull << (x - b0) : 0) : __ballot(base + upto > x);
        if (past) {
            const int k = __builtin_ctzll(past), at = base + dc_of_lane(upto, k) - dc_of_lane(items, k);  // the sequence's first item
            const int tiles = dc_of_lane(t.tiles, k);
            if (tiles) found(dc_span(a.t, b0 + k), b0 + k, at, OF_SEQUENCE ? 0 : x - at, tiles, dc_of_lane(uncut, k), dc_of_lane(parts, k));
            return d;
        }
        base += dc_of_lane(upto, 63);
    }
    return d;
}

// Packed tokens of which no tile is cut: block x / n_h is place x of the tiles' places, of which sequence b has those from
// floor(cu[b] group / tile_rows) + b on, as many as its tiles or one more.  The sequence is found 64 at a time.
__device__ __forceinline__ DcItem dc_packed(const DcPagedAttn &a, int x, int lane) {
    auto place = [&](int b) __attribute__((always_inline)) {
        return (int)((unsigned)(dc_clamp(a.t.cu[b], 0, a.t.n_tokens) * a.group) / (unsigned)a.tile_rows) + b;
    };
    int lo = 0, n = a.n_b;  // the last sequence of [lo, lo + n) whose place is not past x
    while (n > 1) {
        const int step = (n + 63) / 64, b = lo + lane * step;
        const int k = __popcll(__ballot(lane * step < n && place(b) <= x));  // (they do not decrease, so these are the first k lanes)
        const int at = k > 1 ? (k - 1) * step : 0;
        lo += at, n = n - at < step ? n - at : step;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const DcSpan s = dc_span(a.t, lo);
    const int tiles = (int)((unsigned)(s.count * a.group + a.tile_rows - 1) / (unsigned)a.tile_rows), in = x - __builtin_amdgcn_readfirstlane(place(lo));
    if (in < 0 || in >= tiles) return {0, 0, 0, 0, 0};
    return {lo, tiles - 1 - in, 0, 1, 0};
}

// A page's id, or -1 where the table names none that there is.
__device__ __forceinline__ int dc_page_id(const DcPages &p, const int32_t *table, int index) {
    const int id = dc_step_word(table + index);
    return (unsigned)id < (unsigned)p.n_pages ? id : -1;
}

// paged_chunk.hip; join: 0, or the y of the join's grid
int dc_paged_chunk_launch(const DcPagedAttn &a, int hd, unsigned blocks, unsigned join, hipStream_t st);
// Rows of a step; blocks that run at once.
constexpr int dc_chunk_step(int hd) { return hd == 256 ? 32 : 64; }
constexpr int dc_chunk_at_once(int hd) { return hd == 64 ? 1024 : hd == 128 ? 512 : 512; }
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

// x - y of x as it was rounded: a product that the compiler takes into the subtraction would not be, and the largest logit's weight not 1
__device__ __forceinline__ float dc_less(float x, float y) {
    asm("" : "+v"(x));
    return x - y;
}

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

// ---- joining parts --------------------------------------------------------------------------------------------------
__device__ __forceinline__ float dc_weight(float m, float top) { return m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 0.f; }
// a part's share of the sum (one that is no number stays none, whatever its maximum)
__device__ __forceinline__ float dc_share(float m, float l, float top) { return l == l ? dc_weight(m, top) * l : l; }
__device__ __forceinline__ float dc_log_sum(float top, float total) { return total == 0.f ? -INFINITY : (top + log2f(total)) * 0.693147180559945309f; }
