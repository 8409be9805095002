// What the bfloat16 attention kernels over the paged cache share (attention_mfma.hip, attention_weighed_mfma.hip): tiles of 32 keys as
// operands of the matrix cores, the softmax down a column of queries, and how a sequence's tiles are dealt to splits and merged.
// attention_mfma.hip describes the layout.  Compiled once per head size: -DSIA_HEAD_DIM=<multiple of 16, up to 256>.
#pragma once

#include "common.h"

#ifndef SIA_HEAD_DIM
#error "compile with -DSIA_HEAD_DIM=<head size>"
#endif

#ifndef SIA_SCORE_FORMS
#define SIA_SCORE_FORMS 0
#endif
constexpr bool FORMS = SIA_SCORE_FORMS != 0;
constexpr int HD = SIA_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16 up to 256");
constexpr int KSTEPS = (HD + 31) / 32;
constexpr int DBLOCKS = HD / 16;
constexpr int TILE = 32;

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4;

__device__ __forceinline__ bf16x8 load8(const bf16_t* p) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(p));
}
__device__ __forceinline__ bf16x8 zero8() {
    return __builtin_bit_cast(bf16x8, make_uint4(0u, 0u, 0u, 0u));
}
// Two floats to two bfloat16 (round to nearest even) with the hardware's packed conversion.
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float floatx2;
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const floatx2 f = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}
// 2^x by the hardware instruction; arguments here are <= 0 or -inf, results in [0, 1].
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float LOG2E = 1.4426950408889634f;

// The oldest key a query at `pos` sees: all (window = chunk = 0), the last `window`, and/or those of its own block
// of `chunk` absolute positions [b * chunk, (b + 1) * chunk).  It never falls as pos grows.
__device__ __forceinline__ int first_visible(int pos, int window, int chunk) {
    int lo = window > 0 ? max(0, pos - window + 1) : 0;
    if (chunk > 0) lo = max(lo, pos - pos % chunk);
    return lo;
}

// What the two forms add to a kernel's arguments.
struct Forms {
    float rate;       // scale / cap, or 0: no cap
    int keep_first;
};

// Places: place x is position x for x < edge and position x + gap beyond.
struct Places {
    int edge, gap;
};

// lo: the oldest position of the window (of the first query of a workgroup).
__device__ __forceinline__ Places places_of(int lo, int keep_first, int ps_log2) {
    if (!FORMS || keep_first <= 0) return Places{0, 0};
    const int unit = max(1 << ps_log2, TILE);     // both powers of two
    const int edge = (keep_first + unit - 1) & -unit;
    return Places{edge, max(0, (lo & -unit) - edge)};
}

// The first place of the walk that serves a window from place lo on.
__device__ __forceinline__ int walk_begin(int lo, int keep_first) { return FORMS && keep_first > 0 ? 0 : lo; }

// A capped score: tanh of the dot product times `rate` (the cap itself and the change to units of log2 are in the
// softmax's scale).  tanh(x) = 1 - 2 / (e^(2x) + 1), whose absolute error is that of a rounding near 1.
__device__ __forceinline__ float capped(float s, float rate) {
    const float e = __builtin_amdgcn_exp2f(s * rate * (2.f * 1.4426950408889634f));
    return 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
}

// A sink's term of a softmax denominator: sinks[head] is a learned logit of that query head (natural units; the
// score scale does not apply) that takes a share of the weight and carries no value.  Exponentials are taken as 2^(x - ref) with ref in units of log2.
__device__ __forceinline__ float sink_term(const float* __restrict__ sinks, int head, float ref) {
    return sinks ? fast_exp2(sinks[head] * LOG2E - ref) : 0.f;
}

// Maximum and sum over the four lanes r, r+16, r+32, r+48 that share a q column, for every lane, by the
// register swaps between the wave's rows of 16 lanes (no trip through LDS as a general lane shuffle makes):
// v_permlane16_swap exchanges rows 1, 3 of its first operand with rows 0, 2 of its second, v_permlane32_swap
// the upper half of the first with the lower half of the second; either way the two results hold, lane by
// lane, the two values to combine.  The sum is (row 0 + row 1) + (row 2 + row 3) in every lane.
__device__ __forceinline__ float column_max(float v) {
    uint32_t u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    u = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float v) {
    uint32_t u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    u = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 64 consecutive entries of a sequence's block table, one per lane.
struct PageWindow {
    int base;  // index (among the pages of places) of the entry that lane 0 holds
    int mine;
};

__device__ __forceinline__ void pages_load(PageWindow& w, const int* __restrict__ table, int table_width,
                                           int first, int lane, int ps_log2, const Places& places) {
    w.base = first;
    int index = first + lane;
    if (FORMS && index >= places.edge >> ps_log2) index += places.gap >> ps_log2;
    w.mine = table[min(index, table_width - 1)];
}

__device__ __forceinline__ int pages_get(const PageWindow& w, int index) {
    return max(__shfl(w.mine, index - w.base, SIA_WAVE), 0);
}

// Keys and values of one tile of 32 positions, as MFMA operands.
struct Stage {
    bf16x8 k[2][KSTEPS];
    bf16x8 v[DBLOCKS];
};

// Loads the tile at absolute position kb.  [load_lo, load_hi] is the wave-uniform range of keys whose
// pages exist; it must meet the tile.  Addresses of keys outside it are clamped into it, so every
// load is unconditional; what a clamped load brings is masked (scores) or multiplied by a zero
// probability (values).  The pages only ever hold finite numbers.
__device__ __forceinline__ void load_stage(Stage& st, const bf16_t* __restrict__ kp, const bf16_t* __restrict__ vp,
                                           const PageWindow& pages, int ps_log2, int n_kv, int hk, int kb,
                                           int load_lo, int load_hi) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int ps = 1 << ps_log2;
    const int t_lo = max(kb, load_lo), t_hi = min(kb + TILE - 1, load_hi);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int key = min(max(kb + (r >> 2) * 8 + h * 4 + (r & 3), t_lo), t_hi);
        const int page = pages_get(pages, key >> ps_log2);
        const bf16_t* row = kp + (((size_t)page * n_kv + hk) * ps + (key & (ps - 1))) * HD;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
            const int d0 = ks * 32 + g * 8;
            if (HD % 32 == 0 || ks < KSTEPS - 1)
                st.k[h][ks] = load8(row + d0);
            else
                st.k[h][ks] = d0 < HD ? load8(row + d0) : zero8();
        }
    }
    const int key0 = min(max(kb + g * 8, t_lo & ~7), t_hi & ~7);
    const int page = pages_get(pages, key0 >> ps_log2);
    const bf16_t* vbase = vp + ((size_t)page * n_kv + hk) * HD * ps + (key0 & (ps - 1));
#pragma unroll
    for (int db = 0; db < DBLOCKS; ++db) st.v[db] = load8(vbase + (size_t)(db * 16 + r) * ps);
}

// What a wave keeps of the softmax of its q columns, per group n of 16 columns.  A column (one query) lives in the
// four lanes r, r + 16, r + 32, r + 48, each of which sees 8 of a tile's 32 keys.
//   m:   the column's *reference*, in units of log2: exponentials are taken as 2^(s * scale_log2 - m).  It follows
//        the running maximum lazily: it moves up to the maximum only when the maximum has grown more than
//        SOFTMAX_SLACK beyond it.  Exponentials are then at most 2^SOFTMAX_SLACK instead of 1, which float sums and
//        bfloat16 probabilities hold just as well, and (m, l, acc) stay a consistent triple, so acc / l is the
//        same value.  The same in all four lanes of a column.
//   mu:  m, or 0 while the column has seen no key (m = -inf).
//   l:   this lane's part of the sum of exponentials (its 8 keys of every tile); the four lanes' parts are added
//        once, at the end (finish_sums).
// The point of the lazy reference: a tile on which no column's reference moves (nearly all of them) costs no
// exchange between lanes and no rescaling of the accumulators (4 * DBLOCKS registers a column group), only a
// maximum, a multiply-add and an exponential per score.  Whether a column's reference moves depends on that
// column's scores alone, never on its neighbours in the wave.
constexpr float SOFTMAX_SLACK = 8.f;

template <int NQ>
struct Softmax {
    float m[NQ], mu[NQ], l[NQ];
    __device__ __forceinline__ void start() {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n] = -INFINITY;
            mu[n] = 0.f;
            l[n] = 0.f;
        }
    }
    // after the last tile: l becomes the column's whole sum, in every lane
    __device__ __forceinline__ void finish_sums() {
#pragma unroll
        for (int n = 0; n < NQ; ++n) l[n] = column_sum(l[n]);
    }
};

// max without the quieting of signalling NaNs that fmaxf owes the standard (scores are never NaN)
__device__ __forceinline__ float max2(float a, float b) { return __builtin_fmaxf(a, b); }

// Masks the scores of a tile, updates the softmax state of each q column, rescales the accumulators where a
// reference moved, and returns the tile's probabilities as the P^T operand.
//   lo[n], hi[n]: visible keys of this lane's column in group n (hi < lo: none); those below forms.keep_first are visible
//   up to hi[n] too.
//   scale_log2 = scale * log2(e) > 0.
// A tile that every column of the wave sees whole skips the masking (the test is wave-uniform).
template <int NQ>
__device__ __forceinline__ void softmax_update(floatx4 (&s)[NQ][2], int kb, const int (&lo)[NQ], const int (&hi)[NQ],
                                               float scale_log2, Softmax<NQ>& sm, floatx4 (&acc)[NQ][DBLOCKS],
                                               bf16x8 (&p)[NQ], const Forms& forms) {
    const int g = (threadIdx.x & 63) >> 4;
    float top[NQ];
    bool grew = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        if (FORMS && forms.rate > 0.f) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][h][i] = capped(s[n][h][i], forms.rate);
        }
        if (!__all((kb >= lo[n] || (FORMS && kb + TILE <= forms.keep_first)) && kb + TILE - 1 <= hi[n])) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = kb + g * 8 + h * 4 + i;
                    if ((key < lo[n] && !(FORMS && key < forms.keep_first)) || key > hi[n]) s[n][h][i] = -INFINITY;
                }
        }
        top[n] = max2(max2(max2(s[n][0][0], s[n][0][1]), max2(s[n][0][2], s[n][0][3])),
                      max2(max2(s[n][1][0], s[n][1][1]), max2(s[n][1][2], s[n][1][3]))) * scale_log2;
        grew |= top[n] > sm.m[n] + SOFTMAX_SLACK;   // also a column's first visible key (m = -inf)
    }
    if (__builtin_expect(__any(grew), 0)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float mx = column_max(top[n]);
            const bool moved = mx > sm.m[n] + SOFTMAX_SLACK;
            const float alpha = moved ? fast_exp2(sm.m[n] - mx) : 1.f;   // from -inf: 0 (there is nothing yet)
            sm.m[n] = moved ? mx : sm.m[n];
            sm.mu[n] = sm.m[n] == -INFINITY ? 0.f : sm.m[n];
            sm.l[n] *= alpha;
#pragma unroll
            for (int db = 0; db < DBLOCKS; ++db) acc[n][db] *= alpha;
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        float sum = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = fast_exp2(fmaf(s[n][h][i], scale_log2, -sm.mu[n]));
                s[n][h][i] = e;
                sum += e;
            }
        sm.l[n] += sum;
        uint4 u;
        u.x = pack2(s[n][0][0], s[n][0][1]);
        u.y = pack2(s[n][0][2], s[n][0][3]);
        u.z = pack2(s[n][1][0], s[n][1][1]);
        u.w = pack2(s[n][1][2], s[n][1][3]);
        p[n] = __builtin_bit_cast(bf16x8, u);
    }
}

// Scores, online softmax and value product of one tile held in registers.
template <int NQ>
__device__ __forceinline__ void compute_stage(const Stage& st, const bf16x8 (&q)[NQ][KSTEPS], int kb,
                                              const int (&lo)[NQ], const int (&hi)[NQ], float scale,
                                              Softmax<NQ>& sm, floatx4 (&acc)[NQ][DBLOCKS], const Forms& forms) {
    floatx4 s[NQ][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][h] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
                s[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(st.k[h][ks], q[n][ks], s[n][h], 0, 0, 0);
    }
    bf16x8 p[NQ];
    softmax_update<NQ>(s, kb, lo, hi, scale, sm, acc, p, forms);
#pragma unroll
    for (int db = 0; db < DBLOCKS; ++db)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
            acc[n][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(st.v[db], p[n], acc[n][db], 0, 0, 0);
}

// Of the 8 values of positions first .. first + 7, those beyond `last` as zeros: pages may hold anything there, and a weight of 0 times a number
// without bounds is none.
template <typename Words>      // four 32-bit words
__device__ __forceinline__ void clear_beyond(Words& u, int first, int last) {
    const int n = min(max(last - first + 1, 0), 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] &= n >= 2 * i + 2 ? 0xffffffffu : n == 2 * i + 1 ? 0x0000ffffu : 0u;
}
__device__ __forceinline__ void clear_values(Stage& st, int kb, int g, int last) {
    typedef uint32_t words __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int db = 0; db < DBLOCKS; ++db) {
        words u = __builtin_bit_cast(words, st.v[db]);
        clear_beyond(u, kb + 8 * g, last);
        st.v[db] = __builtin_bit_cast(bf16x8, u);
    }
}

// Called before a tile is computed; the default does nothing.
struct NoHook {
    __device__ __forceinline__ void operator()(int, Stage&) const {}
};
struct ClearBeyond {      // values beyond `last` as zeros
    int last, g;
    __device__ __forceinline__ void operator()(int kb, Stage& st) const {
        if (kb + TILE - 1 > last) clear_values(st, kb, g, last);
    }
};

// The tiles w_first, w_first + TILE, ..., w_last, whose block-table entries the window holds; two register
// stages in turn: the loads of tile t+1 are issued before the arithmetic of tile t.  `before(kb, stage)` runs before the
// arithmetic of the tile at kb (it may hand the state on and start it afresh).
template <int NQ, typename Hook>
__device__ __forceinline__ void attend_tiles(const PageWindow& pages, int w_first, int w_last,
                                             const bf16x8 (&q)[NQ][KSTEPS], const bf16_t* __restrict__ kp,
                                             const bf16_t* __restrict__ vp, int ps_log2, int n_kv, int hk,
                                             int range_lo, int range_hi, const int (&lo)[NQ], const int (&hi)[NQ],
                                             float scale, Softmax<NQ>& sm, floatx4 (&acc)[NQ][DBLOCKS], Hook& before,
                                             const Forms& forms) {
    Stage a, b;
    load_stage(a, kp, vp, pages, ps_log2, n_kv, hk, w_first, range_lo, range_hi);
    for (int kb = w_first; kb <= w_last; kb += 2 * TILE) {
        const int kb1 = min(kb + TILE, w_last);  // past the end: the last tile again, never computed
        load_stage(b, kp, vp, pages, ps_log2, n_kv, hk, kb1, range_lo, range_hi);
        before(kb, a);
        compute_stage<NQ>(a, q, kb, lo, hi, scale, sm, acc, forms);
        const int kb2 = min(kb + 2 * TILE, w_last);
        load_stage(a, kp, vp, pages, ps_log2, n_kv, hk, kb2, range_lo, range_hi);
        if (kb + TILE <= w_last) {
            before(kb + TILE, b);
            compute_stage<NQ>(b, q, kb + TILE, lo, hi, scale, sm, acc, forms);
        }
    }
}

// All tiles that meet [range_lo, range_hi] (range_lo <= range_hi).  The block-table window (64 entries,
// starting at the page of the first tile it serves) is loaded outside the pipelined loop, once per 64
// pages: a load inside it would make every iteration wait for all outstanding loads.
template <int NQ, typename Hook>
__device__ __forceinline__ void attend_range(const bf16x8 (&q)[NQ][KSTEPS], const bf16_t* __restrict__ kp,
                                             const bf16_t* __restrict__ vp, const int* __restrict__ table,
                                             int table_width, int ps_log2, int n_kv, int hk, int range_lo,
                                             int range_hi, const int (&lo)[NQ], const int (&hi)[NQ], float scale,
                                             Softmax<NQ>& sm, floatx4 (&acc)[NQ][DBLOCKS], Hook& before,
                                             const Forms& forms, const Places& places) {
    const int lane = threadIdx.x & 63;
    const int kb_first = (range_lo / TILE) * TILE, kb_last = (range_hi / TILE) * TILE;
    for (int w_first = kb_first; w_first <= kb_last;) {
        const int first_page = w_first >> ps_log2;
        const int w_end = (first_page + SIA_WAVE) << ps_log2;  // first key beyond the window, a multiple of TILE
        PageWindow pages;
        pages_load(pages, table, table_width, first_page, lane, ps_log2, places);
        attend_tiles<NQ>(pages, w_first, min(kb_last, w_end - TILE), q, kp, vp, ps_log2, n_kv, hk, range_lo, range_hi,
                         lo, hi, scale, sm, acc, before, forms);
        w_first = w_end;
    }
}

template <int NQ>
__device__ __forceinline__ void attend_range(const bf16x8 (&q)[NQ][KSTEPS], const bf16_t* __restrict__ kp,
                                             const bf16_t* __restrict__ vp, const int* __restrict__ table,
                                             int table_width, int ps_log2, int n_kv, int hk, int range_lo,
                                             int range_hi, const int (&lo)[NQ], const int (&hi)[NQ], float scale,
                                             Softmax<NQ>& sm, floatx4 (&acc)[NQ][DBLOCKS], const Forms& forms,
                                             const Places& places) {
    NoHook none;
    attend_range<NQ>(q, kp, vp, table, table_width, ps_log2, n_kv, hk, range_lo, range_hi, lo, hi, scale, sm, acc,
                     none, forms, places);
}

// q operand of column r: 8 dims d0 .. d0+7 of that column's query row (zeros if the column is unused).
__device__ __forceinline__ void load_q(bf16x8 (&q)[KSTEPS], const bf16_t* row, int g) {
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
        const int d0 = ks * 32 + g * 8;
        q[ks] = (row != nullptr && d0 < HD) ? load8(row + d0) : zero8();
    }
}

// ---------------------------------------------------------------------------------------------------
// decode: sequences with one new token each
// ---------------------------------------------------------------------------------------------------
constexpr int DEC_WAVES = 4;
constexpr int DEC_TILES_PER_SPLIT = 16;  // a split is worth taking from this many tiles (512 keys) on
constexpr int DEC_MAX_SPLITS = 32;
constexpr int DEC_FOLD_LDS = 128 * 1024;  // most LDS a workgroup that does all splits may take for their states

// Workgroups that share one (sequence, kv head) with n_tiles visible key tiles: the largest power of two that
// leaves every workgroup DEC_TILES_PER_SPLIT tiles, at most DEC_MAX_SPLITS.  A function of the sequence's own
// length only; host and device use the same one.
__host__ __device__ inline int decode_splits(int n_tiles) {
    int s = 1;
    while (s < DEC_MAX_SPLITS && 2 * s * DEC_TILES_PER_SPLIT <= n_tiles) s *= 2;
    return s;
}

// out = sum_s w_s acc_s / sum_s w_s l_s over the splits of one (sequence, head), with w_s = 2^(m_s - max m) (the
// maxima are kept in units of log2; a split without keys has m = -inf and weight 0).  One element: `at(s)` gives
// split s's (acc, m, l).  Summed in split order with fused multiply-adds, the same wherever it is called from.
// `beside` is what the denominator holds beside the keys (a sink's term, relative to mx; else 0).
template <typename At>
__device__ __forceinline__ float merge_splits(int n_splits, float mx, float beside, At at) {
    float o = 0.f, denom = beside;
    for (int s0 = 0; s0 < n_splits; s0 += 4) {  // four splits' loads in flight at a time
        float acc[4], m[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) at(min(s0 + j, n_splits - 1), acc[j], m[j], l[j]);  // past the end: the last again, weight 0
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float w = s0 + j < n_splits ? fast_exp2(m[j] - mx) : 0.f;
            denom = __builtin_fmaf(w, l[j], denom);
            o = __builtin_fmaf(w, acc[j], o);
        }
    }
    return o * (1.f / denom);
}

// The states of the four runs of one split, merged for one element of one query head: the split's (acc, m, l).
// `row(w)` is run w's state of that head: acc[HD], m, l.  The same arithmetic wherever it is called from.
template <typename Row>
__device__ __forceinline__ void merge_waves(Row row, int d, float& o, float& mx, float& lsum) {
    const float* rows[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) rows[w] = row(w);
    mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, rows[w][HD]);
    const float mx_use = (mx == -INFINITY) ? 0.f : mx;  // no run had a key: all weights 0, the split counts for nothing
    o = 0.f;
    lsum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float wgt = fast_exp2(rows[w][HD] - mx_use);  // a run without keys has m = -inf: weight 0
        o += wgt * rows[w][d];
        lsum += wgt * rows[w][HD + 1];
    }
}

// One wave's state, finished, into its row of LDS (lanes whose column is no query head of the group write nothing).
__device__ __forceinline__ void leave_state(float* mine, Softmax<1>& sm, const floatx4 (&acc)[1][DBLOCKS], int g,
                                            bool writes) {
    sm.finish_sums();
    if (!writes) return;
    if (g == 0) {
        mine[HD] = sm.m[0];
        mine[HD + 1] = sm.l[0];
    }
#pragma unroll
    for (int db = 0; db < DBLOCKS; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[db * 16 + g * 4 + i] = acc[0][db][i];
}

// The states of the first N splits, beyond `last` that one again.
template <int N>
__device__ __forceinline__ void load_states(int last, const float* __restrict__ acc_at, const float2* __restrict__ ml, float (&acc)[N],
                                            float2 (&state)[N]) {
#pragma unroll
    for (int s = 0; s < N; ++s) acc[s] = acc_at[(size_t)min(s, last) * HD];
#pragma unroll
    for (int s = 0; s < N; ++s) state[s] = ml[min(s, last)];
}

// merge_splits for one element of up to N splits, with its order of sums.  What is held of splits beyond n_splits may be anything.
template <int N>
__device__ __forceinline__ float combine_states(int n_splits, const float (&acc)[N], const float2 (&state)[N], const float* __restrict__ sinks,
                                                int head) {
    float mx = -INFINITY;
#pragma unroll
    for (int s = 0; s < N; ++s) mx = s < n_splits ? fmaxf(mx, state[s].x) : mx;
    float o = 0.f, denom = sink_term(sinks, head, mx);
#pragma unroll
    for (int s = 0; s < N; ++s) {
        const float w = fast_exp2(state[s].x - mx), d = __builtin_fmaf(w, state[s].y, denom), a = __builtin_fmaf(w, acc[s], o);
        denom = s < n_splits ? d : denom;
        o = s < n_splits ? a : o;
    }
    return o * (1.f / denom);
}
template <int N>
__device__ __forceinline__ float combine_all(int n_splits, const float* __restrict__ acc_at, const float2* __restrict__ ml,
                                             const float* __restrict__ sinks, int head) {
    float acc[N];
    float2 state[N];
    load_states(n_splits - 1, acc_at, ml, acc, state);
    return combine_states(n_splits, acc, state, sinks, head);
}
