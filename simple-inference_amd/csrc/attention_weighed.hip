// How much attention weight every cached key got in a step, added to a running sum per (sequence, key/value head, place):
//
//   weights[slot][g][j]  +=  sum over the sequence's tokens t and the query heads h of g of  p[t, h, j]
//   p[t, h, j] = exp(scale q[t, h] . k[j] - lse[t, h])   for j <= the token's place, else 0
//
// The attention that made the output leaves lse (m + log(l) of its softmax, in units of log2: `row_stats`), so that no second pass over
// the values is needed, only the scores again.  A place that the step itself has written begins at zero, whatever lay there.
// All sums are float and have a fixed order, without atomics: over the rows of a chunk in a lane (of every 16th row, and then over 16 lanes, on the
// matrix cores), then over the chunks of a block of keys by a kernel of their own.
//
// Heads of up to 256 in fours go by the float matrix cores (weigh_float_kernel), with keys as rows and queries as columns, single tokens and
// runs alike; bfloat16 heads that the attention kernels take on the bfloat16 matrix cores by attention_weighed_mfma.hip.
// The plain kernel: a wave for 64 consecutive places of one (sequence, key/value head), a lane a key; the queries come one after
// the other through LDS.  It takes every head size, page size and type.
#include "f32_lanes.h"
#include "weighed.h"

#define WEIGH_MAX_HEAD_DIM 640

template <typename T>
__global__ __launch_bounds__(SIA_WAVE) void weigh_plain_kernel(
    const T* __restrict__ q, int q_row_stride, const T* __restrict__ k_pages, const int* __restrict__ block_table, int table_width,
    const int* __restrict__ cu_q, const int* __restrict__ kv_len, const float* __restrict__ row_stats, int n_heads, int n_kv, int head_dim,
    int page_size, int n_pages, float scale, const Weighed w) {
    __shared__ float q_s[WEIGH_MAX_HEAD_DIM];
    const int lane = threadIdx.x, hk = blockIdx.y, seq = blockIdx.z, group = n_heads / n_kv;
    const int first = cu_q[seq], n = cu_q[seq + 1] - first, length = min(kv_len[seq], w.places), start = length - n;
    const int j0 = blockIdx.x * SIA_WAVE, j = j0 + lane;
    float* row = weight_row(w, seq, n_kv, hk);
    if (j0 >= length || !row) return;
    int page = j < length && j / page_size < table_width ? block_table[(size_t)seq * table_width + j / page_size] : -1;
    if (page >= n_pages) page = -1;
    const T* key = k_pages + (((size_t)max(page, 0) * n_kv + hk) * page_size + j % page_size) * head_dim;
    float total = 0.f, sum = 0.f;      // of tokens, and of 64 of them: a long run's small weights are not added one by one to a large sum
    for (int t = max(0, j0 - start); t < n; ++t) {
        for (int h = hk * group; h < (hk + 1) * group; ++h) {
            const T* q_row = q + (size_t)(first + t) * q_row_stride + h * head_dim;
            for (int d = lane; d < head_dim; d += SIA_WAVE) q_s[d] = to_float(q_row[d]);
            __syncthreads();
            float dot = 0.f;
            if (page >= 0)
                for (int d = 0; d < head_dim; ++d) dot = fmaf(q_s[d], to_float(key[d]), dot);
            const float p = exp2f(fmaf(dot * scale, 1.4426950408889634f, -row_stats[(size_t)(first + t) * n_heads + h]));
            sum += page >= 0 && j <= start + t ? p : 0.f;
            __syncthreads();
        }
        if (t % 64 == 63 || t == n - 1) {
            total += sum;
            sum = 0.f;
        }
    }
    if (j < length) row[j] = (j < start ? row[j] : 0.f) + total;
}

template <typename T>
static int weigh_plain(const T* q, int q_row_stride, const T* k_pages, const int* block_table, int table_width, const int* cu_q, const int* kv_len,
                       const float* row_stats, int n_seqs, int max_kv, int n_heads, int n_kv, int head_dim, int page_size, int n_pages, float scale,
                       const Weighed& w, hipStream_t stream) {
    hipLaunchKernelGGL(weigh_plain_kernel<T>, dim3((max_kv + SIA_WAVE - 1) / SIA_WAVE, n_kv, n_seqs), dim3(SIA_WAVE), 0, stream, q, q_row_stride,
                       k_pages, block_table, table_width, cu_q, kv_len, row_stats, n_heads, n_kv, head_dim, page_size, n_pages, scale, w);
    return SIA_LAUNCH_CHECK();
}

// ---------------------------------------------------------------------------------------------------
// heads of up to 256 on the float matrix cores (v_mfma_f32_16x16x4_f32)
// ---------------------------------------------------------------------------------------------------
// A dot product's elements come in the attention kernels' order, so that a score has the bits that went into its row's statistic: what is
// left of a weight's error is that of two exponentials and a sum.  (In the order in which a lane loads them, without the exchange between
// lanes, errors of 8e-7 of the sums where 2e-7 are now.)
constexpr int F32_WAVES = 4;
// Blocks of 16 keys of a wave, and keys of a workgroup: what the registers hold.
constexpr int f32_blocks(int dp) { return dp <= 128 ? 2 : 1; }
constexpr int f32_keys(int dp) { return F32_WAVES * 16 * f32_blocks(dp); }

__device__ __forceinline__ f32x4 load4(const float* p) { return *(const f32x4*)p; }
__device__ __forceinline__ f32x4 load4(const bf16_t* p) {
    const uint2 u = *(const uint2*)p;
    return f32x4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
}

// What bounds it at a few hundred tokens is the chain of loads before the first product; then the float products (157 TFLOP/s).  Three tokens over 200
// and a prompt of 300, 32 heads of 64 on 8: 10.8 us beside an attention of 18.6 and a sum of the chunks of 2.5 to 4.0; the plain kernel 7,400.
// DP: 32, 64, 128 or 256, the head sizes' upper bound.  The items of a key/value head are blocks keys' blocks of each of the first n_direct sequences,
// which bring one token each (one chunk a block: straight into the weights), then most_work pieces of work of each of the others, which have parts as
// weigh_runs_kernel's.  grid (key/value heads, items in rows of gridDim.y).
template <typename T, int DP>
__global__ __launch_bounds__(F32_WAVES* SIA_WAVE) void weigh_float_kernel(
    const T* __restrict__ q, int q_row_stride, const T* __restrict__ k_pages, const int* __restrict__ block_table, int table_width,
    const int* __restrict__ cu_q, const int* __restrict__ kv_len, const float* __restrict__ row_stats, int n_heads, int n_kv, int head_dim,
    int page_size, int n_pages, float scale, int chunk_rows, int most_keys, int n_direct, int blocks, int most_work, int items,
    float* __restrict__ parts, const Weighed w) {
    constexpr int PIECES = DP / 16, F32_BLOCKS = f32_blocks(DP), F32_WAVE_KEYS = 16 * F32_BLOCKS, F32_KEYS = f32_keys(DP);
    const int hk = blockIdx.x, group = n_heads / n_kv;
    const unsigned item = blockIdx.z * gridDim.y + blockIdx.y;
    if (item >= (unsigned)items) return;
    const int piece = (int)item - n_direct * blocks;      // of the others', if not negative
    const unsigned each = piece < 0 ? blocks : most_work, at = piece < 0 ? item : (unsigned)piece, nth = at / each;
    Work run;
    if (!find_work<F32_KEYS>(run, (int)(at - nth * each), (int)nth + (piece < 0 ? 0 : n_direct), cu_q, kv_len, group, chunk_rows, most_keys)) return;
    const int wave = threadIdx.x / SIA_WAVE, lane = threadIdx.x % SIA_WAVE, r = lane & 15, g = lane >> 4;
    const int k0 = run.key0 + wave * F32_WAVE_KEYS;
    if (k0 >= run.length) return;
    const int* table = block_table + (size_t)run.seq * table_width;
    auto load_row = [&](f32x4 (&x)[PIECES], const T* row) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int d = 16 * i + 4 * g;
            x[i] = load4(row + (d < head_dim ? d : 0));
            if (d >= head_dim) x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            across_groups(x[i]);
        }
    };
    f32x4 sum[F32_BLOCKS], kf[F32_BLOCKS][PIECES];
    bool paged[F32_BLOCKS];
#pragma unroll
    for (int b = 0; b < F32_BLOCKS; ++b) {
        sum[b] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int key = min(k0 + b * 16 + r, run.length - 1), page = table[key / page_size];
        paged[b] = page >= 0 && page < n_pages;
        load_row(kf[b], k_pages + (((size_t)(paged[b] ? page : 0) * n_kv + hk) * page_size + key % page_size) * head_dim);
    }
    // the places beyond which this lane's four keys of a block are seen by none: where there is no page, nobody's
    int seen_from[F32_BLOCKS][4];
#pragma unroll
    for (int b = 0; b < F32_BLOCKS; ++b) {
        const unsigned long long pages = __ballot(paged[b]);      // lanes 0 .. 15: the block's keys
#pragma unroll
        for (int i = 0; i < 4; ++i) seen_from[b][i] = pages >> (4 * g + i) & 1 ? k0 + b * 16 + 4 * g + i : 0x7fffffff;
    }
    // from the chunk's first row that sees the wave's first key on
    const int row_first = max(run.row_begin, max(0, k0 - run.start) * group), by_token = 16 / group, by_head = 16 - by_token * group;
    const int last_token = max(run.row_end - 1, 0) / group;
    Column col;
    col.begin(row_first + r, group);
    auto fetch = [&](f32x4 (&qf)[PIECES], float& stat, int& place) {
        const int t = min(col.token, last_token);      // behind the last row: some row of the last token, with weights of 0
        const size_t at = (size_t)(run.q_begin + t);
        load_row(qf, q + at * q_row_stride + (hk * group + col.head) * head_dim);
        const float own = row_stats[at * n_heads + hk * group + col.head];
        stat = col.row < run.row_end ? own : INFINITY;
        place = run.start + t;
        col.next<16>(by_token, by_head, group);
    };
    f32x4 qa[PIECES], qb[PIECES];
    float sa, sb;
    int pa, pb;
    auto compute = [&](const f32x4 (&qf)[PIECES], float stat, int place) {
        f32x4 s[F32_BLOCKS];
#pragma unroll
        for (int b = 0; b < F32_BLOCKS; ++b) s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int b = 0; b < F32_BLOCKS; ++b) s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[b][i][e], qf[i][e], s[b], 0, 0, 0);
#pragma unroll
        for (int b = 0; b < F32_BLOCKS; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = exp2f(fmaf(s[b][i] * scale, 1.4426950408889634f, -stat));
                sum[b][i] += seen_from[b][i] <= place ? p : 0.f;
            }
    };
    if (row_first < run.row_end) fetch(qa, sa, pa);
    for (int row0 = row_first; row0 < run.row_end; row0 += 32) {
        fetch(qb, sb, pb);
        compute(qa, sa, pa);
        if (row0 + 16 >= run.row_end) break;
        fetch(qa, sa, pa);
        compute(qb, sb, pb);
    }
    leave_sums(sum, k0, run, parts && piece >= 0 ? parts + ((size_t)piece * n_kv + hk) * F32_KEYS : nullptr, w, n_kv, hk);
}

// Whether weigh_float_kernel takes such heads and rows.
static bool float_takes(const void* q, int q_row_stride, const void* k_pages, int head_dim, int dtype) {
    return head_dim <= 256 && head_dim % 4 == 0 && q_row_stride % 4 == 0 && ((uintptr_t)q | (uintptr_t)k_pages) % (dtype == SIA_F32 ? 16 : 8) == 0;
}

// How the sequences of a launch are cut: three workgroups are on a compute unit at a time.
constexpr int F32_LEAST_ROWS = 64;
static Cut cut_float(int n_tokens, int q_bound, int n_seqs, int max_kv, int n_heads, int n_kv, int head_dim) {
    return cut_runs(n_tokens, q_bound, n_seqs, max_kv, n_heads / n_kv, n_kv, f32_keys(head_dim), F32_LEAST_ROWS, 768);
}
// Of n_single sequences of a token each, those whose rows fill no chunk: all or none.  They need no parts.
static int direct_of(int n_single, int group) { return group <= F32_LEAST_ROWS ? n_single : 0; }

template <typename T, int DP>
static int weigh_float(const T* q, int q_row_stride, const T* k_pages, const int* block_table, int table_width, const int* cu_q, const int* kv_len,
                       const float* row_stats, float* parts, int n_direct, int n_seqs, int max_kv, int n_heads, int n_kv, int head_dim, int page_size,
                       int n_pages, float scale, const Cut& cut, const Weighed& w, hipStream_t stream) {
    const int most_keys = (int)min((long long)max_kv, (long long)table_width * page_size), blocks = (max_kv + f32_keys(DP) - 1) / f32_keys(DP);
    const long long items = (long long)n_direct * blocks + (long long)(n_seqs - n_direct) * cut.most_work, rows = (items + 65534) / 65535;
    if (blocks > 65535 || items > 0x7fff0000) return SIA_BAD_ARGUMENT;
    hipLaunchKernelGGL((weigh_float_kernel<T, DP>), dim3(n_kv, (unsigned)((items + rows - 1) / rows), (unsigned)rows), dim3(F32_WAVES * SIA_WAVE), 0,
                       stream, q, q_row_stride, k_pages, block_table, table_width, cu_q, kv_len, row_stats, n_heads, n_kv, head_dim, page_size, n_pages,
                       scale, cut.chunk_rows, most_keys, n_direct, blocks, cut.most_work, (int)items, parts, w);
    if (parts)
        hipLaunchKernelGGL(weigh_add_kernel<f32_keys(DP)>, dim3(n_kv, blocks, n_seqs - n_direct), dim3(f32_keys(DP)), 0, stream, parts, cu_q, kv_len,
                           n_heads, n_kv, n_direct, cut.chunk_rows, most_keys, cut.most_work, w);
    return SIA_LAUNCH_CHECK();
}

// ---------------------------------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------------------------------
extern "C" int sia_attention_f32_stats(const float*, int, const float*, const float*, const int*, int, const int*, const int*, float*, int, int, int,
                                       int, int, int, int, int, int, float, const float*, float*, hipStream_t);
extern "C" int sia_attention_generic_stats(const void*, int, const void*, const void*, const int*, int, const int*, const int*, void*, int, int, int,
                                           int, int, int, float, const float*, float*, int, hipStream_t);

// Floats that sia_attention_weighed's workspace holds (arguments as there).
SIA_EXPORT long long sia_attention_weighed_workspace(int n_tokens, int n_single, int q_bound, int n_seqs, int max_kv, int n_heads, int n_kv,
                                                     int head_dim) {
    if (n_tokens <= 0 || q_bound <= 0 || n_seqs <= 0 || n_single < 0 || n_single > n_seqs || max_kv <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv)
        return 0;
    const int n_cut = n_seqs - direct_of(n_single, n_heads / n_kv);
    return (long long)n_tokens * n_heads + cut_float(n_tokens, q_bound, n_cut, max_kv, n_heads, n_kv, head_dim).floats;
}

// The arguments of the attention kernels without window, blocks and forms; q: rows of the step's tokens; n_single: that many sequences, the first
// ones, bring one token each; none of them more than q_bound tokens, n_tokens in all, over at most max_kv places; weights [n_slots][n_kv][places], a
// sequence's row at slots[s].
SIA_EXPORT int sia_attention_weighed(const void* q, int q_row_stride, const void* k_pages, const void* v_pages, const int* block_table, int table_width,
                                     const int* seq_of_token, const int* positions, const int* cu_q, const int* kv_len, void* out, float* ws,
                                     int n_tokens, int n_single, int n_seqs, int q_bound, int max_kv, int n_heads, int n_kv, int head_dim,
                                     int value_dim, int page_size, int n_pages, float scale, const float* sinks, float* weights, const int* slots,
                                     int n_slots, int places, int dtype, hipStream_t stream) {
    if (n_tokens <= 0 || n_seqs <= 0) return 0;
    if ((dtype != SIA_F32 && dtype != SIA_BF16) || head_dim <= 0 || head_dim > WEIGH_MAX_HEAD_DIM || value_dim <= 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv ||
        n_heads > 65535 || n_seqs > 65535 || page_size <= 0 || table_width <= 0 || n_pages <= 0 || q_bound <= 0 || max_kv <= 0 || places < max_kv ||
        n_slots <= 0 || !ws || !weights || n_single < 0 || n_single > n_seqs || (long long)q_bound * (n_heads / n_kv) > 0x7fffff00)
        return SIA_BAD_ARGUMENT;
    float* stats = ws;
    int rc = dtype == SIA_F32 ? sia_attention_f32_stats((const float*)q, q_row_stride, (const float*)k_pages, (const float*)v_pages, block_table, table_width,
                                                        seq_of_token, positions, (float*)out, n_tokens, n_single, n_seqs, max_kv, n_heads, n_kv,
                                                        head_dim, value_dim, page_size, scale, sinks, stats, stream)
                              : sia_attention_generic_stats(q, q_row_stride, k_pages, v_pages, block_table, table_width, seq_of_token, positions, out,
                                                            n_tokens, n_heads, n_kv, head_dim, value_dim, page_size, scale, sinks, stats, dtype, stream);
    if (rc) return rc;
    const Weighed w{weights, slots, nullptr, n_slots, places, 0};
    if (!float_takes(q, q_row_stride, k_pages, head_dim, dtype)) {
        if (dtype == SIA_F32)
            return weigh_plain((const float*)q, q_row_stride, (const float*)k_pages, block_table, table_width, cu_q, kv_len, stats, n_seqs, max_kv, n_heads,
                               n_kv, head_dim, page_size, n_pages, scale, w, stream);
        return weigh_plain((const bf16_t*)q, q_row_stride, (const bf16_t*)k_pages, block_table, table_width, cu_q, kv_len, stats, n_seqs, max_kv, n_heads, n_kv,
                           head_dim, page_size, n_pages, scale, w, stream);
    }
    const int n_direct = direct_of(n_single, n_heads / n_kv);
    const Cut cut = cut_float(n_tokens, q_bound, n_seqs - n_direct, max_kv, n_heads, n_kv, head_dim);
    float* parts = cut.floats ? stats + (long long)n_tokens * n_heads : nullptr;
#define OF_SIZE(T, DP)                                                                                                                                  \
    weigh_float<T, DP>((const T*)q, q_row_stride, (const T*)k_pages, block_table, table_width, cu_q, kv_len, stats, parts, n_direct, n_seqs, max_kv, n_heads, \
                       n_kv, head_dim, page_size, n_pages, scale, cut, w, stream)
#define OF_TYPE(T) (head_dim <= 32 ? OF_SIZE(T, 32) : head_dim <= 64 ? OF_SIZE(T, 64) : head_dim <= 128 ? OF_SIZE(T, 128) : OF_SIZE(T, 256))
    return dtype == SIA_F32 ? OF_TYPE(float) : OF_TYPE(bf16_t);
#undef OF_TYPE
#undef OF_SIZE
}
