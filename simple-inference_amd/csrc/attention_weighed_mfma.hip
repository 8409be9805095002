// bfloat16 attention over the paged cache that also adds up each cached key's weight (attention_weighed.hip says what the sums are),
// on the matrix cores.  Compiled once per head size with attention_mfma.hip, whose tiles it uses.
//
// Single tokens (weighed_decode_kernel): one walk over keys and values.  A weight can be made only when the row's maximum and sum are known, and
// those only when all splits of the sequence are through: the walk leaves every scaled score (float, in units of log2) in a workspace,
// 4 bytes a key and query head beside the 4 * head size bytes a key and key/value head that it reads, and weighed_join_kernel turns
// them into weights while it merges the splits.  A sequence of one split is finished by its one workgroup.
// Runs of tokens (weigh_runs_kernel): the attention kernel leaves every row's statistic, and the scores are made once more, with keys as
// rows and queries as columns: a lane holds 4 keys of 16 columns' scores, so that the sum over the queries stays in its registers to the end.
//
// What is rounded to fewer bits: the probabilities of the value product, to bfloat16 (off by at most 2^-8 of each), as the matrix cores take them and
// as attention without weights has it, so that a layer gives results of the same kind whether it weighs its cache or not.  Against the definition
// in 64 bits results are off by 0.0016 of their size for one row over 40 keys, as with probabilities in float, by 0.0014 for a prompt of 2,048, where those
// give 0.0013, and by 0.0019 against 0.0015 at worst among other lengths: most of it is the result's own rounding.  The sums of weights are made of float exponentials of float scores; a single
// token's scaled scores are rounded to float on their way through the workspace, where its sum of exponentials took them unrounded.
#include "attention_tiles.h"
#include "weighed.h"

// ---------------------------------------------------------------------------------------------------
// single tokens
// ---------------------------------------------------------------------------------------------------
// Keys [j0, j1) of a sequence and head: their weights from the scores, summed over the group's query heads in order.  The last key is the
// step's own: its sum begins at zero.
__device__ __forceinline__ void add_weights(float* __restrict__ row, const float* __restrict__ scores, int row_keys, const float* stat, int group,
                                            int j0, int j1, int length, int first_thread, int threads) {
    for (int j = j0 + first_thread; j < j1; j += threads) {
        float sum = 0.f;
        for (int c = 0; c < group; ++c) sum += fast_exp2(scores[(size_t)c * row_keys + j] - stat[c]);
        row[j] = (j < length - 1 ? row[j] : 0.f) + sum;
    }
}

// Workgroups of four waves that share one (sequence, key/value head) with n_tiles tiles: the largest power of two that leaves each WEIGHED_TILES.  A
// function of the sequence's own length only.  us a call with 4, 8, 16 and 32 tiles a split: one row over 2,048 keys, 32 heads of 128 on 8: 9.4 9.7 11.8 16.3;
// 27 of 24 over about 700 28.9 25.4 31.4 25.1;  8 of 24 over 2,048 25.9 19.2 18.2 19.5;  3 of 32 over 12,000 44.8 42.5 43.8 42.6;  4 of 16 on 1 over
// 6,000 14.0 15.7 19.0 26.6;  64 of 32 over about 900 81.0 70.1 69.7 64.2.
constexpr int WEIGHED_TILES = 8, WEIGHED_MAX_SPLITS = 64;
__host__ __device__ inline int weighed_splits(int n_tiles) {
    int s = 1;
    while (s < WEIGHED_MAX_SPLITS && 2 * s * WEIGHED_TILES <= n_tiles) s *= 2;
    return s;
}

// Scores of a tile as they go into the workspace: lane (r, g) holds keys kb + 8 g .. + 7 of column r.
__device__ __forceinline__ void leave_scores(float* __restrict__ mine, int kb, int g, const floatx4 (&s)[2], float scale) {
    float4* to = reinterpret_cast<float4*>(mine + kb + 8 * g);
    to[0] = make_float4(s[0][0] * scale, s[0][1] * scale, s[0][2] * scale, s[0][3] * scale);
    to[1] = make_float4(s[1][0] * scale, s[1][1] * scale, s[1][2] * scale, s[1][3] * scale);
}

// grid (groups of query heads, sequences, splits), four waves of a run of tiles each, as attn_decode_kernel's plain mode.  The memory bounds it:  8 rows over
// 2,048 keys, 24 heads of 128 on 8, 15.1 us and 3.9 for the join (67 MB: 4.4 TB/s), 3 of 32 over 12,000 37.6 and 5.4 (150 MB: 4.0 TB/s).  With the keys and
// values in the last-level cache a whole call takes 19.1 and 31.3 us, attention alone 18.7 and 29.7.
// kv_share groups of query heads read one key/value head; with more than one, or several splits, the join makes the weights.
__global__ __launch_bounds__(DEC_WAVES* SIA_WAVE) void weighed_decode_kernel(
    const bf16_t* __restrict__ q, int q_row_stride, const bf16_t* __restrict__ kp, const bf16_t* __restrict__ vp,
    const int* __restrict__ block_table, int table_width, const int* __restrict__ cu_q, const int* __restrict__ kv_len,
    float* __restrict__ ws_acc, float* __restrict__ ws_ml, bf16_t* __restrict__ out, int n_heads, int n_groups, int ps_log2, float scale,
    const float* __restrict__ sinks, int max_splits, int kv_share, int most_keys, const Weighed w) {
    extern __shared__ float lds[];  // [waves][group][HD + 2]
    const int hg = blockIdx.x, seq = blockIdx.y, split = blockIdx.z;
    const int wave = threadIdx.x / SIA_WAVE, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int length = min(kv_len[seq], most_keys), last = length - 1, group = n_heads / n_groups;
    if (length <= 0) {      // a row that sees nothing
        for (int i = threadIdx.x; i < group * HD && split == 0; i += DEC_WAVES * SIA_WAVE)
            out[((size_t)cu_q[seq] * n_heads + hg * group) * HD + i] = 0;
        return;
    }
    const int n_tiles = last / TILE + 1, n_splits = min(weighed_splits(n_tiles), max_splits);
    if (split >= n_splits) return;
    scale *= LOG2E;  // exponentials are taken as powers of two
    const int hk = hg / kv_share, n_kv = n_groups / kv_share;
    const int* table = block_table + (size_t)seq * table_width;
    bf16x8 qf[KSTEPS];
    load_q(qf, r < group ? q + (size_t)seq * q_row_stride + (hg * group + r) * HD : nullptr, g);
    const int n_runs = n_splits * DEC_WAVES, run = split * DEC_WAVES + wave;
    const int first = (int)(((long long)run * n_tiles) / n_runs), end = (int)(((long long)(run + 1) * n_tiles) / n_runs);
    float* const scores = w.scores + ((size_t)seq * n_heads + hg * group + min(r, group - 1)) * w.row_keys;

    Softmax<1> sm;
    sm.start();
    floatx4 acc[1][DBLOCKS];
#pragma unroll
    for (int db = 0; db < DBLOCKS; ++db) acc[0][db] = floatx4{0.f, 0.f, 0.f, 0.f};
    const Forms none{0.f, 0};
    const Places all{0, 0};
    const int lo[1] = {r < group ? 0 : 1 << 30}, hi[1] = {r < group ? last : -1};
    auto compute = [&](Stage& st, int kb) {
        floatx4 s[1][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s[0][h] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) s[0][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(st.k[h][ks], qf[ks], s[0][h], 0, 0, 0);
        }
        if (r < group) leave_scores(scores, kb, g, s[0], scale);
        if (kb + TILE - 1 > last) clear_values(st, kb, g, last);
        bf16x8 p[1];
        softmax_update<1>(s, kb, lo, hi, scale, sm, acc, p, none);
#pragma unroll
        for (int db = 0; db < DBLOCKS; ++db) acc[0][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(st.v[db], p[0], acc[0][db], 0, 0, 0);
    };
    const int range_lo = first * TILE, range_hi = min(last, end * TILE - 1), kb_end = (end - 1) * TILE;
    for (int w_first = range_lo; first < end && w_first <= kb_end;) {      // 64 entries of the block table at a time
        const int first_page = w_first >> ps_log2, w_end = (first_page + SIA_WAVE) << ps_log2, w_last = min(kb_end, w_end - TILE);
        PageWindow pages;
        pages_load(pages, table, table_width, first_page, lane, ps_log2, all);
        Stage a, b;
        load_stage(a, kp, vp, pages, ps_log2, n_kv, hk, w_first, range_lo, range_hi);
        for (int kb = w_first; kb <= w_last; kb += 2 * TILE) {      // two register stages in turn
            load_stage(b, kp, vp, pages, ps_log2, n_kv, hk, min(kb + TILE, w_last), range_lo, range_hi);
            compute(a, kb);
            load_stage(a, kp, vp, pages, ps_log2, n_kv, hk, min(kb + 2 * TILE, w_last), range_lo, range_hi);
            if (kb + TILE <= w_last) compute(b, kb + TILE);
        }
        w_first = w_end;
    }
    constexpr int ROW = HD + 2;
    leave_state(lds + (size_t)(wave * group + min(r, group - 1)) * ROW, sm, acc, g, r < group);
    __syncthreads();      // the states are there, and so are the workgroup's scores

    __shared__ float stat[16];
    for (int idx = threadIdx.x; idx < group * HD; idx += DEC_WAVES * SIA_WAVE) {
        const int c = idx / HD, d = idx % HD, head = hg * group + c;
        float o, mx, lsum;
        merge_waves([&](int v) { return lds + (size_t)(v * group + c) * ROW; }, d, o, mx, lsum);
        if (n_splits == 1) {
            const float total = lsum + sink_term(sinks, head, mx);
            out[((size_t)cu_q[seq] * n_heads + head) * HD + d] = float_to_bf16(o * (1.f / total));
            if (d == 0) stat[c] = mx + log2f(total);
        } else {
            ws_acc[(((size_t)seq * n_heads + head) * max_splits + split) * HD + d] = o;
        }
        if (d == 0 && ws_ml) {
            float* ml = ws_ml + (((size_t)seq * n_heads + head) * max_splits + split) * 2;
            ml[0] = mx;
            ml[1] = lsum;
        }
    }
    if (n_splits > 1 || kv_share > 1) return;
    __syncthreads();
    float* row = weight_row(w, seq, n_kv, hk);
    if (row) add_weights(row, w.scores + ((size_t)seq * n_heads + hg * group) * w.row_keys, w.row_keys, stat, group, 0, length, length, threadIdx.x, DEC_WAVES * SIA_WAVE);
}

// grid (key/value heads, sequences, query heads of a group + chunks of JOIN_KEYS keys): the first merge the splits' results of a query head
// each, the others make the weights of their keys from the scores, a thread a key, with the rows' statistics made anew from the splits' (a few hundred
// bytes).  Latency bounds both: what does not depend on another load's result is asked for first.
constexpr int JOIN_KEYS = 256, JOIN_MOST_HEADS = 256;
__global__ __launch_bounds__(JOIN_KEYS) void weighed_join_kernel(
    const float* __restrict__ ws_acc, const float* __restrict__ ws_ml, const int* __restrict__ cu_q, const int* __restrict__ kv_len,
    bf16_t* __restrict__ out, int n_heads, int n_kv, int max_splits, int kv_share, const float* __restrict__ sinks, int most_keys,
    const Weighed w) {
    const int hk = blockIdx.x, seq = blockIdx.y, group = n_heads / n_kv, chunk = (int)blockIdx.z - group;
    const int length = min(kv_len[seq], most_keys);
    if (length <= 0 || chunk * JOIN_KEYS >= length) return;
    const int n_splits = min(weighed_splits((length - 1) / TILE + 1), max_splits);
    if (n_splits == 1 && (kv_share == 1 || chunk < 0)) return;      // finished by its one workgroup
    const size_t base = ((size_t)seq * n_heads + hk * group) * max_splits;
    const float2* const ml = reinterpret_cast<const float2*>(ws_ml) + base;
    if (chunk < 0) {
        const int c = blockIdx.z, head = hk * group + c, d = min((int)threadIdx.x, HD - 1);
        const float* const acc_at = ws_acc + (base + (size_t)c * max_splits) * HD + d;
        const float2* const mine = ml + (size_t)c * max_splits;
        const float o = n_splits <= 8    ? combine_all<8>(n_splits, acc_at, mine, sinks, head)
                        : n_splits <= 16 ? combine_all<16>(n_splits, acc_at, mine, sinks, head)
                        : n_splits <= 32 ? combine_all<32>(n_splits, acc_at, mine, sinks, head)
                                         : combine_all<WEIGHED_MAX_SPLITS>(n_splits, acc_at, mine, sinks, head);
        if (threadIdx.x < HD) out[((size_t)cu_q[seq] * n_heads + head) * HD + d] = float_to_bf16(o);
        return;
    }
    __shared__ float stat[JOIN_MOST_HEADS];
    const int j = min(chunk * JOIN_KEYS + (int)threadIdx.x, length - 1);
    const float* const scores = w.scores + ((size_t)seq * n_heads + hk * group) * w.row_keys + j;
    constexpr int AHEAD = 8;
    float s[AHEAD];
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) s[c] = scores[(size_t)min(c, group - 1) * w.row_keys];
    float* row = weight_row(w, seq, n_kv, hk);
    const float old = row && j < length - 1 ? row[j] : 0.f;      // the last key is the step's own: its sum begins at zero
    // statistics: 16 lanes a query head, a split each at a time
    for (int c0 = threadIdx.x / 16; c0 < (group + JOIN_KEYS / 16 - 1) / (JOIN_KEYS / 16) * (JOIN_KEYS / 16); c0 += JOIN_KEYS / 16) {
        const int c = min(c0, group - 1), lane = threadIdx.x % 16;
        float mx = -INFINITY, total = 0.f;
        for (int s0 = lane; s0 < n_splits; s0 += 16) {
            const float2 state = ml[(size_t)c * max_splits + s0];
            const float top = fmaxf(mx, state.x), was = mx == -INFINITY ? 0.f : total * fast_exp2(mx - top);
            total = state.x == -INFINITY ? was : fmaf(fast_exp2(state.x - top), state.y, was);
            mx = top;
        }
        float top = mx;
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 16));
        total = row_sum(mx == -INFINITY ? 0.f : total * fast_exp2(mx - top)) + sink_term(sinks, hk * group + c, top);
        if (lane == 0 && c0 < group) stat[c] = top + log2f(total);
    }
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) sum += c < group ? fast_exp2(s[c] - stat[min(c, group - 1)]) : 0.f;
    for (int c = AHEAD; c < group; ++c) sum += fast_exp2(scores[(size_t)c * w.row_keys] - stat[c]);
    if (row && chunk * JOIN_KEYS + (int)threadIdx.x < length) row[j] = old + sum;
}

// ---------------------------------------------------------------------------------------------------
// runs of tokens
// ---------------------------------------------------------------------------------------------------
constexpr int RUN_WAVES = 4, WAVE_BLOCKS = 4, WAVE_KEYS = 16 * WAVE_BLOCKS, RUN_KEYS = RUN_WAVES * WAVE_KEYS;

// grid (key/value heads, pieces of work of a run, runs): workgroups go to the chip's dies in turn, so that with 8 key/value heads a die reads
// one head's keys and queries.  A wave holds its 64 keys as operands; the rows come through LDS 32 at a time, two stages of it, the next tile's loads under way while one is computed.  (Read from memory as
// operands, 16 rows of 16 bytes a lane, every lane is an access of its own to the first-level cache: four times as many, and what bound it.)
// What bounds it: a score costs an exponential (16 cycles a wave), a multiply-add and an add (4 each).  2,048 tokens of 24 heads of 128 on 8: 28 us
// (beside an attention of 54), in which 488 workgroups go in one round: 1.1 us for the piece of work, 1.9 (4.3 the longest) until the first rows and the keys
// are there, 14 or 15 tiles of 32 rows of 1.22 us (17 in all, 22 the longest), and 0.5 for the sums.  A tile's 1.22 us are 1,460 cycles at 2.4 GHz for each of the
// two waves of a vector unit, of which the unit's own instructions take 1,016.
// Workgroups for 256, 384, 512, 768 and 1,536 of them 34.5 33.8 28.2 32.4 35.7: two are on a unit at a time, so 512 go in one round.
// parts: [run][piece of work][key/value head][RUN_KEYS], or null where every block has one chunk.
constexpr int TILE_ROWS = 32, PIECES = HD / 8, ROW_STRIDE = HD + ((HD / 16) % 2 == 0 ? 16 : 0);      // as the prefill kernel's key rows
constexpr int RUN_THREADS = RUN_WAVES * SIA_WAVE, PER_THREAD = (TILE_ROWS * PIECES + RUN_THREADS - 1) / RUN_THREADS;
typedef uint32_t piece_t __attribute__((ext_vector_type(4)));      // a plain 16-byte register value

// A thread's part of a tile of rows: pieces of q, and (of the first 32 threads) a row's statistic and place.
struct RowTile {
    piece_t q[PER_THREAD];
    float stat;
    int place;
};

// Lane l of every wave goes with row l % 32 of the tiles; the threads that load the row's pieces ask it for where the row lies.
struct RowWalk {
    Column own;
    int by_token, by_head, last_token, row_end, start, group, n_heads;
    unsigned stride;      // 16-byte pieces from a token's row to the next
    const bf16_t* q;      // the row of the chunk's first token, at the group's first head
    const float* stats;
};

__device__ __forceinline__ void fetch_rows(RowTile& t, RowWalk& w) {
    const int token = min(w.own.token, w.last_token);      // behind the last row: some row of the last token, with weights of 0
    const unsigned at = (unsigned)token * w.stride + w.own.head * PIECES;
    const float stat = w.stats[(size_t)token * w.n_heads + w.own.head];
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        const int c = min((int)threadIdx.x + i * RUN_THREADS, TILE_ROWS * PIECES - 1);
        t.q[i] = reinterpret_cast<const piece_t*>(w.q)[(size_t)(unsigned)__shfl((int)at, c / PIECES, SIA_WAVE) + c % PIECES];
    }
    t.stat = w.own.row < w.row_end ? stat : INFINITY;
    t.place = w.start + token;
    w.own.next<TILE_ROWS>(w.by_token, w.by_head, w.group);
}

__device__ __forceinline__ void store_rows(const RowTile& t, bf16_t* __restrict__ rows, float* __restrict__ stats, int* __restrict__ places) {
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        const int c = threadIdx.x + i * RUN_THREADS;
        if (TILE_ROWS * PIECES % RUN_THREADS == 0 || c < TILE_ROWS * PIECES)
            *reinterpret_cast<piece_t*>(rows + c / PIECES * ROW_STRIDE + c % PIECES * 8) = t.q[i];
    }
    if (threadIdx.x < TILE_ROWS) {
        stats[threadIdx.x] = t.stat;
        places[threadIdx.x] = t.place;
    }
}

// A tile's rows against the wave's keys, which are k0 .. k0 + 63 (k0 the same in all lanes).
__device__ __forceinline__ void weigh_rows(floatx4 (&sum)[WAVE_BLOCKS], const bf16x8 (&kf)[WAVE_BLOCKS][KSTEPS], const bf16_t* __restrict__ rows,
                                           const float* __restrict__ stats, const int* __restrict__ places, int k0, float scale) {
    constexpr int HALVES = TILE_ROWS / 16;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    int place[HALVES];
    float stat[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        place[h] = places[h * 16 + r];
        stat[h] = stats[h * 16 + r];
    }
    if (__builtin_amdgcn_readlane(place[HALVES - 1], 15) < k0) return;      // none of the rows sees one of the wave's keys: places rise with the rows
    floatx4 s[HALVES][WAVE_BLOCKS];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
#pragma unroll
        for (int v = 0; v < WAVE_BLOCKS; ++v) s[h][v] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
            // (beyond HD: some elements of the row once more, which meet zeros of the keys)
            const bf16x8 x = load8(rows + (h * 16 + r) * ROW_STRIDE + (HD % 32 == 0 || ks < KSTEPS - 1 ? ks * 32 + g * 8 : min(ks * 32 + g * 8, HD - 8)));
#pragma unroll
            for (int v = 0; v < WAVE_BLOCKS; ++v) s[h][v] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[v][ks], x, s[h][v], 0, 0, 0);
        }
    }
    const bool whole = __builtin_amdgcn_readfirstlane(place[0]) >= k0 + WAVE_KEYS - 1;
    if (whole) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int v = 0; v < WAVE_BLOCKS; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[v][i] += fast_exp2(fmaf(s[h][v][i], scale, -stat[h]));
        return;
    }
    // A key that a row does not see gets nothing of it, whatever the row's scores and statistic are.
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int v = 0; v < WAVE_BLOCKS; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = fast_exp2(fmaf(s[h][v][i], scale, -stat[h]));
                sum[v][i] += k0 + v * 16 + g * 4 + i <= place[h] ? p : 0.f;
            }
}

__global__ __launch_bounds__(RUN_THREADS) void weigh_runs_kernel(
    const bf16_t* __restrict__ q, int q_row_stride, const bf16_t* __restrict__ kp, const int* __restrict__ block_table, int table_width,
    const int* __restrict__ cu_q, const int* __restrict__ kv_len, const float* __restrict__ row_stats, int n_heads, int n_kv, int ps_log2,
    float scale, int seq_begin, int chunk_rows, int most_keys, float* __restrict__ parts, const Weighed w) {
    __shared__ __attribute__((aligned(16))) bf16_t rows_s[2][TILE_ROWS * ROW_STRIDE];
    __shared__ float stat_s[2][TILE_ROWS];
    __shared__ int place_s[2][TILE_ROWS];
    const int hk = blockIdx.x, group = n_heads / n_kv;
    Work run;
    if (!find_work<RUN_KEYS>(run, blockIdx.y, seq_begin + blockIdx.z, cu_q, kv_len, group, chunk_rows, most_keys)) return;      // the whole workgroup
    float* const part = parts ? parts + (((size_t)blockIdx.z * gridDim.y + blockIdx.y) * n_kv + hk) * RUN_KEYS : nullptr;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int k0 = __builtin_amdgcn_readfirstlane(run.key0 + tid / SIA_WAVE * WAVE_KEYS);
    const int* table = block_table + (size_t)run.seq * table_width;
    scale *= LOG2E;

    const int row_first = run.row_begin;
    RowWalk walk;
    walk.by_token = TILE_ROWS / group;
    walk.by_head = TILE_ROWS - walk.by_token * group;
    walk.last_token = max(run.row_end - 1, 0) / group;
    walk.row_end = run.row_end;
    walk.start = run.start;
    walk.group = group;
    walk.n_heads = n_heads;
    walk.own.begin(row_first + tid % TILE_ROWS, group);
    const int token_first = min(row_first / group, walk.last_token);      // tokens from here on, so that a piece's index stays small
    walk.own.token -= token_first;
    walk.last_token -= token_first;
    walk.start += token_first;
    walk.stride = q_row_stride / 8;
    walk.q = q + (size_t)(run.q_begin + token_first) * q_row_stride + hk * group * HD;
    walk.stats = row_stats + (size_t)(run.q_begin + token_first) * n_heads + hk * group;
    RowTile a, b;
    fetch_rows(a, walk);
    fetch_rows(b, walk);
    floatx4 sum[WAVE_BLOCKS];
    bf16x8 kf[WAVE_BLOCKS][KSTEPS];
#pragma unroll
    for (int v = 0; v < WAVE_BLOCKS; ++v) {
        sum[v] = floatx4{0.f, 0.f, 0.f, 0.f};
        const int key = min(k0 + v * 16 + r, run.length - 1);
        const int page = max(table[key >> ps_log2], 0);
        const bf16_t* row = kp + (((size_t)page * n_kv + hk) * (1 << ps_log2) + (key & ((1 << ps_log2) - 1))) * HD;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
            const int d0 = ks * 32 + g * 8;
            kf[v][ks] = load8(row + (HD % 32 == 0 || ks < KSTEPS - 1 ? d0 : min(d0, HD - 8)));
            if (HD % 32 != 0 && ks == KSTEPS - 1 && d0 >= HD) kf[v][ks] = zero8();
        }
    }
    const bool live = k0 < run.length;
    store_rows(a, rows_s[0], stat_s[0], place_s[0]);
    __syncthreads();
    for (int row0 = row_first; row0 < run.row_end; row0 += 2 * TILE_ROWS) {
        fetch_rows(a, walk);
        if (live) weigh_rows(sum, kf, rows_s[0], stat_s[0], place_s[0], k0, scale);
        store_rows(b, rows_s[1], stat_s[1], place_s[1]);
        __syncthreads();
        fetch_rows(b, walk);
        if (live && row0 + TILE_ROWS < run.row_end) weigh_rows(sum, kf, rows_s[1], stat_s[1], place_s[1], k0, scale);
        store_rows(a, rows_s[0], stat_s[0], place_s[0]);
        __syncthreads();
    }
    if (live) leave_sums(sum, k0, run, part, w, n_kv, hk);
}

// ---------------------------------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------------------------------
static int log2_of(int v) {
    int l = 0;
    while ((1 << l) < v && l < 30) ++l;
    return (1 << l) == v ? l : -1;
}

// Floats from one head's scores (or one chunk's sums) to the next for sequences of up to max_kv places: whole tiles.
static long long row_keys_of(int max_kv) { return ((long long)max_kv + TILE - 1) / TILE * TILE; }
static int splits_of(int max_kv) { return weighed_splits((max_kv + TILE - 1) / TILE); }

// Groups of query heads that share a key/value head: a launch's columns are 16, and the four waves' states lie in 64 KiB.
static int shares_of(int group) {
    for (int s = 1; s < group; ++s)
        if (group % s == 0 && group / s <= 16 && (size_t)DEC_WAVES * (group / s) * (HD + 2) * sizeof(float) <= 64 * 1024) return s;
    return group;
}

// Floats of the single tokens' workspace: scores, and the splits' states.
static long long single_floats(int n_single, int n_heads, int max_kv) {
    return n_single <= 0 ? 0 : (long long)n_single * n_heads * (row_keys_of(max_kv) + (long long)splits_of(max_kv) * (HD + 2));
}

static int attend_single(const bf16_t* q, int q_row_stride, const bf16_t* k_pages, const bf16_t* v_pages, const int* block_table, int table_width,
                         const int* cu_q, const int* kv_len, bf16_t* out, float* ws, int n_single, int n_heads, int n_kv, int ps_log2, float scale,
                         const float* sinks, int max_kv, Weighed w, hipStream_t stream) {
    const int share = shares_of(n_heads / n_kv), n_groups = n_kv * share, max_splits = splits_of(max_kv);
    w.scores = ws;
    w.row_keys = (int)row_keys_of(max_kv);
    const int most_keys = (int)min((long long)max_kv, (long long)table_width << ps_log2);      // what there is room for, whatever kv_len says
    float* acc = ws + (long long)n_single * n_heads * w.row_keys;
    float* ml = acc + (long long)n_single * n_heads * max_splits * HD;
    const size_t lds_bytes = (size_t)DEC_WAVES * (n_heads / n_groups) * (HD + 2) * sizeof(float);
    hipLaunchKernelGGL(weighed_decode_kernel, dim3(n_groups, n_single, max_splits), dim3(DEC_WAVES * SIA_WAVE), lds_bytes, stream, q, q_row_stride,
                       k_pages, v_pages, block_table, table_width, cu_q, kv_len, acc, ml, out, n_heads, n_groups, ps_log2, scale, sinks, max_splits,
                       share, most_keys, w);
    if (max_splits > 1 || share > 1)
        hipLaunchKernelGGL(weighed_join_kernel, dim3(n_kv, n_single, n_heads / n_kv + (max_kv + JOIN_KEYS - 1) / JOIN_KEYS), dim3(JOIN_KEYS), 0,
                           stream, acc, ml, cu_q, kv_len, out, n_heads, n_kv, max_splits, share, sinks, most_keys, w);
    return SIA_LAUNCH_CHECK();
}

// How the runs of a launch are cut.  Two workgroups are on a compute unit at a time: 512 in all.
static Cut cut_of(int run_tokens, int q_bound, int n_runs, int run_kv, int n_heads, int n_kv) {
    return cut_runs(run_tokens, q_bound, n_runs, run_kv, n_heads / n_kv, n_kv, RUN_KEYS, 64, 512);
}

static int weigh_runs(const bf16_t* q, int q_row_stride, const bf16_t* k_pages, const int* block_table, int table_width, const int* cu_q,
                      const int* kv_len, const float* row_stats, float* parts, int seq_begin, int n_runs, const Cut& cut, int n_heads, int n_kv,
                      int ps_log2, float scale, int run_kv, const Weighed& w, hipStream_t stream) {
    const int blocks = (run_kv + RUN_KEYS - 1) / RUN_KEYS, most_keys = (int)min((long long)run_kv, (long long)table_width << ps_log2);
    hipLaunchKernelGGL(weigh_runs_kernel, dim3(n_kv, cut.most_work, n_runs), dim3(RUN_THREADS), 0, stream, q, q_row_stride, k_pages, block_table,
                       table_width, cu_q, kv_len, row_stats, n_heads, n_kv, ps_log2, scale, seq_begin, cut.chunk_rows, most_keys, parts, w);
    if (parts)
        hipLaunchKernelGGL(weigh_add_kernel<RUN_KEYS>, dim3(n_kv, blocks, n_runs), dim3(RUN_KEYS), 0, stream, parts, cu_q, kv_len, n_heads, n_kv,
                           seq_begin, cut.chunk_rows, most_keys, cut.most_work, w);
    return SIA_LAUNCH_CHECK();
}

extern "C" int sia_attn_prefill_stats(const void*, int, const void*, const void*, const int*, int, const int*, const int*, void*, int, int, int, int,
                                      int, int, int, int, int, int, float, const float*, float*, hipStream_t);

// Floats that sia_attn_weighed's workspace holds (arguments as there).
SIA_EXPORT long long sia_attn_weighed_workspace(int n_single, int n_seqs, int n_tokens, int q_bound, int run_kv, int max_kv, int n_heads, int n_kv) {
    if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || max_kv <= 0) return 0;
    long long floats = single_floats(n_single, n_heads, max_kv);
    if (n_single < n_seqs && q_bound > 0 && run_kv > 0)
        floats += (long long)n_tokens * n_heads + cut_of(n_tokens - n_single, q_bound, n_seqs - n_single, run_kv, n_heads, n_kv).floats;
    return floats;
}

// Sequences 0 .. n_single-1 of the step bring one token each, which is row s of q, and none of them is longer than max_kv (without such: no sequence
// is); sequences n_single .. n_seqs-1 bring at most q_bound tokens over at most run_kv places, n_tokens - n_single in all, in row tiles as
// sia_attn_prefill counts them.  weights [n_slots][n_kv][places], a sequence's row at slots[s].
SIA_EXPORT int sia_attn_weighed(const void* q, int q_row_stride, const void* k_pages, const void* v_pages, const int* block_table, int table_width,
                                const int* cu_q, const int* kv_len, void* out, float* ws, int n_single, int n_seqs, int n_tokens, int n_tiles,
                                int n_tiles_split, int n_tiles_long, int q_bound, int run_kv, int max_kv, int n_heads, int n_kv, int page_size,
                                float scale, const float* sinks, float* weights, const int* slots, int n_slots, int places, hipStream_t stream) {
    if (n_seqs <= 0 || n_tokens <= 0) return 0;
    const int ps_log2 = log2_of(page_size), n_runs = n_seqs - n_single;
    const bool runs = n_runs > 0 && q_bound > 0 && n_tokens > n_single;
    if (ps_log2 < 3 || n_kv <= 0 || n_heads % n_kv || n_heads / n_kv > JOIN_MOST_HEADS || n_heads > 65535 || n_seqs > 65535 || n_single < 0 || n_runs < 0 ||
        q_row_stride % 8 || table_width <= 0 || max_kv <= 0 || places < max_kv || n_slots <= 0 || !ws || !weights || !(scale > 0.f) ||
        (runs && (run_kv <= 0 || run_kv > (n_single > 0 ? places : max_kv) || (long long)q_bound * (n_heads / n_kv) > 0x7fffff00)))
        return SIA_BAD_ARGUMENT;
    const Cut cut = runs ? cut_of(n_tokens - n_single, q_bound, n_runs, run_kv, n_heads, n_kv) : Cut{};
    if (runs && (cut.most_work > 65535 || (run_kv + RUN_KEYS - 1) / RUN_KEYS > 65535)) return SIA_BAD_ARGUMENT;
    const Weighed w{weights, slots, nullptr, n_slots, places, 0};
    if (n_single > 0) {
        const int rc = attend_single((const bf16_t*)q, q_row_stride, (const bf16_t*)k_pages, (const bf16_t*)v_pages, block_table, table_width, cu_q, kv_len,
                                     (bf16_t*)out, ws, n_single, n_heads, n_kv, ps_log2, scale, sinks, max_kv, w, stream);
        if (rc) return rc;
    }
    if (!runs) return 0;
    float* stats = ws + single_floats(n_single, n_heads, max_kv);
    float* parts = cut.floats ? stats + (long long)n_tokens * n_heads : nullptr;
    const int rc = sia_attn_prefill_stats(q, q_row_stride, k_pages, v_pages, block_table, table_width, cu_q, kv_len, out, n_single, n_seqs, n_tiles,
                                          n_tiles_split, n_tiles_long, q_bound, run_kv, n_heads, n_kv, page_size, scale, sinks, stats, stream);
    if (rc) return rc;
    return weigh_runs((const bf16_t*)q, q_row_stride, (const bf16_t*)k_pages, block_table, table_width, cu_q, kv_len, stats, parts, n_single, n_runs, cut,
                      n_heads, n_kv, ps_log2, scale, run_kv, w, stream);
}
