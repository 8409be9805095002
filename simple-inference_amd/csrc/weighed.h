// What the kernels that add up the cached keys' attention weight share (attention_weighed.hip, attention_weighed_mfma.hip): where the sums
// lie, and how a run of tokens is cut into pieces of work.
//
// The rows of a key/value head are a run's (token, query head) pairs, token by token; a row sees the keys up to its token's place.  A
// workgroup has a block of KEYS keys and a chunk of the rows that see it: min(tokens, length - first key) tokens' rows, cut into as many
// chunks of equal size as chunk_rows asks for.  So none of the workgroups of the largest run is without work (half of them would be, if all blocks had the
// same chunks), and they are equally long; a shorter run beside it has as many, and those that it has no work for leave at once.  The chunks' sums of
// a block are added in order by a kernel of their own.
#pragma once

#include "common.h"

// Where a launch's sums and scores lie.
struct Weighed {
    float* weights;           // [n_slots][key/value heads][places]
    const int* slots;         // a sequence's row
    float* scores;            // [sequence][query head][row_keys], for single tokens
    int n_slots, places, row_keys;
};

// The sums of one (sequence, head); null for a slot that is none.
__device__ __forceinline__ float* weight_row(const Weighed& w, int seq, int n_kv, int hk) {
    const int slot = w.slots[seq];
    return slot < 0 || slot >= w.n_slots ? nullptr : w.weights + ((size_t)slot * n_kv + hk) * w.places;
}

// Chunks of the rows that see the block of keys at key0.
__host__ __device__ inline int block_chunks(int q_len, int length, int key0, int group, int chunk_rows) {
    const int tokens = q_len < length - key0 ? q_len : length - key0;
    return tokens > 0 ? (tokens * group + chunk_rows - 1) / chunk_rows : 0;
}

// Blocks that all of a run's rows see: every one has as many chunks.
__host__ __device__ inline int full_blocks(int q_len, int length, int keys) { return length >= q_len ? (length - q_len) / keys + 1 : 0; }

// A workgroup's work: a block of keys and rows row_begin .. row_end-1 of a run that begins at token q_begin, place start.
struct Work {
    int seq, q_begin, q_len, length, start, key0, row_begin, row_end;
};

// The index-th piece of work of a run; false if there are not so many.  Behind the blocks that all rows see a lane a block: a walk from one to the next
// would take longer than the work.
template <int KEYS>
__device__ __forceinline__ bool find_work(Work& work, int index, int seq, const int* __restrict__ cu_q, const int* __restrict__ kv_len, int group,
                                          int chunk_rows, int most_keys) {
    const int lane = threadIdx.x % SIA_WAVE, q_begin = cu_q[seq], q_len = cu_q[seq + 1] - q_begin, length = min(kv_len[seq], most_keys);
    const int full = full_blocks(q_len, length, KEYS), each_full = block_chunks(q_len, length, 0, group, chunk_rows);
    if (each_full <= 0) return false;
    auto piece = [&](int key0, int chunk, int chunks) {
        const int tokens = min(q_len, length - key0), rows = tokens * group, first = (q_len - tokens) * group;
        const int each = ((rows + chunks - 1) / chunks + 31) / 32 * 32;
        work = Work{seq, q_begin, q_len, length, length - q_len, key0, first + min(chunk * each, rows), first + min((chunk + 1) * each, rows)};
        return true;
    };
    if (index < full * each_full) return piece(index / each_full * KEYS, index % each_full, each_full);
    index -= full * each_full;
    for (int k0 = full * KEYS; k0 < length; k0 += SIA_WAVE * KEYS) {
        const int mine = block_chunks(q_len, length, k0 + lane * KEYS, group, chunk_rows);
        int upto = mine;
#pragma unroll
        for (int off = 1; off < SIA_WAVE; off *= 2) {
            const int o = __shfl_up(upto, off, SIA_WAVE);
            if (lane >= off) upto += o;
        }
        const unsigned long long behind = __ballot(upto > index);
        if (!behind) {
            index -= __builtin_amdgcn_readlane(upto, SIA_WAVE - 1);
            continue;
        }
        const int at = __builtin_ctzll(behind), chunks = __builtin_amdgcn_readlane(mine, at);
        return piece(k0 + at * KEYS, index - __builtin_amdgcn_readlane(upto, at) + chunks, chunks);
    }
    return false;
}

// A row of a walk that goes on by STEP rows at a time, as its token and query head, without a division.
struct Column {
    int row, token, head;
    __device__ __forceinline__ void begin(int first, int group) {
        row = first;
        token = row / group;
        head = row - token * group;
    }
    template <int STEP>
    __device__ __forceinline__ void next(int by_token, int by_head, int group) {      // STEP / group and STEP % group
        row += STEP;
        token += by_token;
        head += by_head;
        if (head >= group) {
            head -= group;
            ++token;
        }
    }
};

// A thread a key of a block: its chunks' sums in order.  parts: [run][piece of work][key/value head][KEYS], most_work pieces a run.
template <int KEYS>
__global__ __launch_bounds__(KEYS) void weigh_add_kernel(const float* __restrict__ parts, const int* __restrict__ cu_q, const int* __restrict__ kv_len,
                                                         int n_heads, int n_kv, int seq_begin, int chunk_rows, int most_keys, int most_work,
                                                         const Weighed w) {
    const int hk = blockIdx.x, key0 = blockIdx.y * KEYS, seq = seq_begin + blockIdx.z, group = n_heads / n_kv, j = key0 + threadIdx.x;
    const int q_len = cu_q[seq + 1] - cu_q[seq], length = min(kv_len[seq], most_keys), start = length - q_len;
    const int chunks = block_chunks(q_len, length, key0, group, chunk_rows);
    if (chunks <= 0) return;
    // the pieces of the blocks before
    const int full = min(full_blocks(q_len, length, KEYS), (int)blockIdx.y);
    int first = 0;
    for (int k = (full + (int)(threadIdx.x % SIA_WAVE)) * KEYS; k < key0; k += SIA_WAVE * KEYS) first += block_chunks(q_len, length, k, group, chunk_rows);
#pragma unroll
    for (int off = SIA_WAVE / 2; off > 0; off >>= 1) first += __shfl_xor(first, off, SIA_WAVE);
    first += full * block_chunks(q_len, length, 0, group, chunk_rows);
    float* row = weight_row(w, seq, n_kv, hk);
    if (j >= length || !row) return;
    const float old = j < start ? row[j] : 0.f;
    const float* part = parts + (((size_t)blockIdx.z * most_work + first) * n_kv + hk) * KEYS + threadIdx.x;
    const size_t next = (size_t)n_kv * KEYS;
    float sum = 0.f;
    for (int c0 = 0; c0 < chunks; c0 += 8) {      // eight loads under way at a time
        float v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = part[min(c0 + c, chunks - 1) * next];
#pragma unroll
        for (int c = 0; c < 8; ++c) sum += c0 + c < chunks ? v[c] : 0.f;
    }
    row[j] = old + sum;
}

// The sum over the 16 lanes of a row of lanes, in all of them.
__device__ __forceinline__ float row_sum(float x) {
#define ADD_ROTATED(BY) x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x120 + BY, 0xf, 0xf, false))
    ADD_ROTATED(8);
    ADD_ROTATED(4);
    ADD_ROTATED(2);
    ADD_ROTATED(1);
#undef ADD_ROTATED
    return x;
}

// A lane's sums of N blocks of 16 keys from k0 on (rows 4 g .. 4 g + 3 of every block, over its columns), added over the 16 columns and written by a
// lane a key: into the part of its block, or straight into the weights.
template <int N, typename Vec4>
__device__ __forceinline__ void leave_sums(const Vec4 (&sum)[N], int k0, const Work& work, float* part, const Weighed& w, int n_kv, int hk) {
    const int lane = threadIdx.x % SIA_WAVE, r = lane & 15, g = lane >> 4;
    float mine = 0.f;
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float total = row_sum(sum[b][i]);
            mine = r == 4 * b + i ? total : mine;
        }
    const int j = k0 + (r >> 2) * 16 + g * 4 + (r & 3);
    if (r >= 4 * N || j >= work.length) return;
    if (part) {
        part[j - work.key0] = mine;
        return;
    }
    float* to = weight_row(w, work.seq, n_kv, hk);
    if (to) to[j] = (j < work.start ? to[j] : 0.f) + mine;
}

// How a launch for runs of at most q_bound tokens over at most max_kv keys, total_tokens in all, is cut: chunk_rows (a multiple of 32, at least
// `least`) so that there are some `fill` workgroups, which are on the chip at once, or four times as many where they stay long; most_work, the
// pieces of the largest run; floats of the workspace (0: no block has more than one chunk).
struct Cut {
    int chunk_rows, most_work;
    long long floats;
};
inline Cut cut_runs(int total_tokens, int q_bound, int n_runs, int max_kv, int group, int n_kv, int keys, int least, int fill) {
    const double blocks = ((double)max_kv - q_bound + 0.5 * q_bound) / keys + 1.0, work = (double)total_tokens * group * n_kv * blocks;
    double rows = work / fill;
    if (rows > 4096.0) rows = work / fill / 4.0;
    Cut cut;
    cut.chunk_rows = rows < least ? least : rows > 1e9 ? 1 << 30 : ((int)rows + 31) / 32 * 32;
    const int full = full_blocks(q_bound, max_kv, keys);
    cut.most_work = full * block_chunks(q_bound, max_kv, 0, group, cut.chunk_rows);
    for (long long key0 = (long long)full * keys; key0 < max_kv; key0 += keys) cut.most_work += block_chunks(q_bound, max_kv, (int)key0, group, cut.chunk_rows);
    cut.floats = (long long)q_bound * group <= cut.chunk_rows ? 0 : (long long)n_runs * cut.most_work * n_kv * keys;
    return cut;
}
