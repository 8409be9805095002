// What the kernels that add up the cached keys' attention weight share (attention_weighed.hip, attention_weighed_mfma.hip): where the sums
// lie, and how runs of tokens are cut into chunks of rows.
//
// The rows of a key/value head are a sequence's (token, query head) pairs, token by token; a row sees the keys up to its token's place.  A
// workgroup has a block of keys and walks the rows of one chunk; the chunks' sums are added in order by a kernel of their own.
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

// A run: its rows, its keys, and the chunk of its rows that a workgroup has.
struct Run {
    int seq, chunk, q_begin, q_len, length, start, row_end;
};

// The run and chunk of the index-th chunk of sequences seq_begin .. seq_end-1; false if there are not so many.
__device__ __forceinline__ bool find_run(Run& run, int index, const int* __restrict__ cu_q, const int* __restrict__ kv_len, int seq_begin, int seq_end,
                                         int group, int chunk_rows, int most_keys) {
    int seq = seq_begin;
    for (; seq < seq_end; ++seq) {
        const int chunks = ((cu_q[seq + 1] - cu_q[seq]) * group + chunk_rows - 1) / chunk_rows;
        if (index < chunks) break;
        index -= chunks;
    }
    if (seq >= seq_end) return false;
    const int q_begin = cu_q[seq], q_len = cu_q[seq + 1] - q_begin, length = min(kv_len[seq], most_keys);
    run = Run{seq, index, q_begin, q_len, length, length - q_len, min((index + 1) * chunk_rows, q_len * group)};
    return true;
}

// Whether the chunk of rows that ends before row_end has a row that sees a key of the block at key0: the same for the kernel that writes a
// block's sums and the one that reads them.
__device__ __forceinline__ bool chunk_sees(int row_end, int group, int start, int key0) { return start + (row_end - 1) / group >= key0; }

// A lane's column of a walk over rows, 16 rows at a time, as its token and query head: goes on without a division.
struct Column {
    int row, token, head;
    __device__ __forceinline__ void begin(int first, int group) {
        row = first;
        token = row / group;
        head = row - token * group;
    }
    __device__ __forceinline__ void next(int by_token, int by_head, int group) {      // 16 / group and 16 % group
        row += 16;
        token += by_token;
        head += by_head;
        if (head >= group) {
            head -= group;
            ++token;
        }
    }
};

// A thread a key: the sums of the chunks that see its block of RUN_KEYS keys, in order.  parts: [chunk][key/value head][row_keys].
constexpr int ADD_THREADS = 256;
template <int RUN_KEYS>
__global__ __launch_bounds__(ADD_THREADS) void weigh_runs_add_kernel(const float* __restrict__ parts, const int* __restrict__ cu_q,
                                                                     const int* __restrict__ kv_len, int n_heads, int n_kv, int seq_begin,
                                                                     int chunk_rows, int most_keys, const Weighed w) {
    const int hk = blockIdx.y, seq = seq_begin + blockIdx.z, group = n_heads / n_kv, j = blockIdx.x * ADD_THREADS + threadIdx.x;
    const int q_len = cu_q[seq + 1] - cu_q[seq], length = min(kv_len[seq], most_keys), start = length - q_len;
    if (j >= length || q_len <= 0) return;
    int first = 0;      // this sequence's first chunk
    for (int s = seq_begin; s < seq; ++s) first += ((cu_q[s + 1] - cu_q[s]) * group + chunk_rows - 1) / chunk_rows;
    const int rows = q_len * group, chunks = (rows + chunk_rows - 1) / chunk_rows;
    float* row = weight_row(w, seq, n_kv, hk);
    if (!row) return;
    float sum = 0.f;
    for (int c = 0; c < chunks; ++c)
        if (chunk_sees(min((c + 1) * chunk_rows, rows), group, start, j / RUN_KEYS * RUN_KEYS)) sum += parts[((size_t)(first + c) * n_kv + hk) * w.row_keys + j];
    row[j] = (j < start ? row[j] : 0.f) + sum;
}

// A lane's sums of N blocks of 16 keys (rows 4 g .. 4 g + 3 of every block, over its columns), added over the 16 columns and written: into the chunk's
// part, or straight into the weights of a run of one chunk.
template <int N, typename Vec4>
__device__ __forceinline__ void leave_sums(Vec4 (&sum)[N], int k0, const Run& run, float* part, const Weighed& w, int n_kv, int hk) {
    const int lane = threadIdx.x % SIA_WAVE, r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int off = 1; off < 16; off *= 2) sum[b][i] += __shfl_xor(sum[b][i], off, SIA_WAVE);
    float* to = part ? part : weight_row(w, run.seq, n_kv, hk);
    if (r != 0 || !to) return;
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = k0 + b * 16 + g * 4 + i;
            if (j < run.length) to[j] = (part || j >= run.start ? 0.f : to[j]) + sum[b][i];
        }
}
