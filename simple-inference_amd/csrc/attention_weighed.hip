// How much attention weight every cached key got in a step, added to a running sum per (sequence, key/value head, place):
//
//   weights[slot][g][j]  +=  sum over the sequence's tokens t and the query heads h of g of  p[t, h, j]
//   p[t, h, j] = exp(scale q[t, h] . k[j] - lse[t, h])   for j <= the token's place, else 0
//
// The attention that made the output leaves lse (m + log(l) of its softmax, in units of log2: `row_stats`), so that no second pass over
// the values is needed, only the scores again.  A place that the step itself has written begins at zero, whatever lay there.
// All sums are float, each made by one thread in a fixed order.
//
// The plain kernel: a wave for 64 consecutive places of one (sequence, key/value head), a lane a key; the queries come one after
// the other through LDS.  It takes every head size, page size and type.
#include "common.h"

#define WEIGH_MAX_HEAD_DIM 640

// Where the sums of one (sequence, head) lie; null for a slot that is none.
__device__ __forceinline__ float* weight_row(float* weights, const int* __restrict__ slots, int n_slots, int places, int seq, int n_kv, int hk) {
    const int slot = slots[seq];
    return slot < 0 || slot >= n_slots ? nullptr : weights + ((size_t)slot * n_kv + hk) * places;
}

template <typename T>
__global__ __launch_bounds__(SIA_WAVE) void weigh_plain_kernel(
    const T* __restrict__ q, int q_row_stride, const T* __restrict__ k_pages, const int* __restrict__ block_table, int table_width,
    const int* __restrict__ cu_q, const int* __restrict__ kv_len, const int* __restrict__ slots, const float* __restrict__ row_stats,
    float* __restrict__ weights, int n_slots, int places, int n_heads, int n_kv, int head_dim, int page_size, int n_pages, float scale) {
    __shared__ float q_s[WEIGH_MAX_HEAD_DIM];
    const int lane = threadIdx.x, hk = blockIdx.y, seq = blockIdx.z, group = n_heads / n_kv;
    const int first = cu_q[seq], n = cu_q[seq + 1] - first, length = min(kv_len[seq], places), start = length - n;
    const int j0 = blockIdx.x * SIA_WAVE, j = j0 + lane;
    float* row = weight_row(weights, slots, n_slots, places, seq, n_kv, hk);
    if (j0 >= length || !row) return;
    int page = j < length && j / page_size < table_width ? block_table[(size_t)seq * table_width + j / page_size] : -1;
    if (page >= n_pages) page = -1;
    const T* key = k_pages + (((size_t)max(page, 0) * n_kv + hk) * page_size + j % page_size) * head_dim;
    float sum = 0.f;
    for (int t = max(0, j0 - start); t < n; ++t)
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
    if (j < length) row[j] = (j < start ? row[j] : 0.f) + sum;
}

// q: rows of the step's tokens, n_heads * head_dim columns first; cu_q, kv_len, slots: per sequence; row_stats [tokens][n_heads];
// weights [n_slots][n_kv][places]; max_kv: no sequence holds more (what the grid is sized by).
SIA_EXPORT int sia_weigh_plain(const void* q, int q_row_stride, const void* k_pages, const int* block_table, int table_width,
                               const int* cu_q, const int* kv_len, const int* slots, const float* row_stats, float* weights,
                               int n_slots, int places, int n_seqs, int max_kv, int n_heads, int n_kv, int head_dim, int page_size,
                               int n_pages, float scale, int dtype, hipStream_t stream) {
    if (n_seqs <= 0 || max_kv <= 0) return 0;
    if (head_dim <= 0 || head_dim > WEIGH_MAX_HEAD_DIM || n_kv <= 0 || n_heads % n_kv || page_size <= 0 || n_kv > 65535 || n_seqs > 65535 ||
        places <= 0 || table_width <= 0 || n_pages <= 0)
        return SIA_BAD_ARGUMENT;
    const dim3 grid((max_kv + SIA_WAVE - 1) / SIA_WAVE, n_kv, n_seqs);
#define LAUNCH(T)                                                                                                                   \
    hipLaunchKernelGGL(weigh_plain_kernel<T>, grid, dim3(SIA_WAVE), 0, stream, (const T*)q, q_row_stride, (const T*)k_pages,        \
                       block_table, table_width, cu_q, kv_len, slots, row_stats, weights, n_slots, places, n_heads, n_kv, head_dim, \
                       page_size, n_pages, scale)
    if (dtype == SIA_F32) LAUNCH(float);
    else if (dtype == SIA_BF16) LAUNCH(bf16_t);
    else return SIA_BAD_ARGUMENT;
#undef LAUNCH
    return SIA_LAUNCH_CHECK();
}
