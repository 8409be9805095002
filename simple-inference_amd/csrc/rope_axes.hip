// Rotary positions with several axes (time, height and width of a patch of video, say), fused with the write of k and v into the
// cache pages.  Every rotary pair belongs to one axis, and turns by the angle of the token's position on that axis:
//
//   a' = a cos - b sin,  b' = b cos + a sin,  cos and sin = table[position[axis(pair)][token]][pair]
//
// Where the token is written does not follow from its positions: k and v go to the place ctx.positions[token] of its sequence,
// which is another number once axes run apart or cached tokens have been dropped.
// Pairs are dealt to the axes in blocks (the first counts[0] pairs to axis 0, the next counts[1] to axis 1, ..) or in turn (pair j to
// axis j mod n if that is not axis 0 and it has not yet counts[axis] pairs, else to axis 0).  Elements i and i + rotary_dim / 2 are a
// pair, or neighbours.  float arithmetic, rounded once; elements beyond rotary_dim pass through.
// Page layout as in rope_cache.hip.  A position outside the tables is taken at the nearest row.
#include "common.h"

#define AXES_MAX 4
struct Axes {
    int n, cycled;
    int counts[AXES_MAX];
};

__device__ __forceinline__ int axis_of(const Axes& axes, int pair) {
    if (axes.cycled) {
        const int a = pair % axes.n;
        return a > 0 && pair < axes.n * axes.counts[a] ? a : 0;
    }
    int a = 0;
    for (int end = axes.counts[0]; a + 1 < axes.n && pair >= end; end += axes.counts[a]) ++a;
    return a;
}

// A workgroup a token, an element a thread at a time.
template <typename T>
__global__ __launch_bounds__(256) void rope_axes_kernel(
    T* __restrict__ qkv, int row_stride, const float* __restrict__ cos_table, const float* __restrict__ sin_table, int table_rows,
    const int* __restrict__ rotary_positions, const Axes axes, const int* __restrict__ positions, const int* __restrict__ seq_of_token,
    const int* __restrict__ block_table, int table_width, T* __restrict__ k_pages, T* __restrict__ v_pages, int n_pages, int n_tokens,
    int n_heads, int n_kv, int head_dim, int rotary_dim, int neighbours, int page_size) {
    const int n = blockIdx.x, half = rotary_dim / 2;
    T* row = qkv + (size_t)n * row_stride;
    int page = -1, off = 0;
    if (n_kv > 0) {
        const int place = positions[n];
        if (place >= 0 && place / page_size < table_width) page = block_table[(size_t)seq_of_token[n] * table_width + place / page_size];
        if (page >= n_pages) page = -1;      // nowhere to write
        off = place % page_size;
    }
    for (int i = threadIdx.x; i < (n_heads + n_kv) * half; i += blockDim.x) {
        const int h = i / half, j = i % half;
        const int at = min(max(rotary_positions[(size_t)axis_of(axes, j) * n_tokens + n], 0), table_rows - 1);
        const int first = neighbours ? 2 * j : j, second = neighbours ? 2 * j + 1 : j + half;
        T* x = row + h * head_dim;
        float a, b;
        rotate_pair(to_float(x[first]), to_float(x[second]), cos_table[(size_t)at * half + j], sin_table[(size_t)at * half + j], a, b);
        if (h >= n_heads) {
            if (page < 0) continue;
            x = k_pages + (((size_t)page * n_kv + h - n_heads) * page_size + off) * head_dim;
        }
        x[first] = from_float<T>(a);
        x[second] = from_float<T>(b);
    }
    if (page < 0) return;
    const T* k_row = row + n_heads * head_dim;
    const T* v_row = k_row + n_kv * head_dim;
    for (int i = threadIdx.x; i < n_kv * head_dim; i += blockDim.x) {
        const int h = i / head_dim, d = i % head_dim;
        if (d >= rotary_dim) k_pages[(((size_t)page * n_kv + h) * page_size + off) * head_dim + d] = k_row[i];
        v_pages[(((size_t)page * n_kv + h) * head_dim + d) * page_size + off] = v_row[i];
    }
}

SIA_EXPORT int sia_rope_axes_max() { return AXES_MAX; }

// counts: pairs of each of n_axes axes, rotary_dim / 2 in all; rotary_positions [n_axes][n_tokens]; the tables table_rows x rotary_dim / 2.
SIA_EXPORT int sia_rope_axes_kv_write(void* qkv, int row_stride, const float* cos_table, const float* sin_table, int table_rows,
                                      const int* rotary_positions, const int* counts, int n_axes, int cycled, const int* positions,
                                      const int* seq_of_token, const int* block_table, int table_width, void* k_pages, void* v_pages,
                                      int n_pages, int n_tokens, int n_heads, int n_kv, int head_dim, int rotary_dim, int neighbours,
                                      int page_size, int dtype, hipStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (n_axes <= 0 || n_axes > AXES_MAX || rotary_dim <= 0 || rotary_dim > head_dim || (rotary_dim & 1) || table_rows <= 0 || n_heads < 0 || n_kv < 0)
        return SIA_BAD_ARGUMENT;
    if (n_kv > 0 && (!k_pages || !v_pages || !block_table || page_size <= 0 || table_width <= 0)) return SIA_BAD_ARGUMENT;
    Axes axes{n_axes, cycled ? 1 : 0, {}};
    int pairs = 0;
    for (int a = 0; a < n_axes; ++a) {
        if (counts[a] < 0) return SIA_BAD_ARGUMENT;
        pairs += axes.counts[a] = counts[a];
        // in turn: the axis' last pair lies inside the rotation
        if (cycled && a > 0 && counts[a] > 0 && n_axes * (counts[a] - 1) + a >= rotary_dim / 2) return SIA_BAD_ARGUMENT;
    }
    if (pairs != rotary_dim / 2) return SIA_BAD_ARGUMENT;
#define LAUNCH(T)                                                                                                                      \
    hipLaunchKernelGGL(rope_axes_kernel<T>, dim3(n_tokens), dim3(256), 0, stream, (T*)qkv, row_stride, cos_table, sin_table, table_rows, \
                       rotary_positions, axes, positions, seq_of_token, block_table, table_width, (T*)k_pages, (T*)v_pages, n_pages,   \
                       n_tokens, n_heads, n_kv, head_dim, rotary_dim, neighbours, page_size)
    if (dtype == SIA_F32) LAUNCH(float);
    else if (dtype == SIA_BF16) LAUNCH(bf16_t);
    else return SIA_BAD_ARGUMENT;
#undef LAUNCH
    return SIA_LAUNCH_CHECK();
}
