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

// What the kernels are given.
template <typename T>
struct RopeAxes {
    T* qkv;
    T *k_pages, *v_pages;
    const float *cos_table, *sin_table;
    const int *rotary_positions, *positions, *seq_of_token, *block_table;
    int row_stride, table_rows, table_width, n_pages, n_tokens, n_heads, n_kv, head_dim, rotary_dim, page_size;
    Axes axes;
};

// The page of a token's place and the offset in it; page -1 where there is nothing to write to.
template <typename T>
__device__ __forceinline__ int page_of(const RopeAxes<T>& a, int token, int& off) {
    off = 0;
    if (a.n_kv == 0) return -1;
    const int place = a.positions[token], index = place / a.page_size;
    off = place - index * a.page_size;
    if (place < 0 || index >= a.table_width) return -1;
    const int page = a.block_table[(size_t)a.seq_of_token[token] * a.table_width + index];
    return page >= a.n_pages ? -1 : page;
}

template <typename T>
__device__ __forceinline__ void angle_of(const RopeAxes<T>& a, int token, int pair, float& c, float& s) {
    const int row = min(max(a.rotary_positions[(size_t)axis_of(a.axes, pair) * a.n_tokens + token], 0), a.table_rows - 1);
    const size_t at = (size_t)row * (a.rotary_dim / 2) + pair;
    c = a.cos_table[at];
    s = a.sin_table[at];
}

// The plain kernel: a workgroup a token, an element a thread at a time.
template <typename T>
__global__ __launch_bounds__(256) void rope_axes_kernel(const RopeAxes<T> a, int neighbours) {
    const int n = blockIdx.x, half = a.rotary_dim / 2;
    T* row = a.qkv + (size_t)n * a.row_stride;
    int off;
    const int page = page_of(a, n, off);
    for (int i = threadIdx.x; i < (a.n_heads + a.n_kv) * half; i += blockDim.x) {
        const int h = i / half, j = i % half;
        const int first = neighbours ? 2 * j : j, second = neighbours ? 2 * j + 1 : j + half;
        T* x = row + h * a.head_dim;
        float c, s, p, q;
        angle_of(a, n, j, c, s);
        rotate_pair(to_float(x[first]), to_float(x[second]), c, s, p, q);
        if (h >= a.n_heads) {
            if (page < 0) continue;
            x = a.k_pages + (((size_t)page * a.n_kv + h - a.n_heads) * a.page_size + off) * a.head_dim;
        }
        x[first] = from_float<T>(p);
        x[second] = from_float<T>(q);
    }
    if (page < 0) return;
    const T* k_row = row + a.n_heads * a.head_dim;
    const T* v_row = k_row + a.n_kv * a.head_dim;
    for (int i = threadIdx.x; i < a.n_kv * a.head_dim; i += blockDim.x) {
        const int h = i / a.head_dim, d = i % a.head_dim;
        if (d >= a.rotary_dim) a.k_pages[(((size_t)page * a.n_kv + h) * a.page_size + off) * a.head_dim + d] = k_row[i];
        a.v_pages[(((size_t)page * a.n_kv + h) * a.head_dim + d) * a.page_size + off] = v_row[i];
    }
}

// Sixteen bytes of a row: the elements of a piece.
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int N = 4;
    float4 v;
    __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w; }
    __device__ __forceinline__ void set(const float (&x)[4]) { v = make_float4(x[0], x[1], x[2], x[3]); }
};
template <> struct Piece<bf16_t> {
    static constexpr int N = 8;
    uint4 v;
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void set(const float (&x)[8]) {
        v = make_uint4(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]), bf16_pair(x[6], x[7]));
    }
};

// The same in pieces of 16 bytes (head size, row stride and the rotated part in pieces; see `pieces` below).  Two kinds of workgroup:
//   values    tiles of GROUP consecutive tokens by VALUE_ROWS rows (key/value head, dim).  Positions are innermost in a value page, so GROUP tokens
//             that fill an aligned stretch of a page go through LDS and leave it as 16 bytes a lane, neighbouring lanes neighbouring bytes;  a tile
//             has at most one such group beginning in it, and tokens of no whole group are written one by one.  (vt = 1: no groups at all.)
//   rotation  TOKENS tokens: their angles come to LDS once, gathered axis by axis, and serve all heads; a thread has one piece of a head and
//             walks the heads, the pieces of all its tokens under way at a time.
// What bounds a long step is the memory: 16,411 rows of 32 + 2 x 8 heads of 128 in bfloat16 move 412 MB in 93 us (4.4 TB/s; the plain kernel 232), 2,048
// rows of 24 + 2 x 8 43 MB in 11.6 (22.5).  A short one is a chain of loads: 8 rows 3.8 us (7.8).  Steps of fewer than
// 512 tokens have a token a workgroup, so that there are enough of them.
constexpr int TOKENS = 4, MAX_HALF = 256, VALUE_GROUP = 16;

template <typename T>
__device__ __forceinline__ void write_values(const RopeAxes<T>& a, int tile, int chunk, int group, int tid, int n_threads, T* lds) {
    constexpr int N = Piece<T>::N, ROWS = 16384 / sizeof(T) / VALUE_GROUP, STRIDE = ROWS + N;
    const int rows = a.n_kv * a.head_dim, row0 = chunk * ROWS, n_rows = min(ROWS, rows - row0), t0 = tile * group, lane = tid % SIA_WAVE;
    const T* values = a.qkv + (size_t)(a.n_heads + a.n_kv) * a.head_dim + row0;
    // lane i < group of the first wave (others may have fewer lanes): token t0 + i, and whether the aligned stretch of places that it belongs to
    // is whole in this step
    __shared__ int pages_s[VALUE_GROUP], offs_s[VALUE_GROUP], singles_s[VALUE_GROUP], n_singles, group_at;
    if (tid < SIA_WAVE) {
        const int token = min(t0 + lane % group, a.n_tokens - 1), place = a.positions[token], seq = a.seq_of_token[token];
        const int first = token - place % group, last = first + group - 1;
        bool whole = group > 1 && place >= 0 && first >= 0 && last < a.n_tokens;
        if (whole) whole = a.seq_of_token[first] == seq && a.seq_of_token[last] == seq && a.positions[first] == place - place % group && a.positions[last] == a.positions[first] + group - 1;
        const bool mine = lane < group && t0 + lane < a.n_tokens;
        int off;
        const int page = page_of(a, token, off);
        if (lane < group) pages_s[lane] = page, offs_s[lane] = off;
        const unsigned long long alone = __ballot(mine && !whole), starts = __ballot(mine && whole && place % group == 0);
        if (alone >> lane & 1) singles_s[__popcll(alone & ((1ull << lane) - 1))] = lane;
        if (lane == 0) {
            n_singles = __popcll(alone);
            group_at = starts ? __builtin_ctzll(starts) : -1;
        }
    }
    __syncthreads();
    if (group_at >= 0) {
        const int begin = t0 + group_at, page = pages_s[group_at], off = offs_s[group_at];
        const int pieces = n_rows / N;
        for (int i = tid; i < group * pieces; i += n_threads) {
            const int t = i / pieces, c = i - t * pieces;
            *reinterpret_cast<uint4*>(lds + t * STRIDE + c * N) = *reinterpret_cast<const uint4*>(values + (size_t)(begin + t) * a.row_stride + c * N);
        }
        __syncthreads();
        const int parts = group / N;      // 16-byte pieces of a row's stretch
        T* out = a.v_pages + ((size_t)max(page, 0) * rows + row0) * a.page_size + off;
        for (int i = tid; page >= 0 && i < n_rows * parts; i += n_threads) {
            const int r = i / parts, part = i - r * parts;
            __attribute__((aligned(16))) T x[N];
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = lds[(part * N + j) * STRIDE + r];
            *reinterpret_cast<uint4*>(out + (size_t)r * a.page_size + part * N) = *reinterpret_cast<const uint4*>(x);
        }
    }
    const int many = n_singles * n_rows;
    for (int i0 = tid; i0 < many; i0 += 4 * n_threads) {      // four elements under way at a time
        T x[4];
        T* to[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = min(i0 + e * n_threads, many - 1), nth = i / n_rows, r = i - nth * n_rows, at = singles_s[nth];
            x[e] = values[(size_t)(t0 + at) * a.row_stride + r];
            to[e] = i0 + e * n_threads < many && pages_s[at] >= 0 ? a.v_pages + ((size_t)pages_s[at] * rows + row0 + r) * a.page_size + offs_s[at] : nullptr;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (to[e]) *to[e] = x[e];
    }
}

template <typename T, int T_TOKENS, bool NEIGHBOURS>
__global__ __launch_bounds__(256) void rope_axes_pieces_kernel(const RopeAxes<T> a, int value_tiles, int value_chunks, int group) {
    constexpr int N = Piece<T>::N, PAIRS = NEIGHBOURS ? N / 2 : N, SIDES = NEIGHBOURS ? 1 : 2;      // pairs of an item; its pieces
    __shared__ __attribute__((aligned(16))) unsigned char lds[16384 + VALUE_GROUP * 16];
    const int tid = threadIdx.y * blockDim.x + threadIdx.x, n_threads = blockDim.x * blockDim.y;
    if ((int)blockIdx.x < value_tiles * value_chunks) {
        const int tile = blockIdx.x / value_chunks;
        write_values(a, tile, blockIdx.x - tile * value_chunks, group, tid, n_threads, reinterpret_cast<T*>(lds));
        return;
    }
    const int half = a.rotary_dim / 2, t0 = ((int)blockIdx.x - value_tiles * value_chunks) * T_TOKENS, many = min(T_TOKENS, a.n_tokens - t0);
    float* const cos_s = reinterpret_cast<float*>(lds);
    float* const sin_s = cos_s + T_TOKENS * half;
    T* const row = a.qkv + (size_t)t0 * a.row_stride;
    const int piece = threadIdx.x, at = piece * N, heads = a.n_heads + a.n_kv;
    // the first head's pieces are on their way while the angles come
    Piece<T> x[T_TOKENS][SIDES];
    auto load = [&](int h) {
#pragma unroll
        for (int t = 0; t < T_TOKENS; ++t)
#pragma unroll
            for (int e = 0; e < SIDES; ++e)
                x[t][e].v = *reinterpret_cast<const decltype(x[t][e].v)*>(row + (size_t)min(t, many - 1) * a.row_stride + h * a.head_dim + at + e * half);
    };
    int h = threadIdx.y;
    if (h < heads) load(h);
    int page[T_TOKENS], off[T_TOKENS];
#pragma unroll
    for (int t = 0; t < T_TOKENS; ++t) page[t] = page_of(a, t0 + min(t, many - 1), off[t]);
    for (int i = tid; i < many * half; i += n_threads) {
        const int t = i / half;
        angle_of(a, t0 + t, i - t * half, cos_s[i], sin_s[i]);
    }
    __syncthreads();
    for (; h < heads;) {
#pragma unroll
        for (int t = 0; t < T_TOKENS; ++t) {
            if (t >= many) break;
            const float* c = cos_s + t * half + piece * PAIRS;
            const float* s = sin_s + t * half + piece * PAIRS;
            if constexpr (NEIGHBOURS) {
                float v[N];
                x[t][0].get(v);
#pragma unroll
                for (int i = 0; i < PAIRS; ++i) {
                    float p, q;
                    rotate_pair(v[2 * i], v[2 * i + 1], c[i], s[i], p, q);
                    v[2 * i] = p;
                    v[2 * i + 1] = q;
                }
                x[t][0].set(v);
            } else {
                float v[N], w[N];
                x[t][0].get(v);
                x[t][1].get(w);
#pragma unroll
                for (int i = 0; i < PAIRS; ++i) {
                    float p, q;
                    rotate_pair(v[i], w[i], c[i], s[i], p, q);
                    v[i] = p;
                    w[i] = q;
                }
                x[t][0].set(v);
                x[t][1].set(w);
            }
            T* to = h < a.n_heads ? row + (size_t)t * a.row_stride + h * a.head_dim
                    : page[t] < 0 ? nullptr
                                  : a.k_pages + (((size_t)page[t] * a.n_kv + h - a.n_heads) * a.page_size + off[t]) * a.head_dim;
#pragma unroll
            for (int e = 0; e < SIDES; ++e)
                if (to) *reinterpret_cast<decltype(x[t][e].v)*>(to + at + e * half) = x[t][e].v;
        }
        h += blockDim.y;
        if (h < heads) load(h);
    }
    // dims of k beyond the rotation
    const int plain = (a.head_dim - a.rotary_dim) / N;
    for (int i = tid; i < many * a.n_kv * plain; i += n_threads) {
        const int t = i / (a.n_kv * plain), rest = i - t * a.n_kv * plain, g = rest / plain, d = a.rotary_dim + (rest - g * plain) * N;
        int at_page;
        const int to = page_of(a, t0 + t, at_page);
        if (to >= 0)
            *reinterpret_cast<uint4*>(a.k_pages + (((size_t)to * a.n_kv + g) * a.page_size + at_page) * a.head_dim + d) =
                *reinterpret_cast<const uint4*>(row + (size_t)t * a.row_stride + (a.n_heads + g) * a.head_dim + d);
    }
}

template <typename T>
static int launch(const RopeAxes<T>& a, bool neighbours, hipStream_t stream) {
    constexpr int N = Piece<T>::N;
    const int half = a.rotary_dim / 2, items = neighbours ? a.rotary_dim / N : half / N;      // of a head
    const bool pieces = a.head_dim % N == 0 && (neighbours ? a.rotary_dim : half) % N == 0 && a.row_stride % N == 0 && half <= MAX_HALF &&
                        ((uintptr_t)a.qkv | (uintptr_t)a.k_pages | (uintptr_t)a.v_pages) % 16 == 0;
    if (!pieces) {
        hipLaunchKernelGGL(rope_axes_kernel<T>, dim3(a.n_tokens), dim3(256), 0, stream, a, neighbours ? 1 : 0);
        return SIA_LAUNCH_CHECK();
    }
    // tokens whose values are written together: 16 or 8 that fill an aligned stretch of a page, if the step is long enough to have such
    const int group = a.n_tokens < 32 ? 1 : a.page_size % 16 == 0 ? 16 : a.page_size % 8 == 0 ? 8 : 1;
    const int rows_at_once = 16384 / (int)sizeof(T) / VALUE_GROUP, chunks = a.n_kv ? (a.n_kv * a.head_dim + rows_at_once - 1) / rows_at_once : 0;
    const int tiles = a.n_kv ? (a.n_tokens + group - 1) / group : 0, tokens = a.n_tokens < 512 ? 1 : TOKENS;
    const dim3 block(items, max(1, 256 / items)), grid(tiles * chunks + (a.n_tokens + tokens - 1) / tokens);
#define LAUNCH(TOK, NB) hipLaunchKernelGGL((rope_axes_pieces_kernel<T, TOK, NB>), grid, block, 0, stream, a, tiles, chunks, group)
    if (neighbours) {
        if (tokens == 1) LAUNCH(1, true);
        else LAUNCH(TOKENS, true);
    } else {
        if (tokens == 1) LAUNCH(1, false);
        else LAUNCH(TOKENS, false);
    }
#undef LAUNCH
    return SIA_LAUNCH_CHECK();
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
#define ARGS(T)                                                                                                                            \
    RopeAxes<T>{(T*)qkv, (T*)k_pages, (T*)v_pages, cos_table, sin_table, rotary_positions, positions, seq_of_token, block_table, row_stride, \
                table_rows, table_width, n_pages, n_tokens, n_heads, n_kv, head_dim, rotary_dim, page_size, axes}
    if (dtype == SIA_F32) return launch(ARGS(float), neighbours, stream);
    if (dtype == SIA_BF16) return launch(ARGS(bf16_t), neighbours, stream);
#undef ARGS
    return SIA_BAD_ARGUMENT;
}
