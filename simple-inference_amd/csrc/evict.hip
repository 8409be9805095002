// Dropping what got least attention from a paged cache: of every sequence with more than `budget` places, and for every key/value head,
// the first `keep_first` places stay, the last `keep_last`, and of those between the ones with the largest weight (ties: the lowest
// place; a NaN counts as minus infinity).
//
// Attention does not ask in which order a sequence's past lies in its pages, so as little as possible is moved: with edge = budget -
// keep_last, what is kept below the edge stays where it is; the kept places from the edge on, but for the last, fill the holes below it,
// both in order; and the last keep_last move up together to the edge, so that the next eviction finds them at the end again.
//
// select: a workgroup per (sequence, head): the threshold by radix selection over ordered float keys (11 + 11 + 10 bits), then one ordered
// walk that lists holes and movers.  move: a workgroup per (sequence, head, slice of a row): nobody else touches these bytes, so that
// the holes can be filled (their sources lie at or beyond the edge, their targets below it) and then the last moved up, tile after tile,
// in place.
#include "common.h"

typedef long long ll;
#define SELECT_THREADS 1024
#define SELECT_WAVES (SELECT_THREADS / SIA_WAVE)
#define BINS 2048

// Larger floats have larger keys; both zeros have the same.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Sum of v over the threads before this one, and (in total) over all; scratch: SELECT_WAVES ints.
__device__ __forceinline__ int block_prefix(int v, int* scratch, int& total) {
    const int lane = threadIdx.x % SIA_WAVE, wave = threadIdx.x / SIA_WAVE;
    int s = v;
#pragma unroll
    for (int off = 1; off < SIA_WAVE; off *= 2) {
        const int o = __shfl_up(s, off, SIA_WAVE);
        if (lane >= off) s += o;
    }
    if (lane == SIA_WAVE - 1) scratch[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < SELECT_WAVES; ++w) {
        if (w < wave) before += scratch[w];
        total += scratch[w];
    }
    __syncthreads();
    return before + s - v;
}

__global__ __launch_bounds__(SELECT_THREADS) void evict_select_kernel(
    const float* __restrict__ weights, const int* __restrict__ slots, const int* __restrict__ kv_len, int n_slots, int places, int max_kv,
    int n_kv, int budget, int keep_first, int keep_last, int max_moves, int* __restrict__ kept, int* __restrict__ lengths,
    int* __restrict__ from, int* __restrict__ to, int* __restrict__ n_moves) {
    __shared__ int bins[BINS];
    __shared__ int scratch[SELECT_WAVES];
    __shared__ uint32_t found[2];      // the digits so far; how many of the places that match them are still wanted
    const int hk = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
    const size_t unit = (size_t)seq * n_kv + hk;
    const int slot = slots[seq], length = max(0, min(kv_len[seq], min(max_kv, places)));
    if (hk == 0 && tid == 0) lengths[seq] = min(length, budget);
    int* keep_row = kept + unit * budget;
    if (length <= budget || slot < 0 || slot >= n_slots) {
        for (int i = tid; i < budget; i += SELECT_THREADS) keep_row[i] = i < length ? i : -1;
        if (tid == 0) n_moves[unit] = -1;      // nothing moves, the last places neither
        return;
    }
    const float* w = weights + ((size_t)slot * n_kv + hk) * places;
    const int lo = keep_first, hi = length - keep_last, edge = budget - keep_last;      // between: lo .. hi - 1
    const int wanted = edge - lo;                                                        // fewer than there are
    uint32_t digits = 0;
    int left = wanted;
    if (wanted > 0)
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, size = pass == 2 ? 1024 : 2048;
            for (int i = tid; i < BINS; i += SELECT_THREADS) bins[i] = 0;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += SELECT_THREADS) {
                const uint32_t key = order_key(w[j]);
                if (pass == 0 || key >> (pass == 1 ? 21 : 10) == digits) atomicAdd(&bins[(key >> shift) & (size - 1)], 1);
            }
            __syncthreads();
            // the largest digit with `left` places at or above it: threads take two bins each from the top
            const int top = BINS - 1 - 2 * tid, a = bins[top], b = bins[top - 1];
            int total;
            const int above = block_prefix(a + b, scratch, total);
            if (above < left && above + a + b >= left) {
                const bool first = above + a >= left;
                found[0] = first ? top : top - 1;
                found[1] = left - (first ? above : above + a);
            }
            __syncthreads();
            digits = digits << (pass == 2 ? 10 : 11) | found[0];
            left = found[1];
            __syncthreads();
        }
    // keys above `digits` are kept, and of those equal to it the `left` lowest places
    int ties = 0, holes = 0, movers = 0;
    for (int j0 = 0; j0 < hi; j0 += SELECT_THREADS) {
        const int j = j0 + tid;
        const uint32_t key = j >= lo && j < hi ? order_key(w[j]) : 0;
        const bool tie = wanted > 0 && j >= lo && j < hi && key == digits;
        int total;
        const int rank = ties + block_prefix(tie, scratch, total);
        ties += total;
        const bool keep = j < lo || (j < hi && wanted > 0 && (key > digits || (tie && rank < left)));
        const bool hole = !keep && j < edge, mover = keep && j >= edge;
        const int at = block_prefix(hole | (int)mover << 16, scratch, total);
        if (hole && holes + (at & 0xffff) < max_moves) to[unit * max_moves + holes + (at & 0xffff)] = j;
        if (mover && movers + (at >> 16) < max_moves) from[unit * max_moves + movers + (at >> 16)] = j;
        if (keep && j < edge) keep_row[j] = j;
        holes += total & 0xffff;
        movers += total >> 16;
    }
    __syncthreads();
    const int moves = min(movers, max_moves);
    for (int i = tid; i < moves; i += SELECT_THREADS) keep_row[to[unit * max_moves + i]] = from[unit * max_moves + i];
    for (int i = tid; i < keep_last; i += SELECT_THREADS) keep_row[edge + i] = hi + i;
    if (tid == 0) n_moves[unit] = moves;
}

// A sequence's pages and one head of them.
struct Place {
    const int* table;
    int table_width, n_pages, n_kv, hk, page_size, page_log2;
    // index of (page, head) and the place within; negative: no page
    __device__ __forceinline__ ll find(int place, int& off) const {
        const int index = page_log2 >= 0 ? place >> page_log2 : place / page_size;
        off = page_log2 >= 0 ? place & (page_size - 1) : place % page_size;
        const int page = index < table_width ? table[index] : -1;
        return page < 0 || page >= n_pages ? -1 : (ll)page * n_kv + hk;
    }
};

// Pieces of a key's row: `count` pieces P from `first` on.
template <typename P>
struct KeyPieces {
    static constexpr int MOST = 4;
    P* pages;
    Place at;
    int first, count, row;      // pieces of a row
    P held[MOST];
    __device__ __forceinline__ P* where(int place) const {
        int off;
        const ll head = at.find(place, off);
        return head < 0 ? nullptr : pages + (head * at.page_size + off) * row + first;
    }
    __device__ __forceinline__ bool load(int place) {
        const P* p = where(place);
#pragma unroll
        for (int i = 0; i < MOST; ++i)
            if (p && i < count) held[i] = p[i];
        return p != nullptr;
    }
    __device__ __forceinline__ void store(int place) const {
        P* p = where(place);
#pragma unroll
        for (int i = 0; i < MOST; ++i)
            if (p && i < count) p[i] = held[i];
    }
};

// Dimensions first .. first + count - 1 of a value.
template <typename T>
struct ValueDims {
    static constexpr int MOST = 16;
    T* pages;
    Place at;
    int first, count, dim;
    T held[MOST];
    __device__ __forceinline__ T* where(int place) const {
        int off;
        const ll head = at.find(place, off);
        return head < 0 ? nullptr : pages + (head * dim + first) * at.page_size + off;
    }
    __device__ __forceinline__ bool load(int place) {
        const T* p = where(place);
#pragma unroll
        for (int i = 0; i < MOST; ++i)
            if (p && i < count) held[i] = p[(size_t)i * at.page_size];
        return p != nullptr;
    }
    __device__ __forceinline__ void store(int place) const {
        T* p = where(place);
#pragma unroll
        for (int i = 0; i < MOST; ++i)
            if (p && i < count) p[(size_t)i * at.page_size] = held[i];
    }
};

struct Sums {
    float* row;
    float held;
    __device__ __forceinline__ bool load(int place) { held = row[place]; return true; }
    __device__ __forceinline__ void store(int place) const { row[place] = held; }
};

// Fills the holes, then moves the last places up.  Every thread of the workgroup comes here.
template <typename Part>
__device__ __forceinline__ void move_part(Part part, const int* __restrict__ from, const int* __restrict__ to, int moves, int hi, int edge,
                                          int keep_last) {
    for (int i = threadIdx.x; i < moves; i += blockDim.x)
        if (part.load(from[i])) part.store(to[i]);
    if (keep_last == 0) return;
    __syncthreads();      // what lay from the edge on is read
    for (int i0 = 0; i0 < keep_last; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        const bool loaded = i < keep_last && part.load(hi + i);
        __syncthreads();  // read by all before any is written; the next tile's sources lie beyond this one's targets
        if (loaded) part.store(edge + i);
    }
}

template <typename T, typename P>
__global__ __launch_bounds__(256) void evict_move_kernel(
    T* k_pages, T* v_pages, float* weights, const int* __restrict__ slots, const int* __restrict__ kv_len,
    const int* __restrict__ block_table, int table_width, int n_pages, int n_slots, int places, int max_kv, int n_kv, int head_dim, int value_dim,
    int page_size, int page_log2, int budget, int keep_last, int key_slices, int value_slices, int max_moves, const int* __restrict__ from,
    const int* __restrict__ to, const int* __restrict__ n_moves) {
    const int hk = blockIdx.x % n_kv, seq = blockIdx.x / n_kv;
    const size_t unit = blockIdx.x;
    const int moves = n_moves[unit];
    if (moves < 0) return;
    const int length = min(kv_len[seq], min(max_kv, places)), hi = length - keep_last, edge = budget - keep_last;
    from += unit * max_moves;
    to += unit * max_moves;
    const Place at{block_table + (size_t)seq * table_width, table_width, n_pages, n_kv, hk, page_size, page_log2};
    int slice = blockIdx.y;
    if (slice < key_slices) {
        constexpr int PER = sizeof(P) / sizeof(T);
        const int row = head_dim / PER, first = slice * KeyPieces<P>::MOST;
        move_part(KeyPieces<P>{(P*)k_pages, at, first, min(KeyPieces<P>::MOST, row - first), row, {}}, from, to, moves, hi, edge, keep_last);
        return;
    }
    slice -= key_slices;
    if (slice < value_slices) {
        const int first = slice * ValueDims<T>::MOST;
        move_part(ValueDims<T>{v_pages, at, first, min(ValueDims<T>::MOST, value_dim - first), value_dim, {}}, from, to, moves, hi, edge, keep_last);
        return;
    }
    move_part(Sums{weights + ((size_t)slots[seq] * n_kv + hk) * places, 0.f}, from, to, moves, hi, edge, keep_last);
}

// Ints that sia_evict's workspace holds.
static int most_moves(int max_kv, int budget, int keep_last) { return max(0, min(budget - keep_last, max_kv - budget)); }
SIA_EXPORT ll sia_evict_workspace(int n_seqs, int max_kv, int n_kv, int budget, int keep_last) {
    return (ll)n_seqs * n_kv * (1 + 2LL * most_moves(max_kv, budget, keep_last));
}

// kv_len: places of each sequence, none more than max_kv; slots: its row of weights [n_slots][n_kv][places]; kept [n_seqs][n_kv][budget]:
// the old place of what lies at a place now, -1 behind the last; lengths [n_seqs]: what is left.
SIA_EXPORT int sia_evict(void* k_pages, void* v_pages, float* weights, const int* slots, const int* kv_len, const int* block_table,
                         int table_width, int n_pages, int n_slots, int places, int n_seqs, int max_kv, int n_kv, int head_dim, int value_dim,
                         int page_size, int budget, int keep_first, int keep_last, int* kept, int* lengths, int* ws, int dtype,
                         hipStream_t stream) {
    if (n_seqs <= 0) return 0;
    if (n_kv <= 0 || n_kv > 65535 || n_seqs > 65535 || (ll)n_seqs * n_kv > 0x7fffffff || head_dim <= 0 || value_dim <= 0 || page_size <= 0 || budget <= 0 || keep_first < 0 ||
        keep_last < 0 || keep_first > budget - keep_last || places <= 0 || max_kv < 0 || max_kv > places || (ll)table_width * page_size < max_kv ||
        n_pages <= 0 || n_slots <= 0 || !ws || (dtype != SIA_F32 && dtype != SIA_BF16))
        return SIA_BAD_ARGUMENT;
    const int max_moves = most_moves(max_kv, budget, keep_last);
    const ll units = (ll)n_seqs * n_kv;
    int *n_moves = ws, *from = ws + units, *to = from + units * max_moves;
    hipLaunchKernelGGL(evict_select_kernel, dim3(n_kv, n_seqs), dim3(SELECT_THREADS), 0, stream, weights, slots, kv_len, n_slots, places, max_kv,
                       n_kv, budget, keep_first, keep_last, max_moves, kept, lengths, from, to, n_moves);
    if (max_kv <= budget) return SIA_LAUNCH_CHECK();      // nothing moves anywhere
    int page_log2 = -1;
    for (int b = 0; b < 31; ++b)
        if (page_size == 1 << b) page_log2 = b;
    // the widest piece that divides a key's row
    const int size = dtype == SIA_F32 ? 4 : 2, bytes = head_dim * size, piece = bytes % 16 == 0 && (uintptr_t)k_pages % 16 == 0 ? 16 : size;
    const int key_slices = (bytes / piece + 3) / 4, value_slices = (value_dim + 15) / 16;
#define LAUNCH(T, P)                                                                                                                    \
    hipLaunchKernelGGL((evict_move_kernel<T, P>), dim3((unsigned)units, key_slices + value_slices + 1), dim3(256), 0, stream, (T*)k_pages, \
                       (T*)v_pages, weights, slots, kv_len, block_table, table_width, n_pages, n_slots, places, max_kv, n_kv, head_dim, \
                       value_dim, page_size, page_log2, budget, keep_last, key_slices, value_slices, max_moves, from, to, n_moves)
    if (key_slices + value_slices + 1 > 65535) return SIA_BAD_ARGUMENT;
    if (dtype == SIA_F32) {
        if (piece == 16) LAUNCH(float, uint4);
        else LAUNCH(float, float);
    } else {
        if (piece == 16) LAUNCH(bf16_t, uint4);
        else LAUNCH(bf16_t, bf16_t);
    }
#undef LAUNCH
    return SIA_LAUNCH_CHECK();
}
