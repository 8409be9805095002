// Dropping what got least attention from a paged cache: of every sequence with more than `budget` places, and for every key/value head,
// the first `keep_first` places stay, the last `keep_last`, and of those between the ones with the largest weight (ties: the lowest
// place; a NaN counts as minus infinity).
//
// Attention does not ask in which order a sequence's past lies in its pages, so as little as possible is moved: with edge = budget -
// keep_last, what is kept below the edge stays where it is; the kept places from the edge on, but for the last, fill the holes below it,
// both in order; and the last keep_last move up together to the edge, so that the next eviction finds them at the end again.
//
// select: a workgroup per (sequence, head), keys of up to 16,384 places in its registers: the threshold by radix selection over ordered float
// keys (11 + 11 + 10 bits), then holes and movers in order, a wave a stretch of places, so that only the waves' counts cross it.
// move: a workgroup per (sequence, head, slice of a row): nobody else touches these bytes, so that the holes can be filled (their sources lie
// at or beyond the edge, their targets below it) and then the last moved up, tile after tile, in place.  Where there are few sequences, movers from
// beyond the new length, which nothing overwrites, go to further workgroups.
// What bounds both is latency: a chain of loads, each of whose address is the last one's result, and barriers.  us, select and move, 8 key/value heads:
// 8 x 2,112 to 2,048 places, the last 512 kept, heads of 128: 8.2 and 12.7 (39 MB);  one of 16,384 to 4,096 17.5 and 16;  64 of about 700 to 509 in
// float32, heads of 64: 11.6 and 49: a moved value is an element in each of its head's rows of a page, and the memory writes 64 bytes for it.
#include "common.h"

typedef long long ll;
#define SELECT_THREADS 1024
#define SELECT_WAVES (SELECT_THREADS / SIA_WAVE)
#define BINS 2048
#define COPIES 4      // of the histogram: weights crowd into few of the first digit's bins, and lanes that meet in one wait for each other

// Larger floats have larger keys; both zeros have the same.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Sum of v over the lanes up to this one, by moves between lanes within the vector unit (a shuffle goes through LDS and takes ten times as long).
__device__ __forceinline__ int lanes_upto(int v) {
#define ADD_MOVED(CTRL, ROWS) v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false)
    ADD_MOVED(0x111, 0xf);      // rows of 16 lanes, from 1, 2, 4 and 8 lanes below
    ADD_MOVED(0x112, 0xf);
    ADD_MOVED(0x114, 0xf);
    ADD_MOVED(0x118, 0xf);
    ADD_MOVED(0x142, 0xa);      // the last lane of rows 0 and 2 to rows 1 and 3, then that of row 1 to rows 2 and 3
    ADD_MOVED(0x143, 0xc);
#undef ADD_MOVED
    return v;
}

// What the waves' values (the same in all of a wave's lanes) add up to over the waves before this one.  leave, a barrier, then before; nobody may
// still be reading the row of scratch.
__device__ __forceinline__ void leave(int v, int* scratch) {
    if (threadIdx.x % SIA_WAVE == 0) scratch[threadIdx.x / SIA_WAVE] = v;
}
__device__ __forceinline__ int before(const int* scratch, int& all) {
    const int wave = threadIdx.x / SIA_WAVE;
    int sum = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < SELECT_WAVES; ++w) {
        const int x = scratch[w];
        sum += w < wave ? x : 0;
        all += x;
    }
    return sum;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(lanes_upto(v), SIA_WAVE - 1); }

// HELD: places of a wave's stretch that a lane keeps the keys of (64 HELD places a wave); 0: stretches of any length, read again every time.
template <int HELD>
__global__ __launch_bounds__(SELECT_THREADS) void evict_select_kernel(
    const float* __restrict__ weights, const int* __restrict__ slots, const int* __restrict__ kv_len, int n_slots, int places, int max_kv,
    int n_kv, int budget, int keep_first, int keep_last, int max_moves, int* __restrict__ kept, int* __restrict__ lengths,
    int* __restrict__ from, int* __restrict__ to, int2* __restrict__ n_moves) {
    __shared__ int bins[COPIES + 2][BINS];      // of the first digit in copies, of the others
    __shared__ int scratch[7][SELECT_WAVES];    // a row for everything that crosses the waves
    __shared__ uint32_t found[3][2];      // the largest digit that enough places reach; how many of those that have it are still wanted
    const int hk = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid % SIA_WAVE, wave = tid / SIA_WAVE;
    const size_t unit = (size_t)seq * n_kv + hk;
    const int slot = slots[seq], length = max(0, min(kv_len[seq], min(max_kv, places)));
    const bool none = slot < 0 || slot >= n_slots;      // no row of sums: all stays
    if (hk == 0 && tid == 0) lengths[seq] = none ? length : min(length, budget);
    int* keep_row = kept + unit * budget;
    if (length <= budget || none) {
        for (int i = tid; i < budget; i += SELECT_THREADS) keep_row[i] = i < length ? i : -1;
        if (tid == 0) n_moves[unit] = make_int2(-1, -1);      // nothing moves, the last places neither
        return;
    }
    const float* w = weights + ((size_t)slot * n_kv + hk) * places;
    const int lo = keep_first, hi = length - keep_last, edge = budget - keep_last;      // between: lo .. hi - 1
    const int wanted = edge - lo;                                                        // fewer than there are
    from += unit * max_moves;
    to += unit * max_moves;
    // the wave's stretch of the places below hi, 64 of them a step
    const int steps = HELD ? HELD : (hi + SELECT_THREADS - 1) / SELECT_THREADS, begin = wave * steps * SIA_WAVE;
#pragma unroll
    for (int c = 0; c < COPIES + 2; ++c) reinterpret_cast<int2*>(bins[c])[tid] = make_int2(0, 0);
    uint32_t held[HELD ? HELD : 1];
    auto load_key = [&](int j) { return j >= lo && j < hi ? order_key(w[j]) : 0u; };      // no place has the key 0: minus infinity has more
    if constexpr (HELD != 0) {
        float x[HELD];
#pragma unroll
        for (int e = 0; e < HELD; ++e) {
            const int j = begin + e * SIA_WAVE + lane;
            x[e] = w[min(j, hi - 1)];
        }
#pragma unroll
        for (int e = 0; e < HELD; ++e) {
            const int j = begin + e * SIA_WAVE + lane;
            held[e] = j >= lo && j < hi ? order_key(x[e]) : 0u;
        }
    }
    auto key_at = [&](int e) {
        if constexpr (HELD != 0) return held[e];
        else return load_key(begin + e * SIA_WAVE + lane);
    };
    uint32_t digits = 0;
    int left = wanted;
    __syncthreads();
    if (wanted > 0) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, mask = pass == 2 ? 1023 : 2047;
#pragma unroll
            for (int e = 0; e < steps; ++e) {
                const uint32_t key = key_at(e);
                if (key != 0 && (pass == 0 || key >> (pass == 1 ? 21 : 10) == digits))
                    atomicAdd(&bins[pass == 0 ? lane % COPIES : COPIES - 1 + pass][(key >> shift) & mask], 1);
            }
            __syncthreads();
            // threads take two bins each, from the top
            int2 two = make_int2(0, 0);
#pragma unroll
            for (int c = 0; c < (pass == 0 ? COPIES : 1); ++c) {
                const int2 own = reinterpret_cast<const int2*>(bins[pass == 0 ? c : COPIES - 1 + pass])[BINS / 2 - 1 - tid];
                two.x += own.x;
                two.y += own.y;
            }
            const int upto = lanes_upto(two.x + two.y);
            int all;
            leave(__builtin_amdgcn_readlane(upto, SIA_WAVE - 1), scratch[pass]);
            __syncthreads();
            const int above = before(scratch[pass], all) + upto - two.x - two.y;
            if (above < left && above + two.x + two.y >= left) {
                const bool upper = above + two.y >= left;
                found[pass][0] = BINS - 1 - 2 * tid - (upper ? 0 : 1);
                found[pass][1] = left - (upper ? above : above + two.y);
            }
            __syncthreads();
            digits = digits << (pass == 2 ? 10 : 11) | found[pass][0];
            left = found[pass][1];
        }
    }
    // keys above `digits` are kept, and of those equal to it the `left` lowest places (with nothing wanted: none of a key that there is not)
    if (wanted <= 0) digits = 0xffffffffu, left = 0;
    // A wave's stretch: places below lo, between, beyond hi.  First the waves' counts: of ties, and of what is kept but for ties, below the edge, from
    // the edge on, and of that below the new length.
    int ties = 0, stay = 0, beyond = 0, near = 0;      // a lane's own, then the wave's
#pragma unroll
    for (int e = 0; e < steps; ++e) {
        const int j = begin + e * SIA_WAVE + lane;
        const uint32_t key = key_at(e);
        const bool over = key > digits && wanted > 0, tie = key == digits;
        ties += __popcll(__ballot(tie));
        stay += (over || j < lo) && j < edge;
        beyond += over && j >= edge;
        near += over && j >= edge && j < budget;
    }
    int all;
    leave(ties, scratch[3]);
    __syncthreads();
    const int ties_before = before(scratch[3], all);
    const unsigned long long below = (1ull << lane) - 1;
    // of the ties, those with fewer than `left` before them: where they lie matters to the counts only if the wave has some of them and some not
    const int ties_kept = min(max(left - ties_before, 0), ties);
    if (ties_kept > 0) {
        int rank = 0;
#pragma unroll
        for (int e = 0; e < steps; ++e) {
            const int j = begin + e * SIA_WAVE + lane;
            const bool tie = key_at(e) == digits;
            const unsigned long long tied = __ballot(tie);
            if (tied) {
                const bool keep = tie && rank + __popcll(tied & below) < ties_kept;
                stay += keep && j < edge;
                beyond += keep && j >= edge;
                near += keep && j >= edge && j < budget;
                rank += __popcll(tied);
            }
        }
    }
    // the wave's holes: its places below the edge that nothing stays at
    const int reach = steps * SIA_WAVE, upper = min(max(edge - begin, 0), reach);
    leave(upper - wave_total(stay), scratch[4]);
    leave(wave_total(beyond), scratch[5]);
    leave(wave_total(near), scratch[6]);
    __syncthreads();
    int holes = before(scratch[4], all), all_movers, movers = before(scratch[5], all_movers);
    before(scratch[6], all);
    const int total = min(all_movers, max_moves);
    if (tid == 0) n_moves[unit] = make_int2(all, total);
    // then the lists, in order
    int rank = 0;
#pragma unroll
    for (int e = 0; e < steps; ++e) {
        const int j = begin + e * SIA_WAVE + lane;
        const uint32_t key = key_at(e);
        bool keep = j < lo || (key > digits && wanted > 0);
        if (ties_kept > 0) {
            const unsigned long long tied = __ballot(key == digits);
            if (tied) {
                keep |= key == digits && rank + __popcll(tied & below) < ties_kept;
                rank += __popcll(tied);
            }
        }
        const bool hole = !keep && j < edge, mover = keep && j >= edge;
        const unsigned long long h = __ballot(hole), m = __ballot(mover);
        if (h) {
            const int at = holes + __popcll(h & below);
            if (hole && at < max_moves) to[at] = j;
            holes += __popcll(h);
        }
        if (m) {
            const int at = movers + __popcll(m & below);
            if (mover && at < max_moves) from[at] = j;
            movers += __popcll(m);
        }
        if (keep && j < edge) keep_row[j] = j;
    }
    __syncthreads();
    for (int i = tid; i < total; i += SELECT_THREADS) keep_row[to[i]] = from[i];
    for (int i = tid; i < keep_last; i += SELECT_THREADS) keep_row[edge + i] = hi + i;
}

// A sequence's pages and one head of them.  The first entries of its block table lie in LDS: what is moved then waits for one load less.
constexpr int TABLE_HELD = 1024;
struct Place {
    const int *table, *held;
    int table_width, n_pages, n_kv, hk, page_size, page_log2;
    // index of (page, head) and the place within; negative: no page
    __device__ __forceinline__ ll find(int place, int& off) const {
        const int index = page_log2 >= 0 ? place >> page_log2 : place / page_size;
        off = page_log2 >= 0 ? place & (page_size - 1) : place % page_size;
        const int page = index >= table_width ? -1 : index < TABLE_HELD ? held[index] : table[index];
        return page < 0 || page >= n_pages ? -1 : (ll)page * n_kv + hk;
    }
};

constexpr int MOVE_THREADS = 256;
typedef uint32_t piece16 __attribute__((ext_vector_type(4)));      // a plain 16-byte register value

// A slice of a key's row, four pieces P (of 16 bytes, or elements where rows do not lie so): a lane a piece, so that a row's lie in neighbouring lanes.
template <typename P>
struct KeyPieces {
    static constexpr int LANES = 4, BATCH = 4;      // lanes a row (8: 8 x 2,112 to 2,048 12.7 -> 17.6 us); rows of a thread at a time
    P* pages;
    Place at;
    int first, row;      // the slice's first piece, pieces of a row
    P held[BATCH];
    __device__ __forceinline__ P* where(int place) const {
        int off;
        const ll head = at.find(place, off);
        const int piece = first + (int)threadIdx.x % LANES;
        return head < 0 || piece >= row ? nullptr : pages + (head * at.page_size + off) * row + piece;
    }
    __device__ __forceinline__ bool load(int b, int place) {
        const P* p = where(place);
        if (p) held[b] = *p;
        return p != nullptr;
    }
    __device__ __forceinline__ void store(int b, int place) const {
        P* p = where(place);
        if (p) *p = held[b];
    }
};

// Dimensions first .. first + count - 1 of a value, a lane a place.
template <typename T>
struct ValueDims {
    static constexpr int MOST = 16, LANES = 1, BATCH = 2;
    T* pages;
    Place at;
    int first, count, dim;
    T held[BATCH][MOST];
    __device__ __forceinline__ T* where(int place) const {
        int off;
        const ll head = at.find(place, off);
        return head < 0 ? nullptr : pages + (head * dim + first) * at.page_size + off;
    }
    __device__ __forceinline__ bool load(int b, int place) {
        const T* p = where(place);
        if (p) {
#pragma unroll
            for (int i = 0; i < MOST; ++i) held[b][i] = p[(size_t)min(i, count - 1) * at.page_size];
        }
        return p != nullptr;
    }
    __device__ __forceinline__ void store(int b, int place) const {
        T* p = where(place);
        if (!p) return;
#pragma unroll
        for (int i = 0; i < MOST; ++i)
            if (i < count) p[(size_t)i * at.page_size] = held[b][i];
    }
};

struct Sums {
    static constexpr int LANES = 1, BATCH = 2;
    float* row;
    float held[BATCH];
    __device__ __forceinline__ bool load(int b, int place) { held[b] = row[place]; return true; }
    __device__ __forceinline__ void store(int b, int place) const { row[place] = held[b]; }
};

// Moves begin .. end-1 of the lists: from[i] to to[i].
template <typename Part>
__device__ __forceinline__ void fill(Part& part, const int* __restrict__ from, const int* __restrict__ to, int begin, int end) {
    constexpr int ROWS = MOVE_THREADS / Part::LANES;
    for (int i0 = begin + (int)threadIdx.x / Part::LANES; i0 < end; i0 += ROWS * Part::BATCH) {
        int source[Part::BATCH], target[Part::BATCH];
        bool loaded[Part::BATCH];
#pragma unroll
        for (int b = 0; b < Part::BATCH; ++b) {
            const int i = min(i0 + b * ROWS, end - 1);
            source[b] = from[i];
            target[b] = to[i];
        }
#pragma unroll
        for (int b = 0; b < Part::BATCH; ++b) loaded[b] = i0 + b * ROWS < end && part.load(b, source[b]);
#pragma unroll
        for (int b = 0; b < Part::BATCH; ++b)
            if (loaded[b]) part.store(b, target[b]);
    }
}

// A batch of the last places on their way up, from hi + i0 on.
template <typename Part>
struct MoveUp {
    static constexpr int ROWS = MOVE_THREADS / Part::LANES, BATCH = ROWS * Part::BATCH;
    bool loaded[Part::BATCH];
    __device__ __forceinline__ void load(Part& part, int i0, int hi, int keep_last) {
        const int mine = i0 + (int)threadIdx.x / Part::LANES;
#pragma unroll
        for (int b = 0; b < Part::BATCH; ++b) loaded[b] = mine + b * ROWS < keep_last && part.load(b, hi + mine + b * ROWS);
    }
    __device__ __forceinline__ void store(Part& part, int i0, int edge) const {
        const int mine = i0 + (int)threadIdx.x / Part::LANES;
#pragma unroll
        for (int b = 0; b < Part::BATCH; ++b)
            if (loaded[b]) part.store(b, edge + mine + b * ROWS);
    }
};

// A workgroup's share of a part: the first of n_shares has what may be overwritten (all moves, if it is the only one), the others the rest.
template <typename Part>
__device__ __forceinline__ void move_part(Part part, int share, int n_shares, const int* __restrict__ from, const int* __restrict__ to, int2 moves,
                                          int hi, int edge, int keep_last) {
    if (share > 0) {
        const int far = moves.y - moves.x, each = (far + n_shares - 2) / (n_shares - 1);
        fill(part, from, to, moves.x + (share - 1) * each, min(moves.y, moves.x + share * each));
        return;
    }
    // the last places, from hi on, move up to the edge, a batch at a time; the first is read before the holes are filled: nothing is written from hi on
    Part up = part;
    MoveUp<Part> batch;
    batch.load(up, 0, hi, keep_last);
    fill(part, from, to, 0, n_shares == 1 ? moves.y : moves.x);
    for (int i0 = 0; i0 < keep_last; i0 += MoveUp<Part>::BATCH) {
        if (i0 > 0) batch.load(up, i0, hi, keep_last);
        __syncthreads();  // read by all (and what lay from the edge on has filled its holes) before any is written; the next batch's sources lie beyond this one's targets
        batch.store(up, i0, edge);
    }
}

// grid (sequences x heads, slices of keys and values and one for the sums, shares)
template <typename T, typename P>
__global__ __launch_bounds__(MOVE_THREADS) void evict_move_kernel(
    T* k_pages, T* v_pages, float* weights, const int* __restrict__ slots, const int* __restrict__ kv_len,
    const int* __restrict__ block_table, int table_width, int n_pages, int places, int max_kv, int n_kv, int head_dim, int value_dim,
    int page_size, int page_log2, int budget, int keep_last, int key_slices, int value_slices, int max_moves, const int* __restrict__ from,
    const int* __restrict__ to, const int2* __restrict__ n_moves) {
    __shared__ int table_s[TABLE_HELD];
    const int hk = blockIdx.x % n_kv, seq = blockIdx.x / n_kv, share = blockIdx.z, n_shares = gridDim.z;
    const size_t unit = blockIdx.x;
    const int2 moves = n_moves[unit];
    const int* const table = block_table + (size_t)seq * table_width;
#pragma unroll
    for (int i = 0; i < TABLE_HELD; i += MOVE_THREADS)
        if (i + (int)threadIdx.x < table_width) table_s[i + threadIdx.x] = table[i + threadIdx.x];
    __syncthreads();
    const int length = min(kv_len[seq], min(max_kv, places)), hi = length - keep_last, edge = budget - keep_last;
    if (moves.y < 0) return;
    from += unit * max_moves;
    to += unit * max_moves;
    const Place at{table, table_s, table_width, n_pages, n_kv, hk, page_size, page_log2};
    int slice = blockIdx.y;
    if (slice < key_slices) {
        constexpr int PER = sizeof(P) / sizeof(T);
        move_part(KeyPieces<P>{(P*)k_pages, at, slice * KeyPieces<P>::LANES, head_dim / PER, {}}, share, n_shares, from, to, moves, hi, edge, keep_last);
        return;
    }
    slice -= key_slices;
    if (slice < value_slices) {
        const int first = slice * ValueDims<T>::MOST;
        move_part(ValueDims<T>{v_pages, at, first, min(ValueDims<T>::MOST, value_dim - first), value_dim, {}}, share, n_shares, from, to, moves, hi, edge, keep_last);
        return;
    }
    move_part(Sums{weights + ((size_t)slots[seq] * n_kv + hk) * places, {}}, share, n_shares, from, to, moves, hi, edge, keep_last);
}

// Ints that sia_evict's workspace holds.
static int most_moves(int max_kv, int budget, int keep_last) { return max(0, min(budget - keep_last, max_kv - budget)); }
SIA_EXPORT ll sia_evict_workspace(int n_seqs, int max_kv, int n_kv, int budget, int keep_last) {
    return (ll)n_seqs * n_kv * (2 + 2LL * most_moves(max_kv, budget, keep_last));
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
    int2* n_moves = reinterpret_cast<int2*>(ws);
    int *from = ws + 2 * units, *to = from + units * max_moves;
#define SELECT(HELD)                                                                                                                     \
    hipLaunchKernelGGL(evict_select_kernel<HELD>, dim3(n_kv, n_seqs), dim3(SELECT_THREADS), 0, stream, weights, slots, kv_len, n_slots, places, \
                       max_kv, n_kv, budget, keep_first, keep_last, max_moves, kept, lengths, from, to, n_moves)
    if (max_kv <= 2 * SELECT_THREADS) SELECT(2);
    else if (max_kv <= 4 * SELECT_THREADS) SELECT(4);
    else if (max_kv <= 16 * SELECT_THREADS) SELECT(16);
    else SELECT(0);
#undef SELECT
    if (max_kv <= budget) return SIA_LAUNCH_CHECK();      // nothing moves anywhere
    int page_log2 = -1;
    for (int b = 0; b < 31; ++b)
        if (page_size == 1 << b) page_log2 = b;
    // the widest piece that divides a key's row
    const int size = dtype == SIA_F32 ? 4 : 2, bytes = head_dim * size, piece = bytes % 16 == 0 && (uintptr_t)k_pages % 16 == 0 ? 16 : size;
    const int lanes = 4, key_slices = (bytes / piece + lanes - 1) / lanes, value_slices = (value_dim + 15) / 16, slices = key_slices + value_slices + 1;
    if (slices > 65535) return SIA_BAD_ARGUMENT;
    // further workgroups for the movers from beyond the new length, where those that there are leave the chip idle and there may be enough of them
    const ll far = max(0, min(budget - keep_last, max_kv - keep_last - budget)), there = units * slices;
    const int shares = 1 + (int)min((far + 255) / 256, there >= 1024 ? 0 : 1024 / there);
#define LAUNCH(T, P)                                                                                                                    \
    hipLaunchKernelGGL((evict_move_kernel<T, P>), dim3((unsigned)units, slices, shares), dim3(MOVE_THREADS), 0, stream, (T*)k_pages,     \
                       (T*)v_pages, weights, slots, kv_len, block_table, table_width, n_pages, places, max_kv, n_kv, head_dim,           \
                       value_dim, page_size, page_log2, budget, keep_last, key_slices, value_slices, max_moves, from, to, n_moves)
    if (dtype == SIA_F32) {
        if (piece == 16) LAUNCH(float, piece16);
        else LAUNCH(float, float);
    } else {
        if (piece == 16) LAUNCH(bf16_t, piece16);
        else LAUNCH(bf16_t, bf16_t);
    }
#undef LAUNCH
    return SIA_LAUNCH_CHECK();
}
