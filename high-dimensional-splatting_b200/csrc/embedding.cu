// embedding.cu -- the codebook lookup out[i] = f * table[ids[i]] and its gradient
// dtable[v] = f * sum over the i with ids[i] = v of dout[i], both with optional dropout of the looked-up
// elements in the same pass (philox.cuh): f = scale / kept share, dropped elements 0 in both directions.
//
// Lookup.  One pass: the output is written once, the table's rows come from the L2 when the codebook is
// smaller than it.  Bound by the writes: 1.18M x 512 fp32 in 400 to 414 us alone, 2.4 GB at 5.9 to 6.1 TB/s
// (0.90 to 0.93 of the measured copy rate), 444 to 449 us (0.83 to 0.84) in passes over changing inputs;
// with dropout 424 to 442 us alone, where the generator's integer work begins to count.
//
// Gradient.  The rows are put in codeword order by a stable radix sort of (id, row number), and each
// codeword's rows are summed in that order in fp32: no float atomics, so a call's result does not depend
// on timing.  Rows with the padding id or an id outside the table sort behind the last codeword and are
// skipped.
//
// An id outside [0, vocab) that is not the padding id looks up a row of zeros, gets no gradient and
// records HDS_ERR_INVALID in a device status word (hds_device_status); nothing is read or written for it.
#include <algorithm>

#include "elements.cuh"
#include "philox.cuh"

namespace hds {

__device__ int g_embedding_status = 0;

namespace {

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

constexpr int THREADS = 256;
constexpr size_t DEFAULT_SHARED_BYTES = 48 << 10;  // a block may have more on request

// The ids, and which table row each stands for.
struct Ids {
    const void* p;
    int wide;        // int64 (else int32)
    uint32_t vocab;
    int padding_row;  // the padding id if it lies in the table, else -1
    int has_padding;
    int64_t padding_id;

    // The table rows of the ids first, first + step, ... below n: -1 for a row of zeros (padding, or outside
    // the table, which is recorded; and beyond n).  All are loaded before the first is looked at.
    template <int COUNT>
    __device__ __forceinline__ void rows(int first, int step, int n, int (&row)[COUNT]) const {
        const int left = n - first;
        if (wide)
            classify<long long, unsigned long long, COUNT>(first, step, left, row);
        else
            classify<int, unsigned, COUNT>(first, step, left, row);
    }

private:
    template <typename I, typename U, int COUNT>
    __device__ __forceinline__ void classify(int first, int step, int left, int (&row)[COUNT]) const {
        const I* from = static_cast<const I*>(p) + first;
        I id[COUNT];
#pragma unroll
        for (int r = 0; r < COUNT; r++) id[r] = r * step < left ? __ldg(from + r * step) : (I)0;
        bool outside = false;
#pragma unroll
        for (int r = 0; r < COUNT; r++) {
            const bool inside = (U)id[r] < (U)vocab;  // negative ids are large ones
            outside |= !inside;
            row[r] = inside && (int)id[r] != padding_row && r * step < left ? (int)id[r] : -1;
        }
        if (outside) {
#pragma unroll
            for (int r = 0; r < COUNT; r++)
                if (r * step < left && (U)id[r] >= (U)vocab && !(has_padding && (int64_t)id[r] == padding_id))
                    atomicExch(&g_embedding_status, HDS_ERR_INVALID);
        }
    }
};

Ids make_ids(const void* p, int type, int64_t vocab, int has_padding, int64_t padding_id) {
    const bool inside = has_padding && padding_id >= 0 && padding_id < vocab;
    return Ids{p, type == HDS_TYPE_I64, (uint32_t)vocab, inside ? (int)padding_id : -1, has_padding, padding_id};
}

// ---------------------------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------------------------
// Rows in vectors of V elements, V the widest into which rows split and to which both buffers are aligned.
// A thread keeps its column through a few rows: the ids are loaded first, then the table's vectors, then
// the output is stored, and nothing but pointers moves from row to row.  The rows are as many as make 64
// bytes of input or output per thread: with 32 and 128 bytes 1.18M x 512 fp32 from a table of 8192 rows
// takes a tenth longer.
template <typename T, typename O, int V>
constexpr int WIDE_BYTES = V * (sizeof(O) > sizeof(T) ? (int)sizeof(O) : (int)sizeof(T));
template <typename T, typename O, int V>
constexpr int LOOKUP_PASSES = 64 / WIDE_BYTES<T, O, V> < 8 ? 64 / WIDE_BYTES<T, O, V> : 8;

// With dropout the generator's integer work is what the warps wait for: all the blocks that fit (32 registers a
// thread) take 1.18M x 512 from 461 to 434 us.
template <typename T, typename O, int V, bool DROP>
__global__ void __launch_bounds__(THREADS, DROP ? 8 : 1)
    lookup_rows_kernel(int n, int channels, int vectors, int rows_at_once, Divider vectors_of,
                       const T* __restrict__ table, Ids ids, float factor, uint32_t last, Draw draw,
                       O* __restrict__ out) {
    static_assert(V == 8 || !DROP, "a thread draws for whole groups of eight");
    constexpr int PASSES = LOOKUP_PASSES<T, O, V>;
    if (DROP) draw = resolve(draw);
    const uint32_t r = vectors_of.quotient(threadIdx.x);
    const int vector = (int)(blockIdx.y * THREADS + threadIdx.x - r * vectors_of.d);
    if (r >= (uint32_t)rows_at_once || vector >= vectors) return;
    const int row0 = blockIdx.x * (PASSES * rows_at_once) + r, left = n - row0;
    int from[PASSES];
    ids.rows<PASSES>(row0, rows_at_once, n, from);
    const T* column = table + vector * V;
    Vec<T, V> v[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; p++)
        if (from[p] >= 0) v[p] = load_shared_data<T, V>(column + (int64_t)from[p] * channels);
    O* to = out + (int64_t)row0 * channels + vector * V;
    const uint32_t step = (uint32_t)rows_at_once * channels;
    const uint32_t group = (uint32_t)row0 * vectors + vector;
#pragma unroll
    for (int p = 0; p < PASSES; p++) {
        Numbers8 numbers{};
        if (DROP) numbers = philox4x32_10(group + (uint32_t)(p * rows_at_once * vectors), 0, draw);
        float result[V];
#pragma unroll
        for (int j = 0; j < V; j++) result[j] = !DROP || numbers.kept(j, last) ? v[p].get(j) * factor : 0.0f;
        Vec<O, V> packed = Vec<O, V>::pack(result);
        if (from[p] < 0) packed = Vec<O, V>{};
        if (p * rows_at_once < left) store<O, V>(to + p * step, packed);
    }
}

// Rows that split into vectors of two at most, and dropout on rows that do not split into groups of eight.
// Eight rows are whole groups, so a block takes `eights` times eight rows, group by group: one generator
// call still serves eight elements, an id eight of its row's, and the output is one vector.  A group's elements
// come from the table in vectors of V, from two rows at most (any number when rows are narrower than a
// group).  (With a thread per element 1.18M x 75 fp32 took 174 us, 108 like this.)  With scalar loads the L1's
// rate bounds it (98% of its peak at 1.18M x 75 fp32, twice the bytes' floor of 55 us); with dropout in
// 16 bits the integer work (74% of the issue slots, 19% of the memory's rate: 102 us for 1M x 100 bf16,
// floor 33 us).
template <typename T, typename O, int V, bool DROP>
__global__ void __launch_bounds__(THREADS) lookup_groups_kernel(int n, int channels, int eights, Divider rows_of,
                                                                const T* __restrict__ table, Ids ids, float factor,
                                                                uint32_t last, Draw draw, int whole,
                                                                O* __restrict__ out) {
    if (DROP) draw = resolve(draw);
    const int groups = eights * channels;  // of the block
    const int row0 = blockIdx.x * 8 * eights;
    const uint64_t group0 = (uint64_t)blockIdx.x * groups;
    O* to = out + group0 * 8;
    const int here = (int)min((int64_t)groups * 8, ((int64_t)n - row0) * channels);  // elements of the block
    const auto row_of = [&](uint32_t e) -> int {
        return rows_of.d != 0 ? (int)rows_of.quotient(e) : (int)(e / (uint32_t)channels);
    };
    for (int e0 = 8 * threadIdx.x; e0 < here; e0 += 8 * THREADS) {
        Vec<T, V> v[8 / V];
        uint32_t there = 0;  // bit j: element j comes from the table (its first row in the place of no row)
        if (channels >= 8) {
            const int q = row_of(e0), col = e0 - q * channels, left = channels - col;
            int from[2];
            ids.rows<2>(row0 + q, 1, n, from);
            const uint32_t in_a = left >= 8 ? 0xffu : (1u << left) - 1u;
            there = (from[0] >= 0 ? in_a : 0u) | (from[1] >= 0 ? 0xffu & ~in_a : 0u);
            const T* a = table + (int64_t)max(from[0], 0) * channels + col;
            const T* b = table + (int64_t)max(from[1], 0) * channels - left;
#pragma unroll
            for (int k = 0; k < 8 / V; k++) v[k] = load_shared_data<T, V>((k * V < left ? a : b) + k * V);
        } else {
#pragma unroll
            for (int k = 0; k < 8 / V; k++) {
                const int q = row_of(e0 + k * V);
                int from[1];
                ids.rows<1>(row0 + q, 1, n, from);
                if (from[0] >= 0) there |= ((1u << V) - 1u) << (k * V);
                v[k] = load_shared_data<T, V>(table + (int64_t)max(from[0], 0) * channels +
                                              (e0 + k * V - q * channels));
            }
        }
        Numbers8 numbers{};
        if (DROP) numbers = philox4x32_10((uint32_t)group0 + e0 / 8, 0, draw);
        float r[8];
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = !DROP || numbers.kept(j, last) ? v[j / V].get(j % V) * factor : 0.0f;
        if (there != 0xffu) {
#pragma unroll
            for (int j = 0; j < 8; j++) r[j] = (there >> j) & 1u ? r[j] : 0.0f;
        }
        if (whole && e0 + 8 <= here) {
            store<O, 8>(to + e0, Vec<O, 8>::pack(r));
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (e0 + j < here) to[e0 + j] = from_float<O>(r[j]);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// stable radix sort of (codeword, row number)
// ---------------------------------------------------------------------------------------------
// Lanes of the warp with this lane's digit (`bits` bits; among the valid lanes): a vote per bit.  The
// __match_any_sync instruction, which finds the same, took about 100 cycles of an SM here: 17 us for the
// histogram of 100K ids, 8 with votes.
__device__ __forceinline__ uint32_t lanes_alike(uint32_t digit, int bits, bool valid) {
    uint32_t peers = __ballot_sync(FULL_MASK, valid);
    for (int b = 0; b < bits; b++) {
        const bool one = (digit >> b) & 1u;
        const uint32_t ones = __ballot_sync(FULL_MASK, one);
        peers &= one ? ones : ~ones;
    }
    return peers;
}

// Digits of up to 11 bits: one pass for codebooks below 2048 rows, two below 4M.  A pass is a histogram
// per tile and a scatter that ranks the tile's keys, with a scan of the counts between them where they are
// many.  The first pass reads the ids themselves.  No block waits for another.  Bound by latency: the passes
// of 1.18M ids of 8192 codewords take 45 us together, 12% of the gradient's time at 512 channels.
constexpr int SORT_THREADS = 512;
constexpr int SORT_WARPS = SORT_THREADS / 32;
// Keys per thread: 16 (a tile is 8192 keys) when that still gives every SM a tile, else 4.
constexpr int MANY_ROUNDS = 16, SOME_ROUNDS = 4;
constexpr int MAX_DIGIT_BITS = 11;
constexpr int MAX_DIGITS = 1 << MAX_DIGIT_BITS;

// A pass's elements, (key, row) pairs.  The first pass makes them from the ids; all of a thread's ids are
// loaded before the first is looked at, since an id outside the table is recorded, a side effect that
// orders what follows.
struct PairSource {
    const uint2* pairs;  // sorted so far, or NULL in the first pass:
    Ids ids;

    // The elements first, first + step, ... below n (key 0 beyond).
    template <int COUNT>
    __device__ __forceinline__ void load(int first, int step, int n, uint2 (&pair)[COUNT]) const {
        const int left = n - first;
        if (pairs != nullptr) {
#pragma unroll
            for (int r = 0; r < COUNT; r++)
                pair[r] = r * step < left ? __ldg(pairs + first + r * step) : make_uint2(0, 0);
            return;
        }
        int row[COUNT];
        ids.rows<COUNT>(first, step, n, row);
#pragma unroll
        for (int r = 0; r < COUNT; r++) {
            const uint32_t key = row[r] < 0 ? ids.vocab : (uint32_t)row[r];
            pair[r] = make_uint2(r * step < left ? key : 0, (uint32_t)(first + r * step));
        }
    }
};

// counts[digit][tile].
template <int ROUNDS>
__global__ void __launch_bounds__(SORT_THREADS) histogram_kernel(int n, PairSource source, int shift, int bits,
                                                                 int tiles, uint32_t* __restrict__ counts) {
    __shared__ uint32_t hist[MAX_DIGITS];
    const int digits = 1 << bits;
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) hist[d] = 0;
    __syncthreads();
    const int base = blockIdx.x * (SORT_THREADS * ROUNDS) + threadIdx.x;
    const int lane = threadIdx.x & 31;
    uint2 pair[ROUNDS];
    source.load<ROUNDS>(base, SORT_THREADS, n, pair);
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const bool valid = base + r * SORT_THREADS < n;
        const uint32_t d = (pair[r].x >> shift) & (digits - 1);
        // One shared atomic per distinct digit of the warp: popular codewords would serialise otherwise.
        const uint32_t peers = lanes_alike(d, bits, valid);
        if (valid && lane == __ffs(peers) - 1) atomicAdd(&hist[d], __popc(peers));
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) counts[(int64_t)d * tiles + blockIdx.x] = hist[d];
}

// A scatter block sums the counts of the tiles before its own itself where that takes few loads: a thread a
// digit for 16 tiles at most, a warp a digit for 160 tiles and 256 digits at most.
constexpr int FEW_TILES = 16, SOME_TILES = 160, SOME_DIGIT_BITS = 8;

// counts[digit][tile] -> how many keys of that digit the tiles before have, and totals[digit].  A warp per
// digit.
constexpr int SCAN_WARPS = 8;

__global__ void __launch_bounds__(32 * SCAN_WARPS) scan_kernel(int digits, int tiles,
                                                               uint32_t* __restrict__ counts,
                                                               uint32_t* __restrict__ totals) {
    const int lane = threadIdx.x & 31, digit = blockIdx.x * SCAN_WARPS + (threadIdx.x >> 5);
    if (digit >= digits) return;
    uint32_t base = 0;
    uint32_t* row = counts + (int64_t)digit * tiles;
    constexpr int AHEAD = 8;
    for (int t0 = lane; t0 < tiles + lane; t0 += 32 * AHEAD) {
        uint32_t v[AHEAD];
#pragma unroll
        for (int h = 0; h < AHEAD; h++) v[h] = t0 + 32 * h < tiles ? row[t0 + 32 * h] : 0;
#pragma unroll
        for (int h = 0; h < AHEAD; h++) {
            uint32_t x = v[h];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(FULL_MASK, x, o);
                if (lane >= o) x += y;
            }
            if (t0 + 32 * h < tiles) row[t0 + 32 * h] = base + x - v[h];
            base += __shfl_sync(FULL_MASK, x, 31);
        }
    }
    if (lane == 0) totals[digit] = base;
}

// Each warp ranks its own consecutive keys into a count table of its own; a scan over the digits and the
// warps places the tile's pairs in shared memory in sorted order, from where they go out in runs of equal
// digits.  (Stored straight from the registers, each of a warp's pairs is a memory access of its own, and
// the scatter of 1.18M pairs took 20 us instead of 12.)
inline size_t scatter_shared_bytes(int digits, int rounds) {
    return (size_t)digits * (2 * sizeof(uint32_t) + 2 * SORT_WARPS) + (size_t)rounds * SORT_THREADS * sizeof(uint2);
}

template <int ROUNDS>
__global__ void __launch_bounds__(SORT_THREADS) scatter_kernel(int n, PairSource source, int shift, int bits,
                                                               int tiles, int scanned,
                                                               const uint32_t* __restrict__ counts,
                                                               const uint32_t* __restrict__ totals,
                                                               uint2* __restrict__ out) {
    constexpr int TILE = ROUNDS * SORT_THREADS;
    constexpr int OWN = MAX_DIGITS / SORT_THREADS;  // digits per thread in the scan at most
    extern __shared__ uint2 s_pair[];                                        // [TILE] in sorted order
    __shared__ uint2 s_total[SORT_WARPS];
    const int digits = 1 << bits, own = max(1, digits / SORT_THREADS);
    uint32_t* s_move = reinterpret_cast<uint32_t*>(s_pair + TILE);           // [digits]: output - tile position
    uint32_t* s_all = s_move + digits;                                       // [digits]
    uint16_t* s_warp = reinterpret_cast<uint16_t*>(s_all + digits);          // [warps][digits]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tile = blockIdx.x * TILE;
    const int base = tile + warp * (32 * ROUNDS) + lane;
    uint16_t* mine = s_warp + warp * digits;
    uint2 pair[ROUNDS];
    uint16_t rank[ROUNDS];
    source.load<ROUNDS>(base, 32, n, pair);
    // The digit's keys in all tiles, and (s_move for now) in the tiles before this one.
    if (scanned) {
        for (int d = tid; d < digits; d += SORT_THREADS) {
            s_move[d] = counts[(int64_t)d * tiles + blockIdx.x];
            s_all[d] = totals[d];
        }
    } else if (tiles <= FEW_TILES) {
        for (int d = tid; d < digits; d += SORT_THREADS) {
            uint32_t before = 0, all = 0;
#pragma unroll
            for (int t = 0; t < FEW_TILES; t++) {
                const uint32_t c = t < tiles ? counts[(int64_t)d * tiles + t] : 0;
                before += t < (int)blockIdx.x ? c : 0;
                all += c;
            }
            s_move[d] = before;
            s_all[d] = all;
        }
    } else {
#pragma unroll 4
        for (int d = warp; d < digits; d += SORT_WARPS) {
            uint32_t before = 0, all = 0;
#pragma unroll
            for (int t = lane; t < SOME_TILES; t += 32) {
                const uint32_t c = t < tiles ? counts[(int64_t)d * tiles + t] : 0;
                before += t < (int)blockIdx.x ? c : 0;
                all += c;
            }
            before = __reduce_add_sync(FULL_MASK, before);
            all = __reduce_add_sync(FULL_MASK, all);
            if (lane == 0) s_move[d] = before;
            if (lane == 0) s_all[d] = all;
        }
    }
    for (int i = tid; i < digits * SORT_WARPS / 2; i += SORT_THREADS) reinterpret_cast<uint32_t*>(s_warp)[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const bool valid = base + 32 * r < n;
        const uint32_t d = (pair[r].x >> shift) & (digits - 1);
        const uint32_t peers = lanes_alike(d, bits, valid);
        const uint32_t before = mine[d];
        __syncwarp();
        rank[r] = (uint16_t)(before + __popc(peers & ((1u << lane) - 1u)));
        if (valid && lane == __ffs(peers) - 1) mine[d] = (uint16_t)(before + __popc(peers));
        __syncwarp();
    }
    __syncthreads();
    // Where each digit, and in it each warp, starts in the tile.
    uint32_t total[OWN], sum = 0, everywhere[OWN], sum_everywhere = 0;
#pragma unroll
    for (int h = 0; h < OWN; h++) {
        const int d = tid * own + h;
        everywhere[h] = h < own && d < digits ? s_all[d] : 0;
        sum_everywhere += everywhere[h];
        total[h] = 0;
        if (h < own && d < digits)
#pragma unroll
            for (int w = 0; w < SORT_WARPS; w++) total[h] += s_warp[w * digits + d];
        sum += total[h];
    }
    uint32_t inclusive = sum, inclusive_everywhere = sum_everywhere;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(FULL_MASK, inclusive, o);
        const uint32_t z = __shfl_up_sync(FULL_MASK, inclusive_everywhere, o);
        if (lane >= o) inclusive += y;
        if (lane >= o) inclusive_everywhere += z;
    }
    if (lane == 31) s_total[warp] = make_uint2(inclusive, inclusive_everywhere);
    __syncthreads();
    uint32_t run = inclusive - sum, start = inclusive_everywhere - sum_everywhere;
    for (int w = 0; w < warp; w++) {
        run += s_total[w].x;
        start += s_total[w].y;
    }
#pragma unroll
    for (int h = 0; h < OWN; h++) {
        const int d = tid * own + h;
        if (h >= own || d >= digits) break;
        s_move[d] += start - run;
        start += everywhere[h];
#pragma unroll
        for (int w = 0; w < SORT_WARPS; w++) {
            const uint32_t c = s_warp[w * digits + d];
            s_warp[w * digits + d] = (uint16_t)run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        if (base + 32 * r >= n) break;
        const uint32_t d = (pair[r].x >> shift) & (digits - 1);
        s_pair[mine[d] + rank[r]] = pair[r];
    }
    __syncthreads();
    const int here = min(TILE, n - tile);
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const int i = tid + r * SORT_THREADS;
        if (i >= here) break;
        const uint2 p = s_pair[i];
        out[s_move[(p.x >> shift) & (digits - 1)] + i] = p;
    }
}

// ---------------------------------------------------------------------------------------------
// sums by codeword
// ---------------------------------------------------------------------------------------------
// The sorted rows are cut into chunks of equal length whatever the codewords' popularity.  A worker, a
// group of 1 to 32 lanes with 8 columns each, adds up one chunk's rows in registers.  A codeword that
// begins and ends inside the chunk goes straight to the table.  The sum of a codeword that began in an
// earlier chunk is the chunk's head, that of one that goes on into the next its tail; join_kernel adds a
// tail and the heads that follow it.  Bound by the memory: fp32 rows of 512 columns are read at 6.2 TB/s, 0.94
// of the measured copy rate, rows of 128 at 5.9.  With dropout nothing is full (58% of the issue slots, 61% of
// the memory's rate): the generator and the loads take turns in the 30% of the warps that fit.  Odd widths
// load scalars and wait for them (1.18M x 75 fp32: 154 us, 37% of the memory's rate, 24% of the warps).
constexpr int COLUMNS = 8;       // per lane
constexpr int ROWS_AHEAD = 4;    // rows loaded before the first is added

// The sum of no rows is stored as +0 whatever the factor's sign (the addition of 0 turns -0 into it), as the
// memset of the sorted form leaves it.
template <typename T, int V, bool ACCUMULATE>
__device__ __forceinline__ void store_sum(T* p, const float* sum, float factor) {
    Vec<T, V> old;
    if (ACCUMULATE) old = load_once<T, V>(p);
    float r[V];
#pragma unroll
    for (int j = 0; j < V; j++) r[j] = fmaf(factor, sum[j], ACCUMULATE ? old.get(j) : 0.0f);
    store<T, V>(p, Vec<T, V>::pack(r));
}

// Three blocks an SM (85 registers a thread) take 1.18M x 512 with dropout from 598 to 532 us; narrow vectors
// would spill.
template <typename G, typename T, int V, bool DROP, bool ACCUMULATE>
__global__ void __launch_bounds__(THREADS, V == COLUMNS ? 3 : 0)
    chunk_sum_kernel(int64_t n, uint32_t vocab, int channels, int slab, int lanes_log2, int chunk, int slabs,
                     const uint2* __restrict__ pairs, const G* __restrict__ grad, float factor, uint32_t last,
                     Draw draw, T* __restrict__ table, float* __restrict__ heads, float* __restrict__ tails,
                     int stride) {
    constexpr int STEPS = COLUMNS / V;
    if (DROP) draw = resolve(draw);
    const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
    // The slabs of the same chunks are neighbouring blocks, so that they read the rows' halves together.
    const int slab_id = blockIdx.x % slabs;
    const int64_t id = ((int64_t)(blockIdx.x / slabs) * THREADS + threadIdx.x) >> lanes_log2;  // of the chunk
    const int64_t start = id * chunk;
    const int c0 = slab_id * slab, width = min(slab, channels - c0);
    // A lane's vector k, within the slab: interleaved between the lanes, so that narrow vectors coalesce; with
    // dropout the lane's columns are consecutive, since then eight decisions are two neighbouring groups'.
    const auto column = [&](int k) { return DROP ? lane * COLUMNS + k * V : (k * lanes + lane) * V; };
    uint32_t current = start < n ? pairs[start].x : vocab;
    bool began_earlier = start < n && start > 0 && pairs[start - 1].x == current;
    float sum[COLUMNS];
#pragma unroll
    for (int j = 0; j < COLUMNS; j++) sum[j] = 0.0f;

    const auto put = [&](float* partial) {
#pragma unroll
        for (int k = 0; k < STEPS; k++)
            if (column(k) < width)
                store_sum<float, V, false>(partial + id * stride + c0 + column(k), sum + k * V, 1.0f);
    };
    const auto finish = [&]() {  // the current codeword ends here
        if (began_earlier) {
            put(heads);
            return;
        }
#pragma unroll
        for (int k = 0; k < STEPS; k++)
            if (column(k) < width)
                store_sum<T, V, ACCUMULATE>(table + (int64_t)current * channels + c0 + column(k), sum + k * V, factor);
    };

    for (int p = 0; p < chunk; p += ROWS_AHEAD) {
        // Chunks start at multiples of 8, so the four pairs are two 16-byte loads (the buffers are padded
        // beyond n).
        const int64_t pos = start + p;
        uint4 two[2] = {make_uint4(vocab, 0, vocab, 0), make_uint4(vocab, 0, vocab, 0)};
        if (pos < n) {
            two[0] = __ldg(reinterpret_cast<const uint4*>(pairs + pos));
            two[1] = __ldg(reinterpret_cast<const uint4*>(pairs + pos) + 1);
        }
        const uint32_t key[ROWS_AHEAD] = {two[0].x, pos + 1 < n ? two[0].z : vocab, pos + 2 < n ? two[1].x : vocab,
                                          pos + 3 < n ? two[1].z : vocab};
        const uint32_t row[ROWS_AHEAD] = {two[0].y, two[0].w, two[1].y, two[1].w};
        Vec<G, V> g[ROWS_AHEAD][STEPS];
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; u++)
#pragma unroll
            for (int k = 0; k < STEPS; k++)
                if (key[u] != vocab && column(k) < width)
                    g[u][k] = DROP && V < COLUMNS
                                  ? load_shared_data<G, V>(grad + (int64_t)row[u] * channels + c0 + column(k))
                                  : load_once<G, V>(grad + (int64_t)row[u] * channels + c0 + column(k));
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; u++) {
            Numbers8 numbers{};
            uint32_t keep = 0;
            if (DROP) {
                const int64_t e = (int64_t)(key[u] != vocab ? row[u] : 0) * channels + c0;
                numbers = philox4x32_10((uint32_t)(e >> 3) + lane, 0, draw);
                if (V < COLUMNS) {
                    // A row may start inside a group: a lane's columns are then the end of one group and the
                    // beginning of the next lane's.
                    const int into = (int)(e & 7);
                    const uint32_t bits = numbers.bits(last);
                    uint32_t next = __shfl_down_sync(FULL_MASK, bits, 1, lanes);
                    if (into != 0 && lane == lanes - 1 && lane * COLUMNS + COLUMNS - into < width)
                        next = philox4x32_10((uint32_t)(e >> 3) + lanes, 0, draw).bits(last);
                    keep = (bits | next << 8) >> into;
                }
            }
            if (key[u] != current) {
                if (current != vocab) finish();
                current = key[u];
                began_earlier = false;
#pragma unroll
                for (int j = 0; j < COLUMNS; j++) sum[j] = 0.0f;
            }
            if (key[u] == vocab) continue;
#pragma unroll
            for (int k = 0; k < STEPS; k++)
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (!DROP || (V == COLUMNS ? numbers.kept(j, last) : ((keep >> (k * V + j)) & 1u) != 0))
                        sum[k * V + j] += g[u][k].get(j);
        }
    }
    if (current == vocab) return;
    const int64_t end = start + chunk;
    if (end < n && pairs[end].x == current)
        put(began_earlier ? heads : tails);
    else
        finish();
}

// A worker of 4 lanes (32 columns) per chunk: if the chunk's last codeword began in it and goes on, it owns
// that codeword's sum, its tail plus the heads of the following chunks.  Up to 64 heads: the worker adds
// them.  More (a popular codeword): the whole block does, in 64 interleaved runs and a tree, after a
// search for the last head with 256 probes a step.  What the kernel costs is its chain of dependent loads,
// so each step loads all it may need at once.
constexpr int JOIN_LANES = 4;
constexpr int JOIN_WORKERS = THREADS / JOIN_LANES;
constexpr int JOIN_COLUMNS = JOIN_LANES * COLUMNS;
constexpr int HEADS_AHEAD = 8;  // probes, and heads loaded, at once

template <typename T, int V, bool ACCUMULATE>
__global__ void __launch_bounds__(THREADS) join_kernel(int64_t n, uint32_t vocab, int channels, int chunk,
                                                       const uint2* __restrict__ pairs,
                                                       const float* __restrict__ heads,
                                                       const float* __restrict__ tails, int stride, float factor,
                                                       T* __restrict__ table) {
    __shared__ int s_long;
    __shared__ int64_t s_id[JOIN_WORKERS];
    __shared__ float s_sum[JOIN_WORKERS][JOIN_COLUMNS];
    const int worker = threadIdx.x / JOIN_LANES, lane = threadIdx.x % JOIN_LANES;
    const int c = blockIdx.y * JOIN_COLUMNS + lane * COLUMNS;
    const bool there = c < channels;
    const int64_t chunks = (n + chunk - 1) / chunk;
    const int64_t id = (int64_t)blockIdx.x * JOIN_WORKERS + worker;
    if (threadIdx.x == 0) s_long = 0;
    __syncthreads();

    const auto add = [&](float* sum, const Vec<float, COLUMNS>& v) {
#pragma unroll
        for (int j = 0; j < COLUMNS; j++) sum[j] += v.get(j);
    };
    const auto load = [&](const float* partial, int64_t at) {
        return load_shared_data<float, COLUMNS>(partial + at * stride + c);
    };
    const auto write = [&](uint32_t codeword, const float* sum) {
#pragma unroll
        for (int j = 0; j < COLUMNS; j += V)
            if (c + j < channels)
                store_sum<T, V, ACCUMULATE>(table + (int64_t)codeword * channels + c + j, sum + j, factor);
    };

    const int64_t start = id * chunk, end = start + chunk;
    if (end < n) {
        const uint32_t codeword = pairs[end].x, at_end = pairs[end - 1].x, at_start = pairs[start].x;
        const uint32_t before = start > 0 ? pairs[start - 1].x : vocab;
        // The key with which the h-th chunk after the next one begins.
        const auto key_after = [&](int h) { return id + 1 + h < chunks ? pairs[(id + 1 + h) * chunk].x : vocab; };
        uint32_t coarse[HEADS_AHEAD];
#pragma unroll
        for (int h = 0; h < HEADS_AHEAD; h++) coarse[h] = key_after(HEADS_AHEAD * (h + 1));
        if (codeword != vocab && at_end == codeword && (at_start != codeword || before != codeword)) {
            int count = 0;  // heads; the keys are sorted, so equal ones have no gaps
#pragma unroll
            for (int h = 0; h < HEADS_AHEAD; h++) count += coarse[h] == codeword ? HEADS_AHEAD : 0;
            if (count < HEADS_AHEAD * HEADS_AHEAD) {
                int more = 1;
#pragma unroll
                for (int h = 1; h < HEADS_AHEAD; h++) more += key_after(count + h) == codeword ? 1 : 0;
                count += more;
                if (there) {
                    float sum[COLUMNS] = {};
                    add(sum, load(tails, id));
                    for (int h0 = 0; h0 < count; h0 += HEADS_AHEAD) {
                        Vec<float, COLUMNS> head[HEADS_AHEAD];
#pragma unroll
                        for (int h = 0; h < HEADS_AHEAD; h++)
                            if (h0 + h < count) head[h] = load(heads, id + 1 + h0 + h);
#pragma unroll
                        for (int h = 0; h < HEADS_AHEAD; h++)
                            if (h0 + h < count) add(sum, head[h]);
                    }
                    write(codeword, sum);
                }
            } else if (lane == 0) {
                s_id[atomicAdd(&s_long, 1)] = id;
            }
        }
    }
    __syncthreads();
    for (int slot = 0; slot < s_long; slot++) {
        const int64_t from = s_id[slot];
        const uint32_t codeword = pairs[(from + 1) * chunk].x;
        // The last chunk that begins with the codeword lies in [last, beyond).
        int64_t last = from + 1, beyond = chunks;
        while (beyond - last > 1) {
            const int64_t step = (beyond - last + THREADS - 1) / THREADS;
            const int64_t probe = last + (threadIdx.x + 1) * step;
            const int hits = __syncthreads_count(probe < beyond && pairs[probe * chunk].x == codeword);
            last += hits * step;
            beyond = min(beyond, last + step);
        }
        float sum[COLUMNS] = {};
        if (there) {
            if (worker == 0) add(sum, load(tails, from));
            int64_t j = from + 1 + worker;
            for (; j + 3 * JOIN_WORKERS <= last; j += 4 * JOIN_WORKERS) {
                Vec<float, COLUMNS> head[4];
#pragma unroll
                for (int u = 0; u < 4; u++) head[u] = load(heads, j + u * JOIN_WORKERS);
#pragma unroll
                for (int u = 0; u < 4; u++) add(sum, head[u]);
            }
            for (; j <= last; j += JOIN_WORKERS) add(sum, load(heads, j));
        }
#pragma unroll
        for (int j = 0; j < COLUMNS; j++) s_sum[worker][lane * COLUMNS + j] = sum[j];
        __syncthreads();
        for (int half = JOIN_WORKERS / 2; half > 0; half /= 2) {
            for (int i = threadIdx.x; i < half * JOIN_COLUMNS; i += THREADS)
                s_sum[i / JOIN_COLUMNS][i % JOIN_COLUMNS] += s_sum[i / JOIN_COLUMNS + half][i % JOIN_COLUMNS];
            __syncthreads();
        }
        if (worker == 0 && there) write(codeword, s_sum[0] + lane * COLUMNS);
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// few rows: one launch
// ---------------------------------------------------------------------------------------------
// A block owns a range of codewords and a slab of columns and does everything for them: it reads all ids, keeps
// the rows whose codeword is its own, groups them by codeword in shared memory (the scatter's ranking:
// row order stays), adds each codeword's rows and writes every row of its range, zeros included.  Each
// block reads all the ids, which is cheap while there are few; in return nothing waits for a second
// launch.  A worker of 1 to FEW_LANES lanes (8 columns each) adds the rows of a codeword; one with many rows
// is added by the whole block, every worker a run of interleaved rows, and a tree.
//
// Measured against the sorted form, us a call, called in a loop / replayed from a captured graph:
//   4096 x 32 of 256      11.5 / 10.3   sorted 24.8 / 16.4        300 x 64 of 1000   11.5 / 10.3   24.0 / 16.4
//   4096 x 512 of 256     18.5 / 18.4          24.1 / 17.7        4096 x 1000 of 4096  22.6 / 22.6  39.0 / 26.7
//   4096 x 75 of 256      24.6 / 24.6          25.7 / 20.5        8192 x 512: 57 us with events around it, 35 sorted
// so up to 4096 rows it is ahead in a loop (the sorted form's launches cost the host) and level or ahead in
// a graph but for odd widths.  With dropout at odd widths it is not: its decisions for 8 scalar columns of 4
// rows spill (128 registers), and from about 512 rows on it falls behind (4096 x 75 of 256: 54.4 / 53.7 and
// 25.7 / 20.5; 4096 x 501: 117 and 29).  It is taken there all the same: the caller's scratch follows from the
// sizes alone, which tell neither dropout nor alignment.
constexpr int FEW_THREADS = 512;
constexpr int FEW_ROUNDS = 8;                        // ids per thread
constexpr int FEW_ROWS = FEW_THREADS * FEW_ROUNDS;  // 4096
constexpr int FEW_WARPS = FEW_THREADS / 32;
constexpr int FEW_LANES = 8;
constexpr int FEW_RANGE = 2 * FEW_THREADS;  // codewords per block at most
constexpr int FEW_VOCAB = 32768;            // beyond it, rows of zeros are better cleared by a memset
constexpr int SHORT_ROWS = 32;

inline size_t few_rows_shared_bytes(int64_t n, int range) {
    return (size_t)(range + 1) * 4 + (size_t)range * FEW_WARPS * 2 + (size_t)n * 2;
}

template <typename G, typename T, int V, bool DROP, bool ACCUMULATE>
__global__ void __launch_bounds__(FEW_THREADS) few_rows_kernel(int n, int channels, int range, int lanes_log2, Ids ids,
                                                               const G* __restrict__ grad, float factor,
                                                               uint32_t last, Draw draw,
                                                               T* __restrict__ table) {
    constexpr int STEPS = COLUMNS / V;
    extern __shared__ uint32_t s_start[];                                    // [range + 1]
    uint16_t* s_count = reinterpret_cast<uint16_t*>(s_start + range + 1);    // [warps][range]
    uint16_t* s_rows = s_count + FEW_WARPS * range;                          // [n]
    __shared__ float s_sum[FEW_THREADS * COLUMNS];                           // [workers][slab]
    __shared__ uint32_t s_warp[FEW_WARPS];
    __shared__ int s_long;
    __shared__ uint16_t s_long_codeword[FEW_ROWS / SHORT_ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane32 = tid & 31;
    const int first = blockIdx.x * range;
    const int here = min(range, (int)ids.vocab - first);
    const int bits = 32 - __clz(range - 1);  // of a codeword's number in the range
    if (DROP) draw = resolve(draw);
    for (int i = tid; i < FEW_WARPS * range; i += FEW_THREADS) s_count[i] = 0;
    if (tid == 0) s_long = 0;
    __syncthreads();

    // The block's rows by codeword: counts, positions, rows.
    uint16_t* mine = s_count + warp * range;
    const int base = warp * (32 * FEW_ROUNDS) + lane32;
    int row[FEW_ROUNDS];
    ids.rows<FEW_ROUNDS>(base, 32, n, row);
    uint16_t rank[FEW_ROUNDS];  // among the warp's rows of the codeword
#pragma unroll
    for (int r = 0; r < FEW_ROUNDS; r++) {
        row[r] = row[r] >= first && row[r] - first < here ? row[r] - first : -1;
        const uint32_t d = (uint32_t)max(row[r], 0);
        const uint32_t peers = lanes_alike(d, bits, row[r] >= 0);
        const uint32_t before = mine[d];
        __syncwarp();
        rank[r] = (uint16_t)(before + __popc(peers & ((1u << lane32) - 1u)));
        if (row[r] >= 0 && lane32 == __ffs(peers) - 1) mine[d] = (uint16_t)(before + __popc(peers));
        __syncwarp();
    }
    __syncthreads();
    uint32_t total[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; h++)
        if (2 * tid + h < here)
            for (int w = 0; w < FEW_WARPS; w++) total[h] += s_count[w * range + 2 * tid + h];
    uint32_t inclusive = total[0] + total[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(FULL_MASK, inclusive, o);
        if (lane32 >= o) inclusive += y;
    }
    if (lane32 == 31) s_warp[warp] = inclusive;
    __syncthreads();
    uint32_t run = inclusive - total[0] - total[1];
    for (int w = 0; w < warp; w++) run += s_warp[w];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int d = 2 * tid + h;
        if (d >= here) break;
        s_start[d] = run;
        for (int w = 0; w < FEW_WARPS; w++) {
            const uint32_t c = s_count[w * range + d];
            s_count[w * range + d] = (uint16_t)run;
            run += c;
        }
        if (d == here - 1) s_start[here] = run;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < FEW_ROUNDS; r++)
        if (row[r] >= 0) s_rows[mine[row[r]] + rank[r]] = (uint16_t)(base + 32 * r);
    __syncthreads();

    const int lanes = 1 << lanes_log2, worker = tid >> lanes_log2, lane = tid & (lanes - 1);
    const int workers = FEW_THREADS >> lanes_log2, slab = lanes * COLUMNS;
    const unsigned worker_mask = (0xffffffffu >> (32 - lanes)) << (lane32 & ~(lanes - 1));
    const int c0 = blockIdx.y * slab, width = min(slab, channels - c0);
    const auto column = [&](int k) { return (k * lanes + lane) * V; };
    // sum += rows from, from + step, ... below to.
    const auto add_rows = [&](float* sum, uint32_t from, uint32_t to, uint32_t step) {
        for (uint32_t p = from; p < to; p += ROWS_AHEAD * step) {
            Vec<G, V> g[ROWS_AHEAD][STEPS];
            uint32_t keep[ROWS_AHEAD][STEPS];
#pragma unroll
            for (int u = 0; u < ROWS_AHEAD; u++) {
                const bool there = p + u * step < to;
                const int64_t e = (int64_t)(there ? s_rows[p + u * step] : 0) * channels + c0;
#pragma unroll
                for (int k = 0; k < STEPS; k++) {
                    keep[u][k] = there && column(k) < width ? 0xffu : 0u;
                    if (keep[u][k]) g[u][k] = load_once<G, V>(grad + e + column(k));
                }
                if (DROP) {
                    const uint32_t bits = philox4x32_10((uint32_t)(e >> 3) + lane, 0, draw).bits(last);
                    const int into = (int)(e & 7);
                    const uint32_t more = V < COLUMNS && into + width > slab
                                              ? philox4x32_10((uint32_t)(e >> 3) + lanes, 0, draw).bits(last)
                                              : 0;
#pragma unroll
                    for (int k = 0; k < STEPS; k++) {
                        const int b = into + column(k);
                        uint32_t theirs = bits;
                        if (V < COLUMNS) {
                            theirs = __shfl_sync(worker_mask, bits, b >> 3, lanes);
                            theirs = ((b >> 3) < lanes ? theirs : more) >> (b & 7);
                        }
                        keep[u][k] &= theirs;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < ROWS_AHEAD; u++)
#pragma unroll
                for (int k = 0; k < STEPS; k++)
#pragma unroll
                    for (int j = 0; j < V; j++)
                        if ((keep[u][k] >> j) & 1u) sum[k * V + j] += g[u][k].get(j);
        }
    };
    const auto write = [&](int codeword, const float* sum) {
#pragma unroll
        for (int k = 0; k < STEPS; k++)
            if (column(k) < width)
                store_sum<T, V, ACCUMULATE>(table + (int64_t)(first + codeword) * channels + c0 + column(k),
                                            sum + k * V, factor);
    };
    for (int v = worker; v < here; v += workers) {
        const uint32_t from = s_start[v], to = s_start[v + 1];
        if (ACCUMULATE && from == to) continue;
        if (to - from > SHORT_ROWS) {
            if (lane == 0) s_long_codeword[atomicAdd(&s_long, 1)] = (uint16_t)v;
            continue;
        }
        float sum[COLUMNS] = {};
        add_rows(sum, from, to, 1);
        write(v, sum);
    }
    __syncthreads();
    for (int slot = 0; slot < s_long; slot++) {
        const int v = s_long_codeword[slot];
        float sum[COLUMNS] = {};
        add_rows(sum, s_start[v] + worker, s_start[v + 1], workers);
#pragma unroll
        for (int k = 0; k < STEPS; k++)
#pragma unroll
            for (int j = 0; j < V; j++) s_sum[worker * slab + column(k) + j] = sum[k * V + j];
        __syncthreads();
        for (int half = workers / 2; half > 0; half /= 2) {
            for (int i = tid; i < half * slab; i += FEW_THREADS) s_sum[i] += s_sum[i + half * slab];
            __syncthreads();
        }
        if (worker == 0) {
#pragma unroll
            for (int k = 0; k < STEPS; k++)
#pragma unroll
                for (int j = 0; j < V; j++) sum[k * V + j] = s_sum[column(k) + j];
            write(v, sum);
        }
        __syncthreads();
    }
}

int ceil_log2(int64_t x) {
    int bits = 0;
    while ((int64_t(1) << bits) < x) bits++;
    return bits;
}

struct FewRowsPlan {
    int lanes_log2, range;  // codewords per block: enough blocks to fill the machine, FEW_RANGE codewords at most
    int64_t slabs, ranges;
    bool fits;              // few rows, and blocks that all run in two or three waves
    FewRowsPlan(int64_t n, int64_t vocab, int channels) {
        lanes_log2 = ceil_log2(std::min(FEW_LANES, std::max(1, (channels + COLUMNS - 1) / COLUMNS)));
        slabs = (channels + (COLUMNS << lanes_log2) - 1) / (COLUMNS << lanes_log2);
        if (n == 0 || n > FEW_ROWS || vocab == 0 || channels == 0) {
            fits = false;
            return;
        }
        ranges = std::max<int64_t>((vocab + FEW_RANGE - 1) / FEW_RANGE, std::min(vocab, 444 / slabs + 1));
        range = (int)((vocab + ranges - 1) / ranges);
        ranges = (vocab + range - 1) / range;
        fits = vocab <= FEW_VOCAB && ranges * slabs <= 2048;
    }
};

// How the backward splits its work and lays out its scratch.
struct BackwardPlan {
    int rounds;               // of the sort, per thread of a tile
    int64_t tiles;
    int passes, digit_bits;
    int scan;                 // whether a kernel of its own sums the tiles' counts
    int chunk, stride;        // rows per chunk; floats per partial row
    int64_t chunks;
    int slab, lanes_log2;     // columns and lanes of a worker
    size_t pairs_a, pairs_b, counts, totals, heads, tails, bytes;

    BackwardPlan(int64_t n, int64_t vocab, int channels) {
        const size_t nn = (size_t)std::max<int64_t>(n, 1);
        rounds = (int64_t)nn >= 120 * SORT_THREADS * MANY_ROUNDS ? MANY_ROUNDS : SOME_ROUNDS;
        tiles = ((int64_t)nn + SORT_THREADS * rounds - 1) / (SORT_THREADS * rounds);
        const int bits = std::max(1, ceil_log2(vocab + 1));  // keys 0 .. vocab
        passes = (bits + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
        digit_bits = (bits + passes - 1) / passes;
        scan = !(tiles <= FEW_TILES || (tiles <= SOME_TILES && digit_bits <= SOME_DIGIT_BITS));
        // Long chunks write few partial sums (two rows of a chunk at most); but the chunks have to fill the
        // machine.  75,000 lanes with four rows of 32 bytes each in flight are about 10 MB, more than the
        // memory's latency times its rate.  1.18M x 128 of 4096 popular codewords, 128 / 256 / 512 rows at most:
        // 195, 182 and 185 us; 1.18M x 512 of 8192: 472, 456 and 499.
        const int64_t wanted = (int64_t)nn * std::max(channels, 1) / COLUMNS / 75000;
        chunk = 8;
        while (chunk < 256 && chunk < wanted) chunk *= 2;
        chunks = ((int64_t)nn + chunk - 1) / chunk;
        stride = (channels + COLUMNS - 1) / COLUMNS * COLUMNS;
        const int slabs = std::max(1, (channels + 32 * COLUMNS - 1) / (32 * COLUMNS));
        slab = ((channels + slabs - 1) / slabs + COLUMNS - 1) / COLUMNS * COLUMNS;
        lanes_log2 = ceil_log2(std::max(slab / COLUMNS, 1));
        pairs_a = 0;
        pairs_b = pairs_a + align256(nn * sizeof(uint2));
        counts = pairs_b + align256(nn * sizeof(uint2));
        totals = counts + align256(((size_t)tiles << digit_bits) * 4);
        heads = totals + align256(((size_t)1 << digit_bits) * 4);
        tails = heads + align256((size_t)chunks * stride * 4);
        bytes = tails + align256((size_t)chunks * stride * 4);
    }
};

int check_sizes(const char* what, int64_t n, int64_t vocab, int64_t channels) {
    HDS_REQUIRE(n >= 0 && vocab >= 0 && channels >= 0, HDS_ERR_INVALID, "%s: negative size", what);
    // Row numbers are 32-bit, also of the last, partly empty, block.
    constexpr int64_t most = INT32_MAX - (1 << 20);
    HDS_REQUIRE(n <= most && vocab <= most && channels <= HDS_EMBEDDING_MAX_CHANNELS, HDS_ERR_TOO_LARGE,
                "%s: n = %lld, vocab = %lld, channels = %lld is too large", what, (long long)n, (long long)vocab,
                (long long)channels);
    return HDS_OK;
}

// Shared argument checks of both directions.
int check_arguments(const char* what, int64_t n, int64_t vocab, int64_t channels, int table_type, int value_type,
                    int ids_type, double scale, int drop_threshold) {
    if (int rc = check_sizes(what, n, vocab, channels)) return rc;
    HDS_REQUIRE(known_type(table_type) && (value_type == table_type || value_type == HDS_TYPE_F32),
                HDS_ERR_UNSUPPORTED, "%s: values must be of the table's type or fp32", what);
    HDS_REQUIRE(ids_type == HDS_TYPE_I32 || ids_type == HDS_TYPE_I64, HDS_ERR_UNSUPPORTED,
                "%s: ids must be int32 or int64", what);
    HDS_REQUIRE(drop_threshold >= 0 && drop_threshold <= DROP_ONE, HDS_ERR_INVALID,
                "%s: dropout threshold %d outside 0 to 65536", what, drop_threshold);
    // The kernels multiply by the fp32 factor: infinite, it would make NaN of every zero.
    const float factor = keep_factor(scale, drop_threshold);
    HDS_REQUIRE(scale - scale == 0.0 && factor - factor == 0.0f, HDS_ERR_INVALID,
                "%s: scale must be finite, and in fp32 by the kept share's reciprocal too", what);
    // The kernels keep the generator's upper group word out of the lanes: it is 0.
    HDS_REQUIRE(drop_threshold == 0 || n * channels <= HDS_EMBEDDING_MAX_DROPOUT, HDS_ERR_TOO_LARGE,
                "%s: dropout of %lld values (2^35 at most)", what, (long long)(n * channels));
    return HDS_OK;
}

bool misaligned(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) != 0; }

// Calls f(T{}, V{}) with the table's type and the values' type (the table's or fp32).
template <typename F>
int with_types(int table_type, int value_type, F&& f) {
    return with_type(table_type, [&](auto t) -> int {
        if (value_type == HDS_TYPE_F32) return f(t, float{});
        return f(t, t);
    });
}

}  // namespace

int read_and_clear_embedding_status(int* status, cudaStream_t stream) {
    static const int zero = 0;
    HDS_CHECK_CUDA(
        cudaMemcpyFromSymbolAsync(status, g_embedding_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream));
    HDS_CHECK_CUDA(cudaMemcpyToSymbolAsync(g_embedding_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream));
    return HDS_OK;
}

}  // namespace hds

using namespace hds;

extern "C" int hds_embedding_forward(int64_t n, int64_t vocab, int64_t columns, int table_type, const void* table,
                                     int ids_type, const void* ids, int has_padding, int64_t padding_id, double scale,
                                     int drop_threshold, uint64_t seed, uint64_t offset, const int64_t* draw,
                                     int out_type, void* out, hds_stream_t stream) {
    clear_error();
    if (int rc = check_arguments("embedding", n, vocab, columns, table_type, out_type, ids_type, scale,
                                 drop_threshold))
        return rc;
    const int channels = (int)columns;
    if (n == 0 || channels == 0) return HDS_OK;
    HDS_REQUIRE((table != nullptr || vocab == 0) && ids != nullptr && out != nullptr, HDS_ERR_INVALID,
                "embedding: null pointer");
    HDS_REQUIRE(!misaligned(table, element_size(table_type)) && !misaligned(out, element_size(out_type)) &&
                    !misaligned(ids, ids_type == HDS_TYPE_I32 ? 4 : 8) && !misaligned(draw, 8),
                HDS_ERR_INVALID, "embedding: misaligned buffer");
    const Ids id = make_ids(ids, ids_type, vocab, has_padding, padding_id);
    const Draw d{seed, offset, draw};
    const float factor = keep_factor(scale, drop_threshold);
    const int v = widest_vector(channels, {{table, table_type}, {out, out_type}});
    return with_types(table_type, out_type, [&](auto t, auto o) -> int {
        using T = decltype(t);
        using O = decltype(o);
        const T* from = static_cast<const T*>(table);
        O* to = static_cast<O*>(out);
        // (A table without rows goes by rows: that kernel reads none of a row of zeros.)
        if (v == 8 || (drop_threshold == 0 && v == 4) || vocab == 0) {
            const int vectors = channels / (v == 2 ? 1 : v);
            const int rows_at_once = std::max(1, THREADS / vectors);
            const int threads = std::min(THREADS, (rows_at_once * vectors + 31) / 32 * 32);
            // A row's threads: all of a block's when it has more vectors than a block has threads.
            const Divider vectors_of = divider((uint32_t)std::min(vectors, THREADS));
            const auto run = [&](auto* kernel, int passes) -> int {
                const int64_t rows = (int64_t)passes * rows_at_once;  // of a block
                const dim3 grid((unsigned)((n + rows - 1) / rows), (unsigned)((vectors + THREADS - 1) / THREADS));
                kernel<<<grid, threads, 0, stream>>>((int)n, channels, vectors, rows_at_once, vectors_of, from, id,
                                                     factor, below_last(drop_threshold), d, to);
                HDS_CHECK_LAUNCH("lookup_rows_kernel");
                return HDS_OK;
            };
            if (drop_threshold > 0 && v == 8) return run(lookup_rows_kernel<T, O, 8, true>, LOOKUP_PASSES<T, O, 8>);
            if (v == 8) return run(lookup_rows_kernel<T, O, 8, false>, LOOKUP_PASSES<T, O, 8>);
            if (v == 4) return run(lookup_rows_kernel<T, O, 4, false>, LOOKUP_PASSES<T, O, 4>);
            return run(lookup_rows_kernel<T, O, 1, false>, LOOKUP_PASSES<T, O, 1>);
        }
        // Blocks of about 1024 groups.  Quotients of numbers below 8 eights channels (d = 0: too wide for them).
        const int eights = std::max(1, 1024 / channels);
        const Divider rows_of = channels <= 16384 ? divider((uint32_t)channels) : Divider{0, 0};
        const unsigned blocks = (unsigned)((n + 8 * eights - 1) / (8 * eights));
        const int whole = widest_vector(8, {{out, out_type}}) == 8;
        const auto run = [&](auto* kernel) -> int {
            kernel<<<blocks, THREADS, 0, stream>>>((int)n, channels, eights, rows_of, from, id, factor,
                                                   below_last(drop_threshold), d, whole, to);
            HDS_CHECK_LAUNCH("lookup_groups_kernel");
            return HDS_OK;
        };
        const int w = widest_vector(channels, {{table, table_type}});
        if (drop_threshold > 0) {
            if (w >= 4) return run(lookup_groups_kernel<T, O, 4, true>);
            if (w == 2) return run(lookup_groups_kernel<T, O, 2, true>);
            return run(lookup_groups_kernel<T, O, 1, true>);
        }
        if (w >= 4) return run(lookup_groups_kernel<T, O, 4, false>);
        if (w == 2) return run(lookup_groups_kernel<T, O, 2, false>);
        return run(lookup_groups_kernel<T, O, 1, false>);
    });
}

extern "C" size_t hds_embedding_backward_scratch_bytes(int64_t n, int64_t vocab, int64_t columns) {
    // Sizes that hds_embedding_backward refuses need none.
    if (check_sizes("embedding_backward", n, vocab, columns) != HDS_OK) return 0;
    const int channels = (int)columns;
    return FewRowsPlan(n, vocab, channels).fits ? 0 : BackwardPlan(n, vocab, channels).bytes;
}

extern "C" int hds_embedding_backward(int64_t n, int64_t vocab, int64_t columns, int grad_type, const void* grad,
                                      int ids_type, const void* ids, int has_padding, int64_t padding_id,
                                      double scale, int drop_threshold, uint64_t seed, uint64_t offset,
                                      const int64_t* draw, int table_type, void* grad_table, int accumulate,
                                      void* scratch, size_t scratch_bytes, hds_stream_t stream) {
    clear_error();
    if (int rc = check_arguments("embedding_backward", n, vocab, columns, table_type, grad_type, ids_type, scale,
                                 drop_threshold))
        return rc;
    const int channels = (int)columns;
    HDS_REQUIRE(!accumulate || table_type == HDS_TYPE_F32, HDS_ERR_UNSUPPORTED,
                "embedding_backward: only an fp32 gradient buffer can be added to");
    if (vocab == 0 || channels == 0) return HDS_OK;
    HDS_REQUIRE(grad_table != nullptr && !misaligned(grad_table, element_size(table_type)), HDS_ERR_INVALID,
                "embedding_backward: null or misaligned table gradient");
    const BackwardPlan plan(n, vocab, channels);
    const FewRowsPlan few(n, vocab, channels);
    if (n > 0) {
        HDS_REQUIRE(grad != nullptr && ids != nullptr, HDS_ERR_INVALID, "embedding_backward: null pointer");
        HDS_REQUIRE(!misaligned(grad, element_size(grad_type)) && !misaligned(ids, ids_type == HDS_TYPE_I32 ? 4 : 8) &&
                        !misaligned(draw, 8),
                    HDS_ERR_INVALID, "embedding_backward: misaligned buffer");
        HDS_REQUIRE(few.fits ||
                        (scratch != nullptr && scratch_bytes >= plan.bytes && !misaligned(scratch, 256)),
                    HDS_ERR_SCRATCH, "embedding_backward: scratch needs %zu bytes, 256-byte aligned", plan.bytes);
    }
    const Draw d{seed, offset, draw};
    const float factor = keep_factor(scale, drop_threshold);
    const Ids id = make_ids(ids, ids_type, vocab, has_padding, padding_id);
    const int v = widest_vector(channels, {{grad, grad_type}, {grad_table, table_type}});
    // Calls run(G{}, T{}, drop, add) with the types and the two switches.
    const auto with_variant = [&](auto&& run) -> int {
        return with_types(table_type, grad_type, [&](auto t, auto g) -> int {
            if constexpr (std::is_same<decltype(t), float>::value) {
                if (accumulate)
                    return drop_threshold > 0 ? run(g, t, std::true_type{}, std::true_type{})
                                              : run(g, t, std::false_type{}, std::true_type{});
            }
            return drop_threshold > 0 ? run(g, t, std::true_type{}, std::false_type{})
                                      : run(g, t, std::false_type{}, std::false_type{});
        });
    };
    if (few.fits) {
        const dim3 grid((unsigned)few.ranges, (unsigned)few.slabs);
        return with_variant([&](auto g, auto t, auto drop, auto add) -> int {
            using G = decltype(g);
            using T = decltype(t);
            const auto launch = [&](auto* kernel) -> int {
                const size_t shared = few_rows_shared_bytes(n, few.range);
                if (shared > DEFAULT_SHARED_BYTES / 2)  // with the kernel's own 17 KB
                    HDS_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                        (int)few_rows_shared_bytes(FEW_ROWS, FEW_RANGE)));
                kernel<<<grid, FEW_THREADS, shared, stream>>>(
                    (int)n, channels, few.range, few.lanes_log2, id, static_cast<const G*>(grad), factor,
                    below_last(drop_threshold), d, static_cast<T*>(grad_table));
                HDS_CHECK_LAUNCH("few_rows_kernel");
                return HDS_OK;
            };
            // Whole vectors or single elements: at these sizes the widths between would save nothing.
            constexpr bool DROP = decltype(drop)::value, ADD = decltype(add)::value;
            if (v == COLUMNS) return launch(few_rows_kernel<G, T, COLUMNS, DROP, ADD>);
            return launch(few_rows_kernel<G, T, 1, DROP, ADD>);
        });
    }
    // The sums write only the rows of codewords that occur.
    if (!accumulate)
        HDS_CHECK_CUDA(cudaMemsetAsync(grad_table, 0, (size_t)vocab * channels * element_size(table_type), stream));
    if (n == 0) return HDS_OK;

    char* s = static_cast<char*>(scratch);
    auto* pairs = reinterpret_cast<uint2*>(s + plan.pairs_a);
    auto* pairs_other = reinterpret_cast<uint2*>(s + plan.pairs_b);
    auto* counts = reinterpret_cast<uint32_t*>(s + plan.counts);
    auto* totals = reinterpret_cast<uint32_t*>(s + plan.totals);
    auto* heads = reinterpret_cast<float*>(s + plan.heads);
    auto* tails = reinterpret_cast<float*>(s + plan.tails);
    const int digits = 1 << plan.digit_bits, tiles = (int)plan.tiles;
    PairSource source{nullptr, id};
    for (int pass = 0; pass < plan.passes; pass++) {
        const int shift = pass * plan.digit_bits;
        const auto run = [&](auto* histogram, auto* scatter) -> int {
            const size_t shared = scatter_shared_bytes(digits, plan.rounds);
            if (shared > DEFAULT_SHARED_BYTES)
                HDS_CHECK_CUDA(cudaFuncSetAttribute(scatter, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                    (int)scatter_shared_bytes(MAX_DIGITS, plan.rounds)));
            histogram<<<tiles, SORT_THREADS, 0, stream>>>((int)n, source, shift, plan.digit_bits, tiles, counts);
            HDS_CHECK_LAUNCH("histogram_kernel");
            if (plan.scan) {
                scan_kernel<<<(digits + SCAN_WARPS - 1) / SCAN_WARPS, 32 * SCAN_WARPS, 0, stream>>>(
                    digits, tiles, counts, totals);
                HDS_CHECK_LAUNCH("scan_kernel");
            }
            scatter<<<tiles, SORT_THREADS, shared, stream>>>((int)n, source, shift, plan.digit_bits, tiles, plan.scan,
                                                             counts, totals, pairs);
            HDS_CHECK_LAUNCH("scatter_kernel");
            return HDS_OK;
        };
        if (int rc = plan.rounds == MANY_ROUNDS ? run(histogram_kernel<MANY_ROUNDS>, scatter_kernel<MANY_ROUNDS>)
                                                : run(histogram_kernel<SOME_ROUNDS>, scatter_kernel<SOME_ROUNDS>))
            return rc;
        source.pairs = pairs;
        std::swap(pairs, pairs_other);
    }
    const uint2* sorted = source.pairs;

    const int slabs = (channels + plan.slab - 1) / plan.slab;
    const int64_t threads = plan.chunks << plan.lanes_log2;
    const unsigned sum_grid = (unsigned)((threads + THREADS - 1) / THREADS * slabs);
    const dim3 join_grid((unsigned)((plan.chunks + JOIN_WORKERS - 1) / JOIN_WORKERS),
                         (unsigned)((channels + JOIN_COLUMNS - 1) / JOIN_COLUMNS));
    return with_variant([&](auto g, auto t, auto drop, auto add) -> int {
        using G = decltype(g);
        using T = decltype(t);
        if (int rc = with_vector(v, [&](auto width) -> int {
                chunk_sum_kernel<G, T, decltype(width)::value, decltype(drop)::value, decltype(add)::value>
                    <<<sum_grid, THREADS, 0, stream>>>(n, (uint32_t)vocab, channels, plan.slab, plan.lanes_log2,
                                                       plan.chunk, slabs, sorted, static_cast<const G*>(grad), factor,
                                                       below_last(drop_threshold), d, static_cast<T*>(grad_table),
                                                       heads, tails, plan.stride);
                HDS_CHECK_LAUNCH("chunk_sum_kernel");
                return HDS_OK;
            }))
            return rc;
        if (plan.chunks == 1) return HDS_OK;
        const auto join = [&](auto* kernel) -> int {
            kernel<<<join_grid, THREADS, 0, stream>>>(n, (uint32_t)vocab, channels, plan.chunk, sorted, heads,
                                                      tails, plan.stride, factor, static_cast<T*>(grad_table));
            HDS_CHECK_LAUNCH("join_kernel");
            return HDS_OK;
        };
        if (v == COLUMNS) return join(join_kernel<T, COLUMNS, decltype(add)::value>);
        return join(join_kernel<T, 1, decltype(add)::value>);
    });
}
