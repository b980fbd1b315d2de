// embedding.cu -- the codebook lookup out[i] = f * table[ids[i]] and its gradient
// dtable[v] = f * sum over the i with ids[i] = v of dout[i], both with optional dropout of the looked-up
// elements in the same pass (philox.cuh): f = scale / kept share, dropped elements 0 in both directions.
//
// Lookup.  One pass: the output is written once, the table's rows come from the L2 when the codebook is
// smaller than it.
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

struct Padding {
    int present;
    int64_t id;
};

// The table row of an id, or -1 for a row of zeros (padding, or outside the table: recorded).
__device__ __forceinline__ int64_t table_row(int64_t v, int64_t vocab, const Padding& padding) {
    if (padding.present && v == padding.id) return -1;
    if (v < 0 || v >= vocab) {
        atomicExch(&g_embedding_status, HDS_ERR_INVALID);
        return -1;
    }
    return v;
}

constexpr int THREADS = 256;
constexpr size_t DEFAULT_SHARED_BYTES = 48 << 10;  // a block may have more on request

// ---------------------------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------------------------
// A warp writes tiles of 256 consecutive output elements in vectors of V, the widest into which rows
// split and to which both buffers are aligned.  All of a warp's ids are loaded first, then all of its
// table vectors, then it stores: TILES x 8 elements in flight per lane cover the two dependent loads.
// Dropout: lane j draws group j of the tile, the holder of an element fetches its group's decisions with
// a shuffle (itself when V = 8).
constexpr int TILE_ELEMENTS = 256;
constexpr int TILES = 4;
constexpr int LOOKUP_ELEMENTS = THREADS / 32 * TILE_ELEMENTS * TILES;  // per block

struct Ids {
    const void* p;
    int wide;  // int64 (else int32)
    __device__ __forceinline__ int64_t operator[](int64_t i) const {
        return wide ? __ldg(static_cast<const long long*>(p) + i) : (int64_t)__ldg(static_cast<const int*>(p) + i);
    }
    // The ids first, first + step, ... below n (0 beyond), loaded together.
    template <int COUNT>
    __device__ __forceinline__ void load(int64_t first, int64_t step, int64_t n, int64_t (&id)[COUNT]) const {
        if (wide) {
#pragma unroll
            for (int r = 0; r < COUNT; r++)
                id[r] = first + r * step < n ? __ldg(static_cast<const long long*>(p) + first + r * step) : 0;
        } else {
#pragma unroll
            for (int r = 0; r < COUNT; r++)
                id[r] = first + r * step < n ? __ldg(static_cast<const int*>(p) + first + r * step) : 0;
        }
    }
};

template <typename T, typename O, int V, bool DROP>
__global__ void __launch_bounds__(THREADS) lookup_kernel(int64_t total, int64_t vocab, int channels, Divider rows_of,
                                                         const T* __restrict__ table, Ids ids, Padding padding,
                                                         float factor, uint32_t last, Draw draw,
                                                         O* __restrict__ out) {
    constexpr int STEPS = 8 / V;
    if (DROP) draw = resolve(draw);
    const int lane = threadIdx.x & 31;
    const int in_block = (threadIdx.x >> 5) * (TILE_ELEMENTS * TILES);
    const int64_t warp_base = (int64_t)blockIdx.x * LOOKUP_ELEMENTS + in_block;
    if (warp_base >= total) return;
    // A block's groups share the upper counter word: its first is a multiple of their number.
    const uint64_t group0 = (uint64_t)blockIdx.x * (LOOKUP_ELEMENTS / 8);
    const int64_t row0 = warp_base / channels;
    const uint32_t place = (uint32_t)(warp_base - row0 * channels);
    int64_t id[TILES][STEPS];
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            const uint32_t e = t * TILE_ELEMENTS + (k * 32 + lane) * V;
            id[t][k] = warp_base + e < total ? ids[row0 + rows_of.quotient(place + e)] : 0;
        }
    int64_t at[TILES][STEPS];  // the vector's first element in the table, or -1
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            const uint32_t e = t * TILE_ELEMENTS + (k * 32 + lane) * V;
            const int64_t row = warp_base + e < total ? table_row(id[t][k], vocab, padding) : -1;
            const uint32_t q = rows_of.quotient(place + e);
            at[t][k] = row < 0 ? -1 : row * channels + (place + e - q * channels);
        }
    Vec<T, V> v[TILES][STEPS];
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            v[t][k] = Vec<T, V>{};
            if (at[t][k] >= 0) v[t][k] = load_shared_data<T, V>(table + at[t][k]);
        }
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        Numbers8 numbers{};
        uint32_t bits = 0;
        if (DROP) {
            numbers = philox4x32_10((uint32_t)group0 + (in_block + t * TILE_ELEMENTS) / 8 + lane,
                                    (uint32_t)(group0 >> 32), draw);
            if (V < 8) bits = numbers.bits(last);
        }
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            const int e = (k * 32 + lane) * V;
            uint32_t mine = 0;
            if (DROP && V < 8) mine = __shfl_sync(FULL_MASK, bits, e >> 3) >> (e & 7);
            Vec<O, V> r;
#pragma unroll
            for (int j = 0; j < V; j++) {
                // A row of zeros stays one: its table vector was set to zero.
                const bool kept = !DROP || (V == 8 ? numbers.kept(j, last) : ((mine >> j) & 1u) != 0);
                r.set(j, kept ? v[t][k].get(j) * factor : 0.0f);
            }
            const int64_t to = warp_base + t * TILE_ELEMENTS + e;
            if (to < total) store<O, V>(out + to, r);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// stable radix sort of (codeword, row number)
// ---------------------------------------------------------------------------------------------
// Lanes of the warp with this lane's digit (`bits` bits; among the valid lanes): a vote per bit.  The
// __match_any_sync instruction, which finds the same, took about 100 cycles of an SM here: 17 us for a
// tile's histogram that takes 3 with votes.
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
// per tile, a scan that turns the digit-major counts into output positions, and a scatter that ranks the
// tile's keys.  The first pass reads the ids themselves.  No block waits for another.
constexpr int SORT_THREADS = 512;
constexpr int SORT_WARPS = SORT_THREADS / 32;
// Keys per thread: 16 (a tile is 8192 keys) when that still gives every SM a tile, else 4.
constexpr int MANY_ROUNDS = 16, SOME_ROUNDS = 4;
constexpr int MAX_DIGIT_BITS = 11;
constexpr int MAX_DIGITS = 1 << MAX_DIGIT_BITS;

// The keys of a pass.  The first pass makes them from the ids; all of a thread's ids are loaded before the
// first is looked at, since an id outside the table is recorded, a side effect that orders what follows.
struct KeySource {
    const uint32_t* keys;  // sorted so far, or NULL in the first pass:
    const int32_t* rows;
    Ids ids;
    Padding padding;
    int64_t vocab;

    // keys of the elements first, first + step, ... below n (0 beyond).
    template <int COUNT>
    __device__ __forceinline__ void load(int64_t first, int step, int64_t n, uint32_t (&key)[COUNT]) const {
        if (keys != nullptr) {
#pragma unroll
            for (int r = 0; r < COUNT; r++) key[r] = first + r * step < n ? __ldg(keys + first + r * step) : 0;
            return;
        }
        int64_t id[COUNT];
        ids.load<COUNT>(first, step, n, id);
#pragma unroll
        for (int r = 0; r < COUNT; r++) {
            const int64_t row = first + r * step < n ? table_row(id[r], vocab, padding) : 0;
            key[r] = (uint32_t)(row < 0 ? vocab : row);
        }
    }
    template <int COUNT>
    __device__ __forceinline__ void load_rows(int64_t first, int step, int64_t n, int32_t (&row)[COUNT]) const {
#pragma unroll
        for (int r = 0; r < COUNT; r++) {
            const int64_t i = first + r * step;
            row[r] = rows == nullptr ? (int32_t)i : i < n ? __ldg(rows + i) : 0;
        }
    }
};

// counts[digit][tile] and totals[digit] (cleared by the caller; integer adds, so their order is no matter).
template <int ROUNDS>
__global__ void __launch_bounds__(SORT_THREADS) histogram_kernel(int64_t n, KeySource source, int shift, int bits,
                                                                 int tiles, uint32_t* __restrict__ counts,
                                                                 uint32_t* __restrict__ totals) {
    __shared__ uint32_t hist[MAX_DIGITS];
    const int digits = 1 << bits;
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) hist[d] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * (SORT_THREADS * ROUNDS) + threadIdx.x;
    const int lane = threadIdx.x & 31;
    uint32_t key[ROUNDS];
    source.load<ROUNDS>(base, SORT_THREADS, n, key);
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const bool valid = base + r * SORT_THREADS < n;
        const uint32_t d = (key[r] >> shift) & (digits - 1);
        // One shared atomic per distinct digit of the warp: popular codewords would serialise otherwise.
        const uint32_t peers = lanes_alike(d, bits, valid);
        if (valid && lane == __ffs(peers) - 1) atomicAdd(&hist[d], __popc(peers));
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) {
        const uint32_t c = hist[d];
        counts[(int64_t)d * tiles + blockIdx.x] = c;
        if (c) atomicAdd(&totals[d], c);
    }
}

// counts[digit][tile] -> the position of the tile's first key of that digit.  A warp per digit: its base
// is the sum of the totals of all smaller digits, then a scan along the tiles.
constexpr int SCAN_WARPS = 8;

__global__ void __launch_bounds__(32 * SCAN_WARPS) scan_kernel(int digits, int tiles,
                                                               const uint32_t* __restrict__ totals,
                                                               uint32_t* __restrict__ counts) {
    const int lane = threadIdx.x & 31, digit = blockIdx.x * SCAN_WARPS + (threadIdx.x >> 5);
    if (digit >= digits) return;
    uint32_t base = 0;
#pragma unroll 8
    for (int d = lane; d < digit; d += 32) base += totals[d];
    base = __reduce_add_sync(FULL_MASK, base);
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
}

// Each warp ranks its own consecutive keys into a count table of its own; a scan over the warps then
// places the tables one after another.
inline size_t scatter_shared_bytes(int digits) { return (size_t)digits * (sizeof(uint32_t) + 2 * SORT_WARPS); }

template <int ROUNDS>
__global__ void __launch_bounds__(SORT_THREADS) scatter_kernel(int64_t n, KeySource source, int shift, int bits,
                                                               int tiles, const uint32_t* __restrict__ positions,
                                                               uint32_t* __restrict__ keys_out,
                                                               int32_t* __restrict__ rows_out) {
    extern __shared__ uint32_t s_base[];                                  // [digits]
    const int digits = 1 << bits;
    uint16_t* s_warp = reinterpret_cast<uint16_t*>(s_base + digits);      // [warps][digits]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t base = (int64_t)blockIdx.x * (SORT_THREADS * ROUNDS) + warp * (32 * ROUNDS) + lane;
    uint16_t* mine = s_warp + warp * digits;
    uint32_t key[ROUNDS];
    int32_t row[ROUNDS];
    uint16_t rank[ROUNDS];
    source.load<ROUNDS>(base, 32, n, key);
    source.load_rows<ROUNDS>(base, 32, n, row);
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) s_base[d] = positions[(int64_t)d * tiles + blockIdx.x];
    for (int d = threadIdx.x; d < digits * SORT_WARPS / 2; d += SORT_THREADS) reinterpret_cast<uint32_t*>(s_warp)[d] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
        const bool valid = base + 32 * r < n;
        const uint32_t d = (key[r] >> shift) & (digits - 1);
        const uint32_t peers = lanes_alike(d, bits, valid);
        const uint32_t before = mine[d];
        __syncwarp();
        rank[r] = (uint16_t)(before + __popc(peers & ((1u << lane) - 1u)));
        if (valid && lane == __ffs(peers) - 1) mine[d] = (uint16_t)(before + __popc(peers));
        __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) {
        uint32_t run = 0;
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
        const uint32_t d = (key[r] >> shift) & (digits - 1);
        const uint32_t pos = s_base[d] + mine[d] + rank[r];
        keys_out[pos] = key[r];
        rows_out[pos] = row[r];
    }
}

// ---------------------------------------------------------------------------------------------
// sums by codeword
// ---------------------------------------------------------------------------------------------
// The sorted rows are cut into chunks of equal length whatever the codewords' popularity.  A worker, a
// group of 1 to 32 lanes with 8 columns each, adds up one chunk's rows in registers.  A codeword that
// begins and ends inside the chunk goes straight to the table.  The sum of a codeword that began in an
// earlier chunk is the chunk's head, that of one that goes on into the next its tail; join_kernel adds a
// tail and the heads that follow it.
constexpr int COLUMNS = 8;       // per lane
constexpr int ROWS_AHEAD = 4;    // rows loaded before the first is added

template <typename T, int V, bool ACCUMULATE>
__device__ __forceinline__ void store_sum(T* p, const float* sum, float factor) {
    Vec<T, V> r;
    if (ACCUMULATE) r = load_once<T, V>(p);
#pragma unroll
    for (int j = 0; j < V; j++) r.set(j, ACCUMULATE ? fmaf(factor, sum[j], r.get(j)) : factor * sum[j]);
    store<T, V>(p, r);
}

template <typename G, typename T, int V, bool DROP, bool ACCUMULATE>
__global__ void __launch_bounds__(THREADS) chunk_sum_kernel(int64_t n, uint32_t vocab, int channels, int slab,
                                                            int lanes_log2, int chunk,
                                                            const uint32_t* __restrict__ keys,
                                                            const int32_t* __restrict__ rows,
                                                            const G* __restrict__ grad, float factor,
                                                            uint32_t last, Draw draw, T* __restrict__ table,
                                                            float* __restrict__ heads, float* __restrict__ tails,
                                                            int stride) {
    constexpr int STEPS = COLUMNS / V;
    if (DROP) draw = resolve(draw);
    const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
    const int64_t id = ((int64_t)blockIdx.x * THREADS + threadIdx.x) >> lanes_log2;  // of the chunk
    const int64_t start = id * chunk;
    const int c0 = blockIdx.y * slab, width = min(slab, channels - c0);
    const auto column = [&](int k) { return (k * lanes + lane) * V; };  // within the slab
    uint32_t current = start < n ? keys[start] : vocab;
    bool began_earlier = start < n && start > 0 && keys[start - 1] == current;
    float sum[COLUMNS];
#pragma unroll
    for (int j = 0; j < COLUMNS; j++) sum[j] = 0.0f;

    const auto put = [&](float* partial) {
#pragma unroll
        for (int k = 0; k < STEPS; k++)
            if (column(k) < width) store_sum<float, V, false>(partial + id * stride + c0 + column(k), sum + k * V, 1.0f);
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
        // Chunks start at multiples of 8, so the four keys and rows are two 16-byte loads (the buffers are
        // padded beyond n).
        const int64_t pos = start + p;
        uint4 key4 = make_uint4(vocab, vocab, vocab, vocab);
        int4 row4 = make_int4(0, 0, 0, 0);
        if (pos < n) {
            key4 = __ldg(reinterpret_cast<const uint4*>(keys + pos));
            row4 = __ldg(reinterpret_cast<const int4*>(rows + pos));
        }
        const uint32_t key[ROWS_AHEAD] = {key4.x, pos + 1 < n ? key4.y : vocab, pos + 2 < n ? key4.z : vocab,
                                          pos + 3 < n ? key4.w : vocab};
        const int32_t row[ROWS_AHEAD] = {row4.x, row4.y, row4.z, row4.w};
        Vec<G, V> g[ROWS_AHEAD][STEPS];
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; u++)
#pragma unroll
            for (int k = 0; k < STEPS; k++)
                if (key[u] != vocab && column(k) < width)
                    g[u][k] = load_once<G, V>(grad + (int64_t)row[u] * channels + c0 + column(k));
        Numbers8 numbers[ROWS_AHEAD];
        uint32_t keep[ROWS_AHEAD][STEPS];
        if (DROP) {
#pragma unroll
            for (int u = 0; u < ROWS_AHEAD; u++) {
                const int64_t e = (int64_t)(key[u] != vocab ? row[u] : 0) * channels + c0;
                numbers[u] = philox4x32_10((uint64_t)(e >> 3) + lane, draw);
                if (V < COLUMNS) {
                    const uint32_t bits = numbers[u].bits(last);
                    // The row may start inside a group: its last columns then belong to one group more.
                    const int into = (int)(e & 7);
                    const uint32_t more =
                        into + width > 8 * lanes ? philox4x32_10((uint64_t)(e >> 3) + lanes, draw).bits(last) : 0;
#pragma unroll
                    for (int k = 0; k < STEPS; k++) {
                        const int b = into + column(k);
                        const uint32_t theirs = __shfl_sync(FULL_MASK, bits, b >> 3, lanes);
                        keep[u][k] = ((b >> 3) < lanes ? theirs : more) >> (b & 7);
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; u++) {
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
                    if (!DROP || (V == COLUMNS ? numbers[u].kept(j, last) : ((keep[u][k] >> j) & 1u) != 0))
                        sum[k * V + j] += g[u][k].get(j);
        }
    }
    if (current == vocab) return;
    const int64_t end = start + chunk;
    if (end < n && keys[end] == current)
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
                                                       const uint32_t* __restrict__ keys,
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
        const uint32_t codeword = keys[end], at_end = keys[end - 1], at_start = keys[start];
        const uint32_t before = start > 0 ? keys[start - 1] : vocab;
        // The key with which the h-th chunk after the next one begins.
        const auto key_after = [&](int h) { return id + 1 + h < chunks ? keys[(id + 1 + h) * chunk] : vocab; };
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
        const uint32_t codeword = keys[(from + 1) * chunk];
        // The last chunk that begins with the codeword lies in [last, beyond).
        int64_t last = from + 1, beyond = chunks;
        while (beyond - last > 1) {
            const int64_t step = (beyond - last + THREADS - 1) / THREADS;
            const int64_t probe = last + (threadIdx.x + 1) * step;
            const int hits = __syncthreads_count(probe < beyond && keys[probe * chunk] == codeword);
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
// A block owns a range of codewords and 32 columns and does everything for them: it reads all ids, keeps
// the rows whose codeword is its own, groups them by codeword in shared memory (the scatter's ranking:
// row order stays), adds each codeword's rows and writes every row of its range, zeros included.  Each
// block reads all the ids, which is cheap while there are few; in return nothing waits for a second
// launch.  A worker of 4 lanes (8 columns each) adds the rows of a codeword; one with many rows is added
// by the whole block in 128 interleaved runs and a tree.
constexpr int FEW_ROWS = 8192;
constexpr int FEW_THREADS = 512;
constexpr int FEW_WARPS = FEW_THREADS / 32;
constexpr int FEW_WORKERS = FEW_THREADS / JOIN_LANES;
constexpr int FEW_RANGE = 2 * FEW_THREADS;  // codewords per block at most
constexpr int SHORT_ROWS = 32;

inline size_t few_rows_shared_bytes(int64_t n, int range) {
    return (size_t)(range + 1) * 4 + (size_t)range * FEW_WARPS * 2 + (size_t)n * 2;
}

template <typename G, typename T, int V, bool DROP, bool ACCUMULATE>
__global__ void __launch_bounds__(FEW_THREADS) few_rows_kernel(int n, int64_t vocab, int channels, int range, Ids ids,
                                                               Padding padding, const G* __restrict__ grad,
                                                               float factor, uint32_t last, Draw draw,
                                                               T* __restrict__ table) {
    constexpr int STEPS = COLUMNS / V;
    extern __shared__ uint32_t s_start[];                                    // [range + 1]
    uint16_t* s_count = reinterpret_cast<uint16_t*>(s_start + range + 1);    // [warps][range]
    uint16_t* s_rows = s_count + FEW_WARPS * range;                          // [n]
    __shared__ float s_sum[FEW_WORKERS][JOIN_COLUMNS];
    __shared__ uint32_t s_warp[FEW_WARPS];
    __shared__ int s_long;
    __shared__ uint16_t s_long_codeword[FEW_ROWS / SHORT_ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane32 = tid & 31;
    const int64_t first = (int64_t)blockIdx.x * range;
    const int here = (int)min((int64_t)range, vocab - first);
    const int bits = 32 - __clz(range - 1);  // of a codeword's number in the range
    if (DROP) draw = resolve(draw);
    for (int i = tid; i < FEW_WARPS * range; i += FEW_THREADS) s_count[i] = 0;
    if (tid == 0) s_long = 0;
    __syncthreads();

    // The block's rows by codeword: counts, positions, rows.
    const int per_warp = (n + FEW_THREADS - 1) / FEW_THREADS * 32;
    const int begin = warp * per_warp, end = min(n, begin + per_warp);
    uint16_t* mine = s_count + warp * range;
    // The numbers in the range of the codewords of 4 x 32 rows (FEW_RANGE: not in it).
    constexpr int BATCH = 4;
    const auto local_codewords = [&](int i0, uint32_t (&d)[BATCH]) {
        int64_t id[BATCH];
        ids.load<BATCH>(i0 + lane32, 32, end, id);
#pragma unroll
        for (int r = 0; r < BATCH; r++) {
            const int64_t row = i0 + 32 * r + lane32 < end ? table_row(id[r], vocab, padding) : -1;
            d[r] = row >= first && row < first + here ? (uint32_t)(row - first) : (uint32_t)FEW_RANGE;
        }
    };
    for (int i0 = begin; i0 < end; i0 += 32 * BATCH) {
        uint32_t d[BATCH];
        local_codewords(i0, d);
#pragma unroll
        for (int r = 0; r < BATCH; r++) {
            const uint32_t peers = lanes_alike(d[r], bits, d[r] < FEW_RANGE);
            if (d[r] < FEW_RANGE && lane32 == __ffs(peers) - 1) mine[d[r]] = (uint16_t)(mine[d[r]] + __popc(peers));
            __syncwarp();
        }
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
    for (int i0 = begin; i0 < end; i0 += 32 * BATCH) {
        uint32_t d[BATCH];
        local_codewords(i0, d);
#pragma unroll
        for (int r = 0; r < BATCH; r++) {
            const uint32_t peers = lanes_alike(d[r], bits, d[r] < FEW_RANGE);
            const uint32_t at = d[r] < FEW_RANGE ? mine[d[r]] : 0;
            __syncwarp();
            if (d[r] < FEW_RANGE) {
                s_rows[at + __popc(peers & ((1u << lane32) - 1u))] = (uint16_t)(i0 + 32 * r + lane32);
                if (lane32 == __ffs(peers) - 1) mine[d[r]] = (uint16_t)(at + __popc(peers));
            }
            __syncwarp();
        }
    }
    __syncthreads();

    const int worker = tid / JOIN_LANES, lane = tid % JOIN_LANES;
    const unsigned worker_mask = 0xfu << (lane32 & ~(JOIN_LANES - 1));
    const int c0 = blockIdx.y * JOIN_COLUMNS, width = min(JOIN_COLUMNS, channels - c0);
    const auto column = [&](int k) { return (k * JOIN_LANES + lane) * V; };
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
                    const uint32_t bits = philox4x32_10((uint64_t)(e >> 3) + lane, draw).bits(last);
                    const int into = (int)(e & 7);
                    const uint32_t more = V < COLUMNS && into + width > JOIN_COLUMNS
                                              ? philox4x32_10((uint64_t)(e >> 3) + JOIN_LANES, draw).bits(last)
                                              : 0;
#pragma unroll
                    for (int k = 0; k < STEPS; k++) {
                        const int b = into + column(k);
                        uint32_t theirs = bits;
                        if (V < COLUMNS) {
                            theirs = __shfl_sync(worker_mask, bits, b >> 3, JOIN_LANES);
                            theirs = ((b >> 3) < JOIN_LANES ? theirs : more) >> (b & 7);
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
                store_sum<T, V, ACCUMULATE>(table + (first + codeword) * channels + c0 + column(k), sum + k * V,
                                            factor);
    };
    for (int v = worker; v < here; v += FEW_WORKERS) {
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
        add_rows(sum, s_start[v] + worker, s_start[v + 1], FEW_WORKERS);
#pragma unroll
        for (int j = 0; j < COLUMNS; j++) s_sum[worker][lane * COLUMNS + j] = sum[j];
        __syncthreads();
        for (int half = FEW_WORKERS / 2; half > 0; half /= 2) {
            for (int i = tid; i < half * JOIN_COLUMNS; i += FEW_THREADS)
                s_sum[i / JOIN_COLUMNS][i % JOIN_COLUMNS] += s_sum[i / JOIN_COLUMNS + half][i % JOIN_COLUMNS];
            __syncthreads();
        }
        if (worker == 0) write(v, s_sum[0] + lane * COLUMNS);
        __syncthreads();
    }
}

// Codewords per block: enough blocks to fill the machine, at most FEW_RANGE codewords each.
int few_rows_range(int64_t vocab, int channels) {
    const int64_t slabs = (channels + JOIN_COLUMNS - 1) / JOIN_COLUMNS;
    const int64_t blocks = std::max<int64_t>((vocab + FEW_RANGE - 1) / FEW_RANGE, std::min(vocab, 444 / slabs + 1));
    return (int)((vocab + blocks - 1) / blocks);
}

// Few rows, and the blocks' reads of all ids together no more than 16M.
bool few_rows(int64_t n, int64_t vocab, int channels) {
    if (n > FEW_ROWS || vocab == 0 || channels == 0) return false;
    const int64_t slabs = (channels + JOIN_COLUMNS - 1) / JOIN_COLUMNS;
    const int range = few_rows_range(vocab, channels);
    return (vocab + range - 1) / range * slabs * n <= (int64_t(1) << 24);
}

int ceil_log2(int64_t x) {
    int bits = 0;
    while ((int64_t(1) << bits) < x) bits++;
    return bits;
}

// How the backward splits its work and lays out its scratch.
struct BackwardPlan {
    int rounds;               // of the sort, per thread of a tile
    int64_t tiles;
    int passes, digit_bits;
    int chunk, stride;        // rows per chunk; floats per partial row
    int64_t chunks;
    int slab, lanes_log2;     // columns and lanes of a worker
    size_t keys_a, keys_b, rows_a, rows_b, counts, totals, heads, tails, bytes;

    BackwardPlan(int64_t n, int64_t vocab, int channels) {
        const size_t nn = (size_t)std::max<int64_t>(n, 1);
        rounds = (int64_t)nn >= 120 * SORT_THREADS * MANY_ROUNDS ? MANY_ROUNDS : SOME_ROUNDS;
        tiles = ((int64_t)nn + SORT_THREADS * rounds - 1) / (SORT_THREADS * rounds);
        const int bits = std::max(1, ceil_log2(vocab + 1));  // keys 0 .. vocab
        passes = (bits + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
        digit_bits = (bits + passes - 1) / passes;
        // Long chunks write few partial sums (two rows of a chunk at most); but the chunks have to fill the
        // machine.  75,000 lanes with four rows of 32 bytes each in flight are about 10 MB, more than the
        // memory's latency times its rate.
        const int64_t wanted = (int64_t)nn * std::max(channels, 1) / COLUMNS / 75000;
        chunk = 8;
        while (chunk < 128 && chunk < wanted) chunk *= 2;
        chunks = ((int64_t)nn + chunk - 1) / chunk;
        stride = (channels + COLUMNS - 1) / COLUMNS * COLUMNS;
        const int slabs = std::max(1, (channels + 32 * COLUMNS - 1) / (32 * COLUMNS));
        slab = ((channels + slabs - 1) / slabs + COLUMNS - 1) / COLUMNS * COLUMNS;
        lanes_log2 = ceil_log2(std::max(slab / COLUMNS, 1));
        keys_a = 0;
        keys_b = keys_a + align256(nn * 4);
        rows_a = keys_b + align256(nn * 4);
        rows_b = rows_a + align256(nn * 4);
        counts = rows_b + align256(nn * 4);
        totals = counts + align256(((size_t)tiles << digit_bits) * 4);
        heads = totals + align256(((size_t)passes << digit_bits) * 4);
        tails = heads + align256((size_t)chunks * stride * 4);
        bytes = tails + align256((size_t)chunks * stride * 4);
    }
};

// Shared argument checks of both directions.
int check_arguments(const char* what, int64_t n, int64_t vocab, int channels, int table_type, int value_type,
                    int ids_type, double scale, int drop_threshold) {
    HDS_REQUIRE(n >= 0 && vocab >= 0 && channels >= 0, HDS_ERR_INVALID, "%s: negative size", what);
    HDS_REQUIRE(n < INT32_MAX && vocab < INT32_MAX && channels <= HDS_EMBEDDING_MAX_CHANNELS, HDS_ERR_TOO_LARGE,
                "%s: n = %lld, vocab = %lld, channels = %d is too large", what, (long long)n, (long long)vocab,
                channels);
    HDS_REQUIRE(known_type(table_type) && (value_type == table_type || value_type == HDS_TYPE_F32),
                HDS_ERR_UNSUPPORTED, "%s: values must be of the table's type or fp32", what);
    HDS_REQUIRE(ids_type == HDS_TYPE_I32 || ids_type == HDS_TYPE_I64, HDS_ERR_UNSUPPORTED,
                "%s: ids must be int32 or int64", what);
    HDS_REQUIRE(scale - scale == 0.0, HDS_ERR_INVALID, "%s: scale must be finite", what);
    HDS_REQUIRE(drop_threshold >= 0 && drop_threshold <= DROP_ONE, HDS_ERR_INVALID,
                "%s: dropout threshold %d outside 0 to 65536", what, drop_threshold);
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

extern "C" int hds_embedding_forward(int64_t n, int64_t vocab, int channels, int table_type, const void* table,
                                     int ids_type, const void* ids, int has_padding, int64_t padding_id, double scale,
                                     int drop_threshold, uint64_t seed, uint64_t offset, const int64_t* draw,
                                     int out_type, void* out, hds_stream_t stream) {
    clear_error();
    if (int rc = check_arguments("embedding", n, vocab, channels, table_type, out_type, ids_type, scale,
                                 drop_threshold))
        return rc;
    if (n == 0 || channels == 0) return HDS_OK;
    HDS_REQUIRE((table != nullptr || vocab == 0) && ids != nullptr && out != nullptr, HDS_ERR_INVALID,
                "embedding: null pointer");
    HDS_REQUIRE(!misaligned(table, element_size(table_type)) && !misaligned(out, element_size(out_type)) &&
                    !misaligned(ids, ids_type == HDS_TYPE_I32 ? 4 : 8) && !misaligned(draw, 8),
                HDS_ERR_INVALID, "embedding: misaligned buffer");
    const Padding padding{has_padding, padding_id};
    const Draw d{seed, offset, draw};
    const float factor = keep_factor(scale, drop_threshold);
    const int64_t total = n * channels;
    const int64_t blocks = (total + LOOKUP_ELEMENTS - 1) / LOOKUP_ELEMENTS;
    HDS_REQUIRE(blocks <= INT32_MAX, HDS_ERR_TOO_LARGE, "embedding: n = %lld, channels = %d is too large",
                (long long)n, channels);
    const Ids id{ids, ids_type == HDS_TYPE_I64};
    const Divider rows_of = divider((uint32_t)channels);
    return with_types(table_type, out_type, [&](auto t, auto o) -> int {
        using T = decltype(t);
        using O = decltype(o);
        return with_vector(widest_vector(channels, {{table, table_type}, {out, out_type}}), [&](auto width) -> int {
            constexpr int V = decltype(width)::value;
            if (drop_threshold > 0)
                lookup_kernel<T, O, V, true><<<(unsigned)blocks, THREADS, 0, stream>>>(
                    total, vocab, channels, rows_of, static_cast<const T*>(table), id, padding, factor,
                    below_last(drop_threshold), d, static_cast<O*>(out));
            else
                lookup_kernel<T, O, V, false><<<(unsigned)blocks, THREADS, 0, stream>>>(
                    total, vocab, channels, rows_of, static_cast<const T*>(table), id, padding, factor, 0u, d,
                    static_cast<O*>(out));
            HDS_CHECK_LAUNCH("lookup_kernel");
            return HDS_OK;
        });
    });
}

extern "C" size_t hds_embedding_backward_scratch_bytes(int64_t n, int64_t vocab, int channels) {
    return few_rows(n, vocab, channels) ? 0 : BackwardPlan(n, vocab, channels).bytes;
}

extern "C" int hds_embedding_backward(int64_t n, int64_t vocab, int channels, int grad_type, const void* grad,
                                      int ids_type, const void* ids, int has_padding, int64_t padding_id,
                                      double scale, int drop_threshold, uint64_t seed, uint64_t offset,
                                      const int64_t* draw, int table_type, void* grad_table, int accumulate,
                                      void* scratch, size_t scratch_bytes, hds_stream_t stream) {
    clear_error();
    if (int rc = check_arguments("embedding_backward", n, vocab, channels, table_type, grad_type, ids_type, scale,
                                 drop_threshold))
        return rc;
    HDS_REQUIRE(!accumulate || table_type == HDS_TYPE_F32, HDS_ERR_UNSUPPORTED,
                "embedding_backward: only an fp32 gradient buffer can be added to");
    if (vocab == 0 || channels == 0) return HDS_OK;
    HDS_REQUIRE(grad_table != nullptr && !misaligned(grad_table, element_size(table_type)), HDS_ERR_INVALID,
                "embedding_backward: null or misaligned table gradient");
    const BackwardPlan plan(n, vocab, channels);
    if (n > 0) {
        HDS_REQUIRE(grad != nullptr && ids != nullptr, HDS_ERR_INVALID, "embedding_backward: null pointer");
        HDS_REQUIRE(!misaligned(grad, element_size(grad_type)) && !misaligned(ids, ids_type == HDS_TYPE_I32 ? 4 : 8) &&
                        !misaligned(draw, 8),
                    HDS_ERR_INVALID, "embedding_backward: misaligned buffer");
        HDS_REQUIRE(few_rows(n, vocab, channels) ||
                        (scratch != nullptr && scratch_bytes >= plan.bytes && !misaligned(scratch, 256)),
                    HDS_ERR_SCRATCH, "embedding_backward: scratch needs %zu bytes, 256-byte aligned", plan.bytes);
    }
    const Draw d{seed, offset, draw};
    const float factor = keep_factor(scale, drop_threshold);
    const Ids id{ids, ids_type == HDS_TYPE_I64};
    const Padding padding{has_padding, padding_id};
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
    if (n > 0 && few_rows(n, vocab, channels)) {
        const int range = few_rows_range(vocab, channels);
        const dim3 grid((unsigned)((vocab + range - 1) / range), (unsigned)((channels + JOIN_COLUMNS - 1) / JOIN_COLUMNS));
        return with_variant([&](auto g, auto t, auto drop, auto add) -> int {
            using G = decltype(g);
            using T = decltype(t);
            const auto launch = [&](auto* kernel) -> int {
                const size_t shared = few_rows_shared_bytes(n, range);
                if (shared > DEFAULT_SHARED_BYTES / 2)  // with the kernel's own 17 KB
                    HDS_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                        (int)few_rows_shared_bytes(FEW_ROWS, FEW_RANGE)));
                kernel<<<grid, FEW_THREADS, shared, stream>>>(
                    (int)n, vocab, channels, range, id, padding, static_cast<const G*>(grad), factor,
                    below_last(drop_threshold), d, static_cast<T*>(grad_table));
                HDS_CHECK_LAUNCH("few_rows_kernel");
                return HDS_OK;
            };
            // Whole vectors or single elements: at these sizes the widths between would save nothing.
            if (v == COLUMNS) return launch(few_rows_kernel<G, T, COLUMNS, decltype(drop)::value, decltype(add)::value>);
            return launch(few_rows_kernel<G, T, 1, decltype(drop)::value, decltype(add)::value>);
        });
    }
    // The sums write only the rows of codewords that occur.
    if (!accumulate)
        HDS_CHECK_CUDA(cudaMemsetAsync(grad_table, 0, (size_t)vocab * channels * element_size(table_type), stream));
    if (n == 0) return HDS_OK;

    char* s = static_cast<char*>(scratch);
    auto* keys = reinterpret_cast<uint32_t*>(s + plan.keys_a);
    auto* keys_other = reinterpret_cast<uint32_t*>(s + plan.keys_b);
    auto* rows = reinterpret_cast<int32_t*>(s + plan.rows_a);
    auto* rows_other = reinterpret_cast<int32_t*>(s + plan.rows_b);
    auto* counts = reinterpret_cast<uint32_t*>(s + plan.counts);
    auto* totals = reinterpret_cast<uint32_t*>(s + plan.totals);
    auto* heads = reinterpret_cast<float*>(s + plan.heads);
    auto* tails = reinterpret_cast<float*>(s + plan.tails);
    const int digits = 1 << plan.digit_bits, tiles = (int)plan.tiles;
    HDS_CHECK_CUDA(cudaMemsetAsync(totals, 0, (size_t)plan.passes * digits * 4, stream));
    KeySource source{nullptr, nullptr, id, padding, vocab};
    for (int pass = 0; pass < plan.passes; pass++) {
        const int shift = pass * plan.digit_bits;
        const auto run = [&](auto* histogram, auto* scatter) -> int {
            const size_t shared = scatter_shared_bytes(digits);
            if (shared > DEFAULT_SHARED_BYTES)
                HDS_CHECK_CUDA(cudaFuncSetAttribute(scatter, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                    (int)scatter_shared_bytes(MAX_DIGITS)));
            histogram<<<tiles, SORT_THREADS, 0, stream>>>(n, source, shift, plan.digit_bits, tiles, counts,
                                                          totals + pass * digits);
            HDS_CHECK_LAUNCH("histogram_kernel");
            scan_kernel<<<(digits + SCAN_WARPS - 1) / SCAN_WARPS, 32 * SCAN_WARPS, 0, stream>>>(
                digits, tiles, totals + pass * digits, counts);
            HDS_CHECK_LAUNCH("scan_kernel");
            scatter<<<tiles, SORT_THREADS, shared, stream>>>(n, source, shift, plan.digit_bits, tiles, counts, keys,
                                                             rows);
            HDS_CHECK_LAUNCH("scatter_kernel");
            return HDS_OK;
        };
        if (int rc = plan.rounds == MANY_ROUNDS ? run(histogram_kernel<MANY_ROUNDS>, scatter_kernel<MANY_ROUNDS>)
                                                : run(histogram_kernel<SOME_ROUNDS>, scatter_kernel<SOME_ROUNDS>))
            return rc;
        source.keys = keys;
        source.rows = rows;
        std::swap(keys, keys_other);
        std::swap(rows, rows_other);
    }
    const uint32_t* sorted_keys = source.keys;
    const int32_t* sorted_rows = source.rows;

    const int slabs = (channels + plan.slab - 1) / plan.slab;
    const int64_t threads = plan.chunks << plan.lanes_log2;
    const dim3 sum_grid((unsigned)((threads + THREADS - 1) / THREADS), (unsigned)slabs);
    const dim3 join_grid((unsigned)((plan.chunks + JOIN_WORKERS - 1) / JOIN_WORKERS),
                         (unsigned)((channels + JOIN_COLUMNS - 1) / JOIN_COLUMNS));
    return with_variant([&](auto g, auto t, auto drop, auto add) -> int {
        using G = decltype(g);
        using T = decltype(t);
        if (int rc = with_vector(v, [&](auto width) -> int {
                chunk_sum_kernel<G, T, decltype(width)::value, decltype(drop)::value, decltype(add)::value>
                    <<<sum_grid, THREADS, 0, stream>>>(n, (uint32_t)vocab, channels, plan.slab, plan.lanes_log2,
                                                       plan.chunk, sorted_keys, sorted_rows,
                                                       static_cast<const G*>(grad), factor,
                                                       below_last(drop_threshold), d, static_cast<T*>(grad_table), heads, tails, plan.stride);
                HDS_CHECK_LAUNCH("chunk_sum_kernel");
                return HDS_OK;
            }))
            return rc;
        if (plan.chunks == 1) return HDS_OK;
        const auto join = [&](auto* kernel) -> int {
            kernel<<<join_grid, THREADS, 0, stream>>>(n, (uint32_t)vocab, channels, plan.chunk, sorted_keys, heads,
                                                      tails, plan.stride, factor, static_cast<T*>(grad_table));
            HDS_CHECK_LAUNCH("join_kernel");
            return HDS_OK;
        };
        if (v == COLUMNS) return join(join_kernel<T, COLUMNS, decltype(add)::value>);
        return join(join_kernel<T, 1, decltype(add)::value>);
    });
}
