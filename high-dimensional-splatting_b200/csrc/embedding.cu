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
};

template <typename T, typename O, int V, bool DROP>
__global__ void __launch_bounds__(THREADS) lookup_kernel(int64_t total, int64_t vocab, int channels, Divider rows_of,
                                                         const T* __restrict__ table, Ids ids, Padding padding,
                                                         float factor, uint32_t threshold, Draw draw,
                                                         O* __restrict__ out) {
    constexpr int STEPS = 8 / V;
    if (DROP) draw = resolve(draw);
    const int lane = threadIdx.x & 31;
    const int64_t warp_base = (int64_t)blockIdx.x * LOOKUP_ELEMENTS + (threadIdx.x >> 5) * (TILE_ELEMENTS * TILES);
    if (warp_base >= total) return;
    const int64_t row0 = warp_base / channels;
    const uint32_t place = (uint32_t)(warp_base - row0 * channels);
    int64_t at[TILES][STEPS];  // the vector's first element in the table, or -1
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            const uint32_t e = t * TILE_ELEMENTS + (k * 32 + lane) * V;
            at[t][k] = -1;
            if (warp_base + e < total) {
                const uint32_t q = rows_of.quotient(place + e);
                const int64_t row = table_row(ids[row0 + q], vocab, padding);
                if (row >= 0) at[t][k] = row * channels + (place + e - q * channels);
            }
        }
    Vec<T, V> v[TILES][STEPS];
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int k = 0; k < STEPS; k++)
            if (at[t][k] >= 0) v[t][k] = load_shared_data<T, V>(table + at[t][k]);
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        const int64_t tile = warp_base + t * TILE_ELEMENTS;
        const uint32_t bits = DROP ? keep8((uint64_t)(tile >> 3) + lane, draw, threshold) : 0xffu;
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            const int e = (k * 32 + lane) * V;
            uint32_t keep = bits;
            if (DROP && V < 8) keep = __shfl_sync(FULL_MASK, bits, e >> 3) >> (e & 7);
            if (at[t][k] < 0) keep = 0;
            Vec<O, V> r;
#pragma unroll
            for (int j = 0; j < V; j++) r.set(j, (keep >> j) & 1u ? v[t][k].get(j) * factor : 0.0f);
            if (tile + e < total) store<O, V>(out + tile + e, r);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// stable radix sort of (codeword, row number)
// ---------------------------------------------------------------------------------------------
// Digits of up to 11 bits: one pass for codebooks below 2048 rows, two below 4M.  A pass is a histogram
// per tile, a scan that turns the digit-major counts into output positions, and a scatter that ranks the
// tile's keys.  The first pass reads the ids themselves.  No block waits for another.
constexpr int SORT_THREADS = 512;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_ROUNDS = 16;                               // keys per thread
constexpr int SORT_TILE = SORT_THREADS * SORT_ROUNDS;         // 8192
constexpr int MAX_DIGIT_BITS = 11;
constexpr int MAX_DIGITS = 1 << MAX_DIGIT_BITS;

struct KeySource {
    const uint32_t* keys;  // sorted so far, or NULL in the first pass:
    const int32_t* rows;
    Ids ids;
    Padding padding;
    int64_t vocab;
    __device__ __forceinline__ uint32_t key(int64_t i) const {
        if (keys != nullptr) return keys[i];
        const int64_t row = table_row(ids[i], vocab, padding);
        return (uint32_t)(row < 0 ? vocab : row);
    }
    __device__ __forceinline__ int32_t row(int64_t i) const { return rows != nullptr ? rows[i] : (int32_t)i; }
};

// counts[digit][tile] and totals[digit] (cleared by the caller; integer adds, so their order is no matter).
__global__ void __launch_bounds__(SORT_THREADS) histogram_kernel(int64_t n, KeySource source, int shift, int digits,
                                                                 int tiles, uint32_t* __restrict__ counts,
                                                                 uint32_t* __restrict__ totals) {
    __shared__ uint32_t hist[MAX_DIGITS];
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) hist[d] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_TILE;
    const int lane = threadIdx.x & 31;
#pragma unroll 4
    for (int r = 0; r < SORT_ROUNDS; r++) {
        const int64_t i = base + r * SORT_THREADS + threadIdx.x;
        const uint32_t d = i < n ? (source.key(i) >> shift) & (digits - 1) : MAX_DIGITS;
        // One shared atomic per distinct digit of the warp: popular codewords would serialise otherwise.
        const uint32_t peers = __match_any_sync(FULL_MASK, d);
        if (d < MAX_DIGITS && lane == __ffs(peers) - 1) atomicAdd(&hist[d], __popc(peers));
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
    for (int d = lane; d < digit; d += 32) base += totals[d];
    base = __reduce_add_sync(FULL_MASK, base);
    uint32_t* row = counts + (int64_t)digit * tiles;
    for (int t0 = 0; t0 < tiles; t0 += 32) {
        const int t = t0 + lane;
        const uint32_t v = t < tiles ? row[t] : 0;
        uint32_t x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(FULL_MASK, x, o);
            if (lane >= o) x += y;
        }
        if (t < tiles) row[t] = base + x - v;
        base += __shfl_sync(FULL_MASK, x, 31);
    }
}

// Each warp ranks its own 512 consecutive keys with __match_any_sync into a count table of its own; a
// scan over the warps then places the tables one after another.
inline size_t scatter_shared_bytes(int digits) { return (size_t)digits * (sizeof(uint32_t) + 2 * SORT_WARPS); }

__global__ void __launch_bounds__(SORT_THREADS) scatter_kernel(int64_t n, KeySource source, int shift, int digits,
                                                               int tiles, const uint32_t* __restrict__ positions,
                                                               uint32_t* __restrict__ keys_out,
                                                               int32_t* __restrict__ rows_out) {
    extern __shared__ uint32_t s_base[];                                  // [digits]
    uint16_t* s_warp = reinterpret_cast<uint16_t*>(s_base + digits);      // [warps][digits]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int d = threadIdx.x; d < digits; d += SORT_THREADS) s_base[d] = positions[(int64_t)d * tiles + blockIdx.x];
    for (int d = threadIdx.x; d < digits * SORT_WARPS / 2; d += SORT_THREADS) reinterpret_cast<uint32_t*>(s_warp)[d] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * SORT_TILE + warp * (32 * SORT_ROUNDS) + lane;
    uint16_t* mine = s_warp + warp * digits;
    uint32_t key[SORT_ROUNDS];
    uint16_t rank[SORT_ROUNDS];
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; r++) key[r] = base + 32 * r < n ? source.key(base + 32 * r) : 0;
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; r++) {
        const bool valid = base + 32 * r < n;
        const uint32_t d = valid ? (key[r] >> shift) & (digits - 1) : MAX_DIGITS;
        const uint32_t peers = __match_any_sync(FULL_MASK, d);
        const uint32_t before = valid ? mine[d] : 0;
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
    for (int r = 0; r < SORT_ROUNDS; r++) {
        const int64_t i = base + 32 * r;
        if (i >= n) break;
        const uint32_t d = (key[r] >> shift) & (digits - 1);
        const uint32_t pos = s_base[d] + mine[d] + rank[r];
        keys_out[pos] = key[r];
        rows_out[pos] = source.row(i);
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
                                                            uint32_t threshold, Draw draw, T* __restrict__ table,
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
        uint32_t keep[ROWS_AHEAD][STEPS];
        if (DROP) {
#pragma unroll
            for (int u = 0; u < ROWS_AHEAD; u++) {
                const int64_t e = (int64_t)(key[u] != vocab ? row[u] : 0) * channels + c0;
                const uint32_t bits = keep8((uint64_t)(e >> 3) + lane, draw, threshold);
                if (V == COLUMNS) {
                    keep[u][0] = bits;
                } else {
                    // The row may start inside a group: its last columns then belong to one group more.
                    const int into = (int)(e & 7);
                    const uint32_t more =
                        into + width > 8 * lanes ? keep8((uint64_t)(e >> 3) + lanes, draw, threshold) : 0;
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
                    if (!DROP || ((keep[u][k] >> j) & 1u)) sum[k * V + j] += g[u][k].get(j);
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
// that codeword's sum, its tail plus the heads of the following chunks.  Few heads: the worker adds
// them.  Many (a popular codeword): the whole block does, in 64 interleaved runs and a tree.
constexpr int JOIN_LANES = 4;
constexpr int JOIN_WORKERS = THREADS / JOIN_LANES;
constexpr int JOIN_COLUMNS = JOIN_LANES * COLUMNS;
constexpr int FEW_HEADS = 8;

template <typename T, int V, bool ACCUMULATE>
__global__ void __launch_bounds__(THREADS) join_kernel(int64_t n, uint32_t vocab, int channels, int chunk,
                                                       const uint32_t* __restrict__ keys,
                                                       const float* __restrict__ heads,
                                                       const float* __restrict__ tails, int stride, float factor,
                                                       T* __restrict__ table) {
    __shared__ int s_long;
    __shared__ int64_t s_id[JOIN_WORKERS];
    __shared__ int64_t s_last[JOIN_WORKERS];
    __shared__ float s_sum[JOIN_WORKERS][JOIN_COLUMNS];
    const int worker = threadIdx.x / JOIN_LANES, lane = threadIdx.x % JOIN_LANES;
    const int c = blockIdx.y * JOIN_COLUMNS + lane * COLUMNS;
    const bool there = c < channels;
    const int64_t chunks = (n + chunk - 1) / chunk;
    const int64_t id = (int64_t)blockIdx.x * JOIN_WORKERS + worker;
    if (threadIdx.x == 0) s_long = 0;
    __syncthreads();

    const auto add = [&](float* sum, const float* partial, int64_t at) {
        const Vec<float, COLUMNS> v = load_shared_data<float, COLUMNS>(partial + at * stride + c);
#pragma unroll
        for (int j = 0; j < COLUMNS; j++) sum[j] += v.get(j);
    };
    const auto write = [&](uint32_t codeword, const float* sum) {
#pragma unroll
        for (int j = 0; j < COLUMNS; j += V)
            if (c + j < channels)
                store_sum<T, V, ACCUMULATE>(table + (int64_t)codeword * channels + c + j, sum + j, factor);
    };

    const int64_t start = id * chunk, end = start + chunk;
    bool owner = end < n;
    uint32_t codeword = vocab;
    if (owner) {
        codeword = keys[end];
        owner = codeword != vocab && keys[end - 1] == codeword &&
                (keys[start] != codeword || start == 0 || keys[start - 1] != codeword);
    }
    if (owner) {
        // The last chunk that begins with the codeword: doubling steps, then halving ones.
        int64_t last = id + 1, beyond = id + 2;
        for (int64_t step = 1; beyond < chunks && keys[beyond * chunk] == codeword; step *= 2) {
            last = beyond;
            beyond = min(chunks, last + 2 * step);
        }
        while (beyond - last > 1) {
            const int64_t middle = last + (beyond - last) / 2;
            if (middle < chunks && keys[middle * chunk] == codeword) last = middle; else beyond = middle;
        }
        if (last - id <= FEW_HEADS) {
            if (there) {
                float sum[COLUMNS] = {};
                add(sum, tails, id);
                for (int64_t j = id + 1; j <= last; j++) add(sum, heads, j);
                write(codeword, sum);
            }
        } else if (lane == 0) {
            const int slot = atomicAdd(&s_long, 1);
            s_id[slot] = id;
            s_last[slot] = last;
        }
    }
    __syncthreads();
    for (int slot = 0; slot < s_long; slot++) {
        const int64_t from = s_id[slot], last = s_last[slot];
        float sum[COLUMNS] = {};
        if (there) {
            if (worker == 0) add(sum, tails, from);
#pragma unroll 4
            for (int64_t j = from + 1 + worker; j <= last; j += JOIN_WORKERS) add(sum, heads, j);
        }
#pragma unroll
        for (int j = 0; j < COLUMNS; j++) s_sum[worker][lane * COLUMNS + j] = sum[j];
        __syncthreads();
        for (int half = JOIN_WORKERS / 2; half > 0; half /= 2) {
            for (int i = threadIdx.x; i < half * JOIN_COLUMNS; i += THREADS)
                s_sum[i / JOIN_COLUMNS][i % JOIN_COLUMNS] += s_sum[i / JOIN_COLUMNS + half][i % JOIN_COLUMNS];
            __syncthreads();
        }
        if (worker == 0 && there) write(keys[(from + 1) * chunk], s_sum[0] + lane * COLUMNS);
        __syncthreads();
    }
}

int ceil_log2(int64_t x) {
    int bits = 0;
    while ((int64_t(1) << bits) < x) bits++;
    return bits;
}

// How the backward splits its work and lays out its scratch.
struct BackwardPlan {
    int64_t tiles;            // of the sort
    int passes, digit_bits;
    int chunk, stride;        // rows per chunk; floats per partial row
    int64_t chunks;
    int slab, lanes_log2;     // columns and lanes of a worker
    size_t keys_a, keys_b, rows_a, rows_b, counts, totals, heads, tails, bytes;

    BackwardPlan(int64_t n, int64_t vocab, int channels) {
        const size_t nn = (size_t)std::max<int64_t>(n, 1);
        tiles = ((int64_t)nn + SORT_TILE - 1) / SORT_TILE;
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
                    (uint32_t)drop_threshold, d, static_cast<O*>(out));
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
    return BackwardPlan(n, vocab, channels).bytes;
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
        HDS_REQUIRE(scratch != nullptr && scratch_bytes >= plan.bytes && !misaligned(scratch, 256), HDS_ERR_SCRATCH,
                    "embedding_backward: scratch needs %zu bytes, 256-byte aligned", plan.bytes);
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
    HDS_CHECK_CUDA(cudaFuncSetAttribute(scatter_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)scatter_shared_bytes(MAX_DIGITS)));
    KeySource source{nullptr, nullptr, Ids{ids, ids_type == HDS_TYPE_I64}, Padding{has_padding, padding_id}, vocab};
    for (int pass = 0; pass < plan.passes; pass++) {
        const int shift = pass * plan.digit_bits;
        histogram_kernel<<<tiles, SORT_THREADS, 0, stream>>>(n, source, shift, digits, tiles, counts,
                                                             totals + pass * digits);
        HDS_CHECK_LAUNCH("histogram_kernel");
        scan_kernel<<<(digits + SCAN_WARPS - 1) / SCAN_WARPS, 32 * SCAN_WARPS, 0, stream>>>(
            digits, tiles, totals + pass * digits, counts);
        HDS_CHECK_LAUNCH("scan_kernel");
        scatter_kernel<<<tiles, SORT_THREADS, scatter_shared_bytes(digits), stream>>>(n, source, shift, digits, tiles,
                                                                                      counts, keys, rows);
        HDS_CHECK_LAUNCH("scatter_kernel");
        source.keys = keys;
        source.rows = rows;
        std::swap(keys, keys_other);
        std::swap(rows, rows_other);
    }
    const uint32_t* sorted_keys = source.keys;
    const int32_t* sorted_rows = source.rows;

    const Draw d{seed, offset, draw};
    const float factor = keep_factor(scale, drop_threshold);
    const int slabs = (channels + plan.slab - 1) / plan.slab;
    const int64_t threads = plan.chunks << plan.lanes_log2;
    const dim3 sum_grid((unsigned)((threads + THREADS - 1) / THREADS), (unsigned)slabs);
    const dim3 join_grid((unsigned)((plan.chunks + JOIN_WORKERS - 1) / JOIN_WORKERS),
                         (unsigned)((channels + JOIN_COLUMNS - 1) / JOIN_COLUMNS));
    const int v = widest_vector(channels, {{grad, grad_type}, {grad_table, table_type}});
    return with_types(table_type, grad_type, [&](auto t, auto g) -> int {
        using T = decltype(t);
        using G = decltype(g);
        return with_vector(v, [&](auto w) -> int {
            constexpr int V = decltype(w)::value;
            const auto run = [&](auto drop, auto add) -> int {
                chunk_sum_kernel<G, T, V, decltype(drop)::value, decltype(add)::value>
                    <<<sum_grid, THREADS, 0, stream>>>(n, (uint32_t)vocab, channels, plan.slab, plan.lanes_log2,
                                                       plan.chunk, sorted_keys, sorted_rows,
                                                       static_cast<const G*>(grad), factor, (uint32_t)drop_threshold,
                                                       d, static_cast<T*>(grad_table), heads, tails, plan.stride);
                HDS_CHECK_LAUNCH("chunk_sum_kernel");
                if (plan.chunks > 1) {
                    join_kernel<T, V, decltype(add)::value><<<join_grid, THREADS, 0, stream>>>(
                        n, (uint32_t)vocab, channels, plan.chunk, sorted_keys, heads, tails, plan.stride, factor,
                        static_cast<T*>(grad_table));
                    HDS_CHECK_LAUNCH("join_kernel");
                }
                return HDS_OK;
            };
            if constexpr (std::is_same<T, float>::value) {
                if (accumulate)
                    return drop_threshold > 0 ? run(std::true_type{}, std::true_type{})
                                              : run(std::false_type{}, std::true_type{});
            }
            return drop_threshold > 0 ? run(std::true_type{}, std::false_type{})
                                      : run(std::false_type{}, std::false_type{});
        });
    });
}
