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
// stable radix sort of (codeword, row number), 8 bits a pass
// ---------------------------------------------------------------------------------------------
constexpr int RADIX = 256;
constexpr int SORT_TILE = 4096;  // keys per block and pass

template <typename I>
__global__ void __launch_bounds__(THREADS) keys_kernel(int64_t n, int64_t vocab, const I* __restrict__ ids,
                                                       Padding padding, uint32_t* __restrict__ keys,
                                                       int32_t* __restrict__ rows) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int64_t row = table_row(ids[i], vocab, padding);
    keys[i] = (uint32_t)(row < 0 ? vocab : row);
    rows[i] = (int32_t)i;
}

__global__ void __launch_bounds__(THREADS) histogram_kernel(int64_t n, const uint32_t* __restrict__ keys, int shift,
                                                            int blocks, uint32_t* __restrict__ counts) {
    __shared__ uint32_t hist[RADIX];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const int64_t begin = (int64_t)blockIdx.x * SORT_TILE, end = min(n, begin + SORT_TILE);
    for (int64_t i = begin + threadIdx.x; i < end; i += THREADS) atomicAdd(&hist[(keys[i] >> shift) & (RADIX - 1)], 1u);
    __syncthreads();
    counts[(int64_t)threadIdx.x * blocks + blockIdx.x] = hist[threadIdx.x];
}

// Exclusive scan of the digit-major count table by one block.
__global__ void __launch_bounds__(1024) scan_kernel(int64_t items, uint32_t* __restrict__ counts) {
    __shared__ uint32_t warp_sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t carry = 0;
    for (int64_t base = 0; base < items; base += 1024) {
        const int64_t i = base + threadIdx.x;
        const uint32_t v = i < items ? counts[i] : 0;
        uint32_t x = v;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(FULL_MASK, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_sums[warp] = x;
        __syncthreads();
        if (warp == 0) {
            uint32_t w = warp_sums[lane];
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(FULL_MASK, w, o);
                if (lane >= o) w += y;
            }
            warp_sums[lane] = w;
        }
        __syncthreads();
        if (i < items) counts[i] = carry + (warp > 0 ? warp_sums[warp - 1] : 0) + x - v;
        carry += warp_sums[31];
        __syncthreads();
    }
}

__global__ void __launch_bounds__(THREADS) scatter_kernel(int64_t n, const uint32_t* __restrict__ keys_in,
                                                          const int32_t* __restrict__ rows_in, int shift, int blocks,
                                                          const uint32_t* __restrict__ offsets,
                                                          uint32_t* __restrict__ keys_out,
                                                          int32_t* __restrict__ rows_out) {
    constexpr int WARPS = THREADS / 32;
    __shared__ uint32_t s_base[RADIX];
    __shared__ uint32_t s_warp[WARPS][RADIX];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t begin = (int64_t)blockIdx.x * SORT_TILE, end = min(n, begin + SORT_TILE);
    s_base[tid] = offsets[(int64_t)tid * blocks + blockIdx.x];
    for (int64_t base = begin; base < end; base += THREADS) {
        for (int w = 0; w < WARPS; w++) s_warp[w][tid] = 0;
        __syncthreads();
        const int64_t i = base + tid;
        const bool valid = i < end;
        const uint32_t key = valid ? keys_in[i] : 0;
        const uint32_t d = valid ? (key >> shift) & (RADIX - 1) : RADIX;
        const uint32_t peers = __match_any_sync(FULL_MASK, d);
        const uint32_t rank = __popc(peers & ((1u << lane) - 1u));
        if (valid && rank == 0) s_warp[warp][d] = __popc(peers);
        __syncthreads();
        uint32_t run = s_base[tid];
        for (int w = 0; w < WARPS; w++) {
            const uint32_t c = s_warp[w][tid];
            s_warp[w][tid] = run;
            run += c;
        }
        s_base[tid] = run;
        __syncthreads();
        if (valid) {
            const uint32_t pos = s_warp[warp][d] + rank;
            keys_out[pos] = key;
            rows_out[pos] = rows_in[i];
        }
        __syncthreads();
    }
}

// First position of the sorted keys with keys[p] >= v.
__device__ __forceinline__ int64_t lower_bound(const uint32_t* keys, int64_t n, uint32_t v) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < v) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// One block per codeword: its rows' columns summed in row order.
template <typename G, typename T, bool ACCUMULATE>
__global__ void __launch_bounds__(THREADS) segment_sum_kernel(int64_t n, int channels,
                                                              const uint32_t* __restrict__ keys,
                                                              const int32_t* __restrict__ rows,
                                                              const G* __restrict__ grad, float factor,
                                                              uint32_t threshold, Draw draw, T* __restrict__ table) {
    draw = resolve(draw);
    const uint32_t v = blockIdx.x;
    const int64_t begin = lower_bound(keys, n, v), end = lower_bound(keys, n, v + 1);
    for (int c = threadIdx.x; c < channels; c += THREADS) {
        float sum = 0.0f;
        for (int64_t k = begin; k < end; k++) {
            const int64_t e = (int64_t)rows[k] * channels + c;
            if (threshold == 0 || keep_one((uint64_t)e, draw, threshold)) sum += to_float(grad[e]);
        }
        const int64_t at = (int64_t)v * channels + c;
        if (ACCUMULATE) {
            if (begin < end) table[at] = from_float<T>(fmaf(factor, sum, to_float(table[at])));
        } else {
            table[at] = from_float<T>(factor * sum);
        }
    }
}

int sort_blocks(int64_t n) { return (int)((n + SORT_TILE - 1) / SORT_TILE); }

struct BackwardLayout {
    size_t keys_a, keys_b, rows_a, rows_b, counts, bytes;
    explicit BackwardLayout(int64_t n) {
        const size_t nn = (size_t)std::max<int64_t>(n, 1);
        keys_a = 0;
        keys_b = keys_a + align256(nn * 4);
        rows_a = keys_b + align256(nn * 4);
        rows_b = rows_a + align256(nn * 4);
        counts = rows_b + align256(nn * 4);
        bytes = counts + align256((size_t)RADIX * (size_t)sort_blocks((int64_t)nn) * 4);
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
    (void)vocab;
    (void)channels;
    return BackwardLayout(n).bytes;
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
    if (n == 0) {
        if (!accumulate)
            HDS_CHECK_CUDA(cudaMemsetAsync(grad_table, 0, (size_t)vocab * channels * element_size(table_type), stream));
        return HDS_OK;
    }
    HDS_REQUIRE(grad != nullptr && ids != nullptr, HDS_ERR_INVALID, "embedding_backward: null pointer");
    HDS_REQUIRE(!misaligned(grad, element_size(grad_type)) && !misaligned(ids, ids_type == HDS_TYPE_I32 ? 4 : 8) &&
                    !misaligned(draw, 8),
                HDS_ERR_INVALID, "embedding_backward: misaligned buffer");
    const BackwardLayout L(n);
    HDS_REQUIRE(scratch != nullptr && scratch_bytes >= L.bytes && !misaligned(scratch, 256), HDS_ERR_SCRATCH,
                "embedding_backward: scratch needs %zu bytes, 256-byte aligned", L.bytes);
    char* s = static_cast<char*>(scratch);
    auto* keys = reinterpret_cast<uint32_t*>(s + L.keys_a);
    auto* keys_other = reinterpret_cast<uint32_t*>(s + L.keys_b);
    auto* rows = reinterpret_cast<int32_t*>(s + L.rows_a);
    auto* rows_other = reinterpret_cast<int32_t*>(s + L.rows_b);
    auto* counts = reinterpret_cast<uint32_t*>(s + L.counts);
    const Padding padding{has_padding, padding_id};
    const Draw d{seed, offset, draw};
    const float factor = keep_factor(scale, drop_threshold);
    const unsigned blocks = (unsigned)((n + THREADS - 1) / THREADS);
    if (ids_type == HDS_TYPE_I32)
        keys_kernel<int32_t><<<blocks, THREADS, 0, stream>>>(n, vocab, static_cast<const int32_t*>(ids), padding, keys,
                                                             rows);
    else
        keys_kernel<int64_t><<<blocks, THREADS, 0, stream>>>(n, vocab, static_cast<const int64_t*>(ids), padding, keys,
                                                             rows);
    HDS_CHECK_LAUNCH("keys_kernel");
    const int nblocks = sort_blocks(n);
    for (int shift = 0; shift < 32 && (vocab >> shift) != 0; shift += 8) {
        histogram_kernel<<<nblocks, THREADS, 0, stream>>>(n, keys, shift, nblocks, counts);
        HDS_CHECK_LAUNCH("histogram_kernel");
        scan_kernel<<<1, 1024, 0, stream>>>((int64_t)RADIX * nblocks, counts);
        HDS_CHECK_LAUNCH("scan_kernel");
        scatter_kernel<<<nblocks, THREADS, 0, stream>>>(n, keys, rows, shift, nblocks, counts, keys_other, rows_other);
        HDS_CHECK_LAUNCH("scatter_kernel");
        std::swap(keys, keys_other);
        std::swap(rows, rows_other);
    }
    return with_types(table_type, grad_type, [&](auto t, auto g) -> int {
        using T = decltype(t);
        using G = decltype(g);
        if (accumulate)
            segment_sum_kernel<G, T, true><<<(unsigned)vocab, THREADS, 0, stream>>>(
                n, channels, keys, rows, static_cast<const G*>(grad), factor, (uint32_t)drop_threshold, d,
                static_cast<T*>(grad_table));
        else
            segment_sum_kernel<G, T, false><<<(unsigned)vocab, THREADS, 0, stream>>>(
                n, channels, keys, rows, static_cast<const G*>(grad), factor, (uint32_t)drop_threshold, d,
                static_cast<T*>(grad_table));
        HDS_CHECK_LAUNCH("segment_sum_kernel");
        return HDS_OK;
    });
}
