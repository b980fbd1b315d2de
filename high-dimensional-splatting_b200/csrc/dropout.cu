// dropout.cu -- dropout from a counter-based generator: y = kept ? x * f : 0 with f the reciprocal of the
// kept share, the mask drawn anew from (seed, offset) by every call that needs it (philox.cuh).  The
// gradient is the same map of the output's gradient under the same draw, so one kernel serves both
// directions and no mask is stored.  A dropped element is 0 whatever x holds (NaN and infinity too).
//
// Bound by the memory in fp32: a 979 x 546 x 128 image and its gradient take 168 us, 1.09 GB at the measured
// copy rate.  In 16 bits integer work comes level with it (the image in bf16: 46 us a direction, 274 MB at 0.91
// of the copy rate with 74% of the issue slots), and for whole rows it is the bound (bf16 1000003 x 75: 53 us,
// 225 MB, 80% of the issue slots).
#include "elements.cuh"
#include "philox.cuh"

namespace hds {
namespace {

// A warp takes tiles of 256 consecutive elements in vectors of V (8 unless a buffer is aligned to less;
// rows need not be whole vectors).
//
// Elements: lane j draws the eight decisions of group j of the tile, one generator call for eight elements
// whatever V is, and the lane that holds an element fetches its group's decisions with a shuffle; with
// 8-element vectors that is the lane itself.
//
// Whole rows: lane j draws for the rows 8 (r0 / 8 + j) .. + 7 from the tile's first row r0 on.  Of rows at
// least 8 wide a warp's four tiles meet 130 at most, 18 such groups, so one generator call serves them all;
// narrower rows take one for each tile.  Of rows at least V wide a vector meets two at most.  A vector
// all of whose rows are dropped is not read.
constexpr int DROPOUT_THREADS = 256;
constexpr int TILE_ELEMENTS = 256;  // per warp
constexpr int TILES = 4;            // tiles in flight per warp
constexpr int BLOCK_ELEMENTS = DROPOUT_THREADS / 32 * TILE_ELEMENTS * TILES;
constexpr int BLOCK_GROUPS = BLOCK_ELEMENTS / 8;

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_up_to(const T* x, int64_t e, int64_t n) {
    if (e + V <= n) return load_once<T, V>(x + e);
    float v[V];
#pragma unroll
    for (int j = 0; j < V; j++) v[j] = e + j < n ? to_float(x[e + j]) : 0.0f;
    return Vec<T, V>::pack(v);
}

template <typename T, int V>
__device__ __forceinline__ void store_up_to(T* y, int64_t e, int64_t n, const Vec<T, V>& v) {
    if (e + V <= n)
        store<T, V>(y + e, v);
    else
        for (int j = 0; j < V; j++)
            if (e + j < n) y[e + j] = from_float<T>(v.get(j));
}

template <typename T, int V>
__global__ void __launch_bounds__(DROPOUT_THREADS) dropout_kernel(int64_t n, const T* x, float factor, uint32_t last,
                                                                  Draw draw, T* y) {
    constexpr int STEPS = 8 / V;
    draw = resolve(draw);
    const int lane = threadIdx.x & 31;
    const int in_block = (threadIdx.x >> 5) * (TILE_ELEMENTS * TILES);
    const int64_t warp_base = (int64_t)blockIdx.x * BLOCK_ELEMENTS + in_block;
    // A block's groups share the upper counter word: its first is a multiple of their number.
    const uint64_t group0 = (uint64_t)blockIdx.x * BLOCK_GROUPS;
    Vec<T, V> v[TILES][STEPS];
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int k = 0; k < STEPS; k++)
            v[t][k] = load_up_to<T, V>(x, warp_base + t * TILE_ELEMENTS + (k * 32 + lane) * V, n);
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        const Numbers8 numbers = philox4x32_10((uint32_t)group0 + (in_block + t * TILE_ELEMENTS) / 8 + lane,
                                               (uint32_t)(group0 >> 32), draw);
        const uint32_t bits = V == 8 ? 0 : numbers.bits(last);
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            const int at = (k * 32 + lane) * V;
            const uint32_t mine = V == 8 ? 0 : __shfl_sync(FULL_MASK, bits, at >> 3) >> (at & 7);
            float r[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                const bool kept = V == 8 ? numbers.kept(j, last) : ((mine >> j) & 1u) != 0;
                r[j] = kept ? v[t][k].get(j) * factor : 0.0f;
            }
            store_up_to<T, V>(y, warp_base + t * TILE_ELEMENTS + at, n, Vec<T, V>::pack(r));
        }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(DROPOUT_THREADS) dropout_rows_kernel(int64_t n, int64_t row_width, Divider rows_of,
                                                                       const T* x, float factor, uint32_t last,
                                                                       Draw draw, T* y) {
    constexpr int STEPS = 8 / V;
    draw = resolve(draw);
    const int lane = threadIdx.x & 31;
    const int64_t warp_base =
        (int64_t)blockIdx.x * BLOCK_ELEMENTS + (threadIdx.x >> 5) * (TILE_ELEMENTS * TILES);
    const int64_t row0 = warp_base / row_width;          // the warp's first element's row,
    const int64_t place = warp_base - row0 * row_width;  // and its place in it
    // Rows from row0 to the row of an element `at` elements from the warp's first.
    const auto rows_on = [&](uint32_t at) -> uint32_t {
        if (rows_of.d != 0) return rows_of.quotient((uint32_t)place + at);
        return place + at >= row_width ? 1 : 0;
    };
    Vec<T, V> v[TILES][STEPS];
    uint32_t keep[TILES][STEPS];
    uint32_t bits = 0;
    int first = 0;  // of row0 among the decisions in bits
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        if (t == 0 || row_width < 8) {
            const int64_t group0 = (row0 + rows_on(t * TILE_ELEMENTS)) >> 3;
            const uint64_t group = (uint64_t)(group0 + lane);
            bits = philox4x32_10((uint32_t)group, (uint32_t)(group >> 32), draw).bits(last);
            first = (int)(row0 - 8 * group0);
        }
        const auto row_kept = [&](uint32_t on) -> uint32_t {  // the row `on` rows from row0
            const int bit = first + (int)on;
            return (__shfl_sync(FULL_MASK, bits, bit >> 3) >> (bit & 7)) & 1u;
        };
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            const uint32_t at = t * TILE_ELEMENTS + (k * 32 + lane) * V;
            uint32_t mine = 0;
            if (V > 1 && row_width < V) {
#pragma unroll
                for (int j = 0; j < V; j++) mine |= row_kept(rows_on(at + j)) << j;
            } else {
                const uint32_t on = rows_on(at), on_end = rows_on(at + V - 1);
                const uint32_t a = row_kept(on), b = row_kept(on_end);
                // The elements of the vector in its first row: all, or as many as lie before the next one.
                uint32_t low = (1u << V) - 1u;
                if (on_end != on) low = (1u << (int)((int64_t)on_end * row_width - place - at)) - 1u;
                mine = (a ? low : 0u) | (b ? ((1u << V) - 1u) & ~low : 0u);
            }
            keep[t][k] = mine;
            if (mine != 0) v[t][k] = load_up_to<T, V>(x, warp_base + at, n);
        }
    }
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            float r[V];
#pragma unroll
            for (int j = 0; j < V; j++) r[j] = (keep[t][k] >> j) & 1u ? v[t][k].get(j) * factor : 0.0f;
            store_up_to<T, V>(y, warp_base + t * TILE_ELEMENTS + (k * 32 + lane) * V, n, Vec<T, V>::pack(r));
        }
}

}  // namespace
}  // namespace hds

using namespace hds;

extern "C" int hds_dropout(int64_t rows, int64_t channels, int type, const void* x, int drop_threshold, int whole_rows,
                           uint64_t seed, uint64_t offset, const int64_t* draw, void* y, hds_stream_t stream) {
    clear_error();
    HDS_REQUIRE(rows >= 0 && channels >= 0, HDS_ERR_INVALID, "dropout: negative size [%lld, %lld]", (long long)rows,
                (long long)channels);
    HDS_REQUIRE(known_type(type), HDS_ERR_UNSUPPORTED, "dropout: unknown element type %d", type);
    HDS_REQUIRE(drop_threshold >= 0 && drop_threshold <= DROP_ONE, HDS_ERR_INVALID,
                "dropout: threshold %d outside 0 to 65536", drop_threshold);
    if (rows == 0 || channels == 0) return HDS_OK;
    HDS_REQUIRE(rows <= INT64_MAX / 64 / channels, HDS_ERR_TOO_LARGE, "dropout: [%lld, %lld] is too large",
                (long long)rows, (long long)channels);
    HDS_REQUIRE(x != nullptr && y != nullptr, HDS_ERR_INVALID, "dropout: null pointer");
    HDS_REQUIRE((((uintptr_t)x | (uintptr_t)y) & (element_size(type) - 1)) == 0 && ((uintptr_t)draw & 7) == 0,
                HDS_ERR_INVALID, "dropout: misaligned buffer");
    const int64_t n = rows * channels;
    if (drop_threshold == 0) {
        if (x != y)
            HDS_CHECK_CUDA(cudaMemcpyAsync(y, x, (size_t)n * element_size(type), cudaMemcpyDeviceToDevice, stream));
        return HDS_OK;
    }
    const float factor = keep_factor(1.0, drop_threshold);
    const Draw d{seed, offset, draw};
    const int v = widest_vector(8, {{x, type}, {y, type}});
    const int64_t blocks = (n + BLOCK_ELEMENTS - 1) / BLOCK_ELEMENTS;
    HDS_REQUIRE(blocks <= INT32_MAX, HDS_ERR_TOO_LARGE, "dropout: [%lld, %lld] is too large", (long long)rows,
                (long long)channels);
    const uint32_t last = below_last(drop_threshold);
    // d = 0: rows of 2^15 elements and more, found by comparing (a warp's 1024 elements meet two at most).
    const Divider rows_of = channels < (1 << 15) ? divider((uint32_t)channels) : Divider{0, 0};
    return with_type(type, [&](auto t) -> int {
        using T = decltype(t);
        const T* from = static_cast<const T*>(x);
        T* to = static_cast<T*>(y);
        return with_vector(v, [&](auto width) -> int {
            constexpr int V = decltype(width)::value;
            if (whole_rows && channels > 1)  // a row of one element is an element
                dropout_rows_kernel<T, V><<<(unsigned)blocks, DROPOUT_THREADS, 0, stream>>>(n, channels, rows_of, from,
                                                                                           factor, last, d, to);
            else
                dropout_kernel<T, V><<<(unsigned)blocks, DROPOUT_THREADS, 0, stream>>>(n, from, factor, last, d, to);
            HDS_CHECK_LAUNCH("dropout_kernel");
            return HDS_OK;
        });
    });
}
