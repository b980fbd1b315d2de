// dropout.cu -- dropout from a counter-based generator: y = kept ? x * f : 0 with f the reciprocal of the
// kept share, the mask drawn anew from (seed, offset) by every call that needs it (philox.cuh).  The
// gradient is the same map of the output's gradient under the same draw, so one kernel serves both
// directions and no mask is stored.  A dropped element is 0 whatever x holds (NaN and infinity too).
#include "elements.cuh"
#include "philox.cuh"

namespace hds {
namespace {

// A warp takes tiles of 256 consecutive elements: lane j draws the eight decisions of group j of the tile
// (one generator call for eight elements, whatever the vector width), and the lane that holds an
// element fetches its group's decisions with a shuffle.  With 8-element vectors that is the lane itself.
// Whole rows: lane j draws for the rows 8 (r0 / 8 + j) .. + 7 around the tile's first row r0; a tile
// of rows at least two wide spans at most 18 such groups.  A dropped row is not read.
constexpr int DROPOUT_THREADS = 256;
constexpr int TILE_ELEMENTS = 256;  // per warp
constexpr int TILES = 4;            // tiles in flight per warp
constexpr int BLOCK_ELEMENTS = DROPOUT_THREADS / 32 * TILE_ELEMENTS * TILES;

template <typename T, int V, bool ROWS>
__global__ void __launch_bounds__(DROPOUT_THREADS) dropout_kernel(int64_t n, int64_t row_width, Divider rows_of,
                                                                  const T* x, float factor, uint32_t threshold,
                                                                  Draw draw, T* y) {
    constexpr int STEPS = 8 / V;
    draw = resolve(draw);
    const int lane = threadIdx.x & 31;
    const int64_t warp_base =
        (int64_t)blockIdx.x * BLOCK_ELEMENTS + (threadIdx.x >> 5) * (TILE_ELEMENTS * TILES);
    const int64_t row0 = ROWS ? warp_base / row_width : 0;  // the warp's first element's row,
    const int64_t place = warp_base - row0 * row_width;     // and its place in it
    Vec<T, V> v[TILES][STEPS];
    uint32_t keep[TILES][STEPS];
    if (!ROWS) {
#pragma unroll
        for (int t = 0; t < TILES; t++)
#pragma unroll
            for (int k = 0; k < STEPS; k++) {
                const int64_t e = warp_base + t * TILE_ELEMENTS + (k * 32 + lane) * V;
                if (e + V <= n)
                    v[t][k] = load_once<T, V>(x + e);
                else
                    for (int j = 0; j < V; j++) v[t][k].set(j, e + j < n ? to_float(x[e + j]) : 0.0f);
            }
    }
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        const int64_t tile = warp_base + t * TILE_ELEMENTS;
        if (!ROWS) {
            const uint32_t bits = keep8((uint64_t)(tile >> 3) + lane, draw, threshold);
#pragma unroll
            for (int k = 0; k < STEPS; k++) {
                const int at = (k * 32 + lane) * V;
                keep[t][k] = V == 8 ? bits : __shfl_sync(FULL_MASK, bits, at >> 3) >> (at & 7);
            }
        } else {
            const auto row_of = [&](uint32_t at) -> int64_t {  // at: elements from the warp's first
                if (rows_of.d != 0) return row0 + rows_of.quotient((uint32_t)place + at);
                return row0 + (place + at >= row_width ? 1 : 0);
            };
            const int64_t group0 = row_of(t * TILE_ELEMENTS) >> 3;
            const uint32_t bits = keep8((uint64_t)(group0 + lane), draw, threshold);
#pragma unroll
            for (int k = 0; k < STEPS; k++) {
                const int at = t * TILE_ELEMENTS + (k * 32 + lane) * V;
                const int64_t row = row_of(at);
                const uint32_t mine = __shfl_sync(FULL_MASK, bits, (int)((row >> 3) - group0));
                keep[t][k] = (mine >> (row & 7)) & 1u ? 0xffu : 0u;
                if (keep[t][k] && warp_base + at < n) v[t][k] = load_once<T, V>(x + warp_base + at);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TILES; t++)
#pragma unroll
        for (int k = 0; k < STEPS; k++) {
            const int64_t e = warp_base + t * TILE_ELEMENTS + (k * 32 + lane) * V;
            Vec<T, V> r;
#pragma unroll
            for (int j = 0; j < V; j++) r.set(j, (keep[t][k] >> j) & 1u ? v[t][k].get(j) * factor : 0.0f);
            if (e + V <= n)
                store<T, V>(y + e, r);
            else
                for (int j = 0; j < V; j++)
                    if (e + j < n) y[e + j] = from_float<T>(r.get(j));
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
    const float factor = keep_factor(1.0, drop_threshold);
    const Draw d{seed, offset, draw};
    // Rows of one element are elements.  Element by element, vectors need not end with a row: only the
    // alignment bounds them, and the last n % V elements go one by one.
    const bool by_rows = whole_rows && channels > 1;
    const int v = widest_vector(by_rows ? channels : 8, {{x, type}, {y, type}});
    const int64_t blocks = (n + BLOCK_ELEMENTS - 1) / BLOCK_ELEMENTS;
    HDS_REQUIRE(blocks <= INT32_MAX, HDS_ERR_TOO_LARGE, "dropout: [%lld, %lld] is too large", (long long)rows,
                (long long)channels);
    // d = 0: rows of 2^15 elements and more, found by comparing (a warp's 1024 elements span two at most).
    const Divider rows_of = channels < (1 << 15) ? divider((uint32_t)channels) : Divider{0, 0};
    return with_type(type, [&](auto t) -> int {
        using T = decltype(t);
        return with_vector(v, [&](auto width) -> int {
            constexpr int V = decltype(width)::value;
            if (by_rows)
                dropout_kernel<T, V, true><<<(unsigned)blocks, DROPOUT_THREADS, 0, stream>>>(
                    n, channels, rows_of, static_cast<const T*>(x), factor, (uint32_t)drop_threshold, d,
                    static_cast<T*>(y));
            else
                dropout_kernel<T, V, false><<<(unsigned)blocks, DROPOUT_THREADS, 0, stream>>>(
                    n, 1, Divider{0, 0}, static_cast<const T*>(x), factor, (uint32_t)drop_threshold, d,
                    static_cast<T*>(y));
            HDS_CHECK_LAUNCH("dropout_kernel");
            return HDS_OK;
        });
    });
}
