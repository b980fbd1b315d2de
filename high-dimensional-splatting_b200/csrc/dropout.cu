// dropout.cu -- dropout from a counter-based generator: y = kept ? x * f : 0 with f the reciprocal of the
// kept share, the mask drawn anew from (seed, offset) by every call that needs it (philox.cuh).  The
// gradient is the same map of the output's gradient under the same draw, so one kernel serves both
// directions and no mask is stored.  A dropped element is 0 whatever x holds (NaN and infinity too).
#include <algorithm>

#include "elements.cuh"
#include "philox.cuh"

namespace hds {
namespace {

constexpr int DROPOUT_THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(DROPOUT_THREADS) dropout_kernel(int64_t n, int64_t row_width,
                                                                  const T* __restrict__ x, float factor,
                                                                  uint32_t threshold, Draw draw, T* __restrict__ y) {
    draw = resolve(draw);
    const int64_t stride = (int64_t)gridDim.x * blockDim.x;
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += stride) {
        const bool keep = keep_one((uint64_t)(e / row_width), draw, threshold);
        y[e] = keep ? from_float<T>(to_float(x[e]) * factor) : from_float<T>(0.0f);
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
    const int64_t blocks = std::min<int64_t>((n + DROPOUT_THREADS - 1) / DROPOUT_THREADS, 148 * 8);
    return with_type(type, [&](auto t) -> int {
        using T = decltype(t);
        dropout_kernel<T><<<(unsigned)blocks, DROPOUT_THREADS, 0, stream>>>(
            n, whole_rows ? channels : 1, static_cast<const T*>(x), factor, (uint32_t)drop_threshold, d,
            static_cast<T*>(y));
        HDS_CHECK_LAUNCH("dropout_kernel");
        return HDS_OK;
    });
}
