// Dropout: y = x * factor where the element is kept, else 0; its gradient is the same map of the gradient.  Bound by memory, with the generator's
// multiplications close behind (mi8_philox.h): a lane makes the bits of the eight elements it loads, and no mask is stored.
#include "mi8_elements.h"
#include "mi8_philox.h"

namespace mi8 {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const uint8_t* __restrict__ x, uint8_t* __restrict__ y, int64_t n, const Dropout d)
{
    const uint64_t key = d.seed_on_device ? (uint64_t)d.seed_on_device[0] : d.seed;
    const int64_t groups = (n + 7) / 8;
    for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < groups; g += (int64_t)gridDim.x * kThreads) {
        const int64_t at = g * 8 * Eight<T>::kBytes;
        const int left = n - g * 8 < 8 ? (int)(n - g * 8) : 8;
        Eight<T> raw;
        float v[8];
        raw.load(x + at, 0, left);
        const uint32_t m = kept8(g * 8, d.offset, key, d.threshold);
        raw.get(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = m >> e & 1 ? v[e] * d.factor : 0.0f;
        Eight<T>::store(y + at, 0, left, v);
    }
}

template <typename T>
void launch(const void* x, void* y, int64_t n, const Dropout& d, hipStream_t st)
{
    const int64_t blocks = ceil_div(ceil_div(n, 8), kThreads), most = (int64_t)num_compute_units() * 32;
    hipLaunchKernelGGL(dropout_kernel<T>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(kThreads), 0, st, static_cast<const uint8_t*>(x), static_cast<uint8_t*>(y), n, d);
}

}  // namespace
}  // namespace mi8

using namespace mi8;

extern "C" int mi8_dropout(const void* x, int hp_dtype, int64_t n, uint32_t threshold, float factor, uint64_t seed, const int64_t* seed_on_device, uint64_t offset,
                           void* y, void* stream)
{
    MI8_REQUIRE(float_type(hp_dtype), MI8_ERR_ARG, "mi8_dropout: unknown element type %d", hp_dtype);
    MI8_REQUIRE(n >= 0 && threshold <= 65536, MI8_ERR_ARG, "mi8_dropout: bad size or threshold");
    if (n == 0) return MI8_OK;
    MI8_REQUIRE(x != nullptr && y != nullptr, MI8_ERR_ARG, "mi8_dropout: null pointer");
    const Dropout d{seed, offset, seed_on_device, threshold, factor};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (hp_dtype == MI8_BF16)
        launch<half::Bf16>(x, y, n, d, st);
    else if (hp_dtype == MI8_F16)
        launch<half::F16>(x, y, n, d, st);
    else
        launch<F32>(x, y, n, d, st);
    return launch_status("mi8_dropout");
}
