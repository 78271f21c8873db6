// Entry points of the experts' products: checks and operands; the kernels are in experts_kernel.h.
#include "experts_kernel.h"
#include "paia_gemv.h"

namespace paia {

constexpr int kMostExperts = 1024, kMostPairs = 1 << 26, kMostColumns = 1 << 25;     // K; N too

struct ExpertOperands {
    const void *W, *meta, *zeros, *x, *order, *offsets, *bias;
    void* out;
    long long x_stride, out_stride;
    int experts, N, K, pairs, x_rows, gated;
};

template <typename Launch>
static int run_experts(int fmt, const ExpertOperands& o, hipStream_t st, Launch launch)
{
    const bool i4 = fmt == kI4 || fmt == kI4ZP;
    const int step = fmt == kBF16 ? 8 : (fmt == kFP8 ? 16 : kBlockCols);
    if (o.experts <= 0 || o.experts > kMostExperts || o.N <= 0 || o.N > kMostColumns || o.K <= 0 || o.K > kMostColumns || o.K % step ||
        o.pairs < 0 || o.pairs >= kMostPairs || o.x_rows < 0 || (o.gated != 0 && o.gated != 1) || (o.gated && o.N % 2))
        return -2;
    if (o.pairs == 0) return 0;
    if (o.x_rows <= 0 || o.pairs % o.x_rows) return -2;
    const int cols = o.gated ? o.N / 2 : o.N;
    if (o.W == nullptr || o.x == nullptr || o.order == nullptr || o.offsets == nullptr || o.out == nullptr ||
        (fmt != kBF16 && o.meta == nullptr) || (fmt == kI4ZP && o.zeros == nullptr))
        return -2;
    if (!aligned(o.W, 16) || !aligned(o.x, 16) || !aligned(o.order, 4) || !aligned(o.offsets, 4) || !aligned(o.out, 2) ||
        !aligned(o.bias, 2) || !aligned(o.meta, fmt == kFP8 ? 4 : 2) || o.x_stride < 0 || o.x_stride % 8 ||
        (o.x_rows > 1 && o.x_stride < o.K) || o.out_stride < 0 || (o.pairs > 1 && o.out_stride < cols))
        return -2;
    ExpertsParams p;
    p.tiles = p.most = 0;
    p.W = static_cast<const uint8_t*>(o.W);
    p.meta = static_cast<const uint8_t*>(o.meta);
    p.zeros = static_cast<const uint8_t*>(o.zeros);
    p.x = static_cast<const uint16_t*>(o.x);
    p.bias = static_cast<const uint16_t*>(o.bias);
    p.out = static_cast<uint16_t*>(o.out);
    p.order = static_cast<const int32_t*>(o.order);
    p.offsets = static_cast<const int32_t*>(o.offsets);
    p.x_stride = o.x_stride, p.out_stride = o.out_stride;
    p.E = o.experts, p.N = o.N, p.K = o.K, p.R = o.pairs, p.cols = cols;
    p.lane_experts = (o.experts + kWave - 1) / kWave;
    p.row_bytes = (uint32_t)(fmt == kBF16 ? 2 * o.K : (fmt == kFP8 ? o.K : o.K / 2));
    p.G = i4 ? o.K / kBlockCols : 0;
    p.zbytes = (uint32_t)(p.G + 1) / 2;
    const int64_t x_bytes = ((int64_t)(o.x_rows - 1) * o.x_stride + o.K) * 2;
    p.x_bytes = x_bytes < (1ll << 31) ? (uint32_t)x_bytes : 0;
    p.by_pairs = Divisor((uint32_t)(o.pairs / o.x_rows));
    return launch(p, o.gated != 0, st);
}

}  // namespace paia

extern "C" {

int paia_experts_bf16(const void* W, const void* x, long long x_stride, int x_rows, const void* order, const void* offsets,
                      const void* bias, void* out, long long out_stride, int experts, int N, int K, int pairs, int gated,
                      void* stream)
{
    using namespace paia;
    return run_experts(kBF16, {W, nullptr, nullptr, x, order, offsets, bias, out, x_stride, out_stride, experts, N, K, pairs,
                               x_rows, gated}, static_cast<hipStream_t>(stream), launch_experts_bf16);
}

int paia_experts_fp8(const void* Wq, const void* scale, const void* x, long long x_stride, int x_rows, const void* order,
                     const void* offsets, const void* bias, void* out, long long out_stride, int experts, int N, int K,
                     int pairs, int gated, void* stream)
{
    using namespace paia;
    return run_experts(kFP8, {Wq, scale, nullptr, x, order, offsets, bias, out, x_stride, out_stride, experts, N, K, pairs,
                              x_rows, gated}, static_cast<hipStream_t>(stream), launch_experts_fp8);
}

int paia_experts_int4(const void* Wq, const void* scales, const void* x, long long x_stride, int x_rows, const void* order,
                      const void* offsets, void* out, long long out_stride, int experts, int N, int K, int pairs, int gated,
                      void* stream)
{
    using namespace paia;
    return run_experts(kI4, {Wq, scales, nullptr, x, order, offsets, nullptr, out, x_stride, out_stride, experts, N, K, pairs,
                             x_rows, gated}, static_cast<hipStream_t>(stream), launch_experts_int4);
}

int paia_experts_int4_zp(const void* Wq, const void* scales, const void* zeros, const void* x, long long x_stride,
                         int x_rows, const void* order, const void* offsets, const void* bias, void* out,
                         long long out_stride, int experts, int N, int K, int pairs, int gated, void* stream)
{
    using namespace paia;
    return run_experts(kI4ZP, {Wq, scales, zeros, x, order, offsets, bias, out, x_stride, out_stride, experts, N, K, pairs,
                               x_rows, gated}, static_cast<hipStream_t>(stream), launch_experts_int4_zp);
}

}  // extern "C"
