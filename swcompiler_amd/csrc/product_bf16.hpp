// Which tiles a bf16 product takes, and the helpers its callers share: padded copies of operands whose rows do not
// start on 16-byte boundaries, and the joining of partial sums of a product cut along its contraction.
#pragma once
#include "gemm_bf16.hpp"

namespace swc_hip {
namespace mfma16 {

using Big = Cfg<4, 2, 2, 4, 64, 3, 2>;      // 256 x 256, eight wavefronts, one workgroup per CU
using Mid = Cfg<2, 2, 2, 2, 64, 3, 2>;      // 128 x 128, four wavefronts, two workgroups per CU
using Low = Cfg<1, 2, 2, 2, 64, 3, 3>;      // 64 x 128
using Thin = Cfg<1, 1, 1, 4, 64, 4, 4>;     // 32 x 128: few rows, the other operand streams

using Deep = Cfg<4, 4, 2, 2, 64, 3, 2>;  // 256 x 256, four wavefronts of 128 x 128: a third less LDS traffic, a longer end

enum Kind { kBig, kDeep, kMid, kLow, kThin };
struct Plan {
    Kind kind;
    int splits, k_per_split;
    size_t partial_bytes(int m, int n) const { return splits > 1 ? (size_t)splits * m * n * sizeof(float) : 0; }
};

// most memory the partial sums of one product may take
constexpr size_t kMaxPartials = (size_t)256 << 20;

inline Plan plan_product(int m, int n, int k) {
    const int cus = num_cus();
    auto tiles = [&](int bm, int bn) { return (long)((m + bm - 1) / bm) * ((n + bn - 1) / bn); };
    Plan p{kBig, 1, 0};
    long have;
    int per_cu;
    if (m <= 32) p.kind = kThin, have = tiles(32, 128), per_cu = 2;
    else if (m <= 64) p.kind = kLow, have = tiles(64, 128), per_cu = 2;
    else if (tiles(256, 256) * 4 >= 3L * cus) p.kind = k >= 6144 ? kDeep : kBig, have = tiles(256, 256), per_cu = 1;
    else p.kind = kMid, have = tiles(128, 128), per_cu = 2;
    // too few tiles: ranges of the contraction, at least four slices each
    const int slices = (k + 63) / 64;
    long splits = 1;
    if (have < (long)per_cu * cus && slices >= 8) {
        splits = ((long)per_cu * cus + have - 1) / have;
        if (splits > slices / 4) splits = slices / 4;
        while (splits > 1 && (size_t)splits * m * n * sizeof(float) > kMaxPartials) --splits;
        if (splits > 64) splits = 64;
    }
    const int each = (int)((slices + splits - 1) / splits);
    p.splits = slices ? (slices + each - 1) / each : 1;
    p.k_per_split = (each ? each : 1) * 64;
    return p;
}

// The epilogues with arithmetic of their own (kHeavy) do not take the four-wavefront form of the large tile, whose one
// wavefront per SIMD has nothing beside it while they run; those with kTall exist for the large and middle tiles only.
template <Layout LA, Layout LB, class Ep>
int run_product(const Plan &p, const Shape &s, const Ep &ep, const char *who) {
    Shape t = s;
    t.k_per_split = p.k_per_split;
    if constexpr (!Ep::kHeavy)
        if (p.kind == kDeep) return launch_gemm_bf16<Deep, LA, LB>(t, p.splits, ep, who);
    if constexpr (!Ep::kTall) {
        if (p.kind == kLow) return launch_gemm_bf16<Low, LA, LB>(t, p.splits, ep, who);
        if (p.kind == kThin) return launch_gemm_bf16<Thin, LA, LB>(t, p.splits, ep, who);
    }
    if (p.kind == kMid) return launch_gemm_bf16<Mid, LA, LB>(t, p.splits, ep, who);
    return launch_gemm_bf16<Big, LA, LB>(t, p.splits, ep, who);
}

inline bool aligned_rows(const void *p, long ld) { return aligned16(p) && ld % 8 == 0; }
inline long round8(long x) { return (x + 7) & ~7L; }

// A workspace handed out in 256-byte steps; with a null base it only counts.
struct Carver {
    char *base;
    size_t used = 0;
    template <class T> T *take(size_t count) {
        const size_t at = used;
        used += (count * sizeof(T) + 255) & ~(size_t)255;
        return base ? reinterpret_cast<T *>(base + at) : nullptr;
    }
};

// an element in fp32, whichever the type
__device__ __forceinline__ float load_any(const uint16_t *p) { return __builtin_bit_cast(float, (unsigned)*p << 16); }
__device__ __forceinline__ float load_any(const float *p) { return *p; }
__device__ __forceinline__ void store_any(float *p, float x) { *p = x; }
__device__ __forceinline__ void store_any(uint16_t *p, float x) {
#if __HIP_DEVICE_COMPILE__
    *p = __builtin_bit_cast(uint16_t, (__bf16)x);
#endif
}

inline unsigned grid_of(size_t n) {
    const size_t b = (n + 255) / 256;
    return (unsigned)(b > 16384 ? 16384 : b);
}

template <class T> __global__ __launch_bounds__(256) void fill_rows(T *p, long ld, int rows, int cols) {
    const size_t total = (size_t)rows * cols, step = (size_t)gridDim.x * 256;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) p[(i / cols) * ld + i % cols] = T(0);
}
template <class T> int zero_rows(T *p, long ld, int rows, int cols) {
    if (!p || !rows || !cols) return SWC_HIP_OK;
    fill_rows<T><<<grid_of((size_t)rows * cols), 256, 0, stream()>>>(p, ld, rows, cols);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

// dst[r][0..ld) = src[rows ? rows[r] : r][0..cols) and zeros; rows at or beyond *count (when given) become zeros
int copy_rows_bf16(uint16_t *dst, long ld, const uint16_t *src, long lds, int rows, int cols, const int *index, const int *count);
int copy_rows_f32(float *dst, long ld, const float *src, long lds, int rows, int cols, const int *index, const int *count);
// out[j] = sum over parts p of part[p][j], in that order
int sum_parts(uint16_t *out_bf, float *out_f, const float *part, int parts, int n);

} // namespace mfma16

} // namespace swc_hip
