// Which tiles a product of the language-model operators takes, and what their callers share: padded copies of operands
// whose rows do not start on 16-byte boundaries, and the joining of partial sums of a product cut along its contraction.
#pragma once
#include "product_tile.hpp"

namespace swc_hip {
namespace product {

using Big = Cfg<4, 2, 2, 4, 3, 2>;    // 256 x 256, eight wavefronts, one workgroup per CU
using Deep = Cfg<4, 4, 2, 2, 3, 2>;   // 256 x 256, four wavefronts of 128 x 128: a third less LDS traffic, a longer end
using Mid = Cfg<2, 2, 2, 2, 3, 2>;    // 128 x 128, four wavefronts, two workgroups per CU
using Low = Cfg<1, 2, 2, 2, 3, 3>;    // 64 x 128, two
using Small = Cfg<1, 1, 2, 2, 3, 3>;  // 64 x 64, three
using Thin = Cfg<1, 1, 1, 4, 4, 4>;   // 32 x 128, two: few rows, the other operand streams

enum Kind { kBig, kDeep, kMid, kLow, kSmall, kThin };
struct Plan {
    Kind kind;
    int splits, k_per_split;
    int first = 0;        // > 0: these columns on tiles of `kind`, those behind them on tiles of `rest`, uncut
    Kind rest = kMid;
    size_t partial_bytes(int m, int n) const { return splits > 1 ? (size_t)splits * m * n * sizeof(float) : 0; }
};

// most memory the partial sums of one product may take
constexpr size_t kMaxPartials = (size_t)256 << 20;

// The tile and the number of ranges of the contraction with the least estimated time (microseconds):
//     start and end of a workgroup, f, for each round of the chip
//   + slices * max(the time of a slice alone on a CU, workgroups per CU * its share of a busy CU)
//   + the output at 4.5 TB/s, and for a cut contraction the joining kernel: 4 us and the partial sums again.
// The bf16 constants are fits to 10 shapes of 128-2048 x 1024-4096 x 512-50264 at 1 to 32 ranges.  What the model chooses
// there, and the other side measured: 333 x 1411 x 1003 7.0 us (64 x 64 whole; 128 x 128 in four ranges 8.3 and the
// joining), 512 x 4096 x 4096 24.4 (64 x 128 whole; 128 x 128 in two 23.0 and the joining), 2048 x 4096 x 4096 63.5 (128 x
// 128; 256 x 256 83.2), 1400 x 1024 x 50264 175 (256 x 256 in eight; 128 x 128 in four 250).  An fp32 slice is half as many
// products at a sixteenth of the rate: the matrix cores set its time.
// one: only whole contractions.  The cost goes to *cost_of.
template <class T> Plan plan_uniform(int m, int n, int k, bool one, double *cost_of) {
    struct Tile {
        Kind kind;
        int bm, bn, per_cu;
        double f, alone, busy;
    };
    static constexpr Tile kBf16Tiles[] = {{kBig, 256, 256, 1, 10.8, 0.89, 1.2}, {kMid, 128, 128, 2, 4.3, 0.43, 0.46},
                                          {kLow, 64, 128, 2, 4.3, 0.275, 0.32}, {kSmall, 64, 64, 3, 3.3, 0.225, 0.2},
                                          {kThin, 32, 128, 2, 3.0, 0.23, 0.16}};
    static constexpr Tile kFp32Tiles[] = {{kBig, 256, 256, 1, 12, 7.2, 7.2}, {kMid, 128, 128, 2, 5, 2.0, 1.83},
                                          {kLow, 64, 128, 2, 4.5, 1.05, 0.95}, {kSmall, 64, 64, 3, 3.5, 0.55, 0.48},
                                          {kThin, 32, 128, 2, 3.0, 0.55, 0.5}};
    constexpr int kPer = kSlice<T>, E = sizeof(T);
    const int cus = num_cus();
    const int slices = k > 0 ? (k + kPer - 1) / kPer : 1;
    const double operands = (double)E * ((double)m * k + (double)n * k) / 9e6;   // (from the last-level cache)
    Plan best{kMid, 1, slices * kPer};
    double least = 1e30;
    for (const Tile &t : kIsBf16<T> ? kBf16Tiles : kFp32Tiles) {
        if ((t.kind == kThin) != (m <= 32)) continue;
        const long tiles = (long)((m + t.bm - 1) / t.bm) * ((n + t.bn - 1) / t.bn);
        for (int splits = 1; splits <= 64 && splits <= slices; splits += splits < 4 ? 1 : splits < 16 ? 2 : 8) {
            const int each = (slices + splits - 1) / splits, s = (slices + each - 1) / each;
            if (s > 1 && (one || each < 4 || (size_t)s * m * n * sizeof(float) > kMaxPartials)) break;
            const double groups = (double)tiles * s;
            const bool smooth = t.per_cu > 1 && groups >= 4.0 * t.per_cu * cus;   // (ends that do not fall together)
            const double q = groups <= cus ? 1 : smooth ? groups / cus : (double)((long)((groups + cus - 1) / cus));
            const double rounds = q <= t.per_cu ? 1 : q / t.per_cu;
            double work = each * (t.alone > q * t.busy ? t.alone : q * t.busy);
            work = work > operands ? work : operands;
            const double mn = (double)m * n;
            const double cost = rounds * t.f + work + (s > 1 ? 4 + 8 * s * mn / 4.5e6 : E * mn / 4.5e6);
            if (cost < least) least = cost, best = Plan{t.kind, s, each * kPer};
        }
    }
    *cost_of = least;
    return best;
}
// A product on 256 x 256 tiles whose last round is a small part of the chip leaves the columns of that round to smaller tiles
// in a second launch (3 us): bf16 8192 x 8800 x 4096 492 -> 472 us, 2048 x 9000 x 4096 158 -> 139, fp32 1999 x 50257 x 1024
// 1811 -> 1681.
template <class T> Plan plan_product(int m, int n, int k, bool one = false) {
    double cost = 0;
    Plan best = plan_uniform<T>(m, n, k, one, &cost);
    const int cus = num_cus();
    const long tall = (m + 255) / 256, wide = (n + 255) / 256, rounds = tall * wide / cus, cols = rounds * cus / tall;
    if (rounds > 0 && cols > 0 && cols < wide && m > 32) {
        const double f = kIsBf16<T> ? 10.8 : 12, busy = kIsBf16<T> ? 1.2 : 7.2;
        const int slices = (k + kSlice<T> - 1) / kSlice<T>, first = (int)cols * 256;
        double tail = 0;
        const Plan rest = plan_uniform<T>(m, n - first, k, true, &tail);
        const double both = rounds * (f + slices * busy) + sizeof(T) * (double)m * first / 4.5e6 + tail + 3;
        if (both < cost && rest.kind != kBig) best = Plan{kBig, 1, slices * kSlice<T>, first, rest.kind};
    }
    // one wavefront per SIMD pays where the end of a tile is a small part of it: bf16 8192^3 785 -> 757 us, K = 4096 412 -> 417
    if (best.kind == kBig && kIsBf16<T> && best.k_per_split >= 6144) best.kind = kDeep;
    return best;
}

// An epilogue's from(j) is itself for the product's columns from j on.  Those with arithmetic of their own (kHeavy) do not
// take the four-wavefront form of the large tile, whose one wavefront per SIMD has nothing beside it while they run; those
// without kThinToo never run on 32-row tiles.
template <Layout LA, Layout LB, class T, class Ep>
int run_product(const Plan &p, const Shape<T> &s, const Ep &ep, const char *who) {
    Shape<T> t = s;
    t.k_per_split = p.k_per_split, t.splits = p.splits;
    if (p.first > 0 && p.first < s.n) {
        Plan whole = p, rest = p;
        whole.first = rest.first = 0, rest.kind = p.rest;
        t.n = p.first;
        if (int rc = run_product<LA, LB>(whole, t, ep, who)) return rc;
        t.b += LB == kAlongK ? p.first * s.ldb : (long)p.first;
        t.n = s.n - p.first;
        return run_product<LA, LB>(rest, t, ep.from(p.first), who);
    }
    if constexpr (!Ep::kHeavy && kIsBf16<T>)
        if (p.kind == kDeep) return launch_product<T, Deep, LA, LB>(t, ep, who);
    if constexpr (Ep::kThinToo)
        if (p.kind == kThin) return launch_product<T, Thin, LA, LB>(t, ep, who);
    switch (p.kind) {
    case kMid: return launch_product<T, Mid, LA, LB>(t, ep, who);
    case kLow: return launch_product<T, Low, LA, LB>(t, ep, who);
    case kSmall: return launch_product<T, Small, LA, LB>(t, ep, who);
    default: return launch_product<T, Big, LA, LB>(t, ep, who);
    }
}

// what the loads take: rows on 16-byte boundaries
template <class T> bool aligned_rows(const T *p, long ld) { return aligned16(p) && ld % kChunk<T> == 0; }
template <class T> long row_length(long cols) { return (cols + kChunk<T> - 1) / kChunk<T> * kChunk<T>; }

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

#if __HIP_DEVICE_COMPILE__
// `have` (at least one) elements from any address, zeros behind them: four in fp32, or 16 bytes as they are
__device__ __forceinline__ void load4(const bf16 *p, int have, float (&x)[4]) {
    if (have >= 4) {
        const v2u d = *reinterpret_cast<const At<bf16>::four *>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __builtin_bit_cast(float, e & 1 ? d[e / 2] & 0xffff0000u : d[e / 2] << 16);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = e < have ? load_any(p + e) : 0.f;
    }
}
__device__ __forceinline__ void load4(const float *p, int have, float (&x)[4]) {
    if (have >= 4) {
        const v4f d = *reinterpret_cast<const At<float>::four *>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = d[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = e < have ? p[e] : 0.f;
    }
}
__device__ __forceinline__ void store4(bf16 *p, int have, const float (&x)[4]) {
    if (have >= 4) {
        *reinterpret_cast<At<bf16>::four *>(p) = v2u{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < have) store_any(p + e, x[e]);
    }
}
__device__ __forceinline__ void store4(float *p, int have, const float (&x)[4]) {
    if (have >= 4) {
        *reinterpret_cast<At<float>::four *>(p) = v4f{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < have) p[e] = x[e];
    }
}
template <class T> __device__ __forceinline__ v4u chunk_at(const T *p, long have) {
    if (have >= kChunk<T>) return __builtin_bit_cast(v4u, *reinterpret_cast<const typename At<T>::chunk *>(p));
    v4u d = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < kChunk<T>; ++e)
        if (e < have) {
            if constexpr (kIsBf16<T>) d[e / 2] |= (unsigned)p[e] << (16 * (e & 1));
            else d[e] = __builtin_bit_cast(unsigned, p[e]);
        }
    return d;
}
#endif

// dst[r][0..ld) = src[r][0..cols) and zeros behind; dst null: nothing to copy.  dst: rows on 16-byte boundaries, ld =
// row_length(cols).
template <class T> struct Copy {
    T *dst;
    const T *src;
    long ld, lds;
    int rows, cols;
    long chunks() const { return dst ? rows * (ld / kChunk<T>) : 0; }
#if __HIP_DEVICE_COMPILE__
    __device__ __forceinline__ void chunk(long i) const {
        const long per = ld / kChunk<T>, row = i / per, j = (i - row * per) * kChunk<T>;
        *reinterpret_cast<v4u *>(dst + row * ld + j) = chunk_at(src + row * lds + j, cols - j);
    }
#endif
};
// both operands of a product, in one launch
template <class T> int copy_operands(const Copy<T> &a, const Copy<T> &b);
// out[m][n] (rows of ld) = the sum of `parts` matrices, in order
template <class T> int join_parts(T *out, long ld, const float *part, int parts, int m, int n);
// out[j] = sum over parts p of part[p][j], in a fixed order
template <class T> int sum_parts(T *out, const float *part, int parts, int n);

// One product of the gradients: whole tiles straight to the output, or cut along the contraction and joined.
template <Layout LA, Layout LB, class T>
int grad_product(const char *who, const Plan &p, const Shape<T> &s, const Store<T> &out, float *part) {
    if (p.splits == 1) return run_product<LA, LB>(p, s, out, who);
    if (int rc = run_product<LA, LB>(p, s, StorePartial{part, (long)s.m * s.n, s.n, false}, who)) return rc;
    return join_parts<T>(out.out, out.ld, part, p.splits, s.m, s.n);
}

// Both in one launch, dA's (m x k) and dB's (k x n): where their tiles are the small ones and all of their workgroups fit
// the chip at once.  512 x 1024 x 784 fp32 37.9 us in two launches, 33.5 in one, bf16 18.7 and 14.5.
inline bool pairs(const Plan &pa, const Plan &pb, int m, int n, int k) {
    const long a = (long)ceil_div(m, pa.kind == kThin ? 32 : 64) * ceil_div(k, pa.kind == kThin ? 128 : 64) * pa.splits;
    const long b = (long)ceil_div(k, 64) * ceil_div(n, 64) * pb.splits;
    return (pa.kind == kSmall || pa.kind == kThin) && pb.kind == kSmall && a + b <= (pa.kind == kThin ? 2L : 3L) * num_cus();
}
template <class T>
int grad_pair(const Plan &pa, Shape<T> a, const Store<T, true> &out_a, float *part_a, const Plan &pb, Shape<T> b,
              const Store<T, true> &out_b, float *part_b) {
    a.k_per_split = pa.k_per_split, a.splits = pa.splits;
    b.k_per_split = pb.k_per_split, b.splits = pb.splits;
    const StoreEither<T> ea{out_a, {pa.splits > 1 ? part_a : nullptr, (long)a.m * a.n, a.n, false}};
    const StoreEither<T> eb{out_b, {pb.splits > 1 ? part_b : nullptr, (long)b.m * b.n, b.n, false}};
    if (int rc = pa.kind == kThin ? launch_pair<T, Thin, Small>(a, ea, b, eb) : launch_pair<T, Small, Small>(a, ea, b, eb)) return rc;
    if (pa.splits > 1 && out_a.out)
        if (int rc = join_parts<T>(out_a.out, out_a.ld, part_a, pa.splits, a.m, a.n)) return rc;
    return pb.splits > 1 ? join_parts<T>(out_b.out, out_b.ld, part_b, pb.splits, b.m, b.n) : (int)SWC_HIP_OK;
}

} // namespace product

} // namespace swc_hip
