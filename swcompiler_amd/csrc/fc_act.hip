// The fully connected layer with its activation and a second summand (matrixMatrixFCActAdd_f/_bf), next to
// matrixMatrixFCBias_f (gemm.hip):
//
//     Z = A B + bias, C = act(Z) + residual
//
// One product on the core of product_tile.hpp, with everything behind the sums in its epilogue; a product cut along k
// (few tiles) leaves fp32 partial sums in the workspace and ends in fc_finish.  4096 x 16384 x 4096 bf16 with bias, tanh
// gelu and residual: 486 us (the product alone 412, the residual's 134 MB another 30).
#include "act.hpp"
#include "product.hpp"

using namespace swc_hip;
using namespace swc_hip::product;

namespace {

template <class T, int ACT> struct FcEpilogue {
    static constexpr bool kHeavy = true, kThinToo = false;
    const T *bias, *residual;
    T *preact, *c;
    long ldr, ldp, ldc;
    bool vec;   // every matrix given has 16-byte aligned rows, and the bias can be read four elements at a time
#if __HIP_DEVICE_COMPILE__
    template <class P, bool WHOLE, int TM, int TN>
    __device__ __forceinline__ void end(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane) const {
        const int l32 = lane & 31, h = lane >> 5;
        ColumnData<T, P> b;
        RowData<T, P> r;
        if (bias) b.template load<WHOLE>(bias, col0, n, h);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + P::row(tm, l32);
            const bool ok = row < m;
            // a row's second summand is requested together, before its first use
            if (residual) r.template load<WHOLE>(residual + row * ldr, ok, col0, n, vec, h);
            float z[P::kValues], x[P::kValues];
#pragma unroll
            for (int u = 0; u < P::kValues; ++u) z[u] = P::value(acc[tm], u) + (bias ? b.value(u) : 0.f);
            if (preact) store_row<P, WHOLE>(preact + row * ldp, ok, col0, n, vec, h, z);
            if (residual) r.get(x);
#pragma unroll
            for (int u = 0; u < P::kValues; ++u) z[u] = act_value<ACT, kIsBf16<T>>(z[u]) + (residual ? x[u] : 0.f);
            store_row<P, WHOLE>(c + row * ldc, ok, col0, n, vec, h, z);
        }
    }
    template <class P, int TM, int TN>
    __device__ __forceinline__ void finish(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane, int) const {
        if (vec && row0 + 32 * TM <= m && col0 + 32 * TN <= n) end<P, true>(acc, row0, col0, m, n, lane);
        else end<P, false>(acc, row0, col0, m, n, lane);
    }
#endif
};

// The end of a layer from fp32 sums: `parts` matrices of m x n to be added in order, then bias, activation, residual.
// Four columns of a row a thread; VEC: rows of sums on 16-byte boundaries.
template <class T, int ACT, bool VEC>
__global__ __launch_bounds__(256) void fc_finish(const float *part, int parts, long ldpart, long part_stride, const T *bias,
                                                 const T *residual, long ldr, T *preact, long ldp, T *c, long ldc, int m, int n) {
#if __HIP_DEVICE_COMPILE__
    const int j = (blockIdx.x * 64 + (threadIdx.x & 63)) * 4;
    if (j >= n) return;
    float b[4] = {};
    if (bias)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = j + e < n ? load_any(bias + j + e) : 0.f;
    for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < m; r += gridDim.y * 4) {
        float z[4] = {}, x[4] = {};
        const float *p = part + r * ldpart + j;
        if (residual)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = j + e < n ? load_any(residual + r * ldr + j + e) : 0.f;
#pragma unroll 8
        for (int i = 0; i < parts; ++i) {
            if (VEC) {
                const float4 d = *reinterpret_cast<const float4 *>(p + i * part_stride);
                z[0] += d.x, z[1] += d.y, z[2] += d.z, z[3] += d.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] += j + e < n ? p[i * part_stride + e] : 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (j + e >= n) continue;
            z[e] += b[e];
            if (preact) store_any(preact + r * ldp + j + e, z[e]);
            store_any(c + r * ldc + j + e, act_value<ACT, kIsBf16<T>>(z[e]) + x[e]);
        }
    }
#endif
}
template <class T>
int launch_finish(int act, const float *part, int parts, long ldpart, long part_stride, const T *bias, const T *residual, long ldr,
                  T *preact, long ldp, T *c, long ldc, int m, int n) {
    const unsigned rows = ceil_div(m, 4);
    const dim3 grid(ceil_div(n, 256), rows > 16384 ? 16384 : rows);
    const bool vec = aligned16(part) && ldpart % 4 == 0 && part_stride % 4 == 0 && n % 4 == 0;
    return with_act(act, [&]<int ACT>() {
        if (vec) fc_finish<T, ACT, true><<<grid, 256, 0, stream()>>>(part, parts, ldpart, part_stride, bias, residual, ldr, preact, ldp, c, ldc, m, n);
        else fc_finish<T, ACT, false><<<grid, 256, 0, stream()>>>(part, parts, ldpart, part_stride, bias, residual, ldr, preact, ldp, c, ldc, m, n);
        SWC_LAUNCH_CHECK();
        return (int)SWC_HIP_OK;
    });
}

// Rows into a copy whose rows start on 16-byte boundaries, zeros behind their end and in the rows that do not exist:
// 16 bytes a thread.  A source at any alignment is read in the two aligned 16-byte pieces that hold the thread's eight
// values (each of them holds at least one that exists, so neither leaves the allocation's pages), shifted together.
__device__ __forceinline__ uint4 eight_at(const bf16 *p, int have) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint4 *q = reinterpret_cast<const uint4 *>(at & ~(uintptr_t)15);
    const int shift = (int)(at & 15) * 8;
    const uint4 lo = q[0], hi = shift / 16 + have > 8 ? q[1] : make_uint4(0, 0, 0, 0);
    typedef unsigned __int128 u128;
    const u128 l = (u128)(((uint64_t)lo.y << 32) | lo.x) | ((u128)(((uint64_t)lo.w << 32) | lo.z) << 64);
    const u128 h = (u128)(((uint64_t)hi.y << 32) | hi.x) | ((u128)(((uint64_t)hi.w << 32) | hi.z) << 64);
    u128 v = shift ? (l >> shift) | (h << (128 - shift)) : l;
    if (have < 8) v &= ((u128)1 << (16 * have)) - 1;
    const uint64_t a = (uint64_t)v, b = (uint64_t)(v >> 64);
    return make_uint4((unsigned)a, (unsigned)(a >> 32), (unsigned)b, (unsigned)(b >> 32));
}
__device__ __forceinline__ uint4 chunk_at(const bf16 *p, long have) { return eight_at(p, have < 8 ? (int)have : 8); }
__device__ __forceinline__ uint4 chunk_at(const float *p, long have) {
    if (have >= 4 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) return *reinterpret_cast<const uint4 *>(p);
    unsigned v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < have ? __builtin_bit_cast(unsigned, p[e]) : 0u;
    return make_uint4(v[0], v[1], v[2], v[3]);
}
template <class T>
__global__ __launch_bounds__(256) void copy_chunks(T *dst, long ld, const T *src, long lds, int rows, int cols, const int *index,
                                                   const int *count) {
    const int have = count ? *count : rows;
    const long j = ((long)blockIdx.x * 256 + threadIdx.x) * kChunk<T>;
    if (j >= ld) return;
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < have && j < cols) v = chunk_at(src + (index ? index[r] : r) * lds + j, cols - j);
        *reinterpret_cast<uint4 *>(dst + r * ld + j) = v;
    }
}

// 32 columns and eight ranges of the parts a workgroup: a range's parts are added in order, then the ranges in order.
template <class T> __global__ __launch_bounds__(256) void add_parts(T *out, const float *part, int parts, int n) {
    __shared__ float sums[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int j = blockIdx.x * 32 + tx;
    const int each = (parts + 7) / 8, p0 = ty * each, p1 = p0 + each < parts ? p0 + each : parts;
    float s = 0.f;
    if (j < n)
#pragma unroll 4
        for (int p = p0; p < p1; ++p) s += part[(size_t)p * n + j];
    sums[ty][tx] = s;
    __syncthreads();
    if (ty || j >= n) return;
#pragma unroll
    for (int y = 1; y < 8; ++y) s += sums[y][tx];
    store_any(out + j, s);
}

template <class T>
int check_forward(const char *who, int m, int n, int k, const T *a, int lda, const T *b, int ldb, int act, const T *residual,
                  int ldr, const T *preact, int ldp, const T *c, int ldc) {
    if (m < 0 || n < 0 || k < 0) return fail(SWC_HIP_EINVAL, "%s: negative dimension", who);
    if (!known_act(act)) return fail(SWC_HIP_EINVAL, "%s: unknown activation %d", who, act);
    if (m == 0 || n == 0) return SWC_HIP_OK;
    if (!c || (k && (!a || !b))) return fail(SWC_HIP_EINVAL, "%s: null pointer", who);
    if ((k && (lda < k || ldb < n)) || ldc < n || (residual && ldr < n) || (preact && ldp < n))
        return fail(SWC_HIP_EINVAL, "%s: leading dimension smaller than row length", who);
    if ((const void *)c == a || (const void *)c == b || (preact && (preact == a || preact == b || preact == c || preact == residual)))
        return fail(SWC_HIP_EINVAL, "%s: an output is also an input", who);
    if (lda > kMaxLd<T> || ldb > kMaxLd<T>) return fail(SWC_HIP_EUNSUPPORTED, "%s: leading dimension beyond %ld", who, kMaxLd<T>);
    return SWC_HIP_OK;
}

// Few rows, or a cut contraction: sums to the workspace, the end of the layer in fc_finish.
bool partial_sums(const Plan &p) { return p.splits > 1 || p.kind == kThin; }

template <class T> struct Space {
    T *a, *b;
    float *part;
    size_t bytes;
};
template <class T> Space<T> space(char *base, const Plan &p, int m, int n, int k, bool pack_a, bool pack_b) {
    Carver c{base};
    Space<T> s{};
    s.a = pack_a ? c.take<T>((size_t)m * row_length<T>(k)) : nullptr;
    s.b = pack_b ? c.take<T>((size_t)k * row_length<T>(n)) : nullptr;
    s.part = partial_sums(p) ? c.take<float>((size_t)p.splits * m * n) : nullptr;
    s.bytes = c.used;
    return s;
}

template <class T>
int forward(const char *who, int m, int n, int k, const T *a, int lda_, const T *b, int ldb_, const T *bias, int act, const T *residual,
            int ldr, T *preact, int ldp, T *c, int ldc) {
    if (int rc = check_forward(who, m, n, k, a, lda_, b, ldb_, act, residual, ldr, preact, ldp, c, ldc)) return rc;
    if (!ready()) return fail(SWC_HIP_ENOTINIT, "%s: swc_hip_init has not been called", who);
    if (m == 0 || n == 0) return SWC_HIP_OK;
    if (k == 0) return launch_finish<T>(act, nullptr, 0, 0, 0, bias, residual, ldr, preact, ldp, c, ldc, m, n);
    long lda = lda_, ldb = ldb_;
    const Plan p = plan_product<T>(m, n, k);
    const bool pack_a = !aligned_rows(a, lda) || k % kChunk<T>, pack_b = !aligned_rows(b, ldb);
    const size_t need = space<T>(nullptr, p, m, n, k, pack_a, pack_b).bytes;
    Space<T> w{};
    if (need) {
        char *base = static_cast<char *>(workspace(need, who));
        if (!base) return fail_code();
        w = space<T>(base, p, m, n, k, pack_a, pack_b);
    }
    if (pack_a) {
        if (int rc = copy_rows<T>(w.a, row_length<T>(k), a, lda, m, k, nullptr, nullptr)) return rc;
        a = w.a, lda = row_length<T>(k);
    }
    if (pack_b) {
        if (int rc = copy_rows<T>(w.b, row_length<T>(n), b, ldb, k, n, nullptr, nullptr)) return rc;
        b = w.b, ldb = row_length<T>(n);
    }
    const Shape<T> s{a, b, lda, ldb, m, n, k, 0, nullptr};
    if (!partial_sums(p)) {
        const bool vec = (!residual || aligned_rows(residual, ldr)) && (!preact || aligned_rows(preact, ldp)) && aligned_rows(c, ldc) &&
                         reinterpret_cast<uintptr_t>(bias) % (4 * sizeof(T)) == 0;
        return with_act(act, [&]<int ACT>() {
            return run_product<kAlongK, kAcross>(p, s, FcEpilogue<T, ACT>{bias, residual, preact, c, ldr, ldp, ldc, vec}, who);
        });
    }
    if (int rc = run_product<kAlongK, kAcross>(p, s, StorePartial{w.part, (long)m * n, n, false}, who)) return rc;
    return launch_finish<T>(act, w.part, p.splits, n, (long)m * n, bias, residual, ldr, preact, ldp, c, ldc, m, n);
}

} // namespace

namespace swc_hip {
namespace product {

template <class T> int copy_rows(T *dst, long ld, const T *src, long lds, int rows, int cols, const int *index, const int *count) {
    if (!rows || !ld) return SWC_HIP_OK;
    copy_chunks<T><<<dim3(ceil_div(ld / kChunk<T>, 256), rows < 32768 ? rows : 32768), 256, 0, stream()>>>(dst, ld, src, lds, rows, cols,
                                                                                                          index, count);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}
template <class T> int join_parts(T *out, long ld, const float *part, int parts, int m, int n) {
    return launch_finish<T>(SWC_HIP_ACT_NONE, part, parts, n, (long)m * n, nullptr, nullptr, 0, nullptr, 0, out, ld, m, n);
}
template <class T> int sum_parts(T *out, const float *part, int parts, int n) {
    if (!n) return SWC_HIP_OK;
    add_parts<T><<<ceil_div(n, 32), 256, 0, stream()>>>(out, part, parts, n);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}
template int copy_rows<bf16>(bf16 *, long, const bf16 *, long, int, int, const int *, const int *);
template int copy_rows<float>(float *, long, const float *, long, int, int, const int *, const int *);
template int join_parts<bf16>(bf16 *, long, const float *, int, int, int);
template int join_parts<float>(float *, long, const float *, int, int, int);
template int sum_parts<bf16>(bf16 *, const float *, int, int);
template int sum_parts<float>(float *, const float *, int, int);

} // namespace product
} // namespace swc_hip

extern "C" {

int swc_hip_matrixMatrixFCActAdd_f(int m, int n, int k, const float *a, int lda, const float *b, int ldb, const float *bias,
                                   int act, const float *residual, int ldr, float *preact, int ldp, float *c, int ldc) {
    return forward<float>("swc_hip_matrixMatrixFCActAdd_f", m, n, k, a, lda, b, ldb, bias, act, residual, ldr, preact, ldp, c, ldc);
}

int swc_hip_matrixMatrixFCActAdd_bf(int m, int n, int k, const swc_hip_bf16 *a, int lda, const swc_hip_bf16 *b, int ldb,
                                    const swc_hip_bf16 *bias, int act, const swc_hip_bf16 *residual, int ldr,
                                    swc_hip_bf16 *preact, int ldp, swc_hip_bf16 *c, int ldc) {
    return forward<bf16>("swc_hip_matrixMatrixFCActAdd_bf", m, n, k, a, lda, b, ldb, bias, act, residual, ldr, preact, ldp, c, ldc);
}

size_t swc_hip_matrixMatrixFCActAdd_workspace_bytes(int m, int n, int k, int bf) {
    if (!ready() || m <= 0 || n <= 0 || k <= 0) return 0;
    return bf ? space<bf16>(nullptr, plan_product<bf16>(m, n, k), m, n, k, true, true).bytes
              : space<float>(nullptr, plan_product<float>(m, n, k), m, n, k, true, true).bytes;
}

} // extern "C"
