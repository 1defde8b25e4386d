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
            if (residual) r.template load<WHOLE>(residual + row * ldr, ok, col0, n, h);
            float z[P::kValues], x[P::kValues];
#pragma unroll
            for (int u = 0; u < P::kValues; ++u) z[u] = P::value(acc[tm], u) + (bias ? b.value(u) : 0.f);
            if (preact) store_row<P, WHOLE>(preact + row * ldp, ok, col0, n, h, z);
            if (residual) r.get(x);
#pragma unroll
            for (int u = 0; u < P::kValues; ++u) z[u] = act_value<ACT, kIsBf16<T>>(z[u]) + (residual ? x[u] : 0.f);
            store_row<P, WHOLE>(c + row * ldc, ok, col0, n, h, z);
        }
    }
    template <class P, int TM, int TN>
    __device__ __forceinline__ void finish(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane, int) const {
        if (row0 + 32 * TM <= m && col0 + 32 * TN <= n) end<P, true>(acc, row0, col0, m, n, lane);
        else end<P, false>(acc, row0, col0, m, n, lane);
    }
#endif
};

// The end of a layer from fp32 sums: `parts` matrices of m x n to be added in order, then bias, activation, residual.
// Four columns of a row a thread.
template <class T, int ACT>
__global__ __launch_bounds__(256) void fc_finish(const float *part, int parts, long part_stride, const T *bias, const T *residual,
                                                 long ldr, T *preact, long ldp, T *c, long ldc, int m, int n) {
#if __HIP_DEVICE_COMPILE__
    const int j = (blockIdx.x * 64 + (threadIdx.x & 63)) * 4;
    if (j >= n) return;
    const int have = n - j < 4 ? n - j : 4;
    float b[4] = {};
    if (bias) load4(bias + j, have, b);
    for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < m; r += gridDim.y * 4) {
        float z[4] = {}, x[4] = {};
        const float *p = part + (long)r * n + j;
        if (residual) load4(residual + r * ldr + j, have, x);
#pragma unroll 8
        for (int i = 0; i < parts; ++i) {
            float d[4];
            load4(p + i * part_stride, have, d);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] += d[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] += b[e];
        if (preact) store4(preact + r * ldp + j, have, z);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = act_value<ACT, kIsBf16<T>>(z[e]) + x[e];
        store4(c + r * ldc + j, have, z);
    }
#endif
}
template <class T>
int launch_finish(int act, const float *part, int parts, const T *bias, const T *residual, long ldr, T *preact, long ldp, T *c, long ldc,
                  int m, int n) {
    const unsigned rows = ceil_div(m, 4);
    const dim3 grid(ceil_div(n, 256), rows > 16384 ? 16384 : rows);
    return with_act(act, [&]<int ACT>() {
        fc_finish<T, ACT><<<grid, 256, 0, stream()>>>(part, parts, (long)m * n, bias, residual, ldr, preact, ldp, c, ldc, m, n);
        SWC_LAUNCH_CHECK();
        return (int)SWC_HIP_OK;
    });
}

// Rows into copies whose rows start on 16-byte boundaries, zeros behind their end: 16 bytes a thread, both operands of a
// product in one launch.
template <class T> __device__ __forceinline__ void copy_chunk(const Copy<T> &c, long row, long j) {
    *reinterpret_cast<v4u *>(c.dst + row * c.ld + j) = chunk_at(c.src + row * c.lds + j, c.cols - j);
}
template <class T> __global__ __launch_bounds__(256) void copy_chunks(Copy<T> a, Copy<T> b, long chunks_a, long chunks) {
#if __HIP_DEVICE_COMPILE__
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (long)gridDim.x * 256) {
        const bool first = i < chunks_a;
        const long per = (first ? a.ld : b.ld) / kChunk<T>, at = first ? i : i - chunks_a;
        const long row = at / per, j = (at - row * per) * kChunk<T>;
        if (first) copy_chunk(a, row, j);
        else copy_chunk(b, row, j);
    }
#endif
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
    if (k == 0) return launch_finish<T>(act, nullptr, 0, bias, residual, ldr, preact, ldp, c, ldc, m, n);
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
    if (int rc = copy_operands<T>({pack_a ? w.a : nullptr, a, row_length<T>(k), lda, m, k}, {pack_b ? w.b : nullptr, b, row_length<T>(n), ldb, k, n}))
        return rc;
    if (pack_a) a = w.a, lda = row_length<T>(k);
    if (pack_b) b = w.b, ldb = row_length<T>(n);
    const Shape<T> s{a, b, lda, ldb, m, n, k, 0, nullptr};
    if (!partial_sums(p)) {
        return with_act(act, [&]<int ACT>() {
            return run_product<kAlongK, kAcross>(p, s, FcEpilogue<T, ACT>{bias, residual, preact, c, ldr, ldp, ldc}, who);
        });
    }
    if (int rc = run_product<kAlongK, kAcross>(p, s, StorePartial{w.part, (long)m * n, n, false}, who)) return rc;
    return launch_finish<T>(act, w.part, p.splits, bias, residual, ldr, preact, ldp, c, ldc, m, n);
}

} // namespace

namespace swc_hip {
namespace product {

template <class T> int copy_operands(const Copy<T> &a, const Copy<T> &b) {
    const long na = a.dst ? a.rows * (a.ld / kChunk<T>) : 0, nb = b.dst ? b.rows * (b.ld / kChunk<T>) : 0;
    if (!(na + nb)) return SWC_HIP_OK;
    copy_chunks<T><<<grid_of(na + nb), 256, 0, stream()>>>(a, b, na, na + nb);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}
template <class T> int join_parts(T *out, long ld, const float *part, int parts, int m, int n) {
    return launch_finish<T>(SWC_HIP_ACT_NONE, part, parts, nullptr, nullptr, 0, nullptr, 0, out, ld, m, n);
}
template <class T> int sum_parts(T *out, const float *part, int parts, int n) {
    if (!n) return SWC_HIP_OK;
    add_parts<T><<<ceil_div(n, 32), 256, 0, stream()>>>(out, part, parts, n);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}
template int copy_operands<bf16>(const Copy<bf16> &, const Copy<bf16> &);
template int copy_operands<float>(const Copy<float> &, const Copy<float> &);
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
