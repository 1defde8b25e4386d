// The gradients of the fully connected layer with its activation (matrixMatrixFCActAddGrad_f/_bf):
//
//     dZ = dC act'(Z), dA = dZ B^T, dB = A^T dZ, dbias = column sums of dZ
//
// The two products on the core of product_tile.hpp, no matrix transposed in memory; dZ in one pass (three times its size
// at the memory's rate), rounded to the matrices' type once for both products, its column sums before that rounding.  (The
// matrix cores take both operands in one type: a dZ of fp32 would cost bfloat16 a second product for its lower half, and
// twice the memory.  Its rounding brings the error of dA and dB from the 0.0017 of their own last rounding to 0.0024, in the
// norm.)  Without an activation dZ is dC itself.  4096 x 16384 x 4096 bf16 with tanh gelu: 876-896 us, 1240 TFLOP/s.
#include "act.hpp"
#include "product.hpp"

using namespace swc_hip;
using namespace swc_hip::product;

namespace {

// dZ = dC act'(Z) into dz (zeros in columns n .. ld), and each block of rows' column sums of the unrounded values.  64
// threads side by side hold four columns each, four rows at a time.  Bound by memory: three passes over m x n (4096 x 16384
// bf16, 403 MB, 86 us, 4.7 TB/s: the copy's rate less what the slope costs).
template <class T, int ACT>
__global__ __launch_bounds__(256) void act_grad(T *dz, long ld, const T *dc, long ldc, const T *z, long ldz, int m, int n, float *sums,
                                                T *dbias, int each) {
#if __HIP_DEVICE_COMPILE__
    __shared__ float part[4][256];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int j = (blockIdx.x * 64 + tx) * 4;
    const int r0 = blockIdx.y * each;
    const int r1 = r0 + each < m ? r0 + each : m;
    const int have = n - j;
    float sum[4] = {};
    if (have > 0) {
#pragma unroll 8
        for (int r = r0 + ty; r < r1; r += 4) {
            float g[4];
            load4(dc + r * ldc + j, have, g);
            if constexpr (ACT != SWC_HIP_ACT_NONE) {
                float y[4];
                load4(z + r * ldz + j, have, y);
#pragma unroll
                for (int e = 0; e < 4; ++e) g[e] = act_grad_value<ACT, kIsBf16<T>>(y[e], g[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e >= have) g[e] = 0.f;
                sum[e] += g[e];
            }
            if (dz) store4(dz + r * ld + j, (int)ld - j, g);
        }
    } else if (dz && j < ld) {   // the rest of the padding
        const float none[4] = {};
        for (int r = r0 + ty; r < r1; r += 4) store4(dz + r * ld + j, (int)ld - j, none);
    }
    if (!sums && !dbias) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) part[ty][tx * 4 + e] = sum[e];
    __syncthreads();
    const int col = blockIdx.x * 256 + threadIdx.x;
    float s = 0.f;
#pragma unroll
    for (int y = 0; y < 4; ++y) s += part[y][threadIdx.x];
    if (col >= n) return;
    if (dbias) store_any(dbias + col, s);   // (one block of rows)
    else sums[(size_t)blockIdx.y * n + col] = s;
#endif
}

template <class T>
int check_grad(const char *who, int m, int n, int k, const T *dc, int lddc, const T *a, int lda, const T *b, int ldb,
               const T *preact, int ldp, int act, const T *da, int ldda, const T *db, int lddb, const T *dbias) {
    if (m < 0 || n < 0 || k < 0) return fail(SWC_HIP_EINVAL, "%s: negative dimension", who);
    if (!known_act(act)) return fail(SWC_HIP_EINVAL, "%s: unknown activation %d", who, act);
    if (m && n && !dc) return fail(SWC_HIP_EINVAL, "%s: null pointer", who);
    if (act != SWC_HIP_ACT_NONE && m && n && !preact) return fail(SWC_HIP_EINVAL, "%s: preact is needed for this activation", who);
    if ((da && m && n && k && !b) || (db && m && n && k && !a)) return fail(SWC_HIP_EINVAL, "%s: null pointer", who);
    if (lddc < n || (da && (ldda < k || ldb < n)) || (db && (lddb < n || lda < k)) || (act != SWC_HIP_ACT_NONE && ldp < n))
        return fail(SWC_HIP_EINVAL, "%s: leading dimension smaller than row length", who);
    const void *in[4] = {dc, a, b, preact};
    for (const void *p : in)
        if (p && (p == da || p == db || p == dbias)) return fail(SWC_HIP_EINVAL, "%s: an output is also an input", who);
    if ((da && (da == db || da == dbias)) || (db && db == dbias)) return fail(SWC_HIP_EINVAL, "%s: two outputs are the same", who);
    if (lda > kMaxLd<T> || ldb > kMaxLd<T> || lddc > kMaxLd<T> || n > kMaxLd<T> || k > kMaxLd<T>)
        return fail(SWC_HIP_EUNSUPPORTED, "%s: leading dimension beyond %ld", who, kMaxLd<T>);
    if (m > kMaxRows) return fail(SWC_HIP_EUNSUPPORTED, "%s: more than %d rows", who, kMaxRows);
    return SWC_HIP_OK;
}

// Rows a workgroup takes: 32, or 8 where that leaves the chip short of workgroups (with dB and k = 64, 32 / 8: 512 x 1024 13.0 /
// 10.2 us, 64 x 4096 11.2 / 8.2); more where a grid's 65535 rows of workgroups would not cover them.  Up to 32 rows are one
// block where column sums are wanted, with no kernel for the blocks' sums (one block / blocks of 8: 16 x 4096 7.2 / 8.1 us, 32
// x 4096 9.1 / 8.0 and a launch's time on the host).
int sum_rows(int m, int n, bool sums) {
    if (m <= 32 && sums) return 32;
    if ((m + 31) / 32 > 65535) return (m + 65534) / 65535;
    return (long)((m + 31) / 32) * ((n + 255) / 256) >= 4L * swc::devices::HipDevice::computeUnits ? 32 : 8;
}
int sum_blocks(int m, int n, bool sums) { return (m + sum_rows(m, n, sums) - 1) / sum_rows(m, n, sums); }

template <class T>
int launch_act_grad(T *dz, long ld, const T *dc, long lddc, const T *z, long ldz, int act, int m, int n, float *sums, T *dbias) {
    if (!dz) ld = 0;
    const dim3 grid(ceil_div(ld > n ? ld : n, 256), sum_blocks(m, n, dbias));
    return with_act(act, [&]<int ACT>() {
        act_grad<T, ACT><<<grid, 256, 0, stream()>>>(dz, ld, dc, lddc, z, ldz, m, n, sums, sums ? nullptr : dbias, sum_rows(m, n, dbias));
        SWC_LAUNCH_CHECK();
        return (int)SWC_HIP_OK;
    });
}

template <class T> struct Space {
    T *dz, *a, *b;
    float *part, *sums;
    size_t bytes;
};
template <class T>
Space<T> space(char *base, int m, int n, int k, bool own_dz, bool pack_a, bool pack_b, size_t partials, bool bias) {
    Carver c{base};
    Space<T> s{};
    s.dz = own_dz ? c.take<T>((size_t)m * row_length<T>(n)) : nullptr;
    s.a = pack_a ? c.take<T>((size_t)m * row_length<T>(k)) : nullptr;
    s.b = pack_b ? c.take<T>((size_t)k * row_length<T>(n)) : nullptr;
    s.part = partials ? c.take<float>(partials / sizeof(float)) : nullptr;
    s.sums = bias && sum_blocks(m, n, true) > 1 ? c.take<float>((size_t)sum_blocks(m, n, true) * n) : nullptr;
    s.bytes = c.used;
    return s;
}

size_t larger(size_t a, size_t b) { return a > b ? a : b; }

template <class T>
int gradients(const char *who, int m, int n, int k, const T *dc, int lddc, const T *a, int lda_, const T *b, int ldb_, const T *preact,
              int ldp, int act, T *da, int ldda, T *db, int lddb, T *dbias) {
    if (int rc = check_grad(who, m, n, k, dc, lddc, a, lda_, b, ldb_, preact, ldp, act, da, ldda, db, lddb, dbias)) return rc;
    if (!ready()) return fail(SWC_HIP_ENOTINIT, "%s: swc_hip_init has not been called", who);
    if (m == 0 || n == 0) {   // sums of nothing
        if (int rc = zero_rows(da, ldda, m, k)) return rc;
        if (int rc = zero_rows(db, lddb, k, n)) return rc;
        return zero_rows(dbias, n, 1, n);
    }
    if (k == 0) da = db = nullptr;
    long lda = lda_, ldb = ldb_;
    const Plan pa = plan_product<T>(m, k, n), pb = plan_product<T>(k, n, m);
    // dZ is dC itself without an activation; a copy when its rows do not start on 16-byte boundaries, or when dA would
    // read past the end of a row
    const bool tail = da && n % kChunk<T>;
    const bool own_dz = (da || db) && (act != SWC_HIP_ACT_NONE || !aligned_rows(dc, lddc) || tail);
    const bool pack_a = db && !aligned_rows(a, lda), pack_b = da && (!aligned_rows(b, ldb) || tail);
    const bool pair = da && db && pairs(pa, pb, m, n, k);
    const size_t partials = pair ? pa.partial_bytes(m, k) + pb.partial_bytes(k, n)
                                 : larger(da ? pa.partial_bytes(m, k) : 0, db ? pb.partial_bytes(k, n) : 0);
    const size_t need = space<T>(nullptr, m, n, k, own_dz, pack_a, pack_b, partials, dbias).bytes;
    Space<T> w{};
    if (need) {
        char *base = static_cast<char *>(workspace(need, who));
        if (!base) return fail_code();
        w = space<T>(base, m, n, k, own_dz, pack_a, pack_b, partials, dbias);
    }
    const long padded = row_length<T>(n);
    if (own_dz || dbias) {
        if (int rc = launch_act_grad<T>(w.dz, padded, dc, lddc, preact, ldp, act, m, n, w.sums, dbias)) return rc;
        if (w.sums)
            if (int rc = sum_parts<T>(dbias, w.sums, sum_blocks(m, n, true), n)) return rc;
    }
    const T *dz = own_dz ? w.dz : dc;
    const long lddz = own_dz ? padded : lddc;
    if (int rc = copy_operands<T>({pack_a ? w.a : nullptr, a, row_length<T>(k), lda, m, k}, {pack_b ? w.b : nullptr, b, padded, ldb, k, n}))
        return rc;
    if (pack_a) a = w.a, lda = row_length<T>(k);
    if (pack_b) b = w.b, ldb = padded;
    const Shape<T> sa{dz, b, lddz, ldb, m, k, n, 0, 1, nullptr}, sb{a, dz, lda, lddz, k, n, m, 0, 1, nullptr};
    if (pair) return grad_pair<T>(pa, sa, {da, ldda}, w.part, pb, sb, {db, lddb}, w.part + pa.partial_bytes(m, k) / sizeof(float));
    if (da)
        if (int rc = grad_product<kAlongK, kAlongK, T>(who, pa, sa, {da, ldda}, w.part)) return rc;
    if (db)
        if (int rc = grad_product<kAcross, kAcross, T>(who, pb, sb, {db, lddb}, w.part)) return rc;
    return SWC_HIP_OK;
}

template <class T> size_t most(int m, int n, int k) {
    size_t partials = 0;
    if (k > 0) {
        const Plan pa = plan_product<T>(m, k, n), pb = plan_product<T>(k, n, m);
        const size_t a = pa.partial_bytes(m, k), b = pb.partial_bytes(k, n);
        partials = pairs(pa, pb, m, n, k) ? a + b : larger(a, b);
    }
    return space<T>(nullptr, m, n, k > 0 ? k : 0, true, true, true, partials, true).bytes;
}

} // namespace

extern "C" {

int swc_hip_matrixMatrixFCActAddGrad_f(int m, int n, int k, const float *cGrad, int ldcg, const float *a, int lda, const float *b,
                                       int ldb, const float *preact, int ldp, int act, float *aGrad, int ldag, float *bGrad,
                                       int ldbg, float *biasGrad) {
    return gradients<float>("swc_hip_matrixMatrixFCActAddGrad_f", m, n, k, cGrad, ldcg, a, lda, b, ldb, preact, ldp, act, aGrad, ldag,
                            bGrad, ldbg, biasGrad);
}

int swc_hip_matrixMatrixFCActAddGrad_bf(int m, int n, int k, const swc_hip_bf16 *cGrad, int ldcg, const swc_hip_bf16 *a, int lda,
                                        const swc_hip_bf16 *b, int ldb, const swc_hip_bf16 *preact, int ldp, int act,
                                        swc_hip_bf16 *aGrad, int ldag, swc_hip_bf16 *bGrad, int ldbg, swc_hip_bf16 *biasGrad) {
    return gradients<bf16>("swc_hip_matrixMatrixFCActAddGrad_bf", m, n, k, cGrad, ldcg, a, lda, b, ldb, preact, ldp, act, aGrad, ldag,
                           bGrad, ldbg, biasGrad);
}

size_t swc_hip_matrixMatrixFCActAddGrad_workspace_bytes(int m, int n, int k, int bf) {
    if (!ready() || m <= 0 || n <= 0) return 0;
    return bf ? most<bf16>(m, n, k) : most<float>(m, n, k);
}

} // extern "C"
