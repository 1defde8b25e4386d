// The fully connected layer with its activation and a second summand (matrixMatrixFCActAdd_f/_bf) and its gradients,
// next to matrixMatrixFCBias_f (gemm.hip).
//
//     Z = A B + bias, C = act(Z) + residual;    dZ = dC act'(Z), dA = dZ B^T, dB = A^T dZ, dbias = column sums of dZ
//
// bf16: three products on the core of gemm_bf16.hpp with no matrix transposed in memory.  fp32: the kernels of
// gemm.hip (row-major operands; the gradients' operands are transposed into the workspace first), the activation in a
// pass of its own — 12 bytes per element against 2 k flops at the fp32 matrix rate, 4 % at k = 4096.
#include "act.hpp"
#include "product_bf16.hpp"

using namespace swc_hip;
using namespace swc_hip::mfma16;

namespace {

template <int ACT> struct FcEpilogue {
    static constexpr bool kHeavy = true, kThinToo = false;
    const uint16_t *bias, *residual;
    uint16_t *preact, *c;
    long ldr, ldp, ldc;
    bool vec;   // every matrix given has 16-byte aligned rows, and the bias an 8-byte aligned start
#if __HIP_DEVICE_COMPILE__
    template <bool WHOLE, int TM, int TN>
    __device__ __forceinline__ void finish(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane) const {
        const int l32 = lane & 31, h = lane >> 5;
        v2u b[TN][4];
        v4u r[TN][2];
        if (bias)
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) load_columns<WHOLE>(bias, col0 + tn * 32, n, h, b[tn]);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + tm * 32 + l32;
            const bool ok = row < m;
            // a row block's second summand is requested together, before its first use
            if (residual)
#pragma unroll
                for (int tn = 0; tn < TN; ++tn) load_block<WHOLE>(residual + row * ldr, ok, col0 + tn * 32, n, vec, h, r[tn]);
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) {
                const int cb = col0 + tn * 32;
                float z[16], x[16];
#pragma unroll
                for (int v = 0; v < 16; ++v) z[v] = acc[tm][tn][v] + (bias ? column_value(b[tn], v) : 0.f);
                if (preact) store_block<WHOLE>(preact + row * ldp, ok, cb, n, vec, h, z);
                if (residual) unpack_block(r[tn], x);
#pragma unroll
                for (int v = 0; v < 16; ++v) z[v] = act_value<ACT, true>(z[v]) + (residual ? x[v] : 0.f);
                store_block<WHOLE>(c + row * ldc, ok, cb, n, vec, h, z);
            }
        }
    }
    template <int TM, int TN>
    __device__ __forceinline__ void operator()(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane, int) const {
        if (vec && row0 + 32 * TM <= m && col0 + 32 * TN <= n) finish<true>(acc, row0, col0, m, n, lane);
        else finish<false>(acc, row0, col0, m, n, lane);
    }
#endif
};

// The end of a layer from fp32 sums: `parts` matrices of m x n to be added in order, then bias, activation, residual.
// (part may be c itself: fp32, one part.)  Four columns of a row a thread; VEC: rows of sums on 16-byte boundaries.
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
            store_any(c + r * ldc + j + e, act_value<ACT, sizeof(T) == 2>(z[e]) + x[e]);
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
__device__ __forceinline__ uint4 eight_at(const uint16_t *p, int have) {
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
__global__ __launch_bounds__(256) void copy_rows16(uint16_t *dst, long ld, const uint16_t *src, long lds, int rows, int cols,
                                                   const int *index, const int *count) {
    const int have = count ? *count : rows;
    const long j = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
    if (j >= ld) return;
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < have && j < cols) v = eight_at(src + (index ? index[r] : r) * lds + j, cols - j < 8 ? (int)(cols - j) : 8);
        *reinterpret_cast<uint4 *>(dst + r * ld + j) = v;
    }
}
// fp32 (dst and ld as the product wants them: any): four values a thread where everything is aligned
template <bool VEC>
__global__ __launch_bounds__(256) void copy_rows32(float *dst, long ld, const float *src, long lds, int rows, int cols, const int *index,
                                                   const int *count) {
    const int have = count ? *count : rows;
    const long j = ((long)blockIdx.x * 256 + threadIdx.x) * (VEC ? 4 : 1);
    if (j >= ld) return;
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        const float *p = src + (index && r < have ? index[r] : r) * lds + j;
        if (VEC) *reinterpret_cast<float4 *>(dst + r * ld + j) = r < have ? *reinterpret_cast<const float4 *>(p) : make_float4(0, 0, 0, 0);
        else dst[r * ld + j] = r < have && j < cols ? *p : 0.f;
    }
}

// 32 columns and eight ranges of the parts a workgroup: a range's parts are added in order, then the ranges in order.
__global__ __launch_bounds__(256) void add_parts(uint16_t *out_bf, float *out_f, const float *part, int parts, int n) {
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
    if (out_bf) store_any(out_bf + j, s);
    if (out_f) out_f[j] = s;
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
    if (sizeof(T) == 2 && (lda > kMaxLd || ldb > kMaxLd))
        return fail(SWC_HIP_EUNSUPPORTED, "%s: leading dimension beyond %ld", who, kMaxLd);
    return SWC_HIP_OK;
}

// Few rows, or a cut contraction: sums to the workspace, the end of the layer in fc_finish.
bool partial_sums(const Plan &p) { return p.splits > 1 || p.kind == kThin; }

struct ForwardSpace {
    uint16_t *a, *b;
    float *part;
    size_t bytes;
};
ForwardSpace forward_space(char *base, const Plan &p, int m, int n, int k, bool pack_a, bool pack_b) {
    Carver c{base};
    ForwardSpace s{};
    s.a = pack_a ? c.take<uint16_t>((size_t)m * round8(k)) : nullptr;
    s.b = pack_b ? c.take<uint16_t>((size_t)k * round8(n)) : nullptr;
    s.part = partial_sums(p) ? c.take<float>((size_t)p.splits * m * n) : nullptr;
    s.bytes = c.used;
    return s;
}

int forward_bf16(const char *who, int m, int n, int k, const uint16_t *a, long lda, const uint16_t *b, long ldb,
                 const uint16_t *bias, int act, const uint16_t *residual, long ldr, uint16_t *preact, long ldp, uint16_t *c,
                 long ldc) {
    const Plan p = plan_product(m, n, k);
    const bool pack_a = !aligned_rows(a, lda) || k % 8, pack_b = !aligned_rows(b, ldb);
    const size_t need = forward_space(nullptr, p, m, n, k, pack_a, pack_b).bytes;
    ForwardSpace w{};
    if (need) {
        char *base = static_cast<char *>(workspace(need, who));
        if (!base) return fail_code();
        w = forward_space(base, p, m, n, k, pack_a, pack_b);
    }
    if (pack_a) {
        if (int rc = copy_rows_bf16(w.a, round8(k), a, lda, m, k, nullptr, nullptr)) return rc;
        a = w.a, lda = round8(k);
    }
    if (pack_b) {
        if (int rc = copy_rows_bf16(w.b, round8(n), b, ldb, k, n, nullptr, nullptr)) return rc;
        b = w.b, ldb = round8(n);
    }
    const Shape s{a, b, lda, ldb, m, n, k, 0, nullptr};
    if (!partial_sums(p)) {
        const bool vec = (!residual || aligned_rows(residual, ldr)) && (!preact || aligned_rows(preact, ldp)) && aligned_rows(c, ldc) &&
                         (reinterpret_cast<uintptr_t>(bias) & 7) == 0;
        return with_act(act, [&]<int ACT>() {
            return run_product<kAlongK, kAcross>(p, s, FcEpilogue<ACT>{bias, residual, preact, c, ldr, ldp, ldc, vec}, who);
        });
    }
    if (int rc = run_product<kAlongK, kAcross>(p, s, StorePartial{w.part, (long)m * n, n, false}, who)) return rc;
    return launch_finish<uint16_t>(act, w.part, p.splits, n, (long)m * n, bias, residual, ldr, preact, ldp, c, ldc, m, n);
}

} // namespace

int swc_hip::mfma16::join_parts(uint16_t *out, long ld, const float *part, int parts, int m, int n) {
    return launch_finish<uint16_t>(SWC_HIP_ACT_NONE, part, parts, n, (long)m * n, nullptr, nullptr, 0, nullptr, 0, out, ld, m, n);
}
int swc_hip::mfma16::copy_rows_bf16(uint16_t *dst, long ld, const uint16_t *src, long lds, int rows, int cols, const int *index,
                                    const int *count) {
    if (!rows || !ld) return SWC_HIP_OK;
    copy_rows16<<<dim3(ceil_div(ld / 8, 256), rows < 32768 ? rows : 32768), 256, 0, stream()>>>(dst, ld, src, lds, rows, cols, index, count);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}
int swc_hip::mfma16::copy_rows_f32(float *dst, long ld, const float *src, long lds, int rows, int cols, const int *index,
                                   const int *count) {
    if (!rows || !ld) return SWC_HIP_OK;
    const bool vec = aligned16(dst) && aligned16(src) && ld % 4 == 0 && lds % 4 == 0 && cols == ld;
    const dim3 grid(ceil_div(vec ? ld / 4 : ld, 256), rows < 32768 ? rows : 32768);
    if (vec) copy_rows32<true><<<grid, 256, 0, stream()>>>(dst, ld, src, lds, rows, cols, index, count);
    else copy_rows32<false><<<grid, 256, 0, stream()>>>(dst, ld, src, lds, rows, cols, index, count);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}
int swc_hip::mfma16::sum_parts(uint16_t *out_bf, float *out_f, const float *part, int parts, int n) {
    if (!n) return SWC_HIP_OK;
    add_parts<<<ceil_div(n, 32), 256, 0, stream()>>>(out_bf, out_f, part, parts, n);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

extern "C" {

int swc_hip_matrixMatrixFCActAdd_f(int m, int n, int k, const float *a, int lda, const float *b, int ldb, const float *bias,
                                   int act, const float *residual, int ldr, float *preact, int ldp, float *c, int ldc) {
    const char *who = "swc_hip_matrixMatrixFCActAdd_f";
    if (int rc = check_forward(who, m, n, k, a, lda, b, ldb, act, residual, ldr, preact, ldp, c, ldc)) return rc;
    SWC_REQUIRE_INIT();
    if (m == 0 || n == 0) return SWC_HIP_OK;
    // Z goes to preact, or to C, or to the workspace where C still holds the second summand
    const size_t split = k ? swc_hip_gemm_workspace_bytes(m, n, k) : 0;
    const bool apart = !preact && residual == c;
    Carver size{nullptr};
    size.take<float>(split / sizeof(float) + 1);
    if (apart) size.take<float>((size_t)m * n);
    char *base = nullptr;
    if (split || apart) {
        base = static_cast<char *>(workspace(size.used, who));
        if (!base) return fail_code();
    }
    Carver w{base};
    float *part = w.take<float>(split / sizeof(float) + 1);
    float *z = apart ? w.take<float>((size_t)m * n) : preact ? preact : c;
    const int ldz = apart ? n : preact ? ldp : ldc;
    if (k) {
        // (no scratch needed: any address that is not null stands for the empty array)
        if (int rc = gemm_f32(who, m, n, k, a, lda, b, ldb, bias, z, ldz, 0, part ? part : z, split)) return rc;
        bias = nullptr;
    } else {
        if (int rc = zero_rows(z, ldz, m, n)) return rc;
    }
    if (act == SWC_HIP_ACT_NONE && !residual && z == c && !bias) return SWC_HIP_OK;
    return launch_finish<float>(act, z, 1, ldz, 0, bias, residual, ldr, k ? nullptr : preact, ldp, c, ldc, m, n);
}

int swc_hip_matrixMatrixFCActAdd_bf(int m, int n, int k, const swc_hip_bf16 *a, int lda, const swc_hip_bf16 *b, int ldb,
                                    const swc_hip_bf16 *bias, int act, const swc_hip_bf16 *residual, int ldr,
                                    swc_hip_bf16 *preact, int ldp, swc_hip_bf16 *c, int ldc) {
    const char *who = "swc_hip_matrixMatrixFCActAdd_bf";
    if (int rc = check_forward(who, m, n, k, a, lda, b, ldb, act, residual, ldr, preact, ldp, c, ldc)) return rc;
    SWC_REQUIRE_INIT();
    if (m == 0 || n == 0) return SWC_HIP_OK;
    if (k == 0) return launch_finish<uint16_t>(act, nullptr, 0, 0, 0, bias, residual, ldr, preact, ldp, c, ldc, m, n);
    return forward_bf16(who, m, n, k, a, lda, b, ldb, bias, act, residual, ldr, preact, ldp, c, ldc);
}

size_t swc_hip_matrixMatrixFCActAdd_workspace_bytes(int m, int n, int k, int bf) {
    if (!ready() || m <= 0 || n <= 0 || k <= 0) return 0;
    if (bf) return forward_space(nullptr, plan_product(m, n, k), m, n, k, true, true).bytes;
    Carver c{nullptr};
    c.take<float>(swc_hip_gemm_workspace_bytes(m, n, k) / sizeof(float) + 1);
    c.take<float>((size_t)m * n);
    return c.used;
}

} // extern "C"
