// The fully connected layer with its activation and a second summand (matrixMatrixFCActAdd_f/_bf), next to
// matrixMatrixFCBias_f (gemm.hip):
//
//     Z = A B + bias, C = act(Z) + residual
//
// One product on the core of product_tile.hpp, with everything behind the sums in its epilogue; a product cut along k
// (few tiles) leaves fp32 partial sums in the workspace and ends in fc_finish; few rows take fc_stream or fc_few.
// 4096 x 16384 x 4096 bf16 with bias, tanh gelu and residual: 462-467 us, 1180 TFLOP/s (the product alone 412; the residual's 134
// MB another 30).  2048 x 4096 x 4096 fp32 with gelu and residual 500 us, 137 TFLOP/s of the 152 that a large product reaches.
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
    FcEpilogue from(int j) const {
        return {bias ? bias + j : nullptr, residual ? residual + j : nullptr, preact ? preact + j : nullptr, c + j, ldr, ldp, ldc};
    }
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
// Four columns of a row a thread.  Bound by memory: parts + 1 to 3 passes over m x n; where it runs that is a few MB from
// the caches, and its launch (two parts of 512 x 784: 4.1 us).
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

// Up to eight rows in bf16 (decoding): bound by one pass over B.  A workgroup owns 32 columns; its sixteen wavefronts take
// slices of 64 k in turn, each with a ring of two slices of B in LDS to itself — no barrier, the next slice on its way
// while this one is multiplied — and A's fragments straight from memory (the rows are few and shared: cache).  The
// wavefronts' sums meet in LDS once, and the threads end the layer, an element each: one launch, no workspace.  Below 8192
// columns there are fewer workgroups than CUs: 4096 x 4096 runs on 128 of the 256 (8.7-9.2 us, 3.7 TB/s).
// (Workgroups 2 j and 2 j + 1, which share lines of B, are eight apart in launch order: on one XCD's L2.)
constexpr int kStreamWaves = 16, kStreamStage = 64 * 32 * 2;
constexpr size_t kStreamLds = (size_t)kStreamWaves * 2 * kStreamStage;
template <int ACT>
__global__ __launch_bounds__(64 * kStreamWaves) void fc_stream(const bf16 *a, long lda, const bf16 *b, long ldb, const bf16 *bias,
                                                               const bf16 *residual, long ldr, bf16 *preact, long ldp, bf16 *c,
                                                               long ldc, int m, int n, int k) {
#if __HIP_DEVICE_COMPILE__
    extern __shared__ __align__(16) char lds_bytes[];
    const int lane = threadIdx.x & 63, l32 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int whole = (int)(gridDim.x & ~15u), id = blockIdx.x;
    const int n0 = 32 * (id < whole ? (id & ~15) + (id & 7) * 2 + ((id >> 3) & 1) : id);
    char *ring = lds_bytes + wave * 2 * kStreamStage;
    const int slices = (k + 63) / 64;
    Loader<bf16, 32, 1, kAcross, 1> lb;
    lb.init(b, ldb, n, n0, wave * 64 < k ? wave * 64 : 0, k, k, 0, lane);
    Reader<bf16, 32, 1, kAcross> rb;
    rb.init(0, lane);
    v16f acc[1][1];
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[0][0][v] = 0.f;
    // A's chunk at k is read from an address that always exists (so that every slice issues the same number of loads) and
    // replaced by zeros where the row or the k does not.
    const bf16 *row = a + (l32 < m ? l32 : 0) * lda;
    v4u x[2][kSteps];
    auto fetch = [&](int s, int buf) {
#pragma unroll
        for (int j = 0; j < 4; ++j) lb.template issue<false>(ring + buf * kStreamStage, j, 0);
        lb.skip(kStreamWaves);
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
            const int kk = s * 64 + t * 16 + h * 8;
            x[buf][t] = *reinterpret_cast<const At<bf16>::chunk *>(row + (kk < k ? kk : 0));
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int kFetch = 4 + kSteps;
    auto multiply = [&](int s, int buf) {
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
            Frag<bf16> f[1];
            rb.read(f, ring + buf * kStreamStage, t, 0);
            rb.read(f, ring + buf * kStreamStage, t, 1);
            const bool there = l32 < m && s * 64 + t * 16 + h * 8 < k;
            const v4u y = {there ? x[buf][t][0] : 0, there ? x[buf][t][1] : 0, there ? x[buf][t][2] : 0, there ? x[buf][t][3] : 0};
            acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[0].v, __builtin_bit_cast(v8bf, y), acc[0][0], 0, 0, 0);
        }
        // the slice has been read before its stage is filled again
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    auto arrived = [&]() { asm volatile("" ::: "memory"); };   // (behind a wait: LDS may be read now)
    if (wave < slices) {
        fetch(wave, 0);
        int s = wave;
        for (; s + 2 * kStreamWaves < slices; s += 2 * kStreamWaves) {
            fetch(s + kStreamWaves, 1);
            mfma::wait_vmcnt<kFetch>();
            arrived();
            multiply(s, 0);
            fetch(s + 2 * kStreamWaves, 0);
            mfma::wait_vmcnt<kFetch>();
            arrived();
            multiply(s + kStreamWaves, 1);
        }
        if (s + kStreamWaves < slices) {
            fetch(s + kStreamWaves, 1);
            mfma::wait_vmcnt<kFetch>();
            arrived();
            multiply(s, 0);
            mfma::wait_vmcnt<0>();
            arrived();
            multiply(s + kStreamWaves, 1);
        } else {
            mfma::wait_vmcnt<0>();
            arrived();
            multiply(s, 0);
        }
    }
    // Element (lane, v) of every wavefront's sums: row l32, column 8 (v / 4) + 4 h + v % 4.
    float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int v = 0; v < 16; ++v) mine[v * 64 + lane] = acc[0][0][v];
    __syncthreads();
    const int col = n0 + 8 * (wave / 4) + 4 * h + wave % 4;
    if (l32 >= m || col >= n) return;
    float z = 0.f;
#pragma unroll
    for (int w = 0; w < kStreamWaves; ++w) z += reinterpret_cast<const float *>(lds_bytes + w * 2 * kStreamStage)[wave * 64 + lane];
    if (bias) z += load_any(bias + col);
    if (preact) store_any(preact + l32 * ldp + col, z);
    z = act_value<ACT, true>(z);
    if (residual) z += load_any(residual + l32 * ldr + col);
    store_any(c + l32 * ldc + col, z);
#endif
}
// Against the cut 32-row tiles and their joining kernel: 4096 x 4096 10.5 / 12.4 us at one to eight rows, 13.2 / 13.2 at 16;
// 16384 x 4096 25 / 25.5; 4096 x 25088 51 / 38, where 128 workgroups are too few.
bool takes_stream(int m, int k, const bf16 *b, long ldb) { return m <= 8 && k <= 8192 && k % 8 == 0 && aligned_rows(b, ldb); }
bool takes_stream(int, int, const float *, long) { return false; }
int launch_stream(int act, const bf16 *a, long lda, const bf16 *b, long ldb, const bf16 *bias, const bf16 *residual, long ldr,
                  bf16 *preact, long ldp, bf16 *c, long ldc, int m, int n, int k) {
    note_kernel("fc_stream");
    return with_act(act, [&]<int ACT>() {
        static bool attr_set = false;
        if (!attr_set) {
            SWC_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(fc_stream<ACT>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)kStreamLds));
            attr_set = true;
        }
        fc_stream<ACT><<<ceil_div(n, 32), 64 * kStreamWaves, kStreamLds, stream()>>>(a, lda, b, ldb, bias, residual, ldr, preact, ldp, c,
                                                                                     ldc, m, n, k);
        SWC_LAUNCH_CHECK();
        return (int)SWC_HIP_OK;
    });
}
int launch_stream(int, const float *, long, const float *, long, const float *, const float *, long, float *, long, float *, long, int, int,
                  int) {
    return SWC_HIP_OK;   // (fp32 does not take it)
}

// One to four rows in fp32, or one in bf16 where fc_stream does not take the operands: bound by one pass over B.  A
// workgroup owns 64 bytes of B's columns; four lanes side by side read them, 256 rows of B at a time, each a chunk of 16
// bytes from any address, eight rows ahead; the sums over the 256 lanes of a column are joined by lane exchange within a
// wavefront and through LDS between the sixteen of them, and the first threads end the layer.  One launch, no workspace.
// (Workgroups 2 j and 2 j + 1, which share lines of B, are eight apart in launch order: on one XCD's L2.)
constexpr int kFewThreads = 1024;
template <class T, int M, int ACT>
__global__ __launch_bounds__(kFewThreads) void fc_few(const T *a, long lda, const T *b, long ldb, const T *bias, const T *residual,
                                                      long ldr, T *preact, long ldp, T *c, long ldc, int m, int n, int k) {
#if __HIP_DEVICE_COMPILE__
    constexpr int CH = kChunk<T>, kCols = 4 * CH, kLanes = kFewThreads / 4, kAhead = 8;
    __shared__ float sums[kFewThreads / 64][M][kCols];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int whole = (int)(gridDim.x & ~15u), id = blockIdx.x;
    const int block = id < whole ? (id & ~15) + (id & 7) * 2 + ((id >> 3) & 1) : id;
    const int col = block * kCols + (threadIdx.x & 3) * CH;
    const int have = n - col;
    float acc[M][CH] = {};
    if (have > 0)
        for (int k0 = threadIdx.x >> 2; k0 < k; k0 += kAhead * kLanes) {
            v4u d[kAhead];
            float x[kAhead][M];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int kk = k0 + i * kLanes;
                if (kk < k) d[i] = chunk_at(b + (long)kk * ldb + col, have);
#pragma unroll
                for (int r = 0; r < M; ++r) x[i][r] = kk < k && r < m ? load_any(a + r * lda + kk) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (k0 + i * kLanes >= k) break;
#pragma unroll
                for (int e = 0; e < CH; ++e) {
                    const unsigned w = d[i][e * (int)sizeof(T) / 4];
                    const float y = __builtin_bit_cast(float, !kIsBf16<T> ? w : e & 1 ? w & 0xffff0000u : w << 16);
#pragma unroll
                    for (int r = 0; r < M; ++r) acc[r][e] = fmaf(x[i][r], y, acc[r][e]);
                }
            }
        }
#pragma unroll
    for (int r = 0; r < M; ++r)
#pragma unroll
        for (int e = 0; e < CH; ++e) {
#pragma unroll
            for (int off = 4; off < 64; off <<= 1) acc[r][e] += __shfl_xor(acc[r][e], off);
            if (lane < 4) sums[wave][r][lane * CH + e] = acc[r][e];
        }
    __syncthreads();
    const int r = threadIdx.x / kCols, j = block * kCols + threadIdx.x % kCols;
    if (r >= M || r >= m || j >= n) return;
    float z = 0.f;
#pragma unroll
    for (int w = 0; w < kFewThreads / 64; ++w) z += sums[w][r][threadIdx.x % kCols];
    if (bias) z += load_any(bias + j);
    if (preact) store_any(preact + r * ldp + j, z);
    z = act_value<ACT, kIsBf16<T>>(z);
    if (residual) z += load_any(residual + r * ldr + j);
    store_any(c + r * ldc + j, z);
#endif
}
template <class T>
int launch_few(int act, const T *a, long lda, const T *b, long ldb, const T *bias, const T *residual, long ldr, T *preact, long ldp, T *c,
               long ldc, int m, int n, int k) {
    const unsigned blocks = ceil_div(n, 4 * kChunk<T>);
    note_kernel("fc_few<%s,%d>", kIsBf16<T> ? "bf16" : "fp32", m <= 1 ? 1 : m <= 2 ? 2 : 4);
    return with_act(act, [&]<int ACT>() {
        auto kern = fc_few<T, 1, ACT>;
        if constexpr (!kIsBf16<T>)
            if (m > 1) kern = m == 2 ? fc_few<T, 2, ACT> : fc_few<T, 4, ACT>;
        kern<<<blocks, kFewThreads, 0, stream()>>>(a, lda, b, ldb, bias, residual, ldr, preact, ldp, c, ldc, m, n, k);
        SWC_LAUNCH_CHECK();
        return (int)SWC_HIP_OK;
    });
}
// bf16: from two rows on the vector units are the limit (4096 x 4096: one row 12 us, two 16, three 25) and the matrix cores
// take over; fp32, whose matrix rate is a sixteenth: four rows 16 us, 32-row tiles 26.
template <class T> constexpr int kFewRows = kIsBf16<T> ? 1 : 4;

// Rows into copies whose rows start on 16-byte boundaries, zeros behind their end: 16 bytes a thread, both operands of a
// product in one launch.  Bound by memory: 1024 x 50257 bf16, 206 MB, 33 us, 6.2 TB/s.
template <class T> __global__ __launch_bounds__(256) void copy_chunks(Copy<T> a, Copy<T> b, long chunks_a, long chunks) {
#if __HIP_DEVICE_COMPILE__
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (long)gridDim.x * 256) {
        if (i < chunks_a) a.chunk(i);
        else b.chunk(i - chunks_a);
    }
#endif
}

// 32 columns and eight ranges of the parts a workgroup: a range's parts are added in order, then the ranges in order.
// (128 parts of 16384 columns, 8 MB from the caches: 5.3 us.)
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
int check_forward(const char *who, int m, int n, int k, const T *a, int lda, const T *b, int ldb, const T *bias, int act,
                  const T *residual, int ldr, const T *preact, int ldp, const T *c, int ldc) {
    if (m < 0 || n < 0 || k < 0) return fail(SWC_HIP_EINVAL, "%s: negative dimension", who);
    if (!known_act(act)) return fail(SWC_HIP_EINVAL, "%s: unknown activation %d", who, act);
    if (m == 0 || n == 0) return SWC_HIP_OK;
    if (!c || (k && (!a || !b))) return fail(SWC_HIP_EINVAL, "%s: null pointer", who);
    if ((k && (lda < k || ldb < n)) || ldc < n || (residual && ldr < n) || (preact && ldp < n))
        return fail(SWC_HIP_EINVAL, "%s: leading dimension smaller than row length", who);
    const bool c_in = c == a || c == b || c == bias;
    if (c_in || (preact && (preact == a || preact == b || preact == bias || preact == c || preact == residual)))
        return fail(SWC_HIP_EINVAL, "%s: an output is also an input or another output", who);
    if (residual == c && ldr != ldc && m > 1) return fail(SWC_HIP_EINVAL, "%s: the residual is C in rows of another length", who);
    if (lda > kMaxLd<T> || ldb > kMaxLd<T> || n > kMaxLd<T>)
        return fail(SWC_HIP_EUNSUPPORTED, "%s: leading dimension beyond %ld", who, kMaxLd<T>);
    if (m > kMaxRows) return fail(SWC_HIP_EUNSUPPORTED, "%s: more than %d rows", who, kMaxRows);
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
    if (int rc = check_forward(who, m, n, k, a, lda_, b, ldb_, bias, act, residual, ldr, preact, ldp, c, ldc)) return rc;
    if (!ready()) return fail(SWC_HIP_ENOTINIT, "%s: swc_hip_init has not been called", who);
    if (m == 0 || n == 0) return SWC_HIP_OK;
    if (k == 0) return launch_finish<T>(act, nullptr, 0, bias, residual, ldr, preact, ldp, c, ldc, m, n);
    if (takes_stream(m, k, b, ldb_)) return launch_stream(act, a, lda_, b, ldb_, bias, residual, ldr, preact, ldp, c, ldc, m, n, k);
    if (m <= kFewRows<T>) return launch_few<T>(act, a, lda_, b, ldb_, bias, residual, ldr, preact, ldp, c, ldc, m, n, k);
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
    const Shape<T> s{a, b, lda, ldb, m, n, k, 0, 1, nullptr};
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
    const long na = a.chunks(), nb = b.chunks();
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
    if (!ready() || m <= (bf ? kFewRows<bf16> : kFewRows<float>) || n <= 0 || k <= 0) return 0;
    return bf ? space<bf16>(nullptr, plan_product<bf16>(m, n, k), m, n, k, true, true).bytes
              : space<float>(nullptr, plan_product<float>(m, n, k), m, n, k, true, true).bytes;
}

} // extern "C"
