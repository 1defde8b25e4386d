// The softmax loss of a fully connected layer over a large vocabulary, without its logits in memory
// (matrixFCSoftmaxWithLoss_f/_bf), and its gradients, next to matrixSoftmaxWithLoss_f (train.hip).
//
//     z = A B + bias,  lse_r = log sum_j exp z_rj,  loss_r = lse_r - z[r, sel_r]
//     dz_rj = g_r (exp(z_rj - lse_r) - [j = sel_r]),  dA = dz B^T,  dB = A^T dz,  dbias = column sums of dz
//
// Forward: the product's accumulators never leave the registers; a wavefront reduces its 64 (32) columns of each row to a
// maximum and a sum of exponentials, 8 bytes per row and block, which a second kernel joins — sums relative to different
// maxima m_i join as sum_i s_i exp(m_i - max).  Gradients: piece by piece of the vocabulary the logits are computed
// again, become dz in the epilogue (in the matrices' type, in the workspace) and feed the two products; dA is summed
// over the pieces in fp32, each range of the contraction in a buffer of its own, and joined in a fixed order at the end:
// no atomics, the same bits every time.  8 mnk flops for loss and gradients instead of 6 with the logits kept: 8192 x
// 128256 x 4096 bf16 25.4-26 ms, 1340 TFLOP/s of them; 1999 x 50257 x 1024 with 30 % of the rows left out 790 us.
//
// Rows left out (their class outside the vocabulary) are dropped first: the rows that count are gathered into a dense
// copy of A, so the products skip the others' work and nothing in them can reach a sum (0 * NaN is NaN).  Their number
// is known on the device only; the kernels read it there.
#include "product.hpp"

using namespace swc_hip;
using namespace swc_hip::product;

namespace {

// The rows that count, in order, with what the gradients need of each.
struct Rows {
    int *index;    // dense row -> row
    int *place;    // row -> dense row, -1 if left out
    int *sel;      // class of a dense row
    int *count;
    float *lse, *grad;   // of a dense row (gradients only)
};
// What the rows come with: lse and row_grad (may be null) are read for the gradients, row_loss and lse_out of the rows left
// out are set to 0 for the forward call.
struct RowsFrom {
    const int *selected;
    int m, n;
    const float *lse, *row_grad;
    float *row_loss, *lse_out;
};
// a matrix whose rows left out become zeros (null: none)
template <class T> struct Cleared {
    T *out;
    long ld;
    int cols;
};
__device__ __forceinline__ void take_row(const RowsFrom &from, const Rows &to, int r, bool in, int at, int sel) {
    to.place[r] = in ? at : -1;
    if (in) {
        to.index[at] = r, to.sel[at] = sel;
        if (from.lse) to.lse[at] = from.lse[r], to.grad[at] = from.row_grad ? from.row_grad[r] : 1.f;
    } else if (from.row_loss) {
        from.row_loss[r] = 0.f, from.lse_out[r] = 0.f;
    }
}

// Many rows: one workgroup numbers them (8192: 12 us, a chain of eight steps), then copy_dense (8192 x 4096 bf16, 134 MB, 24
// us, 5.7 TB/s).
constexpr int kPickThreads = 1024;
__global__ __launch_bounds__(kPickThreads) void pick_rows(RowsFrom from, Rows to) {
    __shared__ int waves[kPickThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int base = 0;
    for (int r0 = 0; r0 < from.m; r0 += kPickThreads) {
        const int r = r0 + threadIdx.x;
        const int sel = r < from.m ? from.selected[r] : -1;
        const bool in = sel >= 0 && sel < from.n;
        const unsigned long long mask = __ballot(in);
        if (lane == 0) waves[wave] = __popcll(mask);
        __syncthreads();
        int before = base, all = base;
        for (int w = 0; w < kPickThreads / 64; ++w) {
            before += w < wave ? waves[w] : 0;
            all += waves[w];
        }
        if (r < from.m) take_row(from, to, r, in, before + __popcll(mask & ((1ull << lane) - 1)), sel);
        base = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) *to.count = base;
}
template <class T>
__global__ __launch_bounds__(256) void copy_dense(const T *a, long lda, int k, T *dense, long ld, Rows rows) {
#if __HIP_DEVICE_COMPILE__
    const int count = *rows.count;
    const long j = ((long)blockIdx.x * 256 + threadIdx.x) * kChunk<T>;
    if (j >= ld) return;
    for (int r = blockIdx.y; r < count; r += gridDim.y)
        *reinterpret_cast<v4u *>(dense + r * ld + j) = chunk_at(a + rows.index[r] * lda + j, k - j);
#endif
}
// Few rows: a workgroup per row counts the rows before its own and copies it; workgroups behind them copy B onto the 16-byte
// grid where it has to be.  One launch instead of three, and dA's rows may go straight to their places (see direct): 1999 rows
// of 1024 8 us, with 1024 x 50257 of B beside them 37 us.  The counting grows with the square of the rows: bf16, k = 1024, n =
// 256, forward and dA together, this way / the other: 2048 rows 39 / 47 us, 4096 59 / 62, 8192 122 / 89.
constexpr int kCountRows = 4096;
template <class T>
__global__ __launch_bounds__(256) void count_and_copy(RowsFrom from, Rows to, const T *a, long lda, int k, T *dense, long ld,
                                                      Cleared<T> cleared, Copy<T> b, long chunks) {
#if __HIP_DEVICE_COMPILE__
    __shared__ int sums[2][4];
    if ((int)blockIdx.x >= from.m) {
        const long step = (long)(gridDim.x - from.m) * 256;
        for (long i = (long)(blockIdx.x - from.m) * 256 + threadIdx.x; i < chunks; i += step) b.chunk(i);
        return;
    }
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0, all = 0;
    for (int r0 = 0; r0 < from.m; r0 += 256) {
        const int r = r0 + threadIdx.x;
        const int sel = r < from.m ? from.selected[r] : -1;
        const bool in = sel >= 0 && sel < from.n;
        all += __popcll(__ballot(in));
        before += __popcll(__ballot(in && r < row));
    }
    if (lane == 0) sums[0][wave] = before, sums[1][wave] = all;
    __syncthreads();
    const int at = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
    const int sel = from.selected[row];
    const bool in = sel >= 0 && sel < from.n;
    if (threadIdx.x == 0) {
        take_row(from, to, row, in, at, sel);
        if (row == 0) *to.count = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
    }
    if (!in) {
        if (cleared.out)
            for (int j = threadIdx.x; j < cleared.cols; j += 256) cleared.out[row * cleared.ld + j] = T(0);
        return;
    }
    for (long j = threadIdx.x * kChunk<T>; j < ld; j += 256 * kChunk<T>)
        *reinterpret_cast<v4u *>(dense + at * ld + j) = chunk_at(a + row * lda + j, k - j);
#endif
}
// The dense rows, and b's copy; cleared: only with up to kCountRows rows.
template <class T>
int gather_rows(const RowsFrom &from, const Rows &to, const T *a, long lda, int k, T *dense, const Cleared<T> &cleared, const Copy<T> &b) {
    const long ld = row_length<T>(k);
    if (from.m <= kCountRows) {
        const long chunks = b.chunks();
        count_and_copy<T><<<from.m + (chunks ? grid_of(chunks) : 0), 256, 0, stream()>>>(from, to, a, lda, k, dense, ld, cleared, b, chunks);
    } else {
        if (int rc = copy_operands<T>({}, b)) return rc;
        pick_rows<<<1, kPickThreads, 0, stream()>>>(from, to);
        SWC_LAUNCH_CHECK();
        copy_dense<T><<<dim3(ceil_div(ld / kChunk<T>, 256), from.m < 32768 ? from.m : 32768), 256, 0, stream()>>>(a, lda, k, dense, ld, to);
    }
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

// bf16: the exponential instruction (relative error |x| 2^-24 and a little); fp32: the library function.  (Its factor and the
// maximum are not fused into one operation: of values near the type's lowest the product overflows.)
template <class T> __device__ __forceinline__ float exponential(float x) { return kIsBf16<T> ? fast_exp(x) : expf(x); }

// ---------------------------------------------------------------- forward
// Bound by the products where the contraction is long (8192 x 128256 x 4096: 6.6 ms, 1300 TFLOP/s), else by the vector
// units: some five operations and an exponential a logit (7381 x 112020 x 132: 592 us, 1.4e12 logits a second).
template <class T> struct RowStats {
    static constexpr bool kHeavy = true, kThinToo = true;
    float2 *part;     // [row][block]: maximum, sum of exp(z - maximum)
    int blocks;
    float *picked;    // [row]: z of the row's class
    const int *sel;
    const T *bias;
    int first;        // the product's first column
    RowStats from(int j) const { return {part + j / 64, blocks, picked, sel, bias ? bias + j : nullptr, first + j}; }   // (64: Big's)
#if __HIP_DEVICE_COMPILE__
    template <class P, bool WHOLE, int TM, int TN>
    __device__ __forceinline__ void reduce(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane) const {
        const int l32 = lane & 31, h = lane >> 5;
        ColumnData<T, P> b;
        if (bias) b.template load<WHOLE>(bias, col0, n, h);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + P::row(tm, l32);
            const int want = (row < m ? sel[row] : -1) - first - col0;
            float z[P::kValues];
            float top = -__builtin_inff();
#pragma unroll
            for (int u = 0; u < P::kValues; ++u) {
                float x = P::value(acc[tm], u);
                if (bias) x += b.value(u);
                if (!WHOLE && col0 + P::column(u, h) >= n) x = -__builtin_inff();
                z[u] = x;
                top = fmaxf(top, x);
            }
            if (__any(want >= 0 && want < 32 * TN)) {   // a row of these 32 has its class here
#pragma unroll
                for (int u = 0; u < P::kValues; ++u)
                    if (P::column(u, h) == want) picked[row] = z[u];
            }
            top = fmaxf(top, __shfl_xor(top, 32));
            const float from = top == -__builtin_inff() ? 0.f : top;   // a block of impossible classes only
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < P::kValues; ++u) sum += exponential<T>(z[u] - from);
            sum += __shfl_xor(sum, 32);
            if (h == 0 && row < m) part[(size_t)row * blocks + col0 / (32 * TN)] = make_float2(top, sum);
        }
    }
    template <class P, int TM, int TN>
    __device__ __forceinline__ void finish(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane, int) const {
        if (col0 >= n) return;
        if (col0 + 32 * TN <= n) reduce<P, true>(acc, row0, col0, m, n, lane);
        else reduce<P, false>(acc, row0, col0, m, n, lane);
    }
#endif
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off);
    return x;
}

// A wavefront joins a dense row's blocks -> the row's loss: their maxima first, then the sums relative to the largest.
// Bound by memory and its start (8192 rows of 2004 blocks, 131 MB, 45 us; 64 rows and their mean in one launch 6 us).
__device__ __forceinline__ float join_row(int row, int lane, const float2 *part, int blocks, const float *picked, const Rows &rows,
                                          float *row_loss, float *lse) {
    const float2 *p = part + (size_t)row * blocks;
    const float2 first = lane < blocks ? p[lane] : make_float2(-__builtin_inff(), 0.f);
    const float z = picked[row];
    const int r = rows.index[row];
    float top = first.x;
    for (int b = lane + 64; b < blocks; b += 64) top = fmaxf(top, p[b].x);
    top = wave_max(top);
    const float from = top == -__builtin_inff() ? 0.f : top;
    float sum = first.y * expf(first.x - from);
    for (int b = lane + 64; b < blocks; b += 64) sum += p[b].y * expf(p[b].x - from);
    sum = wave_sum(sum);
    const float l = from + logf(sum), loss = l - z;
    if (lane == 0) {
        lse[r] = l;
        row_loss[r] = loss;
    }
    return loss;
}
__global__ __launch_bounds__(256) void join_rows(const float2 *part, int blocks, const float *picked, Rows rows, float *row_loss,
                                                 float *lse) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row < *rows.count) join_row(row, threadIdx.x & 63, part, blocks, picked, rows, row_loss, lse);
}

// *loss = mean over the dense rows, summed in double in a fixed order; JOIN: joins the rows first, sixteen at a time.
template <bool JOIN>
__global__ __launch_bounds__(1024) void mean_loss(const float2 *part, int blocks, const float *picked, Rows rows, float *row_loss,
                                                  float *lse, float *loss) {
    __shared__ double sums[1024];
    const int count = *rows.count;
    double s = 0;
    if (JOIN) {
        const int lane = threadIdx.x & 63;
        for (int i = threadIdx.x >> 6; i < count; i += 16) {
            const float l = join_row(i, lane, part, blocks, picked, rows, row_loss, lse);
            if (lane == 0) s += l;
        }
    } else {
        for (int i = threadIdx.x; i < count; i += 1024) s += row_loss[rows.index[i]];
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    for (int off = 512; off > 0; off >>= 1) {
        if (threadIdx.x < off) sums[threadIdx.x] += sums[threadIdx.x + off];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = count ? (float)(sums[0] / count) : 0.f;
}

// Whether joining and mean take one launch: up to sixteen rows, which go at once, and up to 64 whose blocks are one to a lane.
// (k = 64, one launch / two: 16 x 1000 10.1 / 11.4 us, 16 x 100000 33.8 / 35.0, 32 x 1000 11.1 / 11.4, 64 x 1000 13.1 / 11.4 and
// a launch's time on the host, 32 x 10000 14.9 / 13.1, 64 x 100000 102 / 37.)
bool joins_in_mean(int m, int blocks) { return m <= 16 || (m <= 64 && blocks <= 64); }

// ---------------------------------------------------------------- gradients
// dz of a piece of the vocabulary, zeros in the columns that pad it to whole 16 bytes.  It is held in the matrices' type, which
// is what the products behind it multiply, and the column sums are of the values so held: a lane has rows of its own, and sums
// down the columns before the rounding would take an exchange across 32 lanes for each of its columns.  Off the exact dbias by
// 0.0012-0.0022 of its norm, where its last rounding alone makes 0.0012-0.0017 (40 to 8192 rows, logits flat and sharp).
// Bound by the product (8192 x 16384 x 4096 bf16 862 us, 1276 TFLOP/s), where the contraction is short by writing dz (5981 x
// 17920 x 64: 214 MB, 75 us).
template <class T> struct StoreDz {
    static constexpr bool kHeavy = true, kThinToo = true;
    T *dz;
    long ld;
    int width;       // columns of dz from the product's first one on
    int first;       // class of that column
    const int *sel;
    const float *lse, *grad;
    const T *bias;   // from that class on
    StoreDz from(int j) const { return {dz + j, ld, width - j, first + j, sel, lse, grad, bias ? bias + j : nullptr}; }
#if __HIP_DEVICE_COMPILE__
    template <class P, bool WHOLE, int TM, int TN>
    __device__ __forceinline__ void store(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane) const {
        const int l32 = lane & 31, h = lane >> 5;
        ColumnData<T, P> b;
        if (bias) b.template load<WHOLE>(bias, col0, n, h);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + P::row(tm, l32);
            const bool ok = WHOLE || row < m;
            const int want = (ok ? sel[row] : -1) - first - col0;
            const float l = ok ? lse[row] : 0.f, g = ok ? grad[row] : 0.f;
            float x[P::kValues];
#pragma unroll
            for (int u = 0; u < P::kValues; ++u) {
                float z = P::value(acc[tm], u);
                if (bias) z += b.value(u);
                x[u] = exponential<T>(z - l);
            }
            if (__any(ok && want >= 0 && want < 32 * TN)) {   // a row of these 32 has its class here
#pragma unroll
                for (int u = 0; u < P::kValues; ++u)
                    if (P::column(u, h) == want) x[u] -= 1.f;
            }
#pragma unroll
            for (int u = 0; u < P::kValues; ++u) {
                x[u] *= g;
                if (!WHOLE && col0 + P::column(u, h) >= n) x[u] = 0.f;
            }
            store_row<P, WHOLE>(dz + row * ld, ok, col0, width, h, x);
        }
    }
    template <class P, int TM, int TN>
    __device__ __forceinline__ void finish(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane, int) const {
        if (row0 + 32 * TM <= m && col0 + 32 * TN <= n)
            store<P, true>(acc, row0, col0, m, n, lane);
        else store<P, false>(acc, row0, col0, m, n, lane);
    }
#endif
};

// out[r] = sum of `parts` buffers' dense row of r, zeros for a row left out; four columns a thread where cols allow.  Bound by
// memory (1999 x 1024 of 8 parts, 50 MB of the rows that count, 12 us).
template <class T, bool VEC>
__global__ __launch_bounds__(256) void spread_rows(T *out, long ld, const float *part, int parts, long stride, int m, int cols,
                                                   const int *place) {
    constexpr int kPer = VEC ? 4 : 1;
    const int j = (blockIdx.x * 256 + threadIdx.x) * kPer;
    if (j >= cols) return;
    for (int r = blockIdx.y; r < m; r += gridDim.y) {
        const int at = place[r];
        float s[kPer] = {};
        if (at >= 0)
#pragma unroll 4
            for (int p = 0; p < parts; ++p) {
                const float *q = part + p * stride + (size_t)at * cols + j;
                if constexpr (VEC) {
                    const float4 d = *reinterpret_cast<const float4 *>(q);
                    s[0] += d.x, s[1] += d.y, s[2] += d.z, s[3] += d.w;
                } else {
                    s[0] += *q;
                }
            }
#pragma unroll
        for (int e = 0; e < kPer; ++e) store_any(out + r * ld + j + e, s[e]);
    }
}
template <class T>
int launch_spread(T *out, long ld, const float *part, int parts, long stride, int m, int cols, const int *place) {
    const bool vec = cols % 4 == 0;
    const dim3 grid(ceil_div(vec ? cols / 4 : cols, 256), m < 32768 ? m : 32768);
    if (vec) spread_rows<T, true><<<grid, 256, 0, stream()>>>(out, ld, part, parts, stride, m, cols, place);
    else spread_rows<T, false><<<grid, 256, 0, stream()>>>(out, ld, part, parts, stride, m, cols, place);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

// Few rows: a piece's column sums at once, 32 columns and eight ranges of the rows a workgroup.  One launch instead of two (dz
// and its sums with k = 64, this way / by blocks of rows below: 256 x 1000 10.4 / 11.8 us, 256 x 50000 31.4 / 30.3, 512 x 1000
// 12.6 / 12.2, 512 x 50000 48 / 41).
constexpr int kFewSums = 256;
template <class T> __global__ __launch_bounds__(256) void few_column_sums(const T *dz, long ld, int cols, Rows rows, T *out) {
    __shared__ float sums[8][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, j = blockIdx.x * 32 + tx;
    const int count = *rows.count, each = (count + 7) / 8, r0 = ty * each, r1 = r0 + each < count ? r0 + each : count;
    float s = 0.f;
    if (j < cols)
#pragma unroll 8
        for (int r = r0; r < r1; ++r) s += load_any(dz + r * ld + j);
    sums[ty][tx] = s;
    __syncthreads();
    if (ty || j >= cols) return;
#pragma unroll
    for (int y = 1; y < 8; ++y) s += sums[y][tx];
    store_any(out + j, s);
}
// Sums over blocks of kSumRows dense rows of a piece's columns, four a lane (one: 22 us).  Bound by memory: 3886 rows of 8227
// bf16, 64 MB from the caches, 13 us.
constexpr int kSumRows = 64;
template <class T>
__global__ __launch_bounds__(256) void column_sums(const T *dz, long ld, int cols, Rows rows, float *sums) {
#if __HIP_DEVICE_COMPILE__
    __shared__ float part[4][256];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, j = (blockIdx.x * 64 + tx) * 4;
    const int count = *rows.count, r0 = blockIdx.y * kSumRows;
    const int r1 = r0 + kSumRows < count ? r0 + kSumRows : count;
    float s[4] = {};
    if (j < cols)   // (dz's rows end on a multiple of four)
#pragma unroll 8
        for (int r = r0 + ty; r < r1; r += 4) {
            float x[4];
            load4(dz + r * ld + j, 4, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += x[e];
        }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[ty][tx * 4 + e] = s[e];
    __syncthreads();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= cols) return;
    float all = 0.f;
#pragma unroll
    for (int y = 0; y < 4; ++y) all += part[y][threadIdx.x];
    sums[(size_t)blockIdx.y * cols + col] = all;
#endif
}

// ---------------------------------------------------------------- the calls
template <class T>
int check(const char *who, int m, int n, int k, const T *a, int lda, const T *b, int ldb, const int *selected) {
    if (m < 0 || n < 0 || k < 0) return fail(SWC_HIP_EINVAL, "%s: negative dimension", who);
    if (m && !selected) return fail(SWC_HIP_EINVAL, "%s: selected is null", who);
    if (m && n && k && (!a || !b)) return fail(SWC_HIP_EINVAL, "%s: null pointer", who);
    if (m && n && k && (lda < k || ldb < n)) return fail(SWC_HIP_EINVAL, "%s: leading dimension smaller than row length", who);
    if (lda > kMaxLd<T> || ldb > kMaxLd<T> || k > kMaxLd<T> || n > kMaxLd<T>)
        return fail(SWC_HIP_EUNSUPPORTED, "%s: leading dimension beyond %ld", who, kMaxLd<T>);
    if (m && n && k == 0) return fail(SWC_HIP_EINVAL, "%s: k is 0", who);
    constexpr int kMost = 65535 * kSumRows;
    if (m > kMost) return fail(SWC_HIP_EUNSUPPORTED, "%s: more than %d rows", who, kMost);
    return SWC_HIP_OK;
}

Rows take_rows(Carver &c, int m, bool gradients) {
    Rows r{};
    r.index = c.take<int>(m);
    r.place = c.take<int>(m);
    r.sel = c.take<int>(m);
    r.count = c.take<int>(1);
    if (gradients) r.lse = c.take<float>(m), r.grad = c.take<float>(m);
    return r;
}

// Whole rows of the contraction: the epilogues of this file need finished sums.
template <class T> Plan whole_plan(int m, int n, int k) { return plan_product<T>(m, n, k, true); }
// blocks of columns that RowStats writes for a row
int block_columns(Kind kind) { return kind == kThin || kind == kSmall ? 32 : 64; }
int row_blocks(const Plan &p, int n) {
    if (p.first > 0 && p.first < n) return p.first / block_columns(p.kind) + ceil_div(n - p.first, block_columns(p.rest));
    return ceil_div(n, block_columns(p.kind));
}
static_assert(Big::TN == 2 && Mid::TN == 2 && Low::TN == 2 && Small::TN == 1 && Thin::TN == 1, "columns of a wavefront");

template <class T> struct ForwardSpace {
    Rows rows;
    T *a, *b;
    float2 *part;
    float *picked;
    size_t bytes;
};
template <class T> ForwardSpace<T> forward_space(char *base, const Plan &p, int m, int n, int k, bool pack_b) {
    Carver c{base};
    ForwardSpace<T> s{};
    s.rows = take_rows(c, m, false);
    s.a = c.take<T>((size_t)m * row_length<T>(k));
    s.b = pack_b ? c.take<T>((size_t)k * row_length<T>(n)) : nullptr;
    s.part = c.take<float2>((size_t)m * row_blocks(p, n));
    s.picked = c.take<float>(m);
    s.bytes = c.used;
    return s;
}

// Classes per piece of the gradients' dz: 256 MiB of it, about what the last-level cache holds.  Fewer make dA's sums travel
// more often (4799 x 25615 x 768: 774 us whole, 874 in pieces of 128 MiB, 981 of 64), more leave the cache (7477 x 56867 x 64:
// 786 us, 924 in pieces of 512 MiB; 8192 x 128256 x 4096 gains 1.5 %).
int piece_columns(int m, int n, size_t bytes) {
    size_t p = ((size_t)256 << 20) / bytes / m / 256 * 256;
    if (p < 256) p = 256;
    return p < (size_t)n ? (int)p : n;
}

template <class T> struct GradSpace {
    Rows rows;
    T *a, *b, *dz;
    float *da, *part, *sums;
    int piece;
    Plan pa, pb;
    bool direct, pair;   // dA's rows go straight to their places; both products of the one piece in one launch
    size_t bytes;
};
template <class T> GradSpace<T> grad_space(char *base, int m, int n, int k, bool pack_b, bool da, bool db, bool dbias) {
    Carver c{base};
    GradSpace<T> s{};
    s.piece = piece_columns(m, n, sizeof(T));
    s.pa = plan_product<T>(m, k, s.piece);
    s.pb = plan_product<T>(k, s.piece, m);
    s.direct = s.piece == n && s.pa.splits == 1 && m <= kCountRows;
    s.pair = da && db && s.piece == n && (s.direct || s.pa.splits > 1) && pairs(s.pa, s.pb, m, n, k);
    s.rows = take_rows(c, m, true);
    s.a = c.take<T>((size_t)m * row_length<T>(k));
    s.b = pack_b ? c.take<T>((size_t)k * row_length<T>(n)) : nullptr;
    s.dz = c.take<T>((size_t)m * row_length<T>(s.piece));
    s.da = da && !s.direct ? c.take<float>((size_t)s.pa.splits * m * k) : nullptr;
    s.part = db && s.pb.splits > 1 ? c.take<float>((size_t)s.pb.splits * k * s.piece) : nullptr;
    s.sums = dbias && m > kFewSums ? c.take<float>((size_t)((m + kSumRows - 1) / kSumRows) * s.piece) : nullptr;
    s.bytes = c.used;
    return s;
}

template <class T>
int forward(const char *who, int m, int n, int k, const T *a, int lda, const T *b, int ldb_, const T *bias, const int *selected,
            float *row_loss, float *lse, float *loss) {
    if (int rc = check(who, m, n, k, a, lda, b, ldb_, selected)) return rc;
    if (!loss || (m && (!row_loss || !lse))) return fail(SWC_HIP_EINVAL, "%s: null output", who);
    if (m && (row_loss == lse || row_loss == loss || lse == loss)) return fail(SWC_HIP_EINVAL, "%s: two outputs are the same", who);
    if (!ready()) return fail(SWC_HIP_ENOTINIT, "%s: swc_hip_init has not been called", who);
    if (m == 0 || n == 0) {   // no rows, or no classes: every row is left out
        if (int rc = zero_rows(row_loss, m, m ? 1 : 0, m)) return rc;
        if (int rc = zero_rows(lse, m, m ? 1 : 0, m)) return rc;
        return zero_rows(loss, 1, 1, 1);
    }
    long ldb = ldb_;
    const Plan p = whole_plan<T>(m, n, k);
    const bool pack_b = !aligned_rows(b, ldb);
    char *base = static_cast<char *>(workspace(forward_space<T>(nullptr, p, m, n, k, pack_b).bytes, who));
    if (!base) return fail_code();
    const ForwardSpace<T> w = forward_space<T>(base, p, m, n, k, pack_b);
    if (int rc = gather_rows<T>({selected, m, n, nullptr, nullptr, row_loss, lse}, w.rows, a, lda, k, w.a, {},
                                {w.b, b, row_length<T>(n), ldb, k, n}))
        return rc;
    if (pack_b) b = w.b, ldb = row_length<T>(n);
    const int blocks = row_blocks(p, n);
    const Shape<T> s{w.a, b, row_length<T>(k), ldb, m, n, k, 0, 1, w.rows.count};
    if (int rc = run_product<kAlongK, kAcross>(p, s, RowStats<T>{w.part, blocks, w.picked, w.rows.sel, bias, 0}, who)) return rc;
    if (joins_in_mean(m, blocks)) {
        mean_loss<true><<<1, 1024, 0, stream()>>>(w.part, blocks, w.picked, w.rows, row_loss, lse, loss);
    } else {
        join_rows<<<ceil_div(m, 4), 256, 0, stream()>>>(w.part, blocks, w.picked, w.rows, row_loss, lse);
        SWC_LAUNCH_CHECK();
        mean_loss<false><<<1, 1024, 0, stream()>>>(nullptr, 0, nullptr, w.rows, row_loss, lse, loss);
    }
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

template <class T>
int gradients(const char *who, int m, int n, int k, const T *a, int lda, const T *b, int ldb_, const T *bias, const int *selected,
              const float *lse, const float *row_grad, T *da, int ldda, T *db, int lddb, T *dbias) {
    if (int rc = check(who, m, n, k, a, lda, b, ldb_, selected)) return rc;
    if (m && !lse) return fail(SWC_HIP_EINVAL, "%s: lse is null", who);
    if ((da && ldda < k) || (db && lddb < n)) return fail(SWC_HIP_EINVAL, "%s: leading dimension smaller than row length", who);
    const void *in[3] = {a, b, bias};
    for (const void *p : in)
        if (p && (p == da || p == db || p == dbias)) return fail(SWC_HIP_EINVAL, "%s: an output is also an input", who);
    if ((da && (da == db || da == dbias)) || (db && db == dbias)) return fail(SWC_HIP_EINVAL, "%s: two outputs are the same", who);
    if (!ready()) return fail(SWC_HIP_ENOTINIT, "%s: swc_hip_init has not been called", who);
    if (!da && !db && !dbias) return SWC_HIP_OK;
    if (m == 0 || n == 0) {
        if (int rc = zero_rows(da, ldda, m, k)) return rc;
        if (int rc = zero_rows(db, lddb, k, n)) return rc;
        return zero_rows(dbias, n, 1, n);
    }
    long ldb = ldb_;
    const bool pack_b = !aligned_rows(b, ldb) || (da && n % kChunk<T>);
    char *base = static_cast<char *>(workspace(grad_space<T>(nullptr, m, n, k, pack_b, da, db, dbias).bytes, who));
    if (!base) return fail_code();
    const GradSpace<T> w = grad_space<T>(base, m, n, k, pack_b, da, db, dbias);
    const long ldw = row_length<T>(k);
    if (int rc = gather_rows<T>({selected, m, n, lse, row_grad, nullptr, nullptr}, w.rows, a, lda, k, w.a,
                                {w.direct ? da : nullptr, ldda, k}, {w.b, b, row_length<T>(n), ldb, k, n}))
        return rc;
    if (pack_b) b = w.b, ldb = row_length<T>(n);
    for (int first = 0; first < n; first += w.piece) {
        const int cols = n - first < w.piece ? n - first : w.piece;
        const long ld = row_length<T>(cols);
        const Shape<T> z{w.a, b + first, ldw, ldb, m, cols, k, 0, 1, w.rows.count};
        const StoreDz<T> ep{w.dz, ld, (int)ld, first, w.rows.sel, w.rows.lse, w.rows.grad, bias ? bias + first : nullptr};
        if (int rc = run_product<kAlongK, kAcross>(whole_plan<T>(m, cols, k), z, ep, who)) return rc;
        const Shape<T> sa{w.dz, b + first, ld, ldb, m, k, cols, 0, 1, w.rows.count}, sb{w.a, w.dz, ldw, ld, k, cols, m, 0, 1, w.rows.count};
        const Store<T, true> out_a{w.direct ? da : nullptr, ldda, w.rows.index};
        if (w.pair) {
            // (dA's partial sums stay dense: they are joined by the spreading kernel below)
            if (int rc = grad_pair<T>(w.pa, sa, out_a, w.da, w.pb, sb, {db, lddb}, w.part)) return rc;
        } else {
            const StorePartial sums{w.da, (long)m * k, k, first > 0};
            if (da)
                if (int rc = w.direct ? run_product<kAlongK, kAlongK>(w.pa, sa, out_a, who) : run_product<kAlongK, kAlongK>(w.pa, sa, sums, who))
                    return rc;
            if (db)
                if (int rc = grad_product<kAcross, kAcross, T>(who, w.pb, sb, {db + first, lddb}, w.part)) return rc;
        }
        if (dbias && m <= kFewSums) {
            few_column_sums<T><<<ceil_div(cols, 32), 256, 0, stream()>>>(w.dz, ld, cols, w.rows, dbias + first);
            SWC_LAUNCH_CHECK();
        } else if (dbias) {
            const int parts = (m + kSumRows - 1) / kSumRows;
            column_sums<T><<<dim3(ceil_div(cols, 256), parts), 256, 0, stream()>>>(w.dz, ld, cols, w.rows, w.sums);
            SWC_LAUNCH_CHECK();
            if (int rc = sum_parts<T>(dbias + first, w.sums, parts, cols)) return rc;
        }
    }
    return da && !w.direct ? launch_spread(da, ldda, w.da, w.pa.splits, (long)m * k, m, k, w.rows.place) : (int)SWC_HIP_OK;
}

} // namespace

extern "C" {

int swc_hip_matrixFCSoftmaxWithLoss_f(int m, int n, int k, const float *a, int lda, const float *b, int ldb, const float *bias,
                                      const int *selected, float *rowLoss, float *lse, float *loss) {
    return forward<float>("swc_hip_matrixFCSoftmaxWithLoss_f", m, n, k, a, lda, b, ldb, bias, selected, rowLoss, lse, loss);
}

int swc_hip_matrixFCSoftmaxWithLoss_bf(int m, int n, int k, const swc_hip_bf16 *a, int lda, const swc_hip_bf16 *b, int ldb,
                                       const swc_hip_bf16 *bias, const int *selected, float *rowLoss, float *lse, float *loss) {
    return forward<bf16>("swc_hip_matrixFCSoftmaxWithLoss_bf", m, n, k, a, lda, b, ldb, bias, selected, rowLoss, lse, loss);
}

size_t swc_hip_matrixFCSoftmaxWithLoss_workspace_bytes(int m, int n, int k, int bf) {
    if (!ready() || m <= 0 || n <= 0 || k <= 0) return 0;
    return bf ? forward_space<bf16>(nullptr, whole_plan<bf16>(m, n, k), m, n, k, true).bytes
              : forward_space<float>(nullptr, whole_plan<float>(m, n, k), m, n, k, true).bytes;
}

int swc_hip_matrixFCSoftmaxWithLossGrad_f(int m, int n, int k, const float *a, int lda, const float *b, int ldb, const float *bias,
                                          const int *selected, const float *lse, const float *rowGrad, float *aGrad, int ldag,
                                          float *bGrad, int ldbg, float *biasGrad) {
    return gradients<float>("swc_hip_matrixFCSoftmaxWithLossGrad_f", m, n, k, a, lda, b, ldb, bias, selected, lse, rowGrad, aGrad,
                            ldag, bGrad, ldbg, biasGrad);
}

int swc_hip_matrixFCSoftmaxWithLossGrad_bf(int m, int n, int k, const swc_hip_bf16 *a, int lda, const swc_hip_bf16 *b, int ldb,
                                           const swc_hip_bf16 *bias, const int *selected, const float *lse, const float *rowGrad,
                                           swc_hip_bf16 *aGrad, int ldag, swc_hip_bf16 *bGrad, int ldbg, swc_hip_bf16 *biasGrad) {
    return gradients<bf16>("swc_hip_matrixFCSoftmaxWithLossGrad_bf", m, n, k, a, lda, b, ldb, bias, selected, lse, rowGrad, aGrad,
                           ldag, bGrad, ldbg, biasGrad);
}

size_t swc_hip_matrixFCSoftmaxWithLossGrad_workspace_bytes(int m, int n, int k, int bf) {
    if (!ready() || m <= 0 || n <= 0 || k <= 0) return 0;
    return bf ? grad_space<bf16>(nullptr, m, n, k, true, true, true, true).bytes
              : grad_space<float>(nullptr, m, n, k, true, true, true, true).bytes;
}

} // extern "C"
