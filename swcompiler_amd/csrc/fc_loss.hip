// The softmax loss of a fully connected layer over a large vocabulary, without its logits in memory
// (matrixFCSoftmaxWithLoss_f/_bf), and its gradients, next to matrixSoftmaxWithLoss_f (train.hip).
//
//     z = A B + bias,  lse_r = log sum_j exp z_rj,  loss_r = lse_r - z[r, sel_r]
//     dz_rj = g_r (exp(z_rj - lse_r) - [j = sel_r]),  dA = dz B^T,  dB = A^T dz,  dbias = column sums of dz
//
// bf16 forward: the product's accumulators never leave the registers; a wavefront reduces its 64 (32) columns of each
// row to a maximum and a sum of exponentials, 8 bytes per row and block, which a second kernel joins — sums relative to
// different maxima m_i join as sum_i s_i exp(m_i - max).  Gradients: piece by piece of the vocabulary the logits are
// computed again, become dz in the epilogue (bf16, in the workspace) and feed the two products; dA is summed over the
// pieces in fp32, each range of the contraction in a buffer of its own, and joined in a fixed order at the end: no
// atomics, the same bits every time.  8 mnk flops for loss and gradients instead of 6 with the logits kept.
//
// Rows left out (their class outside the vocabulary) are dropped first: the rows that count are gathered into a dense
// copy of A, so the products skip the others' work and nothing in them can reach a sum (0 * NaN is NaN).  Their number
// is known on the device only; the kernels read it there.
#include "product_bf16.hpp"

using namespace swc_hip;
using namespace swc_hip::mfma16;

namespace {

// The rows that count, in order.
struct Rows {
    int *index;    // dense row -> row
    int *place;    // row -> dense row, -1 if left out
    int *sel;      // class of a dense row
    int *count;
};

constexpr int kPickThreads = 1024;
__global__ __launch_bounds__(kPickThreads) void pick_rows(const int *selected, int m, int n, Rows out, float *row_loss, float *lse) {
    __shared__ int waves[kPickThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int base = 0;
    for (int r0 = 0; r0 < m; r0 += kPickThreads) {
        const int r = r0 + threadIdx.x;
        const int sel = r < m ? selected[r] : -1;
        const bool in = sel >= 0 && sel < n;
        const unsigned long long mask = __ballot(in);
        if (lane == 0) waves[wave] = __popcll(mask);
        __syncthreads();
        int before = base, all = base;
        for (int w = 0; w < kPickThreads / 64; ++w) {
            before += w < wave ? waves[w] : 0;
            all += waves[w];
        }
        if (r < m) {
            const int at = before + __popcll(mask & ((1ull << lane) - 1));
            out.place[r] = in ? at : -1;
            if (in) out.index[at] = r, out.sel[at] = sel;
            else if (row_loss) row_loss[r] = 0.f, lse[r] = 0.f;
        }
        base = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) *out.count = base;
}

// ---------------------------------------------------------------- bf16 forward
struct RowStats {
    static constexpr bool kHeavy = true, kThinToo = true;
    float2 *part;     // [row][block]: maximum, sum of exp(z - maximum)
    int blocks;
    float *picked;    // [row]: z of the row's class
    const int *sel;
    const uint16_t *bias;
#if __HIP_DEVICE_COMPILE__
    template <bool WHOLE, int TM, int TN>
    __device__ __forceinline__ void reduce(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane) const {
        const int l32 = lane & 31, h = lane >> 5;
        v2u b[TN][4];
        if (bias)
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) load_columns<WHOLE>(bias, col0 + tn * 32, n, h, b[tn]);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + tm * 32 + l32;
            const int want = (row < m ? sel[row] : -1) - col0;
            float z[TN * 16];
            float top = -__builtin_inff();
#pragma unroll
            for (int tn = 0; tn < TN; ++tn)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    float x = acc[tm][tn][v];
                    if (bias) x += column_value(b[tn], v);
                    if (!WHOLE && col0 + tn * 32 + 8 * (v / 4) + 4 * h + v % 4 >= n) x = -__builtin_inff();
                    z[tn * 16 + v] = x;
                    top = fmaxf(top, x);
                }
            if (__any(want >= 0 && want < 32 * TN)) {   // a row of these 32 has its class here
#pragma unroll
                for (int v = 0; v < TN * 16; ++v)
                    if (v / 16 * 32 + 8 * (v % 16 / 4) + 4 * h + v % 4 == want) picked[row] = z[v];
            }
            top = fmaxf(top, __shfl_xor(top, 32));
            const float from = top == -__builtin_inff() ? 0.f : top;   // a block of impossible classes only
            float sum = 0.f;
#pragma unroll
            for (int v = 0; v < TN * 16; ++v) sum += fast_exp(z[v] - from);
            sum += __shfl_xor(sum, 32);
            if (h == 0 && row < m) part[(size_t)row * blocks + col0 / (32 * TN)] = make_float2(top, sum);
        }
    }
    template <int TM, int TN>
    __device__ __forceinline__ void operator()(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane,
                                               int) const {
        if (col0 >= n) return;
        if (col0 + 32 * TN <= n && (reinterpret_cast<uintptr_t>(bias) & 7) == 0) reduce<true>(acc, row0, col0, m, n, lane);
        else reduce<false>(acc, row0, col0, m, n, lane);
    }
#endif
};

__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float top = fmaxf(a.x, b.x), from = top == -__builtin_inff() ? 0.f : top;
    return make_float2(top, a.y * expf(a.x - from) + b.y * expf(b.x - from));
}

// One wavefront per dense row joins its blocks.
__global__ __launch_bounds__(256) void join_rows(const float2 *part, int blocks, const float *picked, Rows rows, float *row_loss,
                                                 float *lse) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= *rows.count) return;
    const float2 *p = part + (size_t)row * blocks;
    float2 s = make_float2(-__builtin_inff(), 0.f);
    for (int b = lane; b < blocks; b += 64) s = join(s, p[b]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s = join(s, make_float2(__shfl_xor(s.x, off), __shfl_xor(s.y, off)));
    if (lane == 0) {
        const float l = (s.x == -__builtin_inff() ? 0.f : s.x) + logf(s.y);
        const int r = rows.index[row];
        lse[r] = l;
        row_loss[r] = l - picked[row];
    }
}

// *loss = mean over the dense rows, summed in double in a fixed order
__global__ __launch_bounds__(1024) void mean_loss(const float *row_loss, Rows rows, float *loss) {
    __shared__ double sums[1024];
    const int count = *rows.count;
    double s = 0;
    for (int i = threadIdx.x; i < count; i += 1024) s += row_loss[rows.index[i]];
    sums[threadIdx.x] = s;
    __syncthreads();
    for (int off = 512; off > 0; off >>= 1) {
        if (threadIdx.x < off) sums[threadIdx.x] += sums[threadIdx.x + off];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = count ? (float)(sums[0] / count) : 0.f;
}

// ---------------------------------------------------------------- bf16 gradients
// dz of a piece of the vocabulary whose first class is `first`, zeros in the columns that pad it to whole 16 bytes
struct StoreDz {
    static constexpr bool kHeavy = true, kThinToo = true;
    uint16_t *dz;
    long ld;
    int first;
    const int *sel;
    const float *lse, *grad;
    const uint16_t *bias;   // of the piece
#if __HIP_DEVICE_COMPILE__
    template <bool WHOLE, int TM, int TN>
    __device__ __forceinline__ void store(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane) const {
        const int l32 = lane & 31, h = lane >> 5;
        v2u b[TN][4];
        if (bias)
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) load_columns<WHOLE>(bias, col0 + tn * 32, n, h, b[tn]);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + tm * 32 + l32;
            const bool ok = WHOLE || row < m;
            const int want = (ok ? sel[row] : -1) - first - col0;
            const float l = ok ? lse[row] : 0.f, g = ok ? grad[row] : 0.f;
            const bool here = __any(ok && want >= 0 && want < 32 * TN);   // a row of these 32 has its class here
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) {
                float x[16];
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    float z = acc[tm][tn][v];
                    if (bias) z += column_value(b[tn], v);
                    x[v] = fast_exp(z - l);
                }
                if (here) {
#pragma unroll
                    for (int v = 0; v < 16; ++v)
                        if (tn * 32 + 8 * (v / 4) + 4 * h + v % 4 == want) x[v] -= 1.f;
                }
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    x[v] *= g;
                    if (!WHOLE && col0 + tn * 32 + 8 * (v / 4) + 4 * h + v % 4 >= n) x[v] = 0.f;
                }
                store_block<WHOLE>(dz + row * ld, ok, col0 + tn * 32, (int)ld, true, h, x);
            }
        }
    }
    template <int TM, int TN>
    __device__ __forceinline__ void operator()(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane,
                                               int) const {
        if (row0 + 32 * TM <= m && col0 + 32 * TN <= n && (reinterpret_cast<uintptr_t>(bias) & 7) == 0)
            store<true>(acc, row0, col0, m, n, lane);
        else store<false>(acc, row0, col0, m, n, lane);
    }
#endif
};

// lse and the upstream gradient of the dense rows
__global__ __launch_bounds__(256) void gather_row_values(const float *lse, const float *grad, Rows rows, float *lse_out, float *grad_out) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= *rows.count) return;
    const int r = rows.index[i];
    lse_out[i] = lse[r];
    grad_out[i] = grad ? grad[r] : 1.f;
}

// out[r] = sum of `parts` buffers' dense row of r, zeros for a row left out; four columns a thread where cols allow
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

// sums over blocks of kSumRows dense rows of a piece's columns
constexpr int kSumRows = 64;
template <class T>
__global__ __launch_bounds__(256) void column_sums(const T *dz, long ld, int cols, Rows rows, float *sums) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= cols) return;
    const int count = *rows.count, r0 = blockIdx.y * kSumRows;
    const int r1 = r0 + kSumRows < count ? r0 + kSumRows : count;
    float s = 0.f;
    for (int r = r0; r < r1; ++r) s += load_any(dz + r * ld + j);
    sums[(size_t)blockIdx.y * cols + j] = s;
}

__global__ __launch_bounds__(256) void to_bf16_rows(uint16_t *out, long ld, const float *part, int parts, long stride, int rows, int cols) {
    for (int r = blockIdx.y; r < rows; r += gridDim.y)
        for (int j = blockIdx.x * 256 + threadIdx.x; j < cols; j += gridDim.x * 256) {
            float s = 0.f;
            for (int p = 0; p < parts; ++p) s += part[p * stride + (size_t)r * cols + j];
            store_any(out + r * ld + j, s);
        }
}

// ---------------------------------------------------------------- fp32: pieces of logits in the workspace
// A workgroup per dense row folds a piece into the row's running maximum and sum.
__global__ __launch_bounds__(256) void fold_piece(const float *z, long ld, int cols, int first, Rows rows, float2 *run, float *picked) {
    __shared__ float2 waves[4];
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (row >= *rows.count) return;
    const float *p = z + row * ld;
    float top = -__builtin_inff();
    for (int j = threadIdx.x; j < cols; j += 256) top = fmaxf(top, p[j]);
    const float from = top == -__builtin_inff() ? 0.f : top;
    float sum = 0.f;
    for (int j = threadIdx.x; j < cols; j += 256) sum += expf(p[j] - from);
    float2 s = make_float2(top, sum);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s = join(s, make_float2(__shfl_xor(s.x, off), __shfl_xor(s.y, off)));
    if (lane == 0) waves[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = join(join(waves[0], waves[1]), join(waves[2], waves[3]));
        run[row] = first ? join(run[row], s) : s;
        const int want = rows.sel[row] - first;
        if (want >= 0 && want < cols) picked[row] = p[want];
    }
}

// z -> dz in place, zeros for the rows behind the dense ones
__global__ __launch_bounds__(256) void dz_piece(float *z, long ld, int cols, int first, int m, Rows rows, const float *lse, const float *grad) {
    const int count = *rows.count;
    for (int r = blockIdx.y; r < m; r += gridDim.y) {
        const bool in = r < count;
        const float l = in ? lse[r] : 0.f, g = in ? grad[r] : 0.f;
        const int want = in ? rows.sel[r] - first : -1;
        for (int j = blockIdx.x * 256 + threadIdx.x; j < cols; j += gridDim.x * 256) {
            const float p = in ? expf(z[r * ld + j] - l) : 0.f;
            z[r * ld + j] = in ? g * (j == want ? p - 1.f : p) : 0.f;
        }
    }
}

__global__ __launch_bounds__(256) void add_into(float *acc, const float *x, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) acc[i] += x[i];
}

dim3 rows_grid(int rows, long cols) {
    const unsigned x = ceil_div(cols, 256);
    return dim3(x > 64 ? 64 : x, rows < 32768 ? rows : 32768);
}

template <class T>
int check(const char *who, int m, int n, int k, const T *a, int lda, const T *b, int ldb, const int *selected) {
    if (m < 0 || n < 0 || k < 0) return fail(SWC_HIP_EINVAL, "%s: negative dimension", who);
    if (m && !selected) return fail(SWC_HIP_EINVAL, "%s: selected is null", who);
    if (m && n && k && (!a || !b)) return fail(SWC_HIP_EINVAL, "%s: null pointer", who);
    if (m && n && k && (lda < k || ldb < n)) return fail(SWC_HIP_EINVAL, "%s: leading dimension smaller than row length", who);
    if (sizeof(T) == 2 && (lda > kMaxLd || ldb > kMaxLd || round8(k) > kMaxLd || round8(n) > kMaxLd))
        return fail(SWC_HIP_EUNSUPPORTED, "%s: leading dimension beyond %ld", who, kMaxLd);
    return SWC_HIP_OK;
}

Rows take_rows(Carver &c, int m) {
    Rows r;
    r.index = c.take<int>(m);
    r.place = c.take<int>(m);
    r.sel = c.take<int>(m);
    r.count = c.take<int>(1);
    return r;
}

// Whole rows of the contraction: the epilogues of this file need finished sums.
Plan whole_plan(int m, int n, int k) { return plan_product(m, n, k, true); }
int block_columns(const Plan &p) { return p.kind == kThin || p.kind == kSmall ? 32 : 64; }
static_assert(Big::TN == 2 && Mid::TN == 2 && Low::TN == 2 && Small::TN == 1 && Thin::TN == 1, "columns of a wavefront");

// ---------------------------------------------------------------- spaces
struct ForwardSpace {
    Rows rows;
    uint16_t *a, *b;
    float2 *part;
    float *picked;
    size_t bytes;
};
ForwardSpace forward_space(char *base, const Plan &p, int m, int n, int k, bool pack_b) {
    Carver c{base};
    ForwardSpace s{};
    s.rows = take_rows(c, m);
    s.a = c.take<uint16_t>((size_t)m * round8(k));
    s.b = pack_b ? c.take<uint16_t>((size_t)k * round8(n)) : nullptr;
    s.part = c.take<float2>((size_t)m * ((n + block_columns(p) - 1) / block_columns(p)));
    s.picked = c.take<float>(m);
    s.bytes = c.used;
    return s;
}

// Classes per piece of the gradients' dz: 256 MiB of it.
int piece_columns(int m, int n, size_t bytes) {
    size_t p = ((size_t)256 << 20) / bytes / m / 256 * 256;
    if (p < 256) p = 256;
    return p < (size_t)n ? (int)p : n;
}

struct GradSpace {
    Rows rows;
    uint16_t *a, *b, *dz;
    float *lse, *grad, *da, *part, *sums;
    int piece;
    Plan pa, pb;
    size_t bytes;
};
GradSpace grad_space(char *base, int m, int n, int k, bool pack_b, bool da, bool db, bool dbias) {
    Carver c{base};
    GradSpace s{};
    s.piece = piece_columns(m, n, 2);
    s.pa = plan_product(m, k, s.piece);
    s.pb = plan_product(k, s.piece, m);
    s.rows = take_rows(c, m);
    s.a = c.take<uint16_t>((size_t)m * round8(k));
    s.b = pack_b ? c.take<uint16_t>((size_t)k * round8(n)) : nullptr;
    s.dz = c.take<uint16_t>((size_t)m * round8(s.piece));
    s.lse = c.take<float>(m);
    s.grad = c.take<float>(m);
    s.da = da ? c.take<float>((size_t)s.pa.splits * m * k) : nullptr;
    s.part = db && s.pb.splits > 1 ? c.take<float>((size_t)s.pb.splits * k * s.piece) : nullptr;
    s.sums = dbias ? c.take<float>((size_t)((m + kSumRows - 1) / kSumRows) * s.piece) : nullptr;
    s.bytes = c.used;
    return s;
}

struct SpaceF {
    Rows rows;
    float *a, *z, *picked, *lse, *grad, *da, *tmp, *at, *bt, *part, *sums;
    float2 *run;
    int piece;
    size_t partials, bytes;
};
SpaceF space_f(char *base, int m, int n, int k, bool gradients, bool da, bool db, bool dbias) {
    Carver c{base};
    SpaceF s{};
    s.piece = piece_columns(m, n, 4);
    const int tail = n % s.piece;   // the last piece has a plan of its own
    s.partials = 0;
    for (int p : {s.piece, tail}) {
        if (!p) continue;
        const size_t need[3] = {swc_hip_gemm_workspace_bytes(m, p, k), da ? swc_hip_gemm_workspace_bytes(m, k, p) : 0,
                                db ? swc_hip_gemm_workspace_bytes(k, p, m) : 0};
        for (size_t x : need) s.partials = x > s.partials ? x : s.partials;
    }
    s.rows = take_rows(c, m);
    s.a = c.take<float>((size_t)m * k);
    s.z = c.take<float>((size_t)m * s.piece);
    s.part = c.take<float>(s.partials / sizeof(float) + 1);
    if (!gradients) {
        s.run = c.take<float2>(m);
        s.picked = c.take<float>(m);
    } else {
        s.lse = c.take<float>(m);
        s.grad = c.take<float>(m);
        s.da = da ? c.take<float>((size_t)m * k) : nullptr;
        s.tmp = da && s.piece < n ? c.take<float>((size_t)m * k) : nullptr;
        s.bt = da ? c.take<float>((size_t)k * s.piece) : nullptr;
        s.at = db ? c.take<float>((size_t)m * k) : nullptr;
        s.sums = dbias ? c.take<float>((size_t)((m + kSumRows - 1) / kSumRows) * s.piece) : nullptr;
    }
    s.bytes = c.used;
    return s;
}

// ---------------------------------------------------------------- the calls
int forward_bf16(const char *who, int m, int n, int k, const uint16_t *a, long lda, const uint16_t *b, long ldb,
                 const uint16_t *bias, const int *selected, float *row_loss, float *lse, float *loss) {
    const Plan p = whole_plan(m, n, k);
    const bool pack_b = !aligned_rows(b, ldb);
    char *base = static_cast<char *>(workspace(forward_space(nullptr, p, m, n, k, pack_b).bytes, who));
    if (!base) return fail_code();
    const ForwardSpace w = forward_space(base, p, m, n, k, pack_b);
    pick_rows<<<1, kPickThreads, 0, stream()>>>(selected, m, n, w.rows, row_loss, lse);
    SWC_LAUNCH_CHECK();
    if (int rc = copy_rows_bf16(w.a, round8(k), a, lda, m, k, w.rows.index, w.rows.count)) return rc;
    if (pack_b) {
        if (int rc = copy_rows_bf16(w.b, round8(n), b, ldb, k, n, nullptr, nullptr)) return rc;
        b = w.b, ldb = round8(n);
    }
    const int blocks = (n + block_columns(p) - 1) / block_columns(p);
    const Shape s{w.a, b, round8(k), ldb, m, n, k, 0, w.rows.count};
    if (int rc = run_product<kAlongK, kAcross>(p, s, RowStats{w.part, blocks, w.picked, w.rows.sel, bias}, who)) return rc;
    join_rows<<<ceil_div(m, 4), 256, 0, stream()>>>(w.part, blocks, w.picked, w.rows, row_loss, lse);
    SWC_LAUNCH_CHECK();
    mean_loss<<<1, 1024, 0, stream()>>>(row_loss, w.rows, loss);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

__global__ __launch_bounds__(256) void finish_run(const float2 *run, const float *picked, Rows rows, float *row_loss, float *lse) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= *rows.count) return;
    const float2 s = run[i];
    const float l = (s.x == -__builtin_inff() ? 0.f : s.x) + logf(s.y);
    lse[rows.index[i]] = l;
    row_loss[rows.index[i]] = l - picked[i];
}

int forward_f32(const char *who, int m, int n, int k, const float *a, int lda, const float *b, int ldb, const float *bias,
                const int *selected, float *row_loss, float *lse, float *loss) {
    char *base = static_cast<char *>(workspace(space_f(nullptr, m, n, k, false, false, false, false).bytes, who));
    if (!base) return fail_code();
    const SpaceF w = space_f(base, m, n, k, false, false, false, false);
    pick_rows<<<1, kPickThreads, 0, stream()>>>(selected, m, n, w.rows, row_loss, lse);
    SWC_LAUNCH_CHECK();
    if (int rc = copy_rows_f32(w.a, k, a, lda, m, k, w.rows.index, w.rows.count)) return rc;
    for (int first = 0; first < n; first += w.piece) {
        const int cols = n - first < w.piece ? n - first : w.piece;
        if (int rc = gemm_f32(who, m, cols, k, w.a, k, b + first, ldb, bias ? bias + first : nullptr, w.z, cols, 0, w.part, w.partials))
            return rc;
        fold_piece<<<m, 256, 0, stream()>>>(w.z, cols, cols, first, w.rows, w.run, w.picked);
        SWC_LAUNCH_CHECK();
    }
    finish_run<<<ceil_div(m, 256), 256, 0, stream()>>>(w.run, w.picked, w.rows, row_loss, lse);
    SWC_LAUNCH_CHECK();
    mean_loss<<<1, 1024, 0, stream()>>>(row_loss, w.rows, loss);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

int grad_bf16(const char *who, int m, int n, int k, const uint16_t *a, long lda, const uint16_t *b, long ldb, const uint16_t *bias,
              const int *selected, const float *lse, const float *row_grad, uint16_t *da, long ldda, uint16_t *db, long lddb,
              uint16_t *dbias) {
    const bool pack_b = !aligned_rows(b, ldb) || (da && n % 8);
    char *base = static_cast<char *>(workspace(grad_space(nullptr, m, n, k, pack_b, da, db, dbias).bytes, who));
    if (!base) return fail_code();
    const GradSpace w = grad_space(base, m, n, k, pack_b, da, db, dbias);
    pick_rows<<<1, kPickThreads, 0, stream()>>>(selected, m, n, w.rows, nullptr, nullptr);
    SWC_LAUNCH_CHECK();
    gather_row_values<<<ceil_div(m, 256), 256, 0, stream()>>>(lse, row_grad, w.rows, w.lse, w.grad);
    SWC_LAUNCH_CHECK();
    if (int rc = copy_rows_bf16(w.a, round8(k), a, lda, m, k, w.rows.index, w.rows.count)) return rc;
    if (pack_b) {
        if (int rc = copy_rows_bf16(w.b, round8(n), b, ldb, k, n, nullptr, nullptr)) return rc;
        b = w.b, ldb = round8(n);
    }
    for (int first = 0; first < n; first += w.piece) {
        const int cols = n - first < w.piece ? n - first : w.piece;
        const long ld = round8(cols);
        const Shape z{w.a, b + first, round8(k), ldb, m, cols, k, 0, w.rows.count};
        const StoreDz ep{w.dz, ld, first, w.rows.sel, w.lse, w.grad, bias ? bias + first : nullptr};
        if (int rc = run_product<kAlongK, kAcross>(whole_plan(m, cols, k), z, ep, who)) return rc;
        if (da) {
            const Shape s{w.dz, b + first, ld, ldb, m, k, cols, 0, w.rows.count};
            if (int rc = run_product<kAlongK, kAlongK>(w.pa, s, StorePartial{w.da, (long)m * k, k, first > 0}, who)) return rc;
        }
        if (db) {
            const Shape s{w.a, w.dz, round8(k), ld, k, cols, m, 0, w.rows.count};
            if (w.pb.splits == 1) {
                const StoreBf16 out{db + first, lddb, aligned_rows(db + first, lddb)};
                if (int rc = run_product<kAcross, kAcross>(w.pb, s, out, who)) return rc;
            } else {
                if (int rc = run_product<kAcross, kAcross>(w.pb, s, StorePartial{w.part, (long)k * cols, cols, false}, who)) return rc;
                to_bf16_rows<<<rows_grid(k, cols), 256, 0, stream()>>>(db + first, lddb, w.part, w.pb.splits, (long)k * cols, k, cols);
                SWC_LAUNCH_CHECK();
            }
        }
        if (dbias) {
            const int parts = (m + kSumRows - 1) / kSumRows;
            column_sums<uint16_t><<<dim3(ceil_div(cols, 256), parts), 256, 0, stream()>>>(w.dz, ld, cols, w.rows, w.sums);
            SWC_LAUNCH_CHECK();
            if (int rc = sum_parts(dbias + first, nullptr, w.sums, parts, cols)) return rc;
        }
    }
    return da ? launch_spread(da, ldda, w.da, w.pa.splits, (long)m * k, m, k, w.rows.place) : (int)SWC_HIP_OK;
}

int grad_f32(const char *who, int m, int n, int k, const float *a, int lda, const float *b, int ldb, const float *bias,
             const int *selected, const float *lse, const float *row_grad, float *da, int ldda, float *db, int lddb, float *dbias) {
    char *base = static_cast<char *>(workspace(space_f(nullptr, m, n, k, true, da, db, dbias).bytes, who));
    if (!base) return fail_code();
    const SpaceF w = space_f(base, m, n, k, true, da, db, dbias);
    pick_rows<<<1, kPickThreads, 0, stream()>>>(selected, m, n, w.rows, nullptr, nullptr);
    SWC_LAUNCH_CHECK();
    gather_row_values<<<ceil_div(m, 256), 256, 0, stream()>>>(lse, row_grad, w.rows, w.lse, w.grad);
    SWC_LAUNCH_CHECK();
    if (int rc = copy_rows_f32(w.a, k, a, lda, m, k, w.rows.index, w.rows.count)) return rc;
    if (db)
        if (int rc = swc_hip_matrixTrans_f(m, k, w.a, k, w.at, m)) return rc;
    for (int first = 0; first < n; first += w.piece) {
        const int cols = n - first < w.piece ? n - first : w.piece;
        if (int rc = gemm_f32(who, m, cols, k, w.a, k, b + first, ldb, bias ? bias + first : nullptr, w.z, cols, 0, w.part, w.partials))
            return rc;
        dz_piece<<<rows_grid(m, cols), 256, 0, stream()>>>(w.z, cols, cols, first, m, w.rows, w.lse, w.grad);
        SWC_LAUNCH_CHECK();
        if (da) {
            float *to = first ? w.tmp : w.da;
            if (int rc = swc_hip_matrixTrans_f(k, cols, b + first, ldb, w.bt, k)) return rc;
            if (int rc = gemm_f32(who, m, k, cols, w.z, cols, w.bt, k, nullptr, to, k, 0, w.part, w.partials)) return rc;
            if (first) {
                const unsigned blocks = ceil_div((size_t)m * k, 256);
                add_into<<<blocks > 8192 ? 8192 : blocks, 256, 0, stream()>>>(w.da, w.tmp, (size_t)m * k);
                SWC_LAUNCH_CHECK();
            }
        }
        if (db)
            if (int rc = gemm_f32(who, k, cols, m, w.at, m, w.z, cols, nullptr, db + first, lddb, 0, w.part, w.partials)) return rc;
        if (dbias) {
            const int parts = (m + kSumRows - 1) / kSumRows;
            column_sums<float><<<dim3(ceil_div(cols, 256), parts), 256, 0, stream()>>>(w.z, cols, cols, w.rows, w.sums);
            SWC_LAUNCH_CHECK();
            if (int rc = sum_parts(nullptr, dbias + first, w.sums, parts, cols)) return rc;
        }
    }
    return da ? launch_spread(da, ldda, w.da, 1, 0, m, k, w.rows.place) : (int)SWC_HIP_OK;
}

constexpr int kMaxRows = 65535 * kSumRows;

template <class T, class F>
int forward(const char *who, F call, int m, int n, int k, const T *a, int lda, const T *b, int ldb, const T *bias,
            const int *selected, float *row_loss, float *lse, float *loss) {
    if (int rc = check(who, m, n, k, a, lda, b, ldb, selected)) return rc;
    if (!loss || (m && (!row_loss || !lse))) return fail(SWC_HIP_EINVAL, "%s: null output", who);
    if (m && k == 0 && n) return fail(SWC_HIP_EINVAL, "%s: k is 0", who);
    if (m > kMaxRows) return fail(SWC_HIP_EUNSUPPORTED, "%s: more than %d rows", who, kMaxRows);
    if (!ready()) return fail(SWC_HIP_ENOTINIT, "%s: swc_hip_init has not been called", who);
    if (m == 0) return swc_hip_fill_f(loss, 0.f, 1);
    if (n == 0) {   // no classes: every row is left out
        if (int rc = swc_hip_fill_f(row_loss, 0.f, m)) return rc;
        if (int rc = swc_hip_fill_f(lse, 0.f, m)) return rc;
        return swc_hip_fill_f(loss, 0.f, 1);
    }
    return call(who, m, n, k, a, lda, b, ldb, bias, selected, row_loss, lse, loss);
}

template <class T, class F>
int gradients(const char *who, F call, int m, int n, int k, const T *a, int lda, const T *b, int ldb, const T *bias,
              const int *selected, const float *lse, const float *row_grad, T *da, int ldda, T *db, int lddb, T *dbias) {
    if (int rc = check(who, m, n, k, a, lda, b, ldb, selected)) return rc;
    if (m && !lse) return fail(SWC_HIP_EINVAL, "%s: lse is null", who);
    if ((da && ldda < k) || (db && lddb < n)) return fail(SWC_HIP_EINVAL, "%s: leading dimension smaller than row length", who);
    const void *in[3] = {a, b, bias};
    for (const void *p : in)
        if (p && (p == da || p == db || p == dbias)) return fail(SWC_HIP_EINVAL, "%s: an output is also an input", who);
    if (m && n && k == 0) return fail(SWC_HIP_EINVAL, "%s: k is 0", who);
    if (m > kMaxRows) return fail(SWC_HIP_EUNSUPPORTED, "%s: more than %d rows", who, kMaxRows);
    if (!ready()) return fail(SWC_HIP_ENOTINIT, "%s: swc_hip_init has not been called", who);
    if (!da && !db && !dbias) return SWC_HIP_OK;
    if (m == 0 || n == 0) {
        if (int rc = zero_rows(da, ldda, m, k)) return rc;
        if (int rc = zero_rows(db, lddb, k, n)) return rc;
        return zero_rows(dbias, n, 1, n);
    }
    return call(who, m, n, k, a, lda, b, ldb, bias, selected, lse, row_grad, da, ldda, db, lddb, dbias);
}

} // namespace

extern "C" {

int swc_hip_matrixFCSoftmaxWithLoss_f(int m, int n, int k, const float *a, int lda, const float *b, int ldb, const float *bias,
                                      const int *selected, float *rowLoss, float *lse, float *loss) {
    return forward("swc_hip_matrixFCSoftmaxWithLoss_f", forward_f32, m, n, k, a, lda, b, ldb, bias, selected, rowLoss, lse, loss);
}

int swc_hip_matrixFCSoftmaxWithLoss_bf(int m, int n, int k, const swc_hip_bf16 *a, int lda, const swc_hip_bf16 *b, int ldb,
                                       const swc_hip_bf16 *bias, const int *selected, float *rowLoss, float *lse, float *loss) {
    return forward("swc_hip_matrixFCSoftmaxWithLoss_bf", forward_bf16, m, n, k, a, lda, b, ldb, bias, selected, rowLoss, lse, loss);
}

size_t swc_hip_matrixFCSoftmaxWithLoss_workspace_bytes(int m, int n, int k, int bf) {
    if (!ready() || m <= 0 || n <= 0 || k <= 0) return 0;
    return bf ? forward_space(nullptr, whole_plan(m, n, k), m, n, k, true).bytes : space_f(nullptr, m, n, k, false, false, false, false).bytes;
}

int swc_hip_matrixFCSoftmaxWithLossGrad_f(int m, int n, int k, const float *a, int lda, const float *b, int ldb, const float *bias,
                                          const int *selected, const float *lse, const float *rowGrad, float *aGrad, int ldag,
                                          float *bGrad, int ldbg, float *biasGrad) {
    return gradients("swc_hip_matrixFCSoftmaxWithLossGrad_f", grad_f32, m, n, k, a, lda, b, ldb, bias, selected, lse, rowGrad, aGrad,
                     ldag, bGrad, ldbg, biasGrad);
}

int swc_hip_matrixFCSoftmaxWithLossGrad_bf(int m, int n, int k, const swc_hip_bf16 *a, int lda, const swc_hip_bf16 *b, int ldb,
                                           const swc_hip_bf16 *bias, const int *selected, const float *lse, const float *rowGrad,
                                           swc_hip_bf16 *aGrad, int ldag, swc_hip_bf16 *bGrad, int ldbg, swc_hip_bf16 *biasGrad) {
    return gradients("swc_hip_matrixFCSoftmaxWithLossGrad_bf", grad_bf16, m, n, k, a, lda, b, ldb, bias, selected, lse, rowGrad,
                     aGrad, ldag, bGrad, ldbg, biasGrad);
}

size_t swc_hip_matrixFCSoftmaxWithLossGrad_workspace_bytes(int m, int n, int k, int bf) {
    if (!ready() || m <= 0 || n <= 0 || k <= 0) return 0;
    return bf ? grad_space(nullptr, m, n, k, true, true, true, true).bytes : space_f(nullptr, m, n, k, true, true, true, true).bytes;
}

} // extern "C"
