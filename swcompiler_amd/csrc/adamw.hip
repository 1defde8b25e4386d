// The AdamW step over many tensors at once, with its states in 32 bits or in 8 (adamw_f/_bf, adamw8_f/_bf), next to
// sgd_f (train.hip).
//
// Bound by memory: per element w 8 bytes, the gradient 4 or 2, the states 16 or 4, the bfloat16 copy 2 — and some
// twenty fp32 operations.  One launch covers up to kTensors tensors: their pointers travel by value in the kernel
// arguments (nothing to upload, so a recorded graph needs no buffer of its own), and a workgroup finds its tensor by
// comparing its number with each tensor's first, one a lane.
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

using namespace swc_hip;

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = SWC_HIP_ADAMW_BLOCK;   // elements that share a scale: one wavefront, four elements a lane

struct Header {       // what adamwAdvance leaves for the updates
    int steps;
    int pad;
    float c1, c2;     // 1 / (1 - beta^t)
    int rest[4];
};
static_assert(sizeof(Header) == SWC_HIP_ADAMW_STATE_BYTES, "");

struct Step {
    const Header *state;
    const float *lr_factor, *grad_factor;
    float lr, beta1, beta2, rest1, rest2, eps, decay;   // rest: 1 - beta, from doubles
};

// 1 - beta^t = -expm1(t log beta) in double: the difference of a beta near 1 cancels at the first steps.
__global__ void adamw_advance(Header *state, double log1, double log2) {
    const int t = state->steps + 1;
    state->steps = t;
    state->c1 = (float)(-1.0 / expm1(t * log1));
    state->c2 = (float)(-1.0 / expm1(t * log2));
}

struct Tensor {
    float *w;
    const void *dw;
    void *mom, *var;
    uint16_t *copy;
    size_t size;
};
struct Tensor8 : Tensor {
    float *mom_scale, *var_scale;
};
// (the tables fill the 4 KiB that kernel arguments may take)
template <class T, int N> struct Table {
    T t[N];
    unsigned first[N + 1];   // first chunk of each tensor
    int count, number0;      // number0: the first tensor's number in the call
};
constexpr int kTensors = 64, kTensors8 = 48;
static_assert(sizeof(Table<Tensor, kTensors>) + sizeof(Step) <= 4000 && sizeof(Table<Tensor8, kTensors8>) + sizeof(Step) <= 4000, "");

// The last tensor whose first chunk is not behind this one (one without elements shares its first chunk with the next).
template <class T, int N> __device__ __forceinline__ int tensor_of(const Table<T, N> &tab, unsigned chunk) {
    static_assert(N <= 64, "a lane for each");
    const int lane = threadIdx.x & 63;
    const bool before = lane < tab.count && tab.first[lane < N ? lane : N] <= chunk;
    return __popcll(__ballot(before)) - 1;
}

__device__ __forceinline__ float grad_of(const float *p, size_t i) { return p[i]; }
__device__ __forceinline__ float grad_of(const uint16_t *p, size_t i) { return __builtin_bit_cast(float, (unsigned)p[i] << 16); }
__device__ __forceinline__ uint16_t to_bf16(float x) {
#if __HIP_DEVICE_COMPILE__
    return __builtin_bit_cast(uint16_t, (__bf16)x);
#else
    return 0;
#endif
}

struct Scalars {
    float lr, shrink, g, c1, c2;
};
__device__ __forceinline__ Scalars scalars(const Step &s) {
    Scalars r;
    r.lr = s.lr_factor ? s.lr * *s.lr_factor : s.lr;
    r.shrink = 1.f - r.lr * s.decay;
    r.g = s.grad_factor ? *s.grad_factor : 1.f;
    r.c1 = r.lr * s.state->c1;
    r.c2 = s.state->c2;
    return r;
}
// The states' operations are rounded one by one, as sgd_f's are: they are the same bits wherever they are computed, and
// with them the 8-bit codes that a later step starts from.
__device__ __forceinline__ void step_one(float &w, float g, float &mom, float &var, const Scalars &k, const Step &s) {
    {
#pragma clang fp contract(off)
        g = g * k.g;
        mom = mom * s.beta1 + g * s.rest1;
        var = var * s.beta2 + (g * g) * s.rest2;
    }
    w = w * k.shrink - k.c1 * mom / (sqrtf(var * k.c2) + s.eps);
}

// Four consecutive elements, from any address; NT: past the caches (a model's states do not fit them).
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef f4 f4_any __attribute__((aligned(4)));
typedef u2 u2_any __attribute__((aligned(2)));
typedef unsigned u1_any __attribute__((aligned(1)));
template <bool NT, class V, class P> __device__ __forceinline__ V fetch(const P *p) {
    const V *q = reinterpret_cast<const V *>(p);
    return NT ? __builtin_nontemporal_load(q) : *q;
}
template <bool NT, class V, class P, class X> __device__ __forceinline__ void put(P *p, X x) {
    V *q = reinterpret_cast<V *>(p);
    if (NT) __builtin_nontemporal_store((V)x, q);
    else *q = (V)x;
}
template <bool NT> __device__ __forceinline__ void fetch4(const float *p, float (&x)[4]) {
    const f4 d = fetch<NT, f4_any>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = d[e];
}
template <bool NT> __device__ __forceinline__ void fetch4(const uint16_t *p, float (&x)[4]) {
    const u2 d = fetch<NT, u2_any>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __builtin_bit_cast(float, e & 1 ? d[e / 2] & 0xffff0000u : d[e / 2] << 16);
}
template <bool NT> __device__ __forceinline__ void put4(float *p, const float (&x)[4]) { put<NT, f4_any>(p, f4{x[0], x[1], x[2], x[3]}); }
// (the copy is read by the next step's products: it stays in the caches' reach)
__device__ __forceinline__ void put4_bf16(uint16_t *p, const float (&x)[4]) {
    put<false, u2_any>(p, u2{to_bf16(x[0]) | (unsigned)to_bf16(x[1]) << 16, to_bf16(x[2]) | (unsigned)to_bf16(x[3]) << 16});
}

// A chunk is four consecutive elements a thread: a workgroup's work.  (Four chunks a workgroup: 265M parameters 1341 us
// against 1298, its registers halve the wavefronts.)  A launch has at most 2^32 - 1 threads.
constexpr unsigned kChunk = 4 * kThreads;
constexpr unsigned kMaxChunks = 0xffffffffu / kThreads;

// 265M parameters with bf16 gradients and copies, 7.4 GB: 1286-1300 us, 5.7 TB/s.
template <class G, bool NT>
__global__ __launch_bounds__(kThreads) void adamw_tensors(Table<Tensor, kTensors> tab, Step s) {
    const int which = tensor_of(tab, blockIdx.x);
    const Tensor &t = tab.t[which];
    const Scalars k = scalars(s);
    const size_t i0 = (size_t)(blockIdx.x - tab.first[which]) * kChunk + 4 * threadIdx.x;
    float *mom = static_cast<float *>(t.mom), *var = static_cast<float *>(t.var);
    const G *dw = static_cast<const G *>(t.dw);
    if (i0 + 4 <= t.size) {
        float w[4], g[4], m[4], v[4];
        fetch4<NT>(t.w + i0, w), fetch4<NT>(dw + i0, g), fetch4<NT>(mom + i0, m), fetch4<NT>(var + i0, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) step_one(w[e], g[e], m[e], v[e], k, s);
        put4<NT>(t.w + i0, w), put4<NT>(mom + i0, m), put4<NT>(var + i0, v);
        if (t.copy) put4_bf16(t.copy + i0, w);
        return;
    }
    for (size_t i = i0; i < t.size; ++i) {   // the last thread's one to three
        float w = t.w[i], m = mom[i], v = var[i];
        step_one(w, grad_of(dw, i), m, v, k, s);
        t.w[i] = w, mom[i] = m, var[i] = v;
        if (t.copy) t.copy[i] = to_bf16(w);
    }
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}

// A published 32-bit mixing function (C. Wellons, 2018: two multiplications between shifts, its constants found by a search for
// the least bias).  What goes into it keeps elements, tensors and steps apart: a tensor's number times 2^32 over the golden
// ratio, a step's times an odd constant (from A. Appleby's published 32-bit mixer).
__device__ __forceinline__ unsigned random20(unsigned x) {
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    x = (x ^ (x >> 15)) * 0x846CA68Bu;
    return (x ^ (x >> 16)) >> 12;
}

constexpr float kLargest = 448.f;        // of e4m3
constexpr float kPer = 1.f / 448.f;
constexpr float kTiny = 0x1p-100f;       // a block whose largest magnitude is below this is held as zeros
constexpr unsigned kNan8 = 0x7f;

__device__ __forceinline__ float from_e4m3(unsigned byte) {
#if __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
#else
    return 0.f;
#endif
}
// An fp32 quotient of at most 448 to the nearest value, ties to even.
__device__ __forceinline__ unsigned to_e4m3(float y) {
#if __HIP_DEVICE_COMPILE__
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xffu;
#else
    return 0;
#endif
}
// 0 <= y <= 448 up or down by 20 random bits, which side settled in 64 bits: with the exponent E of y (at least that of the
// least normal value) the values of e4m3 are 2^(E-3) apart, y is that times q + fraction, and the code of (E, q) is
// 8 (E + 7) + q - 8 — also where q reaches 16 (the next exponent's first value) and below 8 at the least exponent (the
// subnormal values).  KEPT: a positive y not to zero.
template <bool KEPT> __device__ __forceinline__ unsigned to_e4m3_random(double y, unsigned bits20) {
    const int e = max((int)(__builtin_bit_cast(unsigned long long, y) >> 52) - 1023, -6);
    const double units = __builtin_bit_cast(double, (unsigned long long)(1023 + 3 - e) << 52);   // 2^(3 - E)
    int q = (int)(y * units + (double)bits20 * 0x1p-20);
    if (KEPT && y > 0) q = max(q, 1);
    return (unsigned)(8 * (e + 7) + q - 8);
}

// A wavefront owns a block of 256 elements, a lane four consecutive ones of them (FULL: the block is whole): a block's scale
// is one exchange within the wavefront.  99M parameters with bf16 gradients and copies, 1.6 GB: 339-351 us, 4.6 TB/s: the
// encodings' arithmetic, two divisions in 64 bits a lane among it, stands beside the memory.
// SLOW: the mean up or down at random too (see slow_mean).
template <class G, bool FULL, bool NT, bool SLOW>
__device__ __forceinline__ void adamw8_block(const Tensor8 &t, size_t block, int lane, unsigned number, const Scalars &k, const Step &s) {
    uint8_t *mom8 = static_cast<uint8_t *>(t.mom), *var8 = static_cast<uint8_t *>(t.var);
    const G *dw = static_cast<const G *>(t.dw);
    const float ms = t.mom_scale[block], vs = t.var_scale[block];
    const size_t i0 = block * kBlock + lane * 4;
    float w[4], g[4], m[4], r[4], top = 0.f, peak = 0.f;
    unsigned mc[4], vc[4];
    bool in[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) in[e] = FULL || i0 + e < t.size;
    if constexpr (FULL) {
        fetch4<NT>(t.w + i0, w), fetch4<NT>(dw + i0, g);
        const unsigned a = fetch<NT, u1_any>(mom8 + i0), b = fetch<NT, u1_any>(var8 + i0);
#pragma unroll
        for (int e = 0; e < 4; ++e) mc[e] = (a >> (8 * e)) & 0xffu, vc[e] = (b >> (8 * e)) & 0xffu;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const size_t i = i0 + e;
            w[e] = in[e] ? t.w[i] : 0.f;
            g[e] = in[e] ? grad_of(dw, i) : 0.f;
            mc[e] = in[e] ? mom8[i] : 0u, vc[e] = in[e] ? var8[i] : 0u;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        m[e] = ms * from_e4m3(mc[e]);
        const float root = vs * from_e4m3(vc[e]);
        float v = root * root;
        step_one(w[e], g[e], m[e], v, k, s);
        r[e] = sqrtf(v);
        if (in[e] && fabsf(m[e]) < __builtin_inff()) top = fmaxf(top, fabsf(m[e]));
        if (in[e] && r[e] < __builtin_inff()) peak = fmaxf(peak, r[e]);
    }
    top = wave_max(top), peak = wave_max(peak);
    const float mscale = top > kTiny ? top * kPer : 0.f, vscale = peak > kTiny ? peak * kPer : 0.f;
    const double im = mscale > 0.f ? 1.0 / (double)mscale : 0.0, iv = vscale > 0.f ? 1.0 / (double)vscale : 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        // (the quotients by a reciprocal in 64 bits: the fp32 quotient of mom correctly rounded)
        const unsigned key = (unsigned)(i0 + e) + number;
        if constexpr (SLOW) {
            const double x = fmin(fabs(m[e] * im), (double)kLargest);
            mc[e] = fabsf(m[e]) < __builtin_inff() ? to_e4m3_random<false>(x, random20(~key)) | (m[e] < 0.f ? 0x80u : 0u) : kNan8;
        } else {
            const float x = fminf(fmaxf((float)(m[e] * im), -kLargest), kLargest);
            mc[e] = fabsf(m[e]) < __builtin_inff() ? to_e4m3(x) : kNan8;
        }
        const double y = fmin(r[e] * iv, (double)kLargest);
        vc[e] = r[e] < __builtin_inff() ? to_e4m3_random<true>(y, random20(key)) : kNan8;
    }
    if constexpr (FULL) {
        put4<NT>(t.w + i0, w);
        put<NT, u1_any>(mom8 + i0, mc[0] | mc[1] << 8 | mc[2] << 16 | mc[3] << 24);
        put<NT, u1_any>(var8 + i0, vc[0] | vc[1] << 8 | vc[2] << 16 | vc[3] << 24);
        if (t.copy) put4_bf16(t.copy + i0, w);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const size_t i = i0 + e;
            if (!in[e]) continue;
            t.w[i] = w[e], mom8[i] = (uint8_t)mc[e], var8[i] = (uint8_t)vc[e];
            if (t.copy) t.copy[i] = to_bf16(w[e]);
        }
    }
    if (lane == 0) {
        t.mom_scale[block] = mscale;
        t.var_scale[block] = vscale;
    }
}

template <class G, bool NT, bool SLOW>
__global__ __launch_bounds__(kThreads) void adamw8_tensors(Table<Tensor8, kTensors8> tab, Step s) {
    const int which = tensor_of(tab, blockIdx.x);
    const Tensor8 &t = tab.t[which];
    const Scalars k = scalars(s);
    const size_t block = (size_t)(blockIdx.x - tab.first[which]) * 4 + (threadIdx.x >> 6);
    if (block * kBlock >= t.size) return;   // whole wavefronts leave together
    const unsigned number = (unsigned)(tab.number0 + which) * 0x9E3779B9u + (unsigned)s.state->steps * 0x85EBCA6Bu;
    if ((block + 1) * kBlock <= t.size) adamw8_block<G, true, NT, SLOW>(t, block, threadIdx.x & 63, number, k, s);
    else adamw8_block<G, false, NT, SLOW>(t, block, threadIdx.x & 63, number, k, s);
}

int check(const char *who, int count, const void *const *w, const void *const *dw, const void *const *mom,
          const void *const *var, const void *const *mom_scale, const void *const *var_scale, const size_t *sizes,
          const void *state, bool eight, float lr, double beta1, double beta2, float eps, float decay) {
    if (count < 0) return fail(SWC_HIP_EINVAL, "%s: count is negative", who);
    if (!state) return fail(SWC_HIP_EINVAL, "%s: state is null", who);
    if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1))
        return fail(SWC_HIP_EINVAL, "%s: beta1 and beta2 must lie in [0, 1)", who);
    if (!(eps >= 0.f) || !(lr == lr) || !(decay == decay)) return fail(SWC_HIP_EINVAL, "%s: eps is negative, or a rate is NaN", who);
    if (count && (!w || !dw || !mom || !var || !sizes || (eight && (!mom_scale || !var_scale))))
        return fail(SWC_HIP_EINVAL, "%s: null array of pointers", who);
    for (int i = 0; i < count; ++i)
        if (sizes[i] && (!w[i] || !dw[i] || !mom[i] || !var[i] || (eight && (!mom_scale[i] || !var_scale[i]))))
            return fail(SWC_HIP_EINVAL, "%s: null pointer for tensor %d", who, i);
    for (int i = 0; i < count; ++i)
        if (sizes[i] > (size_t)kMaxChunks * kChunk) return fail(SWC_HIP_EUNSUPPORTED, "%s: tensor %d has %zu elements", who, i, sizes[i]);
    // one parameter given twice (tied weights) would be stepped by two workgroups at a time
    if (count < 2) return SWC_HIP_OK;
    const std::unique_ptr<const void *[]> seen(new (std::nothrow) const void *[count]);
    if (!seen) return fail(SWC_HIP_ERUNTIME, "%s: out of host memory", who);
    int n = 0;
    for (int i = 0; i < count; ++i)
        if (sizes[i]) seen[n++] = w[i];
    std::sort(seen.get(), seen.get() + n);
    if (std::adjacent_find(seen.get(), seen.get() + n) != seen.get() + n) return fail(SWC_HIP_EINVAL, "%s: a tensor is given twice", who);
    return SWC_HIP_OK;
}

// Fills tables of up to N tensors and launches one kernel for each.
template <class T, int N, class Fill, class Launch>
int launch_tables(int count, const size_t *sizes, Fill fill, Launch launch) {
    Table<T, N> tab;
    int next = 0;
    while (next < count) {
        unsigned chunks = 0;
        tab.count = 0;
        tab.number0 = next;
        for (; next < count && tab.count < N; ++next) {
            const size_t need = (sizes[next] + kChunk - 1) / kChunk;   // (at most kMaxChunks: check)
            if (chunks + need > kMaxChunks) break;
            fill(tab.t[tab.count], next);
            tab.first[tab.count++] = chunks;
            chunks += (unsigned)need;
        }
        tab.first[tab.count] = chunks;
        if (!chunks) continue;
        launch(tab, chunks);
        SWC_LAUNCH_CHECK();
    }
    return SWC_HIP_OK;
}

// A step moves a mean by (1 - beta1) |g - mom|.  Rounded to the nearest value, of which two are up to an eighth of the lower
// one apart, it moves at all only where that is half of it: with 1 - beta1 at most a sixteenth not even a mean whose gradient
// has stopped (g = 0) leaves every value, and one far from its gradient stays.  There the mean is rounded at random, which
// keeps its expectation (99M parameters 380 us, 348 to the nearest).
bool slow_mean(double beta1) { return beta1 >= 15. / 16; }

// Whether the weights of a call are large enough to be streamed past the caches.
bool streams(const size_t *sizes, int count, size_t bytes) {
    size_t all = 0;
    for (int i = 0; i < count; ++i) all += sizes[i];
    return all * bytes >= kStreamingBytes;
}

template <class G>
int adamw(const char *who, int count, float *const *w, const G *const *dw, float *const *mom, float *const *var,
          uint16_t *const *copies, const size_t *sizes, const void *state, float lr, double beta1, double beta2, float eps,
          float decay, const float *lr_factor, const float *grad_factor) {
    if (int rc = check(who, count, (const void *const *)w, (const void *const *)dw, (const void *const *)mom,
                       (const void *const *)var, nullptr, nullptr, sizes, state, false, lr, beta1, beta2, eps, decay))
        return rc;
    if (!ready()) return fail(SWC_HIP_ENOTINIT, "%s: swc_hip_init has not been called", who);
    const Step s{static_cast<const Header *>(state), lr_factor, grad_factor, lr, (float)beta1, (float)beta2, (float)(1. - beta1),
                 (float)(1. - beta2), eps, decay};
    return launch_tables<Tensor, kTensors>(
        count, sizes,
        [&](Tensor &t, int i) { t = Tensor{w[i], dw[i], mom[i], var[i], copies ? copies[i] : nullptr, sizes[i]}; },
        [&](const Table<Tensor, kTensors> &tab, unsigned chunks) {
            auto kern = streams(sizes, count, sizeof(float)) ? adamw_tensors<G, true> : adamw_tensors<G, false>;
            kern<<<chunks, kThreads, 0, stream()>>>(tab, s);
        });
}

template <class G>
int adamw8(const char *who, int count, float *const *w, const G *const *dw, uint8_t *const *mom8, float *const *mom_scale,
           uint8_t *const *var8, float *const *var_scale, uint16_t *const *copies, const size_t *sizes, const void *state,
           float lr, double beta1, double beta2, float eps, float decay, const float *lr_factor, const float *grad_factor) {
    if (int rc = check(who, count, (const void *const *)w, (const void *const *)dw, (const void *const *)mom8,
                       (const void *const *)var8, (const void *const *)mom_scale, (const void *const *)var_scale, sizes,
                       state, true, lr, beta1, beta2, eps, decay))
        return rc;
    if (!ready()) return fail(SWC_HIP_ENOTINIT, "%s: swc_hip_init has not been called", who);
    const Step s{static_cast<const Header *>(state), lr_factor, grad_factor, lr, (float)beta1, (float)beta2, (float)(1. - beta1),
                 (float)(1. - beta2), eps, decay};
    return launch_tables<Tensor8, kTensors8>(
        count, sizes,
        [&](Tensor8 &t, int i) {
            t.w = w[i], t.dw = dw[i], t.mom = mom8[i], t.var = var8[i], t.copy = copies ? copies[i] : nullptr;
            t.size = sizes[i], t.mom_scale = mom_scale[i], t.var_scale = var_scale[i];
        },
        [&](const Table<Tensor8, kTensors8> &tab, unsigned chunks) {
            const bool nt = streams(sizes, count, sizeof(float));
            auto kern = slow_mean(beta1) ? (nt ? adamw8_tensors<G, true, true> : adamw8_tensors<G, false, true>)
                                         : (nt ? adamw8_tensors<G, true, false> : adamw8_tensors<G, false, false>);
            kern<<<chunks, kThreads, 0, stream()>>>(tab, s);
        });
}

} // namespace

extern "C" {

int swc_hip_adamwAdvance(void *state, double beta1, double beta2) {
    SWC_ARG(state);
    SWC_ARG(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1);
    SWC_REQUIRE_INIT();
    // (log 0 is -infinity, and expm1 of that -1: the correction of beta 0 is 1)
    adamw_advance<<<1, 1, 0, stream()>>>(static_cast<Header *>(state), log(beta1), log(beta2));
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

int swc_hip_adamw_f(int count, float *const *w, const float *const *dw, float *const *mom, float *const *var,
                    swc_hip_bf16 *const *copies, const size_t *sizes, const void *state, float lr, double beta1, double beta2,
                    float eps, float decay, const float *lrFactor, const float *gradFactor) {
    return adamw("swc_hip_adamw_f", count, w, dw, mom, var, copies, sizes, state, lr, beta1, beta2, eps, decay, lrFactor, gradFactor);
}

int swc_hip_adamw_bf(int count, float *const *w, const swc_hip_bf16 *const *dw, float *const *mom, float *const *var,
                     swc_hip_bf16 *const *copies, const size_t *sizes, const void *state, float lr, double beta1, double beta2,
                     float eps, float decay, const float *lrFactor, const float *gradFactor) {
    return adamw("swc_hip_adamw_bf", count, w, dw, mom, var, copies, sizes, state, lr, beta1, beta2, eps, decay, lrFactor, gradFactor);
}

int swc_hip_adamw8_f(int count, float *const *w, const float *const *dw, uint8_t *const *mom8, float *const *momScale,
                     uint8_t *const *var8, float *const *varScale, swc_hip_bf16 *const *copies, const size_t *sizes,
                     const void *state, float lr, double beta1, double beta2, float eps, float decay, const float *lrFactor,
                     const float *gradFactor) {
    return adamw8("swc_hip_adamw8_f", count, w, dw, mom8, momScale, var8, varScale, copies, sizes, state, lr, beta1, beta2,
                  eps, decay, lrFactor, gradFactor);
}

int swc_hip_adamw8_bf(int count, float *const *w, const swc_hip_bf16 *const *dw, uint8_t *const *mom8,
                      float *const *momScale, uint8_t *const *var8, float *const *varScale, swc_hip_bf16 *const *copies,
                      const size_t *sizes, const void *state, float lr, double beta1, double beta2, float eps, float decay,
                      const float *lrFactor, const float *gradFactor) {
    return adamw8("swc_hip_adamw8_bf", count, w, dw, mom8, momScale, var8, varScale, copies, sizes, state, lr, beta1, beta2,
                  eps, decay, lrFactor, gradFactor);
}

} // extern "C"
