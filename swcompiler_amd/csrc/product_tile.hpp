// MFMA block-tile core of the products in the language-model operators: C[M,N] = A[M,K] * B[K,N] in bfloat16 or fp32
// with fp32 accumulation, either operand given with its contraction index contiguous in memory or with the other index
// contiguous, and the epilogue a policy.
//
// The three products of a layer and its gradients in row-major storage are exactly these forms:
//     Z  = A * B          A contiguous along k, B along n            <kAlongK, kAcross>
//     dA = dZ * B^T       both contiguous along the contraction (n)  <kAlongK, kAlongK>
//     dB = A^T * dZ       both contiguous across it (m)              <kAcross, kAcross>
// so nothing is ever transposed in memory.
//
// Everything up to the registers counts in bytes and is the same for both types: a slice is 128 bytes of contraction (64
// bf16, 32 fp32), a step 32 bytes (16, 8); in a step a lane of half-wave h = lane / 32 needs the 16 bytes at 16 h of one
// row of A and of one column of B — the operand of one v_mfma_f32_32x32x16_bf16 (k = 8h..8h+7), or of four
// v_mfma_f32_32x32x2_f32 (the sum over k has no order, so the two halves take k = 4h..4h+3).  Result register v of lane l:
// [i = 8*(v/4) + 4h + v%4][j = l % 32], i from the first operand.  The kernels pass B's fragment FIRST: a lane then
// holds one row of C and four consecutive columns per register quad — row reductions (softmax) need one exchange
// between the two half-waves, and stores and residual reads are vectors.
//
// An operand stored across the contraction is turned on its way from LDS into registers:
//   bf16: ds_read_b64_tr_b16 — sixteen lanes fetch a 4 (k) x 16 block, each leaves with a column of it.
//   fp32: the rows are dealt to the T blocks of a wavefront round-robin (lane j of block t: row T j + t of the
//         wavefront's), so that the T values a lane needs at one k lie side by side: one read of 4 T bytes.
//
// Operand tiles travel global -> LDS directly (16 bytes per lane, 1 KiB per instruction; lane l lands at base + 16 l).
// Placement is therefore contiguous and bank conflicts are removed by permuting which 16-byte chunk a lane fetches:
//   along k:  row r of the tile = 8 chunks; chunk q is stored at q ^ ((r >> 1) & 7).  A 128-bit read is served 16 lanes
//             at a time (all 64 banks); 16 consecutive rows, same q, then lie on 16 distinct 16-byte bank groups.
//   across k: bf16: chunk c of k-row k is stored at c ^ key(k), key in units of 4 chunks (64 bytes): the half-wave of a
//             transposing read fetches 64 bytes of each of four consecutive k-rows, which key = k & 3 (ROWS >= 128),
//             (k >> 1) & 1 (64) or 0 (32) puts on disjoint quarters of the banks.  fp32: 32 lanes read 128 T contiguous
//             bytes, which is conflict-free for T >= 2; for T = 1 the half-waves' rows, four apart, are put on opposite
//             halves of the banks.
// Bank conflicts in the counters: none, in any tile and layout.
//
// Elements outside the matrix arrive as zeros (their lanes are given an offset beyond the buffer's record count).  The
// buffer descriptors are based at the tile (and, for an operand stored across k, moved along with k), so that matrices
// of any size are reached with 32-bit offsets.
//
// What bounds the large bf16 tiles is power: on N(0,1) data the clock falls to 1.65-1.8 GHz, where zeros keep 2.4 (8192^3
// without an epilogue: 1370-1395 TFLOP/s against 1980 with four wavefronts, 1290 against 1760 with eight).  The MFMAs alone,
// with neither loads nor LDS reads, reach 1670 on N(0,1), without global loads 1530.  Idle matrix cycles cost power too, so
// what was gained came from keeping the pipe fed (TFLOP/s at 8192^3, one after the other on one card, on which all was some 4 %
// faster than above):
//   one slice of loads in flight, masks and LDS addresses computed in the loop  1280
//   + whole rounds unrolled: no vector instruction between MFMAs                1310
//   + serpentine order, one operand changes from MFMA to MFMA                   1350
//   + A's loads a slice further ahead than B's (three stages and two)           1410
//   + four wavefronts of 128 x 128 for long contractions                        1450
#pragma once
#include "common.hpp"
#include "mfma_dma.hpp"

#include <cstdint>
#include <type_traits>

namespace swc_hip {
namespace product {

using mfma::v16f;
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

typedef uint16_t bf16;   // its bits
template <class T> constexpr bool kIsBf16 = std::is_same_v<T, bf16>;

enum Layout { kAlongK, kAcross };

constexpr int kSliceBytes = 128, kStepBytes = 32, kSteps = kSliceBytes / kStepBytes;
template <class T> constexpr int kSlice = kSliceBytes / (int)sizeof(T);   // contraction indices of a slice
template <class T> constexpr int kChunk = 16 / (int)sizeof(T);            // elements of a 16-byte chunk

// largest leading dimension whose tile offsets stay inside 31 bits (256 rows of it), and most rows: indices of tiles, ranges
// of a contraction and slices loaded past its end all stay inside 31 bits
template <class T> constexpr long kMaxLd = (1L << 31) / (256 * (long)sizeof(T)) - 64;
constexpr int kMaxRows = 1 << 30;

template <class T> struct Shape {
    const T *a;
    const T *b;
    long lda, ldb;
    int m, n, k;
    int k_per_split;   // multiple of the slice
    int splits;        // ranges of the contraction
    const int *rows;   // device count of the rows (of A when along k, of both operands' contraction when across) that
                       // exist, at most m resp. k; null: all of them
};

// TM x TN accumulators of 32 x 32 per wavefront, WM x WN wavefronts; SA slices of A and SB of B in LDS (SA = SB, or
// SA = SB + 1).
template <int TM_, int TN_, int WM_, int WN_, int SA_, int SB_>
struct Cfg {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, SA = SA_, SB = SB_;
    static constexpr int NW = WM * WN;
    static constexpr int kThreads = 64 * NW;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    static constexpr int kABytes = BM * kSliceBytes, kBBytes = BN * kSliceBytes;
    static constexpr int kBBase = SA * kABytes;   // the stages of A, then those of B
    static constexpr int kLdsBytes = SA * kABytes + SB * kBBytes;
    static constexpr int kALoads = kABytes / 1024 / NW, kBLoads = kBBytes / 1024 / NW;
    static constexpr int kLoads = kALoads + kBLoads;
    static constexpr bool kEarlyA = SA > SB;      // A's loads go out a slice ahead of B's (see tile_product)
    static constexpr int kRound = SA == SB ? SA : SA * SB;   // slices after which both rings are where they were
    // loads that may be pending where the next slice must have landed
    static constexpr int kPending = kEarlyA ? (SB - 2) * kBLoads + (SB - 1) * kALoads : (SB - 2) * kLoads;
    static_assert(kALoads * 1024 * NW == kABytes && kBLoads * 1024 * NW == kBBytes, "whole 1-KiB loads per wavefront");
    static_assert(kLdsBytes <= swc::devices::HipDevice::ldsBytesPerCU, "the rings must fit one CU's LDS");
    static_assert(SB >= 2 && (SA == SB || SA == SB + 1) && SB * kLoads < 64, "pending loads must fit the vmcnt field");
};

// Where the values of a wavefront's accumulators lie in its part of C.  A lane's values of a row come in groups q of four
// consecutive columns; value u = 4 q + e of them is column col(q, h) + e.
template <class T, Layout LA, Layout LB, int TM, int TN> struct Place {
    static constexpr bool kDealtRows = !kIsBf16<T> && LA == kAcross, kDealtCols = !kIsBf16<T> && LB == kAcross && TN > 1;
    static constexpr int kGroups = 4 * TN, kValues = 16 * TN;
    static_assert(!kDealtCols || TN == 2 || TN == 4, "");
    static __device__ __forceinline__ int row(int tm, int l32) { return kDealtRows ? TM * l32 + tm : 32 * tm + l32; }
    static __device__ __forceinline__ int col(int q, int h) {
        if (!kDealtCols) return 32 * (q / 4) + 8 * (q % 4) + 4 * h;
        return TN == 2 ? 16 * (q / 2) + 8 * h + 4 * (q % 2) : 32 * (q / 4) + 16 * h + 4 * (q % 4);
    }
    static __device__ __forceinline__ int column(int u, int h) { return col(u / 4, h) + u % 4; }
    static __device__ __forceinline__ float value(const v16f (&acc)[TN], int u) {
        const int q = u / 4, e = u % 4;
        if (!kDealtCols) return acc[q / 4][4 * (q % 4) + e];
        return TN == 2 ? acc[e % 2][4 * (q / 2) + 2 * (q % 2) + e / 2] : acc[e % TN][4 * (q / 4) + q % 4];
    }
};

#if __HIP_DEVICE_COMPILE__

// Accumulators in the AGPR half of the register file: with accumulators in ordinary VGPRs every LDS read that returns
// competes with the matrix core's accumulator traffic.  As inline assembly the instruction is opaque to the compiler's
// hazard recogniser: the loop needs nothing (an accumulator is only read by the next MFMA that accumulates into it,
// which the hardware interlocks), the first ordinary read of the results must be preceded by acc_settle().
__device__ __forceinline__ void mfma_acc(v16f &acc, v8bf first, v8bf second) {
    asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(first), "v"(second));
}

// This wavefront's LDS reads have returned and at most PENDING newer loads are outstanding; then all wavefronts meet.
template <int PENDING> __device__ __forceinline__ void ring_sync() {
    static_assert(PENDING >= 0 && PENDING < 64, "");
    __builtin_amdgcn_s_waitcnt(0x0070 | (PENDING & 15) | ((PENDING >> 4) << 14));   // vmcnt(PENDING) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <class T, int BLOCKS, int ROWS> __device__ __forceinline__ int across_key(int k) {
    if (kIsBf16<T>) return ROWS >= 128 ? (k & 3) << 2 : ROWS == 64 ? ((k >> 1) & 1) << 2 : 0;
    return BLOCKS == 1 && ROWS >= 64 ? ((k >> 2) & 1) << 3 : 0;
}

// One operand's tile: ROWS x a slice, loaded by NW wavefronts; BLOCKS: blocks of 32 rows a wavefront reads.
template <class T, int ROWS, int BLOCKS, Layout L, int NW>
struct Loader {
    static constexpr int E = sizeof(T);
    static constexpr int kLoads = ROWS * kSliceBytes / 1024 / NW;
    const char *base;    // of the tile at the slice being loaded
    long left;           // bytes from base to the end of the matrix
    long step;           // bytes from slice to slice
    int k0, k_end;
    int off[kLoads];     // byte offset of the lane's chunk from base, kOutOfRange outside the matrix
    int kk[kLoads];      // k of the chunk inside a slice

    // rows: how many rows (columns of C or rows of C) the matrix has; k_end: contraction indices at or beyond it do not exist
    __device__ __forceinline__ void init(const T *p, long ld, int rows, int row0, int k_begin, int k_end_, int k_all, int wave,
                                         int lane) {
        k0 = k_begin, k_end = k_end_;
        const long start = L == kAlongK ? (long)row0 * ld + k_begin : (long)k_begin * ld + row0;
        const long total = L == kAlongK ? (long)(rows - 1) * ld + k_all : (long)(k_all - 1) * ld + rows;
        base = reinterpret_cast<const char *>(p + start);
        left = ((total * E + 3) & ~3L) - start * E;   // (the buffer's bounds count whole dwords: an odd last bf16 is in)
        step = L == kAlongK ? (long)kSliceBytes : kSlice<T> * E * ld;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int chunk = (wave * kLoads + j) * 64 + lane;   // position in the tile, in 16-byte chunks
            if (L == kAlongK) {
                const int r = chunk / 8;
                const int q = (chunk % 8) ^ ((r >> 1) & 7);
                kk[j] = q * kChunk<T>;
                off[j] = row0 + r < rows ? r * (int)ld * E + q * 16 : mfma::kOutOfRange;
            } else {
                constexpr int kPer = ROWS * E / 16;
                const int r = chunk / kPer;
                const int q = (chunk % kPer) ^ across_key<T, BLOCKS, ROWS>(r);
                kk[j] = r;
                off[j] = row0 + q * kChunk<T> < rows ? r * (int)ld * E + q * 16 : mfma::kOutOfRange;
            }
        }
    }
    // WHOLE: the slice lies inside the contraction, no chunk has to be checked against its end
    template <bool WHOLE> __device__ __forceinline__ void issue(char *__restrict__ stage, int j, int wave) {
        const long reach = left < 0 ? 0 : left < 0x7fffff00L ? left : 0x7fffff00L;
        const __amdgpu_buffer_rsrc_t rsrc = mfma::make_rsrc(base, (unsigned)reach);
        const int v = WHOLE || k0 + kk[j] < k_end ? off[j] : mfma::kOutOfRange;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (mfma::lds_void_t *)(stage + (wave * kLoads + j) * 1024), 16, v, 0, 0, 0);
    }
    __device__ __forceinline__ void skip(int slices) {
        base += slices * step;
        left -= slices * step;
        k0 += slices * kSlice<T>;
    }
    __device__ __forceinline__ void next() { skip(1); }
};

// What a lane holds of one block of 32 rows for one step: 16 bytes.
template <class T> struct Frag;
template <> struct Frag<bf16> {
    v8bf v;
};
template <> struct Frag<float> {
    v4f v;
};

// A wavefront's fragments of BLOCKS blocks of 32 rows at one step, in kReads LDS instructions.
template <class T, int ROWS, int BLOCKS, Layout L>
struct Reader {
    static constexpr int E = sizeof(T);
    static constexpr int kOffs = L == kAlongK ? kSteps : kIsBf16<T> ? BLOCKS : 1;
    static constexpr int kReads = L == kAlongK ? BLOCKS : kIsBf16<T> ? 2 * BLOCKS : 4;
    int off[kOffs];   // byte offset in the tile: per step (along k), per block (across, bf16), of the first k (across, fp32)

    __device__ __forceinline__ void init(int row0, int lane) {
        const int l32 = lane & 31, h = lane >> 5;
        if (L == kAlongK) {
            const int r = row0 + l32;
#pragma unroll
            for (int s = 0; s < kOffs; ++s) off[s] = r * kSliceBytes + (((2 * s + h) ^ ((r >> 1) & 7)) << 4);
        } else if (kIsBf16<T>) {
            const int i = lane & 15;
            const int krow = 8 * h + (i >> 2);   // of the first of the two reads; the second is four rows down
#pragma unroll
            for (int t = 0; t < kOffs; ++t) {
                const int col = row0 + t * 32 + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
                off[t] = krow * ROWS * E + (((col >> 3) ^ across_key<T, BLOCKS, ROWS>(krow)) << 4) + (col & 4) * E;
            }
        } else {
            const int col = row0 + BLOCKS * l32;
            off[0] = 4 * h * ROWS * E + (((col * E >> 4) ^ across_key<T, BLOCKS, ROWS>(4 * h)) << 4) + (col * E & 15);
        }
    }
    __device__ __forceinline__ void read(Frag<T> (&f)[BLOCKS], const char *__restrict__ tile, int step, int q) const {
        if constexpr (L == kAlongK) {
            f[q].v = *reinterpret_cast<const decltype(f[q].v) *>(tile + off[step] + q * 32 * kSliceBytes);
        } else if constexpr (kIsBf16<T>) {
            // (the key of a k-row repeats every four rows: the rows of a step share the lane's offset)
            typedef __attribute__((address_space(3))) v4s *lds_v4s;
            const int t = q / 2, p = q % 2;
            const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(tile + off[t] + (step * 16 + 4 * p) * ROWS * E));
            v8s whole = __builtin_bit_cast(v8s, f[t].v);
#pragma unroll
            for (int e = 0; e < 4; ++e) whole[4 * p + e] = x[e];
            f[t].v = __builtin_bit_cast(v8bf, whole);
        } else {
            // (the key of a k-row, where there is one, depends on k / 4 % 2 = h alone: steps are 8 k)
            typedef float vec __attribute__((ext_vector_type(BLOCKS)));
            const vec x = *reinterpret_cast<const vec *>(tile + off[0] + (step * 8 + q) * ROWS * E);
#pragma unroll
            for (int t = 0; t < BLOCKS; ++t) f[t].v[q] = x[t];
        }
    }
};

template <class T, class C> struct Frags {
    Frag<T> a[C::TM], b[C::TN];
};

// The tile of this workgroup at (m0, n0), contraction [k_begin, k_end): accumulators of this wavefront.
//
// One barrier per slice, before its last step: by then every wavefront holds the slice's last fragments in registers
// and its own part of the next slice has landed, so behind the barrier the next slice may be read (its first fragments
// are fetched under the last step's MFMAs) and the slice's own stages refilled.  The matrix pipe never waits at a slice
// boundary for LDS.
//
// A load issued behind the barrier has one slice's time to arrive, and if all of a slice's loads are issued there the
// last of them comes too late: 64 KiB per CU in one burst.  With one more stage for A, A's loads are a slice further
// ahead and go out during the slice's other steps: what is behind the barrier is B's half.
template <class T, class C, Layout LA, Layout LB>
__device__ __forceinline__ void tile_product(const Shape<T> &s, int m, int k_all, int m0, int n0, int k_begin, int k_end,
                                             char *__restrict__ lds, v16f (&acc)[C::TM][C::TN]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Loader<T, C::BM, C::TM, LA, C::NW> la;
    Loader<T, C::BN, C::TN, LB, C::NW> lb;
    la.init(s.a, s.lda, m, m0, k_begin, k_end, k_all, wave, lane);
    lb.init(s.b, s.ldb, s.n, n0, k_begin, k_end, k_all, wave, lane);
    Reader<T, C::BM, C::TM, LA> ra;
    Reader<T, C::BN, C::TN, LB> rb;
    ra.init((wave / C::WN) * 32 * C::TM, lane);
    rb.init((wave % C::WN) * 32 * C::TN, lane);
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;

    const int nk = (k_end - k_begin + kSlice<T> - 1) / kSlice<T>;
    // (slices past the end are loaded too, as zeros: the count of pending loads is then the same everywhere)
#pragma unroll
    for (int st = 0; st < C::SB; ++st) {
#pragma unroll
        for (int j = 0; j < C::kALoads; ++j) la.template issue<false>(lds + st * C::kABytes, j, wave);
#pragma unroll
        for (int j = 0; j < C::kBLoads; ++j) lb.template issue<false>(lds + C::kBBase + st * C::kBBytes, j, wave);
        la.next();
        lb.next();
    }
    Frags<T, C> f[2];
    constexpr int kAReads = decltype(ra)::kReads, kReads = kAReads + decltype(rb)::kReads;
    auto read = [&](Frags<T, C> &to, const char *__restrict__ a, const char *__restrict__ b, int step, int q) {
        if (q < kAReads) ra.read(to.a, a, step, q);
        else rb.read(to.b, b, step, q - kAReads);
    };
    ring_sync<(C::SB - 1) * C::kLoads>();
#pragma unroll
    for (int q = 0; q < kReads; ++q) read(f[0], lds, lds + C::kBBase, 0, q);
    constexpr int kBlocks = C::TM * C::TN, kMfmas = kIsBf16<T> ? kBlocks : 4 * kBlocks;
    // a, b: the slice's stages; an, bn: the next slice's; ap: the previous slice's stage of A (to be refilled here
    // when A runs ahead; this slice's otherwise)
    auto slice = [&]<bool WHOLE>(char *__restrict__ a, char *__restrict__ b, const char *__restrict__ an,
                                 const char *__restrict__ bn, char *__restrict__ ap) {
#pragma unroll
        for (int step = 0; step < kSteps; ++step) {
            const bool last = step + 1 == kSteps;
            const Frags<T, C> &now = f[step & 1];
            Frags<T, C> &then = f[(step + 1) & 1];
            if (last) ring_sync<C::kPending>();
#pragma unroll
            for (int i = 0; i < kMfmas; ++i) {
                const int tm = i % kBlocks / C::TN, tn = (tm & 1) ? C::TN - 1 - i % C::TN : i % C::TN;
                if constexpr (kIsBf16<T>) mfma_acc(acc[tm][tn], now.b[tn].v, now.a[tm].v);
                else mfma::mfma_acc(acc[tm][tn], now.b[tn].v[i / kBlocks], now.a[tm].v[i / kBlocks]);
                // the next step's fragments in the first half of the step, loads in the second half or behind the barrier
#pragma unroll
                for (int q = 0; q < kReads; ++q)
                    if (q * ((kMfmas + 1) / 2) / kReads == i) read(then, last ? an : a, last ? bn : b, last ? 0 : step + 1, q);
                constexpr int kLate = C::kEarlyA ? C::kBLoads : C::kLoads;
                if (last) {
#pragma unroll
                    for (int j = 0; j < kLate; ++j)
                        if (j * kMfmas / kLate == i) {
                            if (C::kEarlyA) lb.template issue<WHOLE>(b, j, wave);
                            else if (j < C::kALoads) la.template issue<WHOLE>(a, j, wave);
                            else lb.template issue<WHOLE>(b, j - C::kALoads, wave);
                        }
                } else if (C::kEarlyA) {
                    constexpr int kSlots = (kSteps - 1) * kMfmas;
#pragma unroll
                    for (int j = 0; j < C::kALoads; ++j)
                        if ((2 * j + 1) * kSlots / (2 * C::kALoads) == step * kMfmas + i) la.template issue<WHOLE>(ap, j, wave);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        la.next();
        lb.next();
    };
    // Every vector instruction between the MFMAs costs matrix cycles.  While the slices being loaded lie inside the
    // contraction there are none: whole rounds of the rings, unrolled, so that every LDS address is a lane's constant.
    const int whole = (k_end - k_begin) / kSlice<T> - C::SB;   // slices whose successors in the rings are whole
    int kt = 0;
    for (; kt + C::kRound <= whole; kt += C::kRound) {
#pragma unroll
        for (int st = 0; st < C::kRound; ++st)
            slice.template operator()<true>(lds + st % C::SA * C::kABytes, lds + C::kBBase + st % C::SB * C::kBBytes,
                                            lds + (st + 1) % C::SA * C::kABytes, lds + C::kBBase + (st + 1) % C::SB * C::kBBytes,
                                            lds + (st + C::SA - 1) % C::SA * C::kABytes);
    }
    for (int sa = 0, sb = 0; kt < nk; ++kt) {
        const int na = sa + 1 == C::SA ? 0 : sa + 1, nb = sb + 1 == C::SB ? 0 : sb + 1, pa = sa ? sa - 1 : C::SA - 1;
        slice.template operator()<false>(lds + sa * C::kABytes, lds + C::kBBase + sb * C::kBBytes, lds + na * C::kABytes,
                                         lds + C::kBBase + nb * C::kBBytes, lds + pa * C::kABytes);
        sa = na, sb = nb;
    }
    mfma::wait_vmcnt<0>();   // the trailing loads of zeros still target this workgroup's LDS
    mfma::acc_settle(acc);
}

__device__ __forceinline__ float bf16_to_float(unsigned bits) { return __builtin_bit_cast(float, bits << 16); }
// two floats to two bf16, rounded to nearest even
__device__ __forceinline__ unsigned pack_bf16(float x, float y) {
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    v2bf v;
    v[0] = (__bf16)x;
    v[1] = (__bf16)y;
    return __builtin_bit_cast(unsigned, v);
}

// Vectors at any element's address: one memory instruction (the target takes unaligned global accesses).
template <class T> struct At;
template <> struct At<bf16> {
    typedef v4u chunk __attribute__((aligned(2)));
    typedef v2u four __attribute__((aligned(2)));
};
template <> struct At<float> {
    typedef v4f chunk __attribute__((aligned(4)));
    typedef v4f four __attribute__((aligned(4)));
};

// A lane's part of a row of C (or of a matrix of its shape) to and from memory, `row` the address of the row's first
// column and col0 the wavefront's first.  Every lane of the wavefront calls these; ok: its row exists.  WHOLE: the row
// exists with all the wavefront's columns (the path without control flow: a branch per row makes the compiler wait for
// every store before it).
//
// bf16: the sixteen values of a 32-column block are dealt out again between the half-waves, so that lane h holds columns
// 16 q + 8 h .. + 7 of it: 16-byte accesses.
__device__ __forceinline__ void half_waves_swap(unsigned &lo, unsigned &hi) {   // lo's upper half with hi's lower half
    const auto r = __builtin_amdgcn_permlane32_swap(lo, hi, false, false);
    lo = r[0], hi = r[1];
}

template <class P, bool WHOLE>
__device__ __forceinline__ void store_row(bf16 *row, bool ok, int col0, int n, int h, const float (&x)[P::kValues]) {
#pragma unroll
    for (int b = 0; b < P::kValues / 16; ++b)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const float *v = x + 16 * b + 8 * q;
            unsigned d[4] = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
            half_waves_swap(d[0], d[2]);
            half_waves_swap(d[1], d[3]);
            const int c = col0 + 32 * b + 16 * q + 8 * h;
            if (WHOLE || (ok && c + 8 <= n)) {
                *reinterpret_cast<At<bf16>::chunk *>(row + c) = v4u{d[0], d[1], d[2], d[3]};
            } else if (ok) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < n) row[c + e] = (bf16)(d[e / 2] >> (16 * (e & 1)));
            }
        }
}
template <class P, bool WHOLE>
__device__ __forceinline__ void store_row(float *row, bool ok, int col0, int n, int h, const float (&x)[P::kValues]) {
#pragma unroll
    for (int q = 0; q < P::kGroups; ++q) {
        const int c = col0 + P::col(q, h);
        if (WHOLE || (ok && c + 4 <= n)) {
            *reinterpret_cast<At<float>::chunk *>(row + c) = v4f{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
        } else if (ok) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < n) row[c + e] = x[4 * q + e];
        }
    }
}

// A row's values as loaded, and in the order of the accumulators.
template <class T, class P> struct RowData;
template <class P> struct RowData<bf16, P> {
    v4u d[P::kValues / 8];
    template <bool WHOLE> __device__ __forceinline__ void load(const bf16 *row, bool ok, int col0, int n, int h) {
#pragma unroll
        for (int i = 0; i < P::kValues / 8; ++i) {
            const int c = col0 + 16 * i + 8 * h;
            if (WHOLE || (ok && c + 8 <= n)) {
                d[i] = *reinterpret_cast<const At<bf16>::chunk *>(row + c);
            } else {
                d[i] = v4u{0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (ok && c + e < n) d[i][e / 2] |= (unsigned)row[c + e] << (16 * (e & 1));
            }
        }
    }
    __device__ __forceinline__ void get(float (&x)[P::kValues]) const {
#pragma unroll
        for (int i = 0; i < P::kValues / 8; ++i) {
            unsigned w[4] = {d[i][0], d[i][1], d[i][2], d[i][3]};
            half_waves_swap(w[0], w[2]);
            half_waves_swap(w[1], w[3]);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[8 * i + e] = __builtin_bit_cast(float, e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        }
    }
};
template <class P> struct RowData<float, P> {
    v4f d[P::kGroups];
    template <bool WHOLE> __device__ __forceinline__ void load(const float *row, bool ok, int col0, int n, int h) {
#pragma unroll
        for (int q = 0; q < P::kGroups; ++q) {
            const int c = col0 + P::col(q, h);
            if (WHOLE || (ok && c + 4 <= n)) {
                d[q] = *reinterpret_cast<const At<float>::chunk *>(row + c);
            } else {
                d[q] = v4f{0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (ok && c + e < n) d[q][e] = row[c + e];
            }
        }
    }
    __device__ __forceinline__ void get(float (&x)[P::kValues]) const {
#pragma unroll
        for (int u = 0; u < P::kValues; ++u) x[u] = d[u / 4][u % 4];
    }
};

// The values a lane needs of a vector over the columns (bias), as loaded.  WHOLE: all columns exist.
template <class T, class P> struct ColumnData {
    typedef std::conditional_t<kIsBf16<T>, v2u, v4f> four;
    four d[P::kGroups];
    template <bool WHOLE> __device__ __forceinline__ void load(const T *v, int col0, int n, int h) {
#pragma unroll
        for (int q = 0; q < P::kGroups; ++q) {
            const int c = col0 + P::col(q, h);
            if (WHOLE || c + 4 <= n) {
                d[q] = *reinterpret_cast<const typename At<T>::four *>(v + c);
            } else {
                d[q] = four{};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < n) {
                        if constexpr (kIsBf16<T>) d[q][e / 2] |= (unsigned)v[c + e] << (16 * (e & 1));
                        else d[q][e] = v[c + e];
                    }
            }
        }
    }
    __device__ __forceinline__ float value(int u) const {
        if constexpr (kIsBf16<T>) {
            const unsigned w = d[u / 4][u % 4 / 2];
            return __builtin_bit_cast(float, u & 1 ? w & 0xffff0000u : w << 16);
        } else {
            return d[u / 4][u % 4];
        }
    }
};

#endif  // __HIP_DEVICE_COMPILE__

// Workgroup id -> number of its work, of `total`: those that land on one XCD (every eighth) are consecutive.  Work is
// numbered range by range of the contraction and tile by tile within one, and the tiles in column strips four tall, so that
// the 32 tiles an XCD holds at a time are 4 x 8 of one range: they share operand tiles in its L2.  (Strips of 8: 4096 x 16384
// x 4096 442 us against 430, 8192^3 the same; of 16: 494.)
__device__ __forceinline__ int xcd_order(int id, int total) {
    constexpr int kXcd = swc::devices::HipDevice::xcds;
    const int x = id % kXcd, more = total % kXcd;
    return x * (total / kXcd) + (x < more ? x : more) + id / kXcd;
}
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int &tile_m, int &tile_n) {
    constexpr int kStrip = 4;
    const int strip = id / (kStrip * tiles_n), first = strip * kStrip;
    const int rows = tiles_m - first < kStrip ? tiles_m - first : kStrip;
    const int in = id - strip * kStrip * tiles_n;
    tile_m = first + in % rows;
    tile_n = in / rows;
}

// An epilogue receives, once per wavefront, its accumulators and where they lie:
//     ep.template finish<P>(acc, row0, col0, m, n, lane, split): P a Place, (row0, col0) the wavefront's part of C
#if __HIP_DEVICE_COMPILE__
template <class T, class C, Layout LA, Layout LB, class Ep>
__device__ __forceinline__ void product_tile(const Shape<T> &s, const Ep &ep, int id, char *lds_bytes) {
    int m = s.m, k = s.k;
    if (s.rows) {   // rows left out of a loss: the count is known on the device only
        const int have = __builtin_amdgcn_readfirstlane(*s.rows);
        if (LA == kAlongK) m = have < m ? have : m;
        else k = have < k ? have : k;
    }
    // (of the tiles that exist: with rows left out their work would otherwise fall to some XCDs alone)
    const int tiles_m = (m + C::BM - 1) / C::BM, tiles_n = (s.n + C::BN - 1) / C::BN, tiles = tiles_m * tiles_n;
    if (id >= tiles * s.splits) return;
    id = xcd_order(id, tiles * s.splits);
    const int split = id / tiles;
    int tile_m, tile_n;
    tile_of(id - split * tiles, tiles_m, tiles_n, tile_m, tile_n);
    const int m0 = tile_m * C::BM, n0 = tile_n * C::BN;
    const int k_begin = split * s.k_per_split;
    const int k_end = k_begin + s.k_per_split < k ? k_begin + s.k_per_split : k;
    v16f acc[C::TM][C::TN];
    if (k_begin < k_end) {
        tile_product<T, C, LA, LB>(s, m, k, m0, n0, k_begin, k_end, lds_bytes, acc);
    } else {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int j = 0; j < C::TN; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    ep.template finish<Place<T, LA, LB, C::TM, C::TN>>(acc, m0 + (wave / C::WN) * 32 * C::TM, n0 + (wave % C::WN) * 32 * C::TN, m, s.n,
                                                       (int)(threadIdx.x & 63), split);
}
#endif

template <class T, class C, Layout LA, Layout LB, class Ep>
__global__ __launch_bounds__(C::kThreads) void product_tiles(Shape<T> s, Ep ep) {
#if __HIP_DEVICE_COMPILE__
    extern __shared__ __align__(16) char lds_bytes[];
    product_tile<T, C, LA, LB>(s, ep, (int)blockIdx.x, lds_bytes);
#endif
}
// The two products of a layer's gradients in one launch, dB's workgroups behind dA's `groups`.
template <class T, class CA, class CB, class Ep>
__global__ __launch_bounds__(CA::kThreads) void product_pair(Shape<T> a, Ep ep_a, int groups, Shape<T> b, Ep ep_b) {
    static_assert(CA::kThreads == CB::kThreads, "");
#if __HIP_DEVICE_COMPILE__
    extern __shared__ __align__(16) char lds_bytes[];
    const int id = blockIdx.x;
    if (id < groups) product_tile<T, CA, kAlongK, kAlongK>(a, ep_a, id, lds_bytes);
    else product_tile<T, CB, kAcross, kAcross>(b, ep_b, id - groups, lds_bytes);
#endif
}

// The matrix of the product in its type.  PLACED: its rows go where `rows` says (null: in order).
template <class T, bool PLACED = false> struct Store {
    static constexpr bool kHeavy = false, kThinToo = true;
    T *out;
    long ld;
    const int *rows = nullptr;
    Store from(int j) const { return {out + j, ld, rows}; }
#if __HIP_DEVICE_COMPILE__
    template <class P, bool WHOLE, int TM, int TN>
    __device__ __forceinline__ void store(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane) const {
        const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + P::row(tm, l32);
            float x[P::kValues];
#pragma unroll
            for (int u = 0; u < P::kValues; ++u) x[u] = P::value(acc[tm], u);
            const bool ok = WHOLE || row < m;
            const long at = PLACED && rows && ok ? rows[row] : row;
            store_row<P, WHOLE>(out + at * ld, ok, col0, n, h, x);
        }
    }
    template <class P, int TM, int TN>
    __device__ __forceinline__ void finish(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane, int) const {
        if (row0 + 32 * TM <= m && col0 + 32 * TN <= n) store<P, true>(acc, row0, col0, m, n, lane);
        else store<P, false>(acc, row0, col0, m, n, lane);
    }
#endif
};

// fp32 partial sums of a range (or the whole product when there is one): out[split][m][n], ld = n
struct StorePartial {
    static constexpr bool kHeavy = false, kThinToo = true;
    float *out;
    long split_stride;   // elements between the splits' matrices
    long ld;
    bool add;            // out += : a product summed over several calls
    StorePartial from(int j) const { return {out + j, split_stride, ld, add}; }
#if __HIP_DEVICE_COMPILE__
    template <class P, int TM, int TN>
    __device__ __forceinline__ void finish(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane, int split) const {
        const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + P::row(tm, l32);
            if (row >= m) continue;
            float *p = out + split * split_stride + row * ld;
#pragma unroll
            for (int q = 0; q < P::kGroups; ++q) {
                const int col = col0 + P::col(q, h);
                v4f x = {P::value(acc[tm], 4 * q), P::value(acc[tm], 4 * q + 1), P::value(acc[tm], 4 * q + 2), P::value(acc[tm], 4 * q + 3)};
                if (col + 4 <= n) {
                    auto *o = reinterpret_cast<At<float>::chunk *>(p + col);
                    *o = add ? *o + x : x;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col + e < n) p[col + e] = add ? p[col + e] + x[e] : x[e];
                }
            }
        }
    }
#endif
};

// the one or the other: partial sums where `part.out` is given
template <class T> struct StoreEither {
    Store<T, true> whole;
    StorePartial part;
#if __HIP_DEVICE_COMPILE__
    template <class P, int TM, int TN>
    __device__ __forceinline__ void finish(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane, int split) const {
        if (part.out) part.finish<P>(acc, row0, col0, m, n, lane, split);
        else whole.template finish<P>(acc, row0, col0, m, n, lane, split);
    }
#endif
};

template <class T, class C, Layout LA, Layout LB, class Ep>
int launch_product(const Shape<T> &s, const Ep &ep, const char *who) {
    const long groups = (long)((s.m + C::BM - 1) / C::BM) * ((s.n + C::BN - 1) / C::BN) * s.splits;
    // (a grid has at most 2^32 - 1 threads in each direction)
    if (groups > 0xffffffffL / C::kThreads) return fail(SWC_HIP_EUNSUPPORTED, "%s: too many tiles", who);
    note_kernel("product<%s,%dx%d,%d,%d,%d,%s%s> x%d", kIsBf16<T> ? "bf16" : "fp32", C::BM, C::BN, C::NW, C::SA, C::SB,
                LA == kAlongK ? "k" : "m", LB == kAlongK ? "k" : "n", s.splits);
    auto kern = product_tiles<T, C, LA, LB, Ep>;
    static bool attr_set = false;
    if (!attr_set) {
        SWC_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                        C::kLdsBytes));
        attr_set = true;
    }
    kern<<<(unsigned)groups, C::kThreads, C::kLdsBytes, stream()>>>(s, ep);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

template <class T, class CA, class CB, class Ep>
int launch_pair(const Shape<T> &a, const Ep &ep_a, const Shape<T> &b, const Ep &ep_b) {
    constexpr int kLds = CA::kLdsBytes > CB::kLdsBytes ? CA::kLdsBytes : CB::kLdsBytes;
    note_kernel("product_pair<%s,%dx%d,%dx%d> x%d x%d", kIsBf16<T> ? "bf16" : "fp32", CA::BM, CA::BN, CB::BM, CB::BN, a.splits, b.splits);
    auto kern = product_pair<T, CA, CB, Ep>;
    static bool attr_set = false;
    if (!attr_set) {
        SWC_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
        attr_set = true;
    }
    const unsigned groups = ceil_div(a.m, CA::BM) * ceil_div(a.n, CA::BN) * a.splits;
    const unsigned groups_b = ceil_div(b.m, CB::BM) * ceil_div(b.n, CB::BN) * b.splits;
    kern<<<groups + groups_b, CA::kThreads, kLds, stream()>>>(a, ep_a, (int)groups, b, ep_b);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

} // namespace product
} // namespace swc_hip
