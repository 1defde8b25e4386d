// bf16 MFMA block-tile core: C[M,N] = A[M,K] * B[K,N] with fp32 accumulation, either operand given with its
// contraction index contiguous in memory or with the other index contiguous, and the epilogue a policy.
//
// The three products of a layer and its gradients in row-major storage are exactly these forms:
//     Z  = A * B          A contiguous along k, B along n            <kAlongK, kAcross>
//     dA = dZ * B^T       both contiguous along the contraction (n)  <kAlongK, kAlongK>
//     dB = A^T * dZ       both contiguous across it (m)              <kAcross, kAcross>
// so nothing is ever transposed in memory: an operand stored across the contraction is transposed on its way from
// LDS into registers (ds_read_b64_tr_b16: sixteen lanes fetch a 4 x 16 block, each leaves with a column of it).
//
// v_mfma_f32_32x32x16_bf16, lane l of 64 (h = l / 32): first operand [i = l % 32][k = 8h..8h+7], second operand
// [k = 8h..8h+7][j = l % 32], result register v: [i = 8*(v/4) + 4h + v%4][j = l % 32].  The kernels pass B's fragment
// FIRST: a lane then holds one row of C and four consecutive columns per register quad — row reductions (softmax)
// need one exchange between the two half-waves, and stores and residual reads are vectors.
//
// Operand tiles travel global -> LDS directly (16 bytes per lane, 1 KiB per instruction; lane l lands at base + 16 l).
// Placement is therefore contiguous and bank conflicts are removed by permuting which 16-byte chunk a lane fetches:
//   along k:  row r of the tile = BK/8 chunks; chunk q is stored at q ^ key(r).  A 128-bit read is served 16 lanes at a
//             time (all 64 banks); 16 consecutive rows, same q: with BK = 64 (128-byte rows) key = (r >> 1) & 7, with
//             BK = 32 (64-byte rows) key = (r >> 2) & 3 puts them on 16 distinct 16-byte bank groups.
//   across k: k-row = ROWS/8 chunks; chunk c of row k is stored at c ^ key(k), key in units of 4 chunks (64 bytes): the
//             half-wave of a transposing read fetches 64 bytes of each of four consecutive k-rows, which key = k & 3
//             (ROWS >= 128), (k >> 1) & 1 (64) or 0 (32) puts on disjoint quarters of the banks.
// Elements outside the matrix arrive as zeros (their lanes are given an offset beyond the buffer's record count).  The
// buffer descriptors are based at the tile (and, for an operand stored across k, moved along with k), so that matrices
// of any size are reached with 32-bit offsets.
#pragma once
#include "common.hpp"
#include "mfma_dma.hpp"

#include <cstdint>

namespace swc_hip {
namespace mfma16 {

using mfma::v16f;
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

enum Layout { kAlongK, kAcross };

// largest leading dimension whose tile offsets stay inside 31 bits (256 rows of it)
constexpr long kMaxLd = (1L << 31) / (256 * 2) - 64;

struct Shape {
    const uint16_t *a;
    const uint16_t *b;
    long lda, ldb;
    int m, n, k;
    int k_per_split;   // multiple of the slice; grid.y = number of splits
    const int *rows;   // device count of the rows (of A when along k, of both operands' contraction when across) that
                       // exist, at most m resp. k; null: all of them
};

// TM x TN accumulators of 32 x 32 per wavefront, WM x WN wavefronts, slices of BK; SA slices of A and SB of B in LDS
// (SA = SB, or SA = SB + 1).
template <int TM_, int TN_, int WM_, int WN_, int BK_, int SA_, int SB_>
struct Cfg {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, BK = BK_, SA = SA_, SB = SB_;
    static constexpr int NW = WM * WN;
    static constexpr int kThreads = 64 * NW;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    static constexpr int kABytes = BM * BK * 2, kBBytes = BN * BK * 2;
    static constexpr int kBBase = SA * kABytes;   // the stages of A, then those of B
    static constexpr int kLdsBytes = SA * kABytes + SB * kBBytes;
    static constexpr int kALoads = kABytes / 1024 / NW, kBLoads = kBBytes / 1024 / NW;
    static constexpr int kLoads = kALoads + kBLoads;
    static constexpr int kSteps = BK / 16;
    static constexpr bool kEarlyA = SA > SB;      // A's loads go out a slice ahead of B's (see tile_product)
    static constexpr int kRound = SA == SB ? SA : SA * SB;   // slices after which both rings are where they were
    // loads that may be pending where the next slice must have landed
    static constexpr int kPending = kEarlyA ? (SB - 2) * kBLoads + (SB - 1) * kALoads : (SB - 2) * kLoads;
    static_assert(kALoads * 1024 * NW == kABytes && kBLoads * 1024 * NW == kBBytes, "whole 1-KiB loads per wavefront");
    static_assert(kLdsBytes <= swc::devices::HipDevice::ldsBytesPerCU, "the rings must fit one CU's LDS");
    static_assert(SB >= 2 && (SA == SB || SA == SB + 1) && SB * kLoads < 64, "pending loads must fit the vmcnt field");
    static_assert(BK == 32 || BK == 64, "");
    static_assert(kSteps >= 2, "");
};

#if __HIP_DEVICE_COMPILE__

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

// Wait states between the last MFMA (8 passes) and the first ordinary read of a result.
template <int TM, int TN> __device__ __forceinline__ void acc_settle(v16f (&acc)[TM][TN]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) asm volatile("" : "+a"(acc[i][j]));
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+a"(acc[TM - 1][TN - 1]));
}

// One operand's tile: ROWS x BK elements, loaded by NW wavefronts.
template <int ROWS, Layout L, int BK, int NW>
struct Loader {
    static constexpr int kLoads = ROWS * BK * 2 / 1024 / NW;
    const char *base;    // of the tile at the slice being loaded
    long left;           // bytes from base to the end of the matrix
    long step;           // bytes from slice to slice
    int k0, k_end;
    int off[kLoads];     // byte offset of the lane's chunk from base, kOutOfRange outside the matrix
    int kk[kLoads];      // k of the chunk inside a slice

    // rows: how many rows (columns of C or rows of C) the matrix has; k_end: contraction indices at or beyond it do not exist
    __device__ __forceinline__ void init(const uint16_t *p, long ld, int rows, int row0, int k_begin, int k_end_, int k_all,
                                         int wave, int lane) {
        k0 = k_begin, k_end = k_end_;
        const long start = L == kAlongK ? (long)row0 * ld + k_begin : (long)k_begin * ld + row0;
        const long total = L == kAlongK ? (long)(rows - 1) * ld + k_all : (long)(k_all - 1) * ld + rows;
        base = reinterpret_cast<const char *>(p + start);
        left = ((total + 1) & ~1L) * 2 - start * 2;   // (the buffer's bounds count whole dwords: an odd last element is in)
        step = L == kAlongK ? BK * 2 : BK * 2 * ld;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int chunk = (wave * kLoads + j) * 64 + lane;   // position in the tile, in 16-byte chunks
            if (L == kAlongK) {
                constexpr int kPer = BK / 8;
                const int r = chunk / kPer;
                const int key = BK == 64 ? (r >> 1) & 7 : (r >> 2) & 3;
                kk[j] = ((chunk % kPer) ^ key) * 8;
                off[j] = row0 + r < rows ? r * (int)ld * 2 + kk[j] * 2 : mfma::kOutOfRange;
            } else {
                constexpr int kPer = ROWS / 8;
                const int r = chunk / kPer;
                const int key = ROWS >= 128 ? (r & 3) << 2 : ROWS == 64 ? ((r >> 1) & 1) << 2 : 0;
                const int c = ((chunk % kPer) ^ key) * 8;
                kk[j] = r;
                off[j] = row0 + c < rows ? r * (int)ld * 2 + c * 2 : mfma::kOutOfRange;
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
    __device__ __forceinline__ void next() {
        base += step;
        left -= step;
        k0 += BK;
    }
};

// A wavefront's fragments of T blocks of 32 rows at one step of 16 k.
template <int ROWS, Layout L, int BK, int T>
struct Reader {
    static constexpr int kOffs = L == kAlongK ? BK / 16 : T;
    int off[kOffs];   // byte offset in the tile: per step (along k) or per block (across)

    __device__ __forceinline__ void init(int row0, int lane) {
        const int l32 = lane & 31, h = lane >> 5;
        if (L == kAlongK) {
            const int r = row0 + l32;
            const int key = BK == 64 ? (r >> 1) & 7 : (r >> 2) & 3;
#pragma unroll
            for (int s = 0; s < kOffs; ++s) off[s] = r * BK * 2 + (((2 * s + h) ^ key) << 4);
        } else {
            const int i = lane & 15;
            const int krow = 8 * h + (i >> 2);   // of the first of the two reads; the second is four rows down
            const int key = ROWS >= 128 ? (krow & 3) << 2 : ROWS == 64 ? ((krow >> 1) & 1) << 2 : 0;
#pragma unroll
            for (int t = 0; t < kOffs; ++t) {
                const int col = row0 + t * 32 + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
                off[t] = krow * ROWS * 2 + (((col >> 3) ^ key) << 4) + (col & 4) * 2;
            }
        }
    }
    // The number of LDS instructions a fragment takes.
    static constexpr int kPieces = L == kAlongK ? 1 : 2;
    __device__ __forceinline__ void piece(v8bf &f, const char *__restrict__ tile, int step, int t, int p) const {
        if (L == kAlongK) {
            f = *reinterpret_cast<const v8bf *>(tile + off[step] + t * 32 * BK * 2);
        } else {
            // (the key of a k-row repeats every four (ROWS >= 128, 64) rows: the rows of a step share the lane's offset)
            typedef __attribute__((address_space(3))) v4s *lds_v4s;
            const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_v4s)(tile + off[t] + (step * 16 + 4 * p) * ROWS * 2));
            v8s whole = __builtin_bit_cast(v8s, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) whole[4 * p + e] = x[e];
            f = __builtin_bit_cast(v8bf, whole);
        }
    }
};

template <class C> struct Frags {
    v8bf a[C::TM], b[C::TN];
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
template <class C, Layout LA, Layout LB>
__device__ __forceinline__ void tile_product(const Shape &s, int m, int k_all, int m0, int n0, int k_begin, int k_end,
                                             char *__restrict__ lds, v16f (&acc)[C::TM][C::TN]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Loader<C::BM, LA, C::BK, C::NW> la;
    Loader<C::BN, LB, C::BK, C::NW> lb;
    la.init(s.a, s.lda, m, m0, k_begin, k_end, k_all, wave, lane);
    lb.init(s.b, s.ldb, s.n, n0, k_begin, k_end, k_all, wave, lane);
    Reader<C::BM, LA, C::BK, C::TM> ra;
    Reader<C::BN, LB, C::BK, C::TN> rb;
    ra.init((wave / C::WN) * 32 * C::TM, lane);
    rb.init((wave % C::WN) * 32 * C::TN, lane);
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;

    const int nk = (k_end - k_begin + C::BK - 1) / C::BK;
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
    Frags<C> f[2];
    constexpr int kReads = C::TM * decltype(ra)::kPieces + C::TN * decltype(rb)::kPieces;
    auto read = [&](Frags<C> &to, const char *__restrict__ a, const char *__restrict__ b, int step, int q) {
        constexpr int kA = C::TM * decltype(ra)::kPieces;
        if (q < kA) ra.piece(to.a[q / decltype(ra)::kPieces], a, step, q / decltype(ra)::kPieces, q % decltype(ra)::kPieces);
        else {
            const int t = q - kA;
            rb.piece(to.b[t / decltype(rb)::kPieces], b, step, t / decltype(rb)::kPieces, t % decltype(rb)::kPieces);
        }
    };
    ring_sync<(C::SB - 1) * C::kLoads>();
#pragma unroll
    for (int q = 0; q < kReads; ++q) read(f[0], lds, lds + C::kBBase, 0, q);
    constexpr int kMfmas = C::TM * C::TN;
    // a, b: the slice's stages; an, bn: the next slice's; ap: the previous slice's stage of A (to be refilled here
    // when A runs ahead; this slice's otherwise)
    auto slice = [&]<bool WHOLE>(char *__restrict__ a, char *__restrict__ b, const char *__restrict__ an,
                                 const char *__restrict__ bn, char *__restrict__ ap) {
#pragma unroll
        for (int step = 0; step < C::kSteps; ++step) {
            const bool last = step + 1 == C::kSteps;
            const Frags<C> &now = f[step & 1];
            Frags<C> &then = f[(step + 1) & 1];
            if (last) ring_sync<C::kPending>();
#pragma unroll
            for (int i = 0; i < kMfmas; ++i) {
                const int tm = i / C::TN, tn = (tm & 1) ? C::TN - 1 - i % C::TN : i % C::TN;
                mfma_acc(acc[tm][tn], now.b[tn], now.a[tm]);
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
                    constexpr int kSlots = (C::kSteps - 1) * kMfmas;
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
    const int whole = (k_end - k_begin) / C::BK - C::SB;   // slices whose successors in the rings are whole
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
    acc_settle(acc);
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


// The sixteen values a lane holds of its row in one 32-column block (x[4 g + e]: column 8 g + 4 h + e) are dealt out
// again between the half-waves, so that lane h holds columns 16 q + 8 h .. + 7 in out[q]: 16-byte accesses.
__device__ __forceinline__ void pack_block(const float (&x)[16], v4u (&out)[2]) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        unsigned lo[2], hi[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            lo[i] = pack_bf16(x[8 * q + 2 * i], x[8 * q + 2 * i + 1]);
            hi[i] = pack_bf16(x[8 * q + 4 + 2 * i], x[8 * q + 4 + 2 * i + 1]);
            const auto r = __builtin_amdgcn_permlane32_swap(lo[i], hi[i], false, false);
            out[q][i] = r[0];
            out[q][2 + i] = r[1];
        }
    }
}
// The inverse, for values read from memory in 16-byte pieces.
__device__ __forceinline__ void unpack_block(const v4u (&in)[2], float (&x)[16]) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const auto r = __builtin_amdgcn_permlane32_swap(in[q][i], in[q][2 + i], false, false);
            x[8 * q + 2 * i] = bf16_to_float(r[0] & 0xffffu);
            x[8 * q + 2 * i + 1] = bf16_to_float(r[0] >> 16);
            x[8 * q + 4 + 2 * i] = bf16_to_float(r[1] & 0xffffu);
            x[8 * q + 4 + 2 * i + 1] = bf16_to_float(r[1] >> 16);
        }
}

// A row's 32-column block at column `col` to (from) memory; vec: rows start on 16-byte boundaries.  Every lane of the
// wavefront calls these; `ok` says whether its row exists.  WHOLE: it does, with all its columns and vec (the path
// without control flow: a branch per row makes the compiler wait for every store before it).
template <bool WHOLE>
__device__ __forceinline__ void store_block(uint16_t *row, bool ok, int col, int n, bool vec, int h, const float (&x)[16]) {
    v4u out[2];
    pack_block(x, out);
    if constexpr (WHOLE) {
#pragma unroll
        for (int q = 0; q < 2; ++q) *reinterpret_cast<v4u *>(row + col + 16 * q + 8 * h) = out[q];
    } else {
        if (!ok) return;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int c = col + 16 * q + 8 * h;
            if (vec && c + 8 <= n) {
                *reinterpret_cast<v4u *>(row + c) = out[q];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < n) row[c + e] = (uint16_t)(out[q][e / 2] >> (16 * (e & 1)));
            }
        }
    }
}
template <bool WHOLE>
__device__ __forceinline__ void load_block(const uint16_t *row, bool ok, int col, int n, bool vec, int h, v4u (&in)[2]) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int c = col + 16 * q + 8 * h;
        if constexpr (WHOLE) {
            in[q] = *reinterpret_cast<const v4u *>(row + c);
        } else {
            in[q] = v4u{0, 0, 0, 0};
            if (!ok) continue;
            if (vec && c + 8 <= n) {
                in[q] = *reinterpret_cast<const v4u *>(row + c);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < n) in[q][e / 2] |= (unsigned)row[c + e] << (16 * (e & 1));
            }
        }
    }
}

// The sixteen values a lane needs of a row vector (bias) for its part of the block at column `col`, as loaded: two a
// dword.  WHOLE: all columns exist and the vector lies on an 8-byte boundary.
template <bool WHOLE>
__device__ __forceinline__ void load_columns(const uint16_t *v, int col, int n, int h, v2u (&out)[4]) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int c = col + 8 * g + 4 * h;
        if constexpr (WHOLE) {
            out[g] = *reinterpret_cast<const v2u *>(v + c);
        } else {
            out[g] = v2u{0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < n) out[g][e / 2] |= (unsigned)v[c + e] << (16 * (e & 1));
        }
    }
}
__device__ __forceinline__ float column_value(const v2u (&c)[4], int v) {
    const unsigned d = c[v / 4][(v % 4) / 2];
    return __builtin_bit_cast(float, v & 1 ? d & 0xffff0000u : d << 16);
}

#endif  // __HIP_DEVICE_COMPILE__

// A bf16 matrix of the product, rows 16-byte aligned or not.
struct StoreBf16 {
    static constexpr bool kHeavy = false, kThinToo = true;
    uint16_t *out;
    long ld;
    bool vec;
#if __HIP_DEVICE_COMPILE__
    template <bool WHOLE, int TM, int TN>
    __device__ __forceinline__ void store(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane) const {
        const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + tm * 32 + l32;
#pragma unroll
            for (int tn = 0; tn < TN; ++tn) {
                float x[16];
#pragma unroll
                for (int v = 0; v < 16; ++v) x[v] = acc[tm][tn][v];
                store_block<WHOLE>(out + row * ld, row < m, col0 + tn * 32, n, vec, h, x);
            }
        }
    }
    template <int TM, int TN>
    __device__ __forceinline__ void operator()(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane,
                                               int) const {
        if (vec && row0 + 32 * TM <= m && col0 + 32 * TN <= n) store<true>(acc, row0, col0, m, n, lane);
        else store<false>(acc, row0, col0, m, n, lane);
    }
#endif
};

// An epilogue receives, once per wavefront, its accumulators and where they lie:
//     ep(acc, row0, col0, m, n, lane, split): rows row0 + 32 tm + l % 32, columns col0 + 32 tn + 8 g + 4 (l / 32) + e
template <class C, Layout LA, Layout LB, class Ep>
__global__ __launch_bounds__(C::kThreads) void gemm_bf16(Shape s, Ep ep) {
#if __HIP_DEVICE_COMPILE__
    extern __shared__ __align__(16) char lds_bytes[];
    int m = s.m, k = s.k;
    if (s.rows) {   // rows left out of a loss: the count is known on the device only
        const int have = __builtin_amdgcn_readfirstlane(*s.rows);
        if (LA == kAlongK) m = have < m ? have : m;
        else k = have < k ? have : k;
    }
    int tile_m, tile_n;
    mfma::tile_coords((s.m + C::BM - 1) / C::BM, (s.n + C::BN - 1) / C::BN, tile_m, tile_n);
    const int m0 = tile_m * C::BM, n0 = tile_n * C::BN;
    if (m0 >= m) return;
    const int k_begin = blockIdx.y * s.k_per_split;
    const int k_end = k_begin + s.k_per_split < k ? k_begin + s.k_per_split : k;
    v16f acc[C::TM][C::TN];
    if (k_begin < k_end) {
        tile_product<C, LA, LB>(s, m, k, m0, n0, k_begin, k_end, lds_bytes, acc);
    } else {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int j = 0; j < C::TN; ++j)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
    }
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    ep(acc, m0 + (wave / C::WN) * 32 * C::TM, n0 + (wave % C::WN) * 32 * C::TN, m, s.n, (int)(threadIdx.x & 63),
       (int)blockIdx.y);
#endif
}

// fp32 partial sums of split blockIdx.y (or the whole product when there is one): out[split][m][n], ld = n
struct StorePartial {
    static constexpr bool kHeavy = false, kThinToo = true;
    float *out;
    long split_stride;   // elements between the splits' matrices
    long ld;
    bool add;            // out += (one split only): a product summed over several calls
#if __HIP_DEVICE_COMPILE__
    template <int TM, int TN>
    __device__ __forceinline__ void operator()(const v16f (&acc)[TM][TN], int row0, int col0, int m, int n, int lane,
                                               int split) const {
        const int l32 = lane & 31, h = lane >> 5;
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int row = row0 + tm * 32 + l32;
            if (row >= m) continue;
            float *p = out + split * split_stride + row * ld;
#pragma unroll
            for (int tn = 0; tn < TN; ++tn)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int col = col0 + tn * 32 + g * 8 + h * 4;
                    float4 x = make_float4(acc[tm][tn][4 * g], acc[tm][tn][4 * g + 1], acc[tm][tn][4 * g + 2], acc[tm][tn][4 * g + 3]);
                    if (col + 4 <= n && (ld & 3) == 0) {
                        float4 *q = reinterpret_cast<float4 *>(p + col);
                        if (add) {
                            const float4 o = *q;
                            x.x += o.x, x.y += o.y, x.z += o.z, x.w += o.w;
                        }
                        *q = x;
                    } else {
                        const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (col + e < n) p[col + e] = add ? p[col + e] + v[e] : v[e];
                    }
                }
        }
    }
#endif
};

template <class C, Layout LA, Layout LB, class Ep>
int launch_gemm_bf16(const Shape &s, int splits, const Ep &ep, const char *who) {
    const long tiles = (long)((s.m + C::BM - 1) / C::BM) * ((s.n + C::BN - 1) / C::BN);
    if (tiles > 0x7fffffffL || splits > 65535) return fail(SWC_HIP_EINVAL, "%s: too many tiles", who);
    note_kernel("gemm_bf16<%dx%d,%d,%d,%s%s> x%d", C::BM, C::BN, C::SA, C::SB, LA == kAlongK ? "k" : "m",
                LB == kAlongK ? "k" : "n", splits);
    auto kern = gemm_bf16<C, LA, LB, Ep>;
    static bool attr_set = false;
    if (!attr_set) {
        SWC_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                        C::kLdsBytes));
        attr_set = true;
    }
    kern<<<dim3((unsigned)tiles, (unsigned)splits), C::kThreads, C::kLdsBytes, stream()>>>(s, ep);
    SWC_LAUNCH_CHECK();
    return SWC_HIP_OK;
}

} // namespace mfma16
} // namespace swc_hip
