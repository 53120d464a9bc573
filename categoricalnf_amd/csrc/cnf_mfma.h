// 16-bit matrix products on the matrix cores (v_mfma_f32_16x16x32), shared by the kernels of the linear cross entropy.
//
// A workgroup computes a BM x BN tile of D[m][n] = sum_k A[m][k] B[n][k] in steps of 64 k.  Both operands of a step are copied
// straight into LDS (16 bytes per lane, no registers) while the step before it is multiplied.  Either operand may lie in memory
//   * k-contiguous ([ext][k]: a row of 64 k is 128 bytes = 8 chunks), or
//   * k-major ([k][ext]: fragments are then read with the transposing LDS read, 4 k x 16 columns for 16 lanes).
// Chunks are stored permuted (k-contiguous: chunk c of row r at c ^ (r & 7); k-major: 32-byte unit u of row k at u ^ f(k)), so that
// the 64 lanes of a fragment read touch all banks evenly; the copy applies the permutation to its source addresses.  Chunks outside
// an operand are copied from a block of zeros: edges cost no branch in the inner loop, and nothing outside a tensor is read.
//
// Fragment layout (lane l, g = l / 16): A and B hold k = 8 g ... 8 g + 7 of row l % 16; D holds n = l % 16, m = 4 g ... 4 g + 3.
#pragma once
#include "cnf_dtype.h"

namespace cnf {

typedef __attribute__((address_space(1))) const void glb_cvoid_t;
typedef __attribute__((address_space(3))) void lds_void16_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kStepK = 64;

__device__ const uint32_t kZeroChunk[4] = {0, 0, 0, 0};

template <typename E>
__device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma16<bf16_t>(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec_t<bf16_t, 8>, a), __builtin_bit_cast(vec_t<bf16_t, 8>, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma16<f16_t>(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec_t<f16_t, 8>, a), __builtin_bit_cast(vec_t<f16_t, 8>, b), c, 0, 0, 0);
}

// One operand: `parts` arrays of 16-bit elements, `part` elements apart (fp32 values split into two fp16 parts; 16-bit values: one).
// ld is a multiple of 8 and the base 16-byte aligned; a row has room for its extent rounded up to 8.
struct Operand {
    const void* base;
    int64_t ld, part;
    int ext;            // rows of D (columns) that exist
};

// copies the ext0 ... ext0 + EXT - 1, k0 ... k0 + 63 tile
template <bool KMAJOR, int EXT, int THREADS>
__device__ __forceinline__ void tile_copy(const Operand& o, int part, int ext0, int k0, int k_end, char* lds) {
    constexpr int CH = EXT * 8 / THREADS;
    static_assert(CH * THREADS == EXT * 8, "whole chunks per lane");
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint16_t* base = static_cast<const uint16_t*>(o.base) + (int64_t)part * o.part;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int q = j * THREADS + tid;
        int e, k;
        int64_t off;
        if (!KMAJOR) {
            const int row = q >> 3, c = (q & 7) ^ (row & 7);
            e = ext0 + row;
            k = k0 + c * 8;
            off = (int64_t)e * o.ld + k;
        } else {
            constexpr int CPR = EXT / 8;
            const int kr = q / CPR, slot = q % CPR;
            const int c = (((slot >> 1) ^ ((kr & 3) | ((kr >> 1) & 4))) << 1) | (slot & 1);
            e = ext0 + c * 8;
            k = k0 + kr;
            off = (int64_t)k * o.ld + e;
        }
        const void* src = (e < o.ext && k < k_end) ? static_cast<const void*>(base + off) : static_cast<const void*>(kZeroChunk);
        __builtin_amdgcn_global_load_lds((glb_cvoid_t*)src, (lds_void16_t*)(lds + (j * THREADS + wave * 64) * 16), 16, 0, 0);
    }
}

// the fragments of rows (columns) ext0 + 16 t ... + 15, t = t0 ... t0 + 3, k = 32 kk ... 32 kk + 31 of a tile
template <bool KMAJOR, int EXT>
__device__ __forceinline__ void tile_frags4(const char* lds, int ext0, int t0, int kk, s16x8 (&out)[4]) {
    const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
    if (!KMAJOR) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
            out[t] = *reinterpret_cast<const s16x8*>(lds + (ext0 + (t0 + t) * 16 + i) * 128 + (((kk * 4 + g) ^ (i & 7)) << 4));
    } else {
        // In assembly: in front of the builtin the compiler drains every copy to LDS that is in flight (it cannot tell which stage a
        // transposing read touches), which would undo the overlap.  The reads are waited for in the same block; the outputs are
        // early-clobbered, so no read in flight lands on an address of a later one.
        const int f = (i >> 2) | ((g & 1) << 2);
        const uint32_t row = (uint32_t)(uintptr_t)(lds_void16_t*)lds + (kk * 32 + g * 8 + (i >> 2)) * (EXT * 2) + (i & 3) * 8;
        uint32_t at[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) at[t] = row + (((ext0 >> 4) + t0 + t) ^ f) * 32;
        s16x4 lo[4], hi[4];
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8\n\t"
            "ds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
            "ds_read_b64_tr_b16 %2, %9\n\t"
            "ds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
            "ds_read_b64_tr_b16 %4, %10\n\t"
            "ds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
            "ds_read_b64_tr_b16 %6, %11\n\t"
            "ds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]), "=&v"(hi[3])
            : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(4 * EXT * 2)
            : "memory");
#pragma unroll
        for (int t = 0; t < 4; ++t) out[t] = __builtin_shufflevector(lo[t], hi[t], 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// Which parts are multiplied: 16-bit values (0, 0); fp32 values, scaled so that the largest of their tensor lies in 2^14 ... 2^15, as
// x0 + x1 (each the fp16 nearest to what is left: 2^-23 of the value, or 2^-25 in the scaled unit, stays out): (0, 1), (1, 0), (0, 0).
// What is dropped, x1 y1, is below 2^-22 of |x| |y| and has either sign; fp32 products and sums round by 2^-24 each.
__device__ __forceinline__ int pair_a(int pairs, int s) { return pairs == 3 && s == 1 ? 1 : 0; }
__device__ __forceinline__ int pair_b(int pairs, int s) { return pairs == 3 && s == 0 ? 1 : 0; }

template <typename E, bool KMA, bool KMB, int BM, int BN, int WM, int WN>
struct TileProduct {
    static constexpr int kThreads = WM * WN * 64;
    static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
    static constexpr int kBytesA = BM * kStepK * 2, kBytesB = BN * kStepK * 2, kStage = kBytesA + kBytesB;
    static constexpr int kLds = 2 * kStage;
    static constexpr int kCopies = (BM + BN) * 8 / kThreads;        // copies in flight per lane and step

    static_assert(NT == 4 && MT % 4 == 0, "fragments are read in fours");

    const Operand a, b;
    const int pairs, k_end;         // k < k_end
    char* lds;
    int m_wave, n_wave;             // this wave's corner in the tile

    __device__ __forceinline__ TileProduct(const Operand& a_, const Operand& b_, int pairs_, int k_end_, char* lds_)
        : a(a_), b(b_), pairs(pairs_), k_end(k_end_), lds(lds_) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        m_wave = (wave % WM) * (BM / WM);
        n_wave = (wave / WM) * (BN / WN);
    }

    __device__ __forceinline__ void copy(int m0, int n0, int pair, int k0, int stage) const {
        char* s = lds + stage * kStage;
        tile_copy<KMA, BM, kThreads>(a, pair_a(pairs, pair), m0, k0, k_end, s);
        tile_copy<KMB, BN, kThreads>(b, pair_b(pairs, pair), n0, k0, k_end, s + kBytesA);
    }

    // wait until all copies but the `newer` last ones of this lane have landed, then for the other waves
    template <int NEWER>
    __device__ __forceinline__ static void landed() {
        if (NEWER == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else if (NEWER == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else if (NEWER == 6) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        static_assert(NEWER == 0 || NEWER == 4 || NEWER == 6 || NEWER == 8, "a wait for this many copies is missing");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    // every wave has read its fragments of the stage: it may be overwritten
    __device__ __forceinline__ static void read_done() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    __device__ __forceinline__ void multiply(int stage, f32x4 (&acc)[MT][NT]) const {
        const char* sa = lds + stage * kStage;
        const char* sb = sa + kBytesA;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            s16x8 fb[4];
            tile_frags4<KMB, BN>(sb, n_wave, 0, kk, fb);
#pragma unroll
            for (int m = 0; m < MT; m += 4) {
                s16x8 fa[4];
                tile_frags4<KMA, BM>(sa, m_wave, m, kk, fa);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[m + i][n] = mfma16<E>(fa[i], fb[n], acc[m + i][n]);
            }
        }
    }

    // acc += the tile's product over k0 ... k1 - 1 (k0 a multiple of 64); extra(stage) sees every stage before it is given up
    template <typename Extra>
    __device__ __forceinline__ void run(int m0, int n0, int k0, int k1, f32x4 (&acc)[MT][NT], Extra&& extra) const {
        const int ksteps = (k1 - k0 + kStepK - 1) / kStepK, total = ksteps * pairs;
        if (total <= 0) return;
        int pair = 0, ks = 0, stage = 0;
        copy(m0, n0, 0, k0, 0);
        for (int s = 0; s < total; ++s) {
            if (++ks == ksteps) {
                ks = 0;
                ++pair;
            }
            if (s + 1 < total) {
                copy(m0, n0, pair, k0 + ks * kStepK, stage ^ 1);
                landed<kCopies>();
            } else {
                landed<0>();
            }
            multiply(stage, acc);
            extra(stage);
            read_done();
            stage ^= 1;
        }
    }
};

}  // namespace cnf
