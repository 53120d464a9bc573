// 16-bit matrix products on the matrix cores (v_mfma_f32_16x16x32), shared by the kernels of the linear cross entropy.
//
// A workgroup computes a BM x BN tile of D[m][n] = sum_k A[m][k] B[n][k] in steps of 32 k.  Both operands of a step are copied
// straight into LDS (16 bytes per lane, no registers), three steps ahead into a ring of four stages; a step issues its copies between
// its matrix instructions (issued together in front of them they held every wave for the time the address unit takes), and the steps in
// the middle are unrolled over the ring (its bookkeeping cost 8 %).  In the cross entropy of 8192 x 32000 x 1024 bf16 these products reach
// 0.85 to 1.09 PFLOP/s, the library's product of 8192^3 1.24.  Either operand may lie in memory
//   * k-contiguous ([ext][k]: a row of 32 k is 64 bytes = 4 chunks), or
//   * k-major ([k][ext]: fragments are then read with the transposing LDS read, 4 k x 16 columns for 16 lanes).
// Chunks are stored permuted (k-contiguous: chunk c of row r at c ^ (r / 4 & 3); k-major: 32-byte unit u of row k at u ^ f(k)), so that
// the 64 lanes of a fragment read touch all banks evenly; the copy applies the permutation to its source addresses.  Nothing outside a
// tensor is read.
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

constexpr int kStepK = 32;
constexpr int kStages = 4;

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

// Copies the ext0 ... ext0 + EXT - 1, k0 ... k0 + 31 tile.  A lane's chunk lies at the same offset from the tile's first element in every
// step, so a step whose 32 k all exist costs no vector arithmetic: a scalar base moves on.  Chunks outside `ext` repeat one that exists
// (they reach outputs that are not there); the last, partial step takes chunks behind k_end from a block of zeros.
template <bool KMAJOR, int EXT, int THREADS>
struct TileCopy {
    static constexpr int CH = EXT * 4 / THREADS;
    static_assert(CH * THREADS == EXT * 4, "whole chunks per lane");
    uint32_t off[CH];           // bytes

    __device__ __forceinline__ static void place(int j, int& e, int& k) {
        const int q = j * THREADS + threadIdx.x;
        if (!KMAJOR) {
            const int row = q >> 2;
            e = row;
            k = ((q & 3) ^ ((row >> 2) & 3)) * 8;
        } else {
            constexpr int CPR = EXT / 8;
            const int kr = q / CPR, slot = q % CPR;
            e = (((((slot >> 1) ^ ((kr & 3) | ((kr >> 1) & 4))) << 1) | (slot & 1))) * 8;
            k = kr;
        }
    }
    __device__ __forceinline__ void aim(const Operand& o, int ext0) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            int e, k;
            place(j, e, k);
            if (ext0 + e >= o.ext) e = KMAJOR ? 0 : o.ext - 1 - ext0;
            off[j] = (uint32_t)(KMAJOR ? k * (int)o.ld + e : e * (int)o.ld + k) * 2u;
        }
    }
    // the tile's first element, and how far the next step's is
    __device__ __forceinline__ static const char* base(const Operand& o, int part, int ext0, int k0) {
        return static_cast<const char*>(o.base) + 2 * ((int64_t)part * o.part + (KMAJOR ? (int64_t)k0 * o.ld + ext0 : (int64_t)ext0 * o.ld + k0));
    }
    __device__ __forceinline__ static int64_t advance(const Operand& o) { return 2 * (KMAJOR ? kStepK * o.ld : (int64_t)kStepK); }
    __device__ __forceinline__ void copy_whole(const char* from, char* lds) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int j = 0; j < CH; ++j)
            __builtin_amdgcn_global_load_lds((glb_cvoid_t*)(from + off[j]), (lds_void16_t*)(lds + (j * THREADS + wave * 64) * 16), 16, 0, 0);
    }
    // k0: the step's first k
    __device__ __forceinline__ void copy(const char* from, int k0, int k_end, char* lds) const {
        if (k0 + kStepK <= k_end) return copy_whole(from, lds);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            int e, k;
            place(j, e, k);
            const void* src = k0 + k < k_end ? static_cast<const void*>(from + off[j]) : static_cast<const void*>(kZeroChunk);
            __builtin_amdgcn_global_load_lds((glb_cvoid_t*)src, (lds_void16_t*)(lds + (j * THREADS + wave * 64) * 16), 16, 0, 0);
        }
    }
};

// the fragments of rows (columns) ext0 + 16 t ... + 15, t = t0 ... t0 + 3, of a tile
template <bool KMAJOR, int EXT>
__device__ __forceinline__ void tile_frags4(const char* lds, int ext0, int t0, s16x8 (&out)[4]) {
    const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
    // the stage's address as a scalar of its own: with the unrolled steps' stages folded in, every fragment's address of every stage is
    // kept in a register (26 of them spilled)
    uint32_t stage = (uint32_t)(uintptr_t)(lds_void16_t*)lds;
    asm volatile("" : "+s"(stage));
    if (!KMAJOR) {
        typedef __attribute__((address_space(3))) const s16x8 lds_s16x8;
        const uint32_t at = stage + (ext0 + t0 * 16 + i) * 64 + ((g ^ (i >> 2)) << 4);
#pragma unroll
        for (int t = 0; t < 4; ++t) out[t] = *(lds_s16x8*)(uintptr_t)(at + t * 1024);
    } else {
        // In assembly: in front of the builtin the compiler drains every copy to LDS that is in flight (it cannot tell which stage a
        // transposing read touches), which would undo the overlap.  The reads are waited for in the same block; the outputs are
        // early-clobbered, so no read in flight lands on an address of a later one.
        const int f = (i >> 2) | ((g & 1) << 2);
        const uint32_t row = (g * 8 + (i >> 2)) * (EXT * 2) + (i & 3) * 8;
        uint32_t at[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) at[t] = stage + (row + (((ext0 >> 4) + t0 + t) ^ f) * 32);
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

// two numbers rounded to nearest into one register
template <typename E>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<bf16_t>(float lo, float hi) {
    const vec_t<bf16_t, 2> v = {(bf16_t)lo, (bf16_t)hi};
    return __builtin_bit_cast(uint32_t, v);
}
template <>
__device__ __forceinline__ uint32_t pack2<f16_t>(float lo, float hi) {
    uint32_t v;         // the compiler converts one by one and permutes where both halves are needed again
    asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(v) : "v"(lo), "v"(hi));
    return v;
}
// v - h for both halves of a register of two fp16 numbers, exactly: the mixed fma reads the halves as they lie, where conversions take
// two instructions more per element
__device__ __forceinline__ void minus_halves(uint32_t h, float& lo, float& hi) {
    asm("v_fma_mix_f32 %0, %1, -1.0, %0 op_sel_hi:[1,0,0]" : "+v"(lo) : "v"(h));
    asm("v_fma_mix_f32 %0, %1, -1.0, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(hi) : "v"(h));
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
    static constexpr int kLds = kStages * kStage;
    static constexpr int kCopies = (BM + BN) * 4 / kThreads;        // copies per lane and step

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

    TileCopy<KMA, BM, kThreads> ca;
    TileCopy<KMB, BN, kThreads> cb;

    // wait until this wave's copies but the `NEWER` last steps' have landed and its fragments have been read, then for the other waves:
    // the oldest step in flight is there for everyone, and the stage before it may be overwritten
    template <int NEWER>
    __device__ __forceinline__ static void arrive() {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(NEWER * kCopies) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }

    __device__ __forceinline__ void multiply4(int m, const s16x8 (&fa)[4], const s16x8 (&fb)[4], f32x4 (&acc)[MT][NT]) const {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[m + i][n] = mfma16<E>(fa[i], fb[n], acc[m + i][n]);
        __builtin_amdgcn_s_setprio(0);
    }

    // a step in the middle: its stage is known, three more steps follow, and the one it copies is whole
    template <int STAGE, typename Extra>
    __device__ __forceinline__ void middle_step(const char* pa, const char* pb, int pair, f32x4 (&acc)[MT][NT], Extra&& extra) const {
        constexpr int kAhead = (STAGE + kStages - 1) % kStages;
        arrive<2>();
        const char* sa = lds + STAGE * kStage;
        s16x8 fb[4], fa[MT / 4][4];
        tile_frags4<KMB, BN>(sa + kBytesA, n_wave, 0, fb);
        tile_frags4<KMA, BM>(sa, m_wave, 0, fa[0]);
        ca.copy_whole(pa, lds + kAhead * kStage);
        multiply4(0, fa[0], fb, acc);
        if (MT > 4) tile_frags4<KMA, BM>(sa, m_wave, 4, fa[MT / 4 - 1]);
        cb.copy_whole(pb, lds + kAhead * kStage + kBytesA);
        if (MT > 4) multiply4(MT - 4, fa[MT / 4 - 1], fb, acc);
        extra(STAGE, pair);
    }

    // the tile being multiplied: its corner and k steps; the next step to be copied: its pair, its k step and where it begins
    int m_at, n_at, k_first, ksteps, cp, ck;
    const char *pa, *pb;
    int64_t da, db;             // from one k step to the next

    __device__ __forceinline__ void next() {
        if (++ck == ksteps) {
            ck = 0;
            ++cp;
            pa = ca.base(a, pair_a(pairs, cp), m_at, k_first);
            pb = cb.base(b, pair_b(pairs, cp), n_at, k_first);
        } else {
            pa += da;
            pb += db;
        }
    }

    // starts the product of the tile at m0, n0 over k0 ... k1 - 1 (k0 a multiple of 32): its first copies.  The ring must be free: at the
    // start, or after multiply().  What a wave stores or loads between the two is newer than these copies, so that waiting for all but
    // the newest operations still waits for them.
    __device__ __forceinline__ void begin(int m0, int n0, int k0, int k1) {
        m_at = m0;
        n_at = n0;
        k_first = k0;
        ksteps = (k1 - k0 + kStepK - 1) / kStepK;
        if (ksteps <= 0) return;
        ca.aim(a, m0);
        cb.aim(b, n0);
        cp = ck = 0;
        da = ca.advance(a);
        db = cb.advance(b);
        pa = ca.base(a, pair_a(pairs, 0), m0, k0);
        pb = cb.base(b, pair_b(pairs, 0), n0, k0);
        for (int s = 0; s < kStages - 1 && s < ksteps * pairs; ++s, next()) {
            ca.copy(pa, k0 + ck * kStepK, k_end, lds + s * kStage);
            cb.copy(pb, k0 + ck * kStepK, k_end, lds + s * kStage + kBytesA);
        }
    }

    // acc += the product begun; extra(stage, pair) sees every stage before it is given up
    template <typename Extra>
    __device__ __forceinline__ void multiply(f32x4 (&acc)[MT][NT], Extra&& extra) {
        const int total = ksteps * pairs, k0 = k_first;
        if (total <= 0) return;
        int pair = 0, ks = 0;
        auto done = [&]() {
            if (++ks == ksteps) {
                ks = 0;
                ++pair;
            }
        };
        // whole steps, four at a time; a partial one can only be the last of a pair
        const int whole = k0 + ksteps * kStepK <= k_end ? total : (pairs == 1 ? total - 1 : 0);
        int s = 0;
        for (; s + 2 * kStages - 1 <= whole; s += kStages) {
            middle_step<0>(pa, pb, pair, acc, extra); next(); done();
            middle_step<1>(pa, pb, pair, acc, extra); next(); done();
            middle_step<2>(pa, pb, pair, acc, extra); next(); done();
            middle_step<3>(pa, pb, pair, acc, extra); next(); done();
        }
        for (; s < total; ++s, done()) {
            const int left = total - 1 - s;
            if (left >= 2) arrive<2>();
            else if (left == 1) arrive<1>();
            else arrive<0>();
            const char* sa = lds + (s % kStages) * kStage;
            if (left >= kStages - 1) {
                char* ahead = lds + ((s + kStages - 1) % kStages) * kStage;
                ca.copy(pa, k0 + ck * kStepK, k_end, ahead);
                cb.copy(pb, k0 + ck * kStepK, k_end, ahead + kBytesA);
                next();
            }
            s16x8 fb[4];
            tile_frags4<KMB, BN>(sa + kBytesA, n_wave, 0, fb);
#pragma unroll
            for (int m = 0; m < MT; m += 4) {
                s16x8 fa[4];
                tile_frags4<KMA, BM>(sa, m_wave, m, fa);
                multiply4(m, fa, fb, acc);
            }
            extra(s % kStages, pair);
        }
        // the ring may be used again
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
};

// ---- fp32 products on the fp32 matrix instructions -------------------------------------------------------------------------------------
//
// For operands that two fp16 parts do not hold: v_mfma_f32_16x16x4, an eighth of the rate, over the full range of fp32.  Fragments come
// straight from memory in steps of 16 k (16 rows of 64 bytes each where k is contiguous), and stay in the caches between the workgroups.
// D lies as with the 16-bit instructions; A and B hold one k of row l % 16 a lane: in instruction j of a step, k = 4 (l / 16) + j.

struct Operand32 {
    const float* base;
    int64_t ld, ext;        // ext: rows of D (columns) that exist
};
__device__ __forceinline__ f32x4 mfma32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// elements k ... k + 3 of row (column) e: 0 where e or k is outside, or k is not live
template <bool KMAJOR, typename Live>
__device__ __forceinline__ void load32(const Operand32& o, int64_t e, int64_t k, int64_t k_end, Live&& live, float (&out)[4]) {
    const bool in = e < o.ext;
    if (!KMAJOR && in && k + 4 <= k_end) {
        __builtin_memcpy(out, o.base + e * o.ld + k, 16);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = in && k + j < k_end && (!KMAJOR || live(k + j)) ? o.base[KMAJOR ? (k + j) * o.ld + e : e * o.ld + k + j] : 0.f;
    }
}

// acc += A B over k0 <= k < k1 for this wave's rows m_wave ... and columns n_wave ...; live(k): whether k counts where A is k-major (a dead
// one may hold anything); extra(B's elements) sees every step.  The order of the sums depends on k0 alone, and on nothing of A and B: a
// logit has the same bits wherever it is computed
template <bool KMA, bool KMB, int MT, int NT, typename Live, typename Extra>
__device__ __forceinline__ void product32(const Operand32& a, const Operand32& b, int64_t m_wave, int64_t n_wave, int64_t k0, int64_t k1,
                                          f32x4 (&acc)[MT][NT], Live&& live, Extra&& extra) {
    const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
    for (int64_t k = k0; k < k1; k += 16) {
        float fa[MT][4], fb[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) load32<KMB>(b, n_wave + n * 16 + i, k + 4 * g, k1, [](int64_t) { return true; }, fb[n]);
#pragma unroll
        for (int m = 0; m < MT; ++m) load32<KMA>(a, m_wave + m * 16 + i, k + 4 * g, k1, live, fa[m]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[m][n] = mfma32(fa[m][j], fb[n][j], acc[m][n]);
        extra(fb);
    }
}

}  // namespace cnf
