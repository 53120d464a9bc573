// Linear cross entropy of few features: forward, gradient of the rows, gradient of the weights (formulas: cnf_linear_ce.hip).
//
// A workgroup of four waves keeps 128 rows (for dw: 128 vocabulary entries) as matrix-core operands in registers, 32 a wave, and walks
// through its part of the other side in steps of 64, copied into LDS one step ahead.  Per step and wave:
//   S = walk . own^T            (three fp16 products for fp32 operands, one for 16-bit ones)
//   forward:  running maximum and sum per lane;  backward:  d from S in place, and  out^T += walk^T . d
// S has four consecutive walk entries of one own entry per lane (fragment layout in cnf_mfma.h); two 16-row tiles of it are exactly
// the eight k of a lane in the second product, whose other operand is the transposed LDS read of the same tile: d never moves
// between lanes.  For fp32 d is split into two fp16 parts there.
//
// Bound by the matrix cores and the vector work beside them (exponentials, splitting): 5 products of 2 R V H operations against the
// 3 of the definition — the logits are computed three times — but nothing of size R x V is written or read.  36864 x 10000 x 64 fp32:
// forward 180 us (785 TF of fp16 products), dx 280 us (1010 TF), dw 344 us (820 TF), with fp32 products of wide operands 1.41, 2.02 and 2.24
// ms; in bf16 117, 151 and 223 us.  Matrix cores busy 40 - 50 % of the cycles, vector
// units 50 - 60 %, and a step's products wait for its exponentials.  128 rows a workgroup: the tile of the other side is read from LDS
// once for 32 rows of a wave; 64 rows a wave would leave registers for one wave per SIMD.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "cnf_linear_ce_narrow.h"

namespace cnf {

// LDS tile: [PARTS][64][HP] 16-bit elements; 16-byte chunk c of row r at c ^ f(r): row reads (16 rows, one chunk each) and transposing
// reads (16 rows, 32 bytes each) both touch every bank equally often
template <int HP>
__device__ __forceinline__ int narrow_swizzle(int row) {
    return HP == 32 ? (row >> 2) & 3 : (HP == 64 ? row & 7 : row & 15);
}

template <int HP, int PARTS>
struct NarrowTile {
    static constexpr int kChunks = HP / 8;
    static constexpr int kPart = kNarrowWalk * HP * 2;              // bytes
    static constexpr int kBytes = PARTS * kPart;
    static constexpr int kCopies = PARTS * kNarrowWalk * kChunks / kBlock;

    __device__ static void copy(const Operand& o, int64_t m0, int hidden, char* lds) {
        const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const uint16_t* base = static_cast<const uint16_t*>(o.base);
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
            const int q = j * kBlock + tid;
            const int part = j * kBlock / (kNarrowWalk * kChunks);
            const int row = (q / kChunks) % kNarrowWalk, c = (q % kChunks) ^ narrow_swizzle<HP>(row);
            const int64_t e = m0 + row;
            const void* src = (e < o.ext && c * 8 < hidden) ? static_cast<const void*>(base + (int64_t)part * o.part + e * o.ld + c * 8)
                                                            : static_cast<const void*>(kZeroChunk);
            __builtin_amdgcn_global_load_lds((glb_cvoid_t*)src, (lds_void16_t*)(lds + (j * kBlock + wave * 64) * 16), 16, 0, 0);
        }
    }
    // A tile whose rows and chunks all exist: a copy's rows lie kRows apart, which the swizzle does not see, so a lane has one offset for
    // all of them and the rest is scalar (dw at 36864 x 10000 x 64 fp32: 379 -> 369 us)
    static constexpr int kRows = kBlock / kChunks;
    __device__ static uint32_t lane_offset(const Operand& o) {
        const int row = threadIdx.x / kChunks, c = (threadIdx.x % kChunks) ^ narrow_swizzle<HP>(row);
        return (uint32_t)(row * (int)o.ld + c * 8) * 2u;
    }
    __device__ static void copy_whole(const Operand& o, int64_t m0, uint32_t offset, char* lds) {
        static_assert(kRows % 16 == 0 && kNarrowWalk % kRows == 0, "whole swizzles and parts");
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
            const int part = j * kRows / kNarrowWalk, row = j * kRows % kNarrowWalk;
            const char* base = static_cast<const char*>(o.base) + 2 * (part * o.part + (m0 + row) * o.ld);
            __builtin_amdgcn_global_load_lds((glb_cvoid_t*)(base + offset), (lds_void16_t*)(lds + (j * kBlock + wave * 64) * 16), 16, 0, 0);
        }
    }
    // rows row0 ... row0 + 15, k = 32 kk ...
    __device__ static s16x8 frag(const char* lds, int part, int row0, int kk) {
        const int l = threadIdx.x & 63, row = row0 + (l & 15), c = kk * 4 + (l >> 4);
        return *reinterpret_cast<const s16x8*>(lds + part * kPart + row * (HP * 2) + ((c ^ narrow_swizzle<HP>(row)) << 4));
    }
    // Transposed: columns 16 h ..., k = 32 rows, lane group g holding rows 4 g ... + 3 and 16 + 4 g ... + 3.  The
    // swizzle of a row depends on its place within 16 rows only, so one address per h serves every part and row block through the
    // instruction's offset (held per block, they took 80 registers more).
    __device__ static uint32_t frag_t_base(int h) {
        const int l = threadIdx.x & 63, i = l & 15, row = (l >> 4) * 4 + (i >> 2), c = h * 2 + ((i & 3) >> 1);
        return row * (HP * 2) + ((c ^ narrow_swizzle<HP>(row)) << 4) + (i & 1) * 8;
    }
    // N of them (2 or 4); in assembly, waited for in the same block, like the transposing reads of cnf_mfma.h
    template <int PART, int N>
    __device__ static void frag_t(const uint32_t* base, uint32_t tile_at, s16x8 (&out)[N]) {
        constexpr int kOff = PART * kPart;
        static_assert(N == 2 || N == 4, "two or four");
        uint32_t at[N];
#pragma unroll
        for (int h = 0; h < N; ++h) at[h] = base[h] + tile_at;
        s16x4 v[N][2];
        if constexpr (N == 2)
            asm volatile(
                "ds_read_b64_tr_b16 %0, %4 offset:%6\n\t"
                "ds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
                "ds_read_b64_tr_b16 %2, %5 offset:%6\n\t"
                "ds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1])
                : "v"(at[0]), "v"(at[1]), "n"(kOff), "n"(kOff + 16 * HP * 2)
                : "memory");
        else
            asm volatile(
                "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
                "ds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                "ds_read_b64_tr_b16 %2, %9 offset:%12\n\t"
                "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
                "ds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                "ds_read_b64_tr_b16 %6, %11 offset:%12\n\t"
                "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[2][0]), "=&v"(v[2][1]), "=&v"(v[3][0]), "=&v"(v[3][1])
                : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(kOff), "n"(kOff + 16 * HP * 2)
                : "memory");
#pragma unroll
        for (int h = 0; h < N; ++h) out[h] = __builtin_shufflevector(v[h][0], v[h][1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// fn(integral_constant 0) ... fn(integral_constant N - 1)
template <typename Fn, int... I>
__device__ __forceinline__ void static_for_impl(Fn&& fn, std::integer_sequence<int, I...>) {
    (fn(std::integral_constant<int, I>{}), ...);
}
template <int N, typename Fn>
__device__ __forceinline__ void static_for(Fn&& fn) {
    static_for_impl(static_cast<Fn&&>(fn), std::make_integer_sequence<int, N>{});
}

// forward: two blocks of 16 walk entries (the lane's: m0 + 16 t + i) enter the running maximum and sum of the lane's own rows own0 + 16 n
template <int NT>
__device__ __forceinline__ void lse_step(const NarrowArgs& a, f32x4 (&sc)[2][NT], const float (&back)[NT], const f32x4 (&bias)[2], int64_t m0,
                                         int64_t own0, const int (&want)[NT], float (&mx)[NT], float (&sum)[NT], float (&own_logit)[NT]) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[t][n][i] = __builtin_fmaf(sc[t][n][i], back[n], bias[t][i]);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int64_t at = want[n] - m0;
        if (want[n] >= 0 && at >= 0 && at < 32 && (at & 15) < 4) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at == t * 16 + i) own_logit[n] = sc[t][n][i];
            if (a.splits > 1) a.target_logit[own0 + n * 16] = own_logit[n];
        }
        float top = mx[n];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[t][n][i]);
        const float ref = top == -INFINITY ? 0.f : top;
        float q = sum[n] * __builtin_amdgcn_exp2f(mx[n] - ref);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) q += __builtin_amdgcn_exp2f(sc[t][n][i] - ref);
        sum[n] = q;
        mx[n] = top;
    }
}

// The walk with fp32 products of the operands as they were given (kRowSpan), read where they lie; no lift, and nothing is split
template <int HT, int NT, NarrowJob JOB>
__device__ __forceinline__ void narrow_walk32(const NarrowArgs& a, int64_t first, int64_t last, int64_t n_wave, const RowState (&st)[NT],
                                              const float (&bias_n)[NT], const int (&want)[NT], float (&mx)[NT], float (&sum)[NT],
                                              float (&own_logit)[NT], f32x4 (&acc)[HT][NT]) {
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    float back[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) back[n] = kLog2e;
    for (int64_t m_half = first * kNarrowWalk; m_half < last * kNarrowWalk; m_half += 32) {
        f32x4 sc[2][NT];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        product32<false, false, 2, NT>(a.walk32, a.own32, m_half, n_wave, 0, a.hidden, sc, [](int64_t) { return true; }, [](const float (&)[NT][4]) {});
        const int64_t m0 = m_half + g * 4;
        f32x4 bias[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) bias[t] = JOB == kNarrowDw ? f32x4{0.f, 0.f, 0.f, 0.f} : *reinterpret_cast<const f32x4*>(a.bias + m0 + t * 16);
        if (JOB == kNarrowLse) {
            lse_step(a, sc, back, bias, m0, n_wave + col, want, mx, sum, own_logit);
            continue;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t at = m0 + (e / 4) * 16 + e % 4;                // the walk entry, one of this lane's eight
            // the rows' records are padded to whole tiles
            const RowState q = JOB == kNarrowDw ? a.state[at] : RowState{0.f, 0.f, 0.f, 0};
            float v[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const RowState& row = JOB == kNarrowDw ? q : st[n];
                const float b = JOB == kNarrowDw ? bias_n[n] : bias[e / 4][e % 4];
                v[n] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e / 4][n][e % 4], kLog2e, b) - row.m2) * row.inv_s;
                if (row.target == (JOB == kNarrowDw ? n_wave + n * 16 + col : at)) v[n] -= 1.f;
                if (JOB == kNarrowDw) v[n] *= row.g;                     // dx: at the end
                if (row.target < 0) v[n] = 0.f;                          // an ignored row's logits may be anything
                if (JOB == kNarrowDw) sum[n] += v[n];
            }
            const bool live = at < a.walk32.ext && (JOB == kNarrowDx || q.target >= 0);
#pragma unroll
            for (int h = 0; h < HT; ++h) {
                const int k = h * 16 + col;
                const float f = live && k < a.hidden ? a.walk32.base[at * a.walk32.ld + k] : 0.f;
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[h][n] = mfma32(f, v[n], acc[h][n]);
            }
        }
    }
}

template <typename E, int PARTS, int HP, NarrowJob JOB>
__global__ __launch_bounds__(kBlock, HP <= 64 ? 3 : 2) void ce_narrow_kernel(const NarrowArgs a) {
    typedef NarrowTile<HP, PARTS> Tile;
    constexpr int NT = 2, KK = HP / 32, HT = HP / 16;
    constexpr int HB = HT < 4 || JOB == kNarrowDw ? 2 : 4;           // fragments read together; dw has registers for two
    constexpr int kHalves = JOB == kNarrowLse ? 2 : 1;               // halves of a step in flight: the gradients have registers for one
    constexpr int kAux = JOB == kNarrowDw ? kNarrowWalk * 16 : kNarrowWalk * 4;       // row records, or biases
    constexpr int kStage = Tile::kBytes + kAux;
    __shared__ __align__(16) char lds[2 * kStage];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = blockIdx.x % a.splits;
    const int64_t own_n = JOB == kNarrowDw ? a.vocab : a.rows, walk_n = JOB == kNarrowDw ? a.rows : a.vocab;
    const int64_t n_wave = (int64_t)(blockIdx.x / a.splits) * kNarrowOwn + wave * (NT * 16);
    const int64_t tiles = (walk_n + kNarrowWalk - 1) / kNarrowWalk;
    const int64_t first = tiles * split / a.splits, last = tiles * (split + 1) / a.splits;

    const uint32_t offset = Tile::lane_offset(a.walk);
    auto copy = [&](int64_t tile, int stage) {
        char* s = lds + stage * kStage;
        if (a.hidden > HP - 8 && (tile + 1) * kNarrowWalk <= a.walk.ext) Tile::copy_whole(a.walk, tile * kNarrowWalk, offset, s);
        else Tile::copy(a.walk, tile * kNarrowWalk, a.hidden, s);
        // every wave copies the step's records (the same bytes to the same place): all waves have the same number of copies in flight
        if (JOB == kNarrowDw)
            __builtin_amdgcn_global_load_lds((glb_cvoid_t*)(reinterpret_cast<const char*>(a.state + tile * kNarrowWalk) + lane * 16u),
                                             (lds_void16_t*)(s + Tile::kBytes), 16, 0, 0);
        else
            __builtin_amdgcn_global_load_lds((glb_cvoid_t*)(reinterpret_cast<const char*>(a.bias + tile * kNarrowWalk) + lane * 4u),
                                             (lds_void16_t*)(s + Tile::kBytes), 4, 0, 0);
    };
    // (dx applies g at its end)
    const bool wide = PARTS > 1 && (a.scales->wide[0] | a.scales->wide[1] | (JOB == kNarrowDw && a.scales->wide_g == 2)) != 0;
    const float lift = wide ? 1.f : a.lift;
    if (!wide && first < last) copy(first, 0);

    // this lane's own entries
    RowState st[NT];
    float bias_n[NT];
    int want[NT];
    // a logit (times log2 e) is its product times `back` plus the bias
    float back[NT];
    s16x8 own[PARTS][KK][NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int64_t e = n_wave + n * 16 + col;
        bool in = e < own_n;
        st[n] = RowState{INFINITY, 0.f, 0.f, -1};
        bias_n[n] = 0.f;
        want[n] = -1;
        if (JOB == kNarrowLse) {
            const int64_t t = in ? a.target[e] : -1;
            want[n] = t >= 0 && t < a.vocab && t != a.ignore ? (int)t : -1;
        } else if (JOB == kNarrowDx) {
            if (in) st[n] = a.state[e];
            st[n].inv_s *= lift;
            in = in && st[n].target >= 0;               // an ignored row: operand 0, maximum +inf, so that d = 0 whatever the row holds
        } else {
            bias_n[n] = in ? a.bias[e] : -INFINITY;     // d = 0
        }
        back[n] = a.scaled ? ldexpf(kLog2e, max(min(-(a.scales->ex[0] + a.scales->ex[1]), 126), -300)) : kLog2e;
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                const int k = kk * 32 + g * 8;
                s16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
                own[p][kk][n] = in && k < a.hidden ? *reinterpret_cast<const s16x8*>(static_cast<const uint16_t*>(a.own.base) +
                                                                                       (int64_t)p * a.own.part + e * a.own.ld + k)
                                                   : z;
            }
    }
    uint32_t t_base[HT];
#pragma unroll
    for (int h = 0; h < HT; ++h) t_base[h] = (uint32_t)(uintptr_t)(lds_void16_t*)lds + Tile::frag_t_base(h);
    float mx[NT], sum[NT], own_logit[NT];
    f32x4 acc[HT][NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        mx[n] = -INFINITY;
        sum[n] = own_logit[n] = 0.f;
#pragma unroll
        for (int h = 0; h < HT; ++h) acc[h][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    if constexpr (PARTS > 1) {
        if (wide) narrow_walk32<HT, NT, JOB>(a, first, last, n_wave, st, bias_n, want, mx, sum, own_logit, acc);
    }
    int stage = 0;
    for (int64_t tile = wide ? last : first; tile < last; ++tile, stage ^= 1) {
        if (tile + 1 < last) {
            copy(tile + 1, stage ^ 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(Tile::kCopies + 1) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const char* s = lds + stage * kStage;
        const int64_t m_tile = tile * kNarrowWalk;
#pragma unroll kHalves
        for (int mp = 0; mp < 2; ++mp) {
            f32x4 sc[2][NT];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int n = 0; n < NT; ++n) sc[t][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    s16x8 f[PARTS];
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) f[p] = Tile::frag(s, p, mp * 32 + t * 16, kk);
#pragma unroll
                    for (int order = PARTS - 1; order >= 0; --order)          // smallest products first, w's first part before its second:
#pragma unroll                                                                // the forward's logit to the bit, whichever side is walked
                        for (int i = 0; i <= order; ++i) {
                            const int p = JOB == kNarrowDw ? order - i : i;
#pragma unroll
                            for (int n = 0; n < NT; ++n) sc[t][n] = mfma16<E>(f[p], own[order - p][kk][n], sc[t][n]);
                        }
                }
            }
            const int64_t m0 = m_tile + mp * 32 + g * 4;            // the lane's first walk entry: 16 t + i further
            f32x4 bias[2];
            if (JOB != kNarrowDw) {
#pragma unroll
                for (int t = 0; t < 2; ++t) bias[t] = *reinterpret_cast<const f32x4*>(s + Tile::kBytes + (mp * 32 + t * 16 + g * 4) * 4);
            }
            if (JOB == kNarrowLse) {
                lse_step(a, sc, back, bias, m0, n_wave + col, want, mx, sum, own_logit);
                continue;
            }
            // d, split into its parts: the second product's operand
            // the second product's first fragments, read while the matrix cores work on the first product
            const uint32_t tile_at = stage * kStage + mp * (32 * HP * 2);
            // (dx only: dw has no registers left for them, 393 us against 364 at 36864 x 10000 x 64 fp32)
            s16x8 early[HB];
            if constexpr (JOB == kNarrowDx) Tile::template frag_t<PARTS - 1, HB>(t_base, tile_at, early);
            s16x8 d[PARTS][NT];
            // dw: the records of the lane's rows; target and g are read again where a target is met
            const RowState* row = reinterpret_cast<const RowState*>(s + Tile::kBytes) + mp * 32 + g * 4;
            float row_m2[8], row_scale[8];          // the row's g and the lift in its scale
            bool met = false;                       // targets among the wave's entries: rare
            if (JOB == kNarrowDw) {
                const int e0 = (int)(n_wave + col);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const RowState& q = row[(e / 4) * 16 + e % 4];
                    row_m2[e] = q.m2;
                    row_scale[e] = q.inv_s * q.g * lift;
                    met |= ((q.target - e0) & ~16) == 0;            // entry 0 or 1 of the lane's (NT = 2)
                }
                met = __ballot(met) != 0;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float m = JOB == kNarrowDw ? row_m2[e] : st[n].m2;
                    const float f = JOB == kNarrowDw ? row_scale[e] : st[n].inv_s;      // dx: times the lift; g comes at the end
                    const float b = JOB == kNarrowDw ? bias_n[n] : bias[e / 4][e % 4];
                    // the logit rounded as in the forward, then the difference: the row's maximum gives 1
                    v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e / 4][n][e % 4], back[n], b) - m) * f;
                    // an ignored row of x read as it is: its logits may have overflowed (fp32 ones are laid out as zeros)
                    if (JOB == kNarrowDw && PARTS == 1) v[e] = f == 0.f ? 0.f : v[e];
                }
                if (JOB == kNarrowDx) {
                    const int64_t at = st[n].target - m0;
                    if (__ballot(at >= 0 && at < 32)) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (at == (e / 4) * 16 + e % 4) v[e] -= lift;
                    }
                } else {
                    if (met) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const RowState& q = row[(e / 4) * 16 + e % 4];
                            if (q.target == (int)(n_wave + n * 16 + col)) v[e] -= q.g * lift;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum[n] += v[e];
                }
                vec_t<E, 8> o[PARTS];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        const uint32_t h = pack2<E>(v[e], v[e + 1]);
                        reinterpret_cast<uint32_t*>(&o[p])[e / 2] = h;
                        if (p + 1 < PARTS) minus_halves(h, v[e], v[e + 1]);
                    }
                }
#pragma unroll
                for (int p = 0; p < PARTS; ++p) d[p][n] = __builtin_bit_cast(s16x8, o[p]);
            }
            static_for<HT / HB>([&](auto h_c) {
                constexpr int h = decltype(h_c)::value * HB;
                static_for<PARTS>([&](auto q_c) {
                    constexpr int p = PARTS - 1 - decltype(q_c)::value;          // smallest products first
                    s16x8 f[HB];
                    if constexpr (JOB == kNarrowDx && h == 0 && p == PARTS - 1) {
#pragma unroll
                        for (int i = 0; i < HB; ++i) f[i] = early[i];
                    } else {
                        Tile::template frag_t<p, HB>(t_base + h, tile_at, f);
                    }
#pragma unroll
                    for (int b = PARTS - 1 - p; b >= 0; --b)
#pragma unroll
                        for (int i = 0; i < HB; ++i)
#pragma unroll
                            for (int n = 0; n < NT; ++n) acc[h + i][n] = mfma16<E>(f[i], d[b][n], acc[h + i][n]);
                });
            });
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // this wave has read the stage ...
        __builtin_amdgcn_s_barrier();                               // ... and the others: the next copy may overwrite it
        asm volatile("" ::: "memory");
    }

    if (JOB == kNarrowLse) {
        double total = 0.0, count = 0.0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float m = mx[n], q = sum[n];
#pragma unroll
            for (int x = 16; x <= 32; x <<= 1) {
                const float om = __shfl_xor(m, x, kWave), oq = __shfl_xor(q, x, kWave);
                const float nm = fmaxf(m, om), ref = nm == -INFINITY ? 0.f : nm;
                q = q * __builtin_amdgcn_exp2f(m - ref) + oq * __builtin_amdgcn_exp2f(om - ref);
                m = nm;
            }
            const int64_t r = n_wave + n * 16 + col;
            if (a.splits > 1) {
                if (g == 0 && r < a.rows) a.partial[(int64_t)split * a.rows + r] = make_float2(m, q);
                continue;
            }
            // the whole vocabulary has gone by: one lane of the row's four has met the target
            float t = own_logit[n];
#pragma unroll
            for (int x = 16; x <= 32; x <<= 1) t += __shfl_xor(t, x, kWave);
            if (g == 0 && r < a.rows) {
                const int64_t cat = a.target[r];
                float v = 0.f;
                if (cat != a.ignore) {
                    if (want[n] < 0) raise_flag(a.flags, CNF_FLAG_CATEGORY);
                    v = want[n] < 0 ? NAN : logf(q) + (m - t) * kLn2;
                    total += (double)v;
                    count += 1.0;
                }
                a.row_max[r] = m;
                a.row_sum[r] = q;
                a.loss[r] = v;
            }
        }
        if (a.splits > 1 || !a.reduced) return;
        double* sh = reinterpret_cast<double*>(lds);            // every wave is past its last read of the stages
        total = wave_sum(total);
        count = wave_sum(count);
        if (lane == 0) {
            sh[wave] = total;
            sh[4 + wave] = count;
        }
        __syncthreads();
        if (tid == 0) {
            const double s = ((sh[0] + sh[1]) + sh[2]) + sh[3], c = ((sh[4] + sh[5]) + sh[6]) + sh[7];
            if (gridDim.x == 1) {
                a.reduced[0] = (float)(s / c);
                a.reduced[1] = (float)s;
                a.reduced[2] = (float)c;
            } else {
                a.sums[2 * (int64_t)blockIdx.x] = s;
                a.sums[2 * (int64_t)blockIdx.x + 1] = c;
            }
        }
        return;
    }
    const float down = a.scales->top / lift;
    const int ex_out = a.scaled && !wide ? -a.scales->ex[JOB == kNarrowDw ? 0 : 1] : 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int64_t e = n_wave + n * 16 + col;
        float b = sum[n];
        if (JOB == kNarrowDw) {
#pragma unroll
            for (int x = 16; x <= 32; x <<= 1) b += __shfl_xor(b, x, kWave);
        }
        if (e >= own_n) continue;
        const float scale = JOB == kNarrowDx ? down * st[n].g : down;
        if (JOB == kNarrowDw && a.db && g == 0) {
            if (a.final_dtype >= 0) store_any(a.db, a.db_dtype, e, b * down);
            else static_cast<float*>(a.out)[((int64_t)split * own_n + e) * a.ld + a.ld - 4] = b * down;
        }
#pragma unroll
        for (int h = 0; h < HT; ++h) {
            const int k = h * 16 + g * 4;
            if (k >= a.hidden) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[h][n][i] = ldexpf(acc[h][n][i] * scale, ex_out);
            if (a.final_dtype < 0) {
                *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + ((int64_t)split * own_n + e) * a.ld + k) = acc[h][n];
            } else {
                store4_any(a.out, a.final_dtype, e * a.ld + k, e * a.ld + a.hidden, acc[h][n]);
            }
        }
    }
}

template <typename E, int PARTS, int HP>
static void narrow_job(NarrowJob job, const NarrowArgs& a, hipStream_t st) {
    const int64_t own_n = job == kNarrowDw ? a.vocab : a.rows;
    const dim3 grid((unsigned)((own_n + kNarrowOwn - 1) / kNarrowOwn * a.splits));
    if (job == kNarrowLse) CNF_LAUNCH((ce_narrow_kernel<E, PARTS, HP, kNarrowLse>), grid, dim3(kBlock), 0, st, a);
    else if (job == kNarrowDx) CNF_LAUNCH((ce_narrow_kernel<E, PARTS, HP, kNarrowDx>), grid, dim3(kBlock), 0, st, a);
    else CNF_LAUNCH((ce_narrow_kernel<E, PARTS, HP, kNarrowDw>), grid, dim3(kBlock), 0, st, a);
}

template <typename E, int PARTS>
static void narrow_width(NarrowJob job, const NarrowArgs& a, hipStream_t st) {
    if (a.hidden <= 32) narrow_job<E, PARTS, 32>(job, a, st);
    else if (a.hidden <= 64) narrow_job<E, PARTS, 64>(job, a, st);
    else narrow_job<E, PARTS, 128>(job, a, st);
}

bool narrow_supported(int hidden) { return hidden <= 128; }

int narrow_launch(NarrowJob job, int dtype, const NarrowArgs& a, hipStream_t st) {
    if (dtype == CNF_DTYPE_F32) narrow_width<f16_t, 2>(job, a, st);
    else if (dtype == CNF_DTYPE_BF16) narrow_width<bf16_t, 1>(job, a, st);
    else narrow_width<f16_t, 1>(job, a, st);
    return launch_status("cnf_linear_ce (few features)");
}

}  // namespace cnf
