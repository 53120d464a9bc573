// Softmax cross entropy of a linear layer over a vocabulary, forward and backward, without keeping the logits.
//
//   l_rv = x_r . w_v + b_v,   m_r = max_v l_rv,   s_r = sum_v exp(l_rv - m_r),   loss_r = log s_r + (m_r - l_rt)
//   (the kernels keep l and m in units of log 2: one instruction less per exponential)
//   d_rv = g_r (exp(l_rv - m_r) / s_r - [v = t_r]),   dx = d w,   dw = d^T x,   db_v = sum_r d_rv
//
// Forward: a product whose tiles never leave the registers.  A workgroup owns a block of rows and a part of the vocabulary; every
// lane keeps a running maximum and sum for its rows over the vocabulary entries it sees (four of them are consecutive), the lanes and
// waves of a row are joined once at the end, the parts of the vocabulary by a second launch, which also writes the loss.
// Backward, in pieces of the vocabulary: the piece's logits are computed again and turned into d (rounded to the operands' type, or
// kept as two fp16 parts for fp32), written to a workspace and read by two products: dx += d w over the piece, dw = d^T x complete for
// the piece.  db comes out of the second product: a fragment of ones in place of x.
//
// Bound by the matrix cores and, running one after the other without a pause, by the card's power: 8192 x 32000 x 1024 bf16, 537 GF each:
// forward 587 us (915 TF), d 632 us (850 TF; 525 MB written beside it), dw 515 us (1043 TF), dx 494 us (1087 TF); the library's 8192^3
// product reaches 1236 TF.  256 x 256 tiles read an operand from LDS half as often as 128 x 128 ones (d: 340 us a half against 421);
// those are kept for sizes whose large tiles would leave CUs empty.
//
// Few features (H <= 128) take the kernels of cnf_linear_ce_narrow.hip instead, which write nothing of size R x V.
//
// fp32 inputs are scaled by a power of two per tensor and split once into two fp16 parts (cnf_mfma.h: pair_a): three fp16 products keep
// every product to 2^-22 of its rows' largest elements, and the matrix cores do them at 16 times the fp32 rate.  Tensors with rows below
// 2^-14 of the largest element ("wide", kRowSpan) take fp32 matrix instructions instead, found on the device, in the same kernels and
// order: 8192 x 32000 x 1024 fp32 forward 1.50 ms (1070 TF of fp16 products), wide 7.45 ms (72 TF of fp32 ones, whose peak is 157).  16-bit inputs whose rows are not 16-byte aligned are copied once into padded rows.
// d is computed for g_r / max |g| (for fp16 operands times 2^14, so that small probabilities keep their bits) and the results are scaled
// back: under a mean every row's -1 is then exact, where a rounded -g_r would put the same relative error on every row's largest entry.
#include <algorithm>
#include <type_traits>

#include "cnf_linear_ce_narrow.h"

namespace cnf {

struct CeArgs {
    Operand w, x;                   // [V][H], [R][H]
    int pairs, parts;
    int64_t rows;
    int vocab, hidden, k_end;       // k_end: of the products (copied operands: the padded row)
    const void* bias;
    int bias_dtype;
    const int64_t* target;
    int64_t ignore;
    // forward
    float2* partial;                // [splits][rows]
    float* target_logit;            // [rows]
    int splits;                     // of the vocabulary tiles
    // backward
    const RowState* state;          // [rows]
    const CeScales* scales;
    int scaled;                     // fp32 operands: scales->ex and ->wide hold
    Operand32 w32, x32;             // fp32 operands as they were given
    float lift;                     // of d
    void* d;                        // [parts][rows_pad][piece_ld]
    int64_t d_part, d_ld;
    int v0, v1;                     // the piece
    int g_pass;                     // 1: d for dx, 2: for dw behind it (if g is apart), 0: for both
};

// tiles in the order that lets the workgroups of one XCD (dispatched round-robin over the 8) work on neighbouring tiles
__device__ __forceinline__ unsigned xcd_contiguous(unsigned id, unsigned n) {
    const unsigned xcd = id & 7u, idx = id >> 3, per = n >> 3, rem = n & 7u;
    return xcd * per + (xcd < rem ? xcd : rem) + idx;
}
// tile (i, j) of an ni x nj grid in column groups of 8
__device__ __forceinline__ void grouped_tile(unsigned t, unsigned ni, unsigned nj, unsigned& i, unsigned& j) {
    const unsigned per = 8 * ni, group = t / per, first = group * 8, width = min(8u, nj - first), in = t - group * per;
    j = first + in % width;
    i = in / width;
}

__device__ __forceinline__ float bias_at(const CeArgs& a, int v) { return a.bias && v < a.vocab ? load_any(a.bias, a.bias_dtype, v) : 0.f; }

// what takes a product to its logit, times log2 e
__device__ __forceinline__ float logit_scale(const CeArgs& a) {
    return a.scaled ? ldexpf(kLog2e, max(min(-(a.scales->ex[0] + a.scales->ex[1]), 126), -300)) : kLog2e;
}
// arguments of product32
__device__ __forceinline__ bool all_live(int64_t) { return true; }
struct NoExtra {
    template <typename F>
    __device__ __forceinline__ void operator()(const F&) const {}
};
__device__ __forceinline__ bool wide_rows(const CeScales* s) { return (s->wide[0] | s->wide[1]) != 0; }
// of the backward
__device__ __forceinline__ bool wide_call(const CeScales* s) { return (s->wide[0] | s->wide[1] | (s->wide_g == 2)) != 0; }
// fp16 operands (bf16 has fp32's exponents): whether d comes without g for dx, and then again with it for dw, since x, which the product over
// the rows takes as it lies, cannot carry a row's g
template <typename E, int PARTS>
__device__ __forceinline__ bool g_apart(const CeScales* s) {
    if (!std::is_same<E, f16_t>::value) return false;
    return s->wide_g != 0 && !(PARTS > 1 && wide_call(s));
}

// ---- forward ---------------------------------------------------------------------------------------------------------------------

// D[m = vocabulary][n = row]
template <typename E, int PARTS, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 2) void ce_lse_kernel(const CeArgs a) {
    typedef TileProduct<E, false, false, BM, BN, WM, WN> Tile;
    __shared__ __align__(16) char lds[Tile::kLds];
    Tile tile(a.w, a.x, a.pairs, a.k_end, lds);
    float back = logit_scale(a);
    const unsigned t = xcd_contiguous(blockIdx.x, gridDim.x);
    const int split = t % a.splits;
    const int r0 = (t / a.splits) * BN;
    const int vtiles = (a.vocab + BM - 1) / BM;
    const int first = (int)((int64_t)vtiles * split / a.splits), last = (int)((int64_t)vtiles * (split + 1) / a.splits);
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    float mx[Tile::NT], sum[Tile::NT];
    int want[Tile::NT];
#pragma unroll
    for (int n = 0; n < Tile::NT; ++n) {
        const int64_t r = (int64_t)r0 + tile.n_wave + n * 16 + col;
        mx[n] = -INFINITY;
        sum[n] = 0.f;
        const int64_t tg = r < a.rows ? a.target[r] : -1;
        want[n] = tg >= 0 && tg < a.vocab && tg != a.ignore ? (int)tg : -1;
    }
    auto clear = [](f32x4 (&acc)[Tile::MT][Tile::NT]) {
#pragma unroll
        for (int m = 0; m < Tile::MT; ++m)
#pragma unroll
            for (int n = 0; n < Tile::NT; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    auto enter = [&](f32x4 (&acc)[Tile::MT][Tile::NT], int v0) {
        const int vw = v0 + tile.m_wave + g * 4;        // the lane's first entry
#pragma unroll
        for (int m = 0; m < Tile::MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float b = a.bias ? bias_at(a, vw + m * 16 + i) * kLog2e : 0.f;
#pragma unroll
                for (int n = 0; n < Tile::NT; ++n) acc[m][n][i] = __builtin_fmaf(acc[m][n][i], back, b);
            }
        if (v0 + BM > a.vocab) {                        // entries past the vocabulary
#pragma unroll
            for (int m = 0; m < Tile::MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (vw + m * 16 + i >= a.vocab)
#pragma unroll
                        for (int n = 0; n < Tile::NT; ++n) acc[m][n][i] = -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < Tile::NT; ++n) {
            const int at = want[n] - vw;                // the target's place among the lane's entries: 16 m + i
            if (want[n] >= 0 && at >= 0 && at < Tile::MT * 16 && (at & 15) < 4) {
#pragma unroll
                for (int m = 0; m < Tile::MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (at == m * 16 + i) a.target_logit[(int64_t)r0 + tile.n_wave + n * 16 + col] = acc[m][n][i];
            }
            float top = mx[n];
#pragma unroll
            for (int m = 0; m < Tile::MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, acc[m][n][i]);
            // a lane that has seen only -inf keeps the sum 0 (exp(-inf - 0)); fmaxf drops a NaN, the sum keeps it
            const float ref = top == -INFINITY ? 0.f : top;
            float s = sum[n] * __builtin_amdgcn_exp2f(mx[n] - ref);
#pragma unroll
            for (int m = 0; m < Tile::MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) s += __builtin_amdgcn_exp2f(acc[m][n][i] - ref);
            sum[n] = s;
            mx[n] = top;
        }
    };
    bool wide = false;
    if constexpr (PARTS > 1) {
        wide = wide_rows(a.scales);
        if (wide) back = kLog2e;
        for (int vt = first; wide && vt < last; ++vt) {
            f32x4 acc[Tile::MT][Tile::NT];
            clear(acc);
            product32<false, false>(a.w32, a.x32, vt * BM + tile.m_wave, (int64_t)r0 + tile.n_wave, 0, a.hidden, acc, all_live, NoExtra{});
            enter(acc, vt * BM);
        }
    }
    for (int vt = wide ? last : first; vt < last; ++vt) {
        f32x4 acc[Tile::MT][Tile::NT];
        clear(acc);
        tile.begin(vt * BM, r0, 0, a.k_end);    // (ahead of the last epilogue, as in ce_d_kernel, it spills more and gains nothing: 578 -> 588 us)
        tile.multiply(acc, [](int, int) {});
        enter(acc, vt * BM);
    }
    // join the four lane groups, then the waves that share rows
    float2* sh = reinterpret_cast<float2*>(lds);        // [WM][BN]; every wave is past its last read of the stages
#pragma unroll
    for (int n = 0; n < Tile::NT; ++n) {
        float m = mx[n], s = sum[n];
#pragma unroll
        for (int x = 16; x <= 32; x <<= 1) {
            const float om = __shfl_xor(m, x, kWave), os = __shfl_xor(s, x, kWave);
            const float nm = fmaxf(m, om), ref = nm == -INFINITY ? 0.f : nm;
            s = s * __builtin_amdgcn_exp2f(m - ref) + os * __builtin_amdgcn_exp2f(om - ref);
            m = nm;
        }
        if (g == 0) sh[(tile.m_wave / (BM / WM)) * BN + tile.n_wave + n * 16 + col] = make_float2(m, s);
    }
    __syncthreads();
    for (int n = threadIdx.x; n < BN; n += Tile::kThreads) {
        const int64_t r = (int64_t)r0 + n;
        if (r >= a.rows) continue;
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int w = 0; w < WM; ++w) {
            const float2 o = sh[w * BN + n];
            const float nm = fmaxf(m, o.x), ref = nm == -INFINITY ? 0.f : nm;
            s = s * __builtin_amdgcn_exp2f(m - ref) + o.y * __builtin_amdgcn_exp2f(o.x - ref);
            m = nm;
        }
        a.partial[(int64_t)split * a.rows + r] = make_float2(m, s);
    }
}

// the parts of the vocabulary -> row maximum, sum, loss; a category outside the vocabulary raises its flag and gives NaN.
// `group` lanes (a power of two) share a row: few rows have many parts (one row of 32000 classes in 250 parts: a lane alone takes 40 us).
// sums (with `reduced`): [workgroups][2] sum and number of the rows that are not ignored, in a fixed order; a single workgroup
// writes `reduced` itself
__global__ __launch_bounds__(kBlock) void ce_join_kernel(const float2* partial, const float* target_logit, const int64_t* target,
                                                         int64_t ignore, int vocab, int splits, int group, int64_t rows, float* row_max,
                                                         float* row_sum, float* loss, double* sums, float* reduced, int* flags) {
    const int l = threadIdx.x & (group - 1);
    const int64_t r = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / group;
    float v = 0.f;
    bool counts = false;
    float m = -INFINITY, s = 0.f;
    if (r < rows)
        for (int k = l; k < splits; k += group) m = fmaxf(m, partial[(int64_t)k * rows + r].x);
    for (int x = 1; x < group; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, kWave));
    const float ref = m == -INFINITY ? 0.f : m;
    if (r < rows)
        for (int k = l; k < splits; k += group) {
            const float2 o = partial[(int64_t)k * rows + r];
            s += o.y * __builtin_amdgcn_exp2f(o.x - ref);
        }
    for (int x = 1; x < group; x <<= 1) s += __shfl_xor(s, x, kWave);
    if (r < rows && l == 0) {
        row_max[r] = m;
        row_sum[r] = s;
        const int64_t t = target[r];
        counts = t != ignore;
        if (counts) {
            if (t < 0 || t >= vocab) {
                raise_flag(flags, CNF_FLAG_CATEGORY);
                v = NAN;
            } else {
                v = logf(s) + (m - target_logit[r]) * kLn2;
            }
        }
        loss[r] = v;
    }
    if (!reduced) return;
    __shared__ double sh[2][kWavesPerBlock];
    const double ws = wave_sum((double)v), wc = wave_sum(counts ? 1.0 : 0.0);
    if ((threadIdx.x & 63) == 0) {
        sh[0][threadIdx.x >> 6] = ws;
        sh[1][threadIdx.x >> 6] = wc;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0, c = 0.0;
        for (int w = 0; w < kWavesPerBlock; ++w) {
            s += sh[0][w];
            c += sh[1][w];
        }
        if (gridDim.x == 1) {
            reduced[0] = (float)(s / c);
            reduced[1] = (float)s;
            reduced[2] = (float)c;
        } else {
            sums[2 * (int64_t)blockIdx.x] = s;
            sums[2 * (int64_t)blockIdx.x + 1] = c;
        }
    }
}

// reduced = {mean, sum, number}: one workgroup, fixed order; no row left: 0 / 0 = NaN
__global__ __launch_bounds__(1024) void ce_reduce_kernel(const double* sums, int64_t n, float* reduced) {
    __shared__ double sh[2][16];
    double s = 0.0, c = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        s += sums[2 * i];
        c += sums[2 * i + 1];
    }
    s = wave_sum(s);
    c = wave_sum(c);
    if ((threadIdx.x & 63) == 0) {
        sh[0][threadIdx.x >> 6] = s;
        sh[1][threadIdx.x >> 6] = c;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = c = 0.0;
        for (int w = 0; w < 16; ++w) {
            s += sh[0][w];
            c += sh[1][w];
        }
        reduced[0] = (float)(s / c);
        reduced[1] = (float)s;
        reduced[2] = (float)c;
    }
}

// ---- operand layout ----------------------------------------------------------------------------------------------------------------

constexpr int kMaxBlocks = 256;
// What the layout has to know of an fp32 tensor: the bits of its largest finite |element|, and of the smallest that is largest in its row
// (rows of zeros left out; none: all ones)
struct Extent {
    uint32_t top, least;
};
__device__ __forceinline__ int exponent_of(uint32_t bits) { return max((int)(bits >> 23), 1) - 127; }       // subnormal numbers: as if of -126
__device__ __forceinline__ bool is_wide(Extent e, int span) { return e.least != 0xffffffffu && exponent_of(e.top) - exponent_of(e.least) > span; }

// what this lane's rows say, of fp32 rows `block`, `block` + `blocks`, ... (in units of the rows that a workgroup's lanes share at a time);
// rows with target == ignore do not count (target: nullable).  At most a wave shares a row; four rows are in flight
__device__ __forceinline__ Extent extent_of(const float* src, int64_t stride, int64_t rows, int H, const int64_t* target, int64_t ignore, int block,
                                            int blocks) {
    int g = 1;
    while (g < kWave && g * 4 < H) g <<= 1;
    const int l = threadIdx.x & (g - 1), rpb = blockDim.x / g;
    const bool vec = stride % 4 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    Extent all = {0, 0xffffffffu};
    const int64_t step = (int64_t)blocks * rpb;
    for (int64_t r = (int64_t)block * rpb + threadIdx.x / g; r < rows; r += 4 * step) {
        bool live[4];
        uint32_t top[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) live[k] = r + k * step < rows && (!target || target[r + k * step] != ignore);
        for (int c = l * 4; c < H; c += g * 4) {
            f32x4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float* p = src + (r + k * step) * stride + c;
                v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (r + k * step >= rows) continue;
                if (vec && c + 4 <= H) {
                    v[k] = *reinterpret_cast<const f32x4*>(p);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[k][i] = c + i < H ? p[i] : 0.f;
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t b = __float_as_uint(v[k][i]) & 0x7fffffffu;
                    if (live[k] && b < 0x7f800000u) top[k] = max(top[k], b);
                }
        }
        for (int m = 1; m < g; m <<= 1)
#pragma unroll
            for (int k = 0; k < 4; ++k) top[k] = max(top[k], (uint32_t)__shfl_xor((int)top[k], m, kWave));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            all.top = max(all.top, top[k]);
            if (top[k]) all.least = min(all.least, top[k]);
        }
    }
    return all;
}
// of the workgroup, in every lane
__device__ __forceinline__ Extent block_extent(Extent e, Extent* sh) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        e.top = max(e.top, (uint32_t)__shfl_xor((int)e.top, m, kWave));
        e.least = min(e.least, (uint32_t)__shfl_xor((int)e.least, m, kWave));
    }
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = e;
    __syncthreads();
    for (int k = 0; k < (int)blockDim.x / kWave; ++k) {
        e.top = max(e.top, sh[k].top);
        e.least = min(e.least, sh[k].least);
    }
    return e;
}

// fp32: the extents of x's rows that count (blockIdx.y 0) and of w (1), one for each workgroup
__global__ __launch_bounds__(1024) void ce_extent_kernel(const float* x, int64_t x_stride, int64_t R, const int64_t* target, int64_t ignore,
                                                           const float* w, int64_t w_stride, int V, int H, Extent* extents) {
    __shared__ Extent sh[16];
    const Extent e = block_extent(blockIdx.y ? extent_of(w, w_stride, V, H, nullptr, 0, blockIdx.x, kMaxBlocks)
                                             : extent_of(x, x_stride, R, H, target, ignore, blockIdx.x, kMaxBlocks), sh);
    if (threadIdx.x == 0) extents[blockIdx.y * kMaxBlocks + blockIdx.x] = e;
}

struct LayoutJob {
    const void* src;                // nullable: nothing to do
    int64_t stride, rows;
    void* dst;
};
struct LayoutArgs {
    LayoutJob job[2];               // x, w: [rows][cols] -> `parts` arrays of [rows][ld] 16-bit elements, zeros behind cols
    int cols, vec;                  // vec: bit j: 8 elements of job j's rows may be read as vectors of 16 bytes
    const int64_t* target;          // fp32: ignored rows of x are laid out as zeros, whatever they hold
    int64_t ignore;
    int64_t ld;
    const void* bias;               // -> fp32, times log2 e, -inf behind the vocabulary (nullable: zeros)
    int bias_dtype, vocab, bias_pad;
    float* bias_out;                // nullable
    const Extent* extents;          // fp32: what ce_extent_kernel found (null: every workgroup looks for itself),
    const int* known;               // or the forward's exponents;
    CeScales* scales;               // where what they say goes ...
    int* exponents;                 // ... and here (nullable)
};

// one launch for whatever a call has to lay out: blockIdx.y 0: x, 1: w, 2: the bias.  fp32: scaled, then x0 + x1, each the fp16 nearest to
// what is left
template <typename T, typename E, int PARTS>
__global__ __launch_bounds__(kBlock) void ce_layout_kernel(const LayoutArgs a) {
    if (blockIdx.y == 2) {
        if (a.bias_out)
            for (int v = blockIdx.x * kBlock + threadIdx.x; v < a.bias_pad; v += gridDim.x * kBlock)
                a.bias_out[v] = v >= a.vocab ? -INFINITY : (a.bias ? load_any(a.bias, a.bias_dtype, v) * kLog2e : 0.f);
        return;
    }
    const int which = blockIdx.y;
    const LayoutJob job = a.job[which];
    if (!job.src) return;
    const T* src = static_cast<const T*>(job.src);
    E* dst = static_cast<E*>(job.dst);
    int ex = 0;
    if (PARTS > 1) {
        bool wide;
        if (a.known) {
            wide = a.known[which] >= kWideMark / 2;
            ex = a.known[which] - (wide ? kWideMark : 0);
        } else {
            __shared__ Extent sh[kWavesPerBlock];
            static_assert(kMaxBlocks == kBlock, "a lane reads one workgroup's extent");
            const Extent e = block_extent(a.extents ? a.extents[which * kMaxBlocks + threadIdx.x]
                                                    : extent_of(reinterpret_cast<const float*>(src), job.stride, job.rows, a.cols,
                                                                which ? nullptr : a.target, a.ignore, 0, 1), sh);
            wide = is_wide(e, kRowSpan);
            ex = e.top ? 14 - exponent_of(e.top) : 0;           // the largest into 2^14 ... 2^15; zeros alone stay as they are
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.scales->ex[which] = ex;
            a.scales->wide[which] = wide;
            if (a.exponents) a.exponents[which] = ex + (wide ? kWideMark : 0);
        }
    }
    const int per = (int)(a.ld / 8);
    const int64_t part = job.rows * a.ld, n = job.rows * per;
    for (int64_t q = (int64_t)blockIdx.x * kBlock + threadIdx.x; q < n; q += (int64_t)gridDim.x * kBlock) {
        const int64_t r = q / per;
        const int c0 = (int)(q - r * per) * 8;
        const bool live = PARTS == 1 || which == 1 || a.target[r] != a.ignore;
        vec_t<T, 8> in;
        if (((a.vec >> which) & 1) && c0 + 8 <= a.cols) {
            in = *reinterpret_cast<const vec_t<T, 8>*>(src + r * job.stride + c0);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) in[i] = c0 + i < a.cols ? src[r * job.stride + c0 + i] : (T)0.f;
        }
        vec_t<E, 8> o[PARTS];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v = PARTS > 1 ? (live ? ldexpf((float)in[i], ex) : 0.f) : (float)in[i];
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                o[p][i] = (E)v;
                // infinities and NaN are whole in the first part
                v = PARTS > 1 && __builtin_isfinite(v) ? v - (float)o[p][i] : 0.f;
            }
        }
#pragma unroll
        for (int p = 0; p < PARTS; ++p) *reinterpret_cast<vec_t<E, 8>*>(dst + p * part + r * a.ld + c0) = o[p];
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------

// upstream gradients (per row, or one over the count) -> row records, ignored ones behind the last row up to rows_pad.  Every g is
// divided by the largest |g|, which goes to scales
__global__ __launch_bounds__(1024) void ce_rows_kernel(const float* g, int g_is_row, const float* count, const float* row_max, const float* row_sum,
                                                       const int64_t* target, int64_t ignore, int vocab, int64_t rows, int64_t rows_pad, GradSpan span,
                                                       RowState* state, CeScales* scales) {
    __shared__ Extent sh[16];
    const float shared = g_is_row ? 0.f : *g / *count;
    auto counts = [&](int64_t t) { return t != ignore && t >= 0 && t < vocab; };
    Extent e = {__float_as_uint(shared) & 0x7fffffffu, 0xffffffffu};
    if (g_is_row) {
        for (int64_t r = threadIdx.x; r < rows; r += 1024)
            if (counts(target[r])) {
                const uint32_t bits = __float_as_uint(g[r]) & 0x7fffffffu;
                e.top = max(e.top, bits);
                if (bits) e.least = min(e.least, bits);
            }
        e = block_extent(e, sh);
    }
    // an infinite or NaN one among them: the others are any distance from it
    const bool finite = e.top < 0x7f800000u;
    const int wide = !g_is_row ? 0 : (!finite || is_wide(e, span.plain) ? 2 : (is_wide(e, span.apart) ? 1 : 0));
    // all gradients zero, or an infinite or NaN one among them: as they are
    const float top = e.top != 0 && finite ? __uint_as_float(e.top) : 1.f;
    if (threadIdx.x == 0 && blockIdx.x == 0) {
        scales->top = top;
        scales->wide_g = wide;
    }
    for (int64_t r = (int64_t)blockIdx.x * 1024 + threadIdx.x; r < rows_pad; r += (int64_t)gridDim.x * 1024) {
        const int64_t t = r < rows ? target[r] : -1;
        const bool in = r < rows && counts(t);
        RowState s;
        s.m2 = in ? row_max[r] : INFINITY;
        s.inv_s = in ? 1.f / row_sum[r] : 0.f;
        s.g = in ? (g_is_row ? g[r] : shared) / top : 0.f;
        s.target = in ? (int)t : -1;
        state[r] = s;
    }
}

// d, a few tiles per workgroup (as many workgroups as run at once), so that a tile's first copies land during the epilogue of the one
// before; D[m = vocabulary][n = row].  An XCD's workgroups share one run of tiles.  8192 x 32000 x 1024 bf16: 632 us (850 TF); the copies
// ahead and the 16-byte stores together took 6 % off (726 -> 682 us, measured alone)
template <typename E, int PARTS, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 2) void ce_d_kernel(const CeArgs a) {
    typedef TileProduct<E, false, false, BM, BN, WM, WN> Tile;
    __shared__ __align__(16) char lds[Tile::kLds];
    Tile tile(a.w, a.x, a.pairs, a.k_end, lds);
    const unsigned nv = (a.v1 - a.v0 + BM - 1) / BM, nr = (unsigned)((a.rows + BN - 1) / BN), tiles = nv * nr;
    const unsigned xcds = min(8u, gridDim.x), xcd = blockIdx.x % xcds, step = gridDim.x / xcds + (xcd < gridDim.x % xcds ? 1 : 0);
    const unsigned end = (unsigned)((uint64_t)tiles * (xcd + 1) / xcds);
    unsigned t = (unsigned)((uint64_t)tiles * xcd / xcds) + blockIdx.x / xcds;
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    E* d = static_cast<E*>(a.d);
    int v0 = 0, r0 = 0;
    auto begin = [&]() {
        unsigned ti, tj;
        grouped_tile(t, nv, nr, ti, tj);
        v0 = a.v0 + ti * BM;
        r0 = tj * BN;
        tile.begin(v0, r0, 0, a.k_end);
    };
    if constexpr (PARTS > 1) {
        if (wide_call(a.scales)) {
            if (a.g_pass == 2) return;
            // fp32 products, and d in fp32 where its two parts would be: [rows_pad][piece_ld]
            for (; t < end; t += step) {
                unsigned ti, tj;
                grouped_tile(t, nv, nr, ti, tj);
                const int64_t vw = a.v0 + (int64_t)ti * BM + tile.m_wave + g * 4, rw = (int64_t)tj * BN + tile.n_wave + col;
                f32x4 acc[Tile::MT][Tile::NT];
#pragma unroll
                for (int m = 0; m < Tile::MT; ++m)
#pragma unroll
                    for (int n = 0; n < Tile::NT; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
                product32<false, false>(a.w32, a.x32, vw - g * 4, rw - col, 0, a.hidden, acc, all_live, NoExtra{});
#pragma unroll
                for (int n = 0; n < Tile::NT; ++n) {
                    const RowState q = rw + n * 16 < a.rows ? a.state[rw + n * 16] : RowState{INFINITY, 0.f, 0.f, -1};
#pragma unroll
                    for (int m = 0; m < Tile::MT; ++m) {
                        f32x4 p;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int64_t v = vw + m * 16 + i;
                            const float b = a.bias ? bias_at(a, (int)v) * kLog2e : 0.f;
                            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[m][n][i], kLog2e, b) - q.m2) * q.inv_s;
                            if (v == q.target) p[i] -= 1.f;
                            p[i] = q.target < 0 || v >= a.v1 ? 0.f : p[i] * q.g;
                        }
                        *reinterpret_cast<f32x4*>(static_cast<float*>(a.d) + (rw + n * 16) * a.d_ld + (vw - a.v0) + m * 16) = p;
                    }
                }
            }
            return;
        }
    }
    const bool apart = a.g_pass != 0 && g_apart<E, PARTS>(a.scales), without_g = apart && a.g_pass == 1;
    if (a.g_pass == 2 && !apart) return;
    const float back = logit_scale(a);
    if (t < end) begin();
    while (t < end) {
        f32x4 acc[Tile::MT][Tile::NT];
#pragma unroll
        for (int m = 0; m < Tile::MT; ++m)
#pragma unroll
            for (int n = 0; n < Tile::NT; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        tile.multiply(acc, [](int, int) {});
        const int vw = v0 + tile.m_wave + g * 4;
        const int64_t rw = (int64_t)r0 + tile.n_wave + col;
        const bool edge = v0 + BM > a.v1;
        RowState st[Tile::NT];
        float scale[Tile::NT], own_g[Tile::NT];
        // targets among the wave's entries are rare: their -g is applied behind a branch that most waves do not take
        int at[Tile::NT];
        bool hit = false;
#pragma unroll
        for (int n = 0; n < Tile::NT; ++n) {
            st[n] = rw + n * 16 < a.rows ? a.state[rw + n * 16] : RowState{INFINITY, 0.f, 0.f, -1};
            own_g[n] = without_g ? a.lift : st[n].g * a.lift;
            scale[n] = st[n].inv_s * own_g[n];
            at[n] = st[n].target - vw;
            hit |= st[n].target >= 0 && at[n] >= 0 && at[n] < Tile::MT * 16;
        }
        const bool any_hit = __ballot(hit) != 0;        // the rows' records have arrived: no wait for them behind the copies
        const int v_tile = v0;
        t += step;
        if (t < end) begin();
#pragma unroll
        for (int m = 0; m < Tile::MT; m += 2) {
            f32x4 b[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            if (a.bias) {
#pragma unroll
                for (int i = 0; i < 8; ++i) b[i / 4][i % 4] = bias_at(a, vw + (m + i / 4) * 16 + i % 4) * kLog2e;
            }
#pragma unroll
            for (int n = 0; n < Tile::NT; ++n) {
                uint32_t o[PARTS][2][2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    f32x4 p;
#pragma unroll
                    for (int i = 0; i < 4; ++i)         // the logit rounded as in the forward, then the difference: the row's maximum gives 1
                        p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[m + q][n][i], back, b[q][i]) - st[n].m2) * scale[n];
                    if (any_hit) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (at[n] == (m + q) * 16 + i) p[i] -= own_g[n];        // an ignored row's is negative
                    }
                    if (edge) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (vw + (m + q) * 16 + i >= a.v1) p[i] = 0.f;
                    }
                    // an ignored row, or one that is not there (x may hold anything)
                    if (st[n].target < 0) p = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < 4; i += 2)
#pragma unroll
                        for (int k = 0; k < PARTS; ++k) {
                            o[k][q][i / 2] = pack2<E>(p[i], p[i + 1]);
                            if (k + 1 < PARTS) {
                                float lo = p[i], hi = p[i + 1];
                                minus_halves(o[k][q][i / 2], lo, hi);
                                p[i] = lo;
                                p[i + 1] = hi;
                            }
                        }
                }
                // lanes 16 ... 31 hand their entries 4 ... 7 of block m to lanes 0 ... 15 and get 0 ... 3 of block m + 1 (lanes 48 and 32
                // likewise): a lane then holds 8 consecutive entries, a row's 32 are one 64-byte run
                const int v = v_tile - a.v0 + tile.m_wave + (m + (g & 1)) * 16 + (g >> 1) * 8;
#pragma unroll
                for (int k = 0; k < PARTS; ++k) {
                    vec_t<uint32_t, 4> w;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const auto r = __builtin_amdgcn_permlane16_swap(o[k][0][i], o[k][1][i], false, false);
                        w[i] = r[0];
                        w[2 + i] = r[1];
                    }
                    *reinterpret_cast<vec_t<uint32_t, 4>*>(d + k * a.d_part + (rw + n * 16) * a.d_ld + v) = w;
                }
            }
        }
    }
}

struct GradArgs {
    Operand a, b;           // D[m = hidden][n = row or vocabulary entry]
    Operand32 a32, b32;     // wide operands: the tensor itself, and d in fp32
    const RowState* state;  // over the rows: which of them count; over the vocabulary: their g, where it may be apart, or null
    int pairs, k_end, ksplit;
    int m_end, n_end;       // extent of the output
    void* out;              // final: [n][ld] of the output type; partial: fp32 [ksplit][n][ld]
    int64_t ld;
    int final_dtype;        // -1: partial sums
    int accumulate;         // partial: add to what is there
    const CeScales* scales;
    int scaled;             // fp32: which of scales->ex to take back (1 + index), 0: none
    float lift;
    void* db;               // nullable: row sums of B's operand; partial: in column ld - 4 of out
    int db_dtype;
};

template <typename E, int PARTS, bool KMB, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 2) void ce_grad_kernel(const GradArgs a) {
    typedef TileProduct<E, true, KMB, BM, BN, WM, WN> Tile;
    __shared__ __align__(16) char lds[Tile::kLds];
    Tile tile(a.a, a.b, a.pairs, a.k_end, lds);
    const unsigned nm = (a.m_end + BM - 1) / BM, nn = (a.n_end + BN - 1) / BN, per = nm * nn;
    const unsigned t = xcd_contiguous(blockIdx.x, gridDim.x);
    const unsigned ks = t / per;
    unsigned ti, tj;
    grouped_tile(t - ks * per, nm, nn, ti, tj);
    const int m0 = ti * BM, n0 = tj * BN;
    const int steps = (a.k_end + kStepK - 1) / kStepK;
    const int k0 = (int)((int64_t)steps * ks / a.ksplit) * kStepK, k1 = min(a.k_end, (int)((int64_t)steps * (ks + 1) / a.ksplit) * kStepK);
    const bool sums = KMB && a.db && m0 == 0 && tile.m_wave == 0;
    f32x4 acc[Tile::MT][Tile::NT], acc1[Tile::NT];
#pragma unroll
    for (int n = 0; n < Tile::NT; ++n) {
        acc1[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < Tile::MT; ++m) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    s16x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = __builtin_bit_cast(short, (E)1.f);
    const bool wide = PARTS > 1 && wide_call(a.scales);
    if (wide) {
        product32<true, KMB>(a.a32, a.b32, m0 + tile.m_wave, (int64_t)n0 + tile.n_wave, k0, k1, acc, [&](int64_t k) { return !KMB || a.state[k].target >= 0; },
                             [&](const float (&fb)[Tile::NT][4]) {
                                 if (!sums) return;
#pragma unroll
                                 for (int j = 0; j < 4; ++j)
#pragma unroll
                                     for (int n = 0; n < Tile::NT; ++n) acc1[n] = mfma32(1.f, fb[n][j], acc1[n]);
                             });
    } else {
        // fp32: each part of d is once the partner of part 0 of x: pairs (0, 1) and (0, 0)
        tile.begin(m0, n0, k0, k1);
        tile.multiply(acc, [&](int stage, int pair) {
            if (!sums || pair_a(a.pairs, pair) != 0) return;
            const char* sb = lds + stage * Tile::kStage + Tile::kBytesA;
            s16x8 fb[4];
            tile_frags4<KMB, BN>(sb, tile.n_wave, 0, fb);
#pragma unroll
            for (int n = 0; n < Tile::NT; ++n) acc1[n] = mfma16<E>(ones, fb[n], acc1[n]);
        });
    }
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const bool apart = !KMB && a.state && g_apart<E, PARTS>(a.scales);
    const float all_down = wide ? a.scales->top : a.scales->top / a.lift;
    const int ex = a.scaled && !wide ? -a.scales->ex[a.scaled - 1] : 0;
#pragma unroll
    for (int n = 0; n < Tile::NT; ++n) {
        const int64_t row = (int64_t)n0 + tile.n_wave + n * 16 + col;
        if (row >= a.n_end) continue;
        float down = all_down;
        if (!KMB && apart) down *= a.state[row].g;
#pragma unroll
        for (int m = 0; m < Tile::MT; ++m) {
            const int h = m0 + tile.m_wave + m * 16 + g * 4;
            if (h >= a.m_end) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][n][i] = a.scaled ? ldexpf(acc[m][n][i] * down, ex) : acc[m][n][i] * down;
            if (a.final_dtype < 0) {
                // ld is a multiple of 4: a partial row has room for the whole vector
                f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + ((int64_t)ks * a.n_end + row) * a.ld + h);
                *p = a.accumulate ? *p + acc[m][n] : acc[m][n];
            } else {
                store4_any(a.out, a.final_dtype, row * a.ld + h, row * a.ld + a.m_end, acc[m][n]);
            }
        }
        if (sums && g == 0) {
            if (a.final_dtype < 0) static_cast<float*>(a.out)[((int64_t)ks * a.n_end + row) * a.ld + a.ld - 4] = acc1[n][0] * down;
            else store_any(a.db, a.db_dtype, row, acc1[n][0] * down);
        }
    }
}

struct SumArgs {
    const float* partial;           // [parts][rows][ld]
    int parts;
    int64_t rows, ld;
    int cols;
    void* out;                      // [rows][cols] dense
    int dtype;
    void* db;                       // nullable: [rows], from column ld - 4
    int db_dtype;
};
// where output q lies in a partial matrix
__device__ __forceinline__ int64_t sum_source(const SumArgs& a, int64_t q) {
    const int per = a.cols + (a.db ? 1 : 0);
    const int64_t r = q / per;
    const int c = (int)(q - r * per);
    return r * a.ld + (c < a.cols ? c : a.ld - 4);
}
__device__ __forceinline__ void sum_store(const SumArgs& a, int64_t q, float v) {
    const int per = a.cols + (a.db ? 1 : 0);
    const int64_t r = q / per;
    const int c = (int)(q - r * per);
    if (c < a.cols) store_any(a.out, a.dtype, r * a.cols + c, v);
    else store_any(a.db, a.db_dtype, r, v);
}

// the partial matrices added in their order: a lane per output
__global__ __launch_bounds__(kBlock) void ce_sum_kernel(const SumArgs a) {
    const int64_t n = a.rows * (a.cols + (a.db ? 1 : 0)), part = a.rows * a.ld;
    for (int64_t q = (int64_t)blockIdx.x * kBlock + threadIdx.x; q < n; q += (int64_t)gridDim.x * kBlock) {
        const float* p = a.partial + sum_source(a, q);
        float s = 0.f;
        for (int k = 0; k < a.parts; ++k) s += p[k * part];
        sum_store(a, q, s);
    }
}

// many partial matrices of few outputs (51 classes x 64 features x 288 parts: 67 us with a lane per output): 16 outputs a workgroup,
// 64 lanes each add every 64th part, then the 64 sums are added in order
__global__ __launch_bounds__(1024) void ce_sum_many_kernel(const SumArgs a) {
    __shared__ float sh[64][17];
    const int cl = threadIdx.x & 15, slot = threadIdx.x >> 4;
    const int64_t n = a.rows * (a.cols + (a.db ? 1 : 0)), part = a.rows * a.ld, q = (int64_t)blockIdx.x * 16 + cl;
    float t = 0.f;
    if (q < n) {
        const float* p = a.partial + sum_source(a, q);
        for (int k = slot; k < a.parts; k += 64) t += p[k * part];
    }
    sh[slot][cl] = t;
    __syncthreads();
    if (slot == 0 && q < n) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 64; ++k) v += sh[k][cl];
        sum_store(a, q, v);
    }
}

// ---- host: plan of a call -------------------------------------------------------------------------------------------------------

constexpr int kBig = 256, kSmall = 128;         // tile edges
// what 32-bit loop counters and a tile's 31-bit offsets (256 rows) reach
constexpr int kMaxVocab = 1 << 30, kMaxHidden = 1 << 21;
// d of one piece of the vocabulary.  A second piece costs dx another pass through memory: 8192 x 32000 x 1024 bf16 takes 2197 us as one
// piece, 2285 as two of 256 MiB, which would fit the memory-side cache
constexpr int64_t kPieceBytes = 512ll << 20;

static int64_t round_up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
static int64_t ceil_div(int64_t n, int64_t m) { return (n + m - 1) / m; }

struct CePlan {
    int parts, pairs;
    bool copy_x, copy_w, narrow;
    int64_t ldh;                    // padded row of a copied operand
    int64_t x_off, w_off, bias_off, scales_off, extents_off;
    // forward
    bool big_lse;
    int splits, join_group;
    int64_t partial_off, logit_off, sums_off;
    // backward
    int64_t rows_pad, piece, d_off, state_off, dx_off, dw_off;
    int dx_split, dw_split;
    bool big_d, big_dx, big_dw;
    int64_t bytes;
};

static CePlan ce_plan(int64_t R, int V, int H, int dtype, bool x_ok, bool w_ok, bool backward) {
    CePlan p{};
    p.parts = dtype == CNF_DTYPE_F32 ? 2 : 1;
    p.pairs = dtype == CNF_DTYPE_F32 ? 3 : 1;
    p.copy_x = p.parts > 1 || !x_ok;
    p.copy_w = p.parts > 1 || !w_ok;
    p.narrow = narrow_supported(H);
    p.ldh = round_up(H, p.narrow ? 8 : kStepK);     // whole steps of the products
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += round_up(bytes, 256);
        return o;
    };
    if (p.copy_x) p.x_off = take((int64_t)p.parts * R * p.ldh * 2);
    if (p.copy_w) p.w_off = take((int64_t)p.parts * V * p.ldh * 2);
    p.scales_off = take(sizeof(CeScales));
    if (p.parts > 1) p.extents_off = take(2 * kMaxBlocks * sizeof(Extent));
    if (p.narrow) p.bias_off = take(round_up(V, kNarrowWalk) * 4);
    // about four workgroups for every CU, at least two steps of the walk each
    auto narrow_split = [](int64_t own, int64_t walk) {
        return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(1024, ceil_div(own, kNarrowOwn)), ceil_div(walk, 2 * kNarrowWalk)));
    };
    const int64_t ld4 = round_up(H, 4);
    if (!backward) {
        // 256 x 256 tiles once they fill the chip; the vocabulary is split until there are two workgroups per CU (one of the big)
        p.big_lse = ceil_div(R, kBig) * ceil_div(V, kBig) >= 512;
        const int edge = p.big_lse ? kBig : kSmall;
        const int64_t rt = ceil_div(R, edge), vt = ceil_div(V, edge);
        p.splits = p.narrow ? narrow_split(R, V) : (int)std::min<int64_t>(vt, std::max<int64_t>(1, (p.big_lse ? 256 : 512) / rt));
        p.partial_off = take((int64_t)p.splits * R * 8);
        p.logit_off = take(R * 4);
        p.join_group = 1;
        while (p.join_group < kWave && p.join_group * 4 < p.splits) p.join_group *= 2;
        p.sums_off = take(std::max(ceil_div(R, kNarrowOwn), ceil_div(R * p.join_group, kBlock)) * 16);
        p.bytes = at;
        return p;
    }
    p.rows_pad = round_up(R, kBig);
    p.state_off = take(p.rows_pad * (int64_t)sizeof(RowState));
    if (p.narrow) {
        p.dx_split = narrow_split(R, V);
        p.dw_split = narrow_split(V, R);
        if (p.dx_split > 1) p.dx_off = take((int64_t)p.dx_split * R * ld4 * 4);
        if (p.dw_split > 1) p.dw_off = take((int64_t)p.dw_split * V * (ld4 + 4) * 4);
        p.bytes = at;
        return p;
    }
    const int64_t row_bytes = p.rows_pad * 2 * p.parts;
    p.piece = std::min<int64_t>(round_up(V, kBig), std::max<int64_t>(kBig, kPieceBytes / row_bytes / kBig * kBig));
    p.d_off = take(row_bytes * p.piece);
    const int64_t width = std::min<int64_t>(p.piece, V);
    p.big_d = ceil_div(R, kBig) * ceil_div(width, kBig) >= 256;
    // dx [R][H] over k = the piece; dw [piece][H] over k = R: k is split where the tiles alone do not fill the chip
    auto split = [&](int64_t n, int64_t k, bool& big) {
        big = ceil_div(n, kBig) * ceil_div(H, kBig) >= 128 && H > kSmall;
        const int edge = big ? kBig : kSmall;
        const int64_t tiles = ceil_div(n, edge) * ceil_div(H, edge), steps = ceil_div(k, kStepK);
        return (int)std::max<int64_t>(1, std::min<int64_t>({steps / 8, ceil_div(big ? 256 : 512, tiles), 64}));
    };
    p.dx_split = split(R, width, p.big_dx);
    p.dw_split = split(width, R, p.big_dw);
    if (p.dx_split > 1 || p.piece < V) p.dx_off = take((int64_t)p.dx_split * R * ld4 * 4);
    if (p.dw_split > 1) p.dw_off = take((int64_t)p.dw_split * width * (ld4 + 4) * 4);
    p.bytes = at;
    return p;
}

// calls fn(T{}, E{}, parts): the tensors' type, the products' operand type, the parts of an operand
template <typename Fn>
static int ce_types(int dtype, Fn&& fn) {
    if (dtype == CNF_DTYPE_F32) return fn(float{}, f16_t{}, std::integral_constant<int, 2>{});
    if (dtype == CNF_DTYPE_BF16) return fn(bf16_t{}, bf16_t{}, std::integral_constant<int, 1>{});
    return fn(f16_t{}, f16_t{}, std::integral_constant<int, 1>{});
}

// fp32 rows that vectors of 8 elements may be read from
static bool rows_aligned32(const void* p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0 && stride % 8 == 0; }

template <typename T, typename E, int PARTS>
static void ce_operands(CeArgs& a, const CePlan& p, const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* bias,
                        int bias_dtype, const int64_t* target, int64_t ignore, const int* known, int* exponents, int64_t R, int V, int H,
                        char* ws, hipStream_t st) {
    LayoutArgs l{};
    CeScales* scales = reinterpret_cast<CeScales*>(ws + p.scales_off);
    if constexpr (PARTS > 1) {
        // operands of few elements (at most 32 loads a lane): one launch less; with the rows finished by the walk itself, which saves
        // the join, 64 tokens of 51 classes and 64 features take 11.6 us instead of 17.1
        if (!known && std::max<int64_t>(R, V) * H > 8192) {
            Extent* extents = reinterpret_cast<Extent*>(ws + p.extents_off);
            CNF_LAUNCH(ce_extent_kernel, dim3(kMaxBlocks, 2), dim3(1024), 0, st, static_cast<const float*>(x), x_stride, R, target, ignore,
                       static_cast<const float*>(w), w_stride, V, H, extents);
            l.extents = extents;
        }
        l.known = known;
        l.scales = scales;
        l.exponents = exponents;
        l.target = target;
        l.ignore = ignore;
        a.x32 = Operand32{static_cast<const float*>(x), x_stride, R};
        a.w32 = Operand32{static_cast<const float*>(w), w_stride, V};
    }
    if (p.copy_x) l.job[0] = LayoutJob{x, x_stride, R, ws + p.x_off};
    if (p.copy_w) l.job[1] = LayoutJob{w, w_stride, V, ws + p.w_off};
    l.cols = H;
    // fp32 rows of whole 32-byte groups; 16-bit rows are only copied where they cannot be read that way
    if (sizeof(T) == 4 && H % 8 == 0) l.vec = (rows_aligned32(x, x_stride) ? 1 : 0) | (rows_aligned32(w, w_stride) ? 2 : 0);
    l.ld = p.ldh;
    if (p.narrow) {
        l.bias = bias;
        l.bias_dtype = bias_dtype;
        l.vocab = V;
        l.bias_pad = (int)round_up(V, kNarrowWalk);
        l.bias_out = reinterpret_cast<float*>(ws + p.bias_off);
    }
    if (p.copy_x || p.copy_w || p.narrow) {
        const int64_t chunks = std::max(p.copy_x ? R * (p.ldh / 8) : 0, p.copy_w ? V * (p.ldh / 8) : 0);
        const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(std::max<int64_t>(chunks, l.bias_pad), kBlock), 4096));
        CNF_LAUNCH((ce_layout_kernel<T, E, PARTS>), dim3(grid, 3), dim3(kBlock), 0, st, l);
    }
    a.x = p.copy_x ? Operand{ws + p.x_off, p.ldh, R * p.ldh, (int)R} : Operand{x, x_stride, 0, (int)R};
    a.w = p.copy_w ? Operand{ws + p.w_off, p.ldh, V * p.ldh, V} : Operand{w, w_stride, 0, V};
    a.pairs = p.pairs;
    a.parts = p.parts;
    a.rows = R;
    a.vocab = V;
    a.hidden = H;
    a.k_end = p.copy_x && p.copy_w ? (int)p.ldh : H;
    a.bias = bias;
    a.bias_dtype = bias_dtype;
    a.scales = scales;
    a.scaled = PARTS > 1;
    a.lift = sizeof(E) == 2 && std::is_same<E, f16_t>::value ? 16384.f : 1.f;
}

static NarrowArgs narrow_args(const CeArgs& a, const CePlan& p, bool rows_own, char* ws) {
    NarrowArgs n{};
    n.own = rows_own ? a.x : a.w;
    n.walk = rows_own ? a.w : a.x;
    n.own32 = rows_own ? a.x32 : a.w32;
    n.walk32 = rows_own ? a.w32 : a.x32;
    n.hidden = a.hidden;
    n.vocab = a.vocab;
    n.rows = a.rows;
    n.bias = reinterpret_cast<const float*>(ws + p.bias_off);
    n.target = a.target;
    n.ignore = a.ignore;
    n.partial = a.partial;
    n.target_logit = a.target_logit;
    n.splits = a.splits;
    n.state = a.state;
    n.scales = a.scales;
    n.scaled = a.scaled;
    n.lift = a.lift;
    return n;
}

static void ce_sum(const void* partial, int parts, int64_t rows, int cols, int64_t ld, void* out, int dtype, void* db, int db_dtype,
                   hipStream_t st) {
    const SumArgs a{static_cast<const float*>(partial), parts, rows, ld, cols, out, dtype, db, db_dtype};
    const int64_t n = rows * (cols + (db ? 1 : 0));
    if (parts > 16) CNF_LAUNCH(ce_sum_many_kernel, dim3((unsigned)ceil_div(n, 16)), dim3(1024), 0, st, a);
    else CNF_LAUNCH(ce_sum_kernel, dim3((unsigned)std::min<int64_t>(ceil_div(n, kBlock), 8192)), dim3(kBlock), 0, st, a);
}

// rows that the products may read as they are: whole 16-byte chunks, and 256 of them within reach of a 31-bit offset
static bool ce_aligned(const void* p, int64_t stride, int dtype, int H) {
    return rows_aligned16(p, stride, dtype) && H % 8 == 0 && stride < (1 << 21);
}

}  // namespace cnf

using namespace cnf;

#define CE_CHECK(name)                                                                                                             \
    CNF_REQUIRE(R >= 0 && V > 0 && H > 0 && R <= 0x7fffff00ll && V <= kMaxVocab && H <= kMaxHidden, name ": bad size R=%ld V=%d H=%d", \
                (long)R, V, H);                                                                                                    \
    CNF_REQUIRE(dtype_known(dtype) && dtype_known(bias_dtype), name ": unknown element type");                                     \
    CNF_REQUIRE(x_stride >= 0 && w_stride >= 0, name ": negative stride")

extern "C" {

int64_t cnf_linear_ce_workspace_bytes(int64_t R, int V, int H, int dtype, int backward) {
    if (R <= 0 || R > 0x7fffff00ll || V <= 0 || V > kMaxVocab || H <= 0 || H > kMaxHidden || !dtype_known(dtype)) return 0;
    return ce_plan(R, V, H, dtype, false, false, backward != 0).bytes;
}

int cnf_linear_ce(const void* x, int64_t x_stride, const void* weight, int64_t w_stride, const void* bias, const int64_t* target,
                  int64_t ignore_index, float* loss, float* row_max, float* row_sum, float* reduced, int* exponents, void* workspace, int64_t workspace_bytes,
                  int64_t R, int V, int H, int dtype, int bias_dtype, int* flags, cnf_stream_t stream) {
    CE_CHECK("cnf_linear_ce");
    hipStream_t st = (hipStream_t)stream;
    if (R > 0) {
        CNF_REQUIRE(x && weight && target && loss && row_max && row_sum, "cnf_linear_ce: null tensor");
        CNF_REQUIRE(workspace && workspace_bytes >= cnf_linear_ce_workspace_bytes(R, V, H, dtype, 0),
                    "cnf_linear_ce: workspace smaller than cnf_linear_ce_workspace_bytes");
        CNF_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "cnf_linear_ce: workspace not 16-byte aligned");
        const CePlan p = ce_plan(R, V, H, dtype, ce_aligned(x, x_stride, dtype, H), ce_aligned(weight, w_stride, dtype, H), false);
        char* ws = static_cast<char*>(workspace);
        const int rc = ce_types(dtype, [&](auto t, auto e, auto parts) {
            typedef decltype(t) T;
            typedef decltype(e) E;
            CeArgs a{};
            ce_operands<T, E, decltype(parts)::value>(a, p, x, x_stride, weight, w_stride, bias, bias_dtype, target, ignore_index, nullptr, exponents, R, V, H,
                                                     ws, st);
            a.target = target;
            a.ignore = ignore_index;
            a.partial = reinterpret_cast<float2*>(ws + p.partial_off);
            a.target_logit = reinterpret_cast<float*>(ws + p.logit_off);
            a.splits = p.splits;
            double* sums = reinterpret_cast<double*>(ws + p.sums_off);
            int64_t blocks = ceil_div(R * p.join_group, kBlock);
            if (p.narrow) {
                NarrowArgs n = narrow_args(a, p, true, ws);
                n.row_max = row_max;
                n.row_sum = row_sum;
                n.loss = loss;
                n.sums = sums;
                n.reduced = reduced;
                n.flags = flags;
                const int rc = narrow_launch(kNarrowLse, dtype, n, st);
                if (rc != CNF_OK) return rc;
            } else if (p.big_lse)
                CNF_LAUNCH((ce_lse_kernel<E, decltype(parts)::value, kBig, kBig, 2, 4>), dim3((unsigned)(ceil_div(R, kBig) * p.splits)), dim3(512), 0, st, a);
            else
                CNF_LAUNCH((ce_lse_kernel<E, decltype(parts)::value, kSmall, kSmall, 2, 2>), dim3((unsigned)(ceil_div(R, kSmall) * p.splits)), dim3(256), 0, st, a);
            if (p.narrow && p.splits == 1)
                blocks = ceil_div(R, kNarrowOwn);           // the rows are finished
            else
                CNF_LAUNCH(ce_join_kernel, dim3((unsigned)blocks), dim3(kBlock), 0, st, a.partial, a.target_logit, target, ignore_index, V, p.splits, p.join_group, R,
                           row_max, row_sum, loss, sums, reduced, flags);
            if (reduced && blocks > 1) CNF_LAUNCH(ce_reduce_kernel, dim3(1), dim3(1024), 0, st, sums, blocks, reduced);
            return launch_status("cnf_linear_ce");
        });
        if (rc != CNF_OK) return rc;
    } else if (reduced) {
        CNF_LAUNCH(ce_reduce_kernel, dim3(1), dim3(1024), 0, st, nullptr, (int64_t)0, reduced);
        return launch_status("cnf_linear_ce (no rows)");
    }
    return CNF_OK;
}

int cnf_linear_ce_bwd(const void* x, int64_t x_stride, const void* weight, int64_t w_stride, const void* bias, const int64_t* target,
                      int64_t ignore_index, const float* row_max, const float* row_sum, const int* exponents, const float* g, int g_per_row,
                      const float* count, void* dx, void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, int64_t R, int V, int H, int dtype,
                      int bias_dtype, cnf_stream_t stream) {
    CE_CHECK("cnf_linear_ce_bwd");
    CNF_REQUIRE(R > 0, "cnf_linear_ce_bwd: no rows");
    CNF_REQUIRE(x && weight && target && row_max && row_sum && g && (g_per_row || count) && (dx || dweight) && (dweight || !dbias), "cnf_linear_ce_bwd: null tensor");
    CNF_REQUIRE(workspace && workspace_bytes >= cnf_linear_ce_workspace_bytes(R, V, H, dtype, 1),
                "cnf_linear_ce_bwd: workspace smaller than cnf_linear_ce_workspace_bytes");
    CNF_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "cnf_linear_ce_bwd: workspace not 16-byte aligned");
    const CePlan p = ce_plan(R, V, H, dtype, ce_aligned(x, x_stride, dtype, H), ce_aligned(weight, w_stride, dtype, H), true);
    char* ws = static_cast<char*>(workspace);
    hipStream_t st = (hipStream_t)stream;
    return ce_types(dtype, [&](auto t, auto e, auto parts) {
        typedef decltype(t) T;
        typedef decltype(e) E;
        constexpr int PARTS = decltype(parts)::value;
        CeArgs a{};
        ce_operands<T, E, PARTS>(a, p, x, x_stride, weight, w_stride, bias, bias_dtype, target, ignore_index, exponents, nullptr, R, V, H,
                                 ws, st);
        RowState* state = reinterpret_cast<RowState*>(ws + p.state_off);
        a.state = state;
        // per-row gradients: every workgroup finds the largest |g| itself; few of them
        CNF_LAUNCH(ce_rows_kernel, dim3((unsigned)std::min<int64_t>(ceil_div(p.rows_pad, 1024), g_per_row ? 16 : 1024)), dim3(1024), 0, st, g,
                   g_per_row, count, row_max, row_sum, target, ignore_index, V, R, p.rows_pad, PARTS > 1 ? kGradSpan32 : kGradSpan16, state,
                   reinterpret_cast<CeScales*>(ws + p.scales_off));
        const int64_t ld4 = round_up(H, 4);
        if (p.narrow) {
            if (dx) {
                NarrowArgs n = narrow_args(a, p, true, ws);
                n.splits = p.dx_split;
                n.final_dtype = n.splits > 1 ? -1 : dtype;
                n.out = n.splits > 1 ? static_cast<void*>(ws + p.dx_off) : dx;
                n.ld = n.splits > 1 ? ld4 : H;
                const int rc = narrow_launch(kNarrowDx, dtype, n, st);
                if (rc != CNF_OK) return rc;
                if (n.splits > 1) ce_sum(n.out, n.splits, R, H, ld4, dx, dtype, nullptr, 0, st);
            }
            if (dweight) {
                NarrowArgs n = narrow_args(a, p, false, ws);
                n.splits = p.dw_split;
                n.final_dtype = n.splits > 1 ? -1 : dtype;
                n.out = n.splits > 1 ? static_cast<void*>(ws + p.dw_off) : dweight;
                n.ld = n.splits > 1 ? ld4 + 4 : H;
                n.db = dbias;
                n.db_dtype = bias_dtype;
                const int rc = narrow_launch(kNarrowDw, dtype, n, st);
                if (rc != CNF_OK) return rc;
                if (n.splits > 1) ce_sum(n.out, n.splits, V, H, n.ld, dweight, dtype, dbias, bias_dtype, st);
            }
            return launch_status("cnf_linear_ce_bwd");
        }
        a.d = ws + p.d_off;
        a.d_ld = p.piece;
        a.d_part = p.rows_pad * p.piece;
        const bool dx_partial = p.dx_split > 1 || p.piece < V, dw_partial = p.dw_split > 1;
        for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
            const int64_t v1 = std::min<int64_t>(V, v0 + p.piece), width = v1 - v0;
            a.v0 = (int)v0;
            a.v1 = (int)v1;
            const int edge = p.big_d ? kBig : kSmall;
            const unsigned d_grid = (unsigned)std::min<int64_t>(ceil_div(width, edge) * ceil_div(R, edge), p.big_d ? 256 : 512);
            auto logit_gradient = [&](int pass) {
                a.g_pass = pass;
                if (p.big_d) CNF_LAUNCH((ce_d_kernel<E, PARTS, kBig, kBig, 2, 4>), dim3(d_grid), dim3(512), 0, st, a);
                else CNF_LAUNCH((ce_d_kernel<E, PARTS, kSmall, kSmall, 2, 2>), dim3(d_grid), dim3(256), 0, st, a);
            };
            const bool may_part = std::is_same<E, f16_t>::value && g_per_row && dx;
            logit_gradient(may_part ? 1 : 0);
            const Operand d{a.d, a.d_ld, a.d_part, 0};
            GradArgs q{};
            q.pairs = p.pairs;
            q.m_end = H;
            // dx[r][h] += sum_v w[v][h] d[r][v]
            q.a = Operand{static_cast<const uint16_t*>(a.w.base) + v0 * a.w.ld, a.w.ld, a.w.part, H};
            q.b = d;
            q.b.ext = (int)R;
            q.a32 = Operand32{a.w32.base + v0 * a.w32.ld, a.w32.ld, H};
            q.b32 = Operand32{static_cast<const float*>(a.d), a.d_ld, R};
            q.k_end = (int)width;
            q.n_end = (int)R;
            q.ksplit = p.dx_split;
            q.final_dtype = dx_partial ? -1 : dtype;
            q.out = dx_partial ? static_cast<void*>(ws + p.dx_off) : dx;
            q.ld = dx_partial ? ld4 : H;
            q.accumulate = v0 > 0;
            q.scales = a.scales;
            q.scaled = a.scaled ? 2 : 0;
            q.lift = a.lift;
            auto grad = [&](bool kmb, bool big, int64_t n) {
                const int64_t edge = big ? kBig : kSmall;
                const dim3 grid((unsigned)(ceil_div(n, edge) * ceil_div(H, edge) * q.ksplit));
                if (kmb && big) CNF_LAUNCH((ce_grad_kernel<E, PARTS, true, kBig, kBig, 2, 4>), grid, dim3(512), 0, st, q);
                else if (kmb) CNF_LAUNCH((ce_grad_kernel<E, PARTS, true, kSmall, kSmall, 2, 2>), grid, dim3(256), 0, st, q);
                else if (big) CNF_LAUNCH((ce_grad_kernel<E, PARTS, false, kBig, kBig, 2, 4>), grid, dim3(512), 0, st, q);
                else CNF_LAUNCH((ce_grad_kernel<E, PARTS, false, kSmall, kSmall, 2, 2>), grid, dim3(256), 0, st, q);
            };
            q.state = may_part ? state : nullptr;
            if (dx) grad(false, p.big_dx, R);
            if (!dweight) continue;
            if (may_part) logit_gradient(2);
            // dw[v][h] = sum_r x[r][h] d[r][v]; db[v] = sum_r d[r][v]
            char* dw = static_cast<char*>(dweight) + v0 * H * dtype_bytes(dtype);
            char* db = dbias ? static_cast<char*>(dbias) + v0 * dtype_bytes(bias_dtype) : nullptr;
            q.a = a.x;
            q.a.ext = H;
            q.b = d;
            q.b.ext = (int)width;
            q.a32 = Operand32{a.x32.base, a.x32.ld, H};
            q.b32.ext = width;
            q.state = state;
            q.k_end = (int)R;
            q.n_end = (int)width;
            q.ksplit = p.dw_split;
            q.final_dtype = dw_partial ? -1 : dtype;
            q.out = dw_partial ? static_cast<void*>(ws + p.dw_off) : dw;
            q.ld = dw_partial ? ld4 + 4 : H;
            q.accumulate = 0;
            q.scaled = a.scaled ? 1 : 0;
            q.db = db;
            q.db_dtype = bias_dtype;
            grad(true, p.big_dw, width);
            if (dw_partial) ce_sum(ws + p.dw_off, p.dw_split, width, H, q.ld, dw, dtype, db, bias_dtype, st);
        }
        if (dx && dx_partial) ce_sum(ws + p.dx_off, p.dx_split, R, H, ld4, dx, dtype, nullptr, 0, st);
        return launch_status("cnf_linear_ce_bwd");
    });
}

}  // extern "C"
