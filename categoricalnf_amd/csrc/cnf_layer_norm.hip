// Layer norm over the last axis, forward and backward, with the weight's and bias's gradients.
//
//   xhat = (x - mean) rstd,  y = xhat w + b,  mean and rstd per row in fp32 (variance from the centred values: two passes over
//   registers, so a large common offset of a row does not cancel)
//   dx = rstd (g w - mean_c(g w) - xhat mean_c(g w xhat)),   dw = sum_r g xhat,   db = sum_r g
//
// Bound by HBM: the forward reads x and writes y, the backward reads x and g and writes dx, each once.  A row lives in the
// registers of the lanes that own it — a group of G lanes of a wave (up to 1024 columns; 64 / G rows per wave) or a whole
// workgroup (up to 16 384) —, at most 16 elements per lane.  The backward's lanes own the same columns in every row they walk, so
// the two column sums stay in registers over the whole launch; each workgroup writes one partial row of 2 C sums, and a second
// launch adds the partial rows in their order (the same bits on every run, no atomics).  Longer rows take kernels that read a row
// three times (forward) or twice (backward) and sum the columns in a launch of their own.
//
// Waves in flight are what keeps HBM busy: the forward holds its next row's loads while it works on one; the backward has registers for
// that only at the price of a wave per SIMD, and computes xhat and g w twice instead of holding them (202 -> 166 us).  131072 x 1024 bf16:
// forward 102 us (5.2 TB/s), backward 162 us and 8 for the column sums (4.9 TB/s; a plain copy: 4.97).  Rows that begin at odd addresses
// are read in 16-byte vectors all the same: 4933 x 7438 bf16 forward 44 us, backward 70 us (7440 columns: 27 and 54; floors 30 and 44).
#include <algorithm>
#include <type_traits>

#include "cnf_dtype.h"

namespace cnf {

constexpr int kLnElems = 16;                        // elements of a row one lane holds at most
constexpr int kLnWaveCols = kWave * kLnElems;       // widest row of one wave
constexpr int kLnBlockCols = 1024 * kLnElems;       // widest row of one workgroup
constexpr int kLnMaxPartials = 1024;                // partial rows of the column sums
constexpr int kLnMaxCols = 1 << 30;                 // what 32-bit column counters reach

struct LnArgs {
    const void *x, *dy, *weight, *bias;
    void *y, *dx;
    float *mean, *rstd;
    float* partials;
    int64_t x_stride, dy_stride, y_stride;          // elements between rows (dx has y_stride)
    int64_t rows;
    int cols, wdtype, group;                        // group: lanes per row (wave kernels)
    float eps;
};

// sum over the lanes that share a row: a power-of-two group of a wave, or the workgroup
struct WaveGroup {
    int g;
    __device__ __forceinline__ float sum(float v) const { return group_sum(v, g); }
    __device__ __forceinline__ Sum2 sum(Sum2 v) const { return group_sum(v, g); }
};
struct BlockGroup {
    float* sh;      // 2 x 16 floats
    __device__ __forceinline__ Sum2 sum(Sum2 v) const {
        v = wave_sum(v);
        const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
        __syncthreads();                            // the previous sum has been read
        if ((threadIdx.x & 63) == 0) {
            sh[wave] = v.a;
            sh[16 + wave] = v.b;
        }
        __syncthreads();
        Sum2 t(0);
        for (int w = 0; w < waves; ++w) t += Sum2(sh[w], sh[16 + w]);
        return t;
    }
    __device__ __forceinline__ float sum(float v) const { return sum(Sum2(v, 0.f)).a; }
};

// 16 bytes of a row, at any address its elements may have (the hardware takes them in one access); TAIL: the row's last vector may be
// shorter, and goes element by element
template <bool TAIL, typename T, int VEC>
__device__ __forceinline__ void ln_read(const T* row, int c, int cols, vec_t<T, VEC>& v) {
    if (!TAIL || c + VEC <= cols) {
        __builtin_memcpy(&v, row + c, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + i < cols) v[i] = row[c + i];
    }
}
template <bool TAIL, typename T, int VEC>
__device__ __forceinline__ void ln_write(T* row, int c, int cols, const vec_t<T, VEC>& v) {
    if (!TAIL || c + VEC <= cols) {
        __builtin_memcpy(row + c, &v, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + i < cols) row[c + i] = v[i];
    }
}

template <bool TAIL, typename T, int VEC, int NV>
__device__ __forceinline__ void ln_load(const T* row, int l, int lanes, int cols, bool on, vec_t<T, VEC>* v) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * lanes + l) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] = (T)0.f;
        if (on && c < cols) ln_read<TAIL, T, VEC>(row, c, cols, v[j]);
    }
}

template <int VEC, int NV>
__device__ __forceinline__ void ln_load_weight(const void* w, int wdtype, int l, int lanes, int cols, float fill, float* out) {
#pragma unroll
    for (int e = 0; e < NV * VEC; ++e) out[e] = fill;
    if (!w) return;
    auto load = [&](auto t) {
        typedef decltype(t) W;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * lanes + l) * VEC;
            vec_t<W, VEC> v;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = (W)fill;
            if (c < cols) ln_read<true, W, VEC>(static_cast<const W*>(w), c, cols, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) out[j * VEC + i] = (float)v[i];
        }
    };
    if (wdtype == CNF_DTYPE_F32) load(float{});
    else if (wdtype == CNF_DTYPE_BF16) load(bf16_t{});
    else load(f16_t{});
}

template <bool TAIL, typename T, int VEC, int NV, typename Group>
__device__ __forceinline__ void ln_fwd_row(const LnArgs& a, const vec_t<T, VEC>* xv, int64_t row, bool on, int l, int lanes,
                                           const Group& grp, const float* w, const float* b) {
    float x[NV * VEC], s = 0.f;
#pragma unroll
    for (int e = 0; e < NV * VEC; ++e) {
        x[e] = (float)xv[e / VEC][e % VEC];
        s += x[e];
    }
    const float inv = 1.f / (float)a.cols;
    const float mean = grp.sum(s) * inv;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * lanes + l) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float& v = x[j * VEC + i];
            v = (TAIL ? c + i : c) < a.cols ? v - mean : 0.f;
            q += v * v;
        }
    }
    const float rstd = 1.f / sqrtf(grp.sum(q) * inv + a.eps);
    if (!on) return;
    T* y = static_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * lanes + l) * VEC;
        if (c >= a.cols) continue;
        vec_t<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = (T)(x[j * VEC + i] * rstd * w[j * VEC + i] + b[j * VEC + i]);
        ln_write<TAIL, T, VEC>(y, c, a.cols, o);
    }
    if (l == 0 && a.mean) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
}

template <bool TAIL, typename T, int VEC, int NV>
__global__ __launch_bounds__(kBlock) void ln_fwd_wave_kernel(const LnArgs a) {
    const int g = a.group, rpw = kWave / g;
    const int lane = threadIdx.x & 63, l = lane & (g - 1);
    const int slot = (threadIdx.x >> 6) * rpw + lane / g, rpb = kWavesPerBlock * rpw;
    float w[NV * VEC], b[NV * VEC];
    ln_load_weight<VEC, NV>(a.weight, a.wdtype, l, g, a.cols, 1.f, w);
    ln_load_weight<VEC, NV>(a.bias, a.wdtype, l, g, a.cols, 0.f, b);
    const WaveGroup grp{g};
    // the next row's loads are in flight while a row is worked on
    const int64_t step = (int64_t)gridDim.x * rpb;
    vec_t<T, VEC> now[NV], next[NV];
    int64_t r = (int64_t)blockIdx.x * rpb + slot;
    ln_load<TAIL, T, VEC, NV>(static_cast<const T*>(a.x) + r * a.x_stride, l, g, a.cols, r < a.rows, next);
    for (int64_t r0 = (int64_t)blockIdx.x * rpb; r0 < a.rows; r0 += step, r += step) {
#pragma unroll
        for (int j = 0; j < NV; ++j) now[j] = next[j];
        if (r0 + step < a.rows)
            ln_load<TAIL, T, VEC, NV>(static_cast<const T*>(a.x) + (r + step) * a.x_stride, l, g, a.cols, r + step < a.rows, next);
        ln_fwd_row<TAIL, T, VEC, NV>(a, now, r, r < a.rows, l, g, grp, w, b);
    }
}

template <bool TAIL, typename T, int VEC, int NV>
__global__ __launch_bounds__(1024) void ln_fwd_block_kernel(const LnArgs a) {
    __shared__ float sh[32];
    const BlockGroup grp{sh};
    float w[NV * VEC], b[NV * VEC];
    ln_load_weight<VEC, NV>(a.weight, a.wdtype, threadIdx.x, blockDim.x, a.cols, 1.f, w);
    ln_load_weight<VEC, NV>(a.bias, a.wdtype, threadIdx.x, blockDim.x, a.cols, 0.f, b);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        vec_t<T, VEC> xv[NV];
        ln_load<TAIL, T, VEC, NV>(static_cast<const T*>(a.x) + r * a.x_stride, threadIdx.x, blockDim.x, a.cols, true, xv);
        ln_fwd_row<TAIL, T, VEC, NV>(a, xv, r, true, threadIdx.x, blockDim.x, grp, w, b);
    }
}

// the same values, as if just loaded: the compiler keeps nothing that it has computed from them
template <typename T, int VEC>
__device__ __forceinline__ vec_t<T, VEC> opaque(vec_t<T, VEC> v) {
    if constexpr (sizeof(v) % 4 == 0) {
        typedef vec_t<uint32_t, sizeof(v) / 4> words_t;
        words_t w = __builtin_bit_cast(words_t, v);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(v) / 4); ++i) {
            uint32_t one = w[i];
            asm volatile("" : "+v"(one));
            w[i] = one;
        }
        return __builtin_bit_cast(vec_t<T, VEC>, w);
    }
    return v;
}

// what the backward reads of one row
template <bool TAIL, typename T, int VEC, int NV>
struct LnRow {
    vec_t<T, VEC> x[NV], g[NV];
    float mean, rstd;
    __device__ __forceinline__ void load(const LnArgs& a, int64_t row, bool on, int l, int lanes) {
        ln_load<TAIL, T, VEC, NV>(static_cast<const T*>(a.x) + row * a.x_stride, l, lanes, a.cols, on, x);
        ln_load<TAIL, T, VEC, NV>(static_cast<const T*>(a.dy) + row * a.dy_stride, l, lanes, a.cols, on, g);
        mean = on ? a.mean[row] : 0.f;
        rstd = on ? a.rstd[row] : 0.f;
    }
};

template <bool TAIL, typename T, int VEC, int NV, typename Group>
__device__ __forceinline__ void ln_bwd_row(const LnArgs& a, LnRow<TAIL, T, VEC, NV>& in_row, int64_t row, bool on, int l, int lanes,
                                           const Group& grp, const float* w, float* dw, float* db) {
    vec_t<T, VEC>*xv = in_row.x, *gv = in_row.g;
    const float mean = in_row.mean, rstd = in_row.rstd;
    Sum2 s(0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int e = j * VEC + i;
            // past the last column g is 0
            const float g = (float)gv[j][i], xh = ((float)xv[j][i] - mean) * rstd, gw = g * w[e];
            dw[e] += g * xh;
            db[e] += g;
            s += Sum2(gw, gw * xh);
        }
    }
    s = grp.sum(s);
    // xhat and g w are computed again rather than held: x and g as loaded take half the registers (or fewer)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        xv[j] = opaque<T, VEC>(xv[j]);
        gv[j] = opaque<T, VEC>(gv[j]);
    }
    if (!on) return;
    const float inv = 1.f / (float)a.cols, c1 = s.a * inv, c2 = s.b * inv;
    T* dx = static_cast<T*>(a.dx) + row * a.y_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * lanes + l) * VEC;
        if (c >= a.cols) continue;
        vec_t<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float xh = ((float)xv[j][i] - mean) * rstd, gw = (float)gv[j][i] * w[j * VEC + i];
            o[i] = (T)(rstd * (gw - c1 - xh * c2));
        }
        ln_write<TAIL, T, VEC>(dx, c, a.cols, o);
    }
}

// partials: [gridDim.x][2][cols]
template <bool TAIL, typename T, int VEC, int NV>
__global__ __launch_bounds__(kBlock) void ln_bwd_wave_kernel(const LnArgs a) {
    __shared__ float sh[kWavesPerBlock][kLnWaveCols];
    const int g = a.group, rpw = kWave / g;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & (g - 1);
    const int slot = wave * rpw + lane / g, rpb = kWavesPerBlock * rpw;
    float w[NV * VEC], acc[2][NV * VEC];
    ln_load_weight<VEC, NV>(a.weight, a.wdtype, l, g, a.cols, 1.f, w);
#pragma unroll
    for (int e = 0; e < NV * VEC; ++e) acc[0][e] = acc[1][e] = 0.f;
    const WaveGroup grp{g};
    for (int64_t r0 = (int64_t)blockIdx.x * rpb; r0 < a.rows; r0 += (int64_t)gridDim.x * rpb) {
        LnRow<TAIL, T, VEC, NV> in_row;
        in_row.load(a, r0 + slot, r0 + slot < a.rows, l, g);
        ln_bwd_row<TAIL, T, VEC, NV>(a, in_row, r0 + slot, r0 + slot < a.rows, l, g, grp, w, acc[0], acc[1]);
    }
    if (!a.partials) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int e = 0; e < NV * VEC; ++e) {
            float v = acc[k][e];
            for (int m = g; m < kWave; m <<= 1) v += __shfl_xor(v, m, kWave);       // the wave's row groups
            const int c = ((e / VEC) * g + l) * VEC + e % VEC;
            if (lane < g && c < a.cols) sh[wave][c] = v;
        }
        __syncthreads();
        float* out = a.partials + ((size_t)blockIdx.x * 2 + k) * a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kBlock) {
            float t = 0.f;
#pragma unroll
            for (int q = 0; q < kWavesPerBlock; ++q) t += sh[q][c];
            out[c] = t;
        }
        __syncthreads();
    }
}

// THREADS at most: 1024, or 512 for fp32, whose rows want 134 registers where 1024 threads have 128 (25079 x 3034: 282 -> 250 us)
template <int THREADS, bool TAIL, typename T, int VEC, int NV>
__global__ __launch_bounds__(THREADS) void ln_bwd_block_kernel(const LnArgs a) {
    __shared__ float sh[32];
    const BlockGroup grp{sh};
    float w[NV * VEC], acc[2][NV * VEC];
    ln_load_weight<VEC, NV>(a.weight, a.wdtype, threadIdx.x, blockDim.x, a.cols, 1.f, w);
#pragma unroll
    for (int e = 0; e < NV * VEC; ++e) acc[0][e] = acc[1][e] = 0.f;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        LnRow<TAIL, T, VEC, NV> in_row;
        in_row.load(a, r, true, threadIdx.x, blockDim.x);
        ln_bwd_row<TAIL, T, VEC, NV>(a, in_row, r, true, threadIdx.x, blockDim.x, grp, w, acc[0], acc[1]);
    }
    if (!a.partials) return;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * blockDim.x + threadIdx.x) * VEC;
            vec_t<float, VEC> v;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = acc[k][j * VEC + i];
            if (c < a.cols) ln_write<TAIL, float, VEC>(a.partials + ((size_t)blockIdx.x * 2 + k) * a.cols, c, a.cols, v);
        }
}

// ---- rows wider than a workgroup's registers: the row is read again instead of held ---------------------------------------------

// calls fn(first column, its 16 bytes) for this lane's part of a row
template <typename T, typename Fn>
__device__ __forceinline__ void ln_walk(const T* row, int cols, Fn&& fn) {
    constexpr int V = 16 / (int)sizeof(T);
    for (int c = threadIdx.x * V; c < cols; c += 1024 * V) {
        vec_t<T, V> v;
        ln_read<true, T, V>(row, c, cols, v);
        fn(c, v);
    }
}
template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const LnArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ float sh[32];
    const BlockGroup grp{sh};
    const float inv = 1.f / (float)a.cols;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        T* y = static_cast<T*>(a.y) + r * a.y_stride;
        float s = 0.f, q = 0.f;
        ln_walk<T>(x, a.cols, [&](int c, const vec_t<T, V>& v) {
#pragma unroll
            for (int i = 0; i < V; ++i) s += c + i < a.cols ? (float)v[i] : 0.f;
        });
        const float mean = grp.sum(s) * inv;
        ln_walk<T>(x, a.cols, [&](int c, const vec_t<T, V>& v) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = c + i < a.cols ? (float)v[i] - mean : 0.f;
                q += d * d;
            }
        });
        const float rstd = 1.f / sqrtf(grp.sum(q) * inv + a.eps);
        ln_walk<T>(x, a.cols, [&](int c, const vec_t<T, V>& v) {
            float w[V], b[V];
            ln_load_weight<V, 1>(a.weight, a.wdtype, c / V, 1, a.cols, 1.f, w);
            ln_load_weight<V, 1>(a.bias, a.wdtype, c / V, 1, a.cols, 0.f, b);
            vec_t<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = (T)(((float)v[i] - mean) * rstd * w[i] + b[i]);
            ln_write<true, T, V>(y, c, a.cols, o);
        });
        if (threadIdx.x == 0 && a.mean) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(const LnArgs a) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ float sh[32];
    const BlockGroup grp{sh};
    const float inv = 1.f / (float)a.cols;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        const T* g = static_cast<const T*>(a.dy) + r * a.dy_stride;
        T* dx = static_cast<T*>(a.dx) + r * a.y_stride;
        const float mean = a.mean[r], rstd = a.rstd[r];
        Sum2 s(0);
        ln_walk<T>(x, a.cols, [&](int c, const vec_t<T, V>& v) {
            vec_t<T, V> gv;
            float w[V];
            ln_read<true, T, V>(g, c, a.cols, gv);
            ln_load_weight<V, 1>(a.weight, a.wdtype, c / V, 1, a.cols, 1.f, w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float gw = c + i < a.cols ? (float)gv[i] * w[i] : 0.f, xh = c + i < a.cols ? ((float)v[i] - mean) * rstd : 0.f;
                s += Sum2(gw, gw * xh);
            }
        });
        s = grp.sum(s);
        const float c1 = s.a * inv, c2 = s.b * inv;
        ln_walk<T>(x, a.cols, [&](int c, const vec_t<T, V>& v) {
            vec_t<T, V> gv, o;
            float w[V];
            ln_read<true, T, V>(g, c, a.cols, gv);
            ln_load_weight<V, 1>(a.weight, a.wdtype, c / V, 1, a.cols, 1.f, w);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = (T)(rstd * ((float)gv[i] * w[i] - c1 - ((float)v[i] - mean) * rstd * c2));
            ln_write<true, T, V>(dx, c, a.cols, o);
        });
    }
}

// column sums of long rows: a workgroup owns 256 columns of every gridDim.y-th row
template <typename T>
__global__ __launch_bounds__(kBlock) void ln_columns_kernel(const LnArgs a) {
    const int c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= a.cols) return;
    float dw = 0.f, db = 0.f;
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float g = (float)static_cast<const T*>(a.dy)[r * a.dy_stride + c];
        dw += g * (((float)static_cast<const T*>(a.x)[r * a.x_stride + c] - a.mean[r]) * a.rstd[r]);
        db += g;
    }
    a.partials[((size_t)blockIdx.y * 2) * a.cols + c] = dw;
    a.partials[((size_t)blockIdx.y * 2 + 1) * a.cols + c] = db;
}

// partial rows -> dweight, dbias.  A workgroup owns 16 columns of the 2 C sums (one 64-byte segment per partial row); its 64 row
// slots each add every 64th partial row, then the slots are added in order.
__global__ __launch_bounds__(1024) void ln_reduce_kernel(const float* __restrict__ partials, int nparts, int cols, int wdtype,
                                                         void* dweight, void* dbias) {
    __shared__ float sh[64][17];
    const int cl = threadIdx.x & 15, slot = threadIdx.x >> 4;
    const int64_t width = 2 * (int64_t)cols;
    for (int64_t k = (int64_t)blockIdx.x * 16 + cl; k - cl < width; k += (int64_t)gridDim.x * 16) {
        float t = 0.f;
        if (k < width)
            for (int p = slot; p < nparts; p += 64) t += partials[(size_t)p * width + k];
        sh[slot][cl] = t;
        __syncthreads();
        if (slot == 0 && k < width) {
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < 64; ++q) v += sh[q][cl];
            if (k < cols) {
                if (dweight) store_any(dweight, wdtype, k, v);
            } else if (dbias) {
                store_any(dbias, wdtype, k - cols, v);
            }
        }
        __syncthreads();                            // the sums have been read
    }
}

// How a launch deals rows to lanes.  16-byte vectors where every row allows it; otherwise single elements.
struct LnShape {
    bool tail;      // the last 16-byte vector of a row is shorter
    int nv;         // vectors per lane: 1, or the most that keeps 16 elements
    int group;      // lanes per row; > 64: the workgroup's size
    int kind;       // 0 wave, 1 workgroup, 2 long rows
};
static LnShape ln_shape(int cols, int dtype, bool backward) {
    LnShape s;
    const int width = 16 / dtype_bytes(dtype), units = (cols + width - 1) / width, most = kLnElems / width;
    s.tail = cols % width != 0;
    // Short rows: one vector per lane keeps the lanes of a wave busy; the forward, with less to do per vector, sooner takes more of them
    // (44992 x 128 fp32, 32 vectors a row, one / four a lane: forward 11.2 / 9.6 us, backward 21.3 / 26.1; x 512 bf16, 64 vectors, one /
    // two: 20.8 / 18.7 and 37.1 / 35.5)
    s.nv = units <= (backward ? 32 : 16) ? 1 : most;
    int g = 1;
    while ((int64_t)g * s.nv < units) g <<= 1;
    s.kind = cols > kLnBlockCols ? 2 : (g > kWave ? 1 : 0);
    s.group = s.kind == 1 && g < kBlock ? kBlock : g;
    return s;
}

static int ln_partials(int64_t rows, const LnShape& s) {
    if (s.kind == 2) return (int)std::min<int64_t>(rows, 64);
    const int rpb = s.kind == 1 ? 1 : kWavesPerBlock * (kWave / s.group);
    const int64_t steps = (rows + rpb - 1) / rpb;
    // at least 8 steps of rows per workgroup before there are more than 256 of them: each workgroup writes 2 C sums at its end; of large
    // workgroups no more than run at once
    const int64_t most = s.kind == 1 ? std::min(kLnMaxPartials, 256 * 1024 / s.group) : kLnMaxPartials;
    return (int)std::min<int64_t>(steps, std::max<int64_t>(256, std::min<int64_t>(most, steps / 8)));
}

// calls wave or block with (tail, vector width, vectors per lane) as constants
template <typename T, typename Wave, typename Block>
static void ln_pick(const LnShape& s, Wave&& wave, Block&& block) {
    constexpr int V = 16 / (int)sizeof(T);
    auto pick = [&](auto tail) {
        std::integral_constant<int, V> width;
        std::integral_constant<int, kLnElems / V> most;
        if (s.kind == 1) block(tail, width, most);
        else if (s.nv == 1) wave(tail, width, std::integral_constant<int, 1>{});
        else wave(tail, width, most);
    };
    if (s.tail) pick(std::true_type{});
    else pick(std::false_type{});
}

}  // namespace cnf

using namespace cnf;

extern "C" {

int cnf_layer_norm(const void* x, int64_t x_stride, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                   int64_t rows, int cols, float eps, int dtype, int wdtype, cnf_stream_t stream) {
    CNF_REQUIRE(x && y, "cnf_layer_norm: null tensor");
    CNF_REQUIRE(rows >= 0 && cols > 0 && cols <= kLnMaxCols && x_stride >= 0, "cnf_layer_norm: bad size rows=%ld cols=%d", (long)rows, cols);
    CNF_REQUIRE(dtype_known(dtype) && dtype_known(wdtype), "cnf_layer_norm: unknown element type");
    CNF_REQUIRE(!mean == !rstd, "cnf_layer_norm: mean and rstd come together");
    if (rows == 0) return CNF_OK;
    LnArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.y = y; a.mean = mean; a.rstd = rstd;
    a.x_stride = x_stride; a.y_stride = cols; a.rows = rows; a.cols = cols; a.wdtype = wdtype; a.eps = eps;
    const LnShape s = ln_shape(cols, dtype, false);
    a.group = s.group;
    hipStream_t st = (hipStream_t)stream;
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        if (s.kind == 2) {
            CNF_LAUNCH((ln_fwd_long_kernel<T>), dim3((unsigned)std::min<int64_t>(rows, 2048)), dim3(1024), 0, st, a);
        } else {
            ln_pick<T>(s,
                       [&](auto tail, auto v, auto n) {
                           const int rpb = kWavesPerBlock * (kWave / s.group);
                           const unsigned grid = (unsigned)std::min<int64_t>((rows + rpb - 1) / rpb, 4096);
                           CNF_LAUNCH((ln_fwd_wave_kernel<decltype(tail)::value, T, decltype(v)::value, decltype(n)::value>), dim3(grid), dim3(kBlock), 0, st, a);
                       },
                       [&](auto tail, auto v, auto n) {
                           CNF_LAUNCH((ln_fwd_block_kernel<decltype(tail)::value, T, decltype(v)::value, decltype(n)::value>),
                                      dim3((unsigned)std::min<int64_t>(rows, 4096)), dim3(s.group), 0, st, a);
                       });
        }
        return launch_status("cnf_layer_norm");
    });
}

int64_t cnf_layer_norm_bwd_workspace_floats(int64_t rows, int cols) {
    if (rows <= 0 || cols <= 0 || cols > kLnMaxCols) return 0;
    // the largest partials matrix over the types
    int64_t most = 0;
    for (int dtype : {CNF_DTYPE_F32, CNF_DTYPE_BF16}) most = std::max<int64_t>(most, ln_partials(rows, ln_shape(cols, dtype, true)));
    return most * 2 * cols;
}

int cnf_layer_norm_bwd(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, const void* weight,
                       const float* mean, const float* rstd, void* dx, void* dweight, void* dbias, float* ws, int64_t ws_floats,
                       int64_t rows, int cols, int dtype, int wdtype, cnf_stream_t stream) {
    CNF_REQUIRE(x && dy && mean && rstd && dx, "cnf_layer_norm_bwd: null tensor");
    CNF_REQUIRE(rows >= 0 && cols > 0 && cols <= kLnMaxCols && x_stride >= 0 && dy_stride >= 0, "cnf_layer_norm_bwd: bad size rows=%ld cols=%d", (long)rows, cols);
    CNF_REQUIRE(dtype_known(dtype) && dtype_known(wdtype), "cnf_layer_norm_bwd: unknown element type");
    const bool sums = dweight || dbias;
    CNF_REQUIRE(!sums || rows == 0 || (ws && ws_floats >= cnf_layer_norm_bwd_workspace_floats(rows, cols)),
                "cnf_layer_norm_bwd: workspace smaller than cnf_layer_norm_bwd_workspace_floats");
    LnArgs a{};
    a.x = x; a.dy = dy; a.weight = weight; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd); a.dx = dx;
    a.x_stride = x_stride; a.dy_stride = dy_stride; a.y_stride = cols; a.rows = rows; a.cols = cols; a.wdtype = wdtype;
    a.partials = sums ? ws : nullptr;
    const LnShape s = ln_shape(cols, dtype, true);
    a.group = s.group;
    const int parts = rows > 0 ? ln_partials(rows, s) : 0;
    hipStream_t st = (hipStream_t)stream;
    if (rows > 0) {
        const int rc = with_dtype(dtype, [&](auto t) {
            typedef decltype(t) T;
            if (s.kind == 2) {
                CNF_LAUNCH((ln_bwd_long_kernel<T>), dim3((unsigned)std::min<int64_t>(rows, 2048)), dim3(1024), 0, st, a);
                if (sums)
                    CNF_LAUNCH((ln_columns_kernel<T>), dim3((cols + kBlock - 1) / kBlock, parts), dim3(kBlock), 0, st, a);
            } else {
                ln_pick<T>(s,
                           [&](auto tail, auto v, auto n) {
                               CNF_LAUNCH((ln_bwd_wave_kernel<decltype(tail)::value, T, decltype(v)::value, decltype(n)::value>), dim3(parts), dim3(kBlock), 0, st, a);
                           },
                           [&](auto tail, auto v, auto n) {
                               auto launch = [&](auto threads) {
                                   CNF_LAUNCH((ln_bwd_block_kernel<decltype(threads)::value, decltype(tail)::value, T, decltype(v)::value, decltype(n)::value>),
                                              dim3(parts), dim3(s.group), 0, st, a);
                               };
                               if (sizeof(T) == 4 && s.group <= 512) launch(std::integral_constant<int, sizeof(T) == 4 ? 512 : 1024>{});
                               else launch(std::integral_constant<int, 1024>{});
                           });
            }
            return launch_status("cnf_layer_norm_bwd");
        });
        if (rc != CNF_OK) return rc;
    }
    if (sums) {
        // a grid has less than 2^32 threads: 2^25 columns would reach that
        const unsigned grid = (unsigned)std::min<int64_t>((2 * (int64_t)cols + 15) / 16, 1 << 21);
        CNF_LAUNCH(ln_reduce_kernel, dim3(grid), dim3(1024), 0, st, ws, parts, cols, wdtype, dweight, dbias);
        return launch_status("cnf_layer_norm_bwd (column sums)");
    }
    return CNF_OK;
}

}  // extern "C"
