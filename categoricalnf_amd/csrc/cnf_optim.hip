// One AdamW step over a list of tensors, moments in fp32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Every product, sum, square root and quotient is one correctly rounded fp32 operation in this order (no contraction), so the
// result is that of the same chain of elementwise tensor operations; p in 16 bits is rounded once, to nearest, when it is stored.
//
// 8-bit moments: 256 consecutive elements of a tensor share two fp32 scales.  m = s q |q| with q in -127 .. 127 and s = max|m| / 127^2;
// sqrt(v) = s q^2 with q in 0 .. 255 and s = max sqrt(v) / 255^2.  The quadratic grid is fine near zero, where most moments of a
// block lie (smallest step: 6e-5 of the largest |m|, 1.5e-5 of the largest sqrt(v)).  An element with v > 0 keeps q >= 1: a second
// moment rounded to nothing would divide its step by eps.  The step itself uses the new moments before they are rounded.  A block
// with a non-finite moment gets the scale NaN and codes 0: it reads back as NaN, as the fp32 moments of such an element would.
//
// Bound by HBM: 28 bytes per fp32 element (16 with 8-bit moments, plus 8 / 256).  The tensors' addresses travel in the kernel
// arguments (up to 4 KB: 98 tensors a launch, 70 with scales): nothing is uploaded, so a launch may be captured and replayed, and
// nothing on the device has to outlive it.  A workgroup owns 1024 (2048 with 8-bit moments) consecutive elements of one tensor, found by counting
// the tensors that begin at or before it; each lane has one or two 4-element units of every array in flight.  Measured: 420 M bf16
// elements with fp32 moments 1595 us (5.8 TB/s), 84 M fp32 elements with 8-bit moments 280 us (4.8 TB/s), 27 M elements in 820
// tensors 189 us in 9 launches (4.0 TB/s: a launch of 20 us fills and drains the chip for some of them).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "cnf_dtype.h"

namespace cnf {

// elements of a workgroup, 4 or 8 a lane: fp32 moments want many short workgroups (420 M bf16 elements with 4096, 2048, 1024 each: 1730,
// 1721, 1597 us), 8-bit ones a little arithmetic to hide loads behind (84 M: 340, 285, 308 us)
template <int BITS>
constexpr int kAdamChunk = BITS == 8 ? 2048 : 1024;

struct AdamConst {
    float beta1, one_beta1, beta2, one_beta2, eps, keep, size, root;
};

template <int BITS>
struct AdamArgs {
    static constexpr int kTensors = BITS == 8 ? 70 : 98;
    void* p[kTensors];
    const void* g[kTensors];
    void* m[kTensors];
    void* v[kTensors];
    float* ms[BITS == 8 ? kTensors : 1];
    float* vs[BITS == 8 ? kTensors : 1];
    uint32_t n[kTensors];           // larger tensors are passed in parts
    uint32_t first[kTensors];       // index of the tensor's first chunk
    const float* lr;                // device scalars of a captured step (nullable): the learning rate ...
    const float* step;              // ... and the number of this step
    double log2_beta1, log2_beta2, lr_host, step_host, decay;
    AdamConst c;
    int count;
};
static_assert(sizeof(AdamArgs<32>) <= 4096 && sizeof(AdamArgs<8>) <= 4096, "kernel arguments");

// largest value of the wave, in every lane: within rows of 16 lanes, then row by row into lane 63
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    auto step = [&](auto ctrl) {
        v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, false));
    };
    step(std::integral_constant<int, 0xb1>{});      // lanes 1 0 3 2
    step(std::integral_constant<int, 0x4e>{});      // lanes 2 3 0 1
    step(std::integral_constant<int, 0x141>{});     // mirrored within 8
    step(std::integral_constant<int, 0x140>{});     // mirrored within 16
    step(std::integral_constant<int, 0x142>{});     // lane 15 of a row to the next row
    step(std::integral_constant<int, 0x143>{});     // lane 31 to the upper half
    return (uint32_t)__builtin_amdgcn_readlane((int)v, kWave - 1);
}
__device__ __forceinline__ bool is_finite(float v) { return (__float_as_uint(v) & 0x7fffffffu) < 0x7f800000u; }

// the codes of one block: |values| / s = q^2.  `bits`: the block's largest |value| as bits (a NaN is larger than every number)
__device__ __forceinline__ float code_scale(uint32_t bits, float inv_steps2) {
    const float s = __uint_as_float(bits) * inv_steps2;
    return is_finite(s) ? s : __uint_as_float(0x7fc00000u);
}
// q = rint(sqrt(|x| / s)), quotient and root correctly rounded.  The short form differs from it by less than 2^-21 of the
// root (reciprocal 2^-23, product 2^-24 and quotient 2^-24, halved by the root; the root instruction 2^-23 and the rounded root 2^-24:
// 2^-21.6): it settles every root that is further than that from half an integer, and the wave computes the long form where one of its
// roots is not
struct CodeScale {
    float s, inv;
    bool ok;            // the short form applies
    __device__ __forceinline__ explicit CodeScale(float scale) : s(scale), inv(__builtin_amdgcn_rcpf(scale)), ok(s > 0.f && s < 0x1p100f && inv < 0x1p100f) {}
    __device__ __forceinline__ float exact(float x) const { return s > 0.f ? rintf(sqrtf(fabsf(x) / s)) : 0.f; }
    __device__ __forceinline__ float quick(float x, bool& unsure) const {
        const float y = __builtin_amdgcn_sqrtf(fabsf(x) * inv), q = rintf(y);
        unsure |= !(__builtin_fmaf(y, 0x1p-21f, fabsf(y - q)) < 0.5f);
        return q;
    }
    __device__ __forceinline__ void four(const float* x, float* q) const {
        bool unsure = !ok;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = quick(x[i], unsure);
        if (__ballot(unsure)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = exact(x[i]);
        }
    }
};
// q as whole numbers in fp32: every product of two is exact
__device__ __forceinline__ float decode_m(float q, float s) { return q * fabsf(q) * s; }
__device__ __forceinline__ float decode_v(float q, float s) {
    const float r = q * q * s;
    return r * r;
}

// four consecutive elements; `whole`: a single aligned vector access
template <typename T>
__device__ __forceinline__ void load4(const T* p, int64_t e, int64_t n, bool whole, float* out) {
    if (whole) {
        const vec_t<T, 4> v = *reinterpret_cast<const vec_t<T, 4>*>(p + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = e + i < n ? (float)p[e + i] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t e, int64_t n, bool whole, const float* in) {
    if (whole) {
        vec_t<T, 4> v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (T)in[i];
        *reinterpret_cast<vec_t<T, 4>*>(p + e) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (e + i < n) p[e + i] = (T)in[i];
    }
}

// four codes as bytes: q + bias in 0 .. 255, with the bits of `flip` turned over (127 + 1 and the top bit: two's complement)
template <typename T>
__device__ __forceinline__ void store_codes(T* p, int64_t e, int64_t n, bool whole, const float* q, float bias, uint32_t flip) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w = __builtin_amdgcn_cvt_pk_u8_f32(q[i] + bias, i, w);
    w ^= flip;
    if (whole) {
        *reinterpret_cast<uint32_t*>(p + e) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (e + i < n) p[e + i] = (T)(w >> (8 * i));
    }
}

template <int BITS, typename PT, typename GT>
__global__ __launch_bounds__(kBlock) void adamw_kernel(const AdamArgs<BITS> a) {
    typedef typename std::conditional<BITS == 8, int8_t, float>::type MT;
    typedef typename std::conditional<BITS == 8, uint8_t, float>::type VT;
    const uint32_t chunk = blockIdx.x;
    // the tensor this chunk belongs to: the last one whose first chunk is not behind it
    int t = 0;
    for (int i0 = 0; i0 < a.count; i0 += kWave) {
        const int i = i0 + (threadIdx.x & 63);
        t += __popcll(__ballot(i < a.count && a.first[i] <= chunk));
    }
    t = __builtin_amdgcn_readfirstlane(t - 1);
    PT* p = static_cast<PT*>(a.p[t]);
    const GT* g = static_cast<const GT*>(a.g[t]);
    MT* m = static_cast<MT*>(a.m[t]);
    VT* v = static_cast<VT*>(a.v[t]);
    const int64_t n = a.n[t], base = (int64_t)(chunk - a.first[t]) * kAdamChunk<BITS>;
    const bool aligned = ((reinterpret_cast<uintptr_t>(p) & (4 * sizeof(PT) - 1)) | (reinterpret_cast<uintptr_t>(g) & (4 * sizeof(GT) - 1)) |
                          (reinterpret_cast<uintptr_t>(m) & (4 * sizeof(MT) - 1)) | (reinterpret_cast<uintptr_t>(v) & (4 * sizeof(VT) - 1))) == 0;
    AdamConst c = a.c;
    if (a.step || a.lr) {
        // 1 - b^t in fp64, as on the host
        const double lr = a.lr ? (double)*a.lr : a.lr_host, step = a.step ? (double)*a.step : a.step_host;
        c.keep = (float)(1.0 - lr * a.decay);
        c.size = (float)(lr / (1.0 - exp2(step * a.log2_beta1)));
        c.root = (float)(1.0 / sqrt(1.0 - exp2(step * a.log2_beta2)));
    }
    constexpr int kAdamUnits = kAdamChunk<BITS> / (4 * kBlock);         // 4-element units per lane
    float pv[kAdamUnits][4], gv[kAdamUnits][4], mv[kAdamUnits][4], vv[kAdamUnits][4];
#pragma unroll
    for (int j = 0; j < kAdamUnits; ++j) {
        const int64_t e = base + (int64_t)(j * kBlock + threadIdx.x) * 4;
        const bool whole = aligned && e + 4 <= n;
        load4(p, e, n, whole, pv[j]);
        load4(g, e, n, whole, gv[j]);
        load4(m, e, n, whole, mv[j]);
        load4(v, e, n, whole, vv[j]);
    }
#pragma unroll
    for (int j = 0; j < kAdamUnits; ++j) {
        const int64_t e = base + (int64_t)(j * kBlock + threadIdx.x) * 4;
        const bool whole = aligned && e + 4 <= n;
        const int64_t block = (base + (int64_t)j * (4 * kBlock)) / 256 + (threadIdx.x >> 6);     // the wave's 256 elements
        if (BITS == 8) {
            const bool in = block * 256 < n;
            const float sm = in ? a.ms[t][block] : 0.f, sv = in ? a.vs[t][block] : 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                mv[j][i] = decode_m(mv[j][i], sm);
                vv[j][i] = decode_v(vv[j][i], sv);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float gr = gv[j][i];
            const float mn = mv[j][i] * c.beta1 + gr * c.one_beta1;
            const float vn = vv[j][i] * c.beta2 + (gr * gr) * c.one_beta2;
            const float denom = sqrtf(vn) * c.root + c.eps;
            pv[j][i] = pv[j][i] * c.keep - mn / denom * c.size;
            mv[j][i] = mn;
            vv[j][i] = vn;
        }
        store4(p, e, n, whole, pv[j]);
        if (BITS == 32) {
            store4(m, e, n, whole, mv[j]);
            store4(v, e, n, whole, vv[j]);
        } else {
            // elements past the end decode to 0 and have gradient 0: they do not touch the maxima
            uint32_t am = 0, ar = 0;
            float r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r[i] = sqrtf(vv[j][i]);
                am = max(am, __float_as_uint(mv[j][i]) & 0x7fffffffu);
                ar = max(ar, __float_as_uint(r[i]) & 0x7fffffffu);
            }
            const float sm = code_scale(wave_umax(am), 1.f / 16129.f), sv = code_scale(wave_umax(ar), 1.f / 65025.f);
            float qm[4], qv[4];
            CodeScale(sm).four(mv[j], qm);
            CodeScale(sv).four(r, qv);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                qm[i] = copysignf(fminf(qm[i], 127.f), mv[j][i]);
                qv[i] = r[i] > 0.f && sv > 0.f ? fminf(fmaxf(qv[i], 1.f), 255.f) : 0.f;
            }
            store_codes(m, e, n, whole, qm, 128.f, 0x80808080u);
            store_codes(v, e, n, whole, qv, 0.f, 0u);
            if ((threadIdx.x & 63) == 0 && block * 256 < n) {
                a.ms[t][block] = sm;
                a.vs[t][block] = sv;
            }
        }
    }
}

// the values that a tensor's 8-bit moments stand for
__global__ __launch_bounds__(kBlock) void adamw_moments_kernel(const int8_t* m, const uint8_t* v, const float* ms, const float* vs,
                                                               float* m_out, float* v_out, int64_t n) {
    const bool whole4 = (((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 3) |
                         ((reinterpret_cast<uintptr_t>(m_out) | reinterpret_cast<uintptr_t>(v_out)) & 15)) == 0;
    for (int64_t u = (int64_t)blockIdx.x * kBlock + threadIdx.x; u * 4 < n; u += (int64_t)gridDim.x * kBlock) {
        const int64_t e = u * 4, b = e / 256;
        const bool whole = whole4 && e + 4 <= n;
        float qm[4], qv[4];
        load4(m, e, n, whole, qm);
        load4(v, e, n, whole, qv);
        const float sm = ms[b], sv = vs[b];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            qm[i] = decode_m(qm[i], sm);
            qv[i] = decode_v(qv[i], sv);
        }
        store4(m_out, e, n, whole, qm);
        store4(v_out, e, n, whole, qv);
    }
}

template <int BITS, typename PT, typename GT>
static int adamw_launch(int count, void* const* p, const void* const* g, void* const* m, void* const* v, float* const* ms,
                        float* const* vs, const int64_t* n, AdamArgs<BITS>& a, hipStream_t st) {
    constexpr int64_t kMost = 1ll << 31;            // elements of an entry: whole chunks, blocks of codes and aligned vectors
    static_assert(kMost % kAdamChunk<BITS> == 0 && kMost % 256 == 0, "a part ends where a chunk ends");
    constexpr uint64_t kMostChunks = (1ull << 32) / kBlock - 1;             // a grid has less than 2^32 threads
    int k = 0;
    uint64_t chunks = 0;
    auto flush = [&]() {
        if (k == 0) return (int)CNF_OK;
        a.count = k;
        CNF_LAUNCH((adamw_kernel<BITS, PT, GT>), dim3((unsigned)chunks), dim3(kBlock), 0, st, a);
        k = 0;
        chunks = 0;
        return launch_status("cnf_adamw_step");
    };
    for (int i = 0; i < count; ++i) {
        for (int64_t at = 0; at < n[i]; at += kMost) {
            const int64_t part = std::min<int64_t>(n[i] - at, kMost);
            const uint64_t c = ((uint64_t)part + kAdamChunk<BITS> - 1) / kAdamChunk<BITS>;
            if (k == AdamArgs<BITS>::kTensors || chunks + c > kMostChunks) {
                const int rc = flush();
                if (rc != CNF_OK) return rc;
            }
            a.p[k] = static_cast<PT*>(p[i]) + at;
            a.g[k] = static_cast<const GT*>(g[i]) + at;
            a.m[k] = static_cast<char*>(m[i]) + at * (BITS / 8);
            a.v[k] = static_cast<char*>(v[i]) + at * (BITS / 8);
            if (BITS == 8) {
                a.ms[k] = ms[i] + at / 256;
                a.vs[k] = vs[i] + at / 256;
            }
            a.n[k] = (uint32_t)part;
            a.first[k] = (uint32_t)chunks;
            chunks += c;
            ++k;
        }
    }
    return flush();
}

template <int BITS>
static int adamw_typed(int count, void* const* p, const void* const* g, void* const* m, void* const* v, float* const* ms,
                       float* const* vs, const int64_t* n, int pdtype, int gdtype, AdamArgs<BITS>& a, hipStream_t st) {
    return with_dtype(pdtype, [&](auto pt) {
        typedef decltype(pt) PT;
        if (gdtype == pdtype) return adamw_launch<BITS, PT, PT>(count, p, g, m, v, ms, vs, n, a, st);
        return adamw_launch<BITS, PT, float>(count, p, g, m, v, ms, vs, n, a, st);
    });
}

template <int BITS>
static int adamw_run(int count, void* const* p, const void* const* g, void* const* m, void* const* v, float* const* ms, float* const* vs,
                     const int64_t* n, int pdtype, int gdtype, double lr, double beta1, double beta2, double eps, double decay, double step,
                     const float* lr_dev, const float* step_dev, hipStream_t st) {
    AdamArgs<BITS> a;
    memset(&a, 0, sizeof(a));
    a.lr = lr_dev;
    a.step = step_dev;
    a.log2_beta1 = beta1 > 0.0 ? std::log2(beta1) : -1e30;      // beta = 0: beta^t = 0
    a.log2_beta2 = beta2 > 0.0 ? std::log2(beta2) : -1e30;
    a.lr_host = lr;
    a.step_host = step;
    a.decay = decay;
    a.c.beta1 = (float)beta1;
    a.c.one_beta1 = (float)(1.0 - beta1);
    a.c.beta2 = (float)beta2;
    a.c.one_beta2 = (float)(1.0 - beta2);
    a.c.eps = (float)eps;
    a.c.keep = (float)(1.0 - lr * decay);
    if (!step_dev) {
        a.c.size = (float)(lr / (1.0 - std::pow(beta1, step)));
        a.c.root = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, step)));
    }
    return adamw_typed<BITS>(count, p, g, m, v, ms, vs, n, pdtype, gdtype, a, st);
}

}  // namespace cnf

using namespace cnf;

extern "C" {

int cnf_adamw_step(int count, void* const* params, const void* const* grads, void* const* exp_avg, void* const* exp_avg_sq,
                   float* const* exp_avg_scale, float* const* exp_avg_sq_scale, const int64_t* numel, int pdtype, int gdtype,
                   int state_bits, double lr, double beta1, double beta2, double eps, double weight_decay, double step,
                   const float* lr_dev, const float* step_dev, cnf_stream_t stream) {
    CNF_REQUIRE(count >= 0, "cnf_adamw_step: negative tensor count");
    if (count == 0) return CNF_OK;
    CNF_REQUIRE(params && grads && exp_avg && exp_avg_sq && numel, "cnf_adamw_step: null list");
    CNF_REQUIRE(state_bits == 32 || state_bits == 8, "cnf_adamw_step: moments in 32 or 8 bits, got %d", state_bits);
    CNF_REQUIRE(state_bits == 32 || (exp_avg_scale && exp_avg_sq_scale), "cnf_adamw_step: 8-bit moments need their scales");
    CNF_REQUIRE(dtype_known(pdtype) && (gdtype == pdtype || gdtype == CNF_DTYPE_F32), "cnf_adamw_step: gradients are fp32 or of the parameters' type");
    CNF_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "cnf_adamw_step: betas outside [0, 1)");
    CNF_REQUIRE(step_dev || step >= 1.0, "cnf_adamw_step: the first step is step 1");
    for (int i = 0; i < count; ++i) {
        CNF_REQUIRE(numel[i] >= 0 && numel[i] < ((int64_t)1 << 42), "cnf_adamw_step: tensor %d has %ld elements", i, (long)numel[i]);
        CNF_REQUIRE(numel[i] == 0 || (params[i] && grads[i] && exp_avg[i] && exp_avg_sq[i] &&
                                      (state_bits == 32 || (exp_avg_scale[i] && exp_avg_sq_scale[i]))),
                    "cnf_adamw_step: null tensor %d", i);
    }
    hipStream_t st = (hipStream_t)stream;
    if (state_bits == 8)
        return adamw_run<8>(count, params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, numel, pdtype, gdtype, lr, beta1, beta2,
                            eps, weight_decay, step, lr_dev, step_dev, st);
    return adamw_run<32>(count, params, grads, exp_avg, exp_avg_sq, nullptr, nullptr, numel, pdtype, gdtype, lr, beta1, beta2, eps,
                         weight_decay, step, lr_dev, step_dev, st);
}

int cnf_adamw_moments(const int8_t* exp_avg, const uint8_t* exp_avg_sq, const float* exp_avg_scale, const float* exp_avg_sq_scale,
                      float* m_out, float* v_out, int64_t n, cnf_stream_t stream) {
    CNF_REQUIRE(n >= 0, "cnf_adamw_moments: negative size");
    if (n == 0) return CNF_OK;
    CNF_REQUIRE(exp_avg && exp_avg_sq && exp_avg_scale && exp_avg_sq_scale && m_out && v_out, "cnf_adamw_moments: null tensor");
    const unsigned grid = (unsigned)std::min<int64_t>((n + 4 * kBlock - 1) / (4 * kBlock), 8192);
    CNF_LAUNCH(adamw_moments_kernel, dim3(grid), dim3(kBlock), 0, (hipStream_t)stream, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale,
               m_out, v_out, n);
    return launch_status("cnf_adamw_moments");
}

}  // extern "C"
