// Element types of the operators that take fp32, bf16 and fp16 tensors: loads and stores through 16-byte vectors, arithmetic in fp32.
#pragma once
#include "cnf_common.h"

namespace cnf {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T, int N>
using vec_t = T __attribute__((ext_vector_type(N)));

__host__ __device__ constexpr int dtype_bytes(int dtype) { return dtype == CNF_DTYPE_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype == CNF_DTYPE_F32 || dtype == CNF_DTYPE_BF16 || dtype == CNF_DTYPE_F16; }

// one element of a tensor whose type is known at run time (weights: read once per launch)
__device__ __forceinline__ float load_any(const void* p, int dtype, long i) {
    if (dtype == CNF_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == CNF_DTYPE_BF16) return (float)static_cast<const bf16_t*>(p)[i];
    return (float)static_cast<const f16_t*>(p)[i];
}
__device__ __forceinline__ void store_any(void* p, int dtype, long i, float v) {
    if (dtype == CNF_DTYPE_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == CNF_DTYPE_BF16) static_cast<bf16_t*>(p)[i] = (bf16_t)v;
    else static_cast<f16_t*>(p)[i] = (f16_t)v;
}

// four consecutive elements i ... i + 3, those below `end`; four go in one access, whatever their address
template <typename V4>
__device__ __forceinline__ void store4_any(void* p, int dtype, long i, long end, V4 v) {
    if (i + 4 > end) {
        for (int k = 0; k < 4; ++k)
            if (i + k < end) store_any(p, dtype, i + k, v[k]);
    } else if (dtype == CNF_DTYPE_F32) {
        __builtin_memcpy(static_cast<float*>(p) + i, &v, 16);
    } else if (dtype == CNF_DTYPE_BF16) {
        const vec_t<bf16_t, 4> o = {(bf16_t)v[0], (bf16_t)v[1], (bf16_t)v[2], (bf16_t)v[3]};
        __builtin_memcpy(static_cast<bf16_t*>(p) + i, &o, 8);
    } else {
        const vec_t<f16_t, 4> o = {(f16_t)v[0], (f16_t)v[1], (f16_t)v[2], (f16_t)v[3]};
        __builtin_memcpy(static_cast<f16_t*>(p) + i, &o, 8);
    }
}

// calls fn(T{}) with the element type of `dtype`
template <typename Fn>
inline int with_dtype(int dtype, Fn&& fn) {
    if (dtype == CNF_DTYPE_F32) return fn(float{});
    if (dtype == CNF_DTYPE_BF16) return fn(bf16_t{});
    return fn(f16_t{});
}

// the host's side of "every 16-byte load of these rows is aligned"
inline bool rows_aligned16(const void* p, int64_t stride_elems, int dtype) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride_elems * dtype_bytes(dtype)) % 16 == 0;
}

}  // namespace cnf
