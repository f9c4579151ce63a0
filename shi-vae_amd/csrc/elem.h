// Element types of the sequence operators (conv.hip, ssm.hip, sample.hip): fp32, bf16, fp16 in memory, fp32 in registers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace shivae {

template <class E, int V>
struct alignas(sizeof(E) * V) Pack {
    E v[V];
};

template <class E>
__device__ __forceinline__ float elem_f(E e) { return (float)e; }
// One rounding to nearest even per stored element (v_cvt_pk_bf16_f32, v_cvt_f16_f32).
template <class E>
__device__ __forceinline__ E f_elem(float f) { return (E)f; }

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

// sigmoid(v) and softplus(v) = max(v,0) + log1p(exp(-|v|)) from one v_exp_f32.  log1p(e) = log(w) + (e - (w-1)), w = fl(1+e):
// the second term is what the rounding of w dropped, so small e keep their relative accuracy.
__device__ __forceinline__ float seq_sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-v * kLog2e)); }
__device__ __forceinline__ float seq_softplus(float v) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(v) * kLog2e), w = 1.f + e;
    return fmaxf(v, 0.f) + (__builtin_amdgcn_logf(w) * kLn2 + (e - (w - 1.f)));
}

// Runs a statement with E = the element type of `dtype` (checked by the caller).
#define SV_BY_DTYPE(dtype, ...)                    \
    do {                                           \
        if ((dtype) == SHIVAE_F32) {               \
            using E = float;                       \
            __VA_ARGS__;                           \
        } else if ((dtype) == SHIVAE_BF16) {       \
            using E = __bf16;                      \
            __VA_ARGS__;                           \
        } else {                                   \
            using E = _Float16;                    \
            __VA_ARGS__;                           \
        }                                          \
    } while (0)

// A launch has fewer than 2^32 threads along an axis (hipModuleLaunchKernel).
static inline bool grid_fits(int64_t blocks, int threads) { return blocks < ((int64_t)1 << 32) / threads; }
static inline int elem_bytes(int dtype) { return dtype == SHIVAE_F32 ? 4 : 2; }
static inline bool aligned_to(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

}  // namespace shivae
