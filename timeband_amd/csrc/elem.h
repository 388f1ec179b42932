// Element types of the state space layer's operators (convolution, selective scan, linear with residual): fp32, bf16 and fp16
// in memory, fp32 in registers.  A store rounds once, to nearest even.
#pragma once
#include "common.h"

#define TB_F32 0
#define TB_BF16 1
#define TB_F16 2

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

static inline size_t tb_dtype_size(int dt) { return dt == TB_F32 ? 4 : 2; }
// steps a call: sums of a step and a run or chunk of them stay within 32 bits
#define TB_STEPS_MAX 2147418112L
// a launch has fewer than 2^32 threads
static inline bool tb_grid_ok(long blocks, int threads) { return blocks * threads < 1L << 32; }
static inline bool tb_dtype_ok(int dt) { return dt >= TB_F32 && dt <= TB_F16; }

// N consecutive elements as one access where the address allows it (the caller knows), element by element otherwise
template <typename T, int N>
struct alignas(sizeof(T) * N) TbVec {
  T v[N];
};

// elements an access: at most 16 bytes, and N is made of whole accesses
template <typename T, int N>
constexpr int tb_width() {
  int w = 16 / sizeof(T);
  while (N % w) w /= 2;
  return w;
}

template <typename T, int N>
__device__ __forceinline__ void tb_load_n(const T* p, float (&r)[N]) {
  constexpr int W = tb_width<T, N>();
#pragma unroll
  for (int i = 0; i < N; i += W) {
    const TbVec<T, W> t = *reinterpret_cast<const TbVec<T, W>*>(p + i);
#pragma unroll
    for (int j = 0; j < W; ++j) r[i + j] = (float)t.v[j];
  }
}
template <typename T, int N>
__device__ __forceinline__ void tb_store_n(T* p, const float (&r)[N]) {
  constexpr int W = tb_width<T, N>();
#pragma unroll
  for (int i = 0; i < N; i += W) {
    TbVec<T, W> t;
#pragma unroll
    for (int j = 0; j < W; ++j) t.v[j] = (T)r[i + j];
    *reinterpret_cast<TbVec<T, W>*>(p + i) = t;
  }
}

// The same for addresses that are only aligned to an element: still one access of 16 bytes (the memory path takes any address).
template <typename T, int W>
struct __attribute__((packed, aligned(sizeof(T)))) TbVecU {
  T v[W];
};
template <typename T, int N>
__device__ __forceinline__ void tb_load_u(const T* p, float (&r)[N]) {
  constexpr int W = tb_width<T, N>();
#pragma unroll
  for (int i = 0; i < N; i += W) {
    const TbVecU<T, W> t = *reinterpret_cast<const TbVecU<T, W>*>(p + i);
#pragma unroll
    for (int j = 0; j < W; ++j) r[i + j] = (float)t.v[j];
  }
}
template <typename T, int N>
__device__ __forceinline__ void tb_store_u(T* p, const float (&r)[N]) {
  constexpr int W = tb_width<T, N>();
#pragma unroll
  for (int i = 0; i < N; i += W) {
    TbVecU<T, W> t;
#pragma unroll
    for (int j = 0; j < W; ++j) t.v[j] = (T)r[i + j];
    *reinterpret_cast<TbVecU<T, W>*>(p + i) = t;
  }
}

// A parameter that is kept either in the operator's element type or in fp32 (f32 != 0): read / written once per thread
template <typename T>
__device__ __forceinline__ float tb_load_par(const void* p, long i, int f32) {
  return f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i];
}
template <typename T>
__device__ __forceinline__ void tb_store_par(void* p, long i, float v, int f32) {
  if (f32) static_cast<float*>(p)[i] = v;
  else static_cast<T*>(p)[i] = (T)v;
}

// activations: 0 none, 1 tanh, 2 sigmoid, 3 relu, 4 silu, 5 gelu (the error-function form)
#define TB_ACT_SILU 4
#define TB_ACT_LAST 5

// e^x on the hardware's 2^x alone: results below 2^-126 are 0
__device__ __forceinline__ float tb_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
// 1 / (1 + e^-x) on the hardware exp and reciprocal (1 ulp each): e^-x = inf gives 0, e^-x = 0 gives 1
__device__ __forceinline__ float tb_sig(float x) { return __builtin_amdgcn_rcpf(1.f + tb_exp(-x)); }
__device__ __forceinline__ float tb_silu(float x) { return x * tb_sig(x); }
