// Element types, matrix fragments and LDS tiles shared by the sequence operators (k_norm_rope, k_attn*, k_attn_step).
//
// Elements are fp32, bf16 or fp16; products accumulate in fp32, softmax statistics and norms are fp32.  A fragment holds the
// eight consecutive k values of one row that a lane of v_mfma_f32_32x32x16 / _16x16x32 supplies.  fp32 elements use the same
// fragments: eight v_mfma_f32_32x32x2_f32 (16x16x4), instruction e contracting element e of every lane -- the k values meet
// in another order than in the 16-bit forms, and every kernel written for the fragments serves the three types.
#pragma once
#include "dof_rt.h"

struct DofBf16 { uint16_t u; };
struct DofF16 { uint16_t u; };

// a run of 32-bit words as one load / store of that width (the address must be aligned to it)
template <int N> struct alignas(4 * N) DofWords { uint32_t w[N]; };

template <class T> struct DofElem;
template <> struct DofElem<float> {
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
  template <int N> static __device__ __forceinline__ void unpack(const DofWords<N>& w, float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __builtin_bit_cast(float, w.w[i]);
  }
  template <int N> static __device__ __forceinline__ void pack(const float* v, DofWords<N>& w) {
#pragma unroll
    for (int i = 0; i < N; ++i) w.w[i] = __builtin_bit_cast(uint32_t, v[i]);
  }
};
template <> struct DofElem<DofBf16> {
  static __device__ __forceinline__ float get(const DofBf16* p) { return dof_bf16_to_f32(p->u); }
  static __device__ __forceinline__ void put(DofBf16* p, float v) { p->u = (uint16_t)dof_pack_bf16(v, 0.0f); }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) { return dof_pack_bf16(a, b); }
  template <int N> static __device__ __forceinline__ void unpack(const DofWords<N>& w, float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[2 * i] = dof_bf16_to_f32(w.w[i] & 0xFFFFu);
      v[2 * i + 1] = __builtin_bit_cast(float, w.w[i] & 0xFFFF0000u);
    }
  }
  template <int N> static __device__ __forceinline__ void pack(const float* v, DofWords<N>& w) {
#pragma unroll
    for (int i = 0; i < N; ++i) w.w[i] = dof_pack_bf16(v[2 * i], v[2 * i + 1]);
  }
};
template <> struct DofElem<DofF16> {
  static __device__ __forceinline__ float get(const DofF16* p) { return dof_f16_to_f32(p->u); }
  static __device__ __forceinline__ void put(DofF16* p, float v) { p->u = (uint16_t)dof_pack_f16(v, 0.0f); }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) { return dof_pack_f16(a, b); }
  template <int N> static __device__ __forceinline__ void unpack(const DofWords<N>& w, float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[2 * i] = dof_f16_to_f32(w.w[i] & 0xFFFFu);
      v[2 * i + 1] = dof_f16_to_f32(w.w[i] >> 16);
    }
  }
  template <int N> static __device__ __forceinline__ void pack(const float* v, DofWords<N>& w) {
#pragma unroll
    for (int i = 0; i < N; ++i) w.w[i] = dof_pack_f16(v[2 * i], v[2 * i + 1]);
  }
};

// VEC elements of T at p (aligned to VEC elements, at most 16 bytes) <-> fp32 registers
template <class T, int VEC> __device__ __forceinline__ void dof_load_vec(const T* p, float* v) {
  if constexpr (VEC * sizeof(T) >= 4) {
    const DofWords<(int)(VEC * sizeof(T) / 4)> w = *reinterpret_cast<const DofWords<(int)(VEC * sizeof(T) / 4)>*>(p);
    DofElem<T>::unpack(w, v);
  } else {
    static_assert(VEC == 1, "one element");
    v[0] = DofElem<T>::get(p);
  }
}
template <class T, int VEC> __device__ __forceinline__ void dof_store_vec(T* p, const float* v) {
  if constexpr (VEC * sizeof(T) >= 4) {
    DofWords<(int)(VEC * sizeof(T) / 4)> w;
    DofElem<T>::pack(v, w);
    *reinterpret_cast<DofWords<(int)(VEC * sizeof(T) / 4)>*>(p) = w;
  } else {
    static_assert(VEC == 1, "one element");
    DofElem<T>::put(p, v[0]);
  }
}

// DOF_SEQ_DISPATCH(dtype, T, expr): expr with T = the element type of a DOF_DTYPE_* code
#define DOF_SEQ_DISPATCH(dtype, T, ...)                                          \
  do {                                                                           \
    if ((dtype) == DOF_DTYPE_F32) { using T = float; __VA_ARGS__; }              \
    else if ((dtype) == DOF_DTYPE_BF16) { using T = DofBf16; __VA_ARGS__; }      \
    else { using T = DofF16; __VA_ARGS__; }                                      \
  } while (0)
