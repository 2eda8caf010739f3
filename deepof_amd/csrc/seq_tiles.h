// Matrix fragments and LDS tiles of the attention kernels (see seq_types.h for the element types).
#pragma once
#include "seq_types.h"

// Eight k values of one row, as a lane supplies them to a 32x32x16 or 16x16x32 product.
template <class T> struct DofFrag { uint32_t w[4]; };
template <> struct DofFrag<float> { float v[8]; };

template <class T> __device__ __forceinline__ DofFrag<T> dof_frag_zero() {
  DofFrag<T> f;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = 0.0f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f.w[i] = 0u;
  }
  return f;
}
// eight elements at a 16-byte aligned address
template <class T> __device__ __forceinline__ DofFrag<T> dof_frag_load(const T* p) {
  DofFrag<T> f;
  if constexpr (sizeof(T) == 4) {
    const DofWords<4> a = *reinterpret_cast<const DofWords<4>*>(p), b = *reinterpret_cast<const DofWords<4>*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f.v[i] = __builtin_bit_cast(float, a.w[i]);
      f.v[4 + i] = __builtin_bit_cast(float, b.w[i]);
    }
  } else {
    const DofWords<4> a = *reinterpret_cast<const DofWords<4>*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.w[i] = a.w[i];
  }
  return f;
}
// eight fp32 values as a fragment; 16-bit types: rounded to nearest even
template <class T> __device__ __forceinline__ DofFrag<T> dof_frag_pack(const float* v) {
  DofFrag<T> f;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f.w[i] = DofElem<T>::pack2(v[2 * i], v[2 * i + 1]);
  }
  return f;
}
template <class T> __device__ __forceinline__ void dof_frag_unpack(const DofFrag<T>& f, float* v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f.v[i];
  } else {
    DofWords<4> w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w.w[i] = f.w[i];
    DofElem<T>::unpack(w, v);
  }
}

// what rounding to `f` left of the eight values, as a second fragment: the two carry them to 16 (bf16) or 22 (fp16) bits
template <class T> __device__ __forceinline__ DofFrag<T> dof_frag_rest(const float* v, const DofFrag<T>& f) {
  float r[8];
  dof_frag_unpack<T>(f, r);
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i] - r[i];
  return dof_frag_pack<T>(r);
}

// Sixteen bytes of elements with zeros in the place of infinities and NaN; were there any?
template <class T> __device__ __forceinline__ bool dof_make_finite(DofWords<4>& v) {
  bool any = false;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      const bool bad = (v.w[k] & 0x7F800000u) == 0x7F800000u;
      any |= bad;
      if (bad) v.w[k] = 0u;
    } else {
      constexpr uint32_t m = std::is_same<T, DofBf16>::value ? 0x7F80u : 0x7C00u;
      const bool lo = (v.w[k] & m) == m, hi = (v.w[k] & (m << 16)) == (m << 16);
      any |= lo || hi;
      v.w[k] &= (lo ? 0xFFFF0000u : 0xFFFFFFFFu) & (hi ? 0x0000FFFFu : 0xFFFFFFFFu);
    }
  }
  return any;
}

// c (32 x 32) += a (32 x 16) b (16 x 32); register v of lane l: row 8 (v / 4) + 4 (l >> 5) + v % 4, column l & 31
template <class T> __device__ __forceinline__ dof_f32x16 dof_mma32(const DofFrag<T>& a, const DofFrag<T>& b, dof_f32x16 c) {
  if constexpr (std::is_same<T, DofBf16>::value) {
    return DOF_MFMA_32x32x16_BF16(__builtin_bit_cast(dof_bf16x8, a), __builtin_bit_cast(dof_bf16x8, b), c);
  } else if constexpr (std::is_same<T, DofF16>::value) {
    return DOF_MFMA_32x32x16_F16(__builtin_bit_cast(dof_f16x8, a), __builtin_bit_cast(dof_f16x8, b), c);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = DOF_MFMA_32x32x2_F32(a.v[e], b.v[e], c);
    return c;
  }
}
// c (16 x 16) += a (16 x 32) b (32 x 16); register r of lane l: row 4 (l >> 4) + r, column l & 15
template <class T> __device__ __forceinline__ dof_f32x4 dof_mma16(const DofFrag<T>& a, const DofFrag<T>& b, dof_f32x4 c) {
  if constexpr (std::is_same<T, DofBf16>::value) {
    return DOF_MFMA_16x16x32_BF16(__builtin_bit_cast(dof_bf16x8, a), __builtin_bit_cast(dof_bf16x8, b), c);
  } else if constexpr (std::is_same<T, DofF16>::value) {
    return DOF_MFMA_16x16x32_F16(__builtin_bit_cast(dof_f16x8, a), __builtin_bit_cast(dof_f16x8, b), c);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
  }
}
__device__ __forceinline__ dof_f32x16 dof_zero16() {
  dof_f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}
__device__ __forceinline__ dof_f32x4 dof_zero4() {
  dof_f32x4 z;
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = 0.0f;
  return z;
}

// sum += x with what the addition rounded off collected in `rest` (Knuth's two-sum); an infinite sum stays one
__device__ __forceinline__ void dof_add_rest(float& sum, float& rest, float x) {
  const float s = sum + x, b = s - sum, lost = (sum - (s - b)) + (x - b);
  sum = s;
  rest += fabsf(s) < INFINITY ? lost : 0.0f;
}

// Accumulators of N registers of V for long sums.  A chain of products rounds once per instruction, and where the terms have one sign
// those errors add up: fp32 elements, 65536 equal weights and values, 6e-4 of the result.  There the chain is cut every kTerms
// terms (kTerms / 2 additions of a 32x32x2 product) and added to a sum of such blocks: n terms are off by at most
// (kTerms / 2 + n / kTerms) 2^-24 of the sum of their sizes.  (Keeping the blocks' own rounding errors besides would make that
// independent of n, but its registers cost the kernels for heads of 16 to 64 a wavefront per SIMD.)  16-bit elements have 16 or 32 terms per
// addition and results of 8 or 11 bits: n / 16 additions stay below half a step of bf16 to n = 2^19 terms of one sign, of fp16 to 2^17;
// nothing is kept for them.  ON false: the sum is known to be short (flat tiles of fp32 heads of 128 would keep it in scratch memory:
// 1000 documents of 40 to 60 frames, 8 heads, training, 3.0 ms without, 3.9 with it).
constexpr int kLongTerms = 256;
template <class T, class V, int N, bool ON> struct DofLongSum {
  static constexpr bool kOn = sizeof(T) == 4 && ON;
  static constexpr int kTerms = kLongTerms, kLanes = (int)(sizeof(V) / 4);
  V sum[kOn ? N : 1];
  int n;
  __device__ __forceinline__ void clear() {
    if constexpr (kOn) {
      n = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < kLanes; ++v) sum[i][v] = 0.0f;
    }
  }
  __device__ __forceinline__ void scale(float a) {
    if constexpr (kOn) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < kLanes; ++v) sum[i][v] *= a;
    }
  }
  // `terms` more are in the chain
  __device__ __forceinline__ void count(V* chain, int terms) {
    if constexpr (kOn) {
      n += terms;
      if (n < kTerms) return;
      n = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < kLanes; ++v) {
          sum[i][v] += chain[i][v];
          chain[i][v] = 0.0f;
        }
    }
  }
  // the whole sum, into the chain's registers
  __device__ __forceinline__ void finish(V* chain) {
    if constexpr (kOn) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < kLanes; ++v) chain[i][v] += sum[i][v];
    }
  }
};
// one number that grows once per step; fp32 elements: with its own rounding errors
template <class T> struct DofLongNumber {
  float sum = 0.0f, rest = 0.0f;
  __device__ __forceinline__ void add(float x) {
    if constexpr (sizeof(T) == 4) dof_add_rest(sum, rest, x);
    else sum += x;
  }
  __device__ __forceinline__ void scale(float a) {
    sum *= a;
    if constexpr (sizeof(T) == 4) rest *= a;
  }
  __device__ __forceinline__ float total() const { return sizeof(T) == 4 ? sum + rest : sum; }
};

// An LDS image of ROWS rows x DP elements, read both ways: eight consecutive elements of a row (rowfrag, the operand whose k runs
// along the row) and eight rows of one column (colfrag, the operand whose k runs down the rows).
//
// 16-bit elements: unpadded rows of CH = DP / 8 chunks of 16 bytes, the chunk index XORed with a function of the row, so that both
// readings are free of bank conflicts: sixteen consecutive rows of one chunk (ds_read_b128) and the four rows x four chunks of a
// transposing read (ds_read_b64_tr_b16) each fall into sixteen different 16-byte slots of the 256-byte bank line.
// fp32: rows padded by 16 bytes, columns read as single words.
template <class T, int ROWS, int DP> struct DofTile {
  static constexpr int EPC = 16 / (int)sizeof(T);  // elements per chunk
  static constexpr int CH = DP / EPC;              // chunks per row
  static constexpr int kStride = sizeof(T) == 4 ? DP + 4 : DP;  // elements per row in LDS
  alignas(16) unsigned char mem[ROWS * kStride * (int)sizeof(T)];

  __device__ __forceinline__ static int offset(int row, int chunk) {  // bytes
    if constexpr (sizeof(T) == 4) return (row * kStride + chunk * EPC) * 4;
    int x = (row >> 2) & 3;
    if constexpr (CH % 16 == 0) x |= (row & 3) << 2;
    else if constexpr (CH % 8 == 0) x |= ((row >> 1) & 1) << 2;
    return (row * CH + (chunk ^ x)) * 16;
  }
  __device__ __forceinline__ void put(int row, int chunk, const DofWords<4>& v) {
    *reinterpret_cast<DofWords<4>*>(mem + offset(row, chunk)) = v;
  }
  // elements 8 k8 .. 8 k8 + 7 of a row
  __device__ __forceinline__ DofFrag<T> rowfrag(int row, int k8) const {
    DofFrag<T> f;
    if constexpr (sizeof(T) == 4) {
      return dof_frag_load<T>(reinterpret_cast<const T*>(mem + offset(row, 2 * k8)));
    } else {
      const DofWords<4> v = *reinterpret_cast<const DofWords<4>*>(mem + offset(row, k8));
#pragma unroll
      for (int i = 0; i < 4; ++i) f.w[i] = v.w[i];
      return f;
    }
  }
  // column `col` (16-bit: all 16 lanes of an aligned group read the 16 columns of one aligned block) of the rows ra .. ra + 3 and
  // rb .. rb + 3 (multiples of 4, the same over the group)
  __device__ __forceinline__ DofFrag<T> colfrag(int ra, int rb, int col) const {
    DofFrag<T> f;
    if constexpr (sizeof(T) == 4) {
      const float* m = reinterpret_cast<const float*>(mem);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f.v[i] = m[(ra + i) * kStride + col];
        f.v[4 + i] = m[(rb + i) * kStride + col];
      }
    } else {
      const int q = (int)(threadIdx.x & 15), r = q >> 2, c = (col >> 4) * 2 + ((q & 3) >> 1), b = (q & 1) * 8;
      dof_lds_tr16(reinterpret_cast<const uint16_t*>(mem + offset(ra + r, c) + b), f.w[0], f.w[1]);
      dof_lds_tr16(reinterpret_cast<const uint16_t*>(mem + offset(rb + r, c) + b), f.w[2], f.w[3]);
    }
    return f;
  }
};

// Rows of a tensor on their way into a tile: load() issues the global loads into registers, store() puts them into LDS, so the
// loads of the next tile run under the products of the present one.  Rows from `rows` and elements from `dim` on are zeros.
template <class T, int ROWS, int DP, int NT> struct DofStage {
  using Tile = DofTile<T, ROWS, DP>;
  static constexpr int N = (ROWS * Tile::CH + NT - 1) / NT;
  DofWords<4> reg[N];
  __device__ __forceinline__ void load(const T* base, int64_t stride, int rows, int dim, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + i * NT, r = e / Tile::CH, c = e - r * Tile::CH;
#pragma unroll
      for (int k = 0; k < 4; ++k) reg[i].w[k] = 0u;
      if (r < rows && c * Tile::EPC < dim) reg[i] = *reinterpret_cast<const DofWords<4>*>(base + r * stride + c * Tile::EPC);
    }
  }
  __device__ __forceinline__ void store(Tile& t, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + i * NT, r = e / Tile::CH, c = e - r * Tile::CH;
      if ((ROWS * Tile::CH) % NT == 0 || r < ROWS) t.put(r, c, reg[i]);
    }
  }
  // store() with zeros in the place of infinities and NaN; *found is set if there were any
  __device__ __forceinline__ void store_finite(Tile& t, int tid, int* found) const {
    bool any = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + i * NT, r = e / Tile::CH, c = e - r * Tile::CH;
      DofWords<4> v = reg[i];
      any |= dof_make_finite<T>(v);
      if ((ROWS * Tile::CH) % NT == 0 || r < ROWS) t.put(r, c, v);
    }
    if (any) *found = 1;
  }
};
