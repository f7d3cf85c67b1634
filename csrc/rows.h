// Rows of fp32 / bf16 / fp16 elements at any element offset (csrc/ln.hip,
// csrc/vocab.hip): 16-byte accesses that need no more alignment than their
// elements, and their conversion to fp32.
//
// A row of an odd length starts at every alignment in turn.  Global memory on
// gfx950 takes a 16-byte access at any address (the vector type below says so
// to the compiler, which emits one dwordx4 access); a wave's contiguous
// kilobyte then touches one cache line more than an aligned one.
#pragma once
#include "common.h"

typedef unsigned u32x4n __attribute__((ext_vector_type(4)));
typedef u32x4n u32x4u __attribute__((aligned(2)));

// elements of one 16-byte access
template <int DT> constexpr int row_vec() { return DT == KDT_F32 ? 4 : 8; }

template <int DT> __device__ __forceinline__ void vec_to_f32(const u32x4n v, float* f) {
  if constexpr (DT == KDT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
  } else if constexpr (DT == KDT_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = f16_bits_to_f32((uint16_t)(v[i] & 0xffffu));
      f[2 * i + 1] = f16_bits_to_f32((uint16_t)(v[i] >> 16));
    }
  }
}

template <int DT> __device__ __forceinline__ u32x4n f32_to_vec(const float* f) {
  u32x4n v;
  if constexpr (DT == KDT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = (uint32_t)DTypeTraits<DT>::from_f32(f[2 * i]) |
             ((uint32_t)DTypeTraits<DT>::from_f32(f[2 * i + 1]) << 16);
  }
  return v;
}

// Vector v moved down by s elements (0 <= s < V), zeros moved in.
template <int DT> __device__ __forceinline__ u32x4n vec_shift(u32x4n v, int s) {
  const int words = DT == KDT_F32 ? s : s >> 1;
  if (words & 2) v = (u32x4n){v[2], v[3], 0u, 0u};
  if (words & 1) v = (u32x4n){v[1], v[2], v[3], 0u};
  if (DT != KDT_F32 && (s & 1)) {
    v = (u32x4n){__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16),
                 __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
  }
  return v;
}

// Access at element i of a row of n elements, n >= V = row_vec<DT>(): what lies
// behind the row's end reads as 0.  Branch-free, so that a thread's loads are
// issued back to back: an access past the end is moved into the row -- one that
// holds the end (TAIL: n need not be a multiple of V) to the row's last V
// elements, to be shifted down.
// STREAM: the row is not read again soon (non-temporal).
template <int DT, bool TAIL, bool STREAM = false>
__device__ __forceinline__ u32x4n load_vec(const AS1 typename DTypeTraits<DT>::raw_t* row, int i,
                                           int n) {
  constexpr int V = row_vec<DT>();
  const int at = i + V <= n ? i : TAIL && i < n ? n - V : 0;
  const AS1 u32x4u* p = (const AS1 u32x4u*)(row + at);
  return STREAM ? __builtin_nontemporal_load(p) : *p;
}
template <int DT, bool TAIL>
__device__ __forceinline__ u32x4n clip_vec(u32x4n v, int i, int n) {
  constexpr int V = row_vec<DT>();
  if (TAIL) {
    const int over = i + V - n;
    v = vec_shift<DT>(v, over > 0 && over < V ? over : 0);
  }
  return i < n ? v : (u32x4n)0u;
}
template <int DT, bool TAIL>
__device__ __forceinline__ void store_vec(AS1 typename DTypeTraits<DT>::raw_t* row, int i, int n,
                                          const float* f) {
  constexpr int V = row_vec<DT>();
  if (i + V <= n) {
    *(AS1 u32x4u*)(row + i) = f32_to_vec<DT>(f);
  } else if (TAIL && i < n) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (i + e < n) row[i + e] = DTypeTraits<DT>::from_f32(f[e]);
  }
}
