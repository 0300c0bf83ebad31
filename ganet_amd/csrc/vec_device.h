// Device-side loads, stores and reductions shared by the training operators
// (csrc/layer_norm.hip, csrc/optim.hip).  Internal, not part of the public ABI.
#pragma once

#include "dcn_device.h"

namespace ganet_vec {

using ganet_dcn::bf16_t;
using ganet_dcn::f16_t;

// What a value of T is to the vector types (bf16 travels as its 16 bits).
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  typedef float type;
  __device__ static __forceinline__ float widen(float e) { return e; }
  __device__ static __forceinline__ float narrow(float f) { return f; }
};
template <>
struct Elem<f16_t> {
  typedef _Float16 type;
  __device__ static __forceinline__ float widen(_Float16 e) { return (float)e; }
  __device__ static __forceinline__ _Float16 narrow(float f) { return (_Float16)f; }
};
template <>
struct Elem<bf16_t> {
  typedef unsigned short type;
  __device__ static __forceinline__ float widen(unsigned short e) {
    return __uint_as_float((unsigned)e << 16);
  }
  __device__ static __forceinline__ unsigned short narrow(float f) {
    return ganet_dcn::from_f32<bf16_t>(f).v;
  }
};

// N consecutive values, held as they lie in memory (16-bit values keep half the registers while
// they wait) and widened where they are used.  The memory type is aligned like ONE value: a row
// or a tensor may start anywhere (odd channel counts, views into a flat buffer), and global
// memory takes 4- to 16-byte accesses at any address on gfx950, so one path serves every
// alignment.
template <typename T, int N>
struct Vec {
  typedef typename Elem<T>::type E;
  typedef E Reg __attribute__((ext_vector_type(N)));
  typedef E Mem __attribute__((ext_vector_type(N), aligned(sizeof(E))));
  Reg v;

  __device__ __forceinline__ float get(int i) const { return Elem<T>::widen(v[i]); }
  __device__ __forceinline__ void set(int i, float f) { v[i] = Elem<T>::narrow(f); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (E)0;
  }
  // Every value here is read once and written once by a launch: the accesses are marked as not
  // coming again (nontemporal), which leaves the L2s to what does.  Streams of 400 MB a buffer:
  // copy 5.65 -> 6.30 TB/s, two in and one out 5.48 -> 6.22, AdamW's four in and three out
  // 5.42 -> 5.88 (marking only the stores gains nothing).
  __device__ __forceinline__ void load(const T *p) {
    v = __builtin_nontemporal_load((const GANET_GLOBAL Mem *)(p));
  }
  __device__ __forceinline__ void store(T *p) const {
    __builtin_nontemporal_store((Mem)v, (GANET_GLOBAL Mem *)(p));
  }
  // ... or is read by what follows, or shares its lines with a neighbour
  __device__ __forceinline__ void load_kept(const T *p) { v = *(const GANET_GLOBAL Mem *)(p); }
  __device__ __forceinline__ void load_kept(const T *p, long long k) {
    if (k >= N)
      load_kept(p);
    else
      load(p, k);
  }
  __device__ __forceinline__ void store_kept(T *p) const { *(GANET_GLOBAL Mem *)(p) = (Mem)v; }
  __device__ __forceinline__ void store_kept(T *p, long long k) const {
    if (k >= N)
      store_kept(p);
    else
      store(p, k);
  }
  // To the compiler the values may have changed here: it widens them again afterwards (one
  // instruction a value at most) instead of keeping the wide ones, twice the registers.
  __device__ __forceinline__ void forget() {
    if constexpr (sizeof(Reg) == 16) {
      typedef unsigned int U4 __attribute__((ext_vector_type(4)));
      U4 u = __builtin_bit_cast(U4, v);
      asm volatile("" : "+v"(u));
      v = __builtin_bit_cast(Reg, u);
    } else if constexpr (sizeof(Reg) == 8) {
      typedef unsigned int U2 __attribute__((ext_vector_type(2)));
      U2 u = __builtin_bit_cast(U2, v);
      asm volatile("" : "+v"(u));
      v = __builtin_bit_cast(Reg, u);
    }
  }
  // the first k values only; the rest reads as zero / is left alone
  __device__ __forceinline__ void load(const T *p, long long k) {
    if (k >= N) {
      load(p);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = i < k ? ((const GANET_GLOBAL E *)p)[i] : (E)0;
    }
  }
  __device__ __forceinline__ void store(T *p, long long k) const {
    if (k >= N) {
      store(p);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < k) ((GANET_GLOBAL E *)p)[i] = v[i];
    }
  }
};

// ---- sums over lanes without LDS: DPP within a row of 16, then gfx950's row and half swaps --------
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// a's odd rows of 16 lanes change places with b's even ones: a = {a0, b0, a2, b2}, b = {a1, b1, a3, b3}
__device__ __forceinline__ void swap_rows(float &a, float &b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}
// a's upper 32 lanes change places with b's lower ones: a = {a_low, b_low}, b = {a_high, b_high}
__device__ __forceinline__ void swap_halves(float &a, float &b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}
// A barrier for what passes through LDS.  __syncthreads also waits for every load and store to
// global memory under way; here none of them carries anything to another wavefront, and those for
// the next tile or row are meant to stay under way.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The sum over each group of W neighbouring lanes, in all of them.
template <int W>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (W >= 2) v += dpp<0xB1>(v);      // quad_perm [1,0,3,2]
  if constexpr (W >= 4) v += dpp<0x4E>(v);      // quad_perm [2,3,0,1]
  if constexpr (W >= 8) v += dpp<0x141>(v);     // row_half_mirror
  if constexpr (W >= 16) v += dpp<0x140>(v);    // row_mirror
  if constexpr (W >= 32) {
    float o = v;
    swap_rows(v, o);
    v += o;
  }
  if constexpr (W >= 64) {
    float o = v;
    swap_halves(v, o);
    v += o;
  }
  return v;
}

}  // namespace ganet_vec
