// AdamW over many tensors at once (states in 32 bits or in 8) and the norm of all gradients.
//
// Every operator here reads each value once, works a few tens of operations on it and writes it
// back: HBM bounds them.  What is left to design is (a) that one launch serves many tensors of any
// size, (b) that enough loads are in flight, (c) that nothing but the values moves.
//
// (a) The tensors' addresses travel in the kernel's arguments (no device table, no copy, nothing
// that a captured graph would have to keep alive; argument blocks stay below 4 KiB, longer lists
// take further launches).  A workgroup owns one chunk of one tensor; which one it finds by having
// each lane compare one entry of the running chunk counts and counting the ballot.
#include <math.h>

#include "vec_device.h"

namespace {

using ganet_vec::bf16_t;
using ganet_vec::f16_t;
using ganet_vec::Vec;

constexpr int kThreads = 256;

// The tensors of a launch: PTRS addresses each, the number of its first chunk, and how many values
// its last chunk holds (whole chunks precede it, so no length is needed).
template <int PTRS, int MOST>
struct Table {
  static constexpr int most = MOST;
  void *ptr[PTRS][MOST];
  int first[MOST + 1];               // [count]: all chunks
  unsigned short tail[MOST];
  int count;
};

// The tensor of a workgroup's chunk: the last that starts at or before it (a tensor without values
// has no chunk and starts where its successor does).
template <typename Tab>
__device__ __forceinline__ int find_tensor(const Tab &tab, int chunk) {
  const int lane = threadIdx.x & 63;
  int t = -1;
#pragma unroll
  for (int base = 0; base < Tab::most; base += 64) {
    const int i = base + lane < Tab::most ? base + lane : Tab::most - 1;
    t += __popcll(__ballot(base + lane < tab.count && tab.first[i] <= chunk));
  }
  return __builtin_amdgcn_readfirstlane(t);
}

// ---------------------------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------------------------
struct Hyper {
  float b1, omb1, b2, omb2;     // betas and what is missing to 1 (formed in double)
  float lr_c, rbc2, eps, decay; // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), eps, 1 - lr * wd
  float lr, wd, bc1, lnb1, lnb2;  // for the two pointers below
  unsigned key;                 // of the random words: seed, and the step where the host has it
  int skip;
  const float *stats;           // [norm, coefficient, non-finite] or null
  const long long *step;        // the step number on the device, or null
  const float *lr_dev;
};

struct Coef {
  float lr_c, rbc2, decay, gscale;
  unsigned key;
};

// False: the step is to be left out.
__device__ __forceinline__ bool coefficients(const Hyper &h, Coef &c) {
  c.lr_c = h.lr_c;
  c.rbc2 = h.rbc2;
  c.decay = h.decay;
  c.key = h.key;
  c.gscale = 1.0f;
  if (h.stats) {
    if (h.skip && h.stats[2] != 0.0f) return false;
    c.gscale = h.stats[1];
  }
  if (h.step || h.lr_dev) {
    const float lr = h.lr_dev ? *h.lr_dev : h.lr;
    float bc1 = h.bc1;
    if (h.step) {
      // 1 - b^t as -expm1(t ln b): ln b comes rounded from double, so the relative error of the
      // whole stays at a few 2^-24 even where 1 - b^t is small
      const long long t = *h.step;
      bc1 = -expm1f((float)t * h.lnb1);
      c.rbc2 = 1.0f / sqrtf(-expm1f((float)t * h.lnb2));
      c.key = h.key + (unsigned)t * 0x9E3779B1u;
    }
    c.lr_c = lr / bc1;
    c.decay = 1.0f - lr * h.wd;
  }
  return true;
}

enum { kParam, kGrad, kAvg, kSecond, kMaster32 };
template <bool MASTER>
struct Args32 {
  Table<MASTER ? 5 : 4, MASTER ? 82 : 98> t;
  Hyper h;
};
static_assert(sizeof(Args32<true>) <= 4096 && sizeof(Args32<false>) <= 4096, "kernel arguments");

// A lane takes one vector of 4 values, a workgroup 1024: many short workgroups keep more loads and
// stores under way than few with several vectors a lane (100 M float32 values: one vector 471 us,
// two 479, four 492; 114688 values: 4.0 us and 6.4 with four).
constexpr int kVec = 4;
constexpr int kChunk = kThreads * kVec;

template <typename TP, typename TG, bool MASTER>
__global__ __launch_bounds__(kThreads) void adamw32_kernel(Args32<MASTER> a) {
  Coef c;
  if (!coefficients(a.h, c)) return;
  const int t = find_tensor(a.t, (int)blockIdx.x);
  const long long at = (long long)((int)blockIdx.x - a.t.first[t]) * kChunk;
  const int left = (int)blockIdx.x + 1 == a.t.first[t + 1] ? a.t.tail[t] : kChunk;
  TP *p = (TP *)a.t.ptr[kParam][t] + at;
  const TG *g = (const TG *)a.t.ptr[kGrad][t] + at;
  float *m = (float *)a.t.ptr[kAvg][t] + at, *v = (float *)a.t.ptr[kSecond][t] + at;
  float *w = MASTER ? (float *)a.t.ptr[MASTER ? kMaster32 : 0][t] + at : nullptr;

  const int i = (int)threadIdx.x * kVec, k = left - i;
  if (k <= 0) return;
  Vec<TP, kVec> vp;
  Vec<TG, kVec> vg;
  Vec<float, kVec> vm, vv, vw;
  vg.load(g + i, k);
  vm.load(m + i, k);
  vv.load(v + i, k);
  if constexpr (MASTER)
    vw.load(w + i, k);
  else
    vp.load(p + i, k);
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const float gr = vg.get(j) * c.gscale;
    const float mm = a.h.b1 * vm.get(j) + a.h.omb1 * gr;
    const float sq = a.h.b2 * vv.get(j) + a.h.omb2 * (gr * gr);
    const float old = MASTER ? vw.get(j) : vp.get(j);
    const float now = old * c.decay - c.lr_c * (mm / (sqrtf(sq) * c.rbc2 + a.h.eps));
    vm.set(j, mm);
    vv.set(j, sq);
    if constexpr (MASTER) vw.set(j, now);
    vp.set(j, now);   // 16-bit weights: rounded once, to nearest
  }
  vm.store(m + i, k);
  vv.store(v + i, k);
  if constexpr (MASTER) vw.store(w + i, k);
  vp.store(p + i, k);
}

// ---- states in 8 bits -------------------------------------------------------------------------
// m and r = sqrt(v) are held as e4m3 times one float32 scale for each 256 consecutive values of a
// tensor (scale = the block's largest magnitude / 448).  r and not v: e4m3 spans 2^18, so v spans
// 2^36, and the step divides by r.  Both are rounded up or down at random, with the probability
// that keeps the mean: with beta2 = 0.999 an average moves by a thousandth a step, far less than
// half of e4m3's spacing (2^-4), and rounding to nearest would stop it for good.  An r above zero
// never becomes zero (m over a zero r would be a step of m / eps).
// The new moments, their scales and what is rounded are formed by single float32 operations in a fixed
// order (no contraction; root and reciprocal rounded to nearest): a state is the same bits wherever
// the formula is computed so, and two trainings do not drift apart by roundings that fell otherwise.
constexpr int kBlock = GANET_STATE_BLOCK;
enum { kAvgScale = 4, kSecondScale, kMaster8 };
template <bool MASTER>
struct Args8 {
  Table<MASTER ? 7 : 6, MASTER ? 62 : 70> t;
  int tensor0;                 // the first tensor's place in the whole list
  Hyper h;
};
static_assert(sizeof(Args8<true>) <= 4096 && sizeof(Args8<false>) <= 4096, "kernel arguments");

static_assert(kBlock == 64 * kVec, "a wavefront holds a block");

__device__ __forceinline__ unsigned mix32(unsigned x) {
  x ^= x >> 16;
  x *= 0xBB67AE85u;
  x ^= x >> 15;
  x *= 0x6A09E667u;
  return x ^ (x >> 16);
}

// A value as e4m3 in byte SEL of `to`, up or down by 16 random bits (the upper ones of `random`).
// The instruction adds the upper 20 bits of its second operand to the 20 bits of mantissa that
// e4m3 drops and truncates; below 2^-6, where e4m3 is evenly spaced by 2^-9, to as many bits below
// 2^-9 (both compared with that definition on a million values: no difference).  Bit 15 stands for
// half of the sixteenth bit, so that the numbers are centred.
template <int SEL>
__device__ __forceinline__ unsigned to_e4m3(float v, unsigned random, unsigned to) {
  return (unsigned)__builtin_amdgcn_cvt_sr_fp8_f32(v, (int)(random | 0x8000u), (int)to, SEL);
}

// Root and reciprocal rounded to nearest, by one Newton step on the instructions' estimates (both
// equal sqrtf and 1 / x for every float32 from 1 to 4; the general forms, which also serve the ends
// of the range, cost a step 3 %).  A root of less than 2^-126 is zero here, of infinity NaN.
__device__ __forceinline__ float root(float x) {
  const float y = __builtin_amdgcn_rsqf(x), s = x * y;
  const float r = fmaf(fmaf(-s, s, x), 0.5f * y, s);
  return x < 0x1p-126f ? 0.0f : r;
}
__device__ __forceinline__ float reciprocal(float x) {        // 2^-110 .. 2^126
  const float y = __builtin_amdgcn_rcpf(x);
  return fmaf(fmaf(-x, y, 1.0f), y, y);
}

__device__ __forceinline__ unsigned max3(unsigned a, unsigned b, unsigned c) {
  const unsigned m = b > c ? b : c;
  return a > m ? a : m;
}
// The largest of a wavefront's values, in a scalar register
__device__ __forceinline__ unsigned block_max(unsigned v) {
  auto with = [&](unsigned o) { v = v > o ? v : o; };
  with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
  with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
  with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
  with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
  with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, true));   // row 0 -> 1, 2 -> 3
  with((unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, true));   // row 1 -> 2 and 3
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
constexpr unsigned kInf = 0x7F800000u;

template <typename TP, typename TG, bool MASTER>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(Args8<MASTER> a) {
  Coef c;
  if (!coefficients(a.h, c)) return;
  const int t = find_tensor(a.t, (int)blockIdx.x);
  const long long at = (long long)((int)blockIdx.x - a.t.first[t]) * kChunk;
  const int left = (int)blockIdx.x + 1 == a.t.first[t + 1] ? a.t.tail[t] : kChunk;
  TP *p = (TP *)a.t.ptr[kParam][t] + at;
  const TG *g = (const TG *)a.t.ptr[kGrad][t] + at;
  unsigned char *m = (unsigned char *)a.t.ptr[kAvg][t] + at, *r = (unsigned char *)a.t.ptr[kSecond][t] + at;
  const long long block0 = at / kBlock;
  float *ms = (float *)a.t.ptr[kAvgScale][t] + block0, *rs = (float *)a.t.ptr[kSecondScale][t] + block0;
  float *w = MASTER ? (float *)a.t.ptr[MASTER ? kMaster8 : 0][t] + at : nullptr;
  const unsigned key = mix32(c.key + (unsigned)(a.tensor0 + t) * 0x85EBCA6Bu);
  typedef unsigned char Byte4 __attribute__((ext_vector_type(4), aligned(1)));

  const int i = (int)threadIdx.x * kVec, k = left - i;
  Vec<TP, kVec> vp;
  Vec<TG, kVec> vg;
  Vec<float, kVec> vw;
  unsigned vm = 0, vr = 0;
  float sm = 0.0f, sr = 0.0f;
  vg.zero();
  if (k > 0) {
    vg.load(g + i, k);
    if constexpr (MASTER)
      vw.load(w + i, k);
    else
      vp.load(p + i, k);
    sm = ((const GANET_GLOBAL float *)ms)[i / kBlock];
    sr = ((const GANET_GLOBAL float *)rs)[i / kBlock];
    if (k >= kVec) {
      vm = __builtin_bit_cast(unsigned, __builtin_nontemporal_load((const GANET_GLOBAL Byte4 *)(m + i)));
      vr = __builtin_bit_cast(unsigned, __builtin_nontemporal_load((const GANET_GLOBAL Byte4 *)(r + i)));
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (j < k) {
          vm |= (unsigned)m[i + j] << (8 * j);
          vr |= (unsigned)r[i + j] << (8 * j);
        }
    }
  }
  float nm[kVec], nr[kVec], sq[kVec];
  // Magnitudes are compared as integers: the order is the same, and what is not finite comes out on
  // top.
  unsigned um = 0, ur = 0;
#pragma unroll
  for (int j = 0; j < kVec; j += 2) {
#pragma clang fp contract(off)
    const auto m2 = j ? __builtin_amdgcn_cvt_pk_f32_fp8(vm, true) : __builtin_amdgcn_cvt_pk_f32_fp8(vm, false);
    const auto r2 = j ? __builtin_amdgcn_cvt_pk_f32_fp8(vr, true) : __builtin_amdgcn_cvt_pk_f32_fp8(vr, false);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float gr = vg.get(j + e) * c.gscale;
      const float rr = r2[e] * sr;
      nm[j + e] = m2[e] * sm * a.h.b1 + a.h.omb1 * gr;
      sq[j + e] = rr * rr * a.h.b2 + gr * gr * a.h.omb2;
      nr[j + e] = root(sq[j + e]);
    }
    um = max3(um, __float_as_uint(nm[j]) & 0x7FFFFFFFu, __float_as_uint(nm[j + 1]) & 0x7FFFFFFFu);
    ur = max3(ur, __float_as_uint(nr[j]), __float_as_uint(nr[j + 1]));
  }
  um = block_max(um);
  ur = block_max(ur);
  // What is not finite reaches its own value only: it is left out of the scales.  After a gradient that
  // is not, both codes are e4m3's NaN.  A finite gradient whose square is not leaves a second moment
  // of infinity, as in float32: r's code is NaN over an m that is none, and the value stands still (m over
  // infinity) in this step and in all that follow.
  unsigned bad = 0, held = 0;           // a bit a value: both codes NaN; r's
  if (um >= kInf || ur >= kInf) {
    um = ur = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      // (a NaN of its root by a finite m can only come from r's code)
      const unsigned mb = __float_as_uint(nm[j]) & 0x7FFFFFFFu, rb = __float_as_uint(nr[j]);
      if (mb >= kInf) {
        bad |= 1u << j;
      } else if (rb >= kInf) {
        held |= 1u << j;
        nr[j] = INFINITY;
      } else {
        if (mb > um) um = mb;
        if (rb > ur) ur = rb;
      }
    }
    um = block_max(um);
    ur = block_max(ur);
  }
  if (k <= 0) return;                   // after the exchanges between a block's lanes
  float tm = __uint_as_float(um);
  const float tr = __uint_as_float(ur);
  if (tm < 0x1p-110f) tm = 0.0f;        // 448 / tm would overflow: such a block is held as zeros
  const float im = tm > 0.0f ? 448.0f * reciprocal(tm) : 0.0f;
  const float ir = tr > 0.0f ? 448.0f * reciprocal(tr) : 0.0f;
  const unsigned bkey = mix32(key + (unsigned)(block0 + i / kBlock) * 0xC2B2AE35u);
  unsigned om = 0, orr = 0;
  auto value = [&](auto J) {
    constexpr int j = J.value;
    unsigned h = bkey + (unsigned)((i + j) % kBlock) * 0x9E3779B1u;
    h ^= h >> 16;
    h *= 0xBB67AE85u;
    h ^= h >> 15;
    om = to_e4m3<j>(__builtin_amdgcn_fmed3f(nm[j] * im, -448.0f, 448.0f), h << 16, om);
    // above zero and below e4m3's smallest: the smallest
    orr = to_e4m3<j>(__builtin_amdgcn_fmed3f(nr[j] * ir, nr[j] > 0.0f ? 0x1p-9f : 0.0f, 448.0f),
                     h & 0xFFFF0000u, orr);
    const float old = MASTER ? vw.get(j) : vp.get(j);
    // a root above zero is 2^-63 at least: the bound only keeps a moment over a second moment that
    // counts as zero (and eps = 0) finite
    const float part = nm[j] * __builtin_amdgcn_rcpf(fmaxf(fmaf(nr[j], c.rbc2, a.h.eps), 0x1p-64f));
    const float now = fmaf(-c.lr_c, part, old * c.decay);
    if constexpr (MASTER) vw.set(j, now);
    vp.set(j, now);
  };
  value(std::integral_constant<int, 0>());
  value(std::integral_constant<int, 1>());
  value(std::integral_constant<int, 2>());
  value(std::integral_constant<int, 3>());
  if (bad | held) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      if (bad >> j & 1) om |= 0x7Fu << (8 * j);
      if ((bad | held) >> j & 1) orr |= 0x7Fu << (8 * j);
    }
  }
  if constexpr (MASTER) vw.store(w + i, k);
  vp.store(p + i, k);
  if (k >= kVec) {
    __builtin_nontemporal_store(__builtin_bit_cast(Byte4, om), (GANET_GLOBAL Byte4 *)(m + i));
    __builtin_nontemporal_store(__builtin_bit_cast(Byte4, orr), (GANET_GLOBAL Byte4 *)(r + i));
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (j < k) {
        m[i + j] = (unsigned char)(om >> (8 * j));
        r[i + j] = (unsigned char)(orr >> (8 * j));
      }
  }
  if (i % kBlock == 0) {
    ((GANET_GLOBAL float *)ms)[i / kBlock] = tm * (1.0f / 448.0f);
    ((GANET_GLOBAL float *)rs)[i / kBlock] = tr * (1.0f / 448.0f);
  }
}

// ---------------------------------------------------------------------------------------------
// The norm of all gradients
// ---------------------------------------------------------------------------------------------
// A vector's squares (4 or 8) are added in float32, the vectors in float64: float32 alone would lose
// the small gradients of a long sum, and float64 for every value makes the conversions the bound.
// Where float32 is no safe place for a vector's squares (a sum past 2^100, or under 2^-100 and not
// zero) that vector is added in float64.  Each workgroup leaves one partial sum, a second launch adds
// them in their order: the same inputs give the same bits.
// The list's entries are packed to 12 bytes, so that a launch takes 320 tensors: a lower and an
// upper address word (48 bits), the first chunk (16 bits), the last chunk's values (30) and the type.
constexpr int kTensorsN = 320;
struct ArgsN {
  unsigned low[kTensorsN];
  unsigned high_first[kTensorsN];
  unsigned tail_type[kTensorsN];
  int count;
  unsigned chunks, chunk;
  double *partial;
};
static_assert(sizeof(ArgsN) <= 4096, "kernel arguments");
constexpr int kUnrollN = 4;

template <typename T, int N>
__device__ __forceinline__ double squares(const Vec<T, N> &v) {
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < N; ++k) s = fmaf(v.get(k), v.get(k), s);
  if (s > 0x1p-100f && s < 0x1p100f) return (double)s;
  double d = 0.0;                    // also the way of zeros, infinities and NaN
#pragma unroll
  for (int k = 0; k < N; ++k) d = fma((double)v.get(k), (double)v.get(k), d);
  return d;
}

template <typename T, int N>
__device__ __forceinline__ double sum_squares(const T *g, long long n) {
  double s[kUnrollN] = {0, 0, 0, 0};
  long long i = (long long)threadIdx.x * N;
  constexpr long long step = (long long)kThreads * N;
  for (; i + (kUnrollN - 1) * step + N <= n; i += kUnrollN * step) {
    Vec<T, N> v[kUnrollN];
#pragma unroll
    for (int u = 0; u < kUnrollN; ++u) v[u].load(g + i + u * step);
#pragma unroll
    for (int u = 0; u < kUnrollN; ++u) s[u] += squares(v[u]);
  }
  for (; i < n; i += step) {
    Vec<T, N> v;
    v.load(g + i, n - i);
    s[0] += squares(v);
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(ArgsN a) {
  const int lane = threadIdx.x & 63;
  int t = -1;
#pragma unroll
  for (int base = 0; base < kTensorsN; base += 64)
    t += __popcll(__ballot(base + lane < a.count && (a.high_first[base + lane] & 0xFFFF) <= blockIdx.x));
  t = __builtin_amdgcn_readfirstlane(t);
  const unsigned first = a.high_first[t] & 0xFFFF, type = a.tail_type[t] >> 30;
  const unsigned next = t + 1 < a.count ? a.high_first[t + 1] & 0xFFFF : a.chunks;
  const char *g = (const char *)((unsigned long long)(a.high_first[t] >> 16) << 32 | a.low[t]);
  const long long at = (long long)(blockIdx.x - first) * a.chunk;
  const long long n = blockIdx.x + 1 == next ? a.tail_type[t] & 0x3FFFFFFF : a.chunk;
  double s;
  if (type == GANET_F32)
    s = sum_squares<float, 4>((const float *)g + at, n);
  else if (type == GANET_BF16)
    s = sum_squares<bf16_t, 8>((const bf16_t *)g + at, n);
  else
    s = sum_squares<f16_t, 8>((const f16_t *)g + at, n);
  __shared__ double part[kThreads / 64];
  s = wave_sum(s);
  if (lane == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    for (int w = 0; w < kThreads / 64; ++w) all += part[w];
    a.partial[blockIdx.x] = all;
  }
}

constexpr int kFinish = 1024;
__global__ __launch_bounds__(kFinish) void grad_norm_finish_kernel(const double *partial, long long n,
                                                                   double max_norm, double inv_scale,
                                                                   float *stats) {
  double s = 0.0;
  for (long long i = threadIdx.x; i < n; i += kFinish) s += partial[i];
  s = wave_sum(s);
  __shared__ double part[kFinish / 64];
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = 0.0;
    for (int w = 0; w < kFinish / 64; ++w) all += part[w];
    const double norm = sqrt(all) * fabs(inv_scale);
    const bool fine = (float)norm < INFINITY;       // false for NaN too
    const double clip = max_norm / (norm + 1e-6);
    stats[0] = (float)norm;
    stats[1] = fine ? (float)(inv_scale * (clip < 1.0 ? clip : 1.0)) : 0.0f;
    stats[2] = fine ? 0.0f : 1.0f;
    stats[3] = 0.0f;
  }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
constexpr long long kMostValues = 1ll << 40;      // of one tensor
constexpr long long kMostBlocks = 1ll << 23;      // of one launch: its threads stay below 2^32

bool dtype_ok(int d) { return d == GANET_F32 || d == GANET_BF16 || d == GANET_F16; }

template <typename F>
int with_types(int pd, int gd, bool master, F &&f) {
  auto grad = [&](auto p, auto m) {
    typedef decltype(p) TP;
    if (gd == GANET_F32) return f(TP(), float(), m);
    if (gd == GANET_BF16) return f(TP(), bf16_t(), m);
    return f(TP(), f16_t(), m);
  };
  if (pd == GANET_F32) return grad(float(), std::false_type());
  if (pd == GANET_BF16)
    return master ? grad(bf16_t(), std::true_type()) : grad(bf16_t(), std::false_type());
  return master ? grad(f16_t(), std::true_type()) : grad(f16_t(), std::false_type());
}

// Takes the list in launches; `ptr(x, k)` is the k-th address of a tensor.
template <int PTRS, int MOST, typename Ptr, typename Launch>
int in_launches(const ganet_step_tensor *ts, int count, long long chunk, Table<PTRS, MOST> &tab, Ptr &&ptr,
                Launch &&launch) {
  for (int i = 0; i < count;) {
    const int start = i;
    int k = 0;
    long long blocks = 0;
    for (; i < count && k < MOST; ++i, ++k) {
      const long long n = ts[i].n, need = (n + chunk - 1) / chunk;
      if (blocks + need > kMostBlocks) break;
      tab.first[k] = (int)blocks;
      tab.tail[k] = (unsigned short)(n - (need - 1) * chunk);      // not read where need == 0
      for (int j = 0; j < PTRS; ++j) tab.ptr[j][k] = ptr(ts[i], j);
      blocks += need;
    }
    tab.first[k] = (int)blocks;
    tab.count = k;
    if (blocks == 0) continue;
    const int rc = launch((unsigned)blocks, start);
    if (rc != GANET_OK) return rc;
  }
  return GANET_OK;
}

void *address(const ganet_step_tensor &x, int k) {
  switch (k) {
    case kParam: return x.param;
    case kGrad: return const_cast<void *>(x.grad);
    case kAvg: return x.exp_avg;
    default: return x.second;
  }
}

}  // namespace

extern "C" int ganet_adamw_step(const ganet_step_tensor *tensors, int count, const ganet_adamw_params *p,
                                ganet_stream_t stream) {
  if (!p || (count > 0 && !tensors)) return GANET_ERR_NULL;
  if (count < 0 || !dtype_ok(p->param_dtype) || !dtype_ok(p->grad_dtype) ||
      (p->state_bits != 32 && p->state_bits != 8) || p->reserved != 0)
    return GANET_ERR_BAD_SHAPE;
  if (!(p->lr >= 0.0) || !(p->beta1 >= 0.0 && p->beta1 < 1.0) || !(p->beta2 >= 0.0 && p->beta2 < 1.0) ||
      !(p->eps >= 0.0) || !(p->weight_decay >= 0.0) || isinf(p->lr) || isinf(p->eps) || isinf(p->weight_decay))
    return GANET_ERR_BAD_SHAPE;
  if (!p->step_device && p->step < 1) return GANET_ERR_BAD_SHAPE;
  const bool small = p->state_bits == 8;
  bool master = false, any = false;
  for (int i = 0; i < count; ++i) {
    const ganet_step_tensor &t = tensors[i];
    if (t.n < 0 || t.n > kMostValues) return GANET_ERR_BAD_SHAPE;
    if (t.n == 0) continue;            // has no addresses
    if (!any) master = t.master != nullptr;
    any = true;
    if ((t.master != nullptr) != master) return GANET_ERR_BAD_SHAPE;
    if (!t.param || !t.grad || !t.exp_avg || !t.second) return GANET_ERR_NULL;
    if (small && (!t.exp_avg_scale || !t.second_scale)) return GANET_ERR_NULL;
    if (t.n > kMostBlocks * kChunk) return GANET_ERR_UNSUPPORTED;    // before any tensor is stepped
  }
  if (master && p->param_dtype == GANET_F32) return GANET_ERR_BAD_SHAPE;

  Hyper h;
  h.b1 = (float)p->beta1;
  h.omb1 = (float)(1.0 - p->beta1);
  h.b2 = (float)p->beta2;
  h.omb2 = (float)(1.0 - p->beta2);
  const double t = p->step_device ? 1.0 : (double)p->step;
  const double bc1 = p->beta1 > 0 ? -expm1(t * log(p->beta1)) : 1.0;
  const double bc2 = p->beta2 > 0 ? -expm1(t * log(p->beta2)) : 1.0;
  h.lr_c = (float)(p->lr / bc1);
  h.rbc2 = (float)(1.0 / sqrt(bc2));
  h.eps = (float)p->eps;
  h.decay = (float)(1.0 - p->lr * p->weight_decay);
  h.lr = (float)p->lr;
  h.wd = (float)p->weight_decay;
  h.bc1 = (float)bc1;
  h.lnb1 = (float)log(p->beta1);      // -inf for 0: 1 - exp(-inf) = 1
  h.lnb2 = (float)log(p->beta2);
  h.key = p->seed + (p->step_device ? 0u : (unsigned)p->step * 0x9E3779B1u);
  h.skip = p->skip_nonfinite != 0;
  h.stats = p->grad_stats;
  h.step = (const long long *)p->step_device;
  h.lr_dev = p->lr_device;

  hipStream_t s = (hipStream_t)stream;
  return with_types(p->param_dtype, p->grad_dtype, master, [&](auto tp, auto tg, auto tm) {
    typedef decltype(tp) TP;
    typedef decltype(tg) TG;
    constexpr bool M = decltype(tm)::value;
    if (!small) {
      Args32<M> a;
      a.h = h;
      return in_launches(
          tensors, count, kChunk, a.t,
          [](const ganet_step_tensor &x, int k) { return k == kMaster32 ? (void *)x.master : address(x, k); },
          [&](unsigned blocks, int) {
            adamw32_kernel<TP, TG, M><<<dim3(blocks), dim3(kThreads), 0, s>>>(a);
            return ganet_check_launch();
          });
    }
    Args8<M> a;
    a.h = h;
    return in_launches(
        tensors, count, kChunk, a.t,
        [](const ganet_step_tensor &x, int k) {
          if (k == kAvgScale) return (void *)x.exp_avg_scale;
          if (k == kSecondScale) return (void *)x.second_scale;
          return k == kMaster8 ? (void *)x.master : address(x, k);
        },
        [&](unsigned blocks, int start) {
          a.tensor0 = start;
          adamw8_kernel<TP, TG, M><<<dim3(blocks), dim3(kThreads), 0, s>>>(a);
          return ganet_check_launch();
        });
  });
}

// ---- norm ----
namespace {
// Values of a workgroup: 8192 workgroups for long lists (400 M bf16 values 122 us; 2048 workgroups,
// what the chip holds at once, 131 us), 8192 values (8 float32 vectors a thread) at least.
long long norm_chunk(const int64_t *numel, int count) {
  long long total = 0;
  for (int i = 0; i < count; ++i) total += numel[i];
  const long long unit = 8192;
  const long long even = (total + 8191) / 8192;
  return even <= unit ? unit : (even + unit - 1) / unit * unit;
}
int norm_list_ok(const int64_t *numel, int count) {
  if (count < 0 || count > (1 << 20)) return GANET_ERR_BAD_SHAPE;
  if (count > 0 && !numel) return GANET_ERR_NULL;
  long long total = 0;                 // below 2^40: a chunk's length fits its 30 bits
  for (int i = 0; i < count; ++i) {
    if (numel[i] < 0 || numel[i] > kMostValues || total + numel[i] > kMostValues) return GANET_ERR_BAD_SHAPE;
    total += numel[i];
  }
  return GANET_OK;
}
}  // namespace

extern "C" size_t ganet_grad_norm_workspace_bytes(const int64_t *numel, int count) {
  if (norm_list_ok(numel, count) != GANET_OK) return 0;
  const long long chunk = norm_chunk(numel, count);
  long long blocks = 0;
  for (int i = 0; i < count; ++i) blocks += (numel[i] + chunk - 1) / chunk;
  return ganet_align_up((size_t)(blocks + 1) * sizeof(double), 256);
}

extern "C" int ganet_grad_norm(const void *const *grads, const int64_t *numel, const int32_t *dtypes, int count,
                               double max_norm, double inv_scale, float *stats, void *workspace,
                               size_t workspace_bytes, ganet_stream_t stream) {
  const int bad = norm_list_ok(numel, count);
  if (bad != GANET_OK) return bad;
  if (!stats || !workspace || (count > 0 && (!grads || !dtypes))) return GANET_ERR_NULL;
  if (!(max_norm >= 0.0) || !(fabs(inv_scale) < INFINITY)) return GANET_ERR_BAD_SHAPE;
  for (int i = 0; i < count; ++i) {
    if (!dtype_ok(dtypes[i])) return GANET_ERR_BAD_SHAPE;
    if (numel[i] > 0 && !grads[i]) return GANET_ERR_NULL;
    if ((unsigned long long)grads[i] >> 48) return GANET_ERR_UNSUPPORTED;      // no device address
  }
  if (workspace_bytes < ganet_grad_norm_workspace_bytes(numel, count)) return GANET_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  ArgsN a;
  const long long chunk = norm_chunk(numel, count);
  a.chunk = (unsigned)chunk;
  long long done = 0;
  for (int i = 0; i < count;) {
    int k = 0;
    long long blocks = 0;
    for (; i < count && k < kTensorsN; ++i, ++k) {     // 8192 chunks and one a tensor at most: 16 bits hold them
      const long long need = (numel[i] + chunk - 1) / chunk;
      const unsigned long long at = (unsigned long long)grads[i];
      a.low[k] = (unsigned)at;
      a.high_first[k] = (unsigned)(at >> 32) << 16 | (unsigned)blocks;
      a.tail_type[k] = (unsigned)dtypes[i] << 30 | (need ? (unsigned)(numel[i] - (need - 1) * chunk) : 0);
      blocks += need;
    }
    if (blocks == 0) continue;
    a.count = k;
    a.chunks = (unsigned)blocks;
    a.partial = (double *)workspace + done;
    grad_norm_kernel<<<dim3((unsigned)blocks), dim3(kThreads), 0, s>>>(a);
    const int rc = ganet_check_launch();
    if (rc != GANET_OK) return rc;
    done += blocks;
  }
  grad_norm_finish_kernel<<<dim3(1), dim3(kFinish), 0, s>>>((const double *)workspace, done, max_norm, inv_scale,
                                                          stats);
  return ganet_check_launch();
}
