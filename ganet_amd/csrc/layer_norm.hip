// Layer norm over channels, forward and backward, for rows ([outer][C]: tokens, NHWC pixels) and
// for planes ([outer][C][inner]: NCHW maps, a channel stride of H * W).
//
//   y = (x - mean) rstd w + b;   xh = (x - mean) rstd, a = w dy:
//   dx = rstd (a - mean_C(a) - xh mean_C(a xh)),  dw = sum dy xh,  db = sum dy.
//
// The variance is formed from (x - mean), a second pass over the values: sums of squares would lose
// it where the mean is large.  Where the first sum is rounded even over equal values (kRounded), that pass also
// adds up d = x - mean, which is small: mean += sum d / C, var = sum d^2 / C - (sum d / C)^2.  The mean is then
// right to a rounding of its own, and equal values have no variance (without it a row of 96 times 15538.596
// came out as 0.3 instead of 0).  Everything between the loads and the one rounding of each output is
// float32.  dw and db: every workgroup keeps sums of its own and leaves them in the workspace, a
// second launch adds them in a fixed order; few positions are added in the first (no atomics: the same
// inputs give the same bits).
#include <math.h>

#include <type_traits>

#include "vec_device.h"

namespace {

using ganet_vec::bf16_t;
using ganet_vec::Elem;
using ganet_vec::f16_t;
using ganet_vec::group_sum;
using ganet_vec::Vec;

struct Args {
  const void *x, *g;                // g: grad_y
  const void *w, *b;                // may be null
  void *y;                          // y, or grad_x (may be null in the backward)
  float *mean, *rstd;               // written (forward, may be null) or read
  float *partial;                   // [workgroups][2][C] or null
  void *dw, *db;                    // grad_weight and grad_bias, where the launch writes them itself
  unsigned main;                    // workgroups before those that do
  long long outer, inner, xs, ys, gs;
  int C, wdtype;
  float eps, inv_c, c;              // 1 / C and C
};

__device__ __forceinline__ float load_weight(const void *w, int dtype, int c, float none) {
  if (!w) return none;
  if (dtype == GANET_F32) return ((const GANET_GLOBAL float *)w)[c];
  if (dtype == GANET_BF16)
    return ganet_vec::Elem<bf16_t>::widen(((const GANET_GLOBAL unsigned short *)w)[c]);
  return (float)((const GANET_GLOBAL _Float16 *)w)[c];
}

// Whether a float32 sum of equal values may be rounded: those of up to 16384 bfloat16 values (8 bits each) and
// of up to 8192 float16 ones (11 bits) are exact.
template <typename T>
constexpr bool kRounded = sizeof(T) == 4;

// The mean of c values from the sums of two halves.  Where each half is exact (float16), so is the mean of
// equal values: what the sum of the halves and the division round off goes back in.
__device__ __forceinline__ float mean_of_halves(float a, float b, float c) {
  const float s = a + b, back = s - a, lost = (a - (s - back)) + (b - back);
  const float m = s / c;
  return m + (fmaf(-m, c, s) + lost) / c;
}

// The corrected mean and 1 / deviation from the sums of d and d^2.  A mean smaller than the deviation stays: d
// is rounded to x's spacing, which is more than the first sum lost (rows of 4096 normal values: 4 times as far
// off with `more`).
__device__ __forceinline__ void correct(float sum, float squares, const Args &a, float &mean, float &rstd) {
  const float more = sum / a.c, all = squares * a.inv_c, left = all - more * more;
  // (no number where both are past the largest float32)
  const float var = left > 0.0f ? left : (left <= 0.0f ? 0.0f : all);
  if (mean * mean > var) mean += more;
  rstd = 1.0f / sqrtf(var + a.eps);
}

template <typename T>
__device__ __forceinline__ float load1(const T *p) {
  return Elem<T>::widen(*(const GANET_GLOBAL typename Elem<T>::type *)p);
}
template <typename T>
__device__ __forceinline__ void store1(T *p, float f) {
  *(GANET_GLOBAL typename Elem<T>::type *)p = Elem<T>::narrow(f);
}

template <typename T, int N>
__device__ __forceinline__ void load_some(const T *p, int left, float (&out)[N]) {
  if (left >= N) {
    const typename Vec<T, N>::Reg v = *(const GANET_GLOBAL typename Vec<T, N>::Mem *)p;
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] = Elem<T>::widen(v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] = k < left ? load1(p + k) : 0.0f;
  }
}

// N consecutive weights from column c on, `none` where there are none
template <int N>
__device__ __forceinline__ void load_weights(const void *w, int dtype, int c, int C, float none, float (&out)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) out[k] = none;
  if (!w || c >= C) return;
  if (dtype == GANET_F32)
    load_some<float, N>((const float *)w + c, C - c, out);
  else if (dtype == GANET_BF16)
    load_some<bf16_t, N>((const bf16_t *)w + c, C - c, out);
  else
    load_some<f16_t, N>((const f16_t *)w + c, C - c, out);
}

__device__ __forceinline__ void store_weight(void *w, int dtype, int c, float v) {
  if (!w) return;
  if (dtype == GANET_F32)
    store1((float *)w + c, v);
  else if (dtype == GANET_BF16)
    store1((bf16_t *)w + c, v);
  else
    store1((f16_t *)w + c, v);
}

// Where a backward leaves its sums over positions: nowhere; each workgroup's in the workspace, for a
// second launch; or, for few values, by workgroups of their own in the same launch, which read x and
// grad_y again (from the caches) and need no sums over channels.
enum Sums { kNoSums, kPartial, kApart };

// Adds a value over the lanes that are LANES apart (the row groups of a wavefront).
template <int LANES>
__device__ __forceinline__ float across_groups(float v) {
#pragma unroll
  for (int o = LANES; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// v[0] + ... + v[N - 1] in pairs, N a power of two
template <int N>
__device__ __forceinline__ float tree_sum(const float (&v)[N]) {
  if constexpr (N == 1) {
    return v[0];
  } else {
    float h[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) h[i] = v[i] + v[i + N / 2];
    return tree_sum(h);
  }
}

// ---------------------------------------------------------------------------------------------
// Planes of any C: 64 positions a workgroup, the values read again for each pass
// ---------------------------------------------------------------------------------------------
// More than 1024 channels, or planes of fewer positions than a vector.  Bound by latency: one value a load and
// three passes (4x2048x40x100: float32 forward 219 us, backward 641, bf16 234 and 465; the backward's two sums over a
// wavefront for each channel and tile are the most of it).
constexpr int kThreads = 256;

// Planes: lane l of every wavefront owns position 64 * tile + l, the wavefronts share the channels.
constexpr int kTile = 64;

// The sums of the first and the second two wavefronts.
struct Halves {
  float a, b;
};
__device__ __forceinline__ Halves positions_halves(float v, float (*part)[kTile]) {
  static_assert(kThreads / 64 == 4, "two halves of two");
  const int lane = threadIdx.x & 63;
  part[threadIdx.x >> 6][lane] = v;
  __syncthreads();
  const Halves h = {part[0][lane] + part[1][lane], part[2][lane] + part[3][lane]};
  __syncthreads();
  return h;
}
__device__ __forceinline__ float positions_sum(float v, float (*part)[kTile]) {
  const Halves h = positions_halves(v, part);
  return h.a + h.b;
}

// A wavefront's channels, kAtOnce of them at once: f(i, c, in) for the i-th of each turn; past the last
// `in` is false and c some channel, so that loads need no branch.  Sums are kept for each i by themselves:
// a lane's sum is ceil(C / 64) terms in order and then a tree (all of its C / 4 in order, 16384 equal terms
// lost 2^-14 of a mean).
constexpr int kAtOnce = 16;
constexpr int kWaves = kThreads / 64;
template <typename F>
__device__ __forceinline__ void channels_of_wave(int C, F &&f) {
  for (int c0 = (int)threadIdx.x >> 6; c0 < C; c0 += kAtOnce * kWaves)
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int c = c0 + i * kWaves;
      f(i, c < C ? c : c0, c < C);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_planes_any_fwd(Args a) {
  __shared__ float part[kWaves][kTile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long tiles = (a.inner + kTile - 1) / kTile;
  for (long long i = blockIdx.x; i < a.outer * tiles; i += gridDim.x) {
    const long long b = i / tiles, at = (i % tiles) * kTile + lane;
    const bool valid = at < a.inner;
    const long long pos = valid ? at : a.inner - 1;
    const T *x = (const T *)a.x + b * a.xs + pos;
    T *y = (T *)a.y + b * a.ys + pos;
    float s[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) s[k] = 0.0f;
    channels_of_wave(a.C, [&](int k, int c, bool in) {
      const float v = load1(x + c * a.inner);
      s[k] += in ? v : 0.0f;
    });
    const Halves sum = positions_halves(tree_sum(s), part);
    float mean = mean_of_halves(sum.a, sum.b, a.c), rstd;
    constexpr bool AGAIN = kRounded<T>;
    float more[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) s[k] = more[k] = 0.0f;
    channels_of_wave(a.C, [&](int k, int c, bool in) {
      const float d = load1(x + c * a.inner) - mean;
      s[k] += in ? d * d : 0.0f;
      if constexpr (AGAIN) more[k] += in ? d : 0.0f;
    });
    const float squares = positions_sum(tree_sum(s), part);
    if constexpr (AGAIN)
      correct(positions_sum(tree_sum(more), part), squares, a, mean, rstd);
    else
      rstd = 1.0f / sqrtf(squares * a.inv_c + a.eps);
    if (valid)
#pragma unroll 4
      for (int c = wave; c < a.C; c += kWaves)
        store1(y + c * a.inner, (load1(x + c * a.inner) - mean) * rstd * load_weight(a.w, a.wdtype, c, 1.0f) +
                                    load_weight(a.b, a.wdtype, c, 0.0f));
    if (valid && wave == 0 && a.mean) {
      a.mean[b * a.inner + pos] = mean;
      a.rstd[b * a.inner + pos] = rstd;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_planes_any_bwd(Args a) {
  __shared__ float part[kWaves][kTile];
  extern __shared__ float sums[];               // [2][C]: a wavefront's own channels; 128 KiB at most
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (a.partial)
    for (int c = threadIdx.x; c < 2 * a.C; c += kThreads) sums[c] = 0.0f;
  __syncthreads();
  const long long tiles = (a.inner + kTile - 1) / kTile;
  for (long long i = blockIdx.x; i < a.outer * tiles; i += gridDim.x) {
    const long long b = i / tiles, at = (i % tiles) * kTile + lane;
    const bool valid = at < a.inner;
    const long long pos = valid ? at : a.inner - 1;
    const T *x = (const T *)a.x + b * a.xs + pos;
    const T *g = (const T *)a.g + b * a.gs + pos;
    T *dx = (T *)a.y + b * a.ys + pos;
    const float mean = a.mean[b * a.inner + pos], rstd = a.rstd[b * a.inner + pos];
    float s1[kAtOnce], s2[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) s1[k] = s2[k] = 0.0f;
    channels_of_wave(a.C, [&](int k, int c, bool in) {
      const float xh = (load1(x + c * a.inner) - mean) * rstd, dy = load1(g + c * a.inner);
      const float wa = dy * load_weight(a.w, a.wdtype, c, 1.0f);
      s1[k] += in ? wa : 0.0f;
      s2[k] += in ? wa * xh : 0.0f;
      if (a.partial && in) {                    // a position past the last counts for nothing
        const float dw = group_sum<64>(valid ? dy * xh : 0.0f), db = group_sum<64>(valid ? dy : 0.0f);
        if (lane == 0) {
          sums[c] += dw;
          sums[a.C + c] += db;
        }
      }
    });
    if (!a.y) continue;
    const float m1 = positions_sum(tree_sum(s1), part) * a.inv_c;
    const float m2 = positions_sum(tree_sum(s2), part) * a.inv_c;
    if (valid)
#pragma unroll 4
      for (int c = wave; c < a.C; c += kWaves) {
        const float xh = (load1(x + c * a.inner) - mean) * rstd;
        const float wa = load1(g + c * a.inner) * load_weight(a.w, a.wdtype, c, 1.0f);
        store1(dx + c * a.inner, rstd * (wa - m1 - xh * m2));
      }
  }
  __syncthreads();
  if (a.partial)
    for (int c = threadIdx.x; c < 2 * a.C; c += kThreads)
      a.partial[(long long)blockIdx.x * 2 * a.C + c] = sums[c];
}

// ---------------------------------------------------------------------------------------------
// Rows in registers: each value is read once
// ---------------------------------------------------------------------------------------------
// A row is spread over LANES lanes (a part of a wavefront, one, four or sixteen), NV vectors of 16
// bytes each, and stays in registers from the load to the store: mean, variance and output take one
// pass over memory.  Narrow rows share a wavefront (64 / LANES of them), so that every load moves
// 1 KiB whatever C is.
template <typename T>
constexpr int kN = 16 / (int)sizeof(T);

// The sum over a row's lanes, in each of them.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float *part, int slot) {
  if constexpr (LANES <= 64) {
    return group_sum<LANES>(v);
  } else {
    // `part` holds a set of one float a wavefront for each slot; neighbouring calls use unlike ones, so one
    // barrier a call does
    constexpr int W = LANES / 64;
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) part[slot * W + (threadIdx.x >> 6)] = v;
    ganet_vec::lds_barrier();
    return group_sum<W>(part[slot * W + (threadIdx.x & (W - 1))]);
  }
}
// Two sums over one barrier, in slots 1 and 2.
template <int LANES>
__device__ __forceinline__ void row_sums(float &v, float &w, float *part) {
  if constexpr (LANES <= 64) {
    v = group_sum<LANES>(v);
    w = group_sum<LANES>(w);
  } else {
    constexpr int W = LANES / 64;
    v = group_sum<64>(v);
    w = group_sum<64>(w);
    if ((threadIdx.x & 63) == 0) {
      part[W + (threadIdx.x >> 6)] = v;
      part[2 * W + (threadIdx.x >> 6)] = w;
    }
    ganet_vec::lds_barrier();
    v = group_sum<W>(part[W + (threadIdx.x & (W - 1))]);
    w = group_sum<W>(part[2 * W + (threadIdx.x & (W - 1))]);
  }
}
// The mean of a row from its lanes' sums.
template <typename T, int LANES>
__device__ __forceinline__ float row_mean(float v, float *part, float c) {
  if constexpr (std::is_same<T, f16_t>::value && LANES == 512) {          // more than 8192 columns
    constexpr int W = LANES / 64;
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    ganet_vec::lds_barrier();
    const float half = group_sum<W / 2>(part[threadIdx.x & (W - 1)]);
    return mean_of_halves(half, ganet_vec::dpp<0x141>(half), c);          // mirrored in eight lanes: the other one
  } else {
    return row_sum<LANES>(v, part, 0) / c;
  }
}

// Forward.  R rows of a lane are loaded before the first is worked on.  The accesses are ordinary
// ones: marked as not coming again (as elsewhere here) they cost 2 to 5 % in this kernel.
template <typename T, int LANES, int NV, int R>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void ln_rows_fwd(Args a) {
  constexpr int N = kN<T>;
  constexpr int THREADS = LANES > 256 ? LANES : 256;
  constexpr int ROWS = THREADS / LANES;              // of a workgroup at once
  constexpr bool AGAIN = kRounded<T>;
  __shared__ float part[(AGAIN ? 3 : 2) * (LANES > 64 ? LANES / 64 : 1)];
  const int l = (int)threadIdx.x % LANES;
  const long long row0 = (long long)blockIdx.x * (ROWS * R) + (int)threadIdx.x / LANES;
  Vec<T, N> x[R][NV];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long long row = row0 + r * ROWS;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * LANES + l) * N;
      if (row < a.outer && c < a.C)
        x[r][v].load_kept((const T *)a.x + row * a.xs + c, a.C - c);
      else
        x[r][v].zero();
    }
  }
  float w[NV][N], b[NV][N];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * LANES + l) * N;
    load_weights<N>(a.w, a.wdtype, c, a.C, 1.0f, w[v]);
    load_weights<N>(a.b, a.wdtype, c, a.C, 0.0f, b[v]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long long row = row0 + r * ROWS;
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < N; ++k) s += x[r][v].get(k);
    float mean = row_mean<T, LANES>(s, part, a.c), rstd, more = 0.0f;
    s = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      x[r][v].forget();
      const int left = a.C - (v * LANES + l) * N;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float d = k < left ? x[r][v].get(k) - mean : 0.0f;
        s += d * d;
        if constexpr (AGAIN) more += d;
      }
    }
    if constexpr (AGAIN) {
      row_sums<LANES>(s, more, part);
      correct(more, s, a, mean, rstd);
    } else {
      rstd = 1.0f / sqrtf(row_sum<LANES>(s, part, 1) * a.inv_c + a.eps);
    }
    if (row >= a.outer) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * LANES + l) * N;
      if (c >= a.C) continue;
      x[r][v].forget();
      Vec<T, N> y;
#pragma unroll
      for (int k = 0; k < N; ++k) y.set(k, (x[r][v].get(k) - mean) * rstd * w[v][k] + b[v][k]);
      y.store_kept((T *)a.y + row * a.ys + c, a.C - c);
    }
    if (l == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// Backward.  Workgroups of sixteen wavefronts stay, one on each CU, and take rows in turn; a lane
// keeps its columns' sums of grad_weight and grad_bias in registers and requests the next row
// before it works on this one.  Few, large workgroups: each leaves [2][C] floats to be added.
constexpr int kBwdThreads = 1024;

// kApart: the sums of eight vectors of columns (128 bytes of a row; 64 are slower for wide rows, 512 x
// 5000 float32 17.8 and 14.3 us, and faster for few, 512 x 255 bf16 8.4 and 9.4).  128 groups of eight
// lanes take the rows, four at once.
constexpr int kStrip = 8;
template <typename T>
__device__ __forceinline__ void strip_sums(const Args &a, int strip) {
  constexpr int N = kN<T>, GROUPS = kBwdThreads / kStrip, U = 4;
  __shared__ float part[2][kBwdThreads / 64][kStrip * N];
  const int l = threadIdx.x & (kStrip - 1), c = (strip * kStrip + l) * N;
  float s[2][N];
#pragma unroll
  for (int k = 0; k < N; ++k) s[0][k] = s[1][k] = 0.0f;
  for (int row = (int)threadIdx.x / kStrip; row < (int)a.outer; row += GROUPS * U) {
    Vec<T, N> x[U], g[U];
    float mu[U], rs[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = row + u * GROUPS;
      const bool in = r < (int)a.outer;
      mu[u] = in ? a.mean[r] : 0.0f;
      rs[u] = in ? a.rstd[r] : 0.0f;
      if (in && c < a.C) {
        x[u].load_kept((const T *)a.x + r * a.xs + c, a.C - c);
        g[u].load_kept((const T *)a.g + r * a.gs + c, a.C - c);
      } else {
        x[u].zero();
        g[u].zero();
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float dy = g[u].get(k);
        s[0][k] += dy * ((x[u].get(k) - mu[u]) * rs[u]);
        s[1][k] += dy;
      }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float v = across_groups<kStrip>(s[which][k]);
      if ((threadIdx.x & 63) < kStrip) part[which][threadIdx.x >> 6][l * N + k] = v;
    }
  ganet_vec::lds_barrier();
  const int at = threadIdx.x % (kStrip * N), which = threadIdx.x / (kStrip * N);
  if (which > 1 || strip * kStrip * N + at >= a.C) return;
  float v = 0.0f;
#pragma unroll
  for (int i = 0; i < kBwdThreads / 64; ++i) v += part[which][i][at];
  store_weight(which ? a.db : a.dw, a.wdtype, strip * kStrip * N + at, v);
}

template <typename T, int LANES, int NV, Sums HOW>
__global__ __launch_bounds__(kBwdThreads) void ln_rows_bwd(Args a) {
  if constexpr (HOW == kApart)
    if (blockIdx.x >= a.main) {
      // neighbouring strips on one XCD: rows of odd length share cache lines
      const int i = (int)(blockIdx.x - a.main), strip = (i & 7) * ((int)(gridDim.x - a.main) >> 3) + (i >> 3);
      if (strip * kStrip * kN<T> < a.C) strip_sums<T>(a, strip);
      return;
    }
  constexpr bool SUMS = HOW == kPartial;
  constexpr int N = kN<T>;
  constexpr int ROWS = kBwdThreads / LANES;
  constexpr int W = LANES > 64 ? LANES / 64 : 1;
  __shared__ float part[4 * (kBwdThreads / 64)];
  extern __shared__ __align__(16) float sums[];      // [groups][columns], for the end
  const int l = (int)threadIdx.x % LANES;
  const int group = (int)threadIdx.x / LANES;
  // Weights stay in registers, or, where a lane has 16 columns or more, in LDS.
  constexpr bool LDS_W = NV * N >= 16;
  constexpr int COLS = LANES * NV * N;
  __shared__ __align__(16) float w_lds[LDS_W ? COLS : 1];
  float w_reg[LDS_W ? 1 : NV][N], dw[NV][N], db[NV][N];
  if constexpr (LDS_W) {
    for (int c = threadIdx.x; c < COLS; c += kBwdThreads) w_lds[c] = c < a.C ? load_weight(a.w, a.wdtype, c, 1.0f) : 0.0f;
    ganet_vec::lds_barrier();
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if constexpr (!LDS_W) load_weights<N>(a.w, a.wdtype, (v * LANES + l) * N, a.C, 1.0f, w_reg[v]);
#pragma unroll
    for (int k = 0; k < N; ++k) dw[v][k] = db[v][k] = 0.0f;
  }
  // `at`: l, but not known to be the same in every row, or the loads would move out of the loop and
  // into registers again
  auto weight = [&](int at, int v, int k) {
    return LDS_W ? w_lds[(v * LANES + at) * N + k] : w_reg[LDS_W ? 0 : v][k];
  };
  Vec<T, N> x[NV], g[NV];
  float mean, rstd;
  auto fetch = [&](long long row) {
    const bool in = row < a.outer;
    mean = in ? a.mean[row] : 0.0f;
    rstd = in ? a.rstd[row] : 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * LANES + l) * N;
      if (in && c < a.C) {
        x[v].load((const T *)a.x + row * a.xs + c, a.C - c);
        g[v].load((const T *)a.g + row * a.gs + c, a.C - c);
      } else {
        x[v].zero();
        g[v].zero();
      }
    }
  };
  constexpr bool AHEAD = !LDS_W;                     // 16 columns fill the 128 registers by themselves
  const long long step = (long long)a.main * ROWS;
  const long long first = (long long)blockIdx.x * ROWS;
  if (AHEAD) fetch(first + group);
  int turn = 0;
  for (long long base = first; base < a.outer; base += step) {      // uniform over the workgroup
    const long long row = base + group;
    Vec<T, N> xr[NV], gr[NV];
    if (!AHEAD) fetch(row);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      xr[v] = x[v];
      gr[v] = g[v];
    }
    const float mu = mean, rs = rstd;
    if (AHEAD && base + step < a.outer) fetch(row + step);
    float s1 = 0.0f, s2 = 0.0f;
    int at = l;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      // a vector after the other: widened all at once they would not fit the registers
      if (NV > 1) {
        xr[v].forget();
        gr[v].forget();
        asm volatile("" : "+v"(s1), "+v"(s2), "+v"(at));
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        // zero past the row's end: grad_y is zero there
        const float xh = (xr[v].get(k) - mu) * rs, dy = gr[v].get(k);
        const float wa = dy * weight(at, v, k);
        s1 += wa;
        s2 += wa * xh;
        if constexpr (SUMS) {
          dw[v][k] += dy * xh;
          db[v][k] += dy;
        }
      }
    }
    if (!a.y) continue;
    float m1, m2;
    if constexpr (LANES <= 64) {
      m1 = group_sum<LANES>(s1) * a.inv_c;
      m2 = group_sum<LANES>(s2) * a.inv_c;
    } else {
      s1 = group_sum<64>(s1);
      s2 = group_sum<64>(s2);
      float *p = part + turn * 2 * (kBwdThreads / 64);
      turn ^= 1;                                     // two sets: one barrier a row
      if ((threadIdx.x & 63) == 0) {
        p[threadIdx.x >> 6] = s1;
        p[kBwdThreads / 64 + (threadIdx.x >> 6)] = s2;
      }
      ganet_vec::lds_barrier();
      m1 = m2 = 0.0f;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        m1 += p[group * W + i];
        m2 += p[kBwdThreads / 64 + group * W + i];
      }
      m1 *= a.inv_c;
      m2 *= a.inv_c;
    }
    if (row >= a.outer) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * LANES + l) * N;
      xr[v].forget();
      gr[v].forget();
      if (NV > 1) asm volatile("" : "+v"(at));
      if (c >= a.C) continue;
      Vec<T, N> d;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float xh = (xr[v].get(k) - mu) * rs;
        d.set(k, rs * (gr[v].get(k) * weight(at, v, k) - m1 - xh * m2));
      }
      d.store_kept((T *)a.y + row * a.ys + c, a.C - c);
    }
  }
  if constexpr (SUMS) {
    // The row groups' sums meet in LDS, [groups][columns], the weight's and then the bias's (64 KiB
    // at most), and are added in their order.
    constexpr int GROUPS = LANES < 64 ? kBwdThreads / 64 : ROWS;
    const int mine = LANES < 64 ? (int)threadIdx.x / 64 : group;
    float *out = a.partial + (long long)blockIdx.x * 2 * a.C;
    if constexpr (LANES < 64) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int k = 0; k < N; ++k) {
          dw[v][k] = across_groups<LANES>(dw[v][k]);
          db[v][k] = across_groups<LANES>(db[v][k]);
        }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      ganet_vec::lds_barrier();
      if (LANES >= 64 || ((int)threadIdx.x & 63) < LANES) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int k = 0; k < N; ++k)
            sums[mine * COLS + (v * LANES + l) * N + k] = which ? db[v][k] : dw[v][k];
      }
      ganet_vec::lds_barrier();
      for (int c = threadIdx.x; c < a.C; c += kBwdThreads) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) s += sums[i * COLS + c];
        out[which * a.C + c] = s;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Planes in registers
// ---------------------------------------------------------------------------------------------
// A workgroup owns 16 vectors of neighbouring positions (VB bytes each, 256 bytes of a channel's
// plane at VB = 16) and all channels; a wavefront's four rows of 16 lanes and its WAVES wavefronts
// are 4 WAVES slots, each with up to NC consecutive channels in registers.  Sums over channels: a
// lane's own, then the four rows, then the wavefronts through LDS.
template <typename T, int VB, int NC, int WAVES>
struct Plane {
  static constexpr int N = VB / (int)sizeof(T);
  static constexpr int TILE = 16 * N;
  static constexpr int SLOTS = 4 * WAVES;
  static constexpr int THREADS = 64 * WAVES;
};

// s[M] of each lane, added over the workgroup's slots, in every lane.  First over a wavefront's four
// rows, two values an exchange, so that each row is left with a quarter of the values; these go
// through LDS, where a lane adds what it holds over the wavefronts; then the rows hand each other
// their quarters back.  For M = 16 and 8 wavefronts: 24 exchanges and 9 LDS accesses of 16 bytes
// without conflicts (every lane summing everything: 32 exchanges through LDS and 36 accesses, bf16
// backward 32x256x40x100 61 us instead of 50).
template <int M, int WAVES>
__device__ __forceinline__ void slots_sum(float (&s)[M], float (*part)[64][M / 4]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int Q = M / 4;
#pragma unroll
  for (int i = 0; i < 2 * Q; ++i) {
    ganet_vec::swap_halves(s[i], s[i + 2 * Q]);
    s[i] += s[i + 2 * Q];
  }
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    ganet_vec::swap_rows(s[i], s[i + Q]);
    s[i] += s[i + Q];                   // rows: values i, i + Q, i + 2 Q, i + 3 Q
    part[wave][lane][i] = s[i];
  }
  ganet_vec::lds_barrier();
#pragma unroll
  for (int i = 0; i < Q; ++i) s[i] = WAVES > 1 ? part[0][lane][i] + part[WAVES > 1][lane][i] : part[0][lane][i];
#pragma unroll
  for (int w = 2; w < WAVES; w += 2)                   // two wavefronts at once: half as many sums in order
#pragma unroll
    for (int i = 0; i < Q; ++i) s[i] += part[w][lane][i] + part[w + 1][lane][i];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    s[i + Q] = s[i];
    ganet_vec::swap_rows(s[i], s[i + Q]);
  }
#pragma unroll
  for (int i = 0; i < 2 * Q; ++i) {
    s[i + 2 * Q] = s[i];
    ganet_vec::swap_halves(s[i], s[i + 2 * Q]);
  }
}

// The tiles of a workgroup.  Workgroups go to the eight XCDs in turn, and each XCD has an L2 of its
// own: it gets an eighth of the tiles, neighbours one after another, so that the cache lines that two
// tiles share (planes start at any address) meet in one L2.
struct Share {
  unsigned end, step, at;                            // fewer than 2^31 tiles (with_plane_shape)
  __device__ __forceinline__ Share(unsigned tiles, unsigned workgroups) {
    const unsigned per = (tiles + 7) / 8, from = (blockIdx.x & 7) * per;
    at = from + (blockIdx.x >> 3);
    end = from + per < tiles ? from + per : tiles;
    step = (workgroups + 7 - (blockIdx.x & 7)) >> 3;
  }
};

// Where a lane's N positions begin.  A vector that would pass the plane's end is moved back to end
// there (the plane holds N positions at least): every lane then loads and stores whole vectors; the
// positions it shares with another lane get the same values from both, and `own` says from which
// element on they count in sums over positions (N: none).
template <int N>
__device__ __forceinline__ long long plane_position(long long pos, long long inner, int &own) {
  const long long left = inner - pos;
  own = left >= N ? 0 : (left > 0 ? N - (int)left : N);
  return left >= N ? pos : inner - N;
}

template <typename T, int VB, int NC, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void ln_planes_fwd(Args a, int tiles, int nc) {
  typedef Plane<T, VB, NC, WAVES> P;
  constexpr int N = P::N;
  constexpr bool AGAIN = kRounded<T>;
  constexpr int M = AGAIN ? 2 * N : N;               // sums of the second pass: of d^2, and of d
  __shared__ __align__(16) float part0[WAVES][64][N / 4], part1[WAVES][64][M / 4];
  __shared__ float weights[2][P::SLOTS * NC];
  int own;
  const Share share((unsigned)a.outer * (unsigned)tiles, gridDim.x);
  if (share.at >= share.end) return;
  const unsigned image = share.at / (unsigned)tiles;
  const long long img = image;
  const long long pos = plane_position<N>(
      (long long)(share.at - image * (unsigned)tiles) * P::TILE + (threadIdx.x & 15) * N, a.inner, own);
  const int c0 = (int)(threadIdx.x >> 4) * nc;       // nc <= NC channels of a slot
  const T *x = (const T *)a.x + img * a.xs + (long long)c0 * a.inner + pos;
  Vec<T, N> v[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    v[k].zero();
    if (k < nc && c0 + k < a.C) v[k].load(x + k * a.inner);
  }
  for (int c = threadIdx.x; c < a.C; c += P::THREADS) {
    weights[0][c] = load_weight(a.w, a.wdtype, c, 1.0f);
    weights[1][c] = load_weight(a.b, a.wdtype, c, 0.0f);
  }
  float mean[N], rstd[M];
#pragma unroll
  for (int j = 0; j < N; ++j) mean[j] = 0.0f;
#pragma unroll
  for (int j = 0; j < M; ++j) rstd[j] = 0.0f;
#pragma unroll
  for (int k = 0; k < NC; k += 2)                    // two channels at once: half as many sums in order
#pragma unroll
    for (int j = 0; j < N; ++j) mean[j] += v[k].get(j) + v[k + 1].get(j);
  slots_sum<N, WAVES>(mean, part0);                  // its barrier also covers the weights
#pragma unroll
  for (int k = 0; k < NC; ++k) v[k].forget();
#pragma unroll
  for (int j = 0; j < N; ++j) mean[j] /= a.c;
#pragma unroll
  for (int k = 0; k < NC; k += 2) {
    const bool in0 = k < nc && c0 + k < a.C, in1 = k + 1 < nc && c0 + k + 1 < a.C;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d0 = in0 ? v[k].get(j) - mean[j] : 0.0f, d1 = in1 ? v[k + 1].get(j) - mean[j] : 0.0f;
      rstd[j] += d0 * d0 + d1 * d1;
      if constexpr (AGAIN) rstd[N + j] += d0 + d1;
    }
  }
  slots_sum<M, WAVES>(rstd, part1);
#pragma unroll
  for (int k = 0; k < NC; ++k) v[k].forget();
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (AGAIN)
      correct(rstd[N + j], rstd[j], a, mean[j], rstd[j]);
    else
      rstd[j] = 1.0f / sqrtf(rstd[j] * a.inv_c + a.eps);
  }
  T *y = (T *)a.y + img * a.ys + (long long)c0 * a.inner + pos;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    if (k < nc && c0 + k < a.C) {
      const float w = weights[0][c0 + k], b = weights[1][c0 + k];
      Vec<T, N> o;
#pragma unroll
      for (int j = 0; j < N; ++j) o.set(j, (v[k].get(j) - mean[j]) * rstd[j] * w + b);
      o.store_kept(y + k * a.inner);
    }
  }
  if (threadIdx.x < 16 && a.mean) {
    Vec<float, N> m, r;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      m.set(j, mean[j]);
      r.set(j, rstd[j]);
    }
    m.store(a.mean + img * a.inner + pos);
    r.store(a.rstd + img * a.inner + pos);
  }
}

// Backward: 16 wavefronts a CU (128 registers), however they are grouped.  Loading the next tile into
// registers meanwhile was measured and gains nothing (bf16 32x256x40x100 47.4 and 47.6 us).
// kApart: the sums of one channel, a vector of each image's plane after the other.
template <typename T, int N, int THREADS>
__device__ __forceinline__ void channel_sums(const Args &a, int c) {
  __shared__ float part[2][THREADS / 64];
  constexpr int U = 2;
  const int vecs = (int)((a.inner + N - 1) / N), all = (int)a.outer * vecs;
  float dw = 0.0f, db = 0.0f;
  for (int i = threadIdx.x; i < all; i += THREADS * U) {
    Vec<T, N> x[U], g[U];
    Vec<float, N> mean[U], rstd[U];
    int own[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = i + u * THREADS, image = (at < all ? at : i) / vecs;
      const long long pos = plane_position<N>((long long)((at < all ? at : i) - image * vecs) * N, a.inner, own[u]);
      if (at >= all) own[u] = N;
      x[u].load_kept((const T *)a.x + image * a.xs + c * a.inner + pos);
      g[u].load_kept((const T *)a.g + image * a.gs + c * a.inner + pos);
      mean[u].load_kept(a.mean + image * a.inner + pos);
      rstd[u].load_kept(a.rstd + image * a.inner + pos);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float dy = j >= own[u] ? g[u].get(j) : 0.0f;
        dw += j >= own[u] ? dy * ((x[u].get(j) - mean[u].v[j]) * rstd[u].v[j]) : 0.0f;
        db += dy;
      }
  }
  dw = group_sum<64>(dw);
  db = group_sum<64>(db);
  if ((threadIdx.x & 63) == 0) {
    part[0][threadIdx.x >> 6] = dw;
    part[1][threadIdx.x >> 6] = db;
  }
  ganet_vec::lds_barrier();
  if (threadIdx.x > 1) return;
  float v = 0.0f;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) v += part[threadIdx.x][i];
  store_weight(threadIdx.x ? a.db : a.dw, a.wdtype, c, v);
}

template <typename T, int VB, int NC, int WAVES, Sums HOW>
__global__ __launch_bounds__(64 * WAVES, 4) void ln_planes_bwd(Args a, int tiles, int nc) {
  typedef Plane<T, VB, NC, WAVES> P;
  if constexpr (HOW == kApart)
    if (blockIdx.x >= a.main) return channel_sums<T, P::N, P::THREADS>(a, (int)(blockIdx.x - a.main));
  constexpr bool SUMS = HOW == kPartial;
  constexpr int N = P::N;
  __shared__ __align__(16) float part[2][WAVES][64][N / 2];
  __shared__ float weights[P::SLOTS * NC];
  const int c0 = (int)(threadIdx.x >> 4) * nc;
  for (int c = threadIdx.x; c < a.C; c += P::THREADS) weights[c] = load_weight(a.w, a.wdtype, c, 1.0f);
  ganet_vec::lds_barrier();
  float dw[NC], db[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) dw[k] = db[k] = 0.0f;
  int turn = 0;
  const Share share((unsigned)a.outer * (unsigned)tiles, a.main);
  for (unsigned i = share.at; i < share.end; i += share.step, turn ^= 1) {
    int own;
    const unsigned image = i / (unsigned)tiles;
    const long long img = image;
    const long long pos = plane_position<N>(
        (long long)(i - image * (unsigned)tiles) * P::TILE + (threadIdx.x & 15) * N, a.inner, own);
    const long long c_at = (long long)c0 * a.inner + pos;
    const T *x = (const T *)a.x + img * a.xs + c_at, *g = (const T *)a.g + img * a.gs + c_at;
    Vec<T, N> vx[NC], vg[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      vx[k].zero();
      vg[k].zero();
      if (k < nc && c0 + k < a.C) {
        vx[k].load(x + k * a.inner);
        vg[k].load(g + k * a.inner);
      }
    }
    Vec<float, N> mean, rstd;
    mean.load(a.mean + img * a.inner + pos);
    rstd.load(a.rstd + img * a.inner + pos);
    float m[2 * N];                                  // sums of a, of a xh
#pragma unroll
    for (int j = 0; j < 2 * N; ++j) m[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if (k < nc) {
        const float w = c0 + k < a.C ? weights[c0 + k] : 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float xh = (vx[k].get(j) - mean.v[j]) * rstd.v[j], dy = vg[k].get(j);
          const float wa = dy * w;
          m[j] += wa;
          m[N + j] = fmaf(wa, xh, m[N + j]);
          if constexpr (SUMS) {
            const float counted = j >= own ? dy : 0.0f;
            dw[k] += counted * xh;
            db[k] += counted;
          }
        }
      }
    }
    if (!a.y) continue;
    // two sets of part: the next tile's sums do not wait for this one's readers
    slots_sum<2 * N, WAVES>(m, part[turn]);
#pragma unroll
    for (int j = 0; j < 2 * N; ++j) m[j] *= a.inv_c;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      vx[k].forget();
      vg[k].forget();
    }
    T *dx = (T *)a.y + img * a.ys + c_at;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if (k < nc && c0 + k < a.C) {
        const float w = weights[c0 + k];
        Vec<T, N> o;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float xh = (vx[k].get(j) - mean.v[j]) * rstd.v[j];
          o.set(j, rstd.v[j] * (vg[k].get(j) * w - m[j] - xh * m[N + j]));
        }
        o.store_kept(dx + k * a.inner);
      }
    }
  }
  if constexpr (SUMS) {
    float *out = a.partial + (long long)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const float sw = group_sum<16>(dw[k]), sb = group_sum<16>(db[k]);
      if ((threadIdx.x & 15) == 0 && k < nc && c0 + k < a.C) {
        out[c0 + k] = sw;
        out[a.C + c0 + k] = sb;
      }
    }
  }
}

// Adds the workgroups' sums: 16 channels a workgroup, its 64 groups of 16 lanes take every 64th of
// the `n` partial rows, eight loads at a time: latency is all there is.  blockIdx.y: 0 the weight's
// gradient, 1 the bias's.
constexpr int kFinish = 1024;
constexpr int kFinishCols = 16;
__global__ __launch_bounds__(kFinish) void ln_finish(const float *partial, int n, int C, void *dw, void *db,
                                                     int dtype) {
  constexpr int SLOTS = kFinish / kFinishCols;
  __shared__ float part[kFinish / 64][kFinishCols];
  const int col = threadIdx.x % kFinishCols, slot = threadIdx.x / kFinishCols;
  const int c = blockIdx.x * kFinishCols + col;
  void *out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0.0f;
  const float *p = partial + (long long)blockIdx.y * C + (c < C ? c : 0);
  for (int i = slot; i < n; i += 8 * SLOTS) {
    float f[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) f[u] = i + u * SLOTS < n ? load1(p + (long long)(i + u * SLOTS) * 2 * C) : 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u) s += f[u];
  }
  float o = s;
  ganet_vec::swap_rows(s, o);
  s += o;
  o = s;
  ganet_vec::swap_halves(s, o);
  s += o;
  if ((threadIdx.x & 63) < kFinishCols) part[threadIdx.x >> 6][col] = s;
  __syncthreads();
  if (slot != 0 || c >= C) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < kFinish / 64; ++i) s += part[i][col];
  store_weight(out, dtype, c, s);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
constexpr long long kMostThreads = 1ll << 31;     // of one launch

bool dtype_ok(int d) { return d == GANET_F32 || d == GANET_BF16 || d == GANET_F16; }

int params_ok(const ganet_layer_norm_params *p, bool backward) {
  if (!p) return GANET_ERR_NULL;
  if (p->outer < 0 || p->inner < 1 || p->C < 1 || !dtype_ok(p->dtype) || !dtype_ok(p->weight_dtype) ||
      !(p->eps >= 0.0f))
    return GANET_ERR_BAD_SHAPE;
  if (p->C > GANET_LAYER_NORM_MAX_C) return GANET_ERR_UNSUPPORTED;
  const long long most = 1ll << 40;
  if (p->outer > most || p->inner > most / p->C || (p->outer > 0 && p->inner * p->C > (1ll << 46) / p->outer))
    return GANET_ERR_BAD_SHAPE;
  if (p->outer > 1) {
    const long long one = p->inner * p->C;
    const long long far = (1ll << 60) / p->outer;
    if (p->x_stride < one || p->y_stride < one || (backward && p->g_stride < one)) return GANET_ERR_BAD_SHAPE;
    if (p->x_stride > far || p->y_stride > far || (backward && p->g_stride > far)) return GANET_ERR_BAD_SHAPE;
  }
  return GANET_OK;
}

Args make_args(const ganet_layer_norm_params *p) {
  Args a = {};
  a.outer = p->outer;
  a.inner = p->inner;
  a.xs = p->x_stride;
  a.ys = p->y_stride;
  a.gs = p->g_stride;
  a.C = p->C;
  a.wdtype = p->weight_dtype;
  a.eps = p->eps;
  a.inv_c = 1.0f / (float)p->C;
  a.c = (float)p->C;
  return a;
}

template <typename F>
int with_type(int dtype, F &&f) {
  if (dtype == GANET_F32) return f(float());
  if (dtype == GANET_BF16) return f(bf16_t());
  return f(f16_t());
}

// ---- which kernel ----
// Rows: the narrowest of these that holds C, i.e. LANES * NV vectors of 16 bytes.  Forward: a
// wavefront a row while two vectors a lane do; then four vectors a lane rather than more wavefronts at
// the barriers for 16-bit values (2048 rows of 16384: 512 lanes of four 33 us, 1024 of two 39 us),
// two vectors a lane for float32 (8192 rows of 4096: 512 lanes of two 49 us, 256 of four 58, 1024 of one 54;
// 12000 of 2500: 52, 54 and 63 us).
// Backward: one vector a lane as long as possible, the registers hold the columns' sums and the next
// row (16384 rows of 4096 bf16: 512 lanes of one 70 us, 256 of two, without the next row, 76 us).
template <bool BACKWARD, typename T, typename F>
int with_row_shape(int C, F &&f) {
  const int vecs = (C + kN<T> - 1) / kN<T>;
#define GANET_ROW(LANES, NV) \
  if (vecs <= (LANES) * (NV)) return f(std::integral_constant<int, LANES>(), std::integral_constant<int, NV>())
  GANET_ROW(1, 1);
  GANET_ROW(2, 1);
  GANET_ROW(4, 1);
  GANET_ROW(8, 1);
  GANET_ROW(16, 1);
  GANET_ROW(32, 1);
  GANET_ROW(64, 1);
  if constexpr (BACKWARD) {
    GANET_ROW(128, 1);
    GANET_ROW(256, 1);
    GANET_ROW(512, 1);
  } else {
    GANET_ROW(64, 2);
    GANET_ROW(256, 1);
    GANET_ROW(256, 2);
  }
  if constexpr (!BACKWARD && sizeof(T) == 2) {
    GANET_ROW(256, 4);
    GANET_ROW(512, 4);
  } else {
    if constexpr (BACKWARD) {
      GANET_ROW(1024, 1);
    } else {
      GANET_ROW(512, 2);
    }
    GANET_ROW(1024, 2);
    if constexpr (sizeof(T) == 4) GANET_ROW(1024, 4);
  }
#undef GANET_ROW
  return GANET_ERR_UNSUPPORTED;           // past GANET_LAYER_NORM_MAX_C
}

long long tiles_of(const ganet_layer_norm_params *p, int tile) { return (p->inner + tile - 1) / tile; }

// Planes.  Forward: 16 channels a slot, as many wavefronts as C takes (bf16 128x64x40x100: one
// wavefront 22 us, four with four channels a slot 31 us; float32 44 and 47 us).  Backward, which keeps two maps and the channels' sums: eight channels a slot, and
// four where 16-bit values make eight positions a lane (64x128x40x100: 43 us, with eight 47 us;
// 32x256x40x100: 47 and 48 us; float32 with its four positions the other way round, 75 and 72 us).
enum { kAny = 0 };
template <bool BACKWARD, typename T, typename F>
int with_plane_shape(const ganet_layer_norm_params *p, F &&f) {
#define GANET_PLANE(VB, NC, WAVES)                                                  \
  if (p->C <= 4 * (WAVES) * (NC) && p->inner >= (VB) / (int)sizeof(T) &&            \
      p->outer * tiles_of(p, 16 * (VB) / (int)sizeof(T)) < kMostThreads / (64 * (WAVES)) - 8) \
    return f(std::integral_constant<int, VB>(), std::integral_constant<int, NC>(),  \
             std::integral_constant<int, WAVES>())
  if constexpr (!BACKWARD) {
    GANET_PLANE(16, 16, 1);
    GANET_PLANE(16, 16, 2);
    GANET_PLANE(16, 16, 4);
    GANET_PLANE(16, 16, 8);
    GANET_PLANE(16, 16, 16);
  } else {
    GANET_PLANE(16, 4, 4);
    if constexpr (sizeof(T) == 2) {
      GANET_PLANE(16, 4, 8);
      GANET_PLANE(16, 4, 16);
    } else {
      GANET_PLANE(16, 8, 4);
      GANET_PLANE(16, 8, 8);
    }
    GANET_PLANE(16, 8, 16);
    GANET_PLANE(8, 16, 16);
  }
#undef GANET_PLANE
  return f(std::integral_constant<int, kAny>(), std::integral_constant<int, 1>(), std::integral_constant<int, 1>());
}

// Up to where the sums over positions go to workgroups of the same launch.  One launch less is 3 us
// less for a call that the host bounds (250 rows of 256: 9.5 and 7.2 us), and wide rows leave no
// partial sums as large as themselves (256 x 16384 bf16 35.7 us and 18.7).  What it costs is one
// workgroup's way through all positions of its columns and reading the values twice.  The GPU's time
// over three sets of tensors in turn: 512 rows of 1024 float32 4.7 us (with partial sums 6.7), 1024 rows
// 13.8 (8.4); 4 x 256 x 40 x 100 bf16 11.7 (13.6), 8 x 256 x 40 x 100 19.7 (14.5).
constexpr long long kApartRows = 512, kApartPositions = 1 << 14, kApartValues = 1 << 22;

// Workgroups of the backward, each with sums of its own: what is on the chip at once.
int backward_blocks(const ganet_layer_norm_params *p) {
  int blocks = 0;
  with_type(p->dtype, [&](auto t) {
    typedef decltype(t) T;
    if (p->inner == 1)
      return with_row_shape<true, T>(p->C, [&](auto lanes, auto) {
        const long long need = (p->outer + kBwdThreads / lanes.value - 1) / (kBwdThreads / lanes.value);
        blocks = (int)(need < 256 ? need : 256);
        return GANET_OK;
      });
    return with_plane_shape<true, T>(p, [&](auto vb, auto nc, auto waves) {
      if constexpr (vb.value == kAny) {
        const long long need = p->outer * tiles_of(p, kTile);
        blocks = (int)(need < 512 ? need : 512);
      } else {
        typedef Plane<T, vb.value, nc.value, waves.value> P;
        const long long need = p->outer * tiles_of(p, P::TILE);
        const int most = 256 * 16 / waves.value;              // sixteen wavefronts a CU
        blocks = (int)(need < most ? need : most);
      }
      return GANET_OK;
    });
  });
  return blocks;
}

// Whether the sums go apart, into workgroups of the same launch.
bool sums_apart(const ganet_layer_norm_params *p) {
  const long long positions = p->outer * p->inner;
  if (p->inner == 1) return positions <= kApartRows;
  if (positions > kApartPositions || positions * p->C > kApartValues) return false;
  bool apart = false;
  with_type(p->dtype, [&](auto t) {
    return with_plane_shape<true, decltype(t)>(p, [&](auto vb, auto, auto) {
      apart = vb.value != kAny;
      return GANET_OK;
    });
  });
  return apart;
}

template <typename T>
int launch_forward(const ganet_layer_norm_params *p, const Args &a, hipStream_t s) {
  if (p->inner == 1)
    return with_row_shape<false, T>(p->C, [&](auto lanes, auto nv) {
      constexpr int L = lanes.value, NV = nv.value;
      constexpr int threads = L > 256 ? L : 256, rows = threads / L;
      // Two rows a lane (all their loads first, the weights read once for both) where that leaves
      // half of the chip's threads busy: 512000 rows of 64 bf16 24 us (one: 27, four: 26).
      constexpr int R = 2;
      const long long many = (p->outer + rows * R - 1) / (rows * R);
      const bool deep = many * threads >= 256 * 1024;
      const long long most = kMostThreads / threads * (deep ? rows * R : rows);    // rows of a launch
      Args part = a;
      for (long long at = 0; at < p->outer; at += most) {
        part.outer = p->outer - at < most ? p->outer - at : most;
        part.x = (const T *)a.x + at * a.xs;
        part.y = (T *)a.y + at * a.ys;
        part.mean = a.mean ? a.mean + at : nullptr;
        part.rstd = a.rstd ? a.rstd + at : nullptr;
        if (deep)
          ln_rows_fwd<T, L, NV, R><<<dim3((unsigned)((part.outer + rows * R - 1) / (rows * R))), dim3(threads), 0, s>>>(part);
        else
          ln_rows_fwd<T, L, NV, 1><<<dim3((unsigned)((part.outer + rows - 1) / rows)), dim3(threads), 0, s>>>(part);
        const int rc = ganet_check_launch();
        if (rc != GANET_OK) return rc;
      }
      return (int)GANET_OK;
    });
  return with_plane_shape<false, T>(p, [&](auto vb, auto nc, auto waves) {
    if constexpr (vb.value == kAny) {
      const long long work = p->outer * tiles_of(p, kTile);
      ln_planes_any_fwd<T><<<dim3((unsigned)(work < 8192 ? work : 8192)), dim3(kThreads), 0, s>>>(a);
    } else {
      typedef Plane<T, vb.value, nc.value, waves.value> P;
      const long long tiles = tiles_of(p, P::TILE);
      ln_planes_fwd<T, vb.value, nc.value, waves.value>
          <<<dim3((unsigned)((p->outer * tiles + 7) / 8 * 8)), dim3(P::THREADS), 0, s>>>(a, (int)tiles,
                                                                          (p->C + P::SLOTS - 1) / P::SLOTS);
    }
    return ganet_check_launch();
  });
}

template <typename T, Sums HOW>
int launch_backward(const ganet_layer_norm_params *p, Args a, int blocks, hipStream_t s) {
  a.main = (unsigned)blocks;
  if (p->inner == 1)
    return with_row_shape<true, T>(p->C, [&](auto lanes, auto nv) {
      constexpr int L = lanes.value, NV = nv.value;
      constexpr int groups = L < 64 ? kBwdThreads / 64 : kBwdThreads / L;
      constexpr size_t room = HOW == kPartial ? (size_t)groups * L * NV * kN<T> * sizeof(float) : 0;
      constexpr int columns = 8 * kStrip * kN<T>;              // of eight strips
      const int more = HOW == kApart ? (p->C + columns - 1) / columns * 8 : 0;
      ln_rows_bwd<T, L, NV, HOW><<<dim3(blocks + more), dim3(kBwdThreads), room, s>>>(a);
      return ganet_check_launch();
    });
  return with_plane_shape<true, T>(p, [&](auto vb, auto nc, auto waves) {
    if constexpr (vb.value == kAny) {
      ln_planes_any_bwd<T>
          <<<dim3(blocks), dim3(kThreads), HOW == kPartial ? (size_t)2 * p->C * sizeof(float) : 0, s>>>(a);
    } else {
      typedef Plane<T, vb.value, nc.value, waves.value> P;
      ln_planes_bwd<T, vb.value, nc.value, waves.value, HOW><<<dim3(blocks + (HOW == kApart ? p->C : 0)), dim3(P::THREADS), 0, s>>>(
          a, (int)tiles_of(p, P::TILE), (p->C + P::SLOTS - 1) / P::SLOTS);
    }
    return ganet_check_launch();
  });
}

}  // namespace

extern "C" int ganet_layer_norm_forward(const void *x, const void *weight, const void *bias, void *y, float *mean,
                                        float *rstd, const ganet_layer_norm_params *p, ganet_stream_t stream) {
  const int bad = params_ok(p, false);
  if (bad != GANET_OK) return bad;
  if (p->outer == 0) return GANET_OK;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return GANET_ERR_NULL;
  Args a = make_args(p);
  a.x = x;
  a.w = weight;
  a.b = bias;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  return with_type(p->dtype,
                   [&](auto t) { return launch_forward<decltype(t)>(p, a, (hipStream_t)stream); });
}

extern "C" size_t ganet_layer_norm_backward_workspace_bytes(const ganet_layer_norm_params *p) {
  if (params_ok(p, true) != GANET_OK) return 0;
  const size_t blocks = sums_apart(p) ? 0 : (size_t)backward_blocks(p);
  return ganet_align_up((blocks + 1) * 2 * p->C * sizeof(float), 256);
}

extern "C" int ganet_layer_norm_backward(const void *x, const void *weight, const void *grad_y, const float *mean,
                                         const float *rstd, void *grad_x, void *grad_weight, void *grad_bias,
                                         const ganet_layer_norm_params *p, void *workspace, size_t workspace_bytes,
                                         ganet_stream_t stream) {
  const int bad = params_ok(p, true);
  if (bad != GANET_OK) return bad;
  if (!grad_x && !grad_weight && !grad_bias) return GANET_ERR_NULL;
  const bool sums = grad_weight || grad_bias;
  if (sums && !workspace) return GANET_ERR_NULL;
  if (sums && workspace_bytes < ganet_layer_norm_backward_workspace_bytes(p)) return GANET_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  int blocks = 0;
  if (p->outer > 0) {
    if (!x || !grad_y || !mean || !rstd) return GANET_ERR_NULL;
    Args a = make_args(p);
    a.x = x;
    a.g = grad_y;
    a.w = weight;
    a.y = grad_x;
    a.mean = (float *)mean;
    a.rstd = (float *)rstd;
    a.partial = sums ? (float *)workspace : nullptr;
    blocks = backward_blocks(p);
    const bool apart = sums && sums_apart(p);
    if (apart) {
      a.dw = grad_weight;
      a.db = grad_bias;
    }
    const int rc = with_type(p->dtype, [&](auto t) {
      typedef decltype(t) T;
      if (apart) return launch_backward<T, kApart>(p, a, grad_x ? blocks : 0, s);
      return sums ? launch_backward<T, kPartial>(p, a, blocks, s) : launch_backward<T, kNoSums>(p, a, blocks, s);
    });
    if (rc != GANET_OK || apart) return rc;
  }
  if (!sums) return GANET_OK;
  ln_finish<<<dim3((p->C + kFinishCols - 1) / kFinishCols, 2), dim3(kFinish), 0, s>>>((const float *)workspace, blocks, p->C, grad_weight,
                                                                grad_bias, p->weight_dtype);
  return ganet_check_launch();
}
