// Layer norm over channels, forward and backward, for rows ([outer][C]: tokens, NHWC pixels) and
// for planes ([outer][C][inner]: NCHW maps, a channel stride of H * W).
//
//   y = (x - mean) rstd w + b;   xh = (x - mean) rstd, a = w dy:
//   dx = rstd (a - mean_C(a) - xh mean_C(a xh)),  dw = sum dy xh,  db = sum dy.
//
// The variance is formed from (x - mean), a second pass over the values: sums of squares would lose
// it where the mean is large.  Everything between the loads and the one rounding of each output is
// float32.  dw and db: every workgroup keeps sums of its own and leaves them in the workspace, a
// second launch adds them in a fixed order (no atomics: the same inputs give the same bits).
#include <math.h>

#include "vec_device.h"

namespace {

using ganet_vec::bf16_t;
using ganet_vec::f16_t;
using ganet_vec::group_sum;
using ganet_vec::Vec;

struct Args {
  const void *x, *g;                // g: grad_y
  const void *w, *b;                // may be null
  void *y;                          // y, or grad_x (may be null in the backward)
  float *mean, *rstd;               // written (forward, may be null) or read
  float *partial;                   // [workgroups][2][C] or null
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

template <typename T>
__device__ __forceinline__ float load1(const T *p) {
  Vec<T, 1> v;
  v.load(p);
  return v.get(0);
}
template <typename T>
__device__ __forceinline__ void store1(T *p, float f) {
  Vec<T, 1> v;
  v.set(0, f);
  v.store(p);
}

// The sum over a workgroup of `WAVES` wavefronts, in every lane; `part` [WAVES] is free again
// after the second barrier of the next call.
template <int WAVES>
__device__ __forceinline__ float block_sum(float v, float *part) {
  v = group_sum<64>(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) v += part[i];
  __syncthreads();
  return v;
}

// ---------------------------------------------------------------------------------------------
// Any C: a row (or 64 positions of a plane) per workgroup, the values read again for each pass
// ---------------------------------------------------------------------------------------------
constexpr int kThreads = 256;

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_rows_any_fwd(Args a) {
  __shared__ float part[kThreads / 64];
  for (long long row = blockIdx.x; row < a.outer; row += gridDim.x) {
    const T *x = (const T *)a.x + row * a.xs;
    T *y = (T *)a.y + row * a.ys;
    float s = 0.0f;
    for (int c = threadIdx.x; c < a.C; c += kThreads) s += load1(x + c);
    const float mean = block_sum<kThreads / 64>(s, part) / a.c;   // exact for equal values
    s = 0.0f;
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const float d = load1(x + c) - mean;
      s += d * d;
    }
    const float rstd = 1.0f / sqrtf(block_sum<kThreads / 64>(s, part) * a.inv_c + a.eps);
    for (int c = threadIdx.x; c < a.C; c += kThreads)
      store1(y + c, (load1(x + c) - mean) * rstd * load_weight(a.w, a.wdtype, c, 1.0f) +
                        load_weight(a.b, a.wdtype, c, 0.0f));
    if (threadIdx.x == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_rows_any_bwd(Args a) {
  __shared__ float part[kThreads / 64];
  extern __shared__ float sums[];               // [2][C]: a thread's own columns
  if (a.partial)
    for (int c = threadIdx.x; c < 2 * a.C; c += kThreads) sums[c] = 0.0f;
  __syncthreads();
  for (long long row = blockIdx.x; row < a.outer; row += gridDim.x) {
    const T *x = (const T *)a.x + row * a.xs;
    const T *g = (const T *)a.g + row * a.gs;
    T *dx = (T *)a.y + row * a.ys;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const float xh = (load1(x + c) - mean) * rstd, dy = load1(g + c);
      const float wa = dy * load_weight(a.w, a.wdtype, c, 1.0f);
      s1 += wa;
      s2 += wa * xh;
      if (a.partial) {
        sums[c] += dy * xh;
        sums[a.C + c] += dy;
      }
    }
    if (!a.y) continue;
    const float m1 = block_sum<kThreads / 64>(s1, part) * a.inv_c;
    const float m2 = block_sum<kThreads / 64>(s2, part) * a.inv_c;
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      const float xh = (load1(x + c) - mean) * rstd;
      const float wa = load1(g + c) * load_weight(a.w, a.wdtype, c, 1.0f);
      store1(dx + c, rstd * (wa - m1 - xh * m2));
    }
  }
  __syncthreads();
  if (a.partial)
    for (int c = threadIdx.x; c < 2 * a.C; c += kThreads)
      a.partial[(long long)blockIdx.x * 2 * a.C + c] = sums[c];
}

// Planes: lane l of every wavefront owns position 64 * tile + l, the wavefronts share the channels.
constexpr int kTile = 64;

__device__ __forceinline__ float positions_sum(float v, float (*part)[kTile]) {
  const int lane = threadIdx.x & 63;
  part[threadIdx.x >> 6][lane] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) v += part[i][lane];
  __syncthreads();
  return v;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_planes_any_fwd(Args a) {
  __shared__ float part[kThreads / 64][kTile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long tiles = (a.inner + kTile - 1) / kTile;
  for (long long i = blockIdx.x; i < a.outer * tiles; i += gridDim.x) {
    const long long b = i / tiles, pos = (i % tiles) * kTile + lane;
    const bool in = pos < a.inner;
    const T *x = (const T *)a.x + b * a.xs + pos;
    T *y = (T *)a.y + b * a.ys + pos;
    float s = 0.0f;
    for (int c = wave; c < a.C; c += kThreads / 64)
      if (in) s += load1(x + c * a.inner);
    const float mean = positions_sum(s, part) / a.c;
    s = 0.0f;
    for (int c = wave; c < a.C; c += kThreads / 64)
      if (in) {
        const float d = load1(x + c * a.inner) - mean;
        s += d * d;
      }
    const float rstd = 1.0f / sqrtf(positions_sum(s, part) * a.inv_c + a.eps);
    for (int c = wave; c < a.C; c += kThreads / 64)
      if (in)
        store1(y + c * a.inner, (load1(x + c * a.inner) - mean) * rstd * load_weight(a.w, a.wdtype, c, 1.0f) +
                                    load_weight(a.b, a.wdtype, c, 0.0f));
    if (in && wave == 0 && a.mean) {
      a.mean[b * a.inner + pos] = mean;
      a.rstd[b * a.inner + pos] = rstd;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_planes_any_bwd(Args a) {
  __shared__ float part[kThreads / 64][kTile];
  extern __shared__ float sums[];               // [2][C]: a wavefront's own channels
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (a.partial)
    for (int c = threadIdx.x; c < 2 * a.C; c += kThreads) sums[c] = 0.0f;
  __syncthreads();
  const long long tiles = (a.inner + kTile - 1) / kTile;
  for (long long i = blockIdx.x; i < a.outer * tiles; i += gridDim.x) {
    const long long b = i / tiles, pos = (i % tiles) * kTile + lane;
    const bool in = pos < a.inner;
    const T *x = (const T *)a.x + b * a.xs + pos;
    const T *g = (const T *)a.g + b * a.gs + pos;
    T *dx = (T *)a.y + b * a.ys + pos;
    const float mean = in ? a.mean[b * a.inner + pos] : 0.0f;
    const float rstd = in ? a.rstd[b * a.inner + pos] : 0.0f;
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = wave; c < a.C; c += kThreads / 64) {
      const float xh = in ? (load1(x + c * a.inner) - mean) * rstd : 0.0f;
      const float dy = in ? load1(g + c * a.inner) : 0.0f;
      const float wa = dy * load_weight(a.w, a.wdtype, c, 1.0f);
      s1 += wa;
      s2 += wa * xh;
      if (a.partial) {
        const float dw = group_sum<64>(dy * xh), db = group_sum<64>(dy);
        if (lane == 0) {
          sums[c] += dw;
          sums[a.C + c] += db;
        }
      }
    }
    if (!a.y) continue;
    const float m1 = positions_sum(s1, part) * a.inv_c;
    const float m2 = positions_sum(s2, part) * a.inv_c;
    for (int c = wave; c < a.C; c += kThreads / 64)
      if (in) {
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

// Adds the workgroups' sums: 64 channels a workgroup, its four wavefronts take every fourth of
// the `n` partial rows.  blockIdx.y: 0 the weight's gradient, 1 the bias's.
__global__ __launch_bounds__(kThreads) void ln_finish(const float *partial, int n, int C, void *dw, void *db,
                                                      int dtype) {
  __shared__ float part[kThreads / 64][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  void *out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0.0f;
  if (c < C)
    for (int i = wave; i < n; i += kThreads / 64) s += partial[((long long)i * 2 + blockIdx.y) * C + c];
  part[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= C) return;
  s = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
  if (dtype == GANET_F32)
    store1((float *)out + c, s);
  else if (dtype == GANET_BF16)
    store1((bf16_t *)out + c, s);
  else
    store1((f16_t *)out + c, s);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
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

// Workgroups of the backward, each with sums of its own: two on each of the 256 CUs.
int backward_blocks(const ganet_layer_norm_params *p) {
  const long long work = p->inner == 1 ? p->outer : p->outer * ((p->inner + kTile - 1) / kTile);
  return (int)(work < 512 ? work : 512);
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
  hipStream_t s = (hipStream_t)stream;
  const long long work = p->inner == 1 ? p->outer : p->outer * ((p->inner + kTile - 1) / kTile);
  const unsigned blocks = (unsigned)(work < 8192 ? work : 8192);
  return with_type(p->dtype, [&](auto t) {
    typedef decltype(t) T;
    if (p->inner == 1)
      ln_rows_any_fwd<T><<<dim3(blocks), dim3(kThreads), 0, s>>>(a);
    else
      ln_planes_any_fwd<T><<<dim3(blocks), dim3(kThreads), 0, s>>>(a);
    return ganet_check_launch();
  });
}

extern "C" size_t ganet_layer_norm_backward_workspace_bytes(const ganet_layer_norm_params *p) {
  if (params_ok(p, true) != GANET_OK) return 0;
  return ganet_align_up((size_t)(backward_blocks(p) + 1) * 2 * p->C * sizeof(float), 256);
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
    const size_t lds = sums ? (size_t)2 * p->C * sizeof(float) : 0;
    const int rc = with_type(p->dtype, [&](auto t) {
      typedef decltype(t) T;
      if (p->inner == 1)
        ln_rows_any_bwd<T><<<dim3(blocks), dim3(kThreads), lds, s>>>(a);
      else
        ln_planes_any_bwd<T><<<dim3(blocks), dim3(kThreads), lds, s>>>(a);
      return ganet_check_launch();
    });
    if (rc != GANET_OK) return rc;
  }
  if (!sums) return GANET_OK;
  ln_finish<<<dim3((p->C + 63) / 64, 2), dim3(kThreads), 0, s>>>((const float *)workspace, blocks, p->C, grad_weight,
                                                                grad_bias, p->weight_dtype);
  return ganet_check_launch();
}
