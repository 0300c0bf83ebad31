// Host-only: the size / plan queries of the library under UBSan + ASan with random and extreme
// parameters (tools/asan_plan.sh).  No launch happens in any of these calls; what is checked is
// that no signed overflow, bad shift or out-of-range conversion sits in the host arithmetic.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <random>

#include "ganet_hip.h"

static std::mt19937_64 rng(99);
static int32_t pick(int kind) {
  static const int32_t extreme[] = {0, 1, -1, 2, 3, 7, 31, 32, 33, 63, 64, 65, 127, 128, 255, 256, 257, 1023,
                                    4096, 65535, 65536, 1 << 20, (1 << 24) + 1, 0x3fffffff, 0x7fffffff,
                                    (int32_t)0x80000000, -65536};
  switch (kind) {
    case 0: return (int32_t)(rng() % 9) + 1;
    case 1: return (int32_t)(rng() % 300) + 1;
    case 2: return extreme[rng() % (sizeof extreme / sizeof extreme[0])];
    default: return (int32_t)rng();
  }
}

static int64_t pick64(int kind) {
  static const int64_t far[] = {1ll << 31, (1ll << 33) + 1, 1ll << 40, (1ll << 40) + 1, 1ll << 46, 1ll << 60,
                                INT64_MAX, INT64_MIN, -1};
  return kind < 3 ? pick(kind) : (rng() % 2 ? far[rng() % 9] : (int64_t)rng());
}

int main() {
  unsigned long long acc = 0;
  for (int it = 0; it < 400000; ++it) {
    ganet_dcn_params p;
    std::memset(&p, 0, sizeof p);
    int32_t *f = reinterpret_cast<int32_t *>(&p);
    const int wild = it % 4;
    for (size_t i = 0; i < sizeof p / 4; ++i)
      f[i] = pick(wild == 0 ? (int)(rng() % 2) : (wild == 1 ? (int)(rng() % 3) : (int)(rng() % 4)));
    if (wild < 3) {   // mostly plausible enums so that the plans get past the first checks
      p.dtype = (int32_t)(rng() % 3);
      p.x_layout = (int32_t)(rng() % 2);
      p.out_layout = (int32_t)(rng() % 2);
      p.mfma_bf16 = (int32_t)(rng() % 3);
      p.fuse_relu = p.offset_is_points = p.weight_is_packed = p.debug = 0;
      static const int32_t algos[] = {0, 1, 2, 3, 4, 5, 6, 0x100, 0x102, 0x105, 0x200, 0x300, 0x400};
      p.algo = algos[rng() % 13];
      p.groups = (int32_t)(rng() % 3) + 1;
      p.deformable_groups = (int32_t)(rng() % 3) + 1;
    }
    acc += ganet_deform_conv_workspace_bytes(&p);
    acc += (unsigned)ganet_deform_conv_algorithm(&p);
    acc += ganet_deform_conv_status_offset(&p);
    acc += ganet_deform_conv_y_offset(&p);
    acc += ganet_deform_conv_packed_weight_bytes(&p);
    acc += ganet_deform_conv_backward_workspace_bytes(&p);
    acc += (unsigned)ganet_dcn_out_size(f[2], f[9], f[11], f[5], f[7]);

    ganet_decode_params d;
    std::memset(&d, 0, sizeof d);
    d.B = pick((int)(rng() % 4));
    d.H = pick((int)(rng() % 4));
    d.W = pick((int)(rng() % 4));
    d.max_kpts = pick((int)(rng() % 4));
    d.max_centers = pick((int)(rng() % 4));
    d.max_groups = pick((int)(rng() % 4));
    d.flags = (int32_t)(rng() % 32);
    acc += ganet_decode_workspace_bytes(&d);

    ganet_layer_norm_params n;
    std::memset(&n, 0, sizeof n);
    n.outer = pick64((int)(rng() % 4));
    n.inner = rng() % 3 ? pick64((int)(rng() % 4)) : 1;
    n.C = pick((int)(rng() % 3));
    n.x_stride = rng() % 2 ? n.C * (n.inner & 0xFFFFFFFF) : pick64((int)(rng() % 4));
    n.y_stride = rng() % 2 ? n.x_stride : pick64((int)(rng() % 4));
    n.g_stride = rng() % 2 ? n.x_stride : pick64((int)(rng() % 4));
    n.dtype = (int32_t)(rng() % 3);
    n.weight_dtype = (int32_t)(rng() % 4);
    acc += ganet_layer_norm_backward_workspace_bytes(&n);

    int64_t numel[5];
    for (int64_t &k : numel) k = wild == 3 ? pick64((int)(rng() % 4)) : (int64_t)(rng() % (1ull << (rng() % 41)));
    acc += ganet_grad_norm_workspace_bytes(numel, (int)(rng() % 6));
  }
  std::printf("plan fuzz: 400000 parameter sets, checksum %llu\n", acc);
  return 0;
}
