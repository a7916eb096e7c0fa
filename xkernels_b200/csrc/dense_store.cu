// Dense products that are stored as they are (dense_dev.cuh).
#include "dense_dev.cuh"

namespace xkb {
namespace dense {

namespace {

template <int CG, int BN, int RW> int ask(int width, int* out) {
  using C = Cfg<CG, BN, RW, kStore>;
  auto kernel = dense_kernel<CG, BN, RW, false, kStore>;
  XKB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(width);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = width;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  XKB_CHECK_CUDA(cudaOccupancyMaxActiveClusters(out, kernel, &cfg));
  return XKB_OK;
}

}  // namespace

// (The kernels differ in registers, but not in how many CTAs an SM holds.)
int clusters_at_once(int dev, int cg, int bn, int read_warps, int width, int* out) {
  static std::atomic<int> known[64][4][9];
  const int kind = cg == 2 ? (bn == 256 ? 0 : 1) : read_warps == 8 ? 2 : 3;     // (64 columns take the room of 128)
  int n = dev < 64 ? known[dev][kind][width].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    const int rc = kind == 0   ? ask<2, 256, 8>(width, &n)
                   : kind == 1 ? ask<2, 128, 8>(width, &n)
                   : kind == 2 ? ask<1, 128, 8>(width, &n)
                               : ask<1, 128, 4>(width, &n);
    if (rc != XKB_OK) return rc;
    if (dev < 64) known[dev][kind][width].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return XKB_OK;
}

int run_store(bool b_mn, const Params& p, const Launch& l) {
  return b_mn ? run_variant<true, kStore>(p, l) : run_variant<false, kStore>(p, l);
}
int run_store_long(bool b_mn, const Params& p, const Launch& l) {
  if (l.bn == 256) return b_mn ? run_kernel<2, 256, 8, true, kStoreLong>(p, l) : run_kernel<2, 256, 8, false, kStoreLong>(p, l);
  return b_mn ? run_kernel<2, 128, 8, true, kStoreLong>(p, l) : run_kernel<2, 128, 8, false, kStoreLong>(p, l);
}

}  // namespace dense
}  // namespace xkb
