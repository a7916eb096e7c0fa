// Gradients of moe_sum_reduce (sm_100a).
//
//   dy[m, k, :] = f w[m, k] g[m, :]          dw[m, k] = f sum_h g[m, h] y[m, k, h]          (fp32 sums)
//
// HBM-bound: y is read once, dy written once, g read once.  A block is some slots of one token: a thread holds a piece of g
// and requests the same piece of all its slots' rows before it uses the first.  The sum over h runs in a fixed order (thread,
// warp, block), so the result is the same in every run.
#include "common.cuh"

namespace xkb {
namespace {

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// 16 bytes of a row
template <typename T> struct Vec16;
template <> struct Vec16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <> struct Vec16<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
};

struct Args {
  const void *go, *y, *w;
  void *gy, *gw;
  int64_t M, H;
  int top_k;
  unsigned groups;   // blocks of a token
  float f;
};

constexpr int kMaxThreads = 256;

// SLOTS slots of a token per block.  y (and gw) or gy may be missing.
template <typename T, typename TW, int SLOTS>
__global__ void __launch_bounds__(kMaxThreads)
sum_reduce_grad_kernel(Args a) {
  constexpr int N = Vec16<T>::N;
  __shared__ float s_part[kMaxThreads / 32][SLOTS];
  const int64_t m = blockIdx.x / a.groups;
  const int k0 = (int)(blockIdx.x - m * a.groups) * SLOTS, n = min(SLOTS, a.top_k - k0);
  const int64_t slot0 = m * a.top_k + k0, hv = a.H / N;
  const uint4* g = reinterpret_cast<const uint4*>(static_cast<const T*>(a.go) + m * a.H);
  const uint4* y = reinterpret_cast<const uint4*>(static_cast<const T*>(a.y) + slot0 * a.H);
  uint4* gy = reinterpret_cast<uint4*>(static_cast<T*>(a.gy) + slot0 * a.H);
  float wk[SLOTS], acc[SLOTS];
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) {
    acc[k] = 0.f;
    wk[k] = a.f * (a.w != nullptr && k < n ? as_float(static_cast<const TW*>(a.w)[slot0 + k]) : 1.f);
  }
  for (int64_t i = threadIdx.x; i < hv; i += blockDim.x) {
    uint4 q[SLOTS];
    const uint4 gq = g[i];
    if (a.gw != nullptr) {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k)
        if (k < n) q[k] = __ldcs(y + k * hv + i);
    }
    float gv[N];
    Vec16<T>::unpack(gq, gv);
    if (a.gy != nullptr) {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k) {
        if (k >= n) break;
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = gv[e] * wk[k];
        __stcs(gy + k * hv + i, Vec16<T>::pack(v));
      }
    }
    if (a.gw != nullptr) {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k) {
        if (k >= n) break;
        float v[N];
        Vec16<T>::unpack(q[k], v);
#pragma unroll
        for (int e = 0; e < N; ++e) acc[k] = fmaf(gv[e], v[e], acc[k]);
      }
    }
  }
  if (a.gw == nullptr) return;
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], o);
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5][k] = acc[k];
  }
  __syncthreads();
  if ((int)threadIdx.x < n) {
    float sum = 0.f;
    for (unsigned i = 0; i < blockDim.x / 32; ++i) sum += s_part[i][threadIdx.x];
    put(static_cast<TW*>(a.gw) + slot0 + threadIdx.x, sum * a.f);
  }
}

// Any H, any alignment: a warp per slot.
template <typename T, typename TW>
__global__ void __launch_bounds__(256)
sum_reduce_grad_scalar_kernel(Args a) {
  const int lane = threadIdx.x & 31;
  const int64_t slots = a.M * a.top_k, warps = (int64_t)gridDim.x * 8;
  for (int64_t s = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); s < slots; s += warps) {
    const T* g = static_cast<const T*>(a.go) + s / a.top_k * a.H;
    const float w = a.f * (a.w != nullptr ? as_float(static_cast<const TW*>(a.w)[s]) : 1.f);
    float acc = 0.f;
    for (int64_t h = lane; h < a.H; h += 32) {
      const float x = as_float(g[h]);
      if (a.gy != nullptr) put(static_cast<T*>(a.gy) + s * a.H + h, x * w);
      if (a.gw != nullptr) acc = fmaf(x, as_float(static_cast<const T*>(a.y)[s * a.H + h]), acc);
    }
    if (a.gw == nullptr) continue;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) put(static_cast<TW*>(a.gw) + s, acc * a.f);
  }
}

template <typename T, typename TW, int SLOTS>
int launch_slots(Args a, cudaStream_t s) {
  const int64_t hv = a.H / Vec16<T>::N;
  a.groups = (unsigned)ceil_div(a.top_k, SLOTS);
  const int64_t steps = ceil_div(hv, (int64_t)kMaxThreads);   // as few threads as take the row in as many steps
  const unsigned threads = (unsigned)align_up(ceil_div(hv, steps), 32);
  sum_reduce_grad_kernel<T, TW, SLOTS><<<(unsigned)(a.M * a.groups), threads, 0, s>>>(a);
  XKB_CHECK_LAUNCH("sum_reduce_grad_kernel");
  return XKB_OK;
}

template <typename T, typename TW>
int launch(const Args& a, cudaStream_t s) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.go) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.gy);
  if (a.H % Vec16<T>::N == 0 && bits % 16 == 0 && a.M * a.top_k <= 0x7fffffff) {
    // slots per block: all of them where the tokens fill the chip
    if (a.top_k > 4 && a.M * ceil_div(a.top_k, 8) >= 2 * 148) return launch_slots<T, TW, 8>(a, s);
    if (a.top_k > 2 && a.M * ceil_div(a.top_k, 4) >= 2 * 148) return launch_slots<T, TW, 4>(a, s);
    if (a.top_k > 1 && a.M * ceil_div(a.top_k, 2) >= 2 * 148) return launch_slots<T, TW, 2>(a, s);
    return launch_slots<T, TW, 1>(a, s);
  }
  int64_t blocks = ceil_div(a.M * a.top_k, (int64_t)8);
  if (blocks > 148 * 32) blocks = 148 * 32;
  sum_reduce_grad_scalar_kernel<T, TW><<<(unsigned)blocks, 256, 0, s>>>(a);
  XKB_CHECK_LAUNCH("sum_reduce_grad_scalar_kernel");
  return XKB_OK;
}

}  // namespace
}  // namespace xkb

extern "C" int xkb_moe_sum_reduce_backward(const void* grad_out, int dtype, const void* y, const void* w, int w_dtype, void* grad_y,
                                           void* grad_w, int64_t M, int top_k, int64_t H, float routed_scaling_factor, void* stream) {
  using namespace xkb;
  XKB_REQUIRE(M >= 0 && H >= 0 && top_k >= 0, "moe_sum_reduce_backward: negative dimension");
  XKB_REQUIRE((dtype == XKB_BF16 || dtype == XKB_F32) && (w == nullptr || w_dtype == XKB_BF16 || w_dtype == XKB_F32),
              "moe_sum_reduce_backward: dtype codes must be XKB_BF16 or XKB_F32");
  XKB_REQUIRE(grad_w == nullptr || w != nullptr, "moe_sum_reduce_backward: grad_w without w");
  if (M == 0 || top_k == 0 || (grad_y == nullptr && grad_w == nullptr)) return XKB_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (H == 0) {   // empty sums
    if (grad_w != nullptr) XKB_CHECK_CUDA(cudaMemsetAsync(grad_w, 0, (size_t)(M * top_k) * (w_dtype == XKB_BF16 ? 2 : 4), s));
    return XKB_OK;
  }
  XKB_REQUIRE(grad_out != nullptr && (grad_w == nullptr || y != nullptr), "moe_sum_reduce_backward: null pointer");
  const Args a{grad_out, grad_w != nullptr ? y : nullptr, w, grad_y, grad_w, M, H, top_k, 0, routed_scaling_factor};
  const bool w16 = w != nullptr && w_dtype == XKB_BF16;
  if (dtype == XKB_BF16) return w16 ? launch<__nv_bfloat16, __nv_bfloat16>(a, s) : launch<__nv_bfloat16, float>(a, s);
  return w16 ? launch<float, __nv_bfloat16>(a, s) : launch<float, float>(a, s);
}
