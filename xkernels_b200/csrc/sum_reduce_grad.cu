// Gradients of moe_sum_reduce (sm_100a).
//
//   dy[m, k, :] = f w[m, k] g[m, :]          dw[m, k] = f sum_h g[m, h] y[m, k, h]          (fp32 sums)
//
// HBM-bound: y is read once, dy written once, g read once.  A block is some slots of one token: a thread holds a piece of g
// and requests the same piece of all its slots' rows before it uses the first.  Rows whose ends lie anywhere go in narrower
// accesses, several at once.  The sum over h runs in a fixed order (thread,
// warp, block), so the result is the same in every run.
// 8192 x 8 x 7168 bf16, both gradients: 307 us, 6.5 TB/s.  4096 x 8 rows of 4096 / 4100 / 4098 / 4097 bf16 (accesses of 16 / 8 / 4 / 2 bytes)
// 86 / 98 / 116 / 154 us; of 2048 / 2050 / 2049 fp32 86 / 95 / 106.
#include "common.cuh"

namespace xkb {
namespace {

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// N neighbouring elements, one access
template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = unsigned short; };
template <typename T, int N> using word = typename Word<N * (int)sizeof(T)>::type;

template <int N> __device__ __forceinline__ void unpack(const word<float, N>& q, float (&v)[N], float) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = reinterpret_cast<const float*>(&q)[i];
}
template <int N> __device__ __forceinline__ void unpack(const word<__nv_bfloat16, N>& q, float (&v)[N], __nv_bfloat16) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = bf16_bits_to_float(reinterpret_cast<const unsigned short*>(&q)[i]);
}
template <int N> __device__ __forceinline__ word<float, N> pack(const float (&v)[N], float) {
  word<float, N> q;
#pragma unroll
  for (int i = 0; i < N; ++i) reinterpret_cast<float*>(&q)[i] = v[i];
  return q;
}
template <int N> __device__ __forceinline__ word<__nv_bfloat16, N> pack(const float (&v)[N], __nv_bfloat16) {
  word<__nv_bfloat16, N> q;
  if constexpr (N == 1) {
    q = (unsigned short)pack_bf16(v[0], 0.f);   // (the conversion of a single value runs on the special-function unit)
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) reinterpret_cast<uint32_t*>(&q)[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
  }
  return q;
}

struct Args {
  const void *go, *y, *w;
  void *gy, *gw;
  int64_t M, H;
  int top_k;
  unsigned groups;   // blocks of a token
  float f;
};

constexpr int kMaxThreads = 256;

// SLOTS slots of a token per block, N elements per access (rows of an odd number of elements start anywhere), COLS accesses at once.
// y (and gw) or gy may be missing.
template <typename T, typename TW, int SLOTS, int N, int COLS>
__global__ void __launch_bounds__(kMaxThreads)
sum_reduce_grad_kernel(Args a) {
  using W = word<T, N>;
  __shared__ float s_part[kMaxThreads / 32][SLOTS];
  const int64_t m = blockIdx.x / a.groups;
  const int k0 = (int)(blockIdx.x - m * a.groups) * SLOTS, n = min(SLOTS, a.top_k - k0);
  const int64_t slot0 = m * a.top_k + k0;
  const unsigned hv = (unsigned)(a.H / N);   // SLOTS rows of it stay below 2^31
  const W* g = reinterpret_cast<const W*>(static_cast<const T*>(a.go) + m * a.H);
  const W* y = reinterpret_cast<const W*>(static_cast<const T*>(a.y) + slot0 * a.H);
  W* gy = reinterpret_cast<W*>(static_cast<T*>(a.gy) + slot0 * a.H);
  float wk[SLOTS], acc[SLOTS];
#pragma unroll
  for (int k = 0; k < SLOTS; ++k) {
    acc[k] = 0.f;
    wk[k] = a.f * (a.w != nullptr && k < n ? as_float(static_cast<const TW*>(a.w)[slot0 + k]) : 1.f);
  }
  for (unsigned i0 = threadIdx.x; i0 < hv; i0 += COLS * blockDim.x) {
    W q[COLS][SLOTS], gq[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const unsigned i = i0 + c * blockDim.x;
      if (i >= hv) continue;
      gq[c] = g[i];
      if (a.gw != nullptr) {
#pragma unroll
        for (int k = 0; k < SLOTS; ++k)
          if (k < n) q[c][k] = __ldcs(y + k * hv + i);
      }
    }
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const unsigned i = i0 + c * blockDim.x;
      if (i >= hv) continue;
      float gv[N];
      unpack<N>(gq[c], gv, T());
      if (a.gy != nullptr) {
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
          if (k >= n) break;
          float v[N];
#pragma unroll
          for (int e = 0; e < N; ++e) v[e] = gv[e] * wk[k];
          __stcs(gy + k * hv + i, pack<N>(v, T()));
        }
      }
      if (a.gw != nullptr) {
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
          if (k >= n) break;
          float v[N];
          unpack<N>(q[c][k], v, T());
#pragma unroll
          for (int e = 0; e < N; ++e) acc[k] = fmaf(gv[e], v[e], acc[k]);
        }
      }
    }
  }
  if (a.gw == nullptr) return;
  // Over the lanes: each step halves the slots that a lane adds up, until it has one, then the lanes of that slot.
  const int lane = threadIdx.x & 31;
  int o = 16, slot = 0;
#pragma unroll
  for (int have = SLOTS; have > 1; have /= 2, o /= 2) {
    const bool upper = lane & o;
#pragma unroll
    for (int k = 0; k < have / 2; ++k) {
      const float send = upper ? acc[k] : acc[k + have / 2], keep = upper ? acc[k + have / 2] : acc[k];
      acc[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
    if (upper) slot += have / 2;
  }
#pragma unroll
  for (; o > 0; o /= 2) acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
  if ((lane & (32 / SLOTS - 1)) == 0) s_part[threadIdx.x >> 5][slot] = acc[0];
  __syncthreads();
  if ((int)threadIdx.x < n) {
    float sum = 0.f;
    for (unsigned i = 0; i < blockDim.x / 32; ++i) sum += s_part[i][threadIdx.x];
    put(static_cast<TW*>(a.gw) + slot0 + threadIdx.x, sum * a.f);
  }
}

template <typename T, typename TW, int SLOTS, int N>
int launch_slots(Args a, cudaStream_t s) {
  constexpr int kCols = 16 / (N * (int)sizeof(T)) > 4 ? 4 : 16 / (N * (int)sizeof(T));
  const int64_t hv = a.H / N;
  a.groups = (unsigned)ceil_div(a.top_k, SLOTS);
  const int64_t steps = ceil_div(hv, (int64_t)kMaxThreads * kCols);   // as few threads as take the row in as many steps
  const unsigned threads = (unsigned)align_up(ceil_div(hv, steps * kCols), 32);
  sum_reduce_grad_kernel<T, TW, SLOTS, N, kCols><<<(unsigned)(a.M * a.groups), threads, 0, s>>>(a);
  XKB_CHECK_LAUNCH("sum_reduce_grad_kernel");
  return XKB_OK;
}

template <typename T, typename TW, int N>
int launch_width(const Args& a, cudaStream_t s) {
  // slots per block: all of them where the tokens fill the chip
  if (a.top_k > 4 && a.M * ceil_div(a.top_k, 8) >= 2 * 148) return launch_slots<T, TW, 8, N>(a, s);
  if (a.top_k > 2 && a.M * ceil_div(a.top_k, 4) >= 2 * 148) return launch_slots<T, TW, 4, N>(a, s);
  if (a.top_k > 1 && a.M * ceil_div(a.top_k, 2) >= 2 * 148) return launch_slots<T, TW, 2, N>(a, s);
  return launch_slots<T, TW, 1, N>(a, s);
}

template <typename T, typename TW>
int launch(const Args& a, cudaStream_t s) {
  XKB_REQUIRE(a.H < (1 << 28), "moe_sum_reduce_backward: H must be below 2^28");
  // the widest access whose boundaries all rows start on
  const uintptr_t bits = address_bits(a.go, a.y, a.gy) | (uintptr_t)(a.H * (int64_t)sizeof(T));
  XKB_REQUIRE(bits % sizeof(T) == 0 && address_bits(a.w, a.gw) % sizeof(TW) == 0, "moe_sum_reduce_backward: misaligned tensor");
  if (bits % 16 == 0) return launch_width<T, TW, 16 / sizeof(T)>(a, s);
  if (bits % 8 == 0) return launch_width<T, TW, 8 / sizeof(T)>(a, s);
  if constexpr (sizeof(T) == 2) {
    if (bits % 4 == 0) return launch_width<T, TW, 2>(a, s);
  }
  return launch_width<T, TW, 1>(a, s);
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
  XKB_REQUIRE(M <= 0x7fffffff / top_k, "moe_sum_reduce_backward: M * top_k must be below 2^31");
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
