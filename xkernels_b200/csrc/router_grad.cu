// Balance loss with per-expert counts, and the gradient of the gating logits (sm_100a).
//
//   c_e = slots of expert e, P_e = 1/T sum_t p_te, loss = E sum_e c_e / (k T) P_e            p = softmax(x[t, :]), T tokens
//   dx = p (dp - sum_e p dp),  dp_te = sum of q_tj over the slots j of token t that chose e, + g_loss E c_e / (k T^2)
//   q_j = g_j for weights that are probabilities; (g_j - sum_i g_i w_i) / s for weights w_j = p_j / s, s = sum_j p_j
//
// A warp holds a row of up to 1024 experts in registers, in pieces of P neighbours (16 bytes where the row allows it).
// Loss: warps take rows in turn and keep the sum of every expert's probability in registers; a block adds its warps up and
// leaves one row of partial sums, which a second kernel adds in a fixed order: the result is the same in every run.
#include <cuda_fp16.h>

#include "common.cuh"

namespace xkb {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kWarps = 8;

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T of_float(float v);
template <> __device__ __forceinline__ float of_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 of_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half of_float<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(0xffffffffu, v, o);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(w));
  }
  return v;
}

// A row in registers: the lane's t-th value belongs to expert (t / P * 32 + lane) * P + t % P.
template <typename T, int PER_LANE, int P>
struct Row {
  struct alignas(P * sizeof(T)) Piece { T x[P]; };
  static constexpr int kPieces = PER_LANE / P;
  static __device__ __forceinline__ int expert(int t, int lane) { return (t / P * 32 + lane) * P + t % P; }
  // logits, -inf behind the row
  static __device__ __forceinline__ void load(const T* row, int E, int lane, float (&x)[PER_LANE]) {
    Piece q[kPieces];
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const bool in = (c * 32 + lane) * P < E;
#pragma unroll
      for (int i = 0; i < P; ++i) q[c].x[i] = of_float<T>(-INFINITY);
      if (in) q[c] = reinterpret_cast<const Piece*>(row)[c * 32 + lane];
    }
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) x[t] = to_float(q[t / P].x[t % P]);
  }
  static __device__ __forceinline__ void store(T* row, int E, int lane, const float (&x)[PER_LANE]) {
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      Piece q;
#pragma unroll
      for (int i = 0; i < P; ++i) q.x[i] = of_float<T>(x[c * P + i]);
      if ((c * 32 + lane) * P < E) reinterpret_cast<Piece*>(row)[c * 32 + lane] = q;
    }
  }
  // logits -> probabilities; a row without a live logit has none: 0 everywhere.  NaN and +inf make the row NaN.
  static __device__ __forceinline__ void softmax(float (&x)[PER_LANE]) {
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) asm("max.NaN.f32 %0, %0, %1;" : "+f"(mx) : "f"(x[t]));
    mx = warp_max_nan(mx);
    const bool dead = mx == -INFINITY;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) {
      x[t] = expf(x[t] - (dead ? 0.f : mx));
      sum += x[t];
    }
    sum = warp_add(sum);
    const float inv = dead ? 0.f : 1.f / sum;
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) x[t] *= inv;
  }
};

// ---- loss ---------------------------------------------------------------------------------------------------------
struct LossArgs {
  const void* gating;
  const int32_t* ids;
  const uint8_t* mask;
  float* part_p;        // [blocks, E]
  int32_t* part_c;      // [blocks, E]
  int32_t* part_t;      // [blocks]
  float* loss;
  int32_t* counts;
  float* mean;
  int32_t* tokens;
  int64_t M;
  int E, k, blocks;
};

template <typename T, int PER_LANE, int P>
__global__ void __launch_bounds__(32 * kWarps)
balance_partial_kernel(LossArgs a) {
  using R = Row<T, PER_LANE, P>;
  __shared__ float s_sum[32 * PER_LANE];
  __shared__ int s_count[32 * PER_LANE];
  __shared__ int s_tokens;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < 32 * PER_LANE; e += 32 * kWarps) s_count[e] = 0;
  if (threadIdx.x == 0) s_tokens = 0;
  __syncthreads();
  float acc[PER_LANE];
#pragma unroll
  for (int t = 0; t < PER_LANE; ++t) acc[t] = 0.f;
  int mine = 0;
  for (int64_t m = (int64_t)blockIdx.x * kWarps + warp; m < a.M; m += (int64_t)a.blocks * kWarps) {
    if (a.mask != nullptr && a.mask[m] == 0) continue;
    ++mine;
    float x[PER_LANE];
    R::load(static_cast<const T*>(a.gating) + m * a.E, a.E, lane, x);
    for (int j = lane; j < a.k; j += 32) {
      const int e = a.ids[m * a.k + j];
      if (e >= 0 && e < a.E) atomicAdd(&s_count[e], 1);
    }
    R::softmax(x);
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) acc[t] += x[t];
  }
  if (lane == 0) atomicAdd(&s_tokens, mine);
  // one warp after the other, so that the order is fixed
  for (int w = 0; w < kWarps; ++w) {
    if (warp == w) {
#pragma unroll
      for (int t = 0; t < PER_LANE; ++t) {
        const int e = R::expert(t, lane);
        s_sum[e] = w == 0 ? acc[t] : s_sum[e] + acc[t];
      }
    }
    __syncthreads();
  }
  for (int e = threadIdx.x; e < a.E; e += 32 * kWarps) {
    a.part_p[(int64_t)blockIdx.x * a.E + e] = s_sum[e];
    a.part_c[(int64_t)blockIdx.x * a.E + e] = s_count[e];
  }
  if (threadIdx.x == 0) a.part_t[blockIdx.x] = s_tokens;
}

// Adds the partial rows up: thread (g, e) takes every G-th block of expert e.
__global__ void __launch_bounds__(1024)
balance_join_kernel(LossArgs a) {
  __shared__ float s_p[1024];
  __shared__ int s_c[1024];
  __shared__ double s_loss[32];
  __shared__ int s_tokens;
  const int E = a.E, G = 1024 / E, tid = threadIdx.x, g = tid / E, e = tid - g * E;
  if (tid == 0) s_tokens = 0;
  __syncthreads();
  int t = 0;
  for (int b = tid; b < a.blocks; b += 1024) t += a.part_t[b];
  if (t != 0) atomicAdd(&s_tokens, t);
  float p = 0.f;
  int c = 0;
  if (g < G) {
    for (int b = g; b < a.blocks; b += G) {
      p += a.part_p[(int64_t)b * E + e];
      c += a.part_c[(int64_t)b * E + e];
    }
  }
  s_p[tid] = p;
  s_c[tid] = c;
  __syncthreads();
  const int T = s_tokens;
  double term = 0.0;
  if (tid < E) {
    for (int i = 1; i < G; ++i) { p += s_p[tid + i * E]; c += s_c[tid + i * E]; }
    const float mean = T > 0 ? p / (float)T : 0.f;
    a.mean[tid] = mean;
    a.counts[tid] = c;
    term = (double)c * (double)mean;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) term += __shfl_xor_sync(0xffffffffu, term, o);
  if ((tid & 31) == 0) s_loss[tid >> 5] = term;
  __syncthreads();
  if (tid == 0) {
    double sum = 0.0;
    for (int i = 0; i < 32; ++i) sum += s_loss[i];
    *a.loss = T > 0 && a.k > 0 ? (float)(sum * E / ((double)a.k * T)) : 0.f;
    *a.tokens = T;
  }
}

// ---- gradient -----------------------------------------------------------------------------------------------------
struct GateArgs {
  const void* gating;
  const int32_t* ids;
  const float* g_w;
  int renorm;
  const int32_t* counts;
  const int32_t* tokens;
  const float* g_loss;
  float scale;
  const uint8_t* mask;
  void* out;
  int64_t M;
  int E, k;
};

template <typename T, int PER_LANE, int P>
__global__ void __launch_bounds__(32 * kWarps)
router_grad_kernel(GateArgs a) {
  using R = Row<T, PER_LANE, P>;
  __shared__ float s_share[32 * PER_LANE];          // the balance loss's part of dp
  __shared__ float s_row[kWarps][32 * PER_LANE];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* row = s_row[warp];
  if (a.counts != nullptr) {
    const float n = a.tokens != nullptr ? (float)*a.tokens : (float)a.M;
    const float g = (a.g_loss != nullptr ? *a.g_loss : 1.f) * a.scale;
    const float f = n > 0.f && a.k > 0 ? g * (float)a.E / ((float)a.k * n) / n : 0.f;
    for (int e = threadIdx.x; e < 32 * PER_LANE; e += 32 * kWarps) s_share[e] = e < a.E ? f * (float)a.counts[e] : 0.f;
  }
  __syncthreads();
  for (int64_t m = (int64_t)blockIdx.x * kWarps + warp; m < a.M; m += (int64_t)gridDim.x * kWarps) {
    float p[PER_LANE], dp[PER_LANE];
    R::load(static_cast<const T*>(a.gating) + m * a.E, a.E, lane, p);
    const bool counted = a.counts != nullptr && (a.mask == nullptr || a.mask[m] != 0);
    if (!counted) {   // a row that nothing comes back to (padding) has gradient 0, whatever its logits are
      bool any = false;
      for (int j = lane; j < a.k && a.g_w != nullptr; j += 32) any |= a.g_w[m * a.k + j] != 0.f;
      if (!__any_sync(0xffffffffu, any)) {
#pragma unroll
        for (int t = 0; t < PER_LANE; ++t) p[t] = 0.f;
        R::store(static_cast<T*>(a.out) + m * a.E, a.E, lane, p);
        continue;
      }
    }
    R::softmax(p);
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) dp[t] = counted ? s_share[R::expert(t, lane)] : 0.f;
    if (a.g_w != nullptr) {
      __syncwarp();
#pragma unroll
      for (int t = 0; t < PER_LANE; ++t) row[R::expert(t, lane)] = p[t];
      __syncwarp();
      float sel = 0.f, dot = 0.f;   // of the slots: sum of probabilities, sum of gradient x probability
      for (int j = lane; j < a.k; j += 32) {
        const int e = a.ids[m * a.k + j];
        if (e < 0 || e >= a.E) continue;
        sel += row[e];
        dot = fmaf(a.g_w[m * a.k + j], row[e], dot);
      }
      sel = warp_add(sel);
      dot = warp_add(dot);
      __syncwarp();
#pragma unroll
      for (int t = 0; t < PER_LANE; ++t) row[R::expert(t, lane)] = dp[t];
      __syncwarp();
      for (int j0 = 0; j0 < a.k; j0 += 32) {
        const int j = j0 + lane;
        int e = -1;
        float q = 0.f;
        if (j < a.k) {
          e = a.ids[m * a.k + j];
          if (e < 0 || e >= a.E) e = -1;
          else q = a.g_w[m * a.k + j];
        }
        if (a.renorm) q = sel == 0.f ? 0.f : (q - dot / sel) / sel;
        // an expert that several slots chose takes them one after the other
        const unsigned same = __match_any_sync(0xffffffffu, e);
        const int before = __popc(same & ((1u << lane) - 1u));
        const int rounds = __reduce_max_sync(0xffffffffu, e >= 0 ? before : 0);
        for (int i = 0; i <= rounds; ++i) {
          if (e >= 0 && before == i) row[e] += q;
          __syncwarp();
        }
      }
#pragma unroll
      for (int t = 0; t < PER_LANE; ++t) dp[t] = row[R::expert(t, lane)];
    }
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) s = fmaf(p[t], dp[t], s);
    s = warp_add(s);
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) p[t] *= dp[t] - s;
    R::store(static_cast<T*>(a.out) + m * a.E, a.E, lane, p);
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------
// Calls f<PER_LANE, P>() for the fewest experts per lane that cover the row and the widest piece that the row and
// its address allow.
template <typename T, int PER_LANE, typename F>
int with_piece(int E, uintptr_t bits, F f) {   // bits: the addresses of all rows, or'ed
  constexpr int kMost = PER_LANE < (int)(16 / sizeof(T)) ? PER_LANE : (int)(16 / sizeof(T));
  auto fits = [&](int P) { return E % P == 0 && bits % (P * sizeof(T)) == 0; };
  if constexpr (kMost >= 8) if (fits(8)) return f.template operator()<PER_LANE, 8>();
  if constexpr (kMost >= 4) if (fits(4)) return f.template operator()<PER_LANE, 4>();
  if constexpr (kMost >= 2) if (fits(2)) return f.template operator()<PER_LANE, 2>();
  return f.template operator()<PER_LANE, 1>();
}
template <typename T, typename F>
int with_shape(int E, uintptr_t bits, F f) {
  const int per_lane = (E + 31) / 32;
  if (per_lane <= 1) return with_piece<T, 1>(E, bits, f);
  if (per_lane <= 2) return with_piece<T, 2>(E, bits, f);
  if (per_lane <= 4) return with_piece<T, 4>(E, bits, f);
  if (per_lane <= 8) return with_piece<T, 8>(E, bits, f);
  if (per_lane <= 16) return with_piece<T, 16>(E, bits, f);
  return with_piece<T, 32>(E, bits, f);
}

template <typename T> struct LaunchLoss {
  const LossArgs& a;
  cudaStream_t s;
  template <int PER_LANE, int P> int operator()() const {
    balance_partial_kernel<T, PER_LANE, P><<<a.blocks, 32 * kWarps, 0, s>>>(a);
    XKB_CHECK_LAUNCH("balance_partial_kernel");
    return XKB_OK;
  }
};
template <typename T> struct LaunchGrad {
  const GateArgs& a;
  unsigned blocks;
  cudaStream_t s;
  template <int PER_LANE, int P> int operator()() const {
    router_grad_kernel<T, PER_LANE, P><<<blocks, 32 * kWarps, 0, s>>>(a);
    XKB_CHECK_LAUNCH("router_grad_kernel");
    return XKB_OK;
  }
};

constexpr int64_t kMostBlocks = 2 * 148;
int64_t loss_blocks(int64_t M) {
  const int64_t b = ceil_div(M, (int64_t)kWarps);
  return b < 1 ? 1 : b > kMostBlocks ? kMostBlocks : b;
}

}  // namespace
}  // namespace xkb

extern "C" int64_t xkb_moe_balance_loss_workspace_bytes(int64_t M, int E) {
  using namespace xkb;
  if (M < 0 || E < 1 || E > kMaxExperts) return -1;
  const int64_t blocks = loss_blocks(M);
  return 2 * align_up(blocks * E * 4, 256) + align_up(blocks * 4, 256);
}

extern "C" int xkb_moe_balance_loss(const void* gating_output, int dtype, const int32_t* topk_ids, const uint8_t* token_mask,
                                    float* loss, int32_t* counts, float* mean_probs, int32_t* tokens, int64_t M, int E,
                                    int top_k, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace xkb;
  XKB_REQUIRE(M >= 0 && E >= 1 && E <= kMaxExperts, "moe_balance_loss: bad shape M=%lld E=%d (at most %d experts)", (long long)M, E, kMaxExperts);
  XKB_REQUIRE(top_k >= 0 && M * top_k <= 0x7fffffff, "moe_balance_loss: M * top_k must fit 31 bits (M=%lld, top_k=%d)", (long long)M, top_k);
  XKB_REQUIRE(dtype == XKB_BF16 || dtype == XKB_F32 || dtype == XKB_F16, "moe_balance_loss: unsupported logits dtype code %d", dtype);
  XKB_REQUIRE(loss && counts && mean_probs && tokens && (M == 0 || gating_output) && (M * top_k == 0 || topk_ids),
              "moe_balance_loss: null pointer");
  if (workspace == nullptr || workspace_bytes < xkb_moe_balance_loss_workspace_bytes(M, E))
    return fail(XKB_ERR_WORKSPACE, "moe_balance_loss: the workspace needs %lld bytes (got %lld)",
                (long long)xkb_moe_balance_loss_workspace_bytes(M, E), (long long)(workspace ? workspace_bytes : 0));
  XKB_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "moe_balance_loss: misaligned workspace");
  const int64_t blocks = loss_blocks(M);
  Carver ws(workspace);
  LossArgs a{gating_output, topk_ids, token_mask, nullptr, nullptr, nullptr, loss, counts, mean_probs, tokens, M, E, top_k, (int)blocks};
  a.part_p = ws.take<float>(blocks * E);
  a.part_c = ws.take<int32_t>(blocks * E);
  a.part_t = ws.take<int32_t>(blocks);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(gating_output);
  int rc;
  switch (dtype) {
    case XKB_BF16: rc = with_shape<__nv_bfloat16>(E, bits, LaunchLoss<__nv_bfloat16>{a, s}); break;
    case XKB_F32: rc = with_shape<float>(E, bits, LaunchLoss<float>{a, s}); break;
    default: rc = with_shape<__half>(E, bits, LaunchLoss<__half>{a, s}); break;
  }
  if (rc != XKB_OK) return rc;
  balance_join_kernel<<<1, 1024, 0, s>>>(a);
  XKB_CHECK_LAUNCH("balance_join_kernel");
  return XKB_OK;
}

extern "C" int xkb_moe_router_backward(const void* gating_output, int dtype, const int32_t* topk_ids, const float* grad_weights,
                                       int renormalize, const int32_t* counts, const int32_t* tokens, const float* grad_loss,
                                       float loss_scale, const uint8_t* token_mask, void* grad_gating, int64_t M, int E,
                                       int top_k, void* stream) {
  using namespace xkb;
  XKB_REQUIRE(M >= 0 && E >= 1 && E <= kMaxExperts, "moe_router_backward: bad shape M=%lld E=%d (at most %d experts)", (long long)M, E, kMaxExperts);
  XKB_REQUIRE(top_k >= 0, "moe_router_backward: negative top_k");
  XKB_REQUIRE(dtype == XKB_BF16 || dtype == XKB_F32 || dtype == XKB_F16, "moe_router_backward: unsupported logits dtype code %d", dtype);
  if (M == 0) return XKB_OK;
  XKB_REQUIRE(gating_output && grad_gating && (grad_weights == nullptr || top_k == 0 || topk_ids), "moe_router_backward: null pointer");
  const GateArgs a{gating_output, topk_ids, top_k == 0 ? nullptr : grad_weights, renormalize, counts, tokens, grad_loss, loss_scale,
                   token_mask, grad_gating, M, E, top_k};
  const int64_t want = ceil_div(M, (int64_t)kWarps), most = 148 * 8;
  const unsigned blocks = (unsigned)(want < most ? want : most);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(gating_output) | reinterpret_cast<uintptr_t>(grad_gating);
  switch (dtype) {
    case XKB_BF16: return with_shape<__nv_bfloat16>(E, bits, LaunchGrad<__nv_bfloat16>{a, blocks, s});
    case XKB_F32: return with_shape<float>(E, bits, LaunchGrad<float>{a, blocks, s});
    default: return with_shape<__half>(E, bits, LaunchGrad<__half>{a, blocks, s});
  }
}
