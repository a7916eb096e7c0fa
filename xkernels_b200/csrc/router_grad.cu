// Balance loss with per-expert counts, and the gradient of the gating logits (sm_100a).
//
//   c_e = slots of expert e, P_e = 1/T sum_t p_te, loss = E sum_e c_e / (k T) P_e            p = softmax(x[t, :]), T tokens
//   dx = p (dp - sum_e p dp),  dp_te = sum of q_tj over the slots j of token t that chose e, + g_loss E c_e / (k T^2)
//   q_j = g_j for weights that are probabilities; (g_j - sum_i g_i w_i) / s for weights w_j = p_j / s, s = sum_j p_j
//
// A warp holds a row of up to 1024 experts in registers, in pieces of P neighbours (16 bytes where the row allows it).
//
// Loss: warps take rows in turn and keep the sum of every expert's probability in registers.  A block adds its warps up, a
// cluster of eight its blocks through distributed shared memory, and where there are several clusters a second kernel, which is already
// resident by then, adds theirs.  Floats are added in a fixed order, only counts by atomics: the same bits in every run.
//
// Gradient: bound by instructions, so nothing goes through shared memory.  sum_e p dp splits into sum_e p_e a_e and the slots' part,
// which is sum_j p_j g_j for raw weights and nothing for renormalised ones (they do not change along p); the row is written
// with the first part alone, and the lanes that hold a slot put the chosen experts' gradients in afterwards, from logits
// that they loaded themselves.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace xkb {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxExperts = 1024;
constexpr int kWarps = 8;   // of a block of the gradient kernel
constexpr float kLog2e = 1.44269504088896340736f;

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
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float exp_of(float x) {   // e^x to 2^-22 and the rounding of x log2(e); subnormal results are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * kLog2e));
  return r;
}

// A row in registers: the lane's t-th value belongs to expert (t / P * 32 + lane) * P + t % P.
template <typename T, int PER_LANE, int P>
struct Row {
  struct alignas(P * sizeof(T)) Piece { T x[P]; };
  static constexpr int kPieces = PER_LANE / P;
  static __device__ __forceinline__ int expert(int t, int lane) { return (t / P * 32 + lane) * P + t % P; }
  // logits, -inf behind the row
  struct Raw { Piece q[kPieces]; };
  static __device__ __forceinline__ Raw load(const T* row, int E, int lane) {
    Raw r;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const bool in = (c * 32 + lane) * P < E;
#pragma unroll
      for (int i = 0; i < P; ++i) r.q[c].x[i] = of_float<T>(-INFINITY);
      if (in) r.q[c] = reinterpret_cast<const Piece*>(row)[c * 32 + lane];
    }
    return r;
  }
  static __device__ __forceinline__ void values(const Raw& r, float (&x)[PER_LANE]) {
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) x[t] = to_float(r.q[t / P].x[t % P]);
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
  // logits -> e^(x - max), the maximum (0 for a row without a live logit, whose values become 0) and this lane's sum.  NaN and
  // +inf make the row NaN.
  static __device__ __forceinline__ float exponentials(float (&x)[PER_LANE], float& max) {
    float mx = x[0];
#pragma unroll
    for (int t = 1; t < PER_LANE; ++t) asm("max.NaN.f32 %0, %0, %1;" : "+f"(mx) : "f"(x[t]));
    mx = warp_max_nan(mx);
    max = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) {
      x[t] = exp_of(x[t] - max);
      sum += x[t];
    }
    return sum;
  }
};

// 1 / s to 1 ulp; 0 for 0 (a row or a choice without a live logit).  The sums here are 0 or 2^-126 to 2^10, or NaN.
__device__ __forceinline__ float inverse(float s) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(s));
  return s == 0.f ? 0.f : r;
}

// ---- loss ---------------------------------------------------------------------------------------------------------
struct LossArgs {
  const void* gating;
  const int32_t* ids;
  const uint8_t* mask;
  float* part_p;        // [parts, E]: of every cluster, where there are several
  int32_t* part_c;      // [parts, E]
  int32_t* part_t;      // [parts]
  float* loss;
  int32_t* counts;
  float* mean;
  int32_t* tokens;
  int64_t M;
  int E, k, parts;
};

constexpr int kCluster = 8;
constexpr int loss_warps(int per_lane) { return per_lane > 16 ? 8 : 16; }   // their sums take shared memory side by side

__device__ __forceinline__ void write_loss(const LossArgs& a, float sum, int T) {   // sum of counts x means
  *a.loss = T > 0 && a.k > 0 ? sum * (float)a.E / ((float)a.k * (float)T) : 0.f;
  *a.tokens = T;
}

template <typename T, int PER_LANE, int P>
__global__ void __launch_bounds__(32 * loss_warps(PER_LANE))
balance_kernel(LossArgs a) {
  using R = Row<T, PER_LANE, P>;
  constexpr int kPlaces = 32 * PER_LANE, kWarps = loss_warps(PER_LANE), kThreads = 32 * kWarps;
  __shared__ float s_sum[kWarps][kPlaces];
  __shared__ float s_total[kPlaces];
  __shared__ int s_count[kPlaces];
  __shared__ int s_tokens;
  __shared__ float s_term[4];
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = (int)cluster.block_rank();
  chain_trigger();   // the joining kernel may become resident
  for (int e = threadIdx.x; e < kPlaces; e += kThreads) s_count[e] = 0;
  if (threadIdx.x == 0) s_tokens = 0;
  __syncthreads();
  float acc[PER_LANE];
#pragma unroll
  for (int t = 0; t < PER_LANE; ++t) acc[t] = 0.f;
  int mine = 0;
  const int64_t step = (int64_t)gridDim.x * kWarps, m0 = (int64_t)blockIdx.x * kWarps + warp;
  const T* row = static_cast<const T*>(a.gating) + m0 * a.E;
  const int32_t* ids = a.ids + m0 * a.k + lane;
  auto requested = [&](int64_t m) -> bool { return m < a.M && (a.mask == nullptr || a.mask[m] != 0); };
  bool on = requested(m0);
  typename R::Raw next;
  int e = -1;
  if (on) {
    next = R::load(row, a.E, lane);
    if (lane < a.k) e = *ids;
  }
  for (int64_t m = m0; m < a.M; m += step) {
    const bool now = on;
    const int en = e;
    float x[PER_LANE];
    if (now) R::values(next, x);
    // the next row is on its way while this one is computed
    row += step * a.E;
    ids += step * a.k;
    on = requested(m + step);
    e = -1;
    if (on) {
      next = R::load(row, a.E, lane);
      if (lane < a.k) e = *ids;
    }
    if (!now) continue;
    ++mine;
    if (en >= 0 && en < a.E) atomicAdd(&s_count[en], 1);
    for (int j = lane + 32; j < a.k; j += 32) {
      const int o = a.ids[m * a.k + j];
      if (o >= 0 && o < a.E) atomicAdd(&s_count[o], 1);
    }
    float max;
    const float inv = inverse(warp_add(R::exponentials(x, max)));
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) acc[t] = fmaf(x[t], inv, acc[t]);
  }
  if (lane == 0 && mine != 0) atomicAdd(&s_tokens, mine);
#pragma unroll
  for (int t = 0; t < PER_LANE; ++t) s_sum[warp][R::expert(t, lane)] = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < a.E; i += kThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += s_sum[w][i];
    s_total[i] = sum;
  }
  cluster.sync();
  // every block joins its share of the experts: 128 at most
  const int each = (a.E + kCluster - 1) / kCluster, first = rank * each, n = max(0, min(each, a.E - first));
  const bool alone = gridDim.x == kCluster;
  const int64_t part = blockIdx.x / kCluster;
  if (warp < 4) {
    int tokens = lane < kCluster ? *cluster.map_shared_rank(&s_tokens, lane) : 0;
    float p = 0.f, term = 0.f;
    int c = 0;
    const int i = first + threadIdx.x;
    if ((int)threadIdx.x < n) {
#pragma unroll
      for (int b = 0; b < kCluster; ++b) {
        p += cluster.map_shared_rank(&s_total[0], b)[i];
        c += cluster.map_shared_rank(&s_count[0], b)[i];
      }
    }
    tokens = __reduce_add_sync(0xffffffffu, tokens);
    if (alone) {
      const float mean = tokens > 0 ? p / (float)tokens : 0.f;
      if ((int)threadIdx.x < n) {
        a.mean[i] = mean;
        a.counts[i] = c;
        term = (float)c * mean;
      }
      term = warp_add(term);
      if (lane == 0) s_term[warp] = term;
    } else if ((int)threadIdx.x < n) {
      a.part_p[part * a.E + i] = p;
      a.part_c[part * a.E + i] = c;
    }
    if (threadIdx.x == 0) mine = tokens;   // (used by thread 0 alone)
  }
  if (alone) {
    cluster.sync();   // the terms are there: four of eight blocks, one a lane
    if (rank == 0 && warp == 0) {
      const float term = warp_add(cluster.map_shared_rank(&s_term[0], lane >> 2)[lane & 3]);
      if (lane == 0) write_loss(a, term, mine);
    }
  } else if (rank == 0 && threadIdx.x == 0) {
    a.part_t[part] = mine;
  }
  cluster.sync();   // the others' shared memory is read until here
}

// Adds the clusters' rows up: thread (g, e) takes every G-th row of expert e.
__global__ void __launch_bounds__(1024)
balance_join_kernel(LossArgs a) {
  __shared__ float s_p[1024];
  __shared__ int s_c[1024];
  __shared__ float s_loss[32];
  __shared__ int s_tokens[2];
  const int E = a.E, G = 1024 / E, tid = threadIdx.x, g = tid / E, e = tid - g * E;
  chain_wait();
  // (written by the kernel that this one overlaps: loads from the L2)
  float p = 0.f;
  int c = 0;
  if (g < G) {
    const float* pp = a.part_p + g * E + e;
    const int32_t* pc = a.part_c + g * E + e;
    const int step = G * E;
#pragma unroll 10
    for (int b = g; b < a.parts; b += G, pp += step, pc += step) {
      p += __ldcg(pp);
      c += __ldcg(pc);
    }
  }
  int t = tid < a.parts ? __ldcg(a.part_t + tid) : 0;   // parts <= 64
  if (tid < 64) t = __reduce_add_sync(0xffffffffu, t);
  if (tid == 0 || tid == 32) s_tokens[tid >> 5] = t;
  s_p[tid] = p;
  s_c[tid] = c;
  __syncthreads();
  const int T = s_tokens[0] + s_tokens[1];
  float term = 0.f;
  if (tid < E) {
    for (int i = 1; i < G; ++i) { p += s_p[tid + i * E]; c += s_c[tid + i * E]; }
    const float mean = T > 0 ? p / (float)T : 0.f;
    a.mean[tid] = mean;
    a.counts[tid] = c;
    term = (float)c * mean;
  }
  term = warp_add(term);
  if ((tid & 31) == 0) s_loss[tid >> 5] = term;
  __syncthreads();
  if (tid < 32) {
    const float sum = warp_add(s_loss[tid]);
    if (tid == 0) write_loss(a, sum, T);
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
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool balance = a.counts != nullptr, weights = a.g_w != nullptr;
  if (balance) {
    const float n = a.tokens != nullptr ? (float)*a.tokens : (float)a.M;
    const float g = (a.g_loss != nullptr ? *a.g_loss : 1.f) * a.scale;
    const float f = n > 0.f && a.k > 0 ? g * (float)a.E / ((float)a.k * n) / n : 0.f;
    for (int e = threadIdx.x; e < 32 * PER_LANE; e += 32 * kWarps) s_share[e] = e < a.E ? f * (float)a.counts[e] : 0.f;
    __syncthreads();
  }
  float share[PER_LANE];   // of the lane's experts: the same for all rows
#pragma unroll
  for (int t = 0; t < PER_LANE; ++t) share[t] = balance ? s_share[R::expert(t, lane)] : 0.f;
  // lanes over which the first 32 slots' sums run
  int span = 1;
  while (span < a.k && span < 32) span *= 2;
  if (a.k > 32 || !a.renorm) span = 32;

  const int64_t step = (int64_t)gridDim.x * kWarps, m0 = (int64_t)blockIdx.x * kWarps + warp;
  const T* row = static_cast<const T*>(a.gating) + m0 * a.E;
  T* out = static_cast<T*>(a.out) + m0 * a.E;
  const int32_t* ids = a.ids + m0 * a.k;
  const float* g_w = a.g_w + m0 * a.k;
  for (int64_t m = m0; m < a.M; m += step, row += step * a.E, out += step * a.E, ids += step * a.k, g_w += step * a.k) {
    const typename R::Raw raw = R::load(row, a.E, lane);
    // slot `lane` of the first 32: expert (-1: none), gradient, logit
    int e = -1;
    float g = 0.f, xe = -INFINITY;
    if (weights && lane < a.k) {
      e = ids[lane];
      g = g_w[lane];
      if ((unsigned)e < (unsigned)a.E) {
        xe = to_float(row[e]);
      } else {
        e = -1;
        g = 0.f;
      }
    }
    const bool counted = balance && (a.mask == nullptr || a.mask[m] != 0);
    if (!counted) {   // a row that nothing comes back to (padding) has gradient 0, whatever its logits are
      bool any = g != 0.f;
      if (weights)
        for (int j = lane + 32; j < a.k; j += 32) any |= (unsigned)ids[j] < (unsigned)a.E && g_w[j] != 0.f;
      if (!__any_sync(0xffffffffu, any)) {
        float none[PER_LANE];
#pragma unroll
        for (int t = 0; t < PER_LANE; ++t) none[t] = 0.f;
        R::store(out, a.E, lane, none);
        continue;
      }
    }
    float x[PER_LANE], max;
    R::values(raw, x);
    float sum = R::exponentials(x, max);
    // of the slots: sum of exponentials and of exponential x gradient; the balance loss's sum_e e^x_e a_e
    const float ex = e >= 0 ? exp_of(xe - max) : 0.f;
    float sel = ex, dot = ex * g, even = 0.f;
    if (weights)
      for (int j = lane + 32; j < a.k; j += 32) {
        const int o = ids[j];
        if ((unsigned)o >= (unsigned)a.E) continue;
        const float eo = exp_of(to_float(row[o]) - max);
        sel += eo;
        dot = fmaf(eo, g_w[j], dot);
      }
    if (balance) {
#pragma unroll
      for (int t = 0; t < PER_LANE; ++t) even = fmaf(x[t], share[t], even);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (balance) even += __shfl_xor_sync(0xffffffffu, even, o);
      if (weights && o < span) {
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
        sel += __shfl_xor_sync(0xffffffffu, sel, o);
      }
    }
    const float inv = inverse(sum), s = (counted ? even * inv : 0.f) + (a.renorm ? 0.f : dot * inv);
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) x[t] = x[t] * inv * ((counted ? share[t] : 0.f) - s);
    R::store(out, a.E, lane, x);
    if (!weights) continue;
    // A slot's part is e^x scale (gradient - level); an expert that several slots chose takes all of them, in their order.
    const float scale = a.renorm ? inverse(sel) : inv, level = a.renorm ? dot * scale : 0.f;
    __syncwarp();   // the stores below come after the row's
    if (a.k <= 32) {
      float own = e >= 0 ? g - level : 0.f;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      if (__any_sync(0xffffffffu, e >= 0 && (same & (same - 1)) != 0)) {
        const float q = own;
        own = 0.f;
        for (int j = 0; j < a.k; ++j) {
          const float qj = __shfl_sync(0xffffffffu, q, j);
          if (same >> j & 1) own += qj;
        }
      }
      if (e >= 0) out[e] = of_float<T>(ex * (inv * ((counted ? s_share[e] : 0.f) - s) + scale * own));
    } else {
      for (int j = lane; j < a.k; j += 32) {
        const int o = ids[j];
        if ((unsigned)o >= (unsigned)a.E) continue;
        float own = 0.f;
        for (int i = 0; i < a.k; ++i)
          if (ids[i] == o) own += g_w[i] - level;
        out[o] = of_float<T>(exp_of(to_float(row[o]) - max) * (inv * ((counted ? s_share[o] : 0.f) - s) + scale * own));
      }
    }
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
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.parts * kCluster));
    cfg.blockDim = dim3(32 * loss_warps(PER_LANE));
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    XKB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, balance_kernel<T, PER_LANE, P>, a));
    XKB_CHECK_LAUNCH("balance_kernel");
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

// Clusters of the loss kernel: one, which needs no second kernel, up to eight rows a warp; two blocks per SM at most.
constexpr int64_t kMostParts = 2 * 148 / kCluster;
static_assert(kMostParts <= 64, "the joining kernel reads the clusters' tokens with 64 threads");
int64_t loss_parts(int64_t M) {
  const int64_t rows = kCluster * 16;
  if (M <= 8 * rows) return 1;
  const int64_t p = ceil_div(M, rows);
  return p > kMostParts ? kMostParts : p;
}

}  // namespace
}  // namespace xkb

extern "C" int64_t xkb_moe_balance_loss_workspace_bytes(int64_t M, int E) {
  using namespace xkb;
  if (M < 0 || E < 1 || E > kMaxExperts) return -1;
  const int64_t parts = loss_parts(M);
  return 2 * align_up(parts * E * 4, 256) + align_up(parts * 4, 256);
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
  const int64_t parts = loss_parts(M);
  Carver ws(workspace);
  LossArgs a{gating_output, topk_ids, token_mask, nullptr, nullptr, nullptr, loss, counts, mean_probs, tokens, M, E, top_k, (int)parts};
  a.part_p = ws.take<float>(parts * E);
  a.part_c = ws.take<int32_t>(parts * E);
  a.part_t = ws.take<int32_t>(parts);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(gating_output);
  int rc;
  switch (dtype) {
    case XKB_BF16: rc = with_shape<__nv_bfloat16>(E, bits, LaunchLoss<__nv_bfloat16>{a, s}); break;
    case XKB_F32: rc = with_shape<float>(E, bits, LaunchLoss<float>{a, s}); break;
    default: rc = with_shape<__half>(E, bits, LaunchLoss<__half>{a, s}); break;
  }
  if (rc != XKB_OK || parts == 1) return rc;
  XKB_CHECK_CUDA(launch_chained(balance_join_kernel, dim3(1), dim3(1024), 0, s, a));
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
