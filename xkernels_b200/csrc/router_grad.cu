// The gradient of the gating logits, from the routing weights and the balance loss (sm_100a).
//
//   dx = p (dp - sum_e p dp),  p = softmax(x),  dp_te = sum of q_tj over the slots j of token t that chose e, + a_e
//   q_j = g_j for weights that are probabilities; (g_j - sum_i g_i w_i) / s for weights w_j = p_j / s, s = sum_j p_j
//   a_e = g_loss E c_e / (k T^2)
//
// A warp has one row of up to 1024 experts in registers, two of up to 512 or four of up to 128, as the number of slots allows.  Bound by
// instructions and latency (183 instructions a row, 2.6 of 4 a cycle at a third of the warps), so no row goes through shared memory: sum_e p
// dp splits into sum_e p_e a_e and the slots' part, which is sum_j p_j g_j for raw weights and nothing for renormalised ones (they
// do not change along p); the row is written with the first part alone, and the lanes that hold a slot put the chosen experts'
// gradients in afterwards, from logits that they loaded themselves.
// Both gradients, bf16, top 8: 16384 x 256 6.1 us (2 of them launch), 65536 x 256 16.7 us (4.3 TB/s), 77 x 60 fp32 1.9 us.
#include "gating_dev.cuh"

namespace xkb {
namespace {

constexpr int kWarps = 8;
// Resident blocks, and the grid: a block that follows another has to ask for the counts again.  us, bf16, top 8, 3 / 4 blocks (which leave 85 and 64
// registers a thread): 65536 x 256 with both gradients 16.5 / 22.5, with the weights' alone 13.2 / 13.9, 65536 x 64 7.4 / 7.9, 16384 x 128 fp32
// 3.8 / 3.7; 16384 x 1024 with 1 / 2 36 / 21.
constexpr int blocks_per_sm(int per_lane) { return per_lane > 16 ? 2 : per_lane >= 8 ? 3 : 4; }
constexpr float kFewest = 0x1p-20f;   // of the chosen experts' exponentials, relative to the row's largest

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

template <typename T, int LANES, int PER_LANE, int P, bool BALANCE>
__global__ void __launch_bounds__(32 * kWarps, blocks_per_sm(PER_LANE))
router_grad_kernel(GateArgs a) {
  using R = Row<T, LANES, PER_LANE, P>;
  constexpr int kRows = 32 / LANES, kPlaces = LANES * PER_LANE;
  __shared__ float s_share[BALANCE ? kPlaces : 1];   // the balance loss's part of dp
  __shared__ unsigned char s_who[kWarps][kRows][kPlaces];   // the lane that chose an expert
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LANES, group = lane / LANES;
  const unsigned peers = LANES == 32 ? 0xffffffffu : ((1u << (LANES % 32)) - 1u) << (group * LANES);
  const bool weights = a.g_w != nullptr;
  // the group's rows are m, m + step ...; the warp goes on until its first group has none
  const int64_t step = (int64_t)gridDim.x * kWarps * kRows, w0 = ((int64_t)blockIdx.x * kWarps + warp) * kRows;
  const int64_t row_step = step * a.E, ids_step = step * a.k;
  int64_t m = w0 + group;
  const T* row = static_cast<const T*>(a.gating) + m * a.E;
  T* out = static_cast<T*>(a.out) + m * a.E;
  const int32_t* ids = a.ids + m * a.k;
  const float* g_w = a.g_w + m * a.k;
  // A row's slots are asked for one row ahead, and the first row's before the shares: their logits are then asked for with the row.
  // (The next row itself as well: 16384 x 256 7.3 us instead of 5.9, for the registers that it takes.)
  int e_next = -1;
  float g_next = 0.f;
  if (weights && m < a.M && sub < a.k) {
    e_next = ids[sub];
    g_next = g_w[sub];
  }
  float share[PER_LANE];   // of the lane's experts: the same for all rows
  if constexpr (BALANCE) {
    const float n = a.tokens != nullptr ? (float)*a.tokens : (float)a.M;
    const float g = (a.g_loss != nullptr ? *a.g_loss : 1.f) * a.scale;
    const float f = n > 0.f && a.k > 0 ? g * (float)a.E / ((float)a.k * n) / n : 0.f;
    for (int e = threadIdx.x; e < kPlaces; e += 32 * kWarps) s_share[e] = e < a.E ? f * (float)a.counts[e] : 0.f;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) share[t] = s_share[R::expert(t, sub)];
  }
  for (int64_t w = w0; w < a.M; w += step, m += step, row += row_step, out += row_step, ids += ids_step, g_w += ids_step) {
    const bool there = m < a.M, more_rows = m + step < a.M;
    const typename R::Raw raw = R::load(row, a.E, sub, there);
    // slot `sub` of the first LANES: expert (-1: none), gradient, logit
    int e = e_next;
    float g = g_next, xe = -INFINITY;
    if ((unsigned)e < (unsigned)a.E) {
      xe = to_float(row[e]);
    } else {
      e = -1;
      g = 0.f;
    }
    e_next = -1;
    g_next = 0.f;
    if (weights && more_rows && sub < a.k) {
      e_next = ids[ids_step + sub];
      g_next = g_w[ids_step + sub];
    }
    const bool counted = BALANCE && there && (a.mask == nullptr || a.mask[m] != 0);
    const bool more = LANES == 32 && weights && a.k > LANES;   // (parts of warps have a lane for each slot)
    bool live = counted || g != 0.f;
    if (more)
      for (int j = sub + LANES; j < a.k; j += LANES) live |= (unsigned)ids[j] < (unsigned)a.E && g_w[j] != 0.f;
    live = (__ballot_sync(0xffffffffu, live) & peers) != 0;

    float x[PER_LANE], max;
    float sum = R::exponentials(raw, x, max);
    // of the slots: sum of exponentials and of exponential x gradient; the balance loss's sum_e e^x_e a_e
    const float ex = e >= 0 ? exponential(xe, max) : 0.f;
    float sel = ex, dot = ex * g, even = 0.f;
    if (more)
      for (int j = sub + LANES; j < a.k; j += LANES) {
        const int o = ids[j];
        if ((unsigned)o >= (unsigned)a.E) continue;
        const float eo = exponential(to_float(row[o]), max);
        sel += eo;
        dot = fmaf(eo, g_w[j], dot);
      }
    if constexpr (BALANCE) {
      if constexpr (PER_LANE == 1) {
        even = x[0] * share[0];
      } else {
        Pair sums = pair_of(0.f);
#pragma unroll
        for (int t = 0; t < PER_LANE; t += 2) sums = fma2(pair_of(x[t], x[t + 1]), pair_of(share[t], share[t + 1]), sums);
        float e0, e1;
        split(sums, e0, e1);
        even = e0 + e1;
      }
    }
    lanes_add4<LANES>(sum, even, dot, sel);
    const float inv = inverse(sum), s = (counted ? even * inv : 0.f) + (a.renorm ? 0.f : dot * inv);
    // e^x (inv share - inv s)
    const float f = counted ? inv : 0.f, f0 = -inv * s;
    if (!live) {   // a row that nothing comes back to (padding) has gradient 0, whatever its logits are
#pragma unroll
      for (int t = 0; t < PER_LANE; ++t) x[t] = 0.f;
    } else if constexpr (PER_LANE == 1) {
      x[0] *= BALANCE ? fmaf(f, share[0], f0) : f0;
    } else {
#pragma unroll
      for (int t = 0; t < PER_LANE; t += 2) {
        const Pair d = BALANCE ? fma2(pair_of(f), pair_of(share[t], share[t + 1]), pair_of(f0)) : pair_of(f0);
        split(mul2(pair_of(x[t], x[t + 1]), d), x[t], x[t + 1]);
      }
    }
    if (there) R::store(out, a.E, sub, x);
    if (!weights) continue;
    // A slot's part is e^x scale (gradient - level); an expert that several slots chose takes all of them, in their order.
    const float scale = a.renorm ? inverse(sel) : inv, level = a.renorm ? dot * scale : 0.f;
    // (a row of dropped slots alone has none: 65536 x 256 with a tenth of such rows 16.9 us, 23.8 if they counted)
    const bool few = a.renorm && live && sel < kFewest && (more || e >= 0);
    __syncwarp();   // the stores below come after the row's
    if (!more) {
      float own = e >= 0 ? g - level : 0.f;
      // Of two lanes that chose the same expert, one reads the other's number.  (Asking every row for its equal lanes at once: 65536 x 64
      // 9.9 us instead of 7.2, the time goes with the number of different values.)
      if (e >= 0) s_who[warp][group][e] = (unsigned char)lane;
      __syncwarp();
      const bool seldom = __any_sync(0xffffffffu, (e >= 0 && s_who[warp][group][e] != lane) || few);
      if (seldom) {
        const unsigned same = __match_any_sync(0xffffffffu, e < 0 ? -1 : group << 16 | e);
        const float q = own;
        own = 0.f;
#pragma unroll 1
        for (int j = 0; j < 32; ++j) {
          const float qj = __shfl_sync(0xffffffffu, q, j);
          if (same >> j & 1) own += qj;
        }
      }
      if (e >= 0 && live && !few) out[e] = of_float<T>(ex * ((BALANCE ? fmaf(f, s_share[BALANCE ? e : 0], f0) : f0) + scale * own));
      if (!seldom) continue;
    } else if (live && !few) {
      for (int j = sub; j < a.k; j += LANES) {
        const int o = ids[j];
        if ((unsigned)o >= (unsigned)a.E) continue;
        float own = 0.f;
        for (int i = 0; i < a.k; ++i)
          if (ids[i] == o) own += g_w[i] - level;
        out[o] = of_float<T>(exponential(to_float(row[o]), max) * ((BALANCE ? fmaf(f, s_share[BALANCE ? o : 0], f0) : f0) + scale * own));
      }
    }
    if (!__any_sync(0xffffffffu, few)) continue;
    // Renormalised weights depend on the chosen logits alone.  Where these have less than kFewest of the row's largest exponential (a choice
    // under a bias or within a group), theirs are taken relative to the largest of themselves: relative to the row's they
    // could all be 0, or have a sum whose inverse overflows.  (65536 x 256, top 8, all rows such ones: 40 us instead of 17.)
    float top = -INFINITY;
#pragma unroll 1
    for (int j = sub; few && j < a.k; j += LANES)
      if ((unsigned)ids[j] < (unsigned)a.E) top = fmaxf(top, to_float(row[ids[j]]));   // (no NaN: that row's sum is NaN)
    top = lanes_max_nan<LANES>(top);
    if (top == -INFINITY) top = 0.f;   // no chosen logit is live: their weights are 0
    sel = dot = 0.f;
#pragma unroll 1
    for (int j = sub; few && j < a.k; j += LANES) {
      if ((unsigned)ids[j] >= (unsigned)a.E) continue;
      const float eo = exponential(to_float(row[ids[j]]), top);
      sel += eo;
      dot = fmaf(eo, g_w[j], dot);
    }
    const float own_scale = inverse(lanes_add<LANES>(sel)), own_level = lanes_add<LANES>(dot) * own_scale;
#pragma unroll 1
    for (int j = sub; few && j < a.k; j += LANES) {
      const int o = ids[j];
      if ((unsigned)o >= (unsigned)a.E) continue;
      float own = 0.f;
#pragma unroll 1
      for (int i = 0; i < a.k; ++i)
        if (ids[i] == o) own += g_w[i] - own_level;
      const float xo = to_float(row[o]), part = exponential(xo, max) * (BALANCE ? fmaf(f, s_share[BALANCE ? o : 0], f0) : f0);
      out[o] = of_float<T>(fmaf(exponential(xo, top), own_scale * own, part));   // (part is NaN in a row with +inf)
    }
  }
}

template <typename T> struct LaunchGrad {
  const GateArgs& a;
  cudaStream_t s;
  template <int LANES, int PER_LANE, int P> int operator()() const {
    const int64_t want = ceil_div(a.M, (int64_t)kWarps * 32 / LANES), most = 148 * blocks_per_sm(PER_LANE);
    const unsigned blocks = (unsigned)(want < most ? want : most);
    (a.counts != nullptr ? router_grad_kernel<T, LANES, PER_LANE, P, true>
                         : router_grad_kernel<T, LANES, PER_LANE, P, false>)<<<blocks, 32 * kWarps, 0, s>>>(a);
    XKB_CHECK_LAUNCH("router_grad_kernel");
    return XKB_OK;
  }
};

}  // namespace
}  // namespace xkb

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
  XKB_REQUIRE(address_bits(gating_output, grad_gating) % (dtype == XKB_F32 ? 4 : 2) == 0 &&
                  address_bits(topk_ids, grad_weights, counts, tokens, grad_loss) % 4 == 0,
              "moe_router_backward: a misaligned tensor");
  const GateArgs a{gating_output, topk_ids, top_k == 0 ? nullptr : grad_weights, renormalize, counts, tokens, grad_loss, loss_scale,
                   token_mask, grad_gating, M, E, top_k};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uintptr_t bits = address_bits(gating_output, grad_gating);
  switch (dtype) {
    case XKB_BF16: return with_shape<__nv_bfloat16>(E, top_k, bits, LaunchGrad<__nv_bfloat16>{a, s});
    case XKB_F32: return with_shape<float>(E, top_k, bits, LaunchGrad<float>{a, s});
    default: return with_shape<__half>(E, top_k, bits, LaunchGrad<__half>{a, s});
  }
}
