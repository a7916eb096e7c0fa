// Balance loss with per-expert counts (sm_100a).
//
//   c_e = slots of expert e, P_e = 1/T sum_t p_te, loss = E sum_e c_e / (k T) P_e            p = softmax(x[t, :]), T tokens
//
// A warp has one row of up to 1024 experts in registers, two of up to 512 or four of up to 128.  Warps take rows in turn, the next one on its way
// while one is computed, and keep the sum of every expert's probability in registers; a block adds its warps up.  A few rows
// are one block, or one cluster of eight, joined through distributed shared memory, and one launch; more are a block per SM that leaves a row
// of partial sums each, which a second kernel of eight blocks adds up.  It is launched early, but its blocks (46 registers, 1024
// threads) do not fit an SM beside one of the first kernel's (63 to 128 registers, 512 threads): where there is one on every SM
// they start as those end.  Floats are added in a fixed order, only counts by atomics: the same bits in every run.
// 16384 x 256 bf16 8.8 us: 2.2 of launch, 2.5 for the second kernel, else latency: a lane group has one row's chain of maximum, exponentials, sum and
// reciprocal, and 1.7 of 4 instructions a cycle are issued (65536 rows 16.5 us, 2.2 TB/s).  333 x 48 fp32 4.3 us: launch, the
// cluster's barriers, the chain of sums.
#include <cooperative_groups.h>

#include "gating_dev.cuh"

namespace xkb {
namespace {

namespace cg = cooperative_groups;

struct LossArgs {
  const void* gating;
  const int32_t* ids;
  const uint8_t* mask;
  float* part_p;        // [parts, E]: of every block, where there are more than a cluster's
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
// Warps of a block: their sums take shared memory side by side.  us, 8 / 16 / 32 warps: 333 x 48 4.4 / 4.4 / 5.6, 200 x 64 3.9 / 4.4 / 4.7, 16384 x 256
// 9.8 / 8.7 / 9.8 (64 registers a thread), 65536 x 256 23 / 16.4 / 16.0, 65536 x 64 12.2 / 9.4 / 8.9.
constexpr int loss_warps(int experts) { return experts > 512 ? 8 : 16; }

__device__ __forceinline__ void write_loss(const LossArgs& a, float sum, int T) {   // sum of counts x means
  *a.loss = T > 0 && a.k > 0 ? sum * (float)a.E / ((float)a.k * (float)T) : 0.f;
  *a.tokens = T;
}

// parts == 0: one cluster, which finishes.  Else blocks of their own, which leave a row of partial sums.
template <typename T, int LANES, int PER_LANE, int P>
__global__ void __launch_bounds__(32 * loss_warps(LANES * PER_LANE), 1)
balance_kernel(LossArgs a) {
  using R = Row<T, LANES, PER_LANE, P>;
  constexpr int kPlaces = LANES * PER_LANE, kWarps = loss_warps(kPlaces), kThreads = 32 * kWarps, kRows = 32 / LANES;
  __shared__ float s_sum[kWarps][kPlaces];
  __shared__ float s_total[kPlaces];
  __shared__ int s_count[kPlaces];
  __shared__ int s_tokens;
  __shared__ float s_term[kCluster * kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LANES;
  chain_trigger();   // the joining kernel may start where there is room for it
  float acc[PER_LANE];
#pragma unroll
  for (int t = 0; t < PER_LANE; ++t) acc[t] = 0.f;
  int mine = 0;
  // the group's rows are m, m + step ...; the warp goes on until its first group has none
  const int64_t step = (int64_t)gridDim.x * kWarps * kRows, w0 = ((int64_t)blockIdx.x * kWarps + warp) * kRows;
  int64_t m = w0 + lane / LANES;
  const int64_t row_step = step * a.E, ids_step = step * a.k;
  const T* row = static_cast<const T*>(a.gating) + m * a.E;
  const int32_t* ids = a.ids + m * a.k;
  bool on = m < a.M && (a.mask == nullptr || a.mask[m] != 0);
  typename R::Raw next = R::load(row, a.E, sub, on);
  int e = on && sub < a.k ? ids[sub] : -1;
  for (int i = threadIdx.x; i < kPlaces; i += kThreads) s_count[i] = 0;
  if (threadIdx.x == 0) s_tokens = 0;
  __syncthreads();
  for (int64_t w = w0; w < a.M; w += step) {
    // the next row is on its way while this one is computed
    const bool now = on;
    const int en = e;
    const int32_t* ids_now = ids;
    const typename R::Raw raw = next;
    m += step;
    row += row_step;
    ids += ids_step;
    on = m < a.M && (a.mask == nullptr || a.mask[m] != 0);
    next = R::load(row, a.E, sub, on);
    e = on && sub < a.k ? ids[sub] : -1;
    mine += now;
    if ((unsigned)en < (unsigned)a.E) atomicAdd(&s_count[en], 1);
    if (now)
      for (int j = sub + LANES; j < a.k; j += LANES) {
        const int o = ids_now[j];
        if ((unsigned)o < (unsigned)a.E) atomicAdd(&s_count[o], 1);
      }
    // (a group without a row holds -inf and adds 0)
    float x[PER_LANE], max;
    const float inv = inverse(lanes_add<LANES>(R::exponentials(raw, x, max)));
#pragma unroll
    for (int t = 0; t < PER_LANE; ++t) acc[t] = fmaf(x[t], inv, acc[t]);
  }
  mine = __reduce_add_sync(0xffffffffu, sub == 0 ? mine : 0);
  if (lane == 0 && mine != 0) atomicAdd(&s_tokens, mine);
#pragma unroll
  for (int t = 0; t < PER_LANE; ++t) {
#pragma unroll
    for (int o = LANES; o < 32; o *= 2) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);   // over the warp's rows
    if (lane < LANES) s_sum[warp][R::expert(t, sub)] = acc[t];
  }
  __syncthreads();
  const bool alone = a.parts == 0;
  for (int i = threadIdx.x; i < a.E; i += kThreads) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) sum += s_sum[v][i];
    if (alone) {
      s_total[i] = sum;
    } else {
      a.part_p[(int64_t)blockIdx.x * a.E + i] = sum;
      a.part_c[(int64_t)blockIdx.x * a.E + i] = s_count[i];
    }
  }
  if (!alone) {
    if (threadIdx.x == 0) a.part_t[blockIdx.x] = s_tokens;
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  auto sync = [&] { if (C > 1) cluster.sync(); else __syncthreads(); };
  sync();
  // every block joins its share of the experts
  const int each = (a.E + C - 1) / C, first = rank * each, end = min(first + each, a.E);
  const int tokens = __reduce_add_sync(0xffffffffu, lane < C ? *cluster.map_shared_rank(&s_tokens, lane) : 0);
  float term = 0.f;
  for (int i = first + (int)threadIdx.x; i < end; i += kThreads) {
    float p = 0.f;
    int c = 0;
#pragma unroll 8
    for (int b = 0; b < C; ++b) {
      p += cluster.map_shared_rank(&s_total[0], b)[i];
      c += cluster.map_shared_rank(&s_count[0], b)[i];
    }
    const float mean = tokens > 0 ? p / (float)tokens : 0.f;
    a.mean[i] = mean;
    a.counts[i] = c;
    term += (float)c * mean;
  }
  term = warp_add(term);
  if (lane == 0) cluster.map_shared_rank(&s_term[0], 0)[rank * kWarps + warp] = term;
  sync();
  if (rank == 0 && warp == 0) {
    float sum = 0.f;
    for (int i = lane; i < C * kWarps; i += 32) sum += s_term[i];
    sum = warp_add(sum);
    if (lane == 0) write_loss(a, sum, tokens);
  }
}

// Adds the blocks' rows up: eight blocks, each a share of the experts.  A warp's lanes load neighbouring experts of one row, thread
// (g, i) every G-th row; then a warp adds the G sums of an expert.
__global__ void __launch_bounds__(1024)
balance_join_kernel(LossArgs a) {
  __shared__ float s_p[1024 + 32];      // [G][width + 1]
  __shared__ int s_c[1024 + 32];
  __shared__ int s_tokens[32];
  __shared__ float s_term[kCluster * 32];
  cg::cluster_group cluster = cg::this_cluster();
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  const int rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (a.E + kCluster - 1) / kCluster, first = rank * each, n = max(0, min(each, a.E - first));   // each <= 128
  const int width = each <= 32 ? 32 : each <= 64 ? 64 : 128, G = 1024 / width, g = tid / width, i = tid % width;
  chain_wait();
  // (written by the kernel that this one overlaps: loads from the L2)
  float p = 0.f;
  int c = 0;
  if (i < n) {
    const float* pp = a.part_p + (int64_t)g * a.E + first + i;
    const int32_t* pc = a.part_c + (int64_t)g * a.E + first + i;
    const int64_t step = (int64_t)G * a.E;
#pragma unroll 5
    for (int b = g; b < a.parts; b += G, pp += step, pc += step) {
      p += __ldcg(pp);
      c += __ldcg(pc);
    }
  }
  int t = tid < a.parts ? __ldcg(a.part_t + tid) : 0;   // parts <= 148
  t = __reduce_add_sync(0xffffffffu, t);
  if (lane == 0) s_tokens[warp] = t;
  s_p[g * (width + 1) + i] = p;
  s_c[g * (width + 1) + i] = c;
  __syncthreads();
  const int T = __reduce_add_sync(0xffffffffu, s_tokens[lane]);
  float term = 0.f;
  for (int e = warp; e < n; e += 32) {
    p = warp_add(lane < G ? s_p[lane * (width + 1) + e] : 0.f);
    c = __reduce_add_sync(0xffffffffu, lane < G ? s_c[lane * (width + 1) + e] : 0);
    const float mean = T > 0 ? p / (float)T : 0.f;
    if (lane == 0) {
      a.mean[first + e] = mean;
      a.counts[first + e] = c;
    }
    term += (float)c * mean;
  }
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");   // the first block runs: its memory is there
  if (lane == 0) cluster.map_shared_rank(&s_term[0], 0)[rank * 32 + warp] = term;
  cluster.sync();
  if (rank == 0 && warp == 0) {
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < kCluster; ++b) sum += s_term[b * 32 + lane];
    sum = warp_add(sum);
    if (lane == 0) write_loss(a, sum, T);
  }
}

template <typename... KArgs>
cudaError_t launch_cluster(void (*kernel)(KArgs...), unsigned blocks, unsigned threads, unsigned cluster, bool chained, cudaStream_t s,
                           const LossArgs& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (chained) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T> struct LaunchLoss {
  const LossArgs& a;
  cudaStream_t s;
  template <int LANES, int PER_LANE, int P> int operator()() const {
    // few rows: a block of its own where its warps have at most two, else a cluster
    constexpr int kWarps = loss_warps(LANES * PER_LANE);
    const unsigned cluster = a.parts > 0 || a.M <= 2 * kWarps * 32 / LANES ? 1 : kCluster;
    const unsigned blocks = a.parts > 0 ? (unsigned)a.parts : cluster;
    XKB_CHECK_CUDA(launch_cluster(balance_kernel<T, LANES, PER_LANE, P>, blocks, 32 * kWarps, cluster, false, s, a));
    XKB_CHECK_LAUNCH("balance_kernel");
    return XKB_OK;
  }
};

// Blocks that leave a row of partial sums: none, which is one cluster and no second kernel, up to 512 rows; at most one per SM.
int64_t loss_parts(int64_t M) { return M <= 512 ? 0 : M < 148 * 8 ? ceil_div(M, (int64_t)8) : 148; }

}  // namespace
}  // namespace xkb

extern "C" int64_t xkb_moe_balance_loss_workspace_bytes(int64_t M, int E) {
  using namespace xkb;
  if (M < 0 || E < 1 || E > kMaxExperts) return -1;
  const int64_t parts = loss_parts(M);
  if (parts == 0) return 0;
  return 2 * align_up(parts * E * 4, 256) + align_up(parts * 4, 256);
}

extern "C" int xkb_moe_balance_loss(const void* gating_output, int dtype, const int32_t* topk_ids, const uint8_t* token_mask,
                                    float* loss, int32_t* counts, float* mean_probs, int32_t* tokens, int64_t M, int E,
                                    int top_k, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace xkb;
  XKB_REQUIRE(M >= 0 && E >= 1 && E <= kMaxExperts, "moe_balance_loss: bad shape M=%lld E=%d (at most %d experts)", (long long)M, E, kMaxExperts);
  XKB_REQUIRE(top_k >= 0 && M <= 0x7fffffff / (top_k > 0 ? top_k : 1), "moe_balance_loss: M * top_k must fit 31 bits (M=%lld, top_k=%d)", (long long)M, top_k);
  XKB_REQUIRE(dtype == XKB_BF16 || dtype == XKB_F32 || dtype == XKB_F16, "moe_balance_loss: unsupported logits dtype code %d", dtype);
  XKB_REQUIRE(loss && counts && mean_probs && tokens && (M == 0 || gating_output) && (M * top_k == 0 || topk_ids),
              "moe_balance_loss: null pointer");
  const int64_t need = xkb_moe_balance_loss_workspace_bytes(M, E);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(XKB_ERR_WORKSPACE, "moe_balance_loss: the workspace needs %lld bytes (got %lld)", (long long)need,
                (long long)(workspace ? workspace_bytes : 0));
  XKB_REQUIRE(address_bits(workspace) % 4 == 0, "moe_balance_loss: misaligned workspace");
  XKB_REQUIRE(address_bits(gating_output) % (dtype == XKB_F32 ? 4 : 2) == 0 && address_bits(topk_ids, loss, counts, mean_probs, tokens) % 4 == 0,
              "moe_balance_loss: a misaligned tensor");
  const int64_t parts = loss_parts(M);
  LossArgs a{gating_output, topk_ids, token_mask, nullptr, nullptr, nullptr, loss, counts, mean_probs, tokens, M, E, top_k, (int)parts};
  if (parts > 0) {
    Carver ws(workspace);
    a.part_p = ws.take<float>(parts * E);
    a.part_c = ws.take<int32_t>(parts * E);
    a.part_t = ws.take<int32_t>(parts);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uintptr_t bits = address_bits(gating_output);
  int rc;
  switch (dtype) {
    case XKB_BF16: rc = with_shape<__nv_bfloat16>(E, top_k, bits, LaunchLoss<__nv_bfloat16>{a, s}); break;
    case XKB_F32: rc = with_shape<float>(E, top_k, bits, LaunchLoss<float>{a, s}); break;
    default: rc = with_shape<__half>(E, top_k, bits, LaunchLoss<__half>{a, s}); break;
  }
  if (rc != XKB_OK || parts == 0) return rc;
  XKB_CHECK_CUDA(launch_cluster(balance_join_kernel, kCluster, 1024, kCluster, true, s, a));
  XKB_CHECK_LAUNCH("balance_join_kernel");
  return XKB_OK;
}
