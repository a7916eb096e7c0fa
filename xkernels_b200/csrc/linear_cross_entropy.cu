// Softmax cross entropy of a head's logits z = x W^T that are never stored, and its gradients.
//
// Rows without a label (padding) are no work: one kernel lists the others and copies their hidden states together, and how
// many there are stays on the device.  Forward: the dense product's read-out keeps maximum and sum of exponentials of a
// row's piece of the vocabulary, and one kernel joins the pieces in a fixed order.  Backward: the vocabulary goes by in
// pieces; a piece's logits are multiplied once more and leave the read-out as their gradient d = p (a + b) - a onehot, rounded
// once to 16 bits as the operand of the next products has to be; d W, added up over the pieces in fp32, and d^T x follow as one
// launch.  Three products a piece, 2 M H V each: bound by the tensor cores, and by the weight's bytes where rows are few.
#include "dense_dev.cuh"

namespace xkb {
namespace dense {

int run_ce(int end, const Params& p, const Launch& l) {
  return end == kCeStats ? run_variant<false, kCeStats>(p, l) : run_variant<false, kCeGrad>(p, l);
}

}  // namespace dense

namespace {

constexpr int kListThreads = 256;
constexpr int kJoinThreads = 512;
constexpr int kRowPad = 256;                       // rows of the row arrays are a multiple of this
constexpr int64_t kPieceBytes = 256ll << 20;       // of the logits' gradient that is held at a time

struct Rows {
  int32_t* count;      // rows with a label
  int32_t* rows;       // which they are, in order
  int32_t* labels;     // their labels; V for one outside the vocabulary
  float* inv_scale;    // what undoes the scale of d
  float4* coef;        // backward: m, l, factor of p, what is taken off at the label, times the scale
  uint16_t* x;         // their hidden states
};

struct ListArgs {
  const void* hidden;
  int64_t ld, ld_x;
  const void* labels;
  int ids64, vec;
  int64_t M, H, V;
  const float* stats;
  const float *g_loss, *g_lse;
  int fp16;
  uint16_t* grad_hidden;   // rows without a label are 0 there
  Rows r;
};

__device__ __forceinline__ int64_t label_at(const ListArgs& a, int64_t i) {
  return a.ids64 ? static_cast<const int64_t*>(a.labels)[i] : (int64_t)static_cast<const int32_t*>(a.labels)[i];
}
__device__ __forceinline__ float size_at(const ListArgs& a, int64_t i) {
  return (a.g_loss != nullptr ? fabsf(a.g_loss[i]) : 0.f) + (a.g_lse != nullptr ? fabsf(a.g_lse[i]) : 0.f);
}

// A block has some rows in a line.  It counts the labels before them itself (all blocks read all labels, from L2).
__global__ void __launch_bounds__(kListThreads) list_rows_kernel(const ListArgs a) {
  __shared__ int warp_sum[2][kListThreads / 32];
  __shared__ float warp_top[kListThreads / 32];
  __shared__ int place[kListThreads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = kListThreads / 32;
  const int64_t per = (a.M + gridDim.x - 1) / gridDim.x;
  const int64_t r0 = min((int64_t)blockIdx.x * per, a.M), r1 = min(r0 + per, a.M);
  int before = 0, all = 0;
  float top = 0.f;
  for (int64_t i = tid; i < a.M; i += kListThreads) {
    const bool on = label_at(a, i) >= 0;
    all += on;
    before += on && i < r0;
    if (a.fp16 && on) top = max_nan(top, size_at(a, i));
  }
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(~0u, before, o);
    all += __shfl_xor_sync(~0u, all, o);
    top = max_nan(top, __shfl_xor_sync(~0u, top, o));
  }
  if (lane == 0) warp_sum[0][warp] = before, warp_sum[1][warp] = all, warp_top[warp] = top;
  __syncthreads();
  before = all = 0;
  top = 0.f;
  for (int w = 0; w < warps; ++w) before += warp_sum[0][w], all += warp_sum[1][w], top = max_nan(top, warp_top[w]);
  // fp16 gradients of the logits: times the power of two that brings the largest factor to 2^10 .. 2^11, so that the small
  // probabilities of a large vocabulary do not fall below fp16's steps (2^-24).  |d| <= 2 |a| + |b|: no overflow.
  float scale = 1.f, inv = 1.f;
  if (a.fp16 && top > 0.f && top < INFINITY) {
    int e = 10 - (int)floorf(log2f(top));
    e = e > 100 ? 100 : e < -100 ? -100 : e;
    scale = exp2f((float)e);
    inv = exp2f((float)-e);
  }
  if (blockIdx.x == 0 && tid == 0) {
    *a.r.count = all;
    *a.r.inv_scale = inv;
  }
  // rows of x, a warp each; out: 16 bytes aligned, ld_x a multiple of 8
  auto copy = [&](const uint16_t* from, uint16_t* to) {
    if (from == nullptr) {
      for (int64_t c = lane * 8; c < a.H; c += 256) *reinterpret_cast<uint4*>(to + c) = make_uint4(0, 0, 0, 0);
    } else if (a.vec) {
      for (int64_t c = lane * 8; c < a.H; c += 256) *reinterpret_cast<uint4*>(to + c) = *reinterpret_cast<const uint4*>(from + c);
    } else {
      for (int64_t c = lane; c < a.H; c += 32) to[c] = from[c];
    }
  };
  for (int64_t base = r0; base < r1; base += kListThreads) {
    const int64_t i = base + tid;
    const int64_t label = i < r1 ? label_at(a, i) : -1;
    const bool on = label >= 0;
    const uint32_t vote = __ballot_sync(~0u, on);
    __syncthreads();
    if (lane == 0) warp_sum[0][warp] = __popc(vote);
    __syncthreads();
    int at = before + __popc(vote & ((1u << lane) - 1));
    for (int w = 0; w < warps; ++w) {
      if (w < warp) at += warp_sum[0][w];
      before += warp_sum[0][w];
    }
    place[tid] = on ? at : -1;
    if (on) {
      a.r.rows[at] = (int32_t)i;
      a.r.labels[at] = (int32_t)(label < a.V ? label : a.V);
      if (a.stats != nullptr) {
        float m = a.stats[2 * i], l = a.stats[2 * i + 1];
        if (m == -INFINITY) m = l = 0.f;       // a row without a live logit: its probabilities are 0
        const float ga = a.g_loss != nullptr ? a.g_loss[i] * scale : 0.f, gb = a.g_lse != nullptr ? a.g_lse[i] * scale : 0.f;
        const float bad = label < a.V ? 0.f : NAN;
        a.r.coef[at] = make_float4(m, l, ga + gb + bad, ga);
      }
    }
    __syncthreads();
    const int n = (int)min((int64_t)kListThreads, r1 - base);
    for (int j = warp; j < n; j += warps) {
      if (place[j] >= 0) {
        copy(static_cast<const uint16_t*>(a.hidden) + (base + j) * a.ld, a.r.x + (int64_t)place[j] * a.ld_x);
      } else if (a.grad_hidden != nullptr) {
        for (int64_t c = lane; c < a.H; c += 32) a.grad_hidden[(base + j) * a.H + c] = 0;
      }
    }
  }
  // behind the last row: zeros, as far as a product may read
  const int64_t pad = (all + kRowPad - 1) / kRowPad * kRowPad;
  for (int64_t j = all + blockIdx.x * warps + warp; j < pad; j += (int64_t)gridDim.x * warps) copy(nullptr, a.r.x + j * a.ld_x);
}

struct JoinArgs {
  const float2* part;
  int parts;
  int64_t part_ld;
  const float* given;
  const int32_t *count, *rows, *labels_of_rows;
  const void* labels;
  int ids64;
  int64_t M, V;
  float *loss, *lse, *stats;
};

// Lane = row (32 rows a block), the warps share its pieces.  Blocks beyond the rows' write the padding rows' zeros.
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const JoinArgs a) {
  chain_wait();
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ float sm[kWarps][33], ss[kWarps][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t i = (int64_t)blockIdx.x * 32 + lane;      // row of the batch, for the padding; of the list, for the rest
  if (warp == 0 && i < a.M) {
    const int64_t label = a.ids64 ? static_cast<const int64_t*>(a.labels)[i] : (int64_t)static_cast<const int32_t*>(a.labels)[i];
    if (label < 0) a.loss[i] = a.lse[i] = a.stats[2 * i] = a.stats[2 * i + 1] = 0.f;
  }
  const int count = *a.count;
  if ((int64_t)blockIdx.x * 32 >= count) return;
  const bool on = i < count;
  float m = -INFINITY, s = 0.f;
  if (on) {
    for (int q = warp; q < a.parts; q += kWarps) m = fmaxf(m, a.part[q * a.part_ld + i].x);
    const float ref = m == -INFINITY ? 0.f : m;
    for (int q = warp; q < a.parts; q += kWarps) {
      const float2 f = a.part[q * a.part_ld + i];
      s += f.y * exp2_fast((f.x - ref) * kLog2e);
    }
  }
  sm[warp][lane] = m;
  ss[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || !on) return;
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, sm[w][lane]);
  const float ref = m == -INFINITY ? 0.f : m;
  s = 0.f;
  for (int w = 0; w < kWarps; ++w) s += ss[w][lane] * exp2_fast((sm[w][lane] - ref) * kLog2e);
  // (a piece whose maximum is below all: exp2(-inf) = 0; a NaN or +inf in the row has made its sum a NaN)
  const bool dead = m == -INFINITY && s == 0.f;      // no live logit
  const float l = dead ? 0.f : logf(s);
  const int64_t to = a.rows[i];
  const bool known = a.labels_of_rows[i] < a.V;
  a.loss[to] = !known ? NAN : dead ? INFINITY : (m - a.given[i]) + l;
  a.lse[to] = m + l;
  a.stats[2 * to] = m;
  a.stats[2 * to + 1] = l;
}

int64_t padded(int64_t M) { return align_up(M, kRowPad); }
int64_t pitch8(int64_t n) { return align_up(n, 8); }

int check_sizes(const char* name, int dtype, int64_t M, int64_t H, int64_t V) {
  XKB_REQUIRE(dtype == XKB_BF16 || dtype == XKB_F16, "%s: dtype must be bf16 or fp16", name);
  XKB_REQUIRE(M >= 0 && H >= 1 && V >= 1 && M < (1ll << 28) && H < (1ll << 24) && V < (1ll << 28), "%s: M=%lld H=%lld V=%lld out of range",
              name, (long long)M, (long long)H, (long long)V);
  return XKB_OK;
}

// Columns of the vocabulary that the backward pass takes at a time: what kPieceBytes hold, 256 at least.
int64_t piece_of(int64_t M, int64_t V) {
  const int64_t most = kPieceBytes / 2 / padded(M) / 256 * 256;
  const int64_t piece = most < 256 ? 256 : most;
  const int64_t pieces = ceil_div(V, piece);
  return align_up(ceil_div(V, pieces), 256);     // alike, so that no short one is left
}

struct Work {
  Rows r;
  float2* part;
  float* given;
  uint16_t* d;
  float* acc;
  int64_t bytes;
};

Work carve(void* ws, int64_t M, int64_t H, int64_t V, bool backward) {
  Carver c(ws);
  Work w = {};
  const int64_t P = padded(M);
  w.r.count = c.take<int32_t>(1);
  w.r.inv_scale = c.take<float>(1);
  w.r.rows = c.take<int32_t>(P);
  w.r.labels = c.take<int32_t>(P);
  w.r.x = c.take<uint16_t>(P * pitch8(H));
  if (backward) {
    w.r.coef = c.take<float4>(P);
    const int64_t piece = piece_of(M, V);
    w.d = c.take<uint16_t>(P * piece);
    if (piece < V) w.acc = c.take<float>(P * align_up(H, 32));
  } else {
    w.given = c.take<float>(P);
    w.part = c.take<float2>(dense::ce_parts(M, V, H) * P);
  }
  w.bytes = c.off;
  return w;
}

int check_workspace(const char* name, const void* ws, int64_t bytes, int64_t need) {
  if (ws == nullptr || bytes < need || reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return fail(XKB_ERR_WORKSPACE, "%s: needs a workspace of %lld bytes on 256 bytes", name, (long long)need);
  return XKB_OK;
}

int check_inputs(const char* name, const void* hidden, int64_t ld_h, const void* weight, int64_t ld_w, const void* labels, int ids64, int64_t M,
                 int64_t H) {
  XKB_REQUIRE(hidden != nullptr && weight != nullptr && labels != nullptr, "%s: null input", name);
  XKB_REQUIRE(ids64 == 0 || ids64 == 1, "%s: ids64 must be 0 or 1", name);
  XKB_REQUIRE(reinterpret_cast<uintptr_t>(hidden) % 2 == 0 && reinterpret_cast<uintptr_t>(labels) % (ids64 ? 8 : 4) == 0,
              "%s: misaligned input", name);
  XKB_REQUIRE(ld_h >= 0 && ld_h < (1ll << 32), "%s: row stride of hidden out of range", name);
  XKB_REQUIRE(reinterpret_cast<uintptr_t>(weight) % 16 == 0 && ld_w % 8 == 0 && ld_w >= H && ld_w < (1ll << 32),
              "%s: rows of weight must start on 16 bytes and not overlap (row stride %lld)", name, (long long)ld_w);
  return XKB_OK;
}

int launch_list(const ListArgs& a, cudaStream_t stream) {
  const int64_t blocks = a.M < 296 ? a.M : 296;
  list_rows_kernel<<<(unsigned)blocks, kListThreads, 0, stream>>>(a);
  XKB_CHECK_LAUNCH("list_rows_kernel");
  return XKB_OK;
}

#define XKB_TRY(expr)              \
  do {                             \
    const int _rc = (expr);        \
    if (_rc != XKB_OK) return _rc; \
  } while (0)

}  // namespace
}  // namespace xkb

using namespace xkb;

extern "C" int64_t xkb_linear_cross_entropy_workspace_bytes(int64_t M, int64_t H, int64_t V) {
  if (check_sizes("linear_cross_entropy", XKB_BF16, M, H, V) != XKB_OK) return -1;
  return M == 0 ? 0 : carve(nullptr, M, H, V, false).bytes;
}

extern "C" int xkb_linear_cross_entropy(const void* hidden, int64_t ld_hidden, int dtype, const void* weight, int64_t ld_weight,
                                        const void* labels, int ids64, float* loss, float* lse, float* stats, int64_t M, int64_t H,
                                        int64_t V, void* workspace, int64_t workspace_bytes, void* stream_) {
  const char* name = "linear_cross_entropy";
  XKB_TRY(check_sizes(name, dtype, M, H, V));
  if (M == 0) return XKB_OK;
  XKB_TRY(check_inputs(name, hidden, ld_hidden, weight, ld_weight, labels, ids64, M, H));
  XKB_REQUIRE(loss != nullptr && lse != nullptr && stats != nullptr && address_bits(loss, lse, stats) % 4 == 0,
              "%s: null or misaligned output", name);
  const Work w = carve(workspace, M, H, V, false);
  XKB_TRY(check_workspace(name, workspace, workspace_bytes, w.bytes));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  ListArgs a = {};
  a.hidden = hidden, a.ld = ld_hidden, a.ld_x = pitch8(H);
  a.labels = labels, a.ids64 = ids64;
  a.vec = reinterpret_cast<uintptr_t>(hidden) % 16 == 0 && ld_hidden % 8 == 0 && H % 8 == 0;
  a.M = M, a.H = H, a.V = V;
  a.r = w.r;
  XKB_TRY(launch_list(a, stream));
  dense::Product q = {};
  q.a = {w.r.x, pitch8(H), false, 0, padded(M), H};
  q.b = {weight, ld_weight, false, 0, V, H};
  q.M = M, q.N = V, q.K = H;
  q.live = w.r.count;
  q.end.labels = w.r.labels;
  q.end.part = w.part, q.end.part_ld = padded(M);
  q.end.given = w.given;
  XKB_TRY(dense::launch(&q, 1, dense::kCeStats, dtype, true, false, stream));
  JoinArgs j = {};
  j.part = w.part, j.parts = dense::ce_parts(M, V, H), j.part_ld = padded(M);
  j.given = w.given, j.count = w.r.count, j.rows = w.r.rows, j.labels_of_rows = w.r.labels;
  j.labels = labels, j.ids64 = ids64, j.M = M, j.V = V;
  j.loss = loss, j.lse = lse, j.stats = stats;
  XKB_CHECK_CUDA(launch_chained(join_kernel, dim3((unsigned)ceil_div(M, 32)), dim3(kJoinThreads), 0, stream, j));
  XKB_CHECK_LAUNCH("join_kernel");
  return XKB_OK;
}

extern "C" int64_t xkb_linear_cross_entropy_backward_workspace_bytes(int64_t M, int64_t H, int64_t V) {
  if (check_sizes("linear_cross_entropy_backward", XKB_BF16, M, H, V) != XKB_OK) return -1;
  return M == 0 ? 0 : carve(nullptr, M, H, V, true).bytes;
}

extern "C" int xkb_linear_cross_entropy_backward(const void* hidden, int64_t ld_hidden, int dtype, const void* weight, int64_t ld_weight,
                                                 const void* labels, int ids64, const float* stats, const float* grad_loss,
                                                 const float* grad_lse, void* grad_hidden, void* grad_weight, int64_t M, int64_t H, int64_t V,
                                                 void* workspace, int64_t workspace_bytes, void* stream_) {
  const char* name = "linear_cross_entropy_backward";
  XKB_TRY(check_sizes(name, dtype, M, H, V));
  XKB_REQUIRE(address_bits(grad_hidden, grad_weight) % 2 == 0, "%s: misaligned output", name);
  if (grad_hidden == nullptr && grad_weight == nullptr) return XKB_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (M == 0) {
    if (grad_weight != nullptr) XKB_CHECK_CUDA(cudaMemsetAsync(grad_weight, 0, (size_t)(V * H) * 2, stream));
    return XKB_OK;
  }
  XKB_TRY(check_inputs(name, hidden, ld_hidden, weight, ld_weight, labels, ids64, M, H));
  XKB_REQUIRE(stats != nullptr && address_bits(stats, grad_loss, grad_lse) % 4 == 0, "%s: null or misaligned input", name);
  XKB_REQUIRE(grad_loss != nullptr || grad_lse != nullptr, "%s: no gradient is given", name);
  const Work w = carve(workspace, M, H, V, true);
  XKB_TRY(check_workspace(name, workspace, workspace_bytes, w.bytes));
  ListArgs a = {};
  a.hidden = hidden, a.ld = ld_hidden, a.ld_x = pitch8(H);
  a.labels = labels, a.ids64 = ids64;
  a.vec = reinterpret_cast<uintptr_t>(hidden) % 16 == 0 && ld_hidden % 8 == 0 && H % 8 == 0;
  a.M = M, a.H = H, a.V = V;
  a.stats = stats, a.g_loss = grad_loss, a.g_lse = grad_lse;
  a.fp16 = dtype == XKB_F16;
  a.grad_hidden = static_cast<uint16_t*>(grad_hidden);
  a.r = w.r;
  XKB_TRY(launch_list(a, stream));
  const int64_t piece = piece_of(M, V);
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t n = V - v0 < piece ? V - v0 : piece;
    dense::Product z = {};
    z.a = {w.r.x, pitch8(H), false, 0, padded(M), H};
    z.b = {weight, ld_weight, false, v0, V, H};
    z.M = M, z.N = n, z.K = H;
    z.live = w.r.count;
    z.end.out = w.d, z.end.ld = piece;
    z.end.labels = w.r.labels, z.end.coef = w.r.coef;
    z.end.col0 = (int)v0;
    XKB_TRY(dense::launch(&z, 1, dense::kCeGrad, dtype, true, false, stream));
    dense::Product q[2] = {};
    int count = 0;
    if (grad_hidden != nullptr) {
      dense::Product& g = q[count++];
      g.a = {w.d, piece, false, 0, padded(M), n};
      g.b = {weight, ld_weight, true, v0, V, H};
      g.M = M, g.N = H, g.K = n;
      g.live = w.r.count;
      g.end.out = grad_hidden, g.end.ld = H;
      g.end.row_map = w.r.rows;
      g.end.acc = w.acc, g.end.acc_ld = align_up(H, 32);
      g.end.acc_in = v0 > 0, g.end.acc_out = v0 + n < V;
      if (!g.end.acc_out) g.end.scale = w.r.inv_scale;
    }
    if (grad_weight != nullptr) {
      dense::Product& g = q[count++];
      g.a = {w.d, piece, true, 0, padded(M), n};
      g.b = {w.r.x, pitch8(H), true, 0, padded(M), H};
      g.M = n, g.N = H, g.K = M;
      g.live = w.r.count;
      g.end.out = static_cast<uint16_t*>(grad_weight) + v0 * H, g.end.ld = H;
      g.end.scale = w.r.inv_scale;
    }
    XKB_TRY(dense::launch(q, count, dense::kStore, dtype, true, false, stream));
  }
  return XKB_OK;
}
