// Softmax cross entropy of a head's logits z = x W^T that are never stored, and its gradients.
//
// Rows without a label (padding) are no work: one kernel lists the others and copies their hidden states together, and how
// many there are stays on the device.  Forward: the dense product's read-out keeps maximum and sum of exponentials of a
// row's piece of the vocabulary, and one kernel joins the pieces in a fixed order.  Backward: the vocabulary goes by in
// pieces; a piece's logits are multiplied once more and leave the read-out as their gradient d = p (a + b) - a onehot, rounded
// once to 16 bits as the operand of the next products has to be (up to 16 rows in two terms of them); d W, added up over the pieces in fp32, and d^T x follow as one
// launch.  Three products a piece, 2 M H V each: bound by the tensor cores, and by the weight's bytes where rows are few.
// 4096 x 7168 x 128000, tensor pipe 93 % busy: 4.6 and 13.9 ms between pauses (1470 and 1460 TFLOP/s), 5.5 and 16.2 in a loop, where
// the power limit holds (1230 and 1250).  One row of 4096 x 50001: 76 us in a graph (5.4 TB/s), 84 a call among others.
#include "dense_dev.cuh"

namespace xkb {
namespace dense {

int run_ce(int end, const Params& p, const Launch& l) {
  if (end == kCeStats) return run_variant<false, kCeStats>(p, l);
  return p.prod[0].end.second != 0 ? run_variant<false, kCeGradTwo>(p, l) : run_variant<false, kCeGrad>(p, l);
}

}  // namespace dense

namespace {

constexpr int kListThreads = 512;
constexpr int kListBlocks = 296;                    // two on every SM
constexpr int kSegment = 2048;                      // elements of a row that a warp copies at a time: eight loads a lane in flight
constexpr int kJoinThreads = 128;
constexpr int kRowPad = 256;                       // rows of the row arrays are a multiple of this
// Of the logits' gradient that is held at a time.  4096 x 7168 x 128000, pieces of 64 / 128 / 256 / 512 / 1100 MiB (all of it):
// 15.4 / 14.8 / 15.0 / 14.9 / 15.3 ms, spread of runs 0.3.
constexpr int64_t kPieceBytes = 256ll << 20;

// Up to so many rows d has two 16-bit terms, the second in rows kTwoTerms further, and the hidden states stand there once more: with
// few rows the rounding errors of a row's few large gradients (its label's above all) do not average out.  Error of the gradients in
// the norm, bf16, the worst of eight draws, with one term and two (the result's own rounding is 1.7e-3): 1 x 136 x 25212 3.2e-3 and
// 1.8e-3, 5 x 376 x 1077 3.1e-3 and 1.7e-3; 1 x 4096 x 50001 278 and 292 us.
constexpr int kTwoTerms = 16;

struct Rows {
  int32_t* count;      // rows with a label; rows of d that two terms of them fill
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
  int ids64, vec, vec_grad;
  int second;              // labelled rows are copied to this many rows further too (0: once)
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

// A block has some rows in a line, or with few rows a part of the columns of one.  It counts the labels before them itself
// (all blocks read all labels, from L2).  Bound by the latency of the copies.
__global__ void __launch_bounds__(kListThreads) list_rows_kernel(const ListArgs a, const int col_blocks) {
  chain_trigger();
  constexpr int kWarps = kListThreads / 32;
  __shared__ int warp_sum[2][kWarps];
  __shared__ float warp_top[kWarps];
  __shared__ int place[kListThreads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row_blocks = gridDim.x / col_blocks, block = blockIdx.x / col_blocks, col_block = blockIdx.x - block * col_blocks;
  const int64_t per = (a.M + row_blocks - 1) / row_blocks;
  const int64_t r0 = min((int64_t)block * per, a.M), r1 = min(r0 + per, a.M);
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
  for (int w = 0; w < kWarps; ++w) before += warp_sum[0][w], all += warp_sum[1][w], top = max_nan(top, warp_top[w]);
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
    a.r.count[0] = all;
    a.r.count[1] = all > 0 ? a.second + kTwoTerms : 0;      // (no row: there is no d)
    *a.r.inv_scale = inv;
  }
  const int segments = (int)((a.H + kSegment - 1) / kSegment);
  const int mine = (segments - col_block + col_blocks - 1) / col_blocks;     // segments col_block, col_block + col_blocks, ..
  // a segment of a row of x, by a warp; from nullptr: zeros.  The rows there start on 16 bytes.
  auto copy = [&](const uint16_t* from, uint16_t* to, int segment) {
    const int64_t c0 = (int64_t)segment * kSegment;
    if (from == nullptr || a.vec) {
      uint4 v[kSegment / 256];
#pragma unroll
      for (int j = 0; j < kSegment / 256; ++j) {
        const int64_t c = c0 + j * 256 + lane * 8;
        v[j] = from != nullptr && c < a.H ? *reinterpret_cast<const uint4*>(from + c) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < kSegment / 256; ++j) {
        const int64_t c = c0 + j * 256 + lane * 8;
        if (c < a.H) *reinterpret_cast<uint4*>(to + c) = v[j];
      }
    } else {
#pragma unroll 8
      for (int64_t c = c0 + lane; c < min(c0 + kSegment, a.H); c += 32) to[c] = from[c];
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
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) at += warp_sum[0][w];
      before += warp_sum[0][w];
    }
    place[tid] = on ? at : -1;
    if (on && col_block == 0) {
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
    for (int u = warp; u < n * mine; u += kWarps) {
      const int j = u / mine, segment = (u - j * mine) * col_blocks + col_block;
      if (place[j] >= 0) {
        const uint16_t* from = static_cast<const uint16_t*>(a.hidden) + (base + j) * a.ld;
        copy(from, a.r.x + (int64_t)place[j] * a.ld_x, segment);
        if (a.second != 0) copy(from, a.r.x + (int64_t)(place[j] + a.second) * a.ld_x, segment);
      } else if (a.grad_hidden != nullptr) {
        const int64_t c0 = (int64_t)segment * kSegment, c1 = min(c0 + kSegment, a.H);
        uint16_t* to = a.grad_hidden + (base + j) * a.H;
        if (a.vec_grad) for (int64_t c = c0 + lane * 8; c < c1; c += 256) *reinterpret_cast<uint4*>(to + c) = make_uint4(0, 0, 0, 0);
        else for (int64_t c = c0 + lane; c < c1; c += 32) to[c] = 0;
      }
    }
  }
  // behind the last row: zeros, as far as a product may read
  const int64_t pad = (all + kRowPad - 1) / kRowPad * kRowPad;
  for (int64_t u = (int64_t)blockIdx.x * kWarps + warp; u < (pad - all) * segments; u += (int64_t)gridDim.x * kWarps) {
    const int64_t j = u / segments, row = all + j;
    if (row < a.second || row >= a.second + all) copy(nullptr, a.r.x + row * a.ld_x, (int)(u - j * segments));
  }
}

struct JoinArgs {
  const float2* part;
  int parts;
  const float* given;
  const int32_t *count, *rows;     // nullptr: the rows are the batch's
  const void* labels;
  int ids64;
  int64_t M, V;
  float *loss, *lse, *stats;
};

// A block a row: thread = piece of the vocabulary, in turn.  Block i also writes the zeros of row i of the batch if it is padding.
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const JoinArgs a) {
  chain_wait();
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ float sm[kWarps], ss[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t i = blockIdx.x;
  auto label_of = [&](int64_t r) {
    return a.ids64 ? static_cast<const int64_t*>(a.labels)[r] : (int64_t)static_cast<const int32_t*>(a.labels)[r];
  };
  const bool padding = label_of(i) < 0;
  if (padding && tid == 0) a.loss[i] = a.lse[i] = a.stats[2 * i] = a.stats[2 * i + 1] = 0.f;
  if (a.count != nullptr ? i >= *a.count : padding) return;
  const float2* part = a.part + i * a.parts;
  float m = -INFINITY, s = 0.f;
  for (int q = tid; q < a.parts; q += kJoinThreads) {
    const float2 f = part[q];
    const float top = fmaxf(m, f.x), ref = top == -INFINITY ? 0.f : top;
    // (a piece without a live logit: exp2(-inf) = 0; a NaN or +inf in the row has made its piece's sum a NaN)
    s = s * exp2_fast((m - ref) * kLog2e) + f.y * exp2_fast((f.x - ref) * kLog2e);
    m = top;
  }
  float top = m;
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if (lane == 0) sm[warp] = top;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
  const float ref = top == -INFINITY ? 0.f : top;
  s = warp_add(s * exp2_fast((m - ref) * kLog2e));
  if (lane == 0) ss[warp] = s;
  __syncthreads();
  if (tid != 0) return;
  s = 0.f;
  for (int w = 0; w < kWarps; ++w) s += ss[w];
  const bool dead = top == -INFINITY && s == 0.f;      // no live logit
  const float l = dead ? 0.f : logf(s);
  const int64_t to = a.rows != nullptr ? a.rows[i] : i;
  a.loss[to] = label_of(to) >= a.V ? NAN : dead ? INFINITY : (top - a.given[i]) + l;
  a.lse[to] = top + l;
  a.stats[2 * to] = top;
  a.stats[2 * to + 1] = l;
}

struct AddArgs {
  const float* acc;
  int64_t acc_ld, acc_part, H;
  int parts, fmt, vec;
  const int32_t *count, *rows;
  const float* scale;
  uint16_t* out;
};

// The parts of grad_hidden added up in their order, a block a row.
__global__ void __launch_bounds__(256) add_parts_kernel(const AddArgs a) {
  chain_wait();
  const int64_t i = blockIdx.x;
  if (i >= *a.count) return;
  const float scale = *a.scale;
  uint16_t* to = a.out + (int64_t)a.rows[i] * a.H;
  for (int64_t c = threadIdx.x * 4; c < a.H; c += 1024) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = 0; q < a.parts; ++q) {
      const float4 f = *reinterpret_cast<const float4*>(a.acc + q * a.acc_part + i * a.acc_ld + c);
      s.x += f.x, s.y += f.y, s.z += f.z, s.w += f.w;
    }
    const uint32_t lo = dense::pack16(a.fmt, s.x * scale, s.y * scale), hi = dense::pack16(a.fmt, s.z * scale, s.w * scale);
    if (a.vec) {
      *reinterpret_cast<uint2*>(to + c) = make_uint2(lo, hi);
    } else {
      const uint32_t w[2] = {lo, hi};
      for (int j = 0; j < 4; ++j)
        if (c + j < a.H) to[c + j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    }
  }
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
  int k_parts;
  int64_t bytes;
};

Work carve(void* ws, int64_t M, int64_t H, int64_t V, bool backward) {
  Carver c(ws);
  Work w = {};
  const int64_t P = padded(M);
  w.r.count = c.take<int32_t>(2);
  w.r.inv_scale = c.take<float>(1);
  w.r.rows = c.take<int32_t>(P);
  w.r.labels = c.take<int32_t>(P);
  w.r.x = c.take<uint16_t>(P * pitch8(H));
  if (backward) {
    w.r.coef = c.take<float4>(P);
    const int64_t piece = piece_of(M, V);
    w.d = c.take<uint16_t>(P * piece);
    const int64_t n = V < piece ? V : piece;
    w.k_parts = dense::k_parts_of(M, H, n, n, H, M);
    // (products that add up two terms have one accumulator)
    if (M <= kTwoTerms && w.k_parts < ceil_div(n, 65536)) w.k_parts = (int)ceil_div(n, 65536);
    if (piece < V || w.k_parts > 1) w.acc = c.take<float>(w.k_parts * P * align_up(H, 32));
  } else {
    w.given = c.take<float>(P);
    w.part = c.take<float2>(dense::ce_most_parts(M, V) * P);
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
  const int64_t row_blocks = a.M < kListBlocks ? a.M : kListBlocks, segments = ceil_div(a.H, kSegment);
  const int64_t spare = kListBlocks / row_blocks, col_blocks = spare < segments ? spare : segments;
  list_rows_kernel<<<(unsigned)(row_blocks * col_blocks), kListThreads, 0, stream>>>(a, (int)col_blocks);
  XKB_CHECK_LAUNCH("list_rows_kernel");
  return XKB_OK;
}

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
  const bool aligned = reinterpret_cast<uintptr_t>(hidden) % 16 == 0 && ld_hidden % 8 == 0;
  // One row tile takes as long whatever it holds: the hidden states are then read where they are (listing and copying cost 4 us).
  const bool in_place = M <= dense::kRows && aligned && ld_hidden >= H;
  dense::Product q = {};
  q.b = {weight, ld_weight, false, 0, V, H};
  q.M = M, q.N = V, q.K = H;
  int parts = 0;
  XKB_TRY(dense::ce_parts(M, V, H, &parts));
  q.end.part = w.part, q.end.part_ld = parts;
  q.end.given = w.given;
  JoinArgs j = {};
  if (in_place) {
    q.a = {hidden, ld_hidden, false, 0, M, H};
    if (ids64) q.end.labels64 = static_cast<const int64_t*>(labels);
    else q.end.labels = static_cast<const int32_t*>(labels);
  } else {
    ListArgs a = {};
    a.hidden = hidden, a.ld = ld_hidden, a.ld_x = pitch8(H);
    a.labels = labels, a.ids64 = ids64;
    a.vec = aligned && H % 8 == 0;
    a.M = M, a.H = H, a.V = V;
    a.r = w.r;
    XKB_TRY(launch_list(a, stream));
    q.a = {w.r.x, pitch8(H), false, 0, padded(M), H};
    q.live = w.r.count;
    q.end.labels = w.r.labels;
    j.count = w.r.count, j.rows = w.r.rows;
  }
  XKB_TRY(dense::launch(&q, 1, dense::kCeStats, dtype, !in_place, false, stream));
  j.part = w.part, j.parts = parts, j.given = w.given;
  j.labels = labels, j.ids64 = ids64, j.M = M, j.V = V;
  j.loss = loss, j.lse = lse, j.stats = stats;
  XKB_CHECK_CUDA(launch_chained(join_kernel, dim3((unsigned)M), dim3(kJoinThreads), 0, stream, j));
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
  a.vec_grad = reinterpret_cast<uintptr_t>(grad_hidden) % 16 == 0 && H % 8 == 0;
  a.r = w.r;
  a.second = M <= kTwoTerms ? kTwoTerms : 0;
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
    z.end.second = a.second;
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
      g.end.second = a.second;
      g.k_parts = w.k_parts;
      g.end.acc = w.acc, g.end.acc_ld = align_up(H, 32), g.end.acc_part = padded(M) * align_up(H, 32);
      g.end.acc_in = v0 > 0, g.end.acc_out = v0 + n < V || w.k_parts > 1;
      if (!g.end.acc_out) g.end.scale = w.r.inv_scale;
    }
    if (grad_weight != nullptr) {
      dense::Product& g = q[count++];
      g.a = {w.d, piece, true, 0, padded(M), n};
      g.b = {w.r.x, pitch8(H), true, 0, padded(M), H};
      g.M = n, g.N = H, g.K = a.second != 0 ? 2 * kTwoTerms : M;
      g.live = w.r.count + (a.second != 0 ? 1 : 0);
      g.end.out = static_cast<uint16_t*>(grad_weight) + v0 * H, g.end.ld = H;
      g.end.scale = w.r.inv_scale;
    }
    XKB_TRY(dense::launch(q, count, dense::kStore, dtype, true, false, stream));
  }
  if (grad_hidden != nullptr && w.k_parts > 1) {
    AddArgs s = {};
    s.acc = w.acc, s.acc_ld = align_up(H, 32), s.acc_part = padded(M) * align_up(H, 32), s.H = H;
    s.parts = w.k_parts, s.fmt = dtype == XKB_BF16 ? 1 : 0;
    s.vec = reinterpret_cast<uintptr_t>(grad_hidden) % 8 == 0 && H % 4 == 0;
    s.count = w.r.count, s.rows = w.r.rows, s.scale = w.r.inv_scale;
    s.out = static_cast<uint16_t*>(grad_hidden);
    XKB_CHECK_CUDA(launch_chained(add_parts_kernel, dim3((unsigned)M), dim3(256), 0, stream, s));
    XKB_CHECK_LAUNCH("add_parts_kernel");
  }
  return XKB_OK;
}
