// Host side of the dense products: tensor maps, which tile a product gets, launches.
#include <mutex>

#include "dense_dev.cuh"
#include "tensor_map.h"

namespace xkb {
extern std::atomic<int> g_sm_margin;

namespace dense {

// Status of the last wait that ran out on this device (0: none).  The calls have no workspace of their caller's that
// would outlive them, so it is the library's.
__device__ int g_dense_status;

namespace {

int sm_count(int dev, int* out) {
  static std::atomic<int> known[64];
  int n = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    XKB_CHECK_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return XKB_OK;
}

int status_word(int dev, int** out) {
  static std::atomic<int*> known[64];
  int* p = dev < 64 ? known[dev].load(std::memory_order_relaxed) : nullptr;
  if (p == nullptr) {
    void* at = nullptr;
    XKB_CHECK_CUDA(cudaGetSymbolAddress(&at, g_dense_status));
    p = static_cast<int*>(at);
    if (dev < 64) known[dev].store(p, std::memory_order_relaxed);
  }
  *out = p;
  return XKB_OK;
}

struct Shape { int cg, bn, split; };

// Which tile.  The cost of a shape is its rounds of tiles times the time of a tile: its blocks of K times the clocks of a
// stage, and the read-out.  A stage takes its MMAs (512 clocks for 256 x 256 on a pair, 256 for the halves) or its operands'
// bytes at 64 a clock and SM, whichever is more; and the operands have to come from memory once, at 3500 bytes a clock or 36
// a clock and CTA.  Sharing a tile costs a cluster the exchange of its parts.
// Forced one by one, whole calls of gated_ffn: one row of 7168 x 2048, gate and up in single CTAs of 64 columns shared by
// 2 / 1 / 3 / 4 27.1 / 33.7 / 29.5 / 28.5 us, of 128 by 4 27.4; the second product in 64 columns shared by 1 / 2 / 3 27.1 / 29.1 /
// 33.3, in 128 by 2 29.0.  509 rows of 4096 x 1416: gate and up in pairs of 128 / 256 columns 31.3 / 40.8, 256 shared by 2 34.6,
// single CTAs of 128 by 1 / 2 / 3 44.0 / 34.7 / 33.5.  (64 rows: by 4 28.8, by 2, which the rule takes, 30.1.)
int shape_of(const int64_t* M, const int64_t* N, const int64_t* K, const int* k_parts, int count, int end, bool may_split, bool two_terms,
             int dev, int sms, Shape* best) {
  *best = {2, 256, 1};
  double best_cost = 1e300;
  const bool paired = end == kSwiglu;
  double bytes = 0;
  for (int i = 0; i < count; ++i) bytes += 2.0 * K[i] * (M[i] + N[i] * (paired ? 2 : 1));
  auto consider = [&](Shape s, int64_t ctas, double clocks, double tail) {
    const double rate = ctas * 36.0 < 3500 ? ctas * 36.0 : 3500;
    const double cost = (clocks > bytes / rate ? clocks : bytes / rate) + tail;
    if (cost < best_cost * 0.999) best_cost = cost, *best = s;
  };
  // More of K than one accumulator is to take: pairs whose tile is their own have a way for it.  (Two terms have single CTAs only, and
  // no such K.)
  auto long_sum = [&](int64_t kb, int s) { return end == kStore && !two_terms && ceil_div(kb, s) > kLongBlocks; };
  for (int bn : {256, 128}) {
    // (two terms are single CTAs' alone; logits of one row tile have their shorter sums there: kPartBlocks)
    if (two_terms || ((end == kCeStats || end == kCeGrad) && M[0] <= kRows)) break;
    const int64_t tile_n = paired ? bn / 2 : bn;
    const double stage = bn == 256 ? 520 : 400, readout = bn == 256 ? 3500 : 2000;
    double work = 0;
    int64_t tiles = 0;
    for (int i = 0; i < count; ++i) {
      const int64_t t = ceil_div(M[i], 256) * ceil_div(N[i], tile_n) * k_parts[i], kb = ceil_div(ceil_div(K[i], kBK), k_parts[i]);
      tiles += t;
      // (a short tile takes its read-out's time)
      work += (double)t * (kb * stage > readout ? kb * stage : readout);
    }
    const double mean = work / (double)(tiles > 0 ? tiles : 1);
    consider({2, bn, 1}, 2 * tiles, (double)ceil_div(tiles, sms / 2) * mean, readout);
    if (count == 1 && may_split)
      for (int s = 2; s <= 4; ++s) {
        const int64_t kb = ceil_div(K[0], kBK);
        if (4 * s > kb || tiles * 2 * s > sms || long_sum(kb, s)) continue;
        int most = 0;
        const int rc = clusters_at_once(dev, 2, bn, 8, 2 * s, &most);
        if (rc != XKB_OK) return rc;
        if (tiles <= most) consider({2, bn, s}, 2 * tiles * s, ceil_div(kb, s) * stage, readout + 8000);
      }
  }
  if (count == 1 && may_split) {
    const int warps = single_warps(end);
    const int64_t kb = ceil_div(K[0], kBK), rows = M[0] < kRows ? align_up(M[0], 8) * (two_terms ? 2 : 1) : kRows;
    for (int bn : {128, 64}) {
      if (bn == 64 && warps == 8) continue;
      const int64_t tiles = ceil_div(M[0], kRows) * ceil_div(N[0], paired ? bn / 2 : bn);
      const double mma = bn == 128 ? 275 : 260, stage = 2 * (rows + bn) > mma ? 2 * (rows + bn) : mma;
      if (!long_sum(kb, 1)) consider({1, bn, 1}, tiles, (double)ceil_div(tiles, sms) * kb * stage, 2000);
      for (int s = 2; s <= 8; ++s) {
        if (4 * s > kb || tiles * s > 2 * sms || long_sum(kb, s)) continue;
        int most = 0;
        const int rc = clusters_at_once(dev, 1, bn, warps, s, &most);
        if (rc != XKB_OK) return rc;
        if (tiles <= most) consider({1, bn, s}, tiles * s, (double)(ceil_div(tiles * s, sms) * ceil_div(kb, s)) * stage, 4500 + 500 * s);
      }
    }
  }
  return XKB_OK;
}

int vec_of(const void* p, int64_t ld, int64_t extra = 0) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * 2) | (uintptr_t)(extra * 2);
  return bits % 16 == 0 ? 16 : 2;
}

}  // namespace

int k_parts_of(int64_t M0, int64_t N0, int64_t K0, int64_t M1, int64_t N1, int64_t K1) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || sm_count(dev, &sms) != XKB_OK) sms = 148;
  const int64_t pairs = sms / 2, tiles0 = ceil_div(M0, 256) * ceil_div(N0, 256), kb0 = ceil_div(K0, kBK);
  const int64_t tiles1 = M1 > 0 ? ceil_div(M1, 256) * ceil_div(N1, 256) : 0, kb1 = ceil_div(K1, kBK);
  // K blocks of a pair if all work is dealt out evenly, and of a pair with the most long tiles
  const double even = (double)(tiles0 * kb0 + tiles1 * kb1) / (double)pairs;
  int parts = 1;
  while (parts < 32 && kb0 / (2 * parts) >= 16 && (double)ceil_div(tiles0 * parts, pairs) * ((double)kb0 / parts) > 1.1 * even) parts *= 2;
  return parts;
}

int ce_parts(int64_t M, int64_t N, int64_t K, int* parts) {
  int dev = 0, sms = 0, one = 1;
  XKB_CHECK_CUDA(cudaGetDevice(&dev));
  int rc = sm_count(dev, &sms);
  if (rc != XKB_OK) return rc;
  Shape s;
  rc = shape_of(&M, &N, &K, &one, 1, kCeStats, true, false, dev, sms, &s);
  if (rc != XKB_OK) return rc;
  *parts = (int)(ceil_div(N, s.bn) * (s.split > 1 ? s.bn / 8 : 2));
  return XKB_OK;
}

int64_t ce_most_parts(int64_t M, int64_t N) {
  // shared tiles come in pieces of eight columns, and only tiles of which there are few are shared
  const int64_t own = ceil_div(N, 128) * 2, shared = ceil_div(N, 256) * 32;
  return ceil_div(M, 256) * ceil_div(N, 256) <= 148 ? shared : own;
}

int launch(const Product* products, int count, int end, int dtype, bool chained, bool early_b, cudaStream_t stream) {
  XKB_REQUIRE(count >= 1 && count <= kMaxProblems, "dense products: %d products", count);
  int dev = 0, sms = 0;
  XKB_CHECK_CUDA(cudaGetDevice(&dev));
  int rc = sm_count(dev, &sms);
  if (rc != XKB_OK) return rc;
  Params p = {};
  rc = status_word(dev, &p.status);
  if (rc != XKB_OK) return rc;
  const bool b_mn = products[0].b.k_rows;
  int64_t M[kMaxProblems], N[kMaxProblems], K[kMaxProblems];
  int k_parts[kMaxProblems];
  bool any_a_mn = false, parted = false;
  for (int i = 0; i < count; ++i) {
    M[i] = products[i].M, N[i] = products[i].N, K[i] = products[i].K;
    any_a_mn |= products[i].a.k_rows;
    k_parts[i] = products[i].k_parts > 1 ? products[i].k_parts : 1;
    parted |= k_parts[i] > 1;
    XKB_REQUIRE(M[i] > 0 && N[i] > 0 && K[i] > 0 && M[i] < (1ll << 30) && N[i] < (1ll << 30) && K[i] < (1ll << 30),
                "dense products: sizes out of range");
  }
  const bool two_terms = products[0].a.rest != 0;
  XKB_REQUIRE(!two_terms || (count == 1 && end == kStore && !b_mn && !any_a_mn && M[0] <= 64), "dense products: two terms of this product");
  Shape s;
  rc = shape_of(M, N, K, k_parts, count, end, !any_a_mn && !parted, two_terms, dev, sms, &s);
  if (rc != XKB_OK) return rc;
  const int64_t a_last = M[0] + (end == kStore ? products[0].end.second : 0);      // rows of A that count
  const int a_rows = s.cg == 1 && !any_a_mn && a_last < kRows ? (int)align_up(a_last, 8) : kRows;
  const CUtensorMapDataType dt = dtype == XKB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  p.count = count;
  p.fmt = dtype == XKB_BF16 ? 1 : 0;
  p.split = s.split;
  p.fold = two_terms ? a_rows : 0;
  p.a_bytes = a_rows * 128 * (two_terms ? 2 : 1);
  p.early_b = early_b ? 1 : 0;
  const int read_warps = s.cg == 2 ? 8 : single_warps(end);
  if (s.cg == 1) {      // a stage's place for A is as large as its rows
    const int ring = read_warps == 4 ? Cfg<1, 128, 4, kStore>::kRing : Cfg<1, 128, 8, kCeStats>::kRing;
    p.a_slot = (int)align_up(p.a_bytes, 1024);
    p.stages = ring / ((p.a_slot + s.bn * 128));
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    // An MMA reads 128 rows of A whatever its place holds (the rows behind the last make rows of D that nothing reads), and
    // has to stay within the ring.
    while (p.stages > 1 && (p.stages - 1) * (p.a_slot + s.bn * 128) + kABytes > ring) --p.stages;
  }
  int64_t tiles = 0;
  const int tile_m = kRows * s.cg, tile_n = end == kSwiglu ? s.bn / 2 : s.bn;
  for (int i = 0; i < count; ++i) {
    const Product& q = products[i];
    DevProduct& d = p.prod[i];
    if (two_terms)
      rc = make_map_3d_pitched(&p.a[i], dt, q.a.base, 2, q.a.rows, q.a.cols, (uint64_t)q.a.rest * 2, (uint64_t)q.a.pitch * 2, 2, a_rows, 64,
                               CU_TENSOR_MAP_SWIZZLE_128B, "left operand");
    else
      rc = make_map_2d_pitched(&p.a[i], dt, q.a.base, q.a.rows, q.a.cols, (uint64_t)q.a.pitch * 2, q.a.k_rows ? 64 : a_rows, 64,
                             CU_TENSOR_MAP_SWIZZLE_128B, "left operand");
    if (rc != XKB_OK) return rc;
    if (end == kSwiglu)      // gate rows and up rows are planes
      rc = make_map_3d_pitched(&p.b[i], dt, q.b.base, 2, q.N, q.b.cols, (uint64_t)q.N * q.b.pitch * 2, (uint64_t)q.b.pitch * 2, 2 / s.cg,
                               s.bn / 2, 64, CU_TENSOR_MAP_SWIZZLE_128B, "right operand");
    else
      rc = make_map_2d_pitched(&p.b[i], dt, q.b.base, q.b.rows, q.b.cols, (uint64_t)q.b.pitch * 2, b_mn ? 64 : s.bn / s.cg, 64,
                               CU_TENSOR_MAP_SWIZZLE_128B, "right operand");
    if (rc != XKB_OK) return rc;
    d.M = (int)q.M, d.N = (int)q.N, d.K = (int)q.K, d.b_row0 = (int)q.b.row0;
    d.live = q.live;
    d.live_is_k = d.a_mn = q.a.k_rows;
    d.group = 16;
    d.k_parts = q.k_parts > 1 ? q.k_parts : 1;
    d.end = q.end;
    d.end.vec_out = vec_of(q.end.out, q.end.ld, end == kDswiglu ? q.end.half : 0);
    // whole tiles of pairs, in the order of the rows
    d.end.tma_out = s.split == 1 && s.cg == 2 && d.end.vec_out == 16 && q.end.row_map == nullptr && !q.end.acc_out && !q.end.acc_in &&
                    (end == kStore || end == kCeGrad);
    if (d.end.tma_out) {
      rc = make_map_2d_pitched(&p.out[i], dt, q.end.out, end == kCeGrad ? align_up(q.M, 256) : q.M, q.N, (uint64_t)q.end.ld * 2, 32, 64,
                               CU_TENSOR_MAP_SWIZZLE_128B, "result");
      if (rc != XKB_OK) return rc;
    }
    d.end.vec_h = vec_of(q.end.h, q.end.ld_h);
    d.end.vec_gu = vec_of(q.end.gate_up, q.end.ld_gu, q.end.half);
    tiles += ceil_div(q.M, tile_m) * ceil_div(q.N, tile_n) * d.k_parts;
  }
  XKB_REQUIRE(tiles < (1ll << 31), "dense products: too many tiles");
  Launch l;
  l.dev = dev, l.cg = s.cg, l.bn = s.bn, l.split = s.split, l.chained = chained, l.stream = stream;
  const int margin = g_sm_margin.load(std::memory_order_relaxed);
  if (s.split > 1 || two_terms) {
    XKB_REQUIRE(tiles * s.split * s.cg < (1ll << 31), "dense products: too many tiles");
    l.grid = (int)(tiles * s.split * s.cg);     // one tile a cluster
  } else {
    int64_t most = (sms - margin) / s.cg * (read_warps == 4 ? 2 : 1);
    if (most < 1) most = 1;
    l.grid = (int)(tiles < most ? tiles : most) * s.cg;
  }
  if (end == kStore) {
    bool long_sums = false;
    for (int i = 0; i < count; ++i) long_sums |= ceil_div(ceil_div(K[i], kBK), k_parts[i]) > kLongBlocks;
    // (a kernel of its own: with its registers the ordinary one took 5 % longer, 509 x 4096 x 1416 backward 51.7 -> 54.7 us)
    return long_sums && s.cg == 2 && s.split == 1 && products[0].end.second == 0 ? run_store_long(b_mn, p, l) : run_store(b_mn, p, l);
  }
  if (end == kSwiglu || end == kDswiglu) return run_ffn(end, p, l);
  return run_ce(end, p, l);
}

}  // namespace dense
}  // namespace xkb

namespace xkb {
namespace {

// Matrices laid out once more with rows of whole 16 bytes: a warp copies 256 elements of a row at a time, lane = column, since
// rows start anywhere.  Bound by latency where they are small (why all operands of a call go in one launch), else by memory.
struct LayOut {
  const uint16_t* from[XKB_LAY_OUT_MOST];
  uint16_t* to[XKB_LAY_OUT_MOST];
  int64_t ld[XKB_LAY_OUT_MOST], cols[XKB_LAY_OUT_MOST], first[XKB_LAY_OUT_MOST + 1];      // first: number of its first piece
  int exponent[XKB_LAY_OUT_MOST];      // bits of it: infinities and NaN, which have them all, become 0 (0: they stay)
  int count;
};
constexpr int kPiece = 256;

__global__ void __launch_bounds__(256) lay_out_kernel(const LayOut a) {
  const int lane = threadIdx.x & 31;
  for (int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); u < a.first[a.count]; u += (int64_t)gridDim.x * 8) {
    int i = 0;
    while (i + 1 < a.count && u >= a.first[i + 1]) ++i;
    const int64_t cols = a.cols[i], pieces = (cols + kPiece - 1) / kPiece, v = u - a.first[i];
    const int all = a.exponent[i];
    const int64_t row = v / pieces, c0 = (v - row * pieces) * kPiece, ld_to = (cols + 7) / 8 * 8;
    const uint16_t* from = a.from[i] + row * a.ld[i];
    uint16_t* to = a.to[i] + row * ld_to;
    uint16_t x[kPiece / 32];
#pragma unroll
    for (int j = 0; j < kPiece / 32; ++j) {
      const int64_t c = c0 + j * 32 + lane;
      x[j] = c < cols ? from[c] : (uint16_t)0;
    }
#pragma unroll
    for (int j = 0; j < kPiece / 32; ++j) {
      const int64_t c = c0 + j * 32 + lane;
      if (c < cols) to[c] = all != 0 && (x[j] & all) == all ? (uint16_t)0 : x[j];
    }
  }
}

}  // namespace

int dense::lay_out(const void* const* from_host, const int64_t* ld_host, const int64_t* rows_host, const int64_t* cols_host,
                   void* const* to_host, const int* exponent_host, int count, cudaStream_t stream) {
  XKB_REQUIRE(count >= 0 && count <= XKB_LAY_OUT_MOST, "lay_out_rows: %d matrices", count);
  XKB_REQUIRE(count == 0 || (from_host != nullptr && ld_host != nullptr && rows_host != nullptr && cols_host != nullptr && to_host != nullptr),
              "lay_out_rows: null array");
  LayOut a = {};
  int64_t pieces = 0;
  for (int i = 0; i < count; ++i) {
    XKB_REQUIRE(rows_host[i] >= 0 && rows_host[i] < (1ll << 28) && cols_host[i] >= 1 && cols_host[i] < (1ll << 24) && ld_host[i] >= 0 &&
                    ld_host[i] < (1ll << 32), "lay_out_rows: sizes out of range");
    XKB_REQUIRE(rows_host[i] == 0 || (from_host[i] != nullptr && to_host[i] != nullptr && address_bits(from_host[i], to_host[i]) % 2 == 0),
                "lay_out_rows: null or misaligned matrix");
    a.from[i] = static_cast<const uint16_t*>(from_host[i]);
    a.to[i] = static_cast<uint16_t*>(to_host[i]);
    a.ld[i] = ld_host[i], a.cols[i] = cols_host[i];
    a.exponent[i] = exponent_host != nullptr ? exponent_host[i] : 0;
    a.first[i] = pieces;
    pieces += rows_host[i] * ceil_div(cols_host[i], kPiece);
  }
  a.first[count] = pieces;
  a.count = count;
  if (pieces == 0) return XKB_OK;
  const int64_t blocks = ceil_div(pieces, 8);
  lay_out_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, stream>>>(a);
  XKB_CHECK_LAUNCH("lay_out_kernel");
  return XKB_OK;
}

}  // namespace xkb

extern "C" int xkb_lay_out_rows(const void* const* from_host, const int64_t* ld_host, const int64_t* rows_host, const int64_t* cols_host,
                                void* const* to_host, int count, void* stream_) {
  return xkb::dense::lay_out(from_host, ld_host, rows_host, cols_host, to_host, nullptr, count, static_cast<cudaStream_t>(stream_));
}

extern "C" int xkb_dense_status(void* stream_) {
  using namespace xkb;
  int dev = 0;
  XKB_CHECK_CUDA(cudaGetDevice(&dev));
  int* word = nullptr;
  const int rc = dense::status_word(dev, &word);
  if (rc != XKB_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int host = 0;
  XKB_CHECK_CUDA(cudaMemcpyAsync(&host, word, sizeof(int), cudaMemcpyDeviceToHost, stream));
  XKB_CHECK_CUDA(cudaStreamSynchronize(stream));
  if (host != 0) {
    XKB_CHECK_CUDA(cudaMemsetAsync(word, 0, sizeof(int), stream));     // reported once
    return fail(XKB_ERR_DEVICE, "a kernel of a dense product gave up a bounded wait: status 0x%x (wait site %d)", host, host >> 8);
  }
  return XKB_OK;
}
