// The kernel of the dense products (dense.h): D = A B^T on tcgen05 with fp32 accumulators in tensor memory.
//
// A tile is 128 rows of D per CTA and BN columns; with CG = 2 the two CTAs of a pair hold 128 rows of A and half of the
// columns' rows of B each and one instruction multiplies both halves, so that every SM loads half of B.  Warps: one feeds
// stages of 64 K by TMA, one issues the MMAs, two warpgroups read accumulators out while the next tile is multiplied
// (two accumulator sets).  CTAs (pairs) are persistent and take tiles in turn.  Where there are few tiles (CG = 1), up to
// eight CTAs of a cluster share one: each multiplies a part of K, and adds up a part of the columns in the order of the CTAs.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "dense.h"
#include "softmax_dev.cuh"
#include "tc_common.cuh"

namespace xkb {
namespace dense {

constexpr int kBK = 64;             // K of a stage: 128 bytes, one swizzle row
constexpr int kRows = 128;          // rows of D per CTA
constexpr int kControlWarps = 4;    // 0: TMA of A, 1: MMA, 2: tensor memory, 3: TMA of B; the read-out warps follow
constexpr int kMaxStages = 12;
constexpr int kABytes = kRows * 128;
constexpr int kBoxBytes = 64 * 128;  // a box of 64 K rows by 64 elements
// The tensor cores cut off what an fp32 accumulator cannot hold instead of rounding it, at each step of 16 K, so a long sum
// drifts towards 0 in proportion to K (losses of many rows were 1.4e-6 off at K = 2048).  Logits stay fp32, in the statistics
// (kCeStats) as in their gradient (kCeGrad: d of a token that the head is sure of is a difference of numbers close to 1), so an
// accumulator of theirs takes kPartBlocks of 64 K, and the read-out adds them up in registers while the next is filled.  Error of losses
// in the norm, 4096 x 7168 x 128000 in pairs by 512 / 256 K: 4.0e-7 / 2.1e-7 (an fp32 product on the ordinary cores: 1.1e-6), but 3 to
// 20 % more time, for the read-out of short parts outlasts their MMAs.  Single CTAs, which take up to 128 rows, wait for the
// weight's bytes, and a single row's small loss takes the drift of its largest logit whole: 1 x 4096 x 50001 by 512 / 128 / 64 K
// 2.7e-6 / 8.6e-8 / 1.1e-6 (one number; the ordinary cores' 9.2e-8) in 91 / 92 / 99 us, 128 x 7168 x 32001 4.5e-7 / 1.8e-7 / 2.0e-7 in
// 99 / 99 / 103.  Logits of terms of one sign in the gradient, fp16, in 2^-23 of them: one accumulator of 1024 / 4096 K 44 / 194 off, in
// parts of 512 K 20, of 128 K 3; 4096 x 7168 x 16384 backward 1850 -> 1860 us, 509 x 2048 x 50001 255 -> 262, 77 x 2056 x 32001 130.
// Stored results are rounded to 16 bits, and only sums far longer than a layer is wide drift as far as that: sums over rows of
// one sign lost 6e-9 of themselves a row (1.6e-3 of 2^18 rows in fp16, whose half step is 4.9e-4).  Pairs add sums of more than 16384 K
// up in parts of that the same way (kStoreLong), and single CTAs are not given them.  Other ends contract over a layer's width H,
// in one accumulator.
constexpr int kLongBlocks = 256;
template <int END> constexpr bool kStores = END == kStore || END == kStoreLong;
template <int END> constexpr bool kInParts = END == kCeStats || END == kCeGrad || END == kStoreLong;
template <int END, int CG> constexpr int kPartBlocks = END == kStoreLong ? kLongBlocks : CG == 1 ? 2 : 8;
template <int END, int CG> __device__ __forceinline__ int parts_of(int kb) {      // no blocks are one part too
  return kInParts<END> && kb > 0 ? (kb + kPartBlocks<END, CG> - 1) / kPartBlocks<END, CG> : 1;
}

struct DevProduct {
  int M, N, K, b_row0;
  const int32_t* live;
  int live_is_k, a_mn;
  int group;          // row tiles that are walked side by side
  int k_parts;
  End end;
};

// (What a kernel needs first stands first: a line of parameters that nobody has touched yet is a trip to L2.)
struct Params {
  int count, fmt;       // fmt: 1 bf16, 0 fp16
  int split;            // CTAs (pairs) of a cluster that share a tile, a part of K each
  int a_bytes;          // bytes of A that a stage loads
  int a_slot, stages;   // CG = 1: bytes that a stage has for A, stages
  int early_b;
  int fold;             // CG = 1, kStore: A comes in two terms, row r of the second is row fold + r of the tile (0: one term)
  int* status;
  DevProduct prod[kMaxProblems];
  CUtensorMap a[kMaxProblems], b[kMaxProblems], out[kMaxProblems];      // out: where end.tma_out is set
};

// A product in tiles, in shared memory: a role looks a tile up with a handful of loads side by side.
struct Extent {
  int first, m_tiles, n_tiles, kb, rows, k_parts, group;      // first: number of its first tile; kb: stages of K
  uint32_t strip_inv, group_inv, last_inv;
};

struct Shared {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  int abort_flag;
  uint32_t tmem;
  Extent of[kMaxProblems];
  int tiles, long_tiles, delta, rest;
};

// CG: CTAs of a pair; BN: columns of a tile; RW: read-out warps.  RW = 4 leaves room for two CTAs on an SM.
// (Ends with second terms are instances of their own: as a choice within, they cost calls without 1 to 7 %.)
constexpr int end_of(int way) { return way == kDswigluTwo ? kDswiglu : way == kCeGradTwo ? kCeGrad : way; }
template <int CG, int BN, int RW, int WAY> struct Cfg {
  static constexpr int END = end_of(WAY);
  static constexpr int kThreads = 32 * (kControlWarps + RW);
  static constexpr int kCtas = RW == 4 ? 2 : 1;
  static constexpr int kBBytes = BN / CG * 128;
  // a warp's 32 rows of 64 or 128 bytes on their way; kDswiglu: of its result, of gate and of up
  static constexpr int kRowBytes = 32 * 64 * (CG == 1 ? 1 : END == kDswiglu ? 3 : 2);
  static constexpr int kRing = (RW == 4 ? 102 : CG == 1 ? 209 : END == kDswiglu ? 177 : 193) * 1024;
  static constexpr int kStageBytes = kABytes + kBBytes;      // CG = 2
  static constexpr int kStages = kRing / kStageBytes < 8 ? kRing / kStageBytes : 8;
  static constexpr int kSmem = kRing + RW * kRowBytes + 1024;
  static_assert(kRing >= BN * kRows * 4, "the parts of a sum lie where the stages were");
};

// ---- instructions that tc_common.cuh has no form of ----------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to(uint32_t smem_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void remote_arrive(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if constexpr (CG == 2)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y) : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if constexpr (CG == 2)
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// By the lane whose `leader` is not 0; all lanes of the warp call with the same operands.
template <int CG>
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
  else
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
// Arrives on the barrier at this address (in both CTAs of a pair) once the MMAs issued so far are done.
template <int CG> __device__ __forceinline__ void commit(uint32_t leader, uint32_t bar, uint16_t both) {
  if constexpr (CG == 2)
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
                 "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
                 ::"r"(bar), "h"(both), "r"(leader) : "memory");
  else
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(leader) : "memory");
}
// Barriers by their address.  A wait is bounded (tc_common.cuh).
__device__ __forceinline__ bool probe(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
static __device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, tc::Guard g, int where) {
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (probe(bar, parity)) return true;
    if ((i & 63u) == 0u) {
      if (g.aborted()) return false;
      const uint64_t now = tc::globaltimer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > tc::kWaitBudgetNs) break;
    }
  }
  g.raise(tc::kErrWaitTimeout + (where << 8));
  return false;
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, const tc::Guard& g, int where) {
  return probe(bar, parity) || wait_slow(bar, parity, g, where);
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
template <int CG> __device__ __forceinline__ void tmem_alloc(uint32_t* result, uint32_t cols) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(result)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tc::tmem_alloc(result, cols);
  }
}
template <int CG> __device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
  else
    tc::tmem_dealloc(addr, cols);
}
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[16]) { tc::tmem_ld_32x16(addr, reinterpret_cast<uint32_t(&)[16]>(v)); }
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Operand in shared memory, 128-byte swizzle.  K contiguous: rows of 64 K, groups of eight rows 1024 bytes apart.  Own
// index contiguous: boxes of 64 elements by 64 K rows, 8192 bytes from box to box, groups of eight K rows 1024 apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool k_rows) {
  const uint64_t lbo = k_rows ? (kBoxBytes >> 4) : 1;
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (lbo << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// ---- 16-bit rows ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pack16(int fmt, float lo, float hi) {
  if (fmt) return pack_bf16(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void unpack16(int fmt, uint32_t p, float& lo, float& hi) {
  if (fmt) {
    lo = __uint_as_float(p << 16);
    hi = __uint_as_float(p & 0xFFFF0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
    lo = f.x;
    hi = f.y;
  }
}
// CW consecutive elements of a row, the first n of which exist; vec: what the addresses allow.
template <int CW> __device__ __forceinline__ void store_row(void* base, int64_t at, const uint32_t (&w)[CW / 2], int n, int vec) {
  uint16_t* p = static_cast<uint16_t*>(base) + at;
  if (n >= CW && vec >= 16) {
#pragma unroll
    for (int i = 0; i < CW / 2; i += 4) *reinterpret_cast<uint4*>(p + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < CW; ++i)
      if (i < n) p[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}
template <int CW> __device__ __forceinline__ void load_row(const void* base, int64_t at, uint32_t (&w)[CW / 2], int n, int vec) {
  const uint16_t* p = static_cast<const uint16_t*>(base) + at;
  if (n >= CW && vec >= 16) {
#pragma unroll
    for (int i = 0; i < CW / 2; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 2 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < CW; i += 2)
      w[i / 2] = (i < n ? (uint32_t)p[i] : 0u) | (i + 1 < n ? (uint32_t)p[i + 1] << 16 : 0u);
  }
}

// 64 bytes of 32 rows, lane = row, to memory: through shared memory, so that four lanes write a row's 64 bytes side by side
// (a lane that writes its own row touches one sector of 32 lines an instruction).  to: this lane's row, 16-byte aligned;
// nullptr: not written.  All lanes of the warp call.
__device__ __forceinline__ uint32_t rows_at(uint32_t buf, int row, int unit) { return buf + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4); }
__device__ __forceinline__ void rows_out(uint32_t buf, void* to, const uint32_t* w) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                 ::"r"(rows_at(buf, lane, u)), "r"(w[4 * u]), "r"(w[4 * u + 1]), "r"(w[4 * u + 2]), "r"(w[4 * u + 3]) : "memory");
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 8 + (lane >> 2);
    char* p = reinterpret_cast<char*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(to), row));
    const uint4 v = tc::lds128(rows_at(buf, row, lane & 3));
    if (p != nullptr) *reinterpret_cast<uint4*>(p + (lane & 3) * 16) = v;
  }
  __syncwarp();
}
// The first half of rows_in: starts copies of the rows into the buffer that nothing waits for yet.
__device__ __forceinline__ void rows_start(uint32_t buf, const void* from) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 8 + (lane >> 2);
    const char* p = reinterpret_cast<const char*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(from), row));
    if (p != nullptr)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(rows_at(buf, row, lane & 3)), "l"(p + (lane & 3) * 16) : "memory");
  }
}
__device__ __forceinline__ void rows_take(uint32_t buf, uint32_t* w) {      // of rows that have arrived
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const uint4 x = tc::lds128(rows_at(buf, lane, u));
    w[4 * u] = x.x, w[4 * u + 1] = x.y, w[4 * u + 2] = x.z, w[4 * u + 3] = x.w;
  }
}
__device__ __forceinline__ void rows_in(uint32_t buf, const void* from, uint32_t* w) {
  const int lane = threadIdx.x & 31;
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const char* p = reinterpret_cast<const char*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(from), i * 8 + (lane >> 2)));
    v[i] = p != nullptr ? *reinterpret_cast<const uint4*>(p + (lane & 3) * 16) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                 ::"r"(rows_at(buf, i * 8 + (lane >> 2), lane & 3)), "r"(v[i].x), "r"(v[i].y), "r"(v[i].z), "r"(v[i].w) : "memory");
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const uint4 x = tc::lds128(rows_at(buf, lane, u));
    w[4 * u] = x.x, w[4 * u + 1] = x.y, w[4 * u + 2] = x.z, w[4 * u + 3] = x.w;
  }
  __syncwarp();
}
// The same for rows that start anywhere and for the last n columns: a row at a time, lane = column.
__device__ __forceinline__ void rows_out_any(uint32_t buf, uint16_t* to, const uint32_t* w, int n) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                 ::"r"(rows_at(buf, lane, u)), "r"(w[4 * u]), "r"(w[4 * u + 1]), "r"(w[4 * u + 2]), "r"(w[4 * u + 3]) : "memory");
  __syncwarp();
#pragma unroll 8
  for (int row = 0; row < 32; ++row) {
    uint16_t* p = reinterpret_cast<uint16_t*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(to), row));
    const uint32_t v = tc::lds16(rows_at(buf, row, lane >> 3) + (lane & 7) * 2);
    if (p != nullptr && lane < n) p[lane] = (uint16_t)v;
  }
  __syncwarp();
}
__device__ __forceinline__ void rows_in_any(uint32_t buf, const uint16_t* from, uint32_t* w, int n) {
  const int lane = threadIdx.x & 31;
#pragma unroll 8
  for (int row = 0; row < 32; ++row) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(from), row));
    const uint16_t v = p != nullptr && lane < n ? p[lane] : (uint16_t)0;
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(rows_at(buf, row, lane >> 3) + (lane & 7) * 2), "h"(v) : "memory");
  }
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const uint4 x = tc::lds128(rows_at(buf, lane, u));
    w[4 * u] = x.x, w[4 * u + 1] = x.y, w[4 * u + 2] = x.z, w[4 * u + 3] = x.w;
  }
  __syncwarp();
}
// 16-bit results of 64 columns leave by a copy of their own: the lanes write their rows, halves of 32 columns, into 128-byte
// rows (128-byte swizzle), and one lane starts the copy, which the warp does not wait for until the buffer's next use.
// Full lines reach L2: the products of a head's gradient at 509 x 2048 x 50001, 168 -> 151 us.
__device__ __forceinline__ void half_rows(uint32_t buf, int half, const uint32_t* w) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                 ::"r"(buf + lane * 128 + (((half * 4 + u) ^ (lane & 7)) << 4)), "r"(w[4 * u]), "r"(w[4 * u + 1]), "r"(w[4 * u + 2]),
                   "r"(w[4 * u + 3]) : "memory");
}
__device__ __forceinline__ void rows_copied() {      // what was started has left shared memory
  if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void copy_rows(uint32_t buf, const CUtensorMap* map, int x, int y) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(buf), "r"(x), "r"(y) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
// CW columns of this lane's row: pieces of 32 together, smaller ones each lane its own.
template <int CW>
__device__ __forceinline__ void put_row(uint32_t buf, void* base, int64_t at, bool live, const uint32_t (&w)[CW / 2], int n, int vec) {
  uint16_t* to = live ? static_cast<uint16_t*>(base) + at : nullptr;
  if (CW == 32 && n >= CW && vec >= 16) rows_out(buf, to, w);
  else if (CW == 32) rows_out_any(buf, to, w, n);
  else if (live) store_row<CW>(base, at, w, n, vec);
}
template <int CW>
__device__ __forceinline__ void get_row(uint32_t buf, const void* base, int64_t at, bool live, uint32_t (&w)[CW / 2], int n, int vec) {
  const uint16_t* from = live ? static_cast<const uint16_t*>(base) + at : nullptr;
  if (CW == 32 && n >= CW && vec >= 16) rows_in(buf, from, w);
  else if (CW == 32) rows_in_any(buf, from, w, n);
  else if (live) load_row<CW>(base, at, w, n, vec);
}

// What a rounding to `hi` left of x; nothing of an infinity or a NaN (hi holds it).
__device__ __forceinline__ float finite_rest(float x, float hi) { return fabsf(hi) < INFINITY ? x - hi : 0.f; }
// The sum of first terms and that of second ones; not beside an infinity, for an infinite factor has made them infinite too, of either sign,
// or a NaN.
__device__ __forceinline__ float add_second(float first, float second) { return fabsf(first) < INFINITY ? first + second : first; }
// Two values rounded.  TWO: rows second .. 2 second of a warp's 32 become what the rounding of the rows `second` before them left.
template <bool TWO> __device__ __forceinline__ uint32_t pack_terms(int fmt, int second, int row, float x0, float x1) {
  const uint32_t o = pack16(fmt, x0, x1);
  if constexpr (TWO) {
    float h0, h1;
    unpack16(fmt, o, h0, h1);
    const uint32_t rest = __shfl_sync(~0u, pack16(fmt, finite_rest(x0, h0), finite_rest(x1, h1)), (threadIdx.x & 31) - second);
    return row >= second && row < 2 * second ? rest : o;
  }
  return o;
}
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + exp2_fast(-kLog2e * x)); }

// ---- what becomes of CW columns of a row ---------------------------------------------------------------------
struct RowState {
  float m, s;       // kCeStats: maximum so far, sum of exponentials against it
  int label;        // column of the label within the piece
  float4 coef;      // kCeGrad
  int64_t to;       // kStore: row of `out`
  int half;         // of 64 columns that leave together
  bool here;        // kDswiglu: gate and up of the piece are in the buffers behind `buf`
  const uint16_t* next;   // gate of the next piece (nullptr: none that is copied ahead)
};

template <int END> __device__ __forceinline__ void row_begin(const End& e, int row, bool live, RowState& st) {
  if constexpr (END == kCeStats || END == kCeGrad) {
    st.m = -INFINITY;
    st.s = 0.f;
    st.label = -1;
    if (live) {
      if (END == kCeStats && e.labels64 != nullptr) {
        const int64_t label = e.labels64[row];
        st.label = label >= 0 && label < (1ll << 30) ? (int)label : -1;
      } else {
        st.label = e.labels[row] - e.col0;
      }
    }
    if constexpr (END == kCeGrad) st.coef = live ? e.coef[row] : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if constexpr (kStores<END>) st.to = live && e.row_map != nullptr ? e.row_map[row] : row;
}
template <int END> __device__ __forceinline__ void row_end(const End& e, int row, bool live, int part, const RowState& st) {
  if constexpr (END == kCeStats)
    if (live) e.part[(int64_t)row * e.part_ld + part] = make_float2(st.m, st.s);
}

// v: columns col .. col + CW of D (kSwiglu: of gate, w: of up), n of which exist
template <int END, bool TWO, int CW>
__device__ __forceinline__ void row_piece(const End& e, int fmt, uint32_t buf, int row, bool live, int kpart, int col, int n, float scale, float (&v)[CW],
                                          float (&w)[CW], RowState& st) {
  uint32_t o[CW / 2];
  if constexpr (kStores<END>) {
    if (END == kStore && e.second != 0) {
#pragma unroll
      for (int j = 0; j < CW; ++j) v[j] = add_second(v[j], __shfl_down_sync(~0u, v[j], e.second));
    }
    if (e.acc_in || e.acc_out) {
      float* acc = e.acc + kpart * e.acc_part + (int64_t)row * e.acc_ld + col;
      constexpr int kHalf = CW == 32 ? 16 : CW;
#pragma unroll
      for (int h = 0; h < CW; h += kHalf) {
        if (e.acc_in) {
          uint32_t f[16];
          if constexpr (CW == 32) {
            rows_in(buf, live ? acc + h : nullptr, f);
          } else {
#pragma unroll
            for (int j = 0; j < kHalf; ++j) f[j] = live ? __float_as_uint(acc[j]) : 0u;
          }
#pragma unroll
          for (int j = 0; j < kHalf; ++j) v[h + j] += __uint_as_float(f[j]);
        }
        if (e.acc_out) {
          if constexpr (CW == 32) rows_out(buf, live ? acc + h : nullptr, reinterpret_cast<const uint32_t*>(v + h));
          else if (live)
#pragma unroll
            for (int j = 0; j < kHalf; ++j) acc[j] = v[j];
        }
      }
      if (e.acc_out) return;
    }
    if (scale != 1.f) {
#pragma unroll
      for (int j = 0; j < CW; ++j) v[j] *= scale;
    }
#pragma unroll
    for (int j = 0; j < CW; j += 2) o[j / 2] = pack16(fmt, v[j], v[j + 1]);
    if (CW == 32 && e.tma_out) {
      if (st.half == 0) rows_copied();
      half_rows(buf, st.half, o);
    } else {
      put_row<CW>(buf, e.out, st.to * e.ld + col, live, o, n, e.vec_out);
    }
  } else if constexpr (END == kSwiglu) {
    if (e.gate_up != nullptr) {
#pragma unroll
      for (int j = 0; j < CW; j += 2) o[j / 2] = pack16(fmt, v[j], v[j + 1]);
      put_row<CW>(buf, e.gate_up, (int64_t)row * e.ld_gu + col, live, o, n, e.vec_gu);
#pragma unroll
      for (int j = 0; j < CW; j += 2) o[j / 2] = pack16(fmt, w[j], w[j + 1]);
      put_row<CW>(buf, e.gate_up, (int64_t)row * e.ld_gu + e.half + col, live, o, n, e.vec_gu);
    }
    if (e.h == nullptr) return;
#pragma unroll
    for (int j = 0; j < CW; j += 2) {
      float h[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float g = v[j + i], u = w[j + i];
        if (e.limit > 0.f) {      // (a NaN stays one)
          g = g > e.limit ? e.limit : g;
          u = u > e.limit ? e.limit : u < -e.limit ? -e.limit : u;
        }
        h[i] = g * sigmoid(g) * u;
      }
      v[j] = h[0], v[j + 1] = h[1];
      o[j / 2] = pack16(fmt, h[0], h[1]);
    }
    put_row<CW>(buf, e.h, (int64_t)row * e.ld_h + col, live, o, n, e.vec_h);
    if (e.h_rest != nullptr) {
#pragma unroll
      for (int j = 0; j < CW; j += 2) {
        float hi[2];
        unpack16(fmt, o[j / 2], hi[0], hi[1]);
        o[j / 2] = pack16(fmt, finite_rest(v[j], hi[0]), finite_rest(v[j + 1], hi[1]));
      }
      put_row<CW>(buf, e.h_rest, (int64_t)row * e.ld_h + col, live, o, n, e.vec_h);
    }
  } else if constexpr (END == kDswiglu) {
    uint32_t ug[CW / 2], uu[CW / 2];
    const int64_t half = e.half;
    if (CW == 32 && st.here) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      rows_take(buf + 2048, ug);
      rows_take(buf + 4096, uu);
      __syncwarp();
      if (st.next != nullptr) {      // (the same in all lanes but for rows that are none)
        rows_start(buf + 2048, live ? st.next : nullptr);
        rows_start(buf + 4096, live ? st.next + half : nullptr);
      }
    } else {
      get_row<CW>(buf, e.gate_up, (int64_t)row * e.ld_gu + col, live, ug, n, e.vec_gu);
      get_row<CW>(buf, e.gate_up, (int64_t)row * e.ld_gu + half + col, live, uu, n, e.vec_gu);
    }
#pragma unroll
    for (int j = 0; j < CW; j += 2) {
      float g[2], u[2], dg[2], du[2], h[2];
      unpack16(fmt, ug[j / 2], g[0], g[1]);
      unpack16(fmt, uu[j / 2], u[0], u[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float gc = g[i], uc = u[i];
        if (e.limit > 0.f) {
          gc = gc > e.limit ? e.limit : gc;
          uc = uc > e.limit ? e.limit : uc < -e.limit ? -e.limit : uc;
        }
        const float s = sigmoid(gc), gs = gc * s, d = v[j + i];
        dg[i] = d * uc * (s + gs * (1.f - s));
        du[i] = d * gs;
        h[i] = gs * uc;
        if (e.limit > 0.f) {
          if (g[i] > e.limit) dg[i] = 0.f;
          if (fabsf(u[i]) > e.limit) du[i] = 0.f;
        }
      }
      o[j / 2] = pack_terms<TWO>(fmt, e.second, row, h[0], h[1]);
      ug[j / 2] = pack_terms<TWO>(fmt, e.second, row, dg[0], dg[1]);
      uu[j / 2] = pack_terms<TWO>(fmt, e.second, row, du[0], du[1]);
    }
    const bool kept = live || (TWO && row < 2 * e.second);
    put_row<CW>(buf, e.out, (int64_t)row * e.ld + col, kept, ug, n, e.vec_out);
    put_row<CW>(buf, e.out, (int64_t)row * e.ld + half + col, kept, uu, n, e.vec_out);
    if (e.h != nullptr) put_row<CW>(buf, e.h, (int64_t)row * e.ld_h + col, kept, o, n, e.vec_h);
  } else if constexpr (END == kCeStats) {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < CW; ++j) {
      if (j >= n) v[j] = -INFINITY;
      top = fmaxf(top, v[j]);
    }
    if (top > st.m) {
      st.s *= exp2_fast((st.m - top) * kLog2e);
      st.m = top;
    }
    const float ref = st.m == -INFINITY ? 0.f : st.m;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < CW; j += 2) {
      s0 += exp2_fast((v[j] - ref) * kLog2e);
      s1 += exp2_fast((v[j + 1] - ref) * kLog2e);
    }
    st.s += s0 + s1;
    const int at = st.label - col;
    if (at >= 0 && at < n && at < CW) {
      float x = v[0];
#pragma unroll
      for (int j = 1; j < CW; ++j)
        if (j == at) x = v[j];
      e.given[row] = x;
    }
  } else {
    const float4 c = st.coef;
    const int at = st.label - col;
#pragma unroll
    for (int j = 0; j < CW; j += 2) {
      float d[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        d[i] = exp2_fast(((v[j + i] - c.x) - c.y) * kLog2e) * c.z;
        if (j + i == at) d[i] -= c.w;
        if (!live) d[i] = 0.f;
      }
      o[j / 2] = pack_terms<TWO>(fmt, e.second, row, d[0], d[1]);
    }
    if (CW == 32 && e.tma_out) {
      if (st.half == 0) rows_copied();
      half_rows(buf, st.half, o);
    } else {
      put_row<CW>(buf, e.out, (int64_t)row * e.ld + col, true, o, n, e.vec_out);
    }
  }
}

// ---- the kernel ----------------------------------------------------------------------------------------------
struct Tile { int prod, m, n, kpart, rows, k0, k1; };      // rows: of the product; k0, k1: blocks of K

// n / d by a multiplication: inv = (2^32 - 1) / d, at most one too small before the correction
__device__ __forceinline__ int quotient(int n, int d, uint32_t inv) {
  const int q = (int)__umulhi((uint32_t)n, inv);
  return n - q * d >= d ? q + 1 : q;
}
__device__ __forceinline__ uint32_t inverse(int d) { return d > 0 ? 0xFFFFFFFFu / (uint32_t)d : 0u; }

// The tiles of a cluster in turn: first its share of the long ones (of the first product), every `clusters`-th; then of the
// others, where the clusters that have one long tile more than the rest stay out of the first `delta` rounds.
struct Walk {
  int cluster, clusters, t, round;
  __device__ __forceinline__ void place(const Shared& sh) {
    const int few = clusters - sh.rest;
    t = sh.long_tiles + (round < sh.delta ? round * few + cluster - sh.rest
                                          : sh.delta * few + (round - sh.delta) * clusters + cluster);
  }
  __device__ __forceinline__ Walk(const Shared& sh, int cluster_, int clusters_) : cluster(cluster_), clusters(clusters_), t(cluster_), round(-1) {
    if (t >= sh.long_tiles) start(sh);
  }
  __device__ __forceinline__ void start(const Shared& sh) {
    round = cluster < sh.rest ? sh.delta : 0;
    place(sh);
  }
  __device__ __forceinline__ void next(const Shared& sh) {
    if (round < 0) {
      t += clusters;
      if (t >= sh.long_tiles) start(sh);
    } else {
      ++round;
      place(sh);
    }
  }
  __device__ __forceinline__ bool get(const Shared& sh, Tile& out) const {
    if (t >= sh.tiles) return false;
    const int q = (t >= sh.of[1].first) + (t >= sh.of[2].first);
    const Extent e = sh.of[q];
    int r = t - e.first;
    out.prod = q;
    out.kpart = 0;
    if (e.k_parts > 1) {
      const int each = e.n_tiles * e.m_tiles;
      out.kpart = r / each, r -= out.kpart * each;
    }
    const int strip = e.group * e.n_tiles;
    const int g = quotient(r, strip, e.strip_inv), in = r - g * strip, left = e.m_tiles - g * e.group;
    const int wide = left < e.group ? left : e.group;
    out.n = quotient(in, wide, left < e.group ? e.last_inv : e.group_inv);
    out.m = g * e.group + (in - out.n * wide);
    out.rows = e.rows;
    out.k0 = 0, out.k1 = e.kb;
    if (e.k_parts > 1) out.k0 = e.kb * out.kpart / e.k_parts, out.k1 = e.kb * (out.kpart + 1) / e.k_parts;
    return true;
  }
};

template <int CG, int BN, int RW, bool BMN, int WAY>
__global__ void __launch_bounds__(Cfg<CG, BN, RW, WAY>::kThreads, Cfg<CG, BN, RW, WAY>::kCtas) dense_kernel(const __grid_constant__ Params p) {
  using C = Cfg<CG, BN, RW, WAY>;
  constexpr int END = C::END;
  constexpr bool kTwo = WAY != END;
  constexpr bool kPaired = END == kSwiglu;
  constexpr int kTileN = kPaired ? BN / 2 : BN;    // columns of the result
  constexpr int kTmemCols = 2 * BN;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  const uint32_t ring = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int split = p.split, width = CG * split;   // width: CTAs of a cluster
  const int fold = CG == 1 && END == kStore && !BMN ? p.fold : 0;
  const bool parked = split > 1 || fold != 0;      // sums are put together in shared memory
  const uint32_t rank = width > 1 ? cluster_rank() : 0;
  const int part = (int)rank / CG, half = (int)rank % CG, first_rank = (int)rank - half;   // of K; of the tile's rows
  const int cluster = blockIdx.x / width, clusters = gridDim.x / width;
  const uint32_t stages = CG == 2 ? C::kStages : p.stages, a_slot = CG == 2 ? kABytes : p.a_slot;
  const uint32_t stage_bytes = a_slot + C::kBBytes;
  tc::Guard guard{&sh.abort_flag, p.status};

  if (!p.early_b) chain_wait();
  chain_trigger();
  if (warp == 0) {
    if (lane == 0) {
      sh.abort_flag = 0;
      for (uint32_t s = 0; s < stages; ++s) {
        tc::mbar_init(&sh.full[s], 1);
        tc::mbar_init(&sh.empty[s], 1);
      }
      for (int a = 0; a < 2; ++a) {
        tc::mbar_init(&sh.acc_full[a], 1);
        tc::mbar_init(&sh.acc_empty[a], RW * CG);
      }
      tc::mbar_fence_init();
    }
  } else if (warp == 1) {
    int tiles = 0;
    if (lane < p.count) {
      const DevProduct& q = p.prod[lane];
      Extent& x = sh.of[lane];
      int M = q.M, K = q.K;
      if (q.live != nullptr) {
        const int live = *q.live;
        if (q.live_is_k) K = min(live, K);
        else M = min(live, M);
      }
      x.rows = M;
      x.m_tiles = (M + kRows * CG - 1) / (kRows * CG);
      x.n_tiles = (q.N + kTileN - 1) / kTileN;
      x.kb = (K + kBK - 1) / kBK;
      x.k_parts = q.k_parts;
      x.group = q.group;
      x.strip_inv = inverse(x.group * x.n_tiles);
      x.group_inv = inverse(x.group);
      x.last_inv = inverse(x.m_tiles % x.group);
      tiles = x.m_tiles * x.n_tiles * x.k_parts;
    }
    const int t0 = __shfl_sync(~0u, tiles, 0), t1 = __shfl_sync(~0u, tiles, 1), t2 = __shfl_sync(~0u, tiles, 2);
    if (lane < kMaxProblems) sh.of[lane].first = lane >= p.count ? 0x7FFFFFFF : lane == 0 ? 0 : lane == 1 ? t0 : t0 + t1;
    __syncwarp();
    if (lane == 0) {
      sh.tiles = t0 + t1 + t2;
      // The first product's tiles may be longer than the others': in rounds of the others, none of which takes less than a
      // read-out, the time of 8 blocks of K (5 of a narrow tile).
      sh.long_tiles = p.count > 1 ? t0 : 0;
      sh.rest = sh.long_tiles % clusters;
      const int round = max(sh.of[1].kb, BN == 256 ? 8 : 5);
      sh.delta = p.count > 1 ? max(1, (sh.of[0].kb / sh.of[0].k_parts + 4 + round / 2) / round) : 1;
    }
  } else if (warp == 2) {
    tmem_alloc<CG>(&sh.tmem, kTmemCols);
  } else if (warp == 3 && lane < p.count) {
    tc::prefetch_tensormap(&p.a[lane]);
    tc::prefetch_tensormap(&p.b[lane]);
  }
  // Loads may start when the barriers and the plan are there (for a pair: the other CTA's barriers too); tensor memory can
  // take longer.
  if (CG == 2) cluster_sync();
  else if (warp != 2) asm volatile("bar.sync 1, %0;" ::"n"(C::kThreads - 32) : "memory");

  auto wait_for_tmem = [&]() {      // warps 1, 2 and the read-out's
    tc::tc_fence_before();
    asm volatile("bar.sync 2, %0;" ::"n"(C::kThreads - 64) : "memory");
    tc::tc_fence_after();
    return sh.tmem;
  };
  // what the cluster leaves to this CTA of a tile's blocks of K
  auto share = [&](Tile& t) {
    if (split > 1) t.k0 = t.k1 * part / split, t.k1 = t.k1 * (part + 1) / split;
  };
  if (warp == 0 || warp == 3) {
    // Warp 0 feeds A, warp 3 feeds B.  The whole warp runs the loop and one lane issues: operands then sit in uniform
    // registers (a stage took its issuer 312 clocks in a loop of one lane, 136 so; one warp for both operands was slower
    // than the MMAs, 600 against 512).
    const bool leader = tc::elect_one(), feeds_a = warp == 0;
    if (p.early_b && feeds_a) chain_wait();
    const uint32_t bytes = (uint32_t)(p.a_bytes + C::kBBytes) * CG;
    const uint32_t empty = tc::smem_u32(sh.empty);
    const uint32_t mine = tc::smem_u32(sh.full), full = CG == 2 ? map_to(mine, first_rank) : mine;   // the first CTA's count
    uint32_t slot = 0, parity = 1, dst = ring + (feeds_a ? 0 : a_slot);
    bool ok = true;
    // The bounded waits count this kernel's own time: a role waits for the predecessor before the first that could last, which
    // for B is when the ring is full.
    bool ahead = p.early_b && !feeds_a;
    auto next = [&]() {
      dst += stage_bytes;
      if (++slot == stages) {
        slot = 0, parity ^= 1, dst -= stages * stage_bytes;
        if (ahead) chain_wait();
        ahead = false;
      }
    };
    Tile t;
    for (Walk walk(sh, cluster, clusters); ok && walk.get(sh, t); walk.next(sh)) {
      const DevProduct& q = p.prod[t.prod];
      share(t);
      if (feeds_a) {
        const CUtensorMap* map = &p.a[t.prod];
        const int m0 = t.m * kRows * CG + half * kRows;
        // (a loop for each orientation, one branch in it: with the choice inside an iteration took 250 clocks for 130)
        if (CG == 1 && END == kStore && !BMN && p.fold != 0) {
          for (int k = t.k0 * kBK; k < t.k1 * kBK; k += kBK) {
            if (!wait(empty + 8 * slot, parity, guard, 1)) { ok = false; break; }
            if (leader) {
              expect_tx(mine + 8 * slot, bytes);
              tma_3d<CG>(dst, map, full + 8 * slot, k, m0, 0);
            }
            next();
          }
        } else if (q.a_mn == 0) {
          for (int k = t.k0 * kBK; k < t.k1 * kBK; k += kBK) {
            if (!wait(empty + 8 * slot, parity, guard, 1)) { ok = false; break; }
            if (leader) {
              if (CG == 1 || half == 0) expect_tx(mine + 8 * slot, bytes);
              tma_2d<CG>(dst, map, full + 8 * slot, k, m0);
            }
            next();
          }
        } else {
          for (int k = t.k0 * kBK; k < t.k1 * kBK; k += kBK) {
            if (!wait(empty + 8 * slot, parity, guard, 1)) { ok = false; break; }
            if (leader) {
              if (CG == 1 || half == 0) expect_tx(mine + 8 * slot, bytes);
              tma_2d<CG>(dst, map, full + 8 * slot, m0, k);
              tma_2d<CG>(dst + kBoxBytes, map, full + 8 * slot, m0 + 64, k);
            }
            next();
          }
        }
      } else {
        const CUtensorMap* map = &p.b[t.prod];
        if constexpr (!BMN) {
          // gate and up rows of the same columns (planes of one map): both, or this CTA's half
          const int r0 = kPaired ? t.n * kTileN : q.b_row0 + t.n * BN + half * (BN / 2);
          for (int k = t.k0 * kBK; k < t.k1 * kBK; k += kBK) {
            if (!wait(empty + 8 * slot, parity, guard, 5)) { ok = false; break; }
            if (leader) {
              if constexpr (kPaired) tma_3d<CG>(dst, map, full + 8 * slot, k, r0, half);
              else tma_2d<CG>(dst, map, full + 8 * slot, k, r0);
            }
            next();
          }
        } else {
          const int n0 = t.n * BN + half * (BN / 2), base = q.b_row0;
          for (int k = t.k0 * kBK; k < t.k1 * kBK; k += kBK) {
            if (!wait(empty + 8 * slot, parity, guard, 5)) { ok = false; break; }
            if (leader) {
#pragma unroll
              for (int j = 0; j < BN / CG / 64; ++j) tma_2d<CG>(dst + j * kBoxBytes, map, full + 8 * slot, n0 + 64 * j, base + k);
            }
            next();
          }
        }
      }
    }
  } else if (warp == 2) {
    wait_for_tmem();
  } else if (warp == 1) {
    const uint32_t tmem = wait_for_tmem();
    if (p.early_b) chain_wait();
    if (half == 0) {
      const uint32_t base_idesc = (1u << 4) | ((uint32_t)p.fmt << 7) | ((uint32_t)p.fmt << 10) | ((BMN ? 1u : 0u) << 16) |
                                  ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((kRows * CG) >> 4) << 24);
      const uint32_t leader = tc::elect_one() ? 1u : 0u;
      const uint32_t full = tc::smem_u32(sh.full), empty = tc::smem_u32(sh.empty);
      const uint32_t acc_full = tc::smem_u32(sh.acc_full), acc_empty = tc::smem_u32(sh.acc_empty);
      const uint64_t b_first = operand_desc(ring + a_slot, BMN);
      const uint16_t both = (uint16_t)(3u << first_rank);     // the CTAs of the pair
      uint32_t slot = 0, parity = 0, off = 0, set = 0, set_parity = 1;
      Tile t;
      bool ok = true;
      // the blocks b0 .. b1 of K into accumulator set `set`
      auto multiply = [&](auto a_orientation, int b0, int b1) {
        constexpr bool kAMn = decltype(a_orientation)::value;
        constexpr uint32_t kAStep = kAMn ? 128 : 2, kBStep = BMN ? 128 : 2;    // 16 K further, in units of 16 bytes
        const uint64_t a_first = operand_desc(ring, kAMn);
        const uint32_t idesc = base_idesc | ((kAMn ? 1u : 0u) << 15), d = tmem + set * BN;
        uint32_t accumulate = 0;
        for (int k = b0; k < b1; ++k) {
          if (!wait(full + 8 * slot, parity, guard, 3)) return false;
          tc::tc_fence_after();
          // (Predicated, not in a branch: operands that change or are not constant stay in uniform registers.  Four MMAs of
          // N = 128 take their issuer 270 clocks, in a branch 325; the MMAs themselves 256.)
          const uint64_t a = a_first + off, b = b_first + off;
#pragma unroll
          for (int i = 0; i < kBK / 16; ++i)
            mma_ss<CG>(leader, d, a + i * kAStep, b + i * kBStep, idesc, i == 0 ? accumulate : 1u);
          commit<CG>(leader, empty + 8 * slot, both);
          accumulate = 1;
          off += stage_bytes >> 4;
          if (++slot == stages) slot = 0, parity ^= 1, off = 0;
        }
        return true;
      };
      for (Walk walk(sh, cluster, clusters); ok && walk.get(sh, t); walk.next(sh)) {
        const bool a_mn = p.prod[t.prod].a_mn != 0;
        share(t);
        const int parts = parts_of<END, CG>(t.k1 - t.k0);
        for (int piece = 0; ok && piece < parts; ++piece) {
          if (!wait(acc_empty + 8 * set, set_parity, guard, 2)) { ok = false; break; }
          tc::tc_fence_after();
          constexpr int kPart = kPartBlocks<END, CG>;
          const int b0 = t.k0 + piece * kPart, b1 = kInParts<END> ? min(b0 + kPart, t.k1) : t.k1;
          ok = kStores<END> && BMN && a_mn ? multiply(std::true_type{}, b0, b1) : multiply(std::false_type{}, b0, b1);
          commit<CG>(ok ? leader : 0u, acc_full + 8 * set, both);
          set ^= 1;
          if (set == 0) set_parity ^= 1;
        }
      }
    }
  } else if (warp >= kControlWarps) {
    const uint32_t tmem = wait_for_tmem();
    const uint32_t buf = ring + C::kRing + (warp - kControlWarps) * C::kRowBytes;
    const int wg = (warp - 4) >> 2, quad = warp & 3;
    const int in_tile = quad * 32 + lane;
    constexpr int kMine = kTileN * 4 / RW;  // columns of a warpgroup
    constexpr int kPiece = RW == 4 && END == kDswiglu ? 16 : 32;    // (as many as registers allow)
    {      // the parameters of the end come to the SM while the first tile is multiplied (77 x 2056 x 32001 35.1 -> 34.4 us)
      const End& e = p.prod[0].end;
      asm volatile("" ::"l"(e.out), "l"(e.ld), "l"(e.h), "l"(e.h_rest), "l"(e.gate_up), "l"(e.ld_gu), "r"(e.half), "f"(e.limit), "r"(e.vec_out),
                   "r"(e.vec_h), "r"(e.vec_gu), "r"(e.tma_out), "l"(e.acc), "l"(e.part), "l"(e.given));
    }
    if (p.early_b) chain_wait();
    uint32_t sets = 0;
    Tile t;
    bool ok = true;
    for (Walk walk(sh, cluster, clusters); ok && walk.get(sh, t); walk.next(sh)) {
      const End& e = p.prod[t.prod].end;
      const int N = p.prod[t.prod].N;
      share(t);
      const int row = t.m * kRows * CG + half * kRows + in_tile;
      const bool live = row < t.rows;
      const bool warp_live = row - lane < t.rows;
      auto hand_back = [&](uint32_t set) {      // all loads from the accumulators have come back
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) remote_arrive(map_to(tc::smem_u32(&sh.acc_empty[set]), first_rank));
      };
      auto add_part = [&](uint32_t n, float (&sum)[kMine]) {      // the n-th accumulators in turn, this warp's lanes and columns
        const uint32_t set = n & 1, from = tmem + set * BN + ((uint32_t)(quad * 32) << 16) + wg * kMine;
        if (!wait(tc::smem_u32(&sh.acc_full[set]), (n >> 1) & 1, guard, 4)) return false;
        tc::tc_fence_after();
#pragma unroll
        for (int c = 0; c < kMine; c += 16) {
          uint32_t v[16];
          tc::tmem_ld_32x16(from + c, v);
          tc::tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) sum[c + j] += __uint_as_float(v[j]);
        }
        hand_back(set);
        return true;
      };
      auto park = [&](int c, float x) {         // this CTA's part of a sum, columns of 128 rows, where the stages were
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + (c * kRows + in_tile) * 4), "f"(x) : "memory");
      };
      RowState st;
      row_begin<END>(e, row, live && !parked, st);
      // Gate and up of a piece are copied ahead while the one before it, or the tile, is computed.  (Loaded when they were
      // needed, a piece of 32 columns took 6 us, and the read-out of a tile 21 to 32 beside 41 of its MMAs.)
      const uint16_t* gate_row = nullptr;
      if constexpr (END == kDswiglu && CG == 2) {
        gate_row = static_cast<const uint16_t*>(e.gate_up) + (int64_t)row * e.ld_gu + t.n * kTileN;
        if (!parked && warp_live && e.vec_gu == 16 && t.n * kTileN + wg * kMine + 32 <= N) {
          rows_start(buf + 2048, live ? gate_row + wg * kMine : nullptr);
          rows_start(buf + 4096, live ? gate_row + wg * kMine + e.half : nullptr);
        }
      }
      const float scale = kStores<END> && e.scale != nullptr ? *e.scale : 1.f;
      if constexpr (END == kCeStats || END == kCeGrad) {
        const int parts = parts_of<END, CG>(t.k1 - t.k0);
        float sum[kMine];
#pragma unroll
        for (int j = 0; j < kMine; ++j) sum[j] = 0.f;
        for (int piece = 0; piece < parts; ++piece, ++sets)
          if (!add_part(sets, sum)) { ok = false; break; }
        if (!ok) break;
        if (split > 1) {
          if (warp_live)
#pragma unroll
            for (int j = 0; j < kMine; ++j) park(wg * kMine + j, sum[j]);
          break;
        }
#pragma unroll
        for (int c = 0; c < kMine; c += 32) {
          const int col = t.n * kTileN + wg * kMine + c, n = N - col;
          if (n <= 0) break;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = sum[c + j];
          if constexpr (END == kCeGrad) st.half = (c >> 5) & 1;
          row_piece<END, kTwo, 32>(e, p.fmt, buf, row, live, t.kpart, col, n, scale, v, v, st);
          if constexpr (END == kCeGrad)
            if (e.tma_out && (st.half == 1 || n <= 32)) copy_rows(buf, &p.out[t.prod], col - 32 * st.half, row - lane);
        }
        row_end<END>(e, row, live, t.n * 2 + wg, st);
      } else {
        if constexpr (END == kStoreLong) {
          int left = parts_of<END, CG>(t.k1 - t.k0) - 1;
          if (left > 0) {      // the parts before the last go to its accumulators
            float sum[kMine];
#pragma unroll
            for (int j = 0; j < kMine; ++j) sum[j] = 0.f;
            for (; left > 0; --left, ++sets)
              if (!add_part(sets, sum)) { ok = false; break; }
            const uint32_t set = sets & 1, to = tmem + set * BN + ((uint32_t)(quad * 32) << 16) + wg * kMine;
            if (!ok || !wait(tc::smem_u32(&sh.acc_full[set]), (sets >> 1) & 1, guard, 4)) break;
            tc::tc_fence_after();
#pragma unroll
            for (int c = 0; c < kMine; c += 16) {
              uint32_t v[16];
              tc::tmem_ld_32x16(to + c, v);
              tc::tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(sum[c + j] + __uint_as_float(v[j]));
              tc::tmem_st_32x8(to + c, v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
              tc::tmem_st_32x8(to + c + 8, v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]);
            }
            tc::tmem_wait_st();
          }
        }
        const uint32_t set = sets & 1, from = tmem + set * BN + ((uint32_t)(quad * 32) << 16);
        ++sets;
        if (!wait(tc::smem_u32(&sh.acc_full[set]), ((sets - 1) >> 1) & 1, guard, 4)) break;
        tc::tc_fence_after();
        if (parked) {
          if (fold != 0 ? quad * 32 < 2 * fold : warp_live) {
            for (int c = wg * (BN * 4 / RW); c < (wg + 1) * (BN * 4 / RW); c += 32) {
              float v[32];
              tmem_load(from + c, v);
              tc::tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) park(c + j, v[j]);
            }
          }
          break;
        }
        // The tile before may have been another product's, whose last rows a copy still reads from the buffer.
        if constexpr (kStores<END>)
          if (!e.tma_out) rows_copied();
#pragma unroll 1
        for (int c = wg * kMine; c < (wg + 1) * kMine; c += kPiece) {
          const int col = t.n * kTileN + c, n = N - col;
          const bool none = n <= 0 || !warp_live;
          float v[kPiece], w[kPiece];
          if (!none) {
            tmem_load(from + c, v);
            if constexpr (kPaired) tmem_load(from + BN / 2 + c, w);
            tc::tmem_wait_ld();
          }
          if (none || c + kPiece >= (wg + 1) * kMine || n <= kPiece) {     // the last piece: before it goes to memory
            hand_back(set);
            if (none) break;
          }
          if (t.k1 == t.k0) {
#pragma unroll
            for (int j = 0; j < kPiece; ++j) v[j] = w[j] = 0.f;
          }
          if constexpr (kStores<END>) st.half = ((c - wg * kMine) >> 5) & 1;
          if constexpr (END == kDswiglu) {
            st.here = CG == 2 && e.vec_gu == 16 && n >= 32;
            st.next = CG == 2 && e.vec_gu == 16 && n >= 64 && c + 32 < (wg + 1) * kMine ? gate_row + c + 32 : nullptr;
          }
          row_piece<END, kTwo, kPiece>(e, p.fmt, buf, row, live, t.kpart, col, n, scale, v, w, st);
          if constexpr (kStores<END>)
            if (e.tma_out && (st.half == 1 || n <= kPiece)) copy_rows(buf, &p.out[t.prod], col - 32 * st.half, row - lane);
          if (n <= kPiece) break;
        }
      }
    }
  }
  __syncwarp();
  if (warp >= kControlWarps && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");

  if (parked) {
    if (split > 1) cluster_sync();       // every CTA's part is in its shared memory
    else __syncthreads();
    Tile t;
    if (warp >= kControlWarps && Walk(sh, cluster, clusters).get(sh, t) && !guard.aborted()) {
      // Pieces of eight columns, dealt out to the parts; a warp takes a piece of 32 rows.  Rows behind the last are nothing
      // but for kCeGrad, whose zeros are K of the next product.
      const End& e = p.prod[t.prod].end;
      const int row0 = t.m * kRows * CG + half * kRows, rows = t.rows - row0;
      const int quads = END == kCeGrad ? 4 : rows <= 0 ? 0 : min(4, (rows + 31) / 32);
      const int pieces = (kTileN / 8 - part + split - 1) / split;
      const float scale = kStores<END> && e.scale != nullptr ? *e.scale : 1.f;
#pragma unroll 1
      for (int i = warp - kControlWarps; i < pieces * quads; i += RW) {
        const int quad = i % quads, piece = (i / quads) * split + part;
        const int c = piece * 8, in_tile = quad * 32 + lane, row = row0 + in_tile;
        const int col = t.n * kTileN + c, n = p.prod[t.prod].N - col;
        const bool live = row < t.rows;
        RowState st;
        row_begin<END>(e, row, live, st);
        if constexpr (END == kDswiglu) st.here = false, st.next = nullptr;
        float v[8], w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = w[j] = 0.f;
        if (n > 0 && quad * 32 < rows) {
          // some parts' loads at a time: each is a round trip to another SM
          constexpr int kAtOnce = kPaired ? 2 : 4;
          const uint32_t at = ring + (c * kRows + in_tile) * 4;
          for (int from = 0; from < split; from += kAtOnce) {
            float a[kAtOnce][8], b[kAtOnce][8];      // b: of up, or the second term's
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
              const uint32_t x = map_to(at, min(from + i, split - 1) * CG + half);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                a[i][j] = ld_cluster(x + j * kRows * 4);
                if constexpr (kPaired) b[i][j] = ld_cluster(x + (BN / 2 + j) * kRows * 4);
                else if (fold != 0) b[i][j] = ld_cluster(x + (j * kRows + fold) * 4);
              }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
              if (from + i >= split) break;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                v[j] += a[i][j];
                if constexpr (kPaired) w[j] += b[i][j];
                else if (fold != 0) v[j] = add_second(v[j], b[i][j]);
              }
            }
          }
        }
        if (n > 0) row_piece<END, kTwo, 8>(e, p.fmt, 0, row, live, t.kpart, col, n, scale, v, w, st);
        row_end<END>(e, row, live, t.n * (kTileN / 8) + piece, st);
      }
    }
  }
  // A wait that ran out leaves copies and MMAs in flight: they land within microseconds.
  if (guard.aborted())
    for (int i = 0; i < 100; ++i) __nanosleep(20000);
  tc::tc_fence_before();
  __syncthreads();
  if (width > 1) cluster_sync();
  if (warp == 2) {
    tc::tc_fence_after();
    tmem_dealloc<CG>(sh.tmem, kTmemCols);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------
struct Launch {
  int dev, cg, bn, split, grid;
  bool chained;
  cudaStream_t stream;
};

template <int CG, int BN, int RW, bool BMN, int WAY>
int run_kernel(const Params& p, const Launch& l) {
  using C = Cfg<CG, BN, RW, WAY>;
  auto kernel = dense_kernel<CG, BN, RW, BMN, WAY>;
  static std::atomic<uint64_t> ready{0};      // devices on which this instance is set up
  const uint64_t bit = l.dev < 64 ? 1ull << l.dev : 0;
  if (bit == 0 || !(ready.load(std::memory_order_acquire) & bit)) {
    XKB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    ready.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(l.grid);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = l.stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (CG * l.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = CG * l.split;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (l.chained) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  XKB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  XKB_CHECK_LAUNCH("dense_kernel");
  return XKB_OK;
}

// Read-out warps of a single CTA: eight where the read-out adds up in registers, else four and two CTAs an SM, whose ends
// (and the next kernel's first loads) overlap.
constexpr int single_warps(int end) { return end == kCeStats || end == kCeGrad ? 8 : 4; }

template <bool BMN, int WAY>
int run_variant(const Params& p, const Launch& l) {
  if (l.cg == 2) return l.bn == 256 ? run_kernel<2, 256, 8, BMN, WAY>(p, l) : run_kernel<2, 128, 8, BMN, WAY>(p, l);
  if constexpr (single_warps(end_of(WAY)) == 4)
    if (l.bn == 64) return run_kernel<1, 64, 4, BMN, WAY>(p, l);
  return run_kernel<1, 128, single_warps(end_of(WAY)), BMN, WAY>(p, l);
}

// How many clusters of so many CTAs of one of the kernels' sizes run at once on a device, the current one.
int clusters_at_once(int dev, int cg, int bn, int read_warps, int width, int* out);

// one per translation unit
int run_ffn(int end, const Params& p, const Launch& l);
int run_store(bool b_mn, const Params& p, const Launch& l);
int run_store_long(bool b_mn, const Params& p, const Launch& l);      // of whole tiles of pairs
int run_ce(int end, const Params& p, const Launch& l);

}  // namespace dense
}  // namespace xkb
