// Log-probabilities of given tokens, entropy and top alternatives of wide rows, and their gradient (sm_100a).
//
//   m = max x,  l = ln sum exp(x - m),  logprob = x_t - m - l,  H = l - sum exp(x - m - l) (x - m)
//   dx = -p (G + g_H (ln p + H)) + sum of the gradients given to this column,  p = exp(x - m - l)
//
// Forward: one pass over the row.  A thread adds up e = 2^y and e y with y = x log2(e) - c.  Its reference c follows the
// thread's running maximum lazily: it moves only where a batch exceeds it by kSlack, so that the sums are rescaled once
// or twice a row and not per element; they have 2^104 of headroom left.  The same c stands in every term, its rounding therefore cancels.
// A row belongs to a CTA, or to a cluster of up to eight whose parts are joined through distributed shared memory:
// no workspace, no atomics on floats, the same result in every run.
//
// Top alternatives: every thread keeps the maximum of its elements, which the pass needs anyway.  The k-th largest of
// these maxima, taken by groups of threads, bounds the row's k-th largest element from below, and only threads that reach
// it can hold one of the k: their elements (a tenth of a row at k = 20) are read again, mostly out of the L2, and what
// reaches the bound is ranked.
//
// Forward: HBM-bound where rows fill the chip: 4096 x 128000 bf16 159 us, 6.6 TB/s (182 in a loop of calls, at the power limit).  Few rows are
// bound by latency, half of it behind the pass where alternatives are wanted: 1 x 128000 with 20 of them 6.0 us, 64 x 128000 fp32 with
// 5 9.9 us (3.3 TB/s), 509 x 50001 fp16 with 20 16.4 us (3.1 TB/s).
// Gradient: HBM-bound, read once and written once: 4096 x 128000 bf16 320 us, 6.6 TB/s (344 in a loop).
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <cstddef>
#include <type_traits>

#include "common.cuh"
#include "softmax_dev.cuh"

namespace xkb {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTop = 64;
constexpr float kSlack = 11.f;              // 2^16
constexpr float kNan = __builtin_nanf("");

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// What a type of logits needs: N elements in 16 bytes, a running maximum of whole vectors, ordered keys.
//   kClamp: smaller elements count as this, which keeps -inf out of the products.  A row whose maximum is not between kLow
//   and kHigh, where a clamped element would count or x log2(e) is too coarse, takes the slow pass.
//   key_of: ascending with the value; NaN above all, -0 as +0, never 0 (that is "no element") nor the largest word.
template <typename T> struct Elem;

template <> struct Elem<float> {
  static constexpr int N = 4;
  static constexpr float kClamp = -1e8f, kLow = -1e6f, kHigh = 1e6f;
  static constexpr uint32_t kMaskKey = 0x00800000u;   // of the lowest finite value: one above that of -inf
  using Max = float;
  static __device__ __forceinline__ Max lowest() { return -INFINITY; }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return max_nan(a, b); }
  static __device__ __forceinline__ Max of(const uint4& q) {
    return max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)), max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
  }
  static __device__ __forceinline__ float value(Max a) { return a; }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ void clamped(const uint4& q, float (&v)[4]) {
    unpack(q, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = max_nan(v[i], kClamp);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
  static __device__ __forceinline__ uint32_t key_of(float v) {
    if (v != v) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(v + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
  }
  static __device__ __forceinline__ float of_key(uint32_t k) {
    if (k >= 0xfffffffeu) return kNan;
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
  }
};

template <> struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr float kClamp = -1e8f, kLow = -1e6f, kHigh = 1e6f;
  static constexpr uint32_t kMaskKey = 0x0080u;
  using Max = __nv_bfloat162;
  static __device__ __forceinline__ Max as2(uint32_t u) { return *reinterpret_cast<Max*>(&u); }
  static __device__ __forceinline__ Max lowest() { return as2(0xff80ff80u); }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return __hmax2_nan(a, b); }
  static __device__ __forceinline__ Max of(const uint4& q) {
    return larger(larger(as2(q.x), as2(q.y)), larger(as2(q.z), as2(q.w)));
  }
  static __device__ __forceinline__ float value(Max a) { return max_nan(__low2float(a), __high2float(a)); }
  static __device__ __forceinline__ void pair(uint32_t u, float& a, float& b) {
    a = __uint_as_float(u << 16);
    b = __uint_as_float(u & 0xffff0000u);
  }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
    pair(q.x, v[0], v[1]); pair(q.y, v[2], v[3]); pair(q.z, v[4], v[5]); pair(q.w, v[6], v[7]);
  }
  static __device__ __forceinline__ uint32_t clamp2(uint32_t u) {
    const Max c = __hmax2_nan(as2(u), __float2bfloat162_rn(kClamp));
    return *reinterpret_cast<const uint32_t*>(&c);
  }
  static __device__ __forceinline__ void clamped(const uint4& q, float (&v)[8]) {
    unpack(make_uint4(clamp2(q.x), clamp2(q.y), clamp2(q.z), clamp2(q.w)), v);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint32_t key_of(float v) {
    if (v != v) return 0xffffu;
    const uint32_t u = __float_as_uint(v + 0.f) >> 16;
    return (u & 0x8000u) ? ~u & 0xffffu : u | 0x8000u;
  }
  static __device__ __forceinline__ float of_key(uint32_t k) {
    if (k == 0xffffu) return kNan;
    return __uint_as_float(((k & 0x8000u) ? k & 0x7fffu : ~k & 0xffffu) << 16);
  }
};

template <> struct Elem<__half> {
  static constexpr int N = 8;
  static constexpr float kClamp = -65504.f, kLow = -60000.f, kHigh = 1e6f;
  static constexpr uint32_t kMaskKey = 0x0400u;
  using Max = __half2;
  static __device__ __forceinline__ Max as2(uint32_t u) { return *reinterpret_cast<Max*>(&u); }
  static __device__ __forceinline__ Max lowest() { return as2(0xfc00fc00u); }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return __hmax2_nan(a, b); }
  static __device__ __forceinline__ Max of(const uint4& q) {
    return larger(larger(as2(q.x), as2(q.y)), larger(as2(q.z), as2(q.w)));
  }
  static __device__ __forceinline__ float value(Max a) { return max_nan(__low2float(a), __high2float(a)); }
  static __device__ __forceinline__ void pair(Max h, float& a, float& b) {
    const float2 f = __half22float2(h);
    a = f.x;
    b = f.y;
  }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
    pair(as2(q.x), v[0], v[1]); pair(as2(q.y), v[2], v[3]); pair(as2(q.z), v[4], v[5]); pair(as2(q.w), v[6], v[7]);
  }
  static __device__ __forceinline__ void clamped(const uint4& q, float (&v)[8]) {
    const Max c = __float2half2_rn(kClamp);
    pair(larger(as2(q.x), c), v[0], v[1]); pair(larger(as2(q.y), c), v[2], v[3]);
    pair(larger(as2(q.z), c), v[4], v[5]); pair(larger(as2(q.w), c), v[6], v[7]);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
  }
  static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
  static __device__ __forceinline__ uint32_t key_of(float v) {
    if (v != v) return 0xffffu;
    const uint32_t u = __half_as_ushort(__float2half_rn(v + 0.f));   // exact: v came from a half
    return (u & 0x8000u) ? ~u & 0xffffu : u | 0x8000u;
  }
  static __device__ __forceinline__ float of_key(uint32_t k) {
    if (k == 0xffffu) return kNan;
    return __half2float(__ushort_as_half((unsigned short)((k & 0x8000u) ? k & 0x7fffu : ~k & 0xffffu)));
  }
};

// A row as vectors of 16 aligned bytes: vector j holds columns [j N - skew, (j + 1) N - skew); the first and the last may
// reach over the row's ends, and only what lies in the row is read or written there.
template <typename T>
struct RowView {
  const T* row;
  int skew, V;
  int first_whole, end_whole, vectors;   // vectors [first_whole, end_whole) lie in the row
  __device__ __forceinline__ RowView(const T* r, int v) : row(r), V(v) {
    constexpr int N = Elem<T>::N;
    skew = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    first_whole = skew > 0;
    end_whole = (int)(((int64_t)V + skew) / N);
    vectors = (int)(((int64_t)V + skew + N - 1) / N);
    if (end_whole < first_whole) end_whole = first_whole;
  }
  __device__ __forceinline__ int column(int j) const { return j * Elem<T>::N - skew; }   // of vector j's first element
  __device__ __forceinline__ bool whole(int j) const { return j >= first_whole && j < end_whole; }
  __device__ __forceinline__ uint4 load_whole(int j) const {
    return __ldg(reinterpret_cast<const uint4*>(row - skew) + j);
  }
  // any vector of [0, vectors); `outside` fills what is not in the row
  __device__ __forceinline__ uint4 load(int j, float outside) const {
    if (whole(j)) return load_whole(j);
    constexpr int N = Elem<T>::N;
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = column(j) + i;
      v[i] = at >= 0 && at < V ? Elem<T>::load(row + at) : outside;
    }
    return Elem<T>::pack(v);
  }
};

// The sums of some elements: e = 2^(x log2e - c), S = sum e, T = sum e (x log2e - c).
struct Sums {
  float c, S, T;
  __device__ __forceinline__ void move_to(float to) {
    const float d = c - to, f = exp2_fast(d);
    T = fmaf(d, S, T) * f;
    S *= f;
    c = to;
  }
};

// Parts are (maximum, c, S, T).  Two of them in one, and those of a warp's lanes in one, at the largest c: no factor exceeds 1.
__device__ __forceinline__ float4 joined(float4 p, float4 q) {
  const float to = fmaxf(p.y, q.y);
  Sums a{p.y, p.z, p.w}, b{q.y, q.z, q.w};
  a.move_to(to);
  b.move_to(to);
  return make_float4(max_nan(p.x, q.x), to, a.S + b.S, a.T + b.T);
}
__device__ __noinline__ float4 joined(float4 p) {
  const float mx = warp_max_nan(p.x), to = warp_max(p.y);
  Sums t{p.y, p.z, p.w};
  t.move_to(to);
  return make_float4(mx, to, warp_add(t.S), warp_add(t.T));
}

// S and T of the even and of the odd places of a vector
struct PairSums { Pair S, T; };

template <typename T>
__device__ __forceinline__ void add_vector(const uint4& q, Pair minus_c, PairSums& s) {
  constexpr int N = Elem<T>::N;
  float v[N];
  Elem<T>::clamped(q, v);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const Pair y = fma2(pair_of(v[i], v[i + 1]), pair_of(kLog2e), minus_c);
    float y0, y1;
    split(y, y0, y1);
    const Pair e = pair_of(exp2_fast(y0), exp2_fast(y1));
    s.S = add2(s.S, e);
    s.T = fma2(e, y, s.T);
  }
}

// The largest key that at least k of the warp's 32 PER keys reach (0 if fewer than k are above 0), bit by bit from the first
// one in which the keys differ.
template <int PER>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&key)[PER], int k) {
  uint32_t most = 0, least = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    most = max(most, key[i]);
    least = min(least, key[i]);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  least = __reduce_min_sync(0xffffffffu, least);
  if (most == least) return most;
  uint32_t bit = 0x80000000u >> __clz(most ^ least), t = most & ~(2u * bit - 1u);
#pragma unroll 1
  for (; bit != 0; bit >>= 1) {
    const uint32_t trial = t | bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) n += key[i] >= trial;
    if (__reduce_add_sync(0xffffffffu, n) >= k) t = trial;
  }
  return t;
}

constexpr int kBatch = 4;   // vectors a thread requests before it uses the first

template <int THREADS>
struct TopScratch {
  static constexpr int kRoom = 8 * THREADS + kMaxTop, kGroups = THREADS < 128 ? THREADS : 128;
  static constexpr int kRanked = 32;         // so many candidates are ranked in one step: the places behind the last one hold 0
  static constexpr int kFew = THREADS < 128 ? 128 : THREADS;   // more are cut down to k first
  uint64_t cand[kRoom];                      // value key, ~column: all different, larger is better
  uint64_t top[kMaxTop];                     // the best ones, in order
  alignas(16) uint32_t group[kGroups];       // the maxima of the row's groups of threads
  uint32_t key[THREADS];                     // (long way) of every thread
  int owner[THREADS];                        // threads whose elements are read again, by warp (long way: of the CTA)
  int digits[256], digit, before, inside;    // (too many candidates) how many have a digit, and where the k-th is
  int ties[THREADS / 32];                    // of a warp
  uint32_t least[kGroups / 32];              // of a warp
  int n, owners;
  uint32_t bound;
};
template <int THREADS> struct NoScratch {};
// `group` is read in words of 16 bytes, at multiples of four
template <int THREADS> constexpr bool kWordsOfGroups = alignof(TopScratch<THREADS>) % 16 == 0 && offsetof(TopScratch<THREADS>, group) % 16 == 0 &&
                                                       TopScratch<THREADS>::kGroups % 32 == 0;
static_assert(kWordsOfGroups<32> && kWordsOfGroups<64> && kWordsOfGroups<128> && kWordsOfGroups<256>, "misaligned");

// Leaves the k largest of the n candidates (n >= k) at the front, in any order, and 0 in the places behind them: digits of
// eight bits from the top, until the k-th's digit is one that all who share it are needed.
template <int THREADS>
__device__ __noinline__ void keep_best(TopScratch<THREADS>& s, int k) {
  constexpr int kEach = (TopScratch<THREADS>::kRoom + THREADS - 1) / THREADS;
  const int n = s.n, tid = threadIdx.x;
  uint64_t mine[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int at = tid + i * THREADS;
    mine[i] = at < n ? s.cand[at] : 0;
  }
  uint64_t floor = 0, known = 0;   // digits so far, which bits they are
  int need = k;                    // of those that share them
#pragma unroll 1
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) s.digits[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (mine[i] != 0 && (mine[i] & known) == floor) atomicAdd(&s.digits[mine[i] >> shift & 255], 1);
    __syncthreads();
    if (tid < 32) {   // the digit whose suffix sum reaches `need`: lane l has digits 8 l .. 8 l + 7
      int count[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += count[i] = s.digits[tid * 8 + i];
      int above = sum;             // of the lanes from this one on, then of those behind it
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int more = __shfl_down_sync(0xffffffffu, above, d);
        if (tid + d < 32) above += more;
      }
      above -= sum;
      if (above < need && above + sum >= need) {
        int digit = 7;
#pragma unroll
        for (int i = 7; i >= 0; --i) {
          digit = i;
          if (above + count[i] >= need) break;
          above += count[i];
        }
        s.digit = tid * 8 + digit;
        s.before = above;
        s.inside = s.digits[tid * 8 + digit];
      }
    }
    __syncthreads();
    floor |= (uint64_t)s.digit << shift;
    known |= 255ull << shift;
    need -= s.before;
    const bool all = s.inside == need;
    __syncthreads();
    if (all) break;
  }
  if (tid == 0) s.n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (mine[i] != 0 && (mine[i] & known) >= floor) s.cand[atomicAdd(&s.n, 1)] = mine[i];
  __syncthreads();
  if (tid >= k && tid < TopScratch<THREADS>::kRanked) s.cand[tid] = 0;
  __syncthreads();
}

// The k best of the first n candidates to s.top, in order; unfilled places are 0.
template <int THREADS>
__device__ __forceinline__ void rank_all(TopScratch<THREADS>& s, int n, int k) {
  const int tid = threadIdx.x;
  for (int i = n + tid; i < k; i += THREADS) s.top[i] = 0;
  if (4 * n <= THREADS && THREADS >= 128) {   // four threads a candidate, every fourth place each
    const int i = tid >> 2;
    const uint64_t mine = s.cand[i];
    int rank = 0;
    if (n <= 32) {
#pragma unroll
      for (int j = 0; j < 32; j += 4) rank += s.cand[j + (tid & 3)] > mine;
    } else {
#pragma unroll 4
      for (int j = tid & 3; j < n; j += 4) rank += s.cand[j] > mine;
    }
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if ((tid & 3) == 0 && i < n && rank < k) s.top[rank] = mine;
    return;
  }
#pragma unroll 1
  for (int i = tid; i < n; i += THREADS) {
    const uint64_t mine = s.cand[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += s.cand[j] > mine;
    if (rank < k) s.top[rank] = mine;
  }
}

__device__ __forceinline__ uint64_t candidate(uint32_t key, int col) { return (uint64_t)key << 32 | (uint32_t)~(uint32_t)col; }

template <typename T, int THREADS>
__device__ __forceinline__ void offer(float v, int col, uint32_t floor, uint64_t* to, int* n) {
  const uint32_t key = Elem<T>::key_of(v);
  if (key < floor) return;
  const int place = atomicAdd(n, 1);
  if (place < TopScratch<THREADS>::kRoom) to[place] = candidate(key, col);
}

// Once more the vectors of those threads of the warp whose maximum reaches `floor`: their elements from there on to the list
// `to`, which `n` counts (both perhaps another CTA's).  The warp's lanes share the vectors of an owner, or several small owners.
// The elements before the row's first and behind its last whole vector are looked at in any case, by the CTA that has them.
// Nothing is put behind the list's end: the caller sees by the count that it was too short.
// (This runs a few times in a CTA's life: what costs is latency and fetching the code, so there is one copy of each step.)
template <typename T, int THREADS>
__device__ __forceinline__ void collect(const RowView<T>& r, int lo, int hi, uint32_t floor, uint32_t best, TopScratch<THREADS>& s, uint64_t* to,
                                        int* n) {
  constexpr int N = Elem<T>::N, kLoads = 4;
  const int lane = threadIdx.x & 31, end = min(hi, r.end_whole);
  int edge = -1;   // this thread's column in front of the whole vectors (vector 0) or behind them
  float edge_value = 0.f;
  if (threadIdx.x < 2 * N) {
    const bool head = threadIdx.x < N;
    const int j = head ? 0 : r.end_whole, col = r.column(j) + (int)(threadIdx.x & (N - 1));
    if (j >= lo && j < hi && (head ? r.first_whole > 0 : true) && col >= 0 && col < r.V) {
      edge = col;
      edge_value = Elem<T>::load(r.row + col);   // on its way while the vectors are looked at
    }
  }
  const bool mine = best > 0 && best >= floor;
  const unsigned who = __ballot_sync(0xffffffffu, mine);
  const int owners = __popc(who), per = (hi - lo + THREADS - 1) / THREADS, first = lo + (int)(threadIdx.x & ~31u);
  int* owner = s.owner + (threadIdx.x & ~31u);                          // the warp's own part
  if (mine) owner[__popc(who & ((1u << lane) - 1u))] = lane;
  __syncwarp();
  const float least = Elem<T>::of_key(floor > 0 ? floor : 1u);          // (a NaN, as of key 1, lets everything pass to the keys)
  const int log = per >= 32 ? 5 : per <= 1 ? 0 : 32 - __clz(per - 1);   // lanes of an owner: a power of two
#pragma unroll 1
  for (int o = lane >> log; o < owners; o += kLoads << (5 - log)) {
    int from[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int at = o + (u << (5 - log));
      from[u] = at < owners ? first + owner[at] : end;
    }
#pragma unroll 1
    for (int i = lane & ((1 << log) - 1); i < per; i += 1 << log) {
      uint4 q[kLoads];
      unsigned pass = 0;
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int j = from[u] + i * THREADS;
        if (j < end && j >= r.first_whole) {
          q[u] = r.load_whole(j);
          pass |= 1u << u;
        }
      }
#pragma unroll
      for (int u = 0; u < kLoads; ++u)
        if ((pass >> u & 1) && Elem<T>::value(Elem<T>::of(q[u])) < least) pass &= ~(1u << u);
#pragma unroll 1
      for (; pass != 0; pass &= pass - 1) {   // seldom more than one; the vector comes from the L1 now
        const int u = __ffs(pass) - 1, j = (u == 0 ? from[0] : u == 1 ? from[1] : u == 2 ? from[2] : from[3]) + i * THREADS;
        float v[N];
        Elem<T>::unpack(r.load_whole(j), v);
        unsigned ok = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) ok |= v[e] < least ? 0u : 1u << e;
#pragma unroll 1
        for (; ok != 0; ok &= ok - 1) {
          const int col = r.column(j) + __ffs(ok) - 1;
          offer<T, THREADS>(Elem<T>::load(r.row + col), col, floor, to, n);
        }
      }
    }
  }
  if (edge >= 0) offer<T, THREADS>(edge_value, edge, floor, to, n);
}

// The first k columns of the row whose key is `bound`, to the CTA's list.
template <typename T, int THREADS>
__device__ __noinline__ void collect_first(const T* row, int V, uint32_t bound, int k, TopScratch<THREADS>& s) {
  constexpr int N = Elem<T>::N;
  const RowView<T> r(row, V);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int found = 0;
  for (int j0 = 0; j0 < r.vectors && found < k; j0 += THREADS) {
    const int j = j0 + tid, first = r.column(j);
    unsigned equal = 0;
    if (j < r.vectors) {
      float v[N];
      Elem<T>::unpack(r.load(j, 0.f), v);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (first + i >= 0 && first + i < r.V && Elem<T>::key_of(v[i]) == bound) equal |= 1u << i;
    }
    const int own = __popc(equal);
    int upto = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += below;
    }
    if (lane == 31) s.ties[warp] = upto;
    __syncthreads();
    int place = found + upto - own, all = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) place += s.ties[w];
      all += s.ties[w];
    }
    for (; equal != 0 && place < k; equal &= equal - 1, ++place) {
      const int to = atomicAdd(&s.n, 1);
      if (to < TopScratch<THREADS>::kRoom) s.cand[to] = candidate(bound, first + __ffs(equal) - 1);
    }
    found += all;
    __syncthreads();
  }
}

// The long way, for rows whose candidates do not fit the list: the k largest elements of the whole row to s.top, by one CTA.
template <typename T, int THREADS>
__device__ __noinline__ void select_top(const T* row, int V, int k, TopScratch<THREADS>& s) {
  constexpr int N = Elem<T>::N, kPer = THREADS / 32;
  const RowView<T> r(row, V);
  const int tid = threadIdx.x, lane = tid & 31, per = (r.vectors + THREADS - 1) / THREADS;   // vectors of a thread, at most
  auto search = [&](uint32_t key, int want) -> uint32_t {   // the want-th largest of the threads' keys
    __syncthreads();
    s.key[tid] = key;
    __syncthreads();
    if (tid < 32) {
      uint32_t keys[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) keys[i] = s.key[i * 32 + lane];
      const uint32_t t = kth_largest<kPer>(keys, want);
      if (tid == 0) s.bound = t;
    }
    __syncthreads();
    return s.bound;
  };
  // a vector's elements that lie in the row
  auto each = [&](int j, auto f) {
    float v[N];
    Elem<T>::unpack(r.load(j, 0.f), v);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int col = r.column(j) + i;
      if (col >= 0 && col < r.V) f(Elem<T>::key_of(v[i]), col);
    }
  };
  uint32_t best = 0;
  for (int j = tid; j < r.vectors; j += THREADS) each(j, [&](uint32_t key, int) { best = max(best, key); });
  const uint32_t bound = search(best, k);
  // Of the threads that share the bound those count whose first element of that value comes first, which each looks for.
  uint32_t last = 0xffffffffu;   // an element equal to the bound counts up to this column
  bool mine = best > 0 && best >= bound;
  const int above = __syncthreads_count(best > bound), ties = __syncthreads_count(best > 0 && best == bound);
  if (bound > 0 && above + ties > k) {
    uint32_t at = 0xffffffffu;
    if (best == bound)
      for (int j = tid; j < r.vectors && at == 0xffffffffu; j += THREADS)
        each(j, [&](uint32_t key, int col) { if (key == bound) at = min(at, (uint32_t)col); });
    last = ~search(best == bound ? ~at : 0u, k - above);
    mine = best > bound || (best == bound && at <= last);
  }
  if (tid == 0) s.n = s.owners = 0;
  __syncthreads();
  if (mine) s.owner[atomicAdd(&s.owners, 1)] = tid;
  __syncthreads();
  const int items = s.owners * per;
  for (int base = 0; base < items; base += THREADS) {
    if (base > 0) {   // room for a whole round: what is there is cut down to k
      __syncthreads();
      const int have = s.n;
      __syncthreads();
      if (have > kMaxTop) keep_best<THREADS>(s, k);
    }
    const int it = base + tid, j = it < items ? s.owner[it / per] + it % per * THREADS : r.vectors;
    if (j < r.vectors)
      each(j, [&](uint32_t key, int col) {
        if (key > bound || (key == bound && (uint32_t)col <= last)) s.cand[atomicAdd(&s.n, 1)] = candidate(key, col);
      });
  }
  __syncthreads();
  keep_best<THREADS>(s, k);
}

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  const void* ids;
  int ids64;
  float *logprobs, *entropy, *stats, *top_logprobs;
  int32_t* top_ids;
  int64_t M;
  int V, top_k;
};

__device__ __forceinline__ int64_t id_at(const void* ids, int ids64, int64_t i) {
  return ids64 ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// The statistics of a row from its part: maximum, l, H; `far`: they have to come from the slow pass.
__device__ __forceinline__ void statistics(const float4& part, float low, float high, float& row_max, float& l, float& H, bool& far) {
  row_max = part.x;
  far = false;
  if (row_max != row_max || row_max == INFINITY) {
    l = H = kNan;
  } else if (row_max == -INFINITY) {
    l = H = 0.f;
  } else if (row_max < low || row_max > high) {
    l = H = 0.f;
    far = true;
  } else {
    const float at_max = row_max * kLog2e;
    Sums t{part.y, part.z, part.w};
    t.move_to(at_max);
    // at_max is row_max log2(e) but for its rounding, which is in every e: ln sum exp(x - row_max) = ln2 (log2 S + at_max - row_max log2(e))
    const float off = -fmaf(row_max, kLog2e, -at_max), log2s = log2f(t.S);
    l = (log2s + off) * kLn2;
    H = fmaxf((log2s - t.T / t.S) * kLn2, 0.f);
  }
}

// The slow pass, for a row whose maximum is far from zero: differences from the maximum, in natural units, by one CTA.
template <typename T, int THREADS>
__device__ __noinline__ float2 slow_statistics(const T* row, int V, float row_max, float4* s_warp) {   // l, H
  const RowView<T> r(row, V);
  const int tid = threadIdx.x;
  float S = 0.f, Tn = 0.f;
  for (int j = tid; j < r.vectors; j += THREADS) {
    float v[Elem<T>::N];
    Elem<T>::unpack(r.load(j, -INFINITY), v);
#pragma unroll
    for (int i = 0; i < Elem<T>::N; ++i) {
      const float z = v[i] - row_max, e = exp2_fast(z * kLog2e);
      S += e;
      if (e > 0.f) Tn = fmaf(e, z, Tn);
    }
  }
  S = warp_add(S);
  Tn = warp_add(Tn);
  __syncthreads();
  if ((tid & 31) == 0) s_warp[tid >> 5] = make_float4(S, Tn, 0.f, 0.f);
  __syncthreads();
  S = Tn = 0.f;
  for (int i = 0; i < THREADS / 32; ++i) {
    S += s_warp[i].x;
    Tn += s_warp[i].y;
  }
  const float l = logf(S);
  return make_float2(l, fmaxf(l - Tn / S, 0.f));
}

constexpr int kMostCluster = 8;

// CLUSTERED: a row belongs to the CTAs of a cluster.  They hand their parts to the first one, and their groups' maxima to each other,
// by stores into its shared memory; behind the last barrier only the first one runs on.
template <typename T, int THREADS, bool TOP, bool CLUSTERED>
__global__ void __launch_bounds__(THREADS, (TOP || THREADS < 64 ? 1024 : 1280) / THREADS)   // (4096 x 128000: 182 us with 1024 threads an SM, 176 with 1280, 180 with 1536)
token_logprobs_kernel(LogprobArgs a) {
  using Scratch = TopScratch<THREADS>;
  constexpr int kWarps = THREADS / 32;
  // With 64 groups instead of 128 a bound for 20 alternatives lets through 24 elements instead of 22 and takes a quarter of the
  // comparisons: 9.9 us instead of 10.5 for 64 x 128000 fp32, 16.3 instead of 16.6 for 509 x 50001 fp16 (k = 5 and 20).
  const int groups = Scratch::kGroups == 128 && 3 * a.top_k <= 64 ? 64 : Scratch::kGroups;
  __shared__ float4 s_parts[CLUSTERED ? kMostCluster * kWarps : kWarps];   // of every warp of the row: maximum, c, S, T
  __shared__ float4 s_row;                                                 // maximum, l, H, whether they are still to come
  __shared__ typename std::conditional<TOP, Scratch, NoScratch<THREADS>>::type s_top;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = CLUSTERED ? (int)cluster.num_blocks() : 1, rank = CLUSTERED ? (int)cluster.block_rank() : 0;
  const int64_t m = CLUSTERED ? blockIdx.x / C : blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const RowView<T> r(static_cast<const T*>(a.logits) + m * a.ld, a.V);
  const int per = CLUSTERED ? (r.vectors + C - 1) / C : r.vectors, lo = rank * per, hi = min(lo + per, r.vectors);
  if constexpr (TOP) {
    if (tid < Scratch::kRanked) s_top.cand[tid] = 0;
    if (tid == 0) s_top.n = 0;
  }
  if constexpr (CLUSTERED) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");

  // the given token: requested here, its logit behind the pass, both used at the end
  int64_t id = 0;
  if (rank == 0 && tid == 0) id = id_at(a.ids, a.ids64, m);

  using Max = typename Elem<T>::Max;
  Max best = Elem<T>::lowest();
  float c = Elem<T>::kLow * kLog2e;
  PairSums sums{pair_of(0.f), pair_of(0.f)};
  float move = -INFINITY;   // a maximum above this moves c
  for (int j0 = lo; j0 < hi; j0 += kBatch * THREADS) {
    uint4 q[kBatch];
    if (j0 >= r.first_whole && j0 + kBatch * THREADS <= min(hi, r.end_whole)) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) q[u] = r.load_whole(j0 + u * THREADS + tid);
    } else {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int j = j0 + u * THREADS + tid;
        if (j < hi) {
          q[u] = r.load(j, -INFINITY);
        } else {
          float none[Elem<T>::N];
#pragma unroll
          for (int i = 0; i < Elem<T>::N; ++i) none[i] = -INFINITY;
          q[u] = Elem<T>::pack(none);
        }
      }
    }
    Max here = Elem<T>::of(q[0]);
#pragma unroll
    for (int u = 1; u < kBatch; ++u) here = Elem<T>::larger(here, Elem<T>::of(q[u]));
    best = Elem<T>::larger(best, here);
    const float top = Elem<T>::value(here);
    if (top > move) {
      move = top + kSlack;
      const float to = fmaxf(top, Elem<T>::kLow) * kLog2e, d = c - to;
      const Pair f = pair_of(exp2_fast(d));
      sums.T = mul2(fma2(pair_of(d), sums.S, sums.T), f);
      sums.S = mul2(sums.S, f);
      c = to;
    }
    const Pair minus_c = pair_of(-c);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) add_vector<T>(q[u], minus_c, sums);
  }
  float given = 0.f;
  if (rank == 0 && tid == 0 && id >= 0 && id < a.V) given = Elem<T>::load(r.row + id);

  const float own_max = Elem<T>::value(best);
  float s0, s1, t0, t1;
  split(sums.S, s0, s1);
  split(sums.T, t0, t1);
  const float4 part = joined(make_float4(own_max, c, s0 + s1, t0 + t1));
  if constexpr (CLUSTERED) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");   // the others run: their memory is there
  if (lane == 0) (CLUSTERED ? cluster.map_shared_rank(&s_parts[0], 0) : s_parts)[rank * kWarps + warp] = part;
  uint32_t best_key = 0;
  if constexpr (TOP) {
    if (lo + tid < hi) best_key = Elem<T>::key_of(own_max);   // (a thread without elements holds -inf and has key 0)
    const int each = THREADS / groups * C;                    // threads of a group: 1 to 32 neighbours
    uint32_t most = best_key;
    for (int o = each / 2; o > 0; o /= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const int to = lane % each;                               // the group's maximum goes to every CTA
    if (to < C) (CLUSTERED ? cluster.map_shared_rank(&s_top.group[0], to) : s_top.group)[rank * (groups / C) + tid / each] = most;
  }
  if constexpr (CLUSTERED) cluster.sync(); else __syncthreads();
  if constexpr (TOP) {
    if (tid < groups) {   // the k-th largest of the groups' maxima: the smallest that fewer than k exceed
      const uint32_t mine = s_top.group[tid];
      int more[4] = {0, 0, 0, 0};
#pragma unroll 8
      for (int i = 0; i < groups; i += 4) {
        const uint4 g = *reinterpret_cast<const uint4*>(s_top.group + i);
        more[0] += g.x > mine;
        more[1] += g.y > mine;
        more[2] += g.z > mine;
        more[3] += g.w > mine;
      }
      const uint32_t least = __reduce_min_sync(0xffffffffu, more[0] + more[1] + (more[2] + more[3]) < a.top_k ? mine : 0xffffffffu);
      if (lane == 0) s_top.least[warp] = least;
    }
  } else {
    if (rank != 0) return;
  }
  if (warp == kWarps - 1 && rank == 0) {
    const int n = C * kWarps;
    const float4 none = make_float4(-INFINITY, Elem<T>::kLow * kLog2e, 0.f, 0.f);
    float4 p = lane < n ? s_parts[lane] : none;
    if (CLUSTERED && n > 32) p = joined(p, lane + 32 < n ? s_parts[lane + 32] : none);
    p = joined(p);
    float row_max, l, H;
    bool far;
    statistics(p, Elem<T>::kLow, Elem<T>::kHigh, row_max, l, H, far);
    if (lane == 0) s_row = make_float4(row_max, l, H, far ? 1.f : 0.f);
  }
  __syncthreads();
  if constexpr (TOP) {
    const uint32_t bound = __reduce_min_sync(0xffffffffu, s_top.least[lane % (groups / 32)]);
    // Where many groups share the bound (rows of equal logits), or it is what masks are made of, the first k of the elements that
    // equal it are enough.
    int reach = 0;
    for (int i = 0; i < groups; i += 32) reach += s_top.group[i + lane] >= bound;
    const bool ties = bound > 0 && (bound <= Elem<T>::kMaskKey || __reduce_add_sync(0xffffffffu, reach) > a.top_k + groups / 4);
    collect<T, THREADS>(r, lo, hi, bound + ties, best_key, s_top, CLUSTERED ? cluster.map_shared_rank(&s_top.cand[0], 0) : s_top.cand,
                        CLUSTERED ? cluster.map_shared_rank(&s_top.n, 0) : &s_top.n);
    if (ties && rank == 0) collect_first<T, THREADS>(r.row, r.V, bound, a.top_k, s_top);
    if constexpr (CLUSTERED) cluster.sync(); else __syncthreads();
    if (rank != 0) return;
  }
  const float4 row = s_row;
  const float row_max = row.x;
  float l = row.y, H = row.z;
  if (row.w != 0.f) {
    const float2 slow = slow_statistics<T, THREADS>(r.row, r.V, row_max, s_parts);
    l = slow.x;
    H = slow.y;
  }
  const bool odd = row_max != row_max || row_max == INFINITY, dead = row_max == -INFINITY;
  if (tid == 0) {
    float lp = given - row_max - l;
    if (odd || id >= a.V) lp = kNan;
    else if (dead) lp = -INFINITY;
    if (id < 0) lp = 0.f;
    a.logprobs[m] = lp;
    a.entropy[m] = H;
    a.stats[2 * m] = row_max;
    a.stats[2 * m + 1] = l;
  }
  if constexpr (TOP) {
    const int k = a.top_k;
    int n = s_top.n;
    if (n > Scratch::kFew) {
      __syncthreads();   // everyone has read the count
      if (n > Scratch::kRoom) select_top<T, THREADS>(r.row, r.V, k, s_top);
      else keep_best<THREADS>(s_top, k);
      n = k;
    }
    rank_all<THREADS>(s_top, n, k);
    __syncthreads();
    for (int i = tid; i < k; i += THREADS) {
      const uint64_t key = s_top.top[i];
      const float x = Elem<T>::of_key((uint32_t)(key >> 32));
      a.top_ids[m * k + i] = (int32_t)~(uint32_t)key;
      a.top_logprobs[m * k + i] = odd ? kNan : dead ? -INFINITY : x - row_max - l;
    }
  }
}

// ---- gradient -----------------------------------------------------------------------------------------------------
struct GradArgs {
  const void* logits;
  int64_t ld;
  const void* ids;
  int ids64;
  const float *stats, *entropy, *g_lp, *g_entropy, *g_top;
  const int32_t* top_ids;
  int top_k;
  void* out;
  int64_t ldo;
  int V;
  unsigned chunks;   // CTAs of a row
  int per;           // vectors of a CTA
};

constexpr int kGradThreads = 128;   // at most

// A CTA is a piece of a row: element by element from the saved statistics.  A column that was given a gradient of its own is rounded
// once: the token's is added where its thread comes by, the alternatives' columns are computed once more at the end.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kGradThreads, 8)
token_logprobs_grad_kernel(GradArgs a) {
  constexpr int N = Elem<T>::N, kGiven = TOP ? kMaxTop + 1 : 1;
  __shared__ int s_id[kGiven];
  __shared__ float s_g[kGiven];
  const int64_t m = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x - m * a.chunks), tid = threadIdx.x, threads = blockDim.x;
  const RowView<T> r(static_cast<const T*>(a.logits) + m * a.ld, a.V);
  T* out = static_cast<T*>(a.out) + m * a.ldo;   // at the same place within 16 bytes as the row
  const int lo = chunk * a.per, hi = min(lo + a.per, r.vectors);

  // the first logits are on their way before the row's coefficients are asked for
  uint4 q[kBatch];
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    const int j = lo + u * threads + tid;
    if (j < hi) q[u] = r.load(j, 0.f);
  }
  // what entry i was given: 0 is the token, 1 .. top_k the alternatives
  auto given = [&](int i, int& column, float& g) {
    int64_t id = -1;
    g = 0.f;
    if (i == 0) {
      if (a.g_lp != nullptr) { id = id_at(a.ids, a.ids64, m); g = a.g_lp[m]; }
    } else {
      id = a.top_ids[m * a.top_k + i - 1];
      g = a.g_top[m * a.top_k + i - 1];
    }
    if (id < 0) g = 0.f;
    if (id >= a.V) g = kNan;
    column = id >= 0 && id < a.V ? (int)id : -1;
  };
  const float mx = a.stats[2 * m], l = a.stats[2 * m + 1];
  const float gh = a.g_entropy != nullptr ? a.g_entropy[m] : 0.f;
  const float h = a.g_entropy != nullptr ? a.entropy[m] : 0.f;
  int column = -1;
  float own = 0.f, G = 0.f;
  if constexpr (TOP) {
    for (int i = tid; i <= a.top_k; i += threads) given(i, s_id[i], s_g[i]);
    __syncthreads();
    for (int i = 0; i <= a.top_k; ++i) G += s_g[i];
  } else {
    given(0, column, own);
    G = own;
  }
  const int own_vector = column < 0 ? -1 : (column + r.skew) / N, own_place = (column + r.skew) % N;

  // -p (G + gh (ln p + h)) with ln p = x - mx - l: any value.  A row without a live logit has p = 0; NaN in G, of a token that is no column,
  // is kept there too.
  const bool dead = mx == -INFINITY && G == G;
  const float base = fmaf(gh, h, G);
  auto gradient = [&](float x) -> float {
    const float lp = max_nan(x - mx - l, -200.f);   // e^-200 is 0
    return dead ? 0.f : -exp2_fast(lp * kLog2e) * fmaf(gh, lp, base);
  };
  // The same as 2^y (slope y + level), y = x log2(e) - c: half the instructions, for maxima whose log2(e) multiple is fine
  // enough.  c is mx log2(e) rounded; what the rounding left, and e^-l, are in the factor.
  const bool near = mx >= Elem<T>::kLow && mx <= Elem<T>::kHigh;
  const float c = mx * kLog2e, rest = -fmaf(mx, kLog2e, -c);
  const float scale = -exp2f(rest) * expf(-l);
  const Pair slope = pair_of(scale * gh * kLn2), level = pair_of(scale * fmaf(gh, fmaf(rest, kLn2, -l) + h, G)), minus_c = pair_of(-c);
  for (int j0 = lo; j0 < hi; j0 += kBatch * threads) {
    if (j0 > lo) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int j = j0 + u * threads + tid;
        if (j < hi) q[u] = r.load(j, 0.f);
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int j = j0 + u * threads + tid;
      if (j >= hi) continue;
      float v[N];
      if (near) {
        Elem<T>::clamped(q[u], v);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const Pair y = fma2(pair_of(v[i], v[i + 1]), pair_of(kLog2e), minus_c);
          float y0, y1;
          split(y, y0, y1);
          split(mul2(pair_of(exp2_fast(y0), exp2_fast(y1)), fma2(y, slope, level)), v[i], v[i + 1]);
        }
      } else {
        Elem<T>::unpack(q[u], v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = gradient(v[i]);
      }
      if (!TOP && j == own_vector) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += i == own_place ? own : 0.f;
      }
      if (r.whole(j)) {
        __stcs(reinterpret_cast<uint4*>(out - r.skew) + j, Elem<T>::pack(v));
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int col = r.column(j) + i;
          if (col >= 0 && col < a.V) Elem<T>::store(out + col, v[i]);
        }
      }
    }
  }
  if constexpr (TOP) {
    __syncthreads();   // the columns below were written by other threads of this block
    for (int n = tid; n <= a.top_k; n += threads) {
      const int id = s_id[n];
      const int j = id < 0 ? -1 : (id + r.skew) / N;
      if (id < 0 || j < lo || j >= hi) continue;
      bool first = true;
      float sum = 0.f;
      for (int i = 0; i <= a.top_k; ++i) {   // a column may have been given more than one
        if (s_id[i] != id) continue;
        if (i < n) first = false;
        sum += s_g[i];
      }
      if (first) Elem<T>::store(out + id, gradient(Elem<T>::load(r.row + id)) + sum);
    }
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------
// Threads of a CTA, which is one row.  A small CTA lets more rows overlap their ends with each other's passes, a large one takes
// a row in fewer steps.  So: halved while the rows fill the chip twice over with half the threads (a wave is 148 x 1024) and
// a thread has less than 16 vectors (15 without alternatives).  us, 96 MB of bf16 rows, top 5, 32 / 64 / 128 / 256 threads: V=1000 64 / 123 /
// 263 / 407, 4000 30 / 40 / 69 / 108, 8000 27 / 29 / 43 / 57, 16000 29 / 26 / 30 / 38, 32000 38 / 28 / 26 / 28, 128000 100 / 55 / 34 / 26; no
// alternatives, V=8000 21.2 / 20.2 / 22.3 / 28.9, 16000 23.6 / 21.1 / 20.3 / 23.2; 128 rows of 4000, top 5, 6.3 / 5.3 / 5.0 / 4.8.
// Below 128 threads, which are then the groups, a top_k above a third of them lets more candidates through, and it pays for short
// rows alone (48 MB, top 20, 32 / 64 threads: V=1000 48 / 70, 2000 34 / 39, 4000 28 / 25), above 5/8 not at all (top 32 122 / 83).
int threads_of(int64_t M, int64_t vectors, int top_k) {
  int threads = 256;
  while (threads > 32 && M * threads > 148 * 512) {
    const int groups = threads / 2;
    const int least = top_k == 0 ? 15 : groups >= 128 || 3 * top_k <= groups ? 16 : 8 * top_k <= 5 * groups ? 6 : 0;
    if (vectors >= least * threads) break;
    threads /= 2;
  }
  return threads;
}

// CTAs of a row: long rows are cut, into as many as half fill the chip, or fill it if a piece stays long.  The barriers
// of a cluster cost 1.5 us (less without alternatives), and every piece an end.  us, bf16, top 20, 1 / 2 / 4 / 8: 16 rows of 50001 9.1 / 7.8 / 7.1 / 6.7 (of 32000, top 5,
// 6.0 / 6.7 / 6.2 / 6.7); 64 of 128000 14.7 / 11.2 / 9.4 / 10.6; 128 of 50001 9.9 / 9.8 / 11.1 / 16.5; 300 of 128000 25.4 / 22.9 / 26.5 / 38.5;
// 509 of 50001 17.2 / 22.1 / 33.0 / 54.4.
int cluster_of(int64_t M, int64_t bytes, int top_k) {
  int C = 1;
  if (bytes >= (top_k > 0 ? 64 : 32) * 1024)
    while (C < kMostCluster && (M * C * 2 <= 2 * 148 || (M * C * 2 <= 4 * 148 && bytes / (2 * C) >= 48 * 1024))) C *= 2;
  return C;
}

template <typename T, int THREADS, bool CLUSTERED>
int launch_forward(const LogprobArgs& a, int C, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.M * C));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTERED ? 1 : 0;
  XKB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, a.top_k > 0 ? token_logprobs_kernel<T, THREADS, true, CLUSTERED>
                                                      : token_logprobs_kernel<T, THREADS, false, CLUSTERED>, a));
  XKB_CHECK_LAUNCH("token_logprobs_kernel");
  return XKB_OK;
}

template <typename T>
int forward_typed(const LogprobArgs& a, cudaStream_t s) {
  const int64_t bytes = (int64_t)a.V * (int64_t)sizeof(T);
  switch (threads_of(a.M, ceil_div(bytes, (int64_t)16), a.top_k)) {
    case 32: return launch_forward<T, 32, false>(a, 1, s);
    case 64: return launch_forward<T, 64, false>(a, 1, s);
    case 128: return launch_forward<T, 128, false>(a, 1, s);
  }
  const int C = cluster_of(a.M, bytes, a.top_k);
  return C > 1 ? launch_forward<T, 256, true>(a, C, s) : launch_forward<T, 256, false>(a, 1, s);
}

template <typename T>
int backward_typed(GradArgs a, int64_t M, cudaStream_t s) {
  XKB_REQUIRE((reinterpret_cast<uintptr_t>(a.logits) - reinterpret_cast<uintptr_t>(a.out)) % 16 == 0 &&
                  (M == 1 || (a.ld - a.ldo) * (int64_t)sizeof(T) % 16 == 0),
              "token_logprobs_backward: a row of grad_logits must start at the same place within 16 bytes as the row of logits");
  XKB_REQUIRE(reinterpret_cast<uintptr_t>(a.logits) % sizeof(T) == 0, "token_logprobs_backward: misaligned logits");
  // Pieces of a row: about 16 vectors a thread, or as few as one batch where the rows do not fill the chip (148 x 8 CTAs).  Small CTAs, many
  // of them resident, cover each other's beginnings and ends.  us, bf16, 256 threads in pieces of up to 8192 vectors / here: 4096 x 128000
  // 332 / 320, 1000 x 128000 90 / 84, 5000 x 20000 81 / 69, 12000 x 9000 with 5 alternatives 101 / 77, 40 x 128000 6.6 / 6.2; 592 x 32000
  // 11.6 / 12.1.  Whole rows of up to 1280 vectors take 64 threads (12000 x 9000 with 128: 80; 3171 x 8190 the other way round, 18.5 and 19.0).
  const int64_t vectors = ceil_div((int64_t)a.V + Elem<T>::N - 1, Elem<T>::N), fill = 148 * 8;
  int64_t chunks = ceil_div(vectors, (int64_t)16 * kGradThreads);
  if (M * chunks < fill) {
    const int64_t batches = ceil_div(vectors, (int64_t)kBatch * kGradThreads), want = ceil_div(fill, M);
    chunks = want < batches ? want : batches;
  }
  const int64_t per = ceil_div(vectors, chunks), most = per <= 1280 && M * chunks >= fill ? kGradThreads / 2 : kGradThreads;
  XKB_REQUIRE(M * chunks <= 0x7fffffff, "token_logprobs_backward: %lld rows of %d columns do not fit a grid", (long long)M, a.V);
  a.chunks = (unsigned)chunks;
  a.per = (int)per;
  const int64_t need = align_up(ceil_div(per, (int64_t)kBatch), 32);
  const unsigned threads = (unsigned)(need < most ? need : most);
  (a.top_k > 0 ? token_logprobs_grad_kernel<T, true> : token_logprobs_grad_kernel<T, false>)<<<(unsigned)(M * chunks), threads, 0, s>>>(a);
  XKB_CHECK_LAUNCH("token_logprobs_grad_kernel");
  return XKB_OK;
}

constexpr int64_t kMaxColumns = 0x7fffffff - 4096;   // columns behind the row's end, of threads without a vector, are numbers too

}  // namespace
}  // namespace xkb

extern "C" int xkb_token_logprobs(const void* logits, int dtype, int64_t ld, const void* token_ids, int ids64, float* logprobs,
                                  float* entropy, float* stats, float* top_logprobs, int32_t* top_ids, int64_t M, int64_t V,
                                  int top_k, void* stream) {
  using namespace xkb;
  XKB_REQUIRE(M >= 0 && V >= 1 && V <= kMaxColumns, "token_logprobs: bad shape M=%lld V=%lld", (long long)M, (long long)V);
  XKB_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= V, "token_logprobs: top_k must satisfy 0 <= top_k <= min(V, %d) (got top_k=%d, V=%lld)",
              kMaxTop, top_k, (long long)V);
  XKB_REQUIRE(dtype == XKB_BF16 || dtype == XKB_F32 || dtype == XKB_F16, "token_logprobs: unsupported logits dtype code %d", dtype);
  XKB_REQUIRE(ids64 == 0 || ids64 == 1, "token_logprobs: ids64 must be 0 or 1");
  if (M == 0) return XKB_OK;
  XKB_REQUIRE(ld >= 0 && M <= 0x7fffffff / 8, "token_logprobs: bad row stride or too many rows");
  XKB_REQUIRE(logits && token_ids && logprobs && entropy && stats && (top_k == 0 || (top_logprobs && top_ids)),
              "token_logprobs: null pointer");
  XKB_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == XKB_F32 ? 4 : 2) == 0, "token_logprobs: misaligned logits");
  XKB_REQUIRE(address_bits(token_ids) % (ids64 ? 8 : 4) == 0 && address_bits(logprobs, entropy, stats, top_logprobs, top_ids) % 4 == 0,
              "token_logprobs: a misaligned tensor");
  const LogprobArgs a{logits, ld, token_ids, ids64, logprobs, entropy, stats, top_logprobs, top_ids, M, (int)V, top_k};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case XKB_BF16: return forward_typed<__nv_bfloat16>(a, s);
    case XKB_F32: return forward_typed<float>(a, s);
    default: return forward_typed<__half>(a, s);
  }
}

extern "C" int xkb_token_logprobs_backward(const void* logits, int dtype, int64_t ld, const void* token_ids, int ids64,
                                           const float* stats, const float* entropy, const float* grad_logprobs,
                                           const float* grad_entropy, const int32_t* top_ids, const float* grad_top_logprobs,
                                           int top_k, void* grad_logits, int64_t ld_grad, int64_t M, int64_t V, void* stream) {
  using namespace xkb;
  XKB_REQUIRE(M >= 0 && V >= 1 && V <= kMaxColumns, "token_logprobs_backward: bad shape M=%lld V=%lld", (long long)M, (long long)V);
  XKB_REQUIRE(top_k >= 0 && top_k <= kMaxTop, "token_logprobs_backward: top_k must be between 0 and %d (got %d)", kMaxTop, top_k);
  XKB_REQUIRE(dtype == XKB_BF16 || dtype == XKB_F32 || dtype == XKB_F16,
              "token_logprobs_backward: unsupported logits dtype code %d", dtype);
  XKB_REQUIRE(ids64 == 0 || ids64 == 1, "token_logprobs_backward: ids64 must be 0 or 1");
  if (M == 0) return XKB_OK;
  XKB_REQUIRE(ld >= 0 && (M == 1 || ld_grad >= V) && M <= 0x7fffffff, "token_logprobs_backward: bad row stride or too many rows");
  XKB_REQUIRE(logits && stats && grad_logits, "token_logprobs_backward: null pointer");
  XKB_REQUIRE(grad_logprobs == nullptr || token_ids != nullptr, "token_logprobs_backward: grad_logprobs without token_ids");
  XKB_REQUIRE(grad_entropy == nullptr || entropy != nullptr, "token_logprobs_backward: grad_entropy without entropy");
  XKB_REQUIRE(grad_top_logprobs == nullptr || top_k == 0 || top_ids != nullptr, "token_logprobs_backward: grad_top_logprobs without top_ids");
  XKB_REQUIRE(address_bits(token_ids) % (ids64 ? 8 : 4) == 0 &&
                  address_bits(stats, entropy, grad_logprobs, grad_entropy, top_ids, grad_top_logprobs) % 4 == 0,
              "token_logprobs_backward: a misaligned tensor");
  GradArgs a{logits, ld, token_ids, ids64, stats, entropy, grad_logprobs, grad_entropy, grad_top_logprobs, top_ids,
             grad_top_logprobs == nullptr ? 0 : top_k, grad_logits, ld_grad, (int)V, 0, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case XKB_BF16: return backward_typed<__nv_bfloat16>(a, M, s);
    case XKB_F32: return backward_typed<float>(a, M, s);
    default: return backward_typed<__half>(a, M, s);
  }
}
