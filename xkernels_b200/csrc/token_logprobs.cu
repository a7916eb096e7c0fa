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
// these maxima bounds the row's k-th largest element from below, and only the k threads that reach it can hold one of the k:
// their elements (4 % of a row at k = 20) are read again, out of the L2, and what reaches the bound is ranked.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace xkb {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTop = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kSlack = 11.f;              // 2^16
constexpr float kNan = __builtin_nanf("");

__device__ __forceinline__ float exp2_fast(float x) {   // 2 ulp; subnormal results are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Two fp32 values side by side: one instruction does both.
struct Pair { uint64_t v; };
__device__ __forceinline__ Pair pair_of(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ Pair pair_of(float v) { return pair_of(v, v); }
__device__ __forceinline__ void split(Pair p, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p.v)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}

// What a type of logits needs: N elements in 16 bytes, a running maximum of whole vectors, ordered keys.
//   kClamp: smaller elements count as this, which keeps -inf out of the products.  A row whose maximum is not between kLow
//   and kHigh, where a clamped element would count or x log2(e) is too coarse, takes the slow pass.
//   key_of: ascending with the value; NaN above all, -0 as +0, never 0 (that is "no element").
template <typename T> struct Elem;

template <> struct Elem<float> {
  static constexpr int N = 4;
  static constexpr float kClamp = -1e8f, kLow = -1e6f, kHigh = 1e6f;
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
    if (v != v) return 0xffffffffu;
    const uint32_t u = __float_as_uint(v + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
  }
  static __device__ __forceinline__ float of_key(uint32_t k) {
    if (k == 0xffffffffu) return kNan;
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
  }
};

template <> struct Elem<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr float kClamp = -1e8f, kLow = -1e6f, kHigh = 1e6f;
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

// The largest key t of which at least k of the n keys are >= t (0 if fewer than k are above 0): a search by two bits at a time
// from the first one in which the keys differ, by one warp that holds the keys in registers.
template <int THREADS>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t* keys, int k) {
  const int lane = threadIdx.x & 31;
  uint32_t key[THREADS / 32], most = 0, least = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    key[i] = keys[i * 32 + lane];
    most = max(most, key[i]);
    least = min(least, key[i]);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  least = __reduce_min_sync(0xffffffffu, least);
  if (most == least) return most;
  int b = (31 - __clz(most ^ least)) & ~1;         // the upper of two bits is b + 1
  uint32_t t = b == 30 ? 0u : most >> (b + 2) << (b + 2);
  for (; b >= 0; b -= 2) {
    uint32_t n = 0;   // how many reach t + 1, t + 2, t + 3 in units of this step: fields of ten bits (THREADS < 1024)
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      // (equal bits above the step: everything that is not below t)
      const uint32_t d = key[i] >= t ? min((key[i] - t) >> b, 3u) : 0u;
      n += d == 0 ? 0u : d == 1 ? 1u : d == 2 ? 1u + (1u << 10) : 1u + (1u << 10) + (1u << 20);
    }
    n = __reduce_add_sync(0xffffffffu, n);
    const uint32_t step = (int)(n >> 20) >= k ? 3u : (int)(n >> 10 & 1023u) >= k ? 2u : (int)(n & 1023u) >= k ? 1u : 0u;
    t += step << b;
  }
  return t;
}

constexpr int kBatch = 4;   // vectors a thread requests before it uses the first (select_top names them one by one)

template <int THREADS>
struct TopScratch {
  uint64_t cand[8 * THREADS + kMaxTop];   // value key, ~column: all different, larger is better
  uint64_t top[kMaxTop];                  // the CTA's best ones, in order
  uint32_t key[THREADS];                  // of every thread
  int owner[THREADS];                     // threads whose elements are read again
  int n, owners, want;
  uint32_t bound;
};
template <int THREADS> struct NoScratch {};

// Leaves the k largest of the n candidates (n > k) at the front, in any order.
template <int THREADS>
__device__ __noinline__ void keep_best(TopScratch<THREADS>& s, int k) {
  const int n = s.n;
  uint64_t t = 0;
#pragma unroll 1
  for (int b = 63; b >= 0; --b) {
    const uint64_t trial = t | (1ull << b);
    int mine = 0, all = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) mine += s.cand[i] >= trial;
    // (at most 9 a thread: four counts of one bit)
#pragma unroll
    for (int w = 0; w < 4; ++w) all += __syncthreads_count((mine >> w) & 1) << w;
    if (all >= k) t = trial;
  }
  uint64_t mine[9];   // 9 THREADS > 8 THREADS + kMaxTop
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    const int at = threadIdx.x + i * THREADS;
    mine[i] = at < n ? s.cand[at] : 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 9; ++i)
    if (mine[i] != 0 && mine[i] >= t) s.cand[atomicAdd(&s.n, 1)] = mine[i];
  __syncthreads();
}

// The k best of n <= THREADS candidates, in order, to `to`; unfilled places are 0.
template <int THREADS>
__device__ __forceinline__ void rank_all(const uint64_t* cand, int n, int k, uint64_t* to) {
  for (int i = threadIdx.x; i < k; i += THREADS)
    if (i >= n) to[i] = 0;
  if ((int)threadIdx.x < n) {
    const uint64_t mine = cand[threadIdx.x];
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += cand[i] > mine;
    if (rank < k) to[rank] = mine;
  }
}

// The k largest elements of the CTA's vectors [lo, hi) to s.top, ordered; `best` is the maximum of this thread's vectors.
template <typename T, int THREADS>
__device__ void select_top(const RowView<T>& r, int lo, int hi, uint32_t best, int k, TopScratch<THREADS>& s) {
  constexpr int N = Elem<T>::N;
  const int tid = threadIdx.x, per = (hi - lo + THREADS - 1) / THREADS;   // vectors of a thread, at most
  s.key[tid] = best;
  __syncthreads();
  if (tid < 32) {
    const uint32_t t = kth_largest<THREADS>(s.key, k);
    if (tid == 0) {
      s.bound = t;
      s.n = s.owners = s.want = 0;
    }
  }
  __syncthreads();
  const uint32_t bound = s.bound;
  // Several threads may share the bound.  A few too many are taken; of a crowd (rows of equal logits) only those whose first
  // element of that value comes first, which each looks for in its own vectors.
  uint32_t last = 0xffffffffu;   // an element equal to the bound counts up to this column
  bool mine = best > 0 && best >= bound;
  const int reach = __syncthreads_count(mine);
  if (bound > 0 && reach > 2 * k + 32) {
    const int above = __syncthreads_count(best > bound);
    uint32_t at = 0xffffffffu;
    if (best == bound) {
      for (int j = lo + tid; j < hi && at == 0xffffffffu; j += THREADS) {
        float v[N];
        Elem<T>::unpack(r.load(j, 0.f), v);
#pragma unroll
        for (int i = N - 1; i >= 0; --i) {
          const int col = r.column(j) + i;
          if (col >= 0 && col < r.V && Elem<T>::key_of(v[i]) == bound) at = (uint32_t)col;
        }
      }
    }
    s.key[tid] = best == bound ? ~at : 0u;
    __syncthreads();
    if (tid < 32) {
      const uint32_t t = kth_largest<THREADS>(s.key, k - above);
      if (tid == 0) s.bound = t;
    }
    __syncthreads();
    last = ~s.bound;
    mine = best > bound || (best == bound && at <= last);
  }
  if (mine) s.owner[atomicAdd(&s.owners, 1)] = tid;
  __syncthreads();
  const int items = s.owners * per;
  auto counts = [&](float v, int col) -> bool {
    const uint32_t key = Elem<T>::key_of(v);
    return col >= 0 && col < r.V && (key > bound || (key == bound && (uint32_t)col <= last));
  };
  auto push = [&](float v, int col) {
    s.cand[atomicAdd(&s.n, 1)] = (uint64_t)Elem<T>::key_of(v) << 32 | (uint32_t)~(uint32_t)col;
  };
  for (int base = 0; base < items; base += kBatch * THREADS) {
    // some vectors of every thread at once, their candidates counted before any is put down
    uint4 q[kBatch];
    int at[kBatch], n = 0;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int it = base + u * THREADS + tid;
      at[u] = -1;
      if (it < items) {
        const int j = lo + s.owner[it / per] + it % per * THREADS;
        if (j < hi) {
          at[u] = j;
          q[u] = r.load(j, 0.f);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (at[u] < 0) continue;
      float v[N];
      Elem<T>::unpack(q[u], v);
#pragma unroll
      for (int i = 0; i < N; ++i) n += counts(v[i], r.column(at[u]) + i);
    }
    if (n > 0) atomicAdd(&s.want, n);
    __syncthreads();
    const int have = s.n, want = s.want;
    __syncthreads();
    if (tid == 0) s.want = 0;
    const bool fits = have + want <= 8 * THREADS + kMaxTop;
#pragma unroll 1
    for (int u = 0; u < kBatch; ++u) {
      if (!fits) {   // one vector a thread at a time, what is there cut down to k before
        __syncthreads();
        const int now = s.n;
        __syncthreads();
        if (now > kMaxTop) keep_best<THREADS>(s, k);
      }
      const int j = u == 0 ? at[0] : u == 1 ? at[1] : u == 2 ? at[2] : at[3];
      if (j < 0 || n == 0) continue;
      const uint4 w = u == 0 ? q[0] : u == 1 ? q[1] : u == 2 ? q[2] : q[3];
      float v[N];
      Elem<T>::unpack(w, v);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (counts(v[i], r.column(j) + i)) push(v[i], r.column(j) + i);
    }
    __syncthreads();
  }
  const int found = s.n;
  __syncthreads();
  if (found > THREADS) keep_best<THREADS>(s, k);
  rank_all<THREADS>(s.cand, found > THREADS ? k : found, k, s.top);
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

template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
token_logprobs_kernel(LogprobArgs a) {
  constexpr int kWarps = THREADS / 32;
  __shared__ float4 s_warp[kWarps];                 // a warp's maximum, c, S, T
  __shared__ float4 s_part;                         // the CTA's
  __shared__ typename std::conditional<TOP, TopScratch<THREADS>, NoScratch<THREADS>>::type s_top;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t m = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const RowView<T> r(static_cast<const T*>(a.logits) + m * a.ld, a.V);
  const int per = (r.vectors + C - 1) / C, lo = rank * per, hi = min(lo + per, r.vectors);

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
  Sums s{c, 0.f, 0.f};
  {
    float s0, s1, t0, t1;
    split(sums.S, s0, s1);
    split(sums.T, t0, t1);
    s.S = s0 + s1;
    s.T = t0 + t1;
  }

  // the CTA's sums, at the reference of its maximum
  const float own_max = Elem<T>::value(best);
  auto joined = [](float4 p) -> float4 {   // p: maximum, c, S, T of a lane
    const float mx = warp_max_nan(p.x);
    Sums t{p.y, p.z, p.w};
    float c = p.y;   // the largest c: no factor exceeds 1
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, o));
    t.move_to(c);
    return make_float4(mx, c, warp_add(t.S), warp_add(t.T));
  };
  const float4 w = joined(make_float4(own_max, s.c, s.S, s.T));
  if (lane == 0) s_warp[warp] = w;
  __syncthreads();
  const float4 none = make_float4(-INFINITY, Elem<T>::kLow * kLog2e, 0.f, 0.f);
  if (warp == 0) {
    const float4 all = joined(lane < kWarps ? s_warp[lane] : none);
    if (lane == 0) s_part = all;
  }
  if constexpr (TOP) {
    // (a thread without elements holds -inf: its key must be 0)
    const uint32_t key = lo + tid < hi ? Elem<T>::key_of(own_max) : 0u;
    select_top<T, THREADS>(r, lo, hi, key, a.top_k, s_top);
  }
  __syncthreads();

  // the row's: the parts of all CTAs, one a lane
  float4 part = s_part;
  if (C > 1) {
    cluster.sync();
    part = none;
    if (lane < C) part = *cluster.map_shared_rank(&s_part, lane);
    part = joined(part);
  }
  const float row_max = part.x;
  float l, H;
  const bool odd = row_max != row_max || row_max == INFINITY, dead = row_max == -INFINITY;
  if (!odd && !dead && (row_max < Elem<T>::kLow || row_max > Elem<T>::kHigh)) {
    // slow pass: differences from the maximum, natural units
    if (C > 1) cluster.sync();   // everyone has read the maxima
    float S = 0.f, Tn = 0.f;
    for (int j = lo + tid; j < hi; j += THREADS) {
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
    if (lane == 0) s_warp[warp] = make_float4(0.f, 0.f, S, Tn);
    __syncthreads();
    if (tid == 0) {
      S = Tn = 0.f;
      for (int i = 0; i < kWarps; ++i) { S += s_warp[i].z; Tn += s_warp[i].w; }
      s_part = make_float4(row_max, 0.f, S, Tn);
    }
    if (C > 1) cluster.sync(); else __syncthreads();
    S = Tn = 0.f;
    for (int i = 0; i < C; ++i) {
      const float4 p = C > 1 ? *cluster.map_shared_rank(&s_part, i) : s_part;
      S += p.z;
      Tn += p.w;
    }
    l = logf(S);
    H = fmaxf(l - Tn / S, 0.f);
  } else if (odd) {
    l = H = kNan;
  } else if (dead) {
    l = H = 0.f;
  } else {
    const float at_max = row_max * kLog2e;
    Sums t{part.y, part.z, part.w};
    t.move_to(at_max);
    // at_max is row_max log2(e) but for its rounding, which is in every e: ln sum exp(x - row_max) = ln2 (log2 S + at_max - row_max log2(e))
    const float off = -fmaf(row_max, kLog2e, -at_max), log2s = log2f(t.S);
    l = (log2s + off) * kLn2;
    H = fmaxf((log2s - t.T / t.S) * kLn2, 0.f);
  }
  if (rank == 0 && tid == 0) {
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
    if (rank == 0) {
      const uint64_t* best_of_row = s_top.top;
      if (C > 1) {   // the CTAs' best ones, ranked once more
        for (int i = tid; i < C * k; i += THREADS) s_top.cand[i] = cluster.map_shared_rank(s_top.top, i / k)[i % k];
        __syncthreads();
        uint64_t* to = s_top.cand + 8 * kMaxTop;
        for (int i = tid; i < C * k; i += THREADS) {   // (places a CTA did not fill are 0 and come last)
          const uint64_t mine = s_top.cand[i];
          int above = 0;
          for (int n = 0; n < C * k; ++n) above += s_top.cand[n] > mine;
          if (mine != 0 && above < k) to[above] = mine;
        }
        __syncthreads();
        best_of_row = to;
      }
      for (int i = tid; i < k; i += THREADS) {
        const uint64_t key = best_of_row[i];
        const float x = Elem<T>::of_key((uint32_t)(key >> 32));
        a.top_ids[m * k + i] = (int32_t)~(uint32_t)key;
        a.top_logprobs[m * k + i] = odd ? kNan : dead ? -INFINITY : x - row_max - l;
      }
    }
  }
  if (C > 1) cluster.sync();   // the others' shared memory is read until here
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

constexpr int kGradThreads = 256;

// A CTA is a piece of a row: element by element from the saved statistics, then the columns that were given a gradient of
// their own once more, so that each is rounded once.
template <typename T>
__global__ void __launch_bounds__(kGradThreads)
token_logprobs_grad_kernel(GradArgs a) {
  constexpr int N = Elem<T>::N;
  __shared__ int s_id[kMaxTop + 1];
  __shared__ float s_g[kMaxTop + 1];
  const int64_t m = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x - m * a.chunks), tid = threadIdx.x;
  const RowView<T> r(static_cast<const T*>(a.logits) + m * a.ld, a.V);
  T* out = static_cast<T*>(a.out) + m * a.ldo;   // at the same place within 16 bytes as the row
  const int lo = chunk * a.per, hi = min(lo + a.per, r.vectors);

  // the row's coefficients; entry 0 is the given token, 1 .. top_k the alternatives
  for (int i = tid; i <= a.top_k; i += kGradThreads) {
    int64_t id = -1;
    float g = 0.f;
    if (i == 0) {
      if (a.g_lp != nullptr) { id = id_at(a.ids, a.ids64, m); g = a.g_lp[m]; }
    } else if (a.g_top != nullptr) {
      id = a.top_ids[m * a.top_k + i - 1];
      g = a.g_top[m * a.top_k + i - 1];
    }
    if (id < 0) g = 0.f;
    if (id >= a.V) g = kNan;
    s_id[i] = id >= 0 && id < a.V ? (int)id : -1;
    s_g[i] = g;
  }
  const float mx = a.stats[2 * m], l = a.stats[2 * m + 1];
  const float gh = a.g_entropy != nullptr ? a.g_entropy[m] : 0.f;
  const float h = a.g_entropy != nullptr ? a.entropy[m] : 0.f;
  __syncthreads();
  float G = 0.f;
  for (int i = 0; i <= a.top_k; ++i) G += s_g[i];
  // -p (G + gh (ln p + h)) with ln p = x - mx - l: any value
  const bool dead = mx == -INFINITY;
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
  for (int j0 = lo; j0 < hi; j0 += kBatch * kGradThreads) {
    uint4 q[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int j = j0 + u * kGradThreads + tid;
      if (j < hi) q[u] = r.load(j, 0.f);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int j = j0 + u * kGradThreads + tid;
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
      if (r.whole(j)) {
        *(reinterpret_cast<uint4*>(out - r.skew) + j) = Elem<T>::pack(v);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int col = r.column(j) + i;
          if (col >= 0 && col < a.V) Elem<T>::store(out + col, v[i]);
        }
      }
    }
  }
  __syncthreads();   // the columns below were written by other threads of this block
  if (tid <= a.top_k) {
    const int id = s_id[tid];
    const int j = id < 0 ? -1 : (id + r.skew) / N;
    if (id >= 0 && j >= lo && j < hi) {
      bool first = true;
      float own = 0.f;
      for (int i = 0; i <= a.top_k; ++i) {   // a column may have been given more than one
        if (s_id[i] != id) continue;
        if (i < tid) first = false;
        own += s_g[i];
      }
      if (first) Elem<T>::store(out + id, gradient(Elem<T>::load(r.row + id)) + own);
    }
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------
template <typename T, int THREADS, bool TOP>
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
  cfg.numAttrs = C > 1 ? 1 : 0;
  XKB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, THREADS, TOP>, a));
  XKB_CHECK_LAUNCH("token_logprobs_kernel");
  return XKB_OK;
}

constexpr int kThreads = 256;

// CTAs per row: few rows are cut so that the chip is full, as long as a piece keeps some vectors for every thread.
int cluster_of(int64_t M, int64_t bytes) {
  int C = 1;
  while (C < 8 && M * C * 2 <= 148 * (1024 / kThreads) && bytes / (2 * C) >= 16 * kThreads) C *= 2;
  return C;
}

template <typename T>
int forward_typed(const LogprobArgs& a, cudaStream_t s) {
  const int C = cluster_of(a.M, (int64_t)a.V * (int64_t)sizeof(T));
  return a.top_k > 0 ? launch_forward<T, kThreads, true>(a, C, s) : launch_forward<T, kThreads, false>(a, C, s);
}

template <typename T>
int backward_typed(GradArgs a, int64_t M, cudaStream_t s) {
  XKB_REQUIRE((reinterpret_cast<uintptr_t>(a.logits) - reinterpret_cast<uintptr_t>(a.out)) % 16 == 0 &&
                  (M == 1 || (a.ld - a.ldo) * (int64_t)sizeof(T) % 16 == 0),
              "token_logprobs_backward: a row of grad_logits must start at the same place within 16 bytes as the row of logits");
  XKB_REQUIRE(reinterpret_cast<uintptr_t>(a.logits) % sizeof(T) == 0, "token_logprobs_backward: misaligned logits");
  const int64_t vectors = ceil_div((int64_t)a.V + Elem<T>::N - 1, Elem<T>::N);
  int64_t per = 2 * kBatch * kGradThreads;
  while (per > kGradThreads && M * ceil_div(vectors, per) < 4 * 148) per /= 2;
  const int64_t chunks = ceil_div(vectors, per);
  XKB_REQUIRE(M * chunks <= 0x7fffffff, "token_logprobs_backward: %lld rows of %d columns do not fit a grid", (long long)M, a.V);
  a.chunks = (unsigned)chunks;
  a.per = (int)per;
  token_logprobs_grad_kernel<T><<<(unsigned)(M * chunks), kGradThreads, 0, s>>>(a);
  XKB_CHECK_LAUNCH("token_logprobs_grad_kernel");
  return XKB_OK;
}

constexpr int64_t kMaxColumns = 0x7fffffff - 64;

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
  XKB_REQUIRE(ld >= 0 && (M == 1 || ld_grad >= V), "token_logprobs_backward: bad row stride");
  XKB_REQUIRE(logits && stats && grad_logits, "token_logprobs_backward: null pointer");
  XKB_REQUIRE(grad_logprobs == nullptr || token_ids != nullptr, "token_logprobs_backward: grad_logprobs without token_ids");
  XKB_REQUIRE(grad_entropy == nullptr || entropy != nullptr, "token_logprobs_backward: grad_entropy without entropy");
  XKB_REQUIRE(grad_top_logprobs == nullptr || top_k == 0 || top_ids != nullptr, "token_logprobs_backward: grad_top_logprobs without top_ids");
  GradArgs a{logits, ld, token_ids, ids64, stats, entropy, grad_logprobs, grad_entropy, grad_top_logprobs, top_ids,
             grad_top_logprobs == nullptr ? 0 : top_k, grad_logits, ld_grad, (int)V, 0, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case XKB_BF16: return backward_typed<__nv_bfloat16>(a, M, s);
    case XKB_F32: return backward_typed<float>(a, M, s);
    default: return backward_typed<__half>(a, M, s);
  }
}
