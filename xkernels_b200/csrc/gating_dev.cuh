// Rows of gating logits in registers, shared by the balance loss and the gradient of the gating logits.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "softmax_dev.cuh"

namespace xkb {

constexpr int kMaxExperts = 1024;

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T of_float(float v);
template <> __device__ __forceinline__ float of_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 of_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half of_float<__half>(float v) { return __float2half_rn(v); }

// The larger of two pairs of 16-bit values, NaN where one of them is.
template <typename T> __device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Two values in a word, and a word's two values.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16(lo, hi);
  }
}
template <typename T> __device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  } else {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  }
}

// Over each group of LANES neighbouring lanes.
template <int LANES> __device__ __forceinline__ float lanes_add(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Four sums at once: the first two steps halve the values that a lane adds up instead of adding all four, and the sums are read from
// where they end (22 instructions instead of 40 over a warp).
template <int LANES> __device__ __forceinline__ void lanes_add4(float& a, float& b, float& c, float& d) {
  constexpr int H = LANES / 2, Q = LANES / 4;
  const bool upper = threadIdx.x & H, odd = threadIdx.x & Q;
  float x = upper ? c : a, y = upper ? d : b;
  x += __shfl_xor_sync(0xffffffffu, upper ? a : c, H);
  y += __shfl_xor_sync(0xffffffffu, upper ? b : d, H);
  const float other = __shfl_xor_sync(0xffffffffu, odd ? x : y, Q);
  x = (odd ? y : x) + other;
#pragma unroll
  for (int o = Q / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  a = __shfl_sync(0xffffffffu, x, 0, LANES);
  b = __shfl_sync(0xffffffffu, x, Q, LANES);
  c = __shfl_sync(0xffffffffu, x, H, LANES);
  d = __shfl_sync(0xffffffffu, x, H + Q, LANES);
}
template <int LANES> __device__ __forceinline__ float lanes_max_nan(float v) {
  if constexpr (LANES == 32) {
    return warp_max_nan(v);
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}

// 1 / s to 1 ulp; 0 for 0 (a row or a choice without a live logit).  The sums here are 0 or 2^-127 to 2^11, or NaN.
__device__ __forceinline__ float inverse(float s) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(s));
  return s == 0.f ? 0.f : r;
}

// e^(x - max), but for a factor that all terms of a row share: 2^(x log2(e) - c) with c = max log2(e) rounded, one multiply-add.  Where
// the rounding could come near 1 the difference is taken first.
constexpr float kNear = 1e6f;
__device__ __forceinline__ float exponential(float x, float max) {
  return exp2_fast(fabsf(max) <= kNear ? fmaf(x, kLog2e, -(max * kLog2e)) : (x - max) * kLog2e);
}

// A row over LANES lanes, in pieces of P neighbouring experts: a lane's t-th value belongs to expert (t / P * LANES + lane) * P + t % P.
// A warp has 32 / LANES rows.
template <typename T, int LANES, int PER_LANE, int P>
struct Row {
  struct alignas(P * sizeof(T)) Piece { T x[P]; };
  static constexpr int kPieces = PER_LANE / P;
  struct Raw { Piece q[kPieces]; };
  static __device__ __forceinline__ int expert(int t, int lane) { return (t / P * LANES + lane) * P + t % P; }
  // logits; -inf behind the row, and everywhere if there is none
  static __device__ __forceinline__ Raw load(const T* row, int E, int lane, bool there) {
    Raw r;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      if constexpr (sizeof(T) == 2 && P >= 2) {
#pragma unroll
        for (int i = 0; i < P / 2; ++i) reinterpret_cast<uint32_t*>(&r.q[c])[i] = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
      } else {
#pragma unroll
        for (int i = 0; i < P; ++i) r.q[c].x[i] = of_float<T>(-INFINITY);
      }
      if (there && (c * LANES + lane) * P < E) r.q[c] = reinterpret_cast<const Piece*>(row)[c * LANES + lane];
    }
    return r;
  }
  static __device__ __forceinline__ void store(T* row, int E, int lane, const float (&x)[PER_LANE]) {
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      Piece q;
      if constexpr (sizeof(T) == 2 && P >= 2) {
#pragma unroll
        for (int i = 0; i < P; i += 2) reinterpret_cast<uint32_t*>(&q)[i / 2] = pack2<T>(x[c * P + i], x[c * P + i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < P; ++i) q.x[i] = of_float<T>(x[c * P + i]);
      }
      if ((c * LANES + lane) * P < E) reinterpret_cast<Piece*>(row)[c * LANES + lane] = q;
    }
  }
  // the lane's maximum, NaN if one of its logits is
  static __device__ __forceinline__ float lane_max(const Raw& r, const float (&x)[PER_LANE]) {
    if constexpr (sizeof(T) == 2 && P >= 2) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
      uint32_t m = w[0];
#pragma unroll
      for (int i = 1; i < PER_LANE / 2; ++i) m = larger2<T>(m, w[i]);
      const T* two = reinterpret_cast<const T*>(&m);
      return max_nan(to_float(two[0]), to_float(two[1]));
    } else {
      float m = x[0];
#pragma unroll
      for (int t = 1; t < PER_LANE; ++t) m = max_nan(m, x[t]);
      return m;
    }
  }
  // logits -> exponential(x, max), the row's maximum (0 for a row without a live logit, whose values become 0) and this lane's sum.
  // NaN and +inf make the row NaN.
  static __device__ __forceinline__ float exponentials(const Raw& r, float (&x)[PER_LANE], float& max) {
    if constexpr (sizeof(T) == 2 && P >= 2) {
#pragma unroll
      for (int t = 0; t < PER_LANE; t += 2) unpack2<T>(reinterpret_cast<const uint32_t*>(&r)[t / 2], x[t], x[t + 1]);
    } else {
#pragma unroll
      for (int t = 0; t < PER_LANE; ++t) x[t] = to_float(r.q[t / P].x[t % P]);
    }
    const float mx = lanes_max_nan<LANES>(lane_max(r, x));
    max = mx == -INFINITY ? 0.f : mx;
    if constexpr (PER_LANE == 1) {
      x[0] = exponential(x[0], max);
      return x[0];
    } else {
      if (fabsf(max) <= kNear) {   // (NaN: below)
        const Pair scale = pair_of(kLog2e), minus_c = pair_of(-(max * kLog2e));
#pragma unroll
        for (int t = 0; t < PER_LANE; t += 2) split(fma2(pair_of(x[t], x[t + 1]), scale, minus_c), x[t], x[t + 1]);
      } else {
#pragma unroll
        for (int t = 0; t < PER_LANE; ++t) x[t] = (x[t] - max) * kLog2e;
      }
      Pair sum = pair_of(0.f);
#pragma unroll
      for (int t = 0; t < PER_LANE; t += 2) {
        x[t] = exp2_fast(x[t]);
        x[t + 1] = exp2_fast(x[t + 1]);
        sum = add2(sum, pair_of(x[t], x[t + 1]));
      }
      float s0, s1;
      split(sum, s0, s1);
      return s0 + s1;
    }
  }
};

// Calls f<LANES, PER_LANE, P>() with the widest piece that the row and its address allow.  The sums over lanes, the slots and the loop
// cost a warp the same for one row as for four: rows take as few lanes as hold them with at most 16 values each (32 above 256
// experts) and have a lane for each slot.  us, gradient of both, bf16 top 8, 32 lanes / here: 16384 x 128 6.3 / 4.4, 16384 x 256 7.2 / 6.0,
// 65536 x 256 25 / 18, 65536 x 512 36 / 32.  But 32 lanes above 256 experts where pieces are of one (5003 x 327 6.0 over 16 lanes, 5.1
// over 32; balance loss of 1021 x 271 8.8 / 7.3).  (65536 x 256 over 8 lanes: 16.2, but 16384 x 255 9.8 instead of 7.5.)
template <typename T, int LANES, int PER_LANE, int LEAST = 1, typename F>
int with_piece(int E, uintptr_t bits, F f) {   // bits: the addresses of all rows, or'ed; pieces of LEAST always fit
  constexpr int kMost = PER_LANE < (int)(16 / sizeof(T)) ? PER_LANE : (int)(16 / sizeof(T));
  auto fits = [&](int P) { return E % P == 0 && bits % (P * sizeof(T)) == 0; };
  if constexpr (kMost > 2) if (fits(kMost)) return f.template operator()<LANES, PER_LANE, kMost>();
  if constexpr (kMost >= 2 && LEAST == 1) if (fits(2)) return f.template operator()<LANES, PER_LANE, 2>();
  return f.template operator()<LANES, PER_LANE, LEAST>();
}
template <typename T, typename F>
int with_shape(int E, int top_k, uintptr_t bits, F f) {
  if (top_k <= 8) {
    if (E <= 8) return with_piece<T, 8, 1>(E, bits, f);
    if (E <= 16) return with_piece<T, 8, 2>(E, bits, f);
    if (E <= 32) return with_piece<T, 8, 4>(E, bits, f);
    if (E <= 64) return with_piece<T, 8, 8>(E, bits, f);
    if (E <= 128) return with_piece<T, 8, 16>(E, bits, f);
  }
  if (top_k <= 16) {
    if (E <= 128) return with_piece<T, 16, 8>(E, bits, f);
    if (E <= 256) return with_piece<T, 16, 16>(E, bits, f);
    if (E <= 512 && E % 2 == 0 && bits % (2 * sizeof(T)) == 0) return with_piece<T, 16, 32, 2>(E, bits, f);
  }
  if (E <= 128) return with_piece<T, 32, 4>(E, bits, f);
  if (E <= 256) return with_piece<T, 32, 8>(E, bits, f);
  if (E <= 512) return with_piece<T, 32, 16>(E, bits, f);
  return with_piece<T, 32, 32>(E, bits, f);
}

}  // namespace xkb
