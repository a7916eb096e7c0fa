// Gated feed-forward block: out = (silu(x Wg^T) * (x Wu^T)) W2^T, and its gradients, as dense products with fused ends.
//
// Forward, two products: gate and up columns of one tile lie side by side in tensor memory, so the read-out has both and
// writes their silu(gate) * up, rounded to 16 bits as the operand of the second product has to be (and gate and up, for
// the backward pass, if they are wanted).  8192 rows of 7168 x 2048: 309 + 157 us one at a time, tensor pipe 90 and 82 % busy (1550
// TFLOP/s), 574 us in a loop, where the power limit holds (1260); one row: 30 us a call among others, 24 with the weights in L2.
// Backward, two launches: dh = dout W2 with the derivative of the activation in the read-out, which leaves [dgate dup] and
// the activations once more, each rounded once (up to 16 rows: in two terms); then dx = [dgate dup] W13, dW13 = [dgate dup]^T x and dW2 = dout^T h as one
// launch whose tiles are dealt out over all SMs together.  4096 rows: 105 + 385 us, 58 and 88 % (the first is 128 tiles on 74
// pairs, two rounds), 580 in a loop.
#include "dense_dev.cuh"

namespace xkb {
namespace dense {

int run_ffn(int end, const Params& p, const Launch& l) {
  if (end == kSwiglu) return run_variant<false, kSwiglu>(p, l);
  return p.prod[0].end.second != 0 ? run_variant<true, kDswigluTwo>(p, l) : run_variant<true, kDswiglu>(p, l);
}

}  // namespace dense

namespace {

int64_t pitch8(int64_t n) { return align_up(n, 8); }

// Up to so many rows the activations go into the second product in two 16-bit terms, which leaves of their rounding 2^-16 (bf16)
// or 2^-22 (fp16): a tile of the MMAs has 128 rows whatever they hold, so the second term's rows cost nothing but their copies
// (one row of 7168 x 2048 28.5 -> 29.1 us).  With few rows the rounding errors of a row's few large activations do not
// average out: that row's result was 2.5e-3 off in the norm with one term, and is 1.6e-3 off with two, which its own
// rounding is.  16: the rows of both terms then belong to one read-out warp.
constexpr int64_t kTwoTerms = 16;
// I: as much as single CTAs, which alone take two terms, may add up in one accumulator (a part of it as a rule): 4e-4 lost at most
// where all terms are of one sign.
bool two_terms(int64_t M, int64_t I) { return M <= kTwoTerms && I <= 65536; }
// The gradients' operands too (1 x 7168 x 2048 bf16 2.4e-3 off with one term, 1.7e-3 with two, 58 and 62 us); grad_x contracts over 2 I,
// in one accumulator.
bool two_terms_back(int64_t M, int64_t I) { return two_terms(M, 2 * I); }

int check_sizes(const char* name, int dtype, int64_t M, int64_t H, int64_t I) {
  XKB_REQUIRE(dtype == XKB_BF16 || dtype == XKB_F16, "%s: dtype must be bf16 or fp16", name);
  XKB_REQUIRE(M >= 0 && H >= 1 && I >= 1 && M < (1ll << 28) && H < (1ll << 24) && I < (1ll << 24), "%s: M=%lld H=%lld I=%lld out of range",
              name, (long long)M, (long long)H, (long long)I);
  return XKB_OK;
}

// A matrix that the products read: rows of a multiple of 16 bytes, the first one on 16 bytes.
int check_operand(const char* name, const char* what, const void* p, int64_t ld, int64_t cols) {
  XKB_REQUIRE(p != nullptr, "%s: %s is null", name, what);
  XKB_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && ld >= cols && ld < (1ll << 32),
              "%s: rows of %s must start on 16 bytes and not overlap (row stride %lld)", name, what, (long long)ld);
  return XKB_OK;
}

}  // namespace
}  // namespace xkb

using namespace xkb;

extern "C" int64_t xkb_gated_ffn_workspace_bytes(int64_t M, int64_t H, int64_t I) {
  if (check_sizes("gated_ffn", XKB_BF16, M, H, I) != XKB_OK) return -1;
  return (two_terms(M, I) ? 2 : 1) * align_up(M * pitch8(I) * 2, 256);
}

extern "C" int xkb_gated_ffn(const void* x, int64_t ld_x, int dtype, const void* w13, int64_t ld_w13, const void* w2, int64_t ld_w2,
                             float limit, void* out, void* gate_up, int64_t M, int64_t H, int64_t I, void* workspace,
                             int64_t workspace_bytes, void* stream_) {
  const char* name = "gated_ffn";
  XKB_TRY(check_sizes(name, dtype, M, H, I));
  if (M == 0) return XKB_OK;
  XKB_TRY(check_operand(name, "x", x, ld_x, H));
  XKB_TRY(check_operand(name, "w13", w13, ld_w13, H));
  XKB_TRY(check_operand(name, "w2", w2, ld_w2, I));
  XKB_REQUIRE(out != nullptr && address_bits(out, gate_up) % 2 == 0, "%s: null or misaligned output", name);
  const int64_t need = xkb_gated_ffn_workspace_bytes(M, H, I);
  if (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return fail(XKB_ERR_WORKSPACE, "%s: needs a workspace of %lld bytes on 256 bytes", name, (long long)need);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  using namespace dense;
  Product up = {};
  up.a = {x, ld_x, false, 0, M, H};
  up.b = {w13, ld_w13, false, 0, 2 * I, H};
  up.M = M, up.N = I, up.K = H;
  const int64_t rest = two_terms(M, I) ? align_up(M * pitch8(I) * 2, 256) / 2 : 0;
  up.end.h = workspace, up.end.ld_h = pitch8(I);
  if (rest != 0) up.end.h_rest = static_cast<uint16_t*>(workspace) + rest;
  up.end.gate_up = gate_up, up.end.ld_gu = 2 * I, up.end.half = (int)I;
  up.end.limit = limit;
  XKB_TRY(launch(&up, 1, kSwiglu, dtype, false, false, stream));
  Product down = {};
  down.a = {workspace, pitch8(I), false, 0, M, I, rest};
  down.b = {w2, ld_w2, false, 0, H, I};
  down.M = M, down.N = H, down.K = I;
  down.end.out = out, down.end.ld = H;
  return launch(&down, 1, kStore, dtype, true, true, stream);
}

extern "C" int64_t xkb_gated_ffn_backward_workspace_bytes(int64_t M, int64_t H, int64_t I, int recompute) {
  if (check_sizes("gated_ffn_backward", XKB_BF16, M, H, I) != XKB_OK) return -1;
  const bool few = two_terms_back(M, I);
  const int64_t rows = few ? 2 * M : M;
  return align_up(rows * pitch8(I) * 2, 256) + align_up(rows * pitch8(2 * I) * 2, 256) + (few ? 2 * align_up(rows * pitch8(H) * 2, 256) : 0) +
         (recompute ? align_up(M * pitch8(2 * I) * 2, 256) : 0);
}

extern "C" int xkb_gated_ffn_backward(const void* grad_out, int64_t ld_go, int dtype, const void* x, int64_t ld_x, const void* w13,
                                      int64_t ld_w13, const void* w2, int64_t ld_w2, const void* gate_up, float limit, void* grad_x,
                                      void* grad_w13, void* grad_w2, int64_t M, int64_t H, int64_t I, void* workspace,
                                      int64_t workspace_bytes, void* stream_) {
  const char* name = "gated_ffn_backward";
  XKB_TRY(check_sizes(name, dtype, M, H, I));
  XKB_REQUIRE(address_bits(grad_x, grad_w13, grad_w2, gate_up) % 2 == 0, "%s: misaligned tensor", name);
  if (grad_x == nullptr && grad_w13 == nullptr && grad_w2 == nullptr) return XKB_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (M == 0) {
    if (grad_w13 != nullptr) XKB_CHECK_CUDA(cudaMemsetAsync(grad_w13, 0, (size_t)(2 * I * H) * 2, stream));
    if (grad_w2 != nullptr) XKB_CHECK_CUDA(cudaMemsetAsync(grad_w2, 0, (size_t)(H * I) * 2, stream));
    return XKB_OK;
  }
  XKB_TRY(check_operand(name, "grad_out", grad_out, ld_go, H));
  XKB_TRY(check_operand(name, "x", x, ld_x, H));
  XKB_TRY(check_operand(name, "w13", w13, ld_w13, H));
  XKB_TRY(check_operand(name, "w2", w2, ld_w2, I));
  const int64_t need = xkb_gated_ffn_backward_workspace_bytes(M, H, I, gate_up == nullptr);
  if (workspace == nullptr || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return fail(XKB_ERR_WORKSPACE, "%s: needs a workspace of %lld bytes on 256 bytes", name, (long long)need);
  using namespace dense;
  Carver ws(workspace);
  // Up to 16 rows the operands that the activation's gradient leaves have two terms, M rows apart: grad_x adds its rows of both, and
  // the weights' gradients take the second term's rows as further K, beside x and grad_out once more (but for what is infinite there or
  // a NaN, which the first terms' rows have: a term of the other sign, or of 0, would make a NaN of an infinity).
  const bool few = two_terms_back(M, I);
  const int64_t rows = few ? 2 * M : M;
  void* h = ws.take<uint16_t>(rows * pitch8(I));
  void* d13 = ws.take<uint16_t>(rows * pitch8(2 * I));
  int64_t ld_gu = 2 * I;
  bool chained = false, early = false;      // early: w2 is no output of the predecessor
  if (few) {
    const void* from[4];
    void* to[4];
    int64_t ld[4], each[4], cols[4];
    int exponent[4], copies = 0;
    auto twice = [&](const void*& p, int64_t& pitch) {
      uint16_t* at = ws.take<uint16_t>(rows * pitch8(H));
      for (int i = 0; i < 2; ++i, ++copies) {
        from[copies] = p, ld[copies] = pitch, each[copies] = M, cols[copies] = H, to[copies] = at + i * M * pitch8(H);
        exponent[copies] = i == 0 ? 0 : dtype == XKB_BF16 ? 0x7F80 : 0x7C00;
      }
      p = at, pitch = pitch8(H);
    };
    if (grad_w13 != nullptr) twice(x, ld_x);
    if (grad_w2 != nullptr) twice(grad_out, ld_go);
    if (copies > 0) {
      XKB_TRY(lay_out(from, ld, each, cols, to, exponent, copies, stream));
      chained = true;
    }
  }
  if (gate_up == nullptr) {
    ld_gu = pitch8(2 * I);
    void* again = ws.take<uint16_t>(M * ld_gu);
    Product up = {};
    up.a = {x, ld_x, false, 0, M, H};
    up.b = {w13, ld_w13, false, 0, 2 * I, H};
    up.M = M, up.N = I, up.K = H;
    up.end.gate_up = again, up.end.ld_gu = ld_gu, up.end.half = (int)I;
    XKB_TRY(launch(&up, 1, kSwiglu, dtype, chained, false, stream));
    gate_up = again;
    chained = early = true;
  }
  Product open = {};
  open.a = {grad_out, ld_go, false, 0, M, H};
  open.b = {w2, ld_w2, true, 0, H, I};
  open.M = M, open.N = I, open.K = H;
  open.end.out = d13, open.end.ld = pitch8(2 * I);
  open.end.h = grad_w2 != nullptr ? h : nullptr, open.end.ld_h = pitch8(I);
  open.end.gate_up = const_cast<void*>(gate_up), open.end.ld_gu = ld_gu, open.end.half = (int)I;
  open.end.limit = limit;
  open.end.second = few ? (int)M : 0;
  XKB_TRY(launch(&open, 1, kDswiglu, dtype, chained, early, stream));
  Product q[3] = {};
  int n = 0;
  if (grad_x != nullptr) {
    q[n].a = {d13, pitch8(2 * I), false, 0, rows, 2 * I};
    q[n].b = {w13, ld_w13, true, 0, 2 * I, H};
    q[n].M = M, q[n].N = H, q[n].K = 2 * I;
    q[n].end.out = grad_x, q[n].end.ld = H;
    q[n].end.second = open.end.second;
    ++n;
  }
  if (grad_w13 != nullptr) {
    q[n].a = {d13, pitch8(2 * I), true, 0, rows, 2 * I};
    q[n].b = {x, ld_x, true, 0, rows, H};
    q[n].M = 2 * I, q[n].N = H, q[n].K = rows;
    q[n].end.out = grad_w13, q[n].end.ld = H;
    ++n;
  }
  if (grad_w2 != nullptr) {
    q[n].a = {grad_out, ld_go, true, 0, rows, H};
    q[n].b = {h, pitch8(I), true, 0, rows, I};
    q[n].M = H, q[n].N = I, q[n].K = rows;
    q[n].end.out = grad_w2, q[n].end.ld = I;
    ++n;
  }
  return launch(q, n, kStore, dtype, true, false, stream);
}
