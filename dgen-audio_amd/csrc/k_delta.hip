// Gated delta rule: the entry's checks and how a call is cut (k_delta.h has the
// kernels).
#include "k_delta.h"

#include <cmath>

namespace dgen {

namespace {

constexpr int64_t kMaxK = 128, kMaxV = 1024;

// [batch][T][heads][channels] that is written: no two elements at one address,
// for axes that lie within one another in any order.
bool heads_writable(int64_t sb, int64_t st, int64_t sh, int64_t B, int64_t T, int64_t H, int64_t channels) {
  int64_t stride[3] = {sb, st, sh}, n[3] = {B, T, H};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (stride[j] < stride[i]) std::swap(stride[i], stride[j]), std::swap(n[i], n[j]);
  int64_t extent = channels;
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 1) continue;
    if (stride[i] < extent) return false;
    extent += (n[i] - 1) * stride[i];
  }
  return true;
}

}  // namespace

DeltaPlan delta_plan(const dgen_hip_delta& a, bool backward) {
  DeltaPlan o = {};
  if (delta_steps(a, backward) || a.batch == 0) return o;
  const int64_t bh = a.batch * a.heads, K = a.K <= 32 ? 32 : a.K <= 64 ? 64 : 128;
  o.chunks = (a.T + kC - 1) / kC;
  o.segs = 1;
  o.nvb = (a.V + kVB - 1) / kVB;
  // Segments go through their chunks twice, the second time with their transitions
  // too, and each is a step of the carry: three times the work, so that they pay
  // where the card is a third full at most (with 128 channels, whose steps of the
  // carry are dearer, less).  The square root of the chunks balances both walks.
  // One piece and segments, us, forward, fp32 64 x 64: 1 head of 512 frames 48 and
  // 34, of 65536 3990 and 188, 24 heads of 1024 89 and 67, of 512 52 and 51; bf16
  // 128 x 128: 8 heads of 2048 138 and 85, of 512 46 and 50, 24 of 1024 87 and 98.
  // The limits do not go by the length: with more heads than these, segments would
  // pay for far longer clips (11 heads of 65536 frames, 128 x 128: 4221 and 1435).
  const bool wide = K > 64;
  if (bh * o.nvb <= (wide ? 40 : 96) && o.chunks >= (wide ? 12 : 8))
    o.segs = std::min<int64_t>((int64_t)((wide ? 1.5 : 3.) * std::sqrt((double)o.chunks)), 512 / (bh * o.nvb));
  o.per = (o.chunks + o.segs - 1) / o.segs;
  o.segs = (o.chunks + o.per - 1) / o.per;
  int64_t at = 0;
  auto take = [&](int64_t floats) {
    const int64_t p = at;
    at += align256(floats * 4);
    return p;
  };
  const int64_t n = bh * o.chunks, V = o.nvb * kVB;
  o.X = take(n * kC * kC);
  o.M = take(n * kC * kC);
  if (backward) o.XT = take(n * kC * kC), o.A = take(n * kC * kC);
  o.vec = take(n * kVecs * kC);
  if (backward) {
    o.S = take(n * K * V);
    o.dS = take(n * K * V);
    o.U = take(n * kC * V);
    o.dR = take(n * kC * V);
  }
  if (o.segs > 1) {
    o.ends = take(bh * o.segs * K * (V + K));
    if (backward) o.gends = take(bh * o.segs * K * V);
  }
  o.bytes = at;
  return o;
}

int64_t delta_workspace(const dgen_hip_delta& a, bool backward) { return delta_plan(a, backward).bytes; }

int delta_run(const dgen_hip_delta& a, bool backward, hipStream_t st, bool dry) {
  const char* what = backward ? "gated_delta_rule_backward" : "gated_delta_rule";
  DGEN_REQUIRE(a.struct_size == sizeof(a), "%s: struct_size %u, expected %zu", what, a.struct_size, sizeof(a));
  DGEN_REQUIRE(a.type == DGEN_HIP_F32 || a.type == DGEN_HIP_BF16, "%s: type %d", what, a.type);
  DGEN_REQUIRE(a.batch >= 0 && a.batch <= 1 << 24, "%s: batch %lld outside [0, 2^24]", what, (long long)a.batch);
  DGEN_REQUIRE(a.T >= 1 && a.T <= 1 << 24, "%s: T %lld outside [1, 2^24]", what, (long long)a.T);
  DGEN_REQUIRE(a.heads >= 1 && a.heads <= 1 << 16 && a.key_heads >= 1 && a.heads % a.key_heads == 0,
               "%s: %lld heads, %lld key heads", what, (long long)a.heads, (long long)a.key_heads);
  DGEN_REQUIRE(a.K >= 1 && a.K <= kMaxK, "%s: K %lld outside [1, %lld]", what, (long long)a.K, (long long)kMaxK);
  DGEN_REQUIRE(a.V >= 1 && a.V <= kMaxV, "%s: V %lld outside [1, %lld]", what, (long long)a.V, (long long)kMaxV);
  DGEN_REQUIRE(a.scale > -INFINITY && a.scale < INFINITY && a.scale != 0.f, "%s: scale %g", what, (double)a.scale);
  const int64_t bh = a.batch * a.heads;
  const DeltaPlan o = delta_plan(a, backward);
  // (a launch takes fewer than 2^32 threads)
  DGEN_REQUIRE(bh * std::max<int64_t>(o.chunks, o.segs * (o.nvb + 4)) < int64_t(1) << 23 && bh < int64_t(1) << 18,
               "%s: %lld sequences and heads of %lld frames are too many for one call", what, (long long)bh, (long long)a.T);
  const bool empty = a.batch == 0;
  // (a chunk's rows are addressed in 32 bits)
  auto near = [&](int64_t stride_t) { return stride_t >= 0 && (a.T == 1 || stride_t <= int64_t(1) << 23); };
  auto readable = [&](const dgen_hip_heads& h) { return (h.data || empty) && h.stride_b >= 0 && near(h.stride_t) && h.stride_h >= 0; };
  auto writable = [&](const dgen_hip_heads& h, int64_t heads, int64_t n) {
    return (h.data || empty) && h.stride_b >= 0 && near(h.stride_t) && h.stride_h >= 0 &&
           heads_writable(h.stride_b, h.stride_t, h.stride_h, a.batch, a.T, heads, n);
  };
  DGEN_REQUIRE(readable(a.q) && readable(a.k) && readable(a.v), "%s: q, k or v: null, or a negative stride, or more than 2^23 between frames", what);
  DGEN_REQUIRE(((a.g.data && a.beta.data) || empty) && seq_readable(a.g) && seq_readable(a.beta), "%s: g or beta: null, or a negative stride", what);
  if (!backward) {
    DGEN_REQUIRE(writable(a.y, a.heads, a.V), "%s: y: null, overlapping, or frames too far apart", what);
  } else {
    DGEN_REQUIRE(readable(a.dy), "%s: dy: null, or a negative stride, or more than 2^23 between frames", what);
    DGEN_REQUIRE(writable(a.dq, a.key_heads, a.K) && writable(a.dk, a.key_heads, a.K) && writable(a.dv, a.heads, a.V),
                 "%s: dq, dk or dv: null, overlapping, or frames too far apart", what);
    DGEN_REQUIRE(((a.dg.data && a.dbeta.data) || empty) && seq_writable(a.dg, a.batch, a.T, a.heads) &&
                     seq_writable(a.dbeta, a.batch, a.T, a.heads),
                 "%s: dg or dbeta: null, or overlapping", what);
  }
  DGEN_REQUIRE(o.bytes == 0 || (a.workspace && a.workspace_bytes >= (uint64_t)o.bytes),
               "%s: workspace of %llu bytes, %lld needed", what, (unsigned long long)a.workspace_bytes, (long long)o.bytes);
  if (dry || empty) return 0;
  a.type == DGEN_HIP_BF16 ? delta_enqueue_bf16(a, backward, st) : delta_enqueue_f32(a, backward, st);
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
