// Short depthwise causal convolution with SiLU, forward and backward.
//
// A thread owns four neighbouring channels and a tile of frames and slides a
// window of W frames over them in registers: x is read once (but for the W-1
// frames before a tile, which come from the caches) and y written once; bound
// by memory.  Backward, with du = dy silu'(u): dx[t] = sum_i w[i] du[t+W-1-i]
// needs du up to W-1 frames past the tile, which the thread forms again from
// x; the weight and bias gradients are summed per thread over its tile, over
// the workgroup's tiles in LDS, and over workgroups in a fixed order.
#include "seq.h"

namespace dgen {

namespace {

constexpr int kFwdThreads = 256;
// Backward workgroup: 64 channel groups x 4 tiles.
constexpr int kBwdGroups = 64, kBwdTiles = 4;
constexpr int kMaxTaps = 8;

struct ConvShape {
  int64_t B, T, D, G, tiles, tile;  // G: groups of four channels; tile: frames
};

// Frames of a tile: long enough that the frames before it, read again, cost
// little, short enough that the threads fill the chip (eight waves a CU);
// 8 covers every window's past, so only the first tile reads the state.
ConvShape conv_shape(const dgen_hip_conv& c, bool backward) {
  ConvShape s{c.batch, c.T, c.D, (c.D + 3) / 4, 0, backward ? 32 : 16};
  const int64_t want = 256 * 8 * 64;
  while (s.tile > 8 && s.B * s.G * ((s.T + s.tile - 1) / s.tile) < want) s.tile /= 2;
  s.tiles = std::max<int64_t>(1, (s.T + s.tile - 1) / s.tile);
  return s;
}

__device__ __forceinline__ int64_t live_frames(const int32_t* __restrict__ lengths, int64_t b, int64_t T) {
  if (!lengths) return T;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n < T ? n : T;
}

// Frame t (< 0: of the state, else 0) of four channels.
template <class T, int W>
__device__ __forceinline__ void conv_frame(const T* __restrict__ x, int64_t ld, const T* st, int64_t D, int64_t t,
                                           int valid, float (&o)[4]) {
  if (t >= 0) {
    load_four(x + t * ld, valid, o);
  } else if (st) {
    load_four(st + (t + W - 1) * D, valid, o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = 0.f;
  }
}

template <class T, int W, bool SILU>
__global__ __launch_bounds__(kFwdThreads) void k_conv(ConvShape s, const T* __restrict__ x, int64_t xb, int64_t xt,
                                                      const float* __restrict__ w, const float* __restrict__ bias,
                                                      const int32_t* __restrict__ lengths, const T* state,
                                                      T* state_out, T* __restrict__ y, int64_t yb, int64_t yt) {
  const int64_t i = (int64_t)blockIdx.x * kFwdThreads + threadIdx.x;
  if (i >= s.B * s.tiles * s.G) return;
  const int64_t b = i / (s.tiles * s.G), r = i - b * (s.tiles * s.G), tile = r / s.G;
  const int64_t c = (r - tile * s.G) * 4;
  const int valid = (int)(s.D - c < 4 ? s.D - c : 4);
  const int64_t n = live_frames(lengths, b, s.T), t0 = tile * s.tile, t1 = t0 + s.tile < s.T ? t0 + s.tile : s.T;
  const T* xp = x + b * xb + c;
  const T* sp = state ? state + b * (W - 1) * s.D + c : nullptr;
  T* yp = y + b * yb + c;

  float wt[W][4], bs[4], past[W > 1 ? W - 1 : 1][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    bs[e] = bias && e < valid ? bias[c + e] : 0.f;
#pragma unroll
    for (int q = 0; q < W; ++q) wt[q][e] = e < valid ? w[(c + e) * W + q] : 0.f;
  }
#pragma unroll
  for (int q = 0; q < W - 1; ++q) {
    const int64_t t = t0 - (W - 1) + q;
    conv_frame<T, W>(xp, xt, sp, s.D, t, t < n ? valid : 0, past[q]);
  }
  if (state_out && tile == 0) {
    // The frames before the sequence's end.  The first tile is the only
    // reader of the state (no tile is shorter than the window), and has read
    // all that it needs of it before it stores over it.
    float left[W > 1 ? W - 1 : 1][4];
#pragma unroll
    for (int q = 0; q < W - 1; ++q) conv_frame<T, W>(xp, xt, sp, s.D, n - (W - 1) + q, valid, left[q]);
    T* so = state_out + b * (W - 1) * s.D + c;
#pragma unroll
    for (int q = 0; q < W - 1; ++q) store_four(so + q * s.D, valid, left[q]);
  }
  for (int64_t t = t0; t < t1; ++t) {
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    if (t < n) {
      float v[4];
      load_four(xp + t * xt, valid, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float u = bs[e];
#pragma unroll
        for (int q = 0; q < W - 1; ++q) u = fmaf(wt[q][e], past[q][e], u);
        u = fmaf(wt[W - 1][e], v[e], u);
        o[e] = SILU ? silu(u) : u;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int q = 0; q + 1 < W - 1; ++q) past[q][e] = past[q + 1][e];
        if (W > 1) past[W > 1 ? W - 2 : 0][e] = v[e];
      }
    }
    store_four(yp + t * yt, valid, o);
  }
}

// Workgroup: a tile quad (four tiles) of sequence blockIdx.y and 64 channel
// groups, blockIdx.x = quad * ceil(G / 64) + block of groups; its partial row
// is (sequence, quad).
template <class T, int W, bool SILU>
__global__ __launch_bounds__(kBwdGroups* kBwdTiles) void k_conv_bwd(
    ConvShape s, const T* __restrict__ x, int64_t xb, int64_t xt, const T* __restrict__ dy, int64_t gb, int64_t gt,
    const float* __restrict__ w, const float* __restrict__ bias, const int32_t* __restrict__ lengths,
    const T* __restrict__ state, T* __restrict__ dx, int64_t db, int64_t dt, float* __restrict__ parts, int64_t quads) {
  __shared__ float red[kBwdTiles][kBwdGroups][5];
  const uint32_t gx = (uint32_t)((s.G + kBwdGroups - 1) / kBwdGroups);
  const int64_t b = blockIdx.y, quad = blockIdx.x / gx;
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6;
  const int64_t g = (int64_t)(blockIdx.x % gx) * kBwdGroups + lane, c = g * 4;
  const int valid = (int)(c >= s.D ? 0 : s.D - c < 4 ? s.D - c : 4);
  const int64_t n = live_frames(lengths, b, s.T);
  const int64_t t0 = (quad * kBwdTiles + sub) * s.tile, t1 = t0 + s.tile < s.T ? t0 + s.tile : s.T;
  float wt[W][4], bs[4], dw[W][4] = {}, dbs[4] = {};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    bs[e] = bias && e < valid ? bias[c + e] : 0.f;
#pragma unroll
    for (int q = 0; q < W; ++q) wt[q][e] = e < valid ? w[(c + e) * W + q] : 0.f;
  }
  if (valid && t0 < s.T) {
    const T* xp = x + b * xb + c;
    const T* gp = dy + b * gb + c;
    const T* sp = state ? state + b * (W - 1) * s.D + c : nullptr;
    T* op = dx + b * db + c;
    // win[q]: frame t - (W-1) + q; du[q]: du of frame t - q
    float win[W][4], du[W][4];
#pragma unroll
    for (int q = 0; q < W; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) win[q][e] = du[q][e] = 0.f;
#pragma unroll
    for (int q = 0; q < W - 1; ++q) {
      const int64_t t = t0 - (W - 1) + q;
      conv_frame<T, W>(xp, xt, sp, s.D, t, t < n ? valid : 0, win[q + 1]);
    }
    for (int64_t t = t0; t < t1 + W - 1; ++t) {
#pragma unroll
      for (int q = 0; q + 1 < W; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) win[q][e] = win[q + 1][e];
#pragma unroll
      for (int q = W - 1; q > 0; --q)
#pragma unroll
        for (int e = 0; e < 4; ++e) du[q][e] = du[q - 1][e];
      float d[4];
      load_four(xp + t * xt, t < n ? valid : 0, win[W - 1]);
      load_four(gp + t * gt, t < n ? valid : 0, d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (SILU) {
          float u = bs[e];
#pragma unroll
          for (int q = 0; q < W; ++q) u = fmaf(wt[q][e], win[q][e], u);
          d[e] = t < n ? d[e] * silu_grad(u, sigmoid(u)) : 0.f;
        }
        du[0][e] = d[e];
      }
      if (t < t1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dbs[e] += d[e];
#pragma unroll
          for (int q = 0; q < W; ++q) dw[q][e] = fmaf(d[e], win[q][e], dw[q][e]);
        }
      }
      const int64_t to = t - (W - 1);
      if (to >= t0) {
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[e] = 0.f;
#pragma unroll
          for (int q = 0; q < W; ++q) o[e] = fmaf(wt[q][e], du[q][e], o[e]);
          if (to >= n) o[e] = 0.f;
        }
        store_four(op + to * dt, valid, o);
      }
    }
  }
  // [D][W] weight gradients, then [D] bias gradients
  float* out = parts + (b * quads + quad) * s.D * (W + 1);
#pragma unroll
  for (int q = 0; q <= W; ++q) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e) red[sub][lane][e] = q < W ? dw[q < W ? q : 0][e] : dbs[e];
    __syncthreads();
    // thread (sub, lane): channel 4 lane + sub
    if (sub < valid) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < kBwdTiles; ++k) t += red[k][lane][sub];
      if (q < W) out[(c + sub) * W + q] = t;
      else out[s.D * W + c + sub] = t;
    }
  }
}

int64_t conv_quads(const ConvShape& s) { return (s.tiles + kBwdTiles - 1) / kBwdTiles; }

template <class T, int W, bool SILU>
void conv_launch(const dgen_hip_conv& a, bool backward, hipStream_t st) {
  const ConvShape s = conv_shape(a, backward);
  if (!backward) {
    const int64_t threads = s.B * s.tiles * s.G;
    k_conv<T, W, SILU><<<dim3((unsigned)((threads + kFwdThreads - 1) / kFwdThreads)), kFwdThreads, 0, st>>>(
        s, (const T*)a.x.data, a.x.stride_b, a.x.stride_t, a.weight, a.bias, a.lengths, (const T*)a.state,
        (T*)a.state_out, (T*)a.y.data, a.y.stride_b, a.y.stride_t);
  } else {
    const int64_t quads = conv_quads(s);
    float* parts = (float*)a.workspace;
    k_conv_bwd<T, W, SILU>
        <<<dim3((unsigned)((s.G + kBwdGroups - 1) / kBwdGroups * quads), (unsigned)s.B), kBwdGroups * kBwdTiles, 0,
           st>>>(s, (const T*)a.x.data, a.x.stride_b, a.x.stride_t, (const T*)a.dy.data,
                                            a.dy.stride_b, a.dy.stride_t, a.weight, a.bias, a.lengths,
                                            (const T*)a.state, (T*)a.dx.data, a.dx.stride_b, a.dx.stride_t, parts,
                                            quads);
    enqueue_sum_parts(st, parts, s.B * quads, {{a.dweight, a.dbias, nullptr}, {s.D * W, s.D, 0}});
  }
}

template <class T, bool SILU>
void conv_taps(const dgen_hip_conv& a, bool backward, hipStream_t st) {
  switch (a.width) {
    case 1: return conv_launch<T, 1, SILU>(a, backward, st);
    case 2: return conv_launch<T, 2, SILU>(a, backward, st);
    case 3: return conv_launch<T, 3, SILU>(a, backward, st);
    case 4: return conv_launch<T, 4, SILU>(a, backward, st);
    case 5: return conv_launch<T, 5, SILU>(a, backward, st);
    case 6: return conv_launch<T, 6, SILU>(a, backward, st);
    case 7: return conv_launch<T, 7, SILU>(a, backward, st);
    default: return conv_launch<T, 8, SILU>(a, backward, st);
  }
}

}  // namespace

int64_t conv_workspace(const dgen_hip_conv& a, bool backward) {
  if (!backward) return 0;
  const ConvShape s = conv_shape(a, true);
  return align256(s.B * conv_quads(s) * s.D * (a.width + 1) * (int64_t)sizeof(float));
}

int conv_run(const dgen_hip_conv& a, bool backward, hipStream_t st, bool dry) {
  const char* what = backward ? "causal_conv_backward" : "causal_conv";
  DGEN_REQUIRE(a.struct_size == sizeof(a), "%s: struct_size %u, expected %zu", what, a.struct_size, sizeof(a));
  DGEN_REQUIRE(a.type == DGEN_HIP_F32 || a.type == DGEN_HIP_BF16, "%s: type %d", what, a.type);
  DGEN_REQUIRE(a.width >= 1 && a.width <= kMaxTaps, "%s: width %d outside [1, %d]", what, a.width, kMaxTaps);
  DGEN_REQUIRE(a.batch >= 0 && a.batch <= 65535, "%s: batch %lld outside [0, 65535]", what, (long long)a.batch);
  DGEN_REQUIRE(a.T >= 1 && a.T <= (1 << 24), "%s: T %lld outside [1, 2^24]", what, (long long)a.T);
  DGEN_REQUIRE(a.D >= 1 && a.D <= (1 << 20), "%s: D %lld outside [1, 2^20]", what, (long long)a.D);
  const ConvShape s = conv_shape(a, backward);
  // (a launch takes fewer than 2^32 threads)
  DGEN_REQUIRE(s.B * s.tiles * s.G < (int64_t(1) << 31) &&
                   (s.G + kBwdGroups - 1) / kBwdGroups * conv_quads(s) < (int64_t(1) << 23),
               "%s: batch %lld x T %lld x D %lld is too large for one call", what, (long long)a.batch, (long long)a.T,
               (long long)a.D);
  DGEN_REQUIRE(a.weight, "%s: null weight", what);
  const bool empty = a.batch == 0;
  DGEN_REQUIRE((a.x.data || empty) && seq_readable(a.x), "%s: x missing or with a negative stride", what);
  if (!backward) {
    DGEN_REQUIRE((a.y.data || empty) && seq_writable(a.y, a.batch, a.T, a.D), "%s: y missing or overlapping itself",
                 what);
    DGEN_REQUIRE(a.width > 1 || (!a.state && !a.state_out), "%s: a window of one frame has no state", what);
  } else {
    DGEN_REQUIRE((a.dy.data || empty) && seq_readable(a.dy), "%s: dy missing or with a negative stride", what);
    DGEN_REQUIRE((a.dx.data || empty) && seq_writable(a.dx, a.batch, a.T, a.D), "%s: dx missing or overlapping itself",
                 what);
    DGEN_REQUIRE(a.dweight, "%s: null dweight", what);
    DGEN_REQUIRE(!a.bias || a.dbias, "%s: a bias needs dbias", what);
    DGEN_REQUIRE(a.width > 1 || !a.state, "%s: a window of one frame has no state", what);
    const int64_t need = conv_workspace(a, true);
    DGEN_REQUIRE(empty || (a.workspace && a.workspace_bytes >= (uint64_t)need), "%s: workspace of %llu bytes, %lld needed",
                 what, (unsigned long long)a.workspace_bytes, (long long)need);
  }
  if (dry) return 0;
  if (empty) {
    if (!backward) return 0;
    enqueue_sum_parts(st, a.weight, 0, {{a.dweight, a.dbias, nullptr}, {a.D * a.width, a.D, 0}});  // zeros
  } else if (a.type == DGEN_HIP_BF16) {
    a.silu ? conv_taps<bf16, true>(a, backward, st) : conv_taps<bf16, false>(a, backward, st);
  } else {
    a.silu ? conv_taps<float, true>(a, backward, st) : conv_taps<float, false>(a, backward, st);
  }
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
