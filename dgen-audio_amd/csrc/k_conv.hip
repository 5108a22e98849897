// Short depthwise causal convolution with SiLU, forward and backward.
//
// A thread owns four neighbouring channels and a tile of frames and slides a
// window of W frames over them in registers: x is read once (but for the W-1
// frames before a tile, which come from the caches) and y written once; bound
// by memory.  Backward, with du = dy silu'(u): dx[t] = sum_i w[i] du[t+W-1-i]
// needs du up to W-1 frames past the tile, which the thread forms again from
// x; the weight and bias gradients are summed per thread over its tile, over
// the workgroup's tiles in LDS, and over workgroups in a fixed order.
//
// Measured at 32 x 1000 x 1024, W = 4, on operands that the caches do not hold
// (a large copy: 4.97 TB/s): forward bf16 44 us, 3.0 TB/s, fp32 57 us, 4.6 TB/s;
// backward bf16 53 us, 3.7 TB/s, fp32 91 us, 4.3 TB/s, and 5 us for the partial
// rows of either.  (Calls in a row on two sets of operands, which lie in the
// last cache in part: bf16 30 and 50 us.)  The loads' latency is what is left,
// in bf16 above all: a wave's four channels a lane are 512 bytes a frame and
// tensor, with four frames in flight (eight: 12 and 17 % more time, by their
// registers), and about half of the issue slots go to the sigmoid and the
// window.
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
// 8 covers every window's past, so only the first tile reads the state.  At 32
// x 1000 x 1024 bf16, calls on two sets of operands, tiles of 16, 32 and 64
// frames: forward 36, 33 and 41 us (64 leaves one round of workgroups, half of
// it idle at the end), backward 73, 59 and 55.
ConvShape conv_shape(const dgen_hip_conv& c, bool backward) {
  ConvShape s{c.batch, c.T, c.D, (c.D + 3) / 4, 0, backward ? 64 : 32};
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

// Four channels of a thread: its group's, or the last four where the group
// reaches past the last channel (so that every load is a whole one); of those
// it owns, and stores, the ones from `skip` on.  Tensors of fewer than four
// channels (FEW) are loaded element by element.
struct Channels {
  int64_t c;
  int skip, end;  // owned: [skip, end)
};
template <bool FEW>
__device__ __forceinline__ Channels channels_of(int64_t g, int64_t D) {
  if (FEW) return {0, 0, (int)D};
  const int64_t c = g * 4 < D - 4 ? g * 4 : D - 4;
  const int64_t skip = g * 4 - c;
  return {c, (int)(skip < 4 ? skip : 4), 4};
}
template <bool FEW, class T>
__device__ __forceinline__ Four<T> get_four(const T* __restrict__ p, const Channels& ch) {
  if (!FEW) return *reinterpret_cast<const Four<T>*>(p);
  Four<T> f{};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < ch.end) f.e[e] = p[e];
  return f;
}
template <class T>
__device__ __forceinline__ void put_four(T* __restrict__ p, const Channels& ch, const float (&o)[4]) {
  if (ch.skip == 0 && ch.end == 4) {
    store_four(p, 4, o);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e >= ch.skip && e < ch.end) p[e] = from_f32<T>(o[e]);
  }
}

// Frame t < 0: of the state, else 0.
template <class T, int W, bool FEW>
__device__ __forceinline__ void frame_before(const T* st, int64_t D, int64_t t, const Channels& ch, float (&o)[4]) {
  Four<T> f{};
  if (st) f = get_four<FEW>(st + (t + W - 1) * D, ch);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = to_f32(f.e[e]);
}

template <int W>
struct Taps {
  float w[W][4], bias[4];
  __device__ __forceinline__ void load(const float* __restrict__ wt, const float* __restrict__ bs, const Channels& ch) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t c = ch.c + (e < ch.end ? e : 0);
      bias[e] = bs ? bs[c] : 0.f;
#pragma unroll
      for (int q = 0; q < W; ++q) w[q][e] = wt[c * W + q];
    }
  }
};

constexpr int kGroup = 4;  // frames a thread loads ahead of their use

template <class T, int W, bool SILU, bool FEW>
__global__ __launch_bounds__(kFwdThreads) void k_conv(ConvShape s, const T* __restrict__ x, int64_t xb, int64_t xt,
                                                      const float* __restrict__ w, const float* __restrict__ bias,
                                                      const int32_t* __restrict__ lengths, const T* state,
                                                      T* state_out, T* __restrict__ y, int64_t yb, int64_t yt) {
  const int64_t i = (int64_t)blockIdx.x * kFwdThreads + threadIdx.x;
  if (i >= s.B * s.tiles * s.G) return;
  const int64_t b = i / (s.tiles * s.G), r = i - b * (s.tiles * s.G), tile = r / s.G;
  const Channels ch = channels_of<FEW>(r - tile * s.G, s.D);
  const int64_t n = live_frames(lengths, b, s.T), t0 = tile * s.tile, t1 = t0 + s.tile < s.T ? t0 + s.tile : s.T;
  const int64_t last = n > 0 ? n - 1 : 0;
  const T* xp = x + b * xb + ch.c;
  const T* sp = state ? state + b * (W - 1) * s.D + ch.c : nullptr;
  T* yp = y + b * yb + ch.c;

  Four<T> next[kGroup];
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int k = 0; k < kGroup; ++k) next[k] = get_four<FEW>(xp + (t + k < last ? t + k : last) * xt, ch);
  };
  fetch(t0);
  Taps<W> taps;
  taps.load(w, bias, ch);
  // win[q]: frame t - (W-1) + q of the group's first frame t
  float win[W - 1 + kGroup][4];
#pragma unroll
  for (int q = 0; q < W - 1; ++q) {
    const int64_t t = t0 - (W - 1) + q;
    if (t < 0) {
      frame_before<T, W, FEW>(sp, s.D, t, ch, win[q]);
    } else {
      const Four<T> f = get_four<FEW>(xp + (t < last ? t : last) * xt, ch);
#pragma unroll
      for (int e = 0; e < 4; ++e) win[q][e] = to_f32(f.e[e]);
    }
  }
  if (state_out && tile == 0) {
    // The frames before the sequence's end.  The first tile is the only
    // reader of the state (no tile is shorter than the window), and has read
    // all that it needs of its channels before it stores over them.
    float left[W > 1 ? W - 1 : 1][4];
#pragma unroll
    for (int q = 0; q < W - 1; ++q) {
      const int64_t t = n - (W - 1) + q;
      if (t < 0) {
        frame_before<T, W, FEW>(sp, s.D, t, ch, left[q]);
      } else {
        const Four<T> f = get_four<FEW>(xp + t * xt, ch);
#pragma unroll
        for (int e = 0; e < 4; ++e) left[q][e] = to_f32(f.e[e]);
      }
    }
    T* so = state_out + b * (W - 1) * s.D + ch.c;
#pragma unroll
    for (int q = 0; q < W - 1; ++q) put_four(so + q * s.D, ch, left[q]);
  }
  for (int64_t t = t0; t < t1; t += kGroup) {
#pragma unroll
    for (int k = 0; k < kGroup; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) win[W - 1 + k][e] = to_f32(next[k].e[e]);
    if (t + kGroup < t1) fetch(t + kGroup);
#pragma unroll
    for (int k = 0; k < kGroup; ++k) {
      if (t + k >= t1) break;
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float u = taps.bias[e];
#pragma unroll
        for (int q = 0; q < W; ++q) u = fmaf(taps.w[q][e], win[k + q][e], u);
        o[e] = t + k < n ? (SILU ? silu(u) : u) : 0.f;
      }
      put_four(yp + (t + k) * yt, ch, o);
    }
#pragma unroll
    for (int q = 0; q < W - 1; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) win[q][e] = win[q + kGroup][e];
  }
}

// Workgroup: a tile quad (four tiles) of sequence blockIdx.y and 64 channel
// groups, blockIdx.x = quad * ceil(G / 64) + block of groups; its partial row
// is (sequence, quad).
template <class T, int W, bool SILU, bool FEW>
__global__ __launch_bounds__(kBwdGroups* kBwdTiles) void k_conv_bwd(
    ConvShape s, const T* __restrict__ x, int64_t xb, int64_t xt, const T* __restrict__ dy, int64_t gb, int64_t gt,
    const float* __restrict__ w, const float* __restrict__ bias, const int32_t* __restrict__ lengths,
    const T* __restrict__ state, T* __restrict__ dx, int64_t db, int64_t dt, float* __restrict__ parts, int64_t quads) {
  __shared__ float red[kBwdTiles][kBwdGroups][5];
  const uint32_t gx = (uint32_t)((s.G + kBwdGroups - 1) / kBwdGroups);
  const int64_t b = blockIdx.y, quad = blockIdx.x / gx;
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6;
  const int64_t g = (int64_t)(blockIdx.x % gx) * kBwdGroups + lane;
  const Channels ch = channels_of<FEW>(g < s.G ? g : s.G - 1, s.D);
  const int64_t n = live_frames(lengths, b, s.T), last = n > 0 ? n - 1 : 0;
  const int64_t t0 = (quad * kBwdTiles + sub) * s.tile, t1 = t0 + s.tile < s.T ? t0 + s.tile : s.T;
  float dw[W][4] = {}, dbs[4] = {};
  if (t0 < s.T && g < s.G) {
    const T* xp = x + b * xb + ch.c;
    const T* gp = dy + b * gb + ch.c;
    // (a sequence without frames takes nothing of its state, whatever that holds)
    const T* sp = state && n > 0 ? state + b * (W - 1) * s.D + ch.c : nullptr;
    T* op = dx + b * db + ch.c;
    Four<T> nextx[kGroup], nextg[kGroup];
    auto fetch = [&](int64_t t) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        const int64_t at = t + k < last ? t + k : last;
        nextx[k] = get_four<FEW>(xp + at * xt, ch);
        nextg[k] = get_four<FEW>(gp + at * gt, ch);
      }
    };
    fetch(t0);
    Taps<W> taps;
    taps.load(w, bias, ch);
    // win[q]: frame t - (W-1) + q, du[q]: du of frame t - (W-1) + q
    float win[W - 1 + kGroup][4], du[W - 1 + kGroup][4];
#pragma unroll
    for (int q = 0; q < W - 1; ++q) {
      const int64_t t = t0 - (W - 1) + q;
      if (t < 0) {
        frame_before<T, W, FEW>(sp, s.D, t, ch, win[q]);
      } else {
        const Four<T> f = get_four<FEW>(xp + (t < last ? t : last) * xt, ch);
#pragma unroll
        for (int e = 0; e < 4; ++e) win[q][e] = t < n ? to_f32(f.e[e]) : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) du[q][e] = 0.f;
    }
    for (int64_t t = t0; t < t1 + W - 1; t += kGroup) {
      Four<T> cx[kGroup], cg[kGroup];
#pragma unroll
      for (int k = 0; k < kGroup; ++k) cx[k] = nextx[k], cg[k] = nextg[k];
      if (t + kGroup < t1 + W - 1) fetch(t + kGroup);
      // INSIDE: every frame of the group lies in the tile and the sequence, and
      // the ones that get their gradient now do too
      auto group = [&](auto insidec) {
        constexpr bool INSIDE = decltype(insidec)::value;
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
          const bool in = INSIDE || t + k < n;
          const bool own = INSIDE || t + k < t1;  // (frames past the tile only for the gradients before them)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = to_f32(cx[k].e[e]);
            float d = to_f32(cg[k].e[e]);
            win[W - 1 + k][e] = in ? x : 0.f;
            if (SILU) {
              float u = taps.bias[e];
#pragma unroll
              for (int q = 0; q < W; ++q) u = fmaf(taps.w[q][e], win[k + q][e], u);
              d *= silu_grad(u, sigmoid(u));
            }
            if (!in) d = 0.f;
            du[W - 1 + k][e] = d;
            if (in && own) {  // (0 times a frame before the end is no 0 where that is infinite)
              dbs[e] += d;
#pragma unroll
              for (int q = 0; q < W; ++q) dw[q][e] = fmaf(d, win[k + q][e], dw[q][e]);
            }
          }
          // the frame that has all of its du now
          const int64_t to = t + k - (W - 1);
          if (INSIDE || (to >= t0 && to < t1)) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[e] = 0.f;
              // dx[to] = sum_q w[q] du[to + W-1-q]
#pragma unroll
              for (int q = 0; q < W; ++q) o[e] = fmaf(taps.w[q][e], du[W - 1 + k - q][e], o[e]);
              if (!INSIDE && to >= n) o[e] = 0.f;
            }
            put_four(op + to * dt, ch, o);
          }
        }
      };
      if (t - (W - 1) >= t0 && t + kGroup <= t1 && t + kGroup <= n) group(std::true_type{});
      else group(std::false_type{});
#pragma unroll
      for (int q = 0; q < W - 1; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          win[q][e] = win[q + kGroup][e];
          du[q][e] = du[q + kGroup][e];
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
    // thread (sub, lane): channel `sub` of the lane's four
    if (g < s.G && sub >= ch.skip && sub < ch.end) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < kBwdTiles; ++k) t += red[k][lane][sub];
      if (q < W) out[(ch.c + sub) * W + q] = t;
      else out[s.D * W + ch.c + sub] = t;
    }
  }
}

int64_t conv_quads(const ConvShape& s) { return (s.tiles + kBwdTiles - 1) / kBwdTiles; }

template <class T, int W, bool SILU, bool FEW>
void conv_launch(const dgen_hip_conv& a, bool backward, hipStream_t st) {
  const ConvShape s = conv_shape(a, backward);
  if (!backward) {
    const int64_t threads = s.B * s.tiles * s.G;
    k_conv<T, W, SILU, FEW><<<dim3((unsigned)((threads + kFwdThreads - 1) / kFwdThreads)), kFwdThreads, 0, st>>>(
        s, (const T*)a.x.data, a.x.stride_b, a.x.stride_t, a.weight, a.bias, a.lengths, (const T*)a.state,
        (T*)a.state_out, (T*)a.y.data, a.y.stride_b, a.y.stride_t);
  } else {
    const int64_t quads = conv_quads(s);
    float* parts = (float*)a.workspace;
    k_conv_bwd<T, W, SILU, FEW>
        <<<dim3((unsigned)((s.G + kBwdGroups - 1) / kBwdGroups * quads), (unsigned)s.B), kBwdGroups * kBwdTiles, 0,
           st>>>(s, (const T*)a.x.data, a.x.stride_b, a.x.stride_t, (const T*)a.dy.data, a.dy.stride_b, a.dy.stride_t,
                 a.weight, a.bias, a.lengths, (const T*)a.state, (T*)a.dx.data, a.dx.stride_b, a.dx.stride_t, parts,
                 quads);
    enqueue_sum_parts(st, parts, s.B * quads, {{a.dweight, a.dbias, nullptr}, {s.D * W, s.D, 0}});
  }
}

template <class T, bool SILU, bool FEW>
void conv_taps(const dgen_hip_conv& a, bool backward, hipStream_t st) {
  switch (a.width) {
    case 1: return conv_launch<T, 1, SILU, FEW>(a, backward, st);
    case 2: return conv_launch<T, 2, SILU, FEW>(a, backward, st);
    case 3: return conv_launch<T, 3, SILU, FEW>(a, backward, st);
    case 4: return conv_launch<T, 4, SILU, FEW>(a, backward, st);
    case 5: return conv_launch<T, 5, SILU, FEW>(a, backward, st);
    case 6: return conv_launch<T, 6, SILU, FEW>(a, backward, st);
    case 7: return conv_launch<T, 7, SILU, FEW>(a, backward, st);
    default: return conv_launch<T, 8, SILU, FEW>(a, backward, st);
  }
}

template <class T>
void conv_form(const dgen_hip_conv& a, bool backward, hipStream_t st) {
  if (a.D < 4) a.silu ? conv_taps<T, true, true>(a, backward, st) : conv_taps<T, false, true>(a, backward, st);
  else a.silu ? conv_taps<T, true, false>(a, backward, st) : conv_taps<T, false, false>(a, backward, st);
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
    conv_form<bf16>(a, backward, st);
  } else {
    conv_form<float>(a, backward, st);
  }
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
