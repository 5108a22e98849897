// Gated delta rule, forward and backward.
#include "seq.h"

namespace dgen {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr int kC = 64;  // frames of a chunk
constexpr int kThreads = 256;
constexpr int kStepFrames = 16;  // calls of so few go frame by frame
constexpr float kUnitEps = 1e-6f;

// Parts of fp32 numbers in bf16 products: of what goes into the memory, and of
// what goes into results that are rounded to bf16.
constexpr int kState = 3, kResult = 2;

// ------------------------------------------------------- fragments, products
// Eight consecutive elements of one row, as the matrix instructions take them
// (lane: row lane % 16, elements 8 (lane / 16) and on; for fp32 the four
// instructions' order of the sum is not theirs, but the same for both operands):
// bf16 in P parts, each the rounding of what the ones before leave.
template <class E, int P>
struct Wide;
template <int P>
struct Wide<bf16, P> {
  bf16x8 p[P];
};
template <int P>
struct Wide<float, P> {
  float p[8];
};

template <class E, int P>
__device__ __forceinline__ Wide<E, P> wide(const float (&v)[8]) {
  Wide<E, P> w;
  if constexpr (std::is_same<E, float>::value) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w.p[i] = v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = v[i];
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const __bf16 h = (__bf16)x;
        w.p[q][i] = h;
        x -= (float)h;
      }
    }
  }
  return w;
}

// acc += a b over the eight elements of each of the four lane groups.
template <int PA, int PB>
__device__ __forceinline__ void mma(floatx4& acc, const Wide<bf16, PA>& a, const Wide<bf16, PB>& b) {
  constexpr int most = PA > PB ? PA : PB;
#pragma unroll
  for (int s = most - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (s - i >= 0 && s - i < PB) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[s - i], acc, 0, 0, 0);
}
template <int PA, int PB>
__device__ __forceinline__ void mma(floatx4& acc, const Wide<float, PA>& a, const Wide<float, PB>& b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.p[i], b.p[i], acc, 0, 0, 0);
}
// The first Q parts.
template <int Q, int P>
__device__ __forceinline__ Wide<bf16, Q> first(const Wide<bf16, P>& w) {
  Wide<bf16, Q> o;
#pragma unroll
  for (int i = 0; i < Q; ++i) o.p[i] = w.p[i];
  return o;
}
template <int Q, int P>
__device__ __forceinline__ Wide<float, Q> first(const Wide<float, P>& w) {
  Wide<float, Q> o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o.p[i] = w.p[i];
  return o;
}

// A matrix in LDS whose rows are fragments' rows, split into parts as it is
// written.  Rows are 16 bytes longer than they need be, so that the 16 rows of a
// fragment start in different banks.
template <class E, int P, int ROWS, int COLS>
struct Tile {
  static constexpr bool kFloat = std::is_same<E, float>::value;
  static constexpr int kLd = COLS + (kFloat ? 4 : 8), kParts = kFloat ? 1 : P;
  using T = typename std::conditional<kFloat, float, __bf16>::type;
  alignas(16) T d[kParts][ROWS * kLd];

  __device__ __forceinline__ void put(int row, int col, float x) {
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      const T h = (T)x;
      d[q][row * kLd + col] = h;
      x -= (float)h;
    }
  }
  // Four consecutive columns.
  __device__ __forceinline__ void put4(int row, int col, floatx4 x) {
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      if constexpr (kFloat) {
        *reinterpret_cast<floatx4*>(&d[q][row * kLd + col]) = x;
      } else {
        bf16x4 h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h[i] = (__bf16)x[i];
          x[i] -= (float)h[i];
        }
        *reinterpret_cast<bf16x4*>(&d[q][row * kLd + col]) = h;
      }
    }
  }
  __device__ __forceinline__ Wide<E, P> frag(int row, int col) const {
    Wide<E, P> w;
    if constexpr (kFloat) {
      const floatx4 a = *reinterpret_cast<const floatx4*>(&d[0][row * kLd + col]);
      const floatx4 b = *reinterpret_cast<const floatx4*>(&d[0][row * kLd + col + 4]);
#pragma unroll
      for (int i = 0; i < 4; ++i) w.p[i] = a[i], w.p[4 + i] = b[i];
    } else {
#pragma unroll
      for (int q = 0; q < P; ++q) w.p[q] = *reinterpret_cast<const bf16x8*>(&d[q][row * kLd + col]);
    }
    return w;
  }
  __device__ __forceinline__ float at(int row, int col) const {
    float x = 0.f;
#pragma unroll
    for (int q = 0; q < kParts; ++q) x += (float)d[q][row * kLd + col];
    return x;
  }
};

template <class T>
struct __attribute__((packed, aligned(alignof(T)))) Eight {
  T e[8];
};
// Eight elements of a row, those past its end (or all of a row that is off) 0.
template <class T>
__device__ __forceinline__ void load_eight(const T* __restrict__ p, int left, float (&o)[8]) {
  if (left >= 8) {
    const Eight<T> f = *reinterpret_cast<const Eight<T>*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = to_f32(f.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = i < left ? to_f32(p[i]) : 0.f;
  }
}
template <class E>
__device__ __forceinline__ Wide<E, 1> load_exact(const E* __restrict__ p, int left) {
  float v[8];
  load_eight(p, left, v);
  return wide<E, 1>(v);
}

// ------------------------------------------------------------------ operands
template <class E>
struct Heads {  // [batch][time][head][.]
  E* p;
  int64_t b, t, h;
  __device__ __forceinline__ E* row(int bi, int64_t ti, int hi) const { return p + bi * b + ti * t + hi * h; }
};
struct Gates {  // [batch][time][head]
  float* p;
  int64_t b, t;
};

// Numbers of a chunk's frames, 64 each.
enum Vec { kReadK, kWriteK, kReadQ, kBeta, kGHigh, kGLow, kRootK, kRootQ, kInto, kRest, kVecs };

template <class E>
struct DeltaP {
  Heads<const E> q, k, v, dy;
  Heads<E> y, dq, dk, dv;
  Gates g, beta, dg, dbeta;
  const int32_t* lengths;
  const float* state;
  float* state_out;
  float scale;
  int normalize;
  int B, T, H, shared, K, V;
  int chunks, nvb, segs, per;  // chunks a segment
  float *X, *M, *vec;          // [B H][chunks]: inverse, queries' products with keys [64][64], Vec [kVecs][64]
  float *S, *dS, *U, *dR;      // backward: states entering and adjoints after a chunk [K][V], [64][V]
  float *ends, *gends;         // [B H][segs][K][V + K] (states | transitions), [K][V]
};

__device__ __forceinline__ int live_of(const int32_t* __restrict__ lengths, int b, int T) {
  if (!lengths) return T;
  const int n = lengths[b];
  return n < 0 ? 0 : n < T ? n : T;
}

// ------------------------------------------------------------------- prepare
// Per chunk and head: decays, norms, M and X.
template <class E, int KP>
__global__ __launch_bounds__(kThreads) void k_delta_prepare(DeltaP<E> p) {
  constexpr int NF = KP / 32;
  __shared__ float A[kC][kC + 4], X[kC][kC + 4], part[3][16][20];
  __shared__ float gh[kC], gl[kC], bt[kC], rk[kC], rq[kC];
  const int c = blockIdx.x % (uint32_t)p.chunks, bh = blockIdx.x / (uint32_t)p.chunks, b = bh / p.H, h = bh % p.H;
  const int t0 = c * kC, live = live_of(p.lengths, b, p.T) - t0;
  if (live <= 0) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, g4 = lane >> 4, hk = h / p.shared;
  const int64_t ci = (int64_t)bh * p.chunks + c;
  if (w == 0) {
    const bool on = lane < live;
    float g = on ? p.g.p[b * p.g.b + (int64_t)(t0 + lane) * p.g.t + h] : 0.f;
    g = g < -128.f ? -128.f : g;
    double s = (double)g;
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
      const double o = __shfl_up(s, k, 64);
      if (lane >= k) s += o;
    }
    gh[lane] = (float)s;
    gl[lane] = (float)(s - (double)(float)s);
    bt[lane] = on ? p.beta.p[b * p.beta.b + (int64_t)(t0 + lane) * p.beta.t + h] : 0.f;
  }
  const int row = 16 * w + l16;
  const int left = row < live ? p.K : 0;
  Wide<E, 1> kf[NF], qf[NF];
  {
    float sk = 0.f, sq = 0.f;
    const E *kp = p.k.row(b, t0 + row, hk), *qp = p.q.row(b, t0 + row, hk);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int at = f * 32 + g4 * 8;
      float x[8];
      load_eight(kp + at, left - at, x);
      kf[f] = wide<E, 1>(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) sk = fmaf(x[i], x[i], sk);
      load_eight(qp + at, left - at, x);
      qf[f] = wide<E, 1>(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) sq = fmaf(x[i], x[i], sq);
    }
    sk += __shfl_xor(sk, 16, 64), sk += __shfl_xor(sk, 32, 64);
    sq += __shfl_xor(sq, 16, 64), sq += __shfl_xor(sq, 32, 64);
    if (g4 == 0) {
      rk[row] = p.normalize ? __builtin_amdgcn_rsqf(sk + kUnitEps) : 1.f;
      rq[row] = p.normalize ? __builtin_amdgcn_rsqf(sq + kUnitEps) : 1.f;
    }
  }
  __syncthreads();
  float* Mp = p.M + ci * kC * kC;
#pragma unroll
  for (int tj = 0; tj < 4; ++tj) {
    floatx4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
    const int j = 16 * tj + l16;
    if (tj <= w) {
      const E* kp = p.k.row(b, t0 + j, hk);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int at = f * 32 + g4 * 8;
        const Wide<E, 1> o = load_exact(kp + at, j < live ? p.K - at : 0);
        mma(kk, kf[f], o);
        mma(qk, qf[f], o);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * w + 4 * g4 + r;
      const float d = j <= i ? exp_accurate((gh[i] - gh[j]) + (gl[i] - gl[j])) : 0.f;
      A[i][j] = j < i ? kk[r] * (rk[i] * rk[j]) * d * bt[i] : 0.f;
      Mp[i * kC + j] = j <= i ? qk[r] * (rq[i] * rk[j] * p.scale) * d : 0.f;
      X[i][j] = 0.f;
    }
  }
  __syncthreads();
  // (I + A)^-1: the diagonal blocks by substitution, a column a lane
  if (lane < 16) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == lane ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) s = fmaf(-A[16 * w + i][16 * w + j], x[j], s);
      x[i] = s;
      X[16 * w + i][16 * w + lane] = s;
    }
  }
  __syncthreads();
  // then X[i][j] = -X[i][i] sum over m of A[i][m] X[m][j], diagonal by diagonal
#pragma unroll
  for (int dist = 1; dist < 4; ++dist) {
    if (w + dist < 4) {
      const int bi = w + dist;
      floatx4 s = {0, 0, 0, 0};
      for (int m = w; m < bi; ++m)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          s = __builtin_amdgcn_mfma_f32_16x16x4f32(A[16 * bi + l16][16 * m + 4 * g4 + k], X[16 * m + 4 * g4 + k][16 * w + l16], s,
                                                   0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) part[w][4 * g4 + r][l16] = s[r];
      wave_sync();
      floatx4 o = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        o = __builtin_amdgcn_mfma_f32_16x16x4f32(X[16 * bi + l16][16 * bi + 4 * g4 + k], part[w][4 * g4 + k][l16], o, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) X[16 * bi + 4 * g4 + r][16 * w + l16] = -o[r];
    }
    __syncthreads();
  }
  float* Xp = p.X + ci * kC * kC;
  for (int i = threadIdx.x; i < kC * kC / 4; i += kThreads) {
    const int r = i / (kC / 4), col = i % (kC / 4) * 4;
    *reinterpret_cast<floatx4*>(Xp + r * kC + col) = *reinterpret_cast<const floatx4*>(&X[r][col]);
  }
  if (w == 0) {
    float* v = p.vec + ci * kVecs * kC + lane;
    const float into = exp_accurate(gh[lane] + gl[lane]);
    const float rest = exp_accurate((gh[kC - 1] - gh[lane]) + (gl[kC - 1] - gl[lane]));
    v[kReadK * kC] = into * rk[lane];
    v[kWriteK * kC] = rest * rk[lane];
    v[kReadQ * kC] = into * rq[lane] * p.scale;
    v[kBeta * kC] = bt[lane];
    v[kGHigh * kC] = gh[lane];
    v[kGLow * kC] = gl[lane];
    v[kRootK * kC] = rk[lane];
    v[kRootQ * kC] = rq[lane];
    v[kInto * kC] = into;
    v[kRest * kC] = rest;
  }
}

// --------------------------------------------------------------------- chain
enum Mode { kOut, kEnds, kKeep };

// A workgroup's sequence and head, block of VB values and segment of chunks.
struct Place {
  int b, h, hk, bh, vb, seg;
};
template <class E>
__device__ __forceinline__ Place place_of(const DeltaP<E>& p, int blocks) {
  Place o;
  uint32_t i = blockIdx.x;
  o.vb = i % (uint32_t)blocks, i /= (uint32_t)blocks;
  o.seg = i % (uint32_t)p.segs, i /= (uint32_t)p.segs;
  o.bh = i;
  o.b = o.bh / p.H, o.h = o.bh % p.H;
  o.hk = o.h / p.shared;
  return o;
}

// The memory's states along a segment's chunks.
template <class E, int KP, int VB, Mode MODE>
__global__ __launch_bounds__(kThreads) void k_delta_chain(DeltaP<E> p) {
  constexpr int NF = KP / 32, NV = VB / 16, NT = KP / 16 * NV / 4;
  __shared__ Tile<E, kState, VB, KP> s;
  __shared__ Tile<E, kState, VB, kC> r, wr;
  __shared__ Tile<E, kResult, MODE == kOut ? VB : 1, kC> u;
  __shared__ Tile<E, 1, KP, kC> kt;
  const int nvb = MODE == kEnds ? p.nvb + (p.K + VB - 1) / VB : p.nvb;
  const Place at = place_of(p, nvb);
  const int live = live_of(p.lengths, at.b, p.T);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, g4 = lane >> 4;
  // (ends: the transition is the state's own columns, from the identity on and
  // with nothing written)
  const bool unit = MODE == kEnds && at.vb >= p.nvb;
  const int v0 = (unit ? at.vb - p.nvb : at.vb) * VB, width = unit ? p.K : p.V;
  const int64_t end = ((int64_t)at.bh * p.segs + at.seg) * p.K;
  const int ld = p.V + p.K;
  floatx4 S[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int k = (w * NT + i) / NV * 16 + 4 * g4, v = v0 + (w * NT + i) % NV * 16 + l16;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      S[i][e] = 0.f;
      if (unit) S[i][e] = k + e == v ? 1.f : 0.f;
      else if (MODE != kEnds && k + e < p.K && v < p.V) {
        if (p.segs > 1) S[i][e] = p.ends[(end + k + e) * ld + v];
        else if (p.state) S[i][e] = p.state[((int64_t)at.bh * p.K + k + e) * p.V + v];
      }
    }
    s.put4(v - v0, k, S[i]);
  }
  __syncthreads();
  const int c1 = min((at.seg + 1) * p.per, p.chunks);
  for (int c = at.seg * p.per; c < c1; ++c) {
    const int t0 = c * kC;
    if (t0 >= live) {
      if constexpr (MODE == kOut) {
        for (int i = threadIdx.x; i < kC * VB; i += kThreads) {
          const int t = t0 + i / VB, v = v0 + i % VB;
          if (t < p.T && v < p.V) p.y.row(at.b, t, at.h)[v] = from_f32<E>(0.f);
        }
      }
      continue;
    }
    const int64_t ci = (int64_t)at.bh * p.chunks + c;
    const float* vec = p.vec + ci * kVecs * kC;
    const int row = 16 * w + l16, rows = 16 * w + 4 * g4;
    const int left = t0 + row < live ? p.K : 0;
    Wide<E, 1> kf[NF], qf[MODE == kOut ? NF : 1];
    const E *kp = p.k.row(at.b, t0 + row, at.hk), *qp = p.q.row(at.b, t0 + row, at.hk);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int col = f * 32 + g4 * 8;
      float x[8];
      load_eight(kp + col, left - col, x);
      kf[f] = wide<E, 1>(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) kt.put(col + i, row, x[i]);
      if constexpr (MODE == kOut) qf[f] = load_exact(qp + col, left - col);
    }
    if constexpr (MODE == kKeep) {
      float* out = p.S + ci * p.K * p.V;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int k = (w * NT + i) / NV * 16 + 4 * g4, v = v0 + (w * NT + i) % NV * 16 + l16;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < p.K && v < p.V) out[(int64_t)(k + e) * p.V + v] = S[i][e];
      }
    }
    floatx4 ks[NV] = {}, qs[MODE == kOut ? NV : 1] = {};
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const Wide<E, kState> o = s.frag(16 * v + l16, f * 32 + g4 * 8);
        mma(ks[v], kf[f], o);
        if constexpr (MODE == kOut) mma(qs[v], qf[f], first<kResult>(o));
      }
    const floatx4 beta = *reinterpret_cast<const floatx4*>(vec + kBeta * kC + rows);
    const floatx4 read = *reinterpret_cast<const floatx4*>(vec + kReadK * kC + rows);
    const floatx4 write = *reinterpret_cast<const floatx4*>(vec + kWriteK * kC + rows);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = v0 + 16 * v + l16;
      floatx4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = t0 + rows + e;
        const float val = !unit && t < live && col < p.V ? to_f32(p.v.row(at.b, t, at.h)[col]) : 0.f;
        x[e] = beta[e] * fmaf(-read[e], ks[v][e], val);
      }
      r.put4(16 * v + l16, rows, x);
    }
    __syncthreads();
    floatx4 U[NV] = {};
    {
      const float* X = p.X + (ci * kC + row) * kC + g4 * 8;
      for (int f = 0; f <= w / 2; ++f) {
        float x[8];
        load_eight(X + f * 32, 8, x);
        const Wide<E, kState> o = wide<E, kState>(x);
#pragma unroll
        for (int v = 0; v < NV; ++v) mma(U[v], o, r.frag(16 * v + l16, f * 32 + g4 * 8));
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      wr.put4(16 * v + l16, rows, U[v] * write);
      if constexpr (MODE == kOut) u.put4(16 * v + l16, rows, U[v]);
      if constexpr (MODE == kKeep) {
        const int col = v0 + 16 * v + l16;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col < p.V) p.U[(ci * kC + rows + e) * p.V + col] = U[v][e];
      }
    }
    __syncthreads();
    if constexpr (MODE == kOut) {
      const floatx4 q = *reinterpret_cast<const floatx4*>(vec + kReadQ * kC + rows);
#pragma unroll
      for (int v = 0; v < NV; ++v) qs[v] *= q;
      const float* M = p.M + (ci * kC + row) * kC + g4 * 8;
      for (int f = 0; f <= w / 2; ++f) {
        float x[8];
        load_eight(M + f * 32, 8, x);
        const Wide<E, kResult> o = wide<E, kResult>(x);
#pragma unroll
        for (int v = 0; v < NV; ++v) mma(qs[v], o, u.frag(16 * v + l16, f * 32 + g4 * 8));
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int col = v0 + 16 * v + l16;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = t0 + rows + e;
          if (t < p.T && col < p.V) p.y.row(at.b, t, at.h)[col] = from_f32<E>(t < live ? qs[v][e] : 0.f);
        }
      }
    }
    const float whole = vec[kInto * kC + kC - 1];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int k = (w * NT + i) / NV * 16, v = (w * NT + i) % NV * 16;
      S[i] *= whole;
#pragma unroll
      for (int f = 0; f < 2; ++f) mma(S[i], kt.frag(k + l16, f * 32 + g4 * 8), wr.frag(v + l16, f * 32 + g4 * 8));
      s.put4(v + l16, k + 4 * g4, S[i]);
    }
    __syncthreads();
  }
  float* out = nullptr;
  if (MODE == kOut && at.seg == p.segs - 1) out = p.state_out;
  if (MODE != kEnds && !out) return;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int k = (w * NT + i) / NV * 16 + 4 * g4, v = v0 + (w * NT + i) % NV * 16 + l16;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (k + e >= p.K || v >= width) continue;
      if (MODE == kEnds) p.ends[(end + k + e) * ld + (unit ? p.V : 0) + v] = S[i][e];
      else out[((int64_t)at.bh * p.K + k + e) * p.V + v] = S[i][e];
    }
  }
}

// The states that enter the segments (BACK: the adjoints after them) from the
// segments' ends from zero and their transitions, in the ends' place.
template <class E, int KP, bool BACK>
__global__ __launch_bounds__(kThreads) void k_delta_carry(DeltaP<E> p) {
  constexpr int VB = 32, NF = KP / 32, NV = 2, NT = KP / 16 * NV / 4;
  __shared__ Tile<float, 1, VB, KP> s;
  const int nvb = (p.V + VB - 1) / VB, vb = blockIdx.x % (uint32_t)nvb, bh = blockIdx.x / (uint32_t)nvb, v0 = vb * VB;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, g4 = lane >> 4, ld = p.V + p.K;
  floatx4 S[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int k = (w * NT + i) / NV * 16 + 4 * g4, v = v0 + (w * NT + i) % NV * 16 + l16;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      S[i][e] = !BACK && p.state && k + e < p.K && v < p.V ? p.state[((int64_t)bh * p.K + k + e) * p.V + v] : 0.f;
  }
  for (int n = 0; n < p.segs; ++n) {
    const int seg = BACK ? p.segs - 1 - n : n;
    const int64_t at = ((int64_t)bh * p.segs + seg) * p.K;
#pragma unroll
    for (int i = 0; i < NT; ++i) s.put4((w * NT + i) % NV * 16 + l16, (w * NT + i) / NV * 16 + 4 * g4, S[i]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int kt = (w * NT + i) / NV * 16, k = kt + 4 * g4, v = v0 + (w * NT + i) % NV * 16 + l16;
      floatx4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = 0.f;
        if (k + e < p.K && v < p.V) {
          float* end = BACK ? p.gends + (at + k + e) * p.V + v : p.ends + (at + k + e) * ld + v;
          o[e] = *end;
          *end = S[i][e];
        }
      }
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int col = f * 32 + g4 * 8, row = kt + l16;
        Wide<float, 1> a;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int x = BACK ? col + e : row, y = BACK ? row : col + e;
          a.p[e] = row < p.K && col + e < p.K ? p.ends[(at + x) * ld + p.V + y] : 0.f;
        }
        mma(o, a, s.frag((w * NT + i) % NV * 16 + l16, col));
      }
      S[i] = o;
    }
    __syncthreads();
  }
}

// The adjoints of the memory's states, against time.  Leaves dv, and dR.
template <class E, int KP, int VB, Mode MODE>
__global__ __launch_bounds__(kThreads) void k_delta_back(DeltaP<E> p) {
  constexpr int NF = KP / 32, NV = VB / 16, NT = KP / 16 * NV / 4;
  __shared__ Tile<E, kState, VB, KP> s;
  __shared__ Tile<E, 1, VB, kC> dyt;
  __shared__ Tile<E, kState, VB, kC> qdy, du, dr;
  __shared__ Tile<E, 1, KP, kC> kt, qt;
  const Place at = place_of(p, p.nvb);
  const int live = live_of(p.lengths, at.b, p.T);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, g4 = lane >> 4;
  const int v0 = at.vb * VB;
  const int64_t end = ((int64_t)at.bh * p.segs + at.seg) * p.K;
  floatx4 S[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int k = (w * NT + i) / NV * 16 + 4 * g4, v = v0 + (w * NT + i) % NV * 16 + l16;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      S[i][e] = MODE == kKeep && p.segs > 1 && k + e < p.K && v < p.V ? p.gends[(end + k + e) * p.V + v] : 0.f;
    s.put4(v - v0, k, S[i]);
  }
  __syncthreads();
  const int c0 = at.seg * p.per;
  for (int c = min((at.seg + 1) * p.per, p.chunks) - 1; c >= c0; --c) {
    const int t0 = c * kC;
    if (t0 >= live) {
      if constexpr (MODE == kKeep) {
        for (int i = threadIdx.x; i < kC * VB; i += kThreads) {
          const int t = t0 + i / VB, v = v0 + i % VB;
          if (t < p.T && v < p.V) p.dv.row(at.b, t, at.h)[v] = from_f32<E>(0.f);
        }
      }
      continue;
    }
    const int64_t ci = (int64_t)at.bh * p.chunks + c;
    const float* vec = p.vec + ci * kVecs * kC;
    const int row = 16 * w + l16, rows = 16 * w + 4 * g4;
    const int left = t0 + row < live ? p.K : 0;
    Wide<E, 1> kf[NF];
    const E *kp = p.k.row(at.b, t0 + row, at.hk), *qp = p.q.row(at.b, t0 + row, at.hk);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int col = f * 32 + g4 * 8;
      float x[8];
      load_eight(kp + col, left - col, x);
      kf[f] = wide<E, 1>(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) kt.put(col + i, row, x[i]);
      load_eight(qp + col, left - col, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) qt.put(col + i, row, x[i]);
    }
    if constexpr (MODE == kKeep) {
      float* out = p.dS + ci * p.K * p.V;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int k = (w * NT + i) / NV * 16 + 4 * g4, v = v0 + (w * NT + i) % NV * 16 + l16;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < p.K && v < p.V) out[(int64_t)(k + e) * p.V + v] = S[i][e];
      }
    }
    const floatx4 beta = *reinterpret_cast<const floatx4*>(vec + kBeta * kC + rows);
    const floatx4 read = *reinterpret_cast<const floatx4*>(vec + kReadK * kC + rows);
    const floatx4 write = *reinterpret_cast<const floatx4*>(vec + kWriteK * kC + rows);
    const floatx4 readq = *reinterpret_cast<const floatx4*>(vec + kReadQ * kC + rows);
    floatx4 U[NV] = {};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int col = v0 + 16 * v + l16;
      floatx4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = t0 + rows + e;
        x[e] = t < live && col < p.V ? to_f32(p.dy.row(at.b, t, at.h)[col]) : 0.f;
      }
      dyt.put4(16 * v + l16, rows, x);
      qdy.put4(16 * v + l16, rows, x * readq);
#pragma unroll
      for (int f = 0; f < NF; ++f) mma(U[v], kf[f], s.frag(16 * v + l16, f * 32 + g4 * 8));
      U[v] *= write;
    }
    __syncthreads();
    {
      const float* M = p.M + (ci * kC + g4 * 8) * kC + row;
      for (int f = w / 2; f < 2; ++f) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = M[(f * 32 + i) * kC];
        const Wide<E, kState> o = wide<E, kState>(x);
#pragma unroll
        for (int v = 0; v < NV; ++v) mma(U[v], o, dyt.frag(16 * v + l16, f * 32 + g4 * 8));
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) du.put4(16 * v + l16, rows, U[v]);
    }
    __syncthreads();
    floatx4 R[NV] = {};
    {
      const float* X = p.X + (ci * kC + g4 * 8) * kC + row;
      for (int f = w / 2; f < 2; ++f) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = X[(f * 32 + i) * kC];
        const Wide<E, kState> o = wide<E, kState>(x);
#pragma unroll
        for (int v = 0; v < NV; ++v) mma(R[v], o, du.frag(16 * v + l16, f * 32 + g4 * 8));
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      dr.put4(16 * v + l16, rows, -R[v] * beta * read);
      if constexpr (MODE == kKeep) {
        const int col = v0 + 16 * v + l16;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = t0 + rows + e;
          if (col >= p.V) continue;
          p.dR[(ci * kC + rows + e) * p.V + col] = R[v][e];
          if (t < p.T) p.dv.row(at.b, t, at.h)[col] = from_f32<E>(t < live ? beta[e] * R[v][e] : 0.f);
        }
      }
    }
    __syncthreads();
    const float whole = vec[kInto * kC + kC - 1];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int k = (w * NT + i) / NV * 16, v = (w * NT + i) % NV * 16;
      S[i] *= whole;
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int col = f * 32 + g4 * 8;
        mma(S[i], qt.frag(k + l16, col), qdy.frag(v + l16, col));
        mma(S[i], kt.frag(k + l16, col), dr.frag(v + l16, col));
      }
      s.put4(v + l16, k + 4 * g4, S[i]);
    }
    __syncthreads();
  }
  if constexpr (MODE == kEnds) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int k = (w * NT + i) / NV * 16 + 4 * g4, v = v0 + (w * NT + i) % NV * 16 + l16;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k + e < p.K && v < p.V) p.gends[(end + k + e) * p.V + v] = S[i][e];
    }
  }
}

// -------------------------------------------------------------------- grads
// Per chunk and key head: the gradients of q, k, g and beta from the states
// that enter, the adjoints of those that leave, U and dR.
constexpr int kGradParts = 3;
template <class E, int KP>
struct GradLds {
  union {
    struct {
      Tile<E, kGradParts, KP, 32> s, d;
      Tile<E, kGradParts, kC, 32> u;
    } a;
    struct {
      Tile<E, kGradParts, kC, kC> n, nt;
    } b;
  };
  Tile<E, 1, KP, kC> kt, qt;
  float gh[kC], gl[kC], at[kC], db[kC], red[4][2];
};

template <class E, int KP>
__global__ __launch_bounds__(kThreads) void k_delta_grads(DeltaP<E> p) {
  constexpr int NF = KP / 32, NK = KP / 16;
  __shared__ GradLds<E, KP> L;
  const int G = p.H / p.shared, c = blockIdx.x % (uint32_t)p.chunks, bg = blockIdx.x / (uint32_t)p.chunks;
  const int b = bg / G, hk = bg % G, t0 = c * kC, live = live_of(p.lengths, b, p.T) - t0;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, g4 = lane >> 4;
  const int row = 16 * w + l16, rows = 16 * w + 4 * g4;
  if (live <= 0) {
    for (int i = threadIdx.x; i < kC * p.K; i += kThreads) {
      const int t = t0 + i / p.K, k = i % p.K;
      if (t < p.T) p.dq.row(b, t, hk)[k] = p.dk.row(b, t, hk)[k] = from_f32<E>(0.f);
    }
    for (int i = threadIdx.x; i < kC * p.shared; i += kThreads) {
      const int t = t0 + i / p.shared, h = hk * p.shared + i % p.shared;
      if (t < p.T) p.dg.p[b * p.dg.b + t * p.dg.t + h] = p.dbeta.p[b * p.dbeta.b + t * p.dbeta.t + h] = 0.f;
    }
    return;
  }
  {
    const int left = row < live ? p.K : 0;
    const E *kp = p.k.row(b, t0 + row, hk), *qp = p.q.row(b, t0 + row, hk);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int col = f * 32 + g4 * 8;
      float x[8];
      load_eight(kp + col, left - col, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) L.kt.put(col + i, row, x[i]);
      load_eight(qp + col, left - col, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) L.qt.put(col + i, row, x[i]);
    }
  }
  // Sum over the 16 lanes of a row.
  auto row_total = [](floatx4 v) {
#pragma unroll
    for (int k = 1; k < 16; k *= 2)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], k, 64);
    return v;
  };
  floatx4 DQ[NK] = {}, DK[NK] = {}, qdq = {0, 0, 0, 0}, kdk = {0, 0, 0, 0}, rootk, rootq;
  for (int n = 0; n < p.shared; ++n) {
    const int h = hk * p.shared + n;
    const int64_t ci = ((int64_t)b * p.H + h) * p.chunks + c;
    const float* vec = p.vec + ci * kVecs * kC;
    const float *Sp = p.S + ci * p.K * p.V, *Dp = p.dS + ci * p.K * p.V;
    const float *Up = p.U + ci * kC * p.V, *Rp = p.dR + ci * kC * p.V;
    __syncthreads();
    if (threadIdx.x < kC) L.gh[threadIdx.x] = vec[kGHigh * kC + threadIdx.x], L.gl[threadIdx.x] = vec[kGLow * kC + threadIdx.x];
    floatx4 dq[NK] = {}, z[NK] = {}, wr[NK] = {}, dm[4] = {}, da[4] = {};
    float sd = 0.f, rv = 0.f;
    for (int v0 = 0; v0 < p.V; v0 += 32) {
      if (v0) __syncthreads();
      for (int i = threadIdx.x; i < KP * 8; i += kThreads) {
        const int k = i / 8, v = i % 8 * 4, left = k < p.K ? p.V - v0 - v : 0;
        float x[4], y[4];
        load_four(Sp + (int64_t)k * p.V + v0 + v, left, x);
        load_four(Dp + (int64_t)k * p.V + v0 + v, left, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) sd = fmaf(x[e], y[e], sd);
        L.a.s.put4(k, v, floatx4{x[0], x[1], x[2], x[3]});
        L.a.d.put4(k, v, floatx4{y[0], y[1], y[2], y[3]});
      }
      for (int i = threadIdx.x; i < kC * 8; i += kThreads) {
        const int j = i / 8, v = i % 8 * 4;
        float x[4];
        load_four(Up + (int64_t)j * p.V + v0 + v, p.V - v0 - v, x);
        L.a.u.put4(j, v, floatx4{x[0], x[1], x[2], x[3]});
      }
      __syncthreads();
      const int v = v0 + g4 * 8, left = p.V - v;
      float x[8], y[8];
      const Wide<E, 1> dof = load_exact(p.dy.row(b, t0 + row, h) + v, row < live ? left : 0);
      load_eight(p.v.row(b, t0 + row, h) + v, row < live ? left : 0, x);
      load_eight(Rp + (int64_t)row * p.V + v, left, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) rv = fmaf(x[i], y[i], rv);
      const Wide<E, kGradParts> rf = wide<E, kGradParts>(y);
      load_eight(Up + (int64_t)row * p.V + v, left, x);
      const Wide<E, kGradParts> uf = wide<E, kGradParts>(x);
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        Wide<E, kGradParts> o = L.a.s.frag(16 * k + l16, g4 * 8);
        mma(dq[k], dof, o);
        mma(z[k], rf, o);
        o = L.a.d.frag(16 * k + l16, g4 * 8);
        mma(wr[k], uf, o);
      }
#pragma unroll
      for (int tj = 0; tj < 4; ++tj)
        if (tj <= w) {
          const Wide<E, kGradParts> o = L.a.u.frag(16 * tj + l16, g4 * 8);
          mma(dm[tj], dof, o);
          mma(da[tj], rf, o);
        }
    }
    const floatx4 beta = *reinterpret_cast<const floatx4*>(vec + kBeta * kC + rows);
    const floatx4 into = *reinterpret_cast<const floatx4*>(vec + kInto * kC + rows);
    const floatx4 rest = *reinterpret_cast<const floatx4*>(vec + kRest * kC + rows);
    rootk = *reinterpret_cast<const floatx4*>(vec + kRootK * kC + rows);
    rootq = *reinterpret_cast<const floatx4*>(vec + kRootQ * kC + rows) * p.scale;
    // (keys' and queries' columns, four frames each)
    auto k4 = [&](int k) { return floatx4{L.kt.at(k, rows), L.kt.at(k, rows + 1), L.kt.at(k, rows + 2), L.kt.at(k, rows + 3)}; };
    auto q4 = [&](int k) { return floatx4{L.qt.at(k, rows), L.qt.at(k, rows + 1), L.qt.at(k, rows + 2), L.qt.at(k, rows + 3)}; };
    floatx4 written = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      dq[k] *= into;
      z[k] *= -into;
      wr[k] *= rest;
      written += k4(16 * k + l16) * wr[k];
    }
    // over the chunk's end: what the entering state and the chunk's writes have there
    float over = sd * vec[kInto * kC + kC - 1];
    {
      const floatx4 t = written * rootk;
      over += (t[0] + t[1]) + (t[2] + t[3]);
      over = wave_sum(over);
      rv += __shfl_xor(rv, 16, 64), rv += __shfl_xor(rv, 32, 64);
      if (g4 == 0) L.db[row] = rv;
      if (lane == 0) L.red[w][0] = over;
    }
    // the two triangular matrices, one after the other, by rows and by columns
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int tj = 0; tj < 4; ++tj) {
        if (tj > w + 1 || (tj == w + 1 && (w & 1))) continue;
        const int j = 16 * tj + l16;
        const float rootj = vec[kRootK * kC + j];
        floatx4 by_row, by_col;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = rows + e;
          const float d = (which ? j < i : j <= i) && tj <= w ? exp_accurate((L.gh[i] - L.gh[j]) + (L.gl[i] - L.gl[j])) : 0.f;
          const float x = (which ? -da[tj][e] : dm[tj][e]) * d;
          by_row[e] = x * rootj;
          by_col[e] = x * (which ? beta[e] * rootk[e] : rootq[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) L.b.n.put(rows + e, j, by_row[e]);
        L.b.nt.put4(j, rows, by_col);
      }
      __syncthreads();
      for (int f = 0; f <= w / 2; ++f) {
        const int col = f * 32 + g4 * 8;
        const Wide<E, kGradParts> o = L.b.n.frag(row, col);
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          if (which) mma(z[k], o, L.kt.frag(16 * k + l16, col));
          else mma(dq[k], o, L.kt.frag(16 * k + l16, col));
        }
      }
      for (int f = w / 2; f < 2; ++f) {
        const int col = f * 32 + g4 * 8;
        const Wide<E, kGradParts> o = L.b.nt.frag(row, col);
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          if (which) mma(wr[k], o, L.kt.frag(16 * k + l16, col));
          else mma(wr[k], o, L.qt.frag(16 * k + l16, col));
        }
      }
    }
    floatx4 q = {0, 0, 0, 0}, kr = {0, 0, 0, 0}, kw = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const floatx4 kk = k4(16 * k + l16);
      q += q4(16 * k + l16) * dq[k];
      kr += kk * z[k];
      kw += kk * wr[k];
      DQ[k] += dq[k];
      DK[k] += beta * z[k] + wr[k];
    }
    q = row_total(q) * rootq, kr = row_total(kr) * rootk, kw = row_total(kw) * rootk;
    qdq += q, kdk += beta * kr + kw;
    if (l16 == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        L.at[rows + e] = q[e] + beta[e] * kr[e] - kw[e];
        L.db[rows + e] += kr[e];
      }
    }
    __syncthreads();
    if (w == 0) {
      float a = L.at[lane];
#pragma unroll
      for (int k = 1; k < 64; k *= 2) {
        const float o = __shfl_down(a, k, 64);
        if (lane + k < 64) a += o;
      }
      a += (L.red[0][0] + L.red[1][0]) + (L.red[2][0] + L.red[3][0]);
      const int t = t0 + lane;
      if (t < p.T) {
        const bool on = lane < live;
        p.dg.p[b * p.dg.b + t * p.dg.t + h] = on ? a : 0.f;
        p.dbeta.p[b * p.dbeta.b + t * p.dbeta.t + h] = on ? L.db[lane] : 0.f;
      }
    }
  }
  // through the scales and the norms: x^ = x r, r = 1 / sqrt(|x|^2 + eps)
  floatx4 backq = {0, 0, 0, 0}, backk = {0, 0, 0, 0};
  if (p.normalize) {
    const floatx4 r = rootq * (1.f / p.scale);
    backq = qdq * r * r, backk = kdk * rootk * rootk;
  }
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    const int col = 16 * k + l16;
    if (col >= p.K) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = rows + e;
      if (t0 + i >= p.T) continue;
      const bool on = i < live;
      p.dq.row(b, t0 + i, hk)[col] = from_f32<E>(on ? fmaf(-L.qt.at(col, i), backq[e], rootq[e] * DQ[k][e]) : 0.f);
      p.dk.row(b, t0 + i, hk)[col] = from_f32<E>(on ? fmaf(-L.kt.at(col, i), backk[e], rootk[e] * DK[k][e]) : 0.f);
    }
  }
}

// --------------------------------------------------------------- few frames
// Frame by frame: 32 values of one head a workgroup, a thread holds four of
// them for KP / 32 of the keys' channels.
template <class E, int KP>
__global__ __launch_bounds__(kThreads) void k_delta_step(DeltaP<E> p) {
  constexpr int NR = KP / 32;
  __shared__ float kq[2][2][KP], red[2][4][8][12];
  const int nvb = (p.V + 31) / 32, vb = blockIdx.x % (uint32_t)nvb, bh = blockIdx.x / (uint32_t)nvb;
  const int b = bh / p.H, h = bh % p.H, hk = h / p.shared, live = live_of(p.lengths, b, p.T);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l8 = lane & 7, rt = threadIdx.x >> 3;
  const int v = vb * 32 + l8 * 4, left = p.V - v;
  float S[NR][4];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int k = rt + 32 * i;
    load_four(p.state + ((int64_t)bh * p.K + k) * p.V + v, p.state && k < p.K ? left : 0, S[i]);
  }
  for (int t = 0; t < p.T; ++t) {
    E* yp = p.y.row(b, t, h) + v;
    if (t >= live) {
      if (rt == 0) {
        const float none[4] = {0.f, 0.f, 0.f, 0.f};
        store_four(yp, left, none);
      }
      continue;
    }
    const int at = t & 1;
    if (threadIdx.x < KP) {
      const int k = threadIdx.x;
      kq[at][0][k] = k < p.K ? to_f32(p.k.row(b, t, hk)[k]) : 0.f;
      kq[at][1][k] = k < p.K ? to_f32(p.q.row(b, t, hk)[k]) : 0.f;
    }
    const float beta = p.beta.p[b * p.beta.b + t * p.beta.t + h];
    float g = p.g.p[b * p.g.b + t * p.g.t + h], val[4];
    g = g < -128.f ? -128.f : g;
    load_four(p.v.row(b, t, h) + v, left, val);
    __syncthreads();
    // k.S, q.S, k.q, k.k and q.q in one go
    float o[11] = {};
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const float k = kq[at][0][rt + 32 * i], q = kq[at][1][rt + 32 * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(k, S[i][e], o[e]), o[4 + e] = fmaf(q, S[i][e], o[4 + e]);
      o[8] = fmaf(k, q, o[8]), o[9] = fmaf(k, k, o[9]), o[10] = fmaf(q, q, o[10]);
    }
#pragma unroll
    for (int e = 0; e < 11; ++e) {
#pragma unroll
      for (int k = 8; k < 64; k *= 2) o[e] += __shfl_xor(o[e], k, 64);
      if (lane < 8) red[at][w][l8][e] = o[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 11; ++e) o[e] = (red[at][0][l8][e] + red[at][1][l8][e]) + (red[at][2][l8][e] + red[at][3][l8][e]);
    const float rk = p.normalize ? __builtin_amdgcn_rsqf(o[9] + kUnitEps) : 1.f;
    const float rq = (p.normalize ? __builtin_amdgcn_rsqf(o[10] + kUnitEps) : 1.f) * p.scale;
    const float decay = exp_accurate(g);
    float u[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u[e] = beta * fmaf(-decay * rk, o[e], val[e]);
      y[e] = rq * fmaf(o[8] * rk, u[e], decay * o[4 + e]);
      u[e] *= rk;
    }
    if (rt == 0) store_four(yp, left, y);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const float k = kq[at][0][rt + 32 * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) S[i][e] = fmaf(k, u[e], decay * S[i][e]);
    }
  }
  if (!p.state_out) return;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int k = rt + 32 * i;
    store_four(p.state_out + ((int64_t)bh * p.K + k) * p.V + v, k < p.K ? left : 0, S[i]);
  }
}

// ------------------------------------------------------------------ launches
constexpr int64_t kMaxK = 128, kMaxV = 1024;
constexpr int kVB = 32;

struct Plan {
  int64_t chunks, nvb, segs, per;
  int64_t X, M, vec, S, dS, U, dR, ends, gends, bytes;  // places in the workspace
};

Plan plan_of(const dgen_hip_delta& a, bool backward) {
  Plan o = {};
  if ((!backward && a.T <= kStepFrames) || a.batch == 0) return o;
  const int64_t bh = a.batch * a.heads;
  o.chunks = (a.T + kC - 1) / kC;
  o.nvb = (a.V + kVB - 1) / kVB;
  o.segs = 1;
  if (bh * o.nvb < 256) {
    // (a segment costs its chunks twice, and a step of the carry)
    o.segs = std::min<int64_t>((512 + bh * o.nvb - 1) / (bh * o.nvb), o.chunks / 8);
    if (o.segs < 4) o.segs = 1;
  }
  o.per = (o.chunks + o.segs - 1) / o.segs;
  o.segs = (o.chunks + o.per - 1) / o.per;
  int64_t at = 0;
  auto take = [&](int64_t floats) {
    const int64_t p = at;
    at += align256(floats * 4);
    return p;
  };
  const int64_t n = bh * o.chunks;
  o.X = take(n * kC * kC);
  o.M = take(n * kC * kC);
  o.vec = take(n * kVecs * kC);
  if (backward) {
    o.S = take(n * a.K * a.V);
    o.dS = take(n * a.K * a.V);
    o.U = take(n * kC * a.V);
    o.dR = take(n * kC * a.V);
  }
  if (o.segs > 1) {
    o.ends = take(bh * o.segs * a.K * (a.V + a.K));
    if (backward) o.gends = take(bh * o.segs * a.K * a.V);
  }
  o.bytes = at;
  return o;
}

template <class E, int KP>
void delta_launch(const dgen_hip_delta& a, bool backward, hipStream_t st) {
  const Plan o = plan_of(a, backward);
  DeltaP<E> p;
  auto in = [](const dgen_hip_heads& h) { return Heads<const E>{(const E*)h.data, h.stride_b, h.stride_t, h.stride_h}; };
  auto out = [](const dgen_hip_heads& h) { return Heads<E>{(E*)h.data, h.stride_b, h.stride_t, h.stride_h}; };
  auto gates = [](const dgen_hip_seq& s) { return Gates{(float*)s.data, s.stride_b, s.stride_t}; };
  p.q = in(a.q), p.k = in(a.k), p.v = in(a.v), p.dy = in(a.dy);
  p.y = out(a.y), p.dq = out(a.dq), p.dk = out(a.dk), p.dv = out(a.dv);
  p.g = gates(a.g), p.beta = gates(a.beta), p.dg = gates(a.dg), p.dbeta = gates(a.dbeta);
  p.lengths = a.lengths, p.state = a.state, p.state_out = a.state_out;
  p.scale = a.scale, p.normalize = a.normalize;
  p.B = (int)a.batch, p.T = (int)a.T, p.H = (int)a.heads, p.shared = (int)(a.heads / a.key_heads), p.K = (int)a.K, p.V = (int)a.V;
  p.chunks = (int)o.chunks, p.nvb = (int)o.nvb, p.segs = (int)o.segs, p.per = (int)o.per;
  auto at = [&](int64_t off) { return (float*)((char*)a.workspace + off); };
  p.X = at(o.X), p.M = at(o.M), p.vec = at(o.vec), p.S = at(o.S), p.dS = at(o.dS), p.U = at(o.U), p.dR = at(o.dR);
  p.ends = at(o.ends), p.gends = at(o.gends);
  const int64_t bh = a.batch * a.heads;
  auto grid = [](int64_t n) { return dim3((unsigned)n); };
  if (!backward && a.T <= kStepFrames) {
    k_delta_step<E, KP><<<grid(bh * ((a.V + 31) / 32)), kThreads, 0, st>>>(p);
    return;
  }
  k_delta_prepare<E, KP><<<grid(bh * o.chunks), kThreads, 0, st>>>(p);
  const int64_t blocks = bh * o.nvb * o.segs, carry = bh * ((a.V + 31) / 32);
  if (o.segs > 1) {
    k_delta_chain<E, KP, kVB, kEnds><<<grid(bh * o.segs * (o.nvb + (a.K + kVB - 1) / kVB)), kThreads, 0, st>>>(p);
    k_delta_carry<E, KP, false><<<grid(carry), kThreads, 0, st>>>(p);
  }
  if (!backward) {
    k_delta_chain<E, KP, kVB, kOut><<<grid(blocks), kThreads, 0, st>>>(p);
    return;
  }
  k_delta_chain<E, KP, kVB, kKeep><<<grid(blocks), kThreads, 0, st>>>(p);
  if (o.segs > 1) {
    k_delta_back<E, KP, kVB, kEnds><<<grid(blocks), kThreads, 0, st>>>(p);
    k_delta_carry<E, KP, true><<<grid(carry), kThreads, 0, st>>>(p);
  }
  k_delta_back<E, KP, kVB, kKeep><<<grid(blocks), kThreads, 0, st>>>(p);
  k_delta_grads<E, KP><<<grid(a.batch * a.key_heads * o.chunks), kThreads, 0, st>>>(p);
}

template <class E>
void delta_width(const dgen_hip_delta& a, bool backward, hipStream_t st) {
  if (a.K <= 32) delta_launch<E, 32>(a, backward, st);
  else if (a.K <= 64) delta_launch<E, 64>(a, backward, st);
  else delta_launch<E, 128>(a, backward, st);
}

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

int64_t delta_workspace(const dgen_hip_delta& a, bool backward) { return plan_of(a, backward).bytes; }

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
  const Plan o = plan_of(a, backward);
  // (a launch takes fewer than 2^32 threads)
  DGEN_REQUIRE(bh * std::max<int64_t>(o.chunks, o.segs * (o.nvb + 4)) < int64_t(1) << 23 && bh < int64_t(1) << 18,
               "%s: %lld sequences and heads of %lld frames are too many for one call", what, (long long)bh, (long long)a.T);
  const bool empty = a.batch == 0;
  auto readable = [&](const dgen_hip_heads& h) { return (h.data || empty) && h.stride_b >= 0 && h.stride_t >= 0 && h.stride_h >= 0; };
  auto writable = [&](const dgen_hip_heads& h, int64_t heads, int64_t n) {
    return (h.data || empty) && h.stride_b >= 0 && h.stride_t >= 0 && h.stride_h >= 0 &&
           heads_writable(h.stride_b, h.stride_t, h.stride_h, a.batch, a.T, heads, n);
  };
  DGEN_REQUIRE(readable(a.q) && readable(a.k) && readable(a.v), "%s: q, k or v: null, or a negative stride", what);
  DGEN_REQUIRE(((a.g.data && a.beta.data) || empty) && seq_readable(a.g) && seq_readable(a.beta), "%s: g or beta: null, or a negative stride",
               what);
  if (!backward) {
    DGEN_REQUIRE(writable(a.y, a.heads, a.V), "%s: y: null, or overlapping", what);
  } else {
    DGEN_REQUIRE(readable(a.dy), "%s: dy: null, or a negative stride", what);
    DGEN_REQUIRE(writable(a.dq, a.key_heads, a.K) && writable(a.dk, a.key_heads, a.K) && writable(a.dv, a.heads, a.V),
                 "%s: dq, dk or dv: null, or overlapping", what);
    DGEN_REQUIRE(((a.dg.data && a.dbeta.data) || empty) && seq_writable(a.dg, a.batch, a.T, a.heads) &&
                     seq_writable(a.dbeta, a.batch, a.T, a.heads),
                 "%s: dg or dbeta: null, or overlapping", what);
  }
  DGEN_REQUIRE(o.bytes == 0 || (a.workspace && a.workspace_bytes >= (uint64_t)o.bytes),
               "%s: workspace of %llu bytes, %lld needed", what, (unsigned long long)a.workspace_bytes, (long long)o.bytes);
  if (dry || empty) return 0;
  a.type == DGEN_HIP_BF16 ? delta_width<bf16>(a, backward, st) : delta_width<float>(a, backward, st);
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
