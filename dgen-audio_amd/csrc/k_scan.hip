// Selective state space scan, forward and backward.
//
// Per sequence and channel, N states with decays that depend on the input:
// h[t][n] = exp(step[t] A[n]) h[t-1][n] + step[t] x[t] B[t][n], y = C.h.  Four
// neighbouring lanes share a channel and hold N/4 states each (padded by states
// that stay 0), so a wave has 16 channels and a workgroup of four waves 64.  The
// four lanes take four frames at a time: each evaluates softplus, gate and
// loads of one of the four, and the others read its step by a quad
// permutation; y is summed over the quad the same way.  B and C, which all
// channels share, go through LDS.  What bounds it is the vector unit: per
// (frame, channel, state) one exponential (quarter rate) and four fp32
// operations forward, about four times that backward.
//
// Where the sequences and channels alone do not fill the chip, time is cut
// into chunks: the chunks' end states from zero and their summed steps (which
// give the decay over a chunk, exp(A sum step)), then the states that enter
// each chunk, then the chunks again from those.  The adjoint g[t] = C[t] dy[t] +
// exp(step[t+1] A) g[t+1] is cut in the same way.
//
// The backward pass first runs a chunk forward and stores the state before
// every tile of 16 frames, then takes the tiles from the last: a tile's
// states (kept in LDS) and decays (in registers) are formed again, and the
// adjoint steps down through them.  Sums over channels (gradients of B and C) go over the wave's
// 16 channels in registers, over the four waves in LDS, and over workgroups in
// a fixed order afterwards; no atomics.
//
// Measured, bf16, 32 x 1000 x 1024 x 16: forward in one piece 214 us, backward
// 672 us and 21 for the sums over workgroups (the vector unit issues in 75 to
// 80 % of the cycles; two workgroups a CU by registers and LDS); with 12 states
// 215, 673 and 18, as the padded ones are computed too.  fp32, 1 x 65536 x 64 x
// 16 in 512 chunks: ends 22 us, carry 10, replay 31.  fp32, one frame of 32 x
// 1024 x 16: 8 us, for which the tile's loads are issued as for 32 frames.
#include "seq.h"

namespace dgen {

namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kChannels = 16 * kWaves;
constexpr int kTile = 32;  // frames staged at a time, forward
constexpr float kLog2e = 1.4426950408889634f;

// Frames of a backward tile: its decays are S registers a frame, its states S
// LDS words a lane and frame (64 KB a workgroup at S = 4, two workgroups a CU;
// tiles of 8 frames, 32 x 1000 x 1024 x 16 bf16: 760 us for 712).
template <int S>
constexpr int bwd_tile() { return S <= 4 ? 16 : 64 / S; }

template <class E>
struct Rows {  // [batch][time][.], contiguous last axis
  E* p;
  int64_t b;
  int t;
};

template <class E>
struct ScanP {
  Rows<const E> x, dt, z, B, C, dy;
  Rows<E> y, dx, ddt, dz;
  const float *A, *skip, *bias, *state;
  const int32_t* lengths;
  float* state_out;
  int T, D, N, chunk, chunks, nd, batch;  // nd: blocks of 64 channels
  bool walk;                              // the chunks join their entering states themselves
  float* sums;                         // [batch][chunks][D]: summed steps
  float* ends;                         // [batch][chunks][D][NP]: end states, then the states entering
  float* gends;                        // the same of the adjoint
  float* ckpt;                         // [batch][tiles][D][NP]: states before each backward tile
  float* shared;                       // [nd][batch][T][2 N]: dB | dC per block of channels
  float* parts;                        // [batch chunks][D (N + 2)]: dA | dskip | ddt_bias
};

__device__ __forceinline__ int live_of(const int32_t* __restrict__ lengths, int b, int T) {
  if (!lengths) return T;
  const int n = lengths[b];
  return n < 0 ? 0 : n < T ? n : T;
}

// The value that lane J of each quad holds.
template <int J>
__device__ __forceinline__ float quad(float v) { return dpp<J * 0x55>(v); }
// Sum over the quad, in every lane of it.
__device__ __forceinline__ float quad_sum(float v) {
  v += dpp<0xB1>(v);
  return v + dpp<0x4E>(v);
}

// Sums over the quad of four values: lane q of each quad gets that of v[q].
__device__ __forceinline__ float quad_sums(const float (&v)[4], bool odd, bool upper) {
  const float a = (odd ? v[1] : v[0]) + dpp<0xB1>(odd ? v[0] : v[1]);
  const float b = (odd ? v[3] : v[2]) + dpp<0xB1>(odd ? v[2] : v[3]);
  return (upper ? b : a) + dpp<0x4E>(upper ? a : b);
}

template <int S>
__device__ __forceinline__ void read_states(const float* __restrict__ p, float (&o)[S]) {
  if constexpr (S % 4 == 0) {
#pragma unroll
    for (int s = 0; s < S; s += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + s);
      o[s] = v.x, o[s + 1] = v.y, o[s + 2] = v.z, o[s + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int s = 0; s < S; ++s) o[s] = p[s];
  }
}

template <int S>
__device__ __forceinline__ void write_states(float* __restrict__ p, const float (&v)[S]) {
  if constexpr (S % 4 == 0) {
#pragma unroll
    for (int s = 0; s < S; s += 4) *reinterpret_cast<float4*>(p + s) = make_float4(v[s], v[s + 1], v[s + 2], v[s + 3]);
  } else {
#pragma unroll
    for (int s = 0; s < S; ++s) p[s] = v[s];
  }
}

// A workgroup's place: channel block, chunk, sequence.
struct Place {
  int b, c, d, lane, wave, q;
  bool on;
  int begin, end, live;  // the chunk's frames, and how far they are inside the sequence
  int frames;            // the sequence's
};
template <class E>
__device__ __forceinline__ Place place_of(const ScanP<E>& p) {
  Place w;
  const uint32_t nd = (uint32_t)p.nd, nc = (uint32_t)p.chunks, i = blockIdx.x / nd;
  w.lane = threadIdx.x & 63;
  w.wave = threadIdx.x >> 6;
  w.q = w.lane & 3;
  w.d = (int)(blockIdx.x % nd) * kChannels + w.wave * 16 + (w.lane >> 2);
  w.on = w.d < p.D;
  w.c = i % nc;
  w.b = i / nc;
  w.begin = w.c * p.chunk;
  w.end = w.begin + p.chunk < p.T ? w.begin + p.chunk : p.T;
  w.frames = live_of(p.lengths, w.b, p.T);
  w.live = w.frames < w.end ? w.frames : w.end;
  return w;
}

// The tile's rows of B and C that a thread carries from memory to LDS:
// element i + 256 k of [FRAMES][2][NP].
template <class E, int FRAMES, int NP>
struct Shared {
  static constexpr int K = (FRAMES * 2 * NP + kThreads - 1) / kThreads;
  float v[K];
  __device__ __forceinline__ void load(const ScanP<E>& p, const Place& w, int t0) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = threadIdx.x + k * kThreads, row = i / (2 * NP), col = i % (2 * NP), n = col % NP;
      // (without a branch: what lies outside is loaded from inside and zeroed)
      const int left = w.live - 1 - t0;
      const bool in = row <= left && n < p.N;
      const uint32_t r = row < left ? row : left, c = n < p.N ? n : 0;
      const Rows<const E>& m = col < NP ? p.B : p.C;
      const float x = to_f32((m.p + w.b * m.b + (int64_t)t0 * m.t)[r * (uint32_t)m.t + c]);
      v[k] = in ? x : 0.f;
    }
  }
  __device__ __forceinline__ void store(float* lds) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = threadIdx.x + k * kThreads;
      if (i < FRAMES * 2 * NP) lds[i] = v[k];
    }
  }
};

// One lane's place in a tile of a sequence tensor: its channel and the first
// of its frames, as an offset from the tile's first frame (the host checks
// that it fits).  Frames 4 g + q of the tile are loaded for g < G without any
// branch: past the sequence's end the last frame is loaded again, and lanes
// past the last channel take that one; both are left out by their steps and
// gradients being set to 0.
template <class E>
struct Lane {
  const E* seq;  // the sequence's first frame
  int t;         // elements between frames
  uint32_t at;   // q t + d
  uint32_t d;
  __device__ __forceinline__ Lane(const Rows<const E>& m, const Place& w, int D) {
    seq = m.p + w.b * m.b;
    t = m.t;
    d = (uint32_t)(w.on ? w.d : D - 1);
    at = (uint32_t)w.q * (uint32_t)m.t + d;
  }
  template <int G>
  __device__ __forceinline__ void load(const Place& w, int t0, float (&o)[G]) const {
    const E* p = seq + (int64_t)t0 * t;
    if (t0 + 4 * G <= w.live) {
#pragma unroll
      for (int g = 0; g < G; ++g) o[g] = to_f32((p + (int64_t)(4 * g) * t)[at]);
    } else {
      const uint32_t last = (uint32_t)(w.live - 1 - t0);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t f = 4 * g + w.q;
        o[g] = to_f32(p[(f < last ? f : last) * (uint32_t)t + d]);
      }
    }
  }
};

constexpr int kWalkStates = 4;  // of a lane, at most
// Joins `count` chunks' end states to h, from chunk `first` on in steps of
// `dir`: h = exp(A sum) h + end.  a2: A log2(e).  The loads of 16 chunks
// are in flight at once.
template <class E, int S>
__device__ __forceinline__ void join_chunks(const ScanP<E>& p, const Place& w, const float* __restrict__ ends, int first,
                                            int count, int dir, const float (&a2)[S], float (&h)[S]) {
  constexpr int K = 16;
  const int64_t row = (int64_t)w.b * p.chunks, d = w.on ? w.d : p.D - 1;
  for (int c0 = 0; c0 < count; c0 += K) {
    float sum[K], end[K][S];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = c0 + k < count ? c0 + k : count - 1;
      const int64_t at = (row + first + dir * c) * p.D + d;
      sum[k] = p.sums[at];
      read_states<S>(ends + at * (4 * S) + w.q * S, end[k]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (c0 + k < count)
#pragma unroll
        for (int s = 0; s < S; ++s) h[s] = fmaf(__builtin_amdgcn_exp2f(sum[k] * a2[s]), h[s], end[k][s]);
  }
}

enum Mode { kWhole, kSummary, kReplay, kSummaryBoth };

// What a padded state is fed: 0, as B = 0 does not keep its channel's infinity
// out.  (Its decay is that of A = -1.)  Where whole lanes are padded, that is
// one select a frame, else one a state: calls of 32 x 1000 x 1024 bf16 forward,
// N = 16, 12 and 13: 210, 212 and 225 us (12 and 13 without: 209 and 214).
enum Pad { kNoPad, kLanes, kStates };
template <int PAD, int S>
__device__ __forceinline__ float fed(const bool (&own)[S], int s, float v) {
  return PAD == kNoPad || own[PAD == kLanes ? 0 : s] ? v : 0.f;
}

// Forward: kWhole (one chunk: state to state_out), kReplay (from the state
// that enters the chunk); kSummary: end state from zero and summed steps;
// kSummaryBoth: the adjoint's too, accumulated forwards with the running
// product of decays.
template <class E, int S, int MODE, int PAD>
__global__ __launch_bounds__(kThreads) void k_scan(ScanP<E> p) {
  constexpr int NP = 4 * S, G = kTile / 4;
  constexpr bool OUT = MODE == kWhole || MODE == kReplay, ADJ = MODE == kSummaryBoth;
  __shared__ __align__(16) float bc[2][kTile * 2 * NP];
  const Place w = place_of(p);
  // Where the chunks join their states themselves nobody needs the last one's
  // end, and its place takes the state before the first, which the replay may
  // overwrite (state_out) before all of its workgroups have read it.
  const bool walk = S <= kWalkStates && p.walk, copy = MODE == kSummary && walk && w.c == p.chunks - 1;
  if (!OUT && w.begin >= w.live && !copy) return;  // a chunk past the sequence is left out

  float h[S], a2[S], prod[S], adj[S];
  bool own[S];  // not a padded state
  const float bias = p.bias && w.on ? p.bias[w.d] : 0.f, skip = p.skip && w.on ? p.skip[w.d] : 0.f;
  const int64_t at = ((int64_t)(w.b * p.chunks + w.c) * p.D + w.d) * NP + w.q * S;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int n = w.q * S + s;
    own[s] = n < p.N;
    const bool real = w.on && own[s];
    a2[s] = real ? p.A[(int64_t)w.d * p.N + n] * kLog2e : -kLog2e;
    h[s] = 0.f;
    if ((MODE == kWhole || copy) && p.state && real) h[s] = p.state[((int64_t)w.b * p.D + w.d) * p.N + n];
    prod[s] = 1.f;
    adj[s] = 0.f;
  }
  if (copy) {
    if (w.on) write_states<S>(p.ends + at, h);
    return;
  }
  if (MODE == kReplay && walk) {
    if (w.on) read_states<S>(p.ends + ((int64_t)(w.b * p.chunks + p.chunks - 1) * p.D + w.d) * NP + w.q * S, h);
    if (w.begin < w.live) join_chunks<E, S>(p, w, p.ends, 0, w.c, 1, a2, h);
  } else if (MODE == kReplay && w.on) {
    read_states<S>(p.ends + at, h);
  }

  const bool odd = w.q & 1, upper = w.q & 2;
  float sum = 0.f;
  float x[G], dt[G], z[G], dy[G];
  Shared<E, kTile, NP> bcv;
  const Lane<E> lx(p.x, w, p.D), ldt(p.dt, w, p.D), lz(p.z, w, p.D), ldy(p.dy, w, p.D);
  auto fetch = [&](int t0) {
    bcv.load(p, w, t0);
    lx.load(w, t0, x);
    ldt.load(w, t0, dt);
    if ((OUT || ADJ) && p.z.p) lz.load(w, t0, z);
    if (ADJ) ldy.load(w, t0, dy);
  };
  if (w.begin < w.live) fetch(w.begin);
  E* const yrow = p.y.p + w.b * p.y.b;
  const uint32_t yat = (uint32_t)w.q * (uint32_t)p.y.t + (uint32_t)w.d;
  const bool whole = ((int)(blockIdx.x % (uint32_t)p.nd) + 1) * kChannels <= p.D;
  int buf = 0;
  for (int t0 = w.begin; t0 < w.live; t0 += kTile, buf ^= 1) {
    float* lds = bc[buf];
    bcv.store(lds);
    float cx[G], cdt[G], cz[G], cdy[G];
#pragma unroll
    for (int g = 0; g < G; ++g) cx[g] = x[g], cdt[g] = dt[g], cz[g] = z[g], cdy[g] = dy[g];
    __syncthreads();
    if (t0 + kTile < w.live) fetch(t0 + kTile);
    const int groups = w.live - t0 < kTile ? (w.live - t0 + 3) / 4 : G;
    auto group = [&](int g, auto wholec) {
      const int t = t0 + 4 * g + w.q;
      const bool ok = decltype(wholec)::value || (w.on && t < w.live);
      float slope;
      const float soft = softplus_accurate(cdt[g] + bias, slope);
      const float step = ok ? soft : 0.f, u = ok ? soft * cx[g] : 0.f;
      float gate = 1.f, up = 0.f;
      if ((OUT || ADJ) && p.z.p) gate = silu(cz[g]);
      if (ADJ) up = ok ? cdy[g] * gate : 0.f;
      if (!OUT) sum += step;
      float y4[4];
      auto frame = [&](auto jc) {
        constexpr int J = decltype(jc)::value;
        const float sj = quad<J>(step), uj = quad<J>(u), dj = ADJ ? quad<J>(up) : 0.f;
        const float* row = lds + (4 * g + J) * 2 * NP + w.q * S;
        float bv[S], cv[S], yj = 0.f;
        read_states<S>(row, bv);
        if (OUT || ADJ) read_states<S>(row + NP, cv);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float a = __builtin_amdgcn_exp2f(sj * a2[s]);
          h[s] = fmaf(a, h[s], fed<PAD>(own, s, uj) * bv[s]);
          if (OUT) yj = fmaf(cv[s], h[s], yj);
          if (ADJ) {
            prod[s] *= a;
            adj[s] = fmaf(prod[s] * cv[s], fed<PAD>(own, s, dj), adj[s]);
          }
        }
        y4[J] = yj;
      };
      frame(std::integral_constant<int, 0>{});
      frame(std::integral_constant<int, 1>{});
      frame(std::integral_constant<int, 2>{});
      frame(std::integral_constant<int, 3>{});
      const float y = OUT ? quad_sums(y4, odd, upper) : 0.f;
      const float through = p.skip ? cx[g] : 0.f;
      if (OUT && ok) (yrow + (int64_t)(t0 + 4 * g) * p.y.t)[yat] = from_f32<E>(fmaf(skip, through, y) * gate);
    };
    // a whole tile of whole channels in one piece, without a branch (but with
    // the adjoint's sums one piece takes too many registers)
    if (!ADJ && whole && w.live - t0 >= kTile) {
#pragma unroll
      for (int g = 0; g < G; ++g) group(g, std::true_type{});
    } else {
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (g < groups) group(g, std::false_type{});
    }
  }
  if (!w.on) return;
  if (OUT)
    for (int t = (w.live > w.begin ? w.live : w.begin) + w.q; t < w.end; t += 4)
      p.y.p[w.b * p.y.b + (int64_t)t * p.y.t + w.d] = from_f32<E>(0.f);
  // (of chunks, the one with the sequence's last frame)
  const bool last = MODE == kWhole || (walk && w.frames <= w.end && (w.begin < w.frames || w.c == 0));
  if (OUT && p.state_out && last) {
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (w.q * S + s < p.N) p.state_out[((int64_t)w.b * p.D + w.d) * p.N + w.q * S + s] = h[s];
  }
  if (!OUT) {
    write_states<S>(p.ends + at, h);
    if (ADJ) write_states<S>(p.gends + at, adj);
    sum = quad_sum(sum);
    if (w.q == 0) p.sums[(int64_t)(w.b * p.chunks + w.c) * p.D + w.d] = sum;
  }
}

constexpr int kMaxChunks = 512, kMaxRun = 16;  // chunks, and of a thread in the carry

// Of many chunks: states entering each, in place of the chunks' end states
// (reverse: the adjoints entering from the chunks after).  COLS states a workgroup, SEGS
// threads over the chunks: each joins its run of chunks, the runs are joined
// in LDS, and each walks its run again.
// The backward pass takes both directions in one launch: the second half of
// the grid is the adjoint's.
template <class E, int SEGS, int COLS>
__global__ __launch_bounds__(COLS * SEGS) void k_scan_carry(ScanP<E> p, int np) {
  __shared__ float rsum[SEGS][COLS + 1], rend[SEGS][COLS + 1];
  const int col = threadIdx.x % COLS, seg = threadIdx.x / COLS;
  const int64_t per = (int64_t)p.D * np, blocks = (per + COLS - 1) / COLS;
  const int row = (int)(blockIdx.x / blocks), b = row % p.batch;
  const bool reverse = row >= p.batch;
  float* const ends = reverse ? p.gends : p.ends;
  const int64_t j = (blockIdx.x % blocks) * COLS + col;
  const bool on = j < per;
  const int64_t d = on ? j / np : 0;
  const int n = on ? (int)(j % np) : 0;
  const bool real = on && n < p.N;
  const float a2 = real ? p.A[d * p.N + n] * kLog2e : -kLog2e;
  const int live = live_of(p.lengths, b, p.T), used = (live + p.chunk - 1) / p.chunk;
  const int run = (p.chunks + SEGS - 1) / SEGS, lo = seg * run, hi = lo + run < used ? lo + run : used;
  float* e = ends + (int64_t)b * p.chunks * per + j;
  const float* sm = p.sums + (int64_t)b * p.chunks * p.D + d;
  auto chunk = [&](int k) { return (int64_t)(reverse ? used - 1 - k : k); };  // k-th in walking order
  // the run in registers, loaded at once (past its end: its first chunk again)
  float rs[kMaxRun], re[kMaxRun];
#pragma unroll
  for (int i = 0; i < kMaxRun; i += 4)
    if (i < run)
#pragma unroll
      for (int k = i; k < i + 4; ++k) {
        const int64_t c = on && lo + k < hi ? chunk(lo + k) : 0;
        const float x = on ? sm[c * p.D] : 0.f, y = on ? e[c * per] : 0.f;
        rs[k] = lo + k < hi ? x : 0.f;
        re[k] = lo + k < hi ? y : 0.f;
      }
  float sum = 0.f, end = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxRun; i += 4)
    if (i < run)
#pragma unroll
      for (int k = i; k < i + 4; ++k) {
        // (step 0 and state 0 past the end: the decay is 1)
        end = fmaf(__builtin_amdgcn_exp2f(rs[k] * a2), end, re[k]);
        sum += rs[k];
      }
  rsum[seg][col] = sum;
  rend[seg][col] = end;
  float h = 0.f;
  if (!reverse && real && p.state) h = p.state[((int64_t)b * p.D + d) * p.N + n];
  __syncthreads();
  for (int k = 0; k < seg; ++k) h = fmaf(__builtin_amdgcn_exp2f(rsum[k][col] * a2), h, rend[k][col]);
  if (!on) return;
#pragma unroll
  for (int i = 0; i < kMaxRun; i += 4)
    if (i < run)
#pragma unroll
      for (int k = i; k < i + 4; ++k) {
        if (lo + k < hi) e[chunk(lo + k) * per] = h;
        h = fmaf(__builtin_amdgcn_exp2f(rs[k] * a2), h, re[k]);
      }
  // the thread past the last run has the state after all chunks
  if (!reverse && seg == SEGS - 1 && real && p.state_out) p.state_out[((int64_t)b * p.D + d) * p.N + n] = h;
}

// Sum over the wave's 16 channels (lane bits 2..5) of V values per lane, by
// exchange: after the half-wave and row swaps a lane holds a quarter of the
// values; those are summed over lane bits 2 and 3 by row rotations.  w[k] is
// value index 4 k + 2 (lane bit 4) + (lane bit 5) (V = 2: lane bit 5).
template <int V>
constexpr int kept() { return V >= 4 ? V / 4 : 1; }
template <int V>
__device__ __forceinline__ void channel_sum(const float (&v)[V], float (&w)[kept<V>()]) {
  float r[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) r[i] = swap_add32(v[2 * i], v[2 * i + 1]);
  if constexpr (V >= 4) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k) w[k] = swap_add16(r[2 * k], r[2 * k + 1]);
  } else {
    w[0] = swap_add16(r[0], r[0]);
  }
#pragma unroll
  for (int k = 0; k < kept<V>(); ++k) {
    w[k] += dpp<0x124>(w[k]);  // row_ror:4
    w[k] += dpp<0x128>(w[k]);  // row_ror:8
  }
}

template <class E, int S, int PAD>
__global__ __launch_bounds__(kThreads, S <= 4 ? 2 : 1) void k_scan_bwd(ScanP<E> p) {
  constexpr int NP = 4 * S, TL = bwd_tile<S>(), G = TL / 4;
  __shared__ __align__(16) float bc[2][TL * 2 * NP];
  __shared__ float red[TL][kWaves][2 * NP];
  // the tile's states before each frame, a lane's own
  __shared__ __align__(16) float hs[TL][kThreads][S];
  const Place w = place_of(p);
  const bool walk = S <= kWalkStates && p.walk;
  const int tiles_all = (p.T + TL - 1) / TL, tile0 = w.begin / TL;
  const int tiles = w.live > w.begin ? (w.live - w.begin + TL - 1) / TL : 0;

  float h[S], a[S], g[S], dA[S];
  bool own[S];
  const float bias = p.bias && w.on ? p.bias[w.d] : 0.f, skip = p.skip && w.on ? p.skip[w.d] : 0.f;
  const int64_t at = ((int64_t)(w.b * p.chunks + w.c) * p.D + w.d) * NP + w.q * S;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int n = w.q * S + s;
    own[s] = n < p.N;
    const bool real = w.on && own[s];
    a[s] = real ? p.A[(int64_t)w.d * p.N + n] : -1.f;
    h[s] = (p.chunks == 1 || walk) && p.state && real ? p.state[((int64_t)w.b * p.D + w.d) * p.N + n] : 0.f;
    g[s] = 0.f;
    dA[s] = 0.f;
  }
  if (walk && tiles > 0) {
    float a2[S];
#pragma unroll
    for (int s = 0; s < S; ++s) a2[s] = a[s] * kLog2e;
    const int used = (w.frames + p.chunk - 1) / p.chunk;
    join_chunks<E, S>(p, w, p.ends, 0, w.c, 1, a2, h);
    join_chunks<E, S>(p, w, p.gends, used - 1, used - 1 - w.c, -1, a2, g);
    if (!w.on) {
#pragma unroll
      for (int s = 0; s < S; ++s) h[s] = g[s] = 0.f;
    }
  } else if (p.chunks > 1 && tiles > 0 && w.on) {
    read_states<S>(p.ends + at, h);
    read_states<S>(p.gends + at, g);
  }
  const bool odd = w.q & 1, upper = w.q & 2;
  float dskip = 0.f, dbias = 0.f;
  // (lanes past the last channel read that one's states and store none)
  float* ck = p.ckpt + ((int64_t)(w.b * tiles_all + tile0) * p.D + (w.on ? w.d : p.D - 1)) * NP + w.q * S;
  Shared<E, TL, NP> bcv;
  const Lane<E> lx(p.x, w, p.D), ldt(p.dt, w, p.D), lz(p.z, w, p.D), ldy(p.dy, w, p.D);

  // forward over the chunk: the state before every tile
  {
    float x[G], dt[G];
    auto fetch = [&](int t0) {
      bcv.load(p, w, t0);
      lx.load(w, t0, x);
      ldt.load(w, t0, dt);
    };
    if (tiles > 0) fetch(w.begin);
    for (int i = 0; i < tiles; ++i) {
      if (w.on) write_states<S>(ck + (int64_t)i * p.D * NP, h);
      if (i + 1 == tiles) break;
      float* lds = bc[i & 1];
      bcv.store(lds);
      float cx[G], cdt[G];
#pragma unroll
      for (int k = 0; k < G; ++k) cx[k] = x[k], cdt[k] = dt[k];
      __syncthreads();
      fetch(w.begin + (i + 1) * TL);
#pragma unroll
      for (int k = 0; k < G; ++k) {
        float slope;
        // (every frame of a tile that another follows is inside the sequence)
        const float step = softplus_accurate(cdt[k] + bias, slope), u = step * cx[k], step2 = step * kLog2e;
        auto frame = [&](auto jc) {
          constexpr int J = decltype(jc)::value;
          const float sj = quad<J>(step2), uj = quad<J>(u);
          float bv[S];
          read_states<S>(lds + (4 * k + J) * 2 * NP + w.q * S, bv);
#pragma unroll
          for (int s = 0; s < S; ++s)
            h[s] = fmaf(__builtin_amdgcn_exp2f(sj * a[s]), h[s], fed<PAD>(own, s, uj) * bv[s]);
        };
        frame(std::integral_constant<int, 0>{});
        frame(std::integral_constant<int, 1>{});
        frame(std::integral_constant<int, 2>{});
        frame(std::integral_constant<int, 3>{});
      }
    }
    __syncthreads();
  }

  E *const dxr = p.dx.p + w.b * p.dx.b, *const ddtr = p.ddt.p + w.b * p.ddt.b, *const dzr = p.dz.p + w.b * p.dz.b;
  const uint32_t q = w.q, d = (uint32_t)w.d, dxat = q * (uint32_t)p.dx.t + d, ddtat = q * (uint32_t)p.ddt.t + d,
                 dzat = q * (uint32_t)p.dz.t + d;
  float x[G], dt[G], z[G], dy[G], hn[S];
  auto fetch = [&](int i) {
    const int t0 = w.begin + i * TL;
    bcv.load(p, w, t0);
    lx.load(w, t0, x);
    ldt.load(w, t0, dt);
    if (p.z.p) lz.load(w, t0, z);
    ldy.load(w, t0, dy);
    read_states<S>(ck + (int64_t)i * p.D * NP, hn);
  };
#pragma unroll
  for (int s = 0; s < S; ++s) hn[s] = 0.f;
  if (tiles > 0) fetch(tiles - 1);
  for (int i = tiles - 1; i >= 0; --i) {
    const int t0 = w.begin + i * TL;
    float* lds = bc[i & 1];
    bcv.store(lds);
    float cx[G], cz[G], cdy[G], step[G], slope[G], u[G], up[G], y[G];
#pragma unroll
    for (int s = 0; s < S; ++s) h[s] = w.on ? hn[s] : 0.f;
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const bool ok = w.on && t0 + 4 * k + w.q < w.live;
      cx[k] = x[k], cz[k] = z[k], cdy[k] = dy[k];
      step[k] = softplus_accurate(dt[k] + bias, slope[k]);
      u[k] = step[k] * cx[k];
      up[k] = p.z.p ? cdy[k] * silu(cz[k]) : cdy[k];
      if (!ok) step[k] = slope[k] = u[k] = up[k] = 0.f;
    }
    __syncthreads();
    if (i > 0) fetch(i - 1);

    // the tile's states and decays
    float as[TL][S];
#pragma unroll
    for (int k = 0; k < G; ++k) {
      float y4[4];
      const float step2 = step[k] * kLog2e;
      auto frame = [&](auto jc) {
        constexpr int J = decltype(jc)::value;
        const float sj = quad<J>(step2), uj = quad<J>(u[k]);
        const float* row = lds + (4 * k + J) * 2 * NP + w.q * S;
        float bv[S], cv[S], yj = 0.f;
        read_states<S>(row, bv);
        read_states<S>(row + NP, cv);
        write_states<S>(hs[4 * k + J][threadIdx.x], h);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const float e = __builtin_amdgcn_exp2f(sj * a[s]);
          as[4 * k + J][s] = e;
          h[s] = fmaf(e, h[s], fed<PAD>(own, s, uj) * bv[s]);
          yj = fmaf(cv[s], h[s], yj);
        }
        y4[J] = yj;
      };
      frame(std::integral_constant<int, 0>{});
      frame(std::integral_constant<int, 1>{});
      frame(std::integral_constant<int, 2>{});
      frame(std::integral_constant<int, 3>{});
      y[k] = quad_sums(y4, odd, upper);
    }
    // down through the tile: h is the state after the frame
#pragma unroll
    for (int k = G - 1; k >= 0; --k) {
      float gb4[4], ga4[4];
      auto frame = [&](auto jc) {
        constexpr int J = decltype(jc)::value;
        const int f = 4 * k + J;
        const float sj = quad<J>(step[k]), uj = quad<J>(u[k]), dj = quad<J>(up[k]);
        const float* row = lds + f * 2 * NP + w.q * S;
        float bv[S], cv[S], hb[S], v[2 * S], gbj = 0.f, gaj = 0.f;
        read_states<S>(row, bv);
        read_states<S>(row + NP, cv);
        read_states<S>(hs[f][threadIdx.x], hb);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          g[s] = fmaf(cv[s], fed<PAD>(own, s, dj), g[s]);
          v[s] = g[s] * uj;       // dB
          v[S + s] = h[s] * dj;   // dC
          gbj = fmaf(g[s], bv[s], gbj);
          g[s] *= as[f][s];       // the adjoint of the state before
          h[s] = hb[s];
          const float gh = g[s] * h[s];
          gaj = fmaf(gh, a[s], gaj);
          dA[s] = fmaf(gh, sj, dA[s]);
        }
        gb4[J] = gbj;
        ga4[J] = gaj;
        float sums[kept<2 * S>()];
        channel_sum<2 * S>(v, sums);
        if ((w.lane & 12) == 0) {
#pragma unroll
          for (int m = 0; m < kept<2 * S>(); ++m) {
            const int idx = S >= 2 ? 4 * m + 2 * ((w.lane >> 4) & 1) + (w.lane >> 5) : w.lane >> 5;
            red[f][w.wave][(idx / S) * NP + w.q * S + idx % S] = sums[m];
          }
        }
      };
      frame(std::integral_constant<int, 3>{});
      frame(std::integral_constant<int, 2>{});
      frame(std::integral_constant<int, 1>{});
      frame(std::integral_constant<int, 0>{});
      const float gb = quad_sums(gb4, odd, upper), ga = quad_sums(ga4, odd, upper);
      const int t = t0 + 4 * k + w.q;
      if (w.on && t < w.live) {
        const float draw = fmaf(gb, cx[k], ga) * slope[k];
        dbias += draw;
        dskip = fmaf(up[k], cx[k], dskip);
        const float dthrough = p.skip ? skip * up[k] : 0.f, through = p.skip ? cx[k] : 0.f;
        (dxr + (int64_t)(t0 + 4 * k) * p.dx.t)[dxat] = from_f32<E>(fmaf(step[k], gb, dthrough));
        (ddtr + (int64_t)(t0 + 4 * k) * p.ddt.t)[ddtat] = from_f32<E>(draw);
        if (p.z.p)
          (dzr + (int64_t)(t0 + 4 * k) * p.dz.t)[dzat] =
              from_f32<E>(cdy[k] * fmaf(skip, through, y[k]) * silu_grad(cz[k], sigmoid(cz[k])));
      }
    }
    __syncthreads();
    // dB | dC of the block's channels
    float* out = p.shared + ((int64_t)((int)(blockIdx.x % (uint32_t)p.nd) * p.batch + w.b) * p.T + t0) * 2 * p.N;
    for (int o = threadIdx.x; o < TL * 2 * NP; o += kThreads) {
      const int f = o / (2 * NP), col = o % (2 * NP), n = col % NP;
      if (t0 + f < w.live && n < p.N) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) t += red[f][k][col];
        out[f * 2 * p.N + (col < NP ? 0 : p.N) + n] = t;
      }
    }
  }
  if (!w.on) return;
  for (int t = (w.live > w.begin ? w.live : w.begin) + w.q; t < w.end; t += 4) {
    p.dx.p[w.b * p.dx.b + (int64_t)t * p.dx.t + w.d] = from_f32<E>(0.f);
    p.ddt.p[w.b * p.ddt.b + (int64_t)t * p.ddt.t + w.d] = from_f32<E>(0.f);
    if (p.z.p) p.dz.p[w.b * p.dz.b + (int64_t)t * p.dz.t + w.d] = from_f32<E>(0.f);
  }
  float* part = p.parts + (int64_t)(w.b * p.chunks + w.c) * p.D * (p.N + 2);
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (w.q * S + s < p.N) part[(int64_t)w.d * p.N + w.q * S + s] = dA[s];
  dskip = quad_sum(dskip);
  dbias = quad_sum(dbias);
  if (w.q == 0) {
    part[(int64_t)p.D * p.N + w.d] = dskip;
    part[(int64_t)p.D * (p.N + 1) + w.d] = dbias;
  }
}

// The last sums of the backward pass, in order: workgroups before `first` add
// the channel blocks' dB and dC, the others dA, dskip and ddt_bias.
template <class E>
__global__ __launch_bounds__(kSumThreads) void k_scan_join(ScanP<E> p, Rows<E> dB, Rows<E> dC, uint32_t first, SumOut o,
                                                           int64_t width) {
  __shared__ float red[kSumThreads / kSumCols][kSumCols + 1];
  if (blockIdx.x >= first) {
    sum_parts_block(p.parts, (int64_t)p.batch * p.chunks, o, width, blockIdx.x - first, red);
    return;
  }
  const int64_t N = p.N, T = p.T, total = p.batch * T * 2 * N, i = (int64_t)blockIdx.x * kSumThreads + threadIdx.x;
  if (i >= total) return;
  const int64_t row = i / (2 * N), col = i - row * 2 * N, b = row / T, t = row - b * T;
  float v = 0.f;
  if (t < live_of(p.lengths, (int)b, p.T))
    for (int64_t k = 0; k < p.nd; ++k) v += p.shared[k * total + i];
  const Rows<E>& m = col < N ? dB : dC;
  m.p[b * m.b + t * (int64_t)m.t + (col < N ? col : col - N)] = from_f32<E>(v);
}

struct ScanShape {
  int S;
  int64_t NP, nd, chunk, chunks;
  // workspace, in floats
  int64_t sums, ends, ckpt, shared, parts, total;
};

// Chunks: as many as give every CU four workgroups (backward, whose LDS and
// registers take no more, two), none shorter than 32 frames, and none where
// the sequences and channel blocks come near filling the chip alone, as a
// chunked pass evaluates every decay twice.  Measured, T = 1000, N = 16, bf16,
// whole / chunked: forward 128 blocks 138 / 95 us, 192 140 / 155, 256 141 /
// 168; backward 256 blocks 531 / 476 us, 320 670 / 745.
constexpr int64_t kFill = 1024, kFillBackward = 512, kAlone = 160, kAloneBackward = 288, kMinChunk = 32;
static_assert(2 * kAloneBackward * (kChannels * 64 / 32) * 1024 < int64_t(1) << 32, "threads of the largest carry");
// Chunks up to which, of up to 16 states, each joins the ones before it (and
// after it, backward) by itself; more go through k_scan_carry.  Calls, us,
// joined / carried: N = 16, forward 4 x 256 x 256 (8 chunks) 20 / 22, 2 x 1024
// x 128 (32) 19 / 22, 4 x 2048 x 64 (64) 22 / 22, 1 x 4096 x 64 (128) 28 / 21;
// backward 32 / 34, 33 / 34, 40 / 39, 43 / 36; N = 64, 32 chunks, 41 / 33 and
// 90 / 86.
constexpr int64_t kWalk = 32;

ScanShape scan_shape(const dgen_hip_scan& a, bool backward) {
  ScanShape s{};
  s.S = a.N <= 4 ? 1 : a.N <= 8 ? 2 : a.N <= 16 ? 4 : a.N <= 32 ? 8 : 16;
  s.NP = 4 * s.S;
  s.nd = (a.D + kChannels - 1) / kChannels;
  const int64_t blocks = std::max<int64_t>(1, a.batch * s.nd);
  int64_t chunks = 1;
  if (blocks < (backward ? kAloneBackward : kAlone))
    chunks = std::min({((backward ? kFillBackward : kFill) + blocks - 1) / blocks, (a.T + kMinChunk - 1) / kMinChunk, (int64_t)kMaxChunks});
  s.chunk = (a.T + chunks - 1) / chunks;
  s.chunk = (s.chunk + kTile - 1) / kTile * kTile;
  s.chunks = (a.T + s.chunk - 1) / s.chunk;
  const int64_t lanes = a.batch * a.D;
  auto up = [](int64_t n) { return (n + 63) & ~int64_t(63); };
  if (s.chunks > 1) {
    s.sums = up(s.chunks * lanes);
    s.ends = up(s.chunks * lanes * s.NP);
  }
  if (backward) {
    const int64_t tl = s.S <= 4 ? 16 : 64 / s.S;
    s.ckpt = up((a.T + tl - 1) / tl * lanes * s.NP);
    s.shared = up(s.nd * a.batch * a.T * 2 * a.N);
    s.parts = up(a.batch * s.chunks * a.D * (a.N + 2));
  }
  s.total = s.sums + s.ends * (backward ? 2 : 1) + s.ckpt + s.shared + s.parts;
  return s;
}

// (a single frame's stride says nothing)
template <class E>
Rows<E> rows_of(const dgen_hip_scan& a, const dgen_hip_seq& v) {
  return {(E*)v.data, v.stride_b, a.T > 1 ? (int)v.stride_t : 0};
}

template <class E, int S, int PAD>
void scan_launch(const dgen_hip_scan& a, bool backward, const ScanShape& s, hipStream_t st) {
  float* ws = (float*)a.workspace;
  auto in = [&](const dgen_hip_seq& v) { return rows_of<const E>(a, v); };
  auto out = [&](const dgen_hip_seq& v) { return rows_of<E>(a, v); };
  ScanP<E> p{};
  p.x = in(a.x), p.dt = in(a.dt), p.z = in(a.z), p.B = in(a.B), p.C = in(a.C);
  p.A = a.A, p.skip = a.skip, p.bias = a.dt_bias, p.state = a.state, p.lengths = a.lengths;
  p.T = (int)a.T, p.D = (int)a.D, p.N = (int)a.N, p.chunk = (int)s.chunk, p.chunks = (int)s.chunks, p.nd = (int)s.nd;
  p.batch = (int)a.batch;
  p.walk = S <= kWalkStates && s.chunks > 1 && s.chunks <= kWalk;
  p.sums = ws, p.ends = p.sums + s.sums, p.gends = p.ends + s.ends;
  if (!backward) p.y = out(a.y), p.state_out = a.state_out;
  const dim3 grid((unsigned)(s.nd * s.chunks * a.batch));
  // (threads a state by the number of chunks, for runs of up to 16)
  static_assert(64 / 4 <= kMaxRun && 256 / 16 <= kMaxRun && kMaxChunks / 32 <= kMaxRun, "runs of the carry");
  auto carry = [&]() {
    auto states = [&](int64_t cols) {
      return dim3((unsigned)((a.D * s.NP + cols - 1) / cols * a.batch * (backward ? 2 : 1)));
    };
    if (s.chunks <= 64) k_scan_carry<E, 4, 64><<<states(64), 256, 0, st>>>(p, (int)s.NP);
    else if (s.chunks <= 256) k_scan_carry<E, 16, 64><<<states(64), 1024, 0, st>>>(p, (int)s.NP);
    else k_scan_carry<E, 32, 32><<<states(32), 1024, 0, st>>>(p, (int)s.NP);
  };
  if (!backward) {
    if (s.chunks == 1) {
      k_scan<E, S, kWhole, PAD><<<grid, kThreads, 0, st>>>(p);
    } else {
      k_scan<E, S, kSummary, PAD><<<grid, kThreads, 0, st>>>(p);
      if (!p.walk) carry();
      k_scan<E, S, kReplay, PAD><<<grid, kThreads, 0, st>>>(p);
    }
    return;
  }
  p.dy = in(a.dy), p.dx = out(a.dx), p.ddt = out(a.ddt), p.dz = out(a.dz);
  p.ckpt = p.gends + s.ends, p.shared = p.ckpt + s.ckpt, p.parts = p.shared + s.shared;
  if (s.chunks > 1) {
    k_scan<E, S, kSummaryBoth, PAD><<<grid, kThreads, 0, st>>>(p);
    if (!p.walk) carry();
  }
  k_scan_bwd<E, S, PAD><<<grid, kThreads, 0, st>>>(p);
  const uint32_t first = (uint32_t)((a.batch * a.T * 2 * a.N + kSumThreads - 1) / kSumThreads);
  const int64_t width = a.D * (a.N + 2);
  k_scan_join<E><<<dim3(first + (unsigned)((width + kSumCols - 1) / kSumCols)), kSumThreads, 0, st>>>(
      p, out(a.dB), out(a.dC), first, {{a.dA, a.dskip, a.ddt_bias}, {a.D * a.N, a.D, a.D}}, width);
}

template <class E, int S>
void scan_padded(const dgen_hip_scan& a, bool backward, const ScanShape& s, hipStream_t st) {
  if (a.N == 4 * S) scan_launch<E, S, kNoPad>(a, backward, s, st);
  else if (a.N % S == 0) scan_launch<E, S, kLanes>(a, backward, s, st);
  else if constexpr (S > 1) scan_launch<E, S, kStates>(a, backward, s, st);
}

template <class E>
void scan_states(const dgen_hip_scan& a, bool backward, const ScanShape& s, hipStream_t st) {
  switch (s.S) {
    case 1: return scan_padded<E, 1>(a, backward, s, st);
    case 2: return scan_padded<E, 2>(a, backward, s, st);
    case 4: return scan_padded<E, 4>(a, backward, s, st);
    case 8: return scan_padded<E, 8>(a, backward, s, st);
    default: return scan_padded<E, 16>(a, backward, s, st);
  }
}

}  // namespace

int64_t scan_workspace(const dgen_hip_scan& a, bool backward) {
  return align256(scan_shape(a, backward).total * (int64_t)sizeof(float));
}

int scan_run(const dgen_hip_scan& a, bool backward, hipStream_t st, bool dry) {
  const char* what = backward ? "selective_scan_backward" : "selective_scan";
  DGEN_REQUIRE(a.struct_size == sizeof(a), "%s: struct_size %u, expected %zu", what, a.struct_size, sizeof(a));
  DGEN_REQUIRE(a.type == DGEN_HIP_F32 || a.type == DGEN_HIP_BF16, "%s: type %d", what, a.type);
  DGEN_REQUIRE(a.N >= 1 && a.N <= 64, "%s: N %lld outside [1, 64]", what, (long long)a.N);
  DGEN_REQUIRE(a.batch >= 0 && a.batch <= (1 << 20), "%s: batch %lld outside [0, 2^20]", what, (long long)a.batch);
  DGEN_REQUIRE(a.T >= 1 && a.T <= (1 << 24), "%s: T %lld outside [1, 2^24]", what, (long long)a.T);
  DGEN_REQUIRE(a.D >= 1 && a.D <= (1 << 20), "%s: D %lld outside [1, 2^20]", what, (long long)a.D);
  const ScanShape s = scan_shape(a, backward);
  // (a launch takes fewer than 2^32 threads; the carry's is far from that, as
  // time is cut only where sequences and channel blocks are few)
  DGEN_REQUIRE(s.nd * s.chunks * a.batch < (int64_t(1) << 23) && a.batch * ((a.T + 3) / 4) < (int64_t(1) << 31) &&
                   s.nd * a.batch < (int64_t(1) << 31) &&
                   (!backward || a.batch * a.T * 2 * a.N < (int64_t(1) << 31)),
               "%s: batch %lld x T %lld x D %lld x N %lld is too large for one call", what, (long long)a.batch,
               (long long)a.T, (long long)a.D, (long long)a.N);
  DGEN_REQUIRE(a.A, "%s: null A", what);
  for (const dgen_hip_seq* v : {&a.x, &a.dt, &a.z, &a.B, &a.C, &a.y, &a.dy, &a.dx, &a.ddt, &a.dz, &a.dB, &a.dC})
    DGEN_REQUIRE(a.T == 1 || v->stride_t < (1 << 26), "%s: stride of %lld between frames, at most 2^26", what,
                 (long long)v->stride_t);  // (a tile's offsets are 32 bits: 32 frames)
  const bool empty = a.batch == 0;
  for (const dgen_hip_seq* v : {&a.x, &a.dt, &a.B, &a.C})
    DGEN_REQUIRE((v->data || empty) && seq_readable(*v), "%s: x, dt, B or C missing or with a negative stride", what);
  DGEN_REQUIRE(!a.z.data || seq_readable(a.z), "%s: z has a negative stride", what);
  if (!backward) {
    DGEN_REQUIRE((a.y.data || empty) && seq_writable(a.y, a.batch, a.T, a.D), "%s: y missing or overlapping itself",
                 what);
  } else {
    DGEN_REQUIRE((a.dy.data || empty) && seq_readable(a.dy), "%s: dy missing or with a negative stride", what);
    for (const dgen_hip_seq* v : {&a.dx, &a.ddt})
      DGEN_REQUIRE((v->data || empty) && seq_writable(*v, a.batch, a.T, a.D),
                   "%s: dx or ddt missing or overlapping itself", what);
    for (const dgen_hip_seq* v : {&a.dB, &a.dC})
      DGEN_REQUIRE((v->data || empty) && seq_writable(*v, a.batch, a.T, a.N),
                   "%s: dB or dC missing or overlapping itself", what);
    DGEN_REQUIRE(!a.z.data || (a.dz.data && seq_writable(a.dz, a.batch, a.T, a.D)),
                 "%s: dz missing or overlapping itself", what);
    DGEN_REQUIRE(a.dA && (!a.skip || a.dskip) && (!a.dt_bias || a.ddt_bias), "%s: null dA, dskip or ddt_bias", what);
  }
  const int64_t need = scan_workspace(a, backward);
  DGEN_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= (uint64_t)need && (uintptr_t)a.workspace % 256 == 0),
               "%s: workspace of %llu bytes, %lld needed (256-byte aligned)", what,
               (unsigned long long)a.workspace_bytes, (long long)need);
  if (dry) return 0;
  if (empty) {
    if (!backward) return 0;
    enqueue_sum_parts(st, a.A, 0, {{a.dA, a.dskip, a.ddt_bias}, {a.D * a.N, a.D, a.D}});  // zeros
  } else if (a.type == DGEN_HIP_BF16) {
    scan_states<bf16>(a, backward, s, st);
  } else {
    scan_states<float>(a, backward, s, st);
  }
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
