// Gated delta rule, forward and backward.  Per sequence and head a memory S of
// K x V numbers, frame by frame
//   S' = e^g S,  u = beta (v - S'^T k^),  S = S' + k^ u^T,  y = scale S^T q^
// with q^ and k^ the queries and keys, or these over their norms.
//
// A memory that is rewritten each frame is a chain of outer products; matrix
// instructions need it by chunks.  With G(i) the sum of a chunk's gates up to
// frame i, d(i, j) = e^(G(i) - G(j)) for j <= i and S the memory that enters,
// the u of a chunk's frames solve
//   (I + A) U = r,  A(i, j) = beta(i) d(i, j) k^(i).k^(j) for j < i,
//   r(i) = beta(i) (v(i) - e^G(i) S^T k^(i)),
// so that with X = (I + A)^-1, which does not depend on S,
//   U = X r,  y = scale (e^G S^T q^ + (d q^.k^) U),  S <- e^G(end) S + k^T (d(end, .) U).
// A sum of gates is held in two floats (from a sum in 64 bits): a difference of
// two far sums is then right to the last bits.
//
// Launches: prepare (a workgroup per chunk and head: X, the queries' products
// with the keys, decays, norms), then the chain (a workgroup per head and block
// of values walks the chunks: three products and two of a triangle a chunk, the
// memory in registers, its parts in LDS).  Backward the chain keeps the memory
// that enters each chunk and U; the adjoints' chain, which needs neither, walks
// the other way in the same launch and keeps the adjoint D of the memory after
// each chunk and dR of r; the gradients of q, k, g and beta are then a launch
// with a workgroup per chunk, from products over the values:
//   dq^ = e^G dy S^T + (d dy U^T) k^,  dk^ = -beta (e^G dR S^T + (d dR U^T) k^)
//   + e^(G(end) - G) U D^T + the transposes of these,  dbeta = dR.(v - S'^T k^).
// A gate's gradient is the sum of what passes it:
//   dg(m) = sum over j < m <= i of (M o dy U^T - A o dR U^T)(i, j)   frame to frame,
//   over i >= m of e^G(i) (scale q^.S dy - beta k^.S dR)(i)          from the entering memory,
//   over j < m of e^(G(end) - G(j)) k^.D U(j),  and e^G(end) <S, D>  over the chunk's end.
// Each term has the decay e^g(m) in it, so the sum is as exact as its terms
// however much the gate forgets.  (The differences of q^.dq^ + k^.dk^ as read and
// k^.dk^ as written add up to the same, but terms that do not pass the gate cancel
// there: at g = -16 nothing but their rounding was left.)
// Few heads and a long axis: the chunks are cut into segments.  A segment is an
// affine map of the memory, so each is run from zero and, with the identity as
// its memory and nothing written, as a transition; a short chain over the
// segments' ends gives the memories that enter them (k_delta.hip has when).
//
// A number that is not finite may not reach results of frames before its own: 0
// times it, above a triangle's diagonal, would.  Each chunk's r (backward dy and dU) is
// looked through, eight products with 0 a lane; where a column has such a number, it
// goes on without it, and the rows from that frame on (backward up to it) are made
// NaN after each triangle.  A key, gate or strength that is none says so by its
// frame's scale of what the key reads.
//
// Chunks of 64 frames: a chunk costs 4 K V 64 operations for the memory, a share
// that does not depend on its length, and 64 (K + V) a frame within it, which does;
// at K = V = 128 the two are alike, and its triangles fit next to the memory.  Blocks
// of 32 values and four waves, two of them a CU: of 64 and eight, one a CU, they
// read and turn a chunk's keys half as often, and yet wait longer (400 heads of
// 1000 frames, 128 x 128, when both were built: 469 against 403 us in bf16, 1264
// against 972 in fp32).
//
// Precision: operands that are bf16 go to the bf16 instructions as they are.
// Numbers held in 32 bits (memories, adjoints, U, dR, X, M) are split into three
// bf16 parts, whose products of up to 2^-16 are kept: 24 bits, as fp32 products
// have, at a sixth to a third of the bf16 rate, still above the fp32 instructions'.
// That goes for y too, which may be what is left of larger numbers when it is
// rounded to bf16.  fp32 operands go to the fp32 instructions.
//
// What bounds it: 32 x 1000 x 8 heads of K = V = 128 in bf16 read and write 281 MB
// (55 us at 5.1 TB/s) in 0.265 ms.  (Launches' own times are the profiler's, under
// which they take longer than in a run of calls.)  Prepare has 71 us, the chain 231:
// its vector instructions (parts, turning) issue for 53 % of that, the matrix
// instructions are busy for 24 %, and of a wave's time a third is waiting for issue
// and a quarter for memory or one of three barriers a chunk, with two workgroups of
// four waves a CU (77 KB of LDS).  Backward 463 MB (91 us) take 0.95 ms: prepare 81,
// the two chains 473, gradients 536 us.  The kept memories and adjoints are 0.8 GB
// more, written and read again; a chain that took the gradients as it goes would
// need all of V in one workgroup and the sums over V in its registers, which was
// not built.  A call of few frames goes frame by frame with the memory in registers:
// 32 sequences of 8 heads, fp32, take 10 us for one frame (34 MB: 6.7 us).
#pragma once

#include <cfloat>

#include "seq.h"

namespace dgen {

constexpr int kC = 64;           // frames of a chunk
constexpr int kVB = 32;          // values of a block
constexpr int kVecs = 10;        // numbers of a chunk's frames
constexpr int kStepFrames = 16;  // calls of so few go frame by frame

// How a call is cut, and the places of its parts in the workspace.
struct DeltaPlan {
  int64_t chunks, nvb, segs, per;  // nvb: blocks of values, per: chunks of a segment
  int64_t X, M, XT, A, vec, S, dS, U, dR, ends, gends, bytes;
};
// Whether a call goes frame by frame: a chunk costs its 64 frames, a frame its sums
// over the memory (32 sequences of 8 heads of 128: 32 us in bf16 and 50 in fp32 for
// a chunk, 9 and 1.4 for each frame; 1 sequence of 4 heads of 64: 18 and 20, and 9
// and 0.6).
inline bool delta_steps(const dgen_hip_delta& a, bool backward) {
  return !backward && a.T <= kStepFrames;
}
DeltaPlan delta_plan(const dgen_hip_delta&, bool backward);
void delta_enqueue_f32(const dgen_hip_delta&, bool backward, hipStream_t);
void delta_enqueue_bf16(const dgen_hip_delta&, bool backward, hipStream_t);

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr float kUnitEps = 1e-6f;

// Parts of fp32 numbers in bf16 products.
constexpr int kState = 3;

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
  floatx8 p;
};

template <class E, int P>
__device__ __forceinline__ Wide<E, P> wide(floatx8 x) {
  Wide<E, P> w;
  if constexpr (std::is_same<E, float>::value) {
    w.p = x;
  } else {
#pragma unroll
    for (int q = 0; q < P; ++q) {
      w.p[q] = __builtin_convertvector(x, bf16x8);
      if (q + 1 < P) x -= __builtin_convertvector(w.p[q], floatx8);
    }
  }
  return w;
}

// acc[i][j] += a[i] b[j] over the eight elements of each of the four lane groups,
// the instructions of one sum apart from one another.
template <int PA, int PB, int NA, int NB>
__device__ __forceinline__ void mma(floatx4 (&acc)[NA][NB], const Wide<bf16, PA> (&a)[NA], const Wide<bf16, PB> (&b)[NB]) {
  constexpr int most = PA > PB ? PA : PB;
#pragma unroll
  for (int s = most - 1; s >= 0; --s)
#pragma unroll
    for (int q = 0; q < PA; ++q)
      if (s - q >= 0 && s - q < PB)
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i].p[q], b[j].p[s - q], acc[i][j], 0, 0, 0);
}
template <int PA, int PB, int NA, int NB>
__device__ __forceinline__ void mma(floatx4 (&acc)[NA][NB], const Wide<float, PA> (&a)[NA], const Wide<float, PB> (&b)[NB]) {
#pragma unroll
  for (int q = 0; q < 8; ++q)
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i].p[q], b[j].p[q], acc[i][j], 0, 0, 0);
}
// Loads stay before, products after.
__device__ __forceinline__ void loads_first() { __builtin_amdgcn_sched_barrier(0); }
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// What the parts add up to.
template <int P>
__device__ __forceinline__ floatx8 whole_of(const Wide<bf16, P>& w) {
  floatx8 x = __builtin_convertvector(w.p[P - 1], floatx8);
#pragma unroll
  for (int q = P - 2; q >= 0; --q) x += __builtin_convertvector(w.p[q], floatx8);
  return x;
}
template <int P>
__device__ __forceinline__ floatx8 whole_of(const Wide<float, P>& w) { return w.p; }

// A matrix in LDS whose rows are fragments' rows, split into parts as it is
// written.  A row's 16-byte pieces are permuted by the row, so that the sixteen
// lanes whose pieces are read at once (0-3, 12-15 and 20-27, and so on) find them
// in sixteen different groups of banks.
template <class E, int P, int ROWS, int COLS>
struct Tile {
  static constexpr bool kFloat = std::is_same<E, float>::value;
  static constexpr int kParts = kFloat ? 1 : P, kPiece = kFloat ? 4 : 8, kPieces = COLS / kPiece;
  using T = typename std::conditional<kFloat, float, __bf16>::type;
  alignas(16) T d[kParts][ROWS * COLS];

  static __device__ __forceinline__ int at(int row, int col) {
    const int by = kPieces == 4 ? (0x78 >> (row >> 2 & 3) * 2) & 3 : kPieces == 8 ? ((row >> 1) + 6) & 7 : row & 15;
    return row * COLS + ((col / kPiece) ^ by) * kPiece + col % kPiece;
  }
  // Four consecutive columns, from a multiple of four on.
  __device__ __forceinline__ void put4(int row, int col, floatx4 x) {
    const int i = at(row, col);
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      if constexpr (kFloat) {
        *reinterpret_cast<floatx4*>(&d[q][i]) = x;
      } else {
        const bf16x4 h = __builtin_convertvector(x, bf16x4);
        *reinterpret_cast<bf16x4*>(&d[q][i]) = h;
        if (q + 1 < kParts) x -= __builtin_convertvector(h, floatx4);
      }
    }
  }
  // A fragment, as eight columns of one row or as eight rows of one column.
  __device__ __forceinline__ void put_row(int row, int col, const Wide<E, 1>& w) {
    if constexpr (kFloat) {
      *reinterpret_cast<floatx4*>(&d[0][at(row, col)]) = w.p.lo;
      *reinterpret_cast<floatx4*>(&d[0][at(row, col + 4)]) = w.p.hi;
    } else {
      *reinterpret_cast<bf16x8*>(&d[0][at(row, col)]) = w.p[0];
    }
  }
  __device__ __forceinline__ void put_column(int row, int col, const Wide<E, 1>& w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (kFloat) d[0][at(row + i, col)] = w.p[i];
      else d[0][at(row + i, col)] = w.p[0][i];
    }
  }
  __device__ __forceinline__ Wide<E, P> frag(int row, int col) const {
    Wide<E, P> w;
    if constexpr (kFloat) {
      w.p.lo = *reinterpret_cast<const floatx4*>(&d[0][at(row, col)]);
      w.p.hi = *reinterpret_cast<const floatx4*>(&d[0][at(row, col + 4)]);
    } else {
#pragma unroll
      for (int q = 0; q < P; ++q) w.p[q] = *reinterpret_cast<const bf16x8*>(&d[q][at(row, col)]);
    }
    return w;
  }
  // What four consecutive columns' parts add up to.
  __device__ __forceinline__ floatx4 whole4(int row, int col) const {
    const int i = at(row, col);
    floatx4 x = {0, 0, 0, 0};
#pragma unroll
    for (int q = kParts - 1; q >= 0; --q) {
      if constexpr (kFloat) x = *reinterpret_cast<const floatx4*>(&d[q][i]);
      else x += __builtin_convertvector(*reinterpret_cast<const bf16x4*>(&d[q][i]), floatx4);
    }
    return x;
  }
  __device__ __forceinline__ void clear(int row, int col) {
#pragma unroll
    for (int q = 0; q < kParts; ++q) d[q][at(row, col)] = (T)0.f;
  }
  // Four consecutive columns of the first part.
  __device__ __forceinline__ floatx4 first4(int row, int col) const {
    if constexpr (kFloat) return *reinterpret_cast<const floatx4*>(&d[0][at(row, col)]);
    else return __builtin_convertvector(*reinterpret_cast<const bf16x4*>(&d[0][at(row, col)]), floatx4);
  }
};

// A chunk's keys (or queries), written by rows and read by columns: four frames of
// one channel a lane, of 16 channels from k on.  bf16 stays in rows and is turned
// by the LDS as it is read (of 16 lanes, lane l reads four channels of row l / 4
// and is given channel l of the four rows).
template <class E, int KP>
struct Turned {
  static constexpr bool kFloat = std::is_same<E, float>::value;
  Tile<E, 1, kFloat ? KP : kC, kFloat ? kC : KP> t;

  __device__ __forceinline__ void put(int row, int k, const Wide<E, 1>& w) {
    if constexpr (kFloat) t.put_column(k, row, w);
    else t.put_row(row, k, w);
  }
  __device__ __forceinline__ bf16x4 four(int k, int row, int l16) const {
    typedef __attribute__((address_space(3))) bf16x4 Lds;
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Lds*)&t.d[0][t.at(row + (l16 >> 2), k + 4 * (l16 & 3))]);
  }
  __device__ __forceinline__ Wide<E, 1> frag(int k, int row, int l16) const {
    if constexpr (kFloat) {
      return t.frag(k + l16, row);
    } else {
      const bf16x4 a = four(k, row, l16), b = four(k, row + 4, l16);
      return {{__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)}};
    }
  }
  __device__ __forceinline__ floatx4 first4(int k, int row, int l16) const {
    if constexpr (kFloat) return t.first4(k + l16, row);
    else return __builtin_convertvector(four(k, row, l16), floatx4);
  }
};

// Elements [at, at + 8) of a row of n as they are read, without branches and with
// nothing done to them, so that they can be in flight until they are used: a piece
// past the end is read from the row's last eight, and shifted or dropped then.
template <class T>
struct __attribute__((packed, aligned(alignof(T)))) Eight {
  T e[8];
};
typedef uint32_t uint32x4 __attribute__((ext_vector_type(4)));
template <class E>
struct Raw {
  typename std::conditional<std::is_same<E, float>::value, floatx8, uint32x4>::type x;
};
template <bool WHOLE, class E>
__device__ __forceinline__ void load_raw(Raw<E>& o, const E* __restrict__ p, int at, int n) {
  if (WHOLE || n >= 8) {
    o.x = __builtin_bit_cast(decltype(o.x), *reinterpret_cast<const Eight<E>*>(p + min(at, n - 8)));
  } else {  // (all of the row, its last element again and again)
    Eight<E> e;
#pragma unroll
    for (int i = 0; i < 8; ++i) e.e[i] = p[min(i, n - 1)];
    o.x = __builtin_bit_cast(decltype(o.x), e);
  }
}
// What they stand for: 0 past the row's end, and where `on` is false.  WHOLE: n
// is a multiple of 8.
template <bool WHOLE>
__device__ __forceinline__ Wide<bf16, 1> exact_of(const Raw<bf16>& r, int at, int n, bool on) {
  uint32x4 x = r.x;
  if constexpr (!WHOLE) {
    const int by = at - (n - 8);  // elements that were read too early
    if (n >= 8) {
      const bool four = by > 0 && by & 4, two = by > 0 && by & 2;
      const uint32_t half = by > 0 && by & 1 ? 16 : 0;
      x = four ? uint32x4{x[2], x[3], 0u, 0u} : x;
      x = two ? uint32x4{x[1], x[2], x[3], 0u} : x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_alignbit(i < 3 ? x[i < 3 ? i + 1 : 3] : 0u, x[i], half);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = 2 * i + 1 < n ? x[i] : 2 * i < n ? x[i] & 0xffffu : 0u;
    }
  }
  const bool in = on && at < n;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = in ? x[i] : 0u;
  return {{__builtin_bit_cast(bf16x8, x)}};
}
template <bool WHOLE>
__device__ __forceinline__ Wide<float, 1> exact_of(const Raw<float>& r, int at, int n, bool on) {
  floatx8 x = r.x;
  if constexpr (!WHOLE) {
    const int by = at - (n - 8);
    if (n >= 8) {
#pragma unroll
      for (int k = 4; k > 0; k /= 2) {
        const bool yes = by > 0 && by & k;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = yes ? (i + k < 8 ? x[i + k < 8 ? i + k : 7] : 0.f) : x[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = i < n ? x[i] : 0.f;
    }
  }
  const bool in = on && at < n;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = in ? x[i] : 0.f;
  return {x};
}
template <bool WHOLE, class E>
__device__ __forceinline__ Wide<E, 1> load_exact(const E* __restrict__ p, int at, int n, bool on) {
  Raw<E> r;
  load_raw<WHOLE>(r, p, at, n);
  return exact_of<WHOLE>(r, at, n, on);
}
__device__ __forceinline__ floatx8 floats(const Wide<float, 1>& w) { return w.p; }
__device__ __forceinline__ floatx8 floats(const Wide<bf16, 1>& w) { return __builtin_convertvector(w.p[0], floatx8); }
// Eight and four aligned floats.
__device__ __forceinline__ floatx8 load_row(const float* __restrict__ p) { return *reinterpret_cast<const floatx8*>(p); }
__device__ __forceinline__ floatx4 load_vec(const float* __restrict__ p) { return *reinterpret_cast<const floatx4*>(p); }

// Workgroups in an order in which neighbours share an XCD (they go round the
// eight XCDs), and with it the cache that holds what they share.
__device__ __forceinline__ uint32_t xcd_order(uint32_t i, uint32_t n) {
  const uint32_t x = i & 7, each = n >> 3, more = n & 7;
  return x * each + min(x, more) + (i >> 3);
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
enum Vec { kReadK, kWriteK, kReadQ, kBeta, kGHigh, kGLow, kRootK, kRootQ, kInto, kRest };
static_assert(kRest + 1 == kVecs, "");

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
  int T, H, shared, K, V;
  int chunks, nvb, segs, per;  // chunks a segment
  // The workspace, with KP for K and Vp, whole blocks of values, for V (0 in
  // what is between).
  int Vp;
  // [B H][chunks]: inverse, queries' products with keys [64][64], Vec [kVecs][64];
  // backward: XT, X transposed, and M and A transposed in their own places
  float *X, *M, *XT, *A, *vec;
  // backward: states entering and adjoints after a chunk [KP / 4][Vp][4], [16][Vp][4]:
  // a lane's four rows of a product are one store
  float *S, *dS, *U, *dR;
  float *ends, *gends;     // [B H][segs][KP][Vp + KP] (states | transitions), [KP][Vp]
};

__device__ __forceinline__ int live_of(const int32_t* __restrict__ lengths, int b, int T) {
  if (!lengths) return T;
  const int n = lengths[b];
  return n < 0 ? 0 : n < T ? n : T;
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= FLT_MAX; }
// A chunk's columns with numbers that are not finite, and from which row on (BACK:
// up to which, counted from the last).
template <bool BACK>
struct Spoilt {
  alignas(16) int waves[4];
  int from[4][kVB];

  // Before a barrier: whether a wave's x has any.
  __device__ __forceinline__ void note(const floatx4 (&x)[2], int w) {
    float t = 0.f;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int e = 0; e < 4; ++e) t = fmaf(x[v][e], 0.f, t);
    waves[w] = __ballot(!(t == 0.f)) != 0;
  }
  // After it: the notes, and whether there are any.
  __device__ __forceinline__ int4 notes() const { return *reinterpret_cast<const int4*>(waves); }
  static __device__ __forceinline__ bool any(int4 f) { return __builtin_amdgcn_readfirstlane(f.x | f.y | f.z | f.w) != 0; }
  // If so, which is seldom: 0 in the place of the tile's, which is a
  // wave's rows rows .. rows + 3 of columns l16 and 16 + l16.  `also`: numbers of
  // the same rows that are left.
  template <class E, int P>
  __device__ __forceinline__ void settle(Tile<E, P, kVB, kC>& tile, const floatx4 (&also)[2], int w, int lane, int rows) {
    const int l16 = lane & 15;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const floatx4 x = tile.whole4(16 * v + l16, rows);
      int at = kC;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = is_finite(x[e]);
        if (!in || (BACK && !is_finite(also[v][e]))) at = min(at, BACK ? kC - 1 - rows - e : rows + e);
        if (!in) tile.clear(16 * v + l16, rows + e);
      }
      at = min(at, __shfl_xor(at, 16, 64));
      at = min(at, __shfl_xor(at, 32, 64));
      if (lane < 16) from[w][16 * v + lane] = at;
    }
    lds_barrier();
  }
  // x with `with` in the rows that are spoilt.
  __device__ __forceinline__ void put(floatx4 (&x)[2], float with, int l16, int rows) const {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      int first = kC;
#pragma unroll
      for (int k = 0; k < 4; ++k) first = min(first, from[k][16 * v + l16]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[v][e] = (BACK ? kC - 1 - rows - e : rows + e) >= first ? with : x[v][e];
    }
  }
};

// ------------------------------------------------------------------- prepare
// Per chunk and head: decays, norms, M and X.
template <class E, int KP, bool WHOLE>
__global__ __launch_bounds__(kThreads) void k_delta_prepare(DeltaP<E> p) {
  constexpr int NF = KP / 32;
  __shared__ float A[kC][kC + 4], part[3][16][20];
  __shared__ float gh[kC], gl[kC], bt[kC], rk[kC], rq[kC];
  __shared__ int bad[kC];  // frames whose row of A is not finite
  __shared__ union {
    Tile<E, 1, kC, KP> kt;
    float X[kC][kC + 4];  // (after the products)
  } lds;
  auto& kt = lds.kt;
  auto& X = lds.X;
  const int c = blockIdx.x % (uint32_t)p.chunks, bh = blockIdx.x / (uint32_t)p.chunks, b = bh / p.H, h = bh % p.H;
  const int t0 = c * kC, live = live_of(p.lengths, b, p.T) - t0;
  if (live <= 0) return;
  const int lane = threadIdx.x & 63, w = wave_index(), l16 = lane & 15, g4 = lane >> 4, hk = h / p.shared;
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
    bad[lane] = 0;
  }
  const int row = 16 * w + l16;
  Wide<E, 1> kf[NF], qf[NF];
  {
    float sk = 0.f, sq = 0.f;
    const bool on = row < live;
    const E *kp = p.k.row(b, t0 + min(row, live - 1), hk), *qp = p.q.row(b, t0 + min(row, live - 1), hk);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      kf[f] = load_exact<WHOLE>(kp, f * 32 + g4 * 8, p.K, on);
      qf[f] = load_exact<WHOLE>(qp, f * 32 + g4 * 8, p.K, on);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      kt.put_row(row, f * 32 + g4 * 8, kf[f]);
      const floatx8 x = floats(kf[f]), y = floats(qf[f]);
#pragma unroll
      for (int i = 0; i < 8; ++i) sk = fmaf(x[i], x[i], sk), sq = fmaf(y[i], y[i], sq);
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
    floatx4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0}, a = {0, 0, 0, 0};
    floatx4 acc[2][1] = {};
    const int j = 16 * tj + l16;
    if (tj <= w) {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const Wide<E, 1> both[2] = {kf[f], qf[f]}, o[1] = {kt.frag(j, f * 32 + g4 * 8)};
        mma(acc, both, o);
      }
      kk = acc[0][0], qk = acc[1][0];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * w + 4 * g4 + r;
      const float d = j <= i ? exp_accurate((gh[i] - gh[j]) + (gl[i] - gl[j])) : 0.f;
      a[r] = j < i ? kk[r] * (rk[i] * rk[j]) * d * bt[i] : 0.f;
      if (!is_finite(a[r])) a[r] = 0.f, bad[i] = 1;
      A[i][j] = a[r];
      qk[r] = j <= i ? qk[r] * (rq[i] * rk[j] * p.scale) * d : 0.f;
    }
    // (the quarter above the diagonal, whose products are left out, is not stored)
    if (w < 2 && tj >= 2) continue;
    if (p.XT) {
      *reinterpret_cast<floatx4*>(Mp + j * kC + 16 * w + 4 * g4) = qk;
      *reinterpret_cast<floatx4*>(p.A + ci * kC * kC + j * kC + 16 * w + 4 * g4) = a;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) Mp[(16 * w + 4 * g4 + r) * kC + j] = qk[r];
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
#pragma unroll
  for (int i = 0; i < kC * kC / 4 / kThreads; ++i) {
    const int r = threadIdx.x / 16 + 16 * i, col = threadIdx.x % 16 * 4;
    const floatx4 x = *reinterpret_cast<const floatx4*>(&X[r][col]);
    if (col < 32 || r >= 32) *reinterpret_cast<floatx4*>(Xp + r * kC + col) = col / 16 <= r / 16 ? x : floatx4{0, 0, 0, 0};
    if (p.XT && (col >= 32 || r < 32)) {
      const floatx4 y = {X[col][r], X[col + 1][r], X[col + 2][r], X[col + 3][r]};
      *reinterpret_cast<floatx4*>(p.XT + ci * kC * kC + r * kC + col) = col / 16 >= r / 16 ? y : floatx4{0, 0, 0, 0};
    }
  }
  if (w == 0) {
    float* v = p.vec + ci * kVecs * kC + lane;
    const float into = exp_accurate(gh[lane] + gl[lane]);
    const float rest = exp_accurate((gh[kC - 1] - gh[lane]) + (gl[kC - 1] - gl[lane]));
    v[kReadK * kC] = bad[lane] ? NAN : into * rk[lane];
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

// A workgroup's sequence and head, block of kVB values and segment of chunks.
struct Place {
  int b, h, hk, bh, vb, seg;
};
template <class E>
__device__ __forceinline__ Place place_of(const DeltaP<E>& p, int blocks, uint32_t block, uint32_t of) {
  Place o;
  uint32_t i = xcd_order(block, of);
  o.vb = i % (uint32_t)blocks, i /= (uint32_t)blocks;
  o.seg = i % (uint32_t)p.segs, i /= (uint32_t)p.segs;
  o.bh = i;
  o.b = o.bh / p.H, o.h = o.bh % p.H;
  o.hk = o.h / p.shared;
  return o;
}

// A wave's part: rows 16 w of a chunk's frames with two tiles of values, and
// NKT x NVT tiles of the memory.
template <int KP>
struct Split {
  static constexpr int NF = KP / 32, NV = 2, NT = KP / 32, NVT = NT < 2 ? NT : 2, NKT = NT / NVT;
  int lane, w, l16, g4;
  __device__ __forceinline__ Split() {
    lane = threadIdx.x & 63, w = wave_index(), l16 = lane & 15, g4 = lane >> 4;
  }
  // the memory's tiles: first channel and value
  __device__ __forceinline__ int tile_k(int i) const { return (w * NT / 2 + i) * 16; }
  __device__ __forceinline__ int tile_v(int j) const { return (w * NT % 2 + j) * 16; }
};
// f(i, j, e, k, v) over the memory's tiles and a lane's four channels of each.
#define DGEN_TILES(...)                                                         \
  _Pragma("unroll") for (int i = 0; i < W::NKT; ++i)                            \
  _Pragma("unroll") for (int j = 0; j < W::NVT; ++j) {                          \
    const int k = me.tile_k(i) + 4 * g4, v = v0 + me.tile_v(j) + l16;           \
    _Pragma("unroll") for (int e = 0; e < 4; ++e) { __VA_ARGS__ }               \
  }
// A chunk's frames of one operand and head: their first row (the same in all
// lanes), the step between them, how many there are.
template <class E>
struct Frames {
  E* p;
  uint32_t step;
  int n;
};
template <class E>
__device__ __forceinline__ Frames<E> frames_of(const Heads<E>& a, int b, int h, int t0, int n) {
  return {a.row(b, t0, h), (uint32_t)a.t, n};
}
// Row `row` of K channels, as fragments.
template <bool WHOLE, int NF, class E>
__device__ __forceinline__ void load_rows(const Frames<const E>& a, int row, int g4, int K, Raw<E> (&o)[NF]) {
  const E* p = a.p + (uint32_t)min(row, a.n - 1) * a.step;
#pragma unroll
  for (int f = 0; f < NF; ++f) load_raw<WHOLE>(o[f], p, f * 32 + g4 * 8, K);
}
// Four rows of one column in each of four neighbouring lanes turned into four
// columns of one row, and back.
__device__ __forceinline__ floatx4 turn(floatx4 x, int lane) {
  const bool odd = lane & 1, upper = lane & 2;
  const float a = dpp<0xB1>(odd ? x[0] : x[1]), b = dpp<0xB1>(odd ? x[2] : x[3]);
  x = odd ? floatx4{a, x[1], b, x[3]} : floatx4{x[0], a, x[2], b};
  const float c = dpp<0x4E>(upper ? x[0] : x[2]), d = dpp<0x4E>(upper ? x[1] : x[3]);
  return upper ? floatx4{c, d, x[2], x[3]} : floatx4{x[0], x[1], c, d};
}
// Four values, from column `at` of a row of n, as they are read (moved down where
// the row ends before: right where they are used).
typedef uint32_t uint32x2 __attribute__((ext_vector_type(2)));
template <class E>
struct Quad {
  typename std::conditional<std::is_same<E, float>::value, floatx4, uint32x2>::type x;
};
template <bool WHOLE, class E>
__device__ __forceinline__ void load_quad(Quad<E>& o, const E* __restrict__ row, int at, int n) {
  if (WHOLE || n >= 4) {
    o.x = __builtin_bit_cast(decltype(o.x), *reinterpret_cast<const Four<E>*>(row + min(at, n - 4)));
  } else {
    Four<E> e;
#pragma unroll
    for (int i = 0; i < 4; ++i) e.e[i] = row[min(i, n - 1)];
    o.x = __builtin_bit_cast(decltype(o.x), e);
  }
}
template <bool WHOLE, class E>
__device__ __forceinline__ floatx4 quad_of(const Quad<E>& q, int at, int n, bool on) {
  const Four<E> r = __builtin_bit_cast(Four<E>, q.x);
  floatx4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = to_f32(r.e[i]);
  if constexpr (!WHOLE) {
    const int by = n >= 4 ? at - (n - 4) : 0;
    x = by > 0 && by & 2 ? floatx4{x[2], x[3], 0.f, 0.f} : x;
    x = by > 0 && by & 1 ? floatx4{x[1], x[2], x[3], 0.f} : x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = at + i < n ? x[i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = on && at < n ? x[i] : 0.f;
  return x;
}
// A product's lane has rows 4 g4 .. 4 g4 + 3 of column l16 of its two tiles; of
// memory it takes, or gives, columns 4 (l16 / 4) .. + 3 of row 4 g4 + l16 % 4.
template <bool WHOLE, class E>
__device__ __forceinline__ void load_values(const Frames<const E>& a, int t, int col, int V, Quad<E> (&o)[2]) {
  const E* row = a.p + (uint32_t)min(t, a.n - 1) * a.step;
#pragma unroll
  for (int v = 0; v < 2; ++v) load_quad<WHOLE>(o[v], row, col + 16 * v, V);
}
// Row t of T that are there, zeros behind the sequence.
template <class E>
__device__ __forceinline__ void store_values(const Frames<E>& a, int t, int T, int col, int V, int lane, const floatx4 (&o)[2]) {
  E* row = a.p + (uint32_t)t * a.step;
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    floatx4 x = turn(o[v], lane);
    if (t >= a.n) x = floatx4{0.f, 0.f, 0.f, 0.f};
    const int at = col + 16 * v;
    const float y[4] = {x[0], x[1], x[2], x[3]};
    if (t < T) store_four(row + at, V - at, y);
  }
}
// Zeros in the chunks from c0 on.
template <class E>
__device__ __forceinline__ void store_zeros(const Heads<E>& a, const Place& at, int c0, int c1, int T, int v0, int V) {
  const int t0 = c0 * kC, n = min(c1 * kC, T) - t0;
  for (int i = threadIdx.x; i < n * kVB; i += blockDim.x)
    if (v0 + i % kVB < V) a.row(at.b, t0 + i / kVB, at.h)[v0 + i % kVB] = from_f32<E>(0.f);
}

template <class E, int KP, Mode MODE>
struct ChainLds {
  Tile<E, kState, kVB, KP> s;
  Tile<E, kState, kVB, kC> r, wr;
  Tile<E, kState, MODE == kOut ? kVB : 1, kC> u;
  Turned<E, KP> kt;
  Spoilt<false> bad;
};
// The memory's states along a segment's chunks.
template <class E, int KP, Mode MODE, bool WHOLE>
__device__ __forceinline__ void delta_chain(const DeltaP<E>& p, ChainLds<E, KP, MODE>& L, uint32_t block, uint32_t blocks) {
  using W = Split<KP>;
  constexpr int NF = W::NF, NV = W::NV, NKT = W::NKT, NVT = W::NVT;
  auto &s = L.s;
  auto &r = L.r, &wr = L.wr;
  auto& u = L.u;
  auto& kt = L.kt;
  const W me;
  const int l16 = me.l16, g4 = me.g4;
  const int nvb = MODE == kEnds ? p.nvb + (KP + kVB - 1) / kVB : p.nvb;
  const Place at = place_of(p, nvb, block, blocks);
  const int live = live_of(p.lengths, at.b, p.T);
  // (ends: the transition is the state's own columns, from the identity on and
  // with nothing written)
  const bool unit = MODE == kEnds && at.vb >= p.nvb;
  const int v0 = (unit ? at.vb - p.nvb : at.vb) * kVB;
  const int64_t end = ((int64_t)at.bh * p.segs + at.seg) * KP;
  const int ld = p.Vp + KP;
  floatx4 S[NKT][NVT] = {};
  if (unit) {
    DGEN_TILES(S[i][j][e] = k + e == v ? 1.f : 0.f;)
  } else if (MODE != kEnds && p.segs > 1) {
    DGEN_TILES(S[i][j][e] = p.ends[(end + k + e) * ld + v];)
  } else if (MODE != kEnds && p.state) {
    DGEN_TILES(const float x = p.state[((int64_t)at.bh * p.K + min(k + e, p.K - 1)) * p.V + min(v, p.V - 1)];
               S[i][j][e] = k + e < p.K && v < p.V ? x : 0.f;)
  }
#pragma unroll
  for (int i = 0; i < NKT; ++i)
#pragma unroll
    for (int j = 0; j < NVT; ++j) s.put4(me.tile_v(j) + l16, me.tile_k(i) + 4 * g4, S[i][j]);
  const int c0 = at.seg * p.per, c1 = min(c0 + p.per, p.chunks), cl = min(max((live + kC - 1) / kC, c0), c1);
  const int row = 16 * me.w + l16, rows = 16 * me.w + 4 * g4, col = v0 + l16;
  Raw<E> kr[NF], qr[MODE == kOut ? NF : 1];
  Quad<E> vr[NV];
  const int trow = rows + (l16 & 3), tcol = v0 + (l16 & ~3);  // (turned)
  auto load = [&](int c) {
    const int t0 = c * kC, n = live - t0;
    load_rows<WHOLE>(frames_of(p.k, at.b, at.hk, t0, n), row, g4, p.K, kr);
    if constexpr (MODE == kOut) load_rows<WHOLE>(frames_of(p.q, at.b, at.hk, t0, n), row, g4, p.K, qr);
    load_values<WHOLE>(frames_of(p.v, at.b, at.h, t0, n), trow, tcol, p.V, vr);
  };
  if (c0 < cl) load(c0);
  lds_barrier();
  for (int c = c0; c < cl; ++c) {
    const int t0 = c * kC;
    const int64_t ci = (int64_t)at.bh * p.chunks + c;
    const float* vec = p.vec + ci * kVecs * kC;
    const floatx4 beta = load_vec(vec + kBeta * kC + rows), read = load_vec(vec + kReadK * kC + rows);
    const floatx4 write = load_vec(vec + kWriteK * kC + rows), readq = load_vec(vec + kReadQ * kC + rows);
    const float whole = vec[kInto * kC + kC - 1];
    floatx8 xf[2], mf[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if (f > me.w / 2) break;
      xf[f] = load_row(p.X + ci * kC * kC + (uint32_t)(row * kC + g4 * 8) + f * 32);
      if constexpr (MODE == kOut) mf[f] = load_row(p.M + ci * kC * kC + (uint32_t)(row * kC + g4 * 8) + f * 32);
    }
    if constexpr (MODE == kKeep) {
      float* out = p.S + ci * KP * p.Vp;
#pragma unroll
      for (int i = 0; i < NKT; ++i)
#pragma unroll
        for (int j = 0; j < NVT; ++j)
          *reinterpret_cast<floatx4*>(out + (uint32_t)(((me.tile_k(i) >> 2) + g4) * p.Vp + v0 + me.tile_v(j) + l16) * 4) = S[i][j];
    }
    const int n = live - t0;
    Wide<E, 1> kf[NF], qf[MODE == kOut ? NF : 1];
    floatx4 val[NV];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      kf[f] = exact_of<WHOLE>(kr[f], f * 32 + g4 * 8, p.K, row < n);
      if constexpr (MODE == kOut) qf[f] = exact_of<WHOLE>(qr[f], f * 32 + g4 * 8, p.K, row < n);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) val[v] = turn(quad_of<WHOLE>(vr[v], tcol + 16 * v, p.V, !unit && trow < n), l16);
    // what the keys and queries read of the entering memory
    Wide<E, kState> o[2][NV];
    floatx4 ks[2][1][NV] = {}, qs[1][NV] = {};  // (keys: even and odd fragments apart)
#pragma unroll
    for (int v = 0; v < NV; ++v) o[0][v] = s.frag(16 * v + l16, g4 * 8);
#pragma unroll
    for (int f = 0; f < NF; ++f)
      kt.put(row, f * 32 + g4 * 8, kf[f]);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      if (f + 1 < NF)
#pragma unroll
        for (int v = 0; v < NV; ++v) o[(f + 1) & 1][v] = s.frag(16 * v + l16, (f + 1) * 32 + g4 * 8);
      loads_first();
      const Wide<E, 1> a[1] = {kf[f]};
      mma(ks[f & 1], a, o[f & 1]);
      if constexpr (MODE == kOut) {
        const Wide<E, 1> b[1] = {qf[f]};
        mma(qs, b, o[f & 1]);
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) val[v] = beta * (val[v] - read * (ks[0][0][v] + ks[1][0][v]));
    L.bad.note(val, me.w);
#pragma unroll
    for (int v = 0; v < NV; ++v) r.put4(16 * v + l16, rows, val[v]);
    load(min(c + 1, cl - 1));  // (the next chunk's, in flight through this one's products)
    lds_barrier();
    // U = X r
    const int4 notes = L.bad.notes();
    floatx4 U[1][NV];
    auto solve = [&] {
#pragma unroll
      for (int v = 0; v < NV; ++v) U[0][v] = floatx4{0, 0, 0, 0};
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        if (f > me.w / 2) break;
        Wide<E, kState> x[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) x[v] = r.frag(16 * v + l16, f * 32 + g4 * 8);
        loads_first();
        const Wide<E, kState> a[1] = {wide<E, kState>(xf[f])};
        mma(U, a, x);
      }
    };
    solve();
    const bool some = L.bad.any(notes);
    if (some) {
      L.bad.settle(r, val, me.w, me.lane, rows);
      solve();
      L.bad.put(U[0], 0.f, l16, rows);
    }
    if constexpr (MODE == kOut)
#pragma unroll
      for (int v = 0; v < NV; ++v) u.put4(16 * v + l16, rows, U[0][v]);
    if (some) L.bad.put(U[0], NAN, l16, rows);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      wr.put4(16 * v + l16, rows, U[0][v] * write);
      if constexpr (MODE == kKeep)
        *reinterpret_cast<floatx4*>(p.U + ci * kC * p.Vp + (uint32_t)((rows >> 2) * p.Vp + col + 16 * v) * 4) = U[0][v];
    }
    lds_barrier();
    if constexpr (MODE == kOut) {
      // y = queries' reading + M U
#pragma unroll
      for (int v = 0; v < NV; ++v) qs[0][v] *= readq;
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        if (f > me.w / 2) break;
        Wide<E, kState> x[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) x[v] = u.frag(16 * v + l16, f * 32 + g4 * 8);
        loads_first();
        const Wide<E, kState> a[1] = {wide<E, kState>(mf[f])};
        mma(qs, a, x);
      }
      if (some) L.bad.put(qs[0], NAN, l16, rows);
      store_values(frames_of(p.y, at.b, at.h, t0, n), trow, p.T - t0, tcol, p.V, l16, qs[0]);
    }
    // the memory over the chunk's end
#pragma unroll
    for (int i = 0; i < NKT; ++i)
#pragma unroll
      for (int j = 0; j < NVT; ++j) S[i][j] *= whole;
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      Wide<E, 1> a[NKT];
      Wide<E, kState> x[NVT];
#pragma unroll
      for (int i = 0; i < NKT; ++i) a[i] = kt.frag(me.tile_k(i), f * 32 + g4 * 8, l16);
#pragma unroll
      for (int j = 0; j < NVT; ++j) x[j] = wr.frag(me.tile_v(j) + l16, f * 32 + g4 * 8);
      loads_first();
      mma(S, a, x);
    }
#pragma unroll
    for (int i = 0; i < NKT; ++i)
#pragma unroll
      for (int j = 0; j < NVT; ++j) s.put4(me.tile_v(j) + l16, me.tile_k(i) + 4 * g4, S[i][j]);
    lds_barrier();
  }
  if constexpr (MODE == kOut) {
    store_zeros(p.y, at, cl, c1, p.T, v0, p.V);
    if (p.state_out && at.seg == p.segs - 1) {
      DGEN_TILES(if (k + e < p.K && v < p.V) p.state_out[((int64_t)at.bh * p.K + k + e) * p.V + v] = S[i][j][e];)
    }
  }
  if constexpr (MODE == kEnds) {
    if (unit) {
      DGEN_TILES(if (v < KP) p.ends[(end + k + e) * ld + p.Vp + v] = S[i][j][e];)
    } else {
      DGEN_TILES(p.ends[(end + k + e) * ld + v] = S[i][j][e];)
    }
  }
}

template <class E, int KP, bool WHOLE>
__global__ __launch_bounds__(kThreads) void k_delta_forward(DeltaP<E> p) {
  __shared__ ChainLds<E, KP, kOut> lds;
  delta_chain<E, KP, kOut, WHOLE>(p, lds, blockIdx.x, gridDim.x);
}

// The states that enter the segments (BACK: the adjoints after them) from the
// segments' ends from zero and their transitions, in the ends' place.
template <class E, int KP, bool BACK>
__device__ __forceinline__ void delta_carry(const DeltaP<E>& p, int block, Tile<float, 1, 16, KP> (&s)[2]) {
  constexpr int VB = 16, NF = KP / 32, NT = KP / 64 > 0 ? KP / 64 : 1;  // (16 values a workgroup, tiles of a wave)
  const int nvb = p.Vp / VB, vb = block % nvb, bh = block / nvb;
  const int lane = threadIdx.x & 63, w = wave_index(), l16 = lane & 15, g4 = lane >> 4, ld = p.Vp + KP;
  const int v = vb * VB + l16;
  const bool on = w * 16 < KP;  // (32 channels: two waves)
  floatx4 S[NT][1], E0[NT];
  floatx8 P[NT][NF];
  float* const ends = BACK ? p.gends : p.ends;
  const int le = BACK ? p.Vp : ld;
  auto place = [&](int n) { return ((int64_t)bh * p.segs + (BACK ? p.segs - 1 - n : n)) * KP; };
  auto load = [&](int n) {
    const int64_t at = place(n);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int k = (w + 4 * i) * 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) E0[i][e] = ends[(at + k + 4 * g4 + e) * le + v];
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int col = f * 32 + g4 * 8;
        if constexpr (BACK) {
#pragma unroll
          for (int e = 0; e < 8; ++e) P[i][f][e] = p.ends[(at + col + e) * ld + p.Vp + k + l16];
        } else {
          P[i][f] = load_row(p.ends + (at + k + l16) * ld + p.Vp + col);
        }
      }
    }
  };
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int k = (w + 4 * i) * 16 + 4 * g4;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      S[i][0][e] = !BACK && p.state && k + e < p.K && v < p.V ? p.state[((int64_t)bh * p.K + k + e) * p.V + v] : 0.f;
  }
  if (on) load(0);
  for (int n = 0; n < p.segs; ++n) {
    Tile<float, 1, VB, KP>& t = s[n & 1];
    const int64_t at = place(n);
    floatx4 o[NT][1];
    Wide<float, 1> a[NF][NT];
    if (on) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int k = (w + 4 * i) * 16 + 4 * g4;
        t.put4(l16, k, S[i][0]);
        o[i][0] = E0[i];
#pragma unroll
        for (int f = 0; f < NF; ++f) a[f][i].p = P[i][f];
#pragma unroll
        for (int e = 0; e < 4; ++e) ends[(at + k + e) * le + v] = S[i][0][e];
      }
      load(min(n + 1, p.segs - 1));  // (in flight through this segment's products)
    }
    lds_barrier();
    if (on) {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const Wide<float, 1> x[1] = {t.frag(l16, f * 32 + g4 * 8)};
        mma(o, a[f], x);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) S[i][0] = o[i][0];
    }
  }
}

// (`both`: the first half of the workgroups one way, the second the other)
template <class E, int KP>
__global__ __launch_bounds__(kThreads) void k_delta_carry(DeltaP<E> p, bool both) {
  __shared__ Tile<float, 1, 16, KP> s[2];
  const int n = both ? gridDim.x / 2 : gridDim.x;
  if ((int)blockIdx.x < n) delta_carry<E, KP, false>(p, blockIdx.x, s);
  else delta_carry<E, KP, true>(p, blockIdx.x - n, s);
}

template <class E, int KP>
struct BackLds {
  // (the adjoints' parts are read in a chunk's first products alone: what the
  // later ones take lies in their place)
  union {
    Tile<E, kState, kVB, KP> s;
    Tile<E, kState, kVB, kC> d[2];
  } x;
  Tile<E, 1, kVB, kC> dyt;
  Tile<E, kState, kVB, kC> qdy;
  Turned<E, KP> kt, qt;
  Spoilt<true> bad;
};
// The adjoints of the memory's states, against time.  Leaves dv, and dR.
template <class E, int KP, Mode MODE, bool WHOLE>
__device__ __forceinline__ void delta_back(const DeltaP<E>& p, BackLds<E, KP>& L, uint32_t block, uint32_t blocks) {
  using W = Split<KP>;
  constexpr int NF = W::NF, NV = W::NV, NKT = W::NKT, NVT = W::NVT;
  auto& x = L.x;
  auto& dyt = L.dyt;
  auto& qdy = L.qdy;
  auto &kt = L.kt, &qt = L.qt;
  Tile<E, kState, kVB, KP>& s = x.s;
  Tile<E, kState, kVB, kC>&du = x.d[0], &dr = x.d[1];
  const W me;
  const int l16 = me.l16, g4 = me.g4;
  const Place at = place_of(p, p.nvb, block, blocks);
  const int live = live_of(p.lengths, at.b, p.T);
  const int v0 = at.vb * kVB;
  const int64_t end = ((int64_t)at.bh * p.segs + at.seg) * KP;
  floatx4 S[NKT][NVT] = {};
  if (MODE == kKeep && p.segs > 1) {
    DGEN_TILES(S[i][j][e] = p.gends[(end + k + e) * p.Vp + v];)
  }
#pragma unroll
  for (int i = 0; i < NKT; ++i)
#pragma unroll
    for (int j = 0; j < NVT; ++j) s.put4(me.tile_v(j) + l16, me.tile_k(i) + 4 * g4, S[i][j]);
  const int c0 = at.seg * p.per, c1 = min(c0 + p.per, p.chunks), cl = min(max((live + kC - 1) / kC, c0), c1);
  const int row = 16 * me.w + l16, rows = 16 * me.w + 4 * g4, col = v0 + l16;
  if constexpr (MODE == kKeep) store_zeros(p.dv, at, cl, c1, p.T, v0, p.V);
  Raw<E> kr[NF], qr[NF];
  Quad<E> dyr[NV];
  const int trow = rows + (l16 & 3), tcol = v0 + (l16 & ~3);  // (turned)
  auto load = [&](int c) {
    const int t0 = c * kC, n = live - t0;
    load_rows<WHOLE>(frames_of(p.k, at.b, at.hk, t0, n), row, g4, p.K, kr);
    load_rows<WHOLE>(frames_of(p.q, at.b, at.hk, t0, n), row, g4, p.K, qr);
    load_values<WHOLE>(frames_of(p.dy, at.b, at.h, t0, n), trow, tcol, p.V, dyr);
  };
  if (c0 < cl) load(cl - 1);
  lds_barrier();
  for (int c = cl - 1; c >= c0; --c) {
    const int t0 = c * kC;
    const int64_t ci = (int64_t)at.bh * p.chunks + c;
    const float* vec = p.vec + ci * kVecs * kC;
    const floatx4 beta = load_vec(vec + kBeta * kC + rows), read = load_vec(vec + kReadK * kC + rows);
    const floatx4 write = load_vec(vec + kWriteK * kC + rows), readq = load_vec(vec + kReadQ * kC + rows);
    const float whole = vec[kInto * kC + kC - 1];
    floatx8 xf[2], mf[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if (f >= me.w / 2) mf[f] = load_row(p.M + ci * kC * kC + (uint32_t)(row * kC + g4 * 8) + f * 32);
    }
    if constexpr (MODE == kKeep) {
      float* out = p.dS + ci * KP * p.Vp;
#pragma unroll
      for (int i = 0; i < NKT; ++i)
#pragma unroll
        for (int j = 0; j < NVT; ++j)
          *reinterpret_cast<floatx4*>(out + (uint32_t)(((me.tile_k(i) >> 2) + g4) * p.Vp + v0 + me.tile_v(j) + l16) * 4) = S[i][j];
    }
    const int n = live - t0;
    Wide<E, 1> kf[NF];
    floatx4 dy[NV];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      kf[f] = exact_of<WHOLE>(kr[f], f * 32 + g4 * 8, p.K, row < n);
      kt.put(row, f * 32 + g4 * 8, kf[f]);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) qt.put(row, f * 32 + g4 * 8, exact_of<WHOLE>(qr[f], f * 32 + g4 * 8, p.K, row < n));
#pragma unroll
    for (int v = 0; v < NV; ++v) dy[v] = turn(quad_of<WHOLE>(dyr[v], tcol + 16 * v, p.V, trow < n), l16);
    // the adjoint of U: what the writes reach after the chunk, then within it
    floatx4 part[2][1][NV] = {}, U[1][NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      dyt.put4(16 * v + l16, rows, dy[v]);
      qdy.put4(16 * v + l16, rows, dy[v] * readq);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      Wide<E, kState> o[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) o[v] = s.frag(16 * v + l16, f * 32 + g4 * 8);
      loads_first();
      const Wide<E, 1> a[1] = {kf[f]};
      mma(part[f & 1], a, o);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) U[0][v] = (part[0][0][v] + part[1][0][v]) * write;
    {
      const floatx4 both[NV] = {dy[0] + U[0][0], dy[1] + U[0][1]};
      L.bad.note(both, me.w);
    }
#pragma unroll
    for (int f = 0; f < 2; ++f)
      if (f >= me.w / 2) xf[f] = load_row(p.XT + ci * kC * kC + (uint32_t)(row * kC + g4 * 8) + f * 32);
    load(max(c - 1, c0));  // (the next chunk's, in flight through this one's products)
    lds_barrier();
    const bool some = L.bad.any(L.bad.notes());
    if (some) L.bad.settle(dyt, U[0], me.w, me.lane, rows);
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if (f < me.w / 2) continue;
      Wide<E, 1> x[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) x[v] = dyt.frag(16 * v + l16, f * 32 + g4 * 8);
      loads_first();
      const Wide<E, kState> a[1] = {wide<E, kState>(mf[f])};
      mma(U, a, x);
    }
    if (some) L.bad.put(U[0], 0.f, l16, rows);
#pragma unroll
    for (int v = 0; v < NV; ++v) du.put4(16 * v + l16, rows, U[0][v]);
    lds_barrier();
    // dR = X^T dU
    floatx4 R[1][NV] = {};
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if (f < me.w / 2) continue;
      Wide<E, kState> x[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) x[v] = du.frag(16 * v + l16, f * 32 + g4 * 8);
      loads_first();
      const Wide<E, kState> a[1] = {wide<E, kState>(xf[f])};
      mma(R, a, x);
    }
    if (some) L.bad.put(R[0], NAN, l16, rows);
#pragma unroll
    for (int v = 0; v < NV; ++v) dr.put4(16 * v + l16, rows, -R[0][v] * beta * read);
    if constexpr (MODE == kKeep) {
      floatx4 dv[NV];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        dv[v] = beta * R[0][v];
        *reinterpret_cast<floatx4*>(p.dR + ci * kC * p.Vp + (uint32_t)((rows >> 2) * p.Vp + col + 16 * v) * 4) = R[0][v];
      }
      store_values(frames_of(p.dv, at.b, at.h, t0, n), trow, p.T - t0, tcol, p.V, l16, dv);
    }
    lds_barrier();
    // the memory's adjoint before the chunk
#pragma unroll
    for (int i = 0; i < NKT; ++i)
#pragma unroll
      for (int j = 0; j < NVT; ++j) S[i][j] *= whole;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int at8 = (f & 1) * 32 + g4 * 8;
      Wide<E, 1> a[NKT];
      Wide<E, kState> x[NVT];
#pragma unroll
      for (int i = 0; i < NKT; ++i) a[i] = f < 2 ? qt.frag(me.tile_k(i), at8, l16) : kt.frag(me.tile_k(i), at8, l16);
#pragma unroll
      for (int j = 0; j < NVT; ++j) x[j] = f < 2 ? qdy.frag(me.tile_v(j) + l16, at8) : dr.frag(me.tile_v(j) + l16, at8);
      loads_first();
      mma(S, a, x);
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < NKT; ++i)
#pragma unroll
      for (int j = 0; j < NVT; ++j) s.put4(me.tile_v(j) + l16, me.tile_k(i) + 4 * g4, S[i][j]);
    lds_barrier();
  }
  if constexpr (MODE == kEnds) {
    DGEN_TILES(p.gends[(end + k + e) * p.Vp + v] = S[i][j][e];)
  }
}

// Both ways at once, as neither waits for the other: the first `forward`
// workgroups with time, the others against it.  kEnds: the segments' ends (those
// with time alone in a call that is not backward).
template <class E, int KP, Mode MODE, bool WHOLE>
__global__ __launch_bounds__(kThreads) void k_delta_both(DeltaP<E> p, uint32_t forward) {
  __shared__ union {
    ChainLds<E, KP, MODE> chain;
    BackLds<E, KP> back;
  } lds;
  if (blockIdx.x < forward) delta_chain<E, KP, MODE, WHOLE>(p, lds.chain, blockIdx.x, forward);
  else delta_back<E, KP, MODE, WHOLE>(p, lds.back, blockIdx.x - forward, gridDim.x - forward);
}

// -------------------------------------------------------------------- grads
// Per chunk and key head: the gradients of q, k, g and beta from the states
// that enter, the adjoints of those that leave, U and dR.
constexpr int kGradParts = 3, kGradThreads = 512;
template <class E, int KP>
struct GradLds {
  union {
    struct {
      Tile<E, kGradParts, KP, 32> s, d;
      Tile<E, kGradParts, kC, 32> u, r;
    } a;
    Tile<E, kGradParts, kC, kC> m[2];
  };
  Turned<E, KP> kt, qt;
  alignas(16) float vec[kVecs * kC], dots[2][5][kC];
  float db[kC], over[8], cross[8][kC];
};

// Eight waves: 16 rows (frames) and half the keys' channels each.
template <class E, int KP, bool WHOLE, bool SHARED>
__global__ __launch_bounds__(kGradThreads) void k_delta_grads(DeltaP<E> p) {
  constexpr int NF = KP / 32, NK = KP / 32;  // fragments, tiles of a wave's channels
  __shared__ GradLds<E, KP> L;
  const int G = p.H / p.shared, c = blockIdx.x % (uint32_t)p.chunks, bg = blockIdx.x / (uint32_t)p.chunks;
  const int b = bg / G, hk = bg % G, t0 = c * kC, live = live_of(p.lengths, b, p.T) - t0;
  const int lane = threadIdx.x & 63, wave = wave_index(), half = wave >> 2, w = half ? 7 - wave : wave, l16 = lane & 15, g4 = lane >> 4;
  const int row = 16 * w + l16, rows = 16 * w + 4 * g4, k0 = half * (KP / 2);
  if (live <= 0) {
    for (int i = threadIdx.x; i < kC * p.K; i += kGradThreads) {
      const int t = t0 + i / p.K, k = i % p.K;
      if (t < p.T) p.dq.row(b, t, hk)[k] = p.dk.row(b, t, hk)[k] = from_f32<E>(0.f);
    }
    for (int i = threadIdx.x; i < kC * p.shared; i += kGradThreads) {
      const int t = t0 + i / p.shared, h = hk * p.shared + i % p.shared;
      if (t < p.T) p.dg.p[b * p.dg.b + t * p.dg.t + h] = p.dbeta.p[b * p.dbeta.b + t * p.dbeta.t + h] = 0.f;
    }
    return;
  }
  const bool on = row < live;
  const int64_t tc = t0 + min(row, live - 1);
  {
    // (the waves of the same rows take the keys and the queries)
    const E* x = half ? p.q.row(b, tc, hk) : p.k.row(b, tc, hk);
    Turned<E, KP>& to = half ? L.qt : L.kt;
    Wide<E, 1> o[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) o[f] = load_exact<WHOLE>(x, f * 32 + g4 * 8, p.K, on);
#pragma unroll
    for (int f = 0; f < NF; ++f) to.put(row, f * 32 + g4 * 8, o[f]);
  }
  // Sum over the 16 lanes of a row.
  auto row_total = [](floatx4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] += dpp<0xB1>(v[e]);
      v[e] += dpp<0x4E>(v[e]);
      v[e] += dpp<0x141>(v[e]);  // (the other four of eight, whose sums are alike)
      v[e] += dpp<0x140>(v[e]);  // (the other eight)
    }
    return v;
  };
  floatx4 DQ[SHARED ? NK : 1] = {}, DK[NK] = {}, dqz[2][NK], qdq = {0, 0, 0, 0}, kdk = {0, 0, 0, 0}, rootk, rootq;
  for (int n = 0; n < (SHARED ? p.shared : 1); ++n) {
    const int h = hk * p.shared + n;
    const int64_t ci = ((int64_t)b * p.H + h) * p.chunks + c;
    const float* const vec = L.vec;
    floatx4 vx4 = {0, 0, 0, 0};
    if (threadIdx.x < kVecs * kC / 4) vx4 = load_vec(p.vec + ci * kVecs * kC + threadIdx.x * 4);
    const float *Sp = p.S + ci * KP * p.Vp, *Dp = p.dS + ci * KP * p.Vp;
    const float *Up = p.U + ci * kC * p.Vp, *Rp = p.dR + ci * kC * p.Vp;
    // A block of 32 values to LDS: a thread reads four rows of one value, four times,
    // the first half of the states and their adjoints, the second of U and of dR.
    const bool first_half = wave < 4;
    const int tv = threadIdx.x & 31, each = first_half ? 8 : 4, quad = (threadIdx.x >> 5) & (each - 1);
    const int quads = first_half ? KP / 4 : kC / 4;
    const float *const from = first_half ? Sp : wave < 6 ? Up : Rp, *const also = first_half ? Dp : from;
    struct Ahead {
      floatx4 a[4], b[4];
      Raw<E> dof, vf;
    } ahead;
    auto load = [&](int v0) {
      Ahead& x = ahead;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t at = (uint32_t)(min(quad + each * e, quads - 1) * p.Vp + v0 + tv) * 4;
        x.a[e] = load_vec(from + at), x.b[e] = load_vec(also + at);
      }
      const int v = v0 + g4 * 8;
      load_raw<WHOLE>(x.dof, p.dy.row(b, tc, h), v, p.V);
      load_raw<WHOLE>(x.vf, p.v.row(b, tc, h), v, p.V);
    };
    const int last = p.Vp - 32;  // (no branches: the last block again where there is none)
    if constexpr (!SHARED) load(0);
    lds_barrier();
    if (threadIdx.x < kVecs * kC / 4) *reinterpret_cast<floatx4*>(&L.vec[threadIdx.x * 4]) = vx4;
    // (dqz: gradients of the queries, and what the keys read; wr: what they
    // wrote; m: of the first half dy U^T, of the second dR U^T)
    floatx4 wr[1][NK] = {}, m[1][4] = {};
#pragma unroll
    for (int k = 0; k < NK; ++k) dqz[0][k] = dqz[1][k] = floatx4{0, 0, 0, 0};
    float sd = 0.f, rv = 0.f;
    for (int v0 = 0; v0 < p.V; v0 += 32) {
      if constexpr (SHARED) load(v0);  // (its registers hold the sums over heads)
      if (v0) lds_barrier();
      const int tcol = tv & ~3;
      if (first_half) {
#pragma unroll
        for (int e = 0; e < KP / 32; ++e) {
          const floatx4 xy = ahead.a[e] * ahead.b[e];
          sd += (xy[0] + xy[1]) + (xy[2] + xy[3]);
          const int r = 4 * (quad + 8 * e) + (tv & 3);
          L.a.s.put4(r, tcol, turn(ahead.a[e], lane));
          L.a.d.put4(r, tcol, turn(ahead.b[e], lane));
        }
      } else {
        auto& to = wave < 6 ? L.a.u : L.a.r;
#pragma unroll
        for (int e = 0; e < 4; ++e) to.put4(4 * (quad + 4 * e) + (tv & 3), tcol, turn(ahead.a[e], lane));
      }
      const Wide<E, 1> of[1] = {exact_of<WHOLE>(ahead.dof, v0 + g4 * 8, p.V, on)};
      const floatx8 vx = floats(exact_of<WHOLE>(ahead.vf, v0 + g4 * 8, p.V, on));
      if constexpr (!SHARED) load(min(v0 + 32, last));  // (in flight through this block's products)
      lds_barrier();
      const Wide<E, kGradParts> rf[1] = {L.a.r.frag(row, g4 * 8)}, uf[1] = {L.a.u.frag(row, g4 * 8)};
      const floatx8 rx = whole_of(rf[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) rv = fmaf(vx[i], rx[i], rv);
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const int r = half * (KP / 2) + 16 * k + l16;
        const Wide<E, kGradParts> o[1] = {L.a.s.frag(r, g4 * 8)}, d[1] = {L.a.d.frag(r, g4 * 8)};
        loads_first();
        floatx4 t[3][1][1] = {{{dqz[0][k]}}, {{dqz[1][k]}}, {{wr[0][k]}}};
        mma(t[1], rf, o);
        mma(t[2], uf, d);
        mma(t[0], of, o);
        dqz[0][k] = t[0][0][0], dqz[1][k] = t[1][0][0], wr[0][k] = t[2][0][0];
      }
      Wide<E, kGradParts> x[4];
#pragma unroll
      for (int tj = 0; tj < 4; ++tj) x[tj] = L.a.u.frag(16 * tj + l16, g4 * 8);
      loads_first();
      if (half) mma(m, rf, x);
      else mma(m, of, x);
    }
    const floatx4 beta = load_vec(vec + kBeta * kC + rows), into = load_vec(vec + kInto * kC + rows);
    const floatx4 rest = load_vec(vec + kRest * kC + rows);
    rootk = load_vec(vec + kRootK * kC + rows);
    rootq = load_vec(vec + kRootQ * kC + rows) * p.scale;
    // M (of the second half A), as m lies in the registers
    const float* const tri = (half ? p.A : p.M) + ci * kC * kC + (uint32_t)(l16 * kC + rows);
    floatx4 t[4];
#pragma unroll
    for (int tj = 0; tj < 4; ++tj)
      if (tj <= w) t[tj] = load_vec(tri + tj * 16 * kC);
    // each frame's share of the gates' gradients: reads of the entering memory,
    // and writes over the chunk's end
    floatx4 enter = {0, 0, 0, 0}, enterk = {0, 0, 0, 0}, written = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      dqz[0][k] *= into;
      dqz[1][k] *= -into;
      wr[0][k] *= rest;
      const floatx4 kk = L.kt.first4(k0 + 16 * k, rows, l16);
      enter += L.qt.first4(k0 + 16 * k, rows, l16) * dqz[0][k];
      enterk += kk * dqz[1][k];
      written += kk * wr[0][k];
    }
    enter = row_total(enter * rootq + beta * rootk * enterk), written = row_total(written * rootk);
    if (l16 == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) L.dots[half][3][rows + e] = enter[e], L.dots[half][4][rows + e] = written[e];
    }
    {
      const float over = wave_sum(sd * vec[kInto * kC + kC - 1]);
      if (lane == 0) L.over[wave] = over;
      rv += __shfl_xor(rv, 16, 64), rv += __shfl_xor(rv, 32, 64);
      if (half == 0 && g4 == 0) L.db[row] = rv;
    }
    {
      // frame to frame: a row's sum over the columns before the lane's, added over
      // the rows from the lane's frame on
      floatx4 before = {0, 0, 0, 0};
      float cross = 0.f;
#pragma unroll
      for (int tj = 0; tj < 4; ++tj) {
        if (tj > w) continue;
        floatx4 x = m[0][tj] * (half ? -t[tj] : t[tj]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = tj < w || l16 <= 4 * g4 + e ? x[e] : 0.f;
        const floatx4 all = row_total(x);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float c = x[e];
          c += dpp<0x111>(c), c += dpp<0x112>(c), c += dpp<0x114>(c), c += dpp<0x118>(c);  // (lanes 1, 2, 4 and 8 before)
          c = before[e] + dpp<0x111>(c);
          if (tj < w || l16 <= 4 * g4 + e) sum += c;
        }
        before += all;
        sum = swap_add32(sum, sum);
        sum = swap_add16(sum, sum);
        cross = g4 == tj ? sum : cross;
      }
      L.cross[wave][lane] = cross;
    }
    // the two triangular matrices by rows, then by columns
#pragma unroll
    for (int tj = 0; tj < 4; ++tj) {
      if (tj > w + 1) continue;  // (neither is read further above the diagonal)
      const int j = 16 * tj + l16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = rows + e;
        const float d = exp_accurate((vec[kGHigh * kC + i] - vec[kGHigh * kC + j]) + (vec[kGLow * kC + i] - vec[kGLow * kC + j]));
        m[0][tj][e] = (half ? j < i : j <= i) ? m[0][tj][e] * (half ? -d : d) : 0.f;
      }
    }
    lds_barrier();
#pragma unroll
    for (int tj = 0; tj < 4; ++tj) {
      if (tj > w + 1 || (tj == w + 1 && (w & 1))) continue;
      const float root = vec[kRootK * kC + 16 * tj + l16];
      L.m[half].put4(rows + (l16 & 3), 16 * tj + (l16 & ~3), turn(m[0][tj] * root, l16));
    }
    lds_barrier();
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if (f > w / 2) break;
      const int col = f * 32 + g4 * 8;
      const Wide<E, kGradParts> o[2] = {L.m[0].frag(row, col), L.m[1].frag(row, col)};
      Wide<E, 1> x[NK];
#pragma unroll
      for (int k = 0; k < NK; ++k) x[k] = L.kt.frag(k0 + 16 * k, col, l16);
      loads_first();
      mma(dqz, o, x);
    }
    lds_barrier();
#pragma unroll
    for (int tj = 0; tj < 4; ++tj) {
      if (tj > w + 1 || (tj == w + 1 && (w & 1))) continue;
      L.m[half].put4(16 * tj + l16, rows, m[0][tj] * (half ? beta * rootk : rootq));
    }
    lds_barrier();
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if (f < w / 2) continue;
      const int col = f * 32 + g4 * 8;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const Wide<E, kGradParts> o[1] = {L.m[y].frag(row, col)};
        Wide<E, 1> x[NK];
#pragma unroll
        for (int k = 0; k < NK; ++k) x[k] = y ? L.kt.frag(k0 + 16 * k, col, l16) : L.qt.frag(k0 + 16 * k, col, l16);
        loads_first();
        mma(wr, o, x);
      }
    }
    floatx4 q = {0, 0, 0, 0}, kr = {0, 0, 0, 0}, kw = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const floatx4 kk = L.kt.first4(k0 + 16 * k, rows, l16);
      q += L.qt.first4(k0 + 16 * k, rows, l16) * dqz[0][k];
      kr += kk * dqz[1][k];
      kw += kk * wr[0][k];
      if constexpr (SHARED) DQ[k] += dqz[0][k];
      DK[k] += beta * dqz[1][k] + wr[0][k];
    }
    q = row_total(q), kr = row_total(kr), kw = row_total(kw);
    if (l16 == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        L.dots[half][0][rows + e] = q[e], L.dots[half][1][rows + e] = kr[e], L.dots[half][2][rows + e] = kw[e];
    }
    lds_barrier();
    q = (load_vec(&L.dots[0][0][rows]) + load_vec(&L.dots[1][0][rows])) * rootq;
    kr = (load_vec(&L.dots[0][1][rows]) + load_vec(&L.dots[1][1][rows])) * rootk;
    kw = (load_vec(&L.dots[0][2][rows]) + load_vec(&L.dots[1][2][rows])) * rootk;
    qdq += q, kdk += beta * kr + kw;
    if (wave == 0) {
      const float read = (L.dots[0][1][lane] + L.dots[1][1][lane]) * vec[kRootK * kC + lane];
      float a = L.dots[0][3][lane] + L.dots[1][3][lane], out = L.dots[0][4][lane] + L.dots[1][4][lane];
#pragma unroll
      for (int k = 1; k < 64; k *= 2) {
        const float later = __shfl_down(a, k, 64), earlier = __shfl_up(out, k, 64);
        a += lane + k < 64 ? later : 0.f;
        out += lane >= k ? earlier : 0.f;
      }
      out = __shfl_up(out, 1, 64);
      a += lane > 0 ? out : 0.f;
      float cross = 0.f, over = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) cross += L.cross[k][lane], over += L.over[k];
      a += cross + over;
      const int t = t0 + lane;
      if (t < p.T) {
        const bool in = lane < live;
        p.dg.p[b * p.dg.b + t * p.dg.t + h] = in ? a : 0.f;
        p.dbeta.p[b * p.dbeta.b + t * p.dbeta.t + h] = in ? L.db[lane] + read : 0.f;
      }
    }
  }
  // through the scales and the norms: x^ = x r, r = 1 / sqrt(|x|^2 + eps)
  floatx4 backq = {0, 0, 0, 0}, backk = {0, 0, 0, 0};
  if (p.normalize) {
    const floatx4 r = load_vec(&L.vec[kRootQ * kC + rows]);
    backq = qdq * r * r, backk = kdk * rootk * rootk;
  }
  const int trow = rows + (l16 & 3);
  E *oq = p.dq.row(b, t0 + trow, hk), *ok = p.dk.row(b, t0 + trow, hk);
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    const int col = k0 + 16 * k, at = col + (l16 & ~3);
    floatx4 x = turn(rootq * (SHARED ? DQ[SHARED ? k : 0] : dqz[0][k]) - L.qt.first4(col, rows, l16) * backq, l16);
    floatx4 y = turn(rootk * DK[k] - L.kt.first4(col, rows, l16) * backk, l16);
    if (trow >= live) x = y = floatx4{0.f, 0.f, 0.f, 0.f};
    const float xs[4] = {x[0], x[1], x[2], x[3]}, ys[4] = {y[0], y[1], y[2], y[3]};
    if (t0 + trow >= p.T) continue;
    store_four(oq + at, p.K - at, xs);
    store_four(ok + at, p.K - at, ys);
  }
}

// --------------------------------------------------------------- few frames
// Frame by frame: 32 values of one head a workgroup, a thread holds four of
// them for KP / 32 of the keys' channels.  Bound by the sums' vector instructions
// (the next frame's operands loaded ahead were no faster).
template <class E, int KP>
__global__ __launch_bounds__(kThreads) void k_delta_step(DeltaP<E> p) {
  constexpr int NR = KP / 32;
  __shared__ float kq[2][2][KP];
  __shared__ alignas(16) float red[2][4][8][12];
  const int nvb = (p.V + 31) / 32, vb = blockIdx.x % (uint32_t)nvb, bh = blockIdx.x / (uint32_t)nvb;
  const int b = bh / p.H, h = bh % p.H, hk = h / p.shared, live = live_of(p.lengths, b, p.T);
  const int lane = threadIdx.x & 63, w = wave_index(), l8 = lane & 7, rt = threadIdx.x >> 3;
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
    float o[12] = {};
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const float k = kq[at][0][rt + 32 * i], q = kq[at][1][rt + 32 * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(k, S[i][e], o[e]), o[4 + e] = fmaf(q, S[i][e], o[4 + e]);
      o[8] = fmaf(k, q, o[8]), o[9] = fmaf(k, k, o[9]), o[10] = fmaf(q, q, o[10]);
    }
    // (each exchange halves the sums a lane goes on with)
    float six[6], three[3];
#pragma unroll
    for (int e = 0; e < 6; ++e) six[e] = swap_add32(o[e], o[e + 6]);
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      three[e] = swap_add16(six[e], six[e + 3]);
      three[e] += dpp<0x128>(three[e]);  // (lanes 8 apart)
      if (!(lane & 8)) red[at][w][l8][3 * (lane >> 4) + e] = three[e];
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

template <class E, int KP, bool WHOLE>
void delta_chains(const DeltaP<E>& p, const DeltaPlan& o, int64_t bh, bool backward, hipStream_t st) {
  auto grid = [](int64_t n) { return dim3((unsigned)n); };
  const int64_t blocks = bh * o.nvb * o.segs, carry = bh * (p.Vp / 16);
  if (o.segs > 1) {
    const int64_t ends = bh * o.segs * (o.nvb + (KP + kVB - 1) / kVB);
    k_delta_both<E, KP, kEnds, WHOLE><<<grid(ends + (backward ? blocks : 0)), kThreads, 0, st>>>(p, (uint32_t)ends);
    k_delta_carry<E, KP><<<grid(backward ? 2 * carry : carry), kThreads, 0, st>>>(p, backward);
  }
  if (backward) k_delta_both<E, KP, kKeep, WHOLE><<<grid(2 * blocks), kThreads, 0, st>>>(p, (uint32_t)blocks);
  else k_delta_forward<E, KP, WHOLE><<<grid(blocks), kThreads, 0, st>>>(p);
}

template <class E, int KP, bool WHOLE>
void delta_kernels(const DeltaP<E>& p, const DeltaPlan& o, int64_t bh, bool backward, hipStream_t st) {
  auto grid = [](int64_t n) { return dim3((unsigned)n); };
  k_delta_prepare<E, KP, WHOLE><<<grid(bh * o.chunks), kThreads, 0, st>>>(p);
  delta_chains<E, KP, WHOLE>(p, o, bh, backward, st);
  if (backward) {
    const dim3 n = grid(bh / p.shared * o.chunks);
    p.shared > 1 ? k_delta_grads<E, KP, WHOLE, true><<<n, kGradThreads, 0, st>>>(p)
                 : k_delta_grads<E, KP, WHOLE, false><<<n, kGradThreads, 0, st>>>(p);
  }
}

template <class E, int KP>
void delta_launch(const dgen_hip_delta& a, bool backward, hipStream_t st) {
  const DeltaPlan o = delta_plan(a, backward);
  DeltaP<E> p;
  auto in = [](const dgen_hip_heads& h) { return Heads<const E>{(const E*)h.data, h.stride_b, h.stride_t, h.stride_h}; };
  auto out = [](const dgen_hip_heads& h) { return Heads<E>{(E*)h.data, h.stride_b, h.stride_t, h.stride_h}; };
  auto gates = [](const dgen_hip_seq& s) { return Gates{(float*)s.data, s.stride_b, s.stride_t}; };
  p.q = in(a.q), p.k = in(a.k), p.v = in(a.v), p.dy = in(a.dy);
  p.y = out(a.y), p.dq = out(a.dq), p.dk = out(a.dk), p.dv = out(a.dv);
  p.g = gates(a.g), p.beta = gates(a.beta), p.dg = gates(a.dg), p.dbeta = gates(a.dbeta);
  p.lengths = a.lengths, p.state = a.state, p.state_out = a.state_out;
  p.scale = a.scale, p.normalize = a.normalize;
  p.T = (int)a.T, p.H = (int)a.heads, p.shared = (int)(a.heads / a.key_heads), p.K = (int)a.K, p.V = (int)a.V;
  p.Vp = (int)(o.nvb * kVB);
  p.chunks = (int)o.chunks, p.nvb = (int)o.nvb, p.segs = (int)o.segs, p.per = (int)o.per;
  auto at = [&](int64_t off) { return (float*)((char*)a.workspace + off); };
  p.X = at(o.X), p.M = at(o.M), p.XT = backward ? at(o.XT) : nullptr, p.A = at(o.A), p.vec = at(o.vec), p.S = at(o.S), p.dS = at(o.dS), p.U = at(o.U), p.dR = at(o.dR);
  p.ends = at(o.ends), p.gends = at(o.gends);
  const int64_t bh = a.batch * a.heads;
  if (delta_steps(a, backward))
    k_delta_step<E, KP><<<dim3((unsigned)(bh * ((a.V + 31) / 32))), kThreads, 0, st>>>(p);
  else if (a.K % 8 == 0 && a.V % 8 == 0) delta_kernels<E, KP, true>(p, o, bh, backward, st);
  else delta_kernels<E, KP, false>(p, o, bh, backward, st);
}

template <class E>
void delta_width(const dgen_hip_delta& a, bool backward, hipStream_t st) {
  if (a.K <= 32) delta_launch<E, 32>(a, backward, st);
  else if (a.K <= 64) delta_launch<E, 64>(a, backward, st);
  else delta_launch<E, 128>(a, backward, st);
}

}  // namespace

}  // namespace dgen
