// Gated feed-forward block: h = act(x Wg) * (x Wu), forward and backward, on
// the bf16 matrix cores.
//
// Products, by use:
// - forward: a tile's columns are groups of gate and up columns side by side,
//   so a wave holds both projections of the same outputs and applies the
//   activation and the product in registers;
// - backward, projections again: the same, but the epilogue reads dh and
//   writes dg = dh u act'(g) and du = dh act(g);
// - dx = dg Wg^T + du Wu^T: one product over 2 x hidden;
// - dWg = x^T dg, dWu = x^T du: products over the rows.
// Where tiles alone do not fill the chip, the reductions of dx and dW are cut
// into runs whose parts are added in order.
//
// bfloat16 operands multiply as they are, accumulated in fp32.  dg and du are
// rounded to bfloat16 between the products: gradients of 32000 x 1024 x 2816 are
// then off by 0.0023 of their norm, for 0.0017 by the rounding of the results
// alone.  In two bfloat16 parts each, which would leave that, the products of dx
// and dW would be twice as many (690 us more of 1200).  fp32
// operands are split exactly into three bfloat16 parts on the way to LDS, and
// the six partial products down to 2^-16 are accumulated in fp32, as accurate
// as fp32 products (see k_gemm.hip).  An infinity, or a number past the largest
// bfloat16, has no such parts: its products come out as NaN, and what does is
// formed again from the operands as they are.
//
// Three kernels: k_glu_direct, bfloat16, 256 x 256 tiles on operands that lie
// in whole 16-byte chunks (packed first where they do not); k_glu, operands of
// any layout and type, 128 x 128 (fp32) or 64 x 128 tiles; k_glu_few, a few
// rows.
//
// The matrix instruction's row index is the output's column, so a lane ends
// with four consecutive columns of one output row.
//
// Measured on operands that the caches do not hold (large library products:
// 1227 TFLOP/s of bf16, 154 of fp32): bf16, 32000 x 1024 x 2816 backward:
// projections with their gradients 506 us, dx 342, dW 346, its parts 22 (369
// GFLOP each, 0.73, 1.08 and 1.07 PFLOP/s; the projections' 32 stages a tile
// leave its 192 KB of dh, dg and du and their activations in the open); 20000
// rows forward 257 us, 0.90 PFLOP/s.  fp32, 8003 x 512 x 1365 forward 180 us,
// 124 TFLOP/s (calls in a row: 164, 136); 16000 x 512 x 1408 backward 359, 266
// and 312 us, 128 to 173 TFLOP/s (bound by the six products and the splitting).
// bf16, 8 x 512 x 1408 forward: 7 us (weights in the caches: 5), the latency of
// the launch and of one round of loads.  Between these sizes k_glu's loop, one
// LDS buffer and two barriers a step, and grids of fewer tiles than CUs are
// what bounds: bf16, 2000 x 512 x 1408 forward 20 us, 5 by its products,
// backward 23, 18 and 36 us and 10 of joins, 14 by its products; 61 x 256 x 1792
// backward four launches of 4 to 11 us; fp32, 500 x 512 x 1408 forward 28 us, 7
// by its products, the 16 steps of one tile.
#include "seq.h"

namespace dgen {

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;

enum Use { kForward, kProject, kDx, kDw };

template <class E>
struct GluP {
  // operand rows along the output's columns (n) and rows (m): two matrices
  // each (gate, up), used as columns side by side, as segments of the reduction
  // or as two products
  const E *n0, *n1, *m0, *m1;
  int64_t nld0, nld1, mld0, mld1;
  int64_t M, N, K;  // output rows, columns (of one matrix), reduction length
  E *out0, *out1;
  int64_t old0, old1;
  const E* dh;
  int64_t dhld;
  float* parts;     // [splits][2][M][N]
  int64_t span;     // reduction length of a split
  int act;
  uint32_t tiles_n, tiles_m, splits;
};

// ------------------------------------------------------------- activation
// GELU, tanh form: 0.5 v (1 + tanh(k (v + c v^3))) = v sigmoid(2 k (v + c v^3)).
constexpr float kGeluA = 1.5957691216057308f, kGeluB = 0.044715f;
__device__ __forceinline__ float act_of(int act, float v, float& slope) {
  if (act == DGEN_HIP_SILU) {
    const float p = sigmoid(v);
    slope = silu_grad(v, p);
    return v * p;
  }
  // (past 16 the sigmoid is 0 or 1 to the last bit, and so is the slope: the
  // clamp keeps the powers of v from overflowing into 0 times infinity)
  const float c = v > 16.f ? 16.f : v < -16.f ? -16.f : v;  // (NaN stays)
  const float c2 = c * c, p = sigmoid(kGeluA * c * fmaf(kGeluB, c2, 1.f));
  slope = p * fmaf(c * (1.f - p), kGeluA * fmaf(3.f * kGeluB, c2, 1.f), 1.f);
  return v * p;
}

// ---------------------------------------------------------------- staging
// 8 consecutive k of one row as a 16-byte chunk per plane.
template <class E>
constexpr int planes() { return sizeof(E) == 2 ? 1 : 3; }

struct Chunk {
  uint32_t w[4];
};

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)from_f32<bf16>(a).v | (uint32_t)from_f32<bf16>(b).v << 16;
}
__device__ __forceinline__ float part_of(uint32_t w, int hi) { return __uint_as_float(hi ? w & 0xffff0000u : w << 16); }

// v = h + m + l exactly in bfloat16 parts, two values at a time.
__device__ __forceinline__ void split2(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
  h = pack2(a, b);
  const float ra = a - part_of(h, 0), rb = b - part_of(h, 1);
  m = pack2(ra, rb);
  l = pack2(ra - part_of(m, 0), rb - part_of(m, 1));
}

template <class E, int V>
struct __attribute__((packed, aligned(alignof(E)))) Vec {
  E e[V];
};

// LDS place of chunk c (8 k's) of row r, in chunks of 16 bytes: rows of BK
// k's, the chunks of a row permuted so that neither the fragments' reads (32
// consecutive rows, one chunk) nor the transposing writes (rows 4 or 8 apart)
// meet in a bank.
template <int BK>
__device__ __forceinline__ int place(int r, int c) {
  constexpr int C = BK / 8;
  if constexpr (C == 8) return r * 8 + (c ^ ((r ^ (r >> 3)) & 7));
  else return r * C + (c ^ (((r >> 1) ^ (r >> 3)) & (C - 1)));
}

// One operand's tile of R rows x BK, between memory and LDS.  KC: k is the
// contiguous axis in memory.
template <class E, int R, int BK, bool KC>
struct Stage {
  static constexpr int P = planes<E>();
  static constexpr int kPer = R * BK / kThreads;                     // elements a thread carries
  static constexpr int kMaxV = 16 / (int)sizeof(E);
  static constexpr int V = KC ? 8 : (kPer / 8 < kMaxV ? kPer / 8 : kMaxV);  // elements of a load
  static constexpr int U = kPer / (8 * (KC ? 1 : V));                // chunks (KC) or 8 x V blocks a thread
  static_assert(kPer % 8 == 0 && V >= 1 && U >= 1, "tile too small");
  E v[U][KC ? 1 : 8][V];

  // at(r): the address of row r of the tile (KC), or of element (r, k = 0)
  // (!KC), clamped into the operand; inside(r): how many rows from r on lie in
  // it.  `whole`: the tile is inside the operand (uniform), so that the loads
  // are whole and without a branch; else zeros stand for what lies outside.
  // (Rows past the end of a k-contiguous operand repeat its last one: their
  // results are not stored.)
  template <class At, class Inside>
  __device__ __forceinline__ void load(At at, Inside inside, int64_t ld, int64_t k0, int64_t kend, bool whole) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = threadIdx.x + u * kThreads;
      const int r = KC ? i / (BK / 8) : (i % (R / V)) * V;
      const int64_t k = k0 + (KC ? i % (BK / 8) : i / (R / V)) * 8;
      const E* p = at(r);
      if (whole) {
#pragma unroll
        for (int q = 0; q < (KC ? 1 : 8); ++q) {
          const Vec<E, V> t = *reinterpret_cast<const Vec<E, V>*>(KC ? p + k : p + (k + q) * ld);
#pragma unroll
          for (int e = 0; e < V; ++e) v[u][q][e] = t.e[e];
        }
      } else {
        const int64_t rows = inside(r);
#pragma unroll
        for (int q = 0; q < (KC ? 1 : 8); ++q)
          get(KC ? p + k : p + (k + q) * ld, KC ? kend - k : k + q < kend ? rows : 0, v[u][q]);
      }
    }
  }
  __device__ __forceinline__ static void get(const E* p, int64_t valid, E (&o)[V]) {
    if (valid >= V) {
      const Vec<E, V> t = *reinterpret_cast<const Vec<E, V>*>(p);
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = t.e[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = e < valid ? p[e] : E{};
    }
  }

  __device__ __forceinline__ void store(Chunk* lds) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = threadIdx.x + u * kThreads;
#pragma unroll
      for (int b = 0; b < (KC ? 1 : V); ++b) {
        const int r = KC ? i / (BK / 8) : (i % (R / V)) * V + b;
        const int c = KC ? i % (BK / 8) : i / (R / V);
        Chunk o[P];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const E lo = KC ? v[u][0][KC ? 2 * q : 0] : v[u][KC ? 0 : 2 * q][KC ? 0 : b];
          const E hi = KC ? v[u][0][KC ? 2 * q + 1 : 0] : v[u][KC ? 0 : 2 * q + 1][KC ? 0 : b];
          if constexpr (P == 1) o[0].w[q] = (uint32_t)lo.v | (uint32_t)hi.v << 16;
          else split2(lo, hi, o[0].w[q], o[1].w[q], o[2].w[q]);
        }
#pragma unroll
        for (int pl = 0; pl < P; ++pl) lds[pl * (R * BK / 8) + place<BK>(r, c)] = o[pl];
      }
    }
  }
};

template <class E, int W>
__device__ __forceinline__ void put_four(E* p, int64_t valid, const float (&o)[W]) {
  store_four(p, (int)(valid < 4 ? valid : 4), o);
}

// A wave's accumulators to memory; its tile starts at output row mb, column nb.
template <class E, int USE, int NF, int MF>
__device__ __forceinline__ void finish(const GluP<E>& p, const floatx16 (&acc)[NF][MF], int64_t mb, int64_t nb,
                                       uint32_t split, uint32_t mat) {
  constexpr bool PAIR = USE == kForward || USE == kProject;
  const int lane = threadIdx.x & 63;
  // register 4 q + e of acc[i][j]: output column 8 q + 4 (lane / 32) + e of
  // the fragment's 32, row lane % 32
  const int r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int j = 0; j < MF; ++j) {
    const int64_t m = mb + j * 32 + r;
    if (m >= p.M) continue;
#pragma unroll
    for (int i = 0; i < (PAIR ? NF / 2 : NF); ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = nb + i * 32 + 8 * q + 4 * h;
        if (n >= p.N) continue;
        float a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = acc[i][j][4 * q + e];
        if constexpr (PAIR) {
          float u[4], slope;
#pragma unroll
          for (int e = 0; e < 4; ++e) u[e] = acc[i + NF / 2][j][4 * q + e];
          if constexpr (USE == kForward) {
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = act_of(p.act, a[e], slope) * u[e];
            put_four(p.out0 + m * p.old0 + n, p.N - n, a);
          } else {
            float d[4];
            load_four(p.dh + m * p.dhld + n, (int)(p.N - n < 4 ? p.N - n : 4), d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = act_of(p.act, a[e], slope);
              a[e] = d[e] * u[e] * slope;
              u[e] = d[e] * v;
            }
            put_four(p.out0 + m * p.old0 + n, p.N - n, a);
            put_four(p.out1 + m * p.old1 + n, p.N - n, u);
          }
        } else if constexpr (USE == kDx) {
          if (p.parts) put_four(p.parts + ((int64_t)split * p.M + m) * p.N + n, p.N - n, a);
          else put_four(p.out0 + m * p.old0 + n, p.N - n, a);
        } else {
          if (p.parts) {
            put_four(p.parts + ((int64_t)split * 2 + mat) * p.M * p.N + m * p.N + n, p.N - n, a);
          } else {
            put_four(mat ? p.out1 + m * p.old1 + n : p.out0 + m * p.old0 + n, p.N - n, a);
          }
        }
      }
  }
}

// fp32 products that came out as NaN once more, on the vector unit, from the
// operands in memory.  cols(i, k) and rows(j, k): the lane's address of the
// elements at k of the first of fragment i's columns (consecutive ones nstep()
// apart, `left(i)` of them in the operand) and of its row of fragment j;
// steps(f) calls f(k from, k to, second segment) for the wave's reduction.
// For infinities; a tile without NaN passes by.  (Calls of 8003 x 512 x 1365
// forward: 164 us, with an infinity in a row 1.4 ms, of NaN all over 6.8.)
template <int NF, int MF, class Cols, class Rows, class Left, class Stride, class Steps>
__device__ __forceinline__ void again(floatx16 (&acc)[NF][MF], Cols cols, Rows rows, Left left, Stride nstep,
                                      Steps steps) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
      for (int r = 0; r < 16; r += 2) bad |= __builtin_isunordered(acc[i][j][r], acc[i][j][r + 1]);
  if (!__any(bad)) return;
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // (four at a time: few registers beside the accumulators)
        const int64_t last = left(i) - 1;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        steps([&](int64_t from, int64_t to, bool second) {
#pragma unroll 1
          for (int64_t k = from; k < to; ++k) {
            const float m = *rows(j, k, second), *const p = cols(i, k, second);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int64_t c = 8 * q + e;
              sum[e] = fmaf(p[(c < last ? c : last) * nstep(second)], m, sum[e]);
            }
          }
        });
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = acc[i][j][4 * q + e];
          acc[i][j][4 * q + e] = v != v ? sum[e] : v;
        }
      }
}

// ----------------------------------------------------------------- kernel
// Tile of this workgroup.  Consecutive workgroups go to the eight XCDs in
// turn, so each XCD takes a run of consecutive tiles; a run goes through
// groups of four column tiles, row tiles in turn, so that the tiles an XCD
// works on at a time (32 of the large ones, one a CU) share eight row tiles
// and four column tiles in its L2.
struct TileAt {
  uint32_t n, m, split, mat;
};
template <int USE, class Params>
__device__ __forceinline__ TileAt tile_at(const Params& p) {
  const uint32_t total = gridDim.x, each = total / 8, more = total % 8;
  const uint32_t xcd = blockIdx.x & 7, id = xcd * each + (xcd < more ? xcd : more) + (blockIdx.x >> 3);
  const uint32_t plane = p.tiles_n * p.tiles_m, rest = id / plane, at = id - rest * plane;
  const uint32_t group = at / (4 * p.tiles_m), in = at - group * 4 * p.tiles_m;
  const uint32_t wide = p.tiles_n - group * 4 < 4 ? p.tiles_n - group * 4 : 4;
  return {group * 4 + in % wide, in / wide, USE == kDw || USE == kDx ? rest % p.splits : 0, USE == kDw ? rest / p.splits : 0};
}

// BM x BN: output rows and operand columns of a tile; WM x WN: of a wave.
// (fp32 tiles of 64 rows fit four waves a SIMD but for again's registers.)
template <class E, int BM, int BN, int WM, int WN, int BK, int USE>
__global__ __launch_bounds__(kThreads, sizeof(E) == 2 ? 1 : BM == 64 && USE != kDw ? 4 : 2) void k_glu(GluP<E> p) {
  constexpr int P = planes<E>(), NF = WN / 32, MF = WM / 32;
  constexpr bool PAIR = USE == kForward || USE == kProject;
  constexpr bool NKC = USE == kDx, MKC = USE != kDw;
  static_assert((BM / WM) * (BN / WN) == kThreads / 64, "four waves");
  constexpr int NCH = P * BN * BK / 8, MCH = P * BM * BK / 8;
  __shared__ Chunk lds[NCH + MCH];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wn = wave % (BN / WN), wm = wave / (BN / WN);
  const TileAt t = tile_at<USE>(p);
  const uint32_t split = t.split, mat = t.mat;
  constexpr int COLS = PAIR ? BN / 2 : BN;  // output columns of a tile
  const int64_t n0 = (int64_t)t.n * COLS, m0 = (int64_t)t.m * BM;
  const int64_t kfrom = USE == kDw ? split * p.span : 0;
  const int64_t kend = USE == kDw && kfrom + p.span < p.K ? kfrom + p.span : p.K;
  const int64_t kblocks = kend > kfrom ? (kend - kfrom + BK - 1) / BK : 0;
  const int64_t all = USE == kDx ? 2 * kblocks : kblocks;
  // dx over few tiles: a run of the steps each
  const int64_t first = USE == kDx ? split * p.span : 0;
  const int64_t steps = USE == kDx && first + p.span < all ? first + p.span : all;

  Stage<E, BN, BK, NKC> sn;
  Stage<E, BM, BK, MKC> sm;
  auto load = [&](int64_t step) {
    const bool second = USE == kDx && step >= kblocks;
    const int64_t k0 = kfrom + (second ? step - kblocks : step) * BK;
    const bool n_second = second || (USE == kDw && mat);
    const E *nb = n_second ? p.n1 : p.n0, *mb = second ? p.m1 : p.m0;
    const int64_t nld = n_second ? p.nld1 : p.nld0, mld = second ? p.mld1 : p.mld0;
    // a wave's WN columns are WN / 2 of gate, then the same of up
    auto column = [&](int r) { return PAIR ? n0 + r / WN * (WN / 2) + r % (WN / 2) : n0 + r; };
    auto nat = [&](int r) {
      const int64_t c = column(r), n = c < p.N ? c : p.N - 1;
      if constexpr (PAIR) return ((r % WN) >= WN / 2 ? p.n1 : p.n0) + n;
      else return NKC ? nb + n * nld : nb + n;
    };
    auto nin = [&](int r) { return p.N - column(r); };
    auto mat_at = [&](int r) {
      const int64_t m = m0 + r < p.M ? m0 + r : p.M - 1;
      return MKC ? mb + m * mld : mb + m;
    };
    auto min = [&](int r) { return p.M - (m0 + r); };
    const bool ks = k0 + BK <= kend;
    if constexpr (PAIR) {
      // (the two matrices may have different strides: the block's own is used)
      const bool up = ((threadIdx.x % (BN / Stage<E, BN, BK, NKC>::V)) * Stage<E, BN, BK, NKC>::V) % WN >= WN / 2;
      sn.load(nat, nin, up ? p.nld1 : p.nld0, k0, kend, ks && n0 + COLS <= p.N);
    } else {
      sn.load(nat, nin, nld, k0, kend, ks && (NKC || n0 + COLS <= p.N));
    }
    sm.load(mat_at, min, mld, k0, kend, ks && (MKC || m0 + BM <= p.M));
  };

  floatx16 acc[NF][MF] = {};
  auto compute = [&](const Chunk* b) {
#pragma unroll
    for (int ks = 0; ks < BK / 16; ++ks) {
      bf16x8 nf[NF][P], mf[MF][P];
      const int c = ks * 2 + (lane >> 5), r = lane & 31;
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int pl = 0; pl < P; ++pl)
          nf[i][pl] = __builtin_bit_cast(bf16x8, b[pl * (BN * BK / 8) + place<BK>(wn * WN + i * 32 + r, c)]);
#pragma unroll
      for (int j = 0; j < MF; ++j)
#pragma unroll
        for (int pl = 0; pl < P; ++pl)
          mf[j][pl] = __builtin_bit_cast(bf16x8, b[NCH + pl * (BM * BK / 8) + place<BK>(wm * WM + j * 32 + r, c)]);
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MF; ++j) {
          if constexpr (P == 1) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(nf[i][0], mf[j][0], acc[i][j], 0, 0, 0);
          } else {
            // smallest products first
#define DGEN_PART(a, b2) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(nf[i][a], mf[j][b2], acc[i][j], 0, 0, 0)
            DGEN_PART(2, 0);
            DGEN_PART(0, 2);
            DGEN_PART(1, 1);
            DGEN_PART(1, 0);
            DGEN_PART(0, 1);
            DGEN_PART(0, 0);
#undef DGEN_PART
          }
        }
    }
  };

  if (steps > first) load(first);
  for (int64_t s = first; s < steps; ++s) {
    __syncthreads();
    sn.store(lds);
    sm.store(lds + NCH);
    __syncthreads();
    if (s + 1 < steps) load(s + 1);
    __builtin_amdgcn_sched_barrier(0);  // the loads before the products, which they land behind
    compute(lds);
  }

  const int64_t mb = m0 + wm * WM, nb = n0 + (PAIR ? wn * (WN / 2) : wn * WN);
  if constexpr (P == 3) {
    // the first column of fragment i for this lane (register 4 q + e: column 8 q + e from there)
    auto column = [&](int i) { return nb + (PAIR ? i % (NF / 2) : i) * 32 + 4 * (lane >> 5); };
    auto from = [&](int i) { return column(i) < p.N ? column(i) : p.N - 1; };
    again<NF, MF>(
        acc,
        [&](int i, int64_t k, bool second) {
          const bool up = second || (PAIR ? i >= NF / 2 : USE == kDw && mat);
          const int64_t ld = up ? p.nld1 : p.nld0;
          return (up ? p.n1 : p.n0) + (NKC ? from(i) * ld + k : k * ld + from(i));
        },
        [&](int j, int64_t k, bool second) {
          const int64_t r = mb + j * 32 + (lane & 31), m = r < p.M ? r : p.M - 1, ld = second ? p.mld1 : p.mld0;
          return (second ? p.m1 : p.m0) + (MKC ? m * ld + k : k * ld + m);
        },
        [&](int i) { return p.N - from(i); },
        [&](bool second) { return NKC ? (second ? p.nld1 : p.nld0) : 1; },
        [&](auto f) {
          for (int64_t s = first; s < steps; ++s) {
            const bool second = USE == kDx && s >= kblocks;
            const int64_t k = kfrom + (second ? s - kblocks : s) * BK;
            f(k, k + BK < kend ? k + BK : kend, second);
          }
        });
  }
  finish<E, USE, NF, MF>(p, acc, mb, nb, split, mat);
}

// ------------------------------------------------------- packed operands
// Operand tiles are copied global -> LDS by the load-to-LDS instructions, as
// they lie in memory: 256 x 256 outputs a workgroup of eight waves, 128 x 64 a
// wave (128 accumulators a lane; two waves a SIMD cover each other's LDS reads
// and barriers), stages of 32 k's in four LDS buffers, two to three of them in
// flight.  An operand that is contiguous along its rows is read with the
// transposing LDS load.  Chunks of 16 bytes are permuted within their LDS rows
// through the global addresses, so that the fragments' reads spread over the
// banks: k-contiguous rows (four chunks) by row / 2, row-contiguous k's (32
// chunks) by twice the k.  Results go to memory through LDS in whole rows of
// the tile (stored from the accumulators' layout, 8 bytes to each of 32 rows, a
// tile took 40 us).
constexpr int kDT = 256, kDK = 32, kDThreads = 512, kDChunks = kDT * kDK / 8;  // chunks of an operand's stage

struct GluD {
  const bf16 *n0, *n1, *m0, *m1;  // operands along columns and rows, gate and up
  int64_t nld, mld;               // row strides
  int64_t nx, mx;                 // readable extent of the axis that is not reduced (k-contiguous:
                                  // rows; else columns, a multiple of 8)
  int64_t M, N, K;                // results; reduction of a segment, a multiple of 32
  bf16 *out0, *out1;
  int64_t old0, old1;
  int64_t om, on;                 // project: extent of dg and du (zero past M, N)
  const bf16* dh;
  int64_t dhld;
  float* parts;                   // [splits][mats][M][N] (dx may do without: to out)
  int64_t span;                   // of a split: rows (dW, a multiple of 32) or stages (dx)
  int act, dh_copied;             // dh lies in whole chunks: copied to LDS too
  uint32_t tiles_n, tiles_m, splits;
};

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;

// 16 bytes a lane from `g` to LDS byte `at` + 16 lane (at: uniform).  In
// assembly, since the compiler would wait for every copy in flight before any
// transposing LDS read; the kernel waits for its copies itself.  (M0 is no
// register that the compiler allocates, of which it warns, but one that it
// writes for its own instructions: naming it keeps them apart from these.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy_to_lds(const bf16* g, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(
                   __builtin_amdgcn_readfirstlane(at)),
               "v"(g)
               : "memory", "m0");
}
#pragma clang diagnostic pop

template <bool KC>
__device__ __forceinline__ int chunk_swizzle(int row) { return KC ? (row >> 1) & 3 : (row & 3) << 1; }

// Fragment of 32 rows from `r0` on at k-step ks of a stage.
template <bool KC>
__device__ __forceinline__ bf16x8 fragment(const uint4* b, int r0, int ks, int lane) {
  constexpr int C = kDT / 8;
  if constexpr (KC) {
    const int r = r0 + (lane & 31), c = ks * 2 + (lane >> 5);
    return __builtin_bit_cast(bf16x8, b[r * 4 + (c ^ chunk_swizzle<true>(r))]);
  } else {
    // lane group g = lane / 16: rows 16 (g & 1) + lane % 16, k's 8 (g / 2) ..;
    // each lane addresses four rows of one k and receives four k's of one row
    const int g = lane >> 4, k = ks * 16 + 8 * (g >> 1) + ((lane & 15) >> 2);
    const int r = r0 + 16 * (g & 1) + 4 * (lane & 3);
    struct Two {
      short4v a, b;
    } o;
    const int c = r >> 3, half = (r >> 2) & 1;
    // k + 4 has the same swizzle (k & 3)
    const uint4* p = b + k * C + (c ^ chunk_swizzle<false>(k));
    o.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)((const short*)p + half * 4));
    o.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)((const short*)(p + 4 * C) + half * 4));
    return __builtin_bit_cast(bf16x8, o);
  }
}

// Whole rows of a tile from LDS (C chunks a row, chunk c of row r at
// r C + (c ^ r % 16)) to memory: V elements a chunk, rows below `rows` and
// columns below `cols`.
template <class E, int C, int ROWS>
__device__ __forceinline__ void put_rows(const uint4* tile, E* out, int64_t ld, int64_t m0, int64_t n0, int64_t rows,
                                         int64_t cols) {
  constexpr int V = 16 / (int)sizeof(E);
#pragma unroll 4
  for (int k = 0; k < ROWS * C / kDThreads; ++k) {
    const int id = threadIdx.x + k * kDThreads, r = id / C, c = id % C;
    const int64_t m = m0 + r, n = n0 + c * V;
    const Vec<E, V> v = __builtin_bit_cast(Vec<E, V>, tile[r * C + (c ^ (r & 15))]);
    if (m < rows) {
      if (n + V <= cols) {
        *reinterpret_cast<Vec<E, V>*>(out + m * ld + n) = v;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (n + e < cols) out[m * ld + n + e] = v.e[e];
      }
    }
  }
}

template <int USE>
__global__ __launch_bounds__(kDThreads, 2) void k_glu_direct(GluD p) {
  constexpr bool PAIR = USE == kForward || USE == kProject;
  constexpr bool NKC = USE == kDx, MKC = USE != kDw;
  constexpr int NF = 2, MF = 4, J = kDChunks / kDThreads;  // copies of an operand a lane and stage
  static_assert(J == 2, "the waits below count them");
  __shared__ __align__(1024) uint4 lds[4][2 * kDChunks];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave & 3, wm = wave >> 2;
  const TileAt t = tile_at<USE>(p);
  const int64_t n0 = (int64_t)t.n * (PAIR ? kDT / 2 : kDT), m0 = (int64_t)t.m * kDT;
  const int64_t kfrom = USE == kDw ? t.split * p.span : 0;
  const int64_t kend = USE == kDw && kfrom + p.span < p.K ? kfrom + p.span : p.K;
  const int blocks = (int)((kend - kfrom) / kDK);  // stages of a segment
  const int all = USE == kDx ? 2 * blocks : blocks;
  // dx: a run of the stages
  const int first = USE == kDx ? (int)(t.split * p.span) : 0;
  const int stages = USE == kDx && first + p.span < all ? (int)p.span : all - first;

  // This lane's sources of the copies, at k = 0: chunk 64 (J wave + j) + lane
  // of a stage.
  const bf16 *na[J], *ma[J];
  auto source = [&](bool kc, int id, const bf16* b0, const bf16* b1, int64_t ld, int64_t from, int64_t extent, bool pair) {
    if (kc) {
      const int row = id >> 2, c = (id & 3) ^ chunk_swizzle<true>(row);
      const int64_t r = from + row < extent ? from + row : extent - 1;  // (rows past the end are not stored)
      return b0 + r * ld + c * 8;
    }
    // pair: a wave's 64 columns are 32 of gate, then the same 32 of up
    const int k = id >> 5, c = (id & 31) ^ chunk_swizzle<false>(k);
    const int64_t r = from + (pair ? (c >> 3) * 32 + (c & 3) * 8 : c * 8);
    return (pair && (c & 4) ? b1 : b0) + k * ld + (r < extent ? r : extent - 8);
  };
  const bf16* nbase = USE == kDw && t.mat ? p.n1 : p.n0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int id = (wave * J + j) * 64 + lane;
    na[j] = source(NKC, id, nbase, p.n1, p.nld, n0, p.nx, PAIR);
    ma[j] = source(MKC, id, p.m0, p.m0, p.mld, m0, p.mx, false);
  }
  const int64_t nstep = NKC ? 1 : p.nld, mstep = MKC ? 1 : p.mld;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&lds[0][0];
  auto issue = [&](int stage) {
    const uint32_t at = lds0 + (uint32_t)((stage & 3) * 2 * kDChunks) * 16;
    const int step = first + stage;
    const bool second = USE == kDx && step >= blocks;  // du, w_up
    const int64_t k = kfrom + (int64_t)(second ? step - blocks : step) * kDK;
    const int64_t noff = k * nstep + (second ? p.n1 - p.n0 : 0), moff = k * mstep + (second ? p.m1 - p.m0 : 0);
#pragma unroll
    for (int j = 0; j < J; ++j) copy_to_lds(na[j] + noff, at + (uint32_t)(wave * J + j) * 1024);
#pragma unroll
    for (int j = 0; j < J; ++j) copy_to_lds(ma[j] + moff, at + kDChunks * 16 + (uint32_t)(wave * J + j) * 1024);
  };
  // project: the tile of dh, 128 rows to each of the two buffers that fall
  // free before the last stages (rows of 16 chunks, permuted by row % 16)
  auto copy_dh = [&]() {
#pragma unroll
    for (int k = 0; k < kDT * 16 / kDThreads; ++k) {
      const int id = k * kDThreads + wave * 64 + lane, row = id >> 4, c = (id & 15) ^ (row & 15);
      const int64_t m = m0 + row < p.M ? m0 + row : p.M - 1, n = n0 + c * 8 < p.N ? n0 + c * 8 : p.N - 8;
      const int buf = (stages + (row >> 7)) & 3;
      copy_to_lds(p.dh + m * p.dhld + n,
                  lds0 + (uint32_t)(__builtin_amdgcn_readfirstlane(buf) * 2 * kDChunks) * 16 +
                      (uint32_t)((k * kDThreads + wave * 64) & 2047) * 16);
    }
  };
  const bool dh_copied = USE == kProject && p.dh_copied;

  floatx16 acc[NF][MF] = {};
  bf16x8 nf[2][NF], mf[2][MF];
  auto read = [&](int st, int ks) {
    const uint4 *nb = lds[st & 3], *mb = nb + kDChunks;
#pragma unroll
    for (int i = 0; i < NF; ++i) nf[ks][i] = fragment<NKC>(nb, wn * 64 + i * 32, ks, lane);
#pragma unroll
    for (int j = 0; j < MF; ++j) mf[ks][j] = fragment<MKC>(mb, wm * 128 + j * 32, ks, lane);
  };
  auto multiply = [&](int ks) {
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int j = 0; j < MF; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(nf[ks][i], mf[ks][j], acc[i][j], 0, 0, 0);
  };
  // Stage s + 1 is waited for in the middle of stage s: each wave for its own
  // copies, then for the other waves; after that the buffer of stage s - 1 is
  // free, which every wave has left.  The copies into it go last: ahead of the
  // products they delay the LDS reads (dW: 410 us against 380).
  if (stages > 0) {
    issue(0);
    if (stages > 1) issue(1);
    if (stages > 2) {
      issue(2);
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    asm volatile("s_barrier" ::: "memory");
    read(0, 0);
    int s = 0;
    for (; s + 3 < stages; ++s) {
      read(s, 1);
      __builtin_amdgcn_sched_barrier(0);  // the reads first: they land behind the products
      multiply(0);
      asm volatile("s_waitcnt vmcnt(4)\n\ts_barrier" ::: "memory");
      read(s + 1, 0);
      __builtin_amdgcn_sched_barrier(0);
      multiply(1);
      issue(s + 3);
    }
    if (dh_copied && stages == 1) copy_dh();
    for (; s < stages; ++s) {
      read(s, 1);
      multiply(0);
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      if (dh_copied && s + 2 == stages) copy_dh();
      read(s + 1 < stages ? s + 1 : s, 0);
      multiply(1);
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

  // Register 4 q + e of acc[i][j]: column 8 q + 4 (lane / 32) + e of fragment
  // i's 32, row lane % 32 of fragment j's.
  const int r32 = lane & 31, hi = lane >> 5;
  uint4* tile = lds[0];
  auto four = [&](int i, int j, int q) {
    const floatx16& v = acc[i][j];
    return __builtin_bit_cast(uint4, make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
  };
  if (!PAIR && (USE == kDw || p.parts)) {
    // fp32 parts, 128 rows at a time
    float* out = p.parts + ((int64_t)t.split * (USE == kDw ? 2 : 1) + t.mat) * p.M * p.N;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half) __syncthreads();
      if (wm == half) {
#pragma unroll
        for (int j = 0; j < MF; ++j)
#pragma unroll
          for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int r = j * 32 + r32, c = wn * 16 + i * 8 + 2 * q + hi;
              tile[r * 64 + (c ^ (r & 15))] = four(i, j, q);
            }
      }
      __syncthreads();
      put_rows<float, 64, 128>(tile, out, p.N, m0 + half * 128, n0, p.M, p.N);
    }
    return;
  }
  if constexpr (USE == kProject) {
    // dg and du in place of the projections; dh from LDS, or straight from
    // memory.  Rows past M and columns past N give 0: what reduces over them
    // reads whole stages.
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = j * 32 + r32, c = wn * 4 + q;
        const int64_t m = m0 + wm * 128 + r, n = n0 + wn * 32 + 8 * q + 4 * hi;
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        if (dh_copied) {
          const Four<bf16> f = *(reinterpret_cast<const Four<bf16>*>(lds[(stages + wm) & 3] + r * 16 + (c ^ (r & 15))) + hi);
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e] = to_f32(f.e[e]);
        } else if (m < p.M) {
          load_four(p.dh + m * p.dhld + n, (int)(p.N - n < 4 ? p.N - n : 4), d);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool in = m < p.M && n + e < p.N;
          float slope;
          const float v = act_of(p.act, acc[0][j][4 * q + e], slope), u = acc[1][j][4 * q + e];
          acc[0][j][4 * q + e] = in ? d[e] * u * slope : 0.f;
          acc[1][j][4 * q + e] = in ? d[e] * v : 0.f;
        }
      }
    __syncthreads();
  }
  // bfloat16 rows; dg and du lie side by side
  constexpr int C = PAIR ? 16 : 32, COUNT = USE == kProject ? 2 : 1;
#pragma unroll
  for (int w = 0; w < COUNT; ++w)
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
      for (int i = 0; i < (PAIR ? 1 : NF); ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = wm * 128 + j * 32 + r32, c = (PAIR ? wn * 4 : wn * 8 + i * 4) + q;
          Four<bf16> o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = acc[PAIR ? w : i][j][4 * q + e], slope;
            if constexpr (USE == kForward) v = act_of(p.act, v, slope) * acc[1][j][4 * q + e];
            o.e[e] = from_f32<bf16>(v);
          }
          *(reinterpret_cast<Four<bf16>*>(tile + w * kDT * C + r * C + (c ^ (r & 15))) + hi) = o;
        }
  __syncthreads();
  const int64_t rows = USE == kProject ? p.om : p.M, cols = USE == kProject ? p.on : p.N;
  put_rows<bf16, C, kDT>(tile, p.out0, p.old0, m0, n0, rows, cols);
  if (USE == kProject) put_rows<bf16, C, kDT>(tile + kDT * C, p.out1, p.old1, m0, n0, rows, cols);
}

// An operand in whole chunks: rows of `cols` elements to rows of `ld`, with
// zeros up to `ld` columns and `prows` rows.
__global__ __launch_bounds__(256) void k_glu_pack(const bf16* __restrict__ src, int64_t sld, int64_t rows, int64_t cols,
                                                  bf16* __restrict__ out, int64_t ld, int64_t prows) {
  const int64_t chunks = ld / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= chunks * prows) return;
  const int64_t r = i / chunks, c = (i - r * chunks) * 8;
  Vec<bf16, 8> v{};
  if (r < rows) {
    const bf16* p = src + r * sld + c;
    if (c + 8 <= cols) {
      v = *reinterpret_cast<const Vec<bf16, 8>*>(p);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) v.e[e] = p[e];
    }
  }
  *reinterpret_cast<uint4*>(out + r * ld + c) = __builtin_bit_cast(uint4, v);
}

// dW (two matrices a part) or dx (one) from their parts, in order.
template <class E>
__global__ __launch_bounds__(256) void k_glu_join(const float* __restrict__ parts, uint32_t splits, int mats, int64_t M,
                                                  int64_t N, E* out0, int64_t ld0, E* out1, int64_t ld1) {
  const int64_t groups = (N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= mats * M * groups) return;
  const int64_t mat = i / (M * groups), at = i - mat * M * groups, m = at / groups, n = (at - m * groups) * 4;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  const int valid = (int)(N - n < 4 ? N - n : 4);
  for (uint32_t s = 0; s < splits; ++s) {
    float v[4];
    load_four(parts + ((int64_t)s * mats + mat) * M * N + m * N + n, valid, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] += v[e];
  }
  store_four(mat ? out1 + m * ld1 + n : out0 + m * ld0 + n, valid, t);
}

// Forward for a few rows (single frames of some voices): the weights' reading
// is all that counts, and its latency, so the vector unit multiplies.  A
// workgroup owns COLS columns (two a lane) of 8 rows; the 16 waves' slices take
// every 64th or 128th k, each with all of its loads of a round of 512 k's in
// flight at once (the next round's behind them cost registers: 5.9 us for 5.0
// at 8 x 512 x 1408 bf16); the slices' sums meet by exchange in registers, then
// in LDS.
constexpr int kFewRows = 8, kFewThreads = 1024, kFewRound = 512;
template <class E, int COLS>
__global__ __launch_bounds__(kFewThreads) void k_glu_few(GluP<E> p) {
  constexpr int LANES = COLS / 2, SLICES = kFewThreads / LANES, LOADS = kFewRound / SLICES, ROUND = kFewRound;
  constexpr int XS = ROUND * kFewRows / kFewThreads;
  __shared__ __align__(16) float xs[ROUND][kFewRows];
  __shared__ float red[16][COLS][2][kFewRows + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slice = threadIdx.x / LANES;
  const int64_t m0 = (int64_t)blockIdx.y * kFewRows, f = (int64_t)blockIdx.x * COLS + (lane % LANES) * 2;
  const bool two = f + 1 < p.N;
  const int64_t col = two ? f : f < p.N ? f : p.N - 1;  // (columns past the end are not stored)
  const E *g = p.n0 + col, *u = p.n1 + col;
  float acc[2][2][kFewRows] = {}, xv[XS];
  Vec<E, 2> w[LOADS][2];
  auto load = [&](int64_t k0) {
#pragma unroll
    for (int i = 0; i < XS; ++i) {
      const int id = threadIdx.x + i * kFewThreads, m = id / ROUND, k = id % ROUND;
      xv[i] = k0 + k < p.K && m0 + m < p.M ? to_f32(p.m0[(m0 + m) * p.mld0 + k0 + k]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int64_t k = k0 + slice + SLICES * i, kc = k < p.K ? k : p.K - 1;
      if (two) {
        w[i][0] = *reinterpret_cast<const Vec<E, 2>*>(g + kc * p.nld0);
        w[i][1] = *reinterpret_cast<const Vec<E, 2>*>(u + kc * p.nld1);
      } else {
        w[i][0].e[0] = w[i][0].e[1] = g[kc * p.nld0];
        w[i][1].e[0] = w[i][1].e[1] = u[kc * p.nld1];
      }
    }
  };
  for (int64_t k0 = 0; k0 < p.K; k0 += ROUND) {
    load(k0);
    if (k0 > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < XS; ++i) {
      const int id = threadIdx.x + i * kFewThreads;
      xs[id % ROUND][id / ROUND] = xv[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      // (past the end the weights are a row inside, which may hold anything)
      if (k0 + slice + SLICES * i >= p.K) continue;
#pragma unroll
      for (int m = 0; m < kFewRows; ++m) {
        const float x = xs[slice + SLICES * i][m];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int b = 0; b < 2; ++b) acc[a][b][m] = fmaf(x, to_f32(w[i][a].e[b]), acc[a][b][m]);
      }
    }
  }
  // over the wave's slices: a lane keeps, of four rows, 2 (its bit 4) + (its bit 5)
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int m = 0; m < kFewRows; m += 4) {
        const float* v = acc[a][b] + m;
        float t = swap_add16(swap_add32(v[0], v[1]), swap_add32(v[2], v[3]));
        if constexpr (LANES == 8) t += dpp<0x128>(t);  // row_ror:8
        if ((lane & 15) < LANES) red[wave][lane % LANES * 2 + b][a][m + 2 * ((lane >> 4) & 1) + (lane >> 5)] = t;
      }
  __syncthreads();
  if (threadIdx.x >= COLS * kFewRows) return;
  const int c = threadIdx.x % COLS, m = threadIdx.x / COLS;
  const int64_t n = (int64_t)blockIdx.x * COLS + c;
  float s[2] = {0.f, 0.f}, slope;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    s[0] += red[w][c][0][m];
    s[1] += red[w][c][1][m];
  }
  if (m0 + m < p.M && n < p.N) p.out0[(m0 + m) * p.old0 + n] = from_f32<E>(act_of(p.act, s[0], slope) * s[1]);
}

// ------------------------------------------------------------------ shapes
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t tiles(int64_t n, int64_t of) { return (n + of - 1) / of; }

// Forward by k_glu_few.  It reads the weights once more for every 8 rows and
// multiplies on the vector unit, so it is taken while its workgroups (of 32
// columns and 8 rows) are one round of the 256 CUs, two for fp32, whose tiles
// take three times as long.  Kernels, us, weights in the caches, few /
// tiles (whose time does not change up to 128 rows): bfloat16, 512 x 1408, 16 rows 5 / 10, 40 (220
// workgroups) 6 / 10, 48 (264) 9.9 / 10.3, 96 (528) 14 / 10.5; 1024 x 2816, 16
// (176) 11 / 20, 48 (528) 27 / 20; 1024 x 16384, 8 (512) 28 / 26, 16 (1024) 53
// / 25; 2048 x 512, 128 (256) 17 / 31; fp32, 512 x 1408, 64 (352) 13 / 26; 1024
// x 8192, 16 (512) 30 / 48, 32 (1024) 56 / 48; 1024 x 2816, 96 (1056) 55 / 49.
bool few(const dgen_hip_mlp& a) {
  return a.rows <= 128 && tiles(a.hidden, 32) * tiles(a.rows, kFewRows) <= (a.type == DGEN_HIP_BF16 ? 256 : 512);
}

// bfloat16: packed operands and 256 x 256 tiles where the projections' tiles
// come near to filling the chip's 256 CUs; else small tiles on the operands as
// they are.  Rows x width x hidden, us forward and backward, large / small:
// 132 tiles, 1500 x 1024 x 2816 31 / 50 and 144 / 177, 3000 x 512 x 1408 21 /
// 29 and 105 / 111; 88 tiles, 1024 x 1024 x 2816 30 / 33 and 112 / 118, 2000 x
// 512 x 1408 19 / 19 and 101 / 87; 72 tiles, 9000 x 256 x 256 16 / 15 and 85 /
// 53.
bool large(const dgen_hip_mlp& a) {
  return a.type == DGEN_HIP_BF16 && !few(a) && tiles(a.rows, kDT) * tiles(2 * a.hidden, kDT) >= 128;
}

// Runs of a reduction of `steps`, as many as make the rounds of `count` tiles
// over the CUs' `slots` full, against the time that the parts take: a step of
// a tile takes `step`, writing and reading a tile's part `join` of the whole
// chip, both in us.
int64_t runs_of(int64_t count, int64_t steps, int64_t least, int64_t slots, double step, double join) {
  int64_t best = 1;
  double cost = 0;
  for (int64_t r = 1; r <= std::max<int64_t>(1, std::min<int64_t>(steps / least, 64)); ++r) {
    const double c = (double)(tiles(count * r, slots) * tiles(steps, r)) * step + (r > 1 ? (double)(r * count) * join : 0);
    if (r == 1 || c < cost) best = r, cost = c;
  }
  return best;
}

struct Split {
  int64_t span;  // steps or rows of a run
  uint32_t runs;
};
Split split_of(int64_t n, int64_t runs, int64_t unit) {
  const int64_t span = std::max(unit, up(tiles(n, runs), unit));
  return {span, (uint32_t)std::max<int64_t>(1, tiles(n, span))};
}

// How a call is laid out: which operands are packed, how the reductions are
// cut, and what lies where in the workspace (byte offsets).
struct Plan {
  bool large;
  int64_t width, hidden, rows;  // padded to whole stages
  bool pack_x, pack_w;
  Split dx, dw;                 // stages or steps of dx's runs, rows of dW's
  int64_t dw_rows;              // rows in the runs; the rest (of x as it is) is one more
  int64_t x, xtail, wg, wu, dg, du, parts, total;
};
// k_glu's tile: 128 x 128 for fp32 products that have more tiles (with the runs
// that their reduction can be cut into) than there are CUs, else 64 x 128.
// Forward, us, 128 x 128 / 64 x 128: 500 x 512 x 1408 (88 tiles) 39 / 29, 3000
// x 256 x 700 (264) 33 / 28, 2000 x 512 x 1408 (352) 52 / 54; backward of the
// last 165 / 182, of 4000 x 512 x 512 129 / 141.
template <class E>
bool wide_tile(int64_t rows, int64_t cols, int64_t runs) {
  return sizeof(E) == 4 && tiles(rows, 128) * tiles(cols, 128) * runs >= 320;
}
template <class E>
int64_t runs_small(int64_t rows, int64_t cols, int64_t mats, int64_t steps) {
  // (a step of a 128 x 128 fp32 tile takes about 4 us with two workgroups a
  // CU, of a 64 x 128 tile 1 to 2 us with four; a part 0.03 and 0.02 us)
  if (wide_tile<E>(rows, mats * cols, std::max<int64_t>(1, steps / 8)))
    return runs_of(mats * tiles(rows, 128) * tiles(cols, 128), steps, 8, 512, 4.0, 0.03);
  return runs_of(mats * tiles(rows, 64) * tiles(cols, 128), steps, 8, 1024, 1.5, 0.02);
}
template <class E>
Plan plan_of(const dgen_hip_mlp& a, bool backward) {
  Plan p{};
  p.large = large(a);
  p.rows = up(a.rows, kDK), p.width = up(a.width, kDK), p.hidden = up(a.hidden, p.large ? kDK : 8);
  auto whole = [](const void* q, int64_t ld) { return (uintptr_t)q % 16 == 0 && ld % 8 == 0; };
  p.pack_x = p.large && !(a.width % kDK == 0 && whole(a.x, a.x_stride));
  p.pack_w = p.large && !(a.width % kDK == 0 && a.hidden % kDK == 0 && whole(a.w_gate, a.w_gate_stride) &&
                          whole(a.w_up, a.w_up_stride) && a.w_gate_stride == a.w_up_stride);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  if (p.pack_x) p.x = take(p.rows * p.width * 2);
  if (p.pack_w) p.wg = take(p.width * p.hidden * 2), p.wu = take(p.width * p.hidden * 2);
  if (backward) {
    p.dg = take((p.large ? p.rows : a.rows) * p.hidden * (int64_t)sizeof(E));
    p.du = take((p.large ? p.rows : a.rows) * p.hidden * (int64_t)sizeof(E));
    int64_t parts = 0;
    if (p.large) {
      // (a 256 x 256 x 32 stage takes a CU about 0.9 us; a tile's part, 512
      // KB to and from memory, 0.13 us)
      const int64_t stages = 2 * p.hidden / kDK;
      p.dx = split_of(stages, runs_of(tiles(a.rows, kDT) * tiles(a.width, kDT), stages, 16, 256, 0.9, 0.13), 1);
      p.dw_rows = p.pack_x ? p.rows : a.rows / kDK * kDK;
      const int64_t count = 2 * tiles(a.width, kDT) * tiles(a.hidden, kDT);
      p.dw = split_of(p.dw_rows, runs_of(count, p.dw_rows / kDK, 16, 256, 0.9, 0.13), kDK);
      if (p.dw_rows < a.rows) p.xtail = take(kDK * p.width * 2);
      parts = (int64_t)(p.dw.runs + (p.dw_rows < a.rows ? 1 : 0)) * 2 * a.width * a.hidden * 4;
    } else {
      const int64_t bk = sizeof(E) == 2 ? 64 : 32, steps = 2 * tiles(a.hidden, bk);
      p.dx = split_of(steps, runs_small<E>(a.rows, a.width, 1, steps), 1);
      p.dw_rows = a.rows;
      p.dw = split_of(a.rows, runs_small<E>(a.width, a.hidden, 2, tiles(a.rows, bk)), bk);
      if (p.dw.runs > 1) parts = (int64_t)p.dw.runs * 2 * a.width * a.hidden * 4;
    }
    if (p.dx.runs > 1) parts = std::max(parts, (int64_t)p.dx.runs * a.rows * a.width * 4);
    p.parts = take(parts);
  }
  p.total = at;
  return p;
}

// Whether the packs and joins, a thread for 8 and 4 elements, stay below the
// 2^32 threads of a launch (the products' tiles are limited in mlp_run).
bool fits(const dgen_hip_mlp& a, const Plan& p, bool backward) {
  constexpr int64_t kMost = (int64_t(1) << 32) - 256;
  if (p.pack_x && p.width / 8 * p.rows > kMost) return false;
  if (!backward) return true;
  return (p.dx.runs == 1 || a.rows * tiles(a.width, 4) <= kMost) &&
         ((!p.large && p.dw.runs == 1) || 2 * a.width * tiles(a.hidden, 4) <= kMost);
}

// ----------------------------------------------------------------- launches
template <class E, int USE>
void staged(GluP<E> p, hipStream_t st) {
  constexpr bool PAIR = USE == kForward || USE == kProject;
  const uint32_t more = USE == kDw ? 2 * p.splits : p.splits;
  if constexpr (sizeof(E) == 4) {
    if (wide_tile<E>(p.M, PAIR ? 2 * p.N : p.N, more)) {
      p.tiles_m = (uint32_t)tiles(p.M, 128);
      p.tiles_n = (uint32_t)tiles(p.N, PAIR ? 64 : 128);
      k_glu<E, 128, 128, 64, 64, 32, USE><<<dim3(p.tiles_m * p.tiles_n * more), kThreads, 0, st>>>(p);
      return;
    }
  }
  p.tiles_m = (uint32_t)tiles(p.M, 64);
  p.tiles_n = (uint32_t)tiles(p.N, PAIR ? 64 : 128);
  k_glu<E, 64, 128, 32, 64, sizeof(E) == 2 ? 64 : 32, USE><<<dim3(p.tiles_m * p.tiles_n * more), kThreads, 0, st>>>(p);
}

template <int USE>
void direct(GluD p, hipStream_t st) {
  constexpr bool PAIR = USE == kForward || USE == kProject;
  p.tiles_m = (uint32_t)tiles(USE == kProject ? p.om : p.M, kDT);
  p.tiles_n = (uint32_t)tiles(USE == kProject ? p.on : p.N, PAIR ? kDT / 2 : kDT);
  const uint32_t more = USE == kDw ? 2 * p.splits : p.splits;
  k_glu_direct<USE><<<dim3(p.tiles_m * p.tiles_n * more), kDThreads, 0, st>>>(p);
}

void pack(const void* src, int64_t sld, int64_t rows, int64_t cols, bf16* out, int64_t ld, int64_t prows, hipStream_t st) {
  const int64_t n = ld / 8 * prows;
  k_glu_pack<<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>((const bf16*)src, sld, rows, cols, out, ld, prows);
}

template <class E>
void join(const float* parts, uint32_t runs, int mats, int64_t M, int64_t N, void* out0, int64_t ld0, void* out1,
          int64_t ld1, hipStream_t st) {
  const int64_t n = mats * M * ((N + 3) / 4);
  k_glu_join<E><<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>(parts, runs, mats, M, N, (E*)out0, ld0, (E*)out1, ld1);
}

void launch_large(const dgen_hip_mlp& a, bool backward, const Plan& p, hipStream_t st) {
  char* ws = (char*)a.workspace;
  GluD q{};
  q.act = a.act, q.splits = 1;
  q.K = p.width;
  if (p.pack_x) {
    pack(a.x, a.x_stride, a.rows, a.width, (bf16*)(ws + p.x), p.width, p.rows, st);
    q.m0 = (bf16*)(ws + p.x), q.mld = p.width;
  } else {
    q.m0 = (const bf16*)a.x, q.mld = a.x_stride;
  }
  if (p.pack_w) {
    pack(a.w_gate, a.w_gate_stride, a.width, a.hidden, (bf16*)(ws + p.wg), p.hidden, p.width, st);
    pack(a.w_up, a.w_up_stride, a.width, a.hidden, (bf16*)(ws + p.wu), p.hidden, p.width, st);
    q.n0 = (bf16*)(ws + p.wg), q.n1 = (bf16*)(ws + p.wu), q.nld = p.hidden;
  } else {
    q.n0 = (const bf16*)a.w_gate, q.n1 = (const bf16*)a.w_up, q.nld = a.w_gate_stride;
  }
  q.nx = p.hidden, q.mx = a.rows;
  q.M = a.rows, q.N = a.hidden;
  if (!backward) {
    q.out0 = (bf16*)a.h, q.old0 = a.h_stride;
    direct<kForward>(q, st);
    return;
  }
  bf16 *dg = (bf16*)(ws + p.dg), *du = (bf16*)(ws + p.du);
  float* parts = (float*)(ws + p.parts);
  GluD r = q;
  r.out0 = dg, r.out1 = du, r.old0 = r.old1 = p.hidden;
  r.om = p.rows, r.on = p.hidden;
  r.dh = (const bf16*)a.dh, r.dhld = a.dh_stride;
  r.dh_copied = (uintptr_t)a.dh % 16 == 0 && a.dh_stride % 8 == 0 && a.hidden % 8 == 0;
  direct<kProject>(r, st);

  GluD x = q;
  x.m0 = dg, x.m1 = du, x.mld = p.hidden;
  x.N = a.width, x.K = p.hidden, x.nx = a.width;
  x.out0 = (bf16*)a.dx, x.old0 = a.dx_stride;
  x.splits = p.dx.runs, x.span = p.dx.span;
  x.parts = p.dx.runs > 1 ? parts : nullptr;
  direct<kDx>(x, st);
  if (x.parts) join<bf16>(parts, p.dx.runs, 1, x.M, x.N, a.dx, a.dx_stride, nullptr, 0, st);

  GluD w = q;
  w.n0 = dg, w.n1 = du, w.nld = p.hidden, w.nx = p.hidden;
  w.M = a.width, w.N = a.hidden, w.mx = p.width;
  w.K = p.dw_rows, w.splits = p.dw.runs, w.span = p.dw.span, w.parts = parts;
  if (p.dw_rows > 0) direct<kDw>(w, st);
  uint32_t runs = p.dw_rows > 0 ? p.dw.runs : 0;
  if (p.dw_rows < a.rows) {
    // the last rows of x, less than a stage, with zeros up to it
    bf16* tail = (bf16*)(ws + p.xtail);
    pack((const bf16*)a.x + p.dw_rows * a.x_stride, a.x_stride, a.rows - p.dw_rows, a.width, tail, p.width, kDK, st);
    w.m0 = tail, w.mld = p.width, w.n0 = dg + p.dw_rows * p.hidden, w.n1 = du + p.dw_rows * p.hidden;
    w.K = w.span = kDK, w.splits = 1, w.parts = parts + (int64_t)runs * 2 * a.width * a.hidden;
    direct<kDw>(w, st);
    ++runs;
  }
  join<bf16>(parts, runs, 2, a.width, a.hidden, a.dw_gate, a.dw_gate_stride, a.dw_up, a.dw_up_stride, st);
}

template <class E>
void launch_staged(const dgen_hip_mlp& a, bool backward, const Plan& p, hipStream_t st) {
  GluP<E> q{};
  q.act = a.act;
  q.splits = 1, q.span = int64_t(1) << 40;
  q.n0 = (const E*)a.w_gate, q.n1 = (const E*)a.w_up, q.nld0 = a.w_gate_stride, q.nld1 = a.w_up_stride;
  q.m0 = q.m1 = (const E*)a.x, q.mld0 = q.mld1 = a.x_stride;
  q.M = a.rows, q.N = a.hidden, q.K = a.width;
  if (!backward) {
    q.out0 = (E*)a.h, q.old0 = a.h_stride;
    if (few(a)) {
      // 16 columns a workgroup while there is a CU for each workgroup, else 32
      // (bf16, 16 / 32 columns, us: 8 x 512 x 1408, 88 of 16, 5.0 / 6.3; 8 x 1024
      // x 2816, 176, 12.1 / 12.2; 16 x 1024 x 2816, 352, 19.6 / 12.1)
      const int64_t groups = tiles(a.rows, kFewRows), cols = tiles(a.hidden, 16) * groups <= 256 ? 16 : 32;
      const dim3 grid((unsigned)tiles(a.hidden, cols), (unsigned)groups);
      if (cols == 16) k_glu_few<E, 16><<<grid, kFewThreads, 0, st>>>(q);
      else k_glu_few<E, 32><<<grid, kFewThreads, 0, st>>>(q);
    } else {
      staged<E, kForward>(q, st);
    }
    return;
  }
  E *dg = (E*)((char*)a.workspace + p.dg), *du = (E*)((char*)a.workspace + p.du);
  float* parts = (float*)((char*)a.workspace + p.parts);
  if (a.rows > 0) {
    GluP<E> r = q;
    r.out0 = dg, r.out1 = du, r.old0 = r.old1 = p.hidden;
    r.dh = (const E*)a.dh, r.dhld = a.dh_stride;
    staged<E, kProject>(r, st);
    GluP<E> x = q;
    x.m0 = dg, x.m1 = du, x.mld0 = x.mld1 = p.hidden;
    x.N = a.width, x.K = a.hidden;
    x.out0 = (E*)a.dx, x.old0 = a.dx_stride;
    x.splits = p.dx.runs, x.span = p.dx.span;
    x.parts = p.dx.runs > 1 ? parts : nullptr;
    staged<E, kDx>(x, st);
    if (x.parts) join<E>(parts, p.dx.runs, 1, x.M, x.N, a.dx, a.dx_stride, nullptr, 0, st);
  }
  GluP<E> w = q;
  w.n0 = dg, w.n1 = du, w.nld0 = w.nld1 = p.hidden;
  w.M = a.width, w.N = a.hidden, w.K = a.rows;
  w.out0 = (E*)a.dw_gate, w.old0 = a.dw_gate_stride, w.out1 = (E*)a.dw_up, w.old1 = a.dw_up_stride;
  w.splits = p.dw.runs, w.span = p.dw.span;
  w.parts = p.dw.runs > 1 ? parts : nullptr;
  staged<E, kDw>(w, st);
  if (w.parts) join<E>(parts, p.dw.runs, 2, a.width, a.hidden, a.dw_gate, a.dw_gate_stride, a.dw_up, a.dw_up_stride, st);
}

template <class E>
void mlp_launch(const dgen_hip_mlp& a, bool backward, hipStream_t st) {
  const Plan p = plan_of<E>(a, backward);
  p.large ? launch_large(a, backward, p, st) : launch_staged<E>(a, backward, p, st);
}

}  // namespace

namespace {
Plan plan_for(const dgen_hip_mlp& a, bool backward) {
  return a.type == DGEN_HIP_BF16 ? plan_of<bf16>(a, backward) : plan_of<float>(a, backward);
}
}  // namespace

int64_t mlp_workspace(const dgen_hip_mlp& a, bool backward) { return plan_for(a, backward).total; }

int mlp_run(const dgen_hip_mlp& a, bool backward, hipStream_t st, bool dry) {
  const char* what = backward ? "gated_mlp_backward" : "gated_mlp";
  DGEN_REQUIRE(a.struct_size == sizeof(a), "%s: struct_size %u, expected %zu", what, a.struct_size, sizeof(a));
  DGEN_REQUIRE(a.type == DGEN_HIP_F32 || a.type == DGEN_HIP_BF16, "%s: type %d", what, a.type);
  DGEN_REQUIRE(a.act == DGEN_HIP_SILU || a.act == DGEN_HIP_GELU, "%s: activation %d", what, a.act);
  DGEN_REQUIRE(a.width >= 1 && a.width <= (1 << 17) && a.hidden >= 1 && a.hidden <= (1 << 17),
               "%s: width %lld or hidden %lld outside [1, 2^17]", what, (long long)a.width, (long long)a.hidden);
  // (tiles, of 64 rows at least, times threads stay below 2^32)
  DGEN_REQUIRE(a.rows >= 0 && (a.rows + 63) / 64 * ((2 * a.hidden + 127) / 128 + (a.width + 127) / 128) < (1 << 23),
               "%s: rows %lld too many for one call", what, (long long)a.rows);
  DGEN_REQUIRE(a.w_gate && a.w_up, "%s: null w_gate or w_up", what);
  DGEN_REQUIRE(a.w_gate_stride >= 0 && a.w_up_stride >= 0 && a.x_stride >= 0, "%s: negative stride", what);
  const bool empty = a.rows == 0;
  DGEN_REQUIRE(a.x || empty, "%s: null x", what);
  if (!backward) {
    DGEN_REQUIRE((a.h || empty) && (a.rows <= 1 || a.h_stride >= a.hidden), "%s: h missing or overlapping itself", what);
  } else {
    DGEN_REQUIRE((a.dh || empty) && a.dh_stride >= 0, "%s: dh missing or with a negative stride", what);
    DGEN_REQUIRE((a.dx || empty) && (a.rows <= 1 || a.dx_stride >= a.width), "%s: dx missing or overlapping itself",
                 what);
    DGEN_REQUIRE(a.dw_gate && a.dw_up && (a.width <= 1 || (a.dw_gate_stride >= a.hidden && a.dw_up_stride >= a.hidden)),
                 "%s: dw_gate or dw_up missing or overlapping itself", what);
  }
  const Plan plan = plan_for(a, backward);
  DGEN_REQUIRE(fits(a, plan, backward), "%s: rows %lld x width %lld x hidden %lld is too large for one call", what,
               (long long)a.rows, (long long)a.width, (long long)a.hidden);
  const int64_t need = plan.total;
  DGEN_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= (uint64_t)need && (uintptr_t)a.workspace % 256 == 0),
               "%s: workspace of %llu bytes, %lld needed (256-byte aligned)", what, (unsigned long long)a.workspace_bytes,
               (long long)need);
  if (dry || (empty && !backward)) return 0;
  if (a.type == DGEN_HIP_BF16) mlp_launch<bf16>(a, backward, st);
  else mlp_launch<float>(a, backward, st);
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
