// Gated feed-forward block: h = act(x Wg) * (x Wu), forward and backward, on
// the bf16 matrix cores.
//
// One product kernel serves four uses.  A workgroup of four waves owns a tile
// of the output; operand tiles go from memory through registers to LDS, where
// they lie k-contiguous whatever their layout in memory (an operand that is
// contiguous along its rows is transposed on the way: a thread loads 8 k's of a
// few neighbouring rows and packs them with one byte permutation a dword).
//
// - forward: the tile's columns are 32- or 64-wide groups of gate and up
//   columns side by side, so a wave holds both projections of the same outputs
//   and applies the activation and the product in registers;
// - backward, projections again: the same, but the epilogue reads dh and
//   writes dg = dh u act'(g) and du = dh act(g), in the operands' type;
// - dx = dg Wg^T + du Wu^T: one product over 2 x hidden;
// - dWg = x^T dg, dWu = x^T du: products over the rows, split over row ranges
//   where the tiles alone do not fill the chip; the parts are added in order.
//
// bfloat16 operands multiply as they are, accumulated in fp32.  fp32 operands
// are split exactly into three bfloat16 parts on the way to LDS and the six
// partial products down to 2^-16 are accumulated in fp32, as accurate as fp32
// products (see k_gemm.hip).
//
// The matrix instruction's row index is the output's column, so a lane ends
// with four consecutive columns of one output row.
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
  const float v2 = v * v, p = sigmoid(kGeluA * v * fmaf(kGeluB, v2, 1.f));
  slope = p * fmaf(v * (1.f - p), kGeluA * fmaf(3.f * kGeluB, v2, 1.f), 1.f);
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

  // row(r): the address of row r of the tile (KC) or of element (r, k = 0)
  // (!KC), and how many rows from r on are inside the operand.
  template <class Row>
  __device__ __forceinline__ void load(Row row, int64_t ld, int64_t k0, int64_t kend) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = threadIdx.x + u * kThreads;
      if constexpr (KC) {
        const int r = i / (BK / 8);
        const int64_t k = k0 + (i % (BK / 8)) * 8;
        const E* p;
        const bool in = row(r, p) > 0;
        get<V>(p + k, in ? kend - k : 0, v[u][0]);
      } else {
        const int r = (i % (R / V)) * V;
        const int64_t k = k0 + (i / (R / V)) * 8;
        const E* p;
        const int64_t in = row(r, p);
#pragma unroll
        for (int q = 0; q < 8; ++q) get<V>(p + (k + q) * ld, k + q < kend ? in : 0, v[u][q]);
      }
    }
  }

  template <int W>
  __device__ __forceinline__ static void get(const E* p, int64_t valid, E (&o)[W]) {
    if (valid >= W) {
      const Vec<E, W> t = *reinterpret_cast<const Vec<E, W>*>(p);
#pragma unroll
      for (int e = 0; e < W; ++e) o[e] = t.e[e];
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) o[e] = e < valid ? p[e] : E{};
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
          put_four(p.out0 + m * p.old0 + n, p.N - n, a);
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

// ----------------------------------------------------------------- kernel
// Tile of this workgroup.  Consecutive workgroups go to the eight XCDs in
// turn, so each XCD takes a run of consecutive tiles; a run goes through
// groups of four column tiles, row tiles in turn, so that the tiles an XCD
// works on at a time (32 of the large ones, one a CU) share eight row tiles
// and four column tiles in its L2.
struct TileAt {
  uint32_t n, m, split, mat;
};
template <int USE, class E>
__device__ __forceinline__ TileAt tile_at(const GluP<E>& p) {
  const uint32_t total = gridDim.x, each = total / 8, more = total % 8;
  const uint32_t xcd = blockIdx.x & 7, id = xcd * each + (xcd < more ? xcd : more) + (blockIdx.x >> 3);
  const uint32_t plane = p.tiles_n * p.tiles_m, rest = id / plane, at = id - rest * plane;
  const uint32_t group = at / (4 * p.tiles_m), in = at - group * 4 * p.tiles_m;
  const uint32_t wide = p.tiles_n - group * 4 < 4 ? p.tiles_n - group * 4 : 4;
  return {group * 4 + in % wide, in / wide, USE == kDw ? rest % p.splits : 0, USE == kDw ? rest / p.splits : 0};
}

// BM x BN: output rows and operand columns of a tile; WM x WN: of a wave.
template <class E, int BM, int BN, int WM, int WN, int BK, int BUF, int USE>
__global__ __launch_bounds__(kThreads) void k_glu(GluP<E> p) {
  constexpr int P = planes<E>(), NF = WN / 32, MF = WM / 32;
  constexpr bool PAIR = USE == kForward || USE == kProject;
  constexpr bool NKC = USE == kDx, MKC = USE != kDw;
  static_assert((BM / WM) * (BN / WN) == kThreads / 64, "four waves");
  constexpr int NCH = P * BN * BK / 8, MCH = P * BM * BK / 8;
  __shared__ Chunk lds[BUF][NCH + MCH];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wn = wave % (BN / WN), wm = wave / (BN / WN);
  const TileAt t = tile_at<USE>(p);
  const uint32_t split = t.split, mat = t.mat;
  constexpr int COLS = PAIR ? BN / 2 : BN;  // output columns of a tile
  const int64_t n0 = (int64_t)t.n * COLS, m0 = (int64_t)t.m * BM;
  const int64_t kfrom = USE == kDw ? split * p.span : 0;
  const int64_t kend = USE == kDw && kfrom + p.span < p.K ? kfrom + p.span : p.K;
  const int64_t kblocks = kend > kfrom ? (kend - kfrom + BK - 1) / BK : 0;
  const int64_t steps = USE == kDx ? 2 * kblocks : kblocks;

  Stage<E, BN, BK, NKC> sn;
  Stage<E, BM, BK, MKC> sm;
  auto load = [&](int64_t step) {
    const bool second = USE == kDx && step >= kblocks;
    const int64_t k0 = kfrom + (second ? step - kblocks : step) * BK;
    const bool n_second = second || (USE == kDw && mat), m_second = second;
    const E* nb = n_second ? p.n1 : p.n0;
    const int64_t nld = n_second ? p.nld1 : p.nld0;
    const E* mb = m_second ? p.m1 : p.m0;
    const int64_t mld = m_second ? p.mld1 : p.mld0;
    auto nrow = [&](int r, const E*& at) -> int64_t {
      if constexpr (PAIR) {
        // a wave's WN columns: WN / 2 of gate, then the same of up
        const bool up = (r % WN) >= WN / 2;
        const int64_t f = n0 + r / WN * (WN / 2) + r % (WN / 2);
        at = (up ? p.n1 : p.n0) + f;
        return p.N - f;
      } else {
        const int64_t n = n0 + r;
        at = NKC ? nb + n * nld : nb + n;
        return p.N - n;
      }
    };
    auto mrow = [&](int r, const E*& at) -> int64_t {
      const int64_t m = m0 + r;
      at = MKC ? mb + m * mld : mb + m;
      return p.M - m;
    };
    if constexpr (PAIR) {
      // (the two matrices may have different strides: the block's own is used)
      const bool up = ((threadIdx.x % (BN / Stage<E, BN, BK, NKC>::V)) * Stage<E, BN, BK, NKC>::V) % WN >= WN / 2;
      sn.load(nrow, up ? p.nld1 : p.nld0, k0, kend);
    } else {
      sn.load(nrow, nld, k0, kend);
    }
    sm.load(mrow, mld, k0, kend);
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

  if (steps > 0) load(0);
  if constexpr (BUF == 2) {
    if (steps > 0) {
      sn.store(lds[0]);
      sm.store(lds[0] + NCH);
    }
    __syncthreads();
    for (int64_t s = 0; s < steps; ++s) {
      if (s + 1 < steps) load(s + 1);
      compute(lds[s & 1]);
      if (s + 1 < steps) {
        sn.store(lds[(s + 1) & 1]);
        sm.store(lds[(s + 1) & 1] + NCH);
      }
      __syncthreads();
    }
  } else {
    for (int64_t s = 0; s < steps; ++s) {
      __syncthreads();
      sn.store(lds[0]);
      sm.store(lds[0] + NCH);
      __syncthreads();
      if (s + 1 < steps) load(s + 1);
      compute(lds[0]);
    }
  }

  finish<E, USE, NF, MF>(p, acc, m0 + wm * WM, n0 + (PAIR ? wn * (WN / 2) : wn * WN), split, mat);
}

// ------------------------------------------------- bf16, aligned operands
// The same product with operand tiles copied global -> LDS by the load-to-LDS
// instructions, as they lie in memory: 256 x 256 outputs a workgroup of eight
// waves, 128 x 64 a wave (128 accumulators a lane; two waves a SIMD cover each
// other's LDS reads and barriers), stages of 32 k's in four LDS buffers, two to
// three of them in flight.  An operand that is contiguous along its rows is
// read with the transposing LDS load.  Chunks of 16 bytes are permuted within
// their LDS rows through the global addresses, so that the fragments' reads
// spread over the banks: k-contiguous rows (four chunks) by row / 2, row-
// contiguous k's (32 chunks) by twice the k.  Results go to memory through LDS
// in whole rows of the tile (stored from the accumulators' layout, 8 bytes to
// each of 32 rows, a tile took 40 us).
constexpr int kDM = 256, kDN = 256, kDK = 32, kDBufs = 4, kDThreads = 512;
constexpr int kDMChunks = kDM * kDK / 8, kDNChunks = kDN * kDK / 8;  // of a stage

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;

// 16 bytes a lane from `g` to LDS byte `at` + 16 lane (at: uniform).  In
// assembly, since the compiler would wait for every copy in flight before any
// transposing LDS read; the kernel waits for its copies itself.  (M0 has no
// other use in it.)
__device__ __forceinline__ void copy_to_lds(const bf16* g, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(g) : "memory");
}

template <bool KC>
__device__ __forceinline__ int chunk_swizzle(int row) { return KC ? (row >> 1) & 3 : (row & 3) << 1; }

// Fragment of 32 rows from `r0` on at k-step ks of a stage.
template <bool KC, int ROWS>
__device__ __forceinline__ bf16x8 fragment(const uint4* b, int r0, int ks, int lane) {
  constexpr int C = ROWS / 8;
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

template <int USE>
__global__ __launch_bounds__(kDThreads, 2) void k_glu_direct(GluP<bf16> p) {
  constexpr bool PAIR = USE == kForward || USE == kProject;
  constexpr bool NKC = USE == kDx, MKC = USE != kDw;
  constexpr int NF = 2, MF = 4, NJ = kDNChunks / kDThreads, MJ = kDMChunks / kDThreads;
  __shared__ __align__(1024) uint4 lds[kDBufs][kDNChunks + kDMChunks];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave & 3, wm = wave >> 2;
  const TileAt t = tile_at<USE>(p);
  const int64_t n0 = (int64_t)t.n * (PAIR ? kDN / 2 : kDN), m0 = (int64_t)t.m * kDM;
  const int64_t kfrom = USE == kDw ? t.split * p.span : 0;
  const int64_t kend = USE == kDw && kfrom + p.span < p.K ? kfrom + p.span : p.K;
  const int64_t len = kend > kfrom ? kend - kfrom : 0;
  const int blocks = (int)(len / kDK);  // (len is a multiple of kDK)
  const int stages = USE == kDx ? 2 * blocks : blocks;

  // This lane's sources of the copies: chunk 64 (J wave + j) + lane of a stage.
  const bf16 *na[NJ], *ma[MJ];
  auto source = [&](bool kc, int id, int chunks, const bf16* b0, const bf16* b1, int64_t ld, int64_t first,
                    int64_t limit, bool pair) {
    if (kc) {
      const int row = id >> 2, c = (id & 3) ^ chunk_swizzle<true>(row);
      const int64_t r = first + row < limit ? first + row : limit - 1;  // (rows past the end are not stored)
      return b0 + r * ld + kfrom + c * 8;
    }
    // pair: a wave's 64 columns are 32 of gate, then the same 32 of up
    const int k = id / chunks, c = (id % chunks) ^ chunk_swizzle<false>(k);
    const int64_t r = first + (pair ? (c >> 3) * 32 + (c & 3) * 8 : c * 8);
    return (pair && (c & 4) ? b1 : b0) + (kfrom + k) * ld + (r < limit ? r : limit - 8);
  };
  const bf16* nbase = USE == kDw && t.mat ? p.n1 : p.n0;
#pragma unroll
  for (int j = 0; j < NJ; ++j) na[j] = source(NKC, (wave * NJ + j) * 64 + lane, kDN / 8, nbase, p.n1, p.nld0, n0, p.N, PAIR);
#pragma unroll
  for (int j = 0; j < MJ; ++j) ma[j] = source(MKC, (wave * MJ + j) * 64 + lane, kDM / 8, p.m0, p.m0, p.mld0, m0, p.M, false);
  // to the next stage, and (dx) from the last one of the first segment to the
  // first of the second
  const int64_t nstep = NKC ? kDK : kDK * p.nld0, mstep = MKC ? kDK : kDK * p.mld0;
  const int64_t nturn = USE == kDx ? p.n1 - p.n0 - (int64_t)(blocks - 1) * kDK : 0;
  const int64_t mturn = USE == kDx ? p.m1 - p.m0 - (int64_t)(blocks - 1) * kDK : 0;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&lds[0][0];
  auto issue = [&](int stage, int buf) {
    const uint32_t at = lds0 + (uint32_t)(buf * (kDNChunks + kDMChunks)) * 16;
    const bool turn = USE == kDx && stage + 1 == blocks;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      copy_to_lds(na[j], at + (uint32_t)(wave * NJ + j) * 1024);
      na[j] += turn ? nturn : nstep;
    }
#pragma unroll
    for (int j = 0; j < MJ; ++j) {
      copy_to_lds(ma[j], at + kDNChunks * 16 + (uint32_t)(wave * MJ + j) * 1024);
      ma[j] += turn ? mturn : mstep;
    }
  };

  // project: the tile of dh, 128 rows to each of the two buffers that fall
  // free before the last stages (rows of 16 chunks, permuted by row % 16)
  auto copy_dh = [&]() {
#pragma unroll
    for (int k = 0; k < kDM * 16 / kDThreads; ++k) {
      const int id = k * kDThreads + wave * 64 + lane, row = id >> 4, c = (id & 15) ^ (row & 15);
      const int64_t m = m0 + row < p.M ? m0 + row : p.M - 1, n = n0 + c * 8 < p.N ? n0 + c * 8 : p.N - 8;
      const int buf = (stages + (row >> 7)) & 3;
      copy_to_lds(p.dh + m * p.dhld + n,
                  lds0 + (uint32_t)(__builtin_amdgcn_readfirstlane(buf) * (kDNChunks + kDMChunks)) * 16 +
                      (uint32_t)((k * kDThreads + wave * 64) & 2047) * 16);
    }
  };

  floatx16 acc[NF][MF] = {};
  bf16x8 nf[2][NF], mf[2][MF];
  auto read = [&](int st, int ks) {
    const uint4 *nb = lds[st & 3], *mb = nb + kDNChunks;
#pragma unroll
    for (int i = 0; i < NF; ++i) nf[ks][i] = fragment<NKC, kDN>(nb, wn * 64 + i * 32, ks, lane);
#pragma unroll
    for (int j = 0; j < MF; ++j) mf[ks][j] = fragment<MKC, kDM>(mb, wm * 128 + j * 32, ks, lane);
  };
  auto multiply = [&](int ks) {
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int j = 0; j < MF; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(nf[ks][i], mf[ks][j], acc[i][j], 0, 0, 0);
  };
  if (stages > 0) {
    issue(0, 0);
    if (stages > 1) issue(1, 1);
    if (stages > 2) {
      issue(2, 2);
      asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    asm volatile("s_barrier" ::: "memory");
    read(0, 0);
    int s = 0;
    for (; s + 3 < stages; ++s) {
      read(s, 1);
      __builtin_amdgcn_sched_barrier(0);
      multiply(0);
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(4)\n\ts_barrier" ::: "memory");
      issue(s + 3, (s + 3) & 3);
      read(s + 1, 0);
      __builtin_amdgcn_sched_barrier(0);
      multiply(1);
    }
    if (USE == kProject && stages == 1) copy_dh();
    for (; s < stages; ++s) {
      read(s, 1);
      multiply(0);
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      if (USE == kProject && s + 2 == stages) copy_dh();
      read(s + 1 < stages ? s + 1 : s, 0);
      multiply(1);
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

  // The tile's rows in LDS: chunk c of row r (of C chunks) at r C + (c ^ r % 16).
  // Register 4 q + e of acc[i][j]: column 8 q + 4 (lane / 32) + e of fragment
  // i's 32, row lane % 32 of fragment j's.
  const int r32 = lane & 31, hi = lane >> 5;
  uint4* tile = lds[0];
  if constexpr (USE == kDw) {
    // fp32 parts, 128 rows at a time
    float* out = p.parts + ((int64_t)t.split * 2 + t.mat) * p.M * p.N;
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
              const floatx16& v = acc[i][j];
              tile[r * 64 + (c ^ (r & 15))] = __builtin_bit_cast(
                  uint4, make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
            }
      }
      __syncthreads();
#pragma unroll 4
      for (int k = 0; k < 128 * 64 / kDThreads; ++k) {
        const int id = threadIdx.x + k * kDThreads, r = id >> 6, c = id & 63;
        const int64_t m = m0 + half * 128 + r, n = n0 + c * 4;
        if (m < p.M && n < p.N) *reinterpret_cast<uint4*>(out + m * p.N + n) = tile[r * 64 + (c ^ (r & 15))];
      }
    }
  } else {
    constexpr int C = PAIR ? 16 : 32;  // chunks of a row
    // project: dh lies where dg goes, du in the other two buffers
    uint4* second = PAIR ? lds[(stages + 2) & 3] : nullptr;
    uint4* third = PAIR ? lds[(stages + 3) & 3] : nullptr;
    uint4 *first0 = USE == kProject ? lds[stages & 3] : tile, *first1 = USE == kProject ? lds[(stages + 1) & 3] : tile + 128 * C;
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
      for (int i = 0; i < (PAIR ? 1 : NF); ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = j * 32 + r32, c = (PAIR ? wn * 4 : wn * 8 + i * 4) + q;
          const int at = r * C + (c ^ (r & 15));
          Four<bf16>* o = reinterpret_cast<Four<bf16>*>((wm ? first1 : first0) + at) + hi;
          Four<bf16> w;
          if constexpr (PAIR) {
            float slope;
            if constexpr (USE == kForward) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float v = act_of(p.act, acc[0][j][4 * q + e], slope);
                w.e[e] = from_f32<bf16>(v * acc[NF / 2][j][4 * q + e]);
              }
            } else {
              const Four<bf16> d4 = *o;
              Four<bf16> x;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float v = act_of(p.act, acc[0][j][4 * q + e], slope), d = to_f32(d4.e[e]);
                w.e[e] = from_f32<bf16>(d * acc[NF / 2][j][4 * q + e] * slope);
                x.e[e] = from_f32<bf16>(d * v);
              }
              *(reinterpret_cast<Four<bf16>*>((wm ? third : second) + at) + hi) = x;
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) w.e[e] = from_f32<bf16>(acc[i][j][4 * q + e]);
          }
          *o = w;
        }
    __syncthreads();
    auto put = [&](const uint4* lo, const uint4* up, bf16* out, int64_t ld) {
#pragma unroll 4
      for (int k = 0; k < kDM * C / kDThreads; ++k) {
        const int id = threadIdx.x + k * kDThreads, row = id / C, c = id % C, r = row & 127;
        const int64_t m = m0 + row, n = n0 + c * 8;
        const uint4 v = (row >> 7 ? up : lo)[r * C + (c ^ (r & 15))];
        if (m < p.M && n < p.N) *reinterpret_cast<Vec<bf16, 8>*>(out + m * ld + n) = __builtin_bit_cast(Vec<bf16, 8>, v);
      }
    };
    put(first0, first1, p.out0, p.old0);
    if (USE == kProject) put(second, third, p.out1, p.old1);
  }
}

// dW from the row ranges' parts.
template <class E>
__global__ __launch_bounds__(256) void k_glu_join(const float* __restrict__ parts, uint32_t splits, int64_t M, int64_t N,
                                                  E* out0, int64_t ld0, E* out1, int64_t ld1) {
  const int64_t groups = (N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * M * groups) return;
  const int64_t mat = i / (M * groups), at = i - mat * M * groups, m = at / groups, n = (at - m * groups) * 4;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  const int valid = (int)(N - n < 4 ? N - n : 4);
  for (uint32_t s = 0; s < splits; ++s) {
    float v[4];
    load_four(parts + ((int64_t)s * 2 + mat) * M * N + m * N + n, valid, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] += v[e];
  }
  store_four(mat ? out1 + m * ld1 + n : out0 + m * ld0 + n, valid, t);
}

// Forward for a few rows (single frames of some voices): the weights' reading
// is all that counts, and its latency, so the vector unit multiplies.  A
// workgroup owns 32 columns (16 lanes x 2); the quarter-waves of 16 waves take
// every 64th k, each with all of its 8 loads of a round of 512 k's in flight
// at once; the 64 sums meet in registers, then in LDS.  (64 columns a workgroup
// leave most CUs idle: 512 x 1408, 8 rows: 11.8 us against 9.8.)
constexpr int kFewRows = 8, kFewThreads = 1024, kFewCols = 32, kFewK = 512;
constexpr int kFewLanes = kFewCols / 2, kFewSlices = kFewThreads / kFewLanes, kFewLoads = kFewK / kFewSlices;
template <class E>
__global__ __launch_bounds__(kFewThreads) void k_glu_few(GluP<E> p) {
  __shared__ __align__(16) float xs[kFewK][kFewRows];
  __shared__ float red[16][kFewCols][2][kFewRows + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slice = threadIdx.x / kFewLanes;
  const int64_t m0 = (int64_t)blockIdx.y * kFewRows, f = (int64_t)blockIdx.x * kFewCols + (lane % kFewLanes) * 2;
  const bool two = f + 1 < p.N;
  const int64_t col = two ? f : f < p.N ? f : p.N - 1;  // (columns past the end are not stored)
  float acc[2][2][kFewRows] = {};
  for (int64_t k0 = 0; k0 < p.K; k0 += kFewK) {
    float xv[kFewK * kFewRows / kFewThreads];
#pragma unroll
    for (int i = 0; i < kFewK * kFewRows / kFewThreads; ++i) {
      const int id = threadIdx.x + i * kFewThreads, m = id / kFewK, k = id % kFewK;
      xv[i] = k0 + k < p.K && m0 + m < p.M ? to_f32(p.m0[(m0 + m) * p.mld0 + k0 + k]) : 0.f;
    }
    Vec<E, 2> w[kFewLoads][2];
    const E *g = p.n0 + col, *u = p.n1 + col;
#pragma unroll
    for (int i = 0; i < kFewLoads; ++i) {
      const int64_t k = k0 + slice + kFewSlices * i, kc = k < p.K ? k : p.K - 1;  // (x is 0 past the end)
      if (two) {
        w[i][0] = *reinterpret_cast<const Vec<E, 2>*>(g + kc * p.nld0);
        w[i][1] = *reinterpret_cast<const Vec<E, 2>*>(u + kc * p.nld1);
      } else {
        w[i][0].e[0] = w[i][0].e[1] = g[kc * p.nld0];
        w[i][1].e[0] = w[i][1].e[1] = u[kc * p.nld1];
      }
    }
    if (k0 > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < kFewK * kFewRows / kFewThreads; ++i) {
      const int id = threadIdx.x + i * kFewThreads;
      xs[id % kFewK][id / kFewK] = xv[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kFewLoads; ++i) {
      // (past the end the weights are a row inside, which may hold anything)
      if (k0 + slice + kFewSlices * i >= p.K) continue;
#pragma unroll
      for (int m = 0; m < kFewRows; ++m) {
        const float x = xs[slice + kFewSlices * i][m];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int b = 0; b < 2; ++b) acc[a][b][m] = fmaf(x, to_f32(w[i][a].e[b]), acc[a][b][m]);
      }
    }
  }
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int m = 0; m < kFewRows; ++m) {
        float t = acc[a][b][m];
        t += __shfl_xor(t, 16, 64);
        t += __shfl_xor(t, 32, 64);
        if (lane < kFewLanes) red[wave][lane * 2 + b][a][m] = t;
      }
  __syncthreads();
  if (threadIdx.x >= kFewCols * kFewRows) return;
  const int c = threadIdx.x % kFewCols, m = threadIdx.x / kFewCols;
  const int64_t n = (int64_t)blockIdx.x * kFewCols + c;
  float s[2] = {0.f, 0.f}, slope;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    s[0] += red[w][c][0][m];
    s[1] += red[w][c][1][m];
  }
  if (m0 + m < p.M && n < p.N) p.out0[(m0 + m) * p.old0 + n] = from_f32<E>(act_of(p.act, s[0], slope) * s[1]);
}

// ------------------------------------------------------------------ shapes
// Large tiles where they come near to filling the chip's 256 CUs, else small
// ones.
template <class E>
bool large_tiles(int64_t M, int64_t cols) {
  const int64_t bm = sizeof(E) == 2 ? 256 : 128;
  return ((M + bm - 1) / bm) * ((cols + bm - 1) / bm) >= 128;
}

bool aligned16(const void* p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0; }

template <class E, int USE>
void product(GluP<E> p, bool large, hipStream_t st) {
  constexpr bool PAIR = USE == kForward || USE == kProject;
  constexpr int L = sizeof(E) == 2 ? 256 : 128;
  const int bm = large ? L : 64, bn = large ? L : 128, per = PAIR ? bn / 2 : bn;
  p.tiles_m = (uint32_t)((p.M + bm - 1) / bm);
  p.tiles_n = (uint32_t)((p.N + per - 1) / per);
  const dim3 grid(p.tiles_m * p.tiles_n * (USE == kDw ? 2 * p.splits : 1));
  if (!large) {
    k_glu<E, 64, 128, 32, 64, sizeof(E) == 2 ? 64 : 32, 1, USE><<<grid, kThreads, 0, st>>>(p);
  } else if constexpr (sizeof(E) == 4) {
    k_glu<E, 128, 128, 64, 64, 32, 1, USE><<<grid, kThreads, 0, st>>>(p);
  } else {
    // whole chunks and stages: every row (k-contiguous) or k (row-contiguous)
    // starts at 16 bytes, row-contiguous operands have a multiple of 8 rows,
    // results a multiple of 8 columns, the reduction is a multiple of 32, and
    // the two matrices share a stride
    const bool direct = aligned16(p.n0, p.nld0) && aligned16(p.n1, p.nld1) && aligned16(p.m0, p.mld0) &&
                        aligned16(p.m1, p.mld1) && p.nld0 == p.nld1 && p.mld0 == p.mld1 &&
                        p.N % 8 == 0 && (USE != kDw || p.M % 8 == 0) && p.K % kDK == 0 && p.K > 0 &&
                        (USE != kProject || aligned16(p.dh, p.dhld)) && (USE != kDw || p.parts);
    if (direct) {
      p.tiles_m = (uint32_t)((p.M + kDM - 1) / kDM);
      p.tiles_n = (uint32_t)((p.N + (PAIR ? kDN / 2 : kDN) - 1) / (PAIR ? kDN / 2 : kDN));
      k_glu_direct<USE><<<dim3(p.tiles_m * p.tiles_n * (USE == kDw ? 2 * p.splits : 1)), kDThreads, 0, st>>>(p);
    } else {
      k_glu<E, 256, 256, 128, 128, 64, 2, USE><<<grid, kThreads, 0, st>>>(p);
    }
  }
}

// The weight gradients' products: tiles and row ranges.  As many ranges, of 512
// rows or more, as make the rounds over the 256 CUs full, against the time
// that the partial sums take: a tile's 512 rows take a CU about `unit`, and a
// tile's part takes the whole chip about `join` to write and read.
struct DwShape {
  bool large;
  int64_t rows;     // in the ranges; the rest (bf16 stages are whole) is a part of its own
  int64_t span;     // rows of a range
  uint32_t ranges, parts;
  bool in_parts;    // the products leave fp32 parts (else they write the gradients)
};
template <class E>
DwShape dw_shape(const dgen_hip_mlp& a) {
  constexpr bool kHalf = sizeof(E) == 2;
  const int64_t L = kHalf ? 256 : 128;
  auto count = [&](int64_t bm, int64_t bn) {
    return 2 * ((a.width + bm - 1) / bm) * ((a.hidden + bn - 1) / bn);
  };
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(a.rows / 512, 32));
  DwShape d{};
  d.large = count(L, L) * most >= 128;
  d.rows = kHalf && d.large ? a.rows / kDK * kDK : a.rows;
  const int64_t tiles = d.large ? count(L, L) : count(64, 128);
  const double unit = !d.large ? 4e-6 : kHalf ? 14e-6 : 21e-6, join = d.large ? 0.13e-6 : 0.02e-6;
  int64_t best = 1;
  double least = 0;
  for (int64_t s = 1; s <= most; ++s) {
    const double rounds = (double)((tiles * s + 255) / 256);
    const double cost = rounds * ((double)a.rows / (512.0 * (double)s)) * unit + (s > 1 ? (double)(s * tiles) * join : 0);
    if (s == 1 || cost < least) best = s, least = cost;
  }
  d.span = std::max<int64_t>(64, ((d.rows + best - 1) / best + 63) / 64 * 64);
  d.ranges = (uint32_t)std::max<int64_t>(1, (d.rows + d.span - 1) / d.span);
  d.parts = d.ranges + (d.rows < a.rows ? 1 : 0);
  d.in_parts = d.parts > 1 || (kHalf && d.large);
  return d;
}

// Rows of dg and du start at 16 bytes.
int64_t dg_stride(const dgen_hip_mlp& a) { return (a.hidden + 7) & ~int64_t(7); }

struct MlpWs {
  int64_t dg, du, parts, total;  // bytes
};
MlpWs mlp_ws(const dgen_hip_mlp& a) {
  MlpWs w{};
  const int64_t es = a.type == DGEN_HIP_BF16 ? 2 : 4;
  const DwShape d = a.type == DGEN_HIP_BF16 ? dw_shape<bf16>(a) : dw_shape<float>(a);
  w.dg = w.du = align256(a.rows * dg_stride(a) * es);
  w.parts = d.in_parts ? align256((int64_t)d.parts * 2 * a.width * a.hidden * 4) : 0;
  w.total = w.dg + w.du + w.parts;
  return w;
}

template <class E>
void mlp_launch(const dgen_hip_mlp& a, bool backward, hipStream_t st) {
  GluP<E> p{};
  p.act = a.act;
  p.splits = 1;
  p.n0 = (const E*)a.w_gate, p.n1 = (const E*)a.w_up, p.nld0 = a.w_gate_stride, p.nld1 = a.w_up_stride;
  p.m0 = p.m1 = (const E*)a.x, p.mld0 = p.mld1 = a.x_stride;
  p.M = a.rows, p.N = a.hidden, p.K = a.width;
  if (!backward) {
    p.out0 = (E*)a.h, p.old0 = a.h_stride;
    if (a.rows <= 2 * kFewRows) {
      k_glu_few<E><<<dim3((unsigned)((a.hidden + kFewCols - 1) / kFewCols), (unsigned)((a.rows + kFewRows - 1) / kFewRows)),
                     kFewThreads, 0, st>>>(p);
    } else {
      product<E, kForward>(p, large_tiles<E>(a.rows, 2 * a.hidden), st);
    }
    return;
  }
  const MlpWs w = mlp_ws(a);
  E* dg = (E*)a.workspace;
  E* du = (E*)((char*)a.workspace + w.dg);
  float* parts = (float*)((char*)a.workspace + w.dg + w.du);
  if (a.rows > 0) {
    GluP<E> q = p;
    q.out0 = dg, q.out1 = du, q.old0 = q.old1 = dg_stride(a);
    q.dh = (const E*)a.dh, q.dhld = a.dh_stride;
    product<E, kProject>(q, large_tiles<E>(a.rows, 2 * a.hidden), st);
    q = p;
    q.m0 = dg, q.m1 = du, q.mld0 = q.mld1 = dg_stride(a);
    q.N = a.width, q.K = a.hidden;
    q.out0 = (E*)a.dx, q.old0 = a.dx_stride;
    product<E, kDx>(q, large_tiles<E>(a.rows, a.width), st);
  }
  GluP<E> q = p;
  const DwShape d = dw_shape<E>(a);
  q.n0 = dg, q.n1 = du, q.nld0 = q.nld1 = dg_stride(a);
  q.M = a.width, q.N = a.hidden, q.K = d.rows;
  q.out0 = (E*)a.dw_gate, q.old0 = a.dw_gate_stride, q.out1 = (E*)a.dw_up, q.old1 = a.dw_up_stride;
  q.parts = d.in_parts ? parts : nullptr;
  q.splits = d.ranges, q.span = d.span;
  product<E, kDw>(q, d.large, st);
  if (d.rows < a.rows) {
    GluP<E> r = q;
    r.n0 += d.rows * r.nld0, r.n1 += d.rows * r.nld1, r.m0 += d.rows * r.mld0, r.m1 = r.m0;
    r.K = r.span = a.rows - d.rows;
    r.splits = 1;
    r.parts += (int64_t)d.ranges * 2 * a.width * a.hidden;
    product<E, kDw>(r, d.large, st);
  }
  if (d.in_parts) {
    const int64_t n = 2 * a.width * ((a.hidden + 3) / 4);
    k_glu_join<E><<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>(parts, d.parts, a.width, a.hidden, q.out0, q.old0,
                                                                     q.out1, q.old1);
  }
}

}  // namespace

int64_t mlp_workspace(const dgen_hip_mlp& a, bool backward) { return backward ? mlp_ws(a).total : 0; }

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
    const int64_t need = mlp_workspace(a, true);
    DGEN_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= (uint64_t)need && (uintptr_t)a.workspace % 256 == 0),
                 "%s: workspace of %llu bytes, %lld needed (256-byte aligned)", what,
                 (unsigned long long)a.workspace_bytes, (long long)need);
  }
  if (dry || (empty && !backward)) return 0;
  if (a.type == DGEN_HIP_BF16) mlp_launch<bf16>(a, backward, st);
  else mlp_launch<float>(a, backward, st);
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
