// The norm after a block, its gate, the residual's scale and addition, and the
// norm before the next block, forward and backward.
//
// Forward, per row of n columns: p = x rx post, rx = 1 / sqrt(mean(x^2) + eps),
// s = scale residual + G(gate) p, y = s rs pre, rs = 1 / sqrt(mean(s^2) + eps).
// As one pass: a row's threads hold it in registers, so x, the residual and the
// gate are read once and s and y written once; of three operators in a row two
// more tensors would go to memory and back.  Bound by memory: 32000 x 512, bf16
// with the stream in fp32 and a gate of each row, 229 MB in 52.6 us, 48 of them the
// kernel (4.7 TB/s; a copy reaches 5.1).
//
// Backward, from the stored s, with the gradients dy of y and ds of s:
//   da = rs (dy pre - s rs^2 mean(dy pre s)) + ds       gradient of the sum
//   w  = da G post,  dx = rx (w - x rx^2 mean(w x))
//   dresidual = scale da,  dgate = da p G',  dscale = sum da residual,
//   dpost = sum da G x rx,  dpre = sum dy s rs
// Two sums over the row after one another, in registers again.  Each workgroup
// walks rows and leaves one partial row of the sums over rows, added in a fixed
// order afterwards; where a gate belongs to many rows, a workgroup walks the rows
// of one gate after another.  The same rows backward, a gate for each thousand: 426 MB
// in 102 us, 95 of them the rows (4.5 TB/s) and 8 the sums.
#include "seq.h"

namespace dgen {

namespace {

constexpr int64_t kMaxWidth = 8192;

// Threads per row; each has one to four groups of four columns, of which the
// backward pass holds ten (512 threads leave 256 registers).
template <int TPR>
constexpr int block_threads() { return TPR > 256 ? TPR : 256; }
int row_threads(int64_t n) { return n <= 128 ? 16 : n <= 512 ? 64 : n <= 2048 ? 256 : 512; }

struct Act {
  float g, slope;
};
// The gate's factor and its derivative; e^-|z| keeps both exact far out.
__device__ __forceinline__ Act act_of(float z, int act) {
  if (act == DGEN_HIP_GATE_PLAIN) return {z, 1.f};
  const float e = exp_accurate(-fabsf(z)), p = __builtin_amdgcn_rcpf(1.f + e);
  return {z >= 0.f ? p : e * p, e * p * p};
}

template <class TX, class TS, int TPR, int IT>
__global__ __launch_bounds__(block_threads<TPR>()) void k_block_norm(dgen_hip_block_norms a, float inv_n) {
  constexpr int RPB = block_threads<TPR>() / TPR;
  __shared__ float red[2][16];
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const int c0 = (threadIdx.x % TPR) * 4, n = (int)a.width;
  const bool live = row < a.rows;  // rows of one workgroup end together: no early exit before a barrier
  const TX *xp = (const TX*)a.x + row * a.x_stride, *gp = (const TX*)a.gate;
  const TS* rp = (const TS*)a.residual + row * a.residual_stride;
  if (gp) gp += (a.gate_rows == 1 ? row : row / a.gate_rows) * a.gate_stride;
  const float eps = (float)a.eps;
  float x[IT][4], r[IT][4], g[IT][4];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = c0 + i * TPR * 4, left = live ? n - c : 0;
    load_four(xp + c, left, x[i]);
    load_four(rp + c, left, r[i]);
    if (gp) load_four(gp + c, left, g[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = fmaf(x[i][e], x[i][e], sum);
  }
  const float rx = root_of(fmaf(row_sum<TPR>(sum, red[0]), inv_n, eps));
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = c0 + i * TPR * 4;
    float w[4];
    load_four(a.post + c, n - c, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i][e] *= rx * w[e];
    if (a.scale) {
      load_four(a.scale + c, n - c, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) r[i][e] *= w[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p = gp ? act_of(g[i][e], a.act).g * x[i][e] : x[i][e];
      r[i][e] += p;
      if (c + e < n) sum = fmaf(r[i][e], r[i][e], sum);  // (act(0) p is 0 past the row's end, but for p = NaN)
    }
  }
  const float rs = root_of(fmaf(row_sum<TPR>(sum, red[1]), inv_n, eps));
  if (!live) return;
  TX* yp = (TX*)a.y + row * a.y_stride;
  TS* sp = (TS*)a.s + row * a.s_stride;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = c0 + i * TPR * 4;
    float w[4];
    load_four(a.pre + c, n - c, w);
    store_four(sp + c, n - c, r[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = r[i][e] * rs * w[e];
    store_four(yp + c, n - c, w);
  }
}

// How the backward pass is cut: `blocks` workgroups along the gates (one gate of
// all rows, where each row has its own or none has), `splits` along a gate's rows.
struct Cut {
  int64_t gates, rows;  // of them, and rows of each
  int64_t blocks, splits;
  bool shared;          // gates of many rows
};

template <class TX, class TS, int TPR, int IT>
__global__ __launch_bounds__(block_threads<TPR>(), TPR <= 256 ? 4 : 2) void k_block_norm_bwd(dgen_hip_block_norms a, float inv_n, Cut cut,
                                                                        float* __restrict__ parts,
                                                                        float* __restrict__ gate_parts) {
  constexpr int RPB = block_threads<TPR>() / TPR;
  __shared__ float red[4][16];
  __shared__ float acc[RPB > 1 ? RPB : 1][RPB > 1 ? TPR * 4 : 1];
  const int sub = threadIdx.x / TPR, c0 = (threadIdx.x % TPR) * 4, n = (int)a.width;
  const int64_t block = blockIdx.x / (uint32_t)cut.splits, split = blockIdx.x % (uint32_t)cut.splits;
  const float eps = (float)a.eps;
  float dpost[IT][4] = {}, dpre[IT][4] = {}, dscale[IT][4] = {};

  // A group of four columns summed over the workgroup's rows, in the first of them.
  auto over_rows = [&](float (&v)[4]) {
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[sub][c0 + e] = v[e];
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float t = 0.f;
#pragma unroll
          for (int q = 0; q < RPB; ++q) t += acc[q][c0 + e];
          v[e] = t;
        }
      }
    }
  };

  for (int64_t gate = block; gate < cut.gates; gate += cut.blocks) {
    float dg[IT][4] = {};
    const int64_t base = gate * cut.rows;
    for (int64_t first = split * RPB; first < cut.rows; first += cut.splits * RPB) {
      const bool live = first + sub < cut.rows;
      const int64_t row = base + first + sub;
      const TX* gp = a.gate ? (const TX*)a.gate + (cut.shared ? gate : row) * a.gate_stride : nullptr;
      float x[IT][4], s[IT][4], v[IT][4], d[IT][4] = {}, z[IT][4], r[IT][4], w[4];
      float sx = 0.f, ss = 0.f, dot = 0.f;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = c0 + i * TPR * 4, left = live ? n - c : 0;
        load_four((const TX*)a.x + row * a.x_stride + c, left, x[i]);
        load_four((const TS*)a.s + row * a.s_stride + c, left, s[i]);
        load_four((const TX*)a.dy + row * a.dy_stride + c, left, v[i]);
        if (a.ds) load_four((const TS*)a.ds + row * a.ds_stride + c, left, d[i]);
        if (gp) load_four(gp + c, left, z[i]);
        if (a.scale) load_four((const TS*)a.residual + row * a.residual_stride + c, left, r[i]);
      }
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = c0 + i * TPR * 4;
        load_four(a.pre + c, n - c, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sx = fmaf(x[i][e], x[i][e], sx);
          ss = fmaf(s[i][e], s[i][e], ss);
          dot = fmaf(v[i][e] * w[e], s[i][e], dot);
        }
      }
      sx = row_sum<TPR>(sx, red[0]);
      ss = row_sum<TPR>(ss, red[1]);
      dot = row_sum<TPR>(dot, red[2]);
      const float rx = root_of(fmaf(sx, inv_n, eps)), rs = root_of(fmaf(ss, inv_n, eps));
      const float k = dot * inv_n * rs * rs;
      float dot2 = 0.f;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = c0 + i * TPR * 4;
        float q[4];
        load_four(a.pre + c, n - c, w);
        load_four(a.post + c, n - c, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Act f = gp ? act_of(z[i][e], a.act) : Act{1.f, 0.f};
          const float da = fmaf(rs, fmaf(v[i][e], w[e], -s[i][e] * k), d[i][e]), nx = x[i][e] * rx;
          if (live) {  // (rows past the end hold zeros, and no gradient)
            dpre[i][e] = fmaf(v[i][e], s[i][e] * rs, dpre[i][e]);
            dpost[i][e] = fmaf(da * f.g, nx, dpost[i][e]);
            if (a.scale) dscale[i][e] = fmaf(da, r[i][e], dscale[i][e]);
          }
          d[i][e] = da;
          if (gp) {
            z[i][e] = da * nx * q[e] * f.slope;  // the gate's gradient
            if (cut.shared && live) dg[i][e] += z[i][e];
          }
          v[i][e] = da * f.g * q[e];
          dot2 = fmaf(v[i][e], x[i][e], dot2);
        }
      }
      dot2 = row_sum<TPR>(dot2, red[3]);
      const float k2 = dot2 * inv_n * rx * rx;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = c0 + i * TPR * 4, left = live ? n - c : 0;
        if (gp && !cut.shared) store_four((TX*)a.dgate + row * a.dgate_stride + c, left, z[i]);
        if (a.scale) {
          load_four(a.scale + c, n - c, w);
#pragma unroll
          for (int e = 0; e < 4; ++e) d[i][e] *= w[e];
        }
        store_four((TS*)a.dresidual + row * a.dresidual_stride + c, left, d[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = rx * fmaf(-x[i][e], k2, v[i][e]);
        store_four((TX*)a.dx + row * a.dx_stride + c, left, v[i]);
      }
    }
    if (cut.shared) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = c0 + i * TPR * 4;
        over_rows(dg[i]);
        if (sub != 0) continue;
        if (cut.splits > 1) store_four(gate_parts + (gate * cut.splits + split) * n + c, n - c, dg[i]);
        else store_four((TX*)a.dgate + gate * a.dgate_stride + c, n - c, dg[i]);
      }
    }
  }
  const int sums = a.scale ? 3 : 2;
  float* out = parts + (int64_t)blockIdx.x * sums * n;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = c0 + i * TPR * 4;
    over_rows(dpost[i]);
    over_rows(dpre[i]);
    if (a.scale) over_rows(dscale[i]);
    if (sub != 0) continue;
    store_four(out + c, n - c, dpost[i]);
    store_four(out + n + c, n - c, dpre[i]);
    if (a.scale) store_four(out + 2 * n + c, n - c, dscale[i]);
  }
}

// The last sums: gates' gradients from those of their rows' splits in the first
// workgroups, the partial rows in the others.
template <class TX>
__global__ __launch_bounds__(kSumThreads) void k_block_sums(const float* __restrict__ gate_parts, int64_t gates, int64_t splits,
                                                            int n, TX* __restrict__ out, int64_t stride, int64_t gate_blocks,
                                                            const float* __restrict__ parts, int64_t rows, SumOut sums,
                                                            int64_t width) {
  __shared__ float red[kSumThreads / kSumCols][kSumCols + 1];
  if (blockIdx.x >= gate_blocks) return sum_parts_block(parts, rows, sums, width, blockIdx.x - gate_blocks, red);
  const int64_t at = (int64_t)blockIdx.x * kSumThreads + threadIdx.x;
  if (at >= gates * n) return;
  const int64_t gate = at / n, c = at % n;
  const float* p = gate_parts + gate * splits * n + c;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  int64_t k = 0;
  for (; k + 3 < splits; k += 4)
#pragma unroll
    for (int q = 0; q < 4; ++q) t[q] += p[(k + q) * n];
  for (; k < splits; ++k) t[0] += p[k * n];
  out[gate * stride + c] = from_f32<TX>((t[0] + t[1]) + (t[2] + t[3]));
}

// Two or more steps a workgroup, up to four workgroups a CU, as in the norm.
Cut cut_of(const dgen_hip_block_norms& a) {
  const int tpr = row_threads(a.width);
  const int64_t rpb = tpr > 256 ? 1 : 256 / tpr;
  Cut c;
  c.shared = a.gate && a.gate_rows > 1;
  c.gates = c.shared ? a.rows / a.gate_rows : 1;
  c.rows = c.shared ? a.gate_rows : a.rows;
  const int64_t steps = (c.rows + rpb - 1) / rpb;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>((c.gates * steps + 1) / 2, 1024));
  c.blocks = std::min(c.gates, most);
  c.splits = std::max<int64_t>(1, std::min(most / std::max<int64_t>(c.gates, 1), steps));
  return c;
}

int64_t parts_bytes(const dgen_hip_block_norms& a, const Cut& c) {
  return align256(c.blocks * c.splits * a.width * (a.scale ? 3 : 2) * (int64_t)sizeof(float));
}

template <class TX, class TS, int TPR, int IT>
void block_launch(const dgen_hip_block_norms& a, bool backward, hipStream_t st) {
  constexpr int T = block_threads<TPR>(), RPB = T / TPR;
  const float inv = 1.f / (float)a.width;
  if (!backward) {
    k_block_norm<TX, TS, TPR, IT><<<dim3((unsigned)((a.rows + RPB - 1) / RPB)), T, 0, st>>>(a, inv);
    return;
  }
  const Cut c = cut_of(a);
  float *parts = (float*)a.workspace, *gate_parts = (float*)((char*)a.workspace + parts_bytes(a, c));
  const int64_t groups = c.blocks * c.splits;
  k_block_norm_bwd<TX, TS, TPR, IT><<<dim3((unsigned)groups), T, 0, st>>>(a, inv, c, parts, gate_parts);
  const SumOut sums = {{a.dpost, a.dpre, a.dscale}, {a.width, a.width, a.scale ? a.width : 0}};
  const int64_t width = a.width * (a.scale ? 3 : 2);
  const int64_t gates = c.shared && c.splits > 1 ? (c.gates * a.width + kSumThreads - 1) / kSumThreads : 0;
  k_block_sums<TX><<<dim3((unsigned)(gates + (width + kSumCols - 1) / kSumCols)), kSumThreads, 0, st>>>(
      gate_parts, c.gates, c.splits, (int)a.width, (TX*)a.dgate, a.dgate_stride, gates, parts, groups, sums, width);
}

template <class TX, class TS>
void block_shape(const dgen_hip_block_norms& a, bool backward, hipStream_t st) {
  const int tpr = row_threads(a.width);
  const int64_t it = (a.width + 4 * tpr - 1) / (4 * tpr);
  switch (tpr) {
    case 16: return it > 1 ? block_launch<TX, TS, 16, 2>(a, backward, st) : block_launch<TX, TS, 16, 1>(a, backward, st);
    case 64: return it > 1 ? block_launch<TX, TS, 64, 2>(a, backward, st) : block_launch<TX, TS, 64, 1>(a, backward, st);
    case 256: return it > 1 ? block_launch<TX, TS, 256, 2>(a, backward, st) : block_launch<TX, TS, 256, 1>(a, backward, st);
    default: return it > 2 ? block_launch<TX, TS, 512, 4>(a, backward, st) : block_launch<TX, TS, 512, 2>(a, backward, st);
  }
}

}  // namespace

int64_t block_workspace(const dgen_hip_block_norms& a, bool backward) {
  if (!backward) return 0;
  const Cut c = cut_of(a);
  return parts_bytes(a, c) +
         (c.shared && c.splits > 1 ? align256(c.gates * c.splits * a.width * (int64_t)sizeof(float)) : 0);
}

int block_run(const dgen_hip_block_norms& a, bool backward, hipStream_t st, bool dry) {
  const char* what = backward ? "block_norm_backward" : "block_norm";
  DGEN_REQUIRE(a.struct_size == sizeof(a), "%s: struct_size %u, expected %zu", what, a.struct_size, sizeof(a));
  DGEN_REQUIRE((a.x_type == DGEN_HIP_F32 || a.x_type == DGEN_HIP_BF16) &&
                   (a.s_type == DGEN_HIP_F32 || a.s_type == DGEN_HIP_BF16),
               "%s: types %d, %d", what, a.x_type, a.s_type);
  DGEN_REQUIRE(a.act == DGEN_HIP_GATE_PLAIN || a.act == DGEN_HIP_GATE_SIGMOID, "%s: act %d", what, a.act);
  DGEN_REQUIRE(a.width >= 1 && a.width <= kMaxWidth, "%s: width %lld outside [1, %lld]", what, (long long)a.width,
               (long long)kMaxWidth);
  // (a launch takes fewer than 2^32 threads)
  const int64_t most = (int64_t(1) << 31) / row_threads(a.width);
  DGEN_REQUIRE(a.rows >= 0 && a.rows < most, "%s: rows %lld outside [0, %lld) at width %lld", what, (long long)a.rows,
               (long long)most, (long long)a.width);
  DGEN_REQUIRE(a.gate_rows >= 1 && (a.rows == 0 || a.rows % a.gate_rows == 0), "%s: gate_rows %lld of %lld rows", what,
               (long long)a.gate_rows, (long long)a.rows);
  // (squares of small rows are lost below 2^-149: the least eps stands far above that)
  DGEN_REQUIRE(a.eps >= 1e-30 && a.eps < 1e30, "%s: eps %g outside [1e-30, 1e30)", what, a.eps);
  DGEN_REQUIRE(a.post && a.pre, "%s: null post or pre", what);
  const int64_t gates = a.rows / a.gate_rows;
  // inputs may repeat rows (stride 0); outputs may not
  auto apart = [&](const void* p, int64_t s, int64_t rows) { return !p || rows <= 1 || s >= a.width; };
  DGEN_REQUIRE(a.x_stride >= 0 && a.residual_stride >= 0 && a.gate_stride >= 0, "%s: negative stride", what);
  DGEN_REQUIRE((a.x && a.s) || a.rows == 0, "%s: null x or s", what);
  if (!backward) {
    DGEN_REQUIRE((a.residual && a.y) || a.rows == 0, "%s: null residual or y", what);
    DGEN_REQUIRE(apart(a.y, a.y_stride, a.rows) && apart(a.s, a.s_stride, a.rows), "%s: output rows overlap", what);
  } else {
    DGEN_REQUIRE((a.dy && a.dx && a.dresidual && (a.residual || !a.scale) && (a.dgate || !a.gate)) || a.rows == 0,
                 "%s: null dy, dx, dresidual, residual or dgate", what);
    DGEN_REQUIRE(a.dpost && a.dpre && !a.dscale == !a.scale, "%s: null dpost, dpre or dscale", what);
    DGEN_REQUIRE(a.dy_stride >= 0 && a.s_stride >= 0 && a.ds_stride >= 0, "%s: negative stride", what);
    DGEN_REQUIRE(apart(a.dx, a.dx_stride, a.rows) && apart(a.dresidual, a.dresidual_stride, a.rows) &&
                     apart(a.dgate, a.dgate_stride, gates),
                 "%s: output rows overlap", what);
    const int64_t need = block_workspace(a, true);
    DGEN_REQUIRE(a.rows == 0 || (a.workspace && a.workspace_bytes >= (uint64_t)need),
                 "%s: workspace of %llu bytes, %lld needed", what, (unsigned long long)a.workspace_bytes,
                 (long long)need);
  }
  if (dry || (a.rows == 0 && !backward)) return 0;
  const bool xb = a.x_type == DGEN_HIP_BF16, sb = a.s_type == DGEN_HIP_BF16;
  if (a.rows == 0) {
    // no rows: zeros
    enqueue_sum_parts(st, a.post, 0, {{a.dpost, a.dpre, a.dscale}, {a.width, a.width, a.scale ? a.width : 0}});
  } else if (xb) {
    sb ? block_shape<bf16, bf16>(a, backward, st) : block_shape<bf16, float>(a, backward, st);
  } else {
    sb ? block_shape<float, bf16>(a, backward, st) : block_shape<float, float>(a, backward, st);
  }
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
