// Root-mean-square norm with the residual's addition, forward and backward,
// and the sums over partial rows that the sequence operators' backward passes
// end with.
//
// Forward, per row of n columns: s = x + residual, r = 1 / sqrt(mean(s^2) +
// eps), y = s r w.  One pass: TPR threads hold the row in registers (4 IT
// values each), so x and the residual are read once and y and s written once:
// bound by memory.  Backward: with v = dy w, dx = r (v - s r^2 mean(v s)) +
// ds, again one pass over registers (mean(s^2) is formed again from s, so no
// statistics are kept); each thread adds its columns' dy s r over the rows
// that its workgroup walks, one partial row per workgroup, summed in a fixed
// order afterwards.
//
// Measured on operands that the caches do not hold (a large copy: 4.97 TB/s):
// forward of 32000 x 512, x and y bf16, residual and sum fp32, 40 us, 4.9 TB/s,
// all fp32 48 us, 5.5 TB/s; backward with ds, dy bf16 and the rest fp32, 44 us,
// 5.2 TB/s, and 7 us for the partial rows; backward of 4001 x 1023 fp32 with ds
// 18 us, 3.6 TB/s, and 5 us.
#include "seq.h"

namespace dgen {

namespace {

template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  // butterfly within the wave (every lane gets the sum)
#pragma unroll
  for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += red[i];
  }
  return v;
}

// 1 / sqrt(v); the instruction takes numbers below 2^-126 (small rows without
// an eps) for 0.
__device__ __forceinline__ float root_of(float v) {
  const bool low = v < 0x1p-100f;
  return __builtin_amdgcn_rsqf(low ? v * 0x1p100f : v) * (low ? 0x1p50f : 1.f);
}

template <int TPR>
constexpr int norm_threads() { return TPR > 256 ? TPR : 256; }

template <class TX, class TS, int TPR, int IT>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_rms_norm(
    const TX* x, int64_t xld, const TS* res, int64_t rld, TX* y, int64_t yld, TS* s, int64_t sld,
    const float* __restrict__ w, int64_t rows, int n, float inv_n, float eps) {
  constexpr int RPB = norm_threads<TPR>() / TPR;
  __shared__ float red[16];
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const int c0 = (threadIdx.x % TPR) * 4;
  const bool live = row < rows;  // rows of one workgroup end together: no early exit before a barrier
  float a[IT][4];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = c0 + i * TPR * 4;
    load_four(x + row * xld + c, live ? n - c : 0, a[i]);
    if (res) {
      float b[4];
      load_four(res + row * rld + c, live ? n - c : 0, b);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[i][e] += b[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = fmaf(a[i][e], a[i][e], ss);
  }
  ss = row_sum<TPR>(ss, red);
  if (!live) return;
  const float r = root_of(fmaf(ss, inv_n, eps));
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = c0 + i * TPR * 4;
    float g[4];
    load_four(w + c, n - c, g);
    if (res) store_four(s + row * sld + c, n - c, a[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] = a[i][e] * r * g[e];
    store_four(y + row * yld + c, n - c, g);
  }
}

template <class TX, class TS, int TPR, int IT>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_rms_norm_bwd(
    const TX* dy, int64_t dyld, const TS* s, int64_t sld, const TS* ds, int64_t dsld, TS* dx, int64_t dxld,
    const float* __restrict__ w, float* __restrict__ parts, int64_t rows, int n, float inv_n, float eps) {
  constexpr int RPB = norm_threads<TPR>() / TPR;
  __shared__ float red[2][16];
  __shared__ float acc[RPB > 1 ? RPB : 1][RPB > 1 ? TPR * 4 : 1];
  const int sub = threadIdx.x / TPR, c0 = (threadIdx.x % TPR) * 4;
  float dw[IT][4] = {};
  for (int64_t first = (int64_t)blockIdx.x * RPB; first < rows; first += (int64_t)gridDim.x * RPB) {
    const int64_t row = first + sub;
    const bool live = row < rows;
    float a[IT][4], v[IT][4], g[4];
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = c0 + i * TPR * 4, left = live ? n - c : 0;
      load_four(s + row * sld + c, left, a[i]);
      load_four(dy + row * dyld + c, left, v[i]);
      load_four(w + c, n - c, g);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ss = fmaf(a[i][e], a[i][e], ss);
        dot = fmaf(v[i][e] * g[e], a[i][e], dot);
      }
    }
    ss = row_sum<TPR>(ss, red[0]);
    dot = row_sum<TPR>(dot, red[1]);
    const float r = root_of(fmaf(ss, inv_n, eps));
    const float k = dot * inv_n * r * r;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = c0 + i * TPR * 4, left = live ? n - c : 0;
      float o[4] = {0.f, 0.f, 0.f, 0.f};
      load_four(w + c, n - c, g);
      if (ds) load_four(ds + row * dsld + c, left, o);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // rows past the end hold zeros: r is finite there (eps > 0) or the
        // row's terms are dropped
        if (live) dw[i][e] = fmaf(v[i][e], a[i][e] * r, dw[i][e]);
        o[e] = fmaf(r, fmaf(v[i][e], g[e], -a[i][e] * k), o[e]);
      }
      store_four(dx + row * dxld + c, left, o);
    }
  }
  float* out = parts + (int64_t)blockIdx.x * n;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = c0 + i * TPR * 4;
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[sub][c0 + e] = dw[i][e];
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float t = 0.f;
#pragma unroll
          for (int q = 0; q < RPB; ++q) t += acc[q][c0 + e];
          dw[i][e] = t;
        }
      }
    }
    if (sub == 0) store_four(out + c, n - c, dw[i]);
  }
}

__global__ __launch_bounds__(kSumThreads) void k_sum_parts(const float* __restrict__ ws, int64_t parts, SumOut o,
                                                           int64_t width) {
  __shared__ float red[kSumThreads / kSumCols][kSumCols + 1];
  sum_parts_block(ws, parts, o, width, blockIdx.x, red);
}

constexpr int64_t kMaxWidth = 32768;

// Threads per row and registers (groups of four columns) per thread.
void row_shape(int64_t n, int& tpr, int& it) {
  tpr = n <= 128 ? 16 : n <= 2048 ? 64 : n <= 8192 ? 256 : 1024;
  const int64_t groups = (n + 4 * tpr - 1) / (4 * tpr);
  it = 1;
  while (it < groups) it *= 2;
}

// Workgroups of the backward pass: each walks rows and leaves one partial
// row.  Two or more steps each, up to four workgroups a CU (calls, 32000 x 512:
// 48 us with 1024 workgroups, 64 with 512; 4001 x 1023, 1001 steps: 19.8 us with
// 512, 21.0 with 1001, whose partial rows take longer to add).
int64_t norm_blocks(const dgen_hip_norm& a) {
  int tpr, it;
  row_shape(a.width, tpr, it);
  const int64_t rpb = tpr > 256 ? 1 : 256 / tpr, steps = (a.rows + rpb - 1) / rpb;
  return std::min<int64_t>((steps + 1) / 2, 1024);
}

template <class TX, class TS, int TPR, int IT>
void norm_launch(const dgen_hip_norm& a, bool backward, hipStream_t st) {
  constexpr int T = norm_threads<TPR>(), RPB = T / TPR;
  const float inv = 1.f / (float)a.width;
  if (!backward) {
    k_rms_norm<TX, TS, TPR, IT><<<dim3((unsigned)((a.rows + RPB - 1) / RPB)), T, 0, st>>>(
        (const TX*)a.x, a.x_stride, (const TS*)a.residual, a.residual_stride, (TX*)a.y, a.y_stride, (TS*)a.s,
        a.s_stride, a.weight, a.rows, (int)a.width, inv, a.eps);
  } else {
    const int64_t nb = norm_blocks(a);
    float* parts = (float*)a.workspace;
    k_rms_norm_bwd<TX, TS, TPR, IT><<<dim3((unsigned)nb), T, 0, st>>>(
        (const TX*)a.dy, a.dy_stride, (const TS*)a.s, a.s_stride, (const TS*)a.ds, a.ds_stride, (TS*)a.dx, a.dx_stride,
        a.weight, parts, a.rows, (int)a.width, inv, a.eps);
    enqueue_sum_parts(st, parts, nb, {{a.dweight, nullptr, nullptr}, {a.width, 0, 0}});
  }
}

template <class TX, class TS>
void norm_shape(const dgen_hip_norm& a, bool backward, hipStream_t st) {
  int tpr, it;
  row_shape(a.width, tpr, it);
  switch (tpr * 16 + it) {
    case 16 * 16 + 1: return norm_launch<TX, TS, 16, 1>(a, backward, st);
    case 16 * 16 + 2: return norm_launch<TX, TS, 16, 2>(a, backward, st);
    case 64 * 16 + 1: return norm_launch<TX, TS, 64, 1>(a, backward, st);
    case 64 * 16 + 2: return norm_launch<TX, TS, 64, 2>(a, backward, st);
    case 64 * 16 + 4: return norm_launch<TX, TS, 64, 4>(a, backward, st);
    case 64 * 16 + 8: return norm_launch<TX, TS, 64, 8>(a, backward, st);
    case 256 * 16 + 4: return norm_launch<TX, TS, 256, 4>(a, backward, st);
    case 256 * 16 + 8: return norm_launch<TX, TS, 256, 8>(a, backward, st);
    case 1024 * 16 + 4: return norm_launch<TX, TS, 1024, 4>(a, backward, st);
    default: return norm_launch<TX, TS, 1024, 8>(a, backward, st);
  }
}

}  // namespace

void enqueue_sum_parts(hipStream_t stream, const float* ws, int64_t parts, const SumOut& out) {
  const int64_t width = out.n[0] + out.n[1] + out.n[2];
  k_sum_parts<<<dim3((unsigned)((width + kSumCols - 1) / kSumCols)), kSumThreads, 0, stream>>>(ws, parts, out, width);
}

int64_t norm_workspace(const dgen_hip_norm& a, bool backward) {
  return backward ? align256(norm_blocks(a) * a.width * (int64_t)sizeof(float)) : 0;
}

int norm_run(const dgen_hip_norm& a, bool backward, hipStream_t st, bool dry) {
  const char* what = backward ? "rms_norm_backward" : "rms_norm";
  DGEN_REQUIRE(a.struct_size == sizeof(a), "%s: struct_size %u, expected %zu", what, a.struct_size, sizeof(a));
  DGEN_REQUIRE((a.x_type == DGEN_HIP_F32 || a.x_type == DGEN_HIP_BF16) &&
                   (a.s_type == DGEN_HIP_F32 || a.s_type == DGEN_HIP_BF16),
               "%s: types %d, %d", what, a.x_type, a.s_type);
  DGEN_REQUIRE(a.width >= 1 && a.width <= kMaxWidth, "%s: width %lld outside [1, %lld]", what, (long long)a.width,
               (long long)kMaxWidth);
  int tpr, it;
  row_shape(a.width, tpr, it);
  // (a launch takes fewer than 2^32 threads)
  DGEN_REQUIRE(a.rows >= 0 && a.rows < (int64_t(1) << 31) / tpr, "%s: rows %lld outside [0, %lld) at width %lld", what,
               (long long)a.rows, (long long)((int64_t(1) << 31) / tpr), (long long)a.width);
  DGEN_REQUIRE(a.eps >= 0.f && a.eps < INFINITY, "%s: eps %g", what, (double)a.eps);
  DGEN_REQUIRE(a.weight, "%s: null weight", what);
  auto stride_ok = [&](const void* p, int64_t s) { return !p || a.rows <= 1 || s >= a.width; };
  if (!backward) {
    DGEN_REQUIRE((a.x && a.y) || a.rows == 0, "%s: null x or y", what);
    DGEN_REQUIRE(!a.residual == !a.s, "%s: residual and s come together", what);
    DGEN_REQUIRE(a.residual || a.x_type == a.s_type, "%s: without a residual s_type is x_type", what);
    // inputs may repeat rows (stride 0); outputs may not
    DGEN_REQUIRE(a.x_stride >= 0 && a.residual_stride >= 0, "%s: negative stride", what);
    DGEN_REQUIRE(stride_ok(a.y, a.y_stride) && stride_ok(a.s, a.s_stride), "%s: output rows overlap", what);
  } else {
    DGEN_REQUIRE((a.dy && a.s && a.dx) || a.rows == 0, "%s: null dy, s or dx", what);
    DGEN_REQUIRE(a.dweight, "%s: null dweight", what);
    DGEN_REQUIRE(a.dy_stride >= 0 && a.s_stride >= 0 && a.ds_stride >= 0, "%s: negative stride", what);
    DGEN_REQUIRE(stride_ok(a.dx, a.dx_stride), "%s: output rows overlap", what);
    const int64_t need = norm_workspace(a, true);
    DGEN_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= (uint64_t)need),
                 "%s: workspace of %llu bytes, %lld needed", what, (unsigned long long)a.workspace_bytes,
                 (long long)need);
  }
  if (dry || (a.rows == 0 && !backward)) return 0;
  const bool xb = a.x_type == DGEN_HIP_BF16, sb = a.s_type == DGEN_HIP_BF16;
  if (backward && a.rows == 0) {
    enqueue_sum_parts(st, a.weight, 0, {{a.dweight, nullptr, nullptr}, {a.width, 0, 0}});  // no rows: zeros
  } else if (xb) {
    sb ? norm_shape<bf16, bf16>(a, backward, st) : norm_shape<bf16, float>(a, backward, st);
  } else {
    sb ? norm_shape<float, bf16>(a, backward, st) : norm_shape<float, float>(a, backward, st);
  }
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
