// One AdamW step over many tensors: m' = b1 m + (1 - b1) g, v' = b2 v +
// (1 - b2) g^2, p' = (1 - lr wd) p - lr m^ / (sqrt(v^) + eps), with the
// gradients optionally scaled down to a bound on their norm.
//
// Nothing but memory bounds it: 28 bytes a parameter (fp32 gradients), 2 more
// with the bf16 copy.  The tensors' addresses are the launch's arguments, so
// that one launch takes up to kTensors of any size and a captured step keeps
// them; a workgroup takes 4096 elements of one tensor, all its loads in flight
// before the first store.  The gradients' norm is a launch before: a sum of
// squares per workgroup, added in a fixed order, in 64 bits: the squares of
// gradients past 1e19 are no numbers in 32, and it is such gradients that the
// bound is for.  241 M parameters with bf16 gradients, bounded, and bf16 copies:
// 6.76 GB in 1.39 ms (4.9 TB/s); the squares take 136 us when profiled, their sum
// 12.  7.8 M parameters of 32 tensors: 233 MB in 51 us.
#include <cmath>
#include <vector>

#include "seq.h"

namespace dgen {

namespace {

// (as many tensors as a launch's 4096 bytes of arguments hold)
constexpr int kTensors = 52, kSquares = 200, kThreads = 256, kRuns = 4, kPer = kThreads * 4 * kRuns;

struct Tensor {
  const float *p, *m, *v;
  const void* g;
  float *po, *mo, *vo;
  bf16* copy;
  int64_t n;
};

struct StepP {
  Tensor t[kTensors];
  uint32_t first[kTensors + 1];  // a tensor's first workgroup
  int count;
  float b1, c1, b2, c2, decay, lr, rate, root, eps, ln1, ln2;
  const int64_t* step;
  const double* factor;  // of the gradients
};
static_assert(sizeof(StepP) <= 4096, "a launch's arguments");

struct SquaresP {
  const void* g[kSquares];
  int64_t n[kSquares];
  uint32_t first[kSquares + 1];
  int count;
  double* parts;
};
static_assert(sizeof(SquaresP) <= 4096, "a launch's arguments");

// The tensor that a workgroup works on.
__device__ __forceinline__ int tensor_of(const uint32_t* first, int count) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <class G>
__global__ __launch_bounds__(kThreads) void k_squares(SquaresP a) {
  const int k = tensor_of(a.first, a.count);
  const int64_t at = (int64_t)(blockIdx.x - a.first[k]) * kPer + threadIdx.x * 4;
  const G* g = (const G*)a.g[k];
  float x[kRuns][4];
  double sum = 0.0;
#pragma unroll
  for (int r = 0; r < kRuns; ++r) {
    const int64_t i = at + r * kThreads * 4, left = a.n[k] - i;
    load_four(g + i, left > 4 ? 4 : (int)left, x[r]);
  }
#pragma unroll
  for (int r = 0; r < kRuns; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = fma((double)x[r][e], (double)x[r][e], sum);
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k, 64);
  __shared__ double red[kThreads / 64];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.parts[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// The parts' sum (as many as there are 4096 elements), its root, and what the
// gradients are multiplied by.
__global__ __launch_bounds__(1024) void k_norm_of_squares(const double* __restrict__ parts, int64_t n, double bound,
                                                          float* __restrict__ norm, double* __restrict__ factor) {
  double s = 0.0;
  int64_t i = threadIdx.x;
  for (; i + 7 * 1024 < n; i += 8 * 1024) {  // (eight loads in flight)
    double x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = parts[i + k * 1024];
#pragma unroll
    for (int k = 0; k < 8; ++k) s += x[k];
  }
  for (; i < n; i += 1024) s += parts[i];
  __shared__ double red[1024];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int k = 512; k > 0; k >>= 1) {
    if ((int)threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double root = sqrt(red[0]), f = bound / (root + 1e-6);
    *norm = (float)root;
    *factor = f > 1.0 ? 1.0 : f;  // (a norm that is no number spoils all, as in the formula)
  }
}

// BOUND: the gradients are scaled, in 64 bits, as the factor may be below 2^-126
// (without a bound those multiplications took 56 us where these take 51).
template <class G, bool BOUND>
__global__ __launch_bounds__(kThreads) void k_adamw(StepP a) {
  const int k = tensor_of(a.first, a.count);
  const Tensor t = a.t[k];
  const int64_t at = (int64_t)(blockIdx.x - a.first[k]) * kPer + threadIdx.x * 4;
  float rate = a.rate, root = a.root;
  if (a.step) {
    // 1 - b^t = -(e^(t ln b) - 1)
    const float n = (float)*a.step;
    rate = a.lr / -expm1f(n * a.ln1);
    root = rsqrtf(-expm1f(n * a.ln2));
  }
  const double factor = BOUND ? *a.factor : 1.0;
  float p[kRuns][4], g[kRuns][4], m[kRuns][4], v[kRuns][4];
#pragma unroll
  for (int r = 0; r < kRuns; ++r) {
    const int64_t i = at + r * kThreads * 4, left = t.n - i;
    const int valid = left > 4 ? 4 : (int)left;
    load_four((const G*)t.g + i, valid, g[r]);
    load_four(t.m + i, valid, m[r]);
    load_four(t.v + i, valid, v[r]);
    load_four(t.p + i, valid, p[r]);
  }
#pragma unroll
  for (int r = 0; r < kRuns; ++r) {
    const int64_t i = at + r * kThreads * 4, left = t.n - i;
    const int valid = left > 4 ? 4 : (int)left;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = BOUND ? (float)((double)g[r][e] * factor) : g[r][e];
      m[r][e] = fmaf(a.c1, x, a.b1 * m[r][e]);
      v[r][e] = fmaf(a.c2 * x, x, a.b2 * v[r][e]);  // (x^2 alone may be past the largest number)
      p[r][e] = fmaf(-rate, m[r][e] / fmaf(sqrtf(v[r][e]), root, a.eps), a.decay * p[r][e]);
    }
    store_four(t.mo + i, valid, m[r]);
    store_four(t.vo + i, valid, v[r]);
    store_four(t.po + i, valid, p[r]);
    if (t.copy) store_four(t.copy + i, valid, p[r]);
  }
}

int64_t groups_of(int64_t n) { return (n + kPer - 1) / kPer; }

int64_t total_groups(const dgen_hip_adamw& a) {
  int64_t s = 0;
  for (int64_t i = 0; i < a.count; ++i) s += groups_of(a.tensors[i].n);
  return s;
}

// Memory that a step reads or writes: `what` counts a tensor's addresses in their
// order (0 .. 3 read, 4 .. 7 written).
struct Range {
  uintptr_t begin, end;
  int32_t tensor, what;
  bool out() const { return what >= 4; }
};

// Whether a result lies where something else does, but for a tensor's own
// parameter or moment that it replaces.
int check_apart(const dgen_hip_adamw& a, const char* name) try {
  thread_local std::vector<Range> all;
  all.clear();
  auto add = [&](const void* p, int64_t bytes, int64_t t, int what) {
    if (p && bytes > 0) all.push_back({(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, (int32_t)t, what});
  };
  const int64_t g = a.grad_type == DGEN_HIP_BF16 ? 2 : 4;
  for (int64_t i = 0; i < a.count; ++i) {
    const dgen_hip_adamw_tensor& t = a.tensors[i];
    // (what is replaced in place is there once, as a result)
    if (t.param != t.param_out) add(t.param, t.n * 4, i, 0);
    add(t.grad, t.n * g, i, 1);
    if (t.m != t.m_out) add(t.m, t.n * 4, i, 2);
    if (t.v != t.v_out) add(t.v, t.n * 4, i, 3);
    add(t.param_out, t.n * 4, i, 4), add(t.m_out, t.n * 4, i, 5), add(t.v_out, t.n * 4, i, 6), add(t.copy, t.n * 2, i, 7);
  }
  if (a.max_norm > 0) add(a.norm, 4, -1, 4);
  if (a.step_at) add(a.step_at, 8, -1, 0);
  std::sort(all.begin(), all.end(), [](const Range& x, const Range& y) { return x.begin < y.begin; });
  // against the range so far that reaches furthest, and the result that does
  const Range *far = nullptr, *out = nullptr;
  for (const Range& r : all) {
    for (const Range* q : {far, out})
      DGEN_REQUIRE(!q || q->end <= r.begin || !(q->out() || r.out()), "%s: a result of tensor %d shares memory with tensor %d", name,
                   r.out() ? r.tensor : q->tensor, r.out() ? q->tensor : r.tensor);
    if (!far || r.end > far->end) far = &r;
    if (r.out() && (!out || r.end > out->end)) out = &r;
  }
  return 0;
} catch (...) {
  return fail(DGEN_HIP_E_DEVICE, "%s: out of host memory", name);
}

}  // namespace

// The factor, then the squares' sums.
int64_t adamw_workspace(const dgen_hip_adamw& a) {
  return a.max_norm > 0 ? align256((1 + total_groups(a)) * (int64_t)sizeof(double)) : 0;
}

int adamw_run(const dgen_hip_adamw& a, hipStream_t st, bool dry) {
  const char* what = "adamw";
  if (dry) {
    DGEN_REQUIRE(a.struct_size == sizeof(a), "%s: struct_size %u, expected %zu", what, a.struct_size, sizeof(a));
    DGEN_REQUIRE(a.grad_type == DGEN_HIP_F32 || a.grad_type == DGEN_HIP_BF16, "%s: type %d", what, a.grad_type);
    DGEN_REQUIRE(a.count >= 0 && a.count <= 1 << 20, "%s: count %lld", what, (long long)a.count);
    DGEN_REQUIRE(a.tensors || a.count == 0, "%s: null tensors", what);
    auto in = [](double x, double lo, double hi) { return x >= lo && x < hi; };
    DGEN_REQUIRE(in(a.lr, 0, INFINITY), "%s: lr %g", what, a.lr);
    DGEN_REQUIRE(in(a.beta1, 0, 1) && in(a.beta2, 0, 1), "%s: betas %g, %g outside [0, 1)", what, a.beta1, a.beta2);
    DGEN_REQUIRE(in(a.eps, 0, INFINITY), "%s: eps %g", what, a.eps);
    DGEN_REQUIRE(in(a.weight_decay, 0, INFINITY), "%s: weight_decay %g", what, a.weight_decay);
    DGEN_REQUIRE(in(a.max_norm, 0, INFINITY), "%s: max_norm %g", what, a.max_norm);
    DGEN_REQUIRE(a.step >= 1 || a.step_at, "%s: step %lld, from 1", what, (long long)a.step);
    DGEN_REQUIRE(a.max_norm == 0 || a.norm, "%s: null norm", what);
    for (int64_t i = 0; i < a.count; ++i) {
      const dgen_hip_adamw_tensor& t = a.tensors[i];
      DGEN_REQUIRE(t.n >= 0 && t.n < int64_t(1) << 34, "%s: tensor %lld has %lld elements", what, (long long)i, (long long)t.n);
      DGEN_REQUIRE(t.n == 0 || (t.param && t.grad && t.m && t.v && t.param_out && t.m_out && t.v_out),
                   "%s: tensor %lld: null address", what, (long long)i);
    }
    DGEN_REQUIRE(total_groups(a) < int64_t(1) << 31, "%s: too many elements", what);
    // (the workspace's size does not go by the places)
    if (a.workspace_bytes != ~0ull)
      if (int rc = check_apart(a, what)) return rc;
    const int64_t need = adamw_workspace(a);
    DGEN_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= (uint64_t)need),
                 "%s: workspace of %llu bytes, %lld needed", what, (unsigned long long)a.workspace_bytes, (long long)need);
    return 0;
  }
  const bool half = a.grad_type == DGEN_HIP_BF16;
  // Runs of up to `most` tensors that have elements (and fewer workgroups
  // than a launch takes).
  auto runs = [&](int most, auto take, auto launch) {
    uint32_t at = 0;
    int k = 0;
    for (int64_t i = 0; i <= a.count; ++i) {
      const int64_t g = i < a.count ? groups_of(a.tensors[i].n) : 0;
      if (k && (i == a.count || k == most || at + g >= (1 << 22))) {
        launch(k, at);
        k = 0, at = 0;
      }
      if (g) take(k++, at, a.tensors[i]), at += (uint32_t)g;
    }
  };
  if (a.max_norm > 0) {
    double *const factor = (double*)a.workspace, *const parts = factor + 1;
    SquaresP q;
    q.parts = parts;
    runs(
        kSquares, [&](int k, uint32_t at, const dgen_hip_adamw_tensor& t) { q.g[k] = t.grad, q.n[k] = t.n, q.first[k] = at; },
        [&](int k, uint32_t groups) {
          q.count = k;
          half ? k_squares<bf16><<<groups, kThreads, 0, st>>>(q) : k_squares<float><<<groups, kThreads, 0, st>>>(q);
          q.parts += groups;
        });
    k_norm_of_squares<<<1, 1024, 0, st>>>(parts, q.parts - parts, a.max_norm, a.norm, factor);
  }
  StepP s;
  s.b1 = (float)a.beta1, s.c1 = (float)(1 - a.beta1), s.b2 = (float)a.beta2, s.c2 = (float)(1 - a.beta2);
  s.decay = (float)(1 - a.lr * a.weight_decay), s.lr = (float)a.lr, s.eps = (float)a.eps;
  s.ln1 = (float)std::log(a.beta1), s.ln2 = (float)std::log(a.beta2);
  s.step = a.step_at;
  s.rate = s.root = 0.f;
  if (!a.step_at) {
    s.rate = (float)(a.lr / (1 - std::pow(a.beta1, (double)a.step)));
    s.root = (float)(1 / std::sqrt(1 - std::pow(a.beta2, (double)a.step)));
  }
  s.factor = (const double*)a.workspace;
  runs(
      kTensors,
      [&](int k, uint32_t at, const dgen_hip_adamw_tensor& t) {
        s.t[k] = {t.param, t.m, t.v, t.grad, t.param_out, t.m_out, t.v_out, (bf16*)t.copy, t.n};
        s.first[k] = at;
      },
      [&](int k, uint32_t groups) {
        s.count = k;
        if (a.max_norm > 0)
          half ? k_adamw<bf16, true><<<groups, kThreads, 0, st>>>(s) : k_adamw<float, true><<<groups, kThreads, 0, st>>>(s);
        else
          half ? k_adamw<bf16, false><<<groups, kThreads, 0, st>>>(s) : k_adamw<float, false><<<groups, kThreads, 0, st>>>(s);
      });
  DGEN_LAUNCH_CHECK(what);
  return 0;
}

}  // namespace dgen
