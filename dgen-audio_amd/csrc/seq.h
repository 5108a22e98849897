// Shared by the sequence operators (k_norm, k_conv, k_scan, k_glu, k_delta,
// k_block) and the optimiser's step (k_adamw): element
// types, their loads and stores, and the sums that their backward passes end
// with.
#pragma once

#include <type_traits>

#include "internal.h"

namespace dgen {

// bfloat16 as raw bits; conversions round to nearest even.
struct bf16 {
  uint16_t v;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __uint_as_float((uint32_t)x.v << 16); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) {
  return bf16{__builtin_bit_cast(uint16_t, (__bf16)x)};
}

// Four consecutive elements.  The hardware takes vector accesses at any
// element alignment, so rows of odd widths and offset views use the same
// loads (alignment is declared as one element's).
template <class T>
struct __attribute__((packed, aligned(alignof(T)))) Four {
  T e[4];
};

template <class T>
__device__ __forceinline__ void load_four(const T* __restrict__ p, int valid, float (&o)[4]) {
  if (valid >= 4) {
    const Four<T> f = *reinterpret_cast<const Four<T>*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = to_f32(f.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = i < valid ? to_f32(p[i]) : 0.f;
  }
}

template <class T>
__device__ __forceinline__ void store_four(T* __restrict__ p, int valid, const float (&o)[4]) {
  if (valid >= 4) {
    Four<T> f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.e[i] = from_f32<T>(o[i]);
    *reinterpret_cast<Four<T>*>(p) = f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < valid) p[i] = from_f32<T>(o[i]);
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// Sums across the wave by exchange: each lane gets a's sum over the lanes that
// differ in bit 5 (or 4) if that bit of its own is 0, else b's.
__device__ __forceinline__ float swap_add32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap_add16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// sigmoid(x) = 1 / (1 + e^-x): e^-x overflows to infinity for x < -88, whose
// reciprocal is the right 0.
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + hw_exp(-x)); }
// silu(x) = x sigmoid(x) and its derivative p (1 + x (1 - p)).  x = -inf
// gives -inf * 0 = NaN, as the formula does.
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }
__device__ __forceinline__ float silu_grad(float x, float p) { return p * (1.f + x * (1.f - p)); }

// e^x for x <= 0 with the rounding of x log2(e) carried along (hw_exp alone
// is off by |x| 6e-8); 0 below -104.
__device__ __forceinline__ float exp_accurate(float x) {
  constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = 1.9259629911266175e-08f, kLn2 = 0.69314718055994531f;
  x = x < -104.f ? -104.f : x;
  const float t = x * kLog2e, e = __builtin_amdgcn_exp2f(t);
  return fmaf(e * kLn2, fmaf(x, kLog2eLow, fmaf(x, kLog2e, -t)), e);
}

// softplus(x) = max(x, 0) + ln(1 + e), e = e^-|x|, to fp32 accuracy for
// every e: the rounding of u = 1 + e is divided out again, ln(u) e / (u - 1).
// (internal.h's form, which matches the reference's expression, loses the
// relative accuracy of small results.)  slope: its derivative, the logistic
// function of x.
__device__ __forceinline__ float softplus_accurate(float x, float& slope) {
  const float e = exp_accurate(-fabsf(x)), u = 1.f + e, d = u - 1.f;
  const float l = d == 0.f ? e : hw_ln(u) * (e * __builtin_amdgcn_rcpf(d));
  const float p = __builtin_amdgcn_rcpf(u);
  slope = x >= 0.f ? p : e * p;
  return fmaxf(x, 0.f) + l;
}

// Sum over a row's TPR threads, in every one of them; `red`: LDS of a row of
// more than a wave (16 floats).  Lanes 32, 16, 8, 4, 2 and 1 apart: once those 8
// apart are added, 4 lanes on within the 16 is as good as 4 apart.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (TPR >= 64) v = swap_add32(v, v);
  if constexpr (TPR >= 32) v = swap_add16(v, v);
  v += dpp<0x128>(v);
  v += dpp<0x124>(v);
  v += dpp<0x4E>(v);
  v += dpp<0xB1>(v);
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

// out[j] = sum over p < parts of ws[p][j] for the columns of up to three
// outputs that lie side by side in a row of `ws`; fixed order.
struct SumOut {
  float* out[3];
  int64_t n[3];  // columns of each (0: none); a NULL output is skipped
};
constexpr int kSumThreads = 1024, kSumCols = 64;
// One workgroup's share: columns from 64 `block` on, 16 threads each over the
// rows.
__device__ __forceinline__ void sum_parts_block(const float* __restrict__ ws, int64_t parts, const SumOut& o,
                                                int64_t width, int64_t block, float (*red)[kSumCols + 1]) {
  const int col = threadIdx.x % kSumCols, sub = threadIdx.x / kSumCols;
  const int64_t j = block * kSumCols + col;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (j < width) {
    int64_t p = sub;
    for (; p + 48 < parts; p += 64)
#pragma unroll
      for (int q = 0; q < 4; ++q) a[q] += ws[(p + 16 * q) * width + j];
    for (; p < parts; p += 16) a[0] += ws[p * width + j];
  }
  red[sub][col] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  if (sub == 0 && j < width) {
    float t = 0.f;
#pragma unroll
    for (int q = 0; q < kSumThreads / kSumCols; ++q) t += red[q][col];
    int64_t at = j;
    for (int k = 0; k < 3; ++k) {
      if (at >= 0 && at < o.n[k] && o.out[k]) o.out[k][at] = t;
      at -= o.n[k];
    }
  }
}
void enqueue_sum_parts(hipStream_t stream, const float* ws, int64_t parts, const SumOut& out);

// Device to run on, restored at the end of the scope.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (hipGetDevice(&prev_) != hipSuccess) {
      prev_ = -1;
      return;
    }
    ok_ = prev_ == device || hipSetDevice(device) == hipSuccess;
    moved_ = ok_ && prev_ != device;
    if (!ok_) (void)hipGetLastError();  // reported here, not by the next launch check
  }
  ~DeviceScope() {
    if (moved_) (void)hipSetDevice(prev_);
  }
  bool ok() const { return ok_; }

 private:
  int prev_ = -1;
  bool ok_ = false, moved_ = false;
};

// A sequence tensor of [batch][T][channels] that is read: any strides that
// are not negative (0 repeats a frame or a sequence).
inline bool seq_readable(const dgen_hip_seq& v) { return v.stride_b >= 0 && v.stride_t >= 0; }
// One that is written: no two of its elements may lie at one address.
inline bool seq_writable(const dgen_hip_seq& v, int64_t batch, int64_t T, int64_t channels) {
  if (v.stride_b < 0 || v.stride_t < 0) return false;
  const bool frames = T > 1, seqs = batch > 1;
  if (frames && v.stride_t < channels) return false;
  if (seqs && v.stride_b < channels) return false;
  if (frames && seqs)
    return v.stride_b >= (T - 1) * v.stride_t + channels || v.stride_t >= (batch - 1) * v.stride_b + channels;
  return true;
}

constexpr int64_t align256(int64_t bytes) { return (bytes + 255) & ~int64_t(255); }

// The operators proper: descriptor checks and launches on a stream.  `what`
// names the caller in messages; with `dry` nothing is launched.
int64_t norm_workspace(const dgen_hip_norm&, bool backward);
int norm_run(const dgen_hip_norm&, bool backward, hipStream_t, bool dry);
int64_t conv_workspace(const dgen_hip_conv&, bool backward);
int conv_run(const dgen_hip_conv&, bool backward, hipStream_t, bool dry);
int64_t scan_workspace(const dgen_hip_scan&, bool backward);
int scan_run(const dgen_hip_scan&, bool backward, hipStream_t, bool dry);
int64_t mlp_workspace(const dgen_hip_mlp&, bool backward);
int mlp_run(const dgen_hip_mlp&, bool backward, hipStream_t, bool dry);
int64_t block_workspace(const dgen_hip_block_norms&, bool backward);
int block_run(const dgen_hip_block_norms&, bool backward, hipStream_t, bool dry);
int64_t delta_workspace(const dgen_hip_delta&, bool backward);
int delta_run(const dgen_hip_delta&, bool backward, hipStream_t, bool dry);
int64_t adamw_workspace(const dgen_hip_adamw&);
int adamw_run(const dgen_hip_adamw&, hipStream_t, bool dry);

}  // namespace dgen
