// ops_common.h -- element types, accurate activations and the host-side plumbing of libafc_ops.so
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <exception>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "../../../include/afc_ops.h"

namespace afc_ops {

// ---- host ----
int fail(int code, const std::string &msg);

struct Refused {  // an argument that a check turned down
  std::string why;
};
inline void want(bool ok, const char *why) {
  if (!ok) throw Refused{why};
}
inline void hip(hipError_t e, const char *what) {
  if (e != hipSuccess) throw std::runtime_error(std::string(what) + ": " + hipGetErrorString(e));
}

// makes `device` current for the call and the thread's own device current again after it
struct OnDevice {
  int before = -1;
  explicit OnDevice(int device) {
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n < 1) {
      (void)hipGetLastError();
      throw std::domain_error("no HIP device available (this library has no CPU fallback)");
    }
    want(device >= 0 && device < n, "device ordinal out of range");
    hip(hipGetDevice(&before), "hipGetDevice");
    if (before == device)
      before = -1;
    else
      hip(hipSetDevice(device), "hipSetDevice");
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

inline void launched(const char *what) { hip(hipGetLastError(), what); }

// A launch has fewer than 2^32 threads along x, so more blocks than that go in slices: launch(base, blocks of the slice), the kernel's
// blocks counting from `base`.  (At sizes that real programs have there is one.)
template <class F>
void in_slices(int64_t blocks, int threads, const char *what, F &&launch) {
  const int64_t most = (((int64_t)1 << 32) - 1) / threads;
  for (int64_t base = 0; base < blocks; base += most) {
    launch(base, dim3((unsigned)(blocks - base < most ? blocks - base : most)));
    launched(what);
  }
}
constexpr int64_t kMostBlocks = (int64_t)1 << 31;  // of all slices of a launch

// no exception passes a C entry
template <class F>
int entry(const char *name, F &&f) {
  try {
    f();
    return AFC_OK;
  } catch (const Refused &r) {
    return fail(AFC_EINVAL, std::string(name) + ": " + r.why);
  } catch (const std::domain_error &e) {
    return fail(AFC_ENODEV, std::string(name) + ": " + e.what());
  } catch (const std::exception &e) {
    return fail(AFC_EHIP, std::string(name) + ": " + e.what());
  } catch (...) {
    return fail(AFC_EHIP, std::string(name) + ": unknown error");
  }
}

constexpr int64_t kMostAxis = (int64_t)1 << 30;  // indices along an axis, rounded up to a tile, fit 32 bits

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline uint64_t up256(uint64_t n) { return (n + 255) & ~(uint64_t)255; }

// Everything that is counted or laid out (blocks, partial sums, checkpoints: at most 512 bytes for an element of the sequence) stays
// inside 63 bits
inline void check_axes(int64_t batch, int64_t length, int64_t width) {
  want(batch >= 0 && length >= 0 && width >= 1, "batch, length or width");
  want(length < kMostAxis && width < kMostAxis && batch < kMostAxis, "an axis of 2^30 or more");
  want((__int128)batch * (length > 0 ? length : 1) * width < (__int128)1 << 48, "more than 2^48 elements");
}

// a sequence tensor whose last element's offset stays far inside 63 bits
inline void check_seq(const afc_seq &s, int64_t batch, int64_t length, int64_t groups, const char *why) {
  want(s.data != nullptr && s.stride_batch >= 0 && s.stride_length >= 0 && s.stride_group >= 0, why);
  int64_t p, q, r, t;
  want(!__builtin_mul_overflow(batch, s.stride_batch, &p) && !__builtin_mul_overflow(length, s.stride_length, &q) &&
           !__builtin_mul_overflow(groups, s.stride_group, &r) && !__builtin_add_overflow(p, q, &t) &&
           !__builtin_add_overflow(t, r, &t) && t < (int64_t)1 << 60,
       why);
}

// ---- device ----
template <int DT>
struct ElemT;
template <>
struct ElemT<AFC_F32> {
  typedef float type;
};
template <>
struct ElemT<AFC_BF16> {
  typedef __bf16 type;
};
template <>
struct ElemT<AFC_F16> {
  typedef _Float16 type;
};
template <int DT>
using Elem = typename ElemT<DT>::type;

__device__ inline float exp_(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896341f); }
// log2 e times a decay rate, finite from below: a rate of -inf forgets everything at any step size of 1e-36 and more (2^-340 is zero)
// and nothing at zero, which is that of a position behind a row's end
__device__ inline float rate2(float a) {
  const float r = a * 1.44269504088896341f;
  return r < -3.4e38f ? -3.4e38f : r;
}
__device__ inline float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + exp_(-v)); }
__device__ inline float silu(float v) { return v * sigmoid(v); }
// d/dv v sigmoid(v), with s = sigmoid(v)
__device__ inline float silu_slope(float v, float s) { return s * __builtin_fmaf(v, 1.f - s, 1.f); }

// log(1 + exp(v)) = max(v, 0) + log1p(e), e = exp(-|v|) in (0, 1].  Step sizes near 1e-3 come out of e near 1e-3, where
// log(1 + e) would keep only the digits of e that 1 + e keeps (relative error 6e-5): Kahan's log1p, log(w) e / (w - 1) with
// w = 1 + e as rounded, has the full 24 bits.  No threshold is needed: for large v the sum is v.
// `slope`: sigmoid(v), out of the same exponential.
__device__ inline float softplus(float v, float &slope) {
  const float e = exp_(-__builtin_fabsf(v));
  const float w = 1.f + e, dw = w - 1.f;
  const float l = __builtin_amdgcn_logf(w) * 0.693147180559945309f * (e * __builtin_amdgcn_rcpf(dw));
  slope = __builtin_amdgcn_rcpf(w) * (v < 0.f ? e : 1.f);
  return fmaxf(v, 0.f) + (dw == 0.f ? e : l);
}
__device__ inline float softplus(float v) {
  float slope;
  return softplus(v, slope);
}

// Sum of a column over many rows by a block of 1024: 64 columns, 16 interleaved runs of rows with four sums each in flight, added
// up in a fixed order.  The threads below 64 get it.  (Four runs: 68 us for 1107 rows of 288 columns, which make only five
// blocks.)
__device__ inline float column_sum(const float *from, int64_t rows, int64_t cols, int64_t col, float *red) {
  float a[4] = {};
  if (col < cols) {
    int64_t r = threadIdx.x >> 6;
    for (; r + 48 < rows; r += 64)
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k] += from[(r + 16 * k) * cols + col];
    for (; r < rows; r += 16) a[0] += from[r * cols + col];
  }
  red[threadIdx.x] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  float sum = 0.f;
  if (threadIdx.x < 64)
    for (int k = 0; k < 16; ++k) sum += red[threadIdx.x + 64 * k];
  return sum;
}

__device__ inline int row_length(const int32_t *lengths, int64_t b, int64_t length) {
  if (!lengths) return (int)length;
  const int n = lengths[b];
  return n < 0 ? 0 : n > (int)length ? (int)length : n;
}

}  // namespace afc_ops
