// clip.hip -- global 2-norm of many tensors and clipping by it (afc_clip); the library's error text
#include <algorithm>
#include <stdexcept>
#include <vector>

#include "ops_common.h"

namespace afc_ops {

static thread_local std::string g_err;
int fail(int code, const std::string &msg) {
  try {
    g_err = msg;
  } catch (...) {
  }
  return code;
}

// The tables of pointers travel in the kernel arguments (at most 4 KB): no copy that would have to outlive the call, and a
// captured launch carries its own.
constexpr int kTensors = 110;
constexpr int64_t kChunk = 32768;  // elements of a block

struct Batch {
  const void *in[kTensors];
  void *out[kTensors];
  int64_t numel[kTensors];
  int32_t first[kTensors + 1];  // the batch's first block of each tensor
  uint8_t in_dtype[kTensors], out_dtype[kTensors];
  int32_t count;
};

__device__ inline float load(const void *p, int dtype, int64_t i) {
  if (dtype == AFC_F32) return ((const float *)p)[i];
  if (dtype == AFC_BF16) return (float)((const __bf16 *)p)[i];
  return (float)((const _Float16 *)p)[i];
}
__device__ inline void store(void *p, int dtype, int64_t i, float v) {
  if (dtype == AFC_F32)
    ((float *)p)[i] = v;
  else if (dtype == AFC_BF16)
    ((__bf16 *)p)[i] = (__bf16)v;
  else
    ((_Float16 *)p)[i] = (_Float16)v;
}
__device__ inline int tensor_of(const Batch &T, int block) {
  int lo = 0, hi = T.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    (T.first[mid] <= block ? lo : hi) = mid;
  }
  return lo;
}

__device__ inline double block_sum(double a, double *red) {
  for (int m = 32; m; m >>= 1) a += __shfl_xor(a, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(256) void k_squares(Batch T, double *part) {
  __shared__ double red[4];
  const int t = tensor_of(T, blockIdx.x);
  const int64_t from = (int64_t)(blockIdx.x - T.first[t]) * kChunk, to = min(from + kChunk, T.numel[t]);
  double a = 0;
  for (int64_t i = from + threadIdx.x; i < to; i += 256) {
    const double v = load(T.in[t], T.in_dtype[t], i);
    a = __builtin_fma(v, v, a);
  }
  a = block_sum(a, red);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// coef[0] = what the gradients are multiplied with
__global__ __launch_bounds__(256) void k_norm(const double *part, int64_t n, float max_norm, float *norm, float *coef) {
  __shared__ double red[4];
  double a = 0;
  for (int64_t i = threadIdx.x; i < n; i += 256) a += part[i];
  a = sqrt(block_sum(a, red));
  if (threadIdx.x) return;
  *norm = (float)a;
  const float c = (float)((double)max_norm / (a + 1e-6));
  *coef = c > 1.f ? 1.f : c;  // (a NaN stays one)
}

__global__ __launch_bounds__(256) void k_scale(Batch T, const float *coef) {
  const int t = tensor_of(T, blockIdx.x);
  const int64_t from = (int64_t)(blockIdx.x - T.first[t]) * kChunk, to = min(from + kChunk, T.numel[t]);
  const float c = *coef;
  if (c == 1.f && T.in[t] == T.out[t]) return;
  for (int64_t i = from + threadIdx.x; i < to; i += 256) store(T.out[t], T.out_dtype[t], i, c * load(T.in[t], T.in_dtype[t], i));
}

namespace {

void check(const afc_clip_args *p) {
  want(p != nullptr, "null arguments");
  want(p->count >= 0, "count");
  want(p->count == 0 || (p->in && p->numel && p->in_dtype), "an array is missing");
  for (int i = 0; i < p->count; ++i) {
    want(p->numel[i] >= 0 && p->numel[i] < (int64_t)1 << 45, "numel");
    want(p->numel[i] == 0 || p->in[i], "a tensor is missing");
    want(p->in_dtype[i] >= AFC_F32 && p->in_dtype[i] <= AFC_F16, "dtype must be AFC_F32, AFC_BF16 or AFC_F16");
  }
}

int bytes_of(int dtype) { return dtype == AFC_F32 ? 4 : 2; }

// no element is written twice or read after it was written
void check_outputs(const afc_clip_args *p) {
  struct Range {
    uintptr_t from, to;
    bool out;
  };
  std::vector<Range> r;
  r.reserve(2 * (size_t)p->count);
  for (int i = 0; i < p->count; ++i) {
    want(p->out_dtype[i] >= AFC_F32 && p->out_dtype[i] <= AFC_F16, "dtype must be AFC_F32, AFC_BF16 or AFC_F16");
    if (p->numel[i] == 0) continue;
    want(p->out[i] != nullptr, "an output is missing");
    const uintptr_t a = (uintptr_t)p->in[i], o = (uintptr_t)p->out[i];
    if (a == o)
      want(p->in_dtype[i] == p->out_dtype[i], "an output in place has another type");
    else
      r.push_back({a, a + p->numel[i] * bytes_of(p->in_dtype[i]), false});
    r.push_back({o, o + p->numel[i] * bytes_of(p->out_dtype[i]), true});
  }
  std::sort(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.from < b.from; });
  uintptr_t end = 0, end_out = 0;  // of everything so far, and of the outputs
  for (const Range &q : r) {
    want(q.from >= (q.out ? end : end_out), "two tensors overlap");
    end = std::max(end, q.to);
    if (q.out) end_out = std::max(end_out, q.to);
  }
}

uint64_t workspace(const afc_clip_args *p) {
  uint64_t n = 0;
  for (int i = 0; i < p->count; ++i) n += (uint64_t)ceil_div(p->numel[i], kChunk);
  return 256 + up256(8 * n);
}

template <class F>
void batches(const afc_clip_args *p, F &&go) {
  int i = 0;
  while (i < p->count) {
    Batch t;
    t.count = 0;
    int64_t blocks = 0;
    for (; i < p->count && t.count < kTensors; ++i) {
      const int64_t n = ceil_div(p->numel[i], kChunk);
      if (n == 0) continue;
      want(n < (int64_t)1 << 30, "numel");
      if (blocks + n >= (int64_t)1 << 31) break;
      const int k = t.count++;
      t.in[k] = p->in[i];
      t.out[k] = p->out ? p->out[i] : nullptr;
      t.numel[k] = p->numel[i];
      t.in_dtype[k] = (uint8_t)p->in_dtype[i];
      t.out_dtype[k] = p->out ? (uint8_t)p->out_dtype[i] : 0;
      t.first[k] = (int32_t)blocks;
      blocks += n;
    }
    if (blocks) go(t, blocks);
  }
}

void clip(const afc_clip_args *p, hipStream_t st) {
  check(p);
  want(p->norm != nullptr, "norm is missing");
  if (p->out) {
    want(p->count == 0 || p->out_dtype, "an array is missing");
    want(p->max_norm >= 0.f, "max_norm must not be negative");
    check_outputs(p);
  }
  want(p->workspace && p->workspace_bytes >= workspace(p) && (uintptr_t)p->workspace % 256 == 0, "workspace is missing, too small or not 256-byte aligned");
  OnDevice on(p->device);
  float *coef = (float *)p->workspace;
  double *part = (double *)((char *)p->workspace + 256);
  int64_t n = 0;
  batches(p, [&](const Batch &t, int64_t blocks) {
    k_squares<<<dim3((unsigned)blocks), 256, 0, st>>>(t, part + n);
    launched("k_squares");
    n += blocks;
  });
  k_norm<<<1, 256, 0, st>>>(part, n, p->out ? p->max_norm : 0.f, p->norm, coef);
  launched("k_norm");
  if (!p->out) return;
  batches(p, [&](const Batch &t, int64_t blocks) {
    k_scale<<<dim3((unsigned)blocks), 256, 0, st>>>(t, coef);
    launched("k_scale");
  });
}

}  // namespace
}  // namespace afc_ops

extern "C" {
const char *afc_ops_last_error(void) { return afc_ops::g_err.c_str(); }
int afc_clip(const afc_clip_args *args, void *hip_stream) {
  return afc_ops::entry("afc_clip", [&] { afc_ops::clip(args, (hipStream_t)hip_stream); });
}
int afc_clip_workspace(const afc_clip_args *args, uint64_t *bytes) {
  return afc_ops::entry("afc_clip_workspace", [&] {
    afc_ops::check(args);
    afc_ops::want(bytes != nullptr, "null argument");
    *bytes = afc_ops::workspace(args);
  });
}
}
