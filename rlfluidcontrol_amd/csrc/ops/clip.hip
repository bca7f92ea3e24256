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

// What a block works on
struct Part {
  const void *in;
  void *out;
  int64_t from, n;  // elements of the tensor
  int in_dtype, out_dtype;
};

// The tables of pointers travel in kernel arguments (at most 4 KB a launch): no copy that would have to outlive the call, and a
// captured launch carries its own.  Up to kTensors tensors go with the launches that use them; of more, launches of k_table lay
// down a table in the workspace first, so that one launch each runs over all of them (678 tensors of 40 x 40 and smaller:
// 134 us a call against 142 with a pair of launches for every 110, most of it the host's 0.1 us a tensor).  Up to kFew tensors take
// a small table: 4 KB of arguments cost the host half a microsecond a launch (12 tensors: 10.6 us a call against 11.4).
constexpr int kTensors = 120, kFew = 24;

template <int MOST>
struct Batch {
  const void *in[MOST];
  void *out[MOST];
  int64_t numel[MOST];
  int32_t first[MOST + 1];  // the first block of each tensor
  uint8_t in_dtype[MOST], out_dtype[MOST];
  int32_t count;
  int64_t chunk;  // elements of a block

  __device__ Part part(int block) const {
    int t = 0, hi = count;
    while (hi - t > 1) {
      const int mid = (t + hi) / 2;
      if (first[mid] <= block)
        t = mid;
      else
        hi = mid;
    }
    const int64_t from = (int64_t)(block - first[t]) * chunk;
    return {in[t], out[t], from, min(chunk, numel[t] - from), in_dtype[t], out_dtype[t]};
  }
};

struct Entry {
  const void *in;
  void *out;
  int64_t numel;
  int32_t first;
  uint8_t in_dtype, out_dtype;
};
struct Table {
  Entry *entries;
  int32_t *tensor_of;  // of every block
  int64_t chunk;

  __device__ Part part(int block) const {
    const Entry e = entries[tensor_of[block]];
    const int64_t from = (int64_t)(block - e.first) * chunk;
    return {e.in, e.out, from, min(chunk, e.numel - from), e.in_dtype, e.out_dtype};
  }
};

// one block for each tensor of a batch
__global__ __launch_bounds__(64) void k_table(Batch<kTensors> B, Table T, int base, int first) {
  const int t = blockIdx.x;
  if (threadIdx.x == 0) T.entries[base + t] = {B.in[t], B.out[t], B.numel[t], first + B.first[t], B.in_dtype[t], B.out_dtype[t]};
  for (int i = B.first[t] + threadIdx.x; i < B.first[t + 1]; i += 64) T.tensor_of[first + i] = base + t;
}

// V elements at once (16 bytes of the wider type) from any place: the memory pipeline takes accesses that start inside 16 bytes (a
// tensor may be a slice of a flat buffer), and the compiler is told no more than the element's own alignment.
template <int DT, int V>
struct VecT {
  typedef Elem<DT> type __attribute__((ext_vector_type(V), aligned(sizeof(Elem<DT>))));
};
template <int DT, int V>
using Vec = typename VecT<DT, V>::type;

__device__ inline double block_sum(double a, double *red) {
  for (int m = 32; m; m >>= 1) a += __shfl_xor(a, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = 0;
  for (unsigned i = 0; i < blockDim.x / 64; ++i) a += red[i];
  return a;
}

template <int DT>
__device__ double squares(const Elem<DT> *p, int64_t n) {
  constexpr int V = 16 / sizeof(Elem<DT>);
  double a[4] = {};
  const int64_t body = n / V;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < body; i += 256) {
    const Vec<DT, V> v = *reinterpret_cast<const Vec<DT, V> *>(p + i * V);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const double d = (double)(float)v[k];
      a[k & 3] = __builtin_fma(d, d, a[k & 3]);
    }
  }
  for (int64_t i = body * V + threadIdx.x; i < n; i += 256) {
    const double d = (double)(float)p[i];
    a[0] = __builtin_fma(d, d, a[0]);
  }
  return (a[0] + a[1]) + (a[2] + a[3]);
}

// One partial sum for each block.  Double costs nothing beside the loads (a conversion and a multiply-add for each element):
// 146 us for 641 MB of bf16, 4.4 TB/s (four loads in flight a thread instead of eight: 154 us).
template <class Tensors>
__global__ __launch_bounds__(256) void k_squares(Tensors T, double *part) {
  __shared__ double red[4];
  const Part p = T.part(blockIdx.x);
  double a;
  if (p.in_dtype == AFC_F32)
    a = squares<AFC_F32>((const float *)p.in + p.from, p.n);
  else if (p.in_dtype == AFC_BF16)
    a = squares<AFC_BF16>((const __bf16 *)p.in + p.from, p.n);
  else
    a = squares<AFC_F16>((const _Float16 *)p.in + p.from, p.n);
  a = block_sum(a, red);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// the norm from the partial sums, in their order, and what the gradients are multiplied with
__device__ inline double norm_of(const double *part, int64_t n, double *red) {
  double a = 0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) a += part[i];
  return sqrt(block_sum(a, red));
}
__device__ inline float factor(double norm, float max_norm) {
  const float c = (float)((double)max_norm / (norm + 1e-6));
  return c > 1.f ? 1.f : c;  // (a NaN stays one)
}

__global__ __launch_bounds__(1024) void k_norm(const double *part, int64_t n, float max_norm, float *norm, float *coef) {
  __shared__ double red[16];
  const double a = norm_of(part, n, red);
  if (threadIdx.x) return;
  *norm = (float)a;
  *coef = factor(a, max_norm);
}

template <int DI, int DO>
__device__ void scale(const Elem<DI> *p, Elem<DO> *o, int64_t n, float c) {
  constexpr int V = DI == AFC_F32 || DO == AFC_F32 ? 4 : 8;
  const int64_t body = n / V;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < body; i += 256) {
    const Vec<DI, V> v = *reinterpret_cast<const Vec<DI, V> *>(p + i * V);
    Vec<DO, V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r[k] = (Elem<DO>)(c * (float)v[k]);
    *reinterpret_cast<Vec<DO, V> *>(o + i * V) = r;
  }
  for (int64_t i = body * V + threadIdx.x; i < n; i += 256) o[i] = (Elem<DO>)(c * (float)p[i]);
}
template <int DI>
__device__ void scale_to(const void *in, void *out, int dt, int64_t from, int64_t n, float c) {
  const Elem<DI> *p = (const Elem<DI> *)in + from;
  if (dt == AFC_F32)
    scale<DI, AFC_F32>(p, (float *)out + from, n, c);
  else if (dt == AFC_BF16)
    scale<DI, AFC_BF16>(p, (__bf16 *)out + from, n, c);
  else
    scale<DI, AFC_F16>(p, (_Float16 *)out + from, n, c);
}

// Reads once more and writes: 405 us for 641 MB of bf16 into float, 4.7 TB/s, where rows of odd widths start inside 16 bytes.
// Blocks go backwards over the tensors: what k_squares has read last is still in the last-level cache.  FEW: the partial sums
// are few enough for every block to add them up by itself, which saves k_norm's launch.
template <class Tensors, bool FEW>
__global__ __launch_bounds__(256) void k_scale(Tensors T, const float *coef, const double *part, int64_t n_part, float max_norm, float *norm) {
  __shared__ double red[4];
  const int block = gridDim.x - 1 - blockIdx.x;
  float c;
  if (FEW) {
    const double a = norm_of(part, n_part, red);
    c = factor(a, max_norm);
    if (block == 0 && threadIdx.x == 0) *norm = (float)a;
  } else {
    c = *coef;
  }
  const Part p = T.part(block);
  if (c == 1.f && p.in == p.out) return;
  if (p.in_dtype == AFC_F32)
    scale_to<AFC_F32>(p.in, p.out, p.out_dtype, p.from, p.n, c);
  else if (p.in_dtype == AFC_BF16)
    scale_to<AFC_BF16>(p.in, p.out, p.out_dtype, p.from, p.n, c);
  else
    scale_to<AFC_F16>(p.in, p.out, p.out_dtype, p.from, p.n, c);
}

namespace {

void check(const afc_clip_args *p) {
  want(p != nullptr, "null arguments");
  want(p->count >= 0 && p->count < 1 << 23, "count");  // (with the 4096 blocks that share large ones, 2^24 blocks of 256 in a launch)
  want(p->count == 0 || (p->in && p->numel && p->in_dtype), "an array is missing");
  int64_t all = 0;
  for (int i = 0; i < p->count; ++i) {
    want(p->numel[i] >= 0 && p->numel[i] < (int64_t)1 << 45, "numel");
    want((all += p->numel[i]) < (int64_t)1 << 48, "more than 2^48 elements");
    want(p->numel[i] == 0 || p->in[i], "a tensor is missing");
    want(p->in_dtype[i] >= AFC_F32 && p->in_dtype[i] <= AFC_F16, "dtype must be AFC_F32, AFC_BF16 or AFC_F16");
  }
}

int bytes_of(int dtype) { return dtype == AFC_F32 ? 4 : 2; }

// no element is written twice or read after it was written
void check_outputs(const afc_clip_args *p) {
  struct Range {
    uintptr_t from, to;
  };
  std::vector<Range> ins, outs;  // (what is scaled in place counts as an output)
  ins.reserve((size_t)p->count), outs.reserve((size_t)p->count);
  for (int i = 0; i < p->count; ++i) {
    want(p->out_dtype[i] >= AFC_F32 && p->out_dtype[i] <= AFC_F16, "dtype must be AFC_F32, AFC_BF16 or AFC_F16");
    if (p->numel[i] == 0) continue;
    want(p->out[i] != nullptr, "an output is missing");
    const uintptr_t a = (uintptr_t)p->in[i], o = (uintptr_t)p->out[i];
    if (a == o)
      want(p->in_dtype[i] == p->out_dtype[i], "an output in place has another type");
    else
      ins.push_back({a, a + p->numel[i] * bytes_of(p->in_dtype[i])});
    outs.push_back({o, o + p->numel[i] * bytes_of(p->out_dtype[i])});
  }
  const auto before = [](const Range &a, const Range &b) { return a.from < b.from; };
  for (std::vector<Range> *r : {&ins, &outs})  // (slices of one buffer come in order)
    if (!std::is_sorted(r->begin(), r->end(), before)) std::sort(r->begin(), r->end(), before);
  uintptr_t end = 0, end_in = 0;  // of the outputs and of the inputs so far
  auto in = ins.begin();
  for (const Range &o : outs) {
    for (; in != ins.end() && in->from < o.from; ++in) {
      want(in->from >= end, "two tensors overlap");
      end_in = std::max(end_in, in->to);
    }
    want(o.from >= end && o.from >= end_in, "two tensors overlap");
    end = o.to;
  }
  want(in == ins.end() || in->from >= end, "two tensors overlap");
}

// Elements of a block: some 4096 blocks for all tensors together, so that the partial sums stay few, and 4096 elements at least
int64_t chunk_of(const afc_clip_args *p) {
  int64_t all = 0;
  for (int i = 0; i < p->count; ++i) all += p->numel[i];
  return std::max<int64_t>(4096, ceil_div(ceil_div(all, 4096), 2048) * 2048);
}
int64_t partials(const afc_clip_args *p) {
  const int64_t chunk = chunk_of(p);
  int64_t n = 0;
  for (int i = 0; i < p->count; ++i) n += ceil_div(p->numel[i], chunk);
  return n;
}
// coef, the partial sums, and where there are many tensors the table and the blocks' tensors
struct Layout {
  uint64_t part, entries, tensor_of, all;
};
Layout layout(const afc_clip_args *p) {
  Layout o;
  const uint64_t n = (uint64_t)partials(p), tensors = p->count > kTensors ? (uint64_t)p->count : 0;
  o.part = 256;
  o.entries = o.part + up256(8 * n);
  o.tensor_of = o.entries + up256(sizeof(Entry) * tensors);
  o.all = o.tensor_of + up256(tensors ? 4 * n : 0);
  return o;
}

template <int MOST>
std::vector<Batch<MOST>> batches(const afc_clip_args *p) {
  std::vector<Batch<MOST>> all;
  const int64_t chunk = chunk_of(p);
  int64_t blocks = 0;
  for (int i = 0; i < p->count; ++i) {
    if (p->numel[i] == 0) continue;
    if (all.empty() || all.back().count == MOST) {
      all.emplace_back();
      all.back().count = 0;
      all.back().chunk = chunk;
      blocks = 0;
    }
    Batch<MOST> &t = all.back();
    const int k = t.count++;
    t.in[k] = p->in[i];
    t.out[k] = p->out ? p->out[i] : nullptr;
    t.numel[k] = p->numel[i];
    t.in_dtype[k] = (uint8_t)p->in_dtype[i];
    t.out_dtype[k] = p->out ? (uint8_t)p->out_dtype[i] : 0;
    t.first[k] = (int32_t)blocks;
    blocks += ceil_div(p->numel[i], chunk);
    t.first[k + 1] = (int32_t)blocks;  // (a tensor has at most 4096 blocks, a batch 120 tensors)
  }
  return all;
}

template <class Tensors>
void passes(const afc_clip_args *p, const Tensors &t, int blocks, char *ws, const Layout &o, hipStream_t st) {
  float *coef = (float *)ws;
  double *part = (double *)(ws + o.part);
  const dim3 grid((unsigned)blocks);
  k_squares<<<grid, 256, 0, st>>>(t, part);
  launched("k_squares");
  // Adding up 1024 partial sums in every block costs less than the launch of k_norm: a call with 12 tensors takes 3.5 us less
  const bool few = p->out && blocks <= 1024;
  if (!few) {
    k_norm<<<1, 1024, 0, st>>>(part, blocks, p->out ? p->max_norm : 0.f, p->norm, coef);
    launched("k_norm");
  }
  if (!p->out) return;
  if (few)
    k_scale<Tensors, true><<<grid, 256, 0, st>>>(t, coef, part, blocks, p->max_norm, p->norm);
  else
    k_scale<Tensors, false><<<grid, 256, 0, st>>>(t, coef, part, blocks, p->max_norm, p->norm);
  launched("k_scale");
}

void clip(const afc_clip_args *p, hipStream_t st) {
  check(p);
  want(p->norm != nullptr, "norm is missing");
  if (p->out) {
    want(p->count == 0 || p->out_dtype, "an array is missing");
    want(p->max_norm >= 0.f, "max_norm must not be negative");
    check_outputs(p);
  }
  const Layout o = layout(p);
  want(p->workspace && p->workspace_bytes >= o.all && (uintptr_t)p->workspace % 256 == 0, "workspace is missing, too small or not 256-byte aligned");
  OnDevice on(p->device);
  char *ws = (char *)p->workspace;
  if (p->count > 0 && p->count <= kFew) {
    const std::vector<Batch<kFew>> few = batches<kFew>(p);
    if (!few.empty()) return passes(p, few[0], few[0].first[few[0].count], ws, o, st);
  }
  const std::vector<Batch<kTensors>> all = batches<kTensors>(p);
  if (all.size() > 1) {
    const Table table = {(Entry *)(ws + o.entries), (int32_t *)(ws + o.tensor_of), all[0].chunk};
    int base = 0, first = 0;
    for (const Batch<kTensors> &b : all) {
      k_table<<<dim3((unsigned)b.count), 64, 0, st>>>(b, table, base, first);
      launched("k_table");
      base += b.count, first += b.first[b.count];
    }
    passes(p, table, first, ws, o, st);
  } else if (!all.empty()) {
    passes(p, all[0], all[0].first[all[0].count], ws, o, st);
  } else {
    k_norm<<<1, 1024, 0, st>>>((const double *)(ws + o.part), 0, 0.f, p->norm, (float *)ws);
    launched("k_norm");
  }
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
    *bytes = afc_ops::layout(args).all;
  });
}
}
