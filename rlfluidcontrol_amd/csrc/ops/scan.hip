// scan.hip -- selective state space scan (afc_scan, afc_scan_grad, afc_scan_step)
//
//   delta = softplus(dt + bias)      h[l] = exp(delta A) h[l-1] + delta x B      y = (<C, h> + D x) silu(z)
//   backwards, with dy = dout silu(z):
//   g[l] = dy C + exp(delta A)[l+1] g[l+1]     du = <g, B>     t = g exp(delta A) h[l-1]
//   dx = du delta + D dy     ddelta = du x + <t, A>     dA = sum t delta     dB = sum_w g delta x     dC = sum_w dy h
#include <stdexcept>

#include "ops_common.h"

namespace afc_ops {

// A channel's states lie side by side in NP lanes (a power of two, lanes behind `state` hold zeros), 64 / NP channels in a wave.
template <int NP>
__device__ inline float sum_states(float v) {
  for (int m = 1; m < NP; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

template <int DT, int NP>
__global__ __launch_bounds__(64) void k_scan(afc_scan_args P) {
  typedef Elem<DT> E;
  const int n = threadIdx.x & (NP - 1);
  const int64_t tiles = (P.width + 64 / NP - 1) / (64 / NP);
  const int64_t b = blockIdx.x / tiles, w = (blockIdx.x % tiles) * (64 / NP) + threadIdx.x / NP;
  const bool on = w < P.width, mine = on && n < P.state;
  const int64_t g = on ? w / (P.width / P.groups) : 0;
  const int len = row_length(P.lengths, b, P.length);
  const float A = mine ? P.a[w * P.state + n] : 0.f, D = on && P.d ? P.d[w] : 0.f, bias = on && P.dt_bias ? P.dt_bias[w] : 0.f;
  float h = mine && P.initial_state ? P.initial_state[(b * P.width + w) * P.state + n] : 0.f;
  for (int64_t l = 0; l < P.length; ++l) {
    const int64_t at = b * P.x.stride_batch + l * P.x.stride_length + w;
    float y = 0.f;
    if (l < len) {
      const float x = on ? (float)((const E *)P.x.data)[at] : 0.f;
      const float v = on ? (float)((const E *)P.dt.data)[b * P.dt.stride_batch + l * P.dt.stride_length + w] + bias : 0.f;
      const float delta = P.softplus ? softplus(v) : v;
      const float B = mine ? (float)((const E *)P.b.data)[b * P.b.stride_batch + l * P.b.stride_length + g * P.b.stride_group + n] : 0.f;
      const float C = mine ? (float)((const E *)P.c.data)[b * P.c.stride_batch + l * P.c.stride_length + g * P.c.stride_group + n] : 0.f;
      h = mine ? __builtin_fmaf(exp_(delta * A), h, delta * x * B) : 0.f;
      y = sum_states<NP>(C * h) + D * x;
      if (P.z.data && on) y *= silu((float)((const E *)P.z.data)[b * P.z.stride_batch + l * P.z.stride_length + w]);
    }
    if (mine && P.checkpoints) P.checkpoints[((b * P.length + l) * P.width + w) * P.state + n] = h;
    if (on && n == 0) ((E *)P.y.data)[b * P.y.stride_batch + l * P.y.stride_length + w] = (Elem<DT>)y;
  }
  if (mine && P.final_state) P.final_state[(b * P.width + w) * P.state + n] = h;
}

// per row: sums over its positions (da, dd, ddt_bias rows), the adjoint states of every position for k_scan_grad_bc
template <int DT, int NP>
__global__ __launch_bounds__(64) void k_scan_grad(afc_scan_args P, float *gs, float *da, float *dd, float *dbias) {
  typedef Elem<DT> E;
  const int n = threadIdx.x & (NP - 1);
  const int64_t tiles = (P.width + 64 / NP - 1) / (64 / NP);
  const int64_t b = blockIdx.x / tiles, w = (blockIdx.x % tiles) * (64 / NP) + threadIdx.x / NP;
  const bool on = w < P.width, mine = on && n < P.state;
  const int64_t grp = on ? w / (P.width / P.groups) : 0;
  const int len = row_length(P.lengths, b, P.length);
  const float A = mine ? P.a[w * P.state + n] : 0.f, D = on && P.d ? P.d[w] : 0.f, bias = on && P.dt_bias ? P.dt_bias[w] : 0.f;
  const int64_t st = (b * P.width + w) * P.state + n;
  float g = mine && P.dfinal_state ? P.dfinal_state[st] : 0.f;  // the adjoint of the state that position l hands on
  float sa = 0.f, sd = 0.f, sb = 0.f;
  for (int64_t l = P.length - 1; l >= 0; --l) {
    float dx = 0.f, ddt = 0.f, dz = 0.f, gb = 0.f, dyc = 0.f;
    if (l < len) {
      const float x = on ? (float)((const E *)P.x.data)[b * P.x.stride_batch + l * P.x.stride_length + w] : 0.f;
      const float v = on ? (float)((const E *)P.dt.data)[b * P.dt.stride_batch + l * P.dt.stride_length + w] + bias : 0.f;
      const float delta = P.softplus ? softplus(v) : v;
      const float B = mine ? (float)((const E *)P.b.data)[b * P.b.stride_batch + l * P.b.stride_length + grp * P.b.stride_group + n] : 0.f;
      const float C = mine ? (float)((const E *)P.c.data)[b * P.c.stride_batch + l * P.c.stride_length + grp * P.c.stride_group + n] : 0.f;
      const float h = mine ? P.checkpoints[((b * P.length + l) * P.width + w) * P.state + n] : 0.f;
      float hp = 0.f;
      if (mine)
        hp = l > 0 ? P.checkpoints[((b * P.length + l - 1) * P.width + w) * P.state + n] : P.initial_state ? P.initial_state[st] : 0.f;
      float dy = on ? (float)((const E *)P.dy.data)[b * P.dy.stride_batch + l * P.dy.stride_length + w] : 0.f;
      if (P.z.data) {
        const float z = on ? (float)((const E *)P.z.data)[b * P.z.stride_batch + l * P.z.stride_length + w] : 0.f, s = sigmoid(z);
        dz = dy * (sum_states<NP>(C * h) + D * x) * silu_slope(z, s);
        dy *= z * s;
      }
      g = __builtin_fmaf(dy, C, g);
      const float a = exp_(delta * A), t = g * a * hp;
      const float du = sum_states<NP>(g * B);
      dx = __builtin_fmaf(du, delta, D * dy);
      ddt = __builtin_fmaf(du, x, sum_states<NP>(t * A));
      if (P.softplus) ddt *= sigmoid(v);
      sa = __builtin_fmaf(t, delta, sa);
      sd = __builtin_fmaf(dy, x, sd);
      sb += ddt;
      gb = mine ? g * (delta * x) : 0.f;
      dyc = mine ? dy * h : 0.f;
      g = mine ? g * a : 0.f;
    }
    if (mine) {
      float *o = gs + (((b * P.length + l) * P.width + w) * P.state + n) * 2;
      o[0] = gb;
      o[1] = dyc;
    }
    if (on && n == 0) {
      ((E *)P.dx.data)[b * P.dx.stride_batch + l * P.dx.stride_length + w] = (Elem<DT>)dx;
      ((E *)P.ddt.data)[b * P.ddt.stride_batch + l * P.ddt.stride_length + w] = (Elem<DT>)ddt;
      if (P.dz.data) ((E *)P.dz.data)[b * P.dz.stride_batch + l * P.dz.stride_length + w] = (Elem<DT>)dz;
    }
  }
  if (mine) {
    da[st] = sa;
    if (P.dinitial_state) P.dinitial_state[st] = g;
  }
  if (on && n == 0) {
    dd[b * P.width + w] = sd;
    dbias[b * P.width + w] = sb;
  }
}

template <int DT>
__global__ __launch_bounds__(256) void k_scan_grad_bc(afc_scan_args P, const float *gs) {
  typedef Elem<DT> E;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = P.groups * P.state;
  if (i >= P.batch * P.length * per) return;
  const int64_t row = i / per, g = i % per / P.state, n = i % P.state, b = row / P.length, l = row % P.length, m = P.width / P.groups;
  float sb = 0.f, sc = 0.f;
  for (int64_t w = g * m; w < (g + 1) * m; ++w) {
    const float *o = gs + ((row * P.width + w) * P.state + n) * 2;
    sb += o[0];
    sc += o[1];
  }
  ((E *)P.db.data)[b * P.db.stride_batch + l * P.db.stride_length + g * P.db.stride_group + n] = (Elem<DT>)sb;
  ((E *)P.dc.data)[b * P.dc.stride_batch + l * P.dc.stride_length + g * P.dc.stride_group + n] = (Elem<DT>)sc;
}

// out[i] = sum over rows of part[row][i]
__global__ __launch_bounds__(256) void k_sum_rows(const float *part, int64_t rows, int64_t cols, float *out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= cols) return;
  float a = 0.f;
  for (int64_t r = 0; r < rows; ++r) a += part[r * cols + i];
  out[i] = a;
}

template <int DT, int NP>
__global__ __launch_bounds__(64) void k_scan_step(afc_scan_args P) {
  typedef Elem<DT> E;
  const int n = threadIdx.x & (NP - 1);
  const int64_t tiles = (P.width + 64 / NP - 1) / (64 / NP);
  const int64_t b = blockIdx.x / tiles, w = (blockIdx.x % tiles) * (64 / NP) + threadIdx.x / NP;
  const bool on = w < P.width, mine = on && n < P.state;
  const int64_t g = on ? w / (P.width / P.groups) : 0, st = (b * P.width + w) * P.state + n;
  const float x = on ? (float)((const E *)P.x.data)[b * P.x.stride_batch + w] : 0.f;
  const float v = on ? (float)((const E *)P.dt.data)[b * P.dt.stride_batch + w] + (P.dt_bias ? P.dt_bias[w] : 0.f) : 0.f;
  const float delta = P.softplus ? softplus(v) : v;
  float h = 0.f, yc = 0.f;
  if (mine) {
    const float B = (float)((const E *)P.b.data)[b * P.b.stride_batch + g * P.b.stride_group + n];
    const float C = (float)((const E *)P.c.data)[b * P.c.stride_batch + g * P.c.stride_group + n];
    h = __builtin_fmaf(exp_(delta * P.a[w * P.state + n]), P.final_state[st], delta * x * B);
    P.final_state[st] = h;
    yc = C * h;
  }
  float y = sum_states<NP>(yc);
  if (!on || n) return;
  if (P.d) y = __builtin_fmaf(P.d[w], x, y);
  if (P.z.data) y *= silu((float)((const E *)P.z.data)[b * P.z.stride_batch + w]);
  ((E *)P.y.data)[b * P.y.stride_batch + w] = (Elem<DT>)y;
}

namespace {

void check(const afc_scan_args *p, bool grad, bool step) {
  want(p != nullptr, "null arguments");
  want(p->dtype >= AFC_F32 && p->dtype <= AFC_F16, "dtype must be AFC_F32, AFC_BF16 or AFC_F16");
  want(p->state >= 1 && p->state <= 64, "state must be 1..64");
  want(p->batch >= 0 && p->length >= 0 && p->width >= 1, "batch, length or width");
  want(p->length < (int64_t)1 << 31 && p->width < (int64_t)1 << 31 && p->batch < (int64_t)1 << 31, "an axis of 2^31 or more");
  want(p->groups >= 1 && p->width % p->groups == 0, "groups must divide width");
  want(p->a != nullptr, "a is missing");
  if (step) want(p->length == 1 && !p->lengths && p->final_state && p->final_state == p->initial_state, "a step takes length 1, no lengths, and its state as initial_state and final_state");
  if (p->batch == 0 || p->length == 0) return;
  check_seq(p->x, p->batch, p->length, 0, "x");
  check_seq(p->dt, p->batch, p->length, 0, "dt");
  check_seq(p->b, p->batch, p->length, p->groups, "b");
  check_seq(p->c, p->batch, p->length, p->groups, "c");
  if (p->z.data) check_seq(p->z, p->batch, p->length, 0, "z");
  if (!grad) check_seq(p->y, p->batch, p->length, 0, "y");
  if (grad) {
    check_seq(p->dy, p->batch, p->length, 0, "dy");
    check_seq(p->dx, p->batch, p->length, 0, "dx");
    check_seq(p->ddt, p->batch, p->length, 0, "ddt");
    check_seq(p->db, p->batch, p->length, p->groups, "db");
    check_seq(p->dc, p->batch, p->length, p->groups, "dc");
    if (p->dz.data) check_seq(p->dz, p->batch, p->length, 0, "dz");
    want(p->checkpoints != nullptr, "checkpoints are missing");
  }
}

int lanes(const afc_scan_args *p) {
  int n = 1;
  while (n < p->state) n *= 2;
  return n;
}
int64_t blocks(const afc_scan_args *p) {
  const int64_t n = p->batch * ceil_div(p->width, 64 / lanes(p));
  want(n < (int64_t)1 << 31, "too many blocks");
  return n;
}
uint64_t states(const afc_scan_args *p) { return (uint64_t)p->batch * p->width * p->state * 4; }
uint64_t adjoints(const afc_scan_args *p) { return up256(2 * states(p) * p->length); }

#define SCAN_STATE(DT, ...)                                                                                          \
  switch (lanes(p)) {                                                                                                \
    case 1: SCAN_GO(DT, 1, __VA_ARGS__); break;                                                                      \
    case 2: SCAN_GO(DT, 2, __VA_ARGS__); break;                                                                      \
    case 4: SCAN_GO(DT, 4, __VA_ARGS__); break;                                                                      \
    case 8: SCAN_GO(DT, 8, __VA_ARGS__); break;                                                                      \
    case 16: SCAN_GO(DT, 16, __VA_ARGS__); break;                                                                    \
    case 32: SCAN_GO(DT, 32, __VA_ARGS__); break;                                                                    \
    default: SCAN_GO(DT, 64, __VA_ARGS__); break;                                                                    \
  }
#define SCAN_TYPES(...)                                  \
  if (p->dtype == AFC_F32) {                             \
    SCAN_STATE(AFC_F32, __VA_ARGS__)                     \
  } else if (p->dtype == AFC_BF16) {                     \
    SCAN_STATE(AFC_BF16, __VA_ARGS__)                    \
  } else {                                               \
    SCAN_STATE(AFC_F16, __VA_ARGS__)                     \
  }

void scan(const afc_scan_args *p, hipStream_t st) {
  check(p, false, false);
  OnDevice on(p->device);
  if (p->batch == 0) return;
  const dim3 grid((unsigned)blocks(p));
#define SCAN_GO(DT, NP, ...) k_scan<DT, NP><<<grid, 64, 0, st>>>(*p)
  SCAN_TYPES(0)
#undef SCAN_GO
  launched("k_scan");
}

void scan_step(const afc_scan_args *p, hipStream_t st) {
  check(p, false, true);
  OnDevice on(p->device);
  if (p->batch == 0) return;
  const dim3 grid((unsigned)blocks(p));
#define SCAN_GO(DT, NP, ...) k_scan_step<DT, NP><<<grid, 64, 0, st>>>(*p)
  SCAN_TYPES(0)
#undef SCAN_GO
  launched("k_scan_step");
}

uint64_t grad_workspace(const afc_scan_args *p) { return adjoints(p) + up256(states(p)) + 2 * up256((uint64_t)p->batch * p->width * 4); }

void scan_grad(const afc_scan_args *p, hipStream_t st) {
  check(p, true, false);
  want(p->batch == 0 || (p->workspace && p->workspace_bytes >= grad_workspace(p) && (uintptr_t)p->workspace % 256 == 0),
       "workspace is missing, too small or not 256-byte aligned");
  OnDevice on(p->device);
  char *ws = (char *)p->workspace;
  float *gs = (float *)ws, *da = (float *)(ws + adjoints(p)), *dd = (float *)((char *)da + up256(states(p)));
  float *db = (float *)((char *)dd + up256((uint64_t)p->batch * p->width * 4));
  if (p->batch > 0) {
    const dim3 grid((unsigned)blocks(p));
#define SCAN_GO(DT, NP, ...) k_scan_grad<DT, NP><<<grid, 64, 0, st>>>(*p, gs, da, dd, db)
    SCAN_TYPES(0)
#undef SCAN_GO
    launched("k_scan_grad");
    const int64_t n = ceil_div(p->batch * p->length * p->groups * p->state, 256);
    want(n < (int64_t)1 << 31, "too many blocks");
    if (n) {
      const dim3 gb((unsigned)n);
      if (p->dtype == AFC_F32) k_scan_grad_bc<AFC_F32><<<gb, 256, 0, st>>>(*p, gs);
      if (p->dtype == AFC_BF16) k_scan_grad_bc<AFC_BF16><<<gb, 256, 0, st>>>(*p, gs);
      if (p->dtype == AFC_F16) k_scan_grad_bc<AFC_F16><<<gb, 256, 0, st>>>(*p, gs);
      launched("k_scan_grad_bc");
    }
  }
  auto sum = [&](const float *part, int64_t cols, float *out) {
    if (!out) return;
    k_sum_rows<<<dim3((unsigned)ceil_div(cols, 256)), 256, 0, st>>>(part, p->batch, cols, out);
    launched("k_sum_rows");
  };
  sum(da, p->width * p->state, p->da);
  sum(dd, p->width, p->dd);
  sum(db, p->width, p->ddt_bias);
}

}  // namespace
}  // namespace afc_ops

extern "C" {
int afc_scan(const afc_scan_args *args, void *hip_stream) {
  return afc_ops::entry("afc_scan", [&] { afc_ops::scan(args, (hipStream_t)hip_stream); });
}
int afc_scan_step(const afc_scan_args *args, void *hip_stream) {
  return afc_ops::entry("afc_scan_step", [&] { afc_ops::scan_step(args, (hipStream_t)hip_stream); });
}
int afc_scan_grad(const afc_scan_args *args, void *hip_stream) {
  return afc_ops::entry("afc_scan_grad", [&] { afc_ops::scan_grad(args, (hipStream_t)hip_stream); });
}
int afc_scan_workspace(const afc_scan_args *args, uint64_t *checkpoint_bytes, uint64_t *scan_bytes, uint64_t *grad_bytes) {
  return afc_ops::entry("afc_scan_workspace", [&] {
    afc_ops::want(args && checkpoint_bytes && scan_bytes && grad_bytes, "null argument");
    *checkpoint_bytes = afc_ops::up256(afc_ops::states(args) * args->length);
    *scan_bytes = 0;
    *grad_bytes = afc_ops::grad_workspace(args);
  });
}
}
