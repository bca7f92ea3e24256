// conv.hip -- short causal convolution along the sequence (afc_conv, afc_conv_grad, afc_conv_step)
#include <stdexcept>
#include <type_traits>

#include "ops_common.h"

namespace afc_ops {

// V neighbouring elements at any address that suits one: the memory pipeline takes accesses that start anywhere, so rows of odd
// widths and slices need no other path
template <int DT, int V>
using Vec = Elem<DT> __attribute__((ext_vector_type(V), aligned(sizeof(Elem<DT>))));

template <int DT, int V>
__device__ inline void load(float (&f)[V], const Elem<DT> *p) {
  if constexpr (V == 1) {
    f[0] = (float)*p;
  } else {
    const Vec<DT, V> v = *reinterpret_cast<const Vec<DT, V> *>(p);
    for (int i = 0; i < V; ++i) f[i] = (float)v[i];
  }
}
template <int DT, int V>
__device__ inline void store(Elem<DT> *p, const float (&f)[V]) {
  if constexpr (V == 1) {
    *p = (Elem<DT>)f[0];
  } else {
    Vec<DT, V> v;
    for (int i = 0; i < V; ++i) v[i] = (Elem<DT>)f[i];
    *reinterpret_cast<Vec<DT, V> *>(p) = v;
  }
}

// V neighbouring elements as they were loaded (converted where they are used, so that loads stay in flight)
template <int DT, int V>
struct Raw {
  Vec<DT, V> v;
  __device__ inline void load(const Elem<DT> *p, bool on) {
    v = (Vec<DT, V>)(Elem<DT>)0.f;
    if (on) v = *reinterpret_cast<const Vec<DT, V> *>(p);
  }
  __device__ inline void load_all(const Elem<DT> *p) { v = *reinterpret_cast<const Vec<DT, V> *>(p); }
  __device__ inline float operator[](int i) const { return (float)v[i]; }
};

struct Tiling {
  int log_cx;          // lanes side by side along the channels (the others: positions)
  int run;             // positions of a thread
  int64_t tiles_c, tiles_l;
  int64_t base;        // the slice's first block
};

// A thread takes T.run positions of V channels (16 bytes of a row): the filter and the last K - 1 inputs stay in registers, and
// the next U positions are in flight while U are computed.  It reads and writes each element once (and K - 1 in front of each
// run, mostly from cache): memory bounds it.  3 x 8191 x 4096 bf16: 81 us, 5.0 TB/s (a copy: 5.1; runs of 8 positions loaded at
// once and filters read for each, 124 us; 8 positions in flight, 90 us).
template <int DT, int V, int K, bool SILU>
__global__ __launch_bounds__(256) void k_conv(afc_conv_args P, Tiling T) {
  typedef Elem<DT> E;
  constexpr int U = 4;
  int64_t blk = T.base + blockIdx.x;
  const int64_t ct = blk % T.tiles_c;
  blk /= T.tiles_c;
  const int64_t lt = blk % T.tiles_l, b = blk / T.tiles_l;
  const int cx = 1 << T.log_cx;
  int64_t c = (ct * cx + (threadIdx.x & (cx - 1))) * V;
  if (c >= P.width) return;
  c = min(c, P.width - V);  // (the last vector ends with the row: what two lanes share both write, the same)
  const int64_t l0 = (lt * (256 >> T.log_cx) + (threadIdx.x >> T.log_cx)) * T.run;
  const int len = row_length(P.lengths, b, P.length);
  const E *x = (const E *)P.x.data + b * P.x.stride_batch + c;
  const E *s0 = P.initial_state ? (const E *)P.initial_state + b * (K - 1) * P.width + c : nullptr;
  if (l0 == 0 && P.final_state) {
    for (int j = 0; j < K - 1; ++j) {
      const int64_t p = (int64_t)len - (K - 1) + j;
      float v[V] = {};
      if (p >= 0)
        load<DT, V>(v, x + p * P.x.stride_length);
      else if (s0)
        load<DT, V>(v, s0 + (p + K - 1) * P.width);
      store<DT, V>((E *)P.final_state + (b * (K - 1) + j) * P.width + c, v);
    }
  }
  if (l0 >= P.length) return;
  const int64_t end = min(l0 + T.run, P.length);
  float w[K][V], bias[V] = {}, win[K - 1 + U][V];
  for (int i = 0; i < V; ++i) {
    for (int k = 0; k < K; ++k) w[k][i] = P.weight[(c + i) * K + k];
    if (P.bias) bias[i] = P.bias[c + i];
  }
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const int64_t p = l0 + j - (K - 1);
    for (int i = 0; i < V; ++i) win[j][i] = 0.f;
    if (p < 0) {
      if (s0) load<DT, V>(win[j], s0 + (p + K - 1) * P.width);
    } else if (p < len) {
      load<DT, V>(win[j], x + p * P.x.stride_length);
    }
  }
  E *y = (E *)P.y.data + b * P.y.stride_batch + l0 * P.y.stride_length + c;
  x += l0 * P.x.stride_length;
  Raw<DT, V> ahead[U];
#pragma unroll
  for (int j = 0; j < U; ++j) ahead[j].load(x + j * P.x.stride_length, l0 + j < len && l0 + j < end);
  for (int64_t l = l0; l < end; l += U) {
    x += U * P.x.stride_length;
    Raw<DT, V> now[U];
#pragma unroll
    for (int j = 0; j < U; ++j) now[j] = ahead[j];
#pragma unroll
    for (int j = 0; j < U; ++j) ahead[j].load(x + j * P.x.stride_length, l + U + j < len && l + U + j < end);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        win[K - 1 + j][i] = now[j][i];
        float a = bias[i];
        for (int k = 0; k < K; ++k) a = __builtin_fmaf(w[k][i], win[j + k][i], a);
        v[i] = l + j < len ? (SILU ? silu(a) : a) : 0.f;
      }
      if (l + j < end) store<DT, V>(y, v);
      y += P.y.stride_length;
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
      for (int i = 0; i < V; ++i) win[j][i] = win[j + U][i];
  }
}

template <int DT, int V, int K, bool SILU>
__global__ __launch_bounds__(256) void k_conv_step(afc_conv_args P, int64_t base) {
  typedef Elem<DT> E;
  const int64_t per = P.width / V, t = (base + blockIdx.x) * 256 + threadIdx.x;
  if (t >= P.batch * per) return;
  const int64_t b = t / per, c = (t - b * per) * V;
  E *st = (E *)P.final_state + b * (K - 1) * P.width + c;
  float win[K][V];
#pragma unroll
  for (int j = 0; j < K - 1; ++j) load<DT, V>(win[j], st + j * P.width);
  load<DT, V>(win[K - 1], (const E *)P.x.data + b * P.x.stride_batch + c);
  float v[V];
  for (int i = 0; i < V; ++i) {
    float a = P.bias ? P.bias[c + i] : 0.f;
    for (int k = 0; k < K; ++k) a = __builtin_fmaf(P.weight[(c + i) * K + k], win[k][i], a);
    v[i] = SILU ? silu(a) : a;
  }
#pragma unroll
  for (int j = 0; j < K - 1; ++j) store<DT, V>(st + j * P.width, win[j + 1]);
  store<DT, V>((E *)P.y.data + b * P.y.stride_batch + c, v);
}

// A thread takes T.run positions [s, e) of V channels.  It walks over the positions q = s .. e + K - 2 whose outputs its dx
// depend on, with windows of the last K inputs and of the last K dp = dy f'(pre) in registers; dx[q - K + 1] is complete
// when dp[q] is known.  dweight and dbias: sums of the thread, then of the block, one partial row for each block, so that no
// order of additions depends on timing.  Reads x and dy and writes dx once: 148 us for 3 x 8191 x 4096 bf16, 4.1 TB/s (the
// 21 instructions an element would take some 65 us; without the loads ahead 208 us, with one or four positions ahead 160 and 152,
// half or twice the run or the four waves side by side 148 to 160).  Positions whose neighbours all lie inside the run and the
// row go without conditions: 40 instructions an element fall to 21, the time by 2 us of 150 where memory bounds it.
template <int DT, int V, int K, bool SILU>
__global__ __launch_bounds__(256) void k_conv_grad(afc_conv_args P, Tiling T, float *part) {
  typedef Elem<DT> E;
  __shared__ float red[256 * V];
  int64_t blk = T.base + blockIdx.x;
  const int64_t ct = blk % T.tiles_c;
  blk /= T.tiles_c;
  const int64_t lt = blk % T.tiles_l, b = blk / T.tiles_l;
  const int cx = 1 << T.log_cx, ty = 256 >> T.log_cx;
  const int lane_c = threadIdx.x & (cx - 1), lane_l = threadIdx.x >> T.log_cx;
  int64_t c = (ct * cx + lane_c) * V;
  const bool inside = c < P.width;
  c = inside ? min(c, P.width - V) : c;  // (the last vector ends with the row: what two lanes share both write, the same)
  const int64_t s64 = (lt * ty + lane_l) * (int64_t)T.run;
  const int len = row_length(P.lengths, b, P.length);
  float dw[K + 1][V];
  for (int k = 0; k <= K; ++k)
    for (int i = 0; i < V; ++i) dw[k][i] = 0.f;
  if (inside && (s64 < P.length || s64 == 0)) {
    const int s = (int)s64, e = (int)min(s64 + T.run, P.length);
    const E *x = (const E *)P.x.data + b * P.x.stride_batch + c;
    const E *dy = (const E *)P.dy.data + b * P.dy.stride_batch + c;
    E *dx = (E *)P.dx.data + b * P.dx.stride_batch + c;
    const E *s0 = P.initial_state ? (const E *)P.initial_state + b * (K - 1) * P.width + c : nullptr;
    const E *df = P.dfinal_state ? (const E *)P.dfinal_state + b * (K - 1) * P.width + c : nullptr;
    E *ds = P.dinitial_state ? (E *)P.dinitial_state + b * (K - 1) * P.width + c : nullptr;
    float w[K][V], bias[V] = {}, xw[K][V], dp[K][V];
    for (int i = 0; i < V; ++i) {
      for (int k = 0; k < K; ++k) w[k][i] = P.weight[(c + i) * K + k];
      if (P.bias) bias[i] = P.bias[c + i];
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      for (int i = 0; i < V; ++i) xw[j][i] = dp[j][i] = 0.f;
      const int p = s + j - K;  // xw[1..K-1]: positions s-K+1 .. s-1 (moved down by one at the first step)
      if (j > 0 && p < 0) {
        if (s0) load<DT, V>(xw[j], s0 + (p + K - 1) * P.width);
      } else if (j > 0 && p < len) {
        load<DT, V>(xw[j], x + p * P.x.stride_length);
      }
    }
    constexpr int U = 2;
    const int last = e + K - 1, loads = min(len, last), inner = min(len, e);
    const E *xq = x + s * P.x.stride_length, *dq = dy + s * P.dy.stride_length;
    E *dxl = dx + (int64_t)(s - (K - 1)) * P.dx.stride_length;
    Raw<DT, V> xa[U], da[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      xa[j].load(xq + j * P.x.stride_length, s + j < loads);
      da[j].load(dq + j * P.dy.stride_length, s + j < loads);
    }
    auto positions = [&](auto whole, int q0) {
      constexpr bool WHOLE = decltype(whole)::value;
      xq += U * P.x.stride_length, dq += U * P.dy.stride_length;
      Raw<DT, V> xn[U], dn[U];
#pragma unroll
      for (int j = 0; j < U; ++j) xn[j] = xa[j], dn[j] = da[j];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (WHOLE) {
          xa[j].load_all(xq + j * P.x.stride_length);
          da[j].load_all(dq + j * P.dy.stride_length);
        } else {
          xa[j].load(xq + j * P.x.stride_length, q0 + U + j < loads);
          da[j].load(dq + j * P.dy.stride_length, q0 + U + j < loads);
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int q = q0 + j, l = q - (K - 1), jf = q - len;
        float v[V] = {};
        if (!WHOLE && df && jf >= 0 && jf < K - 1 && q < last) load<DT, V>(v, df + jf * P.width);
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
          for (int k = 0; k + 1 < K; ++k) {
            xw[k][i] = xw[k + 1][i];
            dp[k][i] = dp[k + 1][i];
          }
          xw[K - 1][i] = xn[j][i];
          float d = dn[j][i];
          if (SILU) {
            float a = bias[i];
            for (int k = 0; k < K; ++k) a = __builtin_fmaf(w[k][i], xw[k][i], a);
            d *= silu_slope(a, sigmoid(a));
          }
          d = WHOLE || q < len ? d : 0.f;
          dp[K - 1][i] = d;
          // (where the run or the row has ended nothing is added, not even zero times an input: that one may be infinite)
          if (WHOLE || q < inner) {
            for (int k = 0; k < K; ++k) dw[k][i] = __builtin_fmaf(d, xw[k][i], dw[k][i]);
            dw[K][i] += d;
          }
          for (int k = 0; k < K; ++k) v[i] = WHOLE && k == 0 ? w[0][i] * dp[K - 1][i] : __builtin_fmaf(w[k][i], dp[K - 1 - k][i], v[i]);
          v[i] = WHOLE || l < len ? v[i] : 0.f;
        }
        if (WHOLE || (q < last && l >= s)) {
          store<DT, V>(dxl, v);
        } else if (q < last && l < 0 && s == 0) {
          if (ds) store<DT, V>(ds + (l + K - 1) * P.width, v);
        }
        dxl += P.dx.stride_length;
      }
    };
    for (int q0 = s; q0 < last; q0 += U) {
      if (q0 >= s + K - 1 && q0 + 2 * U <= inner)
        positions(std::true_type(), q0);
      else
        positions(std::false_type(), q0);
    }
  }
  if (!part) return;
  const int64_t row = b * T.tiles_l + lt;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    __syncthreads();
    for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = dw[k][i];
    __syncthreads();
    if (lane_l == 0 && inside) {
      for (int i = 0; i < V; ++i) {
        float a = 0.f;
        for (int r = 0; r < ty; ++r) a += red[((r << T.log_cx) + lane_c) * V + i];
        part[(row * (K + 1) + k) * P.width + c + i] = a;
      }
    }
  }
}

// dweight, dbias: the partial rows summed in their order
__global__ __launch_bounds__(1024) void k_conv_params(const float *part, int64_t rows, int64_t width, int taps, float *dweight,
                                                      float *dbias, int64_t base) {
  __shared__ float red[1024];
  const int64_t cols = (taps + 1) * width, col = (base + blockIdx.x) * 64 + (threadIdx.x & 63);
  const float a = column_sum(part, rows, cols, col, red);
  if (threadIdx.x >= 64 || col >= cols) return;
  const int64_t k = col / width, w = col - k * width;
  if (k < taps) {
    if (dweight) dweight[w * taps + k] = a;
  } else if (dbias) {
    dbias[w] = a;
  }
}

namespace {

int elem_bytes(int dtype) { return dtype == AFC_F32 ? 4 : 2; }

void check_sizes(const afc_conv_args *p) {
  want(p != nullptr, "null arguments");
  want(p->dtype >= AFC_F32 && p->dtype <= AFC_F16, "dtype must be AFC_F32, AFC_BF16 or AFC_F16");
  want(p->taps >= 2 && p->taps <= 4, "taps must be 2, 3 or 4");
  check_axes(p->batch, p->length, p->width);
}

void check(const afc_conv_args *p, bool grad, bool step) {
  check_sizes(p);
  want(p->weight != nullptr, "weight is missing");
  if (step) want(p->length == 1 && !p->lengths && (p->final_state || p->batch == 0) && p->final_state == p->initial_state, "a step takes length 1, no lengths, and its state as initial_state and final_state");
  if (p->batch == 0 || p->length == 0) return;
  check_seq(p->x, p->batch, p->length, 0, "x");
  if (!grad) check_seq(p->y, p->batch, p->length, 0, "y");
  if (grad) {
    check_seq(p->dy, p->batch, p->length, 0, "dy");
    check_seq(p->dx, p->batch, p->length, 0, "dx");
  }
}

Tiling tiling(const afc_conv_args *p, int v, int run) {
  Tiling t;
  const int64_t lanes = ceil_div(p->width, v);
  t.log_cx = 0;
  while (t.log_cx < 6 && (1 << t.log_cx) < lanes) ++t.log_cx;
  t.run = run;
  t.tiles_c = ceil_div(lanes, 1 << t.log_cx);
  t.tiles_l = ceil_div(p->length > 0 ? p->length : 1, (int64_t)run * (256 >> t.log_cx));
  t.base = 0;
  return t;
}
int64_t blocks(const afc_conv_args *p, const Tiling &t) {
  const int64_t n = p->batch * t.tiles_l * t.tiles_c;
  want(n < kMostBlocks, "too many blocks");
  return n;
}
// Positions of a thread: long runs read the filter and the K - 1 positions that neighbours share less often (and leave fewer
// partial rows of the filter's gradient), short ones give the chip enough threads.
Tiling run_tiling(const afc_conv_args *p, int v, int run) {
  Tiling t = tiling(p, v, run);
  while (run > 8 && p->batch * t.tiles_l * t.tiles_c < 1024) t = tiling(p, v, run /= 2);
  return t;
}
// Channels of a gradient thread.  Eight 16-bit ones would make 16 bytes a load, but with the windows of inputs and of dp, the filter and
// its gradient they need 256 registers and more: 265 us against 242 for 3 x 8191 x 4096 forwards and backwards.
constexpr int kGradVector = 4;
Tiling grad_tiling(const afc_conv_args *p, int v) { return run_tiling(p, v, 64); }
uint64_t grad_bytes(const afc_conv_args *p) {
  uint64_t most = 0;
  for (int v : {1, kGradVector}) {
    const Tiling t = grad_tiling(p, v);
    const uint64_t n = up256((uint64_t)p->batch * t.tiles_l * (p->taps + 1) * p->width * 4);
    most = n > most ? n : most;
  }
  return most;
}

#define CONV_SILU(DT, V, K, ...) (p->silu ? CONV_GO(DT, V, K, true, __VA_ARGS__) : CONV_GO(DT, V, K, false, __VA_ARGS__))
#define CONV_TAPS(DT, V, ...) \
  (p->taps == 2 ? CONV_SILU(DT, V, 2, __VA_ARGS__) : p->taps == 3 ? CONV_SILU(DT, V, 3, __VA_ARGS__) : CONV_SILU(DT, V, 4, __VA_ARGS__))
#define CONV_TYPES(wide, VF, VH)                                                                   \
  (p->dtype == AFC_F32 ? (wide ? CONV_TAPS(AFC_F32, VF, 0) : CONV_TAPS(AFC_F32, 1, 0))             \
   : p->dtype == AFC_BF16 ? (wide ? CONV_TAPS(AFC_BF16, VH, 0) : CONV_TAPS(AFC_BF16, 1, 0))        \
                          : (wide ? CONV_TAPS(AFC_F16, VH, 0) : CONV_TAPS(AFC_F16, 1, 0)))

}  // namespace

static void conv(const afc_conv_args *p, hipStream_t st) {
  check(p, false, false);
  const int v = 16 / elem_bytes(p->dtype);
  const bool wide = p->width >= v;
  const Tiling t = run_tiling(p, wide ? v : 1, 32);
  const int64_t n = blocks(p, t);
  OnDevice on(p->device);
  if (p->length == 0 && !p->final_state) return;
  in_slices(n, 256, "k_conv", [&](int64_t base, dim3 grid) {
    Tiling s = t;
    s.base = base;
#define CONV_GO(DT, V, K, S, ...) (k_conv<DT, V, K, S><<<grid, 256, 0, st>>>(*p, s), 0)
    (void)CONV_TYPES(wide, 4, 8);
#undef CONV_GO
  });
}

static void conv_step(const afc_conv_args *p, hipStream_t st) {
  check(p, false, true);
  const int v = 16 / elem_bytes(p->dtype);
  const bool wide = p->width % v == 0;  // (the state is updated in place: no two lanes may share a channel)
  const int64_t n = ceil_div(p->batch * (p->width / (wide ? v : 1)), 256);
  want(n < kMostBlocks, "too many blocks");
  OnDevice on(p->device);
  in_slices(n, 256, "k_conv_step", [&](int64_t base, dim3 grid) {
#define CONV_GO(DT, V, K, S, ...) (k_conv_step<DT, V, K, S><<<grid, 256, 0, st>>>(*p, base), 0)
    (void)CONV_TYPES(wide, 4, 8);
#undef CONV_GO
  });
}

static void conv_grad(const afc_conv_args *p, hipStream_t st) {
  check(p, true, false);
  const bool params = p->dweight || p->dbias;
  const bool wide = p->width >= kGradVector;
  const Tiling t = grad_tiling(p, wide ? kGradVector : 1);
  float *part = params ? (float *)p->workspace : nullptr;
  const int64_t rows = p->batch * t.tiles_l;
  if (params)
    want(p->batch == 0 || (part && p->workspace_bytes >= grad_bytes(p) && (uintptr_t)part % 256 == 0), "workspace is missing, too small or not 256-byte aligned");
  const int64_t n = blocks(p, t);
  OnDevice on(p->device);
  in_slices(n, 256, "k_conv_grad", [&](int64_t base, dim3 grid) {
    Tiling s = t;
    s.base = base;
#define CONV_GO(DT, V, K, S, ...) (k_conv_grad<DT, V, K, S><<<grid, 256, 0, st>>>(*p, s, part), 0)
    (void)CONV_TYPES(wide, 4, 4);
#undef CONV_GO
  });
  if (params)
    in_slices(ceil_div((p->taps + 1) * p->width, 64), 1024, "k_conv_params", [&](int64_t base, dim3 grid) {
      k_conv_params<<<grid, 1024, 0, st>>>(part, rows, p->width, p->taps, p->dweight, p->dbias, base);
    });
}

}  // namespace afc_ops

extern "C" {
int afc_conv(const afc_conv_args *args, void *hip_stream) {
  return afc_ops::entry("afc_conv", [&] { afc_ops::conv(args, (hipStream_t)hip_stream); });
}
int afc_conv_step(const afc_conv_args *args, void *hip_stream) {
  return afc_ops::entry("afc_conv_step", [&] { afc_ops::conv_step(args, (hipStream_t)hip_stream); });
}
int afc_conv_grad(const afc_conv_args *args, void *hip_stream) {
  return afc_ops::entry("afc_conv_grad", [&] { afc_ops::conv_grad(args, (hipStream_t)hip_stream); });
}
int afc_conv_workspace(const afc_conv_args *args, uint64_t *bytes) {
  return afc_ops::entry("afc_conv_workspace", [&] {
    afc_ops::check_sizes(args);
    afc_ops::want(bytes != nullptr, "null argument");
    *bytes = afc_ops::grad_bytes(args);
  });
}
}
