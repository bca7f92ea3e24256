// scan.hip -- selective state space scan (afc_scan, afc_scan_grad, afc_scan_step)
//
//   delta = softplus(dt + bias)      h[l] = exp(delta A) h[l-1] + delta x B      y = (<C, h> + D x) silu(z)
//   backwards, with dy = dout silu(z):
//   g[l] = dy C + exp(delta A)[l+1] g[l+1]     du = <g, B>     t = g exp(delta A) h[l-1]
//   dx = du delta + D dy     ddelta = du x + <t, A>     dA = sum t delta     dB = sum_w g delta x     dC = sum_w dy h
//
// What bounds it: each of batch x length x width x state decays takes an exponential (16 clocks of a SIMD for 64 of them) and
// four multiply-adds forwards, eight more backwards, while the tensors that are read and written are state times smaller.  So
// the states stay in registers, everything that is the same for several states is computed once per position and channel and
// handed over through LDS, and no instruction is spent on a state but the recurrence.
#include <stdexcept>

#include "ops_common.h"

namespace afc_ops {

// ---- how the work lies ----
// A block of four waves takes CB channels of one row, K positions (a chunk) at a time.  In the recurrence a lane holds S states of
// one channel, NL lanes a channel: lane = (c / 4, nl, c % 4), so that sums over nl are rotations inside 16 lanes and sums over
// channels are two half-wave exchanges and two steps inside four lanes.  Before and after it a thread has E neighbouring
// channels of one position (threadIdx.x / 16): whole rows of memory, and the activations once instead of NL times.
constexpr int K = 16;

template <int S, int NL>
struct Shape {
  static constexpr int CPW = 64 / NL, CB = 4 * CPW, E = CB / 16, NP = S * NL, NB = (K * NP + 255) / 256;
};

struct Plan {
  int tiles;       // blocks side by side in a group's channels
  int segs;        // parts of the length that run at the same time
  int seg_chunks;  // chunks of a part
  int chunks;
};

template <int CTRL>
__device__ inline float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kRor4 = 0x124, kRor8 = 0x128;

// lanes 16 (32) apart: a keeps its even rows (lower half) and gets b's, b gets a's odd rows (upper half) and keeps its own
__device__ inline float swap_add16(float a, float b) {
  auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
__device__ inline float swap_add32(float a, float b) {
  auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// the sum over a channel's NL lanes, in all of them
template <int NL>
__device__ inline float sum_states(float v) {
  v += dpp<kRor8>(v);
  v += dpp<kRor4>(v);
  if (NL > 4) v = swap_add16(v, v);
  if (NL > 8) v = swap_add32(v, v);
  return v;
}

// v[i], i < CPW: the lane of channel c gets the sum of v[c] over the wave's channels.  Each step halves the values: a lane keeps
// one half of them and hands the other to its partner (CPW - 1 additions for CPW sums instead of log2 CPW for each).
template <int NL>
__device__ inline float sum_channels(float *v, int lane) {
  constexpr int CPW = 64 / NL;
  int n = CPW / 2;
  if (NL <= 8) {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = swap_add32(v[i], v[i + n]);
    n /= 2;
  }
  if (NL <= 4) {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = swap_add16(v[i], v[i + n]);
    n /= 2;
  }
  const bool two = lane & 2, one = lane & 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float mine = two ? v[i + 2] : v[i], other = two ? v[i] : v[i + 2];
    v[i] = mine + dpp<kXor2>(other);
  }
  const float mine = one ? v[1] : v[0], other = one ? v[0] : v[1];
  return mine + dpp<kXor1>(other);
}

// E neighbouring elements in the form in which they were loaded (converted where they are used, so that loads stay in flight)
template <int DT, int E, bool VEC>
struct Piece {
  Elem<DT> v[E];
  __device__ inline void load(const Elem<DT> *p, int n) {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = i < n ? p[i] : (Elem<DT>)0.f;
  }
  __device__ inline float operator[](int i) const { return (float)v[i]; }
};
template <int DT, int E>
struct Piece<DT, E, true> {
  typedef Elem<DT> V __attribute__((ext_vector_type(E)));
  V v;
  __device__ inline void load(const Elem<DT> *p, int n) {
    v = (V)(Elem<DT>)0.f;
    if (n > 0) v = *reinterpret_cast<const V *>(p);
  }
  __device__ inline float operator[](int i) const { return (float)v[i]; }
};
template <int DT, int E, bool VEC>
__device__ inline void store(Elem<DT> *p, const float *f, int n) {
  if constexpr (VEC) {
    typename Piece<DT, E, true>::V v;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = (Elem<DT>)f[i];
    if (n > 0) *reinterpret_cast<typename Piece<DT, E, true>::V *>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < n) p[i] = (Elem<DT>)f[i];
  }
}
template <int S>
struct States {
  typedef float V __attribute__((ext_vector_type(S)));
};
template <>
struct States<1> {
  typedef float V __attribute__((ext_vector_type(1)));
};
template <int S>
__device__ inline void load_states(float *h, const float *p) {
  const typename States<S>::V v = *reinterpret_cast<const typename States<S>::V *>(p);
#pragma unroll
  for (int s = 0; s < S; ++s) h[s] = v[s];
}
template <int S>
__device__ inline void store_states(float *p, const float *h) {
  typename States<S>::V v;
#pragma unroll
  for (int s = 0; s < S; ++s) v[s] = h[s];
  *reinterpret_cast<typename States<S>::V *>(p) = v;
}

// where a thread is
template <int S, int NL>
struct Place {
  typedef Shape<S, NL> H;
  int b, g, tile, seg, len, nw;  // nw: channels of the block
  int lane, wave, nl, c, cb;     // recurrence: states nl S .. of channel cb of the block
  int r, q, n;                   // before and after it: position r of the chunk, channels q .. q + n of the block
  int64_t w0;                    // the block's first channel
  __device__ Place(const afc_scan_args &P, const Plan &T) {
    unsigned k = blockIdx.x;
    seg = k % T.segs, k /= T.segs;
    tile = k % T.tiles, k /= T.tiles;
    g = k % (unsigned)P.groups, b = k / (unsigned)P.groups;
    const int wg = (int)(P.width / P.groups);
    w0 = (int64_t)g * wg + (int64_t)tile * H::CB;
    nw = min(H::CB, wg - tile * H::CB);
    len = row_length(P.lengths, b, P.length);
    lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    nl = (lane >> 2) & (NL - 1);
    c = lane / (4 * NL) * 4 + (lane & 3);
    cb = wave * H::CPW + c;
    r = threadIdx.x >> 4, q = (threadIdx.x & 15) * H::E;
    n = max(0, min(H::E, nw - q));
  }
  __device__ int first_chunk(const Plan &T) const { return seg * T.seg_chunks; }
  __device__ int end_chunk(const Plan &T) const { return min((seg + 1) * T.seg_chunks, T.chunks); }
  __device__ int live_end(const Plan &T) const { return max(first_chunk(T), min(end_chunk(T), (len + K - 1) / K)); }
};

// rows of B or C: K positions of NP states; what lies behind the row or the state is zero
template <int DT, int S, int NL>
struct Rows {
  typedef Shape<S, NL> H;
  Elem<DT> v[H::NB];
  __device__ inline void load(const afc_seq &s, const Place<S, NL> &at, int l0, int N) {
#pragma unroll
    for (int i = 0; i < H::NB; ++i) {
      const int k = (threadIdx.x + 256 * i) / H::NP, n = (threadIdx.x + 256 * i) % H::NP, l = l0 + k;
      v[i] = (Elem<DT>)0.f;
      if (k < K && n < N && l < at.len) v[i] = ((const Elem<DT> *)s.data)[at.b * s.stride_batch + l * s.stride_length + at.g * s.stride_group + n];
    }
  }
  __device__ inline void put(float *to) const {
#pragma unroll
    for (int i = 0; i < H::NB; ++i)
      if (K * H::NP >= 256 * (i + 1) || threadIdx.x + 256 * i < K * H::NP) to[threadIdx.x + 256 * i] = (float)v[i];
  }
};

template <int DT, int E, bool VEC>
__device__ inline Piece<DT, E, VEC> piece(const afc_seq &s, int64_t b, int64_t l, int64_t w, int n) {
  Piece<DT, E, VEC> p;
  p.load((const Elem<DT> *)s.data + b * s.stride_batch + l * s.stride_length + w, n);
  return p;
}

// decays are computed as 2^(delta A log2 e)
template <int S, int NL>
__device__ inline void decay_rates(float *a2, const afc_scan_args &P, const Place<S, NL> &at) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int n = at.nl * S + s;
    a2[s] = at.cb < at.nw && n < P.state ? P.a[(at.w0 + at.cb) * P.state + n] * 1.44269504088896341f : 0.f;
  }
}
template <int S, int NL>
__device__ inline void state_or_zero(float *h, const float *from, const afc_scan_args &P, const Place<S, NL> &at) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int n = at.nl * S + s;
    h[s] = from && at.cb < at.nw && n < P.state ? from[(at.b * P.width + at.w0 + at.cb) * P.state + n] : 0.f;
  }
}
template <int S, int NL>
__device__ inline void put_state(float *to, const float *h, const afc_scan_args &P, const Place<S, NL> &at) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int n = at.nl * S + s;
    if (to && at.cb < at.nw && n < P.state) to[(at.b * P.width + at.w0 + at.cb) * P.state + n] = h[s];
  }
}

// Parts of the length run at the same time where the rows and channels alone do not fill the chip.  What a part hands on from
// a zero state (`state` [batch, segs, width, NP]) and the sum of its step sizes (`steps` [batch, segs, width]: the decay across it
// is exp(A steps)) come from a pass of their own; each part then works out what reaches it from all the parts before it.
struct Carry {
  float *state, *steps;
};

// ---- forwards ----
// CARRY: only the carries are computed (of all parts but the last)
template <int DT, int S, int NL, bool VEC, bool CARRY>
__global__ __launch_bounds__(256) void k_scan(afc_scan_args P, Plan T, Carry carry) {
  typedef Shape<S, NL> H;
  constexpr int E = H::E;
  __shared__ float2 steps[K][H::CB];  // delta, delta x
  __shared__ __align__(16) float bs[K * H::NP], cs[CARRY ? 4 : K * H::NP];
  __shared__ float ys[CARRY ? 1 : K][H::CB];
  const Place<S, NL> at(P, T);
  if (CARRY && at.seg == T.segs - 1) return;
  float a2[S], h[S], total = 0.f;
  decay_rates<S, NL>(a2, P, at);
  const int64_t w = at.w0 + at.cb;
  if (CARRY) {
    for (int s = 0; s < S; ++s) h[s] = 0.f;
  } else {
    state_or_zero<S, NL>(h, P.initial_state, P, at);
    if (at.cb < at.nw)
      for (int j = 0; j < at.seg; ++j) {
        float e[S];
        load_states<S>(e, carry.state + (((int64_t)at.b * T.segs + j) * P.width + w) * H::NP + at.nl * S);
        const float d = carry.steps[((int64_t)at.b * T.segs + j) * P.width + w];
        for (int s = 0; s < S; ++s) h[s] = __builtin_fmaf(__builtin_amdgcn_exp2f(d * a2[s]), h[s], e[s]);
      }
  }
  float bias[E], D[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    bias[i] = P.dt_bias && i < at.n ? P.dt_bias[at.w0 + at.q + i] : 0.f;
    D[i] = P.d && i < at.n ? P.d[at.w0 + at.q + i] : 0.f;
  }
  const int first = at.first_chunk(T), live = at.live_end(T), end = at.end_chunk(T);
  Piece<DT, E, VEC> x{}, dt{}, z{};
  Rows<DT, S, NL> rb, rc;
  auto fetch = [&](int ch) {
    const int l = ch * K + at.r, n = l < at.len ? at.n : 0;
    x = piece<DT, E, VEC>(P.x, at.b, l, at.w0 + at.q, n);
    dt = piece<DT, E, VEC>(P.dt, at.b, l, at.w0 + at.q, n);
    if (!CARRY && P.z.data) z = piece<DT, E, VEC>(P.z, at.b, l, at.w0 + at.q, n);
    rb.load(P.b, at, ch * K, P.state);
    if (!CARRY) rc.load(P.c, at, ch * K, P.state);
  };
  if (first < live) fetch(first);
  for (int ch = first; ch < live; ++ch) {
    const int l = ch * K + at.r;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float v = dt[i] + bias[i], step = l < at.len && i < at.n ? (P.softplus ? softplus(v) : v) : 0.f;
      steps[at.r][at.q + i] = make_float2(step, step * x[i]);
    }
    rb.put(bs);
    if (!CARRY) rc.put(cs);
    const Piece<DT, E, VEC> x0 = x, z0 = z;
    __syncthreads();
    if (ch + 1 < live) fetch(ch + 1);
    if (!CARRY && P.checkpoints && at.cb < at.nw) store_states<S>(P.checkpoints + (((int64_t)at.b * T.chunks + ch) * P.width + w) * H::NP + at.nl * S, h);
#pragma unroll
    for (int k4 = 0; k4 < K; k4 += 4) {
      float y[4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int k = k4 + kk;
        const float2 d = steps[k][at.cb];
        float B[S], C[S];
        load_states<S>(B, bs + k * H::NP + at.nl * S);
        if (!CARRY) load_states<S>(C, cs + k * H::NP + at.nl * S);
        y[kk] = 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          h[s] = __builtin_fmaf(__builtin_amdgcn_exp2f(d.x * a2[s]), h[s], d.y * B[s]);
          if (!CARRY) y[kk] = s ? __builtin_fmaf(C[s], h[s], y[kk]) : C[s] * h[s];
        }
        if (CARRY)
          total += d.x;
        else
          y[kk] = sum_states<NL>(y[kk]);
      }
      if (!CARRY) {
        const float lo = at.nl & 1 ? y[1] : y[0], hi = at.nl & 1 ? y[3] : y[2];
        if (at.nl < 4) ys[k4 + at.nl][at.cb] = at.nl & 2 ? hi : lo;
      }
    }
    __syncthreads();
    if (!CARRY && l < P.length) {
      float y[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        y[i] = __builtin_fmaf(D[i], x0[i], ys[at.r][at.q + i]);
        if (P.z.data) y[i] *= silu(z0[i]);
        y[i] = l < at.len ? y[i] : 0.f;
      }
      store<DT, E, VEC>((Elem<DT> *)P.y.data + at.b * P.y.stride_batch + l * P.y.stride_length + at.w0 + at.q, y, at.n);
    }
  }
  if (CARRY) {
    if (at.cb < at.nw) {
      store_states<S>(carry.state + (((int64_t)at.b * T.segs + at.seg) * P.width + w) * H::NP + at.nl * S, h);
      if (at.nl == 0) carry.steps[((int64_t)at.b * T.segs + at.seg) * P.width + w] = total;
    }
    return;
  }
  for (int ch = live; ch < end; ++ch) {
    const int l = ch * K + at.r;
    const float zero[E] = {};
    if (l < P.length) store<DT, E, VEC>((Elem<DT> *)P.y.data + at.b * P.y.stride_batch + l * P.y.stride_length + at.w0 + at.q, zero, at.n);
  }
  if (at.seg == T.segs - 1) put_state<S, NL>(P.final_state, h, P, at);
}

// ---- backwards ----
// sums that are finished by k_scan_finish: bc [batch, groups, tiles, length, 2, NP], a [batch, segs, width, NP], d and bias
// [batch, segs, width]
struct Sums {
  float *bc, *a, *d, *bias;
};

// A chunk is run forwards again from its checkpoint with the states and decays of its K positions in registers, then
// backwards.
template <int DT, int S, int NL, bool VEC, bool CARRY>
__global__ __launch_bounds__(256) void k_scan_grad(afc_scan_args P, Plan T, Carry carry, Sums sums) {
  typedef Shape<S, NL> H;
  constexpr int E = H::E, V = 2 * S;
  __shared__ float2 steps[K][H::CB];
  __shared__ float dys[K][H::CB];
  __shared__ __align__(16) float bs[CARRY ? 4 : K * H::NP], cs[K * H::NP];
  __shared__ float ys[CARRY ? 1 : K][H::CB], dus[CARRY ? 1 : K][H::CB], tas[CARRY ? 1 : K][H::CB];
  __shared__ float part[CARRY ? 1 : 4][CARRY ? 1 : K * 2 * H::NP];
  const Place<S, NL> at(P, T);
  if (CARRY && at.seg == 0) return;
  float a2[S], g[S], total = 0.f;
  decay_rates<S, NL>(a2, P, at);
  const int64_t w = at.w0 + at.cb;
  if (CARRY) {
    for (int s = 0; s < S; ++s) g[s] = 0.f;
  } else {
    state_or_zero<S, NL>(g, P.dfinal_state, P, at);
    if (at.cb < at.nw)
      for (int j = T.segs - 1; j > at.seg; --j) {
        float e[S];
        load_states<S>(e, carry.state + (((int64_t)at.b * T.segs + j) * P.width + w) * H::NP + at.nl * S);
        const float d = carry.steps[((int64_t)at.b * T.segs + j) * P.width + w];
        for (int s = 0; s < S; ++s) g[s] = __builtin_fmaf(__builtin_amdgcn_exp2f(d * a2[s]), g[s], e[s]);
      }
  }
  float bias[E], D[E], sum_d[E], sum_b[E], sum_a[S];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    bias[i] = P.dt_bias && i < at.n ? P.dt_bias[at.w0 + at.q + i] : 0.f;
    D[i] = P.d && i < at.n ? P.d[at.w0 + at.q + i] : 0.f;
    sum_d[i] = sum_b[i] = 0.f;
  }
#pragma unroll
  for (int s = 0; s < S; ++s) sum_a[s] = 0.f;
  const int first = at.first_chunk(T), live = at.live_end(T), end = at.end_chunk(T);
  Piece<DT, E, VEC> x{}, dt{}, z{}, dout{};
  Rows<DT, S, NL> rb, rc;
  float h0[S];
  auto fetch = [&](int ch) {
    const int l = ch * K + at.r, n = l < at.len ? at.n : 0;
    if (!CARRY) x = piece<DT, E, VEC>(P.x, at.b, l, at.w0 + at.q, n);
    dt = piece<DT, E, VEC>(P.dt, at.b, l, at.w0 + at.q, n);
    if (P.z.data) z = piece<DT, E, VEC>(P.z, at.b, l, at.w0 + at.q, n);
    dout = piece<DT, E, VEC>(P.dy, at.b, l, at.w0 + at.q, n);
    if (!CARRY) rb.load(P.b, at, ch * K, P.state);
    rc.load(P.c, at, ch * K, P.state);
    if (!CARRY) {
      for (int s = 0; s < S; ++s) h0[s] = 0.f;
      if (at.cb < at.nw) load_states<S>(h0, P.checkpoints + (((int64_t)at.b * T.chunks + ch) * P.width + w) * H::NP + at.nl * S);
    }
  };
  if (!CARRY) {  // behind the row's end
    const float zero[E] = {};
    for (int ch = live; ch < end; ++ch) {
      const int l = ch * K + at.r;
      if (l < P.length) {
        store<DT, E, VEC>((Elem<DT> *)P.dx.data + at.b * P.dx.stride_batch + l * P.dx.stride_length + at.w0 + at.q, zero, at.n);
        store<DT, E, VEC>((Elem<DT> *)P.ddt.data + at.b * P.ddt.stride_batch + l * P.ddt.stride_length + at.w0 + at.q, zero, at.n);
        if (P.dz.data) store<DT, E, VEC>((Elem<DT> *)P.dz.data + at.b * P.dz.stride_batch + l * P.dz.stride_length + at.w0 + at.q, zero, at.n);
      }
      for (int i = threadIdx.x; i < K * 2 * H::NP; i += 256)
        if (ch * K + i / (2 * H::NP) < P.length)
          sums.bc[((((int64_t)at.b * P.groups + at.g) * T.tiles + at.tile) * P.length + ch * K) * 2 * H::NP + i] = 0.f;
    }
  }
  if (first < live) fetch(live - 1);
  for (int ch = live - 1; ch >= first; --ch) {
    const int l = ch * K + at.r;
    float delta[E], dy[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float v = dt[i] + bias[i];
      delta[i] = l < at.len && i < at.n ? (P.softplus ? softplus(v) : v) : 0.f;
      dy[i] = dout[i];
      if (P.z.data) dy[i] *= silu(z[i]);
      steps[at.r][at.q + i] = make_float2(delta[i], CARRY ? 0.f : delta[i] * x[i]);
      dys[at.r][at.q + i] = dy[i];
    }
    if (!CARRY) rb.put(bs);
    rc.put(cs);
    const Piece<DT, E, VEC> x0 = x, dt0 = dt, z0 = z, dout0 = dout;
    float h[S];
    if (!CARRY)
      for (int s = 0; s < S; ++s) h[s] = h0[s];
    __syncthreads();
    if (ch > first) fetch(ch - 1);
    if (CARRY) {
#pragma unroll
      for (int k = K - 1; k >= 0; --k) {
        const float d = steps[k][at.cb].x, dyk = dys[k][at.cb];
        float C[S];
        load_states<S>(C, cs + k * H::NP + at.nl * S);
        total += d;
#pragma unroll
        for (int s = 0; s < S; ++s) g[s] = __builtin_amdgcn_exp2f(d * a2[s]) * __builtin_fmaf(dyk, C[s], g[s]);
      }
      __syncthreads();
      continue;
    }
    float before[K][S], a[K][S];
#pragma unroll
    for (int k4 = 0; k4 < K; k4 += 4) {
      float y[4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int k = k4 + kk;
        const float2 d = steps[k][at.cb];
        float B[S], C[S];
        load_states<S>(B, bs + k * H::NP + at.nl * S);
        load_states<S>(C, cs + k * H::NP + at.nl * S);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          before[k][s] = h[s];
          a[k][s] = __builtin_amdgcn_exp2f(d.x * a2[s]);
          h[s] = __builtin_fmaf(a[k][s], h[s], d.y * B[s]);
          y[kk] = s ? __builtin_fmaf(C[s], h[s], y[kk]) : C[s] * h[s];
        }
        y[kk] = sum_states<NL>(y[kk]);
      }
      const float lo = at.nl & 1 ? y[1] : y[0], hi = at.nl & 1 ? y[3] : y[2];
      if (at.nl < 4) ys[k4 + at.nl][at.cb] = at.nl & 2 ? hi : lo;
    }
    float v[H::CPW > V ? H::CPW : V];
#pragma unroll
    for (int k4 = K - 4; k4 >= 0; k4 -= 4) {
      float du[4], ta[4];
#pragma unroll
      for (int kk = 3; kk >= 0; --kk) {
        const int k = k4 + kk;
        const float2 d = steps[k][at.cb];
        const float dyk = dys[k][at.cb];
        float B[S], C[S];
        load_states<S>(B, bs + k * H::NP + at.nl * S);
        load_states<S>(C, cs + k * H::NP + at.nl * S);
        const int o = (K - 1 - k) * V % (H::CPW > V ? H::CPW : V);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          g[s] = __builtin_fmaf(dyk, C[s], g[s]);
          v[o + s] = g[s] * d.y;
          v[o + S + s] = dyk * (k == K - 1 ? h[s] : before[k < K - 1 ? k + 1 : k][s]);
          du[kk] = s ? __builtin_fmaf(g[s], B[s], du[kk]) : g[s] * B[s];
          g[s] *= a[k][s];
          const float t = g[s] * before[k][s];
          sum_a[s] = __builtin_fmaf(t, d.x, sum_a[s]);
          ta[kk] = s ? __builtin_fmaf(t, a2[s], ta[kk]) : t * a2[s];
        }
        du[kk] = sum_states<NL>(du[kk]);
        ta[kk] = sum_states<NL>(ta[kk]);
        // the set of CPW values that is complete: value i belongs to position K - 1 - i / V of the chunk
        if (o + V >= H::CPW) {
#pragma unroll
          for (int m = 0; m < (H::CPW > V ? H::CPW : V); m += H::CPW) {
            const int i = (K - 1 - k) * V + V - (H::CPW > V ? H::CPW : V) + m + at.c;
            const float sum = sum_channels<NL>(v + m, at.lane);
            part[at.wave][(K - 1 - i / V) * 2 * H::NP + (i % V / S) * H::NP + at.nl * S + i % S] = sum;
          }
        }
      }
      if (at.nl < 4) {
        dus[k4 + at.nl][at.cb] = at.nl & 2 ? (at.nl & 1 ? du[3] : du[2]) : (at.nl & 1 ? du[1] : du[0]);
        tas[k4 + at.nl][at.cb] = at.nl & 2 ? (at.nl & 1 ? ta[3] : ta[2]) : (at.nl & 1 ? ta[1] : ta[0]);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < K * 2 * H::NP; i += 256)
      if (ch * K + i / (2 * H::NP) < P.length)
        sums.bc[((((int64_t)at.b * P.groups + at.g) * T.tiles + at.tile) * P.length + ch * K) * 2 * H::NP + i] =
            (part[0][i] + part[1][i]) + (part[2][i] + part[3][i]);
    if (l < P.length) {
      const bool on = l < at.len;
      float dx[E], ddt[E], dz[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float du = dus[at.r][at.q + i], xi = x0[i];
        dx[i] = on ? __builtin_fmaf(du, delta[i], D[i] * dy[i]) : 0.f;
        ddt[i] = __builtin_fmaf(du, xi, tas[at.r][at.q + i] * 0.693147180559945309f);
        if (P.softplus) ddt[i] *= sigmoid(dt0[i] + bias[i]);
        ddt[i] = on ? ddt[i] : 0.f;
        sum_d[i] = __builtin_fmaf(dy[i], xi, sum_d[i]);
        sum_b[i] += ddt[i];
        const float zi = z0[i];
        dz[i] = on ? dout0[i] * __builtin_fmaf(D[i], xi, ys[at.r][at.q + i]) * silu_slope(zi, sigmoid(zi)) : 0.f;
      }
      store<DT, E, VEC>((Elem<DT> *)P.dx.data + at.b * P.dx.stride_batch + l * P.dx.stride_length + at.w0 + at.q, dx, at.n);
      store<DT, E, VEC>((Elem<DT> *)P.ddt.data + at.b * P.ddt.stride_batch + l * P.ddt.stride_length + at.w0 + at.q, ddt, at.n);
      if (P.dz.data) store<DT, E, VEC>((Elem<DT> *)P.dz.data + at.b * P.dz.stride_batch + l * P.dz.stride_length + at.w0 + at.q, dz, at.n);
    }
  }
  if (CARRY) {
    if (at.cb < at.nw) {
      store_states<S>(carry.state + (((int64_t)at.b * T.segs + at.seg) * P.width + w) * H::NP + at.nl * S, g);
      if (at.nl == 0) carry.steps[((int64_t)at.b * T.segs + at.seg) * P.width + w] = total;
    }
    return;
  }
  const int64_t row = (int64_t)at.b * T.segs + at.seg;
  if (at.cb < at.nw) store_states<S>(sums.a + (row * P.width + w) * H::NP + at.nl * S, sum_a);
  if (at.seg == 0) put_state<S, NL>(P.dinitial_state, g, P, at);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < E; ++i) {
    dus[at.r][at.q + i] = sum_d[i];
    tas[at.r][at.q + i] = sum_b[i];
  }
  __syncthreads();
  if ((int)threadIdx.x < at.nw) {
    float sd = 0.f, sb = 0.f;
#pragma unroll
    for (int r = 0; r < K; ++r) {
      sd += dus[r][threadIdx.x];
      sb += tas[r][threadIdx.x];
    }
    sums.d[row * P.width + at.w0 + threadIdx.x] = sd;
    sums.bias[row * P.width + at.w0 + threadIdx.x] = sb;
  }
}

// db and dc: the sums over a group's tiles.  One thread for each value.
template <int DT>
__global__ __launch_bounds__(256) void k_scan_bc(afc_scan_args P, Plan T, const float *bc, int NP) {
  typedef Elem<DT> E;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = 2 * NP;
  if (i >= P.batch * P.groups * P.length * per) return;
  const int64_t row = i / (P.length * per), l = i / per % P.length, b = row / P.groups, g = row % P.groups;
  const int n = (int)(i % NP), c = (int)(i % per) / NP;
  if (n >= P.state) return;
  const float *from = bc + (row * T.tiles * P.length + l) * per + c * NP + n;
  float a = 0.f;
  for (int t = 0; t < T.tiles; ++t) a += from[t * P.length * per];
  const afc_seq &s = c ? P.dc : P.db;
  ((E *)s.data)[b * s.stride_batch + l * s.stride_length + g * s.stride_group + n] = (E)a;
}

// da, dd, ddt_bias: the sums over rows and parts, 64 columns and four interleaved runs of rows in a block
__global__ __launch_bounds__(256) void k_scan_params(afc_scan_args P, Sums sums, int64_t rows, int NP) {
  __shared__ float red[256];
  const int64_t na = P.width * NP, col = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int which = col < na ? 0 : col < na + P.width ? 1 : 2;
  const int64_t at = which == 0 ? col : col - na - (which - 1) * P.width, cols = which == 0 ? na : P.width;
  const float *from = which == 0 ? sums.a : which == 1 ? sums.d : sums.bias;
  float a = 0.f;
  if (at < cols)
    for (int64_t r = threadIdx.x >> 6; r < rows; r += 4) a += from[r * cols + at];
  red[threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.x >= 64 || at >= cols) return;
  a = (red[threadIdx.x] + red[threadIdx.x + 64]) + (red[threadIdx.x + 128] + red[threadIdx.x + 192]);
  if (which == 0) {
    if (P.da && at % NP < P.state) P.da[at / NP * P.state + at % NP] = a;
  } else if (which == 1) {
    if (P.dd) P.dd[at] = a;
  } else if (P.ddt_bias) {
    P.ddt_bias[at] = a;
  }
}

// ---- single tokens ----
// A channel's states lie side by side in NP lanes (a power of two, lanes behind `state` hold zeros), 64 / NP channels in a wave.
template <int NP>
__device__ inline float sum_lanes(float v) {
  for (int m = 1; m < NP; m <<= 1) v += __shfl_xor(v, m);
  return v;
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
  float y = sum_lanes<NP>(yc);
  if (!on || n) return;
  if (P.d) y = __builtin_fmaf(P.d[w], x, y);
  if (P.z.data) y *= silu((float)((const E *)P.z.data)[b * P.z.stride_batch + w]);
  ((E *)P.y.data)[b * P.y.stride_batch + w] = (Elem<DT>)y;
}

namespace {

void check_sizes(const afc_scan_args *p) {
  want(p != nullptr, "null arguments");
  want(p->dtype >= AFC_F32 && p->dtype <= AFC_F16, "dtype must be AFC_F32, AFC_BF16 or AFC_F16");
  want(p->state >= 1 && p->state <= 64, "state must be 1..64");
  want(p->batch >= 0 && p->length >= 0 && p->width >= 1, "batch, length or width");
  want(p->length < kMostAxis && p->width < kMostAxis && p->batch < kMostAxis, "an axis of 2^30 or more");
  want(p->groups >= 1 && p->width % p->groups == 0, "groups must divide width");
}

void check(const afc_scan_args *p, bool grad, bool step) {
  check_sizes(p);
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

// states of a lane and lanes of a channel: as few lanes as hold the state, four at least
struct Split {
  int s, nl;
};
Split split(const afc_scan_args *p) {
  const int n = p->state;
  return n <= 4 ? Split{1, 4} : n <= 8 ? Split{2, 4} : n <= 16 ? Split{4, 4} : n <= 32 ? Split{4, 8} : Split{4, 16};
}
int padded(const afc_scan_args *p) { return split(p).s * split(p).nl; }

Plan plan(const afc_scan_args *p) {
  Plan t;
  const int cb = 256 / split(p).nl;
  t.tiles = (int)ceil_div(p->width / p->groups, cb);
  t.chunks = (int)ceil_div(p->length, K);
  const int64_t blocks = p->batch * p->groups * t.tiles;
  int64_t segs = 1;
  while (blocks * segs < 512 && t.chunks / (segs * 2) >= 8 && segs < 64) segs *= 2;
  t.seg_chunks = (int)ceil_div(t.chunks > 0 ? t.chunks : 1, segs);
  t.segs = (int)ceil_div(t.chunks > 0 ? t.chunks : 1, t.seg_chunks);
  want(blocks * t.segs < (int64_t)1 << 31, "too many blocks");
  return t;
}

// vectors of E elements along the channels where every row and every tile starts on one
bool vectors(const afc_scan_args *p, std::initializer_list<const afc_seq *> seqs) {
  const int v = 16 / split(p).nl, e = p->dtype == AFC_F32 ? 4 : 2;
  if (p->width / p->groups % v) return false;
  for (const afc_seq *s : seqs)
    if (s->data && ((uintptr_t)s->data % (v * e) || s->stride_batch % v || s->stride_length % v)) return false;
  return true;
}

#define SCAN_SHAPE(DT, VEC, C)                       \
  switch (p->state <= 16 ? split(p).s : split(p).nl) { \
    case 1: SCAN_GO(DT, 1, 4, VEC, C); break;        \
    case 2: SCAN_GO(DT, 2, 4, VEC, C); break;        \
    case 4: SCAN_GO(DT, 4, 4, VEC, C); break;        \
    case 8: SCAN_GO(DT, 4, 8, VEC, C); break;        \
    default: SCAN_GO(DT, 4, 16, VEC, C); break;      \
  }
#define SCAN_VEC(DT, C)          \
  if (wide) {                    \
    SCAN_SHAPE(DT, true, C)      \
  } else {                       \
    SCAN_SHAPE(DT, false, C)     \
  }
#define SCAN_ALL(C)              \
  if (p->dtype == AFC_F32) {     \
    SCAN_VEC(AFC_F32, C)         \
  } else if (p->dtype == AFC_BF16) { \
    SCAN_VEC(AFC_BF16, C)        \
  } else {                       \
    SCAN_VEC(AFC_F16, C)         \
  }

uint64_t carry_bytes(const afc_scan_args *p, const Plan &t) {
  return t.segs > 1 ? up256((uint64_t)p->batch * t.segs * p->width * padded(p) * 4) + up256((uint64_t)p->batch * t.segs * p->width * 4) : 0;
}
Carry carry_at(const afc_scan_args *p, const Plan &t) {
  Carry c;
  c.state = (float *)p->workspace;
  c.steps = (float *)((char *)p->workspace + up256((uint64_t)p->batch * t.segs * p->width * padded(p) * 4));
  return c;
}
void check_workspace(const afc_scan_args *p, uint64_t bytes) {
  want(bytes == 0 || (p->workspace && p->workspace_bytes >= bytes && (uintptr_t)p->workspace % 256 == 0),
       "workspace is missing, too small or not 256-byte aligned");
}

void scan(const afc_scan_args *p, hipStream_t st) {
  check(p, false, false);
  const Plan t = plan(p);
  if (p->batch > 0) check_workspace(p, carry_bytes(p, t));
  want((uintptr_t)p->checkpoints % 16 == 0, "checkpoints must be 16-byte aligned");
  OnDevice on(p->device);
  if (p->batch == 0) return;
  const bool wide = vectors(p, {&p->x, &p->dt, &p->z, &p->y});
  const Carry carry = carry_at(p, t);
  const dim3 grid((unsigned)(p->batch * p->groups * t.tiles * t.segs));
#define SCAN_GO(DT, S, NL, VEC, C) k_scan<DT, S, NL, VEC, C><<<grid, 256, 0, st>>>(*p, t, carry)
  if (t.segs > 1) {
    SCAN_ALL(true)
    launched("k_scan (carry)");
  }
  SCAN_ALL(false)
#undef SCAN_GO
  launched("k_scan");
}

// the workspace of the gradients, one part after the other
struct Layout {
  uint64_t carry, bc, a, d, bias, all;
};
Layout layout(const afc_scan_args *p, const Plan &t) {
  Layout o;
  const uint64_t rows = (uint64_t)p->batch * t.segs * p->width * 4;
  o.carry = 0;
  o.bc = carry_bytes(p, t);
  o.a = o.bc + up256((uint64_t)p->batch * p->groups * t.tiles * p->length * 2 * padded(p) * 4);
  o.d = o.a + up256(rows * padded(p));
  o.bias = o.d + up256(rows);
  o.all = o.bias + up256(rows);
  return o;
}

void scan_grad(const afc_scan_args *p, hipStream_t st) {
  check(p, true, false);
  const Plan t = plan(p);
  const Layout o = layout(p, t);
  if (p->batch > 0) check_workspace(p, o.all);
  want((uintptr_t)p->checkpoints % 16 == 0, "checkpoints must be 16-byte aligned");
  OnDevice on(p->device);
  char *ws = (char *)p->workspace;
  const Carry carry = carry_at(p, t);
  const Sums sums = {(float *)(ws + o.bc), (float *)(ws + o.a), (float *)(ws + o.d), (float *)(ws + o.bias)};
  if (p->batch > 0) {
    const bool wide = vectors(p, {&p->x, &p->dt, &p->z, &p->dy, &p->dx, &p->ddt, &p->dz});
    const dim3 grid((unsigned)(p->batch * p->groups * t.tiles * t.segs));
#define SCAN_GO(DT, S, NL, VEC, C) k_scan_grad<DT, S, NL, VEC, C><<<grid, 256, 0, st>>>(*p, t, carry, sums)
    if (t.segs > 1) {
      SCAN_ALL(true)
      launched("k_scan_grad (carry)");
    }
    SCAN_ALL(false)
#undef SCAN_GO
    launched("k_scan_grad");
    const int64_t n = ceil_div(p->batch * p->length * p->groups * 2 * padded(p), 256);
    want(n < (int64_t)1 << 31, "too many blocks");
    if (n) {
      const dim3 gb((unsigned)n);
      if (p->dtype == AFC_F32) k_scan_bc<AFC_F32><<<gb, 256, 0, st>>>(*p, t, sums.bc, padded(p));
      if (p->dtype == AFC_BF16) k_scan_bc<AFC_BF16><<<gb, 256, 0, st>>>(*p, t, sums.bc, padded(p));
      if (p->dtype == AFC_F16) k_scan_bc<AFC_F16><<<gb, 256, 0, st>>>(*p, t, sums.bc, padded(p));
      launched("k_scan_bc");
    }
  }
  if (p->da || p->dd || p->ddt_bias) {
    const dim3 gp((unsigned)ceil_div(p->width * (padded(p) + 2), 64));
    k_scan_params<<<gp, 256, 0, st>>>(*p, sums, p->batch * t.segs, padded(p));
    launched("k_scan_params");
  }
}

int lanes(const afc_scan_args *p) {
  int n = 1;
  while (n < p->state) n *= 2;
  return n;
}
#define STEP_STATE(DT)                     \
  switch (lanes(p)) {                      \
    case 1: STEP_GO(DT, 1); break;         \
    case 2: STEP_GO(DT, 2); break;         \
    case 4: STEP_GO(DT, 4); break;         \
    case 8: STEP_GO(DT, 8); break;         \
    case 16: STEP_GO(DT, 16); break;       \
    case 32: STEP_GO(DT, 32); break;       \
    default: STEP_GO(DT, 64); break;       \
  }

void scan_step(const afc_scan_args *p, hipStream_t st) {
  check(p, false, true);
  OnDevice on(p->device);
  if (p->batch == 0) return;
  const int64_t n = p->batch * ceil_div(p->width, 64 / lanes(p));
  want(n < (int64_t)1 << 31, "too many blocks");
  const dim3 grid((unsigned)n);
#define STEP_GO(DT, NP) k_scan_step<DT, NP><<<grid, 64, 0, st>>>(*p)
  if (p->dtype == AFC_F32) STEP_STATE(AFC_F32)
  if (p->dtype == AFC_BF16) STEP_STATE(AFC_BF16)
  if (p->dtype == AFC_F16) STEP_STATE(AFC_F16)
#undef STEP_GO
  launched("k_scan_step");
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
    using namespace afc_ops;
    want(args && checkpoint_bytes && scan_bytes && grad_bytes, "null argument");
    check_sizes(args);
    const Plan t = plan(args);
    *checkpoint_bytes = up256((uint64_t)args->batch * t.chunks * args->width * padded(args) * 4);
    *scan_bytes = carry_bytes(args, t);
    *grad_bytes = layout(args, t).all;
  });
}
}
