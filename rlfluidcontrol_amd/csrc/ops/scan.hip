// scan.hip -- selective state space scan (afc_scan, afc_scan_grad, afc_scan_step)
//
//   delta = softplus(dt + bias)      h[l] = exp(delta A) h[l-1] + delta x B      y = (<C, h> + D x) silu(z)
//   backwards, with dy = dout silu(z):
//   g[l] = dy C + exp(delta A)[l+1] g[l+1]     du = <g, B>     t = g exp(delta A) h[l-1]
//   dx = du delta + D dy     ddelta = du x + <t, A>     dA = sum t delta     dB = sum_w g delta x     dC = sum_w dy h
//
// What bounds it: each of the batch x length x width x state decays takes an exponential (8 clocks of a SIMD for 64 of them) and
// four other instructions (4 clocks each) forwards, and 3 + 8 and another exponential backwards, while the tensors that are read
// and written are `state` times smaller.  So the states stay in registers, everything that is the same for several states is
// computed once per position and channel and handed over through LDS, and little is spent on a state but the recurrence.
// 8 x 2048 x 2048 x 16 in bf16: forwards 211 to 223 us, 2.4e12 states/s (the instructions above alone: 85 us; VALU busy 71 % of the
// time at 2.3 GHz, 1.8 TB/s with the checkpoints), backwards 536 to 575 us (200 us; VALU busy 77 % at 2.2 GHz).  What both have to
// read and write would take 106 us at a copy's rate.
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
  unsigned base;   // the slice's first block
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

// The sums of four positions' values over a channel's NL lanes: a lane gets the one of position four_at<NL>(nl).  Where the
// lanes are 16 and 32 apart a step halves the values (a lane keeps two of four, one of two), inside 16 lanes the rotations
// leave the sum in all of them: 11 instructions for four sums whatever NL is.
template <int NL>
__device__ inline int four_at(int nl) {
  return NL == 4 ? nl : NL == 8 ? (nl >> 2) * 2 + (nl & 1) : nl >> 2;
}
__device__ inline float sum_four_lanes(float v) {
  v += dpp<kRor8>(v);
  return v + dpp<kRor4>(v);
}
template <int NL>
__device__ inline float sum_four(float v0, float v1, float v2, float v3, int nl) {
  if (NL == 4) {
    v0 = sum_four_lanes(v0), v1 = sum_four_lanes(v1), v2 = sum_four_lanes(v2), v3 = sum_four_lanes(v3);
    const float lo = nl & 1 ? v1 : v0, hi = nl & 1 ? v3 : v2;
    return nl & 2 ? hi : lo;
  }
  if (NL == 8) {
    v0 = sum_four_lanes(swap_add16(v0, v2)), v1 = sum_four_lanes(swap_add16(v1, v3));
    return nl & 1 ? v1 : v0;
  }
  return sum_four_lanes(swap_add16(swap_add32(v0, v2), swap_add32(v1, v3)));
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

// E neighbouring elements in the form in which they were loaded (converted where they are used, so that loads stay in flight).
// They are loaded and stored together from any address that suits one element: the memory pipeline takes accesses that start
// anywhere, so rows of odd widths and slices need no scalar path.  WHOLE: n is E or 0, as where E divides a group's channels
// (without the branches for a last piece that is cut, 8 x 2048 x 2048 takes 760 us forwards and backwards, with them 880).
template <int DT, int E, bool WHOLE>
struct Piece {
  typedef Elem<DT> V __attribute__((ext_vector_type(E)));
  typedef Elem<DT> Any __attribute__((ext_vector_type(E), aligned(sizeof(Elem<DT>))));
  V v;
  __device__ inline void load(const Elem<DT> *p, int n) {
    v = (V)(Elem<DT>)0.f;
    if (WHOLE ? n > 0 : n == E) {
      v = *reinterpret_cast<const Any *>(p);
    } else if (!WHOLE && n > 0) {
#pragma unroll
      for (int i = 0; i + 1 < E; ++i)
        if (i < n) v[i] = p[i];
    }
  }
  __device__ inline void load_all(const Elem<DT> *p) { v = *reinterpret_cast<const Any *>(p); }
  __device__ inline float operator[](int i) const { return (float)v[i]; }
};
template <int DT, int E, bool WHOLE>
__device__ inline void store(Elem<DT> *p, const float *f, int n) {
  typename Piece<DT, E, WHOLE>::V v;
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = (Elem<DT>)f[i];
  if (WHOLE ? n > 0 : n == E) {
    *reinterpret_cast<typename Piece<DT, E, WHOLE>::Any *>(p) = v;
  } else if (!WHOLE && n > 0) {
#pragma unroll
    for (int i = 0; i + 1 < E; ++i)
      if (i < n) p[i] = v[i];
  }
}
template <int S>
struct States {
  typedef float V __attribute__((ext_vector_type(S)));
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

// a thread's own place in a tensor, moved from chunk to chunk (64-bit products of strides cost more than the loads they serve)
template <int DT>
struct Stream {
  Elem<DT> *p;
  int64_t step;
  __device__ Stream(const afc_seq &s, int64_t b, int64_t l, int64_t w) : p((Elem<DT> *)s.data + b * s.stride_batch + l * s.stride_length + w), step(K * s.stride_length) {}
  __device__ void next() { p += step; }
  __device__ void back() { p -= step; }
};

// where a thread is
template <int S, int NL>
struct Place {
  typedef Shape<S, NL> H;
  int b, g, tile, seg, len, nw;  // nw: channels of the block
  int lane, wave, nl, c, cb;     // recurrence: states nl S .. of channel cb of the block
  int r, q, n;                   // before and after it: position r of the chunk, channels q .. q + n of the block
  int64_t w0;                    // the block's first channel
  __device__ Place(const afc_scan_args &P, const Plan &T) {
    unsigned k = T.base + blockIdx.x;
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
  // where the thread may read rows: a thread without channels reads the block's first ones, and what it reads counts as zero
  __device__ int64_t readable() const { return w0 + (n > 0 ? q : 0); }
  __device__ int first_chunk(const Plan &T) const { return seg * T.seg_chunks; }
  __device__ int end_chunk(const Plan &T) const { return min((seg + 1) * T.seg_chunks, T.chunks); }
  __device__ int live_end(const Plan &T) const { return max(first_chunk(T), min(end_chunk(T), (len + K - 1) / K)); }
};

// rows of B or C: K positions of NP states; what lies behind the row or the state is zero
template <int DT, int S, int NL>
struct Rows {
  typedef Shape<S, NL> H;
  static constexpr int R = 256 / H::NP;  // positions between a thread's values
  const Elem<DT> *p;
  int64_t stride, step;
  int k, n;
  bool on;  // (of a padded state the thread reads the first one's value and puts zero)
  Elem<DT> v[H::NB], ahead[H::NB];
  __device__ Rows(const afc_seq &s, const Place<S, NL> &at, int64_t l0, int N)
      : stride(s.stride_length * R), step(K * s.stride_length), k(threadIdx.x / H::NP), n(threadIdx.x % H::NP), on(n < N) {
    p = (const Elem<DT> *)s.data + at.b * s.stride_batch + (l0 + k) * s.stride_length + at.g * s.stride_group + (on ? n : 0);
  }
  __device__ inline void load_all() {
#pragma unroll
    for (int i = 0; i < H::NB; ++i)
      if (K * H::NP >= 256 * (i + 1) || k + i * R < K) ahead[i] = p[i * stride];
  }
  __device__ void next() { p += step; }
  __device__ void back() { p -= step; }
  __device__ inline void load(int left) {  // left: positions of the chunk within the row
#pragma unroll
    for (int i = 0; i < H::NB; ++i) {
      ahead[i] = (Elem<DT>)0.f;
      if (k + i * R < (left < K ? left : K)) ahead[i] = p[i * stride];
    }
  }
  __device__ inline void take() {
#pragma unroll
    for (int i = 0; i < H::NB; ++i) v[i] = ahead[i];
  }
  __device__ inline void put(float *to) const {
#pragma unroll
    for (int i = 0; i < H::NB; ++i)
      if (K * H::NP >= 256 * (i + 1) || threadIdx.x + 256 * i < K * H::NP) to[threadIdx.x + 256 * i] = on ? (float)v[i] : 0.f;
  }
};

// decays are computed as 2^(delta A log2 e)
template <int S, int NL>
__device__ inline void decay_rates(float *a2, const afc_scan_args &P, const Place<S, NL> &at) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int n = at.nl * S + s;
    a2[s] = at.cb < at.nw && n < P.state ? rate2(P.a[(at.w0 + at.cb) * P.state + n]) : 0.f;
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

// The S states' operands of four positions, loaded one group of positions ahead of their use
template <int S, int NL, bool WITH_B, bool WITH_C>
struct Operands {
  float2 d[4];
  float B[WITH_B ? 4 : 1][S], C[WITH_C ? 4 : 1][S];
  __device__ inline void load(const float2 (*steps)[Shape<S, NL>::CB], const float *bs, const float *cs, int k4, const Place<S, NL> &at) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      d[k] = steps[k4 + k][at.cb];
      if (WITH_B) load_states<S>(B[k], bs + (k4 + k) * S * NL + at.nl * S);
      if (WITH_C) load_states<S>(C[k], cs + (k4 + k) * S * NL + at.nl * S);
    }
  }
};

// What reaches a part from those on its far side: h starts as what the row begins with, `from` is the part at that end.  (The
// loads of eight parts are in flight together.)
template <int S, int NL>
__device__ inline void take_carries(float *h, const float *a2, const Carry &carry, int from, int parts, int way, const afc_scan_args &P, const Plan &T, const Place<S, NL> &at) {
  if (at.cb >= at.nw) return;
  for (int j0 = 0; j0 < parts; j0 += 8) {
    float e[8][S], d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t row = ((int64_t)at.b * T.segs + from + way * min(j0 + j, parts - 1)) * P.width + at.w0 + at.cb;
      load_states<S>(e[j], carry.state + row * S * NL + at.nl * S);
      d[j] = carry.steps[row];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const float next = __builtin_fmaf(__builtin_amdgcn_exp2f(d[j] * a2[s]), h[s], e[j][s]);
        h[s] = j0 + j < parts ? next : h[s];
      }
  }
}

// ---- forwards ----
// One barrier a chunk.  While the recurrence runs over chunk i, whose step sizes and rows lie in LDS, the same threads work out
// the step sizes of chunk i + 1 (into the other half of LDS), finish the outputs of chunk i - 1 and have the loads of chunk
// i + 2 in flight: the chains of the recurrence leave issue slots that the rest fills, also with a single wave on each SIMD.
// CARRY: only the carries are computed (of all parts but the last)
template <int DT, int S, int NL, bool WHOLE, bool CARRY>
__global__ __launch_bounds__(256) void k_scan(afc_scan_args P, Plan T, Carry carry) {
  typedef Shape<S, NL> H;
  constexpr int E = H::E;
  __shared__ float2 steps[2][K][H::CB];  // delta, delta x
  __shared__ __align__(16) float bs[2][K * H::NP], cs[2][CARRY ? 4 : K * H::NP];
  __shared__ float ys[2][CARRY ? 1 : K][H::CB];
  const Place<S, NL> at(P, T);
  if (CARRY && at.seg == T.segs - 1) return;
  float a2[S], h[S], total = 0.f;
  decay_rates<S, NL>(a2, P, at);
  const int64_t w = at.w0 + at.cb;
  if (CARRY) {
    for (int s = 0; s < S; ++s) h[s] = 0.f;
  } else {
    state_or_zero<S, NL>(h, P.initial_state, P, at);
    take_carries<S, NL>(h, a2, carry, 0, at.seg, 1, P, T, at);
  }
  float bias[E], D[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    bias[i] = P.dt_bias && i < at.n ? P.dt_bias[at.w0 + at.q + i] : 0.f;
    D[i] = P.d && i < at.n ? P.d[at.w0 + at.q + i] : 0.f;
  }
  const int first = at.first_chunk(T), live = at.live_end(T), end = at.end_chunk(T);
  Piece<DT, E, WHOLE> x{}, dt{}, z{}, xa{}, dta{}, za{};  // of the chunk whose step sizes come next, and of the one after it
  const int64_t l0 = (int64_t)first * K, lr = l0 + at.r, wq = at.readable();
  Rows<DT, S, NL> rb(P.b, at, l0, P.state), rc(P.c, at, l0, P.state);
  Stream<DT> xs(P.x, at.b, lr, wq), dts(P.dt, at.b, lr, wq), zs(P.z, at.b, lr, wq), out(P.y, at.b, lr, at.w0 + at.q);
  const bool gate = !CARRY && P.z.data, soft = P.softplus, skip = P.d;
  auto fetch = [&](int ch) {
    if (ch >= live) return;  // (what is there stays, unused)
    if (WHOLE && (ch + 1) * K <= at.len) {
      xa.load_all(xs.p);
      dta.load_all(dts.p);
      if (gate) za.load_all(zs.p);
      rb.load_all();
      if (!CARRY) rc.load_all();
    } else {
      const int n = ch * K + at.r < at.len ? at.n : 0, rows = at.len - ch * K;
      xa.load(xs.p, n);
      dta.load(dts.p, n);
      if (gate) za.load(zs.p, n);
      rb.load(rows);
      if (!CARRY) rc.load(rows);
    }
    xs.next(), dts.next(), zs.next(), rb.next(), rc.next();
  };
  auto take = [&] {
    x = xa, dt = dta, z = za;
    rb.take(), rc.take();
  };
  auto step_of = [&](int i, int ch) {
    const float v = dt[i] + bias[i], soft_v = softplus(v);
    return ch * K + at.r < at.len && i < at.n ? (soft ? soft_v : v) : 0.f;
  };
  float step[E];
  auto put = [&](int half) {
#pragma unroll
    for (int i = 0; i < E; ++i) steps[half][at.r][at.q + i] = make_float2(step[i], i < at.n ? step[i] * x[i] : 0.f);
    rb.put(bs[half]);
    if (!CARRY) rc.put(cs[half]);
  };
  Piece<DT, E, WHOLE> x1{}, z1{}, x2{}, z2{};  // of the chunk in the recurrence, and of the one before it
  float y[E];
  auto finish = [&](int i) {
    const float with_x = __builtin_fmaf(D[i], x2[i], y[i]), v = skip ? with_x : y[i], gated = v * silu(z2[i]);
    y[i] = gate ? gated : v;
  };
  auto put_y = [&](int ch) {
    const int l = ch * K + at.r;
    if (l >= P.length) return;
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] = l < at.len ? y[i] : 0.f;
    store<DT, E, WHOLE>(out.p, y, at.n);
    out.next();
  };
  if (first < live) {
    fetch(first);
    take();
    fetch(first + 1);
#pragma unroll
    for (int i = 0; i < E; ++i) step[i] = step_of(i, first);
    put(0);
    x1 = x, z1 = z;
    take();
    __syncthreads();
  }
  for (int ch = first; ch < live; ++ch) {
    const int half = (ch - first) & 1;
    fetch(ch + 2);
    if (!CARRY && P.checkpoints && at.cb < at.nw) store_states<S>(P.checkpoints + (((int64_t)at.b * T.chunks + ch) * P.width + w) * H::NP + at.nl * S, h);
    if (!CARRY) {
#pragma unroll
      for (int i = 0; i < E; ++i) y[i] = ys[half ^ 1][at.r][at.q + i];
    }
    Operands<S, NL, true, !CARRY> now, ahead;
    ahead.load(steps[half], bs[half], cs[half], 0, at);
#pragma unroll
    for (int k4 = 0; k4 < K; k4 += 4) {
      now = ahead;
      if (k4 + 4 < K) ahead.load(steps[half], bs[half], cs[half], k4 + 4, at);
      float yk[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
          h[s] = __builtin_fmaf(__builtin_amdgcn_exp2f(now.d[k].x * a2[s]), h[s], now.d[k].y * now.B[k][s]);
          if (!CARRY) yk[k] = s ? __builtin_fmaf(now.C[k][s], h[s], yk[k]) : now.C[k][s] * h[s];
        }
        if (CARRY) total += now.d[k].x;
      }
      if (!CARRY) {
        ys[half][k4 + four_at<NL>(at.nl)][at.cb] = sum_four<NL>(yk[0], yk[1], yk[2], yk[3], at.nl);
      }
#pragma unroll
      for (int i = k4 / 4 * E / 4; i < (k4 / 4 + 1) * E / 4; ++i) {
        step[i] = step_of(i, ch + 1);
        if (!CARRY) finish(i);
      }
    }
    put(half ^ 1);
    if (!CARRY && ch > first) put_y(ch - 1);
    x2 = x1, z2 = z1, x1 = x, z1 = z;
    take();
    __syncthreads();
  }
  if (CARRY) {
    if (at.cb < at.nw) {
      store_states<S>(carry.state + (((int64_t)at.b * T.segs + at.seg) * P.width + w) * H::NP + at.nl * S, h);
      if (at.nl == 0) carry.steps[((int64_t)at.b * T.segs + at.seg) * P.width + w] = total;
    }
    return;
  }
  if (first < live) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      y[i] = ys[(live - 1 - first) & 1][at.r][at.q + i];
      finish(i);
    }
    put_y(live - 1);
  }
  for (int ch = live; ch < end; ++ch, out.next()) {
    const float zero[E] = {};
    if (ch * K + at.r < P.length) store<DT, E, WHOLE>(out.p, zero, at.n);
  }
  if (at.seg == T.segs - 1) put_state<S, NL>(P.final_state, h, P, at);
}

// ---- backwards ----
// sums that are finished by k_scan_sums: bc [batch, groups, tiles, length, 2, NP], a [batch, segs, width, NP], d
// and bias [batch, segs, width]; others [batch, width, NP]: see kLastChunk
struct Sums {
  float *bc, *a, *d, *bias, *others;
};

// Behind a row's end the step size is zero, but zero times a state or an adjoint that is not finite is NaN, where dA's formula has no
// term at all.  The chunk in which a row ends is the first one that k_scan_grad takes; if its share of dA is NaN the share is left
// out, the others' sum goes to Sums.others and this NaN to Sums.a, and k_scan_sums takes the share over the row's own positions.
constexpr unsigned kLastChunk = 0x7fc0afc1u;

// What a part hands on to the one before it, from a zero adjoint behind it (of all parts but the first)
template <int DT, int S, int NL, bool WHOLE>
__global__ __launch_bounds__(256) void k_scan_grad_carry(afc_scan_args P, Plan T, Carry carry) {
  typedef Shape<S, NL> H;
  constexpr int E = H::E;
  __shared__ float2 steps[2][K][H::CB];  // delta, dy
  __shared__ __align__(16) float cs[2][K * H::NP];
  const Place<S, NL> at(P, T);
  if (at.seg == 0) return;
  float a2[S], g[S] = {}, total = 0.f;
  decay_rates<S, NL>(a2, P, at);
  const int64_t w = at.w0 + at.cb;
  float bias[E];
#pragma unroll
  for (int i = 0; i < E; ++i) bias[i] = P.dt_bias && i < at.n ? P.dt_bias[at.w0 + at.q + i] : 0.f;
  const int first = at.first_chunk(T), live = at.live_end(T);
  Piece<DT, E, WHOLE> dt{}, z{}, dout{}, dta{}, za{}, douta{};
  const int64_t l0 = (int64_t)(live - 1) * K;
  Rows<DT, S, NL> rc(P.c, at, l0, P.state);
  const int64_t lr = l0 + at.r, wq = at.readable();
  Stream<DT> dts(P.dt, at.b, lr, wq), zs(P.z, at.b, lr, wq), douts(P.dy, at.b, lr, wq);
  const bool gate = P.z.data, soft = P.softplus;
  auto fetch = [&](int ch) {
    if (ch < first) return;
    if (WHOLE && (ch + 1) * K <= at.len) {
      dta.load_all(dts.p);
      if (gate) za.load_all(zs.p);
      douta.load_all(douts.p);
      rc.load_all();
    } else {
      const int n = ch * K + at.r < at.len ? at.n : 0;
      dta.load(dts.p, n);
      if (gate) za.load(zs.p, n);
      douta.load(douts.p, n);
      rc.load(at.len - ch * K);
    }
    dts.back(), zs.back(), douts.back(), rc.back();
  };
  auto take = [&] {
    dt = dta, z = za, dout = douta;
    rc.take();
  };
  float step[E], dy[E];
  auto prepare = [&](int i, int ch) {
    const float v = dt[i] + bias[i], soft_v = softplus(v), d = dout[i], gated = d * silu(z[i]);
    step[i] = ch * K + at.r < at.len && i < at.n ? (soft ? soft_v : v) : 0.f;
    dy[i] = i < at.n ? (gate ? gated : d) : 0.f;
  };
  auto put = [&](int half) {
#pragma unroll
    for (int i = 0; i < E; ++i) steps[half][at.r][at.q + i] = make_float2(step[i], dy[i]);
    rc.put(cs[half]);
  };
  if (first < live) {
    fetch(live - 1);
    take();
    fetch(live - 2);
#pragma unroll
    for (int i = 0; i < E; ++i) prepare(i, live - 1);
    put(0);
    take();
    __syncthreads();
  }
  for (int ch = live - 1; ch >= first; --ch) {
    const int half = (live - 1 - ch) & 1;
    fetch(ch - 2);
    Operands<S, NL, false, true> now, ahead;
    ahead.load(steps[half], nullptr, cs[half], K - 4, at);
#pragma unroll
    for (int k4 = K - 4; k4 >= 0; k4 -= 4) {
      now = ahead;
      if (k4) ahead.load(steps[half], nullptr, cs[half], k4 - 4, at);
#pragma unroll
      for (int k = 3; k >= 0; --k) {
        total += now.d[k].x;
#pragma unroll
        for (int s = 0; s < S; ++s) g[s] = __builtin_amdgcn_exp2f(now.d[k].x * a2[s]) * __builtin_fmaf(now.d[k].y, now.C[k][s], g[s]);
      }
#pragma unroll
      for (int i = k4 / 4 * E / 4; i < (k4 / 4 + 1) * E / 4; ++i) prepare(i, ch - 1);
    }
    put(half ^ 1);
    take();
    __syncthreads();
  }
  if (at.cb < at.nw) {
    store_states<S>(carry.state + (((int64_t)at.b * T.segs + at.seg) * P.width + w) * H::NP + at.nl * S, g);
    if (at.nl == 0) carry.steps[((int64_t)at.b * T.segs + at.seg) * P.width + w] = total;
  }
}

// A chunk is run forwards again from its checkpoint with the states and decays of its K positions in registers (beside it, the
// outputs of the chunk behind it are finished), then backwards (beside it, the chunk in front of it is prepared).
template <int DT, int S, int NL, bool WHOLE>
__global__ __launch_bounds__(256) void k_scan_grad(afc_scan_args P, Plan T, Carry carry, Sums sums) {
  typedef Shape<S, NL> H;
  constexpr int E = H::E, V = 2 * S, SET = H::CPW > V ? H::CPW : V, NO = (K * 2 * H::NP + 255) / 256;
  __shared__ float2 steps[2][K][H::CB];  // delta, delta x
  __shared__ float dys[2][K][H::CB], ys[2][K][H::CB], dus[K][H::CB], tas[K][H::CB];
  __shared__ __align__(16) float bs[2][K * H::NP], cs[2][K * H::NP];
  __shared__ float part[4][K * 2 * H::NP];
  const Place<S, NL> at(P, T);
  float a2[S], g[S];
  decay_rates<S, NL>(a2, P, at);
  const int64_t w = at.w0 + at.cb;
  state_or_zero<S, NL>(g, P.dfinal_state, P, at);
  take_carries<S, NL>(g, a2, carry, T.segs - 1, T.segs - 1 - at.seg, -1, P, T, at);
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
  const bool gate = P.z.data, soft = P.softplus, skip = P.d;  // (without D its terms are left out: zero times an infinite input is NaN)
  Piece<DT, E, WHOLE> x{}, dt{}, z{}, dout{}, xa{}, dta{}, za{}, douta{};  // of the chunk that is prepared next, and of the one in front of it
  const int64_t l0 = (int64_t)(live - 1) * K, lr = l0 + at.r, wq = at.readable(), wo = at.w0 + at.q;
  Rows<DT, S, NL> rb(P.b, at, l0, P.state), rc(P.c, at, l0, P.state);
  Stream<DT> xs(P.x, at.b, lr, wq), dts(P.dt, at.b, lr, wq), zs(P.z, at.b, lr, wq), douts(P.dy, at.b, lr, wq), dxs(P.dx, at.b, lr, wo), ddts(P.ddt, at.b, lr, wo),
      dzs(P.dz, at.b, lr, wo);
  auto fetch = [&](int ch) {
    if (ch < first) return;
    if (WHOLE && (ch + 1) * K <= at.len) {
      xa.load_all(xs.p);
      dta.load_all(dts.p);
      if (gate) za.load_all(zs.p);
      douta.load_all(douts.p);
      rb.load_all();
      rc.load_all();
    } else {
      const int n = ch * K + at.r < at.len ? at.n : 0, rows = at.len - ch * K;
      xa.load(xs.p, n);
      dta.load(dts.p, n);
      if (gate) za.load(zs.p, n);
      douta.load(douts.p, n);
      rb.load(rows);
      rc.load(rows);
    }
    xs.back(), dts.back(), zs.back(), douts.back(), rb.back(), rc.back();
  };
  auto take = [&] {
    x = xa, dt = dta, z = za, dout = douta;
    rb.take(), rc.take();
  };
  float h[S], h0[S];
  bool left_out = false;
  auto fetch_state = [&](int ch) {
#pragma unroll
    for (int s = 0; s < S; ++s) h0[s] = 0.f;
    if (ch >= first && at.cb < at.nw) load_states<S>(h0, P.checkpoints + (((int64_t)at.b * T.chunks + ch) * P.width + w) * H::NP + at.nl * S);
  };
  float step[E], dy[E], sz[E], slope[E];  // sz: sigmoid(z); slope: of the softplus
  auto prepare = [&](int i, int ch) {
    const float v = dt[i] + bias[i], soft_v = softplus(v, slope[i]), d = dout[i];
    sz[i] = sigmoid(z[i]);
    const float gated = d * z[i] * sz[i];
    step[i] = ch * K + at.r < at.len && i < at.n ? (soft ? soft_v : v) : 0.f;
    dy[i] = i < at.n ? (gate ? gated : d) : 0.f;
  };
  auto put = [&](int half) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      steps[half][at.r][at.q + i] = make_float2(step[i], i < at.n ? step[i] * x[i] : 0.f);
      dys[half][at.r][at.q + i] = dy[i];
    }
    rb.put(bs[half]);
    rc.put(cs[half]);
  };
  // the chunk in the recurrence, and the one behind it
  struct Kept {
    Piece<DT, E, WHOLE> x, z, dout;
    float step[E], dy[E], sz[E], slope[E];
  } k1{}, k2{};
  auto keep = [&] {
    k2 = k1;
    k1.x = x, k1.z = z, k1.dout = dout;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      k1.step[i] = step[i], k1.dy[i] = dy[i], k1.sz[i] = sz[i], k1.slope[i] = slope[i];
    }
  };
  float dx[E], ddt[E], dz[E], bc[NO];
  auto finish = [&](int i, int half) {
    const float du = dus[at.r][at.q + i], ta = tas[at.r][at.q + i], y = ys[half][at.r][at.q + i], xi = k2.x[i], zi = k2.z[i];
    const float d = __builtin_fmaf(du, xi, ta * 0.693147180559945309f);
    dx[i] = __builtin_fmaf(du, k2.step[i], skip ? D[i] * k2.dy[i] : 0.f);
    ddt[i] = soft ? k2.slope[i] * d : d;
    const float with_x = __builtin_fmaf(D[i], xi, y);
    dz[i] = k2.dout[i] * (skip ? with_x : y) * silu_slope(zi, k2.sz[i]);
  };
  auto finish_bc = [&] {
#pragma unroll
    for (int j = 0; j < NO; ++j) {
      const int i = threadIdx.x + 256 * j;
      bc[j] = K * 2 * H::NP >= 256 * (j + 1) || i < K * 2 * H::NP ? (part[0][i] + part[1][i]) + (part[2][i] + part[3][i]) : 0.f;
    }
  };
  const int length = (int)P.length;
  float *const bc_rows = sums.bc + (((int64_t)at.b * P.groups + at.g) * T.tiles + at.tile) * P.length * 2 * H::NP + threadIdx.x;
  float *bc_to = bc_rows + (int64_t)(live - 1) * K * 2 * H::NP;
  const bool gate_grad = P.dz.data;
  auto put_grads = [&](int ch) {
    const int l = ch * K + at.r;
    if ((ch + 1) * K > at.len) {  // the row ends here: what lies behind it is zero
#pragma unroll
      for (int j = 0; j < NO; ++j) bc[j] = ch * K + (int)(threadIdx.x + 256 * j) / (2 * H::NP) < at.len ? bc[j] : 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        dx[i] = l < at.len ? dx[i] : 0.f;
        ddt[i] = l < at.len ? ddt[i] : 0.f;
        dz[i] = l < at.len ? dz[i] : 0.f;
      }
    }
    const int left = length - ch * K;  // positions that the tensors have
#pragma unroll
    for (int j = 0; j < NO; ++j)
      if ((int)threadIdx.x + 256 * j < (left < K ? left : K) * 2 * H::NP) bc_to[256 * j] = bc[j];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      sum_d[i] = __builtin_fmaf(k2.dy[i], i < at.n ? k2.x[i] : 0.f, sum_d[i]);
      sum_b[i] += ddt[i];
    }
    const int n = at.r < left ? at.n : 0;
    store<DT, E, WHOLE>(dxs.p, dx, n);
    store<DT, E, WHOLE>(ddts.p, ddt, n);
    if (gate_grad) store<DT, E, WHOLE>(dzs.p, dz, n);
    dxs.back(), ddts.back(), dzs.back();
    bc_to -= K * 2 * H::NP;
  };
  {  // behind the row's end
    const float zero[E] = {};
    for (int ch = live; ch < end; ++ch) {
      dxs.next(), ddts.next(), dzs.next();
      if (ch * K + at.r < P.length) {
        store<DT, E, WHOLE>(dxs.p, zero, at.n);
        store<DT, E, WHOLE>(ddts.p, zero, at.n);
        if (gate_grad) store<DT, E, WHOLE>(dzs.p, zero, at.n);
      }
      for (int i = threadIdx.x; i < K * 2 * H::NP; i += 256)
        if (ch * K + i / (2 * H::NP) < length) bc_rows[(int64_t)ch * K * 2 * H::NP + i - threadIdx.x] = 0.f;
    }
    for (int ch = live; ch < end; ++ch) dxs.back(), ddts.back(), dzs.back();
  }
  if (first < live) {
    fetch(live - 1);
    fetch_state(live - 1);
    take();
    fetch(live - 2);
#pragma unroll
    for (int i = 0; i < E; ++i) prepare(i, live - 1);
    put(0);
    keep();
    take();
    __syncthreads();
  }
  for (int ch = live - 1; ch >= first; --ch) {
    const int half = (live - 1 - ch) & 1;
#pragma unroll
    for (int s = 0; s < S; ++s) h[s] = h0[s];
    fetch_state(ch - 1);
    fetch(ch - 2);
    float before[K][S], a[K][S];
    Operands<S, NL, true, true> now, ahead;
    ahead.load(steps[half], bs[half], cs[half], 0, at);
    finish_bc();
#pragma unroll
    for (int k4 = 0; k4 < K; k4 += 4) {
      now = ahead;
      if (k4 + 4 < K) ahead.load(steps[half], bs[half], cs[half], k4 + 4, at);
      float y[4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int k = k4 + kk;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          before[k][s] = h[s];
          a[k][s] = __builtin_amdgcn_exp2f(now.d[kk].x * a2[s]);
          h[s] = __builtin_fmaf(a[k][s], h[s], now.d[kk].y * now.B[kk][s]);
          y[kk] = s ? __builtin_fmaf(now.C[kk][s], h[s], y[kk]) : now.C[kk][s] * h[s];
        }
      }
      ys[half][k4 + four_at<NL>(at.nl)][at.cb] = sum_four<NL>(y[0], y[1], y[2], y[3], at.nl);
#pragma unroll
      for (int i = k4 / 4 * E / 4; i < (k4 / 4 + 1) * E / 4; ++i) finish(i, half ^ 1);
    }
    if (ch < live - 1) put_grads(ch + 1);
    __syncthreads();
    float v[SET];
    ahead.load(steps[half], bs[half], cs[half], K - 4, at);
#pragma unroll
    for (int k4 = K - 4; k4 >= 0; k4 -= 4) {
      now = ahead;
      if (k4) ahead.load(steps[half], bs[half], cs[half], k4 - 4, at);
      float du[4], ta[4];
#pragma unroll
      for (int kk = 3; kk >= 0; --kk) {
        const int k = k4 + kk;
        const float dyk = dys[half][k][at.cb];
        const int o = (K - 1 - k) * V % SET;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          g[s] = __builtin_fmaf(dyk, now.C[kk][s], g[s]);
          v[o + s] = g[s] * now.d[kk].y;
          v[o + S + s] = dyk * (k == K - 1 ? h[s] : before[k < K - 1 ? k + 1 : k][s]);
          du[kk] = s ? __builtin_fmaf(g[s], now.B[kk][s], du[kk]) : g[s] * now.B[kk][s];
          g[s] *= a[k][s];
          const float t = g[s] * before[k][s];
          sum_a[s] = __builtin_fmaf(t, now.d[kk].x, sum_a[s]);
          ta[kk] = s ? __builtin_fmaf(t, a2[s], ta[kk]) : t * a2[s];
        }
        // the set of CPW values that is complete: value i belongs to position K - 1 - i / V of the chunk
        if (o + V >= H::CPW) {
#pragma unroll
          for (int m = 0; m < SET; m += H::CPW) {
            const int i = (K - 1 - k) * V + V - SET + m + at.c;
            const float sum = sum_channels<NL>(v + m, at.lane);
            part[at.wave][(K - 1 - i / V) * 2 * H::NP + (i % V / S) * H::NP + at.nl * S + i % S] = sum;
          }
        }
      }
      dus[k4 + four_at<NL>(at.nl)][at.cb] = sum_four<NL>(du[0], du[1], du[2], du[3], at.nl);
      tas[k4 + four_at<NL>(at.nl)][at.cb] = sum_four<NL>(ta[0], ta[1], ta[2], ta[3], at.nl);
#pragma unroll
      for (int i = k4 / 4 * E / 4; i < (k4 / 4 + 1) * E / 4; ++i) prepare(i, ch - 1);
    }
    if ((ch + 1) * K > at.len) {
#pragma unroll
      for (int s = 0; s < S; ++s) left_out |= sum_a[s] != sum_a[s];
#pragma unroll
      for (int s = 0; s < S; ++s) sum_a[s] = left_out ? 0.f : sum_a[s];
    }
    put(half ^ 1);
    keep();
    take();
    __syncthreads();
  }
  if (first < live) {
#pragma unroll
    for (int i = 0; i < E; ++i) finish(i, (live - 1 - first) & 1);
    finish_bc();
    put_grads(first);
  }
  const int64_t row = (int64_t)at.b * T.segs + at.seg;
  if (left_out && at.cb < at.nw) {
    store_states<S>(sums.others + ((int64_t)at.b * P.width + w) * H::NP + at.nl * S, sum_a);
#pragma unroll
    for (int s = 0; s < S; ++s) sum_a[s] = __builtin_bit_cast(float, kLastChunk);
  }
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

// A row's last chunk's share of dA for one state of one channel, over the row's own positions alone, one after the other, each with the
// state in front of it from the checkpoint on (only where k_scan_grad has left it out: nothing here is fast).
template <int DT>
__device__ inline float last_share(const afc_scan_args &P, const Plan &T, int NP, int64_t b, int64_t w, int n) {
  typedef Elem<DT> E;
  const int len = row_length(P.lengths, b, P.length), chunk = (len - 1) / K, l0 = chunk * K;
  const int64_t g = w / (P.width / P.groups), state = (b * P.width + w) * P.state + n;
  const float a2 = rate2(P.a[w * P.state + n]), bias = P.dt_bias ? P.dt_bias[w] : 0.f;
  auto of = [&](const afc_seq &s, int l, int64_t i) { return (float)((const E *)s.data)[b * s.stride_batch + l * s.stride_length + i]; };
  auto step = [&](int l) {
    const float v = of(P.dt, l, w) + bias;
    return P.softplus ? softplus(v) : v;
  };
  float adjoint = P.dfinal_state ? P.dfinal_state[state] : 0.f, sum = 0.f;
#pragma unroll 1
  for (int l = len - 1; l >= l0; --l) {
    float h = P.checkpoints[((b * T.chunks + chunk) * P.width + w) * NP + n];
#pragma unroll 1
    for (int j = l0; j < l; ++j) {
      const float delta = step(j);
      h = __builtin_fmaf(__builtin_amdgcn_exp2f(delta * a2), h, delta * of(P.x, j, w) * of(P.b, j, g * P.b.stride_group + n));
    }
    const float delta = step(l), dout = of(P.dy, l, w), dy = P.z.data ? dout * silu(of(P.z, l, w)) : dout;
    adjoint = __builtin_amdgcn_exp2f(delta * a2) * __builtin_fmaf(dy, of(P.c, l, g * P.c.stride_group + n), adjoint);
    sum = __builtin_fmaf(adjoint * h, delta, sum);
  }
  return sum;
}

// The sums that the blocks of k_scan_grad leave, in one launch (two cost 1 to 4 us more: 8 x 64 x 256 both ways
// 28.9 against 27.8, 1 x 8191 x 512 164 against 160), in blocks of 1024.
// The first bc_blocks: db and dc, sums over a group's tiles, one thread for each value.  The others: da, dd and ddt_bias, sums
// over rows and parts, 64 columns a block.
template <int DT>
__global__ __launch_bounds__(1024) void k_scan_sums(afc_scan_args P, Plan T, Sums sums, int NP, int64_t bc_blocks) {
  typedef Elem<DT> E;
  __shared__ float red[1024];
  const int64_t block = T.base + blockIdx.x;
  if (block < bc_blocks) {
    const int64_t i = block * 1024 + threadIdx.x, per = 2 * NP;
    if (i >= P.batch * P.groups * P.length * per) return;
    const int64_t row = i / (P.length * per), l = i / per % P.length, b = row / P.groups, g = row % P.groups;
    const int n = (int)(i % NP), c = (int)(i % per) / NP;
    if (n >= P.state) return;
    const float *from = sums.bc + (row * T.tiles * P.length + l) * per + c * NP + n;
    float a = 0.f;
#pragma unroll 8
    for (int t = 0; t < T.tiles; ++t) a += from[t * P.length * per];
    const afc_seq &s = c ? P.dc : P.db;
    ((E *)s.data)[b * s.stride_batch + l * s.stride_length + g * s.stride_group + n] = (E)a;
    return;
  }
  const int64_t rows = P.batch * T.segs, na = P.width * NP, col = (block - bc_blocks) * 64 + (threadIdx.x & 63);
  const int which = col < na ? 0 : col < na + P.width ? 1 : 2;
  const int64_t at = which == 0 ? col : col - na - (which - 1) * P.width, cols = which == 0 ? na : P.width;
  const float *from = which == 0 ? sums.a : which == 1 ? sums.d : sums.bias;
  float a = column_sum(from, rows, cols, at, red);
  if (threadIdx.x >= 64 || at >= cols) return;
  if (which == 0) {
    const int n = (int)(at % NP);
    if (!P.da || n >= P.state) return;
    if (a != a) {
      a = 0.f;
      for (int64_t r = 0; r < rows; ++r) {
        const float v = from[r * cols + at];
        const int64_t b = r / T.segs;
        a += __builtin_bit_cast(unsigned, v) == kLastChunk ? sums.others[b * cols + at] + last_share<DT>(P, T, NP, b, at / NP, n) : v;
      }
    }
    P.da[at / NP * P.state + n] = a;
  } else if (which == 1) {
    if (P.dd) P.dd[at] = a;
  } else if (P.ddt_bias) {
    P.ddt_bias[at] = a;
  }
}

// ---- single tokens ----
// Reading and writing the state is what bounds them.  Where `state` is a multiple of four a lane has four states (16 bytes) of a
// channel, NL lanes a channel, side by side as in memory, and R rows of the batch, whose loads are all in flight before the
// first is used; the channel's parameters are read once for them.
template <int NL>
__device__ inline float sum_side(float v) {
  if (NL > 1) v += dpp<kXor1>(v);
  if (NL > 2) v += dpp<kXor2>(v);
  if (NL > 4) v += dpp<0x141>(v);  // mirrored halves of eight: all four lanes of the other half hold its sum
  if (NL > 8) v += dpp<0x140>(v);  // mirrored sixteen
  return v;
}

template <int DT, int NL, int R>
__global__ __launch_bounds__(256) void k_scan_step4(afc_scan_args P, int tiles, unsigned base) {
  typedef Elem<DT> E;
  typedef float F4 __attribute__((ext_vector_type(4)));
  const unsigned block = base + blockIdx.x;
  const int tile = block % tiles;
  const int64_t b0 = (int64_t)(block / tiles) * R, w = (int64_t)tile * (256 / NL) + threadIdx.x / NL;
  const int n = threadIdx.x % NL * 4, rows = (int)min((int64_t)R, P.batch - b0);
  if (w >= P.width) return;
  const bool on = n < P.state;  // (a lane without states holds zeros: it takes part in the sums)
  const int64_t g = (unsigned)w / (unsigned)(P.width / P.groups), st = (b0 * P.width + w) * P.state + n, row = P.width * P.state;
  F4 h[R];
  typedef E E4 __attribute__((ext_vector_type(4), aligned(sizeof(E))));  // (from any place: B and C may be slices)
  E x[R], dt[R], z[R];
  E4 B[R], C[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rows) continue;
    const int64_t b = b0 + r;
    h[r] = (F4)0.f;
    if (on) h[r] = *reinterpret_cast<const F4 *>(P.final_state + st + r * row);
    x[r] = ((const E *)P.x.data)[b * P.x.stride_batch + w];
    dt[r] = ((const E *)P.dt.data)[b * P.dt.stride_batch + w];
    if (P.z.data) z[r] = ((const E *)P.z.data)[b * P.z.stride_batch + w];
    B[r] = C[r] = (E4)(E)0.f;
    if (on) {
      B[r] = *reinterpret_cast<const E4 *>((const E *)P.b.data + b * P.b.stride_batch + g * P.b.stride_group + n);
      C[r] = *reinterpret_cast<const E4 *>((const E *)P.c.data + b * P.c.stride_batch + g * P.c.stride_group + n);
    }
  }
  F4 a2 = (F4)0.f;
  if (on) a2 = *reinterpret_cast<const F4 *>(P.a + w * P.state + n);
#pragma unroll
  for (int i = 0; i < 4; ++i) a2[i] = rate2(a2[i]);
  const float bias = P.dt_bias ? P.dt_bias[w] : 0.f, D = P.d ? P.d[w] : 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rows) continue;
    const float v = (float)dt[r] + bias, xr = (float)x[r], delta = P.softplus ? softplus(v) : v, u = delta * xr;
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[r][i] = __builtin_fmaf(__builtin_amdgcn_exp2f(delta * a2[i]), h[r][i], u * (float)B[r][i]);
      y = __builtin_fmaf((float)C[r][i], h[r][i], y);
    }
    if (on) *reinterpret_cast<F4 *>(P.final_state + st + r * row) = h[r];
    y = sum_side<NL>(y);
    if (P.d) y = __builtin_fmaf(D, xr, y);
    if (P.z.data) y *= silu((float)z[r]);
    if (n == 0) ((E *)P.y.data)[(b0 + r) * P.y.stride_batch + w] = (E)y;
  }
}

// Any other state: one lane for each, in NP lanes (a power of two, lanes behind `state` hold zeros), 64 / NP channels in a wave.
template <int NP>
__device__ inline float sum_lanes(float v) {
  for (int m = 1; m < NP; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

template <int DT, int NP>
__global__ __launch_bounds__(64) void k_scan_step(afc_scan_args P, unsigned base) {
  typedef Elem<DT> E;
  const int n = threadIdx.x & (NP - 1);
  const int64_t tiles = (P.width + 64 / NP - 1) / (64 / NP), block = base + blockIdx.x;
  const int64_t b = block / tiles, w = (block % tiles) * (64 / NP) + threadIdx.x / NP;
  const bool on = w < P.width, mine = on && n < P.state;
  const int64_t g = on ? w / (P.width / P.groups) : 0, st = (b * P.width + w) * P.state + n;
  const float x = on ? (float)((const E *)P.x.data)[b * P.x.stride_batch + w] : 0.f;
  const float v = on ? (float)((const E *)P.dt.data)[b * P.dt.stride_batch + w] + (P.dt_bias ? P.dt_bias[w] : 0.f) : 0.f;
  const float delta = P.softplus ? softplus(v) : v;
  float h = 0.f, yc = 0.f;
  if (mine) {
    const float B = (float)((const E *)P.b.data)[b * P.b.stride_batch + g * P.b.stride_group + n];
    const float C = (float)((const E *)P.c.data)[b * P.c.stride_batch + g * P.c.stride_group + n];
    h = __builtin_fmaf(__builtin_amdgcn_exp2f(delta * rate2(P.a[w * P.state + n])), P.final_state[st], delta * x * B);
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
  check_axes(p->batch, p->length, p->width);
  want(p->groups >= 1 && p->width % p->groups == 0, "groups must divide width");
}

void check(const afc_scan_args *p, bool grad, bool step) {
  check_sizes(p);
  want(p->a != nullptr, "a is missing");
  if (step) want(p->length == 1 && !p->lengths && (p->final_state || p->batch == 0) && p->final_state == p->initial_state, "a step takes length 1, no lengths, and its state as initial_state and final_state");
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
    want(!p->dz.data || p->z.data, "dz without z");
    if (p->dz.data) check_seq(p->dz, p->batch, p->length, 0, "dz");
    want(p->checkpoints != nullptr, "checkpoints are missing");
  }
}

// States of a lane and lanes of a channel.  Few states a lane leave registers for two and more waves on a SIMD and make more of
// them: a state of 16 in 8 lanes of 2, 4 of 4 and 16 of 1 takes 762, 840 and 962 us at 8 x 2048 x 2048 bf16 forwards and backwards.
// (At 8 x 64 x 256 f32 the kernels take 30, 40 and 25 us, of a call of 100.)
struct Split {
  int s, nl;
};
Split split(const afc_scan_args *p) {
  const int n = p->state;
  const int64_t wg = p->width / p->groups;
  // groups of few channels: more lanes a channel instead of idle ones (37 x 7197 x 7, four groups, state 1: 193 us against 324)
  if (n <= 16 && wg <= 16) return Split{1, 16};
  if (n <= 8 && wg <= 32) return Split{1, 8};
  return n <= 4 ? Split{1, 4} : n <= 8 ? Split{1, 8} : n <= 16 ? Split{2, 8} : n <= 32 ? Split{2, 16} : Split{4, 16};
}
int padded(const afc_scan_args *p) { return split(p).s * split(p).nl; }

Plan plan(const afc_scan_args *p, bool grad) {
  Plan t;
  const int cb = 256 / split(p).nl;
  t.tiles = (int)ceil_div(p->width / p->groups, cb);
  t.chunks = (int)ceil_div(p->length, K);
  const int64_t blocks = p->batch * p->groups * t.tiles;
  // Parts run at the same time, and cost a pass of their own for the carries.  Their number is what an estimate likes best, in us:
  // a chunk of each of n blocks on a CU takes 0.45 + 0.65 n (up to four at once), backwards 1.8 + 1.5 n (two, or one with four
  // states a lane, whose registers fill a SIMD); the carries add two thirds of the forward pass and a quarter of the backward one,
  // 5 and 7 for another launch and start, and 0.2 for each part that the last one has to take up.
  //   1 x 8191 x 2048 (64 blocks) forwards: 578 us whole, 182 in 8 parts, 160 in 16 and in 32
  //   1 x 8191 x 32 (1 block) forwards: 41 us in 256 parts, 29 in 64 and in 128
  //   1 x 1000 x 1024 (32 blocks) both ways: 112 us in 4 parts, 70 in 8, 60 in 16
  //   8 x 128 x 256 (64 blocks) both ways: 43 us whole, 41 in 2 parts, 31 in 4
  //   8 x 128 x 700 (176 blocks) both ways: 48 us whole, 57 in 2 parts
  //   3 x 900 x 1500 (141 blocks) both ways: 239 us whole, 197 in 8 and 4 parts
  //   4 x 4096 x 2048 (256 blocks) both ways: 1116 us whole, 1033 with two parts backwards
  // All of these have a state of 16; other states go by the same constants, untimed.  (Their kernels' registers admit three blocks on a
  // CU in some forms where four, or two backwards, are taken here.)
  const int64_t most = grad ? 512 : 1024, resident = !grad ? 4 : split(p).s == 4 ? 1 : 2;
  const auto chunk = [&](int64_t n) { return n == 0 ? 0. : grad ? 1.8 + 1.5 * (double)n : 0.45 + 0.65 * (double)n; };
  const auto estimate = [&](int64_t segs) {
    const int64_t n = ceil_div(blocks * segs, 256);
    const double whole = (double)ceil_div(t.chunks, segs) * ((double)(n / resident) * chunk(resident) + chunk(n % resident));
    return segs == 1 ? whole : (grad ? whole * 1.25 + 7 : whole * 1.67 + 5) + 0.2 * (double)segs;
  };
  int64_t segs = 1;
  for (int64_t s = 2; blocks * (s / 2) < most && t.chunks / s >= 2; s *= 2)
    if (estimate(s) < estimate(segs)) segs = s;
  t.seg_chunks = (int)ceil_div(t.chunks > 0 ? t.chunks : 1, segs);
  t.segs = (int)ceil_div(t.chunks > 0 ? t.chunks : 1, t.seg_chunks);
  want(blocks * t.segs < kMostBlocks, "too many blocks");
  t.base = 0;
  return t;
}

#define SCAN_SHAPE(DT, WHOLE, C)                 \
  switch (split(p).s * 100 + split(p).nl) {      \
    case 104: SCAN_GO(DT, 1, 4, WHOLE, C); break;  \
    case 108: SCAN_GO(DT, 1, 8, WHOLE, C); break;  \
    case 116: SCAN_GO(DT, 1, 16, true, C); break;  \
    case 208: SCAN_GO(DT, 2, 8, WHOLE, C); break;  \
    case 216: SCAN_GO(DT, 2, 16, true, C); break;  \
    default: SCAN_GO(DT, 4, 16, true, C); break;   \
  }
#define SCAN_WHOLE(DT, C)                                        \
  if (p->width / p->groups % (16 / split(p).nl) == 0) {          \
    SCAN_SHAPE(DT, true, C)                                      \
  } else {                                                       \
    SCAN_SHAPE(DT, false, C)                                     \
  }
#define SCAN_ALL(C)                  \
  if (p->dtype == AFC_F32) {         \
    SCAN_WHOLE(AFC_F32, C)           \
  } else if (p->dtype == AFC_BF16) { \
    SCAN_WHOLE(AFC_BF16, C)          \
  } else {                           \
    SCAN_WHOLE(AFC_F16, C)           \
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

template <class F>
void slices(const afc_scan_args *p, const Plan &t, const char *what, F &&launch) {
  in_slices(p->batch * p->groups * t.tiles * t.segs, 256, what, [&](int64_t base, dim3 grid) {
    Plan s = t;
    s.base = (unsigned)base;
    launch(s, grid);
  });
}

void scan(const afc_scan_args *p, hipStream_t st) {
  check(p, false, false);
  const Plan t = plan(p, false);
  if (p->batch > 0) check_workspace(p, carry_bytes(p, t));
  want((uintptr_t)p->checkpoints % 16 == 0, "checkpoints must be 16-byte aligned");
  OnDevice on(p->device);
  if (p->batch == 0) return;
  const Carry carry = carry_at(p, t);
#define SCAN_GO(DT, S, NL, WHOLE, C) k_scan<DT, S, NL, WHOLE, C><<<grid, 256, 0, st>>>(*p, s, carry)
  if (t.segs > 1) slices(p, t, "k_scan (carry)", [&](const Plan &s, dim3 grid) { SCAN_ALL(true) });
  slices(p, t, "k_scan", [&](const Plan &s, dim3 grid) { SCAN_ALL(false) });
#undef SCAN_GO
}

// the workspace of the gradients, one part after the other
struct Layout {
  uint64_t carry, bc, a, d, bias, others, all;
};
Layout layout(const afc_scan_args *p, const Plan &t) {
  Layout o;
  const uint64_t rows = (uint64_t)p->batch * t.segs * p->width * 4;
  o.carry = 0;
  o.bc = carry_bytes(p, t);
  o.a = o.bc + up256((uint64_t)p->batch * p->groups * t.tiles * p->length * 2 * padded(p) * 4);
  o.d = o.a + up256(rows * padded(p));
  o.bias = o.d + up256(rows);
  o.others = o.bias + up256(rows);
  o.all = o.others + up256((uint64_t)p->batch * p->width * padded(p) * 4);
  return o;
}

void scan_grad(const afc_scan_args *p, hipStream_t st) {
  check(p, true, false);
  const Plan t = plan(p, true);
  const Layout o = layout(p, t);
  const int64_t bc = ceil_div(p->batch * p->length * p->groups * 2 * padded(p), 1024);
  want(bc < kMostBlocks, "too many blocks");
  if (p->batch > 0) check_workspace(p, o.all);
  want((uintptr_t)p->checkpoints % 16 == 0, "checkpoints must be 16-byte aligned");
  OnDevice on(p->device);
  char *ws = (char *)p->workspace;
  const Carry carry = carry_at(p, t);
  const Sums sums = {(float *)(ws + o.bc), (float *)(ws + o.a), (float *)(ws + o.d), (float *)(ws + o.bias), (float *)(ws + o.others)};
#define SCAN_GO(DT, S, NL, WHOLE, C) k_scan_grad_carry<DT, S, NL, WHOLE><<<grid, 256, 0, st>>>(*p, s, carry)
  if (t.segs > 1) slices(p, t, "k_scan_grad_carry", [&](const Plan &s, dim3 grid) { SCAN_ALL(0) });
#undef SCAN_GO
#define SCAN_GO(DT, S, NL, WHOLE, C) k_scan_grad<DT, S, NL, WHOLE><<<grid, 256, 0, st>>>(*p, s, carry, sums)
  slices(p, t, "k_scan_grad", [&](const Plan &s, dim3 grid) { SCAN_ALL(0) });
#undef SCAN_GO
  const int64_t params = p->da || p->dd || p->ddt_bias ? ceil_div(p->width * (padded(p) + 2), 64) : 0;
  in_slices(bc + params, 1024, "k_scan_sums", [&](int64_t base, dim3 grid) {
    Plan s = t;
    s.base = (unsigned)base;
    if (p->dtype == AFC_F32) k_scan_sums<AFC_F32><<<grid, 1024, 0, st>>>(*p, s, sums, padded(p), bc);
    if (p->dtype == AFC_BF16) k_scan_sums<AFC_BF16><<<grid, 1024, 0, st>>>(*p, s, sums, padded(p), bc);
    if (p->dtype == AFC_F16) k_scan_sums<AFC_F16><<<grid, 1024, 0, st>>>(*p, s, sums, padded(p), bc);
  });
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

template <int DT, int NL>
void go_step4(const afc_scan_args *p, hipStream_t st) {
  const int64_t tiles = ceil_div(p->width, 256 / NL);
  // four rows a thread where that leaves four blocks for every CU: 131 x 4096 x 16 bf16 takes 15.0 us with four and 16.6 with
  // one, 1024 x 256 x 16 f32 8.5 and 8.7; below, one row keeps the chip busier
  const int rows = tiles * p->batch >= 4096 ? 4 : 1;
  const int64_t n = tiles * ceil_div(p->batch, rows);
  want(n < kMostBlocks, "too many blocks");
  OnDevice on(p->device);
  in_slices(n, 256, "k_scan_step4", [&](int64_t base, dim3 grid) {
    if (rows == 4)
      k_scan_step4<DT, NL, 4><<<grid, 256, 0, st>>>(*p, (int)tiles, (unsigned)base);
    else
      k_scan_step4<DT, NL, 1><<<grid, 256, 0, st>>>(*p, (int)tiles, (unsigned)base);
  });
}
void step4(const afc_scan_args *p, hipStream_t st) {
#define STEP4(DT)                                                          \
  p->state <= 4 ? go_step4<DT, 1>(p, st) : p->state <= 8 ? go_step4<DT, 2>(p, st) : p->state <= 16 ? go_step4<DT, 4>(p, st) : \
  p->state <= 32 ? go_step4<DT, 8>(p, st) : go_step4<DT, 16>(p, st)
  if (p->dtype == AFC_F32) STEP4(AFC_F32);
  if (p->dtype == AFC_BF16) STEP4(AFC_BF16);
  if (p->dtype == AFC_F16) STEP4(AFC_F16);
}

void scan_step(const afc_scan_args *p, hipStream_t st) {
  check(p, false, true);
  if (p->state % 4 == 0 && (uintptr_t)p->final_state % 16 == 0 && (uintptr_t)p->a % 16 == 0) return step4(p, st);
  const int64_t n = p->batch * ceil_div(p->width, 64 / lanes(p));
  want(n < kMostBlocks, "too many blocks");
  OnDevice on(p->device);
  in_slices(n, 64, "k_scan_step", [&](int64_t base, dim3 grid) {
#define STEP_GO(DT, NP) k_scan_step<DT, NP><<<grid, 64, 0, st>>>(*p, (unsigned)base)
    if (p->dtype == AFC_F32) STEP_STATE(AFC_F32)
    if (p->dtype == AFC_BF16) STEP_STATE(AFC_BF16)
    if (p->dtype == AFC_F16) STEP_STATE(AFC_F16)
#undef STEP_GO
  });
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
    const Plan t = plan(args, false), g = plan(args, true);
    *checkpoint_bytes = up256((uint64_t)args->batch * t.chunks * args->width * padded(args) * 4);
    *scan_bytes = carry_bytes(args, t);
    *grad_bytes = layout(args, g).all;
  });
}
}
