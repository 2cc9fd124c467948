// Linear attention with a decay: the first-order recurrence on a matrix state,
//   S[t] = exp(g[t]) S[t-1] + y[t] z[t]^T,   o[t] = po * x[t]^T S[t]      (g: logarithm of the decay)
// in chunks of C tokens.  With G the running sum of g inside a chunk, E = G[C-1], S the state entering it:
//   o[t]  = po * ( pz * sum_{s<=t} exp(G[t]-G[s]) (x[t].y[s]) z[s]  +  exp(G[t]) x[t]^T S )
//   S'    = exp(E) S + pz * sum_s exp(E-G[s]) y[s] z[s]^T
// The mirrored form (time reversed; the adjoint state entering from the right) exchanges the two row
// weights: the entering state is read with exp(E-G[t]) and tokens join with exp(G[s]).  Every product of
// the operator is one such pass with its operands exchanged:
//   o:  x=q,  y=k,  z=v              dq: x=do, y=v,  z=k   (state: the transpose of S)
//   dk: x=v,  y=do, z=q  mirrored    dv: x=k,  y=q,  z=do  mirrored
// so the backward pass is one launch with the three of them side by side (they share their reads in L2).
//
// Weights are exponentials of DIFFERENCES of sums held in double (in two doubles for float64), never ratios of exponentials: a
// decay of zero (g = -inf, taken as -1e5) or a long row does not overflow or cancel.
#pragma once
#include "launch.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace ptb {

constexpr int kLaMaxDim = 128;       // largest Dk and Dv
constexpr double kLaMinLog = -1e5;   // stands for a decay of zero (exp of it is 0 in double)

struct LaLengths {
  const void* p;   // may be NULL: every sequence has T tokens
  int wide;        // int64, else int32
};

// one pass; x: (B,T,H,M), y: (B,T,H,M), z: (B,T,H,N), o: dense (B,T,H,N); strides in elements (b, t, h)
template <class S>
struct LaPass {
  const void *x, *y, *z, *w;
  int64_t xs[3], ys[3], zs[3], ws[3];
  void* o;
  const S* init;    // entering state per (b,h), NULL: zero; (M,N), or (N,M) when state_t
  S* fin;           // leaving state, may be NULL; laid out like init
  S* bounds;        // may be NULL: the state entering every chunk, [bh][chunk][M][N]
  S* dots;          // may be NULL: per token w[t].o[t] of the part inside the chunk and of the entering state,
                    //   [slice][bh][t][2]
  int M, N, state_t, reverse;
  int out, pitch;   // tcgen05 kernels: which result o is, and its elements from row to row (a multiple of 8)
  int wide;         // o holds float32 beside a 2-byte type (for a normalisation that follows)
  S po, pz;
};

template <class S>
struct LaArgs {
  LaPass<S> p[3];
  const S* g;
  int64_t gs[3];
  LaLengths lengths;        // per b, clamped to 0..T
  int64_t B, T, H;
  int nseg, seg_chunks;     // the time axis is cut into nseg segments of seg_chunks chunks
  S* seg;                   // [role][segment][bh][M*N] entering states of segments (first in pass order unused)
  double* seg_log;          // [role][segment][bh] log decay over the segment
  int64_t seg_stride;       // elements between two states of `seg`
};

__device__ __forceinline__ float la_exp(float v) { return expf(v); }
__device__ __forceinline__ double la_exp(double v) { return exp(v); }

template <class S, class T> __device__ __forceinline__ S la_load(const T* p) { return (S)*p; }
template <> __device__ __forceinline__ float la_load<float, __half>(const __half* p) { return __half2float(*p); }
template <> __device__ __forceinline__ float la_load<float, __nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <class T, class S> __device__ __forceinline__ void la_store(T* p, S v) { *p = (T)v; }
template <> __device__ __forceinline__ void la_store<__half, float>(__half* p, float v) { *p = __float2half_rn(v); }
template <> __device__ __forceinline__ void la_store<__nv_bfloat16, float>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ int64_t la_length(const LaLengths& lengths, int64_t b, int64_t T) {
  if (!lengths.p) return T;
  const int64_t n = lengths.wide ? static_cast<const int64_t*>(lengths.p)[b] : static_cast<const int32_t*>(lengths.p)[b];
  return n < 0 ? 0 : (n > T ? T : n);
}

// one log decay as the kernels use it (NaN stays NaN)
template <class S>
__device__ __forceinline__ double la_log(S g) {
  const double v = (double)g;
  return v < kLaMinLog ? kLaMinLog : v;
}

// A decay over one or more tokens as the factor of a state.  A float32 factor near one is off by up to half a step of 2^-24, always in the
// same direction, and counts once a token (or chunk): exp(-1e-6) as one float acts as exp(-0.954e-6).  So it is two floats:
// 1 + (e^x - 1) keeps its error relative to the decay's distance from one.
template <class S> struct LaDecay;
template <> struct LaDecay<float> {
  float hi, lo;
  LaDecay() = default;
  __device__ __forceinline__ explicit LaDecay(double log) {
    const float x = (float)log;
    if (fabsf(x) <= 1.f) {
      const float q = expm1f(x);
      hi = 1.f + q;
      lo = q - (hi - 1.f);
    } else {
      hi = expf(x);
      lo = 0.f;
    }
  }
  __device__ __forceinline__ float operator()(float state, float more) const {   // (an infinite state stays infinite)
    return fmaf(hi, state, fabsf(state) < INFINITY ? fmaf(lo, state, more) : more);
  }
  // the same up to a decay of 1/16, in few registers (e^x - 1 by its series, the next term is below 2^-29 of it); a single float beyond
  __device__ __forceinline__ static LaDecay of_chunk(double log) {
    const float x = (float)log;
    LaDecay d;
    if (fabsf(x) <= 0.0625f) {
      const float q = x * fmaf(x * 0.5f, fmaf(x * (1.f / 3), fmaf(x * 0.25f, fmaf(x, 0.2f, 1.f), 1.f), 1.f), 1.f);
      d.hi = 1.f + q;
      d.lo = q - (d.hi - 1.f);
    } else {
      d.hi = expf(x);
      d.lo = 0.f;
    }
    return d;
  }
  __device__ __forceinline__ bool single() const { return lo == 0.f; }
};
template <> struct LaDecay<double> {
  double hi;
  LaDecay() = default;
  __device__ __forceinline__ explicit LaDecay(double log) : hi(exp(log)) {}
  __device__ __forceinline__ double operator()(double state, double more) const { return fma(hi, state, more); }
  __device__ __forceinline__ static LaDecay of_chunk(double log) { return LaDecay(log); }
  __device__ __forceinline__ bool single() const { return true; }
};

// Inclusive running sums of a chunk's log decays: G[i] for i < C, tokens from n on count 0.  One warp.  With L, in two doubles G + L:
// differences of sums behind a decay of zero (which is -1e5 in them) lose nothing.  float64 arithmetic needs that; beside
// float32 one double is exact enough.
template <class S, int C>
__device__ __forceinline__ void la_running_logs(double* G, double* L, const S* g, int64_t t_stride, int64_t t0, int n, int lane) {
  constexpr bool kTwo = std::is_same<S, double>::value;
  double carry = 0.0, carry_lo = 0.0;
  auto add = [](double& hi, double& lo, double h, double l) {   // lo takes what the rounding of hi + h loses
    const double s = hi + h, t = s - hi;
    lo += l + ((hi - (s - t)) + (h - t));
    hi = s;
  };
#pragma unroll
  for (int i0 = 0; i0 < C; i0 += 32) {
    const int i = i0 + lane;
    double v = i < n ? la_log(g[(t0 + i) * t_stride]) : 0.0, lo = 0.0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, v, d);
      if constexpr (kTwo) {
        const double ul = __shfl_up_sync(0xffffffffu, lo, d);
        if (lane >= d) add(v, lo, u, ul);
      } else {
        if (lane >= d) v += u;
      }
    }
    if constexpr (kTwo) {
      add(v, lo, carry, carry_lo);
      if (L) L[i] = lo;
      carry_lo = __shfl_sync(0xffffffffu, lo, 31);
    } else {
      v += carry;
    }
    G[i] = v;
    carry = __shfl_sync(0xffffffffu, v, 31);
  }
}

template <class S> struct LaVec4;   // four scalars, in 16-byte accesses
template <> struct LaVec4<float> { float4 v; __device__ __forceinline__ void get(float (&d)[4]) const { d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w; } };
template <> struct LaVec4<double> {
  double2 a, b;
  __device__ __forceinline__ void get(double (&d)[4]) const { d[0] = a.x; d[1] = a.y; d[2] = b.x; d[3] = b.y; }
};
template <class S> __device__ __forceinline__ void la_get4(S (&d)[4], const S* p) { reinterpret_cast<const LaVec4<S>*>(p)->get(d); }

// MD: channels of x and y that fit (64 or 128)
template <class S, int C, int NS, int MD>
struct LaSimtSmem {
  static constexpr int XLD = MD + 4;
  S x[C][XLD], y[C][XLD];
  S z[C][NS];
  S s[MD][NS];
  S p[C][C + 4];
  // two chunks' decays: weight of the entering state per row, weight with which a token joins the state, running sums
  S win[2][C], wout[2][C];
  double G[2][C];
  double L[2][sizeof(S) == 8 ? C : 1];
};

// Float32 / float64 arithmetic on the CUDA cores, any size up to 128: the path of float32, float64 and
// float16 tensors, and of bfloat16 tensors of at most 32 tokens.  A CTA walks one (b, h, segment) in time order with a slice of NS columns of
// the state in registers (8 x 4 per thread in float32) and a copy in shared memory for the products that read it.
// Two CTAs an SM: one's barriers and loads lie under the other's arithmetic.
template <class T, class S, int C, int NS, int MD, bool STATES_ONLY>
__global__ void __launch_bounds__(256, sizeof(S) == 4 ? 2 : 1) la_simt_kernel(const LaArgs<S> a) {
  extern __shared__ __align__(16) unsigned char la_smem[];
  using Sm = LaSimtSmem<S, C, NS, MD>;
  Sm& sm = *reinterpret_cast<Sm*>(la_smem);
  constexpr int TN = NS / 4;              // threads across the columns
  constexpr int MR = MD * TN / 256;       // rows of the state per thread
  static_assert(MR >= 2 && C % 32 == 0, "thread tiles must cover the state");
  constexpr int TR = C / (256 / TN);      // rows of o per thread
  constexpr bool kTwo = std::is_same<S, double>::value;   // sums of log decays in two doubles
  const int role = blockIdx.y;
  const LaPass<S>& p = a.p[role];
  const int slices = (p.N + NS - 1) / NS, seg_count = STATES_ONLY ? a.nseg - 1 : a.nseg;
  int64_t id = blockIdx.x;
  const int slice = (int)(id % ((kLaMaxDim + NS - 1) / NS));
  id /= (kLaMaxDim + NS - 1) / NS;
  const int ord = (int)(id % seg_count);   // the how-manieth segment of the pass, in its own direction
  const int64_t bh = id / seg_count;
  if (slice >= slices) return;
  const int64_t b = bh / a.H, h = bh % a.H, BH = a.B * a.H;
  const int M = p.M, N = p.N, n0 = slice * NS, nw = min(NS, N - n0);
  const int tid = threadIdx.x, lane = tid & 31, tn = tid % TN, tm = tid / TN;
  const int64_t len = la_length(a.lengths, b, a.T);
  const int64_t nchunk = (a.T + C - 1) / C;
  const int seg = p.reverse ? a.nseg - 1 - ord : ord;
  const int64_t c0 = (int64_t)seg * a.seg_chunks, c1 = min(c0 + (int64_t)a.seg_chunks, nchunk);
  const T* x = static_cast<const T*>(p.x) + b * p.xs[0] + h * p.xs[2];
  const T* y = static_cast<const T*>(p.y) + b * p.ys[0] + h * p.ys[2];
  const T* z = static_cast<const T*>(p.z) + b * p.zs[0] + h * p.zs[2] + n0;
  const T* w = static_cast<const T*>(p.w) + b * p.ws[0] + h * p.ws[2] + n0;
  const S* g = a.g + b * a.gs[0] + h * a.gs[2];

  S st[MR][4];
  {
    const S* src = nullptr;
    bool tr = false;
    if (!STATES_ONLY && ord > 0) src = a.seg + ((int64_t)(role * a.nseg + ord) * BH + bh) * a.seg_stride;
    else if (!STATES_ONLY && p.init) { src = p.init + bh * M * N; tr = p.state_t; }
#pragma unroll
    for (int i = 0; i < MR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = tm * MR + i, n = n0 + tn * 4 + j;
        st[i][j] = (src && m < M && n < N) ? src[tr ? (int64_t)n * M + m : (int64_t)m * N + n] : (S)0;
      }
  }
  double seg_log = 0.0;
  const int M4 = (M + 3) & ~3;
  auto chunk_of = [&](int64_t ci) { return p.reverse ? c1 - 1 - (ci - c0) : ci; };
  auto valid = [&](int64_t c) { return (int)max((int64_t)0, min((int64_t)C, len - c * C)); };
  // a chunk's decays, by one warp, a chunk ahead of their use
  auto decays = [&](int64_t ci, int buf) {
    const int64_t c = chunk_of(ci);
    la_running_logs<S, C>(sm.G[buf], sm.L[buf], g, a.gs[1], c * C, valid(c), lane);
    __syncwarp();
    const double E = sm.G[buf][C - 1];
    for (int i = lane; i < C; i += 32) {
      double to_end = E - sm.G[buf][i];
      if constexpr (kTwo) to_end += sm.L[buf][C - 1] - sm.L[buf][i];
      const S up = la_exp((S)sm.G[buf][i]), down = la_exp((S)to_end);
      sm.win[buf][i] = p.reverse ? down : up;
      sm.wout[buf][i] = (p.reverse ? up : down) * p.pz;
    }
  };
  // a warp takes whole rows of the operands: a lane every 32nd value, the next chunk's on their way to
  // registers while this one is worked on
  constexpr int RW = C / 8, ZW = NS / 32;
  constexpr int XW = MD / 32;
  S rx[RW][XW], ry[RW][XW], rz[RW][ZW];
  const int warp = tid >> 5;
  auto fetch = [&](int64_t ci) {
    const int64_t c = chunk_of(ci), t0 = c * C;
    const int n = valid(c);
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int r = warp + 8 * i;
#pragma unroll
      for (int k = 0; k < XW; ++k) {
        const int m = lane + 32 * k;
        const bool ok = r < n && m < M;
        if (!STATES_ONLY) rx[i][k] = ok ? la_load<S, T>(x + (t0 + r) * p.xs[1] + m) : (S)0;
        ry[i][k] = ok ? la_load<S, T>(y + (t0 + r) * p.ys[1] + m) : (S)0;
      }
#pragma unroll
      for (int k = 0; k < ZW; ++k) {
        const int q = lane + 32 * k;
        rz[i][k] = (r < n && q < nw) ? la_load<S, T>(z + (t0 + r) * p.zs[1] + q) : (S)0;
      }
    }
  };
  if (c0 < c1) {
    fetch(c0);
    if (warp == 7) decays(c0, 0);
  }
  for (int64_t ci = c0; ci < c1; ++ci) {
    const int64_t c = chunk_of(ci), t0 = c * C;
    const int n = valid(c), buf = (int)((ci - c0) & 1);
    __syncthreads();   // everything of the previous chunk has been read
    if (n > 0) {
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        const int r = warp + 8 * i;
#pragma unroll
        for (int k = 0; k < XW; ++k) {
          if (!STATES_ONLY) sm.x[r][lane + 32 * k] = rx[i][k];
          sm.y[r][lane + 32 * k] = ry[i][k];
        }
#pragma unroll
        for (int k = 0; k < ZW; ++k) sm.z[r][lane + 32 * k] = rz[i][k];
      }
      if (!STATES_ONLY) {
#pragma unroll
          for (int i = 0; i < MR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sm.s[tm * MR + i][tn * 4 + j] = st[i][j];
        if (p.bounds) {
          S* dst = p.bounds + (bh * nchunk + c) * M * N;
#pragma unroll
          for (int i = 0; i < MR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int m = tm * MR + i, q = n0 + tn * 4 + j;
              if (m < M && q < N) dst[(int64_t)m * N + q] = st[i][j];
            }
        }
      }
    }
    if (ci + 1 < c1) fetch(ci + 1);
    __syncthreads();
    if (warp == 7 && ci + 1 < c1) decays(ci + 1, buf ^ 1);
    if (n == 0) {            // behind the sequence: zeros come out, the state stays
      if (!STATES_ONLY && p.o) {
        for (int i = tid; i < C * nw; i += 256) {
          const int64_t t = t0 + i / nw, at = ((b * a.T + t) * a.H + h) * N + n0 + i % nw;
          if (t >= a.T) continue;
          if (p.wide) static_cast<S*>(p.o)[at] = (S)0;
          else la_store<T, S>(static_cast<T*>(p.o) + at, (S)0);
        }
      }
      continue;
    }
    const double* const G = sm.G[buf];
    const double E = G[C - 1];
    if (!STATES_ONLY) {
      {   // scores inside the chunk with their decays: a CR x CS block per thread, strided over the rows
        constexpr int TS = 16, CR = C / (256 / TS), CS = C / TS;
        const int ts = tid % TS, tr = tid / TS;
        S acc[CR][CS] = {};
#pragma unroll 4
        for (int m = 0; m < M4; m += 4) {
          S xv[CR][4], yv[CS][4];
#pragma unroll
          for (int i = 0; i < CR; ++i) la_get4(xv[i], &sm.x[tr * CR + i][m]);
#pragma unroll
          for (int j = 0; j < CS; ++j) la_get4(yv[j], &sm.y[ts + TS * j][m]);
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < CR; ++i)
#pragma unroll
              for (int j = 0; j < CS; ++j) acc[i][j] += xv[i][k] * yv[j][k];
        }
#pragma unroll
        for (int i = 0; i < CR; ++i)
#pragma unroll
          for (int j = 0; j < CS; ++j) {
            const int t = tr * CR + i, s = ts + TS * j;
            double between = p.reverse ? G[s] - G[t] : G[t] - G[s];
            if constexpr (kTwo) between += p.reverse ? sm.L[buf][s] - sm.L[buf][t] : sm.L[buf][t] - sm.L[buf][s];
            const S w = la_exp((S)between) * p.pz;
            sm.p[t][s] = (p.reverse ? s >= t && s < n : s <= t) ? acc[i][j] * w : (S)0;
          }
      }
      // o: TR rows x 4 columns per thread
      S intra[TR][4] = {}, inter[TR][4] = {};
#pragma unroll 2
      for (int m = 0; m < M4; m += 4) {   // rows of the state from M on are zero
        S sv[4][4], xv[TR][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) la_get4(sv[k], &sm.s[m + k][tn * 4]);
#pragma unroll
        for (int i = 0; i < TR; ++i) la_get4(xv[i], &sm.x[tm * TR + i][m]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < TR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) inter[i][j] += xv[i][k] * sv[k][j];
      }
      __syncthreads();
      // tokens before (mirrored: behind) all of the thread's rows, then the few among them: a masked token is not read,
      // 0 * inf would be NaN
      const int s_lo = p.reverse ? tm * TR + TR : 0, s_hi = p.reverse ? n : tm * TR;
#pragma unroll 4
      for (int s = s_lo; s < s_hi; ++s) {
        S zv[4];
        la_get4(zv, &sm.z[s][tn * 4]);
#pragma unroll
        for (int i = 0; i < TR; ++i) {
          const S pv = sm.p[tm * TR + i][s];
#pragma unroll
          for (int j = 0; j < 4; ++j) intra[i][j] += pv * zv[j];
        }
      }
#pragma unroll
      for (int k = 0; k < TR; ++k) {
        const int s = tm * TR + k;
        S zv[4];
        la_get4(zv, &sm.z[s][tn * 4]);
#pragma unroll
        for (int i = 0; i < TR; ++i) {
          if (p.reverse ? k < i || s >= n : k > i) continue;
          const S pv = sm.p[tm * TR + i][s];
#pragma unroll
          for (int j = 0; j < 4; ++j) intra[i][j] += pv * zv[j];
        }
      }
#pragma unroll
      for (int i = 0; i < TR; ++i) {
        const int r = tm * TR + i;
        const int64_t t = t0 + r;
        const S win = sm.win[buf][r];
        S d0 = 0, d1 = 0;
        const int64_t at = ((b * a.T + t) * a.H + h) * N + n0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int q = tn * 4 + j;
          const S in = intra[i][j] * p.po, ex = inter[i][j] * win * p.po;
          if (p.dots && r < n && q < nw) {
            const S wv = la_load<S, T>(w + t * p.ws[1] + q);
            d0 += in * wv;
            d1 += ex * wv;
          }
          if (p.o && t < a.T && q < nw) {
            const S v = r < n ? in + ex : (S)0;
            if (p.wide) static_cast<S*>(p.o)[at + q] = v;
            else la_store<T, S>(static_cast<T*>(p.o) + at + q, v);
          }
        }
        if (p.dots) {
#pragma unroll
          for (int d = TN / 2; d > 0; d >>= 1) {
            d0 += __shfl_down_sync(0xffffffffu, d0, d, TN);
            d1 += __shfl_down_sync(0xffffffffu, d1, d, TN);
          }
          if (tn == 0 && r < n) {
            S* dst = p.dots + (((int64_t)slice * BH + bh) * a.T + t) * 2;
            dst[0] = d0;
            dst[1] = d1;
          }
        }
      }
    }
    {   // the state moves on by one chunk
      // Where a chunk decays by more than 1/16, the half steps of a single factor come to less than 16 on a state that has decayed
      // to 1/e, which is less than the state's own roundings: one product there instead of two multiply-adds and a test
      // (B=3, T=1999, H=6, Dk=80, Dv=48 in float16, with the join: 99.0 -> 97.4 us)
      const LaDecay<S> dec = LaDecay<S>::of_chunk(E);
      if (dec.single()) {
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) st[i][j] *= dec.hi;
      } else {
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) st[i][j] = dec(st[i][j], (S)0);
      }
      if (tm * MR < M4) {
#pragma unroll 4
        for (int s = 0; s < C; ++s) {   // tokens from n on are zero
          const S wv = sm.wout[buf][s];
          S zv[4], yv[MR];
          la_get4(zv, &sm.z[s][tn * 4]);
          if constexpr (MR >= 4) {
#pragma unroll
            for (int i = 0; i < MR; i += 4) la_get4(*reinterpret_cast<S(*)[4]>(&yv[i]), &sm.y[s][tm * MR + i]);
          } else {
#pragma unroll
            for (int i = 0; i < MR; ++i) yv[i] = sm.y[s][tm * MR + i];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) zv[j] *= wv;
#pragma unroll
          for (int i = 0; i < MR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) st[i][j] += yv[i] * zv[j];
        }
      }
    }
    seg_log += E;
  }
  S* dst = nullptr;
  bool tr = false;
  if (STATES_ONLY) dst = a.seg + ((int64_t)(role * a.nseg + ord + 1) * BH + bh) * a.seg_stride;
  else if (p.fin && ord == a.nseg - 1) { dst = p.fin + bh * M * N; tr = p.state_t; }
  if (dst) {
#pragma unroll
    for (int i = 0; i < MR; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = tm * MR + i, q = n0 + tn * 4 + j;
        if (m < M && q < N) dst[tr ? (int64_t)q * M + m : (int64_t)m * N + q] = st[i][j];
      }
  }
  if (STATES_ONLY && slice == 0 && tid == 0) a.seg_log[(int64_t)(role * a.nseg + ord) * BH + bh] = seg_log;
}

// Entering states of the segments: seg[d+1] = exp(log decay of segment d) * seg[d] + (what segment d added).
template <class S>
__global__ void la_join_kernel(const LaArgs<S> a) {
  const int role = blockIdx.y;
  const LaPass<S>& p = a.p[role];
  const int64_t MN = (int64_t)p.M * p.N, BH = a.B * a.H;
  const int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (e >= BH * MN) return;
  const int64_t bh = e / MN, i = e % MN, m = i / p.N, n = i % p.N;
  S v = p.init ? p.init[bh * MN + (p.state_t ? n * p.M + m : i)] : (S)0;
  const double* log = a.seg_log + (int64_t)role * a.nseg * BH + bh;
  S* slot = a.seg + ((int64_t)(role * a.nseg + 1) * BH + bh) * a.seg_stride + i;
  double lg = *log;
  S more = *slot;
  for (int d = 0; d + 1 < a.nseg; ++d) {
    const LaDecay<S> dec = LaDecay<S>::of_chunk(lg);
    const S add = more;
    S* const at = slot;
    if (d + 2 < a.nseg) {   // the next segment's values are on their way while this one's are worked on
      lg = *(log += BH);
      more = *(slot += BH * a.seg_stride);
    }
    v = dec(v, add);
    *at = v;
  }
}

// Gradient of the log decays.  Token t's decay scales every pair (s < t <= u), so inside a chunk
//   dg[t] = exp(E) <S, R>  +  sum_{u>=t} Xo[u]  +  sum_{s<t} Ko[s]  +  sum_{u>=t} Xi[u] - sum_{s>=t} Ki[s]
// with S the state entering the chunk, R the adjoint state entering it from the right, X. = q.dq and K. = k.dk
// split into their parts inside the chunk (i) and from the entering state (o).  The sums start anew in
// every chunk, so rounding does not accumulate over the row.
template <class S>
struct LaDecayArgs {
  const S *s_bounds, *r_bounds;   // [bh][chunk][MN]
  const S *qd, *kd;               // dots of the two passes, [slice][bh][t][2]
  int q_slices, k_slices;
  const S* g;
  int64_t gs[3];
  LaLengths lengths;
  int64_t B, T, H, MN;            // scalars of a state
  S* dg;           // (B,T,H), or NULL
  double* part;    // [chunk][bh] sums over a chunk, or NULL
};

template <class S, int C>
__global__ void __launch_bounds__(256) la_decay_grad_kernel(const LaDecayArgs<S> a) {
  __shared__ double red[8], G[C];
  const int64_t BH = a.B * a.H, bh = blockIdx.x % BH, c = blockIdx.x / BH, b = bh / a.H, h = bh % a.H;
  const int64_t nchunk = (a.T + C - 1) / C, t0 = c * C, len = la_length(a.lengths, b, a.T);
  const int n = (int)max((int64_t)0, min((int64_t)C, len - t0));
  const int tid = threadIdx.x, lane = tid & 31;
  double acc = 0.0;
  if (n > 0) {
    const S* s = a.s_bounds + (bh * nchunk + c) * a.MN;
    const S* r = a.r_bounds + (bh * nchunk + c) * a.MN;
    if (a.MN % 4 == 0) {   // 16-byte accesses, eight of them on their way
#pragma unroll 4
      for (int64_t i = tid * 4; i < a.MN; i += 1024) {
        S sv[4], rv[4];
        la_get4(sv, s + i);
        la_get4(rv, r + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc += (double)sv[k] * (double)rv[k];
      }
    } else {
      for (int64_t i = tid; i < a.MN; i += 256) acc += (double)s[i] * (double)r[i];
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) acc += __shfl_down_sync(0xffffffffu, acc, d);
  if (lane == 0) red[tid >> 5] = acc;
  __syncthreads();
  if (tid >= 32) return;
  if (n > 0) la_running_logs<S, C>(G, nullptr, a.g + b * a.gs[0] + h * a.gs[2], a.gs[1], t0, n, lane);
  __syncwarp();
  double base = 0.0;
  for (int i = 0; i < 8; ++i) base += red[i];
  if (n > 0) base *= exp(G[C - 1]);
  constexpr int PER = C / 32;
  double suffix[PER], prefix[PER], fs = 0.0, fp = 0.0;   // per lane: PER consecutive tokens
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = lane * PER + j;
    double xi = 0, xo = 0, ki = 0, ko = 0;
    if (i < n) {
      for (int k = 0; k < a.q_slices; ++k) {
        const S* d = a.qd + (((int64_t)k * BH + bh) * a.T + t0 + i) * 2;
        xi += (double)d[0];
        xo += (double)d[1];
      }
      for (int k = 0; k < a.k_slices; ++k) {
        const S* d = a.kd + (((int64_t)k * BH + bh) * a.T + t0 + i) * 2;
        ki += (double)d[0];
        ko += (double)d[1];
      }
    }
    suffix[j] = xi + xo - ki;
    prefix[j] = ko;
    fs += suffix[j];
    fp += prefix[j];
  }
  double after = fs, before = fp;   // inclusive scans over the lanes: from the right, from the left
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double u = __shfl_down_sync(0xffffffffu, after, d), v = __shfl_up_sync(0xffffffffu, before, d);
    if (lane + d < 32) after += u;
    if (lane >= d) before += v;
  }
  double run_p = before - fp, run_s = after, total = 0.0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = lane * PER + j;
    const double v = i < n ? base + run_s + run_p : 0.0;
    if (a.dg && t0 + i < a.T) a.dg[(b * a.T + t0 + i) * a.H + h] = (S)v;
    total += v;
    run_s -= suffix[j];
    run_p += prefix[j];
  }
  if (a.part) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) total += __shfl_down_sync(0xffffffffu, total, d);
    if (lane == 0) a.part[c * BH + bh] = total;
  }
}

// One decay per head: the sum over batch and time, in a fixed order.
template <class S>
__global__ void __launch_bounds__(256) la_decay_sum_kernel(const double* part, int64_t nchunk, int64_t B, int64_t H, S* dg) {
  __shared__ double red[8];
  const int64_t h = blockIdx.x;
  double acc = 0.0;
  for (int64_t i = threadIdx.x; i < nchunk * B; i += 256) acc += part[i * H + h];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) acc += __shfl_down_sync(0xffffffffu, acc, d);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) acc += red[i];
    dg[h] = (S)acc;
  }
}

// One token: state <- exp(g) state + k v^T in place, o = scale * q^T state.  Bound by reading and writing the
// state once.  A CTA owns 32 columns of one (b, h): they need no sum across CTAs, and a row of them is a 128-byte
// line of float32; the 8 warps take the rows in turn.
template <class T, class S>
struct LaStepArgs {
  const T *q, *k, *v;
  int64_t qs[2], ks[2], vs[2];   // strides (b, h)
  const S* g;
  int64_t gs[2];
  S* state;
  int64_t ss[2];
  void* o;                       // dense (B,H,N) of T, or of S when wide
  int64_t H;
  int M, N, wide;
  S scale;
};

template <class T, class S, int V>
__global__ void __launch_bounds__(256) la_step_kernel(const LaStepArgs<T, S> a) {
  constexpr int CW = 32 / V, RW = 256 / CW;   // threads across 32 columns, rows at once
  struct alignas(V * sizeof(S) > 16 ? 16 : V * sizeof(S)) Vec { S v[V]; };
  __shared__ S q[kLaMaxDim], k[kLaMaxDim], red[RW][32 + 1];
  __shared__ LaDecay<S> decay;
  const int64_t bh = blockIdx.x, b = bh / a.H, h = bh % a.H;
  const int n0 = blockIdx.y * 32, tid = threadIdx.x, tc = tid % CW, tr = tid / CW, n = n0 + tc * V;
  S* st = a.state + b * a.ss[0] + h * a.ss[1] + n;
  constexpr int U = kLaMaxDim / RW;           // rows per thread
  Vec s[U];
  const bool on = n < a.N;                    // V > 1 only where N is a multiple of V
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int m = tr + u * RW;
    if (on && m < a.M) s[u] = *reinterpret_cast<const Vec*>(st + (int64_t)m * a.N);
  }
  if (tid < a.M) {
    q[tid] = la_load<S, T>(a.q + b * a.qs[0] + h * a.qs[1] + tid) * a.scale;
    k[tid] = la_load<S, T>(a.k + b * a.ks[0] + h * a.ks[1] + tid);
  }
  if (tid == 255) decay = LaDecay<S>(la_log(a.g[b * a.gs[0] + h * a.gs[1]]));   // (a warp without keys to fetch)
  S v[V], acc[V] = {};
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = on ? la_load<S, T>(a.v + b * a.vs[0] + h * a.vs[1] + n + j) : (S)0;
  __syncthreads();
  const LaDecay<S> dec = decay;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int m = tr + u * RW;
    if (on && m < a.M) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[u].v[j] = dec(s[u].v[j], k[m] * v[j]);
        acc[j] += q[m] * s[u].v[j];
      }
      *reinterpret_cast<Vec*>(st + (int64_t)m * a.N) = s[u];
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) red[tr][tc * V + j] = acc[j];
  __syncthreads();
  if (tid < 32 && n0 + tid < a.N) {
    S sum = 0;
    for (int r = 0; r < RW; ++r) sum += red[r][tid];
    const int64_t at = bh * a.N + n0 + tid;
    if (a.wide) static_cast<S*>(a.o)[at] = sum;
    else la_store<T, S>(static_cast<T*>(a.o) + at, sum);
  }
}

}  // namespace ptb
