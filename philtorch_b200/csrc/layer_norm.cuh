// Layer norm over groups of channels, forward and backward.
//   mu = mean(x), r = 1/sqrt(mean((x-mu)^2) + eps), xh = (x-mu) r, y = xh w + b      (w, b per channel)
//   gu = gy w;  gx = r (gu - mean(gu) - xh mean(gu xh));  gw = sum_rows gy xh;  gb = sum_rows gy
// Both directions are bound by memory: a unit (one group of one row) stays in the registers of L lanes
// between its sums and its result, so x (and gy) are read once.  The mean is subtracted before squaring.
// In the backward kernel a lane keeps the same channels over all the rows it takes, so the parameter
// gradients add up in its registers; a CTA joins its lanes in shared memory and leaves ONE partial row,
// and a second kernel adds the partial rows in a fixed order (bit-reproducible).
#pragma once
#include "linear_attention.cuh"

namespace ptb {

constexpr int kLnMaxWidth = 16384;

template <class S>
struct LnArgs {
  const void *x, *w, *b, *gy;
  int64_t x_stride, gy_stride;     // elements between two rows
  int w_wide;                      // w and b hold S instead of the storage type
  void *y, *gx;                    // dense
  S *mean, *rstd;                  // [row][group]
  S *part_w, *part_b;              // [CTA][channel], may be NULL
  int64_t rows;
  int groups, width;
  S eps;
};

template <class T, class S, int V>
__device__ __forceinline__ void ln_load(S (&d)[V], const T* p) {
  struct alignas(V * sizeof(T)) Raw { T v[V]; };
  const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) d[i] = la_load<S, T>(&r.v[i]);
}
template <class T, class S, int V>
__device__ __forceinline__ void ln_store(T* p, const S (&d)[V]) {
  struct alignas(V * sizeof(T)) Raw { T v[V]; } r;
#pragma unroll
  for (int i = 0; i < V; ++i) la_store<T, S>(&r.v[i], d[i]);
  *reinterpret_cast<Raw*>(p) = r;
}
// parameters: element-wise (they are not asked to be aligned, and stay in L1)
template <class T, class S, int V>
__device__ __forceinline__ void ln_param(S (&d)[V], const void* p, int wide, int64_t at) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    d[i] = wide ? static_cast<const S*>(p)[at + i] : la_load<S, T>(static_cast<const T*>(p) + at + i);
}

// sums over the L lanes of a unit; every lane gets them
template <class S, int L, int K>
__device__ __forceinline__ void ln_sum(S (&v)[K], S* sm) {
  constexpr int W = L < 32 ? L : 32;
#pragma unroll
  for (int d = W / 2; d > 0; d >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], d);
  if constexpr (L > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();   // the previous sums have been read
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) sm[warp * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      S t = 0;
      for (int w = 0; w < L / 32; ++w) t += sm[w * K + k];
      v[k] = t;
    }
  }
}

template <class T, class S, int V, int L, int NV>
__global__ void __launch_bounds__(L > 256 ? L : 256) ln_fwd_kernel(const LnArgs<S> a) {
  constexpr int NT = L > 256 ? L : 256, SLOTS = NT / L;
  __shared__ S sm[32];
  const int l = threadIdx.x % L, slot = threadIdx.x / L;
  const int64_t units = a.rows * a.groups;
  // whole warps stay together: every lane of the CTA runs the same number of rounds
  for (int64_t u0 = (int64_t)blockIdx.x * SLOTS; u0 < units; u0 += (int64_t)gridDim.x * SLOTS) {
    const int64_t u = u0 + slot;
    const bool on = u < units;
    const int64_t row = on ? u / a.groups : 0;
    const int grp = on ? (int)(u % a.groups) : 0;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride + (int64_t)grp * a.width;
    S v[NV][V], sum[1] = {0};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * L + l) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = 0;
      if (on && c < a.width) ln_load<T, S, V>(v[k], x + c);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[0] += v[k][i];
    }
    ln_sum<S, L, 1>(sum, sm);
    const S mu = sum[0] / (S)a.width;
    S sq[1] = {0};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * L + l) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[k][i] -= mu;
        if (c < a.width) sq[0] += v[k][i] * v[k][i];
      }
    }
    ln_sum<S, L, 1>(sq, sm);
    const S r = (S)1 / sqrt(sq[0] / (S)a.width + a.eps);
    if (!on) continue;
    if (l == 0 && a.mean) {
      a.mean[u] = mu;
      a.rstd[u] = r;
    }
    T* y = static_cast<T*>(a.y) + u * a.width;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * L + l) * V;
      if (c >= a.width) continue;
      S w[V], b[V];
      if (a.w) ln_param<T, S, V>(w, a.w, a.w_wide, (int64_t)grp * a.width + c);
      if (a.b) ln_param<T, S, V>(b, a.b, a.w_wide, (int64_t)grp * a.width + c);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        S o = v[k][i] * r;
        if (a.w) o *= w[i];
        if (a.b) o += b[i];
        v[k][i] = o;
      }
      ln_store<T, S, V>(y + c, v[k]);
    }
  }
}

// grid: (row blocks, groups)
template <class T, class S, int V, int L, int NV>
__global__ void __launch_bounds__(L > 256 ? L : 256) ln_bwd_kernel(const LnArgs<S> a) {
  constexpr int NT = L > 256 ? L : 256, SLOTS = NT / L;
  __shared__ S sm[64];
  extern __shared__ __align__(16) unsigned char ln_dyn[];
  S* join = reinterpret_cast<S*>(ln_dyn);     // [slot][width] when SLOTS > 1
  const int l = threadIdx.x % L, slot = threadIdx.x / L, grp = blockIdx.y;
  S aw[NV][V], ab[NV][V], w[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * L + l) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) aw[k][i] = ab[k][i] = 0, w[k][i] = 1;
    if (a.w && c < a.width) ln_param<T, S, V>(w[k], a.w, a.w_wide, (int64_t)grp * a.width + c);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * SLOTS; r0 < a.rows; r0 += (int64_t)gridDim.x * SLOTS) {
    const int64_t row = r0 + slot;
    const bool on = row < a.rows;
    const int64_t u = (on ? row : 0) * a.groups + grp;
    const T* x = static_cast<const T*>(a.x) + (on ? row : 0) * a.x_stride + (int64_t)grp * a.width;
    const T* gy = static_cast<const T*>(a.gy) + (on ? row : 0) * a.gy_stride + (int64_t)grp * a.width;
    const S mu = a.mean[u], r = a.rstd[u];
    S xh[NV][V], g[NV][V], sum[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * L + l) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) xh[k][i] = mu, g[k][i] = 0;
      if (on && c < a.width) {
        ln_load<T, S, V>(xh[k], x + c);
        ln_load<T, S, V>(g[k], gy + c);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xh[k][i] = (xh[k][i] - mu) * r;
        aw[k][i] += g[k][i] * xh[k][i];
        ab[k][i] += g[k][i];
        g[k][i] *= w[k][i];
        sum[0] += g[k][i];
        sum[1] += g[k][i] * xh[k][i];
      }
    if (a.gx) {
      ln_sum<S, L, 2>(sum, sm);
      const S m0 = sum[0] / (S)a.width, m1 = sum[1] / (S)a.width;
      if (on) {
        T* gx = static_cast<T*>(a.gx) + u * a.width;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = (k * L + l) * V;
          if (c >= a.width) continue;
#pragma unroll
          for (int i = 0; i < V; ++i) g[k][i] = r * (g[k][i] - m0 - xh[k][i] * m1);
          ln_store<T, S, V>(gx + c, g[k]);
        }
      }
    }
  }
  if (!a.part_w && !a.part_b) return;
  const int64_t at = (int64_t)blockIdx.x * a.groups * a.width + (int64_t)grp * a.width;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    S* dst = which ? a.part_b : a.part_w;
    if (!dst) continue;
    if constexpr (SLOTS == 1) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = (k * L + l) * V + i;
          if (c < a.width) dst[at + c] = which ? ab[k][i] : aw[k][i];
        }
    } else {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = (k * L + l) * V + i;
          if (c < a.width) join[slot * a.width + c] = which ? ab[k][i] : aw[k][i];
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.width; c += NT) {
        S t = 0;
        for (int s = 0; s < SLOTS; ++s) t += join[s * a.width + c];
        dst[at + c] = t;
      }
    }
  }
}

// gw, gb: sums of the partial rows; 32 channels x 8 parts per CTA
template <class T, class S>
__global__ void __launch_bounds__(256) ln_param_grad_kernel(const S* part_w, const S* part_b, int nparts, int64_t C,
                                                            void* gw, void* gb, int w_wide) {
  __shared__ S sm[8][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int s = threadIdx.x >> 5;
  const S* part = blockIdx.y ? part_b : part_w;
  void* out = blockIdx.y ? gb : gw;
  if (!part) return;
  S t = 0;
  if (c < C)
#pragma unroll 8
    for (int i = s; i < nparts; i += 8) t += part[(int64_t)i * C + c];
  sm[s][threadIdx.x & 31] = t;
  __syncthreads();
  if (s == 0 && c < C) {
    for (int i = 1; i < 8; ++i) t += sm[i][threadIdx.x];
    if (w_wide) static_cast<S*>(out)[c] = t;
    else la_store<T, S>(static_cast<T*>(out) + c, t);
  }
}

}  // namespace ptb
