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
#include "packed.cuh"

namespace ptb {

constexpr int kLnMaxWidth = 16384;

template <class S>
struct LnArgs {
  const void *x, *w, *b, *gy;
  int64_t x_stride, gy_stride;     // elements between two rows
  int w_wide;                      // w and b hold S instead of the storage type
  int w_vec;                       // w and b start on 16 bytes
  void *y, *gx;                    // dense
  S *mean, *rstd;                  // [row][group]
  S *part_w, *part_b;              // [CTA][channel], may be NULL
  int64_t rows;
  int groups, width;
  S eps;
};

template <class T, int V> struct alignas(V * sizeof(T)) LnRaw { T v[V]; };   // one access

template <class T, class S, int V>
__device__ __forceinline__ void ln_widen(S (&d)[V], const LnRaw<T, V>& r) {
#pragma unroll
  for (int i = 0; i < V; ++i) d[i] = la_load<S, T>(&r.v[i]);
}
template <class T, class S, int V>
__device__ __forceinline__ void ln_load(S (&d)[V], const T* p) {
  ln_widen<T, S, V>(d, *reinterpret_cast<const LnRaw<T, V>*>(p));
}
template <class T, class S, int V>
__device__ __forceinline__ void ln_store(T* p, const S (&d)[V]) {
  LnRaw<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) la_store<T, S>(&r.v[i], d[i]);
  *reinterpret_cast<LnRaw<T, V>*>(p) = r;
}
// parameters (they stay in L1): whole accesses where they start on 16 bytes, else element by element
template <class T, class S, int V>
__device__ __forceinline__ void ln_param(S (&d)[V], const void* p, int wide, int vec, int64_t at) {
  if (vec && !wide) {
    ln_load<T, S, V>(d, static_cast<const T*>(p) + at);
  } else if (vec) {
    constexpr int P = V * sizeof(S) > 16 ? 16 / sizeof(S) : V;
#pragma unroll
    for (int i = 0; i < V; i += P) {
      const LnRaw<S, P> r = *reinterpret_cast<const LnRaw<S, P>*>(static_cast<const S*>(p) + at + i);
#pragma unroll
      for (int k = 0; k < P; ++k) d[i + k] = r.v[k];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      d[i] = wide ? static_cast<const S*>(p)[at + i] : la_load<S, T>(static_cast<const T*>(p) + at + i);
  }
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

// V scalars as V / 2 pairs (V = 1: one pair, its second half zero)
template <class S, int V> constexpr int kLnPairs = V > 1 ? V / 2 : 1;
template <class S, int V>
__device__ __forceinline__ void ln_pairs(Pair<S> (&d)[kLnPairs<S, V>], const S (&v)[V]) {
  if constexpr (V == 1) {
    d[0] = Pair<S>(v[0], (S)0);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) d[i] = Pair<S>(v[2 * i], v[2 * i + 1]);
  }
}
template <class S, int V>
__device__ __forceinline__ void ln_scalars(S (&d)[V], const Pair<S> (&v)[kLnPairs<S, V>]) {
  if constexpr (V == 1) {
    d[0] = v[0].get().x;
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const auto f = v[i].get();
      d[2 * i] = f.x;
      d[2 * i + 1] = f.y;
    }
  }
}
__device__ __forceinline__ float ln_rsqrt(float v) { return rsqrtf(v); }
__device__ __forceinline__ double ln_rsqrt(double v) { return rsqrt(v); }

__host__ __device__ constexpr int ln_threads(int L) { return L > 256 ? L : 256; }
// values of one row that a thread holds decide how many CTAs can be resident
__host__ __device__ constexpr int ln_resident(int L, int per_thread) { return L > 256 || per_thread > 32 ? 1 : per_thread > 16 ? 2 : 3; }

// Rows in flight.  What keeps memory busy is bytes on their way: a thread asks for its pieces of the next DEPTH rows with
// 16-byte asynchronous copies into slots of shared memory of its own (nobody else reads them, so there is no
// barrier).  8192 rows of 16 groups of 128 bfloat16: one row ahead in registers 25.5 us
// forward and 58.6 us backward, four ahead 18.5 and 31.3 us (3.6 and 3.2 TB/s; float32 5.0 and 5.5 TB/s: at half
// the bytes per value the instructions count).
// Rows that do not start on 16 bytes, and very wide ones, stay with one row ahead in registers (DEPTH 0).
template <class T, int V, int L, int NV>
__host__ __device__ constexpr int ln_depth(int arrays) {
  const int stage = ln_threads(L) * NV * arrays * 16, d = 65536 / stage;
  return V * (int)sizeof(T) != 16 || d < 2 ? 0 : d > 4 ? 4 : d;
}
template <class T, class S, int V, int L, int NV>
__host__ __device__ constexpr int ln_pipe_bytes(int arrays) {
  return ln_depth<T, V, L, NV>(arrays) * ln_threads(L) * (NV * arrays * 16 + (arrays > 1 ? 2 * (int)sizeof(S) : 0));
}
__device__ __forceinline__ void ln_cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
template <int BYTES> __device__ __forceinline__ void ln_cp(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void ln_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void ln_arrived() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// grid: (row blocks, groups).  A thread keeps its channels, so it keeps its weights and biases, and asks for the
// next row's values while it works on this one's.
template <class T, class TO, class S, int V, int L, int NV>
__global__ void __launch_bounds__(ln_threads(L), ln_resident(L, NV * V)) ln_fwd_kernel(const LnArgs<S> a) {
  constexpr int NT = ln_threads(L), SLOTS = NT / L, P = kLnPairs<S, V>;
  __shared__ S sm[32];
  const int l = threadIdx.x % L, slot = threadIdx.x / L, grp = blockIdx.y;
  Pair<S> w[NV][P], b[NV][P];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * L + l) * V;
    S wv[V], bv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) wv[i] = 1, bv[i] = 0;
    if (a.w && c < a.width) ln_param<TO, S, V>(wv, a.w, a.w_wide, a.w_vec, (int64_t)grp * a.width + c);
    if (a.b && c < a.width) ln_param<TO, S, V>(bv, a.b, a.w_wide, a.w_vec, (int64_t)grp * a.width + c);
    ln_pairs<S, V>(w[k], wv);
    ln_pairs<S, V>(b[k], bv);
  }
  constexpr int D = ln_depth<T, V, L, NV>(1);
  extern __shared__ __align__(16) unsigned char ln_dyn[];
  LnRaw<T, V>* const ring = reinterpret_cast<LnRaw<T, V>*>(ln_dyn);   // [stage][k][thread]
  LnRaw<T, V> rx[NV];
  auto fetch = [&](int64_t row, int stage) {
    if (row < a.rows) {
      const T* x = static_cast<const T*>(a.x) + row * a.x_stride + (int64_t)grp * a.width;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * L + l) * V;
        if (c < a.width) {
          if constexpr (D > 0) ln_cp16(ring + (stage * NV + k) * NT + threadIdx.x, x + c);
          else rx[k] = *reinterpret_cast<const LnRaw<T, V>*>(x + c);
        }
      }
    }
    if constexpr (D > 0) ln_commit();
  };
  const S inv = (S)1 / (S)a.width;
  const int64_t step = (int64_t)gridDim.x * SLOTS;
  int stage = 0;
  for (int d = 0; d < (D > 0 ? D : 1); ++d) fetch((int64_t)blockIdx.x * SLOTS + slot + d * step, d);
  for (int64_t r0 = (int64_t)blockIdx.x * SLOTS; r0 < a.rows; r0 += step) {   // the same rounds for every lane of the CTA
    const int64_t row = r0 + slot;
    const bool on = row < a.rows;
    Pair<S> v[NV][P], acc((S)0, (S)0);
    if constexpr (D > 0) {
      ln_arrived<(D > 0 ? D - 1 : 0)>();
#pragma unroll
      for (int k = 0; k < NV; ++k) rx[k] = ring[(stage * NV + k) * NT + threadIdx.x];
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      S f[V] = {};
      if (on && (k * L + l) * V < a.width) ln_widen<T, S, V>(f, rx[k]);
      ln_pairs<S, V>(v[k], f);
#pragma unroll
      for (int i = 0; i < P; ++i) acc = acc + v[k][i];
    }
    fetch(row + (D > 0 ? D : 1) * step, stage);
    stage = stage + 1 < D ? stage + 1 : 0;
    S sum[1] = {acc.get().x + acc.get().y};
    ln_sum<S, L, 1>(sum, sm);
    const S mu = sum[0] * inv;
    const Pair<S> mu2(mu, V > 1 ? mu : (S)0);
    acc = Pair<S>((S)0, (S)0);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if ((k * L + l) * V < a.width)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          v[k][i] = v[k][i] - mu2;
          acc = fma2(v[k][i], v[k][i], acc);
        }
    sum[0] = acc.get().x + acc.get().y;
    ln_sum<S, L, 1>(sum, sm);
    const S r = ln_rsqrt(sum[0] * inv + a.eps);
    if (on) {
      const int64_t u = row * a.groups + grp;
      if (l == 0 && a.mean) {
        a.mean[u] = mu;
        a.rstd[u] = r;
      }
      TO* y = static_cast<TO*>(a.y) + u * a.width;
      const Pair<S> r2(r, r);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * L + l) * V;
        if (c >= a.width) continue;
#pragma unroll
        for (int i = 0; i < P; ++i) v[k][i] = fma2(v[k][i] * r2, w[k][i], b[k][i]);
        S f[V];
        ln_scalars<S, V>(f, v[k]);
        ln_store<TO, S, V>(y + c, f);
      }
    }
  }
}

// grid: (row blocks, groups)
template <class T, class S, int V, int L, int NV>
__global__ void __launch_bounds__(ln_threads(L), ln_resident(L, 2 * NV * V)) ln_bwd_kernel(const LnArgs<S> a) {
  constexpr int NT = ln_threads(L), SLOTS = NT / L, P = kLnPairs<S, V>;
  __shared__ S sm[64];
  extern __shared__ __align__(16) unsigned char ln_dyn[];
  S* join = reinterpret_cast<S*>(ln_dyn);     // [slot][width] when SLOTS > 1
  const int l = threadIdx.x % L, slot = threadIdx.x / L, grp = blockIdx.y;
  Pair<S> aw2[NV][P], ab2[NV][P];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) aw2[k][i] = ab2[k][i] = Pair<S>((S)0, (S)0);
  // a row's values are asked for while the row before it is worked on
  constexpr int D = ln_depth<T, V, L, NV>(2);
  LnRaw<T, V>* const ring = reinterpret_cast<LnRaw<T, V>*>(ln_dyn);   // [stage][x, gy][k][thread]
  S* const ring_s = reinterpret_cast<S*>(ln_dyn + D * 2 * NV * NT * 16);   // [stage][mean, rstd][thread]
  LnRaw<T, V> rx[NV], rg[NV];
  S next_mu = 0, next_r = 0;
  auto fetch = [&](int64_t row, int stage) {
    if (row < a.rows) {
      const T* x = static_cast<const T*>(a.x) + row * a.x_stride + (int64_t)grp * a.width;
      const T* gy = static_cast<const T*>(a.gy) + row * a.gy_stride + (int64_t)grp * a.width;
      const int64_t u = row * a.groups + grp;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * L + l) * V;
        if (c < a.width) {
          if constexpr (D > 0) {
            ln_cp16(ring + (stage * 2 * NV + k) * NT + threadIdx.x, x + c);
            ln_cp16(ring + ((stage * 2 + 1) * NV + k) * NT + threadIdx.x, gy + c);
          } else {
            rx[k] = *reinterpret_cast<const LnRaw<T, V>*>(x + c);
            rg[k] = *reinterpret_cast<const LnRaw<T, V>*>(gy + c);
          }
        }
      }
      if constexpr (D > 0) {
        ln_cp<sizeof(S)>(ring_s + stage * 2 * NT + threadIdx.x, a.mean + u);
        ln_cp<sizeof(S)>(ring_s + (stage * 2 + 1) * NT + threadIdx.x, a.rstd + u);
      } else {
        next_mu = a.mean[u];
        next_r = a.rstd[u];
      }
    }
    if constexpr (D > 0) ln_commit();
  };
  const S inv = (S)1 / (S)a.width;
  const int64_t step = (int64_t)gridDim.x * SLOTS;
  int stage = 0;
  for (int d = 0; d < (D > 0 ? D : 1); ++d) fetch((int64_t)blockIdx.x * SLOTS + slot + d * step, d);
  for (int64_t r0 = (int64_t)blockIdx.x * SLOTS; r0 < a.rows; r0 += step) {
    const int64_t row = r0 + slot;
    const bool on = row < a.rows;
    if constexpr (D > 0) {
      ln_arrived<(D > 0 ? D - 1 : 0)>();
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        rx[k] = ring[(stage * 2 * NV + k) * NT + threadIdx.x];
        rg[k] = ring[((stage * 2 + 1) * NV + k) * NT + threadIdx.x];
      }
      next_mu = ring_s[stage * 2 * NT + threadIdx.x];
      next_r = ring_s[(stage * 2 + 1) * NT + threadIdx.x];
    }
    const S mu = on ? next_mu : (S)0, r = on ? next_r : (S)0;
    const Pair<S> mu2(mu, mu), r2(r, r);
    Pair<S> xh[NV][P], g[NV][P], s0((S)0, (S)0), s1((S)0, (S)0);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * L + l) * V;
      S fx[V], fg[V] = {}, fw[V];
#pragma unroll
      for (int i = 0; i < V; ++i) fx[i] = mu, fw[i] = 1;
      if (on && c < a.width) {
        ln_widen<T, S, V>(fx, rx[k]);
        ln_widen<T, S, V>(fg, rg[k]);
        if (a.w) ln_param<T, S, V>(fw, a.w, a.w_wide, a.w_vec, (int64_t)grp * a.width + c);
      }
      Pair<S> w[P];
      ln_pairs<S, V>(xh[k], fx);
      ln_pairs<S, V>(g[k], fg);
      ln_pairs<S, V>(w, fw);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        xh[k][i] = (xh[k][i] - mu2) * r2;
        aw2[k][i] = fma2(g[k][i], xh[k][i], aw2[k][i]);
        ab2[k][i] = ab2[k][i] + g[k][i];
        g[k][i] = g[k][i] * w[i];
        s0 = s0 + g[k][i];
        s1 = fma2(g[k][i], xh[k][i], s1);
      }
    }
    fetch(row + (D > 0 ? D : 1) * step, stage);
    stage = stage + 1 < D ? stage + 1 : 0;
    if (a.gx) {
      S sum[2] = {s0.get().x + s0.get().y, s1.get().x + s1.get().y};
      ln_sum<S, L, 2>(sum, sm);
      const S m0 = sum[0] * inv, m1 = -sum[1] * inv;
      const Pair<S> m02(m0, m0), m12(m1, m1);
      if (on) {
        T* gx = static_cast<T*>(a.gx) + (row * a.groups + grp) * a.width;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = (k * L + l) * V;
          if (c >= a.width) continue;
          S f[V];
#pragma unroll
          for (int i = 0; i < P; ++i) g[k][i] = fma2(xh[k][i], m12, g[k][i] - m02) * r2;
          ln_scalars<S, V>(f, g[k]);
          ln_store<T, S, V>(gx + c, f);
        }
      }
    }
  }
  if (!a.part_w && !a.part_b) return;
  if constexpr (D > 0) {
    ln_arrived<0>();
    __syncthreads();   // the slots become the joining array
  }
  S aw[NV][V], ab[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    ln_scalars<S, V>(aw[k], aw2[k]);
    ln_scalars<S, V>(ab[k], ab2[k]);
  }
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
