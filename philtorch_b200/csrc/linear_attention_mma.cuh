// The passes of linear_attention.cuh on the tensor cores, for bfloat16 tensors (mma.sync m16n8k16, float32
// accumulation).  A CTA of four warps walks one (b, h, segment) in time order, 64 tokens at a time; warp w owns a quarter
// of the state's columns n, held TRANSPOSED in accumulator registers (rows n, columns m).  In that layout the
// accumulators of two neighbouring tiles are, packed to bfloat16, exactly the B operand of the product that reads the
// state, so the state never goes through shared memory.
//
// Accuracy.  q, k, v are exact operands; what the products take besides (weights inside a chunk, the decayed z of the
// state's update, the state as an operand) is float32 and has to be rounded.  For a bfloat16 RESULT one rounding of
// it to bfloat16 is as good as the rounding of the result itself.  For a float32 result (the final state, the gradients
// of decays and of the initial state) it is split into three bfloat16 terms (24 bits) and costs three products.
#pragma once
#include "linear_attention.cuh"

namespace ptb {

constexpr int kLaMmaChunk = 64;

__device__ __forceinline__ uint32_t la_pack(float lo, float hi) {   // {lo, hi} in memory order
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// the two values of a packed pair, as float32
__device__ __forceinline__ float la_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float la_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// exp of a difference of log decays given in units of log 2; results below the normal range are zero
__device__ __forceinline__ float la_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void la_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void la_ldm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void la_ldm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void la_cp16(uint32_t dst, const void* src, bool on) {   // off: 16 zero bytes
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void la_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void la_cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// a tile of bfloat16 rows of W columns; 16-byte pieces exchanged by the row's low bits, so that the eight rows
// of a matrix load fall into different banks
template <int W>
__device__ __forceinline__ uint32_t la_at(uint32_t tile, int row, int piece) {
  return tile + row * (W * 2) + ((piece ^ (row & 7)) << 4);
}

template <int W, bool VEC>
__device__ __forceinline__ void la_tile_load(uint32_t tile, unsigned char* tile_ptr, const __nv_bfloat16* src, int64_t t_stride,
                                             int64_t t0, int n, int width, int tid) {
  constexpr int PIECES = W / 8;
  for (int i = tid; i < kLaMmaChunk * PIECES; i += 128) {
    const int r = i / PIECES, p = i % PIECES;
    if constexpr (VEC) {
      const bool on = r < n && p * 8 < width;
      la_cp16(la_at<W>(tile, r, p), on ? src + (t0 + r) * t_stride + p * 8 : src, on);
    } else {
      __align__(16) __nv_bfloat16 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = (r < n && p * 8 + j < width) ? src[(t0 + r) * t_stride + p * 8 + j] : __float2bfloat16_rn(0.f);
      *reinterpret_cast<uint4*>(tile_ptr + (la_at<W>(tile, r, p) - tile)) = *reinterpret_cast<const uint4*>(v);
    }
  }
}

template <int MP, int NP>
struct LaMmaSmem {
  static constexpr int C = kLaMmaChunk;
  static constexpr int X = C * MP * 2, Z = C * NP * 2, STAGE = 2 * X + Z;   // x, y, z
  static constexpr int P = C * C * 2;
  // after the stages: P, G (double), win, wout, row and column sums of the decay's gradient, G in two floats
  static constexpr int MISC = C * 8 + 2 * C * 4 + (4 + 4 + 1 + 2) * C * 4;
  static int bytes(int stages, bool dots) { return stages * STAGE + (dots ? Z : 0) + P + MISC; }
};

// accurate: the state is updated (bit 0) and read (bit 1) in three terms
struct LaMmaFlags {
  int accurate[3];
  int stages;
  int all_segments;   // the pass that only forms states covers the last segment too, and its end is the final state
};

template <int MP, int NP, bool VEC, bool STATES_ONLY>
__global__ void __launch_bounds__(128) la_mma_kernel(const LaArgs<float> a, const LaMmaFlags f) {
  using Sm = LaMmaSmem<MP, NP>;
  constexpr int C = kLaMmaChunk, MT = MP / 8, NJ = NP / 64;   // 8-wide tiles of m; 16-high tiles of n per warp
  extern __shared__ __align__(128) unsigned char la_mma_smem[];
  const int role = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g4 = lane >> 2, t4 = lane & 3;
  const LaPass<float>& p = a.p[role];
  if (STATES_ONLY && f.all_segments && !p.fin && blockIdx.x % a.nseg == a.nseg - 1) return;   // nobody asks for its end
  const bool acc_u = f.accurate[role] & 1, acc_s = f.accurate[role] & 2, dots = !STATES_ONLY && p.dots;
  const int seg_count = STATES_ONLY ? a.nseg - (f.all_segments ? 0 : 1) : a.nseg;
  const int ord = (int)(blockIdx.x % seg_count);
  const int64_t bh = blockIdx.x / seg_count;
  const int64_t b = bh / a.H, h = bh % a.H, BH = a.B * a.H;
  const int M = p.M, N = p.N, nw = warp * (NP / 4);
  const int64_t len = la_length(a.lengths, b, a.T), nchunk = (a.T + C - 1) / C;
  const int seg = p.reverse ? a.nseg - 1 - ord : ord;
  const int64_t c0 = (int64_t)seg * a.seg_chunks, c1 = min(c0 + (int64_t)a.seg_chunks, nchunk);
  const bool rev = p.reverse;
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + b * p.xs[0] + h * p.xs[2];
  const __nv_bfloat16* y = static_cast<const __nv_bfloat16*>(p.y) + b * p.ys[0] + h * p.ys[2];
  const __nv_bfloat16* z = static_cast<const __nv_bfloat16*>(p.z) + b * p.zs[0] + h * p.zs[2];
  const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(p.w) + b * p.ws[0] + h * p.ws[2];
  const float* g = a.g + b * a.gs[0] + h * a.gs[2];

  unsigned char* const misc = la_mma_smem + f.stages * Sm::STAGE + (dots ? Sm::Z : 0);
  unsigned char* const wt_ptr = la_mma_smem + f.stages * Sm::STAGE;
  const uint32_t s_w = smem_u32(wt_ptr), s_p = smem_u32(misc);
  double* const G = reinterpret_cast<double*>(misc + Sm::P);
  float* const win = reinterpret_cast<float*>(G + C);
  float* const wout = win + C;
  float* const cols = wout + C;        // [4][C]
  float* const ext = cols + 4 * C;     // [4][C]: each warp's share of w.o from the entering state
  float* const rows = ext + 4 * C;     // [C]
  float* const Gh = rows + C;          // [C], [C]: the running sums in units of log 2, in two floats (what one float loses of
  float* const Gl = Gh + C;            //   them would be lost to the difference of two tokens behind a strong decay)

  float st[NJ][MT][4];
  {
    const float* src = nullptr;
    bool padded = false;
    if (!STATES_ONLY && ord > 0) { src = a.seg + ((int64_t)(role * (a.nseg + 1) + ord) * BH + bh) * a.seg_stride; padded = true; }
    else if (!STATES_ONLY && p.init) src = p.init + bh * M * N;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = nw + 16 * j + g4 + (e >> 1) * 8, m = 8 * i + 2 * t4 + (e & 1);
          float v = 0.f;
          if (src) {
            if (padded) v = src[n * MP + m];
            else if (m < M && n < N) v = src[p.state_t ? n * M + m : m * N + n];
          }
          st[j][i][e] = v;
        }
  }
  double seg_log = 0.0;

  // the chunks of a segment in pass order
  auto chunk_of = [&](int64_t ci) { return rev ? c1 - 1 - (ci - c0) : ci; };
  auto valid = [&](int64_t c) { return (int)max((int64_t)0, min((int64_t)C, len - c * C)); };
  auto fetch = [&](int64_t ci, int stage) {
    const int64_t c = chunk_of(ci), t0 = c * C;
    const int n = valid(c);
    unsigned char* sp = la_mma_smem + stage * Sm::STAGE;
    const uint32_t sx = smem_u32(sp);
    if (n > 0) {
      if (!STATES_ONLY) la_tile_load<MP, VEC>(sx, sp, x, p.xs[1], t0, n, M, tid);
      la_tile_load<MP, VEC>(sx + Sm::X, sp + Sm::X, y, p.ys[1], t0, n, M, tid);
      la_tile_load<NP, VEC>(sx + 2 * Sm::X, sp + 2 * Sm::X, z, p.zs[1], t0, n, N, tid);
    }
    if (VEC) la_cp_commit();
  };
  if (f.stages == 2 && c0 < c1) fetch(c0, 0);
  for (int64_t ci = c0; ci < c1; ++ci) {
    const int64_t c = chunk_of(ci), t0 = c * C;
    const int n = valid(c), stage = f.stages == 2 ? (int)((ci - c0) & 1) : 0;
    __syncthreads();   // everything of the previous chunk has been read
    if (f.stages == 2) {
      if (ci + 1 < c1) fetch(ci + 1, stage ^ 1);
      else if (VEC) la_cp_commit();
    } else {
      fetch(ci, 0);
    }
    if (n == 0) {      // behind the sequence: zeros come out, the state stays
      if (!STATES_ONLY && p.o) {
        for (int i = tid; i < C * N; i += 128) {
          const int64_t t = t0 + i / N, at = ((b * a.T + t) * a.H + h) * N + i % N;
          if (t >= a.T) continue;
          if (p.wide) static_cast<float*>(p.o)[at] = 0.f;
          else static_cast<__nv_bfloat16*>(p.o)[at] = __float2bfloat16_rn(0.f);
        }
      }
      continue;
    }
    if (dots) {
      la_tile_load<NP, VEC>(s_w, wt_ptr, w, p.ws[1], t0, n, N, tid);
      if (VEC) la_cp_commit();
    }
    if (warp == 0) {
      la_running_logs<float, C>(G, g, a.gs[1], t0, n, lane);
      __syncwarp();
      const double E = G[C - 1];
      for (int i = lane; i < C; i += 32) {
        const float up = expf((float)G[i]), down = expf((float)(E - G[i]));
        win[i] = rev ? down : up;
        wout[i] = (rev ? up : down) * p.pz;
        const double in = (rev ? -G[i] : G[i]) * 1.4426950408889634;
        Gh[i] = (float)in;
        Gl[i] = (float)(in - (double)Gh[i]);
      }
    }
    if (VEC) {
      if (f.stages == 2) la_cp_wait<1>();   // two stages: never with dots, the newest group is the next chunk's
      else la_cp_wait<0>();
    }
    __syncthreads();
    const uint32_t sx = smem_u32(la_mma_smem + stage * Sm::STAGE), sy = sx + Sm::X, sz = sy + Sm::X;
    const double E = G[C - 1];

    if constexpr (!STATES_ONLY) {
      if (p.bounds) {   // [n][m], padded
        float* dst = p.bounds + (bh * nchunk + c) * (int64_t)(MP * NP);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<float2*>(dst + (nw + 16 * j + g4 + e * 8) * MP + 8 * i + 2 * t4) =
                  make_float2(st[j][i][2 * e], st[j][i][2 * e + 1]);
      }
      {   // scores of the rows 16 warp .. 16 warp + 15
        float sc[8][4] = {};
#pragma unroll 1
        for (int kk = 0; kk < MP / 16; ++kk) {
          uint32_t av[4];
          la_ldm(av, la_at<MP>(sx, 16 * warp + (lane & 15), 2 * kk + (lane >> 4)));
#pragma unroll
          for (int jp = 0; jp < 4; ++jp)
            if (rev ? jp >= warp : jp <= warp) {
              uint32_t bv[4];
              la_ldm(bv, la_at<MP>(sy, 16 * jp + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
              la_mma(sc[2 * jp], av, bv[0], bv[1]);
              la_mma(sc[2 * jp + 1], av, bv[2], bv[3]);
            }
        }
        const int r0 = 16 * warp + g4;
        const float2 own0 = make_float2(Gh[r0], Gl[r0]), own1 = make_float2(Gh[r0 + 8], Gl[r0 + 8]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (rev ? j >= 2 * warp : j < 2 * warp + 2) {
            const float2 gh = *reinterpret_cast<const float2*>(Gh + 8 * j + 2 * t4), gl = *reinterpret_cast<const float2*>(Gl + 8 * j + 2 * t4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int s = 8 * j + 2 * t4 + (e & 1), t = r0 + (e >> 1) * 8;
              const float2 own = e >> 1 ? own1 : own0;
              const float d = (own.x - (e & 1 ? gh.y : gh.x)) + (own.y - (e & 1 ? gl.y : gl.x));
              const float w = la_exp2(d) * p.pz;   // (mirrored: the sums are stored negated)
              sc[j][e] = (rev ? s >= t && s < n : s <= t) ? sc[j][e] * w : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int t = r0 + e * 8;
              *reinterpret_cast<uint32_t*>(misc + (la_at<C>(0, t, j) + t4 * 4)) = la_pack(sc[j][2 * e], sc[j][2 * e + 1]);
            }
          }
        if (dots) {   // pairs (t, s) inside the chunk: weight * (x.y)(w.z), summed over rows and over columns
          float s2[8][4] = {};
#pragma unroll 1
          for (int kk = 0; kk < NP / 16; ++kk) {
            uint32_t av[4];
            la_ldm(av, la_at<NP>(s_w, 16 * warp + (lane & 15), 2 * kk + (lane >> 4)));
#pragma unroll
            for (int jp = 0; jp < 4; ++jp)
              if (rev ? jp >= warp : jp <= warp) {
                uint32_t bv[4];
                la_ldm(bv, la_at<NP>(sz, 16 * jp + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
                la_mma(s2[2 * jp], av, bv[0], bv[1]);
                la_mma(s2[2 * jp + 1], av, bv[2], bv[3]);
              }
          }
          float rs[2] = {0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float cs[2] = {0.f, 0.f};
            if (rev ? j >= 2 * warp : j < 2 * warp + 2) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int s = 8 * j + 2 * t4 + (e & 1), t = r0 + (e >> 1) * 8;
                const float v = s == t || sc[j][e] == 0.f ? 0.f : sc[j][e] * s2[j][e] * p.po;   // the diagonal cancels
                rs[e >> 1] += v;
                cs[e & 1] += v;
              }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) cs[e] += __shfl_xor_sync(0xffffffffu, cs[e], d);
              if (g4 == 0) cols[warp * C + 8 * j + 2 * t4 + e] = cs[e];
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            rs[e] += __shfl_xor_sync(0xffffffffu, rs[e], 1);
            rs[e] += __shfl_xor_sync(0xffffffffu, rs[e], 2);
            if (t4 == 0) rows[r0 + e * 8] = rs[e];
          }
        }
      }
      __syncthreads();
      float o[4][NJ * 2][4] = {};
#pragma unroll
      for (int kk = 0; kk < MP / 16; ++kk) {   // the entering state's part
        uint32_t av[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) la_ldm(av[i], la_at<MP>(sx, 16 * i + (lane & 15), 2 * kk + (lane >> 4)));
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float v0 = st[j][2 * kk][2 * hf], v1 = st[j][2 * kk][2 * hf + 1];
            float v2 = st[j][2 * kk + 1][2 * hf], v3 = st[j][2 * kk + 1][2 * hf + 1];
            uint32_t b0 = la_pack(v0, v1), b1 = la_pack(v2, v3);
#pragma unroll
            for (int i = 0; i < 4; ++i) la_mma(o[i][2 * j + hf], av[i], b0, b1);
            if (acc_s) {
#pragma unroll
              for (int term = 0; term < 2; ++term) {
                v0 -= la_lo(b0); v1 -= la_hi(b0); v2 -= la_lo(b1); v3 -= la_hi(b1);
                b0 = la_pack(v0, v1); b1 = la_pack(v2, v3);
#pragma unroll
                for (int i = 0; i < 4; ++i) la_mma(o[i][2 * j + hf], av[i], b0, b1);
              }
            }
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w0 = win[16 * i + g4], w1 = win[16 * i + g4 + 8];
#pragma unroll
        for (int q = 0; q < NJ * 2; ++q) {
          o[i][q][0] *= w0; o[i][q][1] *= w0; o[i][q][2] *= w1; o[i][q][3] *= w1;
        }
        if (dots) {
          float d0 = 0.f, d1 = 0.f;
#pragma unroll
          for (int q = 0; q < NJ * 2; ++q) {
            const int piece = (nw + 8 * q) / 8, r = 16 * i + g4;
            const uint32_t e0 = *reinterpret_cast<const uint32_t*>(wt_ptr + (la_at<NP>(0, r, piece) + t4 * 4));
            const uint32_t e1 = *reinterpret_cast<const uint32_t*>(wt_ptr + (la_at<NP>(0, r + 8, piece) + t4 * 4));
            d0 += o[i][q][0] * la_lo(e0) + o[i][q][1] * la_hi(e0);
            d1 += o[i][q][2] * la_lo(e1) + o[i][q][3] * la_hi(e1);
          }
          d0 += __shfl_xor_sync(0xffffffffu, d0, 1);
          d0 += __shfl_xor_sync(0xffffffffu, d0, 2);
          d1 += __shfl_xor_sync(0xffffffffu, d1, 1);
          d1 += __shfl_xor_sync(0xffffffffu, d1, 2);
          if (t4 == 0) { ext[warp * C + 16 * i + g4] = d0; ext[warp * C + 16 * i + g4 + 8] = d1; }
        }
      }
#pragma unroll 1
      for (int kk = 0; kk < 4; ++kk) {   // the chunk's own tokens
        uint32_t zv[NJ][4];
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          la_ldm_t(zv[j], la_at<NP>(sz, 16 * kk + (lane & 7) + (((lane >> 3) & 1) << 3), (nw + 16 * j) / 8 + (lane >> 4)));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (rev ? kk >= i : kk <= i) {
            uint32_t av[4];
            la_ldm(av, la_at<C>(s_p, 16 * i + (lane & 15), 2 * kk + (lane >> 4)));
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              la_mma(o[i][2 * j], av, zv[j][0], zv[j][1]);
              la_mma(o[i][2 * j + 1], av, zv[j][2], zv[j][3]);
            }
          }
      }
      if (p.o) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 16 * i + g4 + e * 8;
            if (t0 + r >= a.T) continue;
            const int64_t at = ((b * a.T + t0 + r) * a.H + h) * N;
            __nv_bfloat16* row = static_cast<__nv_bfloat16*>(p.o) + at;
            float* wide = static_cast<float*>(p.o) + at;
            const bool on = r < n;
#pragma unroll
            for (int q = 0; q < NJ * 2; ++q) {
              const int col = nw + 8 * q + 2 * t4;
              const float v0 = on ? o[i][q][2 * e] * p.po : 0.f, v1 = on ? o[i][q][2 * e + 1] * p.po : 0.f;
              if (p.wide) {
                if (col < N) wide[col] = v0;
                if (col + 1 < N) wide[col + 1] = v1;
              } else if (VEC) {   // N is a multiple of 8
                if (col < N) *reinterpret_cast<uint32_t*>(row + col) = la_pack(v0, v1);
              } else {
                if (col < N) row[col] = __float2bfloat16_rn(v0);
                if (col + 1 < N) row[col + 1] = __float2bfloat16_rn(v1);
              }
            }
          }
      }
      if (dots) {
        __syncthreads();
        if (tid < n) {
          float in = rows[tid], ex = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            in -= cols[k * C + tid];
            ex += ext[k * C + tid];
          }
          float* d = p.dots + (bh * a.T + t0 + tid) * 2;
          d[0] = rev ? 0.f : in;    // the mirrored pass would give the same pairs again
          d[1] = ex * p.po;
        }
      }
    }
    {   // the state moves on by one chunk
      const float dec = expf((float)E);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) st[j][i][e] *= dec;
#pragma unroll 1
      for (int kk = 0; kk < 4; ++kk) {
        const float w0 = wout[16 * kk + 2 * t4], w1 = wout[16 * kk + 2 * t4 + 1];
        const float w2 = wout[16 * kk + 2 * t4 + 8], w3 = wout[16 * kk + 2 * t4 + 9];
        uint32_t t0v[NJ][4], t1v[NJ][4], t2v[NJ][4];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          uint32_t zv[4];
          la_ldm_t(zv, la_at<NP>(sz, 16 * kk + (lane & 7) + ((lane >> 4) << 3), (nw + 16 * j) / 8 + ((lane >> 3) & 1)));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v0 = la_lo(zv[e]) * (e < 2 ? w0 : w2), v1 = la_hi(zv[e]) * (e < 2 ? w1 : w3);
            t0v[j][e] = la_pack(v0, v1);
            v0 -= la_lo(t0v[j][e]); v1 -= la_hi(t0v[j][e]);
            t1v[j][e] = la_pack(v0, v1);
            v0 -= la_lo(t1v[j][e]); v1 -= la_hi(t1v[j][e]);
            t2v[j][e] = la_pack(v0, v1);
          }
        }
#pragma unroll
        for (int q = 0; q < MT / 2; ++q) {
          uint32_t bv[4];
          la_ldm_t(bv, la_at<MP>(sy, 16 * kk + (lane & 7) + (((lane >> 3) & 1) << 3), 2 * q + (lane >> 4)));
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            // terms added up on their own, smallest first, then to the state: the tensor core's additions truncate, which
            // against the whole state would add up over the chunks
            float u0[4] = {}, u1[4] = {};
            if (acc_u) {
              la_mma(u0, t2v[j], bv[0], bv[1]);
              la_mma(u1, t2v[j], bv[2], bv[3]);
            }
            la_mma(u0, t1v[j], bv[0], bv[1]);
            la_mma(u1, t1v[j], bv[2], bv[3]);
            la_mma(u0, t0v[j], bv[0], bv[1]);
            la_mma(u1, t0v[j], bv[2], bv[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              st[j][2 * q][e] += u0[e];
              st[j][2 * q + 1][e] += u1[e];
            }
          }
        }
      }
    }
    seg_log += E;
  }
  if (VEC) la_cp_wait<0>();
  if (STATES_ONLY) {
    float* dst = a.seg + ((int64_t)(role * (a.nseg + 1) + ord + 1) * BH + bh) * a.seg_stride;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float2*>(dst + (nw + 16 * j + g4 + e * 8) * MP + 8 * i + 2 * t4) =
              make_float2(st[j][i][2 * e], st[j][i][2 * e + 1]);
    if (tid == 0) a.seg_log[(int64_t)(role * a.nseg + ord) * BH + bh] = seg_log;
  } else if (p.fin && ord == a.nseg - 1 && !f.all_segments) {
    float* dst = p.fin + bh * M * N;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int nn = nw + 16 * j + g4 + (e >> 1) * 8, m = 8 * i + 2 * t4 + (e & 1);
          if (m < M && nn < N) dst[p.state_t ? nn * M + m : m * N + nn] = st[j][i][e];
        }
  }
}

// Entering states of the segments for the layout above (slots [role][nseg + 1], padded [n][m]); with all_segments the
// last slot becomes the final state.
template <int MP, int NP>
__global__ void la_mma_join_kernel(const LaArgs<float> a, const LaMmaFlags f) {
  const int role = blockIdx.y;
  const LaPass<float>& p = a.p[role];
  const int64_t BH = a.B * a.H, e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, bh = e / (MP * NP);
  if (bh >= BH) return;
  const int i = (int)(e % (MP * NP)), n = i / MP, m = i % MP;
  const bool on = m < p.M && n < p.N;
  const int64_t at = bh * p.M * p.N + (p.state_t ? n * p.M + m : m * p.N + n);
  float v = p.init && on ? p.init[at] : 0.f;
  const int count = a.nseg - (f.all_segments && p.fin ? 0 : 1);
  for (int d = 0; d < count; ++d) {
    const double lg = a.seg_log[(int64_t)(role * a.nseg + d) * BH + bh];
    float* slot = a.seg + ((int64_t)(role * (a.nseg + 1) + d + 1) * BH + bh) * a.seg_stride + i;
    v = expf((float)lg) * v + *slot;
    *slot = v;
  }
  if (f.all_segments && p.fin && on) p.fin[at] = v;
}

}  // namespace ptb
