// The passes of linear_attention.cuh on the fifth-generation tensor cores (tcgen05, accumulators in tensor memory), for bfloat16
// tensors of more than 32 tokens and any head size (operands that the TMA unit cannot address are copied first: la_move_kernel).
//
// A CTA walks one (b, h, segment) in chunks of 128 tokens with a slice of 64 columns of the state.  Four products per
// chunk, issued by one thread:
//   SC = X Y^T (128 x 128)         OI = X S (128 x 64)        O = P Z (P from tensor memory)        U = Y^T Zw
// around which two groups of eight warps work, two threads per row:
//   rows   P = SC * decays, rounded to bfloat16, back into tensor memory; then o = po (pz O + win OI) to memory, a chunk
//          later: while the next chunk's products run
//   state  S <- exp(E) S + U in registers (float32); S and the weighted Zw go to shared memory as bfloat16 operands
// and single warps drive the TMA loads (no multicast), the products and the running sums of the decays.  U of a
// chunk does not wait for the state, so the chain from chunk to chunk is one multiply-add per element of the state.
//
// Accuracy.  q, k, v are exact operands; what the products take besides (weights inside a chunk, the weighted z, the
// state) is float32 and has to be rounded.  For a bfloat16 RESULT one rounding of P and of S is as good as the
// rounding of the result itself; Zw takes two bfloat16 terms (16 bits), because its rounding would meet that of S.  For
// a float32 result (the final state, the gradient of the decays: DOTS) it is split into three terms (24 bits), and the
// pairs inside a chunk come from the float32 scores themselves.
//
// Why this shape.  128 rows fill the tensor core; 64 columns leave room in shared memory (227 KB) for two stages of
// X, Y and Z beside three terms of Zw, and in tensor memory for a second O and OI; the price is that both slices of
// a head form the scores.  Eight warps a group instead of four: 238 -> 203 us (B=4, T=8192, H=16, D=128, final state).
// Loops instead of straight-line code wherever the tensor-memory tiles allow it: unrolled, the warps' different roles
// did not fit the instruction cache together, and the kernel ran at the rate of the instruction fetch (718 -> 337 us).
// Rows leaving a chunk later: 203 -> 178 us.  Tried and dropped: P in the place of the scores with U in one
// product (194 us: the next scores then wait for O), loading the next scores ahead in registers (216 us),
// prefetching tiles into L2 (no change), 32-byte stores (2.3 -> 3.1 us a chunk).
// What bounds it: 2.5 us a chunk and CTA, in which the row group (weights 1.0, output 0.6 us) and the issue order
// of the products alternate; tensor pipe 29 % busy, DRAM 28 %; with 128 SMs busy the 1000 W limit may hold the clock at
// 1.6 GHz.  157 us without the final state, 186 us with it (537 MB: floor 82 us); 183 and 201 us at 1.6 GHz.
#pragma once
#include "linear_attention.cuh"
#include "packed.cuh"
#include "tensor_map.cuh"

namespace ptb {

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

constexpr int kTcChunk = 128, kTcSlice = 64, kTcDim = 128;
constexpr int kTcPanel = kTcChunk * 128;            // bytes of 128 rows x 64 bfloat16
constexpr int kTcRows = 256, kTcThreads = 2 * kTcRows + 96;   // row and state groups; products, loads, decays
constexpr uint32_t kErrPipelineWait = 8u;

// scalars from row to row of a state that is kept for the decays' gradient: read back in 16-byte accesses
__host__ __device__ __forceinline__ constexpr int la_tc_bound_pitch(int M) { return (M + 3) & ~3; }

struct LaTcMap {
  CUtensorMap map;
  int bmul, hmul;   // 0 where the axis is shared (stride zero)
};
struct LaTcArgs {
  LaArgs<float> a;
  LaTcMap x[3], y[3], z[3], w[3];
  int nu[3], ns[3];   // terms of Zw and of S
  int xy_stages, all_segments;
  long long wait_cycles;
  uint32_t* status;
};

// shared memory: X/Y stages (two panels each), two Z (and W) stages, terms of Zw, terms of S, small arrays
struct LaTcSmem {
  int z, zw, s, misc, total;
  __host__ __device__ LaTcSmem(int xy_stages, bool dots, int nu, int ns) {
    z = xy_stages * 4 * kTcPanel;
    zw = z + 2 * (dots ? 2 : 1) * kTcPanel;
    s = zw + nu * kTcPanel;
    misc = s + ns * kTcPanel;
    total = misc + 2 * kTcChunk * 8 + kTcChunk * 4 + 2 * 64 + 208;
  }
};

__device__ __forceinline__ void tc_alloc(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_dealloc(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t (&r)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_tma(uint32_t dst, const CUtensorMap* map, int d, int t, int h, int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(d), "r"(t), "r"(h), "r"(b), "r"(smem_u32(bar))
      : "memory");
}

using TcPair = Pair<float>;
__device__ __forceinline__ TcPair tc_pair(uint32_t a, uint32_t b) { return TcPair(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ TcPair tc_pair(float a, float b) { return TcPair(a, b); }
__device__ __forceinline__ uint32_t tc_pack(TcPair v) {   // two bfloat16
  const float2 f = v.get();
  return la_pack(f.x, f.y);
}
__device__ __forceinline__ TcPair tc_widen(uint32_t v) { return tc_pair(la_lo(v), la_hi(v)); }
__device__ __forceinline__ bool tc_elect() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on != 0;
}

// Operand descriptors: 128-byte swizzled panels of 64 values a row; groups of 8 rows are 1024 bytes apart, the two
// panels of a 128-wide tile kTcPanel bytes.  The same panel serves with its rows as M/N ("K-major": 16 values of K
// are 32 bytes further along a row) and with its rows as K ("MN-major": 16 values of K are 16 rows further down).
constexpr uint32_t kTcDescHi = (2u << 29) | (1u << 14) | (1024 >> 4);
__device__ __forceinline__ uint32_t tc_desc(uint32_t tile) { return ((uint32_t)(kTcPanel >> 4) << 16) | (tile >> 4); }   // low word
// K / 16 products over one tile: operand a from shared memory (K- or MN-major) or, as packed columns, from tensor memory
enum TcOperand { kKMajor, kMnMajor, kTmem };
template <TcOperand A, TcOperand B>
__device__ __forceinline__ void tc_products(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool fresh, int steps = 8) {
  constexpr uint32_t kRow = 2, kDown = 2048 >> 4, kOver = kTcPanel >> 4;
#pragma unroll 1
  for (int k0 = 0; k0 < steps; k0 += 4) {   // the 64 columns of a panel, or 64 rows
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const uint64_t db = ((uint64_t)kTcDescHi << 32) | (b + kk * (B == kKMajor ? kRow : kDown));
      const uint32_t accumulate = kk > 0 || k0 > 0 || !fresh;
      if constexpr (A == kTmem) tc_mma_ts(d, a + kk * 8, db, idesc, accumulate);
      else tc_mma_ss(d, ((uint64_t)kTcDescHi << 32) | (a + kk * (A == kKMajor ? kRow : kDown)), db, idesc, accumulate);
    }
    a += A == kTmem ? 32 : A == kKMajor ? kOver : 4 * kDown;
    b += B == kKMajor ? kOver : 4 * kDown;
  }
}
// float32 accumulation of bfloat16 operands; a_mn / b_mn: MN-major operand
__host__ __device__ constexpr uint32_t tc_idesc(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// What a chunk's decays come to.  Per token: the sum of the log decays inside its block of 32 tokens, in units of log 2 and
// in two floats (what one float loses of the sums would be lost to the difference of two tokens behind a strong decay),
// negated in a mirrored pass.  Per block: decay from the chunk's start to the block, over the block, from the block
// to the chunk's end.  A weight between two blocks is the product of such exponentials, none of them above one
// for decays below one.
struct __align__(16) TcFactors {
  float before[4], over[4], after[4];
  float dec[2];   // over the chunk, in two floats
};
__device__ __forceinline__ void tc_logs(float* Gs, TcFactors* f, const float (&raw)[4], bool rev, int lane, double* total) {
  constexpr double kLog2E = 1.4426950408889634;
  double v[4];
  v[0] = la_log(raw[0]) * kLog2E;
#pragma unroll
  for (int j = 1; j < 4; ++j) v[j] = v[j - 1] + la_log(raw[j]) * kLog2E;
  double sum = v[3];   // over the lanes of a block: 8 lanes of 4 tokens
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) {
    const double u = __shfl_up_sync(0xffffffffu, sum, d, 8);
    if ((lane & 7) >= d) sum += u;
  }
  double before = __shfl_up_sync(0xffffffffu, sum, 1, 8);   // (not sum - v[3]: a NaN would reach the tokens before it)
  if ((lane & 7) == 0) before = 0.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double in = rev ? -(before + v[j]) : before + v[j];
    const float hi = (float)in;
    Gs[4 * lane + j] = hi;
    Gs[kTcChunk + 4 * lane + j] = (float)(in - (double)hi);
  }
  double end[4], run = 0.0;
#pragma unroll
  for (int k = 0; k < 4; ++k) end[k] = __shfl_sync(0xffffffffu, sum, 8 * k + 7);
  const double E = end[0] + end[1] + end[2] + end[3];
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f->before[k] = la_exp2((float)run);
      f->over[k] = la_exp2((float)end[k]);
      run += end[k];
      f->after[k] = la_exp2((float)(E - run));
    }
    const LaDecay<float> dec(E * 0.69314718055994531);
    f->dec[0] = dec.hi;
    f->dec[1] = dec.lo;
  }
  *total += E;
}
__device__ __forceinline__ void tc_load_logs(float (&raw)[4], const float* g, int64_t t_stride, int64_t t0, int n, int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = 4 * lane + j;
    raw[j] = i < n ? g[(t0 + i) * t_stride] : 0.f;
  }
}

// An infinite or NaN value of z must not meet the zero weights of the tokens that do not see it (0 * inf): it is taken out of the
// tile that P multiplies (Zw keeps it, so the state and everything behind the chunk get it), and at the end the outputs that do see it
// are overwritten with NaN.  Both functions are out of line: they run on such data only.  What looking for it costs: nothing for a
// prompt of B=4, T=8192, H=16, D=128 (with a normalised read-out 281 us), 345 -> 349 us for a training step of B=2, T=4096, H=16, D=128.
// (Rows that looked at each chunk as it left: 353 us; that replaced their values in registers: 366 us.)
// Zeroes the odd values in the 32 columns of a row that a thread of the state group owns.
__device__ __noinline__ void tc_take_out(unsigned char* z_row, int row, int part) {
  for (int q = 4 * part; q < 4 * part + 4; ++q) {
    uint4* const at = reinterpret_cast<uint4*>(z_row + ((q ^ (row & 7)) << 4));
    uint4 v = *at;
    uint32_t* const w = &v.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
      if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu;
    }
    *at = v;
  }
}
// Over the chunks c0 .. c0 + count - 1 again, by a warp of the row group: NaN to a thread's outputs (its row of each chunk, columns from n0
// on, from the element o_at + t * o_step on) and dots that see an odd value of their chunk.
template <bool DOTS, bool WIDE>
__device__ __noinline__ void tc_spoil(const LaPass<float>& p, float* dots, int64_t b, int64_t h, int c0, int count, int len, int row,
                                      int n0, int64_t o_at, int64_t o_step) {
  const int columns = min(32, p.N - n0), lane = row & 31;
  for (int c = c0; c < c0 + count; ++c) {
    const int n = min(kTcChunk, len - c * kTcChunk);
    const unsigned short* const z =
        static_cast<const unsigned short*>(p.z) + b * p.zs[0] + h * p.zs[2] + (int64_t)c * kTcChunk * p.zs[1] + n0;
    auto odd_in = [&](int r) {
      uint32_t m = 0;
      for (int j = 0; j < columns; ++j)
        if ((z[r * p.zs[1] + j] & 0x7f80u) == 0x7f80u) m |= 1u << j;
      return m;
    };
    uint32_t odd = 0;
    for (int r = lane; r < n; r += 32) odd |= odd_in(r);
    if (!__any_sync(0xffffffffu, odd != 0)) continue;
    if (row < n) {   // it sees the tokens up to its own, mirrored: from its own on
      odd = 0;
      for (int r = p.reverse ? row : 0; r < (p.reverse ? n : row + 1); ++r) odd |= odd_in(r);
      const int64_t t = (int64_t)c * kTcChunk + row;
      for (int j = 0; j < columns; ++j)
        if (p.o && odd >> j & 1) {
          if (WIDE) static_cast<float*>(p.o)[o_at + t * o_step + j] = __int_as_float(0x7fffffff);
          else static_cast<unsigned short*>(p.o)[o_at + t * o_step + j] = 0x7fffu;
        }
      if (DOTS && odd) dots[t * 2] = __int_as_float(0x7fffffff);
    }
    __syncwarp();
  }
}

// WIDE: o holds float32 (its own kernel: what a kernel's loops hold of code has to stay in the instruction cache)
template <bool STATES_ONLY, bool DOTS, bool WIDE>
__global__ void __launch_bounds__(kTcThreads, 1) la_tc_kernel(const __grid_constant__ LaTcArgs k) {
  extern __shared__ __align__(1024) unsigned char tc_smem[];
  constexpr int C = kTcChunk;
  const LaArgs<float>& a = k.a;
  const int role = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const LaPass<float>& p = a.p[role];
  const int slices = (p.N + kTcSlice - 1) / kTcSlice;
  const int seg_count = STATES_ONLY ? a.nseg - (k.all_segments ? 0 : 1) : a.nseg;
  const int slice = (int)(blockIdx.x & 1);                       // two slots for slices: neighbours share x and y in L2
  const int ord = (int)((blockIdx.x >> 1) % seg_count);
  const int64_t bh = (blockIdx.x >> 1) / seg_count;
  // The passes with dots let the next kernel on the stream start beside them as soon as all their CTAs run; that kernel
  // may not end before them (what follows it reads the results of both), so its last CTA waits for their end.
  if (DOTS && tid == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const bool last_cta = !STATES_ONLY && !DOTS && tid == 0 && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1;
  if (slice >= slices) {
    if (last_cta) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  if (STATES_ONLY && k.all_segments && !p.fin && ord == a.nseg - 1) return;   // nobody asks for its end
  const int64_t b = bh / a.H, h = bh % a.H, BH = a.B * a.H;
  const int M = p.M, N = p.N, n0 = slice * kTcSlice;
  const bool rev = p.reverse;
  const int T = (int)a.T;   // below 2^31: the TMA unit's coordinates
  const int len = (int)la_length(a.lengths, b, a.T), nchunk = (int)(((int64_t)T + C - 1) / C);
  const int seg = rev ? a.nseg - 1 - ord : ord;
  const int c0 = seg * a.seg_chunks, c1 = min(c0 + a.seg_chunks, nchunk);
  // chunks with tokens: c0 .. c0 + count - 1, visited upwards or downwards
  const int count = max(0, min(c1, (int)(((int64_t)len + C - 1) / C)) - c0);
  const float* g = a.g + b * a.gs[0] + h * a.gs[2];
  auto chunk_of = [&](int i) { return c0 + (rev ? count - 1 - i : i); };
  auto valid = [&](int c) { return min(C, len - c * C); };

  const int nu = k.nu[role], ns = k.ns[role], sxy = k.xy_stages;
  const LaTcSmem L(sxy, DOTS, 3, DOTS ? 3 : 1);
  const uint32_t base = smem_u32(tc_smem);
  float* const Gs = reinterpret_cast<float*>(tc_smem + L.misc);              // [2][2][C] sums inside a block of 32, in two floats
  float* const cs = reinterpret_cast<float*>(tc_smem + L.misc + C * 16);     // [C] column factors
  TcFactors* const fac = reinterpret_cast<TcFactors*>(tc_smem + L.misc + C * 20);   // [2]
  uint64_t* const bars = reinterpret_cast<uint64_t*>(tc_smem + L.misc + C * 20 + 128);
  uint64_t *const xy_full = bars, *const xy_empty = bars + 2, *const zw_full = bars + 4, *const zw_empty = bars + 6;
  uint64_t *const b_sc = bars + 8, *const b_p = bars + 9, *const b_o = bars + 10, *const b_ofree = bars + 20;   // [2]
  uint64_t *const b_zw = bars + 12, *const b_u = bars + 13, *const b_s = bars + 14, *const b_oi = bars + 15;
  uint64_t *const lg_full = bars + 16, *const lg_empty = bars + 18;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
  volatile uint32_t* const gave_up = tmem_slot + 1;
  volatile uint32_t* const odd_seen = tmem_slot + 2;   // some z had an infinite or NaN value
  uint64_t* const b_end = bars + 24;
  // columns of tensor memory.  Without dots O and OI are double: a chunk's rows go out while the next one's weights are
  // formed; with dots the second scores take that place
  constexpr int kLag = DOTS ? 0 : 1;
  constexpr uint32_t kSC = 0, kP = 128, kO = 192, kOI = DOTS ? 256 : 320, kU = DOTS ? 320 : 448, kSC2 = 384;

  if (base & 1023) {   // the swizzled tiles need it; dynamic shared memory starts that way without static arrays
    if (tid == 0 && k.status) atomicOr(k.status, kErrPipelineWait);
    if (last_cta) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  if (warp == 16) tc_alloc(tmem_slot, 512);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(xy_full + i, 1);
      mbar_init(xy_empty + i, 1);
      mbar_init(zw_full + i, 1);
      mbar_init(zw_empty + i, DOTS ? 1 + 8 : 1);
      mbar_init(lg_full + i, 1);
      mbar_init(lg_empty + i, STATES_ONLY ? 8 : 16);
    }
    mbar_init(b_sc, 1);
    mbar_init(b_p, 8);   // one arrival a warp
    mbar_init(b_o, 1);
    mbar_init(b_ofree, 8);
    mbar_init(b_ofree + 1, 8);
    mbar_init(b_zw, 8);
    mbar_init(b_u, 1);
    mbar_init(b_s, 8);
    mbar_init(b_oi, 1);
    mbar_init(b_end, 1);
    *gave_up = 0;
    *odd_seen = 0;
    fence_mbar_init();
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tm = *tmem_slot;
  // a wait that runs out lets every other wait of the CTA fall through: all warps reach the end, results are invalid
  // and the status word says so.  No load is issued from then on: without the waits for their stages the loads would run away,
  // past what a barrier counts
  auto wait = [&](uint64_t* bar, uint32_t parity) {   // by one thread; short code: it is in every loop
    if (mbar_try_wait(bar, parity)) return;
    const long long start = clock64();
#pragma unroll 1
    while (!mbar_try_wait(bar, parity) && !*gave_up)
      if (clock64() - start > k.wait_cycles) *gave_up = 1;
  };
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) {   // by whole warps
    wait(bar, parity);
    __syncwarp();
  };
  auto arrive_warp = [&](uint64_t* bar) {   // for a whole warp, after what each of its threads did
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };

  if (warp == 17) {
    if (lane == 0) {   // loads
      int xy_sent = 0, zw_sent = 0;
#pragma unroll 1
      for (int i = 0; i < count; ++i) {
        const int t0 = chunk_of(i) * C, s = i % sxy, sz = i & 1;
        if (i >= sxy) wait(xy_empty + s, (i / sxy - 1) & 1);
        if (*gave_up) break;
        const uint32_t X = base + s * 4 * kTcPanel, Y = X + 2 * kTcPanel;
        mbar_arrive_expect_tx(xy_full + s, (STATES_ONLY ? 2 : 4) * kTcPanel);
        for (int q = 0; q < 2; ++q) {
          if (!STATES_ONLY)
            tc_tma(X + q * kTcPanel, &k.x[role].map, q * 64, t0, (int)h * k.x[role].hmul, (int)b * k.x[role].bmul, xy_full + s);
          tc_tma(Y + q * kTcPanel, &k.y[role].map, q * 64, t0, (int)h * k.y[role].hmul, (int)b * k.y[role].bmul, xy_full + s);
        }
        xy_sent = i + 1;
        if (i >= 2) wait(zw_empty + sz, (i / 2 - 1) & 1);
        if (*gave_up) break;
        const uint32_t Z = base + L.z + sz * (DOTS ? 2 : 1) * kTcPanel;
        mbar_arrive_expect_tx(zw_full + sz, (DOTS ? 2 : 1) * kTcPanel);
        tc_tma(Z, &k.z[role].map, n0, t0, (int)h * k.z[role].hmul, (int)b * k.z[role].bmul, zw_full + sz);
        if (DOTS) tc_tma(Z + kTcPanel, &k.w[role].map, n0, t0, (int)h * k.w[role].hmul, (int)b * k.w[role].bmul, zw_full + sz);
        zw_sent = i + 1;
      }
      // nothing is on its way when the CTA ends, whatever its waits came to
#pragma unroll 1
      for (int i = max(0, xy_sent - sxy); i < xy_sent; ++i)
        if (!mbar_wait_bounded(xy_full + i % sxy, (i / sxy) & 1, k.wait_cycles / 2)) *gave_up = 1;
#pragma unroll 1
      for (int i = max(0, zw_sent - 2); i < zw_sent; ++i)
        if (!mbar_wait_bounded(zw_full + (i & 1), (i / 2) & 1, k.wait_cycles / 2)) *gave_up = 1;
    }
  } else if (warp == 16) {
    {   // products: the warp stays together (operands in uniform registers), one thread issues
      const bool one = tc_elect();
      constexpr uint32_t kScD = tc_idesc(128, 128, false, false), kOD = tc_idesc(128, 64, false, true),
                         kUD = tc_idesc(128, 64, true, true);
      const uint32_t Zw = tc_desc(base + L.zw), S = tc_desc(base + L.s);
      const int steps = M > 64 ? 8 : 4;   // of 16 channels of x and y
      auto scores = [&](int i) {
        const int s = i % sxy, sz = i & 1;
        const uint32_t X = tc_desc(base + s * 4 * kTcPanel), Y = X + (2 * kTcPanel >> 4);
        wait_warp(xy_full + s, (i / sxy) & 1);
        tc_after();
        if (one) tc_products<kKMajor, kKMajor>(tm + kSC, X, Y, kScD, true, steps);
        if (DOTS) {
          const uint32_t Z = tc_desc(base + L.z + sz * 2 * kTcPanel);
          wait_warp(zw_full + sz, (i / 2) & 1);
          tc_after();
          if (one) tc_products<kKMajor, kKMajor>(tm + kSC2, Z + (kTcPanel >> 4), Z, kScD, true, 4);
        }
        if (one) tc_commit(b_sc);
      };
      if (!STATES_ONLY && count > 0) scores(0);
#pragma unroll 1
      for (int i = 0; i < count; ++i) {
        const int s = i % sxy, sz = i & 1;
        const uint32_t X = tc_desc(base + s * 4 * kTcPanel), Y = X + (2 * kTcPanel >> 4),
                       Z = tc_desc(base + L.z + sz * (DOTS ? 2 : 1) * kTcPanel), at = kLag ? (i & 1) * 64 : 0;
        if (STATES_ONLY) wait_warp(xy_full + s, (i / sxy) & 1);
        wait_warp(b_zw, i & 1);
        tc_after();
#pragma unroll 1
        for (int term = nu - 1; term >= 0; --term)   // smallest first
          if (one) tc_products<kMnMajor, kMnMajor>(tm + kU, Y, Zw + term * (kTcPanel >> 4), kUD, term == nu - 1);
        if (one) tc_commit(b_u);
        if (!STATES_ONLY) {
          wait_warp(b_s, i & 1);
          if (i > kLag) wait_warp(b_ofree + (kLag ? i & 1 : 0), (kLag ? (i >> 1) - 1 : i - 1) & 1);   // O and OI have been read
          tc_after();
#pragma unroll 1
          for (int term = ns - 1; term >= 0; --term)
            if (one) tc_products<kKMajor, kMnMajor>(tm + kOI + at, X, S + term * (kTcPanel >> 4), kOD, term == ns - 1, steps);
          if (one) tc_commit(b_oi);
        }
        if (one) tc_commit(xy_empty + s);
        if (!STATES_ONLY) {
          wait_warp(b_p, i & 1);
          tc_after();
          if (one) tc_products<kTmem, kMnMajor>(tm + kO + at, tm + kP, Z, kOD, true);
          if (one) tc_commit(b_o);
        }
        if (one) tc_commit(zw_empty + sz);
        if (!STATES_ONLY && i + 1 < count) scores(i + 1);
      }
      if (one) tc_commit(b_end);   // every product has ended, whatever the waits came to
      if (!mbar_wait_bounded(b_end, 0, k.wait_cycles / 2)) *gave_up = 1;
    }
  } else if (warp == 18) {   // decays
    float raw[4], next[4];
    double total = 0.0;
    if (count > 0) tc_load_logs(next, g, a.gs[1], (int64_t)chunk_of(0) * C, valid(chunk_of(0)), lane);
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j] = next[j];
      if (i + 1 < count) tc_load_logs(next, g, a.gs[1], (int64_t)chunk_of(i + 1) * C, valid(chunk_of(i + 1)), lane);
      if (i >= 2) wait_warp(lg_empty + (i & 1), ((i >> 1) - 1) & 1);
      tc_logs(Gs + (i & 1) * 2 * C, fac + (i & 1), raw, rev, lane, &total);
      arrive_warp(lg_full + (i & 1));
    }
    if (STATES_ONLY && slice == 0 && lane == 0)
      a.seg_log[(int64_t)(role * a.nseg + ord) * BH + bh] = total * 0.69314718055994531;   // natural
  } else if (warp < 8) {
    if constexpr (!STATES_ONLY) {   // rows
      const int quad = warp & 3, part = warp >> 2, row = 32 * quad + lane;   // two warps share 32 rows and take turns along them
      const uint32_t lanes = tm + ((uint32_t)(32 * quad) << 16);
      {   // blocks that hold no pair stay zero
        uint32_t zero[8] = {};
        for (int q = part; q < 8; q += 2)
          if (rev ? q < 2 * quad : q > 2 * quad + 1) tc_st8(lanes + kP + q * 8, zero);
      }
      const float scale_in = p.po * p.pz;
      float2 row_own;
      float row_mine, row_win, row_mid1, row_mid2, row_col;
      auto decays = [&](int i) {
        wait_warp(lg_full + (i & 1), (i >> 1) & 1);
        const float* const G = Gs + (i & 1) * 2 * C;
        const TcFactors& f = fac[i & 1];
        const float2 whole = make_float2(G[32 * quad + 31], G[C + 32 * quad + 31]);
        row_own = make_float2(G[row], G[C + row]);
        // from the token to its block's end, and from the block's start to it
        const float to_end = la_exp2(rev ? (row_own.x - whole.x) + (row_own.y - whole.y) : (whole.x - row_own.x) + (whole.y - row_own.y));
        const float to_start = la_exp2(rev ? -row_own.x : row_own.x);
        row_col = rev ? to_start : to_end;
        row_mine = rev ? to_end : to_start;
        row_win = row_mine * (rev ? f.after[quad] : f.before[quad]) * p.po;
        row_mid1 = rev ? (quad == 0 ? f.over[1] : f.over[2]) : (quad == 3 ? f.over[2] : f.over[1]);
        row_mid2 = f.over[1] * f.over[2];
      };
      if (count > 0) {
        decays(0);
        if (part == 0) cs[row] = row_col;
      }
      const uint32_t pairs = rev ? ~0u << lane : ~0u >> (31 - lane);   // columns of the own block that count
      const int64_t row_step = a.H * p.pitch, first_row = (b * a.T * a.H + h) * p.pitch + n0 + 32 * part;   // of the thread's columns
      // a chunk's rows to memory
      auto out = [&](int i, float win, float pair_sum) {
        const int t = chunk_of(i) * C + row, n = valid(chunk_of(i)), sz = i & 1;
        const uint32_t at = lanes + (kLag ? (i & 1) * 64 : 0) + part * 32;
        const int64_t first = first_row + (int64_t)t * row_step;
        const bool store = p.o && t < T;
        TcPair ext(0.f, 0.f);
        const TcPair win2(win, win), scale2(scale_in, scale_in);
        uint32_t vi[2][16], vo[2][16];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          tc_ld16(vi[q], at + kOI + q * 16);
          tc_ld16(vo[q], at + kO + q * 16);
        }
        tc_wait_ld();
        tc_before();
        arrive_warp(b_ofree + (kLag ? i & 1 : 0));   // the products may overwrite
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            TcPair r[4];
            const int piece = 2 * (2 * part + q) + e, col = q * 16 + e * 8;   // of a row of Z; of the thread's columns
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = tc_pair(vi[q][e * 8 + 2 * j], vi[q][e * 8 + 2 * j + 1]) * win2;
            if (DOTS) {
              const uint4 wv = *reinterpret_cast<const uint4*>(tc_smem + L.z + (sz * 2 + 1) * kTcPanel + row * 128 +
                                                              ((piece ^ (row & 7)) << 4));
              ext = fma2(r[0], tc_widen(wv.x), fma2(r[1], tc_widen(wv.y), fma2(r[2], tc_widen(wv.z), fma2(r[3], tc_widen(wv.w), ext))));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = fma2(tc_pair(vo[q][e * 8 + 2 * j], vo[q][e * 8 + 2 * j + 1]), scale2, r[j]);
            if (store && n0 + piece * 8 < N) {
              if (WIDE) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const float2 v0 = r[2 * j].get(), v1 = r[2 * j + 1].get();
                  float4 v = make_float4(v0.x, v0.y, v1.x, v1.y);
                  if (row >= n) v = make_float4(0.f, 0.f, 0.f, 0.f);
                  *reinterpret_cast<float4*>(static_cast<float*>(p.o) + first + col + j * 4) = v;
                }
              } else {
                uint4 pk = make_uint4(tc_pack(r[0]), tc_pack(r[1]), tc_pack(r[2]), tc_pack(r[3]));
                if (row >= n) pk = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.o) + first + col) = pk;
              }
            }
          }
        }
        if (DOTS) {
          arrive_warp(zw_empty + sz);
          if (row < n) {
            float2* d = reinterpret_cast<float2*>(p.dots + ((((int64_t)slice * 2 + part) * BH + bh) * a.T + t) * 2);
            const float2 e = ext.get();
            *d = make_float2(pair_sum * scale_in, e.x + e.y);
          }
        }
      };
      float last_win = 0.f;
#pragma unroll 1
      for (int i = 0; i < count; ++i) {
        const int n = valid(chunk_of(i));
        const float* const G = Gs + (i & 1) * 2 * C;
        const TcPair own_hi(row_own.x, row_own.x), own_lo(row_own.y, row_own.y);
        const float mine = row_mine, win = row_win, mid1 = row_mid1, mid2 = row_mid2;
        if (i > 0 && kLag) {   // P has been read, and every row is past its use of the last factors
          wait_warp(b_o, (i - 1) & 1);
          if (part == 0) cs[row] = row_col;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");   // every row's factors are written
        wait_warp(b_sc, i & 1);
        tc_after();
        float rowsum = 0.f;
        // (loops, not unrolled code: straight-line code this long would run at the rate of the instruction fetch)
        const int q0 = rev ? 2 * quad : 0, q1 = rev ? 8 : 2 * quad + 2;
#pragma unroll 1
        for (int q = q0 + part; q < q1; q += 2) {   // 16 columns at a time
          uint32_t v[16], u[16];
          tc_ld16(v, lanes + kSC + q * 16);
          if (DOTS) tc_ld16(u, lanes + kSC2 + q * 16);
          tc_wait_ld();
          if (q >> 1 == quad) {
            const uint32_t on = pairs >> ((q & 1) * 16);
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float2 e = ((own_hi - TcPair(*reinterpret_cast<const uint64_t*>(G + q * 16 + j))) +
                                (own_lo - TcPair(*reinterpret_cast<const uint64_t*>(G + C + q * 16 + j)))).get();
              const float2 w = (tc_pair(v[j], v[j + 1]) * tc_pair(la_exp2(e.x), la_exp2(e.y))).get();
              v[j] = on >> j & 1 ? __float_as_uint(w.x) : 0u;
              v[j + 1] = on >> (j + 1) & 1 ? __float_as_uint(w.y) : 0u;
            }
          } else {
            const int between = (rev ? (q >> 1) - quad : quad - (q >> 1)) - 1;
            const float from1 = mine * (between == 0 ? 1.f : between == 1 ? mid1 : mid2);
            const TcPair from(from1, from1);
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const TcPair c2(*reinterpret_cast<const uint64_t*>(cs + q * 16 + j));
              const float2 w = (tc_pair(v[j], v[j + 1]) * (from * c2)).get();
              v[j] = __float_as_uint(w.x);
              v[j + 1] = __float_as_uint(w.y);
            }
          }
          if (rev && q * 16 + 16 > n) {   // tokens behind the end are not read: they may be infinite or NaN
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (q * 16 + j >= n) v[j] = 0u;
          }
          if (DOTS) {   // pairs of two tokens of the chunk; the diagonal would cancel between q.dq and k.dk
#pragma unroll
            for (int j = 0; j < 16; ++j)
              rowsum += v[j] != 0u && q * 16 + j != row ? __uint_as_float(v[j]) * __uint_as_float(u[j]) : 0.f;
          }
          uint32_t out[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) out[j] = la_pack(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
          tc_st8(lanes + kP + q * 8, out);
        }
        tc_wait_st();
        tc_before();
        arrive_warp(b_p);
        if (lane == 0) mbar_arrive(lg_empty + (i & 1));
        if (i + 1 < count) decays(i + 1);
        if (kLag) {
          if (i > 0) out(i - 1, last_win, 0.f);   // while this chunk's products run
          last_win = win;
        } else {
          wait_warp(b_o, i & 1);
          tc_after();
          if (part == 0 && i + 1 < count) cs[row] = row_col;   // every row is past its use of the last ones
          out(i, win, rowsum);
        }
      }
      if (kLag && count > 0) {
        wait_warp(b_o, (count - 1) & 1);
        tc_after();
        out(count - 1, last_win, 0.f);
      }
      if (__any_sync(0xffffffffu, *odd_seen))
        tc_spoil<DOTS, WIDE>(p, p.dots + (((int64_t)slice * 2 + part) * BH + bh) * a.T * 2, b, h, c0, count, len, row, n0 + 32 * part,
                             first_row, row_step);
      // behind the sequence: zeros
      if (p.o) {
        const int64_t begin = (int64_t)(c0 + count) * C, stop = min(a.T, (int64_t)c1 * C);
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const int pieces = min(8, (p.pitch - n0) / 8) * (WIDE ? 2 : 1), per = WIDE ? 4 : 8;
        for (int64_t t = begin + tid; t < stop; t += kTcRows)
          for (int q = 0; q < pieces; ++q) {
            const int64_t at = (b * a.T * a.H + h) * p.pitch + t * row_step + n0 + q * per;
            *reinterpret_cast<uint4*>(static_cast<char*>(p.o) + at * (16 / per)) = zero;
          }
      }
    }
  } else {   // state: two threads hold a row m, 32 columns each
    const int quad = warp & 3, part = (warp >> 2) & 1, row = 32 * quad + lane, m = row, nc = n0 + 32 * part;
    const uint32_t lanes = tm + ((uint32_t)(32 * quad) << 16);
    float st[32];
    {
      const float* src = nullptr;
      int64_t ms = 0, nstr = 0;
      bool on = true;
      if (!STATES_ONLY && ord > 0) {   // padded, [n][m]
        src = a.seg + ((int64_t)(role * (a.nseg + 1) + ord) * BH + bh) * a.seg_stride;
        ms = 1; nstr = kTcDim;
      } else if (!STATES_ONLY && p.init) {
        src = p.init + bh * M * N;
        ms = p.state_t ? 1 : N; nstr = p.state_t ? M : 1;
        on = m < M;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) st[j] = (src && on && nc + j < N) ? src[m * ms + (nc + j) * nstr] : 0.f;
    }
    float wt = 0.f;
    float2 dec = make_float2(1.f, 0.f), dec_now = dec;
    auto decays = [&](int i) {   // chunk i's: the weight with which token `row` joins the state, the decay over the chunk
      wait_warp(lg_full + (i & 1), (i >> 1) & 1);
      const float* const G = Gs + (i & 1) * 2 * C;
      const TcFactors& f = fac[i & 1];
      const float2 own = make_float2(G[row], G[C + row]), whole = make_float2(G[32 * quad + 31], G[C + 32 * quad + 31]);
      wt = (rev ? la_exp2(-own.x) * f.before[quad] : la_exp2((whole.x - own.x) + (whole.y - own.y)) * f.after[quad]) * p.pz;
      dec_now = make_float2(f.dec[0], f.dec[1]);
      arrive_warp(lg_empty + (i & 1));
    };
    if (count > 0) decays(0);
    auto advance = [&](int i) {   // S <- exp(E) S + U of chunk i
      const TcPair dec_hi(dec.x, dec.x), dec_lo(dec.y, dec.y);
      wait_warp(b_u, i & 1);
      tc_after();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t u[16];
        tc_ld16(u, lanes + kU + part * 32 + q * 16);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const TcPair v = tc_pair(u[j], u[j + 1]);
          const TcPair old = tc_pair(st[q * 16 + j], st[q * 16 + j + 1]);
          const float2 now = fma2(dec_hi, old, fma2(dec_lo, old, v)).get();
          st[q * 16 + j] = now.x;
          st[q * 16 + j + 1] = now.y;
        }
      }
      tc_before();
    };
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      const int c = chunk_of(i);
      const int n = valid(c), sz = i & 1, s = i % sxy;
      if (i > 0) advance(i - 1);
      dec = dec_now;
      wait_warp(zw_full + sz, (i / 2) & 1);
      {
        const int zoff = L.z + sz * (DOTS ? 2 : 1) * kTcPanel + row * 128;
        if (row >= n) {   // what lies behind the sequence is not read: it may be infinite or NaN
          wait(xy_full + s, (i / sxy) & 1);
          const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 1
          for (int q = 0; q < 8; ++q) {   // (two threads write the same zeros)
            *reinterpret_cast<uint4*>(tc_smem + zoff + q * 16) = zero;
            *reinterpret_cast<uint4*>(tc_smem + s * 4 * kTcPanel + 2 * kTcPanel + row * 128 + q * 16) = zero;
            *reinterpret_cast<uint4*>(tc_smem + s * 4 * kTcPanel + 3 * kTcPanel + row * 128 + q * 16) = zero;
          }
        }
        unsigned char* const zw = tc_smem + L.zw + row * 128;
        const TcPair wt2(wt, wt);
        __nv_bfloat162 most = __floats2bfloat162_rn(0.f, 0.f);   // largest magnitudes: infinite or NaN where a value is
#pragma unroll 1
        for (int q = 4 * part; q < 4 * part + 4; ++q) {
          const int at = (q ^ (row & 7)) << 4;
          const uint4 zv = *reinterpret_cast<const uint4*>(tc_smem + zoff + at);
          const uint32_t in[4] = {zv.x, zv.y, zv.z, zv.w};
          uint32_t t[4];
          TcPair v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = tc_widen(in[e]) * wt2;
            if (!STATES_ONLY) most = __hmax2_nan(most, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&in[e])));
            t[e] = tc_pack(v[e]);
          }
          *reinterpret_cast<uint4*>(zw + at) = make_uint4(t[0], t[1], t[2], t[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = v[e] - tc_widen(t[e]);
            t[e] = tc_pack(v[e]);
          }
          *reinterpret_cast<uint4*>(zw + kTcPanel + at) = make_uint4(t[0], t[1], t[2], t[3]);
          if (nu == 3) {
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = tc_pack(v[e] - tc_widen(t[e]));
            *reinterpret_cast<uint4*>(zw + 2 * kTcPanel + at) = make_uint4(t[0], t[1], t[2], t[3]);
          }
        }
        if constexpr (!STATES_ONLY) {
          if (!(__low2float(most) < INFINITY && __high2float(most) < INFINITY)) {
            tc_take_out(tc_smem + zoff, row, part);
            *odd_seen = 1;
          }
        }
      }
      fence_proxy_async_smem();
      arrive_warp(b_zw);
      if constexpr (!STATES_ONLY) {
        if (i > 0) wait_warp(b_oi, (i - 1) & 1);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          unsigned char* const sp = tc_smem + L.s + row * 128 + (((4 * part + q) ^ (row & 7)) << 4);
          uint32_t v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = la_pack(st[q * 8 + 2 * e], st[q * 8 + 2 * e + 1]);
          *reinterpret_cast<uint4*>(sp) = make_uint4(v[0], v[1], v[2], v[3]);
          if (DOTS) {
            uint32_t v1[4], v2[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const TcPair r = tc_pair(st[q * 8 + 2 * e], st[q * 8 + 2 * e + 1]) - tc_widen(v[e]);
              v1[e] = tc_pack(r);
              v2[e] = tc_pack(r - tc_widen(v1[e]));
            }
            *reinterpret_cast<uint4*>(sp + kTcPanel) = make_uint4(v1[0], v1[1], v1[2], v1[3]);
            *reinterpret_cast<uint4*>(sp + 2 * kTcPanel) = make_uint4(v2[0], v2[1], v2[2], v2[3]);
          }
        }
        fence_proxy_async_smem();
        arrive_warp(b_s);
        if (DOTS && p.bounds) {   // [n][m], rows of a multiple of four (the padding is zero)
          const int pitch = la_tc_bound_pitch(M);
          float* dst = p.bounds + (bh * nchunk + c) * N * pitch + (int64_t)nc * pitch + m;
          if (pitch == kTcDim && nc + 32 <= N) {   // (steps known beforehand: 8 us less of 362 at B=2, T=4096, H=16, D=128)
#pragma unroll
            for (int j = 0; j < 32; ++j) dst[j * kTcDim] = st[j];
          } else if (m < pitch) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (nc + j < N) dst[j * pitch] = st[j];
          }
        }
      }
      if (i + 1 < count) decays(i + 1);   // while the products run
    }
    if (count > 0) advance(count - 1);
    if (STATES_ONLY) {
      float* dst = a.seg + ((int64_t)(role * (a.nseg + 1) + ord + 1) * BH + bh) * a.seg_stride + (int64_t)nc * kTcDim + m;
#pragma unroll
      for (int j = 0; j < 32; ++j) dst[j * kTcDim] = st[j];
    } else if (p.fin && ord == a.nseg - 1 && !k.all_segments && m < M) {
      float* dst = p.fin + bh * M * N;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (nc + j < N) dst[p.state_t ? (int64_t)(nc + j) * M + m : (int64_t)m * N + nc + j] = st[j];
    }
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == 16) tc_dealloc(tm, 512);
  if (tid == 0 && *gave_up && k.status) atomicOr(k.status, kErrPipelineWait);
  if (last_cta) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Entering states of the segments (slots [role][nseg + 1] of padded [n][m] matrices): seg[d+1] = exp(log decay of
// segment d) * seg[d] + (what segment d added); with all_segments the last one is the final state.
__global__ void la_tc_join_kernel(const LaArgs<float> a, int all_segments) {
  const int role = blockIdx.y;
  const LaPass<float>& p = a.p[role];
  const int64_t BH = a.B * a.H, e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, bh = e / (kTcDim * kTcDim);
  if (bh >= BH) return;
  const int i = (int)(e % (kTcDim * kTcDim)), n = i / kTcDim, m = i % kTcDim;
  const bool on = m < p.M && n < p.N;
  const int64_t at = bh * p.M * p.N + (p.state_t ? n * p.M + m : m * p.N + n);
  float v = p.init && on ? p.init[at] : 0.f;
  const int count = a.nseg - (all_segments && p.fin ? 0 : 1);
  const double* log = a.seg_log + (int64_t)role * a.nseg * BH + bh;
  float* slot = a.seg + ((int64_t)(role * (a.nseg + 1) + 1) * BH + bh) * a.seg_stride + i;
  double lg = *log;
  float more = *slot;
  for (int d = 0; d < count; ++d) {
    const LaDecay<float> dec = LaDecay<float>::of_chunk(lg);
    const float add = more;
    float* const at = slot;
    if (d + 1 < count) {   // the next segment's values are on their way while this one's are worked on
      lg = *(log += BH);
      more = *(slot += BH * a.seg_stride);
    }
    v = dec(v, add);
    *at = v;
  }
  if (all_segments && p.fin && on) p.fin[at] = v;
}

// Rows moved between layouts: operands that the TMA unit cannot address (rows that do not start on 16 bytes) to rows
// that do, and results from such rows to dense ones.  U: the widest access that all rows allow.  A CTA takes 64 rows,
// whose starts it works out once; its threads then take neighbouring units, so that loads and stores are contiguous.
// What lies between a row's end and the next one's start is never read.
// Measured: q, k, v of B=4, T=2048, H=16, D=60 (8-byte units, 94 MB read and written) 22 us, o 7 us; B=4, T=512, H=8,
// 65 and 127 channels (2-byte units) 11 us.
constexpr int kLaMoveRows = 64;
struct LaMoveArgs {
  const char* src[4];
  char* dst[4];
  int64_t st[4][3], pitch[4];   // bytes: (B, T, H) strides of src, step from row to row of dst
  int width[4];                 // bytes of a row
  int64_t T, H, rows;
};
template <class U>
__global__ void __launch_bounds__(256) la_move_kernel(const LaMoveArgs a) {
  __shared__ int64_t start[kLaMoveRows];
  const int k = blockIdx.y, tid = threadIdx.x;
  const int64_t r0 = (int64_t)blockIdx.x * kLaMoveRows;
  const int rows = (int)min((int64_t)kLaMoveRows, a.rows - r0);
  if (tid < rows) {
    const int64_t r = r0 + tid, bt = r / a.H, h = r - bt * a.H, b = bt / a.T, t = bt - b * a.T;
    start[tid] = b * a.st[k][0] + t * a.st[k][1] + h * a.st[k][2];
  }
  __syncthreads();
  const unsigned units = a.width[k] / (int)sizeof(U);
  char* const dst = a.dst[k] + r0 * a.pitch[k];
  for (unsigned i = tid; i < rows * units; i += 256) {
    const unsigned r = i / units, at = (i - r * units) * (unsigned)sizeof(U);
    *reinterpret_cast<U*>(dst + r * a.pitch[k] + at) = *reinterpret_cast<const U*>(a.src[k] + start[r] + at);
  }
}

}  // namespace ptb
