// C ABI of linear attention with decays (see include/philtorch_b200.h).
#include "linear_attention.cuh"
#include "linear_attention_tc.cuh"

namespace ptb {

template <class S> struct LaGeom;
template <> struct LaGeom<float> { static constexpr int C = 32, NS = 64, PER_SM = 2; };
template <> struct LaGeom<double> { static constexpr int C = 32, NS = 32, PER_SM = 1; };

constexpr int kLaSms = 148;   // CTAs to aim for; only the cut of the time axis depends on it, never a result's meaning

struct LaPlan {
  int C, nseg, seg_chunks;
  int64_t nchunk, seg_off, log_off, qb_off, rb_off, qd_off, kd_off, part_off, total;
  int64_t seg_stride, bound_elems, copy_off[4], out_off[3];
};

// Few (batch, head) pairs: the time axis is cut into segments that run side by side.  Their entering states
// come from a first pass that only forms states (about half the work of a chunk), so a cut into n segments takes
// about 1.5 / n of the time plus two launches.  least: the n from which it pays.  Measured: 2 on the CUDA cores (float32
// training step (2, 509, 3, 33/65): 137 -> 42 us per direction); on the tensor cores two segments of 64 (batch,
// head, slice) CTAs take 89 us against 80 uncut (2, 4096, 16, 128), so 3.
static void la_cut(int64_t ctas, int64_t nchunk, int64_t room, int64_t least, int* nseg, int* seg_chunks) {
  int64_t n = ctas > 0 ? std::min(room / ctas, nchunk / 2) : 1;
  if (n < least || nchunk < 8) n = 1;
  const int64_t per = n > 1 ? (nchunk + n - 1) / n : std::max<int64_t>(nchunk, 1);
  *seg_chunks = (int)per;
  *nseg = n > 1 ? (int)((nchunk + per - 1) / per) : 1;
}

struct LaSize { int64_t B, T, H, Dk, Dv; };

// C: tokens of a chunk; width: columns of a state that a CTA takes; mn, bound: scalars of a segment's state and of one at a chunk's
// end; groups: of threads that share a token's sum for the decays' gradient
template <class S>
static LaPlan la_plan(const LaSize& z, int roles, bool decay_grad, int C, int width, int64_t mn, int64_t bound, int groups,
                      int per_sm, int slots) {
  LaPlan l = {};
  l.C = C;
  const int64_t over_k = (z.Dk + width - 1) / width, over_v = (z.Dv + width - 1) / width;
  const int64_t slices = roles == 1 ? over_v : 2 * over_k + over_v;   // of o; of dq, dk and dv
  l.nchunk = (z.T + C - 1) / C;
  const int64_t BH = z.B * z.H;
  la_cut(BH * slices, l.nchunk, kLaSms * per_sm, C == kTcChunk ? 3 : 2, &l.nseg, &l.seg_chunks);
  l.seg_stride = align_up(mn, 64);
  l.bound_elems = bound;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at = align_up(at + bytes, 256); return o; };
  l.seg_off = take(l.nseg > 1 ? (int64_t)roles * (l.nseg + slots) * BH * l.seg_stride * sizeof(S) : 0);
  l.log_off = take(l.nseg > 1 ? (int64_t)roles * l.nseg * BH * sizeof(double) : 0);
  l.qb_off = take(decay_grad ? BH * l.nchunk * bound * sizeof(S) : 0);
  l.rb_off = take(decay_grad ? BH * l.nchunk * bound * sizeof(S) : 0);
  l.qd_off = take(decay_grad ? groups * over_k * BH * z.T * 2 * sizeof(S) : 0);   // of the passes whose columns are Dk
  l.kd_off = take(decay_grad ? groups * over_k * BH * z.T * 2 * sizeof(S) : 0);
  l.part_off = take(decay_grad ? BH * l.nchunk * sizeof(double) : 0);
  l.total = at;
  return l;
}
template <class S>
static LaPlan la_simt_plan(const LaSize& z, int roles, bool decay_grad) {
  using G = LaGeom<S>;
  return la_plan<S>(z, roles, decay_grad, G::C, G::NS, z.Dk * z.Dv, z.Dk * z.Dv, 1, G::PER_SM, 0);
}
static LaPlan la_tc_plan(const LaSize& z, int roles, bool decay_grad, int copies) {
  LaPlan l = la_plan<float>(z, roles, decay_grad, kTcChunk, kTcSlice, kTcDim * kTcDim, z.Dk * la_tc_bound_pitch((int)z.Dv), 2, 1, 1);
  auto take = [&](int64_t D, int size) {
    const int64_t o = l.total;
    l.total += align_up(z.B * z.T * z.H * align_up(D, 8) * size, 256);
    return o;
  };
  for (int k = 0; k < 4; ++k)   // q, k, v, grad_o on rows that start on 16 bytes
    if (copies >> k & 1) l.copy_off[k] = take(k < 2 ? z.Dk : z.Dv, 2);
  if (roles == 1) {
    if (z.Dv % 8) l.out_off[0] = take(z.Dv, 4);   // o, which may be float32
  } else {
    for (int r = 0; r < 3; ++r)   // dq, dk, dv
      if ((r < 2 ? z.Dk : z.Dv) % 8) l.out_off[r] = take(r < 2 ? z.Dk : z.Dv, 2);
  }
  return l;
}
template <class S>
static LaPlan la_plan_of(bool tensor_cores, const LaSize& z, int roles, bool decay_grad, int copies) {
  if constexpr (std::is_same<S, float>::value)
    if (tensor_cores) return la_tc_plan(z, roles, decay_grad, copies);
  return la_simt_plan<S>(z, roles, decay_grad);
}

// bfloat16 runs on the tensor cores but for one chunk of the CUDA-core kernels: as fast there (B=1, H=4, D=64, T=1: 9.2
// against 11.4 us; T=64: 16.1 against 10.3), and where an output is a sum of a few terms, the rounding of their
// weights to bfloat16 would not average out.
template <class T>
static int64_t la_cuda_core_tokens() {   // the most that they take
  return std::is_same<T, __nv_bfloat16>::value ? LaGeom<float>::C : INT64_MAX;
}
template <class T>
static bool la_tensor_cores(int64_t tokens) { return tokens > la_cuda_core_tokens<T>(); }

template <class T, class S, int MD, bool STATES_ONLY>
static int la_simt_launch(const LaArgs<S>& a, int roles, cudaStream_t st) {
  using G = LaGeom<S>;
  constexpr int smem = sizeof(LaSimtSmem<S, G::C, G::NS, MD>);
  static bool ready[kMaxDevices] = {};
  int dev = 0;
  PTB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return PTB_ERR_ARG;
  {
    std::lock_guard<std::mutex> lock(init_mutex());
    if (!ready[dev]) {
      PTB_CUDA(cudaFuncSetAttribute(la_simt_kernel<T, S, G::C, G::NS, MD, STATES_ONLY>,
                                    cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      ready[dev] = true;
    }
  }
  const int64_t grid = a.B * a.H * (STATES_ONLY ? a.nseg - 1 : a.nseg) * ((kLaMaxDim + G::NS - 1) / G::NS);
  if (grid > 0x7fffffffll) return PTB_ERR_TOO_LARGE;
  la_simt_kernel<T, S, G::C, G::NS, MD, STATES_ONLY><<<dim3((unsigned)grid, roles), 256, smem, st>>>(a);
  PTB_CUDA(cudaGetLastError());
  return PTB_OK;
}

template <class S>
static void la_workspace(LaArgs<S>& a, const LaPlan& l, void* ws) {
  char* w = static_cast<char*>(ws);
  a.nseg = l.nseg;
  a.seg_chunks = l.seg_chunks;
  a.seg_stride = l.seg_stride;
  a.seg = reinterpret_cast<S*>(w + l.seg_off);
  a.seg_log = reinterpret_cast<double*>(w + l.log_off);
}

template <class T, class S, int MD>
static int la_simt_run(LaArgs<S>& a, int roles, cudaStream_t st) {
  if (a.nseg > 1) {
    if (int rc = la_simt_launch<T, S, MD, true>(a, roles, st)) return rc;
    const int64_t elems = a.B * a.H * (int64_t)a.p[0].M * a.p[0].N;
    la_join_kernel<S><<<dim3((unsigned)((elems + 255) / 256), roles), 256, 0, st>>>(a);
    PTB_CUDA(cudaGetLastError());
  }
  return la_simt_launch<T, S, MD, false>(a, roles, st);
}

// ---- tcgen05 kernels
// (Dv | Dk, T, H, B) view of an operand, box 64 x 128 tokens; an axis of stride zero (or of one entry) is left out
static int la_tc_map(LaTcMap* m, const void* base, const int64_t* st, int64_t B, int64_t T, int64_t H, int64_t D) {
  m->bmul = B > 1 && st[0] != 0;
  m->hmul = H > 1 && st[2] != 0;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)T, (cuuint64_t)(m->hmul ? H : 1), (cuuint64_t)(m->bmul ? B : 1)};
  const cuuint64_t strides[3] = {(cuuint64_t)st[1] * 2, (cuuint64_t)(m->hmul ? st[2] * 2 : 16), (cuuint64_t)(m->bmul ? st[0] * 2 : 16)};
  if (!aligned16(base) || st[1] == 0) return PTB_ERR_ARG;
  for (cuuint64_t v : strides)
    if (v % 16 || v >= (1ull << 40)) return PTB_ERR_ARG;
  const cuuint32_t box[4] = {64u, (cuuint32_t)kTcChunk, 1u, 1u};
  const CUresult r = encode_tiled(&m->map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (r == CUDA_SUCCESS) return PTB_OK;
  g_last_cuda_error = (int)r;
  return PTB_ERR_CUDA;
}

static int la_tc_setup(LaTcArgs* k, const LaArgs<float>& a, int roles) {
  for (int r = 0; r < roles; ++r) {
    const LaPass<float>& p = a.p[r];
    if (!aligned16(p.o)) return PTB_ERR_ARG;   // written in pieces of 16 bytes
    if (int rc = la_tc_map(&k->x[r], p.x, p.xs, a.B, a.T, a.H, p.M)) return rc;
    if (int rc = la_tc_map(&k->y[r], p.y, p.ys, a.B, a.T, a.H, p.M)) return rc;
    if (int rc = la_tc_map(&k->z[r], p.z, p.zs, a.B, a.T, a.H, p.N)) return rc;
    if (p.w)
      if (int rc = la_tc_map(&k->w[r], p.w, p.ws, a.B, a.T, a.H, p.N)) return rc;
  }
  return PTB_OK;
}

// n arrays of rows, moved in one launch
static int la_move(LaMoveArgs& m, int n, const LaSize& z, cudaStream_t st) {
  if (n == 0) return PTB_OK;
  m.T = z.T;
  m.H = z.H;
  m.rows = z.B * z.T * z.H;
  uint64_t bits = 16;
  for (int i = 0; i < n; ++i) {
    bits |= reinterpret_cast<uintptr_t>(m.src[i]) | reinterpret_cast<uintptr_t>(m.dst[i]) | m.width[i] | m.pitch[i] | m.st[i][1];
    if (z.B > 1) bits |= m.st[i][0];
    if (z.H > 1) bits |= m.st[i][2];
  }
  const int64_t ctas = (m.rows + kLaMoveRows - 1) / kLaMoveRows;
  if (ctas > 0x7fffffffll) return PTB_ERR_TOO_LARGE;
  const dim3 grid((unsigned)ctas, n);
  switch (bits & (~bits + 1)) {   // the largest power of two that divides all of them
    case 16: la_move_kernel<uint4><<<grid, 256, 0, st>>>(m); break;
    case 8: la_move_kernel<uint2><<<grid, 256, 0, st>>>(m); break;
    case 4: la_move_kernel<uint32_t><<<grid, 256, 0, st>>>(m); break;
    default: la_move_kernel<uint16_t><<<grid, 256, 0, st>>>(m); break;
  }
  PTB_CUDA(cudaGetLastError());
  return PTB_OK;
}

// q, k, v, grad_o of a call; those marked in `copies` move to the workspace, on rows that start on 16 bytes
struct LaOperands {
  const void* p[4];
  int64_t st[4][3];
};
static int la_copy_in(LaOperands* o, int copies, const LaSize& z, const LaPlan& l, void* ws, cudaStream_t st) {
  LaMoveArgs m = {};
  int n = 0;
  for (int k = 0; k < 4; ++k) {
    if (!(copies >> k & 1) || !o->p[k]) continue;
    const int64_t D = k < 2 ? z.Dk : z.Dv, P = align_up(D, 8);
    m.src[n] = static_cast<const char*>(o->p[k]);
    m.dst[n] = static_cast<char*>(ws) + l.copy_off[k];
    for (int i = 0; i < 3; ++i) m.st[n][i] = o->st[k][i] * 2;
    m.width[n] = (int)D * 2;
    m.pitch[n] = P * 2;
    o->p[k] = m.dst[n++];
    o->st[k][0] = z.T * z.H * P;
    o->st[k][1] = z.H * P;
    o->st[k][2] = P;
  }
  return la_move(m, n, z, st);
}

// The rows of results whose head size is no multiple of eight are written to the workspace, as whole 16-byte pieces,
// and moved from there: written in place, element by element, they cost four times the kernel's own time (B=4, T=2048,
// H=16, D=60: 202 against 44 us).
template <class S>
static LaMoveArgs la_results(LaArgs<S>& a, int roles, const LaPlan& l, void* ws, int* n) {
  LaMoveArgs m = {};
  *n = 0;
  for (int r = 0; r < roles; ++r) {
    LaPass<S>& p = a.p[r];
    p.pitch = (int)align_up(p.N, 8);
    if (!p.o || p.pitch == p.N) continue;
    const int64_t size = p.wide ? 4 : 2, P = p.pitch * size;
    m.dst[*n] = static_cast<char*>(p.o);
    p.o = static_cast<char*>(ws) + l.out_off[p.out];
    m.src[*n] = static_cast<const char*>(p.o);
    m.st[*n][0] = a.T * a.H * P;
    m.st[*n][1] = a.H * P;
    m.st[*n][2] = P;
    m.width[*n] = (int)(p.N * size);
    m.pitch[*n] = p.N * size;
    ++*n;
  }
  return m;
}

// beside: may start while the kernel launched before it on the stream is running (it reads nothing that one writes)
template <bool STATES_ONLY, bool DOTS, bool WIDE = false>
static int la_tc_launch(const LaTcArgs& k, int roles, cudaStream_t st, bool beside = false) {
  static bool ready[kMaxDevices] = {};
  int dev = 0;
  PTB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return PTB_ERR_ARG;
  const int smem = LaTcSmem(k.xy_stages, DOTS, 3, DOTS ? 3 : 1).total;
  {
    std::lock_guard<std::mutex> lock(init_mutex());
    if (!ready[dev]) {
      PTB_CUDA(cudaFuncSetAttribute(la_tc_kernel<STATES_ONLY, DOTS, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      ready[dev] = true;
    }
  }
  const int64_t grid = k.a.B * k.a.H * 2 * (STATES_ONLY ? k.a.nseg - (k.all_segments ? 0 : 1) : k.a.nseg);
  if (grid > 0x7fffffffll) return PTB_ERR_TOO_LARGE;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, roles);
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = beside ? 1 : 0;
  PTB_CUDA(cudaLaunchKernelEx(&cfg, la_tc_kernel<STATES_ONLY, DOTS, WIDE>, k));
  return PTB_OK;
}

// The roles with dots come first, then those without
static int la_tc_run(LaTcArgs& k, int roles, cudaStream_t st) {
  const LaArgs<float>& a = k.a;
  bool dots = false;
  for (int r = 0; r < roles; ++r) {
    const bool exact = a.p[r].dots, end = a.p[r].fin && !exact;
    dots = dots || exact;
    k.ns[r] = exact ? 3 : 1;
    k.nu[r] = exact || end ? 3 : 2;
    if (end && a.nseg > 1) k.all_segments = 1;
  }
  if (a.nseg > 1) {
    k.xy_stages = 2;
    if (int rc = la_tc_launch<true, false>(k, roles, st)) return rc;
    const int64_t elems = a.B * a.H * kTcDim * kTcDim;
    if (elems / 256 > 0x7fffffffll) return PTB_ERR_TOO_LARGE;
    la_tc_join_kernel<<<dim3((unsigned)((elems + 255) / 256), roles), 256, 0, st>>>(a, k.all_segments);
    PTB_CUDA(cudaGetLastError());
    for (int r = 0; r < roles; ++r)   // the segments' states are known: the update needs no float32 end any more
      if (!a.p[r].dots) k.nu[r] = 2;
  }
  if (!dots) {
    k.xy_stages = 2;
    return a.p[0].wide ? la_tc_launch<false, false, true>(k, roles, st) : la_tc_launch<false, false>(k, roles, st);
  }
  // the passes with dots, then, beside them, the others (another use of the shared memory).  One launch after the other
  // leaves SMs idle twice: 96 and 48 CTAs at B=1, T=32768, H=4
  LaTcArgs part = k;
  int with = 0, without = 0;
  LaTcArgs plain = k;
  for (int r = 0; r < roles; ++r) {
    LaTcArgs& to = a.p[r].dots ? part : plain;
    const int at = a.p[r].dots ? with++ : without++;
    to.a.p[at] = a.p[r];
    to.x[at] = k.x[r]; to.y[at] = k.y[r]; to.z[at] = k.z[r]; to.w[at] = k.w[r];
    to.nu[at] = k.nu[r]; to.ns[at] = k.ns[r];
  }
  // entering states of segments are found by role: the passes with dots come first in the caller's order
  plain.a.seg = k.a.seg + (int64_t)with * (a.nseg + 1) * a.B * a.H * a.seg_stride;
  part.xy_stages = 1;
  plain.xy_stages = 2;
  if (int rc = la_tc_launch<false, true>(part, with, st)) return rc;
  return without ? la_tc_launch<false, false>(plain, without, st, true) : PTB_OK;
}

template <class T, class S>
static int la_run(LaArgs<S>& a, int roles, const LaPlan& l, void* ws, uint32_t* status, cudaStream_t st) {
  la_workspace(a, l, ws);
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    if (la_tensor_cores<T>(a.T)) {
      LaTcArgs k = {};
      int moved;
      LaMoveArgs m = la_results(a, roles, l, ws, &moved);
      if (int rc = la_tc_setup(&k, a, roles)) return rc;
      k.a = a;
      k.status = status;
      k.wait_cycles = (long long)(g_wait_ns * 2);   // SM clocks are below 2 GHz
      if (int rc = la_tc_run(k, roles, st)) return rc;
      return la_move(m, moved, LaSize{a.B, a.T, a.H, 0, 0}, st);
    }
  int most = 0;   // channels of x and y
  for (int r = 0; r < roles; ++r) most = std::max(most, a.p[r].M);
  return most <= 64 ? la_simt_run<T, S, 64>(a, roles, st) : la_simt_run<T, S, 128>(a, roles, st);
}

static void la_strides(int64_t (&d)[3], const int64_t* s) { for (int i = 0; i < 3; ++i) d[i] = s[i]; }

template <class T, class S>
static int la_fwd(const LaSize& z, LaOperands x, const void* g, const int64_t* gs, LaLengths lengths, const void* init,
                  double scale, int copies, void* o, int o_wide, void* fin, void* ws, int64_t wsb, uint32_t* status,
                  cudaStream_t st) {
  const bool tc = la_tensor_cores<T>(z.T);
  const LaPlan l = la_plan_of<S>(tc, z, 1, false, copies);
  if (l.total && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255u) || wsb < l.total)) return PTB_ERR_WORKSPACE;
  if (tc)
    if (int rc = la_copy_in(&x, copies, z, l, ws, st)) return rc;
  LaArgs<S> a = {};
  LaPass<S>& p = a.p[0];
  p.x = x.p[0]; p.y = x.p[1]; p.z = x.p[2];
  la_strides(p.xs, x.st[0]); la_strides(p.ys, x.st[1]); la_strides(p.zs, x.st[2]);
  p.o = o;
  p.init = static_cast<const S*>(init);
  p.fin = static_cast<S*>(fin);
  p.M = (int)z.Dk; p.N = (int)z.Dv;
  p.po = (S)scale; p.pz = (S)1;
  p.wide = o_wide;
  a.g = static_cast<const S*>(g);
  la_strides(a.gs, gs);
  a.lengths = lengths;
  a.B = z.B; a.T = z.T; a.H = z.H;
  return la_run<T, S>(a, 1, l, ws, status, st);
}

template <class T, class S>
static int la_bwd(const LaSize& z, LaOperands op, const void* g, const int64_t* gs, LaLengths lengths, const void* init,
                  double scale, int copies, const void* gfin, void* gq, void* gk, void* gv, void* gg, int gg_per_token,
                  void* ginit, void* ws, int64_t wsb, uint32_t* status, cudaStream_t st) {
  const bool dec = gg != nullptr, tc = la_tensor_cores<T>(z.T);
  const int64_t B = z.B, H = z.H, Dk = z.Dk, Dv = z.Dv;
  if (!gq && !gk && !gv && !dec && !ginit) return PTB_OK;
  const LaPlan l = la_plan_of<S>(tc, z, 3, dec, copies);
  if (l.total && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255u) || wsb < l.total)) return PTB_ERR_WORKSPACE;
  if (tc)
    if (int rc = la_copy_in(&op, copies, z, l, ws, st)) return rc;
  const void *q = op.p[0], *k = op.p[1], *v = op.p[2], *go = op.p[3];
  const int64_t *qs = op.st[0], *ks = op.st[1], *vs = op.st[2], *gos = op.st[3];
  char* w = static_cast<char*>(ws);
  LaArgs<S> a = {};
  a.g = static_cast<const S*>(g);
  la_strides(a.gs, gs);
  a.lengths = lengths;
  a.B = B; a.T = z.T; a.H = H;
  int roles = 0;
  if (gq || dec) {
    LaPass<S>& p = a.p[roles++];
    p.x = go; p.y = v; p.z = k; p.w = q;
    la_strides(p.xs, gos); la_strides(p.ys, vs); la_strides(p.zs, ks); la_strides(p.ws, qs);
    p.o = gq;
    p.init = static_cast<const S*>(init);
    p.M = (int)Dv; p.N = (int)Dk; p.state_t = 1;
    p.po = (S)scale; p.pz = (S)1;
  }
  if (gk || dec || ginit) {
    LaPass<S>& p = a.p[roles++];
    p.x = v; p.y = go; p.z = q; p.w = k;
    la_strides(p.xs, vs); la_strides(p.ys, gos); la_strides(p.zs, qs); la_strides(p.ws, ks);
    p.o = gk; p.out = 1;
    p.init = static_cast<const S*>(gfin);
    p.fin = static_cast<S*>(ginit);
    p.M = (int)Dv; p.N = (int)Dk; p.state_t = 1; p.reverse = 1;
    p.po = (S)1; p.pz = (S)scale;
  }
  if (gv) {
    LaPass<S>& p = a.p[roles++];
    p.x = k; p.y = q; p.z = go;
    la_strides(p.xs, ks); la_strides(p.ys, qs); la_strides(p.zs, gos);
    p.o = gv; p.out = 2;
    p.init = static_cast<const S*>(gfin);
    p.M = (int)Dk; p.N = (int)Dv; p.reverse = 1;
    p.po = (S)1; p.pz = (S)scale;
  }
  if (dec) {   // the first two passes give what the gradient of the decays is made of
    a.p[0].bounds = reinterpret_cast<S*>(w + l.qb_off);
    a.p[0].dots = reinterpret_cast<S*>(w + l.qd_off);
    a.p[1].bounds = reinterpret_cast<S*>(w + l.rb_off);
    a.p[1].dots = reinterpret_cast<S*>(w + l.kd_off);
  }
  if (int rc = la_run<T, S>(a, roles, l, ws, status, st)) return rc;
  if (dec && l.nchunk > 0) {
    LaDecayArgs<S> d = {};
    d.s_bounds = reinterpret_cast<const S*>(w + l.qb_off);
    d.r_bounds = reinterpret_cast<const S*>(w + l.rb_off);
    d.qd = reinterpret_cast<const S*>(w + l.qd_off);
    d.kd = reinterpret_cast<const S*>(w + l.kd_off);
    const int width = tc ? kTcSlice : LaGeom<S>::NS, slices = (int)((Dk + width - 1) / width);
    d.q_slices = d.k_slices = tc ? 2 * slices : slices;   // there two warps share a row
    d.g = a.g;
    la_strides(d.gs, gs);
    d.lengths = lengths;
    d.B = B; d.T = z.T; d.H = H; d.MN = l.bound_elems;
    if (gg_per_token) d.dg = static_cast<S*>(gg);
    else d.part = reinterpret_cast<double*>(w + l.part_off);
    if (B * H * l.nchunk > 0x7fffffffll) return PTB_ERR_TOO_LARGE;
    const unsigned grid = (unsigned)(B * H * l.nchunk);
    if (tc) la_decay_grad_kernel<S, kTcChunk><<<grid, 256, 0, st>>>(d);
    else la_decay_grad_kernel<S, LaGeom<S>::C><<<grid, 256, 0, st>>>(d);
    PTB_CUDA(cudaGetLastError());
  }
  if (dec && !gg_per_token) {
    la_decay_sum_kernel<S><<<(unsigned)H, 256, 0, st>>>(reinterpret_cast<double*>(w + l.part_off), l.nchunk, B, H,
                                                         static_cast<S*>(gg));
    PTB_CUDA(cudaGetLastError());
  }
  return PTB_OK;
}

template <class T, class S>
static int la_step(int64_t B, int64_t H, int64_t Dk, int64_t Dv, const void* q, const int64_t* qs, const void* k,
                   const int64_t* ks, const void* v, const int64_t* vs, const void* g, const int64_t* gs, double scale,
                   void* state, const int64_t* ss, void* o, int o_wide, cudaStream_t st) {
  LaStepArgs<T, S> a;
  a.q = static_cast<const T*>(q); a.k = static_cast<const T*>(k); a.v = static_cast<const T*>(v);
  for (int i = 0; i < 2; ++i) { a.qs[i] = qs[i]; a.ks[i] = ks[i]; a.vs[i] = vs[i]; a.gs[i] = gs[i]; a.ss[i] = ss[i]; }
  a.g = static_cast<const S*>(g);
  a.state = static_cast<S*>(state);
  a.o = o;
  a.wide = o_wide;
  a.H = H; a.M = (int)Dk; a.N = (int)Dv;
  a.scale = (S)scale;
  constexpr int V = 16 / sizeof(S);
  const dim3 grid((unsigned)(B * H), (unsigned)((Dv + 31) / 32));
  if (aligned16(state) && Dv % V == 0 && ss[0] % V == 0 && ss[1] % V == 0) la_step_kernel<T, S, V><<<grid, 256, 0, st>>>(a);
  else la_step_kernel<T, S, 1><<<grid, 256, 0, st>>>(a);
  PTB_CUDA(cudaGetLastError());
  return PTB_OK;
}

static int la_check(int dtype, int64_t B, int64_t T, int64_t H, int64_t Dk, int64_t Dv) {
  if (dtype != PTB_F32 && dtype != PTB_F64 && dtype != PTB_F16 && dtype != PTB_BF16) return PTB_ERR_ARG;
  if (B < 0 || T < 0 || H < 0 || Dk < 1 || Dv < 1 || Dk > kLaMaxDim || Dv > kLaMaxDim) return PTB_ERR_ARG;
  if (dtype == PTB_BF16 && T > 0x7fffff00ll) return PTB_ERR_TOO_LARGE;   // token numbers there, a chunk past the end too, in 32 bits
  if (B > 0x7fffffffll || H > 0x7fffffffll || B * H > 0x7fffffffll || T > (1ll << 40)) return PTB_ERR_TOO_LARGE;
  return PTB_OK;
}

}  // namespace ptb

using namespace ptb;

#define PTB_LA_TYPES(CALL)                                                                   \
  switch (dtype) {                                                                           \
    case PTB_F64: { using T_ = double; using S_ = double; return CALL; }                     \
    case PTB_F32: { using T_ = float; using S_ = float; return CALL; }                       \
    case PTB_F16: { using T_ = __half; using S_ = float; return CALL; }                      \
    default: { using T_ = __nv_bfloat16; using S_ = float; return CALL; }                    \
  }

static int la_step_entry(int dtype, int64_t B, int64_t H, int64_t Dk, int64_t Dv, const void* q,
                         const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                         const int64_t* v_strides, const void* log_decay, const int64_t* log_decay_strides,
                         double scale, void* state, const int64_t* state_strides, void* o, int o_wide, ptb_stream_t stream) {
  if (int rc = la_check(dtype, B, 1, H, Dk, Dv)) return rc;
  if (B == 0 || H == 0) return PTB_OK;
  if (!q || !k || !v || !log_decay || !state || !o || !q_strides || !k_strides || !v_strides || !log_decay_strides || !state_strides)
    return PTB_ERR_ARG;
  PTB_LA_TYPES((la_step<T_, S_>(B, H, Dk, Dv, q, q_strides, k, k_strides, v, v_strides, log_decay, log_decay_strides,
                                scale, state, state_strides, o, o_wide, (cudaStream_t)stream)))
}

extern "C" {

int64_t ptb_linear_attention_any_rows_tokens(int dtype) {
  return dtype == PTB_BF16 ? la_cuda_core_tokens<__nv_bfloat16>() : la_cuda_core_tokens<float>();
}

int64_t ptb_linear_attention_workspace_bytes(int dtype, int64_t B, int64_t T, int64_t H, int64_t Dk, int64_t Dv,
                                             int backward, int decay_grad, int copies) {
  if (la_check(dtype, B, T, H, Dk, Dv) != PTB_OK) return 0;
  const LaSize z = {B, T, H, Dk, Dv};
  const int roles = backward ? 3 : 1;
  PTB_LA_TYPES((la_plan_of<S_>(la_tensor_cores<T_>(T), z, roles, decay_grad, copies).total))
}

int ptb_linear_attention_fwd(int dtype, int64_t B, int64_t T, int64_t H, int64_t Dk, int64_t Dv, const void* q,
                             const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                             const int64_t* v_strides, const void* log_decay, const int64_t* log_decay_strides,
                             const void* lengths, int lengths_wide, const void* init, double scale, int copies, void* o, int o_wide, void* fin,
                             void* workspace, int64_t workspace_bytes, uint32_t* status, ptb_stream_t stream) {
  if (int rc = la_check(dtype, B, T, H, Dk, Dv)) return rc;
  if (B == 0 || H == 0) return PTB_OK;
  if ((T > 0 && (!q || !k || !v || !o || !log_decay)) || !q_strides || !k_strides || !v_strides || !log_decay_strides) return PTB_ERR_ARG;
  LaOperands x = {{q, k, v, nullptr}, {}};
  la_strides(x.st[0], q_strides); la_strides(x.st[1], k_strides); la_strides(x.st[2], v_strides);
  const LaSize z = {B, T, H, Dk, Dv};
  PTB_LA_TYPES((la_fwd<T_, S_>(z, x, log_decay, log_decay_strides, LaLengths{lengths, lengths_wide}, init, scale, copies, o, o_wide,
                               fin, workspace, workspace_bytes, status, (cudaStream_t)stream)))
}

int ptb_linear_attention_bwd(int dtype, int64_t B, int64_t T, int64_t H, int64_t Dk, int64_t Dv, const void* q,
                             const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                             const int64_t* v_strides, const void* log_decay, const int64_t* log_decay_strides,
                             const void* lengths, int lengths_wide, const void* init, double scale, int copies, const void* grad_o,
                             const int64_t* grad_o_strides, const void* grad_fin, void* grad_q, void* grad_k,
                             void* grad_v, void* grad_log_decay, int grad_log_decay_per_token, void* grad_init,
                             void* workspace, int64_t workspace_bytes, uint32_t* status, ptb_stream_t stream) {
  if (int rc = la_check(dtype, B, T, H, Dk, Dv)) return rc;
  if (B == 0 || H == 0) return PTB_OK;
  if ((T > 0 && (!q || !k || !v || !log_decay || !grad_o)) || !q_strides || !k_strides || !v_strides || !log_decay_strides ||
      !grad_o_strides)
    return PTB_ERR_ARG;
  LaOperands x = {{q, k, v, grad_o}, {}};
  la_strides(x.st[0], q_strides); la_strides(x.st[1], k_strides); la_strides(x.st[2], v_strides);
  la_strides(x.st[3], grad_o_strides);
  const LaSize z = {B, T, H, Dk, Dv};
  PTB_LA_TYPES((la_bwd<T_, S_>(z, x, log_decay, log_decay_strides, LaLengths{lengths, lengths_wide}, init, scale, copies, grad_fin,
                               grad_q, grad_k, grad_v, grad_log_decay, grad_log_decay_per_token, grad_init, workspace,
                               workspace_bytes, status, (cudaStream_t)stream)))
}

int ptb_linear_attention_step(int dtype, int64_t B, int64_t H, int64_t Dk, int64_t Dv, const void* q,
                              const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                              const int64_t* v_strides, const void* log_decay, const int64_t* log_decay_strides,
                              double scale, void* state, const int64_t* state_strides, void* o, ptb_stream_t stream) {
  return la_step_entry(dtype, B, H, Dk, Dv, q, q_strides, k, k_strides, v, v_strides, log_decay, log_decay_strides, scale, state,
                       state_strides, o, 0, stream);
}

int ptb_linear_attention_step_sums(int dtype, int64_t B, int64_t H, int64_t Dk, int64_t Dv, const void* q,
                                   const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                                   const int64_t* v_strides, const void* log_decay, const int64_t* log_decay_strides,
                                   double scale, void* state, const int64_t* state_strides, void* o, ptb_stream_t stream) {
  return la_step_entry(dtype, B, H, Dk, Dv, q, q_strides, k, k_strides, v, v_strides, log_decay, log_decay_strides, scale, state,
                       state_strides, o, 1, stream);
}

}  // extern "C"
