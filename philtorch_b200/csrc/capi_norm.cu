// C ABI of the layer norm over groups of channels (see include/philtorch_b200.h).
#include "layer_norm.cuh"

namespace ptb {

constexpr int kLnSms = 148;

// lanes per unit: the fewest of 8 / 32 / 256 / 1024 that hold a unit in at most 4 vectors each
static int ln_lanes(int width, int V) {
  for (int L : {8, 32, 256})
    if (L * V * 4 >= width) return L;
  return 1024;
}

// CTAs over the rows.  Backward: each leaves one partial row of the parameter gradients, so there are no more of
// them than are resident at once; forward: a few rounds of them, so that the last round is short
static int64_t ln_row_blocks(int64_t rows, int groups, int L, int64_t per_sm) {
  const int slots = ln_threads(L) / L;
  const int64_t want = std::max<int64_t>(1, (kLnSms * per_sm + groups - 1) / groups);
  return std::max<int64_t>(1, std::min<int64_t>(want, (rows + slots - 1) / slots));
}
static int64_t ln_bwd_blocks(int64_t rows, int groups, int L) { return ln_row_blocks(rows, groups, L, L > 256 ? 1 : 2); }

// T: x's type, TO: y's
template <class T, class TO, class S, int V, int L, int NV>
static int ln_launch(const LnArgs<S>& a, bool bwd, int64_t blocks, cudaStream_t st) {
  constexpr int NT = ln_threads(L), SLOTS = NT / L;
  constexpr int kPipe = ln_pipe_bytes<T, S, V, L, NV>(1), kPipeBwd = ln_pipe_bytes<T, S, V, L, NV>(2);
  static bool ready[kMaxDevices] = {};
  int dev = 0;
  PTB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return PTB_ERR_ARG;
  {
    std::lock_guard<std::mutex> lock(init_mutex());
    if (!ready[dev]) {
      PTB_CUDA(cudaFuncSetAttribute(ln_fwd_kernel<T, TO, S, V, L, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPipe));
      if constexpr (std::is_same<T, TO>::value)
        PTB_CUDA(cudaFuncSetAttribute(ln_bwd_kernel<T, S, V, L, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      std::max(kPipeBwd, 48 * 1024)));
      ready[dev] = true;
    }
  }
  if (!bwd) {
    const int64_t grid = ln_row_blocks(a.rows, a.groups, L, 8);
    ln_fwd_kernel<T, TO, S, V, L, NV><<<dim3((unsigned)grid, a.groups), NT, kPipe, st>>>(a);
  } else if constexpr (std::is_same<T, TO>::value) {
    const int join = SLOTS > 1 ? SLOTS * a.width * (int)sizeof(S) : 0;   // at most 256 * V * NV scalars = 32 KB
    ln_bwd_kernel<T, S, V, L, NV><<<dim3((unsigned)blocks, a.groups), NT, std::max(kPipeBwd, join), st>>>(a);
  }
  PTB_CUDA(cudaGetLastError());
  return PTB_OK;
}

template <class T, class TO, class S, int V>
static int ln_pick(const LnArgs<S>& a, bool bwd, int64_t blocks, cudaStream_t st) {
  const int L = ln_lanes(a.width, V), nv = (a.width + L * V - 1) / (L * V);
#define PTB_LN(L_, N_) return ln_launch<T, TO, S, V, L_, N_>(a, bwd, blocks, st)
  if (L == 8) { if (nv <= 1) PTB_LN(8, 1); if (nv <= 2) PTB_LN(8, 2); PTB_LN(8, 4); }
  if (L == 32) { if (nv <= 2) PTB_LN(32, 2); PTB_LN(32, 4); }
  if (L == 256) { if (nv <= 2) PTB_LN(256, 2); PTB_LN(256, 4); }
  constexpr int kMost = (kLnMaxWidth / V + 1023) / 1024;   // 16384 channels: 16, 8, 4 or 2 vectors a lane
  if constexpr (kMost > 4) { if (nv > 4) PTB_LN(1024, kMost); }
  PTB_LN(1024, (kMost < 4 ? kMost : 4));
#undef PTB_LN
}

template <class T, class S>
static int ln_vec(const LnArgs<S>& a) {   // elements per access
  constexpr int V = 16 / sizeof(T);
  bool ok = a.width % V == 0 && aligned16(a.x) && a.x_stride % V == 0;
  ok = ok && (!a.y || aligned16(a.y)) && (!a.gx || aligned16(a.gx));
  ok = ok && (!a.gy || (aligned16(a.gy) && a.gy_stride % V == 0));
  return ok ? V : 1;
}

template <class T, class TO, class S>
static int ln_fwd(const LnArgs<S>& a, cudaStream_t st) {
  if (ln_vec<T, S>(a) == 1) return ln_pick<T, TO, S, 1>(a, false, 0, st);
  return ln_pick<T, TO, S, 16 / sizeof(T)>(a, false, 0, st);
}

template <class T, class S>
static int ln_fwd_to(const LnArgs<S>& a, int y_dtype, cudaStream_t st) {
  if constexpr (std::is_same<T, float>::value) {
    if (y_dtype == PTB_F16) return ln_fwd<float, __half, float>(a, st);
    if (y_dtype == PTB_BF16) return ln_fwd<float, __nv_bfloat16, float>(a, st);
  }
  return ln_fwd<T, T, S>(a, st);
}

template <class T, class S>
static int ln_bwd(LnArgs<S>& a, void* gw, void* gb, void* ws, int64_t wsb, cudaStream_t st) {
  const int V = ln_vec<T, S>(a);
  const int64_t C = (int64_t)a.groups * a.width;
  const int64_t blocks = ln_bwd_blocks(a.rows, a.groups, ln_lanes(a.width, V));
  const int64_t one = align_up(blocks * C * (int64_t)sizeof(S), 256), need = (gw ? one : 0) + (gb ? one : 0);
  if (need && (!ws || (reinterpret_cast<uintptr_t>(ws) & 255u) || wsb < need)) return PTB_ERR_WORKSPACE;
  char* w = static_cast<char*>(ws);
  a.part_w = gw ? reinterpret_cast<S*>(w) : nullptr;
  a.part_b = gb ? reinterpret_cast<S*>(w + (gw ? one : 0)) : nullptr;
  const int rc = V == 1 ? ln_pick<T, T, S, 1>(a, true, blocks, st) : ln_pick<T, T, S, 16 / sizeof(T)>(a, true, blocks, st);
  if (rc != PTB_OK || !need) return rc;
  ln_param_grad_kernel<T, S><<<dim3((unsigned)((C + 31) / 32), 2), 256, 0, st>>>(a.part_w, a.part_b, (int)blocks, C, gw, gb,
                                                                               a.w_wide);
  PTB_CUDA(cudaGetLastError());
  return PTB_OK;
}

static int ln_check(int dtype, int64_t rows, int64_t groups, int64_t width) {
  if (dtype != PTB_F32 && dtype != PTB_F64 && dtype != PTB_F16 && dtype != PTB_BF16) return PTB_ERR_ARG;
  if (rows < 0 || groups < 1 || groups > 65535 || width < 1 || width > kLnMaxWidth) return PTB_ERR_ARG;
  if (rows > (1ll << 40)) return PTB_ERR_TOO_LARGE;
  return PTB_OK;
}

template <class S>
static LnArgs<S> ln_args(int64_t rows, int64_t groups, int64_t width, const void* x, int64_t x_stride, const void* w,
                         const void* b, int w_wide, void* mean, void* rstd) {
  LnArgs<S> a = {};
  a.x = x; a.x_stride = x_stride;
  a.w = w; a.b = b; a.w_wide = w_wide;
  a.w_vec = aligned16(w) && aligned16(b);
  a.mean = static_cast<S*>(mean); a.rstd = static_cast<S*>(rstd);
  a.rows = rows; a.groups = (int)groups; a.width = (int)width;
  return a;
}

}  // namespace ptb

using namespace ptb;

#define PTB_LN_TYPES(BODY)                                                                   \
  switch (dtype) {                                                                           \
    case PTB_F64: { using T_ = double; using S_ = double; BODY }                             \
    case PTB_F32: { using T_ = float; using S_ = float; BODY }                               \
    case PTB_F16: { using T_ = __half; using S_ = float; BODY }                              \
    default: { using T_ = __nv_bfloat16; using S_ = float; BODY }                            \
  }

extern "C" {

int64_t ptb_layer_norm_bwd_workspace_bytes(int dtype, int64_t rows, int64_t groups, int64_t width) {
  if (ln_check(dtype, rows, groups, width) != PTB_OK) return 0;
  const int64_t s = dtype == PTB_F64 ? 8 : 4, vec = dtype == PTB_F64 ? 2 : dtype == PTB_F32 ? 4 : 8;
  int64_t most = 1;   // the pointers' alignment may rule the wide accesses out: room for either choice
  for (int V : {1, (int)vec}) most = std::max(most, ln_bwd_blocks(rows, (int)groups, ln_lanes((int)width, V)));
  return 2 * align_up(most * groups * width * s, 256);
}

int ptb_layer_norm_fwd(int dtype, int64_t rows, int64_t groups, int64_t width, const void* x, int64_t x_stride,
                       const void* weight, const void* bias, int params_wide, double eps, int y_dtype, void* y,
                       void* mean, void* rstd, ptb_stream_t stream) {
  if (int rc = ln_check(dtype, rows, groups, width)) return rc;
  if (y_dtype != dtype && !(dtype == PTB_F32 && (y_dtype == PTB_F16 || y_dtype == PTB_BF16))) return PTB_ERR_ARG;
  if (rows == 0) return PTB_OK;
  if (!x || !y || !mean != !rstd) return PTB_ERR_ARG;
  PTB_LN_TYPES(LnArgs<S_> a = ln_args<S_>(rows, groups, width, x, x_stride, weight, bias, params_wide, mean, rstd);
               a.y = y; a.eps = (S_)eps; return (ln_fwd_to<T_, S_>(a, y_dtype, (cudaStream_t)stream));)
}

int ptb_layer_norm_bwd(int dtype, int64_t rows, int64_t groups, int64_t width, const void* x, int64_t x_stride,
                       const void* weight, int params_wide, const void* mean, const void* rstd, const void* grad_y,
                       int64_t grad_y_stride, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                       int64_t workspace_bytes, uint32_t* status, ptb_stream_t stream) {
  (void)status;
  if (int rc = ln_check(dtype, rows, groups, width)) return rc;
  if (rows == 0) return PTB_OK;
  if (!x || !mean || !rstd || !grad_y) return PTB_ERR_ARG;
  PTB_LN_TYPES(LnArgs<S_> a = ln_args<S_>(rows, groups, width, x, x_stride, weight, nullptr, params_wide,
                                          const_cast<void*>(mean), const_cast<void*>(rstd));
               a.gy = grad_y; a.gy_stride = grad_y_stride; a.gx = grad_x;
               return (ln_bwd<T_, S_>(a, grad_weight, grad_bias, workspace, workspace_bytes, (cudaStream_t)stream));)
}

}  // extern "C"
