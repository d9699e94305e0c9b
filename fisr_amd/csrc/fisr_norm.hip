// C-ABI of group normalisation with an activation and of dropout (include/fisr.h, "normalisation and dropout").  A translation unit of
// its own: its device code is compiled without packed float32 instructions (fisr_amd/lib.py), which the Winograd kernels of
// fisr_api.hip write by hand.
#include <cmath>

#include "../../include/fisr.h"
#include "host_util.h"
#include "train_norm_kernels.h"

using namespace fisr;

#define NORM_HIP_OK(expr)                                                                                             \
  do {                                                                                                                \
    hipError_t e_ = (expr);                                                                                           \
    if (e_ != hipSuccess) return set_error(FISR_EHIP, std::string(#expr) + ": " + hipGetErrorString(e_));             \
  } while (0)

namespace {

// Chunks of one image: about 2048 workgroups for the whole batch (8 a CU), of at least 8192 elements each (32 a thread).  Not a
// function of the vector width: the workspace's size is asked for without the tensors.
void norm_chunks(NormArgs& a) {
  const int want = std::max(1, 2048 / a.n);
  a.ppc = std::max((a.p + want - 1) / want, (8191 + a.c) / a.c);
  a.chunks = (a.p + a.ppc - 1) / a.ppc;
}
void norm_threads(NormArgs& a, int v, dim3& grid) {
  const int cv = (a.c + v - 1) / v, ny = (cv + 255) / 256;
  a.cb = (cv + ny - 1) / ny;
  a.rows = 256 / a.cb;
  grid = dim3(a.n * a.chunks, ny);
}
size_t norm_ws_bytes(const NormArgs& a, bool backward) {
  size_t f2 = (size_t)a.n * a.chunks * a.c;
  if (backward) f2 += (size_t)a.n * a.c + (size_t)a.n * a.groups;
  return f2 * sizeof(float2);
}

// One pixel of a launch's workgroups: vectors of eight channels where all tensors allow 16-byte accesses, else four or two, else one.
template <typename T> int norm_vec(const NormArgs& a) {
  const uintptr_t ptrs = (uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.y;
  const size_t cs = a.xcs | a.ycs | a.dycs;
  for (int v = 8; v > 1; v >>= 1) {
    const size_t bytes = std::min<size_t>(v * sizeof(T), 16);
    if (a.c % v == 0 && ptrs % bytes == 0 && cs * sizeof(T) % bytes == 0) return v;
  }
  return 1;
}

template <typename T, int V> void launch_fwd(NormArgs a, hipStream_t st) {
  dim3 grid;
  norm_threads(a, V, grid);
  hipLaunchKernelGGL((norm_stats_kernel<T, V>), grid, dim3(256), 0, st, a);
  hipLaunchKernelGGL(norm_stats_join_kernel, dim3(a.n * a.groups), dim3(256), 0, st, a);
  hipLaunchKernelGGL((norm_apply_kernel<T, V>), grid, dim3(256), 0, st, a);
}
template <typename T, int V> void launch_bwd(NormArgs a, hipStream_t st) {
  dim3 grid;
  norm_threads(a, V, grid);
  hipLaunchKernelGGL((norm_bwd_sums_kernel<T, V>), grid, dim3(256), 0, st, a);
  hipLaunchKernelGGL(norm_bwd_join_kernel, dim3(a.n * a.groups), dim3(256), 0, st, a);
  hipLaunchKernelGGL((norm_bwd_apply_kernel<T, V>), grid, dim3(256), 0, st, a);
  if (a.dgamma || a.dbeta) hipLaunchKernelGGL(norm_bwd_params_kernel, dim3((a.c + 63) / 64), dim3(256), 0, st, a);
}
template <typename T> void launch(const NormArgs& a, bool backward, hipStream_t st) {
  const int v = norm_vec<T>(a);
#define NORM_V(V) if (v == V) { if (backward) launch_bwd<T, V>(a, st); else launch_fwd<T, V>(a, st); return; }
  NORM_V(8) NORM_V(4) NORM_V(2) NORM_V(1)
#undef NORM_V
}

// The shape's limits keep every pixel index in 31 bits and every grid in HIP's (elements are counted in 64 bits).
const char* norm_shape_error(int n, int h, int w, int c, int groups) {
  if (n <= 0 || h <= 0 || w <= 0 || c <= 0 || groups <= 0) return "a size is not positive";
  if (c % groups) return "the channels are no multiple of the groups";
  if ((long long)h * w > 1 << 30 || c > 1 << 16 || (long long)n * groups > 1 << 22 || n > 1 << 20) return "a size passes the limits (h * w 2^30, c 2^16, n 2^20, n * groups 2^22)";
  return nullptr;
}
const char* drop_error(const fisr_dropout* d, DropArgs& out) {
  out = DropArgs{0, 1.f, 0, 0, nullptr};
  if (!d) return nullptr;
  if (!(d->p >= 0.0 && d->p <= 1.0)) return "dropout: p is not in [0, 1]";
  out.thresh = (uint32_t)std::lrint(d->p * 65536.0);
  out.scale = out.thresh < 65536 ? (float)(65536.0 / (65536.0 - out.thresh)) : 0.f;
  out.seed = d->seed; out.offset = d->offset; out.counter = d->d_counter;
  if ((uintptr_t)d->d_counter % 8) return "dropout: d_counter is not aligned to 8 bytes";
  return nullptr;
}
size_t type_bytes(int type) { return type == FISR_TYPE_F32 ? 4 : type == FISR_TYPE_F16 || type == FISR_TYPE_BF16 ? 2 : 0; }

int norm_call(const char* who, NormArgs& a, bool backward, int n, int h, int w, int c, int groups, int act, const fisr_dropout* drop, int type,
              float* mean_rstd, void* ws, size_t ws_bytes, void* stream) {
  const auto bad = [&](const char* what) { return set_error(FISR_EINVAL, std::string(who) + ": " + what); };
  if (const char* e = norm_shape_error(n, h, w, c, groups)) return bad(e);
  if (!a.x || !a.y || !mean_rstd || (backward && !a.dy)) return bad("null tensor");
  if (a.xcs < (size_t)c || a.ycs < (size_t)c || (backward && a.dycs < (size_t)c)) return bad("a pixel stride is less than the channels");
  const size_t es = type_bytes(type);
  if (!es) return bad("unknown tensor type");
  if (((uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy) % es || ((uintptr_t)a.gamma | (uintptr_t)a.beta | (uintptr_t)mean_rstd | (uintptr_t)a.dgamma | (uintptr_t)a.dbeta) % 4)
    return bad("a pointer is not aligned to its element");
  if (act < FISR_ACT_NONE || act > FISR_ACT_GELU) return bad("unknown activation");
  if (const char* e = drop_error(drop, a.drop)) return bad(e);
  a.n = n; a.p = h * w; a.c = c; a.groups = groups; a.d = c / groups; a.act = act;
  a.mean = mean_rstd; a.rstd = mean_rstd + (size_t)n * groups;
  norm_chunks(a);
  if (!ws || (uintptr_t)ws % 16) return bad("the workspace is null or not aligned to 16 bytes");
  if (ws_bytes < norm_ws_bytes(a, backward)) return set_error(FISR_ENOMEM, std::string(who) + ": workspace too small");
  a.part = (float2*)ws;
  a.ab = a.part + (size_t)a.n * a.chunks * a.c;
  a.s12 = a.ab + (size_t)a.n * a.c;
  DeviceGuard guard(device_of(a.y));
  NORM_HIP_OK(guard.err);
  const hipStream_t st = (hipStream_t)stream;
  if (type == FISR_TYPE_F32) launch<float>(a, backward, st);
  else if (type == FISR_TYPE_F16) launch<f16_t>(a, backward, st);
  else launch<b16_t>(a, backward, st);
  NORM_HIP_OK(hipGetLastError());
  return 0;
}

template <typename T> void launch_dropout(const void* x, const void* res, void* y, size_t count, const DropArgs& d, hipStream_t st) {
  const bool aligned = ((uintptr_t)x | (uintptr_t)res | (uintptr_t)y) % 16 == 0;
  const dim3 grid(grid_for((count + 7) / 8));
  if (aligned) hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(256), 0, st, (const T*)x, (const T*)res, (T*)y, count, d);
  else hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(256), 0, st, (const T*)x, (const T*)res, (T*)y, count, d);
}

}  // namespace

extern "C" {

size_t fisr_train_groupnorm_workspace_bytes(int n, int h, int w, int c, int groups, int backward) {
  if (norm_shape_error(n, h, w, c, groups)) return 0;
  NormArgs a{};
  a.n = n; a.p = h * w; a.c = c; a.groups = groups;
  norm_chunks(a);
  return norm_ws_bytes(a, backward != 0);
}

int fisr_train_groupnorm(const void* x, int x_cs, const float* gamma, const float* beta, void* y, int y_cs, float* mean_rstd, int n, int h, int w,
                         int c, int groups, float eps, int act, const fisr_dropout* drop, int type, void* workspace, size_t workspace_bytes,
                         void* stream) {
  NormArgs a{};
  a.x = x; a.y = y; a.gamma = gamma; a.beta = beta; a.xcs = (size_t)std::max(x_cs, 0); a.ycs = (size_t)std::max(y_cs, 0); a.eps = eps;
  if (!(eps >= 0.f) || !std::isfinite(eps)) return set_error(FISR_EINVAL, "fisr_train_groupnorm: eps is negative or not finite");
  return norm_call("fisr_train_groupnorm", a, false, n, h, w, c, groups, act, drop, type, mean_rstd, workspace, workspace_bytes, stream);
}

int fisr_train_groupnorm_bwd(const void* x, int x_cs, const void* dy, int dy_cs, const float* gamma, const float* beta, const float* mean_rstd,
                             void* dx, int dx_cs, float* dgamma, float* dbeta, int accumulate, int n, int h, int w, int c, int groups, int act,
                             const fisr_dropout* drop, int type, void* workspace, size_t workspace_bytes, void* stream) {
  NormArgs a{};
  a.x = x; a.dy = dy; a.y = dx; a.gamma = gamma; a.beta = beta; a.dgamma = dgamma; a.dbeta = dbeta; a.accumulate = accumulate != 0;
  a.xcs = (size_t)std::max(x_cs, 0); a.dycs = (size_t)std::max(dy_cs, 0); a.ycs = (size_t)std::max(dx_cs, 0);
  return norm_call("fisr_train_groupnorm_bwd", a, true, n, h, w, c, groups, act, drop, type, const_cast<float*>(mean_rstd), workspace,
                   workspace_bytes, stream);
}

int fisr_train_dropout(const void* x, const void* residual, void* y, size_t count, const fisr_dropout* drop, int type, void* stream) {
  const auto bad = [&](const char* what) { return set_error(FISR_EINVAL, std::string("fisr_train_dropout: ") + what); };
  const size_t es = type_bytes(type);
  DropArgs d;
  if (!es) return bad("unknown tensor type");
  if (const char* e = drop_error(drop, d)) return bad(e);
  if (count == 0) return 0;
  if (!x || !y) return bad("null tensor");
  if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) % es) return bad("a pointer is not aligned to its element");
  DeviceGuard guard(device_of(y));
  NORM_HIP_OK(guard.err);
  const hipStream_t st = (hipStream_t)stream;
  if (type == FISR_TYPE_F32) launch_dropout<float>(x, residual, y, count, d, st);
  else if (type == FISR_TYPE_F16) launch_dropout<f16_t>(x, residual, y, count, d, st);
  else launch_dropout<b16_t>(x, residual, y, count, d, st);
  NORM_HIP_OK(hipGetLastError());
  return 0;
}

}  // extern "C"
