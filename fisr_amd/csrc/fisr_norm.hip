// C-ABI of group normalisation with an activation and of dropout (include/fisr.h, "normalisation and dropout").  A translation unit of
// its own: its device code is compiled without packed float32 instructions (fisr_amd/lib.py), which the Winograd kernels of
// fisr_api.hip write by hand.
#include <cmath>
#include <cstdlib>
#include <initializer_list>

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

#ifdef FISR_DIAG
int env_int(const char* name, int def) { const char* e = getenv(name); return e ? atoi(e) : def; }
#else
constexpr int env_int(const char*, int def) { return def; }
#endif

// Chunks of an image's pixels for about `workgroups` in all, of at least `least` elements each.
void chunks_for(const NormArgs& a, int workgroups, int least, int& chunks, int& ppc) {
  const int want = std::max(1, workgroups / a.n);
  ppc = std::max((a.p + want - 1) / want, (least - 1 + a.c) / a.c);
  chunks = (a.p + ppc - 1) / ppc;
}
// Two vectors a thread, 1024 elements at the least: small tensors want many workgroups (5 x 67 x 45 x 36 float32 in 11.4 us at 2 vectors, 14.0 at 8;
// 2 x 40 x 50 x 9 bfloat16 in 8.8 at 1024 elements, 14.0 at 8192)
constexpr int LEAST_ELEMENTS = 1024;
constexpr int least_chunk(int v) { return v * 512 > LEAST_ELEMENTS ? v * 512 : LEAST_ELEMENTS; }
constexpr int MOST_WORKGROUPS = 2048;                          // of a batch, by chunks_for: what the workspace is made for

// Workspace: `part` of n * chunks * c float2, and for the backward pass s12 of n * groups * chunks and ab of n * c.  Not a function of the
// vector width or the form that runs: its size is asked for without the tensors.
struct WsLayout {
  size_t part, s12, ab;
  size_t bytes() const { return (part + s12 + ab) * sizeof(float2); }
};
WsLayout ws_layout(const NormArgs& a, bool backward) {
  int chunks, ppc;
  chunks_for(a, MOST_WORKGROUPS, LEAST_ELEMENTS, chunks, ppc);
  WsLayout w{(size_t)a.n * chunks * a.c, 0, 0};
  if (backward) { w.s12 = (size_t)a.n * a.groups * chunks; w.ab = (size_t)a.n * a.c; }
  return w;
}

// Vectors of 16 bytes where all tensors allow such accesses, else of 8 and so on down to one channel.
template <typename T> int norm_vec(const NormArgs& a) {
  const uintptr_t ptrs = (uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.y;
  const size_t cs = a.xcs | a.ycs | a.dycs;
  for (int v = std::min<int>(16 / sizeof(T), env_int(a.dy ? "NORM_VB" : "NORM_VF", 8)); v > 1; v >>= 1)
    if (a.c % v == 0 && ptrs % (v * sizeof(T)) == 0 && cs * sizeof(T) % (v * sizeof(T)) == 0) return v;
  return 1;
}
uint32_t magic(int y) { return y == 1 ? 0 : (uint32_t)(((1ull << 32) + y - 1) / y); }
// A workgroup's columns, rows and what team_sums goes by.
void set_team(NormArgs& a, int v, int threads, int span) {
  a.span = span; a.cb = span / v; a.rows = threads / a.cb;
  a.slots = a.d % v == 0 ? 1 : v % a.d == 0 ? v / a.d : v;
  a.per_group = a.d * a.slots / v;
  a.by_cb = magic(a.cb); a.by_rows = magic(a.rows); a.by_per_group = magic(a.per_group);
  const int groups = span / a.d;
  for (a.jl = 6; a.jl > 0 && groups > threads >> a.jl;) --a.jl;
}
// Whether a thread's offset within `rows` pixels may pass 32 bits (see Walk).
bool wide_strides(const NormArgs& a, int rows, int elem_bytes) {
  return (unsigned long long)std::max({a.xcs, a.ycs, a.dycs}) * rows * elem_bytes > (1u << 31);
}
// lcm(d, v): the least channels that are whole groups and whole vectors
int span_unit(const NormArgs& a, int v) {
  int unit = a.d;
  while (unit % v) unit += a.d;
  return unit;
}

// One launch, a span of channels of a whole image in a workgroup's registers: which variant holds it (-1: none does, or it would be slower).
// Up to 9 vectors a thread: 48 x 48 pixels of 4 columns.  More were tried in the forward pass (bfloat16, 32 images of 128 channels in 32 groups): 12 take
// 50 x 50 in 17.8 us against 20.6 in two launches and 55 x 55 in 19.3 against 22.6, 16 take 64 x 64 in 23.0 against 26.6 (16 images 21.6 against 19.5);
// the backward pass holds dz as float32 beside them, 72 registers at 9 vectors of 8.
struct TeamVariant { int threads, r; };
constexpr TeamVariant TEAM[] = {{256, 1}, {256, 2}, {256, 4}, {256, 9}, {512, 9}};
int team_variant(NormArgs& a, int v, int elem_bytes, bool backward) {
  const size_t elems = (size_t)a.n * a.p * a.c;
  if (elems > (size_t)env_int("NORM_TEAM_K", 16384) << 10 || wide_strides(a, 512, elem_bytes)) return -1;
  const int unit = span_unit(a, v), most = a.c / unit;
  // Least bytes of a span.  Narrow ones read a cache line many times over (32 x 24 x 24 x 256 bfloat16 in 64 groups, 9.4 MB: 11.9 us at 64 bytes, 12.5 at 16,
  // 13.8 at 128; backward 15.5, 16.1, 18.6), small tensors want the workgroups more (8 x 24 x 24 x 256 in 64 groups, 2.4 MB: 9.0 at 16, 10.9 at 64; but with
  // 32 images of 12 x 12 8.6 and 7.7).  Whole lines of 128 bytes where there are 512 workgroups all the same: 128 x 8 x 8 x 512 bfloat16 in 64 groups 11.7 us
  // against 14.3, backward 14.9 against 19.8; 64 x 16 x 16 x 512 in 32 groups 15.5 against 14.2; without the limit of 512 16 x 24 x 24 x 512 in 32 groups takes
  // 13.7 instead of 11.8, backward 16.7 instead of 15.1.
  const int line = env_int("NORM_LINE", elems * elem_bytes > (size_t)4 << 20 ? 64 : 16);
  int best = -1, best_span = 0;
  for (int k = 1; k <= most; ++k) {
    const int span = k * unit, cols = span / v;
    if (cols > 256) break;
    if (most % k) continue;
    if (best >= 0 && best_span * elem_bytes >= line && (best_span * elem_bytes >= 128 || (long long)a.n * (a.c / span) < 512)) break;
    int fit = -1;
    for (int i = 0; i < (int)(sizeof(TEAM) / sizeof(TEAM[0])) && fit < 0; ++i) {
      const int rows = TEAM[i].threads / cols;
      if ((a.p + rows - 1) / rows <= TEAM[i].r) fit = i;
    }
    if (fit < 0) break;
    best = fit; best_span = span;
  }
  // few workgroups of many vectors a thread: the two launches' finer chunks are faster (one image of 48 x 48 x 128 bf16, 8 workgroups:
  // 12.8 us against 12.3, backward 20.1 against 14.9; with 32 workgroups of at most 4 vectors 8.3 against 11.5, backward 10.6 against 14.4)
  if (best >= 0 && TEAM[best].r > 4 && (backward || TEAM[best].threads > 256) && (long long)a.n * (a.c / best_span) < 64) best = -1;
  if (best >= 0) set_team(a, v, TEAM[best].threads, best_span);
  return best;
}
template <typename T, int V> void launch_team(const NormArgs& a, bool backward, hipStream_t st) {
  const dim3 grid(a.n * (a.c / a.span));
  const bool whole = a.slots == 1;
#define NORM_TEAM(I)                                                                                                                         \
  case I:                                                                                                                                    \
    if (!backward) hipLaunchKernelGGL((norm_team_kernel<T, V, TEAM[I].r, TEAM[I].threads>), grid, dim3(TEAM[I].threads), 0, st, a);           \
    else if (whole) hipLaunchKernelGGL((norm_team_grad_kernel<T, V, TEAM[I].r, TEAM[I].threads, true>), grid, dim3(TEAM[I].threads), 0, st, a);\
    else hipLaunchKernelGGL((norm_team_grad_kernel<T, V, TEAM[I].r, TEAM[I].threads, V == 1>), grid, dim3(TEAM[I].threads), 0, st, a);         \
    break;
  switch (a.team) { NORM_TEAM(0) NORM_TEAM(1) NORM_TEAM(2) NORM_TEAM(3) NORM_TEAM(4) }
#undef NORM_TEAM
  if (backward && (a.dgamma || a.dbeta)) hipLaunchKernelGGL(norm_params_kernel, dim3((a.c + 15) / 16), dim3(256), 0, st, a, a.ab, a.n);
}

// Two launches over chunks of pixels: grids and the channels of a workgroup (all, or the most whole groups that it has threads for).
bool two_tiling(NormArgs& a, int v, int elem_bytes, bool backward) {
  if (wide_strides(a, 256, elem_bytes)) return false;
  const int unit = span_unit(a, v), most = a.c / unit;
  int k = std::min(most, 256 * v / unit);
  while (k > 0 && most % k) --k;
  // (no such span, or one of few columns with more channels beside it: workgroups of any channels read whole lines.  About 4 M elements of 4 images, by
  // columns x spans, this form against that one: 3 x 347 float32 1274 and 49 us, 17 x 61 237 and 48, 41 x 31 137 and 57; 67 x 17 75 and 52, 113 x 11 53 and 59,
  // 100 x 5 42 and 72, 127 x 3 38 and 72; backward 67 x 17 138 and 80, 113 x 11 107 and 82, 100 x 5 84 and 90, 127 x 3 68 and 88)
  if (k == 0 || (k < most && k * unit / v < 64)) return false;
  set_team(a, v, 256, k * unit);
  // First launch: two long-lived workgroups a CU, whose numbers have to be joined.  Second: four a CU, six above 48 MB (272 x 496 x 128 bfloat16,
  // 35 MB: 30.9 us with four, 34.5 with six; 544 x 992 x 64, 69 MB: 48.9 and 47.2); beyond 192 MB pieces of 48 KB, backward 64, at most 64 a CU (twelve
  // 544 x 992 x 64 float16: 407 us in 16384 pieces, 443 in 1536, 422 in 32768; backward 702, 721, 767), or eight times what a workgroup reads to
  // join the first launch's numbers.
  const size_t bytes = (size_t)a.n * a.p * a.c * elem_bytes * (backward ? 2 : 1);
  chunks_for(a, env_int("NORM_SWG", 512), least_chunk(v), a.chunks, a.ppc);
  // (272 x 496 x 128 in 32 groups, backward: 51 us with norm_grad_join_kernel for the 16384 numbers, 60 without; in 512 groups 49 and 626)
  a.join = a.chunks * (a.span / a.d) <= env_int("NORM_JOIN", 2048);
  size_t second = bytes > (size_t)48 << 20 ? 1536 : 1024;
  if (bytes > (size_t)192 << 20) second = std::min<size_t>(bytes / std::max(backward ? 65536 : 49152, a.join * a.chunks * (a.span / a.d) * 64), 16384);
  chunks_for(a, env_int("NORM_AWG", (int)second), least_chunk(v), a.achunks, a.appc);
  return true;
}
template <typename T, int V, bool WHOLE> void launch_two_whole(const NormArgs& a, bool backward, hipStream_t st) {
  constexpr int TH = 256;
  const int ny = a.c / a.span;
  const dim3 g1(a.n * a.chunks, ny);
  if (backward) {
    const int pblocks = a.dgamma || a.dbeta ? (a.c + 15) / 16 : 0;
    hipLaunchKernelGGL((norm_chunk_sums_kernel<T, V, TH, WHOLE>), g1, dim3(TH), 0, st, a);
    if (!a.join) hipLaunchKernelGGL(norm_grad_join_kernel, dim3(a.n * a.groups), dim3(64), 0, st, a);
    hipLaunchKernelGGL((norm_chunk_grad_kernel<T, V, TH, WHOLE>), dim3(pblocks + a.n * a.achunks, ny), dim3(TH), 0, st, a, pblocks);
    return;
  }
  hipLaunchKernelGGL((norm_chunk_stats_kernel<T, V, TH>), g1, dim3(TH), 0, st, a);
  if (!a.join) {
    NormArgs b = a;
    b.jl = 6;
    hipLaunchKernelGGL(norm_join_kernel, dim3(a.n * a.groups), dim3(64), 0, st, b);
  }
  hipLaunchKernelGGL((norm_chunk_apply_kernel<T, V, TH, WHOLE>), dim3(a.n * a.achunks, ny), dim3(TH), 0, st, a);
}
template <typename T, int V> bool launch_two(NormArgs a, bool backward, hipStream_t st) {
  if (!two_tiling(a, V, sizeof(T), backward)) return false;
  const size_t bytes = (size_t)a.n * a.p * a.c * sizeof(T) * (backward ? 2 : 1);
  // Reads go past the caches where the 256 MB last-level cache could not keep them for the second launch (151 MB: 66 us against 69 with
  // non-temporal reads; 830 MB: 408 against 430 without).  Writes always do: what takes this form is beyond the L2 caches or near it, and the
  // last-level cache is read no faster than memory (7.3 against 7.5 TB/s).
  a.nt = bytes > (size_t)env_int("NORM_NT_MB", 256) << 20;
  if (a.slots == 1) launch_two_whole<T, V, true>(a, backward, st);
  else launch_two_whole<T, V, V == 1>(a, backward, st);
  return true;
}

// Any shape.
constexpr int JOIN_WIDE = 4096;                                // numbers a group from which its join takes 1024 threads (4 x 64 x 64 x 1031 float32,
                                                               // one group: 72 us, backward 96; 256 threads 252 and 188)
template <typename T, int V> void launch_any(NormArgs a, bool backward, hipStream_t st) {
  const int cv = (a.c + V - 1) / V, ny = (cv + 255) / 256;
  // (divided by ny: what the joins read is chunks * channels a group.  4 x 64 x 64 x 1031 float32 with joins of 256 threads, one group: 252 us, 1216
  // undivided; 1031 groups: 51 and 90; half as many chunks again 167 and 64)
  chunks_for(a, std::max(a.n, MOST_WORKGROUPS / ny), 8192, a.chunks, a.ppc);
  a.cb = (cv + ny - 1) / ny;
  a.rows = 256 / a.cb;
  const dim3 grid(a.n * a.chunks, ny), joins(a.n * a.groups);
  const bool wide = a.chunks * a.d > JOIN_WIDE && joins.x <= 0xffffffffu / 1024;         // (a grid holds less than 2^32 threads)
  if (!backward) {
    hipLaunchKernelGGL((norm_stats_kernel<T, V>), grid, dim3(256), 0, st, a);
    if (wide) hipLaunchKernelGGL(norm_stats_join_kernel<1024>, joins, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL(norm_stats_join_kernel<256>, joins, dim3(256), 0, st, a);
    hipLaunchKernelGGL((norm_apply_kernel<T, V>), grid, dim3(256), 0, st, a);
    return;
  }
  hipLaunchKernelGGL((norm_bwd_sums_kernel<T, V>), grid, dim3(256), 0, st, a);
  if (wide) hipLaunchKernelGGL(norm_bwd_join_kernel<1024>, joins, dim3(1024), 0, st, a);
  else hipLaunchKernelGGL(norm_bwd_join_kernel<256>, joins, dim3(256), 0, st, a);
  hipLaunchKernelGGL((norm_bwd_apply_kernel<T, V>), grid, dim3(256), 0, st, a);
  if (a.dgamma || a.dbeta) hipLaunchKernelGGL(norm_params_kernel, dim3((a.c + 15) / 16), dim3(256), 0, st, a, a.ab, a.n);
}
template <typename T, int V> void launch_v(const NormArgs& a, bool backward, hipStream_t st) {
  if (a.team >= 0) return launch_team<T, V>(a, backward, st);
  if (!launch_two<T, V>(a, backward, st)) launch_any<T, V>(a, backward, st);
}
template <typename T> void launch(const NormArgs& a, bool backward, hipStream_t st) {
  switch (norm_vec<T>(a)) {
    case 8: if constexpr (sizeof(T) == 2) launch_v<T, 8>(a, backward, st); break;
    case 4: launch_v<T, 4>(a, backward, st); break;
    case 2: launch_v<T, 2>(a, backward, st); break;
    default: launch_v<T, 1>(a, backward, st);
  }
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
// Where an operand lies: runs of `run` bytes, `step` bytes from one to the next, up to `end`; one run has run = step.
struct Place {
  uintptr_t at = 0, end = 0;
  size_t run = 0, step = 0;
  Place(const void* p, size_t bytes) {
    if (p) { at = (uintptr_t)p; end = at + bytes; run = step = bytes; }
  }
  Place(const void* p, size_t pixels, size_t c, size_t cs, size_t elem_bytes) : Place(p, ((pixels - 1) * cs + c) * elem_bytes) {
    if (p && pixels > 1 && cs != c) { run = c * elem_bytes; step = cs * elem_bytes; }
  }
  bool dense() const { return run == step; }
  bool same(const Place& o) const { return at == o.at && end == o.end && run == o.run && step == o.step; }
  // Whether they share a byte (runs at two steps whose ranges meet: taken to)
  bool meets(const Place& o) const {
    if (at >= o.end || o.at >= end || !run || !o.run) return false;
    if (dense() && o.dense()) return true;
    if (!dense() && !o.dense() && step != o.step) return true;
    const size_t every = dense() ? o.step : step;
    const size_t from = at >= o.at ? (at - o.at) % every : (every - (o.at - at) % every) % every;      // where a run of this begins, after one of the other's
    return from < std::min(o.run, every) || from + std::min(run, every) > every;
  }
};
// The device that a call's operands are on, null ones aside; -1 where one is not memory of a GPU or of another one than those before it (every
// pointer that a kernel goes to is among them: one to host memory would be a fault of the GPU), or where one that is written lies across
// another.  IN_PLACE: read, and an OUT may be the very same.
enum Use { READ, IN_PLACE, WRITTEN, OUT };
struct Operand { const char* name; Use use; Place place; };
int operands_device(std::initializer_list<Operand> operands, std::string& error) {
  int dev = -1;
  for (const Operand& o : operands) {
    if (!o.place.at) continue;
    const int d = device_of((const void*)o.place.at);
    if (d < 0) error = std::string(o.name) + " is not memory of a GPU";
    else if (dev >= 0 && d != dev) error = std::string(o.name) + " is memory of another GPU";
    if (!error.empty()) return -1;
    dev = d;
  }
  for (const Operand& w : operands)
    if (w.use >= WRITTEN)
      for (const Operand& o : operands)
        if (&w != &o && w.place.meets(o.place) && !(w.use == OUT && o.use == IN_PLACE && w.place.same(o.place))) {
          error = std::string(w.name) + " overlaps " + o.name;
          return -1;
        }
  return dev;
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
  a.n = n; a.p = h * w; a.c = c; a.groups = groups; a.d = c / groups; a.by_d = magic(a.d); a.act = act; a.inv_m = (float)(1.0 / ((double)a.p * a.d));
  a.mean = mean_rstd; a.rstd = mean_rstd + (size_t)n * groups;
  if ((uintptr_t)ws % 16) return bad("the workspace is not aligned to 16 bytes");
  a.team = team_variant(a, es == 4 ? norm_vec<float>(a) : norm_vec<f16_t>(a), (int)es, backward);
  const bool work = backward || a.team < 0;
  const WsLayout lay = work ? ws_layout(a, backward) : WsLayout{};
  if (work && (!ws || ws_bytes < lay.bytes())) return set_error(FISR_ENOMEM, std::string(who) + ": workspace too small");
  a.part = (float2*)ws;
  a.s12 = a.part + lay.part;
  a.ab = a.s12 + lay.s12;
  std::string error;
  const size_t pixels = (size_t)n * a.p, params = (size_t)c * sizeof(float);
  const int dev = operands_device({{"gamma", READ, {a.gamma, params}}, {"beta", READ, {a.beta, params}}, {"dgamma", WRITTEN, {a.dgamma, params}},
                                   {"dbeta", WRITTEN, {a.dbeta, params}}, {"d_counter", READ, {a.drop.counter, sizeof(uint64_t)}},
                                   {"mean_rstd", backward ? READ : WRITTEN, {mean_rstd, 2 * sizeof(float) * n * groups}},
                                   {"the workspace", WRITTEN, {ws, lay.bytes()}},
                                   {"dy", IN_PLACE, {a.dy, pixels, (size_t)c, a.dycs, es}}, {"x", IN_PLACE, {a.x, pixels, (size_t)c, a.xcs, es}},
                                   {backward ? "dx" : "y", OUT, {a.y, pixels, (size_t)c, a.ycs, es}}}, error);
  if (dev < 0) return bad(error.c_str());
  DeviceGuard guard(dev);
  NORM_HIP_OK(guard.err);
  const hipStream_t st = (hipStream_t)stream;
  if (type == FISR_TYPE_F32) launch<float>(a, backward, st);
  else if (type == FISR_TYPE_F16) launch<f16_t>(a, backward, st);
  else launch<b16_t>(a, backward, st);
  NORM_HIP_OK(hipGetLastError());
  return 0;
}

template <typename T> int launch_dropout(const T* x, const T* res, T* y, size_t count, const DropArgs& d, hipStream_t st) {
  if (((uintptr_t)x | (uintptr_t)res | (uintptr_t)y) % 16) {
    hipLaunchKernelGGL(dropout_any_kernel<T>, dim3(grid_for((count + 7) / 8)), dim3(256), 0, st, x, res, y, count, d);
    return 0;
  }
  const size_t per = (size_t)256 * (16 / sizeof(T)) * DROP_U, grid = (count + per - 1) / per, bytes = count * sizeof(T);
  if (grid >= 1u << 24) return -1;
  const dim3 g((unsigned)grid), b(256);
  // all accesses past the caches beyond 160 MB of reads (float32, 202 MB: 64 us against 74 plain; two inputs of 132 MB 62 against 71, of 94 MB 44.5 against
  // 43.9, of 75 MB 35.9 against 35.3); the writes alone where there is no residual and they pass the L2 caches (75 MB: 22.8 against 24.9; 38 MB 12.3
  // against 12.1, 94 MB 29.4 against 29.8, 132 MB 43.5 against 39.7; with a residual 35.4 against 35.3)
  if (bytes * (res ? 2 : 1) > (size_t)160 << 20) hipLaunchKernelGGL((dropout_kernel<T, true, true>), g, b, 0, st, x, res, y, count, d);
  else if (!res && bytes > (size_t)32 << 20) hipLaunchKernelGGL((dropout_kernel<T, false, true>), g, b, 0, st, x, res, y, count, d);
  else hipLaunchKernelGGL((dropout_kernel<T, false, false>), g, b, 0, st, x, res, y, count, d);
  return 0;
}

}  // namespace

extern "C" {

size_t fisr_train_groupnorm_workspace_bytes(int n, int h, int w, int c, int groups, int backward) {
  if (norm_shape_error(n, h, w, c, groups)) return 0;
  NormArgs a{};
  a.n = n; a.p = h * w; a.c = c; a.groups = groups;
  return ws_layout(a, backward != 0).bytes();
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
  std::string error;
  const int dev = operands_device({{"d_counter", READ, {d.counter, sizeof(uint64_t)}}, {"residual", IN_PLACE, {residual, count * es}}, {"x", IN_PLACE, {x, count * es}},
                                   {"y", OUT, {y, count * es}}}, error);
  if (dev < 0) return bad(error.c_str());
  DeviceGuard guard(dev);
  NORM_HIP_OK(guard.err);
  const hipStream_t st = (hipStream_t)stream;
  const auto run = [&](auto* t) {
    typedef std::remove_pointer_t<decltype(t)> T;
    return launch_dropout<T>((const T*)x, (const T*)residual, (T*)y, count, d, st);
  };
  if ((type == FISR_TYPE_F32 ? run((float*)nullptr) : type == FISR_TYPE_F16 ? run((f16_t*)nullptr) : run((b16_t*)nullptr)) < 0)
    return bad("more than 2^36 elements");
  NORM_HIP_OK(hipGetLastError());
  return 0;
}

}  // extern "C"
