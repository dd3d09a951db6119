// bindings.cpp -- torch-facing wrappers of the extern "C" launchers.
//
// Every op runs on the caller's current CUDA stream (so CUDA-graph capture
// and stream scoping compose with torch), checks devices, dtypes, shapes and
// alignment, and raises on a launcher error instead of returning silently.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cstdint>

#include "gemm_api.h"
#include "kv_budget_api.h"
#include "sched/abi.h"
#include "sp_api.h"

extern "C" {
int sched_attn_decode(const void *q, void *out, const void *k_cache, const void *v_cache,
                      int num_pages, const int32_t *block_table, int bt_stride, const void *items,
                      int num_items, int Hq, int Hkv, float sm_scale, float *part_o,
                      float *part_lse, uint32_t *merge_cnt, int splits, SchedSlots slots,
                      int woven, int acquire, int grid, int pf_blocks, float dT, float dR,
                      float H, const void *stage_k, const void *stage_v, int stage_pages,
                      int stage_split, const void *l2_prefetch, long long l2_prefetch_bytes, int *status,
                      cudaStream_t st);
int sched_attn_merge(const float *part_o, const float *part_lse, const int32_t *merge_req,
                     const int32_t *merge_begin, int rows, int Hq, void *out, cudaStream_t st);
int sched_attn_decode_occupancy(int group);
int sched_attn_decode_smem_bytes();
int sched_attn_prefill(const void *q, int q_rows, void *out, const void *k_cache, const void *v_cache,
                       int num_pages, const int32_t *block_table, int bt_stride,
                       const int32_t *kv_lens, const void *tiles, int num_tiles, int Hq, int Hkv,
                       int page_size, float sm_scale, int *status, cudaStream_t st);
int sched_attn_prefill_tile_rows();
int sched_add_rmsnorm(const void *x, void *res, const void *w, void *y, int T, int H, float eps,
                      cudaStream_t st);
int sched_rope_kv_append(const void *qkv, const int32_t *pos, const int32_t *slot,
                         const float *cos_sin, void *q_out, void *k_cache, void *v_cache, int T,
                         int Hq, int Hkv, int D, int page_size, int num_pages, int *status, cudaStream_t st);
int sched_embedding(const int32_t *ids, const int32_t *prev, int n_prev, const void *table, void *out, int T, int H,
                    int vocab, int *status, cudaStream_t st);
int sched_argmax(const void *logits, int T, int V, int ld, int32_t *ids, float *maxv,
                 int id_offset, cudaStream_t st);
int sched_moe_router(const void *x, const void *wr, int T, int H, int E, int K, int32_t *ids,
                     float *wts, cudaStream_t st);
int sched_moe_quantize(const void *in, int R, int I, void *out, float *scale,
                       const uint32_t *rows_valid, int rows_per_expert, cudaStream_t st);
int sched_moe_combine_norm(const void *c, int K, void *h, const void *w, void *y, int T, int H,
                           float eps, uint32_t *cnt, uint32_t *dropped_step, uint32_t *arrivals,
                           int *status, cudaStream_t st);
}
#include "moe_api.h"
extern "C" int sched_probe_stream(const void *src, size_t bytes, int policy, unsigned *sink, int grid,
                                  cudaStream_t st);
extern "C" int sched_probe_tasks(const uint32_t *cost, int n_tasks, int mode, int grid, int memory,
                                 const void *data, size_t data_bytes, unsigned *hits, unsigned *per_cta,
                                 unsigned *ticket, unsigned *sink, int *status, cudaStream_t st);
extern "C" int sched_probe_tasks_occupancy();
extern "C" void sched_attn_decode_set_trace(unsigned long long *trace);
extern "C" int sched_argmax_exchange(const void *logits, int T, int V, int ld, int32_t *ids, float *maxv,
                                     int id_offset, void *const *lines, int world, int rank, uint32_t *state,
                                     long long set_lines, int *status, cudaStream_t st);
extern "C" int sched_probe_clc_shape(const uint32_t *work, int gx, int gy, int gz, int stride, int cx,
                                     unsigned *hits, unsigned *claimed, unsigned *launched, unsigned *fails,
                                     unsigned *w_nonzero, int *status, cudaStream_t st);
extern "C" int sched_probe_clc_shape_capacity(int cx);
extern "C" int sched_probe_clc(const uint32_t *work, int n_tasks, int mode, int grid, int max_rec, unsigned *hits,
                               unsigned long long *rec, unsigned *n_rec, unsigned *smid, int *status,
                               cudaStream_t st);
extern "C" int sched_probe_mix(const void *R, size_t r_bytes, const void *S, size_t s_bytes, int mode, float frac,
                               unsigned *sink, int grid, cudaStream_t st);
extern "C" int sched_probe_pdl_pairs(float *buf, float *out, int n, const float *table, int work, int prologue,
                                     int pdl, int pairs, cudaStream_t st);
extern "C" int sched_probe_pdl_produce(float *buf, int n, int work, cudaStream_t st);
extern "C" int sched_kv_page_copy(const void *src_k, const void *src_v, long long src_pages, void *dst_k,
                                  void *dst_v, long long dst_pages, const int32_t *pairs, int n_pairs,
                                  const int *n_dev, int layers, int heads, int *status, cudaStream_t st);
extern "C" int sched_kv_page_copy_fp8(const void *src_k, const void *src_v, long long src_pages, void *dst_k,
                                      void *dst_v, long long dst_pages, float *scale_k, float *scale_v, int to_fp8,
                                      const int32_t *pairs, int n_pairs, const int *n_dev, int layers, int heads,
                                      int *status, cudaStream_t st);

namespace {

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_cuda(const at::Tensor &t, const char *name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
}
void check_bf16(const at::Tensor &t, const char *name) {
  check_cuda(t, name);
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bfloat16");
}
void check_i32(const at::Tensor &t, const char *name) {
  check_cuda(t, name);
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
// A launcher's non-zero return code is recorded here instead of thrown:
// throwing a c10::Error out of a binding after its CUDA device guard has
// run crashed the process (SIGSEGV) on the B200 boxes, while throws before
// the guard (argument checks) are translated normally. The Python wrapper
// of every launcher (_ext._Counted) calls take_error() after the call and
// raises there.
namespace {
thread_local int g_last_rc = 0;
thread_local const char *g_last_op = "";
}  // namespace
void check_rc(int rc, const char *op) {
  if (rc != 0 && g_last_rc == 0) {
    g_last_rc = rc;
    g_last_op = op;
  }
}
std::tuple<int64_t, std::string> take_error() {
  std::tuple<int64_t, std::string> r{g_last_rc, std::string(g_last_op)};
  g_last_rc = 0;
  g_last_op = "";
  return r;
}

template <typename T>
T *ptr_or_null(const c10::optional<at::Tensor> &t) {
  return (t.has_value() && t->defined()) ? static_cast<T *>(t->data_ptr()) : nullptr;
}

// ---------------------------------------------------------------- GEMM
int num_sms(const at::Tensor &t) {
  static int n[64] = {0};
  const int d = t.get_device();
  if (d >= 0 && d < 64) {
    if (n[d] == 0) n[d] = at::cuda::getDeviceProperties(d)->multiProcessorCount;
    return n[d];
  }
  return 148;
}

// Diagnostic: when set, every GEMM launch records per-CTA timestamps here.
unsigned long long *g_gemm_trace = nullptr;
void set_attn_trace(int64_t ptr) { sched_attn_decode_set_trace(reinterpret_cast<unsigned long long *>(ptr)); }
void set_gemm_trace(int64_t ptr) { g_gemm_trace = reinterpret_cast<unsigned long long *>(ptr); }

// Residual add + RMSNorm fused after the projection: res += y, out = rmsnorm(res) * nw
// (all [T, N] bf16 except nw [N]); row_cnt int32 [>= T], zero between calls.
void set_norm(GemmArgs &a, const c10::optional<at::Tensor> &res, const c10::optional<at::Tensor> &nw,
              const c10::optional<at::Tensor> &out, const c10::optional<at::Tensor> &row_cnt, double eps) {
  if (!(nw.has_value() && nw->defined())) return;
  TORCH_CHECK(res.has_value() && out.has_value() && row_cnt.has_value(), "fused norm needs res, out and row_cnt");
  check_bf16(*res, "norm res");
  check_bf16(*nw, "norm weight");
  check_bf16(*out, "norm out");
  check_i32(*row_cnt, "row_cnt");
  TORCH_CHECK(res->is_contiguous() && out->is_contiguous() && nw->is_contiguous(), "contiguous norm tensors");
  TORCH_CHECK(res->dim() == 2 && res->size(0) >= a.T && res->size(1) == a.N && out->sizes() == res->sizes() &&
                  nw->numel() == a.N && row_cnt->numel() >= a.T,
              "norm tensors: res/out [>= T, N], weight [N], row_cnt [>= T]");
  a.norm_res = reinterpret_cast<__nv_bfloat16 *>(res->data_ptr());
  a.norm_w = reinterpret_cast<const __nv_bfloat16 *>(nw->data_ptr());
  a.norm_out = reinterpret_cast<__nv_bfloat16 *>(out->data_ptr());
  a.row_cnt = reinterpret_cast<uint32_t *>(row_cnt->data_ptr<int32_t>());
  a.norm_eps = (float)eps;
}

GemmArgs base_args(const at::Tensor &x, const at::Tensor &w, int64_t grid,
                   const c10::optional<at::Tensor> &ws, const c10::optional<at::Tensor> &counters,
                   const c10::optional<at::Tensor> &status) {
  check_bf16(x, "x");
  check_bf16(w, "w");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2, "gemm expects 2-D operands");
  TORCH_CHECK(x.stride(1) == 1 && w.is_contiguous(), "row-major operands");
  TORCH_CHECK(w.size(1) == x.size(1), "K mismatch");
  GemmArgs a{};
  a.x = x.data_ptr();
  a.ldx = x.stride(0);
  a.w = w.data_ptr();
  a.T = x.size(0);
  a.K = x.size(1);
  a.N = w.size(0);
  a.grid = grid;
  a.num_sms = num_sms(x);
  a.trace = g_gemm_trace;
  a.ws = ptr_or_null<float>(ws);
  a.ws_floats = (ws.has_value() && ws->defined()) ? ws->numel() : 0;
  a.counters = ptr_or_null<uint32_t>(counters);
  a.counter_count = (counters.has_value() && counters->defined()) ? counters->numel() : 0;
  a.status = ptr_or_null<int>(status);
  return a;
}

// x_ready: address of the gathered rows' ready flags (0: x is local and ready)
void gemm(const at::Tensor &x, const at::Tensor &w, at::Tensor &y, int64_t epi, int64_t grid,
          const c10::optional<at::Tensor> &ws, const c10::optional<at::Tensor> &counters,
          const c10::optional<at::Tensor> &status, int64_t x_ready, const c10::optional<at::Tensor> &norm_res,
          const c10::optional<at::Tensor> &norm_w, const c10::optional<at::Tensor> &norm_out,
          const c10::optional<at::Tensor> &row_cnt, double norm_eps) {
  GemmArgs a = base_args(x, w, grid, ws, counters, status);
  a.x_ready = reinterpret_cast<const uint32_t *>(x_ready);
  check_bf16(y, "y");
  TORCH_CHECK(y.dim() == 2 && y.stride(1) == 1 && y.size(0) >= a.T, "y [T, ldy]");
  TORCH_CHECK(epi == kEpiStore ? y.size(1) >= a.N : y.size(1) >= a.N / 2, "y columns");
  TORCH_CHECK(epi == kEpiStore || epi == kEpiSwiGLU, "use gemm_qkv_rope for the QKV epilogue");
  a.y = y.data_ptr();
  a.ldy = y.stride(0);
  a.epi = epi;
  TORCH_CHECK(!(norm_w.has_value() && norm_w->defined()) || epi == kEpiStore, "the fused norm follows a plain store");
  set_norm(a, norm_res, norm_w, norm_out, row_cnt, norm_eps);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(x.device());
    rc_ = sched_gemm_run(&a, cur_stream());
  }
  check_rc(rc_, "gemm");
}

void gemm_qkv_rope(const at::Tensor &x, const at::Tensor &w, const at::Tensor &pos,
                   const at::Tensor &slot, const at::Tensor &cos_sin, at::Tensor &q_out,
                   at::Tensor &k_cache, at::Tensor &v_cache, int64_t Hq, int64_t Hkv,
                   int64_t grid, const c10::optional<at::Tensor> &ws,
                   const c10::optional<at::Tensor> &counters,
                   const c10::optional<at::Tensor> &status, int64_t x_ready) {
  GemmArgs a = base_args(x, w, grid, ws, counters, status);
  a.x_ready = reinterpret_cast<const uint32_t *>(x_ready);
  check_i32(pos, "pos");
  check_i32(slot, "slot");
  check_bf16(q_out, "q_out");
  check_bf16(k_cache, "k_cache");
  check_bf16(v_cache, "v_cache");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.is_contiguous(), "cos_sin float32");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.size(3) == 128 && k_cache.is_contiguous(), "cache layout");
  TORCH_CHECK(q_out.is_contiguous() && q_out.numel() >= a.T * Hq * 128, "q_out [T, Hq, 128]");
  a.epi = kEpiRopeKV;
  a.pos = pos.data_ptr<int32_t>();
  a.slot = slot.data_ptr<int32_t>();
  a.cos_sin = cos_sin.data_ptr<float>();
  a.q_out = reinterpret_cast<__nv_bfloat16 *>(q_out.data_ptr());
  a.k_cache = reinterpret_cast<__nv_bfloat16 *>(k_cache.data_ptr());
  a.v_cache = reinterpret_cast<__nv_bfloat16 *>(v_cache.data_ptr());
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.page_size = k_cache.size(2);
  a.kv_pages = k_cache.size(0);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(x.device());
    rc_ = sched_gemm_run(&a, cur_stream());
  }
  check_rc(rc_, "gemm_qkv_rope");
}

// Row-parallel projection with the all-reduce fused into the GEMM epilogue.
// recv/flags: this process's addresses of every rank's slab and flag array.
// ll_state (int32 [2] on this device) selects the low-latency exchange:
// recv then holds every rank's line buffer (two sets of ll_set_lines
// 16-byte lines) and flags is ignored.
void gemm_allreduce(const at::Tensor &x, const at::Tensor &w, at::Tensor &y, int64_t rank,
                    int64_t world, const std::vector<int64_t> &recv,
                    const std::vector<int64_t> &flags, int64_t grid,
                    const c10::optional<at::Tensor> &ws,
                    const c10::optional<at::Tensor> &counters,
                    const c10::optional<at::Tensor> &status,
                    const c10::optional<at::Tensor> &ll_state, int64_t ll_set_lines,
                    const c10::optional<at::Tensor> &norm_res, const c10::optional<at::Tensor> &norm_w,
                    const c10::optional<at::Tensor> &norm_out, const c10::optional<at::Tensor> &row_cnt,
                    double norm_eps, int64_t ll_mc) {
  GemmArgs a = base_args(x, w, grid, ws, counters, status);
  check_bf16(y, "y");
  TORCH_CHECK(y.dim() == 2 && y.stride(1) == 1 && y.size(1) >= a.N, "y [T, >= N]");
  const bool ll = ll_state.has_value() && ll_state->defined();
  TORCH_CHECK(world >= 1 && world <= kMaxWorld && (int64_t)recv.size() == world &&
                  (ll || (int64_t)flags.size() == world),
              "one slab and one flag array per rank");
  if (ll) {
    check_i32(*ll_state, "ll_state");
    TORCH_CHECK(ll_state->numel() >= 2 && ll_state->device() == x.device(), "ll_state: int32 [2] on x's device");
    TORCH_CHECK(ll_set_lines >= world * a.T * (a.N / 4), "line buffer too small for [world, T, N/4] lines");
  }
  a.y = y.data_ptr();
  a.ldy = y.stride(0);
  a.epi = kEpiAllReduce;
  a.rank = rank;
  a.world = world;
  for (int j = 0; j < world; ++j) {
    a.recv[j] = reinterpret_cast<__nv_bfloat16 *>(recv[j]);
    a.flags[j] = ll ? nullptr : reinterpret_cast<uint32_t *>(flags[j]);
  }
  if (ll) {
    a.ll_state = reinterpret_cast<uint32_t *>(ll_state->data_ptr<int32_t>());
    a.ll_set_lines = ll_set_lines;
    a.ll_mc = reinterpret_cast<void *>(ll_mc);
  }
  set_norm(a, norm_res, norm_w, norm_out, row_cnt, norm_eps);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(x.device());
    rc_ = sched_gemm_run(&a, cur_stream());
  }
  check_rc(rc_, "gemm_allreduce");
}

// Row-parallel projection, sequence-parallel output: each finished row goes
// to the slab of the rank that owns the token (kEpiReduceScatter); the owner
// reduces it in sp_reduce_norm. recv/flags: every rank's slab and row flags.
void gemm_reduce_scatter(const at::Tensor &x, const at::Tensor &w, int64_t rank, int64_t world,
                         const std::vector<int64_t> &recv, const std::vector<int64_t> &flags,
                         int64_t grid, const c10::optional<at::Tensor> &ws,
                         const c10::optional<at::Tensor> &counters,
                         const c10::optional<at::Tensor> &status) {
  GemmArgs a = base_args(x, w, grid, ws, counters, status);
  TORCH_CHECK(world >= 1 && world <= kMaxWorld && (int64_t)recv.size() == world &&
                  (int64_t)flags.size() == world,
              "one slab and one flag array per rank");
  a.epi = kEpiReduceScatter;
  a.rank = rank;
  a.world = world;
  for (int j = 0; j < world; ++j) {
    a.recv[j] = reinterpret_cast<__nv_bfloat16 *>(recv[j]);
    a.flags[j] = reinterpret_cast<uint32_t *>(flags[j]);
  }
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(x.device());
    rc_ = sched_gemm_run(&a, cur_stream());
  }
  check_rc(rc_, "gemm_reduce_scatter");
}

// Sequence-parallel reduce + residual + RMSNorm + all-gather push (sp_api.h).
void sp_reduce_norm(int64_t slab, int64_t row_flags, at::Tensor &res, const at::Tensor &w,
                    const c10::optional<at::Tensor> &delta, const std::vector<int64_t> &gather,
                    const std::vector<int64_t> &ready, int64_t clear, int64_t clear_n, int64_t T,
                    int64_t rank, int64_t world, double eps, const c10::optional<at::Tensor> &status) {
  check_bf16(res, "res");
  check_bf16(w, "w");
  TORCH_CHECK(res.dim() == 2 && res.is_contiguous() && res.size(0) >= T, "res [>= T, H] contiguous");
  const int64_t H = res.size(1);
  TORCH_CHECK(w.numel() == H && w.is_contiguous(), "w [H]");
  TORCH_CHECK(world >= 1 && world <= kMaxWorld && (int64_t)gather.size() == world &&
                  (int64_t)ready.size() == world && rank >= 0 && rank < world,
              "one gather buffer and one ready array per rank");
  SpNormArgs a{};
  a.slab = reinterpret_cast<const __nv_bfloat16 *>(slab);
  a.row_flags = reinterpret_cast<uint32_t *>(row_flags);
  a.res = reinterpret_cast<__nv_bfloat16 *>(res.data_ptr());
  a.w = reinterpret_cast<const __nv_bfloat16 *>(w.data_ptr());
  if (delta.has_value() && delta->defined()) {
    check_bf16(*delta, "delta");
    TORCH_CHECK(delta->is_contiguous() && delta->size(0) >= T && delta->size(1) == H, "delta [>= T, H]");
    a.delta = reinterpret_cast<__nv_bfloat16 *>(delta->data_ptr());
  }
  for (int j = 0; j < world; ++j) {
    a.gather[j] = reinterpret_cast<__nv_bfloat16 *>(gather[j]);
    a.ready[j] = reinterpret_cast<uint32_t *>(ready[j]);
  }
  a.clear = reinterpret_cast<uint32_t *>(clear);
  a.clear_n = clear_n;
  a.T = T;
  a.H = H;
  a.rank = rank;
  a.world = world;
  a.eps = (float)eps;
  a.status = ptr_or_null<int>(status);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(res.device());
    rc_ = sched_sp_reduce_norm(&a, cur_stream());
  }
  check_rc(rc_, "sp_reduce_norm");
}

void sp_wait_rows(int64_t ready, int64_t T, const at::Tensor &status) {
  check_cuda(status, "status");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(status.device());
    rc_ = sched_sp_wait_rows(reinterpret_cast<const uint32_t *>(ready), T,
                                static_cast<int *>(status.data_ptr()), cur_stream());
  }
  check_rc(rc_, "sp_wait_rows");
}

int64_t gemm_ws_floats(int64_t T, int64_t N, int64_t K, int64_t grid) {
  return sched_gemm_ws_floats(T, N, K, grid);
}

// ---------------------------------------------------------------- attention
SchedSlots make_slots(const c10::optional<at::Tensor> &order, const c10::optional<at::Tensor> &ctrl,
                      const c10::optional<at::Tensor> &timer, const c10::optional<at::Tensor> &queue,
                      int64_t max_tasks) {
  SchedSlots s{};
  s.order = ptr_or_null<const int32_t>(order);
  s.ctrl = ptr_or_null<const SchedCtrl>(ctrl);
  s.timer = ptr_or_null<unsigned long long>(timer);
  s.queue = ptr_or_null<uint32_t>(queue);
  s.max_tasks = static_cast<uint32_t>(max_tasks);
  return s;
}

void attn_decode(const at::Tensor &q, at::Tensor &out, const at::Tensor &k_cache,
                 const at::Tensor &v_cache, const at::Tensor &block_table, const at::Tensor &items,
                 int64_t num_items, double sm_scale, const c10::optional<at::Tensor> &part_o,
                 const c10::optional<at::Tensor> &part_lse,
                 const c10::optional<at::Tensor> &merge_cnt, int64_t splits,
                 const c10::optional<at::Tensor> &order, const c10::optional<at::Tensor> &ctrl,
                 const c10::optional<at::Tensor> &timer, const c10::optional<at::Tensor> &queue,
                 int64_t max_tasks, int64_t woven, int64_t acquire, int64_t grid,
                 int64_t pf_blocks, double dT, double dR, double H,
                 const c10::optional<at::Tensor> &stage_k, const c10::optional<at::Tensor> &stage_v,
                 int64_t stage_split, const c10::optional<at::Tensor> &status, int64_t l2_prefetch,
                 int64_t l2_prefetch_bytes) {
  check_bf16(q, "q");
  check_bf16(out, "out");
  check_bf16(k_cache, "k_cache");
  const bool staged = stage_k.has_value() && stage_k->defined();
  if (staged) {
    TORCH_CHECK(stage_v.has_value() && stage_v->defined() && stage_k->is_contiguous() && stage_v->is_contiguous() &&
                    stage_k->dim() == 4 && stage_k->size(1) == k_cache.size(1),
                "staging pool [pages, Hkv, 16, 128]");
  }
  check_bf16(v_cache, "v_cache");
  check_i32(block_table, "block_table");
  check_i32(items, "items");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 128 && q.is_contiguous(), "q [B, Hq, 128]");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.size(2) == 16 && k_cache.size(3) == 128 &&
                  k_cache.is_contiguous() && v_cache.sizes() == k_cache.sizes(),
              "cache [pages, Hkv, 16, 128]");
  TORCH_CHECK(items.numel() >= num_items * 4, "items [n, 4]");
  const int Hq = q.size(1), Hkv = k_cache.size(1);
  TORCH_CHECK(Hkv > 0 && Hq % Hkv == 0 && (Hq / Hkv == 1 || Hq / Hkv == 2 || Hq / Hkv == 4 || Hq / Hkv == 8),
              "query heads per KV head must be 1, 2, 4 or 8");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(q.device());
    SchedSlots sl = make_slots(order, ctrl, timer, queue, max_tasks);
    rc_ = sched_attn_decode(q.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                               k_cache.size(0), block_table.data_ptr<int32_t>(),
                               block_table.stride(0), items.data_ptr(), num_items, Hq, Hkv,
                               (float)sm_scale, ptr_or_null<float>(part_o),
                               ptr_or_null<float>(part_lse), ptr_or_null<uint32_t>(merge_cnt),
                               splits, sl, woven, acquire, grid, pf_blocks,
                               (float)dT, (float)dR, (float)H, staged ? stage_k->data_ptr() : nullptr,
                               staged ? stage_v->data_ptr() : nullptr, staged ? (int)stage_k->size(0) : 0,
                               (int)stage_split, reinterpret_cast<const void *>(l2_prefetch),
                               (long long)l2_prefetch_bytes, ptr_or_null<int>(status), cur_stream());
  }
  check_rc(rc_, "attn_decode");
}

void attn_merge(const at::Tensor &part_o, const at::Tensor &part_lse, const at::Tensor &merge_req,
                const at::Tensor &merge_begin, int64_t rows, at::Tensor &out) {
  check_i32(merge_req, "merge_req");
  check_i32(merge_begin, "merge_begin");
  check_bf16(out, "out");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(out.device());
    rc_ = sched_attn_merge(part_o.data_ptr<float>(), part_lse.data_ptr<float>(),
                              merge_req.data_ptr<int32_t>(), merge_begin.data_ptr<int32_t>(), rows,
                              out.size(1), out.data_ptr(), cur_stream());
  }
  check_rc(rc_, "attn_merge");
}

void attn_prefill(const at::Tensor &q, at::Tensor &out, const at::Tensor &k_cache,
                  const at::Tensor &v_cache, const at::Tensor &block_table,
                  const at::Tensor &kv_lens, const at::Tensor &tiles, int64_t num_tiles,
                  double sm_scale, const c10::optional<at::Tensor> &status) {
  check_bf16(q, "q");
  check_bf16(out, "out");
  check_bf16(k_cache, "k_cache");
  check_bf16(v_cache, "v_cache");
  check_i32(block_table, "block_table");
  check_i32(kv_lens, "kv_lens");
  check_i32(tiles, "tiles");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 128 && q.is_contiguous(), "q [T, Hq, 128]");
  TORCH_CHECK(out.sizes() == q.sizes() && out.is_contiguous(), "out like q");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.size(2) == 16 && k_cache.size(3) == 128 &&
                  k_cache.is_contiguous() && v_cache.sizes() == k_cache.sizes() && v_cache.is_contiguous(),
              "cache [pages, Hkv, 16, 128]");
  TORCH_CHECK(k_cache.size(1) > 0 && q.size(1) % k_cache.size(1) == 0, "query heads per KV head");
  TORCH_CHECK(tiles.numel() >= num_tiles * 4 && tiles.is_contiguous(), "tiles [n, 4]");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(q.device());
    rc_ = sched_attn_prefill(q.data_ptr(), q.size(0), out.data_ptr(), k_cache.data_ptr(),
                             v_cache.data_ptr(), k_cache.size(0), block_table.data_ptr<int32_t>(), block_table.stride(0),
                             kv_lens.data_ptr<int32_t>(), tiles.data_ptr(), num_tiles, q.size(1),
                             k_cache.size(1), k_cache.size(2), (float)sm_scale,
                             ptr_or_null<int>(status), cur_stream());
  }
  check_rc(rc_, "attn_prefill");
}

int64_t attn_decode_occupancy(int64_t group) { return sched_attn_decode_occupancy(group); }
int64_t attn_decode_smem_bytes() { return sched_attn_decode_smem_bytes(); }

// ---------------------------------------------------------------- elementwise
void add_rmsnorm(const at::Tensor &x, const c10::optional<at::Tensor> &res, const at::Tensor &w,
                 at::Tensor &y, double eps) {
  check_bf16(x, "x");
  check_bf16(w, "w");
  check_bf16(y, "y");
  TORCH_CHECK(x.is_contiguous() && y.is_contiguous(), "contiguous rows");
  const int H = x.size(-1), T = x.numel() / H;
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(x.device());
    rc_ = sched_add_rmsnorm(x.data_ptr(), res.has_value() ? res->data_ptr() : nullptr,
                               w.data_ptr(), y.data_ptr(), T, H, (float)eps, cur_stream());
  }
  check_rc(rc_, "add_rmsnorm");
}

void rope_kv_append(const at::Tensor &qkv, const at::Tensor &pos, const at::Tensor &slot,
                    const at::Tensor &cos_sin, at::Tensor &q_out, at::Tensor &k_cache,
                    at::Tensor &v_cache, int64_t Hq, int64_t Hkv, const c10::optional<at::Tensor> &status) {
  check_bf16(qkv, "qkv");
  check_i32(pos, "pos");
  check_i32(slot, "slot");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.is_contiguous(), "cos_sin float32");
  const int T = qkv.size(0);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(qkv.device());
    rc_ = sched_rope_kv_append(qkv.data_ptr(), pos.data_ptr<int32_t>(), slot.data_ptr<int32_t>(),
                                  cos_sin.data_ptr<float>(), q_out.data_ptr(), k_cache.data_ptr(),
                                  v_cache.data_ptr(), T, Hq, Hkv, k_cache.size(3), k_cache.size(2),
                                  k_cache.size(0), ptr_or_null<int>(status), cur_stream());
  }
  check_rc(rc_, "rope_kv_append");
}

void embedding(const at::Tensor &ids, const at::Tensor &table, at::Tensor &out,
               const c10::optional<at::Tensor> &status, const c10::optional<at::Tensor> &prev) {
  check_i32(ids, "ids");
  check_bf16(table, "table");
  const bool has_prev = prev.has_value() && prev->defined();
  if (has_prev) check_i32(*prev, "prev");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(ids.device());
    rc_ = sched_embedding(ids.data_ptr<int32_t>(), has_prev ? prev->data_ptr<int32_t>() : nullptr,
                             has_prev ? (int)prev->numel() : 0, table.data_ptr(), out.data_ptr(), ids.numel(),
                             table.size(1), table.size(0), ptr_or_null<int>(status), cur_stream());
  }
  check_rc(rc_, "embedding");
}

void argmax_exchange(const at::Tensor &logits, at::Tensor &ids, int64_t id_offset,
                     const std::vector<int64_t> &lines, int64_t rank, at::Tensor &state, int64_t set_lines,
                     const c10::optional<at::Tensor> &status) {
  check_bf16(logits, "logits");
  check_i32(ids, "ids");
  check_i32(state, "state");
  const int64_t world = (int64_t)lines.size();
  TORCH_CHECK(world >= 1 && world <= 8 && rank >= 0 && rank < world, "one line buffer per rank (<= 8)");
  TORCH_CHECK(state.numel() >= 2 && set_lines >= world * logits.size(0), "state [2]; set_lines >= world x rows");
  std::vector<void *> ptrs(world);
  for (int64_t j = 0; j < world; ++j) ptrs[j] = reinterpret_cast<void *>(lines[j]);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(logits.device());
    rc_ = sched_argmax_exchange(logits.data_ptr(), logits.size(0), logits.size(1), logits.stride(0),
                                ids.data_ptr<int32_t>(), nullptr, id_offset, ptrs.data(), (int)world, (int)rank,
                                reinterpret_cast<uint32_t *>(state.data_ptr<int32_t>()), set_lines,
                                ptr_or_null<int>(status), cur_stream());
  }
  check_rc(rc_, "argmax_exchange");
}

void argmax(const at::Tensor &logits, at::Tensor &ids, const c10::optional<at::Tensor> &maxv,
            int64_t id_offset) {
  check_bf16(logits, "logits");
  check_i32(ids, "ids");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(logits.device());
    rc_ = sched_argmax(logits.data_ptr(), logits.size(0), logits.size(1), logits.stride(0),
                          ids.data_ptr<int32_t>(), ptr_or_null<float>(maxv), id_offset, cur_stream());
  }
  check_rc(rc_, "argmax");
}

// ---------------------------------------------------------------- MoE
void moe_router(const at::Tensor &x, const at::Tensor &wr, at::Tensor &ids, at::Tensor &wts, int64_t k) {
  check_bf16(x, "x");
  check_bf16(wr, "wr");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(x.device());
    rc_ = sched_moe_router(x.data_ptr(), wr.data_ptr(), x.size(0), x.size(1), wr.size(0), k,
                              ids.data_ptr<int32_t>(), wts.data_ptr<float>(), cur_stream());
  }
  check_rc(rc_, "moe_router");
}

// p: dict-like flat vector of int64 arguments (see sched_pass_b200/parallel/ep.py)
void moe_dispatch(const at::Tensor &x, const at::Tensor &ids, const at::Tensor &wts, int64_t T,
                  int64_t K, int64_t E, int64_t E_local, int64_t rank, int64_t world, int64_t capacity,
                  int64_t rows, const std::vector<int64_t> &slab, const std::vector<int64_t> &slab_scale,
                  const std::vector<int64_t> &slab_meta, const std::vector<int64_t> &counter,
                  const std::vector<int64_t> &done, int64_t local_done, int64_t combine_local,
                  int64_t dropped_step, int64_t dropped_total, const c10::optional<at::Tensor> &status) {
  moe::DispatchArgs a{};
  a.x = reinterpret_cast<const __nv_bfloat16 *>(x.data_ptr());
  a.ids = ids.data_ptr<int32_t>();
  a.wts = wts.data_ptr<float>();
  a.T = T;
  a.H = x.size(1);
  a.K = K;
  a.E = E;
  a.E_local = E_local;
  a.rank = rank;
  a.world = world;
  a.capacity = capacity;
  a.rows_per_expert = rows;
  for (int r = 0; r < world; ++r) {
    a.slab[r] = reinterpret_cast<uint8_t *>(slab[r]);
    a.slab_scale[r] = reinterpret_cast<float *>(slab_scale[r]);
    a.slab_meta[r] = reinterpret_cast<int32_t *>(slab_meta[r]);
    a.counter[r] = reinterpret_cast<uint32_t *>(counter[r]);
    a.done[r] = reinterpret_cast<uint32_t *>(done[r]);
  }
  a.local_done = reinterpret_cast<uint32_t *>(local_done);
  a.combine_local = reinterpret_cast<__nv_bfloat16 *>(combine_local);
  a.dropped_step = reinterpret_cast<uint32_t *>(dropped_step);
  a.dropped_total = reinterpret_cast<uint32_t *>(dropped_total);
  a.status = ptr_or_null<int>(status);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(x.device());
    rc_ = sched_moe_dispatch(&a, cur_stream());
  }
  check_rc(rc_, "moe_dispatch");
}

void moe_expert_gemm(int64_t epi, const at::Tensor &w, int64_t x_ptr, int64_t E_local, int64_t N, int64_t K,
                     int64_t rows, const at::Tensor &w_scale, int64_t x_scale, int64_t act, int64_t counter,
                     int64_t done, int64_t rows_valid, int64_t tiles_done, int64_t world, int64_t capacity,
                     int64_t meta, const std::vector<int64_t> &combine, const std::vector<int64_t> &combine_cnt,
                     int64_t k_top, int64_t ws, int64_t tile_counters, int64_t grid, int64_t trace,
                     const c10::optional<at::Tensor> &status) {
  TORCH_CHECK(w.is_cuda() && w.element_size() == 1, "w: fp8 e4m3 [E_local * N, K]");
  moe::ExpertArgs a{};
  a.E_local = E_local;
  a.N = N;
  a.K = K;
  a.rows_per_expert = rows;
  a.w_scale = w_scale.data_ptr<float>();
  a.x_scale = reinterpret_cast<const float *>(x_scale);
  a.act = reinterpret_cast<__nv_bfloat16 *>(act);
  a.counter = reinterpret_cast<uint32_t *>(counter);
  a.done = reinterpret_cast<uint32_t *>(done);
  a.rows_valid = reinterpret_cast<uint32_t *>(rows_valid);
  a.tiles_done = reinterpret_cast<uint32_t *>(tiles_done);
  a.world = world;
  a.capacity = capacity;
  a.meta = reinterpret_cast<const int32_t *>(meta);
  for (size_t r = 0; r < combine.size() && r < moe::kMaxWorld; ++r) {
    a.combine[r] = reinterpret_cast<__nv_bfloat16 *>(combine[r]);
    a.combine_cnt[r] = reinterpret_cast<uint32_t *>(combine_cnt[r]);
  }
  a.k_top = k_top;
  a.ws = reinterpret_cast<float *>(ws);
  a.tile_counters = reinterpret_cast<uint32_t *>(tile_counters);
  a.grid = grid;
  a.trace = reinterpret_cast<unsigned long long *>(trace);
  a.status = ptr_or_null<int>(status);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(w.device());
    rc_ = sched_moe_expert_gemm(epi, w.data_ptr(), reinterpret_cast<const void *>(x_ptr), &a, cur_stream());
  }
  check_rc(rc_, "moe_expert_gemm");
}

void moe_quantize(int64_t in, int64_t R, int64_t I, int64_t out, int64_t scale, int64_t rows_valid,
                  int64_t rows) {
  check_rc(sched_moe_quantize(reinterpret_cast<const void *>(in), R, I, reinterpret_cast<void *>(out),
                              reinterpret_cast<float *>(scale), reinterpret_cast<const uint32_t *>(rows_valid),
                              rows, cur_stream()),
           "moe_quantize");
}

void moe_combine_norm(int64_t c, int64_t K, at::Tensor &h, const at::Tensor &w, at::Tensor &y, int64_t T,
                      double eps, int64_t cnt, int64_t dropped_step, int64_t arrivals,
                      const c10::optional<at::Tensor> &status) {
  check_bf16(h, "h");
  check_bf16(y, "y");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(h.device());
    rc_ = sched_moe_combine_norm(reinterpret_cast<const void *>(c), K, h.data_ptr(), w.data_ptr(), y.data_ptr(), T,
                                    h.size(1), (float)eps, reinterpret_cast<uint32_t *>(cnt),
                                    reinterpret_cast<uint32_t *>(dropped_step), reinterpret_cast<uint32_t *>(arrivals),
                                    ptr_or_null<int>(status), cur_stream());
  }
  check_rc(rc_, "moe_combine_norm");
}

// The status words of a device (int32 x 4, zero), for the life of the process,
// with a CUDA error code (thrown by the caller: see check_rc). They come from
// the driver and not from torch's allocator, and are zeroed before this
// returns, on a stream of their own: so a first use inside a graph capture
// puts neither the memory nor the zero fill into the graph, whose replays
// would erase reports, and a first use on one stream is in order for all.
std::tuple<int64_t, c10::optional<at::Tensor>> status_words(int64_t device) {
  int32_t *p = nullptr;
  cudaError_t rc = cudaSuccess;
  {
    c10::cuda::CUDAGuard g((c10::DeviceIndex)device);
    cudaStream_t st = nullptr;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // of this thread: a capture elsewhere takes no part
    if (rc = cudaThreadExchangeStreamCaptureMode(&mode); rc == cudaSuccess) {
      rc = cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking);
      if (rc == cudaSuccess) rc = cudaMalloc(reinterpret_cast<void **>(&p), 4 * sizeof(int32_t));
      if (rc == cudaSuccess) rc = cudaMemsetAsync(p, 0, 4 * sizeof(int32_t), st);
      if (rc == cudaSuccess) rc = cudaStreamSynchronize(st);
      if (st != nullptr) cudaStreamDestroy(st);
      cudaThreadExchangeStreamCaptureMode(&mode);
    }
  }
  if (rc != cudaSuccess) return {(int64_t)rc, c10::nullopt};
  return {0, at::from_blob(p, {4}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, (c10::DeviceIndex)device))};
}

// ---------------------------------------------------------------- KV budget (kv_budget_api.h)
// Shapes and types are checked before devices, so that a wrong call is refused
// the same way on a machine without a GPU.
int kv_element(const at::Tensor &t, const char *name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name, " must be bfloat16 or float16");
  return t.scalar_type() == at::kHalf ? kKvFp16 : kKvBf16;
}
void check_same(const at::Tensor &t, const at::Tensor &as, const char *name) {
  TORCH_CHECK(t.scalar_type() == as.scalar_type(), name, " must have the cache's type");
}
void check_on(const at::Tensor &t, const at::Tensor &as, const char *name) {
  check_cuda(t, name);
  TORCH_CHECK(t.device() == as.device(), name, " must be on the cache's device");
}
void check_vec(const at::Tensor &t, at::ScalarType type, int64_t n, const char *name, const char *type_name) {
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type_name);
  // (a number streamed into the message crashes the process here; a string does not)
  TORCH_CHECK(t.dim() == 1 && t.is_contiguous() && t.size(0) >= n, name, " must be contiguous with at least ",
              std::to_string(n), " entries");
}
// k, v [pages, Hkv, page_size, D], contiguous, D 64 or 128
void check_cache(const at::Tensor &k, const at::Tensor &v) {
  kv_element(k, "k_cache");
  check_same(v, k, "v_cache");
  TORCH_CHECK(k.dim() == 4 && k.is_contiguous() && v.is_contiguous() && v.sizes() == k.sizes(),
              "k_cache and v_cache must be contiguous [pages, kv heads, page size, head dim] of one shape");
  TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128, "head dim must be 64 or 128");
  TORCH_CHECK(k.size(0) >= 1 && k.size(1) >= 1 && k.size(2) >= 1, "the cache must not be empty");
  TORCH_CHECK(k.size(0) <= INT32_MAX && k.size(1) <= 65535 && k.size(2) <= (1 << 20), "cache dimensions too large");
}
// a tracking tensor beside the cache: [pages, Hkv, page_size], contiguous
void check_track(const at::Tensor &t, const at::Tensor &k, at::ScalarType type, const char *name, const char *type_name) {
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type_name);
  TORCH_CHECK(t.dim() == 3 && t.is_contiguous() && t.size(0) == k.size(0) && t.size(1) == k.size(1) &&
                  t.size(2) == k.size(2),
              name, " must be contiguous [pages, kv heads, page size]");
}
void check_table(const at::Tensor &bt, int64_t rows) {
  TORCH_CHECK(bt.scalar_type() == at::kInt, "block_table must be int32");
  TORCH_CHECK(bt.dim() == 2 && bt.size(0) >= rows && bt.size(1) >= 1 && (bt.stride(1) == 1 || bt.size(1) == 1) &&
                  bt.size(1) <= INT32_MAX,
              "block_table must be [>= requests, pages per request] with contiguous rows");
}
void check_aligned(const at::Tensor &t, const char *name) {
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name, " must start on a 16-byte boundary");
}

void qk_norm_rope_kv_append(const at::Tensor &qkv, const at::Tensor &wq, const at::Tensor &wk, double eps,
                            const at::Tensor &pos, const at::Tensor &slot, const at::Tensor &cos_sin, at::Tensor &q_out,
                            at::Tensor &k_cache, at::Tensor &v_cache, int64_t Hq, int64_t Hkv,
                            const c10::optional<at::Tensor> &scores, const c10::optional<at::Tensor> &positions,
                            const c10::optional<at::Tensor> &status) {
  check_cache(k_cache, v_cache);
  const int64_t D = k_cache.size(3);
  TORCH_CHECK(Hkv == k_cache.size(1), "n_kv_heads must be the cache's");
  TORCH_CHECK(Hq >= 1 && Hq <= 65535, "n_q_heads must be positive");
  check_same(qkv, k_cache, "qkv");
  TORCH_CHECK(qkv.dim() == 2 && qkv.size(1) == (Hq + 2 * Hkv) * D && (qkv.stride(1) == 1 || qkv.size(0) == 0),
              "qkv must be [tokens, (q heads + 2 kv heads) * head dim] with contiguous rows");
  const int64_t T = qkv.size(0);
  TORCH_CHECK(T <= INT32_MAX && T * (Hq + 2 * Hkv) <= INT32_MAX, "too many tokens in one call");
  check_same(wq, k_cache, "q_weight");
  check_same(wk, k_cache, "k_weight");
  TORCH_CHECK(wq.dim() == 1 && wk.dim() == 1 && wq.size(0) == D && wk.size(0) == D && wq.is_contiguous() &&
                  wk.is_contiguous(),
              "q_weight and k_weight must be contiguous [head dim]");
  check_vec(pos, at::kInt, T, "pos", "int32");
  check_vec(slot, at::kInt, T, "slot", "int32");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.dim() == 3 && cos_sin.is_contiguous() &&
                  cos_sin.size(2) == 2 && cos_sin.size(0) >= 1 && cos_sin.size(0) <= INT32_MAX,
              "cos_sin must be contiguous float32 [positions, rotated dims / 2, 2]");
  const int64_t rot = 2 * cos_sin.size(1);
  TORCH_CHECK(rot >= 16 && rot <= D && rot % 16 == 0, "the rotated dims must be a multiple of 16, at most the head dim");
  check_same(q_out, k_cache, "q_out");
  TORCH_CHECK(q_out.dim() == 3 && q_out.size(0) >= T && q_out.size(1) == Hq && q_out.size(2) == D &&
                  q_out.stride(2) == 1 && (q_out.stride(1) == D || Hq == 1),
              "q_out must be [>= tokens, q heads, head dim] with contiguous heads");
  if (scores.has_value()) check_track(*scores, k_cache, at::kFloat, "scores", "float32");
  if (positions.has_value()) check_track(*positions, k_cache, at::kInt, "positions", "int32");
  TORCH_CHECK(T <= 1 || (qkv.stride(0) % 8 == 0 && q_out.stride(0) % 8 == 0 && q_out.stride(0) >= Hq * D),
              "rows of qkv and q_out must not overlap and must start on 16-byte boundaries");
  const std::pair<const at::Tensor *, const char *> on[] = {{&qkv, "qkv"}, {&wq, "q_weight"}, {&wk, "k_weight"},
      {&pos, "pos"}, {&slot, "slot"}, {&cos_sin, "cos_sin"}, {&q_out, "q_out"}, {&v_cache, "v_cache"}};
  check_cuda(k_cache, "k_cache");
  for (const auto &t : on) check_on(*t.first, k_cache, t.second);
  if (scores.has_value()) check_on(*scores, k_cache, "scores");
  if (positions.has_value()) check_on(*positions, k_cache, "positions");
  if (T == 0) return;
  for (const auto &t : on)
    if (t.first != &pos && t.first != &slot) check_aligned(*t.first, t.second);
  check_aligned(k_cache, "k_cache");
  QkNormArgs a{};
  a.qkv = qkv.data_ptr();
  a.ld_qkv = T > 1 ? qkv.stride(0) : 0;
  a.wq = wq.data_ptr();
  a.wk = wk.data_ptr();
  a.eps = (float)eps;
  a.pos = pos.data_ptr<int32_t>();
  a.slot = slot.data_ptr<int32_t>();
  a.cos_sin = cos_sin.data_ptr<float>();
  a.max_pos = cos_sin.size(0);
  a.rot = rot;
  a.q_out = q_out.data_ptr();
  a.ld_q = T > 1 ? q_out.stride(0) : 0;
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.scores = ptr_or_null<float>(scores);
  a.positions = ptr_or_null<int32_t>(positions);
  a.T = T;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.D = D;
  a.page_size = k_cache.size(2);
  a.num_pages = k_cache.size(0);
  a.element = kv_element(k_cache, "k_cache");
  a.num_sms = num_sms(k_cache);
  a.status = ptr_or_null<int>(status);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(k_cache.device());
    rc_ = sched_qk_norm_rope_kv_append(&a, cur_stream());
  }
  check_rc(rc_, "qk_norm_rope_kv_append");
}

// q, out [R, Q, Hq, D] and lse [R, Q, Hq], or without Q for one query; returns
// the number of kernels launched
int64_t attn_decode_scored(const at::Tensor &q, at::Tensor &out, const at::Tensor &k_cache, const at::Tensor &v_cache,
                        const at::Tensor &block_table, const at::Tensor &kv_lens, double sm_scale, at::Tensor &scores,
                        const c10::optional<at::Tensor> &lse, int64_t max_len, const c10::optional<at::Tensor> &status) {
  check_cache(k_cache, v_cache);
  const int64_t D = k_cache.size(3), Hkv = k_cache.size(1), ps = k_cache.size(2);
  TORCH_CHECK(ps % 16 == 0, "the page size must be a multiple of 16");
  check_same(q, k_cache, "q");
  check_same(out, k_cache, "out");
  const int64_t nd = q.dim();
  TORCH_CHECK((nd == 3 || nd == 4) && q.size(-1) == D && q.size(-2) >= 1 && q.size(-2) % Hkv == 0,
              "q must be [requests, (queries,) q heads, head dim] with q heads a multiple of the cache's heads");
  TORCH_CHECK(out.sizes() == q.sizes(), "out must have q's shape");
  const int64_t R = q.size(0), Q = nd == 4 ? q.size(1) : 1, Hq = q.size(-2);
  for (const at::Tensor *t : {&q, (const at::Tensor *)&out})
    TORCH_CHECK(t->numel() == 0 || (t->stride(-1) == 1 && (t->stride(-2) == D || Hq == 1) &&
                                    (Q == 1 || t->stride(1) % 8 == 0) && (R == 1 || t->stride(0) % 8 == 0)),
                "q and out need contiguous heads and rows on 16-byte boundaries");
  TORCH_CHECK(out.numel() == 0 || ((Q == 1 || out.stride(1) >= Hq * D) && (R == 1 || out.stride(0) >= Hq * D) &&
                                   (Q == 1 || R == 1 || out.stride(0) >= Q * out.stride(1) ||
                                    out.stride(1) >= R * out.stride(0))),
              "rows of out must not overlap");
  TORCH_CHECK(R <= 65535 && Q * (Hq / Hkv) <= 8192, "at most 65535 requests and 8192 query rows per KV head");
  check_table(block_table, R);
  check_vec(kv_lens, at::kInt, R, "kv_lens", "int32");
  check_track(scores, k_cache, at::kFloat, "scores", "float32");
  if (lse.has_value()) {
    TORCH_CHECK(lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->dim() == nd - 1 && lse->size(0) == R &&
                    (nd == 3 || lse->size(1) == Q) && lse->size(-1) == Hq,
                "lse must be contiguous float32 of q's shape without the head dim");
  }
  TORCH_CHECK(max_len >= 0, "max_len must not be negative");
  int64_t cap = block_table.size(1) * ps;
  if (max_len > 0 && max_len < cap) cap = max_len;
  TORCH_CHECK(cap < (1 << 30), "contexts of 2^30 tokens or more");
  check_cuda(k_cache, "k_cache");
  const std::pair<const at::Tensor *, const char *> on[] = {{&q, "q"}, {&out, "out"}, {&v_cache, "v_cache"},
      {&block_table, "block_table"}, {&kv_lens, "kv_lens"}, {&scores, "scores"}};
  for (const auto &t : on) check_on(*t.first, k_cache, t.second);
  if (lse.has_value()) check_on(*lse, k_cache, "lse");
  if (R == 0 || Q == 0) return 0;
  check_aligned(q, "q");
  check_aligned(out, "out");
  check_aligned(k_cache, "k_cache");
  check_aligned(v_cache, "v_cache");
  check_aligned(scores, "scores");
  ScoredArgs a{};
  a.q = q.data_ptr();
  a.q_req = R > 1 ? q.stride(0) : 0;
  a.q_query = Q > 1 ? q.stride(1) : 0;
  a.out = out.data_ptr();
  a.out_req = R > 1 ? out.stride(0) : 0;
  a.out_query = Q > 1 ? out.stride(1) : 0;
  a.lse = ptr_or_null<float>(lse);
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.scores = scores.data_ptr<float>();
  a.block_table = block_table.data_ptr<int32_t>();
  a.bt_stride = block_table.stride(0);
  a.bt_pages = block_table.size(1);
  a.kv_lens = kv_lens.data_ptr<int32_t>();
  a.R = R;
  a.Q = Q;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.D = D;
  a.page_size = ps;
  a.num_pages = k_cache.size(0);
  a.max_len = cap;
  a.element = kv_element(k_cache, "k_cache");
  a.num_sms = num_sms(k_cache);
  a.sm_scale = (float)sm_scale;
  a.status = ptr_or_null<int>(status);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(k_cache.device());
    // scratch of this call alone, from the allocator's pool of the current stream (or of the graph being captured)
    const long long floats = sched_attn_scored_ws_floats(a.R, a.Q, a.Hq, a.Hkv, a.D, a.max_len, a.num_sms);
    at::Tensor ws;
    if (floats > 0) ws = at::empty({floats}, scores.options());
    a.ws = floats > 0 ? ws.data_ptr<float>() : nullptr;
    a.ws_floats = floats;
    rc_ = sched_attn_scored(&a, cur_stream());
  }
  check_rc(rc_, "attn_decode_scored");
  return a.ws_floats == 0 ? 1 : 2;
}

// returns new_lens, made here unless given
at::Tensor kv_evict(at::Tensor &k_cache, at::Tensor &v_cache, at::Tensor &scores, at::Tensor &positions,
              const at::Tensor &block_table, const at::Tensor &kv_lens, const at::Tensor &last_pos, int64_t budget,
              int64_t recent, int64_t sink, const c10::optional<at::Tensor> &given, int64_t max_len,
              const c10::optional<at::Tensor> &status) {
  check_cache(k_cache, v_cache);
  const int64_t ps = k_cache.size(2);
  check_track(scores, k_cache, at::kFloat, "scores", "float32");
  check_track(positions, k_cache, at::kInt, "positions", "int32");
  TORCH_CHECK(scores.numel() < 0xffffffffll, "the cache must have fewer than 2^32 - 1 rows");
  TORCH_CHECK(kv_lens.dim() == 1, "kv_lens must be [requests]");
  const int64_t R = kv_lens.size(0);
  check_vec(kv_lens, at::kInt, R, "kv_lens", "int32");
  check_vec(last_pos, at::kInt, R, "last_pos", "int32");
  if (given.has_value()) check_vec(*given, at::kInt, R, "new_lens", "int32");
  check_table(block_table, R);
  TORCH_CHECK(R <= 65535, "at most 65535 requests");
  TORCH_CHECK(budget >= 1 && budget <= INT32_MAX, "budget must be at least 1");
  TORCH_CHECK(recent >= 0 && sink >= 0 && recent <= budget && sink <= budget && recent + sink <= budget,
              "recent and sink must not be negative, and together at most the budget");
  TORCH_CHECK(max_len >= 0, "max_len must not be negative");
  int64_t cap = block_table.size(1) * ps;
  if (max_len > 0 && max_len < cap) cap = max_len;
  TORCH_CHECK(cap < (1 << 30), "contexts of 2^30 tokens or more");
  check_cuda(k_cache, "k_cache");
  const std::pair<const at::Tensor *, const char *> on[] = {{&v_cache, "v_cache"}, {&scores, "scores"},
      {&positions, "positions"}, {&block_table, "block_table"}, {&kv_lens, "kv_lens"}, {&last_pos, "last_pos"}};
  for (const auto &t : on) check_on(*t.first, k_cache, t.second);
  if (given.has_value()) check_on(*given, k_cache, "new_lens");
  at::Tensor new_lens = given.has_value() ? *given : at::empty({R}, kv_lens.options());
  if (R == 0) return new_lens;
  const int32_t *nl = new_lens.data_ptr<int32_t>(), *kl = kv_lens.data_ptr<int32_t>(), *lp = last_pos.data_ptr<int32_t>();
  TORCH_CHECK((nl + R <= kl || kl + R <= nl) && (nl + R <= lp || lp + R <= nl),
              "new_lens must not overlap kv_lens or last_pos: every head reads the old ones");
  check_aligned(k_cache, "k_cache");
  check_aligned(v_cache, "v_cache");
  KvEvictArgs a{};
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.scores = scores.data_ptr<float>();
  a.positions = positions.data_ptr<int32_t>();
  a.block_table = block_table.data_ptr<int32_t>();
  a.bt_stride = block_table.stride(0);
  a.bt_pages = block_table.size(1);
  a.kv_lens = kv_lens.data_ptr<int32_t>();
  a.last_pos = last_pos.data_ptr<int32_t>();
  a.new_lens = new_lens.data_ptr<int32_t>();
  a.R = R;
  a.Hkv = k_cache.size(1);
  a.D = k_cache.size(3);
  a.page_size = ps;
  a.num_pages = k_cache.size(0);
  a.max_len = cap;
  a.budget = budget;
  a.recent = recent;
  a.sink = sink;
  a.num_sms = num_sms(k_cache);
  a.status = ptr_or_null<int>(status);
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(k_cache.device());
    const long long ints = sched_kv_evict_ws_ints(a.R, a.Hkv, a.max_len, a.budget, a.num_sms);
    at::Tensor ws;
    if (ints > 0) ws = at::empty({ints}, kv_lens.options());
    a.ws = ints > 0 ? ws.data_ptr<int32_t>() : nullptr;
    a.ws_ints = ints;
    rc_ = sched_kv_evict(&a, cur_stream());
  }
  check_rc(rc_, "kv_evict");
  return new_lens;
}

void probe_stream(const at::Tensor &src, int64_t policy, at::Tensor &sink, int64_t grid) {
  TORCH_CHECK(src.is_cuda() && src.is_contiguous(), "src on the device");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(src.device());
    rc_ = sched_probe_stream(src.data_ptr(), src.numel() * src.element_size(), policy,
                                reinterpret_cast<unsigned *>(sink.data_ptr()), grid, cur_stream());
  }
  check_rc(rc_, "probe_stream");
}

void probe_tasks(const at::Tensor &cost, int64_t mode, int64_t grid, int64_t memory, const at::Tensor &data,
                 at::Tensor &hits, at::Tensor &per_cta, at::Tensor &ticket, at::Tensor &sink,
                 const c10::optional<at::Tensor> &status) {
  TORCH_CHECK(cost.is_cuda() && cost.scalar_type() == at::kInt, "cost int32 on the device");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(cost.device());
    rc_ = sched_probe_tasks(reinterpret_cast<const uint32_t *>(cost.data_ptr()), cost.numel(), mode, grid, memory,
                               data.data_ptr(), data.numel() * data.element_size(),
                               reinterpret_cast<unsigned *>(hits.data_ptr()),
                               reinterpret_cast<unsigned *>(per_cta.data_ptr()),
                               reinterpret_cast<unsigned *>(ticket.data_ptr()),
                               reinterpret_cast<unsigned *>(sink.data_ptr()), ptr_or_null<int>(status), cur_stream());
  }
  check_rc(rc_, "probe_tasks");
}

// counters: int32 [4n + 1] on the device: hits, claimed, launched, fails
// (n each) and the count of claim answers with a non-zero fourth word.
void probe_clc_shape(const at::Tensor &work, int64_t gx, int64_t gy, int64_t gz, int64_t stride, int64_t cx,
                     at::Tensor &counters, const c10::optional<at::Tensor> &status) {
  TORCH_CHECK(work.is_cuda() && work.scalar_type() == at::kInt && work.is_contiguous(), "work int32 on the device");
  TORCH_CHECK(gx > 0 && gy > 0 && gz > 0 && stride > 0 && cx >= 1 && cx <= 8 && gx % cx == 0,
              "grid dims > 0, stride > 0, cluster 1..8 dividing gx");
  const int64_t n = gx * gy * gz;
  TORCH_CHECK(work.numel() >= n, "work: one entry per CTA");
  TORCH_CHECK(counters.is_cuda() && counters.element_size() == 4 && counters.is_contiguous() &&
                  counters.numel() >= 4 * n + 1,
              "counters: int32 [4 n + 1]");
  unsigned *c = reinterpret_cast<unsigned *>(counters.data_ptr());
  int rc_ = 0;
  {  // the guard is gone before the launch code is recorded
    c10::cuda::CUDAGuard gd(work.device());
    rc_ = sched_probe_clc_shape(reinterpret_cast<const uint32_t *>(work.data_ptr()), (int)gx, (int)gy, (int)gz,
                                (int)stride, (int)cx, c, c + n, c + 2 * n, c + 3 * n, c + 4 * n,
                                ptr_or_null<int>(status), cur_stream());
  }
  check_rc(rc_, "probe_clc_shape");
}

void probe_clc(const at::Tensor &work, int64_t mode, int64_t grid, at::Tensor &hits, at::Tensor &rec,
               at::Tensor &n_rec, at::Tensor &smid, const c10::optional<at::Tensor> &status) {
  TORCH_CHECK(work.is_cuda() && work.scalar_type() == at::kInt && work.is_contiguous(), "work int32 on the device");
  TORCH_CHECK(mode >= 0 && mode <= 2, "mode is 0 (static), 1 (CLC late bound) or 2 (CLC claim-ahead)");
  const int64_t n = work.numel();
  const int64_t g = mode == 0 ? grid : n;
  TORCH_CHECK(g > 0, "grid must be positive");
  TORCH_CHECK(hits.numel() >= n && hits.element_size() == 4, "hits: int32 [n_tasks]");
  TORCH_CHECK(rec.dim() == 2 && rec.size(0) >= g && rec.element_size() == 8 && rec.is_contiguous(),
              "rec: int64 [grid, max_rec]");
  TORCH_CHECK(n_rec.numel() >= g && smid.numel() >= g && n_rec.element_size() == 4 && smid.element_size() == 4,
              "n_rec, smid: int32 [grid]");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard gd(work.device());
    rc_ = sched_probe_clc(reinterpret_cast<const uint32_t *>(work.data_ptr()), (int)n, (int)mode, (int)g,
                             (int)rec.size(1), reinterpret_cast<unsigned *>(hits.data_ptr()),
                             reinterpret_cast<unsigned long long *>(rec.data_ptr()),
                             reinterpret_cast<unsigned *>(n_rec.data_ptr()), reinterpret_cast<unsigned *>(smid.data_ptr()),
                             ptr_or_null<int>(status), cur_stream());
  }
  check_rc(rc_, "probe_clc");
}

void probe_mix(const at::Tensor &R, const at::Tensor &S, int64_t mode, double frac, at::Tensor &sink,
               int64_t grid) {
  TORCH_CHECK(R.is_cuda() && S.is_cuda() && R.is_contiguous() && S.is_contiguous(), "R, S on the device");
  TORCH_CHECK(mode >= 0 && mode <= 2, "mode is 0 (plain), 1 or 2 (pinned fractions)");
  TORCH_CHECK(frac > 0.0 && frac <= 1.0, "the pinned fraction must be in (0, 1]");
  TORCH_CHECK(grid > 0 && sink.numel() >= grid, "sink holds one word per CTA");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(R.device());
    rc_ = sched_probe_mix(R.data_ptr(), R.numel() * R.element_size(), S.data_ptr(), S.numel() * S.element_size(),
                             mode, (float)frac, reinterpret_cast<unsigned *>(sink.data_ptr()), grid, cur_stream());
  }
  check_rc(rc_, "probe_mix");
}

void probe_pdl_pairs(at::Tensor &buf, at::Tensor &out, const at::Tensor &table, int64_t work, int64_t prologue,
                     bool pdl, int64_t pairs) {
  TORCH_CHECK(buf.is_cuda() && buf.scalar_type() == at::kFloat && out.sizes() == buf.sizes() &&
                  out.scalar_type() == at::kFloat && table.numel() >= 256 && table.scalar_type() == at::kFloat,
              "float32 buf/out of one shape and a float32 table of >= 256 entries");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(buf.device());
    rc_ = sched_probe_pdl_pairs(buf.data_ptr<float>(), out.data_ptr<float>(), buf.numel(), table.data_ptr<float>(),
                                   work, prologue, pdl ? 1 : 0, pairs, cur_stream());
  }
  check_rc(rc_, "probe_pdl_pairs");
}

void probe_pdl_produce(at::Tensor &buf, int64_t work) {
  TORCH_CHECK(buf.is_cuda() && buf.scalar_type() == at::kFloat && buf.is_contiguous(), "float32 buf");
  int rc_ = 0;
  {  // the guard is gone before check_rc may throw
    c10::cuda::CUDAGuard g(buf.device());
    rc_ = sched_probe_pdl_produce(buf.data_ptr<float>(), buf.numel(), work, cur_stream());
  }
  check_rc(rc_, "probe_pdl_produce");
}

// Page moves between KV pools (device <-> pinned host); pairs [n, 2] int32 on the device.
// With n_dev (int32 [1] on the device) n_pairs is a capacity and the count is read there.
void kv_page_copy(const at::Tensor &src_k, const at::Tensor &src_v, at::Tensor &dst_k, at::Tensor &dst_v,
                  const at::Tensor &pairs, int64_t n_pairs, const c10::optional<at::Tensor> &n_dev,
                  const c10::optional<at::Tensor> &status) {
  TORCH_CHECK(src_k.dim() == 5 && dst_k.dim() == 5, "pools are [layers, pages, heads, 16, 128]");
  TORCH_CHECK(src_k.size(0) == dst_k.size(0) && src_k.size(2) == dst_k.size(2), "pool shapes differ");
  TORCH_CHECK(src_k.is_contiguous() && src_v.is_contiguous() && dst_k.is_contiguous() && dst_v.is_contiguous(),
              "contiguous pools");
  TORCH_CHECK(pairs.is_cuda() && pairs.scalar_type() == at::kInt && pairs.is_contiguous(), "pairs int32 on device");
  check_rc(sched_kv_page_copy(src_k.data_ptr(), src_v.data_ptr(), src_k.size(1), dst_k.data_ptr(), dst_v.data_ptr(),
                              dst_k.size(1), pairs.data_ptr<int32_t>(), n_pairs, ptr_or_null<int>(n_dev),
                              src_k.size(0), src_k.size(2), ptr_or_null<int>(status), cur_stream()),
           "kv_page_copy");
}

// Page moves between a bf16 pool and an fp8 (uint8 storage) pool; the scales
// [layers, fp8 pool pages, heads] fp32 belong to the fp8 pool.
void kv_page_copy_fp8(const at::Tensor &src_k, const at::Tensor &src_v, at::Tensor &dst_k, at::Tensor &dst_v,
                      at::Tensor &scale_k, at::Tensor &scale_v, bool to_fp8, const at::Tensor &pairs,
                      int64_t n_pairs, const c10::optional<at::Tensor> &n_dev,
                      const c10::optional<at::Tensor> &status) {
  TORCH_CHECK(src_k.dim() == 5 && dst_k.dim() == 5, "pools are [layers, pages, heads, 16, 128]");
  TORCH_CHECK(src_k.size(0) == dst_k.size(0) && src_k.size(2) == dst_k.size(2), "pool shapes differ");
  TORCH_CHECK(src_k.size(3) == 16 && src_k.size(4) == 128 && dst_k.size(3) == 16 && dst_k.size(4) == 128,
              "pages of 16 tokens x head dim 128");
  TORCH_CHECK(src_k.is_contiguous() && src_v.is_contiguous() && dst_k.is_contiguous() && dst_v.is_contiguous() &&
                  scale_k.is_contiguous() && scale_v.is_contiguous(),
              "contiguous pools");
  const at::Tensor &q = to_fp8 ? dst_k : src_k;
  const at::Tensor &b = to_fp8 ? src_k : dst_k;
  TORCH_CHECK(q.element_size() == 1 && b.scalar_type() == at::kBFloat16, "an fp8 (1-byte) pool and a bf16 pool");
  TORCH_CHECK(scale_k.scalar_type() == at::kFloat && scale_k.numel() == q.size(0) * q.size(1) * q.size(2) &&
                  scale_v.numel() == scale_k.numel(),
              "scales [layers, fp8 pages, heads] float32");
  TORCH_CHECK(pairs.is_cuda() && pairs.scalar_type() == at::kInt && pairs.is_contiguous(), "pairs int32 on device");
  check_rc(sched_kv_page_copy_fp8(src_k.data_ptr(), src_v.data_ptr(), src_k.size(1), dst_k.data_ptr(),
                                  dst_v.data_ptr(), dst_k.size(1), scale_k.data_ptr<float>(),
                                  scale_v.data_ptr<float>(), to_fp8 ? 1 : 0, pairs.data_ptr<int32_t>(), n_pairs,
                                  ptr_or_null<int>(n_dev), src_k.size(0), src_k.size(2), ptr_or_null<int>(status),
                                  cur_stream()),
           "kv_page_copy_fp8");
}

}  // namespace

void register_symm(py::module &m);

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  register_symm(m);
  m.def("take_error", &take_error);
  m.def("status_words", &status_words);
  m.def("gemm_allreduce", &gemm_allreduce);
  m.def("gemm_reduce_scatter", &gemm_reduce_scatter);
  m.def("sp_reduce_norm", &sp_reduce_norm);
  m.def("sp_wait_rows", &sp_wait_rows);
  m.doc() = "sched_pass_b200 sm_100a kernels";
  m.def("gemm", &gemm);
  m.def("gemm_qkv_rope", &gemm_qkv_rope);
  m.def("gemm_ws_floats", &gemm_ws_floats);
  m.def("attn_decode", &attn_decode);
  m.def("attn_merge", &attn_merge);
  m.def("qk_norm_rope_kv_append", &qk_norm_rope_kv_append);
  m.def("attn_decode_scored", &attn_decode_scored);
  m.def("kv_evict", &kv_evict);
  m.def("attn_prefill", &attn_prefill);
  m.def("attn_prefill_tile_rows", &sched_attn_prefill_tile_rows);
  m.def("attn_decode_occupancy", &attn_decode_occupancy);
  m.def("attn_decode_smem_bytes", &attn_decode_smem_bytes);
  m.def("add_rmsnorm", &add_rmsnorm);
  m.def("rope_kv_append", &rope_kv_append);
  m.def("embedding", &embedding);
  m.def("argmax", &argmax);
  m.def("argmax_exchange", &argmax_exchange);
  m.def("set_gemm_trace", &set_gemm_trace);
  m.def("set_attn_trace", &set_attn_trace);
  m.def("gemm_plan", [](int64_t T, int64_t N, int64_t K, int64_t epi, int64_t sms) {
    int cs = 0, grid = 0;
    sched_gemm_plan(T, N, K, epi, sms, &cs, &grid);
    return std::make_tuple(cs, grid);
  });
  m.def("gemm_pair_plan", [](int64_t T, int64_t N, int64_t K, int64_t epi, int64_t ws_floats, int64_t counters) {
    int np = 0, whole = 0, splits = 1;
    sched_gemm_pair_plan(T, N, K, epi, ws_floats, counters, &np, &whole, &splits);
    return std::make_tuple(np, whole, splits);
  });
  m.def("moe_router", &moe_router);
  m.def("kv_page_copy", &kv_page_copy);
  m.def("probe_stream", &probe_stream);
  m.def("probe_tasks", &probe_tasks);
  m.def("probe_tasks_occupancy", &sched_probe_tasks_occupancy);
  m.def("probe_mix", &probe_mix);
  m.def("probe_clc", &probe_clc);
  m.def("probe_clc_shape", &probe_clc_shape);
  m.def("probe_clc_shape_capacity", &sched_probe_clc_shape_capacity);
  m.def("kv_page_copy_fp8", &kv_page_copy_fp8);
  m.def("probe_pdl_pairs", &probe_pdl_pairs);
  m.def("probe_pdl_produce", &probe_pdl_produce);
  m.def("moe_dispatch", &moe_dispatch);
  m.def("moe_expert_gemm", &moe_expert_gemm);
  m.def("moe_quantize", &moe_quantize);
  m.def("moe_combine_norm", &moe_combine_norm);
}
