// kv_budget.cu -- the kernels that keep a paged KV cache to a token budget:
//
//   * per-head RMSNorm of queries and keys, the position rotation and the
//     append to the paged cache in one pass (and the start of a new slot's
//     tracking: weight 0, its position);
//   * decode attention that also adds, to every cached token, the attention
//     weight it got from this step's queries;
//   * eviction: each (request, KV head) keeps its newest tokens, its first
//     ones and those of the largest accumulated weight.
//
// The tracking state lies beside the cache: scores and positions are
// [pages, Hkv, page_size], one entry per K row of the cache.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "kv_budget_api.h"
#include "sched/ptx.cuh"

namespace kvb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  return pack_bf16x2(a, b);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t *>(&h);
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &u, float (&f)[8]) {
  const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y), c = unpack2<T>(u.z), d = unpack2<T>(u.w);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = c.x, f[5] = c.y, f[6] = d.x, f[7] = d.y;
}
// Two fp32 values in one register pair: sm_100 multiplies and adds them at once.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 parts(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack_f2(const uint4 &u, F2 (&f)[4]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = unpack2<T>(w[j]);
    f[j] = f2(x.x, x.y);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack_f2(const F2 (&f)[4]) {
  const float2 a = parts(f[0]), b = parts(f[1]), c = parts(f[2]), d = parts(f[3]);
  return make_uint4(pack2<T>(a.x, a.y), pack2<T>(b.x, b.y), pack2<T>(c.x, c.y), pack2<T>(d.x, d.y));
}

// ------------------------------------------------------------------ norm + rotation + append
// y = x / sqrt(mean(x^2) + eps) * w over a head's D values, then the first
// rot values turn in pairs (d, d + rot/2). All in fp32, rounded once.
//
// D/16 lanes share a head: each holds the two 8-value chunks whose values
// pair up (chunks l and l + rot/16; lanes behind the rotated part hold the
// unrotated chunks 2l and 2l + 1), so the rotation needs no exchange and
// every access is a 16-byte vector. A lane group takes NH heads of one kind of
// a token, all requested at once; weight times cos and sin are theirs in
// common. PIPE: the grid is resident at once and strides over the groups, and
// each lane copies its own chunks of the group after next to shared memory
// meanwhile (cp.async: it takes no registers, and nobody else reads them, so
// there is no barrier). Otherwise every lane group takes one group.
constexpr int kNormThreads = 128;
constexpr int kNormStages = 2;
constexpr int kNormResident = 5;  // CTAs per SM

__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(ptx::smem_u32(dst)), "l"(src) : "memory");
}

template <typename T, int D, int NH, bool PIPE>
__global__ void __launch_bounds__(kNormThreads, PIPE ? kNormResident : 6) qk_norm_kernel(const QkNormArgs a) {
  constexpr int LANES = D / 16, ST = PIPE ? kNormStages : 1, BUF = PIPE ? kNormThreads : 1;
  __shared__ uint4 buf[ST][2 * NH][BUF];
  __shared__ int32_t where[ST][2][BUF];  // position, slot
  const int tid = threadIdx.x, l = tid % LANES, nr = a.rot / 16;
  const int c0 = (l < nr ? l : 2 * l) * 8, c1 = (l < nr ? l + nr : 2 * l + 1) * 8;
  const uint32_t gq = (a.Hq + NH - 1) / NH, gk = (a.Hkv + NH - 1) / NH, ng = gq + 2 * gk;
  const uint32_t groups = (uint32_t)a.T * ng, stride = gridDim.x * (kNormThreads / LANES);
  struct Group {
    uint32_t t;
    int kind, h0, heads;  // 0 q, 1 k, 2 v; first head of its kind; number of heads
    const T *src;
  };
  auto group_of = [&](uint32_t i) {
    Group g;
    g.t = i / ng;
    uint32_t r = i - g.t * ng;
    g.kind = r < gq ? 0 : r < gq + gk ? 1 : 2;
    r -= g.kind == 0 ? 0 : g.kind == 1 ? gq : gq + gk;
    g.h0 = (int)r * NH;
    g.heads = min(NH, (g.kind == 0 ? a.Hq : a.Hkv) - g.h0);
    g.src = static_cast<const T *>(a.qkv) + (size_t)g.t * a.ld_qkv +
            (size_t)(g.h0 + (g.kind == 0 ? 0 : g.kind == 1 ? a.Hq : a.Hq + a.Hkv)) * D;
    return g;
  };
  auto request = [&](uint32_t i, int stage) {
    if (i < groups) {
      const Group g = group_of(i);
      cp_async4(&where[stage][0][tid], a.pos + g.t);
      cp_async4(&where[stage][1][tid], a.slot + g.t);
#pragma unroll
      for (int k = 0; k < NH; ++k) {
        if (k < g.heads) {
          cp_async16(&buf[stage][2 * k][tid], g.src + k * D + c0);
          cp_async16(&buf[stage][2 * k + 1][tid], g.src + k * D + c1);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  uint32_t idx = (blockIdx.x * (uint32_t)kNormThreads + tid) / LANES;
  if constexpr (PIPE) {
#pragma unroll
    for (int st = 0; st < ST; ++st) request(idx + st * stride, st);
  }
  for (int stage = 0; idx < groups; idx += stride, stage = stage + 1 == ST ? 0 : stage + 1) {  // whole lane groups
    const Group g = group_of(idx);
    uint4 u0[NH], u1[NH];
    int p, s;
    if constexpr (PIPE) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
      p = where[stage][0][tid];
      s = where[stage][1][tid];
#pragma unroll
      for (int i = 0; i < NH; ++i) u0[i] = buf[stage][2 * i][tid], u1[i] = buf[stage][2 * i + 1][tid];
      request(idx + ST * stride, stage);
    } else {
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        if (i < g.heads) {
          u0[i] = *reinterpret_cast<const uint4 *>(g.src + i * D + c0);
          u1[i] = *reinterpret_cast<const uint4 *>(g.src + i * D + c1);
        }
      }
      p = a.pos[g.t];
      s = a.slot[g.t];
    }
    const bool pos_ok = (uint32_t)p < (uint32_t)a.max_pos;
    const bool slot_ok = s < 0 || (long long)s < (long long)a.num_pages * a.page_size;
    if (g.kind == 0 && g.h0 == 0 && l == 0) {
      if (!pos_ok)
        report_bad_index(a.status, kSiteNormPos, p);
      else if (!slot_ok)
        report_bad_index(a.status, kSiteKvSlot, s);
    }
    if (!slot_ok || !pos_ok) s = -1;  // no cache write
    if (g.kind < 2) {
      F2 w0[4], w1[4];
      const T *w = static_cast<const T *>(g.kind == 0 ? a.wq : a.wk);
      unpack_f2<T>(*reinterpret_cast<const uint4 *>(w + c0), w0);
      unpack_f2<T>(*reinterpret_cast<const uint4 *>(w + c1), w1);
      // y0 = x0 (w0 cos) - x1 (w1 sin), y1 = x1 (w1 cos) + x0 (w0 sin)
      F2 s0[4], s1[4];
      const bool turns = l < nr;
      if (turns) {
        const float4 *cs = reinterpret_cast<const float4 *>(a.cos_sin + ((size_t)(pos_ok ? p : 0) * (a.rot / 2) + l * 8) * 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 v = cs[j];  // (cos, sin) of two pairs
          const F2 c = f2(v.x, v.z), sn = f2(v.y, v.w), ns = f2(-v.y, -v.w);
          s0[j] = w1[j] * ns;
          s1[j] = w0[j] * sn;
          w0[j] = w0[j] * c;
          w1[j] = w1[j] * c;
        }
      }
      // the lanes of a head are aligned neighbours with the same number of heads
      const unsigned mask = ((1u << LANES) - 1u) << (ptx::lane_id() / LANES * LANES);
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        if (i >= g.heads) break;
        F2 x0[4], x1[4], q = f2(0.f, 0.f);
        unpack_f2<T>(u0[i], x0);
        unpack_f2<T>(u1[i], x1);
#pragma unroll
        for (int j = 0; j < 4; ++j) q = fma2(x1[j], x1[j], fma2(x0[j], x0[j], q));
        float ss = parts(q).x + parts(q).y;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float inv = rsqrtf(ss * (1.f / D) + a.eps);
        const F2 iv = f2(inv, inv);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x0[j] = x0[j] * iv;
          x1[j] = x1[j] * iv;
          const F2 y0 = x0[j] * w0[j], y1 = x1[j] * w1[j];
          if (turns) {
            const F2 z0 = fma2(x1[j], s0[j], y0);
            x1[j] = fma2(x0[j], s1[j], y1);
            x0[j] = z0;
          } else {
            x0[j] = y0;
            x1[j] = y1;
          }
        }
        u0[i] = pack_f2<T>(x0);
        u1[i] = pack_f2<T>(x1);
      }
    }
    T *dst;
    size_t pitch = D;
    if (g.kind == 0) {
      dst = static_cast<T *>(a.q_out) + (size_t)g.t * a.ld_q + (size_t)g.h0 * D;
      if (!pos_ok) {
#pragma unroll
        for (int i = 0; i < NH; ++i) u0[i] = u1[i] = make_uint4(0, 0, 0, 0);
      }
    } else {
      if (s < 0) continue;
      const int page = s / a.page_size;
      const size_t row = ((size_t)page * a.Hkv + g.h0) * a.page_size + (s - page * a.page_size);
      pitch = (size_t)a.page_size * D;
      dst = static_cast<T *>(g.kind == 1 ? a.k_cache : a.v_cache) + row * D;
      if (g.kind == 1) {
        for (int i = l; i < g.heads; i += LANES) {
          if (a.scores != nullptr) a.scores[row + (size_t)i * a.page_size] = 0.f;
          if (a.positions != nullptr) a.positions[row + (size_t)i * a.page_size] = p;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NH; ++i) {
      if (i < g.heads) {
        *reinterpret_cast<uint4 *>(dst + i * pitch + c0) = u0[i];
        *reinterpret_cast<uint4 *>(dst + i * pitch + c1) = u1[i];
      }
    }
  }
}

// Heads per lane group, by the lanes that one head each would take per SM.
// Measured with 32 + 8 heads of 128, bf16, cold tensors: 256 tokens (664 lanes)
// 3.4 us with one head, 3.6 with two, 4.5 with four in the pipeline; 1024
// tokens 8.6, 6.6, 7.3; 4097 tokens 31, 25.6, 22.7; 8000 tokens 64, 47, 37
// (5.4 TB/s; copying as many bytes takes 18 us for 4097 tokens, 33 for 8000).
// The pipeline takes about 5.7 us to start and drain and 3.95 us for each stride of
// the resident lane groups over 987 tokens (6.3 TB/s): 17.3 us for three
// strides, 21.7 for four, 25.6 for five; 4097 tokens are 4.15.
template <typename T, int D>
int run_qk_norm(const QkNormArgs &a, cudaStream_t st) {
  const long long lanes = (long long)a.T * (a.Hq + 2 * a.Hkv) * (D / 16);
  const int nh = lanes <= 768ll * a.num_sms ? 1 : lanes <= 4096ll * a.num_sms ? 2 : 4;
  const long long groups = (long long)a.T * ((a.Hq + nh - 1) / nh + 2ll * ((a.Hkv + nh - 1) / nh));
  const long long need = (groups * (D / 16) + kNormThreads - 1) / kNormThreads, most = (long long)a.num_sms * kNormResident;
  if (groups + (kNormStages + 1) * most * kNormThreads > 0xffffffffll) return -1;  // groups are numbered in 32 bits
  const long long grid = nh < 4 || need < most ? need : most;
  launch_pdl(nh == 1   ? qk_norm_kernel<T, D, 1, false>
             : nh == 2 ? qk_norm_kernel<T, D, 2, false>
                       : qk_norm_kernel<T, D, 4, true>,
             dim3((unsigned)grid), dim3(kNormThreads), 0, st, a);
  return cudaPeekAtLastError() == cudaSuccess ? 0 : -4;
}

// ------------------------------------------------------------------ scored decode attention
// For each request, KV head h and query row i (Q queries x the G heads that
// share h): s_ij = sm_scale q_i . k_j for the tokens j a query may see,
// lse_i = log sum_j exp s_ij, out_i = sum_j exp(s_ij - lse_i) v_j, and
// scores_j += sum_i exp(s_ij - lse_i). The weights need the finished lse, so
// the s_ij are kept (fp32, in units of log 2): 4 Q G bytes a token and KV head
// beside the 4 D bytes of K and V that the pass has to read.
//
// Work is cut evenly over warps, not over requests: the 16-token tiles of all
// (request, KV head, row block) tasks form one list, and every warp takes an
// equal run of it, whatever the lengths. A run's part of a task leaves a
// partial result (max, sum, output) in the workspace; a second kernel joins
// them and adds the weights. Runs and tasks advance together through the
// list, so (warp + task) numbers the partial results without gaps to look up.
constexpr int kWarps = 4;      // per CTA of the split kernel
constexpr int kTile = 16;      // tokens per warp step: divides the page size
// CTAs of the split kernel per SM, by its registers. Measured: 64 requests of
// 1664 tokens, 8 heads of 128, 4 query rows each 78 us with three, 90 with two,
// 121 with four (spills); 16 rows 115 with two, 126 with three. 4 heads of 64,
// 64 x 4000 tokens: 4 rows 61 us with four, 69 with three; 16 rows 85 and 89.
// (168 registers with three CTAs: 8 rows of 128 spill 16 to 24 bytes.)
constexpr int resident(int D, int block) { return D == 64 ? 4 : block == 16 ? 2 : 3; }
constexpr int kMinRun = 2;     // tiles per warp at least: bounds the partial results

struct ScoredPlan {
  int rows, lp;         // query rows per KV head, padded length
  int block, blocks;    // rows per task (8 or 16), tasks per (request, KV head)
  int grid;             // CTAs of the split kernel
  int join, o_rows;     // tokens per weight CTA and rows per output CTA of the join (0: no CTAs for outputs alone)
  // workspace: logits [R, Hkv, rows, lp], partial outputs and (max, sum) [parts, block],
  // and for the join: tiles per warp, then (length, tiles in front) of each request
  long long s_off, o_off, ml_off, meta_off, total;
};

inline ScoredPlan scored_plan(int R, int Q, int Hq, int Hkv, int D, int max_len, int num_sms) {
  ScoredPlan p;
  p.rows = Q * (Hq / Hkv);
  p.lp = (max_len + kTile - 1) / kTile * kTile;
  p.block = p.rows <= 8 ? 8 : 16;
  p.blocks = (p.rows + p.block - 1) / p.block;
  const long long heads = (long long)R * Hkv, tasks = heads * p.blocks;
  const long long most = (tasks * (p.lp / kTile) + kMinRun * kWarps - 1) / (kMinRun * kWarps);
  const long long fill = (long long)num_sms * resident(D, p.block);
  p.grid = (int)(most < fill ? most : fill);
  // The join's CTAs all resident at once where that is possible, with each thread having a logit to read. Sized by
  // max_len: of very uneven batches the long requests' weights are few CTAs' work (one request of 32768 tokens among
  // 63 of 100, 8 heads of 128, 4 rows: 86 us, against 38 alone).
  p.join = p.rows >= 16 ? 64 : p.rows >= 8 ? 128 : p.rows >= 4 ? 256 : p.rows >= 2 ? 512 : 1024;
  while (heads * ((max_len + p.join - 1) / p.join) > 4ll * num_sms && p.join < max_len) p.join += p.join < 1024 ? p.join : 1024;
  // and at most 16 partial results per warp, by the average of the tasks (a long request's rows have more)
  p.o_rows = 1;
  while (p.o_rows < 32 && heads * ((p.rows + p.o_rows - 1) / p.o_rows) > (p.o_rows < 8 ? 1 : 4) * num_sms &&
         p.grid * kWarps / tasks * p.o_rows * 2 <= 8 * 16)
    p.o_rows *= 2;
  // up to eight rows and many heads: a warp of the first weight CTA has a row each
  if (p.rows <= 8 && heads > num_sms) p.o_rows = 0;
  p.s_off = 0;
  p.o_off = heads * p.rows * p.lp;
  const long long parts = (long long)p.grid * kWarps + tasks;
  p.ml_off = p.o_off + parts * p.block * D;
  p.meta_off = p.ml_off + parts * p.block * 2;
  p.total = p.meta_off + 1 + 2ll * R;
  return p;
}

template <typename T>
__device__ __forceinline__ void mma16816(float &d0, float &d1, float &d2, float &d3, uint32_t a0, uint32_t a1,
                                         uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float &d0, float &d1, float &d2, float &d3, uint32_t a0,
                                                        uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d0), "+f"(d1), "+f"(d2), "+f"(d3)
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float &d0, float &d1, float &d2, float &d3, uint32_t a0, uint32_t a1,
                                                 uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d0), "+f"(d1), "+f"(d2), "+f"(d3)
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Read once: not kept in L1, and the first to leave L2 (which the logits should
// not). Not the read-only path: the kernel in front may still write the cache
// when this one starts (programmatic dependent launch).
__device__ __forceinline__ uint4 ld_stream(const void *p, uint64_t policy) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.u32 {%0,%1,%2,%3}, [%4], %5;"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p), "l"(policy));
  return v;
}

// A request's length within what the call may address.
__device__ __forceinline__ int checked_len(int n, int cap, int *status, int site, bool tell) {
  if (n > cap) {
    if (tell) report_bad_index(status, site, n);
    n = cap;
  }
  return n < 0 ? 0 : n;
}
__device__ __forceinline__ int table_cap(int max_len, int pages, int page_size) {
  return (int)min((long long)max_len, (long long)pages * page_size);
}

// exp2(m - ref) with m = -inf or an empty row's ref = -inf giving 0
__device__ __forceinline__ float scale_to(float m, float ref) { return ref == -INFINITY ? 0.f : ex2_approx(m - ref); }

// Tiles per warp of the split kernel, for the list's total.
__device__ __forceinline__ uint32_t run_length(uint32_t total, uint32_t warps) {
  const uint32_t per = (total + warps - 1) / warps;
  return per < kMinRun ? kMinRun : per;
}

__device__ __forceinline__ uint4 keep_if(bool k, const uint4 &v) { return k ? v : make_uint4(0, 0, 0, 0); }

// First element of a tile's K (and V) rows, or a negative number for a bad page.
__device__ __forceinline__ long long page_base(const ScoredArgs &a, int page, int h, int tok) {
  if (page < 0 || page >= a.num_pages) {
    if (threadIdx.x % 32 == 0) report_bad_index(a.status, kSiteScoredPage, page);
    return -1;
  }
  return (((long long)page * a.Hkv + h) * a.page_size + tok % a.page_size) * a.D;
}
__device__ __forceinline__ long long tile_base(const ScoredArgs &a, int req, int h, int tok) {
  return page_base(a, a.block_table[(size_t)req * a.bt_stride + tok / a.page_size], h, tok);
}

// A warp's running softmax over 16-token tiles. K and V go from global memory
// straight into the registers of the m16n8k16 operands (K of the next tile is
// requested once this one's logits are done, V once its product is), so a warp
// always has loads in flight and there is no shared-memory staging; Q waits in
// shared memory in operand order. Query rows are the M side (8 of its 16 rows
// where a KV head has at most 8 query rows), tokens the N side of the logits
// and the K side of the output.
//
// Operand layout, for lane 4 r + c: the 16 bytes of K at value 32 kk + 8 c of
// tokens r and r + 8 are the k-slots of two products, Q's registers hold the
// same values; the 16 bytes of V at value 64 i + 8 r of tokens 2c, 2c + 1,
// 2c + 8 and 2c + 9 are column r of the eight products (i, e), column n of
// which is value 64 i + 8 n + e.
template <typename T, int D, int ROWS>
struct RowSoftmax {
  static constexpr int NK = D / 32, RB = ROWS / 8;
  // The weights, at most 1, enter the product with V in the cache's type: fp16
  // keeps its 11 bits only from 2^-14 on, and a context of many tokens behind
  // one heavy one (whose value may be small) is made of lighter ones. So fp16
  // weights are raised to at most 2^15, and hold all bits down to 2^-29 of the
  // largest; o has the same factor until finish(). bf16 has fp32's range.
  static constexpr float kRaise = std::is_same<T, __half>::value ? 32768.f : 1.f;
  typedef uint4 QTile[RB][NK][32];  // each lane reads back only what it wrote
  int lane, r, c;
  uint4 kx[2][NK], vx[D / 64][4];
  float o[D / 8][ROWS / 4];  // product (i, e) = o[8 i + e]: row r's columns 2c, 2c + 1, then row r + 8's
  float m[RB], sum[RB];      // of rows r, r + 8; sum: this lane's tokens only, until finish()
  int lim[RB], all_see;      // tokens that rows r, r + 8 see; tokens that every row of the task sees
  int rows_here;             // rows of the task
  uint64_t policy;

  __device__ __forceinline__ RowSoftmax() : lane(threadIdx.x % 32), r(lane / 4), c(lane % 4), policy(ptx::policy_evict_first()) {}

  __device__ __forceinline__ void enter(const ScoredArgs &a, int rows, int req, int h, int row0, int n, QTile &q_sm) {
    const int G = a.Hq / a.Hkv;
    rows_here = min(ROWS, rows - row0);
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int row = row0 + r + 8 * i;
      lim[i] = 0;
      const T *src = nullptr;
      if (row < rows) {
        const int qi = row / G, g = row - qi * G;
        lim[i] = n - (a.Q - 1 - qi);
        src = static_cast<const T *>(a.q) + (size_t)req * a.q_req + (size_t)qi * a.q_query + (size_t)(h * G + g) * D + c * 8;
      }
#pragma unroll
      for (int kk = 0; kk < NK; ++kk)
        q_sm[i][kk][lane] = src != nullptr ? *reinterpret_cast<const uint4 *>(src + kk * 32) : make_uint4(0, 0, 0, 0);
    }
    all_see = n - (a.Q - 1 - row0 / G);
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int j = 0; j < ROWS / 4; ++j) o[i][j] = 0.f;
#pragma unroll
    for (int i = 0; i < RB; ++i) m[i] = -INFINITY, sum[i] = 0.f;
  }
  __device__ __forceinline__ void load_k(const ScoredArgs &a, long long base) {
    const T *p = static_cast<const T *>(a.k_cache) + (base < 0 ? 0 : base) + r * D + c * 8;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) kx[j][kk] = ld_stream(p + j * 8 * D + kk * 32, policy);
  }
  __device__ __forceinline__ void load_v(const ScoredArgs &a, long long base) {
    const T *p = static_cast<const T *>(a.v_cache) + (base < 0 ? 0 : base) + 2 * c * D + r * 8;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) vx[i][j] = ld_stream(p + ((j & 1) + (j / 2) * 8) * D + i * 64, policy);
  }

  // One tile, whose K and V are loaded or on their way: its logits go to
  // s_out (row 0, the tile's first token; `pitch` between rows). With `more`,
  // the tile at `next` is requested on the way.
  __device__ __forceinline__ void step(const ScoredArgs &a, long long base, int tok, int n, float scale2, const QTile &q_sm,
                                       float *s_out, int pitch, bool more, long long next) {
    float s[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const uint4 q0 = q_sm[0][kk][lane];
      const uint4 q1 = ROWS == 16 ? q_sm[RB - 1][kk][lane] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mma16816<T>(s[j][0], s[j][1], s[j][2], s[j][3], q0.x, q1.x, q0.y, q1.y, kx[j][kk].x, kx[j][kk].y);
        mma16816<T>(s[j][0], s[j][1], s[j][2], s[j][3], q0.z, q1.z, q0.w, q1.w, kx[j][kk].z, kx[j][kk].w);
      }
    }
    if (more) load_k(a, next);
    // tokens from `end` on are not there (behind the request's end, or their page is bad)
    const int end = base < 0 ? tok : n;
    const bool whole = tok + kTile <= min(end, all_see);
    uint32_t pa[2][2] = {{0u, 0u}, {0u, 0u}};  // [row block][tile half]: P as the product's A operand
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      float v[4] = {s[0][2 * i] * scale2, s[0][2 * i + 1] * scale2, s[1][2 * i] * scale2, s[1][2 * i + 1] * scale2};
      if (!whole) {
        const int seen = min(end, lim[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (tok + (j / 2) * 8 + 2 * c + (j & 1) >= seen) v[j] = -INFINITY;
      }
      if (r + 8 * i < rows_here) {
        float *dst = s_out + (size_t)(r + 8 * i) * pitch + 2 * c;
        *reinterpret_cast<float2 *>(dst) = make_float2(v[0], v[1]);
        *reinterpret_cast<float2 *>(dst + 8) = make_float2(v[2], v[3]);
      }
      float top = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(top, m[i]);
      const float ref = top == -INFINITY ? 0.f : top;
      const float f = ex2_approx(m[i] - ref);
      m[i] = top;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = ex2_approx(v[j] - ref);
      sum[i] = sum[i] * f + ((v[0] + v[1]) + (v[2] + v[3]));
      if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
        for (int d = 0; d < D / 8; ++d) o[d][2 * i] *= f, o[d][2 * i + 1] *= f;
      }
      // the weights enter the product in the cache's type (at most half a
      // step of it each, and the sum above is of the unrounded ones)
      pa[i][0] = pack2<T>(v[0] * kRaise, v[1] * kRaise);
      pa[i][1] = pack2<T>(v[2] * kRaise, v[3] * kRaise);
    }
    if (tok + kTile > end) {  // 0 * NaN: values behind the end must not reach the product
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) vx[i][j] = keep_if(tok + (j / 2) * 8 + 2 * c + (j & 1) < end, vx[i][j]);
    }
    bool apart = false;
    if (a.Q > 1 && tok + kTile > all_see) {
      // tokens that only the later queries see: an infinity or a NaN among
      // them must not meet the zero weight of a query that does not
      bool odd = false;
#pragma unroll
      for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float f[8];
          unpack8<T>(vx[i][j], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) odd |= !(fabsf(f[e]) <= 3.4e38f);
        }
      apart = __any_sync(0xffffffffu, odd);
    }
    if (!apart) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          auto word = [&](int j) { return e / 2 == 0 ? vx[i][j].x : e / 2 == 1 ? vx[i][j].y : e / 2 == 2 ? vx[i][j].z : vx[i][j].w; };
          const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
          const uint32_t b0 = __byte_perm(word(0), word(1), sel), b1 = __byte_perm(word(2), word(3), sel);
          float(&acc)[ROWS / 4] = o[i * 8 + e];
          if constexpr (ROWS == 16) {
            mma16816<T>(acc[0], acc[1], acc[2], acc[3], pa[0][0], pa[1][0], pa[0][1], pa[1][1], b0, b1);
          } else {
            float z0 = 0.f, z1 = 0.f;  // rows 8-15 of the product: unused
            mma16816<T>(acc[0], acc[1], z0, z1, pa[0][0], 0u, pa[0][1], 0u, b0, b1);
          }
        }
      }
    } else {  // token by token, each row only with what it sees
      for (int t = 0; t < kTile && tok + t < end; ++t) {
        const T *src = static_cast<const T *>(a.v_cache) + base + t * D + 16 * c;
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          const uint32_t two = __shfl_sync(0xffffffffu, t < 8 ? pa[i][0] : pa[i][1], r * 4 + (t & 7) / 2);
          const float2 pp = unpack2<T>(two);
          const float w = (t & 1) ? pp.y : pp.x;
          if (tok + t < lim[i]) {
#pragma unroll
            for (int d = 0; d < D / 64; ++d) {
              float lo[8], hi[8];
              unpack8<T>(*reinterpret_cast<const uint4 *>(src + d * 64), lo);
              unpack8<T>(*reinterpret_cast<const uint4 *>(src + d * 64 + 8), hi);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                o[d * 8 + e][2 * i] += w * lo[e];
                o[d * 8 + e][2 * i + 1] += w * hi[e];
              }
            }
          }
        }
      }
    }
    if (more) load_v(a, next);
  }

  // The partial result of the tiles since enter(): [rows][D] sums to o_out,
  // (max, sum) to ml_out.
  __device__ __forceinline__ void finish(float *o_out, float2 *ml_out) {
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      const int row = r + 8 * i;
      if (row < rows_here) {
        float *dst = o_out + row * D + 16 * c;
#pragma unroll
        for (int d = 0; d < D / 64; ++d)
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const int x = d * 8 + e % 8, y = 2 * i + e / 8;
            constexpr float lower = 1.f / kRaise;
            *reinterpret_cast<float4 *>(dst + d * 64 + e) =
                make_float4(o[x][y] * lower, o[x + 1][y] * lower, o[x + 2][y] * lower, o[x + 3][y] * lower);
          }
        if (c == 0) ml_out[row] = make_float2(m[i], sum[i]);
      }
    }
  }
  // The same where these were all of the task's tiles: its outputs and lse.
  __device__ __forceinline__ void finish_task(const ScoredArgs &a, int req, int h, int row0, float2 *ml_out) {
    const int G = a.Hq / a.Hkv;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      const int row = r + 8 * i;
      if (row < rows_here) {
        const bool none = m[i] == -INFINITY && sum[i] == 0.f;  // a row that sees nothing
        const float f = none ? 0.f : 1.f / kRaise / sum[i];
        const int qi = (row0 + row) / G, g = row0 + row - qi * G;
        T *dst = static_cast<T *>(a.out) + (size_t)req * a.out_req + (size_t)qi * a.out_query + (size_t)(h * G + g) * D + 16 * c;
#pragma unroll
        for (int d = 0; d < D / 64; ++d)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = o[d * 8 + x][2 * i + e] * f;
            *reinterpret_cast<uint4 *>(dst + d * 64 + 8 * e) =
                make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
          }
        if (c == 0) {
          ml_out[row] = make_float2(m[i], sum[i]);
          if (a.lse != nullptr)
            a.lse[((size_t)req * a.Q + qi) * a.Hq + h * G + g] = none ? -INFINITY : (m[i] + log2f(sum[i])) * kLn2;
        }
      }
    }
  }
};

// One warp: a run of the tile list. Memory bound: 64 requests of 1536 to 1664
// tokens (8 heads of 128, 4 query rows each) take 71 us, 92 % of the copy
// rate, 8 of up to 32768 (8 rows) 150 us, 93 %. With 16 rows the registers
// leave 8 warps an SM, whose one tile ahead does not cover the loads' latency:
// the same 64 requests 95 us at 25 % of the issue slots, 14 % of the tensor
// pipe and 3.5 warps waiting for loads per issue.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kWarps * 32, resident(D, ROWS))
    scored_split_kernel(const ScoredArgs a, const ScoredPlan pl) {
  __shared__ typename RowSoftmax<T, D, ROWS>::QTile q_sm[kWarps];
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  RowSoftmax<T, D, ROWS> x;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int cap = table_cap(a.max_len, a.bt_pages, a.page_size);
  const int HB = a.Hkv * pl.blocks;
  const uint32_t w_id = blockIdx.x * kWarps + warp;
  auto tiles_of = [&](int n) { return (n + kTile - 1) / kTile; };

  // this warp's run of the list (its length fits 31 bits)
  uint32_t total = 0;
  for (int i = lane; i < a.R; i += 32) total += tiles_of(checked_len(a.kv_lens[i], cap, a.status, kSiteScoredLen, w_id == 0));
  total = __reduce_add_sync(0xffffffffu, total) * HB;
  const uint32_t per = run_length(total, gridDim.x * kWarps);
  if (w_id == 0) {  // for the join
    uint32_t *meta = reinterpret_cast<uint32_t *>(a.ws + pl.meta_off);
    uint32_t before = 0;
    for (int i0 = 0; i0 < a.R; i0 += 32) {
      const int len = i0 + lane < a.R ? checked_len(a.kv_lens[i0 + lane], cap, nullptr, 0, false) : 0;
      const uint32_t own = tiles_of(len);
      uint32_t inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (i0 + lane < a.R) meta[1 + 2 * (i0 + lane)] = len, meta[2 + 2 * (i0 + lane)] = before + inc - own;
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) meta[0] = per;
  }
  if ((unsigned long long)w_id * per >= total) return;
  const uint32_t u0 = w_id * per;
  uint32_t left = min(per, total - u0);
  int req = 0, hb = 0, tile = 0;
  {
    uint32_t before = 0;  // tiles (of one head) in front of request i0
    for (int i0 = 0;; i0 += 32) {
      if (i0 >= a.R) return;  // only if kv_lens changes under the kernel
      const uint32_t own = i0 + lane < a.R ? tiles_of(checked_len(a.kv_lens[i0 + lane], cap, nullptr, 0, false)) : 0;
      uint32_t inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, (before + inc) * HB > u0);
      if (past != 0u) {
        const int at = __ffs(past) - 1;
        const uint32_t off = u0 - (before + __shfl_sync(0xffffffffu, inc - own, at)) * HB;
        const uint32_t nt = __shfl_sync(0xffffffffu, own, at);
        req = i0 + at;
        hb = (int)(off / nt);
        tile = (int)(off - (uint32_t)hb * nt);
        break;
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  int n = checked_len(a.kv_lens[req], cap, nullptr, 0, false);
  const float scale2 = a.sm_scale * kLog2e;
  long long base = tile_base(a, req, hb / pl.blocks, tile * kTile);
  x.load_k(a, base);
  x.load_v(a, base);
  while (true) {  // a task
    const int h = hb / pl.blocks, row0 = (hb - h * pl.blocks) * ROWS, nt = tiles_of(n);
    x.enter(a, pl.rows, req, h, row0, n, q_sm[warp]);
    float *s_out = a.ws + pl.s_off + (((size_t)req * a.Hkv + h) * pl.rows + row0) * pl.lp;
    const bool from_start = tile == 0;
    bool to_end;
    int n_req = req, n_hb = hb, n_n = n;
    while (true) {  // a tile
      --left;
      to_end = tile + 1 == nt;
      const bool ends = to_end || left == 0;
      int n_tile = tile + 1;
      long long next = -1;
      if (left > 0) {
        if (ends) {
          n_tile = 0;
          if (++n_hb == HB) {
            n_hb = 0;
            do {  // more tiles follow, so a request with some does
              if (++n_req >= a.R) return;  // only if kv_lens changes under the kernel
              n_n = checked_len(a.kv_lens[n_req], cap, nullptr, 0, false);
            } while (n_n == 0);
          }
        }
        next = tile_base(a, n_req, n_hb / pl.blocks, n_tile * kTile);
      }
      x.step(a, base, tile * kTile, n, scale2, q_sm[warp], s_out + tile * kTile, pl.lp, left > 0, next);
      tile = n_tile;
      base = next;
      if (ends) break;
    }
    const size_t part = (size_t)w_id + (uint32_t)req * HB + hb;
    float2 *ml_out = reinterpret_cast<float2 *>(a.ws + pl.ml_off) + part * ROWS;
    // whole tasks end here with 16 rows (windows of short contexts have many;
    // with 8 rows there are few, and the code costs the loop registers)
    if (ROWS == 16 && from_start && to_end)
      x.finish_task(a, req, h, row0, ml_out);
    else
      x.finish(a.ws + pl.o_off + part * ROWS * D, ml_out);
    if (left == 0) return;
    req = n_req, hb = n_hb, n = n_n;
  }
}

__device__ __forceinline__ void red_add4(float *p, const float4 &v) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
// Adds the weights of tokens tok .. tok + 3 (those below `end`) to their scores.
__device__ __forceinline__ void add_weights(const ScoredArgs &a, int req, int h, int tok, int end, const float4 &w) {
  const int col = tok / a.page_size, page = a.block_table[(size_t)req * a.bt_stride + col];
  if (page < 0 || page >= a.num_pages) return;  // reported where K was read
  float *dst = a.scores + ((size_t)page * a.Hkv + h) * a.page_size + (tok - col * a.page_size);
  if (tok + 4 <= end) {
    red_add4(dst, w);
  } else {
    atomicAdd(dst, w.x);
    if (tok + 1 < end) atomicAdd(dst + 1, w.y);
    if (tok + 2 < end) atomicAdd(dst + 2, w.z);
  }
}
__device__ __forceinline__ void add_weight(float4 &w, const float4 &s, float lse2) {
  w.x += ex2_approx(s.x - lse2);
  w.y += ex2_approx(s.y - lse2);
  w.z += ex2_approx(s.z - lse2);
  w.w += ex2_approx(s.w - lse2);
}

// The same in one kernel, where latency counts: a cluster of C CTAs has a
// (request, KV head), its warps the tiles in turn (so that a warp's first page
// does not depend on the length). The logits stay in shared memory; the CTAs
// exchange (max, sum) and outputs through it, and each then adds its own
// tokens' weights. Eight CTAs of eight warps for few heads, four, two or one of
// four warps for more. Latency bound: a chain of the loads of
// length and page, K and V, the products, two exchanges and the additions (one
// request of 700 tokens: 6.4 us).
constexpr int kCTiles = 8;  // tiles of a warp at most
// CTAs per SM by the registers (a third of four warps with heads of 128 costs more than it gives)
constexpr int one_resident(int D, int warps) { return (D == 64 ? 2 : 1) * (warps == 8 ? 1 : 2); }

template <typename T, int D, int ROWS, int C, int CW>
__global__ void __launch_bounds__(CW * 32, one_resident(D, CW)) scored_cluster_kernel(const ScoredArgs a, int rows, int span) {
  constexpr int NT = CW * 32;
  extern __shared__ __align__(16) float sm[];
  __shared__ typename RowSoftmax<T, D, ROWS>::QTile q_sm[CW];
  __shared__ float2 ml_w[CW][ROWS], ml_c[ROWS];
  __shared__ float lse2[ROWS];                // +inf for a row that sees nothing
  float *o_w = sm;                            // [CW][ROWS][D]; the first [ROWS][D] then hold the CTA's
  float *s_sm = sm + CW * ROWS * D;      // [rows][span]
  const int rank = C > 1 ? (int)ptx::cluster_ctarank() : 0;
  const int req = blockIdx.z, h = blockIdx.y, tid = threadIdx.x, warp = tid / 32;
  const int G = a.Hq / a.Hkv;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int cap = table_cap(a.max_len, a.bt_pages, a.page_size);
  int tile = rank + C * warp;
  const int page0 = tile * kTile < cap ? a.block_table[(size_t)req * a.bt_stride + tile * kTile / a.page_size] : -1;
  const int n = checked_len(a.kv_lens[req], cap, a.status, kSiteScoredLen, h == 0 && rank == 0 && tid == 0);
  const int nt = (n + kTile - 1) / kTile;
  RowSoftmax<T, D, ROWS> x;
  long long base = -1;
  if (tile < nt) {
    base = page_base(a, page0, h, tile * kTile);
    x.load_k(a, base);
    x.load_v(a, base);
  }
  x.enter(a, rows, req, h, 0, n, q_sm[warp]);
  const float scale2 = a.sm_scale * kLog2e;
  for (int at = warp * kTile; tile < nt; at += CW * kTile) {
    const int n_tile = tile + C * CW;
    const long long next = n_tile < nt ? tile_base(a, req, h, n_tile * kTile) : -1;
    x.step(a, base, tile * kTile, n, scale2, q_sm[warp], s_sm + at, span, n_tile < nt, next);
    tile = n_tile;
    base = next;
  }
  x.finish(o_w + warp * ROWS * D, ml_w[warp]);
  __syncthreads();
  // this CTA's sums, in warp order, relative to its own maximum
  for (int i = tid; i < rows * D; i += NT) {
    const int row = i / D;
    float top = -INFINITY, tot = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < CW; ++w) top = fmaxf(top, ml_w[w][row].x);
#pragma unroll
    for (int w = 0; w < CW; ++w) {
      const float f = scale_to(ml_w[w][row].x, top);
      tot += ml_w[w][row].y * f;
      v += o_w[w * ROWS * D + i] * f;
    }
    o_w[i] = v;
    if (i % D == 0) ml_c[row] = make_float2(top, tot);
  }
  if constexpr (C > 1)
    ptx::cluster_sync_all();
  else
    __syncthreads();
  const uint32_t ml_addr = ptx::smem_u32(ml_c), o_addr = ptx::smem_u32(o_w);
  auto peer2 = [&](uint32_t addr, int cta) {
    float2 v;
    if constexpr (C > 1)
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(ptx::mapa_shared(addr, cta)) : "memory");
    else
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
  };
  {  // C lanes to a row: a CTA's (max, sum) each
    const int row = tid / C, at = min(row, rows - 1);
    const float2 mine = peer2(ml_addr + at * 8, tid % C);
    float top = mine.x;
#pragma unroll
    for (int o = C / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float tot = mine.y * scale_to(mine.x, top);
#pragma unroll
    for (int o = C / 2; o > 0; o >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, o);
    const float v = top == -INFINITY && tot == 0.f ? -INFINITY : top + log2f(tot);  // NaN logits stay NaN
    if (row < rows && tid % C == 0) {
      lse2[row] = v == -INFINITY ? INFINITY : v;
      if (rank == 0 && a.lse != nullptr) {
        const int qi = row / G;
        a.lse[((size_t)req * a.Q + qi) * a.Hq + h * G + (row - qi * G)] = v * kLn2;
      }
    }
  }
  __syncthreads();
  // outputs: two values a thread, spread over the cluster
  for (int i = (rank * NT + tid) * 2; i < rows * D; i += C * NT * 2) {
    const int row = i / D, qi = row / G;
    const float ref = lse2[row];
    float2 m[C], p[C], v = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < C; ++k) m[k] = peer2(ml_addr + row * 8, k), p[k] = peer2(o_addr + i * 4, k);
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const float f = ex2_approx(m[k].x - ref);
      if (f != 0.f) v.x += p[k].x * f, v.y += p[k].y * f;
    }
    *reinterpret_cast<uint32_t *>(static_cast<T *>(a.out) + (size_t)req * a.out_req + (size_t)qi * a.out_query +
                                  (size_t)(h * G + row - qi * G) * D + i % D) = pack2<T>(v.x, v.y);
  }
  for (int q = tid; q < span / 4; q += NT) {  // four tokens of a tile that this CTA had
    const int at = q * 4 / kTile, tok = ((at / CW * CW + at % CW) * C + rank) * kTile + q * 4 % kTile;
    if (tok >= n) continue;
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int row = 0; row < rows; ++row) add_weight(w, *reinterpret_cast<const float4 *>(s_sm + row * span + q * 4), lse2[row]);
    add_weights(a, req, h, tok, n, w);
  }
  if constexpr (C > 1) ptx::cluster_sync_all();  // the peers have read this CTA's shared memory
}

// Join. Of a (request, KV head)'s CTAs the first ones join the outputs
// (pl.o_rows rows each, the warps shared evenly by them), the others add the
// weights of pl.join tokens each: a thread has four tokens and every
// groups-th row, whose logits it requests before the rows' lse is known. All
// sums have a fixed order, and one request's pages get one addition per token
// and head from a call.
constexpr int kJoin = 256;
constexpr int kJoinWarps = kJoin / 32;

// Partial results of a task: first index and count.
struct Parts {
  uint32_t first, count;
};
__device__ __forceinline__ Parts parts_of(uint32_t before, uint32_t per, int nt, int HB, int req, int hb) {
  const uint32_t u0 = before * HB + (uint32_t)hb * nt, w0 = u0 / per;
  return {w0 + (uint32_t)req * HB + hb, nt == 0 ? 0u : (u0 + nt - 1) / per - w0 + 1};
}
// log2 of a row's sum over its partial results (NaN where a logit is), by the
// LANES aligned lanes that share the row
template <int LANES>
__device__ __forceinline__ float row_lse2(const float2 *ml, uint32_t count, int pitch) {
  const int lane = threadIdx.x % LANES;
  float top = -INFINITY, tot = 0.f;
#pragma unroll 4
  for (uint32_t k = lane; k < count; k += LANES) {
    const float2 v = ml[(size_t)k * pitch];
    const float t = fmaxf(top, v.x);
    tot = tot * scale_to(top, t) + v.y * scale_to(v.x, t);
    top = t;
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    const float ot = __shfl_xor_sync(0xffffffffu, top, o), os = __shfl_xor_sync(0xffffffffu, tot, o);
    const float t = fmaxf(top, ot);
    tot = tot * scale_to(top, t) + os * scale_to(ot, t);
    top = t;
  }
  return top == -INFINITY && tot == 0.f ? -INFINITY : top + log2f(tot);
}

// This warp's share (every `sub`-th from `part`) of a row's joined output, D / 32 values a lane.
template <int D>
__device__ __forceinline__ void join_row(const ScoredArgs &a, const ScoredPlan &pl, const Parts &pt, int row, float lse2,
                                         int part, int sub, float (&v)[D / 32]) {
  constexpr int V = D / 32;
  const size_t at = (size_t)pt.first * pl.block + row % pl.block;
  const float2 *mr = reinterpret_cast<const float2 *>(a.ws + pl.ml_off) + at;
  const float ref = lse2 == -INFINITY ? INFINITY : lse2;
  const float *src = a.ws + pl.o_off + at * D + threadIdx.x % 32 * V;
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = 0.f;
#pragma unroll 4
  for (uint32_t k = part; k < pt.count; k += sub) {
    const float f = ex2_approx(mr[(size_t)k * pl.block].x - ref);
    float p[V];
    if constexpr (V == 4)
      *reinterpret_cast<float4 *>(p) = *reinterpret_cast<const float4 *>(src + (size_t)k * pl.block * D);
    else
      *reinterpret_cast<float2 *>(p) = *reinterpret_cast<const float2 *>(src + (size_t)k * pl.block * D);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] += f != 0.f ? p[e] * f : 0.f;
  }
}
template <typename T, int D>
__device__ __forceinline__ void put_row(const ScoredArgs &a, int req, int h, int row, const float (&v)[D / 32]) {
  const int G = a.Hq / a.Hkv, qi = row / G;
  T *dst = static_cast<T *>(a.out) + (size_t)req * a.out_req + (size_t)qi * a.out_query + (size_t)(h * G + row - qi * G) * D +
           threadIdx.x % 32 * (D / 32);
  if constexpr (D == 128)
    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  else
    *reinterpret_cast<uint32_t *>(dst) = pack2<T>(v[0], v[1]);
}
__device__ __forceinline__ void put_row_lse(const ScoredArgs &a, int req, int h, int row, float lse2) {
  const int G = a.Hq / a.Hkv, qi = row / G;
  if (a.lse != nullptr) a.lse[((size_t)req * a.Q + qi) * a.Hq + h * G + (row - qi * G)] = lse2 * kLn2;
}

template <typename T, int D>
__global__ void __launch_bounds__(kJoin, 4) scored_join_kernel(const ScoredArgs a, const ScoredPlan pl, int o_ctas) {
  extern __shared__ __align__(16) float sm[];
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int req = blockIdx.z, h = blockIdx.y;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t *meta = reinterpret_cast<const uint32_t *>(a.ws + pl.meta_off);
  const int n = (int)meta[1 + 2 * req];
  const uint32_t before = meta[2 + 2 * req], per = meta[0];
  const int HB = a.Hkv * pl.blocks, nt = (n + kTile - 1) / kTile;
  const float2 *ml = reinterpret_cast<const float2 *>(a.ws + pl.ml_off);

  if ((int)blockIdx.x < o_ctas) {
    constexpr int V = D / 32;  // values per lane
    // up to eight rows: 8 / o_rows warps to a row; more: a warp has every eighth
    const int sub = max(1, kJoinWarps / pl.o_rows), part = warp % sub;
    const int last = min(pl.rows, (int)(blockIdx.x + 1) * pl.o_rows);
    for (int row = blockIdx.x * pl.o_rows + warp / sub; row - warp / sub < last; row += kJoinWarps) {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = 0.f;
      bool done = row >= last;
      if (!done) {
        const Parts pt = parts_of(before, per, nt, HB, req, h * pl.blocks + row / pl.block);
        done = pl.block == 16 && pt.count == 1;  // the warp that had all of the task has written it
        if (!done) {
          const float lse2 = row_lse2<32>(ml + (size_t)pt.first * pl.block + row % pl.block, pt.count, pl.block);
          join_row<D>(a, pl, pt, row, lse2, part, sub, v);
          if (part == 0 && lane == 0) put_row_lse(a, req, h, row, lse2);
        }
      }
      if (sub > 1) {  // (one step: o_rows < 8)
#pragma unroll
        for (int e = 0; e < V; ++e) sm[warp * D + lane * V + e] = v[e];
        __syncthreads();
        for (int w = 1; w < sub && part == 0; ++w)
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] += sm[(warp + w) * D + lane * V + e];
      }
      if (!done && part == 0) put_row<T, D>(a, req, h, row, v);
    }
    return;
  }

  const int t0 = ((int)blockIdx.x - o_ctas) * pl.join, t1 = min(n, t0 + pl.join);
  const bool both = o_ctas == 0 && t0 == 0;  // outputs too
  if (t0 >= n && !both) return;
  constexpr int PRE = 4;
  const int quads = min(pl.join / 4, kJoin), groups = kJoin / quads, grp = tid / quads, quad = tid % quads;
  const float *s_in = a.ws + pl.s_off + ((size_t)req * a.Hkv + h) * pl.rows * pl.lp;
  float4 pre[PRE];
  auto prefetch = [&](int tok) {
    if (tok < t1) {
#pragma unroll
      for (int j = 0; j < PRE; ++j)
        if (grp + j * groups < pl.rows)
          pre[j] = *reinterpret_cast<const float4 *>(s_in + (size_t)(grp + j * groups) * pl.lp + tok);
    }
  };
  prefetch(t0 + quad * 4);
  float4 *part_w = reinterpret_cast<float4 *>(sm);  // [kJoin]
  float *lse2 = sm + 4 * kJoin;                     // [rows]: +inf for a row that sees nothing
  auto put_lse = [&](int row, float v) { lse2[row] = v == -INFINITY ? INFINITY : v; };
  if (pl.rows <= kJoinWarps) {
    if (warp < pl.rows) {
      const Parts pt = parts_of(before, per, nt, HB, req, h);
      const float lse = row_lse2<32>(ml + (size_t)pt.first * pl.block + warp, pt.count, pl.block);
      if (lane == 0) put_lse(warp, lse);
      if (both) {
        float v[D / 32];
        join_row<D>(a, pl, pt, warp, lse, 0, 1, v);
        put_row<T, D>(a, req, h, warp, v);
        if (lane == 0) put_row_lse(a, req, h, warp, lse);
      }
    }
  } else {
    constexpr int LR = 8;  // lanes per row
    for (int row = tid / LR; row - tid / LR < pl.rows; row += kJoin / LR) {
      const int at = min(row, pl.rows - 1);
      const Parts pt = parts_of(before, per, nt, HB, req, h * pl.blocks + at / pl.block);
      const float v = row_lse2<LR>(ml + (size_t)pt.first * pl.block + at % pl.block, pt.count, pl.block);
      if (row < pl.rows && tid % LR == 0) put_lse(row, v);
    }
  }
  __syncthreads();
  for (int tq = t0; tq < t1; tq += quads * 4) {
    const int tok = tq + quad * 4;
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
    if (tok < t1) {
#pragma unroll
      for (int j = 0; j < PRE; ++j)
        if (grp + j * groups < pl.rows) add_weight(w, pre[j], lse2[grp + j * groups]);
#pragma unroll 4
      for (int row = grp + PRE * groups; row < pl.rows; row += groups)
        add_weight(w, *reinterpret_cast<const float4 *>(s_in + (size_t)row * pl.lp + tok), lse2[row]);
    }
    prefetch(tok + quads * 4);
    if (groups > 1) {
      part_w[tid] = w;
      __syncthreads();
      if (grp == 0)
        for (int k = 1; k < groups; ++k) {
          const float4 p = part_w[k * quads + quad];
          w.x += p.x, w.y += p.y, w.z += p.z, w.w += p.w;
        }
      __syncthreads();
    }
    if (grp == 0 && tok < t1) add_weights(a, req, h, tok, t1, w);
  }
}

// ------------------------------------------------------------------ eviction
// Of the n > budget cached tokens of a (request, KV head), the `budget` with
// the largest (key, lowest slot) stay: the key orders the protected tokens
// (position > last - recent, or < sink) above every weight, weights by value,
// NaN and -inf lowest. Kept tokens in slots >= budget then take the slots
// < budget of evicted ones, the i-th the i-th: sources and destinations are
// disjoint, so the moves need no order and only they touch K and V.
constexpr int kBins = 2048;          // of a selection digit: 11, 11 and 10 bits
constexpr int kFew = 256;            // keys that are ranked by comparing all pairs, a thread each
constexpr int kWindow = 1024;        // moves a CTA lists at a time
constexpr int kKeySmem = 40 * 1024;  // slots whose keys fit shared memory; longer contexts keep them in the workspace
constexpr uint32_t kNoRow = 0xffffffffu;

// `after`: the position behind which tokens are recent
__device__ __forceinline__ uint32_t evict_key(float score, int pos, int after, int sink) {
  const uint32_t u = __float_as_uint((score == score ? score : -INFINITY) + 0.f);  // -0 counts as 0
  const uint32_t k = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
  return pos > after || pos < sink ? 0xffffffffu : k;
}

__device__ __forceinline__ uint32_t warp_scan(uint32_t v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += u;
  }
  return v;
}

// Words a CTA needs for n slots: for every block of 128 a key each and four
// flag words (bit l of word e: slot 4 l + e); multiples of 16 bytes.
__host__ __device__ __forceinline__ size_t evict_words(int n) { return (size_t)((n + 127) / 128) * (128 + 4); }

// A cluster has a (request, KV head). Every CTA of it finds the budget-th
// largest key by radix selection over all the keys (8 bytes a token to read;
// doing it once more per CTA costs less than exchanging histograms), and once
// all of them have read the scores, each moves its share of the tokens.
//
// The last key kept and, among its equals, the last slot kept decide each
// slot. A flag marks the slots below the budget that lose their token and the
// slots behind it that keep theirs; as many of the one as of the other, so one
// prefix sum over the flags ranks both.
//
// Measured: 64 requests of 2112 slots to 2048, 8 heads of 128: 19 us, of which
// reading scores and positions would take 3. Its 512 CTAs are one wave and in
// the same phase at once; warps wait for loads (3.0 per issue) and at barriers
// (2.3), with 49 % of the issue slots used. 16 of 8192 to 2048: 52 us, 14 of
// selection and then 206 MB of moves in 38, 83 % of the copy rate: 128 CTAs of
// 1024 threads, one to an SM, leave 20 SMs without one.
template <int D, bool IN_WS>
__global__ void __launch_bounds__(1024) evict_kernel(const KvEvictArgs a, uint32_t *ws, int vec, int page_shift) {
  extern __shared__ __align__(16) uint32_t dyn[];  // evict_words(max_len) unless they are in the workspace (IN_WS)
  __shared__ __align__(16) uint32_t hist[kBins];
  __shared__ uint32_t tot[32], s_bin, s_above, s_count, s_found, s_key;
  __shared__ int s_slot;
  __shared__ __align__(16) uint32_t from[kWindow], to[kWindow];  // slots, then cache rows, of the moves; keys and slots before
  const int tid = threadIdx.x, NT = blockDim.x, NW = NT / 32, warp = tid / 32, lane = tid % 32;
  const int rank = (int)ptx::cluster_ctarank(), C = (int)ptx::cluster_nctarank();
  const int req = blockIdx.z, h = blockIdx.y;
  for (int i = tid; i < kBins; i += NT) hist[i] = 0;
  if (tid == 0) s_found = 0;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int cap = table_cap(a.max_len, a.bt_pages, a.page_size);
  const int n = checked_len(a.kv_lens[req], cap, a.status, kSiteEvictLen, h == 0 && rank == 0 && tid == 0);
  const int b = a.budget;
  if (h == 0 && rank == 0 && tid == 0) a.new_lens[req] = min(n, b);
  if (n <= b) return;  // the whole cluster
  const int32_t *bt = a.block_table + (size_t)req * a.bt_stride;
  const int after = (int)max((long long)a.last_pos[req] - a.recent, -0x80000000ll);
  uint32_t *keys;
  if constexpr (IN_WS)
    keys = ws + (((size_t)req * a.Hkv + h) * C + rank) * evict_words(a.max_len);
  else
    keys = dyn;
  const int nb = (n + 127) / 128;
  uint32_t *flags = keys + (size_t)nb * 128;
  // the row of a slot in the cache and in scores / positions, kNoRow for a bad page
  auto row_of = [&](int j) {
    const int col = page_shift >= 0 ? j >> page_shift : j / a.page_size, page = bt[col];
    return page < 0 || page >= a.num_pages ? kNoRow : ((uint32_t)page * a.Hkv + h) * a.page_size + (j - col * a.page_size);
  };
  auto tell_bad = [&](int j) { report_bad_index(a.status, kSiteEvictPage, bt[j / a.page_size]); };
  __syncthreads();
  // the keys, and the histogram of their first digit. A page outside the
  // cache is reported; its tokens have the lowest key.
  if (vec) {  // four slots of one page at a time, UL such groups of a thread in flight
    constexpr int UL = 3;
    for (int j0 = tid * 4; j0 < n; j0 += NT * 4 * UL) {
      uint32_t row[UL];
      float4 s[UL];
      int4 p[UL];
#pragma unroll
      for (int u = 0; u < UL; ++u) row[u] = j0 + u * NT * 4 < n ? row_of(j0 + u * NT * 4) : kNoRow;
#pragma unroll
      for (int u = 0; u < UL; ++u) {
        const uint32_t at = row[u] == kNoRow ? 0u : row[u];
        s[u] = *reinterpret_cast<const float4 *>(a.scores + at);
        p[u] = *reinterpret_cast<const int4 *>(a.positions + at);
      }
#pragma unroll
      for (int u = 0; u < UL; ++u) {
        const int j = j0 + u * NT * 4;
        if (j >= n) break;
        uint4 k = make_uint4(evict_key(s[u].x, p[u].x, after, a.sink), evict_key(s[u].y, p[u].y, after, a.sink),
                             evict_key(s[u].z, p[u].z, after, a.sink), evict_key(s[u].w, p[u].w, after, a.sink));
        if (row[u] == kNoRow) {
          k = make_uint4(0, 0, 0, 0);
          tell_bad(j);
        }
        *reinterpret_cast<uint4 *>(keys + j) = k;
        atomicAdd(&hist[k.x >> 21], 1u);
        if (j + 1 < n) atomicAdd(&hist[k.y >> 21], 1u);
        if (j + 2 < n) atomicAdd(&hist[k.z >> 21], 1u);
        if (j + 3 < n) atomicAdd(&hist[k.w >> 21], 1u);
      }
    }
  } else {
    for (int j = tid; j < n; j += NT) {
      const uint32_t row = row_of(j);
      uint32_t k = 0u;
      if (row == kNoRow)
        tell_bad(j);
      else
        k = evict_key(a.scores[row], a.positions[row], after, a.sink);
      keys[j] = k;
      atomicAdd(&hist[k >> 21], 1u);
    }
  }

  uint32_t prefix = 0, mask = 0;
  uint32_t need = (uint32_t)b;          // keys still to keep among those that match the prefix
  int last_slot = 0x7fffffff;           // of the keys that match in the end, those up to this slot stay
#pragma unroll 1
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : (digit == 1 ? 10 : 0);
    const uint32_t top = digit == 2 ? 1023u : 2047u;
    if (digit > 0) {
      for (int j = tid * 4; j < n; j += NT * 4) {
        const uint4 k = *reinterpret_cast<const uint4 *>(keys + j);
        if ((k.x & mask) == prefix) atomicAdd(&hist[(k.x >> shift) & top], 1u);
        if ((k.y & mask) == prefix && j + 1 < n) atomicAdd(&hist[(k.y >> shift) & top], 1u);
        if ((k.z & mask) == prefix && j + 2 < n) atomicAdd(&hist[(k.z >> shift) & top], 1u);
        if ((k.w & mask) == prefix && j + 3 < n) atomicAdd(&hist[(k.w >> shift) & top], 1u);
      }
    }
    __syncthreads();
    // bins from the top, 2048 / NT of them a thread, cleared on the way for the next digit
    uint32_t own[8], sum = 0;
    const int per = kBins / NT;  // 8, 4 or 2
    const int hi = kBins - 1 - tid * per;
    if (per == 8) {
      uint4 *q = reinterpret_cast<uint4 *>(hist + hi - 7);
      const uint4 lo4 = q[0], hi4 = q[1];
      q[0] = q[1] = make_uint4(0, 0, 0, 0);
      own[0] = hi4.w, own[1] = hi4.z, own[2] = hi4.y, own[3] = hi4.x;
      own[4] = lo4.w, own[5] = lo4.z, own[6] = lo4.y, own[7] = lo4.x;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) own[i] = i < per ? hist[hi - i] : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < per) hist[hi - i] = 0u;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += own[i];
    const uint32_t inc = warp_scan(sum);
    if (lane == 31) tot[warp] = inc;
    __syncthreads();
    const uint32_t front = warp_scan(lane < NW ? tot[lane] : 0u);
    uint32_t above = inc - sum + (warp > 0 ? __shfl_sync(0xffffffffu, front, warp - 1) : 0u);
    if (above < need && above + sum >= need) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (above < need && above + own[i] >= need) {
          s_bin = (uint32_t)(hi - i);
          s_above = above;
          s_count = own[i];
        }
        above += own[i];
      }
    }
    __syncthreads();
    prefix |= s_bin << shift;
    mask |= top << shift;
    need -= s_above;
    const uint32_t match = s_count;
    if (match == need) break;  // all keys that match the digits so far stay: the other digits decide nothing
    if (match <= kFew) {
      // few keys match: the one that (need - 1) others precede, by key and then slot, is the last kept
      unsigned long long *few = reinterpret_cast<unsigned long long *>(from);
      if (tid == 0) few[match] = 0;  // the list is read in pairs
      for (int j = tid * 4; j < n; j += NT * 4) {
        const uint4 four = *reinterpret_cast<const uint4 *>(keys + j);
        const uint32_t k[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((k[e] & mask) == prefix && j + e < n)
            few[atomicAdd(&s_found, 1u)] = (unsigned long long)k[e] << 32 | (uint32_t)~(j + e);
      }
      __syncthreads();
      if (tid < (int)match) {
        const unsigned long long me = few[tid];
        uint32_t ahead = 0;
#pragma unroll 4
        for (uint32_t i = 0; i < match; i += 2) {
          const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(few + i);
          ahead += (two.x > me) + (two.y > me);
        }
        if (ahead == need - 1) s_key = (uint32_t)(me >> 32), s_slot = (int)~(uint32_t)me;
      }
      __syncthreads();
      prefix = s_key;
      mask = 0xffffffffu;
      last_slot = s_slot;
      break;
    }
    if (digit == 2) last_slot = -1;  // many equal keys: found by the prefix sum below
  }

  // Of the four slots from j on, a bit for each below `bound`.
  auto below = [](int j, int bound) { return (1u << min(max(bound - j, 0), 4)) - 1u; };
  // Sets the flags that f(first of four slots, their keys) gives; returns their number.
  auto flag = [&](auto f) {
    uint32_t mine = 0;
#pragma unroll 2
    for (int w = warp; w < nb; w += NW) {
      const int j = w * 128 + lane * 4;
      const uint4 k = *reinterpret_cast<const uint4 *>(keys + j);
      const uint32_t four = f(j, make_uint4(k.x & mask, k.y & mask, k.z & mask, k.w & mask)) & below(j, n);
      uint32_t word = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t all = __ballot_sync(0xffffffffu, four >> e & 1u);
        mine += __popc(all);
        if (lane == e) word = all;
      }
      if (lane < 4) flags[w * 4 + lane] = word;
    }
    if (lane == 0) tot[warp] = mine;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, lane < NW ? tot[lane] : 0u);
  };
  // Calls f(j, number of flags in front) for the flagged slots of this warp's
  // blocks that wanted(first, end of their numbers) admits; every warp counts
  // all blocks, 32 at a time, for itself.
  auto flagged = [&](auto wanted, auto f) {
    uint32_t front = 0;
    for (int w0 = 0; w0 < nb; w0 += 32) {
      uint32_t c = 0;
      if (w0 + lane < nb) {
        const uint4 v = *reinterpret_cast<const uint4 *>(flags + (w0 + lane) * 4);
        c = __popc(v.x) + __popc(v.y) + __popc(v.z) + __popc(v.w);
      }
      const uint32_t inc = warp_scan(c);
      for (int w = w0 + warp; w < min(nb, w0 + 32); w += NW) {
        const uint32_t base = front + __shfl_sync(0xffffffffu, inc - c, w - w0);
        const uint32_t end = front + __shfl_sync(0xffffffffu, inc, w - w0);
        if (base == end || !wanted((int)base, (int)end)) continue;
        const uint4 v = *reinterpret_cast<const uint4 *>(flags + w * 4);
        const uint32_t word[4] = {v.x, v.y, v.z, v.w}, lower = (1u << lane) - 1u;
        uint32_t at = base + __popc(v.x & lower) + __popc(v.y & lower) + __popc(v.z & lower) + __popc(v.w & lower);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (word[e] >> lane & 1u) f(w * 128 + lane * 4 + e, at++);
        }
      }
      front += __shfl_sync(0xffffffffu, inc, 31);
    }
  };
  auto bits = [](bool a, bool b, bool c, bool d) { return (uint32_t)a | (uint32_t)b << 1 | (uint32_t)c << 2 | (uint32_t)d << 3; };
  if (last_slot < 0) {
    flag([&](int, const uint4 &k) { return bits(k.x == prefix, k.y == prefix, k.z == prefix, k.w == prefix); });
    flagged([&](int base, int end) { return base < (int)need && (int)need <= end; },
            [&](int j, uint32_t at) {
              if (at == need - 1) s_slot = j;
            });
    __syncthreads();
    last_slot = s_slot;
    __syncthreads();
  }
  const int upto = min(last_slot, n - 1) + 1;
  const int moves = (int)(flag([&](int j, const uint4 &k) {
                            const uint32_t more = bits(k.x > prefix, k.y > prefix, k.z > prefix, k.w > prefix);
                            const uint32_t same = bits(k.x == prefix, k.y == prefix, k.z == prefix, k.w == prefix);
                            return (more | (same & below(j, upto))) ^ below(j, b);  // kept and behind the budget, or neither
                          }) / 2);
  if (C > 1) ptx::cluster_sync_all();  // every CTA has read the scores: they may change

  constexpr int LPR = D * 2 / 16;      // lanes per row
  constexpr int TPW = 32 / (2 * LPR);  // tokens a warp moves at once (K and V rows)
  constexpr int U = 4;
  const int sub = lane / (2 * LPR), which = (lane / LPR) & 1, at = lane % LPR;
  uint4 *cache = static_cast<uint4 *>(which ? a.v_cache : a.k_cache);
  // the CTA's share of the ranks, kWindow at a time
  const int share = (moves + C - 1) / C, r0 = min(moves, rank * share), r1 = min(moves, r0 + share);
  for (int q0 = r0; q0 < r1; q0 += kWindow) {
    const int cnt = min(r1 - q0, kWindow);
    flagged([&](int base, int end) { return (base < q0 + cnt && end > q0) || (base < moves + q0 + cnt && end > moves + q0); },
            [&](int j, uint32_t at) {
              int i = (int)at - q0;
              uint32_t *list = to;
              if (j >= b) i -= moves, list = from;
              if (i >= 0 && i < cnt) list[i] = (uint32_t)j;
            });
    __syncthreads();
    for (int i = tid; i < cnt; i += NT) {  // slots to rows, and the tracking entries
      const uint32_t src = row_of((int)from[i]);
      uint32_t dst = row_of((int)to[i]);
      if (src == kNoRow) dst = kNoRow;  // a bad page, reported above
      if (dst != kNoRow) {
        a.scores[dst] = a.scores[src];
        a.positions[dst] = a.positions[src];
      }
      from[i] = src;
      to[i] = dst;
    }
    __syncthreads();
    for (int i = warp * TPW + sub; i - sub < cnt; i += NW * TPW * U) {
      uint4 v[U];
      uint32_t out[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int e = i + u * NW * TPW;
        out[u] = e < cnt ? to[e] : kNoRow;
        if (out[u] != kNoRow) v[u] = cache[(size_t)from[e] * LPR + at];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (out[u] != kNoRow) cache[(size_t)out[u] * LPR + at] = v[u];
    }
    __syncthreads();
  }
}

struct EvictPlan {
  int threads, cluster;
};
inline EvictPlan evict_plan(int R, int Hkv, int max_len, int budget, int num_sms) {
  EvictPlan p;
  const long long heads = (long long)R * Hkv;
  // about eight keys a thread (512 heads of 2112 slots: 20 us with 256 threads, 27 with 512; 128 heads of 8192: 53 us
  // with 1024, 61 with 512)
  p.threads = 256;
  while (p.threads < 1024 && p.threads * 9 < max_len) p.threads *= 2;
  // more CTAs per head while there are many tokens to move and SMs for them (one head of 30001 slots, 6227 moves:
  // 97 us with one CTA, 27 with eight; where the heads fill the SMs a second CTA only selects once more); clusters of
  // four and eight, which lie within a GPC, on three quarters of the SMs at most
  const int list = budget < max_len - budget ? budget : max_len - budget;
  p.cluster = 1;
  while (p.cluster < 8 && list > 128 * p.cluster &&
         heads * p.cluster * 2 * p.threads * 4 <= (p.cluster == 1 ? 4 : 3) * 1024ll * num_sms)
    p.cluster *= 2;
  return p;
}

}  // namespace kvb

// Launch with clusters along x, and programmatic stream serialization as launch_pdl.
template <typename... KArgs, typename... Args>
static int launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, int cluster, size_t smem, cudaStream_t st,
                          Args &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...) == cudaSuccess ? 0 : -4;
}
static inline int launched() { return cudaPeekAtLastError() == cudaSuccess ? 0 : -4; }
static inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
template <typename... P>
static inline bool any_null(P... p) {
  return (... || (p == nullptr));
}
static inline bool overlap(const int32_t *a, const int32_t *b, int n) {  // of n entries each
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b), bytes = (uintptr_t)n * sizeof(int32_t);
  return x < y + bytes && y < x + bytes;
}

extern "C" int sched_qk_norm_rope_kv_append(const QkNormArgs *args, cudaStream_t st) {
  if (args == nullptr) return -1;
  const QkNormArgs &a = *args;
  if (a.T <= 0) return 0;
  if (any_null(a.qkv, a.wq, a.wk, a.pos, a.slot, a.cos_sin, a.q_out, a.k_cache, a.v_cache)) return -1;
  if (a.Hq < 1 || a.Hkv < 1 || a.page_size < 1 || a.num_pages < 1 || a.max_pos < 1 || a.num_sms < 1) return -1;
  if ((a.D != 64 && a.D != 128) || a.rot < 16 || a.rot > a.D || a.rot % 16 != 0) return -1;
  if (a.ld_qkv % 8 != 0 || a.ld_q % 8 != 0 || (a.T > 1 && a.ld_q < (long long)a.Hq * a.D)) return -1;
  if (!aligned16(a.qkv) || !aligned16(a.wq) || !aligned16(a.wk) || !aligned16(a.cos_sin) || !aligned16(a.q_out) ||
      !aligned16(a.k_cache) || !aligned16(a.v_cache))
    return -1;
  if (a.element == kKvFp16) return a.D == 128 ? kvb::run_qk_norm<__half, 128>(a, st) : kvb::run_qk_norm<__half, 64>(a, st);
  return a.D == 128 ? kvb::run_qk_norm<__nv_bfloat16, 128>(a, st) : kvb::run_qk_norm<__nv_bfloat16, 64>(a, st);
}

namespace kvb {
// The one-kernel forms: where all of a call's CTAs are resident at once, with
// as many of them per head as that allows.
struct OneKernel {
  int ctas, warps;  // per (request, KV head); 0: not this form
  int span;         // logits per row in a CTA's shared memory
  size_t smem;
};
inline OneKernel one_kernel(int R, int Hkv, int D, const ScoredPlan &pl, int num_sms) {
  const OneKernel none = {0, 0, 0, 0};
  if (pl.blocks > 1) return none;
  auto tiles_of = [&](int ctas, int warps) { return (pl.lp / kTile + ctas * warps - 1) / (ctas * warps); };
  auto form = [&](int ctas, int warps) {
    const int span = warps * tiles_of(ctas, warps) * kTile;
    return OneKernel{ctas, warps, span, 4 * ((size_t)warps * pl.block * D + (size_t)pl.rows * span)};
  };
  const long long heads = (long long)R * Hkv;
  // Eight CTAs of eight warps: one to an SM with heads of 128 (by its
  // registers), two with 64, and of the SMs about three quarters, since a
  // cluster lies within a GPC (of 148 SMs 14 clusters of one-to-an-SM CTAs fit,
  // which the 8 below admits; 16 do not). One request of 700 tokens, 8 heads of 128: 6.4 us against 9.3 with
  // two kernels, of 8000: 19.2 against 20.7; 16 such heads of 1000 tokens,
  // which do not fit: 12.5 against 11.6.
  if (tiles_of(8, 8) <= kCTiles) {
    const OneKernel wide = form(8, 8);
    const int per_sm = wide.smem <= 90 * 1024 ? one_resident(D, 8) : 1;  // (or by shared memory)
    if (heads * 8 * 4 <= 3ll * num_sms * per_sm + 8) return wide;
  }
  // Four, two or one of four warps, with up to four tiles a warp, or eight if
  // they fill half of the device. 8 heads of 128: 8 requests of 1000 tokens
  // 12.2 us with four CTAs a head against 16.2 with two kernels, 16 of 500
  // 11.7 with two against 16.4 (16.2 with four, which are not resident), 32 of
  // 500 18.5 with one against 23.5; 4 of 2000, a quarter of the device with
  // four of eight tiles, 17.7 against 16.5.
  for (int c = 4; c >= 1; c /= 2) {
    const int tiles = tiles_of(c, 4);
    if (tiles > kCTiles) break;
    const int per_sm = D == 64 && pl.block == 16 && tiles > 4 ? 3 : one_resident(D, 4);  // (3: 57 KB of shared memory each)
    const long long capacity = (long long)per_sm * num_sms;
    if (heads * c <= capacity && (tiles <= 4 || heads * c * 2 > capacity)) return form(c, 4);
  }
  // More heads with contexts of a few tiles: two waves of one CTA each, three
  // with heads of 64 (64 requests of 10 to 64 tokens, 8 heads of 128, 9.5 us
  // against 13.1 with two kernels, of up to 250 18.6 against 17.3, 128 of 64 17.8
  // against 17.4; with heads of 64 200 of up to 250 22.7 against 28.5).
  const long long capacity = (long long)one_resident(D, 4) * num_sms;
  return tiles_of(1, 4) <= (D == 64 ? 4 : 2) && heads <= capacity * (D == 64 ? 3 : 2) ? form(1, 4) : none;
}

template <typename T, int D, int ROWS>
auto one_kernel_for(int ctas) {
  return ctas == 8   ? scored_cluster_kernel<T, D, ROWS, 8, 8>
         : ctas == 4 ? scored_cluster_kernel<T, D, ROWS, 4, 4>
         : ctas == 2 ? scored_cluster_kernel<T, D, ROWS, 2, 4>
                     : scored_cluster_kernel<T, D, ROWS, 1, 4>;
}

template <typename T, int D>
int run_scored(const ScoredArgs &a, const ScoredPlan &pl, cudaStream_t st) {
  if (const OneKernel one = one_kernel(a.R, a.Hkv, D, pl, a.num_sms); one.ctas > 0) {
    auto *k = pl.block == 8 ? one_kernel_for<T, D, 8>(one.ctas) : one_kernel_for<T, D, 16>(one.ctas);
    if (one.smem > 8 * 1024 &&
        cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * one.warps * (16 * D + 16 * kCTiles * kTile)) !=
            cudaSuccess)
      return -4;
    const dim3 grid(one.ctas, a.Hkv, a.R), block(one.warps * 32);
    if (one.ctas > 1) return launch_cluster(k, grid, block, one.ctas, one.smem, st, a, pl.rows, one.span);
    launch_pdl(k, grid, block, one.smem, st, a, pl.rows, one.span);
    return launched();
  }
  auto *split = pl.block == 8 ? scored_split_kernel<T, D, 8> : scored_split_kernel<T, D, 16>;
  launch_pdl(split, dim3(pl.grid), dim3(kWarps * 32), 0, st, a, pl);
  if (cudaPeekAtLastError() != cudaSuccess) return -4;
  const int o_ctas = pl.o_rows > 0 ? (pl.rows + pl.o_rows - 1) / pl.o_rows : 0;
  launch_pdl(scored_join_kernel<T, D>, dim3(o_ctas + (a.max_len + pl.join - 1) / pl.join, a.Hkv, a.R), dim3(kJoin),
             (size_t)(pl.rows + 4 * kJoin) * sizeof(float), st, a, pl, o_ctas);
  return launched();
}
}  // namespace kvb

extern "C" long long sched_attn_scored_ws_floats(int R, int Q, int Hq, int Hkv, int D, int max_len, int num_sms) {
  if (R <= 0 || Q <= 0 || Hkv <= 0 || Hq < Hkv || max_len <= 0) return 0;
  const kvb::ScoredPlan pl = kvb::scored_plan(R, Q, Hq, Hkv, D, max_len, num_sms);
  return kvb::one_kernel(R, Hkv, D, pl, num_sms).ctas > 0 ? 0 : pl.total;
}

extern "C" int sched_attn_scored(const ScoredArgs *args, cudaStream_t st) {
  if (args == nullptr) return -1;
  const ScoredArgs &a = *args;
  if (a.R <= 0 || a.Q <= 0) return 0;
  if (any_null(a.q, a.out, a.k_cache, a.v_cache, a.scores, a.block_table, a.kv_lens) || a.num_sms < 1) return -1;
  if (a.Hkv < 1 || a.Hq < a.Hkv || a.Hq % a.Hkv != 0 || (a.D != 64 && a.D != 128)) return -1;
  if (a.page_size < 16 || a.page_size % 16 != 0 || a.num_pages < 1 || a.max_len < 1 || a.bt_pages < 1) return -1;
  if (a.R > 65535 || a.Hkv > 65535 || a.max_len >= 1 << 30 || (long long)a.Q * (a.Hq / a.Hkv) > 8192) return -1;
  // q, K, V and out are accessed 16 bytes at a time, as are scores and ws
  if (a.q_req % 8 != 0 || a.q_query % 8 != 0 || a.out_req % 8 != 0 || a.out_query % 8 != 0) return -1;
  if (!aligned16(a.q) || !aligned16(a.out) || !aligned16(a.k_cache) || !aligned16(a.v_cache) || !aligned16(a.scores) ||
      !aligned16(a.ws))
    return -1;
  const kvb::ScoredPlan pl = kvb::scored_plan(a.R, a.Q, a.Hq, a.Hkv, a.D, a.max_len, a.num_sms);
  // the tile list is indexed in 32 bits (2^31 tiles are 2^35 cached tokens and heads)
  if ((long long)a.R * a.Hkv * pl.blocks * (pl.lp / kvb::kTile) > 0x7fffffffll) return -1;
  if (kvb::one_kernel(a.R, a.Hkv, a.D, pl, a.num_sms).ctas == 0 && (a.ws == nullptr || a.ws_floats < pl.total)) return -2;
  if (a.element == kKvFp16)
    return a.D == 128 ? kvb::run_scored<__half, 128>(a, pl, st) : kvb::run_scored<__half, 64>(a, pl, st);
  return a.D == 128 ? kvb::run_scored<__nv_bfloat16, 128>(a, pl, st) : kvb::run_scored<__nv_bfloat16, 64>(a, pl, st);
}

// the keys and flags of contexts that shared memory does not hold, for each CTA
extern "C" long long sched_kv_evict_ws_ints(int R, int Hkv, int max_len, int budget, int num_sms) {
  if (R <= 0 || Hkv <= 0 || max_len <= budget || max_len <= kvb::kKeySmem) return 0;
  return (long long)R * Hkv * kvb::evict_plan(R, Hkv, max_len, budget, num_sms).cluster * (long long)kvb::evict_words(max_len);
}

extern "C" int sched_kv_evict(const KvEvictArgs *args, cudaStream_t st) {
  if (args == nullptr) return -1;
  const KvEvictArgs &a = *args;
  if (a.R <= 0) return 0;
  if (any_null(a.k_cache, a.v_cache, a.scores, a.positions, a.block_table, a.kv_lens, a.last_pos, a.new_lens) || a.num_sms < 1)
    return -1;
  if (overlap(a.new_lens, a.kv_lens, a.R) || overlap(a.new_lens, a.last_pos, a.R)) return -1;  // every head reads the old ones
  if (a.Hkv < 1 || (a.D != 64 && a.D != 128) || a.page_size < 1 || a.num_pages < 1 || a.bt_pages < 1) return -1;
  if (a.budget < 1 || a.recent < 0 || a.sink < 0 || (long long)a.recent + a.sink > a.budget || a.max_len < 1) return -1;
  if (a.R > 65535 || a.Hkv > 65535 || a.max_len >= 1 << 30 || !aligned16(a.k_cache) || !aligned16(a.v_cache)) return -1;
  if ((long long)a.num_pages * a.Hkv * a.page_size >= 0xffffffffll) return -1;  // rows are numbered in 32 bits
  const long long need = sched_kv_evict_ws_ints(a.R, a.Hkv, a.max_len, a.budget, a.num_sms);
  if (need > 0 && (a.ws == nullptr || a.ws_ints < need)) return -2;
  if (need > 0 && !aligned16(a.ws)) return -1;  // keys and flags are read 16 bytes at a time
  const kvb::EvictPlan p = kvb::evict_plan(a.R, a.Hkv, a.max_len, a.budget, a.num_sms);
  auto *k = need > 0 ? (a.D == 128 ? kvb::evict_kernel<128, true> : kvb::evict_kernel<64, true>)
                     : (a.D == 128 ? kvb::evict_kernel<128, false> : kvb::evict_kernel<64, false>);
  const size_t smem = need == 0 && a.max_len > a.budget ? kvb::evict_words(a.max_len) * 4 : 0;
  if (smem > 24 * 1024 &&
      cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kvb::evict_words(kvb::kKeySmem) * 4) != cudaSuccess)
    return -4;
  // vectors of four slots where pages hold whole ones
  const int vec = a.page_size % 4 == 0 && aligned16(a.scores) && aligned16(a.positions);
  int shift = -1;  // log2 of the page size where it is a power of two
  if ((a.page_size & (a.page_size - 1)) == 0)
    for (shift = 0; (1 << shift) < a.page_size;) ++shift;
  return launch_cluster(k, dim3(p.cluster, a.Hkv, a.R), dim3(p.threads), p.cluster, smem, st, a,
                        need > 0 ? reinterpret_cast<uint32_t *>(a.ws) : nullptr, vec, shift);
}
