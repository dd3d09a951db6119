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
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16(v);
}
template <>
__device__ __forceinline__ __half narrow<__half>(float v) {
  return __float2half(v);
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &u, float (&f)[8]) {
  const float2 a = unpack2<T>(u.x), b = unpack2<T>(u.y), c = unpack2<T>(u.z), d = unpack2<T>(u.w);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y, f[4] = c.x, f[5] = c.y, f[6] = d.x, f[7] = d.y;
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// ------------------------------------------------------------------ norm + rotation + append
// y = x / sqrt(mean(x^2) + eps) * w over a head's D values, then the first
// rot values turn in pairs (d, d + rot/2). All in fp32, rounded once.
//
// D/16 lanes share a head: each holds the two 8-value chunks whose values
// pair up (chunks l and l + rot/16; lanes behind the rotated part hold the
// unrotated chunks 2l and 2l + 1), so the rotation needs no exchange and
// every access is a 16-byte vector. The grid is flat over (token, head).
template <typename T, int D>
__global__ void __launch_bounds__(256) qk_norm_kernel(const QkNormArgs a) {
  constexpr int LANES = D / 16;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int nheads = a.Hq + 2 * a.Hkv;
  const long long items = (long long)a.T * nheads;
  long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / LANES;
  const bool live = item < items;
  if (!live) item = items - 1;  // takes part in the warp's shuffles, writes nothing
  const int t = (int)(item / nheads), h = (int)(item - (long long)t * nheads);
  const int l = threadIdx.x % LANES;
  const int nr = a.rot / 16;
  const int c0 = l < nr ? l : 2 * l, c1 = l < nr ? l + nr : 2 * l + 1;
  const T *src = static_cast<const T *>(a.qkv) + (size_t)t * a.ld_qkv + (size_t)h * D;
  uint4 u0 = *reinterpret_cast<const uint4 *>(src + c0 * 8);
  uint4 u1 = *reinterpret_cast<const uint4 *>(src + c1 * 8);
  const int p = a.pos[t];
  int s = a.slot[t];
  const bool pos_ok = p >= 0 && p < a.max_pos;
  const bool slot_ok = (long long)s < (long long)a.num_pages * a.page_size;
  if (live && h == 0 && l == 0) {
    if (!pos_ok)
      report_bad_index(a.status, kSiteNormPos, p);
    else if (!slot_ok)
      report_bad_index(a.status, kSiteKvSlot, s);
  }
  if (!slot_ok || !pos_ok) s = -1;  // no cache write
  if (h < a.Hq + a.Hkv) {
    float x0[8], x1[8];
    unpack8<T>(u0, x0);
    unpack8<T>(u1, x1);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += x0[j] * x0[j] + x1[j] * x1[j];
    // the lanes of a head are aligned neighbours and take this branch together
    const unsigned mask = (LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u)) << (ptx::lane_id() / LANES * LANES);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    const float inv = rsqrtf(ss / (float)D + a.eps);
    const T *w = static_cast<const T *>(h < a.Hq ? a.wq : a.wk);
    float w0[8], w1[8];
    unpack8<T>(*reinterpret_cast<const uint4 *>(w + c0 * 8), w0);
    unpack8<T>(*reinterpret_cast<const uint4 *>(w + c1 * 8), w1);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x0[j] *= inv * w0[j];
      x1[j] *= inv * w1[j];
    }
    if (l < nr && pos_ok) {
      const float4 *cs = reinterpret_cast<const float4 *>(a.cos_sin + ((size_t)p * (a.rot / 2) + l * 8) * 2);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 v = cs[j];  // (cos, sin) of two pairs
        const float a0 = x0[2 * j], b0 = x1[2 * j], a1 = x0[2 * j + 1], b1 = x1[2 * j + 1];
        x0[2 * j] = a0 * v.x - b0 * v.y;
        x1[2 * j] = b0 * v.x + a0 * v.y;
        x0[2 * j + 1] = a1 * v.z - b1 * v.w;
        x1[2 * j + 1] = b1 * v.z + a1 * v.w;
      }
    }
    u0 = pack8<T>(x0);
    u1 = pack8<T>(x1);
  }
  if (!live) return;
  T *dst;
  if (h < a.Hq) {
    if (!pos_ok) u0 = u1 = make_uint4(0, 0, 0, 0);
    dst = static_cast<T *>(a.q_out) + (size_t)t * a.ld_q + (size_t)h * D;
  } else {
    if (s < 0) return;
    const int kvh = h < a.Hq + a.Hkv ? h - a.Hq : h - a.Hq - a.Hkv;
    const int page = s / a.page_size;
    const size_t row = ((size_t)page * a.Hkv + kvh) * a.page_size + (s - page * a.page_size);
    dst = static_cast<T *>(h < a.Hq + a.Hkv ? a.k_cache : a.v_cache) + row * D;
    if (l == 0 && h < a.Hq + a.Hkv) {
      if (a.scores != nullptr) a.scores[row] = 0.f;
      if (a.positions != nullptr) a.positions[row] = p;
    }
  }
  *reinterpret_cast<uint4 *>(dst + c0 * 8) = u0;
  *reinterpret_cast<uint4 *>(dst + c1 * 8) = u1;
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
constexpr int kResident = 3;   // CTAs of the split kernel per SM
constexpr int kMinRun = 2;     // tiles per warp at least: bounds the partial results

struct ScoredPlan {
  int rows, lp;         // query rows per KV head, padded length
  int block, blocks;    // rows per task (8 or 16), tasks per (request, KV head)
  int grid, join;       // CTAs of the split kernel, tokens per CTA of the join
  long long s_off, o_off, ml_off, total;
};

inline ScoredPlan scored_plan(int R, int Q, int Hq, int Hkv, int D, int max_len, int num_sms) {
  ScoredPlan p;
  p.rows = Q * (Hq / Hkv);
  p.lp = (max_len + kTile - 1) / kTile * kTile;
  p.block = p.rows <= 8 ? 8 : 16;
  p.blocks = (p.rows + p.block - 1) / p.block;
  const long long heads = (long long)R * Hkv, tasks = heads * p.blocks;
  const long long most = (tasks * (p.lp / kTile) + kMinRun * kWarps - 1) / (kMinRun * kWarps);
  const long long fill = (long long)num_sms * kResident;
  p.grid = (int)(most < fill ? most : fill);
  p.join = 2048;
  while (p.join > 256 && heads * ((max_len + p.join - 1) / p.join) < num_sms) p.join /= 2;
  p.s_off = 0;
  p.o_off = heads * p.rows * p.lp;
  const long long parts = (long long)p.grid * kWarps + tasks;
  p.ml_off = p.o_off + parts * p.block * D;
  p.total = p.ml_off + parts * p.block * 2;
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

__device__ __forceinline__ uint4 ld_stream(const void *p) {  // read once: not kept in L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
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

// One warp: a run of tiles. K and V go from global memory straight into the
// registers of the m16n8k16 operands (K of the next tile is requested once
// this one's logits are done, V once its product is), so a warp always has
// loads in flight and there is no shared-memory staging; Q waits in shared
// memory in operand order. Query rows are the M side (8 of its 16 rows where
// a KV head has at most 8 query rows), tokens the N side of the logits and
// the K side of the output.
//
// Operand layout, for lane 4 r + c: the 16 bytes of K at value 32 kk + 8 c of
// tokens r and r + 8 are the k-slots of two products, Q's registers hold the
// same values; the 16 bytes of V at value 64 i + 8 r of tokens 2c, 2c + 1,
// 2c + 8 and 2c + 9 are column r of the eight products (i, e), column n of
// which is value 64 i + 8 n + e.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kWarps * 32, kResident)
    scored_split_kernel(const ScoredArgs a, const ScoredPlan pl) {
  constexpr int NK = D / 32, RB = ROWS / 8;
  __shared__ uint4 q_sm[kWarps][RB][NK][32];
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int cap = table_cap(a.max_len, a.bt_pages, a.page_size);
  const int G = a.Hq / a.Hkv, HB = a.Hkv * pl.blocks;
  const uint32_t w_id = blockIdx.x * kWarps + warp;
  auto tiles_of = [&](int n) { return (n + kTile - 1) / kTile; };

  // this warp's run of the list (its length fits 31 bits)
  uint32_t total = 0;
  for (int i = lane; i < a.R; i += 32) total += tiles_of(checked_len(a.kv_lens[i], cap, a.status, kSiteScoredLen, w_id == 0));
  total = __reduce_add_sync(0xffffffffu, total) * HB;
  const uint32_t per = run_length(total, gridDim.x * kWarps);
  if ((unsigned long long)w_id * per >= total) return;
  const uint32_t u0 = w_id * per;
  uint32_t left = min(per, total - u0);
  int req = 0, hb = 0, tile = 0;
  {
    uint32_t before = 0;  // tiles (of one head) in front of request i0
    for (int i0 = 0;; i0 += 32) {
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

  int lim[RB], all_see = 0;  // tokens that rows r, r + 8 see; tokens that every row of the task sees
  const float scale2 = a.sm_scale * kLog2e;
  float *s_out = nullptr;
  auto enter_task = [&]() {
    const int h = hb / pl.blocks, row0 = (hb - h * pl.blocks) * ROWS;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      const int row = row0 + r + 8 * i;
      lim[i] = 0;
      const T *src = nullptr;
      if (row < pl.rows) {
        const int qi = row / G, g = row - qi * G;
        lim[i] = n - (a.Q - 1 - qi);
        src = static_cast<const T *>(a.q) + (size_t)req * a.q_req + (size_t)qi * a.q_query + (size_t)(h * G + g) * D + c * 8;
      }
#pragma unroll
      for (int kk = 0; kk < NK; ++kk)  // each lane reads back only what it wrote
        q_sm[warp][i][kk][lane] = src != nullptr ? *reinterpret_cast<const uint4 *>(src + kk * 32) : make_uint4(0, 0, 0, 0);
    }
    all_see = n - (a.Q - 1 - row0 / G);
    s_out = a.ws + pl.s_off + ((size_t)req * a.Hkv + h) * pl.rows * pl.lp + (size_t)(row0 + r) * pl.lp + 2 * c;
  };
  // first element of a tile's K rows, or a negative number for a bad page
  auto tile_row = [&](int q, int hb_, int t) -> long long {
    const int tok = t * kTile, col = tok / a.page_size;
    const int page = a.block_table[(size_t)q * a.bt_stride + col];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) report_bad_index(a.status, kSiteScoredPage, page);
      return -1;
    }
    return (((long long)page * a.Hkv + hb_ / pl.blocks) * a.page_size + (tok - col * a.page_size)) * D;
  };
  uint4 kx[2][NK], vx[D / 64][4];
  auto load_k = [&](long long base) {
    const T *p = static_cast<const T *>(a.k_cache) + (base < 0 ? 0 : base) + r * D + c * 8;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) kx[j][kk] = ld_stream(p + j * 8 * D + kk * 32);
  };
  auto load_v = [&](long long base) {
    const T *p = static_cast<const T *>(a.v_cache) + (base < 0 ? 0 : base) + 2 * c * D + r * 8;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) vx[i][j] = ld_stream(p + ((j & 1) + (j / 2) * 8) * D + i * 64);
  };

  float o[D / 8][ROWS / 4];
  float m[RB], sum[RB];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int j = 0; j < ROWS / 4; ++j) o[i][j] = 0.f;
#pragma unroll
    for (int i = 0; i < RB; ++i) m[i] = -INFINITY, sum[i] = 0.f;
  };

  long long base = tile_row(req, hb, tile);
  load_k(base);
  load_v(base);
  enter_task();
  clear();
  int nt = tiles_of(n);
  while (true) {
    --left;
    int n_req = req, n_hb = hb, n_tile = tile + 1, n_n = n;
    const bool task_ends = n_tile == nt || left == 0;
    long long next = -1;
    if (left > 0) {
      if (n_tile == nt) {
        n_tile = 0;
        if (++n_hb == HB) {
          n_hb = 0;
          do n_n = checked_len(a.kv_lens[++n_req], cap, nullptr, 0, false);
          while (n_n == 0);  // more tiles follow, so a request with some does
        }
      }
      next = tile_row(n_req, n_hb, n_tile);
    }
    float s[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const uint4 q0 = q_sm[warp][0][kk][lane];
      const uint4 q1 = ROWS == 16 ? q_sm[warp][RB - 1][kk][lane] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mma16816<T>(s[j][0], s[j][1], s[j][2], s[j][3], q0.x, q1.x, q0.y, q1.y, kx[j][kk].x, kx[j][kk].y);
        mma16816<T>(s[j][0], s[j][1], s[j][2], s[j][3], q0.z, q1.z, q0.w, q1.w, kx[j][kk].z, kx[j][kk].w);
      }
    }
    if (left > 0) load_k(next);
    // tokens from `end` on are not there (behind the request's end, or their page is bad)
    const int tok = tile * kTile;
    const int end = base < 0 ? tok : n;
    const bool whole = tok + kTile <= min(end, all_see);
    uint32_t pa[2][2] = {{0u, 0u}, {0u, 0u}};  // [row block][tile half]: P as the product's A operand
    const int row0 = (hb % pl.blocks) * ROWS;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      float v[4] = {s[0][2 * i] * scale2, s[0][2 * i + 1] * scale2, s[1][2 * i] * scale2, s[1][2 * i + 1] * scale2};
      if (!whole) {
        const int seen = min(end, lim[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (tok + (j / 2) * 8 + 2 * c + (j & 1) >= seen) v[j] = -INFINITY;
      }
      if (row0 + r + 8 * i < pl.rows) {
        float *dst = s_out + (size_t)(8 * i) * pl.lp + tok;
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
      pa[i][0] = pack2<T>(v[0], v[1]);
      pa[i][1] = pack2<T>(v[2], v[3]);
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
    if (left > 0) load_v(next);
    if (task_ends) {
      const size_t part = (size_t)w_id + (uint32_t)req * HB + hb;
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        const int row = r + 8 * i;
        if (row0 + row < pl.rows) {
          float *dst = a.ws + pl.o_off + (part * ROWS + row) * D + 16 * c;
#pragma unroll
          for (int d = 0; d < D / 64; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const int x = d * 8 + e % 8, y = 2 * i + e / 8;
              *reinterpret_cast<float4 *>(dst + d * 64 + e) = make_float4(o[x][y], o[x + 1][y], o[x + 2][y], o[x + 3][y]);
            }
          if (c == 0) reinterpret_cast<float2 *>(a.ws + pl.ml_off)[part * ROWS + row] = make_float2(m[i], sum[i]);
        }
      }
      if (left == 0) return;
      req = n_req, hb = n_hb, n = n_n;
      nt = tiles_of(n);
      enter_task();
      clear();
    }
    tile = n_tile;
    base = next;
  }
}

__device__ __forceinline__ void red_add4(float *p, const float4 &v) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

// Join. The first CTAs of a (request, KV head) join the outputs of two rows
// each (four warps to a row, each a quarter of the partial results); the
// others add the weights of pl.join tokens each: a thread has four tokens and
// every groups-th row, whose logits it requests before the rows' lse is known.
// All sums have a fixed order, and one request's pages get one addition per
// token and head from a call.
constexpr int kJoin = 256;
constexpr int kJoinRows = 2;

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

template <typename T, int D>
__global__ void __launch_bounds__(kJoin) scored_join_kernel(const ScoredArgs a, const ScoredPlan pl, int o_ctas) {
  extern __shared__ __align__(16) float sm[];
  __shared__ uint32_t red[2][kJoin / 32];
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int req = blockIdx.z, h = blockIdx.y;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int cap = table_cap(a.max_len, a.bt_pages, a.page_size);
  const int n = checked_len(a.kv_lens[req], cap, nullptr, 0, false);
  const bool weigh = (int)blockIdx.x >= o_ctas;
  const int t0 = ((int)blockIdx.x - o_ctas) * pl.join, t1 = min(n, t0 + pl.join);
  if (weigh && t0 >= n) return;
  const int G = a.Hq / a.Hkv, HB = a.Hkv * pl.blocks, nt = (n + kTile - 1) / kTile;

  // this thread's first logits
  constexpr int PRE = 4;
  const int quads = min(pl.join / 4, kJoin), groups = kJoin / quads, grp = tid / quads, quad = tid % quads;
  const float *s_in = a.ws + pl.s_off + ((size_t)req * a.Hkv + h) * pl.rows * pl.lp;
  float4 pre[PRE];
  if (weigh && t0 + quad * 4 < t1) {
#pragma unroll
    for (int j = 0; j < PRE; ++j)
      if (grp + j * groups < pl.rows)
        pre[j] = *reinterpret_cast<const float4 *>(s_in + (size_t)(grp + j * groups) * pl.lp + t0 + quad * 4);
  }
  uint32_t before = 0, total = 0;
  for (int i = tid; i < a.R; i += kJoin) {
    const uint32_t t = (uint32_t)(checked_len(a.kv_lens[i], cap, nullptr, 0, false) + kTile - 1) / kTile;
    total += t;
    if (i < req) before += t;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  total = __reduce_add_sync(0xffffffffu, total);
  if (lane == 0) red[0][warp] = before, red[1][warp] = total;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < kJoin / 32; ++w) before += red[0][w], total += red[1][w];
  const uint32_t per = run_length(total * HB, (uint32_t)(pl.grid * kWarps));
  const float2 *ml = reinterpret_cast<const float2 *>(a.ws + pl.ml_off);

  if (!weigh) {
    constexpr int SUB = kJoin / 32 / kJoinRows, V = D / 32;  // warps per row, values per lane
    const int row = blockIdx.x * kJoinRows + warp / SUB, sub = warp % SUB;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
    if (row < pl.rows) {
      const Parts pt = parts_of(before, per, nt, HB, req, h * pl.blocks + row / pl.block);
      const float2 *mr = ml + (size_t)pt.first * pl.block + row % pl.block;
      const float lse2 = row_lse2<32>(mr, pt.count, pl.block);
      const float ref = lse2 == -INFINITY ? INFINITY : lse2;
      const float *src = a.ws + pl.o_off + ((size_t)pt.first * pl.block + row % pl.block) * D + lane * V;
#pragma unroll 4
      for (uint32_t k = sub; k < pt.count; k += SUB) {
        const float f = ex2_approx(mr[(size_t)k * pl.block].x - ref);
        float p[V];
        if constexpr (V == 4)
          *reinterpret_cast<float4 *>(p) = *reinterpret_cast<const float4 *>(src + (size_t)k * pl.block * D);
        else
          *reinterpret_cast<float2 *>(p) = *reinterpret_cast<const float2 *>(src + (size_t)k * pl.block * D);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += f != 0.f ? p[e] * f : 0.f;
      }
      if (sub == 0 && lane == 0 && a.lse != nullptr) {
        const int qi = row / G;
        a.lse[((size_t)req * a.Q + qi) * a.Hq + h * G + (row - qi * G)] = lse2 * kLn2;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) sm[warp * D + lane * V + e] = v[e];
    __syncthreads();
    if (row < pl.rows && sub == 0) {
      const int qi = row / G;
      T *dst = static_cast<T *>(a.out) + (size_t)req * a.out_req + (size_t)qi * a.out_query + (size_t)(h * G + row - qi * G) * D;
#pragma unroll
      for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int w = 1; w < SUB; ++w) v[e] += sm[(warp + w) * D + lane * V + e];
        dst[lane * V + e] = narrow<T>(v[e]);
      }
    }
    return;
  }

  float4 *part_w = reinterpret_cast<float4 *>(sm);  // [kJoin]
  float *lse2 = sm + 4 * kJoin;                     // [rows]: +inf for a row that sees nothing
  constexpr int LR = 8;                             // lanes per row
  for (int row = tid / LR; row - tid / LR < pl.rows; row += kJoin / LR) {
    const bool in = row < pl.rows;
    const Parts pt = parts_of(before, per, nt, HB, req, h * pl.blocks + (in ? row : 0) / pl.block);
    const float v = row_lse2<LR>(ml + (size_t)pt.first * pl.block + (in ? row : 0) % pl.block, pt.count, pl.block);
    if (in && tid % LR == 0) lse2[row] = v == -INFINITY ? INFINITY : v;
  }
  __syncthreads();
  for (int tq = t0; tq < t1; tq += quads * 4) {
    const int tok = tq + quad * 4;
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4 &s, float ref) {
      w.x += ex2_approx(s.x - ref);
      w.y += ex2_approx(s.y - ref);
      w.z += ex2_approx(s.z - ref);
      w.w += ex2_approx(s.w - ref);
    };
    if (tok < t1) {
#pragma unroll
      for (int j = 0; j < PRE; ++j)
        if (grp + j * groups < pl.rows) add(pre[j], lse2[grp + j * groups]);
#pragma unroll 4
      for (int row = grp + PRE * groups; row < pl.rows; row += groups)
        add(*reinterpret_cast<const float4 *>(s_in + (size_t)row * pl.lp + tok), lse2[row]);
    }
    if (tok + quads * 4 < t1) {
#pragma unroll
      for (int j = 0; j < PRE; ++j)
        if (grp + j * groups < pl.rows)
          pre[j] = *reinterpret_cast<const float4 *>(s_in + (size_t)(grp + j * groups) * pl.lp + tok + quads * 4);
    }
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
    if (grp != 0 || tok >= t1) continue;
    const int col = tok / a.page_size, page = a.block_table[(size_t)req * a.bt_stride + col];
    if (page < 0 || page >= a.num_pages) continue;  // reported by the split kernel
    float *dst = a.scores + ((size_t)page * a.Hkv + h) * a.page_size + (tok - col * a.page_size);
    if (tok + 4 <= t1) {
      red_add4(dst, w);
    } else {
      atomicAdd(dst, w.x);
      if (tok + 1 < t1) atomicAdd(dst + 1, w.y);
      if (tok + 2 < t1) atomicAdd(dst + 2, w.z);
    }
  }
}

// ------------------------------------------------------------------ eviction
// Of the n > budget cached tokens of a (request, KV head), the `budget` with
// the largest (key, lowest slot) stay: the key orders the protected tokens
// (position > last - recent, or < sink) above every weight, weights by value,
// NaN and -inf lowest. Kept tokens in slots >= budget then take the slots
// < budget of evicted ones, the i-th the i-th: sources and destinations are
// disjoint, so the moves need no order and only they touch K and V.
constexpr int kSelThreads = 1024;
constexpr int kSelBins = 4096;

__device__ __forceinline__ uint32_t evict_key(float score, int pos, int last, int recent, int sink) {
  if ((long long)pos > (long long)last - recent || pos < sink) return 0xffffffffu;
  if (!(score == score)) score = -INFINITY;
  const uint32_t u = __float_as_uint(score + 0.f);  // -0 counts as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Radix selection of the budget-th largest key in digits of 12, 10 and 10
// bits, then two ordered sweeps (each warp owns a run of slots, so ranks come
// from ballots and one prefix over the warps) that list the movers and holes.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const KvEvictArgs a, int list_cap,
                                                                   int32_t *key_ws) {
  extern __shared__ uint32_t keys_sm[];  // [max_len] unless the keys are in the workspace
  __shared__ uint32_t hist[kSelBins];
  __shared__ uint32_t wsum[32], s_bin, s_above;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int h = blockIdx.x, req = blockIdx.y;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int cap = min(a.max_len, (int)min((long long)a.bt_pages * a.page_size, 0x7fffffffll));
  const int n = checked_len(a.kv_lens[req], cap, a.status, kSiteEvictLen, h == 0 && tid == 0);
  const int b = a.budget;
  if (h == 0 && tid == 0) a.new_lens[req] = min(n, b);
  const size_t head = (size_t)req * a.Hkv + h;
  int32_t *count = a.ws + head;
  if (n <= b) {
    if (tid == 0 && a.ws != nullptr) *count = 0;
    return;
  }
  uint32_t *keys = key_ws == nullptr ? keys_sm : reinterpret_cast<uint32_t *>(key_ws) + head * (size_t)a.max_len;
  const int32_t *bt = a.block_table + (size_t)req * a.bt_stride;
  const int last = a.last_pos[req];
  for (int j = tid; j < n; j += kSelThreads) {
    const int col = j / a.page_size, page = bt[col];
    uint32_t k = 0u;
    if (page < 0 || page >= a.num_pages) {
      report_bad_index(a.status, kSiteEvictPage, page);
    } else {
      const size_t row = ((size_t)page * a.Hkv + h) * a.page_size + (j - col * a.page_size);
      k = evict_key(a.scores[row], a.positions[row], last, a.recent, a.sink);
    }
    keys[j] = k;
  }
  uint32_t prefix = 0, mask = 0;
  uint32_t need = (uint32_t)b;  // keys still to keep among those that match the prefix
  for (int digit = 0; digit < 3; ++digit) {
    const int bits = digit == 0 ? 12 : 10, shift = digit == 0 ? 20 : (digit == 1 ? 10 : 0);
    const int bins = 1 << bits;
    for (int i = tid; i < bins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += kSelThreads) {
      const uint32_t k = keys[j];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    // bins from the top: thread t owns bins/1024 of them
    const int per = bins / kSelThreads;
    uint32_t own = 0;
    for (int i = 0; i < per; ++i) own += hist[bins - 1 - (tid * per + i)];
    uint32_t inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      uint32_t v = wsum[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      wsum[lane] = v;
    }
    __syncthreads();
    uint32_t above = inc - own + (warp > 0 ? wsum[warp - 1] : 0u);
    for (int i = 0; i < per; ++i) {
      const int bin = bins - 1 - (tid * per + i);
      const uint32_t hv = hist[bin];
      if (above < need && above + hv >= need) {
        s_bin = (uint32_t)bin;
        s_above = above;
      }
      above += hv;
    }
    __syncthreads();
    prefix |= s_bin << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    need -= s_above;
    __syncthreads();
  }
  // keys > prefix stay, and the first `need` that equal it
  const int seg = ((n + 31) / 32 + 31) / 32 * 32;  // slots per warp
  const int w0 = warp * seg, w1 = min(n, w0 + seg);
  uint32_t eq = 0;
  for (int j = w0 + lane; j - lane < w1; j += 32)
    eq += __popc(__ballot_sync(0xffffffffu, j < w1 && keys[j] == prefix));
  if (lane == 0) wsum[warp] = eq;
  __syncthreads();
  uint32_t eq_base = 0;
  for (int w = 0; w < warp; ++w) eq_base += wsum[w];
  __syncthreads();
  int32_t *movers = a.ws + (size_t)a.R * a.Hkv + head * 2 * (size_t)list_cap, *holes = movers + list_cap;
  uint32_t base_h = 0, base_m = 0;
  for (int pass = 0; pass < 2; ++pass) {
    uint32_t eq_at = eq_base, nh = base_h, nm = base_m;
    for (int j = w0 + lane; j - lane < w1; j += 32) {
      const bool in = j < w1;
      const uint32_t k = in ? keys[j] : 0u;
      const uint32_t lower = (1u << lane) - 1u;
      const uint32_t beq = __ballot_sync(0xffffffffu, in && k == prefix);
      const bool keep = in && (k > prefix || (k == prefix && eq_at + __popc(beq & lower) < need));
      eq_at += __popc(beq);
      const bool hole = in && !keep && j < b, mover = keep && j >= b;
      const uint32_t bh = __ballot_sync(0xffffffffu, hole), bm = __ballot_sync(0xffffffffu, mover);
      if (pass == 1) {
        if (hole) holes[nh + __popc(bh & lower)] = j;
        if (mover) movers[nm + __popc(bm & lower)] = j;
      }
      nh += __popc(bh);
      nm += __popc(bm);
    }
    if (pass == 0) {
      if (lane == 0) hist[warp] = nh, hist[32 + warp] = nm;
      __syncthreads();
      uint32_t total = 0;
      for (int w = 0; w < 32; ++w) {
        if (w < warp) base_h += hist[w], base_m += hist[32 + w];
        total += hist[32 + w];
      }
      if (tid == 0) *count = (int)total;
      __syncthreads();
    }
  }
}

// A warp moves a token's K and V rows (and its weight and position): the
// list entry's two rows are found once per 32 entries, one per lane.
template <int D>
__global__ void __launch_bounds__(256) evict_move_kernel(const KvEvictArgs a, int list_cap) {
  constexpr int LPR = D * 2 / 16;         // lanes per row
  constexpr int TPW = 32 / (2 * LPR);     // tokens a warp moves at once (K and V rows)
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int h = blockIdx.y, req = blockIdx.z;
  const size_t head = (size_t)req * a.Hkv + h;
  const int m = a.ws[head];
  const int32_t *movers = a.ws + (size_t)a.R * a.Hkv + head * 2 * (size_t)list_cap, *holes = movers + list_cap;
  const int32_t *bt = a.block_table + (size_t)req * a.bt_stride;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int i0 = (blockIdx.x * 8 + warp) * 32; i0 < m; i0 += gridDim.x * 8 * 32) {
    long long src = -1, dst = -1;
    if (i0 + lane < m) {
      const int js = movers[i0 + lane], jd = holes[i0 + lane];
      const int cs = js / a.page_size, cd = jd / a.page_size;
      const int ps = bt[cs], pd = bt[cd];
      if (ps >= 0 && ps < a.num_pages && pd >= 0 && pd < a.num_pages) {  // bad pages: reported by the selection
        src = ((long long)ps * a.Hkv + h) * a.page_size + (js - cs * a.page_size);
        dst = ((long long)pd * a.Hkv + h) * a.page_size + (jd - cd * a.page_size);
        a.scores[dst] = a.scores[src];
        a.positions[dst] = a.positions[src];
      }
    }
    const int sub = lane / (2 * LPR), which = (lane / LPR) & 1, at = lane % LPR;
    const uint4 *in = static_cast<const uint4 *>(which ? a.v_cache : a.k_cache);
    uint4 *out = static_cast<uint4 *>(which ? a.v_cache : a.k_cache);
    const int cnt = min(32, m - i0);
    for (int i = 0; i < cnt; i += 4 * TPW) {
      uint4 v[4];
      long long to[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = i + u * TPW + sub;
        const long long s = __shfl_sync(0xffffffffu, src, e & 31);
        to[u] = __shfl_sync(0xffffffffu, dst, e & 31);
        if (e >= cnt) to[u] = -1;
        if (to[u] >= 0) v[u] = in[s * LPR + at];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (to[u] >= 0) out[to[u] * LPR + at] = v[u];
    }
  }
}

constexpr int kKeySmem = 40 * 1024;  // keys kept in shared memory (160 KB); longer contexts keep them in the workspace

}  // namespace kvb

static inline int launched() { return cudaPeekAtLastError() == cudaSuccess ? 0 : -4; }
static inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

extern "C" int sched_qk_norm_rope_kv_append(const QkNormArgs *args, cudaStream_t st) {
  if (args == nullptr) return -1;
  const QkNormArgs &a = *args;
  if (a.T <= 0) return 0;
  const int nheads = a.Hq + 2 * a.Hkv;
  if (a.Hq < 1 || a.Hkv < 1 || a.page_size < 1 || a.num_pages < 1 || a.max_pos < 1) return -1;
  if ((a.D != 64 && a.D != 128) || a.rot < 16 || a.rot > a.D || a.rot % 16 != 0) return -1;
  if (a.ld_qkv % 8 != 0 || a.ld_q % 8 != 0) return -1;
  if (!aligned16(a.qkv) || !aligned16(a.wq) || !aligned16(a.wk) || !aligned16(a.cos_sin) || !aligned16(a.q_out) ||
      !aligned16(a.k_cache) || !aligned16(a.v_cache))
    return -1;
  const long long threads = (long long)a.T * nheads * (a.D / 16);
  const long long grid = (threads + 255) / 256;
  if (grid > 0x7fffffffll) return -1;
  auto *k = a.element == kKvFp16 ? (a.D == 128 ? kvb::qk_norm_kernel<__half, 128> : kvb::qk_norm_kernel<__half, 64>)
                                 : (a.D == 128 ? kvb::qk_norm_kernel<__nv_bfloat16, 128>
                                               : kvb::qk_norm_kernel<__nv_bfloat16, 64>);
  launch_pdl(k, dim3((unsigned)grid), dim3(256), 0, st, a);
  return launched();
}

extern "C" long long sched_attn_scored_ws_floats(int R, int Q, int Hq, int Hkv, int D, int max_len, int num_sms) {
  if (R <= 0 || Q <= 0 || Hkv <= 0 || Hq < Hkv || max_len <= 0) return 0;
  return kvb::scored_plan(R, Q, Hq, Hkv, D, max_len, num_sms).total;
}

namespace kvb {
template <typename T, int D>
int run_scored(const ScoredArgs &a, const ScoredPlan &pl, cudaStream_t st) {
  auto *split = pl.block == 8 ? scored_split_kernel<T, D, 8> : scored_split_kernel<T, D, 16>;
  launch_pdl(split, dim3(pl.grid), dim3(kWarps * 32), 0, st, a, pl);
  if (cudaPeekAtLastError() != cudaSuccess) return -4;
  const int o_ctas = (pl.rows + kJoinRows - 1) / kJoinRows;
  launch_pdl(scored_join_kernel<T, D>, dim3(o_ctas + (a.max_len + pl.join - 1) / pl.join, a.Hkv, a.R),
             dim3(kJoin), (size_t)(pl.rows + 4 * kJoin) * sizeof(float), st, a, pl, o_ctas);
  return launched();
}
}  // namespace kvb

extern "C" int sched_attn_scored(const ScoredArgs *args, cudaStream_t st) {
  if (args == nullptr) return -1;
  const ScoredArgs &a = *args;
  if (a.R <= 0 || a.Q <= 0) return 0;
  if (a.Hkv < 1 || a.Hq < a.Hkv || a.Hq % a.Hkv != 0 || (a.D != 64 && a.D != 128)) return -1;
  if (a.page_size < 16 || a.page_size % 16 != 0 || a.num_pages < 1 || a.max_len < 1 || a.bt_pages < 1) return -1;
  if (a.R > 65535 || a.Hkv > 65535 || (long long)a.Q * (a.Hq / a.Hkv) > 8192) return -1;
  if (a.q_req % 8 != 0 || a.q_query % 8 != 0 || !aligned16(a.q) || !aligned16(a.k_cache) || !aligned16(a.v_cache) ||
      !aligned16(a.scores) || !aligned16(a.ws))
    return -1;
  const kvb::ScoredPlan pl = kvb::scored_plan(a.R, a.Q, a.Hq, a.Hkv, a.D, a.max_len, a.num_sms);
  // the tile list is indexed in 32 bits (2^31 tiles are 2^35 cached tokens and heads)
  if ((long long)a.R * a.Hkv * pl.blocks * (pl.lp / kvb::kTile) > 0x7fffffffll) return -1;
  if (a.ws == nullptr || a.ws_floats < pl.total) return -2;
  if (a.element == kKvFp16)
    return a.D == 128 ? kvb::run_scored<__half, 128>(a, pl, st) : kvb::run_scored<__half, 64>(a, pl, st);
  return a.D == 128 ? kvb::run_scored<__nv_bfloat16, 128>(a, pl, st) : kvb::run_scored<__nv_bfloat16, 64>(a, pl, st);
}

// [R * Hkv] counts, [R * Hkv][2][list] mover and hole slots, and the keys of
// contexts that shared memory does not hold
extern "C" long long sched_kv_evict_ws_ints(int R, int Hkv, int max_len, int budget) {
  if (R <= 0 || Hkv <= 0 || max_len <= budget) return 0;
  const long long heads = (long long)R * Hkv;
  const long long list = budget < max_len - budget ? budget : max_len - budget;
  return heads * (1 + 2 * list + (max_len > kvb::kKeySmem ? max_len : 0));
}

extern "C" int sched_kv_evict(const KvEvictArgs *args, cudaStream_t st) {
  if (args == nullptr) return -1;
  const KvEvictArgs &a = *args;
  if (a.R <= 0) return 0;
  if (a.Hkv < 1 || (a.D != 64 && a.D != 128) || a.page_size < 1 || a.num_pages < 1 || a.bt_pages < 1) return -1;
  if (a.budget < 1 || a.recent < 0 || a.sink < 0 || (long long)a.recent + a.sink > a.budget || a.max_len < 1) return -1;
  if (a.R > 65535 || a.Hkv > 65535 || !aligned16(a.k_cache) || !aligned16(a.v_cache)) return -1;
  const int list = a.budget < a.max_len - a.budget ? a.budget : a.max_len - a.budget;
  const long long need = sched_kv_evict_ws_ints(a.R, a.Hkv, a.max_len, a.budget);
  if (need > 0 && (a.ws == nullptr || a.ws_ints < need)) return -2;
  const long long heads = (long long)a.R * a.Hkv;
  int32_t *keys = a.max_len > kvb::kKeySmem ? a.ws + heads * (1 + 2ll * list) : nullptr;
  const size_t smem = keys == nullptr ? (size_t)a.max_len * 4 : 0;
  if (smem + sizeof(uint32_t) * (kvb::kSelBins + 64) > 48 * 1024 &&
      cudaFuncSetAttribute(kvb::evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kvb::kKeySmem * 4) !=
          cudaSuccess)
    return -4;
  launch_pdl(kvb::evict_select_kernel, dim3(a.Hkv, a.R), dim3(kvb::kSelThreads), smem, st, a, list, keys);
  if (cudaPeekAtLastError() != cudaSuccess) return -4;
  if (a.max_len <= a.budget) return 0;
  int x = (list + 255) / 256;
  const long long want = (4ll * a.num_sms + heads - 1) / heads;
  if (x > want) x = (int)want;
  auto *mv = a.D == 128 ? kvb::evict_move_kernel<128> : kvb::evict_move_kernel<64>;
  launch_pdl(mv, dim3(x < 1 ? 1 : x, a.Hkv, a.R), dim3(256), 0, st, a, list);
  return launched();
}
