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
// The tokens of a request are cut into chunks, a CTA each; a second kernel
// joins the chunks' partial results and adds the weights.
constexpr int kWarps = 4;      // per CTA of the split kernel
constexpr int kTile = 16;      // tokens per warp step: divides the page size

struct ScoredPlan {
  int rows, lp, chunk, nch;  // query rows per KV head, padded length, tokens per chunk, chunks
  long long s_off, o_off, ml_off, total;
};

// Chunks of up to 512 tokens; shorter while the grid would leave SMs idle.
inline ScoredPlan scored_plan(int R, int Q, int Hq, int Hkv, int D, int max_len, int num_sms) {
  ScoredPlan p;
  p.rows = Q * (Hq / Hkv);
  p.lp = (max_len + kTile - 1) / kTile * kTile;
  const long long blocks = (long long)R * Hkv * ((p.rows + 15) / 16);
  p.chunk = 512;
  while (p.chunk > kWarps * kTile && blocks * ((max_len + p.chunk - 1) / p.chunk) < 4ll * num_sms) p.chunk /= 2;
  p.nch = (max_len + p.chunk - 1) / p.chunk;
  const long long heads = (long long)R * Hkv;
  p.s_off = 0;
  p.o_off = heads * p.rows * p.lp;
  p.ml_off = p.o_off + heads * p.nch * p.rows * D;
  p.total = p.ml_off + heads * p.nch * p.rows * 2;
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

// exp2(m - ref) with m = -inf or an empty row's ref = -inf giving 0
__device__ __forceinline__ float scale_to(float m, float ref) { return ref == -INFINITY ? 0.f : ex2_approx(m - ref); }

// o += P V for one tile: this lane's V values of tokens 2c, 2c+1, 8+2c, 9+2c
// (vt[i][.]), D in 64-value halves i. ROWS 8: rows 8-15 of the product are
// not used. The column n of product (i, e) is value 64 i + 8 n + e of the
// head, so that a lane's 16 bytes of V feed eight products.
template <typename T, int D, int ROWS>
__device__ __forceinline__ void add_pv(float (&o)[D / 8][ROWS / 4], const uint4 (&vt)[D / 64][4], uint32_t a0, uint32_t a1,
                                       uint32_t a2, uint32_t a3) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const uint32_t t0[4] = {vt[i][0].x, vt[i][0].y, vt[i][0].z, vt[i][0].w};
    const uint32_t t1[4] = {vt[i][1].x, vt[i][1].y, vt[i][1].z, vt[i][1].w};
    const uint32_t t2[4] = {vt[i][2].x, vt[i][2].y, vt[i][2].z, vt[i][2].w};
    const uint32_t t3[4] = {vt[i][3].x, vt[i][3].y, vt[i][3].z, vt[i][3].w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
      const uint32_t b0 = __byte_perm(t0[e / 2], t1[e / 2], sel), b1 = __byte_perm(t2[e / 2], t3[e / 2], sel);
      float(&acc)[ROWS / 4] = o[i * 8 + e];
      if constexpr (ROWS == 16) {
        mma16816<T>(acc[0], acc[1], acc[2], acc[3], a0, a1, a2, a3, b0, b1);
      } else {
        float z0 = 0.f, z1 = 0.f;
        mma16816<T>(acc[0], acc[1], z0, z1, a0, 0u, a2, 0u, b0, b1);
      }
    }
  }
}

__device__ __forceinline__ uint4 keep_if(bool k, const uint4 &v) { return k ? v : make_uint4(0, 0, 0, 0); }

// One CTA: a chunk of one request's tokens for one KV head and ROWS of its
// query rows. Each warp takes every fourth 16-token tile and keeps its own
// running maximum, sum and output; K and V go from global memory straight
// into the registers of the m16n8k16 operands (the next tile's loads are in
// flight while this one is used), so there is no shared-memory staging.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kWarps * 32) scored_split_kernel(const ScoredArgs a, const ScoredPlan pl, int blocks) {
  constexpr int NK = D / 32;
  extern __shared__ float sm[];
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int req = blockIdx.z, h = blockIdx.y;
  const int ch = blockIdx.x / blocks, rb = blockIdx.x % blocks;
  const int cap = min(a.max_len, (int)min((long long)a.bt_pages * a.page_size, 0x7fffffffll));
  const int n = checked_len(a.kv_lens[req], cap, a.status, kSiteScoredLen, blockIdx.x == 0 && h == 0 && threadIdx.x == 0);
  const int t0 = ch * pl.chunk;
  if (t0 >= n) return;
  const int t1 = min(n, t0 + pl.chunk);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = lane / 4, c = lane % 4;
  const int G = a.Hq / a.Hkv, row0 = rb * ROWS;
  const int n_rows = min(ROWS, pl.rows - row0);

  // this lane's query rows r and r + 8: operand registers and token limits
  uint4 qx[ROWS / 8][NK];
  int lim[ROWS / 8];
#pragma unroll
  for (int i = 0; i < ROWS / 8; ++i) {
    const int row = row0 + r + 8 * i;
    lim[i] = 0;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) qx[i][kk] = make_uint4(0, 0, 0, 0);
    if (row < pl.rows) {
      const int qi = row / G, g = row - qi * G;
      lim[i] = n - (a.Q - 1 - qi);
      const T *src = static_cast<const T *>(a.q) + (size_t)req * a.q_req + (size_t)qi * a.q_query +
                     (size_t)(h * G + g) * D + c * 8;
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) qx[i][kk] = *reinterpret_cast<const uint4 *>(src + kk * 32);
    }
  }
  // tokens below all_see are seen by every row of this block
  const int all_see = n - (a.Q - 1 - row0 / G);
  const float scale2 = a.sm_scale * kLog2e;
  const int32_t *bt = a.block_table + (size_t)req * a.bt_stride;
  float *s_out = a.ws + pl.s_off + ((size_t)req * a.Hkv + h) * pl.rows * pl.lp;

  float o[D / 8][ROWS / 4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int j = 0; j < ROWS / 4; ++j) o[i][j] = 0.f;
  float m[ROWS / 8], sum[ROWS / 8];
#pragma unroll
  for (int i = 0; i < ROWS / 8; ++i) m[i] = -INFINITY, sum[i] = 0.f;

  // first element of a tile's K rows, or a negative number for a bad page
  auto tile_row = [&](int tok) -> long long {
    const int col = tok / a.page_size;
    const int page = bt[col];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0 && rb == 0) report_bad_index(a.status, kSiteScoredPage, page);
      return -1;
    }
    return (((long long)page * a.Hkv + h) * a.page_size + (tok - col * a.page_size)) * D;
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
    const T *p = static_cast<const T *>(a.v_cache) + (base < 0 ? 0 : base) + r * 8;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      vx[i][0] = ld_stream(p + (2 * c) * D + i * 64);
      vx[i][1] = ld_stream(p + (2 * c + 1) * D + i * 64);
      vx[i][2] = ld_stream(p + (2 * c + 8) * D + i * 64);
      vx[i][3] = ld_stream(p + (2 * c + 9) * D + i * 64);
    }
  };

  int tok = t0 + warp * kTile;
  long long base = -1;
  if (tok < t1) {
    base = tile_row(tok);
    load_k(base);
    load_v(base);
  }
  for (; tok < t1; tok += kWarps * kTile) {
    const int next = tok + kWarps * kTile;
    const long long next_base = next < t1 ? tile_row(next) : -1;
    float s[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        const uint4 q0 = qx[0][kk], q1 = ROWS == 16 ? qx[ROWS / 8 - 1][kk] : make_uint4(0, 0, 0, 0);
        mma16816<T>(s[j][0], s[j][1], s[j][2], s[j][3], q0.x, q1.x, q0.y, q1.y, kx[j][kk].x, kx[j][kk].y);
        mma16816<T>(s[j][0], s[j][1], s[j][2], s[j][3], q0.z, q1.z, q0.w, q1.w, kx[j][kk].z, kx[j][kk].w);
      }
    }
    if (next < t1) load_k(next_base);
    // tokens from `end` on are not there (behind the request's end, or their page is bad)
    const int end = base < 0 ? tok : n;
    const bool whole = tok + kTile <= min(end, all_see);
    uint32_t pa[2][2] = {{0u, 0u}, {0u, 0u}};  // [row block][tile half]: P as the product's A operand
#pragma unroll
    for (int i = 0; i < ROWS / 8; ++i) {
      float v[4] = {s[0][2 * i] * scale2, s[0][2 * i + 1] * scale2, s[1][2 * i] * scale2, s[1][2 * i + 1] * scale2};
      if (!whole) {
        const int seen = min(end, lim[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (tok + (j / 2) * 8 + 2 * c + (j & 1) >= seen) v[j] = -INFINITY;
      }
      const int row = row0 + r + 8 * i;
      if (row < pl.rows) {
        float *dst = s_out + (size_t)row * pl.lp + tok + 2 * c;
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
      const bool k0 = tok + 2 * c < end, k1 = tok + 2 * c + 1 < end, k2 = tok + 2 * c + 8 < end, k3 = tok + 2 * c + 9 < end;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        vx[i][0] = keep_if(k0, vx[i][0]);
        vx[i][1] = keep_if(k1, vx[i][1]);
        vx[i][2] = keep_if(k2, vx[i][2]);
        vx[i][3] = keep_if(k3, vx[i][3]);
      }
    }
    bool apart = false;
    if (a.Q > 1 && tok + kTile > all_see) {
      // tokens that only the later queries see: if one holds an infinity or
      // a NaN, the queries are added one at a time, each without the tokens
      // that it does not see
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
      add_pv<T, D, ROWS>(o, vx, pa[0][0], pa[1][0], pa[0][1], pa[1][1]);
    } else {
      for (int qi = row0 / G; qi <= (row0 + n_rows - 1) / G; ++qi) {
        const int seen = min(end, n - (a.Q - 1 - qi));
        uint4 vq[D / 64][4];
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) vq[i][j] = keep_if(tok + (j / 2) * 8 + 2 * c + (j & 1) < seen, vx[i][j]);
        const bool mine0 = (row0 + r) / G == qi, mine1 = (row0 + r + 8) / G == qi;
        // rows of the other queries: 0 * NaN again, so their sums are put back
        float old[D / 8][ROWS / 4];
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
#pragma unroll
          for (int j = 0; j < ROWS / 4; ++j) old[d][j] = o[d][j];
        add_pv<T, D, ROWS>(o, vq, pa[0][0], pa[1][0], pa[0][1], pa[1][1]);
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
#pragma unroll
          for (int j = 0; j < ROWS / 4; ++j)
            if (!(j < 2 ? mine0 : mine1)) o[d][j] = old[d][j];
      }
    }
    if (next < t1) load_v(next_base);
    base = next_base;
  }
#pragma unroll
  for (int i = 0; i < ROWS / 8; ++i) {
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
  }

  // join the warps: shared memory holds [warp][ROWS] (max, sum) and [warp][ROWS][D]
  float2 *ml = reinterpret_cast<float2 *>(sm);
  float *os = sm + 2 * kWarps * ROWS;
#pragma unroll
  for (int i = 0; i < ROWS / 8; ++i) {
    if (c == 0) ml[warp * ROWS + r + 8 * i] = make_float2(m[i], sum[i]);
    float *dst = os + ((size_t)warp * ROWS + r + 8 * i) * D;
#pragma unroll
    for (int d = 0; d < D / 8; ++d) {
      dst[(d / 8) * 64 + 16 * c + d % 8] = o[d][2 * i];
      dst[(d / 8) * 64 + 16 * c + 8 + d % 8] = o[d][2 * i + 1];
    }
  }
  __syncthreads();
  const size_t part = ((size_t)req * a.Hkv + h) * pl.nch + ch;
  for (int x = threadIdx.x; x < n_rows * D; x += kWarps * 32) {
    const int row = x / D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * ROWS + row].x);
    float v = 0.f, tot = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = scale_to(ml[w * ROWS + row].x, top);
      v += os[((size_t)w * ROWS + row) * D + x % D] * f;
      tot += ml[w * ROWS + row].y * f;
    }
    const size_t at = part * pl.rows + row0 + row;
    a.ws[pl.o_off + at * D + x % D] = v;
    if (x % D == 0) reinterpret_cast<float2 *>(a.ws + pl.ml_off)[at] = make_float2(top, tot);
  }
}

__device__ __forceinline__ void red_add4(float *p, const float4 &v) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

// Join: every CTA of a request and KV head derives the rows' lse from the
// chunks' (max, sum); each joins the outputs of some rows and adds the weights
// of its own chunk's tokens. Rows are summed in a fixed order, and one
// request's pages get one addition per token and head from a call.
template <typename T, int D>
__global__ void __launch_bounds__(256) scored_join_kernel(const ScoredArgs a, const ScoredPlan pl) {
  extern __shared__ float sm[];
  float *lse2 = sm;                 // [rows]: log2 of the sum; +inf for a row that sees nothing
  float *part_o = sm + pl.rows;     // [256]
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const int req = blockIdx.z, h = blockIdx.y, ch = blockIdx.x;
  const int cap = min(a.max_len, (int)min((long long)a.bt_pages * a.page_size, 0x7fffffffll));
  const int n = checked_len(a.kv_lens[req], cap, nullptr, 0, false);
  const int nce = (n + pl.chunk - 1) / pl.chunk;
  if (ch >= max(nce, 1)) return;
  const int G = a.Hq / a.Hkv;
  const size_t part = ((size_t)req * a.Hkv + h) * pl.nch;
  const float2 *ml = reinterpret_cast<const float2 *>(a.ws + pl.ml_off) + part * pl.rows;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int row = warp; row < pl.rows; row += 8) {
    float top = -INFINITY, tot = 0.f;
    for (int k = lane; k < nce; k += 32) {
      const float2 v = ml[(size_t)k * pl.rows + row];
      const float t = fmaxf(top, v.x);
      tot = tot * scale_to(top, t) + v.y * scale_to(v.x, t);
      top = t;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ot = __shfl_xor_sync(0xffffffffu, top, o), os = __shfl_xor_sync(0xffffffffu, tot, o);
      const float t = fmaxf(top, ot);
      tot = tot * scale_to(top, t) + os * scale_to(ot, t);
      top = t;
    }
    if (lane == 0) {
      const float v = top == -INFINITY && tot == 0.f ? -INFINITY : top + log2f(tot);  // NaN logits stay NaN
      lse2[row] = v == -INFINITY ? INFINITY : v;
      if (ch == 0 && a.lse != nullptr) {
        const int qi = row / G;
        a.lse[((size_t)req * a.Q + qi) * a.Hq + h * G + (row - qi * G)] = v * kLn2;
      }
    }
  }
  __syncthreads();
  const float *o_in = a.ws + pl.o_off + part * pl.rows * D;
  constexpr int GR = 256 / D;
  const int grp = threadIdx.x / D, d = threadIdx.x % D;
  for (int row = ch; row < pl.rows; row += max(nce, 1)) {
    const float ref = lse2[row];
    float v = 0.f;
#pragma unroll 4
    for (int k = grp; k < nce; k += GR) {
      const float f = ex2_approx(ml[(size_t)k * pl.rows + row].x - ref);
      if (f != 0.f) v += o_in[((size_t)k * pl.rows + row) * D + d] * f;
    }
    part_o[threadIdx.x] = v;
    __syncthreads();
    if (grp == 0) {
#pragma unroll
      for (int k = 1; k < GR; ++k) v += part_o[k * D + d];
      const int qi = row / G;
      static_cast<T *>(a.out)[(size_t)req * a.out_req + (size_t)qi * a.out_query + (size_t)(h * G + row - qi * G) * D + d] =
          narrow<T>(v);
    }
    __syncthreads();
  }
  const int t0 = ch * pl.chunk, t1 = min(n, t0 + pl.chunk);
  const float *s_in = a.ws + pl.s_off + ((size_t)req * a.Hkv + h) * pl.rows * pl.lp;
  const int32_t *bt = a.block_table + (size_t)req * a.bt_stride;
  for (int tok = t0 + threadIdx.x * 4; tok < t1; tok += 1024) {
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int row = 0; row < pl.rows; ++row) {
      const float4 s = *reinterpret_cast<const float4 *>(s_in + (size_t)row * pl.lp + tok);
      const float ref = lse2[row];
      w.x += ex2_approx(s.x - ref);
      w.y += ex2_approx(s.y - ref);
      w.z += ex2_approx(s.z - ref);
      w.w += ex2_approx(s.w - ref);
    }
    const int col = tok / a.page_size, page = bt[col];
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
  const bool small = pl.rows <= 8;
  const int per = small ? 8 : 16, blocks = (pl.rows + per - 1) / per;
  const size_t smem = (size_t)kWarps * per * (D + 2) * sizeof(float);
  const long long gx = (long long)pl.nch * blocks;
  if (gx > 0x7fffffffll) return -1;
  auto *split = small ? scored_split_kernel<T, D, 8> : scored_split_kernel<T, D, 16>;
  launch_pdl(split, dim3((unsigned)gx, a.Hkv, a.R), dim3(kWarps * 32), smem, st, a, pl, blocks);
  if (cudaPeekAtLastError() != cudaSuccess) return -4;
  launch_pdl(scored_join_kernel<T, D>, dim3(pl.nch, a.Hkv, a.R), dim3(256), (size_t)(pl.rows + 256) * sizeof(float), st,
             a, pl);
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
