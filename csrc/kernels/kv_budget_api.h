// kv_budget_api.h -- launchers of the kernels that keep a paged KV cache to a
// budget (kv_budget.cu). Plain C structs: no torch, usable from any host.
//
// The launchers return 0, -1 for arguments that they refuse (nothing is
// launched), -2 for scratch that is missing or too small, -4 where the launch
// failed. Pointers not marked "or null" must be there; qkv, the weights,
// cos_sin, q, out, the caches, the scores of the attention, and scratch start
// on 16-byte boundaries, and pitches of q, out and qkv are multiples of 8
// elements. That a pointer's memory is as large as its comment says, and on
// the device, is the caller's part.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

enum KvElement : int { kKvBf16 = 0, kKvFp16 = 1 };

// Per-head RMSNorm of q and k, rotation, and append to the paged cache.
struct QkNormArgs {
  const void *qkv;      // [T] rows of (Hq + 2 Hkv) heads of D, row pitch ld_qkv elements
  long long ld_qkv;
  const void *wq, *wk;  // [D] norm weights
  float eps;
  const int32_t *pos;   // [T]
  const int32_t *slot;  // [T] page * page_size + offset, < 0: no cache write
  const float *cos_sin; // [max_pos, rot / 2, 2]
  int max_pos, rot;
  void *q_out;          // [T] rows of Hq heads, row pitch ld_q elements
  long long ld_q;
  void *k_cache, *v_cache;  // [num_pages, Hkv, page_size, D]
  float *scores;            // [num_pages, Hkv, page_size] or null: set to 0 at the new slots
  int32_t *positions;       // the same shape or null: set to the position
  int T, Hq, Hkv, D, page_size, num_pages, element, num_sms;
  int *status;  // 4 words or null
};
extern "C" int sched_qk_norm_rope_kv_append(const QkNormArgs *args, cudaStream_t st);

// Decode attention that adds every cached token's attention weight to scores.
struct ScoredArgs {
  const void *q;  // [R, Q, Hq, D]: heads contiguous, request and query pitches in elements
  long long q_req, q_query;
  void *out;
  long long out_req, out_query;
  float *lse;  // [R, Q, Hq] or null
  const void *k_cache, *v_cache;
  float *scores;  // [num_pages, Hkv, page_size]
  const int32_t *block_table;
  long long bt_stride;
  int bt_pages;  // columns of the block table
  const int32_t *kv_lens;
  int R, Q, Hq, Hkv, D, page_size, num_pages, max_len, element, num_sms;
  float sm_scale;
  float *ws;  // sched_attn_scored_ws_floats() floats (none for the one-kernel form)
  long long ws_floats;
  int *status;  // 4 words or null
};
extern "C" long long sched_attn_scored_ws_floats(int R, int Q, int Hq, int Hkv, int D, int max_len, int num_sms);
extern "C" int sched_attn_scored(const ScoredArgs *args, cudaStream_t st);

// Eviction of the cached tokens with the least accumulated weight.
struct KvEvictArgs {
  void *k_cache, *v_cache;
  float *scores;
  int32_t *positions;
  const int32_t *block_table;
  long long bt_stride;
  int bt_pages;
  const int32_t *kv_lens, *last_pos;  // [R]
  int32_t *new_lens;                  // [R], apart from kv_lens and last_pos
  int R, Hkv, D, page_size, num_pages, max_len, budget, recent, sink, num_sms;
  int32_t *ws;  // sched_kv_evict_ws_ints() words
  long long ws_ints;
  int *status;  // 4 words or null
};
extern "C" long long sched_kv_evict_ws_ints(int R, int Hkv, int max_len, int budget, int num_sms);
extern "C" int sched_kv_evict(const KvEvictArgs *args, cudaStream_t st);
