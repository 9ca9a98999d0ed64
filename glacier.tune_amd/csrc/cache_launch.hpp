// cache_launch.hpp -- host-side interface of qk_norm.hip (per-head norms of
// queries and keys with the rotation), cache_append.hip and cache_attn.hip
// (the paged cache) for engine.cpp.
#pragma once

#include <hip/hip_runtime.h>

#include "attn_launch.hpp"

namespace glacier {

constexpr int kTurnMaxDim = 256;  // largest head_dim of these kernels

// Revolutions per position of each rotation pair, theta^(-2i/D) / (2 pi).  The
// table goes to a kernel by value: 1 KB of arguments instead of an upload, so
// that a call allocates nothing and can be captured.
struct TurnRates {
  double rev[kTurnMaxDim / 2];
};

// ---- per-head norms of queries and keys (qk_norm.hip) ----------------------
constexpr int kQkMaxGroups = 512;  // workgroups of a backward, each with its partial sums

struct QkNorm {
  int T, hq, hkv, D;
  float eps;
  bool io_bf16, rotate;
  const void *q, *k;            // forward inputs
  const void *dq_out, *dk_out;  // backward: upstream gradients
  const float *wq, *wk;
  const int32_t* positions;  // null: 0 .. T - 1
  void *yq, *yk;             // forward: outputs; backward: dq, dk
  float *dwq, *dwk;          // backward, or null
  float* partials;           // [groups][2 D] when dwq or dwk is given
  int parts;                 // waves that share a token's heads (set by the launch)
};
hipError_t launch_qk_norm_forward(QkNorm a, const TurnRates& r, int n_cu, hipStream_t st);
hipError_t launch_qk_norm_backward(QkNorm a, const TurnRates& r, int n_cu, hipStream_t st);

// ---- the paged cache -------------------------------------------------------
struct CacheView {
  void *k_pages, *v_pages;
  long page_stride;  // elements
  int n_pages, page_shift, hkv, D;
  bool io_bf16;
  const int32_t *cu, *kv_lens, *table;
  long table_stride;
  int n_seqs, T, max_pages;
};

struct CacheAppend {
  CacheView c;
  int hq;  // 0: no queries
  bool rotate;
  const void *k, *v, *q;
  void* q_rot;
  int parts;
};
hipError_t launch_cache_append(CacheAppend a, const TurnRates& r, int n_cu, hipStream_t st);

struct CacheAttn {
  CacheView c;
  int hq, group;
  float scale_log2;  // log2 e / sqrt(D)
  const void* q;
  void* out;
  float* lse;     // or null
  int rows;       // rows of a tile: the kernel variant
  bool long_first;  // tiles of long sequences come first
  int n_splits;   // key splits a tile may take (1: no workspace)
  int split_keys;  // keys of a split, unless a sequence needs more for n_splits of them
  float* part_o;  // [n_splits][T hq][D]
  float2* part_ml;  // [n_splits][T hq] running maximum (log2) and sum
};
// How a call is laid out, from what the host knows (cache_attn.hip).
struct CachePlan {
  int rows, n_splits, split_keys;
  bool long_first;
  size_t bytes;  // workspace
};
CachePlan cache_attn_plan(const CacheView& c, int hq, int max_new, int max_kv, int n_cu);
hipError_t launch_cache_attn(const CacheAttn& a, hipStream_t st);

constexpr int kCacheWideRows = 128;  // rows of a tile of cache_attn_wide.hip
constexpr int kCacheTileJoin = 8;     // up to so many splits it joins them itself, tile by tile;
constexpr int kCacheJoinRows = 2048;  // more, up to so many rows, go to a wave or four per row
hipError_t launch_cache_attn_wide(const CacheAttn& a, hipStream_t st);

}  // namespace glacier
