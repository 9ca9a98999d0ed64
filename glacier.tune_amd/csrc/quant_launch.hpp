// quant_launch.hpp -- host-side interface of qcache_append.hip, qcache_attn.hip (the
// paged cache in 4 bits) and proj_quant.hip (products with 4-bit weights) for
// engine.cpp.
#pragma once

#include "cache_launch.hpp"
#include "proj_launch.hpp"

namespace glacier {

// Groups of 32 columns that a head of D columns is held in.
constexpr int quant_groups(int D) {
  const int g = (D + 31) / 32;
  return g == 5 || g == 7 ? g + 1 : g;
}
// Bytes of one token's head in a page of K, or of V.
constexpr int quant_row_bytes(int D) { return 18 * quant_groups(D); }

// In the CacheView of these calls pages are bytes: page_stride counts bytes, and
// io_bf16 is the tensors' type.
hipError_t launch_qcache_append(CacheAppend a, const TurnRates& r, int n_cu, hipStream_t st);

struct QCacheRead {
  CacheView c;
  void *k, *v;
  int parts;  // set by the launch
};
hipError_t launch_qcache_read(QCacheRead a, int n_cu, hipStream_t st);

// How an attention call is laid out.
struct QCachePlan {
  bool expand;      // the pages' values into the workspace first, then cache_attn
  CachePlan attn;   // of the attention, after the expanded pages in the workspace
  size_t k_bytes;   // of expanded K (and of V), then of the page table
  size_t table_bytes;
  size_t bytes;     // workspace in all
};
QCachePlan qcache_attn_plan(const CacheView& c, int hq, int max_new, int max_kv, int n_cu);
// a.c: the 4-bit cache; a.rows, a.n_splits, ... from plan.attn.
hipError_t launch_qcache_attn(const CacheAttn& a, const QCachePlan& plan, void* workspace, hipStream_t st);

// Where the parts of packed weights begin (bytes).
struct QuantLayout {
  long tiles, blocks, scales, offsets, bytes;
};
constexpr QuantLayout quant_layout(long out, long in, int group, bool offsets) {
  QuantLayout l{};
  l.tiles = (out + 15) / 16;
  l.blocks = (in + 127) / 128;
  l.scales = l.tiles * l.blocks * 1024;
  l.offsets = l.scales + l.tiles * l.blocks * (4096 / group);
  l.bytes = l.offsets + (offsets ? l.tiles * l.blocks * (4096 / group) : 0);
  return l;
}
struct QuantPack {
  int out, in, group;
  const void *numbers, *scales, *offsets;  // offsets: or null
  void* packed;
};
hipError_t launch_quant_pack(const QuantPack& a, hipStream_t st);

// Parts in which x A_p is left for the products.
int quant_low_splits(int T, int in);
// a: x, T, in, rank, io_bf16 and the projections, w packed; low: [adapters][parts][T]
// [rank] for x A_p, or null without adapters; terms: bf16 [3][T][in] for fp32 x.
struct QuantProj {
  ProjLaunch a;
  int group;
  bool offsets;
  float* low;
  void* terms;
};
hipError_t launch_quant_proj(const QuantProj& q, int n_cu, hipStream_t st);

}  // namespace glacier
