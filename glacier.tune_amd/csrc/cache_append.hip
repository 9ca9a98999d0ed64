// cache_append.hip -- new tokens' keys (rotated) and values into a paged
// cache, and their queries rotated, in one launch.
//
// HBM-bound: each row is read once and written once, whole.  A wave takes one
// token, or a share of its heads when there are few tokens; queries, keys and
// values follow each other as heads of that token (turn.hpp).  The token's
// sequence is found by all lanes at once (one load deep up to 64: a binary search would
// chain one per halving), and the first rows are requested before it, since
// only where they go depends on it.
//
// Measured: 16 chunks of up to 512 tokens, 32/8 heads of 128, bf16, 23.1 us (5.7
// TB/s: the rows were written shortly before and are partly in the last-level
// cache), fp32 50.9 (5.5); keys and values alone, as they are, 8.0 and 17.2 (5.1, 5.5);
// 64 sequences of one token 3.4 us in a replayed graph, the launch (3.1 unrotated).
#include "cache_view.hpp"
#include "turn.hpp"

namespace glacier {
namespace {

constexpr int kWavesAp = 4;

template <typename IO, int E, int L>
__global__ __launch_bounds__(64 * kWavesAp) void cache_append_kernel(CacheAppend a, TurnRates rates) {
  constexpr int H = 64 / L;  // heads per step
  __shared__ float2 turns[kWavesAp][kTurnMaxDim / 2];
  const CacheView& c = a.c;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int unit = blockIdx.x * kWavesAp + wave;
  const int t = unit / a.parts, part = unit % a.parts;
  if (t >= c.T) return;
  const int half = c.D / 2, heads = a.hq + 2 * c.hkv;
  const int col = (lane % L) * E;
  const bool in_row = col < half;
  Piece<IO, E> p0, p1;
  // the row of head h (queries, then keys, then values) at this lane's column
  auto fetch = [&](int h) {
    if (!in_row || h >= heads) return;
    const IO* x;
    if (h < a.hq)
      x = static_cast<const IO*>(a.q) + ((long)t * a.hq + h) * c.D;
    else if (h < a.hq + c.hkv)
      x = static_cast<const IO*>(a.k) + ((long)t * c.hkv + (h - a.hq)) * c.D;
    else
      x = static_cast<const IO*>(a.v) + ((long)t * c.hkv + (h - a.hq - c.hkv)) * c.D;
    p0.load(x + col);
    p1.load(x + half + col);
  };
  fetch(part * H + lane / L);
  const CacheSeq s = seq_of_token(c, lane, t);
  if (s.b >= c.n_seqs) return;  // behind the last sequence
  if (t < s.tok0) return;
  const int pos = s.pos0 + (t - s.tok0);
  const int page = cache_page(c, s.b, pos);
  const int row = pos & ((1 << c.page_shift) - 1);
  if (a.rotate) turn_table(turns[wave], LaneRates(rates, half, lane), half, pos, lane);
  for (int h0 = part * H; h0 < heads; h0 += a.parts * H) {
    const int h = h0 + lane / L;
    if (h0 != part * H) fetch(h);
    if (!in_row || h >= heads) continue;
    IO* to;
    if (h < a.hq) {
      to = static_cast<IO*>(a.q_rot) + ((long)t * a.hq + h) * c.D;
    } else {
      if (page < 0) continue;
      const bool is_v = h >= a.hq + c.hkv;
      const int kv = h - a.hq - (is_v ? c.hkv : 0);
      to = static_cast<IO*>(is_v ? c.v_pages : c.k_pages) + page * c.page_stride +
           (((long)kv << c.page_shift) + row) * c.D;
    }
    if (a.rotate && h < a.hq + c.hkv) {
      float x0[E], x1[E];
      p0.get(x0);
      p1.get(x1);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float2 cs = turns[wave][col + e];
        rope_fwd(x0[e], x1[e], cs.x, cs.y, x0[e], x1[e]);
      }
      p0.set(x0);
      p1.set(x1);
    }
    p0.store(to + col);
    p1.store(to + half + col);
  }
}

template <typename IO, int E, int L>
hipError_t append(CacheAppend& a, const TurnRates& r, int n_cu, hipStream_t st) {
  a.parts = turn_parts(a.c.T, (a.hq + 2 * a.c.hkv + 64 / L - 1) / (64 / L), n_cu);
  const long units = (long)a.c.T * a.parts;
  hipLaunchKernelGGL((cache_append_kernel<IO, E, L>), dim3((units + kWavesAp - 1) / kWavesAp),
                     dim3(64 * kWavesAp), 0, st, a, r);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_append(CacheAppend a, const TurnRates& r, int n_cu, hipStream_t st) {
  GL_BY_HEAD(append, a.c.io_bf16, a.c.D, a, r, n_cu, st);
}

}  // namespace glacier
