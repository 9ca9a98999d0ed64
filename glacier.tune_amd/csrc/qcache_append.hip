// qcache_append.hip -- new tokens' keys (rotated) and values into a paged cache in 4
// bits, their queries rotated in the same launch; and tokens back from such pages.
//
// HBM-bound: each row is read once and written once.  A wave takes one token, or a
// share of its heads when there are few tokens.  A lane holds eight columns of a
// head, so a group of 32 is four neighbouring lanes: its largest element is found in
// two exchanges, and a lane's eight numbers are one word of the page.  Two steps' rows
// are in flight, the first from before the token's place is known, and the angles of a
// lane's columns stay in its registers.  5272 tokens of 32 query and 8 KV heads of 128
// (bf16): 30.7 us for 114 MB (3.7 TB/s; with the rows asked for step by step and the
// angles read from LDS 38), read back in 8.0.
//
// The rotation is formed in 64 bits: a key that fp32 rounding moves over the border
// between two numbers would be held a whole step off, so that the cache's contents
// would depend on how the angle was formed.  (q takes the same angles.)
#include "cache_view.hpp"
#include "quant_page.hpp"
#include "turn.hpp"

namespace glacier {
namespace {

constexpr int kWavesQa = 4;

// Angle of position pos and a pair's rate: cos and sin in 64 bits (turn.hpp's, whose
// results are rounded to 32).
__device__ inline double2 turn64(double rev, int pos) {
  double a = rev * (double)pos, s, c;
  a -= rint(a);
  sincospi(2.0 * a, &s, &c);
  return make_double2(c, s);
}

// Eight columns of a row as they are loaded, and the eight that they are rotated with.
template <typename IO>
struct Columns {
  Piece<IO, 4> own[2], other[2];
};

template <typename IO, int G>
__global__ __launch_bounds__(64 * kWavesQa) void qcache_append_kernel(CacheAppend a, TurnRates rates) {
  constexpr int L = 4 * G, H = 64 / L;  // lanes of a head, heads per step
  __shared__ double2 turns[kWavesQa][kTurnMaxDim / 2];
  const CacheView& c = a.c;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int unit = blockIdx.x * kWavesQa + wave;
  const int t = unit / a.parts, part = unit - t * a.parts;
  if (t >= c.T) return;
  const int half = c.D / 2, heads = a.hq + 2 * c.hkv, turned = a.hq + c.hkv;
  const int col8 = lane % L, slot = lane / L, col = 8 * col8;
  const bool in_row = slot < H && col < c.D;
  // (half is a multiple of 4: four columns have their partners together)
  const int at0 = in_row ? col : 0, at1 = at0 + 4;
  const int to0 = at0 < half ? at0 + half : at0 - half, to1 = at1 < half ? at1 + half : at1 - half;
  auto load = [&](Columns<IO>& to, int h0) __attribute__((always_inline)) {
    const int h = min(h0 + slot, heads - 1);
    const IO* const src = h < a.hq ? static_cast<const IO*>(a.q) + ((long)t * a.hq + h) * c.D
                          : h < turned ? static_cast<const IO*>(a.k) + ((long)t * c.hkv + (h - a.hq)) * c.D
                                       : static_cast<const IO*>(a.v) + ((long)t * c.hkv + (h - turned)) * c.D;
    to.own[0].load(src + at0), to.own[1].load(src + at1);
    if (a.rotate && h0 < turned) to.other[0].load(src + to0), to.other[1].load(src + to1);
  };
  // two steps' rows in flight, from before the search for the token's place
  const int first = part * H, stride = a.parts * H;
  Columns<IO> one, two;
  load(one, first);
  if (first + stride < heads) load(two, first + stride);
  const CacheSeq s = seq_of_token(c, lane, t);
  if (s.b >= c.n_seqs || t < s.tok0) return;  // behind the last sequence
  const int pos = s.pos0 + (t - s.tok0);
  const int page = cache_page(c, s.b, pos);
  const int row = pos & ((1 << c.page_shift) - 1);
  // the angles of this lane's columns, the same in every head
  double co[8], si[8];
  if (a.rotate) {
    double2* const turn = turns[wave];
    const int second = lane + 64;
    const double lo = rates.rev[lane < half ? lane : 0], hi = rates.rev[second < half ? second : 0];
    if (lane < half) turn[lane] = turn64(lo, pos);
    if (second < half) turn[second] = turn64(hi, pos);
    wave_lds_order();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = (e < 4 ? at0 : at1) + e % 4;
      const double2 cs = turn[at < half ? at : at - half];
      co[e] = cs.x, si[e] = at < half ? -cs.y : cs.y;
    }
  }
  const long part_bytes = (long)quant_row_bytes(c.D) << c.page_shift;
  auto take = [&](const Columns<IO>& from, int h0) __attribute__((always_inline)) {
    const int h = h0 + slot;
    const bool here = slot < H && h < heads, is_q = h < a.hq, is_k = !is_q && h < turned;
    float x[8];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      float own[4];
      from.own[p].get(own);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * p + e] = in_row ? own[e] : 0.0f;
    }
    if (a.rotate && h0 < turned) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float other[4];
        from.other[p].get(other);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * p + e;
          const float r = (float)fma((double)x[i], co[i], (double)other[e] * si[i]);
          x[i] = in_row && (is_q || is_k) ? r : x[i];
        }
      }
    }
    if (here && is_q && in_row) store8(static_cast<IO*>(a.q_rot) + ((long)t * a.hq + h) * c.D + col, x);
    if (h0 + H <= a.hq || page < 0) return;  // (the wave's heads are queries, or held nowhere)
    // (all lanes: a group's lanes exchange their largest elements)
    f16 scale;
    const unsigned w = quantise8(x, scale);
    if (!here || is_q) return;
    const int kv = h - (is_k ? a.hq : turned);
    char* const to = static_cast<char*>(is_k ? c.k_pages : c.v_pages) + page * c.page_stride + kv * part_bytes;
    f16* const scales = reinterpret_cast<f16*>(to + ((16L * G) << c.page_shift));
    reinterpret_cast<unsigned*>(to)[is_k ? k_word(row, G, col8) : v_word(row, G, col8)] = w;
    if (col8 % 4 == 0) scales[is_k ? k_scale(row, G, col8 / 4) : v_scale(row, G, col8 / 4)] = scale;
  };
  for (int h0 = first; h0 < heads; h0 += 2 * stride) {
    take(one, h0);
    if (h0 + stride >= heads) break;
    if (h0 + 2 * stride < heads) load(one, h0 + 2 * stride);
    take(two, h0 + stride);
    if (h0 + 3 * stride < heads) load(two, h0 + 3 * stride);
  }
}

template <typename IO, int G>
__global__ __launch_bounds__(64 * kWavesQa) void qcache_read_kernel(QCacheRead a) {
  constexpr int L = 4 * G, H = 64 / L;
  const CacheView& c = a.c;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int unit = blockIdx.x * kWavesQa + wave;
  const int t = unit / a.parts, part = unit % a.parts;
  if (t >= c.T) return;
  const CacheSeq s = seq_of_token(c, lane, t);
  if (s.b >= c.n_seqs || t < s.tok0) return;
  const int pos = s.pos0 + (t - s.tok0);
  const int page = cache_page(c, s.b, pos);
  const int row = pos & ((1 << c.page_shift) - 1);
  const int col8 = lane % L, slot = lane / L;
  if (slot >= H || 8 * col8 >= c.D) return;
  const long part_bytes = (long)quant_row_bytes(c.D) << c.page_shift;
  for (int h = part * H + slot; h < 2 * c.hkv; h += a.parts * H) {
    const bool is_k = h < c.hkv;
    const int kv = is_k ? h : h - c.hkv;
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (page >= 0) {
      const char* const from =
          static_cast<const char*>(is_k ? c.k_pages : c.v_pages) + page * c.page_stride + kv * part_bytes;
      const f16* const scales = reinterpret_cast<const f16*>(from + ((16L * G) << c.page_shift));
      const unsigned w = reinterpret_cast<const unsigned*>(from)[is_k ? k_word(row, G, col8) : v_word(row, G, col8)];
      dequantise8(w, (float)scales[is_k ? k_scale(row, G, col8 / 4) : v_scale(row, G, col8 / 4)], x);
    }
    store8(static_cast<IO*>(is_k ? a.k : a.v) + ((long)t * c.hkv + kv) * c.D + 8 * col8, x);
  }
}

template <typename IO, int G>
hipError_t append(CacheAppend& a, const TurnRates& r, int n_cu, hipStream_t st) {
  constexpr int H = 16 / G;
  a.parts = turn_parts(a.c.T, (a.hq + 2 * a.c.hkv + H - 1) / H, n_cu);
  const long units = (long)a.c.T * a.parts;
  hipLaunchKernelGGL((qcache_append_kernel<IO, G>), dim3((units + kWavesQa - 1) / kWavesQa), dim3(64 * kWavesQa), 0,
                     st, a, r);
  return hipGetLastError();
}
template <typename IO, int G>
hipError_t read(QCacheRead& a, int n_cu, hipStream_t st) {
  constexpr int H = 16 / G;
  a.parts = turn_parts(a.c.T, (2 * a.c.hkv + H - 1) / H, n_cu);
  const long units = (long)a.c.T * a.parts;
  hipLaunchKernelGGL((qcache_read_kernel<IO, G>), dim3((units + kWavesQa - 1) / kWavesQa), dim3(64 * kWavesQa), 0,
                     st, a);
  return hipGetLastError();
}

// F<IO, G> for the call's type and head size
#define GL_BY_GROUPS(F, ...)                                              \
  switch (quant_groups(a.c.D)) {                                          \
    case 1: return a.c.io_bf16 ? F<bf16, 1>(__VA_ARGS__) : F<float, 1>(__VA_ARGS__); \
    case 2: return a.c.io_bf16 ? F<bf16, 2>(__VA_ARGS__) : F<float, 2>(__VA_ARGS__); \
    case 3: return a.c.io_bf16 ? F<bf16, 3>(__VA_ARGS__) : F<float, 3>(__VA_ARGS__); \
    case 4: return a.c.io_bf16 ? F<bf16, 4>(__VA_ARGS__) : F<float, 4>(__VA_ARGS__); \
    case 6: return a.c.io_bf16 ? F<bf16, 6>(__VA_ARGS__) : F<float, 6>(__VA_ARGS__); \
    default: return a.c.io_bf16 ? F<bf16, 8>(__VA_ARGS__) : F<float, 8>(__VA_ARGS__); \
  }

}  // namespace

hipError_t launch_qcache_append(CacheAppend a, const TurnRates& r, int n_cu, hipStream_t st) {
  GL_BY_GROUPS(append, a, r, n_cu, st)
}
hipError_t launch_qcache_read(QCacheRead a, int n_cu, hipStream_t st) { GL_BY_GROUPS(read, a, n_cu, st) }

}  // namespace glacier
