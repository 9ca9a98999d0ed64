// qcache_append.hip -- new tokens' keys (rotated) and values into a paged cache in 4
// bits, their queries rotated in the same launch; and tokens back from such pages.
//
// HBM-bound: each row is read once and written once.  A wave takes one token, or a
// share of its heads when there are few tokens.  A lane holds eight columns of a
// head, so a group of 32 is four neighbouring lanes: its largest element is found in
// two exchanges, and a lane's eight numbers are one word of the page.
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

// Four elements at p as floats.
__device__ inline void load4f(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ inline void load4f(const bf16* p, float (&x)[4]) {
  const bf16x4 v = *reinterpret_cast<const bf16x4*>(p);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = (float)v[e];
}

// Angle of position pos and a pair's rate: cos and sin in 64 bits (turn.hpp's, whose
// results are rounded to 32).
__device__ inline double2 turn64(double rev, int pos) {
  double a = rev * (double)pos, s, c;
  a -= rint(a);
  sincospi(2.0 * a, &s, &c);
  return make_double2(c, s);
}

template <typename IO, int G>
__global__ __launch_bounds__(64 * kWavesQa) void qcache_append_kernel(CacheAppend a, TurnRates rates) {
  constexpr int L = 4 * G, H = 64 / L;  // lanes of a head, heads per step
  __shared__ double2 turns[kWavesQa][kTurnMaxDim / 2];
  const CacheView& c = a.c;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int unit = blockIdx.x * kWavesQa + wave;
  const int t = unit / a.parts, part = unit % a.parts;
  if (t >= c.T) return;
  const CacheSeq s = seq_of_token(c, lane, t);
  if (s.b >= c.n_seqs || t < s.tok0) return;  // behind the last sequence
  const int pos = s.pos0 + (t - s.tok0);
  const int page = cache_page(c, s.b, pos);
  const int row = pos & ((1 << c.page_shift) - 1);
  const int half = c.D / 2, heads = a.hq + 2 * c.hkv;
  double2* const turn = turns[wave];
  if (a.rotate) {
    const int second = lane + 64;
    const double lo = rates.rev[lane < half ? lane : 0], hi = rates.rev[second < half ? second : 0];
    wave_lds_order();
    if (lane < half) turn[lane] = turn64(lo, pos);
    if (second < half) turn[second] = turn64(hi, pos);
    wave_lds_order();
  }
  const int col8 = lane % L, slot = lane / L, col = 8 * col8;
  const bool in_row = col < c.D;
  const long part_bytes = (long)quant_row_bytes(c.D) << c.page_shift;
  for (int h0 = part * H; h0 < heads; h0 += a.parts * H) {
    const int h = h0 + slot;
    const bool here = slot < H && h < heads;
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + c.hkv;
    if (here && in_row) {
      const IO* src;
      if (is_q)
        src = static_cast<const IO*>(a.q) + ((long)t * a.hq + h) * c.D;
      else if (is_k)
        src = static_cast<const IO*>(a.k) + ((long)t * c.hkv + (h - a.hq)) * c.D;
      else
        src = static_cast<const IO*>(a.v) + ((long)t * c.hkv + (h - a.hq - c.hkv)) * c.D;
#pragma unroll
      for (int p = 0; p < 2; ++p) {  // (half is a multiple of 4: four columns have their partners together)
        const int at = col + 4 * p;
        float own[4];
        load4f(src + at, own);
        if (a.rotate && (is_q || is_k)) {
          const bool first = at < half;
          float other[4];
          load4f(src + (first ? at + half : at - half), other);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const double2 cs = turn[(first ? at : at - half) + e];
            const double o = first ? -(double)other[e] : (double)other[e];
            own[e] = (float)fma((double)own[e], cs.x, o * cs.y);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * p + e] = own[e];
      }
    }
    if (here && is_q && in_row) store8(static_cast<IO*>(a.q_rot) + ((long)t * a.hq + h) * c.D + col, x);
    if (h0 + H <= a.hq || page < 0) continue;  // (the wave's heads are queries, or held nowhere)
    // (all lanes: a group's lanes exchange their largest elements)
    f16 scale;
    const unsigned w = quantise8(x, scale);
    if (!here || is_q) continue;
    const int kv = h - a.hq - (is_k ? 0 : c.hkv);
    char* const to = static_cast<char*>(is_k ? c.k_pages : c.v_pages) + page * c.page_stride + kv * part_bytes;
    f16* const scales = reinterpret_cast<f16*>(to + ((16L * G) << c.page_shift));
    reinterpret_cast<unsigned*>(to)[is_k ? k_word(row, G, col8) : v_word(row, G, col8)] = w;
    if (col8 % 4 == 0) scales[is_k ? k_scale(row, G, col8 / 4) : v_scale(row, G, col8 / 4)] = scale;
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
