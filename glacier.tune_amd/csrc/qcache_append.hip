// qcache_append.hip -- new tokens' keys (rotated) and values into a paged cache in 4
// bits, their queries rotated in the same launch; and tokens back from such pages.
//
// HBM-bound: each row is read once and written once.  A wave takes one token, or a
// share of its heads when there are few tokens.  A lane holds eight columns of a
// head, so a group of 32 is four neighbouring lanes: its largest element is found in
// two exchanges, and a lane's eight numbers are one word of the page.  A step's rows are
// in flight while the one before is worked on, the first from before the token's place
// is known, and the angles of a lane's columns stay in its registers.  5272 tokens of 32
// query and 8 KV heads of 128 (bf16): 26.4 us for 114 MB (4.3 TB/s), 1600 operations a
// token; with the rows asked for step by step and the angles read from LDS 38, with
// queries in a key's layout, which forms each angle's product twice, and elements rounded
// from 64 bits to bf16 at once 29.4.  Read back in 8.0.
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

// Of a query a lane holds four columns of the first half and the four that they are
// rotated with; of a key eight columns in a row (a word) and their eight partners.
template <typename IO>
struct Columns {
  Piece<IO, 4> own[2], other[2];
};

// x rounded to fp32, kept so: rounded to bf16 from there (the compiler rounds some
// elements from 64 bits otherwise, by eight operations each).
__device__ inline float rounded(double x) {
  float r = (float)x;
  asm("" : "+v"(r));
  return r;
}

template <typename IO, int G>
__global__ __launch_bounds__(64 * kWavesQa) void qcache_append_kernel(CacheAppend a, TurnRates rates) {
  constexpr int L = 4 * G, H = 64 / L;  // lanes of a head, heads per step
  __shared__ double2 turns[kWavesQa][kTurnMaxDim / 2];
  const CacheView& c = a.c;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int unit = blockIdx.x * kWavesQa + wave;
  const int t = unit / a.parts, part = unit - t * a.parts;
  if (t >= c.T) return;
  const int half = c.D / 2, held = 2 * c.hkv, q_steps = (a.hq + H - 1) / H, steps = q_steps + (held + H - 1) / H;
  const int col8 = lane % L, slot = lane / L, col = 8 * col8;
  // queries: pairs (pair + e, half + pair + e) (half is a multiple of 4)
  const bool has_pair = slot < H && 4 * col8 < half;
  const int pair = has_pair ? 4 * col8 : 0;
  const IO* const q = static_cast<const IO*>(a.q) + (long)t * a.hq * c.D;
  auto load_q = [&](Piece<IO, 4> (&to)[2], int step) __attribute__((always_inline)) {
    const IO* const src = q + (long)min(step * H + slot, a.hq - 1) * c.D + pair;
    to[0].load(src), to[1].load(src + half);
  };
  // keys and values, keys first: columns col .. and, rotated, their partners
  const bool in_row = slot < H && col < c.D;
  const int at0 = in_row ? col : 0, at1 = at0 + 4;
  const int to0 = at0 < half ? at0 + half : at0 - half, to1 = at1 < half ? at1 + half : at1 - half;
  auto load_kv = [&](Columns<IO>& to, int step) __attribute__((always_inline)) {
    const int h0 = (step - q_steps) * H, h = min(h0 + slot, held - 1);
    const IO* const src = h < c.hkv ? static_cast<const IO*>(a.k) + ((long)t * c.hkv + h) * c.D
                                    : static_cast<const IO*>(a.v) + ((long)t * c.hkv + (h - c.hkv)) * c.D;
    to.own[0].load(src + at0), to.own[1].load(src + at1);
    if (a.rotate && h0 < c.hkv) to.other[0].load(src + to0), to.other[1].load(src + to1);
  };
  // a step's rows are in flight while the one before is worked on, the first ones from
  // before the search for the token's place
  int step = part;
  const int first_kv = step >= q_steps ? step : step + (q_steps - step + a.parts - 1) / a.parts * a.parts;
  Piece<IO, 4> one[2], two[2];
  Columns<IO> next;
  if (step < q_steps) load_q(one, step);
  if (step + a.parts < q_steps) load_q(two, step + a.parts);
  if (first_kv < steps) load_kv(next, first_kv);
  const CacheSeq s = seq_of_token(c, lane, t);
  if (s.b >= c.n_seqs || t < s.tok0) return;  // behind the last sequence
  const int pos = s.pos0 + (t - s.tok0);
  const int page = cache_page(c, s.b, pos);
  const int row = pos & ((1 << c.page_shift) - 1);
  double2* const turn = turns[wave];
  if (a.rotate) {
    const int second = lane + 64;
    const double lo = rates.rev[lane < half ? lane : 0], hi = rates.rev[second < half ? second : 0];
    if (lane < half) turn[lane] = turn64(lo, pos);
    if (second < half) turn[second] = turn64(hi, pos);
    wave_lds_order();
  }
  if (step < q_steps) {
    double2 cs[4];  // the angles of this lane's pairs, the same in every head
#pragma unroll
    for (int e = 0; e < 4; ++e) cs[e] = turn[pair + e];
    IO* const q_rot = static_cast<IO*>(a.q_rot) + (long)t * a.hq * c.D;
    auto take = [&](const Piece<IO, 4> (&from)[2], int at) __attribute__((always_inline)) {
      const int h = at * H + slot;
      float x[4], y[4], u[4], v[4];
      from[0].get(x), from[1].get(y);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double xd = x[e], yd = y[e];
        u[e] = rounded(fma(xd, cs[e].x, -yd * cs[e].y));
        v[e] = rounded(fma(yd, cs[e].x, xd * cs[e].y));
      }
      if (!has_pair || h >= a.hq) return;
      Piece<IO, 4> to[2];
      to[0].set(u), to[1].set(v);
      to[0].store(q_rot + (long)h * c.D + pair), to[1].store(q_rot + (long)h * c.D + pair + half);
    };
    for (; step < q_steps; step += 2 * a.parts) {
      const int then = step + a.parts;
      take(one, step);
      if (then >= q_steps) break;
      if (then + a.parts < q_steps) load_q(one, then + a.parts);
      take(two, then);
      if (then + 2 * a.parts < q_steps) load_q(two, then + 2 * a.parts);
    }
  }
  if (page < 0) return;  // (held nowhere)
  double co[8], si[8];
  if (a.rotate && (first_kv - q_steps) * H < c.hkv) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = (e < 4 ? at0 : at1) + e % 4;
      const double2 cs = turn[at < half ? at : at - half];
      co[e] = cs.x, si[e] = at < half ? -cs.y : cs.y;
    }
  }
  const long part_bytes = (long)quant_row_bytes(c.D) << c.page_shift;
  for (step = first_kv; step < steps; step += a.parts) {
    const Columns<IO> from = next;
    if (step + a.parts < steps) load_kv(next, step + a.parts);
    const int h0 = (step - q_steps) * H, h = h0 + slot;
    const bool here = slot < H && h < held, is_k = h < c.hkv;
    float x[8];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      float own[4];
      from.own[p].get(own);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * p + e] = in_row ? own[e] : 0.0f;
    }
    if (a.rotate && h0 < c.hkv) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float other[4];
        from.other[p].get(other);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * p + e;
          const float r = (float)fma((double)x[i], co[i], (double)other[e] * si[i]);
          x[i] = in_row && is_k ? r : x[i];
        }
      }
    }
    // (all lanes: a group's lanes exchange their largest elements)
    f16 scale;
    const unsigned w = quantise8(x, scale);
    if (!here) continue;
    const int kv = is_k ? h : h - c.hkv;
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
  a.parts = turn_parts(a.c.T, (a.hq + H - 1) / H + (2 * a.c.hkv + H - 1) / H, n_cu);
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
