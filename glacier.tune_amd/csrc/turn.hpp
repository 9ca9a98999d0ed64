// turn.hpp -- the position rotation of qk_norm.hip and cache_append.hip.
//
// A head's row is walked by L = lanes_of(D) consecutive lanes of a wave: lane
// ch of them holds the E elements ch E .. of the first half and the E elements
// of the second half that they are paired with, so a rotation needs no other
// lane.  A wave takes 64 / L heads of one token at a time.  The token's angles
// are formed once per wave, one pair a lane, and read back from LDS by the
// lanes of every head.
#pragma once

#include "attn_common.hpp"
#include "cache_launch.hpp"

namespace glacier {

// E elements of a row as they are loaded: 8 or 16 bytes of bf16, 16 of fp32.
template <typename IO, int E>
struct Piece {
  static_assert(E == 4 || (E == 8 && sizeof(IO) == 2), "a piece is 8 or 16 bytes");
  typedef IO V __attribute__((ext_vector_type(E)));
  V v;
  __device__ inline void load(const IO* p) { v = *reinterpret_cast<const V*>(p); }
  __device__ inline void store(IO* p) const { *reinterpret_cast<V*>(p) = v; }
  __device__ inline void get(float (&x)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = (float)v[e];
  }
  __device__ inline void set(const float (&x)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (IO)x[e];
  }
};

// cos and sin of pos times pair i's angle.  The number of revolutions is
// formed and reduced to [-1/2, 1/2] in 64 bits, so the angle is right wherever
// pos lies (in fp32 it would be off by pos 2^-24 radians); what rounding it to 32
// bits leaves turns the result by one more step (fp32 gradients of 333 tokens: off by
// 8.1e-8, now 7.4e-8; the weights' 1.78e-7, now 1.28e-7).
__device__ inline float2 turn_of(double rev, int pos) {
  double a = rev * (double)pos;
  a -= rint(a);
  const float near = (float)a;
  const float rest = (float)(a - near) * 6.2831853f;
  float s, c;
  sincospif(2.0f * near, &s, &c);
  return make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
}

// The rates of the pairs whose angles this lane forms.
struct LaneRates {
  double lo, hi;
  __device__ inline LaneRates(const TurnRates& r, int half, int lane) {
    lo = r.rev[lane < half ? lane : 0];
    hi = half > 64 ? r.rev[lane + 64 < half ? lane + 64 : 0] : 0.0;
  }
};

// This wave's angles of position pos into its LDS area [D/2].
__device__ inline void turn_table(float2* area, const LaneRates& r, int half, int pos, int lane) {
  wave_lds_order();
  if (lane < half) area[lane] = turn_of(r.lo, pos);
  if (lane + 64 < half) area[lane + 64] = turn_of(r.hi, pos);
  wave_lds_order();
}

// Waves that share one token's heads: as many as fill the chip with 16 waves a
// CU, each with one step of heads at least.
inline int turn_parts(int tokens, int steps, int n_cu) {
  const long want = 16L * n_cu;
  const long parts = (want + tokens - 1) / (tokens > 0 ? tokens : 1);
  return static_cast<int>(parts < 1 ? 1 : parts > steps ? steps : parts);
}

// Lanes of one head whose lanes take E elements of each half: a power of two, at
// least 4.
inline int lanes_of(int D, int E) {
  int l = 4;
  while (l * E < D / 2) l *= 2;
  return l;
}

// F<IO, 4, L> for the call's dtype and head size, from pieces of 4 elements.
#define GL_BY_HEAD4(F, io_bf16, D, ...)                                 \
  do {                                                                  \
    const int l_ = lanes_of(D, 4);                                      \
    if (l_ == 4) {                                                      \
      if (io_bf16) return F<bf16, 4, 4>(__VA_ARGS__);                   \
      return F<float, 4, 4>(__VA_ARGS__);                               \
    }                                                                   \
    if (l_ == 8) {                                                      \
      if (io_bf16) return F<bf16, 4, 8>(__VA_ARGS__);                   \
      return F<float, 4, 8>(__VA_ARGS__);                               \
    }                                                                   \
    if (l_ == 16) {                                                     \
      if (io_bf16) return F<bf16, 4, 16>(__VA_ARGS__);                  \
      return F<float, 4, 16>(__VA_ARGS__);                              \
    }                                                                   \
    if (io_bf16) return F<bf16, 4, 32>(__VA_ARGS__);                    \
    return F<float, 4, 32>(__VA_ARGS__);                                \
  } while (0)

// F<IO, E, L>: pieces of 8 elements (16 bytes) of bf16 where D allows.
#define GL_BY_HEAD(F, io_bf16, D, ...)                                  \
  do {                                                                  \
    if (!(io_bf16) || (D) % 16 != 0) GL_BY_HEAD4(F, io_bf16, D, __VA_ARGS__); \
    const int l8_ = lanes_of(D, 8);                                     \
    if (l8_ == 4) return F<bf16, 8, 4>(__VA_ARGS__);                    \
    if (l8_ == 8) return F<bf16, 8, 8>(__VA_ARGS__);                    \
    return F<bf16, 8, 16>(__VA_ARGS__);                                 \
  } while (0)

}  // namespace glacier
