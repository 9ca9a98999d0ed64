// qk_norm.hip -- the per-head RMS norms of a layer's queries and keys with the
// position rotation in the same pass, forward and backward:
//   forward   y = R(pos) (x r w),  r = 1 / sqrt(mean x^2 + eps)
//   backward  g = R(-pos) dy,  dx = r w g - (r^3 / D) x sum w g x,
//             dw += sum over tokens and heads of g x r
// (the norms of TransformerBlock.cs:413, :421, :751 and :759, and the rotation
// that follows them).
//
// HBM-bound: each row is read once and written once, a head's sums are one
// fixed-order reduction over the lanes that hold it (turn.hpp), and queries and
// keys share the launch.  Each lane reads its pieces before it writes them, so
// outputs may lie on inputs.  Measured: 4096 tokens of 32/8 heads of 128, bf16,
// 15.3-17 us (5.5-4.9 TB/s: part of it stays in the last-level cache; a 4 GiB copy
// reaches 4.77), 15.2 without the rotation; fp32 30.8 and 28.2 (5.4, 6.0 TB/s); 8
// tokens of 28/4 heads 3.6 us in a replayed graph, the launch (2.9 without).
//
// Weight gradients: a lane meets the same columns in every head and token, so
// it sums them in registers; a workgroup's sums go to the workspace and a second
// launch adds the workgroups in order.  No atomics: results are bitwise
// repeatable.  The backward holds four rows' pieces and four columns' sums a lane,
// so its pieces are 8 bytes in bf16: with 16 it has registers for half the waves
// (4096 tokens of 28/4 heads of 128, bf16, with weight gradients: 35 us against
// 30.8).  Now, in a replayed graph: 27.6 us (3.7 TB/s, of them 4 in the second
// launch), 21.5 without weight gradients; as training calls it, without the rotation,
// 25.7 and 20.1; fp32 37.8 and 32.7 with it, 36.8 and 32.0 without.
#include "turn.hpp"

namespace glacier {
namespace {

constexpr int kWavesQk = 4;
constexpr int kWavesQkBwd = 8;  // with kQkMaxGroups workgroups: 16 waves a CU

template <typename IO, int E, int L>
__global__ __launch_bounds__(64 * kWavesQk) void qk_norm_fwd_kernel(QkNorm a, TurnRates rates) {
  constexpr int H = 64 / L;  // heads per step
  __shared__ float2 turns[kWavesQk][kTurnMaxDim / 2];
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int unit = blockIdx.x * kWavesQk + wave;
  const int t = unit / a.parts, part = unit % a.parts;
  if (t >= a.T) return;
  const int half = a.D / 2, heads = a.hq + a.hkv;
  const int ch = lane % L, col = ch * E;
  const bool in_row = col < half;
  if (a.rotate)
    turn_table(turns[wave], LaneRates(rates, half, lane), half, a.positions != nullptr ? a.positions[t] : t, lane);
  for (int h0 = part * H; h0 < heads; h0 += a.parts * H) {
    const int h = h0 + lane / L;
    const bool ok = in_row && h < heads, is_q = h < a.hq;
    const long at = is_q ? ((long)t * a.hq + h) * a.D : ((long)t * a.hkv + (h - a.hq)) * a.D;
    const float* w = is_q ? a.wq : a.wk;
    float x0[E] = {}, x1[E] = {}, w0[E] = {}, w1[E] = {};
    if (ok) {
      const IO* x = static_cast<const IO*>(is_q ? a.q : a.k) + at + col;
      Piece<IO, E> p0, p1;
      p0.load(x);
      p1.load(x + half);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        w0[e] = w[col + e];
        w1[e] = w[half + col + e];
      }
      p0.get(x0);
      p1.get(x1);
    }
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) ss += x0[e] * x0[e] + x1[e] * x1[e];
    const float r = 1.0f / sqrtf(lanes_sum<L>(ss) / (float)a.D + a.eps);
    if (!ok) continue;
    float y0[E], y1[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      y0[e] = (x0[e] * r) * w0[e];
      y1[e] = (x1[e] * r) * w1[e];
      if (a.rotate) {
        const float2 cs = turns[wave][col + e];
        rope_fwd(y0[e], y1[e], cs.x, cs.y, y0[e], y1[e]);
      }
    }
    IO* y = static_cast<IO*>(is_q ? a.yq : a.yk) + at + col;
    Piece<IO, E> o0, o1;
    o0.set(y0);
    o1.set(y1);
    o0.store(y);
    o1.store(y + half);
  }
}

// DW: the weight gradients are formed.  The wave's steps (a token's heads, H at
// a time) follow each other with the next step's rows requested before this
// one's are used.
template <typename IO, int E, int L, bool DW>
__global__ __launch_bounds__(64 * kWavesQkBwd) void qk_norm_bwd_kernel(QkNorm a, TurnRates rates) {
  constexpr int H = 64 / L;
  __shared__ float2 turns[kWavesQkBwd][kTurnMaxDim / 2];
  __shared__ float sums[DW ? kWavesQkBwd : 1][DW ? 2 * kTurnMaxDim : 1];
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int half = a.D / 2, heads = a.hq + a.hkv;
  const int ch = lane % L, col = ch * E;
  const bool in_row = col < half;
  const LaneRates lane_rates(rates, half, lane);
  float dq0[E] = {}, dq1[E] = {}, dk0[E] = {}, dk1[E] = {};
  const int units = a.T * a.parts;

  struct Step {
    int unit, h0;
  };
  // a step's rows; the place of this lane's head is formed again where it is used
  auto place = [&](const Step& s, bool& is_q) {
    const int t = s.unit / a.parts, h = s.h0 + lane / L;
    is_q = h < a.hq;
    return (is_q ? (long)t * a.hq + h : (long)t * a.hkv + (h - a.hq)) * a.D + col;
  };
  struct Rows {
    Piece<IO, E> x0, x1, d0, d1;
  };
  auto load = [&](const Step& s, Rows& r) {
    bool is_q;
    const long at = place(s, is_q);
    if (s.unit >= units || !in_row || s.h0 + lane / L >= heads) return;
    const IO* x = static_cast<const IO*>(is_q ? a.q : a.k) + at;
    const IO* dy = static_cast<const IO*>(is_q ? a.dq_out : a.dk_out) + at;
    r.x0.load(x);
    r.x1.load(x + half);
    r.d0.load(dy);
    r.d1.load(dy + half);
  };
  auto after = [&](Step s) {
    s.h0 += a.parts * H;
    if (s.h0 >= heads) {
      s.unit += gridDim.x * kWavesQkBwd;
      s.h0 = s.unit % a.parts * H;
    }
    return s;
  };
  auto position = [&](int unit) {
    const int t = unit / a.parts;
    return a.positions != nullptr && a.rotate && unit < units ? a.positions[t] : t;
  };

  Step now;
  now.unit = blockIdx.x * kWavesQkBwd + wave;
  now.h0 = now.unit % a.parts * H;
  Rows rows{}, ahead{};
  load(now, rows);
  int formed = -1, pos = position(now.unit);
  while (now.unit < units) {
    const Step next = after(now);
    load(next, ahead);
    if (now.unit != formed) {
      if (a.rotate) turn_table(turns[wave], lane_rates, half, pos, lane);
      formed = now.unit;
      pos = position(now.unit + gridDim.x * kWavesQkBwd);
    }
    bool is_q;
    const long at = place(now, is_q);
    const bool ok = in_row && now.h0 + lane / L < heads;
    const float* w = is_q ? a.wq : a.wk;
    float x0[E] = {}, x1[E] = {}, g0[E] = {}, g1[E] = {}, w0[E] = {}, w1[E] = {};
    if (ok) {
      rows.x0.get(x0);
      rows.x1.get(x1);
      rows.d0.get(g0);
      rows.d1.get(g1);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        w0[e] = w[col + e];
        w1[e] = w[half + col + e];
      }
    }
    float ss = 0.0f, c = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (a.rotate && in_row) {
        const float2 cs = turns[wave][col + e];
        rope_inv(g0[e], g1[e], cs.x, cs.y, g0[e], g1[e]);
      }
      ss += x0[e] * x0[e] + x1[e] * x1[e];
      c += (w0[e] * g0[e]) * x0[e] + (w1[e] * g1[e]) * x1[e];
    }
    ss = lanes_sum<L>(ss);
    c = lanes_sum<L>(c);
    if (ok) {
      const float r = 1.0f / sqrtf(ss / (float)a.D + a.eps);
      // (by n = x r, whose size is that of 1: r^3 leaves fp32 for rows below 1e-13)
      const float cn = c * r / (float)a.D;
      float o0[E], o1[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float n0 = x0[e] * r, n1 = x1[e] * r;
        o0[e] = r * (w0[e] * g0[e] - n0 * cn);
        o1[e] = r * (w1[e] * g1[e] - n1 * cn);
        if constexpr (DW) {
          const float v0 = g0[e] * n0, v1 = g1[e] * n1;
          dq0[e] += is_q ? v0 : 0.0f;
          dq1[e] += is_q ? v1 : 0.0f;
          dk0[e] += is_q ? 0.0f : v0;
          dk1[e] += is_q ? 0.0f : v1;
        }
      }
      IO* dx = static_cast<IO*>(is_q ? a.yq : a.yk) + at;
      Piece<IO, E> s0, s1;
      s0.set(o0);
      s1.set(o1);
      s0.store(dx);
      s1.store(dx + half);
    }
    rows = ahead;
    now = next;
  }
  if constexpr (DW) {
    // the lanes that hold the same columns (the wave's heads), then the waves
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int s = L; s < 64; s *= 2) {
        dq0[e] += __shfl_xor(dq0[e], s);
        dq1[e] += __shfl_xor(dq1[e], s);
        dk0[e] += __shfl_xor(dk0[e], s);
        dk1[e] += __shfl_xor(dk1[e], s);
      }
      if (lane < L && in_row) {
        sums[wave][col + e] = dq0[e];
        sums[wave][half + col + e] = dq1[e];
        sums[wave][a.D + col + e] = dk0[e];
        sums[wave][a.D + half + col + e] = dk1[e];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.D; i += 64 * kWavesQkBwd) {
      float s = 0.0f;
#pragma unroll
      for (int u = 0; u < kWavesQkBwd; ++u) s += sums[u][i];
      a.partials[(long)blockIdx.x * 2 * a.D + i] = s;
    }
  }
}

// dw[i] += sum over the workgroups' partials: 16 columns a workgroup, 64 rows
// side by side, so that 512 rows are one round of loads deep; then a tree, which
// rounds less than a chain (fp32, 333 tokens of 2 heads: off by 1.75e-7 of the sums, now 1.1e-7).
__global__ __launch_bounds__(1024) void qk_norm_dw_kernel(QkNorm a, int groups) {
  __shared__ float sums[16][16];
  const int x = threadIdx.x & 15, part = threadIdx.x >> 4, i = blockIdx.x * 16 + x;
  float s = 0.0f;
#pragma unroll
  for (int u = 0; u < kQkMaxGroups / 64; ++u) {
    const int g = part + 64 * u;
    s += g < groups ? a.partials[(long)g * 2 * a.D + i] : 0.0f;
  }
  s = col_sum(s);  // the wave's four rows
  if (threadIdx.x % 64 < 16) sums[part / 4][x] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const float total =
      col_sum((sums[4 * part][x] + sums[4 * part + 1][x]) + (sums[4 * part + 2][x] + sums[4 * part + 3][x]));
  if (part != 0) return;
  float* dw = i < a.D ? a.dwq : a.dwk;
  if (dw != nullptr) dw[i < a.D ? i : i - a.D] += total;
}

template <typename IO, int E, int L>
hipError_t fwd(QkNorm& a, const TurnRates& r, int n_cu, hipStream_t st) {
  a.parts = turn_parts(a.T, (a.hq + a.hkv + 64 / L - 1) / (64 / L), n_cu);
  const long units = (long)a.T * a.parts;
  hipLaunchKernelGGL((qk_norm_fwd_kernel<IO, E, L>), dim3((units + kWavesQk - 1) / kWavesQk),
                     dim3(64 * kWavesQk), 0, st, a, r);
  return hipGetLastError();
}

template <typename IO, int E, int L>
hipError_t bwd(QkNorm& a, const TurnRates& r, int n_cu, hipStream_t st) {
  a.parts = turn_parts(a.T, (a.hq + a.hkv + 64 / L - 1) / (64 / L), n_cu);
  const long units = (long)a.T * a.parts;
  const bool dw = a.dwq != nullptr || a.dwk != nullptr;
  const int groups = static_cast<int>(std::min<long>((units + kWavesQkBwd - 1) / kWavesQkBwd, kQkMaxGroups));
  const dim3 block(64 * kWavesQkBwd);
  if (dw)
    hipLaunchKernelGGL((qk_norm_bwd_kernel<IO, E, L, true>), dim3(groups), block, 0, st, a, r);
  else
    hipLaunchKernelGGL((qk_norm_bwd_kernel<IO, E, L, false>), dim3(groups), block, 0, st, a, r);
  GL_CHECK(hipGetLastError());
  if (!dw) return hipSuccess;
  hipLaunchKernelGGL(qk_norm_dw_kernel, dim3(2 * a.D / 16), dim3(1024), 0, st, a, groups);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_qk_norm_forward(QkNorm a, const TurnRates& r, int n_cu, hipStream_t st) {
  GL_BY_HEAD(fwd, a.io_bf16, a.D, a, r, n_cu, st);
}

hipError_t launch_qk_norm_backward(QkNorm a, const TurnRates& r, int n_cu, hipStream_t st) {
  GL_BY_HEAD4(bwd, a.io_bf16, a.D, a, r, n_cu, st);
}

}  // namespace glacier
