// proj_quant.hip -- y_p = x W_p^T + bias_p + s_p (x A_p) B_p with base weights in 4 bits
// and group scales: a step of an answer (few tokens), or a prompt.
//
// Reading the weights bounds it up to some tens of tokens, so they are read once, 16
// bytes a lane, each word being what one lane feeds to one MFMA: 16 outputs by 32
// columns by 16 tokens.  A workgroup takes 16 outputs and up to 16 NT tokens; its
// waves share out the columns and are joined through LDS, where biases and the
// adapters' products are added.  x comes from L2, where every workgroup finds it.
//   bf16: weights as 128 + n (one operation per two), the sum begun at -136 sum(x),
//   which is one more product, with a constant; the scales are applied to the sums of
//   a group.  The sums are 17 to 136 times the product's terms, which costs 4 to 8 of
//   fp32's 24 bits.
//   fp32: weights as n - 8, x in three bf16 terms (24 bits).
// x A_p comes from the kernel of the bf16 projections (proj_lora.hip), in a launch
// before.
#include "quant_page.hpp"

namespace glacier {
namespace {

struct QuantSpec {
  const char* w;
  const float *bias, *l, *b;
  float s;
  int out, first;  // first: its first tile of 16 outputs
  void* y;
};
struct QuantCall {
  const void* x;
  int T, in, blocks, rank, n, tiles, token_blocks;
  QuantSpec p[kMaxProj];
};

// A wave's part of a block of 128 columns.
template <typename IO, int NT, int GP, bool OFF>
struct WBlock {
  u32x4 w;
  unsigned s[2 * GP], o[OFF ? 2 * GP : 1];  // of outputs 4 g ..: halves r GP + group
  typename std::conditional<sizeof(IO) == 2, bf16x8, f32x4[2]>::type x[NT][4];
};

template <int N>
__device__ inline void load_u32(const char* p, unsigned* to) {  // N = 2, 4 or 8
  if constexpr (N == 2) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    to[0] = v[0], to[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(p + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[i + e] = v[e];
    }
  }
}

// GP: groups of a block of 128 columns; OFF: weights have offsets
template <typename IO, int NT, int KS, int GP, bool OFF>
__global__ __launch_bounds__(64 * KS) void quant_proj_kernel(QuantCall a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using B = WBlock<IO, NT, GP, OFF>;
  constexpr bool F32 = sizeof(IO) == 4;
  constexpr int STRIDE = 20;  // floats of a token's 16 outputs in LDS
  __shared__ __align__(16) float red[KS * 16 * NT * STRIDE];
  const int w = wave_id(), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  // the token blocks of a tile of outputs follow each other on one XCD
  const int id = blockIdx.x, round = id / (8 * a.token_blocks);
  const int number = round * 8 + id % 8, t0 = id / 8 % a.token_blocks * 16 * NT;
  if (number >= a.tiles) return;
  int p = 0;
  while (p + 1 < a.n && number >= a.p[p + 1].first) ++p;
  const QuantSpec& job = a.p[p];
  const int tile = number - job.first;
  const long tiles = (job.out + 15) / 16;
  const char* const words = job.w + (long)tile * a.blocks * 1024 + lane * 16;
  const char* const scales = job.w + tiles * a.blocks * 1024 + (long)tile * a.blocks * (32 * GP) + g * (8 * GP);
  const char* const offsets = scales + tiles * a.blocks * (32 * GP);
  const IO* x[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x[n] = static_cast<const IO*>(a.x) + (long)min(t0 + 16 * n + col, a.T - 1) * a.in;
  auto load = [&](B& to, int blk) __attribute__((always_inline)) {
    to.w = *reinterpret_cast<const u32x4*>(words + (long)blk * 1024);
    load_u32<2 * GP>(scales + (long)blk * (32 * GP), to.s);
    if constexpr (OFF) load_u32<2 * GP>(offsets + (long)blk * (32 * GP), to.o);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = min(128 * blk + 32 * i + 8 * g, a.in - 8);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (F32) {
          to.x[n][i][0] = *reinterpret_cast<const f32x4*>(x[n] + k);
          to.x[n][i][1] = *reinterpret_cast<const f32x4*>(x[n] + k + 4);
        } else {
          to.x[n][i] = *reinterpret_cast<const bf16x8*>(x[n] + k);
        }
      }
    }
  };
  const QuantMagic magic;
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  f32x4 y[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) y[n] = zero;
  bf16x8 minus, ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) minus[e] = (bf16)-136.0f, ones[e] = (bf16)1.0f;
  auto take = [&](B& from, int blk) __attribute__((always_inline)) {
    if (128 * blk + 128 > a.in) {  // columns past the last one
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (128 * blk + 32 * i >= a.in)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (F32)
              from.x[n][i][0] = from.x[n][i][1] = zero;
            else
              from.x[n][i] = frag_zero<bf16>();
          }
    }
#pragma unroll
    for (int q = 0; q < GP; ++q) {
      f32x4 d[NT], d0[NT];  // of the group: products, and -136 sum(x) (fp32: sum(x))
      if constexpr (F32) {
#pragma unroll
        for (int n = 0; n < NT; ++n) d[n] = d0[n] = zero;
#pragma unroll
        for (int i = q * 4 / GP; i < (q + 1) * 4 / GP; ++i) {
          const bf16x8 wf = exact8_bf16(from.w[i], magic);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            bf16x8 h, m, l;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float v = from.x[n][i][e / 4][e % 4];
              h[e] = (bf16)v;
              const float r1 = v - (float)h[e];
              m[e] = (bf16)r1;
              l[e] = (bf16)(r1 - (float)m[e]);
            }
            d[n] = Mfma<bf16>::mma(wf, l, d[n]);
            d[n] = Mfma<bf16>::mma(wf, m, d[n]);
            d[n] = Mfma<bf16>::mma(wf, h, d[n]);
            if constexpr (OFF) {
              d0[n] = Mfma<bf16>::mma(ones, l, d0[n]);
              d0[n] = Mfma<bf16>::mma(ones, m, d0[n]);
              d0[n] = Mfma<bf16>::mma(ones, h, d0[n]);
            }
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) d0[n] = zero;
#pragma unroll
        for (int i = q * 4 / GP; i < (q + 1) * 4 / GP; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n) d0[n] = Mfma<bf16>::mma(minus, from.x[n][i], d0[n]);
#pragma unroll
        for (int n = 0; n < NT; ++n) d[n] = d0[n];
#pragma unroll
        for (int i = q * 4 / GP; i < (q + 1) * 4 / GP; ++i) {
          const bf16x8 wf = raw8_bf16(from.w[i], magic);
#pragma unroll
          for (int n = 0; n < NT; ++n) d[n] = Mfma<bf16>::mma(wf, from.x[n][i], d[n]);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float s = half_at(from.s[(r * GP + q) / 2], (r * GP + q) % 2);
#pragma unroll
        for (int n = 0; n < NT; ++n) y[n][r] = fmaf(s, d[n][r], y[n][r]);
        if constexpr (OFF) {
          const float o = half_at(from.o[(r * GP + q) / 2], (r * GP + q) % 2) * (F32 ? 1.0f : -1.0f / 136.0f);
#pragma unroll
          for (int n = 0; n < NT; ++n) y[n][r] = fmaf(o, d0[n][r], y[n][r]);
        }
      }
    }
  };
  B u, v;
  int blk = w;
  if (blk < a.blocks) load(u, blk);
  for (; blk < a.blocks; blk += 2 * KS) {  // two blocks a turn, each loaded while the other is worked on
    if (blk + KS < a.blocks) load(v, blk + KS);
    take(u, blk);
    if (blk + KS >= a.blocks) break;
    if (blk + 2 * KS < a.blocks) load(u, blk + 2 * KS);
    take(v, blk + KS);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) store4(red + ((w * NT + n) * 16 + col) * STRIDE + 4 * g, y[n]);
  __syncthreads();
  for (int idx = threadIdx.x; idx < 64 * NT; idx += 64 * KS) {
    const int t = t0 + idx / 4, o = 16 * tile + 4 * (idx % 4);
    if (t >= a.T || o >= job.out) continue;
    f32x4 sum = zero;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const f32x4 part = *reinterpret_cast<const f32x4*>(red + (k * NT * 16 + idx / 4) * STRIDE + 4 * (idx % 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += part[e];
    }
    if (job.l != nullptr) {
      f32x4 low = zero;
      const float* const l = job.l + (long)t * a.rank;
      for (int j = 0; j < a.rank; ++j) {
        const f32x4 bj = *reinterpret_cast<const f32x4*>(job.b + (long)j * job.out + o);
#pragma unroll
        for (int e = 0; e < 4; ++e) low[e] = fmaf(l[j], bj[e], low[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(job.s, low[e], sum[e]);
    }
    if (job.bias != nullptr)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += job.bias[o + e];
    store4(static_cast<IO*>(job.y) + (long)t * job.out + o, sum);
  }
#endif
}

// ---- laying out ------------------------------------------------------------
__global__ __launch_bounds__(256) void quant_pack_kernel(QuantPack a, QuantLayout l) {
  const long words = l.scales / 4, halves = (l.offsets - l.scales) / 2;
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  if (at < words) {
    const int i = at % 4, entry = at / 4 % 64;
    const long blk = at / 256 % l.blocks, tile = at / 256 / l.blocks;
    const long row = 16 * tile + entry % 16, k = 128 * blk + 32 * i + 8 * (entry / 16);
    unsigned w = kQuantZero;
    if (row < a.out && k < a.in) {
      const unsigned char* const from = static_cast<const unsigned char*>(a.numbers) + row * (a.in / 2) + k / 2;
      w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) w |= (from[j] & 15u) << (4 * j) | static_cast<unsigned>(from[j] >> 4) << (16 + 4 * j);
    }
    reinterpret_cast<unsigned*>(a.packed)[at] = w;
    return;
  }
  const long z = at - words, which = z / halves, x = z % halves;
  if (which > (a.offsets != nullptr ? 1 : 0)) return;
  const int per = 128 / a.group;
  const long q = x % per, r = x / per % 16, blk = x / per / 16 % l.blocks, tile = x / per / 16 / l.blocks;
  const long row = 16 * tile + r, i = blk * per + q, groups = a.in / a.group;
  const auto* const from = static_cast<const unsigned short*>(which == 0 ? a.scales : a.offsets);
  reinterpret_cast<unsigned short*>(static_cast<char*>(a.packed) + l.scales)[z] =
      row < a.out && i < groups ? from[row * groups + i] : static_cast<unsigned short>(0);
}

template <typename IO, int NT, int KS, int GP, bool OFF>
hipError_t project(const QuantCall& c, hipStream_t st) {
  hipLaunchKernelGGL((quant_proj_kernel<IO, NT, KS, GP, OFF>), dim3((c.tiles + 7) / 8 * 8 * c.token_blocks),
                     dim3(64 * KS), 0, st, c);
  return hipGetLastError();
}
template <typename IO, int NT, int KS>
hipError_t by_group(const QuantCall& c, int group, bool off, hipStream_t st) {
  if (group == 32) return off ? project<IO, NT, KS, 4, true>(c, st) : project<IO, NT, KS, 4, false>(c, st);
  if (group == 64) return off ? project<IO, NT, KS, 2, true>(c, st) : project<IO, NT, KS, 2, false>(c, st);
  return off ? project<IO, NT, KS, 1, true>(c, st) : project<IO, NT, KS, 1, false>(c, st);
}
template <typename IO>
hipError_t by_shape(QuantCall c, int group, bool off, int n_cu, hipStream_t st) {
  constexpr int MOST = sizeof(IO) == 2 ? 4 : 2;
  const int nt = c.T <= 16 ? 1 : c.T <= 32 || MOST == 2 ? 2 : 4;
  c.token_blocks = (c.T + 16 * nt - 1) / (16 * nt);
  const bool deep = (long)c.tiles * c.token_blocks < 4L * n_cu;
  if (nt == 1) return deep ? by_group<IO, 1, 8>(c, group, off, st) : by_group<IO, 1, 4>(c, group, off, st);
  if (nt == 2) return deep ? by_group<IO, 2, 8>(c, group, off, st) : by_group<IO, 2, 4>(c, group, off, st);
  if constexpr (MOST == 4)
    return deep ? by_group<IO, 4, 8>(c, group, off, st) : by_group<IO, 4, 4>(c, group, off, st);
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_quant_pack(const QuantPack& a, hipStream_t st) {
  const QuantLayout l = quant_layout(a.out, a.in, a.group, a.offsets != nullptr);
  const long n = l.scales / 4 + (l.bytes - l.scales) / 2;
  hipLaunchKernelGGL(quant_pack_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, st, a, l);
  return hipGetLastError();
}

hipError_t launch_quant_proj(const QuantProj& q, int n_cu, hipStream_t st) {
  const ProjLaunch& a = q.a;
  QuantCall c{};
  c.x = a.x;
  c.T = a.T;
  c.in = a.in;
  c.blocks = (a.in + 127) / 128;
  c.rank = a.rank;
  c.n = a.n_proj;
  float* l[kMaxProj] = {};
  for (int p = 0; p < a.n_proj; ++p) {
    const ProjSpec& s = a.p[p];
    if (s.a != nullptr) l[p] = q.low + (long)p * a.T * a.rank;
    c.p[p] = QuantSpec{static_cast<const char*>(s.w), s.bias, l[p], s.b, s.scaling, s.out, c.tiles, s.y};
    c.tiles += (s.out + 15) / 16;
  }
  GL_CHECK(launch_lowrank_forward(a, l, st));
  return a.io_bf16 ? by_shape<bf16>(c, q.group, q.offsets, n_cu, st)
                   : by_shape<float>(c, q.group, q.offsets, n_cu, st);
}

}  // namespace glacier
