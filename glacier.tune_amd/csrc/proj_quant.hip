// proj_quant.hip -- y_p = x W_p^T + bias_p + s_p (x A_p) B_p with base weights in 4 bits
// and group scales: a step of an answer (few tokens), or a prompt.
//
// Reading the weights bounds it up to some tens of tokens, so they are read once a
// workgroup, 16 bytes a lane, each word being what one lane feeds to one MFMA: 16 outputs
// by 32 columns by 16 tokens.  [1] 3584 -> 18944 twice (76 MB) 18.1 us, 4.2 TB/s with
// start and end; 16 tokens, groups of 128 with offsets, 20.9; 64 tokens 43.5; 512 tokens
// 202 to 224, 620 to 690 TFLOP/s.
//   bf16: weights as 128 + n (one operation per two), the sum begun at -136 sum(x),
//   which is one more product, with a constant; the scales are applied to the sums of
//   a group.  The sums are 17 to 136 times the product's terms, which costs 4 to 8 of
//   fp32's 24 bits.
//   fp32: weights as n - 8, x in three bf16 terms (24 bits), which a launch before writes.
// x A_p comes from a launch before, for more than 16 tokens from the kernel of the bf16
// projections (proj_lora.hip); (x A_p) B_p by fp32 products into the same sums.
#include "lds_mfma.hpp"
#include "quant_grid.hpp"
#include "quant_page.hpp"

#include <algorithm>

namespace glacier {
namespace {

struct QuantSpec {
  const char* w;
  const float *bias, *l, *b;  // l: the parts of x A_p [splits][T][rank], or null
  float s;
  int out, first;  // first: its first tile of 16 RT outputs
  void* y;
};
struct QuantCall {
  const void* x;
  int T, in, blocks, rank, splits, n, tiles, token_blocks;
  QuantSpec p[kMaxProj];
};

#if defined(__HIP_DEVICE_COMPILE__)
template <int N>
__device__ inline void load_u32(__amdgpu_buffer_rsrc_t rs, int voff, int soff, unsigned* to) {  // N = 2, 4 or 8
  if constexpr (N == 2) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b64(rs, voff, soff, 0);
    to[0] = static_cast<unsigned>(v[0]), to[1] = static_cast<unsigned>(v[1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(rs, voff + 4 * i, soff, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[i + e] = static_cast<unsigned>(v[e]);
    }
  }
}
#endif

// A workgroup takes 16 RT RW outputs of 16 NT tokens.  RW waves take 16 RT outputs each and
// walk the columns together, a block of 128 a step; KW such sets take every KW-th block
// and are joined at the end.  x's operands of a block (NT of 1 KB for each 32 columns,
// three times as many for fp32's terms) come by LDS DMA in the order in which lanes read
// them (no bank conflicts, one read an operand), two steps ahead, one barrier a step; a
// wave's weights come into its registers a step ahead.
template <int NT, int RT, int RW, int KW, int GP, bool OFF, int TERMS>
struct TileCfg {
  static constexpr int SLOT = 4096 * NT * TERMS, SLOTS = 3, WAVES = RW * KW;
  static constexpr int STRIDE = 20;  // floats of a token's 16 outputs in the join
  static constexpr int RING = KW * SLOTS * SLOT, JOIN = KW > 1 ? WAVES * RT * NT * 16 * STRIDE * 4 : 0;
  static constexpr int BYTES = RING > JOIN ? RING : JOIN;
  // Offsets of groups of 32, four to a block: one fp32 product for it, of them and the
  // sums of x, which every tile's sums begin with (bf16: -136 of them; fp32: they do not).
  // Larger groups: the sums of x are kept apart and scaled with the others, vector
  // instructions once a group.  [103] 3584 -> 37888 and [16], with offsets, groups of 32:
  // 81 and 24.5 us (kept apart: 109 and 28).
  static constexpr bool FOLD = OFF && GP == 4;
  // -136 sum(x) into the sums of every tile of outputs (one more product each), or kept
  // apart and scaled with them
  static constexpr bool CHAIN = TERMS == 1 && !OFF && (GP == 4 || RT == 1);
  static constexpr bool SUMS = !FOLD && (TERMS == 1 ? !CHAIN : OFF);  // sums of x of their own
  // loads of a step: a wave's share of x's operands, then its weights
  static constexpr int XLOADS = 4 * NT * TERMS / RW, HALVES = GP == 4 ? 2 : 1;
  static constexpr int WLOADS = RT * (1 + HALVES * (OFF && !FOLD ? 2 : 1) + (FOLD ? 1 : 0));
};

template <int NT, int RT, int RW, int KW, int GP, bool OFF, int TERMS>
__global__ __launch_bounds__(64 * RW * KW) void quant_tile_kernel(QuantCall a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using C = TileCfg<NT, RT, RW, KW, GP, OFF, TERMS>;
  using IO = typename std::conditional<TERMS == 1, bf16, float>::type;
  extern __shared__ __align__(16) unsigned char smem[];
  const int w = wave_id() % RW, kw = wave_id() / RW, lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const QuantPlace place = quant_place(blockIdx.x, (a.tiles + RW - 1) / RW, a.token_blocks);
  const int t0 = place.block * 16 * NT;
  int number = RW * place.set + w;
  const bool has_tile = number < a.tiles;
  if (!has_tile) number = a.tiles - 1;  // (its wave takes part in the barriers)
  int p = 0;
  while (p + 1 < a.n && number >= a.p[p + 1].first) ++p;
  const QuantSpec& job = a.p[p];
  const int tile = (number - job.first) * RT, tiles = (job.out + 15) / 16;
  const auto wr = wave_rsrc(job.w, static_cast<int>((long)tiles * a.blocks * (1024 + (OFF ? 64 : 32) * GP)));
  __amdgpu_buffer_rsrc_t xr[TERMS];
#pragma unroll
  for (int z = 0; z < TERMS; ++z)
    xr[z] = wave_rsrc(static_cast<const bf16*>(a.x) + ((long)z * a.T + t0) * a.in, 0x7fffffff);
  const int scales = tiles * a.blocks * 1024, offsets = scales + tiles * a.blocks * 32 * GP;
  int x_at[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x_at[n] = (min(16 * n + col, a.T - 1 - t0) * a.in + 8 * g) * 2;
  unsigned char* const ring = smem + kw * C::SLOTS * C::SLOT;
  // operands (n, w), (n, w + RW), .. of the block of a step: this lane's 16 bytes
  auto request = [&](int slot, int step) __attribute__((always_inline)) {
    const int blk = min(step * KW + kw, a.blocks - 1);
#pragma unroll
    for (int i0 = 0; i0 < 4; i0 += RW) {
      const int i = i0 + w, k = 2 * min(128 * blk + 32 * i, a.in - 32);
#pragma unroll
      for (int z = 0; z < TERMS; ++z)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              xr[z], (GLACIER_LDS void*)(ring + slot * C::SLOT + (4 * (NT * z + n) + i) * 1024), 16, x_at[n], k, 0, 0);
    }
  };
  struct Words {
    u32x4 w[RT];
    unsigned s[RT][2 * GP], o[RT][OFF && !C::FOLD ? 2 * GP : 1];
  };
  auto load = [&](Words& to, int step) __attribute__((always_inline)) {
    const int blk = min(step * KW + kw, a.blocks - 1);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int at = min(tile + r, tiles - 1) * a.blocks + blk;
      to.w[r] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, 16 * lane, at * 1024, 0));
      load_u32<2 * GP>(wr, 8 * GP * g, scales + at * 32 * GP, to.s[r]);
      if constexpr (C::FOLD)  // row col, group g
        to.o[r][0] = __builtin_amdgcn_raw_buffer_load_b16(wr, 8 * col + 2 * g, offsets + at * 128, 0);
      else if constexpr (OFF)
        load_u32<2 * GP>(wr, 8 * GP * g, offsets + at * 32 * GP, to.o[r]);
    }
  };
  const QuantMagic magic;
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  f32x4 y[RT][NT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n) y[r][n] = zero;
  bf16x8 minus;  // of sums of x (fp32: 1)
#pragma unroll
  for (int e = 0; e < 8; ++e) minus[e] = (bf16)(TERMS == 1 ? -136.0f : 1.0f);
  const unsigned ring_at = static_cast<unsigned>(reinterpret_cast<uintptr_t>((GLACIER_LDS unsigned char*)ring)) + 16 * lane;
  auto take = [&](const Words& from, unsigned slot_at) __attribute__((always_inline)) {
    u32x4 f[2][NT * TERMS];
    auto read = [&](int i) __attribute__((always_inline)) {
      u32x4(&to)[NT * TERMS] = f[i % 2];
      if constexpr (TERMS == 1 && !C::FOLD) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
          asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(to[n]) : "v"(slot_at), "i"((4 * n + i) * 1024));
      // (else the compiler lets sums pass through the operands' registers: their writes are
      // waited for)
      } else if constexpr (TERMS == 1 && NT == 1) {
        asm volatile("s_nop 7\n\tds_read_b128 %0, %1 offset:%2" : "=&v"(to[0]) : "v"(slot_at), "i"(i * 1024));
      } else if constexpr (TERMS == 1 && NT == 2) {
        asm volatile("s_nop 7\n\tds_read_b128 %0, %2 offset:%3\n\tds_read_b128 %1, %2 offset:%4"
                     : "=&v"(to[0]), "=&v"(to[1])
                     : "v"(slot_at), "i"(i * 1024), "i"((4 + i) * 1024));
      } else if constexpr (TERMS == 1) {
        static_assert(NT == 4, "reads of one, two or four operands");
        asm volatile(
            "s_nop 7\n\tds_read_b128 %0, %4 offset:%5\n\tds_read_b128 %1, %4 offset:%6\n\tds_read_b128 %2, %4 offset:%7\n\t"
            "ds_read_b128 %3, %4 offset:%8"
            : "=&v"(to[0]), "=&v"(to[1]), "=&v"(to[2]), "=&v"(to[3])
            : "v"(slot_at), "i"(i * 1024), "i"((4 + i) * 1024), "i"((8 + i) * 1024), "i"((12 + i) * 1024));
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
          asm volatile(
              "s_nop 7\n\tds_read_b128 %0, %3 offset:%4\n\tds_read_b128 %1, %3 offset:%5\n\tds_read_b128 %2, %3 offset:%6"
              : "=&v"(to[n]), "=&v"(to[NT + n]), "=&v"(to[2 * NT + n])
              : "v"(slot_at), "i"((4 * n + i) * 1024), "i"((4 * (NT + n) + i) * 1024), "i"((4 * (2 * NT + n) + i) * 1024));
      }
    };
    read(0);
    f32x4 d[RT][NT], d0[NT];
    float of_x[NT];  // of group g's columns and token col
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < 3) {
        read(i + 1);
        lgkm<NT * TERMS>();
      } else {
        lgkm<0>();
      }
#pragma unroll
      for (int n = 0; n < NT * TERMS; ++n) tie_v(f[i % 2][n]);
      if (i * GP % 4 == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n) d0[n] = zero;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n) d[r][n] = zero;
      }
      auto add = [&](const bf16x8& wf, f32x4 (&to)[NT]) __attribute__((always_inline)) {  // smallest terms first
#pragma unroll
        for (int z = TERMS - 1; z >= 0; --z)
#pragma unroll
          for (int n = 0; n < NT; ++n) to[n] = Mfma<bf16>::mma(wf, __builtin_bit_cast(bf16x8, f[i % 2][NT * z + n]), to[n]);
      };
      if constexpr (C::SUMS || C::FOLD) add(minus, d0);
      if constexpr (C::FOLD)
#pragma unroll
        for (int n = 0; n < NT; ++n) of_x[n] = i == 0 || g == i ? d0[n][0] : of_x[n];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if constexpr (C::CHAIN) add(minus, d[r]);
        if constexpr (C::FOLD && TERMS == 1)
#pragma unroll
          for (int n = 0; n < NT; ++n) d[r][n] = d0[n];
        if constexpr (TERMS == 1)
          add(raw8_bf16(from.w[r][i], magic), d[r]);
        else
          add(exact8_bf16(from.w[r][i], magic), d[r]);
      }
      if ((i + 1) * GP % 4 == 0) {  // a group's end
        const int q = i * GP / 4;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float s = half_at(from.s[r][(e * GP + q) / 2], (e * GP + q) % 2);
            float o = s;  // of -136 sum(x)
            if constexpr (OFF && !C::FOLD) {
              o = half_at(from.o[r][(e * GP + q) / 2], (e * GP + q) % 2);
              if constexpr (TERMS == 1) o = fmaf(o, -1.0f / 136.0f, s);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              y[r][n][e] = fmaf(s, d[r][n][e], y[r][n][e]);
              if constexpr (C::SUMS) y[r][n][e] = fmaf(o, d0[n][e], y[r][n][e]);
            }
          }
      }
    }
    if constexpr (C::FOLD)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float o = half_at(from.o[r][0], 0) * (TERMS == 1 ? -1.0f / 136.0f : 1.0f);
#pragma unroll
        for (int n = 0; n < NT; ++n) y[r][n] = Mfma<float>::mma(o, of_x[n], y[r][n]);
      }
  };
  // (columns past the last one: x's last ones again, which meet scales of zero)
  const int steps = (a.blocks + KW - 1) / KW;
  Words u, v;
  request(0, 0);
  request(1, 1);
  load(u, 0);
  auto turn = [&](int step, int slot, const Words& now, Words& next) __attribute__((always_inline)) {
    vmw<C::XLOADS + C::WLOADS>();  // this block of x has come, but for what other waves asked for
    wg_barrier();
    request(slot == 0 ? 2 : slot - 1, step + 2);
    load(next, step + 1);
    if (KW == 1 || step * KW + kw < a.blocks) take(now, ring_at + slot * C::SLOT);
  };
  int slot = 0;
  for (int step = 0; step < steps; step += 2) {
    turn(step, slot, u, v);
    slot = slot == 2 ? 0 : slot + 1;
    if (step + 1 >= steps) break;
    turn(step + 1, slot, v, u);
    slot = slot == 2 ? 0 : slot + 1;
  }
  vmw<0>();
  if (job.l != nullptr) {  // (x A) B by fp32 products of four ranks
    const long step = (long)a.T * a.rank;
    for (int j0 = 4 * kw; j0 < a.rank; j0 += 4 * KW) {
      const int j = j0 + g, jc = min(j, a.rank - 1);
      float low[NT], up[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        up[r] = job.b[(long)jc * job.out + min(16 * (tile + r) + col, job.out - 1)];
        up[r] = j < a.rank ? up[r] : 0.0f;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float* const l = job.l + (long)min(t0 + 16 * n + col, a.T - 1) * a.rank + jc;
        low[n] = 0.0f;
#pragma unroll 8
        for (int z = 0; z < a.splits; ++z) low[n] += l[z * step];
        low[n] = j < a.rank ? job.s * low[n] : 0.0f;
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n) y[r][n] = Mfma<float>::mma(up[r], low[n], y[r][n]);
    }
  }
  auto put = [&](int r, int n, f32x4 sum) __attribute__((always_inline)) {
    const int t = t0 + 16 * n + col, o = 16 * (tile + r) + 4 * g;
    if (!has_tile || t >= a.T || o >= job.out) return;
    if (job.bias != nullptr)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += job.bias[o + e];
    store4(static_cast<IO*>(job.y) + (long)t * job.out + o, sum);
  };
  if constexpr (KW == 1) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) put(r, n, y[r][n]);
  } else {
    __syncthreads();
    float* const mine = reinterpret_cast<float*>(smem) + w * (KW * RT * NT * 16 * C::STRIDE) + col * C::STRIDE + 4 * g;
#pragma unroll
    for (int x = 0; x < RT * NT; ++x) store4(mine + (kw * RT * NT + x) * 16 * C::STRIDE, y[x / NT][x % NT]);
    __syncthreads();
#pragma unroll
    for (int x = 0; x < RT * NT; ++x) {
      if (x % KW != kw) continue;
      f32x4 sum = zero;
#pragma unroll
      for (int k = 0; k < KW; ++k) sum += *reinterpret_cast<const f32x4*>(mine + (k * RT * NT + x) * 16 * C::STRIDE);
      put(x / NT, x % NT, sum);
    }
  }
#endif
}

// ---- x A of few tokens -----------------------------------------------------
// Parts of x A_p over columns z kLowCols .. of x and rows of A_p each: [splits][T][rank]
// of every projection.  Of 32 columns a lane holds eight of one token and the eight rows
// of A that go with them, of one rank each: eight fp32 products of four.  The waves'
// sums are added in order.
constexpr int kLowCols = 256, kLowTokens = 16;
struct LowCall {
  const void* x;
  const float* a[kMaxProj];
  float* l[kMaxProj];
  int T, in, rank, splits;
};
template <typename IO, int NR>  // NR: tiles of 16 ranks
__global__ __launch_bounds__(256) void quant_low_kernel(LowCall c) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ __align__(16) float part[4][NR][16][20];
  const int z = blockIdx.x, w = wave_id(), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const float* const a = c.a[blockIdx.y];
  const int t = min(col, c.T - 1);
  float x[2][8], v[2][NR][8];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int k = z * kLowCols + 64 * w + 32 * u, kc = min(k, c.in - 32) + 8 * g;  // (in is a multiple of 32)
    load8(static_cast<const IO*>(c.x) + (long)t * c.in + kc, x[u]);
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int s = 0; s < 8; ++s) v[u][r][s] = a[(long)(kc + s) * c.rank + min(16 * r + col, c.rank - 1)];
    if (k >= c.in)
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        x[u][s] = 0.0f;
#pragma unroll
        for (int r = 0; r < NR; ++r) v[u][r][s] = 0.0f;
      }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int s = 0; s < 8; ++s) sum = Mfma<float>::mma(v[u][r][s], x[u][s], sum);
    store4(part[w][r][col] + 4 * g, sum);  // token col, ranks 16 r + 4 g ..
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 256 * NR; i += 256) {
    const int j = i % 16, at = i / 16 % 16, r = i / 256;
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) sum += part[u][r][at][j];
    if (at < c.T && 16 * r + j < c.rank) c.l[blockIdx.y][((long)z * c.T + at) * c.rank + 16 * r + j] = sum;
  }
#endif
}

// ---- fp32 x in three bf16 terms, [3][T][in] ---------------------------------
// Cut, not rounded: 8 bits a term, so that the three are x exactly and none overflows.
// What is not finite stays in the first.
__global__ __launch_bounds__(256) void quant_terms_kernel(const float* x, bf16* to, long n) {
  for (long i = 8 * ((long)blockIdx.x * 256 + threadIdx.x); i < n; i += 8L * 256 * gridDim.x) {
    float v[8], h[8];
    load8(x + i, v);
#pragma unroll
    for (int z = 0; z < 3; ++z) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool finite = fabsf(v[e]) < INFINITY;
        h[e] = finite ? __uint_as_float(__float_as_uint(v[e]) & 0xffff0000u) : v[e];
        v[e] = finite ? v[e] - h[e] : 0.0f;
      }
      store8(to + z * n + i, h);
    }
  }
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

template <int NT, int RT, int RW, int KW, int GP, bool OFF, int TERMS>
hipError_t tiled(QuantCall c, hipStream_t st) {
  using C = TileCfg<NT, RT, RW, KW, GP, OFF, TERMS>;
  c.token_blocks = (c.T + 16 * NT - 1) / (16 * NT);
  c.tiles = 0;
  for (int p = 0; p < c.n; ++p) {
    c.p[p].first = c.tiles;
    c.tiles += (c.p[p].out + 16 * RT - 1) / (16 * RT);
  }
  const int grid = quant_grid((c.tiles + RW - 1) / RW, c.token_blocks);
  GL_CHECK(allow_lds((&quant_tile_kernel<NT, RT, RW, KW, GP, OFF, TERMS>), C::BYTES));
  hipLaunchKernelGGL((quant_tile_kernel<NT, RT, RW, KW, GP, OFF, TERMS>), dim3(grid),
                     dim3(64 * C::WAVES), C::BYTES, st, c);
  return hipGetLastError();
}
template <int TERMS, int NT, int RT, int RW, int KW>
hipError_t by_group(const QuantCall& c, int group, bool off, hipStream_t st) {
  if (group == 32) return off ? tiled<NT, RT, RW, KW, 4, true, TERMS>(c, st) : tiled<NT, RT, RW, KW, 4, false, TERMS>(c, st);
  if (group == 64) return off ? tiled<NT, RT, RW, KW, 2, true, TERMS>(c, st) : tiled<NT, RT, RW, KW, 2, false, TERMS>(c, st);
  return off ? tiled<NT, RT, RW, KW, 1, true, TERMS>(c, st) : tiled<NT, RT, RW, KW, 1, false, TERMS>(c, st);
}
// The shape of a workgroup, by how many tiles of 16 outputs by 16 tokens a call has: few
// tiles are cut along the columns, many share the operands of x, and the weights, of a
// workgroup.  In us, the shape named RT RW KW after NT, [tokens] in -> outputs:
//   below 512     1: 1 2 4   [1] 3584 -> 4608: 11.0 (with 1 4 4: 13.2, 1 4 1: 18.1);
//                            fp32: 15.6 (18.0, 24.7)
//     and rows of 8192 or more, up to 16 tokens, bf16
//                 1: 1 1 8   [1] 18944 -> 3584: 13.1 (1 2 4: 20.9); [16]: 23.7 (24.7); but
//                            [1] 3584 -> 4608: 16.2.  (fp32's operands would take twice
//                            the LDS that there is)
//   below 1200    1: 1 4 4   [64] 3584 -> 3584: 9.6 (1 2 4: 13.4, 1 4 1: 11.5);
//                            fp32 [32] 3584 -> 4608: 33.0 (45.6, 40.3)
//   below 3000    1: 1 4 1   [16] 3584 -> 37888: 22.3 (1 2 4: 27.5, 1 4 4: 24.6); [128]
//                            3584 -> 3584: 14.4; fp32 [16] 3584 -> 37888: 45.6 (2: 2 4 1:
//                            63.3)
//   more          2: 2 4 1   [24] 3584 -> 37888: 30.9 (1: 1 4 1: 32.9), [512] 4096 -> 6144:
//                            48; fp32 [512] 3584 -> 4608: 121.7 (1: 1 4 1: 143.9)
//   35000 and more, bf16
//                 4: 2 4 1   [256] 3584 -> 37888: 117 (2: 2 4 1: 127), but [200]: 117 (109)
//                            and [103]: 76 (68); [512]: 202 (213; with weights that
//                            are not in the last-level cache 224; 4: 2 8 1 248, 4: 4 2 1
//                            263), but [512] 4096 -> 6144: 55.  690 TFLOP/s: matrix
//                            instructions are busy 41% of the time, vector ones 52%, and
//                            two waves a SIMD, in step, hardly overlap them
template <int TERMS>
hipError_t by_shape(const QuantCall& c, int group, bool off, hipStream_t st) {
  long units = 0;
  for (int p = 0; p < c.n; ++p) units += (c.p[p].out + 15) / 16;
  units *= (c.T + 15) / 16;
  if constexpr (TERMS == 1)
    if (c.T <= 16 && units < 512 && c.blocks >= 64) return by_group<TERMS, 1, 1, 1, 8>(c, group, off, st);
  if (units < 512) return by_group<TERMS, 1, 1, 2, 4>(c, group, off, st);
  if (units < 1200) return by_group<TERMS, 1, 1, 4, 4>(c, group, off, st);
  if (units < 3000) return by_group<TERMS, 1, 1, 4, 1>(c, group, off, st);
  if constexpr (TERMS == 1)
    if (units >= 35000) return by_group<TERMS, 4, 2, 4, 1>(c, group, off, st);
  return by_group<TERMS, 2, 2, 4, 1>(c, group, off, st);
}

template <typename IO>
hipError_t low(const LowCall& c, int n, hipStream_t st) {
  const dim3 grid(c.splits, n);
  if (c.rank <= 16)
    hipLaunchKernelGGL((quant_low_kernel<IO, 1>), grid, dim3(256), 0, st, c);
  else if (c.rank <= 32)
    hipLaunchKernelGGL((quant_low_kernel<IO, 2>), grid, dim3(256), 0, st, c);
  else
    hipLaunchKernelGGL((quant_low_kernel<IO, 4>), grid, dim3(256), 0, st, c);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_quant_pack(const QuantPack& a, hipStream_t st) {
  const QuantLayout l = quant_layout(a.out, a.in, a.group, a.offsets != nullptr);
  const long n = l.scales / 4 + (l.bytes - l.scales) / 2;
  hipLaunchKernelGGL(quant_pack_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, st, a, l);
  return hipGetLastError();
}

int quant_low_splits(int T, int in) { return T <= kLowTokens ? (in + kLowCols - 1) / kLowCols : 1; }

hipError_t launch_quant_proj(const QuantProj& q, int n_cu, hipStream_t st) {
  const ProjLaunch& a = q.a;
  QuantCall c{};
  c.x = a.x;
  c.T = a.T;
  c.in = a.in;
  c.blocks = (a.in + 127) / 128;
  c.rank = a.rank;
  c.splits = quant_low_splits(a.T, a.in);
  c.n = a.n_proj;
  LowCall low_call{a.x, {}, {}, a.T, a.in, a.rank, c.splits};
  float* l[kMaxProj] = {};
  int adapters = 0;
  for (int p = 0; p < a.n_proj; ++p) {
    const ProjSpec& s = a.p[p];
    if (s.a != nullptr) {
      l[p] = q.low + (long)adapters * c.splits * a.T * a.rank;
      low_call.a[adapters] = s.a;
      low_call.l[adapters++] = l[p];
    }
    c.p[p] = QuantSpec{static_cast<const char*>(s.w), s.bias, l[p], s.b, s.scaling, s.out, 0, s.y};
  }
  if (adapters > 0 && a.T <= kLowTokens)
    GL_CHECK(a.io_bf16 ? low<bf16>(low_call, adapters, st) : low<float>(low_call, adapters, st));
  else if (adapters > 0)
    GL_CHECK(launch_lowrank_forward(a, l, st));
  if (a.io_bf16) return by_shape<1>(c, q.group, q.offsets, st);
  const long n = (long)a.T * a.in;
  c.x = q.terms;
  hipLaunchKernelGGL(quant_terms_kernel, dim3(static_cast<unsigned>(std::min((n + 2047) / 2048, 8L * n_cu))), dim3(256), 0,
                     st, static_cast<const float*>(a.x), static_cast<bf16*>(q.terms), n);
  GL_CHECK(hipGetLastError());
  return by_shape<3>(c, q.group, q.offsets, st);
}

}  // namespace glacier
