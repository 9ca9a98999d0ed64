// qcache_attn.hip -- attention of new tokens over a paged cache in 4 bits.
//
// Tiles, splits and the join are those of cache_attn.hip: 16 rows are (token, head of
// the group) pairs of one KV head, a workgroup's four waves take 32 keys at a time in
// turn, each with its own running maximum and sum, joined through LDS at the end.  K
// and V go from the pages into registers and, unpacked there, straight into the
// matrix cores: a word of a page holds what one lane feeds to one MFMA, and pages are
// laid out so that a lane's words lie together.
//
// S^T = K Q^T, 16 keys by 16 rows, 32 columns (one group) at a time.
//   bf16: K as 128 + n (one operation per two elements), the sum begun at -136 sum(q),
//   and the scales applied to the product: S += s (K' q - 136 sum q).  The sums are 17
//   to 136 times the product's terms, which costs 4 to 8 of fp32's 24 bits.
//   fp32: K as n - 8, q in three bf16 terms (24 bits).
// O^T += V^T P^T, 32 tokens at a time.  Two tokens' words, their halves exchanged, hold
// eight columns of both: a lane's words are the operands of eight products (columns 8 x
// + one of 0 .. 7), of four where a head has at most 64 columns (then two lanes take a
// word's halves).
//   V as bf16 (n - 8) s, exact (five bits by three): (16 + n) s - 24 s, where 16 + n is
//   an fp16 value by one OR, formed by fp32 operations that take fp16 operands, of
//   whose results the upper halves are kept.  The weights in two bf16 terms (16 bits of
//   them; fp32: three).
//
// A held value is NaN only by its scale (it is never infinite).  Where a sum is not
// finite the wave walks its keys once more with such scales of V cleared, and gives
// NaN to the rows that see their tokens.
//
// Long chunks: what the batch's sequences hold is written out first, exactly, and
// cache_attn.hip's kernels read that.
#include "cache_tiles.hpp"
#include "quant_page.hpp"

namespace glacier {
namespace {

constexpr int kWavesQ = 4;
[[maybe_unused]] constexpr int kKeysQ = 32;  // keys of a wave's block: one k-step of the second product

template <int G>
struct QaLayout {
  static constexpr int NV = (G + 3) / 4;    // blocks of 16 words of a token of V
  static constexpr bool HALF = G <= 2;      // two lanes share a word
  static constexpr int NB = HALF ? 4 : 8 * NV;  // 16-column products
  static constexpr int DP = 32 * G;
  static constexpr int OS = DP + 4;         // row stride (floats) of a wave's sums in the join
  static constexpr int WAVE = 16 * (OS + 2);
};

// What a wave loads of 32 keys: two tiles of 16.
template <int G>
struct QBlock {
  static constexpr int NV = QaLayout<G>::NV;
  unsigned k[2][G];      // lane (key l % 16, columns 8 (l / 16) .. of each group)
  unsigned ks[2][2 * G];  // scales of keys 4 (l / 16) ..: halves key G + i
  unsigned v[2][NV][4];   // lane (word l % 16 or its pair, tokens 4 (l / 16) ..)
  unsigned vs[2][NV][2];  // their scales
};

#if defined(__HIP_DEVICE_COMPILE__)
template <int N>
__device__ inline void load_words(__amdgpu_buffer_rsrc_t rs, int voff, int soff, unsigned* to) {
  if constexpr (N >= 4) {
    const auto w = __builtin_amdgcn_raw_buffer_load_b128(rs, voff, soff, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = static_cast<unsigned>(w[e]);
    if constexpr (N > 4) load_words<N - 4>(rs, voff + 16, soff, to + 4);
  } else if constexpr (N == 3) {
    const auto w = __builtin_amdgcn_raw_buffer_load_b96(rs, voff, soff, 0);
#pragma unroll
    for (int e = 0; e < 3; ++e) to[e] = static_cast<unsigned>(w[e]);
  } else if constexpr (N == 2) {
    const auto w = __builtin_amdgcn_raw_buffer_load_b64(rs, voff, soff, 0);
    to[0] = static_cast<unsigned>(w[0]), to[1] = static_cast<unsigned>(w[1]);
  } else {
    to[0] = static_cast<unsigned>(__builtin_amdgcn_raw_buffer_load_b32(rs, voff, soff, 0));
  }
}
#endif

// Halves of a register that are NaN, as a mask (scales are never infinite).
[[maybe_unused]] __device__ inline unsigned nan_halves(unsigned w) {
  return ((((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u) >> 15) * 0xffffu;
}

template <typename T, int G>
__global__ __launch_bounds__(64 * kWavesQ, G <= 4 ? 2 : 1) void qcache_attn_kernel(CacheAttn a) {
#if defined(__HIP_DEVICE_COMPILE__)
  using L = QaLayout<G>;
  using B = QBlock<G>;
  constexpr int NV = L::NV, NB = L::NB;
  constexpr bool F32 = sizeof(T) == 4, HALF = L::HALF;
  __shared__ __align__(16) float all[kWavesQ * L::WAVE];
  const CacheView& c = a.c;
  const int w = wave_id(), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const int D = c.D, numbers = static_cast<int>(gridDim.x / (a.n_splits * c.hkv));
  const int kvh = blockIdx.x / a.n_splits % c.hkv;
  const int number = blockIdx.x / (a.n_splits * c.hkv);
  const int split = (blockIdx.x + number) % a.n_splits;
  int tile;
  CacheSeq s;
  if (a.long_first) {
    s = seq_of_long_tile(a, lane, number, numbers, tile);
  } else {
    s = seq_of_tile(a, lane, number);
    tile = number - first_tile(a, s.b, s.tok0);
  }
  const int b = s.b;
  if (b >= c.n_seqs) return;
  const int r0 = tile * 16, n_rows = s.n * a.group;
  if (tile < 0 || r0 >= n_rows) return;
  const TileKeys tk = tile_keys(a, s, tile);
  if (split >= tk.active) return;
  const int k0 = split * tk.per, k1 = min(tk.kend, k0 + tk.per);

  // this lane's row: its last key and its query, columns 32 i + 8 g .. of each group
  const int row = r0 + col, tok = row / a.group, head = kvh * a.group + (row - tok * a.group);
  const bool has_row = row < n_rows;
  const int limit = has_row ? s.pos0 + tok : -1;
  const T* const q = static_cast<const T*>(a.q) +
                     (has_row ? (long)(s.tok0 + tok) * a.hq + head : (long)(s.tok0 + r0 / a.group) * a.hq) * D;
  constexpr int TERMS = F32 ? 3 : 1;
  bf16x8 qf[TERMS][G];
  f32x4 base[F32 ? 1 : G];  // -136 sum(q) of each group
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int at = 32 * i + 8 * g;
    const bool ok = has_row && at < D;
    float x[8];
    load8(q + (at < D ? at : 0), x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = ok ? x[e] : 0.0f;
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        qf[0][i][e] = (bf16)x[e];
        const float r1 = x[e] - (float)qf[0][i][e];
        qf[1][i][e] = (bf16)r1;
        qf[2][i][e] = (bf16)(r1 - (float)qf[1][i][e]);
      }
    } else {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        qf[0][i][e] = (bf16)x[e];
        sum += x[e];
      }
      sum = -136.0f * col_sum_swap(sum);
      base[i] = f32x4{sum, sum, sum, sum};
    }
  }

  const int part_bytes = quant_row_bytes(D) << c.page_shift, words_bytes = (16 * G) << c.page_shift;
  const long head_at = (long)kvh * part_bytes;
  // this lane's places in 16 keys (bytes): words and scales of K and V
  const int k_at = (col * 4 + g) * G * 4, ks_at = 8 * G * g;
  int v_at[NV], vs_at[NV];
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    const int word = min(HALF ? col >> 1 : 16 * x + col, 4 * G - 1);
    v_at[x] = (g * 4 * G + word) * 16;
    vs_at[x] = (g * G + word / 4) * 8;
  }
  const unsigned pick = HALF && (col & 1) ? 0x07060302u : 0x05040100u;  // which halves of a pair of words
  const auto* const table = (const __attribute__((address_space(4))) int32_t*)(
      reinterpret_cast<uintptr_t>(c.table + (long)b * c.table_stride));
  int page[2];  // of the block to be loaded next
  auto look_up = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int key = j + 16 * p;
      const int at = table[min(key >> c.page_shift, c.max_pages - 1)];
      page[p] = key < k1 && static_cast<unsigned>(at) < static_cast<unsigned>(c.n_pages) ? at : -1;
    }
  };
  // loads block j and looks up the wave's next one
  auto load = [&](B& x, int (&here)[2], int j) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int key = j + 16 * p, in_page = key & ((1 << c.page_shift) - 1);
      here[p] = page[p] < 0 ? 0 : min(16, k1 - key);
      const long at = (page[p] < 0 ? 0 : page[p]) * c.page_stride + head_at;
      const int bytes = page[p] < 0 ? 0 : part_bytes;
      const auto kr = wave_rsrc(static_cast<const char*>(c.k_pages) + at, bytes);
      const auto vr = wave_rsrc(static_cast<const char*>(c.v_pages) + at, bytes);
      const int rows = in_page * 16 * G, scales = words_bytes + in_page * 2 * G;
      load_words<G>(kr, k_at, rows, x.k[p]);
      load_words<2 * G>(kr, ks_at, scales, x.ks[p]);
#pragma unroll
      for (int y = 0; y < NV; ++y) {
        load_words<4>(vr, v_at[y], rows, x.v[p][y]);
        load_words<2>(vr, vs_at[y], scales, x.vs[p][y]);
      }
    }
    look_up(j + kWavesQ * kKeysQ);
  };

  f32x4 acc[NB];
  float m, l;
  const int first_limit = s.pos0 + r0 / a.group;  // the tile's first row sees keys up to here
  auto take = [&](B& x, const int (&here)[2], int j, auto careful) __attribute__((always_inline)) {
    const bool whole = j + kKeysQ - 1 <= first_limit && here[0] == 16 && here[1] == 16;
    // S^T: keys 16 p + 4 g + r of this block, row col
    f32x4 st[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      st[p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < G; ++i) {
        f32x4 d;
        if constexpr (F32) {
          const bf16x8 kf = exact8_bf16(x.k[p][i]);
          d = Mfma<bf16>::mma(kf, qf[2][i], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
          d = Mfma<bf16>::mma(kf, qf[1][i], d);
          d = Mfma<bf16>::mma(kf, qf[0][i], d);
        } else {
          d = Mfma<bf16>::mma(raw8_bf16(x.k[p][i]), qf[0][i], base[i]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) st[p][r] = fmaf(half_at(x.ks[p][(r * G + i) / 2], (r * G + i) % 2), d[r], st[p][r]);
      }
    }
    float top = kLeast;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float y = st[p][r] * a.scale_log2;
        if (!whole) {
          const int at = 4 * g + r;
          y = at < here[p] && j + 16 * p + at <= limit ? y : -INFINITY;
        }
        st[p][r] = y;
        top = fmaxf(top, y);
      }
    const float mn = fmaxf(m, col_max_swap(top));
    if (__any(mn != m)) {
      const float alpha = weight(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[n][r] *= alpha;
    }
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        st[p][r] = weight(st[p][r] - mn);
        l += st[p][r];
      }
    // scales of V that count: not those of keys that are not there
    if (!whole) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int n = here[p] - 4 * g;  // of this lane's four tokens
        const unsigned keep0 = n <= 0 ? 0u : n == 1 ? 0xffffu : ~0u, keep1 = n <= 2 ? 0u : n == 3 ? 0xffffu : ~0u;
#pragma unroll
        for (int y = 0; y < NV; ++y) x.vs[p][y][0] &= keep0, x.vs[p][y][1] &= keep1;
      }
    }
    if constexpr (careful()) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int y = 0; y < NV; ++y)
#pragma unroll
          for (int u = 0; u < 2; ++u) x.vs[p][y][u] &= ~nan_halves(x.vs[p][y][u]);
    }
    // O^T += V^T P^T
    constexpr int PT = F32 ? 3 : 2;
    bf16x8 pf[PT];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float rest = st[e / 4][e % 4];
#pragma unroll
      for (int z = 0; z < PT; ++z) {
        pf[z][e] = (bf16)rest;
        rest -= (float)pf[z][e];
      }
    }
    const f16x2 k24 = {(f16)-24.0f, (f16)-24.0f};
#pragma unroll
    for (int y = 0; y < NV; ++y) {
      f16x2 sc[2][2], off[2][2];
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          sc[p][u] = __builtin_bit_cast(f16x2, x.vs[p][y][u]);
          off[p][u] = sc[p][u] * k24;
        }
#pragma unroll
      for (int z = 0; z < (HALF ? 1 : 2); ++z) {
        const unsigned sel = HALF ? pick : z == 0 ? 0x05040100u : 0x07060302u;
        unsigned both[2][2];  // the halves of two tokens' words
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int u = 0; u < 2; ++u) both[p][u] = __builtin_amdgcn_perm(x.v[p][y][2 * u + 1], x.v[p][y][2 * u], sel);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u32x4 vf;
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              // 16 + n: the number in the four bits above 2^-7 of 16
              const unsigned n = both[p][u];
              const unsigned at = e == 0 ? n << 6 : e == 1 ? n << 2 : e == 2 ? n >> 2 : n >> 6;
              const f16x2 h = __builtin_bit_cast(f16x2, (at & 0x03c003c0u) | 0x4c004c00u);
              vf[2 * p + u] = upper_pair(fmaf((float)h[0], (float)sc[p][u][0], (float)off[p][u][0]),
                                         fmaf((float)h[1], (float)sc[p][u][1], (float)off[p][u][1]));
            }
          const int n = 8 * y + 4 * z + e;
#pragma unroll
          for (int t = PT - 1; t >= 0; --t) acc[n] = Mfma<bf16>::mma(__builtin_bit_cast(bf16x8, vf), pf[t], acc[n]);
        }
      }
    }
  };
  auto walk = [&](auto careful) __attribute__((always_inline)) {
    m = kLeast;
    l = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int STEP = kWavesQ * kKeysQ;
    B x, y;
    int here_x[2], here_y[2];
    int j = k0 + w * kKeysQ;
    if (j < k1) {
      look_up(j);
      load(x, here_x, j);
    }
    for (; j < k1; j += 2 * STEP) {  // two blocks a turn, each loaded while the other is worked on
      if (j + STEP < k1) load(y, here_y, j + STEP);
      take(x, here_x, j, careful);
      if (j + STEP >= k1) break;
      if (j + 2 * STEP < k1) load(x, here_x, j + 2 * STEP);
      take(y, here_y, j + STEP, careful);
    }
  };
  walk(std::false_type{});
  unsigned odd = 0;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) odd |= has_row ? not_finite(acc[n][r]) : 0;
  if (__any(odd != 0)) {
    walk(std::true_type{});
    // a lane's sums of one block belong to one group of columns
    for (int j = k0 + w * kKeysQ; j < k1; j += kWavesQ * kKeysQ)
      for (int key = j; key < min(k1, j + kKeysQ); ++key) {
        const int at = cache_page(c, b, key);
        if (at < 0) continue;
        const f16* const scales = reinterpret_cast<const f16*>(static_cast<const char*>(c.v_pages) + at * c.page_stride +
                                                               head_at + words_bytes);
#pragma unroll
        for (int y = 0; y < NV; ++y) {
          const int i = min(HALF ? g >> 1 : 4 * y + g, G - 1);
          const f16 x = scales[v_scale(key & ((1 << c.page_shift) - 1), G, i)];
          if (x != x && key <= limit)
#pragma unroll
            for (int n = 0; n < (HALF ? 4 : 8); ++n)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[8 * y + n][r] = NAN;
        }
      }
  }

  // join the waves: region of wave u: sums [16][OS], maxima [16], totals [16]
  float* const mine = all + w * L::WAVE;
  const float total_w = col_sum_swap(l);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if constexpr (HALF) {
      if (r % 2) continue;  // rows 4 g + r and + 1 of the products are a word's two halves
      const int word = 2 * g + r / 2;
      if (word >= 4 * G) continue;
      store4(mine + col * L::OS + 8 * word, f32x4{acc[0][r], acc[0][r + 1], acc[1][r], acc[1][r + 1]});
      store4(mine + col * L::OS + 8 * word + 4, f32x4{acc[2][r], acc[2][r + 1], acc[3][r], acc[3][r + 1]});
    } else {
#pragma unroll
      for (int y = 0; y < NV; ++y) {
        const int word = 16 * y + 4 * g + r;
        if (word >= 4 * G) continue;
        const f32x4* const u = acc + 8 * y;
        store4(mine + col * L::OS + 8 * word, f32x4{u[0][r], u[4][r], u[1][r], u[5][r]});
        store4(mine + col * L::OS + 8 * word + 4, f32x4{u[2][r], u[6][r], u[3][r], u[7][r]});
      }
    }
  }
  if (g == 0) {
    mine[16 * L::OS + col] = m;
    mine[16 * (L::OS + 1) + col] = total_w;
  }
  __syncthreads();
  constexpr int CPR = L::DP / 4;
  for (int idx = threadIdx.x; idx < 16 * CPR; idx += 64 * kWavesQ) {
    const int at_row = idx / CPR, d = 4 * (idx % CPR), r = r0 + at_row;
    if (r >= n_rows || d >= D) continue;
    float mx = kLeast;
#pragma unroll
    for (int u = 0; u < kWavesQ; ++u) mx = fmaxf(mx, all[u * L::WAVE + 16 * L::OS + at_row]);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float total = 0.0f;
#pragma unroll
    for (int u = 0; u < kWavesQ; ++u) {
      const float* reg = all + u * L::WAVE;
      const float f = weight(reg[16 * L::OS + at_row] - mx);
      total += f * reg[16 * (L::OS + 1) + at_row];
      const f32x4 v = *reinterpret_cast<const f32x4*>(reg + at_row * L::OS + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += f * v[e];
    }
    const int i = r / a.group, h = kvh * a.group + (r - i * a.group);
    const long t = s.tok0 + i, at = t * a.hq + h;
    if (tk.active > 1) {
      const long slot = (long)split * c.T * a.hq + at;
      store4(a.part_o + slot * D + d, o);
      if (d == 0) a.part_ml[slot] = make_float2(mx, total);
      continue;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;  // no key: the row is zero
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    store4(static_cast<T*>(a.out) + at * D + d, o);
    if (a.lse != nullptr && d == 0)
      a.lse[(long)h * c.T + t] = total == 0.0f ? -INFINITY : (mx + log2f(total)) * kLn2;
  }
#endif
}

// ---- pages written out -----------------------------------------------------
// What sequence b's pages hold, into pages b max_pages + i of a cache of IO, and
// that cache's table.  A workgroup takes one page of one KV head; rows past the
// sequence's end are not written (the attention does not read them).
constexpr int kExpandThreads = 256;
template <typename IO, int G>
__global__ __launch_bounds__(kExpandThreads) void qcache_expand_kernel(CacheView c, IO* k, IO* v, int32_t* table,
                                                                       int pages) {
  const int i = blockIdx.x % pages, kvh = blockIdx.x / pages % c.hkv, b = blockIdx.x / pages / c.hkv;
  const int first = i << c.page_shift, keys = min(c.kv_lens[b] - first, 1 << c.page_shift);
  const bool fresh = clamp_row(c.cu[b + 1], c.T) > clamp_row(c.cu[b], c.T);  // it has new tokens to attend
  const int page = fresh && keys > 0 ? cache_page(c, b, first) : -1;
  const long to = (long)b * pages + i;
  if (kvh == 0 && threadIdx.x == 0) table[to] = page < 0 ? -1 : static_cast<int>(to);
  if (page < 0) return;
  const long part_bytes = (long)quant_row_bytes(c.D) << c.page_shift, from = page * c.page_stride + kvh * part_bytes;
  const char* const kp = static_cast<const char*>(c.k_pages) + from;
  const char* const vp = static_cast<const char*>(c.v_pages) + from;
  const long words_bytes = (16L * G) << c.page_shift, at = (to * c.hkv + kvh) * ((long)c.D << c.page_shift);
  const int per_row = c.D / 8;
  for (int x = threadIdx.x; x < keys * per_row; x += kExpandThreads) {
    const int row = x / per_row, col8 = x % per_row;
    float y[8];
    dequantise8(reinterpret_cast<const unsigned*>(kp)[k_word(row, G, col8)],
                (float)reinterpret_cast<const f16*>(kp + words_bytes)[k_scale(row, G, col8 / 4)], y);
    store8(k + at + (long)row * c.D + 8 * col8, y);
    dequantise8(reinterpret_cast<const unsigned*>(vp)[v_word(row, G, col8)],
                (float)reinterpret_cast<const f16*>(vp + words_bytes)[v_scale(row, G, col8 / 4)], y);
    store8(v + at + (long)row * c.D + 8 * col8, y);
  }
}

template <typename T, int G>
hipError_t attend(const CacheAttn& a, hipStream_t st) {
  hipLaunchKernelGGL((qcache_attn_kernel<T, G>), dim3(tile_numbers(a) * a.c.hkv * a.n_splits), dim3(64 * kWavesQ), 0,
                     st, a);
  return hipGetLastError();
}
template <typename T, int G>
hipError_t expand(const CacheView& c, void* k, void* v, int32_t* table, hipStream_t st) {
  hipLaunchKernelGGL((qcache_expand_kernel<T, G>), dim3((unsigned)((long)c.n_seqs * c.hkv * c.max_pages)),
                     dim3(kExpandThreads), 0, st, c, static_cast<T*>(k), static_cast<T*>(v), table, c.max_pages);
  return hipGetLastError();
}
#define GL_BY_GROUPS(F, D, io_bf16, ...)                                                   \
  switch (quant_groups(D)) {                                                               \
    case 1: return io_bf16 ? F<bf16, 1>(__VA_ARGS__) : F<float, 1>(__VA_ARGS__);           \
    case 2: return io_bf16 ? F<bf16, 2>(__VA_ARGS__) : F<float, 2>(__VA_ARGS__);           \
    case 3: return io_bf16 ? F<bf16, 3>(__VA_ARGS__) : F<float, 3>(__VA_ARGS__);           \
    case 4: return io_bf16 ? F<bf16, 4>(__VA_ARGS__) : F<float, 4>(__VA_ARGS__);           \
    case 6: return io_bf16 ? F<bf16, 6>(__VA_ARGS__) : F<float, 6>(__VA_ARGS__);           \
    default: return io_bf16 ? F<bf16, 8>(__VA_ARGS__) : F<float, 8>(__VA_ARGS__);          \
  }
hipError_t attend_any(const CacheAttn& a, hipStream_t st) { GL_BY_GROUPS(attend, a.c.D, a.c.io_bf16, a, st) }
hipError_t expand_any(const CacheView& c, void* k, void* v, int32_t* table, hipStream_t st) {
  GL_BY_GROUPS(expand, c.D, c.io_bf16, c, k, v, table, st)
}

constexpr size_t up256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

QCachePlan qcache_attn_plan(const CacheView& c, int hq, int max_new, int max_kv, int n_cu) {
  QCachePlan p{};
  p.attn = cache_attn_plan(c, hq, max_new, max_kv, n_cu);
  // Expanded pages lie in the workspace for whatever the table's rows can name (max_kv
  // is a hint only): up to 2^30 bytes of K and V, else tiles of 16 rows read the 4-bit
  // pages however long the chunks are.
  const size_t k_bytes = (size_t)c.n_seqs * c.max_pages * c.hkv * ((size_t)c.D << c.page_shift) * (c.io_bf16 ? 2 : 4);
  p.expand = p.attn.rows > 16 && k_bytes <= (size_t)1 << 29;
  if (p.expand) {
    p.k_bytes = up256(k_bytes);
    p.table_bytes = up256(sizeof(int32_t) * c.n_seqs * c.max_pages);
    p.bytes = 2 * p.k_bytes + p.table_bytes + p.attn.bytes;
    return p;
  }
  const long group = hq / c.hkv, cap = (long)c.max_pages << c.page_shift;
  const long keys = max_kv > 0 && max_kv < cap ? max_kv : cap;
  const long seqs = std::min(c.T, c.n_seqs);
  const long tiles = seqs * ((c.T * group + seqs * 16 - 1) / (seqs * 16));
  p.attn.rows = 16;
  p.attn.long_first = false;
  const long want = 4L * n_cu / std::max(1L, tiles * c.hkv);
  const long most = keys <= 1024 ? 1 : keys / 512;
  const long launch = (1L << 22) / ((long)c.n_seqs * c.hkv);
  p.attn.n_splits = static_cast<int>(std::max(1L, std::min({want, most, (long)kMaxSplits, launch})));
  const long even = (keys + p.attn.n_splits - 1) / p.attn.n_splits;
  p.attn.split_keys = static_cast<int>((even + kSplitUnit - 1) / kSplitUnit * kSplitUnit);
  const size_t rows = (size_t)c.T * hq;
  p.attn.bytes = p.attn.n_splits > 1 ? p.attn.n_splits * rows * (c.D * sizeof(float) + sizeof(float2)) : 0;
  p.bytes = p.attn.bytes;
  return p;
}

hipError_t launch_qcache_attn(const CacheAttn& a, const QCachePlan& plan, void* workspace, hipStream_t st) {
  CacheAttn x = a;
  char* at = static_cast<char*>(workspace);
  if (plan.expand) {
    x.c.k_pages = at;
    x.c.v_pages = at + plan.k_bytes;
    int32_t* const table = reinterpret_cast<int32_t*>(at + 2 * plan.k_bytes);
    at += 2 * plan.k_bytes + plan.table_bytes;
    GL_CHECK(expand_any(a.c, x.c.k_pages, x.c.v_pages, table, st));
    x.c.page_stride = (long)a.c.hkv * ((long)a.c.D << a.c.page_shift);
    x.c.n_pages = a.c.n_seqs * a.c.max_pages;
    x.c.table = table;
    x.c.table_stride = a.c.max_pages;
  }
  if (x.n_splits > 1) {
    x.part_o = reinterpret_cast<float*>(at);
    x.part_ml = reinterpret_cast<float2*>(x.part_o + (size_t)x.n_splits * x.c.T * x.hq * x.c.D);
  }
  if (plan.expand) return launch_cache_attn(x, st);
  GL_CHECK(attend_any(x, st));
  return x.n_splits == 1 ? hipSuccess : launch_cache_join(x, st);
}

}  // namespace glacier
