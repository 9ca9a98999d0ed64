// cache_attn.hip -- attention of new tokens over a paged key/value cache.
//
// The query heads of a KV head's group read the same keys, so a tile's rows
// are (token, head of the group) pairs, token by token: row r of a sequence is
// token r / group, head r % group.  One new token of 7 heads and a long chunk
// are then the same product, and K and V are read once per tile, not per head.
//
// A workgroup takes one tile of 16 or 32 rows of one KV head, and one split of the
// keys the tile sees.  Its waves (four; eight in fp32 up to 128 columns) take keys
// in turn, KB at a time, each with its own LDS tiles and its own running maximum
// and sum of the softmax, so the loop has no barrier; the waves are joined
// through LDS at the end.  Scores are formed
// transposed (S^T = K Q^T, attn_common.hpp), which leaves a lane with
// one row's weights and feeds them to O^T += V^T P^T as they are.
//
// Bound by reading K and V for single tokens: one over 65536 keys, 32/8 heads of
// 128, bf16, 57.4 us (4.67 TB/s of the 4.77 of a large copy); 32 sequences of up to
// 8192 keys, 28/4 heads, 64-65 us (4.3 TB/s, uneven splits); heads of 64 and 256 less
// (8 sequences of up to 16000 keys, 14/2 of 64, 16 us, 2.2 TB/s; 6 of up to 9000, 8/2 of
// 256, 24 us, 3.6); one over 512 keys, 14/2 heads of 64, 6.8 us: four dependent loads
// and four blocks of keys.  Long fp32 chunks are bound by the fp32 MFMAs (1024 tokens
// over 8192 keys, 8/2 heads of 96: 226 us, 107 TFLOP/s of the 154 of a large library
// product; MFMAs busy 66% of the card's cycles), short ones by one workgroup a CU that
// waits for its own loads and LDS (three of up to 120 over up to 1001: 22-23 us on 138
// of the 256 CUs, MFMAs busy 23 thousand cycles there of about 57 thousand; 18% of the
// LDS cycles are bank conflicts).
//
// KV heads alternate over the workgroups, so that an XCD's L2 serves few of them
// (fp32, 16 sequences of up to 8000 keys, one token each: 93 -> 70 us; 512 tokens
// over 4096 keys 375 -> 365; 2 of up to 900 over up to 3000, 8/8 heads of 64: 100 ->
// 81).  In bf16 the splits of a tile alternate first, each tile's from another one
// on: an XCD then gets long and short tiles, first and last splits alike (single
// tokens: 24 sequences of up to 8000 keys, 32/8 heads of 128, 100 -> 93; 32 of up to
// 8192, 28/4, 67.7 -> 65.1).  fp32, with one workgroup a CU, loses by it where an XCD
// gets one more than it has CUs (6 chunks of up to 30 over up to 4000, 12/2 heads of
// 128: 50 -> 71).
//
// A tile's splits write sums and (maximum, sum) to the workspace, and a second
// launch joins them; a tile with one split writes its result itself.
//
// Which tiles exist, which keys they see and how these are split follows from
// device data (cu_tokens, kv_lens) by the same formulas in both launches; the
// grid covers every batch of the call's size, and workgroups without work leave.
#include "cache_tiles.hpp"

namespace glacier {
namespace {

template <typename T>
struct KeyBlock;
template <>
struct KeyBlock<bf16> {
  static constexpr int KB = 32;  // one k-step of the PV product
};
template <>
struct KeyBlock<float> {
  static constexpr int KB = 16;  // two blocks of 256 columns and their copies fit the LDS
};

template <typename T, int DP, int MB, int WAVES>
struct CaLayout {
  static constexpr int KB = KeyBlock<T>::KB;
  static constexpr int S = Lds<T, DP>::STRIDE;
  static constexpr int TILES = WAVES * 2 * KB * S * static_cast<int>(sizeof(T));
  static constexpr int OS = DP + 4;  // row stride (floats) of a wave's sums in the join
  static constexpr int WAVE = 16 * MB * (OS + 2);  // sums, maxima, totals
  static constexpr int JOIN = WAVES * WAVE * 4;
  static constexpr int NOTES = TILES > JOIN ? TILES : JOIN;  // then the noted blocks of each wave
  static constexpr int BYTES = NOTES + WAVES * kNotedBlocks / 8;
  static_assert(BYTES <= 160 * 1024, "exceeds the LDS of a CU");
};

// KB rows of a K or V block in registers between global memory and LDS.
template <typename T, int DP>
struct BlockRegs {
  static constexpr int KB = KeyBlock<T>::KB;
  static constexpr int CE = 16 / sizeof(T);
  static constexpr int CPR = DP / CE;
  static constexpr int LPR = CPR <= 4 ? 4 : CPR <= 8 ? 8 : CPR <= 16 ? 16 : CPR <= 32 ? 32 : 64;
  static constexpr int RPI = 64 / LPR;  // rows per instruction, at most 16
  static constexpr int N = KB / RPI;
  i32x4 w[N];
  // 16 rows of each page piece from base[piece], of which rows[piece] hold
  // keys; rows past them and columns past D arrive as zero (load_within).
  // off: this lane's row lane / LPR and column, in bytes
  __device__ inline void load(const char* const (&base)[KB / 16], const int (&rows)[KB / 16], int rowb,
                              int off) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      constexpr int P = 16 / RPI;  // loads of a piece
      w[i] = load_within(base[i / P], rows[i / P] * rowb, off + i % P * RPI * rowb);
    }
  }
  __device__ inline void store(T* lds, int lane) const {
    const int ch = lane % LPR;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (LPR == CPR || ch < CPR)
        *reinterpret_cast<i32x4*>(lds + (i * RPI + lane / LPR) * Lds<T, DP>::STRIDE + ch * CE) = w[i];
  }
};

template <typename T, int DP, int MB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void cache_attn_kernel(CacheAttn a) {
  using M = Mfma<T>;
  using L = CaLayout<T, DP, MB, WAVES>;
  constexpr int KB = L::KB, NS = KB / 16, ROWS = 16 * MB;
  constexpr int NW = DP * sizeof(T) / 64;  // 16-byte words a lane holds of a row
  extern __shared__ __align__(16) unsigned char smem[];
  const CacheView& c = a.c;
  const int w = wave_id(), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const int D = c.D, numbers = static_cast<int>(gridDim.x / (a.n_splits * c.hkv));
  int kvh, split, number;
  if constexpr (sizeof(T) == 2) {
    kvh = blockIdx.x / a.n_splits % c.hkv;
    number = blockIdx.x / (a.n_splits * c.hkv);
    split = (blockIdx.x + number) % a.n_splits;
  } else {
    kvh = blockIdx.x % c.hkv;
    number = blockIdx.x / c.hkv % numbers;
    split = blockIdx.x / (c.hkv * numbers);
  }
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
  const int r0 = tile * ROWS, n_rows = s.n * a.group;
  if (tile < 0 || r0 >= n_rows) return;
  const TileKeys tk = tile_keys(a, s, tile);
  if (split >= tk.active) return;
  const int k0 = split * tk.per, k1 = min(tk.kend, k0 + tk.per);

  // this lane's rows (one per 16-row block): operand fragments and last key
  i32x4 qw[MB][NW];
  int limit[MB];
  // the first of the 16 bytes of columns that this lane holds in word x of a
  // row of Q or K: one k-step's 8 columns in bf16; in fp32, where a k-step takes
  // one column a lane, those of four steps (step 4 x + e takes column
  // 16 x + 4 g + e: a dot product may take its terms in any order)
  auto first_col = [&](int x) { return sizeof(T) == 2 ? 32 * x + 8 * g : 16 * x + 4 * g; };
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int r = r0 + 16 * mb + col;
    const int i = r / a.group, h = kvh * a.group + (r - i * a.group);
    const bool ok = r < n_rows;
    limit[mb] = ok ? s.pos0 + i : -1;
    // (loaded from the tile's first row where there is none, and cleared after
    // all loads are under way)
    const T* q = static_cast<const T*>(a.q) +
                 (ok ? (long)(s.tok0 + i) * a.hq + h : (long)(s.tok0 + r0 / a.group) * a.hq) * D;
#pragma unroll
    for (int x = 0; x < NW; ++x)
      qw[mb][x] = *reinterpret_cast<const i32x4*>(q + (first_col(x) < D ? first_col(x) : 0));
  }
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int x = 0; x < NW; ++x)
      if (limit[mb] < 0 || first_col(x) >= D) qw[mb][x] = i32x4{0, 0, 0, 0};

  f32x4 acc[MB][DP / 16];
  float m[MB], l[MB];

  T* const kt = reinterpret_cast<T*>(smem) + w * 2 * KB * L::S;
  T* const vt = kt + KB * L::S;
  BlockRegs<T, DP> kr, vr;
  using R = BlockRegs<T, DP>;
  const int rowb = D * static_cast<int>(sizeof(T));
  const int off = lane % R::LPR * R::CE < D ? lane / R::LPR * rowb + lane % R::LPR * 16 : 1 << 20;
  const long head = ((long)kvh << c.page_shift) * rowb, strideb = c.page_stride * sizeof(T);
  // The pages of a block are looked up a block before its rows are requested, by
  // scalar loads (a vector load would wait for the rows in flight).
  const auto* const table = (const __attribute__((address_space(4))) int32_t*)(
      reinterpret_cast<uintptr_t>(c.table + (long)b * c.table_stride));
  int page[NS];  // of the block to be fetched next
  auto look_up = [&](int j) {
#pragma unroll
    for (int p = 0; p < NS; ++p) {
      const int key = j + 16 * p;
      const int at = table[min(key >> c.page_shift, c.max_pages - 1)];
      page[p] = key < k1 && static_cast<unsigned>(at) < static_cast<unsigned>(c.n_pages) ? at : -1;
    }
  };
  int rows[NS];  // keys of the fetched block's pieces
  auto fetch = [&](int j) {
    const char *kb[NS], *vb[NS];
#pragma unroll
    for (int p = 0; p < NS; ++p) {
      const int key = j + 16 * p;
      rows[p] = page[p] < 0 ? 0 : min(16, k1 - key);
      const long at = (page[p] < 0 ? 0 : page[p]) * strideb + head + (key & ((1 << c.page_shift) - 1)) * rowb;
      kb[p] = static_cast<const char*>(c.k_pages) + at;
      vb[p] = static_cast<const char*>(c.v_pages) + at;
    }
    kr.load(kb, rows, rowb, off);
    vr.load(vb, rows, rowb, off);
    look_up(j + WAVES * KB);
  };
  const int first_limit = s.pos0 + r0 / a.group;  // the tile's first row sees keys up to here
  unsigned* const notes = reinterpret_cast<unsigned*>(smem + L::NOTES) + w * (kNotedBlocks / 32);
  auto note_of = [&](int j) { return (j - k0) / (WAVES * KB) % kNotedBlocks; };
  auto walk = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      m[mb] = kLeast;
      l[mb] = 0.0f;
#pragma unroll
      for (int db = 0; db < DP / 16; ++db) acc[mb][db] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int j = k0 + w * KB;
    if (j < k1) {
      look_up(j);
      fetch(j);
    }
    for (; j < k1; j += WAVES * KB) {
      int here[NS];
      bool whole = j + KB - 1 <= first_limit;
#pragma unroll
      for (int p = 0; p < NS; ++p) {
        here[p] = rows[p];
        whole = whole && rows[p] == 16;
      }
      if constexpr (careful()) {
        unsigned found = 0;
#pragma unroll
        for (int i = 0; i < R::N; ++i) found |= clear_not_finite<T>(vr.w[i]);
        if (__any(found != 0) && lane == 0) notes[note_of(j) / 32] |= 1u << note_of(j) % 32;
      }
      wave_lds_order();
      kr.store(kt, lane);
      vr.store(vt, lane);
      wave_lds_order();
      if (j + WAVES * KB < k1) fetch(j + WAVES * KB);
      // S^T: keys 16 p + 4 g + r of this block, row col of each 16-row block
      f32x4 st[MB][NS];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int p = 0; p < NS; ++p) st[mb][p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int p = 0; p < NS; ++p)
#pragma unroll
        for (int x = 0; x < NW; ++x) {
          const i32x4 kw = *reinterpret_cast<const i32x4*>(kt + (16 * p + col) * L::S + first_col(x));
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) {
            if constexpr (sizeof(T) == 2) {
              st[mb][p] = M::mma(__builtin_bit_cast(bf16x8, kw), __builtin_bit_cast(bf16x8, qw[mb][x]), st[mb][p]);
            } else {
              const f32x4 kf = __builtin_bit_cast(f32x4, kw), qf = __builtin_bit_cast(f32x4, qw[mb][x]);
#pragma unroll
              for (int e = 0; e < 4; ++e) st[mb][p] = M::mma(kf[e], qf[e], st[mb][p]);
            }
          }
        }
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        float top = kLeast;
#pragma unroll
        for (int p = 0; p < NS; ++p)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float x = st[mb][p][r] * a.scale_log2;
            if (!whole) {
              const int at = 4 * g + r;
              x = at < here[p] && j + 16 * p + at <= limit[mb] ? x : -INFINITY;
            }
            st[mb][p][r] = x;
            top = fmaxf(top, x);
          }
        const float mn = fmaxf(m[mb], col_max_swap(top));
        const float alpha = weight(m[mb] - mn);
        m[mb] = mn;
        float sum = 0.0f;
#pragma unroll
        for (int p = 0; p < NS; ++p)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = weight(st[mb][p][r] - mn);
            st[mb][p][r] = e;
            sum += e;
          }
        l[mb] = l[mb] * alpha + sum;
#pragma unroll
        for (int db = 0; db < DP / 16; ++db)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[mb][db][r] *= alpha;
      }
      // O^T += V^T P^T; in bf16 each weight in two terms, which leaves 16 bits of
      // it: reading V bounds these calls, and one term would add as much error as
      // the result's own rounding
      if constexpr (sizeof(T) == 2) {
        bf16x8 hi[MB], lo[MB];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p = st[mb][e < 4 ? 0 : NS - 1][e % 4];
            hi[mb][e] = (bf16)p;
            lo[mb][e] = (bf16)(p - (float)hi[mb][e]);
          }
        // (two blocks at a time: a product waits for the one before it on its sums)
#pragma unroll
        for (int db = 0; db < DP / 16; db += 2) {
          bf16x8 vf[2];
#pragma unroll
          for (int x = 0; x < 2; ++x)
            vf[x] = join8(read_tr<L::S>(vt, 0, 16 * (db + x), lane), read_tr<L::S>(vt, 16, 16 * (db + x), lane));
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
            for (int x = 0; x < 2; ++x) acc[mb][db + x] = M::mma(vf[x], lo[mb], acc[mb][db + x]);
#pragma unroll
            for (int x = 0; x < 2; ++x) acc[mb][db + x] = M::mma(vf[x], hi[mb], acc[mb][db + x]);
          }
        }
      } else {
        // V in wide reads: row i of the four blocks 4 x .. 4 x + 3 is column
        // 64 x + 4 i + their number, and of a last pair 64 x + 2 i + its number
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float* const vrow = vt + (4 * g + r) * L::S;
#pragma unroll
          for (int x = 0; x < DP / 64; ++x) {
            const f32x4 vf = *reinterpret_cast<const f32x4*>(vrow + 64 * x + 4 * col);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int mb = 0; mb < MB; ++mb)
                acc[mb][4 * x + e] = M::mma(vf[e], st[mb][0][r], acc[mb][4 * x + e]);
          }
          if constexpr (DP % 64 != 0) {
            const float2 vf = *reinterpret_cast<const float2*>(vrow + DP / 64 * 64 + 2 * col);
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
              acc[mb][DP / 16 - 2] = M::mma(vf.x, st[mb][0][r], acc[mb][DP / 16 - 2]);
              acc[mb][DP / 16 - 1] = M::mma(vf.y, st[mb][0][r], acc[mb][DP / 16 - 1]);
            }
          }
        }
      }
    }
  };
  walk(std::false_type{});
  unsigned odd = 0;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int db = 0; db < DP / 16; ++db)
#pragma unroll
      for (int r = 0; r < 4; ++r) odd |= limit[mb] >= 0 ? not_finite(acc[mb][db][r]) : 0;
  if (__any(odd != 0)) {
    if (lane < kNotedBlocks / 32) notes[lane] = 0;
    wave_lds_order();
    walk(std::true_type{});
    wave_lds_order();
    for (int j = k0 + w * KB; j < k1; j += WAVES * KB) {
      if (!(notes[note_of(j) / 32] >> note_of(j) % 32 & 1)) continue;
      for (int key = j; key < min(k1, j + KB); ++key) {
        const int page = cache_page(c, b, key);
        if (page < 0) continue;
        const char* const v = static_cast<const char*>(c.v_pages) + page * strideb + head +
                              (key & ((1 << c.page_shift) - 1)) * rowb;
        unsigned sees[MB];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) sees[mb] = key <= limit[mb] ? ~0u : 0u;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int db = 0; db < DP / 16; ++db) {
            const bf16x4 x = __builtin_bit_cast(bf16x4, load8_within(v, rowb, 2 * (16 * db + 4 * g)));
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int mb = 0; mb < MB; ++mb) acc[mb][db][r] += given_back((float)x[r], sees[mb]);
          }
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int x = 0; x < DP / 64; ++x) {
              const f32x4 f = __builtin_bit_cast(f32x4, load_within(v, rowb, 4 * (64 * x + 16 * g + 4 * r)));
#pragma unroll
              for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) acc[mb][4 * x + e][r] += given_back(f[e], sees[mb]);
            }
            if constexpr (DP % 64 != 0) {
              const float2 f =
                  __builtin_bit_cast(float2, load8_within(v, rowb, 4 * (DP / 64 * 64 + 8 * g + 2 * r)));
#pragma unroll
              for (int mb = 0; mb < MB; ++mb) {
                acc[mb][DP / 16 - 2][r] += given_back(f.x, sees[mb]);
                acc[mb][DP / 16 - 1][r] += given_back(f.y, sees[mb]);
              }
            }
          }
        }
      }
    }
  }

  // join the waves: region of wave u: sums [ROWS][OS], maxima [ROWS], totals [ROWS]
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(smem) + w * L::WAVE;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const float total = col_sum_swap(l[mb]);
    const int row = 16 * mb + col;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int db = 0; db < DP / 16; ++db)
        store4(mine + row * L::OS + 16 * db + 4 * g, acc[mb][db]);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int x = 0; x < DP / 64; ++x) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[mb][4 * x + e][r];
          store4(mine + row * L::OS + 64 * x + 16 * g + 4 * r, v);
        }
        if constexpr (DP % 64 != 0)
          *reinterpret_cast<float2*>(mine + row * L::OS + DP / 64 * 64 + 8 * g + 2 * r) =
              make_float2(acc[mb][DP / 16 - 2][r], acc[mb][DP / 16 - 1][r]);
      }
    }
    if (g == 0) {
      mine[ROWS * L::OS + row] = m[mb];
      mine[ROWS * (L::OS + 1) + row] = total;
    }
  }
  __syncthreads();
  const float* const all = reinterpret_cast<const float*>(smem);
  constexpr int CPR = DP / 4;
  for (int idx = threadIdx.x; idx < ROWS * CPR; idx += 64 * WAVES) {
    const int row = idx / CPR, d = 4 * (idx % CPR), r = r0 + row;
    if (r >= n_rows || d >= D) continue;
    float mx = kLeast;
#pragma unroll
    for (int u = 0; u < WAVES; ++u) mx = fmaxf(mx, all[u * L::WAVE + ROWS * L::OS + row]);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float total = 0.0f;
#pragma unroll
    for (int u = 0; u < WAVES; ++u) {
      const float* reg = all + u * L::WAVE;
      const float f = weight(reg[ROWS * L::OS + row] - mx);
      total += f * reg[ROWS * (L::OS + 1) + row];
      const f32x4 v = *reinterpret_cast<const f32x4*>(reg + row * L::OS + d);
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
}

// Sum and maximum over a wave's lanes, pair by pair (lanes_sum, swap_sum): no LDS.
__device__ inline float lanes_total(float x) { return col_sum_swap(lanes_sum<16>(x)); }
__device__ inline float lanes_most(float x) {
  auto of = [](float y, float z) { return fmaxf(y, z); };
  x = of(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xB1, 0xF, 0xF, false)));
  x = of(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x4E, 0xF, 0xF, false)));
  x = of(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x141, 0xF, 0xF, false)));
  x = of(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x140, 0xF, 0xF, false)));
  return col_max_swap(x);
}

// Joins the splits of a row.  A split's sums take ceil(D / 4) lanes of 4
// columns, so a wave reads several splits at once where D <= 128, and up to
// eight such loads are in flight.  WAVES waves share a row (1: few splits; 4:
// many, so that 64 splits are one round of loads deep: one wave for them all
// took 20 us of a 77 us call).
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void cache_attn_join_kernel(CacheAttn a) {
  __shared__ f32x4 part[4][64];
  const CacheView& c = a.c;
  const int lane = threadIdx.x & 63, w = wave_id();
  const long at = WAVES == 1 ? (long)blockIdx.x * 4 + w : blockIdx.x;
  if (at >= (long)c.T * a.hq) return;
  const long step = (long)c.T * a.hq;
  // lanes of a split: a power of two that holds D / 4
  const int lanes = c.D <= 32 ? 8 : c.D <= 64 ? 16 : c.D <= 128 ? 32 : 64;
  const int per_load = 64 / lanes, d = 4 * (lane % lanes);
  const int first = (WAVES == 1 ? 0 : w * per_load) + lane / lanes, stride = WAVES * per_load;
  // What the splits may have left is requested before it is known how many of them
  // there are (the workspace holds every one, whatever is in it): one load deep less.
  f32x4 v[8], o = {0.0f, 0.0f, 0.0f, 0.0f};
  auto fetch = [&](int u0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int u = u0 + i * stride + first;
      v[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (u < a.n_splits && d < c.D) v[i] = *reinterpret_cast<const f32x4*>(a.part_o + (u * step + at) * c.D + d);
    }
  };
  float2 ml = make_float2(kLeast, 0.0f);
  if (lane < a.n_splits) ml = a.part_ml[lane * step + at];
  fetch(0);
  const int t = static_cast<int>(at / a.hq), h = static_cast<int>(at % a.hq);
  const CacheSeq s = seq_of_token(c, lane, t);
  if (s.b >= c.n_seqs) return;
  if (t < s.tok0) return;
  const TileKeys tk = tile_keys(a, s, ((t - s.tok0) * a.group + h % a.group) / a.rows);
  if (tk.active <= 1) return;
  if (lane >= tk.active) ml = make_float2(kLeast, 0.0f);
  const float mx = lanes_most(ml.x);
  const float f = weight(ml.x - mx);
  const float total = lanes_total(f * ml.y);
  for (int u0 = 0; u0 < tk.active; u0 += 8 * stride) {
    if (u0 > 0) fetch(u0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int u = u0 + i * stride + first;
      const float fu = __shfl(f, u & 63);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = u < tk.active ? o[e] + fu * v[i][e] : o[e];
    }
  }
  for (int x = lanes; x < 64; x *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
  if constexpr (WAVES > 1) {
    part[w][lane] = o;
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int u = 1; u < WAVES; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += part[u][lane][e];
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if (lane < lanes && d < c.D) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    store4(static_cast<T*>(a.out) + at * c.D + d, o);
  }
  if (a.lse != nullptr && lane == 0)
    a.lse[(long)h * c.T + t] = total == 0.0f ? -INFINITY : (mx + log2f(total)) * kLn2;
}

template <typename T, int DP, int MB, int WAVES>
hipError_t attend(const CacheAttn& a, hipStream_t st) {
  using L = CaLayout<T, DP, MB, WAVES>;
  auto* fn = &cache_attn_kernel<T, DP, MB, WAVES>;
  GL_CHECK(allow_lds(fn, L::BYTES));
  hipLaunchKernelGGL((cache_attn_kernel<T, DP, MB, WAVES>), dim3(tile_numbers(a) * a.c.hkv * a.n_splits),
                     dim3(64 * WAVES), L::BYTES, st, a);
  return hipGetLastError();
}

template <typename T>
hipError_t join(const CacheAttn& a, hipStream_t st) {
  const long rows = (long)a.c.T * a.hq;
  if (a.n_splits <= 8)
    hipLaunchKernelGGL((cache_attn_join_kernel<T, 1>), dim3(static_cast<unsigned>((rows + 3) / 4)),
                       dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((cache_attn_join_kernel<T, 4>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, st, a);
  return hipGetLastError();
}

// 32 rows a tile: fp32 chunks of heads of 65 .. 128 (cache_attn_plan)
constexpr int kRowsMid = 32;

template <typename T>
hipError_t by_head(const CacheAttn& a, hipStream_t st) {
  constexpr int WAVES = sizeof(T) == 2 ? 4 : 8;
  const int d = a.c.D;
  if constexpr (sizeof(T) == 4) {
    if (a.rows == kRowsMid && d <= 96) return attend<T, 96, 2, WAVES>(a, st);
    if (a.rows == kRowsMid) return attend<T, 128, 2, WAVES>(a, st);
  }
  if (d <= 32) return attend<T, 32, 1, WAVES>(a, st);
  if (d <= 64) return attend<T, 64, 1, WAVES>(a, st);
  if (d <= 96) return attend<T, 96, 1, WAVES>(a, st);
  if (d <= 128) return attend<T, 128, 1, WAVES>(a, st);
  return attend<T, 256, 1, 4>(a, st);  // eight waves' fp32 tiles exceed the LDS
}

}  // namespace

CachePlan cache_attn_plan(const CacheView& c, int hq, int max_new, int max_kv, int n_cu) {
  CachePlan p{};
  const long group = hq / c.hkv;
  const long cap = (long)c.max_pages << c.page_shift;
  const long keys = max_kv > 0 && max_kv < cap ? max_kv : cap;
  // where the caller does not say, the new tokens are taken to be spread evenly over
  // the sequences, rounded down (a padded batch of single tokens).  us a call as one
  // chunk of them all and like that: 64 sequences of one token, 14/2 heads of 64, over
  // up to 4096 keys, 32 and 21; 32 of 28/4 heads of 128 over up to 8192, 61 and 53.
  const long seqs = std::min(c.T, c.n_seqs);
  const long longest = max_new > 0 && max_new < c.T ? max_new : max_new > 0 ? c.T : c.T / seqs;
  // tiles of so many rows, spread like that
  auto tiles_of = [&](long rows) { return seqs * ((c.T * group + seqs * rows - 1) / (seqs * rows)); };
  // Tiles of 128 rows for chunks that need more than one of 16, where tiles of 16
  // would read enough keys (tiles x keys x D).  us a call, tiles of 16 and of 128,
  // 28/4 heads of 128 where nothing else is said.  Up to 2048 keys, where the wide
  // tiles find few splits: 64 tokens over 1024 (15e6) 14, 22; 512 over 512 (59e6) 18,
  // 21; 16 chunks of up to 32 over up to 1024 (76e6) 27, 31; 8 of up to 128 over up to
  // 512, 32/8 (109e6) 33, 23; 512 over 1024 (117e6) 31, 32; 512 over 2048 (235e6) 53,
  // 42; 14/2 heads of 64: 1000 over 1000 (56e6) 15, 24; 8 of up to 200 over up to 2048
  // (109e6) 26, 28.  Over more: 16 over 8192 (29e6) 28, 22; 4 of up to 12 over up to
  // 4096 (34e6) 25, 24; 2 of up to 40 over up to 4096 (59e6) 26, 29; 16 of up to 6 over
  // up to 8192 (201e6) 71, 53; 40 over 4096, 12/2 (16e6) 15, 20; 14/2 heads of 64: 4 of
  // up to 100 over up to 4000 (61e6) 25, 24.  Above 128 columns one workgroup of wide
  // tiles fills a CU; 8/2 heads of 256: 256 over 2048 (67e6) 30, 41; 512 over 2048
  // (134e6) 40, 42; 600 over 1000, 16/4 (154e6) 54, 55; 1024 over 2048 (268e6) 70, 48;
  // 200 over 4096 (105e6) 46, 37; 128 over 8192 (134e6) 46, 58; 512 over 4096 (268e6)
  // 72, 52; 1024 over 8192 (1e9) 259, 120.
  const double enough = c.D <= 128 ? (keys <= 2048 ? 110e6 : 25e6) : keys <= 2048 ? 160e6 : 100e6;
  const bool wide =
      c.io_bf16 && longest * group > 16 && (double)tiles_of(16) * c.hkv * keys * c.D > enough;
  // fp32 chunks: tiles of 32 rows read K and V half as often, from 65 columns on (fewer
  // leave too few tiles), up to 128 (their sums fill the registers).  us a call, 16
  // and 32 rows: 512 tokens over 4096 keys, 28/4 heads of 128, 362, 303; 1024 over
  // 8192, 8/2 of 96, 256, 225; 8 chunks of up to 64 over up to 4000, 32/8 of 128, 229,
  // 212; 6 of up to 30 over up to 4000, 12/2 of 128, 55, 50; 4 of up to 300 over up to
  // 4000, 14/2 of 64, 98, 112; 2 of up to 900 over up to 3000, 8/8 of 64, 81, 90; 4 of
  // up to 300 over up to 4000, 8/2 of 256, 352, 391.  Not where they leave CUs idle
  // even in splits: 3 of up to 120 over up to 1001, 8/2 of 96 (54 tiles) 23, 36.
  const bool chunk = !c.io_bf16 && longest * group > 16;
  const long narrow_splits = keys <= 1024 ? 1 : keys / 512;
  const bool mid = chunk && c.D > 64 && c.D <= 128 && tiles_of(kRowsMid) * c.hkv * narrow_splits >= n_cu;
  p.rows = wide ? kCacheWideRows : mid ? kRowsMid : 16;
  // and their long tiles first: 1000 tokens as they come, 40/8 heads of 128, 159 -> 137
  // us; 8 chunks of up to 64 as above 248 -> 205; 4 of up to 300, 14/2 of 64, 97 -> 61;
  // 2 of up to 900, 8/8 of 64, 100 -> 96; bf16 single tokens lose 1 of 67.
  p.long_first = chunk;
  const long groups = tiles_of(p.rows) * c.hkv;
  // Splits of 512 keys or more, as many as fill the workgroups the CUs hold at
  // once (by their LDS); none up to 1024 keys, where the second launch costs
  // more than the shorter chain gives.  us a call, one token a sequence, 28/4
  // heads of 128: one sequence of 2048 keys 11.8 in splits of 512, 15.5 of
  // 1024, 19.4 whole; 8192 keys 12.2, 15.9, 23.2 in splits of 512, 1024, 2048;
  // 32 sequences of up to 1024 keys 12.8 whole, 15.8 in two; of up to 8192 keys
  // 93, 73, 77 for one, two and four workgroups a CU.  14/2 heads of 64, 64
  // sequences of up to 4096 keys: 24.8, 23.2, 21.5.  Eight waves a workgroup
  // instead of four: fp32 128 tokens over 4096 keys 37 -> 30; bf16 64 sequences
  // of up to 512 keys 12.1 -> 15.1.
  //
  // Tiles of 128 rows, two to a CU: as many splits as fill it, of 256 keys or
  // more (512 from 64 workgroups on, 2048 from 256 on), none up to 512 keys.  us
  // a call, 28/4 heads of 128, whole and in 2, 4, 8 splits: 32 tokens over 8192
  // keys (8 workgroups) 189, 106, 61, 41, and 26 in 32; 512 over 4096 (112) 103,
  // 68, 63, 73; 512 over 512 21, 24, 25, 25; 2048 over 8192 (448) 322, 321, 329,
  // 356; 16 chunks of up to 128 over up to 2048 (320) 62, 60, 68, 86; 8 of up to 256
  // over up to 4096 (320) 108, 96, 105, 112; 3 of up to 300 over up to 5000 (132) 122,
  // 77, 69, 78; 8/2 heads of 256, 1024 over 8192 (64) 353, 195, 117, 137.
  const long per_cu = wide ? (c.D <= 128 ? 2 : 1) : !c.io_bf16 ? 1 : c.D <= 64 ? 4 : c.D <= 128 ? 2 : 1;
  const long want = per_cu * n_cu / groups;
  const long least = groups < 64 ? 256 : groups < 256 ? 512 : 2048;
  const long most = !wide ? narrow_splits : keys <= 512 ? 1 : keys / least;
  const long cap_splits = wide && (long)c.T * hq > kCacheJoinRows ? kCacheTileJoin : kMaxSplits;
  const long launch = (1L << 22) / ((long)c.n_seqs * c.hkv);  // threads of a launch, with idle sequences
  p.n_splits = static_cast<int>(std::max(1L, std::min({want, most, cap_splits, launch})));
  const long even = (keys + p.n_splits - 1) / p.n_splits;
  p.split_keys = static_cast<int>((even + kSplitUnit - 1) / kSplitUnit * kSplitUnit);
  if (p.n_splits > 1) {
    const size_t rows = (size_t)c.T * hq;
    p.bytes = p.n_splits * rows * (c.D * sizeof(float) + sizeof(float2));
  }
  return p;
}

hipError_t launch_cache_attn(const CacheAttn& a, hipStream_t st) {
  if (a.rows == kCacheWideRows)
    GL_CHECK(launch_cache_attn_wide(a, st));
  else
    GL_CHECK(a.c.io_bf16 ? by_head<bf16>(a, st) : by_head<float>(a, st));
  // few splits of wide tiles are joined by tiles (launch_cache_attn_wide)
  if (a.n_splits == 1 || (a.rows == kCacheWideRows && a.n_splits <= kCacheTileJoin)) return hipSuccess;
  return launch_cache_join(a, st);
}

hipError_t launch_cache_join(const CacheAttn& a, hipStream_t st) {
  return a.c.io_bf16 ? join<bf16>(a, st) : join<float>(a, st);
}

}  // namespace glacier
