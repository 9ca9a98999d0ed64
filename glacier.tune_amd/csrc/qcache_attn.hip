// qcache_attn.hip -- attention of new tokens over a paged cache in 4 bits.
//
// Tiles, splits and the join are those of cache_attn.hip: 16 rows are (token, head of
// the group) pairs of one KV head, a workgroup's four waves take 32 keys at a time in
// turn, each with its own running maximum and sum, joined through LDS at the end.  K
// and V come from the pages by LDS DMA, as they lie there, into an area of each wave,
// and are unpacked in registers, straight into the matrix cores: a word of a page holds
// what one lane feeds to one MFMA, and pages are laid out so that a lane's words lie
// together.
//
// S^T = K Q^T, 16 keys by 16 rows, 32 columns (one group) at a time.
//   bf16: K as 128 + n (one operation per two elements), the sum begun at -136 sum(q),
//   and the scales applied to the product: S += s (K' q - 136 sum q).  The sums are 17
//   to 136 times the product's terms, which costs 4 to 8 of fp32's 24 bits: scores of
//   random queries are off by 7 x 2^-24 of their terms' length (root of squares; direct
//   sums 1 x 2^-24), far below what rounding q to bf16 has cost.  n - 8 instead would take
//   five operations more for two elements, where unpacking is what bounds single tokens.
//   fp32: K as n - 8, q in three bf16 terms (24 bits).
// O^T += V^T P^T, 32 tokens at a time.  Two tokens' words, their halves exchanged, hold
// eight columns of both: a lane's words are the operands of eight products (columns 8 x
// + one of 0 .. 7), of four where a head has at most 64 columns (then two lanes take a
// word's halves).
//   V as bf16 (n - 8) s, exact (five bits by three): (1024 + n) s - 1032 s, or (64 + n) s
//   - 72 s, where the sum in brackets is an fp16 value by one OR, formed by fp32
//   operations that take fp16 operands, of whose results the upper halves are kept.
//   The weights in two bf16 terms (16 bits of them; fp32: three).
//
// A held value is NaN only by its scale (it is never infinite).  Where a sum is not
// finite the wave walks its keys once more with such scales of V cleared, and gives
// NaN to the rows that see their tokens.
//
// Single tokens read each page once, and unpacking is as long as that: one token over
// 65536 keys, 32/8 heads of 128 (75.5 MB), 23.4 us, 4 of them the join's (vector
// instructions busy 62% of the kernel's 20; the pages alone take 15.4 at a copy's rate);
// 8 over 32768 (302 MB) 72 to 78, 3.9 to 4.2 TB/s.  Twelve waves a CU, one block of K and
// of V under way for each: either is asked for again as soon as it has been read from LDS.
//
// Long chunks: what the batch's sequences hold is written out first, exactly, and
// cache_attn.hip's kernels read that.
#include "cache_tiles.hpp"
#include "quant_page.hpp"

namespace glacier {
namespace {

[[maybe_unused]] constexpr int kKeysQ = 32;  // keys of a wave's block: one k-step of the second product
constexpr int kWavesQ = 4;
[[maybe_unused]] constexpr float kSlack = 8.0f;
// Queries are multiplied as 2^-13 of themselves (exactly, but for bits below 2^-120 of q, which
// no softmax sees), so that 32 of them times 143, of either sign, stay within fp32 whatever
// they are, as they do over a cache in bf16 or fp32.  The scores' scale gives it back.
constexpr float kQueryShare = 0x1p-13f;

// LDS of a workgroup: its queries, operands of the first product (and -136 sum(q), where
// its sums begin), then for each wave one block of K and one of V, words and then scales
// of two tiles of 16 keys, as they lie in the pages.
template <typename T, int G>
struct QaLayout {
  static constexpr int WAVES = kWavesQ;
  static constexpr bool KEEP = sizeof(T) == 2;  // the queries stay in registers (fp32: three times as many)

  static constexpr int NV = (G + 3) / 4;    // blocks of 16 words of a token of V
  static constexpr bool HALF = G <= 2;      // two lanes share a word
  static constexpr int NB = HALF ? 4 : 8 * NV;  // 16-column products
  static constexpr int DP = 32 * G;
  static constexpr int TERMS = sizeof(T) == 4 ? 3 : 1;  // of a query
  static constexpr int QUERY = 1024 * (TERMS == 3 ? 3 : 2);  // bytes of a group's operands
  static constexpr int WORDS = 256 * G, SCALES = 32 * G;  // bytes, of 16 keys
  static constexpr int SIDE = 2 * (WORDS + SCALES);
  static constexpr int ND = (WORDS + 1023) / 1024;  // DMA instructions of a tile's words
  static constexpr int LOADS = 2 * (ND + 1);        // of a side
  static constexpr int RING = G * QUERY + WAVES * 2 * SIDE;
  static constexpr int OS = DP + 4;         // row stride (floats) of a wave's sums in the join
  static constexpr int WAVE = 16 * (OS + 2);
  static constexpr int JOIN = WAVES * WAVE * 4;
  static constexpr int BYTES = RING > JOIN ? RING : JOIN;
  static_assert(BYTES <= 160 * 1024, "exceeds the LDS of a CU");
};

#if defined(__HIP_DEVICE_COMPILE__)
// N words at an LDS address plus OFF, issued only: see settled.
template <int N, int OFF>
struct LdsWords {
  LdsWords<N - 4, OFF + 16> rest;
  u32x4 w;
  __device__ inline void issue(unsigned at) {
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(w) : "v"(at), "i"(OFF));
    rest.issue(at);
  }
  __device__ inline void settled() {
    asm volatile("" : "+v"(w));
    rest.settled();
  }
  __device__ inline unsigned operator[](int i) const { return i < 4 ? w[i] : rest[i - 4]; }
  __device__ inline void keep(int i, unsigned mask) { i < 4 ? (void)(w[i] &= mask) : rest.keep(i - 4, mask); }
};
template <int OFF>
struct LdsWords<3, OFF> {
  typedef unsigned u32x3 __attribute__((ext_vector_type(3)));
  u32x3 w;
  __device__ inline void issue(unsigned at) {
    asm volatile("ds_read_b96 %0, %1 offset:%2" : "=v"(w) : "v"(at), "i"(OFF));
  }
  __device__ inline void settled() { asm volatile("" : "+v"(w)); }
  __device__ inline unsigned operator[](int i) const { return w[i]; }
};
template <int OFF>
struct LdsWords<2, OFF> {
  u32x2 w;
  __device__ inline void issue(unsigned at) {
    asm volatile("ds_read_b64 %0, %1 offset:%2" : "=v"(w) : "v"(at), "i"(OFF));
  }
  __device__ inline void settled() { asm volatile("" : "+v"(w)); }
  __device__ inline unsigned operator[](int i) const { return w[i]; }
  __device__ inline void keep(int i, unsigned mask) { w[i] &= mask; }
};
template <int OFF>
struct LdsWords<1, OFF> {
  unsigned w;
  __device__ inline void issue(unsigned at) {
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(w) : "v"(at), "i"(OFF));
  }
  __device__ inline void settled() { asm volatile("" : "+v"(w)); }
  __device__ inline unsigned operator[](int) const { return w; }
};
template <int OFF>
struct LdsWords<0, OFF> {
  __device__ inline void issue(unsigned) {}
  __device__ inline void settled() {}
  __device__ inline unsigned operator[](int) const { return 0; }
  __device__ inline void keep(int, unsigned) {}
};
#endif

// Halves of a register that are NaN, as a mask (scales are never infinite).
[[maybe_unused]] __device__ inline unsigned nan_halves(unsigned w) {
  return ((((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u) >> 15) * 0xffffu;
}

// 32-bit LDS address.
[[maybe_unused]] __device__ inline unsigned lds_at(unsigned char* p) {
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((GLACIER_LDS unsigned char*)p));
}
// Two floats rounded to bf16, the first in the lower half.
[[maybe_unused]] __device__ inline unsigned pair_of(float a, float b) {
  typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, bf16x2{(bf16)a, (bf16)b});
}

// Division of x by a number known before the launch: one multiplication while x d is
// below 2^32 for every x of the call (the product's error, below x d / 2^32, stays
// under one step then), else a division.  A dozen divisions of 30 instructions each
// were a third of what a workgroup of four short blocks executes.
struct FixedDiv {
  unsigned d, m;
  static FixedDiv by(unsigned d, unsigned long long most) {
    return {d, d > 1 && most * d < (1ull << 32) ? static_cast<unsigned>(((1ull << 32) + d - 1) / d) : 0u};
  }
  __device__ inline int of(int x) const {
    return d == 1 ? x : m != 0 ? static_cast<int>(__umulhi(static_cast<unsigned>(x), m)) : x / static_cast<int>(d);
  }
};
struct TileDivs {
  FixedDiv splits, heads, group;
  unsigned few;  // 2^16 / group, rounded up
  bool by_length;  // tiles as work_by_length has them
  // x / group for x < group + 15
  __device__ inline int few_of(int x, int of) const {
    return of >= 16 ? (x >= of ? 1 : 0) : static_cast<int>(static_cast<unsigned>(x) * few >> 16);
  }
};

// Sum of x over this lane and those before it.
[[maybe_unused]] __device__ inline int lanes_up_to(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // 1, 2, 4, 8 lanes before, in a row of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // the row before's last lane, into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // lane 31, into rows 2 and 3
  return x;
}

// What a workgroup takes: a tile of 16 rows from r0 of sequence s on, one split of its
// keys, one KV head.
struct TileWork {
  CacheSeq s;
  int r0, split, kvh;  // r0: -1 if there is none
  int per, active;  // of the keys, where `last` (else not known yet)
  bool last;  // the sequence's last tile
};
// As everywhere: tiles are numbered through all sequences, a tile's splits from another
// one on.
[[maybe_unused]] __device__ inline TileWork work_by_number(const CacheAttn& a, const TileDivs& f, int lane, int block) {
  const CacheView& c = a.c;
  TileWork x{{c.n_seqs, 0, 0, 0}, -1, 0, 0, 0, 0, false};
  const int rest = f.splits.of(block), number = f.heads.of(rest);
  x.kvh = rest - number * c.hkv;
  x.split = block - rest * a.n_splits + number;
  x.split -= f.splits.of(x.split) * a.n_splits;
  x.s = find_seq(c, lane, number, [&](int b, int to) { return (to * a.group >> 4) + b; });
  if (x.s.b < c.n_seqs) x.r0 = 16 * (number - (x.s.tok0 * a.group >> 4) - x.s.b);
  return x;
}
// Every lane works out how many splits the tiles of one of up to 64 sequences have (splits_a_tile),
// so that workgroups without work come last: a launch holds one for every split that a tile
// may have, and an empty one among others costs them up to 9 ns.  us a call, by number
// and so: 32 sequences of 4096 keys, groups of 7 and 15 heads, 29.6, 27.2 and 31.3, 28.7;
// 64 of up to 4096, 14/2 heads of 64, 19.3, 17.4; 8 of up to 16000, 32/8 heads of 128,
// 33.2, 30.7; groups of one head 25.9, 26.5; 4 chunks of 32 tokens over 8192 64.1, 66.9.
[[maybe_unused]] __device__ inline TileWork work_by_length(const CacheAttn& a, const TileDivs& f, int lane, int block) {
  const CacheView& c = a.c;
  TileWork x{{c.n_seqs, 0, 0, 0}, -1, 0, 0, 0, 0, false};
  const int item = f.heads.of(block);
  x.kvh = block - item * c.hkv;
  const int i = min(lane, c.n_seqs - 1);
  const int from = clamp_row(c.cu[i], c.T), n = lane < c.n_seqs ? max(0, clamp_row(c.cu[i + 1], c.T) - from) : 0;
  const int pos0 = c.kv_lens[i] - n, tiles = (n * a.group + 15) >> 4;
  const long cap = (long)c.max_pages << c.page_shift, len = (long)pos0 + n;
  const int kend = static_cast<int>(len < 0 ? 0 : len < cap ? len : cap);
  KeySplit k{max(1, (kend + kSplitUnit - 1) / kSplitUnit) * kSplitUnit, 1};
  if (a.n_splits > 1) k = split_with(kend, a.n_splits, a.split_keys, div_up);
  const int each = splits_a_tile(tiles, k.active, kend, a.n_splits, a.split_keys, div_up);
  const int items = tiles * each, end = lanes_up_to(items);
  const unsigned long long mine = __ballot(item >= end - items && item < end);
  if (mine == 0) return x;
  const int b = __ffsll(mine) - 1, count = __builtin_amdgcn_readlane(tiles, b);
  x.s.b = b;
  x.s.tok0 = __builtin_amdgcn_readlane(from, b);
  x.s.n = __builtin_amdgcn_readlane(n, b);
  x.s.pos0 = __builtin_amdgcn_readlane(pos0, b);
  x.per = __builtin_amdgcn_readlane(k.per, b);
  x.active = __builtin_amdgcn_readlane(k.active, b);
  const int per_tile = __builtin_amdgcn_readlane(each, b);
  x.split = item - __builtin_amdgcn_readlane(end - items, b);
  int tile = 0;
  if (count > 1) {
    tile = __builtin_amdgcn_readfirstlane(div_up(x.split + 1, per_tile) - 1);
    x.split -= tile * per_tile;
  }
  x.last = tile == count - 1;
  // (more work than the launch has room for, as wrong offsets may have it, can wrap around)
  x.r0 = tile >= 0 && tile < count && x.split >= 0 && x.split < per_tile ? 16 * tile : -1;
  return x;
}

template <typename T, int G>
__global__ __launch_bounds__((64 * QaLayout<T, G>::WAVES), G <= 4 ? 3 : 2) void qcache_attn_kernel(CacheAttn a, TileDivs f) {
#if defined(__HIP_DEVICE_COMPILE__)
  using L = QaLayout<T, G>;
  constexpr int NV = L::NV, NB = L::NB, WAVES = L::WAVES, TERMS = L::TERMS;
  constexpr bool F32 = sizeof(T) == 4, HALF = L::HALF;
  extern __shared__ __align__(16) unsigned char smem[];
  const CacheView& c = a.c;
  const int w = wave_id(), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15, D = c.D;
  const TileWork x = f.by_length ? work_by_length(a, f, lane, blockIdx.x) : work_by_number(a, f, lane, blockIdx.x);
  const CacheSeq& s = x.s;
  const int b = s.b, r0 = x.r0, split = x.split, kvh = x.kvh, n_rows = s.n * a.group;
  if (r0 < 0 || r0 >= n_rows) return;
  const int tok0 = f.group.of(r0), head0 = r0 - tok0 * a.group;  // the tile's first row
  const int last = min(s.n - 1, tok0 + f.few_of(head0 + 15, a.group));
  TileKeys tk;
  if (x.last) {
    const long cap = (long)c.max_pages << c.page_shift, end = (long)s.pos0 + s.n;
    tk = {static_cast<int>(end < 0 ? 0 : end < cap ? end : cap), x.per, x.active};
  } else {
    tk = keys_up_to(a, s, last);
  }
  if (split >= tk.active) return;
  const int k0 = split * tk.per, k1 = min(tk.kend, k0 + tk.per);

  const int part_bytes = quant_row_bytes(D) << c.page_shift, words_bytes = (16 * G) << c.page_shift;
  const long head_at = (long)kvh * part_bytes;
  const auto* const table = (const __attribute__((address_space(4))) int32_t*)(
      reinterpret_cast<uintptr_t>(c.table + (long)b * c.table_stride));
  constexpr int STEP = WAVES * kKeysQ;
  const int first = k0 + w * kKeysQ;
  // The table's entries of the block to be requested next (two pages of 16, or one).
  // They are looked up a block ahead, by scalar loads, and not looked at before they are
  // needed: any wait for LDS is one for them too.
  int entry[2];
  auto look_up = [&](int j) __attribute__((always_inline)) {
    entry[0] = entry[1] = -1;
    if (j < k1) entry[0] = table[min(j >> c.page_shift, c.max_pages - 1)];
    if (c.page_shift == 4 && j + 16 < k1) entry[1] = table[min((j + 16) >> 4, c.max_pages - 1)];
  };
  look_up(first);

  // this lane's row: its last key and its query
  const int over = f.few_of(head0 + col, a.group), tok = tok0 + over, head = kvh * a.group + head0 + col - over * a.group;
  const bool has_row = r0 + col < n_rows;
  const int limit = has_row ? s.pos0 + tok : -1;
  {
    // columns 32 i + 8 g .. of groups i = w, w + WAVES, ..
    const T* const q = static_cast<const T*>(a.q) +
                       (has_row ? (long)(s.tok0 + tok) * a.hq + head : (long)(s.tok0 + tok0) * a.hq) * D;
    bf16x8 minus;
#pragma unroll
    for (int e = 0; e < 8; ++e) minus[e] = (bf16)-136.0f;
#pragma unroll
    for (int i0 = 0; i0 < G; i0 += WAVES) {
      const int i = i0 + w, at = 32 * i + 8 * g;
      if (i >= G) break;
      i32x4 raw[F32 ? 2 : 1];
#pragma unroll
      for (int x = 0; x < (F32 ? 2 : 1); ++x) {
        raw[x] = *reinterpret_cast<const i32x4*>(q + (at < D ? at + 4 * x : 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[x][e] = has_row && at < D ? raw[x][e] : 0;
      }
      unsigned char* const to = smem + i * L::QUERY + 16 * lane;
      if constexpr (F32) {
        bf16x8 term[3];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = kQueryShare * __builtin_bit_cast(f32x4, raw[e / 4])[e % 4];
          term[0][e] = (bf16)x;
          const float r1 = x - (float)term[0][e];
          term[1][e] = (bf16)r1;
          term[2][e] = (bf16)(r1 - (float)term[1][e]);
        }
#pragma unroll
        for (int x = 0; x < 3; ++x) *reinterpret_cast<bf16x8*>(to + 1024 * x) = term[x];
      } else {
        bf16x8 x = __builtin_bit_cast(bf16x8, raw[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (bf16)(kQueryShare * (float)x[e]);
        *reinterpret_cast<bf16x8*>(to) = x;
        *reinterpret_cast<f32x4*>(to + 1024) = Mfma<bf16>::mma(minus, x, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
      }
    }
  }
  __syncthreads();

  // this lane's places (bytes): the queries, words and scales of K and V
  unsigned char* const mine_at = smem + G * L::QUERY + w * 2 * L::SIDE;
  const unsigned q_at = lds_at(smem) + 16 * lane;
  const unsigned side_at = lds_at(mine_at);
  const unsigned k_at = side_at + (col * 4 + g) * G * 4, ks_at = side_at + 2 * L::WORDS + 8 * G * g;
  unsigned v_at[NV], vs_at[NV];
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    const int word = min(HALF ? col >> 1 : 16 * x + col, 4 * G - 1);
    v_at[x] = side_at + L::SIDE + (g * 4 * G + word) * 16;
    vs_at[x] = side_at + L::SIDE + 2 * L::WORDS + (g * G + word / 4) * 8;
  }
  const unsigned pick = HALF && (col & 1) ? 0x07060302u : 0x05040100u;  // which halves of a pair of words

  // A block's pages: K's and V's two tiles of 16 keys, nothing where there is no page.
  // (V's begin as many bytes behind K's as the pages do.)
  long page_at[2];
  int page_bytes[2], rows[2];
  unsigned found = 0, there = 0;  // which tiles of the block requested last, and of this one, have a page
  auto aim = [&](int j) __attribute__((always_inline)) {
    found = 0;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (p == 1 && c.page_shift != 4) {  // the same page
        page_at[1] = page_at[0];
        found |= j + 16 < k1 ? found << 1 : 0;
      } else {
        const bool held = static_cast<unsigned>(entry[p]) < static_cast<unsigned>(c.n_pages);
        page_at[p] = (held ? entry[p] : 0) * c.page_stride + head_at;
        found |= held ? 1u << p : 0u;
      }
      page_bytes[p] = found >> p & 1 ? part_bytes : 0;
      rows[p] = (j + 16 * p) & ((1 << c.page_shift) - 1);
    }
  };
  auto request = [&](const void* pages, unsigned char* to) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const auto rs = wave_rsrc(static_cast<const char*>(pages) + page_at[p], page_bytes[p]);
#pragma unroll
      for (int n = 0; n < L::ND; ++n)
        if (L::WORDS % 1024 == 0 || lane < (L::WORDS - 1024 * n) / 16)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (GLACIER_LDS void*)(to + p * L::WORDS + 1024 * n), 16,
                                                   16 * lane + 1024 * n, rows[p] * 16 * G, 0, 0);
      if (lane < L::SCALES / 16)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (GLACIER_LDS void*)(to + 2 * L::WORDS + p * L::SCALES), 16,
                                                 16 * lane, words_bytes + rows[p] * 2 * G, 0, 0);
    }
  };
  auto start = [&]() __attribute__((always_inline)) {
    aim(first);
    request(c.k_pages, mine_at);
    request(c.v_pages, mine_at + L::SIDE);
    look_up(first + STEP);
  };
  start();
  LdsWords<4, 0> qw[G][TERMS], base[G];
  auto queries = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
      for (int x = 0; x < TERMS; ++x) qw[i][x].issue(q_at + i * L::QUERY + 1024 * x);
      if constexpr (!F32) base[i].issue(q_at + i * L::QUERY + 1024);
    }
  };
  auto queries_settled = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
      for (int x = 0; x < TERMS; ++x) qw[i][x].settled();
      if constexpr (!F32) base[i].settled();
    }
  };
  if constexpr (L::KEEP) {
    queries();
    lgkm<0>();
    queries_settled();
  }

  const QuantMagic magic;
  f32x4 acc[NB];
  float m, l;
  const int first_limit = s.pos0 + tok0;  // the tile's first row sees keys up to here
  // One block.  What it has read of LDS is requested anew for the next block at once, K's
  // before its products and V's before its own, so that either has most of a block's time
  // to come; the counts are of what may still be under way.
  auto take = [&](int j, auto careful) __attribute__((always_inline)) {
    vmw<L::LOADS>();  // K has come
    LdsWords<G, 0> kw[2];
    LdsWords<2 * G, 0> ks[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      kw[p].issue(k_at + p * L::WORDS);
      ks[p].issue(ks_at + p * L::SCALES);
    }
    if constexpr (!L::KEEP) queries();
    lgkm<0>();
#pragma unroll
    for (int p = 0; p < 2; ++p) kw[p].settled(), ks[p].settled();
    if constexpr (!L::KEEP) queries_settled();
    there = found;
    const int here[2] = {there & 1 ? min(16, k1 - j) : 0, there & 2 ? min(16, k1 - j - 16) : 0};
    const bool whole = j + kKeysQ - 1 <= first_limit && here[0] == 16 && here[1] == 16;
    aim(j + STEP);
    request(c.k_pages, mine_at);
    look_up(j + 2 * STEP);
    // S^T: keys 16 p + 4 g + r of this block, row col
    f32x4 st[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) st[p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        f32x4 d;
        if constexpr (F32) {
          const bf16x8 kf = exact8_bf16(kw[p][i], magic);
          d = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int x = TERMS - 1; x >= 0; --x) d = Mfma<bf16>::mma(kf, __builtin_bit_cast(bf16x8, qw[i][x].w), d);
        } else {
          d = Mfma<bf16>::mma(raw8_bf16(kw[p][i], magic), __builtin_bit_cast(bf16x8, qw[i][0].w),
                              __builtin_bit_cast(f32x4, base[i].w));
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) st[p][r] = fmaf(half_at(ks[p][(r * G + i) / 2], (r * G + i) % 2), d[r], st[p][r]);
      }
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[p][r] *= a.scale_log2;
    if (!whole) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = 4 * g + r;
          st[p][r] = at < here[p] && j + 16 * p + at <= limit ? st[p][r] : -INFINITY;
        }
    }
    float top = kLeast;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, st[p][r]);
    // The running maximum follows a row's scores only where they leave it by more than
    // kSlack: weights reach 2^kSlack then, which fp32 sums hold as well, and most blocks
    // of a tile of several rows scale nothing.
    const float high = col_max_swap(top), mn = high > m + kSlack ? high : m;
    if (__any(mn != m)) {
      const float alpha = weight(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[n][r] *= alpha;
    }
    // the weights, and their bf16 terms by pairs
    constexpr int PT = F32 ? 3 : 2;
    u32x4 pf[PT];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float x = weight(st[e / 4][e % 4] - mn), y = weight(st[e / 4][e % 4 + 1] - mn);
      l += x;
      l += y;
#pragma unroll
      for (int z = 0; z < PT; ++z) {
        const unsigned pair = pair_of(x, y);
        pf[z][e / 2] = pair;
        x -= __builtin_bit_cast(float, pair << 16);
        y -= __builtin_bit_cast(float, pair & 0xffff0000u);
      }
    }
    vmw<L::LOADS>();  // V has come
    LdsWords<4, 0> vw[2][NV];
    LdsWords<2, 0> vs[2][NV];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int y = 0; y < NV; ++y) {
        vw[p][y].issue(v_at[y] + p * L::WORDS);
        vs[p][y].issue(vs_at[y] + p * L::SCALES);
      }
    lgkm<0>();
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int y = 0; y < NV; ++y) vw[p][y].settled(), vs[p][y].settled();
    request(c.v_pages, mine_at + L::SIDE);
    // scales of V that count: not those of keys that are not there
    if (!whole) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int n = here[p] - 4 * g;  // of this lane's four tokens
        const unsigned keep0 = n <= 0 ? 0u : n == 1 ? 0xffffu : ~0u, keep1 = n <= 2 ? 0u : n == 3 ? 0xffffu : ~0u;
#pragma unroll
        for (int y = 0; y < NV; ++y) vs[p][y].keep(0, keep0), vs[p][y].keep(1, keep1);
      }
    }
    if constexpr (careful()) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int y = 0; y < NV; ++y)
#pragma unroll
          for (int u = 0; u < 2; ++u) vs[p][y].keep(u, ~nan_halves(vs[p][y][u]));
    }
    // O^T += V^T P^T
#pragma unroll
    for (int y = 0; y < NV; ++y) {
      float off[2][4][2];  // of a token: -1032 s and -72 s
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float sc = half_at(vs[p][y][u / 2], u % 2);
          off[p][u][0] = -1032.0f * sc;
          off[p][u][1] = -72.0f * sc;
        }
#pragma unroll
      for (int z = 0; z < (HALF ? 1 : 2); ++z) {
        const unsigned sel = HALF ? pick : z == 0 ? 0x05040100u : 0x07060302u;
        unsigned both[2][2];  // the halves of two tokens' words
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int u = 0; u < 2; ++u) both[p][u] = __builtin_amdgcn_perm(vw[p][y][2 * u + 1], vw[p][y][2 * u], sel);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u32x4 vf;
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              // 1024 + n from bits 0-3 of a half, 64 + n from bits 4-7
              const unsigned n = e < 2 ? both[p][u] : both[p][u] >> 8;
              const f16x2 h = __builtin_bit_cast(
                  f16x2, e % 2 == 0 ? (n & 0x000f000fu) | magic.h1024 : (n & 0x00f000f0u) | magic.h64);
              vf[2 * p + u] = upper_pair(fmaf((float)h[0], half_at(vs[p][y][u], 0), off[p][2 * u][e % 2]),
                                         fmaf((float)h[1], half_at(vs[p][y][u], 1), off[p][2 * u + 1][e % 2]));
            }
          const int n = 8 * y + 4 * z + e;
#pragma unroll
          for (int t = PT - 1; t >= 0; --t)
            acc[n] = Mfma<bf16>::mma(__builtin_bit_cast(bf16x8, vf), __builtin_bit_cast(bf16x8, pf[t]), acc[n]);
        }
      }
    }
  };
  auto walk = [&](auto careful) __attribute__((always_inline)) {
    m = kLeast;
    l = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int j = first; j < k1; j += STEP) take(j, careful);
  };
  walk(std::false_type{});
  unsigned odd = 0;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) odd |= has_row ? not_finite(acc[n][r]) : 0;
  if (__any(odd != 0)) {
    vmw<0>();  // (the walk requests a block past its last one: nothing)
    look_up(first);
    start();
    walk(std::true_type{});
    // a lane's sums of one block belong to one group of columns
    for (int j = first; j < k1; j += STEP)
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
  vmw<0>();
  __syncthreads();
  float* const all = reinterpret_cast<float*>(smem);
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
  for (int idx = threadIdx.x; idx < 16 * CPR; idx += 64 * WAVES) {
    const int at_row = idx / CPR, d = 4 * (idx % CPR), r = r0 + at_row;
    if (r >= n_rows || d >= D) continue;
    float mx = kLeast;
#pragma unroll
    for (int u = 0; u < WAVES; ++u) mx = fmaxf(mx, all[u * L::WAVE + 16 * L::OS + at_row]);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float total = 0.0f;
#pragma unroll
    for (int u = 0; u < WAVES; ++u) {
      const float* reg = all + u * L::WAVE;
      const float part = weight(reg[16 * L::OS + at_row] - mx);
      total += part * reg[16 * (L::OS + 1) + at_row];
      const f32x4 v = *reinterpret_cast<const f32x4*>(reg + at_row * L::OS + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += part * v[e];
    }
    const int i = f.few_of(head0 + at_row, a.group), h = kvh * a.group + head0 + at_row - i * a.group;
    const long t = s.tok0 + tok0 + i, at = t * a.hq + h;
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
// that cache's table.  A workgroup takes 16 rows of one KV head, whatever the page size;
// rows past the sequence's end are not written (the attention does not read them).  8192
// keys of 4 heads of 128: 15 us of the 307 that a chunk of 2048 tokens takes over them.
constexpr int kExpandThreads = 256;
template <typename IO, int G>
__global__ __launch_bounds__(kExpandThreads) void qcache_expand_kernel(CacheView c, IO* k, IO* v, int32_t* table) {
  const int pieces = c.max_pages << (c.page_shift - 4);
  const int piece = blockIdx.x % pieces, kvh = blockIdx.x / pieces % c.hkv, b = blockIdx.x / pieces / c.hkv;
  const int i = piece >> (c.page_shift - 4), first = 16 * piece, row0 = first & ((1 << c.page_shift) - 1);
  const int keys = min(c.kv_lens[b] - first, 16);
  const bool fresh = clamp_row(c.cu[b + 1], c.T) > clamp_row(c.cu[b], c.T);  // it has new tokens to attend
  const int page = fresh && keys > 0 ? cache_page(c, b, first) : -1;
  const long to = (long)b * c.max_pages + i;
  if (kvh == 0 && row0 == 0 && threadIdx.x == 0) table[to] = page < 0 ? -1 : static_cast<int>(to);
  if (page < 0) return;
  const long part_bytes = (long)quant_row_bytes(c.D) << c.page_shift, from = page * c.page_stride + kvh * part_bytes;
  const char* const kp = static_cast<const char*>(c.k_pages) + from;
  const char* const vp = static_cast<const char*>(c.v_pages) + from;
  const long words_bytes = (16L * G) << c.page_shift, at = (to * c.hkv + kvh) * ((long)c.D << c.page_shift);
  const int per_row = c.D / 8;
  for (int x = threadIdx.x; x < keys * per_row; x += kExpandThreads) {
    const int row = row0 + x / per_row, col8 = x % per_row;
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
hipError_t attend(CacheAttn a, hipStream_t st) {
  a.scale_log2 /= kQueryShare;
  constexpr int BYTES = QaLayout<T, G>::BYTES, WAVES = QaLayout<T, G>::WAVES;
  GL_CHECK(allow_lds(&qcache_attn_kernel<T, G>, BYTES));
  const unsigned groups = tile_numbers(a) * a.c.hkv * a.n_splits;
  // by length: several sequences, mostly of one tile (else few workgroups are empty)
  const bool by_length = a.c.n_seqs > 1 && a.c.n_seqs <= 64 && (long)a.c.T * a.group <= 16L * a.c.n_seqs;
  const TileDivs f{FixedDiv::by(a.n_splits, groups), FixedDiv::by(a.c.hkv, groups),
                   FixedDiv::by(a.group, (unsigned long long)a.c.T * a.group), (65535u + a.group) / a.group, by_length};
  hipLaunchKernelGGL((qcache_attn_kernel<T, G>), dim3(groups), dim3(64 * WAVES), BYTES, st, a, f);
  return hipGetLastError();
}
template <typename T, int G>
hipError_t expand(const CacheView& c, void* k, void* v, int32_t* table, hipStream_t st) {
  const long pieces = (long)c.max_pages << (c.page_shift - 4);
  hipLaunchKernelGGL((qcache_expand_kernel<T, G>), dim3(static_cast<unsigned>(c.n_seqs * c.hkv * pieces)),
                     dim3(kExpandThreads), 0, st, c, static_cast<T*>(k), static_cast<T*>(v), table);
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
  // Pages are written out for chunks that many tiles of 16 rows would read again: from a
  // mean of 256 rows a sequence on.  28/4 heads of 128 over 8192 keys, in us: 4 sequences
  // of 16 tokens 43.4 (written out: 63.2), of 32 66.0 (73.6), of 64 116 (84.4); 16 of 16
  // 117 (153), of 32 214 (189); 32/8 heads in fp32, 4 of 32 over 2048: 36.2 (70.4).  They
  // lie in the workspace for whatever the table's rows can name (max_kv is a hint only):
  // up to 2^30 bytes of K and V, else tiles of 16 rows read the 4-bit pages however long
  // the chunks are.  (Nor is there anything to write out of tables without a column.)  What
  // the mean and the table's width cost: 2048 tokens over 8192 beside 57 single ones over 4096
  // 588, 325 and 40 in two calls; 17 of 128 over 2048 in a table of 32768 tokens 210, of 2048
  // 125; 2048 over 2048 in one of 131072, whose whole width the launch covers, 90, of 2048 75.
  const long group = hq / c.hkv, cap = (long)c.max_pages << c.page_shift;
  const long seqs = std::min(c.T, c.n_seqs);
  const size_t k_bytes = (size_t)c.n_seqs * c.max_pages * c.hkv * ((size_t)c.D << c.page_shift) * (c.io_bf16 ? 2 : 4);
  p.expand = p.attn.rows > 16 && c.T * group > 256 * seqs && k_bytes > 0 && k_bytes <= (size_t)1 << 29;
  if (p.expand) {
    p.k_bytes = up256(k_bytes);
    p.table_bytes = up256(sizeof(int32_t) * c.n_seqs * c.max_pages);
    p.bytes = 2 * p.k_bytes + p.table_bytes + p.attn.bytes;
    return p;
  }
  const long keys = max_kv > 0 && max_kv < cap ? max_kv : cap;
  const long tiles = seqs * ((c.T * group + seqs * 16 - 1) / (seqs * 16));
  p.attn.rows = 16;
  p.attn.long_first = false;
  const long want = 4L * n_cu / std::max(1L, tiles * c.hkv);
  const long most = keys <= 512 ? 1 : keys / 256;
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
