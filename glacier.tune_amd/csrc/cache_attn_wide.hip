// cache_attn_wide.hip -- attention of chunks of new tokens over the paged
// cache on 32x32x16 MFMAs (bf16).
//
// A workgroup takes 128 rows (token, head of the group) of one KV head, 32 a
// wave, and walks the keys 64 at a time; up to 128 columns two workgroups share
// a CU.  K and V tiles come page by page by LDS DMA, two slots each, one barrier
// a tile: while a tile's weights meet V, its successor's scores are formed from
// the K tile that came a step earlier, so matrix and vector instructions of one
// wave have no order between them.  Rows of 16-byte pieces are swizzled (lds_sw,
// lds_mfma.hpp), which keeps both reads free of bank conflicts.
//
// Scores are formed transposed: S^T = K Q^T leaves a lane with 16 keys of one
// row in each accumulator block, and elements 8 s .. 8 s + 7 are the k-slots of
// step s of O^T += V^T P^T, whose V operand comes from two transposing LDS
// reads (the accumulator layout is described in attn_bwd3.hip).  Each weight
// multiplies V as two bf16 terms, as in the 16-row kernel: a token's result is as
// good beside a long chunk as alone (2048 tokens as below, off from 64 bits by
// 0.0017 of the result, the rounding of bf16 itself; one term leaves 0.0024 in
// 223-231 us, two 0.0017 in 304-314).  The sum takes the weights unrounded.
//
// The running maximum is only followed where it has grown by more than 8 (in
// log2): until then weights are taken against the old one, at most 2^8 large,
// and the sums need no rescaling.  The result is the same: any reference value
// cancels in out and lse.  (The second walk, which also takes the sums that leave
// fp32, follows it always: with V from 2^120 on it is those 2^8 that count.)
//
// KV heads alternate over the workgroups, so that an XCD's L2 serves few of
// them, and the tiles of long sequences start first (eight ragged chunks, with one
// term: 117 -> 94 us; now 116-125).
//
// Measured: 2048 tokens over 8192 keys, 28/4 heads of 128: 304-314 us (690-670
// TFLOP/s, 1035 with the second terms' products; a library product of 8192^3
// reaches 1205 on the card).  Of the cycles that the card counts as active (1.95 GHz)
// MFMAs are busy 47% and vector instructions issue 37%; waves spend 42% of theirs ready
// and waiting for the other's instruction; tiles of 448 workgroups on 512 places leave
// an eighth of the card idle.  1024 tokens over 8192 keys, 8/2 heads of 256, one wave a
// SIMD: 116-121 us (550-530 TFLOP/s), MFMAs busy 36%.
//
// Tried and slower (with one term, then at 221-231): tiles through registers (278 us),
// 256 rows on eight waves (295), lines asked for two tiles ahead (245), equal shares of
// all tiles' steps for every workgroup with fragments joined afterwards (278: the
// workgroups lose each other's L2 lines), scheduling hints of the compiler (235-281).
#include "cache_tiles.hpp"

namespace glacier {
namespace {

constexpr int kWavesWide = 4;
constexpr int kRowsWide = 32 * kWavesWide;
constexpr int kKeysWide = 64;
constexpr float kGrowth = 8.0f;

template <int DP>
struct Wide {
  static constexpr int RB = 2 * DP;   // bytes of an LDS row
  static constexpr int PPR = DP / 8;  // 16-byte pieces of a row
  static constexpr int TILE = kKeysWide * RB;
  static constexpr int NOTES = 4 * TILE;  // after K and V, two slots each: the noted tiles
  static constexpr int BYTES = NOTES + kNotedBlocks / 8;
  static constexpr int NKK = DP / 16, NDB = DP / 32;
  static constexpr int ND = 16 * RB / 1024;  // DMA instructions of a page piece
};

__device__ inline f32x16 mma16(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 1 KB of a wave's [base, base + bytes) to LDS, lane l's 16 bytes from `off` to
// to + 16 l; zeros past the end.
__device__ inline void dma16(const void* base, int bytes, int off, unsigned char* to) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(wave_rsrc(base, bytes), (GLACIER_LDS void*)to, 16, off, 0, 0, 0);
#endif
}

// What a wave carries from tile to tile.
template <int DP>
struct WideState {
  f32x16 o[DP / 32];  // O^T
  float m, l, top;    // reference, sum, and the next tile's largest score
};

template <int DP>
__device__ __forceinline__ void wide_scores(f32x16 (&st)[2], const unsigned char* kt, int koff,
                                            const bf16x8 (&qf)[DP / 16]) {
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int e = 0; e < 16; ++e) st[kb][e] = 0.0f;
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
      st[kb] = mma16(*reinterpret_cast<const bf16x8*>(kt + (koff ^ 32 * kk) + kb * 32 * 2 * DP), qf[kk], st[kb]);
}

__device__ __forceinline__ float wide_largest(const f32x16 (&st)[2]) {
  float top = fmaxf(st[0][0], st[1][0]);
#pragma unroll
  for (int e = 1; e < 16; ++e) top = fmaxf(fmaxf(top, st[0][e]), st[1][e]);
  return top;
}

// The weight of a score.  The fused form keeps what rounding the product would
// take off, which is the better value until scores of 2^30 and more leave so much
// of it that a row's largest weight is far from 1, and leaves fp32: the second walk
// rounds the product as the reference was rounded.
template <bool EXACT>
__device__ __forceinline__ float weight_of(float score, float scale_log2, float reference) {
  if constexpr (EXACT) {
#pragma clang fp contract(off)
    const float scaled = score * scale_log2;
    return weight(scaled - reference);
  }
  return weight(fmaf(score, scale_log2, -reference));
}

// Two values rounded to bf16, the first in the lower half.
__device__ __forceinline__ unsigned pair16(float a, float b) {
  typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, bf16x2{(bf16)a, (bf16)b});
}
// Only scalar instructions are moved past it.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(4); }

// One tile: its scores st (formed a tile earlier) become weights and meet V,
// while the next tile's scores are formed into sn.  EXACT (second walk): see weight_of.
// Products and weights alternate, two or four products to two or four weights, and a
// product's K or V is read one such group ahead (324 -> 304 us for 2048 tokens as
// above; left to the compiler, all weights come before all of V's products).  The
// blocks of a row differ by an exclusive or of the address, formed again for each
// tile: kept, they are 14 registers that the kernel has not got.
template <int DP, bool EXACT>
__device__ __forceinline__ void wide_step(WideState<DP>& w, f32x16 (&st)[2], f32x16 (&sn)[2],
                                          const unsigned char* __restrict__ kt,
                                          const unsigned char* __restrict__ vt, int koff, int voff0, int voff1,
                                          const bf16x8 (&qf)[DP / 16], float scale_log2) {
  asm volatile("" : "+v"(koff), "+v"(voff0), "+v"(voff1));  // (not kept from the tile before)
  w.top = swap_max(w.top, false) * scale_log2;
  if (__any(w.top > w.m + (EXACT ? 0.0f : kGrowth))) {
    const float mn = fmaxf(w.m, w.top);
    const float f = weight(w.m - mn);
    w.m = mn;
    w.l *= f;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) w.o[db][e] *= f;
  }
  float sum = 0.0f;
  i32x4 hi[4], lo[4];  // the weights' two terms, 16 keys each
  auto weights = [&](int from, int to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = from; i < to; i += 2) {
      const float p0 = weight_of<EXACT>(st[i / 16][i % 16], scale_log2, w.m);
      const float p1 = weight_of<EXACT>(st[i / 16][i % 16 + 1], scale_log2, w.m);
      const unsigned h = pair16(p0, p1);
      hi[i / 8][i % 8 / 2] = static_cast<int>(h);
      lo[i / 8][i % 8 / 2] = static_cast<int>(
          pair16(p0 - __builtin_bit_cast(float, h << 16), p1 - __builtin_bit_cast(float, h & 0xffff0000u)));
      sum += p0 + p1;
      asm volatile("" : "+v"(sum));  // (here, or the compiler keeps every weight to the end)
    }
  };
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int e = 0; e < 16; ++e) sn[kb][e] = 0.0f;
  constexpr int NKK = DP / 16, NPAIR = DP / 64;
  struct Pair {
    bf16x8 x[2];
  };
  // (of both 32-key halves; of 16 keys, two blocks of columns)
  auto keys = [&](int kk) __attribute__((always_inline)) {
    return Pair{*reinterpret_cast<const bf16x8*>(kt + (koff ^ 32 * kk)),
                *reinterpret_cast<const bf16x8*>(kt + (koff ^ 32 * kk) + 32 * 2 * DP)};
  };
  auto values = [&](int i) __attribute__((always_inline)) {
    const unsigned char* const from = vt + i / NPAIR * 16 * 2 * DP;
    Pair v;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int db = 2 * (i % NPAIR) + x;
      v.x[x] = join8(__builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                         (bf16x4 GLACIER_LDS*)(const_cast<unsigned char*>(from + (voff0 ^ 64 * db)))),
                     __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                         (bf16x4 GLACIER_LDS*)(const_cast<unsigned char*>(from + (voff1 ^ 64 * db)))));
    }
    return v;
  };
  Pair f = keys(0);
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk) {
    const Pair next = kk + 1 < NKK ? keys(kk + 1) : values(0);
    keep_order();
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) sn[kb] = mma16(f.x[kb], qf[kk], sn[kb]);
    weights(2 * (8 * kk / NKK), 2 * (8 * (kk + 1) / NKK));
    keep_order();
    f = next;
  }
#pragma unroll
  for (int i = 0; i < 4 * NPAIR; ++i) {
    const int sp = i / NPAIR, db = 2 * (i % NPAIR);
    Pair next;
    if (i + 1 < 4 * NPAIR) next = values(i + 1);
    keep_order();
#pragma unroll
    for (int x = 0; x < 2; ++x) w.o[db + x] = mma16(f.x[x], __builtin_bit_cast(bf16x8, lo[sp]), w.o[db + x]);
#pragma unroll
    for (int x = 0; x < 2; ++x) w.o[db + x] = mma16(f.x[x], __builtin_bit_cast(bf16x8, hi[sp]), w.o[db + x]);
    if (sp < 2) weights(16 + 8 * i / NPAIR, 16 + 8 * (i + 1) / NPAIR);
    if (i == 2 * NPAIR) w.top = wide_largest(sn);
    keep_order();
    f = next;
  }
  w.l += sum;
}

template <int DP>
__global__ __launch_bounds__(64 * kWavesWide, DP <= 128 ? 2 : 1) void cache_attn_wide_kernel(CacheAttn a) {
  using W = Wide<DP>;
  extern __shared__ __align__(16) unsigned char smem[];
  const CacheView& c = a.c;
  const int w = wave_id(), lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  const int kvh = blockIdx.x % c.hkv, split = blockIdx.y, D = c.D;
  int tile;
  const CacheSeq s = seq_of_long_tile(a, lane, static_cast<int>(blockIdx.x / c.hkv),
                                      static_cast<int>(gridDim.x / c.hkv), tile);
  const int b = s.b;
  if (b >= c.n_seqs) return;
  const int r0 = tile * kRowsWide, n_rows = s.n * a.group;
  if (tile < 0 || r0 >= n_rows) return;
  const TileKeys tk = tile_keys(a, s, tile);
  if (split >= tk.active) return;
  const int k0 = split * tk.per, k1 = min(tk.kend, k0 + tk.per);

  // this lane's row, its query fragments and its last key
  const int r = r0 + 32 * w + col, tok = r / a.group;
  const bool live = r < n_rows;
  const int limit = live ? s.pos0 + tok : -1;
  const long at = (long)(s.tok0 + tok) * a.hq + kvh * a.group + (r - tok * a.group);
  bf16x8 qf[W::NKK];
  {
    // (from the tile's first row where there is none, and cleared after all
    // loads are under way)
    const bf16* const q = static_cast<const bf16*>(a.q) +
                          (live ? at : (long)(s.tok0 + r0 / a.group) * a.hq) * D;
#pragma unroll
    for (int kk = 0; kk < W::NKK; ++kk)
      qf[kk] = *reinterpret_cast<const bf16x8*>(q + (16 * kk + 8 * h < D ? 16 * kk + 8 * h : 0));
#pragma unroll
    for (int kk = 0; kk < W::NKK; ++kk)
      if (!live || 16 * kk + 8 * h >= D) qf[kk] = frag_zero<bf16>();
  }
  // a wave's rows see keys first_limit at least, and none past last_limit
  const int wr = r0 + 32 * w;
  const int first_limit = s.pos0 + wr / a.group;
  const int last_limit = wr < n_rows ? s.pos0 + min(s.n - 1, (wr + 31) / a.group) : -1;

  // LDS offsets of this lane's reads in block 0 (block kk of K is 32 kk away by an
  // exclusive or, block db of V 64 db): K pieces of row col; V pieces of rows
  // 4 h + 8 u + (lane % 16) / 4 at columns 16 (lane / 16 % 2) + 4 (lane % 4)
  const int koff = col * W::RB + 16 * (h ^ lds_sw<DP>(col));
  auto v_off = [&](int u) {
    const int gr = lane >> 4, ra = (lane & 15) >> 2, cb = lane & 3;
    const int row = 8 * u + 4 * h + ra, piece = 2 * (gr & 1) + (cb >> 1);
    return row * W::RB + 16 * (piece ^ lds_sw<DP>(row)) + 8 * (cb & 1);
  };
  const int voff0 = v_off(0), voff1 = v_off(1);

  // A tile is four page pieces of 16 keys; a wave brings one of them, of K and
  // of V.  The piece is read through a buffer resource that
  // ends with its last key (none without a page): what lies past it, and past
  // column D, arrives as zero.
  const int rowb = 2 * D;
  int doff[W::ND];
#pragma unroll
  for (int n = 0; n < W::ND; ++n) {
    const int row = n * (1024 / W::RB) + lane / W::PPR, piece = lane % W::PPR ^ lds_sw<DP>(row);
    doff[n] = 8 * piece < D ? row * rowb + 16 * piece : 1 << 20;
  }
  const int in_page = (1 << c.page_shift) - 1;
  const long head = ((long)kvh << c.page_shift) * rowb, strideb = 2 * c.page_stride;
  // the page of this wave's piece of tile j (-1: none), by a scalar load: a
  // vector load would make the wave wait for every DMA it has in flight
  const auto* const table = (const __attribute__((address_space(4))) int32_t*)(
      reinterpret_cast<uintptr_t>(c.table + (long)b * c.table_stride));
  auto look_up = [&](int j) {
    const int at = (j + 16 * w) >> c.page_shift;
    const int page = table[min(at, c.max_pages - 1)];
    return j + 16 * w < k1 && static_cast<unsigned>(page) < static_cast<unsigned>(c.n_pages) ? page : -1;
  };
  auto bring = [&](const void* pages, unsigned char* to, int j, int page) {
    const int key = j + 16 * w;
    const long off = (page < 0 ? 0 : page) * strideb + head + (key & in_page) * rowb;
    const int bytes = (page < 0 ? 0 : min(16, k1 - key)) * rowb;
#pragma unroll
    for (int n = 0; n < W::ND; ++n)
      dma16(static_cast<const char*>(pages) + off, bytes, doff[n], to + w * 16 * W::RB + 1024 * n);
  };
  auto k_slot = [&](int i) { return smem + i * W::TILE; };
  auto v_slot = [&](int i) { return smem + (2 + i) * W::TILE; };
  unsigned* const notes = reinterpret_cast<unsigned*>(smem + W::NOTES);
  // (second walk) clears what is not finite in this wave's piece of V
  auto look_through = [&](unsigned char* v, int j) {
    unsigned found = 0;
#pragma unroll
    for (int n = 0; n < W::ND; ++n) {
      i32x4* const at = reinterpret_cast<i32x4*>(v + w * 16 * W::RB + 1024 * n + 16 * lane);
      i32x4 x = *at;
      found |= clear_not_finite<bf16>(x);
      *at = x;
    }
    const int block = (j - k0) / kKeysWide % kNotedBlocks;
    if (__any(found != 0) && lane == 0) atomicOr(&notes[block / 32], 1u << block % 32);
  };
  // whether every piece of the keys has a page (if not, each tile is looked at)
  bool clean = true;
  for (int p = (k0 >> c.page_shift) + lane; p <= (k1 - 1) >> c.page_shift; p += 64)
    clean = clean && cache_page(c, b, p << c.page_shift) >= 0;
  clean = __all(clean);

  WideState<DP> ws;
  f32x16 sa[2], sb[2];
  int v_page = -1, k_page = -1;  // of the next V tile and of the K tile after it
  auto tile_step = [&](f32x16 (&st)[2], f32x16 (&sn)[2], int j, int odd, auto careful) __attribute__((always_inline)) {
    bring(c.k_pages, k_slot(odd), j + 2 * kKeysWide, k_page);
    bring(c.v_pages, v_slot(odd ^ 1), j + kKeysWide, v_page);
    v_page = k_page;
    k_page = look_up(j + 3 * kKeysWide);
    __builtin_amdgcn_sched_barrier(0);
    if (j <= last_limit) {
      if (j + kKeysWide - 1 > first_limit || j + kKeysWide > k1 || !clean) {
        const int at = j + 16 * (lane & 3);
        const int held = clean ? 15 : static_cast<int>(__ballot(at < k1 && cache_page(c, b, at) >= 0)) & 15;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = j + 32 * kb + 8 * (e / 4) + 4 * h + e % 4;
            st[kb][e] = (held >> (2 * kb + e / 8) & 1) && key < k1 && key <= limit ? st[kb][e] : -INFINITY;
          }
        ws.top = wide_largest(st);
      }
      wide_step<DP, careful()>(ws, st, sn, k_slot(odd ^ 1), v_slot(odd), koff, voff0, voff1, qf, a.scale_log2);
    }
    vmw<0>();
    if constexpr (careful()) look_through(v_slot(odd ^ 1), j + kKeysWide);
    lgkm<0>();
    wg_barrier();
  };
  auto walk = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < W::NDB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) ws.o[db][e] = 0.0f;
    ws.m = kLeast;
    ws.l = 0.0f;
    ws.top = kLeast;
    if (k0 < k1) {
      const int first = look_up(k0);
      v_page = look_up(k0 + kKeysWide);
      k_page = look_up(k0 + 2 * kKeysWide);
      bring(c.k_pages, k_slot(0), k0, first);
      bring(c.v_pages, v_slot(0), k0, first);
      bring(c.k_pages, k_slot(1), k0 + kKeysWide, v_page);
      vmw<0>();
      if constexpr (careful()) look_through(v_slot(0), k0);
      lgkm<0>();
      wg_barrier();
      wide_scores<DP>(sa, k_slot(0), koff, qf);
      ws.top = wide_largest(sa);
      lgkm<0>();
      wg_barrier();
    }
    for (int j = k0; j < k1; j += 2 * kKeysWide) {
      tile_step(sa, sb, j, 0, careful);
      if (j + kKeysWide < k1) tile_step(sb, sa, j + kKeysWide, 1, careful);
    }
  };
  walk(std::false_type{});
  // not finite, or no weight although the row sees keys (a tile's last row sees
  // them all, so that nothing in V escapes it)
  const float first_sum = swap_sum(ws.l, false);
  unsigned odd = not_finite(first_sum) | not_finite(__builtin_amdgcn_rcpf(first_sum));
#pragma unroll
  for (int db = 0; db < W::NDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) odd |= not_finite(ws.o[db][e]);
  if (__syncthreads_or(odd != 0 && limit >= k0)) {
    if (threadIdx.x < kNotedBlocks / 32) notes[threadIdx.x] = 0;
    __syncthreads();
    walk(std::true_type{});
    __syncthreads();
    for (int j = k0; j < k1; j += kKeysWide) {
      const int block = (j - k0) / kKeysWide % kNotedBlocks;
      if (!(notes[block / 32] >> block % 32 & 1)) continue;
      for (int key = j; key < min(k1, j + kKeysWide); ++key) {
        const int page = cache_page(c, b, key);
        if (page < 0) continue;
        const char* const v = static_cast<const char*>(c.v_pages) + page * strideb + head + (key & in_page) * rowb;
        const unsigned sees = key <= limit ? ~0u : 0u;
#pragma unroll
        for (int db = 0; db < W::NDB; ++db)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const bf16x4 x = __builtin_bit_cast(bf16x4, load8_within(v, rowb, 2 * (32 * db + 8 * q + 4 * h)));
#pragma unroll
            for (int e = 0; e < 4; ++e) ws.o[db][4 * q + e] += given_back((float)x[e], sees);
          }
      }
    }
  }
  f32x16 (&o)[W::NDB] = ws.o;
  const float m = ws.m;
  float l = ws.l;
  if (!live) return;
  l = swap_sum(l, false);
  // elements 4 q .. 4 q + 3 of block db are columns 32 db + 8 q + 4 h ..
  const bool whole = tk.active <= 1;
  const float inv = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;  // no key: the row is zero
  const long slot = (long)split * c.T * a.hq + at;
#pragma unroll
  for (int db = 0; db < W::NDB; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * db + 8 * q + 4 * h;
      if (d >= D) continue;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[db][4 * q + e] * inv;
      if (whole)
        store4(static_cast<bf16*>(a.out) + at * D + d, v);
      else
        store4(a.part_o + slot * D + d, v);
    }
  if (h != 0) return;
  if (!whole)
    a.part_ml[slot] = make_float2(m, l);
  else if (a.lse != nullptr)
    a.lse[(at % a.hq) * c.T + at / a.hq] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

__device__ inline float masked(float x, unsigned kept) {
  return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & kept);
}

// Joins the splits of a tile's rows, 32 of them a workgroup: D / 4 lanes to a
// row, four splits' sums in flight.  (A wave for each row, as after the 16-row
// kernel, spends more on finding the row's sequence than on joining it: 84 us
// for 16 sequences of up to 128 new tokens and 2048 keys that need 54 whole.)
constexpr int kJoinRows = 32;
__global__ __launch_bounds__(256) void cache_join_tiles_kernel(CacheAttn a) {
  const CacheView& c = a.c;
  const int lane = threadIdx.x & 63;
  const int kvh = blockIdx.x % c.hkv, number = blockIdx.x / c.hkv;
  const CacheSeq s = seq_of_tile(a, lane, number);
  if (s.b >= c.n_seqs) return;
  const int tile = number - first_tile(a, s.b, s.tok0);
  const int r0 = tile * kRowsWide + blockIdx.y * kJoinRows, n_rows = s.n * a.group;
  if (tile < 0 || r0 >= n_rows) return;
  const TileKeys tk = tile_keys(a, s, tile);
  if (tk.active <= 1) return;
  const int lanes = c.D <= 64 ? 16 : c.D <= 128 ? 32 : 64, d = 4 * (threadIdx.x % lanes);
  const long step = (long)c.T * a.hq;
  for (int r = r0 + threadIdx.x / lanes; r < min(n_rows, r0 + kJoinRows); r += 256 / lanes) {
    const int tok = r / a.group, h = kvh * a.group + (r - tok * a.group);
    const long t = s.tok0 + tok, at = t * a.hq + h;
    float mx = kLeast, total = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int u0 = 0; u0 < tk.active; u0 += 4) {
      float2 ml[4];
      f32x4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long slot = min(u0 + i, tk.active - 1) * step + at;
        ml[i] = a.part_ml[slot];
        v[i] = *reinterpret_cast<const f32x4*>(a.part_o + slot * c.D + (d < c.D ? d : 0));
      }
      float top = mx;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i].x);
      const float f = weight(mx - top);
      mx = top;
      total *= f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (a weight of zero is not enough where the sums are infinite; by a mask, as a
        // choice becomes a branch with the load in it)
        unsigned kept = u0 + i < tk.active ? ~0u : 0u;
        asm volatile("" : "+v"(kept));
        const float g = masked(weight(ml[i].x - mx), kept);
        total += g * ml[i].y;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += g * masked(v[i][e], kept);
      }
    }
    if (d >= c.D) continue;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    store4(static_cast<bf16*>(a.out) + at * c.D + d, o);
    if (a.lse != nullptr && d == 0)
      a.lse[(long)h * c.T + t] = total == 0.0f ? -INFINITY : (mx + log2f(total)) * kLn2;
  }
}

template <int DP>
hipError_t attend(const CacheAttn& a, hipStream_t st) {
  auto* fn = &cache_attn_wide_kernel<DP>;
  GL_CHECK(allow_lds(fn, Wide<DP>::BYTES));
  hipLaunchKernelGGL((cache_attn_wide_kernel<DP>), dim3(tile_numbers(a) * a.c.hkv, a.n_splits),
                     dim3(64 * kWavesWide), Wide<DP>::BYTES, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_attn_wide(const CacheAttn& a, hipStream_t st) {
  static_assert(kRowsWide == kCacheWideRows, "rows of a wide tile");
  GL_CHECK(a.c.D <= 64 ? attend<64>(a, st) : a.c.D <= 128 ? attend<128>(a, st) : attend<256>(a, st));
  if (a.n_splits == 1 || a.n_splits > kCacheTileJoin) return hipSuccess;
  hipLaunchKernelGGL(cache_join_tiles_kernel, dim3(tile_numbers(a) * a.c.hkv, kRowsWide / kJoinRows),
                     dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace glacier
