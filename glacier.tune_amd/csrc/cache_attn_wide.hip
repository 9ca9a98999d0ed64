// cache_attn_wide.hip -- attention of chunks of new tokens over the paged
// cache on 32x32x16 MFMAs: bf16, head sizes up to 128, many rows.
//
// A workgroup takes 128 rows (token, head of the group) of one KV head, 32 a
// wave, and walks the keys 64 at a time; two workgroups share a CU, so one's
// softmax runs beside the other's products.  K and V tiles come page by page
// through registers into two LDS buffers, the next tile's loads in flight
// during a tile's products, with one barrier a tile.  Rows of 16-byte pieces
// are swizzled (lds_sw, lds_mfma.hpp), which keeps both reads free of bank
// conflicts.
//
// Scores are formed transposed: S^T = K Q^T leaves a lane with 16 keys of one
// row in each accumulator block, and elements 8 s .. 8 s + 7 are the k-slots of
// step s of O^T += V^T P^T, whose V operand comes from two transposing LDS
// reads (the accumulator layout is described in attn_bwd3.hip).
//
// The running maximum is only followed where it has grown by more than 8 (in
// log2): until then weights are taken against the old one, at most 2^8 large,
// and the sums need no rescaling.  The result is the same: any reference value
// cancels in out and lse.
#include "cache_tiles.hpp"

namespace glacier {
namespace {

constexpr int kWavesWide = 4;
constexpr int kRowsWide = 32 * kWavesWide;
constexpr int kKeysWide = 64;
constexpr float kGrowth = 8.0f;

template <int DP>
struct Wide {
  static constexpr int RB = 2 * DP;           // bytes of an LDS row
  static constexpr int PPR = DP / 8;          // 16-byte pieces of a row
  static constexpr int RPI = 64 * kWavesWide / PPR;  // rows one load of all threads covers
  static constexpr int NI = kKeysWide / RPI;  // loads per thread of a K or V tile
  static constexpr int TILE = kKeysWide * RB;
  static constexpr int BYTES = 4 * TILE;  // K and V, two buffers
  static constexpr int NKK = DP / 16, NDB = DP / 32;
};

__device__ inline f32x16 mma16(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <int DP>
__global__ __launch_bounds__(64 * kWavesWide, 2) void cache_attn_wide_kernel(CacheAttn a) {
  using W = Wide<DP>;
  extern __shared__ __align__(16) unsigned char smem[];
  const CacheView& c = a.c;
  const int w = wave_id(), lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  const int kvh = blockIdx.y, split = blockIdx.z, D = c.D;
  // later tiles see more keys: they start first
  const int number = static_cast<int>(gridDim.x - 1 - blockIdx.x);

  const CacheSeq s = seq_of_tile(a, lane, number);
  const int b = s.b;
  if (b >= c.n_seqs) return;
  const int tile = number - first_tile(a, b, s.tok0);
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

  f32x16 o[W::NDB];
#pragma unroll
  for (int db = 0; db < W::NDB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[db][e] = 0.0f;
  float m = kNegBig, l = 0.0f;

  // LDS offsets of this lane's reads: K pieces of row col; V pieces of rows
  // 4 h + 8 u + (lane % 16) / 4 at columns 32 db + 16 (lane / 16 % 2) + 4 (lane % 4)
  int koff[W::NKK], voff[W::NDB][2];
#pragma unroll
  for (int kk = 0; kk < W::NKK; ++kk) koff[kk] = col * W::RB + 16 * ((2 * kk + h) ^ lds_sw<DP>(col));
  {
    const int gr = lane >> 4, ra = (lane & 15) >> 2, cb = lane & 3;
#pragma unroll
    for (int db = 0; db < W::NDB; ++db)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = 8 * u + 4 * h + ra, piece = 4 * db + 2 * (gr & 1) + (cb >> 1);
        voff[db][u] = row * W::RB + 16 * (piece ^ lds_sw<DP>(row)) + 8 * (cb & 1);
      }
  }

  // this thread's share of a tile: rows row0 + RPI i, piece `piece`.  The 16
  // rows of a page piece are read through a buffer resource that ends with the
  // last one that holds a key (none without a page): what lies past it, and
  // past column D, arrives as zero, with no branch and no address arithmetic
  // in vector registers.
  const int piece = threadIdx.x % W::PPR, row0 = threadIdx.x / W::PPR;
  const int wrow0 = w * (64 / W::PPR);  // the wave's rows of one load lie in one page piece
  const int rowb = 2 * D;
  const int loff = 8 * piece < D ? (row0 & 15) * rowb + 16 * piece : 1 << 20;
  int soff[W::NI];
#pragma unroll
  for (int i = 0; i < W::NI; ++i) {
    const int row = row0 + i * W::RPI;
    soff[i] = row * W::RB + 16 * (piece ^ lds_sw<DP>(row));
  }
  const int in_page = (1 << c.page_shift) - 1;
  const long head = ((long)kvh << c.page_shift) * rowb, strideb = 2 * c.page_stride;
  // the pages of a tile's four pieces of 16 keys, one a lane; none (-1) past k1
  auto look_up = [&](int j) {
    const int key = j + 16 * (lane & 3);
    return key < k1 ? cache_page(c, b, key) : -1;
  };
  i32x4 kr[W::NI], vr[W::NI];
  auto fetch = [&](int j, int pages) {
#pragma unroll
    for (int i = 0; i < W::NI; ++i) {
      const int key = j + (wrow0 + i * W::RPI) / 16 * 16;
      const int page = __builtin_amdgcn_readlane(pages, (wrow0 + i * W::RPI) / 16);
      const long off = (page < 0 ? 0 : page) * strideb + head + (key & in_page) * rowb;
      const int rows = page < 0 ? 0 : min(16, k1 - key);
      kr[i] = load_within(static_cast<const char*>(c.k_pages) + off, rows * rowb, loff);
      vr[i] = load_within(static_cast<const char*>(c.v_pages) + off, rows * rowb, loff);
    }
  };
  auto put = [&](int buf) {
    unsigned char* const t = smem + buf * 2 * W::TILE;
#pragma unroll
    for (int i = 0; i < W::NI; ++i) {
      *reinterpret_cast<i32x4*>(t + soff[i]) = kr[i];
      *reinterpret_cast<i32x4*>(t + W::TILE + soff[i]) = vr[i];
    }
  };

  int next = look_up(k0), held = 0;  // held: which pieces of the tile in LDS have a page
  if (k0 < k1) {
    const int pages = next;
    next = look_up(k0 + kKeysWide);
    fetch(k0, pages);
    held = static_cast<int>(__ballot(pages >= 0)) & 15;
    put(0);
  }
  __syncthreads();
  int buf = 0;
  for (int j = k0; j < k1; j += kKeysWide, buf ^= 1) {
    const bool more = j + kKeysWide < k1;
    int held_next = 0;
    if (more) {
      const int pages = next;
      next = look_up(j + 2 * kKeysWide);
      fetch(j + kKeysWide, pages);
      held_next = static_cast<int>(__ballot(pages >= 0)) & 15;
    }
    if (j <= last_limit) {
      const unsigned char* const kt = smem + buf * 2 * W::TILE;
      const unsigned char* const vt = kt + W::TILE;
      f32x16 st[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int e = 0; e < 16; ++e) st[kb][e] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < W::NKK; ++kk)
          st[kb] = mma16(*reinterpret_cast<const bf16x8*>(kt + koff[kk] + kb * 32 * W::RB), qf[kk], st[kb]);
      }
      if (j + kKeysWide - 1 > first_limit || j + kKeysWide > k1 || held != 15) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = j + 32 * kb + 8 * (e / 4) + 4 * h + e % 4;
            st[kb][e] = (held >> (2 * kb + e / 8) & 1) && key < k1 && key <= limit ? st[kb][e] : -INFINITY;
          }
      }
      float top = st[0][0];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, st[kb][e]);
      top = swap_max(top, false) * a.scale_log2;
      if (__any(top > m + kGrowth)) {
        const float mn = fmaxf(m, top);
        const float f = weight(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int db = 0; db < W::NDB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[db][e] *= f;
      }
      bf16x8 pf[4];
      float sum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = weight(fmaf(st[kb][e], a.scale_log2, -m));
          sum += p;
          pf[2 * kb + e / 8][e % 8] = (bf16)p;
        }
      l += sum;
#pragma unroll
      for (int sp = 0; sp < 4; ++sp)
#pragma unroll
        for (int db = 0; db < W::NDB; ++db) {
          const unsigned char* const p = vt + sp * 16 * W::RB;
          const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
              (bf16x4 GLACIER_LDS*)(const_cast<unsigned char*>(p + voff[db][0])));
          const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
              (bf16x4 GLACIER_LDS*)(const_cast<unsigned char*>(p + voff[db][1])));
          o[db] = mma16(join8(lo, hi), pf[sp], o[db]);
        }
    }
    if (more) put(buf ^ 1);
    held = held_next;
    __syncthreads();
  }
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

template <int DP>
hipError_t attend(const CacheAttn& a, hipStream_t st) {
  auto* fn = &cache_attn_wide_kernel<DP>;
  GL_CHECK(allow_lds(fn, Wide<DP>::BYTES));
  hipLaunchKernelGGL((cache_attn_wide_kernel<DP>), dim3(tile_numbers(a), a.c.hkv, a.n_splits),
                     dim3(64 * kWavesWide), Wide<DP>::BYTES, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_attn_wide(const CacheAttn& a, hipStream_t st) {
  static_assert(kRowsWide == kCacheWideRows, "rows of a wide tile");
  return a.c.D <= 64 ? attend<64>(a, st) : attend<128>(a, st);
}

}  // namespace glacier
