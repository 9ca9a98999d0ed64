// cache_attn.hip -- attention of new tokens over a paged key/value cache.
//
// The query heads of a KV head's group read the same keys, so a tile's rows
// are (token, head of the group) pairs, token by token: row r of a sequence is
// token r / group, head r % group.  One new token of 7 heads and a long chunk
// are then the same product, and K and V are read once per tile, not per head.
//
// A workgroup takes one tile of one KV head, and one split of the keys the
// tile sees.  Its four waves take keys in turn, KB at a time, each with its own
// LDS tiles and its own running maximum and sum of the softmax, so the loop
// has no barrier; the waves are joined through LDS at the end.  Scores are
// formed transposed (S^T = K Q^T, attn_common.hpp), which leaves a lane with
// one row's weights and feeds them to O^T += V^T P^T as they are.
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

constexpr int kWavesCa = 4;

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

template <typename T, int DP, int MB>
struct CaLayout {
  static constexpr int KB = KeyBlock<T>::KB;
  static constexpr int S = Lds<T, DP>::STRIDE;
  static constexpr int TILES = kWavesCa * 2 * KB * S * static_cast<int>(sizeof(T));
  static constexpr int OS = DP + 4;  // row stride (floats) of a wave's sums in the join
  static constexpr int WAVE = 16 * MB * (OS + 2);  // sums, maxima, totals
  static constexpr int JOIN = kWavesCa * WAVE * 4;
  static constexpr int BYTES = TILES > JOIN ? TILES : JOIN;
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
  // rows of one page piece (16 keys) each from base[piece]; rows at or past
  // nvalid, pieces without a page and columns at or past D read as zero
  __device__ inline void load(const T* const (&base)[KB / 16], const bool (&held)[KB / 16], int D,
                              int nvalid, int lane) {
    const int ch = lane % LPR;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = i * RPI + lane / LPR;
      w[i] = i32x4{0, 0, 0, 0};
      if (held[i * RPI / 16] && r < nvalid && ch * CE < D)
        w[i] = *reinterpret_cast<const i32x4*>(base[i * RPI / 16] + (long)(r & 15) * D + ch * CE);
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

__device__ inline void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename T, int DP, int MB>
__global__ __launch_bounds__(64 * kWavesCa) void cache_attn_kernel(CacheAttn a) {
  using M = Mfma<T>;
  using L = CaLayout<T, DP, MB>;
  constexpr int KB = L::KB, NS = KB / 16, NKD = DP / M::KSTEP, ROWS = 16 * MB;
  extern __shared__ __align__(16) unsigned char smem[];
  const CacheView& c = a.c;
  const int w = wave_id(), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
  const int kvh = blockIdx.y, split = blockIdx.z, D = c.D;

  const int b = __builtin_amdgcn_readfirstlane(count_prefix(
      c.n_seqs, lane, [&](int i) { return first_tile(a, i + 1) <= static_cast<int>(blockIdx.x); }));
  if (b >= c.n_seqs) return;
  const CacheSeq s = cache_seq(c, b);
  const int tile = static_cast<int>(blockIdx.x) - first_tile(a, b);
  const int r0 = tile * ROWS, n_rows = s.n * a.group;
  if (tile < 0 || r0 >= n_rows) return;
  const TileKeys tk = tile_keys(a, s, tile);
  if (split >= tk.active) return;
  const int k0 = split * tk.per, k1 = min(tk.kend, k0 + tk.per);

  // this lane's rows (one per 16-row block): operand fragments and last key
  typename M::Frag qf[MB][NKD];
  int limit[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int r = r0 + 16 * mb + col;
    const int i = r / a.group, h = kvh * a.group + (r - i * a.group);
    const bool ok = r < n_rows;
    limit[mb] = ok ? s.pos0 + i : -1;
    const T* q = static_cast<const T*>(a.q) + ((long)(s.tok0 + i) * a.hq + h) * D;
#pragma unroll
    for (int kk = 0; kk < NKD; ++kk) {
      qf[mb][kk] = frag_zero<T>();
      if (ok && kk * M::KSTEP + M::KPL * g < D) qf[mb][kk] = frag_global<T>(q, kk, g);
    }
  }

  f32x4 acc[MB][DP / 16];
  float m[MB], l[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    m[mb] = kNegBig;
    l[mb] = 0.0f;
#pragma unroll
    for (int db = 0; db < DP / 16; ++db) acc[mb][db] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  T* const kt = reinterpret_cast<T*>(smem) + w * 2 * KB * L::S;
  T* const vt = kt + KB * L::S;
  BlockRegs<T, DP> kr, vr;
  bool held[NS];
  auto fetch = [&](int j) {
    const T *kb[NS], *vb[NS];
#pragma unroll
    for (int p = 0; p < NS; ++p) {
      const int key = j + 16 * p;
      const int page = key < k1 ? __builtin_amdgcn_readfirstlane(cache_page(c, b, key)) : -1;
      held[p] = page >= 0;
      const long at = (page >= 0 ? page : 0) * c.page_stride +
                      (((long)kvh << c.page_shift) + (key & ((1 << c.page_shift) - 1))) * D;
      kb[p] = static_cast<const T*>(c.k_pages) + at;
      vb[p] = static_cast<const T*>(c.v_pages) + at;
    }
    kr.load(kb, held, D, k1 - j, lane);
    vr.load(vb, held, D, k1 - j, lane);
  };
  const int first_limit = s.pos0 + r0 / a.group;  // the tile's first row sees keys up to here
  int j = k0 + w * KB;
  if (j < k1) fetch(j);
  for (; j < k1; j += kWavesCa * KB) {
    wave_lds_fence();
    kr.store(kt, lane);
    vr.store(vt, lane);
    wave_lds_fence();
    bool here[NS], whole = j + KB - 1 <= first_limit && j + KB <= k1;
#pragma unroll
    for (int p = 0; p < NS; ++p) {
      here[p] = held[p];
      whole = whole && held[p];
    }
    if (j + kWavesCa * KB < k1) fetch(j + kWavesCa * KB);
    // S^T: keys 16 p + 4 g + r of this block, row col of each 16-row block
    f32x4 st[MB][NS];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int p = 0; p < NS; ++p) st[mb][p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int p = 0; p < NS; ++p)
#pragma unroll
      for (int kk = 0; kk < NKD; ++kk) {
        const auto kf = frag_rm<T, DP>(kt, 16 * p + col, kk, g);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) st[mb][p] = M::mma(kf, qf[mb][kk], st[mb][p]);
      }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      float top = kNegBig;
#pragma unroll
      for (int p = 0; p < NS; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = st[mb][p][r] * a.scale_log2;
          if (!whole) {
            const int key = j + 16 * p + 4 * g + r;
            x = here[p] && key < k1 && key <= limit[mb] ? x : -INFINITY;
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
    // O^T += V^T P^T
    if constexpr (sizeof(T) == 2) {
      bf16x8 pf[MB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          pf[mb][r] = (bf16)st[mb][0][r];
          pf[mb][4 + r] = (bf16)st[mb][NS - 1][r];
        }
#pragma unroll
      for (int db = 0; db < DP / 16; ++db) {
        const bf16x4 lo = read_tr<L::S>(vt, 0, 16 * db, lane);
        const bf16x4 hi = read_tr<L::S>(vt, 16, 16 * db, lane);
        bf16x8 vf;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          vf[r] = lo[r];
          vf[4 + r] = hi[r];
        }
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[mb][db] = M::mma(vf, pf[mb], acc[mb][db]);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int db = 0; db < DP / 16; ++db) {
          const float vf = vt[(4 * g + r) * L::S + 16 * db + col];
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) acc[mb][db] = M::mma(vf, st[mb][0][r], acc[mb][db]);
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
#pragma unroll
    for (int db = 0; db < DP / 16; ++db)
      store4(mine + row * L::OS + 16 * db + 4 * g, acc[mb][db]);
    if (g == 0) {
      mine[ROWS * L::OS + row] = m[mb];
      mine[ROWS * (L::OS + 1) + row] = total;
    }
  }
  __syncthreads();
  const float* const all = reinterpret_cast<const float*>(smem);
  constexpr int CPR = DP / 4;
  for (int idx = threadIdx.x; idx < ROWS * CPR; idx += 64 * kWavesCa) {
    const int row = idx / CPR, d = 4 * (idx % CPR), r = r0 + row;
    if (r >= n_rows || d >= D) continue;
    float mx = kNegBig;
#pragma unroll
    for (int u = 0; u < kWavesCa; ++u) mx = fmaxf(mx, all[u * L::WAVE + ROWS * L::OS + row]);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float total = 0.0f;
#pragma unroll
    for (int u = 0; u < kWavesCa; ++u) {
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

// Joins the splits of a row: one wave each, four to a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void cache_attn_join_kernel(CacheAttn a) {
  const CacheView& c = a.c;
  const int lane = threadIdx.x & 63;
  const long at = (long)blockIdx.x * 4 + wave_id();
  if (at >= (long)c.T * a.hq) return;
  const int t = static_cast<int>(at / a.hq), h = static_cast<int>(at % a.hq);
  const int b = __builtin_amdgcn_readfirstlane(
      count_prefix(c.n_seqs, lane, [&](int i) { return c.cu[i + 1] <= t; }));
  if (b >= c.n_seqs) return;
  const CacheSeq s = cache_seq(c, b);
  if (t < s.tok0) return;
  const TileKeys tk = tile_keys(a, s, ((t - s.tok0) * a.group + h % a.group) / a.rows);
  if (tk.active <= 1) return;
  const long step = (long)c.T * a.hq;
  float2 ml = make_float2(kNegBig, 0.0f);
  if (lane < tk.active) ml = a.part_ml[lane * step + at];
  float mx = ml.x;
#pragma unroll
  for (int x = 1; x < 64; x *= 2) mx = fmaxf(mx, __shfl_xor(mx, x));
  const float f = weight(ml.x - mx);
  float total = f * ml.y;
#pragma unroll
  for (int x = 1; x < 64; x *= 2) total += __shfl_xor(total, x);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int d = 4 * lane;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int u = 0; u < tk.active; ++u) {
    const float fu = __shfl(f, u);
    if (d < c.D) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(a.part_o + (u * step + at) * c.D + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += fu * v[e];
    }
  }
  if (d < c.D) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    store4(static_cast<T*>(a.out) + at * c.D + d, o);
  }
  if (a.lse != nullptr && lane == 0)
    a.lse[(long)h * c.T + t] = total == 0.0f ? -INFINITY : (mx + log2f(total)) * kLn2;
}

template <typename T, int DP, int MB>
hipError_t attend(const CacheAttn& a, hipStream_t st) {
  using L = CaLayout<T, DP, MB>;
  auto* fn = &cache_attn_kernel<T, DP, MB>;
  GL_CHECK(allow_lds(fn, L::BYTES));
  hipLaunchKernelGGL((cache_attn_kernel<T, DP, MB>), dim3(tile_numbers(a), a.c.hkv, a.n_splits),
                     dim3(64 * kWavesCa), L::BYTES, st, a);
  return hipGetLastError();
}

template <typename T>
hipError_t join(const CacheAttn& a, hipStream_t st) {
  const long rows = (long)a.c.T * a.hq;
  hipLaunchKernelGGL(cache_attn_join_kernel<T>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0,
                     st, a);
  return hipGetLastError();
}

template <typename T>
hipError_t by_head(const CacheAttn& a, hipStream_t st) {
  const int d = a.c.D;
  if (d <= 32) return attend<T, 32, 1>(a, st);
  if (d <= 64) return attend<T, 64, 1>(a, st);
  if (d <= 96) return attend<T, 96, 1>(a, st);
  if (d <= 128) return attend<T, 128, 1>(a, st);
  return attend<T, 256, 1>(a, st);
}

}  // namespace

CachePlan cache_attn_plan(const CacheView& c, int hq, int max_new, int max_kv, int n_cu) {
  CachePlan p{};
  const long group = hq / c.hkv;
  const long cap = (long)c.max_pages << c.page_shift;
  const long keys = max_kv > 0 && max_kv < cap ? max_kv : cap;
  const long longest = max_new > 0 && max_new < c.T ? max_new : c.T;  // chunk
  p.rows = c.io_bf16 && c.D <= 128 && longest * group > 64 ? kCacheWideRows : 16;
  const long tiles = (c.T * group + p.rows - 1) / p.rows + std::min(c.T, c.n_seqs) / 2;
  // enough workgroups for two on each CU, of 256 keys or more
  const long want = 2L * n_cu / std::max(1L, tiles * c.hkv);
  const long most = (keys + 255) / 256;
  p.n_splits = static_cast<int>(std::max(1L, std::min({want, most, (long)kMaxSplits})));
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
  if (a.n_splits == 1) return hipSuccess;
  return a.c.io_bf16 ? join<bf16>(a, st) : join<float>(a, st);
}

}  // namespace glacier
