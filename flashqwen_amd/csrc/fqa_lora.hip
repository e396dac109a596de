// fqa_lora.hip — low-rank adapters of many requests beside a shared projection (gfx950).
//
// With adapter a of row t, slice s(n) of output column n and that adapter's rank r_a:
//   h[t, s, j] = sum_k x[t, k] A[a, s R + j, k]                                  (j < r_a)
//   y[t, n]    = y_in[t, n] + scale[a] sum_j h[t, s(n), j] B[a, n, j]
// The step's plan groups its rows by adapter, once per step (7.5 us for 64 requests and 16 adapters,
// 12.7 for 2000 and 200: barriers and LDS scans of one workgroup, its bytes are nothing).  A
// projection then takes two launches: the product with A (h, fp32, in the plan's row order, a plane
// for every split of K) and the product with B (added to y_in).  Both are bound by bytes where there
// are many and by loads that wait for one another (item, rows, operands) where there are few; the
// MFMAs are a few percent of either.  On one MI355X, bf16 (us, first product + second):
//   o_proj 4096 -> 4096, 4 rows, rank 16         3.6 + 4.8
//   q|k|v 4096 -> 6144, 64 rows, rank 16         5.3 + 5.2
//   gate|up 4096 -> 24576, 250 rows, 64 adapters of rank 32     11 + 30   (3.0 TB/s of 124 MB)
//   down 12288 -> 4096, 700 rows, rank 64        17.6 + 12.6  (x 17 MB and A 12.6 MB, from 100 CUs)
//   q|k|v, 8192 rows, rank 64                    31 + 72   (y's 201 MB at 2.8 TB/s, and h's planes)
#include "fqa_common.h"

namespace fqa {
namespace {

constexpr int kTileRows = FQA_LORA_TILE_ROWS;

// ---- the plan -------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;
constexpr int kPlanPer = FQA_MAX_REQS / kPlanThreads;  // requests per thread
constexpr int kPlanRows = 4096;                        // rows written per workgroup
constexpr int kDigits = 16;
static_assert(kPlanPer == 2, "two requests per thread");

struct PlanArgs {
  const int32_t* adapter;
  const int32_t* req_map;
  const int32_t* cu;
  const int32_t* meta;
  int reqs_bound, map_bound, rows_bound, n_adapters;
  int32_t* rows;
  int32_t* items;
  int item_cap;
  int32_t* lmeta;
};

// LDS accesses of a wave on either side stay in order (its own run in order on the hardware).
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// Inclusive scans over the workgroup in the order (wave, pair of elements of a lane).
template <bool kMax>
__device__ __forceinline__ int scan_op(int a, int b) {
  return kMax ? (a > b ? a : b) : a + b;
}
template <bool kMax>
__device__ __forceinline__ int wave_scan_incl(int x) {
  if constexpr (!kMax) {
    return wave_incl_scan(x);
  } else {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int y = __shfl_up(x, o, kWave);
      if (lane >= o) x = x > y ? x : y;
    }
    return x;
  }
}
// x0, x1: the thread's elements 2t and 2t + 1 (all values >= 0); replaced by their inclusive
// scan.  Returns the total.
template <bool kMax>
__device__ int block_scan2(int& x0, int& x1, int* sh) {
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x >> 6;
  const int pair = scan_op<kMax>(x0, x1);
  const int incl = wave_scan_incl<kMax>(pair);
  int excl = __shfl_up(incl, 1, kWave);
  if (lane == 0) excl = 0;
  __syncthreads();
  if (lane == kWave - 1) sh[w] = incl;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int i = 0; i < kPlanWaves; ++i) {
    if (i == w) excl = scan_op<kMax>(excl, total);
    total = scan_op<kMax>(total, sh[i]);
  }
  x0 = scan_op<kMax>(excl, x0);
  x1 = scan_op<kMax>(x0, x1);
  return total;
}

// Every workgroup sorts the (at most 2048) requests by adapter and takes the prefixes of their
// rows, the same in each; workgroup g then writes rows [g, g + 1) * kPlanRows of the order, and
// workgroup 0 the items.  The sort is a stable radix sort of (adapter, request) words in LDS,
// 4 bits a pass over the bits that n_adapters needs.
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(PlanArgs a) {
  __shared__ uint32_t word[2][FQA_MAX_REQS];  // adapter << 11 | request
  __shared__ int start[FQA_MAX_REQS];         // first row of the request
  __shared__ int len[FQA_MAX_REQS];
  __shared__ int pos[FQA_MAX_REQS];  // rows before the request in the order
  __shared__ int gend[FQA_MAX_REQS];  // by the group's first request in the order: its rows' end
  __shared__ int cnt[kDigits * kPlanWaves];
  __shared__ int sh[kPlanWaves];
  const int t = threadIdx.x, lane = t & (kWave - 1), w = t >> 6;
  const int R = min(max(a.meta[FQA_META_REQS], 0), a.reqs_bound);
  const int T = min(max(a.meta[FQA_META_ROWS], 0), a.rows_bound);
  const uint32_t none = (uint32_t)a.n_adapters;
#pragma unroll
  for (int k = 0; k < kPlanPer; ++k) {
    const int i = t + k * kPlanThreads;
    uint32_t key = none;
    int c0 = 0, n = 0;
    if (i < R) {
      const int m = a.req_map ? a.req_map[i] : i;
      if ((uint32_t)m < (uint32_t)a.map_bound) key = (uint32_t)a.adapter[m];
      if (key > none) key = none;
      c0 = min(max(a.cu[i], 0), T);
      n = min(max(a.cu[i + 1], c0), T) - c0;
    }
    word[0][i] = key << 11 | (uint32_t)i;
    start[i] = c0;
    len[i] = n;
  }
  __syncthreads();
  int src = 0;
  // wave w holds words [128 w, 128 w + 128) in two runs of 64, in order
  for (int shift = 11; (none << 11 >> shift) != 0; shift += 4) {
    uint32_t v[2];
    int before[2];
    for (int i = t; i < kDigits * kPlanWaves; i += kPlanThreads) cnt[i] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v[k] = word[src][w * 128 + k * 64 + lane];
      const uint32_t d = v[k] >> shift & 15u;
      unsigned long long same = ~0ull;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const unsigned long long m = __ballot(d >> b & 1u);
        same &= (d >> b & 1u) ? m : ~m;
      }
      const int ahead = (int)__popcll(same & ((1ull << lane) - 1ull));
      // the wave's words of this digit in its first run come before those of the second
      const int first_run = cnt[d * kPlanWaves + w];
      before[k] = first_run + ahead;
      wave_fence();
      if (ahead == 0) cnt[d * kPlanWaves + w] = first_run + (int)__popcll(same);
      wave_fence();
    }
    __syncthreads();
    if (t < kDigits * kPlanWaves) {  // 256 counts: exclusive prefix over (digit, wave)
      const int c = cnt[t];
      const int incl = wave_incl_scan(c);
      if (lane == kWave - 1) sh[w] = incl;
      cnt[t] = incl - c;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = (int)(v[k] >> shift & 15u) * kPlanWaves + w;
      int at = before[k] + cnt[c];
      for (int i = 0; i < (c >> 6); ++i) at += sh[i];
      word[src ^ 1][at] = v[k];
    }
    src ^= 1;
    __syncthreads();
  }
  // the order's requests 2t and 2t + 1: rows before them, their group's start, its items
  const uint32_t* ord = word[src];
  const int p0 = 2 * t, p1 = p0 + 1;
  const uint32_t w0 = ord[p0], w1 = ord[p1];
  const uint32_t prev = t ? ord[p0 - 1] : ~0u, next = t < kPlanThreads - 1 ? ord[p1 + 1] : ~0u;
  const int i0 = w0 & 2047, i1 = w1 & 2047;
  const int n0 = len[i0], n1 = len[i1];
  int e0 = n0, e1 = n1;
  const int total = block_scan2<false>(e0, e1, sh);  // rows up to and with the request
  const int b0 = e0 - n0, b1 = e1 - n1;
  pos[p0] = b0;
  pos[p1] = b1;
  int h0 = prev >> 11 != w0 >> 11 ? p0 : 0, h1 = w0 >> 11 != w1 >> 11 ? p1 : 0;
  block_scan2<true>(h0, h1, sh);  // the group's first request in the order
  if (w0 >> 11 != w1 >> 11) gend[h0] = e0;
  if (next >> 11 != w1 >> 11) gend[h1] = e1;
  __syncthreads();
  // items begin every kTileRows rows of a group: those that begin within each request's rows
  const int g0 = pos[h0], g1 = pos[h1];
  const auto tiles = [](int rows) { return (rows + kTileRows - 1) / kTileRows; };
  int m0 = tiles(e0 - g0) - tiles(b0 - g0), m1 = tiles(e1 - g1) - tiles(b1 - g1);
  const int k0 = m0, k1 = m1;
  // adapters' items and rows come before those of no adapter
  const int n_items = block_scan2<false>(m0, m1, sh);
  if (blockIdx.x == 0) {
    const auto put = [&](uint32_t key, int head, int group, int before, int item, int n) {
      for (int k = 0; k < n; ++k, ++item) {
        const int first = group + (tiles(before - group) + k) * kTileRows;
        if (item < a.item_cap) {
          int4 it;
          it.x = key < none ? (int)key : -1;
          it.y = first;
          it.z = min(kTileRows, gend[head] - first);
          it.w = 0;
          reinterpret_cast<int4*>(a.items)[item] = it;
        }
      }
    };
    put(w0 >> 11, h0, g0, b0, m0 - k0, k0);
    put(w1 >> 11, h1, g1, b1, m1 - k1, k1);
    for (int i = n_items + t; i < a.item_cap; i += kPlanThreads)
      reinterpret_cast<int4*>(a.items)[i] = int4{-1, 0, 0, 0};
    // where the requests without an adapter begin (requests past R are among them)
    if (w0 >> 11 == none && (t == 0 || prev >> 11 != none)) {
      a.lmeta[2] = b0;
      a.lmeta[3] = m0 - k0;
    }
    if (w1 >> 11 == none && w0 >> 11 != none) {
      a.lmeta[2] = b1;
      a.lmeta[3] = m1 - k1;
    }
    if (t == kPlanThreads - 1) {
      a.lmeta[0] = n_items;
      a.lmeta[1] = total;
      if (w1 >> 11 != none) {
        a.lmeta[2] = total;
        a.lmeta[3] = n_items;
      }
    }
  }
  // rows of the order: the last request that starts at or before each
  const int r0 = blockIdx.x * kPlanRows, r1 = min(r0 + kPlanRows, min(total, a.rows_bound));
  for (int i = r0 + t; i < r1; i += kPlanThreads) {
    int lo = 0, hi = FQA_MAX_REQS - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pos[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    a.rows[i] = start[ord[lo] & 2047] + (i - pos[lo]);
  }
}

// ---- the products ---------------------------------------------------------------------
constexpr int kLThreads = 256;  // of the second product
constexpr int kLWaves = kLThreads / kWave;
constexpr int kHThreads = 512;  // of the first
constexpr int kHWaves = kHThreads / kWave;
constexpr int kColTile = kLWaves * 64;  // output columns that its waves have at a time
constexpr int kChunk = 64;            // K granularity

struct LoraArgs {
  const uint16_t* x;
  const uint16_t* wa;  // [n][S R][K]
  const uint16_t* wb;  // [n][N][R]
  const float* scale;
  const int32_t* rank;
  const int32_t* rows;
  const int32_t* items;
  const int32_t* lmeta;
  const void* y_in;
  void* y;
  float* h;  // [splits][rows_bound][S R], in the plan's row order
  long long ldx, ldyi, ldy;
  int K, N, S, R, SR;
  int n_adapters, rows_bound, item_bound, subs;
  int splits, jgroups;
  int rounds;  // column tiles of a workgroup of the second product
  int parts;   // workgroups that share an item's rows in the second product
  int slice_end[FQA_LORA_MAX_SLICES];
  int tile_end[FQA_LORA_MAX_SLICES];  // column workgroups up to and with each slice
};

struct Item {
  int adapter, first, count;
};
// The rows that workgroup `blk` of `subs` per item has of its item; count 0 for none.
__device__ __forceinline__ Item item_of(const LoraArgs& a, int blk, int subs) {
  const int i = blk / subs, off = (blk - i * subs) * (kTileRows / subs);
  if (i >= a.item_bound) return {-1, 0, 0};
  const int4 it = reinterpret_cast<const int4*>(a.items)[i];
  const bool ok = i < a.lmeta[0] && it.x < a.n_adapters && it.z > 0 && it.z <= kTileRows &&
                  it.y >= 0 && it.y <= a.rows_bound - it.z;
  return {it.x, it.y + off, ok ? min(it.z - off, kTileRows / subs) : 0};
}

__device__ __forceinline__ int rank_of(const LoraArgs& a, int adapter) {
  return a.rank ? min(max(a.rank[adapter], 0), a.R) : a.R;
}

__device__ __forceinline__ bf16x8 load8(const uint16_t* p) {
  return *reinterpret_cast<const bf16x8*>(p);
}

// h = x A^T: the item's rows (kRB blocks of 16) by kJB blocks of 16 ranks over the split's k.
// The waves take its 64-wide chunks in turn and sum in LDS, a row block at a time (16 KiB and less
// of LDS, so that the registers bound the waves in flight: the loads are what takes the time). A
// lane's MFMA result is 4 consecutive ranks of one row.
template <int kRB, int kJB>
__device__ __forceinline__ void shrink(const LoraArgs& a, const Item& it, int jb0, int njb, int rk,
                                       int split, float4_t* red) {
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int chunks = a.K / kChunk;
  const int c0 = (int)((long long)chunks * split / a.splits);
  const int c1 = (int)((long long)chunks * (split + 1) / a.splits);
  const int kl = (lane >> 4) * 8;
  const uint16_t* xr[kRB];
#pragma unroll
  for (int r = 0; r < kRB; ++r) {
    const int i = min(r * 16 + (lane & 15), it.count - 1);
    const int row = min(max(a.rows[it.first + i], 0), a.rows_bound - 1);
    xr[r] = a.x + (long long)row * a.ldx + kl;
  }
  const uint16_t* ar = a.wa + ((long long)it.adapter * a.SR + jb0 * 16 + (lane & 15)) * a.K + kl;
  bool live[kJB];
#pragma unroll
  for (int j = 0; j < kJB; ++j) live[j] = j < njb && (jb0 + j) * 16 % a.R < rk;
  float4_t acc[kRB][kJB];
#pragma unroll
  for (int r = 0; r < kRB; ++r)
#pragma unroll
    for (int j = 0; j < kJB; ++j) acc[r][j] = float4_t{0.f, 0.f, 0.f, 0.f};
  // a chunk's fragments are on their way while those of the chunk before are multiplied
  bf16x8 xf[kRB][2], af[kJB][2], xn[kRB][2], an[kJB][2];
  const auto load = [&](bf16x8 (&x)[kRB][2], bf16x8 (&f)[kJB][2], int c) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = c * kChunk + h * 32;
#pragma unroll
      for (int j = 0; j < kJB; ++j)
        if (live[j]) f[j][h] = load8(ar + (long long)j * 16 * a.K + k);
#pragma unroll
      for (int r = 0; r < kRB; ++r) x[r][h] = load8(xr[r] + k);
    }
  };
  if (c0 + w < c1) load(xf, af, c0 + w);
  for (int c = c0 + w; c < c1; c += kHWaves) {
    if (c + kHWaves < c1) load(xn, an, c + kHWaves);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < kJB; ++j)  // blocks past the rank too: their sums are not used
#pragma unroll
        for (int r = 0; r < kRB; ++r)
          acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[j][h], xf[r][h], acc[r][j], 0, 0, 0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < kJB; ++j) af[j][h] = an[j][h];
#pragma unroll
      for (int r = 0; r < kRB; ++r) xf[r][h] = xn[r][h];
    }
  }
#pragma unroll
  for (int r = 0; r < kRB; ++r) {
    if (r) __syncthreads();
#pragma unroll
    for (int j = 0; j < kJB; ++j) red[(j * kHWaves + w) * kWave + lane] = acc[r][j];
    __syncthreads();
    if (w < njb && (jb0 + w) * 16 % a.R < rk) {
      float4_t s = red[w * kHWaves * kWave + lane];
#pragma unroll
      for (int k = 1; k < kHWaves; ++k) s += red[(w * kHWaves + k) * kWave + lane];
      const int i = r * 16 + (lane & 15);
      if (i < it.count)
        *reinterpret_cast<float4_t*>(a.h + ((long long)split * a.rows_bound + it.first + i) * a.SR +
                                     (jb0 + w) * 16 + (lane >> 4) * 4) = s;
    }
  }
}

// kRB: blocks of 16 rows multiplied at once.  Workgroups are dealt to the 8 XCDs round robin: the rank
// groups of one block of rows go to one XCD, one after another, so that they share x's rows in its
// L2.
template <int kJB, int kRB>
__global__ void __launch_bounds__(kHThreads, kRB > 2 ? 2 : 4) lora_shrink_kernel(LoraArgs a) {
  __shared__ float4_t red[kJB * kHWaves * kWave];
  const int xcd = blockIdx.x % 8, g = blockIdx.x / 8, group = g % a.jgroups;
  Item it = item_of(a, g / a.jgroups * 8 + xcd, a.subs);
  if (it.count <= 0 || it.adapter < 0) return;
  const int rk = rank_of(a, it.adapter);
  const int total = a.SR / 16, jb0 = group * kJB, njb = min(kJB, total - jb0);
  const int split = blockIdx.y;
  for (int left = it.count; left > 0; left -= kRB * 16, it.first += kRB * 16) {
    it.count = min(left, kRB * 16);
    if (kRB > 1 && it.count <= 16)
      shrink<1, kJB>(a, it, jb0, njb, rk, split, red);
    else
      shrink<kRB, kJB>(a, it, jb0, njb, rk, split, red);
    __syncthreads();
  }
}

// h = x A^T for items of many rows and more than 4 blocks of ranks (q|k|v at a high rank): a workgroup
// takes an item's 128 rows by kJB blocks of 16 ranks.  What bounds it is what the CUs read from L2:
// in lora_shrink_kernel A is read again for every 64 rows and x for every 4 blocks of ranks (400 MB for
// q|k|v at 8192 rows and rank 64, 50 us); here A goes through LDS once for 128 rows and x is read
// once: 31 us.  Wave w multiplies rows 32 (w % 4).. over half w / 4 of each step's two chunks of 64 k.
// A chunk's row of A is 8 pieces of 16 bytes, piece c of row r at c ^ (r / 2 % 8): the 16 rows of a
// fragment read then lie in 16 different bank groups.
template <int kJB>
__global__ void __launch_bounds__(kHThreads, 2) lora_shrink_tile_kernel(LoraArgs a) {
  constexpr int kRowsA = kJB * 16, kBuf = 2 * kRowsA * 8;  // 16-byte pieces of a step
  constexpr int kLoads = kBuf / kHThreads;
  static_assert(kBuf % kHThreads == 0 && kLoads * kHThreads == kBuf, "pieces");
  typedef bf16x8 Piece;
  __shared__ Piece lds[2][kBuf];
  static_assert(4 * 2 * kJB * kWave <= 2 * kBuf, "the halves' sums");
  const int xcd = blockIdx.x % 8, g = blockIdx.x / 8, group = g % a.jgroups;
  const Item it = item_of(a, g / a.jgroups * 8 + xcd, 1);
  if (it.count <= 0 || it.adapter < 0) return;
  const int rk = rank_of(a, it.adapter);
  const int jb0 = group * kJB, njb = min(kJB, a.SR / 16 - jb0);
  const int split = blockIdx.y, chunks = a.K / kChunk;
  const int c0 = (int)((long long)chunks * split / a.splits);
  const int c1 = (int)((long long)chunks * (split + 1) / a.splits);
  const int steps = (c1 - c0 + 1) / 2;
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(t >> 6), half = w >> 2, r0 = (w & 3) * 32;
  const int li = lane & 15, q = lane >> 4;
  const bool busy = r0 < it.count;
  const uint16_t* xr[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = min(r0 + r * 16 + li, it.count - 1);
    const int row = min(max(a.rows[it.first + i], 0), a.rows_bound - 1);
    xr[r] = a.x + (long long)row * a.ldx + q * 8;
  }
  uint32_t live = 0;
#pragma unroll
  for (int j = 0; j < kJB; ++j)
    if (j < njb && (jb0 + j) * 16 % a.R < rk) live |= 1u << j;
  // piece t + 512 i of a step: row / 16 consecutive pieces (two chunks) of it
  const uint16_t* ar[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
    ar[i] = a.wa + ((long long)it.adapter * a.SR + min(jb0 * 16 + i * 32 + (t >> 4), a.SR - 1)) * a.K +
            (t & 15) * 8;
  Piece stage[kLoads], xf[2][2], xn[2][2];
  // (a chunk past the split's end is loaded again and not multiplied)
  const auto load_a = [&](int s) {
    const int c = min(c0 + 2 * s + ((t >> 3) & 1), c1 - 1) - ((t >> 3) & 1);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)  // 32 rows of A each: 2 blocks of ranks
      if (live >> (2 * i) & 3u) stage[i] = load8(ar[i] + (long long)c * kChunk);
  };
  const auto store_a = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = i * 32 + (t >> 4), c = t & 7, h = (t >> 3) & 1;
      lds[buf][(h * kRowsA + row) * 8 + (c ^ ((row >> 1) & 7))] = stage[i];
    }
  };
  const auto load_x = [&](Piece (&x)[2][2], int s) {
    const int c = min(c0 + 2 * s + half, c1 - 1);
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) x[r][h] = load8(xr[r] + (long long)c * kChunk + h * 32);
  };
  float4_t acc[2][kJB];
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int j = 0; j < kJB; ++j) acc[r][j] = float4_t{0.f, 0.f, 0.f, 0.f};
  // what step s + 2 needs is asked for at the end of step s
  const auto step = [&](int s, Piece (&x)[2][2]) {
    if (busy && c0 + 2 * s + half < c1) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < kJB; ++j) {  // blocks past the rank too: their sums are not used
          const int row = j * 16 + li;
          const Piece af = lds[s & 1][(half * kRowsA + row) * 8 + ((h * 4 + q) ^ ((row >> 1) & 7))];
#pragma unroll
          for (int r = 0; r < 2; ++r)
            acc[r][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, x[r][h], acc[r][j], 0, 0, 0);
        }
    }
    if (s + 1 < steps) store_a((s + 1) & 1);
    if (s + 2 < steps) {
      load_a(s + 2);
      load_x(x, s + 2);
    }
    __syncthreads();
  };
  load_a(0);
  load_x(xf, 0);
  store_a(0);
  if (steps > 1) {
    load_a(1);
    load_x(xn, 1);
  }
  __syncthreads();
#pragma nounroll
  for (int s = 0; s < steps; s += 2) {
    step(s, xf);
    if (s + 1 < steps) step(s + 1, xn);
  }
  // the halves' sums
  float4_t* red = reinterpret_cast<float4_t*>(&lds[0][0]);
  if (half)
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int j = 0; j < kJB; ++j) red[(((w & 3) * 2 + r) * kJB + j) * kWave + lane] = acc[r][j];
  __syncthreads();
  if (half || !busy) return;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = r0 + r * 16 + li;
    float* h = a.h + ((long long)split * a.rows_bound + it.first + i) * a.SR + jb0 * 16 + q * 4;
#pragma unroll
    for (int j = 0; j < kJB; ++j)
      if ((live >> j & 1u) && i < it.count)
        *reinterpret_cast<float4_t*>(h + j * 16) = acc[r][j] + red[((w * 2 + r) * kJB + j) * kWave + lane];
  }
}

template <bool kF32>
struct Out;
template <>
struct Out<false> {
  typedef uint16_t T;
};
template <>
struct Out<true> {
  typedef float T;
};

// The parts of v as bf16: the sum of two is v to 2^-16 of its value, of three all of it.  Every part has
// v's sign and is zero only if v is (above 2^-100), so that a product with an infinity is that
// infinity from each: bits are cut off, not rounded, before the last part, and a value that leaves
// nothing for the next part shares itself with it.  An infinity or a NaN is each of its parts.
template <int kParts>
__device__ __forceinline__ void split_bf16(float v, uint16_t (&part)[kParts]) {
#pragma unroll
  for (int p = 0; p < kParts - 1; ++p) {
    const uint32_t all = __float_as_uint(v), cut = all & 0xffff0000u;
    const float g = __uint_as_float(cut) * (all == cut ? 0.5f : 1.f);
    part[p] = (uint16_t)(__float_as_uint(g) >> 16);
    v = (all & 0x7f800000u) == 0x7f800000u ? v : v - bf16_bits_to_f32(part[p]);
  }
  part[kParts - 1] = f32_to_bf16_bits(v);
}

// y = y_in + scale h B^T.  A wave has 64 columns at a time of an item's rows, 16 rows to an MFMA.  One
// MFMA multiplies 16 ranks: its k 0..15 are h's first bf16 parts, 16..31 its second ones, against
// B's 16 values twice, so that h keeps 16 bits (one bf16 would round it to 8); for an fp32 y another
// one adds the halves of the third parts, twice.  Four MFMAs give a lane 16 consecutive columns of one row:
// row i of B that MFMA m takes is column 16 (i / 4) + 4 m + i % 4 of the 64.
template <bool kF32>
struct Expand {
  typedef typename Out<kF32>::T Y;
  static constexpr int kParts = kF32 ? 3 : 2;
  const LoraArgs& a;
  int first, count, adapter;  // rows of the plan, of one adapter
  int slice, col0, n_end;     // first column, end of the slice
  int t, lane, w, q, li, pitch;
  char* lds;  // h's parts, [row][part][rank], and 16 bytes a row against bank conflicts

  __device__ __forceinline__ Expand(const LoraArgs& args, const Item& it, char* shared)
      : a(args), first(it.first), count(it.count), adapter(it.adapter), lds(shared) {
    t = threadIdx.x;
    lane = t & (kWave - 1);
    w = __builtin_amdgcn_readfirstlane(t >> 6);
    q = lane >> 4;
    li = lane & 15;
    pitch = 2 * kParts * a.R + 16;
    slice = 0;
    while (slice < a.S - 1 && (int)blockIdx.x >= a.tile_end[slice]) ++slice;
    const int blk = blockIdx.x - (slice ? a.tile_end[slice - 1] : 0);
    n_end = a.slice_end[slice];
    col0 = (slice ? a.slice_end[slice - 1] : 0) + blk * a.rounds * kColTile;
  }
  __device__ __forceinline__ int row_of(int i) const {
    const int row = i < count ? a.rows[first + i] : -1;
    return row < a.rows_bound ? row : -1;
  }
  // y = y_in, for rows without an adapter
  __device__ __forceinline__ void copy() const {
    const Y* yin = (const Y*)a.y_in;
    Y* y = (Y*)a.y;
    if (yin == y) return;
    constexpr int kPer = 16 / (int)sizeof(Y), kLanes = kColTile / kPer;  // lanes of a row
    for (int c = col0 + t % kLanes * kPer; c < min(n_end, col0 + a.rounds * kColTile); c += kColTile)
#pragma unroll 4
      for (int r = t / kLanes; r < count; r += kLThreads / kLanes) {
        const int row = row_of(r);
        if (row < 0) continue;
        uint4 v;
        __builtin_memcpy(&v, yin + (long long)row * a.ldyi + c, 16);
        __builtin_memcpy(y + (long long)row * a.ldy + c, &v, 16);
      }
  }
  // B's fragment of MFMA m at column c and rank block jb
  __device__ __forceinline__ bf16x8 load_b(int c, int m, int jb) const {
    return load8(a.wb + ((long long)adapter * a.N + c + 16 * (li >> 2) + 4 * m + (li & 3)) * a.R +
                 jb * 16 + (q & 1) * 8);
  }
  // ... with zeros for what it holds past the rank, which is no value
  __device__ __forceinline__ void end_b(bf16x8& f, int jb, int rk) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < rk - jb * 16 - (q & 1) * 8 ? f[e] : (__bf16)0.f;
  }
  // h of rows [row0, row0 + rows) into LDS: summed over the splits, scaled, in parts
  __device__ __forceinline__ void stage(int row0, int rows, int rk, float scale) const {
    const float* h = a.h + (long long)(first + row0) * a.SR + slice * a.R;
    const long long plane = (long long)a.rows_bound * a.SR;
    const int quads = a.R / 4;
    for (int i = t; i < (rows + 15) / 16 * 16 * quads; i += kLThreads) {
      const int r = i / quads, j = (i - r * quads) * 4;
      const float* p = h + (long long)min(r, rows - 1) * a.SR + j;
      float4_t v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int k = 0; k < a.splits; ++k) v += *reinterpret_cast<const float4_t*>(p + k * plane);
      short4_t part[kParts];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint16_t x[kParts];
        split_bf16(j + e < rk ? v[e] * scale : 0.f, x);
        if constexpr (kF32) x[2] = f32_to_bf16_bits(0.5f * bf16_bits_to_f32(x[2]));
#pragma unroll
        for (int k = 0; k < kParts; ++k) part[k][e] = (short)x[k];
      }
#pragma unroll
      for (int k = 0; k < kParts; ++k)
        *reinterpret_cast<short4_t*>(lds + r * pitch + (k * a.R + j) * 2) = part[k];
    }
  }
  // acc += 16 rows (block rb of those staged) by 64 columns over rank block jb
  __device__ __forceinline__ void multiply(const bf16x8 (&f)[4], int rb, int jb, float4_t (&acc)[4]) const {
    const char* p = lds + (rb * 16 + li) * pitch + (q & 1) * 16 + jb * 32;
    if constexpr (kF32) {
      const bf16x8 z = *reinterpret_cast<const bf16x8*>(p + 4 * a.R);
#pragma unroll
      for (int m = 0; m < 4; ++m)
        acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[m], z, acc[m], 0, 0, 0);
    }
    const bf16x8 hf = *reinterpret_cast<const bf16x8*>(p + (q >> 1) * a.R * 2);
#pragma unroll
    for (int m = 0; m < 4; ++m)
      acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[m], hf, acc[m], 0, 0, 0);
  }
  __device__ __forceinline__ void load_y(Y (&v)[16], int row, int c) const {
    if (row >= 0)
      __builtin_memcpy(v, (const Y*)a.y_in + (long long)row * a.ldyi + c + q * 16, sizeof(v));
  }
  __device__ __forceinline__ void add(const Y (&v)[16], const float4_t (&acc)[4], int row, int c) const {
    if (row < 0) return;
    Y out[16];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kF32)
          out[4 * m + e] = v[4 * m + e] + acc[m][e];
        else
          out[4 * m + e] = f32_to_bf16_bits(bf16_bits_to_f32(v[4 * m + e]) + acc[m][e]);
      }
    __builtin_memcpy((Y*)a.y + (long long)row * a.ldy + c + q * 16, out, sizeof(out));
  }
};

// kColTile columns to a workgroup.  What bounds it: y's bytes and those of h, whose planes every
// workgroup of columns reads and sums again (4 planes of 128 rows at rank 64: 131 KB, as much as its
// tile of a bf16 y read and written), and at few rows the loads that wait for one another (item, rank, B
// and h and y).  B's fragments are loaded first and stay in registers for
// all of the item's rows (kJb: blocks of 16 ranks held), h goes through LDS once, and y_in of the next
// 16 rows is on its way while those before are multiplied.  q|k|v at 8192 rows and rank 64: 72 us,
// 201 MB of y at 2.8 TB/s.
template <bool kF32, int kJb, int kRows>
__global__ void __launch_bounds__(kLThreads, kJb > 4 ? 2 : kF32 && kJb > 2 ? 3 : 4)
lora_expand_kernel(LoraArgs a) {
  constexpr int kBlocks = kRows / 16;
  extern __shared__ __align__(16) char lds[];
  const Item it = item_of(a, blockIdx.y, a.parts);
  if (it.count <= 0) return;
  const Expand<kF32> x(a, it, lds);
  if (it.adapter < 0) {
    x.copy();
    return;
  }
  const int c0 = x.col0 + x.w * 64;
  const bool live = c0 < x.n_end;
  const int rk = rank_of(a, it.adapter), njb = (rk + 15) / 16;
  bf16x8 bf[kJb][4];
#pragma unroll
  for (int jb = 0; jb < kJb; ++jb)
    if (jb < njb)
#pragma unroll
      for (int m = 0; m < 4; ++m) bf[jb][m] = x.load_b(live ? c0 : x.col0, m, jb);
  const float scale = a.scale[it.adapter];
  for (int row0 = 0; row0 < it.count; row0 += kRows) {
    const int rows = min(it.count - row0, kRows), nrb = (rows + 15) / 16;
    int row[kBlocks];
#pragma unroll
    for (int rb = 0; rb < kBlocks; ++rb) row[rb] = live ? x.row_of(row0 + rb * 16 + x.li) : -1;
    if (row0) __syncthreads();
    x.stage(row0, rows, rk, scale);
    typename Out<kF32>::T in[kBlocks > 1 ? 2 : 1][16];
    x.load_y(in[0], row[0], c0);
    if (row0 == 0 && (rk & 15))
#pragma unroll
      for (int jb = 0; jb < kJb; ++jb)
        if (jb == njb - 1)
#pragma unroll
          for (int m = 0; m < 4; ++m) x.end_b(bf[jb][m], jb, rk);
    __syncthreads();
    if (!live) continue;
#pragma unroll
    for (int rb = 0; rb < kBlocks; ++rb) {
      if (rb >= nrb) break;
      if constexpr (kBlocks > 1)
        if (rb + 1 < kBlocks) x.load_y(in[(rb + 1) & 1], row[rb + 1], c0);
      float4_t acc[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) acc[m] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int jb = 0; jb < kJb; ++jb)
        if (jb < njb) x.multiply(bf[jb], rb, jb, acc);
      x.add(in[kBlocks > 1 ? rb & 1 : 0], acc, row[rb], c0);
    }
  }
}

// Items of few rows and many columns, as in a decode step: B is most of the bytes, so a workgroup goes
// on over a.rounds column tiles with the next step's B (kG rank blocks of 64 columns) and the next
// tile's y_in on their way under this one's work; 16 rows at a time.  gate|up at 250 rows and 64
// adapters of rank 32: 30 us, 124 MB.
template <bool kF32, int kG>
__global__ void __launch_bounds__(kLThreads, 3) lora_expand_few_kernel(LoraArgs a) {
  extern __shared__ __align__(16) char lds[];
  const Item it = item_of(a, blockIdx.y, 1);
  if (it.count <= 0) return;
  const Expand<kF32> x(a, it, lds);
  if (it.adapter < 0) {
    x.copy();
    return;
  }
  const int c_first = x.col0 + x.w * 64;
  const int tiles = min(a.rounds, max(0, (x.n_end - c_first + kColTile - 1) / kColTile));  // the wave's
  const int rk = rank_of(a, it.adapter), njb = (rk + 15) / 16, groups = max(1, (njb + kG - 1) / kG);
  const int steps = tiles * groups;
  const float scale = a.scale[it.adapter];
  bf16x8 bf[kG][4], bn[kG][4];
  const auto load = [&](bf16x8 (&f)[kG][4], int tile, int g) {
#pragma unroll
    for (int k = 0; k < kG; ++k)
      if (g * kG + k < njb)
#pragma unroll
        for (int m = 0; m < 4; ++m) f[k][m] = x.load_b(c_first + tile * kColTile, m, g * kG + k);
  };
  for (int row0 = 0; row0 < it.count; row0 += 16) {
    const int row = x.row_of(row0 + x.li);
    if (steps > 0) load(bf, 0, 0);
    typename Out<kF32>::T in[16], next[16];
    if (tiles > 0) x.load_y(in, row, c_first);
    if (row0) __syncthreads();
    x.stage(row0, min(it.count - row0, 16), rk, scale);
    __syncthreads();
    float4_t acc[4];
    int tile = 0, g = 0;
#pragma nounroll
    for (int step = 0; step < steps; ++step) {
      const bool last = g + 1 == groups;
      const int tile_n = last ? tile + 1 : tile, g_n = last ? 0 : g + 1;
      if (step + 1 < steps) load(bn, tile_n, g_n);
      if (g == 0) {
        if (tile + 1 < tiles) x.load_y(next, row, c_first + (tile + 1) * kColTile);
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[m] = float4_t{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int k = 0; k < kG; ++k) {
        const int jb = g * kG + k;
        if (jb >= njb) continue;
        if ((rk & 15) && jb == njb - 1)
#pragma unroll
          for (int m = 0; m < 4; ++m) x.end_b(bf[k][m], jb, rk);
        x.multiply(bf[k], 0, jb, acc);
      }
      if (last) {
        x.add(in, acc, row, c_first + tile * kColTile);
#pragma unroll
        for (int e = 0; e < 16; ++e) in[e] = next[e];
      }
#pragma unroll
      for (int k = 0; k < kG; ++k)
#pragma unroll
        for (int m = 0; m < 4; ++m) bf[k][m] = bn[k][m];
      tile = tile_n;
      g = g_n;
    }
  }
}

// How the first product's work is cut.  few: items of a few rows, as in a decode step, whose A is
// most of what is read: 16 rows at once, so that more waves are in flight (and each item's rows one
// after another); otherwise 64, or (tile) 128 through LDS where there are more than 4 blocks of ranks.
// K in splits towards two workgroups for every CU (tile: one), 8 at most, since every workgroup of
// the second product reads them all, and a chunk for every wave at least.  Both products of down at
// 700 rows and rank 64 take 30 us with 8 splits, 37 with 12 and 34 with 16; of q|k|v at 8192 rows and
// rank 64 99 by tiles in 4 splits, 114 in 2, 117 in 8 and 117 without tiles.
// All of it goes by the call's bounds, since the host does not know the items: a decode step planned by
// bounds of 8192 rows and 256 requests takes the forms for many rows (o_proj at 4 rows 9.7 us where its
// own bounds take 7.8, gate|up at 250 rows 47.7 and 34.5, q|k|v at 64 rows of rank 64 31.4 and 18.5).
constexpr int kShrinkWgs = 512, kTileWgs = 300, kMaxSplits = 8;
struct Cut {
  bool few, tile;
  int subs, splits, jgroups, jb;  // jb: blocks of ranks to a workgroup
};
Cut lora_cut(const fqa_lora* w, int item_bound, int rows_bound) {
  Cut c;
  const int blocks = w->n_slices * w->rank_max / 16;
  c.few = rows_bound <= 32ll * item_bound;
  c.tile = !c.few && blocks > 4;
  c.jgroups = (blocks + (c.tile ? 11 : 3)) / (c.tile ? 12 : 4);
  c.jb = (blocks + c.jgroups - 1) / c.jgroups;
  if (c.tile) c.jb = c.jb <= 8 ? 8 : 12;
  c.subs = c.few || c.tile ? 1 : 2;
  const long long wgs = (long long)item_bound * c.jgroups * c.subs;
  const int most = w->n_in / (kChunk * (c.tile ? 2 : kHWaves));
  long long s = wgs > 0 ? (c.tile ? kTileWgs : kShrinkWgs) / wgs : 1;
  if (s > kMaxSplits) s = kMaxSplits;
  if (s > most) s = most;
  c.splits = s < 1 ? 1 : (int)s;
  return c;
}

int check_weights(const fqa_lora* w) {
  if (!w || w->n_adapters < 1 || w->n_adapters > FQA_LORA_MAX_ADAPTERS || w->n_slices < 1 ||
      w->n_slices > FQA_LORA_MAX_SLICES)
    return FQA_EINVAL;
  if (w->rank_max < 16 || w->rank_max > FQA_LORA_MAX_RANK || w->rank_max % 16 || w->n_in < 64 ||
      w->n_in % 64)
    return FQA_EUNSUPPORTED;
  for (int s = 0, prev = 0; s < w->n_slices; prev = w->slice_end[s++])
    if (w->slice_end[s] <= prev || (w->slice_end[s] - prev) % 64 || w->slice_end[s] > FQA_LORA_MAX_COLS)
      return FQA_EUNSUPPORTED;
  return FQA_OK;
}

}  // namespace
}  // namespace fqa

using namespace fqa;

extern "C" {

int32_t fqa_lora_item_bound(int32_t n_reqs, int32_t rows, int32_t n_adapters) {
  if (n_reqs < 0 || rows < 0 || n_adapters < 1) return FQA_EINVAL;
  return rows / kTileRows + (n_reqs < n_adapters + 1 ? n_reqs : n_adapters + 1);
}

int fqa_lora_plan(const int32_t* adapter, int32_t n_ids, const int32_t* req_map,
                  const int32_t* cu_seqlens, const int32_t* meta, int32_t n_reqs_bound,
                  int32_t rows_bound, int32_t n_adapters, int32_t* rows, int32_t* items,
                  int32_t item_cap, int32_t* lora_meta, void* stream) {
  if (n_reqs_bound < 0 || n_reqs_bound > FQA_MAX_REQS || rows_bound < 0 || rows_bound > (1 << 20) ||
      n_ids < 0 || n_adapters < 1 || n_adapters > FQA_LORA_MAX_ADAPTERS ||
      item_cap < fqa_lora_item_bound(n_reqs_bound, rows_bound, n_adapters))
    return FQA_EINVAL;
  if (!meta || !lora_meta || !cu_seqlens || (n_ids && !adapter) || (rows_bound && !rows) ||
      (item_cap && !items) || ((uintptr_t)items & 15))
    return FQA_EINVAL;
  PlanArgs a{adapter, req_map, cu_seqlens, meta, n_reqs_bound, n_ids, rows_bound, n_adapters,
             rows, items, item_cap, lora_meta};
  const int grid = rows_bound > kPlanRows ? (rows_bound + kPlanRows - 1) / kPlanRows : 1;
  hipLaunchKernelGGL(lora_plan_kernel, dim3(grid), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? FQA_OK : FQA_ELAUNCH;
}

int64_t fqa_lora_workspace_bytes(const fqa_lora* w, int32_t rows_bound, int32_t item_bound) {
  const int rc = check_weights(w);
  if (rc != FQA_OK) return rc;
  if (rows_bound < 0 || item_bound < 0) return FQA_EINVAL;
  return (int64_t)lora_cut(w, item_bound, rows_bound).splits * rows_bound * w->n_slices * w->rank_max * 4;
}

int64_t fqa_lora_workspace_most(const fqa_lora* w, int32_t max_rows) {
  const int rc = check_weights(w);
  if (rc != FQA_OK) return rc;
  if (max_rows < 0) return FQA_EINVAL;
  // splits <= kMaxSplits and, where it is above 1, items * splits <= kShrinkWgs; an item bound is
  // rows / kTileRows (rounded down) + 1 at least where there are rows, so splits * rows is below
  // kShrinkWgs * kTileRows or (unsplit) at most max_rows
  const int64_t split = (int64_t)kShrinkWgs * kTileRows, rows = max_rows;
  const int64_t cap = rows * kMaxSplits;
  return (cap < split ? cap : rows > split ? rows : split) * w->n_slices * w->rank_max * 4;
}

int fqa_lora_add(const fqa_lora* w, const void* x, int64_t ldx, const int32_t* rows,
                 const int32_t* items, const int32_t* lora_meta, int32_t rows_bound,
                 int32_t item_bound, const void* y_in, int64_t ldyi, void* y, int64_t ldy,
                 int32_t y_f32, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_weights(w);
  if (rc != FQA_OK) return rc;
  if (rows_bound < 0 || rows_bound > (1 << 20) || item_bound < 0 ||
      item_bound > FQA_LORA_MAX_ITEMS)
    return FQA_EINVAL;
  if (rows_bound == 0 || item_bound == 0) return FQA_OK;
  const int K = w->n_in, S = w->n_slices, R = w->rank_max, N = w->slice_end[S - 1];
  if (!x || !w->a || !w->b || !w->scale || !rows || !items || !lora_meta || !y_in || !y ||
      !workspace || workspace_bytes < fqa_lora_workspace_bytes(w, rows_bound, item_bound))
    return FQA_EINVAL;
  if (ldx < K || ldyi < N || ldy < N || ldx % 8 || ldyi % 4 || ldy % 4) return FQA_EINVAL;
  for (const void* p : {x, (const void*)w->a, (const void*)w->b, (const void*)items, y_in,
                        (const void*)y, (const void*)workspace})
    if ((uintptr_t)p & 15) return FQA_EINVAL;
  if (y_in == y && ldyi != ldy) return FQA_EINVAL;
  LoraArgs a{};
  a.x = (const uint16_t*)x;
  a.wa = w->a;
  a.wb = w->b;
  a.scale = w->scale;
  a.rank = w->rank;
  a.rows = rows;
  a.items = items;
  a.lmeta = lora_meta;
  a.y_in = y_in;
  a.y = y;
  a.h = (float*)workspace;
  a.ldx = ldx;
  a.ldyi = ldyi;
  a.ldy = ldy;
  a.K = K;
  a.N = N;
  a.S = S;
  a.R = R;
  a.SR = S * R;
  a.n_adapters = w->n_adapters;
  a.rows_bound = rows_bound;
  a.item_bound = item_bound;
  const Cut cut = lora_cut(w, item_bound, rows_bound);
  a.subs = cut.subs;
  a.jgroups = cut.jgroups;
  a.splits = cut.splits;
  // Where there are more column tiles than the CUs hold workgroups (3 each), several to one:
  // gate_up's 6336 (250 rows, 64 adapters of rank 32) take 43 us at one to a workgroup and 29 at 8; 33
  // and 39 at 12 and 16.
  const long long all = (long long)((N + kColTile - 1) / kColTile) * item_bound;
  const long long rounds = (all + 384) / 768;
  a.rounds = !cut.few || rounds < 2 ? 1 : rounds < 16 ? (int)rounds : 16;
  int tiles = 0;
  for (int s = 0; s < S; ++s) {
    const int width = w->slice_end[s] - (s ? w->slice_end[s - 1] : 0);
    tiles += (width + a.rounds * kColTile - 1) / (a.rounds * kColTile);
    a.slice_end[s] = w->slice_end[s];
    a.tile_end[s] = tiles;
  }
  const hipStream_t st = (hipStream_t)stream;
  const int blocks = item_bound * a.subs;
  const dim3 g1((blocks + 7) / 8 * 8 * a.jgroups, a.splits), b1(kHThreads), b(kLThreads);
#define FQA_SHRINK(JB)                                                 \
  if (cut.few)                                                         \
    hipLaunchKernelGGL((lora_shrink_kernel<JB, 1>), g1, b1, 0, st, a); \
  else                                                                 \
    hipLaunchKernelGGL((lora_shrink_kernel<JB, 4>), g1, b1, 0, st, a);
  if (cut.tile) {
    if (cut.jb == 8)
      hipLaunchKernelGGL(lora_shrink_tile_kernel<8>, g1, b1, 0, st, a);
    else
      hipLaunchKernelGGL(lora_shrink_tile_kernel<12>, g1, b1, 0, st, a);
  } else {
    switch (cut.jb) {
      case 1: FQA_SHRINK(1) break;
      case 2: FQA_SHRINK(2) break;
      case 3: FQA_SHRINK(3) break;
      default: FQA_SHRINK(4) break;
    }
  }
#undef FQA_SHRINK
  if (hipGetLastError() != hipSuccess) return FQA_ELAUNCH;
  const int row_bytes = (y_f32 ? 6 : 4) * R + 16;
  if (a.rounds > 1) {
    const dim3 g2(tiles, item_bound);
#define FQA_EXPAND(F32, G) \
  hipLaunchKernelGGL((lora_expand_few_kernel<F32, G>), g2, b, 16 * row_bytes, st, a)
    if (R > 16) {
      if (y_f32) FQA_EXPAND(true, 2); else FQA_EXPAND(false, 2);
    } else {
      if (y_f32) FQA_EXPAND(true, 1); else FQA_EXPAND(false, 1);
    }
#undef FQA_EXPAND
  } else {
    // an item of many rows is shared by workgroups until these fill the CUs
    a.parts = cut.few || all >= 1024 ? 1 : all >= 512 ? 2 : 4;
    const dim3 g2(tiles, item_bound * a.parts);
#define FQA_EXPAND(F32, JB, ROWS) \
  hipLaunchKernelGGL((lora_expand_kernel<F32, JB, ROWS>), g2, b, ROWS * row_bytes, st, a)
#define FQA_EXPAND_JB(JB, MANY)                                   \
  if (cut.few) {                                                  \
    if (y_f32) FQA_EXPAND(true, JB, 16); else FQA_EXPAND(false, JB, 16);     \
  } else {                                                        \
    if (y_f32) FQA_EXPAND(true, JB, MANY); else FQA_EXPAND(false, JB, MANY); \
  }
    if (R <= 16) {
      FQA_EXPAND_JB(1, 128)
    } else if (R <= 32) {
      FQA_EXPAND_JB(2, 128)
    } else if (R <= 64) {
      FQA_EXPAND_JB(4, 128)
    } else {
      FQA_EXPAND_JB(8, 64)
    }
#undef FQA_EXPAND_JB
#undef FQA_EXPAND
  }
  return hipGetLastError() == hipSuccess ? FQA_OK : FQA_ELAUNCH;
}

}  // extern "C"
