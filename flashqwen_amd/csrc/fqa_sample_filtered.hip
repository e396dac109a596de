// fqa_sample_filtered.hip — token sampling with temperature, top-k, top-p and min-p (gfx950).
//
// Row b: w_i = exp((l_i - M) inv_temp).  Every filter keeps a prefix of the order (logit
// descending, index ascending), so what is kept is the prefix that ends at one element, the cut
// (logit, index).  The token is the first index at which the running kept mass reaches u times
// the kept mass.
//
// filter_scan_kernel reads the logits once: a row is dealt to parts of 512 x 20 logits, which its
// threads hold in registers, and each part leaves
//  * its largest logit (all a greedy row needs),
//  * for top_k <= 64 a superset of its top_k largest logits, chosen by the top_k-th largest of the
//    512 threads' maxima,
//  * else the masses (and, for a top-k, counts) of its weights by bins of an eighth of an octave, at
//    places that all parts of the row share (bin = round(8 log2(e) inv_temp l)), so that no part has
//    to know the row's largest logit.  Within a bin a weight is 2^(r/8), |r| <= 1/2: a polynomial,
//    in units of 2^-39, and its sum an integer, exact in any order of the LDS atomics.
// filter_merge_kernel (a workgroup per row) adds the parts' bins up, which gives the bin that the
// cut of each filter lies in.  filter_gather_kernel (a workgroup per part) reads the row again and
// collects the logits of those bins; with few rows it does the merge too.  filter_pick_kernel (a
// workgroup per row) has the top_k largest from the parts' lists by sorting networks across lanes;
// or a radix select over the collected logits ends at the cut, the parts' bins above it and the kept
// of its own bin give each part's kept mass, and the part that holds the draw is walked in fp64.
// Rows that the bins do not serve (u = 0, which may pick a weight below all bins, infinite logits or
// inv_temp, |8 log2(e) inv_temp M| > 2^29, more than 8192 logits in the cuts' bins) and vocabularies
// of more than 1024 parts are done by select_row, from the logits alone.
//
// What bounds it, 151936 logits a row (us): 256 rows of wide nuclei take 94 where reading them once
// takes 25 (at 6.2 TB/s) - the scan 31 and the gather 28, each a read at 5 TB/s; the merge 7 and the
// pick 27, which are chains of dependent steps on one CU per row (the walk 3.5, the radix select 3.5,
// both on fp64 weights; a dozen more of 0.5 to 2).  256 rows greedy 35, of top_k 20 46, without a
// filter 54, of every kind 75 (gather 15, pick 22).  64 rows 43 (scan 12, merge 7, gather 7, pick 20).
// One row: greedy 7, top_k 20 17, top-p 29, launches of 1.5 us and the pick's chain.  Rows that
// select_row does take 410 to 650.
#include "fqa_common.h"
#include "fqa_sample_bins.h"

#include <cfloat>

namespace fqa {
namespace {

constexpr int kFThreads = 1024;
constexpr int kFWaves = kFThreads / kWave;
constexpr int kFBins = 2048;

struct FilterArgs {
  const float* logits;
  int vocab;
  long long stride;
  const float* inv_temp;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int32_t* out;
  int rows, parts;  // parts of a row (0: no scan)
  int4* head;           // [rows][parts] {largest key, its lowest index, list length, highest bin}
  unsigned long long* body;  // [rows][parts][kBody]
  struct RowBins* bins;      // [rows]
};

typedef unsigned long long u64;

// A logit as an unsigned integer of the same order: equal logits (0 and -0 too) have one key, NaN
// has that of -inf.
constexpr uint32_t kKeyMasked = 0x007fffffu;  // -inf
constexpr uint32_t kKeyInf = 0xff800000u;     // +inf
__device__ __forceinline__ uint32_t key_of(float l) {
  uint32_t b = __float_as_uint(l);
  if ((b & 0x7fffffffu) > 0x7f800000u) b = 0xff800000u;
  if (b == 0x80000000u) b = 0u;
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key);
}

// A row's settings.
struct Settings {
  bool greedy;
  double it;
  int k;         // 0: no top-k
  double p;      // of masses; >= 1: no top-p
  double min_w;  // smallest weight kept (0: none)
  double u;
  bool extreme;  // inv_temp is infinite
};
__device__ __forceinline__ Settings settings_of(const FilterArgs& a, int row) {
  Settings s;
  const uint32_t it = __float_as_uint(a.inv_temp[row]), p = __float_as_uint(a.top_p[row]);
  const uint32_t q = __float_as_uint(a.min_p[row]), u = __float_as_uint(a.u[row]);
  s.greedy = it == 0 || it > 0x7f800000u;  // not positive, or NaN
  s.it = (double)a.inv_temp[row];
  s.k = a.top_k[row] > 0 && a.top_k[row] < a.vocab ? a.top_k[row] : 0;
  const bool p_nan = (p & 0x7fffffffu) > 0x7f800000u;
  s.p = p_nan ? 1.0 : p >> 31 ? 0.0 : (double)a.top_p[row];
  s.min_w = q == 0 || q > 0x7f800000u ? 0.0 : q > 0x3f800000u ? 1.0 : (double)a.min_p[row];
  s.u = u > 0x7f800000u ? 0.0 : (double)a.u[row];
  s.extreme = it == 0x7f800000u;
  return s;
}

// 64-bit scans and sums over the wave on DPP, as wave_incl_scan's (__shfl goes through LDS, ~100
// cycles a step and 32 bits).
template <int kCtrl, int kRows>
__device__ __forceinline__ u64 dpp64(u64 x) {
  constexpr bool kZero = kRows == 0xf;
  const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, kCtrl, kRows, 0xf, kZero);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), kCtrl, kRows, 0xf, kZero);
  return (u64)(uint32_t)hi << 32 | (uint32_t)lo;
}
template <class T>  // u64 or double
__device__ __forceinline__ T wave_scan64(T x) {
  const auto add = [&](u64 y) { x += __builtin_bit_cast(T, y); };
  add(dpp64<kDppRowShr1, 0xf>(__builtin_bit_cast(u64, x)));
  add(dpp64<kDppRowShr2, 0xf>(__builtin_bit_cast(u64, x)));
  add(dpp64<kDppRowShr4, 0xf>(__builtin_bit_cast(u64, x)));
  add(dpp64<kDppRowShr8, 0xf>(__builtin_bit_cast(u64, x)));
  add(dpp64<kDppRowBcast15, 0xa>(__builtin_bit_cast(u64, x)));
  add(dpp64<kDppRowBcast31, 0xc>(__builtin_bit_cast(u64, x)));
  return x;
}
template <class T>
__device__ __forceinline__ T wave_last64(T x) {  // lane 63's
  const u64 b = __builtin_bit_cast(u64, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, kWave - 1);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), kWave - 1);
  return __builtin_bit_cast(T, (u64)hi << 32 | lo);
}
template <class T>
__device__ __forceinline__ T wave_sum64(T x) {
  return wave_last64(wave_scan64(x));
}
// The largest key of the wave.
__device__ __forceinline__ uint32_t wave_max_key(uint32_t k) {
  return (uint32_t)wave_extreme<true>((int)(k ^ 0x80000000u), (int)0x80000000) ^ 0x80000000u;
}

// What a workgroup of kFThreads shares in sums and scans.
struct BlockLds {
  u64 wsum[kFWaves];
  double wmass[kFWaves];
  u64 above;
  int bin;
  int pick;
};

// The highest of kFBins bins at which the sum of the bins down to it, plus `above`, reaches `need`
// (there is one): the bin, and in `above` the sum of those over it.
__device__ int crossing(const u64* hist, BlockLds& sh, u64 need, u64& above) {
  const int t = threadIdx.x, lane = t & (kWave - 1), w = t >> 6;
  const int b0 = kFBins - 1 - 2 * t;
  const u64 m0 = hist[b0], m1 = hist[b0 - 1];
  const u64 incl = wave_scan64(m0 + m1);
  if (lane == kWave - 1) sh.wsum[w] = incl;
  if (t == 0) sh.bin = 0;
  __syncthreads();
  u64 before = above + incl - m0 - m1;
  for (int i = 0; i < w; ++i) before += sh.wsum[i];
  if (before < need && before + m0 + m1 >= need) {
    const bool first = before + m0 >= need;
    sh.bin = first ? b0 : b0 - 1;
    sh.above = first ? before : before + m0;
  }
  __syncthreads();
  above = sh.above;
  const int bin = sh.bin;
  __syncthreads();
  return bin;
}
// Sum over the workgroup.
__device__ u64 block_sum(u64 n, BlockLds& sh) {
  n = wave_sum64(n);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) sh.wsum[threadIdx.x >> 6] = n;
  __syncthreads();
  u64 z = 0;
  for (int i = 0; i < kFWaves; ++i) z += sh.wsum[i];
  __syncthreads();
  return z;
}

// A mass in two words, in units of 2^-38 and 2^-76 of the largest weight: a double's weight down to
// 2^-76, and the sums of up to 2^24 weights fit each word by itself, so that they are exact in any
// order.  (One word would leave a vocabulary of 2^24 no more than 2^-39: a tail of weights below half
// of that, which together may be 3e-5, would count as nothing.)  Counts go in the first word.
constexpr int kMassBits = 38;
typedef unsigned __int128 u128;
struct Mass {
  u64 hi, lo;
  __device__ __forceinline__ u128 value() const { return ((u128)hi << kMassBits) + lo; }
};
__device__ __forceinline__ Mass mass_from(double w) {  // w in [0, 1]
  const double s = ldexp(w, kMassBits), whole = floor(s);
  return {(u64)whole, (u64)ldexp(s - whole, kMassBits)};
}
struct MassLds {
  u64 hi[kFBins], lo[kFBins];
  u64 wlo[kFWaves];
  u64 above[2];
};
// As crossing, of masses.
__device__ int crossing_mass(MassLds& m, BlockLds& sh, u128 need, u128& above) {
  const int t = threadIdx.x, lane = t & (kWave - 1), w = t >> 6;
  const int b0 = kFBins - 1 - 2 * t;
  const Mass m0{m.hi[b0], m.lo[b0]}, m1{m.hi[b0 - 1], m.lo[b0 - 1]};
  const Mass incl{wave_scan64(m0.hi + m1.hi), wave_scan64(m0.lo + m1.lo)};
  if (lane == kWave - 1) {
    sh.wsum[w] = incl.hi;
    m.wlo[w] = incl.lo;
  }
  if (t == 0) sh.bin = 0;
  __syncthreads();
  Mass ahead{incl.hi - m0.hi - m1.hi, incl.lo - m0.lo - m1.lo};
  for (int i = 0; i < w; ++i) {
    ahead.hi += sh.wsum[i];
    ahead.lo += m.wlo[i];
  }
  const u128 before = above + ahead.value(), with0 = before + m0.value(), with1 = with0 + m1.value();
  if (before < need && with1 >= need) {
    const bool first = with0 >= need;
    sh.bin = first ? b0 : b0 - 1;
    const u128 over = first ? before : with0;
    m.above[0] = (u64)over;
    m.above[1] = (u64)(over >> 64);
  }
  __syncthreads();
  above = (u128)m.above[1] << 64 | m.above[0];
  const int bin = sh.bin;
  __syncthreads();
  return bin;
}

// A row by a whole 1024-thread workgroup, straight from the logits: every selection is a radix
// select over the keys (11, 11, 10 bits), counts or masses in an LDS histogram.  The row is not
// greedy and has a logit above -inf (mk).  A function of its own, out of the way of the code that
// nearly every row runs.
__device__ __noinline__ int select_row(const float* lg, int N, uint32_t mk, double it, int k_top,
                                       double p, double min_w, double u) {
  __shared__ MassLds hist;
  __shared__ BlockLds sh;
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int seg = ((N + kFWaves * kWave - 1) / (kFWaves * kWave)) * kWave;
  const int seg0 = min(w * seg, N), seg1 = min(seg0 + seg, N);
  auto for_each = [&](auto&& f) {
    constexpr int kAhead = 8;  // loads that wait together
    for (int i0 = seg0 + lane; i0 < seg1; i0 += kAhead * kWave) {
      float l[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) l[k] = lg[min(i0 + k * kWave, seg1 - 1)];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (i0 + k * kWave < seg1) f(key_of(l[k]), i0 + k * kWave);
    }
  };
  const double M = (double)logit_of(mk);
  auto weight = [&](uint32_t k) { return k == mk ? 1.0 : exp(((double)logit_of(k) - M) * it); };
  auto mass = [&](uint32_t k) { return mass_from(weight(k)); };
  // the cut: kept are keys above ck, and of those equal the indexes up to ci
  uint32_t ck = kKeyMasked + 1;
  int ci = N;
  auto kept = [&](uint32_t k, int i) { return k > ck || (k == ck && i <= ci); };
  // the prefix of what is kept whose `value`s sum to `need` or more: a new cut
  auto select = [&](u128 need, auto&& value) {
    uint32_t prefix = 0;
    u128 above = 0;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
      for (int b = t; b < kFBins; b += kFThreads) hist.hi[b] = hist.lo[b] = 0;
      __syncthreads();
      for_each([&](uint32_t k, int i) {
        if (kept(k, i) && (level == 0 || (k >> (shift + bits)) == prefix)) {
          const Mass v = value(k);
          const uint32_t b = k >> shift & ((1u << bits) - 1);
          atomicAdd(&hist.hi[b], v.hi);
          if (v.lo) atomicAdd(&hist.lo[b], v.lo);
        }
      });
      __syncthreads();
      prefix = prefix << bits | (uint32_t)crossing_mass(hist, sh, need, above);
    }
    // of the elements with this key, the first q: as many as reach what is left
    const Mass one = value(prefix);
    const u128 each = one.value(), rest = need - above;
    u64 q = 1;
    if (each) {  // the quotient in fp64, then made exact
      const auto f = [](u128 x) { return ldexp((double)(u64)(x >> 64), 64) + (double)(u64)x; };
      q = (u64)fmin(fmax(f(rest) / f(each), 1.0), (double)N);
      while (q < (u64)N && each * q < rest) ++q;
      while (q > 1 && each * (q - 1) >= rest) --q;
    }
    u64 n = 0;
    for_each([&](uint32_t k, int i) { n += k == prefix && kept(k, i) ? 1 : 0; });
    n = wave_sum64(n);
    if (lane == 0) sh.wsum[w] = n;
    if (t == 0) sh.pick = N;
    __syncthreads();
    u64 before = 0;
    for (int i = 0; i < w; ++i) before += sh.wsum[i];
    if (before < q && before + n >= q) {
      for (int s0 = seg0; s0 < seg1; s0 += kWave) {
        const int i = s0 + lane;
        uint32_t k = 0;
        if (i < seg1) k = key_of(lg[i]);
        const u64 hit = __ballot(i < seg1 && k == prefix && kept(k, i));
        const int c = (int)__popcll(hit);
        if (before + c >= q) {
          if ((hit >> lane & 1) && before + __popcll(hit & ((1ull << lane) - 1)) + 1 == q) sh.pick = i;
          break;
        }
        before += c;
      }
    }
    __syncthreads();
    ck = prefix;
    ci = sh.pick;
    __syncthreads();
  };
  if (k_top > 0) {
    u64 n = 0;
    for_each([&](uint32_t k, int i) { n += kept(k, i) ? 1 : 0; });
    if (block_sum(n, sh) > (u64)k_top)
      select((u128)k_top << kMassBits, [](uint32_t) { return Mass{1, 0}; });
  }
  if (p < 1.0) {
    Mass all{0, 0};
    for_each([&](uint32_t k, int i) {
      if (!kept(k, i)) return;
      const Mass v = mass(k);
      all.hi += v.hi;
      all.lo += v.lo;
    });
    all.hi = block_sum(all.hi, sh);
    all.lo = block_sum(all.lo, sh);
    // p times it in units of 2^-38 (p <= 1 - 2^-24, so that rounding does not take it past all)
    const double share = p * ((double)all.hi + ldexp((double)all.lo, -kMassBits)), whole = floor(share);
    const u128 need = ((u128)(u64)whole << kMassBits) + (u64)ceil(ldexp(share - whole, kMassBits));
    select(need > 0 ? need : (u128)1, mass);
  }
  // the pick
  auto kept_weight = [&](uint32_t k, int i) {
    if (!kept(k, i)) return 0.0;
    const double v = weight(k);
    return v >= min_w ? v : 0.0;
  };
  double m = 0.0;
  for_each([&](uint32_t k, int i) { m += kept_weight(k, i); });
  m = wave_sum64(m);
  if (lane == 0) sh.wmass[w] = m;
  if (t == 0) sh.pick = -1;
  __syncthreads();
  double Z = 0.0;
  for (int i = 0; i < kFWaves; ++i) Z += sh.wmass[i];
  const double target = u * Z;
  // the first wave whose running mass reaches the draw (or the last with any mass)
  int owner = -1;
  double before = 0.0, acc = 0.0;
  for (int i = 0; i < kFWaves; ++i) {
    if (sh.wmass[i] > 0.0 && (owner < 0 || acc < target)) {
      owner = i;
      before = acc;
    }
    acc += sh.wmass[i];
  }
  if (w != owner) return -1;
  int last = -1;
  for (int s0 = seg0; s0 < seg1; s0 += kWave) {
    const int i = s0 + lane;
    const double v = i < seg1 ? kept_weight(key_of(lg[i]), i) : 0.0;
    const double incl = wave_scan64(v);
    const u64 has = __ballot(v > 0.0), hit = __ballot(v > 0.0 && before + incl >= target);
    if (hit) {
      last = s0 + (int)__builtin_ctzll(hit);
      break;
    }
    if (has) last = s0 + 63 - (int)__builtin_clzll(has);
    before += wave_last64(incl);
  }
  return lane == 0 ? last : -1;
}

// ---- bins ----------------------------------------------------------------------------
constexpr int kNoBin = -(1 << 30);

// bin_weight_raised with its coefficients in scalar registers (hidden from the compiler, which would
// otherwise move each of them into vector registers for every weight).
struct BinWeight {
  double c[6];
  __device__ __forceinline__ BinWeight() {
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      c[i] = kBinWeight[i];
      if (i == 4)  // an instruction takes one scalar
        asm("" : "+v"(c[i]));
      else
        asm("" : "+s"(c[i]));
    }
  }
  __device__ __forceinline__ double raised(double r) const { return bin_weight_raised(c, r); }
  __device__ __forceinline__ u64 operator()(double r) const {
    return __builtin_bit_cast(u64, raised(r)) & 0xfffffffffffffull;
  }
};

// ---- the parts -----------------------------------------------------------------------
constexpr int kSThreads = 512;
constexpr int kSWaves = kSThreads / kWave;
constexpr int kPer = 20;  // logits of a thread
constexpr int kPartLen = kSThreads * kPer;
constexpr int kSmallK = 64;
constexpr int kListCap = 256;             // a part's list; at most top_k where it would be longer
constexpr int kBody = kBins + kBins / 2;  // masses, and counts of 32 bits
constexpr int kWordCap = 8192;  // logits of the cuts' bins that are selected from

// What the parts make of a row together.
struct RowBins {
  u64 word[kWordCap];      // rank words of the logits in bins that a cut may lie in, in any order
  double mass[kBins + 1];  // of the bins from this one up, in the largest weight's bin's units
  u64 count[kBins + 1];
  int n;                   // words (more than kWordCap: those past it are not there)
  u64 hist[kBins];         // masses of the bins, in their own units
  int bin[3];              // bins that a cut may lie in: top-k's, top-p's highest and lowest
  uint32_t edge[6];        // first and last keys of top-k's bin, top-p's bins, min-p's
};

struct ScanLds {
  float wtop[kSWaves];
  int widx[kSWaves];
  union {
    struct {
      u64 mass[kBins * kBinCols];
      uint32_t count[kBins * kBinCols];
    } h;
    struct {
      u64 list[kListCap];
      uint32_t best[kSThreads];
      uint32_t wcut[kSWaves];
      int wcnt[kSWaves];
      int n;
    } c;
  };
};

// Workgroup -> (row, part).  Workgroups are dealt to the 8 XCDs round robin: all parts of row r go to
// XCD r % 8, and the pick of the row (workgroup r) with them, so that what the parts leave is found
// in that XCD's L2.
// kBack: the last first, for the gather: what the scan read last is still in the caches (256 rows of
// nuclei 2 us faster).
constexpr int kXcds = 8;
template <bool kBack>
__device__ __forceinline__ bool part_of(const FilterArgs& a, int& row, int& part) {
  const int xcd = blockIdx.x % kXcds, n = gridDim.x / kXcds;
  const int i = kBack ? n - 1 - (int)(blockIdx.x / kXcds) : (int)(blockIdx.x / kXcds), group = i / a.parts;
  row = group * kXcds + xcd;
  part = i - group * a.parts;
  return row < a.rows;
}
__device__ __forceinline__ u64 rank_word(uint32_t key, int i) {  // larger: earlier in the order
  return (u64)key << 32 | (uint32_t)~i;
}
// The largest v (of its upper 16 bits) that `need` lanes of the wave reach; 0 if fewer have any.
__device__ __forceinline__ uint32_t wave_nth_largest(uint32_t v, int need) {
  uint32_t cut = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t at = cut | 1u << b;
    if ((int)__popcll(__ballot(v >= at)) >= need) cut = at;
  }
  return cut;
}

// 8 waves a SIMD: the loads of one workgroup go on under the arithmetic of the others.
__global__ void __launch_bounds__(kSThreads, 8) filter_scan_kernel(FilterArgs a) {
  __shared__ ScanLds sh;
  int row, part;
  if (!part_of<false>(a, row, part)) return;
  const int N = a.vocab;
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const float* lg = a.logits + (long long)row * a.stride;
  const int base = part * kPartLen;
  float x[kPer];
#pragma unroll
  for (int j = 0; j < kPer / 4; ++j) {
    const int i = base + (j * kSThreads + t) * 4;
    if (i + 3 < N) {
      __builtin_memcpy(&x[4 * j], lg + i, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * j + e] = i + e < N ? lg[i + e] : -INFINITY;
    }
  }
  const auto index = [&](int e) { return base + ((e >> 2) * kSThreads + t) * 4 + (e & 3); };
  const Settings st = settings_of(a, row);
  const bool lists = !st.greedy && st.k > 0 && st.k <= kSmallK, bins = !st.greedy && !lists;
  if (bins) {
    for (int i = t; i < kBins * kBinCols; i += kSThreads) sh.h.mass[i] = 0;
    if (st.k > 0)
      for (int i = t; i < kBins * kBinCols; i += kSThreads) sh.h.count[i] = 0;
  } else if (t == 0) {
    sh.c.n = 0;
  }
  // the part's largest logit.  v_max of x with itself makes a signalling NaN a quiet one, and of a
  // quiet NaN and a number v_max3 gives the number.
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < kPer; e += 2) {
    float q0, q1;
    asm("v_max_f32 %0, %1, %1" : "=v"(q0) : "v"(x[e]));
    asm("v_max_f32 %0, %1, %1" : "=v"(q1) : "v"(x[e + 1]));
    asm("v_max3_f32 %0, %1, %2, %0" : "+v"(m) : "v"(q0), "v"(q1));
  }
  if (lists) sh.c.best[t] = key_of(m);
  float top = logit_of(wave_max_key(key_of(m)));
  int first = 0x7fffffff;  // its lowest index, for greedy rows
  if (st.greedy) {
#pragma unroll
    for (int e = kPer - 1; e >= 0; --e) first = x[e] == top ? index(e) : first;
    first = wave_extreme<false>(first, 0x7fffffff);
  }
  if (lane == 0) {
    sh.wtop[w] = top;
    sh.widx[w] = first;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSWaves; ++i) top = fmaxf(top, sh.wtop[i]);
  first = 0x7fffffff;
  if (st.greedy)
#pragma unroll
    for (int i = 0; i < kSWaves; ++i) first = sh.wtop[i] == top ? min(first, sh.widx[i]) : first;
  const uint32_t top_key = key_of(top);
  if (part == 0 && t == 0) a.bins[row].n = 0;
  const long long slot = (long long)row * a.parts + part;
  int4 head{(int)top_key, first, 0, kNoBin};
  u64* body = a.body + slot * kBody;
  if (top_key <= kKeyMasked || st.greedy) {
    if (t == 0) a.head[slot] = head;
    return;
  }
  if (lists) {
    // a bound below the part's st.k-th largest: an eighth of them in every wave's share of the
    // threads' maxima (each share from all over the part)
    const uint32_t own = wave_nth_largest(sh.c.best[lane * kSWaves + w], (st.k + kSWaves - 1) / kSWaves);
    if (lane == 0) sh.c.wcut[w] = own;
    __syncthreads();
    uint32_t cut = sh.c.wcut[0];
#pragma unroll
    for (int i = 1; i < kSWaves; ++i) cut = min(cut, sh.c.wcut[i]);
    const float low = logit_of(max(cut, kKeyMasked + 1));
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (x[e] >= low) {
        const int at = atomicAdd(&sh.c.n, 1);
        if (at < kListCap) sh.c.list[at] = rank_word(key_of(x[e]), index(e));
      }
    __syncthreads();
    int n = sh.c.n;
    if (n > kListCap) {
      // many equal or nearly equal logits: the part's first st.k exactly.  The st.k-th largest key:
      uint32_t key = 0;
      for (int b = 31; b >= 0; --b) {
        const uint32_t at = key | 1u << b;
        int c = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) c += (int)__popcll(__ballot(key_of(x[e]) >= at));
        if (lane == 0) sh.c.wcnt[w] = c;
        __syncthreads();
        c = 0;
#pragma unroll
        for (int i = 0; i < kSWaves; ++i) c += sh.c.wcnt[i];
        if (c >= st.k) key = at;
        __syncthreads();
      }
      if (t == 0) sh.c.n = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint32_t k = key_of(x[e]);
        if (k > key) sh.c.list[atomicAdd(&sh.c.n, 1)] = rank_word(k, index(e));
      }
      __syncthreads();
      // ... and of those equal to it the lowest indexes (index order: 4 of a thread, threads, runs)
      n = sh.c.n;
#pragma unroll
      for (int j = 0; j < kPer / 4; ++j) {
        int c = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) c += key_of(x[4 * j + e]) == key ? 1 : 0;
        const int incl = wave_incl_scan(c);
        if (lane == kWave - 1) sh.c.wcnt[w] = incl;
        __syncthreads();
        int at = n + incl - c;
#pragma unroll
        for (int i = 0; i < kSWaves; ++i) {
          if (i < w) at += sh.c.wcnt[i];
          n += sh.c.wcnt[i];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key_of(x[4 * j + e]) == key) {
            if (at < st.k) sh.c.list[at] = rank_word(key, index(4 * j + e));
            ++at;
          }
        __syncthreads();
      }
      n = st.k;
    }
    for (int i = t; i < n; i += kSThreads) body[i] = sh.c.list[i];
    head.z = n;
    if (t == 0) a.head[slot] = head;
    return;
  }
  const double c = kEightLog2e * st.it;
  const double place = (double)top * c;
  if (!st.extreme && top_key < kKeyInf && __builtin_fabs(place) < kMaxPartPlace) {
    double r;
    const int hi = bin_of((double)top, c, r), lo = hi - (kBins - 1);
    // The first logits above the middle of the lowest bin (or, where logits are further apart than
    // the bins reach, the largest alone): what passes the comparison (NaN does not) is in the bins.
    const float mid = (float)((double)lo / c);
    const float low = fminf(logit_of(key_of(fmaxf(mid, -FLT_MAX)) + (mid > -FLT_MAX)), top);
    const uint32_t slots = slot_base(lo, t & (kBinCols - 1));
    const BinWeight bin_weight;
    double round = kRound;
    asm("" : "+s"(round));
    if (st.k > 0) {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (x[e] >= low) {
          const uint32_t at = bin_slot(bin_of((double)x[e], c, r, round), slots);
          atomicAdd(&sh.h.mass[at], bin_weight(r));
          atomicAdd(&sh.h.count[at], 1u);
        }
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (x[e] >= low) {
          const uint32_t at = bin_slot(bin_of((double)x[e], c, r, round), slots);
          atomicAdd(&sh.h.mass[at], bin_weight(r));
        }
    }
    head.w = hi;
  }
  __syncthreads();
  if (t < kBins) {
    u64 mass = 0;
#pragma unroll
    for (int k = 0; k < kBinCols; ++k) mass += sh.h.mass[t * kBinCols + ((k + t) & (kBinCols - 1))];
    body[t] = mass;
    if (st.k > 0) {
      uint32_t n = 0;
#pragma unroll
      for (int k = 0; k < kBinCols; ++k) n += sh.h.count[t * kBinCols + ((k + t) & (kBinCols - 1))];
      reinterpret_cast<uint32_t*>(body + kBins)[t] = n;
    }
  }
  if (t == 0) a.head[slot] = head;
}

// ---- the cuts' bins --------------------------------------------------------------------
// Keys of a row's bins.
struct Keys {
  double c;
  int lo;       // the row's lowest bin
  uint32_t mk;  // its largest key

  // the first key from kKeyMasked + 1 on that `yes` holds for; it holds from some key on, and for mk
  template <class F>
  __device__ __forceinline__ uint32_t first(F&& yes) const {
    const int lane = threadIdx.x & (kWave - 1);
    uint32_t from = kKeyMasked + 1, to = mk;
    while (from < to) {
      const uint32_t step = (to - from) / kWave + 1;
      const u64 reached = __ballot(yes((uint32_t)min((u64)from + (u64)step * lane, (u64)to)));
      if (!reached) {  // past the last lane's
        from += step * (kWave - 1) + 1;
        continue;
      }
      const int f = (int)__builtin_ctzll(reached);
      to = (uint32_t)min((u64)from + (u64)step * f, (u64)to);
      if (f) from += step * (f - 1) + 1;
    }
    return to;
  }
  __device__ __forceinline__ uint32_t first_of_bin(int b) const {
    const auto yes = [&](uint32_t k) {
      const double l = (double)logit_of(k);
      double r;
      return l * c > -kMaxPartPlace && bin_of(l, c, r) >= lo + b;
    };
    // within a few steps of the bin's lower edge, where that is not at an end of the keys
    const uint32_t near = key_of((float)(((double)(lo + b) - 0.5) / c)) - kWave / 2;
    if (near > kKeyMasked && near + kWave <= mk) {
      const u64 reached = __ballot(yes(near + (threadIdx.x & (kWave - 1))));
      if (reached && !(reached & 1)) return near + (uint32_t)__builtin_ctzll(reached);
    }
    return first(yes);
  }
  __device__ __forceinline__ uint32_t last_of_bin(int b) const {
    return b == kBins - 1 ? mk : first_of_bin(b + 1) - 1;
  }
};
// The bin at which min-p cuts (-1: below all).
__device__ __forceinline__ int min_p_bin(const Settings& st, double place, int lo) {
  if (!(st.min_w > 0.0)) return -1;
  double r;
  return max(bin_of(place + 8.0 * log2(st.min_w), 1.0, r) - lo, -1);
}
// Whether the bins serve the row.
__device__ __forceinline__ bool bins_serve(const Settings& st, uint32_t mk, double place) {
  return mk > kKeyMasked && mk < kKeyInf && !st.extreme && st.u != 0.0 &&
         __builtin_fabs(place) <= kMaxPlace;
}

struct MergeLds {
  u64 hist[kBins];
  u64 count[kBins + 1];
  double mass[kBins + 1];
  double wmass[kSWaves];
  u64 wsum[kSWaves];
  int bin[3];        // top-k's; top-p's highest and lowest (its need is known to the top-k's bin)
  uint32_t edge[6];  // key ranges: top-k's bin, top-p's bins, min-p's
};

// A row's bins summed up over its parts by a whole 512-thread workgroup, and the keys of the bins
// that a cut may lie in (sh.edge).  With `leave` the sums go to `out`.  False if the row has
// nothing to gather.
__device__ __forceinline__ bool merge_row(const FilterArgs& a, int row, const Settings& st,
                                          MergeLds& sh, RowBins& out, bool leave) {
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int4* head = a.head + (long long)row * a.parts;
  const u64* body = a.body + (long long)row * a.parts * kBody;
  uint32_t mk = 0;
  for (int p = lane; p < a.parts; p += kWave) mk = max(mk, (uint32_t)head[p].x);
  Keys keys;
  keys.mk = mk = wave_max_key(mk);
  keys.c = kEightLog2e * st.it;
  const double place = (double)logit_of(mk) * keys.c;
  if (!bins_serve(st, mk, place)) return false;
  double r;
  const int hi = bin_of((double)logit_of(mk), keys.c, r), lo = keys.lo = hi - (kBins - 1);
  if (t <= kBins) {
    if (t < kBins) sh.hist[t] = 0;
    sh.count[t] = 0;
    sh.mass[t] = 0.0;
  }
  if (t < 3) sh.bin[t] = -1;
  if (t < 6) sh.edge[t] = t & 1 ? 0u : ~0u;
  __syncthreads();
  constexpr int kRuns = kBins / kWave;  // of 64 bins
  const auto add = [&](int run, u64 m, uint32_t n) {
    const int p = run / kRuns, b = (run - p * kRuns) * kWave + lane - (hi - head[p].w);
    if ((uint32_t)b >= (uint32_t)kBins || !m) return;
    atomicAdd(&sh.hist[b], m);
    if (st.k > 0) atomicAdd(&sh.count[b], (u64)n);
  };
  constexpr int kAhead = 6;
  for (int run0 = w; run0 < a.parts * kRuns; run0 += kAhead * kSWaves) {
    u64 m[kAhead];
    uint32_t n[kAhead] = {};
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int run = min(run0 + k * kSWaves, a.parts * kRuns - 1), p = run / kRuns;
      const u64* from = body + (long long)p * kBody;
      m[k] = from[(run - p * kRuns) * kWave + lane];
      if (st.k > 0)
        n[k] = reinterpret_cast<const uint32_t*>(from + kBins)[(run - p * kRuns) * kWave + lane];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (run0 + k * kSWaves < a.parts * kRuns) add(run0 + k * kSWaves, m[k], n[k]);
  }
  __syncthreads();
  {  // sums from the top down
    const int b = kBins - 1 - t;
    const double m = t < kBins ? (double)sh.hist[b] * exp2((double)(b - (kBins - 1)) * 0.125) : 0.0;
    double mass = wave_scan64(m);
    u64 n = wave_scan64(t < kBins ? sh.count[b] : (u64)0);
    if (lane == kWave - 1) {
      sh.wmass[w] = mass;
      sh.wsum[w] = n;
    }
    __syncthreads();
    for (int i = 0; i < w; ++i) {
      mass += sh.wmass[i];
      n += sh.wsum[i];
    }
    if (t < kBins) {
      sh.mass[b] = mass;
      sh.count[b] = n;
    }
  }
  __syncthreads();
  if (leave && t <= kBins) {
    out.mass[t] = sh.mass[t];
    out.count[t] = sh.count[t];
    if (t < kBins) out.hist[t] = sh.hist[t];
  }
  const bool by_count = st.k > 0 && sh.count[0] > (u64)st.k;
  const int min_bin = min_p_bin(st, place, lo);
  if (!by_count && st.p >= 1.0 && min_bin < 0) return false;
  if (by_count && t < kBins && sh.count[t] >= (u64)st.k && sh.count[t + 1] < (u64)st.k) sh.bin[0] = t;
  __syncthreads();
  if (st.p < 1.0 && t < kBins) {
    // top-p's share is of the mass that top-k leaves: more than that above its bin, at most with it
    const int bk = by_count ? sh.bin[0] : -1;
    const double least = st.p * (by_count ? sh.mass[bk + 1] : sh.mass[0]);
    const double most = st.p * sh.mass[by_count ? bk : 0];
    // (the highest: rounding can leave more than one bin whose sum reaches it and the next's not)
    const bool end = t == kBins - 1;
    if (sh.mass[t] >= least && (end || sh.mass[t + 1] < least)) atomicMax(&sh.bin[1], t);
    if (sh.mass[t] >= most && (end || sh.mass[t + 1] < most)) atomicMax(&sh.bin[2], t);
  }
  __syncthreads();
  const int first = w < 2 ? sh.bin[0] : w < 4 ? sh.bin[2] : min_bin;
  const int last = w < 2 ? sh.bin[0] : w < 4 ? sh.bin[1] : min_bin;
  if (w < 6 && first >= 0 && last >= 0) {
    const uint32_t k = w & 1 ? keys.last_of_bin(last) : keys.first_of_bin(first);
    if (lane == 0) sh.edge[w] = k;
  }
  __syncthreads();
  if (leave && t < 6) out.edge[t] = sh.edge[t];
  if (leave && t < 3) out.bin[t] = sh.bin[t];
  return true;
}
__device__ __forceinline__ bool gathers(const Settings& st) {
  return !st.greedy && !(st.k > 0 && st.k <= kSmallK) && !st.extreme;
}

// The merge alone, a workgroup per row.
__global__ void __launch_bounds__(kSThreads) filter_merge_kernel(FilterArgs a) {
  __shared__ MergeLds sh;
  const int row = blockIdx.x, t = threadIdx.x;
  const Settings st = settings_of(a, row);
  RowBins& out = a.bins[row];
  if (!(gathers(st) && merge_row(a, row, st, sh, out, true)) && t < 6)
    out.edge[t] = t & 1 ? 0u : ~0u;  // nothing to gather
}

// The logits of the bins that a cut may lie in, a workgroup per part.  kMerge: each finds those
// bins itself (the same in each; part 0 leaves the sums for the pick) while its logits are on their
// way, else filter_merge_kernel has, and a row without any is left at once.
template <bool kMerge>
__global__ void __launch_bounds__(kSThreads, kMerge ? 6 : 8) filter_gather_kernel(FilterArgs a) {
  __shared__ int s_n, s_base;
  int row, part;
  if (!part_of<true>(a, row, part)) return;
  const int N = a.vocab;
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const float* lg = a.logits + (long long)row * a.stride;
  const int base = part * kPartLen;
  float x[kPer];
  const auto load = [&] {
#pragma unroll
    for (int j = 0; j < kPer / 4; ++j) {
      const int i = base + (j * kSThreads + t) * 4;
      if (i + 3 < N) {
        __builtin_memcpy(&x[4 * j], lg + i, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * j + e] = i + e < N ? lg[i + e] : -INFINITY;
      }
    }
  };
  RowBins& out = a.bins[row];
  if (t == 0) s_n = 0;
  float low[3], high[3];
  int ranges = 0;  // of logits, in front
  const auto take = [&](const uint32_t* edge) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      low[k] = INFINITY;
      high[k] = -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (edge[2 * k] <= edge[2 * k + 1]) {
        const float l = logit_of(edge[2 * k]), h = logit_of(edge[2 * k + 1]);
#pragma unroll
        for (int i = 0; i < 3; ++i)
          if (i == ranges) {
            low[i] = l;
            high[i] = h;
          }
        ++ranges;
      }
  };
  if constexpr (kMerge) {
    __shared__ MergeLds sh;
    const Settings st = settings_of(a, row);
    const bool cuts = st.k > 0 || st.p < 1.0 || st.min_w > 0.0;
    if (!gathers(st) || (!cuts && part != 0)) return;
    load();
    if (!merge_row(a, row, st, sh, out, part == 0)) return;
    take(sh.edge);
  } else {
    uint32_t edge[6];
#pragma unroll
    for (int k = 0; k < 6; ++k) edge[k] = (uint32_t)__builtin_amdgcn_readfirstlane((int)out.edge[k]);
    take(edge);
  }
  if (ranges == 0) return;
  if constexpr (!kMerge) load();
  // a lane's hits, its first logit in the highest bit
  uint32_t hits = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) hits = hits + hits + (x[e] >= low[0] && x[e] <= high[0] ? 1u : 0u);
  if (ranges > 1)
#pragma unroll
    for (int k = 1; k < 3; ++k) {
      uint32_t more = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) more = more + more + (x[e] >= low[k] && x[e] <= high[k] ? 1u : 0u);
      hits |= more;
    }
  const int mine = (int)__popc(hits), incl = wave_incl_scan(mine);
  const int n = __builtin_amdgcn_readlane(incl, kWave - 1);
  if constexpr (!kMerge) __syncthreads();  // s_n
  int at = 0;
  if (n && lane == 0) at = atomicAdd(&s_n, n);
  at = __builtin_amdgcn_readfirstlane(at) + incl - mine;
  __syncthreads();
  if (t == 0 && s_n) s_base = atomicAdd(&out.n, s_n);
  __syncthreads();
  if (n == 0) return;
  at += s_base;
  // the few there are, read again (from L2): a lane's registers have no index
  for (; hits; hits &= hits - 1, ++at) {
    const int e = kPer - 1 - (int)__builtin_ctz(hits), i = base + ((e >> 2) * kSThreads + t) * 4 + (e & 3);
    if (at < kWordCap) out.word[at] = rank_word(key_of(lg[i]), i);
  }
}

// ---- the pick ------------------------------------------------------------------------
constexpr int kMaxParts = 1024;
constexpr int kMaxRows = 1 << 20;

struct PickLds {
  u64 word[kWordCap];   // rank words: the parts' lists, or the logits of one bin
  u64 hist[kFBins];         // also the short list of pick_listed, select_row's histogram
  u64 listed[kMaxParts];    // by part: kept weights of the cut's bin; offsets of the lists
  double part[kMaxParts];   // ... kept mass
  int hi[kMaxParts];        // ... highest bin
  int len[kMaxParts];       // ... length of the list
  double scale[kBins + 1];  // of a bin's unit, relative to the largest weight's bin
  double mass[kBins + 1];   // what the parts make together: RowBins'
  u64 count[kBins + 1];
  u64 row_hist[kBins];
  int cut_bins[3];
  uint32_t edge[6];
  int bin, n;
  BlockLds b;
};

// The value of lane l ^ kMask, without a trip through LDS: quad permutes, row rotations (by 8 of 16
// lanes) and mirrors, and swaps of rows and halves.
template <int kMask>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
  if constexpr (kMask == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return (threadIdx.x & 32) ? r[0] : r[1];
  } else if constexpr (kMask == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return (threadIdx.x & 16) ? r[0] : r[1];
  } else if constexpr (kMask == 8) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true);  // row_ror:8
  } else if constexpr (kMask == 4) {  // half mirror (l ^ 7), then quads reversed (l ^ 3)
    const int y = __builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true);
    return (uint32_t)__builtin_amdgcn_update_dpp(0, y, 0x1b, 0xf, 0xf, true);
  } else {
    constexpr int kQuad = kMask == 2 ? 0x4e : 0xb1;  // [2,3,0,1], [1,0,3,2]
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kQuad, 0xf, 0xf, true);
  }
}
template <int kMask>
__device__ __forceinline__ u64 lane_xor64(u64 x) {
  return (u64)lane_xor<kMask>((uint32_t)(x >> 32)) << 32 | lane_xor<kMask>((uint32_t)x);
}
template <int kLen, int kMask>
__device__ __forceinline__ u64 sort_step(u64 v) {
  const int lane = threadIdx.x & (kWave - 1);
  const u64 y = lane_xor64<kMask>(v);
  const bool keep_max = ((lane & kMask) == 0) == ((lane & kLen) == 0 || kLen == kWave);
  v = (v > y) == keep_max ? v : y;
  if constexpr (kMask > 1) v = sort_step<kLen, kMask / 2>(v);
  return v;
}
// Descending sorting network over the wave's lanes (steps of length kFrom..64).
template <int kFrom>
__device__ __forceinline__ u64 wave_sort_desc(u64 v) {
  v = sort_step<kFrom, kFrom / 2>(v);
  if constexpr (kFrom < kWave) v = wave_sort_desc<kFrom * 2>(v);
  return v;
}

__device__ __forceinline__ double weight_of(uint32_t k, uint32_t mk, double M, double it) {
  return k == mk ? 1.0 : exp(((double)logit_of(k) - M) * it);
}

// What a thread of the pick asks for at once, before it knows what it needs.
constexpr int kHeld = kBins / kWave;
struct Early {
  u64 held[kHeld];  // top_k <= 64: entry `lane` of part w's list; else part w's masses, 64 of each to a
                    // wave
  double mass;      // RowBins' entries t
  u64 count, hist;
  uint32_t edge;
  int bin, n;
};

// top_k <= 64: the row's top_k from the parts' lists, sorted, in one wave's lanes.  False if the
// lists are longer than LDS holds.
__device__ bool pick_listed(const FilterArgs& a, int row, const Settings& st, uint32_t mk,
                            const Early& early, PickLds& sh) {
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const u64* body = a.body + (long long)row * a.parts * kBody;
  {  // offsets of the lists
    const int n = t < a.parts ? sh.len[t] : 0;
    const int incl = wave_incl_scan(n);
    if (lane == kWave - 1) sh.b.wsum[w] = (u64)incl;
    __syncthreads();
    int at = incl - n;
    for (int i = 0; i < w; ++i) at += (int)sh.b.wsum[i];
    sh.listed[t] = (u64)at;
    if (t == kFThreads - 1) sh.n = at + n;
    __syncthreads();
  }
  int n = sh.n;
  if (n > kWordCap) return false;
  for (int p = w; p < a.parts; p += kFWaves) {
    const int at = (int)sh.listed[p], c = sh.len[p];
    int i = lane;
    if (p < kFWaves) {
      if (i < c) sh.word[at + i] = early.held[0];
      i += kWave;
    }
    for (; i < c; i += kWave) sh.word[at + i] = body[(long long)p * kBody + i];
  }
  __syncthreads();
  const u64* list = sh.word;
  if (n > kWave) {
    // words below a bound of the top_k-th largest are not among the first top_k: a sixteenth of
    // them in every wave's threads' largest
    uint32_t k = 0;
    for (int i = t; i < n; i += kFThreads) k = max(k, (uint32_t)(sh.word[i] >> 32));
    const uint32_t own = wave_nth_largest(k, (st.k + kFWaves - 1) / kFWaves);
    if (lane == 0) sh.b.wsum[w] = own;
    if (t == 0) sh.n = 0;
    __syncthreads();
    uint32_t cut = (uint32_t)sh.b.wsum[0];
#pragma unroll
    for (int i = 1; i < kFWaves; ++i) cut = min(cut, (uint32_t)sh.b.wsum[i]);
    for (int i = t; i < n; i += kFThreads)
      if ((uint32_t)(sh.word[i] >> 32) >= cut) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < kFBins) sh.hist[at] = sh.word[i];
      }
    __syncthreads();
    n = sh.n;
    if (n > kFBins) return false;
    list = sh.hist;
  }
  // each wave's largest 64, then wave 0 merges the waves'
  const int chunks = (n + kWave - 1) / kWave;
  u64 v = 0;
  for (int c = w; c < chunks; c += kFWaves) {
    const int i = c * kWave + lane;
    const u64 y = wave_sort_desc<2>(i < n ? list[i] : 0);
    if (c == w) {
      v = y;
    } else {
      const u64 r = __shfl(y, kWave - 1 - lane, kWave);
      v = wave_sort_desc<kWave>(v > r ? v : r);
    }
  }
  u64* sorted = reinterpret_cast<u64*>(sh.part);  // [waves][64]
  static_assert(kFWaves * kWave <= kMaxParts, "sorted");
  __syncthreads();
  sorted[t] = v;
  __syncthreads();
  if (w != 0) return true;
  for (int i = 1; i < min(chunks, kFWaves); ++i) {
    const u64 r = sorted[i * kWave + kWave - 1 - lane];
    v = wave_sort_desc<kWave>(v > r ? v : r);
  }
  const uint32_t key = (uint32_t)(v >> 32);
  const int idx = (int)~(uint32_t)v;
  const bool valid = lane < st.k && v != 0;
  const double wt = valid ? weight_of(key, mk, (double)logit_of(mk), st.it) : 0.0;
  const double incl = wave_scan64(wt), Z = wave_last64(incl);
  const double before = __builtin_bit_cast(double, dpp64<kDppWaveShr1, 0xf>(__builtin_bit_cast(u64, incl)));
  const bool keep = valid && (lane == 0 || st.p >= 1.0 || before < st.p * Z) && wt >= st.min_w;
  // running masses in the order of the vocabulary: each adds those of lower index
  double total = 0.0, run = 0.0;
  for (u64 left = __ballot(keep); left; left &= left - 1) {
    const int j = (int)__builtin_ctzll(left);
    const u64 bits = __builtin_bit_cast(u64, wt);
    const u64 of_j = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), j) << 32 |
                     (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, j);
    const double wj = __builtin_bit_cast(double, of_j);
    total += wj;
    run += __builtin_amdgcn_readlane(idx, j) <= idx ? wj : 0.0;
  }
  const double target = st.u * total;
  const bool some = keep && wt > 0.0;
  const int first = wave_extreme<false>(some && run >= target ? idx : 0x7fffffff, 0x7fffffff);
  const int last = wave_extreme<true>(some ? idx : -1, -1);
  if (lane == 0) a.out[row] = first != 0x7fffffff ? first : last;
  return true;
}

// The other filters, from the parts' bins.  False where select_row has to do the row.
__device__ bool pick_binned(const FilterArgs& a, int row, const Settings& st, uint32_t mk,
                            const Early& early, PickLds& sh) {
  const int t = threadIdx.x, lane = t & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  Keys keys;
  keys.mk = mk;
  const double M = (double)logit_of(mk), c = keys.c = kEightLog2e * st.it, place = M * c;
  if (!bins_serve(st, mk, place)) return false;
  const RowBins& in = a.bins[row];
  const int n = early.n;
  if (n > kWordCap) return false;
  const u64* body = a.body + (long long)row * a.parts * kBody;
  const float* lg = a.logits + (long long)row * a.stride;
  double r_top;
  const int hi = bin_of(M, c, r_top), lo = keys.lo = hi - (kBins - 1);  // the row's bins: lo..hi
  for (int i = t; i < n; i += kFThreads) sh.word[i] = in.word[i];
  if (t <= kBins) {
    sh.mass[t] = early.mass;
    sh.count[t] = early.count;
    sh.scale[t] = exp2((double)(t - (kBins - 1)) * 0.125);
  }
  if (t < kBins) sh.row_hist[t] = early.hist;
  if (t < 6) sh.edge[t] = early.edge;
  if (t < 3) sh.cut_bins[t] = early.bin;
  sh.listed[t] = 0;
  __syncthreads();
  const BinWeight bin_weight;
  const auto mass_of = [&](uint32_t key) {
    double r;
    bin_of((double)logit_of(key), c, r);
    return bin_weight(r);
  };
  // the highest bin for which `reached` holds
  const auto bin_at = [&](auto&& reached) {
    __syncthreads();
    if (t == 0) sh.bin = 0;
    __syncthreads();
    if (t < kBins && reached(t) && (t == kBins - 1 || !reached(t + 1))) atomicMax(&sh.bin, t);
    __syncthreads();
    return sh.bin;
  };

  u64 cut = 0;       // kept: rank words from the cut on
  int cut_bin = -1;  // the cut's bin: those above are kept whole
  uint32_t k0 = 0, k1 = 0;  // its keys
  const auto in_bin = [&](u64 word) {
    const uint32_t k = (uint32_t)(word >> 32);
    return k >= k0 && k <= k1 && word >= cut;
  };
  double Z = sh.mass[0];
  const int min_bin = min_p_bin(st, place, lo);
#pragma nounroll
  for (int stage = 0; stage < 3; ++stage) {  // top-k, top-p, min-p (one copy of the code for all)
    int b = min_bin;
    double need = 0.0;
    if (stage == 0) {
      if (st.k <= 0 || sh.count[0] <= (u64)st.k) continue;
      b = bin_at([&](int i) { return sh.count[i] >= (u64)st.k; });
    } else if (stage == 1) {
      if (st.p >= 1.0) continue;
      need = st.p * Z;
      b = bin_at([&](int i) { return sh.mass[i] >= need; });
      b = max(min(max(b, sh.cut_bins[2]), sh.cut_bins[1]), cut_bin);  // (Z's last bits are not the merge's)
      if (b < min_bin) continue;
    } else if (min_bin < 0 || min_bin < cut_bin) {
      continue;
    }
    if (b != cut_bin) {
      cut = 0;
      cut_bin = b;
      const int e = stage == 0 ? 0 : stage == 1 ? 2 : 4;
      if (stage != 1 || sh.cut_bins[1] == sh.cut_bins[2]) {
        k0 = sh.edge[e];
        k1 = sh.edge[e + 1];
      } else {
        k0 = keys.first_of_bin(b);
        k1 = keys.last_of_bin(b);
      }
    }
    if (stage == 2) {
      const uint32_t k = keys.first([&](uint32_t x) { return weight_of(x, mk, M, st.it) >= st.min_w; });
      cut = max(cut, (u64)k << 32);
      continue;
    }
    // the last of the first words, in their order, whose counts or masses sum to `want`
    const bool masses = stage == 1;
    const auto value = [&](u64 word) { return masses ? mass_of((uint32_t)(word >> 32)) : (u64)1; };
    u64 all_of = masses ? sh.row_hist[b] : sh.count[b] - sh.count[b + 1];
    if (cut != 0) {
      all_of = 0;
      for (int i = t; i < n; i += kFThreads)
        if (in_bin(sh.word[i])) all_of += value(sh.word[i]);
      all_of = block_sum(all_of, sh.b);
    }
    if (all_of == 0) {
      cut = (u64)(k1 + 1) << 32;
      continue;
    }
    const double rest = masses ? ceil((need - sh.mass[b + 1]) / sh.scale[b])
                               : (double)((u64)st.k - sh.count[b + 1]);
    u64 want = min(rest < 1.0 ? 1 : (u64)rest, all_of), above = 0;
    // a radix select over their keys, then among those of one key over the indexes (below 2^24: of
    // ~index the low 24 bits tell), until no more than a wave's lanes are left
    uint32_t key0 = k0, key1 = k1;
    int bits = k1 > k0 ? 32 - __builtin_clz(k1 - k0) : 0;
    bool by_index = false;
    uint32_t id0 = 0, id1 = 0xffffffu;
#pragma nounroll
    for (;;) {
      const auto left = [&](u64 x) {
        const uint32_t k = (uint32_t)(x >> 32), id = (uint32_t)x & 0xffffffu;
        return k >= key0 && k <= key1 && id >= id0 && id <= id1 && x >= cut;
      };
      if (key0 == key1 && !by_index) {
        by_index = true;
        bits = 24;
      }
      const int d = bits < 11 ? bits : 11;
      bits -= d;
      for (int i = t; i < kFBins; i += kFThreads) sh.hist[i] = 0;
      if (t == 0) sh.n = 0;
      __syncthreads();
      for (int i = t; i < n; i += kFThreads) {
        const u64 x = sh.word[i];
        if (left(x)) {
          const uint32_t y = by_index ? ((uint32_t)x & 0xffffffu) - id0 : (uint32_t)(x >> 32) - key0;
          atomicAdd(&sh.hist[y >> bits], value(x));
        }
      }
      __syncthreads();
      const uint32_t at = (uint32_t)crossing(sh.hist, sh.b, want, above);
      if (by_index) {
        id0 += at << bits;
        id1 = min(id1, id0 + ((1u << bits) - 1));
      } else {
        key0 += at << bits;
        key1 = min(key1, key0 + ((1u << bits) - 1));
      }
      u64* few = reinterpret_cast<u64*>(sh.part);
      for (int i = t; i < n; i += kFThreads)
        if (left(sh.word[i])) {
          const int slot = atomicAdd(&sh.n, 1);
          if (slot < kWave) few[slot] = sh.word[i];
        }
      __syncthreads();
      const int m = sh.n;
      if (m <= kWave) {  // each against all: the word whose running sum reaches `want`
        const u64 mine = lane < m ? few[lane] : 0, own = lane < m ? value(mine) : 0;
        u64 sum = above;
        for (int j = 0; j < m; ++j) {
          const u64 other = few[j];
          sum += other >= mine ? value(other) : 0;
        }
        const u64 hit = __ballot(lane < m && sum >= want && sum - own < want);
        cut = hit ? few[__builtin_ctzll(hit)] : max(cut, (u64)k0 << 32);
        __syncthreads();
        break;
      }
      __syncthreads();
    }
    if (stage == 0 && st.p < 1.0) {
      u64 m = 0;
      for (int i = t; i < n; i += kFThreads)
        if (in_bin(sh.word[i])) m += mass_of((uint32_t)(sh.word[i] >> 32));
      Z = sh.mass[b + 1] + (double)block_sum(m, sh.b) * sh.scale[b];
    }
  }

  // the parts' kept masses
  const int cols = a.parts <= kMaxParts / 16 ? 16 : 1;  // places that a part's words are added to
  if (cut_bin >= 0)
    for (int i = t; i < n; i += kFThreads)
      if (in_bin(sh.word[i]))
        atomicAdd(&sh.listed[~(uint32_t)sh.word[i] / (uint32_t)kPartLen * cols + (t & (cols - 1))],
                  mass_of((uint32_t)(sh.word[i] >> 32)));
  __syncthreads();
  for (int p = w; p < a.parts; p += kFWaves) {
    const u64* from = body + (long long)p * kBody + lane;
    const int b0 = lane - (hi - sh.hi[p]);
    double v = 0.0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int b = b0 + k * kWave;  // the row's bin
      const u64 m = p < kFWaves ? early.held[k] : from[k * kWave];
      v += b > cut_bin && (uint32_t)b < (uint32_t)kBins ? (double)m * sh.scale[b] : 0.0;
    }
    v = wave_sum64(v);
    if (cut_bin >= 0)  // as integers: which place a word was added to differs from run to run
      v += (double)wave_sum64(lane < cols ? sh.listed[p * cols + lane] : (u64)0) * sh.scale[cut_bin];
    if (lane == 0) sh.part[p] = v;
  }
  __syncthreads();
  if (w == 0) {  // the part that holds the draw
    double total = 0.0;
    for (int p0 = 0; p0 < a.parts; p0 += kWave) {
      const double v = p0 + lane < a.parts ? sh.part[p0 + lane] : 0.0;
      total += wave_sum64(v);
    }
    const double target = st.u * total;
    double before = 0.0, start = 0.0;
    int owner = 0;
    for (int p0 = 0; p0 < a.parts; p0 += kWave) {
      const double v = p0 + lane < a.parts ? sh.part[p0 + lane] : 0.0;
      const double incl = wave_scan64(v);
      const u64 has = __ballot(v > 0.0), hit = __ballot(v > 0.0 && before + incl >= target);
      if (has) {  // the first that reaches it, or the last with any mass
        const int l = hit ? (int)__builtin_ctzll(hit) : 63 - (int)__builtin_clzll(has);
        owner = p0 + l;
        start = before + __shfl(incl - v, l, kWave);
      }
      if (hit) break;
      before += wave_last64(incl);
    }
    if (lane == 0) {
      sh.bin = owner;
      sh.b.wmass[0] = target - start;
    }
  }
  if (t == 0) {
    sh.b.pick = 0x7fffffff;
    sh.n = -1;
  }
  __syncthreads();
  // the walk, in the bins' weights too: of equal logits the sums are then exact in every step
  const double target = sh.b.wmass[0];
  constexpr int kWalk = kPartLen / kFThreads;
  const int i0 = sh.bin * kPartLen + t * kWalk;
  float x[kWalk];
#pragma unroll
  for (int e = 0; e < kWalk; ++e) x[e] = lg[min(i0 + e, a.vocab - 1)];
  // kept: logits above the cut's, and those equal to it up to its index (no cut: all above -inf)
  const float low = fmaxf((float)(((double)lo - 2.0) / c), -FLT_MAX);  // as in the scan
  const float cut_l = cut ? logit_of(min((uint32_t)(cut >> 32), kKeyInf)) : -INFINITY;
  const int cut_i = (int)~(uint32_t)cut;  // cuts between keys have 0 there, so every index is up to it
  double wt[kWalk], m = 0.0;
#pragma unroll
  for (int e = 0; e < kWalk; ++e) {
    const int i = i0 + e;
    wt[e] = 0.0;
    if (i < a.vocab && x[e] >= low && (x[e] > cut_l || (x[e] == cut_l && (uint32_t)i <= (uint32_t)cut_i))) {
      double r;
      const int b = bin_of((double)x[e], c, r) - lo;
      if (b >= 0)
        wt[e] = (bin_weight.raised(r) - 4503599627370496.0) * sh.scale[min(b, kBins - 1)];
    }
    m += wt[e];
  }
  const double incl = wave_scan64(m);
  __syncthreads();
  if (lane == kWave - 1) sh.b.wmass[w] = incl;
  __syncthreads();
  double run = incl - m;
  for (int i = 0; i < w; ++i) run += sh.b.wmass[i];
  // the first kept logit whose running sum reaches the draw, or (by rounding) the last kept one; a
  // thread whose last sum falls short of the draw by rounding leaves it to the next
  int pick = 0x7fffffff, last = -1;
#pragma unroll
  for (int e = 0; e < kWalk; ++e) {
    run += wt[e];
    if (wt[e] > 0.0) last = i0 + e;
    if (wt[e] > 0.0 && run >= target) pick = min(pick, i0 + e);
  }
  pick = wave_extreme<false>(pick, 0x7fffffff);
  last = wave_extreme<true>(last, -1);
  if (lane == 0) {
    atomicMin(&sh.b.pick, pick);
    atomicMax(&sh.n, last);
  }
  __syncthreads();
  if (t == 0) a.out[row] = sh.b.pick != 0x7fffffff ? sh.b.pick : sh.n;
  return true;
}

__global__ void __launch_bounds__(kFThreads) filter_pick_kernel(FilterArgs a) {
  __shared__ PickLds sh;
  const int row = blockIdx.x;
  const int t = threadIdx.x, lane = t & (kWave - 1), w = t >> 6;
  const Settings st = settings_of(a, row);
  const bool listed = !st.greedy && a.parts > 0 && st.k > 0 && st.k <= kSmallK;
  const bool binned = !st.greedy && a.parts > 0 && !listed && !st.extreme;
  // what the parts left, asked for at once
  const u64* body = a.body + (long long)row * a.parts * kBody;
  Early early{};
  if (listed) {
    if (w < a.parts) early.held[0] = body[(long long)w * kBody + lane];
  } else if (binned) {
    const RowBins& in = a.bins[row];
    early.n = in.n;
    if (w < a.parts)
#pragma unroll
      for (int k = 0; k < kHeld; ++k) early.held[k] = body[(long long)w * kBody + k * kWave + lane];
    if (t <= kBins) {
      early.mass = in.mass[t];
      early.count = in.count[t];
    }
    if (t < kBins) early.hist = in.hist[t];
    if (t < 6) early.edge = in.edge[t];
    if (t < 3) early.bin = in.bin[t];
  }
  uint32_t mk = 0;
  int mi = 0x7fffffff;
  if (a.parts > 0) {
    if (t < a.parts) {
      const int4 h = a.head[(long long)row * a.parts + t];
      mk = (uint32_t)h.x;
      mi = h.y;
      sh.len[t] = h.z;
      sh.hi[t] = h.w;
    }
  } else {
    const float* lg = a.logits + (long long)row * a.stride;
    for (int i = t; i < a.vocab; i += kFThreads) {
      const uint32_t k = key_of(lg[i]);
      if (k > mk) {
        mk = k;
        mi = i;
      }
    }
  }
  {  // the largest key and its lowest index
    const uint32_t wk = wave_max_key(mk);
    const int wi = wave_extreme<false>(mk == wk ? mi : 0x7fffffff, 0x7fffffff);
    if (lane == 0) sh.b.wsum[w] = rank_word(wk, wi);
    __syncthreads();
    u64 best = sh.b.wsum[0];
#pragma unroll
    for (int i = 1; i < kFWaves; ++i) best = max(best, sh.b.wsum[i]);
    __syncthreads();
    mk = (uint32_t)(best >> 32);
    mi = (int)~(uint32_t)best;
  }
  if (st.greedy || mk <= kKeyMasked) {
    if (t == 0) a.out[row] = mk <= kKeyMasked ? -1 : mi;
    return;
  }
  bool done = false;
  if (listed)
    done = pick_listed(a, row, st, mk, early, sh);
  else if (binned && mk < kKeyInf)
    done = pick_binned(a, row, st, mk, early, sh);
  if (done) return;
  __syncthreads();
  // the token in one lane, -1 in the others
  const int token = select_row(a.logits + (long long)row * a.stride, a.vocab, mk, st.it, st.k, st.p,
                               st.min_w, st.u);
  if (token >= 0) a.out[row] = token;
}

// Parts in all from which the merge is a launch of its own.  Done by every part's gather it costs no
// launch but is repeated.  Nuclei of 0.95 take, so and apart (us): 1 row 30.7 and 32.2, 16 rows 38.4
// and 40.1, 64 rows 54.7 and 51.1, 256 rows 117 and 94.
constexpr int kMergeApart = 512;

int scan_parts(int vocab) {
  const int parts = (vocab + kPartLen - 1) / kPartLen;
  return parts <= kMaxParts ? parts : 0;
}
bool sizes_fit(int n_rows, int vocab) {  // ... also the threads of a launch into 32 bits
  return n_rows >= 0 && n_rows <= kMaxRows && vocab >= 1 && vocab <= (1 << 24) &&
         (int64_t)(n_rows + kXcds) * scan_parts(vocab) * kSThreads <= 0xffffffffll;
}

}  // namespace
}  // namespace fqa

using namespace fqa;

extern "C" int64_t fqa_sample_filtered_workspace_bytes(int32_t n_rows, int32_t vocab) {
  if (!sizes_fit(n_rows, vocab)) return FQA_EINVAL;
  const int64_t parts = scan_parts(vocab);
  return n_rows * (parts * (16 + 8 * kBody) + (parts ? (int64_t)sizeof(RowBins) : 0));
}

extern "C" int fqa_sample_filtered(const float* logits, int32_t n_rows, int32_t vocab,
                                   int64_t row_stride, const float* inv_temp,
                                   const int32_t* top_k, const float* top_p, const float* min_p,
                                   const float* u, int32_t* out, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  if (!sizes_fit(n_rows, vocab) || row_stride < vocab) return FQA_EINVAL;
  if (n_rows == 0) return FQA_OK;
  const int64_t need = fqa_sample_filtered_workspace_bytes(n_rows, vocab);
  if (!logits || !inv_temp || !top_k || !top_p || !min_p || !u || !out ||
      (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))))
    return FQA_EINVAL;
  const int parts = scan_parts(vocab);
  FilterArgs a{logits, vocab, row_stride, inv_temp, top_k, top_p, min_p, u, out, n_rows, parts,
               (int4*)workspace,
               (u64*)((char*)workspace + (int64_t)n_rows * parts * 16),
               (RowBins*)((char*)workspace + (int64_t)n_rows * parts * (16 + 8 * kBody))};
  const hipStream_t st = (hipStream_t)stream;
  if (parts > 0) {
    const dim3 grid((unsigned)((n_rows + kXcds - 1) / kXcds * kXcds * parts)), block(kSThreads);
    hipLaunchKernelGGL(filter_scan_kernel, grid, block, 0, st, a);
    if (hipGetLastError() != hipSuccess) return FQA_ELAUNCH;
    if ((int64_t)n_rows * parts >= kMergeApart) {
      hipLaunchKernelGGL(filter_merge_kernel, dim3((unsigned)n_rows), block, 0, st, a);
      if (hipGetLastError() != hipSuccess) return FQA_ELAUNCH;
      hipLaunchKernelGGL(filter_gather_kernel<false>, grid, block, 0, st, a);
    } else {
      hipLaunchKernelGGL(filter_gather_kernel<true>, grid, block, 0, st, a);
    }
    if (hipGetLastError() != hipSuccess) return FQA_ELAUNCH;
  }
  hipLaunchKernelGGL(filter_pick_kernel, dim3((unsigned)n_rows), dim3(kFThreads), 0, st, a);
  return hipGetLastError() == hipSuccess ? FQA_OK : FQA_ELAUNCH;
}
