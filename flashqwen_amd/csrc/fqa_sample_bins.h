// fqa_sample_bins.h — the bins of fqa_sample_filtered's scan: a weight's bin, its mass in it and its
// place in a part's histogram, apart from the kernels so that a host program can run them too.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fqa {

constexpr int kBins = 384;  // an eighth of an octave each: 48 octaves below the largest weight
constexpr double kEightLog2e = 11.541560327111707;  // 8 log2(e)
constexpr double kRound = 6755399441055744.0;       // 1.5 x 2^52: adding it rounds to an integer
// Places that bins are used for: a row's of its largest logit, and a part's (one below these is none
// that its row has bins for).  They and their differences fit int.
constexpr double kMaxPlace = 536870912.0, kMaxPartPlace = 2 * kMaxPlace;
// Copies of the histogram that a part's lanes add to: fewer of them wait for each other (2, 4 and 8
// are within 1% of one another, at 16 their LDS leaves fewer workgroups to a CU).
constexpr int kBinCols = 4;

// The bin of a logit at place l c, and its distance from the bin's middle; |l c| < 2^31.
__host__ __device__ __forceinline__ int bin_of(double l, double c, double& r, double round = kRound) {
  const double s = __builtin_fma(l, c, round);
  r = __builtin_fma(l, c, round - s);
  return (int)(uint32_t)__builtin_bit_cast(unsigned long long, s);
}

// 2^39 2^(r/8), |r| <= 1/2, to an integer, raised by 2^52 (which rounds it to one, in the low bits): the
// polynomial of degree 5 through the 6 Chebyshev points is within 2^-40.6 of its value, and the rounding
// within 2^-39.9, so a weight is within 2^-39 of its value.
constexpr double kBinUnit = 549755813888.0, kRaise = 4503599627370496.0;  // 2^39, 2^52
constexpr double kBinWeight[6] = {kBinUnit + kRaise,
                                  kBinUnit * 0.08664339756999671,
                                  kBinUnit * 0.0037535391505772045,
                                  kBinUnit * 0.00010840646198027614,
                                  kBinUnit * 2.348396409244877e-06,
                                  kBinUnit * 4.069351772310789e-08};
__host__ __device__ __forceinline__ double bin_weight_raised(const double* c, double r) {
  double p = __builtin_fma(r, c[5], c[4]);
  p = __builtin_fma(r, p, c[3]);
  p = __builtin_fma(r, p, c[2]);
  p = __builtin_fma(r, p, c[1]);
  return __builtin_fma(r, p, c[0]);
}

// The place of bin `bin`, at or above `lo`, in copy `col` of the part's histogram: bin_slot(bin,
// slot_base(lo, col)) = (bin - lo) kBinCols + col.  Places go up to 2^30, so the terms may pass 32
// bits: unsigned, as their sum does not.
__host__ __device__ __forceinline__ uint32_t slot_base(int lo, int col) {
  return (uint32_t)col - (uint32_t)lo * (uint32_t)kBinCols;
}
__host__ __device__ __forceinline__ uint32_t bin_slot(int bin, uint32_t base) {
  return (uint32_t)bin * (uint32_t)kBinCols + base;
}

}  // namespace fqa
