// What fqa_sample_filtered's scan computes of its bins (flashqwen_amd/csrc/fqa_sample_bins.h), on the
// host, for tests/test_sample_bins.py.
#include "../../flashqwen_amd/csrc/fqa_sample_bins.h"

#include <cmath>
#include <cstdio>
#include <cstring>

using namespace fqa;

// Every place that a part's bins may have, for logits of either sign and any inv_temp: the slots of its
// bins are those of the histogram, each bin's its own.
static int slots() {
  long n = 0;
  for (const double sign : {1.0, -1.0})
    for (double top = 1.0; top < kMaxPartPlace; top *= 1.37) {
      const double c = kEightLog2e * 1e4, place = sign * top;  // the largest logit, in places
      double r;
      const int hi = bin_of(place / c, c, r), lo = hi - (kBins - 1);
      for (int col = 0; col < kBinCols; ++col) {
        const uint32_t base = slot_base(lo, col);
        for (int b = 0; b < kBins; ++b, ++n) {
          const int bin = bin_of((double)(lo + b) / c, c, r);
          if (bin < lo || bin > hi) continue;  // (rounded past the end)
          if (bin_slot(bin, base) != (uint32_t)((bin - lo) * kBinCols + col) ||
              bin_slot(bin, base) >= (uint32_t)(kBins * kBinCols)) {
            std::printf("place %.17g: bin %d has slot %u\n", place, bin, bin_slot(bin, base));
            return 1;
          }
        }
      }
    }
  std::printf("%ld slots\n", n);
  return 0;
}

// The largest error of a weight, relative to its value, over the distances from a bin's middle.
static int weights() {
  long double worst = 0;
  const int n = 1 << 21;
  for (int i = -n; i <= n; ++i) {
    const double r = 0.5 * i / n;
    const long double got = bin_weight_raised(kBinWeight, r) - kRaise;
    worst = std::fmax(worst, std::fabs(got / (kBinUnit * std::exp2((long double)r / 8)) - 1));
  }
  std::printf("%.6Lg\n", worst);
  return 0;
}

int main(int argc, char** argv) {
  if (argc == 2 && !std::strcmp(argv[1], "slots")) return slots();
  if (argc == 2 && !std::strcmp(argv[1], "weights")) return weights();
  return 2;
}
