// rank_bins.hpp — ranks of beams' continuations in a histogram.
#pragma once

#include <cfloat>
#include <cmath>

namespace mitok {

// Ranks in BB_BINS equal steps from the lowest to the highest of a range, a monotone
// whole number of each: 0 and above within the range, -1 or 0 below it.  A rank is
// any double above -inf: a masked logit of the type's lowest value gives one of
// -1.8e308, a long hypothesis under a negative length power one of -1e40.  The steps
// are of halves, whose difference stays within the doubles, and never 0, so that no
// infinite rank becomes a NaN; a range too narrow for steps has all its ranks in bin 0.
constexpr int BB_BINS = 256;
struct RankBins {
  double lo, inv;  // half the lowest rank, steps of a unit
  __host__ __device__ __forceinline__ RankBins(double low, double high) : lo(0.5 * fmin(low, DBL_MAX)) {
    const double f = BB_BINS / (0.5 * fmin(high, DBL_MAX) - lo);
    inv = f < INFINITY ? f : 1.0;
  }
  __host__ __device__ __forceinline__ int of(double rank) const {
    return (int)fmin(fmax(fma(0.5, rank, -lo) * inv, -1.0), (double)(BB_BINS - 1));
  }
};

}  // namespace mitok
