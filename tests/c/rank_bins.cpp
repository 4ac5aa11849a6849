/* The bins of a rank (rank_bins.hpp) on the CPU: reads "low high rank" lines, as
 * hexadecimal doubles, and prints each rank's bin. */
#define __host__
#define __device__
#define __forceinline__ inline
#include <cstdio>
#include <cstdlib>

#include "rank_bins.hpp"

int main() {
  char low[64], high[64], rank[64];
  while (scanf("%63s %63s %63s", low, high, rank) == 3)
    printf("%d\n", mitok::RankBins(strtod(low, nullptr), strtod(high, nullptr)).of(strtod(rank, nullptr)));
}
