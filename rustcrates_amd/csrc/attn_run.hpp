// attn_run.hpp — one wave's running softmax over 16-slot tiles of keys and
// values, for the attention kernels of the serving operators (tree_attention.hip,
// paged_attention.hip).
// D[i][j] of a 16x16 tile sits at lane j + 16 * (i % 4), element i / 4.
#pragma once

#include "common.hpp"

namespace mitok {

// For the query lane % 16: the running maximum and sum, and the output (column
// 16 c + 4 e + lane / 16).
template <int DHP>
struct AttnRun {
  static constexpr int CT = DHP / 16;
  v4d o_re[CT], o_im[CT];
  double m = -INFINITY, l = 0.0;  // l over this lane's slots alone
  __device__ __forceinline__ AttnRun() {
#pragma unroll
    for (int c = 0; c < CT; ++c) o_re[c] = o_im[c] = v4d{0.0, 0.0, 0.0, 0.0};
  }
  // A tile's scores become its weights e^(s - m).  Any m near the largest score
  // serves, so it moves only where a score passes it by 8 (weights up to e^8
  // then), which after the first tiles hardly happens: no maximum across the
  // lanes and no rescaling, which costs as much as 8 MFMAs (double arithmetic
  // and double MFMAs take turns on a SIMD: 4 cycles an operation beside 64).
  // Each query goes by its own scores, so its bits do not depend on the others'.
  __device__ __forceinline__ void soften(v4d& s) {
    rescale(s);
    weigh(s);
  }
  __device__ __forceinline__ void rescale(const v4d& s) {
    const double top = fmax(fmax(s[0], s[1]), fmax(s[2], s[3]));
    if (__ballot(top > m + 8.0)) {
      double x, y;
      pair16_f64(top, x, y);
      pair32_f64(fmax(x, y), x, y);
      const double most = fmax(x, y), mn = most > m + 8.0 ? most : m;
      const double keep = mn == m ? 1.0 : exp(m - mn);
      m = mn;
      l *= keep;
#pragma unroll
      for (int c = 0; c < CT; ++c) o_re[c] *= keep, o_im[c] *= keep;
    }
  }
  __device__ __forceinline__ void weigh(v4d& s) {
    const double base = m == -INFINITY ? 0.0 : m;  // nothing seen yet: every weight e^-inf = 0
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = exp(s[e] - base);
      l += s[e];
    }
  }
  __device__ __forceinline__ void output(const v4d& s, int q, int c, double2 v) {
    o_re[c] = __builtin_amdgcn_mfma_f64_16x16x4f64(v.x, s[q], o_re[c], 0, 0, 0);
    o_im[c] = __builtin_amdgcn_mfma_f64_16x16x4f64(v.y, s[q], o_im[c], 0, 0, 0);
  }
  // Values that are not finite are left out of a tile's products, where 0 times
  // them is NaN in the rows of queries that do not see them, and added here to
  // those that do, slot by slot.  row(k): the values of the tile's slot k, of
  // `slots`; bit q of `vis`: this lane's query sees its slot 4 q + lane / 16.
  template <class Row>
  __device__ __forceinline__ void add_left_out(Row&& row, int dh, int slots, const v4d& s, unsigned vis) {
    const int lane = threadIdx.x & 63, node = lane & 15, kq = lane >> 4;
    for (int k = 0; k < 16 && k < slots; ++k) {
      const int from = node + 16 * (k & 3), q = k >> 2;
      const double pk = __shfl(q == 0 ? s[0] : q == 1 ? s[1] : q == 2 ? s[2] : s[3], from);
      const bool see = (__shfl((int)vis, from) >> q) & 1;
      const double2* V = row(k);
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = 16 * c + 4 * e + kq;
          if (see && col < dh) {
            const double2 v = V[col];
            if (!isfinite(v.x)) o_re[c][e] += pk * v.x;
            if (!isfinite(v.y)) o_im[c][e] += pk * v.y;
          }
        }
    }
  }
};
__device__ __forceinline__ bool attn_finite(double2& v) {  // what is not finite becomes 0
  const bool nx = !isfinite(v.x), ny = !isfinite(v.y);
  if (nx) v.x = 0.0;
  if (ny) v.y = 0.0;
  return !(nx || ny);
}

}  // namespace mitok
