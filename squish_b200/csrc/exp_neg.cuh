// exp_neg.cuh — fp64 exponential of the sampler's weights.
#pragma once

namespace sq {

// e^x for x <= 0: x = k ln 2 + r, |r| <= ln 2 / 2 (ln 2 in two parts, Cody and Waite), the Taylor
// polynomial of degree 13 (remainder 4e-18) evaluated in pairs (Estrin), times 2^k; 0 from x = -707 down
// (below 2^-1019). Within 4 ulp (2.1 at most over 350000 arguments). The chain is 11 operations where one after another it would be 20: the
// exponentials are waited for, not many.
__device__ __forceinline__ double exp_neg(double x) {
  const double kx = fma(x, 1.4426950408889634, 6755399441055744.0);  // 1.5 * 2^52: rounds to an integer
  const double k = kx - 6755399441055744.0;
  const double r = fma(k, -1.9082149292705877e-10, fma(k, -6.93147180369123816490e-01, x));
  const double r2 = r * r, r4 = r2 * r2, r8 = r4 * r4;
  const double p01 = 1.0 + r, p23 = fma(r, 1.0 / 6, 0.5), p45 = fma(r, 1.0 / 120, 1.0 / 24),
               p67 = fma(r, 1.0 / 5040, 1.0 / 720), p89 = fma(r, 1.0 / 362880, 1.0 / 40320),
               pab = fma(r, 1.0 / 39916800, 1.0 / 3628800), pcd = fma(r, 1.0 / 6227020800.0, 1.0 / 479001600);
  const double q0 = fma(p23, r2, p01), q1 = fma(p67, r2, p45), q2 = fma(pab, r2, p89);
  const double e = fma(fma(pcd, r4, q2), r8, fma(q1, r4, q0));
  if (!(x > -707.0)) return 0.0;
  return e * __hiloint2double((1023 + __double2loint(kx)) << 20, 0);
}

}  // namespace sq
