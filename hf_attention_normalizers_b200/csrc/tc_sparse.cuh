// Lower bounds of the sparse normalizers' threshold from the largest scores
// seen so far, shared by the tensor-core scans.
#pragma once

#include "common.cuh"
#include "tc_common.cuh"

namespace hfan {
namespace tc {

// A raw-score gate at or a few ulps below z / zs (izs = 1 / zs): a gate that
// is too low only admits a few dead entries, one that is too high could drop
// a candidate.  One multiply instead of a division on the scan's hot path.
__device__ __forceinline__ float raw_gate(float z, float izs) {
  const float r = z * izs;
  return r - fabsf(r) * 0x1p-20f;
}

// Lower bound of tau from the KT largest chunk maxima zz[0] >= ... >= zz[KT-1]
// (z units, -inf when missing): any k distinct scores whose closed-form
// threshold t_k lies at or below the smallest of them give f(t_k) >= 1,
// hence t_k <= tau.  k = 1 is the zmax - 1 bound.
template <int NORM, int KT>
__device__ __forceinline__ float top_bound(const float (&zz)[KT]) {
  // The sizes k whose closed-form threshold t_k stays at or below the k-th
  // value form a prefix, and the largest one gives the set's threshold; the
  // test needs no root or division (1/k is a constant of the unrolled loop),
  // so a single closed form is evaluated at the end.
  const float z1 = zz[0];
  float s1 = 0.f, s2 = 0.f;
  float bt = 0.f, bmean = 0.f, bd = 0.f;  // the largest valid k's closed form (sparsemax) or its parts
  bool any = false;
#pragma unroll
  for (int k = 1; k <= KT; ++k) {
    const float y = zz[k - 1] - z1;
    s1 += y;
    s2 += y * y;
    const float inv = 1.f / float(k);
    bool valid;
    float tk = 0.f, mean = 0.f, d = 0.f;
    if (NORM == HFAN_SPARSEMAX) {
      tk = (s1 - 1.f) * inv;
      valid = tk <= y;
    } else {
      mean = s1 * inv;
      d = (1.f - (s2 - s1 * mean)) * inv;  // t_k = mean - sqrt(d)
      const float g = mean - y;             // t_k <= y  <=>  g <= sqrt(d)
      valid = g <= 0.f || (d >= 0.f && g * g <= d);
    }
    valid = valid && zz[k - 1] > kNegInf;
    if (valid) {
      any = true;
      bt = tk;
      bmean = mean;
      bd = d;
    }
  }
  if (!any) return z1 - 1.f;
  const float t = NORM == HFAN_SPARSEMAX ? bt : bmean - sqrtf(fmaxf(bd, 0.f));
  return fmaxf(z1 - 1.f, z1 + t);
}

// a >= b after the call
__device__ __forceinline__ void cswap(float& a, float& b) {
  const float hi = fmaxf(a, b);
  b = fminf(a, b);
  a = hi;
}

// t[0..3] (descending) becomes the four largest of t and the unsorted c[0..3]:
// c is sorted by a five-comparator network, the two sorted lists are folded
// into the bitonic top four (max of t[i] and c[3 - i]), and two compare
// levels sort it.  Depth 6 instead of the 16 of one insertion after another.
__device__ __forceinline__ void top4_merge(float (&t)[4], const float (&c)[4]) {
  float a = c[0], b = c[1], x = c[2], y = c[3];
  cswap(a, b);
  cswap(x, y);
  cswap(a, x);
  cswap(b, y);
  cswap(b, x);  // a >= b >= x >= y
  float r0 = fmaxf(t[0], y), r1 = fmaxf(t[1], x), r2 = fmaxf(t[2], b), r3 = fmaxf(t[3], a);
  cswap(r0, r2);
  cswap(r1, r3);
  cswap(r0, r1);
  cswap(r2, r3);
  t[0] = r0;
  t[1] = r1;
  t[2] = r2;
  t[3] = r3;
}

}  // namespace tc
}  // namespace hfan
