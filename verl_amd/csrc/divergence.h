// A term of the divergence of a softmax q from a teacher's tokens, shared by the row kernels and the head.
//   forward KL  sum p (t - log q)                                  c = -p
//   reverse KL  sum q (log q - t)                                  c = q (log q - t + 1)
//   JSD         b sum p (t - log w) + (1 - b) sum q (log q - log w)   c = (1 - b) q (log q - log w),  w = b p + (1 - b) q
// with the teacher's log-probability t, p = exp(t), b = beta and c the derivative with respect to log q.
#pragma once
#include "common.h"

namespace vamd {
namespace {

struct Term {
  float loss, slope;  // of a teacher's token, and its derivative with respect to log q
};
// Differences of logarithms are formed from d = log q - t, so that nothing cancels where the two agree.
__device__ __forceinline__ Term divergence_term(int kind, float beta, float t, float lq) {
  const float p = expf(t), q = expf(lq), d = lq - t;
  if (kind == VAMD_DIV_FORWARD_KL) return Term{p > 0.f ? -p * d : 0.f, -p};
  if (kind == VAMD_DIV_REVERSE_KL) {
    const float x = q == 0.f ? 0.f : q * d;
    return Term{x, x + q};
  }
  // t - log w and log q - log w
  float a, b;
  if (d > 0.f) {
    b = -log1pf(beta * expm1f(-d));
    a = b - d;
  } else {
    a = -log1pf((1.f - beta) * expm1f(d));
    b = d + a;
  }
  const float x = q == 0.f ? 0.f : (1.f - beta) * q * b;
  return Term{(p == 0.f ? 0.f : beta * p * a) + x, x};
}

inline int check_divergence(const char* what, int k, int divergence, float beta) {
  VAMD_REQUIRE(k >= 1 && k <= VAMD_TOPK_MAX, "%s: k is %d, of 1 to %d", what, k, VAMD_TOPK_MAX);
  VAMD_REQUIRE(divergence >= VAMD_DIV_FORWARD_KL && divergence <= VAMD_DIV_JSD, "%s: unknown divergence %d", what, divergence);
  VAMD_REQUIRE(divergence != VAMD_DIV_JSD || (beta > 0.f && beta < 1.f), "%s: beta must lie between 0 and 1", what);
  return VAMD_OK;
}

}  // namespace
}  // namespace vamd
