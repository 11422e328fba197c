// The k largest logits of tokens whose logits the head has written out, from the maxima of the groups its epilogue has seen
// (row_topk.hip).
#pragma once
#include "common.h"

namespace vamd {

constexpr int kHeadPickGroups = 12288;  // of a token: 48 KB of LDS

struct HeadPickArgs {
  const float* z;  // [n_tokens][z_ld], unscaled products
  int64_t z_ld, vocab;
  const float* group_max;  // [n_tokens][groups]; group g: the columns 256 (g / 8) + 128 (g / 4 % 2) + 4 (g % 4) + 16 i + 0..3, i < 8
  int groups;
  const float* lse;
  int n_tokens, k;
  float rcp_t;
  float* top;      // [n_tokens][k]
  int64_t* index;  // [n_tokens][k]
};
int launch_head_pick(const HeadPickArgs& a, hipStream_t s);

}  // namespace vamd
