// The prefix pass of shared-prefix decode (shared.hip), which decode.hip's
// entry points launch beside the partial kernel of each sequence's own tokens.
#pragma once

#include "tc_common.hpp"

namespace tc {

struct PrefixArgs {
  const uint16_t* q;        // [B, H, G, D]
  const uint16_t* k;        // prefix [H, n, D], or the K pool
  const uint16_t* v;
  float* o_part;            // [B, H, part_splits, G, D]: this pass writes splits [0, splits)
  float* lse_part;          // [B, H, part_splits, G]
  int64_t sq_b, sq_h, sq_g;
  int64_t sk_h, sk_t, sv_h, sv_t;
  int64_t sk_p, sv_p;       // paged: page strides
  const int32_t* tile_tab;  // paged: the prefix's tiles {page, first slot, rows, -}, or null
  int32_t tiles;            // 16-token tiles of the prefix
  int32_t n;                // tokens (contiguous)
  int32_t pages, page_tokens;
  int heads, group, batch;
  int splits, part_splits;
  float c;                  // |scale| log2(e), > 0
  uint32_t sign;            // 0x80008000 for a negative scale: flips the queries
};

// Splits of the prefix pass for `tiles` tiles, and the launch itself.
int prefix_splits(int batch, int heads, int group, int64_t tiles, int cus);
hipError_t launch_prefix(const PrefixArgs& a, int dtype, hipStream_t stream);

}  // namespace tc
