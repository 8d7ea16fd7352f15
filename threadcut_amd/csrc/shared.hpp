// The partial pass of shared-prefix decode (shared.hip): the prefix for all
// sequences, and each sequence's own tokens, in one launch.
#pragma once

#include "tc_common.hpp"

namespace tc {

struct PartialArgs;  // decode_tile.hpp

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
  int blocks;               // blocks of columns (set by launch_shared)
  float c;                  // |scale| log2(e), > 0
  uint32_t sign;            // 0x80008000 for a negative scale: flips the queries
};

// Splits of the prefix (a.splits) and of the sequences' own tokens for a call on `cus` compute units: prefix tiles of 16
// tokens, own_tokens of the longest sequence.
void shared_splits(int batch, int heads, int group, int64_t prefix_tiles, int64_t own_tokens, bool ragged, int cus,
                   int* prefix, int* own);

// Joins the splits of a call with many rows (sequences x query heads): out_b from o_part and lse_part.
struct JoinArgs {
  const float* o_part;      // [B, H, S, G, D]
  const float* lse_part;    // [B, H, S, G]
  uint16_t* out;
  int64_t so_b, so_h, so_g;
  int heads, group, batch, splits;
};
hipError_t launch_join(const JoinArgs& a, int dtype, hipStream_t stream);

// The launch: a for the prefix; o (its splits from a.splits on) for the own tokens, whose splits may be 0.
hipError_t launch_shared(const PrefixArgs& a, const PartialArgs& o, int dtype, hipStream_t stream);

}  // namespace tc
