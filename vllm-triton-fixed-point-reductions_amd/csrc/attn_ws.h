// The workspace of a split attention launch (host side).
#pragma once

#include "attn_impl.h"

namespace fxpr {
namespace attn {

inline int64_t align256(int64_t x) { return (x + 255) & ~int64_t(255); }

inline int acc_bytes(int int_bits) { return int_bits == 64 ? 8 : 4; }

// Chunks per row that a block-table row of max_blocks pages can hold.
inline int64_t chunk_slots(int max_blocks, int page_size) {
  return cdiv(cdiv(int64_t(max_blocks) * page_size, TILE), CT);
}

// Split-launch workspace: per (token, head) the chunk range, and per
// (token, head, chunk) the row maximum, the integer denominator and the
// integer weighted V row. Unsplit launches need none.
struct WsLayout {
  int64_t crange = -1, pmax = -1, den = -1, wv = -1, total = 0;
};

// (ws_rows: the query tokens that hold records, AttnArgs' W)
inline WsLayout ws_layout(int64_t ws_rows, int num_heads, int head_dim, int int_bits, bool split, int64_t slots) {
  WsLayout w;
  if (!split) return w;
  const int64_t rows = ws_rows * num_heads;
  w.crange = 0;
  w.total = align256(rows * 8);
  w.pmax = w.total;
  w.total += align256(rows * slots * 4);
  w.den = w.total;
  w.total += align256(rows * slots * acc_bytes(int_bits));
  w.wv = w.total;
  w.total += align256(rows * slots * head_dim * acc_bytes(int_bits));
  return w;
}

}  // namespace attn
}  // namespace fxpr
