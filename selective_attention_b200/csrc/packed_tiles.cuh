// packed_tiles.cuh - which query tile of which packed sequence a CTA works on, found on the GPU
// from cu_seqlens.
#pragma once

#include "common.cuh"

namespace ssdb200 {
namespace {

struct PackedTile {
  int seq;   // sequence, or -1 for rows past the last sequence
  int q0;    // the tile's first position in its sequence
  int n;     // the sequence's length
  int tok0;  // the tile's first token
  int rows;  // tokens of the tile; 0: nothing to do
};

// Tiles of all sequences, and of the rows past the last one, that any cu_seqlens over T tokens can have.
inline long long packed_tile_bound(long long T, long long R, int tile) { return T / tile + R + 1; }

// Called by one whole warp. Tiles are ranked by their position in their sequence, the last positions
// first (a tile at position t has t + 1 key tiles, so the longest start first), sequences in order
// within one position; the tile of rank `rank` is found by a binary search over the position,
// each step one sum over the sequences (32 at a time). Offsets are clamped to [0, T], so
// that no cu_seqlens can lead outside the tensors.
__device__ __forceinline__ void find_packed_tile(const int* __restrict__ cu, int R, int T, int rank, int tile,
                                                 PackedTile* out) {
  const int lane = threadIdx.x & 31;
  auto span = [&](int r, int& lo, int& n) {
    lo = min(max(cu[r], 0), T);
    n = max(min(cu[r + 1], T) - lo, 0);
  };
  auto tiles_of = [&](int r) {
    int lo, n;
    span(r, lo, n);
    return (n + tile - 1) / tile;
  };
  // tiles at positions >= t
  auto from = [&](int t) {
    int c = 0;
    for (int r = lane; r < R; r += 32) c += max(tiles_of(r) - t, 0);
    return __reduce_add_sync(0xffffffffu, c);
  };
  int most = 0;
  for (int r = lane; r < R; r += 32) most = max(most, tiles_of(r));
  most = __reduce_max_sync(0xffffffffu, most);
  const int total = from(0);
  PackedTile t{-1, 0, 0, 0, 0};
  if (rank >= total) {
    const int end = min(max(R > 0 ? cu[R] : 0, 0), T);
    const long long first = (long long)end + (long long)(rank - total) * tile;
    t.tok0 = (int)min(first, (long long)T);
    t.rows = min(T - t.tok0, tile);
  } else {
    int lo = 0, hi = most;  // from(lo) > rank >= from(hi)
    int at_hi = 0;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1, c = from(mid);
      if (c > rank) {
        lo = mid;
      } else {
        hi = mid;
        at_hi = c;
      }
    }
    int left = rank - at_hi;  // of the sequences with more than lo tiles, the left-th
    for (int r0 = 0; r0 < R; r0 += 32) {
      const int r = r0 + lane;
      const unsigned has = __ballot_sync(0xffffffffu, r < R && tiles_of(r < R ? r : 0) > lo);
      const int c = __popc(has);
      if (left < c) {
        const int rr = r0 + (int)__fns(has, 0, left + 1);
        int first, n;
        span(rr, first, n);
        t.seq = rr;
        t.q0 = lo * tile;
        t.n = n;
        t.tok0 = first + t.q0;
        t.rows = min(tile, n - t.q0);
        break;
      }
      left -= c;
    }
  }
  if (lane == 0) *out = t;
}

}  // namespace
}  // namespace ssdb200
