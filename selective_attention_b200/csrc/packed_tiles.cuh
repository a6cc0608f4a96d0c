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

// Finds tiles for one whole warp, of 2^SHIFT positions each. Tiles are ranked by their position in their
// sequence, the last positions first (a tile at position t has t + 1 key tiles, so the longest
// start first), sequences in order within one position; the tile of a rank is found by a binary
// search over the position, each step one sum over the sequences. The tile counts of the first
// 128 sequences stay in registers. Offsets are clamped to [0, T], so that no cu_seqlens can lead
// outside the tensors.
template <int SHIFT>
struct PackedFinder {
  static constexpr int kHeld = 4;  // sequences 32 i + lane
  const int* cu;
  int R, T, held[kHeld], most, total;

  __device__ __forceinline__ void span(int r, int& lo, int& n) const {
    lo = min(max(cu[r], 0), T);
    n = max(min(cu[r + 1], T) - lo, 0);
  }
  __device__ __forceinline__ int load_tiles(int r) const {
    if (r >= R) return 0;
    int lo, n;
    span(r, lo, n);
    return (int)(((unsigned)n + (1u << SHIFT) - 1u) >> SHIFT);
  }
  // tiles at positions >= t
  __device__ __forceinline__ int from(int t) const {
    const int lane = threadIdx.x & 31;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) c += max(held[i] - t, 0);
    for (int r = 32 * kHeld + lane; r < R; r += 32) c += max(load_tiles(r) - t, 0);
    return __reduce_add_sync(0xffffffffu, c);
  }
  __device__ __forceinline__ void init(const int* cu_, int R_, int T_) {
    cu = cu_, R = R_, T = T_;
    const int lane = threadIdx.x & 31;
    most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) most = max(most, held[i] = load_tiles(32 * i + lane));
    for (int r = 32 * kHeld + lane; r < R; r += 32) most = max(most, load_tiles(r));
    most = __reduce_max_sync(0xffffffffu, most);
    total = from(0);
  }
  // The `left`-th of sequences 32 i .. 32 i + 31 with more than `pos` tiles, if there are so many.
  __device__ __forceinline__ bool pick(int i, int tiles, int pos, int& left, PackedTile& t) const {
    const unsigned has = __ballot_sync(0xffffffffu, tiles > pos);
    const int c = __popc(has);
    if (left >= c) {
      left -= c;
      return false;
    }
    const int r = 32 * i + (int)__fns(has, 0, left + 1);
    int first, n;
    span(r, first, n);
    t.seq = r;
    t.q0 = pos << SHIFT;
    t.n = n;
    t.tok0 = first + t.q0;
    t.rows = min(1 << SHIFT, n - t.q0);
    return true;
  }
  __device__ __forceinline__ PackedTile find(int rank) const {
    const int lane = threadIdx.x & 31;
    PackedTile t{-1, 0, 0, 0, 0};
    if (rank >= total) {
      const int end = min(max(R > 0 ? cu[R] : 0, 0), T);
      const long long first = (long long)end + ((long long)(rank - total) << SHIFT);
      t.tok0 = (int)min(first, (long long)T);
      t.rows = min(T - t.tok0, 1 << SHIFT);
      return t;
    }
    int lo = 0, hi = most, at_hi = 0;  // from(lo) > rank >= from(hi) = at_hi
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1, c = from(mid);
      if (c > rank) {
        lo = mid;
      } else {
        hi = mid;
        at_hi = c;
      }
    }
    int left = rank - at_hi;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (pick(i, held[i], lo, left, t)) return t;
    for (int i = kHeld; 32 * i < R; ++i)
      if (pick(i, load_tiles(32 * i + lane), lo, left, t)) return t;
    return t;
  }
};

}  // namespace
}  // namespace ssdb200
