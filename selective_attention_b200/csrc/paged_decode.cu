// paged_decode.cu - attention of one query token for each request over the paged 8-bit cache
// (paged.cu): SelectiveMHA.step's attention (modules/selective_attention.py:399-404) with
// grouped heads, requests of different lengths and keys and values held as codes.
//   s_j = scale * q . (code_j * k_scale) + (j < n - 1 ? log_gate_j : 0),  out = softmax(s) . v
// A key whose log-gate is -inf drops out, whatever its codes hold; so does one whose table entry
// is not a page of the cache. A request of length 0 gets zeros.
//
// The step reads every code once and computes 4 operations a code for each of the g = Hq / Hk
// query heads that share it, so it should run at the memory's rate. What decides that is the
// work between a code's arrival and its product; this layout keeps it low:
//   - one warp of a CTA fetches (TMA, 16 tokens of K or V a box, a ring of stages of 64 tokens), four
//     warps compute, 16 tokens of a stage each (32 of 128 for head_dim up to 64); the fetching warp runs
//     ahead from one request to the next, so that memory stays busy where the others join their results;
//   - both products are m16n8k16 tensor-core products with the codes as the 16-row operand A and
//     up to 8 query heads as the 8 columns: S^T = K Q^T has tokens as rows, O^T = V^T P^T has
//     dimensions as rows, so heads pad to 8 and not to 16 (tcgen05 would pad them to 16 columns too,
//     but takes its 128-row operand from shared memory, where the codes would have to be written
//     back as 16-bit values first). The codes become fp16 in registers, exactly
//     (int8: a byte permute builds 1024 + code + 128, one subtraction; e4m3: a conversion);
//   - within a product the contraction index and the rows of A may come in any order that both
//     operands share. A lane takes 16 consecutive bytes of a token's K for four k-steps, and 16
//     consecutive dimensions of V for eight row pairs: shared memory is read with 16-byte loads,
//     K never needs a transposition and V needs one byte permute for each four codes;
//   - the page scales stay outside the products: k_scale multiplies the fp32 scores; v_scale enters
//     P. What P must not exceed is therefore 2^s v_scale, whose largest power of two a warp follows for each
//     head apart from that of 2^s: a page whose values are large takes no bits from the others where
//     its keys have no weight or are dropped.
// Measured: 64 requests of 1 to 8192 tokens (int8, 32 heads on 8 of 128, 547 MB) 106 us a step, 5.1 TB/s, of which 6.2
// in the steady state; one of 131071 tokens (e4m3, 32 heads on 4, 134 MB) 34 us; 24 of 1 to 4097 tokens (fp32
// queries, 24 heads of 64 with gates, 165 MB) 51 us, there bound by instructions: one query head fills an
// eighth of each product.
// Roundings: fp32 accumulation, softmax statistics and O. P is rounded to fp16 (2^-11 of itself),
// offset by 2^7 so that 2^s v_scale down to 2^-21 of the head's largest keeps all bits. q enters
// as fp16 after scaling its row by a power of two, which is exact for fp16 and for bf16 (8 bits)
// down to 2^-29 of the row's largest element; an fp32 q and its P are split into two fp16 parts (22 bits).
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "sm100.cuh"
#include "tmap.cuh"

namespace ssdb200 {
namespace {

using namespace sm100;

constexpr int kDecWarps = 4;                        // computing warps
constexpr int kDecThreads = (kDecWarps + 1) * 32;   // and one that fetches
constexpr int kMinTiles = 8;                        // 16-token tiles that a CTA's share has at least
constexpr int kEachTiles = 32;                      // see decode_launch
constexpr int kStart = 8;                           // a row group's start and join, in tiles' time (see below)
constexpr unsigned int kSiteDecLoad = 0x401, kSiteDecUse = 0x402;
constexpr float kDecLog2e = 1.4426950408889634f;
constexpr float kGrow = 8.0f;      // log2: a head's maxima are followed when one grows by more
constexpr float kOffset = 7.0f;    // log2: P = 2^(s - mv + 7) * v_scale <= 2^15
constexpr float kNone = -3e38f;    // a maximum before the first key (finite: 2^(kNone - kNone) is 1, of nothing)

__device__ __forceinline__ float dec_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The smaller one; NaN if either is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// The exponent of the power of two above |x| (finite, whatever x is).
__device__ __forceinline__ float above(float x) { return (float)((int)((__float_as_uint(x) >> 23) & 0xffu) - 126); }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four codes -> two fp16 pairs (codes 0, 1) and (2, 3), exactly.
template <typename C>
__device__ __forceinline__ void expand4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (std::is_same<C, Int8>::value) {
    const uint32_t x = w ^ 0x80808080u;  // code + 128
    const uint32_t m0 = __byte_perm(x, 0x64646464u, 0x4140), m1 = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    const __half2 h0 = __hsub2(*reinterpret_cast<const __half2*>(&m0), off);
    const __half2 h1 = __hsub2(*reinterpret_cast<const __half2*>(&m1), off);
    lo = *reinterpret_cast<const uint32_t*>(&h0);
    hi = *reinterpret_cast<const uint32_t*>(&h1);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// Where 16-byte chunk `ch` of token row `row` lies in a 16-token tile of K or V (bytes): rows of up
// to 128 bytes, swizzled by the TMA; head_dim 256 is two tiles of 128 columns.
template <int D> __device__ __forceinline__ int tile_at(int row, int ch) {
  if constexpr (D >= 128) return (ch >> 3) * 2048 + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
  if constexpr (D == 64) return row * 64 + ((ch ^ ((row >> 1) & 3)) << 4);
  return row * 32 + ((ch ^ ((row >> 2) & 1)) << 4);
}

// 16-token tiles that a warp takes in one step: two where a tile's work is short next to what a step costs
// anyway (24 requests of up to 4097 tokens, 24 heads of 64: 53 us instead of 59 with cold caches; four stages
// at three CTAs an SM instead of two at four: 55).
template <int D, int NG> constexpr int dec_unroll() { return D <= 64 && NG == 1 ? 2 : 1; }
template <int D, int NG> constexpr int dec_stage_tiles() { return kDecWarps * dec_unroll<D, NG>(); }
template <int D, int NG> constexpr int dec_stages() {
  return D == 256 ? 2 : (D == 128 ? 3 : (D == 64 && NG == 1 ? 2 : 4));
}
template <int D, int NG> constexpr int dec_stage_bytes() { return dec_stage_tiles<D, NG>() * 32 * D; }  // K, V tiles
constexpr int kInfoFloats = 24;                                                  // 16 gates, k_scale, v_scale, live
// Results of two warps on their way to two others: m, l and O of a lane.
template <int D, int NG> constexpr int dec_xchg_words() { return NG * (D / 16 * 4 + 4); }
template <int D, int NG> constexpr size_t dec_smem() {
  return 1024 + (size_t)dec_stages<D, NG>() * (dec_stage_bytes<D, NG>() + dec_stage_tiles<D, NG>() * kInfoFloats * 4) +
         2 * 32 * dec_xchg_words<D, NG>() * 4 + 128;
}

// Adds to the bytes that a barrier's phase waits for, without arriving on it.
__device__ __forceinline__ void mbar_announce(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

struct DecodeArgs {
  const void* q;
  const float *ks, *vs, *gc;
  const int *table, *lengths;
  void* out;
  float *part, *part_ml;  // (2 parts of a CTA, 8 NG heads) partial O and (m, l)
  long long pages;
  int R, W, Hq, Hk, g, ngrp, page_shift, ctas;
  int each;  // a CTA for each row group, nothing to join
  float scale;
};

__device__ __forceinline__ int dec_length(const DecodeArgs& a, int r) {
  return (int)min((long long)max(a.lengths[r], 0), (long long)a.W << a.page_shift);
}
__device__ __forceinline__ int dec_tiles(const DecodeArgs& a, int r) { return (dec_length(a, r) + 15) >> 4; }

// All requests' tiles, request by request and, within one, row group by row group (a row group:
// the up to 8 NG query heads that share one reading of a key head), are one line; CTA i works on
// [i * per, (i + 1) * per) of it. So every CTA has the same share whatever the lengths are, and one
// long request is spread over all of them. Each row group begins with kStart places without a tile,
// for the time that its start and its join take: counted by tiles alone, the CTAs of short requests
// took up to 1.75 times the median (24 requests of 1 to 4097 tokens, 24 heads of 64: 79 us of 45). A row
// group that crosses from one CTA into the next leaves a part in each, which
// paged_decode_join_kernel joins in their order.
__device__ __forceinline__ int dec_places(int tiles) { return tiles > 0 ? tiles + kStart : 0; }

__device__ __forceinline__ long long dec_share(long long units, int ctas) {
  const long long per = (units + ctas - 1) / ctas;
  return per < kMinTiles ? kMinTiles : per;
}

// Called by a whole CTA of N threads: the places of one row group of every request (returned), and those
// before request `upto` (before). sums: 2 * N / 32 words of shared memory.
template <int N>
__device__ __forceinline__ long long dec_count(const DecodeArgs& a, int upto, long long& before, long long* sums) {
  const int tid = threadIdx.x;
  long long all = 0, pre = 0;
  for (int r = tid; r < a.R; r += N) {
    const int t = dec_places(dec_tiles(a, r));
    all += t;
    if (r < upto) pre += t;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, off);
    pre += __shfl_xor_sync(0xffffffffu, pre, off);
  }
  if ((tid & 31) == 0) sums[tid >> 5] = all, sums[N / 32 + (tid >> 5)] = pre;
  __syncthreads();
  all = pre = 0;
#pragma unroll
  for (int w = 0; w < N / 32; ++w) all += sums[w], pre += sums[N / 32 + w];
  before = pre;
  return all;
}

// (kept in step with dec_ctas, which sizes the workspace)
template <int D, int NG> constexpr int dec_ctas_per_sm() {
  return D == 256 || NG == 2 ? 2 : (D == 128 ? 3 : 4);
}

// A run of tiles of one row group (none, where the share ends within the places before the first tile).
struct DecSegment {
  int r, n, group, first, last;
  int places;          // of the line that it takes
  bool whole, begun;   // all of the row group; begun by an earlier CTA
};
// The segment at `at` of the line, r and r_at (the request and its first place on the line) moved on to it.
__device__ __forceinline__ DecSegment dec_segment(const DecodeArgs& a, int groups, long long at, long long end, int& r,
                                                  long long& r_at) {
  DecSegment s;
  int places;
  for (;;) {
    s.n = dec_length(a, r);
    places = dec_places((s.n + 15) >> 4);
    const long long all = (long long)places * groups;
    if (at < r_at + all) break;
    r_at += all;
    ++r;
  }
  s.r = r;
  const long long in = at - r_at;
  s.group = (int)(in / places);
  const int from = (int)(in - (long long)s.group * places), to = (int)min((long long)places, from + (end - at));
  s.places = to - from;
  s.first = max(from - kStart, 0);
  s.last = max(to - kStart, 0);
  s.begun = from > kStart;
  s.whole = !s.begun && to == places;
  return s;
}

template <typename T, typename C, int D, int NG>
__global__ void __launch_bounds__(kDecThreads, dec_ctas_per_sm<D, NG>())
    paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const DecodeArgs a) {
  constexpr bool SPLIT = std::is_same<T, float>::value;
  constexpr int NST = dec_stages<D, NG>(), STAGE = dec_stage_bytes<D, NG>(), TILE = 16 * D;
  constexpr int U = dec_unroll<D, NG>(), GT = dec_stage_tiles<D, NG>();  // tiles of a warp's step and of a stage
  constexpr int KW = D / 16;                 // K words of a lane and row = k-steps
  constexpr int MT = D / 16;                 // 16-row tiles of O^T
  constexpr int VWORDS = D / 32;             // V words of a lane and token
  extern __shared__ uint8_t dsm_raw[];
  __shared__ long long s_sums[2 * (kDecWarps + 1)];
  __shared__ int s_req;
  __shared__ long long s_at;
  uint8_t* ring = align1024_shared(dsm_raw);
  float* infos = reinterpret_cast<float*>(ring + NST * STAGE);
  float* xchg = infos + NST * GT * kInfoFloats;
  uint64_t* bars = reinterpret_cast<uint64_t*>(xchg + 2 * 32 * dec_xchg_words<D, NG>());
  auto full = [&](int s) { return smem_u32(&bars[s]); };
  auto empty = [&](int s) { return smem_u32(&bars[NST + s]); };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, lr = lane >> 2, lc = lane & 3;
  T* out = reinterpret_cast<T*>(a.out);
  asm volatile("griddepcontrol.launch_dependents;");  // the join may be put in place now (it waits for this grid)
  if (tid == 0) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
#pragma unroll
    for (int i = 0; i < NST; ++i) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), kDecWarps);
    }
    fence_mbar_init();
  }
  const int groups = a.Hk * a.ngrp;
  long long begin, end;
  if (a.each) {  // one row group: the line is the request's
    if (tid == 0) s_req = blockIdx.x / groups, s_at = 0;
    const int places = dec_places(dec_tiles(a, blockIdx.x / groups));
    begin = (long long)(blockIdx.x % groups) * places;
    end = begin + places;
  } else {
    long long unused;
    const long long units = dec_count<kDecThreads>(a, 0, unused, s_sums) * groups;
    const long long per = dec_share(units, (int)gridDim.x);
    begin = blockIdx.x * per;
    end = min(begin + per, units);
  }
  for (int r = blockIdx.x; r < a.R; r += gridDim.x) {  // requests without tokens
    if (dec_length(a, r) == 0)
      for (int i = tid; i < a.Hq * D; i += kDecThreads) out[(long long)r * a.Hq * D + i] = from_f32<T>(0.f);
  }
  if (begin >= end) return;
  // the request that holds tile `begin` of the line, by a scan of one warp
  if (warp == 0 && !a.each) {
    long long base = 0;
    for (int r0 = 0; r0 < a.R; r0 += 32) {
      const int t = r0 + lane < a.R ? dec_places(dec_tiles(a, r0 + lane)) : 0;
      long long incl = (long long)t * groups;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += x;
      }
      const long long hi = base + incl, lo = hi - (long long)t * groups;
      if (lo <= begin && begin < hi) s_req = r0 + lane, s_at = lo;
      base = __shfl_sync(0xffffffffu, hi, 31);
      if (base > begin) break;
    }
  }
  __syncthreads();
  int r = s_req;
  long long r_at = s_at;
  int step = 0;  // stages used so far
  const int tiles_page = a.page_shift - 4;  // log2 of a page's tiles

  if (warp == kDecWarps) {
    // ---------------------------------------------------------------- fetch
    // Lanes take the GT tiles of a stage in turn: the first GT lanes their K, then V, gates, scales, and
    // the second column halves of head_dim 256. Page numbers and scales come 32 tiles at a time,
    // one batch ahead.
    bool dead = false;
    for (long long at = begin; at < end;) {
      const DecSegment sg = dec_segment(a, groups, at, end, r, r_at);
      at += sg.places;
      const int hk = sg.group / a.ngrp;
      const int* row = a.table + (long long)sg.r * a.W;
      auto page_of = [&](int t) { return t < sg.last ? row[t >> tiles_page] : -1; };
      auto valid = [&](int id) { return id >= 0 && id < a.pages; };
      int id = page_of(sg.first + lane), id_next = -1;
      float ksc = 0.f, vsc = 0.f, ksc_next = 0.f, vsc_next = 0.f;
      if (valid(id)) ksc = a.ks[(long long)id * a.Hk + hk], vsc = a.vs[(long long)id * a.Hk + hk];
      for (int t = sg.first, i = 0; t < sg.last; t += GT, ++i, ++step) {
        const int in = i & (32 / GT - 1);  // step of the batch
        if (in == 0) {
          if (i > 0) id = id_next, ksc = ksc_next, vsc = vsc_next;
          id_next = page_of(t + 32 + lane);
        } else if (in == 16 / GT) {
          ksc_next = vsc_next = 0.f;
          if (valid(id_next))
            ksc_next = a.ks[(long long)id_next * a.Hk + hk], vsc_next = a.vs[(long long)id_next * a.Hk + hk];
        }
        const int st = step % NST, w = lane & (GT - 1), mt = t + w;
        if (step >= NST && !dead) dead = !mbar_wait_sleep(empty(st), ((step / NST) - 1) & 1, kSiteDecLoad);
        dead = __any_sync(0xffffffffu, dead);
        const int my = __shfl_sync(0xffffffffu, id, GT * in + w);
        const bool live = mt < sg.last && valid(my) && !dead;
        const long long ph = live ? (long long)my * a.Hk + hk : 0;
        const int row0 = (mt & ((1 << tiles_page) - 1)) << 4;
        float* info = infos + (st * GT + w) * kInfoFloats;
        const int role = lane / GT;
        const int n_live = __popc(__ballot_sync(0xffffffffu, live) & ((1u << GT) - 1u));
        // the bytes are announced and asked for; the stage is handed over below, with the scales
        if (lane == 0) mbar_announce(full(st), (uint32_t)(n_live * (2 * TILE + (a.gc ? 64 : 0))));
        __syncwarp();
        if (live) {
          const uint32_t kd = smem_u32(ring + st * STAGE + w * TILE), vd = kd + GT * TILE;
          if (role == 0) tma_load_3d(kd, &tm_k, 0, row0, (int)ph, full(st));
          if (role == 1) tma_load_3d(vd, &tm_v, 0, row0, (int)ph, full(st));
          if (role == 2 && a.gc) bulk_load(smem_u32(info), a.gc + (ph << a.page_shift) + row0, 64, full(st));
          if (D == 256 && role == 4) tma_load_3d(kd + 2048, &tm_k, 128, row0, (int)ph, full(st));
          if (D == 256 && role == 5) tma_load_3d(vd + 2048, &tm_v, 128, row0, (int)ph, full(st));
        }
        const float mk = __shfl_sync(0xffffffffu, ksc, GT * in + w), mv = __shfl_sync(0xffffffffu, vsc, GT * in + w);
        if (role == 3) info[16] = mk, info[17] = mv, info[18] = live ? 1.f : 0.f;
        __syncwarp();
        if (lane == 0) mbar_arrive(full(st));
      }
    }
    // no copy may be in flight when the CTA exits
    if (lane == 0)
      for (int d = 1; d <= NST && d <= step; ++d)
        mbar_wait(full((step - d) % NST), ((step - d) / NST) & 1, kSiteDecLoad);
    return;
  }

  // ------------------------------------------------------------------ compute
  // A wait that ran out sets the error flag; the warp then waits for no more stages but takes every step,
  // so that the barriers below always have their warps.
  bool dead = false;
  for (long long at = begin; at < end;) {
    const DecSegment sg = dec_segment(a, groups, at, end, r, r_at);
    at += sg.places;
    if (sg.first >= sg.last) continue;
    const int hk = sg.group / a.ngrp, hg = sg.group - hk * a.ngrp;
    const int h0 = hk * a.g + hg * 8 * NG, nh = min(a.g - hg * 8 * NG, 8 * NG);
    const int n = sg.n;

    // q as the B operand of S^T: lane (lr, lc) holds head lr, dimensions of its k slots
    uint32_t qb[NG][KW][2], ql[SPLIT ? NG : 1][SPLIT ? KW : 1][2];
    float qf[NG][2];  // per score column 2 lc, 2 lc + 1: scale * log2(e) / the row's power of two
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      const int h = 8 * x + lr;
      const T* qp = reinterpret_cast<const T*>(a.q) + ((long long)sg.r * a.Hq + h0 + h) * D;
      float v[KW][4], m = 0.f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const int d = D == 32 ? 8 * lc + 4 * k : 64 * (k >> 2) + 16 * lc + 4 * (k & 3);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[k][e] = h < nh ? to_f32<T>(qp[d + e]) : 0.f;
          m = fmaxf(m, fabsf(v[k][e]));
        }
      }
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // the largest element goes to [2^14, 2^15); fp16 queries need no scaling
      float up = 1.f, down = 1.f;
      if (!std::is_same<T, __half>::value && m > 0.f && m < INFINITY) {
        const int e = min(max(14 - ilogbf(m), -126), 126);
        up = ldexpf(1.f, e);
        down = ldexpf(1.f, -e);
      }
#pragma unroll
      for (int k = 0; k < KW; ++k) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float x0 = v[k][2 * b] * up, x1 = v[k][2 * b + 1] * up;
          qb[x][k][b] = half2_bits(x0, x1);
          if constexpr (SPLIT) {
            const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&qb[x][k][b]));
            ql[x][k][b] = half2_bits(x0 - hi.x, x1 - hi.y);
          }
        }
      }
      const float f = a.scale * kDecLog2e * down;
      qf[x][0] = __shfl_sync(0xffffffffu, f, (2 * lc) * 4);
      qf[x][1] = __shfl_sync(0xffffffffu, f, (2 * lc + 1) * 4);
    }

    // By head, in log2: m, the largest s, l in units of 2^m; mv, the largest s + log2(v_scale) (rounded up), O in units
    // of 2^mv.
    float o[NG][MT][4], m[NG][2], l[NG][2], mv[NG][2];
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      m[x][0] = m[x][1] = mv[x][0] = mv[x][1] = kNone;
      l[x][0] = l[x][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[x][i][0] = o[x][i][1] = o[x][i][2] = o[x][i][3] = 0.f;
    }
    for (int t = sg.first; t < sg.last; t += GT, ++step) {
      const int st = step % NST;
      if (!dead) dead = !__all_sync(0xffffffffu, mbar_wait_sleep(full(st), (step / NST) & 1, kSiteDecUse));
      const int mine = warp * U;  // the warp's first tile of the stage
      if (t + mine < sg.last) {  // (a tile past the last holds nothing that counts: its `live` is 0)
      const uint8_t* kt = ring + st * STAGE + mine * TILE;
      const uint8_t* vt = kt + GT * TILE;
      const float* info = infos + (st * GT + mine) * kInfoFloats;
      // ---- S^T = K Q^T
      float s[U][NG][4], s2[U][NG][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int x = 0; x < NG; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][x][e] = s2[u][x][e] = 0.f;
        const uint8_t* ku = kt + u * TILE;
        uint32_t kw[2][KW];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if constexpr (D == 32) {
            const uint2 w = *reinterpret_cast<const uint2*>(ku + tile_at<D>(lr + 8 * b, lc >> 1) + (lc & 1) * 8);
            kw[b][0] = w.x, kw[b][1] = w.y;
          } else {
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const uint4 w = *reinterpret_cast<const uint4*>(ku + tile_at<D>(lr + 8 * b, lc + 4 * j));
              kw[b][4 * j] = w.x, kw[b][4 * j + 1] = w.y, kw[b][4 * j + 2] = w.z, kw[b][4 * j + 3] = w.w;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < KW; ++k) {
          uint32_t a0, a1, a2, a3;
          expand4<C>(kw[0][k], a0, a2);
          expand4<C>(kw[1][k], a1, a3);
#pragma unroll
          for (int x = 0; x < NG; ++x) {
            mma16816(k & 1 ? s2[u][x] : s[u][x], a0, a1, a2, a3, qb[x][k][0], qb[x][k][1]);
            if constexpr (SPLIT) mma16816(k & 1 ? s[u][x] : s2[u][x], a0, a1, a2, a3, ql[x][k][0], ql[x][k][1]);
          }
        }
      }
      // ---- scores in log2 units
      bool in0[U], in1[U], grow = false;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* iu = info + u * kInfoFloats;
        const int t0 = (t + mine + u) * 16 + lr, t1 = t0 + 8;
        const float ksc = iu[16];
        const bool live = iu[18] != 0.f;
        in0[u] = live && t0 < n, in1[u] = live && t1 < n;
        float g0 = 0.f, g1 = 0.f;
        if (a.gc) {
          g0 = t0 < n - 1 ? iu[lr] : 0.f;
          g1 = t1 < n - 1 ? iu[lr + 8] : 0.f;
          in0[u] = in0[u] && g0 != -INFINITY;
          in1[u] = in1[u] && g1 != -INFINITY;
          g0 *= kDecLog2e, g1 *= kDecLog2e;
        }
        const float lv = above(iu[17]);
#pragma unroll
        for (int x = 0; x < NG; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = fmaf(s[u][x][e] + s2[u][x][e], qf[x][e & 1] * ksc, e < 2 ? g0 : g1);
            s[u][x][e] = (e < 2 ? in0[u] : in1[u]) ? y : -INFINITY;
            grow |= s[u][x][e] > fminf(m[x][e & 1], mv[x][e & 1] - lv) + kGrow;
          }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int x = 0; x < NG; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float t = fmaxf(s[0][x][e], s[0][x][e + 2]), y = t + above(info[17]);
#pragma unroll
            for (int u = 1; u < U; ++u) {
              const float tu = fmaxf(s[u][x][e], s[u][x][e + 2]);
              t = fmaxf(t, tu);
              y = fmaxf(y, tu + above(info[u * kInfoFloats + 17]));
            }
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, off));
              y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, off));
            }
            t = fmaxf(t, m[x][e]);
            y = fmaxf(y, mv[x][e]);
            l[x][e] *= dec_ex2(m[x][e] - t);
            const float f = dec_ex2(mv[x][e] - y);
            m[x][e] = t;
            mv[x][e] = y;
#pragma unroll
            for (int i = 0; i < MT; ++i) o[x][i][e] *= f, o[x][i][e + 2] *= f;
          }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint8_t* vu = vt + u * TILE;
        // ---- P, as the B operand of O^T (heads as columns, tokens as the contraction). The scale of a tile
        // without a key that counts is nothing's (and may be an infinity or NaN); where r is past
        // the range, P is next to nothing.
        const unsigned b0 = __ballot_sync(0xffffffffu, in0[u]), b1 = __ballot_sync(0xffffffffu, in1[u]);
        const float vs = (b0 | b1) != 0u ? info[u * kInfoFloats + 17] : 0.f;
        uint32_t pb[NG][2], pl[SPLIT ? NG : 1][2];
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          const float r0 = min_nan(vs * dec_ex2(m[x][0] - mv[x][0]), 3e38f);
          const float r1 = min_nan(vs * dec_ex2(m[x][1] - mv[x][1]), 3e38f);
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = dec_ex2(s[u][x][e] - (m[x][e & 1] - kOffset));
          l[x][0] += p[0] + p[2];
          l[x][1] += p[1] + p[3];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float p0 = p[2 * b] * r0, p1 = p[2 * b + 1] * r1;
            const uint32_t w = half2_bits(p0, p1);
            pb[x][b] = transpose8x8(w);
            if constexpr (SPLIT) {
              const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&w));
              pl[x][b] = transpose8x8(half2_bits(p0 - hi.x, p1 - hi.y));
            }
          }
        }
        // ---- O^T += V^T P^T
        uint32_t vw[4][VWORDS];  // tokens 2 lc, 2 lc + 1, 2 lc + 8, 2 lc + 9
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int row = 2 * lc + (b & 1) + (b >> 1) * 8;
          if constexpr (D == 32) {
            vw[b][0] = *reinterpret_cast<const uint32_t*>(vu + tile_at<D>(row, lr >> 2) + (lr & 3) * 4);
          } else if constexpr (D == 64) {
            const uint2 w = *reinterpret_cast<const uint2*>(vu + tile_at<D>(row, lr >> 1) + (lr & 1) * 8);
            vw[b][0] = w.x, vw[b][1] = w.y;
          } else {
#pragma unroll
            for (int j = 0; j < D / 128; ++j) {
              const uint4 w = *reinterpret_cast<const uint4*>(vu + tile_at<D>(row, lr + 8 * j));
              vw[b][4 * j] = w.x, vw[b][4 * j + 1] = w.y, vw[b][4 * j + 2] = w.z, vw[b][4 * j + 3] = w.w;
            }
          }
        }
        if constexpr (std::is_same<C, E4M3>::value) {
          // a NaN code of a token that does not count must not meet its zero weight
          if ((b0 & b1) != 0xffffffffu) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const bool in = ((b < 2 ? b0 : b1) >> (4 * (2 * lc + (b & 1)))) & 1u;
#pragma unroll
              for (int j = 0; j < VWORDS; ++j) vw[b][j] = in ? vw[b][j] : 0u;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < VWORDS; ++j) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362 : 0x5140;
            uint32_t a0, a1, a2, a3;
            expand4<C>(__byte_perm(vw[0][j], vw[1][j], sel), a0, a1);
            expand4<C>(__byte_perm(vw[2][j], vw[3][j], sel), a2, a3);
#pragma unroll
            for (int x = 0; x < NG; ++x) {
              mma16816(o[x][2 * j + half], a0, a1, a2, a3, pb[x][0], pb[x][1]);
              if constexpr (SPLIT) mma16816(o[x][2 * j + half], a0, a1, a2, a3, pl[x][0], pl[x][1]);
            }
          }
        }
      }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(st));
    }

    // ---- join the warps: 2 and 3 hand their results to 0 and 1, then 1 to 0; lanes hold the same places
#pragma unroll
    for (int x = 0; x < NG; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], 4);
        l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], 8);
        l[x][e] += __shfl_xor_sync(0xffffffffu, l[x][e], 16);
        const float f = dec_ex2(mv[x][e] - m[x][e]);
#pragma unroll
        for (int i = 0; i < MT; ++i) o[x][i][e] *= f, o[x][i][e + 2] *= f;
      }
    auto put = [&](float* to) {
      float4* p = reinterpret_cast<float4*>(to) + lane;
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        *p = make_float4(m[x][0], m[x][1], l[x][0], l[x][1]);
        p += 32;
#pragma unroll
        for (int i = 0; i < MT; ++i, p += 32) *p = make_float4(o[x][i][0], o[x][i][1], o[x][i][2], o[x][i][3]);
      }
    };
    auto take = [&](const float* from) {
      const float4* p = reinterpret_cast<const float4*>(from) + lane;
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        const float4 ml = *p;
        p += 32;
        const float n0 = fmaxf(m[x][0], ml.x), n1 = fmaxf(m[x][1], ml.y);
        const float f0 = dec_ex2(m[x][0] - n0), g0 = dec_ex2(ml.x - n0);
        const float f1 = dec_ex2(m[x][1] - n1), g1 = dec_ex2(ml.y - n1);
        m[x][0] = n0, m[x][1] = n1;
        l[x][0] = l[x][0] * f0 + ml.z * g0;  // (a NaN stays one, also times 0)
        l[x][1] = l[x][1] * f1 + ml.w * g1;
#pragma unroll
        for (int i = 0; i < MT; ++i, p += 32) {
          const float4 y = *p;
          o[x][i][0] = o[x][i][0] * f0 + y.x * g0;
          o[x][i][1] = o[x][i][1] * f1 + y.y * g1;
          o[x][i][2] = o[x][i][2] * f0 + y.z * g0;
          o[x][i][3] = o[x][i][3] * f1 + y.w * g1;
        }
      }
    };
    float* x0 = xchg + (warp & 1) * 32 * dec_xchg_words<D, NG>();
    named_bar_sync(1, kDecWarps * 32);  // the last segment's results have been taken
    if (warp >= 2) put(x0);
    named_bar_sync(1, kDecWarps * 32);
    if (warp < 2) {
      take(x0);
      if (warp == 1) put(x0);
      named_bar_sync(2, 64);
      if (warp == 0) {
        take(xchg + 32 * dec_xchg_words<D, NG>());
        const bool whole = sg.whole;
        // parts of a row group: one that an earlier CTA began in place 0, one begun here in place 1
        const long long part = (2ll * blockIdx.x + (sg.begun ? 0 : 1)) * (8 * NG);
#pragma unroll
        for (int x = 0; x < NG; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int h = 8 * x + 2 * lc + e;
            if (h >= nh) continue;
            const float inv = 1.0f / l[x][e];
            constexpr int RUN = D >= 128 ? 8 : MT;  // row pairs of consecutive dimensions
#pragma unroll
            for (int i0 = 0; i0 < MT; i0 += RUN) {
              const int d0 = (i0 ? 128 : 0) + 2 * RUN * lr;
              if (whole) {
                T* op = out + ((long long)sg.r * a.Hq + h0 + h) * D + d0;
#pragma unroll
                for (int i = 0; i < RUN; ++i) {
                  const float y0 = o[x][i0 + i][e] * inv, y1 = o[x][i0 + i][e + 2] * inv;
                  if constexpr (SPLIT) {
                    *reinterpret_cast<float2*>(op + 2 * i) = make_float2(y0, y1);
                  } else {
                    *reinterpret_cast<uint32_t*>(op + 2 * i) = pack2<T>(y0, y1);
                  }
                }
              } else {
                float* op = a.part + (part + h) * D + d0;
#pragma unroll
                for (int i = 0; i < RUN; ++i)
                  *reinterpret_cast<float2*>(op + 2 * i) = make_float2(o[x][i0 + i][e], o[x][i0 + i][e + 2]);
              }
            }
            if (!whole && lr == 0)
              *reinterpret_cast<float2*>(a.part_ml + 2 * (part + h)) = make_float2(m[x][e], l[x][e]);
          }
      }
    }
  }
}

// Joins the parts of the row groups that several CTAs worked on. CTA = (request, query head); a warp
// takes every JW-th part, a lane four dimensions.
// (few rows have many parts each: 16 warps; many rows few: 4, so that all CTAs fit at once)
template <typename T, int D, int NG, int JW>
__global__ void __launch_bounds__(JW * 32) paged_decode_join_kernel(const DecodeArgs a) {
  constexpr int VEC = D >= 128 ? 4 : D / 32, COLS = D / (32 * VEC);  // D = 32: 1 x 1, 64: 2 x 1, 128: 4 x 1, 256: 4 x 2
  __shared__ long long s_sums[2 * JW];
  __shared__ float s_m[JW], s_l[JW];
  __shared__ __align__(16) float s_o[JW][D];
  const int h = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tiles = dec_tiles(a, r);
  const int hk = h / a.g, hg = (h - hk * a.g) / (8 * NG), groups = a.Hk * a.ngrp;
  long long before;
  const long long units = dec_count<JW * 32>(a, r, before, s_sums) * groups;
  const long long per = dec_share(units, a.ctas);
  // the places of the row group's first tile and of the one after its last
  const long long lo = before * groups + (long long)(hk * a.ngrp + hg) * dec_places(tiles) + kStart, hi = lo + tiles;
  const int c0 = (int)(lo / per), c1 = (int)((hi - 1) / per);
  const int hl = h - hk * a.g - hg * 8 * NG;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // every CTA waits: this grid must not end before the first one
  if (tiles == 0 || c0 == c1) return;                 // one CTA had all of it
  float m = -INFINITY, l = 0.f, o[COLS][VEC];
#pragma unroll
  for (int j = 0; j < COLS; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[j][e] = 0.f;
#pragma unroll 4
  for (int c = c0 + warp; c <= c1; c += JW) {
    const long long p = (2ll * c + (c * per > lo ? 0 : 1)) * (8 * NG) + hl;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * p);
    const float mn = fmaxf(m, ml.x);
    const float f = m == -INFINITY ? 0.f : dec_ex2(m - mn), g = ml.x == -INFINITY ? 0.f : dec_ex2(ml.x - mn);
    l = l * f + ml.y * g;
    m = mn;
#pragma unroll
    for (int j = 0; j < COLS; ++j) {
      const float* src = a.part + p * D + j * 128 + lane * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[j][e] = o[j][e] * f + src[e] * g;
    }
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int j = 0; j < COLS; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s_o[warp][j * 128 + lane * VEC + e] = o[j][e];
  __syncthreads();
  for (int d = tid; d < D; d += JW * 32) {
    float mm = -INFINITY, ll = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < JW; ++w) mm = fmaxf(mm, s_m[w]);
#pragma unroll
    for (int w = 0; w < JW; ++w) {
      const float f = s_m[w] == -INFINITY ? 0.f : dec_ex2(s_m[w] - mm);
      ll = fmaf(s_l[w], f, ll);
      acc = fmaf(s_o[w][d], f, acc);
    }
    reinterpret_cast<T*>(a.out)[((long long)r * a.Hq + h) * D + d] = from_f32<T>(acc / ll);
  }
}

// Tensor map over the codes of K or V as (D, page, pages * heads), boxes of 16 tokens.
bool make_map_codes(CUtensorMap* map, const void* base, int D, int page, uint64_t rows) {
  auto enc = tensor_map_encoder();
  if (!enc) return false;
  const int inner = D < 128 ? D : 128;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)page, rows};
  cuuint64_t strides[2] = {(cuuint64_t)D, (cuuint64_t)D * page};
  cuuint32_t box[3] = {(cuuint32_t)inner, 16, 1};
  cuuint32_t es[3] = {1, 1, 1};
  const CUtensorMapSwizzle sw = inner == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                             : (inner == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Query heads of one row group: 16 where more than 8 share a key head (one reading serves twice as
// many; with head_dim 256 the registers hold 8), else 8. With fp32 queries the registers do not quite hold
// them: head_dim 128 with 16 heads spills 220 bytes a thread, head_dim 256 up to 194 (16-bit queries 60 and 24).
// 32 requests of up to 4096 tokens with cold caches, fp32 and bf16 queries: 32 heads on 2 of 128 (36 MB) 37 and 30 us,
// 16 heads on 2 of 256 (73 MB) 42 and 36.
int dec_ng(int g, int D) { return g > 8 && D < 256 ? 2 : 1; }
int dec_ctas(int g, int D) {
  const int per = D == 256 || dec_ng(g, D) == 2 ? 2 : (D == 128 ? 3 : 4);
  return 148 * per;
}

template <typename T, typename C, int D, int NG>
cudaError_t decode_launch(DecodeArgs a, const PagedCache& c, cudaStream_t s) {
  constexpr size_t smem = dec_smem<D, NG>();
  CUtensorMap mk, mv;
  if (!make_map_codes(&mk, c.k, D, c.page, (uint64_t)c.pages * c.nkv) ||
      !make_map_codes(&mv, c.v, D, c.page, (uint64_t)c.pages * c.nkv))
    return cudaErrorInvalidValue;
  static unsigned long long allowed = 0;
  cudaError_t e = allow_smem(paged_decode_kernel<T, C, D, NG>, smem, allowed);
  if (e != cudaSuccess) return e;
  a.ngrp = (a.g + 8 * NG - 1) / (8 * NG);
  // no more CTAs than the table has tiles for
  const long long units = ((((long long)a.W << a.page_shift) + 15) / 16 + kStart) * a.R * a.Hk * a.ngrp;
  const long long want = (units + kMinTiles - 1) / kMinTiles;
  a.ctas = 148 * dec_ctas_per_sm<D, NG>();
  // Few row groups of short tables (up to kEachTiles tiles): a CTA for each, and no second launch. One request
  // of up to 512 tokens takes the same time on the GPU as when it is cut, and the call 14 us instead of 19.
  const long long row_groups = (long long)a.R * a.Hk * a.ngrp;
  a.each = (((long long)a.W << a.page_shift) + 15) / 16 <= kEachTiles && row_groups <= a.ctas;
  if (a.each)
    a.ctas = (int)row_groups;
  else if (want < a.ctas)
    a.ctas = (int)want;
  paged_decode_kernel<T, C, D, NG><<<a.ctas, kDecThreads, smem, s>>>(mk, mv, a);
  if ((e = cudaGetLastError()) != cudaSuccess || a.ctas == 1 || a.each) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)a.Hq, (unsigned)a.R);
  const bool few = (long long)a.R * a.Hq < 148 * 4;
  cfg.blockDim = dim3(few ? 16 * 32 : 4 * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, few ? paged_decode_join_kernel<T, D, NG, 16> : paged_decode_join_kernel<T, D, NG, 4>, a);
}

template <typename T, typename C>
cudaError_t decode_t(const DecodeArgs& a, const PagedCache& c, cudaStream_t s) {
  const int D = c.D;
  const bool wide = dec_ng(a.g, D) == 2;
  switch (D) {
    case 32: return wide ? decode_launch<T, C, 32, 2>(a, c, s) : decode_launch<T, C, 32, 1>(a, c, s);
    case 64: return wide ? decode_launch<T, C, 64, 2>(a, c, s) : decode_launch<T, C, 64, 1>(a, c, s);
    case 128: return wide ? decode_launch<T, C, 128, 2>(a, c, s) : decode_launch<T, C, 128, 1>(a, c, s);
    case 256: return decode_launch<T, C, 256, 1>(a, c, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

size_t paged_decode_workspace(int Hq, int Hk, int D) {
  const int g = Hq / Hk;
  return (size_t)dec_ctas(g, D) * 2 * 8 * dec_ng(g, D) * (D + 2) * sizeof(float);
}

cudaError_t launch_paged_decode(const PagedCache& c, const void* q, const int* table, const int* lengths, void* out,
                                int R, int W, int Hq, float scale, int dtype, void* workspace, cudaStream_t s) {
  DecodeArgs a{};
  a.q = q;
  a.ks = c.ks, a.vs = c.vs, a.gc = c.gate;
  a.table = table, a.lengths = lengths, a.out = out;
  a.pages = c.pages;
  a.R = R, a.W = W, a.Hq = Hq, a.Hk = c.nkv, a.g = Hq / c.nkv, a.page_shift = c.page_shift, a.scale = scale;
  a.part = reinterpret_cast<float*>(workspace);
  a.part_ml = a.part + (size_t)dec_ctas(a.g, c.D) * 2 * 8 * dec_ng(a.g, c.D) * c.D;
  const bool e4m3 = c.code == SSD_CODE_E4M3;
  switch (dtype) {
    case SSD_F32: return e4m3 ? decode_t<float, E4M3>(a, c, s) : decode_t<float, Int8>(a, c, s);
    case SSD_BF16: return e4m3 ? decode_t<__nv_bfloat16, E4M3>(a, c, s) : decode_t<__nv_bfloat16, Int8>(a, c, s);
    case SSD_F16: return e4m3 ? decode_t<__half, E4M3>(a, c, s) : decode_t<__half, Int8>(a, c, s);
  }
  return cudaErrorInvalidValue;
}

SSDB200_DEFINE_ERROR_FETCH(fetch_error_paged)

}  // namespace ssdb200
