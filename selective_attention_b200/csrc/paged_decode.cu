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
//   - a warp takes 16 tokens at a time through its own ring of cp.async stages in shared memory
//     (no barrier between warps, several KB in flight for each warp);
//   - both products are m16n8k16 tensor-core products with the codes as the 16-row operand A and
//     up to 8 query heads as the 8 columns: S^T = K Q^T has tokens as rows, O^T = V^T P^T has
//     dimensions as rows, so heads pad to 8 and not to 16. The codes become fp16 in registers, exactly
//     (int8: a byte permute builds 1024 + code + 128, one subtraction; e4m3: a conversion);
//   - within a product the contraction index and the rows of A may come in any order that both
//     operands share. A lane takes 16 consecutive bytes of a token's K for four k-steps, and 16
//     consecutive dimensions of V for eight row pairs: shared memory is read with 16-byte loads,
//     K never needs a transposition and V needs one byte permute for each four codes;
//   - the page scales stay outside the products: k_scale multiplies the fp32 scores; v_scale enters
//     P relative to the largest one the warp has met (O is rescaled when that grows).
// Roundings: fp32 accumulation, softmax statistics and O. P is rounded to fp16 (2^-11 of itself),
// offset by 2^7 so that products down to 2^-21 of the row's largest keep all bits. q enters
// as fp16 after scaling its row by a power of two, which is exact for fp16 and for bf16 (8 bits)
// down to 2^-29 of the row's largest element; an fp32 q and its P are split into two fp16 parts (22 bits).
#include <cuda_pipeline_primitives.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"

namespace ssdb200 {
namespace {

constexpr int kDecWarps = 4;
constexpr int kMinTiles = 8;       // 16-token tiles that a split has at least
constexpr float kDecLog2e = 1.4426950408889634f;
constexpr float kGrow = 8.0f;      // log2: O is rescaled when a row's maximum grows by more
constexpr float kOffset = 7.0f;    // log2: P = 2^(s - m + 7) <= 2^15

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

// Where 16-byte chunk `ch` of token row `row` lies in a stage's K and V tile (bytes). The reads of
// one 16-byte phase touch two rows x four chunks (K) and four row pairs x two chunks (V); the
// exchanges below spread either over all banks.
template <int D> __device__ __forceinline__ int k_at(int row, int ch) {
  return row * D + ((D >= 128 ? ch ^ ((row & 1) << 2) : ch) << 4);
}
template <int D> __device__ __forceinline__ int v_at(int row, int ch) {
  return row * D + ((D >= 128 ? ch ^ (((row >> 1) & 3) << 1) : (D == 64 ? ch ^ (((row >> 1) & 1) << 1) : ch)) << 4);
}

template <int D> constexpr int dec_stages() { return D == 256 ? 3 : 4; }
template <int D> constexpr int dec_stage_bytes() { return 32 * D + 128; }  // K, V, 16 gates, k_scale, v_scale
template <int D, int NG> constexpr size_t dec_smem() {
  const size_t ring = (size_t)kDecWarps * dec_stages<D>() * dec_stage_bytes<D>();
  const size_t merge = (size_t)kDecWarps * NG * 8 * (D + 2) * 4;
  return ring > merge ? ring : merge;
}

struct DecodeArgs {
  const void* q;
  const unsigned char *kc, *vc;
  const float *ks, *vs, *gc;
  const int *table, *lengths;
  void* out;
  float *part, *part_ml;  // (request, head, split) partial O and (m, l)
  long long pages;
  int W, Hq, Hk, g, page_shift, splits;
  float scale;
};

// Splits of a request that have work, and their tiles each.
__device__ __forceinline__ int dec_split_tiles(int tiles, int splits) {
  return max((tiles + splits - 1) / splits, kMinTiles);
}
__device__ __forceinline__ int dec_length(const DecodeArgs& a, int r) {
  return (int)min((long long)max(a.lengths[r], 0), (long long)a.W << a.page_shift);
}

// CTA = (split of the request's tokens, key head and group of 8 NG query heads, request).
template <typename T, typename C, int D, int NG>
__global__ void __launch_bounds__(kDecWarps * 32, (NG == 2 || D == 256 || std::is_same<T, float>::value) ? 2 : 3)
    paged_decode_kernel(const DecodeArgs a) {
  constexpr bool SPLIT = std::is_same<T, float>::value;
  constexpr int NST = dec_stages<D>(), STAGE = dec_stage_bytes<D>();
  constexpr int KW = D / 16;                 // K words of a lane and row = k-steps
  constexpr int MT = D / 16;                 // 16-row tiles of O^T
  constexpr int VWORDS = D / 32;             // V words of a lane and token
  constexpr int CPR = D / 16;                // 16-byte chunks of a row
  extern __shared__ __align__(16) unsigned char dsm[];
  const int r = blockIdx.z, split = blockIdx.x;
  const int ngrp = (a.g + 8 * NG - 1) / (8 * NG);
  const int hk = blockIdx.y / ngrp, hg = blockIdx.y - hk * ngrp;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, lr = lane >> 2, lc = lane & 3;
  const int n = dec_length(a, r);
  const int tiles = (n + 15) >> 4, per = dec_split_tiles(tiles, a.splits);
  const int first = split * per, last = min(first + per, tiles);
  const int h0 = hk * a.g + hg * 8 * NG, nh = min(a.g - hg * 8 * NG, 8 * NG);
  T* out = reinterpret_cast<T*>(a.out);
  if (n == 0 && split == 0) {
    for (int i = tid; i < nh * D; i += kDecWarps * 32) out[((long long)r * a.Hq + h0) * D + i] = from_f32<T>(0.f);
  }
  if (first >= last) return;

  // q as the B operand of S^T: lane (lr, lc) holds head lr, dimensions of its k slots
  uint32_t qb[NG][KW][2], ql[SPLIT ? NG : 1][SPLIT ? KW : 1][2];
  float qf[NG][2];  // per score column 2 lc, 2 lc + 1: scale * log2(e) / the row's power of two
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    const int h = 8 * x + lr;
    const T* qp = reinterpret_cast<const T*>(a.q) + ((long long)r * a.Hq + h0 + h) * D;
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

  unsigned char* ring = dsm + warp * NST * STAGE;
  const int mine = (last - first - warp + kDecWarps - 1) / kDecWarps;  // this warp's tiles
  const int tiles_page = a.page_shift - 4;                              // log2 of a page's tiles
  int ids = -1;  // page of tile `lane` of the current 32
  auto issue = [&](int it) {
    if ((it & 31) == 0) {
      const int t = first + warp + (it + lane) * kDecWarps;
      ids = t < last ? a.table[(long long)r * a.W + (t >> tiles_page)] : -1;
    }
    const int id = __shfl_sync(0xffffffffu, ids, it & 31);
    if (it < mine) {
      const int t = first + warp + it * kDecWarps;
      unsigned char* st = ring + (it % NST) * STAGE;
      float* info = reinterpret_cast<float*>(st + 32 * D);
      const bool ok = id >= 0 && id < a.pages;
      const long long ph = ok ? (long long)id * a.Hk + hk : 0;
      const int row0 = (t & ((1 << tiles_page) - 1)) << 4;
      const long long tok = (ph << a.page_shift) + row0;
      const size_t zero = ok ? 0 : 16;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int c = lane + 32 * i, row = c / CPR, ch = c % CPR;
        __pipeline_memcpy_async(st + k_at<D>(row, ch), a.kc + tok * D + c * 16, 16, zero);
        __pipeline_memcpy_async(st + 16 * D + v_at<D>(row, ch), a.vc + tok * D + c * 16, 16, zero);
      }
      if (lane < 4) {
        // without gates the 16 floats are unused
        if (a.gc) __pipeline_memcpy_async(info + 4 * lane, a.gc + tok + 4 * lane, 16, zero);
      } else if (lane == 4) {
        __pipeline_memcpy_async(info + 16, a.ks + ph, 4, ok ? 0 : 4);
      } else if (lane == 5) {
        __pipeline_memcpy_async(info + 17, a.vs + ph, 4, ok ? 0 : 4);
      } else if (lane == 6) {
        info[18] = ok ? 1.f : 0.f;
      }
    }
    __pipeline_commit();
  };

  float o[NG][MT][4], m[NG][2], l[NG][2], unit = 0.f;  // O in units of the v_scale `unit`
#pragma unroll
  for (int x = 0; x < NG; ++x) {
    m[x][0] = m[x][1] = -INFINITY;
    l[x][0] = l[x][1] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[x][i][0] = o[x][i][1] = o[x][i][2] = o[x][i][3] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) issue(i);
  for (int it = 0; it < mine; ++it) {
    __pipeline_wait_prior(NST - 2);
    __syncwarp();
    issue(it + NST - 1);  // into the stage that the whole warp has read in the last step
    const unsigned char* st = ring + (it % NST) * STAGE;
    const float* info = reinterpret_cast<const float*>(st + 32 * D);
    const int t0 = (first + warp + it * kDecWarps) * 16 + lr, t1 = t0 + 8;
    // ---- S^T = K Q^T
    float s[NG][4], s2[NG][4];
#pragma unroll
    for (int x = 0; x < NG; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[x][e] = s2[x][e] = 0.f;
    uint32_t kw[2][KW];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if constexpr (D == 32) {
        const uint2 w = *reinterpret_cast<const uint2*>(st + (lr + 8 * b) * D + lc * 8);
        kw[b][0] = w.x, kw[b][1] = w.y;
      } else {
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          const uint4 w = *reinterpret_cast<const uint4*>(st + k_at<D>(lr + 8 * b, lc + 4 * j));
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
        mma16816(k & 1 ? s2[x] : s[x], a0, a1, a2, a3, qb[x][k][0], qb[x][k][1]);
        if constexpr (SPLIT) mma16816(k & 1 ? s[x] : s2[x], a0, a1, a2, a3, ql[x][k][0], ql[x][k][1]);
      }
    }
    // ---- scores in log2 units
    const float ksc = info[16], vsc = info[17];
    bool in0 = t0 < n, in1 = t1 < n;
    float g0 = 0.f, g1 = 0.f;
    if (a.gc) {
      g0 = t0 < n - 1 ? info[lr] * kDecLog2e : 0.f;
      g1 = t1 < n - 1 ? info[lr + 8] * kDecLog2e : 0.f;
      in0 = in0 && g0 != -INFINITY;
      in1 = in1 && g1 != -INFINITY;
    }
    const bool live = info[18] != 0.f;
    in0 = in0 && live;
    in1 = in1 && live;
    bool grow = false;
#pragma unroll
    for (int x = 0; x < NG; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = fmaf(s[x][e] + s2[x][e], qf[x][e & 1] * ksc, e < 2 ? g0 : g1);
        s[x][e] = (e < 2 ? in0 : in1) ? y : -INFINITY;
        grow |= s[x][e] > m[x][e & 1] + kGrow;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int x = 0; x < NG; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float t = fmaxf(s[x][e], s[x][e + 2]);
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
          const float mn = fmaxf(m[x][e], t);
          const float f = m[x][e] == -INFINITY ? 0.f : dec_ex2(m[x][e] - mn);
          if (mn == m[x][e]) continue;  // (uniform over the lanes of a column: no collective below)
          m[x][e] = mn;
          l[x][e] *= f;
#pragma unroll
          for (int i = 0; i < MT; ++i) o[x][i][e] *= f, o[x][i][e + 2] *= f;
        }
    }
    if (vsc > unit) {
      const float f = unit / vsc;
      unit = vsc;
#pragma unroll
      for (int x = 0; x < NG; ++x)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[x][i][e] *= f;
    }
    const float ratio = unit > 0.f ? __fdividef(vsc, unit) : 0.f;
    // ---- P, as the B operand of O^T (heads as columns, tokens as the contraction)
    uint32_t pb[NG][2], pl[SPLIT ? NG : 1][2];
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      const float m0 = m[x][0] == -INFINITY ? 0.f : m[x][0] - kOffset;
      const float m1 = m[x][1] == -INFINITY ? 0.f : m[x][1] - kOffset;
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = dec_ex2(s[x][e] - (e & 1 ? m1 : m0));
      l[x][0] += p[0] + p[2];
      l[x][1] += p[1] + p[3];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float p0 = p[2 * b] * ratio, p1 = p[2 * b + 1] * ratio;
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
      const unsigned char* vp = st + 16 * D;
      if constexpr (D == 32) {
        vw[b][0] = *reinterpret_cast<const uint32_t*>(vp + row * D + lr * 4);
      } else if constexpr (D == 64) {
        const uint2 w = *reinterpret_cast<const uint2*>(vp + v_at<D>(row, lr >> 1) + (lr & 1) * 8);
        vw[b][0] = w.x, vw[b][1] = w.y;
      } else {
#pragma unroll
        for (int j = 0; j < D / 128; ++j) {
          const uint4 w = *reinterpret_cast<const uint4*>(vp + v_at<D>(row, lr + 8 * j));
          vw[b][4 * j] = w.x, vw[b][4 * j + 1] = w.y, vw[b][4 * j + 2] = w.z, vw[b][4 * j + 3] = w.w;
        }
      }
    }
    if constexpr (std::is_same<C, E4M3>::value) {
      // a NaN code of a token that does not count must not meet its zero weight
      const unsigned b0 = __ballot_sync(0xffffffffu, in0), b1 = __ballot_sync(0xffffffffu, in1);
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
  __pipeline_wait_prior(0);
  __syncthreads();  // the ring becomes the warps' results

  // ---- merge the warps
  float* so = reinterpret_cast<float*>(dsm);                    // [warp][head][D]
  float* sml = so + kDecWarps * NG * 8 * D;                     // [warp][head][2]
#pragma unroll
  for (int x = 0; x < NG; ++x)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float t = l[x][e];
      t += __shfl_xor_sync(0xffffffffu, t, 4);
      t += __shfl_xor_sync(0xffffffffu, t, 8);
      t += __shfl_xor_sync(0xffffffffu, t, 16);
      const int h = warp * NG * 8 + 8 * x + 2 * lc + e;
      if (lr == 0) sml[2 * h] = m[x][e], sml[2 * h + 1] = t;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int d = D == 32 ? 4 * lr + 2 * i : (D == 64 ? 8 * lr + 2 * i : 128 * (i >> 3) + 16 * lr + 2 * (i & 7));
        *reinterpret_cast<float2*>(so + h * D + d) = make_float2(o[x][i][e] * unit, o[x][i][e + 2] * unit);
      }
    }
  __syncthreads();
  const bool whole = per >= tiles;  // this split is all of the request
  for (int i = tid; i < nh * D; i += kDecWarps * 32) {
    const int h = i / D, d = i - h * D;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) mm = fmaxf(mm, sml[2 * (w * NG * 8 + h)]);
    float acc = 0.f, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float mw = sml[2 * (w * NG * 8 + h)];
      const float f = mw == -INFINITY ? 0.f : dec_ex2(mw - mm);
      ll = fmaf(sml[2 * (w * NG * 8 + h) + 1], f, ll);  // (a NaN stays one)
      acc = fmaf(so[(w * NG * 8 + h) * D + d], f, acc);
    }
    const long long row = (long long)r * a.Hq + h0 + h;
    if (whole) {
      out[row * D + d] = from_f32<T>(acc / ll);
    } else {
      a.part[(row * a.splits + split) * D + d] = acc;
      if (d == 0) {
        a.part_ml[2 * (row * a.splits + split)] = mm;
        a.part_ml[2 * (row * a.splits + split) + 1] = ll;
      }
    }
  }
}

// Joins the splits of a request; thread = dimension.
template <typename T>
__global__ void paged_decode_join_kernel(const DecodeArgs a, int D) {
  const int h = blockIdx.x, r = blockIdx.y, d = threadIdx.x;
  const int tiles = (dec_length(a, r) + 15) >> 4, per = dec_split_tiles(tiles, a.splits);
  if (per >= tiles) return;
  const int used = (tiles + per - 1) / per;
  const long long row = (long long)r * a.Hq + h;
  const float* ml = a.part_ml + 2 * row * a.splits;
  const float* p = a.part + row * a.splits * D + d;
  float mm = -INFINITY, ll = 0.f, acc = 0.f;
  for (int s = 0; s < used; ++s) mm = fmaxf(mm, ml[2 * s]);
#pragma unroll 4
  for (int s = 0; s < used; ++s) {
    const float mw = ml[2 * s];
    const float f = mw == -INFINITY ? 0.f : dec_ex2(mw - mm);
    ll = fmaf(ml[2 * s + 1], f, ll);
    acc = fmaf(p[(long long)s * D], f, acc);
  }
  reinterpret_cast<T*>(a.out)[row * D + d] = from_f32<T>(acc / ll);
}

// Splits of each request: enough CTAs to fill the 148 SMs several times over, so that requests of
// different lengths even out.
int dec_splits(int R, int W, int Hk, int ngrp, int page_shift) {
  const long long pairs = (long long)R * Hk * ngrp;
  const long long tiles = ((long long)W << page_shift) / 16;
  long long s = (2048 + pairs - 1) / pairs;
  const long long most = (tiles + kMinTiles - 1) / kMinTiles;
  if (s > most) s = most;
  if (s > 128) s = 128;
  return s < 1 ? 1 : (int)s;
}
int dec_groups(int g, int D) { return g > 8 && D < 256 ? (g + 15) / 16 : (g + 7) / 8; }

template <typename T, typename C, int D, int NG>
cudaError_t decode_launch(const DecodeArgs& a, int R, cudaStream_t s) {
  constexpr size_t smem = dec_smem<D, NG>();
  cudaError_t e = cudaFuncSetAttribute(paged_decode_kernel<T, C, D, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)smem);
  if (e != cudaSuccess) return e;
  const int ngrp = (a.g + 8 * NG - 1) / (8 * NG);
  dim3 grid((unsigned)a.splits, (unsigned)(a.Hk * ngrp), (unsigned)R);
  paged_decode_kernel<T, C, D, NG><<<grid, kDecWarps * 32, smem, s>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess || a.splits == 1) return e;
  paged_decode_join_kernel<T><<<dim3((unsigned)a.Hq, (unsigned)R), D, 0, s>>>(a, D);
  return cudaGetLastError();
}

template <typename T, typename C>
cudaError_t decode_t(const DecodeArgs& a, int R, int D, cudaStream_t s) {
  const bool wide = a.g > 8;
  switch (D) {
    case 32: return wide ? decode_launch<T, C, 32, 2>(a, R, s) : decode_launch<T, C, 32, 1>(a, R, s);
    case 64: return wide ? decode_launch<T, C, 64, 2>(a, R, s) : decode_launch<T, C, 64, 1>(a, R, s);
    case 128: return wide ? decode_launch<T, C, 128, 2>(a, R, s) : decode_launch<T, C, 128, 1>(a, R, s);
    case 256: return decode_launch<T, C, 256, 1>(a, R, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

size_t paged_decode_workspace(int R, int W, int Hq, int Hk, int page_shift, int D) {
  const int splits = dec_splits(R, W, Hk, dec_groups(Hq / Hk, D), page_shift);
  return splits == 1 ? 0 : (size_t)R * Hq * splits * (D + 2) * sizeof(float);
}

cudaError_t launch_paged_decode(const PagedCache& c, const void* q, const int* table, const int* lengths, void* out,
                                int R, int W, int Hq, float scale, int dtype, void* workspace, cudaStream_t s) {
  if (R > 65535) return cudaErrorInvalidValue;
  DecodeArgs a{};
  a.q = q;
  a.kc = c.k, a.vc = c.v, a.ks = c.ks, a.vs = c.vs, a.gc = c.gate;
  a.table = table, a.lengths = lengths, a.out = out;
  a.pages = c.pages;
  a.W = W, a.Hq = Hq, a.Hk = c.nkv, a.g = Hq / c.nkv, a.page_shift = c.page_shift, a.scale = scale;
  a.splits = dec_splits(R, W, c.nkv, dec_groups(a.g, c.D), c.page_shift);
  a.part = reinterpret_cast<float*>(workspace);
  a.part_ml = a.part + (size_t)R * Hq * a.splits * c.D;
  const bool e4m3 = c.code == SSD_CODE_E4M3;
  switch (dtype) {
    case SSD_F32: return e4m3 ? decode_t<float, E4M3>(a, R, c.D, s) : decode_t<float, Int8>(a, R, c.D, s);
    case SSD_BF16:
      return e4m3 ? decode_t<__nv_bfloat16, E4M3>(a, R, c.D, s) : decode_t<__nv_bfloat16, Int8>(a, R, c.D, s);
    case SSD_F16: return e4m3 ? decode_t<__half, E4M3>(a, R, c.D, s) : decode_t<__half, Int8>(a, R, c.D, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace ssdb200
