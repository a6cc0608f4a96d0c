// sattn_packed.cu - selective attention over whole prompts of different lengths, packed one
// after another (cu_seqlens), causal, with grouped heads: the prefill of sattn.cu
// (modules/selective_attention.py:27-144, :270-280) without padding.
//   s_ij = scale * q_i . k_j + (j < i ? log_gate_j : 0), j <= i in i's sequence; out_i = softmax(s_i) . v
// Query head h reads key head h / (Hq / Hk). A key whose log-gate is -inf drops out for every later
// query, whatever it holds, and so does every key that a query does not see: a NaN or an infinity
// there changes nothing. Rows past the last sequence are written as zeros.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "packed_tiles.cuh"
#include "sattn_tiles.cuh"
#include "sm100.cuh"
#include "tmap.cuh"

namespace ssdb200 {
namespace {

// Packed fp32 pairs.
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float lo2(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float hi2(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }

// ===========================================================================
// CUDA-core kernel (fp32, and head_dim 16 or 32): CTA = (query head, 64-query tile of a sequence),
// 64-key tiles of K and V staged in shared memory as fp32; thread (tr, tc) owns rows tr + 16 i
// (i < 4), score columns tc + 16 j, output columns 4 tc + 64 g (g < D / 64). Two products an
// instruction (fp32 pairs). At head_dim 128 V takes K's place once the scores are there, so that two CTAs fit
// an SM. A CTA takes the tile of its rank, so that the tiles with most keys start first (the other way round the
// longest ones ended alone: 564 us instead of 488 in the first case below). Bound by reading shared
// memory, whose pipe is 78 % busy (the FMA units 54 %). 8 prompts of up to 1024 tokens: fp32, 16 heads on 4 of 128,
// 488 us (29 TFLOP/s); bf16, the same heads of 32, 222 us; fp32, 24 heads of 64 with gates, 501 us.
// ===========================================================================
template <int D> constexpr bool simt_share() { return D == 128; }
template <int D> constexpr size_t simt_smem() {
  return (size_t)((simt_share<D>() ? 2 : 3) * kPT * (D + 4) + kPT * (kPT + 4) + kPT) * sizeof(float);
}
template <typename T>
__device__ __forceinline__ void stage64(float* dst, int ld, const T* src, long long stride, int rows, int D) {
  const int vpr = D >> 3, nv = kPT * vpr;
  for (int vi = threadIdx.x; vi < nv; vi += 256) {
    const int r = vi / vpr, c = (vi - r * vpr) * 8;
    float v[8];
    if (r < rows) {
      load8<T>(src + r * stride + c, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
    *reinterpret_cast<float4*>(dst + r * ld + c) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(dst + r * ld + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256, 2) sattn_packed_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                           const T* __restrict__ v, const float* __restrict__ lg,
                                                           const int* __restrict__ cu, T* __restrict__ out, int R,
                                                           int Tn, int Hq, int Hk, PackedStrides st,
                                                           float scale) {
  extern __shared__ float4 smem4[];
  __shared__ PackedTile s_tile;
  float* sm = reinterpret_cast<float*>(smem4);
  constexpr int LD = D + 4, LDP = kPT + 4, G = D > 64 ? 2 : 1;
  float* Qs = sm;
  float* Ks = Qs + kPT * LD;
  float* Vs = simt_share<D>() ? Ks : Ks + kPT * LD;
  float* Ps = Vs + kPT * LD;
  float* gs = Ps + kPT * LDP;
  const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;
  if (tid < 32) {
    PackedFinder<6> finder;
    finder.init(cu, R, Tn);
    const PackedTile t = finder.find((int)blockIdx.y);
    if (tid == 0) s_tile = t;
  }
  __syncthreads();
  const PackedTile tile = s_tile;
  if (tile.rows <= 0) return;
  const int hq = blockIdx.x, hk = hq / (Hq / Hk);
  T* ob = out + ((long long)tile.tok0 * Hq + hq) * D;
  if (tile.seq < 0) {  // rows of no sequence
    for (int i = tid; i < tile.rows * D; i += 256) ob[(long long)(i / D) * Hq * D + i % D] = from_f32<T>(0.f);
    return;
  }
  const int q0 = tile.q0, n = tile.n;
  const long long base = tile.tok0 - q0;  // the sequence's first token
  stage64<T>(Qs, LD, q + (long long)tile.tok0 * st.q_ts + hq * st.q_hs, st.q_ts, tile.rows, D);
  uint64_t o[4][2 * G];
  float m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < 2 * G; ++e) o[i][e] = 0;
  }
  int dcol[G];
#pragma unroll
  for (int g = 0; g < G; ++g) dcol[g] = min(4 * tc + 64 * g, D - 4);
  const int qt = q0 / kPT;
  for (int kt = 0; kt <= qt; ++kt) {
    const int k0 = kt * kPT;
    __syncthreads();  // previous tile's K, V, P consumed
    stage64<T>(Ks, LD, k + (base + k0) * st.k_ts + hk * st.k_hs, st.k_ts, min(kPT, n - k0), D);
    if constexpr (!simt_share<D>())
      stage64<T>(Vs, LD, v + (base + k0) * st.v_ts + hk * st.v_hs, st.v_ts, min(kPT, n - k0), D);
    if (tid < kPT) gs[tid] = lg && k0 + tid < n ? lg[(base + k0 + tid) * Hk + hk] : 0.f;
    __syncthreads();
    uint64_t s2[4][4];  // sums over even and over odd dimensions
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s2[i][j] = 0;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      ulonglong2 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const ulonglong2*>(Qs + (tr + 16 * i) * LD + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const ulonglong2*>(Ks + (tc + 16 * j) * LD + d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s2[i][j] = fma2(a[i].y, b[j].y, fma2(a[i].x, b[j].x, s2[i][j]));
    }
    float sc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[i][j] = lo2(s2[i][j]) + hi2(s2[i][j]);
    bool skip = false;  // some row of this thread's half warp does not see some key of the tile
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int qi = q0 + tr + 16 * i;
      float rmax = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int kj = k0 + tc + 16 * j;
        const float g = gs[tc + 16 * j];
        const bool sees = kj < n && (kj == qi || (kj < qi && g != -INFINITY));
        const float s = sees ? sc[i][j] * scale + (kj < qi ? g : 0.f) : -INFINITY;
        skip |= !sees;
        sc[i][j] = s;
        rmax = fmaxf(rmax, s);
      }
      rmax = hw_max(rmax);
      const float mn = fmaxf(m[i], rmax);
      const float corr = m[i] == -INFINITY ? 0.f : expf(m[i] - mn);
      float rs = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = sc[i][j] == -INFINITY ? -0.f : expf(sc[i][j] - mn);  // (a weight is never -0)
        rs += p;
        Ps[(tr + 16 * i) * LDP + tc + 16 * j] = p;
      }
      l[i] = l[i] * corr + hw_sum(rs);
#pragma unroll
      for (int e = 0; e < 2 * G; ++e) o[i][e] = pk2(lo2(o[i][e]) * corr, hi2(o[i][e]) * corr);
      m[i] = mn;
    }
    // a key that a row does not see is left out of its product, not multiplied by zero; one that it sees is
    // multiplied also where its weight has underflowed
    skip = __syncthreads_or(skip);
    if constexpr (simt_share<D>()) {  // (every score has been computed)
      stage64<T>(Vs, LD, v + (base + k0) * st.v_ts + hk * st.v_hs, st.v_ts, min(kPT, n - k0), D);
      __syncthreads();
    }
    auto pv = [&](auto leave_out) {
#pragma unroll 2
      for (int j = 0; j < kPT; j += 4) {
        float4 pa[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pa[i] = *reinterpret_cast<const float4*>(Ps + (tr + 16 * i) * LDP + j);
#pragma unroll
        for (int qq = 0; qq < 4; ++qq) {
          ulonglong2 vv[G];
#pragma unroll
          for (int g = 0; g < G; ++g) vv[g] = *reinterpret_cast<const ulonglong2*>(Vs + (j + qq) * LD + dcol[g]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = qq == 0 ? pa[i].x : (qq == 1 ? pa[i].y : (qq == 2 ? pa[i].z : pa[i].w));
            const uint64_t pp = pk2(p, p);
            const bool out = decltype(leave_out)::value && __float_as_uint(p) == 0x80000000u;
#pragma unroll
            for (int g = 0; g < G; ++g) {
              o[i][2 * g] = fma2(pp, out ? 0 : vv[g].x, o[i][2 * g]);
              o[i][2 * g + 1] = fma2(pp, out ? 0 : vv[g].y, o[i][2 * g + 1]);
            }
          }
        }
      }
    };
    if (skip)
      pv(std::true_type{});
    else
      pv(std::false_type{});
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ri = tr + 16 * i;
    if (ri >= tile.rows) continue;
    const float inv = 1.0f / l[i];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int d = 4 * tc + 64 * g;
      if (d >= D) continue;
      T* op = ob + (long long)ri * Hq * D + d;
#pragma unroll
      for (int e = 0; e < 4; ++e) op[e] = from_f32<T>((e & 1 ? hi2(o[i][2 * g + (e >> 1)]) : lo2(o[i][2 * g + (e >> 1)])) * inv);
    }
  }
}

template <typename T, int D>
cudaError_t packed_simt_d(const PackedArgs& a, cudaStream_t s) {
  constexpr size_t smem = simt_smem<D>();
  static unsigned long long allowed = 0;
  cudaError_t e = allow_smem(sattn_packed_kernel<T, D>, smem, allowed);
  if (e != cudaSuccess) return e;
  dim3 grid((unsigned)a.Hq, (unsigned)packed_tile_bound(a.T, a.R, kPT));
  sattn_packed_kernel<T, D><<<grid, 256, smem, s>>>((const T*)a.q, (const T*)a.k, (const T*)a.v, a.log_gate, a.cu,
                                                    (T*)a.out, a.R, a.T, a.Hq, a.Hk, a.st, a.scale);
  return cudaGetLastError();
}

template <typename T>
cudaError_t packed_simt_t(const PackedArgs& a, cudaStream_t s) {
  switch (a.D) {
    case 16: return packed_simt_d<T, 16>(a, s);
    case 32: return packed_simt_d<T, 32>(a, s);
    case 64: return packed_simt_d<T, 64>(a, s);
    case 128: return packed_simt_d<T, 128>(a, s);
  }
  return cudaErrorInvalidValue;
}

// ===========================================================================
// Tensor-core kernel (16-bit types, head_dim 64 or 128). CTA = two 128-query tiles, w = 0 and 1:
// the same positions of two query heads that share a key head, or (heads that cannot be paired)
// two neighbouring tiles of one head. With two heads both tiles have the same keys, and
// a prompt is cut at 128 positions instead of 256. Warp roles (12 warps):
//   warp 0            loads: the Q tiles once, then 128-key tiles of K and V by TMA into a ring;
//   warp 1            products: S_w = Q_w K_j^T into TMEM; once softmax w has written P_w(j) over
//                     S_w(j): O_w += P_w V_j (A from TMEM), then S_w(j + 1). The tiles alternate, so
//                     that the tensor core works on one while the other's softmax runs;
//   warps 4-7, 8-11   softmax of tile w, thread = query row = TMEM lane, a tile's 128 scores in
//                     registers: running maximum in log2 units (O is rescaled only when it grows by
//                     more than 2^kRescale), P = 2^(s - m + kOffset) rounded to the type, fp32 sums;
//   warps 2-3         what no query may meet: a product multiplies by zero where it should leave
//                     out, which is wrong for infinities and NaN. In the last key tiles (own, later
//                     and other sequences' positions) they set non-finite elements of V to zero, and
//                     the rows that do see one add it at the end (`odd`); with gates, they write the
//                     tile's gates and set the K and V rows of dropped keys to zero.
// The bound is the tensor core (4 D operations a score) together with the special-function unit
// (one exponential a score: 16 a clock and SM, just as long as the products of head_dim 128).
// Every second to eighth pair of exponentials on the FMA pipes instead (a cubic) gained 4 % on a cool card
// and lost 1 to 7 % at the power limit, where such kernels run when there is more than one of them.
// A prompt of 8192 tokens, 32 heads on 8 of 128, bf16: 471 us (1170 TFLOP/s) cool, 548 us (1000) back to
// back; a pair of 128 x 128 tiles takes 3400 cycles, of which its products alone 2040.
// TMEM columns: S_0 [0, 128) S_1 [128, 256) (P_w in the first 64 of S_w) O_0 [256, 256 + D) O_1 [384, 384 + D).
// Every wait is bounded; a role that gives up records a site code and leaves its loop, and the others'
// waits for it run out in turn. A CTA goes from one pair of tiles to the next (cluster launch control:
// it cancels the launch of a CTA that has not begun and takes over its number): the next pair's
// loads and first scores run while the last rows are written.
// ===========================================================================
using namespace sm100;

constexpr int kPkThreads = 384;
constexpr int kCleanSlots = 4;
constexpr float kPkLog2e = 1.4426950408889634f;
// P in bfloat16 has fp32's exponents. In fp16 it would lose bits below 2^-14 and end at 2^-25, while the sums go on:
// 131000 keys of weight e^-16.2, 1 % of a row, came out 29 % too heavy. Up to 2^15 it keeps all bits
// down to 2^-21 of the largest weight, and no weight is off by more than 2^-32 of it.
template <typename T> struct PkRange { static constexpr float kRescale = 8.0f * kPkLog2e, kOffset = 0.0f; };
template <> struct PkRange<__half> { static constexpr float kRescale = 8.0f, kOffset = 7.0f; };
constexpr unsigned int kSitePkLoad = 0x411, kSitePkMma = 0x412, kSitePkSoft = 0x413, kSitePkClean = 0x414;
template <int D> constexpr int pk_tile_bytes() { return 128 * D * 2; }
// One ring for the tiles of K and V in the order of their use, K_0 V_0 K_1 V_1 ...: what shared memory
// holds beside the two Q tiles.
template <int D> constexpr int pk_slots() { return D == 128 ? 5 : 8; }
// Gates of tile j + G may take the place of tile j's: V_{j + G} is loaded when element
// 2 (j + G) + 1 - slots has been used, K_{j + 1} or V_j, that is after the softmaxes of tile j.
template <int D> constexpr int pk_gate_slots() { return D == 128 ? 3 : 4; }
template <int D> constexpr int pk_bar_bytes() { return D == 128 ? 320 : 368; }
template <int D, bool GATED> constexpr size_t pk_smem() {
  return 1024 + (size_t)(2 + pk_slots<D>()) * pk_tile_bytes<D>() + (GATED ? pk_gate_slots<D>() * 128 * 4 : 0) + pk_bar_bytes<D>();
}
static_assert(pk_smem<128, true>() + 96 <= 227 * 1024, "shared memory of a CTA");

__device__ __forceinline__ float pk_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A wait for warps that mostly wait: suspended in the barrier, so that they take neither issue slots nor
// power from the others. Bounded by the number of waits, each of at most about 10 us.
__device__ __forceinline__ bool idle_wait(uint32_t bar, uint32_t parity, unsigned int site) {
  for (uint32_t it = 0; it < 100000u; ++it)
    if (mbar_try_wait(bar, parity, 10000u)) return true;
  record_error(site);
  return false;
}

// Low word of a 128-byte-swizzled operand's descriptor; the high word is the same for all of them (8-row
// groups 1024 bytes apart, descriptor version, swizzle). Addresses below 2^18 only move the low 14 bits.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
  return ((addr >> 4) & 0x3fffu) | ((lbo >> 4) << 16);
}
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 x, {%1, %3};\n\tmov.b64 y, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(kDescHi), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 y, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(kDescHi), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// One lane of the (whole) warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(x));
  return x != 0;
}

// 64 bytes of one thread, as two whole 32-byte sectors where the address allows it.
__device__ __forceinline__ void store64(void* p, const uint32_t (&y)[16], bool wide) {
  if (wide) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<char*>(p) + 32 * i),
                   "r"(y[8 * i]), "r"(y[8 * i + 1]), "r"(y[8 * i + 2]), "r"(y[8 * i + 3]), "r"(y[8 * i + 4]),
                   "r"(y[8 * i + 5]), "r"(y[8 * i + 6]), "r"(y[8 * i + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
  }
}

struct PackedTcArgs {
  const float* lg;
  const int* cu;
  const void* v;
  void* out;
  int R, T, Hq, Hk;
  long long v_ts, v_hs;
  float scale;
};

// A CTA's pair of tiles, as the loading warp hands it to the others.
struct PackedWork {
  int seq0, q0, n;  // the sequence's first token, the (first) tile's position, the sequence's length
  int head;         // the first tile's query head; < 0: no more work
  int odd;          // elements of V were set to zero
  __device__ __forceinline__ int tiles0() const { return q0 / 128 + 1; }                                    // key tiles
  __device__ __forceinline__ int tiles1(bool pair) const { return pair ? q0 / 128 + 1 : (q0 + 128 < n ? q0 / 128 + 2 : 0); }
};

// Asks for the launch of one more CTA of this grid to be cancelled; 16 bytes of answer go to `to`
// and complete on `bar` (PTX ISA, clusterlaunchcontrol).
__device__ __forceinline__ void ask_work(uint32_t to, uint32_t bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(to),
               "r"(bar)
               : "memory");
}
// The answer: the index of the cancelled CTA, x = -1 when there was none left.
__device__ __forceinline__ int2 work_answer(uint32_t from) {
  int2 c;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t.reg .b32 z, w;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "mov.b32 %0, -1;\n\tmov.b32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, %1, z, w}, r;\n\t}"
      : "=r"(c.x), "=r"(c.y)
      : "r"(from)
      : "memory");
  return c;
}

// PAIR: the two tiles are two heads.
template <typename T, int D, bool GATED, bool PAIR>
__global__ void __launch_bounds__(kPkThreads, 1)
    sattn_packed_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, const PackedTcArgs a) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int NS = pk_slots<D>(), TILE = pk_tile_bytes<D>(), NB = D / 64;  // 64-column blocks of 16 KB
  constexpr int GS = pk_gate_slots<D>();
  extern __shared__ uint8_t smraw[];
  uint8_t* base = align1024_shared(smraw);
  uint8_t* sQ = base;
  auto slot_at = [&](int i) { return base + (2 + i % NS) * TILE; };  // of element i: K_j is 2 j, V_j 2 j + 1
  float* gates = reinterpret_cast<float*>(base + (2 + NS) * TILE);
  uint64_t* bars = reinterpret_cast<uint64_t*>(gates + (GATED ? pk_gate_slots<D>() * 128 : 0));
  enum {
    Q_FULL = 0, Q_EMPTY = 1, FULL = 2, EMPTY = FULL + NS, CLEAN = EMPTY + NS, CARE_V = CLEAN + kCleanSlots,
    CARE = CARE_V + 4, S_FULL = CARE + 4, P_FULL = S_FULL + 2, O_DONE = P_FULL + 2, O_FREE = O_DONE + 2,
    W_FULL = O_FREE + 2, W_EMPTY = W_FULL + 2, ANSWERED = W_EMPTY + 2, DRAIN = ANSWERED + 1, NBARS = DRAIN + 1
  };
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + NBARS);
  __shared__ __align__(16) uint8_t s_answer[16];
  __shared__ volatile PackedWork s_work[2];
  static_assert(NBARS * 8 + 8 <= pk_bar_bytes<D>(), "barrier area");
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 1) tmem_alloc(smem_u32(tslot), 512);
  if (tid == 64) {
    prefetch_tmap(&tm_q);
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    for (int i = 0; i < NBARS; ++i) {
      int n = 1;
      if (i >= CLEAN && i < CLEAN + kCleanSlots) n = 2;  // two cleaning warps
      if (i >= CARE && i < CARE + 4) n = 2;
      if (i >= P_FULL && i < P_FULL + 2) n = 4;          // the four warps of a softmax
      if (i >= O_FREE && i < O_FREE + 2) n = 4;
      if (i >= W_EMPTY && i < W_EMPTY + 2) n = 11;       // every warp but the loading one
      mbar_init(bar(i), n);
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  T* out = reinterpret_cast<T*>(a.out);
  constexpr uint32_t T_S = 0, T_O = 256;
  // Registers: launched with 168 a thread (384 x 168 = 64512); warpgroup 0 keeps 56 and the two softmax
  // warpgroups take 208 each: 128 x 56 + 256 x 208 = 60416 <= 64512.
  static_assert(kPkThreads == 384, "register split assumes three warpgroups");
  const int group = a.Hq / a.Hk;

  // Work `it` of this CTA for the roles that use it (whole warps): false when a wait ran out.
  auto next_work = [&](int it, PackedWork& w) {
    if (!__all_sync(0xffffffffu, mbar_wait(bar(W_FULL + (it & 1)), (it >> 1) & 1, kSitePkLoad))) return false;
    volatile PackedWork& s = s_work[it & 1];
    w.seq0 = s.seq0, w.q0 = s.q0, w.n = s.n, w.head = s.head;
    return true;
  };
  // The barriers of a work's one or two last key tiles (c) are those of every other work: the loading and
  // cleaning warps may be a work ahead of the others, but not two (a work's place is free when every
  // role is done with it). `second` counts the works of either kind so far that have two.
  auto care_parity = [&](int it, int c, const int (&second)[2]) { return (c ? second[it & 1] : it >> 1) & 1; };
  auto work_done = [&](int it) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(W_EMPTY + (it & 1)));
  };

  if (warp == 0) {
    // ------------------------------------------------------------ work and loads
    regs_dec<56>();
    int2 c = make_int2((int)blockIdx.x, (int)blockIdx.y);
    bool ok = true;
    int it = 0, asked = 0, i0 = 0;  // works, answers, elements before this work
    PackedFinder<PAIR ? 7 : 8> finder;
    finder.init(a.cu, a.R, a.T);
    for (; c.x >= 0 && ok; ++asked) {
      if (lane == 0) {
        mbar_expect_tx(bar(ANSWERED), 16);
        ask_work(smem_u32(s_answer), bar(ANSWERED));
      }
      const PackedTile tile = finder.find(c.y);
      const int heads = PAIR ? 2 : 1, head = c.x * heads;
      if (tile.seq < 0) {  // nothing, or rows of no sequence
        const int row = heads * D / 8;  // 16-byte words of a token
        for (int i = lane; i < tile.rows * row; i += 32)
          *reinterpret_cast<uint4*>(out + ((long long)(tile.tok0 + i / row) * a.Hq + head) * D + i % row * 8) =
              make_uint4(0u, 0u, 0u, 0u);
      } else {
        PackedWork w{tile.tok0 - tile.q0, tile.q0, tile.n, head, 0};
        const int n0 = w.tiles0(), n1 = w.tiles1(PAIR), nk = max(n0, n1), care = n0 - 1, hk = head / group;
        if (it >= 2) ok = __all_sync(0xffffffffu, idle_wait(bar(W_EMPTY + (it & 1)), ((it >> 1) - 1) & 1, kSitePkLoad));
        if (lane == 0 && ok) {
          volatile PackedWork& s = s_work[it & 1];
          s.seq0 = w.seq0, s.q0 = w.q0, s.n = w.n, s.head = w.head, s.odd = 0;
          mbar_arrive(bar(W_FULL + (it & 1)));
        }
        if (ok && it > 0) ok = __all_sync(0xffffffffu, idle_wait(bar(Q_EMPTY), (it - 1) & 1, kSitePkLoad));
        if (ok) {
          const int nq = n1 > 0 ? 2 : 1;
          if (lane == 0) {
            mbar_expect_tx(bar(Q_FULL), (uint32_t)(nq * TILE));
            for (int t = 0; t < nq; ++t)
#pragma unroll
              for (int b = 0; b < NB; ++b)
                tma_load_3d(smem_u32(sQ + t * TILE + b * 16384), &tm_q, 64 * b, w.seq0 + w.q0 + (PAIR ? 0 : 128 * t),
                            head + (PAIR ? t : 0), bar(Q_FULL));
          }
          for (int e = 0; e < 2 * nk && ok; ++e) {
            const int i = i0 + e, j = e >> 1, sl = i % NS;
            if (i >= NS)
              ok = __all_sync(0xffffffffu, idle_wait(bar(EMPTY + sl), ((i / NS) - 1) & 1, kSitePkLoad));
            if (!ok) break;
            // V tiles that are to be cleaned arrive on a barrier of their own (the ring's goes on)
            const bool special = (e & 1) && j >= care;
            const uint32_t b_in = bar(special ? CARE_V + 2 * (it & 1) + j - care : FULL + sl);
            if (lane == 0) {
              if (special) mbar_arrive(bar(FULL + sl));
              mbar_expect_tx(b_in, (uint32_t)TILE);
#pragma unroll
              for (int b = 0; b < NB; ++b)
                tma_load_3d(smem_u32(slot_at(i) + b * 16384), e & 1 ? &tm_v : &tm_k, 64 * b, w.seq0 + 128 * j, hk, b_in);
            }
          }
          i0 += 2 * nk;
        }
        ++it;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(bar(ANSWERED), asked & 1, kSitePkLoad))) ok = false;
      c = work_answer(smem_u32(s_answer));
      fence_proxy_async_smem();  // the answer has been read before the next one is written
      __syncwarp();
    }
    if (ok && it >= 2) ok = __all_sync(0xffffffffu, idle_wait(bar(W_EMPTY + (it & 1)), ((it >> 1) - 1) & 1, kSitePkLoad));
    if (ok && lane == 0) {
      s_work[it & 1].head = -1;
      mbar_arrive(bar(W_FULL + (it & 1)));
      // No copy may be in flight when the CTA exits: the last work has been used up. (After a wait that
      // ran out, every copy has long arrived.)
      if (it > 0) idle_wait(bar(W_EMPTY + ((it - 1) & 1)), ((it - 1) >> 1) & 1, kSitePkLoad);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    // One warp for both tiles, which keeps them half a period apart. The whole warp runs the role and
    // one elected lane issues: addresses, descriptors and the loop stay in uniform registers, which
    // the instruction takes its operands from.
    regs_dec<56>();
    constexpr uint32_t ID_S = idesc_f16(128, 128, BF16, false, false);
    constexpr uint32_t ID_O = idesc_f16(128, D, BF16, false, true);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t qd = desc_lo(__shfl_sync(0xffffffffu, smem_u32(sQ), 0), 16);
    const uint32_t kd = desc_lo(__shfl_sync(0xffffffffu, smem_u32(slot_at(0)), 0), 16);
    const uint32_t vd = desc_lo(__shfl_sync(0xffffffffu, smem_u32(slot_at(0)), 0), 16384);
    const bool lead = elect_one();
    auto wait = [&](uint32_t b, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_wait(b, parity, kSitePkMma)); };
    int i0 = 0, cleaned = 0, second[2] = {0, 0}, steps[2] = {0, 0}, outs[2] = {0, 0};
    bool fail = false;
    for (int it = 0; !fail; ++it) {
      PackedWork work;
      if (!next_work(it, work)) {
        fail = true;
        break;
      }
      if (work.head < 0) break;
      const int n0 = __shfl_sync(0xffffffffu, work.tiles0(), 0), n1 = __shfl_sync(0xffffffffu, work.tiles1(PAIR), 0);
      const int first_care = n0 - 1, nkt = max(n0, n1);
      auto ready_k = [&](int j) {  // tile j of K, clean where it has to be
        if (GATED && j < first_care) return wait(bar(CLEAN + (cleaned + j) % kCleanSlots), ((cleaned + j) / kCleanSlots) & 1);
        return wait(bar(FULL + (i0 + 2 * j) % NS), ((i0 + 2 * j) / NS) & 1);
      };
      auto ready_v = [&](int j) {
        if (j >= first_care)
          return wait(bar(CARE + 2 * (it & 1) + j - first_care), care_parity(it, j - first_care, second));
        if (GATED) return wait(bar(CLEAN + (cleaned + j) % kCleanSlots), ((cleaned + j) / kCleanSlots) & 1);
        return wait(bar(FULL + (i0 + 2 * j + 1) % NS), ((i0 + 2 * j + 1) / NS) & 1);
      };
      auto issue_s = [&](int w, int j, bool last) {
        const int sl = (i0 + 2 * j) % NS;
        const uint32_t q1 = qd + (uint32_t)(w * (TILE >> 4)), k1 = kd + (uint32_t)(sl * (TILE >> 4));
        if (lead) {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = (uint32_t)(((ks >> 2) * 16384 + (ks & 3) * 32) >> 4);
            mma_ss(tm + T_S + 128 * w, q1 + off, k1 + off, ID_S, ks > 0);
          }
          umma_commit(bar(S_FULL + w));
          if (last) {
            if (!GATED || j < first_care) umma_commit(bar(EMPTY + sl));
            if (j == nkt - 1) umma_commit(bar(Q_EMPTY));
          }
        }
      };
      fail = !wait(bar(Q_FULL), it & 1) || !ready_k(0);
      if (!fail) {
        tc_fence_after();
        issue_s(0, 0, n1 == 0);
        if (n1 > 0) issue_s(1, 0, true);
      }
      for (int j = 0; j < nkt && !fail; ++j) {
        const int sl = (i0 + 2 * j + 1) % NS;
        const uint32_t v1 = vd + (uint32_t)(sl * (TILE >> 4));
        if (!ready_v(j) || (j + 1 < nkt && !ready_k(j + 1))) {
          fail = true;
          break;
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int nw = w ? n1 : n0;
          if (fail || j >= nw) continue;
          // (the first product into O_w: the last work's rows have been read)
          if (!wait(bar(P_FULL + w), steps[w]++ & 1) ||
              (j == 0 && outs[w] > 0 && !wait(bar(O_FREE + w), (outs[w] - 1) & 1))) {
            fail = true;
            continue;
          }
          tc_fence_after();
          if (lead) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
              mma_ts(tm + T_O + 128 * w, tm + T_S + 128 * w + 8 * ks, v1 + (uint32_t)(128 * ks), ID_O, j > 0 || ks > 0);
            if (w == (j < n1 ? 1 : 0)) {
              umma_commit(bar(EMPTY + sl));  // V_j has been used
              // The cleaning warps wait for the last K tiles, too, but hand over nothing before V: only now
              // is it certain that they have seen this one, and its place may be filled again.
              if (GATED && j >= first_care) umma_commit(bar(EMPTY + (i0 + 2 * j) % NS));
            }
          }
          if (j + 1 < nw) {
            issue_s(w, j + 1, w == (j + 1 < n1 ? 1 : 0));  // over P_w(j): products run in the order of their issue
          } else {
            if (lead) umma_commit(bar(O_DONE + w));
            ++outs[w];
          }
        }
      }
      i0 += 2 * nkt;
      cleaned += first_care;
      second[it & 1] += nkt > n0;
      work_done(it);
    }
    // every product has completed before TMEM is released
    if (lead) umma_commit(bar(DRAIN));
    wait(bar(DRAIN), 0);
  } else if (warp < 4) {
    // ------------------------------------------------------------ clean tiles
    regs_dec<56>();
    const int t = tid - 64;  // 0 .. 63: keys t and t + 64 of a tile
    int i0 = 0, cleaned = 0, tiles = 0, second[2] = {0, 0};
    bool ok = true;
    for (int it = 0; ok; ++it) {
      PackedWork work;
      ok = next_work(it, work);
      if (!ok || work.head < 0) break;
      const int care = work.tiles0() - 1, nk = max(work.tiles0(), work.tiles1(PAIR)), hk = work.head / group;
      auto gate_at = [&](int key) {
        if constexpr (!GATED) return 0.f;
        return key < work.n ? a.lg[(long long)(work.seq0 + key) * a.Hk + hk] : 0.f;
      };
      auto in_log2 = [](float x) {  // (only -inf itself drops a key)
        const float y = x * kPkLog2e;
        return y == -INFINITY && x != -INFINITY ? -FLT_MAX : y;
      };
      int j = GATED ? 0 : care;
      float g0 = gate_at(128 * j + t), g1 = gate_at(128 * j + t + 64);
      for (; j < nk; ++j) {
        const int ik = i0 + 2 * j;
        uint8_t *kt = slot_at(ik), *vt = slot_at(ik + 1);
        // (with gates also K of the tiles that are not changed here: the ring's phases are followed one by one)
        if (GATED) ok = idle_wait(bar(FULL + ik % NS), (ik / NS) & 1, kSitePkClean);
        if (j < care)
          ok = ok && idle_wait(bar(FULL + (ik + 1) % NS), ((ik + 1) / NS) & 1, kSitePkClean);
        else
          ok = ok && idle_wait(bar(CARE_V + 2 * (it & 1) + j - care), care_parity(it, j - care, second), kSitePkClean);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if constexpr (GATED) {
          gates[((tiles + j) % GS) * 128 + t] = in_log2(g0);
          gates[((tiles + j) % GS) * 128 + t + 64] = in_log2(g1);
          if (j < care) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if ((half ? g1 : g0) != -INFINITY) continue;
              const int key = t + 64 * half;
#pragma unroll
              for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                  *reinterpret_cast<uint4*>(kt + b * 16384 + key * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                  *reinterpret_cast<uint4*>(vt + b * 16384 + key * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
          }
          g0 = gate_at(128 * (j + 1) + t);
          g1 = gate_at(128 * (j + 1) + t + 64);
        }
        if (j >= care) {
          // x * 0 is 0 but for infinities and NaN: four packed products for 16 bytes see whether there are
          // any; only then are they looked for.
          uint4* ve = reinterpret_cast<uint4*>(vt);
          using T2 = typename std::conditional<BF16, __nv_bfloat162, __half2>::type;
          uint32_t zeros[4] = {0u, 0u, 0u, 0u};
#pragma unroll 8
          for (int i = t; i < TILE / 16; i += 64) {
            const uint4 x = ve[i];
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t zero = 0u;
              const T2 y = __hfma2(*reinterpret_cast<const T2*>(&xs[q]), *reinterpret_cast<const T2*>(&zero),
                                   *reinterpret_cast<const T2*>(&zeros[q]));
              zeros[q] = *reinterpret_cast<const uint32_t*>(&y);
            }
          }
          bool odd = false;
          // (a sum is +0, -0 or NaN)
          if (((zeros[0] | zeros[1] | zeros[2] | zeros[3]) & 0x7fff7fffu) != 0u) {
            constexpr uint32_t EXP = BF16 ? 0x7f80u : 0x7c00u;
            odd = true;
            auto fix = [&](uint32_t w) {
              if ((w & EXP) == EXP) w &= 0xffff0000u;
              if ((w & (EXP << 16)) == (EXP << 16)) w &= 0xffffu;
              return w;
            };
            for (int i = t; i < TILE / 16; i += 64) {
              const uint4 x = ve[i];
              ve[i] = make_uint4(fix(x.x), fix(x.y), fix(x.z), fix(x.w));
            }
          }
          if (odd) s_work[it & 1].odd = 1;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(j >= care ? CARE + 2 * (it & 1) + j - care : CLEAN + (cleaned + j) % kCleanSlots));
      }
      i0 += 2 * nk;
      cleaned += care;
      tiles += nk;
      second[it & 1] += nk > care + 1;
      work_done(it);
    }
  } else {
    // ------------------------------------------------------------ softmax of tile w
    regs_inc<208>();
    const int w = (warp - 4) >> 2;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + tl + T_S + 128 * w, to = tmem + tl + T_O + 128 * w;
    const float scale2 = a.scale * kPkLog2e;
    int tiles = 0, cleaned = 0, second[2] = {0, 0}, steps = 0, outs = 0;
    bool wfail = false;
    auto warp_wait = [&](uint32_t b, uint32_t parity) {
      if (!wfail) wfail = !__all_sync(0xffffffffu, mbar_wait(b, parity, kSitePkSoft));
      return !wfail;
    };
    for (int it = 0; !wfail; ++it) {
      PackedWork work;
      wfail = !next_work(it, work);
      if (wfail || work.head < 0) break;
      const int care = work.tiles0() - 1, nk0 = work.tiles0(), nk1 = work.tiles1(PAIR), my_nk = w ? nk1 : nk0;
      const int qi = work.q0 + (PAIR ? 0 : 128 * w) + r;
      float m_used = -INFINITY, lsum = 0.f;
      for (int j = 0; j < my_nk; ++j) {
        if (!warp_wait(bar(S_FULL + w), steps & 1)) break;
        ++steps;
        if (GATED && !warp_wait(j >= care ? bar(CARE + 2 * (it & 1) + j - care) : bar(CLEAN + (cleaned + j) % kCleanSlots),
                                j >= care ? care_parity(it, j - care, second) : ((cleaned + j) / kCleanSlots) & 1))
          break;
        tc_fence_after();
        uint32_t sv[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, sv[c]);
        tmem_wait_ld();
        const float* g = gates + ((tiles + j) % GS) * 128;
        float mp[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        float mul = scale2;  // what the scores are still to be multiplied by
        if constexpr (GATED) {
          mul = 1.f;
          if (j < care) {
            const uint64_t sc2 = pk2(scale2, scale2);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const float4 gg = *reinterpret_cast<const float4*>(g + 32 * c + e);
                const uint64_t x0 = fma2(pk2(__uint_as_float(sv[c][e]), __uint_as_float(sv[c][e + 1])), sc2, pk2(gg.x, gg.y));
                const uint64_t x1 = fma2(pk2(__uint_as_float(sv[c][e + 2]), __uint_as_float(sv[c][e + 3])), sc2, pk2(gg.z, gg.w));
                sv[c][e] = (uint32_t)x0, sv[c][e + 1] = (uint32_t)(x0 >> 32);
                sv[c][e + 2] = (uint32_t)x1, sv[c][e + 3] = (uint32_t)(x1 >> 32);
              }
          } else {
            // (the keys of these tiles are as they came: a dropped one's score may be a NaN)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const bool own = 128 * j + 32 * c + e == qi;
                const float gg = g[32 * c + e], x = __uint_as_float(sv[c][e]) * scale2;
                sv[c][e] = __float_as_uint(own ? x : (gg == -INFINITY ? -INFINITY : x + gg));
              }
          }
        } else if (!(scale2 > 0.f)) {  // (the largest score is not the largest product's then)
          mul = 1.f;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) sv[c][e] = __float_as_uint(__uint_as_float(sv[c][e]) * scale2);
        }
        if (j >= care) {
          // Later positions. The warp's rows see all keys up to column `edge` of the tile and each lane
          // one more than the lane before it: blocks of 32 columns up to there stay as they are.
          const int edge = qi - lane - 128 * j;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (32 * c + 31 <= edge) continue;
            const int last = edge + lane - 32 * c;  // the block's last column that the row sees
#pragma unroll
            for (int e = 0; e < 32; ++e) sv[c][e] = e > last ? __float_as_uint(-INFINITY) : sv[c][e];
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mp[q] = fmaxf(fmaxf(mp[q], __uint_as_float(sv[c][e + 2 * q])), __uint_as_float(sv[c][e + 2 * q + 1]));
        // (a score of NaN or +inf makes the row's sum NaN or +inf, and its results NaN)
        const float mt = fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])) * mul;
        float f = 1.f;
        bool resc = false;
        if (mt < INFINITY && mt > m_used + PkRange<T>::kRescale) {
          if (m_used != -INFINITY) {  // O and the sum hold earlier tiles: rescale them
            f = pk_ex2(m_used - mt);
            lsum *= f;
            resc = true;
          }
          m_used = mt;
        }
        // S_w(j) is complete, and with it the products before it: O_w holds the tiles up to j - 1
        if (__any_sync(0xffffffffu, resc)) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(to + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(to + 16 * c, o);
          }
        }
        const float mb = m_used == -INFINITY ? 0.f : PkRange<T>::kOffset - m_used;
        const uint64_t mul2 = pk2(mul, mul), mb2 = pk2(mb, mb);
        uint64_t ls[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const uint64_t d = fma2(pk2(__uint_as_float(sv[c][2 * q]), __uint_as_float(sv[c][2 * q + 1])), mul2, mb2);
            const float p0 = pk_ex2(lo2(d)), p1 = pk_ex2(hi2(d));
            ls[q & 1] = add2(ls[q & 1], pk2(p0, p1));
            pk[q] = pack2<T>(p0, p1);
          }
          tmem_st16(ts + 16 * c, pk);  // (the scores of these columns are in registers)
        }
        const uint64_t l2 = add2(ls[0], ls[1]);
        lsum += lo2(l2) + hi2(l2);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FULL + w));
      }
      if (my_nk > 0 && warp_wait(bar(O_DONE + w), outs & 1)) {
        ++outs;
        tc_fence_after();
        const float inv = 1.0f / lsum;
        const bool odd = s_work[it & 1].odd != 0;
        const int hk = work.head / group, head = work.head + (PAIR ? w : 0);
        T* op = out + ((long long)(work.seq0 + qi) * a.Hq + head) * D;
        const bool wide = (reinterpret_cast<uintptr_t>(out) & 31u) == 0;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(to + 32 * c, o);
          tmem_wait_ld();
          if (c == D / 32 - 1) {  // O_w has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(O_FREE + w));
          }
          if (qi < work.n) {
            if (odd) {
              // the elements of V that were set to zero, for the rows that see them
              for (int key = 128 * care; key <= qi; ++key) {
                if (GATED && key < qi && a.lg[(long long)(work.seq0 + key) * a.Hk + hk] == -INFINITY) continue;
                const T* vp = reinterpret_cast<const T*>(a.v) + (work.seq0 + key) * a.v_ts + hk * a.v_hs + 32 * c;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float x = to_f32<T>(vp[e]);
                  if (!(fabsf(x) < INFINITY)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
                }
              }
            }
            uint32_t y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              y[e] = pack2<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
            store64(op + 32 * c, y, wide);
          }
        }
      }
      tiles += max(nk0, nk1);
      cleaned += care;
      second[it & 1] += max(nk0, nk1) > nk0;
      work_done(it);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Tensor map over (D, tokens, heads) of a packed tensor, boxes of 64 columns x 128 tokens.
bool make_map_packed(CUtensorMap* map, const void* base, bool bf16, int D, int T, int H, long long ts, long long hs) {
  auto enc = tensor_map_encoder();
  if (!enc) return false;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)T, (cuuint64_t)H};
  cuuint64_t strides[2] = {(cuuint64_t)ts * 2, (cuuint64_t)hs * 2};
  cuuint32_t box[3] = {64, 128, 1};
  cuuint32_t es[3] = {1, 1, 1};
  return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
             dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool GATED, bool PAIR>
cudaError_t packed_tc_t(const PackedArgs& a, cudaStream_t s) {
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap mq, mk, mv;
  if (!make_map_packed(&mq, a.q, bf16, D, a.T, a.Hq, a.st.q_ts, a.st.q_hs) ||
      !make_map_packed(&mk, a.k, bf16, D, a.T, a.Hk, a.st.k_ts, a.st.k_hs) ||
      !make_map_packed(&mv, a.v, bf16, D, a.T, a.Hk, a.st.v_ts, a.st.v_hs))
    return cudaErrorInvalidValue;
  PackedTcArgs k{};
  k.lg = a.log_gate, k.cu = a.cu, k.v = a.v, k.out = a.out;
  k.R = a.R, k.T = a.T, k.Hq = a.Hq, k.Hk = a.Hk;
  k.v_ts = a.st.v_ts, k.v_hs = a.st.v_hs;
  k.scale = a.scale;
  const long long tiles = packed_tile_bound(a.T, a.R, PAIR ? 128 : 256);
  auto fn = sattn_packed_tc_kernel<T, D, GATED, PAIR>;
  static unsigned long long allowed = 0;
  cudaError_t e = allow_smem(fn, pk_smem<D, GATED>(), allowed);
  if (e != cudaSuccess) return e;
  fn<<<dim3((unsigned)(PAIR ? a.Hq / 2 : a.Hq), (unsigned)tiles), kPkThreads, pk_smem<D, GATED>(), s>>>(mq, mk, mv, k);
  return cudaGetLastError();
}

bool packed_pair(const PackedArgs& a) { return (a.Hq / a.Hk) % 2 == 0; }

template <typename T>
cudaError_t packed_tc(const PackedArgs& a, cudaStream_t s) {
  const bool pair = packed_pair(a);
  if (a.D == 64) {
    if (a.log_gate) return pair ? packed_tc_t<T, 64, true, true>(a, s) : packed_tc_t<T, 64, true, false>(a, s);
    return pair ? packed_tc_t<T, 64, false, true>(a, s) : packed_tc_t<T, 64, false, false>(a, s);
  }
  if (a.log_gate) return pair ? packed_tc_t<T, 128, true, true>(a, s) : packed_tc_t<T, 128, true, false>(a, s);
  return pair ? packed_tc_t<T, 128, false, true>(a, s) : packed_tc_t<T, 128, false, false>(a, s);
}

}  // namespace

bool sattn_packed_fits(const PackedArgs& a) {
  return packed_tile_bound(a.T, a.R, !a.use_tc ? kPT : (packed_pair(a) ? 128 : 256)) <= 65535;
}

bool sattn_packed_tc_supported(int D, int dtype) { return (D == 64 || D == 128) && dtype != SSD_F32; }

cudaError_t launch_sattn_packed(const PackedArgs& a, cudaStream_t s) {
  if (a.use_tc) return a.dtype == SSD_BF16 ? packed_tc<__nv_bfloat16>(a, s) : packed_tc<__half>(a, s);
  switch (a.dtype) {
    case SSD_F32: return packed_simt_t<float>(a, s);
    case SSD_BF16: return packed_simt_t<__nv_bfloat16>(a, s);
    case SSD_F16: return packed_simt_t<__half>(a, s);
  }
  return cudaErrorInvalidValue;
}

SSDB200_DEFINE_ERROR_FETCH(fetch_error_packed)

}  // namespace ssdb200
