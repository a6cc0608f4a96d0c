// sattn_packed.cu - selective attention over whole prompts of different lengths, packed one
// after another (cu_seqlens), causal, with grouped heads: the prefill of sattn.cu
// (modules/selective_attention.py:27-144, :270-280) without padding.
//   s_ij = scale * q_i . k_j + (j < i ? log_gate_j : 0), j <= i in i's sequence; out_i = softmax(s_i) . v
// Query head h reads key head h / (Hq / Hk). A key whose log-gate is -inf drops out for every later
// query, whatever it holds, and so does every key that a query does not see: a NaN or an infinity
// there changes nothing. Rows past the last sequence are written as zeros.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "packed_tiles.cuh"
#include "sattn_tiles.cuh"

namespace ssdb200 {
namespace {

// ===========================================================================
// CUDA-core kernel (fp32, and head_dim 16 or 32): CTA = (query head, 64-query tile of a sequence),
// 64-key tiles of K and V staged in shared memory as fp32; thread (tr, tc) owns rows tr + 16 i
// (i < 4), score columns tc + 16 j, output columns 4 tc + 64 g (g < 2). Bound by FFMA.
// ===========================================================================
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

template <typename T>
__global__ void __launch_bounds__(256) sattn_packed_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                           const T* __restrict__ v, const float* __restrict__ lg,
                                                           const int* __restrict__ cu, T* __restrict__ out, int R,
                                                           int Tn, int Hq, int Hk, int D, PackedStrides st,
                                                           float scale) {
  extern __shared__ float4 smem4[];
  __shared__ PackedTile s_tile;
  float* sm = reinterpret_cast<float*>(smem4);
  const int LD = D + 4, LDP = kPT + 4;
  float* Qs = sm;
  float* Ks = Qs + kPT * LD;
  float* Vs = Ks + kPT * LD;
  float* Ps = Vs + kPT * LD;
  float* gs = Ps + kPT * LDP;
  const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;
  if (tid < 32) find_packed_tile(cu, R, Tn, (int)blockIdx.y, kPT, &s_tile);
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
  float o[4][8], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[i][e] = 0.f;
  }
  int dcol[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) dcol[g] = min(4 * tc + 64 * g, D - 4);
  const int qt = q0 / kPT;
  for (int kt = 0; kt <= qt; ++kt) {
    const int k0 = kt * kPT;
    __syncthreads();  // previous tile's K, V, P consumed
    stage64<T>(Ks, LD, k + (base + k0) * st.k_ts + hk * st.k_hs, st.k_ts, min(kPT, n - k0), D);
    stage64<T>(Vs, LD, v + (base + k0) * st.v_ts + hk * st.v_hs, st.v_ts, min(kPT, n - k0), D);
    if (tid < kPT) gs[tid] = lg && k0 + tid < n ? lg[(base + k0 + tid) * Hk + hk] : 0.f;
    __syncthreads();
    float sc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
    for (int d = 0; d < D; d += 4) {
      float4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(Qs + (tr + 16 * i) * LD + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(Ks + (tc + 16 * j) * LD + d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float t = sc[i][j];
          t = fmaf(a[i].x, b[j].x, t);
          t = fmaf(a[i].y, b[j].y, t);
          t = fmaf(a[i].z, b[j].z, t);
          sc[i][j] = fmaf(a[i].w, b[j].w, t);
        }
    }
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
        const float p = sc[i][j] == -INFINITY ? 0.f : expf(sc[i][j] - mn);
        rs += p;
        Ps[(tr + 16 * i) * LDP + tc + 16 * j] = p;
      }
      l[i] = l[i] * corr + hw_sum(rs);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[i][e] *= corr;
      m[i] = mn;
    }
    // a key that a row does not see is left out of its product, not multiplied by zero
    skip = __syncthreads_or(skip);
#pragma unroll 2
    for (int j = 0; j < kPT; j += 4) {
      float4 pa[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) pa[i] = *reinterpret_cast<const float4*>(Ps + (tr + 16 * i) * LDP + j);
#pragma unroll
      for (int qq = 0; qq < 4; ++qq) {
        float4 vv[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) vv[g] = *reinterpret_cast<const float4*>(Vs + (j + qq) * LD + dcol[g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = qq == 0 ? pa[i].x : (qq == 1 ? pa[i].y : (qq == 2 ? pa[i].z : pa[i].w));
          if (skip && p == 0.f) continue;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            o[i][4 * g] = fmaf(p, vv[g].x, o[i][4 * g]);
            o[i][4 * g + 1] = fmaf(p, vv[g].y, o[i][4 * g + 1]);
            o[i][4 * g + 2] = fmaf(p, vv[g].z, o[i][4 * g + 2]);
            o[i][4 * g + 3] = fmaf(p, vv[g].w, o[i][4 * g + 3]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ri = tr + 16 * i;
    if (ri >= tile.rows) continue;
    const float inv = 1.0f / l[i];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int d = 4 * tc + 64 * g;
      if (d >= D) continue;
      T* op = ob + (long long)ri * Hq * D + d;
#pragma unroll
      for (int e = 0; e < 4; ++e) op[e] = from_f32<T>(o[i][4 * g + e] * inv);
    }
  }
}

template <typename T>
cudaError_t packed_simt_t(const PackedArgs& a, cudaStream_t s) {
  const size_t smem = (size_t)(3 * kPT * (a.D + 4) + kPT * (kPT + 4) + kPT) * sizeof(float);
  cudaError_t e = cudaFuncSetAttribute(sattn_packed_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const long long tiles = packed_tile_bound(a.T, a.R, kPT);
  if (tiles > 65535) return cudaErrorInvalidValue;
  dim3 grid((unsigned)a.Hq, (unsigned)tiles);
  sattn_packed_kernel<T><<<grid, 256, smem, s>>>((const T*)a.q, (const T*)a.k, (const T*)a.v, a.log_gate, a.cu,
                                                 (T*)a.out, a.R, a.T, a.Hq, a.Hk, a.D, a.st, a.scale);
  return cudaGetLastError();
}

}  // namespace

bool sattn_packed_tc_supported(int D, int dtype) {
  (void)D, (void)dtype;
  return false;
}

cudaError_t launch_sattn_packed(const PackedArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case SSD_F32: return packed_simt_t<float>(a, s);
    case SSD_BF16: return packed_simt_t<__nv_bfloat16>(a, s);
    case SSD_F16: return packed_simt_t<__half>(a, s);
  }
  return cudaErrorInvalidValue;
}

SSDB200_DEFINE_ERROR_FETCH(fetch_error_packed)

}  // namespace ssdb200
