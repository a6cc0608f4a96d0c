// paged_decode.cu - attention of one query token for each request over the paged 8-bit cache
// (paged.cu): SelectiveMHA.step's attention (modules/selective_attention.py:399-404) with
// grouped heads, requests of different lengths and keys and values held as codes.
//   s_j = scale * q . (code_j * k_scale) + (j < n - 1 ? log_gate_j : 0),  out = softmax(s) . v
// A key whose log-gate is -inf drops out, whatever its codes hold; so does one whose table entry
// is not a page of the cache. A request of length 0 gets zeros.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "sattn_tiles.cuh"

namespace ssdb200 {
namespace {

// CTA = (request, query head); a group of D/8 lanes owns one key.
constexpr int kDecWarps = 8;

template <typename T, typename C>
__global__ void __launch_bounds__(kDecWarps * 32) paged_decode_kernel(
    const T* __restrict__ q, const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
    const float* __restrict__ ks, const float* __restrict__ vs, const float* __restrict__ gc,
    const int* __restrict__ table, const int* __restrict__ lengths, T* __restrict__ out, long long num_pages, int W,
    int Hq, int Hk, int page_shift, int D, float scale) {
  __shared__ float sm_m[kDecWarps], sm_l[kDecWarps];
  __shared__ float sm_acc[kDecWarps][256];
  const int r = blockIdx.y, hq = blockIdx.x, hk = hq / (Hq / Hk);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int page = 1 << page_shift;
  const int n = (int)min((long long)max(lengths[r], 0), (long long)W << page_shift);
  const int lpk = D >> 3, kpw = 32 / lpk, grp = lane / lpk, sub = lane - grp * lpk;
  float qv[8], acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  load8<T>(q + ((long long)r * Hq + hq) * D + sub * 8, qv);
  float m = -INFINITY, l = 0.f;
  for (int j0 = warp * kpw; j0 < n; j0 += kDecWarps * kpw) {
    const int j = j0 + grp;
    float kv[8], vv[8], d = 0.f, ksc = 0.f, vsc = 0.f, g = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) kv[e] = vv[e] = 0.f;
    if (j < n) {
      const int id = table[(long long)r * W + (j >> page_shift)];
      if (id >= 0 && id < num_pages) {
        const long long ph = (long long)id * Hk + hk, row = ph * page + (j & (page - 1));
        Code<C>::unpack8(*reinterpret_cast<const uint2*>(kc + row * D + sub * 8), kv);
        Code<C>::unpack8(*reinterpret_cast<const uint2*>(vc + row * D + sub * 8), vv);
        ksc = ks[ph];
        vsc = vs[ph];
        g = gc && j < n - 1 ? gc[row] : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) d = fmaf(qv[e], kv[e], d);
    for (int off = 1; off < lpk; off <<= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
    if (g == -INFINITY) continue;
    const float s = d * ksc * scale + g;
    const float mn = fmaxf(m, s);
    const float a = m == -INFINITY ? 0.f : expf(m - mn);
    const float p = expf(s - mn);
    l = l * a + p;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(p * vsc, vv[e], acc[e] * a);
    m = mn;
  }
  __syncwarp();
  // merge the warp's key groups, then the warps
  for (int off = lpk; off < 32; off <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, off), l2 = __shfl_xor_sync(0xffffffffu, l, off);
    const float mn = fmaxf(m, m2);
    const float f1 = m == -INFINITY ? 0.f : expf(m - mn), f2 = m2 == -INFINITY ? 0.f : expf(m2 - mn);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * f1 + __shfl_xor_sync(0xffffffffu, acc[e], off) * f2;
    l = l * f1 + l2 * f2;
    m = mn;
  }
  if (grp == 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sm_acc[warp][sub * 8 + e] = acc[e];
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
  __syncthreads();
  for (int d = tid; d < D; d += kDecWarps * 32) {
    float M = -INFINITY, ls = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, sm_m[w]);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float f = sm_m[w] == -INFINITY ? 0.f : expf(sm_m[w] - M);
      ls = fmaf(sm_l[w], f, ls);
      o = fmaf(sm_acc[w][d], f, o);
    }
    out[((long long)r * Hq + hq) * D + d] = from_f32<T>(ls == 0.f ? 0.f : o / ls);
  }
}

template <typename T, typename C>
cudaError_t decode_t(const PagedCache& c, const void* q, const int* table, const int* lengths, void* out, int R, int W,
                     int Hq, float scale, cudaStream_t s) {
  dim3 grid((unsigned)Hq, (unsigned)R);
  paged_decode_kernel<T, C><<<grid, kDecWarps * 32, 0, s>>>((const T*)q, c.k, c.v, c.ks, c.vs, c.gate, table, lengths,
                                                            (T*)out, c.pages, W, Hq, c.nkv, c.page_shift, c.D, scale);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_decode(const PagedCache& c, const void* q, const int* table, const int* lengths, void* out,
                                int R, int W, int Hq, float scale, int dtype, void* workspace, cudaStream_t s) {
  (void)workspace;
  const bool e4m3 = c.code == SSD_CODE_E4M3;
  switch (dtype) {
    case SSD_F32:
      return e4m3 ? decode_t<float, E4M3>(c, q, table, lengths, out, R, W, Hq, scale, s)
                  : decode_t<float, Int8>(c, q, table, lengths, out, R, W, Hq, scale, s);
    case SSD_BF16:
      return e4m3 ? decode_t<__nv_bfloat16, E4M3>(c, q, table, lengths, out, R, W, Hq, scale, s)
                  : decode_t<__nv_bfloat16, Int8>(c, q, table, lengths, out, R, W, Hq, scale, s);
    case SSD_F16:
      return e4m3 ? decode_t<__half, E4M3>(c, q, table, lengths, out, R, W, Hq, scale, s)
                  : decode_t<__half, Int8>(c, q, table, lengths, out, R, W, Hq, scale, s);
  }
  return cudaErrorInvalidValue;
}

size_t paged_decode_workspace(int R, int W, int Hq, int Hk, int page_shift, int D) {
  (void)R, (void)W, (void)Hq, (void)Hk, (void)page_shift, (void)D;
  return 0;
}

}  // namespace ssdb200
