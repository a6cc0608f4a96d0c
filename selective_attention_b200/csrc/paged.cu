// paged.cu - the paged 8-bit key/value cache of served selective attention: block tables and
// slot maps from request lengths (plan), quantised writes (append) and reads back (read).
// The reference keeps a dense full-precision cache of one capacity per batch
// (inference/selective_attn_cache.py:10-42); this is its form for many requests at once.
//
// A page holds page_size consecutive tokens of one request, for every key head:
//   codes (num_pages, Hkv, page_size, D) 8-bit, scale (num_pages, Hkv) fp32, so that
//   value = code * scale[page, head]; log-gates (num_pages, Hkv, page_size) fp32.
// Slot s is token s % page_size of page s / page_size.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "sattn_tiles.cuh"

namespace ssdb200 {
namespace {

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------
// One launch; a CTA writes the slots and positions of kPlanTokens new tokens. Each CTA sums all
// requests' new tokens and pages by itself (a block scan over pairs, which stop at 2^31), which
// for some hundred requests costs less than a second launch or a wait between CTAs would; the
// requests that begin in or reach into its tokens leave an entry at their first token there, and
// a running maximum over the tokens finds each token's entry. A page's table entry is written by
// the token at its first position, so no two threads write one entry and none is read that
// another writes; so only a request whose tokens are all among the T that are planned is served, or it
// would hold pages that its table does not name. Those that are come first, so that a sum that has stopped
// is never theirs. Bound by latency and each CTA's scan: 256 requests
// of one token each take 4.4 us (captured in a graph), 384 prompts with 393k tokens (386 CTAs) 8.9.
constexpr int kPlanThreads = 256;
constexpr int kPlanPer = 4;
constexpr int kPlanTokens = kPlanThreads * kPlanPer;

struct PlanEntry {
  int r, len, cu, pages_before;  // request, cached tokens, its first new token, pages given before it
  int served;
};

// New tokens and pages, each at most 2^31.
struct PlanSum {
  unsigned tokens, pages;
};
__device__ __forceinline__ unsigned add_up_to(unsigned a, unsigned b) {
  const unsigned c = a + b;
  return c < a ? 0x80000000u : min(c, 0x80000000u);
}
__device__ __forceinline__ PlanSum operator+(PlanSum a, PlanSum b) {
  return PlanSum{add_up_to(a.tokens, b.tokens), add_up_to(a.pages, b.pages)};
}
__device__ __forceinline__ PlanSum shfl_up(PlanSum v, int off) {
  return PlanSum{__shfl_up_sync(0xffffffffu, v.tokens, off), __shfl_up_sync(0xffffffffu, v.pages, off)};
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(
    const int* __restrict__ lengths, const int* __restrict__ new_lengths, int* table, const int* __restrict__ free_pages,
    const long long* __restrict__ free_state, int* __restrict__ lengths_out, int* __restrict__ cu_new,
    long long* __restrict__ slots, int* __restrict__ positions, long long* __restrict__ free_state_out, int R, int W,
    long long F, long long T, int page_shift) {
  __shared__ PlanEntry ent[kPlanTokens];
  __shared__ short start[kPlanTokens];
  __shared__ PlanSum wsum[kPlanThreads / 32];
  __shared__ int wmax[kPlanThreads / 32];
  __shared__ long long s_given;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long t0 = (long long)blockIdx.x * kPlanTokens;
  const long long t1 = min(t0 + kPlanTokens, T);
  const int page = 1 << page_shift;
  const long long head = free_state[0], tail = free_state[1];
  const long long avail = min(tail - head, F);
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) start[tid + i * kPlanThreads] = -1;
  if (tid == 0) s_given = 0;
  __syncthreads();
  PlanSum carry{0u, 0u};
  for (int r0 = 0; r0 < R; r0 += kPlanThreads) {
    const int r = r0 + tid;
    int len = 0, add = 0, need = 0;
    bool fits = true;
    if (r < R) {
      len = max(lengths[r], 0);
      add = max(new_lengths[r], 0);
      const long long end = ((long long)len + add + page - 1) >> page_shift;
      fits = end <= W;
      need = fits ? (int)(end - (((long long)len + page - 1) >> page_shift)) : 0;
    }
    PlanSum incl{(unsigned)add, (unsigned)need};
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const PlanSum o = shfl_up(incl, off);
      if (lane >= off) incl = o + incl;
    }
    if (lane == 31) wsum[warp] = incl;
    PlanSum excl = shfl_up(incl, 1);
    if (lane == 0) excl = PlanSum{0u, 0u};
    __syncthreads();
    PlanSum before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      const PlanSum x = wsum[w];
      if (w < warp) before = before + x;
      all = all + x;
    }
    carry = all;
    incl = before + incl;
    const long long upto = incl.pages, cu = (before + excl).tokens;
    const bool served = r < R && fits && (need == 0 || upto <= avail) && (add == 0 || cu + add <= T);
    if (r < R) {
      if (add > 0 && cu < t1 && cu + add > t0) {
        const int at = (int)(max(cu, t0) - t0);
        ent[at] = PlanEntry{r, len, (int)cu, (int)(upto - need), served};
        start[at] = (short)at;
      }
      if (blockIdx.x == 0) {
        lengths_out[r] = served ? len + add : lengths[r];
        cu_new[r + 1] = (int)min(incl.tokens, 0x7fffffffu);
        if (served && need > 0) atomicMax((unsigned long long*)&s_given, (unsigned long long)upto);
      }
    }
    __syncthreads();  // wsum is rewritten, ent and start are read
  }
  if (blockIdx.x == 0 && tid == 0) {
    cu_new[0] = 0;
    free_state_out[0] = head + s_given;
    free_state_out[1] = tail;
  }
  // the entry of each token: running maximum of start over kPlanPer tokens a thread
  int own[kPlanPer], m = -1;
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    m = max(m, (int)start[tid * kPlanPer + i]);
    own[i] = m;
  }
  int incl = m;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl = max(incl, o);
  }
  if (lane == 31) wmax[warp] = incl;
  __syncthreads();
  int prev = __shfl_up_sync(0xffffffffu, incl, 1);
  if (lane == 0) prev = -1;
  for (int w = 0; w < warp; ++w) prev = max(prev, wmax[w]);
  const long long total = carry.tokens;
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const long long t = t0 + tid * kPlanPer + i;
    if (t >= T) break;
    const int at = max(own[i], prev);
    long long slot = -1;
    int pos = 0;
    if (t < total && at >= 0) {
      const PlanEntry e = ent[at];
      pos = e.len + (int)(t - e.cu);
      if (e.served) {
        const int pg = pos >> page_shift, has = (e.len + page - 1) >> page_shift, in = pos & (page - 1);
        int id;
        if (pg < has) {
          id = table[(long long)e.r * W + pg];
        } else {
          id = free_pages[(head + e.pages_before + (pg - has)) % F];
          if (in == 0) table[(long long)e.r * W + pg] = id;
        }
        slot = (long long)id * page + in;
      }
    }
    slots[t] = slot;
    positions[t] = pos;
  }
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// CTA = (block of `per` tokens, key head, K or V). A segment is a run of tokens with consecutive
// slots in one page; the CTA in whose block it begins writes all of it (up to page - 1 tokens
// past its block), so each page and head has one writer. The rows are loaded once, all loads in
// flight together, and stay in registers as they came (the rows past the first kAppHeld passes
// are read again); then the largest finite magnitude of each row, the segment's scale from its
// rows and the page's old scale, and the codes of the rows and, where the scale grew, of the
// page's older rows. 16k tokens of 8 heads of 128 (fp16 to e4m3, K and V) take 51 us back to back and 57 with cold
// caches, bound by instructions (about 300 for 16 elements of a warp's two rows) between the barriers; the 65 MB
// that they are and the 33 MB of codes would take 15 at the copy rate.
constexpr int kAppThreads = 256;
constexpr int kAppRows = 256;  // rows of one CTA: per + page - 1 <= 255
constexpr int kAppHeld = 8;

// Eight elements as they lie in memory.
template <typename T> struct Raw8 {
  uint4 w[sizeof(T) / 2];
};
template <typename T, bool VEC>
__device__ __forceinline__ void load_raw(const T* p, Raw8<T>& x) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) x.w[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T* d = reinterpret_cast<T*>(x.w);
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = p[e];
  }
}
template <typename T>
__device__ __forceinline__ void floats(const Raw8<T>& x, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = __uint_as_float(x.w[i].x), v[4 * i + 1] = __uint_as_float(x.w[i].y);
      v[4 * i + 2] = __uint_as_float(x.w[i].z), v[4 * i + 3] = __uint_as_float(x.w[i].w);
    }
  } else {
    const float2 a = unpack2<T>(x.w[0].x), b = unpack2<T>(x.w[0].y), c = unpack2<T>(x.w[0].z), d = unpack2<T>(x.w[0].w);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
  }
}

template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(kAppThreads) paged_append_kernel(
    const T* __restrict__ kx, const T* __restrict__ vx, const float* __restrict__ gate,
    const long long* __restrict__ slots, unsigned char* kc, unsigned char* vc, float* ks, float* vs, float* gc,
    long long num_pages, int H, int page_shift, int D, long long Tn, long long k_ts, long long k_hs, long long v_ts,
    long long v_hs, int per) {
  __shared__ int smax[kAppRows];           // at a segment's first row: its largest magnitude (as bits), then its scale
  __shared__ float inverse[kAppRows];      // 1 / the scale
  __shared__ float ratio[kAppRows];        // of a page that grew: old / new scale
  __shared__ short grown[kAppRows];        // first rows of the segments whose pages hold older rows and grew
  __shared__ short head_of[kAppRows];      // row -> its segment's first row, -1 if the row is not this CTA's
  __shared__ long long s_slot[kAppRows];
  __shared__ int wlast[kAppThreads / 32];  // last segment start of each warp's rows
  __shared__ int s_rows, s_grown;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, page = 1 << page_shift;
  const int h = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const T* x = is_v ? vx + h * v_hs : kx + h * k_hs;
  const long long ts = is_v ? v_ts : k_ts;
  unsigned char* codes = is_v ? vc : kc;
  float* scale = is_v ? vs : ks;
  const long long t0 = (long long)blockIdx.x * per;
  const int most = (int)min((long long)per + page - 1, Tn - t0);  // rows that can be this CTA's
  if (tid == 0) s_rows = 0, s_grown = 0;
  // thread = row: where segments begin, then a running maximum of the beginnings
  {
    long long s = -1, before = -2;
    if (tid < most) {
      s = slots[t0 + tid];
      if (t0 + tid > 0) before = slots[t0 + tid - 1];
    }
    const bool in = s >= 0 && s < num_pages << page_shift;
    const bool starts = in && ((s & (page - 1)) == 0 || before != s - 1);
    int m = starts ? tid : -1;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, m, off);
      if (lane >= off) m = max(m, o);
    }
    if (lane == 31) wlast[warp] = m;
    __syncthreads();
    for (int w = 0; w < warp; ++w) m = max(m, wlast[w]);
    const int first = in && m < per ? m : -1;  // (m = -1: begun in an earlier block)
    head_of[tid] = (short)first;
    s_slot[tid] = s;
    smax[tid] = 0;
    const unsigned mine = __ballot_sync(0xffffffffu, first >= 0);
    if (lane == 0 && mine) atomicMax(&s_rows, warp * 32 + 32 - __clz(mine));
  }
  __syncthreads();
  const int rows = s_rows;
  if (rows == 0) return;
  const int lpr = D >> 3, lshift = 31 - __clz(lpr);  // lanes per row, 8 elements each
  const int sub = tid & (lpr - 1), grp = tid >> lshift, ngrp = kAppThreads >> lshift;
  Raw8<T> held[kAppHeld];
#pragma unroll
  for (int u = 0; u < kAppHeld; ++u) {
    const int i = u * ngrp + grp;
    if (i < rows && head_of[i] >= 0) load_raw<T, VEC>(x + (t0 + i) * ts + sub * 8, held[u]);
  }
  // (all lanes of a warp are in the same number of steps: the bound is rounded up to whole passes)
  const int passes = (rows + ngrp - 1) / ngrp;
  auto row_max = [&](int i, const Raw8<T>& raw) {
    float m = 0.f;
    if (i < rows && head_of[i] >= 0) {
      float v[8];
      floats<T>(raw, v);
      // infinities and NaN do not set the scale (a maximum passes over NaN)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
      if (m == INFINITY) {
        m = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
      }
    }
    for (int off = 1; off < lpr; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    // (magnitudes order as their bits do)
    if (i < rows && head_of[i] >= 0 && sub == 0) atomicMax(&smax[head_of[i]], __float_as_int(m));
  };
#pragma unroll
  for (int u = 0; u < kAppHeld; ++u)
    if (u < passes) row_max(u * ngrp + grp, held[u]);
  for (int u = kAppHeld; u < passes; ++u) {
    const int i = u * ngrp + grp;
    Raw8<T> raw;
    if (i < rows && head_of[i] >= 0) load_raw<T, VEC>(x + (t0 + i) * ts + sub * 8, raw);
    row_max(i, raw);
  }
  __syncthreads();
  if (tid < rows && head_of[tid] == tid) {
    const long long s = s_slot[tid];
    const bool older = (s & (page - 1)) != 0;  // a page that begins here has no older rows
    float* sp = scale + (s >> page_shift) * H + h;
    const float was = older ? *sp : 0.f;
    const float now = fmaxf(was, __int_as_float(smax[tid]) * Code<C>::kPerMost);
    *sp = now;
    smax[tid] = __float_as_int(now);
    inverse[tid] = 1.0f / now;
    if (older && now > was) {
      ratio[tid] = __fdiv_rn(was, now);
      grown[atomicAdd(&s_grown, 1)] = (short)tid;
    }
  }
  __syncthreads();
  auto encode = [&](int i, const Raw8<T>& raw) {
    const int first = i < rows ? head_of[i] : -1;
    if (first < 0) return;
    const long long s = s_slot[i];
    const long long row = ((s >> page_shift) * H + h) * page + (s & (page - 1));
    float v[8];
    floats<T>(raw, v);
    // The codes are those of the quotient x / scale. A product with the reciprocal gives the same code but
    // next to the middle between two; there, and where the reciprocal is no normal number, divide.
    const float sc = __int_as_float(smax[first]), inv = inverse[first];
    float y[8];
    bool divide = !(inv < 1e37f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = v[e] * inv;
      divide |= Code<C>::unsure(y[e]);
    }
    if (divide) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = sc > 0.f ? __fdiv_rn(v[e], sc) : 0.f;
    }
    *reinterpret_cast<uint2*>(codes + row * D + sub * 8) = Code<C>::pack8(y);
    if (!is_v && gate && sub == 0) gc[row] = gate[(t0 + i) * H + h];
  };
#pragma unroll
  for (int u = 0; u < kAppHeld; ++u)
    if (u < passes) encode(u * ngrp + grp, held[u]);
  for (int u = kAppHeld; u < passes; ++u) {
    const int i = u * ngrp + grp;
    if (i >= rows || head_of[i] < 0) continue;
    Raw8<T> raw;
    load_raw<T, VEC>(x + (t0 + i) * ts + sub * 8, raw);
    encode(i, raw);
  }
  // older rows of the pages whose scale grew
  for (int k = 0; k < s_grown; ++k) {
    const int i = grown[k];
    const long long s = s_slot[i];
    const int older = (int)(s & (page - 1));
    unsigned char* base = codes + ((s >> page_shift) * H + h) * (long long)page * D;
    for (int j = grp; j < older; j += ngrp) {
      uint2* p = reinterpret_cast<uint2*>(base + (long long)j * D + sub * 8);
      float v[8];
      Code<C>::unpack8(*p, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= ratio[i];
      *p = Code<C>::pack8(v);
    }
  }
}

// ---------------------------------------------------------------------------
// read: values of the given slots, (N, H, D) for K and V; slots outside the cache give zeros.
// One thread reads 8 codes and writes 8 values, fp32 as a whole 32-byte sector. Bound by writing them: 16k slots
// of 8 heads of 128 (33 MB read, 132 MB written) take 33 us with cold caches and 28 back to back, where half of what
// is written stays in L2; at the copy rate they would take 25.
// ---------------------------------------------------------------------------
constexpr int kReadThreads = 256;
constexpr int kReadItems = 4;  // of a thread, their codes all in flight

template <typename T, typename C>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(
    const long long* __restrict__ slots, const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc,
    const float* __restrict__ ks, const float* __restrict__ vs, T* __restrict__ ko, T* __restrict__ vo,
    long long num_pages, int H, int page_shift, int D, long long n, int per) {
  const int lshift = 31 - __clz(D >> 3), page = 1 << page_shift;
  const bool is_v = blockIdx.y != 0;
  const unsigned char* codes = is_v ? vc : kc;
  const float* scale = is_v ? vs : ks;
  T* out = is_v ? vo : ko;
  const long long first = (long long)blockIdx.x * per;              // the CTA's slots, `per` of them
  const unsigned row = (unsigned)H << lshift;                       // items of a slot
  const unsigned items = (unsigned)min((long long)per, n - first) * row;
  const bool wide = (reinterpret_cast<uintptr_t>(out) & 31u) == 0;
  for (unsigned i0 = threadIdx.x; i0 < items; i0 += kReadItems * kReadThreads) {
    uint2 w[kReadItems];
    float sc[kReadItems];
#pragma unroll
    for (int u = 0; u < kReadItems; ++u) {
      const unsigned i = i0 + u * kReadThreads;
      w[u] = make_uint2(0u, 0u);
      sc[u] = 0.f;
      if (i < items) {
        const unsigned t = i / row, in = i - t * row, h = in >> lshift, sub = in & ((1u << lshift) - 1u);
        const long long s = slots[first + t];
        if (s >= 0 && s < num_pages << page_shift) {
          const long long ph = (s >> page_shift) * H + h;
          w[u] = *reinterpret_cast<const uint2*>(codes + (ph * page + (s & (page - 1))) * D + sub * 8);
          sc[u] = scale[ph];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kReadItems; ++u) {
      const unsigned i = i0 + u * kReadThreads;
      if (i >= items) break;
      float v[8];
      Code<C>::unpack8(w[u], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= sc[u];
      store8_wide<T>(out + (first * row + i) * 8, v, wide);
    }
  }
}

template <typename T, typename C>
cudaError_t append_t(const PagedCache& c, const void* k, const void* v, const float* gate, const long long* slots,
                     long long n, long long k_ts, long long k_hs, long long v_ts, long long v_hs, cudaStream_t s) {
  // Few tokens: small blocks, so that many CTAs share them. Many: 128 tokens, which a CTA's threads hold
  // in registers for head_dim 128 (a page of 64 each: 63 us instead of 59 for 16k tokens of 8 heads, events included).
  const int per = n * c.nkv <= 2048 ? 4 : 128;
  const bool vec = (reinterpret_cast<uintptr_t>(k) % 16 == 0) && (reinterpret_cast<uintptr_t>(v) % 16 == 0) &&
                   (k_ts * sizeof(T)) % 16 == 0 && (k_hs * sizeof(T)) % 16 == 0 && (v_ts * sizeof(T)) % 16 == 0 &&
                   (v_hs * sizeof(T)) % 16 == 0;
  const long long blocks = (n + per - 1) / per;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  dim3 grid((unsigned)blocks, (unsigned)c.nkv, 2);
  auto fn = vec ? paged_append_kernel<T, C, true> : paged_append_kernel<T, C, false>;
  fn<<<grid, kAppThreads, 0, s>>>((const T*)k, (const T*)v, gate, slots, c.k, c.v, c.ks, c.vs, c.gate, c.pages,
                                  c.nkv, c.page_shift, c.D, n, k_ts, k_hs, v_ts, v_hs, per);
  return cudaGetLastError();
}

template <typename T, typename C>
cudaError_t read_t(const PagedCache& c, const long long* slots, long long n, void* ko, void* vo, cudaStream_t s) {
  // slots of a CTA: about kReadItems items a thread
  const long long row = (long long)c.nkv * (c.D >> 3);
  const long long per = row >= kReadItems * kReadThreads ? 1 : kReadItems * kReadThreads / row;
  const long long blocks = (n + per - 1) / per;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  dim3 grid((unsigned)blocks, 2);
  paged_read_kernel<T, C><<<grid, kReadThreads, 0, s>>>(slots, c.k, c.v, c.ks, c.vs, (T*)ko, (T*)vo, c.pages, c.nkv,
                                                        c.page_shift, c.D, n, (int)per);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_plan(const int* lengths, const int* new_lengths, int* table, const int* free_pages,
                              const long long* free_state, int* lengths_out, int* cu_new, long long* slots,
                              int* positions, long long* free_state_out, int R, int W, long long F, long long T,
                              int page_shift, cudaStream_t s) {
  long long blocks = (T + kPlanTokens - 1) / kPlanTokens;
  if (blocks < 1) blocks = 1;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  paged_plan_kernel<<<(unsigned)blocks, kPlanThreads, 0, s>>>(lengths, new_lengths, table, free_pages, free_state,
                                                              lengths_out, cu_new, slots, positions, free_state_out, R,
                                                              W, F, T, page_shift);
  return cudaGetLastError();
}

#define PAGED_DISPATCH(fn, ...)                                                     \
  do {                                                                              \
    const bool e4m3 = c.code == SSD_CODE_E4M3;                                      \
    switch (dtype) {                                                                \
      case SSD_F32: return e4m3 ? fn<float, E4M3>(__VA_ARGS__) : fn<float, Int8>(__VA_ARGS__); \
      case SSD_BF16: return e4m3 ? fn<__nv_bfloat16, E4M3>(__VA_ARGS__) : fn<__nv_bfloat16, Int8>(__VA_ARGS__); \
      case SSD_F16: return e4m3 ? fn<__half, E4M3>(__VA_ARGS__) : fn<__half, Int8>(__VA_ARGS__); \
    }                                                                               \
    return cudaErrorInvalidValue;                                                   \
  } while (0)

cudaError_t launch_paged_append(const PagedCache& c, const void* k, const void* v, const float* gate,
                                const long long* slots, long long n, long long k_ts, long long k_hs, long long v_ts,
                                long long v_hs, int dtype, cudaStream_t s) {
  PAGED_DISPATCH(append_t, c, k, v, gate, slots, n, k_ts, k_hs, v_ts, v_hs, s);
}

cudaError_t launch_paged_read(const PagedCache& c, const long long* slots, long long n, void* ko, void* vo, int dtype,
                              cudaStream_t s) {
  PAGED_DISPATCH(read_t, c, slots, n, ko, vo, s);
}

}  // namespace ssdb200
