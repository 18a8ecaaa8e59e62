// Writing new tokens' K/V rows into a paged cache and reading sequences back.
//
// Both are copies, bound by HBM bandwidth: a row of D values of one (token, head) is handled by D / 8
// lanes, each with 16 bytes of BF16.  E4M3 rows get one power-of-two scale: e is the least integer
// with max|x| <= 448 * 2^e (448 is the largest E4M3 value), so x * 2^-e is exact and the conversion
// rounds once; E4M3 is itself a floating format, so a power of two as the scale costs no precision
// against max|x| / 448.  A value that is not finite does not enter the maximum; infinities become
// +-448 * 2^e and NaN stays NaN.
#include <cuda_fp8.h>

#include "paged.cuh"

namespace solattn {

namespace {

constexpr int kCopyThreads = 256;

// 448 * 2^e >= top for the least e, as the biased exponent e + 127 clamped to [0, 254]: with top =
// f * 2^x, 1 <= f < 2, that is x - 8 where f <= 1.75, else x - 7.
__device__ __forceinline__ int scale_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(0, min(254, e));
}

// 8 BF16 values * 2^-e -> 8 E4M3 codes (round to nearest even, saturating).
__device__ __forceinline__ uint2 to_e4m3(const uint4& raw, float f) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __uint_as_float(w[i] << 16) * f, hi = __uint_as_float(w[i] & 0xffff0000u) * f;
    c[i] = __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

__device__ __forceinline__ int seq_of_token(const CacheParams& p, int tok) {
  int lo = 0, hi = p.B;  // the last b with starts[b] <= tok
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(p.starts + mid) <= tok) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace

// Row (token, head) of K or V per group of D / 8 lanes.
template <int D, bool kE4m3>
__global__ void __launch_bounds__(kCopyThreads) cache_write_kernel(const CacheParams p) {
  constexpr int kLanes = D / 8;
  const int sub = threadIdx.x % kLanes;
  const int64_t rows = (int64_t)p.N * p.Hkv;
  const int64_t row = ((int64_t)blockIdx.x * kCopyThreads + threadIdx.x) / kLanes;
  const int z = blockIdx.y;
  const bool in = row < rows;
  const int tok = in ? (int)(row / p.Hkv) : 0, h = in ? (int)(row % p.Hkv) : 0;
  const uint4 raw = in ? __ldg(reinterpret_cast<const uint4*>(p.x[z] + (int64_t)tok * p.sT[z] + (int64_t)h * p.sH[z]) + sub)
                       : make_uint4(0, 0, 0, 0);
  const int b = seq_of_token(p, tok);
  const int start = __ldg(p.starts + b), next = __ldg(p.starts + b + 1);
  bool ok = in && tok >= start && tok < next;  // rows behind the last sequence are left out
  int64_t dst = 0;
  if (ok) {
    const int pos = __ldg(p.lengths + b) - next + tok;
    int page = -1;
    if (pos >= 0 && pos < (p.width << p.page_shift))
      page = __ldg(p.table + (int64_t)b * p.width + (pos >> p.page_shift));
    if (start < 0 || next > p.N || page < 0 || page >= p.npages) {
      note(p.status, kStatusBadIndex);
      ok = false;
    } else {
      dst = (((int64_t)page * p.Hkv + h) << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
    }
  }
  if constexpr (!kE4m3) {
    if (ok) reinterpret_cast<uint4*>(p.pages[z] + dst * D * 2)[sub] = raw;
  } else {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = fabsf(__uint_as_float(w[i] << 16)), hi = fabsf(__uint_as_float(w[i] & 0xffff0000u));
      if (lo < INFINITY) top = fmaxf(top, lo);
      if (hi < INFINITY) top = fmaxf(top, hi);
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int e = scale_exponent(top);
    if (ok) {
      const uint2 c = to_e4m3(raw, __uint_as_float((uint32_t)(254 - e) << 23));
      reinterpret_cast<uint2*>(p.pages[z] + dst * D)[sub] = c;
      if (sub == 0) p.scale[z][dst] = (uint8_t)e;
    }
  }
}

// Row (sequence, token, head) of K or V per group of D / 8 lanes; zeros behind a sequence's end.
template <int D, bool kE4m3>
__global__ void __launch_bounds__(kCopyThreads) cache_read_kernel(const CacheParams p) {
  constexpr int kLanes = D / 8;
  const int sub = threadIdx.x % kLanes;
  const int64_t row = ((int64_t)blockIdx.x * kCopyThreads + threadIdx.x) / kLanes;
  const int z = blockIdx.y;
  if (row >= (int64_t)p.B * p.tokens * p.Hkv) return;
  const int h = (int)(row % p.Hkv);
  const int64_t bt = row / p.Hkv;
  const int b = (int)(bt / p.tokens), pos = (int)(bt % p.tokens);
  int L = __ldg(p.lengths + b);
  const int cap = p.width << p.page_shift;
  if (L < 0 || L > cap) {
    note(p.status, kStatusBadIndex);
    L = L < 0 ? 0 : cap;
  }
  uint4 out = make_uint4(0, 0, 0, 0);
  if (pos < L) {
    const int page = __ldg(p.table + (int64_t)b * p.width + (pos >> p.page_shift));
    if (page < 0 || page >= p.npages) {
      note(p.status, kStatusBadIndex);
    } else {
      const int64_t src = (((int64_t)page * p.Hkv + h) << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
      if constexpr (!kE4m3) {
        out = __ldg(reinterpret_cast<const uint4*>(p.pages[z] + src * D * 2) + sub);
      } else {
        const uint2 c = __ldg(reinterpret_cast<const uint2*>(p.pages[z] + src * D) + sub);
        const float f = e8m0_value(p.scale[z][src]);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t two = ((i & 2) ? c.y : c.x) >> (16 * (i & 1));
          w[i] = pack_bf16(e4m3_value(two & 0xffu) * f, e4m3_value((two >> 8) & 0xffu) * f);
        }
        out = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  reinterpret_cast<uint4*>(p.y[z] + row * D)[sub] = out;
}

cudaError_t launch_cache_write(const CacheParams& p, int D, cudaStream_t stream) {
  const int64_t threads = (int64_t)p.N * p.Hkv * (D / 8);
  const dim3 grid((unsigned)((threads + kCopyThreads - 1) / kCopyThreads), 2);
  if (D == 128) {
    if (p.scale[0]) cache_write_kernel<128, true><<<grid, kCopyThreads, 0, stream>>>(p);
    else cache_write_kernel<128, false><<<grid, kCopyThreads, 0, stream>>>(p);
  } else {
    if (p.scale[0]) cache_write_kernel<64, true><<<grid, kCopyThreads, 0, stream>>>(p);
    else cache_write_kernel<64, false><<<grid, kCopyThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

cudaError_t launch_cache_read(const CacheParams& p, int D, cudaStream_t stream) {
  const int64_t threads = (int64_t)p.B * p.tokens * p.Hkv * (D / 8);
  const dim3 grid((unsigned)((threads + kCopyThreads - 1) / kCopyThreads), 2);
  if (D == 128) {
    if (p.scale[0]) cache_read_kernel<128, true><<<grid, kCopyThreads, 0, stream>>>(p);
    else cache_read_kernel<128, false><<<grid, kCopyThreads, 0, stream>>>(p);
  } else {
    if (p.scale[0]) cache_read_kernel<64, true><<<grid, kCopyThreads, 0, stream>>>(p);
    else cache_read_kernel<64, false><<<grid, kCopyThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace solattn
