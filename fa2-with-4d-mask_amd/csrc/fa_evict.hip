// Eviction from a K/V cache by key weight on gfx950 (MI355X).
//
// Of a sequence's n keys each kv-head keeps the last `recent` and, of the others, the need =
// keep - recent with the largest weight, ties to the lowest index, in ascending order.
//
//   select_kernel  a workgroup per (sequence, kv-head).  Weights become unsigned integers of
//                  the same order; the need-th largest is found digit by digit (11, 11, 10 bits:
//                  a histogram of the digit among the values that agree so far, then the bin
//                  the need-th falls into), then one scan in index order writes the kept indices
//                  and weights.
//   gather_kernel  copies the kept rows of K and V, a 16-byte piece per thread: it moves the
//                  bytes that are kept, once.
#include "fa_cache.h"
#include "fa_common.h"

namespace fa {
namespace {

constexpr int kThreads = 1024, kBins = 2048;

__device__ __forceinline__ int own_length(const EvictArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
}

// Larger weights to larger integers; -0 as 0, every NaN above +inf.
__device__ __forceinline__ uint32_t order(float w) {
  if (w != w) return ~0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of x over the lanes below this one, of the workgroup; *total: of all.
__device__ __forceinline__ uint32_t scan_before(uint32_t x, uint32_t* sums, uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t v = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(v, d);
    if (lane >= d) v += y;
  }
  __syncthreads();   // (sums may still be read)
  if (lane == 63) sums[wave] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const uint32_t y = sums[w];
    before += w < wave ? y : 0;
    all += y;
  }
  *total = all;
  return before + v - x;
}

__global__ __launch_bounds__(kThreads) void select_kernel(const EvictArgs a) {
  __shared__ uint32_t hist[kBins], sums[kThreads / 64], found[2];
  const int bk = blockIdx.x, b = bk / a.Hk, kvh = bk - b * a.Hk;
  const int tid = threadIdx.x;
  const float* w = a.kw + b * a.kwsb + kvh * a.kwsh;
  int64_t* idx = a.idx + (int64_t)bk * a.keep;
  float* kwo = a.kwo + (int64_t)bk * a.keep;
  const int n = own_length(a, b);
  const int last = max(0, n - a.recent);             // keys [last, n) are kept whatever their weight
  const int need = min(a.keep, n) - (n - last);      // of the keys [0, last)
  // thr: keys above it are kept, and `ties` of those equal to it
  uint32_t thr = 0, ties = 0;
  if (need >= last) {
    thr = 0;
    ties = last;        // all (order() of no weight but -NaN is 0; equal ones count as ties)
  } else if (need == 0) {
    thr = ~0u;
    ties = 0;
  } else {
    uint32_t known = 0, left = need;   // the left-th largest of those whose high digits are `thr`'s
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
      __syncthreads();
      for (int j = tid; j < last; j += kThreads) {
        const uint32_t u = order(w[j]);
        if ((u & known) == (thr & known)) atomicAdd(&hist[(u >> shift) & ((1u << bits) - 1)], 1u);
      }
      __syncthreads();
      // bins from the top: thread t has bins kBins - 1 - 2 t and the one below
      const uint32_t hi = hist[kBins - 1 - 2 * tid], lo = hist[kBins - 2 - 2 * tid];
      uint32_t total;
      const uint32_t above = scan_before(hi + lo, sums, &total);
      if (above < left && left <= above + hi + lo) {
        const bool top = left <= above + hi;
        found[0] = kBins - 1 - 2 * tid - (top ? 0 : 1);
        found[1] = left - above - (top ? 0 : hi);
      }
      __syncthreads();
      thr |= found[0] << shift;
      left = found[1];
      known |= ((1u << bits) - 1) << shift;
      __syncthreads();
    }
    ties = left;
  }
  // ---- in index order: thread t's keys are [t per, (t + 1) per) ---------------------------
  const int per = (n + kThreads - 1) / kThreads;
  const int j0 = min(tid * per, n), j1 = min(j0 + per, n);
  uint32_t eq = 0, gt = 0;
  for (int j = j0; j < j1; ++j) {
    if (j >= last) {
      ++gt;
    } else {
      const uint32_t u = order(w[j]);
      gt += u > thr;
      eq += u == thr;
    }
  }
  uint32_t all;
  const uint32_t eq_before = scan_before(eq, sums, &all);
  const uint32_t eq_mine = min(eq, ties - min(ties, eq_before));
  uint32_t at = scan_before(gt + eq_mine, sums, &all), seen = eq_before;
  for (int j = j0; j < j1; ++j) {
    bool kept = j >= last;
    if (!kept) {
      const uint32_t u = order(w[j]);
      kept = u > thr || (u == thr && seen++ < ties);
    }
    if (kept) {
      idx[at] = j;
      kwo[at] = w[j];
      ++at;
    }
  }
  for (int i = (int)all + tid; i < a.keep; i += kThreads) {   // places behind the last key
    idx[i] = -1;
    kwo[i] = 0.f;
  }
}

template <bool VEC>
__global__ __launch_bounds__(256) void gather_kernel(const EvictArgs a) {
  const int CH = VEC ? a.D / 8 : a.D;
  const int64_t n = (int64_t)a.B * a.Hk * a.keep * CH;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < n; x += (int64_t)gridDim.x * 256) {
    const int c = (int)(x % CH) * (VEC ? 8 : 1);
    const int64_t row = x / CH;
    const int i = (int)(row % a.keep), bk = (int)(row / a.keep);
    const int b = bk / a.Hk, kvh = bk - b * a.Hk;
    const int64_t j = a.idx[row];
    const int64_t src_k = b * a.ksb + j * a.kst + kvh * a.ksh + c, src_v = b * a.vsb + j * a.vst + kvh * a.vsh + c;
    const int64_t dst = b * a.osb + i * a.ost + kvh * a.osh + c;
    if constexpr (VEC) {
      u32x4 k = u32x4{0, 0, 0, 0}, v = k;
      if (j >= 0) {
        k = gload16((const uint16_t*)a.k + src_k);
        v = gload16((const uint16_t*)a.v + src_v);
      }
      gstore16((uint16_t*)a.ko + dst, k);
      gstore16((uint16_t*)a.vo + dst, v);
    } else {
      ((uint16_t*)a.ko)[dst] = j >= 0 ? ((const uint16_t*)a.k)[src_k] : (uint16_t)0;
      ((uint16_t*)a.vo)[dst] = j >= 0 ? ((const uint16_t*)a.v)[src_v] : (uint16_t)0;
    }
  }
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(select_kernel, dim3((unsigned)(a.B * a.Hk)), dim3(kThreads), 0, s, a);
  if (const hipError_t e = hipGetLastError()) return e;
  const int64_t n = ((int64_t)a.B * a.Hk * a.keep * (a.vec ? a.D / 8 : a.D) + 255) / 256;
  const dim3 grid((unsigned)min_i64(n, 1 << 20));
  if (a.vec) hipLaunchKernelGGL((gather_kernel<true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((gather_kernel<false>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace fa
