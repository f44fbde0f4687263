// Eviction from a K/V cache by key weight on gfx950 (MI355X).
//
// Of a sequence's n keys each kv-head keeps the last `recent` and, of the others, the need =
// keep - recent with the largest weight, ties to the lowest index, in ascending order.
//
//   evict_kernel  a.nw workgroups of 16 waves per (sequence, kv-head).  Each finds the whole
//                 selection: weights become unsigned integers of the same order; the need-th
//                 largest is found digit by digit (12, 10, 10 bits: a histogram of the digit among
//                 the values that agree so far, then the bin the need-th falls into); one pass in
//                 index order then counts the kept keys.  Each copies its share of the kept rows
//                 of K and V.
//
// The selection is a chain of dependent steps on little data (64 KB of weights for 16384 keys):
// its latency counts, not its work, so that every workgroup of a head repeats it rather than wait
// for one that writes indices to memory and for a second launch to read them.  The weights stay in
// LDS, a stretch of 64-key pieces per wave; the order within a wave comes from ballots.  The copies move the bytes that are kept, once, 16 bytes per lane.
#include "fa_cache.h"
#include "fa_common.h"

namespace fa {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 4096;

__device__ __forceinline__ int own_length(const EvictArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
}

// Larger weights to larger integers; -0 as 0, every NaN above +inf.  No weight's is 0 or
// kKept, the order of the most recent keys, above all.
constexpr uint32_t kKept = ~0u;
__device__ __forceinline__ uint32_t order(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t x = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return w != w ? kKept - 1 : x;
}

// Sum of x over the lanes up to this one (data moved between lanes by the VALU, not through LDS).
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8: rows of 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // lane 15 of a row to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // lane 31 to rows 2 and 3
  return x;
}

// Sum of x over the threads below this one, of the workgroup.
__device__ __forceinline__ uint32_t scan_before(uint32_t x, uint32_t* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t v = wave_scan(x);
  if (lane == 63) sums[wave] = v;   // (last read before the barrier that ended the step before)
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) before += w < wave ? sums[w] : 0;
  return before + v - x;
}

// CAP: weights of a cache that LDS holds (n <= CAP); 0: any number, read again for each step.
// The loops over them stay rolled: unrolled over registers (32 pieces a lane) every step was new
// code, run once, and the instruction fetches took 7 us a step.
template <int CAP, bool VEC>
__global__ __launch_bounds__(kThreads) void evict_kernel(const EvictArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t hist[kBins];
  __shared__ uint32_t sums[kWaves], found[2];
  __shared__ int list[kEvictShare];
  __shared__ uint32_t keys[CAP > 0 ? CAP : 1];
  const int bk = blockIdx.x / a.nw, part = blockIdx.x - bk * a.nw;
  const int b = bk / a.Hk, kvh = bk - b * a.Hk;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* w = a.kw + b * a.kwsb + kvh * a.kwsh;
  const int n = own_length(a, b);
  const int last = max(0, n - a.recent);             // keys [last, n) are kept whatever their weight
  // this wave's stretch: pieces [0, np) of 64 keys from k0 on
  constexpr int U = 4;
  const int np = ((n + kThreads - 1) / kThreads + U - 1) / U * U, k0 = wave * np * 64;
  auto order_at = [&](int j, float x) __attribute__((always_inline)) -> uint32_t {
    return j < last ? order(x) : (j < n ? kKept : 0u);
  };
  if constexpr (CAP > 0) {   // (each wave reads what it wrote; np <= CAP / 1024)
#pragma unroll 4
    for (int i = 0; i < np; i += U) {
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = w[min(k0 + (i + u) * 64 + lane, n - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = k0 + (i + u) * 64 + lane;
        keys[j] = order_at(j, x[u]);
      }
    }
  }
  // fn(key, its order) for every piece, in order
  auto pieces = [&](auto&& fn) __attribute__((always_inline)) {
#pragma unroll 1
    for (int i = 0; i < np; i += U) {
      uint32_t x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = k0 + (i + u) * 64 + lane;
        if constexpr (CAP > 0) x[u] = keys[j];
        else x[u] = order_at(j, w[min(j, n - 1)]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) fn(k0 + (i + u) * 64 + lane, x[u]);
    }
  };
  // keys above thr are kept, and `ties` of those equal to it
  uint32_t thr = 0, ties = 0;
  if (n - last == a.keep) {
    thr = kKept - 1;                     // the most recent ones alone
  } else if (n > a.keep) {
    // the left-th largest weight of those whose high digits are `thr`'s
    uint32_t known = 0, left = a.keep - (n - last);
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 20 : (pass == 1 ? 10 : 0);
      const uint32_t digit = pass == 0 ? 0xfffu : 0x3ffu;
      *(u32x4*)(hist + 4 * tid) = u32x4{0, 0, 0, 0};
      __syncthreads();
      pieces([&](int, uint32_t u) __attribute__((always_inline)) {
        // (weights only: keys past n, and the most recent ones, would all meet in one bin)
        if (u - 1 < kKept - 1 && ((u ^ thr) & known) == 0) atomicAdd(&hist[(u >> shift) & digit], 1u);
      });
      __syncthreads();
      // bins from the top: thread t has the four from kBins - 1 - 4 t down
      const u32x4 h = *(const u32x4*)(hist + kBins - 4 - 4 * tid);
      uint32_t above = scan_before((h[0] + h[1]) + (h[2] + h[3]), sums);
      if (above < left && left <= above + (h[0] + h[1]) + (h[2] + h[3])) {
        int bin = 3;
        while (left > above + h[bin]) above += h[bin--];
        found[0] = kBins - 4 - 4 * tid + bin;
        found[1] = left - above;
      }
      __syncthreads();
      thr |= found[0] << shift;
      left = found[1];
      known |= digit << shift;
    }
    ties = left;
  }
  // ---- kept keys and ties of the waves' stretches, those before this one's added up -----------
  uint32_t gt = 0, eq = 0;   // of the wave, the same in every lane
  pieces([&](int, uint32_t u) __attribute__((always_inline)) {
    gt += __popcll(__builtin_amdgcn_ballot_w64(u > thr));
    eq += __popcll(__builtin_amdgcn_ballot_w64(u == thr));
  });
  const int share = (a.keep + a.nw - 1) / a.nw, i0 = part * share, i1 = min(i0 + share, a.keep);
  for (int i = tid; i < share; i += kThreads) list[i] = -1;
  __syncthreads();   // (hist is free)
  if (lane == 0) {
    hist[wave] = gt;
    hist[kWaves + wave] = eq;
  }
  __syncthreads();
  uint32_t before = 0, seen = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    before += i < wave ? hist[i] : 0;
    seen += i < wave ? hist[kWaves + i] : 0;
  }
  // ---- this workgroup's places [i0, i1), filled by the waves whose keys go there ---------------
  int at = (int)__builtin_amdgcn_readfirstlane(before + min(seen, ties)) - i0;
  seen = __builtin_amdgcn_readfirstlane(seen);
  const int end = at + (int)(gt + min(eq, ties - min(seen, ties)));
  if (end > 0 && at < share) {
    const uint64_t below = (1ull << lane) - 1;
    pieces([&](int j, uint32_t u) __attribute__((always_inline)) {
      bool kept = u > thr;
      const uint64_t te = __builtin_amdgcn_ballot_w64(u == thr);
      if (te != 0) {
        kept = kept || (u == thr && seen + __popcll(te & below) < ties);
        seen += __popcll(te);
      }
      const uint64_t ke = __builtin_amdgcn_ballot_w64(kept);
      const int place = at + __popcll(ke & below);
      if (kept && (uint32_t)place < (uint32_t)share) list[place] = j;
      at += __popcll(ke);
    });
  }
  __syncthreads();
  const int64_t o0 = (int64_t)bk * a.keep;
  for (int i = i0 + tid; i < i1; i += kThreads) {
    const int j = list[i - i0];
    a.idx[o0 + i] = j;
    a.kwo[o0 + i] = j < 0 ? 0.f : w[j];
  }
  // ---- the rows -------------------------------------------------------------------------
  const int CH = VEC ? a.D / 8 : a.D, rpp = max(kThreads / CH, 1), lanes = min(CH, kThreads);
  const int r0 = tid / CH;
  if (r0 >= rpp) return;
  const uint16_t* kp = (const uint16_t*)a.k + b * a.ksb + kvh * a.ksh;
  const uint16_t* vp = (const uint16_t*)a.v + b * a.vsb + kvh * a.vsh;
  uint16_t* ko = (uint16_t*)a.ko + b * a.osb + kvh * a.osh;
  uint16_t* vo = (uint16_t*)a.vo + b * a.osb + kvh * a.osh;
  for (int ch = tid - r0 * CH; ch < CH; ch += lanes) {
    const int c = ch * (VEC ? 8 : 1);
    if constexpr (VEC) {
      constexpr int U = 4;   // rows in flight
      for (int i = i0 + r0; i < i1; i += U * rpp) {
        u32x4 x[U], y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = i + u * rpp < i1 ? list[i + u * rpp - i0] : -1;
          x[u] = gload16_if(j >= 0, kp + (int64_t)max(j, 0) * a.kst + c);
          y[u] = gload16_if(j >= 0, vp + (int64_t)max(j, 0) * a.vst + c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i + u * rpp < i1) {
            gstore16(ko + (int64_t)(i + u * rpp) * a.ost + c, x[u]);
            gstore16(vo + (int64_t)(i + u * rpp) * a.ost + c, y[u]);
          }
      }
    } else {
      for (int i = i0 + r0; i < i1; i += rpp) {
        const int j = list[i - i0];
        ko[(int64_t)i * a.ost + c] = j >= 0 ? kp[(int64_t)j * a.kst + c] : (uint16_t)0;
        vo[(int64_t)i * a.ost + c] = j >= 0 ? vp[(int64_t)j * a.vst + c] : (uint16_t)0;
      }
    }
  }
}

template <int CAP> hipError_t launch_c(const EvictArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.B * a.Hk * a.nw)), block(kThreads);
  if (a.vec) hipLaunchKernelGGL((evict_kernel<CAP, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((evict_kernel<CAP, false>), grid, block, 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t s) {
  if (a.Tk <= 8192) return launch_c<8192>(a, s);
  if (a.Tk <= 32768) return launch_c<32768>(a, s);
  return launch_c<0>(a, s);
}

}  // namespace fa
