// Eviction from a K/V cache by key weight on gfx950 (MI355X).
//
// Of a sequence's n keys each kv-head keeps the last `recent` and, of the others, the need =
// keep - recent with the largest weight, ties to the lowest index, in ascending order.
//
//   evict_kernel  a.nw workgroups of 16 waves per (sequence, kv-head).  Each finds the whole
//                 selection: weights become unsigned integers of the same order; the need-th
//                 largest is found digit by digit (12, 10, 10 bits: a histogram of the digit among
//                 the values that agree so far, then the bin the need-th falls into); one pass then
//                 turns the comparisons with it into bits, 64 keys to a lane, whose counts give every
//                 kept key its place.  Each copies its share of the kept rows of K and V.
//
// The selection is a chain of dependent steps on little data (64 KB of weights for 16384 keys):
// its latency counts, not its work, so that every workgroup of a head repeats it rather than wait
// for one that writes indices to memory and for a second launch to read them.  The weights stay in
// LDS, a stretch of 64-key pieces per wave.  The copies move the bytes that are kept, once, 16 bytes
// per lane.
//
// Measured: B1 Tk 16384 Hk8 D128 keep 4096 16.4 us, 33.7 MB of rows and weights at 2.1 TB/s (head
// dim 8, the selection almost alone, 13.0; the most recent ones alone, without it, 11.4, of which
// a launch takes some 5); B16 Tk 3001 Hk4 D96 keep 1500 19.7 us, 74 MB at 3.7 TB/s; B64 Tk 4096 Hk8 D128
// keep 2048 224 us, 4.8 TB/s.  Past the LDS every workgroup goes over all weights four times: B1 Tk
// 131072 Hk8 D128 keep 32768 130 us, about half of it the copies.
#include "fa_cache.h"
#include "fa_common.h"

namespace fa {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 4096;

__device__ __forceinline__ int own_length(const EvictArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
}

// Larger weights to larger integers, up to kTop; -0 as 0, every NaN above +inf.  No weight's has a
// first digit (12 bits) of 0: 0 stands for keys that are not chosen by their weight.
constexpr uint32_t kTop = ~0u;
__device__ __forceinline__ uint32_t order(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t x = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return w != w ? kTop : x;
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
// code, run once, and the instruction fetches took 7 us a step.  With 32768 a workgroup has a CU's
// LDS to itself; 8192 leaves room for two.
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
  auto order_at = [&](int j, float x) __attribute__((always_inline)) -> uint32_t { return j < last ? order(x) : 0u; };
  // fn(order) for every piece
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
      for (int u = 0; u < U; ++u) fn(x[u], i + u);
    }
  };
  // orders above thr are kept, and `ties` of those equal to it
  const bool select = n > a.keep && n - last < a.keep;
  uint32_t thr = n > a.keep ? kTop : 0u, ties = 0;   // (the most recent ones alone, or all)
  if (select) *(u32x4*)(hist + 4 * tid) = u32x4{0, 0, 0, 0};
  __syncthreads();
  if (CAP > 0 || select) {   // (each wave reads what it wrote; np <= CAP / 1024)
    constexpr int LU = 8;    // loads in flight
#pragma unroll 1
    for (int i = 0; i < np; i += LU) {
      float x[LU];
#pragma unroll
      for (int u = 0; u < LU; ++u) x[u] = w[min(k0 + (i + u) * 64 + lane, n - 1)];
#pragma unroll
      for (int u = 0; u < LU; ++u)
        if (i + u < np) {
          const int j = k0 + (i + u) * 64 + lane;
          const uint32_t o = order_at(j, x[u]);
          if constexpr (CAP > 0) keys[j] = o;
          if (select && o) atomicAdd(&hist[o >> 20], 1u);
        }
    }
  }
  if (select) {
    // the left-th largest of those whose high digits are `thr`'s
    uint32_t known = 0, left = a.keep - (n - last);
    thr = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 20 : (pass == 1 ? 10 : 0);
      if (pass) {   // (order 0's first digit is no weight's)
        *(u32x4*)(hist + 4 * tid) = u32x4{0, 0, 0, 0};
        __syncthreads();
        pieces([&](uint32_t u, int) __attribute__((always_inline)) {
          if ((u & known) == thr) atomicAdd(&hist[(u >> shift) & 0x3ffu], 1u);
        });
      }
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
      known |= (pass ? 0x3ffu : 0xfffu) << shift;
    }
    ties = left;
  }
  // ---- which keys: lane i has the bits of piece c0 + i, kept whatever and equal to thr ----------
  uint64_t more = 0, same = 0;
  auto bits = [&](int c0) __attribute__((always_inline)) {
    more = same = 0;
    const int end = min(np - c0, 64);
#pragma unroll 1
    for (int i = 0; i < end; i += U) {
      uint32_t x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = k0 + (c0 + i + u) * 64 + lane;
        if constexpr (CAP > 0) x[u] = keys[j];
        else x[u] = order_at(j, w[min(j, n - 1)]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint64_t g = __builtin_amdgcn_ballot_w64(x[u] > thr), e = __builtin_amdgcn_ballot_w64(x[u] == thr);
        const bool mine = lane == i + u;
        more = mine ? g : more;
        same = mine ? e : same;
      }
    }
    const int j = k0 + (c0 + lane) * 64;
    auto below = [&](int m) { return m >= 64 ? ~0ull : (m <= 0 ? 0ull : (1ull << m) - 1); };
    if (lane < end) more |= below(n - j) & ~below(last - j);   // the most recent
  };
  // ---- kept keys and ties of the waves' stretches, those before this one's added up -----------
  uint32_t gt = 0, eq = 0;
#pragma unroll 1
  for (int c0 = 0; c0 < np; c0 += 64) {
    bits(c0);
    gt += __popcll(more);
    eq += __popcll(same);
  }
  gt = wave_scan(gt);
  eq = wave_scan(eq);
  const int share = (a.keep + a.nw - 1) / a.nw, i0 = part * share, i1 = min(i0 + share, a.keep);
  for (int i = tid; i < share; i += kThreads) list[i] = -1;
  if (lane == 63) {   // (hist is free: last read before the barrier before this)
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
  const int first = (int)(before + min(seen, ties)) - i0;   // the wave's own places [first, end)
  const int end = (int)(before + __builtin_amdgcn_readlane((int)gt, 63) +
                        min(seen + __builtin_amdgcn_readlane((int)eq, 63), ties)) - i0;
#pragma unroll 1
  for (int c0 = 0; c0 < np && first < share && end > 0; c0 += 64) {
    if constexpr (CAP == 0) bits(c0);   // (else one round: the bits are there)
    const uint32_t ng = __popcll(more), ne = __popcll(same);
    const uint32_t ig = wave_scan(ng), ie = wave_scan(ne), e = seen + ie - ne;
    const uint32_t took = min(e, ties);
    uint32_t take = min(e + ne, ties) - took;   // the first ones of this piece's ties
    uint64_t kept = more;
    if (take == ne) kept |= same;
    else
      for (uint64_t r = same; take; --take, r &= r - 1) kept |= r & (0 - r);
    const int at = (int)(before + ig - ng + took) - i0;   // the piece's first place
    uint64_t todo = __builtin_amdgcn_ballot_w64(kept != 0 && at < share && at + (int)__popcll(kept) > 0);
    while (todo) {
      const int p = __builtin_ctzll(todo);
      todo &= todo - 1;
      const uint64_t m = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(kept >> 32), p) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)kept, p);
      const int place = __builtin_amdgcn_readlane(at, p) + __popcll(m & ((1ull << lane) - 1));
      if ((m >> lane) & 1 && (uint32_t)place < (uint32_t)share) list[place] = k0 + (c0 + p) * 64 + lane;
    }
    before += __builtin_amdgcn_readlane((int)ig, 63);
    seen += __builtin_amdgcn_readlane((int)ie, 63);
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
