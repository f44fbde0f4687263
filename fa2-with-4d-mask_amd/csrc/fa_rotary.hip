// Rotary positions of several axes on gfx950 (MI355X): column pair i of token (b, t) turns by
// positions[axis(i), b, t] * freq[i], queries and keys in one launch.
//
// The angle: freq / 2 pi as a 64-bit binary fraction of a turn, times the position modulo
// 2^64.  Whole turns fall off by themselves and the rest is good to 2^-31 of a turn at positions
// below 2^32 (a product in fp32 has lost 0.06 rad at position 10^6).  Cosines and sines are made
// once per token, into LDS, for all of its heads.
//
// What bounds it: reading and writing queries and keys once, 8192 tokens of 40 heads of 128 at 5.4
// TB/s.  The outputs are stored past the caches (a launch writes more than the L2s hold, and
// lines kept for them push out the inputs: 7996 tokens of 32 heads of 80 24.6 -> 17.0 us).
#include "fa_cache.h"
#include "fa_common.h"

namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;   // head dims up to 256

// V columns per piece: 8 (16 bytes) or 1; kTok tokens per workgroup.
template <typename T, int V, bool ADJ, int kTok>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const RotaryArgs a) {
  __shared__ float cs[2][kTok][kMaxPairs];   // cosines, sines
  const int64_t tok0 = (int64_t)blockIdx.x * kTok, ntok = (int64_t)a.B * a.T;
  const int nt = (int)min_i64(kTok, ntok - tok0);
  const int tid = threadIdx.x;
  for (int x = tid; x < nt * a.R2; x += kThreads) {
    const int tk = x / a.R2, i = x - tk * a.R2;
    const int64_t bt = tok0 + tk;
    const int64_t b = bt / a.T, t = bt - b * a.T;
    int ax = 0;
#pragma unroll
    for (int e = 0; e < kRotaryAxes - 1; ++e) ax += e < a.naxes - 1 && i >= a.ends[e] ? 1 : 0;
    const int64_t at = ax * a.psa + b * a.psb + t * a.pst;
    const int64_t pos = a.pos64 ? ((const int64_t*)a.pos)[at] : ((const int32_t*)a.pos)[at];
    // freq / 2 pi in two doubles: 1 / 2 pi = kTurn + kTurnLo to 2^-110
    constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnLo = -0x1.6b01ec5417056p-57;
    const double f = (double)a.freq[i], turns = f * kTurn;
    const double lo = fma(f, kTurnLo, fma(f, kTurn, -turns));
    float s, c;
    if (fabs(turns) < 0x1p28) {
      const double part = turns - rint(turns);   // exact, in [-1/2, 1/2]
      const uint64_t turn = (uint64_t)(int64_t)rint((part < 0.5 ? part : -0.5) * 0x1p64) + (uint64_t)(int64_t)rint(lo * 0x1p64);
      const int32_t top = (int32_t)((turn * (uint64_t)pos) >> 32);   // in [-1/2, 1/2) turns, times 2^32
      sincospif((float)top * 0x1p-31f, &s, &c);
    } else {
      s = c = __builtin_nanf("");   // no frequency: past 2^30, infinite or NaN
    }
    cs[0][tk][i] = c;
    cs[1][tk][i] = s * a.sign;
  }
  __syncthreads();

  // pieces of a head: NR turned (two at once without ADJ: columns c and c + R2), NC copied
  const int NR = (ADJ ? 2 * a.R2 : a.R2) / V, NC = (a.D - 2 * a.R2) / V, NP = NR + NC;
  const int H = a.Hq + a.Hk, step = kThreads / NP;
  const int pc = tid % NP;
  int h = tid / NP, tk = 0;
  if (h >= step) return;
  auto settle = [&]() __attribute__((always_inline)) {
    while (h >= H) {
      h -= H;
      ++tk;
    }
  };
  settle();
  typedef T TV __attribute__((ext_vector_type(V)));
  const bool turned = pc < NR;
  const int c0 = turned ? pc * V : 2 * a.R2 + (pc - NR) * V;
  const int c1 = ADJ ? (V == 1 && turned ? c0 ^ 1 : c0) : (turned ? c0 + a.R2 : c0);
  // kFly pieces at a time: their loads go out together
  constexpr int kFly = 2;
  while (tk < nt) {
    TV x0[kFly], x1[kFly];
    T* dst[kFly];
    int at[kFly];
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      at[u] = tk;
      if (tk < nt) {
        const int64_t bt = tok0 + tk;
        const int64_t b = bt / a.T, t = bt - b * a.T;
        const bool isq = h < a.Hq;
        const int hh = isq ? h : h - a.Hq;
        const T* src = isq ? (const T*)a.q + b * a.qsb + t * a.qst + hh * a.qsh : (const T*)a.k + b * a.ksb + t * a.kst + hh * a.ksh;
        dst[u] = isq ? (T*)a.qo + b * a.qosb + t * a.qost + hh * a.qosh : (T*)a.ko + b * a.kosb + t * a.kost + hh * a.kosh;
        x0[u] = *(const TV*)(src + c0);
        if (!ADJ || V == 1) x1[u] = *(const TV*)(src + c1);
      }
      h += step;
      settle();
    }
#pragma unroll
    for (int u = 0; u < kFly; ++u) {
      if (at[u] >= nt) continue;
      if (!turned) {
        __builtin_nontemporal_store(x0[u], (TV*)(dst[u] + c0));
      } else if constexpr (ADJ && V == 1) {
        const float co = cs[0][at[u]][c0 >> 1], si = cs[1][at[u]][c0 >> 1];
        const float x = (float)x0[u][0], y = (float)x1[u][0];
        dst[u][c0] = (T)fmaf(x, co, c0 & 1 ? y * si : -(y * si));
      } else if constexpr (ADJ) {
        TV y;
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float co = cs[0][at[u]][(c0 + e) >> 1], si = cs[1][at[u]][(c0 + e) >> 1];
          const float p = (float)x0[u][e], q = (float)x0[u][e + 1];
          y[e] = (T)fmaf(p, co, -(q * si));
          y[e + 1] = (T)fmaf(q, co, p * si);
        }
        __builtin_nontemporal_store(y, (TV*)(dst[u] + c0));
      } else {
        TV y0, y1;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float co = cs[0][at[u]][c0 + e], si = cs[1][at[u]][c0 + e];
          const float p = (float)x0[u][e], q = (float)x1[u][e];
          y0[e] = (T)fmaf(p, co, -(q * si));
          y1[e] = (T)fmaf(q, co, p * si);
        }
        __builtin_nontemporal_store(y0, (TV*)(dst[u] + c0));
        __builtin_nontemporal_store(y1, (TV*)(dst[u] + c1));
      }
    }
  }
}

template <typename T, int TOK> hipError_t launch_n(const RotaryArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)a.B * a.T + TOK - 1) / TOK)), block(kThreads);
  if (a.vec && a.adjacent) hipLaunchKernelGGL((rotary_kernel<T, 8, true, TOK>), grid, block, 0, s, a);
  else if (a.vec) hipLaunchKernelGGL((rotary_kernel<T, 8, false, TOK>), grid, block, 0, s, a);
  else if (a.adjacent) hipLaunchKernelGGL((rotary_kernel<T, 1, true, TOK>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((rotary_kernel<T, 1, false, TOK>), grid, block, 0, s, a);
  return hipGetLastError();
}

// One token per workgroup where the grid is small or a token is 8 KB or more, else two: 32 tokens of
// 40 heads of 128 3.7 us (two 4.6), 8192 of them 30.9 (32.4); 7996 tokens of 32 heads of 80, 5 KB
// each, 20.4 (17.0).
template <typename T> hipError_t launch_t(const RotaryArgs& a, hipStream_t s) {
  const bool one = (int64_t)a.B * a.T <= 1024 || (int64_t)(a.Hq + a.Hk) * a.D * 2 >= 8192;
  return one ? launch_n<T, 1>(a, s) : launch_n<T, 2>(a, s);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, int dtype, hipStream_t s) {
  return dtype == 0 ? launch_t<bf16>(a, s) : launch_t<f16>(a, s);
}

}  // namespace fa
