// Key weights of many query rows on gfx950 (MI355X): for every own key the sum of its
// probability over the rows of its kv-head's group,
//   kw[b, kvh, j] += sum_{h in group, i} exp2(log2(e) scale (q_i k_j + score_ij) - lse_i),
// from the LSE a forward left.  (Few rows: fa_prefix.hip, whose forward keeps its logits.)
//
//   key_weights_kernel   a workgroup of 4 waves per (256 keys (128 at head dim 256), part of
//                        the row tiles, kv-head, sequence).  A wave keeps its 64 (32) keys as MFMA
//                        operands in registers and walks the rows of the group, 64 (32) at a time
//                        from LDS, where the workgroup's waves share them: S^T = K Q^T leaves 16
//                        keys of one row per lane and fragment, which become probabilities and are
//                        added in place; the sum over the lanes (rows) comes once, at the end.
//                        Sums are fp32.
//   key_weights_sum_kernel  adds the parts, in order (deterministic), where few key blocks
//                        leave CUs idle and the row tiles are cut into parts.
//   far_rows_kernel      with a score: rows whose LSE is so large (masks of the type's lowest
//                        value in all of the row) that it no longer holds the sum's logarithm get
//                        their largest raw logit and their sum anew; others leave at once.
//
// What bounds it: the exponentials (6 VALU instructions per MFMA at head dim 128, an exp at a quarter
// of the rate) and the MFMAs, in turn: B1 Tq8192 Tk8192 Hq32/8 D128 causal 399 us, 137 GFLOP at 344
// TFLOP/s, the MFMA busy a third of the time (each wave with its own loads of the rows: 758 us,
// the L1s' rate).  More than two waves per SIMD do not fit beside the keys (three: spills, 5 % slower).
#include "fa_cache.h"
#include "fa_common.h"
#include "fa_pipe.h"

namespace fa {
namespace {

using pipe::IC;

constexpr int kWaves = 4;
template <int D> constexpr int frags() { return D == 256 ? 1 : 2; }       // 32-key fragments per wave
template <int D> constexpr int tile_rows() { return D == 256 ? 32 : 64; }
// Chunk swizzle of the row tiles: 16 rows' reads of one chunk hit 64 distinct banks.
template <int D> __device__ __forceinline__ int swz(int r) { return pipe::swz_q<D == 64 ? 64 : 128>(r); }

__device__ __forceinline__ int own_length(const KeyWArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
}

// A row of a kv-head's group, r = g Tq + tq.
struct Row {
  int g, tq;
};

template <typename T, int DS> __device__ __forceinline__ void load_q(const KeyWArgs& a, u32x4 (&x)[DS], int b, int h, int tq, int hf) {
  load_row(x, (const T*)a.q + b * a.qsb + h * a.qsh + (int64_t)tq * a.qst + hf * 8, a.Dv);
}

// K rows [k0, k0 + 32) as the MFMA's A operand; rows past n read zeros.
template <typename T, int DS> __device__ __forceinline__ void load_keys(const KeyWArgs& a, const T* kp, int k0, int n, int l32, int hf,
                                                                         typename Vec8<T>::type (&kf)[DS]) {
  const int rows = min(n - k0, 32);
  const bool ok = rows > 0;
  const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)(kp + (ok ? (int64_t)k0 * a.kst : 0)), (short)0,
                                                    ok ? (int)((int64_t)(rows - 1) * a.kst * 2 + 2 * a.Dv) : 0, 0x00020000);
  const uint32_t off = (uint32_t)(l32 * a.kst * 2) + (uint32_t)(hf * 16);
#pragma unroll
  for (int ds = 0; ds < DS; ++ds)
    kf[ds] = as_vec8<T>((u32x4)__builtin_amdgcn_raw_buffer_load_b128(rs, off + 32 * ds, 16 * ds < a.Dv ? 0 : kNoRec, 0));
}

// Keep bits (bit 8 gi + e <-> key k0 + 8 gi + 4 hf + e) of a row whose first lim keys count.
__device__ __forceinline__ uint32_t in_row(int lim, int k0, int hf) {
  const int n = lim - (k0 + 4 * hf);
  return n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1u);
}
__device__ __forceinline__ uint32_t mask_bits(const KeyWArgs& a, const uint8_t* mrow, int k0, int hf, int n) {
  uint32_t w = 0;
  const int k = k0 + 4 * hf;
  if (a.mask4 && k0 + 32 <= n) {
    uint32_t x[4];
#pragma unroll
    for (int gi = 0; gi < 4; ++gi) x[gi] = *(const uint32_t*)(mrow + k + 8 * gi);
#pragma unroll
    for (int gi = 0; gi < 4; ++gi)
#pragma unroll
      for (int e = 0; e < 4; ++e) w |= ((x[gi] >> (8 * e)) & 0xffu) != 0 ? 1u << (8 * gi + e) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) w |= mrow[min(k + 8 * (i >> 2) + (i & 3), n - 1)] != 0 ? 1u << (8 * (i >> 2) + (i & 3)) : 0u;
  }
  return w;
}
__device__ __forceinline__ f32x16 scores(const float* srow, int k0, int hf, int n, float sign) {
  f32x16 x;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = sign * srow[min(k0 + 8 * (i >> 2) + 4 * hf + (i & 3), n - 1)];
  return x;
}

template <typename T, int D, bool MASK, bool SCORE>
__global__ __launch_bounds__(kWaves * 64, 2) void key_weights_kernel(const KeyWArgs a) {
  using V8 = typename Vec8<T>::type;
  constexpr int DS = D / 16, NF = frags<D>(), CH = D / 8, RT = tile_rows<D>();
  constexpr int NU = RT * CH / (kWaves * 64);   // 16-byte chunks of a tile per thread
  __shared__ __align__(16) char tiles[2][RT * D * 2];
  __shared__ float lses[2][RT];
  // causal: the first key blocks have the most rows, so all of them start first
  const int n_per = a.B * a.Hk * a.ns, kb = blockIdx.x / n_per, W = blockIdx.x - kb * n_per;
  const int sp = W % a.ns, bk = W / a.ns;
  const int b = bk / a.Hk, kvh = bk - b * a.Hk;
  const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = own_length(a, b);
  const int kb0 = kb * kWaves * NF * 32, k0 = kb0 + wave * NF * 32;   // the workgroup's first key, this wave's
  const int R = a.G * a.Tq, nt = (R + RT - 1) / RT;
  const float c2 = a.scale_log2;
  const uint32_t neg = a.qsign < 0.f ? 0x80008000u : 0u;

  f32x16 acc[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) acc[f] = f32x16{};
  if (kb0 < n) {
    const T* kp = (const T*)a.k + b * a.ksb + kvh * a.ksh;
    V8 kf[NF][DS];
#pragma unroll
    for (int f = 0; f < NF; ++f) load_keys<T, DS>(a, kp, k0 + 32 * f, n, l32, hf, kf[f]);
    // Tile t starts at row (g, tq) of the group, and the tile ns behind it dg heads and dt rows on.
    struct Tile {
      int t, g, tq;
    };
    const int dg = RT * a.ns / a.Tq, dt = RT * a.ns - dg * a.Tq;
    auto behind = [&](Tile x) __attribute__((always_inline)) -> Tile {
      x.t += a.ns;
      x.g += dg;
      x.tq += dt;
      if (x.tq >= a.Tq) {
        x.tq -= a.Tq;
        ++x.g;
      }
      return x;
    };
    // causal: the first tile from x on some row of which sees key kb0 (a tile of one head's last
    // rows and the next one's first: always)
    auto seen = [&](Tile x) __attribute__((always_inline)) -> Tile {
      if (a.causal)
        while (x.t < nt && x.tq + RT <= a.Tq && x.tq + RT <= kb0) x = behind(x);
      return x;
    };
    auto row_in = [&](const Tile& x, int i) __attribute__((always_inline)) -> Row {   // row i (past R: the last)
      if (x.t * RT + i >= R) return {a.G - 1, a.Tq - 1};
      int g = x.g, tq = x.tq + i;
      if (a.Tq >= RT) {
        if (tq >= a.Tq) {
          tq -= a.Tq;
          ++g;
        }
      } else {
        const int y = tq / a.Tq;
        g += y;
        tq -= y * a.Tq;
      }
      return {g, tq};
    };
    // A tile's rows and LSEs, loaded while the one before is worked on.  Rows of one head, as almost
    // always, lie `off` from its first (with every row's address made on its own the kernel issued 13
    // VALU instructions per MFMA, now 8.3: B1 Tq8192 Tk8192 Hq32/8 D128 causal 461 -> 399 us).
    const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
    constexpr int RS = kWaves * 64 / CH;   // rows between a thread's chunks
    const int col = 8 * c < a.Dv ? 8 * c : 0;
    int64_t off[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) off[u] = (r0 + u * RS) * a.qst + col;
    u32x4 x[NU];
    float e = 0.f;
    auto load_tile = [&](const Tile& t) __attribute__((always_inline)) {
      const T* qp = (const T*)a.q + b * a.qsb;
      const float* lp = a.lse + ((int64_t)b * a.Hq + kvh * a.G) * a.Tq;
      if (t.tq + RT <= a.Tq) {
        const T* src = qp + (kvh * a.G + t.g) * a.qsh + (int64_t)t.tq * a.qst;
#pragma unroll
        for (int u = 0; u < NU; ++u) x[u] = gload16(src + off[u]);
        if (threadIdx.x < RT) e = lp[(int64_t)t.g * a.Tq + t.tq + threadIdx.x];
      } else {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const Row q = row_in(t, r0 + u * RS);
          x[u] = gload16(qp + (kvh * a.G + q.g) * a.qsh + (int64_t)q.tq * a.qst + col);
        }
        if (threadIdx.x < RT) {
          const Row q = row_in(t, threadIdx.x);
          // rows past R: +inf, as a row without a kept key
          e = t.t * RT + (int)threadIdx.x < R ? lp[(int64_t)q.g * a.Tq + q.tq] : kPosInf;
        }
      }
    };
    auto keep_tile = [&](int buf) __attribute__((always_inline)) {
      if (neg != 0 || a.Dv < D) {
#pragma unroll
        for (int u = 0; u < NU; ++u) x[u] = zero_unless(8 * c < a.Dv, x[u] ^ neg);
      }
#pragma unroll
      for (int u = 0; u < NU; ++u)
        lds_write16(tiles[buf] + (r0 + u * RS) * 2 * D + ((c ^ swz<D>(r0 + u * RS)) * 16), x[u]);
      if (threadIdx.x < RT) lses[buf][threadIdx.x] = e;
    };
    // probabilities of 32 rows from LDS (this lane's: row q) added to the keys' sums; EDGE: some are
    // dropped
    auto add = [&](auto EDGEc, const char* rows, const Row& q, float lse) __attribute__((always_inline)) {
      const int h = kvh * a.G + q.g;
      V8 qf[DS];
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) qf[ds] = as_vec8<T>(lds_read16(rows + l32 * 2 * D + ((2 * ds + hf) ^ swz<D>(l32)) * 16));
      float sub = 0.f, mul = 1.f;
      if constexpr (SCORE) {
        if (far_max(lse) && lse != kPosInf) {
          const float* ml = a.far_ml + 2 * (((int64_t)b * a.Hq + h) * a.Tq + q.tq);
          sub = ml[0];
          lse = 0.f;
          mul = 1.0f / ml[1];
        }
      }
      // (with a mask or score a fragment at a time: their bits and rows need the registers)
      constexpr int NS = MASK || SCORE ? 1 : NF;
#pragma unroll
      for (int f0 = 0; f0 < NF; f0 += NS) {
        f32x16 s[NS];
#pragma unroll
        for (int f = 0; f < NS; ++f) {
          s[f] = f32x16{};
          if constexpr (SCORE)
            s[f] = scores(a.score + b * a.ssb + h * a.ssh + (int64_t)q.tq * a.ssq, k0 + 32 * (f0 + f), hf, n, a.qsign);
        }
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
          for (int f = 0; f < NS; ++f) s[f] = mfma32(kf[f0 + f][ds], qf[ds], s[f]);
        if constexpr (decltype(EDGEc)::value) {
          const int lim = a.causal ? min(n, q.tq + 1) : n;
#pragma unroll
          for (int f = 0; f < NS; ++f) {
            const int kk = k0 + 32 * (f0 + f);
            uint32_t w = in_row(lim, kk, hf);
            if constexpr (MASK) w &= mask_bits(a, a.mask + b * a.msb + h * a.msh + (int64_t)q.tq * a.msq, kk, hf, n);
#pragma unroll
            for (int j = 0; j < 16; ++j)
              s[f][j] = (w >> (8 * (j >> 2) + (j & 3))) & 1u ? (a.zero_scale ? 0.f : s[f][j]) : kNegInf;
          }
        }
#pragma unroll
        for (int f = 0; f < NS; ++f)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if constexpr (SCORE) acc[f0 + f][j] += exp2_fast(fmaf(s[f][j] - sub, c2, -lse)) * mul;
            else acc[f0 + f][j] += exp2_fast(fmaf(s[f][j], c2, -lse));
          }
        if constexpr (NS < NF) __builtin_amdgcn_sched_barrier(0);
      }
    };
    const bool edge = MASK || a.zero_scale || k0 + 32 * NF > n;
    const int g0 = RT * sp / a.Tq;
    Tile t = seen(Tile{sp, g0, RT * sp - g0 * a.Tq});
    if (t.t < nt) {
      load_tile(t);
      keep_tile(0);
    }
    __syncthreads();
    for (int buf = 0; t.t < nt; buf ^= 1) {
      const Tile now = t;
      t = seen(behind(t));
      if (t.t < nt) load_tile(t);
      if (k0 < n) {
#pragma unroll
        for (int i = 0; i < RT; i += 32) {
          const bool one = now.tq + i + 32 <= a.Tq;   // rows of one head
          if (now.t * RT + i >= R || (a.causal && one && now.tq + i + 32 <= k0)) continue;
          const char* rows = tiles[buf] + i * 2 * D;   // (32 rows on: the same swizzle)
          const float lse = lses[buf][i + l32];
          const Row q = one ? Row{now.g, now.tq + i + l32} : row_in(now, i + l32);
          if (edge || (a.causal && !(one && now.tq + i >= k0 + 32 * NF - 1))) add(IC<1>{}, rows, q, lse);
          else add(IC<0>{}, rows, q, lse);
        }
      }
      if (t.t < nt) keep_tile(buf ^ 1);   // (its last readers: before the barrier before this one)
      __syncthreads();
    }
  }
  // The sums over a half's 32 lanes, half of the values leaving a lane in every step: lane l32 ends
  // with that of fragment l32 / 16, value l32 % 16.
  const bool up = lane & 16;
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float mine = NF == 2 && up ? acc[NF - 1][j] : acc[0][j], other = NF == 2 && !up ? acc[NF - 1][j] : acc[0][j];
    v[j] = mine + __shfl_xor(other, 16);
  }
#pragma unroll
  for (int d = 8; d > 0; d >>= 1)
#pragma unroll
    for (int j = 0; j < d; ++j) {
      const bool high = lane & d;
      const float mine = high ? v[j + d] : v[j], other = high ? v[j] : v[j + d];
      v[j] = mine + __shfl_xor(other, d);
    }
  const int j = k0 + (NF == 2 ? 2 * (lane & 16) : 0) + 8 * ((lane & 15) >> 2) + 4 * hf + (lane & 3);
  if ((NF == 2 || !up) && j < a.Tk) {
    if (a.ns > 1) a.part[((int64_t)sp * a.B * a.Hk + bk) * a.Tk + j] = v[0];
    else a.kw_out[(int64_t)bk * a.Tk + j] = v[0] + (a.kw_in ? a.kw_in[b * a.kwsb + kvh * a.kwsh + j] : 0.f);
  }
}

__global__ __launch_bounds__(256) void key_weights_sum_kernel(const KeyWArgs a) {
  const int64_t n = (int64_t)a.B * a.Hk * a.Tk;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < n; x += (int64_t)gridDim.x * 256) {
    const int j = (int)(x % a.Tk), bk = (int)(x / a.Tk);
    float v = 0.f;
#pragma unroll 8
    for (int i = 0; i < a.ns; ++i) v += a.part[i * n + x];
    a.kw_out[x] = v + (a.kw_in ? a.kw_in[(bk / a.Hk) * a.kwsb + (bk % a.Hk) * a.kwsh + j] : 0.f);
  }
}

// A wave per 32 rows of one head.
template <typename T, int D, bool MASK>
__global__ __launch_bounds__(64) void far_rows_kernel(const KeyWArgs a) {
  using V8 = typename Vec8<T>::type;
  constexpr int DS = D / 16;
  const int nt = (a.Tq + 31) / 32;
  const int t = blockIdx.x % nt, bh = blockIdx.x / nt;
  const int b = bh / a.Hq, h = bh - b * a.Hq;
  const int lane = threadIdx.x, l32 = lane & 31, hf = lane >> 5;
  const int tq = min(t * 32 + l32, a.Tq - 1);
  const int64_t ri = (int64_t)bh * a.Tq + tq;
  const float lse = a.lse[ri];
  if (!wave_any(far_max(lse) && lse != kPosInf)) return;
  const int n = own_length(a, b), lim = a.causal ? min(n, tq + 1) : n;
  const float c2 = a.scale_log2;
  const T* kp = (const T*)a.k + b * a.ksb + (h / a.G) * a.ksh;
  u32x4 x[DS];
  V8 qf[DS], kf[DS];
  load_q<T, DS>(a, x, b, h, tq, hf);
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) qf[ds] = as_vec8<T>(only_cols(x[ds], ds, a.Dv, a.qsign < 0.f ? 0x80008000u : 0u));
  float mr = kNegInf, l = 0.f;
  for (int k0 = 0; k0 < n; k0 += 32) {
    load_keys<T, DS>(a, kp, k0, n, l32, hf, kf);
    f32x16 s = scores(a.score + b * a.ssb + h * a.ssh + (int64_t)tq * a.ssq, k0, hf, n, a.qsign);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) s = mfma32(kf[ds], qf[ds], s);
    uint32_t w = in_row(lim, k0, hf);
    if constexpr (MASK) w &= mask_bits(a, a.mask + b * a.msb + h * a.msh + (int64_t)tq * a.msq, k0, hf, n);
    float mx = kNegInf;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s[j] = (w >> (8 * (j >> 2) + (j & 3))) & 1u ? (a.zero_scale ? 0.f : s[j]) : kNegInf;
      mx = fmaxf(mx, s[j]);
    }
    mx = fmaxf(mr, half_max(mx));
    if (mx > mr) {
      l = mr == kNegInf ? 0.f : l * exp2_fast((mr - mx) * c2);
      mr = mx;
    }
    if (mr > kNegInf) {
#pragma unroll
      for (int j = 0; j < 16; ++j) l += exp2_fast((s[j] - mr) * c2);
    }
  }
  l = half_sum(l);
  if (hf == 0) {
    a.far_ml[2 * ri] = mr;
    a.far_ml[2 * ri + 1] = l;
  }
}

template <typename T, int D>
hipError_t launch_t(const KeyWArgs& a, hipStream_t s) {
  const bool m = a.mask != nullptr, sc = a.score != nullptr;
  if (sc) {
    const dim3 grid((unsigned)(a.B * a.Hq * ((a.Tq + 31) / 32)));
    if (m) hipLaunchKernelGGL((far_rows_kernel<T, D, true>), grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((far_rows_kernel<T, D, false>), grid, dim3(64), 0, s, a);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  const dim3 grid((unsigned)(a.B * a.Hk * a.ns * a.nkb)), block(kWaves * 64);
  if (m && sc) hipLaunchKernelGGL((key_weights_kernel<T, D, true, true>), grid, block, 0, s, a);
  else if (m) hipLaunchKernelGGL((key_weights_kernel<T, D, true, false>), grid, block, 0, s, a);
  else if (sc) hipLaunchKernelGGL((key_weights_kernel<T, D, false, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((key_weights_kernel<T, D, false, false>), grid, block, 0, s, a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && a.ns > 1) {
    const int64_t n = ((int64_t)a.B * a.Hk * a.Tk + 255) / 256;
    hipLaunchKernelGGL(key_weights_sum_kernel, dim3((unsigned)min_i64(n, 1 << 16)), dim3(256), 0, s, a);
    e = hipGetLastError();
  }
  return e;
}

template <typename T> hipError_t launch_d(const KeyWArgs& a, int D, hipStream_t s) {
  if (D == 64) return launch_t<T, 64>(a, s);
  if (D == 128) return launch_t<T, 128>(a, s);
  if (D == 256) return launch_t<T, 256>(a, s);
  return hipErrorInvalidValue;
}

}  // namespace

int keyw_block_keys(int D) { return kWaves * 32 * (D == 256 ? frags<256>() : frags<128>()); }

hipError_t launch_key_weights(const KeyWArgs& a, int D, int dtype, hipStream_t s) {
  return dtype == 0 ? launch_d<bf16>(a, D, s) : launch_d<f16>(a, D, s);
}

}  // namespace fa
