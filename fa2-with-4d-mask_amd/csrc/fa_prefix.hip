// Attention of a few query rows per sequence (decoding, drafts) over a prefix that the whole
// batch shares and each sequence's own keys, on gfx950 (MI355X).
//
//   O = softmax([Q Kp^T, Q K^T + Score] scale) [Vp; V]
//
// One softmax over two key sets, so both are cut into ranges whose partial results (running
// maximum m, sum l and O not divided by l) are joined at the end: O = sum_s 2^(m_s - m) O_s /
// sum_s 2^(m_s - m) l_s.
//
//   prefix_rows_kernel  one workgroup of 4 waves per (32 rows, key range, kv-head), for the
//                       prefix of the rows of *all* sequences (packed r = (b Tq + tq) G + g:
//                       the prefix is read once for the batch, not once per sequence), for own
//                       keys of one sequence's rows.  Both kinds run in one launch.  Each wave
//                       walks every fourth 32-key tile of the range with its own maximum, sum and
//                       O^T, merged through LDS at the end.  Many rows behind a long prefix take
//                       blocks of 128 instead (wide_body), in the same launch.
//   prefix_join_kernel  joins the ranges into O and LSE; with key weights, further workgroups
//                       turn the logits that the own ranges left into probabilities and add them.
//
// K rows go from memory straight into MFMA operands (S^T = K Q^T reads a K row per lane); V
// takes the way through an LDS region of each wave's own for the transpose reads of O^T += V^T P^T.
// P enters that product in two 16-bit parts, the rounded value and its residual: rounded once,
// O would be off by about its own rounding again, and in training Delta = rowsum(dO O) would
// no longer match the P that the backward recomputes (rows that lie on few keys: dQ and dK are
// then sums of terms that cancel, and lost 18 % of their norm).
//
// What bounds it: the bytes of K and V.  B64 Tp 8192, 256 own keys on average, Hq32 Hk8 D128: 136 MB in
// 43 us with the join (35 + 8 in a profile), 3.2 TB/s: 17 MB of fp32 partial results of the
// prefix's ranges go out and come back, and the sequences' own ranges are short.  Own keys alone,
// long enough: B1 Hk8 1e6 keys 667 us, 6.1 TB/s; B16 Tk 4096 with key weights, 208 MB in 55 us.  A few
// rows (B4 Tp1000): latency, 6 + 5 us of two launches beside 11 us of host time.
#include "fa_cache.h"
#include "fa_common.h"

namespace fa {
namespace {

constexpr int kKeys = 32;     // keys per tile
constexpr int kWaves = 4;
constexpr int kScan = 32;     // tiles of a wave whose liveness is looked at together

// chunk swizzle of the V tile's rows: the transpose reads (4 rows x 4 chunks) hit distinct banks
template <int D> __device__ __forceinline__ int swz_v(int r) {
  return D == 64 ? (((r >> 1) & 1) << 2) : ((r & 3) << 2);
}

// The products as fp32 values: O's 16-bit rounding and its residual then come from the same ones.
__device__ __forceinline__ void hold(f32x4& x, f32x4& y) { asm volatile("" : "+v"(x), "+v"(y)); }

__device__ __forceinline__ int own_length(const PrefixArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
}

constexpr int merge_stride(int D) { return D + 4; }   // floats per row of a wave's partial O
template <int D, bool MASK> constexpr int rows_lds() {
  constexpr int work = kWaves * (kKeys * 2 * D + (MASK ? kScan * 256 : 0)), merge = kWaves * 32 * merge_stride(D) * 4;
  return work > merge ? work : merge;
}

// One workgroup's item: OWN a sequence's own keys, else the prefix.  KW: the raw logits are kept.
template <typename T, int D, bool OWN, bool MASK, bool SCORE, bool KW>
__device__ __forceinline__ void rows_body(const PrefixArgs& a, const int W, char* smem, float (*sml)[3][32]) {
  using V8 = typename Vec8<T>::type;
  constexpr int DS = D / 16, NB = D / 32, CH = D / 8, ROWB = 2 * D;
  constexpr int VT = kKeys * ROWB;           // bytes of one V tile
  constexpr int U = kKeys * CH / 64;         // 16-byte V chunks per lane
  constexpr int OS = merge_stride(D);
  constexpr int KEEPB = MASK ? kScan * 256 : 0;

  // ---- which rows and keys: row blocks of a range next to each other (they share its K and V) --
  const int nrb = OWN ? a.nrbo : a.nrbp, ns = OWN ? a.nso : a.nsp;
  const int rb = W % nrb, W1 = W / nrb;
  const int sp = W1 % ns, unit = W1 / ns;
  const int bo = OWN ? unit / a.Hk : 0, kvh = OWN ? unit - bo * a.Hk : unit;
  const int TG = a.Tq * a.G;
  const int R = OWN ? TG : a.B * TG;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hf = lane >> 5;
  auto row_of = [&](int r, int& b, int& tq, int& h) __attribute__((always_inline)) {
    b = OWN ? bo : r / TG;
    const int rr = OWN ? r : r - b * TG;
    tq = rr / a.G;
    h = kvh * a.G + (rr - tq * a.G);
  };
  const int r = min(rb * 32 + l32, R - 1);   // this lane's packed row (rows past R repeat the last)
  int b, tq, h;
  row_of(r, b, tq, h);
  const float c2 = a.scale_log2;
  const int Tk = OWN ? own_length(a, bo) : a.Tp;   // keys past it are not read

  // Q fragment (B of S^T): lane holds Q[row][16 ds + 8 hf .. +7]
  V8 qf[DS];
  {
    const uint32_t neg = a.qsign < 0.f ? 0x80008000u : 0u;
    const T* src = (const T*)a.q + b * a.qsb + h * a.qsh + (int64_t)tq * a.qst + hf * 8;
    u32x4 x[DS];
    load_row(x, src, a.Dv);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qf[ds] = as_vec8<T>(only_cols(x[ds], ds, a.Dv, neg));
  }
  if constexpr (D == 256) {   // in AGPRs, which MFMA reads as well
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) asm volatile("" : "+a"(qf[ds]));
  }
  const int64_t kst = OWN ? a.kst : a.pkst, vst = OWN ? a.vst : a.pvst;
  const T* __restrict__ kp = OWN ? (const T*)a.k + bo * a.ksb + kvh * a.ksh : (const T*)a.pk + kvh * a.pksh;
  const T* __restrict__ vp = OWN ? (const T*)a.v + bo * a.vsb + kvh * a.vsh : (const T*)a.pv + kvh * a.pvsh;
  const uint8_t* mrow = MASK ? a.mask + b * a.msb + h * a.msh + (int64_t)tq * a.msq : nullptr;
  const float* srow = SCORE ? a.score + b * a.ssb + h * a.ssh + (int64_t)tq * a.ssq : nullptr;
  const bool causal = OWN && a.causal;
  const int lim = causal ? min(Tk, tq + 1) : Tk;   // keys [0, lim) of this lane's row
  const int64_t ri = ((int64_t)b * a.Hq + h) * a.Tq + tq;
  float* lrow = KW ? a.logits + ri * a.Tkp : nullptr;
  const bool mine = rb * 32 + l32 < R;

  // ---- key tiles of the workgroup and of this wave ------------------------------
  // (causal: up to the block's last row, rows are packed by tq; KW: of the last row of all, every
  // logit up to there is looked at)
  const int last = KW ? a.Tq : min(rb * 32 + 31, R - 1) / a.G + 1;
  const int nt = ((causal ? min(Tk, last) : Tk) + kKeys - 1) / kKeys;
  const int ct = OWN ? a.cto : a.ctp;
  const int t_lo = min(sp * ct, nt), t_hi = min(t_lo + ct, nt);
  const int t_w = t_lo + wave;
  const int n_w = t_w < t_hi ? (t_hi - t_w + kWaves - 1) / kWaves : 0;   // tiles t_w + 4 i

  // ---- loads ---------------------------------------------------------------------
  u32x4 kf[DS], vr[U];
  uint32_t goff_v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int idx = lane + u * 64;
    goff_v[u] = 8 * (idx % CH) < a.Dv ? (uint32_t)((idx / CH) * vst * 2) + (uint32_t)((idx % CH) * 16) : kNoRec;
  }
  const uint32_t goff_k = (uint32_t)(l32 * kst * 2) + (uint32_t)(hf * 16);
  // rows of tile t through a buffer from its first key; keys past Tk (and a
  // tile that is not there) read zeros
  auto tile_rs = [&](const T* base, int64_t st, int t, bool valid) __attribute__((always_inline)) {
    const int rows = min(Tk - t * kKeys, kKeys);
    const bool ok = valid && rows > 0;
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (ok ? (int64_t)t * kKeys * st : 0)), (short)0,
                                             ok ? (int)((int64_t)(rows - 1) * st * 2 + 2 * a.Dv) : 0, 0x00020000);
  };
  auto load_k = [&](int t, bool valid) __attribute__((always_inline)) {
    const auto rs = tile_rs(kp, kst, t, valid);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) kf[ds] = __builtin_amdgcn_raw_buffer_load_b128(rs, goff_k + 32 * ds, 16 * ds < a.Dv ? 0 : kNoRec, 0);
  };
  auto load_v = [&](int t, bool valid) __attribute__((always_inline)) {
    const auto rs = tile_rs(vp, vst, t, valid);
#pragma unroll
    for (int u = 0; u < U; ++u) vr[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, goff_v[u], 0, 0);
  };
  // scores of tile t at this lane's row (entry 4 gi + e: key 32 t + 8 gi +
  // 4 hf + e); keys past Tk read key Tk - 1 (dropped below)
  auto load_score = [&](int t, f32x16& x) __attribute__((always_inline)) {
    if ((t + 1) * kKeys <= Tk) {
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) {
        struct __attribute__((packed, aligned(4))) F4 { float v[4]; };
        const F4 y = *(const F4*)(srow + t * kKeys + gi * 8 + hf * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[gi * 4 + e] = y.v[e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = srow[min(t * kKeys + 8 * (i >> 2) + 4 * hf + (i & 3), Tk - 1)];
    }
  };
  // keep bits of tile t at this lane's row (bit 8 gi + e <-> entry 4 gi + e)
  auto load_keep = [&](int t) __attribute__((always_inline)) -> uint32_t {
    uint32_t w = 0;
    const int k0 = t * kKeys + 4 * hf;
    if (a.mask4 && (t + 1) * kKeys <= Tk) {   // rows 4-byte aligned: four keys per load
      uint32_t x[4];
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) x[gi] = *(const uint32_t*)(mrow + k0 + 8 * gi);
#pragma unroll
      for (int gi = 0; gi < 4; ++gi)
#pragma unroll
        for (int e = 0; e < 4; ++e) w |= ((x[gi] >> (8 * e)) & 0xffu) != 0 ? 1u << (8 * gi + e) : 0u;
    } else {
      uint8_t x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = mrow[min(k0 + 8 * (i >> 2) + (i & 3), Tk - 1)];
#pragma unroll
      for (int i = 0; i < 16; ++i) w |= x[i] != 0 ? 1u << (8 * (i >> 2) + (i & 3)) : 0u;
    }
    return w;
  };
  // the first lim keys of the row, as keep bits of the tile at k0
  auto in_row = [&](int k0) __attribute__((always_inline)) -> uint32_t {
    const int n = lim - (k0 + 4 * hf);
    return n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1u);
  };

  f32x16 oacc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) oacc[nb] = f32x16{};
  float m_run = kNegInf, l_run = 0.f, mr = kNegInf;
  float m_lift = kNegInf;   // what a tile's maximum has to exceed to move m_run (with a score)
  const int tr_row = 4 * hf + ((lane >> 2) & 3);
  const int tr_col = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
  char* vt = smem + wave * VT;
  uint32_t* keep = (uint32_t*)(smem + kWaves * VT + wave * KEEPB);

  for (int ic = 0; ic < n_w; ic += kScan) {
    // ---- live tiles among the next kScan of this wave (KW: all, each leaves its logits) ----
    const int cnt = min(kScan, n_w - ic);
    uint32_t live = cnt == 32 ? ~0u : (1u << cnt) - 1u;
    if constexpr (MASK) {
      uint32_t any = 0;
#pragma unroll 2
      for (int i = 0; i < cnt; ++i) {
        const int t = t_w + kWaves * (ic + i);
        const uint32_t w = in_row(t * kKeys) & load_keep(t);
        keep[i * 64 + lane] = w;
        any |= wave_any(w != 0) ? 1u << i : 0u;
      }
      if constexpr (!KW) live = any;
    }
    if (live == 0) continue;

    // ---- the tiles: K(next) and V(next) are loaded while this one is worked on ----
    f32x16 sc = f32x16{};
    int i = __builtin_ctz(live);
    live &= live - 1;
    load_k(t_w + kWaves * (ic + i), true);
    if constexpr (SCORE) load_score(t_w + kWaves * (ic + i), sc);
    load_v(t_w + kWaves * (ic + i), true);
    for (;;) {
      const int k0 = (t_w + kWaves * (ic + i)) * kKeys;
      const bool more = live != 0;
      const int i_nx = more ? __builtin_ctz(live) : i;
      const int t_nx = t_w + kWaves * (ic + i_nx);
      live &= live - 1;
      f32x16 s;
      if constexpr (SCORE) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = a.qsign < 0.f ? -sc[j] : sc[j];
      } else {
        s = f32x16{};
      }
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) s = mfma32(as_vec8<T>(kf[ds]), qf[ds], s);
      load_k(t_nx, more);
      if constexpr (SCORE) load_score(t_nx, sc);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int idx = lane + u * 64, rr = idx / CH, c = idx % CH;
        lds_write16(vt + rr * ROWB + ((c ^ swz_v<D>(rr)) * 16), vr[u]);
      }
      load_v(t_nx, more);
      // dropped entries to -inf (kept ones to 0 with scale 0)
      if (MASK || a.zero_scale || causal || k0 + kKeys > Tk) {
        uint32_t w = in_row(k0);
        if constexpr (MASK) w &= keep[i * 64 + lane];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const bool kept = (w >> (8 * (j >> 2) + (j & 3))) & 1u;
          s[j] = kept ? (a.zero_scale ? 0.f : s[j]) : kNegInf;
        }
      }
      if constexpr (KW) {
        if (mine) {
#pragma unroll
          for (int gi = 0; gi < 4; ++gi) {
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = s[4 * gi + e];
            *(f32x4*)(lrow + k0 + 8 * gi + 4 * hf) = x;
          }
        }
      }
      // running maximum: the first kept tile's, then raised in whole steps (the
      // rounded P then does not depend on which tile raised it)
      float mx = s[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j]);
      mx = half_max(mx);
      if constexpr (SCORE && KW) mr = fmaxf(mr, mx);
      const float mc = mx * c2;
      float mneg = m_run == kNegInf ? 0.f : -m_run;
      if (wave_any(mc > (SCORE ? m_lift : m_run))) {   // (-inf for rows of far_max(): with every tile)
        const float m_new = m_run == kNegInf ? mc : raise_max(m_run, mc);
        const float alpha = m_run == kNegInf ? 0.f : exp2_fast(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) oacc[nb] *= alpha;
        m_run = m_new;
        mneg = m_run == kNegInf ? 0.f : -m_run;
        if constexpr (SCORE) {
          m_lift = far_max(m_run) ? kNegInf : m_run;
          const bool far = far_max(m_run) && mx > kNegInf;
          const float sub = far ? mx : 0.f;
#pragma unroll
          for (int j = 0; j < 16; ++j) s[j] -= sub;
          if (far) mneg = mc - m_run;
        }
      }
      V8 pk[2], pkl[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = exp2_fast(fmaf(s[8 * c + e], c2, mneg));
          l_run += p[e];
        }
        pk[c] = pack8<T>(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]);
        float q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = p[e] - (float)(T)p[e];
        pkl[c] = pack8<T>(q[0], q[1], q[2], q[3], q[4], q[5], q[6], q[7]);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = 16 * c + tr_row;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int col = nb * 32 + tr_col;
          const char* p = vt + row * ROWB + (((col >> 3) ^ swz_v<D>(row)) * 16) + (col & 7) * 2;
          const V8 va = cat_tr<T>(lds_read_tr(p), lds_read_tr(p + 8 * ROWB));
          oacc[nb] = mfma32(va, pk[c], oacc[nb]);
          oacc[nb] = mfma32(va, pkl[c], oacc[nb]);
        }
      }
      if (!more) break;
      i = i_nx;
    }
  }

  // ---- merge the waves, leave the range's partial result ------------------------------
  const float l_tot = half_sum(l_run);
  if (hf == 0) {
    sml[wave][0][l32] = m_run;
    sml[wave][1][l32] = l_tot;
    if constexpr (SCORE && KW) sml[wave][2][l32] = mr;
  }
  __syncthreads();   // also: every wave is done with its V tile and keep words
  auto merged = [&](int which, int row) __attribute__((always_inline)) -> float {
    return fmaxf(fmaxf(sml[0][which][row], sml[1][which][row]), fmaxf(sml[2][which][row], sml[3][which][row]));
  };
  auto weight = [&](float m, float mm) __attribute__((always_inline)) -> float {
    return m == kNegInf ? 0.f : exp2_fast(m - mm);
  };
  {
    const float w = weight(m_run, merged(0, l32));
    float* st = (float*)smem + (wave * 32 + l32) * OS;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = oacc[nb][gi * 4 + e] * w;
        *(f32x4*)(st + nb * 32 + gi * 8 + hf * 4) = x;
      }
  }
  __syncthreads();
  const int64_t rows = (int64_t)a.B * a.Hq * a.Tq;
  const int slot = OWN ? a.nsp + sp : sp;
#pragma unroll
  for (int u = 0; u < 32 * CH / (kWaves * 64); ++u) {
    const int idx = tid + u * kWaves * 64, row = idx / CH, c = idx % CH;
    const int rr = rb * 32 + row;
    if (rr >= R) continue;
    int b_, q_, h_;
    row_of(rr, b_, q_, h_);
    const int64_t pr = slot * rows + ((int64_t)b_ * a.Hq + h_) * a.Tq + q_;
    const float mm = merged(0, row);
    float l = 0.f;
    f32x4 x0 = f32x4{}, x1 = f32x4{};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      l += sml[w][1][row] * weight(sml[w][0][row], mm);
      const float* st = (const float*)smem + (w * 32 + row) * OS + c * 8;
      x0 += *(const f32x4*)st;
      x1 += *(const f32x4*)(st + 4);
    }
    if (c == 0) *(f32x4*)(a.part_ml + 4 * pr) = f32x4{mm, l, SCORE && KW ? merged(2, row) : kNegInf, 0.f};
    if (mm == kNegInf || 8 * c >= a.Dv) continue;   // nothing kept: the join does not look
    float* po = a.part_o + pr * D + c * 8;
    *(f32x4*)po = x0;
    *(f32x4*)(po + 4) = x1;
  }
}

// The prefix for many rows (a.wide: at least kWideRows of a kv-head over the batch): 128 rows per
// workgroup, 32 per wave, every wave walks all 64-key tiles of the range, which the workgroup
// stages once in LDS (two buffers, one barrier per tile).  Against rows_body, whose waves have 32
// rows in common and cut the keys: K and V come from memory once per 128 rows, two independent
// chains of S products per wave hide each other's latency, and there is no merge.
constexpr int kWideKeys = 64;
// K rows are read 16 consecutive ones of a chunk at a time, V as 4 rows x 4 chunks.
template <int D> __device__ __forceinline__ int swz_wk(int r) { return D == 128 ? (r & 15) : ((r >> 1) & 7); }

template <typename T, int D>
__device__ __forceinline__ void wide_body(const PrefixArgs& a, const int W, char* smem) {
  using V8 = typename Vec8<T>::type;
  constexpr int DS = D / 16, NB = D / 32, CH = D / 8, ROWB = 2 * D;
  constexpr int TB = kWideKeys * ROWB;             // bytes of a K or V tile
  constexpr int U = kWideKeys * CH / (kWaves * 64);   // 16-byte chunks per thread and kind
  const int nrb = a.nrbp;
  const int rb = W % nrb, W1 = W / nrb;
  const int sp = W1 % a.nsp, kvh = W1 / a.nsp;
  const int TG = a.Tq * a.G, R = a.B * TG;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hf = lane >> 5;
  const int row = rb * kWideRows + wave * 32 + l32;
  const int r = min(row, R - 1);
  const int b = r / TG, rr = r - b * TG, tq = rr / a.G, h = kvh * a.G + (rr - tq * a.G);
  const float c2 = a.scale_log2;
  const int Tk = a.Tp;

  V8 qf[DS];
  {
    const uint32_t neg = a.qsign < 0.f ? 0x80008000u : 0u;
    u32x4 x[DS];
    load_row(x, (const T*)a.q + b * a.qsb + h * a.qsh + (int64_t)tq * a.qst + hf * 8, a.Dv);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qf[ds] = as_vec8<T>(only_cols(x[ds], ds, a.Dv, neg));
  }
  const T* __restrict__ kp = (const T*)a.pk + kvh * a.pksh;
  const T* __restrict__ vp = (const T*)a.pv + kvh * a.pvsh;
  const int nt = (Tk + kWideKeys - 1) / kWideKeys;
  const int t_lo = min(sp * a.ctp, nt), t_hi = min(t_lo + a.ctp, nt);

  // staging: thread -> chunk c of tile row tr + u (256 / CH)
  uint32_t gk[U], gv[U], lk[U], lv[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int idx = tid + u * kWaves * 64, tr = idx / CH, c = idx % CH;
    gk[u] = 8 * c < a.Dv ? (uint32_t)(tr * a.pkst * 2) + (uint32_t)(c * 16) : kNoRec;
    gv[u] = 8 * c < a.Dv ? (uint32_t)(tr * a.pvst * 2) + (uint32_t)(c * 16) : kNoRec;
    lk[u] = tr * ROWB + ((c ^ swz_wk<D>(tr)) * 16);
    lv[u] = TB + tr * ROWB + ((c ^ swz_v<D>(tr)) * 16);
  }
  u32x4 kr[U], vr[U];
  auto rs_of = [&](const T* base, int64_t st, int t) __attribute__((always_inline)) {
    const int rows = t < t_hi ? min(Tk - t * kWideKeys, kWideKeys) : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (rows > 0 ? (int64_t)t * kWideKeys * st : 0)), (short)0,
                                             rows > 0 ? (int)((int64_t)(rows - 1) * st * 2 + 2 * a.Dv) : 0, 0x00020000);
  };
  auto load = [&](int t) __attribute__((always_inline)) {   // (past the range: zeros)
    const auto rk = rs_of(kp, a.pkst, t), rv = rs_of(vp, a.pvst, t);
#pragma unroll
    for (int u = 0; u < U; ++u) kr[u] = __builtin_amdgcn_raw_buffer_load_b128(rk, gk[u], 0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) vr[u] = __builtin_amdgcn_raw_buffer_load_b128(rv, gv[u], 0, 0);
  };
  auto store = [&](int buf) __attribute__((always_inline)) {
    char* p = smem + buf * 2 * TB;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      lds_write16(p + lk[u], kr[u]);
      lds_write16(p + lv[u], vr[u]);
    }
  };

  f32x16 oacc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) oacc[nb] = f32x16{};
  float m_run = kNegInf, l_run = 0.f;
  const int tr_row = 4 * hf + ((lane >> 2) & 3);
  const int tr_col = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;

  if (t_lo < t_hi) {
    load(t_lo);
    store(0);
    __syncthreads();
  }
  for (int t = t_lo; t < t_hi; ++t) {
    const char* kt = smem + ((t - t_lo) & 1) * 2 * TB;
    const char* vt = kt + TB;
    load(t + 1);
    f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
    for (int ds = 0; ds < DS; ++ds)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int kr_ = kb * 32 + l32;
        s[kb] = mfma32(as_vec8<T>(lds_read16(kt + kr_ * ROWB + (((2 * ds + hf) ^ swz_wk<D>(kr_)) * 16))), qf[ds], s[kb]);
      }
    const int k0 = t * kWideKeys;
    if (a.zero_scale || k0 + kWideKeys > Tk) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          s[kb][j] = k0 + 32 * kb + 8 * (j >> 2) + 4 * hf + (j & 3) < Tk ? (a.zero_scale ? 0.f : s[kb][j]) : kNegInf;
    }
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[kb][j]);
    mx = half_max(mx);
    const float mc = mx * c2;
    if (wave_any(mc > m_run)) {   // raised in whole steps, as in rows_body
      const float m_new = m_run == kNegInf ? mc : raise_max(m_run, mc);
      const float alpha = m_run == kNegInf ? 0.f : exp2_fast(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) oacc[nb] *= alpha;
      m_run = m_new;
    }
    const float mneg = m_run == kNegInf ? 0.f : -m_run;
#pragma unroll
    for (int c = 0; c < 4; ++c) {   // 16 keys
      float p[8], q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = exp2_fast(fmaf(s[c >> 1][8 * (c & 1) + e], c2, mneg));
        q[e] = p[e] - (float)(T)p[e];
      }
      l_run += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      const V8 hi = pack8<T>(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]);
      const V8 lo = pack8<T>(q[0], q[1], q[2], q[3], q[4], q[5], q[6], q[7]);
      const int vrow = 16 * c + tr_row;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int col = nb * 32 + tr_col;
        const char* x = vt + vrow * ROWB + (((col >> 3) ^ swz_v<D>(vrow)) * 16) + (col & 7) * 2;
        const V8 va = cat_tr<T>(lds_read_tr(x), lds_read_tr(x + 8 * ROWB));
        oacc[nb] = mfma32(va, hi, oacc[nb]);
        oacc[nb] = mfma32(va, lo, oacc[nb]);
      }
    }
    if (t + 1 < t_hi) {
      store((t + 1 - t_lo) & 1);   // (read last in tile t - 1, before the barrier that ended it)
      __syncthreads();
    }
  }
  const float l_tot = half_sum(l_run);
  if (row >= R) return;
  const int64_t pr = ((int64_t)sp * a.B * a.Hq + (int64_t)b * a.Hq + h) * a.Tq + tq;
  if (hf == 0) *(f32x4*)(a.part_ml + 4 * pr) = f32x4{m_run, l_tot, kNegInf, 0.f};
  if (m_run == kNegInf) return;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int gi = 0; gi < 4; ++gi) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = oacc[nb][gi * 4 + e];
      *(f32x4*)(a.part_o + pr * D + nb * 32 + gi * 8 + hf * 4) = x;
    }
}

template <typename T, int D, bool MASK, bool SCORE, bool KW>
__global__ __launch_bounds__(kWaves * 64, D == 256 ? 1 : 2) void prefix_rows_kernel(const PrefixArgs a) {
  __shared__ __attribute__((aligned(1024))) char smem[rows_lds<D, MASK>()];
  __shared__ float sml[kWaves][3][32];       // running maximum, sum, largest raw logit per wave and row
  // the prefix ranges first: the longest ones
  if constexpr (D <= 128) {
    static_assert(4 * kWideKeys * 2 * D <= rows_lds<D, MASK>(), "two buffers of K and V");
    if (a.wide && (int)blockIdx.x < a.np) {
      wide_body<T, D>(a, xcd_remap(blockIdx.x, a.np), smem);
      return;
    }
  }
  if ((int)blockIdx.x < a.np) rows_body<T, D, false, false, false, false>(a, xcd_remap(blockIdx.x, a.np), smem, sml);
  else rows_body<T, D, true, MASK, SCORE, KW>(a, xcd_remap(blockIdx.x - a.np, a.no), smem, sml);
}

// Maximum, sum and largest raw logit of row ri over all its slots, in every lane of the wave;
// w0 / w1: this lane's slots' (lane, lane + 64) weights 2^(m - mm), 0 where nothing was kept.
__device__ __forceinline__ void join_stats(const PrefixArgs& a, int64_t rows, int64_t ri, int lane, float& mm, float& l,
                                           float& mr, float& w0, float& w1) {
  const int ns = a.nsp + a.nso;
  const f32x4 none = f32x4{kNegInf, 0.f, kNegInf, 0.f};
  const f32x4 x0 = lane < ns ? *(const f32x4*)(a.part_ml + 4 * (lane * rows + ri)) : none;
  const f32x4 x1 = lane + 64 < ns ? *(const f32x4*)(a.part_ml + 4 * ((lane + 64) * rows + ri)) : none;
  mm = fmaxf(x0[0], x1[0]);
  mr = fmaxf(x0[2], x1[2]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    mm = fmaxf(mm, __shfl_xor(mm, d));
    mr = fmaxf(mr, __shfl_xor(mr, d));
  }
  w0 = x0[0] == kNegInf ? 0.f : exp2_fast(x0[0] - mm);
  w1 = x1[0] == kNegInf ? 0.f : exp2_fast(x1[0] - mm);
  l = x0[1] * w0 + x1[1] * w1;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
}

// NW waves per row: a wave's lanes in groups of D / 8, each group's share of the slots summed
// over the groups at the end (fixed order: deterministic).  One wave for few slots; four, a
// workgroup per row, for many.
template <typename T, int D, int NW>
__global__ __launch_bounds__(256) void prefix_join_kernel(const PrefixArgs a, const int nrow_wg) {
  using V8 = typename Vec8<T>::type;
  constexpr int CH = D / 8, GW = 64 / CH, NG = NW * GW, RPB = 4 / NW;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t rows = (int64_t)a.B * a.Hq * a.Tq;
  const int ns = a.nsp + a.nso;
  if ((int)blockIdx.x < nrow_wg) {
    const int c = lane % CH, grp = (NW == 1 ? 0 : wave * GW) + lane / CH;
    const int64_t rb = (int64_t)blockIdx.x * RPB + (NW == 1 ? wave : 0);
    const int64_t ri = min_i64(rb, rows - 1);
    const int q = (int)(ri % a.Tq);
    const int64_t bh = ri / a.Tq;
    const int b = (int)(bh / a.Hq), h = (int)(bh - (int64_t)b * a.Hq);
    float mm, lt, mr, w0, w1;
    join_stats(a, rows, ri, lane, mm, lt, mr, w0, w1);
    f32x4 x0 = f32x4{}, x1 = f32x4{};
    // (every load goes out, also of slots where nothing was kept: their values are not used)
#pragma unroll 8
    for (int i = grp; i < (ns + NG - 1) / NG * NG; i += NG) {
      const float wa = __shfl(w0, i & 63), wb = __shfl(w1, i & 63);
      const float wi = i < 64 ? wa : wb;
      const float* p = a.part_o + ((int64_t)min(i, ns - 1) * rows + ri) * D + c * 8;
      const f32x4 y0 = *(const f32x4*)p, y1 = *(const f32x4*)(p + 4);
      if (i < ns && wi != 0.f) {
        x0 += y0 * wi;
        x1 += y1 * wi;
      }
    }
#pragma unroll
    for (int d = CH; d < 64; d <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x0[e] += __shfl_xor(x0[e], d);
        x1[e] += __shfl_xor(x1[e], d);
      }
    if constexpr (NW > 1) {   // lane c of each wave holds the wave's sum
      __shared__ f32x4 part[NW][CH][2];
      if (lane < CH) {
        part[wave][c][0] = x0;
        part[wave][c][1] = x1;
      }
      __syncthreads();
      x0 = part[0][c][0];
      x1 = part[0][c][1];
#pragma unroll
      for (int i = 1; i < NW; ++i) {
        x0 += part[i][c][0];
        x1 += part[i][c][1];
      }
    }
    if (grp != 0 || rb >= rows || 8 * c >= a.Dv) return;
    const float inv = 1.0f / lt;   // (a row that keeps nothing: 0 times inf, NaN)
    x0 *= inv;
    x1 *= inv;
    hold(x0, x1);
    const V8 o = pack8<T>(x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]);
    gstore16((T*)a.o + b * a.osb + h * a.osh + (int64_t)q * a.ost + c * 8, as_u32x4<T>(o));
    if (a.olo) {
      const V8 lo = pack8<T>(x0[0] - (float)o[0], x0[1] - (float)o[1], x0[2] - (float)o[2], x0[3] - (float)o[3],
                             x1[0] - (float)o[4], x1[1] - (float)o[5], x1[2] - (float)o[6], x1[3] - (float)o[7]);
      gstore16((T*)a.olo + b * a.olsb + h * a.olsh + (int64_t)q * a.olst + c * 8, as_u32x4<T>(lo));
    }
    if (c == 0) a.lse[ri] = lt > 0.f ? mm + log2_fast(lt) : kPosInf;
    return;
  }
  // ---- key weights: 1024 keys of one (sequence, kv-head) ----------------------------------
  // p = exp2(s c - m) / l; a row whose maximum is so far from zero that the fused product and
  // the rounded maximum no longer meet (far_max) takes s - its largest raw logit first.
  __shared__ f32x4 st[kPrefixKwRows];
  const int W = blockIdx.x - nrow_wg, nch = (a.Tk + 1023) / 1024;
  const int ch = W % nch, bk = W / nch;
  const int b = bk / a.Hk, kvh = bk - b * a.Hk, TG = a.Tq * a.G;
  const int64_t r0 = ((int64_t)b * a.Hq + kvh * a.G) * a.Tq;   // the group's rows are neighbours: (g, tq)
  for (int r = wave; r < TG; r += 4) {
    float mm, l, mr, w0, w1;
    join_stats(a, rows, r0 + r, lane, mm, l, mr, w0, w1);
    const bool far = a.score && far_max(mm) && mr > kNegInf;
    float mc = mr * a.scale_log2;
    asm volatile("" : "+v"(mc));   // rounded, as the ranges' maxima are
    // {subtracted from s, from the product, 1 / sum (0: nothing kept)}
    if (lane == 0)
      st[r] = f32x4{far ? mr : 0.f, far ? mm - mc : (mm == kNegInf ? 0.f : mm),
                    mm == kNegInf || !(l != 0.f) ? 0.f : 1.0f / l, 0.f};
  }
  __syncthreads();
  const int j = ch * 1024 + threadIdx.x * 4;
  if (j >= a.Tk) return;
  const int n = own_length(a, b), lim = a.causal ? min(n, a.Tq) : n;
  f32x4 w = f32x4{};
  if (j < lim) {
    const float* lp = a.logits + r0 * a.Tkp + j;
#pragma unroll 8
    for (int r = 0; r < TG; ++r) {
      const f32x4 s = *(const f32x4*)(lp + (int64_t)r * a.Tkp);
      const f32x4 t = st[r];
      if (t[2] != 0.f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] += exp2_fast(fmaf(s[e] - t[0], a.scale_log2, -t[1])) * t[2];
      }
    }
  }
  const float* in = a.kw_in ? a.kw_in + b * a.kwsb + kvh * a.kwsh + j : nullptr;
  float* out = a.kw_out + (int64_t)bk * a.Tk + j;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j + e < a.Tk) out[e] = (in ? in[e] : 0.f) + (j + e < lim ? w[e] : 0.f);
}

template <typename T, int D>
hipError_t launch_rows_t(const PrefixArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.np + a.no)), block(kWaves * 64);
  const bool m = a.mask != nullptr, sc = a.score != nullptr;
  if (a.kw_out) {
    if (m && sc) hipLaunchKernelGGL((prefix_rows_kernel<T, D, true, true, true>), grid, block, 0, s, a);
    else if (m) hipLaunchKernelGGL((prefix_rows_kernel<T, D, true, false, true>), grid, block, 0, s, a);
    else if (sc) hipLaunchKernelGGL((prefix_rows_kernel<T, D, false, true, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((prefix_rows_kernel<T, D, false, false, true>), grid, block, 0, s, a);
  } else {
    if (m && sc) hipLaunchKernelGGL((prefix_rows_kernel<T, D, true, true, false>), grid, block, 0, s, a);
    else if (m) hipLaunchKernelGGL((prefix_rows_kernel<T, D, true, false, false>), grid, block, 0, s, a);
    else if (sc) hipLaunchKernelGGL((prefix_rows_kernel<T, D, false, true, false>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((prefix_rows_kernel<T, D, false, false, false>), grid, block, 0, s, a);
  }
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_join_t(const PrefixArgs& a, hipStream_t s) {
  const int64_t rows = (int64_t)a.B * a.Hq * a.Tq;
  const int64_t kw = a.kw_out ? (int64_t)a.B * a.Hk * ((a.Tk + 1023) / 1024) : 0;
  if (a.nsp + a.nso <= 16) {
    const int64_t n = (rows + 3) / 4;
    hipLaunchKernelGGL((prefix_join_kernel<T, D, 1>), dim3((unsigned)(n + kw)), dim3(256), 0, s, a, (int)n);
  } else {
    hipLaunchKernelGGL((prefix_join_kernel<T, D, 4>), dim3((unsigned)(rows + kw)), dim3(256), 0, s, a, (int)rows);
  }
  return hipGetLastError();
}

}  // namespace

int prefix_tile_keys() { return kKeys; }

#define FA_BY_DIM(fn, a, D, s)                                                  \
  (dtype == 0 ? (D == 64 ? fn<bf16, 64>(a, s) : D == 128 ? fn<bf16, 128>(a, s) : \
                 D == 256 ? fn<bf16, 256>(a, s) : hipErrorInvalidValue)          \
              : (D == 64 ? fn<f16, 64>(a, s) : D == 128 ? fn<f16, 128>(a, s) :   \
                 D == 256 ? fn<f16, 256>(a, s) : hipErrorInvalidValue))

hipError_t launch_prefix_rows(const PrefixArgs& a, int D, int dtype, hipStream_t s) { return FA_BY_DIM(launch_rows_t, a, D, s); }
hipError_t launch_prefix_join(const PrefixArgs& a, int D, int dtype, hipStream_t s) { return FA_BY_DIM(launch_join_t, a, D, s); }

}  // namespace fa
