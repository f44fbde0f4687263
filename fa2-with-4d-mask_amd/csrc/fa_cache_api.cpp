// C ABI of the cache operators (shared prefixes, key weights, eviction, rotary positions):
// argument validation, planning, launches.  As in fa_api.cpp every entry point checks its
// arguments on the host before any HIP call.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "fa2_4d_mask.h"
#include "fa_cache.h"
#include "fa_kernels.h"
#include "fa_status.h"

namespace {

using fa::aligned16;
using fa::check_operand;
using fa::fail;
using fa::launch_status;

constexpr int64_t kMaxRows = (1LL << 31) - (1LL << 16);   // as fa_api.cpp: 32-bit row indices
constexpr int64_t kMaxGrid = 1LL << 23;                   // workgroups of 256 threads: below 2^31 threads

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// (of positive sizes below 2^31)
bool rows_fit(int64_t a, int64_t b, int64_t c) { return a * b < kMaxRows && a * b * c < kMaxRows; }

struct Sizes {
  int32_t B, Tq, Tk, Hq, Hk, D, Din, dtype;
  float scale;
};

// min_q / min_k: smallest lengths the entry point takes.
int check_sizes(const Sizes& z, int min_k) {
  if (z.B < 1 || z.Tq < 1 || z.Tk < min_k || z.Hq < 1 || z.Hk < 1)
    return fail(FA_ERR_SHAPE, "sizes must be >= 1 (B=%d Tq=%d Tk=%d Hq=%d Hk=%d)", z.B, z.Tq, z.Tk, z.Hq, z.Hk);
  if (z.Hq % z.Hk != 0) return fail(FA_ERR_SHAPE, "query heads (%d) must be divisible by key/value heads (%d)", z.Hq, z.Hk);
  if (z.D != 64 && z.D != 128 && z.D != 256) return fail(FA_ERR_HEAD_DIM, "head_dim %d not supported (64, 128, 256)", z.D);
  if (z.Din < 0 || z.Din > z.D || z.Din % 16)
    return fail(FA_ERR_HEAD_DIM, "head_dim_in %d must be a multiple of 16 up to head_dim %d (0: head_dim)", z.Din, z.D);
  if (z.dtype != FA_DTYPE_BF16 && z.dtype != FA_DTYPE_FP16) return fail(FA_ERR_DTYPE, "unsupported dtype code %d", z.dtype);
  if (!std::isfinite(z.scale)) return fail(FA_ERR_SCALE, "scale must be finite");
  if (!rows_fit(z.B, z.Hq, z.Tq) || !rows_fit(z.B, z.Hk, z.Tk))
    return fail(FA_ERR_SHAPE, "problem too large for 32-bit row indices (B*H*T must stay below 2^31 - 2^16)");
  return FA_OK;
}

int check_step(const char* name, int64_t st) {
  if (st < 0 || st >= (1LL << 24)) return fail(FA_ERR_STRIDE, "%s time stride %lld must lie in [0, 2^24) elements", name, (long long)st);
  return FA_OK;
}

int check_nonneg(const char* name, int64_t a, int64_t b, int64_t c) {
  if (a < 0 || b < 0 || c < 0) return fail(FA_ERR_STRIDE, "%s strides must be non-negative", name);
  return FA_OK;
}

bool mask_by_words(const uint8_t* m, int64_t sb, int64_t sh, int64_t sq) {
  return (uintptr_t)m % 4 == 0 && sb % 4 == 0 && sh % 4 == 0 && sq % 4 == 0;
}

void scales(float scale, float* scale_log2, float* qsign, int* zero) {
  *zero = scale == 0.f;
  *qsign = scale < 0.f ? -1.f : 1.f;
  *scale_log2 = *zero ? 1.f : std::fabs(scale) * 1.4426950408889634f;
}

// ---- shared prefix ------------------------------------------------------------------------

// Few rows per sequence: packed in blocks (fa_prefix.hip), the prefix read once for the batch.
// Beyond, the 256-row blocks of fa_fwd.hip run over both key sets in turn, every range leaving its
// partial result for one combine.  (Head dim 256: always packed; its own forward leaves no
// partial results.)  In us, packed / not (bf16): 8 sequences behind 2000 shared keys, Hq 16, D 128, Tq
// 48 33 / 69, 100 48 / 71, 200 70 / 84; one sequence behind 16000, Hq 32, Tq 48
// 43 / 101, 100 70 / 108, 200 137 / 125; own keys alone, B16 Tk Tq + 500 Hq16 D64, Tq 48 21 / 28, 100
// 34 / 30, 200 58 / 37.
bool few_rows(const FaPrefixParams* p) {
  return p->head_dim > 128 || p->seqlen_q <= (p->seqlen_p >= p->seqlen_k ? 128 : 64);
}

struct PrefixPlan {
  bool few, wide;
  int ctp, cto, nsp, nso, nrbp, nrbo;
  int64_t np, no, rows, bytes;
  int Tkp;
};

PrefixPlan prefix_plan(const FaPrefixParams* p) {
  PrefixPlan f{};
  const int G = p->heads_q / p->heads_k, kt = fa::prefix_tile_keys();
  const int64_t TG = (int64_t)G * p->seqlen_q;
  f.rows = (int64_t)p->batch * p->heads_q * p->seqlen_q;
  f.few = few_rows(p);
  if (!f.few) {
    auto ranges = [&](int64_t Tk, bool causal) -> int {
      if (Tk == 0) return 0;
      const int64_t nt = ceil_div(causal ? std::min<int64_t>(Tk, p->seqlen_q) : Tk, fa::kFwdKeys);
      return fa::fwd_key_split((int64_t)p->batch * p->heads_q * ceil_div(p->seqlen_q, fa::kFwdRows), nt, f.rows, p->head_dim,
                               true, false);
    };
    f.nsp = ranges(p->seqlen_p, false);
    f.nso = ranges(p->seqlen_k, p->is_causal != 0);
    // (a single range writes O itself)
    f.bytes = f.nsp + f.nso == 1 ? 0 : f.rows * (f.nsp + f.nso) * (p->head_dim + 2) * (int64_t)sizeof(float);
    return f;
  }
  // The prefix in blocks of 128 rows sharing its 64-key tiles, where those give every CU four tiles;
  // else in blocks of 32.  In us, wide / not (bf16, Hq 32, Hk 8, D 128, one row of B sequences):
  // B24 Tp8192 20.7 / 23.1, B48 Tp8192 and 256 own 32.5 / 34.4, B32 Tp32000 54.3 / 64.4, B20 Tq16
  // Hq16 Hk4 Tp4000 37 / 44; with less B32 Tp1000 17.4 / 16.4, B60 Hk1 D64 Tp4000 20.7 / 19.2.
  const int64_t wide_tiles = p->heads_k * ceil_div(TG * p->batch, fa::kWideRows) * ceil_div(p->seqlen_p, 64);
  f.wide = p->head_dim <= 128 && TG * p->batch > 64 && wide_tiles >= 4 * fa::kCus;
  const int rows_p = f.wide ? fa::kWideRows : 32, keys_p = f.wide ? 64 : kt;
  const int64_t rbp = ceil_div(TG * p->batch, rows_p), rbo = ceil_div(TG, 32);
  const int64_t ntp = ceil_div(p->seqlen_p, keys_p), nto = ceil_div(p->seqlen_k, kt);
  const int64_t base_p = ntp ? p->heads_k * rbp : 0, base_o = nto ? (int64_t)p->batch * p->heads_k * rbo : 0;
  // Tiles per range: one round of workgroups (two per CU; wide ones beside the own keys': one), four
  // tiles for every wave where there are as many, fewer only until every CU has a workgroup; no
  // more slots than the join holds.  (B16 Tp8192: ranges of 4 tiles 26.7 us, 16 16.9, 24 18.0; own keys of
  // B64 Tk512 in two rounds 28.3, in one 24.8; B1 Hq32 Hk8 own 1000: ranges of 16 tiles 11.8, of 4 8.6;
  // B12 Tq7 Hq24 Hk8 Tp1000: 16 15.0, 8 13.7, 4, two workgroups per CU, 17.8.)
  const int64_t slots = (p->head_dim > 128 ? 1 : 2) * fa::kCus;
  const int64_t work = (f.wide ? 0 : base_p * ntp) + base_o * nto;
  const int64_t per = std::max(std::min<int64_t>(16, std::max<int64_t>(4, ceil_div(work, fa::kCus))), ceil_div(work, slots));
  const int64_t per_p = f.wide ? std::max<int64_t>(4, ceil_div(wide_tiles, fa::kCus)) : per;
  // (half of the join's slots for each key set, and those the other leaves)
  const int64_t want_p = ceil_div(ntp, per_p), want_o = ceil_div(nto, per);
  auto ranges = [&](int64_t nt, int64_t want, int64_t other, int* ct) -> int {
    const int64_t ns = std::min<int64_t>(std::max<int64_t>(fa::kPrefixSlots / 2, fa::kPrefixSlots - other), want);
    *ct = ns ? (int)ceil_div(nt, ns) : 1;
    return ns ? (int)ceil_div(nt, *ct) : 0;
  };
  f.nsp = ranges(ntp, want_p, want_o, &f.ctp);
  f.nso = ranges(nto, want_o, want_p, &f.cto);
  f.np = base_p * f.nsp;
  f.no = base_o * f.nso;
  f.nrbp = (int)rbp;
  f.nrbo = (int)rbo;
  f.Tkp = (int)(nto * kt);
  f.bytes = f.rows * (f.nsp + f.nso) * (p->head_dim + 4) * (int64_t)sizeof(float);
  if (p->kw_out) f.bytes += f.rows * f.Tkp * (int64_t)sizeof(float);
  return f;
}

int check_prefix(const FaPrefixParams* p) {
  if (!p) return fail(FA_ERR_NULL, "params is NULL");
  const Sizes z{p->batch, p->seqlen_q, p->seqlen_k, p->heads_q, p->heads_k, p->head_dim, p->head_dim_in, p->dtype, p->scale};
  if (const int st = check_sizes(z, 0)) return st;
  if (p->seqlen_p < 0 || (int64_t)p->seqlen_p + p->seqlen_k < 1 || (int64_t)p->heads_k * p->seqlen_p >= kMaxRows)
    return fail(FA_ERR_SHAPE, "seqlen_p=%d seqlen_k=%d: at least one key, and 32-bit row indices", p->seqlen_p, p->seqlen_k);
  // what either way launches: below 2^31 threads
  const PrefixPlan f = prefix_plan(p);
  if (f.few ? f.np + f.no >= kMaxGrid || f.rows + (int64_t)p->batch * p->heads_k * ceil_div(p->seqlen_k, 1024) >= kMaxGrid
            : f.rows * std::max(f.nsp, f.nso) >= kMaxGrid * 128)
    return fail(FA_ERR_SHAPE, "problem too large for one launch");
  return FA_OK;
}

bool kw_fits(const FaPrefixParams* p) {
  return few_rows(p) && (int64_t)(p->heads_q / p->heads_k) * p->seqlen_q <= fa::kPrefixKwRows;
}

// Both key sets through the 256-row forward, then one combine of all ranges.
int prefix_many(const FaPrefixParams* p, const PrefixPlan& f) {
  fa::FwdArgs a{};
  a.q = p->q; a.o = p->o; a.lse = p->lse; a.olo = p->o_lo;
  a.qsb = p->q_stride_b; a.qst = p->q_stride_t; a.qsh = p->q_stride_h;
  a.osb = p->o_stride_b; a.ost = p->o_stride_t; a.osh = p->o_stride_h;
  a.olsb = p->o_lo_stride_b; a.olst = p->o_lo_stride_t; a.olsh = p->o_lo_stride_h;
  a.B = p->batch; a.Tq = p->seqlen_q; a.Hq = p->heads_q; a.Hk = p->heads_k; a.G = p->heads_q / p->heads_k;
  a.Dv = p->head_dim_in ? p->head_dim_in : p->head_dim;
  scales(p->scale, &a.scale_log2, &a.qsign, &a.zero_scale);
  a.nqt = (int)ceil_div(p->seqlen_q, fa::kFwdRows);   // (the precise forms' blocks)
  a.fine = 1;
  const int64_t rows = f.rows, ns = f.nsp + f.nso;
  float* part_o = ns > 1 ? (float*)p->workspace : nullptr;
  float* part_ml = ns > 1 ? part_o + rows * ns * p->head_dim : nullptr;
  const hipStream_t s = (hipStream_t)p->stream;
  int st;
  if (f.nsp) {
    fa::FwdArgs x = a;
    x.k = p->pk; x.v = p->pv;   // every sequence's: batch stride 0
    x.kst = p->pk_stride_t; x.ksh = p->pk_stride_h; x.vst = p->pv_stride_t; x.vsh = p->pv_stride_h;
    x.Tk = p->seqlen_p;
    x.ns = f.nsp; x.part_o = part_o; x.part_ml = part_ml;
    if ((st = launch_status(fa::launch_fwd(x, p->head_dim, p->dtype, false, s), "fa_prefix_fwd"))) return st;
  }
  if (f.nso) {
    fa::FwdArgs x = a;
    const bool causal = p->is_causal != 0;
    x.k = p->k; x.v = p->v; x.mask = p->mask; x.score = p->score;
    x.ksb = p->k_stride_b; x.kst = p->k_stride_t; x.ksh = p->k_stride_h;
    x.vsb = p->v_stride_b; x.vst = p->v_stride_t; x.vsh = p->v_stride_h;
    x.msb = p->mask_stride_b; x.msh = p->mask_stride_h; x.msq = p->mask_stride_q;
    x.ssb = p->score_stride_b; x.ssh = p->score_stride_h; x.ssq = p->score_stride_q;
    x.Tk = p->seqlen_k; x.lengths = p->lengths;
    x.causal = causal;
    if (p->mask) {
      x.mws = (const char*)p->mask_ws;
      x.ml = fa::mask_layout(p->batch, p->heads_q, p->seqlen_q, p->seqlen_k, p->mask_stride_b == 0, p->mask_stride_h == 0);
    }
    x.ns = f.nso;
    if (ns > 1) {
      x.part_o = part_o + f.nsp * rows * p->head_dim;
      x.part_ml = part_ml + 2 * f.nsp * rows;
    }
    if ((st = launch_status(fa::launch_fwd(x, p->head_dim, p->dtype, causal, s), "fa_prefix_fwd own"))) return st;
  }
  if (ns == 1) return FA_OK;
  a.ns = (int)ns; a.part_o = part_o; a.part_ml = part_ml;
  return launch_status(fa::launch_fwd_combine(a, p->head_dim, p->dtype, s), "fa_prefix_fwd combine");
}

}  // namespace

extern "C" {

int fa_prefix_plan(const FaPrefixParams* p, FaPrefixPlan* plan) {
  if (const int st = check_prefix(p)) return st;
  if (!plan) return fail(FA_ERR_NULL, "plan is NULL");
  const PrefixPlan f = prefix_plan(p);
  *plan = FaPrefixPlan{f.few && (!p->kw_out || kw_fits(p)) ? 1 : 0, f.nsp, f.nso, f.few ? 0 : 1, f.bytes, f.wide ? 1 : 0, 0};
  return FA_OK;
}

int fa_prefix_fwd(const FaPrefixParams* p) {
  int st = check_prefix(p);
  if (st) return st;
  if ((st = check_operand("q", p->q, p->q_stride_b, p->q_stride_t, p->q_stride_h))) return st;
  if (p->seqlen_p > 0) {
    if ((st = check_operand("pk", p->pk, 0, p->pk_stride_t, p->pk_stride_h))) return st;
    if ((st = check_operand("pv", p->pv, 0, p->pv_stride_t, p->pv_stride_h))) return st;
    if ((st = check_step("pk", p->pk_stride_t)) || (st = check_step("pv", p->pv_stride_t))) return st;
  }
  if (p->seqlen_k > 0) {
    if ((st = check_operand("k", p->k, p->k_stride_b, p->k_stride_t, p->k_stride_h))) return st;
    if ((st = check_operand("v", p->v, p->v_stride_b, p->v_stride_t, p->v_stride_h))) return st;
    if ((st = check_step("k", p->k_stride_t)) || (st = check_step("v", p->v_stride_t))) return st;
  }
  if ((st = check_operand("o", p->o, p->o_stride_b, p->o_stride_t, p->o_stride_h))) return st;
  if (p->o_lo && (st = check_operand("o_lo", p->o_lo, p->o_lo_stride_b, p->o_lo_stride_t, p->o_lo_stride_h))) return st;
  if (!p->lse) return fail(FA_ERR_NULL, "lse is NULL");
  if (p->mask && (st = check_nonneg("mask", p->mask_stride_b, p->mask_stride_h, p->mask_stride_q))) return st;
  if (p->score && (st = check_nonneg("score", p->score_stride_b, p->score_stride_h, p->score_stride_q))) return st;
  if (p->kw_in && (st = check_nonneg("kw", p->kw_stride_b, p->kw_stride_h, 0))) return st;
  const PrefixPlan f = prefix_plan(p);
  const bool own = p->seqlen_k > 0;
  if (p->kw_out && !(f.few && kw_fits(p)))
    return fail(FA_ERR_SHAPE, "more query rows than key weights are taken with (fa_prefix_plan: few_rows 0)");
  if (!f.few) {
    if (p->lengths && own && (p->mask || p->score))
      return fail(FA_ERR_SHAPE, "lengths beside a mask or score are taken with few rows only (fa_prefix_plan: few_rows 0)");
    if (own && p->mask && !p->mask_ws)
      return fail(FA_ERR_WORKSPACE, "a mask needs its prepared workspace (fa_mask_prepare): mask_ws is NULL");
    if (own && p->mask && (uintptr_t)p->mask_ws % 256) return fail(FA_ERR_STRIDE, "mask_ws must be 256-byte aligned");
    if (own && p->score && (31 * p->score_stride_q + (int64_t)p->seqlen_k + 64) * 4 >= (1LL << 32))
      return fail(FA_ERR_STRIDE, "score query stride %lld: 32 score rows must span less than 4 GiB", (long long)p->score_stride_q);
  }
  if (f.bytes && (!p->workspace || p->workspace_bytes < f.bytes))
    return fail(FA_ERR_WORKSPACE, "workspace of %lld bytes needed, %lld given", (long long)f.bytes,
                (long long)(p->workspace ? p->workspace_bytes : 0));
  if (f.bytes && !aligned16(p->workspace)) return fail(FA_ERR_STRIDE, "workspace must be 16-byte aligned");
  if (!f.few) return prefix_many(p, f);

  fa::PrefixArgs a{};
  a.q = p->q; a.pk = p->pk; a.pv = p->pv; a.k = p->k; a.v = p->v;
  a.o = p->o; a.olo = p->o_lo; a.lse = p->lse;
  a.mask = own ? p->mask : nullptr; a.score = own ? p->score : nullptr; a.lengths = p->lengths;
  a.kw_in = p->kw_in; a.kw_out = own ? p->kw_out : nullptr;
  a.qsb = p->q_stride_b; a.qst = p->q_stride_t; a.qsh = p->q_stride_h;
  a.pkst = p->pk_stride_t; a.pksh = p->pk_stride_h; a.pvst = p->pv_stride_t; a.pvsh = p->pv_stride_h;
  a.ksb = p->k_stride_b; a.kst = p->k_stride_t; a.ksh = p->k_stride_h;
  a.vsb = p->v_stride_b; a.vst = p->v_stride_t; a.vsh = p->v_stride_h;
  a.osb = p->o_stride_b; a.ost = p->o_stride_t; a.osh = p->o_stride_h;
  a.olsb = p->o_lo_stride_b; a.olst = p->o_lo_stride_t; a.olsh = p->o_lo_stride_h;
  a.msb = p->mask_stride_b; a.msh = p->mask_stride_h; a.msq = p->mask_stride_q;
  a.ssb = p->score_stride_b; a.ssh = p->score_stride_h; a.ssq = p->score_stride_q;
  a.kwsb = p->kw_stride_b; a.kwsh = p->kw_stride_h;
  a.B = p->batch; a.Tq = p->seqlen_q; a.Tp = p->seqlen_p; a.Tk = p->seqlen_k;
  a.Hq = p->heads_q; a.Hk = p->heads_k; a.G = p->heads_q / p->heads_k;
  a.Dv = p->head_dim_in ? p->head_dim_in : p->head_dim;
  scales(p->scale, &a.scale_log2, &a.qsign, &a.zero_scale);
  a.causal = p->is_causal != 0;
  a.mask4 = mask_by_words(p->mask, p->mask_stride_b, p->mask_stride_h, p->mask_stride_q);
  a.nsp = f.nsp; a.nso = f.nso; a.ctp = f.ctp; a.cto = f.cto; a.nrbp = f.nrbp; a.nrbo = f.nrbo;
  a.np = (int)f.np; a.no = (int)f.no;
  a.wide = f.wide;
  a.part_o = (float*)p->workspace;
  a.part_ml = a.part_o + f.rows * (f.nsp + f.nso) * p->head_dim;
  a.logits = a.part_ml + f.rows * (f.nsp + f.nso) * 4;
  a.Tkp = f.Tkp;
  const hipStream_t s = (hipStream_t)p->stream;
  if ((st = launch_status(fa::launch_prefix_rows(a, p->head_dim, p->dtype, s), "fa_prefix_fwd"))) return st;
  return launch_status(fa::launch_prefix_join(a, p->head_dim, p->dtype, s), "fa_prefix_fwd join");
}

}  // extern "C"

namespace {

// ---- key weights --------------------------------------------------------------------------

struct KeyWPlan {
  int nkb, ns;
  int64_t far_elems, part_elems;
  int64_t bytes() const { return (far_elems + part_elems) * (int64_t)sizeof(float); }
};

KeyWPlan keyw_plan(const FaKeyWeightsParams* p) {
  KeyWPlan f{};
  const int64_t base = (int64_t)p->batch * p->heads_k;
  f.nkb = (int)ceil_div(p->seqlen_k, fa::keyw_block_keys(p->head_dim));
  const int64_t nt = ceil_div((int64_t)(p->heads_q / p->heads_k) * p->seqlen_q, 32);
  // parts of the row tiles: two rounds of two workgroups per CU, at least eight tiles each
  f.ns = (int)std::max<int64_t>(1, std::min<int64_t>({4 * fa::kCus / (base * f.nkb), nt / 8, 64}));
  f.far_elems = p->score ? 2 * (int64_t)p->batch * p->heads_q * p->seqlen_q : 0;
  f.far_elems = (f.far_elems + 3) & ~3LL;
  f.part_elems = f.ns > 1 ? f.ns * base * p->seqlen_k : 0;
  return f;
}

int check_keyw(const FaKeyWeightsParams* p) {
  if (!p) return fail(FA_ERR_NULL, "params is NULL");
  const Sizes z{p->batch, p->seqlen_q, p->seqlen_k, p->heads_q, p->heads_k, p->head_dim, p->head_dim_in, p->dtype, p->scale};
  if (const int st = check_sizes(z, 1)) return st;
  if ((int64_t)p->batch * p->heads_k * ceil_div(p->seqlen_k, fa::keyw_block_keys(p->head_dim)) >= kMaxGrid ||
      (int64_t)p->batch * p->heads_q * ceil_div(p->seqlen_q, 32) >= kMaxGrid)
    return fail(FA_ERR_SHAPE, "problem too large for one launch");
  return FA_OK;
}

}  // namespace

extern "C" {

int fa_key_weights_plan(const FaKeyWeightsParams* p, int64_t* workspace_bytes) {
  if (const int st = check_keyw(p)) return st;
  if (!workspace_bytes) return fail(FA_ERR_NULL, "workspace_bytes is NULL");
  *workspace_bytes = keyw_plan(p).bytes();
  return FA_OK;
}

int fa_key_weights(const FaKeyWeightsParams* p) {
  int st = check_keyw(p);
  if (st) return st;
  if ((st = check_operand("q", p->q, p->q_stride_b, p->q_stride_t, p->q_stride_h))) return st;
  if ((st = check_operand("k", p->k, p->k_stride_b, p->k_stride_t, p->k_stride_h)) || (st = check_step("k", p->k_stride_t))) return st;
  if (!p->lse || !p->kw_out) return fail(FA_ERR_NULL, "lse or kw_out is NULL");
  if (p->mask && (st = check_nonneg("mask", p->mask_stride_b, p->mask_stride_h, p->mask_stride_q))) return st;
  if (p->score && (st = check_nonneg("score", p->score_stride_b, p->score_stride_h, p->score_stride_q))) return st;
  if (p->kw_in && (st = check_nonneg("kw", p->kw_stride_b, p->kw_stride_h, 0))) return st;
  const KeyWPlan f = keyw_plan(p);
  if (f.bytes() && (!p->workspace || p->workspace_bytes < f.bytes()))
    return fail(FA_ERR_WORKSPACE, "workspace of %lld bytes needed, %lld given", (long long)f.bytes(),
                (long long)(p->workspace ? p->workspace_bytes : 0));
  if (f.bytes() && !aligned16(p->workspace)) return fail(FA_ERR_STRIDE, "workspace must be 16-byte aligned");
  fa::KeyWArgs a{};
  a.q = p->q; a.k = p->k; a.lse = p->lse;
  a.mask = p->mask; a.score = p->score; a.lengths = p->lengths;
  a.kw_in = p->kw_in; a.kw_out = p->kw_out;
  a.qsb = p->q_stride_b; a.qst = p->q_stride_t; a.qsh = p->q_stride_h;
  a.ksb = p->k_stride_b; a.kst = p->k_stride_t; a.ksh = p->k_stride_h;
  a.msb = p->mask_stride_b; a.msh = p->mask_stride_h; a.msq = p->mask_stride_q;
  a.ssb = p->score_stride_b; a.ssh = p->score_stride_h; a.ssq = p->score_stride_q;
  a.kwsb = p->kw_stride_b; a.kwsh = p->kw_stride_h;
  a.B = p->batch; a.Tq = p->seqlen_q; a.Tk = p->seqlen_k; a.Hq = p->heads_q; a.Hk = p->heads_k;
  a.G = p->heads_q / p->heads_k;
  a.Dv = p->head_dim_in ? p->head_dim_in : p->head_dim;
  scales(p->scale, &a.scale_log2, &a.qsign, &a.zero_scale);
  a.causal = p->is_causal != 0;
  a.mask4 = mask_by_words(p->mask, p->mask_stride_b, p->mask_stride_h, p->mask_stride_q);
  a.ns = f.ns;
  a.nkb = f.nkb;
  a.far_ml = (float*)p->workspace;
  a.part = a.far_ml + f.far_elems;
  return launch_status(fa::launch_key_weights(a, p->head_dim, p->dtype, (hipStream_t)p->stream), "fa_key_weights");
}

// ---- eviction -----------------------------------------------------------------------------

int fa_evict(const FaEvictParams* p) {
  if (!p) return fail(FA_ERR_NULL, "params is NULL");
  if (p->batch < 1 || p->seqlen_k < 1 || p->heads_k < 1 || p->head_dim < 1)
    return fail(FA_ERR_SHAPE, "sizes must be >= 1 (B=%d Tk=%d Hk=%d D=%d)", p->batch, p->seqlen_k, p->heads_k, p->head_dim);
  if (p->head_dim > 65536 || (int64_t)p->batch * p->heads_k >= (1 << 21) || !rows_fit(p->batch, p->heads_k, p->seqlen_k))
    return fail(FA_ERR_SHAPE, "problem too large (B*H*T below 2^31 - 2^16, B*H below 2^21)");
  if (p->keep < 1 || p->keep > p->seqlen_k) return fail(FA_ERR_SHAPE, "keep %d must lie in [1, %d]", p->keep, p->seqlen_k);
  if (p->recent < 0 || p->recent > p->keep) return fail(FA_ERR_SHAPE, "recent %d must lie in [0, keep = %d]", p->recent, p->keep);
  if (!p->k || !p->v || !p->kw || !p->k_out || !p->v_out || !p->kw_out || !p->index_out)
    return fail(FA_ERR_NULL, "a required pointer is NULL");
  const int64_t st[] = {p->k_stride_b, p->k_stride_t, p->k_stride_h, p->v_stride_b, p->v_stride_t, p->v_stride_h,
                        p->out_stride_b, p->out_stride_t, p->out_stride_h};
  for (int64_t s : st)
    if (s < 0) return fail(FA_ERR_STRIDE, "strides must be non-negative");
  if (p->kw_stride_b < 0 || p->kw_stride_h < 0) return fail(FA_ERR_STRIDE, "strides must be non-negative");
  fa::EvictArgs a{};
  a.k = p->k; a.v = p->v; a.kw = p->kw; a.lengths = p->lengths;
  a.ko = p->k_out; a.vo = p->v_out; a.kwo = p->kw_out; a.idx = p->index_out;
  a.ksb = p->k_stride_b; a.kst = p->k_stride_t; a.ksh = p->k_stride_h;
  a.vsb = p->v_stride_b; a.vst = p->v_stride_t; a.vsh = p->v_stride_h;
  a.kwsb = p->kw_stride_b; a.kwsh = p->kw_stride_h;
  a.osb = p->out_stride_b; a.ost = p->out_stride_t; a.osh = p->out_stride_h;
  a.B = p->batch; a.Tk = p->seqlen_k; a.Hk = p->heads_k; a.D = p->head_dim; a.keep = p->keep; a.recent = p->recent;
  a.vec = p->head_dim % 8 == 0 && aligned16(p->k) && aligned16(p->v) && aligned16(p->k_out) && aligned16(p->v_out);
  for (int64_t s : st) a.vec = a.vec && s % 8 == 0;
  // A workgroup per CU, each with 64 rows to copy at least: two would make each other wait for the
  // same selection (B1 Tk 16384 Hk8 D128 keep 4096: 16.4 us, with two 26.9; B16 Tk 3001 Hk4 D96 keep
  // 1500: 19.7 and 25.5; half as many: 17.3 and 20.3).
  const int64_t heads = (int64_t)p->batch * p->heads_k;
  a.nw = (int)std::max(ceil_div(p->keep, fa::kEvictShare), std::min<int64_t>(std::max<int64_t>(fa::kCus / heads, 1), ceil_div(p->keep, 64)));
  if (heads * a.nw >= (1 << 21)) return fail(FA_ERR_SHAPE, "problem too large for one launch");
  return launch_status(fa::launch_evict(a, (hipStream_t)p->stream), "fa_evict");
}

// ---- rotary positions ---------------------------------------------------------------------

int fa_rotary(const FaRotaryParams* p) {
  if (!p) return fail(FA_ERR_NULL, "params is NULL");
  if (p->batch < 1 || p->seqlen < 1 || p->heads_q < 1 || p->heads_k < 0 || p->head_dim < 1 || p->head_dim > 256)
    return fail(FA_ERR_SHAPE, "sizes must be >= 1, head_dim up to 256 (B=%d T=%d Hq=%d Hk=%d D=%d)", p->batch, p->seqlen,
                p->heads_q, p->heads_k, p->head_dim);
  if ((int64_t)p->batch * p->seqlen >= (1LL << 25) || (int64_t)p->heads_q + p->heads_k >= (1 << 16))
    return fail(FA_ERR_SHAPE, "problem too large (B*T below 2^25, heads below 2^16)");
  if (p->rotary < 2 || p->rotary % 2 || p->rotary > p->head_dim)
    return fail(FA_ERR_HEAD_DIM, "rotary %d must be even and lie in [2, head_dim = %d]", p->rotary, p->head_dim);
  if (p->axes < 1 || p->axes > FA_ROTARY_AXES) return fail(FA_ERR_SHAPE, "axes %d must lie in [1, %d]", p->axes, (int)FA_ROTARY_AXES);
  if (p->dtype != FA_DTYPE_BF16 && p->dtype != FA_DTYPE_FP16) return fail(FA_ERR_DTYPE, "unsupported dtype code %d", p->dtype);
  if (p->sign != 1 && p->sign != -1) return fail(FA_ERR_SHAPE, "sign must be 1 or -1");
  if (!p->q || !p->q_out || (p->heads_k && (!p->k || !p->k_out)) || !p->positions || !p->inv_freq)
    return fail(FA_ERR_NULL, "a required pointer is NULL");
  fa::RotaryArgs a{};
  int64_t sum = 0;
  for (int i = 0; i < p->axes; ++i) {
    if (p->sections[i] < 0) return fail(FA_ERR_SHAPE, "section %d is negative", i);
    sum += p->sections[i];
    a.ends[i] = (int)std::min<int64_t>(sum, INT32_MAX);
  }
  if (sum != p->rotary / 2) return fail(FA_ERR_SHAPE, "sections add up to %lld pairs, rotary has %d", (long long)sum, p->rotary / 2);
  a.q = p->q; a.k = p->k; a.qo = p->q_out; a.ko = p->k_out; a.pos = p->positions; a.freq = p->inv_freq;
  a.qsb = p->q_stride_b; a.qst = p->q_stride_t; a.qsh = p->q_stride_h;
  a.ksb = p->k_stride_b; a.kst = p->k_stride_t; a.ksh = p->k_stride_h;
  a.qosb = p->qo_stride_b; a.qost = p->qo_stride_t; a.qosh = p->qo_stride_h;
  a.kosb = p->ko_stride_b; a.kost = p->ko_stride_t; a.kosh = p->ko_stride_h;
  a.psa = p->pos_stride_a; a.psb = p->pos_stride_b; a.pst = p->pos_stride_t;
  a.B = p->batch; a.T = p->seqlen; a.Hq = p->heads_q; a.Hk = p->heads_k; a.D = p->head_dim; a.R2 = p->rotary / 2;
  a.naxes = p->axes;
  a.pos64 = p->positions_64 != 0;
  a.adjacent = p->adjacent != 0;
  a.sign = (float)p->sign;
  const int64_t st[] = {a.qsb, a.qst, a.qsh, a.ksb, a.kst, a.ksh, a.qosb, a.qost, a.qosh, a.kosb, a.kost, a.kosh};
  a.vec = p->head_dim % 8 == 0 && p->rotary % (a.adjacent ? 8 : 16) == 0 && aligned16(p->q) && aligned16(p->k) &&
          aligned16(p->q_out) && aligned16(p->k_out);
  for (int64_t s : st) a.vec = a.vec && s % 8 == 0;
  return launch_status(fa::launch_rotary(a, p->dtype, (hipStream_t)p->stream), "fa_rotary");
}

}  // extern "C"
