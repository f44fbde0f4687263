// Kernel argument blocks and launchers of the cache operators (internal to the library).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fa {

// Few query rows per sequence over a shared prefix and own keys (fa_prefix.hip).
// A problem's partial results: slot s < nsp is range s of the prefix, slot nsp + s range s
// of the own keys.  Row ri = (b Hq + h) Tq + tq leaves, in slot s, its O (not divided by its
// sum) at part_o[(s rows + ri) D ..], and at part_ml[4 (s rows + ri) ..] its running maximum
// (base 2; -inf: nothing kept, no O written), its sum and its largest raw logit (with a score).
struct PrefixArgs {
  const void* q; const void* pk; const void* pv; const void* k; const void* v;
  void* o; void* olo; float* lse;
  const uint8_t* mask; const float* score; const int32_t* lengths;
  const float* kw_in; float* kw_out;
  int64_t qsb, qst, qsh, pkst, pksh, pvst, pvsh, ksb, kst, ksh, vsb, vst, vsh, osb, ost, osh, olsb, olst, olsh;
  int64_t msb, msh, msq, ssb, ssh, ssq, kwsb, kwsh;
  int B, Tq, Tp, Tk, Hq, Hk, G;
  int Dv;               // columns that exist (a multiple of 16)
  float scale_log2, qsign;
  int zero_scale, causal, mask4;
  int nsp, nso;         // key ranges
  int ctp, cto;         // 32-key tiles of each range (the last may have fewer)
  int nrbp, nrbo;       // 32-row blocks: of a kv-head's rows over the batch, of one sequence's
  int np, no;           // workgroups: prefix, own
  int wide;             // the prefix in blocks of kWideRows rows (ctp counts 64-key tiles then)
  float* part_o;
  float* part_ml;
  float* logits;        // with kw_out: raw logits [rows][Tkp] of the own keys (-inf: dropped)
  int Tkp;
};
constexpr int kPrefixSlots = 128;     // most key ranges of a problem: two per lane of the joining wave
constexpr int kWideRows = 128;
// Most rows of a kv-head's group with kw_out: each leaves its logits, 4 bytes a key to write and read
// again; past them a pass of its own over K is shorter.  Together / apart in us (bf16, D 128): B1
// Tk16000 Hq32 Hk8 4 rows of a group 20 / 30, 16 27.4 / 30.3, 32 38 / 31, 64 65 / 38; B8 Tk8000 16
// 78 / 94, 32 95 / 97, 64 160 / 118; B1 Tk3000 32 30 / 21.6; B16 Tk<=4096 Hq32 Hk8 4 55 / 85.
constexpr int kPrefixKwRows = 16;
int prefix_tile_keys();
hipError_t launch_prefix_rows(const PrefixArgs& a, int D, int dtype, hipStream_t s);
hipError_t launch_prefix_join(const PrefixArgs& a, int D, int dtype, hipStream_t s);

// Key weights from an LSE (fa_keyw.hip).
struct KeyWArgs {
  const void* q; const void* k; const float* lse;
  const uint8_t* mask; const float* score; const int32_t* lengths;
  const float* kw_in; float* kw_out;
  int64_t qsb, qst, qsh, ksb, kst, ksh, msb, msh, msq, ssb, ssh, ssq, kwsb, kwsh;
  int B, Tq, Tk, Hq, Hk, G, Dv;
  float scale_log2, qsign;
  int zero_scale, causal, mask4;
  int ns;               // parts of the row tiles; with ns > 1 each part leaves its sums in part
  int nkb;              // key blocks
  float* part;          // [ns][B Hk][Tk]
  float* far_ml;        // with a score: [rows][2] largest raw logit and sum, of rows that need them
};
int keyw_block_keys(int D);
hipError_t launch_key_weights(const KeyWArgs& a, int D, int dtype, hipStream_t s);

struct EvictArgs {
  const void* k; const void* v; const float* kw; const int32_t* lengths;
  void* ko; void* vo; float* kwo; int64_t* idx;
  int64_t ksb, kst, ksh, vsb, vst, vsh, kwsb, kwsh, osb, ost, osh;
  int B, Tk, Hk, D, keep, recent;
  int vec;              // rows of 16-byte pieces, aligned
  int nw;               // workgroups per (sequence, kv-head), each with ceil(keep / nw) places
};
constexpr int kEvictShare = 2048;   // most places of a workgroup
hipError_t launch_evict(const EvictArgs& a, hipStream_t s);

constexpr int kRotaryAxes = 8;
struct RotaryArgs {
  const void* q; const void* k; void* qo; void* ko;
  const void* pos; const float* freq;
  int64_t qsb, qst, qsh, ksb, kst, ksh, qosb, qost, qosh, kosb, kost, kosh, psa, psb, pst;
  int B, T, Hq, Hk, D, R2;    // R2: pairs
  int naxes, ends[kRotaryAxes];   // pairs [ends[a - 1], ends[a]) belong to axis a
  int pos64, adjacent;
  float sign;
  int vec;              // pieces of 8 columns, 16-byte aligned
};
hipError_t launch_rotary(const RotaryArgs& a, int dtype, hipStream_t s);

}  // namespace fa
