// Device helpers shared by the tree-decoding kernels: the paged cache, a tree's rows and mask.
#pragma once
#include "common.cuh"
#include "exactb200.h"

namespace exb {

// Arguments of the tree attention kernels (see exb_tree_attention).
struct TreeArgs {
  exb_kv_view kv;
  const int16_t* q = nullptr;
  const int32_t* qs = nullptr;
  const int32_t* table = nullptr;
  const int32_t* ctx = nullptr;
  const int32_t* row_start = nullptr;
  const uint64_t* mask = nullptr;
  const int32_t* exp_t = nullptr;
  int64_t* out = nullptr;
  int32_t* status = nullptr;
  int R = 0, H = 0, rep = 0, B = 0, MP = 0, W = 0;
  int64_t cap = 0;                       // positions a table row can name: MP * page
  int64_t inv = 0;                       // round(2^16 / sqrt(hd))
};

// One sequence's rows and positions, cut to what the arguments can hold.
struct TreeSeq {
  int r0 = 0, T = 0;                     // first row, nodes
  int ctx = 0;                           // positions that every row sees
  int S = 0;                             // ctx + nodes that have a position in the table
};

EXB_DEV TreeSeq tree_seq(const TreeArgs& a, int b, bool report) {
  TreeSeq s;
  const int lo = a.row_start[b], hi = a.row_start[b + 1], c = a.ctx[b];
  bool bad = lo < 0 || hi > a.R || hi < lo || c < 0;
  if (!bad) {
    s.r0 = lo;
    s.T = hi - lo;
    s.ctx = (int)min((int64_t)c, a.cap);
    s.S = (int)min((int64_t)s.ctx + min(s.T, 64 * a.W), a.cap);
    bad = (int64_t)c + s.T > a.cap || s.T > 64 * a.W;
  }
  if (bad && report) set_err(a.status, ERR_BOUNDS);
  return s;
}

// page of position pos, or -1 (reported) where the table names none
EXB_DEV int page_of(const exb_kv_view& kv, const int32_t* __restrict__ row, int pos, int& off, int32_t* status) {
  const int i = pos / kv.page;
  off = pos - i * kv.page;
  const int pg = row[i];
  if ((unsigned)pg < (unsigned)kv.pages) return pg;
  set_err(status, ERR_BOUNDS);
  return -1;
}

// exp table at d = max - score (exact_llm.py:109-115).  d is not negative unless the difference left
// 64 bits, and then it is past the table's end in truth: both compare as large.
EXB_DEV int64_t tree_exp(const int32_t* __restrict__ T, uint64_t d) {
  return d >= (40ull << 16) ? 0 : exp_lookup(T, (int64_t)d);
}

}  // namespace exb
