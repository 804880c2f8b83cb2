// Exact attention of a tree of drafted tokens over a paged K/V cache (exb_tree_attention).
//
//   s_t = shr((q . k_t) * INV, 32 - qs - ks_t)     over the visible positions t
//   e_t = exp table at (max s - s_t), Q24;  p_t = (e_t << 20) // sum(e);  out = shr(sum p_t v_t, 20)
//
// p needs the row's final maximum and sum (a floor division by the sum: no rescaling afterwards
// gives the same bits), so a row goes over its positions three times.
#include <cmath>

#include "exb_internal.h"
#include "treedev.cuh"

namespace exb {

// One CTA per (row, head): the scores are computed anew in each of the three passes.
constexpr int TS_THREADS = 128;

__global__ void __launch_bounds__(TS_THREADS) k_tree_simple(const TreeArgs a) {
  __shared__ int64_t red[TS_THREADS / 32];
  __shared__ int64_t pt[TS_THREADS];
  __shared__ const int32_t* vrow[TS_THREADS];
  __shared__ int16_t qsm[128];
  const int r = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const exb_kv_view& kv = a.kv;
  const int hd = kv.hd, j = h / a.rep;
  if (r == 0 && h == 0)                                // every sequence is looked over once
    for (int i = tid; i < a.B; i += TS_THREADS) tree_seq(a, i, true);
  int b = -1;
  for (int i = 0; i < a.B; ++i)
    if (r >= a.row_start[i] && r < a.row_start[i + 1]) { b = i; break; }
  int64_t* out = a.out + ((size_t)r * a.H + h) * hd;
  TreeSeq sq;
  if (b >= 0) sq = tree_seq(a, b, false);
  const uint64_t* mask = a.mask + (size_t)r * a.W;
  const int32_t* row = a.table + (size_t)(b < 0 ? 0 : b) * a.MP;
  const int qs = a.qs[(size_t)r * a.H + h];
  if (tid < hd) qsm[tid] = a.q[((size_t)r * a.H + h) * hd + tid];
  __syncthreads();
  auto seen = [&](int t) { return t < sq.ctx || ((mask[(t - sq.ctx) >> 6] >> ((t - sq.ctx) & 63)) & 1); };
  // score of position t; false where it is hidden
  auto score = [&](int t, int64_t& s, int& pg, int& off) {
    if (t >= sq.S || !seen(t)) return false;
    pg = page_of(kv, row, t, off, a.status);
    if (pg < 0) return false;
    const int16_t* k = kv.k + (int64_t)pg * kv.k_page + (int64_t)j * kv.k_head + (int64_t)off * kv.k_pos;
    int64_t acc = 0;
    for (int d = 0; d < hd; ++d) acc += (int)qsm[d] * (int)k[d];
    const int ks = kv.ks[(int64_t)pg * kv.s_page + (int64_t)j * kv.s_head + (int64_t)off * kv.s_pos];
    s = shr64((int64_t)((uint64_t)acc * (uint64_t)a.inv), 32 - qs - ks);
    return true;
  };
  auto block_max = [&](int64_t v) {
    for (int o = 16; o > 0; o >>= 1) { const int64_t w = __shfl_xor_sync(0xffffffffu, v, o); v = w > v ? w : v; }
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = v;
    __syncthreads();
    for (int i = 0; i < TS_THREADS / 32; ++i) v = red[i] > v ? red[i] : v;
    return v;
  };
  int64_t s;
  int pg, off;
  int64_t m = INT64_MIN;
  for (int t = tid; t < sq.S; t += TS_THREADS)
    if (score(t, s, pg, off)) m = s > m ? s : m;
  m = block_max(m);
  int64_t sum = 0;
  for (int t = tid; t < sq.S; t += TS_THREADS)
    if (score(t, s, pg, off)) sum += tree_exp(a.exp_t, (uint64_t)m - (uint64_t)s);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if ((tid & 31) == 0) red[tid >> 5] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < TS_THREADS / 32; ++i) sum += red[i];
  uint64_t acc = 0;
  for (int t0 = 0; t0 < sq.S; t0 += TS_THREADS) {
    int64_t p = 0;
    const int32_t* v = nullptr;
    if (score(t0 + tid, s, pg, off)) {
      p = (int64_t)(((uint64_t)tree_exp(a.exp_t, (uint64_t)m - (uint64_t)s) << 20) / (uint64_t)sum);
      v = kv.v + (int64_t)pg * kv.v_page + (int64_t)j * kv.v_head + (int64_t)off * kv.v_pos;
    }
    __syncthreads();
    pt[tid] = p;
    vrow[tid] = v;
    __syncthreads();
    if (tid < hd)
      for (int t = 0; t < TS_THREADS; ++t)
        if (pt[t]) acc += (uint64_t)pt[t] * (uint64_t)(int64_t)vrow[t][tid];
  }
  if (tid < hd) out[tid] = shr64((int64_t)acc, 20);
}

static cudaError_t launch_tree_attention(const TreeArgs& a, cudaStream_t st) {
  k_tree_simple<<<dim3(a.R, a.H), TS_THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

// what is wrong with a cache description, or nullptr
const char* kv_view_error(const exb_kv_view* kv) {
  if (!kv || !kv->k || !kv->ks || !kv->v) return "null cache pointer";
  if (kv->layers < 1 || kv->pages < 1 || kv->KV < 1 || kv->page < 1) return "layers, pages, KV and page must be positive";
  if (kv->hd != 16 && kv->hd != 32 && kv->hd != 64 && kv->hd != 128) return "hd must be 16, 32, 64 or 128";
  if (((uintptr_t)kv->k | (uintptr_t)kv->v) & 15) return "k and v must be 16-byte aligned";
  if ((kv->k_layer | kv->k_page | kv->k_head | kv->k_pos) & 7) return "K strides must be multiples of 8 elements";
  if ((kv->v_layer | kv->v_page | kv->v_head | kv->v_pos) & 3) return "V strides must be multiples of 4 elements";
  return nullptr;
}

}  // namespace exb

using namespace exb;

#define TREE_FAIL(code, msg)                    \
  do {                                          \
    set_last_error(msg);                        \
    return code;                                \
  } while (0)

extern "C" {

size_t exb_tree_attention_workspace_bytes(int R, int H, int KV, int hd) {
  (void)R; (void)H; (void)KV; (void)hd;
  return 256;
}

int exb_tree_attention(const exb_kv_view* kv, const int16_t* q, const int32_t* qs, int R, int H, const int32_t* table,
                       int B, int max_pages, const int32_t* ctx, const int32_t* row_start, const uint64_t* mask,
                       int mask_words, const int32_t* exp_t, int64_t* out, void* workspace, size_t workspace_bytes,
                       int32_t* status, void* stream) {
  if (const char* why = kv_view_error(kv)) TREE_FAIL(EXB_EINVAL, std::string("exb_tree_attention: ") + why);
  if (R < 0 || B < 0) TREE_FAIL(EXB_EINVAL, "exb_tree_attention: negative R or B");
  if (R == 0) return EXB_OK;
  if (H < 1 || H % kv->KV) TREE_FAIL(EXB_EINVAL, "exb_tree_attention: H must be a positive multiple of KV");
  if (!q || !qs || !exp_t || !out || !mask || (B && (!table || !ctx)) || !row_start)
    TREE_FAIL(EXB_EINVAL, "exb_tree_attention: null argument");
  if (mask_words < 1 || mask_words > 64 || max_pages < 1) TREE_FAIL(EXB_EINVAL, "exb_tree_attention: 1 <= mask_words <= 64 and max_pages >= 1");
  if ((int64_t)max_pages * kv->page >= (1ll << 30)) TREE_FAIL(EXB_EINVAL, "exb_tree_attention: a table row names 2^30 positions or more");
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) TREE_FAIL(EXB_EINVAL, "exb_tree_attention: q, out and workspace must be 16-byte aligned");
  if (!workspace || workspace_bytes < exb_tree_attention_workspace_bytes(R, H, kv->KV, kv->hd))
    TREE_FAIL(EXB_EINVAL, "exb_tree_attention: workspace too small");
  TreeArgs a;
  a.kv = *kv; a.q = q; a.qs = qs; a.table = table; a.ctx = ctx; a.row_start = row_start; a.mask = mask;
  a.exp_t = exp_t; a.out = out; a.status = status; a.R = R; a.H = H; a.rep = H / kv->KV; a.B = B; a.MP = max_pages;
  a.W = mask_words; a.cap = (int64_t)max_pages * kv->page;
  a.inv = (int64_t)std::nearbyint(65536.0 / std::sqrt((double)kv->hd));
  const cudaError_t e = launch_tree_attention(a, (cudaStream_t)stream);
  if (e != cudaSuccess) TREE_FAIL(EXB_ECUDA, std::string("exb_tree_attention: ") + cudaGetErrorString(e));
  return EXB_OK;
}

}  // extern "C"
