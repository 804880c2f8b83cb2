// Verification of drafted trees (exb_tree_verify): the target's own token of every row, from a
// given random number or as the argmax, then the walk along the drafted tokens that agree.
//
//   y = shr(logit * tnum, 16), p = (e << 20) // sum(e) with e the exp table at (max y - y),
//   token = first index whose running sum of p exceeds (u20 * sum(p)) >> 20     (exact_llm.py:243-259)
#include "exb_internal.h"
#include "treedev.cuh"

namespace exb {

constexpr int TV_THREADS = 1024;

struct VerArgs {
  const int64_t* logits = nullptr; int64_t ld = 0;
  const int32_t* u20 = nullptr;
  int64_t tnum = 0;
  const int32_t *tokens = nullptr, *parent = nullptr, *row_start = nullptr, *exp_t = nullptr;
  int32_t *sampled = nullptr, *n = nullptr, *path = nullptr, *out_tokens = nullptr;
  int R = 0, V = 0, B = 0, max_len = 0;
};

// One CTA per row; thread t owns the t-th of 1024 contiguous slices of the row.
__global__ void __launch_bounds__(TV_THREADS) k_tree_sample(const VerArgs a) {
  __shared__ uint64_t red[TV_THREADS / 32];
  __shared__ int64_t scan[TV_THREADS];
  __shared__ int tok;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t* row = a.logits + (int64_t)r * a.ld;
  const int u = a.u20[r];
  const int c0 = (int)((int64_t)a.V * tid / TV_THREADS), c1 = (int)((int64_t)a.V * (tid + 1) / TV_THREADS);
  auto y_at = [&](int i) {
    return u < 0 ? row[i] : shr64((int64_t)((uint64_t)row[i] * (uint64_t)a.tnum), 16);
  };
  auto block_max = [&](int64_t v) {
    for (int o = 16; o > 0; o >>= 1) { const int64_t w = __shfl_xor_sync(0xffffffffu, v, o); v = w > v ? w : v; }
    __syncthreads();
    if (lane == 0) red[warp] = (uint64_t)v;
    __syncthreads();
    for (int i = 0; i < TV_THREADS / 32; ++i) v = (int64_t)red[i] > v ? (int64_t)red[i] : v;
    return v;
  };
  int64_t m = INT64_MIN;
  int first = INT32_MAX;
  for (int i = c0; i < c1; ++i) {
    const int64_t y = y_at(i);
    if (y > m || first == INT32_MAX) { m = y; first = i; }
  }
  const int64_t M = block_max(m);
  if (tid == 0) tok = a.V - 1;
  __syncthreads();
  if (u < 0) {
    if (m == M && first != INT32_MAX) atomicMin(&tok, first);
  } else {
    int64_t s = 0;
    for (int i = c0; i < c1; ++i) s += tree_exp(a.exp_t, (uint64_t)M - (uint64_t)y_at(i));
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();
    if (lane == 0) red[warp] = (uint64_t)s;
    __syncthreads();
    uint64_t S = 0;
    for (int i = 0; i < TV_THREADS / 32; ++i) S += red[i];
    auto p_at = [&](int i) { return ((uint64_t)tree_exp(a.exp_t, (uint64_t)M - (uint64_t)y_at(i)) << 20) / S; };
    int64_t ps = 0;
    for (int i = c0; i < c1; ++i) ps += (int64_t)p_at(i);
    scan[tid] = ps;
    __syncthreads();
    for (int o = 1; o < TV_THREADS; o <<= 1) {
      const int64_t add = tid >= o ? scan[tid - o] : 0;
      __syncthreads();
      scan[tid] += add;
      __syncthreads();
    }
    const int64_t before = scan[tid] - ps;
    const int64_t target = (int64_t)(((uint64_t)u * (uint64_t)scan[TV_THREADS - 1]) >> 20);
    if (before <= target && target < before + ps) {
      int64_t cum = before;
      for (int i = c0; i < c1; ++i) {
        cum += (int64_t)p_at(i);
        if (cum > target) { tok = i; break; }
      }
    }
  }
  __syncthreads();
  if (tid == 0) a.sampled[r] = tok;
}

// One warp per sequence walks from node 0: 32 candidates at a time, the lowest one that fits.
__global__ void __launch_bounds__(32) k_tree_walk(const VerArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  int r0 = a.row_start[b], r1 = a.row_start[b + 1];
  if (r0 < 0 || r1 > a.R || r1 < r0) r1 = r0 = 0;
  const int T = r1 - r0;
  int len = 0, cur = T > 0 ? 0 : -1;
  while (cur >= 0 && len < a.max_len) {
    const int t = a.sampled[r0 + cur];
    if (lane == 0) {
      a.path[(size_t)b * a.max_len + len] = cur;
      a.out_tokens[(size_t)b * a.max_len + len] = t;
    }
    ++len;
    int next = -1;
    for (int i0 = cur + 1; i0 < T && next < 0; i0 += 32) {         // children come after their parent
      const int i = i0 + lane;
      const bool hit = i < T && a.parent[r0 + i] == cur && a.tokens[r0 + i] == t;
      const unsigned m = __ballot_sync(0xffffffffu, hit);
      if (m) next = i0 + __ffs(m) - 1;
    }
    cur = next;
  }
  for (int i = len + lane; i < a.max_len; i += 32)
    a.path[(size_t)b * a.max_len + i] = a.out_tokens[(size_t)b * a.max_len + i] = -1;
  if (lane == 0) a.n[b] = len;
}

static cudaError_t launch_tree_verify(const VerArgs& a, cudaStream_t st) {
  if (a.R) k_tree_sample<<<a.R, TV_THREADS, 0, st>>>(a);
  if (a.B) k_tree_walk<<<a.B, 32, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace exb

using namespace exb;

extern "C" int exb_tree_verify(const int64_t* logits, int64_t ld, int R, int V, const int32_t* u20, int64_t tnum,
                               const int32_t* tokens, const int32_t* parent, const int32_t* row_start, int B,
                               int max_len, const int32_t* exp_t, int32_t* sampled, int32_t* n, int32_t* path,
                               int32_t* out_tokens, void* stream) {
  auto fail = [](const char* m) { set_last_error(std::string("exb_tree_verify: ") + m); return EXB_EINVAL; };
  if (R < 0 || B < 0 || V < 1 || max_len < 1) return fail("R, B >= 0 and V, max_len >= 1");
  if (ld < V) return fail("row stride below V");
  if (tnum < 1 || tnum > (1ll << 32)) return fail("temperature multiplier in [1, 2^32]");
  if (!exp_t || (R && (!logits || !u20 || !tokens || !parent || !sampled)) ||
      (B && (!row_start || !n || !path || !out_tokens)))
    return fail("null argument");
  VerArgs a;
  a.logits = logits; a.ld = ld; a.u20 = u20; a.tnum = tnum; a.tokens = tokens; a.parent = parent;
  a.row_start = row_start; a.exp_t = exp_t; a.sampled = sampled; a.n = n; a.path = path; a.out_tokens = out_tokens;
  a.R = R; a.V = V; a.B = B; a.max_len = max_len;
  const cudaError_t e = launch_tree_verify(a, (cudaStream_t)stream);
  if (e != cudaSuccess) {
    set_last_error(std::string("exb_tree_verify: ") + cudaGetErrorString(e));
    return EXB_ECUDA;
  }
  return EXB_OK;
}
