// Verification of drafted trees (exb_tree_verify): the target's own token of every row, from a
// given random number or as the argmax, then the walk along the drafted tokens that agree.
//
//   y = shr(logit * tnum, 16), p = (e << 20) // sum(e) with e the exp table at (max y - y),
//   token = first index whose running sum of p exceeds (u20 * sum(p)) >> 20     (exact_llm.py:243-259);
//           the last index where none does
#include <cooperative_groups.h>

#include "exb_internal.h"
#include "treedev.cuh"

namespace cg = cooperative_groups;

namespace exb {

struct VerArgs {
  const int64_t* logits = nullptr; int64_t ld = 0;
  const int32_t* u20 = nullptr;
  int64_t tnum = 0;
  const int32_t *tokens = nullptr, *parent = nullptr, *row_start = nullptr, *exp_t = nullptr;
  int32_t *sampled = nullptr, *n = nullptr, *path = nullptr, *out_tokens = nullptr;
  int R = 0, V = 0, B = 0, max_len = 0;
};

// A row by one CTA of NT threads that reads it again for every step: any length, any values.
// Thread t owns the t-th of NT contiguous slices of the row.
template <int NT>
__device__ __noinline__ void sample_row(const VerArgs& a, int r) {
  __shared__ uint64_t red[NT / 32];
  __shared__ int64_t scan[NT];
  __shared__ int tok;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t* row = a.logits + (int64_t)r * a.ld;
  const int u = a.u20[r];
  const int c0 = (int)((int64_t)a.V * tid / NT), c1 = (int)((int64_t)a.V * (tid + 1) / NT);
  auto y_at = [&](int i) {
    return u < 0 ? row[i] : shr64((int64_t)((uint64_t)row[i] * (uint64_t)a.tnum), 16);
  };
  int64_t m = INT64_MIN;
  int first = INT32_MAX;
  for (int i = c0; i < c1; ++i) {
    const int64_t y = y_at(i);
    if (y > m || first == INT32_MAX) { m = y; first = i; }
  }
  int64_t M = m;
  for (int o = 16; o > 0; o >>= 1) { const int64_t w = __shfl_xor_sync(0xffffffffu, M, o); M = w > M ? w : M; }
  if (lane == 0) red[warp] = (uint64_t)M;
  if (tid == 0) tok = a.V - 1;
  __syncthreads();
  for (int i = 0; i < NT / 32; ++i) M = (int64_t)red[i] > M ? (int64_t)red[i] : M;
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
    for (int i = 0; i < NT / 32; ++i) S += red[i];
    auto p_at = [&](int i) { return ((uint64_t)tree_exp(a.exp_t, (uint64_t)M - (uint64_t)y_at(i)) << 20) / S; };
    int64_t ps = 0;
    for (int i = c0; i < c1; ++i) ps += (int64_t)p_at(i);
    scan[tid] = ps;
    __syncthreads();
    for (int o = 1; o < NT; o <<= 1) {
      const int64_t add = tid >= o ? scan[tid - o] : 0;
      __syncthreads();
      scan[tid] += add;
      __syncthreads();
    }
    const int64_t before = scan[tid] - ps;
    const int64_t target = (int64_t)(((uint64_t)u * (uint64_t)scan[NT - 1]) >> 20);
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

__global__ void __launch_bounds__(1024) k_tree_sample_long(const VerArgs a) { sample_row<1024>(a, blockIdx.x); }

// A row by a cluster: CTA c holds a slice of up to 1024 IT logits in registers (two neighbouring ones a
// thread and step), so the row is read once while the cluster agrees on its maximum and its sum.  What
// stays is the scaled logit as 32 bits, then e, then p; the sum of all p is at most 2^20, so 32-bit sums
// do from there.  A row with a scaled logit of 2^30 or more goes to sample_row instead.
// Measured on one B200 (device time in a graph): 420 rows of 152064 logits 259 us, 2.0 TB/s (a copy moves
// 6.6: the loads, the look-ups in the exp table and three agreements of the cluster follow one another within a
// row, and two or three CTAs an SM cover one another's only in part); 26 rows 22 us, one greedy row 8 us with
// the walk.
constexpr int TV_THREADS = 512;

template <int IT>
__global__ void __launch_bounds__(TV_THREADS, IT > 10 ? 2 : 3) k_tree_sample(const VerArgs a, int slice, int ahead) {
  extern __shared__ __align__(128) unsigned char sm[];
  int32_t* T = reinterpret_cast<int32_t*>(sm);
  constexpr int NW = TV_THREADS / 32;
  __shared__ int red[NW];
  __shared__ uint64_t red64[NW];
  __shared__ uint32_t seg[IT * NW];
  __shared__ int lmax, lwide, lfirst, gmax, gwide;
  __shared__ uint64_t lsum, linv;
  __shared__ uint32_t lps, gps[2];
  __shared__ uint64_t tbar;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), c = (int)cluster.block_rank();
  const int r = (int)blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = c * slice, n = max(0, min(a.V - i0, slice));
  const int64_t* row = a.logits + (int64_t)r * a.ld + i0;
  const int u = a.u20[r];
  if (tid == 0 && u >= 0) {
    mbar_init(&tbar, 1);
    mbar_fence_init();
    mbar_expect_tx(&tbar, 40960);
    bulk_g2s(T, a.exp_t, 40960, &tbar);
  }
  if (tid < EXP_LEN - 10240) T[10240 + tid] = 0;              // from 40.0 on (exp_sm_flat)
  const bool pair = ((((uintptr_t)row) & 15) == 0);
  // a logit of 32 bits times tnum < 2^31, scaled; `big` gathers what leaves the range (|y| < 2^30)
  const int tn = u < 0 ? 1 << 16 : (int)a.tnum;
  int y[2 * IT];
  int m = INT32_MIN;
  uint32_t big = 0;
  auto scaled = [&](long long x) {
    const int lo = (int)x, hi = (int)(x >> 32);
    const int64_t w = mad_wide_s32(lo, tn, 1 << 15);
    const int wh = (int)(w >> 32);
    big |= (uint32_t)(hi ^ (lo >> 31)) | ((uint32_t)(wh + (1 << 14)) >> 15);
    return (int)__funnelshift_r((uint32_t)w, (uint32_t)wh, 16);
  };
  constexpr int NB = IT < 4 ? IT : IT % 5 ? 4 : 5;            // loads in flight a thread
  static_assert(IT % NB == 0, "whole batches");
#pragma unroll
  for (int it0 = 0; it0 < IT; it0 += NB) {
    longlong2 v[NB];
    const bool full = (it0 + NB) * 2 * TV_THREADS <= n;
    const int64_t* at = row + it0 * 2 * TV_THREADS + 2 * tid;
    if (full && pair) {
#pragma unroll
      for (int k = 0; k < NB; ++k) v[k] = __ldcs(reinterpret_cast<const longlong2*>(at + k * 2 * TV_THREADS));
    } else {
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const int i = (it0 + k) * 2 * TV_THREADS + 2 * tid;
        v[k].x = i < n ? row[i] : 0;
        v[k].y = i + 1 < n ? row[i + 1] : 0;
      }
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int i = (it0 + k) * 2 * TV_THREADS + 2 * tid;
      const int y0 = scaled(v[k].x), y1 = scaled(v[k].y);     // past the end: no term, never the maximum
      y[2 * (it0 + k)] = full || i < n ? y0 : INT32_MIN;
      y[2 * (it0 + k) + 1] = full || i + 1 < n ? y1 : INT32_MIN;
      m = max(m, max(y[2 * (it0 + k)], y[2 * (it0 + k) + 1]));
    }
  }
  // the same slice of the row that is read when this one is done: into L2 while the cluster confers
  if (r + ahead < a.R) {
    const char* p = reinterpret_cast<const char*>(row + (int64_t)ahead * a.ld);
    const char* p0 = reinterpret_cast<const char*>((uintptr_t)p & ~(uintptr_t)15);
    const int bytes = n * 8 & ~15;
    for (int o = tid * 2048; o < bytes; o += TV_THREADS * 2048) prefetch_l2_bulk(p0 + o, min(2048, bytes - o));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) red[warp] = m;
  const int any_big = __syncthreads_or(big != 0);
  if (warp == 0) {
    m = __reduce_max_sync(0xffffffffu, red[lane & (NW - 1)]);
    // where the table did not come within the wait's limit, the row goes to sample_row, which reads it in place
    const bool late = u >= 0 && !mbar_wait(&tbar, 0);
    if (lane == 0) { lmax = m; lwide = any_big || late; }
  }
  cluster.sync();
  // one warp reads the peers' words, all at once, and leaves the result to the CTA: a word of another
  // SM is dear (16 warps reading 8 peers took 0.9 us a time)
  const int peer = lane & (C - 1);
  if (warp == 0) {
    const int M0 = __reduce_max_sync(0xffffffffu, *cluster.map_shared_rank(&lmax, peer));
    const bool w0 = __any_sync(0xffffffffu, *cluster.map_shared_rank(&lwide, peer));
    if (lane == 0) { gmax = M0; gwide = w0; }
  }
  __syncthreads();
  const int M = gmax;
  const bool wide = gwide;
  if (wide) {
    if (c == 0) sample_row<TV_THREADS>(a, r);
    if (u >= 0) mbar_wait(&tbar, 0);                          // no copy is left in flight
    cluster.sync();
    return;
  }
  if (u < 0) {                                                // the lowest index of the maximum
    int first = INT32_MAX;
#pragma unroll
    for (int k = 2 * IT - 1; k >= 0; --k)
      if (y[k] == M) first = (k >> 1) * 2 * TV_THREADS + 2 * tid + (k & 1);
    first = (int)__reduce_min_sync(0xffffffffu, (unsigned)first);
    if (lane == 0) red[warp] = first;
    __syncthreads();
    if (warp == 0) {
      first = (int)__reduce_min_sync(0xffffffffu, (unsigned)red[lane & (NW - 1)]);
      if (lane == 0) lfirst = first == INT32_MAX ? first : first + i0;
    }
    cluster.sync();
    if (c == 0 && warp == 0) {
      const int best = __reduce_min_sync(0xffffffffu, *cluster.map_shared_rank(&lfirst, peer));
      if (lane == 0) a.sampled[r] = best;
    }
    cluster.sync();
    return;
  }
  mbar_wait(&tbar, 0);                                        // (complete: warp 0 has seen it; every thread reads the copy)
  uint32_t es = 0;                                            // at most 2^24 each, 40 a thread
#pragma unroll
  for (int k = 0; k < 2 * IT; ++k) {
    const uint32_t e = exp_sm_flat(T, (uint32_t)M - (uint32_t)y[k]);
    y[k] = (int)e;
    es += e;
  }
  uint64_t s = es;
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) red64[warp] = s;
  __syncthreads();
  if (warp == 0) {
    s = lane < NW ? red64[lane] : 0;
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) lsum = s;
  }
  cluster.sync();
  if (warp == 0) {                                            // the reciprocal once, not by every thread
    uint64_t S = lane < C ? *cluster.map_shared_rank(&lsum, lane) : 0;
    for (int o = 16; o > 0; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
    if (lane == 0) linv = prob_inverse(S);
  }
  __syncthreads();
  const uint64_t inv = linv;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    uint32_t p = 0;
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const uint32_t e = (uint32_t)y[2 * it + f];
      y[2 * it + f] = (int)prob_of(e, inv);
      p += (uint32_t)y[2 * it + f];
    }
    p = __reduce_add_sync(0xffffffffu, p);                    // 64 neighbouring logits
    if (lane == 0) seg[it * NW + warp] = p;
  }
  __syncthreads();
  if (warp == 0) {
    uint32_t t = 0;
    for (int k = lane; k < IT * NW; k += 32) t += seg[k];
    t = __reduce_add_sync(0xffffffffu, t);
    if (lane == 0) lps = t;
  }
  cluster.sync();
  if (warp == 0) {
    const uint32_t t = lane < C ? *cluster.map_shared_rank(&lps, lane) : 0;
    const uint32_t t0 = __reduce_add_sync(0xffffffffu, t), t1 = __reduce_add_sync(0xffffffffu, lane < c ? t : 0);
    if (lane == 0) { gps[0] = t0; gps[1] = t1; }
  }
  auto all_read = cluster.barrier_arrive();                  // this CTA reads no other's memory any more
  __syncthreads();
  const uint32_t total = gps[0], before = gps[1];
  const uint32_t target = (uint32_t)(((uint64_t)u * total) >> 20);
  if (target >= total) {                                      // every p rounds to 0, or u20 is 2^20 or more
    if (c == 0 && tid == 0) a.sampled[r] = a.V - 1;
  } else if (before <= target && target < before + lps) {     // one CTA: its segment, then its lane
    // every warp looks for the segment, a lane over NS neighbouring ones; the segment's own warp goes on
    constexpr int NS = (IT * NW + 31) / 32;
    uint32_t x[NS], mine = 0;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      x[i] = lane * NS + i < IT * NW ? seg[lane * NS + i] : 0;
      mine += x[i];
    }
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const uint32_t w = __shfl_up_sync(0xffffffffu, inc, o); inc += lane >= o ? w : 0; }
    const int own = __ffs(__ballot_sync(0xffffffffu, before + inc > target)) - 1;
    uint32_t at = before + inc - mine;
    int k = lane * NS;
#pragma unroll
    for (int i = 0; i + 1 < NS; ++i)
      if (k == lane * NS + i && at + x[i] <= target) { at += x[i]; ++k; }
    k = __shfl_sync(0xffffffffu, k, own);
    at = __shfl_sync(0xffffffffu, at, own);
    if (warp == k % NW) {
      uint32_t pa = 0, pb = 0;
#pragma unroll
      for (int it = 0; it < IT; ++it)
      {                                                       // masks: a select by index would put y in memory
        const uint32_t is = 0u - (uint32_t)(it == k / NW);
        pa |= (uint32_t)y[2 * it] & is;
        pb |= (uint32_t)y[2 * it + 1] & is;
      }
      inc = pa + pb;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const uint32_t w = __shfl_up_sync(0xffffffffu, inc, o); inc += lane >= o ? w : 0; }
      const unsigned hit = __ballot_sync(0xffffffffu, at + inc > target);
      if (lane == __ffs(hit) - 1) {
        const bool first = at + inc - pb > target;
        a.sampled[r] = i0 + (k / NW) * 2 * TV_THREADS + 2 * tid + (first ? 0 : 1);
      }
    }
  }
  cluster.barrier_wait(std::move(all_read));                 // this CTA's words stay until they are read
}

// One warp per sequence walks from node 0: 32 candidates at a time, the lowest one that fits.
__global__ void __launch_bounds__(32) k_tree_walk(const VerArgs a) {
  pdl_wait();
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

template <int IT>
static cudaError_t launch_sample_rows(const VerArgs& a, int C, cudaStream_t st) {
  static DevOnce attr_set;
  if (!attr_set.done()) {
    cudaError_t e = cudaFuncSetAttribute(k_tree_sample<IT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 41024);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_tree_sample<IT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    attr_set.set();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)C * (unsigned)a.R);
  cfg.blockDim = dim3(TV_THREADS);
  cfg.dynamicSmemBytes = 41024;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_tree_sample<IT>, a, (a.V + 2 * C - 1) / (2 * C) * 2, 2 * 148 / C);
}

static cudaError_t launch_tree_verify(const VerArgs& a, cudaStream_t st) {
  if (a.R) {
    cudaError_t e;
    // slices of a row over 8 CTAs, as few steps of 1024 logits as hold them
    const int per = (a.V + 8191) / 8192;
    if (a.tnum >= (1ll << 31)) {
      k_tree_sample_long<<<a.R, 1024, 0, st>>>(a);
      e = cudaGetLastError();
    } else if (per <= 2) e = launch_sample_rows<2>(a, 8, st);
    else if (per <= 8) e = launch_sample_rows<8>(a, 8, st);
    else if (per <= 20) e = launch_sample_rows<20>(a, 8, st);
    else if (per <= 40) e = launch_sample_rows<20>(a, 16, st);
    else {
      k_tree_sample_long<<<a.R, 1024, 0, st>>>(a);
      e = cudaGetLastError();
    }
    if (e != cudaSuccess) return e;
  }
  if (a.B) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.B);
    cfg.blockDim = dim3(32);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_tree_walk, a);
  }
  return cudaSuccess;
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
  if ((uintptr_t)exp_t & 15) return fail("exp_t must be 16-byte aligned");
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
