// Exact attention of a tree of drafted tokens over a paged K/V cache (exb_tree_attention).
//
//   s_t = shr((q . k_t) * INV, 32 - qs - ks_t)     over the visible positions t
//   e_t = exp table at (max s - s_t), Q24;  p_t = (e_t << 20) // sum(e);  out = shr(sum p_t v_t, 20)
//
// p needs the row's final maximum and sum (a floor division by the sum: no rescaling afterwards
// gives the same bits), so a row goes over its scores three times.  Here the scores stay in shared memory
// meanwhile; tree_tc.cu computes them anew each time, for many rows and long caches.
//
// Measured on one B200 (device time in a graph): 32 single tokens of 28 heads after up to 1000 tokens 28.8 us
// (11.4 us would be the 75 MB at the rate of a copy; every SM reads rows of 256 and 512 bytes by look-up, and
// what it has in flight covers the latency of L2 and HBM in part: 126 registers a thread and the shared memory
// each leave room for two CTAs); a tree of 26 nodes of 28 heads after 513 tokens 21.9 us and one token of an
// empty sequence 9.4 us (cluster barriers and the chain from the lengths over the table to the rows: no bytes to
// speak of).  Width 16 with 8 rows a tile spills one register (4 bytes stored, 8 loaded), no other does.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "exb_internal.h"
#include "tree_tc.h"

namespace cg = cooperative_groups;

namespace exb {

// ---------------------------------------------------------------- few rows: one cluster per row tile
// A cluster of CTAs takes one (sequence, KV head) and NR = 8 NT of its query rows (a group's heads of
// neighbouring nodes together, so each K/V byte is read once for all of them); its CTAs split the
// positions.  Scores are int8 tensor-core products over byte digits, x = 256 hi + lo (hi signed, lo
// not): q.k = 65536 hh + 256 (hl + lh) + ll, each digit sum over 128 dims below 2^31.  They stay in
// shared memory as 32-bit numbers (rows above 2^31: as distances from the CTA's own maximum) while
// the cluster exchanges maxima and sums, so K and V are read once.  p < 2^21 is three byte digits,
// V four: twelve digit products, the ones of equal weight 2^(8 s) summed in int32 (at most 3 * 2^16 per
// position and 8192 positions a CTA) and put together in 64 bits at the end.
constexpr int TC_THREADS_T = 256;
constexpr int TREE_SMEM_MAX = 220 * 1024;
constexpr int EXP_BULK = 40960;                    // bytes of the table that one bulk copy brings

template <int HD, int NT>
struct TreeGeo {
  static constexpr int NR = 8 * NT;
  static constexpr int DG = HD < 32 ? 1 : HD / 32;           // 32-dim groups of the output
  static constexpr int KP = 8 / DG;                          // warps that share a dim group: key parts
  static constexpr int KS = HD < 32 ? 1 : HD / 32;           // 32-dim steps of a score
  static constexpr int OUT = KP * NR * HD;                   // partial outputs (int64)
  // exp table, partial outputs, then per position: scores, the place of its V row (and of its K row where that
  // is another number of elements), its shift
  static size_t smem(int ldk, bool same) { return 41024 + (size_t)OUT * 8 + (size_t)ldk * (NR * 4 + (same ? 10 : 18)); }
};
// score row pitch for n positions: 4 mod 16 words, so a warp's stores and loads hit 32 banks
inline int tree_pitch(int64_t n) { return (int)((n + 15) / 16 * 16 + 4); }

// zeros in the rows that no sequence owns, the gaps between the ranges taken (see TreeOrder): `n` values of a row
static __device__ __noinline__ void zero_rows(const int32_t* row_start, const int32_t* ctx, int B, int R, int64_t* out, int pitch, int n) {
  int end = 0, top = INT32_MIN;
  for (int b = 0; b <= B; ++b) {
    const int lo = b < B ? row_start[b] : R, hi = b < B ? row_start[b + 1] : R;
    const bool taken = lo >= max(top, 0) && hi >= lo && hi <= R && (b == B || (hi > lo && ctx[b] >= 0));
    if (b < B) top = max(top, lo);
    if (!taken && b < B) continue;
    for (int64_t e = threadIdx.x; e < (int64_t)(lo - end) * n; e += TC_THREADS_T) {
      const int64_t r = e / n;
      out[(end + r) * pitch + (e - r * n)] = 0;
    }
    end = hi;
  }
}

template <int HD, int NT>
__global__ void __launch_bounds__(TC_THREADS_T, NT == 1 ? 2 : 1) k_tree_cluster(const TreeArgs a, int ldk, bool same) {
  using G = TreeGeo<HD, NT>;
  constexpr int NR = G::NR;
  extern __shared__ __align__(128) unsigned char sm[];
  int32_t* T = reinterpret_cast<int32_t*>(sm);                               // exp table
  int64_t* pout = reinterpret_cast<int64_t*>(sm + 41024);                    // KP x NR x HD
  int32_t* sc = reinterpret_cast<int32_t*>(sm + 41024 + (size_t)G::OUT * 8); // NR x ldk
  int64_t* vat = reinterpret_cast<int64_t*>(sc + (size_t)NR * ldk);          // V row of every position, in elements
  int64_t* kat = same ? vat : vat + ldk;                                     // and K row
  int16_t* ksh = reinterpret_cast<int16_t*>(kat + ldk);                      // its shift, -1: there is no such position
  __shared__ int64_t lmax[NR], lsum[NR];
  __shared__ int64_t wmax[8][NR];
  __shared__ uint64_t pinv[NR];
  __shared__ int32_t base[NR];
  __shared__ int qsh[NR];
  __shared__ const uint64_t* rmask[NR];
  __shared__ int find[2];
  __shared__ int odd_sh;
  __shared__ uint64_t tbar;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), c = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
  const int j = blockIdx.y, ct = (int)blockIdx.x / C;
  const exb_kv_view& kv = a.kv;

  // ---- this cluster's sequence and row tile: tiles of all sequences in order
  if (warp == 0) {
    int at = 0, fb = -1, ft = 0;
    bool odd = lane == 0 && (a.B == 0 || a.row_start[0] != 0 || a.row_start[a.B] != a.R);
    TreeOrder order;
    for (int b0 = 0; b0 < a.B && (fb < 0 || blockIdx.x == 0); b0 += 32) {
      const int b = b0 + lane;
      TreeSeq s;
      if (b < a.B) {
        s = tree_seq(a, b, blockIdx.x == 0 && j == 0);
        odd |= s.T != s.hi - s.lo;
      }
      tree_in_order(b < a.B, lane, s, order);
      const int nt = (s.T * a.rep + NR - 1) / NR;
      int inc = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int w = __shfl_up_sync(0xffffffffu, inc, o); inc += lane >= o ? w : 0; }
      const unsigned hit = __ballot_sync(0xffffffffu, ct < at + inc && ct >= at + inc - nt);
      if (hit && fb < 0) {
        const int l = __ffs(hit) - 1;
        fb = b0 + l;
        ft = ct - at - __shfl_sync(0xffffffffu, inc - nt, l);
      }
      at += __shfl_sync(0xffffffffu, inc, 31);
    }
    odd = __any_sync(0xffffffffu, odd);
    if (lane == 0) { find[0] = fb; find[1] = ft; odd_sh = odd; }
    if (lane == 0) {
      mbar_init(&tbar, 1);
      mbar_fence_init();
    }
  }
  __syncthreads();
  if (blockIdx.x == 0 && odd_sh) zero_rows(a.row_start, a.ctx, a.B, a.R, a.out + j * a.rep * HD, a.H * HD, a.rep * HD);
  const int b = find[0];
  if (b < 0) return;                                         // the whole cluster leaves together
  const TreeSeq sq = tree_seq(a, b, false);
  if (tid == 0) {                                            // the table arrives during the scores
    mbar_expect_tx(&tbar, EXP_BULK);
    bulk_g2s(T, a.exp_t, EXP_BULK, &tbar);
  }
  if (tid < EXP_LEN - EXP_BULK / 4) T[EXP_BULK / 4 + tid] = 0;       // from 40.0 on (exp_sm_flat)
  const int32_t* trow = a.table + (size_t)b * a.MP;
  const int g0 = find[1] * NR, ng = min(NR, sq.T * a.rep - g0);
  // row i of the tile: node (g0 + i) / rep, head (g0 + i) % rep of the group
  auto q_index = [&](int i) {
    const int node = (g0 + i) / a.rep;
    return (size_t)(sq.r0 + node) * a.H + (size_t)j * a.rep + (g0 + i - node * a.rep);
  };
  if (tid < NR) {
    const bool live = tid < ng;
    qsh[tid] = live ? a.qs[q_index(tid)] : 0;
    rmask[tid] = a.mask + (size_t)(live ? sq.r0 + (g0 + tid) / a.rep : 0) * a.W;
  }
  // positions of this CTA, a multiple of 16 apart
  const int chunk = ((sq.S + C - 1) / C + 15) & ~15;
  const int t0 = min(sq.S, c * chunk), n = min(sq.S, t0 + chunk) - t0;
  const int n32 = (n + 31) & ~31;

  // ---- where the rows lie; all of them are on their way to L2 before the first is used
  for (int t = tid; t < n32; t += TC_THREADS_T) {
    int off = 0;
    const int pg = t < n ? page_of(a, trow, t0 + t, off) : -1;
    int64_t vo = 0, ko = 0;                                  // (a position that is not there: some row, hidden)
    int sh = -1;
    if (pg >= 0) {
      const int16_t* kr = k_row(kv, j, pg, off);
      const int32_t* vr = v_row(kv, j, pg, off);
#pragma unroll
      for (int o = 0; o < HD * 2; o += 128) prefetch_l2_line(reinterpret_cast<const char*>(kr) + o);
#pragma unroll
      for (int o = 0; o < HD * 4; o += 128) prefetch_l2_line(reinterpret_cast<const char*>(vr) + o);
      sh = (uint8_t)k_shift(kv, j, pg, off);
      ko = kr - kv.k;
      vo = vr - kv.v;
    }
    vat[t] = vo;
    if (!same) kat[t] = ko;
    ksh[t] = (int16_t)sh;
  }
  // ---- query digits: operand B of the scores; contraction slots 4 tq + i and 16 + 4 tq + i of a step
  // hold dims 8 tq + i and 8 tq + 4 + i, so that a key row is read 16 bytes at a time
  uint32_t ql[NT][G::KS][2], qh[NT][G::KS][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int i = nt * 8 + g;
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) {
      int4 v = make_int4(0, 0, 0, 0);
      if (i < ng && ks * 32 + 8 * tq < HD)
        v = *reinterpret_cast<const int4*>(a.q + q_index(i) * HD + ks * 32 + 8 * tq);
      uint2 lo, hi;
      int16_digits(v, lo, hi);
      ql[nt][ks][0] = lo.x; ql[nt][ks][1] = lo.y;
      qh[nt][ks][0] = hi.x; qh[nt][ks][1] = hi.y;
    }
  }
  __syncthreads();
  int qmax = 0;
  bool qneg = false;
#pragma unroll
  for (int i = 0; i < NR; ++i) { qmax = max(qmax, qsh[i]); qneg |= qsh[i] < 0; }
  int qs_r[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int f = 0; f < 2; ++f) qs_r[nt][f] = qsh[nt * 8 + 2 * tq + f];

  // ---- phase 1: scores of 16 positions a warp and step (operand A: keys g and g + 8), 64-bit maxima.
  // 19 <= 32 - qs - ks <= 32 for every row and key: |score| < 2^31 and a 32-bit shift gives it.
  // Where some shift is outside, the CTA goes over its keys twice: maxima, then clamped distances.
  const int c2 = (int)(a.inv << 16), c1 = (int)(a.inv << 8), c0 = (int)a.inv;
  int64_t mx[NT][2];
  int mx32[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) mx32[nt][0] = mx32[nt][1] = INT32_MIN;
  // one step's keys, fetched a step ahead
  struct Keys {
    int4 k[2][G::KS];
    int sh[2];                                               // -1: no such key
  };
  auto fetch = [&](int u, Keys& x) {
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int t = u + g + 8 * f;
      const int16_t* kr = kv.k + kat[t] + 8 * tq;
      x.sh[f] = ksh[t];
#pragma unroll
      for (int ks = 0; ks < G::KS; ++ks)
        x.k[f][ks] = ks * 32 + 8 * tq < HD ? __ldg(reinterpret_cast<const int4*>(kr + ks * 32)) : make_int4(0, 0, 0, 0);
    }
  };
  // one sweep over the keys: `wide` scores in 64 bits, `store` into sc
  auto sweep = [&](auto wide_t, bool store, bool track) {
    constexpr bool wide = decltype(wide_t)::value;
    bool fits = true;
    Keys next;
    if (warp * 16 < n) fetch(warp * 16, next);
#pragma unroll 1
    for (int u = warp * 16; u < n; u += 128) {
      const Keys x = next;
      if (u + 128 < n) fetch(u + 128, next);
      const int sh[2] = {max(x.sh[0], 0), max(x.sh[1], 0)};
      if (!wide) fits &= sh[0] + qmax <= 13 && sh[1] + qmax <= 13;
      int ll[NT][4], md[NT][4], hh[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int f = 0; f < 4; ++f) ll[nt][f] = md[nt][f] = hh[nt][f] = 0;
#pragma unroll
      for (int ks = 0; ks < G::KS; ++ks) {
        uint2 l0, h0, l1, h1;
        int16_digits(x.k[0][ks], l0, h0);
        int16_digits(x.k[1][ks], l1, h1);
        const uint32_t al[4] = {l0.x, l1.x, l0.y, l1.y}, ah[4] = {h0.x, h1.x, h0.y, h1.y};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_digits<false, false>(ll[nt], al, ql[nt][ks][0], ql[nt][ks][1]);
          mma_digits<false, true>(md[nt], al, qh[nt][ks][0], qh[nt][ks][1]);
          mma_digits<true, false>(md[nt], ah, ql[nt][ks][0], ql[nt][ks][1]);
          mma_digits<true, true>(hh[nt], ah, qh[nt][ks][0], qh[nt][ks][1]);
        }
      }
      const bool all = __all_sync(0xffffffffu, x.sh[0] >= 0 && x.sh[1] >= 0) && t0 + u + 15 < sq.ctx;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const int kf = f >> 1, i = nt * 8 + 2 * tq + (f & 1), t = u + g + 8 * kf;
          bool see = true;
          if (!all) {
            see = x.sh[kf] >= 0;
            if (see && t0 + t >= sq.ctx) {
              const int node = t0 + t - sq.ctx;
              see = (rmask[i][node >> 6] >> (node & 63)) & 1;
            }
          }
          const int sft = 32 - qs_r[nt][f & 1] - sh[kf];
          if (!wide) {
            const int64_t w = mad_wide_s32(hh[nt][f], c2, mad_wide_s32(md[nt][f], c1, mad_wide_s32(ll[nt][f], c0,
                                                                        (int64_t)(1u << ((sft - 1) & 31)))));
            const int s = see ? shift_low(w, sft) : INT32_MIN;
            mx32[nt][f & 1] = max(mx32[nt][f & 1], s);
            sc[i * ldk + t] = s;
          } else {
            const int64_t acc = mad_wide_s32(hh[nt][f], 65536, mad_wide_s32(md[nt][f], 256, (int64_t)ll[nt][f]));
            const int64_t s = shr64((int64_t)((uint64_t)acc * (uint64_t)a.inv), sft);
            if (track && see && s > mx[nt][f & 1]) mx[nt][f & 1] = s;
            if (store) {                                     // s - the CTA's maximum, clamped
              const uint64_t d = see ? (uint64_t)lmax[i] - (uint64_t)s : ~0ull;
              sc[i * ldk + t] = d < (1ull << 30) ? -(int)d : INT32_MIN;
            }
          }
        }
    }
    return fits;
  };
  // row maxima of the CTA: lanes of a row (stride 4), then the warps
  auto cta_max = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        int64_t m = mx[nt][f];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) { const int64_t w = __shfl_xor_sync(0xffffffffu, m, o); m = w > m ? w : m; }
        if (g == 0) wmax[warp][nt * 8 + 2 * tq + f] = m;
      }
    __syncthreads();
    if (tid < NR) {
      int64_t m = wmax[0][tid];
#pragma unroll
      for (int w = 1; w < 8; ++w) m = wmax[w][tid] > m ? wmax[w][tid] : m;
      lmax[tid] = m;
    }
    __syncthreads();
  };
  const unsigned live = NR * C - (tid & ~31) >= 32 ? 0xffffffffu : (1u << max(NR * C - (tid & ~31), 0)) - 1u;   // lanes below NR C
  const bool fits = sweep(std::false_type{}, true, true);
  const bool wide = __syncthreads_or(!fits || qneg);
  if (wide) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mx[nt][0] = mx[nt][1] = INT64_MIN;
    sweep(std::true_type{}, false, true);
    cta_max();
    sweep(std::true_type{}, true, false);
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int f = 0; f < 2; ++f) mx[nt][f] = mx32[nt][f] == INT32_MIN ? INT64_MIN : mx32[nt][f];
    cta_max();
  }
  // hidden rows of the tail, so that the loops below take whole steps of 32
  for (int e = tid; e < NR * (n32 - n); e += TC_THREADS_T) {
    const int i = e / (n32 - n), t = n + e - i * (n32 - n);
    sc[i * ldk + t] = INT32_MIN;
  }
  cluster.sync();
  // thread (row, peer): every peer's word at once, then over the C lanes of the row (C a power of two)
  if (tid < NR * C) {
    const int i = tid / C;
    int64_t m = cluster.map_shared_rank(lmax, tid & (C - 1))[i];
    for (int o = 1; o < C; o <<= 1) { const int64_t w = __shfl_xor_sync(live, m, o); m = w > m ? w : m; }
    // distance of a stored score: base - sc as 32 bits without a sign
    if ((tid & (C - 1)) == 0) {
      if (wide) {
        const uint64_t d = (uint64_t)m - (uint64_t)lmax[i];
        base[i] = d < (1ull << 30) ? (int)d : (1 << 30);
      } else {
        // another CTA's scores may be far above; 32-bit ones are above -1.6e9, so a lower maximum has none
        // here, and 0 keeps the hidden ones far
        base[i] = m > INT32_MAX ? INT32_MAX : m < -(3ll << 29) ? 0 : (int)m;
      }
    }
  }
  if (!mbar_wait(&tbar, 0)) {                                // the table
    set_err(a.status, ERR_WAIT_TIMEOUT);
    mbar_wait(&tbar, 0);                                     // no copy is left in flight
  }
  __syncthreads();
  // ---- phase 2: e over the stored scores, row sums
#pragma unroll 1
  for (int i = warp; i < NR; i += 8) {
    int64_t s = 0;
    const int bs = base[i];
    for (int t = lane; t < n32; t += 32) {
      // a hidden position (INT32_MIN) is at 2^29 or more from any base: e = 0
      const uint32_t e = exp_sm_flat(T, (uint32_t)bs - (uint32_t)sc[i * ldk + t]);
      sc[i * ldk + t] = (int)e;
      s += e;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) lsum[i] = s;
  }
  cluster.sync();
  if (tid < NR * C) {
    uint64_t s = (uint64_t)cluster.map_shared_rank(lsum, tid & (C - 1))[tid / C];
    for (int o = 1; o < C; o <<= 1) s += __shfl_xor_sync(live, s, o);
    if ((tid & (C - 1)) == 0) pinv[tid / C] = prob_inverse(s);       // 0 for a row that sees nothing: p = 0
  }
  __syncthreads();
  // ---- phase 3: out += p . v.  Warp: 32 dims (its group) x every KP-th step of 32 positions.  Operand
  // A: V digits, tile pair rows (tile 0: g, g + 8; tile 1: g, g + 8) = dims 4 g .. 4 g + 3, contraction
  // slots 4 tq + i, 16 + 4 tq + i = positions tq + 4 i, tq + 16 + 4 i; operand B: p digits, row g.
  {
    const int dg = warp % G::DG, part = warp / G::DG;
    const bool dlive = HD >= 32 || g < 4;
    int acc[NT][2][6][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int w = 0; w < 6; ++w)
#pragma unroll
          for (int f = 0; f < 4; ++f) acc[nt][mt][w][f] = 0;
    uint64_t inv[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) inv[nt] = pinv[nt * 8 + g];
    const int32_t* vbase = kv.v + (dlive ? dg * 32 + 4 * g : 0);
    auto load_v = [&](int u, int4* v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = __ldg(reinterpret_cast<const int4*>(vbase + vat[u + tq + 4 * i]));           // past the CTA's keys p is 0
      }
    };
    // 16 rows: the next step's V rows are fetched a step ahead; 8 rows: two CTAs an SM hide them, and the
    // registers that it takes would spill (32 single tokens after 1000: 55 us with it, 47 without)
    int4 v[8];
    if (NT > 1 && part * 32 < n) load_v(part * 32, v);
#pragma unroll 1
    for (int u = part * 32; u < n; u += 32 * G::KP) {
      if (NT == 1) load_v(u, v);
      uint32_t va[2][4][4];                                  // tile, digit, fragment
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t* x = reinterpret_cast<const uint32_t*>(&v[4 * h]);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          uint32_t o[4];
          byte_planes(x[d], x[4 + d], x[8 + d], x[12 + d], o);
#pragma unroll
          for (int p = 0; p < 4; ++p) va[d >> 1][p][(d & 1) + 2 * h] = o[p];
        }
      }
      if (NT > 1 && u + 32 * G::KP < n) load_v(u + 32 * G::KP, v);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t pb[2][4];                                   // half, digit
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t e = (uint32_t)sc[(nt * 8 + g) * ldk + u + tq + 16 * h + 4 * i];
            p[i] = prob_of(e, inv[nt]);
          }
          byte_planes(p[0], p[1], p[2], p[3], pb[h]);
        }
#pragma unroll
        for (int pd = 0; pd < 3; ++pd)
#pragma unroll
          for (int vd = 0; vd < 4; ++vd)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
              if (vd == 3) mma_digits<true, false>(acc[nt][mt][pd + vd], va[mt][vd], pb[0][pd], pb[1][pd]);
              else mma_digits<false, false>(acc[nt][mt][pd + vd], va[mt][vd], pb[0][pd], pb[1][pd]);
            }
      }
    }
    // the weights put together; fragment f: dim 4 g + 2 mt + (f >> 1), row 2 tq + (f & 1)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          uint64_t s = 0;
#pragma unroll
          for (int w = 0; w < 6; ++w) s += (uint64_t)(int64_t)acc[nt][mt][w][f] << (8 * w);
          if (dlive) pout[(size_t)(part * NR + nt * 8 + 2 * tq + (f & 1)) * HD + dg * 32 + 4 * g + 2 * mt + (f >> 1)] = (int64_t)s;
        }
  }
  __syncthreads();
  if (G::KP > 1) {
    for (int e = tid; e < NR * HD; e += TC_THREADS_T) {
      int64_t s = pout[e];
#pragma unroll
      for (int k = 1; k < G::KP; ++k) s += pout[k * NR * HD + e];
      pout[e] = s;
    }
  }
  cluster.sync();
  // ---- the cluster's partial sums: CTA c finishes a slice of the rows
  const int tot = ng * HD, per = (tot + C - 1) / C;
  for (int e = c * per + tid; e < min(tot, (c + 1) * per); e += TC_THREADS_T) {
    int64_t s = 0;
    for (int c0 = 0; c0 < C; c0 += 8) {
      int64_t w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = c0 + k < C ? cluster.map_shared_rank(pout, c0 + k)[e] : 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += w[k];
    }
    const int i = e / HD;
    a.out[q_index(i) * HD + (e - i * HD)] = shr64(s, 20);
  }
  cluster.sync();                                            // peers' shared memory stays until it is read
}

template <int HD, int NT>
static cudaError_t launch_cluster(const TreeArgs& a, int C, int ldk, bool same, cudaStream_t st) {
  using G = TreeGeo<HD, NT>;
  static DevOnce attr_set;
  if (!attr_set.done()) {
    cudaError_t e = cudaFuncSetAttribute(k_tree_cluster<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, TREE_SMEM_MAX);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_tree_cluster<HD, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    attr_set.set();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)C * (unsigned)((int64_t)a.R * a.rep / G::NR + a.B), a.kv.KV);
  cfg.blockDim = dim3(TC_THREADS_T);
  cfg.dynamicSmemBytes = G::smem(ldk, same);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_tree_cluster<HD, NT>, a, ldk, same);
}

template <int NT>
static cudaError_t launch_cluster_hd(const TreeArgs& a, int C, int ldk, bool same, cudaStream_t st) {
  switch (a.kv.hd) {
    case 16: return launch_cluster<16, NT>(a, C, ldk, same, st);
    case 32: return launch_cluster<32, NT>(a, C, ldk, same, st);
    case 64: return launch_cluster<64, NT>(a, C, ldk, same, st);
    default: return launch_cluster<128, NT>(a, C, ldk, same, st);
  }
}

// The tensor-core kernels from about 7 million scores of 128 dims on, with rows enough in a group to fill
// their tiles.  The lengths are on the device, so the rule takes a.cap, what a table row has room for: the figures
// are of tables as wide as the cache is long.  In wider ones the choice, the cluster size and the shared memory are
// those of the longer cache (a tree of 26 nodes of 28 heads after 513 tokens in tables of 1024, 4096, 16384
// positions 22, 33, 62 us; 32 single tokens after 1000 in 1024, 4096, 16384, 32768, 131072: 29, 40, 111, 218, 97).
// Measured both ways (28 heads of 128, 4 groups; one tree of 16, 32, 64 nodes): after 2000
// tokens 28, 43, 83 us here and 61, 72, 97 there; after 8000 tokens 68, 129, 254 here and 91, 120, 179
// there; 8 trees of 16 nodes of 40 heads, 8 groups, after 1000, 2000, 4000 tokens 78, 147, 239 and 99, 145,
// 212; at half the width it takes twice the scores (64 nodes of 14 heads after 8000, 16000 tokens: 90, 176
// and 110, 164).  With fewer than 24 rows a group most of a tile is empty (8 trees of 4 nodes of 28 heads after
// 16000 tokens: 263 and 270).
static bool use_tc(const TreeArgs& a) {
  return (int64_t)a.R * a.rep >= 24ll * a.B && (int64_t)a.R * a.H * a.kv.hd >= ((7ll << 27) + a.cap - 1) / a.cap;
}

static cudaError_t launch_tree_attention(const TreeArgs& a, void* workspace, cudaStream_t st) {
  // rows per tile: 16 where the trees have that many in a group
  const int NT = (int64_t)a.R * a.rep > 8ll * a.B ? 2 : 1, NR = 8 * NT;
  // CTAs per cluster: as many as keep every cluster resident at once, each with 64 positions at least; more
  // where the scores need the room.  A GPU processing cluster's SMs bound what fits together: at one CTA an
  // SM (16 rows, or a long score array) 14 clusters of 8, and a second round doubles the time (8 nodes of
  // 28 heads after 2000 tokens: 16 clusters of 8 37 us, of 4 28 us)
  const int64_t clusters = std::max<int64_t>(a.B, ((int64_t)a.R * a.rep + NR - 1) / NR) * a.kv.KV;
  auto pitch = [&](int c) { return tree_pitch(((a.cap + c - 1) / c + 31) / 16 * 16); };
  const exb_kv_view& kv = a.kv;
  const bool same = kv.k_page == kv.v_page && kv.k_head == kv.v_head && kv.k_pos == kv.v_pos;
  auto smem_of = [&](int c) { return 41024 + (size_t)2048 * NR + (size_t)pitch(c) * (NR * 4 + (same ? 10 : 18)); };
  int C = 0;
  for (int c = 1; c <= 16; c *= 2) {
    if (smem_of(c) > (size_t)TREE_SMEM_MAX) continue;
    const int slots = (NT == 2 || smem_of(c) > 110 * 1024 ? 112 : 256) / (c == 16 ? 2 : 1);
    if (!C || ((int64_t)(c / 2) * 64 < a.cap && clusters * c <= slots)) C = c;
  }
  if (!C || use_tc(a)) return launch_tree_tc(a, workspace, st);
  const int ldk = pitch(C);
  return NT == 2 ? launch_cluster_hd<2>(a, C, ldk, same, st) : launch_cluster_hd<1>(a, C, ldk, same, st);
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

size_t exb_tree_attention_workspace_bytes(int R, int H, int B) {
  return R < 1 || H < 1 || B < 0 ? 0 : tt_workspace_bytes(R, H, B);
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
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)exp_t | (uintptr_t)workspace) & 15) TREE_FAIL(EXB_EINVAL, "exb_tree_attention: q, exp_t, out and workspace must be 16-byte aligned");
  if (!workspace || workspace_bytes < exb_tree_attention_workspace_bytes(R, H, B))
    TREE_FAIL(EXB_EINVAL, "exb_tree_attention: workspace too small");
  TreeArgs a;
  a.kv = *kv; a.q = q; a.qs = qs; a.table = table; a.ctx = ctx; a.row_start = row_start; a.mask = mask;
  a.exp_t = exp_t; a.out = out; a.status = status; a.R = R; a.H = H; a.rep = H / kv->KV; a.B = B; a.MP = max_pages;
  a.W = mask_words; a.cap = (int64_t)max_pages * kv->page; a.page_div = fast_div(kv->page);
  a.inv = (int64_t)std::nearbyint(65536.0 / std::sqrt((double)kv->hd));
  const cudaError_t e = B ? launch_tree_attention(a, workspace, (cudaStream_t)stream)
                          : cudaMemsetAsync(out, 0, (size_t)R * H * kv->hd * 8, (cudaStream_t)stream);
  if (e != cudaSuccess) TREE_FAIL(EXB_ECUDA, std::string("exb_tree_attention: ") + cudaGetErrorString(e));
  return EXB_OK;
}

}  // extern "C"
