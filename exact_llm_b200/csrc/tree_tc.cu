// Tree attention on the 5th-generation tensor cores, for many rows or caches past a cluster's shared
// memory: three kernels over the same scores (row maxima; sums of e; p . v), each on an even share of the
// work per SM.
//
//   work unit   128 positions x one tile of NR query rows of one (sequence, KV head); a CTA takes a
//               contiguous range of units, whatever the lengths of the sequences are
//   scores      D[position][row] = K Q^T: kind::i8 MMAs on byte digits, x = 256 hi + lo; three int32 sums
//               ll, hl + lh, hh in TMEM, put together as (hh INV 2^16 + md INV 2^8 + ll INV + half) >> n
//   p . v       D[dim][row] = V^T P^T: four byte digits of V times three of p < 2^21, twelve products; the
//               ones of equal weight 2^(8 s) share one of six int32 accumulators that stay in TMEM for
//               the whole run of units (at most 3 * 255^2 * 4096 positions < 2^31)
//   digits      cache rows come through registers: K in 16-byte pieces, V in blocks of 4 positions x 4
//               dims that byte permutations turn into words of 4 positions per digit
// Scores are computed anew in each kernel: keeping them would move 12 bytes a score, more than the MMAs
// and the three multiply-adds that make one cost.
#include <algorithm>

#include "exb_internal.h"
#include "tcdev.cuh"
#include "treedev.cuh"
#include "tree_tc.h"

namespace exb {

constexpr int TT_THREADS = 512;
constexpr int TT_BK = 128;                         // positions per unit
constexpr int TT_CHUNK = 32;                       // units of one run: row tiles of a chunk follow one another,
                                                   // so its cache rows are read from L2 by all but the first
constexpr int TT_RING = 8;

template <int PASS>
struct TtGeo {
  static constexpr int NR = PASS == 2 ? 48 : 80;   // rows per tile (MMA N)
  static constexpr int RPT = NR / 4;               // rows per thread: four column groups of four warps
  static constexpr int QB = NR * 128;              // one digit plane of the query rows
  static constexpr int KB = TT_BK * 128;           // one digit plane of the keys
  static constexpr int OFF_K = 2 * QB;
  static constexpr int OFF_V = OFF_K + 4 * KB;     // two buffers of two planes
  static constexpr int OFF_P = OFF_V + (PASS == 2 ? 4 * 16384 : 0);
  static constexpr int OFF_T = OFF_P + (PASS == 2 ? 3 * QB : 0);
  static constexpr int OFF_RING = OFF_T + (PASS ? 41088 : 0);
  static constexpr int SMEM = OFF_RING + TT_RING * TT_BK * 24 + 1024;
  static constexpr int ACC = 3 * NR;               // first column of the p . v accumulators
};

struct TtPlace {                                   // a position's rows in the cache, in elements
  int64_t k, v, s;                                 // k = -1: there is none
};

struct TtRow {
  int qs, base;                                    // base: the row's maximum, at most INT32_MAX
  uint32_t ilo, ihi;                               // reciprocal of its sum (prob_inverse)
};

// 4 consecutive 32-bit TMEM columns of this thread's lane
EXB_DEV void tmem_ld4(uint32_t taddr, int32_t* v) {
  uint32_t r[4];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (int32_t)r[i];
}
// int32 sums, A and B signed or not, both K-major, M = 128
EXB_DEV constexpr uint32_t tt_idesc(bool as, bool bs, int n) {
  return (2u << 4) | ((as ? 1u : 0u) << 7) | ((bs ? 1u : 0u) << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
EXB_DEV void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 64-bit values in an order that an unsigned maximum keeps; 0 is below all of them
EXB_DEV unsigned long long tt_key(int64_t s) { return (unsigned long long)s ^ (1ull << 63); }
EXB_DEV int64_t tt_value(unsigned long long k) { return (int64_t)(k ^ (1ull << 63)); }

// ---------------------------------------------------------------- before: zeros, and the units of every sequence
__global__ void __launch_bounds__(256) k_tt_init(const TreeArgs a, const TtWork w) {
  const int64_t nout = (int64_t)a.R * a.H * a.kv.hd, nst = (int64_t)a.R * a.H * 2;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nout; i += (int64_t)gridDim.x * 256) a.out[i] = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nst; i += (int64_t)gridDim.x * 256) w.rowmax[i] = 0;
  if (blockIdx.x == 0 && threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int64_t at0 = 0, at1 = 0;
    if (lane == 0) w.pre[0] = w.pre[a.B + 1] = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      TreeSeq s;
      if (b0 + lane < a.B) s = tree_seq(a, b0 + lane, true);
      const int64_t rows = (int64_t)s.T * a.rep, nk = (s.S + TT_BK - 1) / TT_BK;
      int64_t u0 = (rows + 79) / 80 * nk * a.kv.KV, u1 = (rows + 47) / 48 * nk * a.kv.KV;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x0 = __shfl_up_sync(0xffffffffu, u0, o), x1 = __shfl_up_sync(0xffffffffu, u1, o);
        if (lane >= o) { u0 += x0; u1 += x1; }
      }
      if (b0 + lane < a.B) {
        w.pre[b0 + lane + 1] = at0 + u0;
        w.pre[a.B + 1 + b0 + lane + 1] = at1 + u1;
      }
      at0 += __shfl_sync(0xffffffffu, u0, 31);
      at1 += __shfl_sync(0xffffffffu, u1, 31);
    }
  }
}

__global__ void __launch_bounds__(256) k_tt_finish(int64_t* out, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) out[i] = shr64(out[i], 20);
}

// ---------------------------------------------------------------- PASS 0: maxima, 1: sums of e, 2: p . v
template <int HD, int PASS>
__global__ void __launch_bounds__(TT_THREADS, 1) k_tt(const TreeArgs a, const TtWork w) {
  using G = TtGeo<PASS>;
  constexpr int NR = G::NR, RPT = G::RPT;
  constexpr int KS = HD < 32 ? 1 : HD / 32;                  // 32-byte steps of a score
  constexpr int KCH = HD / 8;                                // 16-byte pieces of a key row
  constexpr int KC = TT_BK * KCH >= TT_THREADS ? TT_BK * KCH / TT_THREADS : 1;
  constexpr int VB = HD >= 128 ? 2 : 1;                      // V blocks (16 positions x 32 dims) a warp
  constexpr int RS = HD < 32 ? 8 : HD / 4;                   // dim 4 c + d is MMA row d RS + c
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  int32_t* T = reinterpret_cast<int32_t*>(sm + G::OFF_T);
  TtPlace* ring = reinterpret_cast<TtPlace*>(sm + G::OFF_RING);
  __shared__ TtRow rowc[NR];
  __shared__ const uint64_t* rmask[NR];
  __shared__ int64_t rmax[NR];
  __shared__ uint64_t sbar[2], pvbar;
  __shared__ uint32_t tmem_sh;
  __shared__ int qmax_sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int quarter = warp & 3, cg = warp >> 2;              // TMEM lanes 32 quarter .., rows RPT cg ..
  const int key = quarter * 32 + lane;
  const exb_kv_view& kv = a.kv;

  if (tid == 0) {
    mbar_init(&sbar[0], 1);
    mbar_init(&sbar[1], 1);
    mbar_init(&pvbar, 1);
    mbar_fence_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_sh)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (PASS) {
    for (int i = tid; i < 10240 / 4; i += TT_THREADS) reinterpret_cast<int4*>(T)[i] = reinterpret_cast<const int4*>(a.exp_t)[i];
    if (tid < 2) T[10240 + tid] = 0;                         // from 40.0 on (exp_sm_flat)
  }
  if (HD == 16)                                              // bytes 16..31 of the digit rows: no dims
    for (int i = tid; i < G::OFF_V / 16; i += TT_THREADS) reinterpret_cast<int4*>(sm)[i] = make_int4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh, tlane = tmem + ((uint32_t)(quarter * 32) << 16);
  const int64_t* pre = w.pre + (PASS == 2 ? a.B + 1 : 0);
  const int64_t total = pre[a.B];
  int64_t u = total * blockIdx.x / gridDim.x;
  const int64_t uend = total * (blockIdx.x + 1) / gridDim.x;
  const int c2 = (int)(a.inv << 16), c1 = (int)(a.inv << 8), c0 = (int)a.inv;
  uint32_t sph[2] = {0, 0}, pvph = 0;                        // phases of the barriers
  bool late = false;                                         // a wait gave up

  while (u < uend) {
    // ---- the run that starts at unit u
    int b = 0;
    {
      int lo = 0, hi = a.B - 1;                              // last sequence that begins at or before u
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] <= u) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
    }
    const TreeSeq sq = tree_seq(a, b, false);
    const int nrt = (sq.T * a.rep + NR - 1) / NR, nkt = (sq.S + TT_BK - 1) / TT_BK;
    const int64_t x = u - pre[b];
    const int64_t per_head = (int64_t)nrt * nkt;
    const int j = (int)(x / per_head);
    const int y = (int)(x - j * per_head);
    const int ch = min(y / (TT_CHUNK * nrt), (nkt - 1) / TT_CHUNK);
    const int len = min(TT_CHUNK, nkt - ch * TT_CHUNK);
    const int z = y - ch * TT_CHUNK * nrt, rt = z / len, k0 = z - rt * len;
    const int kt0 = ch * TT_CHUNK + k0;
    const int nk = (int)min((int64_t)(len - k0), uend - u);
    u += nk;
    const int g0 = rt * NR, ng = min(NR, sq.T * a.rep - g0);
    const int32_t* trow = a.table + (size_t)b * a.MP;
    auto q_index = [&](int i) {                              // row i of the tile: node (g0 + i) / rep
      const int node = (g0 + i) / a.rep;
      return (size_t)(sq.r0 + node) * a.H + (size_t)j * a.rep + (g0 + i - node * a.rep);
    };
    auto place = [&](int pg, int off) {                      // where an offset of a page lies
      TtPlace p = {-1, 0, 0};
      if (pg >= 0) {
        p.k = (int64_t)pg * kv.k_page + (int64_t)j * kv.k_head + (int64_t)off * kv.k_pos;
        p.v = (int64_t)pg * kv.v_page + (int64_t)j * kv.v_head + (int64_t)off * kv.v_pos;
        p.s = (int64_t)pg * kv.s_page + (int64_t)j * kv.s_head + (int64_t)off * kv.s_pos;
      }
      return p;
    };
    __syncthreads();                                         // the last run is done with shared memory
    if (tid == 0) qmax_sh = 0;
    {
      const int i = tid >> 7;                                // the first four units' places
      if (i < nk) {
        const int t = (kt0 + i) * TT_BK + (tid & 127);
        int off = 0;
        const int pg = t < sq.S ? page_of(a, trow, t, off) : -1;
        ring[i * TT_BK + (tid & 127)] = place(pg, off);
      }
    }
    for (int e = tid; e < NR * KCH; e += TT_THREADS) {       // query digits
      const int r = e / KCH, c = e - r * KCH;
      int4 v = make_int4(0, 0, 0, 0);
      if (r < ng) v = *reinterpret_cast<const int4*>(a.q + q_index(r) * HD + c * 8);
      uint2 lo, hi;
      int16_digits(v, lo, hi);
      const int o = r * 128 + (((c >> 1) ^ (r & 7)) << 4) + (c & 1) * 8;
      *reinterpret_cast<uint2*>(sm + o) = lo;
      *reinterpret_cast<uint2*>(sm + G::QB + o) = hi;
    }
    __syncthreads();
    if (tid < NR) {
      TtRow r = {0, INT32_MIN, 0, 0};
      int64_t m = INT64_MIN;
      if (tid < ng) {
        const size_t qi = q_index(tid);
        r.qs = a.qs[qi];
        rmask[tid] = a.mask + (size_t)(sq.r0 + (g0 + tid) / a.rep) * a.W;
        if (PASS) {
          m = tt_value(w.rowmax[qi]);
          r.base = m > INT32_MAX ? INT32_MAX : (int)m;
        }
        if (PASS == 2) {
          const uint64_t inv = prob_inverse(w.rowsum[qi]);
          r.ilo = (uint32_t)inv;
          r.ihi = (uint32_t)(inv >> 32);
        }
        atomicMax(&qmax_sh, r.qs < 0 ? 64 : r.qs);
      }
      rowc[tid] = r;
      rmax[tid] = m;
    }

    // ---- cache rows through registers
    int4 kraw[KC];
    int4 vraw[PASS == 2 ? VB * 4 : 1];
    auto load_k = [&](int i) {
      const TtPlace* p = ring + (i & (TT_RING - 1)) * TT_BK;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int e = tid + c * TT_THREADS, r = e / KCH;
        kraw[c] = make_int4(0, 0, 0, 0);
        if (TT_BK * KCH >= TT_THREADS || e < TT_BK * KCH) {
          const int64_t at = p[r].k;
          if (at >= 0) kraw[c] = __ldg(reinterpret_cast<const int4*>(kv.k + at) + (e - r * KCH));
        }
      }
    };
    auto store_k = [&](int buf) {
      unsigned char* d = sm + G::OFF_K + buf * 2 * G::KB;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int e = tid + c * TT_THREADS, r = e / KCH, ch8 = e - r * KCH;
        if (TT_BK * KCH >= TT_THREADS || e < TT_BK * KCH) {
          uint2 lo, hi;
          int16_digits(kraw[c], lo, hi);
          const int o = r * 128 + (((ch8 >> 1) ^ (r & 7)) << 4) + (ch8 & 1) * 8;
          *reinterpret_cast<uint2*>(d + o) = lo;
          *reinterpret_cast<uint2*>(d + G::KB + o) = hi;
        }
      }
    };
    // V block n of this warp: 16 positions kg, dims 32 dgp ..; lane: 4 dims (piece cl), positions 4 aq ..
    const int cl = lane & 7, aq = lane >> 3;
    auto load_v = [&](int i) {
      const TtPlace* p = ring + (i & (TT_RING - 1)) * TT_BK;
#pragma unroll
      for (int n = 0; n < VB; ++n) {
        const int blk = warp + 16 * n, kg = blk & 7, c = (blk >> 3) * 8 + cl;
#pragma unroll
        for (int f = 0; f < 4; ++f)
          vraw[4 * n + f] = c < HD / 4 ? __ldg(reinterpret_cast<const int4*>(kv.v + p[kg * 16 + aq * 4 + f].v) + c)
                                       : make_int4(0, 0, 0, 0);
      }
    };
    auto store_v = [&]() {
#pragma unroll
      for (int n = 0; n < VB; ++n) {
        const int blk = warp + 16 * n, kg = blk & 7, c = (blk >> 3) * 8 + cl;
        if (c < HD / 4) {
          const uint32_t* x4 = reinterpret_cast<const uint32_t*>(&vraw[4 * n]);
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            uint32_t o4[4];
            byte_planes(x4[d], x4[4 + d], x4[8 + d], x4[12 + d], o4);
            const int r = d * RS + c, o = r * 128 + ((kg ^ (r & 7)) << 4) + aq * 4;
#pragma unroll
            for (int p = 0; p < 4; ++p) *reinterpret_cast<uint32_t*>(sm + G::OFF_V + p * 16384 + o) = o4[p];
          }
        }
      }
    };
    // shift of this thread's key in unit i; -1: no such key
    auto key_shift = [&](int i) {
      const TtPlace p = ring[(i & (TT_RING - 1)) * TT_BK + key];
      return p.k < 0 ? -1 : (int)(uint8_t)__ldg(kv.ks + p.s);
    };
    // places of unit i + 4 are written while unit i runs; its page was looked up a unit earlier
    int pg_next = -1;
    auto look_up = [&](int i) {
      const int t = (kt0 + i) * TT_BK + tid;
      pg_next = -1;
      if (tid < TT_BK && i < nk && t < sq.S) pg_next = __ldg(trow + div_by(t, a.page_div));
    };
    auto put_place = [&](int i) {
      if (tid < TT_BK && i < nk) {
        const int t = (kt0 + i) * TT_BK + tid;
        TtPlace p = {-1, 0, 0};
        if (t < sq.S) {
          if ((unsigned)pg_next < (unsigned)kv.pages) p = place(pg_next, t - div_by(t, a.page_div) * kv.page);
          else set_err(a.status, ERR_BOUNDS);
        }
        ring[(i & (TT_RING - 1)) * TT_BK + tid] = p;
      }
    };
    auto issue_scores = [&](int kbuf, int col) {             // one thread
      const unsigned char* kd = sm + G::OFF_K + kbuf * 2 * G::KB;
#pragma unroll
      for (int k = 0; k < KS; ++k) tc_mma_i8(tmem + col, tc_desc(kd, k), tc_desc(sm, k), tt_idesc(false, false, NR), k > 0);
#pragma unroll
      for (int k = 0; k < KS; ++k)
        tc_mma_i8(tmem + col + NR, tc_desc(kd, k), tc_desc(sm + G::QB, k), tt_idesc(false, true, NR), k > 0);
#pragma unroll
      for (int k = 0; k < KS; ++k)
        tc_mma_i8(tmem + col + NR, tc_desc(kd + G::KB, k), tc_desc(sm, k), tt_idesc(true, false, NR), true);
#pragma unroll
      for (int k = 0; k < KS; ++k)
        tc_mma_i8(tmem + col + 2 * NR, tc_desc(kd + G::KB, k), tc_desc(sm + G::QB, k), tt_idesc(true, true, NR), k > 0);
    };
    auto wait = [&](uint64_t* bar, uint32_t& ph) {
      late |= !mbar_wait(bar, ph, TC_WAIT_LIMIT);
      ph ^= 1;
      __syncwarp();                                          // the TMEM loads that follow are the whole warp's
      tc_fence_after();
    };
    const int live = max(0, min(RPT, ng - cg * RPT));        // this thread's rows that exist
    // a score's three sums to its 32-bit value: every key of the warp visible, shifts within [0, 13]
    auto score32 = [&](int ll, int md, int hh, int sft) {
      return shift_low(mad_wide_s32(hh, c2, mad_wide_s32(md, c1, mad_wide_s32(ll, c0, (int64_t)(1u << ((sft - 1) & 31))))), sft);
    };
    auto score64 = [&](int ll, int md, int hh, int sft) {
      const int64_t acc = mad_wide_s32(hh, 65536, mad_wide_s32(md, 256, (int64_t)ll));
      return shr64((int64_t)((uint64_t)acc * (uint64_t)a.inv), sft);
    };
    auto seen = [&](int i, int t) {
      if (t < sq.ctx) return true;
      const int node = t - sq.ctx;
      return (bool)((rmask[i][node >> 6] >> (node & 63)) & 1);
    };

    if constexpr (PASS < 2) {
      int mx[RPT];
      uint32_t es[RPT];
#pragma unroll
      for (int r = 0; r < RPT; ++r) { mx[r] = INT32_MIN; es[r] = 0; }
      load_k(0);
      store_k(0);
      if (nk > 1) load_k(1);
      int ksh = key_shift(0), ksh_next = -1;
      look_up(4);
      fence_async_smem();
      tc_fence_before();
      __syncthreads();
      if (tid == 0) {
        tc_fence_after();
        issue_scores(0, 0);
        tc_commit(&sbar[0]);
      }
      const int qmax = qmax_sh;
#pragma unroll 1
      for (int i = 0; i < nk; ++i) {
        const int buf = i & 1;
        if (i + 1 < nk) {
          store_k(buf ^ 1);
          fence_async_smem();
          tc_fence_before();
          __syncthreads();                                   // unit i - 1 is read, unit i + 1 is in place
          if (tid == 0) {
            tc_fence_after();
            issue_scores(buf ^ 1, (buf ^ 1) * 3 * NR);
            tc_commit(&sbar[buf ^ 1]);
          }
          if (i + 2 < nk) load_k(i + 2);
          ksh_next = key_shift(i + 1);
          put_place(i + 4);
          look_up(i + 5);
        }
        const int t = (kt0 + i) * TT_BK + key;
        const bool fast = __all_sync(0xffffffffu, ksh >= 0 && ksh + qmax <= 13 && t < sq.ctx);
        wait(&sbar[buf], sph[buf]);
        const uint32_t col = tlane + buf * 3 * NR + cg * RPT;
#pragma unroll
        for (int r0 = 0; r0 < RPT; r0 += 4) {
          if (r0 < live) {
            int ll[4], md[4], hh[4];
            tmem_ld4(col + r0, ll);
            tmem_ld4(col + NR + r0, md);
            tmem_ld4(col + 2 * NR + r0, hh);
            tmem_wait_ld();
            if (fast) {
#pragma unroll
              for (int f = 0; f < 4; ++f) {
                const TtRow rc = rowc[cg * RPT + r0 + f];
                const int s = score32(ll[f], md[f], hh[f], 32 - rc.qs - ksh);
                if (PASS == 0) mx[r0 + f] = max(mx[r0 + f], s);
                else es[r0 + f] += exp_sm_flat(T, (uint32_t)rc.base - (uint32_t)s);
              }
            } else {
#pragma unroll 1
              for (int f = 0; f < 4; ++f) {
                const int i2 = cg * RPT + r0 + f;
                const bool see = ksh >= 0 && i2 < ng && seen(i2, t);
                // (a constant-index select keeps the sums in registers)
                const int l = f == 0 ? ll[0] : f == 1 ? ll[1] : f == 2 ? ll[2] : ll[3];
                const int m = f == 0 ? md[0] : f == 1 ? md[1] : f == 2 ? md[2] : md[3];
                const int h = f == 0 ? hh[0] : f == 1 ? hh[1] : f == 2 ? hh[2] : hh[3];
                const int64_t s = score64(l, m, h, 32 - rowc[i2].qs - max(ksh, 0));
                if (PASS == 0) {
                  int64_t best = see ? s : INT64_MIN;
                  for (int o = 16; o > 0; o >>= 1) { const int64_t v = __shfl_xor_sync(0xffffffffu, best, o); best = v > best ? v : best; }
                  if (lane == 0 && i2 < ng && best != INT64_MIN) atomicMax(w.rowmax + q_index(i2), tt_key(best));
                } else {
                  const uint64_t d = see ? (uint64_t)rmax[i2] - (uint64_t)s : ~0ull;
                  const uint32_t e = exp_sm_flat(T, d < (1ull << 31) ? (uint32_t)d : 1u << 31);
#pragma unroll
                  for (int k = 0; k < 4; ++k) es[r0 + k] += k == f ? e : 0u;
                }
              }
            }
          }
        }
        ksh = ksh_next;
        tc_fence_before();                                   // these TMEM reads before the next barrier
      }
      // the run's maxima and sums, over the warp's keys
#pragma unroll
      for (int r = 0; r < RPT; ++r) {
        if (PASS == 0) {
          const int m = __reduce_max_sync(0xffffffffu, mx[r]);
          if (lane == 0 && r < live && m != INT32_MIN) atomicMax(w.rowmax + q_index(cg * RPT + r), tt_key(m));
        } else {                                             // 32 lanes x 32 units x 2^24 < 2^34: two halves
          const uint32_t lo = __reduce_add_sync(0xffffffffu, es[r] & 0xffffu), hi = __reduce_add_sync(0xffffffffu, es[r] >> 16);
          const unsigned long long s = lo + ((unsigned long long)hi << 16);
          if (lane == 0 && r < live && s) atomicAdd(w.rowsum + q_index(cg * RPT + r), s);
        }
      }
    } else {
      load_k(0);
      store_k(0);
      if (nk > 1) { load_k(1); store_k(1); }
      load_v(0);
      if (nk > 2) load_k(2);
      int ksh = key_shift(0);
      look_up(4);
      fence_async_smem();
      tc_fence_before();
      __syncthreads();
      if (tid == 0) {
        tc_fence_after();
        issue_scores(0, 0);
        tc_commit(&sbar[0]);
      }
      const int qmax = qmax_sh;
#pragma unroll 1
      for (int i = 0; i < nk; ++i) {
        const int t = (kt0 + i) * TT_BK + key;
        const bool fast = __all_sync(0xffffffffu, ksh >= 0 && ksh + qmax <= 13 && t < sq.ctx);
        int ll[RPT], md[RPT], hh[RPT];
        wait(&sbar[0], sph[0]);
#pragma unroll
        for (int r0 = 0; r0 < RPT; r0 += 4) {
          tmem_ld4(tlane + cg * RPT + r0, ll + r0);
          tmem_ld4(tlane + NR + cg * RPT + r0, md + r0);
          tmem_ld4(tlane + 2 * NR + cg * RPT + r0, hh + r0);
        }
        tmem_wait_ld();
        tc_fence_before();
        __syncthreads();                                     // the sums are in registers
        if (tid == 0 && i + 1 < nk) {
          tc_fence_after();
          issue_scores((i + 1) & 1, 0);
          tc_commit(&sbar[0]);
        }
        // p of this key for the thread's rows, over ll
        uint32_t big = 0;
        if (fast) {
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            const TtRow rc = rowc[cg * RPT + r];
            const int s = score32(ll[r], md[r], hh[r], 32 - rc.qs - ksh);
            const uint32_t e = exp_sm_flat(T, (uint32_t)rc.base - (uint32_t)s);
            const uint32_t p = prob_of(e, ((uint64_t)rc.ihi << 32) | rc.ilo);
            ll[r] = (int)p;
            big |= p;
          }
        } else {
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            const int i2 = cg * RPT + r;
            uint32_t p = 0;
            if (ksh >= 0 && i2 < ng && seen(i2, t)) {
              const TtRow rc = rowc[i2];
              const uint64_t d = (uint64_t)rmax[i2] - (uint64_t)score64(ll[r], md[r], hh[r], 32 - rc.qs - ksh);
              const uint32_t e = exp_sm_flat(T, d < (1ull << 31) ? (uint32_t)d : 1u << 31);
              p = prob_of(e, ((uint64_t)rc.ihi << 32) | rc.ilo);
            }
            ll[r] = (int)p;
            big |= p;
          }
        }
        if (i > 0) wait(&pvbar, pvph);                       // V, P and the other key buffer are free
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
          const int i2 = cg * RPT + r;
          unsigned char* d = sm + G::OFF_P + i2 * 128 + (((key >> 4) ^ (i2 & 7)) << 4) + (key & 15);
          d[0] = (unsigned char)ll[r];
          d[G::QB] = (unsigned char)((uint32_t)ll[r] >> 8);
          d[2 * G::QB] = (unsigned char)((uint32_t)ll[r] >> 16);
        }
        store_v();
        if (i + 2 < nk) store_k(i & 1);
        fence_async_smem();
        tc_fence_before();
        const int top = __syncthreads_or(big >> 16);         // the third digit of p: only where there is one
        if (tid == 0) {
          tc_fence_after();
#pragma unroll 1
          for (int pd = 0; pd < (top || i == 0 ? 3 : 2); ++pd)
#pragma unroll
            for (int vd = 0; vd < 4; ++vd)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc_mma_i8(tmem + G::ACC + (pd + vd) * NR, tc_desc(sm + G::OFF_V + vd * 16384, k),
                          tc_desc(sm + G::OFF_P + pd * G::QB, k), tt_idesc(vd == 3, false, NR),
                          i > 0 || k > 0 || !(pd == 0 || vd == 3));       // a weight's first product starts it
          tc_commit(&pvbar);
        }
        if (i + 1 < nk) {
          load_v(i + 1);
          if (i + 3 < nk) load_k(i + 3);
          ksh = key_shift(i + 1);
          put_place(i + 4);
          look_up(i + 5);
        }
      }
      wait(&pvbar, pvph);
      // the run's sums: lane = dim, columns = rows
      const int m = key, c = m % RS, dim = 4 * c + m / RS;
      const bool has = m < 4 * RS && c < HD / 4;
#pragma unroll
      for (int r0 = 0; r0 < RPT; r0 += 4) {
        if (r0 < live) {
          int v[6][4];
#pragma unroll
          for (int s = 0; s < 6; ++s) tmem_ld4(tlane + G::ACC + s * NR + cg * RPT + r0, v[s]);
          tmem_wait_ld();
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            uint64_t o = 0;
#pragma unroll
            for (int s = 0; s < 6; ++s) o += (uint64_t)(int64_t)v[s][f] << (8 * s);
            if (has && r0 + f < live && o)
              atomicAdd(reinterpret_cast<unsigned long long*>(a.out) + q_index(cg * RPT + r0 + f) * HD + dim, o);
          }
        }
      }
      tc_fence_before();
    }
  }
  if (late) set_err(a.status, ERR_WAIT_TIMEOUT);
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

size_t tt_workspace_bytes(int R, int H, int B) {
  return ((size_t)R * H * 16 + (size_t)(B + 1) * 16 + 255) / 256 * 256;
}

template <int HD, int PASS>
static cudaError_t launch_tt(const TreeArgs& a, const TtWork& w, cudaStream_t st) {
  static DevOnce attr_set;
  if (!attr_set.done()) {
    cudaError_t e = cudaFuncSetAttribute(k_tt<HD, PASS>, cudaFuncAttributeMaxDynamicSharedMemorySize, TtGeo<PASS>::SMEM);
    if (e != cudaSuccess) return e;
    attr_set.set();
  }
  k_tt<HD, PASS><<<148, TT_THREADS, TtGeo<PASS>::SMEM, st>>>(a, w);
  return cudaGetLastError();
}

template <int HD>
static cudaError_t launch_tt_all(const TreeArgs& a, const TtWork& w, cudaStream_t st) {
  cudaError_t e = launch_tt<HD, 0>(a, w, st);
  if (e == cudaSuccess) e = launch_tt<HD, 1>(a, w, st);
  if (e == cudaSuccess) e = launch_tt<HD, 2>(a, w, st);
  return e;
}

cudaError_t launch_tree_tc(const TreeArgs& a, void* workspace, cudaStream_t st) {
  TtWork w;
  w.rowmax = reinterpret_cast<unsigned long long*>(workspace);
  w.rowsum = w.rowmax + (size_t)a.R * a.H;
  w.pre = reinterpret_cast<int64_t*>(w.rowsum + (size_t)a.R * a.H);
  const int64_t n = (int64_t)a.R * a.H * a.kv.hd;
  k_tt_init<<<(unsigned)std::min<int64_t>((n + 1023) / 1024, 592), 256, 0, st>>>(a, w);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  switch (a.kv.hd) {
    case 16: e = launch_tt_all<16>(a, w, st); break;
    case 32: e = launch_tt_all<32>(a, w, st); break;
    case 64: e = launch_tt_all<64>(a, w, st); break;
    default: e = launch_tt_all<128>(a, w, st); break;
  }
  if (e != cudaSuccess) return e;
  k_tt_finish<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a.out, n);
  return cudaGetLastError();
}

}  // namespace exb
