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
//               the whole run of units (at most 3 * 255^2 * 8064 positions < 2^31)
//   digits      cache rows come through registers: K in 16-byte pieces, V in blocks of 4 positions x 4
//               dims that byte permutations turn into words of 4 positions per digit
//   warps       16 that turn scores into maxima, sums or probabilities (TMEM lane = position, four column
//               groups), 8 that load cache rows and make digits of them, 3 that issue the MMAs (one alone took 90
//               cycles an MMA next to the others, twice what the tensor core takes) and one that looks up the
//               pages; they meet on mbarriers only, so the look-ups, the loads, the digits, the MMAs and the
//               softmax of neighbouring units overlap
// Scores are computed anew in each kernel: keeping them would move 12 bytes a score, more than the MMAs
// and the three multiply-adds that make one cost.
//
// Measured on one B200 (device time in a graph): a tree of 61 nodes of 40 heads after 32768 tokens 817 us,
// 24 digit products of 128 dims a score, 0.60 POP/s; 8 trees of up to 63 nodes of 28 heads after up to 4097
// tokens 491 us.  Every kernel spills (width 128, bytes stored and loaded: 40 and 132, 52 and 148, 68 and 296):
// 72 registers are all that 896 threads can start with.  A unit of the third kernel takes about 9000 cycles: 17
// thousand warp instructions (the exact exp table with its interpolation, the division by the sum, byte digits) at
// 2.0 a cycle, and of the shared memory's cycles 4400 for their loads and stores (1900 are conflicts of the table's
// random look-ups) and 2800 for the MMAs' operands; the tensor cores are busy a sixth of the time.
#include <algorithm>
#include <type_traits>

#include "exb_internal.h"
#include "tcdev.cuh"
#include "treedev.cuh"
#include "tree_tc.h"

namespace exb {

constexpr int TT_CW = 16;                          // softmax warps
constexpr int TT_COMPUTE = 32 * TT_CW;
constexpr int TT_LW = 8;                           // loading warps
constexpr int TT_LOAD = 32 * TT_LW;
constexpr int TT_THREADS = TT_COMPUTE + TT_LOAD + 128;       // and four: MMAs (two or three), places
constexpr int TT_BK = 128;                         // positions per unit
constexpr int TT_CHUNK = 32;                       // a chunk is 32 to 63 units of positions (all, if fewer): its row
                                                   // tiles follow one another, so its cache rows are read from L2
                                                   // by all but the first; a run is a part of a chunk
constexpr uint32_t TT_WAIT_LIMIT = 1u << 20;       // polls of a wait
constexpr int TT_RING = 8;                         // units whose rows' places are kept

struct TtPlaces {                                  // where a unit's cache rows lie, in elements, and the shifts
  int64_t k[TT_BK], v[TT_BK];
  int s[TT_BK];                                    // -1: there is no such position (the places are some row's)
};

template <int PASS>
struct TtGeo {
  static constexpr int NT = PASS == 2 ? 48 : 80;   // rows of one score tile (MMA N)
  static constexpr int SUB = PASS == 2 ? 1 : 2;    // score tiles that share a unit's keys
  static constexpr int NR = NT * SUB;              // rows of a unit
  static constexpr int RPT = NT / 4;               // rows per thread and tile: four column groups of warps
  static constexpr int QB = NT * 128;              // one digit plane of a tile's query rows
  static constexpr int KB = TT_BK * 128;           // one digit plane of the keys
  static constexpr int OFF_K = 2 * SUB * QB;
  static constexpr int OFF_V = OFF_K + 4 * KB;     // two buffers of two planes
  static constexpr int OFF_P = OFF_V + (PASS == 2 ? 4 * 16384 : 0);
  static constexpr int OFF_T = OFF_P + (PASS == 2 ? 3 * QB : 0);
  static constexpr int OFF_RING = OFF_T + (PASS ? 41088 : 0);
  static constexpr int SMEM = OFF_RING + TT_RING * (int)sizeof(TtPlaces) + 1024;
  static constexpr int ACC = 3 * NT;               // first column of the p . v accumulators
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
// the loads into these registers are complete (they pass through, so no use of them moves before)
EXB_DEV void tmem_wait12(int (&a)[4], int (&b)[4], int (&c)[4]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(b[0]), "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(c[0]),
                 "+r"(c[1]), "+r"(c[2]), "+r"(c[3])::"memory");
}
// int32 sums, A and B signed or not, both K-major, M = 128
EXB_DEV constexpr uint32_t tt_idesc(bool as, bool bs, int n) {
  return (2u << 4) | ((as ? 1u : 0u) << 7) | ((bs ? 1u : 0u) << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// stores to shared memory by 32-bit address
EXB_DEV void sts64(uint32_t a, uint32_t x, uint32_t y) { asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(a), "r"(x), "r"(y) : "memory"); }
EXB_DEV void sts32(uint32_t a, uint32_t x) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(x) : "memory"); }
EXB_DEV void sts8(uint32_t a, uint32_t x) {
  asm volatile("{\n .reg .b16 t;\n cvt.u16.u32 t, %1;\n st.shared.u8 [%0], t;\n}\n" ::"r"(a), "r"(x) : "memory");
}
// one MMA with its descriptors put together inside: low words base + constant, the common high word.  Few
// registers live across a row of them (the MMA warp has 48; a spilled operand is a trip to L2)
constexpr uint32_t TT_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);    // as tc_desc
template <int DOFF, int AOFF, int BOFF, uint32_t IDESC>
EXB_DEV void tt_mma(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b32 x, y, z, w;\n .reg .b64 da, db;\n"
      " setp.ne.b32 p, %3, 0;\n add.u32 z, %0, %4;\n add.u32 x, %1, %5;\n add.u32 y, %2, %6;\n"
      " mov.b32 w, %8;\n mov.b64 da, {x, w};\n mov.b64 db, {y, w};\n mov.b32 x, %7;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [z], da, db, x, p;\n}\n"
      ::"r"(d), "r"(a), "r"(b), "r"((uint32_t)accumulate), "n"(DOFF), "n"(AOFF), "n"(BOFF), "n"(IDESC), "n"(TT_DESC_HI)
      : "memory");
}
EXB_DEV uint32_t tt_desc_lo(const void* tile) { return ((smem_u32(tile) >> 4) & 0x3FFF) | (1u << 16); }
// the K steps of one product
template <int KS, int DOFF, int AOFF, int BOFF, uint32_t IDESC>
EXB_DEV void tt_product(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  tt_mma<DOFF, AOFF, BOFF, IDESC>(d, a, b, accumulate);
  if constexpr (KS > 1) tt_mma<DOFF, AOFF + 2, BOFF + 2, IDESC>(d, a, b, true);
  if constexpr (KS > 2) {
    tt_mma<DOFF, AOFF + 4, BOFF + 4, IDESC>(d, a, b, true);
    tt_mma<DOFF, AOFF + 6, BOFF + 6, IDESC>(d, a, b, true);
  }
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
    TreeOrder order;
    if (lane == 0) w.pre[0] = w.pre[a.B + 1] = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      TreeSeq s;
      if (b0 + lane < a.B) s = tree_seq(a, b0 + lane, true);
      tree_in_order(b0 + lane < a.B, lane, s, order);
      const int64_t rows = (int64_t)s.T * a.rep, nk = (s.S + TT_BK - 1) / TT_BK;
      int64_t u0 = (rows + TtGeo<0>::NR - 1) / TtGeo<0>::NR * nk * a.kv.KV;
      int64_t u1 = (rows + TtGeo<2>::NR - 1) / TtGeo<2>::NR * nk * a.kv.KV;
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
// A run of units of one row tile, found from its first unit: every role walks the same runs.
struct TtRun {
  int b = 0, j = 0, rt = 0, kt0 = 0, nk = 0;
};
// units of positions in a chunk: near equal parts of 32 to 63
EXB_DEV int tt_chunk(int nkt) {
  const int n = max(1, nkt / TT_CHUNK);
  return (nkt + n - 1) / n;
}
EXB_DEV TtRun tt_run(const TreeArgs& a, const int64_t* pre, int NR, int64_t u, int64_t uend) {
  TtRun r;
  int lo = 0, hi = a.B - 1;                                  // last sequence that begins at or before u
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  r.b = lo;
  const TreeSeq sq = tree_seq(a, lo, false);
  const int nrt = (sq.T * a.rep + NR - 1) / NR, nkt = (sq.S + TT_BK - 1) / TT_BK;
  const int64_t x = u - pre[lo], per_head = (int64_t)nrt * nkt;
  // (a 64-bit division takes longer than the rest of this)
  r.j = (int)(x < (1ll << 31) && per_head < (1ll << 31) ? (int)x / (int)per_head : x / per_head);
  const int64_t y = x - r.j * per_head;
  const int L = tt_chunk(nkt);
  const int64_t chunk = (int64_t)L * nrt;
  const int ch = (int)(y < (1ll << 31) ? (int)min(chunk, (int64_t)INT32_MAX) > (int)y ? 0 : (int)y / (int)chunk : y / chunk);
  const int len = min(L, nkt - ch * L), z = (int)(y - ch * chunk), k0 = z % len;
  r.rt = z / len;
  r.kt0 = ch * L + k0;
  r.nk = (int)min((int64_t)(len - k0), uend - u);
  return r;
}

template <int HD, int PASS>
__global__ void __launch_bounds__(TT_THREADS, 1) k_tt(const TreeArgs a, const TtWork w) {
  using G = TtGeo<PASS>;
  constexpr int NT = G::NT, RPT = G::RPT, SUB = G::SUB;
  constexpr int KS = HD < 32 ? 1 : HD / 32;                  // 32-byte steps of a score
  constexpr int KCH = HD / 8;                                // 16-byte pieces of a key row
  constexpr int KC = TT_BK * KCH / TT_LOAD;                  // of a loading thread
  constexpr int VB = HD >= 64 ? 2 : 1;                       // V blocks (16 positions x 32 dims) a warp loads at once
  constexpr int VH = HD >= 128 ? 2 : 1;                      // and how often
  constexpr int RS = HD < 32 ? 8 : HD / 4;                   // dim 4 c + d is MMA row d RS + c
  extern __shared__ unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  int32_t* T = reinterpret_cast<int32_t*>(sm + G::OFF_T);
  TtPlaces* ring = reinterpret_cast<TtPlaces*>(sm + G::OFF_RING);
  __shared__ TtRow rowc[G::NR];
  __shared__ const uint64_t* rmask[G::NR];
  __shared__ int64_t rmax[PASS ? G::NR : 1];
  __shared__ int64_t rowq[G::NR];                            // row of q, qs and out
  __shared__ unsigned long long row_sh[PASS < 2 ? G::NR : 1];
  // Barriers by unit or tile number, two of a kind where the second to next depends on the wait for this one:
  //   bar_s   a score tile is complete        bar_f   every softmax warp has read it
  //   bar_k   a unit's keys are in place      bar_kf  its score MMAs are complete (the buffer is free)
  //   bar_v   V is in place                   bar_w   P is in place
  //   bar_p   the p . v products are complete
  //   bar_q   a run's query digits are in place, and what the last run left in shared memory is used up
  //           (two by turns as well: a warp that issues scores has no part in a run of one tile, but in the next)
  //   ring_full, ring_free   a unit's places are written, every warp is done with them
  //   bar_x   an issuing warp's MMAs are all complete
  __shared__ uint64_t bar_s[2], bar_f[2], bar_k[2], bar_kf[2], bar_v[2], bar_w[2], bar_p, bar_q[2], ring_full[TT_RING], ring_free[TT_RING], bar_x[3];
  __shared__ uint32_t tmem_sh;
  __shared__ int qmax_sh;
  __shared__ volatile uint32_t top_sh[2];                    // the last unit (+ 1) with a third digit in some p
  __shared__ volatile uint32_t late_sh;                      // a wait has given up: every role leaves at its next unit
  __shared__ uint32_t stop_sh;                               // the same, as the softmax warps agree on it at a run's start
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const exb_kv_view& kv = a.kv;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_s[i], 1);
      mbar_init(&bar_f[i], TT_CW);
      mbar_init(&bar_k[i], TT_LW);
      mbar_init(&bar_kf[i], PASS < 2 ? 2 : 1);               // two warps issue the scores of a unit's two tiles
      mbar_init(&bar_v[i], TT_LW);
      mbar_init(&bar_w[i], TT_CW);
      mbar_init(&bar_q[i], TT_CW);
    }
    for (int i = 0; i < TT_RING; ++i) {
      mbar_init(&ring_full[i], 1);
      mbar_init(&ring_free[i], TT_CW + TT_LW);
    }
    mbar_init(&bar_p, 2);                                    // two warps issue the products
    for (int i = 0; i < 3; ++i) mbar_init(&bar_x[i], 1);
    top_sh[0] = top_sh[1] = late_sh = 0;
    mbar_fence_init();
  }
  if (warp == TT_CW + TT_LW) {
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
  const uint32_t tmem = tmem_sh, sb = smem_u32(sm);
  const int64_t* pre = w.pre + (PASS == 2 ? a.B + 1 : 0);
  const int64_t total = pre[a.B];
  int64_t u = total * blockIdx.x / gridDim.x;
  const int64_t uend = total * (blockIdx.x + 1) / gridDim.x;
  bool gave_up = false;                                      // a wait of this thread
  uint32_t tiles = 0, units = 0, runs = 0;                   // of this CTA so far
  // the n-th completion (from 0) of a barrier.  Where a wait gives up, every warp ends the unit it is in (a few
  // waits, each with its limit) and the kernel leaves with a status.  The flag is looked at once a unit: 828 us
  // against 806 without (61 nodes after 32768 tokens); a branch at every wait took 1033
  auto wait = [&](uint64_t* bar, uint32_t n) {
    gave_up |= !mbar_wait(bar, n & 1, TT_WAIT_LIMIT);
  };
  auto late = [&]() {                                        // asked by a warp once a unit
    if (gave_up) late_sh = 1;
    return (bool)__any_sync(0xffffffffu, late_sh);
  };
  auto wait2 = [&](uint64_t* bar, uint32_t n) { wait(bar + (n & 1), n >> 1); };          // one of two, by turns
  auto arrive = [&](uint64_t* bar) {                         // this warp, after all its lanes
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  auto await_places = [&](uint32_t unit) { wait(&ring_full[unit % TT_RING], unit / TT_RING); };

  // 896 threads start with 72 registers each, 64512 in all; 512 x 80 + 256 x 64 + 128 x 48 = 63488
  if (warp >= TT_CW + TT_LW) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    const int role = warp - TT_CW - TT_LW;
    if (role == 3) {
      // ---- places: four positions a lane; the pages of the next unit are looked up meanwhile
      const int32_t* trow = nullptr;
      int pg[4], S = 0, j = 0, t0 = 0;
      TtRun run;
      int i = 0;                                             // unit of the run whose pages are in pg
      auto next_pages = [&]() {                              // false: there are no more units
        if (i >= run.nk) {
          if (u >= uend) return false;
          run = tt_run(a, pre, G::NR, u, uend);
          u += run.nk;
          i = 0;
          S = tree_seq(a, run.b, false).S;
          trow = a.table + (size_t)run.b * a.MP;
        }
        j = run.j;
        t0 = (run.kt0 + i) * TT_BK + lane;
        ++i;
#pragma unroll
        for (int f = 0; f < 4; ++f) pg[f] = t0 + 32 * f < S ? __ldg(trow + div_by(t0 + 32 * f, a.page_div)) : -1;
        return true;
      };
      bool more = next_pages();
      while (more && !late()) {
        const uint32_t slot = units % TT_RING;
        TtPlaces& out = ring[slot];
        int64_t k[4], v[4];
        int sh[4];
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const int t = t0 + 32 * f, off = t - div_by(t, a.page_div) * kv.page;
          k[f] = v[f] = 0;
          sh[f] = -1;
          if ((unsigned)pg[f] < (unsigned)kv.pages) {
            k[f] = pg[f] * kv.k_page + off * kv.k_pos + j * kv.k_head;
            v[f] = pg[f] * kv.v_page + off * kv.v_pos + j * kv.v_head;
            sh[f] = (uint8_t)__ldg(kv.ks + pg[f] * kv.s_page + off * kv.s_pos + j * kv.s_head);
          } else if (t < S) {
            set_err(a.status, ERR_BOUNDS);
          }
        }
        more = next_pages();
        if (units >= TT_RING) wait(&ring_free[slot], units / TT_RING - 1);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          out.k[lane + 32 * f] = k[f];
          out.v[lane + 32 * f] = v[f];
          out.s[lane + 32 * f] = sh[f];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ring_full[slot]);
        ++units;
      }
    } else if (lane == 0) {
      // ---- MMAs, one lane.  Scores: warp 16, with two score tiles warps 16 and 17, a TMEM buffer each;
      // p . v: warps 17 and 18, half of the weights each
      const uint32_t qlo = tt_desc_lo(sm), klo = tt_desc_lo(sm + G::OFF_K), vlo = tt_desc_lo(sm + G::OFF_V),
                     plo = tt_desc_lo(sm + G::OFF_P);
      constexpr int QP = G::QB >> 4, KP = G::KB >> 4, VP = 16384 >> 4;       // planes, in 16 bytes
      auto issue_scores = [&](int sub, int kbuf, int col) {
        const uint32_t k = klo + kbuf * 2 * KP, q = qlo + sub * 2 * QP, d = tmem + col;
        tt_product<KS, 0, 0, 0, tt_idesc(false, false, NT)>(d, k, q, false);
        tt_product<KS, NT, 0, QP, tt_idesc(false, true, NT)>(d, k, q, false);
        tt_product<KS, NT, KP, 0, tt_idesc(true, false, NT)>(d, k, q, true);
        tt_product<KS, 2 * NT, KP, QP, tt_idesc(true, true, NT)>(d, k, q, false);
      };
      // digit PD of p times digit VD of V, added to weight PD + VD
      auto product = [&](auto pd_t, auto vd_t, bool add) {
        constexpr int PD = decltype(pd_t)::value, VD = decltype(vd_t)::value;
        tt_product<4, G::ACC + (PD + VD) * NT, VD * VP, PD * QP, tt_idesc(VD == 3, false, NT)>(tmem, vlo, plo, add);
      };
      using C0 = std::integral_constant<int, 0>;
      using C1 = std::integral_constant<int, 1>;
      using C2 = std::integral_constant<int, 2>;
      using C3 = std::integral_constant<int, 3>;
      while (u < uend && !late_sh) {
        const TtRun run = tt_run(a, pre, G::NR, u, uend);
        u += run.nk;
        if constexpr (PASS < 2) {
          bool begun = false;
          const TreeSeq sq = tree_seq(a, run.b, false);
          const int nh = sq.T * a.rep - run.rt * G::NR > NT ? 2 : 1;
          for (int i = 0; i < run.nk && !late_sh; ++i, ++units) {
            for (int h = 0; h < nh; ++h, ++tiles) {
              const int s = tiles & 1;
              if (role != s) continue;
              if (!begun) wait2(bar_q, runs);
              begun = true;
              wait2(bar_k, units);
              if (tiles >= 2) wait2(bar_f, tiles - 2);
              tc_fence_after();
              issue_scores(h, units & 1, s * 3 * NT);
              tc_commit(&bar_s[s]);
              tc_commit(&bar_kf[units & 1]);
              if (nh == 1) tc_commit(&bar_kf[units & 1]);
            }
          }
        } else if (role == 0) {
          wait2(bar_q, runs);
          for (int i = 0; i < run.nk && !late_sh; ++i, ++units) {
            wait2(bar_k, units);
            if (i > 0) wait(&bar_f[0], units - 1);
            tc_fence_after();
            issue_scores(0, units & 1, 0);
            tc_commit(&bar_s[0]);
            tc_commit(&bar_kf[units & 1]);
          }
        } else if (role < 3) {
          for (int i = 0; i < run.nk && !late_sh; ++i, ++units) {
            wait2(bar_v, units);
            wait2(bar_w, units);
            tc_fence_after();
            const bool add = i > 0;                          // the first unit's first product of a weight starts it
            const bool top = !add || top_sh[units & 1] == units + 1;
            if (role == 1) {
              product(C0{}, C0{}, add);
              product(C0{}, C3{}, add);
              product(C1{}, C2{}, true);
              product(C1{}, C3{}, add);
              if (top) {
                product(C2{}, C1{}, true);
                product(C2{}, C2{}, true);
              }
            } else {
              product(C0{}, C1{}, add);
              product(C1{}, C0{}, true);
              product(C0{}, C2{}, add);
              product(C1{}, C1{}, true);
              if (top) {
                product(C2{}, C0{}, true);
                product(C2{}, C3{}, add);
              }
            }
            tc_commit(&bar_p);
          }
        }
        ++runs;
      }
      tc_commit(&bar_x[role]);                               // none is left in flight, however this warp got here
      mbar_wait(&bar_x[role], 0, TT_WAIT_LIMIT);
    }
    __syncwarp();
  } else if (warp >= TT_CW) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // ---- loading warps: a thread's pieces have fixed places in the planes
    const int lt = tid - TT_COMPUTE, lw = warp - TT_CW;
    const int kr = lt / KCH, kc = lt % KCH;                  // first key and piece, then KSTEP keys on
    constexpr int KSTEP = TT_LOAD / KCH;
    const uint32_t ka = sb + G::OFF_K + kr * 128 + (((kc >> 1) ^ (kr & 7)) << 4) + (kc & 1) * 8;
    // V block: 16 positions (group lw), 32 dims; lane: 4 dims (piece vc), positions 4 aq ..
    const int vc = lane & 7, aq = lane >> 3;
    const uint32_t va = sb + G::OFF_V + vc * 128 + ((lw ^ vc) << 4) + aq * 4;
    auto load_v = [&](const TtPlaces& p, int half, int4* x) {
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int4* at = reinterpret_cast<const int4*>(kv.v + p.v[lw * 16 + aq * 4 + f]) + vc + 16 * half;
#pragma unroll
        for (int n = 0; n < VB; ++n)
          if (HD >= 32 || vc < HD / 4) x[4 * n + f] = __ldg(at + 8 * n);
      }
    };
    auto store_v = [&](int half, const int4* x) {
#pragma unroll
      for (int n = 0; n < VB; ++n) {
        if (HD >= 32 || vc < HD / 4) {
          uint32_t o4[4][4];
          byte_planes(x[4 * n].x, x[4 * n + 1].x, x[4 * n + 2].x, x[4 * n + 3].x, o4[0]);
          byte_planes(x[4 * n].y, x[4 * n + 1].y, x[4 * n + 2].y, x[4 * n + 3].y, o4[1]);
          byte_planes(x[4 * n].z, x[4 * n + 1].z, x[4 * n + 2].z, x[4 * n + 3].z, o4[2]);
          byte_planes(x[4 * n].w, x[4 * n + 1].w, x[4 * n + 2].w, x[4 * n + 3].w, o4[3]);
          const uint32_t d0 = va + (16 * half + 8 * n) * 128;
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int p = 0; p < 4; ++p) sts32(d0 + p * 16384 + d * RS * 128, o4[d][p]);
        }
      }
    };
    auto keys = [&](uint32_t n) {                            // of unit n
      await_places(n);
      const TtPlaces& p = ring[n % TT_RING];
      int4 x[KC];
#pragma unroll
      for (int c = 0; c < KC; ++c) x[c] = __ldg(reinterpret_cast<const int4*>(kv.k + p.k[kr + c * KSTEP]) + kc);
      if (n >= 2) wait2(bar_kf, n - 2);                      // the buffer's last scores
      const uint32_t d = ka + (n & 1) * 2 * G::KB;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        uint2 lo, hi;
        int16_digits(x[c], lo, hi);
        sts64(d + c * KSTEP * 128, lo.x, lo.y);
        sts64(d + G::KB + c * KSTEP * 128, hi.x, hi.y);
      }
      fence_async_smem();
      arrive(&bar_k[n & 1]);
    };
    const uint32_t all = (uint32_t)(uend - u);
    if constexpr (PASS < 2) {
      for (; units < all && !late(); ++units) {
        keys(units);
        arrive(&ring_free[units % TT_RING]);
      }
    } else {
      if (all) keys(0);
      while (u < uend && !late()) {
        const TtRun run = tt_run(a, pre, G::NR, u, uend);
        u += run.nk;
        for (int i = 0; i < run.nk && !late(); ++i, ++units) {
          if (units + 1 < all) keys(units + 1);              // a unit ahead of V, which waits for the products
          const TtPlaces& p = ring[units % TT_RING];
          int4 x[VB * 4];
          load_v(p, 0, x);
          if (units) wait(&bar_p, units - 1);                // V's last products
          if (i == 0) wait2(bar_q, runs);                    // and the last run's sums, which went through V's planes
#pragma unroll
          for (int half = 0; half < VH; ++half) {
            if (half) load_v(p, half, x);
            store_v(half, x);
          }
          fence_async_smem();
          arrive(&bar_v[units & 1]);
          arrive(&ring_free[units % TT_RING]);
        }
        ++runs;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 80;");
    const int quarter = warp & 3, cg = warp >> 2;            // TMEM lanes 32 quarter .., rows RPT cg ..
    const int key = quarter * 32 + lane;
    const uint32_t tlane = tmem + ((uint32_t)(quarter * 32) << 16);
    const int c2 = (int)(a.inv << 16), c1 = (int)(a.inv << 8), c0 = (int)a.inv;
    while (u < uend) {
      const TtRun run = tt_run(a, pre, G::NR, u, uend);
      const TreeSeq sq = tree_seq(a, run.b, false);
      const int kt0 = run.kt0, nk = run.nk;
      u += nk;
      const int g0 = run.rt * G::NR, ng = min(G::NR, sq.T * a.rep - g0);
      const int nh = PASS < 2 && ng > NT ? 2 : 1;
      if (gave_up) late_sh = 1;
      named_sync(1, TT_COMPUTE);                             // the last run is done with shared memory
      if (tid == 0) {
        qmax_sh = 0;
        stop_sh = late_sh;
      }
      if (tid < G::NR && tid < ng) {                         // row i of the tile: node (g0 + i) / rep
        const int node = (g0 + tid) / a.rep;
        rowq[tid] = (int64_t)(sq.r0 + node) * a.H + (int64_t)run.j * a.rep + (g0 + tid - node * a.rep);
        rmask[tid] = a.mask + (size_t)(sq.r0 + node) * a.W;
      }
      named_sync(1, TT_COMPUTE);
      if (stop_sh) break;                                    // all of them or none
      for (int e = tid; e < nh * NT * KCH; e += TT_COMPUTE) {          // query digits
        const int r = e / KCH, c = e - r * KCH;
        int4 v = make_int4(0, 0, 0, 0);
        if (r < ng) v = *reinterpret_cast<const int4*>(a.q + rowq[r] * HD + c * 8);
        uint2 lo, hi;
        int16_digits(v, lo, hi);
        const int sub = r / NT, n = r - sub * NT;
        const int o = sub * 2 * G::QB + n * 128 + (((c >> 1) ^ (n & 7)) << 4) + (c & 1) * 8;
        *reinterpret_cast<uint2*>(sm + o) = lo;
        *reinterpret_cast<uint2*>(sm + G::QB + o) = hi;
      }
      if (tid < G::NR) {
        TtRow r = {0, INT32_MIN, 0, 0};
        if (tid < ng) {
          const int64_t qi = rowq[tid];
          r.qs = a.qs[qi];
          if (PASS) {
            const int64_t m = tt_value(w.rowmax[qi]);
            // (32-bit scores are above -1.6e9: a lower maximum has none, and 0 keeps hidden ones far)
            r.base = m > INT32_MAX ? INT32_MAX : m < -(3ll << 29) ? 0 : (int)m;
            rmax[tid] = m;
          }
          if (PASS == 2) {
            const uint64_t inv = prob_inverse(w.rowsum[qi]);
            r.ilo = (uint32_t)inv;
            r.ihi = (uint32_t)(inv >> 32);
          }
          atomicMax(&qmax_sh, r.qs < 0 ? 64 : r.qs);
        }
        rowc[tid] = r;
      }

      fence_async_smem();
      named_sync(1, TT_COMPUTE);                             // query digits, rows and maxima are in place
      arrive(&bar_q[runs & 1]);
      ++runs;
      const int qmax = qmax_sh;
      // ---- a score's sums put together, sh = qs + ks: n = 32 - sh, so the 64-bit sum shifted left by sh has the
      // score in its high words.  MODE 0: every position visible and sh in [0, 13], |score| < 2^31; MODE 3: the
      // same with the mask (a hidden score is INT32_MIN, 2^29 or more from any base); MODE 1: sh in [0, 31], with
      // the mask and 64-bit distances; MODE 2: any shift
      auto sum64 = [&](int ll, int md, int hh, int sh) {     // sh in [0, 31]: with the rounding half
        return mad_wide_s32(hh, c2, mad_wide_s32(md, c1, mad_wide_s32(ll, c0, (int64_t)(0x80000000u >> sh))));
      };
      auto high = [&](int64_t x, int sh) { return (int)__funnelshift_l((uint32_t)x, (uint32_t)((uint64_t)x >> 32), sh); };
      auto score64 = [&](auto mode, int ll, int md, int hh, int sh) -> int64_t {
        if (decltype(mode)::value == 1) {
          const int64_t x = sum64(ll, md, hh, sh);
          const int top = (int)(x >> 32);
          const int up = (int)__funnelshift_rc((uint32_t)top, (uint32_t)(top >> 31), 32 - sh);
          return (int64_t)(((uint64_t)(uint32_t)up << 32) | (uint32_t)high(x, sh));
        }
        const int64_t acc = mad_wide_s32(hh, 65536, mad_wide_s32(md, 256, (int64_t)ll));
        return shr64((int64_t)((uint64_t)acc * (uint64_t)a.inv), 32 - sh);
      };
      auto mode_of = [&](int ksh, int t, int qmax) {
        if (__all_sync(0xffffffffu, ksh + qmax <= 13)) return __all_sync(0xffffffffu, ksh >= 0 && t < sq.ctx) ? 0 : 3;
        return __all_sync(0xffffffffu, ksh + qmax <= 31) ? 1 : 2;
      };
      auto seen = [&](int i, int ksh, int t) {               // row i of the unit, this thread's key
        if (ksh < 0 || i >= ng) return false;
        if (t < sq.ctx) return true;
        const int node = t - sq.ctx;
        return (bool)((rmask[i][node >> 6] >> (node & 63)) & 1);
      };
      auto e_far = [&](int i, int64_t s) {                   // e at a 64-bit distance
        const uint64_t d = (uint64_t)rmax[i] - (uint64_t)s;
        return exp_sm_flat(T, (d >> 32) ? 0xffffffffu : (uint32_t)d);
      };
      using M1 = std::integral_constant<int, 1>;
      using M2 = std::integral_constant<int, 2>;

      if constexpr (PASS < 2) {
        int mx[SUB][RPT];
        uint32_t es[SUB][RPT];
#pragma unroll
        for (int h = 0; h < SUB; ++h)
#pragma unroll
          for (int r = 0; r < RPT; ++r) { mx[h][r] = INT32_MIN; es[h][r] = 0; }
#pragma unroll 1
        for (int i = 0; i < nk && !late(); ++i, ++units) {
          await_places(units);
          const int ksh = ring[units % TT_RING].s[key];      // shift of this thread's key; -1: no such position
          const int t = (kt0 + i) * TT_BK + key;
          const int mode = mode_of(ksh, t, qmax);
#pragma unroll
          for (int h = 0; h < SUB; ++h) {
            if (h < nh) {
              const int s = tiles & 1;
              const int live = max(0, min(RPT, ng - h * NT - cg * RPT));          // this thread's rows that exist
              wait2(bar_s, tiles);
              __syncwarp();
              tc_fence_after();
              const uint32_t col = tlane + s * 3 * NT + cg * RPT;
#pragma unroll
              for (int r0 = 0; r0 < RPT; r0 += 4) {
                if (r0 < live) {
                  int ll[4], md[4], hh[4];
                  tmem_ld4(col + r0, ll);
                  tmem_ld4(col + NT + r0, md);
                  tmem_ld4(col + 2 * NT + r0, hh);
                  tmem_wait12(ll, md, hh);
                  int way = mode;
                  if (way == 0) {
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                      const TtRow rc = rowc[h * NT + cg * RPT + r0 + f];
                      const int sh = rc.qs + ksh, sc = high(sum64(ll[f], md[f], hh[f], sh), sh);
                      if (PASS == 0) mx[h][r0 + f] = max(mx[h][r0 + f], sc);
                      else es[h][r0 + f] += exp_sm_flat(T, (uint32_t)rc.base - (uint32_t)sc);
                    }
                  }
                  if (way == 3) {
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                      const int i2 = h * NT + cg * RPT + r0 + f;
                      const TtRow rc = rowc[i2];
                      const int sh = rc.qs + max(ksh, 0);
                      const int sc = seen(i2, ksh, t) ? high(sum64(ll[f], md[f], hh[f], sh), sh) : INT32_MIN;
                      if (PASS == 0) mx[h][r0 + f] = max(mx[h][r0 + f], sc);
                      else es[h][r0 + f] += exp_sm_flat(T, (uint32_t)rc.base - (uint32_t)sc);
                    }
                  }
                  if (way == 1) {
                    bool far = false;
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                      const int i2 = h * NT + cg * RPT + r0 + f;
                      const bool see = seen(i2, ksh, t);
                      const int64_t sc = score64(M1{}, ll[f], md[f], hh[f], rowc[i2].qs + max(ksh, 0));
                      if (PASS == 0) {
                        const bool fits = sc == (int)sc && (int)sc != INT32_MIN;     // (INT32_MIN: nothing seen)
                        far |= see && !fits;                 // (its row is done anew below)
                        if (see && fits) mx[h][r0 + f] = max(mx[h][r0 + f], (int)sc);
                      } else if (see) {
                        es[h][r0 + f] += e_far(i2, sc);
                      }
                    }
                    if (PASS == 0 && __any_sync(0xffffffffu, far)) way = 2;
                  }
                  if (way == 2) {                            // (rare: one row at a time, in little code)
#pragma unroll 1
                    for (int f = 0; f < 4; ++f) {
                      const int i2 = h * NT + cg * RPT + r0 + f;
                      const bool see = seen(i2, ksh, t);
                      const int64_t sc = score64(M2{}, f < 2 ? (f ? ll[1] : ll[0]) : (f == 2 ? ll[2] : ll[3]),
                                                 f < 2 ? (f ? md[1] : md[0]) : (f == 2 ? md[2] : md[3]),
                                                 f < 2 ? (f ? hh[1] : hh[0]) : (f == 2 ? hh[2] : hh[3]),
                                                 rowc[i2].qs + max(ksh, 0));
                      if (PASS == 0) {
                        int64_t best = see ? sc : INT64_MIN;
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) { const int64_t v = __shfl_xor_sync(0xffffffffu, best, o); best = v > best ? v : best; }
                        if (lane == 0 && i2 < ng && best != INT64_MIN) atomicMax(w.rowmax + rowq[i2], tt_key(best));
                      } else {
                        const uint32_t e = see ? e_far(i2, sc) : 0u;
#pragma unroll
                        for (int k = 0; k < 4; ++k) es[h][r0 + k] += k == f ? e : 0u;
                      }
                    }
                  }
                }
              }
              tc_fence_before();
              arrive(&bar_f[s]);
              ++tiles;
            }
          }
          arrive(&ring_free[units % TT_RING]);
        }
        // the run's maxima and sums: over the warp's keys, lane r of a warp keeping row r's, over the four warps
        // of a column group in shared memory, then one atomic a row
        for (int i = tid; i < G::NR; i += TT_COMPUTE) row_sh[i] = 0;
        named_sync(1, TT_COMPUTE);
#pragma unroll
        for (int h = 0; h < SUB; ++h) {
          if (h < nh) {
            unsigned long long mine = 0;
#pragma unroll
            for (int r = 0; r < RPT; ++r) {
              unsigned long long v;
              if (PASS == 0) {
                const int m = __reduce_max_sync(0xffffffffu, mx[h][r]);
                v = m == INT32_MIN ? 0ull : tt_key(m);
              } else {                                       // 32 lanes x 63 units x 2^24 < 2^35: two halves
                const uint32_t lo = __reduce_add_sync(0xffffffffu, es[h][r] & 0xffffu), hi = __reduce_add_sync(0xffffffffu, es[h][r] >> 16);
                v = lo + ((unsigned long long)hi << 16);
              }
              mine = lane == r ? v : mine;
            }
            if (lane < RPT) {
              if (PASS == 0) atomicMax(&row_sh[h * NT + cg * RPT + lane], mine);
              else atomicAdd(&row_sh[h * NT + cg * RPT + lane], mine);
            }
          }
        }
        named_sync(1, TT_COMPUTE);
        if (tid < ng && row_sh[tid]) {
          if (PASS == 0) atomicMax(w.rowmax + rowq[tid], row_sh[tid]);
          else atomicAdd(w.rowsum + rowq[tid], row_sh[tid]);
        }
      } else {
        const int live = max(0, min(RPT, ng - cg * RPT));    // this thread's rows that exist
        // row r of column group cg is row 4 r + cg of the P planes: two places of the key in them
        const uint32_t p0 = sb + G::OFF_P + cg * 128 + (((key >> 4) ^ cg) << 4) + (key & 15);
        const uint32_t p1 = sb + G::OFF_P + cg * 128 + (((key >> 4) ^ (4 + cg)) << 4) + (key & 15);
#pragma unroll 1
        for (int i = 0; i < nk && !late(); ++i, ++units) {
          await_places(units);
          const int ksh = ring[units % TT_RING].s[key];      // shift of this thread's key; -1: no such position
          const int t = (kt0 + i) * TT_BK + key;
          const int mode = mode_of(ksh, t, qmax);
          uint32_t pr[RPT];                                  // p of this key for the thread's rows
          wait(&bar_s[0], units);
          __syncwarp();
          tc_fence_after();
#pragma unroll
          for (int r0 = 0; r0 < RPT; r0 += 4) {
            if (r0 < live) {
              int ll[4], md[4], hh[4];
              tmem_ld4(tlane + cg * RPT + r0, ll);
              tmem_ld4(tlane + NT + cg * RPT + r0, md);
              tmem_ld4(tlane + 2 * NT + cg * RPT + r0, hh);
              tmem_wait12(ll, md, hh);
              if (mode == 0) {
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                  const TtRow rc = rowc[cg * RPT + r0 + f];
                  const int sh = rc.qs + ksh, sc = high(sum64(ll[f], md[f], hh[f], sh), sh);
                  pr[r0 + f] = prob_of(exp_sm_flat(T, (uint32_t)rc.base - (uint32_t)sc), ((uint64_t)rc.ihi << 32) | rc.ilo);
                }
              } else if (mode == 3) {
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                  const int i2 = cg * RPT + r0 + f;
                  const TtRow rc = rowc[i2];
                  const int sh = rc.qs + max(ksh, 0);
                  const int sc = seen(i2, ksh, t) ? high(sum64(ll[f], md[f], hh[f], sh), sh) : INT32_MIN;
                  pr[r0 + f] = prob_of(exp_sm_flat(T, (uint32_t)rc.base - (uint32_t)sc), ((uint64_t)rc.ihi << 32) | rc.ilo);
                }
              } else {
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                  const int i2 = cg * RPT + r0 + f;
                  const TtRow rc = rowc[i2];
                  const int sh = rc.qs + max(ksh, 0);
                  const int64_t sc = mode == 1 ? score64(M1{}, ll[f], md[f], hh[f], sh) : score64(M2{}, ll[f], md[f], hh[f], sh);
                  pr[r0 + f] = seen(i2, ksh, t) ? prob_of(e_far(i2, sc), ((uint64_t)rc.ihi << 32) | rc.ilo) : 0u;
                }
              }
            }
          }
          tc_fence_before();
          arrive(&bar_f[0]);                                 // the next unit's scores may come
          if (units) wait(&bar_p, units - 1);                // P's planes are free
          uint32_t big = 0;
#pragma unroll
          for (int r = 0; r < RPT; ++r) {
            if (r < live) {
              const uint32_t d = ((r & 1) ? p1 : p0) + r * 512;
              sts8(d, pr[r]);
              sts8(d + G::QB, pr[r] >> 8);
              sts8(d + 2 * G::QB, pr[r] >> 16);
              big |= pr[r];
            }
          }
          if (__any_sync(0xffffffffu, big >> 16) && lane == 0) top_sh[units & 1] = units + 1;
          fence_async_smem();
          arrive(&bar_w[units & 1]);
          arrive(&ring_free[units % TT_RING]);
        }
        wait(&bar_p, units - 1);
        __syncwarp();
        tc_fence_after();
        // the run's sums: lane = dim, columns = rows; through shared memory (V's planes), so that a warp's
        // atomics are of neighbouring dims
        int64_t* stage = reinterpret_cast<int64_t*>(sm + G::OFF_V);          // [row][MMA row], 48 x 128
#pragma unroll
        for (int r0 = 0; r0 < RPT; r0 += 4) {
          int v[6][4];
#pragma unroll
          for (int s = 0; s < 6; ++s) tmem_ld4(tlane + G::ACC + s * NT + cg * RPT + r0, v[s]);
          tmem_wait12(v[0], v[1], v[2]);
          tmem_wait12(v[3], v[4], v[5]);
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            int64_t o = mad_wide_s32(v[3][f], 1 << 24, mad_wide_s32(v[2][f], 1 << 16, mad_wide_s32(v[1][f], 256, (int64_t)v[0][f])));
            o += (int64_t)(((uint64_t)(uint32_t)v[4][f] + ((uint64_t)(uint32_t)v[5][f] << 8)) << 32);
            stage[(cg * RPT + r0 + f) * 128 + key] = o;
          }
        }
        tc_fence_before();
        named_sync(1, TT_COMPUTE);
        for (int e = tid; e < NT * HD; e += TT_COMPUTE) {
          const int col = e / HD, dim = e - col * HD, i2 = (col & 3) * RPT + (col >> 2);
          const int64_t o = stage[col * 128 + (dim & 3) * RS + (dim >> 2)];
          if (i2 < ng && o) atomicAdd(reinterpret_cast<unsigned long long*>(a.out) + rowq[i2] * HD + dim, (unsigned long long)o);
        }
        tc_fence_before();
      }
    }
  }
  if (gave_up) late_sh = 1;
  __syncthreads();
  if (tid == 0 && late_sh) set_err(a.status, ERR_WAIT_TIMEOUT);
  if (warp == TT_CW + TT_LW)
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
