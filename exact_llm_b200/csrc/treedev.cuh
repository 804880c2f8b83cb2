// Device helpers shared by the tree-decoding kernels: the paged cache, a tree's rows and mask.
#pragma once
#include "common.cuh"
#include "exactb200.h"

namespace exb {

// n / d for 0 <= n < 2^30 by one multiplication: m = floor(2^(32+s) / d) + 1 with s = floor(log2 d), so
// n * (m d - 2^(32+s)) < 2^30 * 2^(s+1) stays below 2^(32+s) and the quotient is exact; m = 0: a power of two
struct FastDiv {
  uint32_t m = 0;
  int s = 0;
};
inline FastDiv fast_div(int d) {
  FastDiv f;
  while ((d >> f.s) > 1) ++f.s;
  f.m = (d & (d - 1)) ? (uint32_t)((1ull << (32 + f.s)) / (uint32_t)d) + 1 : 0;
  return f;
}
EXB_DEV int div_by(int n, FastDiv f) { return (int)((f.m ? __umulhi((uint32_t)n, f.m) : (uint32_t)n) >> f.s); }

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
  FastDiv page_div;
};

// One sequence's rows and positions, cut to what the arguments can hold.
struct TreeSeq {
  int r0 = 0, T = 0;                     // first row, nodes
  int ctx = 0;                           // positions that every row sees
  int S = 0;                             // ctx + nodes that have a position in the table
  int lo = 0, hi = 0;                    // row_start as it is
};

EXB_DEV TreeSeq tree_seq(const TreeArgs& a, int b, bool report) {
  TreeSeq s;
  const int lo = a.row_start[b], hi = a.row_start[b + 1], c = a.ctx[b];
  s.lo = lo;
  s.hi = hi;
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

// A warp over all sequences in order, 32 at a time: where row_start falls (tree_seq has reported it), ranges may
// overlap, and one that begins below an earlier entry is left out too.  So no row belongs to two sequences.
struct TreeOrder {
  bool fell = false;
  int top = 0;                           // the largest entry so far, once it fell
};
// (m: this lane's entry, or the lowest number; returns the largest entry up to it)
static __device__ __noinline__ int tree_top(int m) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    const int w = __shfl_up_sync(0xffffffffu, m, i);
    if (lane >= i) m = max(m, w);
  }
  return m;
}
EXB_DEV void tree_in_order(bool there, int lane, TreeSeq& s, TreeOrder& o) {
  if (!__any_sync(0xffffffffu, s.hi < s.lo) && !o.fell) return;
  int m = there ? s.lo : INT32_MIN;
  if (o.fell && lane == 0) m = max(m, o.top);                // (where it rose so far, nothing is above this entry)
  m = tree_top(m);
  if (there && s.lo < m) s.T = s.S = 0;
  o.fell = true;
  o.top = __shfl_sync(0xffffffffu, m, 31);
}

// page of position pos, or -1 (reported) where the table names none
EXB_DEV int page_of(const TreeArgs& a, const int32_t* __restrict__ row, int pos, int& off) {
  const int i = div_by(pos, a.page_div);
  off = pos - i * a.kv.page;
  const int pg = __ldg(row + i);
  if ((unsigned)pg < (unsigned)a.kv.pages) return pg;
  set_err(a.status, ERR_BOUNDS);
  return -1;
}
// the 128-byte line of an address into L2 (for rows of cache lines a third of the time of bulk prefetches)
EXB_DEV void prefetch_l2_line(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p) : "memory"); }
EXB_DEV const int16_t* k_row(const exb_kv_view& kv, int head, int pg, int off) {
  return kv.k + (int64_t)pg * kv.k_page + (int64_t)head * kv.k_head + (int64_t)off * kv.k_pos;
}
EXB_DEV const int32_t* v_row(const exb_kv_view& kv, int head, int pg, int off) {
  return kv.v + (int64_t)pg * kv.v_page + (int64_t)head * kv.v_head + (int64_t)off * kv.v_pos;
}
EXB_DEV int k_shift(const exb_kv_view& kv, int head, int pg, int off) {
  return kv.ks[(int64_t)pg * kv.s_page + (int64_t)head * kv.s_head + (int64_t)off * kv.s_pos];
}

// p = (e << 20) // sum for 0 <= e <= 2^24 by two multiplications, p = (e * inv) >> 66.  The row's largest term
// alone is 2^24 (entry 0 of the table), so a smaller sum is a row that sees nothing: inv = 0 and p = 0.
//   2^24 <= sum < 2^42 (up to 2^18 terms): inv = ceil(2^86 / sum); e * (inv * sum - 2^86) < 2^24 * 2^42 = 2^66
//     keeps the quotient exact
//   sum >= 2^42: p is at most 4, the number of j in 1..4 with e >= t_j = ceil(j * sum / 2^20).  inv is the largest
//     ceil(j * 2^66 / t_j): no smaller one takes t_j to j, and t_j - 1 stays below j, since 2^86 / sum lies between
//     all j * 2^66 / t_j and all j * 2^66 / (t_j - 1), and two such fractions that differ are 2^18 apart or more
static __device__ __noinline__ uint64_t prob_inverse_long(uint64_t sum) {
  uint64_t inv = 0;
#pragma unroll 1
  for (uint64_t j = 1; j <= 4; ++j) {
    const uint64_t t = (j * sum + (1u << 20) - 1) >> 20;
    if (t > (1ull << 24)) break;
    const uint64_t q = (j << 60) / t, r = (j << 60) - q * t;
    inv = max(inv, (q << 6) + ((r << 6) + t - 1) / t);
  }
  return inv;
}
EXB_DEV uint64_t prob_inverse(uint64_t sum) {
  if (sum < (1ull << 24)) return 0;
  if (sum >= (1ull << 42)) return prob_inverse_long(sum);
  // a double's estimate is within 2^10 of the quotient (below 2^62 + 1), so the remainder 2^86 - q sum is
  // below 2^53 and its low 64 bits are all of it; the second estimate is within one of the rest
  const double rc = __drcp_rn((double)sum);
  int64_t q = (int64_t)(rc * 77371252455336267181195264.0);             // 2^86
  int64_t r = (int64_t)(0ull - (uint64_t)q * sum);
  const int64_t dq = (int64_t)floor((double)r * rc);
  q += dq;
  r -= dq * (int64_t)sum;
  while (r < 0) { r += (int64_t)sum; --q; }
  while (r >= (int64_t)sum) { r -= (int64_t)sum; ++q; }
  return (uint64_t)q + (r ? 1 : 0);
}
EXB_DEV uint32_t prob_of(uint32_t e, uint64_t inv) {
  const uint64_t t = (uint64_t)e * (uint32_t)inv;
  const uint64_t h = (uint64_t)e * (uint32_t)(inv >> 32) + (t >> 32);
  return (uint32_t)(h >> 34);
}

// the table value at distance d, from a copy of the table in shared memory
EXB_DEV uint32_t exp_sm(const int32_t* T, uint32_t d) {
  if (d >= (40u << 16)) return 0;
  const int a = T[d >> 8], b = T[(d >> 8) + 1];
  return (uint32_t)(a - (((a - b) * (int)(d & 255) + 128) >> 8));
}

// the same without a branch: entries 10240 and 10241 of the copy hold 0
EXB_DEV uint32_t exp_sm_flat(const int32_t* T, uint32_t d) {
  d = min(d, 40u << 16);
  const int a = T[d >> 8], b = T[(d >> 8) + 1];
  return (uint32_t)(a - (((a - b) * (int)(d & 255) + 128) >> 8));
}

// 8 int16 -> their low bytes (unsigned digits) and high bytes (signed digits), in order
EXB_DEV void int16_digits(const int4 v, uint2& lo, uint2& hi) {
  lo = make_uint2(__byte_perm((uint32_t)v.x, (uint32_t)v.y, 0x6420), __byte_perm((uint32_t)v.z, (uint32_t)v.w, 0x6420));
  hi = make_uint2(__byte_perm((uint32_t)v.x, (uint32_t)v.y, 0x7531), __byte_perm((uint32_t)v.z, (uint32_t)v.w, 0x7531));
}
// byte planes of four words: o[i] = byte i of a, b, c, d in order
EXB_DEV void byte_planes(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t* o) {
  const uint32_t l0 = __byte_perm(a, b, 0x5140), l1 = __byte_perm(c, d, 0x5140);
  const uint32_t h0 = __byte_perm(a, b, 0x7362), h1 = __byte_perm(c, d, 0x7362);
  o[0] = __byte_perm(l0, l1, 0x5410);
  o[1] = __byte_perm(l0, l1, 0x7632);
  o[2] = __byte_perm(h0, h1, 0x5410);
  o[3] = __byte_perm(h0, h1, 0x7632);
}

// D += A (16 x 32) . B (32 x 8) in int8 digits, signed or not by operand, int32 sums
template <bool AS, bool BS>
EXB_DEV void mma_digits(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (!AS && !BS)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else if constexpr (!AS && BS)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else if constexpr (AS && !BS)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
EXB_DEV int64_t mad_wide_s32(int a, int b, int64_t t) {
  int64_t d;
  asm("mad.wide.s32 %0, %1, %2, %3;" : "=l"(d) : "r"(a), "r"(b), "l"(t));
  return d;
}
// low word of a 64-bit arithmetic shift right by n in [0, 32]
EXB_DEV int shift_low(int64_t x, int n) {
  return (int)__funnelshift_rc((uint32_t)x, (uint32_t)((uint64_t)x >> 32), n);
}

// exp table at d = max - score (exact_llm.py:109-115).  d is not negative unless the difference left
// 64 bits, and then it is past the table's end in truth: both compare as large.
EXB_DEV int64_t tree_exp(const int32_t* __restrict__ T, uint64_t d) {
  return d >= (40ull << 16) ? 0 : exp_lookup(T, (int64_t)d);
}

}  // namespace exb
