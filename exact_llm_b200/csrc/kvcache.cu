// Cache rows moved on the device: the accepted path of a drafted tree (exb_kv_compact), pages
// copied to other pages (exb_kv_copy_pages).  Both move bytes and nothing else.
#include "exb_internal.h"
#include "treedev.cuh"

namespace exb {

const char* kv_view_error(const exb_kv_view* kv);

// ---------------------------------------------------------------- compaction
// One CTA per (sequence, layer x KV head).  A thread owns one 16-byte column of the K or V rows (or
// the shifts) and moves the path's rows in order: a strictly increasing path has path[j] >= j, so a
// row is read before any later step writes it.  A path's rows follow one another (a load and a store each), so
// its length is what a call takes: 8 paths of up to 9 rows in 28 layers of 4 heads of 128 7.6 us, one path of 4 in
// 24 layers 4.6 us (device time in a graph), a launch and the chain.
constexpr int KC_THREADS = 64;                     // 16 K columns + 32 V columns + the shifts

struct CompactArgs {
  exb_kv_view kv;
  const int32_t *table = nullptr, *ctx = nullptr, *path = nullptr, *n = nullptr;
  int32_t *new_ctx = nullptr, *status = nullptr;
  int MP = 0, ld_path = 0;
  int64_t cap = 0;
};

__global__ void __launch_bounds__(KC_THREADS) k_kv_compact(const CompactArgs a) {
  const exb_kv_view& kv = a.kv;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int layer = blockIdx.y / kv.KV, head = blockIdx.y - layer * kv.KV;
  const int c = a.ctx[b], n = a.n[b];
  const int32_t* path = a.path + (size_t)b * a.ld_path;
  const int32_t* row = a.table + (size_t)b * a.MP;
  // the whole path is checked before anything moves
  bool bad = c < 0 || n < 0 || n > a.ld_path;
  if (!bad)
    for (int j = tid; j < n; j += KC_THREADS) {
      const int p = path[j], before = j ? path[j - 1] : -1;
      if (p <= before || (int64_t)c + p >= a.cap) { bad = true; break; }
      const int64_t s = c + p, d = c + j;
      bad |= (unsigned)row[s / kv.page] >= (unsigned)kv.pages || (unsigned)row[d / kv.page] >= (unsigned)kv.pages;
    }
  bad = __syncthreads_or(bad);
  if (blockIdx.y == 0 && tid == 0) {
    a.new_ctx[b] = bad ? c : c + n;
    if (bad) set_err(a.status, ERR_BOUNDS);
  }
  if (bad) return;
  const int kcol = kv.hd / 8, vcol = kv.hd / 4;
  if (tid > kcol + vcol) return;
  for (int j = 0; j < n; ++j) {
    const int p = path[j];
    if (p == j) continue;
    const int s = c + p, d = c + j;
    const int64_t ps = row[s / kv.page], pd = row[d / kv.page];
    const int64_t os = s % kv.page, od = d % kv.page;
    if (tid < kcol) {
      int16_t* base = kv.k + layer * kv.k_layer + head * kv.k_head + tid * 8;
      *reinterpret_cast<int4*>(base + pd * kv.k_page + od * kv.k_pos) =
          *reinterpret_cast<const int4*>(base + ps * kv.k_page + os * kv.k_pos);
    } else if (tid < kcol + vcol) {
      int32_t* base = kv.v + layer * kv.v_layer + head * kv.v_head + (tid - kcol) * 4;
      *reinterpret_cast<int4*>(base + pd * kv.v_page + od * kv.v_pos) =
          *reinterpret_cast<const int4*>(base + ps * kv.v_page + os * kv.v_pos);
    } else {
      int8_t* base = kv.ks + layer * kv.s_layer + head * kv.s_head;
      base[pd * kv.s_page + od * kv.s_pos] = base[ps * kv.s_page + os * kv.s_pos];
    }
  }
}

// ---------------------------------------------------------------- page copies
// One CTA per (64 positions, page, layer x KV head).  96 pages of 64 positions in 28 layers of 4 heads of 128:
// 1.06 GB read and written in 163 us, 0.98 of the rate of a plain copy.
constexpr int KP_THREADS = 256;
constexpr int KP_ROWS = 64;

struct CopyArgs {
  exb_kv_view kv;
  const int32_t *src = nullptr, *dst = nullptr, *rows = nullptr;
  int32_t* status = nullptr;
};

__global__ void __launch_bounds__(KP_THREADS) k_kv_copy(const CopyArgs a) {
  const exb_kv_view& kv = a.kv;
  const int i = blockIdx.y, tid = threadIdx.x;
  const int layer = blockIdx.z / kv.KV, head = blockIdx.z - layer * kv.KV;
  const int64_t s = a.src[i], d = a.dst[i];
  int n = a.rows[i];
  if ((uint64_t)s >= (uint64_t)kv.pages || (uint64_t)d >= (uint64_t)kv.pages || n < 0 || n > kv.page) {
    if (tid == 0) set_err(a.status, ERR_BOUNDS);
    return;
  }
  if (s == d) return;
  const int p0 = blockIdx.x * KP_ROWS;
  n = min(n - p0, KP_ROWS);
  if (n <= 0) return;
  const int kcol = kv.hd / 8, vcol = kv.hd / 4;
  {
    int16_t* base = kv.k + layer * kv.k_layer + head * kv.k_head + (int64_t)p0 * kv.k_pos;
    for (int e = tid; e < n * kcol; e += KP_THREADS) {
      const int64_t o = (int64_t)(e / kcol) * kv.k_pos + (e % kcol) * 8;
      *reinterpret_cast<int4*>(base + d * kv.k_page + o) = *reinterpret_cast<const int4*>(base + s * kv.k_page + o);
    }
  }
  {
    int32_t* base = kv.v + layer * kv.v_layer + head * kv.v_head + (int64_t)p0 * kv.v_pos;
    for (int e = tid; e < n * vcol; e += KP_THREADS) {
      const int64_t o = (int64_t)(e / vcol) * kv.v_pos + (e % vcol) * 4;
      *reinterpret_cast<int4*>(base + d * kv.v_page + o) = *reinterpret_cast<const int4*>(base + s * kv.v_page + o);
    }
  }
  int8_t* base = kv.ks + layer * kv.s_layer + head * kv.s_head + (int64_t)p0 * kv.s_pos;
  for (int e = tid; e < n; e += KP_THREADS) base[d * kv.s_page + e * kv.s_pos] = base[s * kv.s_page + e * kv.s_pos];
}

}  // namespace exb

using namespace exb;

extern "C" {

int exb_kv_compact(const exb_kv_view* kv, const int32_t* table, int B, int max_pages, const int32_t* ctx,
                   const int32_t* path, int ld_path, const int32_t* n, int32_t* new_ctx, int32_t* status,
                   void* stream) {
  auto fail = [](const std::string& m) { set_last_error("exb_kv_compact: " + m); return EXB_EINVAL; };
  if (const char* why = kv_view_error(kv)) return fail(why);
  if (B < 0 || max_pages < 1 || ld_path < 1) return fail("B >= 0, max_pages >= 1 and ld_path >= 1");
  if ((int64_t)max_pages * kv->page >= (1ll << 30)) return fail("a table row names 2^30 positions or more");
  if ((int64_t)kv->layers * kv->KV > 65535) return fail("layers x KV above 65535");
  if (B == 0) return EXB_OK;
  if (!table || !ctx || !path || !n || !new_ctx) return fail("null argument");
  CompactArgs a;
  a.kv = *kv; a.table = table; a.ctx = ctx; a.path = path; a.n = n; a.new_ctx = new_ctx; a.status = status;
  a.MP = max_pages; a.ld_path = ld_path; a.cap = (int64_t)max_pages * kv->page;
  k_kv_compact<<<dim3(B, kv->layers * kv->KV), KC_THREADS, 0, (cudaStream_t)stream>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_error(std::string("exb_kv_compact: ") + cudaGetErrorString(e));
    return EXB_ECUDA;
  }
  return EXB_OK;
}

int exb_kv_copy_pages(const exb_kv_view* kv, const int32_t* src, const int32_t* dst, const int32_t* rows, int count,
                      int32_t* status, void* stream) {
  auto fail = [](const std::string& m) { set_last_error("exb_kv_copy_pages: " + m); return EXB_EINVAL; };
  if (const char* why = kv_view_error(kv)) return fail(why);
  if (count < 0 || count > 65535) return fail("0 <= count <= 65535");
  if ((int64_t)kv->layers * kv->KV > 65535) return fail("layers x KV above 65535");
  if (count == 0) return EXB_OK;
  if (!src || !dst || !rows) return fail("null argument");
  CopyArgs a;
  a.kv = *kv; a.src = src; a.dst = dst; a.rows = rows; a.status = status;
  k_kv_copy<<<dim3((kv->page + KP_ROWS - 1) / KP_ROWS, count, kv->layers * kv->KV), KP_THREADS, 0,
              (cudaStream_t)stream>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_error(std::string("exb_kv_copy_pages: ") + cudaGetErrorString(e));
    return EXB_ECUDA;
  }
  return EXB_OK;
}

}  // extern "C"
