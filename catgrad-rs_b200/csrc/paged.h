// paged.h — what the operators on a paged key/value cache share (paged.cu, paged_attn.cu, beam.cu): the layout as the
// kernels see it, and the checks of their arguments.
//
// Keys and values lie in pages [n_pages, nkv, page, d], page a power of two.  Row r of a batch has the packed tokens
// starts[r] .. starts[r + 1], of its cached tokens lens[r] count (the new ones among them, so token i of n stands at
// position lens[r] - n + i), and position p lies in page table[r][p / page] at place p % page.  Everything that comes
// from device memory is checked where it is used: what is out of range raises the context's error word and is left out.
#pragma once

#include "runtime.h"

namespace cg {

struct PagedRows {
  const uint32_t* starts;   // [rows + 1]
  const uint32_t* lens;     // [rows]
  const uint32_t* table;    // [rows, cols]
  int64_t rows, cols, M;    // M: packed tokens of the batch's tensors
  int64_t n_pages;
  int lg;                   // page = 1 << lg
  int32_t* err;
};

#ifdef __CUDACC__
#define CG_HD __host__ __device__ __forceinline__
#else
#define CG_HD inline
#endif
// The new tokens of a row: the first one's place, how many, and the row's length with them.  False: there is nothing to do, or
// (raised) what the tables say cannot be.
CG_HD bool row_span(const PagedRows& p, int64_t row, int64_t most, int64_t* tok0, int64_t* n, int64_t* len) {
  const int64_t a = p.starts[row], b = p.starts[row + 1];
  *tok0 = a;
  *n = b - a;
  *len = p.lens[row];
  if (a == b) return false;
  const bool ok = a < b && b <= p.M && b - a <= most && b - a <= *len && *len <= (p.cols << p.lg);
  if (!ok) *p.err = DEV_INDEX;
  return ok;
}
// The page of a position below cols * page; -1 (raised) where the table names none.
CG_HD int64_t page_of(const PagedRows& p, int64_t row, int64_t pos) {
  const int64_t id = p.table[row * p.cols + (pos >> p.lg)];
  if (id < p.n_pages) return id;
  *p.err = DEV_INDEX;
  return -1;
}

// Groups of neighbouring rows that have their first tokens in common.
struct PagedGroups {
  const uint32_t* rows;    // [n + 1], ascending: group g has the rows rows[g] .. rows[g + 1]
  const uint32_t* shared;  // [n]: the tokens in common
  int64_t n;
  int64_t most;            // tokens in common, at most
};
// A group's first row, packed tokens and shared tokens.  False (raised): its numbers cannot be.
CG_HD bool group_span(const PagedRows& p, const PagedGroups& s, int64_t g, int64_t* row0, int64_t* rows, int64_t* tok0, int64_t* n, int64_t* shared) {
  const int64_t a = s.rows[g], b = s.rows[g + 1], keys = s.shared[g];
  *row0 = a;
  *rows = b - a;
  *shared = keys;
  *tok0 = *n = 0;
  bool ok = a <= b && b <= p.rows && keys <= s.most && keys <= (p.cols << p.lg);
  if (ok) {
    const int64_t t0 = p.starts[a], t1 = p.starts[b];
    *tok0 = t0;
    *n = t1 - t0;
    ok = t0 <= t1 && t1 <= p.M;
  }
  if (!ok) *p.err = DEV_INDEX;
  return ok;
}
// The row of a packed token of the rows row0 .. row0 + rows (by halving; rows without tokens are passed over), and where the token stands.
CG_HD int64_t position_of(const PagedRows& p, int64_t row0, int64_t rows, int64_t token) {
  int64_t lo = row0, hi = row0 + rows;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if ((int64_t)p.starts[mid] <= token) lo = mid;
    else hi = mid;
  }
  return (int64_t)p.lens[lo] - (int64_t)p.starts[lo + 1] + token;
}

// The context's device is current while this lives.
struct OnDevice {
  int before = -1;
  explicit OnDevice(const cg_ctx* c) {
    int now = -1;
    if (cudaGetDevice(&now) == cudaSuccess && now != c->core->device && cudaSetDevice(c->core->device) == cudaSuccess) before = now;
  }
  ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};

// ---- checks of arguments (host) ----

inline int same_device(cg_ctx* c, const cg_tensor* t, const char* what) {
  if (!t->buf) return fail(c, CG_ERR_INVALID, std::string(what) + " is recorded in another context");
  if (t->buf->core->device != c->core->device) return fail(c, CG_ERR_INVALID, std::string(what) + " is on another device");
  return CG_OK;
}
// `t` has this rank (and, where given >= 0, these dims), is F32 or U32, and contiguous where that is asked for (one without elements is).
inline int check_tensor(cg_ctx* c, const cg_tensor* t, const char* what, int tag, int rank, const int64_t* dims, bool contiguous = true) {
  if (!t) return fail(c, CG_ERR_INVALID, std::string(what) + " is null");
  if (t->tag != tag) return fail(c, CG_ERR_DTYPE, std::string(what) + (tag == CG_F32 ? " wants F32" : " wants U32"));
  bool ok = t->rank == rank;
  for (int i = 0; ok && i < rank; ++i) ok = dims[i] < 0 || t->dims[i] == dims[i];
  if (!ok) return fail(c, CG_ERR_SHAPE, std::string("Shape mismatch in operation: ") + what);
  if (contiguous && t->numel() && !t->contiguous()) return fail(c, CG_ERR_UNSUPPORTED, std::string(what) + " must be contiguous");
  return same_device(c, t, what);
}
// Where a tensor's memory lies (its whole extent); nowhere: null or without elements.
struct Extent {
  uintptr_t lo = 0, hi = 0;
  Extent() = default;
  Extent(const cg_tensor* t) {
    if (!t) return;
    int64_t last = 0;
    for (int i = 0; i < t->rank; ++i) {
      if (t->dims[i] == 0) return;
      last += (t->dims[i] - 1) * t->strides[i];
    }
    lo = (uintptr_t)t->data();
    hi = lo + (size_t)(last + 1) * t->esize();
  }
};
inline bool overlap(const Extent& a, const Extent& b) { return a.lo < b.hi && b.lo < a.hi; }
// Whether what is written touches an input, or one of the others that are written.
template <int NI, int NO>
inline bool overlap_any(const cg_tensor* const (&in)[NI], const cg_tensor* const (&out)[NO]) {
  Extent o[NO];
  for (int i = 0; i < NO; ++i) {
    o[i] = Extent(out[i]);
    for (int j = 0; j < i; ++j)
      if (overlap(o[i], o[j])) return true;
  }
  for (const cg_tensor* t : in) {
    const Extent e(t);
    for (const Extent& x : o)
      if (overlap(e, x)) return true;
  }
  return false;
}
// The pages: k and v alike, [n_pages, nkv, page, d] (with `layers`, [layers, n_pages, nkv, page, d]).
inline int check_pages(cg_ctx* c, const cg_tensor* k, const cg_tensor* v, bool layers, int* lg) {
  const int64_t any[5] = {-1, -1, -1, -1, -1};
  const int rank = layers ? 5 : 4;
  if (!k || !v) return fail(c, CG_ERR_INVALID, "pages are null");
  CG_TRY(check_tensor(c, k, "k_pages", CG_F32, rank, any));
  CG_TRY(check_tensor(c, v, "v_pages", CG_F32, rank, k->dims));
  if (k->storage != v->storage) return fail(c, CG_ERR_DTYPE, "k_pages and v_pages are stored differently");
  const int64_t page = k->dims[rank - 2], d = k->dims[rank - 1];
  if (page < 8 || page > 1024 || (page & (page - 1))) return fail(c, CG_ERR_UNSUPPORTED, "a page holds 8, 16, .. 1024 tokens");
  if (d < 8 || d > 256 || d % 8) return fail(c, CG_ERR_UNSUPPORTED, "head sizes are multiples of 8 up to 256");
  if (k->dims[rank - 4] > 0xFFFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "too many pages");
  if (((uintptr_t)k->data() | (uintptr_t)v->data()) % 16) return fail(c, CG_ERR_UNSUPPORTED, "pages begin on a 16-byte boundary");
  int b = 0;
  while ((int64_t)1 << b < page) ++b;
  *lg = b;
  return CG_OK;
}

// The rows' tables against M packed tokens and pages of [n_pages, ..].
inline int check_rows(cg_ctx* c, const cg_tensor* table, const cg_tensor* starts, const cg_tensor* lens, int64_t M, int64_t n_pages, int lg,
                      PagedRows* out) {
  const int64_t any[2] = {-1, -1};
  CG_TRY(check_tensor(c, table, "table", CG_U32, 2, any));
  const int64_t rows = table->dims[0], r1[1] = {rows + 1}, r0[1] = {rows};
  CG_TRY(check_tensor(c, starts, "starts", CG_U32, 1, r1));
  CG_TRY(check_tensor(c, lens, "lens", CG_U32, 1, r0));
  if (rows > 65535) return fail(c, CG_ERR_UNSUPPORTED, "at most 65535 rows");
  if (M > 0x7FFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "too many tokens");
  if (table->dims[1] > (1ll << 40) >> lg) return fail(c, CG_ERR_UNSUPPORTED, "too many columns");
  out->starts = (const uint32_t*)starts->data();
  out->lens = (const uint32_t*)lens->data();
  out->table = (const uint32_t*)table->data();
  out->rows = rows;
  out->cols = table->dims[1];
  out->M = M;
  out->n_pages = n_pages;
  out->lg = lg;
  out->err = c->core->dev_err;
  return CG_OK;
}

}  // namespace cg
