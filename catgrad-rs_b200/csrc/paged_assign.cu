// paged_assign.cu — pages for the next step: which rows' new tokens fit, the pages they get, and the tables, starts, positions
// and slots that the operators on the cache read (paged.h).
//
// With h pages held, f of them not the row's own, l cached and w new tokens a row needs max(ceil((l + w) / page) - h, 0) more; ended
// rows first put their pages f .. h on the stack.  Rows that run (l > f page) come before rows that begin; within a kind a row fits if the
// sum of needs up to and with it is no more than the stack, and the sum of tokens no more than the budget: two prefix sums, and a third
// over what fits for the starts.  So nobody overtakes another of its kind, and a row without needs is held up by tokens alone.
//
// What bounds it is the chain loads -> sums -> sums -> pages -> stores, some 0.5 to 1 us each, and the call.  Every block of a cluster makes the sums for itself (which
// needs no memory for them) and has its part of the tokens and of the pages that are given back: the row of each is looked up in shared memory, by halving, so that
// long prompts and single tokens cost the same.  The first token of a page that is new also writes the table.  8 rows 4.9 us, most of it the call; 391 rows,
// some ended, prompts that wait, 16384 places 10.6 us.
#include <algorithm>

#include "paged.h"
#include "tc_common.cuh"

namespace cg {

namespace {

struct AssignArgs {
  const uint32_t *lens, *fresh, *done, *first, *held, *n_free;  // fresh: the new tokens; done, first may be null
  uint32_t *free, *table, *starts, *lens_out, *held_out, *n_free_out, *positions, *slots;  // positions, slots may be null
  int64_t rows, cols, budget, room;  // budget: most tokens; room: of the stack
  int lg;
  int32_t* err;
};

// What a row asks for.
struct Ask {
  int64_t len, fresh, held, first;
  int64_t need;    // pages
  int64_t back;    // pages given back
  bool ended, runs;
};
__device__ __forceinline__ Ask ask_of(const AssignArgs& a, int64_t row, bool valid) {
  Ask x = {};
  if (row >= a.rows) return x;
  x.len = a.lens[row];
  x.held = a.held[row];
  x.first = a.first ? a.first[row] : 0;
  x.ended = a.done && a.done[row];
  const int64_t want = x.ended ? 0 : a.fresh[row], pages = (x.len + want + ((int64_t)1 << a.lg) - 1) >> a.lg;
  // (what cannot be: raised, and the row stays as it is)
  const bool ok = x.held <= a.cols && x.first <= x.held && (x.ended || (x.len <= x.held << a.lg && (want == 0 || pages <= a.cols)));
  if (!ok) *a.err = DEV_INDEX;
  if (!ok || !valid) {
    x.ended = false;
    return x;
  }
  if (x.ended) {
    x.back = x.held - x.first;
  } else {
    x.fresh = want;
    x.need = want > 0 ? max(pages - x.held, (int64_t)0) : 0;
    x.runs = x.len > x.first << a.lg;
  }
  return x;
}

constexpr int CHUNK = 1024;  // rows whose sums are made at a time, a thread each

// Exclusive sums over the block's threads, and over all; `sm` [32][N]
template <int N>
__device__ __forceinline__ void block_sums(const int64_t (&x)[N], int64_t (&before)[N], int64_t (&all)[N], int64_t* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t inc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) inc[i] = x[i];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc[i], o);
      if (lane >= o) inc[i] += y;
    }
  __syncthreads();  // (nobody reads what the last sums left)
  if (lane == 31)
#pragma unroll
    for (int i = 0; i < N; ++i) sm[warp * N + i] = inc[i];
  __syncthreads();
  // (every warp sums the warps' sums for itself)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t mine = lane < warps ? sm[lane * N + i] : 0;
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    before[i] = __shfl_sync(0xffffffffu, sum - mine, warp) + inc[i] - x[i];
    all[i] = __shfl_sync(0xffffffffu, sum, 31);
  }
}
// The last of the places 0 .. n whose start is at or before i
__device__ __forceinline__ int row_of(const uint32_t* start, int n, uint32_t i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(CHUNK) k_paged_assign(AssignArgs a) {
  __shared__ int64_t sums[32 * 4];
  __shared__ int64_t s_take[CHUNK];                      // pages taken before the row's, in the order in which they are taken
  __shared__ uint32_t s_start[CHUNK + 1];                // the rows' tokens among the chunk's
  __shared__ uint32_t s_len[CHUNK], s_held[CHUNK];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, threads = blockDim.x, blocks = gridDim.x, block = blockIdx.x, lane = tid & 31;
  const int64_t chunks = (a.rows + threads - 1) / threads;
  const int64_t n_free = *a.n_free;
  bool valid = n_free <= a.room;
  if (!valid) *a.err = DEV_INDEX;

  // ---- what is given back, and the totals ----
  int64_t back = 0, needs = 0, tokens = 0;  // all rows'; needs and tokens of those that run
  Ask mine = {};
  for (int64_t c = 0; c < chunks; ++c) {
    const int64_t row = c * threads + tid;
    mine = ask_of(a, row, valid);
    const int64_t x[3] = {mine.back, mine.runs ? mine.need : 0, mine.runs ? mine.fresh : 0};
    int64_t before[3], all[3];
    block_sums<3>(x, before, all, sums);
    if (all[0] > 0) {
      // the chunk's pages, dealt to all threads of the cluster
      s_start[tid] = (uint32_t)min(before[0], (int64_t)0xFFFFFFFF);
      s_held[tid] = (uint32_t)mine.first;
      __syncthreads();
      for (int64_t i = (int64_t)block * threads + tid; i < all[0] && n_free + back + i < a.room; i += (int64_t)blocks * threads) {
        const int r = row_of(s_start, threads, (uint32_t)i);
        a.free[n_free + back + i] = a.table[(c * threads + r) * a.cols + s_held[r] + (i - s_start[r])];
      }
    }
    back += all[0];
    needs += all[1];
    tokens += all[2];
  }
  if (n_free + back > a.room) {  // the stack cannot hold what is given back: nothing happens
    *a.err = DEV_INDEX;
    valid = false;
  }
  const int64_t count = valid ? n_free + back : n_free;
  if (blocks > 1) tc::cluster_sync_all();  // what was given back is on the stack
  else __syncthreads();

  // ---- who fits ----
  struct Got {
    int64_t n, take;
  };
  int64_t run_needs, run_tokens, new_needs, new_tokens, start, taken;  // totals so far
  auto clear = [&]() {
    run_needs = run_tokens = 0;
    new_needs = needs;  // (rows that begin come behind all that run)
    new_tokens = tokens;
    start = taken = 0;
  };
  auto chunk = [&](int64_t c, const Ask& x, int64_t* at, int64_t* chunk_tokens) {
    const int64_t y[4] = {x.runs ? x.need : 0, x.runs ? x.fresh : 0, x.runs ? 0 : x.need, x.runs ? 0 : x.fresh};
    int64_t before[4], all[4];
    block_sums<4>(y, before, all, sums);
    const int64_t pages = x.runs ? run_needs + before[0] : new_needs + before[2], toks = x.runs ? run_tokens + before[1] : new_tokens + before[3];
    const bool fits = x.fresh > 0 && (x.need == 0 || pages + x.need <= count) && toks + x.fresh <= a.budget;
    Got g = {fits ? x.fresh : 0, fits ? x.need : 0};
    const int64_t z[2] = {g.n, g.take};
    int64_t b2[2], a2[2];
    block_sums<2>(z, b2, a2, sums);
    s_start[tid] = (uint32_t)b2[0];
    if (tid == 0) s_start[threads] = (uint32_t)a2[0];
    s_take[tid] = pages;
    s_len[tid] = (uint32_t)x.len;
    s_held[tid] = (uint32_t)x.held;
    *at = start + b2[0];
    *chunk_tokens = a2[0];
    run_needs += all[0];
    run_tokens += all[1];
    new_needs += all[2];
    new_tokens += all[3];
    start += a2[0];
    taken += a2[1];
    return g;
  };
  auto keep = [&](int64_t row, const Ask& x, const Got& g, int64_t at) {  // by one block
    if (row >= a.rows) return;
    a.starts[row + 1] = (uint32_t)(at + g.n);
    a.lens_out[row] = (uint32_t)(x.ended ? 0 : x.len + g.n);
    a.held_out[row] = (uint32_t)(x.ended ? x.first : x.held + g.take);
  };
  clear();
  Got got = {};
  int64_t at = 0;
  for (int64_t c = 0; c < chunks; ++c) {
    if (chunks > 1 || !valid) mine = ask_of(a, c * threads + tid, valid);
    int64_t n;
    const int64_t start0 = start;
    got = chunk(c, mine, &at, &n);
    __syncthreads();
    for (int64_t i = (int64_t)block * threads + tid; i < n; i += (int64_t)blocks * threads) {
      const int lo = row_of(s_start, threads, (uint32_t)i);
      const int64_t row = c * threads + lo, pos = (int64_t)s_len[lo] + (i - s_start[lo]), col = pos >> a.lg, in_page = pos & (((int64_t)1 << a.lg) - 1);
      const int64_t j = col - s_held[lo];
      const bool names = j >= 0 && in_page == 0;
      if (!a.slots && !a.positions && !names) continue;
      uint32_t id = 0;
      if (j >= 0) id = a.free[count - 1 - (s_take[lo] + j)];
      else if (a.slots) id = a.table[row * a.cols + col];
      if (names) a.table[row * a.cols + col] = id;
      if (a.positions) a.positions[start0 + i] = (uint32_t)pos;
      if (a.slots) {
        const uint64_t slot = ((uint64_t)id << a.lg) + (uint64_t)in_page;
        if (slot >> 32) *a.err = DEV_INDEX;
        a.slots[start0 + i] = slot >> 32 ? 0xFFFFFFFFu : (uint32_t)slot;
      }
    }
  }
  // ---- the rows' new lengths: where inputs may be, so when all blocks have read them ----
  if (blocks > 1) tc::cluster_sync_all();
  else __syncthreads();
  if (block != 0) return;
  if (chunks == 1) {
    keep(tid, mine, got, at);
  } else {
    clear();
    for (int64_t c = 0; c < chunks; ++c) {
      const int64_t row = c * threads + tid;
      mine = ask_of(a, row, valid);
      int64_t n;
      got = chunk(c, mine, &at, &n);
      keep(row, mine, got, at);
    }
  }
  if (tid == 0) {
    a.starts[0] = 0;
    *a.n_free_out = (uint32_t)(count - taken);
  }
}

}  // namespace

}  // namespace cg

using namespace cg;

extern "C" int32_t cg_paged_assign(cg_ctx* c, const cg_tensor* lens, const cg_tensor* fresh, const cg_tensor* done, const cg_tensor* first, int64_t page,
                                   int64_t max_tokens, const cg_tensor* held, const cg_tensor* n_free, cg_tensor* free, cg_tensor* table, cg_tensor* starts,
                                   cg_tensor* lens_out, cg_tensor* held_out, cg_tensor* n_free_out, cg_tensor* positions, cg_tensor* slots) {
  if (!c) return CG_ERR_INVALID;
  CG_LAZY_EAGER_SCOPE(c);
  OnDevice on(c);
  if (!lens || !fresh || !held || !n_free || !free || !table || !starts || !lens_out || !held_out || !n_free_out) return fail(c, CG_ERR_INVALID, "null argument");
  const int64_t any[2] = {-1, -1};
  CG_TRY(check_tensor(c, table, "table", CG_U32, 2, any));
  const int64_t rows = table->dims[0], cols = table->dims[1], r0[1] = {rows}, r1[1] = {rows + 1}, one[1] = {1};
  CG_TRY(check_tensor(c, lens, "lens", CG_U32, 1, r0));
  CG_TRY(check_tensor(c, fresh, "new", CG_U32, 1, r0));
  if (done) CG_TRY(check_tensor(c, done, "done", CG_U32, 1, r0));
  if (first) CG_TRY(check_tensor(c, first, "first", CG_U32, 1, r0));
  CG_TRY(check_tensor(c, held, "held", CG_U32, 1, r0));
  CG_TRY(check_tensor(c, n_free, "n_free", CG_U32, 1, one));
  CG_TRY(check_tensor(c, free, "free", CG_U32, 1, any));
  CG_TRY(check_tensor(c, starts, "starts", CG_U32, 1, r1));
  CG_TRY(check_tensor(c, lens_out, "lens_out", CG_U32, 1, r0));
  CG_TRY(check_tensor(c, held_out, "held_out", CG_U32, 1, r0));
  CG_TRY(check_tensor(c, n_free_out, "n_free_out", CG_U32, 1, one));
  if (positions) CG_TRY(check_tensor(c, positions, "positions", CG_U32, 1, any));
  if (slots) CG_TRY(check_tensor(c, slots, "slots", CG_U32, 1, any));
  if (positions && slots && positions->dims[0] != slots->dims[0]) return fail(c, CG_ERR_SHAPE, "Shape mismatch in operation: slots");
  if (page < 8 || page > 1024 || (page & (page - 1))) return fail(c, CG_ERR_UNSUPPORTED, "a page holds 8, 16, .. 1024 tokens");
  if (max_tokens < 0) return fail(c, CG_ERR_INVALID, "bad argument");
  AssignArgs a = {};
  while ((int64_t)1 << a.lg < page) ++a.lg;
  if (rows > 65535) return fail(c, CG_ERR_UNSUPPORTED, "at most 65535 rows");
  if (cols > 0xFFFFFFFFll >> a.lg) return fail(c, CG_ERR_UNSUPPORTED, "too many columns");
  if (free->dims[0] > 0xFFFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "too many pages");
  // (lens, held and n_free may be written over their own)
  auto unless = [](const cg_tensor* in, const cg_tensor* out) {
    const Extent x(in), y(out);
    return x.lo == y.lo && x.hi == y.hi ? nullptr : in;
  };
  if (overlap_any({unless(lens, lens_out), fresh, done, first, unless(held, held_out), unless(n_free, n_free_out)},
                  {free, table, starts, lens_out, held_out, n_free_out, positions, slots}))
    return fail(c, CG_ERR_INVALID, "what is written overlaps an input or each other");
  a.budget = 0x7FFFFFFFll;  // (places of tokens are 31 bits everywhere)
  if (max_tokens > 0) a.budget = std::min(a.budget, max_tokens);
  if (positions) a.budget = std::min(a.budget, positions->dims[0]);
  if (slots) a.budget = std::min(a.budget, slots->dims[0]);
  a.lens = (const uint32_t*)lens->data();
  a.fresh = (const uint32_t*)fresh->data();
  a.done = done ? (const uint32_t*)done->data() : nullptr;
  a.first = first ? (const uint32_t*)first->data() : nullptr;
  a.held = (const uint32_t*)held->data();
  a.n_free = (const uint32_t*)n_free->data();
  a.free = (uint32_t*)free->data();
  a.table = (uint32_t*)table->data();
  a.starts = (uint32_t*)starts->data();
  a.lens_out = (uint32_t*)lens_out->data();
  a.held_out = (uint32_t*)held_out->data();
  a.n_free_out = (uint32_t*)n_free_out->data();
  a.positions = positions && positions->dims[0] ? (uint32_t*)positions->data() : nullptr;
  a.slots = slots && slots->dims[0] ? (uint32_t*)slots->data() : nullptr;
  a.rows = rows;
  a.cols = cols;
  a.room = free->dims[0];
  a.err = c->core->dev_err;
  for (cg_tensor* t : {free, table, starts, lens_out, held_out, n_free_out, positions, slots})
    if (t) written(t);
  // A thread per row, as far as a block goes; more blocks where a block's threads would have many tokens each.
  const int threads = rows <= 128 ? 128 : rows <= 512 ? 512 : CHUNK;
  const int blocks = std::min<int64_t>(a.budget, rows << 8) > 4 * threads ? 8 : 1;
  CG_CUDA(c, launch_kernel(c, k_paged_assign, dim3((unsigned)blocks), dim3((unsigned)threads), 0, -blocks, a));
  CG_LAUNCHED(c);
  return CG_OK;
}
