// paged_attn.h — the arguments of attention over a paged cache, and the kernels it is run on.
#pragma once

#include "mma.cuh"
#include "paged.h"

namespace cg {

// Attention over keys that groups of rows have in common, in three launches: the first has all of a group's queries and a chunk of
// the shared keys in a block, the second a row's own keys; both leave, per token and head, the output against their own maximum, that maximum (of scores in
// units of log2) and the sum of exponentials, and the third joins these parts.
struct SharedParts {
  PagedGroups groups;
  int64_t chunk;   // keys of a chunk
  int chunks;      // of the longest prefix
  float* out;      // [chunks + 1][M][heads][d], the last for the rows' own keys
  float2* ml;      // [chunks + 1][M][heads]
  // keys of a row behind the prefix, by the table's width (which stands for the lengths)
  int64_t own(int64_t longest) const { return longest > groups.most ? longest - groups.most : longest; }
};

// Which keys of a row a kernel takes: ALL of them; CHUNK: the queries are a group's, the keys a chunk of what its rows have in common; OWN: those behind that.
// What comes before the launch of the chunks is complete when that lets the next one begin, so OWN waits for nothing until it ends; its last block does then, so
// that what waits for it waits for the chunks too. (While all its blocks did, those that ended beside the chunks kept their
// room on an SM to themselves: 64 rows behind 16001 tokens, 8 key heads of 128, 70.5 us instead of 56.4.)
enum KeysOf { ALL, CHUNK, OWN };

struct PagedAttnArgs {
  PagedRows rows;
  const void *q, *k_pages, *v_pages;
  void* out;
  int64_t q_ld, q_hs;   // from one token and one head of q to the next
  int64_t most;         // new tokens of a row, at most
  int64_t window;       // 0 = none
  float scale, cap;     // cap 0 = none
  int nh, nkv, d;
  SharedParts sh;       // (of shared attention)
};

// Soft-caps c tanh(x / c), in units of log2: kernels take c log2(e) and the factors of a product q k in x / c (`in`) and in the exponent
// of 2 of exp(-2 x / c) (`unit`).  tanh(y) / y in y^2 up to y = 3/4, fitted to the least largest relative error: 3e-8, half a step
// of f32.  Beyond that 2 / (1 + e^-2y) - 1, which would lose what is small against 1.
constexpr CG_HD float tanh_term(int i) {
  return i == 0 ? 1.f : i == 1 ? -0.33332958817481995f : i == 2 ? 0.1332540661096573f : i == 3 ? -0.05334442853927612f
       : i == 4 ? 0.019582903012633324f : -0.004716253839433193f;
}
#ifdef __CUDACC__
__device__ __forceinline__ bool last_block() { return blockIdx.x + 1 == gridDim.x && blockIdx.y + 1 == gridDim.y && blockIdx.z + 1 == gridDim.z; }
// A group of rows that a tile belongs to: its first row, rows, first packed token, tokens and shared tokens, and the tile's number in it.
struct GroupTile {
  int64_t row0, rows, tok0, n, shared, tile;
};
// By a whole warp: the group of tile `t` of all groups' tiles; false if there is none.  A token has `heads` query rows of a tile's `size`.
__device__ __forceinline__ bool group_of_tile(const PagedRows& p, const PagedGroups& s, int64_t t, int64_t heads, int64_t size, GroupTile* out) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int64_t g0 = 0; g0 < s.n; g0 += 32) {
    GroupTile x = {};
    int64_t mine = 0;
    if (g0 + lane < s.n && group_span(p, s, g0 + lane, &x.row0, &x.rows, &x.tok0, &x.n, &x.shared) && x.shared > 0) mine = (x.n * heads + size - 1) / size;
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const uint32_t has = __ballot_sync(0xffffffffu, t < before + sum);
    if (has) {
      const int at = __ffs(has) - 1;
      out->tile = t - (before + __shfl_sync(0xffffffffu, sum - mine, at));
      out->row0 = __shfl_sync(0xffffffffu, x.row0, at);
      out->rows = __shfl_sync(0xffffffffu, x.rows, at);
      out->tok0 = __shfl_sync(0xffffffffu, x.tok0, at);
      out->n = __shfl_sync(0xffffffffu, x.n, at);
      out->shared = __shfl_sync(0xffffffffu, x.shared, at);
      return true;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}
// By a whole warp: the group of a row (-1: it has none) and the tokens that it shares.
__device__ __forceinline__ int64_t group_of_row(const PagedGroups& s, int64_t row, int64_t* shared) {
  const int lane = threadIdx.x & 31;
  for (int64_t g0 = 0; g0 < s.n; g0 += 32) {
    const int64_t g = g0 + lane;
    uint32_t a = 0, b = 0, keys = 0;
    if (g < s.n) {
      a = s.rows[g];
      b = s.rows[g + 1];
      keys = s.shared[g];
    }
    const uint32_t has = __ballot_sync(0xffffffffu, (int64_t)a <= row && row < (int64_t)b);
    if (has) {
      const int at = __ffs(has) - 1;
      *shared = __shfl_sync(0xffffffffu, keys, at);
      return g0 + at;
    }
  }
  *shared = 0;
  return -1;
}
// By a whole warp: of the rows row0 .. row0 + rows those that end at or before a packed token (32 places at a time, so that thousands of rows take three
// loads); row0 + that is the token's row.
__device__ __forceinline__ int64_t rows_before(const PagedRows& p, int64_t row0, int64_t rows, int64_t token) {
  const int lane = threadIdx.x & 31;
  int64_t base = 0, len = rows;
  while (len > 0) {
    const int64_t step = (len + 31) / 32, r = base + (lane + 1) * step - 1;
    const bool before = r < base + len && (int64_t)p.starts[row0 + r + 1] <= token;
    const int64_t k = __popc(__ballot_sync(0xffffffffu, before)), skip = min(k * step, len);
    base += skip;
    len = step == 1 ? 0 : min(len - skip, step - 1);  // (the next probe's row is not before the token)
  }
  return base;
}
// By a whole warp: where the new tokens of the rows of the packed tokens t0 .. t1 (of rows row0 .. row0 + rows) stand, the first and the last position.
__device__ __forceinline__ void tile_positions(const PagedRows& p, int64_t row0, int64_t rows, int64_t t0, int64_t t1, int64_t* first, int64_t* last) {
  const int64_t r0 = rows_before(p, row0, rows, t0), r1 = min(rows_before(p, row0, rows, t1), rows - 1);
  uint32_t lo = 0xffffffffu, hi = 0;
  for (int64_t i = r0 + (threadIdx.x & 31); i <= r1; i += 32) {
    const uint32_t len = p.lens[row0 + i], n = p.starts[row0 + i + 1] - p.starts[row0 + i];
    if (n > 0 && n <= len) {
      lo = min(lo, len - n);
      hi = max(hi, len - 1);
    }
  }
  *first = __reduce_min_sync(0xffffffffu, lo);
  *last = __reduce_max_sync(0xffffffffu, hi);
}
// The chunks of what a row's new tokens tok0 .. tok0 + n have in common with others; -1 (raised): what the tables say cannot be.
__device__ __forceinline__ int chunks_of(const PagedRows& p, const SharedParts& s, int64_t group, int64_t tok0, int64_t n) {
  if (group < 0) return 0;
  int64_t row0, rows, t0, tokens, shared;
  if (!group_span(p, s.groups, group, &row0, &rows, &t0, &tokens, &shared)) return -1;
  if (tok0 < t0 || tok0 + n > t0 + tokens) {  // (starts that do not ascend: the chunks have other tokens)
    *p.err = DEV_INDEX;
    return -1;
  }
  return (int)((shared + s.chunk - 1) / s.chunk);
}
__device__ __forceinline__ float soft_cap_near(float y, float cap_log2e) {
  const float u = y * y;
  float f = tanh_term(5);
#pragma unroll
  for (int i = 4; i >= 0; --i) f = fmaf(f, u, tanh_term(i));
  return cap_log2e * y * f;
}
__device__ __forceinline__ float soft_cap(float x, float cap_log2e, float in, float unit) {
  const float y = x * in, far = fmaf(2.f * cap_log2e, rcp_newton(1.f + fast_exp2(x * unit)), -cap_log2e);
  float v;  // (both are worked out: a branch per score costs more)
  asm("{\n\t.reg .pred p;\n\tsetp.le.f32 p, %1, 0f3F400000;\n\tselp.f32 %0, %2, %3, p;\n\t}" : "=f"(v) : "f"(fabsf(y)), "f"(soft_cap_near(y, cap_log2e)), "f"(far));
  return v;
}
#endif

// Prompts in bf16 on tcgen05 (paged_fa.cu)
bool paged_fa_supported(const PagedAttnArgs& a);
int paged_fa(cg_ctx* c, const PagedAttnArgs& a);
bool paged_fa_prefix_supported(const PagedAttnArgs& a);
int paged_fa_prefix(cg_ctx* c, const PagedAttnArgs& a);  // the chunks of shared keys
int paged_fa_own(cg_ctx* c, const PagedAttnArgs& a);     // the rows' own keys
int64_t paged_fa_chunk(const PagedAttnArgs& a);
int64_t paged_fa_slots(const PagedAttnArgs& a);          // blocks that chunks are cut for
constexpr int SHARED_CHUNK = 128;                        // keys of a chunk, at least
// A few tokens per row, bf16 (paged_dec.cu)
bool paged_dec_supported(const PagedAttnArgs& a);
int paged_dec(cg_ctx* c, const PagedAttnArgs& a);
int paged_dec_own(cg_ctx* c, const PagedAttnArgs& a);    // the rows' own keys

// ---- into how many shares a row's keys are cut ----
constexpr int SHARES = 5;  // 1, 2, 4, 8 or 16: the blocks of a cluster

// Clusters of 1, 2, .. blocks along z that run at a time (asked once per kernel, which keeps `known`); -1: none.
struct AtATime {
  int n[64][SHARES] = {};
};
template <typename... KArgs>
int at_a_time(AtATime& known, int device, int i, void (*kernel)(KArgs...), int threads, size_t smem) {
  int& n = known.n[device & 63][i];
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1024, 1, 1u << i);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1u << i;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      got = 0;
    }
    n = got > 0 ? got : -1;
  }
  return n;
}
// The shares of least time: a block takes `base` us and `round` for each of its rounds of `keys` keys, joining 2 to 4.5.  What does not run
// at the same time takes turns (between whole turns and their mean, as rows differ): clusters beyond at_a_time, and, where one
// block keeps an SM's units busy, blocks beyond the SMs; part_seen is what of a row a query sees in the mean, 0 where that
// does not count.
template <typename F>
int pick_shares(F&& n_of, int most, int64_t clusters, int64_t keys_of_row, int keys, double base, double round, double part_seen) {
  constexpr double join[SHARES] = {0., 2., 2., 2.5, 4.5};
  int shares = 1;
  double best = 1e300;
  for (int i = 0; i < SHARES && 1 << i <= most; ++i) {
    const int n = n_of(i);
    if (n <= 0) continue;
    auto turns_of = [](double x) { return 0.5 * (x + (double)(int64_t)(x + 0.999999)); };
    double turns = turns_of((double)clusters / n);
    const double by_sm = turns_of((double)(clusters << i) * part_seen / 148.);
    if (part_seen > 0. && by_sm > turns) turns = by_sm;
    const int64_t tiles = keys_of_row / keys + 1;
    const double cost = (turns > 1. ? turns : 1.) * (base + join[i] + round * (double)((tiles + (1 << i) - 1) >> i));
    if (cost < best) {
      best = cost;
      shares = 1 << i;
    }
  }
  return shares;
}

}  // namespace cg
