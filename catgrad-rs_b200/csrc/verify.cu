// verify.cu — drafted tokens before the target's probabilities (speculative decoding), from given random numbers.
//
// A row has run its last token and its drafts x_1 .. x_k; logits l_i stand behind each.  With p_i = softmax(l_i / T) and the drafter's
// probabilities q_i, draft i + 1 stands while u_i q_i(x) < p_i(x); behind the first that does not (place a) the next token is drawn from
// max(p_a - q_a, 0), behind all of them from p_k: the first token whose inclusive sum is above u times the whole.  What is put out is then
// distributed as if the target had drawn it token by token.  T = 0: the draft has to be the largest logit, which comes next anyway.
//
// The token that a random number falls on depends on sums over the vocabulary to their last bits (100000 borders: an error of 2^-24
// moves 1 % of the draws to a neighbour), so the weights that are drawn from and their sums have 64 bits; the sums that drafts are judged by
// have exponentials in f32, which moves a border by 2^-22 of itself.
//
// A cluster has a row, its blocks equal slices of the vocabulary.  Logits are read once: a position's slice stays in shared memory, where
// the draw finds it; positions behind the first rejected draft are not read unless they were asked for ahead.
#include <algorithm>

#include "mma.cuh"
#include "paged.h"
#include "tc_common.cuh"

namespace cg {

namespace {

using namespace tc;

constexpr int VT = 512;          // threads of a block
constexpr int MOST_BLOCKS = 16;  // of a cluster
constexpr int MOST_AHEAD = 8;    // positions in shared memory
constexpr uint32_t NONE = 0xFFFFFFFFu;
constexpr float NO_LOGIT = -INFINITY;

struct VerifyArgs {
  const void *logits, *probs;  // probs may be null: a draft is its drafter's only token
  int64_t l_ld, q_ld;          // from one place to the next
  const uint32_t *tokens, *starts, *lens;  // lens may be null
  const float *uniform, *temperature;      // temperature may be null: 1
  uint32_t *accepted, *next, *lens_out;
  int64_t rows, M, V, most;
  int slice;                   // tokens of a block
  int ahead;                   // positions asked for at a time
  int probs16;
  uint32_t stride;             // bytes of a position in shared memory
  int32_t* err;
};

template <typename T>
__device__ __forceinline__ float widen(T x);
template <>
__device__ __forceinline__ float widen<float>(float x) { return x; }
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// (NaN counts as -inf)
template <typename T>
__device__ __forceinline__ float logit(T x) { return fmaxf(widen(x), NO_LOGIT); }

__device__ __forceinline__ double exp64(double x) { return exp(x); }

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
// Of the lanes' parts x of a sum that begins at `begin`: the first one with which it is above t, and the sum before it; without one (`none`), the
// last part above 0.  (Sums of other lanes come in another order: a part of 0 may seem to be above.)
__device__ __forceinline__ int first_above(double x, double begin, double t, double* before, bool* none) {
  const int lane = threadIdx.x & 31;
  double sum = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  const uint32_t above = __ballot_sync(0xffffffffu, x > 0.0 && begin + sum > t), some = __ballot_sync(0xffffffffu, x > 0.0);
  const double lower = __shfl_up_sync(0xffffffffu, sum, 1);
  *none = above == 0;
  const int at = above ? __ffs(above) - 1 : some ? 31 - __clz(some) : 0;
  *before = begin + __shfl_sync(0xffffffffu, lane ? lower : 0.0, at);
  return at;
}
__device__ __forceinline__ void put_remote(const void* p, uint32_t rank, double x) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(x) : "memory");
}
__device__ __forceinline__ void put_remote(const void* p, uint32_t rank, uint32_t x) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(x) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(VT) k_verify_drafts(VerifyArgs a) {
  constexpr int E = 16 / sizeof(T);  // values of a vector
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ double w_sum[VT / 32];
  __shared__ float w_top[VT / 32];
  __shared__ uint32_t w_at[VT / 32], w_last[VT / 32];
  __shared__ double told_sum[2][MOST_AHEAD][MOST_BLOCKS], total[2][MOST_BLOCKS];
  __shared__ uint32_t told_top[2][MOST_AHEAD][MOST_BLOCKS], told_at[2][MOST_AHEAD][MOST_BLOCKS];
  __shared__ double pos_sum[MOST_AHEAD];
  __shared__ float pos_top[MOST_AHEAD];
  __shared__ uint32_t pos_at[MOST_AHEAD];
  __shared__ int verdict;            // of a group's positions: the place of the first that ends the row, or -1
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int blocks = (int)gridDim.x, block = (int)blockIdx.x;
  const int64_t row = blockIdx.y;
  // (the same in all blocks of a cluster, as everything that decides which way they go)
  const int64_t s0 = a.starts[row], s1 = a.starts[row + 1], n = s1 - s0;
  if (n == 0) return;
  bool ok = s0 < s1 && s1 <= a.M && n <= a.most && (!a.lens || a.lens[row] >= n - 1);
  if (ok) {
    bool bad = false;
    for (int64_t i = 1 + tid; i < n; i += VT) bad = bad || a.tokens[s0 + i] >= a.V;
    ok = !__syncthreads_or(bad);
  }
  if (!ok) {
    if (tid == 0) *a.err = DEV_INDEX;
    return;
  }
  // (nothing is put into another block's memory before it runs: waited for ahead of the first put)
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const float heat_in = a.temperature ? a.temperature[row] : 1.f;
  const bool greedy = !(heat_in > 0.f);
  // (temperatures beyond 2^+-100 act as these)
  const float heat = fminf(fmaxf(heat_in, 0x1p-100f), 0x1p100f), unit = 1.4426950408889634f / heat;
  const double cold = 1.0 / (double)heat;
  const int64_t lo = std::min<int64_t>((int64_t)block * a.slice, a.V), hi = std::min<int64_t>(lo + a.slice, a.V);
  const int count = (int)(hi - lo);

  // ---- a position's slice into shared memory: whole vectors as they lie, ragged ends value by value ----
  auto place = [&](int64_t pos) { return (const T*)a.logits + (s0 + pos) * a.l_ld + lo; };
  auto phase_of = [&](int64_t pos) { return (int)(((uintptr_t)place(pos) & 15) / sizeof(T)); };
  auto request = [&](int64_t pos, int buffer) {
    const T* src = place(pos);
    const int phase = phase_of(pos), vectors = (phase + count + E - 1) / E;
    uint8_t* dst = ring + (size_t)buffer * a.stride;
    const T* base = src - phase;
    for (int v = tid; v < vectors; v += VT) {
      const int j0 = v * E - phase;
      if (j0 >= 0 && j0 + E <= count) {
        cp_async16(smem_u32(dst + v * 16), base + v * E, 16);
      } else {
        T* to = (T*)(dst + v * 16);
        for (int e = 0; e < E; ++e) to[e] = j0 + e >= 0 && j0 + e < count ? src[j0 + e] : (T)NO_LOGIT;
      }
    }
    cp_async_commit();
  };

  int64_t first = 0;  // of the group
  int parity = 0, group = (int)std::min<int64_t>(a.ahead, n), stop = -1;
  for (;;) {
    for (int j = 0; j < group; ++j) request(first + j, j);
    // what the drafts are judged by, asked for meanwhile
    float draft_logit = 0.f, u = 0.f, q = 1.f;
    uint32_t draft = NONE;
    if (tid < group) {
      const int64_t pos = first + tid, m = s0 + pos;
      if (pos < n - 1) {
        draft = a.tokens[m + 1];
        u = a.uniform[m];
        draft_logit = logit(((const T*)a.logits)[m * a.l_ld + draft]);
        if (a.probs) {
          q = a.probs16 ? __bfloat162float(((const __nv_bfloat16*)a.probs)[m * a.q_ld + draft]) : ((const float*)a.probs)[m * a.q_ld + draft];
          q = q > 0.f ? q : 0.f;
        }
      }
    }
    cp_async_wait_all();
    __syncthreads();
    if (first == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    for (int j = 0; j < group; ++j) {
      const int phase = phase_of(first + j), vectors = (phase + count + E - 1) / E;
      const uint4* src = (const uint4*)(ring + (size_t)j * a.stride);
      float top = NO_LOGIT, sum = 0.f;
      uint32_t at = NONE;
      for (int v = tid; v < vectors; v += VT) {
        const uint4 w = src[v];
        const T* x = (const T*)&w;
        float y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = logit(x[e]);
        if (greedy) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (y[e] > top) {
              top = y[e];
              at = (uint32_t)(lo + v * E + e - phase);
            }
        } else {
          float t = y[0];
#pragma unroll
          for (int e = 1; e < E; ++e) t = fmaxf(t, y[e]);
          if (t > top) {
            sum *= fast_exp2((top - t) * unit);
            top = t;
          }
          if (top > NO_LOGIT) {
#pragma unroll
            for (int e = 0; e < E; ++e) sum += fast_exp2((y[e] - top) * unit);
          }
        }
      }
      // the block's
      float t = top;
#pragma unroll
      for (int o = 16; o; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
      double s = top > NO_LOGIT ? (double)sum * (double)fast_exp2((top - t) * unit) : 0.0;
      s = warp_sum(s);
      const uint32_t i = __reduce_min_sync(0xffffffffu, top == t ? at : NONE);
      if (lane == 0) {
        w_top[warp] = t;
        w_sum[warp] = s;
        w_at[warp] = i;
      }
      __syncthreads();
      if (warp == 0) {
        const bool there = lane < VT / 32;
        float wt = there ? w_top[lane] : NO_LOGIT, bt = wt;
#pragma unroll
        for (int o = 16; o; o >>= 1) bt = fmaxf(bt, __shfl_xor_sync(0xffffffffu, bt, o));
        double ws = there && wt > NO_LOGIT ? w_sum[lane] * (double)fast_exp2((wt - bt) * unit) : 0.0;
        ws = warp_sum(ws);
        const uint32_t wi = __reduce_min_sync(0xffffffffu, there && wt == bt ? w_at[lane] : NONE);
        if (lane < blocks) {
          put_remote(&told_sum[parity][j][block], (uint32_t)lane, ws);
          put_remote(&told_top[parity][j][block], (uint32_t)lane, __float_as_uint(bt));
          put_remote(&told_at[parity][j][block], (uint32_t)lane, wi);
        }
      }
      __syncthreads();
    }
    cluster_sync_all();
    // ---- the verdicts, in every block alike ----
    if (warp == 0) {
      bool ends = false;
      if (lane < group) {
        float top = NO_LOGIT;
        for (int b = 0; b < blocks; ++b) top = fmaxf(top, __uint_as_float(told_top[parity][lane][b]));
        double sum = 0.0;
        uint32_t at = NONE;
        for (int b = 0; b < blocks; ++b) {
          const float t = __uint_as_float(told_top[parity][lane][b]);
          if (t > NO_LOGIT) sum += told_sum[parity][lane][b] * (double)fast_exp2((t - top) * unit);
          if (t == top) at = min(at, told_at[parity][lane][b]);
        }
        const bool some = top > NO_LOGIT && top < INFINITY;  // (else nothing has a probability)
        pos_top[lane] = top;
        pos_sum[lane] = sum;
        pos_at[lane] = at;
        ends = first + lane == n - 1;
        if (!ends) {
          const bool stands = greedy ? draft == at : (double)u * (double)q * sum < exp64(((double)draft_logit - (double)top) * cold);
          ends = !(some && stands);
        }
      }
      const uint32_t which = __ballot_sync(0xffffffffu, ends);
      if (lane == 0) verdict = which ? __ffs(which) - 1 : -1;
    }
    parity ^= 1;
    __syncthreads();
    stop = verdict;
    if (stop >= 0) break;
    first += group;
    group = (int)std::min<int64_t>(a.ahead, n - first);
  }

  // ---- the next token, at position first + stop ----
  const int64_t pos = first + stop, m = s0 + pos;
  const float top = pos_top[stop];
  uint32_t token = NONE;
  bool write = block == 0 && tid == 0;
  if (!(top > NO_LOGIT && top < INFINITY)) {
    token = NONE;
  } else if (greedy) {
    token = pos_at[stop];
  } else {
    const T* values = (const T*)(ring + (size_t)stop * a.stride) + phase_of(pos);
    const double t64 = (double)top;
    // a warp has the same number of neighbouring tokens
    const int per = ((count + VT / 32 - 1) / (VT / 32) + 31) & ~31, v0 = min(warp * per, count), v1 = min(v0 + per, count);
    const uint32_t draft = pos < n - 1 ? a.tokens[m + 1] : NONE;
    const __nv_bfloat16* q16 = (const __nv_bfloat16*)a.probs + m * a.q_ld + lo;
    const float* q32 = (const float*)a.probs + m * a.q_ld + lo;
    auto weight = [&](int j) { return exp64(((double)logit(values[j]) - t64) * cold); };
    double whole = 0.0;  // sum of the weights, of all tokens
    int mode = pos < n - 1 ? (a.probs ? 2 : 1) : 0;  // what is drawn from: 0 weights, 1 weights but the draft's, 2 what the drafter's probabilities leave
    auto rest = [&](int j) {
      const double e = weight(j);
      if (mode == 0) return e;
      if (mode == 1) return lo + j == draft ? 0.0 : e;
      const float q = a.probs16 ? __bfloat162float(q16[j]) : q32[j];
      const double left = e - (double)(q > 0.f ? q : 0.f) * whole;
      return left > 0.0 ? left : 0.0;
    };
    // sums of the warps (left in w_sum), and of all blocks (in total[parity])
    auto sums = [&](auto f) {
      double s = 0.0;
      for (int j = v0 + lane; j < v1; j += 32) s += f(j);
      s = warp_sum(s);
      __syncthreads();
      if (lane == 0) w_sum[warp] = s;
      __syncthreads();
      if (warp == 0) {
        double b = lane < VT / 32 ? w_sum[lane] : 0.0;
        b = warp_sum(b);
        if (lane < blocks) put_remote(&total[parity][block], (uint32_t)lane, b);
      }
      cluster_sync_all();
      double all = 0.0;
      for (int b = 0; b < blocks; ++b) all += total[parity][b];
      parity ^= 1;
      return all;
    };
    double all = 0.0;
    if (mode == 2) whole = sums(weight);
    all = sums(rest);
    if (!(all > 0.0)) {  // nothing is left: from the weights themselves
      mode = 0;
      all = sums(rest);
    }
    // ---- the first token whose inclusive sum is above u times the whole ----
    const double t = (double)a.uniform[s1 - 1] * all;
    double before;
    bool lasts;  // (u is 1, or no number: the last token with a weight)
    const int winner = first_above(lane < blocks ? total[parity ^ 1][lane] : 0.0, 0.0, t, &before, &lasts);
    write = block == winner && tid == 0;
    if (block == winner) {
      bool fallen;  // (sums of warps in another order than the blocks': the border is the block's end)
      const int w = first_above(lane < VT / 32 ? w_sum[lane] : 0.0, before, lasts ? INFINITY : t, &before, &fallen);
      // that warp's tokens, neighbours to each thread
      const int a0 = min(w * per, count), a1 = min(a0 + per, count), each = (a1 - a0 + VT - 1) / VT, j0 = min(a0 + tid * each, a1), j1 = min(j0 + each, a1);
      double s = 0.0;
      for (int j = j0; j < j1; ++j) s += rest(j);
      double inc = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      __syncthreads();
      if (lane == 31) w_sum[warp] = inc;
      __syncthreads();
      double lower = before;
      for (int i = 0; i < warp; ++i) lower += w_sum[i];
      lower += inc - s;
      // the first token above t, or the last one with a weight (1 more than it, 0 if there is none)
      uint32_t above = NONE, weighs = 0;
      double run = lower;
      for (int j = j0; j < j1; ++j) {
        const double x = rest(j);
        run += x;
        if (x > 0.0) weighs = (uint32_t)(lo + j) + 1u;
        if (x > 0.0 && !lasts && !fallen && above == NONE && run > t) above = (uint32_t)(lo + j);
      }
      above = __reduce_min_sync(0xffffffffu, above);
      weighs = __reduce_max_sync(0xffffffffu, weighs);
      if (lane == 0) {
        w_at[warp] = above;
        w_last[warp] = weighs;
      }
      __syncthreads();
      for (int i = 0; i < VT / 32; ++i) {
        above = min(above, w_at[i]);
        weighs = max(weighs, w_last[i]);
      }
      token = above != NONE ? above : weighs - 1u;
    }
  }
  if (write) {
    a.accepted[row] = (uint32_t)pos;
    a.next[row] = token;
    if (a.lens) a.lens_out[row] = (uint32_t)(a.lens[row] - (n - 1 - pos));
  }
}

// [M, V], the values of a place next to each other
int check_places(cg_ctx* c, const cg_tensor* t, const char* what, int64_t M, int64_t V) {
  const int64_t dims[2] = {M, V};
  CG_TRY(check_tensor(c, t, what, CG_F32, 2, dims, false));
  if (t->numel() && ((V > 1 && t->strides[1] != 1) || (t->dims[0] > 1 && t->strides[0] < V)))
    return fail(c, CG_ERR_UNSUPPORTED, std::string(what) + ": the last axis must be contiguous");
  return CG_OK;
}

template <typename T>
int launch(cg_ctx* c, VerifyArgs& a) {
  static PerDeviceFlag configured_on;
  bool& configured = configured_on.at(c->core->device);
  constexpr int64_t smem_most = 200 * 1024;
  if (!configured) {
    CG_CUDA(c, cudaFuncSetAttribute(k_verify_drafts<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_most));
    CG_CUDA(c, cudaFuncSetAttribute(k_verify_drafts<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    configured = true;
  }
  int blocks = MOST_BLOCKS;
  auto stride_of = [&](int b) { return ((a.V + b - 1) / b * (int64_t)sizeof(T) + 31) / 16 * 16; };
  while (blocks > 1 && a.rows * blocks > 2 * 148 && stride_of(blocks / 2) * 2 <= smem_most) blocks /= 2;
  a.slice = (int)((a.V + blocks - 1) / blocks);
  a.stride = (uint32_t)stride_of(blocks);
  a.ahead = (int)std::min<int64_t>(std::min<int64_t>(smem_most / a.stride, a.most), MOST_AHEAD);
  const size_t smem = (size_t)a.ahead * a.stride;
  CG_CUDA(c, launch_kernel(c, k_verify_drafts<T>, dim3((unsigned)blocks, (unsigned)a.rows), dim3(VT), smem, -blocks, a));
  CG_LAUNCHED(c);
  return CG_OK;
}

}  // namespace

}  // namespace cg

using namespace cg;

extern "C" int32_t cg_verify_drafts(cg_ctx* c, const cg_tensor* logits, const cg_tensor* probs, const cg_tensor* tokens, const cg_tensor* starts,
                                    const cg_tensor* uniform, const cg_tensor* temperature, const cg_tensor* lens, int64_t max_new, cg_tensor* accepted,
                                    cg_tensor* next, cg_tensor* lens_out) {
  if (!c) return CG_ERR_INVALID;
  CG_LAZY_EAGER_SCOPE(c);
  OnDevice on(c);
  if (!logits || !tokens || !starts || !uniform || !accepted || !next || !lens != !lens_out) return fail(c, CG_ERR_INVALID, "null argument");
  const int64_t any[2] = {-1, -1};
  CG_TRY(check_tensor(c, logits, "logits", CG_F32, 2, any, false));
  const int64_t M = logits->dims[0], V = logits->dims[1], m1[1] = {M};
  CG_TRY(check_places(c, logits, "logits", M, V));
  if (probs) CG_TRY(check_places(c, probs, "probs", M, V));
  CG_TRY(check_tensor(c, tokens, "tokens", CG_U32, 1, m1));
  CG_TRY(check_tensor(c, starts, "starts", CG_U32, 1, any));
  if (starts->dims[0] < 1) return fail(c, CG_ERR_SHAPE, "Shape mismatch in operation: starts");
  const int64_t rows = starts->dims[0] - 1, r0[1] = {rows};
  CG_TRY(check_tensor(c, uniform, "uniform", CG_F32, 1, m1));
  if (temperature) CG_TRY(check_tensor(c, temperature, "temperature", CG_F32, 1, r0));
  if (uniform->storage != ST_F32 || (temperature && temperature->storage != ST_F32)) return fail(c, CG_ERR_DTYPE, "random numbers and temperatures are f32");
  CG_TRY(check_tensor(c, accepted, "accepted", CG_U32, 1, r0));
  CG_TRY(check_tensor(c, next, "next", CG_U32, 1, r0));
  if (lens) {
    CG_TRY(check_tensor(c, lens, "lens", CG_U32, 1, r0));
    CG_TRY(check_tensor(c, lens_out, "lens_out", CG_U32, 1, r0));
  }
  if (rows > 65535) return fail(c, CG_ERR_UNSUPPORTED, "at most 65535 rows");
  if (M > 0x7FFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "too many tokens");
  if (V > 1 << 19) return fail(c, CG_ERR_UNSUPPORTED, "at most 2^19 tokens in the vocabulary");
  if (max_new < 0) return fail(c, CG_ERR_INVALID, "bad argument");
  const Extent x(lens), y(lens_out);
  const cg_tensor* lens_in = x.lo == y.lo && x.hi == y.hi ? nullptr : lens;  // (may be written over its own)
  if (overlap_any({logits, probs, tokens, starts, uniform, temperature, lens_in}, {accepted, next, lens_out}))
    return fail(c, CG_ERR_INVALID, "what is written overlaps an input or each other");
  if (rows == 0 || M == 0) return CG_OK;
  if (V == 0) return fail(c, CG_ERR_SHAPE, "no vocabulary");
  VerifyArgs a = {};
  a.logits = logits->data();
  a.probs = probs ? probs->data() : nullptr;
  a.l_ld = logits->strides[0];
  a.q_ld = probs ? probs->strides[0] : 0;
  a.probs16 = probs && probs->storage == ST_BF16;
  a.tokens = (const uint32_t*)tokens->data();
  a.starts = (const uint32_t*)starts->data();
  a.uniform = (const float*)uniform->data();
  a.temperature = temperature ? (const float*)temperature->data() : nullptr;
  a.lens = lens ? (const uint32_t*)lens->data() : nullptr;
  a.accepted = (uint32_t*)accepted->data();
  a.next = (uint32_t*)next->data();
  a.lens_out = lens_out ? (uint32_t*)lens_out->data() : nullptr;
  a.rows = rows;
  a.M = M;
  a.V = V;
  a.most = max_new > 0 ? std::min(max_new, M) : M;
  a.err = c->core->dev_err;
  written(accepted);
  written(next);
  if (lens_out) written(lens_out);
  return logits->storage == ST_BF16 ? launch<__nv_bfloat16>(c, a) : launch<float>(c, a);
}
