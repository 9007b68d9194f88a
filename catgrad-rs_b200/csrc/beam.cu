// beam.cu — one step of beam search: the best continuations over beams and vocabulary.
//
// For the beams j of a group with scores s_j (sums of log-probabilities) and logits x_j
//   total(j, v) = s_j + ((x_jv - M_j) - ln sum_u exp(x_ju - M_j)),  M_j = max_u x_ju,
// and the K largest are taken, equal ones in the order of j V + v.  A beam that is finished has one continuation,
// total(j, end) = s_j.  What has no number (NaN logits; all of a beam whose largest logit or own score is not finite)
// is -inf, as are masked logits.
//
// The logits are read once, 32 values a thread at a time, and stay in registers.  Within a beam totals are in the
// order of the logits, so a block keeps the K largest of each piece it reads: the K-th largest of 32 disjoint groups'
// maxima is no larger than the piece's K-th largest value, and the few values that reach it are ranked by counting.
// Where more reach it than the list holds (masked or level logits) the block takes K rounds of a block-wide
// maximum instead.  Exponentials are f32, their sums over more than a warp, the logarithm and the totals 64 bits: totals of
// different beams may lie close together.  A group is a thread-block cluster: its blocks share the vocabulary, each then
// finishes some of the beams from all blocks' lists, and the first one takes the K best of those.
#include <algorithm>

#include "mma.cuh"
#include "paged.h"

namespace cg {

namespace {

constexpr int BT = 256;            // threads
constexpr int PER = 32;            // values a thread holds
constexpr int PIECE = BT * PER;    // values of a piece
constexpr int LIST = 512;          // values that may reach the bound

struct SelectArgs {
  const void* logits;
  int64_t ld_b, ld_j;               // from one group and one beam to the next
  const float* scores;              // [B, J]
  const uint32_t* finished;         // [B, J] or null
  uint32_t end;
  int J, K, pieces;                 // pieces per block and beam
  int pool;                         // keys that the pool holds: LIST or all lists of a beam
  int64_t V, share;                 // share: values per block, a multiple of 16 bytes
  float* out_scores;                // [B, K]
  uint32_t *out_tokens, *out_parents, *out_finished;
};

// order-preserving: larger numbers have larger bits; the low word prefers lower indices
__device__ __forceinline__ uint32_t up(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float down(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)up(x) << 32 | (0xffffffffu - i); }
__device__ __forceinline__ uint64_t up64(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double down64(uint64_t u) { return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u)); }

__device__ __forceinline__ uint32_t remote_addr(const void* local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint64_t remote_ld64(uint32_t at) {
  uint64_t v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void remote_st64(uint32_t at, uint64_t v) { asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// number, -0 as 0, NaN as -inf
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.f : -INFINITY; }

template <typename T>
__device__ __forceinline__ void load_piece(const T* row, int64_t first, int64_t stop, float* x, int* valid) {
  // value i of vector w: place first + (w BT + tid) per + i
  constexpr int per = 16 / sizeof(T), vectors = PER / per;
  *valid = 0;
#pragma unroll
  for (int w = 0; w < vectors; ++w) {
    const int64_t at = first + (int64_t)(w * BT + (int)threadIdx.x) * per;
    const T* p = row + at;
    float* to = x + w * per;
    if (at + per <= stop && ((uintptr_t)p & 15) == 0) {
      const uint4 u = __ldg((const uint4*)p);
      const uint32_t b[4] = {u.x, u.y, u.z, u.w};
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = clean(__uint_as_float(b[i]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          to[2 * i] = clean(__uint_as_float(b[i] << 16));
          to[2 * i + 1] = clean(__uint_as_float(b[i] & 0xffff0000u));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < per; ++i) to[i] = at + i < stop ? clean((float)p[i]) : -INFINITY;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(BT) k_beam_select(SelectArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int per = 16 / sizeof(T);
  extern __shared__ uint64_t smem[];
  const int J = a.J, K = a.K, units = J * a.pieces;
  // every block's: the K largest keys, maximum and sum of each unit (beam, piece); the beams' scores and marks
  uint64_t* lists = smem;                       // [units][K]
  uint64_t* top = lists + units * K;            // first block: [J][K] totals of the beams' best
  uint64_t* place = top + J * K;                // first block: [J][K] j V + v
  double* sums = (double*)(place + J * K);      // [units]
  uint64_t* pool = (uint64_t*)(sums + units);   // [a.pool]
  float* tops = (float*)(pool + a.pool);        // [units]
  uint32_t* marks = (uint32_t*)(tops + units);  // [J]
  __shared__ float groups[32], bound_s, peak_s;
  __shared__ float part[BT / 32];
  __shared__ uint64_t best_s[BT / 32];
  __shared__ int count;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t rank, n_ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n_ranks));
  const int64_t b = blockIdx.y;
  const T* logits = (const T*)a.logits + b * a.ld_b;
  if (tid < J) marks[tid] = a.finished ? a.finished[b * J + tid] : 0;
  const int64_t lo = (int64_t)rank * a.share, hi = lo + a.share < a.V ? lo + a.share : a.V;

  for (int u = 0; u < units; ++u) {
    const int j = u / a.pieces;
    const T* row = logits + (int64_t)j * a.ld_j;
    const int64_t first = lo + (int64_t)(u - j * a.pieces) * PIECE, stop = first + PIECE < hi ? first + PIECE : hi;
    float x[PER];
    int valid;
    load_piece(row, first, stop, x, &valid);
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) mx = fmaxf(mx, x[i]);
    if (tid == 0) count = 0;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((lane & 7) == 0) groups[tid >> 3] = mx;
    __syncthreads();
    if (warp == 0) {
      const float g = groups[lane];
      float peak = g;
#pragma unroll
      for (int o = 16; o; o >>= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, o));
      int above = 0;  // groups before this one in the order of size, then number
#pragma unroll
      for (int o = 0; o < 32; ++o) {
        const float other = __shfl_sync(0xffffffffu, g, o);
        above += other > g || (other == g && o < lane);
      }
      if (above == K - 1) bound_s = g;
      if (lane == 0) peak_s = peak;
    }
    __syncthreads();
    const float bound = bound_s, peak = peak_s;
    const bool live = peak > -INFINITY && peak < INFINITY;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (live) sum += fast_exp2((x[i] - peak) * 1.4426950408889634f);
      const int64_t at = first + (int64_t)((i / per) * BT + tid) * per + i % per;
      if (x[i] >= bound && at < stop) {
        const int n = atomicAdd(&count, 1);
        if (n < LIST) pool[n] = key_of(x[i], (uint32_t)at);
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    const int n = count;
    if (tid == 0) {
      double s = 0.;
      for (int i = 0; i < BT / 32; ++i) s += (double)part[i];
      sums[u] = s;
      tops[u] = peak;
    }
    if (n <= LIST) {
      for (int i = tid; i < K; i += BT) if (i >= n) lists[u * K + i] = 0;
      for (int i = tid; i < n; i += BT) {
        const uint64_t key = pool[i];
        int above = 0;
        for (int o = 0; o < n; ++o) above += pool[o] > key;
        if (above < K) lists[u * K + above] = key;
      }
    } else {
      uint64_t last = ~0ull;
      for (int r = 0; r < K; ++r) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int64_t at = first + (int64_t)((i / per) * BT + tid) * per + i % per;
          const uint64_t key = at < stop ? key_of(x[i], (uint32_t)at) : 0;
          if (key < last && key > best) best = key;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
          best = other > best ? other : best;
        }
        if (lane == 0) best_s[warp] = best;
        __syncthreads();
        for (int w = 0; w < BT / 32; ++w) best = best_s[w] > best ? best_s[w] : best;
        if (tid == 0) lists[u * K + r] = best;
        last = best;
        __syncthreads();
      }
    }
    __syncthreads();
  }
  cluster_barrier();

  // this block's beams: the K largest of all blocks' lists, and their totals, into the first block
  const uint32_t top0 = remote_addr(top, 0), place0 = remote_addr(place, 0);
  for (int j = (int)rank; j < J; j += (int)n_ranks) {
    const int per_rank = a.pieces * K, n = (int)n_ranks * per_rank;
    uint64_t* all = pool;
    for (int i = tid; i < n; i += BT) all[i] = remote_ld64(remote_addr(lists + j * per_rank + i % per_rank, (uint32_t)(i / per_rank)));
    __shared__ double sum_s;
    __shared__ float max_s;
    if (warp == 0) {
      const int parts = (int)n_ranks * a.pieces;
      float m = -INFINITY;
      for (int i = lane; i < parts; i += 32) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote_addr(tops + j * a.pieces + i % a.pieces, (uint32_t)(i / a.pieces))) : "memory");
        m = fmaxf(m, v);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      double s = 0.;
      for (int i = lane; i < parts; i += 32) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote_addr(tops + j * a.pieces + i % a.pieces, (uint32_t)(i / a.pieces))) : "memory");
        const double part_sum = __longlong_as_double((long long)remote_ld64(remote_addr(sums + j * a.pieces + i % a.pieces, (uint32_t)(i / a.pieces))));
        if (part_sum > 0.) s += part_sum * exp((double)v - (double)m);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) { sum_s = s; max_s = m; }
    }
    __syncthreads();
    const double score = (double)a.scores[b * J + j], log_sum = log(sum_s);
    const float m = max_s;
    const bool dead = !(m > -INFINITY && m < INFINITY) || !(score > -INFINITY && score < INFINITY);
    const uint64_t j0 = (uint64_t)j * (uint64_t)a.V;
    if (dead || marks[j]) {
      // -inf all over, in the order of the vocabulary, behind the end token of a finished beam
      for (int i = tid; i < K; i += BT) {
        const bool ends = marks[j] && score > -INFINITY && score < INFINITY;
        uint64_t v = (uint64_t)i;
        double total = -INFINITY;
        if (ends) {
          v = i == 0 ? a.end : (uint64_t)(i - 1) + ((uint32_t)(i - 1) >= a.end ? 1u : 0u);
          if (i == 0) total = score;
        }
        remote_st64(top0 + (uint32_t)(j * K + i) * 8u, up64(total));
        remote_st64(place0 + (uint32_t)(j * K + i) * 8u, j0 + v);
      }
    } else {
      for (int i = tid; i < n; i += BT) {
        const uint64_t key = all[i];
        int above = 0;
        for (int o = 0; o < n; ++o) above += all[o] > key;
        if (above < K && key) {
          const float x = down((uint32_t)(key >> 32));
          const double total = score + (((double)x - (double)m) - log_sum);
          remote_st64(top0 + (uint32_t)(j * K + above) * 8u, up64(total));
          remote_st64(place0 + (uint32_t)(j * K + above) * 8u, j0 + (0xffffffffu - (uint32_t)key));
        }
      }
    }
    __syncthreads();
  }
  cluster_barrier();

  if (rank == 0) {
    for (int i = tid; i < J * K; i += BT) {
      const uint64_t t = top[i], p = place[i];
      int above = 0;
      for (int o = 0; o < J * K; ++o) above += top[o] > t || (top[o] == t && place[o] < p);
      if (above < K) {
        const uint32_t parent = (uint32_t)(p / (uint64_t)a.V), token = (uint32_t)(p - parent * (uint64_t)a.V);
        const int64_t at = b * K + above;
        a.out_scores[at] = (float)down64(t);
        a.out_tokens[at] = token;
        a.out_parents[at] = parent;
        a.out_finished[at] = marks[parent] || token == a.end;
      }
    }
  }
}

size_t select_smem(const SelectArgs& a) {
  const size_t units = (size_t)a.J * a.pieces;
  return (units * a.K + 2 * (size_t)a.J * a.K + units + a.pool) * 8 + units * 4 + (size_t)a.J * 4;
}

template <typename T>
int launch_select(cg_ctx* c, SelectArgs a, int64_t B) {
  // blocks of a group: enough that each has about one piece of a beam, at most 8
  int ranks = 1;
  while (ranks < 8 && (int64_t)ranks * PIECE < a.V) ranks *= 2;
  constexpr int64_t per = 16 / sizeof(T);
  a.share = ((a.V + ranks - 1) / ranks + per - 1) / per * per;
  a.pieces = (int)((a.share + PIECE - 1) / PIECE);
  if (a.pieces > 64) return fail(c, CG_ERR_UNSUPPORTED, "vocabulary too large");
  a.pool = std::max(LIST, ranks * a.pieces * a.K);
  const size_t smem = select_smem(a);
  if (smem > 200 * 1024) return fail(c, CG_ERR_UNSUPPORTED, "beams times vocabulary too large");
  static PerDeviceFlag configured_on;
  bool& configured = configured_on.at(c->core->device);
  if (!configured) {
    CG_CUDA(c, cudaFuncSetAttribute(k_beam_select<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    configured = true;
  }
  CG_CUDA(c, launch_kernel(c, k_beam_select<T>, dim3((unsigned)ranks, (unsigned)B), dim3(BT), smem, -ranks, a));
  CG_LAUNCHED(c);
  return CG_OK;
}

}  // namespace

}  // namespace cg

using namespace cg;

extern "C" int32_t cg_beam_select(cg_ctx* c, const cg_tensor* logits, const cg_tensor* scores, const cg_tensor* finished, uint32_t end,
                                  cg_tensor* scores_out, cg_tensor* tokens_out, cg_tensor* parents_out, cg_tensor* finished_out) {
  if (!c) return CG_ERR_INVALID;
  CG_LAZY_EAGER_SCOPE(c);
  OnDevice on(c);
  if (!logits || !scores || !scores_out || !tokens_out || !parents_out || !finished_out) return fail(c, CG_ERR_INVALID, "null argument");
  const int64_t any[3] = {-1, -1, -1};
  CG_TRY(check_tensor(c, logits, "logits", CG_F32, 3, any, false));
  const int64_t B = logits->dims[0], J = logits->dims[1], V = logits->dims[2];
  CG_TRY(check_tensor(c, scores, "scores", CG_F32, 2, logits->dims));
  if (finished) CG_TRY(check_tensor(c, finished, "finished", CG_U32, 2, logits->dims));
  const int64_t to[2] = {B, -1};
  CG_TRY(check_tensor(c, scores_out, "scores_out", CG_F32, 2, to));
  const int64_t K = scores_out->dims[1];
  for (const cg_tensor* o : {tokens_out, parents_out, finished_out}) CG_TRY(check_tensor(c, o, "an output", CG_U32, 2, scores_out->dims));
  if (scores->storage != ST_F32 || scores_out->storage != ST_F32) return fail(c, CG_ERR_DTYPE, "scores are f32");
  if (B > 0 && V > 1 && logits->strides[2] != 1) return fail(c, CG_ERR_UNSUPPORTED, "logits: the last axis must be contiguous");
  if (J > 32 || K > 32) return fail(c, CG_ERR_UNSUPPORTED, "at most 32 beams");
  if (B > 65535) return fail(c, CG_ERR_UNSUPPORTED, "at most 65535 groups");
  if (K > V) return fail(c, CG_ERR_SHAPE, "more beams than the vocabulary has");
  if (V > 0x7FFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "vocabulary too large");
  if (finished && (int64_t)end >= V) return fail(c, CG_ERR_INVALID, "the end token is not in the vocabulary");
  // the scores and marks of a group are read before its new ones are written, so they may take their place
  const cg_tensor* outs[4] = {scores_out, tokens_out, parents_out, finished_out};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j])) return fail(c, CG_ERR_INVALID, "outputs overlap");
    const bool whole = K == J;
    const bool bad = overlap(outs[i], logits) || (overlap(outs[i], scores) && !(whole && i == 0 && scores_out->data() == scores->data())) ||
                     (finished && overlap(outs[i], finished) && !(whole && i == 3 && finished_out->data() == finished->data()));
    if (bad) return fail(c, CG_ERR_INVALID, "an output overlaps an input");
  }
  if (B == 0 || K == 0) return CG_OK;
  if (J == 0) return fail(c, CG_ERR_SHAPE, "no beams");
  SelectArgs a = {};
  a.logits = logits->data();
  a.ld_b = logits->strides[0]; a.ld_j = logits->strides[1];
  a.scores = (const float*)scores->data();
  a.finished = finished ? (const uint32_t*)finished->data() : nullptr;
  a.end = end;
  a.J = (int)J; a.K = (int)K; a.V = V;
  a.out_scores = (float*)scores_out->data();
  a.out_tokens = (uint32_t*)tokens_out->data();
  a.out_parents = (uint32_t*)parents_out->data();
  a.out_finished = (uint32_t*)finished_out->data();
  for (cg_tensor* t : {scores_out, tokens_out, parents_out, finished_out}) written(t);
  return logits->storage == ST_BF16 ? launch_select<__nv_bfloat16>(c, a, B) : launch_select<float>(c, a, B);
}
