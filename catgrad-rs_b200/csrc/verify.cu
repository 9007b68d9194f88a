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
// A cluster has a row, its blocks equal slices of the vocabulary.  Positions are judged a few at a time, and none behind the first rejected draft but those of its
// group; the draw reads the slice again, out of L2, in one pass for the sum of the weights and for what q leaves of them.
//
// Bytes do not bound it (40 rows of up to 4 drafts over 151936 tokens, bf16: 41 MB in 42 us, 0.15 of the copy rate) but a row's chain: a round of positions is loads,
// maxima and sums, the cluster's barrier, the verdict, 3 to 5 us; the draw's 64-bit exponentials 9 us at full rate, its sums and the search for the token
// 4 to 7.  Rows of several rounds go on when the others' SMs are idle: an SM has work for 0.69 of the time, the busiest issues 1.66 times the mean.  One row of 4 drafts over
// 128256, f32: 14 us; 32 rows of 7 over 256000 45.5; greedy, 16 rows of 3 over 50257, f32: 7.4.  Rows of one token, which draw from their logits: 64 over 128256, bf16, 26.6 us,
// one in f32 9.4.
#include <algorithm>
#include <type_traits>

#include "mma.cuh"
#include "paged.h"
#include "tc_common.cuh"

namespace cg {

namespace {

using namespace tc;

constexpr int MOST_BLOCKS = 16;  // of a cluster
constexpr int MOST_AHEAD = 8;    // positions judged at a time
constexpr uint32_t NONE = 0xFFFFFFFFu;
constexpr float NO_LOGIT = -INFINITY;

struct VerifyArgs {
  const void *logits, *probs;  // probs may be null: a draft is its drafter's only token
  int64_t l_ld, q_ld;          // from one place to the next
  const uint32_t *tokens, *starts, *lens;  // lens may be null
  const float *uniform, *temperature;      // temperature may be null: 1
  uint32_t *accepted, *next, *lens_out;
  int64_t rows, M, most;
  int V;
  int slice;                   // tokens of a block
  int ahead;                   // positions judged at a time
  int probs16;
  int staged;                  // the drafter's probabilities that are drawn from go through shared memory
  int32_t* err;
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
// Word i of a vector, and value i of it as it is stored (i is known when compiling)
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
template <typename T>
__device__ __forceinline__ float value_of(const uint4& v, int i) {
  if (sizeof(T) == 4) return __uint_as_float(word_of(v, i));
  return __uint_as_float(i & 1 ? word_of(v, i / 2) & 0xffff0000u : word_of(v, i / 2) << 16);
}
// (NaN counts as -inf)
template <typename T>
__device__ __forceinline__ float logit(T x) { return fmaxf(widen(x), NO_LOGIT); }

// e^x for x <= 0 by Tang's method (1989), to 2^-49 down to e^-30 and 2^-45 down to e^-700 (ln2 / 16 is off by 2^-59, the whole numbers by which it is taken go up to 16158): x = (16 m + j) ln2 / 16 + r, 2^(j/16) from a table (whose 16 values lie in different
// banks), e^r by its series: 12 operations in 64 bits, where exp() takes twice as many, and no branch, so that several are under way.
// Below e^-700 it is 0.
__device__ __forceinline__ double exp64(double x, const double* power) {
  const double magic = 6755399441055744.0;  // 1.5 2^52: sums with it are rounded to whole numbers
  const double t = fma(x, 23.083120654223414, magic), r = fma(t - magic, -0.04332169878499658, x);
  const int k = __double2loint(t);
  double p = fma(r, 1.0 / 720.0, 1.0 / 120.0);
  p = fma(r, p, 1.0 / 24.0);
  p = fma(r, p, 1.0 / 6.0);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0) * power[k & 15];
  return x < -700.0 ? 0.0 : __hiloint2double(__double2hiint(p) + ((k >> 4) << 20), __double2loint(p));
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
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
// A slice of `count` values from `src` on: `head` up to a 16-byte boundary, whole vectors, the rest.  The ends are one more value of the first threads.
template <typename T>
struct Slice {
  static constexpr int E = 16 / sizeof(T);
  const T* src;
  int head, vectors, tail;
  __device__ __forceinline__ Slice(const T* s, int count) : src(s) {
    head = min((E - (int)(((uintptr_t)s & 15) / sizeof(T))) % E, count);
    vectors = (count - head) / E;
    tail = count - head - vectors * E;
  }
  __device__ __forceinline__ int end_of(int tid) const { return tid < head ? tid : tid >= E && tid < E + tail ? head + vectors * E + tid - E : -1; }
};

// VT: threads.  Of a position a thread has every VT-th vector, U a step; the next step's are on their way while these are judged.
template <typename T, int VT, int ON_SM>
__global__ void __launch_bounds__(VT, ON_SM) k_verify_drafts(VerifyArgs a) {
  constexpr int E = 16 / sizeof(T), W = VT / 32, U = 16 / E;  // values of a vector, warps, vectors of a step
  constexpr int SUB = 32 / W;                            // parts of a warp's tokens, of which there are sums
  extern __shared__ __align__(16) uint8_t staging[];  // the drafter's probabilities at a position
  __shared__ double power[16];
  __shared__ double w_sum[MOST_AHEAD][W];
  __shared__ float w_top[MOST_AHEAD][W];
  __shared__ uint32_t w_at[MOST_AHEAD][W];
  // what the blocks tell each other of positions (two buffers, which take turns), and of what is drawn from
  __shared__ double told_sum[2][MOST_AHEAD][MOST_BLOCKS], told_rest[4][MOST_BLOCKS];
  __shared__ uint32_t told_top[2][MOST_AHEAD][MOST_BLOCKS], told_at[2][MOST_AHEAD][MOST_BLOCKS];
  __shared__ double pos_sum[MOST_AHEAD];
  __shared__ float pos_top[MOST_AHEAD];
  __shared__ uint32_t pos_at[MOST_AHEAD];
  __shared__ int pos_ends[MOST_AHEAD];
  __shared__ double r_sum[3][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int blocks = (int)gridDim.x, block = (int)blockIdx.x;
  const int64_t row = blockIdx.y;
  if (tid < 16) power[tid] = exp2(tid / 16.0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // (the same in all blocks of a cluster, as everything that decides which way they go)
  const uint32_t s0 = a.starts[row], s1 = a.starts[row + 1];
  const float heat_in = a.temperature ? a.temperature[row] : 1.f;
  const uint32_t len = a.lens ? a.lens[row] : 0xFFFFFFFFu;
  if (s0 == s1) return;
  const int n = (int)(s1 - s0);  // (places are 31 bits)
  if (!(s0 < s1 && s1 <= a.M && n <= a.most && len >= (uint32_t)n - 1u)) {
    if (tid == 0) *a.err = DEV_INDEX;
    return;
  }
  // (nothing is put into another block's memory before it runs: waited for ahead of the first put)
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int lo = std::min(block * a.slice, a.V), count = std::min(lo + a.slice, a.V) - lo;
  auto place = [&](int pos) { return (const T*)a.logits + (int64_t)(s0 + pos) * a.l_ld + lo; };
  // A position's slice as this thread reads it: U of its vectors at a time, VT apart, and its value of the ends.
  struct Cursor {
    const uint4* at;  // the next vector
    int left;         // vectors from that on, those of other threads among them
    uint4 x[U];       // on their way
    T end;
  };
  auto load = [&](Cursor& c) {
    if ((U - 1) * VT < c.left) {
#pragma unroll
      for (int i = 0; i < U; ++i) c.x[i] = __ldg(c.at + i * VT);
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        constexpr uint32_t none = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;  // (-inf)
        c.x[i] = make_uint4(none, none, none, none);
        if (i * VT < c.left) c.x[i] = __ldg(c.at + i * VT);
      }
    }
    c.at += U * VT;
    c.left -= U * VT;
  };
  auto begin = [&](Cursor& c, int pos) {
    const Slice<T> f(place(pos), count);
    c.at = (const uint4*)(f.src + f.head) + tid;
    c.left = f.vectors - tid;
    load(c);
    const int e = f.end_of(tid);
    c.end = e >= 0 ? f.src[e] : (T)NO_LOGIT;
  };
  int first = 0, parity = 0, group = std::min(a.ahead, n), stop = -1;  // first: of the positions judged at a time
  Cursor ahead;
  begin(ahead, 0);

  bool bad = false;
  for (int i = 1 + tid; i < n; i += VT) bad = bad || a.tokens[s0 + i] >= (uint32_t)a.V;
  const float u_next = a.uniform[s1 - 1];
  const bool greedy = !(heat_in > 0.f);
  // (temperatures beyond 2^+-100 act as these)
  const float heat = fminf(fmaxf(heat_in, 0x1p-100f), 0x1p100f), unit = 1.4426950408889634f / heat;
  const double cold = 1.0 / (double)heat;
  if (__syncthreads_or(bad)) {
    if (tid == 0) *a.err = DEV_INDEX;
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    return;
  }
  for (;;) {
    // what the drafts are judged by, a warp each (used behind the sums)
    struct Judged {
      uint32_t draft, q;  // (q as it is stored)
      float u;
      T logit;
    };
    auto judge = [&](int j) {
      Judged x = {NONE, 0, 0.f, (T)NO_LOGIT};
      if (j >= group || first + j >= n - 1) return x;
      const int64_t m = (int64_t)s0 + first + j;
      x.draft = a.tokens[m + 1];
      x.u = a.uniform[m];
      x.logit = ((const T*)a.logits)[m * a.l_ld + x.draft];
      if (a.probs) x.q = a.probs16 ? (uint32_t)((const uint16_t*)a.probs)[m * a.q_ld + x.draft] << 16 : ((const uint32_t*)a.probs)[m * a.q_ld + x.draft];
      else x.q = 0x3F800000u;
      return x;
    };
    const Judged mine = judge(warp);
    for (int j = 0; j < group; ++j) {
      float top = NO_LOGIT, sum = 0.f, end = logit(ahead.end);  // (the ends count once)
      uint32_t at = NONE;
      for (int step = 0;; ++step) {
        uint4 now[U];
#pragma unroll
        for (int i = 0; i < U; ++i) now[i] = ahead.x[i];
        auto value = [&](int i) { return value_of<T>(now[i / E], i % E); };  // (unpacked where it is used, which keeps registers)
        const bool more_steps = ahead.left > 0;
        if (more_steps) load(ahead);
        else if (first + j + 1 < n) begin(ahead, first + j + 1);
        float t[4] = {end, NO_LOGIT, NO_LOGIT, NO_LOGIT};
        if constexpr (sizeof(T) == 2) {  // (two values at a time)
          uint32_t m[2] = {0xFF80FF80u, 0xFF80FF80u};
#pragma unroll
          for (int i = 0; i < U * E / 2; ++i) asm("max.bf16x2 %0, %0, %1;" : "+r"(m[i & 1]) : "r"(word_of(now[i / 4], i % 4)));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            t[2 * i] = fmaxf(t[2 * i], __uint_as_float(m[i] << 16));
            t[2 * i + 1] = fmaxf(t[2 * i + 1], __uint_as_float(m[i] & 0xffff0000u));
          }
        } else {
#pragma unroll
          for (int i = 0; i < U * E; ++i) t[i & 3] = fmaxf(t[i & 3], value(i));
        }
        t[0] = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        if (greedy) {
          // (a thread's places ascend from step to step, but for the ends: before all others or behind them)
          if (t[0] > NO_LOGIT && t[0] >= top) {
            const Slice<T> f(place(first + j), count);
            if (t[0] > top) at = NONE;
            top = t[0];
            if (end == top) at = min(at, (uint32_t)(lo + f.end_of(tid)));
#pragma unroll
            for (int i = 0; i < U * E; ++i)
              if (value(i) == top) at = min(at, (uint32_t)(lo + f.head + (tid + (step * U + i / E) * VT) * E + i % E));
          }
        } else {
          if (t[0] > top) {
            sum *= fast_exp2((top - t[0]) * unit);
            top = t[0];
          }
          if (top > NO_LOGIT) {
            float s[4] = {fast_exp2((end - top) * unit), 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < U * E; ++i) s[i & 3] += fast_exp2((value(i) - top) * unit);
            float more = (s[0] + s[1]) + (s[2] + s[3]);
            if (more != more) {  // (some are no numbers)
              more = fast_exp2((end - top) * unit);
#pragma unroll
              for (int i = 0; i < U * E; ++i) more += value(i) == value(i) ? fast_exp2((value(i) - top) * unit) : 0.f;
            }
            sum += more;
          }
        }
        end = NO_LOGIT;
        if (!more_steps) break;
      }
      const float t = warp_max(top);
      if (greedy) {
        at = __reduce_min_sync(0xffffffffu, top == t ? at : NONE);
      } else {
        sum = top > NO_LOGIT ? sum * fast_exp2((top - t) * unit) : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      }
      if (lane == 0) {
        w_top[j][warp] = t;
        w_sum[j][warp] = (double)sum;
        w_at[j][warp] = at;
      }
    }
    __syncthreads();
    if (first == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (warp < group) {
      const bool there = lane < W;
      const float wt = there ? w_top[warp][lane] : NO_LOGIT, bt = warp_max(wt);
      const double ws = greedy ? 0.0 : warp_sum(there && wt > NO_LOGIT ? w_sum[warp][lane] * (double)fast_exp2((wt - bt) * unit) : 0.0);
      const uint32_t wi = __reduce_min_sync(0xffffffffu, there && wt == bt ? w_at[warp][lane] : NONE);
      if (lane < blocks) {
        put_remote(&told_sum[parity][warp][block], (uint32_t)lane, ws);
        put_remote(&told_top[parity][warp][block], (uint32_t)lane, __float_as_uint(bt));
        put_remote(&told_at[parity][warp][block], (uint32_t)lane, wi);
      }
    }
    cluster_sync_all();
    // ---- the verdicts, in every block alike ----
    if (warp < group) {
      const float q = __uint_as_float(mine.q);
      const bool there = lane < blocks;
      const float t = there ? __uint_as_float(told_top[parity][warp][lane]) : NO_LOGIT, top = warp_max(t);
      const bool some = top > NO_LOGIT && top < INFINITY;  // (else nothing has a probability)
      const double sum = greedy ? 0.0 : warp_sum(there && t > NO_LOGIT ? told_sum[parity][warp][lane] * (double)fast_exp2((t - top) * unit) : 0.0);
      const uint32_t at = __reduce_min_sync(0xffffffffu, there && t == top ? told_at[parity][warp][lane] : NONE);
      bool ends = first + warp == n - 1;
      if (!ends) {
        const bool stands = greedy ? mine.draft == at
                                   : (double)mine.u * (double)(q > 0.f ? q : 0.f) * sum < exp64(((double)logit(mine.logit) - (double)top) * cold, power);
        ends = !(some && stands);
      }
      if (lane == 0) {
        pos_top[warp] = top;
        pos_sum[warp] = sum;
        pos_at[warp] = at;
        pos_ends[warp] = ends;
      }
    }
    parity ^= 1;
    __syncthreads();
    const uint32_t which = __ballot_sync(0xffffffffu, lane < group && pos_ends[lane]);
    if (which) {
      stop = __ffs(which) - 1;
      break;
    }
    first += group;
    group = std::min(a.ahead, n - first);
  }

  // ---- the next token, at position first + stop ----
  const int pos = first + stop;
  const int64_t m = (int64_t)s0 + pos;
  const float top = pos_top[stop];
  uint32_t token = NONE;
  bool write = block == 0 && tid == 0;
  if (!(top > NO_LOGIT && top < INFINITY)) {
    token = NONE;
  } else if (greedy) {
    token = pos_at[stop];
  } else {
    const T* values = place(pos);
    int mode = pos < n - 1 ? (a.probs ? 2 : 1) : 0;  // what is drawn from: 0 weights e, 1 weights but the draft's, 2 what q leaves of them, max(e - q sum e, 0)
    const __nv_bfloat16* q16 = (const __nv_bfloat16*)a.probs + m * a.q_ld + lo;
    const float* q32 = (const float*)a.probs + m * a.q_ld + lo;
    const double t64 = (double)top;
    // 32 parts of neighbouring tokens, of which a warp has SUB
    const int unit = count >= 4096 ? 127 : 31, per = ((count + 31) / 32 + unit) & ~unit;  // (whole batches, of long slices)
    auto part_begin = [&](int i) { return min(i * per, count); };
    const uint32_t draft = pos < n - 1 ? a.tokens[m + 1] : NONE;
    auto weigh = [&](float x) { return exp64(((double)x - t64) * cold, power); };
    auto drafter = [&](int j) {
      const float q = a.probs16 ? __bfloat162float(q16[j]) : q32[j];
      return q > 0.f ? q : 0.f;
    };
    // One pass for the sum of e, and for what is left once that is known: of the tokens with e > q s, where s is the sum that drafts were judged by,
    // the sums of e and of q.  (Tokens on the wrong side of that border, 2^-20 of themselves from it, would add as little.)  Where less than 2^-10 of the whole is left
    // that is too much, as of a drafter that agrees with the target to the last bits, and what is left is summed by itself: 7 us for so rare a row.
    const double s = mode == 2 ? pos_sum[stop] : 0.0;
    auto sums = [&](auto probs) {  // (probs: of which type, or none)
      typedef decltype(probs) Q;
      constexpr bool HAS = !std::is_same<Q, char>::value;
      constexpr int B = 4;  // logits of a thread at a time; the next ones are on their way
      const int w0 = part_begin(warp * SUB), w1 = part_begin(warp * SUB + SUB);  // this warp's tokens
      const Q* q_at = (const Q*)a.probs + m * a.q_ld + lo;
      if constexpr (HAS) {
        if (a.staged) {
          // this warp's probabilities, whole vectors as they lie (before the row is the one before it, but in front of all)
          constexpr int QE = 16 / sizeof(Q);
          const int phase = (int)(((uintptr_t)(q_at + w0) & 15) / sizeof(Q));
          uint8_t* to = staging + ((size_t)w0 * sizeof(Q) + 15) / 16 * 16 + warp * 16;
          for (int v = lane; w0 < w1 && v * QE < phase + w1 - w0; v += 32) {
            const int j0 = v * QE - phase;
            if (j0 < 0 && m == 0 && lo + w0 == 0) {
              for (int e = phase; e < QE; ++e)
                if (e - phase < w1) ((Q*)to)[e] = q_at[e - phase];
            } else {
              cp_async16(smem_u32(to + v * 16), q_at + w0 + j0, std::min(QE, a.V - lo - w0 - j0) * (int)sizeof(Q));
            }
          }
          cp_async_commit();
          q_at = (const Q*)to + phase - w0;
        }
      }
      T x[B];
      auto load = [&](int b) {
        if (b + 32 * B <= w1) {
#pragma unroll
          for (int i = 0; i < B; ++i) x[i] = values[b + lane + 32 * i];
        }
      };
      int have = w0;  // x are the logits from here on
      load(w0);
      if (HAS && a.staged) {
        cp_async_wait_group<0>();
        __syncwarp();
      }
      for (int k = warp * SUB; k < warp * SUB + SUB; ++k) {
        double e_all = 0.0, e_left = 0.0, q_left = 0.0;
        auto add = [&](float y, float q) {
          const double e = weigh(y);
          e_all += e;
          if constexpr (HAS) {
            const double p = (double)(q > 0.f ? q : 0.f);
            if (e > p * s) {
              e_left += e;
              q_left += p;
            }
          }
        };
        const int v0 = part_begin(k), v1 = part_begin(k + 1);
        int b = v0;
        if (have != b) load(b);
        while (b + 32 * B <= v1) {
          float y[B], q[B];
#pragma unroll
          for (int i = 0; i < B; ++i) {
            y[i] = logit(x[i]);
            q[i] = 0.f;
            if constexpr (HAS) q[i] = widen(q_at[b + lane + 32 * i]);
          }
          b += 32 * B;
          load(b);
#pragma unroll
          for (int i = 0; i < B; ++i) add(y[i], q[i]);
        }
        have = b;
        for (; b < v1; b += 32) {
          const int j = b + lane;
          float q = 0.f;
          if constexpr (HAS) q = j < v1 ? widen(q_at[j]) : 0.f;
          add(j < v1 ? logit(values[j]) : NO_LOGIT, q);
        }
        e_all = warp_sum(e_all);
        if (HAS) {
          e_left = warp_sum(e_left);
          q_left = warp_sum(q_left);
        } else if (mode == 1) {
          const int d = (int)draft - lo;
          e_left = e_all - (d >= v0 && d < v1 ? weigh(logit(values[d])) : 0.0);
        }
        if (lane == 0) {
          r_sum[0][k] = e_all;
          r_sum[1][k] = e_left;
          r_sum[2][k] = q_left;
        }
      }
    };
    if (mode != 2) sums((char)0);
    else if (a.probs16) sums(__nv_bfloat16());
    else sums(0.f);
    __syncthreads();
    if (warp < 3) {
      const double b = warp_sum(r_sum[warp][lane]);
      if (lane < blocks) put_remote(&told_rest[warp][block], (uint32_t)lane, b);
    }
    cluster_sync_all();
    const double b_e = lane < blocks ? told_rest[0][lane] : 0.0, b_left = lane < blocks ? told_rest[1][lane] : 0.0, b_q = lane < blocks ? told_rest[2][lane] : 0.0;
    const double whole = mode == 2 ? warp_sum(b_e) : 0.0;
    double part = mode == 0 ? b_e : mode == 1 ? b_left : fmax(b_left - b_q * whole, 0.0), all = warp_sum(part);
    auto rest = [&](int j) {
      const double e = weigh(logit(values[j]));
      if (mode == 0) return e;
      if (mode == 1) return (uint32_t)(lo + j) == draft ? 0.0 : e;
      return fmax(e - (double)drafter(j) * whole, 0.0);
    };
    if (mode == 2 && all < 0x1p-10 * whole) {  // (the same in all blocks)
#pragma unroll 1
      for (int k = warp * SUB; k < warp * SUB + SUB; ++k) {
        double left = 0.0;
#pragma unroll 1
        for (int j = part_begin(k) + lane; j < part_begin(k + 1); j += 32) left += rest(j);
        left = warp_sum(left);
        if (lane == 0) {
          r_sum[1][k] = left;
          r_sum[2][k] = 0.0;
        }
      }
      __syncthreads();
      if (warp == 0) {
        const double b = warp_sum(r_sum[1][lane]);
        if (lane < blocks) put_remote(&told_rest[3][block], (uint32_t)lane, b);
      }
      cluster_sync_all();
      part = lane < blocks ? told_rest[3][lane] : 0.0;
      all = warp_sum(part);
    }
    if (!(all > 0.0)) {  // nothing is left: from the weights themselves
      mode = 0;
      part = b_e;
      all = warp_sum(part);
    }
    // ---- the first token whose inclusive sum is above u times the whole ----
    const double t = (double)u_next * all;
    double before;
    bool lasts;  // (u is 1, or no number: the last token with a weight)
    const int winner = first_above(part, 0.0, t, &before, &lasts);
    write = block == winner && tid == 0;
    if (block == winner) {
      bool fallen;  // (sums of parts in another order than the blocks': the border is the block's end)
      const double mine = mode == 0 ? r_sum[0][lane] : mode == 1 ? r_sum[1][lane] : fmax(r_sum[1][lane] - r_sum[2][lane] * whole, 0.0);
      const int w = first_above(mine, before, lasts ? INFINITY : t, &before, &fallen);
      // that part's tokens, neighbours to each thread
      constexpr int KEPT = 4;  // (what they add, as far as it is kept)
      const int a0 = part_begin(w), a1 = part_begin(w + 1), each = (a1 - a0 + VT - 1) / VT, j0 = min(a0 + tid * each, a1), j1 = min(j0 + each, a1);
      double kept[KEPT], s = 0.0;
#pragma unroll
      for (int i = 0; i < KEPT; ++i) {
        kept[i] = j0 + i < j1 ? rest(j0 + i) : 0.0;
        s += kept[i];
      }
      for (int j = j0 + KEPT; j < j1; ++j) s += rest(j);
      double inc = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      if (lane == 31) w_sum[0][warp] = inc;
      __syncthreads();
      double run = before + warp_sum(lane < warp ? w_sum[0][lane] : 0.0) + (inc - s);
      // the first token above t, or the last one with a weight (1 more than it, 0 if there is none)
      uint32_t above = NONE, weighs = 0;
      auto look = [&](int j, double x) {
        run += x;
        if (x > 0.0) weighs = (uint32_t)(lo + j) + 1u;
        if (x > 0.0 && !lasts && !fallen && above == NONE && run > t) above = (uint32_t)(lo + j);
      };
#pragma unroll
      for (int i = 0; i < KEPT; ++i) look(j0 + i, kept[i]);
      for (int j = j0 + KEPT; j < j1; ++j) look(j, rest(j));
      above = __reduce_min_sync(0xffffffffu, above);
      weighs = __reduce_max_sync(0xffffffffu, weighs);
      if (lane == 0) {
        w_at[0][warp] = above;
        w_at[1][warp] = weighs;
      }
      __syncthreads();
      above = __reduce_min_sync(0xffffffffu, lane < W ? w_at[0][lane] : NONE);
      weighs = __reduce_max_sync(0xffffffffu, lane < W ? w_at[1][lane] : 0u);
      token = above != NONE ? above : weighs - 1u;
    }
  }
  if (write) {
    a.accepted[row] = (uint32_t)pos;
    a.next[row] = token;
    if (a.lens) a.lens_out[row] = len - (uint32_t)(n - 1 - pos);
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

template <typename T, int VT, int ON_SM>
int launch_threads(cg_ctx* c, VerifyArgs& a, int blocks) {
  constexpr int smem_most = 210 * 1024 / ON_SM;
  static PerDeviceFlag configured_on;
  bool& configured = configured_on.at(c->core->device);
  if (!configured) {
    CG_CUDA(c, cudaFuncSetAttribute(k_verify_drafts<T, VT, ON_SM>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_most));
    CG_CUDA(c, cudaFuncSetAttribute(k_verify_drafts<T, VT, ON_SM>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    configured = true;
  }
  a.slice = (int)((a.V + blocks - 1) / blocks);
  // Positions judged at a time: two, where bytes count, so that few behind a rejected draft are read; of short ones all, for fewer rounds of
  // sums and verdicts.  (Us with 2 / 8: 32 rows of 7 drafts x 256000, bf16, 39.7  52.8, 40 of 4 x 151936 42.2  43.4; 16 of 3 x 50257, f32, greedy 8.3  7.4, 4 of 4 x 128256, bf16, 15.4  13.4.)
  a.ahead = a.rows * a.V * (int64_t)sizeof(T) > 8 << 20 ? 2 : MOST_AHEAD;
  const int64_t staging = a.probs ? (int64_t)a.slice * (a.probs16 ? 2 : 4) + 32 * (VT / 32 + 1) : 0;
  a.staged = staging > 0 && staging <= smem_most;
  const size_t smem = a.staged ? (size_t)staging : 0;
  CG_CUDA(c, launch_kernel(c, k_verify_drafts<T, VT, ON_SM>, dim3((unsigned)blocks, (unsigned)a.rows), dim3(VT), smem, -blocks, a));
  CG_LAUNCHED(c);
  return CG_OK;
}
template <typename T>
int launch(cg_ctx* c, VerifyArgs& a) {
  // Blocks of a row, and their threads and how many run on an SM (those of 512, 2 have 64 registers and spill 60 to 170 bytes, of 256, 3 some 80 and 0 to 16), us, [the rule's]:
  //                                                 16 x 512, 1   8 x 512, 2   8 x 256, 2   8 x 256, 3   4 x 256, 2
  //   1 row x 128256, f32, 4 drafts                 [14.1]        20           24           24           41
  //   16 x 50257, f32, 3, greedy                     16           10.0         [7.5]        8.1          10
  //   25 x 54301, f32, 4                             45           24           [22.0]       25.7         30
  //   32 x 256000, bf16, 7, no probabilities         86           [45.6]       59           59           77
  //   40 x 151936, bf16, 4                           84           54           53           [42.9]       59
  //   38 x 2736, f32, 3                              46           23           13.6         13.6         [11.5]
  // More threads for a row hide the draw's 64-bit chains, more registers let more of them be under way; more blocks than run at a time wait for whole clusters to
  // end.
  int blocks = a.V >= 65536 && a.rows * MOST_BLOCKS <= 148 ? MOST_BLOCKS : 8;
  while (blocks > 1 && (a.rows * blocks > 3 * 148 || a.V < 512 * blocks)) blocks /= 2;
  const int64_t all = a.rows * blocks;
  if (all <= 74 && a.V >= 2048 * blocks) return launch_threads<T, 512, 1>(c, a, blocks);
  if (all > 148 && all <= 2 * 148 && a.V >= 16384 * blocks) return launch_threads<T, 512, 2>(c, a, blocks);
  if (all <= 2 * 148) return launch_threads<T, 256, 2>(c, a, blocks);
  return launch_threads<T, 256, 3>(c, a, blocks);
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
  a.V = (int)V;
  a.most = max_new > 0 ? std::min(max_new, M) : M;
  a.err = c->core->dev_err;
  written(accepted);
  written(next);
  if (lens_out) written(lens_out);
  return logits->storage == ST_BF16 ? launch<__nv_bfloat16>(c, a) : launch<float>(c, a);
}
