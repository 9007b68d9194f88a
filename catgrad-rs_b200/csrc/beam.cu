// beam.cu — one step of beam search: the best continuations over beams and vocabulary.
//
// For the beams j of a group with scores s_j (sums of log-probabilities) and logits x_j
//   total(j, v) = s_j + ((x_jv - M_j) - ln sum_u exp(x_ju - M_j)),  M_j = max_u x_ju,
// and the K largest are taken, equal ones in the order of j V + v.  A beam that is finished has one continuation,
// total(j, end) = s_j.  What has no number (NaN logits; all of a beam whose largest logit or own score is not finite)
// is -inf, as are masked logits.
//
// The logits are read once: 256 threads take 32 KB of a beam at a time and hold them in registers.
// Within a beam totals are in the order of the logits, so of each such piece the K largest are kept: the smallest of K disjoint groups'
// maxima is no larger than the piece's K-th largest value, and the few values that reach it (some K ln K) are ranked by
// counting, several pieces at a time so that a warp has each.  Where more reach it than a list holds, the K-th largest of 32
// groups' maxima is the bound, what is above it is taken, and of what is equal to it (masked, level logits) the first K;
// where even that is too much (logits in descending order), K rounds of a common maximum.
// A group of beams is a thread-block cluster, over whose blocks, each of up to four times 256 threads, the pieces of its beams are
// dealt; a warp then joins all sorted lists of a beam, and one warp those of the beams.
//
// 24 groups of 8 beams over 256000 tokens in bf16: 98 MB in 42.6 us, 2.3 TB/s (24 clusters of 10 blocks of 512 threads, two blocks on most SMs).
// Neither bytes nor issue (33 % of its slots) is used up: between two of a warp's instructions 15 clocks pass, 4.8 of them at barriers and 2.3
// for logits, none of which are on their way while a piece is ranked.  One group of 4 beams over 128256 in f32: 9.6 us, a chain of loads, barriers and joins behind a call of 4.
//
// Rows that begin off a 16-byte boundary take two loads a vector: 51.2 us over 255999.
//
// Exponentials are f32, their sums over more than a warp, the logarithm and the totals 64 bits: totals of different
// beams may lie close together.
#include <algorithm>

#include "mma.cuh"
#include "paged.h"

namespace cg {

namespace {

constexpr int BT = 256;            // threads that share a piece
constexpr int VECS = 8;            // 16-byte vectors of a piece that a thread holds
constexpr float LOG2E = 1.4426950408889634f;

struct SelectArgs {
  const void* logits;
  int64_t ld_b, ld_j;               // from one group and one beam to the next
  const float* scores;              // [B, J]
  const uint32_t* finished;         // [B, J] or null
  uint32_t end;
  int J, K, V;
  int pieces, rounds;               // of a beam; of a block (each of its times 256 threads has a piece a round)
  int joiners;                      // warps of a block that join lists
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

__device__ __forceinline__ uint64_t key_at(float x, int i) { return key_of(x == x ? x + 0.f : -INFINITY, (uint32_t)i); }  // (NaN as -inf, -0 as 0)

// the largest of the warp's keys, and the first lane that has it
__device__ __forceinline__ uint64_t warp_best(uint64_t key, int* lane) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32) == hi ? (uint32_t)key : 0u);
  const uint64_t best = (uint64_t)hi << 32 | lo;
  *lane = __ffs(__ballot_sync(0xffffffffu, key == best)) - 1;
  return best;
}

constexpr int MAX_OWN = 4;         // pieces of a beam: at most 32 times this
constexpr int POOL = 1024;         // values that reach their bounds, of several pieces
struct PieceWork {                 // of 256 threads
  float groups[2][32];             // (taking turns)
  int count[8];                    // by slot: up to 8 pieces are ranked together
  float peak[8], part[8][BT / 32];
  uint64_t best[BT / 32];
  int equal[BT / 32];
  uint64_t pool[POOL];
};

// Sums of 2^((x - peak) log2 e), two values at a time on the packed f32 units.
struct ExpSums {
  uint64_t s = 0, less, unit;
  __device__ __forceinline__ explicit ExpSums(float peak) {
    const float minus = -peak, l = LOG2E;
    asm("mov.b64 %0, {%1, %1};" : "=l"(less) : "f"(minus));
    asm("mov.b64 %0, {%1, %1};" : "=l"(unit) : "f"(l));
  }
  __device__ __forceinline__ void add(uint32_t x0, uint32_t x1) {
    uint64_t x, d, e;
    float e0, e1;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "r"(x0), "r"(x1));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(less));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(e) : "l"(d), "l"(unit));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(e0), "=f"(e1) : "l"(e));
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(fast_exp2(e0)), "f"(fast_exp2(e1)));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(s) : "l"(x));
  }
  __device__ __forceinline__ float sum() const {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(s));
    return a + b;
  }
};

// word i of 16, which stay in registers
__device__ __forceinline__ uint32_t word_of(const uint32_t* w, int i) {
  uint32_t a[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) a[k] = i & 1 ? w[2 * k + 1] : w[2 * k];
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = i & 2 ? a[2 * k + 1] : a[2 * k];
#pragma unroll
  for (int k = 0; k < 2; ++k) a[k] = i & 4 ? a[2 * k + 1] : a[2 * k];
  return i & 8 ? a[1] : a[0];
}

// Four 16-byte vectors' values (16 words).  (-inf stands for what lies outside.)
template <typename T>
struct Values;
template <>
struct Values<float> {
  static constexpr int per = 4, n = 16;
  static constexpr uint32_t lowest = 0xff800000u;
  static __device__ __forceinline__ float at(const uint32_t* w, int i) { return __uint_as_float(w[i]); }
  static __device__ __forceinline__ float largest(const uint32_t* w) {  // (NaNs are passed over)
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < n; ++i) m = fmaxf(m, at(w, i));
    return m;
  }
  static __device__ __forceinline__ uint32_t reach(const uint32_t* w, float bound) {  // a bit per value
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < n; ++i) m |= at(w, i) >= bound ? 1u << i : 0u;
    return m;
  }
  static __device__ __forceinline__ int value_of(int bit) { return bit; }
  static __device__ __forceinline__ float pick(const uint32_t* w, int i) { return __uint_as_float(word_of(w, i)); }
  static __device__ __forceinline__ float exps(const uint32_t* w, float peak) {
    ExpSums s(peak);
#pragma unroll
    for (int i = 0; i < n; i += 2) s.add(w[i], w[i + 1]);
    return s.sum();
  }
};
template <>
struct Values<__nv_bfloat16> {
  static constexpr int per = 8, n = 32;
  static constexpr uint32_t lowest = 0xff80ff80u;
  static __device__ __forceinline__ float at(const uint32_t* w, int i) { return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); }
  static __device__ __forceinline__ float largest(const uint32_t* w) {
    __nv_bfloat162 m = *(const __nv_bfloat162*)&w[0];
#pragma unroll
    for (int i = 1; i < n / 2; ++i) m = __hmax2(m, *(const __nv_bfloat162*)&w[i]);
    const float lo = __low2float(m), hi = __high2float(m);
    return fmaxf(fmaxf(lo, hi), -INFINITY);
  }
  // (bit i: value 2 i, bit 16 + i: value 2 i + 1)
  static __device__ __forceinline__ uint32_t reach(const uint32_t* w, float bound) {
    const __nv_bfloat162 b = __float2bfloat162_rn(bound);  // (a value of the piece)
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) m |= __hge2_mask(*(const __nv_bfloat162*)&w[i], b) & (0x00010001u << i);
    return m;
  }
  static __device__ __forceinline__ int value_of(int bit) { return bit < 16 ? 2 * bit : 2 * bit - 31; }
  static __device__ __forceinline__ float pick(const uint32_t* w, int i) {
    const uint32_t two = word_of(w, i >> 1);
    return __uint_as_float(i & 1 ? two & 0xffff0000u : two << 16);
  }
  static __device__ __forceinline__ float exps(const uint32_t* w, float peak) {
    ExpSums s(peak);
#pragma unroll
    for (int i = 0; i < n / 2; ++i) s.add(w[i] << 16, w[i] & 0xffff0000u);
    return s.sum();
  }
};

// A vector's values one at a time: -inf from `limit` on.
template <typename T>
__device__ __noinline__ uint4 load_edge(const T* row, int at, int limit) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = at + i < limit ? *(const uint32_t*)(row + at + i) : Values<T>::lowest;
    } else {
      const int lo = at + 2 * i, hi = lo + 1;
      w[i] = (lo < limit ? *(const uint16_t*)(row + lo) : Values<T>::lowest & 0xffffu) |
             (hi < limit ? *(const uint16_t*)(row + hi) : Values<T>::lowest & 0xffffu) << 16;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The vector that begins `shift` values into the aligned vector x and ends in the next one.
template <typename T>
__device__ __forceinline__ void realign(uint32_t* x, uint4 next, int shift) {
  const uint32_t a[8] = {x[0], x[1], x[2], x[3], next.x, next.y, next.z, next.w};
  const int words = shift * (int)sizeof(T) / 4;
  uint32_t b[6], c[5];
#pragma unroll
  for (int i = 0; i < 6; ++i) b[i] = words & 2 ? a[i + 2] : a[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) c[i] = words & 1 ? b[i + 1] : b[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = sizeof(T) == 4 ? c[i] : __funnelshift_r(c[i], c[i + 1], shift & 1 ? 16u : 0u);
}

// What is rare is kept out of the kernel's way (instructions are read once a call, so their number counts).
// The largest values of a piece whose list ran over: those above the K-th largest of 32 groups' maxima and, in the order of their
// places, K that are equal to it; or K rounds of a common maximum.  By all of its 256 threads.
template <typename T>
__device__ __noinline__ void rank_again(PieceWork& w, const T* row, int at0, int V, int K, int room, int slot) {
  constexpr int per = Values<T>::per;
  const int sb = threadIdx.x / BT, tid = threadIdx.x % BT, warp = tid >> 5, lane = tid & 31;
  auto sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(sb + 1), "r"(BT) : "memory"); };
  auto take = [&](int at, float v) {
    const int n = atomicAdd(&w.count[slot], 1);
    if (n < room) w.pool[slot * room + n] = key_at(v, at);
  };
  float mx = -INFINITY;
#pragma unroll 1
  for (int v = 0; v < VECS; ++v)
#pragma unroll
    for (int i = 0; i < per; ++i) {
      const int at = at0 + v * BT * per + i;
      if (at < V) mx = fmaxf(mx, (float)row[at]);
    }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  sync();
  if ((lane & 7) == 0) w.groups[0][tid >> 3] = mx;
  if (tid == 0) w.count[slot] = 0;
  sync();
  uint32_t left = up(w.groups[0][lane]), kth = 0;
  for (int r = 0; r < K; ++r) {
    kth = __reduce_max_sync(0xffffffffu, left);
    if (lane == __ffs(__ballot_sync(0xffffffffu, left == kth)) - 1) left = 0;
  }
  const float bound = down(kth);
  auto side = [&](int at) {  // 1 above the bound, 0 at it, -1 below
    const float v = (float)row[at], c = v == v ? v : -INFINITY;
    return c > bound ? 1 : c == bound ? 0 : -1;
  };
  if (mx > bound)
#pragma unroll 1
    for (int v = 0; v < VECS; ++v)
#pragma unroll 1
      for (int i = 0; i < per; ++i) {
        const int at = at0 + v * BT * per + i;
        if (at < V && side(at) > 0) take(at, (float)row[at]);
      }
  sync();
  const int above = w.count[slot];
  if (above + K <= room) {
    int have = 0;
#pragma unroll 1
    for (int v = 0; v < VECS && have < K; ++v) {
      uint32_t level = 0;
#pragma unroll
      for (int i = 0; i < per; ++i) {
        const int at = at0 + v * BT * per + i;
        if (at < V && side(at) == 0) level |= 1u << i;
      }
      int before = __popc(level);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int more = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += more;
      }
      if (lane == 31) w.equal[warp] = before;
      sync();
      before -= __popc(level);
      int all_of = 0;
      for (int i = 0; i < BT / 32; ++i) {
        if (i < warp) before += w.equal[i];
        all_of += w.equal[i];
      }
      for (int n = have + before; level && n < K; ++n, level &= level - 1) {
        const int at = at0 + v * BT * per + __ffs(level) - 1;
        w.pool[slot * room + above + n] = key_at((float)row[at], at);
      }
      have += all_of;
      sync();
    }
    if (tid == 0) w.count[slot] = above + min(have, K);
  } else {
    uint64_t last = ~0ull;
    for (int r = 0; r < K; ++r) {
      uint64_t best = 0;
#pragma unroll 1
      for (int v = 0; v < VECS; ++v)
#pragma unroll
        for (int i = 0; i < per; ++i) {
          const int at = at0 + v * BT * per + i;
          const uint64_t key = at < V ? key_at((float)row[at], at) : 0;
          if (key < last && key > best) best = key;
        }
      int who;
      best = warp_best(best, &who);
      if (lane == 0) w.best[warp] = best;
      sync();
      for (int i = 0; i < BT / 32; ++i) best = w.best[i] > best ? w.best[i] : best;
      if (tid == 0) w.pool[slot * room + r] = best;
      last = best;
      sync();
    }
    if (tid == 0) w.count[slot] = K;  // (places without a value are 0)
  }
  sync();
}
// This thread's sum of exponentials where some values are NaN, rounded as that of Values::exps is, so that NaN counts as a mask does.
template <typename T>
__device__ __noinline__ float sum_of_numbers(const T* row, int at0, int V, float peak) {
  constexpr int per = Values<T>::per;
  float sum = 0.f;
#pragma unroll 1
  for (int q = 0; q < VECS; q += 4) {
    float even = 0.f, odd = 0.f;
#pragma unroll 1
    for (int v = q; v < q + 4; ++v)
#pragma unroll 1
      for (int i = 0; i < per; i += 2) {
        const int at = at0 + v * BT * per + i;
        const float x = at < V ? (float)row[at] : -INFINITY, y = at + 1 < V ? (float)row[at + 1] : -INFINITY;
        if (x == x) even += fast_exp2((x - peak) * LOG2E);
        if (y == y) odd += fast_exp2((y - peak) * LOG2E);
      }
    sum += even + odd;
  }
  return sum;
}

__device__ __forceinline__ double total_of(float score, float x, float m, double log_sum) { return (double)score + (((double)x - (double)m) - log_sum); }
// Where 64 bits do not tell some totals of a beam apart (scores such as -1e30, logits next to 0): of those that equal the K-th the
// lowest tokens, all in the order of totals, then tokens.  By a warp: lane i has the (i + 1)-th largest logit's total and token, and afterwards
// those of the beam's (i + 1)-th continuation.  What is larger than the K-th total is among the K; what equals it is looked for in the beam up to
// the last of these.  `found`: room for K tokens.
struct Total {
  double total;
  uint32_t token;
};
template <typename T>
__device__ __noinline__ Total settle(const T* row, float score, float m, double log_sum, int V, int K, uint64_t* found, double total, uint32_t token) {
  const int lane = threadIdx.x & 31;
  const double least = __shfl_sync(0xffffffffu, total, K - 1);
  const int above = __popc(__ballot_sync(0xffffffffu, lane < K && total > least));
  const uint32_t last = __reduce_max_sync(0xffffffffu, lane >= above && lane < K ? token : 0u);
  int n = above;
  for (uint32_t v0 = 0; v0 <= last && n < K; v0 += 32) {
    const uint32_t v = v0 + lane;
    const float x = v < (uint32_t)V ? (float)row[v] : -INFINITY;
    const bool hit = v < (uint32_t)V && total_of(score, x == x ? x : -INFINITY, m, log_sum) == least;
    const uint32_t hits = __ballot_sync(0xffffffffu, hit);
    const int to = n + __popc(hits & ((1u << lane) - 1u));
    if (hit && to < K) found[to] = v;
    n += __popc(hits);
  }
  __syncwarp();
  if (lane >= above && lane < K) {
    total = least;
    token = (uint32_t)found[lane];
  }
  int rank = 0;
  for (int o = 0; o < K; ++o) {
    const double t = __shfl_sync(0xffffffffu, total, o);
    const uint32_t v = __shfl_sync(0xffffffffu, token, o);
    rank += t > total || (t == total && v < token);
  }
  __syncwarp();
  if (lane < K) found[rank] = (uint64_t)lane;
  __syncwarp();
  const int from = lane < K ? (int)found[lane] : lane;
  return {__shfl_sync(0xffffffffu, total, from), __shfl_sync(0xffffffffu, token, from)};
}

// dynamic shared memory: PieceWork [SB]; lists u64 [rounds][SB][K]; sums f64 [rounds][SB]; totals u64 [J][K]; places u64 [J][K];
// tops f32 [rounds][SB]; marks u32 [J]; then per joining warp a beam's lists of all blocks, u64 [pieces][K]
template <typename T, int SB>
__global__ void __launch_bounds__(SB * BT, 4 / SB) k_beam_select(SelectArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using Vals = Values<T>;
  constexpr int per = Vals::per;
  extern __shared__ uint64_t smem[];
  const int J = a.J, K = a.K, units = J * a.pieces;
  PieceWork* works = (PieceWork*)smem;
  uint64_t* lists = (uint64_t*)(works + SB);
  double* sums = (double*)(lists + a.rounds * SB * K);
  uint64_t* totals = (uint64_t*)(sums + a.rounds * SB);
  uint64_t* places = totals + J * K;
  float* tops = (float*)(places + J * K);
  uint32_t* marks = (uint32_t*)(tops + a.rounds * SB);
  uint64_t* all = (uint64_t*)(((uintptr_t)(marks + J) + 7) & ~(uintptr_t)7);

  const int sb = threadIdx.x / BT, tid = threadIdx.x % BT, warp = tid >> 5, lane = tid & 31;
  PieceWork& w = works[sb];
  auto sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(sb + 1), "r"(BT) : "memory"); };
  uint32_t rank, n_ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n_ranks));
  const int64_t b = blockIdx.y;
  if ((int)threadIdx.x < J) marks[threadIdx.x] = a.finished ? a.finished[b * J + threadIdx.x] : 0;
  if (tid < 8) w.count[tid] = 0;
  const int room = K <= 8 ? 128 : K <= 16 ? 256 : 512, slots = POOL / room;  // (more than `room` in one piece in 10^6)
  int least_groups = 1;
  while (least_groups < K) least_groups *= 2;

  // Unit u, piece u % pieces of beam u / pieces, belongs to round i of 256 threads of a block where u = (i n_ranks + rank) SB + sb.
  // A piece's vectors are counted from the beam's first value, wherever that lies in memory: sums of exponentials then depend on the logits
  // alone, and beams with the same logits have the same totals.  This thread's vectors are BT apart.
  const T* row;
  int at0;
  auto locate = [&](int u) {
    const int j = u / a.pieces;
    row = (const T*)a.logits + b * a.ld_b + (int64_t)j * a.ld_j;
    at0 = ((u - j * a.pieces) * (BT * VECS) + tid) * per;
  };
  auto load = [&](uint32_t* x) {
    const int shift = (int)(((uintptr_t)row & 15) / sizeof(T));  // values from a 16-byte boundary to a vector's first one
    if (shift == 0 && at0 - tid * per + BT * VECS * per <= a.V) {  // (all of the piece's)
      const uint4* from = (const uint4*)(row + at0);
#pragma unroll
      for (int v = 0; v < VECS; ++v) {
        const uint4 q = __ldg(from + v * BT);
        x[4 * v] = q.x; x[4 * v + 1] = q.y; x[4 * v + 2] = q.z; x[4 * v + 3] = q.w;
      }
      return;
    }
    // (all whole vectors are asked for before any is waited for: of those off a boundary the two aligned ones that they lie in, the
    // second of which a neighbour has asked for as its first)
    const int whole_to = a.V - per - (shift ? per - shift : 0);  // first values of whole vectors: from `shift` up to here
    bool edge = false;
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = at0 + v * BT * per;
      uint4 q = make_uint4(Vals::lowest, Vals::lowest, Vals::lowest, Vals::lowest);
      const bool whole = at >= shift && at <= whole_to;
      if (whole) q = __ldg((const uint4*)(row + at - shift));
      edge = edge || (!whole && at < a.V);
      x[4 * v] = q.x; x[4 * v + 1] = q.y; x[4 * v + 2] = q.z; x[4 * v + 3] = q.w;
    }
    if (shift)
#pragma unroll
      for (int v = 0; v < VECS; ++v) {
        const int at = at0 + v * BT * per;
        if (at >= shift && at <= whole_to) realign<T>(x + 4 * v, __ldg((const uint4*)(row + at - shift + per)), shift);
      }
    if (edge)
#pragma unroll
      for (int v = 0; v < VECS; ++v) {
        const int at = at0 + v * BT * per;
        if (!(at >= shift && at <= whole_to) && at < a.V) {
          const uint4 q = load_edge<T>(row, at, a.V);
          x[4 * v] = q.x; x[4 * v + 1] = q.y; x[4 * v + 2] = q.z; x[4 * v + 3] = q.w;
        }
      }
  };
  int slot = 0, begun = 0;  // the round of slot 0
  for (int i = 0; i < a.rounds; ++i) {
    const int u = (i * (int)n_ranks + (int)rank) * SB + sb;
    if (u < units) {
      locate(u);
      uint32_t x[4 * VECS];
      load(x);
      float mine = Vals::largest(x);
#pragma unroll
      for (int q = 16; q < 4 * VECS; q += 16) mine = fmaxf(mine, Vals::largest(x + q));
      float mx = mine;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if ((lane & 7) == 0) w.groups[i & 1][tid >> 3] = mx;
      sync();
      // every warp finds the smallest of 1, 2, .. 32 >= K groups' maxima
      uint32_t g = up(w.groups[i & 1][lane]);
      const uint32_t none = up(-INFINITY);
      const float peak = down(__reduce_max_sync(0xffffffffu, g));
      for (int o = 16; o >= least_groups; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
      // (groups without a value are left out where the others are enough)
      const int some = __popc(__ballot_sync(0xffffffffu, g > none));
      if (g == none && some >= K * (32 / least_groups)) g = 0xffffffffu;
      const float bound = down(__reduce_min_sync(0xffffffffu, g));
      if (bound == -INFINITY) {
        if (tid == 0) w.count[slot] = room + 1;
      } else if (__any_sync(0xffffffffu, mine >= bound)) {
        // places in the list for all of the warp's at once
        uint32_t m[VECS / 4];
        int mine_n = 0;
#pragma unroll
        for (int q = 0; q < VECS / 4; ++q) {
          m[q] = Vals::reach(x + 16 * q, bound);
          mine_n += __popc(m[q]);
        }
        int n = mine_n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int more = __shfl_up_sync(0xffffffffu, n, o);
          if (lane >= o) n += more;
        }
        int from = 0;
        if (lane == 31) from = atomicAdd(&w.count[slot], n);
        n += __shfl_sync(0xffffffffu, from, 31) - mine_n;
        if (mine_n) {
#pragma unroll
          for (int q = 0; q < VECS / 4; ++q)
            for (; m[q]; m[q] &= m[q] - 1, ++n) {
              const int e = Vals::value_of(__ffs(m[q]) - 1);
              if (n < room) w.pool[slot * room + n] = key_at(Vals::pick(x + 16 * q, e), at0 + (4 * q + e / per) * BT * per + e % per);
            }
        }
      }
      // (differences to the peak first: the largest value's term is exactly 1, so that equal beams stay equal)
      float sum = 0.f;
      if (peak > -INFINITY && peak < INFINITY) {
#pragma unroll
        for (int q = 0; q < 4 * VECS; q += 16) sum += Vals::exps(x + q, peak);
        if (!(sum == sum)) sum = sum_of_numbers<T>(row, at0, a.V, peak);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) w.part[slot][warp] = sum;
      if (tid == 0) w.peak[slot] = peak;
      ++slot;
    }
    if (slot > 0 && (slot == slots || i + 1 == a.rounds)) {  // the slots' lists: a warp has slots warp, warp + 8
      sync();
      for (int q = 0; q < slot; ++q)
        if (w.count[q] > room) {
          locate(((begun + q) * (int)n_ranks + (int)rank) * SB + sb);
          rank_again<T>(w, row, at0, a.V, K, room, q);
        }
      for (int q = warp; q < slot; q += BT / 32) {
        const int place = (begun + q) * SB + sb, n = w.count[q];
        double s = lane < BT / 32 ? (double)w.part[q][lane] : 0.;
#pragma unroll
        for (int o = 4; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) {
          sums[place] = s;
          tops[place] = w.peak[q];
        }
        const uint64_t* keys = w.pool + q * room;
        uint64_t* list = lists + place * K;
        if (lane < K) list[lane] = 0;
        __syncwarp();
        for (int k = lane; k < n; k += 32) {
          const uint64_t key = keys[k];
          int above = 0;
#pragma unroll 8
          for (int o = 0; o < n; ++o) above += (int)(keys[o] > key);
          if (above < K && key) list[above] = key;
        }
        __syncwarp();
        if (lane == 0) w.count[q] = 0;
      }
      sync();
      slot = 0;
      begun = i + 1;
    }
  }
  __syncthreads();
  cluster_barrier();

  // A warp joins a beam's sorted lists, and puts its K best totals into the first block.
  const uint32_t totals0 = remote_addr(totals, 0), places0 = remote_addr(places, 0);
  const int me = sb * (BT / 32) + warp, P = a.pieces;
  if (me < a.joiners)
    for (int j = (int)rank + me * (int)n_ranks; j < J; j += a.joiners * (int)n_ranks) {
      uint64_t* mine = all + me * P * K;
      // (a lane has pieces lane, lane + 32, ..: their list, maximum and sum)
      float m = -INFINITY, v[MAX_OWN];
      double part[MAX_OWN];
      const float score = a.scores[b * J + j];
#pragma unroll
      for (int i = 0; i < MAX_OWN; ++i) {
        const int p = lane + 32 * i;
        v[i] = -INFINITY;
        part[i] = 0.;
        if (p < P) {
          const int u = j * P + p, block = u / SB, round = block / (int)n_ranks, at = round * SB + u % SB;
          const uint32_t r = (uint32_t)(block - round * (int)n_ranks), from = remote_addr(lists + at * K, r);
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[i]) : "r"(remote_addr(tops + at, r)) : "memory");
          part[i] = __longlong_as_double((long long)remote_ld64(remote_addr(sums + at, r)));
          for (int k = 0; k < K; k += 4) {  // (four on their way at a time)
            uint64_t four[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) four[q] = k + q < K ? remote_ld64(from + (uint32_t)(k + q) * 8u) : 0;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (k + q < K) mine[p * K + k + q] = four[q];
          }
          m = fmaxf(m, v[i]);
        }
      }
      m = down(__reduce_max_sync(0xffffffffu, up(m)));
      double s = 0.;
#pragma unroll
      for (int i = 0; i < MAX_OWN; ++i)
        if (part[i] > 0.) s += part[i] * (double)fast_exp2((v[i] - m) * LOG2E);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      const double log_sum = log(s);
      const bool known = score > -INFINITY && score < INFINITY;
      const uint64_t j0 = (uint64_t)j * (uint64_t)a.V;
      auto put = [&](int i, double total, uint64_t v) {
        remote_st64(totals0 + (uint32_t)(j * K + i) * 8u, up64(total));
        remote_st64(places0 + (uint32_t)(j * K + i) * 8u, j0 + v);
      };
      if (marks[j] && known) {
        // the end token, then -inf in the order of the vocabulary
        for (int i = lane; i < K; i += 32) put(i, i == 0 ? (double)score + 0. : -INFINITY, i == 0 ? a.end : (uint32_t)(i - 1) + ((uint32_t)(i - 1) >= a.end ? 1u : 0u));
      } else if (!known || !(m > -INFINITY && m < INFINITY)) {
        for (int i = lane; i < K; i += 32) put(i, -INFINITY, (uint64_t)i);
      } else {
        __syncwarp();
        // K times the largest of the lists' heads; a lane has lists lane, lane + 32, ..
        uint64_t got = 0;
        int taken = 0;  // of list `lane`, where that is the lane's only one
        for (int r = 0; r < K; ++r) {
          uint64_t best = 0;
          int from = lane, who;
          if (P <= 32) {
            if (lane < P && taken < K) best = mine[lane * K + taken];
          } else {
            for (int l = lane; l < P; l += 32)
              if (mine[l * K] > best) { best = mine[l * K]; from = l; }
          }
          const uint64_t top = warp_best(best, &who);
          if (lane == who) {  // (keys differ: they hold the token)
            if (P <= 32) {
              ++taken;
            } else {
              uint64_t* list = mine + from * K;
              for (int i = 0; i + 1 < K && list[i]; ++i) list[i] = list[i + 1];
              list[K - 1] = 0;
            }
          }
          if (lane == (r & 31)) got = top;
          __syncwarp();
        }
        const float x = lane < K ? down((uint32_t)(got >> 32)) : INFINITY;
        Total best = {total_of(score, x, m, log_sum), 0xffffffffu - (uint32_t)got};
        // (rare: a step of f32, at least 2^-24 of a logit, may be less than what the total's three roundings in 64 bits take: 2^-48 of its
        // largest term; ln V < 32)
        if (__any_sync(0xffffffffu, fabsf(x) * 0x1p24f < fmaxf(fmaxf(fabsf(score), fabsf(m)), 32.f)))
          best = settle<T>((const T*)a.logits + b * a.ld_b + (int64_t)j * a.ld_j, score, m, log_sum, a.V, K, mine, best.total, best.token);
        if (lane < K) put(lane, best.total, best.token);
      }
    }
  cluster_barrier();

  // the best of the beams' sorted totals: a lane has a beam
  if (rank == 0 && threadIdx.x < 32) {
    int at = 0, beam = 0, place = 0;  // lane r keeps the r-th best's beam, and its place there
    uint64_t total = 0;
    for (int r = 0; r < K; ++r) {
      const uint64_t key = lane < J && at < K ? totals[lane * K + at] : 0;
      int who;
      const uint64_t best = warp_best(key, &who);  // (of equal totals the lowest beam's)
      const int from = __shfl_sync(0xffffffffu, at, who);
      if (lane == r) { beam = who; place = from; total = best; }
      if (lane == who) ++at;
    }
    if (lane < K) {
      const uint32_t token = (uint32_t)(places[beam * K + place] - (uint64_t)beam * (uint64_t)a.V);
      const int64_t to = b * K + lane;
      a.out_scores[to] = (float)down64(total);
      a.out_tokens[to] = token;
      a.out_parents[to] = (uint32_t)beam;
      a.out_finished[to] = marks[beam] || token == a.end;
    }
  }
}

template <typename T, int SB>
struct Blocks {
  static cudaError_t configure(int device) {
    static PerDeviceFlag configured_on;
    bool& configured = configured_on.at(device);
    if (configured) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(k_beam_select<T, SB>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_beam_select<T, SB>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    configured = e == cudaSuccess;
    return e;
  }
  // clusters of this many blocks that run at a time (asked once)
  static int at_a_time(int device, int ranks) {
    static int known[64][17];
    int& n = known[device & 63][ranks];
    if (n == 0) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)ranks, 1024);
      cfg.blockDim = dim3(SB * BT);
      cfg.dynamicSmemBytes = SB * sizeof(PieceWork) + 16384;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = (unsigned)ranks;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      int got = 0;
      if (configure(device) != cudaSuccess || cudaOccupancyMaxActiveClusters(&got, k_beam_select<T, SB>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        got = 0;
      }
      n = got > 0 ? got : -1;
    }
    return n;
  }
  static int launch(cg_ctx* c, SelectArgs a, int64_t B, int ranks) {
    a.rounds = (int)(((int64_t)a.J * a.pieces + ranks * SB - 1) / (ranks * SB));
    const size_t places = (size_t)a.rounds * SB, list = (size_t)a.pieces * a.K * 8;
    const size_t fixed = SB * sizeof(PieceWork) + (places * a.K + places + 2 * (size_t)a.J * a.K) * 8 + (places + a.J) * 4 + 8;
    a.joiners = std::min(SB * BT / 32, (a.J + ranks - 1) / ranks);
    while (a.joiners > 1 && fixed + a.joiners * list > (SB == 4 ? 160 : 50) * 1024) --a.joiners;
    const size_t smem = fixed + a.joiners * list;
    if (smem > 200 * 1024) return fail(c, CG_ERR_UNSUPPORTED, "beams times vocabulary too large");
    CG_CUDA(c, configure(c->core->device));
    CG_CUDA(c, launch_kernel(c, k_beam_select<T, SB>, dim3((unsigned)ranks, (unsigned)B), dim3(SB * BT), smem, -ranks, a));
    CG_LAUNCHED(c);
    return CG_OK;
  }
};

template <typename T>
int launch_select(cg_ctx* c, SelectArgs a, int64_t B) {
  constexpr int64_t per = 16 / sizeof(T), piece = BT * VECS;  // vectors of a piece
  const int64_t all = (a.V + per - 1) / per;                  // a beam's vectors
  const int64_t pieces = (all + piece - 1) / piece, units = a.J * pieces;
  if (pieces > 32 * MAX_OWN) return fail(c, CG_ERR_UNSUPPORTED, "vocabulary too large");
  a.pieces = (int)pieces;
  // Blocks of a group and times 256 threads of a block: what takes the least time by rounds of pieces, a round being a chain of
  // 1.5 us and 0.4 per 256 threads that an SM has.  Us for blocks x times, of the ten numbers of blocks and three of times, the rule's first:
  //   24 groups of 8 over 256000 in bf16    10 x 2: 42.8    5 x 4: 44.0   16 x 1: 45.3   8 x 2: 47.7   5 x 2: 52.0
  //   1 of 4 over 128256 in f32             16 x 4: 9.6    16 x 2: 10.2   8 x 4: 12.4   10 x 2: 14.1
  //   64 of 4 over 32000                     4 x 2: 12.8    8 x 1: 12.7    2 x 4: 13.3   2 x 2: 14.9
  //   190 of 1 over 50257 in bf16            1 x 2: 16.8    2 x 1: 18.0    1 x 1: 18.6   4 x 1: 19.1  (rows off a boundary)
  //   12 of 8 over 151936 in bf16           16 x 2: 21.7   16 x 1: 21.3    8 x 4: 22.0   6 x 4: 25.7
  int best_ranks = 0, best_sb = 1;
  double best = 1e300;
  const int device = c->core->device;
  for (int ranks : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16})
    for (int sb : {1, 2, 4}) {
      if (ranks * sb > 1 && (ranks * sb + 1) / 2 >= units + 1) continue;
      const int n = sb == 1 ? Blocks<T, 1>::at_a_time(device, ranks) : sb == 2 ? Blocks<T, 2>::at_a_time(device, ranks) : Blocks<T, 4>::at_a_time(device, ranks);
      if (n <= 0) continue;
      const double waves = (double)((B + n - 1) / n), rounds = (double)((units + ranks * sb - 1) / (ranks * sb));
      if (rounds * sb * a.K * 8 > 100 * 1024) continue;
      const double per_sm = std::max((double)sb, (double)(std::min<int64_t>(B, n) * ranks * sb) / 148.);
      const double cost = waves * rounds * (1.5 + 0.4 * per_sm) + 0.1 * ranks;
      if (cost < best) {
        best = cost;
        best_ranks = ranks;
        best_sb = sb;
      }
    }
  if (best_ranks == 0) return fail(c, CG_ERR_UNSUPPORTED, "beams times vocabulary too large");
  if (best_sb == 4) return Blocks<T, 4>::launch(c, a, B, best_ranks);
  if (best_sb == 2) return Blocks<T, 2>::launch(c, a, B, best_ranks);
  return Blocks<T, 1>::launch(c, a, B, best_ranks);
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
  if (V > 1ll << 30) return fail(c, CG_ERR_UNSUPPORTED, "vocabulary too large");
  if (finished && (int64_t)end >= V) return fail(c, CG_ERR_INVALID, "the end token is not in the vocabulary");
  // the scores and marks of a group are read before its new ones are written, so they may take their place
  const bool whole = K == J, same_scores = whole && scores_out->data() == scores->data(), same_marks = whole && finished && finished_out->data() == finished->data();
  if (overlap_any({logits, same_scores ? nullptr : scores, same_marks ? nullptr : finished}, {scores_out, tokens_out, parents_out, finished_out}) ||
      (same_scores && finished && overlap(Extent(scores), Extent(finished))) || (same_marks && overlap(Extent(finished), Extent(scores))))
    return fail(c, CG_ERR_INVALID, "an output overlaps an input or another one");
  if (B == 0 || K == 0) return CG_OK;
  if (J == 0) return fail(c, CG_ERR_SHAPE, "no beams");
  SelectArgs a = {};
  a.logits = logits->data();
  a.ld_b = logits->strides[0]; a.ld_j = logits->strides[1];
  a.scores = (const float*)scores->data();
  a.finished = finished ? (const uint32_t*)finished->data() : nullptr;
  a.end = end;
  a.J = (int)J; a.K = (int)K; a.V = (int)V;
  a.out_scores = (float*)scores_out->data();
  a.out_tokens = (uint32_t*)tokens_out->data();
  a.out_parents = (uint32_t*)parents_out->data();
  a.out_finished = (uint32_t*)finished_out->data();
  for (cg_tensor* t : {scores_out, tokens_out, parents_out, finished_out}) written(t);
  return logits->storage == ST_BF16 ? launch_select<__nv_bfloat16>(c, a, B) : launch_select<float>(c, a, B);
}
