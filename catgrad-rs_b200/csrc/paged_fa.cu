// paged_fa.cu — attention of prompts over a paged cache on tcgen05 / TMEM, in bf16.  D is the head size, rounded up to 64, 128
// or 256: what is read beyond a head is zeros.
//
// A tile is 128 query rows, the query heads of a key head side by side: row r of a tile that begins at token i0 is token
// i0 + r / rep, head r % rep of the group.  Keys come 64 at a time, by one TMA box per page (or per 64 keys of a longer
// one) and 64 components.  Per query tile
//   S = Q K^T    128 x 64, f32, two buffers in TMEM, the next one computed while this one's softmax runs
//   P            bf16 over its scores in TMEM, the A operand of
//   O += P V     128 x D, f32 in TMEM
// and four warps, a thread per row, make P from S: they hold a row's 64 scores in registers, so that scores are read once.
//
// Exponentials are taken against a reference that lags behind the row's maximum by up to 2^8: O and the sum are rescaled
// only when it would be more.  bf16 has the same relative step everywhere, so this costs no precision but for
// the largest probability, which is exactly 1 against the exact maximum; the denominator sums the
// probabilities as bf16 holds them, so that a row that one key decides loses nothing either way.  Probabilities are one bf16 operand: a
// second part, as the decode form has, would double the second product, which is half of this kernel's work.  Their rounding
// (2^-9 of each, of either sign) adds to the output's: errors against 64 bits 0.0021 of the result, where the output's alone are 0.0016.  Those of chunks of shared
// keys (CHUNK below) have the second part, and the denominator sums them unrounded, so that sharing costs no bits: 0.00166, for 56.4 us instead of 53.9 (64 rows of 1 behind
// 16001), 36.2 instead of 35.1 (30 of up to 5 in 3 groups behind 4003).  The rows' own keys in OWN have one, as these tokens' have in the form of prompts (with two 43.3).
//
// Where there are few tiles, or a little more than a whole number of turns, a cluster of 2 or 4 blocks shares a tile's keys; their outputs
// are joined through shared memory.
//
// One row of 8191 tokens, 32 heads and 8 key heads of 128: 564 us, 975 TFLOP/s at about 1690 MHz under the power limit; the tensor pipe is
// busy 51 % of the time, the exponentials' unit as much: what bounds it is the chain scores -> softmax -> product, which two tiles per SM
// hide in part.  128-key tiles with one score buffer: 619 us.  6 rows of up to 700 behind 5003, 8 heads and 4 of 256, cap and
// window: 150 us, 566 TFLOP/s, with one tile per SM (soft-caps as branches 523, as exponentials 214).
//
// Every mbarrier wait is bounded; on expiry the error word is raised, all roles leave their loops, TMEM is freed and the kernel
// returns.
#include <algorithm>

#include "mma.cuh"
#include "paged_attn.h"
#include "tc_common.cuh"

namespace cg {

namespace {

using namespace tc;

constexpr int KT = 64;            // keys of a tile
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LAG = 8.f;        // of the exponents' reference, in powers of 2

struct FaArgs {
  PagedRows rows;
  __nv_bfloat16* out;
  int64_t most, window, pool_rows;  // pool_rows: rows of d values in each pool, n_pages nkv page
  int nh, nkv, rep, per, d;         // per: tokens of a query tile
  int slices;                       // blocks that share a tile's keys
  float scale_log2e, cap_log2e, cap_unit;  // soft-cap c: c log2(e), -2 log2(e) score factor / c
  float cap_in, cap_poly[6];               // score factor / c; c log2(e) times tanh's series
  float lag;                               // LAG in products q k
  SharedParts sh;
};

// B operand stored [k rows][n contiguous] in 128-byte-swizzled boxes of [rows, 64 elements], chunk_bytes apart
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t chunk_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((chunk_bytes >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]),
        "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
        "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// A from TMEM (bf16, two consecutive k per column), B from shared memory
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }

// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}

template <int D, int NQ>
__host__ __device__ constexpr int fa_stages() { return NQ == 2 ? 4 : D == 64 ? 4 : 2; }
template <int D, int NQ>
__host__ __device__ constexpr size_t fa_smem() {
  return 1024 + (size_t)(D / 64) * (NQ * 128 * 128 + 2 * fa_stages<D, NQ>() * KT * 128) + 8 * (1 + 4 * fa_stages<D, NQ>() + 5 * NQ + 2) + 16;
}

// Warps: 0 loads, 1 and 3 issue the products of query tiles 0 and 1, 2 clears values that nobody sees, 4 to 7 and 8 to 11 are the rows
// of tiles 0 and 1.
//
// CHUNK: the queries are those of a group of rows, the keys a chunk of what the group has in common (through its first row's table), and
// the outputs parts that are joined with the rows' own keys' (OWN).  A token's position is then its row's, and masks are only looked at
// where a query stands inside the prefix or a window ends there.  64 rows, 32 heads and 8 key heads of 128, over 16001 shared keys in chunks of 1280: 2.6 us to the
// first loads, 2.2 to the first scores, 1.2 per 64 keys where an SM has two blocks (1.07 with one part of the probabilities), 2 to write the parts (4 in 16-byte pieces).
template <int D, int NQ, bool CAP, int MODE>
__global__ void __launch_bounds__(NQ == 2 ? 384 : 256, NQ == 2 || D > 128 ? 1 : 2)
k_paged_fa(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, FaArgs p) {
  constexpr bool SHARED = MODE == KeysOf::CHUNK, OWN = MODE == KeysOf::OWN, PART = SHARED || OWN;
  constexpr int SUB = D / 64, KS = fa_stages<D, NQ>();
  constexpr uint32_t BOX = 128 * 128, KBOX = KT * 128;
  constexpr uint32_t Q_BYTES = SUB * BOX, KV_BYTES = SUB * KBOX;
  constexpr uint32_t TILE_COLS = 2 * KT + D;                       // two score buffers, then O
  constexpr uint32_t NCOLS = NQ * TILE_COLS <= 256 ? 256 : 512;
  static_assert(NQ * TILE_COLS <= NCOLS, "TMEM");

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - raw);
  const uint32_t sq = base, sk = sq + NQ * Q_BYTES, sv = sk + KS * KV_BYTES, bars = sv + KS * KV_BYTES;
  const uint32_t b_q = bars, b_k_full = b_q + 8, b_v_full = b_k_full + 8 * KS, b_k_empty = b_v_full + 8 * KS, b_v_empty = b_k_empty + 8 * KS,
                 b_tile = b_v_empty + 8 * KS,  // per query tile: scores [2], probabilities [2], output
                 b_v_last = b_tile + 40 * NQ, b_v_ready = b_v_last + 8;
  volatile uint32_t* tmem_slot = (volatile uint32_t*)(gen + (b_v_ready + 8 - base));
  volatile int* cta_abort = (volatile int*)(gen + (b_v_ready + 12 - base));

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;  // (warp: known to be uniform)
  // q, the tables and the pages are written by the preceding kernels
  auto dependency = []() { asm volatile("griddepcontrol.wait;" ::: "memory"); };
  if (!OWN) dependency();
  const int slice = (int)blockIdx.x % p.slices;
  const int kvh = blockIdx.y;
  int64_t qt = ((int)gridDim.x - 1 - (int)blockIdx.x) / p.slices;  // longest first
  int64_t row = blockIdx.z, tok0, n, len, rows = 0, shared = 0;  // (OWN: shared are the keys in front)
  int64_t group = -1;
  if (SHARED) {
    const int64_t tiles = (int)gridDim.x / (p.slices * p.sh.chunks), t = (int)blockIdx.x / p.slices % tiles;
    GroupTile g;
    if (!group_of_tile(p.rows, p.sh.groups, t, 1, (int64_t)NQ * p.per, &g)) return;  // uniform over the CTA, before anything is allocated
    row = g.row0;
    rows = g.rows;
    tok0 = g.tok0;
    n = g.n;
    shared = g.shared;
    qt = g.tile;
    len = 0;
  } else {
    if (OWN) group = group_of_row(p.sh.groups, row, &shared);
    if (!row_span(p.rows, row, p.most, &tok0, &n, &len)) n = 0;
  }
  const int64_t i0 = qt * NQ * p.per;                            // first token of the first tile
  const int chunk = OWN ? p.sh.chunks : SHARED ? (int)blockIdx.x / p.slices / ((int)gridDim.x / (p.slices * p.sh.chunks)) : 0;
  if (SHARED && chunk * p.sh.chunk >= shared) n = 0;
  if (OWN && i0 >= n && last_block()) dependency();
  if (i0 >= n) return;
  const int64_t pos0 = SHARED ? 0 : len - n;
  const int64_t last = SHARED ? min(shared, (chunk + 1) * p.sh.chunk) - 1 : pos0 + min(n, i0 + NQ * p.per) - 1;  // the last key, position of the last query
  const int64_t lo = SHARED ? chunk * p.sh.chunk : max(p.window > 0 ? max((int64_t)0, pos0 + i0 - p.window + 1) : 0, OWN ? min(shared, last + 1) : 0);  // first visible key
  // this block's share of the key tiles: [j0, j0 + nt)
  const int all = max((int)(last / KT + 1 - lo / KT), 0), share = (all + p.slices - 1) / p.slices;
  const int64_t j0 = lo / KT + (int64_t)slice * share;
  const int nt = min(share, max(0, all - slice * share));
  // Keys of the last tile that some query sees.  The values behind them (what nothing or another sequence wrote) are
  // cleared in shared memory: a probability of 0 times an infinity would not be 0
  const int seen = nt > 0 && slice * share + nt == all ? (int)(last % KT) + 1 : KT;

  if (tid == 0) {
    mbar_init(b_q, 1);
    for (int i = 0; i < KS; ++i) {
      mbar_init(b_k_full + 8 * i, 1);
      mbar_init(b_v_full + 8 * i, 1);
      mbar_init(b_k_empty + 8 * i, NQ);
      mbar_init(b_v_empty + 8 * i, NQ);
    }
    for (int t = 0; t < NQ; ++t) {
      mbar_init(b_tile + 40 * t, 1);
      mbar_init(b_tile + 40 * t + 8, 1);
      mbar_init(b_tile + 40 * t + 16, 4);  // (a warp each)
      mbar_init(b_tile + 40 * t + 24, 4);
      mbar_init(b_tile + 40 * t + 32, 1);
    }
    mbar_init(b_v_last, 1);
    mbar_init(b_v_ready, 1);
    *cta_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  // TMEM between the dependency and the trigger: all kernels before have given their columns back, and none behind can
  // take columns that this one still waits for
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)), "r"(NCOLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  float m = -INFINITY, l = 0.f;  // of a row (m in units of log2: what a score is in the exponent of 2)
  float limit = -INFINITY;       // the product q k from which m follows
  if (warp == 0 && nt > 0) {
    // ---- loads ----
    if (lane == 0) {
      mbar_expect_tx(b_q, NQ * SUB * (uint32_t)(p.per * p.rep) * 128u);
      for (int t = 0; t < NQ; ++t)
        for (int s = 0; s < SUB; ++s) load_3d(sq + t * Q_BYTES + s * BOX, &map_q, s * 64, kvh * p.rep, (int)(tok0 + i0 + t * p.per), b_q);
    }
    // A lane has a page of the tile (or the whole tile, if pages are longer).  Pages that hold no visible key are not looked up:
    // a box behind the pool's end reads as zeros.
    const int lg = p.rows.lg, box = min(1 << lg, KT), pages = KT / box;
    const int off_end = (int)p.pool_rows;
    auto place = [&](int64_t j) {  // this lane's first row of the pool in key tile j
      const int64_t key = j * KT + lane * box;
      if (lane >= pages || key > last || key + box <= lo) return off_end;
      const int64_t id = page_of(p.rows, row, key);
      return id < 0 ? off_end : (int)(((id * p.nkv + kvh) << lg) + (key & ((1 << lg) - 1)));
    };
    int at = place(j0), j = 0;
    bool ok = true, half = false;  // half: of tile j the keys have been asked for
    for (; j < nt; ++j) {
      const int stage = j % KS;
      const uint32_t ph = (uint32_t)(j / KS) & 1u;
      const int next = j + 1 < nt ? place(j0 + j + 1) : off_end;  // (on its way while this tile waits for room)
      half = false;
      if (j >= KS) ok = __all_sync(0xffffffffu, mbar_wait(b_k_empty + 8 * stage, ph ^ 1u, cta_abort, p.rows.err));
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(b_k_full + 8 * stage, KV_BYTES);
      __syncwarp();
      if (lane < pages)
        for (int s = 0; s < SUB; ++s) tma_load_2d(sk + stage * KV_BYTES + s * KBOX + lane * box * 128, &map_k, s * 64, at, b_k_full + 8 * stage);
      half = true;
      if (j >= KS) ok = __all_sync(0xffffffffu, mbar_wait(b_v_empty + 8 * stage, ph ^ 1u, cta_abort, p.rows.err));
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(b_v_full + 8 * stage, KV_BYTES);
      __syncwarp();
      if (lane < pages)
        for (int s = 0; s < SUB; ++s) tma_load_2d(sv + stage * KV_BYTES + s * KBOX + lane * box * 128, &map_v, s * 64, at, b_v_full + 8 * stage);
      at = next;
    }
    if (!ok)  // the block does not leave before its copies have arrived
      for (int i = max(0, j - KS + 1); i <= j; ++i) {
        if (i < j || half) mbar_drain(b_k_full + 8 * (i % KS), (uint32_t)(i / KS) & 1u, p.rows.err);
        if (i < j) mbar_drain(b_v_full + 8 * (i % KS), (uint32_t)(i / KS) & 1u, p.rows.err);
      }
  } else if (nt > 0 && (warp == 1 || (NQ == 2 && warp == 3))) {
    // ---- products ----
    // The whole warp goes through the loop and one lane issues: descriptors then are uniform values, which an issue takes as they are.
    // (A single lane's loop: some 70 cycles an issue where a product of 64 keys takes 48.)
    const int t = warp >> 1;
    const bool issues = elect_one();
    constexpr uint32_t idesc_s = umma_idesc(KT), idesc_o = umma_idesc(D) | (1u << 16);  // (V: MN-major)
    const uint64_t dq = umma_desc(sq + t * Q_BYTES), dk = umma_desc(sk), dv = desc_mn(sv, KBOX);
    const uint32_t cols = tmem_base + t * TILE_COLS, o_cols = cols + 2 * KT;
    const uint32_t b_s = b_tile + 40 * t, b_p = b_s + 16, b_o = b_s + 32;
    auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, cta_abort, p.rows.err)) != 0; };
    auto qk = [&](int j) {
      const uint32_t buf = (uint32_t)j & 1u, stage = (uint32_t)(j % KS);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (issues) {
        const uint64_t dks = dk + ((stage * KV_BYTES) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / UMMA_K; ++kk) {
          const uint64_t oq = ((uint32_t)(kk / 4) * BOX + (uint32_t)(kk % 4) * 32u) >> 4, ok = ((uint32_t)(kk / 4) * KBOX + (uint32_t)(kk % 4) * 32u) >> 4;
          umma_bf16(cols + buf * KT, dq + oq, dks + ok, idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(b_s + 8 * buf);
        umma_commit(b_k_empty + 8 * stage);
      }
      __syncwarp();
    };
    auto pv = [&](int j) {
      const uint32_t buf = (uint32_t)j & 1u, stage = (uint32_t)(j % KS);
      if (j == nt - 1 && seen < KT) {
        // (warp 2 clears what no query sees while the softmax runs)
        if (t == 0 && issues) arrive(b_v_last);
        if (!wait(b_v_ready, 0)) return false;
      }
      if (!wait(b_p + 8 * buf, (uint32_t)(j >> 1) & 1u)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (issues) {
        const uint64_t dvs = dv + ((stage * KV_BYTES) >> 4);
#pragma unroll
        for (int kk = 0; kk < KT / UMMA_K; ++kk)
          umma_ts(o_cols, cols + buf * KT + kk * (UMMA_K / 2), dvs + (((uint32_t)kk * (UMMA_K * 128u)) >> 4), idesc_o, j > 0 || kk > 0 ? 1u : 0u);
        if (SHARED)  // (the probabilities' second parts, in the other half of the columns)
#pragma unroll
          for (int kk = 0; kk < KT / UMMA_K; ++kk) umma_ts(o_cols, cols + buf * KT + KT / 2 + kk * (UMMA_K / 2), dvs + (((uint32_t)kk * (UMMA_K * 128u)) >> 4), idesc_o, 1u);
        umma_commit(b_o);
        umma_commit(b_v_empty + 8 * stage);
      }
      __syncwarp();
      return true;
    };
    // Scores overwrite the probabilities that lay in their columns, and products with different accumulators are not
    // ordered among themselves: the product that reads them is waited for.
    auto done = [&](int j) { return wait(b_o, (uint32_t)j & 1u); };
    auto keys = [&](int j) { return j >= nt || wait(b_k_full + 8 * (j % KS), (uint32_t)(j / KS) & 1u); };
    auto values = [&](int j) { return j >= nt || wait(b_v_full + 8 * (j % KS), (uint32_t)(j / KS) & 1u); };
    bool ok = wait(b_q, 0) && keys(0);
    if (ok) qk(0);
    ok = ok && keys(1) && values(0);
    for (int j = 0; j < nt && ok; ++j) {
      if (j + 1 < nt) {
        ok = j == 0 || done(j - 1);
        if (!ok) break;
        qk(j + 1);
      }
      // (the next tiles' arrival is waited for behind the products, off the chain from one softmax to the next)
      ok = pv(j) && keys(j + 2) && values(j + 1);
    }
  } else if (warp == 2) {
    if (seen < KT) {
      const uint32_t stage = (uint32_t)((nt - 1) % KS);
      if (mbar_wait(b_v_last, 0, cta_abort, p.rows.err)) {  // the last values have arrived
        for (int i = lane; i < SUB * (KT - seen) * 8; i += 32) {
          const int sub = i / ((KT - seen) * 8), x = i - sub * ((KT - seen) * 8);
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + stage * KV_BYTES + sub * KBOX + (uint32_t)seen * 128u + (uint32_t)x * 16u), "r"(0)
                       : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(b_v_ready);
      }
    }
  } else if (warp >= 4) {
    // ---- rows ----
    const int t = (warp - 4) >> 2, q = warp & 3;
    const int r = q * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lane_base = tmem_base + t * TILE_COLS + ((uint32_t)(q * 32) << 16);
    const uint32_t o_addr = lane_base + 2 * KT;
    const uint32_t b_s = b_tile + 40 * t, b_p = b_s + 16, b_o = b_s + 32;
    const int64_t first = i0 + t * p.per;                       // the tile's first token
    const int64_t ti = first + r / p.rep;                       // this row's
    const int head = kvh * p.rep + r % p.rep;
    const bool mine = r < p.per * p.rep && ti < n;              // (others have what follows in q, or nothing that was loaded)
    int64_t qpos = pos0 + ti, tile_last = min(pos0 + first + p.per - 1, last), tile_first = pos0 + first;
    if (SHARED) {
      tile_positions(p.rows, row, rows, tok0 + first, tok0 + min(first + p.per, n) - 1, &tile_first, &tile_last);
      qpos = last;
      if (tile_first < last || (p.window > 0 && tile_last >= p.window + lo)) {
        if (mine) qpos = position_of(p.rows, row, rows, tok0 + ti);
        tile_first = min(tile_first, last);
      } else {  // all of them see all of the chunk
        tile_first = last;
        tile_last = 0;
      }
    }
    bool ok = true;
    for (int j = 0; j < nt && ok; ++j) {
      const int buf = j & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(b_s + 8 * buf, (uint32_t)(j >> 1) & 1u, cta_abort, p.rows.err));  // (a warp leaves whole)
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int64_t k0 = (j0 + j) * KT;
      const uint32_t s_addr = lane_base + buf * KT;
      uint32_t v[KT];
      ld32(s_addr, v);
      ld32(s_addr + 32, v + 32);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      // uniform: some key may be masked for some row
      const bool masked = k0 + KT - 1 > tile_first || (p.window > 0 && k0 <= tile_last - p.window) || (OWN && k0 < shared);
      uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
      if (masked) {
        // column c is visible to this row iff low <= c <= lim
        const int64_t lim64 = (SHARED ? min(qpos, last) : qpos) - k0, low64 = max(p.window > 0 ? qpos - k0 - p.window + 1 : 0, OWN ? shared - k0 : 0);
        const int lim = lim64 > KT ? KT : (lim64 < -1 ? -1 : (int)lim64), low = low64 < 0 ? 0 : (low64 > KT ? KT : (int)low64);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          vis[c] = bits_below(lim + 1 - c * 32) & ~bits_below(low - c * 32);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[c * 32 + i] = vis[c] & (1u << i) ? v[c * 32 + i] : 0xff800000u;
        }
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < KT; i += 2) mx4[i / 2 & 3] = fmaxf(fmaxf(mx4[i / 2 & 3], __uint_as_float(v[i])), __uint_as_float(v[i + 1]));
      const float raw_max = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      bool small = false;  // (uniform) no score of the sequence's rows is beyond 3/4 of the cap
      if (CAP) {
        if (masked)
#pragma unroll
          for (int i = 0; i < KT; ++i) v[i] = vis[i / 32] >> (i & 31) & 1u ? v[i] : 0u;  // (their probabilities are cleared)
        float low4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KT; i += 2) low4[i / 2 & 3] = fminf(fminf(low4[i / 2 & 3], __uint_as_float(v[i])), __uint_as_float(v[i + 1]));
        const float far = fmaxf(raw_max, -fminf(fminf(low4[0], low4[1]), fminf(low4[2], low4[3])));
        small = __all_sync(0xffffffffu, !mine || far * p.cap_in <= 0.75f);
      }
      // (the soft-cap is monotone, and what a score grows by is no less than what its cap does)
      auto reference = [&]() {
        if (CAP) return raw_max == -INFINITY ? -INFINITY : soft_cap(raw_max, p.cap_log2e, p.cap_in, p.cap_unit);
        return raw_max * p.scale_log2e;
      };
      if (j == 0) {
        m = reference();
        limit = raw_max + p.lag;
      } else {
        const bool grown = raw_max > limit;
        if (__any_sync(0xffffffffu, grown)) {
          const float m_new = grown ? reference() : m;
          limit = grown ? raw_max + p.lag : limit;
          const float corr = grown ? fast_exp2(m - m_new) : 1.f;  // 0 while m is -inf
          // (the product before the last was complete before this tile's scores could be issued, so the parity is that
          // of the last)
          ok = __all_sync(0xffffffffu, mbar_wait(b_o, (uint32_t)(j - 1) & 1u, cta_abort, p.rows.err));
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(o_addr + c, o);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            st16(o_addr + c, o);
          }
          l *= corr;
          m = m_new;
        }
      }
      const float mc = m == -INFINITY ? 0.f : m;
      float ls[2] = {0.f, 0.f};
      // Two probabilities as bf16, and (of shared keys) what their rounding left, in the place of the scores.
      auto split = [&](uint32_t* pk, int c, int i, float e0, float e1) {
        if (SHARED) {
          if (CAP && masked) {
            e0 = vis[c] >> i & 1u ? e0 : 0.f;
            e1 = vis[c] >> i & 2u ? e1 : 0.f;
          }
          ls[0] += e0;
          ls[1] += e1;
        }
        pk[i / 2] = pack_bf16(e0, e1);
        if (SHARED) v[c * 32 + i / 2] = pack_bf16(e0 - __uint_as_float(pk[i / 2] << 16), e1 - __uint_as_float(pk[i / 2] & 0xffff0000u));
      };
      // All go to TMEM; of one part, masked ones are cleared here and the sum is of what the products use.
      auto put = [&](uint32_t* pk, int c) {
        if (!SHARED) {
          if (CAP && masked)
#pragma unroll
            for (int i = 0; i < 32; i += 2) pk[i / 2] &= (vis[c] >> i & 1u ? 0xffffu : 0u) | (vis[c] >> i & 2u ? 0xffff0000u : 0u);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            ls[0] += __uint_as_float(pk[i] << 16);
            ls[1] += __uint_as_float(pk[i] & 0xffff0000u);
          }
        }
        st16(s_addr + (uint32_t)c * 16u, pk);
        if (SHARED) st16(s_addr + KT / 2 + (uint32_t)c * 16u, v + c * 32);
      };
      // probabilities of a half of the tile; `exponent` of a score
      auto half = [&](int c, auto exponent) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) split(pk, c, i, fast_exp2(exponent(__uint_as_float(v[c * 32 + i]))), fast_exp2(exponent(__uint_as_float(v[c * 32 + i + 1]))));
        put(pk, c);
      };
      if (CAP && small) {
        // c tanh(y), |y| <= 3/4, as y times a polynomial of y^2, two scores at a time: one exponential a score instead of two and a
        // reciprocal
        auto two = [](float a, float b) {
          uint64_t w;
          asm("mov.b64 %0, {%1, %2};" : "=l"(w) : "f"(a), "f"(b));
          return w;
        };
        auto mul = [](uint64_t a, uint64_t b) {
          uint64_t w;
          asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(w) : "l"(a), "l"(b));
          return w;
        };
        auto fma = [](uint64_t a, uint64_t b, uint64_t c) {
          uint64_t w;
          asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(w) : "l"(a), "l"(b), "l"(c));
          return w;
        };
        const uint64_t in = two(p.cap_in, p.cap_in), less = two(-mc, -mc);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const uint64_t y = mul(two(__uint_as_float(v[c * 32 + i]), __uint_as_float(v[c * 32 + i + 1])), in), u = mul(y, y);
            uint64_t f = two(p.cap_poly[5], p.cap_poly[5]);
#pragma unroll
            for (int q = 4; q >= 0; --q) f = fma(f, u, two(p.cap_poly[q], p.cap_poly[q]));
            f = fma(f, y, less);
            float x0, x1;
            asm("mov.b64 {%0, %1}, %2;" : "=f"(x0), "=f"(x1) : "l"(f));
            split(pk, c, i, fast_exp2(x0), fast_exp2(x1));
          }
          put(pk, c);
        }
      } else
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (CAP) half(c, [&](float x) { return soft_cap(x, p.cap_log2e, p.cap_in, p.cap_unit) - mc; });
        else half(c, [&](float x) { return fmaf(x, p.scale_log2e, -mc); });
      }
      // (This warp may be a whole product ahead of the tensor core, and a parity tells only neighbouring phases apart: the
      // last product but one is waited for here, where the last cannot have been issued.)
      if (j > 0 && j + 1 == nt) ok = mbar_wait(b_o, (uint32_t)(j - 1) & 1u, cta_abort, p.rows.err);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(b_p + 8 * buf);
      l += ls[0] + ls[1];
    }
    ok = ok && (nt == 0 || mbar_wait(b_o, (uint32_t)(nt - 1) & 1u, cta_abort, p.rows.err));
    ok = __all_sync(0xffffffffu, ok);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const bool out = ok && mine;
    const int64_t part_at = ((int64_t)chunk * p.rows.M + tok0 + ti) * p.nh + head;
    if (PART && p.slices == 1 && out) p.sh.ml[part_at] = make_float2(m, l);
    __nv_bfloat16* dst = p.out + ((tok0 + ti) * p.nh + head) * (int64_t)p.d;
#pragma unroll 1
    for (int c0 = 0; c0 < D && p.slices == 1; c0 += 32) {
      uint32_t v[32];
      ld32(o_addr + c0, v);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (PART) {  // (without keys nothing was written: the sum says so)
        float* to = p.sh.out + part_at * p.d + c0;
#pragma unroll
        for (int u = 0; u < 32; u += 8)  // (whole sectors: a row's values are a thread's)
          if (out && c0 + u < p.d)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + u), "r"(v[u]), "r"(v[u + 1]), "r"(v[u + 2]), "r"(v[u + 3]), "r"(v[u + 4]),
                         "r"(v[u + 5]), "r"(v[u + 6]), "r"(v[u + 7])
                         : "memory");
      } else if (out) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (c0 + 8 * u >= p.d) break;
          uint32_t x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = pack_bf16(__uint_as_float(v[8 * u + 2 * i]) * inv, __uint_as_float(v[8 * u + 2 * i + 1]) * inv);
          *(uint4*)(dst + c0 + 8 * u) = make_uint4(x[0], x[1], x[2], x[3]);
        }
      }
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  // ---- the blocks' shares ----
  constexpr int LD = D + 4;
  static_assert((size_t)NQ * 128 * LD * 4 <= NQ * Q_BYTES + 2 * KS * KV_BYTES, "the outputs lie over the tiles");
  float* const part = (float*)gen;  // [NQ][128][LD] outputs of this block, for the cluster
  __shared__ float part_m[NQ * 128], part_l[NQ * 128];
  if (p.slices > 1) {
    if (warp >= 4) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int x = tid - 128, q = warp & 3;
      const uint32_t o_addr = tmem_base + (uint32_t)(x >> 7) * TILE_COLS + ((uint32_t)(q * 32) << 16) + 2 * KT;
      part_m[x] = m;
      part_l[x] = l;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t v[32];
        ld32(o_addr + c0, v);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *(uint4*)(part + x * LD + c0 + i) = l != 0.f ? make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]) : make_uint4(0u, 0u, 0u, 0u);  // (without tiles nothing was written)
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(NCOLS) : "memory");
  }
  if (p.slices == 1) {
    if (OWN && last_block()) dependency();
    return;
  }
  __shared__ float weight[4][NQ * 128];  // of the blocks' outputs of a row
  cluster_sync_all();
  if (tid < NQ * 128) {
    float ms[4], ls[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      ms[s] = s < p.slices ? ld_cluster_f32(smem_u32(&part_m[tid]), (uint32_t)s) : -INFINITY;
      ls[s] = s < p.slices ? ld_cluster_f32(smem_u32(&part_l[tid]), (uint32_t)s) : 0.f;
    }
    const float top = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])), at = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      ms[s] = fast_exp2(ms[s] - at);
      sum = fmaf(ls[s], ms[s], sum);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) weight[s][tid] = PART ? ms[s] : sum != 0.f ? ms[s] / sum : 0.f;
    if (PART && slice == 0) {
      const int r = tid & 127;
      const int64_t ti = i0 + (tid >> 7) * p.per + r / p.rep;
      if (r < p.per * p.rep && ti < n) p.sh.ml[((int64_t)chunk * p.rows.M + tok0 + ti) * p.nh + kvh * p.rep + r % p.rep] = make_float2(top, sum);
    }
  }
  __syncthreads();
  constexpr int U = 4;  // values of a thread on their way, 4 columns each
  const int step = (int)blockDim.x * p.slices;
  for (int i = slice * (int)blockDim.x + tid; i < NQ * 128 * (D / 4); i += U * step) {
    float4 os[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        os[u][s] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int k = i + u * step;
        if (s < p.slices && k < NQ * 128 * (D / 4)) {
          uint32_t at;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(part + k / (D / 4) * LD + k % (D / 4) * 4)), "r"(s));
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(os[u][s].x), "=f"(os[u][s].y), "=f"(os[u][s].z), "=f"(os[u][s].w) : "r"(at));
        }
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = i + u * step, x = k / (D / 4), c = k % (D / 4) * 4, r = x & 127;
      const int64_t ti = i0 + (x >> 7) * p.per + r / p.rep;
      if (k >= NQ * 128 * (D / 4) || r >= p.per * p.rep || ti >= n || c >= p.d) continue;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const float f = weight[s][x];
        v.x = fmaf(os[u][s].x, f, v.x); v.y = fmaf(os[u][s].y, f, v.y); v.z = fmaf(os[u][s].z, f, v.z); v.w = fmaf(os[u][s].w, f, v.w);
      }
      const int64_t at = ((tok0 + ti) * p.nh + kvh * p.rep + r % p.rep) * (int64_t)p.d + c;
      if (PART) *(float4*)(p.sh.out + (int64_t)chunk * p.rows.M * p.nh * p.d + at) = v;
      else *(uint2*)(p.out + at) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    }
  }
  cluster_sync_all();
  if (OWN && last_block()) dependency();
}

// q as [tokens, heads, d] in boxes of [per tokens, rep heads, 64 components]
int make_q_map(cg_ctx* c, CUtensorMap* map, const PagedAttnArgs& a, int per, int rep) {
  cuuint64_t gdim[3] = {(cuuint64_t)a.d, (cuuint64_t)a.nh, (cuuint64_t)a.rows.M};
  cuuint64_t gstr[2] = {(cuuint64_t)a.q_hs * 2, (cuuint64_t)a.q_ld * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)rep, (cuuint32_t)per};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = ((EncodeTiledFn)c->encode_tiled)(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), gdim, gstr, box, estr,
                                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(c, CG_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return CG_OK;
}

// How a kernel is set up: once per device, and its arguments.
template <int D, int NQ, bool CAP, int MODE>
int configure(cg_ctx* c, const PagedAttnArgs& a, FaArgs* out, CUtensorMap* mq, CUtensorMap* mk, CUtensorMap* mv) {
  constexpr size_t smem = fa_smem<D, NQ>();
  static PerDeviceFlag configured_on;
  bool& configured = configured_on.at(c->core->device);
  if (!configured) {
    CG_CUDA(c, cudaFuncSetAttribute(k_paged_fa<D, NQ, CAP, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured = true;
  }
  FaArgs& p = *out;
  p.rows = a.rows;
  p.sh = a.sh;
  p.out = (__nv_bfloat16*)a.out;
  p.most = a.most;
  p.window = a.window;
  p.pool_rows = (a.rows.n_pages * a.nkv) << a.rows.lg;
  p.nh = a.nh; p.nkv = a.nkv;
  p.rep = a.nh / a.nkv;
  p.per = 128 / p.rep;
  p.d = a.d;
  p.scale_log2e = a.scale * LOG2E;
  p.cap_log2e = p.cap_unit = p.cap_in = 0.f;
  for (float& f : p.cap_poly) f = 0.f;
  p.lag = std::min(LAG / p.scale_log2e, 1e38f);
  if (CAP) {
    p.cap_log2e = a.cap * LOG2E;
    p.cap_unit = -2.f * p.scale_log2e / a.cap;
    for (int i = 0; i < 6; ++i) p.cap_poly[i] = p.cap_log2e * tanh_term(i);
    p.cap_in = a.scale / a.cap;
  }
  const int box = std::min(1 << a.rows.lg, KT);
  CG_TRY(make_map(c, mk, a.k_pages, p.pool_rows, a.d, a.d, box));
  CG_TRY(make_map(c, mv, a.v_pages, p.pool_rows, a.d, a.d, box));
  return make_q_map(c, mq, a, p.per, p.rep);
}

template <int D, int NQ, bool CAP, int MODE>
int launch(cg_ctx* c, const PagedAttnArgs& a) {
  constexpr size_t smem = fa_smem<D, NQ>();
  FaArgs p;
  CUtensorMap mq, mk, mv;
  CG_TRY((configure<D, NQ, CAP, MODE>(c, a, &p, &mq, &mk, &mv)));
  const int64_t tiles = (a.most + (int64_t)NQ * p.per - 1) / ((int64_t)NQ * p.per), width = a.rows.cols << a.rows.lg, longest = MODE == OWN ? a.sh.own(width) : width;
  // Shares of the keys (of several rows four fifths of the tiles count: they differ).  Us with 1 / 2 / 4, [the rule's]:
  //   6 rows of 480 behind 3720, 4 x 2 heads of 256, window 4096    182  [157]  187
  //   1 of 63 behind 2937, the same, no window                     61.6   38.0 [24.6]
  //   1 of 49 behind 3951, 8 x 4 heads of 128                      65.5   40.8 [26.0]
  //   1 of 2000, the same                                         [59.7]  71.5  118
  //   4 of 300 behind 1700, the same                              [72.1]  75.7  94
  //   3 of 200 behind 8800, heads of 64                            139    145  [124]
  // (The table's width stands for the lengths, and 4 shares of a short tile of queries leave SMs idle: the second and third rows' bytes take 2 to 3 us.)
  static AtATime known;
  const int64_t clusters = tiles * a.nkv * a.rows.rows;
  p.slices = pick_shares([&](int i) { return at_a_time(known, c->core->device, i, k_paged_fa<D, NQ, CAP, MODE>, NQ == 2 ? 384 : 256, smem); }, 4,
                         a.rows.rows > 1 ? std::max<int64_t>(clusters * 4 / 5, 1) : clusters, a.window > 0 ? std::min(longest, a.window + p.per * NQ) : longest, KT, 6.,
                         D == 256 ? 1.25 : NQ == 2 ? 1.1 : 0.9, 0.);
  CG_CUDA(c, launch_kernel(c, k_paged_fa<D, NQ, CAP, MODE>, dim3((unsigned)(tiles * p.slices), (unsigned)a.nkv, (unsigned)a.rows.rows), dim3(NQ == 2 ? 384 : 256), smem, -p.slices,
                           mq, mk, mv, p));
  CG_LAUNCHED(c);
  return CG_OK;
}

template <int D>
int pick(cg_ctx* c, const PagedAttnArgs& a) {
  const bool cap = a.cap > 0.f;
  if constexpr (D <= 128) {
    const int per = 128 / (a.nh / a.nkv);
    if (a.most > per) return cap ? launch<D, 2, true, ALL>(c, a) : launch<D, 2, false, ALL>(c, a);
  }
  return cap ? launch<D, 1, true, ALL>(c, a) : launch<D, 1, false, ALL>(c, a);
}

// ---- shared keys ----

// (Two tiles of queries that share their keys in a block are no faster here: 64 rows over 16001 keys, heads of 128, 62 us where one took 60.5, and
// a group's second tile is often all but empty.)
int64_t prefix_tiles(const PagedAttnArgs& a) {
  const int64_t tokens = 128 / (a.nh / a.nkv);
  return (a.rows.M + a.sh.groups.n * (tokens - 1)) / tokens;  // (a group's last one may not be full)
}
template <int D, bool CAP>
int launch_prefix(cg_ctx* c, const PagedAttnArgs& a) {
  FaArgs p;
  CUtensorMap mq, mk, mv;
  CG_TRY((configure<D, 1, CAP, CHUNK>(c, a, &p, &mq, &mk, &mv)));
  p.slices = 1;
  const int64_t blocks = prefix_tiles(a) * a.sh.chunks;
  if (blocks > 0x7FFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "too many tokens");
  CG_CUDA(c, launch_kernel(c, k_paged_fa<D, 1, CAP, CHUNK>, dim3((unsigned)blocks, (unsigned)a.nkv), dim3(256), fa_smem<D, 1>(), 1, mq, mk, mv, p));
  CG_LAUNCHED(c);
  return CG_OK;
}
template <int D>
int pick_prefix(cg_ctx* c, const PagedAttnArgs& a) { return a.cap > 0.f ? launch_prefix<D, true>(c, a) : launch_prefix<D, false>(c, a); }
template <int D>
int pick_own(cg_ctx* c, const PagedAttnArgs& a) {
  return a.cap > 0.f ? launch<D, 1, true, OWN>(c, a) : launch<D, 1, false, OWN>(c, a);  // (a row's tokens do not fill a tile)
}

}  // namespace

bool paged_fa_supported(const PagedAttnArgs& a) {
  const int64_t rep = a.nh / a.nkv;
  return rep <= 128 && a.most > 1 && a.most * rep > 16 && a.nkv <= 65535 &&
         ((a.rows.n_pages * a.nkv) << a.rows.lg) < 0x7FFFFFFFll && ((uintptr_t)a.q % 16) == 0 && ((uintptr_t)a.out % 16) == 0 && a.q_ld % 8 == 0 &&
         a.q_hs % 8 == 0 && a.q_ld > 0 && a.q_hs > 0 && a.q_ld < (1ll << 38) && a.q_hs < (1ll << 38);
}

int paged_fa(cg_ctx* c, const PagedAttnArgs& a) {
  if (a.d <= 64) return pick<64>(c, a);
  if (a.d <= 128) return pick<128>(c, a);
  return pick<256>(c, a);
}

bool paged_fa_prefix_supported(const PagedAttnArgs& a) {
  return a.nh / a.nkv <= 128 && ((a.rows.n_pages * a.nkv) << a.rows.lg) < 0x7FFFFFFFll && ((uintptr_t)a.q % 16) == 0 && a.q_ld % 8 == 0 && a.q_hs % 8 == 0 && a.q_ld > 0 &&
         a.q_hs > 0 && a.q_ld < (1ll << 38) && a.q_hs < (1ll << 38);
}
int paged_fa_prefix(cg_ctx* c, const PagedAttnArgs& a) {
  if (a.d <= 64) return pick_prefix<64>(c, a);
  if (a.d <= 128) return pick_prefix<128>(c, a);
  return pick_prefix<256>(c, a);
}
int paged_fa_own(cg_ctx* c, const PagedAttnArgs& a) {
  if (a.d <= 64) return pick_own<64>(c, a);
  if (a.d <= 128) return pick_own<128>(c, a);
  return pick_own<256>(c, a);
}
// Keys of a chunk: as many chunks as make a block per SM, or 1.4 where two fit (the rows' own keys then run beside them), in one wave however the
// tokens are dealt to the groups.  Us with 1 / 1.25 / 1.4 / 1.5 / 2 on an SM:
//   64 rows of 1 behind 16001, 8 key heads of 128              57.1  55.9 [56.4] 57.5  62.3
//   30 of up to 5 in 3 groups behind 4003, 4 of 128            38.0  35.8 [36.2] 36.3  39.5
//   14 of 5 in 4 groups behind 3588, 8 of 128                  31.0  26.7 [26.0] 26.0  24.1
//   26 of 1 behind 13661, 4 of 128                             26.0  27.2 [26.5] 27.1  28.2
int64_t paged_fa_slots(const PagedAttnArgs& a) { return a.d <= 128 ? 204 : 148; }
int64_t paged_fa_chunk(const PagedAttnArgs& a) {
  const int64_t slots = paged_fa_slots(a), queries = a.rows.M * (a.nh / a.nkv), tiles = std::max<int64_t>((queries + a.sh.groups.n * 127) / 128, 1) * a.nkv;
  const int64_t chunks = std::max<int64_t>(slots / tiles, 1), keys = (a.sh.groups.most + chunks - 1) / chunks;
  return std::max<int64_t>((keys + KT - 1) / KT * KT, SHARED_CHUNK);
}

}  // namespace cg
