// paged_dec.cu — attention of a few tokens per row over a paged cache in bf16: the form of decode steps.
//
// The query rows of a key head (token x / rep, head x % rep of the group) fill the rows of one mma.sync tile, 8 or
// 16 at a time, so a key is read once for all of them.  A cluster has a row's keys and a key head; its blocks have equal
// shares of the keys, a block's W warps every W-th tile of KT keys, each through a ring of its own that TMA fills.
//   S [rows, keys] = Q K^T     (Q's fragments stay in registers)
//   O^T [d, rows] += V^T P^T   (S's accumulators are P^T's fragments; 8 rows fill the 8 columns)
// What bounds it is the bytes of the cache, and for short contexts the chain tables -> page table -> keys -> product -> joining.
//
// 7 rows of up to 32002 tokens, 32 heads and 8 key heads of 128: 623 MB in 100 us, 6.2 TB/s, 0.95 of a copy.  8 rows of 578, heads of 64:
// 6.4 us (7.4 while a page's number was waited for before the next one was asked for, and one block of a cluster joined all).  A warp per
// query with plain loads: 1194 and 36.7 us.
//
// Probabilities are split into two bf16 parts (the second product costs nothing where bytes bound the kernel), so that the output is
// rounded once.  Exponents' references lag behind the maxima by up to 2^8, so that tiles need no shuffles.
#include <algorithm>

#include "mma.cuh"
#include "paged_attn.h"
#include "tc_common.cuh"

namespace cg {

namespace {

using namespace tc;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LAG = 8.f;

struct DecArgs {
  PagedRows rows;
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  int64_t q_ld, q_hs, most, window, pool_rows;
  int nh, nkv, rep, d;
  float scale_log2e, cap_log2e, cap_in, cap_unit;
  SharedParts sh;
};

// Keys of a warp's tile, tiles of its ring, warps.  (Four warps of heads of 256 fill an SM; two blocks of two deal rows of different lengths out more evenly: 14 rows behind
// 3001 tokens, 4 key heads of 256, window, 41.3 us with four, 39.2 with two, 39.2 with one.  Rows that read all their keys keep four.)
template <int D>
__host__ __device__ constexpr int dec_keys() { return D == 64 ? 32 : 16; }
constexpr int RING = 3;
template <int D, int MODE>
__host__ __device__ constexpr int dec_warps() { return MODE == OWN && D == 256 ? 2 : 4; }
template <int D, int MODE>
__host__ __device__ constexpr size_t dec_ring() { return (size_t)dec_warps<D, MODE>() * RING * 2 * dec_keys<D>() * D * 2; }
template <int D, int MODE>
__host__ __device__ constexpr size_t dec_smem() { return 1024 + dec_ring<D, MODE>() + dec_warps<D, MODE>() * RING * 8; }

template <int D, int ROWS, bool CAP, int MODE>
__global__ void __launch_bounds__(dec_warps<D, MODE>() * 32)
k_paged_dec(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, DecArgs p) {
  constexpr bool OWN = MODE == KeysOf::OWN;
  constexpr int KT = dec_keys<D>(), SUB = D / 64, NB = ROWS / 8, KS = D / 16, LD = D + 4, W = dec_warps<D, MODE>();
  constexpr uint32_t BOX = KT * 128, TILE = SUB * BOX;  // bytes of 64 components, of a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ float red_m[W][ROWS], red_l[W][ROWS], cta_m[ROWS], cta_l[ROWS];
  __shared__ int aborted;
  static_assert((size_t)W * ROWS * LD * 4 + (size_t)ROWS * LD * 4 <= dec_ring<D, MODE>(), "the warps' outputs lie over the ring");
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  float* red_o = (float*)(smem_raw + (base - raw));       // [W][ROWS][LD]
  float* part = red_o + W * ROWS * LD;                    // [ROWS][LD]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t2 = (lane & 3) * 2;
  const uint32_t ring = base + warp * (RING * 2 * TILE), bars = base + (uint32_t)dec_ring<D, MODE>() + warp * (RING * 8);
  if (lane == 0)
    for (int i = 0; i < RING; ++i) mbar_init(bars + 8 * i, 1);
  if (tid == 0) aborted = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  // (query rows fit into 31 bits, and the blocks of a cluster are a power of two)
  const uint32_t kvh = blockIdx.x % (uint32_t)p.nkv, x0 = blockIdx.x / (uint32_t)p.nkv * ROWS, rep = (uint32_t)p.rep;
  const uint32_t i0 = x0 / rep, i_end = (x0 + ROWS - 1) / rep;
  const int64_t row = blockIdx.y;
  const int slices = (int)gridDim.z, slice = (int)blockIdx.z, lg_slices = 31 - __clz(slices);
  const int lg = p.rows.lg, box = min(1 << lg, KT), parts = KT / box;
  const int my_part = lane % parts, my_sub = lane / parts % SUB, my_pool = lane / (parts * SUB);  // (keys, values; others have nothing)
  auto depend = []() { asm volatile("griddepcontrol.wait;" ::: "memory"); };
  if (!OWN) depend();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  int64_t tok0, n, len;
  int64_t from = 0, group = -1;  // OWN: the first key, the row's group
  if (OWN) group = group_of_row(p.sh.groups, row, &from);
  if (!row_span(p.rows, row, p.most, &tok0, &n, &len) || x0 >= n * rep) {  // (the same in all blocks of a cluster)
    if (OWN && last_block()) depend();
    return;
  }
  const int64_t pos0 = len - n, i1 = min(n - 1, (int64_t)i_end);
  const int64_t hi = pos0 + i1, lo = max(p.window > 0 ? max((int64_t)0, pos0 + i0 - p.window + 1) : 0, OWN ? min(from, hi + 1) : 0);
  const int64_t first = (int64_t)((uint64_t)lo / KT), tiles = (int64_t)((uint64_t)hi / KT) + 1 - first, share = (tiles + slices - 1) >> lg_slices;
  const int64_t end = min(first + tiles, first + (slice + 1) * share);

  // A lane has a box of a tile: 64 components of a page's keys or values (of the whole tile's, if pages are longer).  Pages without a
  // visible key are not looked up and read as zeros (a box behind the pool's end).
  const int off_end = (int)p.pool_rows;
  const uint32_t* pages = p.rows.table + row * p.rows.cols;
  // (asked for apart from what is made of it: several are on their way at once)
  auto ask = [&](int64_t t) {
    const int64_t key = t * KT + my_part * box;
    return t < end && key <= hi && key + box > lo ? (int64_t)pages[key >> lg] : (int64_t)-1;
  };
  auto place = [&](int64_t t, int64_t id) {
    if (id >= p.rows.n_pages) {
      *p.rows.err = DEV_INDEX;
      id = -1;
    }
    return id < 0 ? off_end : (int)(((id * p.nkv + kvh) << lg) + ((t * KT + my_part * box) & ((1 << lg) - 1)));
  };
  auto request = [&](int stage, int at) {
    const uint32_t bar = bars + 8 * stage;
    if (lane == 0) mbar_expect_tx(bar, 2 * TILE);
    __syncwarp();
    if (my_pool < 2)
      tma_load_2d(ring + stage * (2 * TILE) + my_pool * TILE + my_sub * BOX + my_part * box * 128, my_pool ? &map_v : &map_k, my_sub * 64, at, bar);
  };
  int64_t t = first + slice * share + warp;
  int64_t ahead_id;  // page of the tile that is asked for next
  {
    int64_t id[RING + 1];
#pragma unroll
    for (int i = 0; i <= RING; ++i) id[i] = ask(t + W * i);
#pragma unroll
    for (int i = 0; i < RING; ++i)
      if (t + W * i < end) request(i, place(t + W * i, id[i]));
    ahead_id = id[RING];
  }

  // rows g and g + 8 of the tile
  uint32_t qf[KS][2 * NB];
  int64_t qpos[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t x = x0 + g + 8 * b, i = x / rep;
    const bool there = x < n * rep;
    qpos[b] = pos0 + i;
    const __nv_bfloat16* src = p.q + (tok0 + (there ? i : 0u)) * p.q_ld + (int64_t)(kvh * rep + (there ? x - i * rep : 0u)) * p.q_hs;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int c = k * 16 + t2;
      qf[k][b] = there && c < p.d ? *(const uint32_t*)(src + c) : 0u;
      qf[k][NB + b] = there && c + 8 < p.d ? *(const uint32_t*)(src + c + 8) : 0u;
    }
  }
  float o[KS][NB][4], m[NB], l[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    m[b] = -INFINITY;
    l[b] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) o[k][b][0] = o[k][b][1] = o[k][b][2] = o[k][b][3] = 0.f;
  }
  // ldmatrix: lane's key and 16-byte piece within 16 keys x 16 components
  const int lkey = (lane >> 4) * 8 + (lane & 7), lpiece = (lane >> 3) & 1;
  bool ok = true;
  int it = 0;
  for (; t < end; t += W, ++it) {
    const int stage = it % RING;
    const int64_t ahead = t + W * RING;
    const int64_t next = ask(ahead + W);  // (a whole round before it is asked for)
    ok = __all_sync(0xffffffffu, mbar_wait(bars + 8 * stage, (uint32_t)(it / RING) & 1u, &aborted, p.rows.err));
    if (!ok) break;
    const uint32_t kt = ring + stage * (2 * TILE), vt = kt + TILE;
    const int64_t k0 = t * KT;
    if (k0 + KT - 1 > hi) {
      // the values behind the last visible key are nobody's: a probability of 0 times an infinity would not be 0.  (The row's last
      // tile: nothing is loaded over it.)
      for (int i = lane; i < SUB * (int)(k0 + KT - 1 - hi) * 8; i += 32) {
        const int rows = (int)(k0 + KT - 1 - hi), s = i / (rows * 8), x = i - s * rows * 8;
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vt + s * BOX + (uint32_t)(KT - rows) * 128u + (uint32_t)x * 16u), "r"(0) : "memory");
      }
      __syncwarp();
    }
    float s[KT / 8][4], s2[KT / 8][4];  // (even and odd 16 components: two shorter chains)
#pragma unroll
    for (int i = 0; i < KT / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = s2[i][0] = s2[i][1] = s2[i][2] = s2[i][3] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < KT / 16; ++i) {
        const int key = i * 16 + lkey, piece = (k * 2 + lpiece) & 7;
        uint32_t b0, b1, b2, b3;
        ldsm_x4(kt + (k / 4) * BOX + key * 128 + ((piece ^ (key & 7)) << 4), b0, b1, b2, b3);
        float (*to)[4] = k & 1 ? s2 : s;
        mma_bf16(to[2 * i], qf[k][0], NB == 2 ? qf[k][1] : 0u, qf[k][NB], NB == 2 ? qf[k][NB + 1] : 0u, b0, b1);
        mma_bf16(to[2 * i + 1], qf[k][0], NB == 2 ? qf[k][1] : 0u, qf[k][NB], NB == 2 ? qf[k][NB + 1] : 0u, b2, b3);
      }
#pragma unroll
    for (int i = 0; i < KT / 8; ++i)
#pragma unroll
      for (int e = 0; e < 2 * NB; ++e) s[i][e] += s2[i][e];
    const bool masked = k0 + KT - 1 > pos0 + i0 || (p.window > 0 && k0 <= hi - p.window) || (OWN && k0 < from);
    float top[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) top[b] = -INFINITY;
#pragma unroll
    for (int i = 0; i < KT / 8; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[i][2 * b + e];
          if (CAP) x = soft_cap(x, p.cap_log2e, p.cap_in, p.cap_unit);
          else x *= p.scale_log2e;
          if (masked) {
            const int64_t key = k0 + i * 8 + t2 + e;
            if (key > qpos[b] || (p.window > 0 && key <= qpos[b] - p.window) || (OWN && key < from)) x = -INFINITY;
          }
          top[b] = fmaxf(top[b], x);
        }
    bool grown = false;
#pragma unroll
    for (int b = 0; b < NB; ++b) grown = grown || top[b] > m[b] + LAG;
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float w = fmaxf(top[b], __shfl_xor_sync(0xffffffffu, top[b], 1));
        w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 2));
        const float m_new = fmaxf(m[b], w), corr = m_new == -INFINITY ? 1.f : fast_exp2(m[b] - m_new);
        m[b] = m_new;
        l[b] *= corr;
        const float c0 = __shfl_sync(0xffffffffu, corr, t2 * 4), c1 = __shfl_sync(0xffffffffu, corr, t2 * 4 + 4);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          o[k][b][0] *= c0; o[k][b][1] *= c1;
          o[k][b][2] *= c0; o[k][b][3] *= c1;
        }
      }
    }
    uint32_t ph[KT / 8][NB], pl[KT / 8][NB];  // probabilities, and what their rounding left
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float mc = m[b] == -INFINITY ? 0.f : m[b];
#pragma unroll
      for (int i = 0; i < KT / 8; ++i) {
        const float e0 = fast_exp2(s[i][2 * b] - mc), e1 = fast_exp2(s[i][2 * b + 1] - mc);
        l[b] += e0 + e1;
        ph[i][b] = pack_bf16(e0, e1);
        pl[i][b] = pack_bf16(e0 - __uint_as_float(ph[i][b] << 16), e1 - __uint_as_float(ph[i][b] & 0xffff0000u));
      }
    }
#pragma unroll
    for (int i = 0; i < KT / 16; ++i)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int key = i * 16 + lkey, piece = (k * 2 + lpiece) & 7;
        uint32_t a0, a1, a2, a3;
        ldsm_x4_t(vt + (k / 4) * BOX + key * 128 + ((piece ^ (key & 7)) << 4), a0, a1, a2, a3);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          mma_bf16(o[k][b], a0, a1, a2, a3, ph[2 * i][b], ph[2 * i + 1][b]);
          mma_bf16(o[k][b], a0, a1, a2, a3, pl[2 * i][b], pl[2 * i + 1][b]);
        }
      }
    __syncwarp();
    if (ahead < end) request(stage, place(ahead, ahead_id));
    ahead_id = next;
  }
  if (!ok) {  // copies on their way are waited for: what lies over the ring is written next
    for (int i = 0; i < RING && t + W * i < end; ++i) mbar_drain(bars + 8 * ((it + i) % RING), (uint32_t)((it + i) / RING) & 1u, p.rows.err);
    aborted = 1;
  }

  // ---- the warps' shares ----
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    l[b] += __shfl_xor_sync(0xffffffffu, l[b], 1);
    l[b] += __shfl_xor_sync(0xffffffffu, l[b], 2);
    if (t2 == 0) { red_m[warp][g + 8 * b] = m[b]; red_l[warp][g + 8 * b] = l[b]; }
  }
  __syncthreads();  // (all rings are empty, or given up on)
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) red_o[(warp * ROWS + b * 8 + t2 + (e & 1)) * LD + k * 16 + g + (e >> 1) * 8] = o[k][b][e];
  __syncthreads();
  auto out_at = [&](uint32_t x) { return p.out + ((tok0 + x / rep) * p.nh + kvh * rep + x % rep) * (int64_t)p.d; };
  auto put_part = [&](uint32_t x, int c, float top, float sum, float4 v) {
    const int64_t at = ((int64_t)p.sh.chunks * p.rows.M + tok0 + x / rep) * p.nh + kvh * rep + x % rep;
    *(float4*)(p.sh.out + at * p.d + c) = v;
    if (c == 0) p.sh.ml[at] = make_float2(top, sum);
  };
  for (int i = tid; i < ROWS * (D / 4); i += W * 32) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float top = red_m[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, red_m[w][r]);
    const float mc = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = fast_exp2(red_m[w][r] - mc);
      const float4 u = *(const float4*)(red_o + (w * ROWS + r) * LD + c);
      sum += red_l[w][r] * f;
      v.x = fmaf(u.x, f, v.x); v.y = fmaf(u.y, f, v.y); v.z = fmaf(u.z, f, v.z); v.w = fmaf(u.w, f, v.w);
    }
    if (slices > 1) {
      *(float4*)(part + r * LD + c) = v;
      if (c == 0) { cta_m[r] = top; cta_l[r] = sum; }
    } else if (x0 + r < n * rep && c < p.d && !aborted) {
      const float f = sum > 0.f ? 1.f / sum : 0.f;
      if (OWN) put_part(x0 + r, c, top, sum, v);
      else *(uint2*)(out_at(x0 + r) + c) = make_uint2(pack_bf16(v.x * f, v.y * f), pack_bf16(v.z * f, v.w * f));
    }
  }
  if (slices == 1) {
    if (OWN && last_block()) depend();
    return;
  }

  // ---- the blocks' shares: each finishes some of the values ----
  cluster_sync_all();
  const int rows = (int)min((int64_t)ROWS, n * rep - x0);
  for (int i = tid * slices + slice; i < rows * (D / 4); i += W * 32 * slices) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    // (four shares on their way at a time)
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < slices; s0 += 4) {
      float ms[4], ls[4];
      float4 us[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        ms[s] = -INFINITY;
        ls[s] = 0.f;
        us[s] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s0 + s < slices) {
          uint32_t at;
          ms[s] = ld_cluster_f32(smem_u32(&cta_m[r]), (uint32_t)(s0 + s));
          ls[s] = ld_cluster_f32(smem_u32(&cta_l[r]), (uint32_t)(s0 + s));
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(part + r * LD + c)), "r"(s0 + s));
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(us[s].x), "=f"(us[s].y), "=f"(us[s].z), "=f"(us[s].w) : "r"(at) : "memory");
        }
      }
      const float before = top;
      top = fmaxf(fmaxf(fmaxf(top, ms[0]), fmaxf(ms[1], ms[2])), ms[3]);
      const float mc = top == -INFINITY ? 0.f : top, f0 = fast_exp2(before - mc);
      sum *= f0;
      v.x *= f0; v.y *= f0; v.z *= f0; v.w *= f0;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const float f = fast_exp2(ms[s] - mc);
        sum = fmaf(ls[s], f, sum);
        v.x = fmaf(us[s].x, f, v.x); v.y = fmaf(us[s].y, f, v.y); v.z = fmaf(us[s].z, f, v.z); v.w = fmaf(us[s].w, f, v.w);
      }
    }
    if (c < p.d && !aborted) {
      const float f = sum > 0.f ? 1.f / sum : 0.f;
      if (OWN) put_part(x0 + r, c, top, sum, v);
      else *(uint2*)(out_at(x0 + r) + c) = make_uint2(pack_bf16(v.x * f, v.y * f), pack_bf16(v.z * f, v.w * f));
    }
  }
  cluster_sync_all();
  if (OWN && last_block()) depend();
}

template <int D, int ROWS, bool CAP, int MODE>
int launch(cg_ctx* c, const PagedAttnArgs& a) {
  constexpr size_t smem = dec_smem<D, MODE>();
  constexpr int W = dec_warps<D, MODE>();
  static PerDeviceFlag configured_on;
  bool& configured = configured_on.at(c->core->device);
  if (!configured) {
    CG_CUDA(c, cudaFuncSetAttribute(k_paged_dec<D, ROWS, CAP, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    CG_CUDA(c, cudaFuncSetAttribute(k_paged_dec<D, ROWS, CAP, MODE>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    configured = true;
  }
  DecArgs p;
  p.rows = a.rows;
  p.sh = a.sh;
  p.q = (const __nv_bfloat16*)a.q;
  p.out = (__nv_bfloat16*)a.out;
  p.q_ld = a.q_ld; p.q_hs = a.q_hs;
  p.most = a.most;
  p.window = a.window;
  p.pool_rows = (a.rows.n_pages * a.nkv) << a.rows.lg;
  p.nh = a.nh; p.nkv = a.nkv; p.rep = a.nh / a.nkv; p.d = a.d;
  p.scale_log2e = a.scale * LOG2E;
  p.cap_log2e = p.cap_in = p.cap_unit = 0.f;
  if (CAP) {
    p.cap_log2e = a.cap * LOG2E;
    p.cap_in = a.scale / a.cap;
    p.cap_unit = -2.f * p.scale_log2e / a.cap;
  }
  CUtensorMap mk, mv;
  const int box = std::min(1 << a.rows.lg, dec_keys<D>());
  CG_TRY(make_map(c, &mk, a.k_pages, p.pool_rows, a.d, a.d, box));
  CG_TRY(make_map(c, &mv, a.v_pages, p.pool_rows, a.d, a.d, box));
  const int64_t groups = (a.most * p.rep + ROWS - 1) / ROWS * a.nkv, width = a.rows.cols << a.rows.lg, longest = MODE == OWN ? a.sh.own(width) : width;
  // Shares of the keys.  Us with 1 / 2 / 4 / 8 / 16, [the rule's]:
  //   8 rows x 8 key heads, 578 keys, d 64      7.9   7.4 [6.5]  11.0  27.5
  //   8 x 8, 2000, d 128                       29.9  19.3 [15.9] 22.1  39.6
  //   1 x 8, 4096, d 128                       53.8  30.3  17.6  11.4 [9.7]
  //   1 x 8, 32000, d 128                      410   211   108   57.7 [37.3]
  //   32 x 8, 530, d 128                      [15.7] 23.5  31.7  53.6  119
  //   4 x 4, 2080, d 256                       39.8  23.7 [15.2] 20.9  25.7
  //   12 x 4, 167, d 256                        7.5 [7.9]  12.7  24.8  47.7
  // (Lengths are on the device, so the table's width stands for them: 32 x 8 rows of 530 with columns for 32768 tokens get 2 shares, 23.4 us.)
  static AtATime known;
  const int slices = pick_shares([&](int i) { return at_a_time(known, c->core->device, i, k_paged_dec<D, ROWS, CAP, MODE>, W * 32, smem); }, 16, groups * a.rows.rows, longest,
                                 W * dec_keys<D>(), 4., D == 64 ? 0.7 : D == 128 ? 0.75 : 1.25, 0.);
  CG_CUDA(c, launch_kernel(c, k_paged_dec<D, ROWS, CAP, MODE>, dim3((unsigned)groups, (unsigned)a.rows.rows, (unsigned)slices), dim3(W * 32), smem, slices, mk, mv, p));
  CG_LAUNCHED(c);
  return CG_OK;
}

template <int D, int MODE>
int pick(cg_ctx* c, const PagedAttnArgs& a) {
  const bool cap = a.cap > 0.f;
  if (a.most * (a.nh / a.nkv) <= 8) return cap ? launch<D, 8, true, MODE>(c, a) : launch<D, 8, false, MODE>(c, a);
  return cap ? launch<D, 16, true, MODE>(c, a) : launch<D, 16, false, MODE>(c, a);
}

}  // namespace

bool paged_dec_supported(const PagedAttnArgs& a) {
  return ((a.rows.n_pages * a.nkv) << a.rows.lg) < 0x7FFFFFFFll && (a.most * (a.nh / a.nkv) + 7) / 8 * a.nkv < 0x7FFFFFFFll && ((uintptr_t)a.q % 4) == 0 && a.most * (a.nh / a.nkv) < 0x7FFFFF00ll &&
         ((uintptr_t)a.out % 8) == 0 && a.q_ld % 2 == 0 && a.q_hs % 2 == 0;
}

int paged_dec(cg_ctx* c, const PagedAttnArgs& a) {
  if (a.d <= 64) return pick<64, ALL>(c, a);
  if (a.d <= 128) return pick<128, ALL>(c, a);
  return pick<256, ALL>(c, a);
}

int paged_dec_own(cg_ctx* c, const PagedAttnArgs& a) {
  if (a.d <= 64) return pick<64, OWN>(c, a);
  if (a.d <= 128) return pick<128, OWN>(c, a);
  return pick<256, OWN>(c, a);
}

}  // namespace cg
