// paged_attn.cu — causal attention of new tokens over a paged key/value cache:
//   o = sum_t softmax_t(cap tanh(scale q k_t / cap)) v_t   over   p - window < t <= p
// for a query at position p (catgrad-llm/src/models/llama.rs:97-108 after repeat_kv, helpers.rs:147-161), one pass over the
// keys with the running maximum and sum of the softmax in f32.
#include <algorithm>

#include "mma.cuh"
#include "paged_attn.h"

namespace cg {

namespace {

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* x) {
  const uint4 u = *(const uint4*)p;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store_as(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ float load_as(const float* p) { return *p; }
__device__ __forceinline__ float load_as(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// An f32 as the sum of two tf32 values of 11 bits, operands of the tensor cores.  The upper one is rounded to nearest (an infinity stays
// one, near the largest value it may become one), so that the lower one has either sign; of that the product reads the upper 11 bits.
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// f32, and bf16 that the other kernels do not take (its values are widened on the way in).  Operands are split into two parts of
// 11 bits, and three of the four products are summed in f32: what is left out is 2^-24 of a product.  The tensor cores cut sums off
// instead of rounding them, so sums over more than a tile are made outside.  Error against 64 bits, 3 rows of up to 1713
// tokens, heads of 64: 6.7e-7, of f32 sums 8.3e-7 (with one accumulator for all 2.1e-6, with parts cut off 3.1e-6).  On the
// CUDA cores the same tiles are bound by shared memory, eight vectors for 16 x 4 products of a thread: 43 us, here 29.8 (of which two blocks on
// an SM take 6700 clocks for a tile of each, 3000 of them for Q K^T: loads, splitting and products share the schedulers).
//
// A block has QR queries of one row and key head (query x is token x / rep, head x % rep of the group) and a share of the visible
// keys, GK at a time; its four warps share the rows (QR = 64) or the keys (QR = 16) of a tile, 16 rows each.  The blocks of a
// cluster share the keys and are joined through shared memory.  Tiles come by asynchronous copies, a ring of them ahead, their pages
// asked for before that.  Components, and columns, are dealt to the fragments so that a lane reads 16 bytes at a time and has eight
// neighbouring output values.  D: head size, rounded up to 64, 128 or 256.
template <int D, int QR>
struct Shape {
  static constexpr int GK = QR == 64 ? (D == 256 ? 16 : 32) : (D == 64 ? 128 : D == 128 ? 64 : 32);
  static constexpr int LK = D + 16, LV = D + 4;  // rows of keys (and queries), of values: conflict-free reads
  static constexpr int STAGE = GK * (LK + LV);   // floats of a tile
};
template <typename T>
constexpr int any_ring() { return sizeof(T) == 2 ? 1 : 2; }
template <typename T, int D, int QR>
constexpr size_t any_smem() {
  using S = Shape<D, QR>;
  const size_t ring = (size_t)any_ring<T>() * S::STAGE, joined = (size_t)(QR == 64 ? 64 : 80) * S::LV;
  return ((size_t)2 * QR * S::LK + (ring > joined ? ring : joined)) * 4;
}
template <typename T, int D, int QR, int MODE>
__global__ void __launch_bounds__(128) k_paged_attn(PagedAttnArgs a) {
  using S = Shape<D, QR>;
  constexpr int GK = S::GK, LK = S::LK, LV = S::LV, RING = any_ring<T>();
  constexpr int WK = QR == 64 ? 1 : 4, NT = GK / WK / 8;  // warps that share the keys, 8 keys of a warp
  constexpr int DG = D / 32;                             // 32 columns of the output
  extern __shared__ __align__(16) float sm[];
  float* qh = sm;                       // [QR][LK] upper and
  float* ql = qh + QR * LK;             // lower parts of the queries
  float* ring = ql + QR * LK;           // [RING] keys [GK][LK], values [GK][LV]
  float* part = ring;                   // behind the loop: the warps' outputs [4][16][LV] and, with WK = 4, the block's [16][LV]
  __shared__ float red[2][64], ml[2][QR];
  __shared__ int64_t places[2][GK];     // of the keys of the next tile to be asked for; -1: zeros
  auto depend = []() { asm volatile("griddepcontrol.wait;" ::: "memory"); };
  if (MODE != OWN) depend();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int rep = a.nh / a.nkv, kvh = (int)blockIdx.x % a.nkv;
  int64_t row = blockIdx.y, x0 = (int64_t)(blockIdx.x / a.nkv) * QR;
  const int slices = (int)gridDim.z, slice = (int)blockIdx.z;
  int64_t tok0, n, len, rows_of = 0, from = 0, group = -1;  // CHUNK: the group's rows; OWN: the first key, the group
  if constexpr (MODE == CHUNK) {
    GroupTile t;
    if (!group_of_tile(a.rows, a.sh.groups, blockIdx.x / a.nkv, rep, QR, &t) || (int64_t)blockIdx.y * a.sh.chunk >= t.shared) return;
    row = t.row0;
    rows_of = t.rows;
    tok0 = t.tok0;
    n = t.n;
    x0 = t.tile * QR;
    len = n + min(t.shared, ((int64_t)blockIdx.y + 1) * a.sh.chunk);  // (so that the keys end before it)
  } else {
    if constexpr (MODE == OWN) group = group_of_row(a.sh.groups, row, &from);
    if (!row_span(a.rows, row, a.most, &tok0, &n, &len) || x0 >= n * rep) {  // (the same in all blocks of a cluster)
      if (MODE == OWN && last_block()) depend();
      return;
    }
  }
  const int64_t pos0 = len - n, i0 = x0 / rep, i1 = min(n - 1, (x0 + QR - 1) / rep);
  const int64_t hi = MODE == CHUNK ? pos0 - 1 : pos0 + i1;
  const int64_t lo = MODE == CHUNK ? (int64_t)blockIdx.y * a.sh.chunk : max(a.window > 0 ? max((int64_t)0, pos0 + i0 - a.window + 1) : 0, MODE == OWN ? min(from, hi + 1) : 0);
  const int64_t first = lo / GK, tiles = hi / GK + 1 - first, per = (tiles + slices - 1) / slices;
  const int64_t t0 = first + slice * per, t1 = min(first + tiles, t0 + per);
  const int64_t page_mask = ((int64_t)1 << a.rows.lg) - 1;
  // By the first GK threads: the page of a key of tile t, asked for early and written down late.
  auto ask = [&](int64_t t) {
    const int64_t key = t * GK + tid;
    const bool seen = tid < GK && t < t1 && key >= lo && key <= hi;
    return seen ? (int64_t)a.rows.table[row * a.rows.cols + (key >> a.rows.lg)] : -1;
  };
  auto note = [&](int64_t t, int64_t page) {
    if (page >= a.rows.n_pages) {
      *a.rows.err = DEV_INDEX;
      page = -1;
    }
    if (tid < GK) places[t & 1][tid] = page < 0 ? -1 : (((page * a.nkv + kvh) << a.rows.lg) + ((t * GK + tid) & page_mask)) * a.d;
  };
  auto request = [&](int64_t t) {
    float* ks = ring + (int)((t - t0) % RING) * S::STAGE;
    float* vs = ks + GK * LK;
    if constexpr (sizeof(T) == 4) {
      if (t < t1)
        for (int i = tid; i < GK * (D / 4); i += 128) {
          const int r = i / (D / 4), c = i % (D / 4) * 4;
          const int64_t at = places[t & 1][r];
          const bool there = at >= 0 && c < a.d;
          const float* k = (const float*)a.k_pages + (there ? at + c : 0);
          const float* v = (const float*)a.v_pages + (there ? at + c : 0);
          cp_async16((uint32_t)__cvta_generic_to_shared(ks + r * LK + c), k, there ? 16 : 0);
          cp_async16((uint32_t)__cvta_generic_to_shared(vs + r * LV + c), v, there ? 16 : 0);
        }
      cp_async_commit();
    } else {
      for (int i = tid; i < GK * (D / 8); i += 128) {
        const int r = i / (D / 8), c = i % (D / 8) * 8;
        const int64_t at = places[t & 1][r];
        float kx[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, vx[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (at >= 0 && c < a.d) {
          load8((const T*)a.k_pages + at + c, kx);
          load8((const T*)a.v_pages + at + c, vx);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ks[r * LK + c + e] = kx[e];
          vs[r * LV + c + e] = vx[e];
        }
      }
    }
  };
  note(t0, ask(t0));
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) {  // (two tiles' places take turns)
    request(t0 + i);
    note(t0 + i + 1, ask(t0 + i + 1));
    __syncthreads();
  }
  for (int i = tid; i < QR * (D / 8); i += 128) {
    const int r = i / (D / 8), c = i % (D / 8) * 8;
    const int64_t x = x0 + r;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (x < n * rep && c < a.d) {
      const T* p = (const T*)a.q + (tok0 + x / rep) * a.q_ld + (kvh * rep + x % rep) * a.q_hs + c;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = load_as(p + e);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t h, l;
      split(v[e], h, l);
      qh[r * LK + c + e] = __uint_as_float(h);
      ql[r * LK + c + e] = __uint_as_float(l);
    }
  }
  // this lane's rows g and g + 8 of the warp's 16
  const int r0 = (QR == 64 ? warp * 16 : 0) + g, key0 = QR == 64 ? 0 : warp * (GK / 4);
  int64_t qpos[2] = {pos0 + (x0 + r0) / rep, pos0 + (x0 + r0 + 8) / rep};
  if constexpr (MODE == CHUNK)  // (a token stands where its row says)
#pragma unroll
    for (int q = 0; q < 2; ++q) qpos[q] = x0 + r0 + 8 * q < n * rep ? position_of(a.rows, row, rows_of, tok0 + (x0 + r0 + 8 * q) / rep) : hi;
  const float scale = a.scale * 1.4426950408889634f, cap2 = a.cap * 1.4426950408889634f, cap_in = a.cap > 0.f ? a.scale / a.cap : 0.f, cap_unit = -2.f * 1.4426950408889634f * cap_in;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[DG][4][4];
#pragma unroll
  for (int c = 0; c < DG; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[c][i][0] = o[c][i][1] = o[c][i][2] = o[c][i][3] = 0.f;
  for (int64_t t = t0; t < t1; ++t) {
    int64_t page;
    if constexpr (RING > 1) {
      cp_async_wait_group<RING - 2>();
      __syncthreads();  // tile t is there, and everyone is done with the one before
      request(t + RING - 1);
      page = ask(t + RING);
    } else {
      __syncthreads();
      request(t);
      __syncthreads();
      page = ask(t + 1);
    }
    const float* ks = ring + (int)((t - t0) % RING) * S::STAGE;
    const float* vs = ks + GK * LK;
    ks += key0 * LK;
    vs += key0 * LV;
    const int64_t k0 = t * GK + key0;
    float s[NT][4], less[NT][4];  // (the small products apart)
#pragma unroll
    for (int i = 0; i < NT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = less[i][0] = less[i][1] = less[i][2] = less[i][3] = 0.f;
#pragma unroll (D == 64 ? 4 : 2)
    for (int c = 0; c < D; c += 16) {  // components c + 4 t4 .. + 3: places t4 and t4 + 4 of two products
      uint32_t ah[2][4], al[2][4];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint4 h = *(const uint4*)(qh + (r0 + 8 * q) * LK + c + 4 * t4), w = *(const uint4*)(ql + (r0 + 8 * q) * LK + c + 4 * t4);
        ah[0][q] = h.x; ah[0][2 + q] = h.y; ah[1][q] = h.z; ah[1][2 + q] = h.w;
        al[0][q] = w.x; al[0][2 + q] = w.y; al[1][q] = w.z; al[1][2 + q] = w.w;
      }
      // (products with the same sum as far apart as there are sums)
      uint32_t h[NT][4], w[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float4 k = *(const float4*)(ks + (i * 8 + g) * LK + c + 4 * t4);
        split(k.x, h[i][0], w[i][0]); split(k.y, h[i][1], w[i][1]); split(k.z, h[i][2], w[i][2]); split(k.w, h[i][3], w[i][3]);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < NT; ++i) mma_tf32(less[i], al[u], h[i][2 * u], h[i][2 * u + 1]);
#pragma unroll
        for (int i = 0; i < NT; ++i) mma_tf32(s[i], ah[u], h[i][2 * u], h[i][2 * u + 1]);
#pragma unroll
        for (int i = 0; i < NT; ++i) mma_tf32(less[i], ah[u], w[i][2 * u], w[i][2 * u + 1]);
      }
    }
    // (scores and maxima in units of log2)
    const bool masked = MODE == CHUNK || k0 + GK / WK - 1 > pos0 + i0 || k0 < lo || (a.window > 0 && k0 <= hi - a.window);
    // (conditions stand around the loops: one per score would cut them up)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] += less[i][e];
    if (a.cap > 0.f) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = soft_cap(s[i][e], cap2, cap_in, cap_unit);
    } else {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] *= scale;
    }
    if (masked) {
      // key k0 + x is visible to row q iff low <= x <= lim
      int low[2], lim[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int64_t x = qpos[q] - k0, y = MODE == CHUNK ? min(x, hi - k0) : x;
        lim[q] = y > GK ? GK : y < -1 ? -1 : (int)y;
        low[q] = a.window > 0 ? (x - a.window >= GK ? GK : x - a.window < -1 ? 0 : (int)(x - a.window) + 1) : 0;
        if (MODE != ALL) low[q] = max(low[q], (int)min(max((MODE == OWN ? from : lo) - k0, (int64_t)0), (int64_t)GK));  // (chunks may begin inside a tile)
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = i * 8 + 2 * t4 + (e & 1);
          s[i][e] = x <= lim[e >> 1] && x >= low[e >> 1] ? s[i][e] : -INFINITY;
        }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[i][e]);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 1));
      top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 2));
      top[q] = fmaxf(top[q], m[q]);
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
      const float f0 = top[0] == -INFINITY ? 1.f : fast_exp2(m[0] - top[0]), f1 = top[1] == -INFINITY ? 1.f : fast_exp2(m[1] - top[1]);
      m[0] = top[0];
      m[1] = top[1];
      l[0] *= f0;
      l[1] *= f1;
#pragma unroll
      for (int c = 0; c < DG; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[c][i][0] *= f0; o[c][i][1] *= f0;
          o[c][i][2] *= f1; o[c][i][3] *= f1;
        }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
    // probabilities of 8 keys as they lie are the left operand whose places t4 and t4 + 4 are keys 2 t4 and 2 t4 + 1
    uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = fast_exp2(s[i][e] - base[e >> 1]);
        l[e >> 1] += x;
        split(x, ph[i][(e & 1) * 2 + (e >> 1)], pl[i][(e & 1) * 2 + (e >> 1)]);
      }
    // (a tile's sums begin at 0 and are added to the output by rounded additions: the tensor cores' own cut bits off, which over a
    // long row would lean one way)
#pragma unroll
    for (int c = 0; c < DG; ++c) {  // columns 32 c + 4 g + j are place g of product j
      float sum[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j][0] = sum[j][1] = sum[j][2] = sum[j][3] = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float4 v0 = *(const float4*)(vs + (i * 8 + 2 * t4) * LV + 32 * c + 4 * g), v1 = *(const float4*)(vs + (i * 8 + 2 * t4 + 1) * LV + 32 * c + 4 * g);
        const float b0[4] = {v0.x, v0.y, v0.z, v0.w}, b1[4] = {v1.x, v1.y, v1.z, v1.w};
        uint32_t h0[4], w0[4], h1[4], w1[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          split(b0[j], h0[j], w0[j]);
          split(b1[j], h1[j], w1[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_tf32(sum[j], pl[i], h0[j], h1[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_tf32(sum[j], ph[i], w0[j], w1[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_tf32(sum[j], ph[i], h0[j], h1[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][j][e] += sum[j][e];
    }
    note(t + RING, page);
  }
  if constexpr (RING > 1) cp_async_wait_group<0>();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    l[q] += __shfl_xor_sync(0xffffffffu, l[q], 1);
    l[q] += __shfl_xor_sync(0xffffffffu, l[q], 2);
    if (t4 == 0) { red[0][warp * 16 + g + 8 * q] = m[q]; red[1][warp * 16 + g + 8 * q] = l[q]; }
  }
  __syncthreads();  // (nobody reads the ring any more)
#pragma unroll
  for (int c = 0; c < DG; ++c)
#pragma unroll
    for (int q = 0; q < 2; ++q)  // columns 32 c + 8 t4 .. + 7
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *(float4*)(part + (warp * 16 + g + 8 * q) * LV + 32 * c + 8 * t4 + 4 * e) = make_float4(o[c][0][2 * q + e], o[c][1][2 * q + e], o[c][2][2 * q + e], o[c][3][2 * q + e]);
  __syncthreads();
  // the output of query x at four components, v against `top`, whose exponentials' sum is `sum`
  auto finish = [&](int x, int col, float4 v, float top, float sum) {
    if (x0 + x >= n * rep || col >= a.d) return;
    const int64_t at = (tok0 + (x0 + x) / rep) * a.nh + kvh * rep + (x0 + x) % rep;
    if constexpr (MODE != ALL) {
      const int64_t to = (MODE == OWN ? (int64_t)a.sh.chunks : (int64_t)blockIdx.y) * a.rows.M * a.nh + at;
      *(float4*)(a.sh.out + to * a.d + col) = v;
      if (col == 0) a.sh.ml[to] = make_float2(top, sum);
      return;
    }
    const float f = sum > 0.f ? 1.f / sum : 0.f;
    T* to = (T*)a.out + at * a.d + col;
    store_as(to, v.x * f); store_as(to + 1, v.y * f); store_as(to + 2, v.z * f); store_as(to + 3, v.w * f);
  };
  const float* joined = QR == 64 ? part : part + 64 * LV;
  if (QR == 16 || slices == 1)
    for (int i = tid; i < QR * (D / 4); i += 128) {
      const int x = i / (D / 4), c = i % (D / 4) * 4;
      float top = red[0][x], sum = red[1][x];
      float4 v = *(const float4*)(part + x * LV + c);
      if (QR == 16) {  // the warps' shares of the keys
        top = fmaxf(fmaxf(red[0][x], red[0][16 + x]), fmaxf(red[0][32 + x], red[0][48 + x]));
        const float at = top == -INFINITY ? 0.f : top;
        sum = 0.f;
        v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = fast_exp2(red[0][w * 16 + x] - at);
          const float4 u = *(const float4*)(part + (w * 16 + x) * LV + c);
          sum = fmaf(red[1][w * 16 + x], f, sum);
          v.x = fmaf(u.x, f, v.x); v.y = fmaf(u.y, f, v.y); v.z = fmaf(u.z, f, v.z); v.w = fmaf(u.w, f, v.w);
        }
      }
      if (slices == 1) {
        finish(x, c, v, top, sum);
      } else {
        *(float4*)(part + (64 + x) * LV + c) = v;
        if (c == 0) { ml[0][x] = top; ml[1][x] = sum; }
      }
    }
  if (slices == 1) {
    if (MODE == OWN && last_block()) depend();
    return;
  }
  if (QR == 64 && tid < QR) { ml[0][tid] = red[0][tid]; ml[1][tid] = red[1][tid]; }

  // the blocks' shares: a block has some of the values
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  auto remote = [](const float* p, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"((uint32_t)rank));
    return at;
  };
  const int rows = (int)min((int64_t)QR, n * rep - x0);
  for (int i = slice * 128 + tid; i < rows * (D / 4); i += 128 * slices) {
    const int x = i / (D / 4), c = i % (D / 4) * 4;
    float ms[8], ls[8];
    float4 os[8];  // (all on their way at once)
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      ms[s] = -INFINITY;
      ls[s] = 0.f;
      os[s] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s < slices) {
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ms[s]) : "r"(remote(&ml[0][x], s)) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(ls[s]) : "r"(remote(&ml[1][x], s)) : "memory");
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(os[s].x), "=f"(os[s].y), "=f"(os[s].z), "=f"(os[s].w) : "r"(remote(joined + x * LV + c, s)) : "memory");
      }
    }
    float top = ms[0];
#pragma unroll
    for (int s = 1; s < 8; ++s) top = fmaxf(top, ms[s]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const float f = fast_exp2(ms[s] - base);
      sum = fmaf(ls[s], f, sum);
      v.x = fmaf(os[s].x, f, v.x); v.y = fmaf(os[s].y, f, v.y); v.z = fmaf(os[s].z, f, v.z); v.w = fmaf(os[s].w, f, v.w);
    }
    finish(x, c, v, top, sum);
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (MODE == OWN && last_block()) depend();
}

template <typename T, int D, int QR, int MODE>
int launch_any(cg_ctx* c, const PagedAttnArgs& a) {
  constexpr size_t smem = any_smem<T, D, QR>();
  static PerDeviceFlag configured_on;
  bool& configured = configured_on.at(c->core->device);
  if (!configured) {
    CG_CUDA(c, cudaFuncSetAttribute(k_paged_attn<T, D, QR, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured = true;
  }
  const int64_t rep = a.nh / a.nkv, width = a.rows.cols << a.rows.lg, longest = MODE == OWN ? a.sh.own(width) : width;
  const int64_t tiles = (MODE == CHUNK ? (a.rows.M * rep + a.sh.groups.n * (QR - 1)) / QR : (a.most * rep + QR - 1) / QR) * a.nkv;  // (a group's last tile may not be full)
  if (tiles > 0x7FFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "too many tokens");
  if (MODE == CHUNK) {
    CG_CUDA(c, launch_kernel(c, k_paged_attn<T, D, QR, MODE>, dim3((unsigned)tiles, (unsigned)a.sh.chunks), dim3(128), smem, 1, a));
    CG_LAUNCHED(c);
    return CG_OK;
  }
  // Shares of the keys.  Us in f32, heads of 64, with 1 / 2 / 4 / 8, [the rule's] (the table's width stands for the lengths):
  //   3 rows of 213 behind 1500, 2 x 2 heads    117  63.1  50.2 [54.7]
  //   1 row of 1000                             70.3 40.8 [30.2] 32.3
  //   8 single tokens of 600                    16.2 12.6 [10.4] 13.9
  //   32 of 1800                                42.2 [26.5] 31.2 49.6
  //   1 of 4000                                 80.4 43.5  24.5 [15.1]
  static AtATime known;
  const int slices = pick_shares([&](int i) { return at_a_time(known, c->core->device, i, k_paged_attn<T, D, QR, MODE>, 128, smem); }, 8, tiles * a.rows.rows, longest,
                                 Shape<D, QR>::GK, QR == 16 ? 4.5 : 3.5, QR == 16 ? 2.8 : D == 64 ? 2.4 : D == 128 ? 4.5 : 5.,
                                 std::max(0.5, 1. - 0.5 * (double)a.most / (double)std::max<int64_t>(longest, 1)));
  CG_CUDA(c, launch_kernel(c, k_paged_attn<T, D, QR, MODE>, dim3((unsigned)tiles, (unsigned)a.rows.rows, (unsigned)slices), dim3(128), smem, slices, a));
  CG_LAUNCHED(c);
  return CG_OK;
}

template <typename T, int MODE>
int launch_typed(cg_ctx* c, const PagedAttnArgs& a) {
  // (of a group there are more queries than of a row)
  const bool few = (MODE == CHUNK ? a.rows.M : a.most) * (a.nh / a.nkv) <= 32;
  if (a.d <= 64) return few ? launch_any<T, 64, 16, MODE>(c, a) : launch_any<T, 64, 64, MODE>(c, a);
  if (a.d <= 128) return few ? launch_any<T, 128, 16, MODE>(c, a) : launch_any<T, 128, 64, MODE>(c, a);
  return few ? launch_any<T, 256, 16, MODE>(c, a) : launch_any<T, 256, 64, MODE>(c, a);
}

// The parts of a token's head, joined: o = sum_c o_c 2^(m_c - m) / sum_c l_c 2^(m_c - m), m the largest m_c.  A thread has four components, a block
// 256 / (d / 4) vectors or more; what the tables say is looked up before the parts are waited for.  What bounds it is that chain and the parts' way out of L2: 64 x 32
// heads of 128 and 14 parts, 15 MB, some 5 us behind the others.  (A launch of its own: in the blocks of the rows' own keys the loads of parts would stand in the way of the
// next block's keys.)
template <typename T>
__global__ void __launch_bounds__(256) k_paged_join(PagedAttnArgs a) {
  const int quads = a.d / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, vector = i / quads, m = vector / a.nh;
  const int col = (int)(i - vector * quads) * 4;
  const int64_t m0 = ((int64_t)blockIdx.x * 256 + (threadIdx.x & ~31)) / quads / a.nh, m1 = ((int64_t)blockIdx.x * 256 + (threadIdx.x | 31)) / quads / a.nh;  // tokens of the warp's ends
  int chunks = -1;
  for (int64_t t = m0; t <= m1 && t < a.rows.M; ++t) {
    const int64_t row = rows_before(a.rows, 0, a.rows.rows, t);
    int64_t tok0, n, len, shared;
    if (row >= a.rows.rows || !row_span(a.rows, row, a.most, &tok0, &n, &len) || t < tok0 || t >= tok0 + n) continue;
    const int64_t group = group_of_row(a.sh.groups, row, &shared);
    const int c = chunks_of(a.rows, a.sh, group, tok0, n);
    if (t == m) chunks = c;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (m >= a.rows.M || chunks < 0) return;
  const int64_t per_chunk = a.rows.M * a.nh;
  constexpr int U = 8;  // (on their way at a time)
  float top = -INFINITY, sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c0 = 0; c0 <= chunks; c0 += U) {
    float2 ml[U];
    float4 o[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      if (c0 + k <= chunks) {
        const int64_t x = (c0 + k < chunks ? c0 + k : a.sh.chunks) * per_chunk + vector;
        ml[k] = __ldcg(a.sh.ml + x);
        o[k] = __ldcg((const float4*)(a.sh.out + x * a.d + col));
      }
    }
    const float before = top;
#pragma unroll
    for (int k = 0; k < U; ++k) top = fmaxf(top, ml[k].x);
    const float base = top == -INFINITY ? 0.f : top, f0 = fast_exp2(before - base);
    sum *= f0;
    v.x *= f0; v.y *= f0; v.z *= f0; v.w *= f0;
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (ml[k].y != 0.f) {  // (a part without keys holds anything; a sum that is no number is one, and all that it is joined with)
        const float f = fast_exp2(ml[k].x - base);
        sum = fmaf(ml[k].y, f, sum);
        v.x = fmaf(o[k].x, f, v.x); v.y = fmaf(o[k].y, f, v.y); v.z = fmaf(o[k].z, f, v.z); v.w = fmaf(o[k].w, f, v.w);
      }
  }
  const float f = sum != 0.f ? 1.f / sum : 0.f;
  T* to = (T*)a.out + vector * a.d + col;
  if constexpr (sizeof(T) == 4) {
    store_as(to, v.x * f); store_as(to + 1, v.y * f); store_as(to + 2, v.z * f); store_as(to + 3, v.w * f);
  } else if ((uintptr_t)a.out % 8 == 0) {
    *(uint2*)to = make_uint2(pack_bf16(v.x * f, v.y * f), pack_bf16(v.z * f, v.w * f));
  } else {
    store_as(to, v.x * f); store_as(to + 1, v.y * f); store_as(to + 2, v.z * f); store_as(to + 3, v.w * f);
  }
}
template <typename T>
int launch_join(cg_ctx* c, const PagedAttnArgs& a) {
  const int64_t blocks = (a.rows.M * a.nh * (a.d / 4) + 255) / 256;
  if (blocks > 0x7FFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "too many tokens");
  CG_CUDA(c, launch_kernel(c, k_paged_join<T>, dim3((unsigned)blocks), dim3(256), 0, 1, a));
  CG_LAUNCHED(c);
  return CG_OK;
}

// What both kinds of attention check of their arguments, and their form for the kernels; `nothing`: there is nothing to do.
int attention_args(cg_ctx* c, const cg_tensor* q, const cg_tensor* k_pages, const cg_tensor* v_pages, const cg_tensor* table, const cg_tensor* starts,
                   const cg_tensor* lens, int64_t max_new, float scale, int64_t window, float softcap, const cg_tensor* out, PagedAttnArgs* args, bool* nothing) {
  PagedAttnArgs& a = *args;
  if (!q || !out) return fail(c, CG_ERR_INVALID, "null argument");
  int lg;
  CG_TRY(check_pages(c, k_pages, v_pages, false, &lg));
  const int64_t nkv = k_pages->dims[1], d = k_pages->dims[3], any[3] = {-1, -1, d};
  CG_TRY(check_tensor(c, q, "q", CG_F32, 3, any, false));
  const int64_t M = q->dims[0], nh = q->dims[1];
  CG_TRY(check_tensor(c, out, "out", CG_F32, 3, q->dims));
  CG_TRY(check_rows(c, table, starts, lens, M, k_pages->dims[0], lg, &a.rows));
  if (q->storage != k_pages->storage || out->storage != k_pages->storage) return fail(c, CG_ERR_DTYPE, "q and out are stored as the pages are");
  if (M > 0 && q->strides[2] != 1) return fail(c, CG_ERR_UNSUPPORTED, "q: the last axis must be contiguous");
  if (nkv < 1 || nkv > 65535 || nh > 65535) return fail(c, CG_ERR_UNSUPPORTED, "too many heads");
  if (nh % nkv) return fail(c, CG_ERR_SHAPE, "query heads are a multiple of key heads");
  if (max_new < 0 || window < 0 || !(softcap >= 0.f) || !(scale >= 0.f) || scale > 3e38f || softcap > 3e38f) return fail(c, CG_ERR_INVALID, "bad argument");
  if (overlap_any({q, k_pages, v_pages, table, starts, lens}, {out})) return fail(c, CG_ERR_INVALID, "out overlaps an input");
  if (M == 0 || nh == 0 || a.rows.rows == 0) {
    *nothing = true;
    return CG_OK;
  }
  if (k_pages->dims[0] == 0) return fail(c, CG_ERR_SHAPE, "no pages");
  a.q = q->data(); a.k_pages = k_pages->data(); a.v_pages = v_pages->data(); a.out = out->data();
  a.q_ld = q->strides[0]; a.q_hs = q->strides[1];
  a.most = max_new > 0 ? std::min(max_new, M) : M;
  a.window = window < a.rows.cols << lg ? window : 0;  // (one that reaches over all positions is none)
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)d);
  // (caps beyond 2^+-100 act as these: all scores are far below the one, and differ by nothing that an exponential shows under the other)
  a.cap = softcap > 0.f ? fminf(fmaxf(softcap, 0x1p-100f), 0x1p100f) : 0.f;
  a.nh = (int)nh; a.nkv = (int)nkv; a.d = (int)d;
  return CG_OK;
}
// Attention over all of a row's keys.
int attend(cg_ctx* c, const PagedAttnArgs& a, bool bf16) {
  if (bf16 && paged_fa_supported(a)) return paged_fa(c, a);
  if (bf16 && paged_dec_supported(a)) return paged_dec(c, a);
  return bf16 ? launch_typed<__nv_bfloat16, ALL>(c, a) : launch_typed<float, ALL>(c, a);
}

// Into how many chunks shared keys are cut (0: rows read them for themselves, out of L2).  A function of sizes alone, as the workspace's is.
// Rows of so many tokens that they fill half a tile of 128 queries gain little by others' beside them, and blocks find their group by walking them (32 at
// a time, 1 us).  Two launches more pay where 32 MB need not be read again, whatever the type, and 12 keys for each query, whose parts are written, read and
// joined.  Us with chunks / row by row, [the rule's], rows of 1, 4 and 8 tokens:
//   12 rows behind  500, 8 key heads of 128, saves  23 MB    10.4 [10.0]    14.4 [12.9]    16.3 [13.1]
//   40 behind       500, 4 of 128,                  40 MB    13.1 [13.1]    23.8 [15.5]    30.4 [15.6]
//   12 behind      1500, 4 of 128,                  34 MB    12.3 [12.2]    15.9 [18.3]    18.6 [18.3]
//   40 behind       500, 8 of 128,                  80 MB   [15.4] 23.5    [26.7] 29.3     32.4 [26.5]
//   40 behind      1500, 4 of 128,                 120 MB   [17.6] 26.6    [27.2] 29.5    [35.4] 29.6
//   40 behind      5000, 8 of 128,                 799 MB   [23.8] 119     [39.1] 144     [67.0] 150
//    4 behind      5000, 8 of 64,                   31 MB    15.7 [10.4]    17.2 [13.6]    16.1 [20.2]
//   12 behind      1500, 4 of 256 with a cap,       68 MB   [13.9] 20.7    [15.6] 21.6    [28.1] 29.8
//   40 behind       500, 2 of 64, f32,              20 MB    19.3 [16.7]    19.4 [16.9]    21.3 [17.0]
//   40 behind      1500, 2 of 64, f32,              60 MB   [19.9] 42.5    [26.4] 42.8    [32.4] 43.0
constexpr int SHARED_QUERIES = 64;  // of a row and key head, at most, in the mean
// (In the mean: a prompt among rows that run does not keep these from sharing, and takes the chunks' tiles as they do.  64 rows of 1, 8 key heads of 128, and with them one of
// 100 or 500, behind 500: [45] and 109 us, row by row 62 and [89]; behind 4000: [60] and [135], 269 and 301; behind 16000: [139] and [345], 1073 and 1046.)
int64_t mean_new(const PagedAttnArgs& a) { return std::min(a.most, (a.rows.M + a.rows.rows - 1) / a.rows.rows); }
// Under a window rows read no more than that of the prefix, and the chunks all of it.  Us with chunks / row by row, the rule's with a *, windows of 512, 1024 and 4096 for
// 4 key heads of 256, then for 8 of 128:
//   14 rows behind  3000    21.5  11.4*   21.4* 16.1    20.8* 34.7       18.1   9.8*   18.0* 13.3    18.1* 27.6
//   14 behind      16000    31.8  17.0*   31.8  22.1*   31.8* 50.3       26.4  15.0*   26.2  18.8*   26.0* 40.4
//   40 behind      16000    37.7  41.1*   37.7* 54.1    37.4* 125        41.1  35.9*   41.2* 45.3    41.1* 98.8
//    2 behind      16000    31.1  15.1*   31.0  17.4*   30.7  23.0*      25.3   6.9*   24.9   7.8*   24.8  13.2*
bool saves_enough(const cg_ctx* c, const PagedAttnArgs& a, bool bf16, int64_t queries) {
  const double most = (double)a.sh.groups.most, seen = a.window > 0 ? std::min(most, (double)(a.window + mean_new(a) - 1)) : most;
  const double keys = (double)a.rows.rows * seen - (double)a.sh.groups.n * most - 12. * (double)queries;  // (wide tables name more bytes than 63 bits hold)
  return a.sh.groups.n > 0 && a.sh.groups.n <= 256 && a.sh.groups.most > 0 && c->opt_shared != 0 && (c->opt_shared != 1 || keys * (2. * a.nkv * a.d * (bf16 ? 2 : 4)) >= 32 << 20);
}
constexpr int ANY_SLOTS = 2 * 148;  // blocks of 64 queries, or 16, in f32: two or four on an SM
void plan_chunks(const cg_ctx* c, PagedAttnArgs* args, bool bf16) {
  PagedAttnArgs& a = *args;
  const int64_t rep = a.nh / a.nkv;
  a.sh.chunks = 0;
  a.sh.chunk = 0;
  if (mean_new(a) * rep > SHARED_QUERIES || !saves_enough(c, a, bf16, a.rows.M * rep)) return;
  if (bf16) {
    a.sh.chunk = paged_fa_chunk(a);
  } else {
    const int64_t size = a.rows.M * rep <= 32 ? 16 : 64, tiles = std::max((a.rows.M * rep + size - 1) / size, a.sh.groups.n) * a.nkv;
    const int64_t chunks = std::max<int64_t>(ANY_SLOTS / tiles, 1);
    a.sh.chunk = std::max<int64_t>(((a.sh.groups.most + chunks - 1) / chunks + 63) / 64 * 64, SHARED_CHUNK);
  }
  a.sh.chunks = (int)std::min<int64_t>((a.sh.groups.most + a.sh.chunk - 1) / a.sh.chunk, 0x7FFFFFFF);
}
// Parts of a head, at most, of all calls of up to M tokens: fewer tokens are cut into more chunks, so their number times the tokens does not ascend with these.  A chunk
// has SHARED_CHUNK keys or more, and there are no more chunks than slots / tiles, or one, where tiles of `size` queries are M rep nkv / size or more:
//   (chunks + 1) M <= min(M most / SHARED_CHUNK, max(M, slots size / nh)) + M
int64_t most_parts(const PagedAttnArgs& a, bool bf16) {
  const int64_t slots = bf16 ? paged_fa_slots(a) : ANY_SLOTS, size = bf16 ? 128 : 64, M = a.rows.M;
  const int64_t chunks = std::min((a.sh.groups.most + SHARED_CHUNK - 1) / SHARED_CHUNK, slots);
  return std::min(M * chunks, std::max(M, slots * size / a.nh)) + M;
}

}  // namespace

}  // namespace cg

using namespace cg;

extern "C" int32_t cg_paged_attention(cg_ctx* c, const cg_tensor* q, const cg_tensor* k_pages, const cg_tensor* v_pages, const cg_tensor* table,
                                      const cg_tensor* starts, const cg_tensor* lens, int64_t max_new, float scale, int64_t window, float softcap,
                                      cg_tensor* out) {
  if (!c) return CG_ERR_INVALID;
  CG_LAZY_EAGER_SCOPE(c);
  OnDevice on(c);
  PagedAttnArgs a = {};
  bool nothing = false;
  CG_TRY(attention_args(c, q, k_pages, v_pages, table, starts, lens, max_new, scale, window, softcap, out, &a, &nothing));
  if (nothing) return CG_OK;
  written(out);
  return attend(c, a, q->storage == ST_BF16);
}

extern "C" int64_t cg_paged_shared_floats(cg_ctx* c, const cg_tensor* q, const cg_tensor* k_pages, const cg_tensor* table, const cg_tensor* groups,
                                          int64_t max_new, int64_t max_shared) {
  if (!c || !q || !k_pages || !table || !groups || q->rank != 3 || k_pages->rank != 4 || table->rank != 2 || groups->rank != 1 || groups->dims[0] < 1 || max_new < 0 ||
      max_shared < 0 || k_pages->dims[1] < 1 || q->dims[1] % k_pages->dims[1] || q->dims[1] > 65535)
    return -1;
  PagedAttnArgs a = {};
  a.rows.M = q->dims[0];
  a.rows.rows = table->dims[0];
  a.nh = (int)q->dims[1];
  a.nkv = (int)k_pages->dims[1];
  a.d = (int)k_pages->dims[3];
  if (a.rows.M == 0 || a.nh == 0 || a.rows.rows == 0) return 0;
  a.most = max_new > 0 ? std::min(max_new, a.rows.M) : a.rows.M;
  const int64_t longest = table->dims[1] * k_pages->dims[2];
  a.sh.groups.n = groups->dims[0] - 1;
  a.sh.groups.most = max_shared > 0 ? std::min(max_shared, longest) : longest;
  const bool bf16 = q->storage == ST_BF16;
  const int64_t rep = a.nh / a.nkv;
  if (mean_new(a) * rep > SHARED_QUERIES) {
    // Rows read for themselves in this step, but not in all smaller ones.  (Where prefixes are always read once, for tests, it is the step's own.)
    if (c->opt_shared != 1) return 0;
    a.rows.M = std::min(a.rows.M, a.rows.rows * (SHARED_QUERIES / rep));
  }
  return a.rows.M > 0 && saves_enough(c, a, bf16, 0) ? most_parts(a, bf16) * a.nh * (a.d + 2) : 0;
}

extern "C" int32_t cg_paged_shared_attention(cg_ctx* c, const cg_tensor* q, const cg_tensor* k_pages, const cg_tensor* v_pages, const cg_tensor* table,
                                             const cg_tensor* starts, const cg_tensor* lens, const cg_tensor* groups, const cg_tensor* shared, int64_t max_new,
                                             int64_t max_shared, float scale, int64_t window, float softcap, cg_tensor* work, cg_tensor* out) {
  if (!c) return CG_ERR_INVALID;
  CG_LAZY_EAGER_SCOPE(c);
  OnDevice on(c);
  PagedAttnArgs a = {};
  bool nothing = false;
  CG_TRY(attention_args(c, q, k_pages, v_pages, table, starts, lens, max_new, scale, window, softcap, out, &a, &nothing));
  const int64_t any[1] = {-1};
  CG_TRY(check_tensor(c, groups, "groups", CG_U32, 1, any));
  if (groups->dims[0] < 1) return fail(c, CG_ERR_SHAPE, "Shape mismatch in operation: groups");
  const int64_t G[1] = {groups->dims[0] - 1};
  CG_TRY(check_tensor(c, shared, "shared", CG_U32, 1, G));
  CG_TRY(check_tensor(c, work, "work", CG_F32, 1, any));
  if (work->storage != ST_F32) return fail(c, CG_ERR_DTYPE, "work is f32");
  if (G[0] > 65535) return fail(c, CG_ERR_UNSUPPORTED, "at most 65535 groups");
  if (max_shared < 0) return fail(c, CG_ERR_INVALID, "bad argument");
  if (overlap_any({q, k_pages, v_pages, table, starts, lens, groups, shared}, {out, work})) return fail(c, CG_ERR_INVALID, "what is written overlaps an input or each other");
  if (nothing) return CG_OK;
  const int64_t longest = a.rows.cols << a.rows.lg;
  a.sh.groups.rows = (const uint32_t*)groups->data();
  a.sh.groups.shared = (const uint32_t*)shared->data();
  a.sh.groups.n = G[0];
  a.sh.groups.most = max_shared > 0 ? std::min(max_shared, longest) : longest;
  const bool bf16 = q->storage == ST_BF16;
  plan_chunks(c, &a, bf16);
  const int64_t parts = a.sh.chunks ? (a.sh.chunks + 1) * a.rows.M * a.nh : 0;
  if (work->dims[0] < parts * (a.d + 2)) return fail(c, CG_ERR_SHAPE, "work holds less than cg_paged_shared_floats");
  if (parts > 0 && (uintptr_t)work->data() % 32) return fail(c, CG_ERR_UNSUPPORTED, "work begins on a 32-byte boundary");
  written(out);
  if (parts == 0) return attend(c, a, bf16);
  if (a.sh.chunks > 65535) return fail(c, CG_ERR_UNSUPPORTED, "too many tokens");
  written(work);
  a.sh.out = (float*)work->data();
  a.sh.ml = (float2*)(a.sh.out + parts * a.d);
  if (bf16 && paged_fa_prefix_supported(a)) CG_TRY(paged_fa_prefix(c, a));
  else CG_TRY((bf16 ? launch_typed<__nv_bfloat16, CHUNK>(c, a) : launch_typed<float, CHUNK>(c, a)));
  if (bf16 && paged_fa_supported(a)) CG_TRY(paged_fa_own(c, a));
  else if (bf16 && paged_dec_supported(a)) CG_TRY(paged_dec_own(c, a));
  else CG_TRY((bf16 ? launch_typed<__nv_bfloat16, OWN>(c, a) : launch_typed<float, OWN>(c, a)));
  return bf16 ? launch_join<__nv_bfloat16>(c, a) : launch_join<float>(c, a);
}
