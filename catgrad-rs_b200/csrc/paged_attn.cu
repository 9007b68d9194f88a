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
template <typename T, int D, int QR>
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
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int rep = a.nh / a.nkv, kvh = (int)blockIdx.x % a.nkv;
  const int64_t row = blockIdx.y, x0 = (int64_t)(blockIdx.x / a.nkv) * QR;
  const int slices = (int)gridDim.z, slice = (int)blockIdx.z;
  int64_t tok0, n, len;
  if (!row_span(a.rows, row, a.most, &tok0, &n, &len) || x0 >= n * rep) return;  // (the same in all blocks of a cluster)
  const int64_t pos0 = len - n, i0 = x0 / rep, i1 = min(n - 1, (x0 + QR - 1) / rep);
  const int64_t lo = a.window > 0 ? max((int64_t)0, pos0 + i0 - a.window + 1) : 0, hi = pos0 + i1;
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
  const int64_t qpos[2] = {pos0 + (x0 + r0) / rep, pos0 + (x0 + r0 + 8) / rep};
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
    const bool masked = k0 + GK / WK - 1 > pos0 + i0 || k0 < lo || (a.window > 0 && k0 <= hi - a.window);
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
        const int64_t x = qpos[q] - k0;
        lim[q] = x > GK ? GK : x < -1 ? -1 : (int)x;
        low[q] = a.window > 0 ? (x - a.window >= GK ? GK : x - a.window < -1 ? 0 : (int)(x - a.window) + 1) : 0;
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
  auto put4 = [&](int x, int col, float4 v, float f) {
    if (x0 + x >= n * rep || col >= a.d) return;
    T* to = (T*)a.out + ((tok0 + (x0 + x) / rep) * a.nh + kvh * rep + (x0 + x) % rep) * a.d + col;
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
        put4(x, c, v, sum > 0.f ? 1.f / sum : 0.f);
      } else {
        *(float4*)(part + (64 + x) * LV + c) = v;
        if (c == 0) { ml[0][x] = top; ml[1][x] = sum; }
      }
    }
  if (slices == 1) return;
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
    put4(x, c, v, sum > 0.f ? 1.f / sum : 0.f);
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int D, int QR>
int launch_any(cg_ctx* c, const PagedAttnArgs& a) {
  constexpr size_t smem = any_smem<T, D, QR>();
  static PerDeviceFlag configured_on;
  bool& configured = configured_on.at(c->core->device);
  if (!configured) {
    CG_CUDA(c, cudaFuncSetAttribute(k_paged_attn<T, D, QR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured = true;
  }
  const int64_t tiles = (a.most * (a.nh / a.nkv) + QR - 1) / QR * a.nkv, longest = a.rows.cols << a.rows.lg;
  if (tiles > 0x7FFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "too many tokens");
  // Shares of the keys.  Us in f32, heads of 64, with 1 / 2 / 4 / 8, [the rule's] (the table's width stands for the lengths):
  //   3 rows of 213 behind 1500, 2 x 2 heads    117  63.1  50.2 [54.7]
  //   1 row of 1000                             70.3 40.8 [30.2] 32.3
  //   8 single tokens of 600                    16.2 12.6 [10.4] 13.9
  //   32 of 1800                                42.2 [26.5] 31.2 49.6
  //   1 of 4000                                 80.4 43.5  24.5 [15.1]
  static AtATime known;
  const int slices = pick_shares([&](int i) { return at_a_time(known, c->core->device, i, k_paged_attn<T, D, QR>, 128, smem); }, 8, tiles * a.rows.rows, longest,
                                 Shape<D, QR>::GK, QR == 16 ? 4.5 : 3.5, QR == 16 ? 2.8 : D == 64 ? 2.4 : D == 128 ? 4.5 : 5.,
                                 std::max(0.5, 1. - 0.5 * (double)a.most / (double)std::max<int64_t>(longest, 1)));
  CG_CUDA(c, launch_kernel(c, k_paged_attn<T, D, QR>, dim3((unsigned)tiles, (unsigned)a.rows.rows, (unsigned)slices), dim3(128), smem, slices, a));
  CG_LAUNCHED(c);
  return CG_OK;
}

template <typename T>
int launch_typed(cg_ctx* c, const PagedAttnArgs& a) {
  const bool few = a.most * (a.nh / a.nkv) <= 32;
  if (a.d <= 64) return few ? launch_any<T, 64, 16>(c, a) : launch_any<T, 64, 64>(c, a);
  if (a.d <= 128) return few ? launch_any<T, 128, 16>(c, a) : launch_any<T, 128, 64>(c, a);
  return few ? launch_any<T, 256, 16>(c, a) : launch_any<T, 256, 64>(c, a);
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
  if (!q || !out) return fail(c, CG_ERR_INVALID, "null argument");
  PagedAttnArgs a = {};
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
  if (M == 0 || nh == 0 || a.rows.rows == 0) return CG_OK;
  if (k_pages->dims[0] == 0) return fail(c, CG_ERR_SHAPE, "no pages");
  a.q = q->data(); a.k_pages = k_pages->data(); a.v_pages = v_pages->data(); a.out = out->data();
  a.q_ld = q->strides[0]; a.q_hs = q->strides[1];
  a.most = max_new > 0 ? std::min(max_new, M) : M;
  a.window = window < a.rows.cols << lg ? window : 0;  // (one that reaches over all positions is none)
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)d);
  // (caps beyond 2^+-100 act as these: all scores are far below the one, and differ by nothing that an exponential shows under the other)
  a.cap = softcap > 0.f ? fminf(fmaxf(softcap, 0x1p-100f), 0x1p100f) : 0.f;
  a.nh = (int)nh; a.nkv = (int)nkv; a.d = (int)d;
  written(out);
  if (q->storage == ST_BF16 && paged_fa_supported(a)) return paged_fa(c, a);
  if (q->storage == ST_BF16 && paged_dec_supported(a)) return paged_dec(c, a);
  return q->storage == ST_BF16 ? launch_typed<__nv_bfloat16>(c, a) : launch_typed<float>(c, a);
}
