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

// two f32 at a time
__device__ __forceinline__ void fma2(uint64_t& c, uint64_t a, uint64_t b) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b)); }
__device__ __forceinline__ void mul2(uint64_t& c, uint64_t a) { asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(c) : "l"(a)); }
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ float2 both(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}

// f32, and whatever the tensor-core kernels do not take, on the CUDA cores.  A block has QR queries of one row and key head (query x
// is token x / rep, head x % rep of the group) and a share of the visible keys, 32 at a time; the blocks of a cluster share the
// keys and are joined through shared memory.  Eight lanes have a query row (or four rows): a score is a key's, an output value
// four neighbouring columns', so that for a thread's 4 x 4 products eight vectors are read; two products are
// one instruction, and probabilities lie in shared memory twice for that.  f32 keys and values come by
// asynchronous copies, a ring of tiles ahead, their places looked up a tile before that.  D: head size, rounded up to 64,
// 128 or 256.
constexpr int GK = 32;  // keys of a tile
template <typename T, int D>
__host__ __device__ constexpr int any_ring() { return sizeof(T) == 2 ? 1 : D == 256 ? 2 : 3; }
template <typename T, int D, int QR>
__host__ __device__ constexpr size_t any_smem() { return (size_t)((QR + 2 * any_ring<T, D>() * GK) * (D + 4) + 2 * QR * (GK + 1)) * 4; }
template <typename T, int D, int QR>
__global__ void __launch_bounds__(128) k_paged_attn(PagedAttnArgs a) {
  constexpr int LD = D + 4, RING = any_ring<T, D>();
  constexpr int RT = QR / 16;      // query rows of a thread
  constexpr int CT = D / 32;       // groups of four output columns of a thread
  extern __shared__ __align__(16) float sm[];
  float* qs = sm;                  // [QR][LD]
  float* ring = qs + QR * LD;      // [RING] keys [GK][LD], values [GK][LD]
  uint64_t* ps = (uint64_t*)(ring + RING * 2 * GK * LD);  // [QR][GK + 1]: each probability twice
  __shared__ float ml[2][QR];
  __shared__ int64_t places[2][GK];  // of the keys of the next tile to be asked for; -1: zeros
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, ty = tid >> 3, tx = tid & 7;
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
  auto look_up = [&](int64_t t) {  // by the first warp
    const int64_t key = t * GK + tid;
    int64_t at = -1;
    if (t < t1 && key >= lo && key <= hi) {
      const int64_t page = page_of(a.rows, row, key);
      if (page >= 0) at = (((page * a.nkv + kvh) << a.rows.lg) + (key & page_mask)) * a.d;
    }
    places[t & 1][tid] = at;
  };
  auto request = [&](int64_t t) {
    float* ks = ring + (int)((t - t0) % RING) * 2 * GK * LD;
    float* vs = ks + GK * LD;
    if constexpr (sizeof(T) == 4) {
      if (t < t1)
        for (int i = tid; i < GK * (D / 4); i += 128) {
          const int r = i / (D / 4), c = i % (D / 4) * 4;
          const int64_t at = places[t & 1][r];
          const bool there = at >= 0 && c < a.d;
          const float* k = (const float*)a.k_pages + (there ? at + c : 0);
          const float* v = (const float*)a.v_pages + (there ? at + c : 0);
          cp_async16((uint32_t)__cvta_generic_to_shared(ks + r * LD + c), k, there ? 16 : 0);
          cp_async16((uint32_t)__cvta_generic_to_shared(vs + r * LD + c), v, there ? 16 : 0);
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
          ks[r * LD + c + e] = kx[e];
          vs[r * LD + c + e] = vx[e];
        }
      }
    }
  };
  if (tid < GK) look_up(t0);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) {  // (two tiles' places take turns)
    request(t0 + i);
    if (tid < GK) look_up(t0 + i + 1);
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
    for (int e = 0; e < 8; ++e) qs[r * LD + c + e] = v[e];
  }
  float m[RT], l[RT];
  uint64_t o[RT][CT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < CT; ++c) o[r][c][0] = o[r][c][1] = 0;
  }
  for (int64_t t = t0; t < t1; ++t) {
    if constexpr (RING > 1) {
      cp_async_wait_group<RING - 2>();
      __syncthreads();  // tile t is there, and everyone is done with the one before
      request(t + RING - 1);
      if (tid < GK) look_up(t + RING);
    } else {
      __syncthreads();
      request(t);
      __syncthreads();
      if (tid < GK) look_up(t + 1);
    }
    const float* ks = ring + (int)((t - t0) % RING) * 2 * GK * LD;
    const float* vs = ks + GK * LD;
    uint64_t s2[RT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r) s2[r][0] = s2[r][1] = s2[r][2] = s2[r][3] = 0;
#pragma unroll 4
    for (int c = 0; c < D; c += 4) {
      ulonglong2 kk[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) kk[j] = *(const ulonglong2*)(ks + (tx + 8 * j) * LD + c);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const ulonglong2 qq = *(const ulonglong2*)(qs + (ty * RT + r) * LD + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) fma2(s2[r][j], qq.x, kk[j].x);
#pragma unroll
        for (int j = 0; j < 4; ++j) fma2(s2[r][j], qq.y, kk[j].y);
      }
    }
    const bool masked = t * GK + GK - 1 > pos0 + i0 || (a.window > 0 && t * GK <= hi - a.window);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int64_t pos = masked ? pos0 + (x0 + ty * RT + r) / rep : 0;
      float top = -INFINITY, s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t key = t * GK + tx + 8 * j;
        const float2 f = both(s2[r][j]);
        float x = (f.x + f.y) * a.scale;
        if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
        if (masked && !(key <= pos && (a.window <= 0 || key > pos - a.window))) x = -INFINITY;
        s[j] = x;
        top = fmaxf(top, x);
      }
#pragma unroll
      for (int w = 4; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float m_new = fmaxf(m[r], top), base = m_new == -INFINITY ? 0.f : m_new;
      const float corr = expf(m[r] - base);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = expf(s[j] - base);
        sum += e;
        ps[(ty * RT + r) * (GK + 1) + tx + 8 * j] = pair(e, e);
      }
      l[r] = l[r] * corr + sum;  // (of this lane's keys)
      m[r] = m_new;
      if (corr != 1.f)
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          mul2(o[r][c][0], pair(corr, corr));
          mul2(o[r][c][1], pair(corr, corr));
        }
    }
    __syncwarp();
#pragma unroll 4
    for (int k = 0; k < GK; ++k) {
      uint64_t p[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) p[r] = ps[(ty * RT + r) * (GK + 1) + k];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const ulonglong2 v = *(const ulonglong2*)(vs + k * LD + tx * 4 + c * 32);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          fma2(o[r][c][0], p[r], v.x);
          fma2(o[r][c][1], p[r], v.y);
        }
      }
    }
    __syncwarp();
  }
  if constexpr (RING > 1) cp_async_wait_group<0>();
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int w = 4; w; w >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
  auto values = [&](int r, int c, float f) {
    const float2 u = both(o[r][c][0]), w = both(o[r][c][1]);
    return make_float4(u.x * f, u.y * f, w.x * f, w.y * f);
  };
  auto put4 = [&](int64_t x, int col, float4 v) {
    if (x >= n * rep || col >= a.d) return;
    T* to = (T*)a.out + ((tok0 + x / rep) * a.nh + kvh * rep + x % rep) * a.d + col;
    store_as(to, v.x); store_as(to + 1, v.y); store_as(to + 2, v.z); store_as(to + 3, v.w);
  };
  if (slices == 1) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float f = l[r] > 0.f ? 1.f / l[r] : 0.f;
#pragma unroll
      for (int c = 0; c < CT; ++c) put4(x0 + ty * RT + r, tx * 4 + c * 32, values(r, c, f));
    }
    return;
  }
  // the shares are joined: a block has some of the values
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int x = ty * RT + r;
    if (tx == 0) { ml[0][x] = m[r]; ml[1][x] = l[r]; }
#pragma unroll
    for (int c = 0; c < CT; ++c) *(float4*)(qs + x * LD + tx * 4 + c * 32) = values(r, c, 1.f);
  }
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
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(os[s].x), "=f"(os[s].y), "=f"(os[s].z), "=f"(os[s].w) : "r"(remote(qs + x * LD + c, s)) : "memory");
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
      const float f = expf(ms[s] - base);
      sum = fmaf(ls[s], f, sum);
      v.x = fmaf(os[s].x, f, v.x); v.y = fmaf(os[s].y, f, v.y); v.z = fmaf(os[s].z, f, v.z); v.w = fmaf(os[s].w, f, v.w);
    }
    const float f = sum > 0.f ? 1.f / sum : 0.f;
    put4(x0 + x, c, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
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
  // Blocks that share the keys: until there are two per SM, but no shares of less than two tiles.
  int slices = 1;
  while (slices < 8 && tiles * a.rows.rows * slices < 148 * 2 && (int64_t)slices * 2 * GK < longest) slices *= 2;
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
  a.q = q->data(); a.k_pages = k_pages->data(); a.v_pages = v_pages->data(); a.out = out->data();
  a.q_ld = q->strides[0]; a.q_hs = q->strides[1];
  a.most = max_new > 0 ? std::min(max_new, M) : M;
  a.window = window;
  a.scale = scale > 0.f ? scale : 1.f / sqrtf((float)d);
  a.cap = softcap;
  a.nh = (int)nh; a.nkv = (int)nkv; a.d = (int)d;
  written(out);
  if (q->storage == ST_BF16 && paged_fa_supported(a)) return paged_fa(c, a);
  if (q->storage == ST_BF16 && paged_dec_supported(a)) return paged_dec(c, a);
  return q->storage == ST_BF16 ? launch_typed<__nv_bfloat16>(c, a) : launch_typed<float>(c, a);
}
