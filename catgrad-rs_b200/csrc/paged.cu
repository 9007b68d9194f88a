// paged.cu — appending to a paged key/value cache, and its reordering behind a step of beam search.
//
// cg_paged_append: per new token and head x^ = x / sqrt(mean x^2 + eps) g (optional, queries and keys;
// catgrad-llm/src/models/qwen3.rs:187-217), then the rotation of catgrad-llm/src/helpers.rs:202-221,
// (a, b) -> (a cos - b sin, b cos + a sin), then one rounding to the pages' type.
// cg_paged_reorder: beam j of a group goes on from parents[j]: the pages that are full are shared by naming them, the one
// that has begun is copied, in all layers.
#include <algorithm>

#include "paged.h"

namespace cg {

namespace {

struct AppendArgs {
  PagedRows rows;
  const void *q, *k, *v;
  int64_t q_ld, k_ld, v_ld, q_hs, k_hs, v_hs;  // from one token and one head to the next
  const float *q_gain, *k_gain;
  float eps;
  int plus_one;
  const float *cos_t, *sin_t;  // [T, half] or null
  int64_t T;
  int half, rot_half;
  void *q_out, *k_pages, *v_pages;
  int nh, nkv, d;
};

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Every head size and alignment (k_paged_append_vec takes the usual ones; its long case below takes 225 us here).  A warp per vector (a head of a token); a lane has pairs lane, lane + 32, ..: with `rot_half` pair i < half is components
// (i, i + half), else (2 i, 2 i + 1); pairs from `half` on are (2 i, 2 i + 1) and not turned.
template <typename TI, typename TO>
__global__ void __launch_bounds__(256) k_paged_append(AppendArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int heads = a.nh + 2 * a.nkv;
  const int64_t vec = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t m = vec / heads;
  const int h = (int)(vec - m * heads);
  if (m >= a.rows.M) return;
  // the token's row: as many rows as end at or before it
  int64_t row = 0;
  for (int64_t i = lane; i - lane < a.rows.rows; i += 32)
    row += __popc(__ballot_sync(0xffffffffu, i < a.rows.rows && a.rows.starts[i + 1] <= m));
  if (row >= a.rows.rows) return;  // behind the last row
  int64_t tok0, n, len;
  if (!row_span(a.rows, row, a.rows.M, &tok0, &n, &len) || m < tok0) return;
  if (m >= tok0 + n) {  // (starts that do not ascend)
    *a.rows.err = DEV_INDEX;
    return;
  }
  const int64_t pos = len - n + (m - tok0);
  if (a.cos_t && pos >= a.T) {
    *a.rows.err = DEV_INDEX;
    return;
  }
  const int which = h < a.nh ? 0 : h < a.nh + a.nkv ? 1 : 2;
  const int hh = which == 0 ? h : which == 1 ? h - a.nh : h - a.nh - a.nkv;
  const TI* src = which == 0 ? (const TI*)a.q + m * a.q_ld + hh * a.q_hs : which == 1 ? (const TI*)a.k + m * a.k_ld + hh * a.k_hs : (const TI*)a.v + m * a.v_ld + hh * a.v_hs;
  TO* dst;
  if (which == 0) {
    dst = (TO*)a.q_out + (m * a.nh + hh) * a.d;
  } else {
    const int64_t page = page_of(a.rows, row, pos);
    if (page < 0) return;
    dst = (which == 1 ? (TO*)a.k_pages : (TO*)a.v_pages) + ((((page * a.nkv + hh) << a.rows.lg) + (pos & ((1 << a.rows.lg) - 1))) * a.d);
  }
  const int pairs = a.d / 2;
  float x[4], y[4];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = lane + 32 * i;
    x[i] = y[i] = 0.f;
    if (p < pairs) {
      const bool halves = a.rot_half && p < a.half;
      x[i] = load1(src + (halves ? p : 2 * p));
      y[i] = load1(src + (halves ? p + a.half : 2 * p + 1));
    }
    ss += x[i] * x[i] + y[i] * y[i];
  }
  const float* gain = which == 0 ? a.q_gain : which == 1 ? a.k_gain : nullptr;
  float f = 1.f;
  if (gain) {
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    f = 1.f / sqrtf(ss / (float)a.d + a.eps);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = lane + 32 * i;
    if (p >= pairs) continue;
    const bool halves = a.rot_half && p < a.half;
    const int c0 = halves ? p : 2 * p, c1 = halves ? p + a.half : 2 * p + 1;
    float u = x[i], w = y[i];
    if (gain) {
      const float one = a.plus_one ? 1.f : 0.f;
      u = u * f * (one + gain[c0]);
      w = w * f * (one + gain[c1]);
    }
    if (which < 2 && p < a.half) {
      const float cs = a.cos_t[pos * a.half + p], sn = a.sin_t[pos * a.half + p];
      const float t = u * cs - w * sn;
      w = w * cs + u * sn;
      u = t;
    }
    store1(dst + c0, u);
    store1(dst + c1, w);
  }
}

// Eight neighbouring values, loaded as they are stored.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = __ldg((const float4*)p); b = __ldg((const float4*)p + 1); }
  __device__ __forceinline__ void get(float* x) const { x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w; }
  static __device__ __forceinline__ void put(float* p, const float* x) {
    *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
    *((float4*)p + 1) = make_float4(x[4], x[5], x[6], x[7]);
  }
};
template <>
struct Eight<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = __ldg((const uint4*)p); }
  __device__ __forceinline__ void get(float* x) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *(const uint32_t*)&v;
    }
    *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// The same for head sizes 16 G, G a power of two, aligned vectors and angles in eights: G lanes have a vector, each two pieces of eight values,
// which are the two sides of its eight pairs (with `rot_half` where they turn), or 16 neighbours.  A warp has one of `parts` shares of a
// token's heads, U times 32 / G of them, all on their way before the token's row is looked up.
//
// Bytes should bound it (read once, written once).  They do not (0.68 of the copy rate), nor does issue (56 % of its slots): 96 registers leave a scheduler 4
// warps, each of which waits 6.8 clocks from one instruction to the next, 1.9 for dependent arithmetic, 0.8 for the norm's shuffles, 0.8 for memory.  6 rows of up to 2903 tokens, 32 + 2 x 4 heads of 128 with norms, bf16: 251 MB in 56.8 us, 4.4 TB/s.  The steps
// there, from 225 us: vectors in eights 77, all of a lane's vectors on their way at once 62, neighbouring heads in a warp, so that
// gains stay in registers, 57.  Of a single step's tokens the call's 4.9 us are all.
template <typename TI>
constexpr int append_vectors() { return sizeof(TI) == 2 ? 4 : 2; }
template <typename TI, typename TO, int G>
__global__ void __launch_bounds__(128, 5) k_paged_append_vec(AppendArgs a, int parts) {
  constexpr int VPI = 32 / G, U = append_vectors<TI>();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, g = lane % G;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), m = w / parts;
  if (m >= a.rows.M) return;
  const int heads = a.nh + 2 * a.nkv, share = (heads + VPI * parts - 1) / (VPI * parts);  // (at most U)
  const int h0 = (int)(w - m * parts) * share * VPI + lane / G, stop = min(heads, h0 - lane / G + share * VPI);
  // this lane's two pieces of every vector
  const int turned = a.half / 8;  // lanes whose pairs turn, with rot_half
  const int c0 = a.rot_half ? (g < turned ? 8 * g : 2 * a.half + 16 * (g - turned)) : 16 * g, c1 = a.rot_half && g < turned ? c0 + a.half : c0 + 8;
  auto source = [&](int h) {
    return h < a.nh ? (const TI*)a.q + m * a.q_ld + h * a.q_hs
                    : h < a.nh + a.nkv ? (const TI*)a.k + m * a.k_ld + (h - a.nh) * a.k_hs : (const TI*)a.v + m * a.v_ld + (h - a.nh - a.nkv) * a.v_hs;
  };
  Eight<TI> in[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (h0 + u * VPI < stop) {
      const TI* src = source(h0 + u * VPI);
      in[u][0].load(src + c0);
      in[u][1].load(src + c1);
    }
  // the token's row (as many rows as end at or before it), position and page
  int64_t row = 0;
  for (int64_t i = lane; i - lane < a.rows.rows; i += 32)
    row += __popc(__ballot_sync(0xffffffffu, i < a.rows.rows && a.rows.starts[i + 1] <= m));
  if (row >= a.rows.rows) return;  // behind the last row
  int64_t tok0, n, len;
  if (!row_span(a.rows, row, a.rows.M, &tok0, &n, &len) || m < tok0) return;
  if (m >= tok0 + n) {  // (starts that do not ascend)
    *a.rows.err = DEV_INDEX;
    return;
  }
  const int64_t pos = len - n + (m - tok0);
  if (a.cos_t && pos >= a.T) {
    *a.rows.err = DEV_INDEX;
    return;
  }
  const int64_t page = page_of(a.rows, row, pos);
  const int64_t at = page < 0 ? 0 : (((page * a.nkv) << a.rows.lg) + (pos & ((1 << a.rows.lg) - 1))) * a.d;
  // (pair i: components c0 + i and c1 + i with rot_half, else neighbours c0 + 2 i and c0 + 2 i + 1)
  float cs[8], sn[8];
  const bool turns = a.rot_half ? g < turned : 8 * g < a.half;
  if (turns) {
    Eight<float> t;
    t.load(a.cos_t + pos * a.half + 8 * g);
    t.get(cs);
    t.load(a.sin_t + pos * a.half + 8 * g);
    t.get(sn);
  }
  const float one = a.plus_one ? 1.f : 0.f, over_d = 1.f / (float)a.d;
  const float* have = nullptr;
  float gx[8], gy[8];  // the gains at `have`
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * VPI;
    if (h - lane / G >= stop) break;  // (uniform)
    float x[8], y[8];
    in[u][0].get(x);
    in[u][1].get(y);
    const int which = h < a.nh ? 0 : h < a.nh + a.nkv ? 1 : 2;
    const float* gain = which == 0 ? a.q_gain : which == 1 ? a.k_gain : nullptr;
    if (a.q_gain || a.k_gain) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
#pragma unroll
      for (int o = G / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (gain) {
        if (gain != have) {
          Eight<float> t;
          t.load(gain + c0);
          t.get(gx);
          t.load(gain + c1);
          t.get(gy);
#pragma unroll
          for (int i = 0; i < 8; ++i) { gx[i] += one; gy[i] += one; }
          have = gain;
        }
        const float f = rsqrtf(ss * over_d + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = x[i] * f * gx[i];
          y[i] = y[i] * f * gy[i];
        }
      }
    }
    if (turns && which < 2) {
      if (a.rot_half) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float t = x[i] * cs[i] - y[i] * sn[i];
          y[i] = y[i] * cs[i] + x[i] * sn[i];
          x[i] = t;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float t = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i], r = y[2 * i] * cs[4 + i] - y[2 * i + 1] * sn[4 + i];
          x[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
          y[2 * i + 1] = y[2 * i + 1] * cs[4 + i] + y[2 * i] * sn[4 + i];
          x[2 * i] = t;
          y[2 * i] = r;
        }
      }
    }
    if (h < stop && (which == 0 || page >= 0)) {
      TO* dst = which == 0 ? (TO*)a.q_out + (m * a.nh + h) * a.d
                           : (which == 1 ? (TO*)a.k_pages : (TO*)a.v_pages) + at + ((int64_t)(h - a.nh - (which == 2 ? a.nkv : 0)) << a.rows.lg) * a.d;
      Eight<TO>::put(dst + c0, x);
      Eight<TO>::put(dst + c1, y);
    }
  }
}

struct ReorderArgs {
  const uint32_t *parents, *lens, *own;
  uint32_t* table;
  char *k_pages, *v_pages;
  int64_t cols, n_pages, layer_bytes;  // bytes of a layer's pages
  int lg, K, nkv, token_bytes;         // bytes of a head's token
  int pools;                           // layers, keys and values
  int32_t* err;
};

// Group blockIdx.y.  All of a group's copies go through the registers of the thread that makes them: it has read the K sources of
// its 16 bytes before it writes them, so pages may change places.  The sources are the parents' own pages, which nobody
// else's targets are.  What bounds it is the bytes; a block looks its group up once and then has pieces of all layers.  12 groups of 8
// beams, 8 layers of 8 heads of 128: 77 MB in 18.4 us, 4.2 TB/s (with the call's 3.8 us, which is all that one group of 4 takes).
template <int KM>
__global__ void __launch_bounds__(256) k_paged_reorder(ReorderArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int64_t src[KM], dst[KM];
  __shared__ int par[KM];
  const int64_t row0 = (int64_t)blockIdx.y * a.K;
  const int j = threadIdx.x;
  const int64_t len = a.lens[row0], cur = len >> a.lg;
  const int begun = (int)(len & ((1 << a.lg) - 1));
  bool ok = true;
  if (j < a.K) {
    const uint32_t p = a.parents[row0 + j];
    ok = p < (uint32_t)a.K && a.lens[row0 + j] == len && cur + (begun > 0) <= a.cols;
    par[j] = (int)p;
    src[j] = dst[j] = 0;
    if (ok && begun) {
      src[j] = a.own[(row0 + p) * a.cols + cur];
      dst[j] = a.own[(row0 + j) * a.cols + cur];
      ok = src[j] < a.n_pages && dst[j] < a.n_pages;
    }
  }
  __syncthreads();
  if (begun && j < a.K)
    for (int i = 0; i < j; ++i) ok = ok && dst[i] != dst[j];  // (a page of its own)
  if (__syncthreads_or(!ok)) {
    if (j == 0) *a.err = DEV_INDEX;
    return;
  }
  const int64_t t0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
  if (begun) {
    const uint32_t head_bytes = (uint32_t)a.token_bytes << a.lg, per = (uint32_t)begun * (uint32_t)a.token_bytes / 16;  // 16-byte pieces of a head
    const int64_t page_bytes = (int64_t)a.nkv * head_bytes, all = (int64_t)per * a.nkv * a.pools;
    for (int64_t i = t0; i < all; i += step) {
      const int64_t ph = i / per;
      const uint32_t pool = (uint32_t)(ph / a.nkv), h = (uint32_t)(ph - (int64_t)pool * a.nkv), off = (uint32_t)(i - ph * per) * 16u;
      char* base = (pool & 1 ? a.v_pages : a.k_pages) + (int64_t)(pool >> 1) * a.layer_bytes + (int64_t)h * head_bytes + off;
      uint4 x[KM];
#pragma unroll
      for (int q = 0; q < KM; ++q)
        if (q < a.K && par[q] != q) x[q] = *(const uint4*)(base + src[q] * page_bytes);
#pragma unroll
      for (int q = 0; q < KM; ++q)
        if (q < a.K && par[q] != q) *(uint4*)(base + dst[q] * page_bytes) = x[q];
    }
  }
  for (int64_t p = t0; p < a.cols; p += step) {
    uint32_t x[KM];
#pragma unroll
    for (int q = 0; q < KM; ++q)
      if (q < a.K) x[q] = p < cur ? a.table[(row0 + par[q]) * a.cols + p] : a.own[(row0 + q) * a.cols + p];
#pragma unroll
    for (int q = 0; q < KM; ++q)
      if (q < a.K) a.table[(row0 + q) * a.cols + p] = x[q];
  }
}

// [M, heads, d], the components next to each other
int check_vectors(cg_ctx* c, const cg_tensor* t, const char* what, int64_t M, int64_t heads, int64_t d) {
  const int64_t dims[3] = {M, heads, d};
  CG_TRY(check_tensor(c, t, what, CG_F32, 3, dims, false));
  if (t->strides[2] != 1 && M > 0) return fail(c, CG_ERR_UNSUPPORTED, std::string(what) + ": the last axis must be contiguous");
  return CG_OK;
}

template <typename TI, typename TO, int G>
int launch_vec(cg_ctx* c, const AppendArgs& a) {
  // Shares of a token: as many vectors as a lane holds; of few tokens smaller ones, until every SM has 32 warps.
  const int heads = a.nh + 2 * a.nkv, most = (heads + 32 / G - 1) / (32 / G);
  int parts = (most + append_vectors<TI>() - 1) / append_vectors<TI>();
  while (2 * parts <= most && a.rows.M * parts < 148 * 32) parts *= 2;
  CG_CUDA(c, launch_kernel(c, k_paged_append_vec<TI, TO, G>, dim3((unsigned)((a.rows.M * parts + 3) / 4)), dim3(128), 0, 1, a, parts));
  CG_LAUNCHED(c);
  return CG_OK;
}

template <typename TI, typename TO>
int launch_append(cg_ctx* c, const AppendArgs& a) {
  constexpr int64_t in = 16 / sizeof(TI);
  const bool aligned = ((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.cos_t | (uintptr_t)a.sin_t | (uintptr_t)a.q_gain |
                        (uintptr_t)a.k_gain) % 16 == 0 &&
                       (a.q_ld | a.q_hs | a.k_ld | a.k_hs | a.v_ld | a.v_hs) % in == 0 && a.half % 8 == 0;
  if (aligned) {
    if (a.d == 32) return launch_vec<TI, TO, 2>(c, a);
    if (a.d == 64) return launch_vec<TI, TO, 4>(c, a);
    if (a.d == 128) return launch_vec<TI, TO, 8>(c, a);
    if (a.d == 256) return launch_vec<TI, TO, 16>(c, a);
  }
  const int64_t vectors = a.rows.M * (a.nh + 2 * a.nkv);
  CG_CUDA(c, launch_kernel(c, k_paged_append<TI, TO>, dim3((unsigned)((vectors + 7) / 8)), dim3(256), 0, 1, a));
  CG_LAUNCHED(c);
  return CG_OK;
}

template <int KM>
int launch_reorder(cg_ctx* c, const ReorderArgs& a, int64_t groups) {
  // At most what runs at a time (four blocks of 256 per SM), at least a block per group.
  const int64_t pieces = std::max<int64_t>((((int64_t)a.nkv * a.token_bytes) << a.lg) / 16 * a.pools, a.cols);
  const int64_t blocks = std::min<int64_t>((pieces + 255) / 256, std::max<int64_t>(148 * 4 / groups, 1));
  CG_CUDA(c, launch_kernel(c, k_paged_reorder<KM>, dim3((unsigned)blocks, (unsigned)groups), dim3(256), 0, 1, a));
  CG_LAUNCHED(c);
  return CG_OK;
}

}  // namespace

}  // namespace cg

using namespace cg;

extern "C" {

int32_t cg_paged_append(cg_ctx* c, const cg_tensor* q, const cg_tensor* k, const cg_tensor* v, const cg_tensor* q_gain, const cg_tensor* k_gain,
                        float eps, int32_t plus_one, const cg_tensor* cos_t, const cg_tensor* sin_t, int32_t rot_half, const cg_tensor* table,
                        const cg_tensor* starts, const cg_tensor* lens, cg_tensor* k_pages, cg_tensor* v_pages, cg_tensor* q_out) {
  if (!c) return CG_ERR_INVALID;
  CG_LAZY_EAGER_SCOPE(c);
  OnDevice on(c);
  if (!k || !v || !q != !q_out) return fail(c, CG_ERR_INVALID, "null argument");
  AppendArgs a = {};
  int lg;
  CG_TRY(check_pages(c, k_pages, v_pages, false, &lg));
  const int64_t nkv = k_pages->dims[1], d = k_pages->dims[3], any[3] = {-1, -1, -1};
  CG_TRY(check_tensor(c, k, "k", CG_F32, 3, any, false));
  const int64_t M = k->dims[0];
  CG_TRY(check_vectors(c, k, "k", M, nkv, d));
  CG_TRY(check_vectors(c, v, "v", M, nkv, d));
  CG_TRY(check_rows(c, table, starts, lens, M, k_pages->dims[0], lg, &a.rows));
  a.nh = 0;
  if (q) {
    CG_TRY(check_tensor(c, q, "q", CG_F32, 3, any, false));
    CG_TRY(check_vectors(c, q, "q", M, q->dims[1], d));
    CG_TRY(check_tensor(c, q_out, "q_out", CG_F32, 3, q->dims));
    if (q_out->storage != k_pages->storage) return fail(c, CG_ERR_DTYPE, "q_out is stored as the pages are");
    if (q->dims[1] > 65535) return fail(c, CG_ERR_UNSUPPORTED, "too many heads");
    a.nh = (int)q->dims[1];
  }
  if (nkv > 65535) return fail(c, CG_ERR_UNSUPPORTED, "too many heads");
  if (k->storage != v->storage || (q && q->storage != k->storage)) return fail(c, CG_ERR_DTYPE, "q, k and v are stored differently");
  const int64_t dd[1] = {d};
  for (const cg_tensor* g : {q_gain, k_gain})
    if (g) {
      CG_TRY(check_tensor(c, g, "gain", CG_F32, 1, dd));
      if (g->storage != ST_F32) return fail(c, CG_ERR_DTYPE, "gains are f32");
    }
  if (!cos_t != !sin_t) return fail(c, CG_ERR_INVALID, "cos without sin");
  if (cos_t) {
    CG_TRY(check_tensor(c, cos_t, "cos", CG_F32, 2, any));
    CG_TRY(check_tensor(c, sin_t, "sin", CG_F32, 2, cos_t->dims));
    if (cos_t->storage != ST_F32 || sin_t->storage != ST_F32) return fail(c, CG_ERR_DTYPE, "angles are f32");
    if (2 * cos_t->dims[1] > d) return fail(c, CG_ERR_SHAPE, "more angles than pairs of a head");
  }
  if (overlap_any({q, k, v, q_gain, k_gain, cos_t, sin_t, table, starts, lens}, {k_pages, v_pages, q_out}))
    return fail(c, CG_ERR_INVALID, "what is written overlaps an input or each other");
  if (M == 0 || a.rows.rows == 0 || a.nh + 2 * nkv == 0) return CG_OK;
  a.q = q ? q->data() : nullptr; a.k = k->data(); a.v = v->data();
  if (q) { a.q_ld = q->strides[0]; a.q_hs = q->strides[1]; }
  a.k_ld = k->strides[0]; a.k_hs = k->strides[1];
  a.v_ld = v->strides[0]; a.v_hs = v->strides[1];
  a.q_gain = q_gain ? (const float*)q_gain->data() : nullptr;
  a.k_gain = k_gain ? (const float*)k_gain->data() : nullptr;
  a.eps = eps; a.plus_one = plus_one;
  if (cos_t) {
    a.cos_t = (const float*)cos_t->data(); a.sin_t = (const float*)sin_t->data();
    a.T = cos_t->dims[0]; a.half = (int)cos_t->dims[1];
  }
  a.rot_half = rot_half;
  a.q_out = q_out ? q_out->data() : nullptr;
  a.k_pages = k_pages->data(); a.v_pages = v_pages->data();
  a.nkv = (int)nkv; a.d = (int)d;
  if ((M * (a.nh + 2 * nkv) + 7) / 8 > 0x7FFFFFFFll) return fail(c, CG_ERR_UNSUPPORTED, "too many tokens");
  written(k_pages);
  written(v_pages);
  if (q_out) written(q_out);
  const bool in16 = k->storage == ST_BF16, out16 = k_pages->storage == ST_BF16;
  if (in16) return out16 ? launch_append<__nv_bfloat16, __nv_bfloat16>(c, a) : launch_append<__nv_bfloat16, float>(c, a);
  return out16 ? launch_append<float, __nv_bfloat16>(c, a) : launch_append<float, float>(c, a);
}

int32_t cg_paged_reorder(cg_ctx* c, const cg_tensor* parents, const cg_tensor* lens, const cg_tensor* own, cg_tensor* table, cg_tensor* k_pages,
                         cg_tensor* v_pages) {
  if (!c) return CG_ERR_INVALID;
  CG_LAZY_EAGER_SCOPE(c);
  OnDevice on(c);
  if (!parents || !lens || !own || !table || !k_pages || !v_pages) return fail(c, CG_ERR_INVALID, "null argument");
  ReorderArgs a = {};
  const bool layers = k_pages->rank == 5;
  CG_TRY(check_pages(c, k_pages, v_pages, layers, &a.lg));
  const int64_t any[2] = {-1, -1}, *dims = k_pages->dims + (layers ? 1 : 0);
  CG_TRY(check_tensor(c, parents, "parents", CG_U32, 2, any));
  const int64_t B = parents->dims[0], K = parents->dims[1], L = layers ? k_pages->dims[0] : 1;
  const int64_t rows[1] = {B * K}, tab[2] = {B * K, -1};
  CG_TRY(check_tensor(c, lens, "lens", CG_U32, 1, rows));
  CG_TRY(check_tensor(c, table, "table", CG_U32, 2, tab));
  CG_TRY(check_tensor(c, own, "own", CG_U32, 2, table->dims));
  if (K > 32) return fail(c, CG_ERR_UNSUPPORTED, "at most 32 beams");
  if (B > 65535 || L > 1ll << 24 || dims[1] > 65535) return fail(c, CG_ERR_UNSUPPORTED, "too many groups, layers or heads");
  if (overlap_any({parents, lens, own}, {table, k_pages, v_pages})) return fail(c, CG_ERR_INVALID, "what is written overlaps an input or each other");
  if (B == 0 || K == 0 || table->dims[1] == 0 || L == 0) return CG_OK;
  a.parents = (const uint32_t*)parents->data();
  a.lens = (const uint32_t*)lens->data();
  a.own = (const uint32_t*)own->data();
  a.table = (uint32_t*)table->data();
  a.k_pages = (char*)k_pages->data();
  a.v_pages = (char*)v_pages->data();
  a.cols = table->dims[1];
  a.n_pages = dims[0];
  a.K = (int)K;
  a.nkv = (int)dims[1];
  a.token_bytes = (int)(dims[3] * k_pages->esize());
  a.layer_bytes = dims[0] * dims[1] * dims[2] * a.token_bytes;
  a.pools = (int)(2 * L);
  a.err = c->core->dev_err;
  written(table);
  written(k_pages);
  written(v_pages);
  if (K <= 4) return launch_reorder<4>(c, a, B);
  if (K <= 8) return launch_reorder<8>(c, a, B);
  if (K <= 16) return launch_reorder<16>(c, a, B);
  return launch_reorder<32>(c, a, B);
}

}  // extern "C"
