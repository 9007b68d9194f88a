// paged_attn.h — the arguments of attention over a paged cache, and the kernels it is run on.
#pragma once

#include "mma.cuh"
#include "paged.h"

namespace cg {

struct PagedAttnArgs {
  PagedRows rows;
  const void *q, *k_pages, *v_pages;
  void* out;
  int64_t q_ld, q_hs;   // from one token and one head of q to the next
  int64_t most;         // new tokens of a row, at most
  int64_t window;       // 0 = none
  float scale, cap;     // cap 0 = none
  int nh, nkv, d;
};

// Soft-caps c tanh(x / c), in units of log2: kernels take c log2(e) and the factors of a product q k in x / c (`in`) and in the exponent
// of 2 of exp(-2 x / c) (`unit`).  tanh(y) / y in y^2 up to y = 3/4, fitted to the least largest relative error: 3e-8, half a step
// of f32.  Beyond that 2 / (1 + e^-2y) - 1, which would lose what is small against 1.
constexpr CG_HD float tanh_term(int i) {
  return i == 0 ? 1.f : i == 1 ? -0.33332958817481995f : i == 2 ? 0.1332540661096573f : i == 3 ? -0.05334442853927612f
       : i == 4 ? 0.019582903012633324f : -0.004716253839433193f;
}
#ifdef __CUDACC__
__device__ __forceinline__ float soft_cap_near(float y, float cap_log2e) {
  const float u = y * y;
  float f = tanh_term(5);
#pragma unroll
  for (int i = 4; i >= 0; --i) f = fmaf(f, u, tanh_term(i));
  return cap_log2e * y * f;
}
__device__ __forceinline__ float soft_cap(float x, float cap_log2e, float in, float unit) {
  const float y = x * in, far = fmaf(2.f * cap_log2e, rcp_newton(1.f + fast_exp2(x * unit)), -cap_log2e);
  float v;  // (both are worked out: a branch per score costs more)
  asm("{\n\t.reg .pred p;\n\tsetp.le.f32 p, %1, 0f3F400000;\n\tselp.f32 %0, %2, %3, p;\n\t}" : "=f"(v) : "f"(fabsf(y)), "f"(soft_cap_near(y, cap_log2e)), "f"(far));
  return v;
}
#endif

// Prompts in bf16 on tcgen05 (paged_fa.cu)
bool paged_fa_supported(const PagedAttnArgs& a);
int paged_fa(cg_ctx* c, const PagedAttnArgs& a);
// A few tokens per row, bf16 (paged_dec.cu)
bool paged_dec_supported(const PagedAttnArgs& a);
int paged_dec(cg_ctx* c, const PagedAttnArgs& a);

// ---- into how many shares a row's keys are cut ----
constexpr int SHARES = 5;  // 1, 2, 4, 8 or 16: the blocks of a cluster

// Clusters of 1, 2, .. blocks along z that run at a time (asked once per kernel, which keeps `known`); -1: none.
struct AtATime {
  int n[64][SHARES] = {};
};
template <typename... KArgs>
int at_a_time(AtATime& known, int device, int i, void (*kernel)(KArgs...), int threads, size_t smem) {
  int& n = known.n[device & 63][i];
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1024, 1, 1u << i);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1u << i;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int got = 0;
    if (cudaOccupancyMaxActiveClusters(&got, kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      got = 0;
    }
    n = got > 0 ? got : -1;
  }
  return n;
}
// The shares of least time: a block takes `base` us and `round` for each of its rounds of `keys` keys, joining 2 to 4.5.  What does not run
// at the same time takes turns (between whole turns and their mean, as rows differ): clusters beyond at_a_time, and, where one
// block keeps an SM's units busy, blocks beyond the SMs; part_seen is what of a row a query sees in the mean, 0 where that
// does not count.
template <typename F>
int pick_shares(F&& n_of, int most, int64_t clusters, int64_t keys_of_row, int keys, double base, double round, double part_seen) {
  constexpr double join[SHARES] = {0., 2., 2., 2.5, 4.5};
  int shares = 1;
  double best = 1e300;
  for (int i = 0; i < SHARES && 1 << i <= most; ++i) {
    const int n = n_of(i);
    if (n <= 0) continue;
    auto turns_of = [](double x) { return 0.5 * (x + (double)(int64_t)(x + 0.999999)); };
    double turns = turns_of((double)clusters / n);
    const double by_sm = turns_of((double)(clusters << i) * part_seen / 148.);
    if (part_seen > 0. && by_sm > turns) turns = by_sm;
    const int64_t tiles = keys_of_row / keys + 1;
    const double cost = (turns > 1. ? turns : 1.) * (base + join[i] + round * (double)((tiles + (1 << i) - 1) >> i));
    if (cost < best) {
      best = cost;
      shares = 1 << i;
    }
  }
  return shares;
}

}  // namespace cg
