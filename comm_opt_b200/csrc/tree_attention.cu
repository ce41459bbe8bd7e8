// Attention of a tree of drafted tokens over the paged KV cache.
//
// One warp per (sequence, drafted token, query head): the lanes share the head's components, the running maximum
// and sum of the softmax are in fp32, and the warp walks the row's visible slots.
#include "common.cuh"
#include "serve_ops.h"

namespace cob {
namespace {

constexpr int kPage = 16, kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) k_tree_attn(const __grid_constant__ TreeAttnParams p) {
  constexpr int E = D / 32;  // components per lane
  pdl_wait_then_trigger();
  const long long r = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= (long long)p.batch * p.tree * p.nq) return;
  const int h = (int)(r % p.nq), t = (int)(r / p.nq % p.tree), b = (int)(r / p.nq / p.tree);
  const int tl = p.tree_lens ? min(max(p.tree_lens[b], 0), p.tree) : p.tree;
  if (t >= tl) return;
  const int cap = p.max_blocks * kPage;
  const int ctx = min(max(p.ctx_lens[b], 0), cap), end = min(ctx + tl, cap);
  const unsigned long long bits =
      p.mask ? (unsigned long long)p.mask[b * p.mask_sb + t] : (t < 63 ? (2ull << t) - 1ull : ~0ull);
  const int kvh = h / (p.nq / p.nkv);
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_sb + t * p.q_st + h * p.q_sh;
  float qf[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    qf[i] = to_f(q[lane + 32 * i]) * p.scale * kLog2e;
    o[i] = 0.f;
  }
  for (int s = 0; s < end; ++s) {
    if (s >= ctx && !((bits >> (s - ctx)) & 1ull)) continue;
    const int blk = p.block_tables[(size_t)b * p.max_blocks + s / kPage];
    const bool ok = blk >= 0 && blk < p.num_blocks;  // a page outside the cache reads as zeros
    const size_t base = (((size_t)(ok ? blk : 0) * p.nkv + kvh) * kPage + s % kPage) * D;
    const T* k = reinterpret_cast<const T*>(p.k_cache) + base;
    const T* v = reinterpret_cast<const T*>(p.v_cache) + base;
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) d += qf[i] * (ok ? to_f(k[lane + 32 * i]) : 0.f);
    d = warp_sum(d);
    const float mn = fmaxf(m, d);
    const float a = m == -INFINITY ? 0.f : exp2f(m - mn), w = exp2f(d - mn);
    m = mn;
    l = l * a + w;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * a + w * (ok ? to_f(v[lane + 32 * i]) : 0.f);
  }
  T* out = reinterpret_cast<T*>(p.out) + b * p.o_sb + t * p.o_st + h * p.o_sh;
#pragma unroll
  for (int i = 0; i < E; ++i) out[lane + 32 * i] = from_f<T>(l == 0.f ? 0.f : o[i] / l);
}

template <typename T>
cudaError_t launch(const TreeAttnParams& p, cudaStream_t s) {
  const long long rows = (long long)p.batch * p.tree * p.nq;
  const dim3 grid((unsigned)((rows + kWarps - 1) / kWarps));
  return p.head_dim == 128 ? launch_k(k_tree_attn<T, 128>, grid, dim3(kWarps * 32), 0, s, p)
                           : launch_k(k_tree_attn<T, 64>, grid, dim3(kWarps * 32), 0, s, p);
}

}  // namespace

cudaError_t tree_attention(const TreeAttnParams& p, cudaStream_t s) {
  if ((p.head_dim != 64 && p.head_dim != 128) || p.batch <= 0 || p.tree <= 0 || p.tree > 64 || p.nkv <= 0 ||
      p.nq <= 0 || p.nq % p.nkv != 0 || p.max_blocks <= 0 || p.num_blocks <= 0)
    return cudaErrorInvalidValue;
  if (p.dtype == kBF16) return launch<__nv_bfloat16>(p, s);
  if (p.dtype == kF16) return launch<__half>(p, s);
  return cudaErrorInvalidValue;
}

}  // namespace cob
