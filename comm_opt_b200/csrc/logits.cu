// Repetition, frequency and presence penalties, sparse biases and grammar masks on logits, in one pass.
//
// A CTA owns one row and a chunk of its vocabulary. It counts the row's token history inside its chunk in shared
// memory (integer atomics: any order gives the same counts; the top bit says that the prompt held the id, the
// rest how often the output did), sums the row's sparse biases in their order, and then streams the chunk once:
// load, penalise, mask, round, store - and, for greedy decoding, fold the stored value into the row's argmax
// key. Nothing is kept between calls. Bound by the logits' bytes; each CTA also reads the row's whole history
// from L2, so chunks grow with the history.
#include <algorithm>

#include "common.cuh"
#include "serve_ops.h"

namespace cob {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kInPrompt = 0x80000000u;

__device__ __forceinline__ unsigned long long greedy_key(float v, uint32_t idx) {
  uint32_t u = __float_as_uint(v);
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (0xFFFFFFFFu - idx);
}

// The row's scalars, and one id's chain of roundings. Products and differences are rounded one by one (no fused
// multiply-add), so the result is that of the same formula written in elementwise fp32 operations.
struct RowScalars {
  float rep, freq, pres;
  bool has_rep, has_freq, has_pres;
  __device__ __forceinline__ float apply(float x, uint32_t c) const {
    if (c != 0) {
      if (has_rep) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      const uint32_t n = c & ~kInPrompt;
      if (n != 0) {
        if (has_freq) x = __fsub_rn(x, __fmul_rn(freq, (float)n));
        if (has_pres) x = __fsub_rn(x, pres);
      }
    }
    return x;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) k_penalize(const __grid_constant__ LogitsParams p, int chunk, int counts,
                                                       int biases) {
  using V = Vec<T>;
  extern __shared__ __align__(16) uint32_t sm[];
  __shared__ float sval[32];
  __shared__ unsigned long long skey[kThreads / 32];
  pdl_wait_then_trigger();
  const int row = blockIdx.x;
  const T* in = reinterpret_cast<const T*>(p.logits) + row * p.ld_in;
  T* out = reinterpret_cast<T*>(p.out) + row * p.ld_out;
  // ids up to the row's first 16-byte boundary belong to the first chunk; every chunk then starts on one
  const int lead = min(p.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(in) & 15)) & 15) / (int)sizeof(T));
  const long long body0 = lead + (long long)blockIdx.y * chunk;
  const int v0 = (int)min((long long)p.vocab, body0);
  const int v1 = (int)min((long long)p.vocab, body0 + chunk);
  const int lo = blockIdx.y == 0 ? 0 : v0;  // first id of this CTA
  const int n = v1 - lo;
  if (n <= 0) return;
  const int slots = chunk + V::N;
  uint32_t* cnt = sm;
  float* bsum = reinterpret_cast<float*>(sm + (counts ? slots : 0));
  const int words = (counts ? slots : 0) + (biases ? slots : 0);
  for (int i = threadIdx.x; i < words; i += kThreads) sm[i] = 0u;
  __syncthreads();
  const int g0 = p.vocab_offset + lo;  // global id of slot 0
  if (counts) {
    const int32_t* tok = p.tokens + row * p.ld_tokens;
    const int len = p.lens ? min(max(p.lens[row], 0), p.history) : p.history;
    const int plen = p.prompt_lens ? p.prompt_lens[row] : 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < len; i += kThreads) {
      const unsigned id = (unsigned)(tok[i] - g0);
      if (tok[i] >= g0 && id < (unsigned)n) {
        if (i < plen)
          atomicOr(cnt + id, kInPrompt);
        else
          atomicAdd(cnt + id, 1u);
      }
    }
  }
  if (biases && threadIdx.x < 32) {  // one warp, 32 entries at a time: equal ids add up in their order
    const int32_t* ids = p.bias_ids + (size_t)row * p.biases;
    const float* val = p.bias + (size_t)row * p.biases;
    const int lane = threadIdx.x;
    for (int i0 = 0; i0 < p.biases; i0 += 32) {
      const int i = i0 + lane;
      const int id = i < p.biases ? ids[i] : -1;
      const bool mine = id >= g0 && (unsigned)(id - g0) < (unsigned)n;
      if (!__any_sync(0xffffffffu, mine)) continue;
      sval[lane] = mine ? val[i] : 0.f;
      const unsigned same = __match_any_sync(0xffffffffu, mine ? id : -1 - lane);
      __syncwarp();
      if (mine && (same & ((1u << lane) - 1u)) == 0) {
        float s = bsum[id - g0];
        for (unsigned m = same; m; m &= m - 1) s = __fadd_rn(s, sval[__ffs(m) - 1]);
        bsum[id - g0] = s;
      }
      __syncwarp();
    }
  }
  __syncthreads();
  RowScalars r;
  r.has_rep = p.repetition != nullptr;
  r.has_freq = p.frequency != nullptr;
  r.has_pres = p.presence != nullptr;
  r.rep = r.has_rep ? p.repetition[row] : 1.f;
  r.freq = r.has_freq ? p.frequency[row] : 0.f;
  r.pres = r.has_pres ? p.presence[row] : 0.f;
  const uint32_t* mask = p.allowed ? p.allowed + row * p.ld_mask : nullptr;
  unsigned long long best = 0ull;
  auto one = [&](float x, int v) {  // v: id within this shard
    if (counts) x = r.apply(x, cnt[v - lo]);
    if (biases) x = __fadd_rn(x, bsum[v - lo]);
    if (mask) {
      const int g = p.vocab_offset + v;
      if (!((__ldg(mask + (g >> 5)) >> (g & 31)) & 1u)) x = -INFINITY;
    }
    return x;
  };
  auto single = [&](int v) {
    const T o = from_f<T>(one(to_f(in[v]), v));
    out[v] = o;
    if (p.keys) best = max(best, greedy_key(to_f(o), (uint32_t)(p.vocab_offset + v)));
  };
  const int nv = (v1 - v0) / V::N;  // whole vectors
  const bool vec_store = ((reinterpret_cast<uintptr_t>(out + v0)) & 15) == 0;
  for (int i = threadIdx.x; i < nv; i += kThreads) {
    const int v = v0 + i * V::N;
    float f[V::N];
    V::to_float(*reinterpret_cast<const uint4*>(in + v), f);
#pragma unroll
    for (int j = 0; j < V::N; ++j) f[j] = one(f[j], v + j);
    const uint4 o = V::from_float(f);
    if (vec_store) {
      *reinterpret_cast<uint4*>(out + v) = o;
    } else {
#pragma unroll
      for (int j = 0; j < V::N; ++j) out[v + j] = from_f<T>(f[j]);
    }
    if (p.keys) {
      V::to_float(o, f);
#pragma unroll
      for (int j = 0; j < V::N; ++j) best = max(best, greedy_key(f[j], (uint32_t)(p.vocab_offset + v + j)));
    }
  }
  for (int v = lo + threadIdx.x; v < v0; v += kThreads) single(v);
  for (int v = v0 + nv * V::N + threadIdx.x; v < v1; v += kThreads) single(v);
  if (!p.keys) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((threadIdx.x & 31) == 0) skey[threadIdx.x >> 5] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) best = max(best, skey[w]);
    atomicMax(p.keys + row, best);
  }
}

template <typename T>
cudaError_t launch(const LogitsParams& p, cudaStream_t s) {
  const int counts = p.tokens != nullptr && p.history > 0 && (p.repetition || p.frequency || p.presence);
  const int biases = p.bias != nullptr && p.biases > 0;
  int chunk = 4096;
  while (chunk > 1024 && (long long)p.rows * ((p.vocab + chunk - 1) / chunk) < 148 * 2) chunk /= 2;
  const size_t smem = (size_t)(counts + biases) * (chunk + Vec<T>::N) * 4;
  // the leading ids (fewer than a vector) shift the chunks by at most one vector
  const dim3 grid(p.rows, (p.vocab + chunk - 1) / chunk);
  return launch_k(k_penalize<T>, grid, dim3(kThreads), smem, s, p, chunk, counts, biases);
}

}  // namespace

cudaError_t penalize_logits(const LogitsParams& p, cudaStream_t s) {
  if (p.rows <= 0 || p.vocab <= 0 || p.vocab > (1 << 26)) return cudaErrorInvalidValue;
  switch (p.dtype) {
    case kF32: return launch<float>(p, s);
    case kF16: return launch<__half>(p, s);
    case kBF16: return launch<__nv_bfloat16>(p, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace cob
