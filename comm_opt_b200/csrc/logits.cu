// Repetition, frequency and presence penalties, sparse biases and grammar masks on logits, in one pass.
//
// A CTA owns one row and a chunk of its vocabulary. It counts the row's token history inside its chunk in shared
// memory (integer atomics: any order gives the same counts; the top bit says that the prompt held the id, the
// rest how often the output did), sums the row's sparse biases in their order, and then streams the chunk once:
// penalise the ids that a bit word marks as touched, mask, round, store - and, for greedy decoding, fold the stored value
// into the row's argmax key. Nothing is kept between calls. All first loads are issued together.
//
// Meant to be bound by the logits' bytes; each CTA also reads the row's whole history from L2. Measured on one B200, 128 rows
// of 152064 fp32 logits (159 MB): 25.6 us with nothing to do (6.2 TB/s), 41 us with histories of up to 2048 tokens (10 us),
// grammar masks (3.5) and 64 biases (2.7). Chunks of 4096 ids by 256 threads: 2048 took 46, 8192 60 us, when there was more
// to do per id. One row of 128256: 5.3 us with argmax_combine.
#include <algorithm>

#include "common.cuh"
#include "serve_ops.h"

namespace cob {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kInPrompt = 0x80000000u;

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

// `chunk` ids of one row; MAXV: 16-byte vectors of them per thread
template <typename T, int MAXV>
__global__ void __launch_bounds__(kThreads) k_penalize(const __grid_constant__ LogitsParams p, int chunk, int counts,
                                                       int biases) {
  using V = Vec<T>;
  constexpr int N = V::N;
  extern __shared__ __align__(16) uint32_t sm[];
  __shared__ int s_id[kThreads];
  __shared__ float s_val[kThreads];
  __shared__ unsigned long long s_key[kThreads / 32];
  pdl_wait_then_trigger();
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
  const int nv = (v1 - v0) / N;  // whole vectors
  const int g0 = p.vocab_offset + lo;  // first global id
  // Everything this CTA reads first is requested at once: the chunk, its mask words, the row's scalars, a tile of the
  // biases and a tile of the history (whose length is only applied afterwards), one memory latency for all.
  uint4 raw[MAXV];
  const uint32_t* mask = p.allowed ? p.allowed + row * p.ld_mask : nullptr;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int e = tid + i * kThreads;
    if (e < nv) {
      raw[i] = *reinterpret_cast<const uint4*>(in + v0 + e * N);
    }
  }
  // bit words of the chunk's ids v0 + 32 w ..: allowed, and touched by the history or a bias
  constexpr int kWords = MAXV * N * kThreads / 32, kPer = (kWords + kThreads - 1) / kThreads;
  __shared__ uint32_t s_mask[kWords], s_mark[kWords];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int w = tid + i * kThreads;
    const int g = (int)((unsigned)(p.vocab_offset + v0) + 32u * w);
    if (w < kWords) {
      s_mark[w] = 0;
      if (mask && 32 * w < v1 - v0) {
        const uint32_t a = __ldg(mask + (g >> 5));
        const uint32_t b = (g & 31) && (g | 31) < p.vocab_offset + p.vocab - 1 ? __ldg(mask + (g >> 5) + 1) : 0u;  // (ids reach 2^31 - 2)
        s_mask[w] = __funnelshift_r(a, b, g & 31);
      }
    }
  }
  constexpr int kTile = 4;
  const int32_t* tok = p.tokens + row * p.ld_tokens;
  int t[kTile];
  int len = 0, plen = 0;
  if (counts) {
    len = p.lens ? min(max(p.lens[row], 0), p.history) : p.history;
    plen = p.prompt_lens ? p.prompt_lens[row] : 0;
#pragma unroll
    for (int k = 0; k < kTile; ++k) t[k] = tid + k * kThreads < p.history ? tok[tid + k * kThreads] : -1;
  }
  const int32_t* ids = p.bias_ids + (size_t)row * p.biases;
  const float* val = p.bias + (size_t)row * p.biases;
  int bid = -1;
  float bval = 0.f;
  if (biases && tid < p.biases) bid = ids[tid], bval = val[tid];
  RowScalars r;
  r.has_rep = p.repetition != nullptr;
  r.has_freq = p.frequency != nullptr;
  r.has_pres = p.presence != nullptr;
  r.rep = r.has_rep ? p.repetition[row] : 1.f;
  r.freq = r.has_freq ? p.frequency[row] : 0.f;
  r.pres = r.has_pres ? p.presence[row] : 0.f;
  // id v has slot v - v0 + N of the tables (the few ids before v0 sit in the first N), so vectors are aligned there too
  const int slots = chunk + 2 * N, base = N - v0;
  uint32_t* cnt = sm;
  float* bsum = reinterpret_cast<float*>(sm + (counts ? slots : 0));
  const int words4 = ((counts ? slots : 0) + (biases ? slots : 0)) / 4;
  for (int i = tid; i < words4; i += kThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
  const int gs = p.vocab_offset - base;  // global id of slot 0
  auto mark = [&](int slot) {  // (the ids before v0 look their tables up without it)
    if (slot >= N) atomicOr(&s_mark[(slot - N) >> 5], 1u << ((slot - N) & 31));
  };
  // biases in tiles of one entry per thread; each warp takes the ids of one residue and adds them up 32 entries at a
  // time, equal ids in their order
  for (int i0 = 0;;) {
    const bool mine = (unsigned)bid - (unsigned)g0 < (unsigned)n;
    s_id[tid] = mine ? bid - gs : -1;
    s_val[tid] = bval;
    const int here = biases ? min(kThreads, p.biases - i0) : 0;
    i0 += kThreads;
    const bool more = biases && i0 < p.biases;
    if (more) {
      bid = i0 + tid < p.biases ? ids[i0 + tid] : -1;
      bval = i0 + tid < p.biases ? val[i0 + tid] : 0.f;
    }
    __syncthreads();  // (the first also completes the tables' zeros)
    for (int t0 = 0; t0 < here; t0 += 32) {
      const int e = s_id[t0 + lane], at = e >= 0 && e % (kThreads / 32) == warp ? e : -1;
      if (!__any_sync(0xffffffffu, at >= 0)) continue;
      const unsigned same = __match_any_sync(0xffffffffu, at >= 0 ? at : -1 - lane);
      if (at >= 0 && (same & ((1u << lane) - 1u)) == 0) {
        float s = bsum[at];
        for (unsigned m = same; m; m &= m - 1) s = __fadd_rn(s, s_val[t0 + __ffs(m) - 1]);
        bsum[at] = s;
        mark(at);
      }
      __syncwarp();
    }
    if (!more) break;
    __syncthreads();
  }
  if (counts) {
    for (int i0 = tid; i0 < len;) {
      int ahead[kTile];  // the next tile is on its way while this one is counted
#pragma unroll
      for (int k = 0; k < kTile; ++k) {
        const int i = i0 + (kTile + k) * kThreads;
        ahead[k] = i < len ? tok[i] : -1;
      }
#pragma unroll
      for (int k = 0; k < kTile; ++k) {
        const int i = i0 + k * kThreads;
        // (one unsigned comparison: ids below 2^31 and negative ones never wrap into the chunk)
        if (i < len && (unsigned)t[k] - (unsigned)g0 < (unsigned)n) {
          mark(t[k] - gs);
          if (i < plen)
            atomicOr(cnt + (t[k] - gs), kInPrompt);
          else
            atomicAdd(cnt + (t[k] - gs), 1u);
        }
      }
      i0 += kTile * kThreads;
#pragma unroll
      for (int k = 0; k < kTile; ++k) t[k] = ahead[k];
    }
  }
  unsigned long long best = 0ull;
  __syncthreads();
  auto single = [&](int v) {
    float x = to_f(in[v]);
    if (counts) x = r.apply(x, cnt[v + base]);
    if (biases) x = __fadd_rn(x, bsum[v + base]);
    const int g = p.vocab_offset + v;
    if (mask && !((__ldg(mask + (g >> 5)) >> (g & 31)) & 1u)) x = -INFINITY;
    const T o = from_f<T>(x);
    out[v] = o;
    if (p.keys) best = max(best, greedy_key(to_f(o), (uint32_t)g));
  };
  const bool vec_store = ((reinterpret_cast<uintptr_t>(out + v0)) & 15) == 0;
#pragma unroll
  for (int i = 0; i < MAXV; ++i) {
    const int e = tid + i * kThreads;
    if (e >= nv) break;
    const int v = v0 + e * N, slot = N + e * N, g = p.vocab_offset + v;
    float f[N];
    V::to_float(raw[i], f);
    const int word = e * N >> 5, bit = e * N & 31;  // a vector's bits lie in one word
    if ((s_mark[word] >> bit) & ((1u << N) - 1u)) {
      if (counts) {
        uint32_t c[N];
#pragma unroll
        for (int j = 0; j < N; j += 4) *reinterpret_cast<uint4*>(c + j) = *reinterpret_cast<const uint4*>(cnt + slot + j);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = r.apply(f[j], c[j]);
      }
      if (biases) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
          const float4 b = *reinterpret_cast<const float4*>(bsum + slot + j);
          f[j] = __fadd_rn(f[j], b.x), f[j + 1] = __fadd_rn(f[j + 1], b.y);
          f[j + 2] = __fadd_rn(f[j + 2], b.z), f[j + 3] = __fadd_rn(f[j + 3], b.w);
        }
      }
    }
    if (mask) {
      const uint32_t bits = s_mask[word] >> bit;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!((bits >> j) & 1u)) f[j] = -INFINITY;
    }
    const uint4 o = V::from_float(f);
    if (vec_store) {
      *reinterpret_cast<uint4*>(out + v) = o;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) out[v + j] = from_f<T>(f[j]);
    }
    if (p.keys) {
      V::to_float(o, f);
#pragma unroll
      for (int j = 0; j < N; ++j) best = max(best, greedy_key(f[j], (uint32_t)(g + j)));
    }
  }
  for (int v = lo + tid; v < v0; v += kThreads) single(v);
  for (int v = v0 + nv * N + tid; v < v1; v += kThreads) single(v);
  if (!p.keys) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) s_key[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 32; ++w) best = max(best, s_key[w]);
    atomicMax(p.keys + row, best);
  }
}

template <typename T>
cudaError_t launch(const LogitsParams& p, cudaStream_t s) {
  const int counts = p.tokens != nullptr && p.history > 0 && (p.repetition || p.frequency || p.presence);
  const int biases = p.bias != nullptr && p.biases > 0;
  constexpr int N = Vec<T>::N, kChunk = 4096;
  int chunk = kChunk;
  while (chunk > 1024 && (long long)p.rows * ((p.vocab + chunk - 1) / chunk) < 148 * 2) chunk /= 2;
  const size_t smem = (size_t)(counts + biases) * (chunk + 2 * N) * 4;
  // the leading ids (fewer than a vector) shift the chunks by less than one vector
  const dim3 grid(p.rows, (p.vocab + chunk - 1) / chunk);
  return launch_k(k_penalize<T, kChunk / N / kThreads>, grid, dim3(kThreads), smem, s, p, chunk, counts, biases);
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
