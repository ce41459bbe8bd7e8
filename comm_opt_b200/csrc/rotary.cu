// Rotary positions, alone or after an RMSNorm of every head, for training rows and for rows that enter the
// paged KV cache.
//
//   n = x * rstd * w,  rstd = 1 / sqrt(mean(x^2) + eps)        (only with norm weights)
//   y[a] = n[a] cos - n[b] sin,  y[b] = n[b] cos + n[a] sin     for the pairs (a, b) of the first `rot` components
//
// and backward, with g = the gradient rotated back and h = x * rstd:
//   dw = sum over rows and heads of g h,   dx = rstd * (w g - h mean(w g h)).
//
// All of it is bound by the bytes of the heads: each is read once and written once. A head is held by a group of
// 2^k lanes; a lane owns "slots", each of two vectors of V components chosen so that every pair of the rotation
// lies inside one lane: half layout, slot s < rot / 2 / V holds vectors s and s + rot / 2 / V; all other slots,
// and the interleaved layout, hold vectors 2s and 2s + 1. No shuffles but the norm's sum. Statistics, products
// and sums are fp32; every output is rounded once, at its store.
#include <algorithm>

#include "common.cuh"
#include "serve_ops.h"

namespace cob {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kPage = 16;  // tokens per cache page

// V components of T as one load
template <typename T, int V>
struct Pack {
  static constexpr int kBytes = V * (int)sizeof(T);
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void to_float(float* f) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        f[i] = to_f(*reinterpret_cast<const T*>(&h));
      }
    }
  }
  __device__ __forceinline__ void from_float(const float* f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const T lo = from_f<T>(f[2 * i]);
        w[i] = *reinterpret_cast<const uint16_t*>(&lo);
        if constexpr (V > 1) {
          const T hi = from_f<T>(f[2 * i + 1]);
          w[i] |= (uint32_t) * reinterpret_cast<const uint16_t*>(&hi) << 16;
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes == 16)
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (kBytes == 8)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (kBytes == 4)
      *reinterpret_cast<uint32_t*>(p) = w[0];
    else
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
  }
};

// what a lane needs of its slots: component offsets of the two vectors, and which pairs rotate
template <int V>
struct Slot {
  int a, b;     // first component of each vector
  int j;        // first pair index (into the tables)
  bool on;      // slot exists
};
template <int V>
__device__ __forceinline__ Slot<V> slot_of(int s, int nslots, int rot, int interleaved) {
  Slot<V> r;
  r.on = s < nslots;
  r.j = s * V;
  const int half = rot / 2;
  if (!interleaved && r.j < half) {
    r.a = r.j;
    r.b = r.j + half;
  } else {
    r.a = 2 * r.j;
    r.b = r.a + V;
  }
  return r;
}

// cos / sin of the lane's pairs at one table row; pairs past rot / 2 do not rotate
template <int V>
__device__ __forceinline__ void load_angles(const float* ct, const float* st, size_t row, int j, int half, bool on,
                                            float* c, float* sn) {
  if (on && V % 4 == 0 && half % 4 == 0 && j + V <= half) {
#pragma unroll
    for (int i = 0; i + 3 < V; i += 4) {
      const float4 cv = __ldg(reinterpret_cast<const float4*>(ct + row * half + j + i));
      const float4 sv = __ldg(reinterpret_cast<const float4*>(st + row * half + j + i));
      c[i] = cv.x, c[i + 1] = cv.y, c[i + 2] = cv.z, c[i + 3] = cv.w;
      sn[i] = sv.x, sn[i + 1] = sv.y, sn[i + 2] = sv.z, sn[i + 3] = sv.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const bool r = on && j + i < half;
    c[i] = r ? __ldg(ct + row * half + j + i) : 1.f;
    sn[i] = r ? __ldg(st + row * half + j + i) : 0.f;
  }
}

// (a, b) turned by the angle of (c, s); the roundings are spelled out, so that every variant gives the same bits
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = a, y = b;
  a = __fmaf_rn(x, c, -__fmul_rn(y, s));
  b = __fmaf_rn(y, c, __fmul_rn(x, s));
}

// rotate a slot's 2 V components in place; components past `half` pairs pass through untouched (not as x * 1 -
// y * 0, which an infinity next to them would turn into NaN)
template <int V>
__device__ __forceinline__ void rotate(float* x, const float* c, const float* sn, int j, int half, int interleaved) {
  if (!interleaved) {
    if (j < half) {
#pragma unroll
      for (int i = 0; i < V; ++i) turn(x[i], x[V + i], c[i], sn[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (j + i < half) turn(x[2 * i], x[2 * i + 1], c[i], sn[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void load_weights(const void* w, int f32, int off, float* o) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    o[i] = f32 ? __ldg(reinterpret_cast<const float*>(w) + off + i) : to_f(__ldg(reinterpret_cast<const T*>(w) + off + i));
}

__device__ __forceinline__ float group_sum(float v, int gl) {
  for (int o = gl >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct RotaryArgs {
  RotaryParams p;
  int gl;          // lanes per head
  int hb;          // heads per warp and step
  int blocks[3];   // head blocks of q, k, v per row
};

// One warp takes `hb` heads of one row: 32 / gl heads side by side, HPT after one another with all their loads
// in flight; cos, sin and the weights are loaded once for them.
template <typename T, int V, int NSL, int HPT>
__global__ void __launch_bounds__(kThreads) k_rotary(const __grid_constant__ RotaryArgs args) {
  const RotaryParams& p = args.p;
  pdl_wait_then_trigger();
  const int hblocks = args.blocks[0] + args.blocks[1] + args.blocks[2];
  const long long unit = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const long long row = unit / hblocks;
  if (row >= (long long)p.batch * p.seq) return;
  int hblk = (int)(unit - row * hblocks), kind = 0;
  while (kind < 2 && hblk >= args.blocks[kind]) hblk -= args.blocks[kind++];
  const int b = (int)(row / p.seq), s = (int)(row - (long long)b * p.seq);
  const int lane = threadIdx.x & 31, gl = args.gl, l = lane & (gl - 1), sub = lane / gl, per = 32 / gl;
  const int half = p.rot / 2, nslots = p.D / (2 * V);
  const int pos = p.pos[b * p.pos_sb + s * p.pos_ss];
  const bool in_table = pos >= 0 && pos < p.max_pos;
  long long cache_row = -1;  // append: (block * nkv) * page + slot within it, in rows of the head's page
  int page_off = 0;
  if (p.append) {
    if (!in_table || (p.lens && s >= p.lens[b])) return;
    if (kind > 0) {
      const int start = p.starts[b];
      const long long slot = (long long)start + s;
      if (start < 0 || slot >= (long long)p.max_blocks * kPage) return;
      const int blk = p.block_tables[(size_t)b * p.max_blocks + (int)(slot / kPage)];
      if (blk < 0 || blk >= p.num_blocks) return;
      page_off = (int)(slot % kPage);
      cache_row = (long long)blk * p.in[kind].heads;
    }
  }
  const HeadView& in = p.in[kind];
  const T* src = reinterpret_cast<const T*>(in.p) + b * in.sb + s * in.ss;
  Slot<V> sl[NSL];
  Pack<T, V> raw[HPT][NSL][2];
#pragma unroll
  for (int n = 0; n < NSL; ++n) sl[n] = slot_of<V>(l + n * gl, nslots, p.rot, p.interleaved);
#pragma unroll
  for (int h = 0; h < HPT; ++h) {
    const int head = hblk * args.hb + h * per + sub;
#pragma unroll
    for (int n = 0; n < NSL; ++n)
      if (head < in.heads && sl[n].on) {
        raw[h][n][0].load(src + head * in.sh + sl[n].a);
        raw[h][n][1].load(src + head * in.sh + sl[n].b);
      }
  }
  float c[NSL][V], sn[NSL][V], w[NSL][2 * V];
  const bool norm = kind < 2 && p.w[0] != nullptr;
  if (kind < 2) {
#pragma unroll
    for (int n = 0; n < NSL; ++n) {
      load_angles<V>(p.cos_t, p.sin_t, in_table ? pos : 0, sl[n].j, half, sl[n].on, c[n], sn[n]);
      if (p.inverse) {
#pragma unroll
        for (int i = 0; i < V; ++i) sn[n][i] = -sn[n][i];
      }
      if (norm && sl[n].on) {
        load_weights<T, V>(p.w[kind], p.w_f32, sl[n].a, w[n]);
        load_weights<T, V>(p.w[kind], p.w_f32, sl[n].b, w[n] + V);
      }
    }
  }
  T* dst;
  long long dst_sh;
  if (p.append && kind > 0) {
    T* cache = reinterpret_cast<T*>(kind == 1 ? p.k_cache : p.v_cache);
    dst = cache + (cache_row * kPage + page_off) * p.D;
    dst_sh = (long long)kPage * p.D;
  } else {
    const HeadView& o = p.out[kind];
    dst = reinterpret_cast<T*>(const_cast<void*>(o.p)) + b * o.sb + s * o.ss;
    dst_sh = o.sh;
  }
  const int head0 = (kind > 0 ? p.in[0].heads : 0) + (kind > 1 ? p.in[1].heads : 0);  // bias order: q, k, v
#pragma unroll
  for (int h = 0; h < HPT; ++h) {
    const int head = hblk * args.hb + h * per + sub;
    const bool live = head < in.heads;
    float x[NSL][2 * V], ss = 0.f;
#pragma unroll
    for (int n = 0; n < NSL; ++n) {
      if (live && sl[n].on) {
        raw[h][n][0].to_float(x[n]);
        raw[h][n][1].to_float(x[n] + V);
        if (p.bias) {
          const T* bp = reinterpret_cast<const T*>(p.bias) + (size_t)(head0 + head) * p.D;
          float bf[2 * V];
          load_weights<T, V>(bp, 0, sl[n].a, bf);
          load_weights<T, V>(bp, 0, sl[n].b, bf + V);
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) x[n][i] += bf[i];
        }
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) ss += x[n][i] * x[n][i];
      }
    }
    if (norm) {
      const float rstd = rsqrtf(group_sum(ss, gl) / (float)p.D + p.eps);
#pragma unroll
      for (int n = 0; n < NSL; ++n)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) x[n][i] = x[n][i] * rstd * w[n][i];
    }
#pragma unroll
    for (int n = 0; n < NSL; ++n)
      if (live && sl[n].on) {
        if (kind < 2) rotate<V>(x[n], c[n], sn[n], sl[n].j, half, p.interleaved);
        if (!in_table) {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) x[n][i] = 0.f;
        }
        Pack<T, V> o;
        o.from_float(x[n]);
        o.store(dst + head * dst_sh + sl[n].a);
        o.from_float(x[n] + V);
        o.store(dst + head * dst_sh + sl[n].b);
      }
  }
}

// Backward of norm + rotation. The first nb[0] blocks walk the query heads, the others the key heads, each with a
// fixed share of (row, head block) units, so a thread's share of dw stays in its registers and the sums have one
// order: thread, lanes of equal slots, warps, blocks (k_weight_grad).
struct RotaryBwdArgs {
  RotaryParams p;
  int gl, hb, blocks[2], nb[2];
  float* ws;  // [nb[0] + nb[1]][D]
};

template <typename T, int V, int NSL, int HPT>
__global__ void __launch_bounds__(kThreads) k_rotary_norm_bwd(const __grid_constant__ RotaryBwdArgs args) {
  const RotaryParams& p = args.p;
  extern __shared__ float sdw[];  // [kWarps][D]
  pdl_wait_then_trigger();
  const int kind = (int)blockIdx.x < args.nb[0] ? 0 : 1;
  const int blk = kind ? (int)blockIdx.x - args.nb[0] : (int)blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gl = args.gl, l = lane & (gl - 1), sub = lane / gl, per = 32 / gl;
  const int half = p.rot / 2, nslots = p.D / (2 * V), hblocks = args.blocks[kind];
  const HeadView &in = p.in[kind], &gr = p.grad[kind], &o = p.out[kind];
  Slot<V> sl[NSL];
  float w[NSL][2 * V], dw[NSL][2 * V];
#pragma unroll
  for (int n = 0; n < NSL; ++n) {
    sl[n] = slot_of<V>(l + n * gl, nslots, p.rot, p.interleaved);
    if (sl[n].on) {
      load_weights<T, V>(p.w[kind], p.w_f32, sl[n].a, w[n]);
      load_weights<T, V>(p.w[kind], p.w_f32, sl[n].b, w[n] + V);
    }
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) dw[n][i] = 0.f;
  }
  const long long units = (long long)p.batch * p.seq * hblocks;
  const float inv_d = 1.f / (float)p.D;
  for (long long u = (long long)blk * kWarps + warp; u < units; u += (long long)args.nb[kind] * kWarps) {
    const long long row = u / hblocks;
    const int hblk = (int)(u - row * hblocks);
    const int b = (int)(row / p.seq), s = (int)(row - (long long)b * p.seq);
    const T* xs = reinterpret_cast<const T*>(in.p) + b * in.sb + s * in.ss;
    const T* gs = reinterpret_cast<const T*>(gr.p) + b * gr.sb + s * gr.ss;
    T* ds = reinterpret_cast<T*>(const_cast<void*>(o.p)) + b * o.sb + s * o.ss;
    Pack<T, V> rx[HPT][NSL][2], rg[HPT][NSL][2];
#pragma unroll
    for (int h = 0; h < HPT; ++h) {
      const int head = hblk * args.hb + h * per + sub;
#pragma unroll
      for (int n = 0; n < NSL; ++n)
        if (head < in.heads && sl[n].on) {
          rx[h][n][0].load(xs + head * in.sh + sl[n].a);
          rx[h][n][1].load(xs + head * in.sh + sl[n].b);
          rg[h][n][0].load(gs + head * gr.sh + sl[n].a);
          rg[h][n][1].load(gs + head * gr.sh + sl[n].b);
        }
    }
    const int pos = p.pos[b * p.pos_sb + s * p.pos_ss];
    const bool in_table = pos >= 0 && pos < p.max_pos;
    float c[NSL][V], sn[NSL][V];
#pragma unroll
    for (int n = 0; n < NSL; ++n) {
      load_angles<V>(p.cos_t, p.sin_t, in_table ? pos : 0, sl[n].j, half, sl[n].on, c[n], sn[n]);
#pragma unroll
      for (int i = 0; i < V; ++i) sn[n][i] = -sn[n][i];
    }
#pragma unroll
    for (int h = 0; h < HPT; ++h) {
      const int head = hblk * args.hb + h * per + sub;
      const bool live = head < in.heads;
      float x[NSL][2 * V], g[NSL][2 * V], ss = 0.f, sg = 0.f;
#pragma unroll
      for (int n = 0; n < NSL; ++n)
        if (live && sl[n].on) {
          rx[h][n][0].to_float(x[n]);
          rx[h][n][1].to_float(x[n] + V);
          rg[h][n][0].to_float(g[n]);
          rg[h][n][1].to_float(g[n] + V);
          rotate<V>(g[n], c[n], sn[n], sl[n].j, half, p.interleaved);
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) {
            ss += x[n][i] * x[n][i];
            sg += x[n][i] * g[n][i] * w[n][i];
          }
        }
      ss = group_sum(ss, gl);
      sg = group_sum(sg, gl);
      const float rstd = rsqrtf(ss * inv_d + p.eps);
      const float m = sg * rstd * inv_d;  // mean(w g h)
#pragma unroll
      for (int n = 0; n < NSL; ++n)
        if (live && sl[n].on) {
          float d[2 * V];
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) {
            const float hx = x[n][i] * rstd;
            d[i] = in_table ? rstd * (w[n][i] * g[n][i] - hx * m) : 0.f;
            if (in_table) dw[n][i] += g[n][i] * hx;
          }
          Pack<T, V> ov;
          ov.from_float(d);
          ov.store(ds + head * o.sh + sl[n].a);
          ov.from_float(d + V);
          ov.store(ds + head * o.sh + sl[n].b);
        }
    }
  }
#pragma unroll
  for (int n = 0; n < NSL; ++n)
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) {
      float v = dw[n][i];
      for (int k = gl; k < 32; k <<= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
      if (sub == 0 && sl[n].on) sdw[warp * p.D + (i < V ? sl[n].a + i : sl[n].b + i - V)] = v;
    }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += sdw[k * p.D + d];
    args.ws[(size_t)blockIdx.x * p.D + d] = v;
  }
}

// dw[kind][d] = sum of the blocks' partial rows: block (column group, kind), 32 columns x 32 row lanes
template <typename W>
__global__ void __launch_bounds__(1024) k_weight_grad(const float* __restrict__ ws, int nb0, int nb1, int D, W* dwq,
                                                      W* dwk) {
  __shared__ float sm[32][33];
  pdl_wait_then_trigger();
  const int kind = blockIdx.y, d = blockIdx.x * 32 + threadIdx.x;
  const float* base = ws + (kind ? (size_t)nb0 * D : 0);
  const int nb = kind ? nb1 : nb0;
  float v = 0.f;
  if (d < D)
    for (int r = threadIdx.y; r < nb; r += 32) v += base[(size_t)r * D + d];
  sm[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  const float t = warp_sum(sm[threadIdx.x][threadIdx.y]);  // column threadIdx.y of the group
  const int dc = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && dc < D) (kind ? dwk : dwq)[dc] = from_f<W>(t);
}

// Largest vector (in components) that every operand's address and strides, the head size and the layout allow.
int vector_of(const RotaryParams& p, int esize, bool backward) {
  int v = 16 / esize;
  auto fits = [&](const HeadView& h, int vv) {
    const long long bytes = (long long)vv * esize;
    return h.heads == 0 || (reinterpret_cast<uintptr_t>(h.p) % bytes == 0 && h.sb % vv == 0 && h.ss % vv == 0 && h.sh % vv == 0);
  };
  for (; v > 1; v /= 2) {
    bool ok = p.D % (2 * v) == 0 && (p.interleaved || (p.rot / 2) % v == 0);
    for (int i = 0; i < 3; ++i) ok = ok && fits(p.in[i], v);
    for (int i = 0; i < 2; ++i) {
      if (p.append && i == 1) continue;  // k and v go to the caches, whose rows are D apart (the binding checks 16-byte bases)
      ok = ok && fits(p.out[i], v) && (!backward || fits(p.grad[i], v));
    }
    if (ok) break;
  }
  return v;
}

int lanes_of(int nslots) {
  int gl = 1;
  while (gl < 32 && gl < nslots) gl *= 2;
  return gl;
}

bool valid(const RotaryParams& p) {
  return p.D >= 2 && p.D <= 512 && p.D % 2 == 0 && p.rot >= 2 && p.rot <= p.D && p.rot % 2 == 0 && p.batch > 0 &&
         p.seq > 0 && p.max_pos > 0;
}

template <typename T, int V, int NSL, int HPT>
cudaError_t launch_fwd(const RotaryParams& p, cudaStream_t s) {
  RotaryArgs a;
  a.p = p;
  a.gl = lanes_of(p.D / (2 * V));
  a.hb = 32 / a.gl * HPT;
  long long hblocks = 0;
  for (int i = 0; i < 3; ++i) hblocks += a.blocks[i] = (p.in[i].heads + a.hb - 1) / a.hb;
  const long long units = hblocks * p.batch * p.seq, grid = (units + kWarps - 1) / kWarps;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  if (grid == 0) return cudaSuccess;
  return launch_k(k_rotary<T, V, NSL, HPT>, dim3((unsigned)grid), dim3(kThreads), 0, s, a);
}

template <typename T>
cudaError_t forward_t(const RotaryParams& p, cudaStream_t s) {
  constexpr int VM = 16 / (int)sizeof(T);
  const int v = vector_of(p, sizeof(T), false);
  if (v == VM && p.D / (2 * VM) <= 32) {
    const long long heads = (long long)p.batch * p.seq * (p.in[0].heads + p.in[1].heads + p.in[2].heads);
    const int per = 32 / lanes_of(p.D / (2 * VM));
    return heads >= 148ll * 64 * per ? launch_fwd<T, VM, 1, 4>(p, s) : launch_fwd<T, VM, 1, 1>(p, s);
  }
  if (v >= 4) return launch_fwd<T, 4, 2, 1>(p, s);
  if (v == 2) return launch_fwd<T, 2, 4, 1>(p, s);
  return launch_fwd<T, 1, 8, 1>(p, s);
}

// blocks of the backward: enough to fill the GPU, shared between q and k by their heads
void bwd_blocks(const RotaryParams& p, int nb[2]) {
  const long long rows = (long long)p.batch * p.seq;
  const int total = 148 * 6;
  for (int i = 0; i < 2; ++i) {
    const long long share = (long long)total * p.in[i].heads / (p.in[0].heads + p.in[1].heads);
    nb[i] = (int)std::max<long long>(1, std::min<long long>(share, rows * ((p.in[i].heads + 7) / 8)));
  }
}

template <typename T, int V, int NSL, int HPT>
cudaError_t launch_bwd(const RotaryParams& p, float* ws, cudaStream_t s) {
  RotaryBwdArgs a;
  a.p = p;
  a.gl = lanes_of(p.D / (2 * V));
  a.hb = 32 / a.gl * HPT;
  a.ws = ws;
  bwd_blocks(p, a.nb);
  for (int i = 0; i < 2; ++i) a.blocks[i] = (p.in[i].heads + a.hb - 1) / a.hb;
  return launch_k(k_rotary_norm_bwd<T, V, NSL, HPT>, dim3(a.nb[0] + a.nb[1]), dim3(kThreads),
                  (size_t)kWarps * p.D * sizeof(float), s, a);
}

template <typename T>
cudaError_t backward_t(const RotaryParams& p, float* ws, cudaStream_t s) {
  constexpr int VM = 16 / (int)sizeof(T);
  const int v = vector_of(p, sizeof(T), true);
  if (v == VM && p.D / (2 * VM) <= 32) return launch_bwd<T, VM, 1, 2>(p, ws, s);
  if (v >= 4) return launch_bwd<T, 4, 2, 1>(p, ws, s);
  if (v == 2) return launch_bwd<T, 2, 4, 1>(p, ws, s);
  return launch_bwd<T, 1, 8, 1>(p, ws, s);
}

}  // namespace

cudaError_t rotary_forward(const RotaryParams& p, cudaStream_t s) {
  if (!valid(p)) return cudaErrorInvalidValue;
  switch (p.dtype) {
    case kF32: return forward_t<float>(p, s);
    case kF16: return forward_t<__half>(p, s);
    case kBF16: return forward_t<__nv_bfloat16>(p, s);
    default: return cudaErrorInvalidValue;
  }
}

int rotary_backward_blocks(const RotaryParams& p) {
  int nb[2];
  bwd_blocks(p, nb);
  return nb[0] + nb[1];
}

cudaError_t rotary_norm_backward(const RotaryParams& p, float* ws, void* dwq, void* dwk, cudaStream_t s) {
  if (!valid(p) || !p.w[0] || !p.w[1] || p.in[0].heads <= 0 || p.in[1].heads <= 0) return cudaErrorInvalidValue;
  cudaError_t e;
  switch (p.dtype) {
    case kF32: e = backward_t<float>(p, ws, s); break;
    case kF16: e = backward_t<__half>(p, ws, s); break;
    case kBF16: e = backward_t<__nv_bfloat16>(p, ws, s); break;
    default: return cudaErrorInvalidValue;
  }
  if (e != cudaSuccess) return e;
  int nb[2];
  bwd_blocks(p, nb);
  const dim3 grid((p.D + 31) / 32, 2), block(32, 32);
  if (p.w_f32 || p.dtype == kF32)
    return launch_k(k_weight_grad<float>, grid, block, 0, s, (const float*)ws, nb[0], nb[1], p.D,
                    reinterpret_cast<float*>(dwq), reinterpret_cast<float*>(dwk));
  if (p.dtype == kF16)
    return launch_k(k_weight_grad<__half>, grid, block, 0, s, (const float*)ws, nb[0], nb[1], p.D,
                    reinterpret_cast<__half*>(dwq), reinterpret_cast<__half*>(dwk));
  return launch_k(k_weight_grad<__nv_bfloat16>, grid, block, 0, s, (const float*)ws, nb[0], nb[1], p.D,
                  reinterpret_cast<__nv_bfloat16*>(dwq), reinterpret_cast<__nv_bfloat16*>(dwk));
}

}  // namespace cob
