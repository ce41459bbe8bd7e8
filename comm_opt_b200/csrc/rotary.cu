// Rotary positions, alone or after an RMSNorm of every head, for training rows and for rows that enter the
// paged KV cache.
//
//   n = x * rstd * w,  rstd = 1 / sqrt(mean(x^2) + eps)        (only with norm weights)
//   y[a] = n[a] cos - n[b] sin,  y[b] = n[b] cos + n[a] sin     for the pairs (a, b) of the first `rot` components
//
// and backward, with g = the gradient rotated back and h = x * rstd:
//   dw = sum over rows and heads of g h,   dx = rstd * (w g - h mean(w g h)).
//
// All of it is meant to be bound by the bytes of the heads: each is read once and written once. A head is held by a
// group of 2^k lanes; a lane owns "slots", each of two vectors of V components chosen so that every pair of the rotation
// lies inside one lane: half layout, slot s < rot / 2 / V holds vectors s and s + rot / 2 / V; all other slots,
// and the interleaved layout, hold vectors 2s and 2s + 1. No shuffles but the norm's sums. V is the widest vector that
// every operand's address and strides, the weights and the layout allow (16 bytes for contiguous heads of 64, 128, 256).
// Statistics, products and sums are fp32, two components an instruction; the norm's weights are folded into the angles'
// coefficients once per row; every output is rounded once, at its store.
//
// Measured on one B200: 32763 rows of 64 fp16 heads, half of each rotated (1.08 GB): 169 us, 6.4 TB/s, the rate of a copy.
// With the norm neither memory nor the issue slots are full (backward: 50 and 38 %; prompts into the cache: 30 and 42 %): 12 to
// 16 warps an SM have too few bytes on their way. 8 x 2048 rows of 32 + 8 bf16 heads, forward and backward with the weights'
// gradients (841 MB): 194 us, 4.3 TB/s; padded prompts of 4 x 2048 rows into the cache: 47 us. 8 rows of one decode step: 1.8 us
// (rotation), 2.6 us (norm, rotation, append): a launch. Narrow vectors are far from the bytes' rate, since their lanes are
// given slots by the vector's width alone and most of them repeat the last: half layout, bf16 heads of 96 with 24 rotated 1.1
// TB/s (interleaved, whose vectors stay wide, 5.2), fp32 heads of 80 with 20 rotated 0.8, heads of 64 off a 4-byte boundary 0.2.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "packed.cuh"
#include "serve_ops.h"

namespace cob {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kPage = 16;  // tokens per cache page
// heads that a lane takes per step where there are many rows (measured: 3 without the norm's registers, 166.7 us for the
// long prompt against 177 with 2; 2 with them, 47.0 us for the padded prompts against 50.7 with 3)
constexpr int kSteps = 3, kStepsNorm = 2;

// two 16-bit components of a word
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));  // bf16: the upper half of an fp32
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

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
    } else if constexpr (V == 1) {
      const uint16_t h = (uint16_t)w[0];
      f[0] = to_f(*reinterpret_cast<const T*>(&h));
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const float2 t = unpack2<T>(w[i]);
        f[2 * i] = t.x, f[2 * i + 1] = t.y;
      }
    }
  }
  __device__ __forceinline__ void from_float(const float* f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(f[i]);
    } else if constexpr (V == 1) {
      const T t = from_f<T>(f[0]);
      w[0] = *reinterpret_cast<const uint16_t*>(&t);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
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

// what a lane needs of one of its slots
template <int V>
struct Slot {
  int a, b;  // first component of each vector
  int j;     // first rotation pair (index into the tables)
  bool on;   // the slot exists
};
template <int V, bool INTER>
__device__ __forceinline__ Slot<V> slot_of(int s, int nslots, int half) {
  Slot<V> r;
  r.on = s < nslots;
  r.j = s * V;
  if (!INTER && r.j < half) {
    r.a = r.j;
    r.b = r.j + half;
  } else {
    r.a = 2 * r.j;
    r.b = r.a + V;
  }
  return r;
}

// V weights (fp32 or T) from component `off`, a multiple of V (the launcher's vectors fit the weights' alignment too)
template <typename T, int V>
__device__ __forceinline__ void load_weights(const void* w, int f32, int off, float* o) {
  if (f32) {
    constexpr int N = V < 4 ? V : 4;
#pragma unroll
    for (int i = 0; i < V; i += N) {
      Pack<float, N> r;
      r.load(reinterpret_cast<const float*>(w) + off + i);
      r.to_float(o + i);
    }
  } else {
    Pack<T, V> r;
    r.load(reinterpret_cast<const T*>(w) + off);
    r.to_float(o);
  }
}

// A slot's 2 V components in fp32 as V register pairs: pair k holds components 2k, 2k + 1 of (first vector, second
// vector). `within`: the two components of a pair turn with each other (interleaved layout, and V = 1); otherwise pair k
// of the first vector turns with pair k of the second.
template <typename T, int V>
__device__ __forceinline__ void to_pairs(const Pack<T, V>& lo, const Pack<T, V>& hi, uint64_t* x) {
  float f[2 * V];
  lo.to_float(f);
  hi.to_float(f + V);
#pragma unroll
  for (int k = 0; k < V; ++k) x[k] = pair(f[2 * k], f[2 * k + 1]);
}
template <typename T, int V>
__device__ __forceinline__ void store_zeros(T* lo, T* hi) {
  Pack<T, V> o;
#pragma unroll
  for (int i = 0; i < Pack<T, V>::kWords; ++i) o.w[i] = 0;
  o.store(lo);
  o.store(hi);
}
template <typename T, int V>
__device__ __forceinline__ void store_pairs(const uint64_t* x, T* lo, T* hi) {
  float f[2 * V];
#pragma unroll
  for (int k = 0; k < V; ++k) unpair(x[k], f[2 * k], f[2 * k + 1]);
  Pack<T, V> o;
  o.from_float(f);
  o.store(lo);
  o.from_float(f + V);
  o.store(hi);
}

// What turns a slot by one position's angles: pair k becomes x c + mate(x) s, with the rotation's signs in s and, where
// weights are given, each coefficient times the weight of the component that it multiplies. Pairs past the rotary part get
// c = 1 (or the weight) and are only multiplied.
template <int V, bool INTER>
struct Turn {
  static constexpr bool kWithin = INTER || V == 1;
  uint64_t c[V], s[V];
  __device__ __forceinline__ void load(const float* ct, const float* st, size_t row, int j, int half, float sign,
                                       const float* w) {
    float cv[V], sv[V];
    ct += row * half + j;
    st += row * half + j;
    if (V % 4 == 0 && half % 4 == 0 && j + V <= half) {
#pragma unroll
      for (int i = 0; i + 3 < V; i += 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(ct + i)), b = __ldg(reinterpret_cast<const float4*>(st + i));
        cv[i] = a.x, cv[i + 1] = a.y, cv[i + 2] = a.z, cv[i + 3] = a.w;
        sv[i] = b.x, sv[i + 1] = b.y, sv[i + 2] = b.z, sv[i + 3] = b.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool turns = j + i < half;
        cv[i] = turns ? __ldg(ct + i) : 1.f;
        sv[i] = turns ? __ldg(st + i) : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float a[2], b[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = 2 * k + h, m = kWithin ? e ^ 1 : (e < V ? e + V : e - V);  // component and its mate
        const int at = kWithin ? k : e % V;                                     // their angle
        const bool second = kWithin ? h == 1 : e >= V;
        a[h] = w ? cv[at] * w[e] : cv[at];
        b[h] = second ? sv[at] * sign : sv[at] * -sign;
        if (w) b[h] *= w[m];
      }
      c[k] = pair(a[0], a[1]);
      s[k] = pair(b[0], b[1]);
    }
  }
  // the roundings are those of fma(x, c, mate * s) in every variant; what does not rotate is not x c + mate 0, which an
  // infinity in the mate would turn into NaN
  __device__ __forceinline__ void apply(uint64_t* x, int j, int half, bool weighted) const {
    if (INTER ? j + V <= half : j < half) {
      uint64_t y[V];
#pragma unroll
      for (int k = 0; k < V; ++k) y[k] = mul2(mate(x, k), s[k]);
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] = fma2(x[k], c[k], y[k]);
    } else if (INTER && j < half) {  // the rotary part ends inside the slot
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] = j + k < half ? fma2(x[k], c[k], mul2(mate(x, k), s[k])) : mul2(x[k], c[k]);
    } else if (weighted) {
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] = mul2(x[k], c[k]);
    }
  }
  static __device__ __forceinline__ uint64_t mate(const uint64_t* x, int k) {
    if constexpr (kWithin) {
      float a, b;
      unpair(x[k], a, b);
      return pair(b, a);
    } else {
      return x[k < V / 2 ? k + V / 2 : k - V / 2];
    }
  }
};

__device__ __forceinline__ float group_sum(float v, int gl) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < gl) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// a parameter array's element by value (indexed parameters would be read from constant memory at every use)
template <typename A>
__device__ __forceinline__ A pick(const A (&a)[3], int i) {
  return i == 0 ? a[0] : i == 1 ? a[1] : a[2];
}
template <typename A>
__device__ __forceinline__ A pick(const A (&a)[2], int i) {
  return i == 0 ? a[0] : a[1];
}

// What a kernel is compiled for: kAnything decides at run time (the narrow-vector forms)
enum Mode : int { kPlain = 0, kNorm = 1, kAppend = 2, kAppendNorm = 3, kAnything = 4 };

struct RotaryArgs {
  RotaryParams p;
  int gl, gl_shift;  // lanes per head
  int hb;            // heads per step of a warp
  int blocks[3];     // head blocks (steps) of q, k, v per row
  int groups[3];     // warps that share them: `inner` steps each
  int inner;
  int wh_shift;      // log2 of the warps of a block side by side on one row's groups (they share its angles in L1)
  uint32_t seq_inv;  // ceil(2^32 / seq): row / seq = high word of row * seq_inv; 0: divide
};
__device__ __forceinline__ int batch_of(int row, int seq, uint32_t inv) {
  return inv ? (int)__umulhi((uint32_t)row, inv) : row / seq;
}

// One warp takes `inner` steps of one row's q, k or v heads, the angles and weights loaded and combined once for them. A
// step is 32 / gl heads side by side, HPT after one another; the next step's loads are in flight while one is computed.
template <typename T, int V, int NSL, int HPT, int MODE, bool INTER>
__global__ void __launch_bounds__(kThreads, HPT > 1 ? 4 : NSL == 1 ? 6 : 1)
    k_rotary(const __grid_constant__ RotaryArgs args) {
  const RotaryParams& p = args.p;
  pdl_wait_then_trigger();
  const int warp = threadIdx.x >> 5;
  const int row = (int)blockIdx.x * (kWarps >> args.wh_shift) + (warp >> args.wh_shift);
  int group = ((int)blockIdx.y << args.wh_shift) + (warp & ((1 << args.wh_shift) - 1)), kind = 0;
  if (row >= p.batch * p.seq || group >= args.groups[0] + args.groups[1] + args.groups[2]) return;
  while (kind < 2 && group >= args.groups[kind]) group -= args.groups[kind++];
  const bool append = MODE == kAnything ? p.append != 0 : MODE >= kAppend;
  const bool norm = kind < 2 && (MODE == kAnything ? p.w[0] != nullptr : (MODE & kNorm) != 0);
  const bool has_bias = (MODE == kAnything || MODE >= kAppend) && p.bias != nullptr;
  const int b = batch_of(row, p.seq, args.seq_inv), s = row - b * p.seq;
  const int lane = threadIdx.x & 31, gl = args.gl, l = lane & (gl - 1), sub = lane >> args.gl_shift, per = 32 >> args.gl_shift;
  const int half = p.rot / 2, nslots = p.D / (2 * V);
  const int pos = p.pos[b * p.pos_sb + s * p.pos_ss];
  const bool in_table = pos >= 0 && pos < p.max_pos;
  const int start = append && kind > 0 ? p.starts[b] : 0;
  if (append && (!in_table || (p.lens && s >= p.lens[b]))) return;
  const HeadView in = pick(p.in, kind);
  // Lanes without a slot, and heads past the last one in a warp's row of them, work on copies of real ones and only do not
  // store, so the arithmetic has no branches; whole steps past the last head are left out.
  int hblk = group * args.inner;
  const int hend = min(pick(args.blocks, kind), hblk + args.inner);
  Slot<V> sl[NSL];
#pragma unroll
  for (int n = 0; n < NSL; ++n) {
    sl[n] = slot_of<V, INTER>(min(l + n * gl, nslots - 1), nslots, half);
    sl[n].on = l + n * gl < nslots;
  }
  const T* src = reinterpret_cast<const T*>(in.p) + b * in.sb + s * in.ss;
  Pack<T, V> raw[HPT][NSL][2];
  auto fetch = [&](int hblk, Pack<T, V>(&r)[HPT][NSL][2]) {
#pragma unroll
    for (int h = 0; h < HPT; ++h)
      if (HPT == 1 || hblk * args.hb + h * per < in.heads) {
        const T* at = src + min(hblk * args.hb + h * per + sub, in.heads - 1) * in.sh;
#pragma unroll
        for (int n = 0; n < NSL; ++n) {
          r[h][n][0].load(at + sl[n].a);
          r[h][n][1].load(at + sl[n].b);
        }
      }
  };
  fetch(hblk, raw);
  Turn<V, INTER> turn[NSL];
  if (kind < 2) {
    const void* wp = pick(p.w, kind);
#pragma unroll
    for (int n = 0; n < NSL; ++n) {
      float w[2 * V];
      if (norm) {
        load_weights<T, V>(wp, p.w_f32, sl[n].a, w);
        load_weights<T, V>(wp, p.w_f32, sl[n].b, w + V);
      }
      turn[n].load(p.cos_t, p.sin_t, in_table ? pos : 0, sl[n].j, half, p.inverse ? -1.f : 1.f, norm ? w : nullptr);
    }
  }
  T* dst;
  long long dst_sh;
  if (append && kind > 0) {
    const long long slot = (long long)start + s;
    if (start < 0 || slot >= (long long)p.max_blocks * kPage) return;
    const int blk = p.block_tables[(size_t)b * p.max_blocks + (int)(slot / kPage)];
    if (blk < 0 || blk >= p.num_blocks) return;
    T* cache = reinterpret_cast<T*>(kind == 1 ? p.k_cache : p.v_cache);
    dst = cache + ((long long)blk * in.heads * kPage + slot % kPage) * p.D;
    dst_sh = (long long)kPage * p.D;
  } else {
    const HeadView o = pick(p.out, kind);
    dst = reinterpret_cast<T*>(const_cast<void*>(o.p)) + b * o.sb + s * o.ss;
    dst_sh = o.sh;
  }
  const int bias0 = (kind > 0 ? p.in[0].heads : 0) + (kind > 1 ? p.in[1].heads : 0);  // bias order: q, k, v heads
  const float inv_d = 1.f / (float)p.D;
  Pack<T, V> ahead[HPT][NSL][2];
  for (;;) {
    const bool more = HPT > 1 && hblk + 1 < hend;  // (HPT = 1 is launched with one step a warp)
    if (more) fetch(hblk + 1, ahead);
#pragma unroll
  for (int h = 0; h < HPT; ++h) {
    if (HPT > 1 && hblk * args.hb + h * per >= in.heads) break;
    const int head = hblk * args.hb + h * per + sub;
    T* to = dst + head * dst_sh;
    uint64_t x[NSL][V];
    if (!append && !in_table) {  // a padded row
#pragma unroll
      for (int n = 0; n < NSL; ++n)
        if (head < in.heads && sl[n].on) store_zeros<T, V>(to + sl[n].a, to + sl[n].b);
      continue;
    }
#pragma unroll
    for (int n = 0; n < NSL; ++n) to_pairs(raw[h][n][0], raw[h][n][1], x[n]);
    if (has_bias) {
      const T* bias = reinterpret_cast<const T*>(p.bias) + (size_t)(bias0 + min(head, in.heads - 1)) * p.D;
#pragma unroll
      for (int n = 0; n < NSL; ++n) {
        Pack<T, V> b0, b1;
        b0.load(bias + sl[n].a);
        b1.load(bias + sl[n].b);
        uint64_t bf[V];
        to_pairs(b0, b1, bf);
#pragma unroll
        for (int k = 0; k < V; ++k) x[n][k] = add2(x[n][k], bf[k]);
      }
    }
    uint64_t rstd = 0;
    if (norm) {
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NSL; ++n) {
        uint64_t ss = mul2(x[n][0], x[n][0]);
#pragma unroll
        for (int k = 1; k < V; ++k) ss = fma2(x[n][k], x[n][k], ss);
        sum += sl[n].on ? sum2(ss) : 0.f;
      }
      const float r = rsqrtf(group_sum(sum, gl) * inv_d + p.eps);
      rstd = pair(r, r);
    }
#pragma unroll
    for (int n = 0; n < NSL; ++n) {
      if (kind < 2) turn[n].apply(x[n], sl[n].j, half, norm);
      if (norm) {
#pragma unroll
        for (int k = 0; k < V; ++k) x[n][k] = mul2(x[n][k], rstd);
      }
      if (head < in.heads && sl[n].on) store_pairs<T, V>(x[n], to + sl[n].a, to + sl[n].b);
    }
  }
    if (!more) break;
    ++hblk;
#pragma unroll
    for (int h = 0; h < HPT; ++h)
#pragma unroll
      for (int n = 0; n < NSL; ++n) raw[h][n][0] = ahead[h][n][0], raw[h][n][1] = ahead[h][n][1];
  }
}

// Backward of norm + rotation. The first nb[0] blocks walk the query heads, the others the key heads, each with a
// fixed share of (row, head block) units, so a thread's share of dw stays in its registers and the sums have one
// order: thread, lanes of equal slots, warps, blocks (k_weight_grad).
// what a row costs the backward beside its heads (angles, addresses), in heads: it divides the blocks between q and k.
// Measured at 32 / 8 heads of 128, 16384 rows, forward and backward: 208 us with 2, 195 with 6, 193 with 12
constexpr int kRowCost = 12;
constexpr int kInner = 4;  // steps of a row that a warp of the backward takes, where rows alone fill the GPU
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src)
               : "memory");
}
// until at most n (0 .. 3) of this thread's groups are on their way
__device__ __forceinline__ void cp_async_wait(int n) {
  if (n == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  if (n == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  if (n == 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
}
struct RotaryBwdArgs {
  RotaryParams p;
  int gl, gl_shift, hb, blocks[2], nb[2];
  int inner, groups[2];  // head blocks that a warp takes with one load of the angles; groups of them in a row
  uint32_t seq_inv, groups_inv[2];
  float* ws;  // [nb[0] + nb[1]][D]
};

template <typename T, int V, int NSL, int HPT, bool INTER>
__global__ void __launch_bounds__(kThreads) k_rotary_norm_bwd(const __grid_constant__ RotaryBwdArgs args) {
  const RotaryParams& p = args.p;
  // [kWarps][D] sums at the end, then (wide vectors) what each thread has on its way: [kInner][HPT][4][kThreads] vectors
  extern __shared__ __align__(16) float sdw[];
  constexpr bool ASYNC = Pack<T, V>::kBytes == 16 && NSL == 1;
  uint4* ring = reinterpret_cast<uint4*>(sdw + kWarps * args.p.D) + threadIdx.x;
  pdl_wait_then_trigger();
  const int kind = (int)blockIdx.x < args.nb[0] ? 0 : 1;
  const int blk = kind ? (int)blockIdx.x - args.nb[0] : (int)blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gl = args.gl, l = lane & (gl - 1), sub = lane >> args.gl_shift, per = 32 >> args.gl_shift;
  const int half = p.rot / 2, nslots = p.D / (2 * V), hblocks = args.blocks[kind];
  const HeadView in = pick(p.in, kind), gr = pick(p.grad, kind), o = pick(p.out, kind);
  const void* wp = pick(p.w, kind);
  Slot<V> sl[NSL];
  uint64_t w[NSL][V], dw[NSL][V];
#pragma unroll
  for (int n = 0; n < NSL; ++n) {
    sl[n] = slot_of<V, INTER>(min(l + n * gl, nslots - 1), nslots, half);
    sl[n].on = l + n * gl < nslots;
    float f[2 * V];
    load_weights<T, V>(wp, p.w_f32, sl[n].a, f);
    load_weights<T, V>(wp, p.w_f32, sl[n].b, f + V);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      w[n][k] = pair(f[2 * k], f[2 * k + 1]);
      dw[n][k] = pair(0.f, 0.f);
    }
  }
  const int groups = args.groups[kind], units = p.batch * p.seq * groups;  // (the launcher keeps them below 2^30)
  const float inv_d = 1.f / (float)p.D;
  const long long dstep = per * o.sh;
  for (int u = blk * kWarps + warp; u < units; u += args.nb[kind] * kWarps) {
    const int row = groups == 1 ? u : batch_of(u, groups, args.groups_inv[kind]), group = u - row * groups;
    const int b = batch_of(row, p.seq, args.seq_inv), s = row - b * p.seq;
    const T* xs = reinterpret_cast<const T*>(in.p) + b * in.sb + s * in.ss;
    const T* gs = reinterpret_cast<const T*>(gr.p) + b * gr.sb + s * gr.ss;
    const int hbeg = group * args.inner, hend = min(hblocks, hbeg + args.inner);
    if constexpr (ASYNC) {
      // all of the row's vectors are requested at once, into shared memory: in registers there is room for one step
#pragma unroll
      for (int q = 0; q < kInner; ++q) {
#pragma unroll
        for (int h = 0; h < HPT; ++h)
          if (hbeg + q < hend && (hbeg + q) * args.hb + h * per < in.heads) {
            const int head = min((hbeg + q) * args.hb + h * per + sub, in.heads - 1);
            const T *xa = xs + head * in.sh, *ga = gs + head * gr.sh;
            uint4* to = ring + (q * HPT + h) * 4 * kThreads;
            cp_async16(to, xa + sl[0].a);
            cp_async16(to + kThreads, xa + sl[0].b);
            cp_async16(to + 2 * kThreads, ga + sl[0].a);
            cp_async16(to + 3 * kThreads, ga + sl[0].b);
          }
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
    }
    const int pos = p.pos[b * p.pos_sb + s * p.pos_ss];
    const bool in_table = pos >= 0 && pos < p.max_pos;
    Turn<V, INTER> turn[NSL];
#pragma unroll
    for (int n = 0; n < NSL; ++n)
      turn[n].load(p.cos_t, p.sin_t, in_table ? pos : 0, sl[n].j, half, -1.f, nullptr);
#pragma unroll(ASYNC ? kInner : 1)
    for (int q = 0; q < (ASYNC ? kInner : args.inner); ++q) {
      const int hblk = hbeg + q;
      if (hblk >= hend) break;
      if constexpr (ASYNC) cp_async_wait(kInner - 1 - q);
      const int head0 = hblk * args.hb + sub;  // lanes and heads past the last as in the forward
      T* ds = reinterpret_cast<T*>(const_cast<void*>(o.p)) + b * o.sb + s * o.ss + head0 * o.sh;
      auto has = [&](int h) { return hblk * args.hb + h * per < in.heads; };
      if (!in_table) {  // a padded row: zeros, and no share of dw
#pragma unroll
        for (int h = 0; h < HPT; ++h, ds += dstep)
#pragma unroll
          for (int n = 0; n < NSL; ++n)
            if (head0 + h * per < in.heads && sl[n].on) store_zeros<T, V>(ds + sl[n].a, ds + sl[n].b);
        continue;
      }
      Pack<T, V> rx[HPT][NSL][2], rg[HPT][NSL][2];
#pragma unroll
      for (int h = 0; h < HPT; ++h)
        if (!ASYNC && has(h)) {
          const int head = min(head0 + h * per, in.heads - 1);
          const T *xa = xs + head * in.sh, *ga = gs + head * gr.sh;
#pragma unroll
          for (int n = 0; n < NSL; ++n) {
            rx[h][n][0].load(xa + sl[n].a);
            rx[h][n][1].load(xa + sl[n].b);
            rg[h][n][0].load(ga + sl[n].a);
            rg[h][n][1].load(ga + sl[n].b);
          }
        }
#pragma unroll
      for (int h = 0; h < HPT; ++h, ds += dstep) {
        if (!has(h)) break;
        const bool live = head0 + h * per < in.heads;
        if constexpr (ASYNC) {
          const uint4* from = ring + (q * HPT + h) * 4 * kThreads;
          rx[h][0][0].load(reinterpret_cast<const T*>(from));
          rx[h][0][1].load(reinterpret_cast<const T*>(from + kThreads));
          rg[h][0][0].load(reinterpret_cast<const T*>(from + 2 * kThreads));
          rg[h][0][1].load(reinterpret_cast<const T*>(from + 3 * kThreads));
        }
        uint64_t x[NSL][V], g[NSL][V];
        float sx = 0.f, sxg = 0.f;
#pragma unroll
        for (int n = 0; n < NSL; ++n) {
          to_pairs(rx[h][n][0], rx[h][n][1], x[n]);
          to_pairs(rg[h][n][0], rg[h][n][1], g[n]);
          turn[n].apply(g[n], sl[n].j, half, false);
          uint64_t ss = mul2(x[n][0], x[n][0]), sg = mul2(x[n][0], mul2(g[n][0], w[n][0]));
#pragma unroll
          for (int k = 1; k < V; ++k) {
            ss = fma2(x[n][k], x[n][k], ss);
            sg = fma2(x[n][k], mul2(g[n][k], w[n][k]), sg);
          }
          sx += sl[n].on ? sum2(ss) : 0.f;
          sxg += sl[n].on ? sum2(sg) : 0.f;
        }
        sx = group_sum(sx, gl);
        sxg = group_sum(sxg, gl);
        const float r = rsqrtf(sx * inv_d + p.eps);
        const float m = -(r * sxg * inv_d) * r * r;  // -rstd^2 mean(w g h): dx = rstd w g + m x
        const uint64_t r2 = pair(r, r), m2 = pair(m, m);
        if (live) {
#pragma unroll
          for (int n = 0; n < NSL; ++n) {
            uint64_t d[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
              const uint64_t gr2 = mul2(g[n][k], r2);  // rstd g
              d[k] = fma2(x[n][k], m2, mul2(gr2, w[n][k]));
              dw[n][k] = fma2(gr2, x[n][k], dw[n][k]);
            }
            if (sl[n].on) store_pairs<T, V>(d, ds + sl[n].a, ds + sl[n].b);
          }
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NSL; ++n)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float v[2];
      unpair(dw[n][k], v[0], v[1]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        for (int q = gl; q < 32; q <<= 1) v[h] += __shfl_xor_sync(0xffffffffu, v[h], q);
        const int e = 2 * k + h;
        if (sub == 0 && sl[n].on) sdw[warp * p.D + (e < V ? sl[n].a + e : sl[n].b + e - V)] = v[h];
      }
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
    const size_t wb = p.w_f32 ? std::min(16, 4 * v) : (size_t)esize * v;
    for (const void* w : p.w) ok = ok && reinterpret_cast<uintptr_t>(w) % wb == 0;
    ok = ok && reinterpret_cast<uintptr_t>(p.bias) % ((size_t)esize * v) == 0;
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

int log2_of(int x) {
  int r = 0;
  while ((1 << r) < x) ++r;
  return r;
}
// the high word of row * inverse is row / seq for all rows below `rows` while rows * seq < 2^32; else 0, and the kernels divide
uint32_t inverse_of(long long rows, int seq) {
  return seq > 1 && rows * seq < (1ll << 32) ? (uint32_t)(((1ull << 32) + seq - 1) / seq) : 0u;
}

template <typename T, int V, int NSL, int HPT, int MODE, bool INTER>
cudaError_t launch_fwd(const RotaryParams& p, cudaStream_t s) {
  RotaryArgs a;
  a.p = p;
  a.gl = lanes_of(p.D / (2 * V));
  a.gl_shift = log2_of(a.gl);
  a.hb = 32 / a.gl * HPT;
  const long long rows = (long long)p.batch * p.seq;
  long long hblocks = 0;
  for (int i = 0; i < 3; ++i) hblocks += a.blocks[i] = (p.in[i].heads + a.hb - 1) / a.hb;
  // as many steps in a warp as leave the GPU full
  a.inner = HPT == 1 ? 1 : (int)std::max<long long>(1, std::min<long long>(hblocks, rows * hblocks / (148 * 32)));
  hblocks = 0;
  for (int i = 0; i < 3; ++i) hblocks += a.groups[i] = (a.blocks[i] + a.inner - 1) / a.inner;
  a.wh_shift = hblocks >= 4 ? 2 : hblocks >= 2 ? 1 : 0;
  const int wh = 1 << a.wh_shift;
  a.seq_inv = inverse_of(rows, p.seq);
  const int per = kWarps / wh;
  if (rows >= 0x7fffffffll - kWarps || hblocks > 65535ll * wh) return cudaErrorInvalidValue;
  if (hblocks == 0) return cudaSuccess;
  return launch_k(k_rotary<T, V, NSL, HPT, MODE, INTER>, dim3((unsigned)((rows + per - 1) / per), (unsigned)((hblocks + wh - 1) / wh)),
                  dim3(kThreads), 0, s, a);
}

template <typename T, bool MANY, bool INTER>
cudaError_t wide_fwd(const RotaryParams& p, cudaStream_t s) {
  constexpr int VM = 16 / (int)sizeof(T), A = MANY ? kSteps : 1, N = MANY ? kStepsNorm : 1;
  if (p.append) return p.w[0] ? launch_fwd<T, VM, 1, N, kAppendNorm, INTER>(p, s) : launch_fwd<T, VM, 1, A, kAppend, INTER>(p, s);
  return p.w[0] ? launch_fwd<T, VM, 1, N, kNorm, INTER>(p, s) : launch_fwd<T, VM, 1, A, kPlain, INTER>(p, s);
}

template <typename T>
cudaError_t forward_t(const RotaryParams& p, cudaStream_t s) {
  constexpr int VM = 16 / (int)sizeof(T);
  const int v = vector_of(p, sizeof(T), false);
  if (v == VM && p.D / (2 * VM) <= 32) {
    const long long heads = (long long)p.batch * p.seq * (p.in[0].heads + p.in[1].heads + p.in[2].heads);
    const int per = 32 / lanes_of(p.D / (2 * VM));
    const bool many = heads >= 148ll * 64 * per;
    if (p.interleaved) return many ? wide_fwd<T, true, true>(p, s) : wide_fwd<T, false, true>(p, s);
    return many ? wide_fwd<T, true, false>(p, s) : wide_fwd<T, false, false>(p, s);
  }
  auto narrow = [&](auto inter) {
    constexpr bool I = decltype(inter)::value;
    if (v >= 4) return launch_fwd<T, 4, 2, 1, kAnything, I>(p, s);
    if (v == 2) return launch_fwd<T, 2, 4, 1, kAnything, I>(p, s);
    return launch_fwd<T, 1, 8, 1, kAnything, I>(p, s);
  };
  return p.interleaved ? narrow(std::true_type{}) : narrow(std::false_type{});
}

// blocks of the backward: those that are resident together (three per SM), shared between q and k by what their rows cost
void bwd_blocks(const RotaryParams& p, int nb[2]) {
  const long long rows = (long long)p.batch * p.seq;
  const int total = 148 * 3;
  const int cost[2] = {p.in[0].heads + kRowCost, p.in[1].heads + kRowCost};
  for (int i = 0; i < 2; ++i) {
    const long long share = (long long)total * cost[i] / (cost[0] + cost[1]);
    nb[i] = (int)std::max<long long>(1, std::min<long long>(share, rows * ((p.in[i].heads + 7) / 8)));
  }
}

template <typename T, int V, int NSL, int HPT, bool INTER>
cudaError_t launch_bwd(const RotaryParams& p, float* ws, cudaStream_t s) {
  RotaryBwdArgs a;
  a.p = p;
  a.gl = lanes_of(p.D / (2 * V));
  a.hb = 32 / a.gl * HPT;
  a.ws = ws;
  bwd_blocks(p, a.nb);
  const long long rows = (long long)p.batch * p.seq;
  a.gl_shift = log2_of(a.gl);
  a.seq_inv = inverse_of(rows, p.seq);
  // rows alone fill the GPU: a warp keeps a row's angles for four head blocks, else for one
  a.inner = rows >= 148 * 24 ? kInner : 1;
  for (int i = 0; i < 2; ++i) {
    a.blocks[i] = (p.in[i].heads + a.hb - 1) / a.hb;
    a.groups[i] = (a.blocks[i] + a.inner - 1) / a.inner;
    a.groups_inv[i] = inverse_of(rows * a.groups[i], a.groups[i]);
    if (rows * a.groups[i] >= (1ll << 30)) return cudaErrorInvalidValue;
  }
  auto fn = k_rotary_norm_bwd<T, V, NSL, HPT, INTER>;
  size_t smem = (size_t)kWarps * p.D * sizeof(float);
  if (Pack<T, V>::kBytes == 16 && NSL == 1) {
    smem += (size_t)kInner * HPT * 4 * kThreads * 16;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return launch_k(fn, dim3(a.nb[0] + a.nb[1]), dim3(kThreads), smem, s, a);
}

template <typename T>
cudaError_t backward_t(const RotaryParams& p, float* ws, cudaStream_t s) {
  constexpr int VM = 16 / (int)sizeof(T);
  const int v = vector_of(p, sizeof(T), true);
  auto go = [&](auto inter) {
    constexpr bool I = decltype(inter)::value;
    if (v == VM && p.D / (2 * VM) <= 32) return launch_bwd<T, VM, 1, 2, I>(p, ws, s);
    if (v >= 4) return launch_bwd<T, 4, 2, 1, I>(p, ws, s);
    if (v == 2) return launch_bwd<T, 2, 4, 1, I>(p, ws, s);
    return launch_bwd<T, 1, 8, 1, I>(p, ws, s);
  };
  return p.interleaved ? go(std::true_type{}) : go(std::false_type{});
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
