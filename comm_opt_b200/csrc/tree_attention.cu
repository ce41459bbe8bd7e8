// Attention of a tree of drafted tokens over the paged KV cache, on the tcgen05 tensor cores.
//
// For one (sequence, KV head) the rows are all drafted tokens of all its query heads, r = t * G + g, so every cache
// byte is read once per 256 rows. A CTA owns NT row tiles of 128 rows (NT = 2 above 128 rows) and walks 128-token
// tiles of the cache, 64 tokens a step, with the online softmax
//   S = Q K^T;  m' = max(m, row max);  P = 2^((S - m') c);  l = l 2^((m - m') c) + sum P;  O = O 2^((m - m') c) + P V
// with c = scale log2(e). A row tile's row is one TMEM lane and one thread of a softmax warpgroup, so maxima and
// sums need no shuffles. Roles: one warp loads K tiles, one V tiles (8 pages of 16 tokens as 64-column TMA boxes
// whose 128-byte swizzle makes them tcgen05 operands: K is K-major, V N-major), one issues the MMAs, NT warpgroups do
// the softmax. S is written by the tensor cores into one of a row tile's two TMEM buffers, P goes back over it in 16 bits
// and is the A operand of P V straight from TMEM; O stays in TMEM. Q K^T of the next step runs while the softmax works
// on this one, which is what two buffers of 64 columns per row tile are for (one of 128 left the softmax waiting 1 us a
// tile for its scores; two of 128 fit beside one row tile's O, but not beside two). O is rescaled only where a row's maximum rose by more than 2^8 (bf16; fp16 2^4, see kRise), which
// after the first tiles hardly happens; O / l is the same number.
//
// Work is cut into equal shares of the flattened (sequence, KV head, tile) space by the sequences' actual lengths,
// each (sequence, KV head) charged two tiles for its start and end, so ragged batches and few long sequences both fill
// the GPU; the RB CTAs that hold the row blocks of one share walk it side by side and meet each other's cache tiles in
// L2. A (sequence, head) cut between shares leaves unnormalised partials (at most two per CTA) that a second kernel,
// launched early, joins in the shares' order.
//
// Bounds, measured on one B200 at 4 x 64 drafted tokens over 32k, 64 / 8 heads of 128 (0.55 GB, 275 GFLOP): 280 us, 0.98
// PFLOP/s, over the same inputs again and again, 335 us (0.82) with inputs that change from call to call. Without the softmax
// the same walk takes 222 us, of which Q K^T 97 us: M = 128, N = 64 from shared memory reads
// 6 KB per 32 cycles of arithmetic and the memory gives 128 bytes a cycle, but 128 columns do not fit beside O twice.
// Exponentials on the FMA pipe (a degree-5 polynomial for 2 to 4 of 8), 16 softmax warps of 16 rows each (16x256b TMEM
// accesses) and 128-column steps were all measured and no faster (288 - 303, 306, 305 us against 290 then); the two row
// tiles taking turns at the exponential unit took it from 290 to 276.
// Small: 8 drafted tokens over 1k, 32 / 8 heads: 11.0 us, latencies (lengths, page indices and first pages 3.2, one tile
// 1.5, output 1, the join 3). 8 x 16 over up to 2k, 64 / 8 heads (38 MB): 22 us. One row tile over long caches: 16 drafts over
// 4 x 32k, 64 / 8 heads of 128: 112 us, 4.8 TB/s of cache; 8 x 8k, 32 / 8 heads: 60 us, 4.5 TB/s, and of 64 56 us, 2.4 TB/s
// (the steps take as long with half the bytes, one CTA an SM).
//
// What a row does not see must not reach it, even when it is not finite: scores are replaced, not added to; slots past
// the last token are zeroed in the V tile; a non-finite component of a drafted token's v is zeroed there too, and
// added back at the end to the rows that see it.
#include <algorithm>

#include "common.cuh"
#include "packed.cuh"
#include "serve_ops.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace cob {
namespace {

using namespace sm100;

constexpr int kPage = 16, kTile = 128, kTilePages = kTile / kPage;
constexpr int kMaxBatch = 128;  // sequences of one launch (their lengths and tile counts live in shared memory)
constexpr int kBarBytes = 320;  // barriers and flags of a CTA
constexpr int kPieceCost = 2;   // of starting and ending a piece of a (sequence, KV head), in tiles
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint64_t kDrain = 1000000000ull;  // most that a CTA waits for its own copies and MMAs before it ends, ns
__device__ int g_gave_up;                   // per device: set where a wait ran out (kept until the host clears it)

// ----------------------------------------------------------------------------- TMEM accesses of this kernel
// 32 lanes x 32 columns, asynchronous: the registers are valid after tmem_landed()
__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a)
      : "memory");
}
// waits for this thread's TMEM loads; the registers pass through, so no use of them can move above the wait
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29])
               :
               : "memory");
  asm volatile("" : "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The MMA warp runs its loop as a whole and one elected lane issues: what feeds the instructions is then the same in all
// lanes and stays in uniform registers (behind a branch on the lane, moving it there took 100 cycles per MMA).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e;
}
// Shared-memory matrix descriptors as (low, high) words; a step along the operand adds its bytes / 16 to the low word.
// K-major: 128-byte swizzle, 8-row groups 1024 bytes apart. N-major: 64-column groups `lbo` bytes apart, 8-row groups 1024.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3FFFu) | (lbo >> 4) << 16; }
// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "mov.b64 da, {%1, %6};\n\tmov.b64 db, {%2, %6};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(leader), "n"(kDescHigh)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], 16-bit A packed two components to a column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "mov.b64 db, {%2, %6};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(leader), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
      "r"(leader)
      : "memory");
}
constexpr uint32_t kBNMajor = 1u << 16;  // instruction descriptor: B is N-major
constexpr uint32_t kNegateA = 1u << 13;  // instruction descriptor: A enters with its sign changed

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 16 bytes global -> shared without registers, zeros where `real` is false (nothing is read then)
__device__ __forceinline__ void cp_async16_or_zero(void* dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(real ? 16 : 0) : "memory");
}
// NaN if any is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
constexpr uint32_t kExpMask = 0x7C00u;  // exponent bits of __half: all set in infinities and NaN
template <>
constexpr uint32_t kExpMask<__nv_bfloat16> = 0x7F80u;

// Weights are P = 2^(x + kShift), x relative to a reference maximum that lies at most kRise below the row's (and both cancel in
// O / l). They are rounded to the cache's 16 bits, which is what the tensor cores take beside a 16-bit V: at most half a step
// each, of numbers that the sum l counts in fp32. bf16 has fp32's range. fp16 ends at 2^16 and loses bits below 2^-14, so its
// weights sit as high as they can: they are normal numbers from 2^-25 of the row's largest on (without the shift from 2^-14 on,
// and nothing below 2^-25: 4000 tokens at 2^-26 behind one strong token vanished from O while l counted them). The smaller kRise
// costs a rescaling of O now and then.
template <typename T>
constexpr float kRise = 4.f;
template <typename T>
constexpr float kShift = 11.f;
template <>
constexpr float kRise<__nv_bfloat16> = 8.f;
template <>
constexpr float kShift<__nv_bfloat16> = 0.f;

// zeroes the non-finite halves of a vector; non-zero if there were any
template <typename T>
__device__ __forceinline__ uint32_t drop_odd(uint4& v) {
  uint32_t odd = 0;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if ((w[x] & kExpMask<T>) == kExpMask<T>) w[x] &= 0xFFFF0000u, odd = 1;
    if (((w[x] >> 16) & kExpMask<T>) == kExpMask<T>) w[x] &= 0x0000FFFFu, odd = 1;
  }
  return odd;
}

// 4 x 4 vectors across the lanes of a quad, transposed: v[j] becomes lane j's v[this lane's place in the quad]
__device__ __forceinline__ void quad_transpose(uint4 (&v)[4], int lane) {
  auto swap = [&](uint4& a, uint4& b, int bit) {  // lanes with the bit clear give b and get a's mate, the others the reverse
    const bool up = lane & bit;
    uint4 s = up ? a : b;
    s.x = __shfl_xor_sync(0xffffffffu, s.x, bit);
    s.y = __shfl_xor_sync(0xffffffffu, s.y, bit);
    s.z = __shfl_xor_sync(0xffffffffu, s.z, bit);
    s.w = __shfl_xor_sync(0xffffffffu, s.w, bit);
    if (up)
      a = s;
    else
      b = s;
  };
  swap(v[0], v[1], 1);
  swap(v[2], v[3], 1);
  swap(v[0], v[2], 2);
  swap(v[1], v[3], 2);
}

// Bounded wait of a whole warp, one verdict for all lanes (and reconverged: the TMEM accesses that follow need it). The
// timer and the failure flag are only looked at every 64 tries. Every waiter of a barrier sees every phase of it in turn, so
// the parity is never ambiguous (but for the softmax's waits for V tiles, where it is for another reason, stated there).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* fail, uint64_t limit) {
  uint64_t t0 = 0;
  for (uint32_t tries = 1;; ++tries) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((tries & 63u) == 0) {
      const uint64_t t = globaltimer();
      if (t0 == 0) t0 = t;
      if (__any_sync(0xffffffffu, t - t0 > limit || *fail != 0)) {
        *fail = 1;
        return false;
      }
    }
  }
}

// ----------------------------------------------------------------------------- geometry
template <int D, int NT>
struct Geo {
  static constexpr int ROWS = NT * 128;
  static constexpr int HALVES = D / 64;
  static constexpr int HALF_BYTES = kTile * 128;          // 64 columns of a tile
  static constexpr int TILE_BYTES = kTile * D * 2;        // Q, K or V tile
  static constexpr int KS = 3, VS = NT == 2 ? 2 : 3;      // ring stages (227 KB per CTA at D = 128)
  // 4 softmax warps per row tile, 2 loading, 1 issuing MMAs, 1 idle (with 11 warps the compiler spills)
  static constexpr int WARPS = 4 * NT + 4;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int SMEM = 1024 + NT * TILE_BYTES + (KS + VS) * TILE_BYTES + kBarBytes + (3 * kMaxBatch + 1) * 4;
  static constexpr int STEP = 64;                         // tokens of a score buffer: two per row tile fit beside O
  static constexpr int PER = kTile / STEP;                // steps of a tile
  static constexpr uint32_t O0 = 256;                     // TMEM columns: score buffers [tile][2] of STEP, then O of each tile
};

struct alignas(64) TreeArgs {
  CUtensorMap tk, tv;  // caches as [num_blocks * nkv * 16, D], box 16 x 64, 128-byte swizzle
  TreeAttnParams p;
  int group;           // G = nq / nkv
  uint32_t group_inv;  // ceil(2^32 / G): row / G = high word of row * group_inv (rows * G < 2^32); 0 for G = 1
  int rb;              // row blocks of a (sequence, KV head)
  int shares;          // equal shares of the flattened (sequence, KV head, piece cost + tile) space
  float* part_o;       // [shares * rb][2][D / 4][ROWS][4]
  float* part_ml;      // [shares * rb][2][ROWS][2]: reference maximum and sum
};

struct SeqLen {
  int ctx, tl, len;  // cached tokens, drafted tokens, slots in all
};
__device__ __forceinline__ SeqLen seq_len(const TreeAttnParams& p, int ctx, int tl) {
  SeqLen s;
  const int cap = p.max_blocks * kPage;
  s.tl = min(max(tl, 0), p.tree);
  s.ctx = min(max(ctx, 0), cap);
  s.len = min(s.ctx + s.tl, cap);
  return s;
}
// scores to exponents of 2: a negative scale negates Q K^T in the MMA; a zero scale is a tiny one (masked scores are -inf: not
// times 0)
__device__ __forceinline__ float scale_log2(const TreeAttnParams& p) { return fmaxf(fabsf(p.scale) * kLog2e, 1e-37f); }
__device__ __forceinline__ int token_of(int row, uint32_t inv) { return inv ? (int)__umulhi((uint32_t)row, inv) : row; }
__device__ __forceinline__ int tiles_of(const SeqLen& s) { return s.tl > 0 ? (s.len + kTile - 1) / kTile : 0; }

// The batch's lengths, and the positions of its work: (sequence b, KV head h) covers the positions
// [cum[b] + h * (kPieceCost + tiles), ...), kPieceCost of them for starting it and one for every tile.
struct Lens {
  int *ctx, *tl, *cum;  // [kMaxBatch], [kMaxBatch], [kMaxBatch + 1]
  __device__ __forceinline__ explicit Lens(int* mem) : ctx(mem), tl(mem + kMaxBatch), cum(mem + 2 * kMaxBatch) {}
  __device__ __forceinline__ SeqLen at(const TreeAttnParams& p, int b) const { return seq_len(p, ctx[b], tl[b]); }
  // by the whole block; ends with a barrier
  __device__ __forceinline__ void fill(const TreeAttnParams& p) {
    for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
      ctx[b] = p.ctx_lens[b];
      tl[b] = p.tree_lens ? p.tree_lens[b] : p.tree;
      const int t = tiles_of(at(p, b));
      cum[b + 1] = t ? (t + kPieceCost) * p.nkv : 0;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      int carry = 0;
      if (lane == 0) cum[0] = 0;
      for (int i0 = 0; i0 < p.batch; i0 += 32) {
        int v = i0 + lane < p.batch ? cum[i0 + lane + 1] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += u;
        }
        v += carry;
        if (i0 + lane < p.batch) cum[i0 + lane + 1] = v;
        carry = __shfl_sync(0xffffffffu, v, 31);
      }
    }
    __syncthreads();
  }
};

// One contiguous piece of a share: tiles [t0, t1) of (b, kvh), of nt in all.
struct Segment {
  int b, kvh, t0, t1, nt;
  bool first;  // of the (sequence, KV head) that holds the share's first position (partial slot 0, else 1)
};
// steps of a piece: STEP tokens each, up to the last one that holds a token
template <int STEP>
__device__ __forceinline__ int steps_of(const Segment& s, int len) {
  return (s.t1 - s.t0) * (kTile / STEP) - (s.t1 == s.nt ? (s.nt * kTile - len) / STEP : 0);
}
struct Walk {
  const int* cum;
  int batch, nkv, g, beg, end;
  __device__ __forceinline__ bool next(Segment& s) {
    while (g < end) {
      int lo = 0, hi = batch - 1;  // last b with cum[b] <= g
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cum[mid] <= g)
          lo = mid;
        else
          hi = mid - 1;
      }
      const int cost = (cum[lo + 1] - cum[lo]) / nkv, rem = g - cum[lo];
      s.b = lo;
      s.nt = cost - kPieceCost;
      s.kvh = rem / cost;
      const int at = g - (rem - s.kvh * cost);  // position of the (sequence, KV head)
      s.t0 = max(0, g - at - kPieceCost);
      s.t1 = min(s.nt, end - at - kPieceCost);
      s.first = g == beg;
      g = min(end, at + cost);
      if (s.t0 < s.t1) return true;  // (a share may end inside the starting cost)
    }
    return false;
  }
};
__device__ __forceinline__ int share_beg(int c, int total, int shares) { return (int)((long long)c * total / shares); }
__device__ __forceinline__ int share_of(int g, int total, int shares) {
  return (int)((((long long)g + 1) * shares - 1) / total);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Geo<D, NT>::THREADS, 1) k_tree_attn(const __grid_constant__ TreeArgs args) {
  using C = Geo<D, NT>;
  constexpr bool BF16 = kExpMask<T> == 0x7F80u;
  const TreeAttnParams& p = args.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = base;
  uint8_t* sK = sQ + NT * C::TILE_BYTES;
  uint8_t* sV = sK + C::KS * C::TILE_BYTES;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sV + C::VS * C::TILE_BYTES);
  uint64_t* k_empty = k_full + C::KS;
  uint64_t* v_full = k_empty + C::KS;
  uint64_t* v_empty = v_full + C::VS;
  uint64_t* s_full = v_empty + C::VS;    // [NT][2] scores of a buffer are in TMEM
  uint64_t* p_ready = s_full + 2 * NT;   // [NT][2] and its weights
  uint64_t* o_done = p_ready + 2 * NT;   // [NT] one more P V of a row tile has completed
  uint64_t* q_ready = o_done + NT;       // [NT] query tile staged
  uint64_t* turn = q_ready + NT;         // [NT][4] a warp's turn at the exponential unit
  uint64_t* drain = turn + 4 * NT;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* s_fail = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_odd = reinterpret_cast<int*>(tmem_slot + 2);  // a drafted v of this segment is not finite
  Lens lens(reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(k_full) + kBarBytes));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int WK = 4 * NT, WV = WK + 1, WM = WK + 2;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::KS; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < C::VS; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2 * NT; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_ready[i], 4);
    for (int i = 0; i < NT; ++i) mbar_init(&o_done[i], 1), mbar_init(&q_ready[i], 4);
    for (int i = 0; i < 4 * NT; ++i) mbar_init(&turn[i], 1);
    mbar_init(drain, 1);
    *s_fail = p.timeout_ns == 0;
    *s_odd = 0;
    fence_barrier_init();
    prefetch_tmap(&args.tk);
    prefetch_tmap(&args.tv);
  }
  if (warp == WM) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  // The dependents may start once every CTA has triggered, and may want tensor memory too: no thread triggers before its
  // CTA's allocation is done, or a dependent's CTA could take columns first and wait for this kernel, which waits for them.
  __syncthreads();
  pdl_wait_then_trigger();
  lens.fill(p);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int total = lens.cum[p.batch];
  const int share = (int)blockIdx.x / args.rb, rblk = (int)blockIdx.x - share * args.rb;
  const int shares = min(args.shares, total);  // no share is empty, the CTAs past them are idle
  const int beg = share < shares ? share_beg(share, total, shares) : 0, end = share < shares ? share_beg(share + 1, total, shares) : 0;
  Walk walk{lens.cum, p.batch, p.nkv, beg, beg, end};
  Segment sg;

  if (warp == WK || warp == WV) {
    // ------------------------------------------------ loads: a lane per (page, 64-column half) box
    const bool is_k = warp == WK;
    const CUtensorMap* map = is_k ? &args.tk : &args.tv;
    uint8_t* ring = is_k ? sK : sV;
    uint64_t *full = is_k ? k_full : v_full, *empty = is_k ? k_empty : v_empty;
    const int stages = is_k ? C::KS : C::VS;
    const int page = lane / C::HALVES, half = lane % C::HALVES;
    int st = 0, ph = 0, issued = 0;
    bool okay = p.timeout_ns != 0;
    while (okay && walk.next(sg)) {
      const SeqLen sl = lens.at(p, sg.b);
      const int pages = (sl.len + kPage - 1) / kPage;
      const int* bt = p.block_tables + (size_t)sg.b * p.max_blocks;
      auto entry = [&](int t) {
        const int pg = t * kTilePages + page;
        return page < kTilePages && pg < pages ? __ldg(bt + pg) : -1;
      };
      int blk = entry(sg.t0);
      for (int t = sg.t0; t < sg.t1; ++t) {
        const int nxt = t + 1 < sg.t1 ? entry(t + 1) : -1;
        okay = warp_wait(&empty[st], ph ^ 1, s_fail, p.timeout_ns);
        if (!okay) break;
        const int np = min(kTilePages, pages - t * kTilePages);
        if (lane == 0) mbar_arrive_expect_tx(&full[st], np * C::HALVES * 2048);
        __syncwarp();
        if (page < np) {
          // a page index outside the cache: rows past its end, which the load fills with zeros
          const int row = blk >= 0 && blk < p.num_blocks ? (blk * p.nkv + sg.kvh) * kPage : p.num_blocks * p.nkv * kPage;
          tma_load_2d(ring + st * C::TILE_BYTES + half * C::HALF_BYTES + page * 2048, map, &full[st], 64 * half, row);
        }
        ++issued;
        blk = nxt;
        if (++st == stages) st = 0, ph ^= 1;
      }
    }
    // copies in flight must land before the CTA's memory is given back: those who wait for them may have given up
    for (int i = max(0, issued - stages); i < issued; ++i) mbar_wait(&full[i % stages], (i / stages) & 1, kDrain);
  } else if (warp == WM) {
    // ------------------------------------------------ MMAs: step s of row tile q is S[q][s & 1] = Q K^T, O[q] += P V
    const uint32_t leader = elect_one();
    const uint32_t id_qk = idesc_f16(128, C::STEP, BF16) | (p.scale < 0.f ? kNegateA : 0u);
    constexpr uint32_t id_pv = idesc_f16(128, D, BF16) | kBNMajor;
    const uint32_t q_desc = desc_low(smem_addr(sQ), 16), k_desc = desc_low(smem_addr(sK), 16);
    const uint32_t v_desc = desc_low(smem_addr(sV), C::HALF_BYTES);
    int n0 = 0, i0 = 0, seg = 0;  // steps, KV tiles and segments before this segment
    bool okay = p.timeout_ns != 0;
    while (okay && walk.next(sg)) {
      for (int q = 0; q < NT && okay; ++q) okay = warp_wait(&q_ready[q], seg & 1, s_fail, p.timeout_ns);
      const int steps = steps_of<C::STEP>(sg, lens.at(p, sg.b).len);
      auto qk = [&](int s, int q) {
        const int i = i0 + s / C::PER, st = i % C::KS, n = n0 + s;
        if (q == 0 && s % C::PER == 0) {
          if (!warp_wait(&k_full[st], (i / C::KS) & 1, s_fail, p.timeout_ns)) return false;
          tc_fence_after();
        }
        const uint32_t a = q_desc + q * (C::TILE_BYTES >> 4);
        const uint32_t b = k_desc + (st * C::TILE_BYTES + s % C::PER * (C::STEP * 128) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk / 4 * C::HALF_BYTES + kk % 4 * 32) >> 4;
          mma_ss(tmem + (2 * q + (n & 1)) * C::STEP, a + off, b + off, id_qk, kk > 0, leader);
        }
        commit(&s_full[2 * q + (n & 1)], leader);
        if (q == NT - 1 && (s % C::PER == C::PER - 1 || s + 1 == steps)) commit(&k_empty[st], leader);
        return true;
      };
      for (int s = 0; s < min(steps, 2) && okay; ++s)
        for (int q = 0; q < NT && okay; ++q) okay = qk(s, q);
      for (int s = 0; s < steps && okay; ++s) {
        const int n = n0 + s, i = i0 + s / C::PER, st = i % C::VS;
        const uint32_t b = v_desc + (st * C::TILE_BYTES + s % C::PER * (C::STEP * 128) >> 4);
#pragma unroll
        for (int q = 0; q < NT; ++q) {
          okay = okay && warp_wait(&p_ready[2 * q + (n & 1)], (n >> 1) & 1, s_fail, p.timeout_ns);
          if (q == 0 && s % C::PER == 0) okay = okay && warp_wait(&v_full[st], (i / C::VS) & 1, s_fail, p.timeout_ns);
          if (!okay) break;
          tc_fence_after();
          const uint32_t a = tmem + (2 * q + (n & 1)) * C::STEP;
#pragma unroll
          for (int kk = 0; kk < C::STEP / 16; ++kk)
            mma_ts(tmem + C::O0 + q * D, a + kk * 8, b + kk * (2048 >> 4), id_pv, s > 0 || kk > 0, leader);
          commit(&o_done[q], leader);
          if (q == NT - 1 && (s % C::PER == C::PER - 1 || s + 1 == steps)) commit(&v_empty[st], leader);
          if (s + 2 < steps) okay = qk(s + 2, q);
        }
      }
      n0 += steps;
      i0 += sg.t1 - sg.t0;
      ++seg;
    }
    // MMAs in flight must end before their memory is given back: those who wait for them may have given up
    commit(drain, leader);
    mbar_wait(drain, 0, kDrain);
    __syncwarp();
  } else if (warp < WK) {
    // ------------------------------------------------ softmax and epilogue: warpgroup `tile`, thread = row
    const int tile = warp >> 2, wq = warp & 3;
    const uint32_t lanes = (uint32_t)(wq * 32) << 16;
    const int row0 = rblk * C::ROWS + tile * 128 + wq * 32;  // first row of this warp
    const int r = row0 + lane;
    const int t_row = token_of(r, args.group_inv), g_row = r - t_row * args.group;
    const float c = scale_log2(p);
    uint8_t* myQ = sQ + tile * C::TILE_BYTES;
    // this warp's 32 rows, 128-byte-swizzled K-major, missing rows as zeros: asynchronous, q_staged() ends it
    auto stage_q = [&](const Segment& s) {
      constexpr int CH = D / 8;
      const int tl = lens.at(p, s.b).tl, ch = lane % CH;
      const T* q = reinterpret_cast<const T*>(p.q) + s.b * p.q_sb + (long long)s.kvh * args.group * p.q_sh + ch * 8;
#pragma unroll
      for (int it = 0; it < CH; ++it) {
        const int tr = wq * 32 + (it * 32 + lane) / CH;
        const int row = rblk * C::ROWS + tile * 128 + tr, t = token_of(row, args.group_inv), g = row - t * args.group;
        const T* src = q + t * p.q_st + g * p.q_sh;
        cp_async16_or_zero(myQ + (ch / 8) * C::HALF_BYTES + tr * 128 + (((ch % 8) ^ (tr & 7)) << 4), t < tl ? src : q, t < tl);
      }
    };
    auto q_staged = [&]() {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[tile]);
    };
    // The two row tiles' warps of one scheduler take turns at their exponentials. Left alone they fall into step, share the
    // exponential unit while both need it and leave it idle while neither does.
    auto my_turn = [&](int n) {
      return NT == 1 || (tile == 0 && n == 0) || warp_wait(&turn[tile * 4 + wq], (tile ? n : n - 1) & 1, s_fail, p.timeout_ns);
    };
    int n0 = 0, i0 = 0;
    bool okay = p.timeout_ns != 0, have = walk.next(sg);
    if (have) {
      stage_q(sg);
      q_staged();
    }
    while (have && okay) {
      const Segment cur = sg;
      const SeqLen sl = lens.at(p, cur.b);
      const bool live = t_row < sl.tl;
      const bool warp_live = token_of(row0, args.group_inv) < sl.tl;
      unsigned long long bits = 0ull;
      if (live) {
        bits = p.mask ? (unsigned long long)p.mask[cur.b * p.mask_sb + t_row] : (t_row < 63 ? (2ull << t_row) - 1ull : ~0ull);
        const int nodes = sl.len - sl.ctx;  // drafted tokens that have a slot
        if (nodes < 64) bits &= (1ull << nodes) - 1ull;
      }
      float m = -INFINITY, l = 0.f;
      const int steps = steps_of<C::STEP>(cur, sl.len);
      const uint32_t obuf = tmem + lanes + C::O0 + tile * D;
      for (int st = 0; st < steps; ++st) {
        const int n = n0 + st, i = i0 + st / C::PER, s0 = cur.t0 * kTile + st * C::STEP;
        const uint32_t sbuf = tmem + lanes + (2 * tile + (n & 1)) * C::STEP;
        const bool tail = s0 + C::STEP > sl.ctx;
        okay = warp_wait(&s_full[2 * tile + (n & 1)], (n >> 1) & 1, s_fail, p.timeout_ns);
        if (!okay) break;
        tc_fence_after();
        if (st + 1 == steps) {  // every Q K^T of this piece has completed: the next piece's queries may be staged
          have = walk.next(sg);
          if (have) stage_q(sg);
        }
        if (tail && tile == 0) {
          // 128 / STEP threads per slot of the step's V rows: zero them past the last token, and zero non-finite components
          // of drafted tokens
          constexpr int CELLS = C::HALVES * 8 * C::STEP / 128;
          const int vs = i % C::VS, at = threadIdx.x % C::STEP, sr = st % C::PER * C::STEP + at, slot = s0 + at;
          const int part = threadIdx.x / C::STEP;
          // These warps skip the phases of tiles without a tail, but the one before this is over all the same: the scores just
          // seen were issued after the P V of two steps ago (a piece's first two after all of the previous piece's), which had
          // waited for a V tile that is later than the one that held this stage before.
          static_assert(C::VS >= 2 && C::PER <= 2, "the parity of v_full");
          okay = warp_wait(&v_full[vs], (i / C::VS) & 1, s_fail, p.timeout_ns);
          if (!okay) break;
          if (slot >= sl.ctx) {
            uint8_t* vr = sV + vs * C::TILE_BYTES + sr * 128;
            auto cell = [&](int k) {  // this thread's part of the row, in an order free of bank conflicts
              const int e = part * CELLS + k;
              return reinterpret_cast<uint4*>(vr + e / 8 * C::HALF_BYTES + (((e + lane) & 7) << 4));
            };
            if (slot >= sl.len) {
#pragma unroll
              for (int k = 0; k < CELLS; ++k) *cell(k) = make_uint4(0, 0, 0, 0);
            } else {
              uint4 v[CELLS];
              uint32_t odd = 0;
#pragma unroll
              for (int k = 0; k < CELLS; ++k) v[k] = *cell(k);
#pragma unroll
              for (int k = 0; k < CELLS; ++k) odd |= drop_odd<T>(v[k]);
              if (odd) {
#pragma unroll
                for (int k = 0; k < CELLS; ++k) *cell(k) = v[k];
                *s_odd = 1;
              }
            }
          }
          fence_proxy_async();
          __syncwarp();  // (lanes went their own ways; the TMEM accesses are the whole warp's)
        }
        constexpr int G = C::STEP / 32;
        uint32_t w[G / 2][32];
        if (warp_live) {
          uint32_t s[G][32];
#pragma unroll
          for (int k = 0; k < G; ++k) tmem_ld32(sbuf + 32 * k, s[k]);
#pragma unroll
          for (int k = 0; k < G; ++k) tmem_landed(s[k]);
          if (tail) {  // scores of slots that the row does not see
#pragma unroll
            for (int k = 0; k < G; k += 2) {
              const int node = s0 + 32 * k - sl.ctx;  // drafted token of the 64 columns' first
              const unsigned long long see = node >= 64   ? 0ull
                                             : node >= 0  ? bits >> node
                                             : node > -64 ? (bits << -node) | ((1ull << -node) - 1ull)
                                                          : ~0ull;
#pragma unroll
              for (int x = 0; x < 64; ++x)
                if (!((see >> x) & 1ull)) s[k + x / 32][x % 32] = 0xff800000u;
            }
          }
          float mx[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int x = 0; x < 32; x += 4)
#pragma unroll
            for (int k = 0; k < G; ++k) {
              mx[k % 2 * 2] = max3(mx[k % 2 * 2], __uint_as_float(s[k][x]), __uint_as_float(s[k][x + 1]));
              mx[k % 2 * 2 + 1] = max3(mx[k % 2 * 2 + 1], __uint_as_float(s[k][x + 2]), __uint_as_float(s[k][x + 3]));
            }
          float mn = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
          if (mn == INFINITY) mn = __uint_as_float(0x7fc00000u);  // inf - inf
          const bool rise = st == 0 || !((mn - m) * c <= kRise<T>);
          const float f = !rise || mn == m ? 1.f : ex2((m - mn) * c);
          if (rise) m = mn;  // (by row: no row's result depends on another's)
          l *= f;
          if (st > 0 && __any_sync(0xffffffffu, rise)) {  // rescale rows of O, which the previous P V has finished
            okay = warp_wait(&o_done[tile], (n - 1) & 1, s_fail, p.timeout_ns);
            if (!okay) break;
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < D / 32; ++k) {
              uint32_t o[32];
              tmem_ld32(obuf + 32 * k, o);
              tmem_landed(o);
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st32(obuf + 32 * k, o);
            }
          }
          okay = my_turn(n);
          if (!okay) break;
          // x = (s - m) c + kShift, the difference first: s c - m c would round m c, for large scores (2^24 and more) by more than
          // the exponents that are left above P, and give infinities. The subtraction costs 2 % of the wide case; differences for
          // the rows that need them alone, behind a branch, cost 7.
          const float ref = m == -INFINITY ? 0.f : m;
          const uint64_t ref2 = pair(-ref, -ref), c2 = pair(c, c), up2 = pair(kShift<T>, kShift<T>);
          uint64_t sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
          for (int x = 0; x < 16 * G; ++x) {
            float a, b;
            const uint64_t d = add2(pair(__uint_as_float(s[x / 16][x % 16 * 2]), __uint_as_float(s[x / 16][x % 16 * 2 + 1])), ref2);
            unpair(kShift<T> == 0.f ? mul2(d, c2) : fma2(d, c2, up2), a, b);
            a = ex2(a);
            b = ex2(b);
            sum[x & 1] = add2(sum[x & 1], pair(a, b));
            w[x / 32][x % 32] = pack2<T>(a, b);
          }
          l += sum2(add2(sum[0], sum[1]));
        } else {
          okay = my_turn(n);
          if (!okay) break;
        }
        if (NT == 2) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&turn[(tile ^ 1) * 4 + wq]);
          __syncwarp();
        }
        if (st > 0) {  // the previous P V has long ended; seeing its phase keeps this warp's parity in step
          okay = warp_wait(&o_done[tile], (n - 1) & 1, s_fail, p.timeout_ns);
          if (!okay) break;
        }
        if (warp_live) {
#pragma unroll
          for (int k = 0; k < G / 2; ++k) tmem_st32(sbuf + 32 * k, w[k]);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[2 * tile + (n & 1)]);
      }
      if (!okay) break;
      if (have) q_staged();
      const int tiles = cur.t1 - cur.t0;
      okay = warp_wait(&o_done[tile], (n0 + steps - 1) & 1, s_fail, p.timeout_ns);
      if (!okay) break;
      tc_fence_after();
      n0 += steps;
      i0 += tiles;
      const bool whole = tiles == cur.nt;
      const bool odd = *reinterpret_cast<volatile int*>(s_odd) != 0;  // (kept set: a re-check, not a result)
      // partials of a slot: [D / 4][ROWS] vectors of 4 components, and [ROWS] pairs (maximum, sum)
      const size_t slot = (size_t)blockIdx.x * 2 + (cur.first ? 0 : 1);
      const int prow = tile * 128 + wq * 32 + lane;
      uint4* po = reinterpret_cast<uint4*>(args.part_o + slot * C::ROWS * D) + prow;
      T* out = reinterpret_cast<T*>(p.out) + cur.b * p.o_sb + (long long)cur.kvh * args.group * p.o_sh;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (warp_live) {
        const uint32_t obuf = tmem + lanes + C::O0 + tile * D;
#pragma unroll 1
        for (int k = 0; k < D / 32; ++k) {
          uint32_t o[32];
          __syncwarp();  // (rows differ in what they add back and store)
          tmem_ld32(obuf + 32 * k, o);
          tmem_landed(o);
          if (odd && live) {  // non-finite components of drafted tokens that this row sees, from this segment's tiles
            const int lo = max(sl.ctx, cur.t0 * kTile), hi = min(sl.len, cur.t1 * kTile);
            for (int s = lo; s < hi; ++s) {
              const int blk = p.block_tables[(size_t)cur.b * p.max_blocks + s / kPage];
              if (!((bits >> (s - sl.ctx)) & 1ull) || blk < 0 || blk >= p.num_blocks) continue;
              const T* v = reinterpret_cast<const T*>(p.v_cache) +
                           (((size_t)blk * p.nkv + cur.kvh) * kPage + s % kPage) * D + 32 * k;
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                const float f = to_f(v[x]);
                if (!isfinite(f)) o[x] = __float_as_uint(__uint_as_float(o[x]) + f);
              }
            }
          }
          if (whole) {
            // four lanes trade their rows' vectors, so that each stores 16 of 64 contiguous bytes
            uint4 v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              float f[8];
#pragma unroll
              for (int y = 0; y < 8; ++y) f[y] = l == 0.f ? 0.f : __uint_as_float(o[8 * x + y]) * inv;
              v[x] = Vec<T>::from_float(f);
            }
            quad_transpose(v, lane);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int row = row0 + (lane & ~3) + x, t = token_of(row, args.group_inv), g = row - t * args.group;
              if (t < sl.tl) *reinterpret_cast<uint4*>(out + t * p.o_st + g * p.o_sh + 32 * k + (lane & 3) * 8) = v[x];
            }
          } else if (live) {
#pragma unroll
            for (int x = 0; x < 8; ++x)
              po[(size_t)(8 * k + x) * C::ROWS] = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
          }
        }
        if (live && !whole)
          reinterpret_cast<float2*>(args.part_ml)[slot * C::ROWS + prow] = make_float2(m, l);
      }
      tc_fence_before();
    }
    if (!okay) {
      // a wait gave up: what this CTA still owed reads as NaN
      asm volatile("cp.async.wait_all;" ::: "memory");
      const float nan = __uint_as_float(0x7fc00000u);
      Walk again{lens.cum, p.batch, p.nkv, beg, beg, end};
      while (again.next(sg)) {
        if (t_row >= lens.at(p, sg.b).tl) continue;
        if (sg.t1 - sg.t0 == sg.nt) {
          T* out = reinterpret_cast<T*>(p.out) + sg.b * p.o_sb + t_row * p.o_st + (long long)(sg.kvh * args.group + g_row) * p.o_sh;
          for (int d = 0; d < D; ++d) out[d] = from_f<T>(nan);
        } else {
          const size_t slot = ((size_t)blockIdx.x * 2 + (sg.first ? 0 : 1)) * C::ROWS + tile * 128 + wq * 32 + lane;
          reinterpret_cast<float2*>(args.part_ml)[slot] = make_float2(0.f, nan);
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (threadIdx.x == 0 && *s_fail) atomicOr(&g_gave_up, 1);
  if (warp == WM) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the partials of (sequence, head) rows that were cut between shares, in the shares' order:
// M = max m_i, out = sum 2^((m_i - M) c) O_i / sum 2^((m_i - M) c) l_i. A lane holds one row and 16 of its components, so
// that the partials' vectors are read 512 bytes at a time and a row is written by whole sectors.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(128) k_tree_join(const __grid_constant__ TreeArgs args) {
  using C = Geo<D, NT>;
  constexpr int PARTS = D / 16, kBatch = 8;
  const TreeAttnParams& p = args.p;
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = blockIdx.y;
  const int unit = (int)blockIdx.x * 4 + (threadIdx.x >> 5), part = unit % PARTS, r = unit / PARTS * 32 + lane;
  const int t = token_of(r, args.group_inv), g = r - t * args.group;
  const int rblk = r / C::ROWS, rr = r - rblk * C::ROWS;
  // the lengths were complete before the attention started (it waited for its predecessor before it let this kernel
  // start), so the arithmetic on them runs beside the attention
  __shared__ int mem[3 * kMaxBatch + 1];
  Lens lens(mem);
  lens.fill(p);
  const int c0 = lens.cum[b], c1 = lens.cum[b + 1], total = lens.cum[p.batch];
  const bool live = c1 > c0 && t < lens.at(p, b).tl;
  const int cost = (c1 - c0) / p.nkv, nt = cost - kPieceCost, at = c0 + kvh * cost, i0 = at + kPieceCost;
  const int shares = max(1, min(args.shares, total));
  const int s0 = live ? share_of(i0, total, shares) : 0, s1 = live ? share_of(i0 + nt - 1, total, shares) : 0;
  pdl_wait_then_trigger();  // by every thread: what follows this kernel in the stream counts on the attention's end
  if (s0 == s1) return;     // one share held it whole and wrote it
  const int first = share_beg(s0, total, shares) >= at ? 0 : 1;
  auto slot = [&](int s) { return (size_t)(s * args.rb + rblk) * 2 + (s == s0 ? first : 0); };
  const float2* ml = reinterpret_cast<const float2*>(args.part_ml) + rr;
  const float4* po = reinterpret_cast<const float4*>(args.part_o) + (size_t)part * 4 * C::ROWS + rr;
  const float c = scale_log2(p);
  float M = -INFINITY, L = 0.f;
  float4 o[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int q0 = s0; q0 <= s1; q0 += kBatch) {  // kBatch shares' loads in flight together
    float2 e[kBatch];
    float4 v[kBatch][4];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      e[q] = make_float2(-INFINITY, 0.f);
      if (q0 + q <= s1) {
        const size_t k = slot(q0 + q) * C::ROWS;
        e[q] = ml[k];
#pragma unroll
        for (int x = 0; x < 4; ++x) v[q][x] = po[k * (D / 4) + x * C::ROWS];
      }
    }
    float mn = M;
#pragma unroll
    for (int q = 0; q < kBatch; ++q) mn = fmaxf(mn, e[q].x);
    if (mn > M) {
      const float f = exp2f((M - mn) * c);
      M = mn;
      L *= f;
#pragma unroll
      for (int x = 0; x < 4; ++x) o[x].x *= f, o[x].y *= f, o[x].z *= f, o[x].w *= f;
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q)
      if (e[q].x != -INFINITY) {  // (a piece in which the row sees nothing, or no piece)
        const float f = exp2f((e[q].x - M) * c);
        L += f * e[q].y;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          o[x].x += f * v[q][x].x;
          o[x].y += f * v[q][x].y;
          o[x].z += f * v[q][x].z;
          o[x].w += f * v[q][x].w;
        }
      }
  }
  T* out = reinterpret_cast<T*>(p.out) + b * p.o_sb + t * p.o_st + (long long)(kvh * args.group + g) * p.o_sh + part * 16;
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    float f[8] = {o[2 * x].x, o[2 * x].y, o[2 * x].z, o[2 * x].w, o[2 * x + 1].x, o[2 * x + 1].y, o[2 * x + 1].z, o[2 * x + 1].w};
#pragma unroll
    for (int y = 0; y < 8; ++y) f[y] = L == 0.f ? 0.f : f[y] * inv;
    reinterpret_cast<uint4*>(out)[x] = Vec<T>::from_float(f);
  }
}

struct Plan {
  int nt, rb, shares, max_tiles;
};
Plan plan_of(const TreeAttnParams& p) {
  Plan pl;
  const int rows = p.tree * (p.nq / p.nkv);
  pl.nt = rows > 128 ? 2 : 1;
  pl.rb = (rows + pl.nt * 128 - 1) / (pl.nt * 128);
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  pl.max_tiles = (p.max_blocks + kTilePages - 1) / kTilePages;
  const long long most = (long long)std::min(p.batch, kMaxBatch) * p.nkv * (pl.max_tiles + kPieceCost);
  pl.shares = (int)std::max<long long>(1, std::min<long long>(most, sms / pl.rb));
  return pl;
}

size_t part_floats(const TreeAttnParams& p, const Plan& pl) {
  return (size_t)pl.shares * pl.rb * 2 * pl.nt * 128 * (p.head_dim + 2);
}

template <typename T, int D, int NT>
cudaError_t launch(TreeArgs a, const Plan& pl, cudaStream_t s) {
  using C = Geo<D, NT>;
  auto fn = k_tree_attn<T, D, NT>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  e = launch_k(fn, dim3(pl.shares * pl.rb), dim3(C::THREADS), C::SMEM, s, a);
  if (e != cudaSuccess || pl.max_tiles == 1) return e;  // one tile per (sequence, head): nothing is ever cut
  const int units = (a.p.tree * a.group + 31) / 32 * (D / 16);  // warps per (sequence, KV head)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((units + 3) / 4, a.p.nkv, a.p.batch);
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // starts during the attention, waits for its end
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_tree_join<T, D, NT>, a);
}

}  // namespace

cudaError_t tree_attention_error_word(int** word) { return cudaGetSymbolAddress(reinterpret_cast<void**>(word), g_gave_up); }

size_t tree_attention_scratch_bytes(const TreeAttnParams& p) {
  return part_floats(p, plan_of(p)) * sizeof(float);
}

cudaError_t tree_attention(const TreeAttnParams& p, void* scratch, cudaStream_t s) {
  if ((p.head_dim != 64 && p.head_dim != 128) || p.batch <= 0 || p.tree <= 0 || p.tree > 64 || p.nkv <= 0 ||
      p.nq <= 0 || p.nq % p.nkv != 0 || p.nkv > 65535 || p.max_blocks <= 0 || p.num_blocks <= 0 || (p.dtype != kBF16 && p.dtype != kF16))
    return cudaErrorInvalidValue;
  const Plan pl = plan_of(p);
  if (pl.rb > 148 || (long long)std::min(p.batch, kMaxBatch) * p.nkv * (pl.max_tiles + kPieceCost) >= (1ll << 31)) return cudaErrorInvalidValue;
  const bool bf16 = p.dtype == kBF16;
  TreeArgs a;
  a.p = p;
  a.group = p.nq / p.nkv;
  a.group_inv = a.group > 1 ? (uint32_t)(((1ull << 32) + a.group - 1) / a.group) : 0u;
  a.rb = pl.rb;
  a.shares = pl.shares;
  a.part_o = reinterpret_cast<float*>(scratch);
  a.part_ml = a.part_o + (size_t)pl.shares * pl.rb * 2 * pl.nt * 128 * p.head_dim;
  const uint64_t rows = (uint64_t)p.num_blocks * p.nkv * kPage;
  cudaError_t e = tensor_map_2d(p.k_cache, rows, p.head_dim, p.head_dim * 2, kPage, 64, bf16, &a.tk);
  if (e == cudaSuccess) e = tensor_map_2d(p.v_cache, rows, p.head_dim, p.head_dim * 2, kPage, 64, bf16, &a.tv);
  for (int b0 = 0; b0 < p.batch && e == cudaSuccess; b0 += kMaxBatch) {  // the launches share the scratch in stream order
    a.p.batch = std::min(kMaxBatch, p.batch - b0);
    a.p.q = static_cast<const char*>(p.q) + b0 * p.q_sb * 2;
    a.p.out = static_cast<char*>(p.out) + b0 * p.o_sb * 2;
    a.p.block_tables = p.block_tables + (size_t)b0 * p.max_blocks;
    a.p.ctx_lens = p.ctx_lens + b0;
    a.p.tree_lens = p.tree_lens ? p.tree_lens + b0 : nullptr;
    a.p.mask = p.mask ? p.mask + b0 * p.mask_sb : nullptr;
    auto go = [&](auto t) {
      using T = decltype(t);
      if (p.head_dim == 128) return pl.nt == 2 ? launch<T, 128, 2>(a, pl, s) : launch<T, 128, 1>(a, pl, s);
      return pl.nt == 2 ? launch<T, 64, 2>(a, pl, s) : launch<T, 64, 1>(a, pl, s);
    };
    e = bf16 ? go(__nv_bfloat16{}) : go(__half{});
  }
  return e;
}

}  // namespace cob
