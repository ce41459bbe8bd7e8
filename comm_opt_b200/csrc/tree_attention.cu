// Attention of a tree of drafted tokens over the paged KV cache, on the tcgen05 tensor cores.
//
// For one (sequence, KV head) the rows are all drafted tokens of all its query heads, r = t * G + g, so every cache
// byte is read once per 256 rows. A CTA owns NT row tiles of 128 rows (NT = 2 above 128 rows) and walks 128-token
// tiles of the cache with the online softmax
//   S = Q K^T;  m' = max(m, row max);  P = 2^((S - m') c);  l = l 2^((m - m') c) + sum P;  O = O 2^((m - m') c) + P V
// with c = scale log2(e). A row tile's row is one TMEM lane and one thread of a softmax warpgroup, so maxima and
// sums need no shuffles. Roles: one warp loads K tiles, one V tiles (8 pages of 16 tokens as 64-column TMA boxes
// whose 128-byte swizzle makes them tcgen05 operands: K is K-major, V N-major), one issues the MMAs, NT warpgroups do
// the softmax. S is written by the tensor cores into one of two TMEM buffers, P goes back over it in 16 bits and is
// the A operand of P V straight from TMEM; O stays in TMEM. The two buffers belong to the two row tiles (NT = 2) or to
// alternate KV tiles (NT = 1), so the tensor cores work on one while the other is in the softmax.
// O is rescaled only when a row's maximum rose by more than 2^8 (P stays below 2^8, far inside the 16-bit types;
// O / l is the same number), which after the first tiles hardly happens.
//
// Work is cut into equal shares of the flattened (sequence, KV head, tile) space by the sequences' actual lengths, so
// ragged batches and few long sequences both fill the GPU; the RB CTAs that hold the row blocks of one share walk
// it side by side and meet each other's cache tiles in L2. A (sequence, head) cut between shares leaves
// unnormalised partials (at most two per CTA) that a second kernel joins in the shares' order.
//
// What a row does not see must not reach it, even when it is not finite: scores are replaced, not added to; slots past
// the last token are zeroed in the V tile; a non-finite component of a drafted token's v is zeroed there too, and
// added back at the end to the rows that see it.
#include <algorithm>

#include "common.cuh"
#include "serve_ops.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace cob {
namespace {

using namespace sm100;

constexpr int kPage = 16, kTile = 128, kTilePages = kTile / kPage;
constexpr int kMaxBatch = 256;  // sequences of one launch (their tile counts are scanned in shared memory)
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint64_t kTimeout = 1000000000ull;  // of every wait, ns

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

// D[tmem] (+)= A[tmem] * B[smem], 16-bit A packed two components to a column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// N-major operand, 128-byte swizzle: 64-column groups `lbo` bytes apart, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t desc_n_sw128(uint32_t addr, uint32_t lbo) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(lbo >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}
constexpr uint32_t kBNMajor = 1u << 16;  // instruction descriptor: B is N-major

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
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

// Bounded wait of a whole warp, one verdict for all lanes (and reconverged: the TMEM accesses that follow need it).
// Every waiter of a barrier sees every phase of it in turn, so the parity is never ambiguous.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* fail) {
  const bool good = mbar_wait(bar, parity, kTimeout) && *fail == 0;
  if (__all_sync(0xffffffffu, good)) return true;
  *fail = 1;
  return false;
}

// ----------------------------------------------------------------------------- geometry
template <int D, int NT>
struct Geo {
  static constexpr int ROWS = NT * 128;
  static constexpr int HALVES = D / 64;
  static constexpr int HALF_BYTES = kTile * 128;          // 64 columns of a tile
  static constexpr int TILE_BYTES = kTile * D * 2;        // Q, K or V tile
  static constexpr int KS = 3, VS = NT == 2 ? 2 : 3;      // ring stages (227 KB per CTA at D = 128)
  static constexpr int WARPS = 4 * NT + 3;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int SMEM = 1024 + NT * TILE_BYTES + (KS + VS) * TILE_BYTES + 256 + (kMaxBatch + 1) * 4;
  static constexpr uint32_t S0 = 0, S1 = 128, O0 = 256;   // TMEM columns
};

struct alignas(64) TreeArgs {
  CUtensorMap tk, tv;  // caches as [num_blocks * nkv * 16, D], box 16 x 64, 128-byte swizzle
  TreeAttnParams p;
  int group;           // G = nq / nkv
  int rb;              // row blocks of a (sequence, KV head)
  int shares;          // equal shares of the flattened (sequence, KV head, tile) space
  int* cum;            // [batch + 1] scanned tile counts, for the joining kernel
  float* part_o;       // [shares * rb][2][ROWS][D]
  float* part_ml;      // [shares * rb][2][ROWS][2]: maximum (times c) and sum
};

struct SeqLen {
  int ctx, tl, len;  // cached tokens, drafted tokens, slots in all
};
__device__ __forceinline__ SeqLen seq_len(const TreeAttnParams& p, int b) {
  SeqLen s;
  const int cap = p.max_blocks * kPage;
  s.tl = p.tree_lens ? min(max(p.tree_lens[b], 0), p.tree) : p.tree;
  s.ctx = min(max(p.ctx_lens[b], 0), cap);
  s.len = min(s.ctx + s.tl, cap);
  return s;
}
__device__ __forceinline__ int tiles_of(const SeqLen& s) { return s.tl > 0 ? (s.len + kTile - 1) / kTile : 0; }

// One contiguous piece of a share: tiles [t0, t1) of (b, kvh), of nt in all.
struct Segment {
  int b, kvh, t0, t1, nt;
  bool first;  // starts where the share starts (partial slot 0, else 1)
};
struct Walk {
  const int* cum;
  int batch, nkv, g, beg, end;
  __device__ __forceinline__ bool next(Segment& s) {
    if (g >= end) return false;
    int lo = 0, hi = batch - 1;  // last b with cum[b] <= g
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum[mid] <= g)
        lo = mid;
      else
        hi = mid - 1;
    }
    s.b = lo;
    s.nt = (cum[lo + 1] - cum[lo]) / nkv;
    const int rem = g - cum[lo];
    s.kvh = rem / s.nt;
    s.t0 = rem - s.kvh * s.nt;
    s.t1 = min(s.nt, s.t0 + (end - g));
    s.first = g == beg;
    g += s.t1 - s.t0;
    return true;
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
  uint64_t* s_full = v_empty + C::VS;  // [2] scores of a buffer are in TMEM
  uint64_t* p_ready = s_full + 2;      // [2] weights of a buffer are in TMEM
  uint64_t* o_done = p_ready + 2;      // [NT] one more P V of a row tile has completed
  uint64_t* q_ready = o_done + 2;      // [NT] query tile staged
  uint64_t* drain = q_ready + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* s_fail = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_odd = reinterpret_cast<int*>(tmem_slot + 2);  // a drafted v of this segment is not finite
  int* cum = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(k_full) + 256);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int WK = 4 * NT, WV = WK + 1, WM = WK + 2;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::KS; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < C::VS; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&q_ready[i], 4);
    }
    mbar_init(drain, 1);
    *s_fail = 0;
    *s_odd = 0;
    fence_barrier_init();
    prefetch_tmap(&args.tk);
    prefetch_tmap(&args.tv);
  }
  if (warp == WM) tmem_alloc(tmem_slot, 512);
  pdl_wait_then_trigger();
  for (int i = threadIdx.x; i < p.batch; i += C::THREADS) cum[i + 1] = tiles_of(seq_len(p, i)) * p.nkv;
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
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
  tc_fence_after();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= p.batch; i += C::THREADS) args.cum[i] = cum[i];
  const uint32_t tmem = *tmem_slot;
  const int total = cum[p.batch];
  const int share = (int)blockIdx.x / args.rb, rblk = (int)blockIdx.x - share * args.rb;
  const int shares = min(args.shares, total);  // no share is empty, the CTAs past them are idle
  const int beg = share < shares ? share_beg(share, total, shares) : 0, end = share < shares ? share_beg(share + 1, total, shares) : 0;
  Walk walk{cum, p.batch, p.nkv, beg, beg, end};
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
    bool okay = true;
    while (okay && walk.next(sg)) {
      const SeqLen sl = seq_len(p, sg.b);
      const int pages = (sl.len + kPage - 1) / kPage;
      const int* bt = p.block_tables + (size_t)sg.b * p.max_blocks;
      auto entry = [&](int t) {
        const int pg = t * kTilePages + page;
        return page < kTilePages && pg < pages ? __ldg(bt + pg) : -1;
      };
      int blk = entry(sg.t0);
      for (int t = sg.t0; t < sg.t1; ++t) {
        const int nxt = t + 1 < sg.t1 ? entry(t + 1) : -1;
        okay = warp_wait(&empty[st], ph ^ 1, s_fail);
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
    if (!okay)  // copies in flight must land before the CTA's memory is given back
      for (int i = max(0, issued - stages); i < issued; ++i) mbar_wait(&full[i % stages], (i / stages) & 1, kTimeout);
  } else if (warp == WM) {
    // ------------------------------------------------ MMAs: S(n) = Q K^T into buffer n & 1, O += P(n) V
    if (lane == 0) {
      constexpr uint32_t id_qk = idesc_f16(128, kTile, BF16), id_pv = idesc_f16(128, D, BF16) | kBNMajor;
      int n0 = 0, i0 = 0, seg = 0;  // row-tile steps, KV tiles and segments before this segment
      bool okay = true;
      while (okay && walk.next(sg)) {
        for (int q = 0; q < NT && okay; ++q)
          if (!mbar_wait(&q_ready[q], seg & 1, kTimeout) || *s_fail) okay = false;
        if (!okay) break;
        const int steps = (sg.t1 - sg.t0) * NT;
        auto qk = [&](int m) {
          const int i = i0 + m / NT, st = i % C::KS, tile = m % NT;
          if (!mbar_wait(&k_full[st], (i / C::KS) & 1, kTimeout) || *s_fail) return false;
          tc_fence_after();
          const uint32_t a = smem_addr(sQ + tile * C::TILE_BYTES), b = smem_addr(sK + st * C::TILE_BYTES);
          const uint32_t d = tmem + (((n0 + m) & 1) ? C::S1 : C::S0);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk / 4) * C::HALF_BYTES + (kk % 4) * 32;
            mma_f16(d, desc_k_sw128(a + off), desc_k_sw128(b + off), id_qk, kk > 0);
          }
          mma_commit(&s_full[(n0 + m) & 1]);
          if (tile == NT - 1) mma_commit(&k_empty[st]);
          return true;
        };
        okay = qk(0) && (steps < 2 || qk(1));
        for (int m = 0; m < steps && okay; ++m) {
          const int n = n0 + m, i = i0 + m / NT, st = i % C::VS, tile = m % NT;
          if (!mbar_wait(&p_ready[n & 1], (n >> 1) & 1, kTimeout) || !mbar_wait(&v_full[st], (i / C::VS) & 1, kTimeout) ||
              *s_fail) {
            okay = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = tmem + ((n & 1) ? C::S1 : C::S0), b = smem_addr(sV + st * C::TILE_BYTES);
          const uint32_t d = tmem + C::O0 + tile * D;
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk)
            mma_ts(d, a + kk * 8, desc_n_sw128(b + kk * 2048, C::HALF_BYTES), id_pv, m >= NT || kk > 0);
          mma_commit(&o_done[tile]);
          if (tile == NT - 1) mma_commit(&v_empty[st]);
          if (m + 2 < steps) okay = qk(m + 2);
        }
        n0 += steps;
        i0 += sg.t1 - sg.t0;
        ++seg;
      }
      if (!okay) {  // MMAs in flight must end before their memory is given back
        *s_fail = 1;
        mma_commit(drain);
        mbar_wait(drain, 0, kTimeout);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------ softmax and epilogue: warpgroup `tile`, thread = row
    const int tile = warp >> 2, wq = warp & 3;
    const uint32_t lanes = (uint32_t)(wq * 32) << 16;
    const int row0 = rblk * C::ROWS + tile * 128 + wq * 32;  // first row of this warp
    const int r = row0 + lane;
    const int t_row = r / args.group, g_row = r - t_row * args.group;
    // negative scales become a sign of q; a zero scale a tiny one (masked scores are -inf: not times 0)
    const bool neg = p.scale < 0.f;
    const float c = fmaxf(fabsf(p.scale) * kLog2e, 1e-37f);
    uint8_t* myQ = sQ + tile * C::TILE_BYTES;
    auto stage_q = [&](const Segment& s) {  // this warp's 32 rows, 128-byte-swizzled K-major; missing rows are zeros
      constexpr int CH = D / 8;
      const int tl = seq_len(p, s.b).tl;
      const T* q = reinterpret_cast<const T*>(p.q) + s.b * p.q_sb;
#pragma unroll 4
      for (int it = 0; it < CH; ++it) {
        const int idx = it * 32 + lane, rr = idx / CH, ch = idx % CH;
        const int row = row0 + rr, t = row / args.group, g = row - t * args.group;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (t < tl) {
          v = ld_nc_v4(q + t * p.q_st + (long long)(s.kvh * args.group + g) * p.q_sh + ch * 8);
          if (neg) v.x ^= 0x80008000u, v.y ^= 0x80008000u, v.z ^= 0x80008000u, v.w ^= 0x80008000u;
        }
        const int tr = wq * 32 + rr;
        *reinterpret_cast<uint4*>(myQ + (ch / 8) * C::HALF_BYTES + tr * 128 + (((ch % 8) ^ (tr & 7)) << 4)) = v;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[tile]);
    };
    int n0 = 0, i0 = 0;
    bool okay = true, have = walk.next(sg);
    if (have) stage_q(sg);
    while (have && okay) {
      const SeqLen sl = seq_len(p, sg.b);
      const bool live = t_row < sl.tl;
      const bool warp_live = row0 / args.group < sl.tl;
      unsigned long long bits = 0ull;
      if (live) {
        bits = p.mask ? (unsigned long long)p.mask[sg.b * p.mask_sb + t_row] : (t_row < 63 ? (2ull << t_row) - 1ull : ~0ull);
        const int nodes = sl.len - sl.ctx;  // drafted tokens that have a slot
        if (nodes < 64) bits &= (1ull << nodes) - 1ull;
      }
      float m = -INFINITY, l = 0.f;
      for (int t = sg.t0; t < sg.t1; ++t) {
        const int j = t - sg.t0, n = n0 + (NT == 1 ? j : 2 * j + tile), i = i0 + j;
        const uint32_t sbuf = tmem + lanes + ((n & 1) ? C::S1 : C::S0), obuf = tmem + lanes + C::O0 + tile * D;
        const int s0 = t * kTile;
        const bool tail = s0 + kTile > sl.ctx;
        okay = warp_wait(&s_full[n & 1], (n >> 1) & 1, s_fail);
        if (!okay) break;
        tc_fence_after();
        if (tail && tile == 0) {
          // thread = slot of the V tile: zero it past the last token, and zero non-finite components of drafted tokens
          const int st = i % C::VS, slot = s0 + (int)threadIdx.x;
          okay = warp_wait(&v_full[st], (i / C::VS) & 1, s_fail);
          if (!okay) break;
          if (slot >= sl.ctx) {
            uint8_t* vr = sV + st * C::TILE_BYTES + threadIdx.x * 128;
#pragma unroll
            for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                uint4* cell = reinterpret_cast<uint4*>(vr + h * C::HALF_BYTES + (((k + lane) & 7) << 4));
                if (slot >= sl.len) {
                  *cell = make_uint4(0, 0, 0, 0);
                } else {
                  uint4 v = *cell;
                  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
                  bool odd = false;
#pragma unroll
                  for (int x = 0; x < 4; ++x) {
                    if ((w[x] & kExpMask<T>) == kExpMask<T>) w[x] &= 0xFFFF0000u, odd = true;
                    if (((w[x] >> 16) & kExpMask<T>) == kExpMask<T>) w[x] &= 0x0000FFFFu, odd = true;
                  }
                  if (odd) {
                    *cell = v;
                    *s_odd = 1;
                  }
                }
              }
          }
          fence_proxy_async();
        }
        if (warp_live) {
          uint32_t s[4][32];
#pragma unroll
          for (int k = 0; k < 4; ++k) tmem_ld32(sbuf + 32 * k, s[k]);
#pragma unroll
          for (int k = 0; k < 4; ++k) tmem_landed(s[k]);
          if (tail) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int node = s0 + 32 * k - sl.ctx;  // drafted token of the group's first column
              const uint32_t see = node >= 64 ? 0u
                                   : node >= 0 ? (uint32_t)(bits >> node)
                                   : node > -32 ? (uint32_t)(bits << -node) | ((1u << -node) - 1u)
                                                : 0xffffffffu;
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (!((see >> x) & 1u)) s[k][x] = 0xff800000u;
            }
          }
          float mx[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mx[k] = __uint_as_float(s[k][0]);
#pragma unroll
            for (int x = 1; x < 32; ++x) mx[k] = fmaxf(mx[k], __uint_as_float(s[k][x]));
          }
          const float mn = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          if (j == 0) {
            m = mn;
          } else if (__any_sync(0xffffffffu, (mn - m) * c > 8.f)) {
            // rescale this warp's rows of O, which the previous P V has finished
            const float f = mn == m ? 1.f : ex2((m - mn) * c);
            m = mn;
            l *= f;
            okay = warp_wait(&o_done[tile], (i - 1) & 1, s_fail);
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
          const float mu = m == -INFINITY ? 0.f : m * c;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t w[32];
#pragma unroll
            for (int x = 0; x < 32; ++x) {
              const int e = 2 * x;  // column 64 k + e
              const float a = ex2(fmaf(__uint_as_float(s[2 * k + e / 32][e % 32]), c, -mu));
              const float b = ex2(fmaf(__uint_as_float(s[2 * k + e / 32][e % 32 + 1]), c, -mu));
              sum[x & 1] += a;
              sum[2 + (x & 1)] += b;
              w[x] = pack2<T>(a, b);
            }
            tmem_st32(sbuf + 32 * k, w);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_wait_st();
        }
        if (j > 0) {  // the previous P V has long ended; seeing its phase keeps this warp's parity in step
          okay = warp_wait(&o_done[tile], (i - 1) & 1, s_fail);
          if (!okay) break;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[n & 1]);
      }
      if (!okay) break;
      // every Q K^T of this segment has completed: the next segment's queries may be staged
      Segment cur = sg;
      have = walk.next(sg);
      if (have) stage_q(sg);
      const int tiles = cur.t1 - cur.t0, last = i0 + tiles - 1;
      okay = warp_wait(&o_done[tile], last & 1, s_fail);
      if (!okay) break;
      tc_fence_after();
      n0 += NT * tiles;
      i0 += tiles;
      const bool whole = tiles == cur.nt;
      const bool odd = *reinterpret_cast<volatile int*>(s_odd) != 0;  // (kept set: a re-check, not a result)
      const size_t slot = ((size_t)blockIdx.x * 2 + (cur.first ? 0 : 1)) * C::ROWS + tile * 128 + wq * 32 + lane;
      float* po = args.part_o + slot * D;
      T* out = reinterpret_cast<T*>(p.out) + cur.b * p.o_sb + t_row * p.o_st + (long long)(cur.kvh * args.group + g_row) * p.o_sh;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (warp_live) {
        const uint32_t obuf = tmem + lanes + C::O0 + tile * D;
#pragma unroll 1
        for (int k = 0; k < D / 32; ++k) {
          uint32_t o[32];
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
          if (live && whole) {
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
              float f[8];
#pragma unroll
              for (int y = 0; y < 8; ++y) f[y] = l == 0.f ? 0.f : __uint_as_float(o[x + y]) * inv;
              *reinterpret_cast<uint4*>(out + 32 * k + x) = Vec<T>::from_float(f);
            }
          } else if (live) {
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<uint4*>(po + 32 * k + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
          }
        }
        if (live && !whole) {
          args.part_ml[slot * 2] = m == -INFINITY ? -INFINITY : m * c;
          args.part_ml[slot * 2 + 1] = l;
        }
      }
      tc_fence_before();
    }
    if (!okay) {
      // a wait gave up: what this CTA still owed reads as NaN
      const float nan = __uint_as_float(0x7fc00000u);
      Walk again{cum, p.batch, p.nkv, beg, beg, end};
      while (again.next(sg)) {
        if (t_row >= seq_len(p, sg.b).tl) continue;
        if (sg.t1 - sg.t0 == sg.nt) {
          T* out = reinterpret_cast<T*>(p.out) + sg.b * p.o_sb + t_row * p.o_st + (long long)(sg.kvh * args.group + g_row) * p.o_sh;
          for (int d = 0; d < D; ++d) out[d] = from_f<T>(nan);
        } else {
          const size_t slot = ((size_t)blockIdx.x * 2 + (sg.first ? 0 : 1)) * C::ROWS + tile * 128 + wq * 32 + lane;
          args.part_ml[slot * 2] = 0.f;
          args.part_ml[slot * 2 + 1] = nan;
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == WM) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the partials of (sequence, head) rows that were cut between shares, one warp per row, in the shares' order:
// M = max m_i, out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(128) k_tree_join(const __grid_constant__ TreeArgs args) {
  using C = Geo<D, NT>;
  constexpr int E = D / 32;
  const TreeAttnParams& p = args.p;
  pdl_wait_then_trigger();
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= (long long)p.batch * p.tree * p.nq) return;
  const int h = (int)(row % p.nq), t = (int)(row / p.nq % p.tree), b = (int)(row / p.nq / p.tree);
  const int c0 = args.cum[b], c1 = args.cum[b + 1], total = args.cum[p.batch];
  if (c1 == c0) return;
  if (p.tree_lens && t >= p.tree_lens[b]) return;
  const int nt = (c1 - c0) / p.nkv, kvh = h / args.group, r = t * args.group + (h - kvh * args.group);
  const int i0 = c0 + kvh * nt, rblk = r / C::ROWS, rr = r - rblk * C::ROWS;
  const int shares = min(args.shares, total);
  const int s0 = share_of(i0, total, shares), s1 = share_of(i0 + nt - 1, total, shares);
  if (s0 == s1) return;  // one share held it whole and wrote it
  auto slot = [&](int s) {
    const int first = s > s0 || share_beg(s, total, shares) == i0 ? 0 : 1;
    return ((size_t)(s * args.rb + rblk) * 2 + first) * C::ROWS + rr;
  };
  float M = -INFINITY;
  for (int s = s0 + lane; s <= s1; s += 32) M = fmaxf(M, args.part_ml[slot(s) * 2]);
  M = warp_max(M);
  float L = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int s = s0; s <= s1; ++s) {
    const size_t k = slot(s);
    const float2 ml = *reinterpret_cast<const float2*>(args.part_ml + k * 2);
    if (ml.x == -INFINITY) continue;
    const float f = exp2f(ml.x - M);
    L += f * ml.y;
    float v[E];
    if constexpr (E == 4)
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(args.part_o + k * D + lane * E);
    else
      *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(args.part_o + k * D + lane * E);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += f * v[e];
  }
  T* out = reinterpret_cast<T*>(p.out) + b * p.o_sb + t * p.o_st + h * p.o_sh + lane * E;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint32_t w[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2) w[e / 2] = L == 0.f ? 0u : pack2<T>(o[e] * inv, o[e + 1] * inv);
  if constexpr (E == 4)
    *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(out) = w[0];
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
  const long long most = (long long)std::min(p.batch, kMaxBatch) * p.nkv * pl.max_tiles;
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
  const long long rows = (long long)a.p.batch * a.p.tree * a.p.nq;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((rows + 3) / 4));
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

size_t tree_attention_scratch_bytes(const TreeAttnParams& p) {
  return (kMaxBatch + 4) * sizeof(int) + part_floats(p, plan_of(p)) * sizeof(float);
}

cudaError_t tree_attention(const TreeAttnParams& p, void* scratch, cudaStream_t s) {
  if ((p.head_dim != 64 && p.head_dim != 128) || p.batch <= 0 || p.tree <= 0 || p.tree > 64 || p.nkv <= 0 ||
      p.nq <= 0 || p.nq % p.nkv != 0 || p.max_blocks <= 0 || p.num_blocks <= 0 || (p.dtype != kBF16 && p.dtype != kF16))
    return cudaErrorInvalidValue;
  const Plan pl = plan_of(p);
  if (pl.rb > 148 || (long long)std::min(p.batch, kMaxBatch) * p.nkv * pl.max_tiles >= (1ll << 31)) return cudaErrorInvalidValue;
  const bool bf16 = p.dtype == kBF16;
  TreeArgs a;
  a.p = p;
  a.group = p.nq / p.nkv;
  a.rb = pl.rb;
  a.shares = pl.shares;
  a.cum = reinterpret_cast<int*>(scratch);
  a.part_o = reinterpret_cast<float*>(a.cum + kMaxBatch + 4);
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
