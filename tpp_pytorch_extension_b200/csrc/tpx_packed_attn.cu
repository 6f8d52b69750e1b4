// Attention over whole prompts of different lengths laid end to end, on the 5th-generation tensor cores.
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j    over the keys j of the same sequence, j <= i when causal
//
// Rows of a tile are (token, group member) pairs of one key head, 128 / R tokens by R members, so that grouped heads share their keys
// and short prompts fill tiles. A unit of work is two such tiles A and B, consecutive in their sequence, that walk the same keys in tiles
// of 128: while the softmax warps work on one tile's scores the tensor core works on the other's, and every key tile is fetched once for
// 256 rows (at one fetch per 128 rows L2 would bound it: 64 bytes per clock and SM).
//   S = Q K^T   A = 128 rows in shared memory, B = 128 keys, D = 128 fp32 columns of tensor memory
//   O += P V    A = P in tensor memory (bf16, over the columns of S that it came from), B = 128 keys read MN-major, D = H columns
//   warp 0: TMA, keys and values through a ring of four tiles; warp 1: tensor memory, MMAs; warp 2: which unit comes next;
//   warps 4-7, 8-11: softmax and output of tile A, B, one row per thread; they take the registers that warps 0-3 give back
// O stays in tensor memory. The maximum that scores are taken off is a reference that follows the running maximum only when a score
// passes it by 2^8: the row's O and sum are then rescaled by the softmax thread itself (O is complete up to the tile before whenever
// scores arrive, since commits cover all earlier MMAs). P is rounded to bf16 for the MMA, the row sum adds the unrounded weights.
//
// 8192 tokens, 32/8 heads of 128: 535-549 us, 1.00-1.03 PFLOP/s. The tensor pipe is busy 60 % of the time, the exponentials 57 %; instructions are what the
// loop is short of next (issue slots 32 %, but from code that does not stay in the nearest instruction cache), so less code per step is faster code. 16
// prompts of up to 2048: 75 us; 24 of up to 300, 32/32 heads of 64: 29 us, where each unit is one chain of dependent steps.
//
// Values in places that a row does not see must not reach it, whatever they are (0 * NaN is NaN): in key tiles that not all rows see in
// full, softmax warps look through the values in shared memory, zero what is not finite, and add it back at the end to rows that see it.
#include "tpx_tc_ptx.cuh"
#include "../../include/tpx_packed.h"

namespace tpx {

static __device__ unsigned g_packed_err;  // set when a bounded wait gave up; read and cleared by tpx_packed_status

constexpr int kPkThreads = 384;   // TMA, MMA and unit warps (and one that idles), two warpgroups of softmax
constexpr int kPkBuckets = 1024;  // sequences are found through prefix sums over at most so many runs of them

template <int H>
struct PkCfg {
  static constexpr int HALVES = H / 64;
  static constexpr int HALF_BYTES = 128 * 128;
  static constexpr int TILE_BYTES = HALVES * HALF_BYTES;  // 128 rows
  static constexpr int SLOTS = H == 128 ? 4 : 8;
  static constexpr size_t SMEM = (2 + SLOTS) * TILE_BYTES + 1024;
  static constexpr uint32_t COL_S = 0, COL_O = 256;  // + 128 per tile; P over the first 64 columns of S
};

struct PkParams {
  const int32_t *cu, *cached;  // cached: the tokens cached of each sequence, for calls of the new ones alone
  const uint16_t* v;
  uint16_t* out;
  int64_t ldv;
  int T, B, Nq, Nkv, R, TPT, causal;  // TPT: tokens of a tile
  float sc2;
};

__device__ __forceinline__ void pk_tma_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
      "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void pk_tma_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void pk_mma_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n  tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(adesc),
               "l"(bdesc), "r"(idesc), "r"(acc)
               : "memory");
}
__device__ __forceinline__ void pk_mma_ts(uint32_t d, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n  tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a_tmem),
               "l"(bdesc), "r"(idesc), "r"(acc)
               : "memory");
}
// MN-major operand in 128-byte swizzle: rows of 128 bytes are consecutive keys, 8-key groups 1024 bytes apart, the next 64 values of the
// head `lbo` bytes further
__device__ __forceinline__ uint64_t pk_desc_mn(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void pk_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pk_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void pk_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pk_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float pk_ex2(float x) {  // 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pk_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// pairs of fp32 in 64-bit registers
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pk_pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void pk_halves(f32x2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a)); }
__device__ __forceinline__ f32x2 pk_fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 pk_add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 pk_mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t pk_pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Rows first .. first + n - 1 of sequence b. PART: sequences of which tokens are cached have none (a kernel of its own: the test in the one for all
// sequences took 543-548 us for 536-540, 8192 tokens, and 30.6 for 29.4, 24 short prompts)
template <bool PART>
__device__ __forceinline__ void pk_sequence(const PkParams& p, int b, int& first, int& n) {
  first = min(max(p.cu[b], 0), p.T);
  n = max(min(max(p.cu[b + 1], 0), p.T) - first, 0);
  if (PART && p.cached[b] > 0) n = 0;
}
// Units of a sequence. One that fills a single tile has its key heads in pairs, a tile each with keys of its own: units of one tile leave half of a
// block idle and every step of it waiting for the one before (24 prompts of up to 300 tokens, 32 heads of 64: 42.7 us)
template <bool PART>
__device__ __forceinline__ int pk_units(const PkParams& p, int b) {
  int first, n;
  pk_sequence<PART>(p, b, first, n);
  return n <= p.TPT ? (n > 0 ? (p.Nkv + 1) / 2 : 0) : (n + 2 * p.TPT - 1) / (2 * p.TPT) * p.Nkv;
}

struct __align__(16) PkUnit {
  int tok0, n;            // first row of the sequence, its tokens
  int t0[2], head[2];     // first token and key head of tile A and B
  int tiles[2];           // key tiles that they walk; 0: no such tile
  int split;              // the tiles have keys of their own, one tile each: ring slots are K A, K B, V A, V B (K, V without a tile B)
};
constexpr int kPkAhead = 4;      // units that are looked up ahead
constexpr int kPkSorted = 128;   // sequences, at most, whose units are dealt by length
// The units of a block: rounds over all blocks, every other one backwards, since units get shorter from round to round
__device__ __forceinline__ int pk_nth(int round) { return round * (int)gridDim.x + ((round & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x); }
template <bool PART>
__device__ __forceinline__ void pk_fill(const PkParams& p, PkUnit& w, int b, bool split, int pair, int head) {
  pk_sequence<PART>(p, b, w.tok0, w.n);
  w.split = split;
  if (split) {
    w.t0[0] = w.t0[1] = 0;
    w.head[0] = 2 * head;
    w.head[1] = 2 * head + 1;
    w.tiles[0] = 1;
    w.tiles[1] = 2 * head + 1 < p.Nkv;
    return;
  }
  w.head[0] = w.head[1] = head;
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const int first = (2 * pair + x) * p.TPT, last = min(first + p.TPT, w.n) - 1;
    w.t0[x] = first;
    w.tiles[x] = first >= w.n ? 0 : ((p.causal ? last + 1 : w.n) + 127) / 128;
  }
}
// Unit u of the call, sequences in order: the last tokens (with the most keys) of a sequence first, heads of the same tokens side by side
template <bool PART>
__device__ __forceinline__ void pk_in_order(const PkParams& p, PkUnit& w, const int* pre, int buckets, int stride, int u) {
  int lo = 0, hi = buckets;  // pre[lo] <= u < pre[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (pre[m] <= u) lo = m;
    else hi = m;
  }
  int at = pre[lo], b = lo * stride, units = 0;
  for (; b < p.B; b++) {
    units = pk_units<PART>(p, b);
    if (u < at + units) break;
    at += units;
  }
  b = min(b, p.B - 1);
  int first, n;
  pk_sequence<PART>(p, b, first, n);
  const int k = u - at;
  if (n <= p.TPT) pk_fill<PART>(p, w, b, true, 0, k);
  else pk_fill<PART>(p, w, b, false, units / p.Nkv - 1 - k / p.Nkv, k % p.Nkv);
}
// Unit u of the call, those with the most keys first: pair by pair of tiles from the end of the longest sequence down, the pairs of all sequences that
// are as long side by side, sequences of a single tile last. A warp looks one up together: pairs[i] are those of its sequence 32 i + lane, 0 in a
// single tile (single: such a sequence). Units in order of the sequences: 16 prompts of up to 2048 tokens 85.3 us
template <bool PART>
__device__ __forceinline__ void pk_by_length(const PkParams& p, PkUnit& w, const int (&pairs)[kPkSorted / 32], const unsigned (&single)[kPkSorted / 32], int most, int u) {
  auto above = [&](int k) {  // units of pairs k and later
    int v = 0;
#pragma unroll
    for (int i = 0; i < kPkSorted / 32; i++) v += max(pairs[i] - k, 0);
    return __reduce_add_sync(0xffffffffu, v) * p.Nkv;
  };
  int lo = 0, hi = most;  // above(hi) <= u; above(lo) > u unless the unit is one of a single tile
  int behind = 0, all = above(0);
  const bool in_pairs = u < all;
  while (in_pairs && hi - lo > 1) {
    const int m = (lo + hi) >> 1, v = above(m);
    if (v > u) {
      lo = m;
    } else {
      hi = m;
      behind = v;
    }
  }
  const int r = u - (in_pairs ? behind : all), each = in_pairs ? p.Nkv : (p.Nkv + 1) / 2;
  int m = r / each, b = -1;  // the sequence is the m-th of those that have one
#pragma unroll
  for (int i = 0; i < kPkSorted / 32; i++) {
    const unsigned has = in_pairs ? __ballot_sync(0xffffffffu, pairs[i] > lo) : single[i];
    const int n = __popc(has);
    if (b < 0 && m < n) b = 32 * i + __fns(has, 0, m + 1);
    m -= n;
  }
  pk_fill<PART>(p, w, max(b, 0), !in_pairs, lo, r % each);
}

template <int H, bool PART>
__global__ void __launch_bounds__(kPkThreads, 1)
packed_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const PkParams p) {
  using C = PkCfg<H>;
  extern __shared__ unsigned char pk_smem_raw[];
  __shared__ __align__(8) unsigned long long q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], o_free[2], kv_full[C::SLOTS], kv_empty[C::SLOTS],
      u_full[kPkAhead], u_empty[kPkAhead];
  __shared__ PkUnit ring[kPkAhead];  // the block's units, a few ahead
  __shared__ uint32_t tmem_holder;
  __shared__ int dirty;  // some value in a tile's margin is not finite
  __shared__ int pre[kPkBuckets + 1], warp_sum[kPkThreads / 32];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (tc_smem_u32(pk_smem_raw) + 1023u) & ~1023u;
  const uint32_t q_s = smem, kv_s = smem + 2 * C::TILE_BYTES;

  if (threadIdx.x == 0) {
    dirty = 0;
    for (int x = 0; x < 2; x++) {
      tc_mbar_init(tc_smem_u32(&q_full[x]), 1);
      tc_mbar_init(tc_smem_u32(&q_empty[x]), 1);
      tc_mbar_init(tc_smem_u32(&s_full[x]), 1);
      tc_mbar_init(tc_smem_u32(&p_full[x]), 128);
      tc_mbar_init(tc_smem_u32(&o_full[x]), 1);
      tc_mbar_init(tc_smem_u32(&o_free[x]), 128);
    }
    for (int s = 0; s < C::SLOTS; s++) {
      tc_mbar_init(tc_smem_u32(&kv_full[s]), 1);
      tc_mbar_init(tc_smem_u32(&kv_empty[s]), 1);
    }
    for (int s = 0; s < kPkAhead; s++) {
      tc_mbar_init(tc_smem_u32(&u_full[s]), 1);
      tc_mbar_init(tc_smem_u32(&u_empty[s]), 2 + 8);  // TMA, MMA, eight softmax warps
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(&tmem_holder)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_trigger();
  pdl_wait();

  // ---- units before each run of `stride` sequences
  const int stride = (p.B + kPkBuckets - 1) / kPkBuckets, buckets = (p.B + stride - 1) / stride;
  int total;
  {
    const int per = (buckets + kPkThreads - 1) / kPkThreads, lo = min((int)threadIdx.x * per, buckets), hi = min(lo + per, buckets);
    int mine = 0;
    for (int b = lo * stride; b < min(hi * stride, p.B); b++) mine += pk_units<PART>(p, b);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int at = incl - mine;
    total = 0;
    for (int i = 0; i < kPkThreads / 32; i++) {
      if (i < warp) at += warp_sum[i];
      total += warp_sum[i];
    }
    for (int k = lo; k < hi; k++) {
      pre[k] = at;
      for (int b = k * stride; b < min((k + 1) * stride, p.B); b++) at += pk_units<PART>(p, b);
    }
    if (threadIdx.x == 0) pre[buckets] = total;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  const int units = total;

  // 384 x 168 registers at launch = 256 x 216 + 128 x 72
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (tc_elect()) {
      const uint32_t q_bytes = (uint32_t)(C::HALVES * p.TPT * p.R * 128);
      int seen[2] = {0, 0}, c = 0;  // units of each tile, ring slots so far
      bool ok = true;
      for (int round = 0; ok && round * (int)gridDim.x < units; round++) {
        if (pk_nth(round) >= units) break;
        const int slot = round % kPkAhead;
        if (!tc_wait(tc_smem_u32(&u_full[slot]), (uint32_t)((round / kPkAhead) & 1))) { ok = false; break; }
        const PkUnit w = ring[slot];
        tc_mbar_arrive(tc_smem_u32(&u_empty[slot]));
        const int n = max(w.tiles[0], w.tiles[1]);
        auto load_q = [&](int x) {
          if (w.tiles[x] == 0) return;
          if (seen[x] && !tc_wait(tc_smem_u32(&q_empty[x]), (uint32_t)((seen[x] - 1) & 1))) { ok = false; return; }
          seen[x]++;
          const uint32_t bar = tc_smem_u32(&q_full[x]);
          tc_mbar_expect_tx(bar, q_bytes);
#pragma unroll
          for (int h = 0; h < C::HALVES; h++)  // 64 values x R members x 1 key head x TPT tokens
            pk_tma_4d(q_s + x * C::TILE_BYTES + h * C::HALF_BYTES, &tmQ, h * 64, 0, w.head[x], w.tok0 + w.t0[x], bar);
        };
        auto load_kv = [&](const CUtensorMap* map, int j, int x) {
          const int s = c % C::SLOTS;
          if (c >= C::SLOTS && !tc_wait(tc_smem_u32(&kv_empty[s]), (uint32_t)((c / C::SLOTS - 1) & 1))) { ok = false; return; }
          c++;
          const uint32_t bar = tc_smem_u32(&kv_full[s]);
          tc_mbar_expect_tx(bar, C::TILE_BYTES);
#pragma unroll
          for (int h = 0; h < C::HALVES; h++)
            pk_tma_3d(kv_s + s * C::TILE_BYTES + h * C::HALF_BYTES, map, h * 64, w.head[x], w.tok0 + j * 128, bar);
        };
        load_q(0);
        if (ok) load_kv(&tmK, 0, 0);
        if (ok) load_q(1);
        if (w.split) {
          if (ok && w.tiles[1]) load_kv(&tmK, 0, 1);
          if (ok) load_kv(&tmV, 0, 0);
          if (ok && w.tiles[1]) load_kv(&tmV, 0, 1);
          continue;
        }
        for (int j = 0; ok && j < n; j++) {
          load_kv(&tmV, j, 0);
          if (ok && j + 1 < n) load_kv(&tmK, j + 1, 0);
        }
      }
      if (!ok) {  // copies in flight land before this block gives its shared memory back
        atomicExch(&g_packed_err, 1u);
        for (int k = max(0, c - C::SLOTS); k < c; k++) tc_wait(tc_smem_u32(&kv_full[k % C::SLOTS]), (uint32_t)((k / C::SLOTS) & 1));
        for (int x = 0; x < 2; x++)
          if (seen[x]) tc_wait(tc_smem_u32(&q_full[x]), (uint32_t)((seen[x] - 1) & 1));
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (tc_elect()) {
      const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
      const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(H >> 3) << 17) | ((128u >> 4) << 24);
      int seen[2] = {0, 0}, steps[2] = {0, 0}, c = 0;  // c: ring slots used up
      bool ok = true;
      auto wait = [&](unsigned long long* bar, int parity) {
        if (ok && !tc_wait(tc_smem_u32(bar), (uint32_t)(parity & 1))) {
          ok = false;
          atomicExch(&g_packed_err, 2u);
        }
        return ok;
      };
      auto scores = [&](int x, int slot) {
        tc_fence_after();
        const uint64_t q0 = tc_smem_desc(q_s + x * C::TILE_BYTES), k0 = tc_smem_desc(kv_s + slot * C::TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < H / 16; kk++) {
          const uint64_t off = (uint64_t)((kk >> 2) * (C::HALF_BYTES / 16) + (kk & 3) * 2);
          pk_mma_ss(tmem + C::COL_S + x * 128, q0 + off, k0 + off, idesc_s, kk > 0 ? 1u : 0u);
        }
        tc_commit(tc_smem_u32(&s_full[x]));
      };
      for (int round = 0; ok && round * (int)gridDim.x < units; round++) {
        if (pk_nth(round) >= units || !wait(&u_full[round % kPkAhead], round / kPkAhead)) break;
        const PkUnit w = ring[round % kPkAhead];
        tc_mbar_arrive(tc_smem_u32(&u_empty[round % kPkAhead]));
        const int n = max(w.tiles[0], w.tiles[1]);
        for (int x = 0; ok && x < 2; x++) {  // scores of the first keys
          if (w.tiles[x] == 0) continue;
          if ((x == 0 || w.split) && !wait(&kv_full[c % C::SLOTS], c / C::SLOTS)) break;
          if (!wait(&q_full[x], seen[x])) break;
          scores(x, c % C::SLOTS);
          if (w.split) {
            tc_commit(tc_smem_u32(&kv_empty[c % C::SLOTS]));
            c++;
          }
        }
        if (!ok) break;
        if (!w.split) {
          tc_commit(tc_smem_u32(&kv_empty[c % C::SLOTS]));
          c++;
        }
        for (int j = 0; ok && j < n; j++) {
          int vs = c % C::SLOTS;
          const int ks = (c + 1) % C::SLOTS;
          if (!wait(&kv_full[vs], c / C::SLOTS)) break;
          if (j + 1 < n && !wait(&kv_full[ks], (c + 1) / C::SLOTS)) break;
          for (int x = 0; ok && x < 2; x++) {
            if (j >= w.tiles[x]) continue;
            if (w.split && x == 1) {  // values of its own
              tc_commit(tc_smem_u32(&kv_empty[vs]));
              c++;
              vs = c % C::SLOTS;
              if (!wait(&kv_full[vs], c / C::SLOTS)) break;
            }
            if (j == 0 && seen[x] && !wait(&o_free[x], seen[x] - 1)) break;
            if (!wait(&p_full[x], steps[x])) break;
            tc_fence_after();
            const uint64_t v0 = pk_desc_mn(kv_s + vs * C::TILE_BYTES, C::HALF_BYTES);
#pragma unroll
            for (int kk = 0; kk < 8; kk++)  // 16 keys: 8 columns of packed weights, two 8-key groups of values
              pk_mma_ts(tmem + C::COL_O + x * 128, tmem + C::COL_S + x * 128 + kk * 8, v0 + kk * 128, idesc_o,
                        j > 0 || kk > 0 ? 1u : 0u);
            steps[x]++;
            if (j + 1 < w.tiles[x]) {
              scores(x, ks);
            } else {
              tc_commit(tc_smem_u32(&o_full[x]));
              tc_commit(tc_smem_u32(&q_empty[x]));
              seen[x]++;
            }
          }
          if (!ok) break;
          tc_commit(tc_smem_u32(&kv_empty[vs]));
          c++;
          if (j + 1 < n) {
            tc_commit(tc_smem_u32(&kv_empty[ks]));
            c++;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------ units, ahead of those who work on them
    // By length, as long as a warp can hold the sizes of all sequences: 16 prompts of up to 2048 72.5 us, in order of the sequences 84.4; 120 of up to 1000
    // 283 and 308; 200, with twice the table, 508-532 and 543. Not causal, every pair of a sequence takes all of its keys, and the order of the
    // sequences is the faster one for many: 200 prompts 807 us by length, 722 in order (16: 120 and 118)
    const bool sorted = p.causal && p.B <= kPkSorted;
    int pairs[kPkSorted / 32], most = 0;
    unsigned single[kPkSorted / 32];
#pragma unroll
    for (int i = 0; i < kPkSorted / 32; i++) {
      int first, n = 0;
      if (sorted && 32 * i + lane < p.B) pk_sequence<PART>(p, 32 * i + lane, first, n);
      pairs[i] = n <= p.TPT ? 0 : (n + 2 * p.TPT - 1) / (2 * p.TPT);
      single[i] = __ballot_sync(0xffffffffu, n > 0 && n <= p.TPT);
      most = max(most, pairs[i]);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    for (int round = 0; round * (int)gridDim.x < units; round++) {
      const int u = pk_nth(round), slot = round % kPkAhead;
      if (u >= units) break;
      if (round >= kPkAhead && !tc_wait_warp(tc_smem_u32(&u_empty[slot]), (uint32_t)((round / kPkAhead - 1) & 1))) {
        if (lane == 0) atomicExch(&g_packed_err, 4u);
        break;
      }
      PkUnit w;
      if (sorted) pk_by_length<PART>(p, w, pairs, single, most, u);
      else pk_in_order<PART>(p, w, pre, buckets, stride, u);
      if (lane == 0) {
        ring[slot] = w;
        tc_mbar_arrive(tc_smem_u32(&u_full[slot]));
      }
      __syncwarp();
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------ softmax and output, a row per thread
    const int x = (warp >> 2) - 1, quarter = warp & 3, rl = quarter * 32 + lane, wg_tid = threadIdx.x & 127;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_t = tmem + lane_base + C::COL_S + x * 128, o_t = tmem + lane_base + C::COL_O + x * 128;
    const int tok = rl / p.R, member = rl % p.R;
    int seen = 0, steps = 0, c = 0;
    bool ok = true;
    auto wait = [&](unsigned long long* bar, int parity) {
      if (ok && !tc_wait_warp(tc_smem_u32(bar), (uint32_t)(parity & 1))) {
        ok = false;
        if (lane == 0) atomicExch(&g_packed_err, 3u);
      }
      return ok;
    };
    for (int round = 0; ok && round * (int)gridDim.x < units; round++) {
      if (pk_nth(round) >= units || !wait(&u_full[round % kPkAhead], round / kPkAhead)) break;
      const volatile PkUnit& w = ring[round % kPkAhead];  // read where it is needed: registers are short
      auto release = [&]() {
        __syncwarp();
        if (lane == 0) tc_mbar_arrive(tc_smem_u32(&u_empty[round % kPkAhead]));
      };
      const int n = w.tiles[x];
      const int v0 = c + (w.split ? w.tiles[0] + w.tiles[1] + x : 1);  // values of key tile j are in ring slot v0 + 2 j
      c += w.split ? 2 * (w.tiles[0] + w.tiles[1]) : 2 * max(w.tiles[0], w.tiles[1]);
      if (n == 0) {
        release();
        continue;
      }
      const int t = w.t0[x] + tok;
      const bool live = tok < p.TPT && t < w.n;
      const int klim = p.causal ? min(t + 1, w.n) : w.n;               // keys [0, klim) are seen (dead rows: anything)
      const int whole = (p.causal ? w.t0[0] + 1 : w.n) / 128;              // key tiles that every row of the unit sees in full
      float m_ref = -INFINITY;
      f32x2 l2[2] = {0, 0};  // partial sums of the weights
      for (int j = 0; j < n; j++) {
        if (!wait(&s_full[x], steps)) break;
        steps++;
        tc_fence_after();
        uint32_t v[128];
#pragma unroll
        for (int i = 0; i < 4; i++) pk_ld32(s_t + i * 32, v + i * 32);
        pk_ld_wait();
        float* s = reinterpret_cast<float*>(v);
        const bool margin = j >= whole;
        if (margin) {
          const int lim = klim - j * 128;
#pragma unroll
          for (int i = 0; i < 128; i++)
            if (i >= lim) s[i] = -INFINITY;
        }
        float unit = p.sc2;
        float top8[8];
#pragma unroll
        for (int k = 0; k < 8; k++) top8[k] = fmaxf(pk_max3(s[2 * k], s[2 * k + 1], s[16 + 2 * k]), s[17 + 2 * k]);
#pragma unroll
        for (int i = 32; i < 128; i += 16)
#pragma unroll
          for (int k = 0; k < 8; k++) top8[k] = pk_max3(top8[k], s[i + 2 * k], s[i + 2 * k + 1]);
        float top = fmaxf(pk_max3(pk_max3(top8[0], top8[1], top8[2]), top8[3], top8[4]), pk_max3(top8[5], top8[6], top8[7]));
        // The multiply-add below takes the rounded reference off an unrounded score, which is nothing for ordinary scores; large ones are
        // rounded first, so that the largest weight is what it should be (for all rows of a warp, so rows of no token have no say in it)
        if (__any_sync(0xffffffffu, live && !(fabsf(top) * unit < 4096.0f)) && unit != 1.0f) {
#pragma unroll
          for (int i = 0; i < 128; i++) s[i] *= unit;
          top *= unit;
          unit = 1.0f;
        }
        top *= unit;
        const bool pass = top > m_ref + 8.0f;
        if (__any_sync(0xffffffffu, pass)) {
          const float m_new = pass ? top : m_ref, alpha = pass ? pk_ex2(m_ref - m_new) : 1.0f;
          m_ref = m_new;
          l2[0] = pk_mul2(l2[0], pk_pair(alpha, alpha));
          l2[1] = pk_mul2(l2[1], pk_pair(alpha, alpha));
          if (j > 0) {
#pragma unroll
            for (int i = 0; i < H / 32; i++) {
              uint32_t o[32];
              pk_ld32(o_t + i * 32, o);
              pk_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              pk_st32(o_t + i * 32, o);
            }
          }
        }
        if (margin) {
          const int vc = v0 + 2 * j;
          if (!wait(&kv_full[vc % C::SLOTS], vc / C::SLOTS)) break;
          const uint32_t base = kv_s + (vc % C::SLOTS) * C::TILE_BYTES + wg_tid * 16;
          const __nv_bfloat162 zero = __floats2bfloat162_rn(0.0f, 0.0f);
          __nv_bfloat162 bad[4] = {zero, zero, zero, zero};  // 0 * x summed: a NaN where any x is not finite
#pragma unroll
          for (int i = 0; i < C::TILE_BYTES / 2048; i++) {
            uint32_t a[4];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(base + i * 2048));
#pragma unroll
            for (int k = 0; k < 4; k++) bad[k] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a[k]), zero, bad[k]);
          }
          const __nv_bfloat162 sum = __hadd2(__hadd2(bad[0], bad[1]), __hadd2(bad[2], bad[3]));
          if (__hisnan(sum.x) || __hisnan(sum.y)) {
            *reinterpret_cast<volatile int*>(&dirty) = 1;
            __threadfence_block();
            for (int i = 0; i < C::TILE_BYTES / 2048; i++) {
              for (int k = 0; k < 8; k++) {
                uint16_t e;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(e) : "r"(base + i * 2048 + 2 * k));
                if ((e & 0x7f80) == 0x7f80) asm volatile("st.shared.u16 [%0], %1;" ::"r"(base + i * 2048 + 2 * k), "h"((uint16_t)0) : "memory");
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        const float ref = m_ref == -INFINITY ? 0.0f : m_ref;
        const f32x2 unit2 = pk_pair(unit, unit), ref2 = pk_pair(-ref, -ref);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          uint32_t pw[32];
#pragma unroll
          for (int k = 0; k < 32; k++) {
            float a, b;
            pk_halves(pk_fma2(pk_pair(s[64 * i + 2 * k], s[64 * i + 2 * k + 1]), unit2, ref2), a, b);
            a = pk_ex2(a);
            b = pk_ex2(b);
            l2[k & 1] = pk_add2(l2[k & 1], pk_pair(a, b));
            pw[k] = pk_pack(a, b);
          }
          pk_st32(s_t + i * 32, pw);
        }
        __syncwarp();
        pk_st_wait();
        tc_fence_before();
        tc_mbar_arrive(tc_smem_u32(&p_full[x]));
      }
      if (!wait(&o_full[x], seen)) break;
      seen++;
      tc_fence_after();
      float l[4];
      pk_halves(l2[0], l[0], l[1]);
      pk_halves(l2[1], l[2], l[3]);
      const float inv = 1.0f / ((l[0] + l[1]) + (l[2] + l[3]));
      const bool mend = *reinterpret_cast<volatile int*>(&dirty) != 0;
      uint16_t* dst = p.out + ((int64_t)(w.tok0 + (live ? t : 0)) * p.Nq + w.head[x] * p.R + member) * H;
#pragma unroll
      for (int i = 0; i < H / 32; i++) {
        uint32_t o[32];
        pk_ld32(o_t + i * 32, o);
        pk_ld_wait();
        if (live && mend) {
          for (int key = whole * 128; key < klim; key++) {
            const uint16_t* src = p.v + (int64_t)(w.tok0 + key) * p.ldv + w.head[x] * H + i * 32;
#pragma unroll
            for (int k = 0; k < 32; k++) {
              const uint16_t e = src[k];
              if ((e & 0x7f80) == 0x7f80) o[k] = __float_as_uint(__uint_as_float(o[k]) + bf16_bits_to_f32(e));
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          if (!live) break;
          uint32_t r[4];
#pragma unroll
          for (int e = 0; e < 4; e++) r[e] = pk_pack(__uint_as_float(o[k + 2 * e]) * inv, __uint_as_float(o[k + 2 * e + 1]) * inv);
          *reinterpret_cast<uint4*>(dst + i * 32 + k) = make_uint4(r[0], r[1], r[2], r[3]);
        }
        __syncwarp();
      }
      tc_fence_before();
      tc_mbar_arrive(tc_smem_u32(&o_free[x]));
      release();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---------------------------------------------------------------- host side
typedef CUresult (*PkEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static PkEncodeFn pk_encode_fn() {
  static PkEncodeFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PkEncodeFn>(ptr);
  }
  return fn;
}

static int pk_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  PkEncodeFn fn = pk_encode_fn();
  TPX_REQUIRE(fn, TPX_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TPX_REQUIRE(r == CUDA_SUCCESS, TPX_ERR_CUDA, "packed attention: cuTensorMapEncodeTiled failed with %d", (int)r);
  return TPX_OK;
}

template <int H, bool PART>
static int pk_launch(const TpxPackedAttention& a, PkParams& p, cudaStream_t st) {
  using C = PkCfg<H>;
  CUtensorMap mq, mk, mv;
  const cuuint64_t R = p.R, Nkv = p.Nkv, T = p.T;
  const cuuint64_t qd[4] = {H, R, Nkv, T}, qs[3] = {H * 2, R * H * 2, (cuuint64_t)a.ldq * 2}, kd[3] = {H, Nkv, T}, ks[2] = {H * 2, (cuuint64_t)a.ldk * 2},
                   vs[2] = {H * 2, (cuuint64_t)a.ldv * 2};
  const cuuint32_t qb[4] = {64, (cuuint32_t)R, 1, (cuuint32_t)p.TPT}, kb[3] = {64, 1, 128};
  int rc;
  if ((rc = pk_map(&mq, a.q, 4, qd, qs, qb)) || (rc = pk_map(&mk, a.k, 3, kd, ks, kb)) || (rc = pk_map(&mv, a.v, 3, kd, vs, kb))) return rc;
  static bool opted[16] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16 || !opted[dev]) {
    TPX_CUDA_OK(cudaFuncSetAttribute(packed_attn_kernel<H, PART>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
    if (dev >= 0 && dev < 16) opted[dev] = true;
  }
  const int64_t most = ((int64_t)p.T / (2 * p.TPT) + p.B) * p.Nkv;  // units at most, whatever the lengths
  TPX_CUDA_OK(launch_pdl(packed_attn_kernel<H, PART>, dim3((unsigned)(most < sm_count() ? most : sm_count())), dim3(kPkThreads), C::SMEM, st, mq, mk, mv, p));
  return TPX_OK;
}

}  // namespace tpx

using namespace tpx;

static int packed_attention(const TpxPackedAttention* a, const int32_t* cached, void* stream) {
  TPX_REQUIRE(a && a->cu_seqlens && (a->T == 0 || (a->q && a->k && a->v && a->out)), TPX_ERR_ARG, "packed_attention: null pointer");
  TPX_REQUIRE(a->H == 64 || a->H == 128, TPX_ERR_UNSUPPORTED, "packed_attention: head size %ld not supported (64 or 128)", (long)a->H);
  TPX_REQUIRE(a->Nkv > 0 && a->Nkv <= 1024 && a->Nq > 0 && a->Nq % a->Nkv == 0, TPX_ERR_ARG, "packed_attention: %ld query heads for %ld key heads", (long)a->Nq,
              (long)a->Nkv);
  TPX_REQUIRE(a->Nq / a->Nkv <= 128, TPX_ERR_UNSUPPORTED, "packed_attention: more than 128 query heads per key head");
  TPX_REQUIRE(a->T >= 0 && a->B > 0 && a->B <= (1 << 24) && a->T + 1024 < (1ll << 31) && (a->T + a->B) * a->Nkv < (1ll << 31), TPX_ERR_ARG,
              "packed_attention: %ld tokens of %ld sequences", (long)a->T, (long)a->B);
  TPX_REQUIRE((((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) & 15) == 0 && (a->ldq | a->ldk | a->ldv) % 8 == 0, TPX_ERR_ARG,
              "packed_attention: tensors and their rows must be 16-byte aligned");
  TPX_REQUIRE(a->scale > 0.0f && a->scale < INFINITY, TPX_ERR_ARG, "packed_attention: a scale of %g (it must be positive)", (double)a->scale);
  if (a->T == 0) return TPX_OK;
  PkParams p = {};
  p.cu = a->cu_seqlens;
  p.cached = cached;
  p.v = a->v;
  p.out = a->out;
  p.ldv = a->ldv;
  p.T = (int)a->T;
  p.B = (int)a->B;
  p.Nq = (int)a->Nq;
  p.Nkv = (int)a->Nkv;
  p.R = (int)(a->Nq / a->Nkv);
  p.TPT = 128 / p.R;
  p.causal = a->causal;
  p.sc2 = a->scale * 1.4426950408889634f;
  cudaStream_t st = (cudaStream_t)stream;
  if (cached) return a->H == 128 ? pk_launch<128, true>(*a, p, st) : pk_launch<64, true>(*a, p, st);
  return a->H == 128 ? pk_launch<128, false>(*a, p, st) : pk_launch<64, false>(*a, p, st);
}

extern "C" int tpx_packed_attention(const TpxPackedAttention* a, void* stream) { return packed_attention(a, nullptr, stream); }

extern "C" int tpx_packed_attention_new(const TpxPackedAttention* a, const int32_t* lengths, void* stream) {
  TPX_REQUIRE(lengths, TPX_ERR_ARG, "packed_attention_new: null pointer");
  return packed_attention(a, lengths, stream);
}

extern "C" int tpx_packed_status(void* stream, unsigned* status_host) {
  TPX_REQUIRE(status_host, TPX_ERR_ARG, "packed_status: null pointer");
  static void* ptrs[64] = {};
  int dev = 0;
  TPX_CUDA_OK(cudaGetDevice(&dev));
  TPX_REQUIRE(dev >= 0 && dev < 64, TPX_ERR_UNSUPPORTED, "packed_status: device index %d out of range", dev);
  if (!ptrs[dev]) TPX_CUDA_OK(cudaGetSymbolAddress(&ptrs[dev], g_packed_err));
  TPX_CUDA_OK(cudaMemcpyAsync(status_host, ptrs[dev], 4, cudaMemcpyDeviceToHost, (cudaStream_t)stream));
  TPX_CUDA_OK(cudaMemsetAsync(ptrs[dev], 0, 4, (cudaStream_t)stream));
  TPX_CUDA_OK(cudaStreamSynchronize((cudaStream_t)stream));
  return TPX_OK;
}
