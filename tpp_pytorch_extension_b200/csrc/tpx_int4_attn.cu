// Attention of a few new tokens per sequence over the 4-bit cache of tpx_packed.h.
//
//   out = softmax(scale * q K^T) V,   K[t][d] = kz + ks * kc[t][d],  V alike, with codes 0..15 and a scale and a minimum per 64 values
//
// The loop over the cache is bound by instructions per code, not by the matrix unit, so codes go to mma.sync as nearly as they lie there,
// scales and minima around them (tcgen05 has no form this narrow: it would need 128 query rows or keys):
//   q.K  = sum over groups of 64:  ks (q . kc) + kz sum(q)
//          m16n8k32 u8 x s8 on the bytes as they lie: a byte is 16 odd + even, and
//          q_even even + q_odd odd = (q_odd / 16) byte + (q_even - q_odd / 16) (byte & 15), so eight codes cost one AND. The two
//          factors are whole numbers of 2^-21 of the row's largest value (q_odd: 2^-17), cut into three signed digits of 8 bits, each a
//          column: products and sums are exact in 32 bits. Columns (2 r, 2 r + 1) are the upper digits of row r, so that a lane has
//          whole scores; the accumulator starts at the bits of 1.5 * 2^23, which makes it a float.
//   P V  = sum over t: (p vs) (vc - 8) + p (vz + 8 vs)
//          m16n8k16 fp16: a byte of two codes in the mantissa of 1024 is an fp16, and so is its lower code alone; both go to the matrix unit
//          centred (one addition per pair) and the upper code's sum is the difference / 16. Centred, since p vs is rounded to fp16 and that
//          should not be weighed with the range's offset. p vs is kept in units of a power of two that every row and group of 64 has for
//          itself and that follows the largest p vs it has met: products from 2^-20 of that one up have all bits of fp16, smaller ones are
//          off by 2^-31 of it at most, however the scales of the groups, of the tokens and of the rows' weights differ.
// The cache is the 16-row operand: 16 tokens for keys, 16 of the head's dimensions for values. Weights get to the second product by movmatrix.
//
// A page of a head (4608 bytes at H = 128) is one warp's work item, fetched by cp.async into a ring of the warp's own: no barrier in the
// loop. The (sequence, key head, row chunk) segments, each rounded up to whole quanta of GW pages (GW warps work on one segment at a
// time), are laid end to end and cut evenly between all groups of GW warps of the GPU, whatever the sequences' lengths, which are read
// on the device. A segment that is cut leaves partial results in scratch, which the group that finishes it last adds up in the order of
// the pieces: results do not depend on who is last. Arrivals are counted in words that carry the call's own number, so that scratch may
// hold anything before, and calls share none.
// One sequence of 131072 tokens, 32/8 heads of 128: 42.9 us, of which 12 are the launch's start and end (1024 tokens: 12.4 us; a launch without work: 4.4) and the rest
// pages at 4.9 TB/s, 55 % of issue slots. 16 of 2048: 19.4 us; 64 of up to 4096 with 64/8 heads: 35.5 us; 8 times 5 tokens over up to 1500, 32/32 heads of 64: 15.8 us.
#include "tpx_int4.cuh"

namespace tpx {

constexpr int kI4Warps = 16;

struct I4Params {
  const uint16_t* q;
  uint16_t* out;
  const int32_t* cu;
  I4Cache c;
  float* part;                   // [workers][2][ROWS][H + 2]: maximum, sum, output of each row
  unsigned long long* counters;  // [workers]
  unsigned long long nonce;      // low 16 bits zero
  int64_t ldq;
  int T, Nq, R, causal, behind;  // behind: only sequences of which tokens are cached before the call have a part in it
  float sc2;                     // scale * log2(e)
};

constexpr uint32_t kI4Magic = 0x4B400000u;  // 1.5 * 2^23: a float whose low bits count whole numbers
__device__ __forceinline__ float i4_count(int v) { return __int_as_float(v) - __uint_as_float(kI4Magic); }

// d = a b + c with c the magic number in every place (first) or d
__device__ __forceinline__ void i4_mma_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y), "r"(kI4Magic));
}
__device__ __forceinline__ void i4_mma_u8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ void i4_mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t i4_transpose(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ float i4_ex2(float x) {  // 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t i4_pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t i4_pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float i4_pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ float i4_inverse(float pow2) { return __uint_as_float(0x7f000000u - __float_as_uint(pow2)); }  // of 2^-126 .. 2^126
// a += e b, and d = e b c, over the groups of a head: pairs of fp32 in one operation
template <int G>
__device__ __forceinline__ void i4_fma(float (&a)[G], float e, const float (&b)[G]) {
  if (G == 2)
    asm("{ .reg .b64 x, y, z;\n  mov.b64 x, {%2, %2};\n  mov.b64 y, {%3, %4};\n  mov.b64 z, {%0, %1};\n  fma.rn.f32x2 z, x, y, z;\n  mov.b64 {%0, %1}, z; }"
        : "+f"(a[0]), "+f"(a[G - 1])
        : "f"(e), "f"(b[0]), "f"(b[G - 1]));
  else
    a[0] = fmaf(e, b[0], a[0]);
}
template <int G>
__device__ __forceinline__ void i4_mul(float (&d)[G], float e, const float (&b)[G], const float (&c)[G]) {
  if (G == 2)
    asm("{ .reg .b64 x, y, z;\n  mov.b64 x, {%2, %2};\n  mov.b64 y, {%3, %4};\n  mov.b64 z, {%5, %6};\n  mul.rn.f32x2 x, x, y;\n  mul.rn.f32x2 x, x, z;\n  mov.b64 {%0, %1}, x; }"
        : "=f"(d[0]), "=f"(d[G - 1])
        : "f"(e), "f"(b[0]), "f"(b[G - 1]), "f"(c[0]), "f"(c[G - 1]));
  else
    d[0] = e * b[0] * c[0];
}
__device__ __forceinline__ uint32_t i4_add_f16(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two codes of two keys: the bytes B (0: bits 0..7, 1: bits 8..15) of both halves of w, minus 136, and their lower codes, minus 8, as fp16
template <int B>
__device__ __forceinline__ void i4_centred(uint32_t w, uint32_t& both, uint32_t& lower) {
  const uint32_t v = __byte_perm(w, 0x64646464u, B == 0 ? 0x4240 : 0x4341);  // 1024 + byte
  both = i4_add_f16(v, 0xe488e488u);                                        // - 1160
  lower = i4_add_f16(v & 0xff0fff0fu, 0xe408e408u);                         // - 1032
}
__device__ __forceinline__ void i4_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N>
__device__ __forceinline__ void i4_lds(const unsigned char* a, uint32_t (&v)[N]) {  // N words, 4 N-byte aligned
  if (N == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(a);
    v[0] = x.x; v[1 % N] = x.y; v[2 % N] = x.z; v[3 % N] = x.w;
  } else if (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(a);
    v[0] = x.x; v[1 % N] = x.y;
  } else {
    v[0] = *reinterpret_cast<const uint32_t*>(a);
  }
}

// Work of one sequence. A quantum is GW pages, one per warp of a group; a piece is what is never cut between groups: one quantum, or
// four where there is too little work for all groups anyway (more quanta in a row cost less than adding up partial results).
constexpr int kI4PieceShift = 2;
// Quanta that the start and the end of a run take the time of: without them a group that drew six short segments took 54 us where one
// with a part of a long segment took 27 (64 sequences of 1 to 4096 tokens)
constexpr int kI4Start = 2;
struct I4Seq {
  int n, keys, pages, chunks;  // tokens of the call, keys, their pages, row chunks
};
__device__ __forceinline__ I4Seq i4_seq(const I4Params& p, int b, int rows) {
  I4Seq s;
  if (p.cu) {
    const int lo = min(max(p.cu[b], 0), p.T), hi = min(max(p.cu[b + 1], 0), p.T);
    s.n = max(hi - lo, 0);
  } else {
    s.n = 1;
  }
  if (p.behind && p.c.lengths[b] <= 0) s.n = 0;
  const long long keys = (long long)max(p.c.lengths[b], 0) + s.n, cap = (long long)p.c.cols * kI4Page;
  s.keys = (int)min(keys, cap);
  s.pages = (s.keys + kI4Page - 1) / kI4Page;
  s.chunks = (int)(((long long)s.n * p.R + rows - 1) / rows);
  return s;
}
// Counts one arrival at a segment of `want` parts; whether it is the last. The word starts as anything but this call's number (that of another
// call, or none): who finds that (`was`: what it held some time ago) sets it up by one exchange, which fails only where another has; then
// everyone adds one. No retries: nineteen groups that finish together took 14 us to count themselves by compare-and-swap. The
// addition releases what the group has written before it met at a barrier, and acquires the others'.
__device__ __forceinline__ bool i4_arrive(unsigned long long* word, unsigned long long was, unsigned long long nonce, unsigned want) {
  if ((was & ~0xffffull) != nonce) atomicCAS(word, was, nonce);
  unsigned long long seen;
  asm volatile("atom.acq_rel.gpu.global.add.u64 %0, [%1], %2;" : "=l"(seen) : "l"(word), "l"(1ull) : "memory");
  const bool last = (unsigned)(seen & 0xffffull) + 1 == want;
  if (last) *reinterpret_cast<volatile unsigned long long*>(word) = 0;  // a replayed call starts anew
  return last;
}

// RT: query rows per lane, 4 RT in a chunk
template <int H, int RT>
struct I4Cfg {
  static constexpr int ROWS = 4 * RT;
  static constexpr int STAGES = 2;
  static constexpr int WARP_SHIFT = RT < 4 ? 4 : 3, WARPS = 1 << WARP_SHIFT;
  static_assert(WARPS <= kI4Warps, "scratch");
  // The run's place in the share, which its pages do not need, waits in shared memory while they are walked. With 8 rows it saves spills (64 sequences of up to
  // 4096 tokens, 64/8 heads of 128: 38.1 -> 34.6 us); with 4 rows it costs more than it saves (one of 131072, 32/8 heads: 44.2 -> 45.9 us)
  static constexpr bool PARK = RT == 2;
  static constexpr int TILES = RT + (RT + 1) / 2;          // n-tiles of q digits: upper two of 4 rows each, lowest of 8
  static constexpr int PITCH = H + 4;                      // floats of a row in the merge buffer
  static constexpr int MERGE = (ROWS * PITCH + 2 * ROWS) * 4;
  static constexpr int QBUF = TILES * (H / 32) * 256 + ROWS * 16;  // digits, then (scale, sums of q) of each row: a group's, over its first warp's merge buffer
  static constexpr int WARP_BYTES = STAGES * I4<H>::BYTES + (MERGE > QBUF ? MERGE : QBUF);
  static constexpr int SMEM = WARPS * WARP_BYTES;
};

template <int H, int RT>
__global__ void __launch_bounds__(I4Cfg<H, RT>::WARPS * 32, 1) int4_attn_kernel(const I4Params p) {
  using C = I4Cfg<H, RT>;
  using L = I4<H>;
  constexpr int ROWS = C::ROWS, G = L::G, WPK = H / 32, VT = (RT + 1) / 2;  // WPK: words of a lane per key row; VT: n-tiles of weights
  extern __shared__ __align__(16) unsigned char i4_smem[];
  __shared__ int scan[3][C::WARPS], start_off[C::WARPS];
  __shared__ int start_b[C::WARPS];
  __shared__ int parked[C::WARPS][C::PARK ? 12 : 1];
  pdl_trigger();
  pdl_wait();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  // ---- how many segments, how many pages, how many at most in one
  const int per_thread = (p.c.B + blockDim.x - 1) / blockDim.x;
  const int b_lo = min((int)threadIdx.x * per_thread, p.c.B), b_hi = min(b_lo + per_thread, p.c.B);
  int segments = 0, all_pages = 0, most_pages = 0;
  for (int b = b_lo; b < b_hi; b++) {
    const I4Seq s = i4_seq(p, b, ROWS);
    segments += s.chunks * p.c.Nkv;
    all_pages += s.chunks * p.c.Nkv * s.pages;
    if (s.chunks) most_pages = max(most_pages, s.pages);
  }
  segments = __reduce_add_sync(0xffffffffu, segments);
  all_pages = __reduce_add_sync(0xffffffffu, all_pages);
  most_pages = __reduce_max_sync(0xffffffffu, most_pages);
  if (lane == 0) {
    scan[0][warp] = segments;
    scan[1][warp] = all_pages;
    scan[2][warp] = most_pages;
  }
  __syncthreads();
  segments = all_pages = most_pages = 0;
  for (int i = 0; i < C::WARPS; i++) {
    segments += scan[0][i];
    all_pages += scan[1][i];
    most_pages = max(most_pages, scan[2][i]);
  }
  // Warps work on segments of their own where there are segments enough and none is so long that adding up its parts would take
  // long: no warp waits for another. Else groups of four, or the whole block: its warps' results meet in shared memory.
  // Measured with 8 key heads of 128 (us for warps / fours / blocks): 16 sequences of 2048 (128 segments) 29.2 / 20.9 / 18.0, 19 of them (152) 29.8 / 21.6 / 26.2;
  // 100 of 200 to 900: 27.2 / 29.6 / 42.2; 64 of 2000: 44.9 / 43.0 / 51.6; 64 of up to 4096, 64 query heads: 50.9 / 30.0 / 46.7; 39 of up to 100 beside one of
  // 100000: 176 / 47.1 / 46.2. Half of both limits takes 49.5 instead of 32.4 us for the 64 of up to 4096, twice both 30.0 instead of 22.5 for the 19
  const int even = (all_pages + (int)gridDim.x * C::WARPS - 1) / ((int)gridDim.x * C::WARPS);  // pages per warp
  const bool many = segments >= (int)gridDim.x;
  const int gsh = !many ? C::WARP_SHIFT : most_pages <= 8 * even ? 0 : most_pages <= 64 * even ? 2 : C::WARP_SHIFT, GW = 1 << gsh;
  const int grp = warp >> gsh, w = warp & (GW - 1), gtid = threadIdx.x - grp * GW * 32;
  const int workers = (int)gridDim.x * (C::WARPS >> gsh), me = (int)blockIdx.x * (C::WARPS >> gsh) + grp;
  auto group_sync = [&]() {
    if (GW == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "r"(GW * 32) : "memory");
  };

  // ---- the units of all segments, and this group's share of them
  auto quanta_of = [&](int pages) { return (pages + GW - 1) >> gsh; };
  int mine[2] = {0, 0};  // in quanta, in pieces of four
  for (int b = b_lo; b < b_hi; b++) {
    const I4Seq s = i4_seq(p, b, ROWS);
    const int n = s.chunks * p.c.Nkv, quanta = quanta_of(s.pages);
    mine[0] += n * (quanta + kI4Start);
    mine[1] += n * ((quanta + (1 << kI4PieceShift) - 1) >> kI4PieceShift);
  }
  int incl[2] = {mine[0], mine[1]};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int v = __shfl_up_sync(0xffffffffu, incl[k], o);
      if (lane >= o) incl[k] += v;
    }
  }
  __syncthreads();
  if (lane == 31) {
    scan[0][warp] = incl[0];
    scan[1][warp] = incl[1];
  }
  __syncthreads();
  int before[2] = {0, 0}, totals[2] = {0, 0};
  for (int i = 0; i < C::WARPS; i++) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
      if (i < warp) before[k] += scan[k][i];
      totals[k] += scan[k][i];
    }
  }
  const bool few = totals[1] <= workers;
  // Segments lie end to end in units: pieces of four quanta, or single quanta behind kI4Start units for what a run costs besides
  auto units_of = [&](int quanta) { return few ? (quanta + (1 << kI4PieceShift) - 1) >> kI4PieceShift : quanta + kI4Start; };
  auto quantum_at = [&](int unit, int quanta) { return min(few ? unit << kI4PieceShift : max(unit - kI4Start, 0), quanta); };
  const int start = few ? 0 : kI4Start;
  const int total = few ? totals[1] : totals[0], held_here = few ? mine[1] : mine[0], excl = few ? before[1] + incl[1] - mine[1] : before[0] + incl[0] - mine[0];
  const int per = (total + workers - 1) / workers;
  // where each group starts: the thread whose sequences hold that unit says so
  for (int k = 0; k < C::WARPS >> gsh; k++) {
    const int s0 = ((int)blockIdx.x * (C::WARPS >> gsh) + k) * per;
    if (s0 < total && excl <= s0 && s0 < excl + held_here) {
      int acc = excl;
      for (int b = b_lo; b < b_hi; b++) {
        const I4Seq s = i4_seq(p, b, ROWS);
        const int n = units_of(quanta_of(s.pages)) * s.chunks * p.c.Nkv;
        if (s0 < acc + n) {
          start_b[k] = b;
          start_off[k] = s0 - acc;
          break;
        }
        acc += n;
      }
    }
  }
  __syncthreads();
  const int q0 = me * per, q1 = min(q0 + per, total);
  if (q0 >= q1) return;  // whole groups leave; what follows synchronises groups only

  // ---- the share as runs: parts of one segment each
  struct Run {
    int b, n, chunk, seg0;     // sequence (-1: none left), key head, row chunk, first unit of the segment
    int qi, qend, left;        // quanta of the segment, units of the share behind this run
    int keys, quanta, chunks;  // of the sequence
  };
  auto clip = [&](Run& r, int unit) {  // the run starts at that unit of the segment
    const int take = min(units_of(r.quanta) - unit, r.left);
    r.left -= take;
    r.qi = quantum_at(unit, r.quanta);
    r.qend = quantum_at(unit + take, r.quanta);
  };
  auto enter = [&](Run& r) {
    const I4Seq s = i4_seq(p, r.b, ROWS);
    r.keys = s.keys;
    r.quanta = quanta_of(s.pages);
    r.chunks = s.chunks;
  };
  auto next = [&](Run& r) {
    do {
      if (r.left == 0) {
        r.b = -1;
        return;
      }
      r.seg0 += units_of(r.quanta);
      if (++r.chunk == r.chunks) {
        r.chunk = 0;
        if (++r.n == p.c.Nkv) {
          r.n = 0;
          do {
            if (++r.b >= p.c.B) {
              r.b = -1;
              return;
            }
            enter(r);
          } while (r.quanta * r.chunks == 0);
        }
      }
      clip(r, 0);
    } while (r.qi == r.qend);
  };
  Run now;
  {
    now.b = start_b[grp];
    enter(now);
    const int units = units_of(now.quanta), at = start_off[grp], segment = at / units, unit = at % units;
    now.n = segment / now.chunks;
    now.chunk = segment % now.chunks;
    now.seg0 = q0 - unit;
    now.left = q1 - q0;
    clip(now, unit);
    if (now.qi == now.qend) next(now);
  }

  unsigned char* base = i4_smem + warp * C::WARP_BYTES;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(base);
  float* merge = reinterpret_cast<float*>(base + C::STAGES * L::BYTES);
  unsigned char* group_base = i4_smem + grp * GW * C::WARP_BYTES + C::STAGES * L::BYTES;

  // The table's entry for this warp's page of a run's quantum, asked for one round before it is needed (-1: no page)
  auto entry = [&](const Run& r) -> int {
    const int pg = r.qi * GW + w;
    return r.b >= 0 && pg * kI4Page < r.keys ? p.c.table[(int64_t)r.b * p.c.cols + pg] : -1;
  };
  // Fetches that page; the keys that it holds (0: no page)
  auto fetch = [&](const Run& r, int page, int stage) -> int {
    if ((unsigned)page >= (unsigned)p.c.pages) return 0;
    const uint8_t* src = p.c.pool + ((int64_t)page * p.c.Nkv + r.n) * L::BYTES + lane * 16;
    const uint32_t dst = ring + stage * L::BYTES + lane * 16;
#pragma unroll
    for (int k = 0; k < L::BYTES / 512; k++) i4_cp16(dst + k * 512, src + k * 512);
    if (L::BYTES % 512 && lane < L::BYTES % 512 / 16) i4_cp16(dst + L::BYTES / 512 * 512, src + L::BYTES / 512 * 512);
    return min(r.keys - (r.qi * GW + w) * kI4Page, kI4Page);
  };
  auto step = [&](Run& r) {
    if (r.b >= 0 && ++r.qi == r.qend) next(r);
  };

  Run ahead = now;
  int ahead_page = entry(ahead), held[2];
  static_assert(C::STAGES == 2, "held");
  {
    const Run first = ahead;
    const int first_page = ahead_page;
    step(ahead);
    ahead_page = entry(ahead);  // both entries are asked for before either is used
    held[0] = fetch(first, first_page, 0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    held[1] = fetch(ahead, ahead_page, 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    step(ahead);
    ahead_page = entry(ahead);
  }

  uint2 qf[C::TILES][WPK];
  float qsc[RT], qs[RT][G];                // per row: 2^-k scale log2(e), and sums of q times scale log2(e)
  float acc[VT][G][4][4], zacc[RT][G], m_run[RT], l_run[RT];
  float unit[RT][G];                       // acc holds sums times this power of two
  int klim[RT], klim_min = 0;
  const int kr = (g >> 1) + 4 * (g & 1);   // row g of a 16-row tile is key kr of its first 8, row g + 8 of its last 8

  int stage = 0;
  for (; now.b >= 0; next(now)) {
    int n_tok = i4_seq(p, now.b, ROWS).n, tok0 = p.cu ? min(max(p.cu[now.b], 0), p.T) : now.b;
    int w0 = (now.seg0 + start) / per, w1 = (now.seg0 + units_of(now.quanta) - 1) / per;  // the groups that share the segment
    unsigned long long word_was = 0;
    if (w0 != w1 && gtid == 0) word_was = *reinterpret_cast<volatile unsigned long long*>(p.counters + w0);
    {  // the segment's query rows, as digits, by the group together
      constexpr int LR = H / 8;  // lanes per row
      uint2* frag = reinterpret_cast<uint2*>(group_base);
      float4* info = reinterpret_cast<float4*>(group_base + C::TILES * WPK * 256);
      for (int r0 = w * (32 / LR); r0 < ROWS; r0 += GW * (32 / LR)) {
        const int r = r0 + lane / LR, u = lane % LR, row = now.chunk * ROWS + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < ROWS && row < n_tok * p.R)
          v = *reinterpret_cast<const uint4*>(p.q + (int64_t)(tok0 + row / p.R) * p.ldq + (int64_t)(now.n * p.R + row % p.R) * H + 8 * u);
        const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
        float x[8], top = 0.0f, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          x[2 * i] = __uint_as_float(vw[i] << 16);
          x[2 * i + 1] = __uint_as_float(vw[i] & 0xffff0000u);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x[i])));
          sum += x[i];
        }
#pragma unroll
        for (int o = LR / 2; o > 0; o >>= 1) {
          const float v2 = __shfl_xor_sync(0xffffffffu, top, o);
          asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(v2));
          if (o < 8) sum += __shfl_xor_sync(0xffffffffu, sum, o);  // within a group of 64
        }
        const float other = __shfl_xor_sync(0xffffffffu, sum, LR / 2);
        const int k = min(21 - ((int)((__float_as_uint(top) >> 23) & 255) - 127), 120);  // top * 2^k in [2^21, 2^22)
        const float up = i4_pow2(k), up16 = i4_pow2(k - 4);
        uint32_t d[3][2];  // digits: bytes of the factors of (byte & 15), of the whole byte
        {
          uint32_t e[4], f[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t Qo = __float_as_uint(fmaf(x[2 * i + 1], up16, __uint_as_float(kI4Magic)));
            const uint32_t Qe = __float_as_uint(fmaf(x[2 * i], up, __uint_as_float(kI4Magic)));
            // bytes 0..2 become signed digits, the lowest first
            e[i] = (Qe - Qo + 0x8080u) ^ 0x8080u;
            f[i] = (Qo - kI4Magic + 0x8080u) ^ 0x8080u;
          }
#pragma unroll
          for (int half = 0; half < 2; half++) {
            const uint32_t* b = half ? f : e;
            const uint32_t p01 = __byte_perm(b[0], b[1], 0x5140), p23 = __byte_perm(b[2], b[3], 0x5140);
            d[2][half] = __byte_perm(p01, p23, 0x5410);
            d[1][half] = __byte_perm(p01, p23, 0x7632);
            d[0][half] = __byte_perm(__byte_perm(b[0], b[1], 0x0062), __byte_perm(b[2], b[3], 0x0062), 0x5410);
          }
        }
        const float bad = top * 0.0f;  // a NaN where any value is not finite
        if (r < ROWS) {
          const int tile = r / 4, col = 2 * (r % 4), i = u / 4, tt = u % 4;
          frag[(tile * WPK + i) * 32 + col * 4 + tt] = make_uint2(d[0][0], d[0][1]);
          frag[(tile * WPK + i) * 32 + (col + 1) * 4 + tt] = make_uint2(d[1][0], d[1][1]);
          frag[((RT + tile / 2) * WPK + i) * 32 + (col + (tile & 1)) * 4 + tt] = make_uint2(d[2][0], d[2][1]);
          if (u == 0) info[r] = make_float4(i4_pow2(-k) * p.sc2 + bad, sum * p.sc2, G == 2 ? other * p.sc2 : 0.0f, 0.0f);
        }
      }
      group_sync();
#pragma unroll
      for (int i = 0; i < C::TILES; i++)
#pragma unroll
        for (int k = 0; k < WPK; k++) qf[i][k] = frag[(i * WPK + k) * 32 + lane];
      const long long cap = (long long)p.c.cols * kI4Page, first = max(p.c.lengths[now.b], 0);
#pragma unroll
      for (int j = 0; j < RT; j++) {
        const float4 f = info[4 * j + t];
        qsc[j] = f.x;
        qs[j][0] = f.y;
        if (G == 2) qs[j][G - 1] = f.z;
        // rows behind the last are computed with the last token's keys and not written
        const int tok = min((now.chunk * ROWS + 4 * j + t) / p.R, n_tok - 1);
        klim[j] = p.causal ? (int)min(cap, first + tok + 1) : now.keys;
        m_run[j] = -INFINITY;
        l_run[j] = 0.0f;
#pragma unroll
        for (int h = 0; h < G; h++) {
          zacc[j][h] = 0.0f;
          unit[j][h] = i4_pow2(126);
        }
      }
      klim_min = p.causal ? (int)min(cap, first + now.chunk * ROWS / p.R + 1) : now.keys;
#pragma unroll
      for (int v = 0; v < VT; v++)
#pragma unroll
        for (int h = 0; h < G; h++)
#pragma unroll
          for (int i = 0; i < 4; i++) acc[v][h][i][0] = acc[v][h][i][1] = acc[v][h][i][2] = acc[v][h][i][3] = 0.0f;
    }

    volatile int* const lot = parked[warp];
    if (C::PARK && lane == 0) {
      const int v[12] = {now.b, now.n, now.chunk, now.seg0, now.left, now.keys, now.quanta, now.chunks, tok0, n_tok, w0, w1};
#pragma unroll
      for (int i = 0; i < 12; i++) lot[i] = v[i];
    }
    for (; now.qi < now.qend; now.qi++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 1) : "memory");
    __syncwarp();
    const int have = held[0];
    if (have > 0) {
      const unsigned char* st = base + stage * L::BYTES;
      const int key0 = (now.qi * GW + w) * kI4Page;
      // ---- scores of 32 keys, in units of log2(e): x[row][tile of 16 keys][its first or last 8]
      float x[RT][2][2];
      uint32_t vparam[2][2][G];
#pragma unroll
      for (int m = 0; m < 2; m++) {
        uint32_t kw[2][WPK], kp[2][G];
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const int key = 16 * m + 8 * r + kr;
          i4_lds(st + L::KC + key * (H / 2) + t * (WPK * 4), kw[r]);
          i4_lds(st + L::KP + key * (G * 4), kp[r]);
          i4_lds(st + L::VP + key * (G * 4), vparam[m][r]);
        }
#pragma unroll
        for (int h = 0; h < G; h++) {
          int d[C::TILES][4];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const uint32_t a = kw[0][2 * h + i], b = kw[1][2 * h + i];
            const uint32_t a0 = a & 0x0f0f0f0fu, a1 = b & 0x0f0f0f0fu;
#pragma unroll
            for (int n = 0; n < C::TILES; n++) {
              if (i == 0) i4_mma_first(d[n], a0, a1, a, b, qf[n][2 * h]);
              else i4_mma_u8(d[n], a0, a1, a, b, qf[n][2 * h + 1]);
            }
          }
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const float s = __uint_as_float(kp[r][h] << 16), z = __uint_as_float(kp[r][h] & 0xffff0000u);
#pragma unroll
            for (int j = 0; j < RT; j++) {
              const float f = fmaf(fmaf(i4_count(d[j][2 * r]), 256.0f, i4_count(d[j][2 * r + 1])), 256.0f, i4_count(d[RT + j / 2][2 * r + (j & 1)]));
              x[j][m][r] = fmaf(s * qsc[j], f, h == 0 ? z * qs[j][0] : fmaf(z, qs[j][h], x[j][m][r]));
            }
          }
        }
      }
      bool odd = false;  // a key that some row sees and another does not has no finite value
      if (key0 + kI4Page > klim_min || have < kI4Page) {
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const int key = 16 * m + 8 * r + kr;
#pragma unroll
            for (int j = 0; j < RT; j++)
              if (key0 + key >= klim[j]) x[j][m][r] = -INFINITY;
#pragma unroll
            for (int h = 0; h < G; h++) {
              if (key >= have) vparam[m][r][h] = 0;  // places behind the last token may hold anything
              odd |= (vparam[m][r][h] & 0x7f800000u) == 0x7f800000u;
            }
          }
        odd = __any_sync(0xffffffffu, odd);
      }
      // ---- the running maximum is a reference that has to follow only when a score passes it by 2^8, a unit when a weight times a scale
      // may pass 2^15.9 of it: the leading bits of a positive float, as the mantissa of 256, are 256 + 127 + its log2, to 0.09 below. (The products
      // themselves, once rounded, as the test: 46.4 us for 44.0, 131072 tokens)
      bool pass = false;
      float top[RT], ref[RT];
      float size[G];
#pragma unroll
      for (int h = 0; h < G; h++)
        size[h] = __uint_as_float(0x43800000u | (__vmaxu2(__vmaxu2(vparam[0][0][h], vparam[0][1][h]), __vmaxu2(vparam[1][0][h], vparam[1][1][h])) & 0xffffu) << 8);
#pragma unroll
      for (int j = 0; j < RT; j++) {
        top[j] = fmaxf(fmaxf(x[j][0][0], x[j][0][1]), fmaxf(x[j][1][0], x[j][1][1]));
        const float over = top[j] - m_run[j];
        pass |= over > 8.0f;
#pragma unroll
        for (int h = 0; h < G; h++) pass |= over + size[h] > 2 * 383.0f + 15.8f - __uint_as_float(0x43800000u + (__float_as_uint(unit[j][h]) >> 8));
      }
      if (__any_sync(0xffffffffu, pass)) {
        float down[RT][G];
#pragma unroll
        for (int j = 0; j < RT; j++) {
          float v = top[j];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
          // a whole number: the sums change by powers of two, those of the values not at all, but for their units
          const float m_new = fmaxf(m_run[j], ceilf(v)), d = m_new == m_run[j] ? 0.0f : m_new - m_run[j];
          const float alpha = d <= 126.0f ? i4_pow2(-(int)d) : 0.0f, grow = i4_pow2((int)fminf(d, 126.0f)), r0 = m_new == -INFINITY ? 0.0f : m_new;
          m_run[j] = m_new;
          l_run[j] *= alpha;
#pragma unroll
          for (int h = 0; h < G; h++) {
            float most = 0.0f;  // the largest weight times scale; what is not finite has no say
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
              for (int r = 0; r < 2; r++) {
                const float w = i4_ex2(x[j][m][r] - r0) * __uint_as_float(vparam[m][r][h] << 16);
                most = w < INFINITY ? fmaxf(most, w) : most;
              }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            float u = d <= 126.0f ? fminf(unit[j][h] * grow, i4_pow2(126)) : i4_pow2(126);
            if (most * u >= 32768.0f) u = i4_pow2(6 + 127 - (int)(__float_as_uint(most) >> 23));  // it becomes 2^6 .. 2^7 units
            down[j][h] = u * alpha * i4_inverse(unit[j][h]);
            unit[j][h] = u;
            zacc[j][h] *= alpha;
          }
        }
#pragma unroll
        for (int v = 0; v < VT; v++)
#pragma unroll
          for (int h = 0; h < G; h++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
              for (int k = 0; k < 4; k++) acc[v][h][i][k] *= RT == 1 ? down[0][h] : down[2 * v + (k & 1)][h];
      }
#pragma unroll
      for (int j = 0; j < RT; j++) ref[j] = m_run[j] == -INFINITY ? 0.0f : m_run[j];
      // ---- weights, and values of 16 keys at a time
#pragma unroll
      for (int m = 0; m < 2; m++) {
        uint32_t pb[VT][RT == 1 ? 1 : G][2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
          float vs[G], z[G], ps[RT][G];  // ps: weight times scale, in its unit
#pragma unroll
          for (int h = 0; h < G; h++) {
            vs[h] = __uint_as_float(vparam[m][r][h] << 16);
            z[h] = fmaf(8.0f, vs[h], __uint_as_float(vparam[m][r][h] & 0xffff0000u));
          }
#pragma unroll
          for (int j = 0; j < RT; j++) {
            const float e = i4_ex2(x[j][m][r] - ref[j]);
            l_run[j] += e;
            if (odd && x[j][m][r] == -INFINITY) {  // what a row does not see leaves it alone
#pragma unroll
              for (int h = 0; h < G; h++) ps[j][h] = 0.0f;
            } else {
              i4_mul(ps[j], e, vs, unit[j]);
              i4_fma(zacc[j], e, z);
            }
          }
          if (RT == 1) {  // columns (row t, group): both groups' products share the operand
            pb[0][0][r] = i4_transpose(i4_pack_f16(ps[0][0], G == 2 ? ps[0][G - 1] : 0.0f));
          } else {        // columns (row t, row t + 4) of each group
#pragma unroll
            for (int v = 0; v < VT; v++)
#pragma unroll
              for (int h = 0; h < G; h++) pb[v][RT == 1 ? 0 : h][r] = i4_transpose(i4_pack_f16(ps[RT == 1 ? 0 : 2 * v][h], ps[RT == 1 ? 0 : 2 * v + 1][h]));
          }
        }
        uint32_t va[2 * G], vb[2 * G];  // [key t, key t + 4][group] of the first and the last 8 keys
        i4_lds(st + L::VC + (((2 * m) * 8 + g) * 4 + t) * (8 * G), va);
        i4_lds(st + L::VC + (((2 * m + 1) * 8 + g) * 4 + t) * (8 * G), vb);
#pragma unroll
        for (int h = 0; h < G; h++) {
          // low halves: dimensions 64 h + 8 g + 0..3 of the keys t and t + 4, high halves: + 4..7
          const uint32_t xa = __byte_perm(va[h], va[G + h], 0x5410), ya = __byte_perm(va[h], va[G + h], 0x7632);
          const uint32_t xb = __byte_perm(vb[h], vb[G + h], 0x5410), yb = __byte_perm(vb[h], vb[G + h], 0x7632);
          uint32_t f[2][8];  // [codes 2 i + 1 with 2 i, codes 2 i alone]: i = 0, 1
          i4_centred<0>(xa, f[1][0], f[0][0]);
          i4_centred<0>(ya, f[1][1], f[0][1]);
          i4_centred<0>(xb, f[1][2], f[0][2]);
          i4_centred<0>(yb, f[1][3], f[0][3]);
          i4_centred<1>(xa, f[1][4], f[0][4]);
          i4_centred<1>(ya, f[1][5], f[0][5]);
          i4_centred<1>(xb, f[1][6], f[0][6]);
          i4_centred<1>(yb, f[1][7], f[0][7]);
#pragma unroll
          for (int v = 0; v < VT; v++) {
            const uint32_t(&b)[2] = pb[v][RT == 1 ? 0 : h];
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t* a = &f[i & 1][(i >> 1) * 4];
              i4_mma_f16(acc[v][h][i], a[0], a[1], a[2], a[3], b[0], b[1]);
            }
          }
        }
      }
    }
    __syncwarp();  // the stage has been read by every lane
    held[0] = held[1];
    held[1] = fetch(ahead, ahead_page, stage);
    asm volatile("cp.async.commit_group;" ::: "memory");
    step(ahead);
    ahead_page = entry(ahead);
    stage ^= 1;
    }

    // ---- the run's end: rows of (maximum, sum, output); a lane has 8 dimensions 64 h + 8 g + .. of the rows 4 j + t
    if (C::PARK) {
      __syncwarp();
      now = Run{lot[0], lot[1], lot[2], lot[3], now.qi, now.qend, lot[4], lot[5], lot[6], lot[7]};
      tok0 = lot[8], n_tok = lot[9], w0 = lot[10], w1 = lot[11];
    }
    const bool whole = w0 == w1;
    const int rows = min(ROWS, n_tok * p.R - now.chunk * ROWS);
    // A part is [RT][G][2][32 lanes] float4 as the lanes have them, then maxima and sums; one of a share's first, one of its last segment
    auto part_of = [&](int k) { return p.part + ((int64_t)k * 2 + (now.seg0 + start < k * per ? 0 : 1)) * ROWS * (H + 2); };
    auto row_out = [&](int r) {
      const int row = now.chunk * ROWS + r;
      return p.out + ((int64_t)(tok0 + row / p.R) * p.Nq + now.n * p.R + row % p.R) * H;
    };
    float o[RT][G][8];
    {
#pragma unroll
      for (int j = 0; j < RT; j++) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          l_run[j] += __shfl_xor_sync(0xffffffffu, l_run[j], k);
#pragma unroll
          for (int h = 0; h < G; h++) zacc[j][h] += __shfl_xor_sync(0xffffffffu, zacc[j][h], k);
        }
#pragma unroll
        for (int h = 0; h < G; h++)
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int c = i & 3, e = (RT == 1 ? h : j & 1) + 2 * (i >> 2);  // accumulators c odd hold 16 times their code's sum and that of c - 1
            const float sum = c & 1 ? (acc[j / 2][h][c][e] - acc[j / 2][h][c - 1][e]) * 0.0625f : acc[j / 2][h][c][e];
            o[j][h][i] = fmaf(sum, i4_inverse(unit[j][h]), zacc[j][h]);
          }
      }
    }
    auto write_out = [&]() {
#pragma unroll
      for (int j = 0; j < RT; j++) {
        if (4 * j + t >= rows) continue;
        const float inv = l_run[j] == 0.0f ? 0.0f : 1.0f / l_run[j];  // 0: no keys
        uint16_t* dst = row_out(4 * j + t);
#pragma unroll
        for (int h = 0; h < G; h++) {
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = i4_pack_bf16(o[j][h][2 * i] * inv, o[j][h][2 * i + 1] * inv);
          *reinterpret_cast<uint4*>(dst + 64 * h + 8 * g) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
    };
    if (GW == 1) {
      if (whole) {
        write_out();
      } else {
        float* part = part_of(me);
#pragma unroll
        for (int j = 0; j < RT; j++) {
#pragma unroll
          for (int h = 0; h < G; h++)
#pragma unroll
            for (int q = 0; q < 2; q++)
              reinterpret_cast<float4*>(part)[((j * G + h) * 2 + q) * 32 + lane] = make_float4(o[j][h][4 * q], o[j][h][4 * q + 1], o[j][h][4 * q + 2], o[j][h][4 * q + 3]);
          if (g == 0) {
            part[ROWS * H + 4 * j + t] = m_run[j];
            part[ROWS * H + ROWS + 4 * j + t] = l_run[j];
          }
        }
        __syncwarp();
        bool last = false;
        if (lane == 0) last = i4_arrive(p.counters + w0, word_was, p.nonce, (unsigned)(w1 - w0 + 1));
        last = __shfl_sync(0xffffffffu, (int)last, 0);
        __syncwarp();  // orders what lane 0 has acquired before the other lanes' reads; the shuffle orders no memory
        if (last) {
#pragma unroll
          for (int j = 0; j < RT; j++) {
            m_run[j] = -INFINITY;
            l_run[j] = 0.0f;
#pragma unroll
            for (int h = 0; h < G; h++)
#pragma unroll
              for (int i = 0; i < 8; i++) o[j][h][i] = 0.0f;
          }
#pragma unroll 2
          for (int k = w0; k <= w1; k++) {
            const float* from = part_of(k);
            float4 v[RT][G][2];
            float pm[RT], pl[RT];
#pragma unroll
            for (int j = 0; j < RT; j++) {
              pm[j] = __ldcg(from + ROWS * H + 4 * j + t);
              pl[j] = __ldcg(from + ROWS * H + ROWS + 4 * j + t);
#pragma unroll
              for (int h = 0; h < G; h++)
#pragma unroll
                for (int q = 0; q < 2; q++) v[j][h][q] = __ldcg(reinterpret_cast<const float4*>(from) + ((j * G + h) * 2 + q) * 32 + lane);
            }
#pragma unroll
            for (int j = 0; j < RT; j++) {
              if (pl[j] == 0.0f) continue;  // saw nothing of this row (scores that are all NaN leave the maximum behind, but a sum)
              const float m_new = fmaxf(m_run[j], pm[j]), fo = i4_ex2(m_run[j] - m_new), fn = i4_ex2(pm[j] - m_new);
              m_run[j] = m_new;
              l_run[j] = fmaf(l_run[j], fo, pl[j] * fn);
#pragma unroll
              for (int h = 0; h < G; h++)
#pragma unroll
                for (int q = 0; q < 2; q++) {
                  const float x4[4] = {v[j][h][q].x, v[j][h][q].y, v[j][h][q].z, v[j][h][q].w};
#pragma unroll
                  for (int i = 0; i < 4; i++) o[j][h][4 * q + i] = fmaf(o[j][h][4 * q + i], fo, x4[i] * fn);
                }
            }
          }
          write_out();
        }
      }
    } else {
      float* ml = merge + ROWS * C::PITCH;
      group_sync();  // the first warp's buffer has held the digits
#pragma unroll
      for (int j = 0; j < RT; j++) {
        const int r = 4 * j + t;
        if (r < rows) {
          if (g == 0) {
            ml[r] = m_run[j];
            ml[ROWS + r] = l_run[j];
          }
#pragma unroll
          for (int h = 0; h < G; h++)
#pragma unroll
            for (int q = 0; q < 2; q++)
              *reinterpret_cast<float4*>(merge + r * C::PITCH + 64 * h + 8 * g + 4 * q) =
                  make_float4(o[j][h][4 * q], o[j][h][4 * q + 1], o[j][h][4 * q + 2], o[j][h][4 * q + 3]);
        }
      }
      group_sync();
      float* part = part_of(me);
      auto store = [&](int r, int d, float l, const float4& v) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        *reinterpret_cast<uint2*>(row_out(r) + d) = make_uint2(i4_pack_bf16(v.x * inv, v.y * inv), i4_pack_bf16(v.z * inv, v.w * inv));
      };
      auto add = [&](float4& v, float fo, const float4& x, float fn) {
        v.x = fmaf(v.x, fo, x.x * fn);
        v.y = fmaf(v.y, fo, x.y * fn);
        v.z = fmaf(v.z, fo, x.z * fn);
        v.w = fmaf(v.w, fo, x.w * fn);
      };
      for (int e = gtid; e < ROWS * H / 4; e += GW * 32) {  // in the order of a part
        const int le = e & 31, q = (e >> 5) & 1, h = (e >> 6) % G, r = 4 * ((e >> 6) / G) + (le & 3), d = 64 * h + 8 * (le >> 2) + 4 * q;
        if (r >= rows) continue;
        float m = -INFINITY, l = 0.0f;
        for (int k = 0; k < GW; k++) m = fmaxf(m, reinterpret_cast<const float*>(group_base + k * C::WARP_BYTES)[ROWS * C::PITCH + r]);
        const float ref = m == -INFINITY ? 0.0f : m;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < GW; k++) {
          const float* from = reinterpret_cast<const float*>(group_base + k * C::WARP_BYTES);
          const float pm = from[ROWS * C::PITCH + r], pl = from[ROWS * C::PITCH + ROWS + r];
          if (pl == 0.0f) continue;  // a warp that saw nothing of this row
          const float f = i4_ex2(pm - ref);
          l = fmaf(pl, f, l);
          add(v, 1.0f, *reinterpret_cast<const float4*>(from + r * C::PITCH + d), f);
        }
        if (whole) {
          store(r, d, l, v);
        } else {
          reinterpret_cast<float4*>(part)[e] = v;
          if (d == 0) {
            part[ROWS * H + r] = m;
            part[ROWS * H + ROWS + r] = l;
          }
        }
      }
      if (!whole) {
        group_sync();
        int* flag = reinterpret_cast<int*>(group_base + (ROWS * C::PITCH + 2 * ROWS - 1) * 4);  // the last float of the first warp's buffer: read by now
        if (gtid == 0) *flag = i4_arrive(p.counters + w0, word_was, p.nonce, (unsigned)(w1 - w0 + 1));
        group_sync();
        if (*flag) {
          // the parts, by every thread of the group: a piece of four values each, or where there are more threads some of the parts each
          constexpr int ITEMS = ROWS * H / 4;
          const int splits = max(GW * 32 / ITEMS, 1), first = gtid / ITEMS;
          for (int e = gtid % ITEMS; e < ITEMS; e += GW * 32) {
            const int le = e & 31, q = (e >> 5) & 1, h = (e >> 6) % G, r = 4 * ((e >> 6) / G) + (le & 3), d = 64 * h + 8 * (le >> 2) + 4 * q;
            float m = -INFINITY, l = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            constexpr int U = 8;  // parts whose loads are in flight together
            for (int k0 = w0 + first; k0 <= w1; k0 += U * splits) {
              float pm[U], pl[U];
              float4 x[U];
#pragma unroll
              for (int k = 0; k < U; k++) {
                const float* from = part_of(min(k0 + k * splits, w1));
                pm[k] = __ldcg(from + ROWS * H + r);
                pl[k] = __ldcg(from + ROWS * H + ROWS + r);
                x[k] = __ldcg(reinterpret_cast<const float4*>(from) + e);
              }
#pragma unroll
              for (int k = 0; k < U; k++) {
                if (k0 + k * splits > w1 || pl[k] == 0.0f) continue;
                const float m_new = fmaxf(m, pm[k]), fo = i4_ex2(m - m_new), fn = i4_ex2(pm[k] - m_new);
                m = m_new;
                l = fmaf(l, fo, pl[k] * fn);
                add(v, fo, x[k], fn);
              }
            }
            if (splits > 1) {  // once around this loop: every thread has one item
              float* mine_of = merge + lane * 6;
              if (first > 0) {
                mine_of[0] = m; mine_of[1] = l; mine_of[2] = v.x; mine_of[3] = v.y; mine_of[4] = v.z; mine_of[5] = v.w;
              }
              group_sync();
              if (first > 0) break;
              for (int k = 1; k < splits; k++) {
                const float* from = reinterpret_cast<const float*>(group_base + (w + k * (ITEMS / 32)) * C::WARP_BYTES) + lane * 6;
                if (from[1] == 0.0f) continue;
                const float m_new = fmaxf(m, from[0]), fo = i4_ex2(m - m_new), fn = i4_ex2(from[0] - m_new);
                m = m_new;
                l = fmaf(l, fo, from[1] * fn);
                add(v, fo, make_float4(from[2], from[3], from[4], from[5]), fn);
              }
            }
            if (r < rows) store(r, d, l, v);
          }
        }
      }
    }
    group_sync();  // the buffers are free again
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---------------------------------------------------------------- host side
// Query rows per lane: chunks of 4, 8 or 16 rows, the least that holds a sequence's rows if all have as many tokens (the lengths are on the device; a
// sequence of more rows has more chunks). With 1, 2, 4 rows per lane, us: 16 sequences of 2048, 4 rows each: 19.1 / 23.9 / 33.4; 64 of up to 4096, 8 rows:
// 35.1 / 32.3 / 41.0; 8 of up to 1500 with five tokens and 20 rows: 18.8 / 24.4 / 20.2
static int i4_rows(int64_t T, int64_t B, int64_t Nq, int64_t Nkv) {
  const int64_t rows = (T + B - 1) / B * (Nq / Nkv);
  return rows <= 4 ? 1 : rows <= 8 ? 2 : 4;
}
static size_t i4_scratch(int rt, int64_t H) { return (size_t)sm_count() * kI4Warps * (8 + 2 * (size_t)(4 * rt) * (H + 2) * 4); }

template <int H, int RT>
static int i4_launch(I4Params& p, cudaStream_t st) {
  using C = I4Cfg<H, RT>;
  static bool opted[16] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16 || !opted[dev]) {
    TPX_CUDA_OK(cudaFuncSetAttribute(int4_attn_kernel<H, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    if (dev >= 0 && dev < 16) opted[dev] = true;
  }
  const int64_t most = ((int64_t)p.T * p.R / C::ROWS + p.c.B) * p.c.Nkv * (p.c.cols + C::WARPS);
  TPX_REQUIRE(most < (1ll << 31), TPX_ERR_UNSUPPORTED, "int4_attention: more than 2^31 pages may be walked in one call");
  TPX_CUDA_OK(launch_pdl(int4_attn_kernel<H, RT>, dim3(sm_count()), dim3(C::WARPS * 32), C::SMEM, st, p));
  return TPX_OK;
}

}  // namespace tpx

using namespace tpx;

extern "C" size_t tpx_int4_attention_scratch_bytes(int64_t T, int64_t B, int64_t Nq, int64_t kv_heads, int64_t H) {
  if (T <= 0 || B <= 0 || kv_heads <= 0 || Nq <= 0) return 0;
  return i4_scratch(i4_rows(T, B, Nq, kv_heads), H);
}

static int int4_attention(const TpxInt4Attention* a, int behind, void* stream) {
  TPX_REQUIRE(a && a->cache && (a->T == 0 || (a->q && a->out)), TPX_ERR_ARG, "int4_attention: null pointer");
  I4Params p = {};
  const int rc = i4_cache_of(a->cache, &p.c);
  if (rc) return rc;
  const int64_t H = a->cache->H, Nkv = a->cache->kv_heads;
  TPX_REQUIRE(a->T >= 0 && a->T < (1ll << 31) / 4096 && (a->cu_seqlens || a->T == a->cache->B), TPX_ERR_ARG, "int4_attention: %ld tokens for %ld sequences", (long)a->T,
              (long)a->cache->B);
  TPX_REQUIRE(a->Nq > 0 && a->Nq <= 4096 && a->Nq % Nkv == 0, TPX_ERR_ARG, "int4_attention: %ld query heads for %ld key heads", (long)a->Nq, (long)Nkv);
  TPX_REQUIRE((((uintptr_t)a->q | (uintptr_t)a->out) & 15) == 0 && a->ldq % 8 == 0, TPX_ERR_ARG, "int4_attention: q, its rows and out must be 16-byte aligned");
  TPX_REQUIRE(a->scale - a->scale == 0.0f, TPX_ERR_ARG, "int4_attention: a scale of %g", (double)a->scale);
  if (a->T == 0) return TPX_OK;
  const int rt = i4_rows(a->T, a->cache->B, a->Nq, Nkv);
  TPX_REQUIRE(a->scratch && ((uintptr_t)a->scratch & 255) == 0 && a->scratch_bytes >= i4_scratch(rt, H), TPX_ERR_SCRATCH,
              "int4_attention: scratch of %zu bytes, %zu are needed (256-byte aligned)", a->scratch_bytes, i4_scratch(rt, H));
  // a number of its own for every call: 48 bits, from an origin that differs between processes
  static unsigned long long calls = 0;
  static const unsigned long long origin = (unsigned long long)(uintptr_t)&calls * 0x9E3779B97F4A7C15ull;
  p.nonce = ((origin >> 16) + __atomic_add_fetch(&calls, 1ull, __ATOMIC_RELAXED)) << 16;
  if (p.nonce == 0) p.nonce = 1ull << 16;
  p.q = a->q;
  p.out = a->out;
  p.cu = a->cu_seqlens;
  p.counters = (unsigned long long*)a->scratch;
  p.part = (float*)((char*)a->scratch + (size_t)sm_count() * kI4Warps * 8);
  p.ldq = a->ldq;
  p.T = (int)a->T;
  p.Nq = (int)a->Nq;
  p.R = (int)(a->Nq / Nkv);
  p.causal = a->causal;
  p.behind = behind;
  p.sc2 = a->scale * 1.4426950408889634f;
  cudaStream_t st = (cudaStream_t)stream;
  if (H == 128) return rt == 1 ? i4_launch<128, 1>(p, st) : rt == 2 ? i4_launch<128, 2>(p, st) : i4_launch<128, 4>(p, st);
  return rt == 1 ? i4_launch<64, 1>(p, st) : rt == 2 ? i4_launch<64, 2>(p, st) : i4_launch<64, 4>(p, st);
}

extern "C" int tpx_int4_attention(const TpxInt4Attention* a, void* stream) { return int4_attention(a, 0, stream); }
extern "C" int tpx_int4_attention_behind(const TpxInt4Attention* a, void* stream) { return int4_attention(a, 1, stream); }
