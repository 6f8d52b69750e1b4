// Attention of a few new tokens per sequence over the 4-bit cache of tpx_packed.h.
//
//   out = softmax(scale * q K^T) V,   K[t][d] = kz + ks * kc[t][d],  V alike, with codes 0..15 and a scale and a minimum per 64 values
//
// Codes go to the matrix instructions as they are, scales and minima around them, so that a value costs an AND-OR (and a shift):
//   q.K  = sum over groups of 64:  ks (q . (16 + kc)) + (kz - 16 ks) sum(q)    16 + code is a bf16 with the code as its mantissa
//   P V  = sum over t: (p vs) (vc - 8) + p (vz + 8 vs)                          codes are centred: p vs is rounded to bf16, and that
//                                                                              rounding should not be weighed with the range's offset
// mma.sync m16n8k16 with the cache as the 16-row operand and the query rows ((token, group member) pairs of one key head) as its 8
// columns: at most 8 or 16 rows share one pass over the keys (tcgen05 has no form this narrow: it would need 128 of either). Keys: M is
// 16 tokens. Values: M is 16 of the head's dimensions, K 16 tokens; the weights get there by movmatrix.
//
// A page of a head (4608 bytes at H = 128) is one warp's work item, fetched by cp.async into a ring of the warp's own: no barrier in the
// loop. The (sequence, key head, row chunk) segments, each rounded up to whole quanta of GW pages (GW warps work on one segment at a
// time), are laid end to end and cut evenly between all groups of GW warps of the GPU, whatever the sequences' lengths, which are read
// on the device. A segment that is cut leaves partial results in scratch, which the group that finishes it last adds up in the order of
// the pieces: results do not depend on who is last. Arrivals are counted in words that carry the call's own number, so that scratch may
// hold anything before, and calls share none.
#include "tpx_int4.cuh"

namespace tpx {

constexpr int kI4Warps = 16;

struct I4Params {
  const uint16_t* q;
  uint16_t* out;
  const int32_t* cu;
  I4Cache c;
  float* part;                  // [workers][2][ROWS][H + 2]: maximum, sum, output of each row
  unsigned long long* counters;  // [workers]
  unsigned long long nonce;     // low 16 bits zero
  int64_t ldq;
  int T, Nq, R, GW, causal;
  float sc2;                    // scale * log2(e)
};

__device__ __forceinline__ void i4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
__device__ __forceinline__ uint32_t i4_pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Codes j and j + 4 of a word as bf16 pairs: 16 + code, or code - 8
template <int J>
__device__ __forceinline__ uint32_t i4_plus16(uint32_t w) {
  const uint32_t s = J == 0 ? w << 3 : w >> (4 * J - 3);
  return (s & 0x00780078u) | 0x41804180u;
}
template <int J>
__device__ __forceinline__ uint32_t i4_minus8(uint32_t w) {
  const uint32_t v = ((w >> (4 * J)) & 0x000f000fu) | 0x43004300u;  // 128 + code
  const uint32_t off = 0x43084308u;                                  // 136
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void i4_cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void i4_lds(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
}
__device__ __forceinline__ void i4_lds(uint32_t a, uint32_t (&v)[2]) {
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a));
}
__device__ __forceinline__ void i4_lds(uint32_t a, uint32_t (&v)[1]) { asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(a)); }

// Work of one sequence
struct I4Seq {
  int n, keys, quanta, chunks;  // tokens of the call, keys, quanta of a segment, row chunks
};
__device__ __forceinline__ I4Seq i4_seq(const I4Params& p, int b, int rows) {
  I4Seq s;
  if (p.cu) {
    const int lo = min(max(p.cu[b], 0), p.T), hi = min(max(p.cu[b + 1], 0), p.T);
    s.n = max(hi - lo, 0);
  } else {
    s.n = 1;
  }
  const long long keys = (long long)max(p.c.lengths[b], 0) + s.n, cap = (long long)p.c.cols * kI4Page;
  s.keys = (int)min(keys, cap);
  s.quanta = ((s.keys + kI4Page - 1) / kI4Page + p.GW - 1) / p.GW;
  s.chunks = (int)(((long long)s.n * p.R + rows - 1) / rows);
  return s;
}

template <int H, int NT>
struct I4Cfg {
  static constexpr int ROWS = 8 * NT;
  static constexpr int STAGES = 2;
  static constexpr int WARPS = NT == 1 ? kI4Warps : kI4Warps / 2;
  static constexpr int PITCH = H + 4;                     // floats of a row in the merge buffer
  static constexpr int MERGE = (ROWS * PITCH + 2 * ROWS) * 4;
  static constexpr int WARP_BYTES = STAGES * I4<H>::BYTES + MERGE;
  static constexpr int SMEM = WARPS * WARP_BYTES;
};

template <int H, int NT>
__global__ void __launch_bounds__(I4Cfg<H, NT>::WARPS * 32, 1) int4_attn_kernel(const I4Params p) {
  using C = I4Cfg<H, NT>;
  using L = I4<H>;
  constexpr int ROWS = C::ROWS, G = L::G, WPK = H / 32;  // WPK: words of a lane per key row
  extern __shared__ __align__(16) unsigned char i4_smem[];
  __shared__ long long scan[C::WARPS + 1];
  __shared__ int start_b;
  __shared__ long long start_off;
  pdl_trigger();
  pdl_wait();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int GW = p.GW, grp = warp / GW, w = warp % GW, gtid = threadIdx.x - grp * GW * 32;
  const long long workers = (long long)gridDim.x * (C::WARPS / GW), me = (long long)blockIdx.x * (C::WARPS / GW) + grp;
  auto group_sync = [&]() {
    if (GW == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "r"(GW * 32) : "memory");
  };

  // ---- the quanta of all segments, and this group's share of them
  long long total;
  const int per_thread = (p.c.B + blockDim.x - 1) / blockDim.x;
  const int b_lo = min((int)threadIdx.x * per_thread, p.c.B), b_hi = min(b_lo + per_thread, p.c.B);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; b++) {
    const I4Seq s = i4_seq(p, b, ROWS);
    mine += (long long)s.quanta * s.chunks * p.c.Nkv;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) scan[warp + 1] = incl;
  if (threadIdx.x == 0) scan[0] = 0;
  __syncthreads();
  long long before = 0;
  total = 0;
  for (int i = 0; i < C::WARPS; i++) {
    if (i < warp) before += scan[i + 1];
    total += scan[i + 1];
  }
  const long long excl = before + incl - mine;
  const long long per = (total + workers - 1) / workers;
  // where each group starts: the thread whose sequences hold that quantum says so, one group after the other
  long long q0 = 0, q1 = 0, at = 0;
  int b0 = 0;
  for (int k = 0; k < C::WARPS / GW; k++) {
    const long long s0 = ((long long)blockIdx.x * (C::WARPS / GW) + k) * per, s1 = min(s0 + per, total);
    __syncthreads();
    if (s0 < s1 && excl <= s0 && s0 < excl + mine) {
      long long acc = excl;
      for (int b = b_lo; b < b_hi; b++) {
        const I4Seq s = i4_seq(p, b, ROWS);
        const long long n = (long long)s.quanta * s.chunks * p.c.Nkv;
        if (s0 < acc + n) {
          start_b = b;
          start_off = s0 - acc;
          break;
        }
        acc += n;
      }
    }
    __syncthreads();
    if (k == grp) {
      q0 = s0;
      q1 = s1;
      b0 = start_b;
      at = start_off;
    }
  }
  if (q0 >= q1) return;  // whole groups leave; what follows synchronises groups only

  // ---- iterators over the quanta of the share
  struct Iter {
    int b, n, chunk, qi;  // sequence, key head, row chunk, quantum of the segment
    I4Seq s;
  };
  auto begin = [&]() {
    Iter i;
    i.b = b0;
    i.s = i4_seq(p, b0, ROWS);
    const long long per_head = (long long)i.s.quanta * i.s.chunks;
    i.n = (int)(at / per_head);
    const int r = (int)(at % per_head);
    i.chunk = r / i.s.quanta;
    i.qi = r % i.s.quanta;
    return i;
  };
  auto advance = [&](Iter& i) {  // only while quanta are left
    if (++i.qi < i.s.quanta) return;
    i.qi = 0;
    if (++i.chunk < i.s.chunks) return;
    i.chunk = 0;
    if (++i.n < p.c.Nkv) return;
    i.n = 0;
    do {
      i.b++;
      if (i.b >= p.c.B) return;
      i.s = i4_seq(p, i.b, ROWS);
    } while (i.s.quanta * i.s.chunks == 0);
  };

  unsigned char* base = i4_smem + warp * C::WARP_BYTES;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(base);
  float* merge = reinterpret_cast<float*>(base + C::STAGES * L::BYTES);
  unsigned char* group_base = i4_smem + grp * GW * C::WARP_BYTES + C::STAGES * L::BYTES;

  // Fetches this warp's page of the iterator's quantum; the keys that it holds (0: no page)
  auto fetch = [&](const Iter& i, int stage) -> int {
    const int pg = i.qi * GW + w;
    int live = i.s.keys - pg * kI4Page;
    if (live > 0) {
      const int page = p.c.table[(int64_t)i.b * p.c.cols + pg];
      if (page >= 0 && page < p.c.pages) {
        const uint8_t* src = p.c.pool + ((int64_t)page * p.c.Nkv + i.n) * L::BYTES + lane * 16;
        const uint32_t dst = ring + stage * L::BYTES + lane * 16;
#pragma unroll
        for (int k = 0; k < L::BYTES / 512; k++) i4_cp16(dst + k * 512, src + k * 512);
        if (L::BYTES % 512 && lane < L::BYTES % 512 / 16) i4_cp16(dst + L::BYTES / 512 * 512, src + L::BYTES / 512 * 512);
      } else {
        live = 0;
      }
    }
    return min(max(live, 0), kI4Page);
  };

  Iter ahead = begin(), now = ahead;
  long long qa = q0;
  int held[C::STAGES];
#pragma unroll
  for (int s = 0; s < C::STAGES; s++) {
    held[s] = 0;
    if (qa < q1) {
      held[s] = fetch(ahead, s);
      if (++qa < q1) advance(ahead);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  uint32_t qf[NT][WPK][4];
  float qs[NT][G][2];                        // sums of q over each group, rows 2t and 2t + 1
  float acc[NT][G][4][4], zacc[NT][G][2], m_run[NT][2], l_run[NT][2];
  int klim[NT][2], klim_min = 0;
  bool fresh = true;

  for (long long qc = q0; qc < q1; qc++) {
    const int stage = (int)((qc - q0) % C::STAGES);
    if (fresh) {  // a new segment: its query rows
      fresh = false;
      const int tok0 = p.cu ? min(max(p.cu[now.b], 0), p.T) : now.b;
      const long long cap = (long long)p.c.cols * kI4Page, first = max(p.c.lengths[now.b], 0);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        const int row = now.chunk * ROWS + nt * 8 + g;
        const bool live = row < now.s.n * p.R;
        const uint16_t* src = p.q + (int64_t)(tok0 + (live ? row / p.R : 0)) * p.ldq + (int64_t)(now.n * p.R + (live ? row % p.R : 0)) * H;
        float sum[G];
#pragma unroll
        for (int h = 0; h < G; h++) sum[h] = 0.0f;
#pragma unroll
        for (int i = 0; i < WPK; i++) {
          const uint4 v = live ? *reinterpret_cast<const uint4*>(src + 32 * i + 8 * t) : make_uint4(0, 0, 0, 0);
          qf[nt][i][0] = __byte_perm(v.x, v.z, 0x5410);  // values 0 and 4 of the lane's 8
          qf[nt][i][1] = __byte_perm(v.x, v.z, 0x7632);  // 1 and 5
          qf[nt][i][2] = __byte_perm(v.y, v.w, 0x5410);
          qf[nt][i][3] = __byte_perm(v.y, v.w, 0x7632);
#pragma unroll
          for (int j = 0; j < 4; j++) sum[i / 2] += __uint_as_float(qf[nt][i][j] << 16) + __uint_as_float(qf[nt][i][j] & 0xffff0000u);
        }
#pragma unroll
        for (int h = 0; h < G; h++) {
          float s = sum[h];
          s += __shfl_xor_sync(0xffffffffu, s, 1);
          s += __shfl_xor_sync(0xffffffffu, s, 2);
          qs[nt][h][0] = __shfl_sync(0xffffffffu, s, 8 * t);
          qs[nt][h][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
          zacc[nt][h][0] = zacc[nt][h][1] = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; i++) acc[nt][h][i][0] = acc[nt][h][i][1] = acc[nt][h][i][2] = acc[nt][h][i][3] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
          // rows behind the last are computed with the last token's keys and not written
          const int tok = min((now.chunk * ROWS + nt * 8 + 2 * t + e) / p.R, now.s.n - 1);
          klim[nt][e] = p.causal ? (int)min(cap, first + tok + 1) : now.s.keys;
          m_run[nt][e] = -INFINITY;
          l_run[nt][e] = 0.0f;
        }
      }
      klim_min = p.causal ? (int)min(cap, first + now.chunk * ROWS / p.R + 1) : now.s.keys;
    }

    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 1) : "memory");
    __syncwarp();
    const int have = held[0];
    if (have > 0) {
      const uint32_t st = ring + stage * L::BYTES;
      const int key0 = (now.qi * GW + w) * kI4Page;
      // ---- scores of 32 keys: rows of two m16 tiles; row i of a tile is key i / 2 + 4 (i % 2) of its first 8, then of its last 8
      float x[NT][2][4];
      uint32_t vparam[2][2][G];
      const int kr = (g >> 1) + 4 * (g & 1);
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
        for (int nt = 0; nt < NT; nt++) x[nt][m][0] = x[nt][m][1] = x[nt][m][2] = x[nt][m][3] = 0.0f;
#pragma unroll
        for (int h = 0; h < G; h++) {
          float d[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; nt++) d[nt][0] = d[nt][1] = d[nt][2] = d[nt][3] = 0.0f;
#pragma unroll
          for (int i = 2 * h; i < 2 * h + 2; i++) {
            const uint32_t a = kw[0][i], b = kw[1][i];
            const uint32_t f[8] = {i4_plus16<0>(a), i4_plus16<0>(b), i4_plus16<1>(a), i4_plus16<1>(b),
                                   i4_plus16<2>(a), i4_plus16<2>(b), i4_plus16<3>(a), i4_plus16<3>(b)};
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              i4_mma(d[nt], f[0], f[1], f[2], f[3], qf[nt][i][0], qf[nt][i][1]);
              i4_mma(d[nt], f[4], f[5], f[6], f[7], qf[nt][i][2], qf[nt][i][3]);
            }
          }
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const float s = __uint_as_float(kp[r][h] << 16), z = fmaf(-16.0f, s, __uint_as_float(kp[r][h] & 0xffff0000u));
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
              for (int e = 0; e < 2; e++) x[nt][m][2 * r + e] = fmaf(s, d[nt][2 * r + e], fmaf(z, qs[nt][h][e], x[nt][m][2 * r + e]));
          }
        }
      }
      const bool edge = key0 + kI4Page > klim_min || have < kI4Page;
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            x[nt][m][i] *= p.sc2;
            if (edge && key0 + 16 * m + 8 * (i >> 1) + kr >= klim[nt][i & 1]) x[nt][m][i] = -INFINITY;
          }
      // ---- the running maximum is a reference that has to follow only when a score passes it by 2^8
      bool pass = false;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          top[nt][e] = fmaxf(fmaxf(x[nt][0][e], x[nt][0][2 + e]), fmaxf(x[nt][1][e], x[nt][1][2 + e]));
          pass |= top[nt][e] > m_run[nt][e] + 8.0f;
        }
      if (__any_sync(0xffffffffu, pass)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float v = top[nt][e];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
            const float m_new = fmaxf(m_run[nt][e], v);
            const float alpha = m_new == m_run[nt][e] ? 1.0f : i4_ex2(m_run[nt][e] - m_new);
            m_run[nt][e] = m_new;
            l_run[nt][e] *= alpha;
#pragma unroll
            for (int h = 0; h < G; h++) {
              zacc[nt][h][e] *= alpha;
#pragma unroll
              for (int i = 0; i < 4; i++) {
                acc[nt][h][i][e] *= alpha;
                acc[nt][h][i][2 + e] *= alpha;
              }
            }
          }
      }
      // ---- weights, and values of 16 keys at a time
#pragma unroll
      for (int m = 0; m < 2; m++) {
        uint32_t pb[NT][G][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float e4[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float ref = m_run[nt][i & 1];
            e4[i] = ref == -INFINITY ? 0.0f : i4_ex2(x[nt][m][i] - ref);
            l_run[nt][i & 1] += e4[i];
          }
#pragma unroll
          for (int h = 0; h < G; h++) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
              const float s = __uint_as_float(vparam[m][r][h] << 16), z = fmaf(8.0f, s, __uint_as_float(vparam[m][r][h] & 0xffff0000u));
              float a = e4[2 * r] * s, b = e4[2 * r + 1] * s, za = e4[2 * r] * z, zb = e4[2 * r + 1] * z;
              if (edge) {  // what a row does not see leaves it alone, whatever it is
                if (x[nt][m][2 * r] == -INFINITY) a = za = 0.0f;
                if (x[nt][m][2 * r + 1] == -INFINITY) b = zb = 0.0f;
              }
              zacc[nt][h][0] += za;
              zacc[nt][h][1] += zb;
              pb[nt][h][r] = i4_transpose(i4_pack(a, b));
            }
          }
        }
        uint32_t va[2 * G], vb[2 * G];  // [key t, key t + 4][group] of the first and the last 8 keys
        i4_lds(st + L::VC + (((2 * m) * 8 + g) * 4 + t) * (8 * G), va);
        i4_lds(st + L::VC + (((2 * m + 1) * 8 + g) * 4 + t) * (8 * G), vb);
#pragma unroll
        for (int h = 0; h < G; h++) {
          const uint32_t xa = __byte_perm(va[h], va[G + h], 0x5410), ya = __byte_perm(va[h], va[G + h], 0x7632);
          const uint32_t xb = __byte_perm(vb[h], vb[G + h], 0x5410), yb = __byte_perm(vb[h], vb[G + h], 0x7632);
#define TPX_I4_V(I)                                                                                                    \
  {                                                                                                                    \
    const uint32_t f0 = i4_minus8<I>(xa), f1 = i4_minus8<I>(ya), f2 = i4_minus8<I>(xb), f3 = i4_minus8<I>(yb);         \
    _Pragma("unroll") for (int nt = 0; nt < NT; nt++) i4_mma(acc[nt][h][I], f0, f1, f2, f3, pb[nt][h][0], pb[nt][h][1]); \
  }
          TPX_I4_V(0) TPX_I4_V(1) TPX_I4_V(2) TPX_I4_V(3)
#undef TPX_I4_V
        }
      }
    }
    __syncwarp();  // the stage has been read by every lane
#pragma unroll
    for (int s = 0; s + 1 < C::STAGES; s++) held[s] = held[s + 1];
    held[C::STAGES - 1] = 0;
    if (qa < q1) {
      held[C::STAGES - 1] = fetch(ahead, stage);
      if (++qa < q1) advance(ahead);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");

    const bool last_of_segment = now.qi + 1 == now.s.quanta;
    if (last_of_segment || qc + 1 == q1) {
      // ---- this group's part of the segment: rows of (maximum, sum, output), merged over its warps
      float* ml = merge + ROWS * C::PITCH;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float l = l_run[nt][e], z[G];
#pragma unroll
          for (int h = 0; h < G; h++) z[h] = zacc[nt][h][e];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
            for (int h = 0; h < G; h++) z[h] += __shfl_xor_sync(0xffffffffu, z[h], o);
          }
          const int r = nt * 8 + 2 * t + e;
          if (g == 0) {
            ml[r] = m_run[nt][e];
            ml[ROWS + r] = l;
          }
#pragma unroll
          for (int h = 0; h < G; h++) {
            float* dst = merge + r * C::PITCH + 64 * h + 8 * g;
            *reinterpret_cast<float4*>(dst) = make_float4(acc[nt][h][0][e] + z[h], acc[nt][h][1][e] + z[h], acc[nt][h][2][e] + z[h], acc[nt][h][3][e] + z[h]);
            *reinterpret_cast<float4*>(dst + 4) =
                make_float4(acc[nt][h][0][2 + e] + z[h], acc[nt][h][1][2 + e] + z[h], acc[nt][h][2][2 + e] + z[h], acc[nt][h][3][2 + e] + z[h]);
          }
        }
      }
      group_sync();
      const long long seg0 = qc - now.qi, seg1 = seg0 + now.s.quanta;  // the segment's quanta
      const long long w0 = seg0 / per, w1 = (seg1 - 1) / per;          // the groups that share it
      const bool whole = w0 == w1;
      const int slot = seg0 < q0 ? 0 : 1;
      float* part = p.part + ((int64_t)me * 2 + slot) * ROWS * (H + 2);
      const int tok0 = p.cu ? min(max(p.cu[now.b], 0), p.T) : now.b;
      const int rows = min(ROWS, now.s.n * p.R - now.chunk * ROWS);
      auto store = [&](int r, int d, float inv, float a, float b) {
        const int row = now.chunk * ROWS + r;
        uint16_t* dst = p.out + ((int64_t)(tok0 + row / p.R) * p.Nq + now.n * p.R + row % p.R) * H + d;
        *reinterpret_cast<uint32_t*>(dst) = i4_pack(a * inv, b * inv);
      };
      for (int i = gtid; i < rows * (H / 2); i += GW * 32) {
        const int r = i / (H / 2), d = i % (H / 2) * 2;
        float m = -INFINITY;
        for (int k = 0; k < GW; k++) m = fmaxf(m, reinterpret_cast<float*>(group_base + k * C::WARP_BYTES)[ROWS * C::PITCH + r]);
        const float ref = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, a = 0.0f, b = 0.0f;
        for (int k = 0; k < GW; k++) {
          const float* o = reinterpret_cast<const float*>(group_base + k * C::WARP_BYTES);
          const float f = i4_ex2(o[ROWS * C::PITCH + r] - ref);
          if (o[ROWS * C::PITCH + r] == -INFINITY) continue;  // a warp that saw nothing of this row
          l = fmaf(o[ROWS * C::PITCH + ROWS + r], f, l);
          a = fmaf(o[r * C::PITCH + d], f, a);
          b = fmaf(o[r * C::PITCH + d + 1], f, b);
        }
        if (whole) {
          store(r, d, m == -INFINITY ? 0.0f : 1.0f / l, a, b);
        } else {
          if (d == 0) {
            part[r * (H + 2)] = m;
            part[r * (H + 2) + 1] = l;
          }
          *reinterpret_cast<float2*>(part + r * (H + 2) + 2 + d) = make_float2(a, b);
        }
      }
      if (!whole) {
        __threadfence();
        group_sync();
        int* flag = reinterpret_cast<int*>(group_base + ROWS * C::PITCH * 4 + 2 * ROWS * 4 - 4);  // the last float of the first warp's buffer: read by now
        if (gtid == 0) {
          unsigned long long* word = p.counters + w0;
          const unsigned long long want = (unsigned long long)(w1 - w0 + 1);
          unsigned long long old = *reinterpret_cast<volatile unsigned long long*>(word), next;
          for (;;) {  // lock-free: a failed exchange means that another group has arrived
            next = (old & ~0xffffull) == p.nonce ? old + 1 : p.nonce + 1;
            const unsigned long long seen = atomicCAS(word, old, next);
            if (seen == old) break;
            old = seen;
          }
          const bool last = (next & 0xffffull) == want;
          if (last) *word = 0;  // a replayed call starts anew
          *flag = last;
          __threadfence();
        }
        group_sync();
        if (*flag) {
          for (int i = gtid; i < rows * (H / 2); i += GW * 32) {
            const int r = i / (H / 2), d = i % (H / 2) * 2;
            float m = -INFINITY, l = 0.0f, a = 0.0f, b = 0.0f;
            for (long long k = w0; k <= w1; k++) {
              const float* o = p.part + ((int64_t)k * 2 + (seg0 < k * per ? 0 : 1)) * ROWS * (H + 2) + r * (H + 2);
              const float2 ml2 = __ldcg(reinterpret_cast<const float2*>(o)), v = __ldcg(reinterpret_cast<const float2*>(o + 2 + d));
              if (ml2.x == -INFINITY) continue;
              const float m_new = fmaxf(m, ml2.x), fo = i4_ex2(m - m_new), fn = i4_ex2(ml2.x - m_new);
              l = l * fo + ml2.y * fn;
              a = a * fo + v.x * fn;
              b = b * fo + v.y * fn;
              m = m_new;
            }
            store(r, d, m == -INFINITY ? 0.0f : 1.0f / l, a, b);
          }
        }
      }
      group_sync();  // the buffers are free again
      fresh = true;
    }
    if (qc + 1 < q1) advance(now);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---------------------------------------------------------------- host side
static int i4_tiles(int64_t T, int64_t B, int64_t Nq, int64_t Nkv) { return (T > B ? 2 : 1) * (Nq / Nkv) > 8 ? 2 : 1; }
static size_t i4_scratch(int nt, int64_t H) { return (size_t)sm_count() * kI4Warps * (8 + 2 * (size_t)(8 * nt) * (H + 2) * 4); }

template <int H, int NT>
static int i4_launch(I4Params& p, cudaStream_t st) {
  using C = I4Cfg<H, NT>;
  static bool opted[16] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16 || !opted[dev]) {
    TPX_CUDA_OK(cudaFuncSetAttribute(int4_attn_kernel<H, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    if (dev >= 0 && dev < 16) opted[dev] = true;
  }
  p.GW = C::WARPS;
  TPX_CUDA_OK(launch_pdl(int4_attn_kernel<H, NT>, dim3(sm_count()), dim3(C::WARPS * 32), C::SMEM, st, p));
  return TPX_OK;
}

}  // namespace tpx

using namespace tpx;

extern "C" size_t tpx_int4_attention_scratch_bytes(int64_t T, int64_t B, int64_t Nq, int64_t kv_heads, int64_t H) {
  if (T <= 0 || kv_heads <= 0 || Nq <= 0) return 0;
  return i4_scratch(i4_tiles(T, B, Nq, kv_heads), H);
}

extern "C" int tpx_int4_attention(const TpxInt4Attention* a, void* stream) {
  TPX_REQUIRE(a && a->cache && (a->T == 0 || (a->q && a->out)), TPX_ERR_ARG, "int4_attention: null pointer");
  I4Params p = {};
  const int rc = i4_cache_of(a->cache, &p.c);
  if (rc) return rc;
  const int64_t H = a->cache->H, Nkv = a->cache->kv_heads;
  TPX_REQUIRE(a->T >= 0 && a->T < (1ll << 31) / 4096 && (a->cu_seqlens || a->T == a->cache->B), TPX_ERR_ARG, "int4_attention: %ld tokens for %ld sequences", (long)a->T,
              (long)a->cache->B);
  TPX_REQUIRE(a->Nq > 0 && a->Nq <= 4096 && a->Nq % Nkv == 0, TPX_ERR_ARG, "int4_attention: %ld query heads for %ld key heads", (long)a->Nq, (long)Nkv);
  TPX_REQUIRE((((uintptr_t)a->q | (uintptr_t)a->out) & 15) == 0 && a->ldq % 8 == 0, TPX_ERR_ARG, "int4_attention: q, its rows and out must be 16-byte aligned");
  if (a->T == 0) return TPX_OK;
  const int nt = i4_tiles(a->T, a->cache->B, a->Nq, Nkv);
  TPX_REQUIRE(a->scratch && ((uintptr_t)a->scratch & 255) == 0 && a->scratch_bytes >= i4_scratch(nt, H), TPX_ERR_SCRATCH,
              "int4_attention: scratch of %zu bytes, %zu are needed (256-byte aligned)", a->scratch_bytes, i4_scratch(nt, H));
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
  p.sc2 = a->scale * 1.4426950408889634f;
  cudaStream_t st = (cudaStream_t)stream;
  if (H == 128) return nt == 1 ? i4_launch<128, 1>(p, st) : i4_launch<128, 2>(p, st);
  return nt == 1 ? i4_launch<64, 1>(p, st) : i4_launch<64, 2>(p, st);
}
