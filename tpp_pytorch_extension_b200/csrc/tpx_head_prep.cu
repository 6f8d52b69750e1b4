// The pass over the heads behind a q/k/v linear: per-head RMS norm, rotation, and keys and values into the 4-bit cache.
//
//   y = x / sqrt(mean(x^2) + eps) * w          over the H values of a query or key head, statistics in fp32
//   (y_i, y_i+rot/2) -> (y_i c - y_i+rot/2 s, y_i+rot/2 c + y_i s)
// and for the cache, per 64 values of the bf16 row: code = round((x - min) / scale). One read of q/k/v, one write of q and k, 36 bytes
// per 64 cached values. Single tokens are bound by the launch and one chain of dependent loads; prompts by latencies (see the counters below: neither HBM
// nor the issue slots are full), the append by the ranges' shuffles and the codes.
//
// H / 16 lanes share a head (two pieces of 8 values per lane, which are the two halves of its rotary pairs), so that norms and ranges
// of 64 values are a few shuffles. A warp works on heads of one kind of one token: a thread does up to UNITS of them, whose loads go out
// together, with the products of norm weights, cosines and sines kept in registers. 8191 tokens, 32/8 heads of 128, norms and rotation: 45 us (3.8 TB/s
// of inputs and outputs, HBM busy 36 %, 53 % of issue slots); one token: 5.4 us with the call. 8 key heads of 128, 32768 tokens: append alone 132 us (1.3 TB/s),
// read-back alone 33.5 us (5.1 TB/s, HBM); 4071 tokens: 21.3 and 7.1 us.
#include <numeric>

#include "tpx_int4.cuh"

namespace tpx {

struct PrepParams {
  const uint16_t *q, *k, *v;
  const void *q_norm, *k_norm;
  const float* ep;
  const int64_t* pos;
  const int32_t* cu;
  uint16_t *q_out, *k_out;
  I4Cache c;
  int64_t ldq, ldk, ldv, max_pos, ld_ep;
  int T, Nq, Nkv, H, rot, wq, wkv, wpt;  // warps per token for queries, for keys and for values each, in all
  int stride;                                 // resident warps that walk the items
  float eps, inv_h;
  int norm_f32, cached;
};

__device__ __forceinline__ void prep_unpack(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; j++) {
    x[2 * j] = __uint_as_float(w[j] << 16);
    x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 prep_pack(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
    w[j] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void prep_weights(const void* w, int f32, int d, float (&g)[8]) {
  if (f32) {
    const float4 a = *reinterpret_cast<const float4*>((const float*)w + d), b = *reinterpret_cast<const float4*>((const float*)w + d + 4);
    g[0] = a.x; g[1] = a.y; g[2] = a.z; g[3] = a.w; g[4] = b.x; g[5] = b.y; g[6] = b.z; g[7] = b.w;
  } else {
    prep_unpack(*reinterpret_cast<const uint4*>((const uint16_t*)w + d), g);
  }
}
// bf16 pairs: a NaN in either operand is the result
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// A lane's two pieces of a bf16 row (dimensions dlo.., dhi..) into place t of a page's head. All lanes of the head's group call it; `dst` null:
// nothing is written.
template <int LANES>
__device__ __forceinline__ void prep_to_cache(uint8_t* dst, int t, bool is_v, int H, int dlo, int dhi, uint4 lo, uint4 hi, int sub) {
  auto range = [](uint4 a, uint32_t& mn, uint32_t& mx) {  // of 8 values, in both halves of a word
    mn = min2_nan(min2_nan(a.x, a.y), min2_nan(a.z, a.w));
    mx = max2_nan(max2_nan(a.x, a.y), max2_nan(a.z, a.w));
    mn = min2_nan(mn, __byte_perm(mn, 0, 0x1032));
    mx = max2_nan(mx, __byte_perm(mx, 0, 0x1032));
  };
  uint32_t mnl, mxl, mnh, mxh;
  range(lo, mnl, mxl);
  range(hi, mnh, mxh);
  // low half of a word: the first 64 dimensions, high half: the others
  const int gl = dlo / kI4Group, gh = dhi / kI4Group;
  const uint32_t INF = 0x7f807f80u, NINF = 0xff80ff80u;
  auto only = [](uint32_t v, uint32_t none, int g) { return g == 0 ? (v & 0xffffu) | (none & 0xffff0000u) : (v & 0xffff0000u) | (none & 0xffffu); };
  uint32_t mn = min2_nan(only(mnl, INF, gl), only(mnh, INF, gh)), mx = max2_nan(only(mxl, NINF, gl), only(mxh, NINF, gh));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    mn = min2_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = max2_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (!dst) return;
  uint32_t param[2];
  float least[2], step[2], back[2];  // halves of minimum and scale: the range of a row may pass the largest float
#pragma unroll
  for (int g = 0; g < 2; g++) {
    const uint32_t a = g ? mn & 0xffff0000u : mn << 16, b = g ? mx & 0xffff0000u : mx << 16;
    least[g] = 0.5f * __uint_as_float(a);
    const float half_range = 0.5f * __uint_as_float(b) - least[g];
    const bool fine = (a & 0x7f800000u) != 0x7f800000u && (b & 0x7f800000u) != 0x7f800000u;
    const uint32_t s = fine ? f32_to_bf16_bits(__fdiv_rn(half_range, 7.5f)) : 0x7fc0u;
    step[g] = 0.5f * __uint_as_float(s << 16);
    back[g] = __frcp_rn(step[g]);
    param[g] = s | (fine ? a & 0xffff0000u : 0x7fc00000u);
  }
  uint32_t* codes = reinterpret_cast<uint32_t*>(dst + (is_v ? H / 2 * kI4Page + H / kI4Group * 4 * kI4Page : 0));
  uint32_t* params = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(codes) + H / 2 * kI4Page) + t * (H / kI4Group);
#pragma unroll
  for (int half = 0; half < 2; half++) {
    const int d = half ? dhi : dlo, g = half ? gh : gl;
    float x[8];
    prep_unpack(half ? hi : lo, x);
    const float base = g ? least[1] : least[0], s = g ? step[1] : step[0], y = g ? back[1] : back[0];
    uint32_t word = 0;
    if (s > 1e-30f && s < 1e30f) {
      // v / s: the product with the reciprocal, corrected once by the remainder that a multiply-add leaves exactly (P. W. Markstein, "Computation of
      // elementary functions on the IBM RISC System/6000 processor", IBM J. Res. Dev. 34, 1990). What codes need of it follows from s having 8
      // bits: a quotient halfway between two codes has 5 bits and comes out as it is, since the corrected value is off by 2^-46 of itself before it is
      // rounded; rounding is monotone, so no other quotient gets past that point. 1.5 * 2^23 then rounds it to a whole number.
      // Where remainders might not be normal numbers: the division itself.
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 7; i >= 0; i--) {
        const float v = fmaf(0.5f, x[i], -base), q = v * y, r = fmaf(fmaf(-q, s, v), y, q);
        sum[i >> 2] = fmaf(sum[i >> 2], 16.0f, fminf((r + 12582912.0f) - 12582912.0f, 15.0f));
      }
      word = (__float_as_uint(sum[0] + 12582912.0f) & 0xffffu) | __float_as_uint(sum[1] + 12582912.0f) << 16;
    } else if (s > 0.0f) {
      for (int i = 0; i < 8; i++) word |= (uint32_t)fminf(rintf(__fdiv_rn(fmaf(0.5f, x[i], -base), s)), 15.0f) << (4 * i);
    }
    codes[is_v ? i4_v_word(H, t, d) : i4_k_word(H, t, d)] = word;
  }
  if (sub == 0)
    for (int g = 0; g < H / kI4Group; g++) params[g] = param[g];
}

// Pairs of fp32 in one operation, kept in 64-bit registers
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 prep_pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void prep_halves(f32x2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a)); }
__device__ __forceinline__ f32x2 prep_fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 prep_mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void prep_pairs(uint4 v, f32x2 (&x)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; j++) x[j] = prep_pair(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
}
__device__ __forceinline__ uint4 prep_pack(const f32x2 (&x)[4]) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; j++) prep_halves(x[j], f[2 * j], f[2 * j + 1]);
  return prep_pack(f);
}

// What a warp works on: heads of one kind of one token
struct PrepItem {
  int row, kind, N, groups, base;  // queries, keys, values; heads, distance of a thread's heads, the warp's first group
  int seq;                         // -1: a row of no sequence
  int64_t place, pos;              // of the token in the cache, in the rotation table (outside: no rotation)
};
__device__ __forceinline__ bool prep_turns(const PrepParams& p, const PrepItem& it) { return (unsigned long long)it.pos < (unsigned long long)p.max_pos; }
template <int LANES>
__device__ __forceinline__ PrepItem prep_item(const PrepParams& p, int row, int in_row) {
  PrepItem it;
  it.row = row;
  it.kind = in_row < p.wq ? 0 : in_row < p.wq + p.wkv ? 1 : 2;
  it.N = it.kind ? p.Nkv : p.Nq;
  it.groups = (it.kind ? p.wkv : p.wq) * (32 / LANES);
  it.base = (in_row - (it.kind == 0 ? 0 : it.kind == 1 ? p.wq : p.wq + p.wkv)) * (32 / LANES);
  it.seq = 0;
  it.place = 0;
  if (p.cached) {
    it.seq = i4_sequence(p.cu, p.c.B, it.row);
    if (it.seq >= 0) it.place = (int64_t)max(p.c.lengths[it.seq], 0) + (p.cu ? it.row - p.cu[it.seq] : 0);
  }
  it.pos = it.kind == 2 || p.rot == 0 ? -1 : p.pos ? p.pos[it.row] : it.place;  // looked at when the item is fetched, not here
  return it;
}
// A lane's pieces of a head: the first rot / 16 lanes hold rotary pairs, the others two pieces side by side
struct PrepLane {
  int sub, dlo, dhi;
  bool live, turns;  // head sizes that are no power of two leave lanes idle
};
template <int LANES>
__device__ __forceinline__ PrepLane prep_lane(const PrepParams& p, int lane) {
  PrepLane l;
  l.sub = lane % LANES;
  l.live = l.sub * 16 < p.H;
  l.turns = l.sub * 16 < p.rot;
  l.dlo = l.turns ? l.sub * 8 : l.sub * 16;
  l.dhi = l.turns ? l.dlo + p.rot / 2 : l.dlo + 8;
  return l;
}
__device__ __forceinline__ const uint16_t* prep_source(const PrepParams& p, const PrepItem& it) {
  return it.kind == 0 ? p.q + it.row * p.ldq : it.kind == 1 ? p.k + it.row * p.ldk : p.v + it.row * p.ldv;
}

// The heads of an item: load(u, lo, hi) gives the thread's pieces of its head u, weights(wl, wh) those of the norm (or ones),
// angles(cs, sn) its cosines and sines
template <int LANES, int UNITS, class Load, class Weights, class Angles>
__device__ __forceinline__ void prep_heads(const PrepParams& p, const PrepItem& it, const PrepLane& l, int lane, Load load, Weights weights, Angles angles) {
  const bool norm = it.kind == 0 ? p.q_norm != nullptr : it.kind == 1 && p.k_norm != nullptr;
  const bool rotate = l.turns && prep_turns(p, it), turned = __all_sync(0xffffffffu, rotate || !l.live);
  const int first = it.base + lane / LANES;
  // out_lo = x_lo (w_lo c) - x_hi (w_hi s), out_hi = x_hi (w_hi c) + x_lo (w_lo s)
  f32x2 lc[4], hs[4], hc[4], ls[4];
  if (it.kind < 2) {
    f32x2 wl[4], wh[4];
    weights(wl, wh);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      lc[i] = wl[i];
      hc[i] = wh[i];
      hs[i] = ls[i] = 0;
    }
    if (rotate) {
      f32x2 cs[4], sn[4];
      angles(cs, sn);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        lc[i] = prep_mul2(wl[i], cs[i]);
        hc[i] = prep_mul2(wh[i], cs[i]);
        ls[i] = prep_mul2(wl[i], sn[i]);
        hs[i] = prep_mul2(wh[i], sn[i]) ^ 0x8000000080000000ull;
      }
    }
  }
  uint16_t* const out0 = it.kind == 0 ? p.q_out : p.k_out;
#pragma unroll
  for (int u = 0; u < UNITS; u++) {
    if (u * it.groups >= it.N) break;
    const int h = first + u * it.groups;
    const bool write = l.live && h < it.N;
    uint4 lo, hi;
    load(u, lo, hi);
    if (it.kind < 2) {
      f32x2 a[4], b[4];
      prep_pairs(lo, a);
      prep_pairs(hi, b);
      if (norm) {
        f32x2 s2 = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) s2 = prep_fma2(b[i], b[i], prep_fma2(a[i], a[i], s2));
        float s0, s1;
        prep_halves(s2, s0, s1);
        float ss = s0 + s1;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(fmaf(ss, p.inv_h, p.eps));
        const f32x2 inv2 = prep_pair(inv, inv);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          a[i] = prep_mul2(a[i], inv2);
          b[i] = prep_mul2(b[i], inv2);
        }
      }
      if (norm || p.rot) {
        f32x2 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          x[i] = prep_mul2(a[i], lc[i]);
          y[i] = prep_mul2(b[i], hc[i]);
        }
        if (turned || rotate) {  // the whole warp, or the lanes that do: elsewhere 0 * infinity would be added
#pragma unroll
          for (int i = 0; i < 4; i++) {
            x[i] = prep_fma2(b[i], hs[i], x[i]);
            y[i] = prep_fma2(a[i], ls[i], y[i]);
          }
        }
        lo = prep_pack(x);
        hi = prep_pack(y);
      }
      if (write && out0) {
        uint16_t* out = out0 + ((int64_t)it.row * it.N + h) * p.H;
        *reinterpret_cast<uint4*>(out + l.dlo) = lo;
        *reinterpret_cast<uint4*>(out + l.dhi) = hi;
      }
    }
    if (LANES == 4 || LANES == 8) {  // the head sizes of the cache
      if (p.cached && it.kind > 0)   // the whole warp takes part in the ranges' shuffles
        prep_to_cache<LANES>(write ? i4_head(p.c, it.seq, it.place, h, 36 * p.H) : nullptr, (int)(it.place % kI4Page), it.kind == 2, p.H, l.dlo, l.dhi, lo, hi, l.sub);
    }
  }
}

// Few tokens: a warp per item, a head per thread, loads straight to registers
template <int LANES>
__global__ void __launch_bounds__(256) head_prep_kernel(const PrepParams p) {
  pdl_trigger();
  pdl_wait();
  const int item = (int)(((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5), lane = threadIdx.x & 31;
  if (item >= p.T * p.wpt) return;  // a warp as a whole
  const PrepLane l = prep_lane<LANES>(p, lane);
  const PrepItem it = prep_item<LANES>(p, item / p.wpt, item % p.wpt);
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (l.live && it.base + lane / LANES < it.N) {
    const uint16_t* src = prep_source(p, it) + (it.base + lane / LANES) * p.H;
    lo = *reinterpret_cast<const uint4*>(src + l.dlo);
    hi = *reinterpret_cast<const uint4*>(src + l.dhi);
  }
  if (it.seq < 0) return;  // a row of no sequence
  const void* norm = it.kind == 0 ? p.q_norm : p.k_norm;
  auto pairs = [](const float(&f)[8], f32x2(&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = prep_pair(f[2 * i], f[2 * i + 1]);
  };
  prep_heads<LANES, 1>(
      p, it, l, lane,
      [&](int, uint4& a, uint4& b) {
        a = lo;
        b = hi;
      },
      [&](f32x2(&wl)[4], f32x2(&wh)[4]) {
        float f[8] = {1, 1, 1, 1, 1, 1, 1, 1}, h[8] = {1, 1, 1, 1, 1, 1, 1, 1};
        if (norm && l.live) {
          prep_weights(norm, p.norm_f32, l.dlo, f);
          prep_weights(norm, p.norm_f32, l.dhi, h);
        }
        pairs(f, wl);
        pairs(h, wh);
      },
      [&](f32x2(&cs)[4], f32x2(&sn)[4]) {
        float f[8];
        prep_weights(p.ep + it.pos * p.ld_ep, 1, l.dlo, f);
        pairs(f, cs);
        prep_weights(p.ep + (p.max_pos + it.pos) * p.ld_ep, 1, l.dlo, f);
        pairs(f, sn);
      });
}

// Many tokens: resident warps walk the tokens, four heads per thread. The next token's pieces and angles come by cp.async while this one is
// worked on, each lane's into places of its own (no barrier): with loads to registers 16 warps per SM had too little in flight (8191
// tokens, 40 heads of 128: 51 us, 3.4 TB/s).
// Four heads: with three 52.7 us, with two 57.9 (102 with three blocks per SM), against 45.2
constexpr int kPrepUnits = 4, kPrepWarps = 8;
constexpr int kPrepStage = (2 * kPrepUnits + 4) * 512;  // bytes per warp: two pieces of each head, four of cosines and sines
template <int LANES>
__global__ void __launch_bounds__(kPrepWarps * 32, 2) head_prep_many_kernel(const PrepParams p) {
  extern __shared__ __align__(16) unsigned char prep_smem[];
  __shared__ __align__(16) float norms[2][LANES * 16];  // weights of queries and of keys, or ones
  pdl_trigger();
  pdl_wait();
  for (int i = threadIdx.x; i < 2 * LANES * 16; i += kPrepWarps * 32) {
    const void* w = i < LANES * 16 ? p.q_norm : p.k_norm;
    const int d = i % (LANES * 16);
    norms[i / (LANES * 16)][d] = !w || d >= p.H ? 1.0f : p.norm_f32 ? ((const float*)w)[d] : bf16_bits_to_f32(((const uint16_t*)w)[d]);
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = p.stride, items = p.T * p.wpt;
  int i = blockIdx.x * kPrepWarps + warp;
  if (i >= min(warps, items)) return;
  const PrepLane l = prep_lane<LANES>(p, lane);
  unsigned char* mine = prep_smem + warp * 2 * kPrepStage + lane * 16;
  const uint32_t mine_s = (uint32_t)__cvta_generic_to_shared(mine);
  // what is not there (no such head, a lane without values, a token without angles) is filled with zeros
  auto copy = [&](int piece, int stage, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(mine_s + stage * kPrepStage + piece * 512), "l"(src), "r"(valid ? 16 : 0) : "memory");
  };
  auto fetch = [&](const PrepItem& it, int stage) {
    const uint16_t* src = prep_source(p, it);
    const int h0 = it.base + lane / LANES;
#pragma unroll
    for (int u = 0; u < kPrepUnits; u++) {
      const bool valid = l.live && h0 + u * it.groups < it.N;
      const uint16_t* head = src + (valid ? (h0 + u * it.groups) * p.H : 0);
      copy(2 * u, stage, head + (valid ? l.dlo : 0), valid);
      copy(2 * u + 1, stage, head + (valid ? l.dhi : 0), valid);
    }
    if (p.rot && it.kind < 2) {
      const bool valid = l.turns && prep_turns(p, it);
      const float *c = p.ep + (valid ? it.pos * p.ld_ep + l.dlo : 0), *s = c + (valid ? p.max_pos * p.ld_ep : 0);
      copy(2 * kPrepUnits, stage, c, valid);
      copy(2 * kPrepUnits + 1, stage, c + (valid ? 4 : 0), valid);
      copy(2 * kPrepUnits + 2, stage, s, valid);
      copy(2 * kPrepUnits + 3, stage, s + (valid ? 4 : 0), valid);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // items of one warp are taken in the order of the rows; the one after the next is looked up a round ahead
  int row = i / p.wpt, in_row = i % p.wpt;
  const int rows_on = warps / p.wpt, in_row_on = warps % p.wpt;
  auto onward = [&]() {
    row += rows_on;
    in_row += in_row_on;
    if (in_row >= p.wpt) {
      in_row -= p.wpt;
      row++;
    }
  };
  PrepItem now = prep_item<LANES>(p, row, in_row), ahead = now;
  fetch(now, 0);
  onward();
  if (i + warps < items) ahead = prep_item<LANES>(p, row, in_row);
  for (int stage = 0; i < items; i += warps, stage ^= 1) {
    if (i + warps < items) fetch(ahead, stage ^ 1);
    else asm volatile("cp.async.commit_group;" ::: "memory");
    PrepItem later = ahead;
    onward();
    if (i + 2 * warps < items) later = prep_item<LANES>(p, row, in_row);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const unsigned char* at = mine + stage * kPrepStage;
    auto four = [](const void* from, f32x2& a, f32x2& b) {  // of 16 bytes
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(from);
      a = v.x;
      b = v.y;
    };
    if (now.seq >= 0)
      prep_heads<LANES, kPrepUnits>(
          p, now, l, lane,
          [&](int u, uint4& a, uint4& b) {
            a = *reinterpret_cast<const uint4*>(at + 2 * u * 512);
            b = *reinterpret_cast<const uint4*>(at + (2 * u + 1) * 512);
          },
          [&](f32x2(&wl)[4], f32x2(&wh)[4]) {
            const float* w = norms[now.kind];
            four(w + l.dlo, wl[0], wl[1]);
            four(w + l.dlo + 4, wl[2], wl[3]);
            four(w + l.dhi, wh[0], wh[1]);
            four(w + l.dhi + 4, wh[2], wh[3]);
          },
          [&](f32x2(&cs)[4], f32x2(&sn)[4]) {
            four(at + 2 * kPrepUnits * 512, cs[0], cs[1]);
            four(at + (2 * kPrepUnits + 1) * 512, cs[2], cs[3]);
            four(at + (2 * kPrepUnits + 2) * 512, sn[0], sn[1]);
            four(at + (2 * kPrepUnits + 3) * 512, sn[2], sn[3]);
          });
    now = ahead;
    ahead = later;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// A thread has one piece of 8 values of up to UNITS heads of a token: where the token is found once, and the loads go out together.
template <int H, int UNITS>
__global__ void __launch_bounds__(256) int4_read_kernel(I4Cache c, const int32_t* __restrict__ cu, int T, int groups, uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out) {
  pdl_trigger();
  pdl_wait();
  using L = I4<H>;
  constexpr int PIECES = H / 8;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int d = (int)(idx % PIECES) * 8;
  const int64_t rest = idx / PIECES;
  const int first = (int)(rest % groups);
  const int64_t row = rest / groups;
  if (row >= T) return;
  const int seq = i4_sequence(cu, c.B, (int)row);
  if (seq < 0) return;
  const int64_t place = (int64_t)max(c.lengths[seq], 0) + (cu ? (int)row - cu[seq] : 0);
  const int t = (int)(place % kI4Page);
  const uint8_t* page = i4_head(c, seq, place, 0, L::BYTES);
  uint32_t word[UNITS][2], param[UNITS][2];
#pragma unroll
  for (int u = 0; u < UNITS; u++)
#pragma unroll
    for (int is_v = 0; is_v < 2; is_v++) {
      word[u][is_v] = param[u][is_v] = 0;
      if (page && first + u * groups < c.Nkv) {
        const uint8_t* codes = page + (int64_t)(first + u * groups) * L::BYTES + (is_v ? L::VC : L::KC);
        word[u][is_v] = reinterpret_cast<const uint32_t*>(codes)[is_v ? i4_v_word(H, t, d) : i4_k_word(H, t, d)];
        param[u][is_v] = reinterpret_cast<const uint32_t*>(codes + L::CODES)[t * L::G + d / kI4Group];
      }
    }
#pragma unroll
  for (int u = 0; u < UNITS; u++)
#pragma unroll
    for (int is_v = 0; is_v < 2; is_v++) {
      uint16_t* out = is_v ? v_out : k_out;
      if (!out || first + u * groups >= c.Nkv) continue;
      const float s = __uint_as_float(param[u][is_v] << 16), z = __uint_as_float(param[u][is_v] & 0xffff0000u);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = fmaf((float)(word[u][is_v] >> (4 * i) & 15), s, z);
      *reinterpret_cast<uint4*>(out + (row * c.Nkv + first + u * groups) * H + d) = prep_pack(x);
    }
}

template <int H>
static int read_launch(const I4Cache& c, const int32_t* cu, int T, uint16_t* k_out, uint16_t* v_out, cudaStream_t st) {
  const bool many = (int64_t)T * c.Nkv * (H / 8) >= (int64_t)sm_count() * 2048;
  const int units = many ? 4 : 1, groups = (c.Nkv + units - 1) / units;
  const int64_t grid = ((int64_t)T * groups * (H / 8) + 255) / 256;
  TPX_REQUIRE(grid < (1ll << 31), TPX_ERR_UNSUPPORTED, "int4_read: too many tokens in one call");
  TPX_CUDA_OK(many ? launch_pdl(int4_read_kernel<H, 4>, dim3((unsigned)grid), dim3(256), 0, st, c, cu, T, groups, k_out, v_out)
                   : launch_pdl(int4_read_kernel<H, 1>, dim3((unsigned)grid), dim3(256), 0, st, c, cu, T, groups, k_out, v_out));
  return TPX_OK;
}

int i4_cache_of(const TpxInt4Cache* a, I4Cache* c) {
  TPX_REQUIRE(a->pool && a->table && a->lengths, TPX_ERR_ARG, "int4 cache: null pointer");
  TPX_REQUIRE(((uintptr_t)a->pool & 15) == 0, TPX_ERR_ARG, "int4 cache: the pool must be 16-byte aligned");
  TPX_REQUIRE(a->H == 64 || a->H == 128, TPX_ERR_UNSUPPORTED, "int4 cache: head size %ld not supported (64 or 128)", (long)a->H);
  TPX_REQUIRE(a->B > 0 && a->B <= 65536 && a->kv_heads > 0 && a->kv_heads <= 1024 && a->pages > 0 && a->pages < (1ll << 31) && a->table_cols > 0 &&
                  a->table_cols <= (1 << 25),
              TPX_ERR_ARG, "int4 cache: %ld sequences, %ld heads, %ld pages, %ld table columns", (long)a->B, (long)a->kv_heads, (long)a->pages,
              (long)a->table_cols);
  *c = I4Cache{a->pool, a->table, a->lengths, (int)a->pages, (int)a->table_cols, (int)a->B, (int)a->kv_heads};
  return TPX_OK;
}

template <int LANES>
static int prep_launch(PrepParams& p, cudaStream_t st) {
  const int heads = p.Nq + p.Nkv + (p.cached ? p.Nkv : 0);
  // Four heads per thread and resident warps once that gives every warp an item or more
  const bool many = (int64_t)p.T * heads * LANES >= (int64_t)sm_count() * 2048 && heads <= 2048;
  const int per_warp = 32 / LANES * (many ? kPrepUnits : 1);
  p.wq = (p.Nq + per_warp - 1) / per_warp;
  p.wkv = (p.Nkv + per_warp - 1) / per_warp;
  p.wpt = p.wq + (p.cached ? 2 : 1) * p.wkv;
  TPX_REQUIRE((int64_t)p.T * p.wpt < (1ll << 30), TPX_ERR_UNSUPPORTED, "head_prep: too many tokens in one call");
  if (!many) {
    TPX_CUDA_OK(launch_pdl(head_prep_kernel<LANES>, dim3((p.T * p.wpt + 7) / 8), dim3(256), 0, st, p));
    return TPX_OK;
  }
  // no common factor with the items of a token: every warp then meets all kinds, which take different times
  p.stride = 2 * sm_count() * kPrepWarps;
  while (std::gcd(p.stride, p.wpt) != 1) p.stride--;
  constexpr int SMEM = kPrepWarps * 2 * kPrepStage;
  static bool opted[16] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 16 || !opted[dev]) {
    TPX_CUDA_OK(cudaFuncSetAttribute(head_prep_many_kernel<LANES>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev >= 0 && dev < 16) opted[dev] = true;
  }
  TPX_CUDA_OK(launch_pdl(head_prep_many_kernel<LANES>, dim3(2 * sm_count()), dim3(kPrepWarps * 32), SMEM, st, p));
  return TPX_OK;
}

}  // namespace tpx

using namespace tpx;

extern "C" int tpx_head_prep(const TpxHeadPrep* a, void* stream) {
  TPX_REQUIRE(a, TPX_ERR_ARG, "head_prep: null pointer");
  TPX_REQUIRE(a->T >= 0 && a->T < (1ll << 31) && a->Nq >= 0 && a->Nkv >= 0 && a->Nq + a->Nkv > 0 && a->Nq <= 4096 && a->Nkv <= 1024, TPX_ERR_ARG,
              "head_prep: %ld tokens, %ld query and %ld key heads", (long)a->T, (long)a->Nq, (long)a->Nkv);
  TPX_REQUIRE(a->H >= 16 && a->H <= 256 && a->H % 16 == 0, TPX_ERR_UNSUPPORTED, "head_prep: head size %ld (multiples of 16 up to 256)", (long)a->H);
  TPX_REQUIRE(!a->ep || (a->rot >= 16 && a->rot <= a->H && a->rot % 16 == 0 && a->max_pos > 0 && a->ld_ep >= a->rot / 2 && a->ld_ep % 4 == 0), TPX_ERR_ARG,
              "head_prep: %ld rotated values of %ld (a multiple of 16), %ld positions in rows of %ld", (long)a->rot, (long)a->H, (long)a->max_pos, (long)a->ld_ep);
  TPX_REQUIRE(a->T == 0 || ((a->Nq == 0 || (a->q && a->q_out)) && (a->Nkv == 0 || a->k) && (!a->cache || a->Nkv == 0 || a->v)), TPX_ERR_ARG, "head_prep: null pointer");
  TPX_REQUIRE(!a->cu_seqlens || a->cache, TPX_ERR_ARG, "head_prep: sequences are those of a cache");
  uintptr_t bits = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q_out | (uintptr_t)a->k_out | (uintptr_t)a->q_norm |
                   (uintptr_t)a->k_norm | (uintptr_t)a->ep;
  TPX_REQUIRE((bits & 15) == 0 && (a->ldq | a->ldk | a->ldv) % 8 == 0, TPX_ERR_ARG, "head_prep: tensors and their rows must be 16-byte aligned");
  PrepParams p = {a->q, a->k, a->v, a->q_norm, a->k_norm, a->ep, a->pos, a->cu_seqlens, a->q_out, a->k_out, {}, a->ldq, a->ldk, a->ldv, a->max_pos, a->ld_ep,
                  (int)a->T, (int)a->Nq, (int)a->Nkv, (int)a->H, a->ep ? (int)a->rot : 0, 0, 0, 0, 0, a->eps, 1.0f / (float)a->H, a->norm_is_f32, 0};
  if (a->cache) {
    const int rc = i4_cache_of(a->cache, &p.c);
    if (rc) return rc;
    TPX_REQUIRE(a->cache->H == a->H && a->cache->kv_heads == a->Nkv, TPX_ERR_ARG, "head_prep: %ld key heads of %ld, the cache has %ld of %ld", (long)a->Nkv,
                (long)a->H, (long)a->cache->kv_heads, (long)a->cache->H);
    TPX_REQUIRE(a->cu_seqlens || a->T == a->cache->B, TPX_ERR_ARG, "head_prep: %ld tokens for %ld sequences of one token", (long)a->T, (long)a->cache->B);
    p.cached = 1;
  }
  if (a->T == 0) return TPX_OK;
  cudaStream_t st = (cudaStream_t)stream;
  if (a->H <= 16) return prep_launch<1>(p, st);
  if (a->H <= 32) return prep_launch<2>(p, st);
  if (a->H <= 64) return prep_launch<4>(p, st);
  if (a->H <= 128) return prep_launch<8>(p, st);
  return prep_launch<16>(p, st);
}

extern "C" int tpx_int4_read(const TpxInt4Cache* cache, const int32_t* cu_seqlens, int64_t T, uint16_t* k_out, uint16_t* v_out, void* stream) {
  TPX_REQUIRE(cache, TPX_ERR_ARG, "int4_read: null pointer");
  I4Cache c;
  const int rc = i4_cache_of(cache, &c);
  if (rc) return rc;
  TPX_REQUIRE(T >= 0 && T < (1ll << 31) && (cu_seqlens || T == cache->B), TPX_ERR_ARG, "int4_read: %ld tokens for %ld sequences", (long)T, (long)cache->B);
  TPX_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, TPX_ERR_ARG, "int4_read: outputs must be 16-byte aligned");
  if (T == 0) return TPX_OK;
  return cache->H == 128 ? read_launch<128>(c, cu_seqlens, (int)T, k_out, v_out, (cudaStream_t)stream)
                         : read_launch<64>(c, cu_seqlens, (int)T, k_out, v_out, (cudaStream_t)stream);
}
