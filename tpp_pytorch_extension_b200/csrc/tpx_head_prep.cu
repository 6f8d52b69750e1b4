// The pass over the heads behind a q/k/v linear: per-head RMS norm, rotation, and keys and values into the 4-bit cache.
//
//   y = x / sqrt(mean(x^2) + eps) * w          over the H values of a query or key head, statistics in fp32
//   (y_i, y_i+rot/2) -> (y_i c - y_i+rot/2 s, y_i+rot/2 c + y_i s)
// and for the cache, per 64 values of the bf16 row: code = round((x - min) / scale). One read of q/k/v, one write of q and k, 36 bytes
// per 64 cached values: bound by HBM for prompts, by the launch and one chain of dependent loads for single tokens.
//
// H / 16 lanes share a head (two pieces of 8 values per lane, which are the two halves of its rotary pairs), so that norms and ranges
// of 64 values are a few shuffles. A thread does UNITS heads of one token: their loads go out together and share its cosines and sines.
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
  int T, Nq, Nkv, H, rot, per_token;  // per_token: threads per token
  float eps;
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
  float least[2], step[2];  // halves of minimum and scale: the range of a row may pass the largest float
#pragma unroll
  for (int g = 0; g < 2; g++) {
    const uint32_t a = g ? mn & 0xffff0000u : mn << 16, b = g ? mx & 0xffff0000u : mx << 16;
    least[g] = 0.5f * __uint_as_float(a);
    const float half_range = 0.5f * __uint_as_float(b) - least[g];
    const bool fine = (a & 0x7f800000u) != 0x7f800000u && (b & 0x7f800000u) != 0x7f800000u;
    const uint32_t s = fine ? f32_to_bf16_bits(__fdiv_rn(half_range, 7.5f)) : 0x7fc0u;
    step[g] = 0.5f * __uint_as_float(s << 16);
    param[g] = s | (fine ? a & 0xffff0000u : 0x7fc00000u);
  }
  uint32_t* codes = reinterpret_cast<uint32_t*>(dst + (is_v ? H / 2 * kI4Page + H / kI4Group * 4 * kI4Page : 0));
  uint32_t* params = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(codes) + H / 2 * kI4Page) + t * (H / kI4Group);
#pragma unroll
  for (int half = 0; half < 2; half++) {
    const int d = half ? dhi : dlo, g = half ? gh : gl;
    float x[8];
    prep_unpack(half ? hi : lo, x);
    const float base = g ? least[1] : least[0], s = g ? step[1] : step[0];
    uint32_t word = 0;
    if (s > 0.0f) {
#pragma unroll
      for (int i = 0; i < 8; i++) word |= (uint32_t)fminf(rintf(__fdiv_rn(fmaf(0.5f, x[i], -base), s)), 15.0f) << (4 * i);
    }
    codes[is_v ? i4_v_word(H, t, d) : i4_k_word(H, t, d)] = word;
  }
  if (sub == 0)
    for (int g = 0; g < H / kI4Group; g++) params[g] = param[g];
}

template <int LANES, int UNITS>
__global__ void head_prep_kernel(PrepParams p) {
  pdl_trigger();
  pdl_wait();
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int row = (int)(idx / p.per_token), in_row = (int)(idx % p.per_token);
  const int sub = in_row % LANES, first = in_row / LANES, groups = p.per_token / LANES;
  const int heads = p.Nq + p.Nkv + (p.cached ? p.Nkv : 0);
  const bool live_lane = sub * 16 < p.H && row < p.T;  // head sizes that are no power of two leave lanes idle
  // a lane's pieces: the first rot / 16 lanes hold rotary pairs, the others two pieces side by side
  const bool turns = sub * 16 < p.rot;
  const int dlo = turns ? sub * 8 : sub * 16, dhi = turns ? dlo + p.rot / 2 : dlo + 8;

  uint4 lo[UNITS], hi[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; u++) {
    const int h = first + u * groups;
    lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
    if (live_lane && h < heads) {
      const uint16_t* src = h < p.Nq ? p.q + row * p.ldq + h * p.H
                                     : h < p.Nq + p.Nkv ? p.k + row * p.ldk + (h - p.Nq) * p.H : p.v + row * p.ldv + (h - p.Nq - p.Nkv) * p.H;
      lo[u] = *reinterpret_cast<const uint4*>(src + dlo);
      hi[u] = *reinterpret_cast<const uint4*>(src + dhi);
    }
  }
  int seq = -1;
  int64_t place = 0;
  const bool placed = p.cached || p.cu;
  if (row < p.T && placed) {
    seq = i4_sequence(p.cu, p.c.B, row);
    if (seq >= 0 && p.cached) place = (int64_t)max(p.c.lengths[seq], 0) + (p.cu ? row - p.cu[seq] : 0);
  }
  const bool live = row < p.T && (!placed || seq >= 0);
  float cs[8], sn[8];
  bool rotate = turns && live && p.ep;
  if (rotate) {
    const int64_t pos = p.pos ? p.pos[row] : place;
    rotate = pos >= 0 && pos < p.max_pos;
    if (rotate) {
      prep_weights(p.ep + pos * p.ld_ep, 1, dlo, cs);
      prep_weights(p.ep + (p.max_pos + pos) * p.ld_ep, 1, dlo, sn);
    }
  }
#pragma unroll
  for (int u = 0; u < UNITS; u++) {
    const int h = first + u * groups;
    const bool is_q = h < p.Nq, is_v = h >= p.Nq + p.Nkv;
    const void* norm = is_q ? p.q_norm : p.k_norm;
    float a[8], b[8];
    prep_unpack(lo[u], a);
    prep_unpack(hi[u], b);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!is_v && (norm || rotate)) {
      if (norm && live_lane) {
        const float inv = 1.0f / sqrtf(ss / (float)p.H + p.eps);
        float g[8];
        prep_weights(norm, p.norm_f32, dlo, g);
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = a[i] * inv * g[i];
        prep_weights(norm, p.norm_f32, dhi, g);
#pragma unroll
        for (int i = 0; i < 8; i++) b[i] = b[i] * inv * g[i];
      }
      if (rotate) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float x = a[i], y = b[i];
          a[i] = x * cs[i] - y * sn[i];
          b[i] = y * cs[i] + x * sn[i];
        }
      }
      lo[u] = prep_pack(a);
      hi[u] = prep_pack(b);
    }
    const bool write = live && live_lane && h < heads;
    uint16_t* out = is_q ? p.q_out : is_v ? nullptr : p.k_out;
    if (write && out) {
      out += is_q ? ((int64_t)row * p.Nq + h) * p.H : ((int64_t)row * p.Nkv + h - p.Nq) * p.H;
      *reinterpret_cast<uint4*>(out + dlo) = lo[u];
      *reinterpret_cast<uint4*>(out + dhi) = hi[u];
    }
    if (LANES == 4 || LANES == 8) {  // the head sizes of the cache
      // the whole warp takes part in the ranges' shuffles
      if (p.cached && __any_sync(0xffffffffu, write && !is_q)) {
        const int n = is_v ? h - p.Nq - p.Nkv : h - p.Nq;
        uint8_t* dst = write && !is_q ? i4_head(p.c, seq, place, n, 36 * p.H) : nullptr;
        prep_to_cache<LANES>(dst, (int)(place % kI4Page), is_v, p.H, dlo, dhi, lo[u], hi[u], sub);
      }
    }
  }
}

template <int H>
__global__ void int4_read_kernel(I4Cache c, const int32_t* __restrict__ cu, int T, uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out) {
  pdl_trigger();
  pdl_wait();
  constexpr int PIECES = H / 8;
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int d = (int)(idx % PIECES) * 8;
  const int64_t rest = idx / PIECES;
  const int n = (int)(rest % c.Nkv);
  const int64_t row = rest / c.Nkv;
  if (row >= T) return;
  const int seq = i4_sequence(cu, c.B, (int)row);
  if (seq < 0) return;
  const int64_t place = (int64_t)max(c.lengths[seq], 0) + (cu ? (int)row - cu[seq] : 0);
  const uint8_t* src = i4_head(c, seq, place, n, I4<H>::BYTES);
  const int t = (int)(place % kI4Page);
#pragma unroll
  for (int is_v = 0; is_v < 2; is_v++) {
    uint16_t* out = is_v ? v_out : k_out;
    if (!out) continue;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (src) {
      const uint8_t* codes = src + (is_v ? I4<H>::VC : I4<H>::KC);
      const uint32_t word = reinterpret_cast<const uint32_t*>(codes)[is_v ? i4_v_word(H, t, d) : i4_k_word(H, t, d)];
      const uint32_t param = reinterpret_cast<const uint32_t*>(codes + I4<H>::CODES)[t * I4<H>::G + d / kI4Group];
      const float s = __uint_as_float(param << 16), z = __uint_as_float(param & 0xffff0000u);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = fmaf((float)(word >> (4 * i) & 15), s, z);
      w = prep_pack(x);
    }
    *reinterpret_cast<uint4*>(out + ((int64_t)row * c.Nkv + n) * H + d) = w;
  }
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
  // Four heads per thread once that still fills the GPU
  const bool many = (int64_t)p.T * heads * LANES >= (int64_t)sm_count() * 2048;
  const int units = many ? 4 : 1, block = 256;
  p.per_token = (heads + units - 1) / units * LANES;
  const int64_t grid = ((int64_t)p.T * p.per_token + block - 1) / block;
  TPX_REQUIRE(grid < (1ll << 31), TPX_ERR_UNSUPPORTED, "head_prep: too many tokens in one call");
  TPX_CUDA_OK(many ? launch_pdl(head_prep_kernel<LANES, 4>, dim3((unsigned)grid), dim3(block), 0, st, p)
                   : launch_pdl(head_prep_kernel<LANES, 1>, dim3((unsigned)grid), dim3(block), 0, st, p));
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
                  (int)a->T, (int)a->Nq, (int)a->Nkv, (int)a->H, a->ep ? (int)a->rot : 0, 0, a->eps, a->norm_is_f32, 0};
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
  const int64_t grid = (T * c.Nkv * (cache->H / 8) + 255) / 256;
  TPX_REQUIRE(grid < (1ll << 31), TPX_ERR_UNSUPPORTED, "int4_read: too many tokens in one call");
  cudaStream_t st = (cudaStream_t)stream;
  TPX_CUDA_OK(cache->H == 128 ? launch_pdl(int4_read_kernel<128>, dim3((unsigned)grid), dim3(256), 0, st, c, cu_seqlens, (int)T, k_out, v_out)
                              : launch_pdl(int4_read_kernel<64>, dim3((unsigned)grid), dim3(256), 0, st, c, cu_seqlens, (int)T, k_out, v_out));
  return TPX_OK;
}
