// AdamW over many tensors, the gradient norm over many tensors, and the
// 8-bit form of AdamW's moments.  Beside the SGD/EMA kernels of
// multi_tensor.hip, but with the tensor table in the kernel's arguments: no
// device-side table is built, so nothing is kept from one call to the next.
//
//   g  = coef * grad              coef = min(1, max_norm / (norm + 1e-6))
//   m' = b1 m + (1 - b1) g        v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd)
//        - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// m' and v' are rounded operation by operation (no contraction into fma), as
// a plain elementwise program in 32 bits does, and the root is rounded
// correctly, so that what is rounded to 8 bits afterwards falls on the same
// codes (a root that is off by an ulp moves one code in 2e5, and with it later
// steps).  What reaches the weights alone takes the hardware's reciprocal, off
// by an ulp at most, and fma.
#include "common.h"
#include "launchers.h"

#pragma clang fp contract(off)

namespace {

constexpr int THREADS = 256;
constexpr int CHUNK = ADAMW_CHUNK;  // elements of one table chunk
constexpr int QBLOCK = 256;         // elements that share a pair of scales
constexpr float TINY = 1e-30f;      // least block maximum a scale stands for
constexpr float TOP_M = 448.f;      // largest e4m3 value
constexpr float TOP_R = 1.9375f;    // largest value of a code of sqrt(v)
static_assert(sizeof(AdamwTable) + sizeof(AdamwScalars) + 16 <= 4096 &&
                  sizeof(GradTable) + 8 <= 4096,
              "kernel arguments");
static_assert(CHUNK == THREADS * 16, "a thread handles 16 elements");

// Where chunk c lies.  first[] ascends, so its tensor is the last one whose
// first chunk is not behind c; a lane looks at one tensor in 64.
struct Place {
  int tensor;
  int64_t at;  // first element
  int left;    // elements, CHUNK at most
};
template <typename Table>
__device__ __forceinline__ Place find_chunk(const Table& tab, uint32_t c) {
  const int lane = threadIdx.x % WAVE;
  int t = -1;
  for (int b = 0; b < tab.count; b += WAVE) {
    const int i = b + lane;
    t += __popcll(__ballot(i < tab.count && tab.first[i] <= c));
  }
  const bool last = c + 1 == (t + 1 < tab.count ? tab.first[t + 1]
                                                : tab.chunks);
  return {t, (int64_t)(c - tab.first[t]) * CHUNK, last ? tab.tail[t] : CHUNK};
}

// V elements of type T as they lie in memory.  Tensors may be views that
// begin anywhere: only the element's own alignment is assumed.  ONCE: past
// the caches, for what will not be there when it is next used.
typedef uint32_t word4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T, int V>
struct Raw {
  static constexpr int W = sizeof(T) * V / 16;
  word4 w[W];
  template <bool ONCE>
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      w[i] = ONCE ? __builtin_nontemporal_load((const word4*)p + i)
                  : *((const word4*)p + i);
  }
  __device__ __forceinline__ void floats(float (&out)[V]) const {
    T t[V];
    __builtin_memcpy(t, w, sizeof(t));
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)t[i];
  }
};

template <bool ONCE, typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
  T t[V];
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = (T)in[i];  // to nearest even
  word4 w[sizeof(t) / 16];
  __builtin_memcpy(w, t, sizeof(t));
#pragma unroll
  for (int i = 0; i < (int)sizeof(t) / 16; ++i) {
    if (ONCE) __builtin_nontemporal_store(w[i], (word4*)p + i);
    else *((word4*)p + i) = w[i];
  }
}

// the first `n` of them (n may be <= 0); zeros behind
template <typename T, int V>
__device__ __forceinline__ void load_part(const T* p, float (&out)[V],
                                          int n) {
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = i < n ? (float)p[i] : 0.f;
}

template <typename T, int V>
__device__ __forceinline__ void store_part(T* p, const float (&in)[V],
                                           int n) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) p[i] = (T)in[i];
}

// min(1, max_norm / (norm + 1e-6)); a NaN norm stays a NaN
__device__ __forceinline__ float clip_coef(const float* norm,
                                           float max_norm) {
  if (norm == nullptr) return 1.f;
  const float c = max_norm / (*norm + 1e-6f);
  return c > 1.f ? 1.f : c;
}

// The square root, rounded correctly, of any v.  The hardware's is off by an
// ulp at most for normal v (and zero for subnormal ones), so it is that, or its
// neighbour below or above: by Tuckerman's test (Agarwal et al., "New scalar
// and vector elementary functions for the IBM System/370", 1986), r is the root
// rounded to nearest where r (r - ulp) < v <= r (r + ulp).  An fma gives those
// differences' signs exactly where they are normal numbers, so a v below 2^-96
// is scaled up first, by an even power of two.  (A zero, an infinity and a NaN
// compare false.)
__device__ __forceinline__ float root(float v) {
  const bool small = v < 0x1p-96f;
  v = small ? v * 0x1p96f : v;
  const float r = __builtin_amdgcn_sqrtf(v);
  const float below = __uint_as_float(__float_as_uint(r) - 1u);
  const float above = __uint_as_float(__float_as_uint(r) + 1u);
  float s = fmaf(-below, r, v) <= 0.f ? below : r;
  s = fmaf(-above, r, v) > 0.f ? above : s;
  return small ? s * 0x1p-48f : s;
}

// one element; r is sqrt(v')
__device__ __forceinline__ void adamw_element(const AdamwScalars& h,
                                              float coef, float g, float& p,
                                              float& m, float& v, float& r) {
  g = g * coef;
  m = m * h.beta1 + g * h.one_minus_beta1;
  v = v * h.beta2 + (g * g) * h.one_minus_beta2;
  r = root(v);
  // what reaches the weights alone
  const float q = m * __builtin_amdgcn_rcpf(fmaf(r, h.inv_root_bc2, h.eps));
  p = fmaf(-q, h.step_size, p * h.decay);
}

// 28 bytes an fp32 element (22 a 16-bit one) and some 30 operations: bound
// by memory.  All loads of a chunk are issued before the first is used (the
// barrier keeps the compiler from holding some back to save registers).
// 2e8 bf16 weights: 803 us, 5.5 TB/s, where a copy of 4 GB reaches 4.75.
template <typename T, bool ONCE>
__global__ __launch_bounds__(THREADS) void adamw_kernel(
    const AdamwTable tab, const AdamwScalars h, const float* norm) {
  constexpr int V = 16 / sizeof(T);
  constexpr int NV = CHUNK / (THREADS * V);
  const auto [t, at, left] = find_chunk(tab, blockIdx.x);
  T* p = (T*)tab.p[t] + at;
  const T* g = (const T*)tab.g[t] + at;
  float* m = (float*)tab.m[t] + at;
  float* v = (float*)tab.v[t] + at;
  const float coef = clip_coef(norm, h.max_norm);
  float gf[V], pf[V], mf[V], vf[V], r;
  const int i0 = threadIdx.x * V;
  if (left == CHUNK) {
    Raw<T, V> gr[NV], pr[NV];
    Raw<float, V> mr[NV], vr[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = i0 + j * THREADS * V;
      gr[j].template load<ONCE>(g + i);
      pr[j].template load<ONCE>(p + i);
      mr[j].template load<ONCE>(m + i);
      vr[j].template load<ONCE>(v + i);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = i0 + j * THREADS * V;
      gr[j].floats(gf);
      pr[j].floats(pf);
      mr[j].floats(mf);
      vr[j].floats(vf);
#pragma unroll
      for (int k = 0; k < V; ++k)
        adamw_element(h, coef, gf[k], pf[k], mf[k], vf[k], r);
      store_vec<ONCE>(p + i, pf);
      store_vec<ONCE>(m + i, mf);
      store_vec<ONCE>(v + i, vf);
    }
  } else {
    for (int i = i0; i < left; i += THREADS * V) {
      const int n = left - i;
      load_part(g + i, gf, n);
      load_part(p + i, pf, n);
      load_part(m + i, mf, n);
      load_part(v + i, vf, n);
#pragma unroll
      for (int k = 0; k < V; ++k)
        adamw_element(h, coef, gf[k], pf[k], mf[k], vf[k], r);
      store_part(p + i, pf, n);
      store_part(m + i, mf, n);
      store_part(v + i, vf, n);
    }
  }
}

// ---- 8-bit moments ---------------------------------------------------------
// m: an e4m3 code times the block's scale (its largest |m| / 448), rounded
// to nearest; b1 = 0.9 moves m by whole steps.
// v: kept as sqrt(v), which has half the octaves: an unsigned code of 4
// exponent and 4 fraction bits, value 2^(e-15) (1 + f/16) (e = 0: 2^-14
// f/16), times the block's scale (its largest root / 1.9375).  19 octaves,
// 38 of v.  Rounded stochastically: b2 = 0.999 moves sqrt(v) by 0.05% a
// step where codes are 3 to 6% apart, so rounding to nearest would hold it
// still.  A value above zero keeps a code above zero, since m / (sqrt(v) +
// eps) has no bound where v is lost and m is not.

__device__ __forceinline__ float decode_root(uint32_t code) {
  return __uint_as_float(code << 19) * 0x1p112f;
}

__device__ __forceinline__ uint32_t encode_root(float q, uint32_t dither) {
  const uint32_t c = (__float_as_uint(q * 0x1p-112f) + dither) >> 19;
  return min(max(c, min(__float_as_uint(q), 1u)), 255u);  // 1 if q > 0
}

// 19 random bits of one element: a multiplicative hash of its counter (the
// golden ratio's and sqrt(3)'s fractions as odd multipliers), folded twice
__device__ __forceinline__ uint32_t dither19(uint32_t x) {
  x *= 0x9E3779B9u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  x ^= x >> 16;
  return x >> 13;
}

// Largest of 16 neighbouring lanes.  On the bits of non-negative floats, so
// that a NaN is larger than every number and reaches the scale.
__device__ __forceinline__ uint32_t max16(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));
  x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));
  x = max(x,
          (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, true));
  x = max(x,
          (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x140, 0xF, 0xF, true));
  return x;
}

__device__ __forceinline__ void decode8(const uint2 mc, const uint2 vc,
                                        float (&m)[8], float (&r)[8]) {
  const uint32_t mw[2] = {mc.x, mc.y}, vw[2] = {vc.x, vc.y};
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const auto f = (k & 2)
        ? __builtin_amdgcn_cvt_pk_f32_fp8(mw[k / 4], true)
        : __builtin_amdgcn_cvt_pk_f32_fp8(mw[k / 4], false);
    m[k] = f[0];
    m[k + 1] = f[1];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    r[k] = decode_root((vw[k / 4] >> (8 * (k % 4))) & 255u);
}

__device__ __forceinline__ uint2 pack_m(const float (&q)[8]) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; k += 4) {
    int x = __builtin_amdgcn_cvt_pk_fp8_f32(q[k], q[k + 1], 0, false);
    w[k / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(q[k + 2], q[k + 3], x, true);
  }
  return make_uint2(w[0], w[1]);
}

// bytes [0, n) of a code word, zeros behind
typedef uint32_t word2 __attribute__((ext_vector_type(2), aligned(1)));
template <bool ONCE>
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int n) {
  uint2 w = make_uint2(0, 0);
  if (n >= 8) {
    const word2 x = ONCE ? __builtin_nontemporal_load((const word2*)p)
                         : *(const word2*)p;
    w = make_uint2(x.x, x.y);
  } else {
    for (int k = 0; k < n; ++k) {
      const uint32_t b = p[k];
      if (k < 4) w.x |= b << (8 * k);
      else w.y |= b << (8 * (k - 4));
    }
  }
  return w;
}

__device__ __forceinline__ void store_codes(uint8_t* p, uint2 w, int n) {
  if (n >= 8) {
    __builtin_memcpy(p, &w, 8);
  } else {
    for (int k = 0; k < n; ++k)
      p[k] = (uint8_t)((k < 4 ? w.x >> (8 * k) : w.y >> (8 * (k - 4))));
  }
}

// 16 lanes share a block of 256 elements: lane l holds elements l*8.. of
// each half, so that a wave reads whole lines and the block's maximum needs
// no shared memory (four DPP steps).  16 bytes an fp32 element (10 a 16-bit
// one) against some 65 operations, which leaves the vector units little to
// spare: 2e8 bf16 weights 361 us, 5.6 TB/s, of which the root's scaling of
// values below 2^-96 takes some 7; with the library's root and a rounded
// quotient they were the limit, at 430.  Codes go through the caches in any
// case: their next reader may find them there.
template <typename T, bool ONCE>
__global__ __launch_bounds__(THREADS) void adamw8_kernel(
    const AdamwTable tab, const AdamwScalars h, const float* norm,
    uint32_t seed) {
  const auto [t, at, left] = find_chunk(tab, blockIdx.x);
  T* p = (T*)tab.p[t] + at;
  const T* g = (const T*)tab.g[t] + at;
  uint8_t* m = (uint8_t*)tab.m[t] + at;
  uint8_t* v = (uint8_t*)tab.v[t] + at;
  const int b = threadIdx.x / 16, l = threadIdx.x % 16;
  float2* scale = (float2*)tab.s[t] + at / QBLOCK + b;
  const bool full = left == CHUNK;
  const float coef = clip_coef(norm, h.max_norm);
  const int i0 = b * QBLOCK + l * 8;
  const bool live = b * QBLOCK < left;  // the same for the 16 lanes
  float pf[2][8], gf[2][8], mf[2][8], rf[2][8];
  uint2 mc[2], vc[2];
  const float2 s = live ? *scale : make_float2(0.f, 0.f);
  if (full) {
    Raw<T, 8> gr[2], pr[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = i0 + j * 128;
      gr[j].template load<ONCE>(g + i);
      pr[j].template load<ONCE>(p + i);
      mc[j] = load_codes<false>(m + i, 8);
      vc[j] = load_codes<false>(v + i, 8);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 2; ++j) gr[j].floats(gf[j]), pr[j].floats(pf[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = i0 + j * 128;
      load_part(g + i, gf[j], left - i);
      load_part(p + i, pf[j], left - i);
      mc[j] = load_codes<false>(m + i, left - i);
      vc[j] = load_codes<false>(v + i, left - i);
    }
  }
  uint32_t top_m = __float_as_uint(TINY), top_r = __float_as_uint(TINY);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    decode8(mc[j], vc[j], mf[j], rf[j]);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float r = rf[j][k] * s.y;
      float v2 = r * r;
      mf[j][k] *= s.x;
      adamw_element(h, coef, gf[j][k], pf[j][k], mf[j][k], v2, rf[j][k]);
      top_m = max(top_m, __float_as_uint(mf[j][k]) & 0x7FFFFFFFu);
      top_r = max(top_r, __float_as_uint(rf[j][k]));
    }
  }
  float sm = __uint_as_float(max16(top_m)) * (float)(1.0 / 448.0);
  float sr = __uint_as_float(max16(top_r)) * (float)(1.0 / 1.9375);
  // an infinity in the block: all of it becomes a NaN, whatever the codes
  if (!(sm < INFINITY)) sm = NAN;
  if (!(sr < INFINITY)) sr = NAN;
  const float im = 1.f / sm, ir = 1.f / sr;
  const uint32_t key =
      seed + (tab.list_base + tab.number[t]) * 0x3C6EF372u + (uint32_t)at;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = i0 + j * 128;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      // (where this is a NaN so is the scale: the code says nothing)
      mf[j][k] = __builtin_amdgcn_fmed3f(mf[j][k] * im, -TOP_M, TOP_M);
      w[k / 4] |= encode_root(rf[j][k] * ir, dither19(key + i + k))
                  << (8 * (k % 4));
    }
    const uint2 mw = pack_m(mf[j]);
    if (full) {
      store_vec<ONCE>(p + i, pf[j]);
      store_codes(m + i, mw, 8);
      store_codes(v + i, make_uint2(w[0], w[1]), 8);
    } else {
      store_part(p + i, pf[j], left - i);
      store_codes(m + i, mw, left - i);
      store_codes(v + i, make_uint2(w[0], w[1]), left - i);
    }
  }
  if (live && l == 0) *scale = make_float2(sm, sr);
}

// the moments of 8-bit codes, into p (m) and g (v) of the table
template <typename T>
__global__ __launch_bounds__(THREADS) void adamw8_values_kernel(
    const AdamwTable tab) {
  const auto [t, at, left] = find_chunk(tab, blockIdx.x);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = (j * THREADS + threadIdx.x) * 8;
    const int n = left - i;
    if (n <= 0) break;
    const uint2 mc = load_codes<true>((const uint8_t*)tab.m[t] + at + i, n);
    const uint2 vc = load_codes<true>((const uint8_t*)tab.v[t] + at + i, n);
    const float2 s = ((const float2*)tab.s[t])[(at + i) / QBLOCK];
    float m[8], v[8];
    decode8(mc, vc, m, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] *= s.x;
      const float r = v[k] * s.y;
      v[k] = r * r;
    }
    T* om = (T*)tab.p[t] + at + i;
    T* ov = (T*)const_cast<void*>(tab.g[t]) + at + i;
    if (n >= 8) {
      store_vec<true>(om, m);
      store_vec<true>(ov, v);
    } else {
      store_part(om, m, n);
      store_part(ov, v, n);
    }
  }
}

// ---- gradient norm ---------------------------------------------------------
// Squares and sums in 64 bits: a square of a 32-bit value is exact there,
// and the order of the sum hardly ever reaches the 32-bit result (its value
// would have to lie within some 2^-42 of a border between two).  The order is
// that of the list, so the same list gives the same bits.  Bound by reading 4
// (2) bytes an element: 300 MB in bf16 take 53 us, 5.7 TB/s.

// root of the sum over a workgroup of 1024
__device__ __forceinline__ void finish_norm(double acc, float* out) {
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, WAVE);
  __shared__ double part[1024 / WAVE];
  if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = acc;
  __syncthreads();
  if (threadIdx.x != 0) return;
  acc = 0.0;
#pragma unroll
  for (int i = 0; i < 1024 / WAVE; ++i) acc += part[i];
  *out = (float)sqrt(acc);
}

template <typename T, bool ONCE>
__global__ __launch_bounds__(THREADS) void sumsq_kernel(
    const GradTable tab, double* __restrict__ partial) {
  constexpr int V = 16 / sizeof(T);
  constexpr int NV = CHUNK / (THREADS * V);
  double acc = 0.0;
  float gf[V];
  for (uint32_t c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
    const auto [t, at, left] = find_chunk(tab, c);
    const T* g = (const T*)tab.g[t] + at + threadIdx.x * V;
    if (left == CHUNK) {
      Raw<T, V> r[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j)
        r[j].template load<ONCE>(g + j * THREADS * V);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        r[j].floats(gf);
#pragma unroll
        for (int k = 0; k < V; ++k) acc += (double)gf[k] * (double)gf[k];
      }
    } else {
      for (int i = threadIdx.x * V; i < left; i += THREADS * V) {
        load_part((const T*)tab.g[t] + at + i, gf, left - i);
#pragma unroll
        for (int k = 0; k < V; ++k) acc += (double)gf[k] * (double)gf[k];
      }
    }
  }
  for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off, WAVE);
  __shared__ double part[THREADS / WAVE];
  if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = acc;
  __syncthreads();
  if (threadIdx.x == 0)
    partial[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// Up to NORM_SMALL_CHUNKS chunks in one launch: a wave takes a chunk, with 8
// loads a lane on their way, one workgroup all of them.  With so few it is
// the launches that count: 4096 fp32 elements take 5.5 us instead of 9.5, 32
// chunks 7.0 instead of 9.6, and a few more would take longer than two
// launches.
template <typename T>
__global__ __launch_bounds__(1024) void norm_small_kernel(
    const GradTable tab, float* __restrict__ out) {
  constexpr int V = 16 / sizeof(T);
  constexpr int NV = 8;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int lane = threadIdx.x % WAVE;
  double acc = 0.0;
  float gf[V];
  for (uint32_t c = wave; c < tab.chunks; c += 1024 / WAVE) {
    const auto [t, at, left] = find_chunk(tab, c);
    const T* g = (const T*)tab.g[t] + at;
    int i = lane * V;
    for (; left == CHUNK && i < CHUNK; i += NV * WAVE * V) {
      Raw<T, V> r[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j)
        r[j].template load<false>(g + i + j * WAVE * V);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        r[j].floats(gf);
#pragma unroll
        for (int k = 0; k < V; ++k) acc += (double)gf[k] * (double)gf[k];
      }
    }
    for (; i < left; i += WAVE * V) {
      load_part(g + i, gf, left - i);
#pragma unroll
      for (int k = 0; k < V; ++k) acc += (double)gf[k] * (double)gf[k];
    }
  }
  finish_norm(acc, out);
}

// (1024 threads: a launch's 2048 partial sums at most are two loads a thread)
__global__ __launch_bounds__(1024) void norm_final_kernel(
    const double* __restrict__ partial, int n, float* __restrict__ out) {
  double acc = 0.0;
#pragma unroll 2
  for (int i = threadIdx.x; i < n; i += 1024) acc += partial[i];
  finish_norm(acc, out);
}

template <typename T>
void go_adamw(hipStream_t s, const AdamwTable& tab, const AdamwScalars& h,
              const float* norm, bool once) {
  if (once)
    adamw_kernel<T, true><<<dim3(tab.chunks), THREADS, 0, s>>>(tab, h, norm);
  else
    adamw_kernel<T, false><<<dim3(tab.chunks), THREADS, 0, s>>>(tab, h, norm);
}

template <typename T>
void go_adamw8(hipStream_t s, const AdamwTable& tab, const AdamwScalars& h,
               const float* norm, bool once, uint32_t seed) {
  if (once)
    adamw8_kernel<T, true>
        <<<dim3(tab.chunks), THREADS, 0, s>>>(tab, h, norm, seed);
  else
    adamw8_kernel<T, false>
        <<<dim3(tab.chunks), THREADS, 0, s>>>(tab, h, norm, seed);
}

template <typename T>
void go_values(hipStream_t s, const AdamwTable& tab) {
  adamw8_values_kernel<T><<<dim3(tab.chunks), THREADS, 0, s>>>(tab);
}

template <typename T>
void go_sumsq(hipStream_t s, const GradTable& tab, double* partial,
              int blocks, bool once) {
  if (once)
    sumsq_kernel<T, true><<<dim3(blocks), THREADS, 0, s>>>(tab, partial);
  else
    sumsq_kernel<T, false><<<dim3(blocks), THREADS, 0, s>>>(tab, partial);
}

template <typename T>
void go_small(hipStream_t s, const GradTable& tab, float* out) {
  norm_small_kernel<T><<<dim3(1), 1024, 0, s>>>(tab, out);
}

#define BY_DTYPE(dtype, fn, ...)                        \
  switch (dtype) {                                      \
    case 0: fn<float>(__VA_ARGS__); break;              \
    case 1: fn<__bf16>(__VA_ARGS__); break;             \
    case 2: fn<_Float16>(__VA_ARGS__); break;           \
    default: return (int)hipErrorInvalidValue;          \
  }

}  // namespace

extern "C" int launch_adamw(void* stream, const AdamwTable* tab,
                            const AdamwScalars* h, const float* norm,
                            int dtype, bool once) {
  if (tab->chunks == 0) return 0;
  BY_DTYPE(dtype, go_adamw, (hipStream_t)stream, *tab, *h, norm, once)
  HIP_CHECK_LAST();
  return 0;
}

extern "C" int launch_adamw8(void* stream, const AdamwTable* tab,
                             const AdamwScalars* h, const float* norm,
                             int dtype, bool once, uint32_t seed) {
  if (tab->chunks == 0) return 0;
  BY_DTYPE(dtype, go_adamw8, (hipStream_t)stream, *tab, *h, norm, once,
           seed)
  HIP_CHECK_LAST();
  return 0;
}

extern "C" int launch_adamw8_values(void* stream, const AdamwTable* tab,
                                    int dtype) {
  if (tab->chunks == 0) return 0;
  BY_DTYPE(dtype, go_values, (hipStream_t)stream, *tab)
  HIP_CHECK_LAST();
  return 0;
}

extern "C" int launch_sumsq(void* stream, const GradTable* tab, int dtype,
                            double* partial, int blocks, bool once) {
  if (tab->chunks == 0 || blocks == 0) return 0;
  BY_DTYPE(dtype, go_sumsq, (hipStream_t)stream, *tab, partial, blocks, once)
  HIP_CHECK_LAST();
  return 0;
}

extern "C" int launch_norm_final(void* stream, const double* partial, int n,
                                 float* out) {
  norm_final_kernel<<<dim3(1), 1024, 0, (hipStream_t)stream>>>(partial, n,
                                                               out);
  HIP_CHECK_LAST();
  return 0;
}

extern "C" int launch_norm_small(void* stream, const GradTable* tab,
                                 int dtype, float* out) {
  if (tab->chunks > NORM_SMALL_CHUNKS) return (int)hipErrorInvalidValue;
  BY_DTYPE(dtype, go_small, (hipStream_t)stream, *tab, out)
  HIP_CHECK_LAST();
  return 0;
}
