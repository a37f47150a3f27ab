// The norms after and before a residual block, with its gate and residual
// scale, in one pass over a row:
//
//   n = post(h)                    RMSNorm, LayerNorm or nothing
//   r = x + scale * act(gate) * n  gate per element or per row
//   y = pre(r)                     of r before it is rounded
//
// A norm is hat * w + b with hat = (v - mean) * rstd over the row; an RMSNorm
// has mean = 0.  Statistics are 32-bit and taken in two passes over the
// registers that hold the row (mean, then centred squares).
//
// Backward, with d_r and d_y given and r, hats recomputed in 32 bits from the
// inputs and the saved statistics:
//
//   t  = d_y w2;   d = d_r + rstd_r (t - [mean t] - rhat mean(t rhat));  dx = d
//   dn = d scale a;   dgate = act'(gate) d scale n (summed over a row's gate)
//   t1 = dn w1;    dh = rstd_h (t1 - [mean t1] - hhat mean(t1 hhat))
//   over rows: S0 = sum d a hhat, S1 = sum d a, S2 = sum d_y rhat, S3 = sum d_y
//   dw1 = scale S0, db1 = scale S1, dscale = w1 S0 + b1 S1, dw2 = S2, db2 = S3
//   ([..], S1 and S3 only with a LayerNorm)
//
// Both directions are bound by memory: each input is read and each output
// written once.  NT threads share a row, 8 neighbouring elements a thread
// and K such groups, so that the row stays in registers between its
// reductions.  Column sums stay in registers over a workgroup's rows, go to
// memory once per workgroup, and a second kernel adds those: no atomics, the
// same bits every time.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "launchers.h"

namespace {

constexpr int BLOCK = 256;  // threads of a workgroup, at least
// threads of a forward grid at most: 1024 on each of 256 CUs, which is what
// their registers let be there at once; beyond that workgroups take more rows
constexpr int FWD_THREADS = 256 * 1024;

// V elements as they lie in memory: registers hold whole words until an
// element is used, so that several loads are on their way at once
template <typename T, int V>
struct Raw {
  static constexpr int N = V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1;
  uint32_t w[N];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __bf16>::value) {
      return __uint_as_float(i % 2 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    } else {
      const uint16_t u = (uint16_t)(i % 2 ? w[i / 2] >> 16 : w[i / 2]);
      return (float)__builtin_bit_cast(_Float16, u);
    }
  }
};

// The V neighbouring elements that a thread has of a row.  Where the width is
// no multiple of V the last thread's begin early enough to end with the row:
// it then has `skip` elements in common with its neighbour, computes and
// stores the same values for them, and leaves them out of row sums.  So every
// access is a whole vector (of the element's own alignment).  A thread that
// has none (skip = V) reads the row's first, and stores nothing.
template <int V>
struct Cols {
  uint32_t col;
  int skip;
  __device__ __forceinline__ void set(int c0, int width, bool row = true) {
    const bool live = row && c0 < width;
    const int c = min(c0, width - V);
    col = live ? c : 0;
    skip = live ? c0 - c : V;
  }
  __device__ __forceinline__ bool live() const { return skip < V; }
};

// off (to the row) is the same for a wave: it stays in scalar registers, and
// one 32-bit offset serves all arrays of a type.  The empty asm keeps the
// offset's widening to 64 bits beside the access, where it is part of the
// instruction; moved out of the row loop it costs two registers an array (141
// instead of 126 in the backward pass, a workgroup a CU less).
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const void* base, int64_t off,
                                              const Cols<V>& c,
                                              bool wanted = true) {
  Raw<T, V> r;
  if (wanted) {
    uint32_t at = c.col * (uint32_t)sizeof(T);
    asm volatile("" : "+v"(at));
    const char* p = (const char*)base + off * (int64_t)sizeof(T) + at;
    if constexpr (V * sizeof(T) < 4) {
      uint16_t u;
      __builtin_memcpy(&u, p, 2);
      r.w[0] = u;
    } else {
      __builtin_memcpy(r.w, p, sizeof(r.w));
    }
  } else {
#pragma unroll
    for (int i = 0; i < Raw<T, V>::N; ++i) r.w[i] = 0;
  }
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_f(void* base, int64_t off,
                                        const Cols<V>& c,
                                        const float (&f)[V]) {
  T r[V];
  char* p = (char*)base + off * (int64_t)sizeof(T);
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = (T)f[i];  // to nearest even
  uint32_t at = c.col * (uint32_t)sizeof(T);
  asm volatile("" : "+v"(at));
  if (c.live()) __builtin_memcpy(p + at, r, sizeof(r));
}

// a per-channel vector (fp32 or TH), or a constant
template <typename TH, int V>
__device__ __forceinline__ void load_vec(const void* p, bool f32,
                                         const Cols<V>& c, float none,
                                         float (&out)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = none;
  } else if (f32) {
    const Raw<float, V> r = load_raw<float>(p, 0, c);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = r[i];
  } else {
    const Raw<TH, V> r = load_raw<TH>(p, 0, c);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = r[i];
  }
}

// Sum over the N lanes (8 to 64) that share a row, the same in all of them:
// inside rows of 16 lanes by DPP, a wave's four through scalar registers.
// (Six ds_bpermute steps take some 400 cycles of latency, twice or more a
// row.)
template <int N>
__device__ __forceinline__ float lane_sum(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(
        0, __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>());   // lane ^ 1
  v += dpp(v, std::integral_constant<int, 0x4E>());   // lane ^ 2
  v += dpp(v, std::integral_constant<int, 0x141>());  // half row mirrored
  if constexpr (N >= 16)
    v += dpp(v, std::integral_constant<int, 0x140>());  // row mirrored
  if constexpr (N == 32) v += __shfl_xor(v, 16, WAVE);
  if constexpr (N < WAVE) return v;
  const int b = __float_as_int(v);
  return (__int_as_float(__builtin_amdgcn_readlane(b, 0)) +
          __int_as_float(__builtin_amdgcn_readlane(b, 16))) +
         (__int_as_float(__builtin_amdgcn_readlane(b, 32)) +
          __int_as_float(__builtin_amdgcn_readlane(b, 48)));
}

// the group of NT threads that this one belongs to: where that is whole
// waves, in a scalar register, and so is what is made of it
template <int NT>
__device__ __forceinline__ int group_of() {
  return NT < WAVE ? threadIdx.x / NT
                   : __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
}

// sums of M values over the NT threads of a row, in a fixed order
template <int NT, int M>
struct RowSum {
  static constexpr int WAVES = NT / WAVE;  // of this row (0: part of one)
  // two slots in turn: one barrier a reduction
  float slot[2][M][WAVES > 1 ? WAVES : 1];

  __device__ __forceinline__ void operator()(float (&v)[M], int turn) {
#pragma unroll
    for (int j = 0; j < M; ++j) v[j] = lane_sum<(NT < WAVE ? NT : WAVE)>(v[j]);
    if constexpr (WAVES > 1) {
      const int wave = threadIdx.x / WAVE % WAVES;
      if (threadIdx.x % WAVE == 0)
#pragma unroll
        for (int j = 0; j < M; ++j) slot[turn & 1][j][wave] = v[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < M; ++j) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s += slot[turn & 1][j][w];
        v[j] = s;
      }
    }
  }
};

// 1 / (1 + exp(-g)) by the hardware's exp2 and reciprocal: off by
// (5 + 1.25 |g|) U of itself, U = 2^-24: an ulp (2U) each and U for the sum,
// and g log2(e) is off by its rounding, U, and its constant's, 0.22 U, which
// the exponential makes |g| times as much.  An eighth of expf's and a
// division's instructions.
__device__ __forceinline__ float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(
      1.f + __builtin_amdgcn_exp2f(g * -1.44269504088896341f));
}

// s[] becomes act(g), g[] becomes act'(g)
template <int V>
__device__ __forceinline__ void activate(int act, float (&g)[V],
                                         float (&s)[V]) {
  if (act == NORM_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float sig = sigmoid(g[i]);
      s[i] = g[i] * sig;
      g[i] = sig + s[i] * (1.f - sig);
    }
  } else if (act == NORM_ACT_SIGMOID) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[i] = sigmoid(g[i]);
      g[i] = s[i] * (1.f - s[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[i] = g[i];
      g[i] = 1.f;
    }
  }
}

// mean (LayerNorm) and 1/std of a row held as f[K][V]
template <int NT, int K, int V, bool LAYER>
__device__ __forceinline__ void row_stats(const float (&f)[K][V],
                                          const Cols<V> (&c)[K], int kind,
                                          float inv_c, float eps,
                                          RowSum<NT, 1>& sum, int& turn,
                                          float& mean, float& rstd) {
  float s[1] = {0.f};
  mean = 0.f;
  if (LAYER && kind == NORM_LAYER) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += i >= c[k].skip ? f[k][i] : 0.f;
    sum(s, turn++);
    mean = s[0] * inv_c;
    s[0] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = i >= c[k].skip ? f[k][i] - mean : 0.f;
      s[0] += d * d;
    }
  sum(s, turn++);
  rstd = rsqrtf(s[0] * inv_c + eps);
}

// a row's inputs on their way
template <typename TX, typename TH, int K, int V>
struct FwdRow {
  Raw<TX, V> x[K];
  Raw<TH, V> h[K], g[K];
  float row_gate;

  __device__ __forceinline__ void load(const NormArgs& a, int64_t row,
                                       const Cols<V> (&c)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x[k] = load_raw<TX>(a.x, row * a.ld_x, c[k]);
      h[k] = load_raw<TH>(a.h, row * a.ld_h, c[k], a.h != nullptr);
      g[k] = load_raw<TH>(a.gate, row * a.ld_g, c[k],
                          a.gate_kind == NORM_GATE_FULL);
    }
    row_gate = a.gate_kind == NORM_GATE_ROW
                   ? (float)((const TH*)a.gate)[row * a.ld_g]
                   : 1.f;
  }
};

// LAYER: whether one norm is a LayerNorm.  A workgroup keeps its columns'
// weights in registers (K = 1) over its rows, and the next row's inputs are on
// their way while this one's sums are taken.  16384 x 4096 bf16, gated: 125
// us, 5.4 TB/s, where a copy of 4 GB reaches 4.75 (one row a workgroup, its
// weights read each time: 170 us).  Above 8192 columns (K = 2) 4.0 TB/s; fp32
// blocks spill 4 to 10 registers there.
template <typename TX, typename TH, int NT, int K, int V, bool LAYER>
__global__ __launch_bounds__(NT < BLOCK ? BLOCK : NT) void norm_fwd_kernel(
    const NormArgs a) {
  constexpr int GROUPS = NT < BLOCK ? BLOCK / NT : 1;
  constexpr bool KEEP = K == 1;
  __shared__ RowSum<NT, 1> sums[GROUPS];
  const int group = group_of<NT>();
  const int t = threadIdx.x % NT;
  RowSum<NT, 1>& sum = sums[group];
  int turn = 0;
  const float inv_c = 1.f / (float)a.width;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  // the groups of a workgroup take the same turns (they share barriers); one
  // that is behind the last row repeats that row and stores nothing
  int64_t base = (int64_t)blockIdx.x * GROUPS;
  auto row_of = [&](int64_t b) {
    return b + group < a.rows ? b + group : a.rows - 1;
  };
  Cols<V> c[K];
#pragma unroll
  for (int k = 0; k < K; ++k) c[k].set((k * NT + t) * V, a.width);
  FwdRow<TX, TH, K, V> next;
  next.load(a, row_of(base), c);
  float w1[K][V], b1[K][V], w2[K][V], b2[K][V], sc[K][V];
  auto vectors = [&](int k) {
    load_vec<TH>(a.w1, a.f32 & 1, c[k], 1.f, w1[k]);
    if (LAYER) load_vec<TH>(a.b1, a.f32 & 2, c[k], 0.f, b1[k]);
    load_vec<TH>(a.w2, a.f32 & 4, c[k], 1.f, w2[k]);
    if (LAYER) load_vec<TH>(a.b2, a.f32 & 8, c[k], 0.f, b2[k]);
    load_vec<TH>(a.scale, a.f32 & 16, c[k], a.scale_value, sc[k]);
  };
  if (KEEP) vectors(0);
  for (; base < a.rows; base += step) {
    const bool in = base + group < a.rows;
    const int64_t row = row_of(base);
    FwdRow<TX, TH, K, V> cur = next;
    if (base + step < a.rows) next.load(a, row_of(base + step), c);
    float f[K][V];  // h, later r
    if (a.h == nullptr) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) f[k][i] = cur.x[k][i];
    } else {
      float row_slope[1] = {cur.row_gate}, row_act[1] = {1.f};
      if (a.gate_kind == NORM_GATE_ROW)
        activate(a.act, row_slope, row_act);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) f[k][i] = cur.h[k][i];
      float mean = 0.f, rstd = 1.f;
      if (a.post != NORM_NONE) {
        row_stats<NT, K, V, LAYER>(f, c, a.post, inv_c, a.post_eps, sum, turn,
                                   mean, rstd);
        if (t == 0 && in && a.stats != nullptr) {
          a.stats[row] = mean;
          a.stats[a.rows + row] = rstd;
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!KEEP) vectors(k);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          f[k][i] = (LAYER ? f[k][i] - mean : f[k][i]) * (rstd * w1[k][i]);
          if (LAYER) f[k][i] += b1[k][i];
        }
        float act[V], slope[V];
#pragma unroll
        for (int i = 0; i < V; ++i) act[i] = row_act[0];
        if (a.gate_kind == NORM_GATE_FULL) {
#pragma unroll
          for (int i = 0; i < V; ++i) slope[i] = cur.g[k][i];
          activate(a.act, slope, act);
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
          f[k][i] = cur.x[k][i] + sc[k][i] * act[i] * f[k][i];
        if (in) store_f<TX>(a.r, row * a.width, c[k], f[k]);
      }
    }
    if (a.pre == NORM_NONE) continue;
    float mean, rstd;
    row_stats<NT, K, V, LAYER>(f, c, a.pre, inv_c, a.pre_eps, sum, turn, mean,
                               rstd);
    if (t == 0 && in && a.stats != nullptr) {
      a.stats[2 * a.rows + row] = mean;
      a.stats[3 * a.rows + row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!KEEP) vectors(k);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[k][i] = (LAYER ? f[k][i] - mean : f[k][i]) * (rstd * w2[k][i]);
        if (LAYER) f[k][i] += b2[k][i];
      }
      if (in) store_f<TH>(a.y, row * a.width, c[k], f[k]);
    }
  }
}

// Column sums of a workgroup, S0 to S3
constexpr int SUMS = 4;

// LAYER: whether one norm is a LayerNorm (or has a bias).  What bounds this
// pass after memory is the number of vector instructions, some 50 an element,
// and registers, which bound how many rows are on their way per CU.  So hats
// and weighted values are made again rather than kept, and the weights are
// read from LDS (K = 1), where a workgroup puts them once.  16384 x 4096
// bf16, gated: 205 us, 5.2 TB/s (321 us with twice the instructions and the
// weights from L2).  Above 8192 columns (K = 2) the registers do not suffice
// for two vectors a thread, and 44 to 306 are spilled: 2048 x 16384 194 us, 2.8
// TB/s.  (Two LayerNorm forms under an fp32 stream spill one or two from 4097
// columns on.)
template <typename TX, typename TH, int NT, int K, int V, bool LAYER>
__global__ __launch_bounds__(NT < BLOCK ? BLOCK : NT,
                             LAYER && NT < 1024 ? 3 : 4) void
norm_bwd_kernel(const NormArgs a, const NormGrads o) {
  constexpr int GROUPS = NT < BLOCK ? BLOCK / NT : 1;
  constexpr bool KEEP = K == 1;
  constexpr int KEPT = LAYER ? 4 : 3;  // w1, scale, w2, b1
  constexpr int P = LAYER ? 2 : 1, Q3 = LAYER ? 3 : 2;  // row sums of a step
  __shared__ RowSum<NT, P> pre_sums[GROUPS];
  __shared__ RowSum<NT, Q3> post_sums[GROUPS];
  // [vector][four elements][thread]: neighbouring threads' reads of 16 bytes
  // lie side by side
  constexpr int Q = V >= 4 ? V / 4 : 1, W = V / Q;
  __shared__ float kept[KEEP ? KEPT : 1][KEEP ? Q : 1][KEEP ? NT : 1][W];
  __shared__ float across[GROUPS > 1 ? GROUPS : 1]
                         [GROUPS > 1 ? NT * K * V : 1];
  const int group = group_of<NT>();
  const int t = threadIdx.x % NT;
  RowSum<NT, P>& pre_sum = pre_sums[group];
  RowSum<NT, Q3>& post_sum = post_sums[group];
  const float inv_c = 1.f / (float)a.width;
  const bool full = a.gate_kind == NORM_GATE_FULL;
  const bool per_row = a.gate_kind == NORM_GATE_ROW;
  Cols<V> c[K];
#pragma unroll
  for (int k = 0; k < K; ++k) c[k].set((k * NT + t) * V, a.width);
  auto fetch = [&](int which, int k, float (&v)[V]) {
    switch (which) {
      case 0: load_vec<TH>(a.w1, a.f32 & 1, c[k], 1.f, v); break;
      case 1: load_vec<TH>(a.scale, a.f32 & 16, c[k], a.scale_value, v); break;
      case 2: load_vec<TH>(a.w2, a.f32 & 4, c[k], 1.f, v); break;
      default: load_vec<TH>(a.b1, a.f32 & 2, c[k], 0.f, v); break;
    }
  };
  if constexpr (KEEP) {
    if (group == 0) {
#pragma unroll
      for (int j = 0; j < KEPT; ++j) {
        float v[V];
        fetch(j, 0, v);
#pragma unroll
        for (int i = 0; i < V; ++i) kept[j][i / W][t][i % W] = v[i];
      }
    }
    __syncthreads();
  }
  auto vec = [&](int which, int k, float (&v)[V]) {
    if constexpr (KEEP) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = kept[which][i / W][t][i % W];
    } else {
      fetch(which, k, v);
    }
  };
  float acc[SUMS][K][V];
#pragma unroll
  for (int j = 0; j < SUMS; ++j)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[j][k][i] = 0.f;
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  // AHEAD: the next row's inputs are on their way during this one, where the
  // registers hold them (4096 x 8192 117 to 112 us)
  constexpr bool AHEAD = !LAYER && K == 1 && sizeof(TX) == 2;
  struct In {
    Raw<TX, V> x[K], dr[K];
    Raw<TH, V> h[K], g[K], dy[K];
  } next;
  auto fetch_row = [&](In& n, int64_t base) {
    const bool in = base + group < a.rows;
    const int64_t row = in ? base + group : a.rows - 1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      n.x[k] = load_raw<TX>(a.x, row * a.ld_x, c[k], o.d_y != nullptr);
      n.h[k] = load_raw<TH>(a.h, row * a.ld_h, c[k], a.h != nullptr);
      n.g[k] = load_raw<TH>(a.gate, row * a.ld_g, c[k], full);
      // zeros behind the last row: nothing is added to the column sums
      n.dr[k] = load_raw<TX>(o.d_r, row * a.width, c[k],
                             o.d_r != nullptr && in);
      n.dy[k] = load_raw<TH>(o.d_y, row * a.width, c[k],
                             o.d_y != nullptr && in);
    }
  };
  if (AHEAD) fetch_row(next, (int64_t)blockIdx.x * GROUPS);
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < a.rows;
       base += step, ++turn) {
    const bool in = base + group < a.rows;
    const int64_t row = in ? base + group : a.rows - 1;
    In cur;
    if (AHEAD) {
      cur = next;
      if (base + step < a.rows) fetch_row(next, base + step);
    } else {
      fetch_row(cur, base);
    }
    auto &x = cur.x, &dr = cur.dr;
    auto &h = cur.h, &g = cur.g, &dy = cur.dy;
    float mean_h = 0.f, rstd_h = 1.f, mean_r = 0.f, rstd_r = 0.f;
    if (a.h != nullptr && a.post != NORM_NONE) {
      if (LAYER) mean_h = a.stats[row];
      rstd_h = a.stats[a.rows + row];
    }
    if (o.d_y != nullptr) {
      if (LAYER) mean_r = a.stats[2 * a.rows + row];
      rstd_r = a.stats[3 * a.rows + row];
    }
    float row_act[1] = {1.f}, row_slope[1] = {0.f};
    if (per_row) {
      row_slope[0] = (float)((const TH*)a.gate)[row * a.ld_g];
      activate(a.act, row_slope, row_act);
    }
    float d[K][V], act[V], slope[V];
    auto gate = [&](int k) {
#pragma unroll
      for (int i = 0; i < V; ++i) act[i] = row_act[0], slope[i] = 1.f;
      if (full) {
#pragma unroll
        for (int i = 0; i < V; ++i) slope[i] = g[k][i];
        activate(a.act, slope, act);
      }
    };
    if (K == 1) gate(0);
    auto hat_h = [&](int k, int i) {
      return (LAYER ? h[k][i] - mean_h : h[k][i]) * rstd_h;
    };
    // the norm before the next block: its row sums need r
    float p[P] = {};
    if (o.d_y != nullptr) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float v[V];
        if (K > 1) gate(k);
        if (a.h != nullptr) {
          vec(0, k, v);
#pragma unroll
          for (int i = 0; i < V; ++i) d[k][i] = hat_h(k, i) * v[i];
          if (LAYER) {
            vec(3, k, v);
#pragma unroll
            for (int i = 0; i < V; ++i) d[k][i] += v[i];
          }
          vec(1, k, v);
#pragma unroll
          for (int i = 0; i < V; ++i)
            d[k][i] = x[k][i] + v[i] * act[i] * d[k][i];
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) d[k][i] = x[k][i];
        }
        vec(2, k, v);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          d[k][i] = (LAYER ? d[k][i] - mean_r : d[k][i]) * rstd_r;  // hat
          const float tt = i >= c[k].skip ? dy[k][i] * v[i] : 0.f;
          acc[2][k][i] += dy[k][i] * d[k][i];
          if (LAYER) acc[3][k][i] += dy[k][i];
          p[0] += tt * d[k][i];
          if constexpr (LAYER) p[1] += tt;
        }
      }
      pre_sum(p, turn);
      p[0] *= inv_c;
      if constexpr (LAYER) p[1] = a.pre == NORM_LAYER ? p[1] * inv_c : 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float v[V];
        vec(2, k, v);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float back = dy[k][i] * v[i] - d[k][i] * p[0];
          d[k][i] = dr[k][i] + rstd_r * (LAYER ? back - p[P - 1] : back);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) d[k][i] = dr[k][i];
    }
    if (o.d_x != nullptr && in) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        store_f<TX>(o.d_x, row * a.width, c[k], d[k]);
    }
    if (a.h == nullptr) continue;
    // the gate, the scale and the norm after the block
    float q[Q3] = {};  // of t1 hhat, of the gate, of t1
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float w[V], s[V], nf[V];
      if (K > 1) gate(k);
      vec(0, k, w);
#pragma unroll
      for (int i = 0; i < V; ++i) nf[i] = hat_h(k, i) * w[i];
      if (LAYER) {
        float b[V];
        vec(3, k, b);
#pragma unroll
        for (int i = 0; i < V; ++i) nf[i] += b[i];
      }
      vec(1, k, s);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float da = d[k][i] * act[i];
        slope[i] *= d[k][i] * s[i] * nf[i];
        acc[0][k][i] += da * hat_h(k, i);
        if (LAYER) acc[1][k][i] += da;
        d[k][i] = da * s[i] * w[i];  // t1 from here on
        const float t1 = i >= c[k].skip ? d[k][i] : 0.f;
        q[0] += t1 * hat_h(k, i);
        if constexpr (LAYER) q[2] += t1;
      }
      if (full && o.d_gate != nullptr && in)
        store_f<TH>(o.d_gate, row * a.width, c[k], slope);
      if (per_row) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          q[1] += i >= c[k].skip ? slope[i] : 0.f;
      }
    }
    if (a.post != NORM_NONE || per_row) post_sum(q, turn);
    if (per_row && o.d_gate != nullptr && t == 0 && in)
      ((TH*)o.d_gate)[row] = (TH)(q[1] * row_slope[0]);
    if (o.d_h == nullptr || !in) continue;
    const float m1 = a.post != NORM_NONE ? q[0] * inv_c : 0.f;
    const float m0 =
        LAYER && a.post == NORM_LAYER ? q[Q3 - 1] * inv_c : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float back = d[k][i] - hat_h(k, i) * m1;
        d[k][i] = rstd_h * (LAYER ? back - m0 : back);
      }
      store_f<TH>(o.d_h, row * a.width, c[k], d[k]);
    }
  }
  // the workgroup's column sums: its groups' are added in LDS first
#pragma unroll
  for (int j = 0; j < SUMS; ++j) {
    if (o.partial[j] == nullptr) continue;
    float* out = o.partial[j] + (int64_t)blockIdx.x * a.width;
    if constexpr (GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k)
        store_f<float>(across[group], 0, c[k], acc[j][k]);
      __syncthreads();
      for (int i = threadIdx.x; i < a.width; i += BLOCK) {
        float s = 0.f;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) s += across[gr][i];
        out[i] = s;
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) store_f<float>(out, 0, c[k], acc[j][k]);
    }
  }
}

__device__ __forceinline__ void store_any(void* p, int type, int c, float f) {
  switch (type) {
    case 0: ((float*)p)[c] = f; break;
    case 1: ((__bf16*)p)[c] = (__bf16)f; break;
    default: ((_Float16*)p)[c] = (_Float16)f; break;
  }
}

// a vector of fp32 or the block's type, or a constant
__device__ __forceinline__ float load_any(const void* p, int type, int c,
                                          float none) {
  if (p == nullptr) return none;
  return type == 0   ? ((const float*)p)[c]
         : type == 1 ? (float)((const __bf16*)p)[c]
                     : (float)((const _Float16*)p)[c];
}

// The workgroups' column sums added, and the vectors' gradients of them.  A
// workgroup has 32 columns (a line of memory) and adds S0 and S1, or S2 and
// S3; 32 parts of the rows of partial sums side by side with 8 loads each on
// their way (16 parts and one load at a time took 10 us for 512 rows of any
// width).
__global__ __launch_bounds__(1024) void norm_columns_kernel(
    const NormArgs a, const NormGrads o, int blocks) {
  const int lane = threadIdx.x % 32, part = threadIdx.x / 32;
  const bool in = (int)blockIdx.x * 32 + lane < a.width;
  const int c = in ? blockIdx.x * 32 + lane : a.width - 1;
  const int first = 2 * blockIdx.y;
  __shared__ float lds[2][32][33];
  for (int j = 0; j < 2; ++j) {
    const float* p = o.partial[first + j];
    float s = 0.f;
    if (p != nullptr) {
      p += c;
      int b = part;
      for (; b + 7 * 32 < blocks; b += 8 * 32) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = p[(int64_t)(b + i * 32) * a.width];
#pragma unroll
        for (int i = 0; i < 8; ++i) s += f[i];
      }
      for (; b < blocks; b += 32) s += p[(int64_t)b * a.width];
    }
    lds[j][part][lane] = s;
  }
  __syncthreads();
  if (part != 0 || !in) return;
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    s[0] += lds[0][j][lane];
    s[1] += lds[1][j][lane];
  }
  const int t = a.type_h;
  auto type = [&](int bit) { return a.f32 >> bit & 1 ? 0 : t; };
  if (first) {
    if (o.d_w2 != nullptr) store_any(o.d_w2, type(2), c, s[0]);
    if (o.d_b2 != nullptr) store_any(o.d_b2, type(3), c, s[1]);
    return;
  }
  const float w = load_any(a.w1, type(0), c, 1.f);
  const float b = load_any(a.b1, type(1), c, 0.f);
  const float scale = load_any(a.scale, type(4), c, a.scale_value);
  if (o.d_w1 != nullptr) store_any(o.d_w1, type(0), c, scale * s[0]);
  if (o.d_b1 != nullptr) store_any(o.d_b1, type(1), c, scale * s[1]);
  if (o.d_scale != nullptr)
    store_any(o.d_scale, type(4), c,
              a.b1 != nullptr ? w * s[0] + b * s[1] : w * s[0]);
}

template <typename TX, typename TH, int NT, int K, int V>
void go(hipStream_t s, const NormArgs& a, const NormGrads* o, int blocks) {
  constexpr int GROUPS = NT < BLOCK ? BLOCK / NT : 1;
  constexpr int THREADS = NT < BLOCK ? BLOCK : NT;
  const bool layer = a.post == NORM_LAYER || a.pre == NORM_LAYER;
  if (o == nullptr) {
    const int64_t grid = std::min<int64_t>((a.rows + GROUPS - 1) / GROUPS,
                                           FWD_THREADS / THREADS);
    if (layer)
      norm_fwd_kernel<TX, TH, NT, K, V, true>
          <<<dim3((unsigned)grid), THREADS, 0, s>>>(a);
    else
      norm_fwd_kernel<TX, TH, NT, K, V, false>
          <<<dim3((unsigned)grid), THREADS, 0, s>>>(a);
  } else if (layer) {
    norm_bwd_kernel<TX, TH, NT, K, V, true>
        <<<dim3(blocks), THREADS, 0, s>>>(a, *o);
  } else {
    norm_bwd_kernel<TX, TH, NT, K, V, false>
        <<<dim3(blocks), THREADS, 0, s>>>(a, *o);
  }
}

// 8 elements a thread, and the fewest threads a row that hold it: narrow rows
// share waves (65536 x 64: 18 us backward, a wave a row 76), wide ones spread
// over up to 16 (4096 columns over 512 threads: 2 rows on their way per CU
// where 256 threads with twice the registers had 1).
template <typename TX, typename TH>
int go_width(hipStream_t s, const NormArgs& a, const NormGrads* o,
             int blocks) {
  if (a.width < 8) go<TX, TH, 8, 1, 1>(s, a, o, blocks);
  else if (a.width <= 64) go<TX, TH, 8, 1, 8>(s, a, o, blocks);
  else if (a.width <= 128) go<TX, TH, 16, 1, 8>(s, a, o, blocks);
  else if (a.width <= 256) go<TX, TH, 32, 1, 8>(s, a, o, blocks);
  else if (a.width <= 512) go<TX, TH, 64, 1, 8>(s, a, o, blocks);
  else if (a.width <= 1024) go<TX, TH, 128, 1, 8>(s, a, o, blocks);
  else if (a.width <= 2048) go<TX, TH, 256, 1, 8>(s, a, o, blocks);
  else if (a.width <= 4096) go<TX, TH, 512, 1, 8>(s, a, o, blocks);
  else if (a.width <= 8192) go<TX, TH, 1024, 1, 8>(s, a, o, blocks);
  else if (a.width <= NORM_MAX_WIDTH) go<TX, TH, 1024, 2, 8>(s, a, o, blocks);
  else return (int)hipErrorInvalidValue;
  HIP_CHECK_LAST();
  return 0;
}

int go_types(hipStream_t s, const NormArgs& a, const NormGrads* o,
             int blocks) {
  switch (a.type_x * 3 + a.type_h) {
    case 0: return go_width<float, float>(s, a, o, blocks);
    case 1: return go_width<float, __bf16>(s, a, o, blocks);
    case 2: return go_width<float, _Float16>(s, a, o, blocks);
    case 4: return go_width<__bf16, __bf16>(s, a, o, blocks);
    case 8: return go_width<_Float16, _Float16>(s, a, o, blocks);
    default: return (int)hipErrorInvalidValue;
  }
}

}  // namespace

extern "C" int launch_norm_fwd(void* stream, const NormArgs* a) {
  if (a->rows == 0) return 0;
  return go_types((hipStream_t)stream, *a, nullptr, 0);
}

// Workgroups of the backward pass: enough to fill 256 CUs, and no more, since
// each writes its column sums once: one a CU of 1024 threads, 2 of 512, and up
// to 4 of 256 where each still has 8 turns.  Half of that with LayerNorms,
// whose four sums weigh more.  16384 x 2048 bf16 RMSNorms: 512 workgroups take
// 118 us, 1024 take 112; fp32 and bf16 LayerNorms 124 and 131; 8192 x 4096 of
// those 149 us with 256 and 157 with 512, the sums' addition included.
extern "C" int norm_bwd_blocks(const NormArgs* a) {
  const int64_t groups = a->width <= 64    ? 32
                         : a->width <= 128 ? 16
                         : a->width <= 256 ? 8
                         : a->width <= 512 ? 4
                         : a->width <= 1024 ? 2
                                            : 1;
  const bool layer = a->post == NORM_LAYER || a->pre == NORM_LAYER;
  const int64_t turns = (a->rows + groups - 1) / groups;
  int64_t most = 512;
  if (a->width > 4096 || (layer && a->width > 2048)) most = 256;
  else if (a->width <= 2048 && !layer)
    most = std::min<int64_t>(std::max<int64_t>(512, turns / 8), 1024);
  return (int)std::min(turns, most);
}

extern "C" int launch_norm_bwd(void* stream, const NormArgs* a,
                               const NormGrads* o, int blocks) {
  if (a->rows == 0) return 0;
  return go_types((hipStream_t)stream, *a, o, blocks);
}

extern "C" int launch_norm_columns(void* stream, const NormArgs* a,
                                   const NormGrads* o, int blocks) {
  norm_columns_kernel<<<dim3((unsigned)((a->width + 31) / 32), 2), 1024, 0,
                        (hipStream_t)stream>>>(*a, *o, blocks);
  HIP_CHECK_LAST();
  return 0;
}
