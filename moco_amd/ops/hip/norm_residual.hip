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
//   dw2 = sum d_y rhat, db2 = sum d_y, dw1 = sum dn hhat, db1 = sum dn,
//   dscale = sum d a n      over rows; [..] only in a LayerNorm.
//
// Both directions are bound by memory: each input is read and each output
// written once.  NT threads share a row, 8 neighbouring elements a thread
// and K such groups, so that the row stays in registers between its
// reductions.  Column sums stay in registers over a workgroup's rows, go to
// memory once per workgroup, and a second kernel adds those: no atomics, the
// same bits every time.
#include <algorithm>

#include "common.h"
#include "launchers.h"

namespace {

constexpr int V = 8;        // neighbouring elements of a thread
constexpr int BLOCK = 256;  // threads of a workgroup, at least

template <typename T>
struct Raw {
  T v[V];
};

// the first n (<= 0: none) of V elements, zeros behind; only the element's
// own alignment is assumed
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const void* base, int64_t off,
                                           int n) {
  Raw<T> r;
  const T* p = (const T*)base + off;
  if (n >= V) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store_f(void* base, int64_t off,
                                        const float (&f)[V], int n) {
  Raw<T> r;
  T* p = (T*)base + off;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = (T)f[i];  // to nearest even
  if (n >= V) {
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = r.v[i];
  }
}

// a per-channel vector (fp32 or TH), or a constant
template <typename TH>
__device__ __forceinline__ void load_vec(const void* p, bool f32, int col,
                                         int n, float none, float (&out)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = none;
  } else if (f32) {
    const Raw<float> r = load_raw<float>(p, col, n);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = r.v[i];
  } else {
    const Raw<TH> r = load_raw<TH>(p, col, n);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)r.v[i];
  }
}

// sums of M values over the NT threads of a row, in a fixed order
template <int NT, int M>
struct RowSum {
  static constexpr int WAVES = NT / WAVE;
  // two slots in turn: one barrier a reduction
  float slot[2][M][WAVES > 1 ? WAVES : 1];

  __device__ __forceinline__ void operator()(float (&v)[M], int turn) {
#pragma unroll
    for (int j = 0; j < M; ++j) v[j] = wave_reduce_sum(v[j]);
    if constexpr (WAVES > 1) {
      const int wave = threadIdx.x / WAVE;
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

__device__ __forceinline__ float sigmoid(float g) {
  return 1.f / (1.f + expf(-g));
}

__device__ __forceinline__ float act_of(int act, float g) {
  if (act == NORM_ACT_NONE) return g;
  const float s = sigmoid(g);
  return act == NORM_ACT_SILU ? g * s : s;
}

__device__ __forceinline__ float act_slope(int act, float g) {
  if (act == NORM_ACT_NONE) return 1.f;
  const float s = sigmoid(g);
  return act == NORM_ACT_SILU ? s * (1.f + g * (1.f - s)) : s * (1.f - s);
}

// mean (LayerNorm) and 1/std of a row held as f[K][V]
template <int NT, int K>
__device__ __forceinline__ void row_stats(const float (&f)[K][V],
                                          const int (&n)[K], int kind,
                                          float inv_c, float eps,
                                          RowSum<NT, 1>& sum, int& turn,
                                          float& mean, float& rstd) {
  float s[1] = {0.f};
  mean = 0.f;
  if (kind == NORM_LAYER) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += f[k][i];  // zeros behind the row
    sum(s, turn++);
    mean = s[0] * inv_c;
    s[0] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = i < n[k] ? f[k][i] - mean : 0.f;
      s[0] += d * d;
    }
  sum(s, turn++);
  rstd = rsqrtf(s[0] * inv_c + eps);
}

template <typename TX, typename TH, int NT, int K>
__global__ __launch_bounds__(NT < BLOCK ? BLOCK : NT) void norm_fwd_kernel(
    const NormArgs a) {
  constexpr int GROUPS = NT < BLOCK ? BLOCK / NT : 1;
  __shared__ RowSum<NT, 1> sums[GROUPS];
  const int group = threadIdx.x / NT, t = threadIdx.x % NT;
  RowSum<NT, 1>& sum = sums[group];
  int turn = 0;
  const float inv_c = 1.f / (float)a.width;
  // several groups share a workgroup only where they are single waves,
  // which need no barrier
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + group; row < a.rows;
       row += (int64_t)gridDim.x * GROUPS) {
    int n[K];
    Raw<TX> x[K];
    Raw<TH> g[K];
    float f[K][V];  // h, later r
  #pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * NT + t) * V;
      n[k] = a.width - col;
      x[k] = load_raw<TX>(a.x, row * a.ld_x + col, n[k]);
      if (a.h != nullptr) {
        const Raw<TH> h = load_raw<TH>(a.h, row * a.ld_h + col, n[k]);
  #pragma unroll
        for (int i = 0; i < V; ++i) f[k][i] = (float)h.v[i];
      }
      if (a.gate_kind == NORM_GATE_FULL)
        g[k] = load_raw<TH>(a.gate, row * a.ld_g + col, n[k]);
    }
    if (a.h == nullptr) {
  #pragma unroll
      for (int k = 0; k < K; ++k)
  #pragma unroll
        for (int i = 0; i < V; ++i) f[k][i] = (float)x[k].v[i];
    } else {
      float row_gate = 1.f;
      if (a.gate_kind == NORM_GATE_ROW)
        row_gate = act_of(a.act, (float)((const TH*)a.gate)[row * a.ld_g]);
      float mean = 0.f, rstd = 1.f;
      if (a.post != NORM_NONE) {
        row_stats<NT, K>(f, n, a.post, inv_c, a.post_eps, sum, turn, mean,
                         rstd);
        if (t == 0 && a.stats != nullptr) {
          a.stats[row] = mean;
          a.stats[a.rows + row] = rstd;
        }
      }
  #pragma unroll
      for (int k = 0; k < K; ++k) {
        const int col = (k * NT + t) * V;
        float w[V], b[V], s[V];
        load_vec<TH>(a.w1, a.f32 & 1, col, n[k], 1.f, w);
        load_vec<TH>(a.b1, a.f32 & 2, col, n[k], 0.f, b);
        load_vec<TH>(a.scale, a.f32 & 16, col, n[k], a.scale_value, s);
  #pragma unroll
        for (int i = 0; i < V; ++i) {
          const float hat = (f[k][i] - mean) * rstd;
          const float ga = a.gate_kind == NORM_GATE_FULL
                               ? act_of(a.act, (float)g[k].v[i])
                               : row_gate;
          f[k][i] = (float)x[k].v[i] + s[i] * ga * (hat * w[i] + b[i]);
          if (i >= n[k]) f[k][i] = 0.f;
        }
        if (a.r != nullptr)
          store_f<TX>(a.r, row * a.width + col, f[k], n[k]);
      }
    }
    if (a.pre == NORM_NONE) continue;
    float mean, rstd;
    row_stats<NT, K>(f, n, a.pre, inv_c, a.pre_eps, sum, turn, mean, rstd);
    if (t == 0 && a.stats != nullptr) {
      a.stats[2 * a.rows + row] = mean;
      a.stats[3 * a.rows + row] = rstd;
    }
  #pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * NT + t) * V;
      float w[V], b[V];
      load_vec<TH>(a.w2, a.f32 & 4, col, n[k], 1.f, w);
      load_vec<TH>(a.b2, a.f32 & 8, col, n[k], 0.f, b);
  #pragma unroll
      for (int i = 0; i < V; ++i)
        f[k][i] = (f[k][i] - mean) * rstd * w[i] + b[i];
      store_f<TH>(a.y, row * a.width + col, f[k], n[k]);
    }
  }
}

// Column sums of a workgroup, in the order of NormGrads::partial: dw1, db1,
// dw2, db2, dscale.
constexpr int VECS = 5;

template <typename TX, typename TH, int NT, int K>
__global__ __launch_bounds__(NT < BLOCK ? BLOCK : NT) void norm_bwd_kernel(
    const NormArgs a, const NormGrads o) {
  constexpr int GROUPS = NT < BLOCK ? BLOCK / NT : 1;
  __shared__ RowSum<NT, 2> sums2[GROUPS];
  __shared__ RowSum<NT, 3> sums3[GROUPS];
  __shared__ float across[GROUPS > 1 ? GROUPS * NT * K * V : 1];
  const int group = threadIdx.x / NT, t = threadIdx.x % NT;
  RowSum<NT, 2>& sum2 = sums2[group];
  RowSum<NT, 3>& sum3 = sums3[group];
  const float inv_c = 1.f / (float)a.width;
  float acc[VECS][K][V];
#pragma unroll
  for (int j = 0; j < VECS; ++j)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) acc[j][k][i] = 0.f;
  int n[K];
#pragma unroll
  for (int k = 0; k < K; ++k) n[k] = a.width - (k * NT + t) * V;
  int turn = 0;
  // the same number of turns for all threads of a group; several groups
  // share a workgroup only where they need no barrier
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + group; row < a.rows;
       row += (int64_t)gridDim.x * GROUPS, ++turn) {
    Raw<TX> x[K], dr[K];
    Raw<TH> h[K], g[K], dy[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * NT + t) * V;
      x[k] = load_raw<TX>(a.x, row * a.ld_x + col, n[k]);
      if (a.h != nullptr)
        h[k] = load_raw<TH>(a.h, row * a.ld_h + col, n[k]);
      if (a.gate_kind == NORM_GATE_FULL)
        g[k] = load_raw<TH>(a.gate, row * a.ld_g + col, n[k]);
      dr[k] = load_raw<TX>(o.d_r, row * a.width + col,
                           o.d_r != nullptr ? n[k] : 0);
      dy[k] = load_raw<TH>(o.d_y, row * a.width + col,
                           o.d_y != nullptr ? n[k] : 0);
    }
    float mean_h = 0.f, rstd_h = 1.f, mean_r = 0.f, rstd_r = 0.f;
    if (a.h != nullptr && a.post != NORM_NONE) {
      mean_h = a.stats[row];
      rstd_h = a.stats[a.rows + row];
    }
    if (o.d_y != nullptr) {
      mean_r = a.stats[2 * a.rows + row];
      rstd_r = a.stats[3 * a.rows + row];
    }
    float row_raw = 0.f, row_gate = 1.f;
    if (a.gate_kind == NORM_GATE_ROW) {
      row_raw = (float)((const TH*)a.gate)[row * a.ld_g];
      row_gate = act_of(a.act, row_raw);
    }
    // n = hhat w1 + b1 and r, then the norm before the next block
    float nf[K][V], hat[K][V], ga[K][V], d[K][V];
    float p[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * NT + t) * V;
      float w[V], b[V], s[V];
      if (a.h != nullptr) {
        load_vec<TH>(a.w1, a.f32 & 1, col, n[k], 1.f, w);
        load_vec<TH>(a.b1, a.f32 & 2, col, n[k], 0.f, b);
        load_vec<TH>(a.scale, a.f32 & 16, col, n[k], a.scale_value, s);
      }
      float w2[V];
      load_vec<TH>(a.w2, a.f32 & 4, col, n[k], 1.f, w2);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float r = (float)x[k].v[i];
        if (a.h != nullptr) {
          hat[k][i] = ((float)h[k].v[i] - mean_h) * rstd_h;
          nf[k][i] = hat[k][i] * w[i] + b[i];
          ga[k][i] = a.gate_kind == NORM_GATE_FULL
                         ? act_of(a.act, (float)g[k].v[i])
                         : row_gate;
          r += s[i] * ga[k][i] * nf[k][i];
        }
        const float rhat =
            i < n[k] && o.d_y != nullptr ? (r - mean_r) * rstd_r : 0.f;
        const float dyf = (float)dy[k].v[i];
        const float tt = dyf * w2[i];
        acc[2][k][i] += dyf * rhat;
        acc[3][k][i] += dyf;
        p[0] += tt * rhat;
        p[1] += tt;
        d[k][i] = rhat;  // until the sums are there
      }
    }
    if (o.d_y != nullptr) {
      sum2(p, turn);
      p[0] *= inv_c;
      p[1] = a.pre == NORM_LAYER ? p[1] * inv_c : 0.f;
    }
    float q[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * NT + t) * V;
      float w2[V], w[V], s[V];
      load_vec<TH>(a.w2, a.f32 & 4, col, n[k], 1.f, w2);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float dn =
            rstd_r * ((float)dy[k].v[i] * w2[i] - p[1] - d[k][i] * p[0]);
        d[k][i] = (float)dr[k].v[i] + (o.d_y != nullptr ? dn : 0.f);
      }
      if (o.d_x != nullptr)
        store_f<TX>(o.d_x, row * a.width + col, d[k], n[k]);
      if (a.h == nullptr) continue;
      load_vec<TH>(a.w1, a.f32 & 1, col, n[k], 1.f, w);
      load_vec<TH>(a.scale, a.f32 & 16, col, n[k], a.scale_value, s);
      float dg[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (i >= n[k]) d[k][i] = 0.f;
        const float dsn = d[k][i] * nf[k][i];
        acc[4][k][i] += dsn * ga[k][i];
        const float da = dsn * s[i];
        q[2] += da;
        if (a.gate_kind == NORM_GATE_FULL)
          dg[i] = da * act_slope(a.act, (float)g[k].v[i]);
        const float dn = d[k][i] * s[i] * ga[k][i];
        acc[0][k][i] += dn * hat[k][i];
        acc[1][k][i] += dn;
        d[k][i] = dn * w[i];  // t1 from here on
        q[0] += d[k][i] * hat[k][i];
        q[1] += d[k][i];
      }
      if (a.gate_kind == NORM_GATE_FULL && o.d_gate != nullptr)
        store_f<TH>(o.d_gate, row * a.width + col, dg, n[k]);
    }
    if (a.h == nullptr) continue;
    if (a.post != NORM_NONE || a.gate_kind == NORM_GATE_ROW) sum3(q, turn);
    if (a.gate_kind == NORM_GATE_ROW && o.d_gate != nullptr && t == 0)
      ((TH*)o.d_gate)[row] = (TH)(q[2] * act_slope(a.act, row_raw));
    if (o.d_h == nullptr) continue;
    const float m1 = a.post != NORM_NONE ? q[0] * inv_c : 0.f;
    const float m0 = a.post == NORM_LAYER ? q[1] * inv_c : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (k * NT + t) * V;
#pragma unroll
      for (int i = 0; i < V; ++i)
        d[k][i] = rstd_h * (d[k][i] - m0 - hat[k][i] * m1);
      store_f<TH>(o.d_h, row * a.width + col, d[k], n[k]);
    }
  }
  // the workgroup's column sums: its groups' are added in LDS first
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    if (o.partial[j] == nullptr) continue;
    float* out = o.partial[j] + (int64_t)blockIdx.x * a.width;
    if constexpr (GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
          across[((group * K + k) * NT + t) * V + i] = acc[j][k][i];
      __syncthreads();
      for (int c = threadIdx.x; c < a.width; c += BLOCK) {
        float s = 0.f;
#pragma unroll
        for (int gr = 0; gr < GROUPS; ++gr) s += across[gr * K * NT * V + c];
        out[c] = s;
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
        store_f<float>(out, (k * NT + t) * V, acc[j][k], n[k]);
    }
  }
}

// out[c] = sum over blocks of partial[b][c], for up to VECS vectors; one
// workgroup adds 64 columns, 16 parts of the blocks side by side
__global__ __launch_bounds__(1024) void norm_columns_kernel(
    const NormColumns v, int blocks, int width) {
  const float* p = v.partial[blockIdx.y];
  const int c = blockIdx.x * 64 + threadIdx.x % 64;
  const int part = threadIdx.x / 64;
  float s = 0.f;
  if (c < width)
    for (int b = part; b < blocks; b += 16) s += p[(int64_t)b * width + c];
  __shared__ float lds[16][64];
  lds[part][threadIdx.x % 64] = s;
  __syncthreads();
  if (part != 0 || c >= width) return;
  s = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) s += lds[j][threadIdx.x];
  void* out = v.out[blockIdx.y];
  switch (v.dtype[blockIdx.y]) {
    case 0: ((float*)out)[c] = s; break;
    case 1: ((__bf16*)out)[c] = (__bf16)s; break;
    default: ((_Float16*)out)[c] = (_Float16)s; break;
  }
}

template <typename TX, typename TH, int NT, int K>
void go(hipStream_t s, const NormArgs& a, const NormGrads* o, int blocks) {
  constexpr int GROUPS = NT < BLOCK ? BLOCK / NT : 1;
  constexpr int THREADS = NT < BLOCK ? BLOCK : NT;
  if (o == nullptr) {
    // a grid holds fewer than 2^32 threads
    const int64_t grid = std::min<int64_t>((a.rows + GROUPS - 1) / GROUPS,
                                           1 << 20);
    norm_fwd_kernel<TX, TH, NT, K><<<dim3((unsigned)grid), THREADS, 0, s>>>(a);
  } else {
    norm_bwd_kernel<TX, TH, NT, K><<<dim3(blocks), THREADS, 0, s>>>(a, *o);
  }
}

template <typename TX, typename TH>
int go_width(hipStream_t s, const NormArgs& a, const NormGrads* o,
             int blocks) {
  if (a.width <= 512) go<TX, TH, 64, 1>(s, a, o, blocks);
  else if (a.width <= 1024) go<TX, TH, 64, 2>(s, a, o, blocks);
  else if (a.width <= 2048) go<TX, TH, 256, 1>(s, a, o, blocks);
  else if (a.width <= 4096) go<TX, TH, 256, 2>(s, a, o, blocks);
  else if (a.width <= 8192) go<TX, TH, 1024, 1>(s, a, o, blocks);
  else if (a.width <= NORM_MAX_WIDTH) go<TX, TH, 1024, 2>(s, a, o, blocks);
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

extern "C" int norm_bwd_blocks(int64_t rows, int64_t width) {
  const int64_t groups = width <= 1024 ? BLOCK / WAVE : 1;
  const int64_t most = (rows + groups - 1) / groups;
  return (int)(most < 512 ? most : 512);
}

extern "C" int launch_norm_bwd(void* stream, const NormArgs* a,
                               const NormGrads* o, int blocks) {
  if (a->rows == 0) return 0;
  return go_types((hipStream_t)stream, *a, o, blocks);
}

extern "C" int launch_norm_columns(void* stream, const NormColumns* v,
                                   int vecs, int blocks, int64_t width) {
  if (vecs == 0 || width == 0) return 0;
  norm_columns_kernel<<<dim3((unsigned)((width + 63) / 64), vecs), 1024, 0,
                        (hipStream_t)stream>>>(*v, blocks, (int)width);
  HIP_CHECK_LAST();
  return 0;
}
