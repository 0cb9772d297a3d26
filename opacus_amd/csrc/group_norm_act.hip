// Group normalisation with an affine map and an activation on channels-last tensors, forward and
// backward, the backward pass with PER-SAMPLE weight and bias gradients.
//
//   x[n,S,C], G groups of Cg = C / G neighbouring channels;  xh = (x - mu) rstd;  z = w xh + b;  y = act(z)
//   dz = dy act'(z);  gw[n,c] = sum_s dz xh;  gb[n,c] = sum_s dz
//   dx = rstd (w dz - S1 - xh S2),  S1 = mean of w dz, S2 = mean of w dz xh over the statistics' elements
//
// Statistics per sample (nn.GroupNorm: over all S positions and the group's channels): S1 and S2
// are sums over the group's channels of w gb and w gw, so the per-sample parameter gradients that a
// DP step needs ARE the sums the input gradient waits for, and one reading of x and dy forms both.
// Statistics per position (each position's groups on their own, a norm per attention or recurrence
// head): the sums stay within a few lanes, and gw, gb are kept in registers along the rows.
//
// Means and variances are two-step (the mean first, then squares around it) within what a thread
// holds, and put together from (count, mean, M2) triples, so that a large mean costs no digits.
// All arithmetic is fp32; every reduction runs in a fixed order.
//
// Training passes (forward and backward), inputs that change from pass to pass: 256 x 1024 x 64 fp32, 32 groups: 81 us
// for 336 MB (kernels 24 and 44 us, 4.9 TB/s), memory; per position 16 x 1024 x 2048 bf16, 16 heads: 76 us for 335 MB
// (kernels 28, 46 and 5 us), memory and, backward, arithmetic (three quarters of the issue slots); 3 x 40000 x 128 bf16,
// 32 groups, gelu: 81 us in six launches that move eight streams of 31 MB (x; x, y; x, dy; x, dy, dx: 50 us at 4.9 TB/s),
// half of the issue slots arithmetic (gelu takes about 23 instructions a value in each of three passes), 10 us merges.
#include <type_traits>

#include "vec_io.h"

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 8;           // rows a thread has in flight in the statistics kernel
constexpr int kApplyRows = 4;      // and where it also computes
constexpr int64_t kWantBlocks = 2048;

constexpr int kRelu = DPK_ACT_RELU, kSilu = DPK_ACT_SILU, kGelu = DPK_ACT_GELU;

// Phi(z) = (1 + erf(z / sqrt 2)) / 2 and E = exp(-z^2 / 2), by formula 7.1.26 of Abramowitz and Stegun:
// erfc(x) = t (a1 + ... + a5 t^4) exp(-x^2) with t = 1 / (1 + p x), off by at most 1.5e-7. Its
// exponential is the one act' needs, and for z < 0 no 1 - erf cancels. Against the exact gelu that is 7e-7 of the value
// for |z| < 1 (the erf form in fp32: 2e-7) and 2e-7 absolute below -1 (5e-8), so 5e-5 of the value at -3.
__device__ __forceinline__ float normal_cdf(float z, float& E) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f));
  E = __builtin_amdgcn_exp2f(x * x * -kLog2e);
  float q = fmaf(t, 1.061405429f, -1.453152027f);
  q = fmaf(t, q, 1.421413741f);
  q = fmaf(t, q, -0.284496736f);
  q = fmaf(t, q, 0.254829592f);
  q *= 0.5f * t * E;
  return z < 0.f ? q : 1.0f - q;
}

// z -> act(z) for N values; one uniform branch for all of them.
template <int N>
__device__ __forceinline__ void activate(float (&z)[N], int act) {
  if (act == kSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] *= sigmoid_f(z[i]);
  } else if (act == kGelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float E;
      z[i] *= normal_cdf(z[i], E);
    }
  } else if (act == kRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] > 0.f ? z[i] : (z[i] != z[i] ? z[i] : 0.f);
  }
}
// z -> act'(z)
template <int N>
__device__ __forceinline__ void slope(float (&z)[N], int act) {
  if (act == kSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = sigmoid_f(z[i]);
      z[i] = s * fmaf(z[i], 1.0f - s, 1.0f);
    }
  } else if (act == kGelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float E;
      const float phi = normal_cdf(z[i], E);
      z[i] = fmaf(z[i] * 0.39894228040143268f, E, phi);
    }
  } else if (act == kRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] > 0.f ? 1.0f : (z[i] != z[i] ? z[i] : 0.f);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = 1.0f;
  }
}

struct NormArgs {
  const void* x;
  const void* dy;
  const void* w;        // null: 1
  const void* b;        // null: 0
  void* y;              // or dx
  float2* stats;        // [n,G] (mean, rstd); per position [n*S,G] in the workspace
  float2* part;         // [n,J,C] (mean, M2) or (sum dz, sum dz xh)
  float2* sums;         // [n,G] (S1, S2)
  float* gw;            // [n,C] or null
  float* gb;
  int64_t n, S;
  int C, G, Cg;
  int cl;               // vectors of a row that a block covers
  int lg;               // lanes of a group (statistics per position), or groups of a slab
  int wide;             // groups of a row that a wave takes, a power of two
  int cblocks;          // blocks along a row
  int J;                // row chunks of a sample
  int64_t chunk;        // rows of one
  int param_bf16, act;
  float eps;
};

__device__ __forceinline__ float param_at(const void* p, int is_bf16, int c, float none) {
  if (!p) return none;
  return is_bf16 ? bf16_to_f32(static_cast<const bf16_t*>(p)[c]) : static_cast<const float*>(p)[c];
}

// V neighbouring parameters from channel c on, in 16-byte loads where they are aligned to that.
template <int V>
__device__ __forceinline__ void params_at(const void* p, int is_bf16, int c, float none, float* v) {
  if (p && !is_bf16 && V % 4 == 0 && ((reinterpret_cast<uintptr_t>(p) >> 2) + c) % 4 == 0) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 q = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + c + j);
      v[j] = q.x, v[j + (V > 1)] = q.y, v[j + 2 * (V > 2)] = q.z, v[j + 3 * (V > 3)] = q.w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = param_at(p, is_bf16, c + j, none);
}

// What a thread of the streaming kernels works on: vector column c of rows r0 + rg, r0 + rg + step, ...
struct Span {
  int64_t b, r0, r1;
  int c, rg, step, j;
  bool on;
};
template <int V>
__device__ __forceinline__ Span span_of(const NormArgs& p) {
  Span s;
  int64_t bid = blockIdx.x;
  const int cb = static_cast<int>(bid % p.cblocks);
  bid /= p.cblocks;
  s.j = static_cast<int>(bid % p.J);
  s.b = bid / p.J;
  const int lane = threadIdx.x % p.cl;
  s.rg = threadIdx.x / p.cl;
  s.step = kThreads / p.cl;
  s.c = (cb * p.cl + lane) * V;
  s.on = s.rg < s.step && s.c < p.C;
  s.r0 = s.j * p.chunk;
  s.r1 = s.r0 + p.chunk < p.S ? s.r0 + p.chunk : p.S;
  return s;
}

// ---- statistics per sample: partial sums, merged sums, application ------------------------

// part[n,j,c] = (mean, M2) of channel c over the rows of chunk j.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void sample_stat_kernel(NormArgs p) {
  typedef vec_io<T, V> io;
  __shared__ float lds[2][kThreads * V];
  const Span s = span_of<V>(p);
  const T* x = static_cast<const T*>(p.x) + (s.b * p.S) * p.C + s.c;
  float mean[V], m2[V], cnt = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) mean[j] = m2[j] = 0.f;
  if (s.on) {
    for (int64_t r = s.r0 + s.rg; r < s.r1; r += static_cast<int64_t>(s.step) * kRows) {
      typename io::raw raw[kRows];
      int m = 0;
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const int64_t at = r + static_cast<int64_t>(k) * s.step;
        raw[k] = typename io::raw();
        if (at < s.r1) {
          raw[k] = io::load(x + at * p.C);
          ++m;
        }
      }
      const float fm = static_cast<float>(m), inv = 1.0f / fm, all = cnt + fm, share = fm / all;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < kRows; ++k) t += k < m ? io::get(raw[k], j) : 0.f;
        t *= inv;
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
          const float d = k < m ? io::get(raw[k], j) - t : 0.f;
          q = fmaf(d, d, q);
        }
        const float delta = t - mean[j];
        mean[j] = fmaf(delta, share, mean[j]);
        m2[j] += q + delta * delta * (cnt * share);
      }
      cnt = all;
    }
  }
  const int W = p.cl * V, lane = threadIdx.x % p.cl;
  if (s.rg < s.step) {
#pragma unroll
    for (int j = 0; j < V; ++j) lds[0][s.rg * W + lane * V + j] = mean[j], lds[1][s.rg * W + lane * V + j] = m2[j];
  }
  __syncthreads();
  // row group g of the block saw ceil((rows - g) / step) rows
  const int64_t rows = s.r1 - s.r0;
  const int groups = rows < s.step ? static_cast<int>(rows) : s.step;
  const float most = static_cast<float>((rows + s.step - 1) / s.step);
  const int extra = static_cast<int>(rows - (rows + s.step - 1) / s.step * s.step) + s.step;  // groups below it saw `most`
  const int c0 = s.c - lane * V;
  for (int i = threadIdx.x; i < W && c0 + i < p.C; i += kThreads) {
    float t = 0.f, q = 0.f;
    for (int g = 0; g < groups; ++g) t = fmaf(g < extra ? most : most - 1.f, lds[0][g * W + i], t);
    t /= static_cast<float>(rows);
    for (int g = 0; g < groups; ++g) {
      const float d = lds[0][g * W + i] - t;
      q += fmaf(d * d, g < extra ? most : most - 1.f, lds[1][g * W + i]);
    }
    p.part[(s.b * p.J + s.j) * p.C + c0 + i] = make_float2(t, q);
  }
}

// stats[n,g] from the (mean, M2) of its channels and chunks. One block per (n, g).
__global__ __launch_bounds__(kThreads) void sample_stat_merge_kernel(NormArgs p) {
  __shared__ float red[kThreads / DPK_WAVE];
  __shared__ float share;
  const int64_t b = blockIdx.x / p.G;
  const int g = static_cast<int>(blockIdx.x % p.G);
  const float2* part = p.part + b * p.J * p.C + g * p.Cg;
  const int items = p.J * p.Cg;
  const float total = static_cast<float>(p.S) * static_cast<float>(p.Cg);
  float t = 0.f;
  for (int i = threadIdx.x; i < items; i += kThreads) {
    const int j = i / p.Cg;
    const int64_t rows = p.S - j * p.chunk < p.chunk ? p.S - j * p.chunk : p.chunk;
    t += static_cast<float>(rows) * part[static_cast<int64_t>(j) * p.C + (i - j * p.Cg)].x;
  }
  t = block_sum<kThreads / DPK_WAVE>(t, red);
  if (threadIdx.x == 0) share = t / total;
  __syncthreads();
  const float mean = share;
  float q = 0.f;
  for (int i = threadIdx.x; i < items; i += kThreads) {
    const int j = i / p.Cg;
    const int64_t rows = p.S - j * p.chunk < p.chunk ? p.S - j * p.chunk : p.chunk;
    const float2 v = part[static_cast<int64_t>(j) * p.C + (i - j * p.Cg)];
    const float d = v.x - mean;
    q += fmaf(d * d, static_cast<float>(rows), v.y);
  }
  q = block_sum<kThreads / DPK_WAVE>(q, red);
  if (threadIdx.x == 0) p.stats[blockIdx.x] = make_float2(mean, 1.0f / sqrtf(q / total + p.eps));
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void sample_apply_kernel(NormArgs p) {
  typedef vec_io<T, V> io;
  const Span s = span_of<V>(p);
  if (!s.on) return;
  const T* x = static_cast<const T*>(p.x) + (s.b * p.S) * p.C + s.c;
  T* y = static_cast<T*>(p.y) + (s.b * p.S) * p.C + s.c;
  float mean[V], f[V], shift[V];
  params_at<V>(p.w, p.param_bf16, s.c, 1.f, f);
  params_at<V>(p.b, p.param_bf16, s.c, 0.f, shift);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float2 st = p.stats[s.b * p.G + (s.c + j) / p.Cg];
    mean[j] = st.x;
    f[j] *= st.y;
  }
  for (int64_t r = s.r0 + s.rg; r < s.r1; r += static_cast<int64_t>(s.step) * kApplyRows) {
    typename io::raw raw[kApplyRows];
#pragma unroll
    for (int k = 0; k < kApplyRows; ++k) {
      const int64_t at = r + static_cast<int64_t>(k) * s.step;
      raw[k] = typename io::raw();
      if (at < s.r1) raw[k] = io::load(x + at * p.C);
    }
    float z[kApplyRows * V];
#pragma unroll
    for (int k = 0; k < kApplyRows; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) z[k * V + j] = fmaf(io::get(raw[k], j) - mean[j], f[j], shift[j]);
    }
    activate(z, p.act);
#pragma unroll
    for (int k = 0; k < kApplyRows; ++k) {
      const int64_t at = r + static_cast<int64_t>(k) * s.step;
      if (at < s.r1) io::store(y + at * p.C, z + k * V);
    }
  }
}

// part[n,j,c] = (sum dz, sum dz xh) of channel c over the rows of chunk j.
template <typename T, int V, bool PER_POSITION>
__global__ __launch_bounds__(kThreads) void channel_sums_kernel(NormArgs p) {
  typedef vec_io<T, V> io;
  constexpr int R = 4;
  __shared__ float lds[2][kThreads * V];
  const Span s = span_of<V>(p);
  const T* x = static_cast<const T*>(p.x) + (s.b * p.S) * p.C + s.c;
  const T* dy = static_cast<const T*>(p.dy) + (s.b * p.S) * p.C + s.c;
  float A[V], B[V];
#pragma unroll
  for (int j = 0; j < V; ++j) A[j] = B[j] = 0.f;
  if (s.on) {
    float2 st[V];
    float w[V], shift[V];
    int grp[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      grp[j] = (s.c + j) / p.Cg;
      if (!PER_POSITION) st[j] = p.stats[s.b * p.G + grp[j]];
    }
    params_at<V>(p.w, p.param_bf16, s.c, 1.f, w);
    params_at<V>(p.b, p.param_bf16, s.c, 0.f, shift);
    for (int64_t r = s.r0 + s.rg; r < s.r1; r += static_cast<int64_t>(s.step) * R) {
      typename io::raw rx[R], rd[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int64_t at = r + static_cast<int64_t>(k) * s.step;
        rx[k] = rd[k] = typename io::raw();
        if (at < s.r1) {
          rx[k] = io::load(x + at * p.C);
          rd[k] = io::load(dy + at * p.C);
        }
      }
      float xh[R * V], z[R * V];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const int64_t at = r + static_cast<int64_t>(k) * s.step;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (PER_POSITION) st[j] = at < s.r1 ? p.stats[(s.b * p.S + at) * p.G + grp[j]] : make_float2(0.f, 0.f);
          xh[k * V + j] = (io::get(rx[k], j) - st[j].x) * st[j].y;
          z[k * V + j] = fmaf(xh[k * V + j], w[j], shift[j]);
        }
      }
      slope(z, p.act);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (r + static_cast<int64_t>(k) * s.step < s.r1) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float dz = io::get(rd[k], j) * z[k * V + j];
            A[j] += dz;
            B[j] = fmaf(dz, xh[k * V + j], B[j]);
          }
        }
      }
    }
  }
  const int W = p.cl * V, lane = threadIdx.x % p.cl, c0 = s.c - lane * V;
  if (s.rg < s.step) {
#pragma unroll
    for (int j = 0; j < V; ++j) lds[0][s.rg * W + lane * V + j] = A[j], lds[1][s.rg * W + lane * V + j] = B[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < W && c0 + i < p.C; i += kThreads) {
    float t = 0.f, q = 0.f;
    for (int g = 0; g < s.step; ++g) t += lds[0][g * W + i], q += lds[1][g * W + i];
    p.part[(s.b * p.J + s.j) * p.C + c0 + i] = make_float2(t, q);
  }
}

// gw, gb from the chunks' sums, and S1, S2 of the group. One block per (n, g): up to 256 channels side
// by side, and as many threads for the chunks of each as that leaves.
__global__ __launch_bounds__(kThreads) void sample_grad_merge_kernel(NormArgs p) {
  __shared__ float red[kThreads / DPK_WAVE];
  __shared__ float2 lds[kThreads];
  const int64_t b = blockIdx.x / p.G;
  const int g = static_cast<int>(blockIdx.x % p.G);
  const int across = p.Cg < kThreads ? p.Cg : kThreads, down = kThreads / across;
  const int lane = threadIdx.x % across, row = threadIdx.x / across;
  float s1 = 0.f, s2 = 0.f;
  for (int i0 = 0; i0 < p.Cg; i0 += across) {
    const int c = g * p.Cg + i0 + lane;
    const bool on = i0 + lane < p.Cg && row < down;
    float A = 0.f, B = 0.f;
    if (on) {
      const float2* part = p.part + b * p.J * p.C + c;
#pragma unroll 4
      for (int j = row; j < p.J; j += down) {
        const float2 v = part[static_cast<int64_t>(j) * p.C];
        A += v.x;
        B += v.y;
      }
    }
    __syncthreads();
    lds[threadIdx.x] = make_float2(A, B);
    __syncthreads();
    if (on && row == 0) {
      A = B = 0.f;
      for (int r = 0; r < down; ++r) A += lds[r * across + lane].x, B += lds[r * across + lane].y;
      if (p.gb) p.gb[b * p.C + c] = A;
      if (p.gw) p.gw[b * p.C + c] = B;
      const float w = param_at(p.w, p.param_bf16, c, 1.f);
      s1 = fmaf(w, A, s1);
      s2 = fmaf(w, B, s2);
    }
  }
  s1 = block_sum<kThreads / DPK_WAVE>(s1, red);
  s2 = block_sum<kThreads / DPK_WAVE>(s2, red);
  const float inv = 1.0f / (static_cast<float>(p.S) * static_cast<float>(p.Cg));
  if (threadIdx.x == 0) p.sums[blockIdx.x] = make_float2(s1 * inv, s2 * inv);
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void sample_dx_kernel(NormArgs p) {
  typedef vec_io<T, V> io;
  constexpr int R = 4;
  const Span s = span_of<V>(p);
  if (!s.on) return;
  const T* x = static_cast<const T*>(p.x) + (s.b * p.S) * p.C + s.c;
  const T* dy = static_cast<const T*>(p.dy) + (s.b * p.S) * p.C + s.c;
  T* dx = static_cast<T*>(p.y) + (s.b * p.S) * p.C + s.c;
  float2 st[V], sm[V];
  float w[V], shift[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int64_t g = s.b * p.G + (s.c + j) / p.Cg;
    st[j] = p.stats[g];
    sm[j] = p.sums[g];
  }
  params_at<V>(p.w, p.param_bf16, s.c, 1.f, w);
  params_at<V>(p.b, p.param_bf16, s.c, 0.f, shift);
  for (int64_t r = s.r0 + s.rg; r < s.r1; r += static_cast<int64_t>(s.step) * R) {
    typename io::raw rx[R], rd[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int64_t at = r + static_cast<int64_t>(k) * s.step;
      rx[k] = rd[k] = typename io::raw();
      if (at < s.r1) {
        rx[k] = io::load(x + at * p.C);
        rd[k] = io::load(dy + at * p.C);
      }
    }
    float xh[R * V], z[R * V];
#pragma unroll
    for (int k = 0; k < R; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xh[k * V + j] = (io::get(rx[k], j) - st[j].x) * st[j].y;
        z[k * V + j] = fmaf(xh[k * V + j], w[j], shift[j]);
      }
    }
    slope(z, p.act);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = io::get(rd[k], j) * z[k * V + j] * w[j];
        o[j] = st[j].y * (d - sm[j].x - xh[k * V + j] * sm[j].y);
      }
      const int64_t at = r + static_cast<int64_t>(k) * s.step;
      if (at < s.r1) io::store(dx + at * p.C, o);
    }
  }
}

// ---- statistics per sample, where a block holds all positions of some whole groups ---------------
//
// A block takes gs neighbouring groups (a slab of 128 bytes of each row or more) of one sample, a thread
// one vector column of every step-th row, all in registers: x (and dy) are read once. At 256 x 1024 x 64
// fp32: 23 us forward and 44 us backward, against 73 and 74 us with partial sums, their merge and a second
// reading (three launches each); 33 x 49 x 210: 7 us against 21. Slabs of 64 bytes, two blocks a CU instead of one:
// 29 and 59 us.
// What a thread holds ends the route: 64 values, so 1024 positions of 64 channels in 32 groups in fp32 and 512 in bf16.
// A call forward and backward, on its two sides: 256 x 1024 x 64 fp32 24 and 49 us, 1088 positions 49 and 87; 256 x 512 x
// 64 bf16 15 and 19 us, 1024 positions 34 and 61.
constexpr int kSlabThreads = 512;
constexpr int kSlabWidth = 2048;  // channels at most: 40 KB of LDS with 16 KB for the row groups of 8-element vectors

// s[i] (i < groups of the slab) = sum over the slab's channels i * Cg ... of w * v, v[V] being this
// thread's value for its columns: first over the row groups, then over the channels. `chan` keeps the
// channels' unweighted sums. lds: [step][W]. One thread adds up a group's channels, which is nothing for a few and
// most of the time for very wide groups: 64 x 16 x 2048 fp32 takes 26 us forward in 32 groups and 169 us in one.
template <int V>
__device__ __forceinline__ void slab_sums(const float (&v)[V], bool on, int rg, int lane, int step, int W, int Cg, float* lds,
                                          float* chan, float* s, const float* w) {
  __syncthreads();
  if (on) {
#pragma unroll
    for (int j = 0; j < V; ++j) lds[rg * W + lane * V + j] = v[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < W; i += kSlabThreads) {
    float t = 0.f;
#pragma unroll 4
    for (int g = 0; g < step; ++g) t += lds[g * W + i];
    chan[i] = t;
  }
  __syncthreads();
  for (int g = threadIdx.x; g < W / Cg; g += kSlabThreads) {
    float t = 0.f;
    for (int i = g * Cg; i < (g + 1) * Cg; ++i) t = w ? fmaf(w[i], chan[i], t) : t + chan[i];
    s[g] = t;
  }
  __syncthreads();
}

template <typename T, int V, int R, bool BACKWARD>
__global__ __launch_bounds__(kSlabThreads) void slab_kernel(NormArgs p) {
  typedef vec_io<T, V> io;
  extern __shared__ float shared[];  // [step][W], 2 x [W], 2 x [groups], [W]
  const int slabs = p.cblocks;
  const int64_t b = blockIdx.x / slabs;
  const int slab = static_cast<int>(blockIdx.x - b * slabs);
  const int g0 = slab * p.lg, gs = p.G - g0 < p.lg ? p.G - g0 : p.lg;  // p.lg: groups of a slab
  const int W = gs * p.Cg, cl = W / V, step = kSlabThreads / cl;
  float* lds = shared;
  float* chan[2] = {lds + kSlabThreads * V, lds + kSlabThreads * V + W};
  float* grp[2] = {chan[1] + W, chan[1] + W + gs};
  float* wts = grp[1] + gs;
  const int lane = threadIdx.x % cl, rg = threadIdx.x / cl;
  const bool on = rg < step;
  const int in = lane * V, c = g0 * p.Cg + in;
  const int S = static_cast<int>(p.S);
  const T* x = static_cast<const T*>(p.x) + b * p.S * p.C + c;
  const T* dy = static_cast<const T*>(p.dy) + b * p.S * p.C + c;
  T* y = static_cast<T*>(p.y) + b * p.S * p.C + c;
  typename io::raw rx[R], rd[BACKWARD ? R : 1];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int r = rg + k * step;
    rx[k] = typename io::raw();
    if (BACKWARD) rd[BACKWARD ? k : 0] = typename io::raw();
    if (on && r < S) {
      rx[k] = io::load(x + static_cast<int64_t>(r) * p.C);
      if (BACKWARD) rd[BACKWARD ? k : 0] = io::load(dy + static_cast<int64_t>(r) * p.C);
    }
  }
  float w[V], shift[V];
  params_at<V>(p.w, p.param_bf16, c, 1.f, w);
  params_at<V>(p.b, p.param_bf16, c, 0.f, shift);
  if (BACKWARD && rg == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) wts[in + j] = w[j];
  }
  const float inv = 1.0f / (static_cast<float>(S) * static_cast<float>(p.Cg));
  float mean[V], rstd[V], t[V];
  if (!BACKWARD) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      t[j] = 0.f;
#pragma unroll
      for (int k = 0; k < R; ++k) t[j] += io::get(rx[k], j);
    }
    slab_sums<V>(t, on, rg, lane, step, W, p.Cg, lds, chan[0], grp[0], nullptr);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      mean[j] = grp[0][(in + j) / p.Cg] * inv;
      t[j] = 0.f;
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const float d = io::get(rx[k], j) - mean[j];
        t[j] = rg + k * step < S ? fmaf(d, d, t[j]) : t[j];
      }
    }
    slab_sums<V>(t, on, rg, lane, step, W, p.Cg, lds, chan[0], grp[1], nullptr);
    for (int g = threadIdx.x; g < gs; g += kSlabThreads)
      p.stats[b * p.G + g0 + g] = make_float2(grp[0][g] * inv, 1.0f / sqrtf(fmaf(grp[1][g], inv, p.eps)));
#pragma unroll
    for (int j = 0; j < V; ++j) rstd[j] = w[j] / sqrtf(fmaf(grp[1][(in + j) / p.Cg], inv, p.eps));
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const int r = rg + k * step;
      float z[V];
#pragma unroll
      for (int j = 0; j < V; ++j) z[j] = fmaf(io::get(rx[k], j) - mean[j], rstd[j], shift[j]);
      activate(z, p.act);
      if (on && r < S) io::store(y + static_cast<int64_t>(r) * p.C, z);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float2 st = p.stats[b * p.G + g0 + (in + j) / p.Cg];
    mean[j] = st.x;
    rstd[j] = st.y;
    t[j] = 0.f;
  }
  float dz[R][V], u[V];
#pragma unroll
  for (int j = 0; j < V; ++j) u[j] = 0.f;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    float z[V], xh[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      xh[j] = (io::get(rx[k], j) - mean[j]) * rstd[j];
      z[j] = fmaf(xh[j], w[j], shift[j]);
    }
    slope(z, p.act);
    const bool live = rg + k * step < S;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      dz[k][j] = live ? io::get(rd[BACKWARD ? k : 0], j) * z[j] : 0.f;
      t[j] += dz[k][j];
      u[j] = live ? fmaf(dz[k][j], xh[j], u[j]) : u[j];
    }
  }
  slab_sums<V>(t, on, rg, lane, step, W, p.Cg, lds, chan[0], grp[0], wts);
  slab_sums<V>(u, on, rg, lane, step, W, p.Cg, lds, chan[1], grp[1], wts);
  for (int i = threadIdx.x; i < W; i += kSlabThreads) {
    if (p.gb) p.gb[b * p.C + g0 * p.Cg + i] = chan[0][i];
    if (p.gw) p.gw[b * p.C + g0 * p.Cg + i] = chan[1][i];
  }
  float s1[V], s2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    s1[j] = grp[0][(in + j) / p.Cg] * inv;
    s2[j] = grp[1][(in + j) / p.Cg] * inv;
  }
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int r = rg + k * step;
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float xh = (io::get(rx[k], j) - mean[j]) * rstd[j];
      o[j] = rstd[j] * (dz[k][j] * w[j] - s1[j] - xh * s2[j]);
    }
    if (on && r < S) io::store(y + static_cast<int64_t>(r) * p.C, o);
  }
}

// ---- statistics per position: the groups of a row side by side in the lanes of a wave ------------
//
// A group takes `lg` lanes (the least power of two that holds its vectors, NI vectors a lane where 64
// lanes are not enough), a wave `wide` groups of a row and, where a row has fewer, as many rows side by
// side as fill it; then the same groups of the next rows. A row's sums are a few lane exchanges, and
// the columns a lane holds never change: weight and bias stay in registers, and so do the
// per-sample sums along the rows. Nothing is read twice.

// v[i] = sum of v[i] over the lg lanes of the group, in all of them.
template <int R>
__device__ __forceinline__ void lane_sum(float (&v)[R], int lg) {
#define DPK_DPP_STEP(at, ctrl)                                                                                       \
  if (lg > at) {                                                                                                     \
    _Pragma("unroll") for (int i = 0; i < R; ++i) v[i] += __int_as_float(                                            \
        __builtin_amdgcn_update_dpp(0, __float_as_int(v[i]), ctrl, 0xf, 0xf, true));                                 \
  }
  DPK_DPP_STEP(1, 0xb1)   // quad_perm [1,0,3,2]
  DPK_DPP_STEP(2, 0x4e)   // quad_perm [2,3,0,1]
  DPK_DPP_STEP(4, 0x141)  // row_half_mirror
  DPK_DPP_STEP(8, 0x140)  // row_mirror
#undef DPK_DPP_STEP
  if (lg > 16) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] += __shfl_xor(v[i], 16, DPK_WAVE);
  }
  if (lg > 32) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] += __shfl_xor(v[i], 32, DPK_WAVE);
  }
}

template <typename T, int V, int NI, int R, bool BACKWARD>
__global__ __launch_bounds__(kThreads, NI * V <= 8 ? 3 : 1) void position_rows_kernel(NormArgs p) {
  typedef vec_io<T, V> io;
  constexpr int N = NI * V, kWaves = kThreads / DPK_WAVE;
  __shared__ float lds[BACKWARD ? 2 : 1][BACKWARD ? kWaves : 1][BACKWARD ? DPK_WAVE * N : 1];
  const int lane = threadIdx.x % DPK_WAVE, wave = threadIdx.x / DPK_WAVE;
  const int cb = static_cast<int>(blockIdx.x % p.cblocks);
  const int64_t rest = blockIdx.x / p.cblocks;
  // forward: row chunks of the whole tensor; backward: of one sample
  const int64_t b = BACKWARD ? rest / p.J : 0, j = BACKWARD ? rest - b * p.J : rest;
  const int64_t rows = BACKWARD ? p.S : p.n * p.S;
  const int64_t r0 = j * p.chunk, r1 = r0 + p.chunk < rows ? r0 + p.chunk : rows;
  const int across = p.lg * p.wide, side = DPK_WAVE / across, sub = lane / across;  // rows side by side, and this lane's
  const int g = cb * p.wide + lane % across / p.lg, at = lane % p.lg;
  const bool mine = g < p.G;
  bool on[NI];
  int c[NI];
  float w[N], shift[N];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int in = (i * p.lg + at) * V;
    on[i] = mine && in < p.Cg;
    c[i] = on[i] ? g * p.Cg + in : 0;
    params_at<V>(p.w, p.param_bf16, c[i], 1.f, w + i * V);
    params_at<V>(p.b, p.param_bf16, c[i], 0.f, shift + i * V);
#pragma unroll
    for (int k = 0; k < V; ++k) {  // a lane without a channel adds zeros to its group's sums
      w[i * V + k] = on[i] ? w[i * V + k] : 0.f;
      shift[i * V + k] = on[i] ? shift[i * V + k] : 0.f;
    }
  }
  const float inv = 1.0f / static_cast<float>(p.Cg);
  const T* x = static_cast<const T*>(p.x) + b * p.S * p.C;
  const T* dy = static_cast<const T*>(p.dy) + b * p.S * p.C;
  T* y = static_cast<T*>(p.y) + b * p.S * p.C;
  float A[N], B[N];
#pragma unroll
  for (int k = 0; k < N; ++k) A[k] = B[k] = 0.f;

  typename io::raw nx[R][NI], nd[BACKWARD ? R : 1][NI];
  const auto fetch = [&](int64_t r) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        nx[q][i] = typename io::raw();
        if (BACKWARD) nd[BACKWARD ? q : 0][i] = typename io::raw();
        if (on[i] && r + q * side < r1) {
          nx[q][i] = io::load(x + (r + q * side) * p.C + c[i]);
          if (BACKWARD) nd[BACKWARD ? q : 0][i] = io::load(dy + (r + q * side) * p.C + c[i]);
        }
      }
    }
  };
  fetch(r0 + wave * R * side + sub);
  // (the bound is the wave's: its lanes exchange values, so they stay together)
  for (int64_t r = r0 + wave * R * side + sub; r - sub < r1; r += kWaves * R * side) {
    typename io::raw rx[R][NI], rd[BACKWARD ? R : 1][NI];
#pragma unroll
    for (int q = 0; q < R; ++q) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        rx[q][i] = nx[q][i];
        if (BACKWARD) rd[BACKWARD ? q : 0][i] = nd[BACKWARD ? q : 0][i];
      }
    }
    fetch(r + kWaves * R * side);  // the next rows, under this batch's arithmetic
    float mean[R], rstd[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) mean[q] += io::get(rx[q][i], k);
      }
    }
    lane_sum(mean, p.lg);
    // A lane without a channel takes 0 for the mean, a row behind the last one 0 for rstd: their x and dy
    // are zeros, so every term they add is zero too and no element has to be masked.
    float at_mean[R][NI];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] *= inv;
      rstd[q] = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        at_mean[q][i] = on[i] ? mean[q] : 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float d = io::get(rx[q][i], k) - at_mean[q][i];
          rstd[q] = fmaf(d, d, rstd[q]);
        }
      }
    }
    lane_sum(rstd, p.lg);
#pragma unroll
    for (int q = 0; q < R; ++q) rstd[q] = r + q * side < r1 ? 1.0f / sqrtf(fmaf(rstd[q], inv, p.eps)) : 0.f;
    if (!BACKWARD) {
#pragma unroll
      for (int q = 0; q < R; ++q) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          float z[V];
#pragma unroll
          for (int k = 0; k < V; ++k)
            z[k] = fmaf((io::get(rx[q][i], k) - at_mean[q][i]) * rstd[q], w[i * V + k], shift[i * V + k]);
          activate(z, p.act);
          if (on[i] && r + q * side < r1) io::store(y + (r + q * side) * p.C + c[i], z);
        }
      }
    } else {
      float s1[R], s2[R], xh[R][N], d[R][N];
#pragma unroll
      for (int q = 0; q < R; ++q) {
        s1[q] = s2[q] = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          float z[V];
#pragma unroll
          for (int k = 0; k < V; ++k) {
            xh[q][i * V + k] = (io::get(rx[q][i], k) - at_mean[q][i]) * rstd[q];
            z[k] = fmaf(xh[q][i * V + k], w[i * V + k], shift[i * V + k]);
          }
          slope(z, p.act);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float dz = io::get(rd[BACKWARD ? q : 0][i], k) * z[k];
            A[i * V + k] += dz;
            B[i * V + k] = fmaf(dz, xh[q][i * V + k], B[i * V + k]);
            d[q][i * V + k] = dz * w[i * V + k];
            s1[q] += d[q][i * V + k];
            s2[q] = fmaf(d[q][i * V + k], xh[q][i * V + k], s2[q]);
          }
        }
      }
      lane_sum(s1, p.lg);
      lane_sum(s2, p.lg);
#pragma unroll
      for (int q = 0; q < R; ++q) {
        s1[q] *= inv;
        s2[q] *= inv;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          float o[V];
#pragma unroll
          for (int k = 0; k < V; ++k) o[k] = rstd[q] * (d[q][i * V + k] - s1[q] - xh[q][i * V + k] * s2[q]);
          if (on[i] && r + q * side < r1) io::store(y + (r + q * side) * p.C + c[i], o);
        }
      }
    }
  }
  if (!BACKWARD) return;
  if (!p.gw && !p.gb) return;
  for (int o = DPK_WAVE / 2; o >= across; o /= 2) {  // the rows side by side
#pragma unroll
    for (int k = 0; k < N; ++k) A[k] += __shfl_xor(A[k], o, DPK_WAVE), B[k] += __shfl_xor(B[k], o, DPK_WAVE);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) lds[0][wave][k * DPK_WAVE + lane] = A[k], lds[BACKWARD][wave][k * DPK_WAVE + lane] = B[k];
  __syncthreads();
  if (wave != 0 || sub != 0) return;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float t = 0.f, u = 0.f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        t += lds[0][BACKWARD ? v : 0][(i * V + k) * DPK_WAVE + lane];
        u += lds[BACKWARD][BACKWARD ? v : 0][(i * V + k) * DPK_WAVE + lane];
      }
      if (!on[i]) continue;
      if (p.J > 1) {
        p.part[(b * p.J + j) * p.C + c[i] + k] = make_float2(t, u);
      } else {
        if (p.gb) p.gb[b * p.C + c[i] + k] = t;
        if (p.gw) p.gw[b * p.C + c[i] + k] = u;
      }
    }
  }
}

// ---- statistics per position, groups that no wave holds: one wave per (row, group) ---------------
//
// The simplest form: single elements, x read three times and more (from a cache after the first). 8 x 1024 x 4096 in one
// group, forward and backward: bf16 83 and 235 us (floor 27 and 41), fp32 116 and 282 (55 and 82); 16 x 1024 x 2048 fp32
// in one group 110 and 253, where the bf16 row, which a wave holds, takes 29 and 62.

template <typename T, bool BACKWARD>
__global__ __launch_bounds__(kThreads) void position_kernel(NormArgs p) {
  typedef vec_io<T, 1> io;
  const int64_t wave = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / DPK_WAVE;
  const int lane = threadIdx.x & (DPK_WAVE - 1);
  if (wave >= p.n * p.S * p.G) return;
  const int64_t row = wave / p.G;
  const int g = static_cast<int>(wave - row * p.G);
  const int c0 = g * p.Cg;
  const T* x = static_cast<const T*>(p.x) + row * p.C + c0;
  T* y = static_cast<T*>(p.y) + row * p.C + c0;
  const float inv = 1.0f / static_cast<float>(p.Cg);
  float t = 0.f;
  for (int i = lane; i < p.Cg; i += DPK_WAVE) t += io::get(x[i], 0);
  const float mean = wave_sum(t) * inv;
  t = 0.f;
  for (int i = lane; i < p.Cg; i += DPK_WAVE) {
    const float d = io::get(x[i], 0) - mean;
    t = fmaf(d, d, t);
  }
  const float rstd = 1.0f / sqrtf(wave_sum(t) * inv + p.eps);
  if (!BACKWARD) {
    for (int i = lane; i < p.Cg; i += DPK_WAVE) {
      float z[1] = {fmaf((io::get(x[i], 0) - mean) * rstd, param_at(p.w, p.param_bf16, c0 + i, 1.f),
                         param_at(p.b, p.param_bf16, c0 + i, 0.f))};
      activate(z, p.act);
      io::store(y + i, z);
    }
    return;
  }
  if (lane == 0) p.stats[wave] = make_float2(mean, rstd);
  const T* dy = static_cast<const T*>(p.dy) + row * p.C + c0;
  float s1 = 0.f, s2 = 0.f;
  for (int i = lane; i < p.Cg; i += DPK_WAVE) {
    const float w = param_at(p.w, p.param_bf16, c0 + i, 1.f), xh = (io::get(x[i], 0) - mean) * rstd;
    float z[1] = {fmaf(xh, w, param_at(p.b, p.param_bf16, c0 + i, 0.f))};
    slope(z, p.act);
    const float d = io::get(dy[i], 0) * z[0] * w;
    s1 += d;
    s2 = fmaf(d, xh, s2);
  }
  s1 = wave_sum(s1) * inv;
  s2 = wave_sum(s2) * inv;
  for (int i = lane; i < p.Cg; i += DPK_WAVE) {
    const float w = param_at(p.w, p.param_bf16, c0 + i, 1.f), xh = (io::get(x[i], 0) - mean) * rstd;
    float z[1] = {fmaf(xh, w, param_at(p.b, p.param_bf16, c0 + i, 0.f))};
    slope(z, p.act);
    const float o[1] = {rstd * (io::get(dy[i], 0) * z[0] * w - s1 - xh * s2)};
    io::store(y + i, o);
  }
}

// gw, gb[n,c] from the chunks' sums.
__global__ __launch_bounds__(kThreads) void chunk_merge_kernel(NormArgs p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= p.n * p.C) return;
  const int64_t b = i / p.C;
  const float2* part = p.part + b * p.J * p.C + (i - b * p.C);
  float A = 0.f, B = 0.f;
#pragma unroll 8
  for (int j = 0; j < p.J; ++j) {
    const float2 v = part[static_cast<int64_t>(j) * p.C];
    A += v.x;
    B += v.y;
  }
  if (p.gb) p.gb[i] = A;
  if (p.gw) p.gw[i] = B;
}

// ---- host ------------------------------------------------------------------------------------

// The cut of [S, C] into blocks: a block covers up to 256 vectors of a row and as many rows at once as
// its threads allow; S is cut into enough chunks to fill the GPU. `sums`: the chunks leave partial sums
// of 8 bytes a channel, and there are no more of them than it takes to give each 64 rows, or 8 for a thread (rounded up
// and then evened out: of 65 rows, two chunks of 33).
void plan(NormArgs* p, int V, bool sums) {
  const int vecs = p->C / V;
  p->cl = vecs < kThreads ? vecs : kThreads;
  p->cblocks = static_cast<int>(dpk_cdiv(vecs, p->cl));
  const int step = kThreads / p->cl;
  int64_t least = static_cast<int64_t>(step) * (sums ? 8 : kApplyRows);
  if (sums && least < 64) least = 64;
  int64_t J = dpk_cdiv(kWantBlocks, p->n * p->cblocks);
  const int64_t most = dpk_cdiv(p->S, least);
  if (J > most) J = most;
  if (J < 1) J = 1;
  p->chunk = dpk_cdiv(p->S, J);
  p->J = static_cast<int>(dpk_cdiv(p->S, p->chunk));
}

int grid_of(const char* fn, const NormArgs& p, dim3* grid) {
  const int64_t blocks = p.n * p.cblocks * p.J;
  DPK_REQUIRE(dpk_grid_fits(blocks, kThreads), DPK_E_SHAPE, "%s: too large", fn);
  *grid = dim3(static_cast<unsigned>(blocks));
  return DPK_OK;
}

int width_of(const NormArgs& p, int dtype) {
  for (int V = dtype == DPK_BF16 ? 8 : 4; V > 1; V /= 2) {
    const size_t al = dpk_elsize(dtype) * V;
    if (p.C % V == 0 && dpk_aligned(p.x, al) && dpk_aligned(p.dy, al) && dpk_aligned(p.y, al)) return V;
  }
  return 1;
}

// Statistics per sample: the slab of whole groups a block of 512 threads can hold in registers, at most
// 64 values a thread. False if S is too long for the narrowest one.
bool plan_slabs(NormArgs* p, int V, int dtype, int* R) {
  const int64_t es = static_cast<int64_t>(dpk_elsize(dtype));
  int gs = 1;
  while (gs < p->G && (static_cast<int64_t>(gs) * p->Cg * es < 128 || static_cast<int64_t>(gs) * p->Cg % V != 0)) ++gs;
  const int64_t cl = static_cast<int64_t>(gs) * p->Cg / V;
  if (cl > kSlabThreads || cl * V > kSlabWidth) return false;
  const int64_t rows = dpk_cdiv(p->S, kSlabThreads / cl);
  const int most = V == 8 ? 8 : 16;
  if (rows > most) return false;
  *R = rows <= 4 ? 4 : most;
  p->lg = gs;
  p->cblocks = static_cast<int>(dpk_cdiv(p->G, gs));
  return true;
}

// Statistics per position: the widest loads for which a group's vectors fit into a wave, up to 4 a
// lane. False if none do.
bool plan_rows(NormArgs* p, int dtype, bool backward, int* V, int* NI) {
  for (*V = dtype == DPK_BF16 ? 8 : 4;; *V /= 2) {
    const size_t al = dpk_elsize(dtype) * *V;
    if (p->Cg % *V == 0 && dpk_aligned(p->x, al) && dpk_aligned(p->dy, al) && dpk_aligned(p->y, al)) break;
  }
  const int vecs = p->Cg / *V;
  for (p->lg = 1; p->lg < vecs && p->lg < DPK_WAVE;) p->lg *= 2;
  for (*NI = 1; *NI * p->lg < vecs;) *NI *= 2;
  if (*NI > 4) return false;
  for (p->wide = 1; p->wide < p->G && p->wide * p->lg < DPK_WAVE;) p->wide *= 2;
  p->cblocks = static_cast<int>(dpk_cdiv(p->G, p->wide));
  const int64_t rows = backward ? p->S : p->n * p->S, samples = backward ? p->n : 1;
  // enough blocks to fill the GPU; backward, no more chunks than chunks of 64 rows, or of 32 for every one that lies side
  // by side in a wave, would be, evened out (the partial sums of a chunk cost 8 bytes a channel and a reduction over the
  // block)
  int64_t J = dpk_cdiv(backward ? 768 : kWantBlocks, samples * p->cblocks);
  const int64_t side = DPK_WAVE / (p->lg * p->wide);
  const int64_t most = dpk_cdiv(rows, !backward ? 4 * side : side > 2 ? 32 * side : 64);
  if (J > most) J = most;
  if (J < 1) J = 1;
  p->chunk = dpk_cdiv(rows, J);
  p->J = static_cast<int>(dpk_cdiv(rows, p->chunk));
  return true;
}

// A group of up to 256 channels fits a wave, whatever its alignment.
bool wave_holds(int64_t C, int64_t G) { return C / G <= 4 * DPK_WAVE; }
// The partial sums of the chunks, for whichever type and width the call has; nothing where the kernels
// that need none run for all of them.
size_t part_bytes(int64_t n, int64_t S, int64_t C, int64_t G, int per_position) {
  const size_t chunk = static_cast<size_t>(n) * C * sizeof(float2);
  size_t most = 0;
  if (per_position) {
    // a sample is cut into no more chunks than 64-row ones, nor than it takes to fill the GPU
    int64_t J = dpk_cdiv(S, 64);
    if (J > dpk_cdiv(kWantBlocks, n)) J = dpk_cdiv(kWantBlocks, n);
    if (J > 1) most = chunk * J;
  }
  if (!per_position || !wave_holds(C, G)) {
    for (int V = 1; V <= 8 && C % V == 0; V *= 2) {
      NormArgs p = {};
      p.n = n, p.S = S, p.C = static_cast<int>(C), p.G = static_cast<int>(G), p.Cg = p.C / p.G;
      int R;
      bool slabs = !per_position;
      for (const int dtype : {DPK_BF16, DPK_F32})
        if (V * dpk_elsize(dtype) <= 16) slabs = slabs && plan_slabs(&p, V, dtype, &R);
      if (slabs) continue;
      plan(&p, V, true);
      if (chunk * p.J > most) most = chunk * p.J;
    }
  }
  return dpk_align_up(most, 256);
}
// (mean, rstd) of every position's groups where no wave may hold one, or (S1, S2) of every sample's.
size_t group_bytes(int64_t n, int64_t S, int64_t G, int per_position) {
  return dpk_align_up(static_cast<size_t>(n) * (per_position ? S : 1) * G * sizeof(float2), 256);
}

int check_common(const char* fn, const NormArgs& p, int dtype, int param_dtype, int64_t C, int64_t G, int per_position,
                 const void* ws, size_t ws_bytes, bool* nothing) {
  *nothing = false;
  DPK_REQUIRE(p.n >= 0 && p.S >= 0 && C >= 1 && G >= 1, DPK_E_SHAPE, "%s: bad size (n=%lld S=%lld C=%lld groups=%lld)", fn,
              (long long)p.n, (long long)p.S, (long long)C, (long long)G);
  DPK_REQUIRE(C % G == 0, DPK_E_SHAPE, "%s: %lld channels do not divide into %lld groups", fn, (long long)C, (long long)G);
  DPK_REQUIRE(C <= (1 << 24) && p.n < (1LL << 31) && p.S < (1LL << 40), DPK_E_SHAPE, "%s: too large", fn);
  DPK_REQUIRE(dpk_dtype_ok(dtype) && dpk_dtype_ok(param_dtype), DPK_E_DTYPE, "%s: dtype %d / %d not supported", fn, dtype,
              param_dtype);
  DPK_REQUIRE(p.act >= DPK_ACT_NONE && p.act <= DPK_ACT_GELU, DPK_E_ARG, "%s: unknown activation %d", fn, p.act);
  DPK_REQUIRE(per_position == 0 || per_position == 1, DPK_E_ARG, "%s: per_position must be 0 or 1", fn);
  DPK_REQUIRE(p.eps >= 0.f, DPK_E_ARG, "%s: eps must not be negative", fn);
  if (p.n == 0 || p.S == 0) {
    *nothing = true;
    return DPK_OK;
  }
  const size_t es = dpk_elsize(dtype), ps = dpk_elsize(param_dtype);
  DPK_REQUIRE(p.x && p.y, DPK_E_ARG, "%s: a tensor is NULL", fn);
  DPK_REQUIRE(dpk_aligned(p.x, es) && dpk_aligned(p.y, es) && dpk_aligned(p.dy, es) && dpk_aligned(p.w, ps) &&
                  dpk_aligned(p.b, ps) && dpk_aligned(p.gw, 4) && dpk_aligned(p.gb, 4) && dpk_aligned(p.stats, 8),
              DPK_E_ALIGN, "%s: a tensor is not aligned to its element size", fn);
  // (in floating point: the product of sizes no tensor has must not wrap around)
  const double groups = static_cast<double>(p.n) * static_cast<double>(G) * (per_position ? static_cast<double>(p.S) / 4 + 1 : 1.0);
  DPK_REQUIRE(groups <= static_cast<double>(DPK_MAX_GRID_X), DPK_E_SHAPE, "%s: too many groups", fn);
  const size_t need = dpk_group_norm_act_workspace_bytes(p.n, p.S, C, G, per_position);
  DPK_REQUIRE(need == 0 || (ws && ws_bytes >= need), DPK_E_WORKSPACE, "%s: workspace too small (%zu < %zu)", fn, ws_bytes, need);
  DPK_REQUIRE(dpk_aligned(ws, 16), DPK_E_ALIGN, "%s: workspace not 16-byte aligned", fn);
  return DPK_OK;
}

template <typename T, int V, bool BACKWARD>
void launch_rows(const NormArgs& p, int NI, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((BACKWARD ? p.n : 1) * p.J * p.cblocks)), block(kThreads);
  if (NI == 1) hipLaunchKernelGGL((position_rows_kernel<T, V, 1, BACKWARD ? 2 : 4, BACKWARD>), grid, block, 0, s, p);
  else if (NI == 2) hipLaunchKernelGGL((position_rows_kernel<T, V, 2, BACKWARD ? 1 : 2, BACKWARD>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((position_rows_kernel<T, V, 4, 1, BACKWARD>), grid, block, 0, s, p);
}

template <typename T, int V, bool BACKWARD>
void launch_slabs(const NormArgs& p, int R, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.n * p.cblocks)), block(kSlabThreads);
  const size_t lds = (kSlabThreads * V + 3 * p.lg * p.Cg + 2 * p.lg) * sizeof(float);
  if (R == 4) hipLaunchKernelGGL((slab_kernel<T, V, 4, BACKWARD>), grid, block, lds, s, p);
  else hipLaunchKernelGGL((slab_kernel<T, V, (V == 8 ? 8 : 16), BACKWARD>), grid, block, lds, s, p);
}

// Calls body(T{}, integral_constant<V>) for the tensor's type and width.
template <typename F>
void by_width(int dtype, int V, F&& body) {
  if (dtype == DPK_BF16) {
    if (V == 8) body(bf16_t(), std::integral_constant<int, 8>());
    else if (V == 4) body(bf16_t(), std::integral_constant<int, 4>());
    else if (V == 2) body(bf16_t(), std::integral_constant<int, 2>());
    else body(bf16_t(), std::integral_constant<int, 1>());
  } else {
    if (V == 4) body(float(), std::integral_constant<int, 4>());
    else if (V == 2) body(float(), std::integral_constant<int, 2>());
    else body(float(), std::integral_constant<int, 1>());
  }
}

}  // namespace

extern "C" size_t dpk_group_norm_act_workspace_bytes(int64_t n, int64_t S, int64_t C, int64_t groups, int per_position) {
  if (n <= 0 || S <= 0 || C <= 0 || groups <= 0 || C > (1 << 24) || C % groups) return 0;  // nothing to do, or refused
  const size_t part = part_bytes(n, S, C, groups, per_position);
  if (per_position ? wave_holds(C, groups) : part == 0) return part;
  return part + group_bytes(n, S, groups, per_position);
}

extern "C" int dpk_group_norm_act(const void* x, int dtype, const void* weight, const void* bias, int param_dtype, void* y,
                                  float* stats, int64_t n, int64_t S, int64_t C, int64_t groups, float eps, int act,
                                  int per_position, void* ws, size_t ws_bytes, dpk_stream_t stream) {
  const char* fn = "dpk_group_norm_act";
  NormArgs p = {};
  p.x = x, p.w = weight, p.b = bias, p.y = y, p.stats = reinterpret_cast<float2*>(stats);
  p.n = n, p.S = S, p.act = act, p.eps = eps, p.param_bf16 = param_dtype == DPK_BF16;
  bool nothing;
  if (int rc = check_common(fn, p, dtype, param_dtype, C, groups, per_position, ws, ws_bytes, &nothing)) return rc;
  if (nothing) return DPK_OK;
  DPK_REQUIRE(stats || per_position, DPK_E_ARG, "%s: stats is NULL", fn);
  p.C = static_cast<int>(C), p.G = static_cast<int>(groups), p.Cg = p.C / p.G;
  hipStream_t s = static_cast<hipStream_t>(stream);
  int V, NI;
  if (per_position && plan_rows(&p, dtype, false, &V, &NI)) {
    DPK_REQUIRE(dpk_grid_fits(static_cast<int64_t>(p.J) * p.cblocks, kThreads), DPK_E_SHAPE, "%s: too large", fn);
    by_width(dtype, V, [&](auto t, auto v) { launch_rows<decltype(t), decltype(v)::value, false>(p, NI, s); });
  } else if (per_position) {
    DPK_REQUIRE(dpk_grid_fits(dpk_cdiv(n * S * groups, kThreads / DPK_WAVE), kThreads), DPK_E_SHAPE, "%s: too large", fn);
    const unsigned grid = static_cast<unsigned>(dpk_cdiv(n * S * groups, kThreads / DPK_WAVE));
    if (dtype == DPK_BF16) hipLaunchKernelGGL((position_kernel<bf16_t, false>), dim3(grid), dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((position_kernel<float, false>), dim3(grid), dim3(kThreads), 0, s, p);
  } else {
    V = width_of(p, dtype);
    int R;
    if (plan_slabs(&p, V, dtype, &R)) {
      DPK_REQUIRE(dpk_grid_fits(n * p.cblocks, kSlabThreads), DPK_E_SHAPE, "%s: too large", fn);
      by_width(dtype, V, [&](auto t, auto v) { launch_slabs<decltype(t), decltype(v)::value, false>(p, R, s); });
      DPK_LAUNCH_CHECK(fn);
      return DPK_OK;
    }
    DPK_REQUIRE(dpk_grid_fits(n * groups, kThreads), DPK_E_SHAPE, "%s: too many groups", fn);
    plan(&p, V, true);
    p.part = static_cast<float2*>(ws);
    dim3 grid;
    if (int rc = grid_of(fn, p, &grid)) return rc;
    by_width(dtype, V, [&](auto t, auto v) {
      hipLaunchKernelGGL((sample_stat_kernel<decltype(t), decltype(v)::value>), grid, dim3(kThreads), 0, s, p);
    });
    hipLaunchKernelGGL(sample_stat_merge_kernel, dim3(static_cast<unsigned>(n * groups)), dim3(kThreads), 0, s, p);
    plan(&p, V, false);
    if (int rc = grid_of(fn, p, &grid)) return rc;
    by_width(dtype, V, [&](auto t, auto v) {
      hipLaunchKernelGGL((sample_apply_kernel<decltype(t), decltype(v)::value>), grid, dim3(kThreads), 0, s, p);
    });
  }
  DPK_LAUNCH_CHECK(fn);
  return DPK_OK;
}

extern "C" int dpk_group_norm_act_backward(const void* x, const void* grad_out, int dtype, const void* weight,
                                           const void* bias, int param_dtype, const float* stats, void* grad_x,
                                           float* grad_weight, float* grad_bias, int64_t n, int64_t S, int64_t C,
                                           int64_t groups, float eps, int act, int per_position, void* ws, size_t ws_bytes,
                                           dpk_stream_t stream) {
  const char* fn = "dpk_group_norm_act_backward";
  NormArgs p = {};
  p.x = x, p.dy = grad_out, p.w = weight, p.b = bias, p.y = grad_x;
  p.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  p.gw = grad_weight, p.gb = grad_bias;
  p.n = n, p.S = S, p.act = act, p.eps = eps, p.param_bf16 = param_dtype == DPK_BF16;
  bool nothing;
  if (int rc = check_common(fn, p, dtype, param_dtype, C, groups, per_position, ws, ws_bytes, &nothing)) return rc;
  if (nothing) return DPK_OK;
  DPK_REQUIRE(grad_out, DPK_E_ARG, "%s: grad_out is NULL", fn);
  DPK_REQUIRE(stats || per_position, DPK_E_ARG, "%s: stats is NULL", fn);
  p.C = static_cast<int>(C), p.G = static_cast<int>(groups), p.Cg = p.C / p.G;
  hipStream_t s = static_cast<hipStream_t>(stream);
  p.part = static_cast<float2*>(ws);
  int V, NI;
  if (per_position && plan_rows(&p, dtype, true, &V, &NI)) {
    DPK_REQUIRE(dpk_grid_fits(n * p.J * p.cblocks, kThreads), DPK_E_SHAPE, "%s: too large", fn);
    by_width(dtype, V, [&](auto t, auto v) { launch_rows<decltype(t), decltype(v)::value, true>(p, NI, s); });
    if (p.J > 1 && (p.gw || p.gb))
      hipLaunchKernelGGL(chunk_merge_kernel, dim3(static_cast<unsigned>(dpk_cdiv(n * C, kThreads))), dim3(kThreads), 0, s, p);
    DPK_LAUNCH_CHECK(fn);
    return DPK_OK;
  }
  V = width_of(p, dtype);
  int R;
  if (!per_position && plan_slabs(&p, V, dtype, &R)) {
    DPK_REQUIRE(dpk_grid_fits(n * p.cblocks, kSlabThreads), DPK_E_SHAPE, "%s: too large", fn);
    by_width(dtype, V, [&](auto t, auto v) { launch_slabs<decltype(t), decltype(v)::value, true>(p, R, s); });
    DPK_LAUNCH_CHECK(fn);
    return DPK_OK;
  }
  plan(&p, V, true);
  dim3 grid;
  if (int rc = grid_of(fn, p, &grid)) return rc;
  float2* groups_ws = reinterpret_cast<float2*>(static_cast<char*>(ws) + part_bytes(n, S, C, groups, per_position));
  if (per_position) {
    DPK_REQUIRE(dpk_grid_fits(dpk_cdiv(n * S * groups, kThreads / DPK_WAVE), kThreads), DPK_E_SHAPE, "%s: too large", fn);
    p.stats = groups_ws;
    const unsigned waves = static_cast<unsigned>(dpk_cdiv(n * S * groups, kThreads / DPK_WAVE));
    if (dtype == DPK_BF16) hipLaunchKernelGGL((position_kernel<bf16_t, true>), dim3(waves), dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((position_kernel<float, true>), dim3(waves), dim3(kThreads), 0, s, p);
    if (p.gw || p.gb) {
      by_width(dtype, V, [&](auto t, auto v) {
        hipLaunchKernelGGL((channel_sums_kernel<decltype(t), decltype(v)::value, true>), grid, dim3(kThreads), 0, s, p);
      });
      hipLaunchKernelGGL(chunk_merge_kernel, dim3(static_cast<unsigned>(dpk_cdiv(n * C, kThreads))), dim3(kThreads), 0, s, p);
    }
  } else {
    DPK_REQUIRE(dpk_grid_fits(n * groups, kThreads), DPK_E_SHAPE, "%s: too many groups", fn);
    p.sums = groups_ws;
    by_width(dtype, V, [&](auto t, auto v) {
      hipLaunchKernelGGL((channel_sums_kernel<decltype(t), decltype(v)::value, false>), grid, dim3(kThreads), 0, s, p);
    });
    hipLaunchKernelGGL(sample_grad_merge_kernel, dim3(static_cast<unsigned>(n * groups)), dim3(kThreads), 0, s, p);
    plan(&p, V, false);
    if (int rc = grid_of(fn, p, &grid)) return rc;
    by_width(dtype, V, [&](auto t, auto v) {
      hipLaunchKernelGGL((sample_dx_kernel<decltype(t), decltype(v)::value>), grid, dim3(kThreads), 0, s, p);
    });
  }
  DPK_LAUNCH_CHECK(fn);
  return DPK_OK;
}
