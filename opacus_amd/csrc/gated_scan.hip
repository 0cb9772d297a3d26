// The gated linear recurrence of the DPGatedRNN layer, forward, backward and one token at a time.
//
//   gates[n,T,3D] = values x | decay gates r | input gates i,   decay lam[D]
//   rho = sigma(r);  L = -softplus(lam) rho;  a = exp(L);  u = sqrt(1 - a^2) sigma(i) x
//   h_t = a_t h_{t-1} + u_t,   out_t = h_t
//
// The recurrence is a composition of affine maps h -> A h + B, so T is cut at will: every thread
// runs K positions of its channels in registers, the 16 time groups of a block exchange their
// (A, B) through LDS and fold them in order, and where the batch has too few rows to fill the
// GPU, T is also cut into segments whose (A, B) a first launch leaves in the workspace. Every fold runs in
// position order: the same inputs give the same bits.
//
// Backward: g_t = dy_t + a_{t+1} g_{t+1} runs the same maps the other way (same A, other B), and
//   q = 1 - a,  m = sqrt(q (1 + a)),  kappa = -L / m,  s = sigma(i)
//   dx = g m s;  di = dx x (1 - s);  w = g (L a h_{t-1} + s x a^2 kappa);  dr = w (1 - rho)
//   dlam[sample] = sigma(lam) / softplus(lam) * sum_t w
// (dL/dr = L (1 - rho) and dL/dlam = L sigma(lam) / softplus(lam), so w = L dloss/dL serves both; in
// this form nothing is divided by m alone, which vanishes as the gate closes.) h_{t-1} is formed
// again from the fp32 state the forward pass kept at every 64th position, so no rounded output
// enters a gradient.
#include <initializer_list>

#include "vec_io.h"

namespace {

constexpr int kThreads = 256;
constexpr int kCL = 16;                  // lanes across channels
constexpr int kTG = kThreads / kCL;      // time groups of a block
constexpr int kChunk = DPK_SCAN_CHUNK;   // positions between kept states
constexpr int kFwdK = 8;                 // positions per thread and tile
constexpr int kBwdK = 4;
constexpr int kFwdTile = kTG * kFwdK;    // 128
constexpr int kBwdTile = kTG * kBwdK;    // 64
static_assert(kBwdTile == kChunk && kFwdTile % kChunk == 0, "a backward tile starts at a kept state");
// Blocks wanted before T is left whole: four per CU of the MI355X.
constexpr int64_t kWantBlocks = 1024;
constexpr int kMaxSegments = 64;

// softplus(v) = max(v, 0) + log1p(exp(-|v|))
__device__ __forceinline__ float softplus_f(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }
// sigma(v) / softplus(v); 1 in the limit v -> -inf, where both are exp(v)
__device__ __forceinline__ float decay_ratio(float v) {
  const float sp = softplus_f(v);
  return sp > 0.f ? (1.0f / (1.0f + expf(-v))) / sp : 1.0f;
}

// a = exp(L) and q = 1 - a for L <= 0, each to its own relative accuracy: q from its series
// -L (1 + L/2 + L^2/6 + ...) while |L| < 0.35 (the first dropped term is below 2e-8), from a beyond.
// A layer starts out with every L in the series' range, so the exponential is behind a branch
// that a wave takes only if one of its lanes needs it.
__device__ __forceinline__ void decay_of(float L, float& a, float& q) {
  float p = fmaf(L, 1.0f / 5040.0f, 1.0f / 720.0f);
  p = fmaf(L, p, 1.0f / 120.0f);
  p = fmaf(L, p, 1.0f / 24.0f);
  p = fmaf(L, p, 1.0f / 6.0f);
  p = fmaf(L, p, 0.5f);
  p = fmaf(L, p, 1.0f);
  q = -L * p;
  a = 1.0f - q;
  if (!(L > -0.35f)) {
    a = __builtin_amdgcn_exp2f(L * kLog2e);
    q = 1.0f - a;
  }
}
// 1 / sqrt(1 - a^2) from q. A q of zero gives a finite factor, so that m = (1 - a^2) * this and
// kappa = -L * this are zero there.
__device__ __forceinline__ float inv_scale(float q2) { return __builtin_amdgcn_rsqf(fmaxf(q2, 1e-37f)); }

struct ScanArgs {
  const void* gates;
  const void* decay;
  const float* state;      // [n,D] or null
  const int64_t* lengths;  // [n] or null
  void* out;
  float* last;
  float* kept;             // [n, ceil(T/chunk), D] or null
  float* sum_a;            // [S,n,D] summaries of the segments
  float* sum_b;
  int64_t n, T, D, sn, st;
  int decay_bf16, reverse;
  int S;                   // segments of T
  int64_t seg;             // positions of a segment, a multiple of the tile
};

struct ScanBwdArgs {
  const void* gates;
  const void* decay;
  const float* kept;
  const int64_t* lengths;
  const void* dy;
  const float* dlast;      // [n,D] or null
  void* dgates;            // [n,T,3D]
  float* dstate;           // [n,D] or null
  float* dlam;             // [S,n,D]: the rows themselves when S == 1
  float* sum_a;
  float* sum_b;
  int64_t n, T, D, sn, st;
  int decay_bf16, reverse;
  int S;
  int64_t seg;
};

template <int V>
__device__ __forceinline__ void load_decay(const void* decay, int is_bf16, int64_t c, float* lam) {
#pragma unroll
  for (int j = 0; j < V; ++j)
    lam[j] = is_bf16 ? bf16_to_f32(static_cast<const bf16_t*>(decay)[c + j]) : static_cast<const float*>(decay)[c + j];
}

__device__ __forceinline__ int64_t live_length(const int64_t* lengths, int64_t b, int64_t T) {
  if (!lengths) return T;
  const int64_t l = lengths[b];
  return l < 0 ? 0 : (l < T ? l : T);
}

// One block: 16 * V channels of one sample, one segment of T, walked tile by tile.
// SUMMARY: only (A, B) of the segment are wanted.
template <typename T, int V, bool SUMMARY>
__global__ __launch_bounds__(kThreads) void scan_fwd_kernel(ScanArgs p) {
  typedef vec_io<T, V> io;
  constexpr int W = kCL * V;
  __shared__ float lds_a[2][kTG][W];
  __shared__ float lds_b[2][kTG][W];
  const int cl = threadIdx.x % kCL, tg = threadIdx.x / kCL;
  const int64_t cbs = (p.D + W - 1) / W;
  int64_t bid = blockIdx.x;
  const int64_t cb = bid % cbs;
  bid /= cbs;
  const int64_t b = bid % p.n;
  const int seg = static_cast<int>(bid / p.n);
  const int64_t c = cb * W + cl * V;
  const bool on = c < p.D;
  const int64_t len = live_length(p.lengths, b, p.T);
  const int64_t s0 = seg * p.seg;
  const int64_t s1 = s0 + p.seg < p.T ? s0 + p.seg : p.T;
  const T* gx = static_cast<const T*>(p.gates) + b * p.sn + c;
  T* out = static_cast<T*>(p.out) + b * p.T * p.D + c;
  const int64_t nD = p.n * p.D, row = b * p.D + c;

  float sp[V], h_in[V], prod[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sp[j] = h_in[j] = 0.f, prod[j] = 1.f;
  if (on) {
    load_decay<V>(p.decay, p.decay_bf16, c, sp);
#pragma unroll
    for (int j = 0; j < V; ++j) sp[j] = softplus_f(sp[j]);
    if (!SUMMARY) {
      if (p.state) {
#pragma unroll
        for (int j = 0; j < V; ++j) h_in[j] = p.state[row + j];
      }
      for (int k = 0; k < seg; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          h_in[j] = fmaf(p.sum_a[k * nD + row + j], h_in[j], p.sum_b[k * nD + row + j]);
      }
    }
  }

  int buf = 0;
  for (int64_t tile = s0; tile < s1; tile += kFwdTile, buf ^= 1) {
    const int64_t s = tile + tg * kFwdK;
    typename io::raw rx[kFwdK], rr[kFwdK], ri[kFwdK];
    bool live[kFwdK];
#pragma unroll
    for (int k = 0; k < kFwdK; ++k) {
      const int64_t pos = p.reverse ? p.T - 1 - (s + k) : s + k;
      live[k] = on && s + k < s1 && pos < len;
      rx[k] = rr[k] = ri[k] = typename io::raw();
      if (live[k]) {
        const T* q = gx + pos * p.st;
        rx[k] = io::load(q);
        rr[k] = io::load(q + p.D);
        ri[k] = io::load(q + 2 * p.D);
      }
    }
    float a[kFwdK][V], u[kFwdK][V], A[V], B[V];
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = 1.f, B[j] = 0.f;
#pragma unroll
    for (int k = 0; k < kFwdK; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float q;
        const float L = live[k] ? -sp[j] * sigmoid_f(io::get(rr[k], j)) : 0.f;
        decay_of(L, a[k][j], q);
        const float m2 = q * (1.0f + a[k][j]);
        u[k][j] = m2 * inv_scale(m2) * sigmoid_f(io::get(ri[k], j)) * io::get(rx[k], j);
        A[j] *= a[k][j];
        B[j] = fmaf(a[k][j], B[j], u[k][j]);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) lds_a[buf][tg][cl * V + j] = A[j], lds_b[buf][tg][cl * V + j] = B[j];
    __syncthreads();  // the other buffer's readers are past it once every thread is here
    float h[V];
#pragma unroll
    for (int g = 0; g < kTG; ++g) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (g == tg) h[j] = h_in[j];
        const float ga = lds_a[buf][g][cl * V + j];
        h_in[j] = fmaf(ga, h_in[j], lds_b[buf][g][cl * V + j]);
        if (SUMMARY) prod[j] *= ga;
      }
    }
    if (!SUMMARY) {
      if (p.kept && on && s < s1 && s % kChunk == 0) {
        float* kp = p.kept + (b * ((p.T + kChunk - 1) / kChunk) + s / kChunk) * p.D + c;
#pragma unroll
        for (int j = 0; j < V; ++j) kp[j] = h[j];
      }
#pragma unroll
      for (int k = 0; k < kFwdK; ++k) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          h[j] = fmaf(a[k][j], h[j], u[k][j]);
          o[j] = live[k] ? h[j] : 0.f;
        }
        if (on && s + k < s1) io::store(out + (p.reverse ? p.T - 1 - (s + k) : s + k) * p.D, o);
      }
    }
  }
  if (on && tg == 0) {
    if (SUMMARY) {
#pragma unroll
      for (int j = 0; j < V; ++j) p.sum_a[seg * nD + row + j] = prod[j], p.sum_b[seg * nD + row + j] = h_in[j];
    } else if (seg == p.S - 1) {
#pragma unroll
      for (int j = 0; j < V; ++j) p.last[row + j] = h_in[j];
    }
  }
}

// The reverse recurrence's (A, B) of a segment: needs the decay gates and the output gradients only.
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void scan_bwd_summary_kernel(ScanBwdArgs p) {
  typedef vec_io<T, V> io;
  constexpr int W = kCL * V;
  __shared__ float lds_a[2][kTG][W];
  __shared__ float lds_b[2][kTG][W];
  const int cl = threadIdx.x % kCL, tg = threadIdx.x / kCL;
  const int64_t cbs = (p.D + W - 1) / W;
  int64_t bid = blockIdx.x;
  const int64_t cb = bid % cbs;
  bid /= cbs;
  const int64_t b = bid % p.n;
  const int seg = static_cast<int>(bid / p.n);
  const int64_t c = cb * W + cl * V;
  const bool on = c < p.D;
  const int64_t len = live_length(p.lengths, b, p.T);
  const int64_t s0 = seg * p.seg;
  const int64_t s1 = s0 + p.seg < p.T ? s0 + p.seg : p.T;
  const T* gr = static_cast<const T*>(p.gates) + b * p.sn + p.D + c;
  const T* dy = static_cast<const T*>(p.dy) + b * p.T * p.D + c;
  float sp[V], R[V], prod[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sp[j] = R[j] = 0.f, prod[j] = 1.f;
  if (on) {
    load_decay<V>(p.decay, p.decay_bf16, c, sp);
#pragma unroll
    for (int j = 0; j < V; ++j) sp[j] = softplus_f(sp[j]);
  }
  int buf = 0;
  const int64_t tiles = s1 > s0 ? (s1 - s0 + kFwdTile - 1) / kFwdTile : 0;
  for (int64_t i = tiles - 1; i >= 0; --i, buf ^= 1) {
    const int64_t s = s0 + i * kFwdTile + tg * kFwdK;
    typename io::raw rr[kFwdK], rd[kFwdK];
    bool live[kFwdK];
#pragma unroll
    for (int k = 0; k < kFwdK; ++k) {
      const int64_t pos = p.reverse ? p.T - 1 - (s + k) : s + k;
      live[k] = on && s + k < s1 && pos < len;
      rr[k] = rd[k] = typename io::raw();
      if (live[k]) {
        rr[k] = io::load(gr + pos * p.st);
        rd[k] = io::load(dy + pos * p.D);
      }
    }
    float A[V], B[V];
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = 1.f, B[j] = 0.f;
#pragma unroll
    for (int k = kFwdK - 1; k >= 0; --k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float a, q;
        decay_of(live[k] ? -sp[j] * sigmoid_f(io::get(rr[k], j)) : 0.f, a, q);
        A[j] *= a;
        B[j] = a * (io::get(rd[k], j) + B[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) lds_a[buf][tg][cl * V + j] = A[j], lds_b[buf][tg][cl * V + j] = B[j];
    __syncthreads();
#pragma unroll
    for (int g = kTG - 1; g >= 0; --g) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float ga = lds_a[buf][g][cl * V + j];
        R[j] = fmaf(ga, R[j], lds_b[buf][g][cl * V + j]);
        prod[j] *= ga;
      }
    }
  }
  if (on && tg == 0) {
    const int64_t nD = p.n * p.D, row = b * p.D + c;
#pragma unroll
    for (int j = 0; j < V; ++j) p.sum_a[seg * nD + row + j] = prod[j], p.sum_b[seg * nD + row + j] = R[j];
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void scan_bwd_kernel(ScanBwdArgs p) {
  typedef vec_io<T, V> io;
  constexpr int W = kCL * V, K = kBwdK;
  __shared__ float lds_a[2][kTG][W];
  __shared__ float lds_b[2][kTG][W];
  __shared__ float lds_g[2][kTG][W];
  const int cl = threadIdx.x % kCL, tg = threadIdx.x / kCL;
  const int64_t cbs = (p.D + W - 1) / W;
  int64_t bid = blockIdx.x;
  const int64_t cb = bid % cbs;
  bid /= cbs;
  const int64_t b = bid % p.n;
  const int seg = static_cast<int>(bid / p.n);
  const int64_t c = cb * W + cl * V;
  const bool on = c < p.D;
  const int64_t len = live_length(p.lengths, b, p.T);
  const int64_t s0 = seg * p.seg;
  const int64_t s1 = s0 + p.seg < p.T ? s0 + p.seg : p.T;
  const int64_t chunks = (p.T + kChunk - 1) / kChunk;
  const T* gx = static_cast<const T*>(p.gates) + b * p.sn + c;
  const T* dy = static_cast<const T*>(p.dy) + b * p.T * p.D + c;
  T* dg = static_cast<T*>(p.dgates) + b * p.T * 3 * p.D + c;
  const int64_t nD = p.n * p.D, row = b * p.D + c;

  float sp[V], ratio[V], R[V], acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sp[j] = ratio[j] = R[j] = acc[j] = 0.f;
  if (on) {
    load_decay<V>(p.decay, p.decay_bf16, c, sp);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      ratio[j] = decay_ratio(sp[j]);
      sp[j] = softplus_f(sp[j]);
      if (p.dlast) R[j] = p.dlast[row + j];
    }
    for (int k = p.S - 1; k > seg; --k) {
#pragma unroll
      for (int j = 0; j < V; ++j) R[j] = fmaf(p.sum_a[k * nD + row + j], R[j], p.sum_b[k * nD + row + j]);
    }
  }

  int buf = 0;
  const int64_t tiles = s1 > s0 ? (s1 - s0 + kBwdTile - 1) / kBwdTile : 0;
  for (int64_t i = tiles - 1; i >= 0; --i, buf ^= 1) {
    const int64_t tile = s0 + i * kBwdTile;
    const int64_t s = tile + tg * K;
    typename io::raw rx[K], rr[K], ri[K], rd[K];
    bool live[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t pos = p.reverse ? p.T - 1 - (s + k) : s + k;
      live[k] = on && s + k < s1 && pos < len;
      rx[k] = rr[k] = ri[k] = rd[k] = typename io::raw();
      if (live[k]) {
        const T* q = gx + pos * p.st;
        rx[k] = io::load(q);
        rr[k] = io::load(q + p.D);
        ri[k] = io::load(q + 2 * p.D);
        rd[k] = io::load(dy + pos * p.D);
      }
    }
    float h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = on ? p.kept[(b * chunks + tile / kChunk) * p.D + c + j] : 0.f;

    float a[K][V], ms[K][V], sx[K][V], s1m[K][V], r1m[K][V], Lv[K][V], ak[K][V];
    float A[V], B[V], G[V];
#pragma unroll
    for (int j = 0; j < V; ++j) A[j] = 1.f, B[j] = G[j] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float q;
        const float rho = sigmoid_f(io::get(rr[k], j));
        const float L = live[k] ? -sp[j] * rho : 0.f;
        decay_of(L, a[k][j], q);
        const float m2 = q * (1.0f + a[k][j]), im = inv_scale(m2), m = m2 * im;
        const float sg = sigmoid_f(io::get(ri[k], j)), x = io::get(rx[k], j);
        Lv[k][j] = L * a[k][j];
        ak[k][j] = a[k][j] * a[k][j] * (-L * im);
        sx[k][j] = sg * x;
        ms[k][j] = m * sg;
        s1m[k][j] = x * (1.0f - sg);
        r1m[k][j] = 1.0f - rho;
        A[j] *= a[k][j];
        B[j] = fmaf(a[k][j], B[j], m * sx[k][j]);
      }
    }
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
#pragma unroll
      for (int j = 0; j < V; ++j) G[j] = a[k][j] * (io::get(rd[k], j) + G[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      lds_a[buf][tg][cl * V + j] = A[j];
      lds_b[buf][tg][cl * V + j] = B[j];
      lds_g[buf][tg][cl * V + j] = G[j];
    }
    __syncthreads();
    float g[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      for (int t = 0; t < tg; ++t) h[j] = fmaf(lds_a[buf][t][cl * V + j], h[j], lds_b[buf][t][cl * V + j]);
    }
#pragma unroll
    for (int t = kTG - 1; t >= 0; --t) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (t == tg) g[j] = R[j];
        R[j] = fmaf(lds_a[buf][t][cl * V + j], R[j], lds_g[buf][t][cl * V + j]);
      }
    }
    float hp[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        hp[k][j] = h[j];
        h[j] = fmaf(a[k][j], h[j], ms[k][j] * io::get(rx[k], j));
      }
    }
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
      float ox[V], orr[V], oi[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float gt = io::get(rd[k], j) + g[j];
        g[j] = a[k][j] * gt;
        const float w = gt * fmaf(Lv[k][j], hp[k][j], sx[k][j] * ak[k][j]);
        const float dx = gt * ms[k][j];
        acc[j] += w;
        ox[j] = live[k] ? dx : 0.f;
        orr[j] = live[k] ? w * r1m[k][j] : 0.f;
        oi[j] = live[k] ? dx * s1m[k][j] : 0.f;
      }
      if (on && s + k < s1) {
        T* q = dg + (p.reverse ? p.T - 1 - (s + k) : s + k) * 3 * p.D;
        io::store(q, ox);
        io::store(q + p.D, orr);
        io::store(q + 2 * p.D, oi);
      }
    }
  }
  // sum_t w of the segment over the time groups, in order
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) lds_a[0][tg][cl * V + j] = acc[j];
  __syncthreads();
  if (on && tg == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float t = 0.f;
      for (int g = 0; g < kTG; ++g) t += lds_a[0][g][cl * V + j];
      if (p.dlam) p.dlam[seg * nD + row + j] = t * ratio[j];
      if (p.dstate && seg == 0) p.dstate[row + j] = R[j];
    }
  }
}

__global__ __launch_bounds__(kThreads) void scan_dlam_kernel(const float* __restrict__ part, int S, int64_t nD,
                                                             float* __restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= nD) return;
  float t = 0.f;
  for (int s = 0; s < S; ++s) t += part[s * nD + i];
  out[i] = t;
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void scan_step_kernel(const T* __restrict__ gates, const void* __restrict__ decay,
                                                             int decay_bf16, float* __restrict__ state,
                                                             T* __restrict__ out, int64_t n, int64_t D, int64_t sn) {
  typedef vec_io<T, V> io;
  const int64_t Dv = D / V;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n * Dv) return;
  const int64_t b = i / Dv, c = (i - b * Dv) * V;
  const T* g = gates + b * sn + c;
  const typename io::raw rx = io::load(g), rr = io::load(g + D), ri = io::load(g + 2 * D);
  const typename vec_io<float, V>::raw rh = vec_io<float, V>::load(state + b * D + c);
  float lam[V], h[V];
  load_decay<V>(decay, decay_bf16, c, lam);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float a, q;
    decay_of(-softplus_f(lam[j]) * sigmoid_f(io::get(rr, j)), a, q);
    const float m2 = q * (1.0f + a);
    h[j] = fmaf(a, vec_io<float, V>::get(rh, j), m2 * inv_scale(m2) * sigmoid_f(io::get(ri, j)) * io::get(rx, j));
  }
  vec_io<float, V>::store(state + b * D + c, h);
  io::store(out + b * D + c, h);
}

// Segments of T for n samples of D channels: enough blocks to fill the GPU, whole tiles each.
void segments_of(int64_t n, int64_t T, int64_t D, int V, int* S, int64_t* seg) {
  const int64_t rows = n * dpk_cdiv(D, kCL * V), tiles = dpk_cdiv(T, kFwdTile);
  int64_t want = rows > 0 ? dpk_cdiv(kWantBlocks, rows) : 1;
  if (rows * 2 > kWantBlocks) want = 1;
  if (want > kMaxSegments) want = kMaxSegments;
  if (want > tiles) want = tiles;
  if (want < 1) want = 1;
  const int64_t per = dpk_cdiv(tiles > 0 ? tiles : 1, want);
  *S = static_cast<int>(dpk_cdiv(tiles > 0 ? tiles : 1, per));
  *seg = per * kFwdTile;
}

int vec_of(int64_t D, int dtype, int64_t sn, int64_t st, int64_t n, int64_t T, std::initializer_list<const void*> elems,
           std::initializer_list<const void*> floats) {
  for (int V = 4; V > 1; V /= 2) {
    bool ok = D % V == 0 && (n == 1 || sn % V == 0) && (T == 1 || st % V == 0);
    for (const void* e : elems) ok = ok && dpk_aligned(e, dpk_elsize(dtype) * V);
    for (const void* f : floats) ok = ok && dpk_aligned(f, 4 * V);
    if (ok) return V;
  }
  return 1;
}

int check_common(const char* fn, const void* gates, int dtype, const void* decay, int decay_dtype, int64_t n, int64_t T,
                 int64_t D, int64_t sn, int64_t st) {
  DPK_REQUIRE(n >= 0 && T >= 0 && D >= 0, DPK_E_SHAPE, "%s: negative size (n=%lld T=%lld D=%lld)", fn, (long long)n,
              (long long)T, (long long)D);
  DPK_REQUIRE(dpk_dtype_ok(dtype) && dpk_dtype_ok(decay_dtype), DPK_E_DTYPE, "%s: dtype %d / %d not supported", fn, dtype,
              decay_dtype);
  if (n == 0 || D == 0) return DPK_OK;
  DPK_REQUIRE(decay, DPK_E_ARG, "%s: decay is NULL", fn);
  DPK_REQUIRE(gates || T == 0, DPK_E_ARG, "%s: gates is NULL", fn);
  DPK_REQUIRE(dpk_aligned(gates, dpk_elsize(dtype)) && dpk_aligned(decay, dpk_elsize(decay_dtype)), DPK_E_ALIGN,
              "%s: gates or decay not aligned to its element size", fn);
  DPK_REQUIRE(sn >= 0 && st >= 0, DPK_E_ARG, "%s: negative stride", fn);
  DPK_REQUIRE(n * dpk_cdiv(D, kCL) * kMaxSegments <= DPK_MAX_GRID_X, DPK_E_SHAPE, "%s: n * D too large", fn);
  return DPK_OK;
}

}  // namespace

extern "C" size_t dpk_gated_scan_workspace_bytes(int64_t n, int64_t T, int64_t D) {
  if (n <= 0 || T <= 0 || D <= 0) return 0;
  int S;
  int64_t seg, most = 1;
  for (int V = 1; V <= 4; V *= 2) {  // whichever width the pointers allow
    segments_of(n, T, D, V, &S, &seg);
    if (S > most) most = S;
  }
  return most > 1 ? dpk_align_up(static_cast<size_t>(3) * most * n * D * 4, 256) : 0;
}

extern "C" int dpk_gated_scan(const void* gates, int dtype, const void* decay, int decay_dtype, const float* state,
                              const int64_t* lengths, void* out, float* last, float* kept, int64_t n, int64_t T, int64_t D,
                              int64_t gates_stride_n, int64_t gates_stride_t, int reverse, void* ws, size_t ws_bytes,
                              dpk_stream_t stream) {
  const char* fn = "dpk_gated_scan";
  if (int rc = check_common(fn, gates, dtype, decay, decay_dtype, n, T, D, gates_stride_n, gates_stride_t)) return rc;
  DPK_REQUIRE(reverse == 0 || reverse == 1, DPK_E_ARG, "%s: reverse must be 0 or 1", fn);
  if (n == 0 || D == 0) return DPK_OK;
  DPK_REQUIRE(last && (out || T == 0), DPK_E_ARG, "%s: out or last is NULL", fn);
  DPK_REQUIRE(dpk_aligned(out, dpk_elsize(dtype)) && dpk_aligned(last, 4) && dpk_aligned(state, 4) && dpk_aligned(kept, 4) &&
                  dpk_aligned(lengths, 8),
              DPK_E_ALIGN, "%s: a tensor is not aligned to its element size", fn);
  const int V = vec_of(D, dtype, gates_stride_n, gates_stride_t, n, T, {gates, out}, {last, state, kept});
  ScanArgs p = {gates, decay, state, lengths, out, last, kept, nullptr, nullptr, n, T, D, gates_stride_n, gates_stride_t,
                decay_dtype == DPK_BF16, reverse, 1, 0};
  segments_of(n, T, D, V, &p.S, &p.seg);
  if (p.S > 1) {
    DPK_REQUIRE(ws && ws_bytes >= dpk_gated_scan_workspace_bytes(n, T, D), DPK_E_WORKSPACE, "%s: workspace too small (%zu)",
                fn, ws_bytes);
    DPK_REQUIRE(dpk_aligned(ws, 16), DPK_E_ALIGN, "%s: workspace not 16-byte aligned", fn);
    p.sum_a = static_cast<float*>(ws);
    p.sum_b = p.sum_a + static_cast<int64_t>(p.S) * n * D;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t rows = n * dpk_cdiv(D, kCL * V);
#define DPK_SCAN_FWD(TT, VV)                                                                                              \
  do {                                                                                                                    \
    if (p.S > 1)                                                                                                          \
      hipLaunchKernelGGL((scan_fwd_kernel<TT, VV, true>), dim3((unsigned)(rows * (p.S - 1))), dim3(kThreads), 0, s, p);   \
    hipLaunchKernelGGL((scan_fwd_kernel<TT, VV, false>), dim3((unsigned)(rows * p.S)), dim3(kThreads), 0, s, p);          \
  } while (0)
  if (dtype == DPK_BF16) {
    if (V == 4) DPK_SCAN_FWD(bf16_t, 4);
    else if (V == 2) DPK_SCAN_FWD(bf16_t, 2);
    else DPK_SCAN_FWD(bf16_t, 1);
  } else {
    if (V == 4) DPK_SCAN_FWD(float, 4);
    else if (V == 2) DPK_SCAN_FWD(float, 2);
    else DPK_SCAN_FWD(float, 1);
  }
#undef DPK_SCAN_FWD
  DPK_LAUNCH_CHECK(fn);
  return DPK_OK;
}

extern "C" int dpk_gated_scan_backward(const void* gates, int dtype, const void* decay, int decay_dtype, const float* kept,
                                       const int64_t* lengths, const void* grad_out, const float* grad_last,
                                       void* grad_gates, float* grad_decay, float* grad_state, int64_t n, int64_t T,
                                       int64_t D, int64_t gates_stride_n, int64_t gates_stride_t, int reverse, void* ws,
                                       size_t ws_bytes, dpk_stream_t stream) {
  const char* fn = "dpk_gated_scan_backward";
  if (int rc = check_common(fn, gates, dtype, decay, decay_dtype, n, T, D, gates_stride_n, gates_stride_t)) return rc;
  DPK_REQUIRE(reverse == 0 || reverse == 1, DPK_E_ARG, "%s: reverse must be 0 or 1", fn);
  if (n == 0 || D == 0) return DPK_OK;
  DPK_REQUIRE((kept && grad_out && grad_gates) || T == 0, DPK_E_ARG, "%s: kept, grad_out or grad_gates is NULL", fn);
  DPK_REQUIRE(dpk_aligned(grad_out, dpk_elsize(dtype)) && dpk_aligned(grad_gates, dpk_elsize(dtype)) && dpk_aligned(kept, 4) &&
                  dpk_aligned(grad_last, 4) && dpk_aligned(grad_decay, 4) && dpk_aligned(grad_state, 4) &&
                  dpk_aligned(lengths, 8),
              DPK_E_ALIGN, "%s: a tensor is not aligned to its element size", fn);
  const int V = vec_of(D, dtype, gates_stride_n, gates_stride_t, n, T, {gates, grad_out, grad_gates},
                       {kept, grad_last, grad_decay, grad_state});
  ScanBwdArgs p = {gates, decay, kept, lengths, grad_out, grad_last, grad_gates, grad_state, grad_decay, nullptr, nullptr,
                   n, T, D, gates_stride_n, gates_stride_t, decay_dtype == DPK_BF16, reverse, 1, 0};
  segments_of(n, T, D, V, &p.S, &p.seg);
  if (p.S > 1) {
    DPK_REQUIRE(ws && ws_bytes >= dpk_gated_scan_workspace_bytes(n, T, D), DPK_E_WORKSPACE, "%s: workspace too small (%zu)",
                fn, ws_bytes);
    DPK_REQUIRE(dpk_aligned(ws, 16), DPK_E_ALIGN, "%s: workspace not 16-byte aligned", fn);
    p.sum_a = static_cast<float*>(ws);
    p.sum_b = p.sum_a + static_cast<int64_t>(p.S) * n * D;
    if (grad_decay) p.dlam = p.sum_b + static_cast<int64_t>(p.S) * n * D;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t rows = n * dpk_cdiv(D, kCL * V);
#define DPK_SCAN_BWD(TT, VV)                                                                                            \
  do {                                                                                                                  \
    if (p.S > 1)                                                                                                        \
      hipLaunchKernelGGL((scan_bwd_summary_kernel<TT, VV>), dim3((unsigned)(rows * p.S)), dim3(kThreads), 0, s, p);     \
    hipLaunchKernelGGL((scan_bwd_kernel<TT, VV>), dim3((unsigned)(rows * p.S)), dim3(kThreads), 0, s, p);               \
  } while (0)
  if (dtype == DPK_BF16) {
    if (V == 4) DPK_SCAN_BWD(bf16_t, 4);
    else if (V == 2) DPK_SCAN_BWD(bf16_t, 2);
    else DPK_SCAN_BWD(bf16_t, 1);
  } else {
    if (V == 4) DPK_SCAN_BWD(float, 4);
    else if (V == 2) DPK_SCAN_BWD(float, 2);
    else DPK_SCAN_BWD(float, 1);
  }
#undef DPK_SCAN_BWD
  if (p.S > 1 && grad_decay)
    hipLaunchKernelGGL(scan_dlam_kernel, dim3((unsigned)dpk_cdiv(n * D, kThreads)), dim3(kThreads), 0, s, p.dlam, p.S, n * D,
                       grad_decay);
  DPK_LAUNCH_CHECK(fn);
  return DPK_OK;
}

extern "C" int dpk_gated_scan_step(const void* gates, int dtype, const void* decay, int decay_dtype, float* state, void* out,
                                   int64_t n, int64_t D, int64_t gates_stride_n, dpk_stream_t stream) {
  const char* fn = "dpk_gated_scan_step";
  if (int rc = check_common(fn, gates, dtype, decay, decay_dtype, n, 1, D, gates_stride_n, 0)) return rc;
  if (n == 0 || D == 0) return DPK_OK;
  DPK_REQUIRE(state && out, DPK_E_ARG, "%s: state or out is NULL", fn);
  DPK_REQUIRE(dpk_aligned(out, dpk_elsize(dtype)) && dpk_aligned(state, 4), DPK_E_ALIGN,
              "%s: a tensor is not aligned to its element size", fn);
  const int V = vec_of(D, dtype, gates_stride_n, 0, n, 1, {gates, out}, {state});
  const unsigned grid = static_cast<unsigned>(dpk_cdiv(n * (D / V), kThreads));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int db = decay_dtype == DPK_BF16;
#define DPK_SCAN_STEP(TT, VV)                                                                                              \
  hipLaunchKernelGGL((scan_step_kernel<TT, VV>), dim3(grid), dim3(kThreads), 0, s, static_cast<const TT*>(gates), decay, db, \
                     state, static_cast<TT*>(out), n, D, gates_stride_n)
  if (dtype == DPK_BF16) {
    if (V == 4) DPK_SCAN_STEP(bf16_t, 4);
    else if (V == 2) DPK_SCAN_STEP(bf16_t, 2);
    else DPK_SCAN_STEP(bf16_t, 1);
  } else {
    if (V == 4) DPK_SCAN_STEP(float, 4);
    else if (V == 2) DPK_SCAN_STEP(float, 2);
    else DPK_SCAN_STEP(float, 1);
  }
#undef DPK_SCAN_STEP
  DPK_LAUNCH_CHECK(fn);
  return DPK_OK;
}
