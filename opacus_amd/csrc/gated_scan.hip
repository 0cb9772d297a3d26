// The gated linear recurrence of the DPGatedRNN layer, forward, backward and one token at a time.
//
//   gates[n,T,3D] = values x | decay gates r | input gates i,   decay lam[D]
//   rho = sigma(r);  L = -softplus(lam) rho;  a = exp(L);  u = sqrt(1 - a^2) sigma(i) x
//   h_t = a_t h_{t-1} + u_t,   out_t = h_t
//
// The recurrence is a composition of affine maps h -> A h + B, so T is cut at will. A block takes one
// tile of positions for 32 * V channels of a sample: every thread runs K positions of its channels in
// registers, the block's time groups exchange their (A, B) through lanes and LDS, and the tiles of a
// row pass the state on in one launch (see "the chain" below), or one block walks through all of them where
// that is faster (bwd_walks), so every input is read once and every output written once. What is folded, and in which
// order, depends on sizes and alignment alone: the same bits on every run. n is among the sizes backward (bwd_walks), so a
// sample's gradients are not the same bits in every batch: a walking thread adds up the decay's gradient over all of its
// positions, the chain tile by tile.
//
// Backward: g_t = dy_t + a_{t+1} g_{t+1} runs the same maps the other way (same A, other B), and
//   q = 1 - a,  m = sqrt(q (1 + a)),  kappa = -L / m,  s = sigma(i)
//   dx = g m s;  di = dx x (1 - s);  w = g (L a h_{t-1} + s x a^2 kappa);  dr = w (1 - rho)
//   dlam[sample] = sigma(lam) / softplus(lam) * sum_t w
// (dL/dr = L (1 - rho) and dL/dlam = L sigma(lam) / softplus(lam), so w = L dloss/dL serves both; in
// this form nothing is divided by m alone, which vanishes as the gate closes.) h_{t-1} is formed
// again from the fp32 state the forward pass kept at every 64th position, so no rounded output
// enters a gradient.
//
// Bounds, at 16 x 1024 x 2048, kernels alone, inputs in no cache: forward bf16 59 us for 272 MB (4.6 TB/s; a large copy
// reaches 4.9 to 5.4), fp32 110 us for 541 MB (4.9 TB/s): memory. Backward fp32 187 us for 948 MB (5.1 TB/s): memory.
// Backward bf16 106 us for 478 MB (4.5 TB/s) in a loop of such calls, 101 us among other kernels: half the cycles issue
// arithmetic (55 vector instructions an element, 5 of them transcendental), and the two waves a SIMD that their
// registers leave cover the loads for the rest. There a block walks: 109 us a call in a loop, in the chain 119, about 10
// of them its clearing and the sum of the decay gradients. Tried for the walk and slower (us a call in that loop): the
// next tile's inputs sent ahead into registers (116 us, fp32 242), three waves (129 us). For the chain:
// 4 positions a thread in blocks of 512 (four waves a SIMD, 130 us), two waves with nothing spilled (134 us),
// four with spills (211 us against 126 then), two rows a block with the second one's inputs sent ahead into
// LDS (140 us against 126 then). One 16384-token row of 2048 channels: 66 us for 268 MB (4.1 TB/s), with the clearing
// and the launches 80 us a call (70 with the same inputs call after call; a summary launch in front instead of the
// chain took 127 us then).
// Spills: the chain forward in bf16 4 registers (of the 128 that four waves a SIMD have), the chain backward 7 in bf16
// and 6 in fp32 (of the 168 that three have).
#include <initializer_list>

#include "vec_io.h"

namespace {

constexpr int kThreads = 256;            // of the forward kernel and the small ones
constexpr int kBwdThreads = 256;
constexpr int kCL = 32;                  // lanes across channels: a wave holds two time groups
constexpr int kChunk = DPK_SCAN_CHUNK;   // positions between kept states
constexpr int kBwdK = 8;                 // positions per thread
constexpr int kBwdTile = kBwdThreads / kCL * kBwdK;  // 64
constexpr int kFwdTile = 128;            // forward: 16 positions per thread, or 8 where T is 64 at most or a block walks
constexpr int kWalkTile = 64;
static_assert(kBwdTile == kChunk && kFwdTile % kChunk == 0, "tiles start at kept states");
// Byte offsets inside a tile are 32 bits wide.
constexpr int64_t kMaxStride = DPK_SCAN_MAX_STRIDE;
static_assert(kMaxStride == (1LL << 31) / (kFwdTile * 4) - 1, "the largest offset inside a tile of fp32 fits 31 bits");

// softplus(v) = max(v, 0) + log1p(exp(-|v|)), with log1p(e) = log(1 + e) * e / ((1 + e) - 1): the
// quotient corrects what the rounding of 1 + e did, so the result keeps its relative accuracy as
// e vanishes. Hardware exp2, log2 and reciprocal.
__device__ __forceinline__ float softplus_f(float v) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(v) * kLog2e), u = 1.0f + e, d = u - 1.0f;
  const float l = d > 0.f ? __builtin_amdgcn_logf(u) * 0.69314718055994531f * (e * __builtin_amdgcn_rcpf(d)) : e;
  return fmaxf(v, 0.f) + l;
}
// For the decay gates of one position: L = -softplus(lam) sigma(r), a = exp(L) and q = 1 - a, each
// to its own relative accuracy: q = -L P(L) while L > -0.7, P the degree-5 polynomial nearest to
// (exp(L) - 1) / L there (1e-8 of it off; found by Remez exchange), q = 1 - a beyond. A layer starts out
// with every L in the polynomial's range; the exponentials are behind one branch for the V elements,
// which a wave takes only if one of its lanes needs it.
template <int V>
__device__ __forceinline__ void decay_of(const float (&L)[V], float (&a)[V], float (&q)[V]) {
  float low = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    low = fminf(low, L[j]);
    float p = fmaf(L[j], 0.0010301340371370316f, 0.008062456734478474f);
    p = fmaf(L[j], p, 0.04156935214996338f);
    p = fmaf(L[j], p, 0.16665059328079224f);
    p = fmaf(L[j], p, 0.4999990165233612f);
    p = fmaf(L[j], p, 1.0f);
    q[j] = -L[j] * p;
    a[j] = 1.0f - q[j];
  }
  if (__any(low <= -0.7f)) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float e = __builtin_amdgcn_exp2f(L[j] * kLog2e);
      const bool far = L[j] <= -0.7f;
      a[j] = far ? e : a[j];
      q[j] = far ? 1.0f - e : q[j];
    }
  }
}
// 1 / sqrt(1 - a^2) from 1 - a^2. A zero gives a finite factor, so that m = (1 - a^2) * this and
// kappa = -L * this are zero there.
__device__ __forceinline__ float inv_scale(float q2) { return __builtin_amdgcn_rsqf(fmaxf(q2, 1e-37f)); }

// ---- the chain: tiles of one row hand the state on within a launch -----------------------------
//
// A row is 32 * V channels of one sample; its tiles are numbered by a ticket each block draws when
// it starts, so a block only ever waits for blocks that are already running and that never wait
// for it. Every tile but the row's last publishes its (A, B); 16 tiles form a run, and the last
// tile of a run publishes the state after it. A tile waits for the (A, B) of the tiles before it in its
// run and for the state the run started from, and folds them in position order. What it adds up
// never depends on timing, so the bits repeat; the serial part of a row is one hop per run.
// A word is 64 bits, stored and read whole at agent scope (the XCDs' L2s are not coherent), with
// the pattern kEmpty in its low half until it is written; a NaN is published as the usual quiet one.
// (One row of 128 tiles of 2048 channels, same inputs: 68 us with runs of 16, 70 with 8, 32 or 64; two rows backward:
// 123, 125, 124, 132.)
constexpr int kRun = 16;
constexpr uint32_t kEmpty = 0xffffffffu;

struct Chain {
  uint32_t* tickets;  // [rows], zero at the start
  uint64_t* maps;     // [rows, tiles, W]
  uint64_t* states;   // [rows, runs, W]
  int64_t rows;
  int tiles, runs;
};

__device__ __forceinline__ void publish(uint64_t* w, float a, float b) {
  const uint32_t lo = a != a ? 0x7fc00000u : __float_as_uint(a);
  __hip_atomic_store(w, (static_cast<uint64_t>(__float_as_uint(b)) << 32) | lo, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Waits until all V words are written. A block waits microseconds; what would keep it for 2^21 reads (seconds
// of running) is a workspace that another call wrote to meanwhile, against the rules of the C interface. The
// wait then ends with NaN for the state, so that even such a launch drains.
constexpr uint32_t kMostReads = 1u << 21;
template <int V>
__device__ __forceinline__ void await(const uint64_t* w, float* a, float* b) {
  uint64_t v[V];
  bool there = false;
  for (uint32_t reads = 0; !there && reads < kMostReads; ++reads) {
    if (reads) __builtin_amdgcn_s_sleep(1);
    there = true;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      v[j] = __hip_atomic_load(w + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      there = there && static_cast<uint32_t>(v[j]) != kEmpty;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    a[j] = there ? __uint_as_float(static_cast<uint32_t>(v[j])) : __uint_as_float(0x7fc00000u);
    b[j] = there ? __uint_as_float(static_cast<uint32_t>(v[j] >> 32)) : __uint_as_float(0x7fc00000u);
  }
}

// pairs: 16-byte pairs of words; the tickets lie in front of them.
__global__ __launch_bounds__(kThreads) void chain_clear_kernel(uint32_t* tickets, int64_t rows, uint4* pairs, int64_t count) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads, first = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  for (int64_t i = first; i < count; i += step) pairs[i] = make_uint4(kEmpty, kEmpty, kEmpty, kEmpty);
  for (int64_t i = first; i < rows; i += step) tickets[i] = 0;
}

// This block's tile number in its row, in the order of the chain: drawn first, read once the work that
// does not depend on it is under way.
__device__ __forceinline__ void draw_tile(const Chain& ch, int64_t row, int* lds) {
  if (threadIdx.x == 0)
    *lds = ch.tiles == 1 ? 0 : static_cast<int>(__hip_atomic_fetch_add(ch.tickets + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ int drawn_tile(const int* lds) {
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*lds);
}

// Tile t's own map (TA, TB), for the tiles behind it in its run. `owner`: the lanes that hold it.
template <int V>
__device__ __forceinline__ void publish_map(const Chain& ch, int64_t row, int t, int cl, bool owner, const float (&TA)[V],
                                            const float (&TB)[V]) {
  if (owner && t + 1 < ch.tiles && t % kRun + 1 < kRun) {
    uint64_t* w = ch.maps + (row * ch.tiles + t) * (kCL * V) + cl * V;
#pragma unroll
    for (int j = 0; j < V; ++j) publish(w + j, TA[j], TB[j]);
  }
}
// The state that enters tile t, in `in`, which holds the row's first state. All threads call it, TG
// time groups; lds_m: [2][kRun][W], lds_s: [W], used by nothing else.
template <int V, int TG>
__device__ __forceinline__ void state_before(const Chain& ch, int64_t row, int t, int cl, int tg, bool owner,
                                             const float (&TA)[V], const float (&TB)[V], float (&in)[V], float* lds_m,
                                             float* lds_s) {
  constexpr int W = kCL * V;
  const int run = t / kRun, k = t - run * kRun;
  if (t > 0) {
    float x[V], y[V];
    for (int g = tg; g < k; g += TG) {
      await<V>(ch.maps + (row * ch.tiles + run * kRun + g) * W + cl * V, x, y);
#pragma unroll
      for (int j = 0; j < V; ++j) lds_m[g * W + cl * V + j] = x[j], lds_m[(kRun + g) * W + cl * V + j] = y[j];
    }
    if (tg == TG - 1 && run > 0) {
      await<V>(ch.states + (row * ch.runs + run) * W + cl * V, x, y);
#pragma unroll
      for (int j = 0; j < V; ++j) lds_s[cl * V + j] = y[j];
    }
    __syncthreads();
    if (run > 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) in[j] = lds_s[cl * V + j];
    }
    for (int g = 0; g < k; ++g) {
#pragma unroll
      for (int j = 0; j < V; ++j) in[j] = fmaf(lds_m[g * W + cl * V + j], in[j], lds_m[(kRun + g) * W + cl * V + j]);
    }
  }
  if (owner && t + 1 < ch.tiles && k + 1 == kRun) {
    uint64_t* w = ch.states + (row * ch.runs + run + 1) * W + cl * V;
#pragma unroll
    for (int j = 0; j < V; ++j) publish(w + j, 0.f, fmaf(TA[j], in[j], TB[j]));
  }
}

// The same for a block that walks a row: the state lies in LDS from one tile to the next. Every thread has
// passed a barrier since the last tile's owner wrote it, and passes the one here before the next tile's
// maps overwrite what it folded.
template <int V>
__device__ __forceinline__ void pass_state(int t, int cw, bool owner, const float (&TA)[V], const float (&TB)[V], float (&in)[V],
                                           float* lds_s) {
  if (t > 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) in[j] = lds_s[cw + j];
  }
  __syncthreads();
  if (owner) {
#pragma unroll
    for (int j = 0; j < V; ++j) lds_s[cw + j] = fmaf(TA[j], in[j], TB[j]);
  }
}

struct ScanArgs {
  const void* gates;
  const void* decay;
  const float* state;      // [n,D] or null
  const int64_t* lengths;  // [n] or null
  void* out;
  float* last;
  float* kept;             // [n, ceil(T/chunk), D] or null
  int64_t n, T, D, sn, st;
  int decay_bf16, reverse;
  Chain ch;
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
  float* dlam;             // [tiles,n,D] (the result itself if a block takes the whole row) or null
  int64_t n, T, D, sn, st;
  int decay_bf16, reverse;
  Chain ch;
};

template <int V>
__device__ __forceinline__ void load_decay(const void* decay, int is_bf16, int64_t c, float* lam) {
#pragma unroll
  for (int j = 0; j < V; ++j)
    lam[j] = is_bf16 ? bf16_to_f32(static_cast<const bf16_t*>(decay)[c + j]) : static_cast<const float*>(decay)[c + j];
}

// The row of a block: consecutive block numbers walk the rows, so that all rows advance together.
// Blocks go to the XCDs in turn; where a row is one 128-byte line wide (2-byte elements), each XCD gets neighbouring rows
// instead, so that it walks through contiguous memory (16 x 1024 x 2048 bf16 backward: 128 -> 118 us; wider rows
// do not gain: fp32 forward 110 -> 120 us, backward 200 -> 197 us).
template <typename T>
__device__ __forceinline__ int64_t row_of(int64_t rows) {
  const uint32_t n = static_cast<uint32_t>(rows), i = blockIdx.x % n;
  return sizeof(T) == 2 ? xcd_contiguous_id(i, n) : i;
}

// softplus of the decays of V channels from c on; 0 behind the last channel
template <int V>
__device__ __forceinline__ void softplus_of(const void* decay, int is_bf16, int64_t D, int64_t c, float (&sp)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) sp[j] = 0.f;
  if (c >= D) return;
  load_decay<V>(decay, is_bf16, c, sp);
#pragma unroll
  for (int j = 0; j < V; ++j) sp[j] = softplus_f(sp[j]);
}

__device__ __forceinline__ int64_t live_length(const int64_t* lengths, int64_t b, int64_t T) {
  if (!lengths) return T;
  const int64_t l = lengths[b];
  return l < 0 ? 0 : (l < T ? l : T);
}

// The positions of one tile, in the order of the scan: local position l is position
// (reverse ? T - 1 - s0 - l : s0 + l); those of [lo, hi) are live, those below count exist. `at(l)` is the
// element offset of l from the tile's lowest position at the given stride.
struct Tile {
  int64_t low;  // lowest position
  int lo, hi, count;
  bool reverse;
  __device__ __forceinline__ int at(int l, int stride) const { return (reverse ? count - 1 - l : l) * stride; }
};
// Where position k of a thread's K lies in a FULL tile: the same 32-bit byte offset for all k, and
// for each k a step of the block's base, which is scalar arithmetic.
template <int K>
__device__ __forceinline__ uint32_t first_of(const Tile& t, int tg, int stride_bytes) {
  return (t.reverse ? t.count - K - tg * K : tg * K) * stride_bytes;
}
template <int K>
__device__ __forceinline__ int64_t step_of(const Tile& t, int k, int stride) {
  return static_cast<int64_t>(t.reverse ? K - 1 - k : k) * stride;
}

template <typename T, int V>
__device__ __forceinline__ typename vec_io<T, V>::raw load_at(const T* base, uint32_t bytes) {
  return vec_io<T, V>::load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + bytes));
}
template <typename T, int V>
__device__ __forceinline__ void store_at(T* base, uint32_t bytes, const float* v) {
  vec_io<T, V>::store(reinterpret_cast<T*>(reinterpret_cast<char*>(base) + bytes), v);
}
template <int SIZE>
__device__ __forceinline__ Tile tile_of(int64_t T, int64_t len, int64_t s0, int reverse) {
  Tile t;
  t.reverse = reverse != 0;
  t.count = static_cast<int>(T - s0 < SIZE ? T - s0 : SIZE);
  t.low = t.reverse ? T - s0 - t.count : s0;
  // live positions are those below len: in scan order a prefix, or in reverse a suffix
  int64_t n = len - t.low;
  n = n < 0 ? 0 : (n < t.count ? n : t.count);
  t.lo = t.reverse ? t.count - static_cast<int>(n) : 0;
  t.hi = t.reverse ? t.count : static_cast<int>(n);
  return t;
}

// The value of the wave's other time group.
template <int V>
__device__ __forceinline__ void other_group(const float (&v)[V], float (&o)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = __shfl_xor(v[j], 32, DPK_WAVE);
}
// P = the composition of the waves [from, to) in steps of `step`, whose maps lie in LDS. The bounds
// are the same for the whole wave, so nothing is folded that a lane does not need.
template <int V>
__device__ __forceinline__ void fold_waves(const float (*la)[kCL * V], const float (*lb)[kCL * V], int cw, int from, int to,
                                           int step, float (&PA)[V], float (&PB)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) PA[j] = 1.f, PB[j] = 0.f;
  for (int w = from; w != to; w += step) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float a = la[w][cw + j];
      PB[j] = fmaf(a, PB[j], lb[w][cw + j]);
      PA[j] *= a;
    }
  }
}

// FULL: every position and channel of the tile is live. WALK: the block takes the tiles of its row one after the
// other, and the state between them lies in lds_s.
template <typename T, int V, int K, bool FULL, bool WALK>
__device__ __forceinline__ void fwd_tile(const ScanArgs& p, int t, int64_t r, int64_t b, int64_t cb, const Tile& tl,
                                         const float (&sp)[V], float (*lds_a)[kCL * V], float (*lds_b)[kCL * V], float* lds_m, float* lds_s) {
  typedef vec_io<T, V> io;
  constexpr int W = kCL * V, E = sizeof(T), kWaves = kThreads / DPK_WAVE, TILE = kThreads / kCL * K;
  const int cl = threadIdx.x % kCL, tg = threadIdx.x / kCL;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / DPK_WAVE);
  const bool late = tg & 1;  // the later one of the wave's two time groups
  const int cw = cl * V, c = static_cast<int>(cb) * W + cw;
  const bool on = FULL || c < p.D;
  const int D = static_cast<int>(p.D), st = static_cast<int>(p.st);
  const T* gx = static_cast<const T*>(p.gates) + b * p.sn + tl.low * p.st + cb * W;
  const T *gr = gx + D, *gi = gr + D;

  typename io::raw rx[K], rr[K], ri[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int l = tg * K + k;
    if (!FULL) rx[k] = rr[k] = ri[k] = typename io::raw();
    if (FULL || (on && l >= tl.lo && l < tl.hi)) {
      const uint32_t q = (FULL ? first_of<K>(tl, tg, st * E) : tl.at(l, st * E)) + cw * E;
      const int64_t at = FULL ? step_of<K>(tl, k, st) : 0;
      rx[k] = load_at<T, V>(gx + at, q);
      rr[k] = load_at<T, V>(gr + at, q);
      ri[k] = load_at<T, V>(gi + at, q);
    }
  }
  const int64_t row = b * p.D + c;
  float h[V];
#pragma unroll
  for (int j = 0; j < V; ++j) h[j] = on && p.state && t < (WALK ? 1 : kRun) ? p.state[row + j] : 0.f;
  float a[K][V], u[K][V], A[V], B[V];
#pragma unroll
  for (int j = 0; j < V; ++j) A[j] = 1.f, B[j] = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool live = FULL || (tg * K + k >= tl.lo && tg * K + k < tl.hi);
    float L[V], q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) L[j] = live ? -sp[j] * sigmoid_f(io::get(rr[k], j)) : 0.f;
    decay_of<V>(L, a[k], q);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float m = __builtin_amdgcn_sqrtf(fmaf(q[j], a[k][j], q[j]));
      u[k][j] = m * sigmoid_f(io::get(ri[k], j)) * io::get(rx[k], j);
      A[j] *= a[k][j];
      B[j] = fmaf(a[k][j], B[j], u[k][j]);
    }
  }
  float Ao[V], Bo[V], TA[V], TB[V], PA[V], PB[V];
  other_group<V>(A, Ao);
  other_group<V>(B, Bo);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    TA[j] = A[j] * Ao[j];
    TB[j] = late ? fmaf(A[j], Bo[j], B[j]) : fmaf(Ao[j], B[j], Bo[j]);
    if (!late) lds_a[wave][cw + j] = TA[j], lds_b[wave][cw + j] = TB[j];
  }
  __syncthreads();
  fold_waves<V>(lds_a, lds_b, cw, 0, wave, 1, PA, PB);
  const bool owner = wave == kWaves - 1 && !late;
#pragma unroll
  for (int j = 0; j < V; ++j) TB[j] = fmaf(TA[j], PB[j], TB[j]), TA[j] *= PA[j];  // the tile's map, in the last wave
  if (WALK) {
    pass_state<V>(t, cw, owner, TA, TB, h, lds_s);
  } else {
    publish_map<V>(p.ch, r, t, cl, owner, TA, TB);
    state_before<V, kThreads / kCL>(p.ch, r, t, cl, tg, owner, TA, TB, h, lds_m, lds_s);
  }
  if (on && owner && t + 1 == p.ch.tiles) {
#pragma unroll
    for (int j = 0; j < V; ++j) p.last[row + j] = fmaf(TA[j], h[j], TB[j]);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    h[j] = fmaf(PA[j], h[j], PB[j]);
    h[j] = late ? fmaf(Ao[j], h[j], Bo[j]) : h[j];
  }
  if (!on || tg * K >= tl.count) return;
  if (p.kept && (tg * K) % kChunk == 0) {
    const int64_t s = static_cast<int64_t>(t) * TILE + tg * K;
    vec_io<float, V>::store(p.kept + (b * ((p.T + kChunk - 1) / kChunk) + s / kChunk) * p.D + c, h);
  }
  T* out = static_cast<T*>(p.out) + (b * p.T + tl.low) * p.D + cb * W;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int l = tg * K + k;
    const bool live = FULL || (l >= tl.lo && l < tl.hi);
    float o[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      h[j] = fmaf(a[k][j], h[j], u[k][j]);
      o[j] = live ? h[j] : 0.f;
    }
    if (FULL) store_at<T, V>(out + step_of<K>(tl, k, D), first_of<K>(tl, tg, D * E) + cw * E, o);
    else if (l < tl.count) store_at<T, V>(out, tl.at(l, D * E) + cw * E, o);
  }
}

// One block: one tile of 8 * K positions of 32 * V channels of one sample, or (WALK) all of them in turn.
template <typename T, int V, int K, bool WALK>
__global__ __launch_bounds__(kThreads, WALK ? 2 : sizeof(T) == 2 ? 4 : 3) void scan_fwd_kernel(ScanArgs p) {
  constexpr int W = kCL * V, kWaves = kThreads / DPK_WAVE, TILE = kThreads / kCL * K;
  static_assert(TILE % kChunk == 0 && kChunk % K == 0, "a time group starts where a state is kept");
  __shared__ float lds_a[kWaves][W];
  __shared__ float lds_b[kWaves][W];
  __shared__ float lds_m[WALK ? 1 : 2 * kRun * W];
  __shared__ float lds_s[W];
  __shared__ int lds_t;
  const int64_t cbs = (p.D + W - 1) / W, r = row_of<T>(p.ch.rows), b = r / cbs, cb = r - b * cbs;
  if (!WALK) draw_tile(p.ch, r, &lds_t);
  float sp[V];
  softplus_of<V>(p.decay, p.decay_bf16, p.D, cb * W + (threadIdx.x % kCL) * V, sp);
  int t = WALK ? 0 : drawn_tile(&lds_t);
  if (t >= p.ch.tiles) return;  // never, unless another call used the workspace meanwhile
  const int64_t len = live_length(p.lengths, b, p.T);
  do {
    const Tile tl = tile_of<TILE>(p.T, len, static_cast<int64_t>(t) * TILE, p.reverse);
    if (tl.hi - tl.lo == TILE && (cb + 1) * W <= p.D)
      fwd_tile<T, V, K, true, WALK>(p, t, r, b, cb, tl, sp, lds_a, lds_b, lds_m, lds_s);
    else
      fwd_tile<T, V, K, false, WALK>(p, t, r, b, cb, tl, sp, lds_a, lds_b, lds_m, lds_s);
  } while (WALK && ++t < p.ch.tiles);
}

// acc: this thread's share of the decay's gradient, over its tiles.
template <typename T, int V, bool FULL, bool WALK>
__device__ __forceinline__ void bwd_tile(const ScanBwdArgs& p, int t, int64_t r, int64_t b, int64_t cb, const Tile& tl,
                                         const float (&sp)[V], float (&acc)[V], float (*lds_a)[kCL * V], float (*lds_b)[kCL * V],
                                         float (*lds_g)[kCL * V], float* lds_m, float* lds_s) {
  typedef vec_io<T, V> io;
  constexpr int W = kCL * V, K = kBwdK, E = sizeof(T), kWaves = kBwdThreads / DPK_WAVE;
  const int cl = threadIdx.x % kCL, tg = threadIdx.x / kCL;
  const int cw = cl * V, c = static_cast<int>(cb) * W + cw;
  const bool on = FULL || c < p.D;
  const int D = static_cast<int>(p.D), st = static_cast<int>(p.st);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / DPK_WAVE);
  const bool late = tg & 1;  // the later one of the wave's two time groups
  const int tile = p.ch.tiles - 1 - t;
  const T* gx = static_cast<const T*>(p.gates) + b * p.sn + tl.low * p.st + cb * W;
  const T *gr = gx + D, *gi = gr + D;
  const T* dy = static_cast<const T*>(p.dy) + (b * p.T + tl.low) * p.D + cb * W;

  typename io::raw rx[K], rr[K], ri[K], rd[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int l = tg * K + k;
    if (!FULL) rx[k] = rr[k] = ri[k] = rd[k] = typename io::raw();
    if (FULL || (on && l >= tl.lo && l < tl.hi)) {
      const uint32_t q = (FULL ? first_of<K>(tl, tg, st * E) : tl.at(l, st * E)) + cw * E;
      const uint32_t q1 = (FULL ? first_of<K>(tl, tg, D * E) : tl.at(l, D * E)) + cw * E;
      const int64_t at = FULL ? step_of<K>(tl, k, st) : 0, at1 = FULL ? step_of<K>(tl, k, D) : 0;
      rx[k] = load_at<T, V>(gx + at, q);
      rr[k] = load_at<T, V>(gr + at, q);
      ri[k] = load_at<T, V>(gi + at, q);
      rd[k] = load_at<T, V>(dy + at1, q1);
    }
  }
  const int64_t row = b * p.D + c;
  float h[V], g[V];
  typename vec_io<float, V>::raw kh = typename vec_io<float, V>::raw();
  if (on && p.T > 0) kh = vec_io<float, V>::load(p.kept + (b * p.ch.tiles + tile) * p.D + c);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    h[j] = vec_io<float, V>::get(kh, j);
    g[j] = on && p.dlast && t < (WALK ? 1 : kRun) ? p.dlast[row + j] : 0.f;
  }
  // what the second half needs of each element; the rest is a product or two away
  float a[K][V], ms[K][V], is[K][V], sg[K][V], rho[K][V];  // ms = m s, is = s / m
  float A[V], B[V], G[V];
#pragma unroll
  for (int j = 0; j < V; ++j) A[j] = 1.f, B[j] = G[j] = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool live = FULL || (tg * K + k >= tl.lo && tg * K + k < tl.hi);
    float L[V], q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      rho[k][j] = sigmoid_f(io::get(rr[k], j));
      L[j] = live ? -sp[j] * rho[k][j] : 0.f;
    }
    decay_of<V>(L, a[k], q);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float m2 = fmaf(q[j], a[k][j], q[j]);
      sg[k][j] = sigmoid_f(io::get(ri[k], j));
      is[k][j] = inv_scale(m2) * sg[k][j];
      ms[k][j] = m2 * is[k][j];
      A[j] *= a[k][j];
      B[j] = fmaf(a[k][j], B[j], ms[k][j] * io::get(rx[k], j));
    }
  }
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
#pragma unroll
    for (int j = 0; j < V; ++j) G[j] = a[k][j] * (io::get(rd[k], j) + G[j]);
  }
  // Ao, Bo, Go: the other group's; T: the pair's, then (in wave 0, the first in time) the tile's
  float Ao[V], Bo[V], Go[V], TA[V], TG[V], PA[V], PG[V];
  other_group<V>(A, Ao);
  other_group<V>(B, Bo);
  other_group<V>(G, Go);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    TA[j] = A[j] * Ao[j];
    TG[j] = late ? fmaf(Ao[j], G[j], Go[j]) : fmaf(A[j], Go[j], G[j]);
    if (!late) {
      lds_a[wave][cw + j] = TA[j];
      lds_b[wave][cw + j] = fmaf(Ao[j], B[j], Bo[j]);
      lds_g[wave][cw + j] = TG[j];
    }
  }
  __syncthreads();
  fold_waves<V>(lds_a, lds_g, cw, kWaves - 1, wave, -1, PA, PG);
  const bool owner = wave == 0 && !late;
#pragma unroll
  for (int j = 0; j < V; ++j) TG[j] = fmaf(TA[j], PG[j], TG[j]), TA[j] *= PA[j];
  if (!WALK) publish_map<V>(p.ch, r, t, cl, owner, TA, TG);
  // the states inside the tile, while the words of the chain are on their way
  for (int w = 0; w < wave; ++w) {
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = fmaf(lds_a[w][cw + j], h[j], lds_b[w][cw + j]);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) h[j] = late ? fmaf(Ao[j], h[j], Bo[j]) : h[j];
  // The products below are formed again, not kept from the first half: the empty asm makes the
  // compiler take the factors as new values, which keeps a thread's registers down.
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int j = 0; j < V; ++j) asm volatile("" : "+v"(ms[k][j]), "+v"(sg[k][j]), "+v"(rho[k][j]), "+v"(is[k][j]));
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
  if (WALK) pass_state<V>(t, cw, owner, TA, TG, g, lds_s);
  else state_before<V, kBwdThreads / kCL>(p.ch, r, t, cl, tg, owner, TA, TG, g, lds_m, lds_s);
  if (on && owner && p.dstate && tile == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) p.dstate[row + j] = fmaf(TA[j], g[j], TG[j]);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    g[j] = fmaf(PA[j], g[j], PG[j]);
    g[j] = late ? g[j] : fmaf(Ao[j], g[j], Go[j]);
  }
  T* dg = static_cast<T*>(p.dgates) + (b * p.T + tl.low) * 3 * p.D + cb * W;
  T *dr = dg + D, *di = dr + D;
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
    const int l = tg * K + k;
    const bool live = FULL || (l >= tl.lo && l < tl.hi);
    float ox[V], orr[V], oi[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float gt = io::get(rd[k], j) + g[j], x = io::get(rx[k], j);
      g[j] = a[k][j] * gt;
      // w = g (L a h_{t-1} + s x a^2 kappa) with kappa = -L / m and L = -softplus rho:
      // w / -softplus = a g rho (h_{t-1} - a x s / m)
      const float v = g[j] * rho[k][j] * fmaf(-is[k][j], x * a[k][j], hp[k][j]);
      const float w = -sp[j] * v;
      const float dx = gt * ms[k][j];
      acc[j] += live ? v : 0.f;
      ox[j] = live ? dx : 0.f;
      orr[j] = live ? fmaf(-w, rho[k][j], w) : 0.f;
      oi[j] = live ? dx * fmaf(-x, sg[k][j], x) : 0.f;
    }
    if (FULL || (on && l < tl.count)) {
      const uint32_t q = (FULL ? first_of<K>(tl, tg, 3 * D * E) : tl.at(l, 3 * D * E)) + cw * E;
      const int64_t at = FULL ? step_of<K>(tl, k, 3 * D) : 0;
      store_at<T, V>(dg + at, q, ox);
      store_at<T, V>(dr + at, q, orr);
      store_at<T, V>(di + at, q, oi);
    }
  }
}

// The decay's gradient of the block's tiles, `to` [n,D]: acc summed over the time groups, in order.
template <int V>
__device__ __forceinline__ void store_decay_sums(const ScanBwdArgs& p, float* to, int64_t b, int c, const float (&sp)[V],
                                                 const float (&acc)[V], float (*lds_g)[kCL * V]) {
  const int cw = threadIdx.x % kCL * V, wave = threadIdx.x / DPK_WAVE;
  const bool late = threadIdx.x / kCL & 1;
  float other[V];
  other_group<V>(acc, other);
  __syncthreads();
  if (!late) {
#pragma unroll
    for (int j = 0; j < V; ++j) lds_g[wave][cw + j] = acc[j] + other[j];
  }
  __syncthreads();
  if (c < p.D && wave == 0 && !late) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kBwdThreads / DPK_WAVE; ++w) sum += lds_g[w][cw + j];
      // v lacks the factor -softplus(lam) of w, and dlam = sigma(lam) / softplus(lam) sum_t w;
      // sigma(lam) = 1 - exp(-softplus(lam))
      to[b * p.D + c + j] = expm1f(-sp[j]) * sum;
    }
  }
}

// One block: one tile of 64 positions, or (WALK) all of them in turn, from the row's last to its first.
template <typename T, int V, bool WALK>
__global__ __launch_bounds__(kBwdThreads, WALK ? 2 : 3) void scan_bwd_kernel(ScanBwdArgs p) {
  constexpr int W = kCL * V, kWaves = kBwdThreads / DPK_WAVE;
  __shared__ float lds_a[kWaves][W];
  __shared__ float lds_b[kWaves][W];
  __shared__ float lds_g[kWaves][W];
  __shared__ float lds_m[WALK ? 1 : 2 * kRun * W];
  __shared__ float lds_s[W];
  __shared__ int lds_t;
  const int64_t cbs = (p.D + W - 1) / W, r = row_of<T>(p.ch.rows), b = r / cbs, cb = r - b * cbs;
  if (!WALK) draw_tile(p.ch, r, &lds_t);
  float sp[V];
  softplus_of<V>(p.decay, p.decay_bf16, p.D, cb * W + (threadIdx.x % kCL) * V, sp);
  int t = WALK ? 0 : drawn_tile(&lds_t);  // 0 is the last tile of the scan
  if (t >= p.ch.tiles) return;  // never, unless another call used the workspace meanwhile
  const int64_t len = live_length(p.lengths, b, p.T);
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  do {
    const Tile tl = tile_of<kBwdTile>(p.T, len, static_cast<int64_t>(p.ch.tiles - 1 - t) * kBwdTile, p.reverse);
    if (tl.hi - tl.lo == kBwdTile && (cb + 1) * W <= p.D)
      bwd_tile<T, V, true, WALK>(p, t, r, b, cb, tl, sp, acc, lds_a, lds_b, lds_g, lds_m, lds_s);
    else
      bwd_tile<T, V, false, WALK>(p, t, r, b, cb, tl, sp, acc, lds_a, lds_b, lds_g, lds_m, lds_s);
  } while (WALK && ++t < p.ch.tiles);
  if (p.dlam) {
    float* to = p.dlam + (WALK ? 0 : (p.ch.tiles - 1 - t) * p.n * p.D);
    store_decay_sums<V>(p, to, b, static_cast<int>(cb * W) + threadIdx.x % kCL * V, sp, acc, lds_g);
  }
}

// out[i] = sum over the tiles of part[tile][i], in order: 64 sums a block, its 16 waves on 16 neighbouring
// runs of tiles, and those in order.
__global__ __launch_bounds__(1024) void scan_dlam_kernel(const float* __restrict__ part, int tiles, int64_t nD,
                                                         float* __restrict__ out) {
  __shared__ float lds[16][DPK_WAVE];
  const int lane = threadIdx.x % DPK_WAVE, wave = threadIdx.x / DPK_WAVE, waves = blockDim.x / DPK_WAVE;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * DPK_WAVE + lane;
  const int run = (tiles + waves - 1) / waves, k0 = wave * run, k1 = k0 + run < tiles ? k0 + run : tiles;
  float t = 0.f;
  if (i < nD) {
#pragma unroll 8
    for (int k = k0; k < k1; ++k) t += part[k * nD + i];
  }
  lds[wave][lane] = t;
  __syncthreads();
  if (wave == 0 && i < nD) {
    t = 0.f;
    for (int w = 0; w < waves; ++w) t += lds[w][lane];
    out[i] = t;
  }
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
  float L[V], a[V], q[V];
#pragma unroll
  for (int j = 0; j < V; ++j) L[j] = -softplus_f(lam[j]) * sigmoid_f(io::get(rr, j));
  decay_of<V>(L, a, q);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float m = __builtin_amdgcn_sqrtf(fmaf(q[j], a[j], q[j]));
    h[j] = fmaf(a[j], vec_io<float, V>::get(rh, j), m * sigmoid_f(io::get(ri, j)) * io::get(rx, j));
  }
  vec_io<float, V>::store(state + b * D + c, h);
  io::store(out + b * D + c, h);
}

int tiles_of(int64_t T, int tile) { return T > tile ? static_cast<int>(dpk_cdiv(T, tile)) : 1; }

// The chain's part of the workspace for rows of 32 * V channels: tickets, maps, states.
size_t chain_bytes(int64_t n, int64_t D, int V, int tiles) {
  if (tiles == 1) return 0;
  const size_t rows = static_cast<size_t>(n * dpk_cdiv(D, kCL * V));
  return dpk_align_up(rows * 4, 256) + rows * kCL * V * 8 * (tiles + dpk_cdiv(tiles, kRun));
}
// Sets up and, but where blocks walk, clears the chain of a launch; returns the first byte behind it.
char* chain_of(Chain* ch, int64_t n, int64_t D, int V, int tiles, bool walk, void* ws, hipStream_t s) {
  ch->rows = n * dpk_cdiv(D, kCL * V);
  ch->tiles = tiles;
  ch->runs = static_cast<int>(dpk_cdiv(tiles, kRun));
  if (tiles == 1 || walk) return static_cast<char*>(ws);
  const int64_t W = kCL * V, words = ch->rows * W * (tiles + ch->runs);
  char* at = static_cast<char*>(ws);
  ch->tickets = reinterpret_cast<uint32_t*>(at);
  at += dpk_align_up(static_cast<size_t>(ch->rows) * 4, 256);
  ch->maps = reinterpret_cast<uint64_t*>(at);
  ch->states = ch->maps + ch->rows * tiles * W;
  const int64_t blocks = dpk_cdiv(words, kThreads * 2);  // one 16-byte store a thread
  hipLaunchKernelGGL(chain_clear_kernel, dim3(static_cast<unsigned>(blocks < 8192 ? blocks : 8192)), dim3(kThreads), 0, s,
                     ch->tickets, ch->rows, reinterpret_cast<uint4*>(ch->maps), words / 2);
  return at + words * 8;
}

// Where one block takes all tiles of its row in turn, and no chain is set up. Few tiles: two launches and the
// workspace saved are more than the tiles one after the other cost (us in a loop of calls, chain and walk: forward
// 8 x 256 x 512 fp32 15.8 and 13.0, 64 x 192 x 1024 bf16 30.7 and 21.4, 7 x 333 x 130 fp32 15.8 and 20.6;
// backward 8 x 192 x 512 fp32 19.3 and 14.5, 8 x 256 x 512 19.4 and 18.2, 7 x 333 x 130 19.1 and 25.5).
// Backward also where rows fill the GPU's 512 places for such blocks to 85 % or more, whatever T: they lose nothing by
// waiting for one another (16 x 1024 x 2048 bf16 119 and 109, fp32 201 and 187, 64 x 4096 x 500 bf16 483 and 416;
// but half the rows, 8 x 1024 x 2048 bf16, 54 and 57, and three quarters of the places, 24 x 512 x 2048, 87 and 92).
bool fwd_walks(int64_t T) { return T > kFwdTile && T <= 4 * kWalkTile; }
bool bwd_walks(int64_t n, int64_t T, int64_t D) {
  const int64_t rows = n * dpk_cdiv(D, 2 * kCL), places = dpk_cdiv(rows, 512) * 512;
  return T > kBwdTile && (T <= 3 * kBwdTile || 20 * rows >= 17 * places);
}

int vec_of(int most, int64_t D, int dtype, int64_t sn, int64_t st, int64_t n, int64_t T, std::initializer_list<const void*> elems,
           std::initializer_list<const void*> floats) {
  for (int V = most; V > 1; V /= 2) {
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
  DPK_REQUIRE(3 * D <= kMaxStride && (T <= 1 || st <= kMaxStride), DPK_E_SHAPE,
              "%s: a position's features span more than %lld elements", fn, (long long)kMaxStride);
  // (in floating point: the product of sizes no tensor has must not wrap around)
  const double blocks = static_cast<double>(n) * static_cast<double>(D / kCL + 1) * static_cast<double>(T / kBwdTile + 1);
  DPK_REQUIRE(blocks <= static_cast<double>(DPK_MAX_GRID_X), DPK_E_SHAPE, "%s: n * T * D too large", fn);
  return DPK_OK;
}

}  // namespace

extern "C" size_t dpk_gated_scan_workspace_bytes(int64_t n, int64_t T, int64_t D) {
  if (n <= 0 || T <= kBwdTile || D <= 0 || ((T <= kFwdTile || fwd_walks(T)) && bwd_walks(n, T, D))) return 0;
  const int tiles = tiles_of(T, kBwdTile);  // the backward pass cuts finer
  size_t most = 0;
  for (int V = 1; V <= 2; V *= 2) {  // whichever width the pointers allow
    const size_t need = chain_bytes(n, D, V, tiles);
    if (need > most) most = need;
  }
  return dpk_align_up(most + static_cast<size_t>(tiles) * n * D * 4, 256);
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
  const int V = vec_of(2, D, dtype, gates_stride_n, gates_stride_t, n, T, {gates, out}, {last, state, kept});
  const bool walk = fwd_walks(T);
  const int tiles = tiles_of(T, walk ? kWalkTile : kFwdTile);
  DPK_REQUIRE(dpk_grid_fits(n * dpk_cdiv(D, kCL * V) * tiles, kThreads), DPK_E_SHAPE, "%s: n * T * D too large", fn);
  const size_t need = walk ? 0 : chain_bytes(n, D, V, tiles);
  DPK_REQUIRE(need == 0 || (ws && ws_bytes >= need), DPK_E_WORKSPACE, "%s: workspace too small (%zu < %zu)", fn, ws_bytes, need);
  DPK_REQUIRE(dpk_aligned(ws, 16), DPK_E_ALIGN, "%s: workspace not 16-byte aligned", fn);
  hipStream_t s = static_cast<hipStream_t>(stream);
  ScanArgs p = {gates, decay, state, lengths, out, last, kept, n, T, D, gates_stride_n, gates_stride_t,
                decay_dtype == DPK_BF16, reverse, {}};
  chain_of(&p.ch, n, D, V, tiles, walk, ws, s);
  const dim3 grid(static_cast<unsigned>(p.ch.rows * (walk ? 1 : tiles)));
// 16 positions a thread; 8 where a tile of 128 would be half empty (256 x 64 x 2048 bf16: 92 us with 16,
// 56 with 8; 128 x 128 x 2048: 48 with 16, 63 with 8; 4 x 4096 x 2048: 57 and 69)
#define DPK_SCAN_FWD(TT, VV)                                                                                           \
  do {                                                                                                                 \
    if (walk) hipLaunchKernelGGL((scan_fwd_kernel<TT, VV, 8, true>), grid, dim3(kThreads), 0, s, p);                  \
    else if (T <= kChunk) hipLaunchKernelGGL((scan_fwd_kernel<TT, VV, 8, false>), grid, dim3(kThreads), 0, s, p);      \
    else hipLaunchKernelGGL((scan_fwd_kernel<TT, VV, 16, false>), grid, dim3(kThreads), 0, s, p);                      \
  } while (0)
  if (dtype == DPK_BF16) {
    if (V == 2) DPK_SCAN_FWD(bf16_t, 2);
    else DPK_SCAN_FWD(bf16_t, 1);
  } else {
    if (V == 2) DPK_SCAN_FWD(float, 2);
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
  const int V = vec_of(2, D, dtype, gates_stride_n, gates_stride_t, n, T, {gates, grad_out, grad_gates},
                       {kept, grad_last, grad_decay, grad_state});
  const int tiles = tiles_of(T, kBwdTile);
  const bool walk = bwd_walks(n, T, D), parts = tiles > 1 && !walk && grad_decay;
  DPK_REQUIRE(dpk_grid_fits(n * dpk_cdiv(D, kCL * V) * tiles, kBwdThreads), DPK_E_SHAPE, "%s: n * T * D too large", fn);
  const size_t need = walk ? 0 : chain_bytes(n, D, V, tiles) + (parts ? static_cast<size_t>(tiles) * n * D * 4 : 0);
  DPK_REQUIRE(need == 0 || (ws && ws_bytes >= need), DPK_E_WORKSPACE, "%s: workspace too small (%zu < %zu)", fn, ws_bytes, need);
  DPK_REQUIRE(dpk_aligned(ws, 16), DPK_E_ALIGN, "%s: workspace not 16-byte aligned", fn);
  hipStream_t s = static_cast<hipStream_t>(stream);
  ScanBwdArgs p = {gates, decay, kept, lengths, grad_out, grad_last, grad_gates, grad_state, grad_decay, n, T, D,
                   gates_stride_n, gates_stride_t, decay_dtype == DPK_BF16, reverse, {}};
  char* behind = chain_of(&p.ch, n, D, V, tiles, walk, ws, s);
  if (parts) p.dlam = reinterpret_cast<float*>(behind);
  const dim3 grid(static_cast<unsigned>(p.ch.rows * (walk ? 1 : tiles)));
#define DPK_SCAN_BWD(TT, VV)                                                                                \
  do {                                                                                                      \
    if (walk) hipLaunchKernelGGL((scan_bwd_kernel<TT, VV, true>), grid, dim3(kBwdThreads), 0, s, p);        \
    else hipLaunchKernelGGL((scan_bwd_kernel<TT, VV, false>), grid, dim3(kBwdThreads), 0, s, p);            \
  } while (0)
  if (dtype == DPK_BF16) {
    if (V == 2) DPK_SCAN_BWD(bf16_t, 2);
    else DPK_SCAN_BWD(bf16_t, 1);
  } else {
    if (V == 2) DPK_SCAN_BWD(float, 2);
    else DPK_SCAN_BWD(float, 1);
  }
#undef DPK_SCAN_BWD
  if (parts)
    hipLaunchKernelGGL(scan_dlam_kernel, dim3(static_cast<unsigned>(dpk_cdiv(n * D, DPK_WAVE))),
                       dim3(DPK_WAVE * (tiles <= 32 ? 4 : 16)), 0, s, p.dlam, tiles, n * D, grad_decay);
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
  const int V = vec_of(4, D, dtype, gates_stride_n, 0, n, 1, {gates, out}, {state});
  DPK_REQUIRE(dpk_grid_fits(dpk_cdiv(n * (D / V), kThreads), kThreads), DPK_E_SHAPE, "%s: n * D too large", fn);
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
