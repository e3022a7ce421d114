// recur.cu -- the minGRU recurrence over whole sequences, and its gradient.
//
//   z = sigmoid(zl)   c = hr >= 0 ? hr + 1/2 : sigmoid(hr)
//   h_t = a_t h_{t-1} + z_t c_t,   a_t = 1 - z_t
//
// (the cell of MinGRUBlockGPU, boa_gpu.hpp:652-693).  With g_t the gradient
// that reaches h_t,
//
//   g_t = dh_t + a_{t+1} g_{t+1}
//   dzl = g z a (c - h_{t-1})    dhr = g z c'(hr)    dh0 = a_0 g_0
//
// where c' is 1 for hr >= 0 and c (1 - c) below.  The state is fp32
// throughout.  The forward pass leaves the state before every kSpan-th
// position, and the backward pass recomputes the states between from those:
// it reads the gates and the state's gradient once and never reads h.
//
// Both directions are linear in what they carry: over a run of positions the
// state goes from x to A x + B, with A the product of the run's a.  A group is
// 32 * V chains (a chain is one channel of one chunk) and is taken along the
// time axis by one block, or by a cluster of up to kMaxCluster blocks when
// there are too few groups to fill the GPU.  In a step of the walk every warp
// holds P positions of every chain in registers, forms their (A, B), and
// issues the loads of its next step; the warps' maps meet in shared memory,
// the blocks' in each other's (pushed there, double-buffered, one barrier a
// step); the state that enters a warp's positions is the walk's state with the
// maps before it applied in order, and the outputs come from the registers.
// So the gates are read once, nothing waits on another block outside its
// cluster, and the result does not depend on timing.
#include "kernels.cuh"
#include "ptx.cuh"
#include "train_ops.cuh"

namespace boa {

constexpr int kSpan = 32;         // positions between two saved states
constexpr int kMaxWarps = 16;     // warps of a block
constexpr int kMaxCluster = 8;    // blocks of a cluster (the portable limit)
constexpr int kScanSteps = 8;     // positions a warp holds, forward
constexpr int kGradSteps = 4;     // and backward, which holds twice the values

// n / d for n < 2^31 by a multiplication: with 2^(s-1) < d <= 2^s and
// mul = floor(2^(31+s) / d) + 1, mul d exceeds 2^(31+s) by at most d, and
// n d < 2^(31+s).
struct FastDiv {
  uint32_t d, mul, shift;
};
static FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {d, d == 1 ? 0u : (uint32_t)((1ull << (31 + s)) / d + 1), s ? s - 1 : 0u};
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, FastDiv f) {
  return f.d == 1 ? n : __umulhi(n, f.mul) >> f.shift;
}

__device__ __forceinline__ float ex2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The cell's gates.  Both sigmoids are taken of -|x|, so the exponentials are
// at most 1, the smaller of z and 1 - z comes without a cancellation, and one
// reciprocal of the two denominators' product (1 .. 4) serves both: three
// special-function operations instead of four, which would run out before HBM
// does with 16-bit gates.  The larger of z and 1 - z is 1 minus the smaller,
// so a closed gate keeps the state exactly, however many positions long.
struct Cell {
  float a, z, c;
};
__device__ __forceinline__ Cell mingru_cell(float zl, float hr) {
  constexpr float kLog2e = 1.44269504f;
  const float e = ex2_fast(-fabsf(zl) * kLog2e), f = ex2_fast(-fabsf(hr) * kLog2e);
  const float p = 1.f + e, q = 1.f + f;
  const float r = rcp_fast(p * q);
  const float small = e * (q * r), big = 1.f - small;  // e / p and 1 / p
  Cell k;
  k.z = zl >= 0.f ? big : small;
  k.a = zl >= 0.f ? small : big;
  k.c = hr >= 0.f ? hr + 0.5f : f * (p * r);
  return k;
}

static long long spans_of(int T) { return ((long long)T + kSpan - 1) / kSpan; }
size_t mingru_states_floats(int B, int T, int d) { return (size_t)spans_of(T) * B * d; }

// The map of a run of positions for V chains: x -> A x + B.
template <int V>
struct alignas(8 * V) Map {
  float A[V], B[V];
};
template <int V>
__device__ __forceinline__ Map<V> identity_map() {
  Map<V> m;
#pragma unroll
  for (int v = 0; v < V; ++v) { m.A[v] = 1.f; m.B[v] = 0.f; }
  return m;
}
template <int V>
__device__ __forceinline__ void apply(const Map<V>& m, float (&x)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = __fmaf_rn(m.A[v], x[v], m.B[v]);
}
// m, then n
template <int V>
__device__ __forceinline__ void then(Map<V>& m, const Map<V>& n) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    m.B[v] = __fmaf_rn(n.A[v], m.B[v], n.B[v]);
    m.A[v] *= n.A[v];
  }
}

// Shared memory of a walk.  Everything is double-buffered by the step's
// parity: what a step writes was last read two steps ago, and every warp
// passes one barrier in between.
template <int V>
struct Walk {
  Map<V> warp[2][kMaxWarps][32];      // the warps' maps
  Map<V> block[2][kMaxCluster][32];   // the cluster's blocks' maps (pushed by their owners)
  float state[2][kMaxWarps][32][V];   // the walk's state, left by the group's last warp (no cluster)
};

// Where a warp works.  A block's warps form groups of `warps` (a power of
// two); more than one group per block only when a group's whole sequence fits
// its warps.
struct Place {
  long long chain;
  bool in;
  int b, c, lane, warp, warps, first;  // warp within its group, the group's first warp
  int rank, ranks;                     // block within its cluster
};
template <int V>
__device__ __forceinline__ Place place_of(int warps, int ranks, long long chains, int d, FastDiv by_d) {
  Place p;
  p.lane = threadIdx.x & 31;
  const int w = threadIdx.x >> 5, per = (int)(blockDim.x >> 5) / warps;
  p.warps = warps;
  p.warp = w % warps;
  p.first = w - p.warp;
  p.ranks = ranks;
  p.rank = ranks > 1 ? (int)cluster_rank() : 0;
  const long long group = (long long)(blockIdx.x / ranks) * per + w / warps;
  p.chain = group * (32 * V) + p.lane * V;
  p.in = p.chain < chains;
  p.b = p.in ? (int)div_by((uint32_t)p.chain, by_d) : 0;
  p.c = p.in ? (int)(p.chain - (long long)p.b * d) : 0;
  return p;
}

template <int V>
__device__ __forceinline__ void store_map_cluster(uint32_t addr, const Map<V>& m) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr + 4 * v), "f"(m.A[v]) : "memory");
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr + 4 * (V + v)), "f"(m.B[v]) : "memory");
  }
}

// One step's exchange.  `mine`: the map of this warp's positions, `x`: the
// walk's state before the step; afterwards `s` is the state before this warp's
// positions, and (in a cluster) `x` the state after the step.  REVERSE runs
// from the last warp and block to the first.  Without a cluster the caller
// hands the state on through leave().
template <int V, bool REVERSE>
__device__ __forceinline__ void exchange(Walk<V>& K, const Place& p, int parity, const Map<V>& mine, float (&x)[V],
                                         float (&s)[V], bool first_step) {
  const int order = REVERSE ? p.warps - 1 - p.warp : p.warp;  // place of this warp along the walk
  Map<V>(*maps)[32] = K.warp[parity] + p.first;
  maps[order][p.lane] = mine;
  __syncthreads();
  if (p.ranks == 1) {
    if (!first_step)
#pragma unroll
      for (int v = 0; v < V; ++v) x[v] = K.state[parity][p.first][p.lane][v];
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = x[v];
  } else {
    const int turn = REVERSE ? p.ranks - 1 - p.rank : p.rank;
    if (p.warp < p.ranks) {  // warp r takes the block's map to block r
      Map<V> all = maps[0][p.lane];
      for (int w = 1; w < p.warps; ++w) then<V>(all, maps[w][p.lane]);
      store_map_cluster<V>(cluster_addr(&K.block[parity][turn][p.lane], (uint32_t)p.warp), all);
    }
    cluster_sync_all();
    for (int r = 0; r < p.ranks; ++r) {
      if (r == turn)
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = x[v];
      apply<V>(K.block[parity][r][p.lane], x);
    }
  }
  for (int w = 0; w < order; ++w) apply<V>(maps[w][p.lane], s);
}
// The state after the step, for the next one (no cluster): the group's last
// warp along the walk has it.
template <int V, bool REVERSE>
__device__ __forceinline__ void leave(Walk<V>& K, const Place& p, int parity, const float (&s)[V]) {
  if (p.ranks == 1 && (REVERSE ? p.warp == 0 : p.warp == p.warps - 1))
#pragma unroll
    for (int v = 0; v < V; ++v) K.state[parity ^ 1][p.first][p.lane][v] = s[v];
}

// P rows of V elements from `x`, the first `live` of them; the others as `fill`
template <int P, typename T_, int V>
__device__ __forceinline__ void load_rows(Pack<T_, V> (&to)[P], const T_* x, long long row, int live, float fill) {
#pragma unroll
  for (int p = 0; p < P; ++p) {
    if (p < live) {
      to[p] = *reinterpret_cast<const Pack<T_, V>*>(x + p * row);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) to[p].v[v] = from_f32<T_>(fill);
    }
  }
}

// Positions that are not a chunk's get a gate logit of -inf: a = 1 and z = 0
// exactly, which leaves the state alone.
// ------------------------------------------------------------------ forward
template <typename T_, int V>
__global__ void __launch_bounds__(kMaxWarps * 32, V == 1 ? 2 : 1)
mingru_scan_kernel(const T_* __restrict__ zh, RowStrides zs, int T, int d, FastDiv by_d, long long chains, int warps,
                   int ranks, const int* __restrict__ lengths, const float* h0, T_* __restrict__ h, RowStrides hs,
                   float* h_last, float* __restrict__ states) {
  constexpr int P = kScanSteps;
  __shared__ Walk<V> K;
  if (ranks > 1) cluster_sync_all();  // the others' shared memory is there from here on
  const Place at = place_of<V>(warps, ranks, chains, d, by_d);
  int len = at.in ? T : 0;
  if (at.in && lengths) len = min(max(lengths[at.b], 0), T);
  const int step = ranks * warps * P;  // positions of a step of the walk
  long long t = (long long)(at.rank * warps + at.warp) * P;
  const T_* x = zh + at.b * zs.chunk + t * zs.row + at.c;
  T_* o = h + at.b * hs.chunk + t * hs.row + at.c;
  Pack<T_, V> zl[P], hr[P];
  auto count = [&](int end, long long from) { return (int)max(min((long long)P, end - from), 0ll); };
  int live = count(len, t);
  load_rows(zl, x, zs.row, live, -INFINITY);
  load_rows(hr, x + d, zs.row, live, 0.f);
  float s[V], walk[V];
#pragma unroll
  for (int v = 0; v < V; ++v) walk[v] = at.in && h0 ? h0[at.chain + v] : 0.f;
  const int steps = (T + step - 1) / step;
  for (int i = 0; i < steps; ++i) {
    float ga[P][V], gb[P][V];
    Map<V> m = identity_map<V>();
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Cell k = mingru_cell(to_f32(zl[p].v[v]), to_f32(hr[p].v[v]));
        ga[p][v] = k.a;
        gb[p][v] = k.z * k.c;
        m.B[v] = __fmaf_rn(k.a, m.B[v], gb[p][v]);
        m.A[v] *= k.a;
      }
    const int rows = at.in ? count(T, t) : 0, was = live;
    if (i + 1 < steps) {
      x += step * zs.row;
      live = count(len, t + step);
      load_rows(zl, x, zs.row, live, -INFINITY);
      load_rows(hr, x + d, zs.row, live, 0.f);
    }
    exchange<V, false>(K, at, i & 1, m, walk, s, i == 0);
    if (states && rows > 0 && t % kSpan == 0)
#pragma unroll
      for (int v = 0; v < V; ++v) states[t / kSpan * chains + at.chain + v] = s[v];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      Pack<T_, V> y;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s[v] = __fmaf_rn(ga[p][v], s[v], gb[p][v]);
        y.v[v] = from_f32<T_>(p < was ? s[v] : 0.f);
      }
      if (p < rows) *reinterpret_cast<Pack<T_, V>*>(o + p * hs.row) = y;
    }
    if (i + 1 < steps) leave<V, false>(K, at, i & 1, s);
    t += step;
    o += step * hs.row;
  }
  // the state after the last position: the walk's last warp has applied all
  if (h_last && at.in && at.rank == ranks - 1 && at.warp == warps - 1)
#pragma unroll
    for (int v = 0; v < V; ++v) h_last[at.chain + v] = s[v];
}

// ----------------------------------------------------------------- backward
template <typename T_, int V>
__global__ void __launch_bounds__(kMaxWarps * 32, V == 1 ? 2 : 1)
mingru_grad_kernel(const T_* __restrict__ zh, RowStrides zs, int T, int d, FastDiv by_d, long long chains, int warps,
                   int ranks, const int* __restrict__ lengths, const float* __restrict__ states,
                   const T_* __restrict__ dh, RowStrides dhs, const float* dh_last, T_* __restrict__ dzh,
                   RowStrides dzs, float* dh0) {
  constexpr int P = kGradSteps;
  __shared__ Walk<V> K;
  __shared__ Map<V> forward[2][kMaxWarps][32];  // the warps' maps of the state
  if (ranks > 1) cluster_sync_all();  // the others' shared memory is there from here on
  const Place at = place_of<V>(warps, ranks, chains, d, by_d);
  int len = at.in ? T : 0;
  if (at.in && lengths) len = min(max(lengths[at.b], 0), T);
  const int step = ranks * warps * P;
  const int steps = (T + step - 1) / step;
  long long t = (long long)(steps - 1) * step + (at.rank * warps + at.warp) * P;
  // the saved state that this warp's positions follow, and the warps between
  const int since = min(warps, kSpan / P), lead = at.warp % since;
  const T_* x = zh + at.b * zs.chunk + t * zs.row + at.c;
  const T_* u = dh + at.b * dhs.chunk + t * dhs.row + at.c;
  T_* o = dzh + at.b * dzs.chunk + t * dzs.row + at.c;
  Pack<T_, V> zl[P], hr[P], du[P];
  float saved[V];
  auto count = [&](int end, long long from) { return (int)max(min((long long)P, end - from), 0ll); };
  auto load_all = [&](int n) {
    load_rows(zl, x, zs.row, n, -INFINITY);
    load_rows(hr, x + d, zs.row, n, 0.f);
    load_rows(du, u, dhs.row, n, 0.f);
    const long long k = t / kSpan;
#pragma unroll
    for (int v = 0; v < V; ++v) saved[v] = n > 0 ? states[k * chains + at.chain + v] : 0.f;
  };
  int live = count(len, t);
  load_all(live);
  float s[V], g[V], walk[V];
#pragma unroll
  for (int v = 0; v < V; ++v) walk[v] = at.in && dh_last ? dh_last[at.chain + v] : 0.f;
  for (int i = 0; i < steps; ++i) {
    // c carries its branch in its sign: c >= 0, and a negative hr makes it -c
    float ga[P][V], gz[P][V], gc[P][V], gu[P][V];
    Map<V> m = identity_map<V>(), r = identity_map<V>();
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float raw = to_f32(hr[p].v[v]);
        const Cell k = mingru_cell(to_f32(zl[p].v[v]), raw);
        ga[p][v] = k.a;
        gz[p][v] = k.z;
        gc[p][v] = copysignf(k.c, raw);
        gu[p][v] = to_f32(du[p].v[v]);
        m.B[v] = __fmaf_rn(k.a, m.B[v], k.z * k.c);
        m.A[v] *= k.a;
      }
#pragma unroll
    for (int p = P - 1; p >= 0; --p)
#pragma unroll
      for (int v = 0; v < V; ++v) r.B[v] = ga[p][v] * (r.B[v] + gu[p][v]);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      r.A[v] = m.A[v];
      s[v] = saved[v];
    }
    const int rows = at.in ? count(T, t) : 0, was = live;
    if (i + 1 < steps) {
      x -= step * zs.row;
      u -= step * dhs.row;
      t -= step;
      live = count(len, t);
      load_all(live);
    }
    forward[i & 1][at.first + at.warp][at.lane] = m;
    exchange<V, true>(K, at, i & 1, r, walk, g, i == 0);
    for (int w = at.warp - lead; w < at.warp; ++w) apply<V>(forward[i & 1][at.first + w][at.lane], s);
    float before[P][V];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        before[p][v] = s[v];
        s[v] = __fmaf_rn(ga[p][v], s[v], gz[p][v] * fabsf(gc[p][v]));
      }
#pragma unroll
    for (int p = P - 1; p >= 0; --p) {
      Pack<T_, V> yz, yr;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float k = fabsf(gc[p][v]);
        g[v] += gu[p][v];
        const float z = g[v] * gz[p][v];
        const float dz = z * ga[p][v] * (k - before[p][v]);
        const float dr = signbit(gc[p][v]) ? z * (k - k * k) : z;
        g[v] *= ga[p][v];
        yz.v[v] = from_f32<T_>(p < was ? dz : 0.f);
        yr.v[v] = from_f32<T_>(p < was ? dr : 0.f);
      }
      if (p < rows) {
        *reinterpret_cast<Pack<T_, V>*>(o + p * dzs.row) = yz;
        *reinterpret_cast<Pack<T_, V>*>(o + p * dzs.row + d) = yr;
      }
    }
    if (i + 1 < steps) leave<V, true>(K, at, i & 1, g);
    o -= step * dzs.row;
  }
  if (dh0 && at.in && at.rank == 0 && at.warp == 0)
#pragma unroll
    for (int v = 0; v < V; ++v) dh0[at.chain + v] = g[v];
}

// ------------------------------------------------------------- few positions
// Up to kScanSteps positions (the decode step): a thread takes V chains through
// all of them, all loads issued first.
template <typename T_, int V, int STEPS>
__global__ void __launch_bounds__(256)
mingru_step_kernel(const T_* __restrict__ zh, RowStrides zs, int T, int d, FastDiv by_d, long long chains,
                   const int* __restrict__ lengths, const float* h0, T_* __restrict__ h, RowStrides hs,
                   float* h_last, float* __restrict__ states) {
  const long long chain = ((long long)blockIdx.x * 256 + threadIdx.x) * V;
  if (chain >= chains) return;
  const int b = (int)div_by((uint32_t)chain, by_d), c = (int)(chain - (long long)b * d);
  const int len = lengths ? min(max(lengths[b], 0), T) : T;
  Pack<T_, V> zl[STEPS], hr[STEPS];
  const T_* x = zh + b * zs.chunk + c;
#pragma unroll
  for (int p = 0; p < STEPS; ++p)
    if (p < len) {
      zl[p] = *reinterpret_cast<const Pack<T_, V>*>(x + p * zs.row);
      hr[p] = *reinterpret_cast<const Pack<T_, V>*>(x + p * zs.row + d);
    }
  float s[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s[v] = h0 ? h0[chain + v] : 0.f;
    if (states && T > 0) states[chain + v] = s[v];
  }
  T_* o = h + b * hs.chunk + c;
#pragma unroll
  for (int p = 0; p < STEPS; ++p) {
    if (p >= T) break;
    Pack<T_, V> y;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      y.v[v] = from_f32<T_>(0.f);
      if (p < len) {
        const Cell k = mingru_cell(to_f32(zl[p].v[v]), to_f32(hr[p].v[v]));
        s[v] = k.a * s[v] + k.z * k.c;
        y.v[v] = from_f32<T_>(s[v]);
      }
    }
    *reinterpret_cast<Pack<T_, V>*>(o + p * hs.row) = y;
  }
  if (h_last)
#pragma unroll
    for (int v = 0; v < V; ++v) h_last[chain + v] = s[v];
}

// ------------------------------------------------------------------ launches
// Two chains per lane where every row lets pairs be moved whole.
static bool pairs_ok(int d, int type, std::initializer_list<std::pair<const void*, RowStrides>> rows) {
  if (d % 2) return false;
  for (const auto& r : rows)
    if (r.second.row % 2 || r.second.chunk % 2 || !aligned_to(r.first, 2 * type_bytes(type))) return false;
  return true;
}

// The shape of a walk over `groups` groups of T positions, P to a warp.
struct Shape {
  int warps, ranks;     // warps of a group in a block, blocks of a group
  unsigned blocks, threads;
};
static Shape shape_of(long long groups, int T, int P) {
  Shape s{1, 1, 0, 0};
  const int block_warps = groups < 300 ? kMaxWarps : kMaxWarps / 2;
  while (s.warps < block_warps && (long long)s.warps * P < T) s.warps *= 2;
  const int per = (long long)s.warps * P >= T ? block_warps / s.warps : 1;  // groups of a block
  while (s.ranks < kMaxCluster && groups * s.ranks * 2 <= 148 && (long long)s.ranks * s.warps * P < T) s.ranks *= 2;
  s.blocks = (unsigned)((groups + per - 1) / per * s.ranks);
  s.threads = (unsigned)(s.warps * per * 32);
  return s;
}
template <typename K, typename... A>
static cudaError_t launch_walk(K kernel, const Shape& s, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(s.blocks);
  cfg.blockDim = dim3(s.threads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)s.ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = s.ranks > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_mingru_scan(const void* zh, int type, RowStrides zs, int B, int T, int d, const int* lengths,
                               const float* h0, void* h, RowStrides hs, float* h_last, float* states,
                               cudaStream_t st) {
  const long long chains = (long long)B * d;
  const FastDiv by_d = fast_div((uint32_t)d);
  const bool pairs = pairs_ok(d, type, {{zh, zs}, {h, hs}});
  return with_type(type, [&](auto t) {
    using E = decltype(t);
    const E* x = static_cast<const E*>(zh);
    E* o = static_cast<E*>(h);
    auto go = [&](auto vec) -> cudaError_t {
      constexpr int V = decltype(vec)::value;
      if (T <= kScanSteps) {
        const unsigned blocks = (unsigned)((chains + 256 * V - 1) / (256 * V));
        if (T <= 1)
          mingru_step_kernel<E, V, 1><<<blocks, 256, 0, st>>>(x, zs, T, d, by_d, chains, lengths, h0, o, hs, h_last,
                                                              states);
        else
          mingru_step_kernel<E, V, kScanSteps><<<blocks, 256, 0, st>>>(x, zs, T, d, by_d, chains, lengths, h0, o, hs,
                                                                       h_last, states);
        return cudaGetLastError();
      }
      const Shape s = shape_of((chains + 32 * V - 1) / (32 * V), T, kScanSteps);
      return launch_walk(mingru_scan_kernel<E, V>, s, st, x, zs, T, d, by_d, chains, s.warps, s.ranks, lengths, h0, o,
                         hs, h_last, states);
    };
    return pairs && (sizeof(E) == 2 || T <= kScanSteps) ? go(std::integral_constant<int, 2>{})
                                                        : go(std::integral_constant<int, 1>{});
  });
}

cudaError_t launch_mingru_scan_grad(const void* zh, int type, RowStrides zs, int B, int T, int d, const int* lengths,
                                    const float* states, const void* dh, RowStrides dhs, const float* dh_last,
                                    void* dzh, RowStrides dzs, float* dh0, cudaStream_t st) {
  const long long chains = (long long)B * d;
  if (T == 0) {  // the state's gradient passes through
    if (!dh0 || dh0 == dh_last) return cudaSuccess;
    return dh_last ? cudaMemcpyAsync(dh0, dh_last, (size_t)chains * 4, cudaMemcpyDeviceToDevice, st)
                   : cudaMemsetAsync(dh0, 0, (size_t)chains * 4, st);
  }
  const FastDiv by_d = fast_div((uint32_t)d);
  const bool pairs = pairs_ok(d, type, {{zh, zs}, {dh, dhs}, {dzh, dzs}});
  return with_type(type, [&](auto t) {
    using E = decltype(t);
    auto go = [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      const Shape s = shape_of((chains + 32 * V - 1) / (32 * V), T, kGradSteps);
      return launch_walk(mingru_grad_kernel<E, V>, s, st, static_cast<const E*>(zh), zs, T, d, by_d, chains, s.warps,
                         s.ranks, lengths, states, static_cast<const E*>(dh), dhs, dh_last, static_cast<E*>(dzh), dzs,
                         dh0);
    };
    return pairs && sizeof(E) == 2 ? go(std::integral_constant<int, 2>{}) : go(std::integral_constant<int, 1>{});
  });
}

}  // namespace boa
