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
// G * V chains (a chain is one channel of one chunk) and is taken along the
// time axis by one block, or by a cluster of up to kMaxCluster blocks when
// there are too few groups to fill the GPU.  A team of G lanes (a warp, or half
// of one where groups are few) has V chains a lane.  In a step of the walk every
// team holds P positions of every chain in registers, forms their (A, B), and
// issues the loads of its next step; the teams' maps meet in shared memory,
// the blocks' in each other's (pushed there, double-buffered, one barrier a
// step); the state that enters a team's positions is the walk's state with the
// maps before it applied in order, and the outputs come from the registers.
// So the gates are read once, nothing waits on another block outside its
// cluster, and the result does not depend on timing.
//
// Measured on a B200 (floor: the bytes at the 6561 GB/s of a copy).  Many 32-bit
// chains run at the memory's rate: 256 x 1024 x 256 forward 142 us (0.87),
// backward 245 us (0.84).  16-bit rows are paced by instruction issue, 30 a value
// forward and 56 backward: 64 x 4096 x 256 bf16 105 us (0.58) and 171 us (0.60);
// their 256 blocks also leave 40 of the SMs with one instead of two.
// Few chains are paced by the SMs that clusters reach: 1 x 262144 x 512 fp32
// 383 us (0.64) and 680 us (0.60).  One position, 16384 x 256: 13.5 to 14.4 us
// in four captures (0.95 to 0.89); 8 positions 68 us (0.98).  Backward one to
// eight positions take the walk too: 162 and 178 us (0.11, 0.60).
#include "ptx.cuh"
#include "train_ops.cuh"

namespace boa {

constexpr int kSpan = 32;         // positions between two saved states
constexpr int kMaxCluster = 8;    // blocks of a cluster (the portable limit)
constexpr int kFew = 8;           // up to here, one thread takes a chain through all positions
// Positions that a warp holds, and registers a thread, for V chains a lane.
// Long runs spread the exchange and the walk's bookkeeping over more
// positions, which is what paces 16-bit rows and few chains (32 x 4096 x 256
// bf16 forward: 8 positions at 80 registers 69 us, 16 at 128 60 us).  With many
// 32-bit chains there are bytes enough to wait for, and more warps win
// (256 x 1024 x 256 forward: 4 positions at 64 registers 146 us, 8 at 80
// 169 us).  Backward a position holds twice the values (8 at 128: 95 us, 4 at
// 80: 134 us).
template <typename T_, int V>
constexpr int scan_steps() { return V == 2 && sizeof(T_) == 4 ? 4 : 16; }
template <typename T_, int V>
constexpr int scan_regs() { return V == 1 ? 96 : sizeof(T_) == 4 ? 64 : 128; }
constexpr int kGradSteps = 8;
template <int V>
constexpr int grad_regs() { return V == 1 ? 96 : 128; }
// Warps of a block that has an SM to itself (as many as those registers let
// in); of the blocks that share one, half of 16.
template <int V>
constexpr int alone_warps() { return V == 1 ? 20 : 16; }
constexpr int kSharedWarps = 8;

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

// V chains of a lane.  (Packed pairs, f32x2, were measured slower: they run on
// one of the two FMA pipes only, and most of the arithmetic here is FMA work.)
template <int V>
struct Vec {
  float v[V];
};
template <int V>
__device__ __forceinline__ Vec<V> all_of(float x) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = x;
  return r;
}
template <int V>
__device__ __forceinline__ Vec<V> vfma(const Vec<V>& a, const Vec<V>& b, const Vec<V>& c) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = __fmaf_rn(a.v[i], b.v[i], c.v[i]);
  return r;
}
template <int V>
__device__ __forceinline__ Vec<V> vmul(const Vec<V>& a, const Vec<V>& b) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = __fmul_rn(a.v[i], b.v[i]);
  return r;
}

__device__ __forceinline__ float max_or_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// The cell's gates for V chains.  One reciprocal of both denominators'
// product serves both sigmoids: three special-function operations an element
// instead of four.  With e = exp(-zl), f = exp(-|hr|), p = 1 + e, q = 1 + f and
// r = 1 / (p q):
//
//   z = q r = f r + r     sigmoid(-|hr|) = f (p r)     a = 1 - z
//
// zl is cut off at -88, where p q stays below 2^128 and its reciprocal is
// below 2^-126, which the instruction flushes: from there down z is 0 and
// a is 1, exactly (the candidate then has no weight).  A closed gate so keeps
// the state however many positions long.
//
// For zl >= 0 a is taken as e z: 1 - z would leave few of its digits, and none
// from zl = 17 on, and the gate's gradient is proportional to it.  Below 0
// the difference has all digits, and e z would not be 1 for a closed gate.
template <int V>
struct Cell {
  Vec<V> a, b;  // 1 - z, z c
  Vec<V> z, w;  // z, z c'(hr): for the gradient
};
template <int V, bool GRAD>
__device__ __forceinline__ Cell<V> mingru_cell(const Vec<V>& zl, const Vec<V>& hr) {
  Cell<V> k;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float e = ex2_fast(max_or_nan(zl.v[v], -88.f) * -kLog2e), f = ex2_fast(fabsf(hr.v[v]) * -kLog2e);
    const float p = 1.f + e;
    const float r = rcp_fast(__fmaf_rn(p, f, p));
    const float z = __fmaf_rn(f, r, r), low = f * (p * r);
    // hr + 1/2 lies below sigmoid(hr) for hr < 0 (slopes 1 and at most 1/4
    // from the same value at 0), and above sigmoid(-hr) <= 1/2 otherwise
    const float c = fmaxf(hr.v[v] + 0.5f, low);
    k.a.v[v] = zl.v[v] >= 0.f ? e * z : 1.f - z;
    k.b.v[v] = z * c;
    k.z.v[v] = z;
    if (GRAD) k.w.v[v] = z * (hr.v[v] >= 0.f ? 1.f : __fmaf_rn(-low, low, low));
  }
  return k;
}

static long long spans_of(int T) { return ((long long)T + kSpan - 1) / kSpan; }
size_t mingru_states_floats(int B, int T, int d) { return (size_t)spans_of(T) * B * d; }

// The map of a run of positions for V chains: x -> A x + B.
template <int V>
struct alignas(8 * V) Map {
  Vec<V> A, B;
};
template <int V>
__device__ __forceinline__ Vec<V> apply(const Map<V>& m, const Vec<V>& x) { return vfma(m.A, x, m.B); }
// m, then n
template <int V>
__device__ __forceinline__ Map<V> then(const Map<V>& m, const Map<V>& n) {
  return {vmul(m.A, n.A), vfma(n.A, m.B, n.B)};
}

// Shared memory of a walk, for a block of `teams` teams.  Everything is
// double-buffered by the step's parity: what a step writes was last read two
// steps ago, and every warp passes one barrier in between.
template <int V, int G>
struct Walk {
  Map<V>* maps;     // [2][teams][G]: the teams' maps
  Map<V>* forward;  // [2][teams][G]: backward, their maps of the state
  Map<V>* block;    // [2][ranks][G]: the cluster's blocks' maps, pushed by their owners (ranks > 1)
  Vec<V>* state;    // [2][G]: the walk's state, left by the last team (ranks = 1)
  uint64_t* full;   // [2]: barriers that count the bytes pushed into `block` (ranks > 1)
  uint8_t* stages;
  int teams, ranks;
  uint64_t limit_ns;  // of a wait
  __device__ __forceinline__ Walk(uint8_t* at, int ranks_, bool both, uint64_t limit_ns_ = kWaitLimitNs)
      : teams(blockDim.x / G), ranks(ranks_), limit_ns(limit_ns_) {
    maps = reinterpret_cast<Map<V>*>(at);
    forward = maps + 2 * G * teams;
    block = forward + (both ? 2 * G * teams : 0);
    state = reinterpret_cast<Vec<V>*>(block + (ranks > 1 ? 2 * G * ranks : 0));
    full = reinterpret_cast<uint64_t*>(state + 2 * G);
    stages = reinterpret_cast<uint8_t*>(full + 2);
  }
  static size_t bytes(int threads, int ranks, bool both) {
    return sizeof(Map<V>) * 2 * ((both ? 2 : 1) * threads + (ranks > 1 ? ranks * G : 0)) + sizeof(Vec<V>) * 2 * G + 16;
  }
  // Called by all threads before anything else; afterwards the cluster's
  // blocks have started and their barriers are ready.
  __device__ __forceinline__ void start() const {
    if (ranks == 1) return;
    if (threadIdx.x == 0) {
      mbar_init(full, 1);
      mbar_init(full + 1, 1);
      fence_mbar_init();
    }
    __syncwarp();  // the barrier is for whole warps
    cluster_sync_all();
  }
  // No block leaves before the others' last pushes have gone out.  One that
  // has stopped waiting did not see them arrive, and stays a little longer.
  __device__ __forceinline__ void finish(bool waiting) const {
    if (ranks == 1) return;
    __syncwarp();
    cluster_sync_all();
    if (!waiting)
      for (const uint64_t t0 = global_ns(); global_ns() - t0 < 100000;) {
      }
  }
};

// Where a team works.  A block serves one group of chains with all its teams,
// or several groups with `teams` teams each when a group's whole sequence fits
// them.
struct Place {
  long long chain;
  bool in;
  int b, c, lane, team, teams, first;  // lane within the team, team within its group, the group's first team
  int rank, ranks;                     // block within its cluster
};
template <int V, int G>
__device__ __forceinline__ Place place_of(int teams, int ranks, long long chains, int d, FastDiv by_d) {
  Place p;
  p.lane = threadIdx.x % G;
  const int w = threadIdx.x / G, per = (int)(blockDim.x / G) / teams;
  p.teams = teams;
  p.team = w % teams;
  p.first = w - p.team;
  p.ranks = ranks;
  p.rank = ranks > 1 ? (int)cluster_rank() : 0;
  const long long group = (long long)(blockIdx.x / ranks) * per + w / teams;
  p.chain = group * (G * V) + p.lane * V;
  p.in = p.chain < chains;
  p.b = p.in ? (int)div_by((uint32_t)p.chain, by_d) : 0;
  p.c = p.in ? (int)(p.chain - (long long)p.b * d) : 0;
  return p;
}

// Writes a map into another block's shared memory; its bytes are counted on
// that block's barrier.  The barrier, and not a release by this block, says
// that the map is there: a release would also wait for the block's stores to
// HBM, a full memory latency in every step.
template <int V>
__device__ __forceinline__ void push_map(uint32_t addr, const Map<V>& m, uint32_t bar) {
  if constexpr (V == 1)
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(addr),
                 "f"(m.A.v[0]), "f"(m.B.v[0]), "r"(bar)
                 : "memory");
  else
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::
                     "r"(addr), "f"(m.A.v[0]), "f"(m.A.v[V - 1]), "f"(m.B.v[0]), "f"(m.B.v[V - 1]), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for a phase.  When the wait runs out `waiting` is cleared: this
// thread's state becomes NaN, and with it all that it writes from there on (a
// handle-free call has no error word to set).  It neither waits nor pushes
// again: a slot that it filled without waiting could still be in use, and
// would give another block a wrong map.  The others miss its maps and run
// out in the next step, so every value written is right or NaN.
__device__ __forceinline__ void await_maps(uint32_t bar, uint32_t parity, uint64_t limit_ns, bool& waiting) {
  if (waiting && !try_wait_cluster(bar, parity)) {
    const uint64_t t0 = global_ns();
    while (waiting && !try_wait_cluster(bar, parity)) waiting = global_ns() - t0 <= limit_ns;
  }
  __syncwarp();  // lanes may leave the loop apart
}

// One step's exchange.  `mine`: the map of this team's positions, `x`: the
// walk's state before the step.  Returns the state before this team's
// positions; in a cluster x becomes the state after the step.  REVERSE runs
// from the last team and block to the first.  Without a cluster the state
// after the step is handed on through leave().
//
// In a cluster, a slot of `block` is written again two steps on.  Its writer
// has then seen this block's map of the step between, which goes out after
// the barrier below, that is after all teams here have read the slot.
template <int V, int G, bool REVERSE>
__device__ __forceinline__ Vec<V> exchange(const Walk<V, G>& K, const Place& p, int step, const Map<V>& mine,
                                           Vec<V>& x, bool& waiting) {
  const int parity = step & 1;
  const int order = REVERSE ? p.teams - 1 - p.team : p.team;  // place of this team along the walk
  Map<V>* maps = K.maps + (parity * K.teams + p.first) * G + p.lane;
  maps[order * G] = mine;
  __syncthreads();
  Vec<V> s;
  if (p.ranks == 1) {
    s = step == 0 ? x : K.state[parity * G + p.lane];
  } else {
    if (threadIdx.x == 0 && waiting) mbar_arrive_expect_tx(K.full + parity, (uint32_t)(p.ranks * G * sizeof(Map<V>)));
    const int turn = REVERSE ? p.ranks - 1 - p.rank : p.rank;
    if (p.team < p.ranks && waiting) {  // team r takes the block's map to block r
      Map<V> all = maps[0];
#pragma unroll 4
      for (int w = 1; w < p.teams; ++w) all = then<V>(all, maps[w * G]);
      push_map<V>(cluster_addr(K.block + (parity * p.ranks + turn) * G + p.lane, (uint32_t)p.team), all,
                  cluster_addr(K.full + parity, (uint32_t)p.team));
    }
    await_maps(smem_u32(K.full + parity), (uint32_t)(step >> 1) & 1u, K.limit_ns, waiting);
    if (!waiting) x = all_of<V>(__int_as_float(0x7fffffff));
    for (int r = 0; r < p.ranks; ++r) {
      if (r == turn) s = x;
      x = apply<V>(K.block[(parity * p.ranks + r) * G + p.lane], x);
    }
  }
#pragma unroll 4
  for (int w = 0; w < order; ++w) s = apply<V>(maps[w * G], s);
  return s;
}
// The state after the step, for the next one (no cluster): the group's last
// team along the walk has it.
template <int V, int G, bool REVERSE>
__device__ __forceinline__ void leave(const Walk<V, G>& K, const Place& p, int parity, const Vec<V>& s) {
  if (p.ranks == 1 && (REVERSE ? p.team == 0 : p.team == p.teams - 1)) K.state[(parity ^ 1) * G + p.lane] = s;
}

// Rows on their way from HBM to a team's stage, [row][G lanes] packs a
// stream.  QUADS: 16 bytes a lane, several rows an instruction, where every
// row lets them be moved whole (a lane then brings packs that other lanes of
// its team use).  Otherwise every lane brings its own packs; one of 2 bytes
// (odd widths) is too small for an asynchronous copy and is moved by a load
// and a store.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T_, int V>
__device__ __forceinline__ Vec<V> widen(const Pack<T_, V>& p) {
  Vec<V> r;
  widen_pack(p, r.v);
  return r;
}
// a row that is not there as `fill`
template <typename T_, int V>
__device__ __forceinline__ Vec<V> widen(const Pack<T_, V>& p, bool there, float fill) {
  Vec<V> r = widen(p);
#pragma unroll
  for (int v = 0; v < V; ++v) r.v[v] = there ? r.v[v] : fill;
  return r;
}
template <typename T_, int V>
__device__ __forceinline__ void store_rounded(T_* to, const Vec<V>& x) {
  *reinterpret_cast<Pack<T_, V>*>(to) = narrow_pack<T_>(x.v);
}

// A team's stages, [stage][stream][P][G].  Half-warp teams lie half the banks
// apart, so that the two of a warp read without conflicts.
template <int G>
__host__ __device__ constexpr int packs_of_team(int stages, int streams, int P) {
  return stages * streams * P * G + (G == 32 ? 0 : G);
}
template <typename T_, int V, int G, int P, int STREAMS>
__device__ __forceinline__ Pack<T_, V>* team_stages(uint8_t* stages, int S) {
  return reinterpret_cast<Pack<T_, V>*>(stages) + (threadIdx.x / G) * packs_of_team<G>(S, STREAMS, P);
}
// row p after `x`, `row` bytes each: one multiply-add of 32 bits to 64
template <typename P_>
__device__ __forceinline__ P_* row_at(P_* x, uint32_t row, int p) {
  using B_ = typename std::conditional<std::is_const<P_>::value, const char, char>::type;
  return reinterpret_cast<P_*>(reinterpret_cast<B_*>(x) + (unsigned long long)row * (uint32_t)p);
}
// Which part of a team's rows a lane brings: elements `c` on of chunk `b`, of
// rows first, first + EVERY, ...; `at` bytes into the stage.
template <typename T_, int V, int G, bool QUADS>
struct Carrier {
  static constexpr int kBytes = QUADS ? 16 : (int)sizeof(T_) * V;
  static constexpr int kRow = G * (int)sizeof(T_) * V;       // bytes of a row in the stage
  static constexpr int kEvery = G * kBytes / kRow;           // rows of an instruction
  int b, c, first, len;
  uint32_t at;
  __device__ __forceinline__ Carrier(const Place& p, int T, int d, FastDiv by_d, long long chains, const int* lengths) {
    const int piece = p.lane % (G / kEvery);
    first = p.lane / (G / kEvery);
    at = (uint32_t)(p.lane * kBytes);
    const long long chain = p.chain - p.lane * V + piece * (kBytes / (int)sizeof(T_));
    const bool in = chain < chains;
    b = in ? (int)div_by((uint32_t)chain, by_d) : 0;
    c = in ? (int)(chain - (long long)b * d) : 0;
    len = in ? T : 0;
    if (in && lengths) len = min(max(lengths[b], 0), T);
  }
  // the rows of [t, t + P) that are there (`whole`: all); x is at row t + first
  template <int P>
  __device__ __forceinline__ void copy(Pack<T_, V>* stage, const T_* x, uint32_t row, int t, bool whole) const {
    const uint32_t to = smem_u32(stage) + at;
    if constexpr (kBytes == 2) {  // all loads, then all stores
      unsigned short v[P];
#pragma unroll
      for (int k = 0; k < P; ++k)
        v[k] = whole || t + k < len ? __ldg(reinterpret_cast<const unsigned short*>(row_at(x, row, k))) : 0;
#pragma unroll
      for (int k = 0; k < P; ++k) asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + k * kRow), "h"(v[k]) : "memory");
    } else if (whole) {
#pragma unroll
      for (int k = 0; k < P / kEvery; ++k) copy_async<kBytes>(to + k * kEvery * kRow, row_at(x, row, k * kEvery));
    } else {
#pragma unroll
      for (int k = 0; k < P / kEvery; ++k)
        if (t + first + k * kEvery < len)
          copy_async<kBytes>(to + k * kEvery * kRow, row_at(x, row, k * kEvery));
    }
  }
};
// rows of [from, from + P) before `end`
template <int P>
__device__ __forceinline__ int rows_left(int from, int end) { return max(min(P, end - from), 0); }

constexpr int kStages = 2;  // the step in use, and the next one on its way

// Positions that are not a chunk's get a gate logit of -inf: a = 1 and b = 0
// exactly, which leaves the state alone.  (p r = 0 there, and so is f (p r).)
// A warp whose rows are all there (`whole`, the same for its lanes: `later` is
// how much later its last team's positions begin) takes a form without those
// tests.
// ------------------------------------------------------------------ forward
template <typename T_, int V, int G, bool QUADS>
__global__ void __maxnreg__((scan_regs<T_, V>()))
mingru_scan_kernel(const T_* __restrict__ zh, RowStrides zs, int T, int d, FastDiv by_d, long long chains,
                   const int* __restrict__ lengths, const float* h0, T_* __restrict__ h, RowStrides hs,
                   float* h_last, float* __restrict__ states, int teams, int ranks) {
  constexpr int P = scan_steps<T_, V>(), S = kStages, STAGE = 2 * P * G;
  extern __shared__ __align__(16) uint8_t walk_smem[];
  const Walk<V, G> K(walk_smem, ranks, false);
  K.start();
  const Place at = place_of<V, G>(teams, ranks, chains, d, by_d);
  int len = at.in ? T : 0;
  if (at.in && lengths) len = min(max(lengths[at.b], 0), T);
  const int end = at.in ? T : 0;
  const int all_len = __reduce_min_sync(~0u, len);  // positions that all of the warp's chains have
  const int later = P * ((32 / G - 1) - at.team % (32 / G));
  const int step = ranks * teams * P;  // positions of a step of the walk
  int t = (at.rank * teams + at.team) * P;
  const Carrier<T_, V, G, QUADS> by(at, T, d, by_d, chains, lengths);
  const T_* x = zh + by.b * zs.chunk + (t + by.first) * zs.row + by.c;
  T_* o = h + at.b * hs.chunk + t * hs.row + at.c;
  Pack<T_, V>* const stages = team_stages<T_, V, G, P, 2>(K.stages, S);
  const long long x_step = step * zs.row, o_step = step * hs.row;
  const uint32_t x_row = (uint32_t)(zs.row * sizeof(T_)), o_row = (uint32_t)(hs.row * sizeof(T_));
  const int steps = (T + step - 1) / step;
  int t_next = t, put = 0, got = 0;  // the next step to fetch, its stage, and the stage in use
  auto fetch = [&](bool more) {
    if (more) {
      const bool whole = t_next + later + P <= all_len;
      by.template copy<P>(stages + put * STAGE, x, x_row, t_next, whole);
      by.template copy<P>(stages + put * STAGE + P * G, x + d, x_row, t_next, whole);
      x += x_step;
      t_next += step;
      put = put + 1 == S ? 0 : put + 1;
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch(i < steps);
  Vec<V> walk = all_of<V>(0.f), s = walk;
  bool waiting = true;
  if (at.in && h0)
#pragma unroll
    for (int v = 0; v < V; ++v) walk.v[v] = h0[at.chain + v];
  for (int i = 0; i < steps; ++i) {
    copies_wait<S - 2>();
    __syncwarp();  // the other lanes' copies too
    const Pack<T_, V>*zl = stages + got * STAGE + at.lane, *hr = zl + P * G;
    got = got + 1 == S ? 0 : got + 1;
    const int live = rows_left<P>(t, len), rows = rows_left<P>(t, end);
    const bool whole = t + later + P <= all_len;
    Vec<V> ga[P], gb[P];
    Map<V> m;
    auto gates = [&](auto all) {
      constexpr bool ALL = decltype(all)::value;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const bool there = ALL || p < live;
        const Cell<V> k = mingru_cell<V, false>(widen(zl[p * G], there, -INFINITY),
                                                widen(hr[p * G], there, 0.f));
        ga[p] = k.a;
        gb[p] = k.b;
        m = p ? then<V>(m, {k.a, k.b}) : Map<V>{k.a, k.b};
      }
    };
    if (whole) gates(std::true_type{});
    else gates(std::false_type{});
    fetch(i + S - 1 < steps);
    s = exchange<V, G, false>(K, at, i, m, walk, waiting);
    if (states && rows > 0 && t % kSpan == 0)
#pragma unroll
      for (int v = 0; v < V; ++v) states[t / kSpan * chains + at.chain + v] = s.v[v];
    auto finish = [&](auto all) {
      constexpr bool ALL = decltype(all)::value;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        s = vfma(ga[p], s, gb[p]);
        if (ALL || p < rows)
          store_rounded<T_, V>(row_at(o, o_row, p), ALL || p < live ? s : all_of<V>(0.f));
      }
    };
    if (whole) finish(std::true_type{});
    else finish(std::false_type{});
    if (i + 1 < steps) leave<V, G, false>(K, at, i & 1, s);
    t += step;
    o += o_step;
  }
  // The state after the last position: the walk's last team has applied all.
  // h_last may be h0: a push orders nothing before it, so only the cluster's
  // last barrier says that the other blocks have read h0.
  K.finish(waiting);
  if (h_last && at.in && at.rank == ranks - 1 && at.team == teams - 1)
#pragma unroll
    for (int v = 0; v < V; ++v) h_last[at.chain + v] = s.v[v];
}

// ----------------------------------------------------------------- backward
template <typename T_, int V, int G, bool QUADS>
__global__ void __maxnreg__(grad_regs<V>())
mingru_grad_kernel(const T_* __restrict__ zh, RowStrides zs, int T, int d, FastDiv by_d, long long chains,
                   const int* __restrict__ lengths, const float* __restrict__ states, const T_* __restrict__ dh,
                   RowStrides dhs, const float* dh_last, T_* __restrict__ dzh, RowStrides dzs, float* dh0, int teams,
                   int ranks) {
  constexpr int P = kGradSteps, S = kStages, STAGE = 3 * P * G;
  extern __shared__ __align__(16) uint8_t walk_smem[];
  const Walk<V, G> K(walk_smem, ranks, true);
  K.start();
  const Place at = place_of<V, G>(teams, ranks, chains, d, by_d);
  int len = at.in ? T : 0;
  if (at.in && lengths) len = min(max(lengths[at.b], 0), T);
  const int end = at.in ? T : 0;
  const int all_len = __reduce_min_sync(~0u, len);  // positions that all of the warp's chains have
  const int later = P * ((32 / G - 1) - at.team % (32 / G));
  const int step = ranks * teams * P;
  const int steps = (T + step - 1) / step;
  // steps are taken from the last
  int t = (steps - 1) * step + (at.rank * teams + at.team) * P;
  // the teams between the saved state and this team's positions
  const int lead = at.team % min(teams, kSpan / P);
  const Carrier<T_, V, G, QUADS> by(at, T, d, by_d, chains, lengths);
  const T_* x = zh + by.b * zs.chunk + (t + by.first) * zs.row + by.c;
  const T_* u = dh + by.b * dhs.chunk + (t + by.first) * dhs.row + by.c;
  T_* o = dzh + at.b * dzs.chunk + t * dzs.row + at.c;
  const long long x_step = step * zs.row, u_step = step * dhs.row, o_step = step * dzs.row;
  const uint32_t x_row = (uint32_t)(zs.row * sizeof(T_)), u_row = (uint32_t)(dhs.row * sizeof(T_)),
                 o_row = (uint32_t)(dzs.row * sizeof(T_));
  Vec<V> next_saved = all_of<V>(0.f);  // the saved state of the step after the current one
  Pack<T_, V>* const stages = team_stages<T_, V, G, P, 3>(K.stages, S);
  int t_next = t, put = 0, got = 0;  // the next step to fetch, its stage, and the stage in use
  auto fetch = [&](bool more) {
    if (more) {
      const bool whole = t_next + later + P <= all_len;
      by.template copy<P>(stages + put * STAGE, x, x_row, t_next, whole);
      by.template copy<P>(stages + put * STAGE + P * G, x + d, x_row, t_next, whole);
      by.template copy<P>(stages + put * STAGE + 2 * P * G, u, u_row, t_next, whole);
      x -= x_step;
      u -= u_step;
      t_next -= step;
      put = put + 1 == S ? 0 : put + 1;
    }
    copies_commit();
  };
  auto load_saved = [&](int from) {
    if (from < len)
#pragma unroll
      for (int v = 0; v < V; ++v) next_saved.v[v] = states[from / kSpan * chains + at.chain + v];
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch(i < steps);
  load_saved(t);
  Vec<V> walk = all_of<V>(0.f), g = walk;
  bool waiting = true;
  if (at.in && dh_last)
#pragma unroll
    for (int v = 0; v < V; ++v) walk.v[v] = dh_last[at.chain + v];
  for (int i = 0; i < steps; ++i) {
    copies_wait<S - 2>();
    __syncwarp();  // the other lanes' copies too, and all have read the stage that is filled next
    const Pack<T_, V>*zl = stages + got * STAGE + at.lane, *hr = zl + P * G, *du = hr + P * G;
    got = got + 1 == S ? 0 : got + 1;
    const int live = rows_left<P>(t, len), rows = rows_left<P>(t, end);
    Vec<V> s = next_saved;
    if (i + 1 < steps) load_saved(t - step);
    const bool whole = t + later + P <= all_len;
    Vec<V> ga[P], gb[P], gz[P], gw[P];
    Map<V> m, r;
    auto gates = [&](auto all) {
      constexpr bool ALL = decltype(all)::value;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const bool there = ALL || p < live;
        const Cell<V> k = mingru_cell<V, true>(widen(zl[p * G], there, -INFINITY),
                                               widen(hr[p * G], there, 0.f));
        ga[p] = k.a;
        gb[p] = k.b;
        gz[p] = k.z;
        gw[p] = k.w;
        m = p ? then<V>(m, {k.a, k.b}) : Map<V>{k.a, k.b};
      }
    };
    if (whole) gates(std::true_type{});
    else gates(std::false_type{});
    // the gradient that reaches each state: G_p = u_p + a_{p+1} G_{p+1}
    r.A = m.A;
    r.B = widen(du[(P - 1) * G], P - 1 < live, 0.f);
#pragma unroll
    for (int p = P - 2; p >= 0; --p) r.B = vfma(ga[p + 1], r.B, widen(du[p * G], p < live, 0.f));
    r.B = vmul(ga[0], r.B);
    fetch(i + S - 1 < steps);
    Map<V>* forward = K.forward + ((i & 1) * K.teams + at.first) * G + at.lane;
    forward[at.team * G] = m;
    g = exchange<V, G, true>(K, at, i, r, walk, waiting);
#pragma unroll 4
    for (int w = at.team - lead; w < at.team; ++w) s = apply<V>(forward[w * G], s);
    // dzl / G = a (z c - z h'), h' the state before
#pragma unroll
    for (int p = 0; p < P; ++p) {
      Vec<V> gap;
#pragma unroll
      for (int v = 0; v < V; ++v) gap.v[v] = __fmaf_rn(-gz[p].v[v], s.v[v], gb[p].v[v]);
      gz[p] = vmul(ga[p], gap);
      s = vfma(ga[p], s, gb[p]);
    }
    auto finish = [&](auto all) {
      constexpr bool ALL = decltype(all)::value;
#pragma unroll
      for (int p = P - 1; p >= 0; --p) {
        const bool there = ALL || p < live;
        const Vec<V> u_p = widen(du[p * G], there, 0.f);
        g = vfma(p == P - 1 ? all_of<V>(1.f) : ga[p + 1], g, u_p);
        if (ALL || p < rows) {
          T_* y = row_at(o, o_row, p);
          store_rounded<T_, V>(y, there ? vmul(g, gz[p]) : all_of<V>(0.f));
          store_rounded<T_, V>(y + d, there ? vmul(g, gw[p]) : all_of<V>(0.f));
        }
      }
      g = vmul(g, ga[0]);
    };
    if (whole) finish(std::true_type{});
    else finish(std::false_type{});
    if (i + 1 < steps) leave<V, G, true>(K, at, i & 1, g);
    t -= step;
    o -= o_step;
  }
  K.finish(waiting);  // dh0 may be dh_last, as above
  if (dh0 && at.in && at.rank == 0 && at.team == 0)
#pragma unroll
    for (int v = 0; v < V; ++v) dh0[at.chain + v] = g.v[v];
}

// A walk of a cluster of two blocks whose second stops pushing its maps at step `silent`: what the exchange
// gives each thread, [step][thread of the cluster].  Every run of positions adds 1.
__global__ void __launch_bounds__(64)
walk_selftest_kernel(int steps, int silent, FastDiv by_32, uint64_t limit_ns, float* out) {
  extern __shared__ __align__(16) uint8_t walk_smem[];
  const Walk<1, 32> K(walk_smem, 2, false, limit_ns);
  K.start();
  const Place at = place_of<1, 32>(2, 2, 32, 32, by_32);
  Vec<1> walk = all_of<1>(0.f);
  bool waiting = true;
  for (int i = 0; i < steps; ++i) {
    if (i >= silent && at.rank == 1) waiting = false;
    out[(i * 2 + at.rank) * 64 + threadIdx.x] =
        exchange<1, 32, false>(K, at, i, {all_of<1>(1.f), all_of<1>(1.f)}, walk, waiting).v[0];
  }
  K.finish(waiting);
}
cudaError_t launch_walk_selftest(int steps, int silent, uint64_t limit_ns, float* out, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2);
  cfg.blockDim = dim3(64);
  cfg.dynamicSmemBytes = Walk<1, 32>::bytes(64, 2, false);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, walk_selftest_kernel, steps, silent, fast_div(32), limit_ns, out);
}

// ------------------------------------------------------------- few positions
// Up to kFew positions (the decode step): a thread takes V chains through
// all of them, all loads issued first.
// The cell and the state's update are the same operations for every V, T_ and
// STEPS, so that any cut of a sequence into such calls gives the same bits:
// the header promises that, for an encoder and a decoder that must agree.
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
  Vec<V> s;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s.v[v] = h0 ? h0[chain + v] : 0.f;
    if (states && T > 0) states[chain + v] = s.v[v];
  }
  T_* o = h + b * hs.chunk + c;
#pragma unroll
  for (int p = 0; p < STEPS; ++p) {
    if (p >= T) break;
    Vec<V> y = all_of<V>(0.f);
    if (p < len) {
      const Cell<V> k = mingru_cell<V, false>(widen(zl[p], true, 0.f), widen(hr[p], true, 0.f));
      y = s = vfma(k.a, s, k.b);
    }
    store_rounded<T_, V>(o + p * hs.row, y);
  }
  if (h_last)
#pragma unroll
    for (int v = 0; v < V; ++v) h_last[chain + v] = s.v[v];
}

// ------------------------------------------------------------------ launches
// Whether every row lets `n` elements be moved whole: the pointers and strides
// are multiples of them, and so is d.
static bool moved_whole(int n, int d, int type, std::initializer_list<std::pair<const void*, RowStrides>> rows) {
  if (d % n) return false;
  for (const auto& r : rows)
    if (r.second.row % n || r.second.chunk % n || !aligned_to(r.first, n * type_bytes(type))) return false;
  return true;
}

// Clusters of `ranks` blocks that the device holds at once: a property of the
// kernel and the device, asked once for each.
template <auto KERNEL>
static int clusters_at_once(int ranks, unsigned threads, size_t smem) {
  static std::atomic<int> known[64][kMaxCluster + 1];  // + 1; 0 = not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  const int k = known[dev][ranks].load(std::memory_order_relaxed);
  if (k) return k - 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ranks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  known[dev][ranks].store(n + 1, std::memory_order_relaxed);
  return n;
}

// The shape of a walk of T positions, P to a team: teams and blocks of a group,
// groups of a block, threads and shared memory of a block, and how many SMs
// have work.
struct Shape {
  int teams, ranks, per, threads;
  size_t smem;
  long long reach;
};
template <auto KERNEL, int V, int G, typename M>
static cudaError_t shape_of(long long chains, int T, int P, M smem, Shape& s) {
  const long long groups = (chains + G * V - 1) / (G * V);
  const bool shared = groups >= 148;  // enough groups to give every SM blocks of its own
  const int block_teams = (shared ? kSharedWarps : alone_warps<V>()) * (32 / G);
  s = {1, 1, 1, 0, 0, 0};
  while (s.teams < block_teams && (long long)s.teams * P < T) s.teams *= 2;
  if (s.teams > block_teams) s.teams = block_teams;
  // short sequences: several groups a block, as long as there are two blocks an SM
  if ((long long)s.teams * P >= T)
    while (s.per * 2 * s.teams <= block_teams && groups / (s.per * 2) >= 2 * 148) s.per *= 2;
  s.threads = s.teams * s.per * G;
  if (s.threads < 32) s.threads = 32;  // two half-warp teams, of two groups
  if (s.threads > s.teams * s.per * G) s.per = s.threads / (s.teams * G);
  // clusters are packed: two of their blocks on one SM while another stays
  // empty, unless a block takes more than half of the shared memory
  const size_t widest = smem(alone_warps<V>() * 32, kMaxCluster), alone = widest < 116 * 1024 ? 116 * 1024 : widest;
  // The limit belongs to the kernel on the device, not to this launch: a
  // constant, so that two threads that launch different shapes agree on it.
  const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)alone);
  if (e != cudaSuccess) return e;
  if (s.teams == block_teams && groups * 2 <= 148)
    for (int r = kMaxCluster; r > 1; --r)
      if ((long long)(r - 1) * s.teams * P < T && groups * r <= 148 &&
          clusters_at_once<KERNEL>(r, (unsigned)s.threads, alone) >= groups) {
        s.ranks = r;
        break;
      }
  s.smem = s.ranks > 1 ? alone : smem(s.threads, 1);
  s.reach = (groups + s.per - 1) / s.per * s.ranks;
  return cudaSuccess;
}
template <auto KERNEL, typename... A>
static cudaError_t launch_walk(const Shape& s, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)s.reach);
  cfg.blockDim = dim3((unsigned)s.threads);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)s.ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = s.ranks > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, KERNEL, args..., s.teams, s.ranks);
  return e != cudaSuccess ? e : cudaGetLastError();
}
// Shared memory of a block.
template <typename E, int V, int G>
static size_t scan_smem(int threads, int ranks) {
  return Walk<V, G>::bytes(threads, ranks, false) +
         (size_t)packs_of_team<G>(kStages, 2, scan_steps<E, V>()) * (threads / G) * sizeof(Pack<E, V>);
}
template <typename E, int V, int G>
static size_t grad_smem(int threads, int ranks) {
  return Walk<V, G>::bytes(threads, ranks, true) +
         (size_t)packs_of_team<G>(kStages, 3, kGradSteps) * (threads / G) * sizeof(Pack<E, V>);
}
// Half-warp teams make twice the groups.  They are taken where more SMs then
// have work (as first measured, 1 x 262144 x 512 fp32 forward: 16 clusters of 6,
// 473 us, against 32 of 4, 392 us; 1 x 65536 x 64: 95 us and 56 us), not where as many have
// (4 x 16384 x 256: 53 us and 58 us).
static bool half_reaches_further(const Shape& half, const Shape& warp) {
  return half.reach <= 148 && half.reach > warp.reach;
}

cudaError_t launch_mingru_scan(const void* zh, int type, RowStrides zs, int B, int T, int d, const int* lengths,
                               const float* h0, void* h, RowStrides hs, float* h_last, float* states,
                               cudaStream_t st) {
  const long long chains = (long long)B * d;
  const FastDiv by_d = fast_div((uint32_t)d);
  const bool pairs = moved_whole(2, d, type, {{zh, zs}, {h, hs}});
  const bool quads = moved_whole(16 / type_bytes(type), d, type, {{zh, zs}});
  return with_type(type, [&](auto t) {
    using E = decltype(t);
    const E* x = static_cast<const E*>(zh);
    E* o = static_cast<E*>(h);
    auto go = [&](auto vec, auto whole) -> cudaError_t {
      constexpr int V = decltype(vec)::value;
      constexpr bool Q = decltype(whole)::value;
      if (T <= kFew) {
        const unsigned blocks = (unsigned)((chains + 256 * V - 1) / (256 * V));
        if (T <= 1)
          mingru_step_kernel<E, V, 1><<<blocks, 256, 0, st>>>(x, zs, T, d, by_d, chains, lengths, h0, o, hs, h_last,
                                                              states);
        else
          mingru_step_kernel<E, V, kFew><<<blocks, 256, 0, st>>>(x, zs, T, d, by_d, chains, lengths, h0, o, hs,
                                                                       h_last, states);
        return cudaGetLastError();
      }
      constexpr auto kernel = mingru_scan_kernel<E, V, 32, Q>;
      constexpr int P = scan_steps<E, V>();
      Shape s, n;
      cudaError_t e = shape_of<kernel, V, 32>(chains, T, P, scan_smem<E, V, 32>, s);
      if (e != cudaSuccess) return e;
      if constexpr (!(V == 2 && sizeof(E) == 4)) {  // those have groups enough
        constexpr auto narrow = mingru_scan_kernel<E, V, 16, Q>;
        if (s.reach < 148) {
          e = shape_of<narrow, V, 16>(chains, T, P, scan_smem<E, V, 16>, n);
          if (e != cudaSuccess) return e;
          if (half_reaches_further(n, s))
            return launch_walk<narrow>(n, st, x, zs, T, d, by_d, chains, lengths, h0, o, hs, h_last, states);
        }
      }
      return launch_walk<kernel>(s, st, x, zs, T, d, by_d, chains, lengths, h0, o, hs, h_last, states);
    };
    // two chains a lane: always for 16 bits; for 32 bits where that leaves
    // groups enough to fill the GPU.  (16 bytes a lane mean 16-bit pairs, so
    // 16-bit single chains never go with them.)
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    if (pairs && (sizeof(E) == 2 || T <= kFew || chains >= 148 * 64))
      return quads && T > kFew ? go(two, std::true_type{}) : go(two, std::false_type{});
    if constexpr (sizeof(E) == 4)
      if (quads) return go(one, std::true_type{});
    return go(one, std::false_type{});
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
  const bool pairs = moved_whole(2, d, type, {{zh, zs}, {dh, dhs}, {dzh, dzs}});
  const bool quads = moved_whole(16 / type_bytes(type), d, type, {{zh, zs}, {dh, dhs}});
  return with_type(type, [&](auto t) {
    using E = decltype(t);
    auto go = [&](auto vec, auto whole) -> cudaError_t {
      constexpr int V = decltype(vec)::value;
      constexpr bool Q = decltype(whole)::value;
      constexpr auto kernel = mingru_grad_kernel<E, V, 32, Q>;
      const E *x = static_cast<const E*>(zh), *u = static_cast<const E*>(dh);
      E* o = static_cast<E*>(dzh);
      Shape s, n;
      cudaError_t e = shape_of<kernel, V, 32>(chains, T, kGradSteps, grad_smem<E, V, 32>, s);
      if (e != cudaSuccess) return e;
      if (s.reach < 148) {
        constexpr auto narrow = mingru_grad_kernel<E, V, 16, Q>;
        e = shape_of<narrow, V, 16>(chains, T, kGradSteps, grad_smem<E, V, 16>, n);
        if (e != cudaSuccess) return e;
        if (half_reaches_further(n, s))
          return launch_walk<narrow>(n, st, x, zs, T, d, by_d, chains, lengths, states, u, dhs, dh_last, o, dzs, dh0);
      }
      return launch_walk<kernel>(s, st, x, zs, T, d, by_d, chains, lengths, states, u, dhs, dh_last, o, dzs, dh0);
    };
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    if constexpr (sizeof(E) == 2) {
      if (pairs) return quads ? go(two, std::true_type{}) : go(two, std::false_type{});
    } else {
      if (quads) return go(one, std::true_type{});
    }
    return go(one, std::false_type{});
  });
}

}  // namespace boa
