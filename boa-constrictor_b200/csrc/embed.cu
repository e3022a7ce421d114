// embed.cu -- embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = s * E[t_i]          dE[v] = s * sum_{i : t_i = v} dout[i]
//
// Lookup.  n * d elements leave, and the table (at most 1024 rows) is read
// from the caches, so the stores set the pace.
//
// Gradient.  Every row of dout is read once, whatever its token: the
// positions are first ordered by token with a stable counting sort (at most
// 1024 tokens, so one pass), and the sums then run over consecutive sorted
// positions in registers.  The sorted positions of a token are cut into
// pieces, so that a token that makes up most of the input (the zero byte of
// binary records) is summed by as many blocks as its share of the rows; the
// block that finishes a token last adds its pieces' sums in their order.
// Nothing is added atomically in floating point, and the same input gives the
// same bits.
//
// Measured on a B200: 1M x 256 fp32 lookup 148 us (7.2 TB/s of stores); its
// gradient 191 us; profiled one by one, the row sums take 167 us (6.4 TB/s) and
// the sort's three launches 26 us.  bf16: 115 us (floor 82).
#include "pieces.h"
#include "ptx.cuh"
#include "train_ops.cuh"

namespace boa {

// ------------------------------------------------------------------ lookup
// A block writes `rows` rows; an item of a row is H packs of N elements, d / H
// apart, and thread k takes items k, k + 256, ... of the block's rows * q.  The
// row of item l is umulhi(l, magic) with magic = ceil(2^32 / q), exact while
// l * q < 2^32.  A pack has 16 bytes in the wider of the two types: with more, a
// warp's loads from the table would skip every other 16 bytes and take twice
// the L1 cycles.
constexpr int kEmbedThreads = 256;

template <typename Tok, typename TI, typename TO, int N, int H, int U>
__global__ void __launch_bounds__(kEmbedThreads)
embed_kernel(const Tok* __restrict__ tok, long long n, const TI* __restrict__ table, long long ld_table, int vocab,
             int q, uint32_t magic, int rows, float scale, TO* __restrict__ out, long long ld_out) {
  const long long r0 = (long long)blockIdx.x * rows;
  const int here = (int)(n - r0 < rows ? n - r0 : rows);
  const int items = here * q, apart = q * N;
  for (int l0 = threadIdx.x; l0 < items; l0 += kEmbedThreads * U) {
    int row[U], idx[U];
    Pack<TI, N> e[U][H];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int l = l0 + u * kEmbedThreads;
      row[u] = q == 1 ? l : (int)__umulhi((uint32_t)l, magic);
      idx[u] = l < items ? token_index(tok[r0 + row[u]], vocab) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const TI* from = table + idx[u] * ld_table + (l0 + u * kEmbedThreads - row[u] * q) * N;
#pragma unroll
      for (int k = 0; k < H; ++k)
        if (idx[u] >= 0) e[u][k] = *reinterpret_cast<const Pack<TI, N>*>(from + k * apart);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int l = l0 + u * kEmbedThreads;
      if (l >= items) break;
      TO* to = out + (r0 + row[u]) * ld_out + (l - row[u] * q) * N;
#pragma unroll
      for (int k = 0; k < H; ++k) {
        float o[N];
        if (idx[u] >= 0) widen_pack(e[u][k], o);
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = idx[u] >= 0 ? scale * o[j] : 0.f;
        *reinterpret_cast<Pack<TO, N>*>(to + k * apart) = narrow_pack<TO>(o);
      }
    }
  }
}

template <typename Tok, typename TI, typename TO, int N, int H, int U>
static cudaError_t embed_run(const Tok* tok, long long n, const TI* table, long long ld_table, int vocab, int d,
                             float scale, TO* out, long long ld_out, cudaStream_t st) {
  const int q = d / (N * H);
  // about two rounds of kEmbedThreads * U items per block
  int rows = 2 * kEmbedThreads * U / q;
  rows = rows < 1 ? 1 : rows;
  const long long blocks = (n + rows - 1) / rows;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const uint32_t magic = (uint32_t)(((1ull << 32) + q - 1) / q);
  embed_kernel<Tok, TI, TO, N, H, U><<<(unsigned)blocks, kEmbedThreads, 0, st>>>(
      tok, n, table, ld_table, vocab, q, magic, rows, scale, out, ld_out);
  return cudaGetLastError();
}

cudaError_t launch_embed(const void* tokens, int tok_t, long long n, const void* table, int table_t,
                         long long ld_table, int vocab, int d, float scale, void* out, int out_t, long long ld_out,
                         cudaStream_t st) {
  return with_token(tok_t, [&](auto tk) {
    return with_type(table_t, [&](auto ti) {
      return with_type(out_t, [&](auto to) {
        using Tok = decltype(tk);
        using TI = decltype(ti);
        using TO = decltype(to);
        constexpr int N = 16 / (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO));
        const Tok* t = static_cast<const Tok*>(tokens);
        const TI* e = static_cast<const TI*>(table);
        TO* o = static_cast<TO*>(out);
        const bool wide = d % N == 0 && ld_out % N == 0 && ld_table % N == 0 &&
                          aligned_to(o, (int)alignof(Pack<TO, N>)) && aligned_to(e, (int)alignof(Pack<TI, N>));
        // Four packs an item share a token's lookup where rows are long (1M x 512,
        // fp32 table, bf16 out: 177 us, two 198 us, one 276 us); short rows want
        // items of more rows at once instead (1M x 64 bf16: two packs 31 us, four
        // 40 us; 1M x 16 fp32: one 13.5 us, two 17 us).
        const int packs = d / N;
        if (!wide) return embed_run<Tok, TI, TO, 1, 1, 4>(t, n, e, ld_table, vocab, d, scale, o, ld_out, st);
        if (packs >= 64 && packs % 4 == 0)
          return embed_run<Tok, TI, TO, N, 4, 1>(t, n, e, ld_table, vocab, d, scale, o, ld_out, st);
        if (packs >= 8 && packs % 2 == 0)
          return embed_run<Tok, TI, TO, N, 2, 2>(t, n, e, ld_table, vocab, d, scale, o, ld_out, st);
        return embed_run<Tok, TI, TO, N, 1, 4>(t, n, e, ld_table, vocab, d, scale, o, ld_out, st);
      });
    });
  });
}

// ---------------------------------------------------------------- gradient
// Workspace, as 32-bit words: counts [V][tiles], then exclusive along the
// tiles; total [V]; done [V], finished pieces of each token; order [n];
// pieces [most] of four words (and their number before them); and the pieces'
// sums [most][d] in fp32.
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortHeld = 8;                               // tokens that a lane holds at once
constexpr int kTile = kSortThreads * kSortHeld;            // least tokens of a tile
constexpr int kMaxTiles = 1024;
constexpr int kSumThreads = 256;
constexpr int kSumChunk = 1024;    // positions of a piece in shared memory at once
constexpr int kSmallRows = 4096;   // up to here one kernel does all
constexpr int kSmallPacks = 16;

struct GradPlan {
  int tiles, tile;                 // tiles of the sort, tokens of a tile
  int rows;                        // rows of a piece (more for a token of over kMaxPieces * rows)
  long long most;                  // pieces there can be
  size_t counts, total, done, order, pieces, part, words;  // offsets in words
};
static GradPlan grad_plan(long long n, int vocab, int d) {
  GradPlan p{};
  long long tile = (n + kMaxTiles - 1) / kMaxTiles;
  tile = (tile + kTile - 1) / kTile * kTile;
  p.tile = (int)tile;
  p.tiles = (int)((n + tile - 1) / tile);
  // about sixteen blocks per SM
  const long long rows = (n + 148 * 16 - 1) / (148 * 16);
  p.rows = (int)(rows < 128 ? 128 : (rows + 31) / 32 * 32);
  p.most = n / p.rows + vocab;     // at least the sum of pieces_of(total)
  auto up4 = [](size_t x) { return (x + 3) & ~(size_t)3; };
  p.counts = 0;
  p.total = up4(p.counts + (size_t)vocab * p.tiles);
  p.done = up4(p.total + vocab);
  p.order = up4(p.done + vocab);
  p.pieces = up4(p.order + (size_t)n);
  p.part = p.pieces + 4 * (size_t)(p.most + 1);
  p.words = p.part + (size_t)p.most * d;
  return p;
}
size_t embed_grad_workspace(long long n, int vocab, int d) {
  return n > kSmallRows ? grad_plan(n, vocab, d).words * 4 : 0;
}
struct alignas(16) Piece {
  int tok_pieces;  // token, and its pieces << 16
  int at, rows;    // sorted positions
  int first;       // the token's first piece
};

// The tokens of 32 * kSortHeld positions from `at`, lane by lane; -1 past `end`.
template <typename Tok>
__device__ __forceinline__ void load_tokens(const Tok* __restrict__ tok, long long at, long long end, int vocab,
                                            int (&v)[kSortHeld]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < kSortHeld; ++j) {
    const long long i = at + j * 32 + lane;
    v[j] = i < end ? token_index(tok[i], vocab) : -1;
  }
}

// Counts of each token in each tile; warp w owns the w-th part of the tile.
template <typename Tok>
__global__ void __launch_bounds__(kSortThreads)
embed_count_kernel(const Tok* __restrict__ tok, long long n, int vocab, int tile, int tiles, int* __restrict__ counts) {
  extern __shared__ int hist[];  // [kSortWarps][vocab]
  const int warp = threadIdx.x >> 5;
  const int span = tile / kSortWarps;
  const long long w0 = (long long)blockIdx.x * tile + (long long)warp * span;
  const long long w1 = w0 + span < n ? w0 + span : n;
  int v[kSortHeld];
  load_tokens(tok, w0, w1, vocab, v);
  for (int i = threadIdx.x; i < kSortWarps * vocab; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  int* mine = hist + warp * vocab;
  for (long long at = w0; at < w1; at += 32 * kSortHeld) {
    if (at > w0) load_tokens(tok, at, w1, vocab, v);
#pragma unroll
    for (int j = 0; j < kSortHeld; ++j)
      if (v[j] >= 0) atomicAdd(mine + v[j], 1);
  }
  __syncthreads();
  for (int k = threadIdx.x; k < vocab; k += kSortThreads) {
    int s = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) s += hist[w * vocab + k];
    counts[(size_t)k * tiles + blockIdx.x] = s;
  }
}

// Exclusive prefix of one int per thread over the block; scratch [threads / 32].
template <int THREADS>
__device__ __forceinline__ int block_prefix(int x, int* scratch, int& sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, s, o);
    if (lane >= o) s += y;
  }
  if (lane == 31) scratch[warp] = s;
  __syncthreads();
  int before = s - x;
  sum = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += scratch[w];
    sum += scratch[w];
  }
  __syncthreads();
  return before;
}

// counts of one token -> exclusive prefix along the tiles, and the total
constexpr int kPrefixThreads = 128;
__global__ void __launch_bounds__(kPrefixThreads)
embed_prefix_kernel(int* __restrict__ counts, int tiles, int* __restrict__ total, int* __restrict__ done) {
  __shared__ int scratch[kPrefixThreads / 32];
  constexpr int PER = kMaxTiles / kPrefixThreads;
  int* c = counts + (size_t)blockIdx.x * tiles;
  int x[PER], sum = 0, all;
  const int t0 = threadIdx.x * PER;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    x[k] = t0 + k < tiles ? c[t0 + k] : 0;
    sum += x[k];
  }
  int before = block_prefix<kPrefixThreads>(sum, scratch, all);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (t0 + k < tiles) c[t0 + k] = before;
    before += x[k];
  }
  if (threadIdx.x == 0) {
    total[blockIdx.x] = all;
    done[blockIdx.x] = 0;
  }
}

// Exclusive prefix over the tokens of f(total[v]), written to out[0..vocab].
template <typename F>
__device__ __forceinline__ void vocab_prefix(const int* __restrict__ total, int vocab, F f, int* out, int* scratch) {
  constexpr int PER = kMaxVocab / kSortThreads;
  int x[PER], sum = 0, all;
  const int v0 = threadIdx.x * PER;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    x[k] = v0 + k < vocab ? f(total[v0 + k]) : 0;
    sum += x[k];
  }
  int before = block_prefix<kSortThreads>(sum, scratch, all);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (v0 + k < vocab) out[v0 + k] = before;
    before += x[k];
  }
  if (threadIdx.x == 0) out[vocab] = all;
  __syncthreads();
}

// Writes each position to its place in token order, and the pieces.  A warp takes its part of
// the tile 32 tokens at a time: lanes that hold the same token find each
// other with a match, so equal tokens keep the order of their positions.
template <typename Tok>
__global__ void __launch_bounds__(kSortThreads)
embed_order_kernel(const Tok* __restrict__ tok, long long n, int vocab, int tile, int tiles, int rows,
                   const int* __restrict__ counts, const int* __restrict__ total, Piece* __restrict__ pieces,
                   int* __restrict__ order) {
  // [kSortWarps][vocab] next places, base and first piece [vocab + 1] each, scratch [kSortWarps]
  extern __shared__ int hist[];
  int* base = hist + kSortWarps * vocab;
  int* first = base + vocab + 1;
  int* scratch = first + vocab + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int span = tile / kSortWarps;
  const long long w0 = (long long)blockIdx.x * tile + (long long)warp * span;
  const long long w1 = w0 + span < n ? w0 + span : n;
  int v[kSortHeld];
  load_tokens(tok, w0, w1, vocab, v);
  for (int i = threadIdx.x; i < kSortWarps * vocab; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  int* next = hist + warp * vocab;
  for (long long at = w0; at < w1; at += 32 * kSortHeld) {
    if (at > w0) load_tokens(tok, at, w1, vocab, v);
#pragma unroll
    for (int j = 0; j < kSortHeld; ++j)
      if (v[j] >= 0) atomicAdd(next + v[j], 1);
  }
  vocab_prefix(total, vocab, [&](int c) { return pieces_of(c, rows); }, first, scratch);
  vocab_prefix(total, vocab, [](int c) { return c; }, base, scratch);
  // the pieces, for the kernel that follows; pieces[0].at is their number
  if (blockIdx.x == 0 && threadIdx.x == 0) pieces[0].at = first[vocab];
  for (int k = blockIdx.x; k < vocab; k += gridDim.x) {
    const int count = base[k + 1] - base[k], size = rows_of_piece(count, rows), n_pieces = first[k + 1] - first[k];
    for (int j = threadIdx.x; j < n_pieces; j += kSortThreads)
      pieces[1 + first[k] + j] = {k | n_pieces << 16, base[k] + j * size, max(0, min(size, count - j * size)), first[k]};
  }
  for (int k = threadIdx.x; k < vocab; k += kSortThreads) {
    int at = base[k] + counts[(size_t)k * tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = hist[w * vocab + k];
      hist[w * vocab + k] = at;
      at += c;
    }
  }
  __syncthreads();
  for (long long at = w0; at < w1; at += 32 * kSortHeld) {
    if (span > 32 * kSortHeld) load_tokens(tok, at, w1, vocab, v);
#pragma unroll
    for (int j = 0; j < kSortHeld; ++j) {
      const unsigned same = __match_any_sync(~0u, v[j]);
      const int rank = __popc(same & ((1u << lane) - 1));
      const int to = v[j] >= 0 ? next[v[j]] + rank : 0;
      __syncwarp();
      if (v[j] >= 0) {
        if (rank == 0) next[v[j]] = to + __popc(same);
        order[to] = (int)(at + j * 32 + lane);
      }
      __syncwarp();
    }
  }
}

// Up to kClusterRows rows: one cluster of eight blocks sorts instead of three
// launches of the kernels above (the whole gradient of 5000 x 256: 23 us against
// 35 us, of 20000 x 160 over 1000 tokens 24 and 40; from 65536 rows on the
// eight SMs are slower, 29.5 and 27.5).  A block counts its eighth of the
// positions, 32 warps with a row of counts each; the blocks read each other's
// totals, and go on as above.
constexpr int kClusterBlocks = 8, kClusterThreads = 1024, kClusterWarps = kClusterThreads / 32;
constexpr int kClusterHeld = 6;   // tokens of a lane
constexpr int kClusterRows = kClusterBlocks * kClusterThreads * kClusterHeld;
constexpr int cluster_smem(int vocab) { return ((kClusterWarps + 2) * vocab + kClusterWarps) * 4; }

template <typename Tok>
__global__ void __launch_bounds__(kClusterThreads)
embed_sort_kernel(const Tok* __restrict__ tok, int n, int span, int vocab, int rows, Piece* __restrict__ pieces,
                  int* __restrict__ done, int* __restrict__ order) {
  // [kClusterWarps][vocab] counts, the block's totals [vocab], first places [vocab], scratch
  extern __shared__ int hist[];
  int* mine = hist + kClusterWarps * vocab;
  int* start = mine + vocab;
  int* scratch = start + vocab;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_rank();
  const int w0 = (rank * kClusterWarps + warp) * span, w1 = min(n, w0 + span);
  int v[kClusterHeld];
#pragma unroll
  for (int j = 0; j < kClusterHeld; ++j) {
    const int i = w0 + j * 32 + lane;
    v[j] = i < w1 ? token_index(tok[i], vocab) : -1;
  }
  for (int i = threadIdx.x; i < kClusterWarps * vocab; i += kClusterThreads) hist[i] = 0;
  __syncthreads();
  int* next = hist + warp * vocab;
#pragma unroll
  for (int j = 0; j < kClusterHeld; ++j)
    if (v[j] >= 0) atomicAdd(next + v[j], 1);
  __syncthreads();
  const int k = threadIdx.x;  // this thread's token
  if (k < vocab) {
    int sum = 0;
#pragma unroll 8
    for (int w = 0; w < kClusterWarps; ++w) {
      const int c = hist[w * vocab + k];
      hist[w * vocab + k] = sum;
      sum += c;
    }
    mine[k] = sum;
  }
  __syncwarp();  // the barrier is for whole warps, and the alphabet may end inside one
  cluster_sync_all();
  int before = 0, count = 0, all;  // of the blocks before this one, and of all
  if (k < vocab)
#pragma unroll
    for (int r = 0; r < kClusterBlocks; ++r) {
      int c;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c) : "r"(cluster_addr(mine + k, r)) : "memory");
      if (r < rank) before += c;
      count += c;
    }
  __syncwarp();
  cluster_sync_all();  // no block leaves while its totals are read
  const int n_pieces = k < vocab ? pieces_of(count, rows) : 0;
  const int base = block_prefix<kClusterThreads>(count, scratch, all);
  const int first = block_prefix<kClusterThreads>(n_pieces, scratch, all);
  if (k < vocab) {
    start[k] = base + before;
    if (k % kClusterBlocks == rank) {
      const int size = rows_of_piece(count, rows);
      for (int j = 0; j < n_pieces; ++j)
        pieces[1 + first + j] = {k | n_pieces << 16, base + j * size, max(0, min(size, count - j * size)), first};
      done[k] = 0;
    }
  }
  if (rank == 0 && k == 0) pieces[0].at = all;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kClusterHeld; ++j) {
    const unsigned same = __match_any_sync(~0u, v[j]);
    const int place = __popc(same & ((1u << lane) - 1));
    const int to = v[j] >= 0 ? next[v[j]] : 0;
    __syncwarp();
    if (v[j] >= 0) {
      if (place == 0) next[v[j]] = to + __popc(same);
      order[start[v[j]] + to + place] = w0 + j * 32 + lane;
    }
    __syncwarp();
  }
}

// out (+)= scale * sum of N columns
template <typename TD, int N>
__device__ __forceinline__ void store_grad(TD* out, const float (&sum)[N], float scale, int accumulate) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float r = sum[k] * scale;
    out[k] = from_f32<TD>(accumulate ? r + to_f32(out[k]) : r);
  }
}
// Adds up what the `groups` groups of `per_row` threads hold, N columns a
// thread, in the order of the groups; the result is group 0's.
template <int N>
__device__ __forceinline__ void join_groups(float (&acc)[N], float* s_sum, int g, int groups, int col, int per_row) {
#pragma unroll
  for (int k = 0; k < N; ++k) s_sum[k * kSumThreads + threadIdx.x] = acc[k];
  __syncthreads();
  if (g == 0)
    for (int j = 1; j < groups; ++j)
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += s_sum[k * kSumThreads + j * per_row + col];
  __syncthreads();
}

// Sum of one piece: the block's threads form groups of `per_row` threads, one
// pack of N columns each; group g takes the piece's rows g, g + groups, ...
// The block that finishes a token's pieces last adds them up.
template <typename TG, typename TD, int N>
__global__ void __launch_bounds__(kSumThreads)
embed_sum_kernel(const TG* __restrict__ dout, long long ld, int d, int per_row, const Piece* __restrict__ all,
                 const int* __restrict__ order, int* __restrict__ done, float* __restrict__ part, float scale,
                 int accumulate, TD* dtable, long long ld_dtable) {
  __shared__ int s_last, s_order[kSumChunk];
  __shared__ float s_sum[kSumThreads * N];
  const int p = blockIdx.x;
  const Piece me = all[1 + p];
  if (p >= all[0].at) return;
  const int v = me.tok_pieces & 0xffff, pieces = me.tok_pieces >> 16, rows = me.rows;
  const int* mine = order + me.at;
  const int groups = kSumThreads / per_row, g = threadIdx.x / per_row, col = threadIdx.x - g * per_row;
  const int q = d / N;
  for (int c0 = 0; c0 < q; c0 += per_row) {
    const int c = c0 + col;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    for (int r0 = 0; r0 < rows; r0 += kSumChunk) {
      const int here = min(kSumChunk, rows - r0);
      if (r0 || !c0) {
        if (r0) __syncthreads();
        for (int i = threadIdx.x; i < here; i += kSumThreads) s_order[i] = mine[r0 + i];
        __syncthreads();
      } else if (rows > kSumChunk) {  // the first chunk again, for the next columns
        for (int i = threadIdx.x; i < here; i += kSumThreads) s_order[i] = mine[i];
        __syncthreads();
      }
      if (g < groups && c < q) {
        const TG* x = dout + (size_t)c * N;
#pragma unroll 8
        for (int r = g; r < here; r += groups) {
          float y[N];
          widen_pack(load_once<TG, N>(x + s_order[r] * ld), y);
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += y[k];
        }
      }
    }
    join_groups<N>(acc, s_sum, g, groups, col, per_row);
    if (g == 0 && c < q) {
      if (pieces == 1) {
        store_grad<TD, N>(dtable + v * ld_dtable + c * N, acc, scale, accumulate);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) __stcg(part + (size_t)p * d + c * N + k, acc[k]);
      }
    }
  }
  if (pieces == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(done + v, 1) == pieces - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int c0 = 0; c0 < q; c0 += per_row) {
    const int c = c0 + col;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    if (g < groups && c < q) {
      const float* x = part + (size_t)me.first * d + c * N;
#pragma unroll 8
      for (int r = g; r < pieces; r += groups)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += __ldcg(x + (size_t)r * d + k);
    }
    join_groups<N>(acc, s_sum, g, groups, col, per_row);
    if (g == 0 && c < q) store_grad<TD, N>(dtable + v * ld_dtable + c * N, acc, scale, accumulate);
  }
}

// Few rows: one kernel instead of the cluster's sort and the sums.  On the GPU,
// fp32 rows spread over 256 tokens: 1024 x 64 4.8 us against 10.3, 4096 x 256 8.2
// against 11.3, 8192 x 256 11.5 against 11.6.  It is the slower one where few blocks
// have the work (4096 rows of one token 37 against 14) and for large alphabets
// (4096 x 160 bf16 over 1000 tokens 23 against 15); the rule sees the number of
// rows alone.  A block takes `per` tokens and up to kSmallPacks packs
// of columns; it reads all tokens into shared memory, and for each of its own
// tokens lists the positions in order (a lane keeps the match mask of every
// 32 positions of its warp's part) and sums their rows.
template <typename Tok, typename TG, typename TD, int N>
__global__ void __launch_bounds__(kSumThreads)
embed_small_kernel(const Tok* __restrict__ tok, int n, const TG* __restrict__ dout, long long ld, int vocab, int d,
                   int per, float scale, int accumulate, TD* dtable, long long ld_dtable) {
  static_assert(kSmallRows <= 32 * 32 * (kSumThreads / 32), "a lane holds one mask");
  __shared__ short s_tok[kSmallRows], s_order[kSmallRows];
  __shared__ int s_count[kSumThreads / 32];
  __shared__ float s_sum[kSumThreads * N];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int q = d / N, c0 = blockIdx.y * kSmallPacks, packs = min(kSmallPacks, q - c0);
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += kSumThreads) s_tok[i] = (short)token_index(tok[i], vocab);
  __syncthreads();
  // this warp's part of the positions: whole groups of 32, at most 16 of them
  const int span = (n + kSumThreads - 1) / kSumThreads * 32, w0 = warp * span, w1 = min(n, w0 + span);
  const int groups = kSumThreads / packs, g = threadIdx.x / packs, col = threadIdx.x - g * packs;
  const int v1 = min(vocab, (int)(blockIdx.x + 1) * per);
  for (int v = blockIdx.x * per; v < v1; ++v) {
    unsigned mask = 0;
    for (int j = 0; w0 + j * 32 < w1; ++j) {
      const int i = w0 + j * 32 + lane;
      const unsigned m = __ballot_sync(~0u, i < w1 && s_tok[i] == v);
      if (lane == j) mask = m;
    }
    int at = __popc(mask), sum = at;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, at, o);
      if (lane >= o) at += y;
    }
    if (lane == 31) s_count[warp] = at;
    at -= sum;
    __syncthreads();
    int rows = 0;
#pragma unroll
    for (int w = 0; w < kSumThreads / 32; ++w) {
      if (w < warp) at += s_count[w];
      rows += s_count[w];
    }
    for (; mask; mask &= mask - 1) s_order[at++] = (short)(w0 + lane * 32 + __ffs(mask) - 1);
    __syncthreads();
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    if (g < groups) {
      const TG* x = dout + (size_t)(c0 + col) * N;
#pragma unroll 8
      for (int r = g; r < rows; r += groups) {
        float y[N];
        widen_pack(load_once<TG, N>(x + s_order[r] * ld), y);
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += y[k];
      }
    }
    join_groups<N>(acc, s_sum, g, groups, col, packs);
    if (g == 0 && (rows || !accumulate))
      store_grad<TD, N>(dtable + v * ld_dtable + (c0 + col) * N, acc, scale, accumulate);
  }
}

template <typename TD>
__global__ void __launch_bounds__(256) embed_zero_kernel(TD* dtable, long long ld, int d) {
  for (int c = threadIdx.x; c < d; c += 256) dtable[blockIdx.x * ld + c] = from_f32<TD>(0.f);
}

template <typename Tok>
static cudaError_t launch_sort(const Tok* tok, int n, int vocab, int rows, Piece* pieces, int* done, int* order,
                               cudaStream_t st) {
  const auto kernel = embed_sort_kernel<Tok>;
  const int warps = kClusterBlocks * kClusterWarps, span = ((n + warps - 1) / warps + 31) / 32 * 32;
  // the limit is the kernel's, whatever thread launches it: always the largest alphabet's
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, cluster_smem(kMaxVocab));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kClusterBlocks);
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = (size_t)cluster_smem(vocab);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = kClusterBlocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, tok, n, span, vocab, rows, pieces, done, order);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename Tok, typename TG, typename TD, int N>
static cudaError_t grad_run(const Tok* tok, long long n, const TG* dout, long long ld, int vocab, int d, float scale,
                            bool accumulate, TD* dtable, long long ld_dtable, int* w, cudaStream_t st) {
  const int q = d / N;
  if (n <= kSmallRows) {
    const int per = (vocab + 147) / 148;
    embed_small_kernel<Tok, TG, TD, N><<<dim3((vocab + per - 1) / per, (q + kSmallPacks - 1) / kSmallPacks), kSumThreads, 0, st>>>(
        tok, (int)n, dout, ld, vocab, d, per, scale, accumulate ? 1 : 0, dtable, ld_dtable);
    return cudaGetLastError();
  }
  const GradPlan p = grad_plan(n, vocab, d);
  Piece* pieces = reinterpret_cast<Piece*>(w + p.pieces);
  cudaError_t e;
  if (n <= kClusterRows) {
    e = launch_sort(tok, (int)n, vocab, p.rows, pieces, w + p.done, w + p.order, st);
  } else {
    const size_t hist_bytes = (size_t)kSortWarps * vocab * 4;
    embed_count_kernel<Tok><<<p.tiles, kSortThreads, hist_bytes, st>>>(tok, n, vocab, p.tile, p.tiles, w + p.counts);
    embed_prefix_kernel<<<vocab, kPrefixThreads, 0, st>>>(w + p.counts, p.tiles, w + p.total, w + p.done);
    embed_order_kernel<Tok><<<p.tiles, kSortThreads, hist_bytes + (2 * (vocab + 1) + kSortWarps) * 4, st>>>(
        tok, n, vocab, p.tile, p.tiles, p.rows, w + p.counts, w + p.total, pieces, w + p.order);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  embed_sum_kernel<TG, TD, N><<<(unsigned)p.most, kSumThreads, 0, st>>>(
      dout, ld, d, q < kSumThreads ? q : kSumThreads, pieces, w + p.order, w + p.done,
      reinterpret_cast<float*>(w + p.part), scale, accumulate ? 1 : 0, dtable, ld_dtable);
  return cudaGetLastError();
}

cudaError_t launch_embed_grad(const void* tokens, int tok_t, long long n, const void* dout, int dout_t,
                              long long ld_dout, int vocab, int d, float scale, bool accumulate, void* dtable,
                              int dtable_t, long long ld_dtable, void* ws, cudaStream_t st) {
  return with_type(dtable_t, [&](auto td) {
    using TD = decltype(td);
    TD* out = static_cast<TD*>(dtable);
    if (n == 0) {
      if (accumulate) return cudaSuccess;
      embed_zero_kernel<TD><<<vocab, 256, 0, st>>>(out, ld_dtable, d);
      return cudaGetLastError();
    }
    return with_type(dout_t, [&](auto tg) {
      return with_token(tok_t, [&](auto tk) {
        using TG = decltype(tg);
        using Tok = decltype(tk);
        constexpr int N = 16 / sizeof(TG);
        const TG* x = static_cast<const TG*>(dout);
        const Tok* t = static_cast<const Tok*>(tokens);
        int* w = static_cast<int*>(ws);
        const bool wide = d % N == 0 && ld_dout % N == 0 && aligned_to(x, 16);
        return wide ? grad_run<Tok, TG, TD, N>(t, n, x, ld_dout, vocab, d, scale, accumulate, out, ld_dtable, w, st)
                    : grad_run<Tok, TG, TD, 1>(t, n, x, ld_dout, vocab, d, scale, accumulate, out, ld_dtable, w, st);
      });
    });
  });
}

}  // namespace boa
