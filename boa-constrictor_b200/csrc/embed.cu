// embed.cu -- embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i] = s * E[t_i]          dE[v] = s * sum_{i : t_i = v} dout[i]
//
// Forward.  n * d elements leave, and the table (at most 1024 rows) is read
// from the caches, so the stores set the pace.
//
// Gradient.  Every row of dout is read once, whatever its token: the
// positions are first ordered by token with a stable counting sort (at most
// 1024 tokens, so one pass), and the sums then run over consecutive sorted
// positions in registers.  The sorted positions of a token are cut into
// pieces of equal length, so that a token that makes up most of the input
// (the zero byte of binary records) is summed by as many blocks as its share
// of the rows; the pieces' sums are added in order.  Nothing is added
// atomically in floating point, and the same input gives the same bits.
#include "kernels.cuh"
#include "ptx.cuh"
#include "train_ops.cuh"

namespace boa {

// ------------------------------------------------------------------ lookup
// A block writes `rows` rows of q packs of N elements; thread k takes packs
// k, k + 256, ...  The row of pack l is umulhi(l, magic) with
// magic = ceil(2^32 / q), exact while l * q < 2^32.
constexpr int kEmbedThreads = 256;
constexpr int kEmbedUnroll = 4;

template <typename Tok, typename TI, typename TO, int N>
__global__ void __launch_bounds__(kEmbedThreads)
embed_kernel(const Tok* __restrict__ tok, long long n, const TI* __restrict__ table, long long ld_table, int vocab,
             int q, uint32_t magic, int rows, float scale, TO* __restrict__ out, long long ld_out) {
  const long long r0 = (long long)blockIdx.x * rows;
  const int here = (int)(n - r0 < rows ? n - r0 : rows);
  const int items = here * q;
  for (int l0 = threadIdx.x; l0 < items; l0 += kEmbedThreads * kEmbedUnroll) {
    int row[kEmbedUnroll], idx[kEmbedUnroll];
    Pack<TI, N> e[kEmbedUnroll];
#pragma unroll
    for (int u = 0; u < kEmbedUnroll; ++u) {
      const int l = l0 + u * kEmbedThreads;
      row[u] = q == 1 ? l : (int)__umulhi((uint32_t)l, magic);
      idx[u] = l < items ? token_index(tok[r0 + row[u]], vocab) : -1;
    }
#pragma unroll
    for (int u = 0; u < kEmbedUnroll; ++u) {
      const int c = (l0 + u * kEmbedThreads - row[u] * q) * N;
      if (idx[u] >= 0) e[u] = *reinterpret_cast<const Pack<TI, N>*>(table + idx[u] * ld_table + c);
    }
#pragma unroll
    for (int u = 0; u < kEmbedUnroll; ++u) {
      const int l = l0 + u * kEmbedThreads;
      if (l >= items) break;
      const int c = (l - row[u] * q) * N;
      Pack<TO, N> o;
#pragma unroll
      for (int k = 0; k < N; ++k) o.v[k] = from_f32<TO>(idx[u] >= 0 ? scale * to_f32(e[u].v[k]) : 0.f);
      *reinterpret_cast<Pack<TO, N>*>(out + (r0 + row[u]) * ld_out + c) = o;
    }
  }
}

template <typename Tok, typename TI, typename TO, int N>
static cudaError_t embed_run(const Tok* tok, long long n, const TI* table, long long ld_table, int vocab, int d,
                             float scale, TO* out, long long ld_out, cudaStream_t st) {
  const int q = d / N;
  // about two rounds of kEmbedThreads * kEmbedUnroll packs per block
  int rows = 2 * kEmbedThreads * kEmbedUnroll / q;
  rows = rows < 1 ? 1 : rows;
  const long long blocks = (n + rows - 1) / rows;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const uint32_t magic = (uint32_t)(((1ull << 32) + q - 1) / q);
  embed_kernel<Tok, TI, TO, N><<<(unsigned)blocks, kEmbedThreads, 0, st>>>(tok, n, table, ld_table, vocab, q, magic,
                                                                           rows, scale, out, ld_out);
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
        constexpr int N = 16 / sizeof(TO);
        const Tok* t = static_cast<const Tok*>(tokens);
        const TI* e = static_cast<const TI*>(table);
        TO* o = static_cast<TO*>(out);
        const bool wide = d % N == 0 && ld_out % N == 0 && ld_table % N == 0 && aligned_to(o, 16) &&
                          aligned_to(e, (int)alignof(Pack<TI, N>));
        return wide ? embed_run<Tok, TI, TO, N>(t, n, e, ld_table, vocab, d, scale, o, ld_out, st)
                    : embed_run<Tok, TI, TO, 1>(t, n, e, ld_table, vocab, d, scale, o, ld_out, st);
      });
    });
  });
}

// ---------------------------------------------------------------- gradient
// Workspace, as 32-bit words: counts [V][tiles], then exclusive along the
// tiles; total [V]; base [V + 1] and piece_base [V + 1], the first sorted
// position and the first piece of each token; order [n]; and the pieces'
// sums [pieces][d] in fp32.
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kPieceRows = 512;
constexpr int kSumThreads = 256;

struct GradPlan {
  int tiles;           // tiles of the sort
  int tile;            // tokens per tile, a multiple of 32 * kSortWarps
  long long pieces;    // most pieces there can be
  size_t counts, total, base, piece_base, order, part, words;  // offsets in words
};

static GradPlan grad_plan(long long n, int vocab, int d) {
  GradPlan p{};
  // at least 4096 tokens a tile, at most about two tiles per SM
  long long tile = (n + 295) / 296;
  if (tile < 4096) tile = 4096;
  tile = (tile + kSortThreads - 1) / kSortThreads * kSortThreads;
  p.tile = (int)tile;
  p.tiles = (int)((n + tile - 1) / tile);
  p.pieces = n / kPieceRows + vocab;  // sum of ceil(total / kPieceRows)
  auto up4 = [](size_t x) { return (x + 3) & ~(size_t)3; };
  p.counts = 0;
  p.total = up4(p.counts + (size_t)vocab * p.tiles);
  p.base = up4(p.total + vocab);
  p.piece_base = up4(p.base + vocab + 1);
  p.order = up4(p.piece_base + vocab + 1);
  p.part = up4(p.order + (size_t)n);
  p.words = p.part + (size_t)p.pieces * d;
  return p;
}
size_t embed_grad_workspace(long long n, int vocab, int d) { return n > 0 ? grad_plan(n, vocab, d).words * 4 : 0; }

// Counts of each token in each tile, per warp in shared memory: warp w owns
// the w-th contiguous part of the tile.  Returns with `mine` complete.
template <typename Tok>
__device__ __forceinline__ void count_tile(const Tok* __restrict__ tok, long long w0, long long w1, int vocab,
                                           int* mine) {
  const int lane = threadIdx.x & 31;
  for (long long i = w0 + lane; i < w1; i += 32) {
    const int v = token_index(tok[i], vocab);
    if (v >= 0) atomicAdd(mine + v, 1);
  }
}

template <typename Tok>
__global__ void __launch_bounds__(kSortThreads)
embed_count_kernel(const Tok* __restrict__ tok, long long n, int vocab, int tile, int tiles, int* __restrict__ counts) {
  extern __shared__ int hist[];  // [kSortWarps][vocab]
  const int warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kSortWarps * vocab; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  const int span = tile / kSortWarps;
  const long long w0 = (long long)blockIdx.x * tile + (long long)warp * span;
  const long long w1 = w0 + span < n ? w0 + span : n;
  count_tile(tok, w0, w1, vocab, hist + warp * vocab);
  __syncthreads();
  for (int v = threadIdx.x; v < vocab; v += kSortThreads) {
    int s = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) s += hist[w * vocab + v];
    counts[(size_t)v * tiles + blockIdx.x] = s;
  }
}

// counts of one token -> exclusive prefix along the tiles, and the total
__global__ void __launch_bounds__(32) embed_prefix_kernel(int* __restrict__ counts, int tiles, int* __restrict__ total) {
  const int v = blockIdx.x, lane = threadIdx.x;
  int* c = counts + (size_t)v * tiles;
  int run = 0;
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    const int x = t0 + lane < tiles ? c[t0 + lane] : 0;
    int s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, s, o);
      if (lane >= o) s += y;
    }
    if (t0 + lane < tiles) c[t0 + lane] = run + s - x;
    run += __shfl_sync(~0u, s, 31);
  }
  if (lane == 0) total[v] = run;
}

// Exclusive prefix over the tokens of f(total[v]), written to out[0..vocab];
// whole block, vocab <= 4 * kSortThreads.
template <typename F>
__device__ __forceinline__ void vocab_prefix(const int* __restrict__ total, int vocab, F f, int* out, int* scratch) {
  constexpr int PER = kMaxVocab / kSortThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x[PER], sum = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int v = threadIdx.x * PER + k;
    x[k] = v < vocab ? f(total[v]) : 0;
    sum += x[k];
  }
  int s = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, s, o);
    if (lane >= o) s += y;
  }
  if (lane == 31) scratch[warp] = s;
  __syncthreads();
  int before = s - sum;
  for (int w = 0; w < warp; ++w) before += scratch[w];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int v = threadIdx.x * PER + k;
    if (v <= vocab) out[v] = before;  // out[vocab] = the sum of all
    before += x[k];
  }
  if (threadIdx.x == kSortThreads - 1 && kMaxVocab == vocab) out[vocab] = before;
  __syncthreads();
}

// Writes each position to its place in token order.  A warp takes its part of
// the tile 32 tokens at a time: lanes that hold the same token find each
// other with a match, so equal tokens keep the order of their positions.
template <typename Tok>
__global__ void __launch_bounds__(kSortThreads)
embed_order_kernel(const Tok* __restrict__ tok, long long n, int vocab, int tile, int tiles,
                   const int* __restrict__ counts, const int* __restrict__ total, int* __restrict__ base_out,
                   int* __restrict__ piece_base, int* __restrict__ order) {
  extern __shared__ int hist[];  // [kSortWarps][vocab] next places, base [vocab + 1], scratch [kSortWarps]
  int* base = hist + kSortWarps * vocab;
  int* scratch = base + vocab + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * vocab; i += kSortThreads) hist[i] = 0;
  __syncthreads();
  const int span = tile / kSortWarps;
  const long long w0 = (long long)blockIdx.x * tile + (long long)warp * span;
  const long long w1 = w0 + span < n ? w0 + span : n;
  count_tile(tok, w0, w1, vocab, hist + warp * vocab);
  if (blockIdx.x == 0) {  // the pieces of each token, for the kernels that follow
    vocab_prefix(total, vocab, [](int c) { return (c + kPieceRows - 1) / kPieceRows; }, base, scratch);
    for (int v = threadIdx.x; v <= vocab; v += kSortThreads) piece_base[v] = base[v];
    __syncthreads();
  }
  vocab_prefix(total, vocab, [](int c) { return c; }, base, scratch);
  if (blockIdx.x == 0)
    for (int v = threadIdx.x; v <= vocab; v += kSortThreads) base_out[v] = base[v];
  for (int v = threadIdx.x; v < vocab; v += kSortThreads) {
    int at = base[v] + counts[(size_t)v * tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = hist[w * vocab + v];
      hist[w * vocab + v] = at;
      at += c;
    }
  }
  __syncthreads();
  int* next = hist + warp * vocab;
  for (long long i0 = w0; i0 < w1; i0 += 32) {
    const long long i = i0 + lane;
    const int v = i < w1 ? token_index(tok[i], vocab) : -1;
    const unsigned same = __match_any_sync(~0u, v);
    const int rank = __popc(same & ((1u << lane) - 1));
    int at = 0;
    if (v >= 0) at = next[v] + rank;
    __syncwarp();
    if (v >= 0 && rank == 0) next[v] = at + __popc(same);
    __syncwarp();
    if (v >= 0) order[at] = (int)i;
  }
}

// Sum of one piece: the block's threads form groups of `per_row` threads, one
// pack of N columns each; group g takes the piece's rows g, g + groups, ...
template <typename TG, int N>
__global__ void __launch_bounds__(kSumThreads)
embed_sum_kernel(const TG* __restrict__ dout, long long ld, int vocab, int d, int per_row,
                 const int* __restrict__ base, const int* __restrict__ piece_base, const int* __restrict__ order,
                 float* __restrict__ part) {
  __shared__ int s_tok, s_order[kPieceRows];
  __shared__ float s_sum[kSumThreads * N];
  const int p = blockIdx.x;
  if (p >= piece_base[vocab]) return;
  for (int v = threadIdx.x; v < vocab; v += kSumThreads)
    if (piece_base[v] <= p && p < piece_base[v + 1]) s_tok = v;
  __syncthreads();
  const int v = s_tok;
  const int first = base[v] + (p - piece_base[v]) * kPieceRows;
  const int rows = min(kPieceRows, base[v + 1] - first);
  for (int i = threadIdx.x; i < rows; i += kSumThreads) s_order[i] = order[first + i];
  __syncthreads();
  const int groups = kSumThreads / per_row;
  const int g = threadIdx.x / per_row, col = threadIdx.x - g * per_row;
  const int q = d / N;
  for (int c0 = 0; c0 < q; c0 += per_row) {
    const int c = c0 + col;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    if (g < groups && c < q) {
      const TG* col_ptr = dout + (size_t)c * N;
#pragma unroll 8
      for (int r = g; r < rows; r += groups) {
        const Pack<TG, N> x = *reinterpret_cast<const Pack<TG, N>*>(col_ptr + s_order[r] * ld);
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += to_f32(x.v[k]);
      }
    }
    if (c0) __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) s_sum[k * kSumThreads + threadIdx.x] = acc[k];
    __syncthreads();
    if (g == 0 && c < q) {
      for (int j = 1; j < groups; ++j)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += s_sum[k * kSumThreads + j * per_row + col];
#pragma unroll
      for (int k = 0; k < N; ++k) part[(size_t)p * d + c * N + k] = acc[k];
    }
  }
}

// dtable[v][c] = scale * the sum of the token's pieces, in order (fp64: one
// add per 512 rows): eight threads a column take contiguous runs of pieces.
template <typename TD>
__global__ void __launch_bounds__(256)
embed_join_kernel(const float* __restrict__ part, const int* __restrict__ piece_base, int d, float scale,
                  int accumulate, TD* __restrict__ dtable, long long ld) {
  __shared__ double s[8][32];
  const int v = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
  const int p0 = piece_base ? piece_base[v] : 0, p1 = piece_base ? piece_base[v + 1] : 0;
  const int run = (p1 - p0 + 7) / 8;
  const int a = p0 + g * run, b = min(p1, a + run);
  double sum = 0.0;
  if (c < d)
#pragma unroll 8
    for (int p = a; p < b; ++p) sum += (double)part[(size_t)p * d + c];
  s[g][threadIdx.x & 31] = sum;
  __syncthreads();
  if (g == 0 && c < d) {
    for (int j = 1; j < 8; ++j) sum += s[j][threadIdx.x];
    TD* out = dtable + v * ld + c;
    float r = (float)(sum * (double)scale);
    if (accumulate) r += to_f32(*out);
    *out = from_f32<TD>(r);
  }
}

template <typename TG, int N>
static void sum_run(const TG* dout, long long ld, int vocab, int d, const GradPlan& p, int* w, cudaStream_t st) {
  const int q = d / N;
  const int per_row = q < kSumThreads ? q : kSumThreads;
  embed_sum_kernel<TG, N><<<(unsigned)p.pieces, kSumThreads, 0, st>>>(
      dout, ld, vocab, d, per_row, w + p.base, w + p.piece_base, w + p.order, reinterpret_cast<float*>(w + p.part));
}

cudaError_t launch_embed_grad(const void* tokens, int tok_t, long long n, const void* dout, int dout_t,
                              long long ld_dout, int vocab, int d, float scale, bool accumulate, void* dtable,
                              int dtable_t, long long ld_dtable, void* ws, cudaStream_t st) {
  int* w = static_cast<int*>(ws);
  const GradPlan p = grad_plan(n > 0 ? n : 1, vocab, d);
  cudaError_t e = cudaSuccess;
  if (n > 0) {
    e = with_token(tok_t, [&](auto tk) {
      using Tok = decltype(tk);
      const Tok* t = static_cast<const Tok*>(tokens);
      const size_t hist_bytes = (size_t)kSortWarps * vocab * 4;
      embed_count_kernel<Tok><<<p.tiles, kSortThreads, hist_bytes, st>>>(t, n, vocab, p.tile, p.tiles, w + p.counts);
      embed_prefix_kernel<<<vocab, 32, 0, st>>>(w + p.counts, p.tiles, w + p.total);
      embed_order_kernel<Tok><<<p.tiles, kSortThreads, hist_bytes + (vocab + 1 + kSortWarps) * 4, st>>>(
          t, n, vocab, p.tile, p.tiles, w + p.counts, w + p.total, w + p.base, w + p.piece_base, w + p.order);
      return cudaGetLastError();
    });
    if (e != cudaSuccess) return e;
    e = with_type(dout_t, [&](auto tg) {
      using TG = decltype(tg);
      constexpr int N = 16 / sizeof(TG);
      const TG* x = static_cast<const TG*>(dout);
      if (d % N == 0 && ld_dout % N == 0 && aligned_to(x, 16)) sum_run<TG, N>(x, ld_dout, vocab, d, p, w, st);
      else sum_run<TG, 1>(x, ld_dout, vocab, d, p, w, st);
      return cudaGetLastError();
    });
    if (e != cudaSuccess) return e;
  } else if (accumulate) {
    return cudaSuccess;
  }
  return with_type(dtable_t, [&](auto td) {
    using TD = decltype(td);
    embed_join_kernel<TD><<<dim3((d + 31) / 32, vocab), 256, 0, st>>>(
        n > 0 ? reinterpret_cast<const float*>(w + p.part) : nullptr, n > 0 ? w + p.piece_base : nullptr, d, scale,
        accumulate ? 1 : 0, static_cast<TD*>(dtable), ld_dtable);
    return cudaGetLastError();
  });
}

}  // namespace boa
