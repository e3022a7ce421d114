// loss.cu -- next-token cross entropy and its gradient in one pass.
//
//   p = softmax(s x),  s = 1 / temperature
//   loss = -log p[target]        dx = w s (p - onehot(target))
//
// A few lanes hold a row (at most 1024 logits) in registers: the logits are
// read once, the maximum, the sum and the gradient come from the same
// registers, and the gradient is written once, so a row costs its bytes in
// and its bytes out.  The maximum is subtracted before scaling, so a mask of
// the type's lowest value underflows to p = 0 instead of overflowing.
//
// Measured on a B200, loss and gradient: 1M x 256 fp32 319 us (the rate of a copy),
// bf16 172 us (0.95 of it), 262144 x 1024 bf16 168 us (0.97).  Eight lanes a row
// of up to 256 logits keep more rows in flight and reduce in three exchanges
// (32 lanes: 376 us and 258 us).  The target's logit is read by the lane that
// forms the loss, before the exchanges (by all lanes: 200 us for 1M x 256 bf16).
#include <cfloat>

#include "train_ops.cuh"

namespace boa {

constexpr int kLossThreads = 128;

// L lanes take a row; a lane holds C packs of N logits, pack k at element
// (k * L + lane) * N.
template <typename T_, typename Tok, int N, int C, int L>
__global__ void __launch_bounds__(kLossThreads)
token_loss_kernel(const T_* logits, long long ld, long long rows, int vocab, const Tok* __restrict__ targets,
                  float inv_t, const float* __restrict__ dloss, float grad_scale, float* __restrict__ loss,
                  T_* grad, long long ld_grad) {
  const long long row = (long long)blockIdx.x * (kLossThreads / L) + threadIdx.x / L;
  if (row >= rows) return;
  const int lane = threadIdx.x % L;
  const unsigned lanes = L == 32 ? ~0u : ((1u << L) - 1) << (threadIdx.x & 31 & ~(L - 1));
  const int target = token_index(targets[row], vocab);
  T_* g = grad + row * ld_grad;
  if (target < 0) {  // a row that pads the batch: its logits are not read
    if (loss && lane == 0) loss[row] = 0.f;
    if (grad) {
      const float zero[N] = {};
      for (int c = lane * N; c < vocab; c += L * N) store_once<T_, N>(g + c, narrow_pack<T_>(zero));
    }
    return;
  }
  const T_* x = logits + row * ld;
  const float hit = lane == 0 ? to_f32(x[target]) : 0.f;
  float v[C][N];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = (k * L + lane) * N;
    if (c < vocab) {
      widen_pack(load_once<T_, N>(x + c), v[k]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[k][j] = -INFINITY;
    }
  }
#pragma unroll
  for (int k = 0; k < C; ++k)
#pragma unroll
    for (int j = 0; j < N; ++j) m = fmaxf(m, v[k][j]);
#pragma unroll
  for (int o = L / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(lanes, m, o));
  // every logit -inf: no distribution is left, all weights come out 0 (not NaN)
  if (m == -INFINITY) m = 0.f;
  // cut off where the product passes fp32: from there on any two logits whose difference is a normal number are apart
  const float scale = fminf(inv_t * kLog2e, FLT_MAX);
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < C; ++k)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v[k][j] = ex2_fast((v[k][j] - m) * scale);
      sum += v[k][j];
    }
#pragma unroll
  for (int o = L / 2; o; o >>= 1) sum += __shfl_xor_sync(lanes, sum, o);
  if (loss && lane == 0) loss[row] = sum == 0.f ? INFINITY : logf(sum) - (hit - m) * inv_t;
  if (grad) {
    __syncwarp(lanes);  // in place: all logits, the target's too, are read before a gradient is written over them
    const float w = sum == 0.f ? 0.f : (dloss ? dloss[row] * grad_scale : grad_scale) * inv_t;
    const float r = sum == 0.f ? 0.f : w / sum;
    const int pack = target / N, own = pack % L == lane ? pack / L : -1;  // the pack that holds the target
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int c = (k * L + lane) * N;
      if (c >= vocab) continue;
#pragma unroll
      for (int j = 0; j < N; ++j) v[k][j] *= r;
      if (k == own) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[k][j] -= j == target % N ? w : 0.f;
      }
      store_once<T_, N>(g + c, narrow_pack<T_>(v[k]));
    }
  }
}

cudaError_t launch_token_loss(const void* logits, int type, long long ld, long long rows, int vocab,
                              const void* targets, int tok_t, float inv_t, const float* dloss, float grad_scale,
                              float* loss, void* dlogits, long long ld_grad, cudaStream_t st) {
  return with_type(type, [&](auto ty) {
    return with_token(tok_t, [&](auto tk) {
      using E = decltype(ty);
      using Tok = decltype(tk);
      constexpr int W = 16 / sizeof(E);
      const bool wide = vocab % W == 0 && ld % W == 0 && aligned_to(logits, 16) &&
                        (!dlogits || (ld_grad % W == 0 && aligned_to(dlogits, 16)));
      auto go = [&](auto kernel, int lanes) {
        const long long blocks = (rows + kLossThreads / lanes - 1) / (kLossThreads / lanes);
        kernel<<<(unsigned)blocks, kLossThreads, 0, st>>>(static_cast<const E*>(logits), ld, rows, vocab,
                                                          static_cast<const Tok*>(targets), inv_t, dloss, grad_scale,
                                                          loss, static_cast<E*>(dlogits), ld_grad);
        return cudaGetLastError();
      };
      if (wide && vocab <= 256) return go(token_loss_kernel<E, Tok, W, 256 / (8 * W), 8>, 8);
      if (wide) return go(token_loss_kernel<E, Tok, W, kMaxVocab / (32 * W), 32>, 32);
      if (vocab <= 256) return go(token_loss_kernel<E, Tok, 1, 256 / 32, 32>, 32);
      return go(token_loss_kernel<E, Tok, 1, kMaxVocab / 32, 32>, 32);
    });
  });
}

}  // namespace boa
