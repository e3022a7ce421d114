// loss.cu -- next-token cross entropy and its gradient in one pass.
//
//   p = softmax(s x),  s = 1 / temperature
//   loss = -log p[target]        dx = w s (p - onehot(target))
//
// One warp holds a row (at most 1024 logits) in registers: the logits are
// read once, the maximum, the sum and the gradient come from the same
// registers, and the gradient is written once, so a row costs its bytes in
// and its bytes out.  The maximum is subtracted before scaling, so a mask of
// the type's lowest value underflows to p = 0 instead of overflowing.
#include "kernels.cuh"
#include "ptx.cuh"
#include "train_ops.cuh"

namespace boa {

constexpr int kLossThreads = 256;

// A lane holds C packs of N logits, pack k at element (k * 32 + lane) * N.
template <typename T_, typename Tok, int N, int C>
__global__ void __launch_bounds__(kLossThreads)
token_loss_kernel(const T_* logits, long long ld, long long rows, int vocab, const Tok* __restrict__ targets,
                  float inv_t, const float* __restrict__ dloss, float grad_scale, float* __restrict__ loss,
                  T_* grad, long long ld_grad) {
  const long long row = (long long)blockIdx.x * (kLossThreads / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  const int target = token_index(targets[row], vocab);
  if (target < 0) {  // a row that pads the batch: its logits are not read
    if (loss && lane == 0) loss[row] = 0.f;
    if (grad) {
      Pack<T_, N> zero;
#pragma unroll
      for (int j = 0; j < N; ++j) zero.v[j] = from_f32<T_>(0.f);
      for (int c = lane * N; c < vocab; c += 32 * N) *reinterpret_cast<Pack<T_, N>*>(grad + row * ld_grad + c) = zero;
    }
    return;
  }
  const T_* x = logits + row * ld;
  float v[C * N];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = (k * 32 + lane) * N;
    if (c < vocab) {
      const Pack<T_, N> p = *reinterpret_cast<const Pack<T_, N>*>(x + c);
#pragma unroll
      for (int j = 0; j < N; ++j) v[k * N + j] = to_f32(p.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[k * N + j] = -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) m = fmaxf(m, v[k * N + j]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  // every logit -inf: no distribution is left, all weights come out 0 (not NaN)
  if (m == -INFINITY) m = 0.f;
  float sum = 0.f;
  float at = 0.f;  // s (x[target] - m)
#pragma unroll
  for (int k = 0; k < C; ++k)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float y = (v[k * N + j] - m) * inv_t;
      if ((k * 32 + lane) * N + j == target) at = y;
      v[k * N + j] = __expf(y);
      sum += v[k * N + j];
    }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    sum += __shfl_xor_sync(~0u, sum, o);
  }
  if (loss) {
    const int owner = target / N % 32;
    at = __shfl_sync(~0u, at, owner);
    if (lane == 0) loss[row] = sum == 0.f ? INFINITY : logf(sum) - at;
  }
  if (grad) {
    const float w = (dloss ? dloss[row] * grad_scale : grad_scale) * inv_t;
    const float r = sum == 0.f ? 0.f : w / sum;
    const float hit = sum == 0.f ? 0.f : w;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int c = (k * 32 + lane) * N;
      if (c >= vocab) continue;
      Pack<T_, N> p;
#pragma unroll
      for (int j = 0; j < N; ++j) p.v[j] = from_f32<T_>(v[k * N + j] * r - (c + j == target ? hit : 0.f));
      *reinterpret_cast<Pack<T_, N>*>(grad + row * ld_grad + c) = p;
    }
  }
}

cudaError_t launch_token_loss(const void* logits, int type, long long ld, long long rows, int vocab,
                              const void* targets, int tok_t, float inv_t, const float* dloss, float grad_scale,
                              float* loss, void* dlogits, long long ld_grad, cudaStream_t st) {
  const long long blocks = (rows + kLossThreads / 32 - 1) / (kLossThreads / 32);
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  return with_type(type, [&](auto ty) {
    return with_token(tok_t, [&](auto tk) {
      using E = decltype(ty);
      using Tok = decltype(tk);
      constexpr int W = 16 / sizeof(E);
      const bool wide = vocab % W == 0 && ld % W == 0 && aligned_to(logits, 16) &&
                        (!dlogits || (ld_grad % W == 0 && aligned_to(dlogits, 16)));
      auto go = [&](auto kernel) {
        kernel<<<(unsigned)blocks, kLossThreads, 0, st>>>(static_cast<const E*>(logits), ld, rows, vocab,
                                                          static_cast<const Tok*>(targets), inv_t, dloss, grad_scale,
                                                          loss, static_cast<E*>(dlogits), ld_grad);
        return cudaGetLastError();
      };
      if (wide) {
        if (vocab <= 256) return go(token_loss_kernel<E, Tok, W, 256 / (32 * W)>);
        return go(token_loss_kernel<E, Tok, W, kMaxVocab / (32 * W)>);
      }
      if (vocab <= 256) return go(token_loss_kernel<E, Tok, 1, 8>);
      return go(token_loss_kernel<E, Tok, 1, kMaxVocab / 32>);
    });
  });
}

}  // namespace boa
