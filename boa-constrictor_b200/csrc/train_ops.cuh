// train_ops.cuh -- launchers and element types of the operators a predictor
// is trained and stepped with (embedding, minGRU recurrence, next-token loss
// and their gradients).  They work on caller-owned device buffers of several
// element types; all arithmetic is fp32 or wider, and a result is rounded
// once, to nearest, when it is stored.
#pragma once
#include <atomic>
#include <cstdint>
#include <initializer_list>
#include <type_traits>
#include <utility>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace boa {

// element types, in the order of BOA_F32 / BOA_F16 / BOA_BF16
enum : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };
// token types, in the order of BOA_TOK_U8 / BOA_TOK_I32 / BOA_TOK_I64
enum : int { TOK_U8 = 0, TOK_I32 = 1, TOK_I64 = 2 };

constexpr int kMaxVocab = 1024;   // the coder's largest alphabet
constexpr int kMaxWidth = 65536;  // widest row; keeps in-block index products below 2^32

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements, moved in pieces of up to 16 bytes.
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  T v[N];
};

// A pack as fp32 and back.  Pairs of 16 bits are taken as the 32-bit words that
// they are: taken as halves they cost twice the instructions.
template <typename T, int N>
__device__ __forceinline__ void widen_pack(const Pack<T, N>& p, float (&r)[N]) {
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&p);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        r[2 * k] = __uint_as_float(w[k] << 16);
        r[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
      } else {
        __half2 h;
        *reinterpret_cast<uint32_t*>(&h) = w[k];
        const float2 f = __half22float2(h);
        r[2 * k] = f.x;
        r[2 * k + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = to_f32(p.v[k]);
  }
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> narrow_pack(const float (&x)[N]) {
  Pack<T, N> p;
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&r);
      } else {
        const __half2 r = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&r);
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) p.v[k] = from_f32<T>(x[k]);
  }
  return p;
}
// A pack that is read once, or written and not read again here.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_once(const T* p) {
  if constexpr (N * sizeof(T) == 16) {
    const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p));
    return *reinterpret_cast<const Pack<T, N>*>(&w);
  } else {
    return *reinterpret_cast<const Pack<T, N>*>(p);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_once(T* p, const Pack<T, N>& x) {
  if constexpr (N * sizeof(T) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&x));
  else *reinterpret_cast<Pack<T, N>*>(p) = x;
}
// 2^x and 1 / x to about one step of fp32; results below 2^-126 are 0
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
constexpr float kLog2e = 1.44269504f;

// A token as an index, or -1 when it lies outside [0, vocab): such a token
// pads a batch, and no address is formed from it.
template <typename Tok>
__device__ __forceinline__ int token_index(Tok t, int vocab) {
  const long long x = (long long)t;
  return x >= 0 && x < vocab ? (int)x : -1;
}

// Calls f with a value of the element type `t` (f(float{}), f(__half{}) ...).
template <typename F>
cudaError_t with_type(int t, F&& f) {
  switch (t) {
    case DT_F32: return f(float{});
    case DT_F16: return f(__half{});
    case DT_BF16: return f(__nv_bfloat16{});
  }
  return cudaErrorInvalidValue;
}
template <typename F>
cudaError_t with_token(int t, F&& f) {
  switch (t) {
    case TOK_U8: return f(uint8_t{});
    case TOK_I32: return f(int32_t{});
    case TOK_I64: return f(int64_t{});
  }
  return cudaErrorInvalidValue;
}
inline int type_bytes(int t) { return t == DT_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

// out[i] = scale * table[tokens[i]]; a token outside [0, vocab) gives a zero row
cudaError_t launch_embed(const void* tokens, int tok_t, long long n, const void* table, int table_t,
                         long long ld_table, int vocab, int d, float scale, void* out, int out_t, long long ld_out,
                         cudaStream_t st);

// dtable[v] (+)= scale * sum over i with tokens[i] == v of dout[i]
size_t embed_grad_workspace(long long n, int vocab, int d);
cudaError_t launch_embed_grad(const void* tokens, int tok_t, long long n, const void* dout, int dout_t,
                              long long ld_dout, int vocab, int d, float scale, bool accumulate, void* dtable,
                              int dtable_t, long long ld_dtable, void* ws, cudaStream_t st);

// Rows of a [B][T][width] tensor: element (b, t, c) is at b * chunk + t * row + c.
struct RowStrides {
  long long row, chunk;
};

// minGRU over T positions per chunk; see recur.cu
size_t mingru_states_floats(int B, int T, int d);
cudaError_t launch_mingru_scan(const void* zh, int type, RowStrides zs, int B, int T, int d, const int* lengths,
                               const float* h0, void* h, RowStrides hs, float* h_last, float* states,
                               cudaStream_t st);
cudaError_t launch_mingru_scan_grad(const void* zh, int type, RowStrides zs, int B, int T, int d, const int* lengths,
                                    const float* states, const void* dh, RowStrides dhs, const float* dh_last,
                                    void* dzh, RowStrides dzs, float* dh0, cudaStream_t st);

// What the walk's exchange gives when one of a cluster's two blocks falls silent: [steps][128], see recur.cu
cudaError_t launch_walk_selftest(int steps, int silent, uint64_t limit_ns, float* out, cudaStream_t st);

// Next-token cross entropy per row and its gradient; see loss.cu
cudaError_t launch_token_loss(const void* logits, int type, long long ld, long long rows, int vocab,
                              const void* targets, int tok_t, float inv_t, const float* dloss, float grad_scale,
                              float* loss, void* dlogits, long long ld_grad, cudaStream_t st);

}  // namespace boa
