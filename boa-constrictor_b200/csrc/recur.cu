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
#include "kernels.cuh"
#include "ptx.cuh"
#include "train_ops.cuh"

namespace boa {

constexpr int kSpan = 128;  // positions between two saved states

struct Cell {
  float a, z, c;
};
__device__ __forceinline__ Cell mingru_cell(float zl, float hr) {
  Cell r;
  const float e = __expf(-fabsf(zl)), i = __fdividef(1.f, 1.f + e);
  const float small = e * i;  // the smaller of z and 1 - z, without cancellation
  r.z = zl >= 0.f ? i : small;
  r.a = zl >= 0.f ? small : i;
  if (zl != zl) r.z = r.a = zl;
  r.c = hr >= 0.f ? hr + 0.5f : __fdividef(1.f, 1.f + __expf(-hr));
  return r;
}

size_t mingru_states_floats(int B, int T, int d) { return (size_t)((T + kSpan - 1) / kSpan) * B * d; }
size_t mingru_workspace(int, int, int) { return 0; }

// One thread per chain (chunk b, channel c), position after position.
template <typename T_>
__global__ void __launch_bounds__(256)
mingru_scan_kernel(const T_* __restrict__ zh, RowStrides zs, int B, int T, int d, const int* __restrict__ lengths,
                   const float* h0, T_* __restrict__ h, RowStrides hs, float* h_last, float* __restrict__ states) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x, chains = (long long)B * d;
  if (i >= chains) return;
  const int b = (int)(i / d), c = (int)(i - (long long)b * d);
  const int len = lengths ? min(max(lengths[b], 0), T) : T;
  float s = h0 ? h0[i] : 0.f;
  const T_* x = zh + b * zs.chunk + c;
  T_* o = h + b * hs.chunk + c;
  for (int t = 0; t < T; ++t) {
    if (states && t % kSpan == 0) states[(t / kSpan) * chains + i] = s;
    if (t < len) {
      const Cell k = mingru_cell(to_f32(x[t * zs.row]), to_f32(x[t * zs.row + d]));
      s = k.a * s + k.z * k.c;
      o[t * hs.row] = from_f32<T_>(s);
    } else {
      o[t * hs.row] = from_f32<T_>(0.f);
    }
  }
  if (h_last) h_last[i] = s;
}

template <typename T_>
__global__ void __launch_bounds__(256)
mingru_scan_grad_kernel(const T_* __restrict__ zh, RowStrides zs, int B, int T, int d, const int* __restrict__ lengths,
                        const float* __restrict__ states, const T_* __restrict__ dh, RowStrides dhs,
                        const float* __restrict__ dh_last, T_* __restrict__ dzh, RowStrides dzs,
                        float* __restrict__ dh0) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x, chains = (long long)B * d;
  if (i >= chains) return;
  const int b = (int)(i / d), c = (int)(i - (long long)b * d);
  const int len = lengths ? min(max(lengths[b], 0), T) : T;
  float g = dh_last ? dh_last[i] : 0.f;
  const T_* x = zh + b * zs.chunk + c;
  const T_* u = dh + b * dhs.chunk + c;
  T_* o = dzh + b * dzs.chunk + c;
  float before[kSpan];
  for (int k = T > 0 ? (T - 1) / kSpan : -1; k >= 0; --k) {
    float s = states[k * chains + i];
    const int t0 = k * kSpan, n = min(kSpan, T - t0);
    for (int j = 0; j < n && t0 + j < len; ++j) {
      const long long t = t0 + j;
      const Cell q = mingru_cell(to_f32(x[t * zs.row]), to_f32(x[t * zs.row + d]));
      before[j] = s;
      s = q.a * s + q.z * q.c;
    }
    for (int j = n - 1; j >= 0; --j) {
      const long long t = t0 + j;
      float dz = 0.f, dr = 0.f;
      if (t < len) {
        const float hr = to_f32(x[t * zs.row + d]);
        const Cell q = mingru_cell(to_f32(x[t * zs.row]), hr);
        g += to_f32(u[t * dhs.row]);
        dz = g * q.z * q.a * (q.c - before[j]);
        dr = g * q.z * (hr >= 0.f ? 1.f : q.c * (1.f - q.c));
        g *= q.a;
      }
      o[t * dzs.row] = from_f32<T_>(dz);
      o[t * dzs.row + d] = from_f32<T_>(dr);
    }
  }
  if (dh0) dh0[i] = g;
}

cudaError_t launch_mingru_scan(const void* zh, int type, RowStrides zs, int B, int T, int d, const int* lengths,
                               const float* h0, void* h, RowStrides hs, float* h_last, float* states, void*,
                               cudaStream_t st) {
  const long long blocks = ((long long)B * d + 255) / 256;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  return with_type(type, [&](auto t) {
    using E = decltype(t);
    mingru_scan_kernel<E><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const E*>(zh), zs, B, T, d, lengths, h0,
                                                            static_cast<E*>(h), hs, h_last, states);
    return cudaGetLastError();
  });
}

cudaError_t launch_mingru_scan_grad(const void* zh, int type, RowStrides zs, int B, int T, int d, const int* lengths,
                                    const float* states, const void* dh, RowStrides dhs, const float* dh_last,
                                    void* dzh, RowStrides dzs, float* dh0, void*, cudaStream_t st) {
  const long long blocks = ((long long)B * d + 255) / 256;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  return with_type(type, [&](auto t) {
    using E = decltype(t);
    mingru_scan_grad_kernel<E><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const E*>(zh), zs, B, T, d, lengths,
                                                                 states, static_cast<const E*>(dh), dhs, dh_last,
                                                                 static_cast<E*>(dzh), dzs, dh0);
    return cudaGetLastError();
  });
}

}  // namespace boa
