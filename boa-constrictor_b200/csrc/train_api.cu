// train_api.cu -- C entry points of the operators a predictor is trained and
// stepped with: handle-free, on caller-owned device buffers and the caller's
// stream, like the step-wise coder (coder_api.cu).  Arguments are checked
// here; nothing is allocated and nothing is synchronised, so every call can be
// captured into a CUDA graph (but for the walk's self-test).
#include <cmath>

#include "train_ops.cuh"

namespace {

// Checks shared by the entry points.  The message goes to a buffer of the
// calling thread: these calls have no handle to hold it, and several threads
// may make them at once.
int train_fail(int code, const char* fn, const char* what) {
  std::snprintf(t_call_error, sizeof t_call_error, "%s: %s", fn, what);
  return code;
}
// Runs a launcher.  An error that an earlier call left behind is not this
// call's, and this call's is not left to a later one: a launch's outcome is
// read back from the thread's last error.  A launch into a stream that is not
// of the current device fails as an invalid handle.  Asking for the stream's
// device beforehand is no choice: the query ends a stream capture.
template <typename F>
int train_launch(const char* fn, F&& launch) {
  cudaGetLastError();
  const cudaError_t e = launch();
  if (e == cudaSuccess) return BOA_OK;
  cudaGetLastError();
  if (e == cudaErrorInvalidResourceHandle)
    return train_fail(BOA_E_INVALID, fn, "the stream belongs to another device");
  return train_fail(BOA_E_CUDA, fn, cudaGetErrorString(e));
}
bool type_ok(int t) { return t == BOA_F32 || t == BOA_F16 || t == BOA_BF16; }
bool token_ok(int t) { return t == BOA_TOK_U8 || t == BOA_TOK_I32 || t == BOA_TOK_I64; }
bool elem_aligned(const void* p, int type) { return boa::aligned_to(p, boa::type_bytes(type)); }
bool token_aligned(const void* p, int t) {
  return boa::aligned_to(p, t == BOA_TOK_U8 ? 1 : t == BOA_TOK_I32 ? 4 : 8);
}
// Rows are below 4 GiB apart, and b * chunk stays within 63 bits.  Rows that are read may
// coincide (an expanded gradient has strides of 0); rows that are written may
// not, with the chunks outside the positions or inside.
bool in_strides_ok(int64_t row, int64_t chunk, int B, int T, int type) {
  return row >= 0 && row < (1ll << 40) && (T <= 1 || row * boa::type_bytes(type) <= 0xffffffffll) && chunk >= 0 &&
         chunk <= ((int64_t)1 << 60) / (B + 1ll);
}
bool out_strides_ok(int64_t row, int64_t chunk, int B, int T, int width, int type) {
  if (!in_strides_ok(row, chunk, B, T, type)) return false;
  if (T == 0) return true;
  if (B <= 1 || T <= 1) return (T <= 1 || row >= width) && (B <= 1 || chunk >= width);
  return (row >= width && chunk >= (T - 1) * row + width) || (chunk >= width && row >= (B - 1) * chunk + width);
}

}  // namespace

#define BOA_REQUIRE(cond, what) \
  if (!(cond)) return train_fail(BOA_E_INVALID, __func__, what)

extern "C" {

int boa_embed(const void* d_tokens, int token_type, int64_t n, const void* d_table, int table_type, int64_t ld_table,
              int vocab, int d, float scale, void* d_out, int out_type, int64_t ld_out, void* stream) {
  BOA_REQUIRE(token_ok(token_type) && type_ok(table_type) && type_ok(out_type), "unknown element or token type");
  BOA_REQUIRE(n >= 0 && n <= 0x7fffffff, "n must be 0 .. 2^31 - 1");
  BOA_REQUIRE(vocab >= 1 && vocab <= boa::kMaxVocab, "vocab must be 1 .. 1024");
  BOA_REQUIRE(d >= 1 && d <= boa::kMaxWidth, "d must be 1 .. 65536");
  BOA_REQUIRE(ld_table >= d && ld_out >= d && ld_table < (1ll << 31) && ld_out < (1ll << 31),
              "ld_table and ld_out must be d .. 2^31 - 1");
  if (n == 0) return BOA_OK;
  BOA_REQUIRE(d_tokens && d_table && d_out, "null buffer");
  BOA_REQUIRE(token_aligned(d_tokens, token_type) && elem_aligned(d_table, table_type) &&
                  elem_aligned(d_out, out_type),
              "a buffer is not aligned to its element");
  return train_launch(__func__, [&] {
    return boa::launch_embed(d_tokens, token_type, n, d_table, table_type, ld_table, vocab, d, scale, d_out, out_type,
                             ld_out, (cudaStream_t)stream);
  });
}

size_t boa_embed_backward_workspace(int64_t n, int vocab, int d) {
  if (n < 0 || n > 0x7fffffff || vocab < 1 || vocab > boa::kMaxVocab || d < 1 || d > boa::kMaxWidth) return 0;
  return boa::embed_grad_workspace(n, vocab, d);
}

int boa_embed_backward(const void* d_tokens, int token_type, int64_t n, const void* d_dout, int dout_type,
                       int64_t ld_dout, int vocab, int d, float scale, int accumulate, void* d_dtable,
                       int dtable_type, int64_t ld_dtable, void* d_workspace, size_t workspace_bytes, void* stream) {
  BOA_REQUIRE(token_ok(token_type) && type_ok(dout_type) && type_ok(dtable_type), "unknown element or token type");
  BOA_REQUIRE(n >= 0 && n <= 0x7fffffff, "n must be 0 .. 2^31 - 1");
  BOA_REQUIRE(vocab >= 1 && vocab <= boa::kMaxVocab, "vocab must be 1 .. 1024");
  BOA_REQUIRE(d >= 1 && d <= boa::kMaxWidth, "d must be 1 .. 65536");
  BOA_REQUIRE(ld_dout >= d && ld_dtable >= d && ld_dout < (1ll << 31) && ld_dtable < (1ll << 31),
              "ld_dout and ld_dtable must be d .. 2^31 - 1");
  BOA_REQUIRE(d_dtable && elem_aligned(d_dtable, dtable_type), "d_dtable is null or not aligned to its element");
  if (n > 0) {
    BOA_REQUIRE(d_tokens && d_dout, "null buffer");
    BOA_REQUIRE(token_aligned(d_tokens, token_type) && elem_aligned(d_dout, dout_type),
                "a buffer is not aligned to its element");
    const size_t need = boa::embed_grad_workspace(n, vocab, d);
    BOA_REQUIRE(need == 0 || (d_workspace && boa::aligned_to(d_workspace, 16) && workspace_bytes >= need),
                "the workspace is null, not aligned to 16 bytes or below boa_embed_backward_workspace");
  }
  return train_launch(__func__, [&] {
    return boa::launch_embed_grad(d_tokens, token_type, n, d_dout, dout_type, ld_dout, vocab, d, scale, accumulate != 0,
                                  d_dtable, dtable_type, ld_dtable, d_workspace, (cudaStream_t)stream);
  });
}

uint64_t boa_mingru_states_floats(int n_chunks, int T, int d) {
  if (n_chunks < 0 || T < 0 || d < 1 || d > boa::kMaxWidth) return 0;
  return boa::mingru_states_floats(n_chunks, T, d);
}
int boa_mingru_scan(const void* d_zh, int type, int64_t zh_row, int64_t zh_chunk, int n_chunks, int T, int d,
                    const int32_t* d_lengths, const float* d_h0, void* d_h, int64_t h_row, int64_t h_chunk,
                    float* d_h_last, float* d_states, void* stream) {
  BOA_REQUIRE(type_ok(type), "unknown element type");
  BOA_REQUIRE(n_chunks >= 0 && T >= 0 && T <= 1 << 30, "n_chunks must not be negative, T must be 0 .. 2^30");
  BOA_REQUIRE(d >= 1 && d <= boa::kMaxWidth, "d must be 1 .. 65536");
  BOA_REQUIRE((int64_t)n_chunks * d <= 0x7fffffff, "n_chunks * d must be at most 2^31 - 1");
  BOA_REQUIRE(in_strides_ok(zh_row, zh_chunk, n_chunks, T, type) &&
                  out_strides_ok(h_row, h_chunk, n_chunks, T, d, type),
              "a stride is negative or too large, or the rows of h overlap");
  if (n_chunks == 0) return BOA_OK;
  BOA_REQUIRE(T == 0 || (d_zh && d_h), "null buffer");
  BOA_REQUIRE(elem_aligned(d_zh, type) && elem_aligned(d_h, type) && boa::aligned_to(d_lengths, 4) &&
                  boa::aligned_to(d_h0, 4) && boa::aligned_to(d_h_last, 4) && boa::aligned_to(d_states, 4),
              "a buffer is not aligned to its element");
  return train_launch(__func__, [&] {
    return boa::launch_mingru_scan(d_zh, type, {zh_row, zh_chunk}, n_chunks, T, d, d_lengths, d_h0, d_h, {h_row,
                                   h_chunk}, d_h_last, d_states, (cudaStream_t)stream);
  });
}

int boa_mingru_scan_backward(const void* d_zh, int type, int64_t zh_row, int64_t zh_chunk, int n_chunks, int T, int d,
                             const int32_t* d_lengths, const float* d_states, const void* d_dh, int64_t dh_row,
                             int64_t dh_chunk, const float* d_dh_last, void* d_dzh, int64_t dzh_row,
                             int64_t dzh_chunk, float* d_dh0, void* stream) {
  BOA_REQUIRE(type_ok(type), "unknown element type");
  BOA_REQUIRE(n_chunks >= 0 && T >= 0 && T <= 1 << 30, "n_chunks must not be negative, T must be 0 .. 2^30");
  BOA_REQUIRE(d >= 1 && d <= boa::kMaxWidth, "d must be 1 .. 65536");
  BOA_REQUIRE((int64_t)n_chunks * d <= 0x7fffffff, "n_chunks * d must be at most 2^31 - 1");
  BOA_REQUIRE(in_strides_ok(zh_row, zh_chunk, n_chunks, T, type) &&
                  in_strides_ok(dh_row, dh_chunk, n_chunks, T, type) &&
                  out_strides_ok(dzh_row, dzh_chunk, n_chunks, T, 2 * d, type),
              "a stride is negative or too large, or the rows of dzh overlap");
  if (n_chunks == 0) return BOA_OK;
  BOA_REQUIRE(T == 0 || (d_zh && d_states && d_dh && d_dzh), "null buffer");
  BOA_REQUIRE(elem_aligned(d_zh, type) && elem_aligned(d_dh, type) && elem_aligned(d_dzh, type) &&
                  boa::aligned_to(d_lengths, 4) && boa::aligned_to(d_states, 4) && boa::aligned_to(d_dh_last, 4) &&
                  boa::aligned_to(d_dh0, 4),
              "a buffer is not aligned to its element");
  return train_launch(__func__, [&] {
    return boa::launch_mingru_scan_grad(d_zh, type, {zh_row, zh_chunk}, n_chunks, T, d, d_lengths, d_states, d_dh,
                                        {dh_row, dh_chunk}, d_dh_last, d_dzh, {dzh_row, dzh_chunk}, d_dh0,
                                        (cudaStream_t)stream);
  });
}

int boa_selftest_walk_timeout(int device, int n_steps, int silent_from, uint32_t limit_us, float* out) {
  int n_dev = 0;
  if (cudaGetDeviceCount(&n_dev) != cudaSuccess) {
    cudaGetLastError();
    n_dev = 0;
  }
  BOA_REQUIRE(device >= 0 && device < n_dev, "no such CUDA device");
  BOA_REQUIRE(n_steps >= 1 && n_steps <= 64 && silent_from >= 0, "n_steps must be 1 .. 64, silent_from not negative");
  BOA_REQUIRE(limit_us >= 1 && limit_us <= 1000000u, "limit_us must be in [1, 1e6]");
  BOA_REQUIRE(out, "null buffer");
  DeviceGuard dev(device);
  return train_launch(__func__, [&] {
    const size_t bytes = (size_t)n_steps * 128 * sizeof(float);
    float* d_out = nullptr;
    cudaError_t e = cudaMalloc(&d_out, bytes);
    if (e != cudaSuccess) return e;
    e = boa::launch_walk_selftest(n_steps, silent_from, limit_us * 1000ull, d_out, nullptr);
    if (e == cudaSuccess) e = cudaMemcpy(out, d_out, bytes, cudaMemcpyDeviceToHost);
    cudaFree(d_out);
    return e;
  });
}

int boa_token_loss(const void* d_logits, int type, int64_t ld, int64_t n_rows, int vocab, const void* d_targets,
                   int token_type, float inv_temperature, const float* d_dloss, float grad_scale, float* d_loss,
                   void* d_dlogits, int64_t ld_dlogits, void* stream) {
  BOA_REQUIRE(type_ok(type) && token_ok(token_type), "unknown element or token type");
  BOA_REQUIRE(n_rows >= 0 && n_rows <= 0x7fffffff, "n_rows must be 0 .. 2^31 - 1");
  BOA_REQUIRE(vocab >= 1 && vocab <= boa::kMaxVocab, "vocab must be 1 .. 1024");
  BOA_REQUIRE(ld >= vocab && ld < (1ll << 31), "ld must be vocab .. 2^31 - 1");
  BOA_REQUIRE(!d_dlogits || (ld_dlogits >= vocab && ld_dlogits < (1ll << 31)),
              "ld_dlogits must be vocab .. 2^31 - 1");
  BOA_REQUIRE(d_dlogits != d_logits || !d_dlogits || ld_dlogits == ld, "in place needs ld_dlogits == ld");
  BOA_REQUIRE(std::isfinite(inv_temperature) && inv_temperature > 0.f, "inv_temperature must be finite and positive");
  if (n_rows == 0) return BOA_OK;
  BOA_REQUIRE(d_logits && d_targets && (d_loss || d_dlogits), "null buffer");
  BOA_REQUIRE(elem_aligned(d_logits, type) && token_aligned(d_targets, token_type) && boa::aligned_to(d_dloss, 4) &&
                  boa::aligned_to(d_loss, 4) && elem_aligned(d_dlogits, type),
              "a buffer is not aligned to its element");
  return train_launch(__func__, [&] {
    return boa::launch_token_loss(d_logits, type, ld, n_rows, vocab, d_targets, token_type, inv_temperature, d_dloss,
                                  grad_scale, d_loss, d_dlogits, ld_dlogits, (cudaStream_t)stream);
  });
}

}  // extern "C"
#undef BOA_REQUIRE
