// boa_all.cu -- the library's main translation unit.  Kernels, launchers and
// the host runtime are compiled together so that device globals (the error
// word read back by the host) have exactly one definition without relocatable
// device code.  embed.cu, recur.cu and loss.cu (the training operators), which
// never touch the error word, are compiled on their own.
#include "gemm.cu"
#include "mlp.cu"
#include "mamba.cu"
#include "rnn.cu"
#include "runtime.cpp"
#include "container.cpp"
#include "noalloc.cu"
#include "coder_api.cu"
#include "pyrc.cu"
#include "train_api.cu"
