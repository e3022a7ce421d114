// pieces.h -- how the positions of one token are cut into pieces for the sums
// of the table gradient (embed.cu).  Plain integers, for host and device: a
// token may make up all of 2^31 - 1 positions, so a ceiling is formed without
// adding to the total first.
#pragma once

#ifdef __CUDACC__
#define BOA_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define BOA_HOST_DEVICE inline
#endif

namespace boa {

constexpr int kMaxPieces = 256;  // of one token: what its last block adds up

BOA_HOST_DEVICE int ceil_div(int x, int by) { return x / by + (x % by != 0); }
// Rows of a token's pieces (`rows`, or more for a token of over kMaxPieces * rows), and the number of pieces
// (one, of no rows, for a token that does not occur).
BOA_HOST_DEVICE int rows_of_piece(int total, int rows) {
  const int r = ceil_div(total, kMaxPieces);
  return r > rows ? r : rows;
}
BOA_HOST_DEVICE int pieces_of(int total, int rows) {
  const int n = ceil_div(total, rows_of_piece(total, rows));
  return n > 1 ? n : 1;
}

}  // namespace boa
