// The few-row attention kernels for head dimension 128 (a unit of its own: they take the build's
// longest to compile).
#include "ma_decode.cuh"

namespace ma {

int launch_decode_d128(const DecodeParams& p, int rows, bool wide, bool fast, cudaStream_t st) {
  return launch_decode_d<128>(p, rows, wide, fast, st);
}

}  // namespace ma
