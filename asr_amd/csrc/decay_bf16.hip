// The chunk kernels of the causal decay attention (decay_core.h) for bf16 tensors, all head widths.
#include <type_traits>

#include "decay_core.h"

namespace lmufft {

int decay_chunk_bf16(int dk, int dv) {
  int n = 0;
  DECAY_FOR_WIDTHS(__bf16, dk, dv, n, (DecGeo<__bf16, DK, DV>::C));
  return n;
}

int decay_launch_bf16(const DecayArgs& a, int roles, int dk, int dv, hipStream_t st) {
  int rc = 1;
  DECAY_FOR_WIDTHS(__bf16, dk, dv, rc, (decay_launch<__bf16, DK, DV>(a, roles, st)));
  return rc;
}

}  // namespace lmufft
