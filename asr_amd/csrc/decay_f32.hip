// The chunk kernels of the causal decay attention (decay_core.h) for f32 tensors, all head widths.
#include <type_traits>

#include "decay_core.h"

namespace lmufft {

int decay_chunk_f32(int dk, int dv) {
  int n = 0;
  DECAY_FOR_WIDTHS(float, dk, dv, n, (DecGeo<float, DK, DV>::C));
  return n;
}

int decay_launch_f32(const DecayArgs& a, int roles, int dk, int dv, hipStream_t st) {
  int rc = 1;
  DECAY_FOR_WIDTHS(float, dk, dv, rc, (decay_launch<float, DK, DV>(a, roles, st)));
  return rc;
}

}  // namespace lmufft
