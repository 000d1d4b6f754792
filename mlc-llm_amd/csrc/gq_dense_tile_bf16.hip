// The tile forms of gq_dense_tile.hpp for bfloat16: a file of its own, so that the two are compiled at the same time.
#include "gq_dense_tile.hpp"

namespace gq {

hipError_t launch_dense_part_bf16(const DenseArgs& a, const DensePlan& plan, int part, hipStream_t s) {
  return a.gated ? launch_form<true, true>(a, plan, part, s) : launch_form<true, false>(a, plan, part, s);
}

}  // namespace gq
