// SPDX-License-Identifier: Apache-2.0
//
// The dense products over f16 rows.
#include "linear_kernels.hpp"

namespace uniserve {
namespace linear {

void launch_f16(const LinearParams &p, bool gated, hipStream_t stream) {
  gated ? launch<F16, true>(p, stream) : launch<F16, false>(p, stream);
}

}  // namespace linear
}  // namespace uniserve
