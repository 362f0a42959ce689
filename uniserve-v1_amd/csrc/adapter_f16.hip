// SPDX-License-Identifier: Apache-2.0
//
// The dense products with low-rank adapters over f16 rows.
#include "linear_kernels.hpp"

namespace uniserve {
namespace linear {

void launch_adapters_f16(const AdapterParams &p, bool gated, hipStream_t stream) {
  launch_low_rank<F16>(p, gated, stream);
  gated ? launch<F16, true>(p, stream) : launch<F16, false>(p, stream);
}

}  // namespace linear
}  // namespace uniserve
