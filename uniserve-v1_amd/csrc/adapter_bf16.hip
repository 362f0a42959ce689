// SPDX-License-Identifier: Apache-2.0
//
// The dense products with low-rank adapters over bf16 rows.
#include "linear_kernels.hpp"

namespace uniserve {
namespace linear {

void launch_adapters_bf16(const AdapterParams &p, bool gated, hipStream_t stream) {
  launch_low_rank<Bf16>(p, gated, stream);
  gated ? launch<Bf16, true>(p, stream) : launch<Bf16, false>(p, stream);
}

}  // namespace linear
}  // namespace uniserve
