// SPDX-License-Identifier: Apache-2.0
//
// The dense products over bf16 rows.
#include "linear_kernels.hpp"

namespace uniserve {
namespace linear {

void launch_bf16(const LinearParams &p, bool gated, hipStream_t stream) {
  gated ? launch<Bf16, true>(p, stream) : launch<Bf16, false>(p, stream);
}

}  // namespace linear
}  // namespace uniserve
