// smoe_linear_mm_any.hip — the tiled kernels of linear_act for operands of any
// row length, stride and alignment: small tiles, loaded by way of registers.
#include "smoe_linear_mm.h"

namespace smoe {

int linear_mm_any(const LinArgs& a, int what, int dtype, hipStream_t s) {
  return dtype == SMOE_BF16 ? linear_mm_c<bf16_t, MmSmall, true>(a, what, s) : linear_mm_c<f16_t, MmSmall, true>(a, what, s);
}

}  // namespace smoe
