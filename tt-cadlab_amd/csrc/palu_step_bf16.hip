// Decode of batches that share prefixes over bf16 page pools, row-major or tiled (palu_step.h).
#include "palu_step.h"

namespace palu {

int step_bf16(const StepArgs& a, int layout, const char* who, hipStream_t s) {
  return layout == PALU_LAYOUT_TILED ? step_run<PALU_LAYOUT_TILED>(a, who, s) : step_run<PALU_LAYOUT_ROWS>(a, who, s);
}

}  // namespace palu
