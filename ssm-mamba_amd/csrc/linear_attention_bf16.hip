// The linear-attention pass for bf16 operands (linear_attention.cuh).
#include "linear_attention_heads.cuh"

namespace ssm {

// mode 0: results in bf16 alone; 1: the end state is wanted in float32; 2: the
// row dots too; 3: a summary
hipError_t launch_linear_attention_bf16(const LaPass& p, int mode, int blocks, hipStream_t st) {
  using T = __hip_bfloat16;
  if (mode == 0) return la::launch_dims<T, 2, 2, false, false>(p, blocks, st);
  if (mode == 1) return la::launch_dims<T, 3, 2, false, false>(p, blocks, st);
  if (mode == 2) return la::launch_dims<T, 3, 3, true, false>(p, blocks, st);
  return la::launch_dims<T, 3, 1, false, true>(p, blocks, st);
}

// the same for sums over p.subs parts of a group's heads (modes 0 to 2)
hipError_t launch_linear_attention_heads(const LaPass& p, int mode, int blocks, hipStream_t st) {
  using T = __hip_bfloat16;
  if (mode == 0) return la::launch_heads_dims<T, 2, 2, false>(p, blocks, st);
  if (mode == 1) return la::launch_heads_dims<T, 3, 2, false>(p, blocks, st);
  return la::launch_heads_dims<T, 3, 3, true>(p, blocks, st);
}

}  // namespace ssm
