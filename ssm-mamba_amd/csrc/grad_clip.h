// Parameter structs of the gradient-clipping kernels.
#pragma once

#include <stdint.h>

namespace ssm {

constexpr int kClipTensors = 96;  // of one launch: its table rides in the kernel arguments

// What a call gives, host arrays of `count` entries.
struct ClipList {
  int64_t count;
  const void* const* grads;
  void* const* outs;
  const int64_t* sizes;
  const int *dtypes, *out_dtypes;  // 0: float32, 1: bf16
};

// kClipTensors tensors: tensor i's chunks (kChunk elements, grad_clip.hip) are the
// workgroups first[i] .. first[i + 1] - 1
struct ClipTable {
  int count;
  int first[kClipTensors + 1];
  const void* grad[kClipTensors];
  void* out[kClipTensors];
  int64_t n[kClipTensors];
  uint8_t type[kClipTensors];  // 1: bf16 gradient, 2: bf16 output, 4: 16-byte aligned
};

}  // namespace ssm
