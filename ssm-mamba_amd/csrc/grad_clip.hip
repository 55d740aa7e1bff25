// The global norm of many gradients, and their scaling to a largest norm.
// gfx950.
//
//   norm = sqrt(sum g^2),  g <- g min(1, max_norm / (norm + 1e-6))
//
// Traffic alone: every gradient is read for the norm, and read and written for
// the scaling.  Launches take up to kClipTensors tensors, whose table rides in
// the kernel arguments (no copy to the device, nothing to keep alive, and
// capturable).  A workgroup takes one chunk of one tensor.  Squares are added
// in 64 bits (no overflow of a large gradient's square, no loss over many
// elements; the double adds hide behind the loads), one sum a workgroup, and the
// sums in one workgroup in a fixed order: the norm has the same bits every time.
// The scaling goes through the chunks from the last to the first: what the norm
// read last is still in the last-level cache.  211M bf16 gradients in 218 tensors into
// float32 ones (MI355X): 376 us, 1.69 GB with the second read at 4.5 TB/s; 25M
// float32 ones in place: 23 us, out of that cache.
#include "grad_clip.h"
#include "ss_common.cuh"
#include "ss_prof.h"

namespace ssm {

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 16384;  // elements of a workgroup

__device__ double block_sum(double v, double* s) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// the tensor of workgroup `blk`
__device__ __forceinline__ int find(const ClipTable& t, int blk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= blk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ double chunk_squares(const T* g, int cnt, bool vec) {
  constexpr int kE = Elem<T>::kVec;
  double sum = 0.0;
  const int whole = vec ? cnt / kE * kE : 0;
#pragma unroll 4
  for (int i = threadIdx.x * kE; i < whole; i += kThreads * kE) {
    float v[kE];
    Elem<T>::loadv(g + i, v);
#pragma unroll
    for (int e = 0; e < kE; ++e) sum = fma((double)v[e], (double)v[e], sum);
  }
  for (int i = whole + threadIdx.x; i < cnt; i += kThreads) {
    const double v = (double)Elem<T>::load1(g + i);
    sum = fma(v, v, sum);
  }
  return sum;
}

__global__ __launch_bounds__(kThreads) void clip_squares_kernel(const ClipTable t, double* part) {
  __shared__ double s[4];
  const int i = find(t, blockIdx.x);
  const int64_t at = (int64_t)(blockIdx.x - t.first[i]) * kChunk;
  const int cnt = (int)min((int64_t)kChunk, t.n[i] - at);
  const bool vec = t.type[i] & 4;
  const double v = t.type[i] & 1
      ? chunk_squares(static_cast<const __hip_bfloat16*>(t.grad[i]) + at, cnt, vec)
      : chunk_squares(static_cast<const float*>(t.grad[i]) + at, cnt, vec);
  const double sum = block_sum(v, s);
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

constexpr int kNormThreads = 1024;

__global__ __launch_bounds__(kNormThreads) void clip_norm_kernel(const double* part, int n, float max_norm,
                                                                 float* norm, float* coef) {
  __shared__ double s[kNormThreads / 64];
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += 8 * kNormThreads) {  // eight loads in flight
    double x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = part[min(i + u * kNormThreads, n - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) v += i + u * kNormThreads < n ? x[u] : 0.0;
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  double sum = 0.0;
  for (int k = 0; k < kNormThreads / 64; ++k) sum += s[k];
  if (threadIdx.x == 0) {
    const float x = (float)sqrt(sum);
    *norm = x;
    const float c = max_norm / (x + 1e-6f);
    *coef = c > 1.f ? 1.f : c;  // NaN stays
  }
}

template <typename T, typename O>
__device__ void chunk_scale(const T* g, O* o, int cnt, bool vec, float c) {
  constexpr int kE = Elem<T>::kVec;
  const int whole = vec ? cnt / kE * kE : 0;
#pragma unroll 4
  for (int i = threadIdx.x * kE; i < whole; i += kThreads * kE) {
    float v[kE];
    Elem<T>::loadv(g + i, v);
#pragma unroll
    for (int e = 0; e < kE; ++e) v[e] *= c;
    if constexpr (Elem<O>::kVec == kE) {
      Elem<O>::storev(o + i, v);
    } else if constexpr (kE == 8) {  // bf16 to float32
      *reinterpret_cast<float4*>(o + i) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(o + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {                          // float32 to bf16
      *reinterpret_cast<uint2*>(o + i) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
  }
  for (int i = whole + threadIdx.x; i < cnt; i += kThreads)
    Elem<O>::store1(o + i, Elem<T>::load1(g + i) * c);
}

__global__ __launch_bounds__(kThreads) void clip_scale_kernel(const ClipTable t, const float* coef) {
  const int blk = gridDim.x - 1 - blockIdx.x;
  const int i = find(t, blk);
  const float c = *coef;
  // in place and nothing to scale: a product with 1 would write what is there
  if (c == 1.f && t.grad[i] == t.out[i]) return;
  const int64_t at = (int64_t)(blk - t.first[i]) * kChunk;
  const int cnt = (int)min((int64_t)kChunk, t.n[i] - at);
  const bool vec = t.type[i] & 4;
  using B = __hip_bfloat16;
  const B* gb = static_cast<const B*>(t.grad[i]) + at;
  const float* gf = static_cast<const float*>(t.grad[i]) + at;
  B* ob = static_cast<B*>(t.out[i]) + at;
  float* of = static_cast<float*>(t.out[i]) + at;
  if (t.type[i] & 1) {
    if (t.type[i] & 2) chunk_scale(gb, ob, cnt, vec, c);
    else chunk_scale(gb, of, cnt, vec, c);
  } else {
    if (t.type[i] & 2) chunk_scale(gf, ob, cnt, vec, c);
    else chunk_scale(gf, of, cnt, vec, c);
  }
}

}  // namespace

int64_t clip_chunks(int64_t n) { return n / kChunk + (n % kChunk != 0); }

// In launches of kClipTensors entries of the list.  ws: a double per chunk and
// one float.
hipError_t launch_grad_clip(const ClipList& list, int64_t chunks, float max_norm, float* norm, void* ws,
                            hipStream_t st) {
  double* const part = static_cast<double*>(ws);
  float* const coef = reinterpret_cast<float*>(part + chunks);
  ClipTable t;
  auto table = [&](int64_t batch) {  // workgroups of entries kClipTensors * batch ..
    t.count = 0;
    int blocks = 0;
    for (int64_t i = batch * kClipTensors; i < list.count && i < (batch + 1) * kClipTensors; ++i) {
      if (list.sizes[i] == 0) continue;
      const int k = t.count++;
      t.first[k] = blocks;
      t.grad[k] = list.grads[i];
      t.out[k] = list.outs[i];
      t.n[k] = list.sizes[i];
      const bool vec = ((reinterpret_cast<uintptr_t>(t.grad[k]) | reinterpret_cast<uintptr_t>(t.out[k])) & 15) == 0;
      t.type[k] = (uint8_t)((list.dtypes[i] ? 1 : 0) | (list.out_dtypes[i] ? 2 : 0) | (vec ? 4 : 0));
      blocks += (int)clip_chunks(t.n[k]);
    }
    t.first[t.count] = blocks;
    return blocks;
  };
  const int64_t batches = (list.count + kClipTensors - 1) / kClipTensors;
  {
    ProfScope prof("grad_norm", st);
    int64_t at = 0;
    for (int64_t k = 0; k < batches; ++k) {
      const int blocks = table(k);
      if (blocks)
        hipLaunchKernelGGL(clip_squares_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, t,
                           part + at);
      at += blocks;
    }
    hipLaunchKernelGGL(clip_norm_kernel, dim3(1), dim3(kNormThreads), 0, st, part, (int)at, max_norm,
                       norm, coef);
  }
  ProfScope prof("grad_scale", st);
  for (int64_t k = batches; k-- > 0;) {
    const int blocks = batches == 1 ? t.first[t.count] : table(k);
    if (blocks)
      hipLaunchKernelGGL(clip_scale_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, t, coef);
  }
  return hipGetLastError();
}

}  // namespace ssm
