// Linear attention around the chunked pass (linear_attention.cuh): the fold of
// segment summaries, the decays' gradient, sums over value heads that share a
// query and key head, and the single-token step.  gfx950.
#include "linear_attention.h"
#include "ss_common.cuh"
#include "ss_prof.h"

namespace ssm {

hipError_t launch_linear_attention_bf16(const LaPass& p, int mode, int blocks, hipStream_t st);
hipError_t launch_linear_attention_f32(const LaPass& p, int mode, int blocks, hipStream_t st);
hipError_t launch_linear_attention_heads(const LaPass& p, int mode, int blocks, hipStream_t st);

namespace {

constexpr int kThreads = 256;
constexpr float kLowest = -256.f;  // as linear_attention.cuh

// Summaries to starts, in place: slot s holds what the segment in front of s
// (in the pass's time order) adds, and its decay; a thread runs one element
// through the segments.
__global__ __launch_bounds__(kThreads) void la_fold_kernel(const LaFold p) {
  const int e = blockIdx.x * kThreads + threadIdx.x, bh = blockIdx.y;
  if (e >= p.elems) return;
  float x = p.first ? p.first[(int64_t)bh * p.elems + e] : 0.f;
  for (int k = 0; k < p.nseg; ++k) {
    const int s = p.reverse ? p.nseg - 1 - k : k;
    float* slot = p.slots + ((int64_t)s * p.bh + bh) * p.elems + e;
    if (k) x = fmaf(fast_exp2(p.decay[(int64_t)s * p.bh + bh]), x, *slot);
    *slot = x;
  }
  if (p.last) {
    float* last = p.last + (int64_t)bh * p.elems + e;
    *last = fmaf(fast_exp2(p.decay[(int64_t)p.nseg * p.bh + bh]), x, *last);
  }
}

__device__ double block_sum(double v, double* s) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  return v;
}

__device__ bool valid(int t, int seqlen, const int64_t* length, int b, int pad_right) {
  if (t < 0 || t >= seqlen) return false;
  if (!length) return true;
  return pad_right ? t < length[b] : t >= seqlen - length[b];
}

// dg_t = sum of A_ij over the pairs j < t <= i.  Inside a segment ending
// before token t1: the reversed running sum of row_i - col_j (row_i = q_i . dq_i
// sums A over j, col_j = k_j . dk_j over i) plus what crosses its end,
// a_{t1} <D_{t1}, S_{t1 - 1}>, from the two passes' states there: rounding
// errors of the running sum do not pass a segment.  A workgroup per segment.
__global__ __launch_bounds__(kThreads) void la_decay_grad_kernel(const LaDecayGrad p) {
  __shared__ double s[4];
  const int seg = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int bh = b * p.heads + h, nbh = p.batch * p.heads;
  const int t0 = seg * p.seg_len, t1 = min(t0 + p.seg_len, p.seqlen);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float *S = nullptr, *D = nullptr;
  float w = 1.f;
  if (seg < p.nseg - 1) {
    S = p.starts + ((int64_t)(seg + 1) * nbh + bh) * p.elems;
    D = p.rstarts + ((int64_t)seg * nbh + bh) * p.elems;
    if (valid(t1, p.seqlen, p.length, b, p.pad_right)) {
      const float v = p.g[b * p.g_sb + t1 * p.g_st + h] * kLog2e;
      w = fast_exp2(v < kLowest ? kLowest : v);
    }
  } else if (p.last && p.dlast) {
    S = p.last + (int64_t)bh * p.elems;
    D = p.dlast + (int64_t)bh * p.elems;
  }
  double carry = 0.0;
  if (S) {
    double x = 0.0;
    // products in float32, sums of a thread's few in 64 bits
    const int quads = p.elems / 4 * 4;
#pragma unroll 4
    for (int e = threadIdx.x * 4; e < quads; e += kThreads * 4) {
      float a[4], c[4];
      if (p.elems % 4 == 0) {
        Elem<float>::loadv(S + e, a);
        Elem<float>::loadv(D + e, c);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = S[e + k], c[k] = D[e + k];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) x += (double)(a[k] * c[k]);
    }
    if (quads + (int)threadIdx.x < p.elems) x += (double)S[quads + threadIdx.x] * (double)D[quads + threadIdx.x];
    carry = (double)w * block_sum(x, s);
  }
  double sum = 0.0;
  const int64_t base = (int64_t)bh * p.seqlen;
  for (int end = t1; end > t0; end -= kThreads) {
    const int t = end - 1 - (int)threadIdx.x;
    double x = t >= t0 ? (double)p.row[base + t] - (double)p.col[base + t] : 0.0;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const double o = __shfl_up(x, m, 64);
      if (lane >= m) x += o;
    }
    if (lane == 63) s[wave] = x;
    __syncthreads();
    for (int k = 0; k < wave; ++k) x += s[k];
    const double total = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (t >= t0) {
      const bool ok = valid(t, p.seqlen, p.length, b, p.pad_right);
      const double v = ok ? carry + x : 0.0;
      if (p.part) sum += v;
      else p.dg[((int64_t)b * p.seqlen + t) * p.heads + h] = (float)v;
    }
    carry += total;
  }
  if (p.part) {
    sum = block_sum(sum, s);
    if (threadIdx.x == 0) p.part[((int64_t)b * p.nseg + seg) * p.heads + h] = (float)sum;
  }
}

// one decay per head: the sum of its segments' parts, in order
__global__ __launch_bounds__(kThreads) void la_decay_sum_kernel(const float* part, int rows, int heads,
                                                                float* dg) {
  const int h = blockIdx.x * kThreads + threadIdx.x;
  if (h >= heads) return;
  double v = 0.0;
  for (int r = 0; r < rows; ++r) v += (double)part[(int64_t)r * heads + h];
  dg[h] = (float)v;
}

// out = sum over the `rep` heads of a group, in order: part (rows, groups, rep, dim)
// in quads of elements (dim a multiple of 4), or single ones
template <typename T, int kE>
__global__ __launch_bounds__(kThreads) void la_head_sum_kernel(const float* part, int rep, int dim,
                                                               int64_t n, T* out) {
  const int per = dim / kE;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n * per;
       i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / per;
    const int c = (int)(i - row * per) * kE;
    const float* p = part + row * rep * dim + c;
    float v[kE] = {};
    for (int s = 0; s < rep; s += 8) {
      float x[8][kE];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float* q = p + (int64_t)min(s + u, rep - 1) * dim;
        if constexpr (kE == 4) Elem<float>::loadv(q, x[u]);
        else x[u][0] = *q;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s + u < rep) {
#pragma unroll
          for (int e = 0; e < kE; ++e) v[e] += x[u][e];
        }
    }
    T* o = out + row * dim + c;
    if constexpr (kE == 4 && sizeof(T) == 4) {
      Elem<float>::storev(o, v);
    } else if constexpr (kE == 4) {
      *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else {
      Elem<T>::store1(o, v[0]);
    }
  }
}

// One token: S <- a S + k v^T, o = scale S^T q.  Pure traffic of the state, so
// a workgroup takes 4 * kQ columns of one head: kQ lanes with 4 columns each
// side by side, 256 / kQ rows at a time, and adds the rows' parts of o through
// LDS.  128 rows of 32 heads of 128 x 64, 134 MB of states: 54 us from HBM, 5.0 TB/s,
// what a copy reaches, 42 where the last-level cache still has them; one row of 16
// heads of 128 x 128: 5.2 us, the launch.
template <typename T, int kQ, bool kVec>
__global__ __launch_bounds__(kThreads) void la_step_kernel(const LaStep p, int tiles) {
  constexpr int kRows = kThreads / kQ;
  __shared__ float s_q[kLaMaxDim], s_k[kLaMaxDim];
  __shared__ float s_o[kRows][4 * kQ];
  const int tile = blockIdx.x % tiles;
  const int bh = blockIdx.x / tiles, b = bh / p.heads, h = bh % p.heads;
  const int col = (threadIdx.x % kQ) * 4, row = threadIdx.x / kQ;
  const int v0 = tile * 4 * kQ + col;
  const T* q = static_cast<const T*>(p.q.p) + b * p.q.sb + (h / p.q.rep) * p.q.sh;
  const T* k = static_cast<const T*>(p.k.p) + b * p.k.sb + (h / p.k.rep) * p.k.sh;
  const T* v = static_cast<const T*>(p.v.p) + b * p.v.sb + h * p.v.sh;
  if ((int)threadIdx.x < p.key) {
    s_q[threadIdx.x] = Elem<T>::load1(q + threadIdx.x);
    s_k[threadIdx.x] = Elem<T>::load1(k + threadIdx.x);
  }
  const float gl = p.g[b * p.g_sb + h] * kLog2e;
  const float a = fast_exp2(gl < kLowest ? kLowest : gl);
  float* st = p.state + (int64_t)bh * p.key * p.value;
  float vv[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 4; ++c) vv[c] = v0 + c < p.value ? Elem<T>::load1(v + v0 + c) : 0.f;
  __syncthreads();
  if (v0 < p.value) {
#pragma unroll 4
    for (int d = row; d < p.key; d += kRows) {
      float* s = st + (int64_t)d * p.value + v0;
      float x[4];
      if constexpr (kVec) {
        Elem<float>::loadv(s, x);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = v0 + c < p.value ? s[c] : 0.f;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[c] = fmaf(s_k[d], vv[c], a * x[c]);
        o[c] = fmaf(s_q[d], x[c], o[c]);
      }
      if constexpr (kVec) {
        Elem<float>::storev(s, x);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (v0 + c < p.value) s[c] = x[c];
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) s_o[row][col + c] = o[c];
  __syncthreads();
  if (threadIdx.x < 4 * kQ) {
    const int z = tile * 4 * kQ + threadIdx.x;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) sum += s_o[r][threadIdx.x];
    if (z < p.value)
      Elem<T>::store1(static_cast<T*>(p.out) + (int64_t)bh * p.value + z, sum * p.scale);
  }
}

template <typename T, int kQ>
hipError_t launch_step(const LaStep& p, bool vec, hipStream_t st) {
  ProfScope prof("linear_attention_step", st);
  const int tiles = (p.value + 4 * kQ - 1) / (4 * kQ);
  const dim3 grid((unsigned)((int64_t)p.batch * p.heads * tiles));
  if (vec) hipLaunchKernelGGL((la_step_kernel<T, kQ, true>), grid, dim3(kThreads), 0, st, p, tiles);
  else hipLaunchKernelGGL((la_step_kernel<T, kQ, false>), grid, dim3(kThreads), 0, st, p, tiles);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_step_t(const LaStep& p, bool vec, hipStream_t st) {
  // few heads: 16 columns a workgroup, so that there are workgroups for more CUs
  if ((int64_t)p.batch * p.heads < 512 || p.value <= 16) return launch_step<T, 4>(p, vec, st);
  if (p.value <= 32) return launch_step<T, 8>(p, vec, st);
  if (p.value <= 64) return launch_step<T, 16>(p, vec, st);
  return launch_step<T, 32>(p, vec, st);
}

}  // namespace

// Parts of a group's heads: of bf16 several heads share a workgroup (see
// linear_attention_heads.cuh), of float32, whose tiles fill LDS, each has its own.
int la_subs(int64_t rep, int64_t ydim, int bf16) {
  const int64_t heads = !bf16 ? 1 : ydim <= 64 ? 4 : 2;
  return (int)((rep + heads - 1) / heads);
}

// Tokens per segment: one whole sequence where its workgroups alone fill the machine,
// or of up to 4 chunks; else as many segments as do, of at least 2 chunks each (a
// segment costs a summary of its tokens and reads of its start).  8 heads of 128 x
// 128: 256 tokens forward took 18 us in one segment and 26 in two, 1024 forward and
// backward 110 with segments of 2 chunks, 127 with 3, 191 with 6.  A pass over 128
// columns, of float32, or over the heads of a group has one workgroup a CU, one over
// 64 columns two: 4 x 2048 tokens of 16 heads of 128 x 128 forward and backward took
// 318 us with 256 workgroups and 375 with 512.
int la_segment_len(int64_t batch, int64_t seqlen, int64_t heads, int64_t groups, int64_t key,
                   int64_t value, int bf16) {
  const int64_t rep = heads / groups;
  const bool two = bf16 && rep == 1 && std::min(key, value) <= 64;
  const int64_t units = batch * groups * la_subs(rep, value, bf16);
  const int64_t chunks = (seqlen + kLaChunk - 1) / kLaChunk;
  const int64_t want = ((two ? 512 : 256) + units - 1) / units;
  const int64_t per = std::max<int64_t>((chunks + want - 1) / want, chunks <= 4 ? 4 : 2);
  return (int)(std::min(per, chunks) * kLaChunk);
}

hipError_t launch_la_pass(const LaPass& p, int bf16, int mode, hipStream_t st) {
  if (p.part && bf16)
    return launch_linear_attention_heads(
        p, mode, (int)((int64_t)p.batch * (p.heads / p.rep) * p.subs * p.nseg), st);
  const int blocks = (int)((int64_t)p.batch * p.heads * p.nseg);
  return bf16 ? launch_linear_attention_bf16(p, mode, blocks, st)
              : launch_linear_attention_f32(p, mode, blocks, st);
}

hipError_t launch_la_fold(const LaFold& p, hipStream_t st) {
  ProfScope prof("linear_attention_fold", st);
  const dim3 grid((unsigned)((p.elems + kThreads - 1) / kThreads), (unsigned)p.bh);
  hipLaunchKernelGGL(la_fold_kernel, grid, dim3(kThreads), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_la_decay_grad(const LaDecayGrad& p, hipStream_t st) {
  ProfScope prof("linear_attention_decay_grad", st);
  hipLaunchKernelGGL(la_decay_grad_kernel, dim3(p.nseg, p.heads, p.batch), dim3(kThreads), 0, st, p);
  if (p.part)
    hipLaunchKernelGGL(la_decay_sum_kernel, dim3((p.heads + kThreads - 1) / kThreads), dim3(kThreads),
                       0, st, p.part, p.batch * p.nseg, p.heads, p.dg);
  return hipGetLastError();
}

// part (rows, rep, dim) float32 -> out (rows, dim)
hipError_t launch_la_head_sum(int bf16, const float* part, int rep, int dim, int64_t rows, void* out,
                              hipStream_t st) {
  ProfScope prof("linear_attention_head_sum", st);
  const int e = dim % 4 ? 1 : 4;
  const dim3 grid((unsigned)std::min<int64_t>((rows * (dim / e) + kThreads - 1) / kThreads, 1 << 20));
  auto go = [&](auto* kernel, auto* o) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, part, rep, dim, rows, o);
  };
  if (bf16) {
    using T = __hip_bfloat16;
    if (e == 4) go(la_head_sum_kernel<T, 4>, static_cast<T*>(out));
    else go(la_head_sum_kernel<T, 1>, static_cast<T*>(out));
  } else {
    if (e == 4) go(la_head_sum_kernel<float, 4>, static_cast<float*>(out));
    else go(la_head_sum_kernel<float, 1>, static_cast<float*>(out));
  }
  return hipGetLastError();
}

hipError_t launch_la_step(const LaStep& p, int bf16, bool vec, hipStream_t st) {
  return bf16 ? launch_step_t<__hip_bfloat16>(p, vec, st) : launch_step_t<float>(p, vec, st);
}

}  // namespace ssm
