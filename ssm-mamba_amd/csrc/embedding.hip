// Embedding lookup with scaling, and its weight gradient by sorted tokens.
// gfx950.
//
//   out[i] = scale W[ids[i]],   dW[v] = scale sum over i with ids[i] = v of dout[i]
//
// Both are traffic: the lookup reads 8 bytes and a row and writes a row per
// token; the gradient reads every dout row once and writes every row of dW
// once.  The gradient's sums have a fixed order (no atomics on values): the
// positions are sorted by token, stably, and each row adds up its run.
//
// 32768 bf16 tokens of 1024 over 50280 rows (MI355X): lookup 23 us (5.7 TB/s), two
// digits of the sort 2 x 10.5 (latency: 64 workgroups, one to read all counts), the
// runs and pieces 7, the rows of dW 37 (4.2 TB/s with the dout rows); 105 with the
// gaps of seven launches.
//
// The sort is a radix sort of (token, position) pairs over as few digits of at
// most kMaxBits as cover the vocabulary, two launches a digit: each workgroup
// counts the digits of its own stretch of positions; then it finds where its
// stretch's pairs of each digit begin from all workgroups' counts and places
// them in order.  Inside a wave, a pair's rank is the number of lower lanes
// with the same digit, found by one ballot a bit.
#include "ss_common.cuh"
#include "ss_prof.h"

namespace ssm {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxBits = 10;           // of a digit
constexpr int kBins = 1 << kMaxBits;
constexpr int kMaxBlocks = 128;        // workgroups of the sort
constexpr int kMinPer = 512;           // positions a workgroup sorts, at least
constexpr int kPiece = 32;             // sorted positions summed ahead for long runs
constexpr int kSmall = 4096;           // positions that one workgroup sorts in one launch
constexpr int kNoPieces = 1024;        // positions whose runs are summed one by one
constexpr int kMaxGrid = 1 << 23;      // workgroups of a launch: fewer than 2^32 threads

// ---------------------------------------------------------------- lookup


// 16-byte pieces of rows: kThreads pieces a workgroup, in order
template <typename T, bool kVec>
__global__ __launch_bounds__(kThreads) void embed_kernel(const int64_t* __restrict__ ids,
                                                         const T* __restrict__ w, T* __restrict__ out,
                                                         int64_t n, int vocab, int dim, int pieces,
                                                         float scale) {
  constexpr int kE = kVec ? Elem<T>::kVec : 1;
  const int64_t total = n * pieces;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * kThreads) {
    const int64_t t = i / pieces;
    const int c = (int)(i - t * pieces) * kE;
    const int64_t id = ids[t];
    const bool ok = id >= 0 && id < vocab;  // else NaN: a wrong token shows, and reads nothing
    const T* src = w + (ok ? id : 0) * dim + c;
    T* dst = out + t * dim + c;
    if constexpr (kVec) {
      float v[kE];
      Elem<T>::loadv(src, v);
#pragma unroll
      for (int e = 0; e < kE; ++e) v[e] = ok ? v[e] * scale : __builtin_nanf("");
      Elem<T>::storev(dst, v);
    } else {
      Elem<T>::store1(dst, ok ? Elem<T>::load1(src) * scale : __builtin_nanf(""));
    }
  }
}

// ---------------------------------------------------------------- sort

struct Digit {
  int shift, bits;
};

// a position's token for sorting: what has no gradient (padding, outside the
// vocabulary) goes behind every row, as token `vocab`
__device__ __forceinline__ uint32_t sort_key(int64_t id, int vocab, int64_t pad) {
  return id < 0 || id >= vocab || id == pad ? (uint32_t)vocab : (uint32_t)id;
}

// counts[block][digit] of a workgroup's stretch; the first pass reads the
// tokens themselves and clears the rows' runs.
__global__ __launch_bounds__(kThreads) void sort_count_kernel(const int64_t* __restrict__ ids,
                                                              const uint2* __restrict__ in, int n,
                                                              int per, int vocab, int64_t pad, Digit d,
                                                              int* __restrict__ counts,
                                                              uint4* __restrict__ runs) {
  __shared__ int s[kBins];
  const int bins = 1 << d.bits;
  for (int k = threadIdx.x; k < bins; k += kThreads) s[k] = 0;
  if (runs)
    for (int v = blockIdx.x * kThreads + threadIdx.x; v <= vocab; v += gridDim.x * kThreads)
      runs[v] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const int lo = blockIdx.x * per, hi = min(lo + per, n);
  const uint32_t m = (1u << d.bits) - 1;
  for (int i = lo + threadIdx.x; i < hi; i += kThreads) {
    const uint32_t key = ids ? sort_key(ids[i], vocab, pad) : in[i].x;
    atomicAdd(&s[(key >> d.shift) & m], 1);  // whole numbers: any order
  }
  __syncthreads();
  for (int k = threadIdx.x; k < bins; k += kThreads) counts[blockIdx.x * bins + k] = s[k];
}

__global__ __launch_bounds__(kThreads) void sort_place_kernel(const int64_t* __restrict__ ids,
                                                              const uint2* __restrict__ in,
                                                              uint2* __restrict__ out, int n, int per,
                                                              int vocab, int64_t pad, Digit d,
                                                              const int* __restrict__ counts) {
  __shared__ int s_at[kBins];                // where this workgroup's next pair of a digit goes
  __shared__ int s_wave[kWaves][kBins];      // its waves' counts of a round
  __shared__ int s_sum[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bins = 1 << d.bits, nb = gridDim.x;
  // of each digit: pairs in front of this workgroup, and of smaller digits in all
  // (a thread has kBins / kThreads adjacent digits; 32 loads in flight)
  constexpr int kPer = kBins / kThreads;
  const int per_thread = max(bins / kThreads, 1);
  int before[kPer], all[kPer], total = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    before[k] = all[k] = 0;
    const int digit = threadIdx.x * per_thread + k;
    if (k < per_thread && digit < bins) {
      for (int b0 = 0; b0 < nb; b0 += 32) {
        int c[32];
#pragma unroll
        for (int u = 0; u < 32; ++u) c[u] = counts[min(b0 + u, nb - 1) * bins + digit];
#pragma unroll
        for (int u = 0; u < 32; ++u) {
          if (b0 + u < (int)blockIdx.x) before[k] += c[u];
          if (b0 + u < nb) all[k] += c[u];
        }
      }
    }
    total += all[k];
  }
  int run = total;  // running sum over threads, and so digits
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(run, m, 64);
    if (lane >= m) run += o;
  }
  if (lane == 63) s_sum[wave] = run;
  __syncthreads();
  for (int k = 0; k < wave; ++k) run += s_sum[k];
  run -= total;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int digit = threadIdx.x * per_thread + k;
    if (k < per_thread && digit < bins) s_at[digit] = run + before[k];
    run += all[k];
  }
  const int lo = blockIdx.x * per, hi = min(lo + per, n);
  const uint32_t mask = (1u << d.bits) - 1;
  for (int r0 = lo; r0 < hi; r0 += kThreads) {
    for (int v = threadIdx.x; v < bins; v += kThreads)
#pragma unroll
      for (int k = 0; k < kWaves; ++k) s_wave[k][v] = 0;
    __syncthreads();
    const int i = r0 + threadIdx.x;
    const bool ok = i < hi;
    uint2 kv = make_uint2(0, 0);
    if (ok) kv = ids ? make_uint2(sort_key(ids[i], vocab, pad), (uint32_t)i) : in[i];
    const uint32_t digit = (kv.x >> d.shift) & mask;
    uint64_t same = __ballot(ok);
    for (int bit = 0; bit < d.bits; ++bit) {
      const bool one = (digit >> bit) & 1;
      const uint64_t ones = __ballot(one);
      same &= one ? ones : ~ones;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (ok && rank == 0) s_wave[wave][digit] = __popcll(same);
    __syncthreads();
    if (ok) {
      int at = s_at[digit] + rank;
      for (int k = 0; k < wave; ++k) at += s_wave[k][digit];
      out[at] = kv;
    }
    __syncthreads();
    if (r0 + kThreads < hi)
      for (int v = threadIdx.x; v < bins; v += kThreads) {
        int add = 0;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) add += s_wave[k][v];
        s_at[v] += add;
      }
    __syncthreads();
  }
}

// Up to kSmall positions (what LDS holds twice): every pass in one workgroup, in LDS,
// and the runs.  The call's host time counts there, and this is one launch or two in
// place of four to six: 3000 tokens of 512 over 50280 rows, forward and backward, 59 us
// by digits over workgroups, 54 this way.  Where there are many rows (kRunsHere) their
// runs have been cleared by a launch before; few it clears itself.
constexpr int kRunsHere = 16384;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;

__global__ __launch_bounds__(kThreads) void clear_runs_kernel(uint4* runs, int vocab) {
  const int v = blockIdx.x * kThreads + threadIdx.x;
  if (v <= vocab) runs[v] = make_uint4(0, 0, 0, 0);
}

__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(const int64_t* __restrict__ ids,
                                                                  uint2* __restrict__ out, int n,
                                                                  int vocab, int64_t pad, int bits,
                                                                  uint4* __restrict__ runs) {
  constexpr int kDigit = 8, kD = 1 << kDigit;
  __shared__ uint2 s_kv[2][kSmall];
  __shared__ int s_at[kD], s_wave[kSortWaves][kD], s_sum[kD / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (vocab < kRunsHere)
    for (int v = tid; v <= vocab; v += kSortThreads) runs[v] = make_uint4(0, 0, 0, 0);
  for (int i = tid; i < n; i += kSortThreads)
    s_kv[0][i] = make_uint2(sort_key(ids[i], vocab, pad), (uint32_t)i);
  int from = 0;
  for (int shift = 0; shift < bits; shift += kDigit, from ^= 1) {
    if (tid < kD) s_at[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSortThreads) atomicAdd(&s_at[(s_kv[from][i].x >> shift) & (kD - 1)], 1);
    __syncthreads();
    // where each digit begins
    const int all = tid < kD ? s_at[tid] : 0;
    int run = all;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(run, m, 64);
      if (lane >= m) run += o;
    }
    if (tid < kD && lane == 63) s_sum[wave] = run;
    __syncthreads();
    if (tid < kD) {
      for (int k = 0; k < wave; ++k) run += s_sum[k];
      s_at[tid] = run - all;
    }
    for (int r0 = 0; r0 < n; r0 += kSortThreads) {
      for (int k = tid; k < kSortWaves * kD; k += kSortThreads) s_wave[k / kD][k % kD] = 0;
      __syncthreads();
      const int i = r0 + tid;
      const bool ok = i < n;
      const uint2 kv = ok ? s_kv[from][i] : make_uint2(0, 0);
      const uint32_t digit = (kv.x >> shift) & (kD - 1);
      uint64_t same = __ballot(ok);
#pragma unroll
      for (int bit = 0; bit < kDigit; ++bit) {
        const bool one = (digit >> bit) & 1;
        const uint64_t ones = __ballot(one);
        same &= one ? ones : ~ones;
      }
      const int rank = __popcll(same & ((1ull << lane) - 1));
      if (ok && rank == 0) s_wave[wave][digit] = __popcll(same);
      __syncthreads();
      if (tid < kD) {  // waves' counts to where each wave's pairs of the digit go
        int at = s_at[tid];
#pragma unroll
        for (int k = 0; k < kSortWaves; ++k) {
          const int c = s_wave[k][tid];
          s_wave[k][tid] = at;
          at += c;
        }
        s_at[tid] = at;
      }
      __syncthreads();
      if (ok) s_kv[from ^ 1][s_wave[wave][digit] + rank] = kv;
      __syncthreads();
    }
  }
  for (int i = tid; i < n; i += kSortThreads) {
    const uint2 kv = s_kv[from][i];
    out[i] = kv;
    if (i == 0 || s_kv[from][i - 1].x != kv.x) {
      runs[kv.x].x = i;
      runs[kv.x].z = kv.y;
    }
    if (i == n - 1 || s_kv[from][i + 1].x != kv.x) runs[kv.x].y = i + 1;
  }
}

// ---------------------------------------------------------------- sums

// kE elements as they are in memory (half the registers of bf16 on their way)
template <typename T, int kE>
struct Raw {
  using V = std::conditional_t<kE == Elem<T>::kVec, uint4, T>;
  V v;
  __device__ __forceinline__ void get(const T* p) { v = *reinterpret_cast<const V*>(p); }
  __device__ __forceinline__ void add(float (&sum)[kE]) const {
    T e[kE];
    __builtin_memcpy(e, &v, sizeof(V));
#pragma unroll
    for (int k = 0; k < kE; ++k) sum[k] += to_f32(e[k]);
  }
};

// Per piece of kPiece sorted positions, from piece `first` on: the beginnings and ends
// of runs in it go to runs[token] (begin, end, first position: a token that occurs once,
// as most do, needs no more); and a piece that lies inside one run is summed ahead, so
// that a frequent token's row adds pieces and not single positions.
template <typename T, int kE>
__global__ __launch_bounds__(kThreads) void embed_piece_kernel(const uint2* __restrict__ sorted, int n,
                                                               int first, int vocab, const T* __restrict__ dout,
                                                               int dim, uint4* __restrict__ runs,
                                                               float* __restrict__ part) {
  __shared__ uint32_t s_pos[kPiece];
  const int piece = first + blockIdx.x, lo = piece * kPiece, cnt = min(kPiece, n - lo);
  if ((int)threadIdx.x < cnt) {
    const int i = lo + threadIdx.x;
    const uint2 kv = sorted[i];
    s_pos[threadIdx.x] = kv.y;
    if (i == 0 || sorted[i - 1].x != kv.x) {
      runs[kv.x].x = i;
      runs[kv.x].z = kv.y;
    }
    if (i == n - 1 || sorted[i + 1].x != kv.x) runs[kv.x].y = i + 1;
  }
  const uint32_t token = sorted[lo].x;
  if (cnt < kPiece || token == (uint32_t)vocab || sorted[lo + kPiece - 1].x != token) return;
  __syncthreads();
  for (int c = threadIdx.x * kE; c < dim; c += kThreads * kE) {
    float sum[kE] = {};
    for (int k = 0; k < kPiece; k += 16) {
      Raw<T, kE> v[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u].get(dout + (int64_t)s_pos[k + u] * dim + c);
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u].add(sum);
    }
    float* o = part + (int64_t)piece * dim + c;
#pragma unroll
    for (int e = 0; e < kE; ++e) o[e] = sum[e];
  }
}

// A workgroup of kX * kY threads takes kY rows of dW, from row `first` on; a row's run
// is single positions up to the first whole piece, pieces, and single positions, kIn of
// them read at once.
template <typename T, int kE, int kX, int kIn>
__global__ __launch_bounds__(kThreads) void embed_rows_kernel(const uint2* __restrict__ sorted,
                                                              const uint4* __restrict__ runs, int first,
                                                              int vocab, const T* __restrict__ dout, int dim,
                                                              const float* __restrict__ part, int pieces,
                                                              float scale, T* __restrict__ dw) {
  const int row = first + blockIdx.x * (kThreads / kX) + threadIdx.x / kX;
  if (row >= vocab) return;
  const uint4 run = runs[row];
  const int lo = run.x, hi = run.y;
  const int p0 = (lo + kPiece - 1) / kPiece, p1 = pieces ? hi / kPiece : 0;  // whole pieces
  const int head = p0 < p1 ? p0 * kPiece : hi, tail = p0 < p1 ? p1 * kPiece : hi;
  for (int c = (threadIdx.x % kX) * kE; c < dim; c += kX * kE) {
    float sum[kE] = {};
    auto single = [&](int i0, int i1) {
      for (int i = i0; i < i1; i += kIn) {
        Raw<T, kE> v[kIn];
#pragma unroll
        for (int u = 0; u < kIn; ++u) v[u].get(dout + (int64_t)sorted[min(i + u, i1 - 1)].y * dim + c);
#pragma unroll
        for (int u = 0; u < kIn; ++u)
          if (i + u < i1) v[u].add(sum);
      }
    };
    if (head > lo) {
      const T* p = dout + (int64_t)run.z * dim + c;
      if constexpr (kE == Elem<T>::kVec) Elem<T>::loadv(p, sum);
      else sum[0] = Elem<T>::load1(p);
      single(lo + 1, head);
    }
    constexpr int kPieces = kE == 8 ? kIn / 2 : kIn;
    for (int k = p0; k < p1; k += kPieces) {
      float v[kPieces][kE];
#pragma unroll
      for (int u = 0; u < kPieces; ++u) {
        const float* p = part + (int64_t)min(k + u, p1 - 1) * dim + c;
#pragma unroll
        for (int e = 0; e < kE; ++e) v[u][e] = p[e];
      }
#pragma unroll
      for (int u = 0; u < kPieces; ++u)
        if (k + u < p1) {
#pragma unroll
          for (int e = 0; e < kE; ++e) sum[e] += v[u][e];
        }
    }
    single(tail, hi);
#pragma unroll
    for (int e = 0; e < kE; ++e) sum[e] *= scale;
    T* o = dw + (int64_t)row * dim + c;
    if constexpr (kE == Elem<T>::kVec) Elem<T>::storev(o, sum);
    else Elem<T>::store1(o, sum[0]);
  }
}

template <typename T, int kE, int kX>
void launch_rows(const uint2* sorted, const uint4* runs, int n, int vocab, const T* dout, int dim,
                 const float* part, float scale, T* dw, hipStream_t st) {
  constexpr int kY = kThreads / kX;
  auto go = [&](auto* kernel) {
    const int blocks = (vocab + kY - 1) / kY;
    for (int k = 0; k < blocks; k += kMaxGrid)
      hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(blocks - k, kMaxGrid)), dim3(kThreads), 0, st, sorted,
                         runs, k * kY, vocab, dout, dim, part, (int)(n > kNoPieces), scale, dw);
  };
  // long runs on average: their latency counts; else the registers do
  if (n / vocab >= 8) go(embed_rows_kernel<T, kE, kX, 16>);
  else go(embed_rows_kernel<T, kE, kX, 8>);
}

template <typename T, int kE>
hipError_t launch_sums(const uint2* sorted, uint4* runs, int n, int vocab, const T* dout, int dim,
                       float* part, float scale, T* dw, hipStream_t st) {
  ProfScope prof("embedding_grad", st);
  const int parts = n > kNoPieces ? (n + kPiece - 1) / kPiece : 0;
  for (int k = 0; k < parts; k += kMaxGrid)
    hipLaunchKernelGGL((embed_piece_kernel<T, kE>), dim3((unsigned)std::min(parts - k, kMaxGrid)),
                       dim3(kThreads), 0, st, sorted, n, k, vocab, dout, dim, runs, part);
  // a row as wide as the threads that share it
  const int pieces = (dim + kE - 1) / kE;
  if (pieces <= 64) launch_rows<T, kE, 64>(sorted, runs, n, vocab, dout, dim, part, scale, dw, st);
  else if (pieces <= 128) launch_rows<T, kE, 128>(sorted, runs, n, vocab, dout, dim, part, scale, dw, st);
  else launch_rows<T, kE, 256>(sorted, runs, n, vocab, dout, dim, part, scale, dw, st);
  return hipGetLastError();
}

int key_bits(int vocab) {  // of tokens 0 .. vocab
  int bits = 1;
  while (bits < 31 && (vocab >> bits)) ++bits;
  return bits;
}

}  // namespace

struct EmbedPlan {
  int per, blocks, pieces;
  size_t a, b, counts, runs, part, total;
};

EmbedPlan embed_plan(int n, int vocab, int dim) {
  EmbedPlan w{};
  w.per = std::max(kMinPer, ((n + kMaxBlocks - 1) / kMaxBlocks + kThreads - 1) / kThreads * kThreads);
  w.blocks = (int)(((int64_t)n + w.per - 1) / w.per);
  w.pieces = (n + kPiece - 1) / kPiece;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  };
  w.a = take((size_t)n * 8);
  w.b = take((size_t)n * 8);
  w.counts = take((size_t)w.blocks * kBins * 4);
  w.runs = take(((size_t)vocab + 1) * 16);
  w.part = take((size_t)w.pieces * dim * 4);
  w.total = at;
  return w;
}

size_t embed_bwd_workspace(int n, int vocab, int dim) { return embed_plan(n, vocab, dim).total; }

hipError_t launch_embed(int bf16, const int64_t* ids, const void* w, void* out, int64_t n, int vocab,
                        int dim, float scale, bool vec, hipStream_t st) {
  ProfScope prof("embedding", st);
  const int e = !vec ? 1 : bf16 ? 8 : 4;
  const int pieces = dim / e;
  const dim3 grid((unsigned)std::min<int64_t>((n * pieces + kThreads - 1) / kThreads, 1 << 20));
  auto go = [&](auto* kernel, auto* wp, auto* op) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, ids, wp, op, n, vocab, dim, pieces, scale);
  };
  if (bf16) {
    using T = __hip_bfloat16;
    auto* wp = static_cast<const T*>(w);
    auto* op = static_cast<T*>(out);
    if (vec) go(embed_kernel<T, true>, wp, op);
    else go(embed_kernel<T, false>, wp, op);
  } else {
    auto* wp = static_cast<const float*>(w);
    auto* op = static_cast<float*>(out);
    if (vec) go(embed_kernel<float, true>, wp, op);
    else go(embed_kernel<float, false>, wp, op);
  }
  return hipGetLastError();
}

hipError_t launch_embed_bwd(int bf16, const int64_t* ids, const void* dout, void* dw, int n, int vocab,
                            int dim, float scale, int64_t pad, bool vec, void* ws, hipStream_t st) {
  const EmbedPlan w = embed_plan(n, vocab, dim);
  char* const base = static_cast<char*>(ws);
  uint2* a = reinterpret_cast<uint2*>(base + w.a);
  uint2* b = reinterpret_cast<uint2*>(base + w.b);
  int* counts = reinterpret_cast<int*>(base + w.counts);
  uint4* runs = reinterpret_cast<uint4*>(base + w.runs);
  float* part = reinterpret_cast<float*>(base + w.part);
  {
    ProfScope prof("embedding_sort", st);
    const int bits = key_bits(vocab);
    if (n <= kSmall) {
      if (vocab >= kRunsHere)
        hipLaunchKernelGGL(clear_runs_kernel, dim3((unsigned)(vocab / kThreads + 1)), dim3(kThreads), 0, st,
                           runs, vocab);
      hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(kSortThreads), 0, st, ids, b, n, vocab, pad, bits,
                         runs);
    }
    const int passes = n <= kSmall ? 0 : (bits + kMaxBits - 1) / kMaxBits;
    const int each = (bits + passes - 1) / std::max(passes, 1);
    for (int p = 0; p < passes; ++p) {
      const Digit d{p * each, each};
      const int64_t* src = p ? nullptr : ids;
      hipLaunchKernelGGL(sort_count_kernel, dim3(w.blocks), dim3(kThreads), 0, st, src, b, n, w.per,
                         vocab, pad, d, counts, p ? nullptr : runs);
      hipLaunchKernelGGL(sort_place_kernel, dim3(w.blocks), dim3(kThreads), 0, st, src, b, a, n, w.per,
                         vocab, pad, d, counts);
      std::swap(a, b);
    }
  }
  if (hipError_t e = hipGetLastError()) return e;
  if (bf16) {
    using T = __hip_bfloat16;
    auto* dp = static_cast<const T*>(dout);
    auto* wp = static_cast<T*>(dw);
    return vec ? launch_sums<T, 8>(b, runs, n, vocab, dp, dim, part, scale, wp, st)
               : launch_sums<T, 1>(b, runs, n, vocab, dp, dim, part, scale, wp, st);
  }
  auto* dp = static_cast<const float*>(dout);
  auto* wp = static_cast<float*>(dw);
  return vec ? launch_sums<float, 4>(b, runs, n, vocab, dp, dim, part, scale, wp, st)
             : launch_sums<float, 1>(b, runs, n, vocab, dp, dim, part, scale, wp, st);
}

}  // namespace ssm
