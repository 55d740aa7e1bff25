// Linear attention with a decay for each head, over chunks of 64 tokens on the
// matrix cores (gfx950).
//
//   S_t = a_t S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t,   a_t = exp(g_t)
//
// The output and the gradients of q, k and v are one and the same sum,
//
//   out_i = sum_{j <= i} W_ij (x_i . y_j) z_j,   W_ij = exp(g_{j+1} + ... + g_i):
//
//   o:  x = q,  y = k,  z = v              dq: x = do, y = v,  z = k
//   dk: x = v,  y = do, z = q, reversed    dv: x = k,  y = q,  z = do, reversed
//
// (in reversed time token t's predecessor is t + 1 and its decay g_{t+1}), so
// one kernel serves all four.  A workgroup of four or eight waves runs one
// segment of one head chunk after chunk with the state S = sum w y z^T in
// registers: each wave owns 16 columns of z and all rows.  Per chunk, c_i the running
// sum of the decays from the chunk's start:
//
//   P_ij  = exp(c_i - c_j) x_i . y_j for j <= i   (a wave per 16 rows i; to LDS)
//   out_i = exp(c_i) S^T x_i + sum_j P_ij z_j     (a wave's own columns)
//   S     = exp(c_n) S + sum_j y_j (exp(c_n - c_j) z_j)^T
//
// so the state never leaves the registers inside a segment.  Segments of one
// sequence run at once, from starts that a summary pass (the update alone) and
// a fold over the segments provide.
//
// Products are v_mfma_f32_16x16x32_bf16, or eight v_mfma_f32_16x16x4_f32 for
// float32.  A fragment is 8 values of one row (or column) index l % 16 for lane
// l: contraction indexes 4 (l / 16) + {0..3} of one 16-wide tile and of the next.  Any
// order does for a contraction as long as both operands have it, and in this one a
// result tile's lane layout (4 consecutive rows of one column) is an operand's: the
// state is used as it lies in the accumulators, and P is written and read 4 values at a
// time.  bf16 contracts over columns in order, 8 (l / 16) + {0..7}, one 16-byte piece of
// a row; the rows of a state stand for columns accordingly (state_row()).
//
// Roundings (bf16): x, y, z enter the matrix cores as they are; P, z times its decay and
// the state as an operand each as a sum of two bf16 terms, 2^-16 of them at most.  One
// term of the state would leave 2^-8 of the part of the result that it carries, which is
// most of it where decays are slow: 2.2e-3 of the result's norm at decays of 1 - 2^-8,
// where the result's own rounding is 1.66e-3 (and what is here leaves no more than that).
// Where the result is float32 (a last state, the decays' gradient) z and the state are
// three terms, which hold all 24 bits, so their products are float32's.  The decays'
// gradient needs r_i . out_i (r the partner of out: q of dq, k of dk): the state's part
// from the float32 accumulators, the chunk's own as sum_j W_ij (x_i . y_j)(r_i . z_j), two
// products of exact operands.  Sums, states and decays stay in float32, running sums of
// decays in 64 bits (two float32 terms where weights of P are made from them).
//
// What bounds it (MI355X, 4 x 2048 tokens of 16 heads of 128 x 128, bf16; one
// workgroup of eight waves a CU, 8 chunks each): a pass for o or dv takes 48 us, 151
// MB of rows and starts at 3.1 TB/s.  (With one term of the state, 44; then without its
// loads and stores 26, without its products 35: the two overlap in part.)  A wave issues
// 81 matrix instructions of 16 cycles a chunk and about 530 vector ones, in phases
// between two barriers.  A pass with row dots takes 68 us, 124 matrix and 800 vector
// instructions (the splits into three terms); a summary 26.  A prompt of 32768 tokens of
// those heads takes 248 us in a row of calls; in a trace, whose launches are longer, its
// pass is 184 and the summary, which reads k and v once more, 92.  In float32 it takes
// 793 (traced 580 and 238): half of the matrix rate, the eight waves' phases are not
// hidden by another workgroup, for which LDS has no room.
#pragma once

#include "linear_attention.h"
#include "ss_common.cuh"
#include "ss_prof.h"

namespace ssm {

namespace la {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kC = kLaChunk;
// decays below 2^kLowest are zero in float32: the floor keeps sums finite for
// a decay of zero (g = -inf)
constexpr float kLowest = -256.f;

// A tile of 64 rows of kDim elements in LDS, the 16-byte pieces of a row permuted by
// an xor with f(row), which spreads what one instruction asks of LDS (64 banks, 256
// bytes, a cycle) over the banks.  bf16: a row fragment is one piece of 16 rows, a
// column read four quads of four rows; f, linear over xor, sends the row's bits that
// do not choose banks by themselves to 4, 8, 2 and 3, with which 16 lanes' pieces are
// apart in either of the orders that LDS may take the lanes in.  Measured alone, with
// an xor of the row's 3 low bits a row fragment took 16 cycles and a column read 8;
// asked in this order 4 and 4 (a column read wants half a piece of each row), and
// conflicts went from 6.3 to 1.4 million cycles a pass, its time from 45.5 to 44 us.
// float32: a piece is a quad, and f the row's bits.  An address is (a lane's base ^ a
// constant of the block) + a constant.
template <typename E, int kDim>
struct Tile {
  static constexpr int kRow = kDim * (int)sizeof(E);    // bytes
  static constexpr int kBytes = kC * kRow;
  static constexpr int kVec = 16 / (int)sizeof(E);
  static constexpr int kPieces = kRow / 16;
  static constexpr bool kHalf = sizeof(E) == 2;
  static constexpr int kShift = kRow >= 128 ? 0 : 1;    // float32: rows per 128 bytes

  __device__ static __forceinline__ uint32_t permuted(uint32_t row, uint32_t piece) {
    if constexpr (!kHalf) return piece ^ ((row >> kShift) & 7);
    const uint32_t f = ((row >> 2 ^ row >> 3) & 1) << 1 | (row >> 3 & 1);
    const uint32_t high = kRow == 256 ? (row & 3) << 2 : kRow == 128 ? (row & 2) << 1 : 0;
    return piece ^ f ^ high;
  }
  // the byte of the quad of columns 4 u ..
  __device__ static __forceinline__ uint32_t quad(uint32_t row, uint32_t u) {
    if constexpr (!kHalf) return row * kRow + permuted(row, u) * 16;
    return row * kRow + permuted(row, u >> 1) * 16 + (u & 1) * 8;
  }
  // what lane has of a row fragment of rows 0 to 15, and of the ks-th 32 columns
  __device__ static __forceinline__ uint32_t row_base(int lane) {
    return quad(lane & 15, kHalf ? 2 * (lane >> 4) : lane >> 4);
  }
  __device__ static __forceinline__ uint32_t row_tile(uint32_t base, int ks) { return base ^ (ks * (kHalf ? 64 : 128)); }
  // quad lane / 16 of row lane % 16, and the same of 16-column tile ct
  __device__ static __forceinline__ uint32_t quad_base(int lane) { return quad(lane & 15, lane >> 4); }
  __device__ static __forceinline__ uint32_t quad_tile(uint32_t base, int ct) { return base ^ (ct * (kHalf ? 32 : 64)); }
  // what lane asks of 16 columns in order: see column()
  __device__ static __forceinline__ uint32_t col_base(int lane) {
    const uint32_t r = lane & 15, g = lane >> 4;
    return kHalf ? quad(4 * g + (r >> 2), r & 3) : quad(4 * g, r >> 2) + (r & 3) * 4;
  }
  // and of those that the at-th 16 rows of a state stand for: see state_row()
  __device__ static __forceinline__ uint32_t state_base(int lane) {
    const uint32_t r = lane & 15, g = lane >> 4;
    return kHalf ? quad(4 * g + (r >> 2), 2 * (r & 3)) : col_base(lane);
  }
  __device__ static __forceinline__ uint32_t state_tile(uint32_t base, int at) {
    return kHalf ? (base ^ ((at >> 1) * 64)) + (at & 1) * 8 : quad_tile(base, at);
  }
};

// the column of y that row 4 gq of the at-th 16 rows of a state stands for: such that
// two tiles of a state make a fragment over columns
template <typename T>
__device__ __forceinline__ int state_row(int at, int gq) {
  return sizeof(T) == 2 ? at / 2 * 32 + gq * 8 + (at & 1) * 4 : at * 16 + gq * 4;
}

template <typename T> struct Mat;

template <> struct Mat<__hip_bfloat16> {
  using E = __bf16;
  using Frag = bf16x8;
  using Quad = bf16x4;
  __device__ static __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // column lane % 16, rows row0 + 4 (lane / 16) + {0..3}: a transposed LDS read, lane r
  // of 16 giving row r / 4 and its quad r % 4
  template <typename Tl>
  __device__ static __forceinline__ Quad column(const char* t, uint32_t at, int row0) {
    const char* p = t + at + row0 * Tl::kRow;
    return __builtin_bit_cast(Quad, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4*)p));
  }
};

template <> struct Mat<float> {
  using E = float;
  using Frag = f32x8;
  using Quad = f32x4;
  __device__ static __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  template <typename Tl>
  __device__ static __forceinline__ Quad column(const char* t, uint32_t at, int row0) {
    Quad q;
#pragma unroll
    for (int e = 0; e < 4; ++e)  // row 4 g + e: its xor is that of row 4 g, ^ (e >> kShift)
      q[e] = *reinterpret_cast<const float*>(t + (at ^ ((e >> Tl::kShift) << 4)) +
                                             (row0 + e) * Tl::kRow);
    return q;
  }
};

template <typename T>
__device__ __forceinline__ typename Mat<T>::Frag join(typename Mat<T>::Quad a,
                                                      typename Mat<T>::Quad b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// row lane % 16 of the tile at t, the ks-th 32 columns; base: row_base(lane)
template <typename T, typename Tl>
__device__ __forceinline__ typename Mat<T>::Frag row_frag(const char* t, uint32_t base, int ks) {
  using Quad = typename Mat<T>::Quad;
  const uint32_t at = Tl::row_tile(base, ks);
  if constexpr (Tl::kHalf) return *reinterpret_cast<const typename Mat<T>::Frag*>(t + at);
  return join<T>(*reinterpret_cast<const Quad*>(t + at), *reinterpret_cast<const Quad*>(t + (at ^ 64)));
}

// column lane % 16 of the 16 columns at `at` (quad_tile of col_base, state_tile of
// state_base), rows row0 + 0..31
template <typename T, typename Tl>
__device__ __forceinline__ typename Mat<T>::Frag col_frag(const char* t, uint32_t at, int row0) {
  return join<T>(Mat<T>::template column<Tl>(t, at, row0),
                 Mat<T>::template column<Tl>(t, at, row0 + 16));
}

// bf16 terms that P is a sum of: one would be off by up to 2^-8, as much as the result's
// own rounding; with two, that is what counts
template <typename T> constexpr int kP = sizeof(T) == 2 ? 2 : 1;

// v as a sum of kN operands (float32: itself)
template <typename T, int kN>
__device__ __forceinline__ void split(f32x8 v, typename Mat<T>::Frag (&out)[kN]) {
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    out[n] = __builtin_convertvector(v, typename Mat<T>::Frag);
    if (n + 1 < kN) v -= __builtin_convertvector(out[n], f32x8);
  }
}

// log2 of a token's decay, zero (no decay) where the token is padding
__device__ __forceinline__ float la_log2_decay(const float* g, int64_t sb, int64_t st, int b, int t,
                                               int h, bool ok) {
  if (!ok) return 0.f;
  const float v = g[b * sb + t * st + h] * kLog2e;
  return v < kLowest ? kLowest : v;  // NaN stays
}

template <int kCtrl, int kRows>
__device__ __forceinline__ double dpp_add(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kCtrl, kRows, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), kCtrl, kRows, 0xF, false);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// running sum over the 64 lanes: shifts inside rows of 16 lanes, then the ends
// of rows 0 and 2 to rows 1 and 3, then that of row 1 to rows 2 and 3
__device__ __forceinline__ double wave_scan(double x) {
  x = dpp_add<0x111, 0xF>(x);
  x = dpp_add<0x112, 0xF>(x);
  x = dpp_add<0x114, 0xF>(x);
  x = dpp_add<0x118, 0xF>(x);
  x = dpp_add<0x142, 0xA>(x);
  return dpp_add<0x143, 0xC>(x);
}

// The 64 token rows of an operand on their way to LDS (row r: token first + step *
// r).  The loads go through a buffer descriptor of the valid tokens among them, lo
// to hi - 1: whatever is outside (other tokens, pieces past dim) reads as zero and
// touches no memory, so a chunk needs no branch and no mask.  A thread takes one
// 16-byte column of every kRows-th row.
template <typename T, typename Tl, int kThreads>
struct Rows {
  using E = typename Mat<T>::E;
  static constexpr int kRows = kThreads / Tl::kPieces;
  static constexpr int kN = (kC + kRows - 1) / kRows;
  static constexpr int kSpan = kC / kN;                 // rows apart; more threads than rows: 64
  typedef uint32_t V __attribute__((ext_vector_type(4)));
  V v[kN];
  uint32_t off;   // of the window's row threadIdx.x / kPieces, in bytes
  uint32_t at;    // in the tile

  __device__ __forceinline__ void init(const LaTensor& x, bool reverse) {
    const int q = threadIdx.x % kThreads / Tl::kPieces, piece = threadIdx.x % kThreads % Tl::kPieces;
    off = piece * Tl::kVec < x.dim ? q * (uint32_t)x.st * (uint32_t)sizeof(E) + piece * 16 : 0x80000000u;
    at = Tl::quad((reverse ? kSpan - 1 - q : q) & (kC - 1), Tl::kHalf ? 2 * piece : piece);
  }
  // the 64 tokens from `window` on, of which [lo, hi) are valid
  __device__ __forceinline__ void get(const LaTensor& x, const E* src, int window, int lo, int hi,
                                      bool reverse) {
    const uint32_t row = (uint32_t)x.st * (uint32_t)sizeof(E);
    const int n = max(hi - lo, 0);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<E*>(src + (n ? lo : 0) * x.st), 0, (int)(n * row), 0x00020000);
    const uint32_t from = (uint32_t)(window - lo) * row;  // at most 0, modulo 2^32
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const uint32_t k = reverse ? kN - 1 - i : i;
      v[i] = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off + (from + k * kSpan * row),
                                                                         0, 0));
    }
  }
  __device__ __forceinline__ void put(char* tile, int dim) {
    if (kRows > kC && threadIdx.x % kThreads / Tl::kPieces >= kC) return;
    if (dim % Tl::kVec) {  // of the piece that holds the last columns
      using Bits = std::conditional_t<sizeof(E) == 2, uint16_t, uint32_t>;
      const int c = threadIdx.x % kThreads % Tl::kPieces * Tl::kVec;
      E e[Tl::kVec];
#pragma unroll
      for (int k = 0; k < Tl::kVec; ++k) e[k] = __builtin_bit_cast(E, (Bits)(c + k < dim ? ~0u : 0u));
      V keep;
      __builtin_memcpy(&keep, e, 16);
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] &= keep;
    }
    // a thread's rows have one xor (a multiple of 16 apart; float32's has 8 values)
    static_assert(kSpan % (Tl::kHalf ? 16 : 8) == 0, "rows that a thread takes");
#pragma unroll
    for (int i = 0; i < kN; ++i) *reinterpret_cast<V*>(tile + i * kSpan * Tl::kRow + at) = v[i];
  }
};

// a chunk's rows, lane column l % 16 of 16-row tile it, four columns of z; o: the
// (batch, seqlen, heads, zdim) array's row of this batch row's token 0 and this head
template <typename E>
__device__ __forceinline__ void store_rows(E* o, const f32x4 (&out)[4], int first, int step, int n,
                                           int64_t next, int zdim, int wave, int lane) {
  typedef E Quad __attribute__((ext_vector_type(4)));
  const int l16 = lane & 15, z = wave * 16 + (lane >> 4) * 4;
  const uint32_t off = (step > 0 ? l16 : 15 - l16) * (uint32_t)next + z;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    E* const p = o + (step > 0 ? first + it * 16 : first - it * 16 - 15) * next;
    if (it * 16 + l16 >= n) continue;
    const Quad q = __builtin_convertvector(out[it], Quad);
    if ((zdim & 3) == 0) {
      if (z < zdim) *reinterpret_cast<Quad*>(p + off) = q;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (z + r < zdim) p[off + r] = q[r];
    }
  }
}

// A state between memory and the accumulators (rows state_row(at, lane / 16) + r of
// column 16 wave + lane % 16) by way of LDS, whole rows at a time, zeros around it.
// Memory is (ydim, zdim), or (zdim, ydim) with trans.
template <typename T, int kA, int kB, int kThreads>
__device__ __forceinline__ void load_state(char* smem, const float* src, int trans, int ydim, int zdim,
                                           int zcol, int gq, f32x4 (&st)[kA / 16]) {
  float* const s = reinterpret_cast<float*>(smem);
  const int tid = threadIdx.x % kThreads;
  if (src) {
    const int rows = trans ? zdim : ydim, cols = trans ? ydim : zdim, ld = trans ? kA : kB;
    constexpr int kN = kA * kB / 4 / kThreads;
    f32x4 v[kN];
#pragma unroll
    for (int u = 0; u < kN; ++u) {
      const int i = (tid + u * kThreads) * 4, r = i / ld, c = i % ld;  // ld: a power of two
      const float* const q = src + min(r, rows - 1) * cols;
      if (cols % 4 == 0) {
        v[u] = *reinterpret_cast<const f32x4*>(q + min(c, cols - 4));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[u][e] = q[min(c + e, cols - 1)];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[u][e] = r < rows && c + e < cols ? v[u][e] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kN; ++u) *reinterpret_cast<f32x4*>(s + (tid + u * kThreads) * 4) = v[u];
    __syncthreads();
  }
#pragma unroll
  for (int at = 0; at < kA / 16; ++at) {
    st[at] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (src) {
      const int a = state_row<T>(at, gq);
      if (trans) {
        st[at] = *reinterpret_cast<const f32x4*>(s + zcol * kA + a);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) st[at][r] = s[(a + r) * kB + zcol];
      }
    }
  }
}

template <typename T, int kA, int kB, int kThreads>
__device__ __forceinline__ void store_state(char* smem, float* dst, float w, int trans, int ydim, int zdim,
                                            int zcol, int gq, const f32x4 (&st)[kA / 16]) {
  __syncthreads();  // what was in LDS is read
  float* const s = reinterpret_cast<float*>(smem);
  const int tid = threadIdx.x % kThreads;
#pragma unroll
  for (int at = 0; at < kA / 16; ++at) {
    const int a = state_row<T>(at, gq);
    const f32x4 v = st[at] * w;
    if (trans) {
      *reinterpret_cast<f32x4*>(s + zcol * kA + a) = v;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) s[(a + r) * kB + zcol] = v[r];
    }
  }
  __syncthreads();
  const int rows = trans ? zdim : ydim, cols = trans ? ydim : zdim, ld = trans ? kA : kB;
  if (cols % 4 == 0) {
    for (int i = tid * 4; i < rows * ld; i += kThreads * 4) {
      const int r = i / ld, c = i % ld;
      if (c < cols) *reinterpret_cast<f32x4*>(dst + r * cols + c) = *reinterpret_cast<const f32x4*>(s + i);
    }
  } else {
    for (int i = tid; i < rows * ld; i += kThreads) {
      const int r = i / ld, c = i % ld;
      if (c < cols) dst[r * cols + c] = s[i];
    }
  }
}

// out^T = S^T x for the 64 rows x: lane column i = lane % 16 of each 16-row tile,
// four columns z
template <typename T, typename TA, int kO, bool kSkip, int kAT>
__device__ __forceinline__ void state_rows(const char* sx, uint32_t row_a, const f32x4 (&st)[kAT], int ydim,
                                           f32x4 (&out)[4]) {
  using Frag = typename Mat<T>::Frag;
#pragma unroll
  for (int it = 0; it < 4; ++it) out[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < kAT / 2; ++ks) {
    if (kSkip && ks * 32 >= ydim) break;
    Frag fs[kO], f[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) f[it] = row_frag<T, TA>(sx + it * 16 * TA::kRow, row_a, ks);
    split<T, kO>(__builtin_shufflevector(st[2 * ks], st[2 * ks + 1], 0, 1, 2, 3, 4, 5, 6, 7), fs);
#pragma unroll
    for (int s = 0; s < kO; ++s)
#pragma unroll
      for (int it = 0; it < 4; ++it) out[it] = Mat<T>::mma(fs[s], f[it], out[it]);
  }
}

// the dot of a row's quad in LDS with out's, summed over the 16 columns of a wave
template <typename T>
__device__ __forceinline__ float quad_dot(const char* r, f32x4 out) {
  const f32x4 v = __builtin_convertvector(*reinterpret_cast<const typename Mat<T>::Quad*>(r), f32x4);
  float dot = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) dot = fmaf(v[e], out[e], dot);
  dot += __shfl_xor(dot, 16, 64);
  return dot + __shfl_xor(dot, 32, 64);
}

// P (lane column i, four rows j) as a sum of kP operands, to row i of as many tiles
template <typename T, typename TP>
__device__ __forceinline__ void put_p(char* p, f32x4 v) {
#pragma unroll
  for (int k = 0; k < kP<T>; ++k) {
    const auto q = __builtin_convertvector(v, typename Mat<T>::Quad);
    *reinterpret_cast<typename Mat<T>::Quad*>(p + k * TP::kBytes) = q;
    if (k + 1 < kP<T>) v -= __builtin_convertvector(q, f32x4);
  }
}

// 0, or NaN if a value is not finite
__device__ __forceinline__ float zero_or_nan(f32x4 v) {
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) sum = fmaf(v[e], 0.f, sum);
  return sum;
}
__device__ __forceinline__ float zero_or_nan(f32x8 v) {
  return zero_or_nan(__builtin_shufflevector(v, v, 0, 1, 2, 3)) + zero_or_nan(__builtin_shufflevector(v, v, 4, 5, 6, 7));
}
__device__ __forceinline__ float zero_or_nan(bf16x8 v) { return zero_or_nan(__builtin_convertvector(v, f32x8)); }

// out^T += Z^T P^T one row of z after the other, to its own row out and later ones
template <typename T, typename TB, typename TP>
__device__ __forceinline__ void add_rows(const char* sz, const char* sp, int wave, f32x4 (&out)[4]) {
  using E = typename Mat<T>::E;
  const int lane = threadIdx.x & 63, l16 = lane & 15, gq = lane >> 4;
#pragma unroll 1
  for (int j = 0; j < kC; ++j) {
    const f32x4 z = __builtin_convertvector(
        *reinterpret_cast<const typename Mat<T>::Quad*>(sz + TB::quad(j, wave * 4 + gq)), f32x4);
    const int jt = j >> 4, jq = j >> 2 & 3;
    const int u = TP::kHalf ? (jt >> 1) * 8 + jq * 2 + (jt & 1) : jt * 4 + jq;  // as put_p() has it
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int i = it * 16 + l16;
      if (i < j) continue;
      const char* const at = sp + TP::quad(i, u) + (j & 3) * sizeof(E);
      float w = 0.f;
#pragma unroll
      for (int k = 0; k < kP<T>; ++k) w += (float)*reinterpret_cast<const E*>(at + k * TP::kBytes);
      out[it] += w * z;
    }
  }
}

// out^T += Z^T P^T, P's blocks above the diagonal left out.  Inside the others P is zero
// above it, which is still NaN times a later row of z that is not finite.  The last 16
// rows out have a product with every row of z: only where one of them is not finite is z
// looked through, and a chunk with such a value taken row by row.
template <typename T, typename TB, typename TP>
__device__ __forceinline__ void add_chunk(const char* sz, const char* sp, uint32_t col_b, uint32_t row_p,
                                          int wave, f32x4 (&out)[4]) {
  using Frag = typename Mat<T>::Frag;
  const f32x4 before[4] = {out[0], out[1], out[2], out[3]};
#pragma unroll
  for (int js = 0; js < 2; ++js) {
    const Frag fz = col_frag<T, TB>(sz, TB::quad_tile(col_b, wave), js * 32);
    Frag fp[4];
#pragma unroll
    for (int k = 0; k < kP<T>; ++k) {
#pragma unroll
      for (int it = 2 * js; it < 4; ++it)
        fp[it] = row_frag<T, TP>(sp + k * TP::kBytes + it * 16 * TP::kRow, row_p, js);
#pragma unroll
      for (int it = 2 * js; it < 4; ++it) out[it] = Mat<T>::mma(fz, fp[it], out[it]);
    }
  }
  if (__any(__builtin_isnan(zero_or_nan(out[3])))) {
    float z = 0.f;
#pragma unroll
    for (int js = 0; js < 2; ++js) z += zero_or_nan(col_frag<T, TB>(sz, TB::quad_tile(col_b, wave), js * 32));
    if (__any(__builtin_isnan(z))) {
#pragma unroll
      for (int it = 0; it < 4; ++it) out[it] = before[it];
      add_rows<T, TB, TP>(sz, sp, wave, out);
    }
  }
}

// S <- exp(total) S + sum_j y_j (in_j z_j)^T; in: of row 4 (lane / 16)
template <typename T, typename TA, typename TB, int kU, bool kSkip, int kAT>
__device__ __forceinline__ void update_state(const char* sy, const char* sz, uint32_t col_a, uint32_t col_b,
                                             int wave, float total, const float* in, int ydim,
                                             f32x4 (&st)[kAT]) {
  using Frag = typename Mat<T>::Frag;
  const float keep = fast_exp2(total);
#pragma unroll
  for (int at = 0; at < kAT; ++at) st[at] *= keep;
#pragma unroll
  for (int js = 0; js < 2; ++js) {
    Frag fz[kU];
    const f32x8 w = join<float>(*reinterpret_cast<const f32x4*>(in + js * 32),
                                *reinterpret_cast<const f32x4*>(in + js * 32 + 16));
    split<T, kU>(__builtin_convertvector(col_frag<T, TB>(sz, TB::quad_tile(col_b, wave), js * 32), f32x8) * w, fz);
#pragma unroll
    for (int at = 0; at < kAT; ++at) {
      if (kSkip && at * 16 >= ydim) break;
      const Frag fy = col_frag<T, TA>(sy, TA::state_tile(col_a, at), js * 32);
#pragma unroll
      for (int s = 0; s < kU; ++s) st[at] = Mat<T>::mma(fy, fz[s], st[at]);
    }
  }
}

// log2 decays of 64 rows (lane by lane) to what a chunk needs of them: their running
// sum in two float32 terms, the weights of a row's value in the state past the chunk
// and of the state in a row
__device__ __forceinline__ void put_decays(float g, bool ok, int lane, float scale_in, float scale_out,
                                           float* hi, float* lo, float* in, float* out, float* sum) {
  const float d = g * kLog2e;
  const double s = wave_scan(!ok ? 0.0 : d < kLowest ? (double)kLowest : (double)d);  // NaN stays
  const double total = __shfl(s, 63, 64);
  const float h = (float)s, l = (float)(s - h);
  hi[lane] = h;
  lo[lane] = l;
  in[lane] = fast_exp2((float)(total - s)) * scale_in;
  out[lane] = fast_exp2(h) * fmaf(l, kLn2, 1.f) * scale_out;
  if (lane == 0) *sum = (float)total;
}

// kW waves of 16 columns each, of kH heads that share x and y: the workgroup has their
// tiles and x . y once, and z, P, decays and states for each.  kU, kO: bf16 terms of z times its decay and of the
// state as an operand; kDot: row dots with r.
// Two waves a SIMD: two workgroups of four waves a CU, or one of eight, whose tiles
// are in LDS twice (kBuf): the next chunk's go there while this one's are read.
template <typename T, int kA, int kW, int kU, int kO, bool kDot, bool kSummary, int kBuf, int kH>
__global__ __launch_bounds__(64 * kW, kBuf == 2 || sizeof(T) == 2 ? 2 : kW / 4) void linear_attention_kernel(const LaPass p) {
  static_assert(kH == 1 || !kDot, "row dots are of one head");
  using M = Mat<T>;
  using E = typename M::E;
  using Frag = typename M::Frag;
  constexpr int kThreads = 64 * kW, kWh = kW / kH, kB = 16 * kWh, kAT = kA / 16, kAS = kA / 32, kBS = kB / 32;
  // float32 products, 16 times as long, are left out where a block is padding
  constexpr bool kSkip = sizeof(E) == 4;
  using TA = Tile<E, kA>;
  using TB = Tile<E, kB>;
  using TP = Tile<E, kC>;
  constexpr int kState = kA * kB * (int)sizeof(float);
  extern __shared__ __align__(16) char smem[];
  // y, z, then x (not in a summary), r (with kDot); P behind the last buffer
  constexpr int kZ = TA::kBytes, kX = kZ + kH * TB::kBytes, kR = kX + TA::kBytes;
  constexpr int kTiles = kSummary ? kX : kDot ? kR + TB::kBytes : kR;
  char* const sp = smem + kBuf * kTiles;
  __shared__ __align__(16) float s_hi[kBuf][kH][kC], s_lo[kBuf][kH][kC], s_in[kBuf][kH][kC], s_out[kBuf][kH][kC];
  __shared__ float s_total[kBuf][kH], s_dot[kDot ? 2 : 1][kDot ? kW + kW / 4 : 1][kC];

  const int lane = threadIdx.x & 63, wave = wave_id_uniform();
  const int l16 = lane & 15, gq = lane >> 4;
  const int ct = wave % kWh, hw = wave / kWh;  // a wave's 16 columns, of which head
  // Workgroups go to the 8 XCDs in turn: a run of the (batch row, group, segment,
  // head) order to each, so that the heads that share rows share an L2
  int unit = blockIdx.x;
  if (gridDim.x % 8 == 0) unit = unit % 8 * (gridDim.x / 8) + unit / 8;
  const int h_in = unit % (p.rep / kH) * kH + hw;
  unit /= p.rep / kH;
  int seg = unit % p.nseg;
  unit /= p.nseg;
  const int groups = p.heads / p.rep;
  const int b = unit / groups, h = unit % groups * p.rep + h_in;
  if (kSummary) seg = p.reverse ? seg + 1 : seg;  // grid: nseg - 1 segments a head
  const int t0 = seg * p.seg_len, t1 = min(t0 + p.seg_len, p.seqlen);
  const int nchunks = (t1 - t0 + kC - 1) / kC;
  const int step = p.reverse ? -1 : 1;
  const int ydim = p.y.dim, zdim = p.z.dim;
  const int64_t elems = (int64_t)ydim * zdim;
  const int zcol = ct * 16 + l16;
  // valid tokens
  int v0 = 0, v1 = p.seqlen;
  if (p.length) {
    const int64_t n = min(max(p.length[b], (int64_t)0), (int64_t)p.seqlen);
    if (p.pad_right) v1 = (int)n;
    else v0 = p.seqlen - (int)n;
  }

  const int bh = b * p.heads + h;
  const auto head = [&](const LaTensor& x) {
    return static_cast<const E*>(x.p) + (int64_t)b * x.sb + (int64_t)(h / x.rep) * x.sh;
  };
  const E* const px = kSummary ? nullptr : head(p.x);
  const E* const py = head(p.y);
  const E* const pz = head(p.z);
  const E* const pr = kDot ? head(p.r) : nullptr;
  Rows<T, TA, kThreads> rx, ry;
  Rows<T, TB, kThreads / kH> rz, rr;  // a head's z by its own waves
  float dec;
  bool dec_ok;
  ry.init(p.y, p.reverse);
  rz.init(p.z, p.reverse);
  if constexpr (!kSummary) rx.init(p.x, p.reverse);
  if constexpr (kDot) rr.init(p.r, p.reverse);
  // the rows and decays of chunk c, into registers; past the last chunk nothing
  auto fetch = [&](int c) {
    const int first = p.reverse ? t1 - 1 - c * kC : t0 + c * kC;
    const int n = min(kC, t1 - t0 - c * kC);
    const int window = p.reverse ? first - kC + 1 : first;
    const int lo = max(max(window, t0), v0), hi = min(min(window + kC, t1), v1);
    ry.get(p.y, py, window, lo, hi, p.reverse);
    rz.get(p.z, pz, window, lo, hi, p.reverse);
    if constexpr (!kSummary) rx.get(p.x, px, window, lo, hi, p.reverse);
    if constexpr (kDot) rr.get(p.r, pr, window, lo, hi, p.reverse);
    // the decay in front of row `lane`
    const int t = p.reverse ? first - lane + 1 : first + lane;
    dec_ok = lane < n && t >= v0 && t < v1;
    dec = p.g[b * p.g_sb + min(max(t, 0), p.seqlen - 1) * p.g_st + h];
  };
  fetch(0);

  f32x4 st[kAT];
  load_state<T, kA, kB, kThreads / kH>(smem + hw * kState, kSummary || !p.start ? nullptr : p.start + seg * p.start_ss + bh * elems,
                               p.trans, ydim, zdim, zcol, gq, st);
  float seg_total = 0.f;
  uint32_t row_a = TA::row_base(lane), col_a = TA::state_base(lane);
  uint32_t row_b = TB::row_base(lane), col_b = TB::col_base(lane), row_p = TP::row_base(lane);
  uint32_t quad_b = TB::quad_base(lane);
  // a wave computes P's rows i = 16 strip + lane % 16, tiles j half, half + kW / 4, ..;
  // waves 4 apart share a SIMD, so one has a strip of many tiles and one of few
  const int strip = wave < 4 ? wave : 7 - wave, half = wave >> 2;
  const float p_scale = p.scale_in * p.scale_out;

  // chunk c's rows and decays, from registers to buffer c % kBuf, and the loads of
  // the next
  auto put = [&](int c) {
    const int k = c % kBuf;
    char* const t = smem + k * kTiles;
    ry.put(t, ydim);
    rz.put(t + kZ + hw * TB::kBytes, zdim);
    if constexpr (!kSummary) rx.put(t + kX, ydim);
    if constexpr (kDot) rr.put(t + kR, zdim);
    if (ct == 0)
      put_decays(dec, dec_ok, lane, p.scale_in, p.scale_out, s_hi[k][hw], s_lo[k][hw], s_in[k][hw],
                 s_out[k][hw], &s_total[k][hw]);
    fetch(c + 1);
  };
  // chunk c's row dots, from the waves' parts
  auto put_dots = [&](int c) {
    const int n = min(kC, t1 - t0 - c * kC);
    if (wave == 0 && lane < n) {
      float dot = 0.f;
#pragma unroll
      for (int w = 0; w < kW + kW / 4; ++w) dot += s_dot[c & 1][w][lane];
      p.dot[(int64_t)bh * p.seqlen + (p.reverse ? t1 - 1 - c * kC : t0 + c * kC) + step * lane] = dot;
    }
  };
  __syncthreads();  // the start is read
  put(0);

  for (int c = 0; c < nchunks; ++c) {
    // the fragments' addresses are made again in each chunk (an xor each): kept over
    // the loop they cost 30 registers
    asm volatile("" : "+v"(row_a), "+v"(col_a), "+v"(row_b), "+v"(col_b), "+v"(row_p), "+v"(quad_b));
    const int n = min(kC, t1 - t0 - c * kC);
    const int first = p.reverse ? t1 - 1 - c * kC : t0 + c * kC;
    const int mine = first + step * lane;
    const uint64_t mask = __ballot(lane < n && mine >= v0 && mine < v1);
    const int buf = c % kBuf;
    char* const sy = smem + buf * kTiles;
    char* const sz = sy + kZ;
    char* const sx = sy + kX;
    char* const sr = sy + kR;
    __syncthreads();  // this chunk's tiles are written
    if constexpr (kDot) {
      if (c) put_dots(c - 1);
    }

    if constexpr (!kSummary) {
      // P transposed: lane column i, four rows j
      const int i = strip * 16 + l16;
      float own = 0.f;  // sum_j W_ij (x_i . y_j)(r_i . z_j) over this lane's j
      Frag fx[kAS], fr[kDot ? kBS : 1];
#pragma unroll
      for (int ks = 0; ks < kAS; ++ks) fx[ks] = row_frag<T, TA>(sx + strip * 16 * TA::kRow, row_a, ks);
      if constexpr (kDot) {
#pragma unroll
        for (int ks = 0; ks < kBS; ++ks) fr[ks] = row_frag<T, TB>(sr + strip * 16 * TB::kRow, row_b, ks);
      }
#pragma unroll
      for (int k = 0; k < 16 / kW; ++k) {
        const int jt = half + k * (kW / 4);
        if (jt > (strip | 1)) break;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f}, par = {0.f, 0.f, 0.f, 0.f};
        if (jt <= strip) {
          const char* const ty = sy + jt * 16 * TA::kRow;
#pragma unroll
          for (int ks = 0; ks < kAS; ++ks) {
            if (kSkip && ks * 32 >= ydim) break;
            acc = M::mma(row_frag<T, TA>(ty, row_a, ks), fx[ks], acc);
          }
          if constexpr (kDot) {
            const char* const tz = sz + jt * 16 * TB::kRow;
#pragma unroll
            for (int ks = 0; ks < kBS; ++ks) {
              if (kSkip && ks * 32 >= zdim) break;
              par = M::mma(row_frag<T, TB>(tz, row_b, ks), fr[ks], par);
            }
          }
        }
        // the same x . y for all heads
#pragma unroll
        for (int hh = 0; hh < kH; ++hh) {
          f32x4 pij = acc;
          if (jt <= strip) {
            f32x4 d = s_hi[buf][hh][i] - *reinterpret_cast<const f32x4*>(s_hi[buf][hh] + jt * 16 + gq * 4);
            d += s_lo[buf][hh][i] - *reinterpret_cast<const f32x4*>(s_lo[buf][hh] + jt * 16 + gq * 4);
#pragma unroll
            for (int r = 0; r < 4; ++r) pij[r] *= fast_exp2(d[r]) * p_scale;
            if (jt == strip) {
#pragma unroll
              for (int r = 0; r < 4; ++r) pij[r] = gq * 4 + r <= l16 ? pij[r] : 0.f;
            }
            if constexpr (kDot) {
#pragma unroll
              for (int r = 0; r < 4; ++r) own = fmaf(pij[r], par[r], own);
            }
          }
          put_p<T, TP>(sp + hh * kP<T> * TP::kBytes + strip * 16 * TP::kRow + TP::state_tile(row_p, jt), pij);
        }
      }
      if constexpr (kDot) {
        own += __shfl_xor(own, 16, 64);
        own += __shfl_xor(own, 32, 64);
        if (gq == 0) s_dot[c & 1][kW + half][i] = own;
      }
      __syncthreads();  // P is written; the other buffer is read
      if constexpr (kBuf == 2) put(c + 1);

      // out^T: lane column i, four columns z
      f32x4 out[4];
      state_rows<T, TA, kO, kSkip>(sx, row_a, st, ydim, out);
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        out[it] *= s_out[buf][hw][it * 16 + l16];
        if constexpr (kDot) {
          const float dot = quad_dot<T>(sr + it * 16 * TB::kRow + TB::quad_tile(quad_b, wave), out[it]);
          if (gq == 0) s_dot[c & 1][wave][it * 16 + l16] = dot;
        }
      }
      add_chunk<T, TB, TP>(sz + hw * TB::kBytes, sp + hw * kP<T> * TP::kBytes, col_b, row_p, ct, out);
      if (mask != ~0ull) {  // zeros outside the length, whatever the state holds
#pragma unroll
        for (int it = 0; it < 4; ++it)
          if (!((mask >> (it * 16 + l16)) & 1)) out[it] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      const int64_t next = (int64_t)p.heads * zdim, o = (int64_t)b * p.seqlen * next + h * zdim;
      if (p.part) store_rows(p.part + o, out, first, step, n, next, zdim, ct, lane);
      else store_rows(static_cast<E*>(p.out) + o, out, first, step, n, next, zdim, ct, lane);
    } else {
      if constexpr (kBuf == 2) put(c + 1);
    }

    // the state past this chunk
    seg_total += s_total[buf][hw];
    update_state<T, TA, TB, kU, kSkip>(sy, sz + hw * TB::kBytes, col_a, col_b, ct, s_total[buf][hw],
                                       s_in[buf][hw] + gq * 4, ydim, st);
    if constexpr (kBuf == 1) {
      __syncthreads();  // the tiles are read
      put(c + 1);
    }
  }
  if constexpr (kDot) {
    __syncthreads();
    put_dots(nchunks - 1);
  }

  const bool last = p.reverse ? seg == 0 : seg == p.nseg - 1;
  float* dst = nullptr;
  float w = 1.f;
  if constexpr (kSummary) {
    const int slot = p.reverse ? seg - 1 : seg + 1;
    dst = slot == p.slots ? p.end + bh * elems
                          : p.seg_end + ((int64_t)slot * p.batch * p.heads + bh) * elems;
    if (threadIdx.x % (kThreads / kH) == 0) p.seg_decay[(int64_t)slot * p.batch * p.heads + bh] = seg_total;
  } else if (p.end && last) {
    dst = p.end + bh * elems;
    if (p.end_decay) w = fast_exp2(la_log2_decay(p.g, p.g_sb, p.g_st, b, 0, h, v0 == 0 && v1 > 0));
  }
  if (dst) store_state<T, kA, kB, kThreads / kH>(smem + hw * kState, dst, w, p.trans, ydim, zdim, zcol, gq, st);
}

template <typename T, int kA, int kW, int kU, int kO, bool kDot, bool kSummary, int kH = 1>
hipError_t launch_one(const LaPass& p, int blocks, hipStream_t stream) {
  using E = typename Mat<T>::E;
  constexpr int kBuf = sizeof(E) == 2 && kW == 8 ? 2 : 1;
  const size_t tiles = (Tile<E, kA>::kBytes * (kSummary ? 1 : 2) +
                         Tile<E, 16 * kW / kH>::kBytes * (kDot ? 2 : kH)) * kBuf +
                       (kSummary ? 0 : kH * kP<T> * Tile<E, kC>::kBytes);
  // a state passes through the same memory
  const size_t lds = std::max(tiles, (size_t)kA * 16 * kW * sizeof(float));
  auto* kernel = linear_attention_kernel<T, kA, kW, kU, kO, kDot, kSummary, kBuf, kH>;
  if (lds > 48 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  ProfScope prof(kSummary ? "linear_attention_summary" : "linear_attention", stream);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks / kH)), dim3(64 * kW), lds, stream, p);
  return hipGetLastError();
}

template <typename T, int kU, int kO, bool kDot, bool kSummary>
hipError_t launch_dims(const LaPass& p, int blocks, hipStream_t stream) {
  const int a = p.y.dim, b = p.z.dim;
  if (b <= 64) {
    if constexpr (sizeof(T) == 2 && !kDot && !kSummary) {
      // Two heads that share x and y, where that leaves a workgroup for each CU: 4 x
      // 2048 tokens of 32 heads of 128 x 64 over one group 96 -> 89 us forward.  Over
      // 64 rows a head's x . y is not what counts (64 x 64: 66 both ways), nor are
      // there products to share in a summary (30 -> 33).
      if (a > 64 && p.rep % 2 == 0 && blocks >= 512)
        return launch_one<T, 128, 8, kU, kO, kDot, kSummary, 2>(p, blocks, stream);
    }
    if (a <= 32) return launch_one<T, 32, 4, kU, kO, kDot, kSummary>(p, blocks, stream);
    if (a <= 64) return launch_one<T, 64, 4, kU, kO, kDot, kSummary>(p, blocks, stream);
    return launch_one<T, 128, 4, kU, kO, kDot, kSummary>(p, blocks, stream);
  }
  if (a <= 32) return launch_one<T, 32, 8, kU, kO, kDot, kSummary>(p, blocks, stream);
  if (a <= 64) return launch_one<T, 64, 8, kU, kO, kDot, kSummary>(p, blocks, stream);
  return launch_one<T, 128, 8, kU, kO, kDot, kSummary>(p, blocks, stream);
}

}  // namespace la

}  // namespace ssm
