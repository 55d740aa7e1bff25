// Parameter structs of the linear-attention kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ssm {

constexpr int kLaChunk = 64;    // tokens per chunk
constexpr int kLaMaxDim = 128;  // key and value size

// A (batch, seqlen, heads, dim) operand with a unit inner stride; a value
// head h reads its head h / rep.
struct LaTensor {
  const void* p;     // rows 16-byte aligned and readable to whole 16 bytes
  int64_t sb, st, sh;
  int dim, rep;
};

// One pass out_i = sum_{j <= i} W_ij (x_i . y_j) z_j over one direction of time
// (see linear_attention.cuh).
struct LaPass {
  int batch, seqlen, heads, seg_len, nseg, reverse;
  int rep;                // heads that share rows
  LaTensor x, y, z, r;    // r: the partner of the row dots (p NULL: no dots)
  const float* g;         // log decays
  int64_t g_sb, g_st;     // strides of batch and token (heads adjacent; 0, 0: one per head)
  const int64_t* length;
  int pad_right;
  float scale_in, scale_out;
  // states (batch, heads, ydim, zdim), or (batch, heads, zdim, ydim) with trans
  int trans;
  const float* start;     // of each segment (slot stride: start_ss), or NULL: zero
  int64_t start_ss;
  float* end;             // the state after the last token, or NULL
  int end_decay;          // multiply `end` by the first token's decay (reversed time)
  float* seg_end;         // summary: segment s's own state to slot s + 1 (s - 1 reversed), and to
  int slots;              //   `end` where that is this one
  float* seg_decay;       // summary: (slots + 1, batch * heads) log2 of the segment's decay
  // outputs: (batch, seqlen, heads, zdim) in the streamed type, or (batch, seqlen,
  // groups, subs, zdim) float32, each of a part of a group's heads
  void* out;
  float* part;
  int subs;
  float* dot;             // (batch, heads, seqlen): r_i . out_i
};

// The fold of segment summaries into segment starts, in place.
struct LaFold {
  int bh, nseg, elems, reverse;
  const float* first;     // start of the first segment in time order of the pass, or NULL
  float* slots;           // (nseg, bh, elems)
  const float* decay;     // (nseg, bh) log2; with last nseg + 1
  float* last;            // the last segment's own state, to the last state; or NULL
};

struct LaDecayGrad {
  int batch, seqlen, heads, seg_len, nseg, elems;
  const float *row, *col;         // (batch, heads, seqlen)
  const float* starts;            // forward starts (nseg, bh, elems)
  const float* rstarts;           // reversed starts (nseg, bh, elems)
  const float *last, *dlast;      // (bh, elems) or NULL
  const float* g;
  int64_t g_sb, g_st;
  const int64_t* length;
  int pad_right;
  float* dg;                      // (batch, seqlen, heads), or NULL with
  float* part;                    // (batch * nseg, heads) sums over the segment's tokens
};

struct LaStep {
  int batch, heads, key, value;
  float* state;
  LaTensor q, k, v;               // st unused
  const float* g;
  int64_t g_sb;
  float scale;
  void* out;
};

}  // namespace ssm
