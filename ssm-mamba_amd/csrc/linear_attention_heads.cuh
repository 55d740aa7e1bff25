// The pass of linear_attention.cuh where its result is a sum over the value heads
// that share a query and key head (dq and dk), in bf16: a workgroup takes kH heads of
// a group, and goes through a chunk head by head.  z and r are the group's own rows,
// loaded once for all heads; the heads' P are added before the product with z, and
// their rows out in the accumulators, so one float32 row leaves for kH heads.  With a
// workgroup a head that row went out for each: 134 MB written and read again for 4 x
// 2048 tokens of 32 heads of 128 x 64 over one group, and z and r were read 32
// times; 95 us and 21 for the sum of the rows, now 88 and 7.  What is left is issue:
// 16 steps a CU of about 5 us, most of it the splits into three terms, some of it
// registers: at 256 of them the compiler spills 38 (108 bytes a lane) and 132 scalar
// ones into vector ones (64 rows, eight waves, with row dots; up to 99 with four waves).
//
// Tiles of x and y are in LDS twice, for this head and the next, those of z and r
// for this chunk and the next: a head costs one barrier.
#pragma once

#include "linear_attention.cuh"

namespace ssm {

namespace la {

template <typename T, int kA, int kW, int kU, int kO, bool kDot, int kH>
__global__ __launch_bounds__(64 * kW, 2) void linear_attention_heads_kernel(const LaPass p) {
  using M = Mat<T>;
  using E = typename M::E;
  using Frag = typename M::Frag;
  constexpr int kThreads = 64 * kW, kB = 16 * kW, kAT = kA / 16, kAS = kA / 32, kBS = kB / 32;
  constexpr int kJ = 16 / kW;  // 16-row tiles of P a wave has
  using TA = Tile<E, kA>;
  using TB = Tile<E, kB>;
  using TP = Tile<E, kC>;
  extern __shared__ __align__(16) char smem[];
  constexpr int kXY = 2 * TA::kBytes, kZR = (kDot ? 2 : 1) * TB::kBytes;
  char* const s_zr = smem + 2 * kXY;
  char* const sp = s_zr + 2 * kZR;
  __shared__ __align__(16) float s_hi[2][kC], s_lo[2][kC], s_in[2][kC], s_out[2][kC];
  __shared__ float s_total[2], s_dot[kDot ? 2 : 1][kDot ? kW + kW / 4 : 1][kC];

  const int lane = threadIdx.x & 63, wave = wave_id_uniform();
  const int l16 = lane & 15, gq = lane >> 4;
  // runs of the (batch row, group, segment, part) order to each of the 8 XCDs
  int unit = blockIdx.x;
  if (gridDim.x % 8 == 0) unit = unit % 8 * (gridDim.x / 8) + unit / 8;
  const int sub = unit % p.subs;
  unit /= p.subs;
  const int seg = unit % p.nseg;
  unit /= p.nseg;
  const int groups = p.heads / p.rep, grp = unit % groups, b = unit / groups;
  const int h0 = grp * p.rep + sub * kH, nh = min(kH, p.rep - sub * kH);
  const int t0 = seg * p.seg_len, t1 = min(t0 + p.seg_len, p.seqlen);
  const int nchunks = (t1 - t0 + kC - 1) / kC;
  const int step = p.reverse ? -1 : 1;
  const int ydim = p.y.dim, zdim = p.z.dim;
  const int64_t elems = (int64_t)ydim * zdim;
  const int zcol = wave * 16 + l16;
  int v0 = 0, v1 = p.seqlen;
  if (p.length) {
    const int64_t n = min(max(p.length[b], (int64_t)0), (int64_t)p.seqlen);
    if (p.pad_right) v1 = (int)n;
    else v0 = p.seqlen - (int)n;
  }
  const auto row_of = [&](const LaTensor& x, int h) {
    return static_cast<const E*>(x.p) + (int64_t)b * x.sb + (int64_t)(h / x.rep) * x.sh;
  };
  const auto first_of = [&](int c) { return p.reverse ? t1 - 1 - c * kC : t0 + c * kC; };
  Rows<T, TA, kThreads> rx, ry;
  Rows<T, TB, kThreads> rz, rr;
  rx.init(p.x, p.reverse);
  ry.init(p.y, p.reverse);
  rz.init(p.z, p.reverse);
  if constexpr (kDot) rr.init(p.r, p.reverse);
  float dec;
  bool dec_ok;
  // into registers: head hh's rows and decays of chunk c; z and r of chunk c.  Past
  // the last chunk nothing.
  auto fetch_xy = [&](int c, int hh) {
    const int first = first_of(c), window = p.reverse ? first - kC + 1 : first;
    const int lo = max(max(window, t0), v0), hi = min(min(window + kC, t1), v1), h = h0 + hh;
    ry.get(p.y, row_of(p.y, h), window, lo, hi, p.reverse);
    rx.get(p.x, row_of(p.x, h), window, lo, hi, p.reverse);
    const int n = min(kC, t1 - t0 - c * kC);
    const int t = p.reverse ? first - lane + 1 : first + lane;
    dec_ok = lane < n && t >= v0 && t < v1;
    dec = p.g[b * p.g_sb + min(max(t, 0), p.seqlen - 1) * p.g_st + h];
  };
  auto fetch_zr = [&](int c) {
    const int first = first_of(c), window = p.reverse ? first - kC + 1 : first;
    const int lo = max(max(window, t0), v0), hi = min(min(window + kC, t1), v1);
    rz.get(p.z, row_of(p.z, h0), window, lo, hi, p.reverse);
    if constexpr (kDot) rr.get(p.r, row_of(p.r, h0), window, lo, hi, p.reverse);
  };
  // step s = c nh + hh, to buffer s % 2, and the loads of the step after
  auto put_xy = [&](int c, int hh) {
    const int k = (c * nh + hh) & 1;
    char* const t = smem + k * kXY;
    ry.put(t, ydim);
    rx.put(t + TA::kBytes, ydim);
    if (wave == 0)
      put_decays(dec, dec_ok, lane, p.scale_in, p.scale_out, s_hi[k], s_lo[k], s_in[k], s_out[k], &s_total[k]);
    fetch_xy(hh + 1 < nh ? c : c + 1, hh + 1 < nh ? hh + 1 : 0);
  };
  auto put_zr = [&](int c) {
    char* const t = s_zr + (c & 1) * kZR;
    rz.put(t, zdim);
    if constexpr (kDot) rr.put(t + TB::kBytes, zdim);
    fetch_zr(c + 1);
  };
  auto put_dots = [&](int c, int hh) {
    const int n = min(kC, t1 - t0 - c * kC);
    if (wave == 0 && lane < n) {
      float dot = 0.f;
#pragma unroll
      for (int w = 0; w < kW + kW / 4; ++w) dot += s_dot[(c * nh + hh) & 1][w][lane];
      p.dot[(int64_t)(b * p.heads + h0 + hh) * p.seqlen + first_of(c) + step * lane] = dot;
    }
  };
  fetch_zr(0);
  fetch_xy(0, 0);
  f32x4 st[kH][kAT];
#pragma unroll
  for (int hh = 0; hh < kH; ++hh) {
    const bool ok = hh < nh && p.start;
    load_state<T, kA, kB, kThreads>(
        smem, ok ? p.start + seg * p.start_ss + (int64_t)(b * p.heads + h0 + hh) * elems : nullptr, p.trans,
        ydim, zdim, zcol, gq, st[hh]);
    __syncthreads();
  }
  uint32_t row_a = TA::row_base(lane), col_a = TA::state_base(lane);
  uint32_t row_b = TB::row_base(lane), col_b = TB::col_base(lane), row_p = TP::row_base(lane);
  uint32_t quad_b = TB::quad_base(lane);
  const int strip = wave < 4 ? wave : 7 - wave, half = wave >> 2;
  const float p_scale = p.scale_in * p.scale_out;
  put_zr(0);
  put_xy(0, 0);

  for (int c = 0; c < nchunks; ++c) {
    asm volatile("" : "+v"(row_a), "+v"(col_a), "+v"(row_b), "+v"(col_b), "+v"(row_p), "+v"(quad_b));
    const int n = min(kC, t1 - t0 - c * kC), first = first_of(c), mine = first + step * lane;
    const uint64_t mask = __ballot(lane < n && mine >= v0 && mine < v1);
    char* const sz = s_zr + (c & 1) * kZR;
    char* const sr = sz + TB::kBytes;
    f32x4 out[4], sum[kJ], par[kJ];
#pragma unroll
    for (int it = 0; it < 4; ++it) out[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kJ; ++k) sum[k] = par[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int hh = 0; hh < kH; ++hh) {
      if (hh >= nh) break;
      const int buf = (c * nh + hh) & 1;
      char* const sy = smem + buf * kXY;
      char* const sx = sy + TA::kBytes;
      __syncthreads();  // this step's tiles are written, the other buffers read
      if constexpr (kDot) {
        if (hh) put_dots(c, hh - 1);
        else if (c) put_dots(c - 1, nh - 1);
        if (hh == 0) {  // r_i . z_j: the heads' own
          Frag fr[kBS];
#pragma unroll
          for (int ks = 0; ks < kBS; ++ks) fr[ks] = row_frag<T, TB>(sr + strip * 16 * TB::kRow, row_b, ks);
#pragma unroll
          for (int k = 0; k < kJ; ++k) {
            const int jt = half + k * (kW / 4);
            if (jt > strip) break;
#pragma unroll
            for (int ks = 0; ks < kBS; ++ks)
              par[k] = M::mma(row_frag<T, TB>(sz + jt * 16 * TB::kRow, row_b, ks), fr[ks], par[k]);
          }
        }
      }
      // this head's part of P, as in linear_attention.cuh
      const int i = strip * 16 + l16;
      const float ihi = s_hi[buf][i], ilo = s_lo[buf][i];
      float own = 0.f;
      Frag fx[kAS];
#pragma unroll
      for (int ks = 0; ks < kAS; ++ks) fx[ks] = row_frag<T, TA>(sx + strip * 16 * TA::kRow, row_a, ks);
#pragma unroll
      for (int k = 0; k < kJ; ++k) {
        const int jt = half + k * (kW / 4);
        if (jt > strip) break;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < kAS; ++ks)
          acc = M::mma(row_frag<T, TA>(sy + jt * 16 * TA::kRow, row_a, ks), fx[ks], acc);
        f32x4 d = ihi - *reinterpret_cast<const f32x4*>(s_hi[buf] + jt * 16 + gq * 4);
        d += ilo - *reinterpret_cast<const f32x4*>(s_lo[buf] + jt * 16 + gq * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] *= fast_exp2(d[r]) * p_scale;
        if (jt == strip) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[r] = gq * 4 + r <= l16 ? acc[r] : 0.f;
        }
        if constexpr (kDot) {
#pragma unroll
          for (int r = 0; r < 4; ++r) own = fmaf(acc[r], par[k][r], own);
        }
        sum[k] += acc;
      }
      if constexpr (kDot) {
        own += __shfl_xor(own, 16, 64);
        own += __shfl_xor(own, 32, 64);
        if (gq == 0) s_dot[buf][kW + half][i] = own;
      }
      if (hh == nh - 1) {  // the heads' sum, and zeros next to an odd diagonal
#pragma unroll
        for (int k = 0; k < kJ; ++k) {
          const int jt = half + k * (kW / 4);
          if (jt > (strip | 1)) break;
          put_p<T, TP>(sp + strip * 16 * TP::kRow + TP::state_tile(row_p, jt), sum[k]);
        }
        put_zr(c + 1);
      }
      put_xy(hh + 1 < nh ? c : c + 1, hh + 1 < nh ? hh + 1 : 0);
      f32x4 part[4];
      state_rows<T, TA, kO, false>(sx, row_a, st[hh], ydim, part);
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        part[it] *= s_out[buf][it * 16 + l16];
        if constexpr (kDot) {
          const float dot = quad_dot<T>(sr + it * 16 * TB::kRow + TB::quad_tile(quad_b, wave), part[it]);
          if (gq == 0) s_dot[buf][wave][it * 16 + l16] = dot;
        }
        out[it] += part[it];
      }
      update_state<T, TA, TB, kU, false>(sy, sz, col_a, col_b, wave, s_total[buf], s_in[buf] + gq * 4, ydim,
                                         st[hh]);
    }
    __syncthreads();  // P is written
    add_chunk<T, TB, TP>(sz, sp, col_b, row_p, wave, out);
    if (mask != ~0ull) {  // zeros outside the length, whatever the states hold
#pragma unroll
      for (int it = 0; it < 4; ++it)
        if (!((mask >> (it * 16 + l16)) & 1)) out[it] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int64_t next = (int64_t)groups * p.subs * zdim;
    store_rows(p.part + (int64_t)b * p.seqlen * next + (grp * p.subs + sub) * zdim, out, first, step, n, next,
               zdim, wave, lane);
  }
  if constexpr (kDot) {
    __syncthreads();
    put_dots(nchunks - 1, nh - 1);
  }
  if (p.end && (p.reverse ? seg == 0 : seg == p.nseg - 1)) {
#pragma unroll
    for (int hh = 0; hh < kH; ++hh) {
      if (hh >= nh) break;
      const int h = h0 + hh;
      float w = 1.f;
      if (p.end_decay) w = fast_exp2(la_log2_decay(p.g, p.g_sb, p.g_st, b, 0, h, v0 == 0 && v1 > 0));
      store_state<T, kA, kB, kThreads>(smem, p.end + (int64_t)(b * p.heads + h) * elems, w, p.trans, ydim, zdim,
                                    zcol, gq, st[hh]);
    }
  }
}

template <typename T, int kA, int kW, int kU, int kO, bool kDot, int kH>
hipError_t launch_heads(const LaPass& p, int blocks, hipStream_t stream) {
  using E = typename Mat<T>::E;
  constexpr size_t tiles = 4 * (size_t)Tile<E, kA>::kBytes + (kDot ? 4 : 2) * (size_t)Tile<E, 16 * kW>::kBytes +
                           kP<T> * (size_t)Tile<E, kC>::kBytes;
  constexpr size_t lds = std::max(tiles, (size_t)kA * 16 * kW * sizeof(float));
  auto* kernel = linear_attention_heads_kernel<T, kA, kW, kU, kO, kDot, kH>;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (e != hipSuccess) return e;
  ProfScope prof("linear_attention_heads", stream);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * kW), lds, stream, p);
  return hipGetLastError();
}

// Four heads to a workgroup, whose states are in its registers, where y has up to 64
// rows, two past that (la_subs())
template <typename T, int kU, int kO, bool kDot>
hipError_t launch_heads_dims(const LaPass& p, int blocks, hipStream_t stream) {
  const int a = p.y.dim, b = p.z.dim;
  if (b <= 64) {
    if (a <= 64) return launch_heads<T, 64, 4, kU, kO, kDot, 4>(p, blocks, stream);
    return launch_heads<T, 128, 4, kU, kO, kDot, 2>(p, blocks, stream);
  }
  if (a <= 64) return launch_heads<T, 64, 8, kU, kO, kDot, 4>(p, blocks, stream);
  return launch_heads<T, 128, 8, kU, kO, kDot, 2>(p, blocks, stream);
}

}  // namespace la

}  // namespace ssm
