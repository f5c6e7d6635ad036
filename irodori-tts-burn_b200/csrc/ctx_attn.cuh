// Row loads and stores and the merge of split keys, shared by the kernels of the
// attention over context states.
#pragma once

#include <cooperative_groups.h>

#include "ctx_attn.hpp"

namespace irt {

// Eight values of a row from 16-byte aligned memory, or one by one.
template <bool BF>
__device__ __forceinline__ void load8(const void* base, long off, bool vec, float (&x)[8]) {
  if (BF) {
    const bf16* p = static_cast<const bf16*>(base) + off;
    if (vec) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __bfloat162float(p[i]);
    }
  } else {
    const float* p = static_cast<const float*>(base) + off;
    if (vec) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
  }
}

template <bool BF>
__device__ __forceinline__ void store8(void* base, long off, bool vec, const float (&x)[8]) {
  if (BF) {
    bf16* p = static_cast<bf16*>(base) + off;
    if (vec) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<uint32_t*>(&t);
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(x[i]);
    }
  } else {
    float* p = static_cast<float*>(base) + off;
    if (vec) {
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = x[i];
    }
  }
}

// Whether rows can be read or written 16 bytes at a time.
inline bool rows_vec(const irt_rows& r, int bf16_io) {
  const long per = bf16_io ? 8 : 4;  // elements in 16 bytes
  return (reinterpret_cast<uintptr_t>(r.data) & 15) == 0 && r.row_stride % per == 0 && r.head_stride % per == 0;
}

// Eight codes (one word) of a 4-bit group with scale s.
__device__ __forceinline__ void kv4_unpack8(uint32_t w, float s, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)((int)((w >> (4 * j)) & 15u) - 8) * s;
}

// Joins the partial softmax states of R packed query rows (from row0 on) that
// W warps of each CTA of a cluster hold over their shares of the keys, in a
// fixed order, and writes the rows: out = gate sum_w 2^(m_w - m) O_w /
// sum_w 2^(m_w - m) l_w.  part [W][R][hd], pm (base-2 maxima) and pl (sums)
// [W][R] are this CTA's; cpart [R][hd], cm and cl [R] hold its joined state for
// the cluster.  Called by every thread of every CTA of the cluster, after the
// CTA's warps have written their parts.
template <bool BF, int R, int W>
__device__ __forceinline__ void merge_partials(const CtxAttnParams& p, const irt_attn_seq& sd, int split, int rank,
                                               int hk, int row0, const float* part, const float* pm, const float* pl,
                                               float* cpart, float* cm, float* cl) {
  namespace cg = cooperative_groups;
  constexpr float LN2 = 0.6931471805599453f;
  const int hd = p.hd, G = p.G;
  __syncthreads();
  for (int e = threadIdx.x; e < R * hd; e += 32 * W) {
    const int r = e / hd, d = e % hd;
    float mc = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) mc = fmaxf(mc, pm[w * R + r]);
    const float base = mc == -INFINITY ? 0.f : mc;
    float lc = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = exp2f(pm[w * R + r] - base);
      lc = fmaf(pl[w * R + r], f, lc);
      x = fmaf(part[(w * R + r) * hd + d], f, x);
    }
    cpart[e] = x;
    if (d == 0) {
      cm[r] = mc;
      cl[r] = lc;
    }
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (split > 1) cluster.sync();
  else __syncthreads();
  // each CTA finishes a share of the rows' values
  for (int e = rank * 32 * W + threadIdx.x; e < R * hd; e += split * 32 * W) {
    const int r = e / hd, d = e % hd, pr = row0 + r;
    if (pr >= sd.q_len * G) continue;
    float mt = -INFINITY;
    for (int c = 0; c < split; ++c) mt = fmaxf(mt, split > 1 ? cluster.map_shared_rank(cm, c)[r] : cm[r]);
    const float base = mt == -INFINITY ? 0.f : mt;
    float lt = 0.f, x = 0.f;
    for (int c = 0; c < split; ++c) {
      const float* om = split > 1 ? cluster.map_shared_rank(cm, c) : cm;
      const float* ol = split > 1 ? cluster.map_shared_rank(cl, c) : cl;
      const float* op = split > 1 ? cluster.map_shared_rank(cpart, c) : cpart;
      const float f = exp2f(om[r] - base);
      lt = fmaf(ol[r], f, lt);
      x = fmaf(op[e], f, x);
    }
    x *= lt == 0.f ? 0.f : 1.f / lt;
    const long row = (long)sd.q_start + pr / G;
    const int head = hk * G + pr % G;
    if (p.gate.data) {
      const long off = row * p.gate.row_stride + head * p.gate.head_stride + d;
      x *= BF ? __bfloat162float(static_cast<const bf16*>(p.gate.data)[off])
              : static_cast<const float*>(p.gate.data)[off];
    }
    const long off = row * p.out.row_stride + head * p.out.head_stride + d;
    if (BF) static_cast<bf16*>(p.out.data)[off] = __float2bfloat16_rn(x);
    else static_cast<float*>(p.out.data)[off] = x;
    if (p.lse && d == 0) p.lse[row * p.H + head] = lt == 0.f ? -INFINITY : fmaf(mt, LN2, logf(lt));
  }
  if (split > 1) cluster.sync();  // the others may still read this CTA's part
}

}  // namespace irt
