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

// Eight codes u -> eight bf16 values (u - 8) s, in order.  Under the exponent
// of 16 a code is the bf16 number 16 + u; for a scale of 5 significant bits
// (16 + u) s - 24 s is exact in one fused step, since 24 s has at most 7.  n2 =
// -24 s, twice.  BIG: 24 s is not a bf16 number; (16 + u - 24) s in two steps,
// the second one rounded where s has more than 5 bits.
template <bool BIG>
__device__ __forceinline__ uint4 kv4_bf16x8(uint32_t w, __nv_bfloat162 s2, __nv_bfloat162 n2) {
  const uint32_t lo = ((w << 3) & 0x78787878u) | 0x80808080u;                        // codes 0 2 4 6, low bytes
  const uint32_t hi = ((w >> 1) & 0x78787878u) | 0x80808080u;                        // codes 1 3 5 7
  const uint32_t a = __byte_perm(lo, hi, 0x5140), b = __byte_perm(lo, hi, 0x7362);  // 0 1 2 3 / 4 5 6 7
  uint32_t r[4] = {__byte_perm(a, 0x41414141u, 0x4140), __byte_perm(a, 0x41414141u, 0x4342),
                   __byte_perm(b, 0x41414141u, 0x4140), __byte_perm(b, 0x41414141u, 0x4342)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 u = *reinterpret_cast<__nv_bfloat162*>(&r[i]);
    const __nv_bfloat162 v = BIG ? __hmul2(__hsub2(u, __floats2bfloat162_rn(24.f, 24.f)), s2) : __hfma2(u, s2, n2);
    r[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Eight codes (one word) of a 4-bit group with scale s, bf16 bits `sb`: exact
// in f32 for every s.  A code u under the exponent of 2^23 is 2^23 + u.
__device__ __forceinline__ void kv4_unpack8(uint32_t w, uint16_t sb, float (&x)[8]) {
  const float s = __uint_as_float((uint32_t)sb << 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (__uint_as_float((w >> (4 * i) & 0xfu) | 0x4b000000u) - 8388616.f) * s;
}

// SMs of the current device, looked up once per device.
inline int device_sms() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  IRT_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  IRT_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}
// Lets a kernel use `bytes` of dynamic shared memory on the current device;
// `done` is the kernel's own mask of the devices it has been told on.
template <class K>
void allow_smem(K kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  IRT_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit & done.load(std::memory_order_relaxed)) return;
  IRT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
}

// Four values of a row of the output (or gate).
template <bool BF>
__device__ __forceinline__ float4 load4(const void* base, long off, bool vec) {
  if (BF) {
    const bf16* p = static_cast<const bf16*>(base) + off;
    if (vec) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                         __uint_as_float(u.y & 0xffff0000u));
    }
    return make_float4(__bfloat162float(p[0]), __bfloat162float(p[1]), __bfloat162float(p[2]), __bfloat162float(p[3]));
  }
  const float* p = static_cast<const float*>(base) + off;
  if (vec) return *reinterpret_cast<const float4*>(p);
  return make_float4(p[0], p[1], p[2], p[3]);
}
template <bool BF>
__device__ __forceinline__ void store4(void* base, long off, bool vec, float4 x) {
  if (BF) {
    bf16* p = static_cast<bf16*>(base) + off;
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    if (vec) {
      *reinterpret_cast<uint2*>(p) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
      p[0] = a.x; p[1] = a.y; p[2] = b.x; p[3] = b.y;
    }
  } else {
    float* p = static_cast<float*>(base) + off;
    if (vec) {
      *reinterpret_cast<float4*>(p) = x;
    } else {
      p[0] = x.x; p[1] = x.y; p[2] = x.z; p[3] = x.w;
    }
  }
}

constexpr int MAX_SPLIT = 8;  // CTAs of a cluster that share a query block's keys

// Shared memory of merge_partials in floats: part [W][R][hd], the CTA's own
// joined rows [R][hd], and maxima, sums and weights.
constexpr __host__ __device__ int merge_floats(int R, int W, int hd) { return (W + 1) * R * hd + (3 * W + 2) * R; }

// Joins the partial softmax states of the packed query rows [row0, row0 + R)
// that W warps of each CTA of a cluster hold over their shares of the keys, in
// a fixed order, and writes the rows:
//   out = gate sum_w 2^(m_w - m) O_w / sum_w 2^(m_w - m) l_w.
// sm: part [W][R][hd], then pm [W][R] (base-2 maxima) and pl [W][R] (sums),
// written by the warps; the rest is used here.  16-byte aligned.  Called by
// every thread of every CTA of the cluster.  vec: rows of out and gate can be
// accessed four values at a time.  HEADROOM: how far (log2) the m_w lie above
// the maxima; the log of the sum moves it over, so that it loses nothing to it.
template <bool BF, int R, int W, int HEADROOM = 0>
__device__ __forceinline__ void merge_partials(const CtxAttnParams& p, const irt_attn_seq& sd, int split, int rank,
                                               int hk, int row0, float* sm, bool vec) {
  namespace cg = cooperative_groups;
  constexpr float LN2 = 0.6931471805599453f;
  const int hd = p.hd, G = p.G, rows = min(R, sd.q_len * G - row0), q4 = hd / 4;
  float* cpart = sm + W * R * hd;  // joined rows; before them the parts, behind them the statistics
  float* pm = cpart + R * hd;
  float* pl = pm + W * R;
  float* pf = pl + W * R;
  float* cm = pf + W * R;
  float* cl = cm + R;
  __syncthreads();
  for (int e = threadIdx.x; e < W * rows; e += 32 * W) {
    const int r = e / W, w = e % W;
    float mc = -INFINITY;
#pragma unroll
    for (int i = 0; i < W; ++i) mc = fmaxf(mc, pm[i * R + r]);
    const float base = mc == -INFINITY ? 0.f : mc;
    pf[w * R + r] = exp2f(pm[w * R + r] - base);
    if (w == 0) {
      float lc = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) lc = fmaf(pl[i * R + r], exp2f(pm[i * R + r] - base), lc);
      cm[r] = mc;
      cl[r] = lc;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * q4; e += 32 * W) {
    const int r = e / q4, d = e % q4 * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = pf[w * R + r];
      const float4 o = *reinterpret_cast<const float4*>(sm + (w * R + r) * hd + d);
      x.x = fmaf(o.x, f, x.x);
      x.y = fmaf(o.y, f, x.y);
      x.z = fmaf(o.z, f, x.z);
      x.w = fmaf(o.w, f, x.w);
    }
    *reinterpret_cast<float4*>(cpart + r * hd + d) = x;
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (split > 1) cluster.sync();
  else __syncthreads();
  // each CTA finishes a share of the rows' values
  for (int e = rank * 32 * W + threadIdx.x; e < rows * q4; e += split * 32 * W) {
    const int r = e / q4, d = e % q4 * 4, pr = row0 + r;
    float om[MAX_SPLIT], ol[MAX_SPLIT];
    float4 o[MAX_SPLIT];
    float mt = -INFINITY;
#pragma unroll
    for (int c = 0; c < MAX_SPLIT; ++c)
      if (c < split) {
        om[c] = split > 1 ? cluster.map_shared_rank(cm, c)[r] : cm[r];
        ol[c] = split > 1 ? cluster.map_shared_rank(cl, c)[r] : cl[r];
        o[c] = *reinterpret_cast<const float4*>((split > 1 ? cluster.map_shared_rank(cpart, c) : cpart) + r * hd + d);
        mt = fmaxf(mt, om[c]);
      }
    const float base = mt == -INFINITY ? 0.f : mt;
    float lt = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < MAX_SPLIT; ++c)
      if (c < split) {
        const float f = exp2f(om[c] - base);
        lt = fmaf(ol[c], f, lt);
        x.x = fmaf(o[c].x, f, x.x);
        x.y = fmaf(o[c].y, f, x.y);
        x.z = fmaf(o[c].z, f, x.z);
        x.w = fmaf(o[c].w, f, x.w);
      }
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
    const long row = (long)sd.q_start + pr / G;
    const int head = hk * G + pr % G;
    if (p.gate.data) {
      const float4 g = load4<BF>(p.gate.data, row * p.gate.row_stride + head * p.gate.head_stride + d, vec);
      x.x *= g.x; x.y *= g.y; x.z *= g.z; x.w *= g.w;
    }
    store4<BF>(p.out.data, row * p.out.row_stride + head * p.out.head_stride + d, vec, x);
    if (p.lse && d == 0)
      p.lse[row * p.H + head] =
          lt == 0.f ? -INFINITY : fmaf(mt - HEADROOM, LN2, logf(lt * (float)(1 << HEADROOM)));
  }
  if (split > 1) cluster.sync();  // the others may still read this CTA's part
}

}  // namespace irt
