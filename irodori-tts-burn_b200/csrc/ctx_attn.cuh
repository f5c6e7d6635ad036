// Row loads and stores shared by the kernels of ctx_attn.cu and kv4.cu.
#pragma once

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

}  // namespace irt
