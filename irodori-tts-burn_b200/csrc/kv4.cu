// The 4-bit context cache: quantising rows into it and reading them back.
//
// A group of 32 values of one row of one KV head is s * c, c in [-7, 7], s of
// 5 significant bits: s = min{t : 7 t >= max|x|}.  c = x / s rounded half away
// from zero.  Both are decided by comparisons that are exact in f32: 7 t and
// the borders (c + 1/2) s have at most 9 significant bits, so neither result
// depends on how a quotient was rounded.  c s has at most 8 significant bits:
// it is a bf16 number.
#include "ctx_attn.cuh"

namespace irt {

namespace {

constexpr float KV4_MIN_MAX = 7.88860905e-31f; // 2^-100: smaller groups hold zeros

// Scale of a group with largest magnitude `amax` (finite).
__device__ __forceinline__ float kv4_scale(float amax) {
  if (amax < KV4_MIN_MAX) return 0.f;
  // largest 5-bit number <= amax / 7, then the next one up where 7 s < amax
  const uint32_t t = __float_as_uint(amax / 7.f) & 0xfff80000u;
  float s = __uint_as_float(t);
  if (7.f * s < amax) s = __uint_as_float(t + 0x80000u);
  return fminf(s, __uint_as_float(0x7e100000u));  // 1.125 * 2^125
}

// Code + 8 of x in a group of scale s > 0, inv ~ 1 / s.
__device__ __forceinline__ uint32_t kv4_code(float x, float s, float inv) {
  const float a = fabsf(x);
  float c = rintf(a * inv);
  // a * inv may have been rounded across a border
  if (a >= (c + 0.5f) * s) c += 1.f;
  else if (a < (c - 0.5f) * s) c -= 1.f;
  const int u = (int)fminf(c, 7.f);
  return (uint32_t)(8 + (x < 0.f ? -u : u));
}

struct Kv4Side {
  irt_rows x;
  uint8_t* codes;
  bf16* scales;
  int vec;  // rows of x can be read or written 16 bytes at a time
};
struct Kv4Args {
  Kv4Side side[2];  // K, V
  long rows, row_start, n, src_rows;
  int hd, groups;
  const int* idx;
};

constexpr int KV4_TILE = 64;  // rows of one head per CTA

// Four lanes hold a group, eight values each: its maximum takes two shuffles
// and every lane stores its eight codes as one word.  A CTA covers 64 rows of
// one head, whose codes and scales are contiguous in the cache.  Bound by
// memory: 2 (or 4) bytes a value in, 4.5 bits out.
template <bool BF>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ Kv4Args a) {
  const Kv4Side& sd = a.side[blockIdx.z];
  const int h = blockIdx.y;
  const int octs = 4 * a.groups;  // lanes of a row, the last group's missing ones included
  const long r0 = (long)blockIdx.x * KV4_TILE;
  const int items = KV4_TILE * octs;
#pragma unroll 2
  for (int i = threadIdx.x; i < items; i += 256) {  // items is a multiple of 32: whole warps stay together
    const long r = r0 + i / octs;
    const int o = i % octs;
    long src = -1;
    if (r < a.n) {
      src = a.idx ? a.idx[r] : r;
      if (src >= a.src_rows) src = -1;
    }
    const bool in = src >= 0 && 8 * o < a.hd;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (in) load8<BF>(sd.x.data, src * sd.x.row_stride + h * sd.x.head_stride + 8 * o, sd.vec, x);
    float m = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m = fmaxf(m, fabsf(x[j]));
      bad |= !(fabsf(x[j]) <= 3.402823466e+38f);  // NaN or infinity
    }
    if (bad) m = INFINITY;  // fmaxf drops NaN
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    float s = m == INFINITY ? __uint_as_float(0x7fc00000u) : kv4_scale(m);
    uint32_t w = 0x88888888u;
    if (s > 0.f) {  // not for zero or NaN
      const float inv = 1.f / s;
      w = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) w |= kv4_code(x[j], s, inv) << (4 * j);
    } else if (s != 0.f) {
      w = 0x99999999u;
    }
    if (in) {
      const long row = (long)h * a.rows + a.row_start + r;
      *reinterpret_cast<uint32_t*>(sd.codes + row * (a.hd / 2) + 4 * o) = w;
      if ((o & 3) == 0) sd.scales[row * a.groups + o / 4] = __float2bfloat16_rn(s);
    }
  }
}

template <bool BF>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4Args a) {
  const Kv4Side& sd = a.side[blockIdx.z];
  const int h = blockIdx.y;
  const int octs = a.hd / 8;
  const long r0 = (long)blockIdx.x * KV4_TILE;
  const int items = KV4_TILE * octs;
#pragma unroll 2
  for (int i = threadIdx.x; i < items; i += 256) {
    const long r = r0 + i / octs;
    const int o = i % octs;
    if (r >= a.n) break;
    const long row = (long)h * a.rows + a.row_start + r;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(sd.codes + row * (a.hd / 2) + 4 * o);
    const float s = __bfloat162float(sd.scales[row * a.groups + o / 4]);
    float x[8];
    kv4_unpack8(w, s, x);
    store8<BF>(sd.x.data, r * sd.x.row_stride + h * sd.x.head_stride + 8 * o, sd.vec, x);
  }
}

Kv4Args kv4_args(const irt_kv4_cache& c, int bf16_io, long row_start, long n, const irt_rows& k, const irt_rows& v) {
  Kv4Args a{};
  a.side[0] = {k, c.k_codes, reinterpret_cast<bf16*>(c.k_scales), rows_vec(k, bf16_io)};
  a.side[1] = {v, c.v_codes, reinterpret_cast<bf16*>(c.v_scales), rows_vec(v, bf16_io)};
  a.rows = c.rows;
  a.row_start = row_start;
  a.n = n;
  a.hd = c.head_dim;
  a.groups = kv4_groups(c.head_dim);
  return a;
}

}  // namespace

void kv4_append(const irt_kv4_cache& c, int bf16_io, long row_start, long n, const irt_rows& k, const irt_rows& v,
                long src_rows, const int* idx, cudaStream_t s) {
  if (n <= 0) return;
  Kv4Args a = kv4_args(c, bf16_io, row_start, n, k, v);
  a.src_rows = src_rows;
  a.idx = idx;
  const dim3 grid((unsigned)((n + KV4_TILE - 1) / KV4_TILE), c.kv_heads, 2);
  if (bf16_io) kv4_append_kernel<true><<<grid, 256, 0, s>>>(a);
  else kv4_append_kernel<false><<<grid, 256, 0, s>>>(a);
  IRT_CHECK_LAUNCH();
}

void kv4_read(const irt_kv4_cache& c, int bf16_io, long row_start, long n, const irt_rows& k, const irt_rows& v,
              cudaStream_t s) {
  if (n <= 0) return;
  const Kv4Args a = kv4_args(c, bf16_io, row_start, n, k, v);
  const dim3 grid((unsigned)((n + KV4_TILE - 1) / KV4_TILE), c.kv_heads, 2);
  if (bf16_io) kv4_read_kernel<true><<<grid, 256, 0, s>>>(a);
  else kv4_read_kernel<false><<<grid, 256, 0, s>>>(a);
  IRT_CHECK_LAUNCH();
}

}  // namespace irt
