// The 4-bit context cache: quantising rows into it and reading them back.
//
// A group of 32 values of one row of one KV head is s * c, c in [-7, 7], s of
// 5 significant bits: s = min{t : 7 t >= max|x|}.  c = x / s rounded half away
// from zero.  Both are exact: 7 t and the borders (c + 1/2) s have at most 9
// significant bits, so comparisons with them in f32 decide, and neither result
// depends on how a quotient was rounded.  c s has at most 8 significant bits:
// it is a bf16 number.
#include "ctx_attn.cuh"
#include "tc_common.cuh"

namespace irt {

namespace {

using tcx::f2_add;
using tcx::f2_fma;
using tcx::f2_pack;
using tcx::f2_unpack;

__device__ __forceinline__ uint64_t f2_both(float x) { return f2_pack(__float_as_uint(x), __float_as_uint(x)); }

constexpr float KV4_MIN_MAX = 7.88860905e-31f;  // 2^-100: smaller groups hold zeros
constexpr float MAGIC = 12582912.f;              // 1.5 * 2^23: adding it rounds to a whole number

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Scale of a group with largest magnitude `amax` (finite).
__device__ __forceinline__ float kv4_scale(float amax) {
  if (amax < KV4_MIN_MAX) return 0.f;
  // a 5-bit number at or just below amax / 7, then the next ones up while 7 s < amax
  uint32_t t = __float_as_uint(amax * 0.14285709f) & 0xfff80000u;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (7.f * __uint_as_float(t) < amax) t += 0x80000u;
  return fminf(__uint_as_float(t), __uint_as_float(0x7e100000u));  // 1.125 * 2^125
}

// x / s rounded half away from zero.  inv is a little below 1 / s, so the
// first rounding ends on a border's inner side at worst; the remainder x - c s
// is exact and tells.
__device__ __forceinline__ float kv4_code(float x, float s, float half, float inv) {
  float c = fmaf(x, inv, MAGIC) - MAGIC;
  const float e = fmaf(-c, s, x);
  if (fabsf(e) >= half) c += copysignf(1.f, x);
  return c;
}
// Codes of eight values, plus 8, in one word: four are a whole number below
// 2^16 that f32 multiply-adds put together exactly.
__device__ __forceinline__ uint32_t kv4_pack(const float (&c)[8]) {
  const float lo = fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]) + (MAGIC + 34952.f);  // 0x8888
  const float hi = fmaf(fmaf(fmaf(c[7], 16.f, c[6]), 16.f, c[5]), 16.f, c[4]) + (MAGIC + 34952.f);
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x5410);
}

// Eight bf16 values x as codes of scale s, inv a little above 1 / s (one part in
// 2^20).  x and the borders (c + 1/2) s have at most 8 and 9 significant bits,
// so x is on a border or at least one part in 2^9 away from it: inv takes the
// former outwards and the latter nowhere.  Values i and i + 4 are a packed pair.
__device__ __forceinline__ uint32_t kv4_codes_bf16(uint4 v, float inv) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  const uint64_t inv2 = f2_both(inv), magic = f2_both(MAGIC), back = f2_both(-MAGIC), sixteen = f2_both(16.f);
  uint64_t c[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    c[2 * i] = f2_pack(w[i] << 16, w[i + 2] << 16);
    c[2 * i + 1] = f2_pack(w[i] & 0xffff0000u, w[i + 2] & 0xffff0000u);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = f2_add(f2_fma(c[i], inv2, magic), back);
  const uint64_t word = f2_add(f2_fma(f2_fma(f2_fma(c[3], sixteen, c[2]), sixteen, c[1]), sixteen, c[0]),
                               f2_both(MAGIC + 34952.f));  // 0x8888
  float lo, hi;
  f2_unpack(word, lo, hi);
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x5410);
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
constexpr int KV4_APPEND_THREADS = 128, KV4_READ_THREADS = 256;

// Eight values as they are in memory; zeros where `in` is false.
template <bool BF>
struct Raw {
  uint4 v[BF ? 1 : 2];
};
template <bool BF>
__device__ __forceinline__ void load_raw(const Kv4Side& sd, long off, bool in, Raw<BF>& r) {
  constexpr int N = BF ? 1 : 2;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = make_uint4(0, 0, 0, 0);
  if (!in) return;
  const uint8_t* p = static_cast<const uint8_t*>(sd.x.data) + off * (BF ? 2 : 4);
  if (sd.vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = BF ? (uint32_t) reinterpret_cast<const uint16_t*>(p)[2 * k] |
                        (uint32_t) reinterpret_cast<const uint16_t*>(p)[2 * k + 1] << 16
                  : reinterpret_cast<const uint32_t*>(p)[4 * i + k];
      r.v[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
// Eight f32 values.
__device__ __forceinline__ void expand(const Raw<false>& r, float (&x)[8]) {
  const uint32_t w[8] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w, r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
}

// Largest magnitude of eight values; NaN if one is NaN.
template <bool BF>
__device__ __forceinline__ float amax8(const Raw<BF>& r) {
  if constexpr (BF) {  // two at a time as they are
    const uint32_t a[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
    __nv_bfloat162 m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = a[i] & 0x7fff7fffu;
      m[i] = *reinterpret_cast<const __nv_bfloat162*>(&u);
    }
    const __nv_bfloat162 t = __hmax2_nan(__hmax2_nan(m[0], m[1]), __hmax2_nan(m[2], m[3]));
    return max_nan(__bfloat162float(t.x), __bfloat162float(t.y));
  } else {
    float x[8], m = 0.f;
    expand(r, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(x[j]));
    return m;
  }
}

// Two lanes hold a group, sixteen values each: one shuffle joins its maximum.
// A CTA covers 64 rows of one head (NG groups a row), whose codes and scales
// are contiguous in the cache; a thread's loads are in flight together.  Bound
// by memory and, for bf16, the issue of instructions (2 bytes a value in, 4.5
// bits out): K and V of 25,600 rows of 16 heads of 128 in 54 us, 5.0 TB/s (66 us
// with the f32 values' exact remainders); f32 90 us, 5.3 TB/s; 576 rows 8 us.
template <bool BF, int NG>
__global__ void __launch_bounds__(KV4_APPEND_THREADS) kv4_append_kernel(const __grid_constant__ Kv4Args a) {
  constexpr int HALVES = 2 * NG, N = KV4_TILE * HALVES / KV4_APPEND_THREADS;  // half groups of a row, missing ones included
  constexpr int B = BF ? (N < 4 ? N : 4) : (N < 2 ? N : 2);          // of a thread, in flight
  const Kv4Side& sd = a.side[blockIdx.z];
  const int h = blockIdx.y;
  const long r0 = (long)blockIdx.x * KV4_TILE, head = h * sd.x.head_stride;
  uint8_t* codes = sd.codes + ((long)h * a.rows + a.row_start + r0) * (a.hd / 2);
  bf16* scales = sd.scales + ((long)h * a.rows + a.row_start + r0) * NG;
#pragma unroll 1
  for (int i0 = 0; i0 < N; i0 += B) {
    Raw<BF> raw[B][2];
    bool in[B][2];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int e = threadIdx.x + KV4_APPEND_THREADS * (i0 + i), d = e % HALVES * 16;
      const long r = r0 + e / HALVES;
      long src = -1;
      if (r < a.n && (N % B == 0 || i0 + i < N)) {
        src = a.idx ? a.idx[r] : r;
        if (src >= a.src_rows) src = -1;
      }
      const long off = src * sd.x.row_stride + head + d;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        in[i][u] = src >= 0 && d + 8 * u < a.hd;
        load_raw<BF>(sd, off + 8 * u, in[i][u], raw[i][u]);
      }
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int e = threadIdx.x + KV4_APPEND_THREADS * (i0 + i), half = e % HALVES;
      float m = max_nan(amax8<BF>(raw[i][0]), amax8<BF>(raw[i][1]));
      m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
      float s = kv4_scale(m), inv;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
      // more than rcp.approx is off: one part in 2^20 above, or in 2.5e6 below
      inv *= BF ? 1.00000095f : 0.9999996f;
      float hs = 0.5f * s;
      if (s == 0.f) {  // the values are too small: codes 0
        inv = 0.f;
        hs = INFINITY;
      }
      const bool bad = !(m <= 3.402823466e+38f);  // NaN or infinity
      if (bad) s = __uint_as_float(0x7fc00000u);
      const int row = e / HALVES;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t w;
        if constexpr (BF) {
          w = kv4_codes_bf16(raw[i][u].v[0], inv);
        } else {
          float x[8];
          expand(raw[i][u], x);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = kv4_code(x[j], s, hs, inv);
          w = kv4_pack(x);
        }
        if (bad) w = 0x99999999u;
        if (in[i][u]) *reinterpret_cast<uint32_t*>(codes + row * (a.hd / 2) + half * 8 + 4 * u) = w;
      }
      if (in[i][0] && !(half & 1)) scales[row * NG + half / 2] = __float2bfloat16_rn(s);
    }
  }
}

// A thread has one word of codes of several rows in flight and writes 16
// bytes for each.  Bound by memory: 25,600 rows as above in 49 us, 5.5 TB/s.
template <int NG>
__global__ void __launch_bounds__(KV4_READ_THREADS) kv4_read_bf16_kernel(const __grid_constant__ Kv4Args a) {
  constexpr int OCTS = 4 * NG, N = KV4_TILE * OCTS / KV4_READ_THREADS;
  const Kv4Side& sd = a.side[blockIdx.z];
  const int h = blockIdx.y;
  const long r0 = (long)blockIdx.x * KV4_TILE;
  uint32_t w[N];
  uint16_t sb[N];
  bool in[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = threadIdx.x + KV4_READ_THREADS * i, o = e % OCTS;
    in[i] = r0 + e / OCTS < a.n && 8 * o < a.hd;
    const long row = (long)h * a.rows + a.row_start + r0 + e / OCTS;
    w[i] = in[i] ? *reinterpret_cast<const uint32_t*>(sd.codes + row * (a.hd / 2) + 4 * o) : 0u;
    sb[i] = in[i] ? reinterpret_cast<const uint16_t*>(sd.scales)[row * NG + o / 4] : 0;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = threadIdx.x + KV4_READ_THREADS * i, o = e % OCTS;
    const long r = r0 + e / OCTS;
    if (!in[i]) continue;
    const long off = r * sd.x.row_stride + h * sd.x.head_stride + 8 * o;
    if (sd.vec) {  // the values as the tensor cores get them
      const uint32_t s = (uint32_t)sb[i] << 16 | sb[i];
      const __nv_bfloat162 s2 = *reinterpret_cast<const __nv_bfloat162*>(&s);
      *reinterpret_cast<uint4*>(static_cast<bf16*>(sd.x.data) + off) = kv4_bf16x8<true>(w[i], s2, s2);
    } else {
      float x[8];
      kv4_unpack8(w[i], sb[i], x);
      store8<true>(sd.x.data, off, false, x);
    }
  }
}

// The same into f32: four values a thread, so that the lanes of a store write
// side by side: 88 us, 5.4 TB/s (two 16-byte stores a lane, 32 bytes apart:
// 102 us).
template <int NG>
__global__ void __launch_bounds__(KV4_READ_THREADS) kv4_read_f32_kernel(const __grid_constant__ Kv4Args a) {
  constexpr int QUADS = 8 * NG, N = KV4_TILE * QUADS / KV4_READ_THREADS;
  const Kv4Side& sd = a.side[blockIdx.z];
  const int h = blockIdx.y;
  const long r0 = (long)blockIdx.x * KV4_TILE;
  uint16_t w[N], sb[N];
  bool in[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = threadIdx.x + KV4_READ_THREADS * i, o = e % QUADS;
    in[i] = r0 + e / QUADS < a.n && 4 * o < a.hd;
    const long row = (long)h * a.rows + a.row_start + r0 + e / QUADS;
    w[i] = in[i] ? *reinterpret_cast<const uint16_t*>(sd.codes + row * (a.hd / 2) + 2 * o) : 0;
    sb[i] = in[i] ? reinterpret_cast<const uint16_t*>(sd.scales)[row * NG + o / 8] : 0;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = threadIdx.x + KV4_READ_THREADS * i, o = e % QUADS;
    if (!in[i]) continue;
    const float s = __uint_as_float((uint32_t)sb[i] << 16);
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)  // a code u under the exponent of 2^23 is 2^23 + u
      x[j] = (__uint_as_float(((uint32_t)w[i] >> (4 * j) & 0xfu) | 0x4b000000u) - 8388616.f) * s;
    store4<false>(sd.x.data, (r0 + e / QUADS) * sd.x.row_stride + h * sd.x.head_stride + 4 * o, sd.vec,
                  make_float4(x[0], x[1], x[2], x[3]));
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

template <int NG>
void launch(const Kv4Args& a, int bf16_io, bool read, dim3 grid, cudaStream_t s) {
  if (read) {
    if (bf16_io) kv4_read_bf16_kernel<NG><<<grid, KV4_READ_THREADS, 0, s>>>(a);
    else kv4_read_f32_kernel<NG><<<grid, KV4_READ_THREADS, 0, s>>>(a);
  } else {
    if (bf16_io) kv4_append_kernel<true, NG><<<grid, KV4_APPEND_THREADS, 0, s>>>(a);
    else kv4_append_kernel<false, NG><<<grid, KV4_APPEND_THREADS, 0, s>>>(a);
  }
}

void launch(const Kv4Args& a, int kv_heads, int bf16_io, bool read, cudaStream_t s) {
  using F = void (*)(const Kv4Args&, int, bool, dim3, cudaStream_t);
  static const F by_groups[8] = {launch<1>, launch<2>, launch<3>, launch<4>, launch<5>, launch<6>, launch<7>, launch<8>};
  by_groups[a.groups - 1](a, bf16_io, read, dim3((unsigned)((a.n + KV4_TILE - 1) / KV4_TILE), kv_heads, 2), s);
  IRT_CHECK_LAUNCH();
}

}  // namespace

void kv4_append(const irt_kv4_cache& c, int bf16_io, long row_start, long n, const irt_rows& k, const irt_rows& v,
                long src_rows, const int* idx, cudaStream_t s) {
  if (n <= 0) return;
  Kv4Args a = kv4_args(c, bf16_io, row_start, n, k, v);
  a.src_rows = src_rows;
  a.idx = idx;
  launch(a, c.kv_heads, bf16_io, false, s);
}

void kv4_read(const irt_kv4_cache& c, int bf16_io, long row_start, long n, const irt_rows& k, const irt_rows& v,
              cudaStream_t s) {
  if (n <= 0) return;
  launch(kv4_args(c, bf16_io, row_start, n, k, v), c.kv_heads, bf16_io, true, s);
}

}  // namespace irt
