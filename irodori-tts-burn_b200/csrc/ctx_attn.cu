// Attention over context states: argument checks, choice of kernel, and the
// row kernel that handles every type, head dimension, stride and alignment.
//
//   out_i = gate_i * sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - m_i)
//
// over a sequence's own rows (if given) and its allowed context rows, native
// or 4-bit.  One pass over the keys with a running maximum and sum; keys are
// split over lanes, warps and the CTAs of a cluster, whose partial
// (maximum, sum, output) triples are merged in a fixed order: results do not
// depend on timing, and no workspace is needed.
#include <algorithm>
#include <numeric>
#include <type_traits>

#include "ctx_attn.cuh"
#include "tc_common.cuh"

namespace irt {

namespace {

using tcx::ex2;
using tcx::f2_add;
using tcx::f2_fma;
using tcx::f2_pack;
using tcx::f2_unpack;

constexpr float LOG2E = 1.4426950408889634f;

constexpr int ROW_WARPS = 8;

struct RowArgs {
  CtxAttnParams p;
  int lanes;  // lanes that share a key: a power of two >= head_dim / (8 VC)
  int split;  // CTAs of a cluster over the keys of one row block
  int q_vec, k_vec, v_vec, ks_vec, vs_vec, out_vec;
  int wide;  // a lane's two chunks of codes are one load
};

// Eight values as packed pairs.
__device__ __forceinline__ void pairs(const float (&x)[8], uint64_t (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = f2_pack(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]));
}
// Eight codes u as pairs of f32 u - 8, exact: a code under the exponent of 2^23
// is 2^23 + u.
__device__ __forceinline__ void code_pairs(uint32_t w, uint64_t (&r)[4]) {
  const uint64_t off = f2_pack(0xcb000008u, 0xcb000008u);  // -(2^23 + 8)
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = f2_add(f2_pack(((w >> (8 * i)) & 0xfu) | 0x4b000000u, ((w >> (8 * i + 4)) & 0xfu) | 0x4b000000u), off);
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float bf_value(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// R packed query rows (query x grouped head) of one KV head per CTA.  A key is
// held by `lanes` lanes, VC chunks of eight values each; a warp works on
// 32 / lanes keys at a time, U of them in flight per lane group, each group
// with its own running maximum.  4-bit context: a lane's chunks are side by
// side within a group of 32, whose scale goes to the score and to the weight;
// the codes of the next keys are read meanwhile.
template <bool BF, bool CTX4, int R, int U, int VC>
__global__ void __launch_bounds__(32 * ROW_WARPS, 2) ctx_attn_rows_kernel(const __grid_constant__ RowArgs a) {
  const CtxAttnParams& p = a.p;
  irt_attn_seq sd;
  if (!ctx_attn_seq(p, blockIdx.z, sd)) return;
  const int split = a.split, rank = blockIdx.x % split;
  const int hk = blockIdx.y, G = p.G, hd = p.hd;
  const int row0 = (blockIdx.x / split) * R;
  if (row0 >= sd.q_len * G) return;  // the whole cluster
  extern __shared__ __align__(16) float sm[];
  // states of the warps, see merge_partials
  float* part = sm;
  float* pm = part + (ROW_WARPS + 1) * R * hd;
  float* pl = pm + ROW_WARPS * R;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int LK = a.lanes, sub = lane / LK, o = lane % LK, per = 32 / LK;
  auto at = [&](int c) { return 8 * (CTX4 ? o * VC + c : o + LK * c); };  // first value of a chunk
  const float qscale = p.scale * LOG2E;
  uint64_t q[R][VC][4], acc[R][VC][4];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int pr = row0 + r;
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
      if (at(c) < hd && pr < sd.q_len * G)
        load8<BF>(p.q.data, (sd.q_start + pr / G) * p.q.row_stride + (hk * G + pr % G) * p.q.head_stride + at(c), a.q_vec,
                  x);
      pairs(x, q[r][c]);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][c][i] = 0;
    }
    m[r] = -INFINITY;
    l[r] = 0.f;
  }

  // U keys of each lane group: scores times ks, weights times vs
  auto step = [&](const uint64_t (&k)[U][VC][4], const float (&ks)[U], const uint64_t (&v)[U][VC][4],
                  const float (&vs)[U], const bool (&ok)[U], auto scaled) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s[U];
      float mx = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint64_t d2 = 0;
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) d2 = f2_fma(q[r][c][i], k[u][c][i], d2);
        float d, d1;
        f2_unpack(d2, d, d1);
        d += d1;
        if (scaled) d *= ks[u];
        for (int w = LK / 2; w > 0; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
        s[u] = ok[u] ? d * qscale : -INFINITY;
        mx = fmaxf(mx, s[u]);
      }
      const float base = mx == -INFINITY ? 0.f : mx;  // NaN scores stay NaN in p and the sum
      if (__any_sync(0xffffffffu, mx > m[r])) {
        const float corr = ex2(m[r] - base);
        m[r] = mx;
        l[r] *= corr;
        const uint64_t c2 = f2_pack(__float_as_uint(corr), __float_as_uint(corr));
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][c][i] = f2_mul(acc[r][c][i], c2);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = ex2(s[u] - base), f = scaled ? e * vs[u] : e;
        l[r] += e;
        const uint64_t f2 = f2_pack(__float_as_uint(f), __float_as_uint(f));
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][c][i] = f2_fma(f2, v[u][c][i], acc[r][c][i]);
      }
    }
  };
  const int chunk = per * U, first = (rank * ROW_WARPS + warp) * chunk + sub, stride = split * ROW_WARPS * chunk;
  const float one[U] = {};
  // native rows: the own ones (keys [0, q_len), unmasked), or the context
  auto native = [&](const irt_rows& kr, const irt_rows& vr, int k_vec, int v_vec, long start, int n, const uint8_t* mask) {
    for (int j0 = first; j0 - sub < n; j0 += stride) {
      uint64_t k[U][VC][4], v[U][VC][4];
      bool ok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * per;
        const long row = start + j;
        ok[u] = j < n && (!mask || mask[row]);
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          float x[8], y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
          if (ok[u] && at(c) < hd) {
            load8<BF>(kr.data, row * kr.row_stride + hk * kr.head_stride + at(c), k_vec, x);
            load8<BF>(vr.data, row * vr.row_stride + hk * vr.head_stride + at(c), v_vec, y);
          }
          pairs(x, k[u][c]);
          pairs(y, v[u][c]);
        }
      }
      step(k, one, v, one, ok, std::false_type{});
    }
  };
  if (p.ks.data) native(p.ks, p.vs, a.ks_vec, a.vs_vec, sd.q_start, sd.q_len, nullptr);
  if constexpr (!CTX4) {
    native(p.k, p.v, a.k_vec, a.v_vec, sd.k_start, sd.k_len, p.mask);
  } else {
    const int groups = kv4_groups(hd);
    struct {
      uint32_t k[U][VC], v[U][VC];
      uint16_t ks[U], vs[U];
      bool ok[U];
    } next;
    auto words = [&](const uint8_t* codes, bool in, uint32_t (&w)[VC]) {
#pragma unroll
      for (int c = 0; c < VC; ++c) w[c] = 0;
      if (!in) return;
      if (VC == 2 && a.wide) {
        const uint2 x = *reinterpret_cast<const uint2*>(codes);
        w[0] = x.x; w[1 % VC] = x.y;
      } else {
#pragma unroll
        for (int c = 0; c < VC; ++c)
          if (at(c) < hd) w[c] = *reinterpret_cast<const uint32_t*>(codes + 4 * c);
      }
    };
    auto fetch = [&](int j0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * per;
        const long row = (long)sd.k_start + j, cr = (long)hk * p.k_rows + row;
        next.ok[u] = j < sd.k_len && (!p.mask || p.mask[row]);
        const bool in = next.ok[u] && at(0) < hd;
        words(p.kc + cr * (hd / 2) + at(0) / 2, in, next.k[u]);
        words(p.vc + cr * (hd / 2) + at(0) / 2, in, next.v[u]);
        next.ks[u] = in ? reinterpret_cast<const uint16_t*>(p.kscale)[cr * groups + at(0) / KV4_GROUP] : 0;
        next.vs[u] = in ? reinterpret_cast<const uint16_t*>(p.vscale)[cr * groups + at(0) / KV4_GROUP] : 0;
      }
    };
    if (first - sub < sd.k_len) fetch(first);
    for (int j0 = first; j0 - sub < sd.k_len; j0 += stride) {
      const auto cur = next;
      if (j0 - sub + stride < sd.k_len) fetch(j0 + stride);
      uint64_t k[U][VC][4], v[U][VC][4];
      float ks[U], vs[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ks[u] = bf_value(cur.ks[u]);
        vs[u] = bf_value(cur.vs[u]);
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          code_pairs(cur.k[u][c], k[u][c]);
          code_pairs(cur.v[u][c], v[u][c]);
        }
      }
      step(k, ks, v, vs, cur.ok, std::true_type{});
    }
  }

  // lane groups of the warp
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float mw = m[r];
    for (int w = LK; w < 32; w <<= 1) mw = fmaxf(mw, __shfl_xor_sync(0xffffffffu, mw, w));
    const float f = ex2(m[r] - (mw == -INFINITY ? 0.f : mw));
    float lw = l[r] * f;
    for (int w = LK; w < 32; w <<= 1) lw += __shfl_xor_sync(0xffffffffu, lw, w);
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x, y;
        f2_unpack(acc[r][c][i], x, y);
        x *= f;
        y *= f;
        for (int w = LK; w < 32; w <<= 1) {
          x += __shfl_xor_sync(0xffffffffu, x, w);
          y += __shfl_xor_sync(0xffffffffu, y, w);
        }
        if (sub == 0 && at(c) < hd)
          *reinterpret_cast<float2*>(part + (warp * R + r) * hd + at(c) + 2 * i) = make_float2(x, y);
      }
    if (lane == 0) {
      pm[warp * R + r] = mw;
      pl[warp * R + r] = lw;
    }
  }
  merge_partials<BF, R, ROW_WARPS>(p, sd, split, rank, hk, row0, sm, a.out_vec);
}

template <bool BF, bool CTX4, int R, int U, int VC>
void launch_rows(const CtxAttnParams& p, cudaStream_t s) {
  RowArgs a{};
  a.p = p;
  a.lanes = 1;
  while (a.lanes * VC < p.hd / 8) a.lanes *= 2;
  a.q_vec = rows_vec(p.q, BF);
  a.k_vec = rows_vec(p.k, BF);
  a.v_vec = rows_vec(p.v, BF);
  a.ks_vec = rows_vec(p.ks, BF);
  a.vs_vec = rows_vec(p.vs, BF);
  a.out_vec = rows_vec(p.out, BF) && (!p.gate.data || rows_vec(p.gate, BF));
  a.wide = p.hd % 16 == 0;
  const long blocks = ((long)p.max_q * p.G + R - 1) / R;
  const long ctas = blocks * p.Hkv * p.nseq;
  const long keys = (long)p.max_k + (p.ks.data ? p.max_q : 0);
  // Keys are split over a cluster while there are fewer than two CTAs per SM
  // and every warp keeps a chunk (one query over 200 / 576 f32 rows 7.2 / 9.2
  // us, 8.6 / 9.4 with two chunks, 7.6 / 9.4 with half a one).
  const int sms = device_sms();
  const long least = 2L * ROW_WARPS * U * (32 / a.lanes);
  a.split = 1;
  while (a.split < MAX_SPLIT && ctas * a.split * 2 <= 2L * sms && keys >= a.split * least) a.split *= 2;
  const size_t smem = (size_t)merge_floats(R, ROW_WARPS, p.hd) * sizeof(float);
  auto kernel = ctx_attn_rows_kernel<BF, CTX4, R, U, VC>;  // smem <= 37.3 KB (R = 4, head_dim 256)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks * a.split), p.Hkv, p.nseq);
  cfg.blockDim = dim3(32 * ROW_WARPS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)a.split, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  IRT_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  IRT_CHECK_LAUNCH();
}

// Rows, keys in flight and chunks as measured, all with two CTAs an SM: 16
// streams of 16 heads of 128 over 8192 f32 rows with 1 / 2 / 4 queries 324 / 392
// / 611 us (reading them 328 us), without the split of U and VC by R 557 / 896 /
// 1066; 4-bit rows 202 / 264 / 590 us (reading them 46 us: bound by unpacking
// and multiplying in f32), one utterance of 576 9.4 / 11.6 / 13.9.  Twice the
// chunks a lane took 175 / 243 / 531, but 11.0 / 14.5 / 27.4 there.
template <bool BF>
void rows_path(const CtxAttnParams& p, cudaStream_t s) {
  const long rows = (long)p.max_q * p.G;
  if (p.kc) {
    if (rows == 1) launch_rows<BF, true, 1, 2, 2>(p, s);
    else if (rows == 2) launch_rows<BF, true, 2, 1, 2>(p, s);
    else launch_rows<BF, true, 4, 1, 1>(p, s);
  } else {
    if (rows == 1) launch_rows<BF, false, 1, 3, 1>(p, s);
    else if (rows == 2) launch_rows<BF, false, 2, 3, 1>(p, s);
    else launch_rows<BF, false, 4, 2, 1>(p, s);
  }
}

// ---- argument checks -------------------------------------------------------

// Rows of a tensor: a sequence's own and context rows together stay below 2^31.
constexpr long MAX_ROWS = (1L << 30) - 1;

Error arg_error(const std::string& m) { return Error(IRT_E_INVALID_ARG, m); }

// First and one-past-last byte of a tensor.  For rows of heads also the windows
// that its bytes repeat in: every byte is in [lo + i period, + extent) for some
// i, with the step that rows and heads share, that of the rows, and that of the
// heads as the period (0: no such window).
struct Span {
  uintptr_t lo, hi;
  struct {
    uintptr_t period, extent;
  } win[3];
};
Span span_of(const irt_rows& r, long rows, int heads, int hd, int esz) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(r.data);
  if (!r.data || rows <= 0) return {lo, lo, {}};
  // a stride that nothing steps by says nothing
  const long row = rows > 1 ? r.row_stride : 0, head = heads > 1 ? r.head_stride : 0;
  const uintptr_t in_row = (heads - 1) * head + hd, in_head = (rows - 1) * row + hd;
  Span s{lo, lo + ((rows - 1) * row + in_row) * esz, {}};
  s.win[0] = {(uintptr_t)std::gcd(row, head) * esz, (uintptr_t)hd * esz};
  s.win[1] = {(uintptr_t)row * esz, in_row * esz};
  s.win[2] = {(uintptr_t)head * esz, in_head * esz};
  return s;
}
Span span_of(const void* data, long bytes) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(data);
  return {lo, data ? lo + bytes : lo, {}};
}
bool overlap(const Span& a, const Span& b) {
  if (a.lo == a.hi || b.lo == b.hi || a.lo >= b.hi || b.lo >= a.hi) return false;
  // inside one tensor: apart where windows of the same period lie side by side
  for (const auto& x : a.win)
    for (const auto& y : b.win) {
      const uintptr_t p = x.period;
      if (p == 0 || p != y.period) continue;
      const uintptr_t d = b.lo >= a.lo ? (b.lo - a.lo) % p : (p - (a.lo - b.lo) % p) % p;
      if (d >= x.extent && d + y.extent <= p) return false;
    }
  return true;
}

void check_rows(const char* name, const irt_rows& r, long rows, int heads, int esz) {
  if (!r.data && rows > 0) throw arg_error(std::string(name) + " is NULL");
  if (reinterpret_cast<uintptr_t>(r.data) % esz) throw arg_error(std::string(name) + " is not aligned to its type");
  if (r.row_stride < 0 || r.head_stride < 0) throw shape_error(std::string(name) + " has a negative stride");
  // a tensor of more than 2^48 elements is a mistake, and keeps 64-bit offsets from overflowing
  const long lim = 1L << 48;
  if (r.row_stride > lim || r.head_stride > lim || (rows > 0 && r.row_stride > lim / rows) ||
      (heads > 0 && r.head_stride > lim / heads))
    throw shape_error(std::string(name) + " has a stride beyond 2^48 elements");
}

// A tensor that is written must not overlap itself.
void check_own(const char* name, const irt_rows& r, long rows, int heads, int hd) {
  const bool row_major = (heads == 1 || r.head_stride >= hd) &&
                         (rows <= 1 || r.row_stride >= (heads - 1) * r.head_stride + hd);
  const bool head_major = (rows <= 1 || r.row_stride >= hd) &&
                          (heads == 1 || r.head_stride >= (rows - 1) * r.row_stride + hd);
  if (!row_major && !head_major) throw shape_error(std::string(name) + "'s rows overlap one another");
}

void check_heads(int heads, int kv_heads, int hd) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads)
    throw shape_error("heads " + std::to_string(heads) + " must be a positive multiple of kv_heads " +
                      std::to_string(kv_heads));
  if (kv_heads > 65535) throw shape_error("at most 65535 KV heads");
  if (hd < 8 || hd > 256 || hd % 8)
    throw shape_error("head_dim " + std::to_string(hd) + " must be a multiple of 8 in 8..256");
}

}  // namespace

void kv4_check_cache(const irt_kv4_cache& c) {
  check_heads(c.kv_heads, c.kv_heads, c.head_dim);
  if (c.rows < 0 || c.rows > MAX_ROWS) throw shape_error("cache rows " + std::to_string(c.rows) + " out of range");
  const void* const ps[4] = {c.k_codes, c.k_scales, c.v_codes, c.v_scales};
  for (const void* q : ps) {
    if (!q && c.rows > 0) throw arg_error("a cache buffer is NULL");
    if (reinterpret_cast<uintptr_t>(q) & 15) throw arg_error("cache buffers must be aligned to 16 bytes");
  }
}

namespace {

constexpr const char* KV4_NAMES[4] = {"k_codes", "k_scales", "v_codes", "v_scales"};
void kv4_spans(const irt_kv4_cache& c, Span (&s)[4]) {
  const long n = c.rows * c.kv_heads, codes = n * (c.head_dim / 2), scales = n * kv4_groups(c.head_dim) * 2;
  s[0] = span_of(c.k_codes, codes);
  s[1] = span_of(c.k_scales, scales);
  s[2] = span_of(c.v_codes, codes);
  s[3] = span_of(c.v_scales, scales);
}

}  // namespace

void kv4_check_rows(const irt_kv4_cache& c, int dtype, long row_start, long n, const irt_rows& k, const irt_rows& v,
                    long ext_rows, const int* idx, bool written) {
  if (dtype != IRT_PREC_BF16 && dtype != IRT_PREC_F32) throw arg_error("dtype must be an irt_precision");
  kv4_check_cache(c);
  if (row_start < 0 || n < 0 || row_start > c.rows || n > c.rows - row_start)
    throw shape_error("rows [" + std::to_string(row_start) + ", " + std::to_string(row_start) + " + " +
                      std::to_string(n) + ") are outside the cache's " + std::to_string(c.rows));
  if (ext_rows < 0 || ext_rows > MAX_ROWS) throw shape_error("source rows must be in 0..2^30 - 1");
  const int esz = dtype == IRT_PREC_BF16 ? 2 : 4;
  check_rows("k", k, ext_rows, c.kv_heads, esz);
  check_rows("v", v, ext_rows, c.kv_heads, esz);
  if (written) {
    check_own("k", k, ext_rows, c.kv_heads, c.head_dim);
    check_own("v", v, ext_rows, c.kv_heads, c.head_dim);
  }
  const Span sk = span_of(k, ext_rows, c.kv_heads, c.head_dim, esz), sv = span_of(v, ext_rows, c.kv_heads, c.head_dim, esz);
  if (written && overlap(sk, sv)) throw arg_error("k overlaps v");
  Span buf[4];
  kv4_spans(c, buf);
  if (reinterpret_cast<uintptr_t>(idx) % 4) throw arg_error("the source index must be aligned to 4 bytes");
  const Span si = span_of(idx, 4 * n);
  for (int i = 0; i < 4; ++i) {
    const std::string name = std::string("the cache's ") + KV4_NAMES[i];
    if (overlap(sk, buf[i])) throw arg_error("k overlaps " + name);
    if (overlap(sv, buf[i])) throw arg_error("v overlaps " + name);
    if (overlap(si, buf[i])) throw arg_error("the source index overlaps " + name);
    for (int j = 0; j < i && !written; ++j)
      if (overlap(buf[j], buf[i])) throw arg_error(std::string(KV4_NAMES[j]) + " overlaps " + name);
  }
}

CtxAttnParams ctx_attn_params(const irt_attn_args& a, const irt_kv4_cache* cache, const irt_rows* k,
                              const irt_rows* v, long k_rows, const irt_rows* k_self, const irt_rows* v_self) {
  if (a.dtype != IRT_PREC_BF16 && a.dtype != IRT_PREC_F32) throw arg_error("dtype must be an irt_precision");
  check_heads(a.heads, a.kv_heads, a.head_dim);
  if (a.num_seqs < 0 || a.num_seqs > 65535) throw shape_error("num_seqs must be in 0..65535");
  if (a.max_q_len < 0 || a.max_k_len < 0) throw shape_error("max_q_len and max_k_len must not be negative");
  if (a.q_rows < 0 || k_rows < 0 || a.q_rows > MAX_ROWS || k_rows > MAX_ROWS)
    throw shape_error("q_rows and the context rows must be in 0..2^30 - 1");
  if ((long)a.max_q_len * (a.heads / a.kv_heads) > (1L << 26)) throw shape_error("max_q_len is too large");
  const float s2 = a.scale * LOG2E;  // as the kernels use it
  if (s2 - s2 != 0.f) throw arg_error("scale must be finite, and below 2^127");
  if (!a.seqs && ((long)a.num_seqs * a.max_q_len > a.q_rows || (long)a.num_seqs * a.max_k_len > k_rows))
    throw shape_error("without a sequence table q needs num_seqs * max_q_len rows and the context num_seqs * max_k_len");
  const bool bf = a.dtype == IRT_PREC_BF16;
  const int esz = bf ? 2 : 4;
  CtxAttnParams p{};
  p.bf16_io = bf;
  p.H = a.heads;
  p.Hkv = a.kv_heads;
  p.hd = a.head_dim;
  p.G = a.heads / a.kv_heads;
  p.nseq = a.num_seqs;
  p.max_q = a.max_q_len;
  p.max_k = a.max_k_len;
  p.scale = a.scale;
  p.q_rows = a.q_rows;
  p.k_rows = k_rows;
  p.seqs = a.seqs;
  p.q = a.q;
  p.gate = a.gate;
  p.out = a.out;
  p.mask = a.key_mask;
  p.lse = a.lse;
  check_rows("q", a.q, a.q_rows, a.heads, esz);
  check_rows("out", a.out, a.q_rows, a.heads, esz);
  check_own("out", a.out, a.q_rows, a.heads, a.head_dim);
  if (a.gate.data) check_rows("gate", a.gate, a.q_rows, a.heads, esz);
  const Span so = span_of(a.out, a.q_rows, a.heads, a.head_dim, esz), sl = span_of(a.lse, a.q_rows * a.heads * 4);
  if (reinterpret_cast<uintptr_t>(a.lse) % 4 || reinterpret_cast<uintptr_t>(a.seqs) % 4)
    throw arg_error("lse and seqs must be aligned to 4 bytes");
  auto apart_span = [&](const char* name, const Span& x) {
    if (overlap(so, x)) throw arg_error("out overlaps " + std::string(name));
    if (overlap(sl, x)) throw arg_error("lse overlaps " + std::string(name));
  };
  auto apart = [&](const char* name, const irt_rows& r, long rows, int heads) {
    apart_span(name, span_of(r, rows, heads, a.head_dim, esz));
  };
  if (overlap(so, sl)) throw arg_error("out overlaps lse");
  apart_span("key_mask", span_of(a.key_mask, k_rows));
  apart_span("seqs", span_of(a.seqs, a.num_seqs * (long)sizeof(irt_attn_seq)));
  apart("q", a.q, a.q_rows, a.heads);
  apart("gate", a.gate, a.q_rows, a.heads);
  if (cache) {
    kv4_check_cache(*cache);
    if (cache->kv_heads != a.kv_heads || cache->head_dim != a.head_dim)
      throw shape_error("the cache holds " + std::to_string(cache->kv_heads) + " heads of " +
                        std::to_string(cache->head_dim) + ", the call has " + std::to_string(a.kv_heads) + " of " +
                        std::to_string(a.head_dim));
    Span buf[4];
    kv4_spans(*cache, buf);
    for (int i = 0; i < 4; ++i) apart_span(KV4_NAMES[i], buf[i]);
    p.kc = cache->k_codes;
    p.vc = cache->v_codes;
    p.kscale = reinterpret_cast<const bf16*>(cache->k_scales);
    p.vscale = reinterpret_cast<const bf16*>(cache->v_scales);
  } else {
    check_rows("k", *k, k_rows, a.kv_heads, esz);
    check_rows("v", *v, k_rows, a.kv_heads, esz);
    apart("k", *k, k_rows, a.kv_heads);
    apart("v", *v, k_rows, a.kv_heads);
    p.k = *k;
    p.v = *v;
  }
  const bool s0 = k_self && k_self->data, s1 = v_self && v_self->data;
  if (s0 != s1) throw missing_input("k_self and v_self go together");
  if (s0) {
    check_rows("k_self", *k_self, a.q_rows, a.kv_heads, esz);
    check_rows("v_self", *v_self, a.q_rows, a.kv_heads, esz);
    apart("k_self", *k_self, a.q_rows, a.kv_heads);
    apart("v_self", *v_self, a.q_rows, a.kv_heads);
    p.ks = *k_self;
    p.vs = *v_self;
  }
  return p;
}

void ctx_attention(const CtxAttnParams& p, cudaStream_t s) {
  if (p.nseq == 0 || p.max_q == 0 || p.q_rows == 0) return;
  if (ctx_attention_kv4_rows(p, s) || ctx_attention_tc(p, s) || ctx_attention_tile(p, s)) return;
  if (p.bf16_io) rows_path<true>(p, s);
  else rows_path<false>(p, s);
}

}  // namespace irt
