// Attention of few query rows over a 4-bit context cache (bf16, head_dim 64 or
// 128, up to 16 packed query rows a KV head): the newest frames of a stream
// against its context.  tcgen05 unpacks a tile once for up to 128 rows: with 8 /
// 16 / 24 rows, 16 streams over 20000 rows take 184 / 309 / 508 us here and 456
// us there, over 576 rows 14 / 25 / 35 and 22 us, one stream over 576 rows 9 / 9
// / 11 and 12 us.
//
// Bound by reading the cache, 4.5 bits a value, and nearly as much by taking
// the codes apart: 7 integer instructions for 8 codes, 65 % of that pipe at
// 4.95 TB/s (0.75 of the copy peak; 16 streams over 20000 to 32768 rows in
// 205 us; one frame over 576 rows 6.5 us).  Codes go into mma.sync.m16n8k16 as integers
// and the scales, constant over 32 values of a key, are applied to the sums:
//   score(q, j)  = sum_G sK[j][G] * (sum_{d in G} q_d c_jd)
//   out(q, d)    = sum_j (p_qj sV[j][G(d)]) c_jd
// The small products are exact; p sV is rounded to bf16 as p would be.
//
//   codes: a word holds eight codes u = c + 8; (w >> 4i) & 0xf000f are codes i
//     and i + 4, and under the exponent of 128 (16, shifted to bit 3) they are
//     the bf16 pair 136 + c (24 + c): one or two instructions for two values.
//     K: the sum of q over a group's offsets is subtracted from its score sum.
//     V: the offset is subtracted from the pair, which is exact (it would grow
//     with the number of keys in the output).
//   K as the A operand [key][d]: ldmatrix hands lane (g, t) word t of keys g
//     and g + 8 of a group, whose pairs are the k slots of two MMAs; q, the B
//     operand, is laid out alike.
//   V as the A operand [d][key]: ldmatrix.trans hands lane (g, t) the codes
//     4g..4g+3 of keys 2t and 2t + 1 side by side, so each nibble pair is an
//     operand register.  The weights come out of the scores' layout [key][row]
//     by movmatrix.
//
// A warp takes 32 keys at a time through its own ring of asynchronous copies
// (no CTA barrier in the loop); warps and the CTAs of a cluster share the keys
// and join their states at the end.
#include <algorithm>
#include <cmath>

#include "ctx_attn.cuh"
#include "tc_common.cuh"

namespace irt {

namespace {

using tcx::ex2;
using tcx::pack_bf16x2;
using tcx::smem_u32;

constexpr int WARPS = 8, STAGES = 3, KEYS = 32, SUB = KEYS / 16;
// m starts 2^8 above a row's maximum and is raised only when a score passes it:
// weights are at most 1, and weights times scales no larger than the scales.
constexpr int HEADROOM_LOG2 = 8;

template <int NGR>
struct Ring {
  static constexpr int CODES = KEYS * NGR * 16, SCALES = KEYS * NGR * 2;  // bytes of K (and of V)
  static constexpr int OFF_V = CODES, OFF_SK = 2 * CODES;  // then the scales of K and of V
  static constexpr int STAGE = 2 * (CODES + SCALES);
};

struct Kv4RowArgs {
  CtxAttnParams p;
  float scale_log2;
  int split;
  int out_vec;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_small_or_zero(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? BYTES : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// 8 x 8 transpose of 16-bit elements across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Codes i and i + 4 of a word (or code i of two keys' half words) as the bf16
// pair OFF<i> + c: codes 0 and 4 stay in place under the exponent of 128, the
// others are shifted to bit 3 under the exponent of 16.
// exps = {0x43004300, 0x41804180}: registers, so that mask and exponent are
// one three-input instruction.
struct Exponents {
  uint32_t e128 = 0x43004300u, e16 = 0x41804180u;
};
template <int I>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, const Exponents& x) {
  uint32_t r;
  if constexpr (I == 0)
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(r) : "r"(w), "r"(x.e128));  // (a & b) | c
  else
    asm("lop3.b32 %0, %1, 0x00780078, %2, 0xea;" : "=r"(r) : "r"(w >> (4 * I - 3)), "r"(x.e16));
  return r;
}
constexpr float OFF0 = 136.f, OFFX = 24.f;
// Both halves minus an offset.
__device__ __forceinline__ uint32_t sub2(uint32_t x, float off) {
  __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&x), __floats2bfloat162_rn(off, off));
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// N scales at `a` (one key's, or the two of a lane) as f32.
template <int N>
__device__ __forceinline__ void load_scales(uint32_t a, float (&s)[N]) {
  uint32_t w[N / 2];
  if constexpr (N == 4) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(a));
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = (i & 1) ? bf_hi(w[i / 2]) : bf_lo(w[i / 2]);
}

// The ring of one warp: 32 keys a stage.
template <int NGR>
struct Loader {
  using RG = Ring<NGR>;
  static constexpr int HD = 32 * NGR, KPL = 32 / NGR;
  // This lane's chunks of a tile: every KPL-th key from ckey on, one group; and
  // the scales of one K and one V row.
  const CtxAttnParams& p;
  const uint8_t *kptr, *vptr;
  const bf16 *ksp, *vsp;
  uint32_t cdst, sdst;
  int ckey, lane, te, k_len;

  __device__ __forceinline__ Loader(const CtxAttnParams& p_, const irt_attn_seq& sd, int hk, int first, int te_,
                                    uint32_t ring, int lane_)
      : p(p_), lane(lane_), te(te_), k_len(sd.k_len) {
    ckey = lane / NGR;
    const int G = lane % NGR;
    const long row = (long)hk * p.k_rows + sd.k_start + (long)first * KEYS;
    kptr = p.kc + (row + ckey) * (HD / 2) + G * 16;
    vptr = p.vc + (row + ckey) * (HD / 2) + G * 16;
    ksp = p.kscale + (row + lane) * NGR;
    vsp = p.vscale + (row + lane) * NGR;
    // chunks swizzled so that the eight rows of a matrix fall on different banks (the same for keys KPL apart)
    cdst = ring + (ckey * NGR + (NGR == 4 ? G ^ ((ckey >> 1) & 3) : G ^ ((ckey >> 2) & 1))) * 16;
    sdst = ring + RG::OFF_SK + lane * NGR * 2;
  }
  // Starts the copies of a tile (the warp's next one) into a stage.
  __device__ __forceinline__ void issue(int tile, uint32_t stage_off) {
    const int left = k_len - tile * KEYS;
    if (tile < te && left >= KEYS) {
#pragma unroll
      for (int i = 0; i < KEYS / KPL; ++i) {
        cp16(cdst + stage_off + i * KPL * NGR * 16, kptr + i * KPL * (HD / 2));
        cp16(cdst + stage_off + i * KPL * NGR * 16 + RG::OFF_V, vptr + i * KPL * (HD / 2));
      }
      cp_small<2 * NGR>(sdst + stage_off, ksp);
      cp_small<2 * NGR>(sdst + stage_off + RG::SCALES, vsp);
    } else if (tile < te) {  // the last rows: zeros behind them
#pragma unroll
      for (int i = 0; i < KEYS / KPL; ++i) {
        const bool ok = ckey + i * KPL < left;
        cp16_or_zero(cdst + stage_off + i * KPL * NGR * 16, ok ? kptr + i * KPL * (HD / 2) : p.kc, ok);
        cp16_or_zero(cdst + stage_off + i * KPL * NGR * 16 + RG::OFF_V, ok ? vptr + i * KPL * (HD / 2) : p.vc, ok);
      }
      cp_small_or_zero<2 * NGR>(sdst + stage_off, lane < left ? ksp : p.kscale, lane < left);
      cp_small_or_zero<2 * NGR>(sdst + stage_off + RG::SCALES, lane < left ? vsp : p.vscale, lane < left);
    }
    kptr += WARPS * KEYS * (HD / 2);
    vptr += WARPS * KEYS * (HD / 2);
    ksp += WARPS * KEYS * NGR;
    vsp += WARPS * KEYS * NGR;
    cp_commit();
  }
};

// NGR = head_dim / 32 groups.  The eight columns of the score and output
// products are
//   FEW: (query row, group) pairs of R = 8 / NGR packed query rows (2 at
//     head_dim 128).  Column (r, G) of Q holds q in group G and zeros
//     elsewhere, so one accumulator gathers the group sums and a lane scales
//     its own two groups'; column (r, G) of P has p sV[G], and of the product
//     with the codes of group G only the columns of G are kept.
//   otherwise: R = 8 packed query rows, each group's sums in an accumulator of
//     its own.
template <int NGR, bool FEW>
__global__ void __launch_bounds__(32 * WARPS, 2) ctx_attn_kv4_rows_kernel(const __grid_constant__ Kv4RowArgs a) {
  using RG = Ring<NGR>;
  constexpr int HD = 32 * NGR, R = FEW ? 8 / NGR : 8;
  constexpr int NC = FEW ? 1 : 2;  // query rows of a lane's two columns
  const CtxAttnParams& p = a.p;
  irt_attn_seq sd;
  if (!ctx_attn_seq(p, blockIdx.z, sd)) return;
  const int split = a.split, rank = blockIdx.x % split;
  const int row0 = (blockIdx.x / split) * R, nrows = sd.q_len * p.G;
  if (row0 >= nrows) return;  // the whole cluster
  const int hk = blockIdx.y;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const uint32_t ring_s = smem_u32(smem) + warp * STAGES * RG::STAGE;
  const int ntiles = (sd.k_len + KEYS - 1) / KEYS;
  const int tb = (int)((long)ntiles * rank / split), te = (int)((long)ntiles * (rank + 1) / split);
  const int first = tb + warp;
  Loader<NGR> ld(p, sd, hk, first, te, ring_s, lane);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) ld.issue(first + s * WARPS, s * RG::STAGE);

  // q of column g: lane t has values 8t..8t+7 of each group, paired (e, e + 4)
  // as the codes are; bias: minus the codes' offsets times q, summed over the
  // group, of this lane's columns 2t and 2t + 1
  uint32_t qf[NGR][2][2];
  float bias[FEW ? 1 : NGR][2];
  const int qrow = row0 + (FEW ? g / NGR : g);
#pragma unroll
  for (int G = 0; G < NGR; ++G) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (qrow < nrows && (!FEW || g % NGR == G))
      v = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q.data) +
                                          ((long)sd.q_start + qrow / p.G) * p.q.row_stride +
                                          (hk * p.G + qrow % p.G) * p.q.head_stride + 32 * G + 8 * t);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t e = s ? v.y : v.x, f = s ? v.w : v.z;  // values 2s, 2s + 1 and 2s + 4, 2s + 5
      qf[G][s][0] = __byte_perm(e, f, 0x5410);
      qf[G][s][1] = __byte_perm(e, f, 0x7632);
    }
    // values 0 and 4 have the offset OFF0
    float x = OFF0 * (bf_lo(v.x) + bf_lo(v.z)) +
              OFFX * ((bf_hi(v.x) + bf_hi(v.z)) + (bf_lo(v.y) + bf_hi(v.y)) + (bf_lo(v.w) + bf_hi(v.w)));
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    const float b0 = -__shfl_sync(0xffffffffu, x, 8 * t), b1 = -__shfl_sync(0xffffffffu, x, 8 * t + 4);
    if (FEW) {  // a column has one group
      bias[0][0] = G == 0 ? b0 : bias[0][0] + b0;
      bias[0][1] = G == 0 ? b1 : bias[0][1] + b1;
    } else {
      bias[FEW ? 0 : G][0] = b0;
      bias[FEW ? 0 : G][1] = b1;
    }
  }
  Exponents ex;
  asm volatile("" : "+r"(ex.e128), "+r"(ex.e16));  // opaque: they stay in registers

  float o[NGR][2][4];
#pragma unroll
  for (int G = 0; G < NGR; ++G)
#pragma unroll
    for (int i = 0; i < 8; ++i) o[G][i / 4][i % 4] = 0.f;
  float m[NC], l[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
  }
  uint32_t stage_off = 0;
  // ldmatrix row of this lane: matrix lane / 8 = (group of the pair, key half)
  const int lkey = (lane & 7) + ((lane >> 3) & 1) * 8, lG = lane >> 4;
  const uint32_t lrow = ring_s + lkey * NGR * 16;
  const uint32_t lchunk = (NGR == 4 ? lG ^ ((lkey >> 1) & 3) : lG ^ ((lkey >> 2) & 1)) * 16;
  const uint32_t srow = ring_s + RG::OFF_SK + (g * NGR + (FEW ? 2 * t % NGR : 0)) * 2;
  constexpr int NS = FEW ? 2 : NGR;  // scales of a key that a lane uses
  for (int tile = first; tile < te; tile += WARPS) {
    const int left = sd.k_len - tile * KEYS;
    uint32_t on = 0xffffffffu;  // keys that count
    if (left < KEYS) on = (1u << left) - 1;
    if (p.mask) on &= __ballot_sync(0xffffffffu, lane < left && p.mask[(long)sd.k_start + tile * KEYS + lane]);
    cp_wait<STAGES - 2>();
    __syncwarp();

    // scores of keys 16 u + 8 h + g
    float sc[SUB][2][NC];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      float sk[2][NS];
#pragma unroll
      for (int h = 0; h < 2; ++h) load_scales<NS>(srow + stage_off + (16 * u + 8 * h) * NGR * 2, sk[h]);
      float c[4];
#pragma unroll
      for (int hG = 0; hG < NGR / 2; ++hG) {
        uint32_t w[4];
        ldsm4(lrow + stage_off + u * 16 * NGR * 16 + (lchunk ^ (hG << 5)), w);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int G = 2 * hG + x;
          const uint32_t w0 = w[2 * x], w1 = w[2 * x + 1];  // keys g and g + 8
          const uint32_t a0[4] = {code_pair<0>(w0, ex), code_pair<0>(w1, ex), code_pair<1>(w0, ex), code_pair<1>(w1, ex)};
          const uint32_t a1[4] = {code_pair<2>(w0, ex), code_pair<2>(w1, ex), code_pair<3>(w0, ex), code_pair<3>(w1, ex)};
          if (G == 0 || !FEW) mma0(c, a0, qf[G][0][0], qf[G][0][1]);
          else mma(c, a0, qf[G][0][0], qf[G][0][1]);
          mma(c, a1, qf[G][1][0], qf[G][1][1]);
          if constexpr (!FEW) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float& s = sc[u][i / 2][i % 2 % NC];
              s = fmaf(sk[i / 2][G % NS], c[i] + bias[G % (FEW ? 1 : NGR)][i % 2], G == 0 ? 0.f : s);
            }
          }
        }
      }
      if constexpr (FEW) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float s = fmaf(sk[h][0], c[2 * h] + bias[0][0], sk[h][1] * (c[2 * h + 1] + bias[0][1]));
          if (NGR == 4) s += __shfl_xor_sync(0xffffffffu, s, 1);  // the row's other two groups
          sc[u][h][0] = s;
        }
      }
    }
    if (on != 0xffffffffu) {
#pragma unroll
      for (int i = 0; i < 2 * SUB; ++i)
        if (!((on >> (8 * i + g)) & 1)) {
#pragma unroll
          for (int n = 0; n < NC; ++n) sc[i / 2][i % 2][n] = -INFINITY;
        }
    }
    bool raise = false;
    float mx[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      mx[n] = sc[0][0][n];
#pragma unroll
      for (int i = 1; i < 2 * SUB; ++i) mx[n] = fmaxf(mx[n], sc[i / 2][i % 2][n]);
      mx[n] *= a.scale_log2;
      raise |= mx[n] > m[n];
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        float mn = mx[n];
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, w));
        mn = mn > m[n] ? mn + HEADROOM_LOG2 : m[n];
        const float corr = m[n] == mn ? 1.f : ex2(m[n] - mn);
        m[n] = mn;
        l[n] *= corr;
#pragma unroll
        for (int G = 0; G < NGR; ++G)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (FEW || i % 2 == n) o[G][i / 4][i % 4] *= corr;
      }
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      float sv[2][NS];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_scales<NS>(srow + stage_off + RG::SCALES + (16 * u + 8 * h) * NGR * 2, sv[h]);
        if (on != 0xffffffffu && !((on >> (16 * u + 8 * h + g)) & 1)) {  // a masked key's scale may be NaN
#pragma unroll
          for (int i = 0; i < NS; ++i) sv[h][i] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          const float base = m[n] == -INFINITY ? 0.f : -m[n];
          const float e = ex2(fmaf(sc[u][h][n], a.scale_log2, base));
          l[n] += e;
          sc[u][h][n] = e;
        }
      }
      uint32_t b[2];
      if constexpr (FEW) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          b[h] = transpose8(pack_bf16x2(sc[u][h][0] * sv[h][0], sc[u][h][0] * sv[h][1]));
      }
#pragma unroll
      for (int hG = 0; hG < NGR / 2; ++hG) {
        uint32_t w[4];
        ldsm4_trans(lrow + stage_off + RG::OFF_V + u * 16 * NGR * 16 + (lchunk ^ (hG << 5)), w);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int G = 2 * hG + x;
          const uint32_t w0 = w[2 * x], w1 = w[2 * x + 1];  // keys 2t, 2t + 1 and those + 8
          const uint32_t a0[4] = {sub2(code_pair<0>(w0, ex), OFF0), sub2(code_pair<1>(w0, ex), OFFX),
                                  sub2(code_pair<0>(w1, ex), OFF0), sub2(code_pair<1>(w1, ex), OFFX)};
          const uint32_t a1[4] = {sub2(code_pair<2>(w0, ex), OFFX), sub2(code_pair<3>(w0, ex), OFFX),
                                  sub2(code_pair<2>(w1, ex), OFFX), sub2(code_pair<3>(w1, ex), OFFX)};
          if constexpr (!FEW) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              b[h] = transpose8(pack_bf16x2(sc[u][h][0] * sv[h][G % NS], sc[u][h][NC - 1] * sv[h][G % NS]));
          }
          mma(o[G][0], a0, b[0], b[1]);
          mma(o[G][1], a1, b[0], b[1]);
        }
      }
    }
    // the stage that the previous iteration read
    ld.issue(tile + (STAGES - 1) * WARPS, stage_off == 0 ? (STAGES - 1) * RG::STAGE : stage_off - RG::STAGE);
    stage_off = stage_off == (STAGES - 1) * RG::STAGE ? 0 : stage_off + RG::STAGE;
  }
  cp_wait<0>();
  __syncthreads();  // the rings become the partial states

  float* part = reinterpret_cast<float*>(smem);
  float* pm = part + (WARPS + 1) * R * HD;
  float* pl = pm + WARPS * R;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], w);
    const int r = FEW ? 2 * t / NGR : 2 * t + n;
    if (g == 0 && (!FEW || 2 * t % NGR == 0)) {
      pm[warp * R + r] = m[n];
      pl[warp * R + r] = l[n];
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // columns 2t, 2t + 1
    const int col = 2 * t + k, r = FEW ? col / NGR : col;
    float* dst = part + (warp * R + r) * HD + 4 * g;
    if (row0 + r >= nrows) continue;
    if constexpr (FEW) {  // the column's group: k, or 2 + k in odd lanes
      const bool upper = NGR == 4 && (t & 1);
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
        *reinterpret_cast<float2*>(dst + (upper ? 64 : 0) + 32 * k + 2 * mt) =
            make_float2(upper ? o[(2 + k) % NGR][mt][k] : o[k][mt][k],
                        upper ? o[(2 + k) % NGR][mt][2 + k] : o[k][mt][2 + k]);
    } else {
#pragma unroll
      for (int G = 0; G < NGR; ++G)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
          *reinterpret_cast<float2*>(dst + 32 * G + 2 * mt) = make_float2(o[G][mt][k], o[G][mt][2 + k]);
    }
  }
  merge_partials<true, R, WARPS, HEADROOM_LOG2>(p, sd, split, rank, hk, row0, part, a.out_vec);
}

template <int NGR, int R>
void launch(void (*kernel)(Kv4RowArgs), const CtxAttnParams& p, cudaStream_t s) {
  constexpr int HD = 32 * NGR;
  constexpr size_t merge = merge_floats(R, WARPS, HD) * sizeof(float);
  constexpr size_t smem = std::max((size_t)WARPS * STAGES * Ring<NGR>::STAGE, merge);
  Kv4RowArgs a{};
  a.p = p;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  a.out_vec = rows_vec(p.out, 1) && (!p.gate.data || rows_vec(p.gate, 1));
  const int sms = device_sms();
  const long blocks = ((long)p.max_q * p.G + R - 1) / R;
  const long ctas = blocks * p.Hkv * p.nseq;
  // Keys are shared by a cluster where that pays.  Microseconds, of a CTA that
  // starts with the launch 6.8, of one that waits for its place what the work
  // beside it leaves of them; `key` for a key of one head, twice that where two
  // CTAs share an SM, in as many rounds of CTAs as it takes (the last one, if not
  // full, counts the less the more there are); of the longest sequences what they
  // are longer than the mean (the rows of the cache over the sequences); and the
  // merge.  head_dim 128, 1 / 2 / 4 / 8 CTAs, 16 heads of 1 stream over
  // 8192 rows 35.5 / 21.4 / 13.8 / 13.8 us; of 4 streams over 2000 13.0 / 10.3 /
  // 10.5 / 15.5; of 16 over 576 11.2 / 16.3 / 26.5 / 49.4, over 20000 to 32768 215
  // / 209 / 207 / 224.
  const float key = 3.6e-3f * (HD == 64 ? 0.65f : 1.f) * (R == 8 ? 1.25f : 1.f);
  const float places = 2.f * sms, longest = (float)p.max_k, mean = std::min(longest, (float)p.k_rows / p.nseq);
  float best = 0.f;
  for (int n = 1; n <= MAX_SPLIT && (n == 1 || p.max_k > (n / 2) * KEYS * WARPS / 2); n *= 2) {
    const float rounds = ctas * n / places, share = ctas * n > sms ? 2.f : 1.f, one = mean / n * key;
    const float late = std::max(0.f, rounds - 1.f) / (1.f + one * 2.f / 40.f);
    const float all = std::max(1.f, rounds + 0.5f * (std::ceil(rounds) - rounds) / rounds) * one * share +
                      (longest - mean) / n * key;
    const float t = 6.8f * (1.f + late) + std::max(all, longest / n * key * share) + (n > 1 ? 0.8f + 0.15f * n : 0.f);
    if (n == 1 || t < best) {
      best = t;
      a.split = n;
    }
  }
  static std::atomic<uint64_t> told{0};
  allow_smem(kernel, smem, told);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks * a.split), p.Hkv, p.nseq);
  cfg.blockDim = dim3(32 * WARPS);
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

template <int NGR>
void launch_rows(long rows, const CtxAttnParams& p, cudaStream_t s) {
  if (rows <= 8 / NGR) launch<NGR, 8 / NGR>(ctx_attn_kv4_rows_kernel<NGR, true>, p, s);
  else launch<NGR, 8>(ctx_attn_kv4_rows_kernel<NGR, false>, p, s);
}

}  // namespace

bool ctx_attention_kv4_rows(const CtxAttnParams& p, cudaStream_t s) {
  const long rows = (long)p.max_q * p.G;
  // the maximum is taken before the scale, so the scale must be positive
  if (!p.bf16_io || !p.kc || p.ks.data || (p.hd != 64 && p.hd != 128) || rows > 16 || !(p.scale > 0.f) ||
      !rows_vec(p.q, 1))
    return false;
  if (p.hd == 128) launch_rows<4>(rows, p, s);
  else launch_rows<2>(rows, p, s);
  return true;
}

}  // namespace irt
