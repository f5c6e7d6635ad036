// Attention of few query rows over a 4-bit context cache (bf16, head_dim 64 or
// 128, up to 16 packed query rows a KV head): the newest frames of a stream
// against its context.
//
// Bound by reading the cache: 4.5 bits a value, so a value may cost no more
// than two or three instructions.  Codes go into mma.sync.m16n8k16 as integers
// and the scales, constant over 32 values of a key, are applied to the sums:
//   score(q, j)  = sum_G sK[j][G] * (sum_{d in G} q_d c_jd)
//   out(q, d)    = sum_j (p_qj sV[j][G(d)]) c_jd
// The small products are exact; p sV is rounded to bf16 as p would be.
//
//   codes: a word holds eight codes u = c + 8; (w >> 4i) & 0xf000f are codes i
//     and i + 4, and shifted to bit 3 under the exponent of 16 they are the
//     bf16 pair 16 + u.  The sum over d of q (24 + c) is started at -24 sum(q)
//     (K); 24 is subtracted exactly where the error would not cancel (V).
//   K as the B operand [d][key]: ldmatrix hands lane (g, t) word t of key g of
//     a group, whose pairs are the k slots of two MMAs; q is laid out alike.
//   V as the A operand [d][key]: ldmatrix.trans hands lane (g, t) the codes
//     4g..4g+3 of keys 2t and 2t + 1 side by side, so each nibble pair is an
//     operand register; the scores' registers are the B operand as they are.
//
// A warp takes 16 keys at a time through its own ring of asynchronous copies
// (no CTA barrier in the loop); warps and the CTAs of a cluster share the keys
// and join their states at the end.
#include <algorithm>

#include "ctx_attn.cuh"
#include "tc_common.cuh"

namespace irt {

namespace {

using tcx::ex2;
using tcx::pack_bf16x2;
using tcx::smem_u32;

constexpr int WARPS = 8, STAGES = 4, KEYS = 16;
constexpr float RESCALE_LOG2 = 8.f;  // raise the running maximum only beyond 2^8 growth

template <int NGR>
struct Ring {
  static constexpr int CODES = KEYS * NGR * 16, SCALES = KEYS * NGR * 2;  // bytes of K (and of V)
  static constexpr int OFF_V = CODES, OFF_SK = 2 * CODES, OFF_SV = OFF_SK + SCALES;
  static constexpr int STAGE = 2 * (CODES + SCALES);
};

struct Kv4RowArgs {
  CtxAttnParams p;
  float scale_log2;
  int split;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src, bool ok) {
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

// Codes i and i + 4 of a word (or code i of two keys' half words) as the bf16
// pair 16 + u.
template <int I>
__device__ __forceinline__ uint32_t pair16(uint32_t w) {
  const uint32_t x = I == 0 ? w << 3 : w >> (4 * I - 3);
  return (x & 0x00780078u) | 0x41804180u;
}
// The same as c = u - 8.
template <int I>
__device__ __forceinline__ uint32_t pair_c(uint32_t w) {
  uint32_t x = pair16<I>(w);
  __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&x), __floats2bfloat162_rn(24.f, 24.f));
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Scales of keys 2t and 2t + 1 (both halves of the 16 keys): s[half][key][G].
template <int NGR>
__device__ __forceinline__ void load_scales(const uint8_t* base, int t, float (&s)[2][2][NGR]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[NGR];
    const uint8_t* a = base + (8 * h + 2 * t) * NGR * 2;
    if constexpr (NGR == 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(a);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(a);
      w[0] = v.x; w[1] = v.y;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int G = 0; G < NGR; ++G) {
        const uint32_t x = w[(k * NGR + G) / 2];
        s[h][k][G] = (G & 1) ? bf_hi(x) : bf_lo(x);
      }
  }
}

// NGR = head_dim / 32 groups, NQ = packed query rows / 8.
template <int NGR, int NQ>
__global__ void __launch_bounds__(32 * WARPS, 2) ctx_attn_kv4_rows_kernel(const __grid_constant__ Kv4RowArgs a) {
  using RG = Ring<NGR>;
  constexpr int HD = 32 * NGR, R = 8 * NQ;
  const CtxAttnParams& p = a.p;
  irt_attn_seq sd;
  if (!ctx_attn_seq(p, blockIdx.z, sd)) return;
  const int split = a.split, rank = blockIdx.x % split;
  const int row0 = (blockIdx.x / split) * R, nrows = sd.q_len * p.G;
  if (row0 >= nrows) return;  // the whole cluster
  const int hk = blockIdx.y;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  uint8_t* ring = smem + warp * STAGES * RG::STAGE;
  const uint32_t ring_s = smem_u32(ring);

  // q of rows g (and g + 8): lane t has values 8t..8t+7 of each group, paired
  // (e, e + 4) as the codes are
  uint32_t qf[NGR][2][4];
  float bias[NGR][NQ];  // -24 sum of q over the group
#pragma unroll
  for (int G = 0; G < NGR; ++G) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      uint4 v = make_uint4(0, 0, 0, 0);
      const int pr = row0 + g + 8 * n;
      if (n < NQ && pr < nrows)
        v = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q.data) +
                                            ((long)sd.q_start + pr / p.G) * p.q.row_stride +
                                            (hk * p.G + pr % p.G) * p.q.head_stride + 32 * G + 8 * t);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t e = s ? v.y : v.x, f = s ? v.w : v.z;  // values 2s, 2s + 1 and 2s + 4, 2s + 5
        qf[G][s][n] = __byte_perm(e, f, 0x5410);
        qf[G][s][n + 2] = __byte_perm(e, f, 0x7632);
      }
      if (n < NQ) {
        float x = (bf_lo(v.x) + bf_hi(v.x)) + (bf_lo(v.y) + bf_hi(v.y)) + (bf_lo(v.z) + bf_hi(v.z)) +
                  (bf_lo(v.w) + bf_hi(v.w));
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        bias[G][n] = -24.f * x;
      }
    }
  }

  const int ntiles = (sd.k_len + KEYS - 1) / KEYS;
  const int tb = (int)((long)ntiles * rank / split), te = (int)((long)ntiles * (rank + 1) / split);
  const long head_row = (long)hk * p.k_rows + sd.k_start;
  auto issue = [&](int tile, int stage) {
    if (tile < te) {
      const uint32_t dst = ring_s + stage * RG::STAGE;
      const int k0 = tile * KEYS;
#pragma unroll
      for (int i = 0; i < KEYS * NGR / 32; ++i) {
        const int c = lane + 32 * i, key = c / NGR, G = c % NGR;
        const bool ok = k0 + key < sd.k_len;
        const long off = (head_row + k0 + (ok ? key : 0)) * (HD / 2) + G * 16;
        // 16-byte chunks swizzled so that the eight rows of a matrix fall on different banks
        const int sw = NGR == 4 ? G ^ ((key >> 1) & 3) : G ^ ((key >> 2) & 1);
        cp16(dst + (key * NGR + sw) * 16, p.kc + off, ok);
        cp16(dst + RG::OFF_V + (key * NGR + sw) * 16, p.vc + off, ok);
      }
      const int key = lane % 16;
      const bool ok = k0 + key < sd.k_len;
      const bf16* sc = (lane < 16 ? p.kscale : p.vscale) + (head_row + k0 + (ok ? key : 0)) * NGR;
      cp_small<2 * NGR>(dst + (lane < 16 ? RG::OFF_SK : RG::OFF_SV) + key * NGR * 2, sc, ok);
    }
    cp_commit();
  };
  float o[NQ][NGR][2][4];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
#pragma unroll
    for (int G = 0; G < NGR; ++G)
#pragma unroll
      for (int i = 0; i < 8; ++i) o[n][G][i / 4][i % 4] = 0.f;
    m[n] = -INFINITY;
    l[n] = 0.f;
  }
  const int first = tb + warp;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(first + s * WARPS, s);
  int stage = 0;
  // ldmatrix row of this lane: matrix lane / 8 = (group of the pair, key half)
  const int lkey = (lane & 7) + ((lane >> 3) & 1) * 8, lG = lane >> 4;
  for (int tile = first; tile < te; tile += WARPS) {
    const int k0 = tile * KEYS;
    uint32_t on = 0xffffu;  // keys that count
    if (p.mask) on = __ballot_sync(0xffffffffu, lane < KEYS && k0 + lane < sd.k_len && p.mask[(long)sd.k_start + k0 + lane]);
    else if (sd.k_len - k0 < KEYS) on = (1u << (sd.k_len - k0)) - 1;
    cp_wait<STAGES - 2>();
    __syncwarp();
    const uint32_t st = ring_s + stage * RG::STAGE;
    const uint8_t* sb = ring + stage * RG::STAGE;

    // scores of keys 2t, 2t + 1 (+ 8) for query rows g (and g + 8)
    float sc[NQ][2][2];
    {
      float sk[2][2][NGR];
      load_scales<NGR>(sb + RG::OFF_SK, t, sk);
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][i / 2][i % 2] = 0.f;
#pragma unroll
      for (int hG = 0; hG < NGR / 2; ++hG) {
        const int G0 = 2 * hG + lG;
        const int sw = NGR == 4 ? G0 ^ ((lkey >> 1) & 3) : G0 ^ ((lkey >> 2) & 1);
        uint32_t w[4];
        ldsm4(st + (lkey * NGR + sw) * 16, w);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int G = 2 * hG + x / 2, h = x % 2;
          float c[4] = {bias[G][0], bias[G][0], bias[G][NQ - 1], bias[G][NQ - 1]};
          mma(c, qf[G][0], pair16<0>(w[x]), pair16<1>(w[x]));
          mma(c, qf[G][1], pair16<2>(w[x]), pair16<3>(w[x]));
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) sc[n][h][k] = fmaf(sk[h][k][G], c[2 * n + k], sc[n][h][k]);
        }
      }
    }
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float& s = sc[n][i / 2][i % 2];
        s *= a.scale_log2;
        if (on != 0xffffu && !((on >> (8 * (i / 2) + 2 * t + i % 2)) & 1)) s = -INFINITY;
        mx = fmaxf(mx, s);
      }
      raise |= mx > m[n] + RESCALE_LOG2 || (m[n] == -INFINITY && mx > -INFINITY);
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float mx = fmaxf(fmaxf(sc[n][0][0], sc[n][0][1]), fmaxf(sc[n][1][0], sc[n][1][1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx = fmaxf(mx, m[n]);
        const float corr = m[n] == -INFINITY ? 0.f : ex2(m[n] - mx);
        m[n] = mx;
        l[n] *= corr;
        // the outputs' columns are query rows 2t and 2t + 1
        const float c0 = __shfl_sync(0xffffffffu, corr, 8 * t), c1 = __shfl_sync(0xffffffffu, corr, 8 * t + 4);
#pragma unroll
        for (int G = 0; G < NGR; ++G)
#pragma unroll
          for (int i = 0; i < 8; ++i) o[n][G][i / 4][i % 4] *= (i & 1) ? c1 : c0;
      }
    }
    float sv[2][2][NGR];
    load_scales<NGR>(sb + RG::OFF_SV, t, sv);
    if (on != 0xffffu) {  // a masked key's scale may be NaN
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!((on >> (8 * (i / 2) + 2 * t + i % 2)) & 1)) {
#pragma unroll
          for (int G = 0; G < NGR; ++G) sv[i / 2][i % 2][G] = 0.f;
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float base = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = ex2(sc[n][i / 2][i % 2] - base);
        sc[n][i / 2][i % 2] = e;
        l[n] += e;
      }
    }
#pragma unroll
    for (int hG = 0; hG < NGR / 2; ++hG) {
      const int G0 = 2 * hG + lG;
      const int sw = NGR == 4 ? G0 ^ ((lkey >> 1) & 3) : G0 ^ ((lkey >> 2) & 1);
      uint32_t w[4];
      ldsm4_trans(st + RG::OFF_V + (lkey * NGR + sw) * 16, w);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int G = 2 * hG + x;
        const uint32_t w0 = w[2 * x], w1 = w[2 * x + 1];  // keys 2t, 2t + 1 and those + 8
        const uint32_t a0[4] = {pair_c<0>(w0), pair_c<1>(w0), pair_c<0>(w1), pair_c<1>(w1)};
        const uint32_t a1[4] = {pair_c<2>(w0), pair_c<3>(w0), pair_c<2>(w1), pair_c<3>(w1)};
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const uint32_t b0 = pack_bf16x2(sc[n][0][0] * sv[0][0][G], sc[n][0][1] * sv[0][1][G]);
          const uint32_t b1 = pack_bf16x2(sc[n][1][0] * sv[1][0][G], sc[n][1][1] * sv[1][1][G]);
          mma(o[n][G][0], a0, b0, b1);
          mma(o[n][G][1], a1, b0, b1);
        }
      }
    }
    issue(tile + (STAGES - 1) * WARPS, stage == 0 ? STAGES - 1 : stage - 1);
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  }
  cp_wait<0>();
  __syncthreads();  // the rings become the partial states

  float* part = reinterpret_cast<float*>(smem);
  float* pm = part + WARPS * R * HD;
  float* pl = pm + WARPS * R;
  float* cpart = pl + WARPS * R;
  float* cm = cpart + R * HD;
  float* cl = cm + R;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float ls = l[n];
    ls += __shfl_xor_sync(0xffffffffu, ls, 1);
    ls += __shfl_xor_sync(0xffffffffu, ls, 2);
    if (t == 0) {
      pm[warp * R + 8 * n + g] = m[n];
      pl[warp * R + 8 * n + g] = ls;
    }
#pragma unroll
    for (int G = 0; G < NGR; ++G)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int d = 32 * G + 4 * g + 2 * mt;
        const float* c = o[n][G][mt];
        float* dst = part + (warp * R + 8 * n + 2 * t) * HD + d;
        *reinterpret_cast<float2*>(dst) = make_float2(c[0], c[2]);
        *reinterpret_cast<float2*>(dst + HD) = make_float2(c[1], c[3]);
      }
  }
  merge_partials<true, R, WARPS>(p, sd, split, rank, hk, row0, part, pm, pl, cpart, cm, cl);
}

template <int NGR, int NQ>
void launch(const CtxAttnParams& p, cudaStream_t s) {
  constexpr int R = 8 * NQ, HD = 32 * NGR;
  constexpr size_t merge = ((WARPS + 1) * R * HD + 2 * (WARPS + 1) * R) * sizeof(float);
  constexpr size_t smem = std::max((size_t)WARPS * STAGES * Ring<NGR>::STAGE, merge);
  Kv4RowArgs a{};
  a.p = p;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  int dev = 0, sms = 0;
  IRT_CUDA(cudaGetDevice(&dev));
  IRT_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const long blocks = ((long)p.max_q * p.G + R - 1) / R;
  const long ctas = blocks * p.Hkv * p.nseq;
  a.split = 1;
  while (a.split < 8 && ctas * a.split * 2 <= 8L * sms && p.max_k >= 2L * a.split * WARPS * KEYS) a.split *= 2;
  auto kernel = ctx_attn_kv4_rows_kernel<NGR, NQ>;
  IRT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
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

}  // namespace

bool ctx_attention_kv4_rows(const CtxAttnParams& p, cudaStream_t s) {
  const long rows = (long)p.max_q * p.G;
  if (!p.bf16_io || !p.kc || p.ks.data || (p.hd != 64 && p.hd != 128) || rows > 16 || !rows_vec(p.q, 1)) return false;
  if (p.hd == 128) {
    if (rows <= 8) launch<4, 1>(p, s);
    else launch<4, 2>(p, s);
  } else {
    if (rows <= 8) launch<2, 1>(p, s);
    else launch<2, 2>(p, s);
  }
  return true;
}

}  // namespace irt
