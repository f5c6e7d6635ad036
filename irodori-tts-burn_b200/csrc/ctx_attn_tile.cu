// Attention over context states in f32 arithmetic for many query rows: the f32
// mode, and bf16 tensors that the tcgen05 kernel does not take (strides or
// bases that are not multiples of 16 bytes, a scale that is not positive).
// head_dim <= 128.
//
// One CTA = 64 (32) packed query rows (query x grouped head) of one KV head, in
// tiles of 64 keys; 256 threads as 16 x 16, each with 4 x 4 (2 x 4) scores (rows
// r + 16 i, keys c + 16 j) and 4 x HDT / 16 outputs, so both products run from
// registers at 8 multiply-adds a thread for each 16-byte shared-memory load, as
// packed f32 pairs along the head dimension (half the instructions of scalar
// ones).  Bound by the FP32 pipe (61 %) and shared-memory passes (73 %): two
// sequences of 750 queries over 576 rows 223 us, with own rows and a 4-bit
// context 530 us, 31 to 33 TFLOP/s.  8 x 4 scores a thread halve the passes and
// the warps: 241 us.  tf32 halves on the tensor cores with sums handed over in
// chunks, as the f32 GEMM has them, have not been tried for these products.
// Query rows are scaled by scale log2(e) on the way in.  K of the next tile is
// loaded during softmax and P V, V during the next scores.  Shared rows of Q, K,
// V are f32, their 16-byte chunks XOR-swizzled by the row against bank
// conflicts.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "ctx_attn.cuh"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace irt {

namespace {

using tcx::f2_fma;
using tcx::f2_unpack;
using tcx::smem_u32;

constexpr int KT = 64, THREADS = 256;
constexpr float LN2 = 0.6931471805599453f;

struct TileArgs {
  CtxAttnParams p;
  int split;
  int q_vec, k_vec, v_vec, ks_vec, vs_vec, out_vec;
};

template <int HDT, int RT>
struct Smem {
  static constexpr int QT = 16 * RT;  // query rows of a CTA
  static constexpr int CH = HDT / 4;  // 16-byte chunks of a row
  static constexpr int OFF_K = QT * HDT, OFF_V = OFF_K + KT * HDT, OFF_P = OFF_V + KT * HDT, OFF_B = OFF_P + KT * QT;
  static constexpr int FLOATS = OFF_B + KT;
  // cluster merge over the tiles: O rows (padded against bank conflicts), m, l and weights
  static constexpr int OLD = HDT + 4;
  static_assert(QT * (OLD + 2 + MAX_SPLIT) <= OFF_P, "merge state fits Q, K and V");
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  return tcx::f2_pack(__float_as_uint(lo), __float_as_uint(hi));
}

// RT: query rows of a thread.
template <bool BF, bool CTX4, int HDT, int RT>
__global__ void __launch_bounds__(THREADS, 2) ctx_attn_tile_kernel(const __grid_constant__ TileArgs a) {
  using S = Smem<HDT, RT>;
  constexpr int QT = S::QT, CH = S::CH, OC = HDT / 8, NV = HDT / 64;  // NV: output chunks of four values per thread and row
  const CtxAttnParams& p = a.p;
  irt_attn_seq sd;
  if (!ctx_attn_seq(p, blockIdx.z, sd)) return;
  const int split = a.split, rank = blockIdx.x % split;
  const int hk = blockIdx.y, G = p.G, hd = p.hd;
  const int row0 = (blockIdx.x / split) * QT, nrows = sd.q_len * G;
  if (row0 >= nrows) return;  // the whole cluster
  extern __shared__ __align__(16) float sm[];
  float* sq = sm;
  float* sk = sm + S::OFF_K;
  float* sv = sm + S::OFF_V;
  float* sp = sm + S::OFF_P;
  float* sb = sm + S::OFF_B;  // 0 or -inf per key
  const int tid = threadIdx.x, r = tid / 16, c = tid % 16;
  const int n_self = p.ks.data ? (sd.q_len + KT - 1) / KT : 0;
  const int n_all = n_self + (sd.k_len + KT - 1) / KT;
  const int t0 = (int)((long)n_all * rank / split), nt = (int)((long)n_all * (rank + 1) / split) - t0;

  // Q rows, scaled
  const float qs = p.scale * 1.4426950408889634f;
  for (int e = tid; e < QT * OC; e += THREADS) {
    const int row = e / OC, o = e % OC, pr = row0 + row;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (pr < nrows && 8 * o < hd)
      load8<BF>(p.q.data, ((long)sd.q_start + pr / G) * p.q.row_stride + (hk * G + pr % G) * p.q.head_stride + 8 * o,
                a.q_vec, x);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<float4*>(sq + row * HDT + (((2 * o + i) ^ (row & 7)) * 4)) =
          make_float4(x[4 * i] * qs, x[4 * i + 1] * qs, x[4 * i + 2] * qs, x[4 * i + 3] * qs);
  }

  // K (or V) rows of local tile j into shared memory; rows that do not count
  // become zeros, whatever they hold
  auto load_tile = [&](int j, bool is_v) {
    const int t = t0 + j;
    const bool own = t < n_self;
    const int k0 = own ? t * KT : (t - n_self) * KT;
    const int left = (own ? sd.q_len : sd.k_len) - k0;
    const long base = (long)(own ? sd.q_start : sd.k_start) + k0;
    const uint8_t* mask = own || !p.mask ? nullptr : p.mask + base;
    float* dst = is_v ? sv : sk;
    const irt_rows& src = own ? (is_v ? p.vs : p.ks) : (is_v ? p.v : p.k);
    const bool vec = own ? (is_v ? a.vs_vec : a.ks_vec) : (is_v ? a.v_vec : a.k_vec);
    if (!is_v && tid < KT) sb[tid] = tid < left && (!mask || mask[tid]) ? 0.f : -INFINITY;
    if (!BF && vec && (own || !CTX4)) {
      const float* x = static_cast<const float*>(src.data) + base * src.row_stride + hk * src.head_stride;
#pragma unroll
      for (int i = 0; i < KT * CH / THREADS; ++i) {
        const int e = tid + i * THREADS, key = e / CH, ch = e % CH;
        const bool ok = key < left && 4 * ch < hd && (!mask || mask[key]);
        cp16(smem_u32(dst + key * HDT + ((ch ^ (key & 7)) * 4)), ok ? x + key * src.row_stride + 4 * ch : x, ok);
      }
      return;
    }
    constexpr int N = KT * OC / THREADS;
    float x[N][8];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + i * THREADS, key = e / OC, o = e % OC;
#pragma unroll
      for (int u = 0; u < 8; ++u) x[i][u] = 0.f;
      if (key >= left || 8 * o >= hd || (mask && !mask[key])) continue;
      if (CTX4 && !own) {
        const long cr = (long)hk * p.k_rows + base + key;
        const uint8_t* codes = is_v ? p.vc : p.kc;
        const bf16* sc = is_v ? p.vscale : p.kscale;
        kv4_unpack8(*reinterpret_cast<const uint32_t*>(codes + cr * (hd / 2) + 4 * o),
                    reinterpret_cast<const uint16_t*>(sc)[cr * kv4_groups(hd) + o / 4], x[i]);
      } else {
        load8<BF>(src.data, (base + key) * src.row_stride + hk * src.head_stride + 8 * o, vec, x[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + i * THREADS, key = e / OC, o = e % OC;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        *reinterpret_cast<float4*>(dst + key * HDT + (((2 * o + u) ^ (key & 7)) * 4)) =
            make_float4(x[i][4 * u], x[i][4 * u + 1], x[i][4 * u + 2], x[i][4 * u + 3]);
    }
  };

  uint64_t acc[RT][2 * NV];
  float m[RT], l[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
#pragma unroll
    for (int d = 0; d < 2 * NV; ++d) acc[i][d] = 0;
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  if (nt > 0) {
    load_tile(0, false);
    cp_commit();
    load_tile(0, true);
    cp_commit();
  }
  for (int j = 0; j < nt; ++j) {
    cp_wait<1>();  // K of this tile (its V may still fly)
    __syncthreads();
    float s[RT][4];
    {
      uint64_t s2[RT][4];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n) s2[i][n] = 0;
      const ulonglong2* q2 = reinterpret_cast<const ulonglong2*>(sq);
      const ulonglong2* k2 = reinterpret_cast<const ulonglong2*>(sk);
#pragma unroll 4
      for (int ch = 0; ch < CH; ++ch) {
        ulonglong2 qa[RT], kb[4];
#pragma unroll
        for (int i = 0; i < RT; ++i) qa[i] = q2[(r + 16 * i) * CH + (ch ^ (r & 7))];
#pragma unroll
        for (int n = 0; n < 4; ++n) kb[n] = k2[(c + 16 * n) * CH + (ch ^ (c & 7))];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int n = 0; n < 4; ++n) s2[i][n] = f2_fma(qa[i].y, kb[n].y, f2_fma(qa[i].x, kb[n].x, s2[i][n]));
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const bool off = sb[c + 16 * n] != 0.f;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          float x, y;
          f2_unpack(s2[i][n], x, y);
          s[i][n] = off ? -INFINITY : x + y;
        }
      }
    }
    __syncthreads();  // every thread is done with K of this tile
    if (j + 1 < nt) load_tile(j + 1, false);
    cp_commit();

    // online softmax: a row's scores are in the 16 threads of a half warp
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      float mx = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      mx = fmaxf(mx, m[i]);
      const float base = mx == -INFINITY ? 0.f : mx;  // NaN scores stay NaN in P and the sum
      const float corr = exp2f(m[i] - base);
      m[i] = mx;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        s[i][n] = exp2f(s[i][n] - base);
        sum += s[i][n];
      }
      l[i] = fmaf(l[i], corr, sum);
      const uint64_t c2 = pack2(corr, corr);
#pragma unroll
      for (int d = 0; d < 2 * NV; ++d) acc[i][d] = f2_fma(acc[i][d], c2, 0);
    }
    // P transposed: the rows of a thread are one chunk of a key
    using Chunk = typename std::conditional<RT == 4, float4, float2>::type;
    Chunk* pc = reinterpret_cast<Chunk*>(sp);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int key = c + 16 * n;
      float* t = reinterpret_cast<float*>(&pc[key * 16 + (r ^ (key & 15))]);
      if constexpr (RT == 4) *reinterpret_cast<float4*>(t) = make_float4(s[0][n], s[1][n], s[2][n], s[3][n]);
      else *reinterpret_cast<float2*>(t) = make_float2(s[0][n], s[1][n]);
    }
    cp_wait<1>();  // V of this tile (K of the next may still fly)
    __syncthreads();
    const ulonglong2* v2 = reinterpret_cast<const ulonglong2*>(sv);
#pragma unroll 4
    for (int key = 0; key < KT; ++key) {
      const Chunk pr = pc[key * 16 + (r ^ (key & 15))];
      ulonglong2 v[NV];
#pragma unroll
      for (int u = 0; u < NV; ++u) v[u] = v2[key * CH + ((c + 16 * u) ^ (key & 7))];
      const float* pv = reinterpret_cast<const float*>(&pr);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const uint64_t pp = pack2(pv[i], pv[i]);
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          acc[i][2 * u] = f2_fma(pp, v[u].x, acc[i][2 * u]);
          acc[i][2 * u + 1] = f2_fma(pp, v[u].y, acc[i][2 * u + 1]);
        }
      }
    }
    __syncthreads();  // every thread is done with V and P of this tile
    if (j + 1 < nt) load_tile(j + 1, true);
    cp_commit();
  }
  cp_wait<0>();

#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
  auto write = [&](int row, int d, float4 x, float inv) {  // four values from d of a row of the block
    x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
    const int pr = row0 + row;
    const long q = (long)sd.q_start + pr / G;
    const int head = hk * G + pr % G;
    if (p.gate.data) {
      const float4 g = load4<BF>(p.gate.data, q * p.gate.row_stride + head * p.gate.head_stride + d, a.out_vec);
      x.x *= g.x; x.y *= g.y; x.z *= g.z; x.w *= g.w;
    }
    store4<BF>(p.out.data, q * p.out.row_stride + head * p.out.head_stride + d, a.out_vec, x);
  };
  auto write_lse = [&](int row, float ms, float ls) {
    const int pr = row0 + row;
    if (p.lse)
      p.lse[((long)sd.q_start + pr / G) * p.H + hk * G + pr % G] = ls == 0.f ? -INFINITY : fmaf(ms, LN2, logf(ls));
  };
  if (split == 1) {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int row = r + 16 * i;
      if (row0 + row >= nrows) continue;
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
      if (c == 0) write_lse(row, m[i], l[i]);
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int d = 4 * (c + 16 * u);
        float4 x;
        f2_unpack(acc[i][2 * u], x.x, x.y);
        f2_unpack(acc[i][2 * u + 1], x.z, x.w);
        if (d < hd) write(row, d, x, inv);
      }
    }
    return;
  }
  // this CTA's rows for the others, over its tiles
  __syncthreads();
  float* so = sm;
  float* sml = sm + QT * S::OLD;
  float* wt = sml + 2 * QT;  // [row of this CTA][MAX_SPLIT]
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int row = r + 16 * i;
#pragma unroll
    for (int u = 0; u < NV; ++u)
      *reinterpret_cast<ulonglong2*>(so + row * S::OLD + 4 * (c + 16 * u)) =
          make_ulonglong2(acc[i][2 * u], acc[i][2 * u + 1]);
    if (c == 0) {
      sml[row] = m[i];
      sml[QT + row] = l[i];
    }
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int valid = min(QT, nrows - row0), per_row = hd / 4;
  const int mine = (valid - rank + split - 1) / split;  // rows dealt out to this CTA
  for (int i = tid; i < mine; i += THREADS) {
    const int row = i * split + rank;
    float mc[MAX_SPLIT], lc[MAX_SPLIT], mt = -INFINITY, lt = 0.f;
#pragma unroll
    for (int u = 0; u < MAX_SPLIT; ++u)
      if (u < split) {
        const float* o = cluster.map_shared_rank(sml, u);
        mc[u] = o[row];
        lc[u] = o[QT + row];
        mt = fmaxf(mt, mc[u]);
      }
    const float base = mt == -INFINITY ? 0.f : mt;
#pragma unroll
    for (int u = 0; u < MAX_SPLIT; ++u)
      if (u < split) {
        mc[u] = exp2f(mc[u] - base);
        lt = fmaf(lc[u], mc[u], lt);
      }
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
#pragma unroll
    for (int u = 0; u < MAX_SPLIT; ++u)
      if (u < split) wt[i * MAX_SPLIT + u] = mc[u] * inv;
    write_lse(row, mt, lt);
  }
  __syncthreads();
  for (int e = tid; e < mine * per_row; e += THREADS) {
    const int i = e / per_row, d = (e - i * per_row) * 4, row = i * split + rank;
    float4 o[MAX_SPLIT], x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < MAX_SPLIT; ++u)
      if (u < split) o[u] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(so, u) + row * S::OLD + d);
#pragma unroll
    for (int u = 0; u < MAX_SPLIT; ++u)
      if (u < split) {
        const float f = wt[i * MAX_SPLIT + u];
        x.x = fmaf(o[u].x, f, x.x);
        x.y = fmaf(o[u].y, f, x.y);
        x.z = fmaf(o[u].z, f, x.z);
        x.w = fmaf(o[u].w, f, x.w);
      }
    write(row, d, x, 1.f);
  }
  cluster.sync();  // the others may still read this CTA's rows
}

template <bool BF, bool CTX4, int HDT, int RT>
void launch(const CtxAttnParams& p, cudaStream_t s) {
  TileArgs a{};
  a.p = p;
  a.q_vec = rows_vec(p.q, BF);
  a.k_vec = rows_vec(p.k, BF);
  a.v_vec = rows_vec(p.v, BF);
  a.ks_vec = rows_vec(p.ks, BF);
  a.vs_vec = rows_vec(p.vs, BF);
  a.out_vec = rows_vec(p.out, BF) && (!p.gate.data || rows_vec(p.gate, BF));
  const int sms = device_sms();
  constexpr int QT = Smem<HDT, RT>::QT;
  const long blocks = ((long)p.max_q * p.G + QT - 1) / QT;
  const long ctas = blocks * p.Hkv * p.nseq;
  const long ktiles = (p.max_k + KT - 1L) / KT + (p.ks.data ? (p.max_q + KT - 1L) / KT : 0);
  a.split = 1;
  while (a.split < MAX_SPLIT && ctas * a.split * 2 <= 2L * sms && a.split * 2 <= ktiles) a.split *= 2;
  constexpr size_t smem = Smem<HDT, RT>::FLOATS * sizeof(float);
  auto kernel = ctx_attn_tile_kernel<BF, CTX4, HDT, RT>;
  static std::atomic<uint64_t> told{0};
  allow_smem(kernel, smem, told);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks * a.split), p.Hkv, p.nseq);
  cfg.blockDim = dim3(THREADS);
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

// Blocks of 32 rows up to 32 (half the work of a key tile), of 64 beyond.
template <bool BF, bool CTX4>
void launch_hd(const CtxAttnParams& p, cudaStream_t s) {
  const bool few = (long)p.max_q * p.G <= 32;
  if (p.hd <= 64) {
    if (few) launch<BF, CTX4, 64, 2>(p, s);
    else launch<BF, CTX4, 64, 4>(p, s);
  } else {
    if (few) launch<BF, CTX4, 128, 2>(p, s);
    else launch<BF, CTX4, 128, 4>(p, s);
  }
}

}  // namespace

bool ctx_attention_tile(const CtxAttnParams& p, cudaStream_t s) {
  // Fewer rows are the row kernel's: 16 streams over 8192 f32 rows, 8 / 12 packed
  // rows 1176 / 1765 us there and 1530 us here; 4-bit rows, 8 / 12 / 16 packed
  // rows 1172 / 1757 / 2340 us there and 1935 us here.
  if (p.hd > 128 || (long)p.max_q * p.G <= (p.kc ? 12 : 8)) return false;
  if (p.bf16_io) {
    if (p.kc) launch_hd<true, true>(p, s);
    else launch_hd<true, false>(p, s);
  } else {
    if (p.kc) launch_hd<false, true>(p, s);
    else launch_hd<false, false>(p, s);
  }
  return true;
}

}  // namespace irt
