// Attention over context states on tcgen05 (bf16, head_dim <= 128).
//
// One CTA = one (sequence, head group, tile of 128 packed query rows); with
// grouped heads the rows of a tile are query x head of the group (row r =
// query r / Gp, head r % Gp; Gp a power of two), so the group's K and V are read once.  Two CTAs
// share an SM.  Key tiles of 64: a sequence's own rows first, then its context
// rows.  Warps:
//   0..3  softmax: thread = query row.  Per tile: scores from TMEM, masked
//         keys to -inf, P = exp2(s - m) as packed bf16 over the first half of
//         the score buffer (the A operand of P V).  m starts 2^8 above a row's
//         maximum and is raised, and O rescaled, only when a score passes it, so
//         weights are at most 1 and O no larger than the values' sum.  Warps
//         without a query row take no part.
//   4     TMA: Q once, K and V of native tiles (2-stage rings, K two tiles
//         ahead of V).
//   5     tcgen05.mma issue: S_j = Q K_j^T, O += P_j V_j.
//   6..9  (4-bit context) codes -> bf16 K and V tiles in the same swizzled
//         layout.  A value c s has at most 8 significant bits, so the bf16 tile
//         is exact and the products are those of the cache's values.
// Keys that do not count (past the sequence, masked) must not meet the P V
// product even with weight 0, since 0 * NaN is NaN: their V rows are zeroed in
// shared memory before the product (native tiles: by the softmax warps, only
// in tiles that have such keys).
//
// Few query tiles: the key tiles of one query tile are shared by a cluster of
// 2, 4 or 8 CTAs, which merge their (m, l, O) through distributed shared
// memory in rank order.  No workspace, no atomics.
//
// Many queries: bound by the latency of a CTA's chain (load, scores, softmax,
// product, rows out), of which an SM runs two: 256 of its 512 TMEM columns
// each, for two score tiles and O.  About 6.5 us a CTA and 0.9 us a key tile:
// 64 x 16 heads, 768 queries over 64 / 640 / 1280 keys without a gate 130 / 303 /
// 535 us, the last at 0.96 PFLOP/s; 64 utterances of 50 to 750 frames over 141 to 632 rows
// 158 us.  4-bit context with own rows 338 us, there also bound by the issue of
// instructions of the code warps.  One query: bound by reading K and V, 6.1
// TB/s over 5000 to 8192 rows.  Fewer keys a tile would leave the tensor pipe
// waiting for softmax.  All 512 columns for one CTA (128 keys a tile, or two
// query tiles that share each K and V tile) have not been measured.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstring>
#include <mutex>

#include "ctx_attn.cuh"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace irt {

namespace {

using namespace tcx;

constexpr int QT = 128, KT = 64, NKV = 2;
constexpr float HEADROOM_LOG2 = 8.f;  // of m above the maximum when it is raised
constexpr float LN2 = 0.6931471805599453f;

template <int HDT, bool CTX4>
struct Cfg {
  static constexpr int CODE_WARPS = CTX4 ? 4 : 0, THREADS = 192 + 32 * CODE_WARPS;
  // The native kernel's 6 warps stay within 128 registers: with more, two CTAs
  // fill the register file and a CTA's successor starts late (64 utterances 188
  // us at 149 registers against 159).
  static constexpr uint32_t Q_HALF = QT * 128, Q_BYTES = Q_HALF * (HDT / 64);  // 64-column halves
  static constexpr uint32_t HALF = KT * 128, TILE = HALF * (HDT / 64);
  static constexpr uint32_t OFF_K = Q_BYTES, OFF_V = OFF_K + NKV * TILE, OFF_BAR = OFF_V + NKV * TILE;
  static constexpr size_t SMEM = OFF_BAR + 256 + 1024;
  static constexpr uint32_t IDESC_S = idesc_bf16(128, KT, false), IDESC_O = idesc_bf16(128, HDT, true);
  static constexpr uint32_t TM_S = 0, TM_O = 2 * KT, TM_COLS = 256;
  // arrivals that fill a K or V stage: the TMA thread and the code warps of K or V
  static constexpr uint32_t FULL_COUNT = 1 + CODE_WARPS / 2;
  // cluster merge: f32 O rows (padded against bank conflicts), m and l
  static constexpr int OLD = HDT + 4;
  static_assert((uint32_t)QT * (OLD + 2 + MAX_SPLIT) * 4 <= OFF_BAR, "merge buffers fit the tiles");
};

struct TcArgs {
  CtxAttnParams p;
  float scale_log2;
  int log_gp; // heads packed into a query tile, a power of two
  int split;  // CTAs of the cluster
  int tma_out;  // a warp's 32 rows are a box of the output's map
  int heads;    // head groups of the listed grid (see list_tiles), or 0
};

__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(db), "r"(idesc), "r"(acc));
}

// 32 lanes x 16 or 32 columns from the warp's registers.
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[32]) { tmem_st32(taddr, r); }
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Bounded wait as tcx::mbar_wait, reported to `status` in the place of the
// file's own flag.
__device__ __forceinline__ void wait_or_report(uint32_t bar, uint32_t parity, int* status) {
  if (mbar_try_wait(bar, parity)) return;
  volatile int* flag = status;
  if (*flag) return;
  const uint64_t limit = *reinterpret_cast<volatile unsigned long long*>(&g_wait_limit_ns);
  const uint64_t t0 = globaltimer();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (mbar_try_wait(bar, parity)) return;
    if (*flag) return;
    if (globaltimer() - t0 > limit) {
      atomicExch(status, 1);
      return;
    }
  }
}
// For a CTA with an expired wait, before it leaves: tells the host, and stays.
// What it started (loads, products) may still be on its way and must not reach
// the shared memory of the CTA that takes its place; a millisecond is a
// thousand times what a load takes.  Not inlined, and looked for where the
// chain does not wait: next to the softmax a few instructions more in every
// wait cost the 4-bit kernel 5 %.
__device__ __noinline__ void settle(int* host) {
  if (host) *reinterpret_cast<volatile int*>(host) = 1;
  const uint64_t t0 = globaltimer();
  for (int i = 0; i < 10000 && globaltimer() - t0 < 1000000; ++i) __nanosleep(200);
}

// Box of a (d, head, row) tensor.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
__device__ __forceinline__ void ld_shared16(uint32_t addr, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}

// m log 2 + log l, the headroom moved from one to the other: their sum loses nothing to it.
__device__ __forceinline__ float lse_of(float m, float l) {
  return fmaf(m - HEADROOM_LOG2, LN2, logf(l * exp2f(HEADROOM_LOG2)));
}

// Listed grids (4-bit context): ragged sequences of several query tiles are
// numbered through, tile after tile, so that no CTA starts for a tile that its
// sequence does not have.  The 20 warps of two CTAs fill the register file, and
// an empty CTA held up the next one for about 7 us: 16 / 64 / 250 utterances of
// 50 to 750 frames 113 / 382 / 1466 us, listed 100 / 339 / 1400 us.  The native
// kernel leaves room, and looking for the tile costs what the empty CTAs do: 49
// / 162 / 605 us, listed 48 / 161 / 691.
// Tiles to start, QT packed rows (`group` heads a query) each: at least as many
// as there are, since query ranges do not overlap.  0: the grid is [tiles of
// max_q, head groups, sequences], because it is no larger, or there are too
// many sequences to look through.
constexpr int MAX_LISTED = 256;
inline long list_tiles(const CtxAttnParams& p, int group, int QT) {
  const long per = ((long)p.max_q * group + QT - 1) / QT, most = p.q_rows * group / QT + p.nseq;
  return p.seqs && p.nseq <= MAX_LISTED && per > 1 && most < per * p.nseq ? most : 0;
}
// Sequence of listed tile `tile` and the tile's number in it, or -1 (the same
// in every thread).  Called by whole warps.
__device__ __forceinline__ int listed_tile(const CtxAttnParams& p, int tile, int group, int QT, irt_attn_seq& sd) {
  const int lane = threadIdx.x % 32;
  auto entry = [&](int n, irt_attn_seq& e) {
    return n < p.nseq && ctx_attn_seq(p, n, e) ? (e.q_len * group + QT - 1) / QT : 0;
  };
  irt_attn_seq e, next{};
  int t_next = entry(lane, next), before = 0;
  for (int c = 0; c < p.nseq; c += 32) {
    e = next;
    const int t = t_next;
    t_next = entry(c + 32 + lane, next);
    int sum = t;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, w);
      if (lane >= w) sum += o;
    }
    const uint32_t behind = __ballot_sync(0xffffffffu, before + sum > tile);
    if (behind) {
      const int f = __ffs(behind) - 1;
      sd = {__shfl_sync(0xffffffffu, e.q_start, f), __shfl_sync(0xffffffffu, e.q_len, f),
            __shfl_sync(0xffffffffu, e.k_start, f), __shfl_sync(0xffffffffu, e.k_len, f)};
      return tile - before - __shfl_sync(0xffffffffu, sum - t, f);
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return -1;
}

template <int HDT, bool CTX4>
__global__ void __launch_bounds__(Cfg<HDT, CTX4>::THREADS, 2)
    ctx_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmKS,
                       const __grid_constant__ CUtensorMap tmVS, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmG,
                       const __grid_constant__ CUtensorMap tmO, const __grid_constant__ TcArgs a) {
  using C = Cfg<HDT, CTX4>;
  if (threadIdx.x == 128) {  // the TMA thread's first descriptors, while the predecessor may still run
    prefetch_map(&tmQ);
    if (!CTX4) {
      prefetch_map(&tmK);
      prefetch_map(&tmV);
    }
  }
  pdl_wait();
  pdl_trigger();
  const CtxAttnParams& p = a.p;
  // read by the TMA thread: after an expired wait nothing is loaded
  const bool go = threadIdx.x != 128 || *reinterpret_cast<volatile int*>(p.expired) == 0;
  irt_attn_seq sd;
  const int split = a.split, rank = blockIdx.x % split, lg = a.log_gp, gmask = (1 << lg) - 1;
  int q0, head0;  // first query and first head of the tile
  if (CTX4 && a.heads) {
    const int tile = blockIdx.x / a.heads;
    head0 = (blockIdx.x - tile * a.heads) << lg;
    q0 = listed_tile(p, tile, 1 << lg, QT, sd) * (QT >> lg);
    if (q0 < 0) return;
  } else {
    if (!ctx_attn_seq(p, blockIdx.z, sd)) return;
    q0 = (blockIdx.x / split) * (QT >> lg);
    if (q0 >= sd.q_len) return;  // the whole cluster
    head0 = blockIdx.y << lg;
  }
  const int hk = head0 / p.G;
  const int rows = min(QT, (sd.q_len - q0) << lg);  // packed query rows of the tile
  const int n_self = p.ks.data ? (sd.q_len + KT - 1) / KT : 0;
  const int n_all = n_self + (sd.k_len + KT - 1) / KT;
  const int t0 = (int)((long)n_all * rank / split), nt = (int)((long)n_all * (rank + 1) / split) - t0;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  const uint32_t Q_FULL = bar(0), O_DONE = bar(1), O_FINAL = bar(2);
  auto K_FULL = [&](int s) { return bar(3 + s); };
  auto K_EMPTY = [&](int s) { return bar(3 + NKV + s); };
  auto V_FULL = [&](int s) { return bar(3 + 2 * NKV + s); };
  auto V_EMPTY = [&](int s) { return bar(3 + 3 * NKV + s); };
  auto S_FULL = [&](int b) { return bar(3 + 4 * NKV + b); };
  auto P_FULL = [&](int b) { return bar(5 + 4 * NKV + b); };
  const uint32_t G_FULL = bar(7 + 4 * NKV);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 8 + 4 * NKV);
  auto bar_wait = [&](uint32_t b, uint32_t parity) { wait_or_report(b, parity, p.expired); };

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int sm_warps = (rows + 31) / 32;  // softmax warps that have a query row
  const uint32_t sQ = smem_u32(sm);
  auto sK = [&](int s) { return smem_u32(sm + C::OFF_K + s * C::TILE); };
  auto sV = [&](int s) { return smem_u32(sm + C::OFF_V + s * C::TILE); };
  // first row and valid keys of local tile j
  auto row_of = [&](int j) {
    const int t = t0 + j;
    return t < n_self ? sd.q_start + t * KT : sd.k_start + (t - n_self) * KT;
  };
  auto keys_of = [&](int j) {
    const int t = t0 + j;
    return min(KT, t < n_self ? sd.q_len - t * KT : sd.k_len - (t - n_self) * KT);
  };

  // K (V) rows of local tile j, by the TMA thread
  auto load = [&](int j, uint32_t full, uint32_t empty, uint32_t dst, const CUtensorMap* self, const CUtensorMap* ctx) {
    bar_wait(empty, ((j / NKV) & 1) ^ 1);
    if (!mbar_try_wait(empty, ((j / NKV) & 1) ^ 1)) return;  // gave up: nothing more is started
    const bool own = t0 + j < n_self;
    if (CTX4 && !own) {  // the code warps fill this one
      mbar_arrive(full);
      return;
    }
    mbar_expect_tx(full, C::TILE);
    const CUtensorMap* m = own ? self : ctx;
#pragma unroll
    for (int h = 0; h < HDT / 64; ++h) tma_load_3d(dst + h * C::HALF, m, full, 64 * h, hk, row_of(j));
  };
  auto load_k = [&](int j) { load(j, K_FULL(j % NKV), K_EMPTY(j % NKV), sK(j % NKV), &tmKS, &tmK); };
  auto load_v = [&](int j) { load(j, V_FULL(j % NKV), V_EMPTY(j % NKV), sV(j % NKV), &tmVS, &tmV); };

  // The TMA thread sets up the barriers and starts the first loads; TMEM is
  // allocated meanwhile.
  if (threadIdx.x == 128) {
    mbar_init(Q_FULL, 1);
    mbar_init(O_DONE, 1);
    mbar_init(O_FINAL, 1);
    mbar_init(G_FULL, 1);
    for (int r = 0; r < NKV; ++r) {
      mbar_init(K_FULL(r), C::FULL_COUNT);
      mbar_init(K_EMPTY(r), 1);
      mbar_init(V_FULL(r), C::FULL_COUNT);
      mbar_init(V_EMPTY(r), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(S_FULL(b), 1);
      mbar_init(P_FULL(b), sm_warps);
    }
    mbar_fence_init();
    fence_proxy_async();
    if (nt > 0 && go) {
      mbar_expect_tx(Q_FULL, C::Q_BYTES);
#pragma unroll
      for (int h = 0; h < HDT / 64; ++h) tma_load_3d(sQ + h * C::Q_HALF, &tmQ, Q_FULL, 64 * h, head0, sd.q_start + q0);
      load_k(0);
      if (nt > 1) load_k(1);
      load_v(0);
    }
  }
  __syncwarp();
  if (warp == 5) tmem_alloc(smem_u32(tmem_slot), C::TM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  float m_run = -INFINITY, l_run = 0.f;
  if (nt > 0) {
    if (warp == 4) {
      // ---------------- TMA ----------------
      if (lane == 0 && go) {
        for (int j = 0; j + 1 < nt; ++j) {  // K two tiles ahead of V, as the products are issued
          if (j + 2 < nt) load_k(j + 2);
          load_v(j + 1);
        }
        // the gate takes Q's place once the last scores are done
        if (split == 1 && p.gate.data) {
          bar_wait(K_EMPTY((nt - 1) % NKV), ((nt - 1) / NKV) & 1);
          mbar_expect_tx(G_FULL, C::Q_BYTES);
#pragma unroll
          for (int h = 0; h < HDT / 64; ++h)
            tma_load_3d(sQ + h * C::Q_HALF, &tmG, G_FULL, 64 * h, head0, sd.q_start + q0);
        }
      }
    } else if (warp == 5) {
      // ---------------- MMA ----------------
      if (lane == 0) {
        bar_wait(Q_FULL, 0);
        tc_fence_after();
        auto issue_s = [&](int j) {
          const int r = j % NKV, b = j & 1;
          bar_wait(K_FULL(r), (j / NKV) & 1);
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < HDT / 16; ++kk) {
            const uint64_t da = sdesc_kmajor(sQ + (kk >> 2) * C::Q_HALF + (kk & 3) * 32);
            const uint64_t db = sdesc_kmajor(sK(r) + (kk >> 2) * C::HALF + (kk & 3) * 32);
            umma_f16(tmem + C::TM_S + b * KT, da, db, C::IDESC_S, kk != 0);
          }
          umma_commit(S_FULL(b));
          umma_commit(K_EMPTY(r));
        };
        issue_s(0);
        if (nt > 1) issue_s(1);
        for (int j = 0; j < nt; ++j) {
          const int s = j & 1, r = j % NKV;
          bar_wait(V_FULL(r), (j / NKV) & 1);
          bar_wait(P_FULL(s), (j >> 1) & 1);
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < KT / 16; ++kk) {
            const uint64_t db = sdesc_sw128(sV(r) + kk * 16 * 128, C::HALF, 1024);
            umma_ts(tmem + C::TM_O, tmem + C::TM_S + s * KT + kk * 8, db, C::IDESC_O, (j | kk) != 0);
          }
          umma_commit(V_EMPTY(r));
          umma_commit(O_DONE);
          if (j + 2 < nt) issue_s(j + 2);  // overwrites S_j / P_j after P_j V_j in the tensor pipe's order
        }
        umma_commit(O_FINAL);
        // a wait has given up before (read while the last rows are written)
        if (*reinterpret_cast<volatile int*>(p.expired)) settle(p.expired_host);
      }
    } else if (CTX4 && warp >= 6) {
      // ---------------- codes -> bf16 tiles ----------------
      // Warps 6 and 7 fill the K tiles, 8 and 9 the V tiles, each half of the
      // head dimension; a lane has keys lane and lane + 32, so the eight
      // 16-byte chunks that a quarter warp stores fall on different banks under
      // the swizzle.  The codes of a tile are read while the one before it is
      // written.  One small copy of the code: unrolled over tiles it outgrew
      // the instruction cache next to the softmax (64 utterances 523 us
      // against 429 us before the other steps).
      constexpr int W = HDT / 16;   // words of eight codes per key and lane
      constexpr int NG = HDT / 64;  // groups of 32
      const bool is_v = warp >= 8;
      const int part = warp & 1, hd = p.hd, groups = kv4_groups(hd);
      const long row0 = (long)hk * p.k_rows + sd.k_start + lane;
      const uint8_t* codes = (is_v ? p.vc : p.kc) + row0 * (hd / 2) + part * W * 4;
      const bf16* scales = (is_v ? p.vscale : p.kscale) + row0 * groups + part * NG;
      const uint8_t* mask = p.mask ? p.mask + sd.k_start + lane : nullptr;
      struct Codes {
        uint4 w[2][NG];
        uint16_t s[2][NG];
      } next;
      auto fetch = [&](int j) {
        const int k0 = (t0 + j - n_self) * KT;
        if (k0 < 0) return;  // a tile of own rows
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int k = k0 + 32 * e;  // of lane 0
          const bool ok = k + lane < sd.k_len && (!mask || mask[k]);
#pragma unroll
          for (int g = 0; g < NG; ++g) {  // scale 0: a row that does not count, or what is behind head_dim, becomes zeros
            const bool in = ok && part * NG + g < groups;
            next.w[e][g] = in ? *reinterpret_cast<const uint4*>(codes + (long)k * (hd / 2) + 16 * g) : make_uint4(0, 0, 0, 0);
            next.s[e][g] = in ? reinterpret_cast<const uint16_t*>(scales)[(long)k * groups + g] : 0;
          }
        }
      };
      fetch(0);
#pragma unroll 1
      for (int j = 0; j < nt; ++j) {
        const Codes cur = next;
        if (j + 1 < nt) fetch(j + 1);
        const int r = j % NKV;
        bar_wait(is_v ? V_EMPTY(r) : K_EMPTY(r), ((j / NKV) & 1) ^ 1);
        if (t0 + j >= n_self) {
          const uint32_t dst = is_v ? sV(r) : sK(r);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t row = dst + (lane + 32 * e) * 128;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const uint32_t sb = (uint32_t)cur.s[e][g] << 16 | cur.s[e][g];
              const __nv_bfloat162 s2 = *reinterpret_cast<const __nv_bfloat162*>(&sb);
              const __nv_bfloat162 n2 = __hmul2(s2, __floats2bfloat162_rn(-24.f, -24.f));
              const uint32_t w[4] = {cur.w[e][g].x, cur.w[e][g].y, cur.w[e][g].z, cur.w[e][g].w};
              const int c0 = part * W + 4 * g;  // 16-byte chunk of the row
              const uint32_t at = row + (c0 >> 3) * C::HALF;
              // below 2^123 and of 5 significant bits, as append writes it; a caller's own may be any bf16 number
              if (cur.s[e][g] < 0x7d00 && (cur.s[e][g] & 7) == 0) {
#pragma unroll
                for (int o = 0; o < 4; ++o)
                  st_shared16(at + ((((c0 + o) & 7) ^ (lane & 7)) << 4), kv4_bf16x8<false>(w[o], s2, n2));
              } else {
                uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
#pragma unroll 1
                for (int o = 0; o < 4; ++o) {
                  st_shared16(at + ((((c0 + o) & 7) ^ (lane & 7)) << 4), kv4_bf16x8<true>((uint32_t)lo, s2, n2));
                  lo = lo >> 32 | hi << 32;
                  hi >>= 32;
                }
              }
            }
          }
          fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(is_v ? V_FULL(r) : K_FULL(r));
      }
    } else if (warp < sm_warps) {
      // ---------------- softmax ----------------
      const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
      // mask bytes of keys lane and lane + 32 of a tile, read a tile ahead
      uint8_t next0 = 1, next1 = 1;
      auto fetch_mask = [&](int j) {
        if (!p.mask || j >= nt || t0 + j < n_self) return;
        const uint8_t* mk = p.mask + row_of(j) + lane;
        const int n = keys_of(j) - lane;
        next0 = n > 0 ? mk[0] : 0;
        next1 = n > 32 ? mk[32] : 0;
      };
      fetch_mask(0);
      for (int j = 0; j < nt; ++j) {
        const int b = j & 1;
        const bool own = t0 + j < n_self;
        const int nkeys = keys_of(j);
        // bit i: key i counts
        uint32_t on0 = nkeys >= 32 ? 0xffffffffu : (1u << nkeys) - 1;
        uint32_t on1 = nkeys >= 64 ? 0xffffffffu : nkeys > 32 ? (1u << (nkeys - 32)) - 1 : 0u;
        if (p.mask && !own) {
          on0 &= __ballot_sync(0xffffffffu, next0);
          on1 &= __ballot_sync(0xffffffffu, next1);
        }
        fetch_mask(j + 1);
        const bool partial = (on0 & on1) != 0xffffffffu;
        bar_wait(S_FULL(b), (j >> 1) & 1);
        tc_fence_after();
        // Scores in halves of 32 columns.  One register copy of a tile's scores
        // (native context), or two readings of them: 96 registers a thread
        // leave room for the code warps.
        constexpr int HC = CTX4 ? 32 : KT;
        uint32_t sr[HC];
        auto load_scores = [&](int col) {
#pragma unroll
          for (int g = 0; g < HC / 32; ++g)
            tmem_ld32(tmem + lane_off + C::TM_S + b * KT + col + 32 * g, *reinterpret_cast<uint32_t(*)[32]>(&sr[32 * g]));
          tmem_wait_ld();
          if (partial) {
#pragma unroll
            for (int i = 0; i < HC; ++i) {
              const uint32_t on = i < 32 ? (col ? on1 : on0) : on1;
              if (!((on >> (i & 31)) & 1)) sr[i] = __float_as_uint(-INFINITY);
            }
          }
        };
        float mx = -INFINITY;
#pragma unroll 1
        for (int col = 0; col < KT; col += HC) {
          load_scores(col);
          float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
          for (int i = 0; i < HC; i += 4) {
            mx0 = fmaxf(mx0, __uint_as_float(sr[i]));
            mx1 = fmaxf(mx1, __uint_as_float(sr[i + 1]));
            mx2 = fmaxf(mx2, __uint_as_float(sr[i + 2]));
            mx3 = fmaxf(mx3, __uint_as_float(sr[i + 3]));
          }
          mx = fmaxf(mx, fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)));
        }
        mx *= a.scale_log2;
        if (partial && (!CTX4 || own)) {  // V rows that do not count: zeros
          bar_wait(V_FULL(j % NKV), (j / NKV) & 1);
          constexpr int CH = HDT / 8, KW = 32 / CH;  // 16-byte chunks of a row, rows of a warp at a time
          const uint32_t at = sV(j % NKV) + (lane % CH >> 3) * C::HALF + (lane & 7) * 16;
#pragma unroll 4
          for (int key = warp * KW + lane / CH; key < KT; key += sm_warps * KW)
            if (!((key < 32 ? on0 >> key : on1 >> (key - 32)) & 1)) st_shared16(at + key * 128, make_uint4(0, 0, 0, 0));
          fence_proxy_async();
        }
        float corr = 1.f;
        const bool raise = mx > m_run;
        if (raise) {
          const float m_new = mx + HEADROOM_LOG2;
          corr = ex2(m_run - m_new);
          m_run = m_new;
        }
        const float nbase = m_run == -INFINITY ? 0.f : -m_run;
        // P_{j-1} V_{j-1} must be done before O is read; the phase in flight
        // is j - 1 or already j
        if (__any_sync(0xffffffffu, raise) && j > 0) {
          bar_wait(O_DONE, (j - 1) & 1);
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HDT / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(tmem + lane_off + C::TM_O + c * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
            tmem_st32(tmem + lane_off + C::TM_O + c * 32, r);
          }
        }
        const uint64_t sc2 = f2_pack(__float_as_uint(a.scale_log2), __float_as_uint(a.scale_log2));
        const uint64_t nb2 = f2_pack(__float_as_uint(nbase), __float_as_uint(nbase));
        uint64_t rs2 = 0;
#pragma unroll 1
        for (int col = 0; col < KT; col += HC) {
          if (CTX4) load_scores(col);
          uint32_t pk[HC / 2];
#pragma unroll
          for (int c = 0; c < HC / 2; ++c) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(sr[2 * c], sr[2 * c + 1]), sc2, nb2), x0, x1);
            const float p0 = ex2(x0), p1 = ex2(x1);
            rs2 = f2_add(rs2, f2_pack(__float_as_uint(p0), __float_as_uint(p1)));
            pk[c] = pack_bf16x2(p0, p1);
          }
          // P of these columns: half as many, over scores that have been read
          tmem_st_cols(tmem + lane_off + C::TM_S + b * KT + col / 2, pk);
        }
        float rs0, rs1;
        f2_unpack(rs2, rs0, rs1);
        tmem_wait_st();
        l_run = l_run * corr + (rs0 + rs1);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(P_FULL(b));
      }
      bar_wait(O_FINAL, 0);
      if (!__all_sync(0xffffffffu, mbar_try_wait(O_FINAL, 0))) settle(p.expired_host);
      tc_fence_after();
    }
  }

  // ---------------- output ----------------
  const int qrow = warp * 32 + lane;
  if (split == 1) {
    // Rows go through shared memory in Q's place (all products that read Q are
    // done): the 32 rows of a warp leave as boxes of the output's map, or,
    // where they are not all of this sequence, 256 contiguous bytes of a row at
    // a time (a thread's own 16-byte stores, a row apart, took twice as long;
    // without the boxes 64 utterances 163.5 us against 158.8).
    if (warp < sm_warps) {
      const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
      const bool gated = p.gate.data && nt > 0;
      if (gated) {
        bar_wait(G_FULL, 0);
        if (!__all_sync(0xffffffffu, mbar_try_wait(G_FULL, 0))) settle(p.expired_host);
      }
#pragma unroll 1
      for (int c = 0; c < HDT; c += 32) {
        uint32_t r[32], g[4][4];
        auto addr = [&](int u) {
          return sQ + (c >> 6) * C::Q_HALF + qrow * 128 + (((((c & 63) >> 3) + u) ^ (qrow & 7)) << 4);
        };
        if (nt > 0) {
          tmem_ld32(tmem + lane_off + C::TM_O + c, r);
          if (gated) {
#pragma unroll
            for (int u = 0; u < 4; ++u) ld_shared16(addr(u), g[u]);
          }
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t op[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float x = __uint_as_float(r[u * 8 + 2 * k]) * inv, y = __uint_as_float(r[u * 8 + 2 * k + 1]) * inv;
            if (gated) {
              x *= __uint_as_float(g[u][k] << 16);
              y *= __uint_as_float(g[u][k] & 0xffff0000u);
            }
            op[k] = pack_bf16x2(x, y);
          }
          st_shared16(addr(u), make_uint4(op[0], op[1], op[2], op[3]));
        }
      }
      fence_proxy_async();
      __syncwarp();
      const bool boxes = a.tma_out && warp * 32 + 32 <= rows;
      if (boxes && lane == 0) {
#pragma unroll
        for (int h = 0; h < HDT / 64; ++h)
          tma_store_3d(&tmO, sQ + h * C::Q_HALF + warp * 4096, 64 * h, head0, sd.q_start + q0 + ((warp * 32) >> lg));
        bulk_commit();
      }
      if (qrow < rows && p.lse)
        p.lse[((long)sd.q_start + q0 + (qrow >> lg)) * p.H + head0 + (qrow & gmask)] =
            l_run == 0.f ? -INFINITY : lse_of(m_run, l_run);
      constexpr int LPR = HDT / 8;  // lanes of a row
      const int chunk = lane % LPR;
      if (!boxes && 8 * chunk < p.hd) {
        bf16* out = static_cast<bf16*>(p.out.data) + 8 * chunk;
#pragma unroll 4
        for (int i = lane / LPR; i < 32; i += 32 / LPR) {
          const int row = warp * 32 + i;
          if (row >= rows) break;
          uint32_t v[4];
          ld_shared16(sQ + (chunk >> 3) * C::Q_HALF + row * 128 + (((chunk & 7) ^ (row & 7)) << 4), v);
          *reinterpret_cast<uint4*>(out + ((long)sd.q_start + q0 + (row >> lg)) * p.out.row_stride +
                                    (head0 + (row & gmask)) * p.out.head_stride) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
      if (boxes && lane == 0) bulk_wait_read0();
    }
  } else {
    // this CTA's O, m and l over its tiles (all products are done, so nothing
    // else uses the shared memory)
    float* so = reinterpret_cast<float*>(sm);
    float* sml = so + QT * C::OLD;  // m, then l
    if (warp < sm_warps) {
      const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
      sml[qrow] = m_run;
      sml[QT + qrow] = l_run;
#pragma unroll 1
      for (int c = 0; c < HDT / 32; ++c) {
        uint32_t r[32];
        if (nt > 0) {
          tmem_ld32(tmem + lane_off + C::TM_O + c * 32, r);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<uint4*>(so + qrow * C::OLD + c * 32 + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
      }
    }
    cg::cluster_group cluster = cg::this_cluster();
    __syncwarp();
    cluster.sync();
    // weights of the CTAs' states for the rows dealt out to this one
    float* wt = sml + 2 * QT;  // [row of this CTA][MAX_SPLIT]
    const int mine = (rows - rank + split - 1) / split;
    for (int i = threadIdx.x; i < mine; i += C::THREADS) {
      const int r = i * split + rank;
      float m[MAX_SPLIT], l[MAX_SPLIT], mt = -INFINITY, lt = 0.f;
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c)
        if (c < split) {
          const float* o = cluster.map_shared_rank(sml, c);
          m[c] = o[r];
          l[c] = o[QT + r];
          mt = fmaxf(mt, m[c]);
        }
      const float base = mt == -INFINITY ? 0.f : mt;
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c)
        if (c < split) {
          m[c] = ex2(m[c] - base);
          lt = fmaf(l[c], m[c], lt);
        }
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c)
        if (c < split) wt[i * MAX_SPLIT + c] = m[c] * inv;
      if (p.lse)
        p.lse[((long)sd.q_start + q0 + (r >> lg)) * p.H + head0 + (r & gmask)] =
            lt == 0.f ? -INFINITY : lse_of(mt, lt);
    }
    __syncthreads();
    const int per_row = p.hd / 4;
    for (int e = threadIdx.x; e < mine * per_row; e += C::THREADS) {
      const int i = e / per_row, d = (e - i * per_row) * 4, r = i * split + rank;
      float4 o[MAX_SPLIT], x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c)
        if (c < split) o[c] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(so, c) + r * C::OLD + d);
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c)
        if (c < split) {
          const float f = wt[i * MAX_SPLIT + c];
          x.x = fmaf(o[c].x, f, x.x);
          x.y = fmaf(o[c].y, f, x.y);
          x.z = fmaf(o[c].z, f, x.z);
          x.w = fmaf(o[c].w, f, x.w);
        }
      const long row = (long)sd.q_start + q0 + (r >> lg);
      const int head = head0 + (r & gmask);
      if (p.gate.data) {
        const float4 g = load4<true>(p.gate.data, row * p.gate.row_stride + head * p.gate.head_stride + d, true);
        x.x *= g.x; x.y *= g.y; x.z *= g.z; x.w *= g.w;
      }
      store4<true>(p.out.data, row * p.out.row_stride + head * p.out.head_stride + d, true, x);
    }
    __syncwarp();
    cluster.sync();  // the others may still read this CTA's part
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TM_COLS);
  }
}

// (d, head, row) map with boxes of 64 values x `heads` x `rows`; false when
// the strides cannot be encoded.
bool rows_map(CUtensorMap& m, const irt_rows& r, long rows, int heads, int hd, int box_heads, int box_rows) {
  const cuuint64_t dim[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t stride[2] = {(cuuint64_t)r.head_stride * 2, (cuuint64_t)r.row_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  const cuuint32_t step[3] = {1, 1, 1};
  return tma_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, r.data, dim, stride, box, step,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HDT, bool CTX4>
bool launch(const CtxAttnParams& p, cudaStream_t s) {
  using C = Cfg<HDT, CTX4>;
  TcArgs a{};
  a.p = p;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  const int gp = QT % p.G == 0 ? p.G : 1;
  while ((1 << a.log_gp) < gp) ++a.log_gp;
  CUtensorMap q, ks, vs, k, v, g, o;
  if (!rows_map(q, p.q, p.q_rows, p.H, p.hd, gp, QT / gp)) return false;
  ks = vs = k = v = g = o = q;
  if (p.gate.data && !rows_map(g, p.gate, p.q_rows, p.H, p.hd, gp, QT / gp)) return false;
  if (p.ks.data && (!rows_map(ks, p.ks, p.q_rows, p.Hkv, p.hd, 1, KT) ||
                    !rows_map(vs, p.vs, p.q_rows, p.Hkv, p.hd, 1, KT)))
    return false;
  if (p.k.data && p.k_rows > 0 &&
      (!rows_map(k, p.k, p.k_rows, p.Hkv, p.hd, 1, KT) || !rows_map(v, p.v, p.k_rows, p.Hkv, p.hd, 1, KT)))
    return false;
  const int sms = device_sms();
  const long qtiles = ((long)p.max_q * gp + QT - 1) / QT;
  const long ctas = qtiles * (p.H / gp) * p.nseq;
  const long ktiles = (p.max_k + KT - 1L) / KT + (p.ks.data ? (p.max_q + KT - 1L) / KT : 0);
  // Key tiles are shared by a cluster where that pays: the least of
  //   5 + 0.82 (tiles of a CTA) (1.6 where CTAs share SMs) + 1 + 2.2 rows / 128
  // microseconds, the last two for the merge; at most two CTAs per SM.  One
  // sequence of 16 heads, 1 / 2 / 4 / 8 CTAs: 1 query over 576 keys 11.3 / 9.3
  // / 8.1 / 7.9 us; 128 over 2048 31.4 / 21.9 / 14.8 / 14.3; 750 over 576 13.2
  // / 16.1 / 22.9 / 36.3; 750 over 2048 32.5 / 26.8 / 32.3 / 44.8.
  const float rows = (float)std::min(128L, (long)p.max_q * gp);
  float best = 0.f;
  for (int n = 1; n <= MAX_SPLIT && (n == 1 || (ctas * n <= 2L * sms && n <= ktiles)); n *= 2) {
    const float share = ctas * n > sms ? 1.6f : 1.f;
    const float t = 5.f + 0.82f * ((ktiles + n - 1) / n) * share + (n > 1 ? 1.f + 2.2f / 128.f * rows : 0.f);
    if (n == 1 || t < best) {
      best = t;
      a.split = n;
    }
  }
  a.tma_out = a.split == 1 && (long)p.max_q * gp >= 32 && gp <= 32 &&
              rows_map(o, p.out, p.q_rows, p.H, p.hd, gp, 32 / gp);
  const long listed = CTX4 && a.split == 1 ? list_tiles(p, gp, QT) : 0;
  if (listed && listed * (p.H / gp) < (1L << 31)) a.heads = p.H / gp;
  auto kernel = ctx_attn_tc_kernel<HDT, CTX4>;
  static std::atomic<uint64_t> told{0};
  allow_smem(kernel, C::SMEM, told);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = a.heads ? dim3((unsigned)(listed * a.heads)) : dim3((unsigned)(qtiles * a.split), p.H / gp, p.nseq);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)a.split, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  IRT_CUDA(cudaLaunchKernelEx(&cfg, kernel, q, ks, vs, k, v, g, o, a));
  IRT_CHECK_LAUNCH();
  return true;
}

}  // namespace

bool ctx_attention_tc(const CtxAttnParams& p, cudaStream_t s) {
  // The row maximum is taken before the scale, so the scale must be positive;
  // tensors must be readable and writable 16 bytes at a time.
  if (!p.bf16_io || p.hd > 128 || !(p.scale > 0.f) || p.H / (QT % p.G == 0 ? p.G : 1) > 65535) return false;
  const irt_rows* const rows[7] = {&p.q, &p.out, &p.gate, &p.k, &p.v, &p.ks, &p.vs};
  for (const irt_rows* r : rows)
    if (r->data && !rows_vec(*r, 1)) return false;
  // whole groups of codes, 16 bytes each
  if (p.kc && p.hd % KV4_GROUP) return false;
  if (p.kc) return p.hd > 64 ? launch<128, true>(p, s) : launch<64, true>(p, s);
  return p.hd > 64 ? launch<128, false>(p, s) : launch<64, false>(p, s);
}

CtxAttnStatus ctx_attn_status(int dev) {
  constexpr int MAX_DEVICES = 64;
  static std::atomic<int*> known[MAX_DEVICES];
  static std::atomic<int*> words{nullptr};
  static std::mutex mu;
  if (dev >= MAX_DEVICES) throw unsupported("more than 64 devices");
  int* w = words.load(std::memory_order_acquire);
  if (!w) {
    std::lock_guard<std::mutex> lk(mu);
    if (!(w = words.load(std::memory_order_acquire))) {
      // the first call of a process may be captured into a graph; this allocation is no part of it
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      IRT_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
      const cudaError_t e =
          cudaHostAlloc(reinterpret_cast<void**>(&w), MAX_DEVICES * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
      cudaThreadExchangeStreamCaptureMode(&mode);
      IRT_CUDA(e);
      std::memset(w, 0, MAX_DEVICES * sizeof(int));
      words.store(w, std::memory_order_release);
    }
  }
  int* p = known[dev].load(std::memory_order_relaxed);
  if (!p) {
    IRT_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_watchdog));
    known[dev].store(p, std::memory_order_relaxed);
  }
  return {p, w + dev};
}

void ctx_attn_report(CtxAttnParams& p, int dev) {
  const CtxAttnStatus st = ctx_attn_status(dev);
  if (*reinterpret_cast<volatile int*>(st.host))
    throw Error(IRT_E_CUDA,
                "a bounded wait inside an earlier attention operator expired: its outputs are invalid "
                "(irt_attention_check reports it and lets calls through again)");
  p.expired = st.device;
  p.expired_host = st.host;
}

int read_and_clear_ctx_attn_error(int dev) {
  const CtxAttnStatus st = ctx_attn_status(dev);
  const int v = read_and_clear_flag();
  *reinterpret_cast<volatile int*>(st.host) = 0;
  return v;
}

namespace {
__global__ void wait_probe_kernel(int waits, CtxAttnStatus report, unsigned long long* elapsed_ns) {
  __shared__ __align__(8) uint64_t bar;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar), 1);
    const uint64_t t0 = globaltimer();
    for (int i = 0; i < waits; ++i)
      wait_or_report(smem_u32(&bar), 0, report.device);  // phase 0 never completes
    *elapsed_ns = globaltimer() - t0;
    if (*reinterpret_cast<volatile int*>(report.device)) settle(report.host);
  }
}
}  // namespace

void ctx_attn_watchdog_probe(unsigned long long limit_ns, int waits, unsigned long long* elapsed_ns,
                             const CtxAttnStatus& report) {
  DevBuf d(sizeof(*elapsed_ns));
  IRT_CUDA(set_wait_limit_ns(limit_ns));
  wait_probe_kernel<<<1, 32>>>(waits, report, d.as<unsigned long long>());
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  IRT_CUDA(set_wait_limit_ns(DEFAULT_WAIT_LIMIT_NS));
  IRT_CUDA(e);
  IRT_CUDA(cudaMemcpy(elapsed_ns, d.p, sizeof(*elapsed_ns), cudaMemcpyDeviceToHost));
}

}  // namespace irt
