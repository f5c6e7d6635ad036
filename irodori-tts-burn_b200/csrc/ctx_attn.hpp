// Attention over context states (cross attention and attention over the 4-bit
// context cache): the parameter block that the entry points fill and every
// kernel reads, and the 4-bit format.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "common.hpp"
#include "kernels.hpp"

namespace irt {

// Values of one KV head's row that share a scale.
constexpr int KV4_GROUP = 32;
inline __host__ __device__ int kv4_groups(int hd) { return (hd + KV4_GROUP - 1) / KV4_GROUP; }

struct CtxAttnParams {
  int bf16_io;               // element type of q, k, v, gate, out: bf16 or f32
  int H, Hkv, hd, G;         // G = H / Hkv query heads read one KV head
  int nseq, max_q, max_k;
  float scale;
  long q_rows, k_rows;
  const irt_attn_seq* seqs;  // null: nseq sequences of max_q x max_k rows
  irt_rows q, gate, out;
  irt_rows k, v;             // native context (null data: none)
  irt_rows ks, vs;           // own rows (null data: none)
  const uint8_t *kc, *vc;    // 4-bit context codes (null: none)
  const bf16 *kscale, *vscale;
  const uint8_t* mask;       // [k_rows] or null
  float* lse;                // [q_rows, H] or null
  // Device memory that a bounded wait sets to 1 when it runs out; once it is
  // set, every wait that reports here gives up at once and later launches load
  // nothing: what they write means nothing.  The operators have one word per device (ctx_attn_status),
  // an engine has its own.
  int* expired;
  int* expired_host;         // a word in mapped host memory that a CTA with such a wait sets, or null
};

// Range of sequence n; false when its table entry reaches outside the tensors
// or the bounds that the launch was sized for (the sequence is skipped).
__device__ __forceinline__ bool ctx_attn_seq(const CtxAttnParams& p, int n, irt_attn_seq& sd) {
  if (!p.seqs) {
    sd = {n * p.max_q, p.max_q, n * p.max_k, p.max_k};  // checked on the host
    return true;
  }
  sd = p.seqs[n];
  return sd.q_start >= 0 && sd.q_len >= 0 && sd.q_len <= p.max_q && (long)sd.q_start + sd.q_len <= p.q_rows &&
         sd.k_start >= 0 && sd.k_len >= 0 && sd.k_len <= p.max_k && (long)sd.k_start + sd.k_len <= p.k_rows;
}

// Queues the attention on s (checks of arguments are done by the caller).
void ctx_attention(const CtxAttnParams& p, cudaStream_t s);

// The same on tcgen05 (ctx_attn_tc.cu): bf16, head_dim <= 128, 16-byte rows.
// Returns false, with nothing queued, where the call is outside what it handles.
bool ctx_attention_tc(const CtxAttnParams& p, cudaStream_t s);
// Few query rows over a 4-bit cache (ctx_attn_kv4.cu); false as above.
bool ctx_attention_kv4_rows(const CtxAttnParams& p, cudaStream_t s);
// Many query rows in f32 arithmetic, head_dim <= 128 (ctx_attn_tile.cu); false as above.
bool ctx_attention_tile(const CtxAttnParams& p, cudaStream_t s);
// Where waits of the operators on device `dev`, the current one, report: `device` as
// CtxAttnParams::expired, `host` as expired_host.  The host's word lets a call
// see an expired wait without waiting for the GPU; reading clears both.
struct CtxAttnStatus {
  int *device, *host;
};
CtxAttnStatus ctx_attn_status(int dev);
// Sets p's words to the operators'; throws while an expired wait is unreported.
void ctx_attn_report(CtxAttnParams& p, int dev);
int read_and_clear_ctx_attn_error(int dev);
// Test hook: `waits` bounded waits of the kernels on a barrier that nothing
// arrives on, with a limit of limit_ns each, reported to `expired`.
void ctx_attn_watchdog_probe(unsigned long long limit_ns, int waits, unsigned long long* elapsed_ns,
                             const CtxAttnStatus& report);

// cache rows [row_start, row_start + n) from source rows idx[i] (or i); see
// irt_kv4_append / irt_kv4_read.
void kv4_append(const irt_kv4_cache& c, int bf16_io, long row_start, long n, const irt_rows& k, const irt_rows& v,
                long src_rows, const int* idx, cudaStream_t s);
void kv4_read(const irt_kv4_cache& c, int bf16_io, long row_start, long n, const irt_rows& k, const irt_rows& v,
              cudaStream_t s);

// Checked argument blocks of the C entry points.
CtxAttnParams ctx_attn_params(const irt_attn_args& a, const irt_kv4_cache* cache, const irt_rows* k,
                              const irt_rows* v, long k_rows, const irt_rows* k_self, const irt_rows* v_self);
void kv4_check_cache(const irt_kv4_cache& c);
// Cache rows [row_start, row_start + n) against `ext_rows` rows of k and v
// (written: they are outputs) and n source indices (or null).
void kv4_check_rows(const irt_kv4_cache& c, int dtype, long row_start, long n, const irt_rows& k, const irt_rows& v,
                    long ext_rows, const int* idx, bool written);

// Sets the current device for one call and puts the caller's back.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    IRT_CUDA(cudaGetDevice(&prev));
    if (prev == dev) prev = -1;
    else IRT_CUDA(cudaSetDevice(dev));
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
};

}  // namespace irt
