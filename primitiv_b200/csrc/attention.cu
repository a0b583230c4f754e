// Entry points of attention, and the pass over rows in front of the gradients.
#include <cmath>

#include "attention.h"
#include "ops_common.cuh"

namespace b200 {
namespace {

// Whether row t lies in a sequence.
__device__ __forceinline__ bool in_sequence(const uint32_t *starts, const uint32_t *lens, uint32_t pitch, uint32_t rows, uint32_t longest,
                                            uint32_t seqs, uint32_t t) {
  uint32_t i;
  if (starts) {
    uint32_t lo = 0, hi = seqs + 1;   // the last start at or before t
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (starts[mid] <= t) lo = mid + 1;
      else hi = mid;
    }
    if (lo == 0 || lo == seqs + 1) return false;
    i = lo - 1;
  } else {
    i = pitch ? t / pitch : seqs;
    if (i >= seqs) return false;
  }
  uint32_t first, len;
  attn_range(starts, lens, pitch, rows, longest, i, first, len);
  return t >= first && t - first < len;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// delta[h][t] = sum_d gy y, and the squares' sums that the kernels for halves take their scales from; one warp a head
// of a row.  Gradients of rows outside every sequence, which no other kernel touches, are stored as zeros here.
template <typename T>
__global__ void __launch_bounds__(256) attention_rows_kernel(AttnArgs a) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31u;
  const u64 nq = static_cast<u64>(a.rows_q) * a.heads_q, nk = static_cast<u64>(a.rows_k) * a.heads_k;
  for (u64 w = static_cast<u64>(blockIdx.x) * 8 + (threadIdx.x >> 5); w < nq + nk; w += static_cast<u64>(gridDim.x) * 8) {
    if (w < nq) {
      const uint32_t t = static_cast<uint32_t>(w / a.heads_q), h = static_cast<uint32_t>(w - static_cast<u64>(t) * a.heads_q);
      if (!in_sequence(a.q_starts, a.q_lens, a.q_pitch, a.rows_q, a.max_q, a.seqs, t)) {
        if (!a.accumulate)
          for (uint32_t d = lane; d < a.head; d += 32) st(static_cast<T *>(a.gq), t * a.q_ld + static_cast<u64>(h) * a.head + d, 0.f);
        continue;
      }
      const T *gy = static_cast<const T *>(a.gy) + t * a.y_ld + static_cast<u64>(h) * a.head;
      const T *y = static_cast<const T *>(a.y_in) + t * a.y_ld + static_cast<u64>(h) * a.head;
      float dot = 0.f, sq = 0.f;
      for (uint32_t d = lane; d < a.head; d += 32) {
        const float g = ld(gy, d);
        dot += g * ld(y, d);
        sq += g * g;
      }
      dot = warp_sum(dot);
      sq = warp_sum(sq);
      if (lane == 0) {
        a.delta[static_cast<u64>(h) * a.rows_q + t] = dot;
        a.gy_norm[static_cast<u64>(h) * a.rows_q + t] = sq;
      }
    } else {
      const u64 wk = w - nq;
      const uint32_t t = static_cast<uint32_t>(wk / a.heads_k), h = static_cast<uint32_t>(wk - static_cast<u64>(t) * a.heads_k);
      if (!in_sequence(a.k_starts, a.k_lens, a.k_pitch, a.rows_k, a.max_k, a.seqs, t)) {
        if (!a.accumulate)
          for (uint32_t d = lane; d < a.head; d += 32) {
            st(static_cast<T *>(a.gk), t * a.k_ld + static_cast<u64>(h) * a.head + d, 0.f);
            st(static_cast<T *>(a.gv), t * a.v_ld + static_cast<u64>(h) * a.head + d, 0.f);
          }
        continue;
      }
      const T *v = static_cast<const T *>(a.v) + t * a.v_ld + static_cast<u64>(h) * a.head;
      float sq = 0.f;
      for (uint32_t d = lane; d < a.head; d += 32) {
        const float x = ld(v, d);
        sq += x * x;
      }
      sq = warp_sum(sq);
      if (lane == 0) a.v_norm[static_cast<u64>(h) * a.rows_k + t] = sq;
    }
  }
}

int check_plan(const b200_attention *p, AttnArgs *a) {
  if (!p || p->head == 0 || p->heads_q == 0 || p->heads_k == 0 || p->heads_q % p->heads_k != 0) return B200_ERR_INVALID_ARG;
  if (p->head > kAttnMaxHead) return B200_ERR_TOO_LARGE;
  if (!std::isfinite(p->scale)) return B200_ERR_INVALID_ARG;
  // tiles are numbered in 32 bits
  if (static_cast<u64>(p->rows_q) * p->heads_q > 0x7fffffffu || static_cast<u64>(p->rows_k) * p->heads_k > 0x7fffffffu || p->seqs > 0x3fffffffu ||
      p->heads_k > 65535u)
    return B200_ERR_TOO_LARGE;
  *a = AttnArgs{};
  a->head = p->head, a->heads_q = p->heads_q, a->heads_k = p->heads_k, a->group = p->heads_q / p->heads_k;
  a->rows_q = p->rows_q, a->rows_k = p->rows_k, a->seqs = p->seqs;
  a->max_q = p->max_q && p->max_q < p->rows_q ? p->max_q : p->rows_q;
  a->max_k = p->max_k && p->max_k < p->rows_k ? p->max_k : p->rows_k;
  a->q_starts = p->q_starts, a->q_lens = p->q_lens, a->k_starts = p->k_starts, a->k_lens = p->k_lens;
  if (p->seqs) a->q_pitch = p->rows_q / p->seqs, a->k_pitch = p->rows_k / p->seqs;
  if (!a->q_starts && a->q_pitch < a->max_q) a->max_q = a->q_pitch;
  if (!a->k_starts && a->k_pitch < a->max_k) a->max_k = a->k_pitch;
  a->causal = p->causal != 0, a->scale = p->scale;
  const u64 dense_q = static_cast<u64>(p->heads_q) * p->head, dense_k = static_cast<u64>(p->heads_k) * p->head;
  a->q_ld = p->q_ld ? p->q_ld : dense_q, a->y_ld = p->y_ld ? p->y_ld : dense_q;
  a->k_ld = p->k_ld ? p->k_ld : dense_k, a->v_ld = p->v_ld ? p->v_ld : dense_k;
  if (a->q_ld < dense_q || a->y_ld < dense_q || a->k_ld < dense_k || a->v_ld < dense_k) return B200_ERR_INVALID_ARG;
  return B200_OK;
}

bool known_mode(int mode) { return mode >= B200_MODE_FP32_3XTF32 && mode <= B200_MODE_FP32_3XFP16; }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200_attention_bw_scratch(const b200_attention *plan_host, uint64_t *floats_host) {
  AttnArgs a;
  if (!floats_host) return B200_ERR_INVALID_ARG;
  if (const int rc = check_plan(plan_host, &a)) return rc;
  *floats_host = 2 * static_cast<u64>(a.rows_q) * a.heads_q + static_cast<u64>(a.rows_k) * a.heads_k;
  return B200_OK;
}

int b200_attention_fw(b200_ctx *ctx, int mode, const b200_attention *plan_host, const void *q, const void *k, const void *v, void *y,
                      float *lse, void *stream) {
  B200_OPS_PROLOGUE(ctx);
  AttnArgs a;
  if (const int rc = check_plan(plan_host, &a)) return rc;
  if (!known_mode(mode)) return B200_ERR_INVALID_ARG;
  if (a.rows_q == 0 || a.seqs == 0 || a.max_q == 0) return B200_OK;
  if (!q || !y || (a.rows_k > 0 && (!k || !v))) return B200_ERR_INVALID_ARG;
  a.q = q, a.k = k, a.v = v, a.y = y, a.lse = lse;
  ProfScope prof(ctx, kProfElementwise, s);
  int rc;
  if (static_cast<u64>(a.max_q) * a.group <= 32u && a.max_k > 0) rc = attention_tokens_fw(ctx, mode, a, s);
  else if (a.max_q > 64 && attention_tc_fw_eligible(ctx, mode, a)) rc = attention_tc_fw(ctx, a, s);
  else rc = attention_mma_fw(ctx, mode, a, s);
  if (rc != B200_OK) return rc;
  B200_OPS_EPILOGUE(ctx);
}

int b200_attention_bw(b200_ctx *ctx, int mode, const b200_attention *plan_host, const void *q, const void *k, const void *v, const void *y,
                      const float *lse, const void *gy, void *gq, void *gk, void *gv, float *scratch, int accumulate, void *stream) {
  B200_OPS_PROLOGUE(ctx);
  AttnArgs a;
  if (const int rc = check_plan(plan_host, &a)) return rc;
  if (!known_mode(mode)) return B200_ERR_INVALID_ARG;
  if (a.rows_q == 0 && a.rows_k == 0) return B200_OK;
  if (a.rows_q > 0 && (!q || !y || !lse || !gy || !gq)) return B200_ERR_INVALID_ARG;
  if (a.rows_k > 0 && (!k || !v || !gk || !gv)) return B200_ERR_INVALID_ARG;
  if (!scratch) return B200_ERR_INVALID_ARG;
  a.q = q, a.k = k, a.v = v, a.y_in = y, a.lse = const_cast<float *>(lse), a.gy = gy, a.gq = gq, a.gk = gk, a.gv = gv;
  a.accumulate = accumulate != 0;
  a.delta = scratch;
  a.gy_norm = a.delta + static_cast<u64>(a.rows_q) * a.heads_q;
  a.v_norm = a.gy_norm + static_cast<u64>(a.rows_q) * a.heads_q;
  ProfScope prof(ctx, kProfElementwise, s);
  const u64 rows = static_cast<u64>(a.rows_q) * a.heads_q + static_cast<u64>(a.rows_k) * a.heads_k;
  B200_DISPATCH_MODE(mode, { b200::launch(ctx, attention_rows_kernel<T>, dim3(grid_for(ctx, rows, 8)), dim3(256), 0, s, 1u, a); });
  ++ctx->launches;
  const int rc = attention_tc_bw_eligible(ctx, mode, a) ? attention_tc_bw(ctx, a, s) : attention_mma_bw(ctx, mode, a, s);
  if (rc != B200_OK) return rc;
  B200_OPS_EPILOGUE(ctx);
}

}  // extern "C"
