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

// Eight elements of a head's row from d on, zeros past `head`; one 16- or 32-byte piece where `wide`.
template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T *p, uint32_t d, uint32_t head, bool wide) {
  if (wide) {
    constexpr int N = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      Vec<T> x;
      if (d + i < head) x.load(p + d + i);
#pragma unroll
      for (int j = 0; j < N; ++j) v[i + j] = d + i < head ? x.get(j) : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = d + i < head ? ld(p, d + i) : 0.f;
  }
}

// delta[h][t] = sum_d gy y and, for halves, the squares' sums that their kernels take the scales of ds from.  Gradients of rows
// outside every sequence, which no other kernel touches, are stored as zeros here.  A warp takes a row; a group of lanes (the least
// power of two that holds a head at eight elements a lane) takes a head.  y and gy are read once, and v for halves; a warp that has
// its row's heads one after another waits for them (50 us at 29 % of DRAM for 4096 tokens, 37 heads of 128 each).
template <typename T>
__global__ void __launch_bounds__(256) attention_rows_kernel(AttnArgs a, uint32_t lanes, int wide) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31u, at = lane & (lanes - 1), group = lane / lanes, groups = 32u / lanes, d = at * 8u;
  constexpr bool kHalf = sizeof(T) == 2;
  const u64 rows = static_cast<u64>(a.rows_q) + a.rows_k;
  for (u64 w = static_cast<u64>(blockIdx.x) * 8 + (threadIdx.x >> 5); w < rows; w += static_cast<u64>(gridDim.x) * 8) {
    if (w < a.rows_q) {
      const uint32_t t = static_cast<uint32_t>(w);
      if (!in_sequence(a.q_starts, a.q_lens, a.q_pitch, a.rows_q, a.max_q, a.seqs, t)) {
        if (!a.accumulate)
          for (uint32_t i = lane; i < a.heads_q * a.head; i += 32) st(static_cast<T *>(a.gq), t * a.q_ld + i, 0.f);
        continue;
      }
      const T *gy = static_cast<const T *>(a.gy) + t * a.y_ld, *y = static_cast<const T *>(a.y_in) + t * a.y_ld;
#pragma unroll 2
      for (uint32_t h0 = 0; h0 < a.heads_q; h0 += groups) {
        const uint32_t h = h0 + group;
        float g[8], v[8], dot = 0.f, sq = 0.f;
        load8(g, gy + static_cast<u64>(h) * a.head, h < a.heads_q ? d : a.head, a.head, wide);
        load8(v, y + static_cast<u64>(h) * a.head, h < a.heads_q ? d : a.head, a.head, wide);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dot += g[i] * v[i];
          if constexpr (kHalf) sq += g[i] * g[i];
        }
        for (uint32_t o = 1; o < lanes; o <<= 1) {
          dot += __shfl_xor_sync(0xffffffffu, dot, o);
          if constexpr (kHalf) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        }
        if (at == 0 && h < a.heads_q) {
          a.delta[static_cast<u64>(h) * a.rows_q + t] = dot;
          if constexpr (kHalf) a.gy_norm[static_cast<u64>(h) * a.rows_q + t] = sq;
        }
      }
    } else {
      const uint32_t t = static_cast<uint32_t>(w - a.rows_q);
      if (!in_sequence(a.k_starts, a.k_lens, a.k_pitch, a.rows_k, a.max_k, a.seqs, t)) {
        if (!a.accumulate)
          for (uint32_t i = lane; i < a.heads_k * a.head; i += 32) {
            st(static_cast<T *>(a.gk), t * a.k_ld + i, 0.f);
            st(static_cast<T *>(a.gv), t * a.v_ld + i, 0.f);
          }
        continue;
      }
      if constexpr (!kHalf) continue;
      const T *v = static_cast<const T *>(a.v) + t * a.v_ld;
      for (uint32_t h0 = 0; h0 < a.heads_k; h0 += groups) {
        const uint32_t h = h0 + group;
        float x[8], sq = 0.f;
        load8(x, v + static_cast<u64>(h) * a.head, h < a.heads_k ? d : a.head, a.head, wide);
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += x[i] * x[i];
        for (uint32_t o = 1; o < lanes; o <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        if (at == 0 && h < a.heads_k) a.v_norm[static_cast<u64>(h) * a.rows_k + t] = sq;
      }
    }
  }
}

int check_plan(const b200_attention *p, AttnArgs *a) {
  if (!p || p->head == 0 || p->heads_q == 0 || p->heads_k == 0 || p->heads_q % p->heads_k != 0) return B200_ERR_INVALID_ARG;
  if (p->head > kAttnMaxHead) return B200_ERR_TOO_LARGE;
  if (!std::isfinite(p->scale)) return B200_ERR_INVALID_ARG;
  // Tiles, the rows of one that ends behind the last row, and the elements of a token are numbered in 32 bits.
  constexpr u64 kMostRows = 0x7fff0000u;
  if (static_cast<u64>(p->rows_q) * p->heads_q > kMostRows || static_cast<u64>(p->rows_k) * p->heads_k > kMostRows || p->seqs > 0x3fffffffu ||
      p->heads_k > 65535u || static_cast<u64>(p->heads_q) * p->head > 0x7fffffffu)
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
  uint32_t lanes = 1;
  while (lanes * 8 < a.head) lanes *= 2;
  const u64 es = elem_bytes(mode);
  const bool wide = aligned16(gy) && aligned16(y) && aligned16(v) && a.y_ld * es % 16 == 0 && a.v_ld * es % 16 == 0 && a.head * es % 16 == 0;
  B200_DISPATCH_MODE(mode, {
    b200::launch(ctx, attention_rows_kernel<T>, dim3(grid_for(ctx, static_cast<u64>(a.rows_q) + a.rows_k, 8)), dim3(256), 0, s, 1u, a, lanes, wide);
  });
  ++ctx->launches;
  const int rc = attention_tc_bw_eligible(ctx, mode, a) ? attention_tc_bw(ctx, a, s) : attention_mma_bw(ctx, mode, a, s);
  if (rc != B200_OK) return rc;
  B200_OPS_EPILOGUE(ctx);
}

}  // extern "C"
