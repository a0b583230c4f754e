// Shared pieces of the attention kernels (attention.cu, attention_mma.cu).
#ifndef PRIMITIV_B200_CSRC_ATTENTION_H_
#define PRIMITIV_B200_CSRC_ATTENTION_H_

#include <cuda_fp16.h>

#include "../../include/primitiv_b200_attention.h"
#include "ctx.h"

namespace b200 {

constexpr uint32_t kAttnMaxHead = 256;

// One call, strides filled in.  Pointers of the pass that runs are set, the others null.
struct AttnArgs {
  const void *q, *k, *v, *y_in, *gy;
  void *y, *gq, *gk, *gv;
  float *lse;
  // scratch of the backward pass: [heads_q][rows_q] sums of gy y, as many squares' sums of gy, and
  // [heads_k][rows_k] squares' sums of v (kernels for halves only)
  float *delta, *gy_norm, *v_norm;
  unsigned long long q_ld, k_ld, v_ld, y_ld;
  const uint32_t *q_starts, *q_lens, *k_starts, *k_lens;
  uint32_t head, heads_q, heads_k, group;
  uint32_t rows_q, rows_k, seqs, max_q, max_k;
  uint32_t q_pitch, k_pitch;   // rows per sequence where there are no starts
  uint32_t q_each, k_each;     // how tiles are numbered, see attn_tiles
  int causal, accumulate;
  float scale;
};

// attention_mma.cu: every type, head and alignment
int attention_mma_fw(b200_ctx *ctx, int mode, const AttnArgs &a, cudaStream_t s);
int attention_mma_bw(b200_ctx *ctx, int mode, const AttnArgs &a, cudaStream_t s);

// attention_tokens.cu: a few queries per sequence
int attention_tokens_fw(b200_ctx *ctx, int mode, const AttnArgs &a, cudaStream_t s);
// attention_tc.cu: halves on tcgen05
bool attention_tc_fw_eligible(const b200_ctx *ctx, int mode, const AttnArgs &a);
int attention_tc_fw(b200_ctx *ctx, const AttnArgs &a, cudaStream_t s);
bool attention_tc_bw_eligible(const b200_ctx *ctx, int mode, const AttnArgs &a);
int attention_tc_bw(b200_ctx *ctx, const AttnArgs &a, cudaStream_t s);

#ifdef __CUDACC__

struct AttnSeq {
  uint32_t q0, lq, k0, lk;
};

// First row and length of sequence i on one side.  Whatever the arrays hold, what comes back lies within `rows`.
__device__ __forceinline__ void attn_range(const uint32_t *starts, const uint32_t *lens, uint32_t pitch, uint32_t rows, uint32_t longest,
                                           uint32_t i, uint32_t &first, uint32_t &len) {
  uint32_t span = pitch;
  if (starts) {
    first = min(starts[i], rows);
    const uint32_t end = min(starts[i + 1], rows);
    span = end > first ? end - first : 0u;
  } else {
    first = i * pitch;
  }
  len = min(min(span, lens ? lens[i] : span), longest);
}

__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs &a, uint32_t i) {
  AttnSeq s;
  attn_range(a.q_starts, a.q_lens, a.q_pitch, a.rows_q, a.max_q, i, s.q0, s.lq);
  attn_range(a.k_starts, a.k_lens, a.k_pitch, a.rows_k, a.max_k, i, s.k0, s.lk);
  return s;
}

// Sequence i has ceil(length * per / rows) tiles.  They are numbered through all sequences; or, if `each` is not 0, sequence i has
// the numbers from i * each on.  Finds the sequence of one tile and the tile's number within it, in the first case by the first
// warp for the whole block, 32 sequences a step.  False: there is no such tile.  kKeys: the keys are what is cut into tiles.
template <bool kKeys>
__device__ __forceinline__ bool attn_find_tile(const AttnArgs &a, uint32_t tile, uint32_t per, uint32_t rows, uint32_t *s_at, uint32_t &seq,
                                               uint32_t &within) {
  const uint32_t each = kKeys ? a.k_each : a.q_each;
  if (each) {
    __syncthreads();   // (as below: callers set up shared memory before)
    seq = tile / each;
    within = tile - seq * each;
    if (seq >= a.seqs) return false;
    uint32_t first, len;
    if (kKeys) attn_range(a.k_starts, a.k_lens, a.k_pitch, a.rows_k, a.max_k, seq, first, len);
    else attn_range(a.q_starts, a.q_lens, a.q_pitch, a.rows_q, a.max_q, seq, first, len);
    return static_cast<unsigned long long>(within) * rows < static_cast<unsigned long long>(len) * per;
  }
  if (threadIdx.x < 32u) {
    const uint32_t lane = threadIdx.x;
    uint32_t before = 0, found = 0xffffffffu, in = 0;
    for (uint32_t base = 0; base < a.seqs; base += 32u) {
      uint32_t n = 0;
      if (base + lane < a.seqs) {
        uint32_t first, len;
        if (kKeys) attn_range(a.k_starts, a.k_lens, a.k_pitch, a.rows_k, a.max_k, base + lane, first, len);
        else attn_range(a.q_starts, a.q_lens, a.q_pitch, a.rows_q, a.max_q, base + lane, first, len);
        n = static_cast<uint32_t>((static_cast<unsigned long long>(len) * per + rows - 1) / rows);
      }
      uint32_t sum = n;
#pragma unroll
      for (uint32_t o = 1; o < 32u; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, before + sum > tile);
      if (hit != 0u) {
        const uint32_t who = __ffs(hit) - 1u;
        found = base + who;
        in = tile - before - (__shfl_sync(0xffffffffu, sum, who) - __shfl_sync(0xffffffffu, n, who));
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) s_at[0] = found, s_at[1] = in;
  }
  __syncthreads();
  seq = s_at[0];
  within = s_at[1];
  return seq != 0xffffffffu;
}

__device__ __forceinline__ float attn_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The scale of ds for halves: the power of two that takes the largest |ds| possible to at most 2^14.  |dp - delta| <= |gy| |v| + |delta|.
__device__ __forceinline__ float attn_ds_scale(float gy_sq, float v_sq, float delta) {
  const float bound = sqrtf(gy_sq) * sqrtf(v_sq) + delta;
  if (!(bound > 1e-30f) || !(bound < 1e30f)) return 1.f;
  return exp2f(fminf(fmaxf(13.f - ceilf(log2f(bound)), -100.f), 100.f));
}
// The larger one, without x if that is an infinity or a NaN: what holds one has such gradients whatever the scale, and the others keep theirs.
__device__ __forceinline__ float attn_finite_max(float top, float x) { return x < INFINITY ? fmaxf(top, x) : top; }

#endif  // __CUDACC__

// The tiles of all sequences together, a bound, and how they are numbered.  Through all sequences there are few beyond those that exist, but
// a block looks for its own among the sequences, 0.1 us for 32 of them; with `each` numbers for every sequence it need not look, and
// blocks without a tile cost half a microsecond.  Returns 2^31 where there are too many.
inline unsigned long long attn_tiles(uint32_t total, uint32_t longest, uint32_t seqs, uint32_t per, uint32_t rows, uint32_t *each) {
  const unsigned long long through = static_cast<unsigned long long>(total) * per / rows + seqs;
  const unsigned long long one = (static_cast<unsigned long long>(longest) * per + rows - 1) / rows, apart = seqs * one;
  const bool look = apart > through && through * (seqs / 32 + 1) < 5 * apart;
  *each = look ? 0u : static_cast<uint32_t>(one);
  const unsigned long long n = look ? through : apart;
  return n < (1ull << 31) ? n : (1ull << 31);
}

}  // namespace b200

#endif  // PRIMITIV_B200_CSRC_ATTENTION_H_
