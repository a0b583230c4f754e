// Pieces of the mma.sync attention kernels (attention_mma.cu, attention_tokens.cu): fragments and products of 16 rows per warp,
// tiles in shared memory, dispatch.
#ifndef PRIMITIV_B200_CSRC_ATTENTION_MMA_CUH_
#define PRIMITIV_B200_CSRC_ATTENTION_MMA_CUH_

#include <type_traits>

#include "attention.h"

namespace b200 {
namespace {   // each translation unit instantiates its own kernels

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ uint32_t smem_at(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---- fragments and products --------------------------------------------------------------------------------

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// x = hi + lo: hi is x rounded to TF32 by integer instructions; of what is left the tensor core takes the first 11 bits, all but one.
// A product loses 2^-21 of itself that way.  (cvt.rna.tf32 for both, with infinities kept, took seven instructions, and two thirds of the
// kernels' time.)  A NaN stays one, an infinity becomes one.
template <int kPass>
__device__ __forceinline__ void split(float x, uint32_t &hi, uint32_t &lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  if constexpr (kPass == 3) lo = __float_as_uint(x - __uint_as_float(hi));
  else if (x != x) hi = __float_as_uint(x);
}

// Row pitch of a tile in shared memory, in elements: 16 bytes more than the row, so that eight rows start in eight different
// groups of banks.
template <typename T, int kD> constexpr int kPitch = kD + 16 / static_cast<int>(sizeof(T));

// c[16 rows of this warp][8 NT] = X . Y^T, X and Y with contiguous rows of kD elements.
template <int kD, int NT, int kPass>
__device__ __forceinline__ void product_abt(float (&c)[NT][4], const __half *x, const __half *y) {
  constexpr int P = kPitch<__half, kD>;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t xa = smem_at(x) + ((lane & 15u) * P + (lane >> 4) * 8u) * 2u;
  const uint32_t ya = smem_at(y) + (((lane & 7u) + (lane >> 4) * 8u) * P + ((lane >> 3) & 1u) * 8u) * 2u;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[n][i] = 0.f;
#pragma unroll
  for (int kk = 0; kk < kD / 16; ++kk) {
    uint32_t a[4], b[4];
    ldsm4(a, xa + kk * 32);
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      ldsm4(b, ya + (n * 8 * P + kk * 16) * 2);
      mma_f16(c[n], a, b[0], b[1]);
      mma_f16(c[n + 1], a, b[2], b[3]);
    }
  }
}
template <int kD, int NT, int kPass>
__device__ __forceinline__ void product_abt(float (&c)[NT][4], const float *x, const float *y) {
  constexpr int P = kPitch<float, kD>;
  const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
  const float *xa = x + g * P + t, *ya = y + g * P + t;
  float small[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[n][i] = small[n][i] = 0.f;
#pragma unroll 4
  for (int kk = 0; kk < kD / 8; ++kk) {
    uint32_t ah[4], al[4];
    split<kPass>(xa[kk * 8], ah[0], al[0]);
    split<kPass>(xa[8 * P + kk * 8], ah[1], al[1]);
    split<kPass>(xa[kk * 8 + 4], ah[2], al[2]);
    split<kPass>(xa[8 * P + kk * 8 + 4], ah[3], al[3]);
    // The passes of one sum are NT instructions apart: behind one another they wait 30 clocks each.  The small terms have a sum of
    // their own, so that the large one is truncated once a step.
    uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      split<kPass>(ya[n * 8 * P + kk * 8], bh[n][0], bl[n][0]);
      split<kPass>(ya[n * 8 * P + kk * 8 + 4], bh[n][1], bl[n][1]);
    }
    if constexpr (kPass == 3) {
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_tf32(small[n], al, bh[n][0], bh[n][1]);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_tf32(small[n], ah, bl[n][0], bl[n][1]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) mma_tf32(c[n], ah, bh[n][0], bh[n][1]);
  }
  if constexpr (kPass == 3) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[n][i] += small[n][i];
  }
}

// acc[16 rows][kCols columns from col0] = acc * keep[row half] + P . Y, P in the accumulator layout [NT tiles of 8], Y of 8 NT rows.
template <int kD, int kCols, int NT, int kPass>
__device__ __forceinline__ void product_py(float (&acc)[kCols / 8][4], const float (&p)[NT][4], const __half *y, int col0, float keep0, float keep1) {
  constexpr int P = kPitch<__half, kD>;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t ya = smem_at(y) + ((lane & 15u) * P + (lane >> 4) * 8u + col0) * 2u;
  uint32_t a[NT / 2][4];
#pragma unroll
  for (int j = 0; j < NT / 2; ++j) {
    a[j][0] = half2_of(p[2 * j][0], p[2 * j][1]);
    a[j][1] = half2_of(p[2 * j][2], p[2 * j][3]);
    a[j][2] = half2_of(p[2 * j + 1][0], p[2 * j + 1][1]);
    a[j][3] = half2_of(p[2 * j + 1][2], p[2 * j + 1][3]);
  }
#pragma unroll
  for (int n = 0; n < kCols / 8; n += 2) {
    float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
      uint32_t b[4];
      ldsm4t(b, ya + (j * 16 * P + n * 8) * 2);
      mma_f16(c0, a[j], b[0], b[1]);
      mma_f16(c1, a[j], b[2], b[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float keep = i < 2 ? keep0 : keep1;
      acc[n][i] = acc[n][i] * keep + c0[i];
      acc[n + 1][i] = acc[n + 1][i] * keep + c1[i];
    }
  }
}
// The accumulator has columns 2t, 2t+1 where the left operand wants k = t, t+4: the rows of Y are taken in that order instead.
template <int kD, int kCols, int NT, int kPass>
__device__ __forceinline__ void product_py(float (&acc)[kCols / 8][4], const float (&p)[NT][4], const float *y, int col0, float keep0, float keep1) {
  constexpr int P = kPitch<float, kD>;
  const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
  const float *ya = y + 2 * t * P + g + col0;
  uint32_t ah[NT][4], al[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    split<kPass>(p[j][0], ah[j][0], al[j][0]);
    split<kPass>(p[j][2], ah[j][1], al[j][1]);
    split<kPass>(p[j][1], ah[j][2], al[j][2]);
    split<kPass>(p[j][3], ah[j][3], al[j][3]);
  }
  // four sums side by side, for the same reason as above
#pragma unroll
  for (int n0 = 0; n0 < kCols / 8; n0 += 4) {
    float c[4][4], small[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[n][i] = small[n][i] = 0.f;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      uint32_t bh[4][2], bl[4][2];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        split<kPass>(ya[j * 8 * P + (n0 + n) * 8], bh[n][0], bl[n][0]);
        split<kPass>(ya[j * 8 * P + P + (n0 + n) * 8], bh[n][1], bl[n][1]);
      }
      if constexpr (kPass == 3) {
#pragma unroll
        for (int n = 0; n < 4; ++n) mma_tf32(small[n], al[j], bh[n][0], bh[n][1]);
#pragma unroll
        for (int n = 0; n < 4; ++n) mma_tf32(small[n], ah[j], bl[n][0], bl[n][1]);
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) mma_tf32(c[n], ah[j], bh[n][0], bh[n][1]);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n0 + n][i] = acc[n0 + n][i] * (i < 2 ? keep0 : keep1) + (c[n][i] + small[n][i]);
  }
}

// ---- tiles ---------------------------------------------------------------------------------------------

// Rows [row0, row0 + ROWS) of a side into shared memory, zeros past `rows` and past `head`.  Row r is token r / per, head
// r % per behind `base` (per = 1: plain rows).  Copied in 16-byte pieces where every address allows, and then still in
// flight on return.
// `tid` of kThreads threads that load together.
template <typename T, int kD, int ROWS, int kThreads>
__device__ __forceinline__ void load_rows(T *dst, const T *base, unsigned long long ld, uint32_t per, uint32_t row0, uint32_t rows, uint32_t head, bool wide,
                                          uint32_t tid = threadIdx.x) {
  constexpr int P = kPitch<T, kD>, N = 16 / sizeof(T);
  if (wide) {
    constexpr uint32_t kPer = kD / N;
    for (uint32_t i = tid; i < ROWS * kPer; i += kThreads) {
      const uint32_t r = i / kPer, c = (i % kPer) * N, row = row0 + r;
      const T *from = base;
      uint32_t bytes = 0;
      if (row < rows && c < head) {
        const uint32_t tok = per == 1u ? row : row / per;
        from = base + tok * ld + static_cast<unsigned long long>(row - tok * per) * head + c;
        bytes = 16;
      }
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_at(dst + r * P + c)), "l"(from), "r"(bytes) : "memory");
    }
  } else {
    for (uint32_t i = tid; i < ROWS * kD; i += kThreads) {
      const uint32_t r = i / kD, c = i % kD, row = row0 + r;
      T v = T(0.f);
      if (row < rows && c < head) {
        const uint32_t tok = per == 1u ? row : row / per;
        v = base[tok * ld + static_cast<unsigned long long>(row - tok * per) * head + c];
      }
      dst[r * P + c] = v;
    }
  }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T> __device__ __forceinline__ T round_to(float v);
template <> __device__ __forceinline__ float round_to<float>(float v) { return v; }
template <> __device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }

// One row's columns of an accumulator: columns col0 + 8n + 2t, + 1.  Zeros in their place where not `some`, whatever they are.
template <typename T, int kCols>
__device__ __forceinline__ void store_row(T *out, const float (&acc)[kCols / 8][4], int half, int col0, uint32_t head, float factor, int accumulate,
                                          bool some = true) {
  const uint32_t t = threadIdx.x & 3u;
#pragma unroll
  for (int n = 0; n < kCols / 8; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t c = col0 + n * 8 + 2 * t + e;
      if (c < head) {
        float v = some ? acc[n][half * 2 + e] * factor : 0.f;
        if (accumulate) v += static_cast<float>(out[c]);
        out[c] = round_to<T>(v);
      }
    }
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
template <typename T> __device__ __forceinline__ float exp2_of(float x) {
  if constexpr (sizeof(T) == 2) return attn_exp2(x);
  else return exp2f(x);
}

// Shared memory of another block of the cluster.
__device__ __forceinline__ float ld_cluster(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

enum { kWideQ = 1, kWideK = 2, kWideV = 4, kWideGy = 8 };

int find_wide(const AttnArgs &a, size_t es) {
  auto ok = [&](const void *p, unsigned long long ld) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * es % 16 == 0 && a.head * es % 16 == 0;
  };
  return (ok(a.q, a.q_ld) ? kWideQ : 0) | (ok(a.k, a.k_ld) ? kWideK : 0) | (ok(a.v, a.v_ld) ? kWideV : 0) | (ok(a.gy, a.y_ld) ? kWideGy : 0);
}

// cudaFuncSetAttribute once per kernel and device would do; it is cheap beside a launch and needs no state.
template <typename K>
int allow_smem(K kernel, size_t smem) {
  return static_cast<int>(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
}

template <typename T, int kPass, typename F>
int with_head(uint32_t head, F f) {
  if (head <= 64) return f(std::integral_constant<int, 64>());
  if (head <= 128) return f(std::integral_constant<int, 128>());
  return f(std::integral_constant<int, 256>());
}

template <typename F>
int with_type(int mode, F f) {
  if (mode == B200_MODE_FP16) return f(__half(), std::integral_constant<int, 1>());
  if (mode == B200_MODE_TF32) return f(float(), std::integral_constant<int, 1>());
  return f(float(), std::integral_constant<int, 3>());
}

}  // namespace
}  // namespace b200

#endif  // PRIMITIV_B200_CSRC_ATTENTION_MMA_CUH_
