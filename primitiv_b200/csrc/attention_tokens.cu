// Attention of a few queries per sequence against many keys: a step of generation, forward only.
//
// Bound by the cache, which is read once: 16 rows (queries times the heads of a group) share a key head's keys, and a 16-row
// mma.sync product costs less than its operands take to arrive.  A sequence's keys are cut over the blocks of a
// cluster and over the four warps of a block; every warp has a ring of its own, three steps deep, fed by cp.async,
// so that no warp waits for another while the keys stream.  Each keeps a running softmax; the parts are joined in
// shared memory and then across the cluster through distributed shared memory, in rank order: one launch, no scratch,
// the same bits every run.
#include <algorithm>
#include <atomic>

#include "attention_mma.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr uint32_t kWarps = 4, kThreads = kWarps * 32, kStages = 3;
constexpr uint32_t kMaxSplits = 16;
template <typename T> constexpr int kStep = sizeof(T) == 2 ? 16 : 8;   // keys per step of a warp
template <typename T, int kD> constexpr uint32_t kWarpBytes = kStages * 2 * kStep<T> * kPitch<T, kD> * sizeof(T);
// the ring, which the parts of the warps take over
template <typename T, int kD>
constexpr uint32_t kSmem = std::max<uint32_t>(kWarps * kWarpBytes<T, kD>, kWarps * 16 * kD * 4) + 16 * kPitch<T, kD> * sizeof(T);

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

template <typename T, int kD, int kPass>
__global__ void __launch_bounds__(kThreads) attention_tokens_kernel(AttnArgs a, uint32_t row_tiles, uint32_t splits, int wide) {
  pdl_enter();
  constexpr int BN = kStep<T>, NT = BN / 8, P = kPitch<T, kD>;
  extern __shared__ __align__(16) unsigned char s_raw[];
  __shared__ float s_m[kWarps][16], s_l[kWarps][16], s_top[16], s_sum[16], s_weight[kMaxSplits][16];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
  const uint32_t rank = splits > 1 ? blockIdx.x % splits : 0u, item = blockIdx.x / splits;
  const uint32_t row_tile = item % row_tiles, hk = item / row_tiles % a.heads_k, seq = item / row_tiles / a.heads_k;
  const AttnSeq q = attn_seq(a, seq);
  const uint32_t rows = q.lq * a.group, row0 = row_tile * 16u;
  if (row0 >= rows) return;   // the whole cluster
  T *sq = reinterpret_cast<T *>(s_raw), *ring = sq + 16 * P;
  T *mine = ring + warp * (kStages * 2 * BN * P);
  const T *qb = static_cast<const T *>(a.q) + q.q0 * a.q_ld + static_cast<unsigned long long>(hk) * a.group * a.head;
  const T *kb = static_cast<const T *>(a.k) + q.k0 * a.k_ld + static_cast<unsigned long long>(hk) * a.head;
  const T *vb = static_cast<const T *>(a.v) + q.k0 * a.v_ld + static_cast<unsigned long long>(hk) * a.head;
  const long long shift = static_cast<long long>(q.lk) - q.lq;
  uint32_t keys = q.lk;
  if (a.causal) {
    const long long seen = static_cast<long long>((min(row0 + 16u, rows) - 1u) / a.group) + shift + 1;
    keys = seen <= 0 ? 0u : min(keys, static_cast<uint32_t>(seen));
  }
  // this block's keys, in whole rounds of the four warps
  constexpr uint32_t kRound = kWarps * BN;
  const uint32_t rounds = (keys + kRound - 1) / kRound, per = (rounds + splits - 1) / splits;
  const uint32_t from = min(rank * per, rounds) * kRound, to = min(keys, min((rank + 1) * per, rounds) * kRound);
  const uint32_t first = from + warp * BN, steps = first < to ? (to - first + kRound - 1) / kRound : 0u;

  auto load_step = [&](uint32_t i) {
    if (i < steps) {
      T *at = mine + i % kStages * (2 * BN * P);
      load_rows<T, kD, BN, 32>(at, kb, a.k_ld, 1, first + i * kRound, to, a.head, wide & kWideK, lane);
      load_rows<T, kD, BN, 32>(at + BN * P, vb, a.v_ld, 1, first + i * kRound, to, a.head, wide & kWideV, lane);
    }
    copies_commit();
  };
  load_rows<T, kD, 16, kThreads>(sq, qb, a.q_ld, a.group, row0, rows, a.head, wide & kWideQ);
  copies_commit();
  load_step(0);
  load_step(1);
  copies_wait<2>();
  __syncthreads();

  uint32_t row[2];
  long long last[2];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    row[r] = row0 + g + r * 8;
    last[r] = row[r] >= rows ? -1 : (a.causal ? static_cast<long long>(row[r] / a.group) + shift : static_cast<long long>(q.lk) - 1);
    last[r] = min(last[r], static_cast<long long>(to) - 1);
  }
  float acc[kD / 8][4];
#pragma unroll
  for (int n = 0; n < kD / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  const float to2 = a.scale * kLog2e;

  for (uint32_t i = 0; i < steps; ++i) {
    copies_wait<1>();
    __syncwarp();          // every lane's copies of this step are in, and the step before is read
    load_step(i + 2);
    const T *sk = mine + i % kStages * (2 * BN * P);
    float s[NT][4];
    product_abt<kD, NT, kPass>(s, sq, sk);
    const uint32_t key0 = first + i * kRound;
    float top[2] = {-INFINITY, -INFINITY}, keep[2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool seen = static_cast<long long>(key0 + n * 8 + 2 * t + (e & 1)) <= last[e >> 1];
        s[n][e] = seen ? s[n][e] * to2 : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float now = fmaxf(m[r], quad_max(top[r])), base = now == -INFINITY ? 0.f : now;
      keep[r] = exp2_of<T>(m[r] - base);
      m[r] = now;
      l[r] *= keep[r];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_of<T>(s[n][r * 2 + e] - base);
          s[n][r * 2 + e] = p;
          l[r] += p;
        }
    }
    product_py<kD, kD, NT, kPass>(acc, s, sk + BN * P, 0, keep[0], keep[1]);
  }
  copies_wait<0>();

  // ---- the warps' parts ----
  float *part = reinterpret_cast<float *>(ring);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] = quad_sum(l[r]);
    if (t == 0) s_m[warp][g + r * 8] = m[r], s_l[warp][g + r * 8] = l[r];
  }
  __syncthreads();         // (and the ring is read)
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint32_t at = g + r * 8;
    float top = s_m[0][at];
#pragma unroll
    for (uint32_t w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][at]);
    const float factor = m[r] == -INFINITY ? 0.f : exp2_of<T>(m[r] - top);
    float *out = part + (warp * 16 + at) * kD + 2 * t;
#pragma unroll
    for (int n = 0; n < kD / 8; ++n) *reinterpret_cast<float2 *>(out + n * 8) = make_float2(acc[n][r * 2] * factor, acc[n][r * 2 + 1] * factor);
  }
  if (threadIdx.x < 16) {
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][threadIdx.x]);
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) sum += s_m[w][threadIdx.x] == -INFINITY ? 0.f : exp2_of<T>(s_m[w][threadIdx.x] - top) * s_l[w][threadIdx.x];
    s_top[threadIdx.x] = top, s_sum[threadIdx.x] = sum;
  }
  __syncthreads();
  const uint32_t here = min(rows - row0, 16u);
  for (uint32_t i = threadIdx.x; i < here * (kD / 4); i += kThreads) {
    float4 v = *reinterpret_cast<const float4 *>(part + i * 4);
#pragma unroll
    for (uint32_t w = 1; w < kWarps; ++w) {
      const float4 o = *reinterpret_cast<const float4 *>(part + w * 16 * kD + i * 4);
      v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
    }
    *reinterpret_cast<float4 *>(part + i * 4) = v;
  }

  // ---- the blocks' parts ----
  if (splits > 1) cluster_sync_all();
  else __syncthreads();
  if (threadIdx.x < 16) {
    float top = -INFINITY, sum = 0.f;
    float tops[kMaxSplits];
#pragma unroll
    for (uint32_t r = 0; r < kMaxSplits; ++r) {
      if (r < splits) {
        tops[r] = splits > 1 ? ld_cluster(map_to_cta(smem_u32(&s_top[threadIdx.x]), r)) : s_top[threadIdx.x];
        s_weight[r][threadIdx.x] = splits > 1 ? ld_cluster(map_to_cta(smem_u32(&s_sum[threadIdx.x]), r)) : s_sum[threadIdx.x];
        top = fmaxf(top, tops[r]);
      }
    }
#pragma unroll
    for (uint32_t r = 0; r < kMaxSplits; ++r)
      if (r < splits) {
        const float w = tops[r] == -INFINITY ? 0.f : exp2_of<T>(tops[r] - top);
        sum += w * s_weight[r][threadIdx.x];
        s_weight[r][threadIdx.x] = w;
      }
    const float inv = top == -INFINITY ? 0.f : 1.f / sum;
    for (uint32_t r = 0; r < splits; ++r) s_weight[r][threadIdx.x] *= inv;
    if (rank == 0 && a.lse && threadIdx.x < here) {
      const uint32_t tok = (row0 + threadIdx.x) / a.group, h = hk * a.group + row0 + threadIdx.x - tok * a.group;
      a.lse[static_cast<unsigned long long>(h) * a.rows_q + q.q0 + tok] = top == -INFINITY ? -INFINITY : top * kLn2 + logf(sum);
    }
  }
  __syncthreads();
  for (uint32_t i = rank * kThreads + threadIdx.x; i < here * (kD / 4); i += splits * kThreads) {
    const uint32_t at = i / (kD / 4), c = i % (kD / 4) * 4;
    if (c >= a.head) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t r = 0; r < splits; ++r) {
      const float4 o = splits > 1 ? ld_cluster4(map_to_cta(smem_u32(part + i * 4), r)) : *reinterpret_cast<const float4 *>(part + i * 4);
      const float w = s_weight[r][at];
      v[0] += w * o.x, v[1] += w * o.y, v[2] += w * o.z, v[3] += w * o.w;
    }
    const uint32_t tok = (row0 + at) / a.group, h = hk * a.group + row0 + at - tok * a.group;
    T *out = static_cast<T *>(a.y) + (q.q0 + tok) * a.y_ld + static_cast<unsigned long long>(h) * a.head + c;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < a.head) out[e] = round_to<T>(v[e]);
  }
  if (splits > 1) cluster_sync_all();   // nobody leaves while another reads its part
}

template <typename T, int kD, int kPass>
int launch_tokens(b200_ctx *ctx, const AttnArgs &a, cudaStream_t s) {
  constexpr uint32_t smem = kSmem<T, kD>;
  auto kernel = attention_tokens_kernel<T, kD, kPass>;
  if (const int rc = allow_smem(kernel, smem)) return rc;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return static_cast<int>(e);
  const uint32_t row_tiles = (a.max_q * a.group + 15u) / 16u;
  const unsigned long long items = static_cast<unsigned long long>(a.seqs) * a.heads_k * row_tiles;
  // Two blocks for every SM, and no more than 1024 keys for one, so that sequences of different lengths even out; two rounds of
  // the warps at least.
  const unsigned long long sms = static_cast<unsigned long long>(ctx->sm_count);
  const unsigned long long want = std::max((2 * sms + items - 1) / items, (a.max_k + 1023ull) / 1024ull);
  uint32_t splits = 1;
  while (splits < kMaxSplits && splits < want && a.max_k / (2 * splits) >= 2 * kWarps * kStep<T>) splits *= 2;
  if (items * splits > 0x7fffffffull) return B200_ERR_TOO_LARGE;
  b200::launch(ctx, kernel, dim3(static_cast<uint32_t>(items * splits)), dim3(kThreads), smem, s, splits, a, row_tiles, splits, find_wide(a, sizeof(T)));
  return B200_OK;
}

}  // namespace

int attention_tokens_fw(b200_ctx *ctx, int mode, const AttnArgs &a, cudaStream_t s) {
  return with_type(mode, [&](auto type, auto pass) {
    using T = decltype(type);
    return with_head<T, decltype(pass)::value>(a.head, [&](auto d) { return launch_tokens<T, decltype(d)::value, decltype(pass)::value>(ctx, a, s); });
  });
}

}  // namespace b200
