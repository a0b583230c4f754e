// Attention of a few queries per sequence against many keys: a step of generation, forward only.
//
// Bound by the cache, which is read once: 16 rows (queries times the heads of a group) share a key head's keys, and a 16-row
// mma.sync product costs less than its operands take to arrive, if little stands beside it.  So copies' addresses are one addition each, the
// queries stay in registers, masks are looked at in steps that need one, and y is rescaled only when the running maximum moves.
// (With addresses formed anew 16 keys took 860 instructions.  One bulk copy per row instead: an SM starts one in 30 clocks, which is
// 8 bytes a clock.)
// A sequence's keys are cut over the blocks of a cluster and over the four warps of a block; every warp has a ring of its own, so that no
// warp waits for another while the keys stream.  Each keeps a running softmax; the parts are joined in shared memory and then across
// the cluster through distributed shared memory, in rank order: one launch, no scratch, the same bits every run.
#include <algorithm>

#include "attention_mma.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr uint32_t kWarps = 4, kThreads = kWarps * 32;
constexpr uint32_t kMaxSplits = 16;
template <typename T> constexpr int kStep = sizeof(T) == 2 ? 16 : 8;   // keys per step of a warp
template <typename T, int kD> constexpr uint32_t kRing = sizeof(T) * kD > 512 ? 2 : 3;           // steps in a warp's ring
template <typename T, int kD> constexpr uint32_t kWarpBytes = kRing<T, kD> * 2 * kStep<T> * kPitch<T, kD> * sizeof(T);
template <typename T, int kD> constexpr uint32_t kQueryBytes = (sizeof(T) == 2 ? 1 : 2) * 16 * kPitch<T, kD> * sizeof(T);   // fp32: hi and lo
// the ring, which the parts of the warps take over
template <typename T, int kD>
constexpr uint32_t kSmem = std::max<uint32_t>(kWarps * kWarpBytes<T, kD>, kWarps * 16 * kD * 4) + kQueryBytes<T, kD>;

// s[16 rows][8 NT] = q k^T.  Halves: q in registers.
template <int kD, int NT>
__device__ __forceinline__ void scores(float (&s)[NT][4], const uint32_t (&qf)[kD / 16][4], const __half *k) {
  constexpr int P = kPitch<__half, kD>;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t ya = smem_at(k) + (((lane & 7u) + (lane >> 4) * 8u) * P + ((lane >> 3) & 1u) * 8u) * 2u;
  float even[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};   // two chains of sums for each tile of eight keys
  static_assert(NT == 2, "16 keys a step");
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
  for (int kk = 0; kk < kD / 16; ++kk) {
    uint32_t b[4];
    ldsm4(b, ya + kk * 32);
    if (kk & 1) {
      mma_f16(even, qf[kk], b[0], b[1]);
      mma_f16(odd, qf[kk], b[2], b[3]);
    } else {
      mma_f16(s[0], qf[kk], b[0], b[1]);
      mma_f16(s[1], qf[kk], b[2], b[3]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[0][i] += even[i], s[1][i] += odd[i];
}
// fp32: q split beforehand into planes hi and lo.
template <int kD, int NT, int kPass>
__device__ __forceinline__ void scores(float (&s)[NT][4], const float *q_hi, const float *q_lo, const float *k) {
  constexpr int P = kPitch<float, kD>;
  const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
  const uint32_t *hi = reinterpret_cast<const uint32_t *>(q_hi) + g * P + t, *lo = reinterpret_cast<const uint32_t *>(q_lo) + g * P + t;
  const float *ka = k + g * P + t;
  static_assert(NT == 1, "8 keys a step");
  float c[3][4] = {};   // hi hi, and a chain for either small term
#pragma unroll 4
  for (int kk = 0; kk < kD / 8; ++kk) {
    const uint32_t ah[4] = {hi[kk * 8], hi[8 * P + kk * 8], hi[kk * 8 + 4], hi[8 * P + kk * 8 + 4]};
    uint32_t bh[2], bl[2];
    split<kPass>(ka[kk * 8], bh[0], bl[0]);
    split<kPass>(ka[kk * 8 + 4], bh[1], bl[1]);
    if constexpr (kPass == 3) {
      const uint32_t al[4] = {lo[kk * 8], lo[8 * P + kk * 8], lo[kk * 8 + 4], lo[8 * P + kk * 8 + 4]};
      mma_tf32(c[1], al, bh[0], bh[1]);
      mma_tf32(c[2], ah, bl[0], bl[1]);
    }
    mma_tf32(c[0], ah, bh[0], bh[1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[0][i] = c[0][i] + (c[1][i] + c[2][i]);
}

// y += p v of one step.  Halves: summed by the tensor core (which truncates: 16384 keys lose 3e-5 of a sum, a tenth of its rounding).  p is rounded
// to half, which makes the error of y 2.7e-4 of its norm instead of 2.1e-4.  (With p as the sum of two halves, and two products, y is as good as
// its storage allows, but the instructions no longer hide behind the cache's way in: one token against 32768 keys 42.6 us instead of 38.2, 64
// tokens against up to 8192 keys 207 instead of 195.)
template <int kD, int kPass>
__device__ __forceinline__ void add_values(float (&acc)[kD / 8][4], const float (&p)[2][4], const __half *v) {
  constexpr int P = kPitch<__half, kD>;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t va = smem_at(v) + ((lane & 15u) * P + (lane >> 4) * 8u) * 2u;
  const uint32_t a[4] = {half2_of(p[0][0], p[0][1]), half2_of(p[0][2], p[0][3]), half2_of(p[1][0], p[1][1]), half2_of(p[1][2], p[1][3])};
#pragma unroll
  for (int n = 0; n < kD / 8; n += 2) {
    uint32_t b[4];
    ldsm4t(b, va + n * 16);
    mma_f16(acc[n], a, b[0], b[1]);
    mma_f16(acc[n + 1], a, b[2], b[3]);
  }
}
template <int kD, int kPass>
__device__ __forceinline__ void add_values(float (&acc)[kD / 8][4], const float (&p)[1][4], const float *v) {
  product_py<kD, kD, 1, kPass>(acc, p, v, 0, 1.f, 1.f);
}

template <typename T, int kD, int kPass>
__global__ void __launch_bounds__(kThreads) attention_tokens_kernel(AttnArgs a, uint32_t row_tiles, uint32_t splits, int wide) {
  pdl_enter();
  constexpr int BN = kStep<T>, NT = BN / 8, P = kPitch<T, kD>;
  constexpr uint32_t kStages = kRing<T, kD>;
  constexpr bool kHalf = sizeof(T) == 2;
  extern __shared__ __align__(16) unsigned char s_raw[];
  __shared__ float s_m[kWarps][16], s_l[kWarps][16], s_top[16], s_sum[16], s_weight[kMaxSplits][16];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
  const uint32_t rank = splits > 1 ? blockIdx.x % splits : 0u, item = blockIdx.x / splits;
  const uint32_t row_tile = item % row_tiles, hk = item / row_tiles % a.heads_k, seq = item / row_tiles / a.heads_k;
  const AttnSeq q = attn_seq(a, seq);
  const uint32_t rows = q.lq * a.group, row0 = row_tile * 16u;
  if (row0 >= rows) return;   // the whole cluster
  T *sq = reinterpret_cast<T *>(s_raw), *ring_at = reinterpret_cast<T *>(s_raw + kQueryBytes<T, kD>);
  T *mine = ring_at + warp * (kStages * 2 * BN * P);
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

  // Copies of a step: 32 lanes take whole rows or parts of them, 16 bytes each; a lane keeps its column and adds row strides.
  constexpr uint32_t kPer = kD * sizeof(T) / 16, kLanes = kPer < 32 ? kPer : 32, kRowsAt = 32 / kLanes, kParts = kPer / kLanes;
  const bool apart = (wide & (kWideK | kWideV)) != (kWideK | kWideV);
  const uint32_t lane_row = lane / kLanes, lane_col = lane % kLanes * (16 / sizeof(T));
  const unsigned long long lane_key = first + lane_row;
  const T *k_from = kb + lane_key * a.k_ld + lane_col, *v_from = vb + lane_key * a.v_ld + lane_col;
  const unsigned long long k_rows = kRowsAt * a.k_ld, v_rows = kRowsAt * a.v_ld;
  const uint32_t lane_to = smem_at(mine + lane_row * P + lane_col);
  uint32_t load_at = 0;
  auto copy_rows = [&](uint32_t to_at, const T *from_at, unsigned long long stride, uint32_t have) {
#pragma unroll
    for (uint32_t i = 0; i < BN / kRowsAt; ++i) {
#pragma unroll
      for (uint32_t part = 0; part < kParts; ++part) {
        const uint32_t col = part * kLanes * (16 / sizeof(T));
        const bool in = lane_col + col < a.head && i * kRowsAt + lane_row < have;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to_at + static_cast<uint32_t>((i * kRowsAt * P + col) * sizeof(T))), "l"(in ? from_at + col : kb), "r"(in ? 16u : 0u) : "memory");
      }
      from_at += stride;
    }
  };
  auto load_step = [&](uint32_t i) {
    if (i < steps) {
      const uint32_t key0 = first + i * kRound, have = min(to - key0, static_cast<uint32_t>(BN));
      if (apart) {
        T *at = mine + load_at * (2 * BN * P);
        load_rows<T, kD, BN, 32>(at, kb, a.k_ld, 1, key0, to, a.head, false, lane);
        load_rows<T, kD, BN, 32>(at + BN * P, vb, a.v_ld, 1, key0, to, a.head, false, lane);
      } else {
        const uint32_t to_at = lane_to + load_at * static_cast<uint32_t>(2 * BN * P * sizeof(T));
        copy_rows(to_at, k_from, k_rows, have);
        copy_rows(to_at + static_cast<uint32_t>(BN * P * sizeof(T)), v_from, v_rows, have);
        k_from += kRound * a.k_ld, v_from += kRound * a.v_ld;
      }
      if (++load_at == kStages) load_at = 0;
    }
    copies_commit();
  };
  load_rows<T, kD, 16, kThreads>(sq, qb, a.q_ld, a.group, row0, rows, a.head, wide & kWideQ);
  copies_commit();
#pragma unroll
  for (uint32_t i = 0; i + 1 < kStages; ++i) load_step(i);
  copies_wait<kStages - 1>();
  __syncthreads();          // queries
  uint32_t qf[kHalf ? kD / 16 : 1][4];
  if constexpr (kHalf) {
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk) ldsm4(qf[kk], smem_at(sq) + ((lane & 15u) * P + (lane >> 4) * 8u + kk * 16) * 2u);
  } else {
    for (uint32_t i = threadIdx.x; i < 16 * P; i += kThreads) {
      uint32_t hi, lo = 0;
      split<kPass>(sq[i], hi, lo);
      sq[i] = __uint_as_float(hi), sq[16 * P + i] = __uint_as_float(lo);
    }
    __syncthreads();
  }

  // the last key that each of this lane's two rows sees, and the first step in which one of the warp's rows does not see all
  uint32_t row[2];
  int last[2];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    row[r] = row0 + g + r * 8;
    long long see = row[r] >= rows ? static_cast<long long>(to) - 1 : (a.causal ? static_cast<long long>(row[r] / a.group) + shift : static_cast<long long>(q.lk) - 1);
    see = min(see, static_cast<long long>(to) - 1);
    last[r] = static_cast<int>(max(see, -1ll));
  }
  const int all = __reduce_min_sync(0xffffffffu, min(last[0], last[1])) + 1;   // keys that every row sees
  float acc[kD / 8][4];
#pragma unroll
  for (int n = 0; n < kD / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  const float to2 = a.scale * kLog2e;

  uint32_t at = 0;
  int key0 = static_cast<int>(first);
  for (uint32_t i = 0; i < steps; ++i, key0 += kRound) {
    copies_wait<kStages - 2>();
    __syncwarp();          // every lane's copies of this step are in, and the slot of the step before is read
    load_step(i + kStages - 1);
    const T *sk = mine + at * (2 * BN * P);
    float s[NT][4];
    if constexpr (kHalf) scores<kD, NT>(s, qf, sk);
    else scores<kD, NT, kPass>(s, sq, sq + 16 * P, sk);
    if (key0 + BN > all) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key0 + n * 8 + static_cast<int>(2 * t) + (e & 1) > last[e >> 1]) s[n][e] = -INFINITY;
          else s[n][e] *= to2;
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] *= to2;
    }
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
    top[0] = quad_max(top[0]), top[1] = quad_max(top[1]);
    if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float keep = top[r] == m[r] ? 1.f : exp2_of<T>(m[r] - top[r]);
        m[r] = top[r];
        l[r] *= keep;
#pragma unroll
        for (int n = 0; n < kD / 8; ++n) acc[n][2 * r] *= keep, acc[n][2 * r + 1] *= keep;
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float base = m[r] == -INFINITY ? 0.f : m[r];   // nothing seen yet: every p below is exp2(-inf)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_of<T>(s[n][r * 2 + e] - base);
          s[n][r * 2 + e] = p;
          l[r] += p;
        }
    }
    add_values<kD, kPass>(acc, s, sk + BN * P);
    if (++at == kStages) at = 0;
  }
  copies_wait<0>();

  // ---- the warps' parts ----
  float *part = reinterpret_cast<float *>(ring_at);
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
    for (uint32_t w = 0; w < kWarps; ++w)   // (a maximum of -infinity leaves out NaNs, so the sum counts all the same)
      sum += (s_m[w][threadIdx.x] == -INFINITY ? 0.f : exp2_of<T>(s_m[w][threadIdx.x] - top)) * s_l[w][threadIdx.x];
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
  // a query that sees no key has zeros, whatever the values that the others see hold
  auto sees_any = [&](uint32_t tok) { return a.causal ? static_cast<long long>(tok) + shift >= 0 : q.lk > 0u; };
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
    // (a row that sees scores of -infinity alone has 0 / 0)
    const uint32_t tok = (row0 + threadIdx.x) / a.group;
    const bool sees = sees_any(tok);
    const float inv = 1.f / sum;
    for (uint32_t r = 0; r < splits; ++r) s_weight[r][threadIdx.x] *= inv;
    if (rank == 0 && a.lse && threadIdx.x < here) {
      const uint32_t h = hk * a.group + row0 + threadIdx.x - tok * a.group;
      a.lse[static_cast<unsigned long long>(h) * a.rows_q + q.q0 + tok] = sees ? (top == -INFINITY ? 0.f : top * kLn2) + logf(sum) : -INFINITY;
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
    const bool sees = sees_any(tok);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < a.head) out[e] = round_to<T>(sees ? v[e] : 0.f);
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
  // Two blocks for every SM, and no more than 4096 keys for one, so that sequences of different lengths even out (64 sequences of up to
  // 8192 keys, after a pause: 182 us; with 1024 for one 251, more joins); two rounds of the warps at least.
  const unsigned long long sms = static_cast<unsigned long long>(ctx->sm_count);
  const unsigned long long want = std::max((2 * sms + items - 1) / items, (a.max_k + 4095ull) / 4096ull);
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
