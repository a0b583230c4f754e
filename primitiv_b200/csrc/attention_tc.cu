// Attention of halves on the tcgen05 tensor cores, for heads of up to 128 elements that TMA can address.
//
// Forward.  A block has two tiles of 128 queries that share their keys: two heads of one group where the group is
// even, else 256 queries of one head.  Warp 0 issues every matrix instruction, warp 1 every copy; warps 4-7 and
// 8-11 are the softmax of one tile each, a thread a row.  Keys and values come through a ring each.
//   tensor memory: s of tile 0, s of tile 1 (128 columns each), y of tile 0, y of tile 1
// p is written over s as halves, and is the left operand of p v from there: it never passes through shared memory.  While one
// tile's rows are in their softmax, the tensor core has the other tile's two products: per 128 keys of one tile 1024 clocks of
// matrix instructions stand against 16384 exponentials, which are 1024 clocks of the special function units.  The products run
// in the order in which they were issued, so p(j) v is read before s(j + 1) overwrites it.
// 16384 causal tokens of 32 heads of 128 on 8: 1.84 ms, 1.19 PFLOP/s, in ten calls after a pause; 2.08 ms, 1.06 PFLOP/s, in a long run, where
// the GPU's 1000 W hold the clock at about 1.55 GHz; 60 % of the tensor core's clocks.  (Figures of forms that were compared, here and below,
// are of ten calls after a pause, on one GPU each; this form had 1.82 ms there.)
// What is left is the way round: a softmax of 1700 clocks, two products, 600 clocks of waking one another.  Tried and no better: one place
// for s, which the tiles have in turn, p beside it (1.83 ms); the same with pairs of blocks that share each tile of keys and
// values, so that the tensor core reads less of shared memory (2.03 ms).
//
// The running maximum that scales y is only moved when a row has passed it by more than 2^8: until then p may exceed one (at most
// 256, exact enough in halves), and y stays in tensor memory untouched.  Moving it costs a pass over y, by the softmax
// warps themselves, a few times per row.
//
// Every wait is bounded, as in gemm_tc.cu.
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>

#include "attention.h"
#include "f32x2.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr uint32_t kTile = 128;                      // queries and keys of a tile
constexpr uint32_t kChunk = kTile * 128;             // bytes of 64 columns of a tile: 128-byte lines, swizzled
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// ---- matrix instructions ------------------------------------------------------------------------------------

// The instruction cache is what these warps wait for most: their code runs once per tile between two others that are unrolled over a
// row, and each line of it comes from afar (a wait that had nothing to wait for took 300 clocks, loop and bookkeeping as
// much again).  So a product is one run of eight instructions with little between them, waits keep their rare part elsewhere, and
// one lane is elected once.
// fp32 accumulator, both operands halves, M = 128, N columns; `mn`: the right operand lies N-major (its rows are k).
constexpr uint32_t idesc_of(uint32_t n, uint32_t mn) { return (1u << 4) | (mn << 16) | ((n >> 3) << 17) | ((kTile >> 4) << 24); }
// 128-byte swizzle, groups of eight lines 1024 bytes apart
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);


#define B200_MMA_SS "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, "
#define B200_MMA_TS "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %4, "
#define B200_NEXT_SS "add.u64 da, da, 2; add.u64 db, db, 2;\n\t"
#define B200_NEXT_TS(COLUMNS) "add.u32 a, a, " COLUMNS "; add.u64 db, db, 128;\n\t"

// d[128][128] = A . B^T over kD columns, both tiles of 128-byte lines in chunks of 64 columns.  All lanes of a converged warp, uniform
// arguments; `leader`: not 0 in the one lane that issues.
#define B200_NT_HEAD \
  "{\n\t.reg .pred e, t, f;\n\t.reg .b64 da, db;\n\t" \
  "setp.ne.b32 e, %5, 0; setp.eq.b32 t, %3, %3; setp.ne.b32 f, %3, %3;\n\tmov.b64 da, {%1, %3}; mov.b64 db, {%2, %3};\n\t"
#define B200_NT_FOUR(FIRST) \
  B200_MMA_SS FIRST ";\n\t" B200_NEXT_SS B200_MMA_SS "t;\n\t" B200_NEXT_SS B200_MMA_SS "t;\n\t" B200_NEXT_SS B200_MMA_SS "t;\n\t"
#define B200_NT_ARGS ::"r"(d), "r"((a & 0x3FFFFu) >> 4), "r"((b & 0x3FFFFu) >> 4), "r"(kDescHi), "r"(idesc), "r"(leader) : "memory"
template <int kD>
__device__ __forceinline__ void product_nt(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t leader) {
  static_assert(kChunk / 16 - 6 == 1018, "the step from the last of a chunk to the first of the next");
  if constexpr (kD == 64) asm volatile(B200_NT_HEAD B200_NT_FOUR("f") "}\n" B200_NT_ARGS);
  else asm volatile(B200_NT_HEAD B200_NT_FOUR("f") "add.u64 da, da, 1018; add.u64 db, db, 1018;\n\t" B200_NT_FOUR("t") "}\n" B200_NT_ARGS);
}
// d[128][N] (+)= P . B, P of 128 halves a row in tensor memory, B a tile of 128 rows in chunks of 64 columns.  kGap: p lies in runs of
// 16 columns, 32 apart.
#define B200_PN(EVEN) \
  "{\n\t.reg .pred e, t, f;\n\t.reg .b32 a;\n\t.reg .b64 db;\n\t" \
  "setp.ne.b32 e, %5, 0; setp.eq.b32 t, %3, %3; setp.ne.b32 f, %6, 0;\n\tmov.b32 a, %1; mov.b64 db, {%2, %3};\n\t" \
  B200_MMA_TS "f;\n\t" B200_NEXT_TS("8") B200_MMA_TS "t;\n\t" B200_NEXT_TS(EVEN) B200_MMA_TS "t;\n\t" B200_NEXT_TS("8") B200_MMA_TS "t;\n\t" \
  B200_NEXT_TS(EVEN) B200_MMA_TS "t;\n\t" B200_NEXT_TS("8") B200_MMA_TS "t;\n\t" B200_NEXT_TS(EVEN) B200_MMA_TS "t;\n\t" B200_NEXT_TS("8") \
  B200_MMA_TS "t;\n\t}\n"
#define B200_PN_ARGS \
  ::"r"(d), "r"(p), "r"(((b & 0x3FFFFu) >> 4) | ((kChunk >> 4) << 16)), "r"(kDescHi), "r"(idesc), "r"(leader), "r"(first ? 0u : 1u) : "memory"
template <bool kGap = false>
__device__ __forceinline__ void product_pn(uint32_t d, uint32_t p, uint32_t b, uint32_t idesc, bool first, uint32_t leader) {
  if constexpr (kGap) asm volatile(B200_PN("24") B200_PN_ARGS);
  else asm volatile(B200_PN("8") B200_PN_ARGS);
}
// Arrives on `bar` when every product issued so far is done.
__device__ __forceinline__ void commit(uint32_t bar, uint32_t leader) {
  asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar), "r"(leader) : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}\n" : "=r"(is));
  return is;
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- arithmetic ---------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t halves_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// The larger one, or a NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x without the special function unit: x = n + r, |r| <= 1/2, n by adding and taking away 1.5 2^23, whose last bits it then is; 2^r by a
// polynomial of degree 4 fitted for the least relative error (2.7e-6, a hundredth of what rounding to a half
// costs); 2^n is n in an exponent's place.  Below 2^-126: next to nothing, as it should be.  A NaN stays one.
__device__ __forceinline__ void exp2_by_products(f32x2 x, float &u, float &w) {
  constexpr float kMagic = 12582912.f;
  unpair(x, u, w);
  x = pair_of(max_nan(u, -126.f), max_nan(w, -126.f));
  const f32x2 t = add2(x, pair_of(kMagic, kMagic)), r = fma2(add2(t, pair_of(-kMagic, -kMagic)), pair_of(-1.f, -1.f), x);
  f32x2 y = fma2(r, pair_of(0.009570102f, 0.009570102f), pair_of(0.055917863f, 0.055917863f));
  y = fma2(y, r, pair_of(0.240247443f, 0.240247443f));
  y = fma2(y, r, pair_of(0.693121791f, 0.693121791f));
  y = fma2(y, r, pair_of(0.999999285f, 0.999999285f));
  unpair(t, u, w);
  unpair(mul2(y, pair_of(__uint_as_float((__float_as_uint(u) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(w) << 23) + 0x3f800000u))), u, w);
}
// Of eight pairs, kByProducts go that way: the special function units of an SM do 16 elements a clock, as many as its tensor core needs of
// them at full rate.  More of them cost more instructions than they save: a warp is alone on its scheduler for most of its softmax.
// (0, 1, 2 of 8: 1.84, 1.82, 1.86 ms for the 16384 tokens above.)
constexpr int kByProducts = 1;
__device__ __forceinline__ void exp2_pair(int nth, f32x2 x, float &u, float &w) {
  if ((nth & 7) < kByProducts) {
    exp2_by_products(x, u, w);
  } else {
    unpair(x, u, w);
    u = attn_exp2(u), w = attn_exp2(w);
  }
}

// All lanes of the warp.
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
  if (__builtin_expect(__all_sync(0xffffffffu, mbar_try_wait(bar, parity)), 1)) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// ---- forward ------------------------------------------------------------------------------------------------

struct alignas(64) FwParams {
  CUtensorMap q, k, v;
  AttnArgs a;
  uint32_t tiles, columns;   // tiles of all sequences (a bound); blocks per tile: heads, or pairs of them
  uint32_t two_heads;        // a block's two tiles are two heads; else 256 queries of one
  int *status;
};

// Three warps on each quarter of an SM; two of the first four only lend their registers.  (16384 tokens, 32 heads of 128 on 8, after a pause: 1812 us; with
// two threads a row, as the gradients have them, 2030, for what they have to tell one another; with p handed over in halves 1843.)
constexpr uint32_t kFwThreads = 384;
// Slots for tiles of keys and of values.
template <int kD> constexpr uint32_t kFwK = kD == 128 ? 2u : 4u;
template <int kD> constexpr uint32_t kFwV = kD == 128 ? 3u : 4u;
template <int kD> constexpr uint32_t kFwSmem = (2 + kFwK<kD> + kFwV<kD>) * kTile * kD * 2 + 1024;

template <int kD>
__global__ void __launch_bounds__(kFwThreads, 1) attention_fw_tc_kernel(const __grid_constant__ FwParams p) {
  constexpr uint32_t kBytes = kTile * kD * 2, kSlotsK = kFwK<kD>, kSlotsV = kFwV<kD>, kChunks = kD / 64;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full, k_full[kSlotsK], k_empty[kSlotsK], v_full[kSlotsV], v_empty[kSlotsV], s_full[2], p_full[2], y_done[2], v_clean, drain_bar;
  __shared__ uint32_t tmem_slot, s_at[2];
  __shared__ int s_abort;
  pdl_release_next();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u, k_ring = smem + 2 * kBytes, v_ring = k_ring + kSlotsK * kBytes;
  volatile int *abort_flag = &s_abort;
  const AttnArgs &a = p.a;
  if (threadIdx.x == 32u) {
    for (const CUtensorMap *m : {&p.q, &p.k, &p.v}) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<unsigned long long>(m)) : "memory");
  }
  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(smem_u32(&q_full), 1);
    for (uint32_t i = 0; i < kSlotsK; ++i) mbar_init(smem_u32(&k_full[i]), 1), mbar_init(smem_u32(&k_empty[i]), 1);
    for (uint32_t i = 0; i < kSlotsV; ++i) mbar_init(smem_u32(&v_full[i]), 1), mbar_init(smem_u32(&v_empty[i]), 1);
    for (uint32_t x = 0; x < 2; ++x) mbar_init(smem_u32(&s_full[x]), 1), mbar_init(smem_u32(&p_full[x]), 4), mbar_init(smem_u32(&y_done[x]), 1);
    mbar_init(smem_u32(&v_clean), 1);
    mbar_init(smem_u32(&drain_bar), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait_previous();
  tc_fence_before();
  // the last tiles of a causal sequence have the most keys: they go first
  const uint32_t column = blockIdx.x % p.columns, unit = p.two_heads ? kTile : 2 * kTile;
  uint32_t seq, tile;
  const bool any = attn_find_tile<false>(a, p.tiles - 1u - blockIdx.x / p.columns, 1, unit, s_at, seq, tile);
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (any) {
    const AttnSeq q = attn_seq(a, seq);
    const long long shift = static_cast<long long>(q.lk) - q.lq;
    const uint32_t head0 = p.two_heads ? 2 * column : column, kv_head = head0 / a.group, first_tok = tile * unit;
    auto head_of = [&](uint32_t x) { return head0 + (p.two_heads ? x : 0u); };
    auto tok_of = [&](uint32_t x) { return first_tok + (p.two_heads ? 0u : x * kTile); };
    // the keys that any of them sees: of two tiles of one head the first sees fewer, and has its last steps masked
    uint32_t keys = q.lk;
    if (a.causal) {
      const long long seen = static_cast<long long>(min(first_tok + unit, q.lq)) + shift;
      keys = seen <= 0 ? 0u : min(keys, static_cast<uint32_t>(seen));
    }
    const uint32_t steps = (keys + kTile - 1) / kTile, count = p.two_heads || first_tok + kTile < q.lq ? 2u : 1u;
    const uint32_t left = keys % kTile;   // keys in the last tile, 0 = all

    // 168 registers a thread at launch: 56 + 2 * 224 = 3 * 168
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 1) {
      // ------------------------------ copies ------------------------------
      if (steps > 0) {
        auto copy = [&](const CUtensorMap *map, uint32_t full, uint32_t dst, uint32_t j) {
          if (lane == 0) {
            mbar_arrive_expect_tx(full, kBytes);
            for (uint32_t c = 0; c < kChunks; ++c) tma_load_3d(dst + c * kChunk, map, full, c * 64, kv_head, q.k0 + j * kTile);
          }
          __syncwarp();
        };
        if (lane == 0) {
          mbar_arrive_expect_tx(smem_u32(&q_full), count * kBytes);
          for (uint32_t x = 0; x < count; ++x)
            for (uint32_t c = 0; c < kChunks; ++c) tma_load_3d(smem + x * kBytes + c * kChunk, &p.q, smem_u32(&q_full), c * 64, head_of(x), q.q0 + tok_of(x));
        }
        __syncwarp();
        uint32_t copied_k = 0, copied_v = 0;
        for (uint32_t j = 0; j < steps; ++j) {
          const uint32_t ks = j % kSlotsK, vs = j % kSlotsV;
          if (!wait_all(smem_u32(&k_empty[ks]), (j / kSlotsK & 1u) ^ 1u, abort_flag)) break;
          copy(&p.k, smem_u32(&k_full[ks]), k_ring + ks * kBytes, j);
          copied_k = j + 1;
          if (!wait_all(smem_u32(&v_empty[vs]), (j / kSlotsV & 1u) ^ 1u, abort_flag)) break;
          copy(&p.v, smem_u32(&v_full[vs]), v_ring + vs * kBytes, j);
          copied_v = j + 1;
        }
        // The last tile of values: rows behind the last key hold another sequence's, or anything; p is zero there, but zero
        // times an infinity is not.
        const uint32_t end = steps - 1u, last_at = v_ring + end % kSlotsV * kBytes;
        if (copied_v == steps && left != 0u && wait_all(smem_u32(&v_full[end % kSlotsV]), end / kSlotsV & 1u, abort_flag)) {
          for (uint32_t c = 0; c < kChunks; ++c)
            for (uint32_t at = left * 128u + lane * 16u; at < kChunk; at += 512u)
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(last_at + c * kChunk + at), "r"(0u) : "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&v_clean));
        }
        if (*abort_flag) {   // the copies in flight land before shared memory is given up
          mbar_wait_quiet(smem_u32(&q_full), 0);
          for (uint32_t j = copied_k > kSlotsK ? copied_k - kSlotsK : 0u; j < copied_k; ++j) mbar_wait_quiet(smem_u32(&k_full[j % kSlotsK]), j / kSlotsK & 1u);
          for (uint32_t j = copied_v > kSlotsV ? copied_v - kSlotsV : 0u; j < copied_v; ++j) mbar_wait_quiet(smem_u32(&v_full[j % kSlotsV]), j / kSlotsV & 1u);
        }
      }
    } else if (warp == 0) {
      // ------------------------------ products ------------------------------
      if (steps > 0) {
        constexpr uint32_t kS = idesc_of(kTile, 0), kY = idesc_of(kD, 1);
        const uint32_t leader = elect_one();
        const uint32_t s_done = smem_u32(&s_full[0]), p_done = smem_u32(&p_full[0]), made = smem_u32(&y_done[0]);
        uint32_t k_at = 0, k_phase = 0, v_at = 0, v_phase = 0;
        auto make_s = [&](uint32_t x) {
          if (x == 0 && !wait_all(smem_u32(&k_full[0]) + 8 * k_at, k_phase, abort_flag)) return false;
          product_nt<kD>(tmem + x * kTile, smem + x * kBytes, k_ring + k_at * kBytes, kS, leader);
          commit(s_done + 8 * x, leader);
          if (x + 1 == count) {
            commit(smem_u32(&k_empty[0]) + 8 * k_at, leader);
            if (++k_at == kSlotsK) k_at = 0, k_phase ^= 1u;
          }
          return true;
        };
        bool ok = wait_all(smem_u32(&q_full), 0, abort_flag) && make_s(0) && (count == 1u || make_s(1));
        for (uint32_t j = 0; ok && j < steps; ++j) {
          ok = wait_all(smem_u32(&v_full[0]) + 8 * v_at, v_phase, abort_flag) && (j + 1 < steps || left == 0u || wait_all(smem_u32(&v_clean), 0, abort_flag));
          for (uint32_t x = 0; ok && x < count; ++x) {
            if (!wait_all(p_done + 8 * x, j & 1u, abort_flag)) { ok = false; break; }
            tc_fence_after();
            product_pn(tmem + 2 * kTile + x * kD, tmem + x * kTile, v_ring + v_at * kBytes, kY, j == 0, leader);
            commit(made + 8 * x, leader);
            if (j + 1 < steps) ok = make_s(x);
          }
          commit(smem_u32(&v_empty[0]) + 8 * v_at, leader);
          if (++v_at == kSlotsV) v_at = 0, v_phase ^= 1u;
        }
        if (*abort_flag) {   // retire whatever was issued before tensor memory is freed
          __syncwarp();
          mma_commit(smem_u32(&drain_bar));
          mbar_wait_quiet(smem_u32(&drain_bar), 0);
        }
      }
    } else if (warp >= 4) {
      // ------------------------------ softmax ------------------------------
      asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
      const uint32_t x = (warp >> 2) - 1u, quarter = warp & 3u;
      const uint32_t lanes = (quarter * 32u) << 16, s_tmem = tmem + lanes + x * kTile, y_tmem = tmem + lanes + 2 * kTile + x * kD;
      const uint32_t tok = tok_of(x) + quarter * 32u + lane, n = x < count ? steps : 0u;
      // keys that this row sees
      long long sees = q.lk;
      if (a.causal) sees = min(sees, max(0ll, static_cast<long long>(tok) + 1 + shift));
      const float to2 = a.scale * kLog2e;
      float m = -INFINITY, l = 0.f;     // maximum in units of s, and the sum at that maximum
      bool ok = true;
      for (uint32_t j = 0; j < n; ++j) {
        if (!wait_all(smem_u32(&s_full[x]), j & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32_issue(s_tmem + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_wait(s[c]);
        const int seen = static_cast<int>(max(-1ll, min(sees - static_cast<long long>(j) * kTile, static_cast<long long>(kTile))));
        if (__any_sync(0xffffffffu, seen < static_cast<int>(kTile))) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= seen) s[c][i] = 0xff800000u;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2) top[(i >> 1) & 3] = max3_nan(top[(i >> 1) & 3], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
        const float now = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3]));
        // (a row that has seen nothing has m = -inf, and zeros for its sum and y; a NaN moves, and stays in both)
        const bool move = now != m && !((now - m) * to2 <= 8.f);
        if (j == 0) {
          m = now;
        } else if (__any_sync(0xffffffffu, move)) {
          const float keep = move ? attn_exp2((m - now) * to2) : 1.f;
          if (move) m = now;
          l *= keep;
          if (!wait_all(smem_u32(&y_done[x]), (j - 1) & 1u, abort_flag)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kD / 32; ++c) {
            uint32_t y[32];
            tmem_ld32(y_tmem + c * 32, y);
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * keep);
            tmem_st32(y_tmem + c * 32, y);
          }
        }
        const float base = m == -INFINITY ? 0.f : -m * to2;
        const f32x2 to22 = pair_of(to2, to2), base2 = pair_of(base, base);
        f32x2 sum[2] = {0ull, 0ull};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t out[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int c = h * 2 + i / 16, e = (i % 16) * 2;
            float u, w;
            exp2_pair(i, fma2(pair_of(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])), to22, base2), u, w);
            sum[i & 1] = add2(sum[i & 1], pair_of(u, w));
            out[i] = halves_of(u, w);
          }
          tmem_st32(s_tmem + h * 32, out);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_full[x]));
        float u, w;
        unpair(add2(sum[0], sum[1]), u, w);
        l += u + w;
      }
      if (ok && n > 0) ok = wait_all(smem_u32(&y_done[x]), (n - 1) & 1u, abort_flag);
      tc_fence_after();
      if (ok && x < count) {
        // a row that sees no key has zeros, one that sees scores of -infinity alone 0 / 0
        const bool some = sees > 0, mine = tok < q.lq;
        if (m == -INFINITY) l *= 0.f;         // next to nothing from exp2_by_products, or a NaN from before the row's last keys
        const float inv = 1.f / l;
        const uint32_t head = head_of(x);
        __half *out = static_cast<__half *>(a.y) + (q.q0 + tok) * a.y_ld + static_cast<unsigned long long>(head) * a.head;
#pragma unroll
        for (int c = 0; c < kD / 32; ++c) {
          uint32_t y[32];
          if (n > 0) tmem_ld32(y_tmem + c * 32, y);
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            if (mine && c * 32 + i < a.head) {
              uint4 o = make_uint4(0u, 0u, 0u, 0u);
              if (some) {
                o.x = halves_of(__uint_as_float(y[i]) * inv, __uint_as_float(y[i + 1]) * inv);
                o.y = halves_of(__uint_as_float(y[i + 2]) * inv, __uint_as_float(y[i + 3]) * inv);
                o.z = halves_of(__uint_as_float(y[i + 4]) * inv, __uint_as_float(y[i + 5]) * inv);
                o.w = halves_of(__uint_as_float(y[i + 6]) * inv, __uint_as_float(y[i + 7]) * inv);
              }
              *reinterpret_cast<uint4 *>(out + c * 32 + i) = o;
            }
          }
        }
        if (a.lse && mine) a.lse[static_cast<unsigned long long>(head) * a.rows_q + q.q0 + tok] = some ? (m == -INFINITY ? 0.f : m * to2 * kLn2) + logf(l) : -INFINITY;
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && s_abort) report_status(p.status, B200_ERR_KERNEL_TIMEOUT);
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ---- backward -----------------------------------------------------------------------------------------------
//
// Blocks of two kinds and one shape, as in attention_mma.cu, so that no sum needs atomics: with 128 keys at rest (gk and gv; the queries of
// all heads of the group pass by) and with 128 queries at rest (gq; the keys pass by).  X1, X2 rest, tiles Y1, Y2 come
// through a ring:
//   keys at rest     X1 = k, X2 = v, Y1 = q, Y2 = gy:   s' = k q^T, dp' = v gy^T,  gv += p' gy,  gk += ds' q
//   queries at rest  X1 = q, X2 = gy, Y1 = k, Y2 = v:   s = q k^T,  dp = gy v^T,   gq += ds k
// Transposed where the keys rest, so that p and ds are always the left operand, from tensor memory, and a tile in shared memory
// serves both as the right operand of the first products and of the second.  Sixteen warps share a tile: a thread has 32 of a
// row's 128 columns.  Four warps on a scheduler fill one another's waits, and 96 registers are enough without moving any.  (6 packed sequences of up to 4096 tokens, 16 heads of 128 on 4,
// forward and backward, ten calls after a pause: 794 us with eight warps of 64 columns a thread, 753 with sixteen; 868 with sixteen in a long run.)
//   keys at rest: the sums take half of tensor memory, so s and dp have one place between them: s(i) is in registers when dp(i) is
//     issued, and dp(i) is when s(i+1) is.  Order of the products: dp(i) s(i+1) gv(i), dp(i+1) gk(i) ...
//     (With places of their own, p written over s and ds over dp, s(i+1) waited for gv(i) and that for p(i): 3250 clocks a step.)
//   queries at rest: s(i+1) dp(i+1) gq(i), ds over dp, which has two buffers
// Bound by the tensor core, 2048 + 1536 clocks per 128 x 128 pairs, and as much by what shared memory has to read for it; the
// exponentials are 1024 of the special function units in each, of which exp2_pair takes a part over.
//
// p and ds are halves, which tensor memory and the products' rate ask for: the error of gk and gq against 64 bits is 3.1e-4 of their norm,
// where rounding the result alone makes 2.1e-4.  p is stored as 2^13 p; ds after a scale by a power of two from the largest |ds| that the norms of gy and v
// allow, over all that the block sees (keys at rest) or per query: without it the ds of long rows lie below the smallest half.

struct alignas(64) BwParams {
  CUtensorMap q, k, v, gy;
  AttnArgs a;
  uint32_t q_tiles, k_blocks;   // tiles of queries of all sequences (a bound); blocks with keys at rest, which come first
  int *status;
};

constexpr uint32_t kBwWarps = 16;                       // for p and ds; four more for products, copies and preparing tiles
constexpr uint32_t kBwThreads = (4 + kBwWarps) * 32;
constexpr float kPBits = 13.f;
// Slots of the rings.  Y1 is needed first and given back last, by the product that ends a step: with two slots its copy started a step
// late, and a step with queries at rest took 3500 clocks instead of 1900.
template <int kD> constexpr uint32_t kY1 = kD == 128 ? 3u : 4u;
template <int kD> constexpr uint32_t kY2 = kD == 128 ? 2u : 3u;
constexpr uint32_t kStats = 2;
constexpr uint32_t kBwHead = 3 * 1024;   // bytes in front of the tiles; with 7 tiles of 32 KB that is all there is
template <int kD> constexpr uint32_t kBwSmem = kBwHead + (2 + kY1<kD> + kY2<kD>) * kTile * kD * 2;

struct BwShared {
  float stat[kStats][2][kTile];      // keys at rest: 13 - lse log2(e), and -delta scaled, of the queries that pass by
  uint64_t x_full, full1[4], ready1[4], empty1[4], full2[4], ready2[4], empty2[4], s_full, s_read, dp_full[2], dp_read, p_full, ds_full[2], acc_done, drain;
  float top[3][kBwThreads / 32];
  uint32_t tmem, at[2];
  int abort;
};
static_assert(sizeof(BwShared) <= kBwHead, "no room");

// A position in a ring.
template <uint32_t kSlots>
struct Slot {
  uint32_t at = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++at == kSlots) at = 0, phase ^= 1u;
  }
};

// Four floats of shared memory as two pairs.
__device__ __forceinline__ void stat4(const float *p, f32x2 &a, f32x2 &b) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(p);
  a = v.x, b = v.y;
}

template <int kD, bool kKeys>
__device__ __forceinline__ void attention_bw_side(const BwParams &p, uint8_t *smem_raw) {
  constexpr uint32_t kBytes = kTile * kD * 2, kChunks = kD / 64, kSlots1 = kY1<kD>, kSlots2 = kY2<kD>;
  BwShared &sh = *reinterpret_cast<BwShared *>(smem_raw);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t smem = smem_u32(smem_raw) + kBwHead, ring1 = smem + 2 * kBytes, ring2 = ring1 + kSlots1 * kBytes;
  volatile int *abort_flag = &sh.abort;
  const AttnArgs &a = p.a;
  if (threadIdx.x == 32u) {
    for (const CUtensorMap *m : {&p.q, &p.k, &p.v, &p.gy}) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<unsigned long long>(m)) : "memory");
  }
  if (threadIdx.x == 0) {
    sh.abort = 0;
    for (uint64_t *one : {&sh.x_full, &sh.s_full, &sh.dp_full[0], &sh.dp_full[1], &sh.acc_done, &sh.drain}) mbar_init(smem_u32(one), 1);
    for (uint32_t i = 0; i < 4; ++i)
      for (uint64_t *one : {&sh.full1[i], &sh.ready1[i], &sh.empty1[i], &sh.full2[i], &sh.ready2[i], &sh.empty2[i]}) mbar_init(smem_u32(one), 1);
    for (uint64_t *warps : {&sh.s_read, &sh.dp_read, &sh.p_full, &sh.ds_full[0], &sh.ds_full[1]}) mbar_init(smem_u32(warps), kBwWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait_previous();
  tc_fence_before();
  // heaviest first: the first keys of a causal sequence are seen by the most queries, its last queries see the most keys
  const uint32_t block = kKeys ? blockIdx.x : blockIdx.x - p.k_blocks, columns = kKeys ? a.heads_k : a.heads_q;
  const uint32_t column = block % columns, nth = block / columns;
  uint32_t seq, tile;
  const bool any = attn_find_tile<kKeys>(a, kKeys ? nth : p.q_tiles - 1u - nth, 1, kTile, sh.at, seq, tile);
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  // columns of tensor memory.  Keys at rest: s and then dp, p, ds, two sums; queries at rest: s, two of dp and ds, the sum
  constexpr uint32_t kP = kTile, kDs = kTile + 64u, kDp = kTile, kAcc1 = 2 * kTile, kAcc2 = kKeys ? 2 * kTile + kD : 3 * kTile;

  if (any) {
    const AttnSeq q = attn_seq(a, seq);
    const long long shift = static_cast<long long>(q.lk) - q.lq;
    const uint32_t kv_head = kKeys ? column : column / a.group, q_head = kKeys ? column * a.group : column;
    const uint32_t row0 = tile * kTile, rows = kKeys ? q.lk : q.lq;
    // what passes by: `per` tiles from `from` on, for each head of the group where those are queries
    uint32_t from = 0, to = kKeys ? q.lq : q.lk;
    if (a.causal) {
      if (kKeys) {
        const long long first = static_cast<long long>(row0) - shift;
        from = first <= 0 ? 0u : (first >= q.lq ? q.lq : static_cast<uint32_t>(first));
      } else {
        const long long seen = static_cast<long long>(min(row0 + kTile, q.lq)) + shift;
        to = seen <= 0 ? 0u : min(to, static_cast<uint32_t>(seen));
      }
    }
    const uint32_t per = to > from ? (to - from + kTile - 1) / kTile : 0u, steps = kKeys ? per * a.group : per;
    const uint32_t left = (to - from) % kTile;
    const unsigned long long stat = static_cast<unsigned long long>(q_head) * a.rows_q + q.q0;

    // the scale of ds
    float gm = 0.f, dm = 0.f, vm = 0.f, ds_scale;
    {
      if constexpr (kKeys) {
        for (uint32_t g = 0; g < a.group; ++g)
#pragma unroll 4
          for (uint32_t t = from + threadIdx.x; t < q.lq; t += kBwThreads) {
            const unsigned long long i = stat + static_cast<unsigned long long>(g) * a.rows_q + t;
            gm = attn_finite_max(gm, a.gy_norm[i]);
            dm = attn_finite_max(dm, fabsf(a.delta[i]));
          }
      }
      const uint32_t k_from = kKeys ? row0 : 0u, k_to = kKeys ? min(row0 + kTile, rows) : to;
#pragma unroll 4
      for (uint32_t t = k_from + threadIdx.x; t < k_to; t += kBwThreads)
        vm = attn_finite_max(vm, a.v_norm[static_cast<unsigned long long>(kv_head) * a.rows_k + q.k0 + t]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
        dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, o));
        vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
      }
      if (lane == 0) sh.top[0][warp] = gm, sh.top[1][warp] = dm, sh.top[2][warp] = vm;
      __syncthreads();
#pragma unroll
      for (uint32_t w = 0; w < kBwThreads / 32; ++w) gm = fmaxf(gm, sh.top[0][w]), dm = fmaxf(dm, sh.top[1][w]), vm = fmaxf(vm, sh.top[2][w]);
      ds_scale = attn_ds_scale(gm, vm, dm);
    }

    if (warp == 1) {
      // ------------------------------ copies ------------------------------
      if (steps > 0) {
        const int x_row = (kKeys ? q.k0 : q.q0) + row0, x_head = kKeys ? kv_head : q_head;
        if (lane == 0) {
          mbar_arrive_expect_tx(smem_u32(&sh.x_full), 2 * kBytes);
          for (uint32_t c = 0; c < kChunks; ++c) {
            tma_load_3d(smem + c * kChunk, kKeys ? &p.k : &p.q, smem_u32(&sh.x_full), c * 64, x_head, x_row);
            tma_load_3d(smem + kBytes + c * kChunk, kKeys ? &p.v : &p.gy, smem_u32(&sh.x_full), c * 64, x_head, x_row);
          }
        }
        __syncwarp();
        Slot<kSlots1> s1;
        Slot<kSlots2> s2;
        uint32_t g = 0, t = 0, armed1 = 0, armed2 = 0, parity1 = 0, parity2 = 0;
        auto copy = [&](const CUtensorMap *map, uint32_t bar, uint32_t dst) {
          if (lane == 0) {
            const int head = kKeys ? q_head + g : kv_head, row = (kKeys ? q.q0 : q.k0) + from + t * kTile;
            mbar_arrive_expect_tx(bar, kBytes);
            for (uint32_t c = 0; c < kChunks; ++c) tma_load_3d(dst + c * kChunk, map, bar, c * 64, head, row);
          }
          __syncwarp();
        };
        for (uint32_t i = 0; i < steps; ++i) {
          if (!wait_all(smem_u32(&sh.empty1[s1.at]), s1.phase ^ 1u, abort_flag)) break;
          copy(kKeys ? &p.q : &p.k, smem_u32(&sh.full1[s1.at]), ring1 + s1.at * kBytes);
          armed1 |= 1u << s1.at, parity1 = (parity1 & ~(1u << s1.at)) | (s1.phase << s1.at);
          if (!wait_all(smem_u32(&sh.empty2[s2.at]), s2.phase ^ 1u, abort_flag)) break;
          copy(kKeys ? &p.gy : &p.v, smem_u32(&sh.full2[s2.at]), ring2 + s2.at * kBytes);
          armed2 |= 1u << s2.at, parity2 = (parity2 & ~(1u << s2.at)) | (s2.phase << s2.at);
          if (++t == per) t = 0, ++g;
          s1.next(), s2.next();
        }
        if (*abort_flag) {   // the copies in flight land before shared memory is given up
          mbar_wait_quiet(smem_u32(&sh.x_full), 0);
          for (uint32_t s = 0; s < 4; ++s) {
            if (armed1 & (1u << s)) mbar_wait_quiet(smem_u32(&sh.full1[s]), (parity1 >> s) & 1u);
            if (armed2 & (1u << s)) mbar_wait_quiet(smem_u32(&sh.full2[s]), (parity2 >> s) & 1u);
          }
        }
      }
    } else if (warp == 2) {
      // -------------------- what a tile needs before use: its rows' numbers, zeros behind its last row --------------------
      Slot<kSlots1> s1;
      Slot<kSlots2> s2;
      uint32_t g = 0, t = 0;
      auto clean = [&](uint32_t base) {   // p and ds are zero there, but zero times an infinity is not
        for (uint32_t c = 0; c < kChunks; ++c)
          for (uint32_t at = left * 128u + lane * 16u; at < kChunk; at += 512u)
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(base + c * kChunk + at), "r"(0u) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      };
      const float f = ds_scale * exp2f(-kPBits);
      for (uint32_t i = 0; i < steps; ++i) {
        if constexpr (kKeys) {
          float lse[4], delta[4];
#pragma unroll
          for (uint32_t c = 0; c < 4; ++c) {
            const uint32_t tok = from + t * kTile + c * 32u + lane;
            const unsigned long long at = stat + static_cast<unsigned long long>(g) * a.rows_q + tok;
            lse[c] = tok < q.lq ? a.lse[at] : 0.f;
            delta[c] = tok < q.lq ? a.delta[at] : 0.f;
          }
          // the numbers of two steps ago are done with when that step's ds is
          if (i >= kStats && !wait_all(smem_u32(&sh.ds_full[i & 1u]), ((i - kStats) >> 1) & 1u, abort_flag)) break;
#pragma unroll
          for (uint32_t c = 0; c < 4; ++c) {
            // (scores of -infinity alone have an lse of that too, and p is a NaN)
            sh.stat[i % kStats][0][c * 32u + lane] = from + t * kTile + c * 32u + lane < q.lq ? kPBits - lse[c] * kLog2e : -INFINITY;
            sh.stat[i % kStats][1][c * 32u + lane] = -delta[c] * f;
          }
        }
        const bool cut = t + 1 == per && left != 0u;
        if (!wait_all(smem_u32(&sh.full1[s1.at]), s1.phase, abort_flag)) break;
        if (cut) clean(ring1 + s1.at * kBytes);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.ready1[s1.at]));
        if (!wait_all(smem_u32(&sh.full2[s2.at]), s2.phase, abort_flag)) break;
        if (cut) clean(ring2 + s2.at * kBytes);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.ready2[s2.at]));
        if (++t == per) t = 0, ++g;
        s1.next(), s2.next();
      }
    } else if (warp == 0) {
      // ------------------------------ products ------------------------------
      if (steps > 0) {
        constexpr uint32_t kS = idesc_of(kTile, 0), kG = idesc_of(kD, 1);
        const uint32_t leader = elect_one();
        Slot<kSlots1> s1;   // of the next step
        Slot<kSlots2> s2;
        // (`ready` follows `full`, which is what orders the copies before the products)
        auto make_s = [&]() {
          if (!wait_all(smem_u32(&sh.ready1[s1.at]), s1.phase, abort_flag) || !wait_all(smem_u32(&sh.full1[s1.at]), s1.phase, abort_flag)) return false;
          product_nt<kD>(tmem, smem, ring1 + s1.at * kBytes, kS, leader);
          commit(smem_u32(&sh.s_full), leader);
          return true;
        };
        auto make_dp = [&](uint32_t d, uint32_t b) {
          if (!wait_all(smem_u32(&sh.ready2[s2.at]), s2.phase, abort_flag) || !wait_all(smem_u32(&sh.full2[s2.at]), s2.phase, abort_flag)) return false;
          product_nt<kD>(tmem + d, smem + kBytes, ring2 + s2.at * kBytes, kS, leader);
          commit(smem_u32(&sh.dp_full[b]), leader);
          if (!kKeys) commit(smem_u32(&sh.empty2[s2.at]), leader);
          return true;
        };
        auto heard = [&](uint64_t *bar, uint32_t parity) {
          if (!wait_all(smem_u32(bar), parity, abort_flag)) return false;
          tc_fence_after();
          return true;
        };
        bool ok = wait_all(smem_u32(&sh.x_full), 0, abort_flag) && make_s();
        if constexpr (kKeys) {
          ok = ok && heard(&sh.s_read, 0) && make_dp(0, 0);
          for (uint32_t i = 0; ok && i < steps; ++i) {
            const uint32_t at1 = s1.at, at2 = s2.at;
            const bool more = i + 1 < steps;
            s1.next(), s2.next();
            if (more) ok = heard(&sh.dp_read, i & 1u) && make_s();
            if (!ok || !heard(&sh.p_full, i & 1u)) { ok = false; break; }
            product_pn(tmem + kAcc1, tmem + kP, ring2 + at2 * kBytes, kG, i == 0, leader);
            commit(smem_u32(&sh.empty2[at2]), leader);
            if (more) ok = heard(&sh.s_read, (i + 1) & 1u) && make_dp(0, 0);
            if (!ok || !heard(&sh.ds_full[i & 1u], (i >> 1) & 1u)) { ok = false; break; }
            product_pn(tmem + kAcc2, tmem + kDs, ring1 + at1 * kBytes, kG, i == 0, leader);
            commit(smem_u32(&sh.empty1[at1]), leader);
          }
        } else {
          ok = ok && make_dp(kDp, 0);
          for (uint32_t i = 0; ok && i < steps; ++i) {
            const uint32_t at1 = s1.at, b = i & 1u;
            s1.next(), s2.next();
            if (i + 1 < steps) ok = heard(&sh.s_read, b) && make_s() && make_dp(kDp + (b ^ 1u) * kTile, b ^ 1u);
            if (!ok || !heard(&sh.ds_full[b], (i >> 1) & 1u)) { ok = false; break; }
            product_pn<true>(tmem + kAcc2, tmem + kDp + b * kTile, ring1 + at1 * kBytes, kG, i == 0, leader);
            commit(smem_u32(&sh.empty1[at1]), leader);
          }
        }
        if (ok) commit(smem_u32(&sh.acc_done), leader);
        if (*abort_flag) {   // retire whatever was issued before tensor memory is freed
          __syncwarp();
          mma_commit(smem_u32(&sh.drain));
          mbar_wait_quiet(smem_u32(&sh.drain), 0);
        }
      }
    } else if (warp >= 4) {
      // ------------------------------ p and ds ------------------------------
      const uint32_t part = (warp >> 2) - 1u, quarter = warp & 3u, col0 = part * 32u;   // a thread has 32 of a row's 128 columns
      const uint32_t lanes = (quarter * 32u) << 16, s_tmem = tmem + lanes + col0;
      const uint32_t row = row0 + quarter * 32u + lane;
      const float to2 = a.scale * kLog2e;
      float base = 0.f, minus_delta = 0.f;
      long long sees = q.lk;
      if constexpr (!kKeys) {
        if (a.causal) sees = min(sees, max(0ll, static_cast<long long>(row) + 1 + shift));
        if (row < rows) {
          base = sees > 0 ? -a.lse[stat + row] * kLog2e : 0.f;   // (a query that sees nothing: every column below is masked)
          const float delta = a.delta[stat + row];
          ds_scale = attn_ds_scale(a.gy_norm[stat + row], vm, fabsf(delta));
          minus_delta = -delta * ds_scale;
        }
      }
      const float f = kKeys ? ds_scale * exp2f(-kPBits) : ds_scale;
      const f32x2 to22 = pair_of(to2, to2), f2 = pair_of(f, f), base2 = pair_of(base, base), minus_delta2 = pair_of(minus_delta, minus_delta);
      Slot<kSlots1> s1;
      uint32_t t = 0;
      bool ok = true;
      for (uint32_t i = 0; i < steps; ++i) {
        const uint32_t b = i & 1u, dp_tmem = tmem + lanes + (kKeys ? 0u : kDp + b * kTile) + col0;
        const float *stat0 = sh.stat[i % kStats][0] + col0, *stat1 = sh.stat[i % kStats][1] + col0;
        if (kKeys && !wait_all(smem_u32(&sh.ready1[s1.at]), s1.phase, abort_flag)) { ok = false; break; }
        if (!wait_all(smem_u32(&sh.s_full), i & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        uint32_t s[32];
        tmem_ld32(s_tmem, s);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.s_read));
        // columns of this thread that its row has no part in: [0, skip) where queries pass by, [skip, 32) where keys do
        int skip;
        if constexpr (kKeys) {
          const long long first = a.causal ? static_cast<long long>(row) - shift - (from + static_cast<long long>(t) * kTile) - col0 : 0ll;
          skip = static_cast<int>(max(0ll, min(first, 32ll)));
        } else {
          skip = static_cast<int>(max(0ll, min(sees - static_cast<long long>(i) * kTile - col0, 32ll)));
        }
        if (__any_sync(0xffffffffu, kKeys ? skip > 0 : skip < 32)) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (kKeys ? e < skip : e >= skip) s[e] = 0xff800000u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          f32x2 add[2] = {base2, base2};
          if constexpr (kKeys) stat4(stat0 + e, add[0], add[1]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int at = e + 2 * k;
            float u, w;
            exp2_pair(at / 2, fma2(pair_of(__uint_as_float(s[at]), __uint_as_float(s[at + 1])), to22, add[k]), u, w);
            s[at] = __float_as_uint(u), s[at + 1] = __float_as_uint(w);
          }
        }
        if (!wait_all(smem_u32(&sh.dp_full[kKeys ? 0u : b]), (kKeys ? i : i >> 1) & 1u, abort_flag)) { ok = false; break; }
        tc_fence_after();
        uint32_t d[32], out[16];
        tmem_ld32(dp_tmem, d);
        if constexpr (kKeys) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh.dp_read));
          // (dp(i) is issued behind gv(i - 1), so p(i - 1) is read)
#pragma unroll
          for (int e = 0; e < 16; ++e) out[e] = halves_of(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
          tmem_st16(tmem + lanes + kP + part * 16u, out);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sh.p_full));
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          f32x2 add[2] = {minus_delta2, minus_delta2};
          if constexpr (kKeys) stat4(stat1 + e, add[0], add[1]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int at = e + 2 * k;
            float u, w;
            unpair(mul2(pair_of(__uint_as_float(s[at]), __uint_as_float(s[at + 1])),
                        fma2(pair_of(__uint_as_float(d[at]), __uint_as_float(d[at + 1])), f2, add[k])), u, w);
            out[at / 2] = halves_of(u, w);
          }
        }
        if constexpr (kKeys) {   // gk(i - 1) has read its ds
          if (i > 0 && !wait_all(smem_u32(&sh.empty1[(i - 1) % kSlots1]), ((i - 1) / kSlots1) & 1u, abort_flag)) { ok = false; break; }
          tc_fence_after();
        }
        tmem_st16(kKeys ? tmem + lanes + kDs + part * 16u : dp_tmem, out);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.ds_full[b]));
        if (++t == per) t = 0;
        s1.next();
      }
      if (ok && steps > 0) ok = wait_all(smem_u32(&sh.acc_done), 0, abort_flag);
      tc_fence_after();
      if (ok) {
        // keys at rest: half of gv's columns by either of the first two fours of warps, of gk's by the others; queries at rest: a quarter
        // of gq's columns each
        const bool is_v = kKeys && part < 2u;
        const float undo = is_v ? exp2f(-kPBits) : a.scale / ds_scale;
        const bool some = steps > 0 && (kKeys || sees > 0);   // a query that sees no key has zeros, whatever it and the keys hold
        constexpr int kCols = kKeys ? kD / 2 : kD / 4;
        const uint32_t c0 = (kKeys ? part & 1u : part) * kCols;
        const uint32_t acc = tmem + lanes + (is_v ? kAcc1 : kAcc2) + c0;
        __half *out;
        if constexpr (kKeys)
          out = is_v ? static_cast<__half *>(a.gv) + (q.k0 + static_cast<unsigned long long>(row)) * a.v_ld + static_cast<unsigned long long>(kv_head) * a.head
                     : static_cast<__half *>(a.gk) + (q.k0 + static_cast<unsigned long long>(row)) * a.k_ld + static_cast<unsigned long long>(kv_head) * a.head;
        else
          out = static_cast<__half *>(a.gq) + (q.q0 + static_cast<unsigned long long>(row)) * a.q_ld + static_cast<unsigned long long>(q_head) * a.head;
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
          uint32_t y[16];
          if (steps > 0) tmem_ld16(acc + c, y);
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            if (row < rows && c0 + c + e < a.head) {
              float v[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] = some ? __uint_as_float(y[e + k]) * undo : 0.f;
              uint4 *to16 = reinterpret_cast<uint4 *>(out + c0 + c + e);
              if (a.accumulate) {
                const uint4 old = *to16;
                const uint32_t words[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float2 o = __half22float2(*reinterpret_cast<const __half2 *>(&words[k]));
                  v[2 * k] += o.x, v[2 * k + 1] += o.y;
                }
              }
              *to16 = make_uint4(halves_of(v[0], v[1]), halves_of(v[2], v[3]), halves_of(v[4], v[5]), halves_of(v[6], v[7]));
            }
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && sh.abort) report_status(p.status, B200_ERR_KERNEL_TIMEOUT);
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// Both kinds in one launch: either alone leaves SMs idle behind its last blocks.
template <int kD>
__global__ void __launch_bounds__(kBwThreads, 1) attention_bw_tc_kernel(const __grid_constant__ BwParams p) {
  pdl_release_next();   // (pdl_wait_previous(); comes behind the set-up, in either)
  extern __shared__ __align__(1024) uint8_t bw_smem[];
  if (blockIdx.x < p.k_blocks) attention_bw_side<kD, true>(p, bw_smem);
  else attention_bw_side<kD, false>(p, bw_smem);
}

// ---- launches ------------------------------------------------------------------------------------------------

// Shape({head, heads, rows}) in boxes of 64 elements of one head of 128 rows; what lies past the head or the rows reads as zero.
int encode(const b200_ctx *ctx, CUtensorMap *map, const void *p, uint32_t head, uint32_t heads, uint32_t rows, unsigned long long ld) {
  cuuint64_t dims[3] = {head, heads, rows}, strides[2] = {head * 2ull, ld * 2ull};
  cuuint32_t box[3] = {64, 1, kTile}, step[3] = {1, 1, 1};
  const CUresult r = ctx->encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(p), dims, strides, box, step,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200_OK : B200_ERR_DRIVER;
}

bool addressable(const void *p, unsigned long long ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && ld * 2 < (1ull << 40); }

template <int kD>
int launch_fw(b200_ctx *ctx, const FwParams &p, cudaStream_t s) {
  auto kernel = attention_fw_tc_kernel<kD>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kFwSmem<kD>));
  if (e != cudaSuccess) return static_cast<int>(e);
  b200::launch(ctx, kernel, dim3(p.tiles * p.columns), dim3(kFwThreads), kFwSmem<kD>, s, 1u, p);
  return B200_OK;
}

template <int kD>
int launch_bw(b200_ctx *ctx, const BwParams &p, uint32_t blocks, cudaStream_t s) {
  auto kernel = attention_bw_tc_kernel<kD>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kBwSmem<kD>));
  if (e != cudaSuccess) return static_cast<int>(e);
  b200::launch(ctx, kernel, dim3(blocks), dim3(kBwThreads), kBwSmem<kD>, s, 1u, p);
  return B200_OK;
}

}  // namespace

bool attention_tc_fw_eligible(const b200_ctx *ctx, int mode, const AttnArgs &a) {
  return mode == B200_MODE_FP16 && ctx->encode_tiled && a.head <= 128 && a.head % 8 == 0 && a.scale > 0.f && a.max_k > 0 &&
         addressable(a.q, a.q_ld) && addressable(a.k, a.k_ld) && addressable(a.v, a.v_ld) && addressable(a.y, a.y_ld);
}

int attention_tc_fw(b200_ctx *ctx, const AttnArgs &a, cudaStream_t s) {
  FwParams p;
  std::memset(&p, 0, sizeof(p));
  p.a = a;
  p.two_heads = a.group % 2 == 0;
  p.columns = p.two_heads ? a.heads_q / 2 : a.heads_q;
  const unsigned long long tiles = attn_tiles(a.rows_q, a.max_q, a.seqs, 1, p.two_heads ? kTile : 2 * kTile, &p.a.q_each);
  if (tiles * p.columns > 0x7fffffffull) return B200_ERR_TOO_LARGE;
  p.tiles = static_cast<uint32_t>(tiles);
  p.status = ctx->d_status;
  int rc = encode(ctx, &p.q, a.q, a.head, a.heads_q, a.rows_q, a.q_ld);
  if (rc == B200_OK) rc = encode(ctx, &p.k, a.k, a.head, a.heads_k, a.rows_k, a.k_ld);
  if (rc == B200_OK) rc = encode(ctx, &p.v, a.v, a.head, a.heads_k, a.rows_k, a.v_ld);
  if (rc != B200_OK) return rc;
  return a.head <= 64 ? launch_fw<64>(ctx, p, s) : launch_fw<128>(ctx, p, s);
}

bool attention_tc_bw_eligible(const b200_ctx *ctx, int mode, const AttnArgs &a) {
  return mode == B200_MODE_FP16 && ctx->encode_tiled && a.head <= 128 && a.head % 8 == 0 && a.max_k > 0 && a.max_q > 0 && a.seqs > 0 &&
         addressable(a.q, a.q_ld) && addressable(a.k, a.k_ld) && addressable(a.v, a.v_ld) && addressable(a.gy, a.y_ld) &&
         addressable(a.gq, a.q_ld) && addressable(a.gk, a.k_ld) && addressable(a.gv, a.v_ld) && a.scale > 0.f;
}

int attention_tc_bw(b200_ctx *ctx, const AttnArgs &a, cudaStream_t s) {
  BwParams p;
  std::memset(&p, 0, sizeof(p));
  p.a = a, p.status = ctx->d_status;
  int rc = encode(ctx, &p.q, a.q, a.head, a.heads_q, a.rows_q, a.q_ld);
  if (rc == B200_OK) rc = encode(ctx, &p.k, a.k, a.head, a.heads_k, a.rows_k, a.k_ld);
  if (rc == B200_OK) rc = encode(ctx, &p.v, a.v, a.head, a.heads_k, a.rows_k, a.v_ld);
  if (rc == B200_OK) rc = encode(ctx, &p.gy, a.gy, a.head, a.heads_q, a.rows_q, a.y_ld);
  if (rc != B200_OK) return rc;
  const unsigned long long k_tiles = attn_tiles(a.rows_k, a.max_k, a.seqs, 1, kTile, &p.a.k_each), q_tiles = attn_tiles(a.rows_q, a.max_q, a.seqs, 1, kTile, &p.a.q_each);
  const unsigned long long blocks = k_tiles * a.heads_k + q_tiles * a.heads_q;
  if (blocks > 0x7fffffffull) return B200_ERR_TOO_LARGE;
  if (blocks == 0) return B200_OK;
  p.q_tiles = static_cast<uint32_t>(q_tiles), p.k_blocks = static_cast<uint32_t>(k_tiles * a.heads_k);
  return a.head <= 64 ? launch_bw<64>(ctx, p, static_cast<uint32_t>(blocks), s) : launch_bw<128>(ctx, p, static_cast<uint32_t>(blocks), s);
}

}  // namespace b200
