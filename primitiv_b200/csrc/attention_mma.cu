// Attention with mma.sync: every storage type, head size, stride and alignment.
//
// One block has 64 rows of one key head and walks the other side in tiles, everything between two products staying in
// registers: the accumulator of s = q k^T has the layout that the next product wants of its left operand.  A row is a
// query of one of the `group` heads that share a key head, so those read its keys once: row r of a sequence is query
// r / group, head r % group.
//
// forward:  the running maximum m and sum l of a softmax; y = y 2^(m - m') + p v, one pass over the keys.
// backward: p is computed again from lse.  Blocks of two kinds and one shape, with the keys at rest (gk, gv) and with
//   the queries (gq): s and dp are computed twice, which costs 7 products instead of 5 and needs neither atomics nor
//   a sum over blocks, so the same call has the same bits.
//
// With few tiles a cluster of blocks shares each, every one with a part of what passes by; their sums are joined through distributed
// shared memory, in rank order.
//
// fp32 storage: a product is three TF32 passes on x = hi + lo split in registers (one in B200_MODE_TF32).  The tensor core
// truncates as it adds into its accumulator, so no sum runs longer than one tile there: each tile's product starts from zero and
// is added in fp32 instructions.  Halves: p and ds are rounded to half for the second product, ds after a scale by a power of
// two (see attn_ds_scale), without which the ds of a long row, p / row length times a small gy, would lie below the
// smallest half.
#include <algorithm>
#include "attention_mma.cuh"
#include "tcgen05.cuh"

namespace b200 {
namespace {

constexpr uint32_t kRows = 64;       // rows at rest per block
constexpr float kPScale = 8192.f;    // backward, halves: p in [0, 1] times this

// ---- forward ---------------------------------------------------------------------------------------------

template <typename T, int kD> constexpr int kFwCols = sizeof(T) == 2 ? 64 : 32;

template <typename T, int kD, int kPass>
__global__ void __launch_bounds__(128) attention_fw_kernel(AttnArgs a, uint32_t tiles, uint32_t splits, int wide) {
  pdl_enter();
  constexpr int BN = kFwCols<T, kD>, NT = BN / 8, P = kPitch<T, kD>;
  extern __shared__ __align__(16) unsigned char s_raw[];
  __shared__ uint32_t s_at[2];
  T *sq = reinterpret_cast<T *>(s_raw), *sk = sq + kRows * P, *sv = sk + 2 * BN * P;
  __shared__ float s_m[kRows], s_l[kRows];
  const uint32_t rank = splits > 1 ? blockIdx.x % splits : 0u;
  // the last tiles of a causal sequence have the most keys: they go first
  uint32_t seq, tile;
  if (!attn_find_tile<false>(a, tiles - 1u - blockIdx.x / splits, a.group, kRows, s_at, seq, tile)) return;   // the whole cluster
  const AttnSeq q = attn_seq(a, seq);
  const uint32_t hk = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
  const uint32_t rows = q.lq * a.group, row0 = tile * kRows;
  const T *qb = static_cast<const T *>(a.q) + q.q0 * a.q_ld + static_cast<unsigned long long>(hk) * a.group * a.head;
  const T *kb = static_cast<const T *>(a.k) + q.k0 * a.k_ld + static_cast<unsigned long long>(hk) * a.head;
  const T *vb = static_cast<const T *>(a.v) + q.k0 * a.v_ld + static_cast<unsigned long long>(hk) * a.head;
  const long long shift = static_cast<long long>(q.lk) - q.lq;   // query i sees keys up to i + shift
  uint32_t keys = q.lk;
  if (a.causal) {
    const long long seen = static_cast<long long>((min(row0 + kRows, rows) - 1u) / a.group) + shift + 1;
    keys = seen <= 0 ? 0u : min(keys, static_cast<uint32_t>(seen));
  }
  const uint32_t all_steps = (keys + BN - 1) / BN, share = (all_steps + splits - 1) / splits;   // steps of one block of the cluster
  const uint32_t step0 = min(rank * share, all_steps), steps = min(step0 + share, all_steps) - step0, first_key = step0 * BN;

  load_rows<T, kD, kRows, 128>(sq, qb, a.q_ld, a.group, row0, rows, a.head, wide & kWideQ);
  if (steps) {
    load_rows<T, kD, BN, 128>(sk, kb, a.k_ld, 1, first_key, keys, a.head, wide & kWideK);
    load_rows<T, kD, BN, 128>(sv, vb, a.v_ld, 1, first_key, keys, a.head, wide & kWideV);
  }
  copies_commit();

  uint32_t row[2];
  long long last[2];       // the last key that each of this lane's two rows sees
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    row[r] = row0 + warp * 16 + g + r * 8;
    last[r] = row[r] >= rows ? -1 : (a.causal ? static_cast<long long>(row[r] / a.group) + shift : static_cast<long long>(q.lk) - 1);
  }
  float acc[kD / 8][4];
#pragma unroll
  for (int n = 0; n < kD / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  const float to2 = a.scale * kLog2e;

  for (uint32_t step = 0; step < steps; ++step) {
    const uint32_t at = step & 1u;
    copies_wait<0>();
    __syncthreads();
    if (step + 1 < steps) {
      const uint32_t next = first_key + (step + 1) * BN;
      load_rows<T, kD, BN, 128>(sk + (at ^ 1u) * BN * P, kb, a.k_ld, 1, next, keys, a.head, wide & kWideK);
      load_rows<T, kD, BN, 128>(sv + (at ^ 1u) * BN * P, vb, a.v_ld, 1, next, keys, a.head, wide & kWideV);
      copies_commit();
    }
    float s[NT][4];
    product_abt<kD, NT, kPass>(s, sq + warp * 16 * P, sk + at * BN * P);
    const uint32_t key0 = first_key + step * BN;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool seen = static_cast<long long>(key0 + n * 8 + 2 * t + (i & 1)) <= last[i >> 1];
        s[n][i] = seen ? s[n][i] * to2 : -INFINITY;
        top[i >> 1] = fmaxf(top[i >> 1], s[n][i]);
      }
    float keep[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float now = fmaxf(m[r], quad_max(top[r]));
      const float base = now == -INFINITY ? 0.f : now;   // nothing seen yet: every p below is exp2(-inf)
      keep[r] = exp2_of<T>(m[r] - base);
      m[r] = now;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_of<T>(s[n][r * 2 + e] - base);
          s[n][r * 2 + e] = p;
          sum += p;
        }
      l[r] = l[r] * keep[r] + sum;
    }
    product_py<kD, kD, NT, kPass>(acc, s, sv + at * BN * P, 0, keep[0], keep[1]);
  }
  if (splits > 1) {
    // the blocks' parts: each lays down its own, and joins the rows that fall to it, in rank order
    float *part = reinterpret_cast<float *>(sk);
    copies_wait<0>();
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t at = warp * 16 + g + r * 8;
      l[r] = quad_sum(l[r]);
      if (t == 0) s_m[at] = m[r], s_l[at] = l[r];
#pragma unroll
      for (int n = 0; n < kD / 8; ++n) *reinterpret_cast<float2 *>(part + at * kD + n * 8 + 2 * t) = make_float2(acc[n][2 * r], acc[n][2 * r + 1]);
    }
    cluster_sync_all();
    const uint32_t mine = kRows / splits, at0 = rank * mine;
    for (uint32_t i = threadIdx.x; i < mine * (kD / 4); i += 128) {
      const uint32_t at = at0 + i / (kD / 4), c = i % (kD / 4) * 4, rw = row0 + at;
      if (rw >= rows || c >= a.head) continue;
      float top = -INFINITY, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
      for (uint32_t s = 0; s < splits; ++s) top = fmaxf(top, ld_cluster(map_to_cta(smem_at(s_m + at), s)));
      for (uint32_t s = 0; s < splits; ++s) {
        const float ms = ld_cluster(map_to_cta(smem_at(s_m + at), s)), w = ms == -INFINITY ? 0.f : exp2_of<T>(ms - top);
        const float4 o = ld_cluster4(map_to_cta(smem_at(part + at * kD + c), s));
        sum += w * ld_cluster(map_to_cta(smem_at(s_l + at), s));
        v[0] += w * o.x, v[1] += w * o.y, v[2] += w * o.z, v[3] += w * o.w;
      }
      const uint32_t tok = rw / a.group, h = hk * a.group + rw - tok * a.group;
      const bool sees = a.causal ? static_cast<long long>(tok) + shift >= 0 : q.lk > 0u;
      T *out = static_cast<T *>(a.y) + (q.q0 + tok) * a.y_ld + static_cast<unsigned long long>(h) * a.head + c;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < a.head) out[e] = round_to<T>(sees ? v[e] / sum : 0.f);
      if (a.lse && c == 0) a.lse[static_cast<unsigned long long>(h) * a.rows_q + q.q0 + tok] = sees ? (top == -INFINITY ? 0.f : top * kLn2) + logf(sum) : -INFINITY;
    }
    cluster_sync_all();   // nobody leaves while another reads its part
    return;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] = quad_sum(l[r]);
    if (row[r] >= rows) continue;
    const uint32_t tok = row[r] / a.group, h = hk * a.group + row[r] - tok * a.group;
    // a row that sees no key has zeros, one that sees scores of -infinity alone 0 / 0; a maximum of -infinity also leaves out NaNs
    const bool sees = last[r] >= 0;
    store_row<T, kD>(static_cast<T *>(a.y) + (q.q0 + tok) * a.y_ld + static_cast<unsigned long long>(h) * a.head, acc, r, 0, a.head,
                     1.f / l[r], 0, sees);
    if (a.lse && t == 0)
      a.lse[static_cast<unsigned long long>(h) * a.rows_q + q.q0 + tok] = sees ? (m[r] == -INFINITY ? 0.f : m[r] * kLn2) + logf(l[r]) : -INFINITY;
  }
}

// ---- backward ----------------------------------------------------------------------------------------------

template <typename T, int kD> constexpr int kBwCols = sizeof(T) == 2 && kD == 64 ? 64 : 32;
template <typename T, int kD> constexpr int kBwThreads = kD == 256 ? 256 : 128;   // 256 columns: a warp has half of them
// fp32: one stage, so that more blocks share an SM.  A training step of 8 x 509 tokens, 8 heads of 64: 467 us; two stages, or four blocks to an
// SM (128 registers, some in memory), are 4 to 8 % slower.
template <typename T, int kD> constexpr int kBwStages = sizeof(T) == 4 ? 1 : 2;
template <typename T, int kD> constexpr int kBwBlocks = sizeof(T) == 4 && kD == 64 ? 3 : 1;

// kKeys: the keys rest, the queries of all heads of the group pass by (gk, gv).  Else the queries rest (gq).
template <typename T, int kD, int kPass, bool kKeys>
__device__ __forceinline__ void attention_bw_side(const AttnArgs &a, uint32_t nth, uint32_t tiles, uint32_t splits, int wide) {
  constexpr int BN = kBwCols<T, kD>, NT = BN / 8, P = kPitch<T, kD>, kThreads = kBwThreads<T, kD>, kStages = kBwStages<T, kD>;
  constexpr int kCols = kD == 256 ? 128 : kD;
  constexpr bool kHalf = sizeof(T) == 2;
  // p = exp(s - lse).  fp32: the difference first, then its multiple of log2(e): lse log2(e), rounded, would cost p half of 2^-20
  constexpr float kLseUnit = kHalf ? kLog2e : 1.f;
  extern __shared__ __align__(16) unsigned char s_raw[];
  __shared__ uint32_t s_at[2];
  __shared__ float s_lse[2][BN], s_delta[2][BN], s_max[3][8], s_undo[kRows];
  __shared__ int s_last[2][BN];   // the last key that a query sees
  T *x1 = reinterpret_cast<T *>(s_raw), *x2 = x1 + kRows * P, *y1 = x2 + kRows * P, *y2 = y1 + kStages * BN * P;
  uint32_t seq, tile;
  if (!attn_find_tile<kKeys>(a, kKeys ? nth : tiles - 1u - nth, kKeys ? 1u : a.group, kRows, s_at, seq, tile)) return;   // the whole cluster
  const uint32_t rank = splits > 1 ? blockIdx.x % splits : 0u;
  const AttnSeq q = attn_seq(a, seq);
  const uint32_t hk = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
  const uint32_t wrow = (warp & 3u) * 16u, col0 = (warp >> 2) * kCols;
  const uint32_t qrows = q.lq * a.group, row0 = tile * kRows, rows = kKeys ? q.lk : qrows;
  const unsigned long long hq_at = static_cast<unsigned long long>(hk) * a.group * a.head, hk_at = static_cast<unsigned long long>(hk) * a.head;
  const T *qb = static_cast<const T *>(a.q) + q.q0 * a.q_ld + hq_at, *gyb = static_cast<const T *>(a.gy) + q.q0 * a.y_ld + hq_at;
  const T *kb = static_cast<const T *>(a.k) + q.k0 * a.k_ld + hk_at, *vb = static_cast<const T *>(a.v) + q.k0 * a.v_ld + hk_at;
  const long long shift = static_cast<long long>(q.lk) - q.lq;
  // what passes by: queries from the first that sees a key of the tile, or keys up to the last that a query of the tile sees
  uint32_t from = 0, to = kKeys ? qrows : q.lk;
  if (a.causal) {
    if (kKeys) {
      const long long first = static_cast<long long>(row0) - shift;
      from = first <= 0 ? 0u : (first >= q.lq ? qrows : static_cast<uint32_t>(first) * a.group);
    } else {
      const long long seen = static_cast<long long>((min(row0 + kRows, rows) - 1u) / a.group) + shift + 1;
      to = seen <= 0 ? 0u : min(to, static_cast<uint32_t>(seen));
    }
  }
  const uint32_t all_steps = to > from ? (to - from + BN - 1) / BN : 0u, share = (all_steps + splits - 1) / splits;   // steps of one block of the cluster
  const uint32_t step0 = min(rank * share, all_steps), steps = min(step0 + share, all_steps) - step0;
  const unsigned long long stat = static_cast<unsigned long long>(hk) * a.group * a.rows_q + q.q0;   // of query 0, first head

  auto last_key = [&](uint32_t tok) {
    const long long see = a.causal ? min(static_cast<long long>(tok) + shift, static_cast<long long>(q.lk) - 1) : static_cast<long long>(q.lk) - 1;
    return static_cast<int>(max(see, -1ll));
  };
  auto load_step = [&](uint32_t step, uint32_t at) {
    const uint32_t r0 = from + (step0 + step) * BN;
    if constexpr (kKeys) {
      load_rows<T, kD, BN, kThreads>(y1 + at * BN * P, qb, a.q_ld, a.group, r0, to, a.head, wide & kWideQ);
      load_rows<T, kD, BN, kThreads>(y2 + at * BN * P, gyb, a.y_ld, a.group, r0, to, a.head, wide & kWideGy);
      if (threadIdx.x < BN) {
        const uint32_t r = r0 + threadIdx.x, tok = r / a.group;
        const unsigned long long i = stat + static_cast<unsigned long long>(r - tok * a.group) * a.rows_q + tok;
        s_lse[at][threadIdx.x] = r < to ? a.lse[i] * kLseUnit : 0.f;
        s_last[at][threadIdx.x] = r < to ? last_key(tok) : -1;
        s_delta[at][threadIdx.x] = r < to ? a.delta[i] : 0.f;
      }
    } else {
      load_rows<T, kD, BN, kThreads>(y1 + at * BN * P, kb, a.k_ld, 1, r0, to, a.head, wide & kWideK);
      load_rows<T, kD, BN, kThreads>(y2 + at * BN * P, vb, a.v_ld, 1, r0, to, a.head, wide & kWideV);
    }
    copies_commit();
  };
  if constexpr (kKeys) {
    load_rows<T, kD, kRows, kThreads>(x1, kb, a.k_ld, 1, row0, rows, a.head, wide & kWideK);
    load_rows<T, kD, kRows, kThreads>(x2, vb, a.v_ld, 1, row0, rows, a.head, wide & kWideV);
  } else {
    load_rows<T, kD, kRows, kThreads>(x1, qb, a.q_ld, a.group, row0, rows, a.head, wide & kWideQ);
    load_rows<T, kD, kRows, kThreads>(x2, gyb, a.y_ld, a.group, row0, rows, a.head, wide & kWideGy);
  }
  if (steps) load_step(0, 0);
  else copies_commit();

  // Scale of ds: with the keys at rest one for all that this block sees, since it must not change on the way; with the queries at rest one per
  // query, so that none loses bits to another with a larger gradient.
  float ds_scale[2] = {1.f, 1.f};
  float vm = 0.f;
  if constexpr (kHalf) {
    const uint32_t k_from = kKeys ? row0 : 0u, k_to = kKeys ? min(row0 + kRows, rows) : to;
    float gm = 0.f, dm = 0.f;
    if constexpr (kKeys) {
      for (uint32_t r = from + threadIdx.x; r < qrows; r += kThreads) {
        const uint32_t tok = r / a.group;
        const unsigned long long i = stat + static_cast<unsigned long long>(r - tok * a.group) * a.rows_q + tok;
        gm = attn_finite_max(gm, a.gy_norm[i]);
        dm = attn_finite_max(dm, fabsf(a.delta[i]));
      }
    }
    for (uint32_t r = k_from + threadIdx.x; r < k_to; r += kThreads)
      vm = attn_finite_max(vm, a.v_norm[static_cast<unsigned long long>(hk) * a.rows_k + q.k0 + r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
      dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, o));
      vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
    }
    if (lane == 0) s_max[0][warp] = gm, s_max[1][warp] = dm, s_max[2][warp] = vm;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 32; ++w) gm = fmaxf(gm, s_max[0][w]), dm = fmaxf(dm, s_max[1][w]), vm = fmaxf(vm, s_max[2][w]);
    if constexpr (kKeys) ds_scale[0] = ds_scale[1] = attn_ds_scale(gm, vm, dm);
  }

  uint32_t row[2];
  int row_last[2];   // queries at rest: the last key that the row sees; keys at rest: the row's key
  float row_lse[2] = {0.f, 0.f}, row_delta[2] = {0.f, 0.f};
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    row[r] = row0 + wrow + g + r * 8;
    const uint32_t tok = row[r] / a.group;
    row_last[r] = kKeys ? static_cast<int>(row[r]) : (row[r] < rows ? last_key(tok) : -1);
    if (!kKeys && row[r] < rows) {
      const unsigned long long at = stat + static_cast<unsigned long long>(row[r] - tok * a.group) * a.rows_q + tok;
      row_lse[r] = a.lse[at] * kLseUnit;
      row_delta[r] = a.delta[at];
      if constexpr (kHalf) ds_scale[r] = attn_ds_scale(a.gy_norm[at], vm, fabsf(row_delta[r]));
    }
  }
  float acc1[kKeys ? kCols / 8 : 1][4], acc2[kCols / 8][4];
#pragma unroll
  for (int n = 0; n < kCols / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc2[n][i] = 0.f;
      if constexpr (kKeys) acc1[n][i] = 0.f;
    }
  const float to2 = a.scale * kLog2e;

  for (uint32_t step = 0; step < steps; ++step) {
    const uint32_t at = kStages == 2 ? step & 1u : 0u;
    if (kStages == 1 && step > 0) {
      __syncthreads();
      load_step(step, 0);
    }
    copies_wait<0>();
    __syncthreads();
    if (kStages == 2 && step + 1 < steps) load_step(step + 1, at ^ 1u);
    float p[NT][4], ds[NT][4];
    product_abt<kD, NT, kPass>(p, x1 + wrow * P, y1 + at * BN * P);
    product_abt<kD, NT, kPass>(ds, x2 + wrow * P, y2 + at * BN * P);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = n * 8 + 2 * t + e, key = static_cast<int>(from + (step0 + step) * BN) + c;
        const int col_last = kKeys ? s_last[at][c] : 0;
        const float col_lse = kKeys ? s_lse[at][c] : 0.f, col_delta = kKeys ? s_delta[at][c] : 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int i = 2 * r + e;
          const bool seen = kKeys ? row_last[r] <= col_last : key <= row_last[r];
          const float lse = kKeys ? col_lse : row_lse[r];
          const float x = !seen ? 0.f : kHalf ? exp2_of<T>(fmaf(p[n][i], to2, -lse)) : exp2_of<T>(fmaf(p[n][i], a.scale, -lse) * kLog2e);
          ds[n][i] = seen ? x * (ds[n][i] - (kKeys ? col_delta : row_delta[r])) * ds_scale[r] : 0.f;
          p[n][i] = kHalf ? x * kPScale : x;
        }
      }
    if constexpr (kKeys) product_py<kD, kCols, NT, kPass>(acc1, p, y2 + at * BN * P, col0, 1.f, 1.f);
    product_py<kD, kCols, NT, kPass>(acc2, ds, y1 + at * BN * P, col0, 1.f, 1.f);
  }
  const float undo[2] = {a.scale / ds_scale[0], a.scale / ds_scale[1]};
  if (splits > 1) {
    // the blocks' sums: each lays down its own, and adds the rows that fall to it, in rank order
    float *part = reinterpret_cast<float *>(s_raw);
    copies_wait<0>();
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (t == 0) s_undo[wrow + g + r * 8] = undo[r];
#pragma unroll
      for (int n = 0; n < kCols / 8; ++n) {
        float *at = part + (wrow + g + r * 8) * kD + col0 + n * 8 + 2 * t;
        *reinterpret_cast<float2 *>(at) = make_float2(acc2[n][2 * r], acc2[n][2 * r + 1]);
        if constexpr (kKeys) *reinterpret_cast<float2 *>(at + kRows * kD) = make_float2(acc1[n][2 * r], acc1[n][2 * r + 1]);
      }
    }
    cluster_sync_all();
    const uint32_t mine = kRows / splits, at0 = rank * mine;
    for (uint32_t i = threadIdx.x; i < (kKeys ? 2u : 1u) * mine * (kD / 4); i += kThreads) {
      const uint32_t which = i / (mine * (kD / 4)), in = i - which * mine * (kD / 4);   // gk or gq, then gv
      const uint32_t at = at0 + in / (kD / 4), c = in % (kD / 4) * 4, rw = row0 + at;
      if (rw >= rows || c >= a.head) continue;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      for (uint32_t s = 0; s < splits; ++s) {
        const float4 o = ld_cluster4(map_to_cta(smem_at(part + (which * kRows + at) * kD + c), s));
        v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
      }
      const float factor = which ? (kHalf ? 1.f / kPScale : 1.f) : s_undo[at];
      T *out;
      bool some = true;
      if constexpr (kKeys) {
        out = which ? static_cast<T *>(a.gv) + (q.k0 + rw) * a.v_ld + hk_at : static_cast<T *>(a.gk) + (q.k0 + rw) * a.k_ld + hk_at;
      } else {
        const uint32_t tok = rw / a.group;
        some = last_key(tok) >= 0;
        out = static_cast<T *>(a.gq) + (q.q0 + tok) * a.q_ld + hq_at + static_cast<unsigned long long>(rw - tok * a.group) * a.head;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < a.head) out[c + e] = round_to<T>((some ? v[e] * factor : 0.f) + (a.accumulate ? static_cast<float>(out[c + e]) : 0.f));
    }
    cluster_sync_all();   // nobody leaves while another reads its part
    return;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (row[r] >= rows) continue;
    if constexpr (kKeys) {
      store_row<T, kCols>(static_cast<T *>(a.gv) + (q.k0 + row[r]) * a.v_ld + hk_at, acc1, r, col0, a.head, kHalf ? 1.f / kPScale : 1.f, a.accumulate);
      store_row<T, kCols>(static_cast<T *>(a.gk) + (q.k0 + row[r]) * a.k_ld + hk_at, acc2, r, col0, a.head, undo[r], a.accumulate);
    } else {
      const uint32_t tok = row[r] / a.group;
      store_row<T, kCols>(static_cast<T *>(a.gq) + (q.q0 + tok) * a.q_ld + hq_at + static_cast<unsigned long long>(row[r] - tok * a.group) * a.head,
                          acc2, r, col0, a.head, undo[r], a.accumulate, row_last[r] >= 0);
    }
  }
}

// Both sides in one launch: either alone leaves SMs idle behind its last blocks.
template <typename T, int kD, int kPass>
__global__ void __launch_bounds__(kBwThreads<T, kD>, kBwBlocks<T, kD>) attention_bw_kernel(AttnArgs a, uint32_t k_tiles, uint32_t q_tiles, uint32_t splits, int wide) {
  pdl_enter();
  const uint32_t item = blockIdx.x / splits;
  if (item < k_tiles) attention_bw_side<T, kD, kPass, true>(a, item, k_tiles, splits, wide);
  else attention_bw_side<T, kD, kPass, false>(a, item - k_tiles, q_tiles, splits, wide);
}

// ---- launches ----------------------------------------------------------------------------------------------

// Blocks of a cluster that share a tile: as many as bring four on every SM, while each has two steps of the longest.
uint32_t split_of(const b200_ctx *ctx, unsigned long long blocks, unsigned long long steps) {
  uint32_t splits = 1;
  while (splits < 8 && blocks * splits < 4ull * ctx->sm_count && steps / (2 * splits) >= 2) splits *= 2;
  return splits;
}

template <typename T, int kD, int kPass>
int launch_fw(b200_ctx *ctx, AttnArgs a, cudaStream_t s) {
  constexpr size_t smem = sizeof(T) * kPitch<T, kD> * (kRows + 4 * kFwCols<T, kD>);
  const unsigned long long bound = attn_tiles(a.rows_q, a.max_q, a.seqs, a.group, kRows, &a.q_each);
  if (bound >= 1ull << 31) return B200_ERR_TOO_LARGE;
  const uint32_t tiles = static_cast<uint32_t>(bound);
  auto kernel = attention_fw_kernel<T, kD, kPass>;
  if (const int rc = allow_smem(kernel, smem)) return rc;
  const uint32_t splits = split_of(ctx, static_cast<unsigned long long>(tiles) * a.heads_k, a.max_k / kFwCols<T, kD>);
  if (static_cast<unsigned long long>(tiles) * splits > 0x7fffffffull) return B200_ERR_TOO_LARGE;
  b200::launch(ctx, kernel, dim3(tiles * splits, a.heads_k), dim3(128), smem, s, splits, a, tiles, splits, find_wide(a, sizeof(T)));
  return B200_OK;
}

template <typename T, int kD, int kPass>
int launch_bw(b200_ctx *ctx, AttnArgs a, cudaStream_t s) {
  constexpr size_t smem = sizeof(T) * kPitch<T, kD> * (2 * kRows + 2 * kBwStages<T, kD> * kBwCols<T, kD>);
  const unsigned long long k_bound = attn_tiles(a.rows_k, a.max_k, a.seqs, 1, kRows, &a.k_each);
  const unsigned long long q_bound = attn_tiles(a.rows_q, a.max_q, a.seqs, a.group, kRows, &a.q_each);
  if (k_bound + q_bound >= 1ull << 31) return B200_ERR_TOO_LARGE;
  const uint32_t k_tiles = static_cast<uint32_t>(k_bound), q_tiles = static_cast<uint32_t>(q_bound);
  if (k_tiles + q_tiles == 0) return B200_OK;
  auto kernel = attention_bw_kernel<T, kD, kPass>;
  if (const int rc = allow_smem(kernel, smem)) return rc;
  const uint32_t splits = split_of(ctx, static_cast<unsigned long long>(k_tiles + q_tiles) * a.heads_k,
                                   std::max<unsigned long long>(a.max_k, static_cast<unsigned long long>(a.max_q) * a.group) / kBwCols<T, kD>);
  b200::launch(ctx, kernel, dim3((k_tiles + q_tiles) * splits, a.heads_k), dim3(kBwThreads<T, kD>), smem, s, splits, a, k_tiles, q_tiles, splits,
               find_wide(a, sizeof(T)));
  return B200_OK;
}

}  // namespace

int attention_mma_fw(b200_ctx *ctx, int mode, const AttnArgs &a, cudaStream_t s) {
  return with_type(mode, [&](auto type, auto pass) {
    using T = decltype(type);
    return with_head<T, decltype(pass)::value>(a.head, [&](auto d) { return launch_fw<T, decltype(d)::value, decltype(pass)::value>(ctx, a, s); });
  });
}

int attention_mma_bw(b200_ctx *ctx, int mode, const AttnArgs &a, cudaStream_t s) {
  return with_type(mode, [&](auto type, auto pass) {
    using T = decltype(type);
    return with_head<T, decltype(pass)::value>(a.head, [&](auto d) {
      return launch_bw<T, decltype(d)::value, decltype(pass)::value>(ctx, a, s);
    });
  });
}

}  // namespace b200
