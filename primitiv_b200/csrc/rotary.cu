// Rotary positions, and norms of queries and keys with the rotation in the same pass.
//
//   rotary        (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t),  t = position * freqs[pair]
//   norm_rotary   n = x r, r = 1 / sqrt(mean(x^2) + eps);  y = turned (n gain)
//   backward      g = gy turned back (t -> -t);  ggain += sum g n;  gx += r (g gain - n mean(g gain n))
//
// Bound by memory, one read and one write of every element (three with a backward norm), if the instructions beside
// it are few.  A group of lanes (a power of two) holds one head of one token in registers, so the norm's sums are a few shuffles and
// nothing is read twice.  A lane's unit is the two vectors that turn with one another: in the HALVES layout they lie rot/2
// apart, in the PAIRS layout side by side.
//
// The cosines depend on the token alone.  A block takes a tile of tokens and forms their angles once, in shared memory: with each head
// forming its own, 40 heads of 128 would cost 2.6 million 64-bit products and sines per 1024 tokens instead of 65 thousand.  A
// group stays with one token and goes over its heads, with the token's cosines and the gain in registers; arithmetic is on pairs of floats.
// (A group that took any row, and read cosines and gain for it, spent two to three times the instructions: 71 us forward, 91 us with norms,
// 266 us for their gradient, where this takes 61, 82 and 117; 16384 tokens of 40 heads of 128 halves.)
// An angle is formed in turns, with what its products round off, and reduced in 64 bits, so the last position, 2^32 - 1, has the same
// error (2^-26 of a turn) as position 1; its sine and cosine are 32-bit.
//
// With norms a block takes the heads of one gain only.  Gradients of gains are sums over every token and head: a thread keeps its
// elements' sums in registers over all that its block takes, a block writes one partial row and a second kernel adds the
// rows in order: no atomics, the same bits every run.
#include <algorithm>
#include <cmath>

#include "../../include/primitiv_b200_attention.h"
#include "f32x2.cuh"
#include "ops_common.cuh"

namespace b200 {
namespace {

constexpr unsigned kThreads = 256;
constexpr unsigned kWarps = kThreads / 32;
constexpr uint32_t kMaxHead = 256;
constexpr uint32_t kHeadsEach = 8;
constexpr uint32_t kSumBlocks = 3;         // blocks per SM that keep sums
constexpr uint32_t kMaxPartials = B200_NORM_ROTARY_SCRATCH / kMaxHead;

struct RotaryArgs {
  const void *x, *g;        // forward: x; backward: g = gy, and x where there is a norm
  void *y;                  // y or gx
  const void *gain_q, *gain_k;
  float *partial;           // [block][head], or null
  const double *freqs;
  const uint32_t *positions;
  u64 x_ld, g_ld, y_ld;
  uint32_t head, heads, heads_q, tokens, rot;
  uint32_t units, lanes_log2;         // units of a head; lanes of a group
  // Blocks 0 .. blocks_q - 1 take the first heads_q heads, the others the rest.  Of a block's groups 2^split_log2 share a token.
  uint32_t blocks_q, split_q_log2, split_k_log2;
  float amplitude, eps;
  int accumulate;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// The two vectors of unit u: their first elements.  At or past `head`: there is none.
template <int V, int kLayout>
__device__ __forceinline__ void unit_at(uint32_t u, uint32_t rot, uint32_t &c0, uint32_t &c1) {
  if constexpr (kLayout == B200_ROTARY_HALVES) {
    const uint32_t turned = rot / (2 * V);
    if (u < turned) {
      c0 = u * V;
      c1 = c0 + rot / 2;
      return;
    }
    c0 = rot + 2 * (u - turned) * V;
  } else {
    c0 = 2 * u * V;
  }
  c1 = c0 + V;
}

// V floats, as pairs where there are two.
template <int V>
struct Lane {
  f32x2 p[V > 1 ? V / 2 : 1];
  __device__ __forceinline__ void put(int j, float v) {
    float a, b;
    unpair(p[j / 2], a, b);
    p[j / 2] = (j & 1) ? pair_of(a, v) : pair_of(v, b);
  }
  __device__ __forceinline__ float get(int j) const {
    float a, b;
    unpair(p[j / 2], a, b);
    return (j & 1) ? b : a;
  }
};
template <int V> __device__ __forceinline__ Lane<V> operator*(const Lane<V> &x, const Lane<V> &y) {
  Lane<V> z;
#pragma unroll
  for (int i = 0; i < (V > 1 ? V / 2 : 1); ++i) z.p[i] = mul2(x.p[i], y.p[i]);
  return z;
}
template <int V> __device__ __forceinline__ Lane<V> fma(const Lane<V> &x, const Lane<V> &y, const Lane<V> &c) {
  Lane<V> z;
#pragma unroll
  for (int i = 0; i < (V > 1 ? V / 2 : 1); ++i) z.p[i] = fma2(x.p[i], y.p[i], c.p[i]);
  return z;
}
template <int V> __device__ __forceinline__ Lane<V> all_of(float v) {
  Lane<V> z;
#pragma unroll
  for (int i = 0; i < (V > 1 ? V / 2 : 1); ++i) z.p[i] = pair_of(v, V > 1 ? v : 0.f);
  return z;
}
template <int V> __device__ __forceinline__ float sum_of(const Lane<V> &x) {
  f32x2 s[V > 1 ? V / 2 : 1];
#pragma unroll
  for (int i = 0; i < (V > 1 ? V / 2 : 1); ++i) s[i] = x.p[i];
#pragma unroll
  for (int n = V / 4; n > 0; n /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) s[i] = add2(s[i], s[i + n]);
  float a, b;
  unpair(s[0], a, b);
  return V > 1 ? a + b : a;
}

// A unit's pairs: a[j] turns with b[j].
template <int V>
struct Unit {
  Lane<V> a, b;
};

// A unit as it lies in memory.
template <typename T, int V>
struct Raw {
  Pack<T, V> first, second;
};

template <typename T, int V>
__device__ __forceinline__ void load_raw(Raw<T, V> &raw, const T *p, uint32_t c0, uint32_t c1, uint32_t head) {
  if (c0 < head) raw.first = *reinterpret_cast<const Pack<T, V> *>(p + c0);
  if (c1 < head) raw.second = *reinterpret_cast<const Pack<T, V> *>(p + c1);
}
// What there is none of counts as zero.
template <typename T, int V, int kLayout>
__device__ __forceinline__ Unit<V> unit_of(const Raw<T, V> &raw, bool has0, bool has1) {
  Unit<V> u;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    // element e of the two vectors' 2 V
    const int ea = kLayout == B200_ROTARY_HALVES ? j : 2 * j, eb = kLayout == B200_ROTARY_HALVES ? j + V : 2 * j + 1;
    const float x = ea < V ? (has0 ? to_float(raw.first.v[ea < V ? ea : 0]) : 0.f) : (has1 ? to_float(raw.second.v[ea < V ? 0 : ea - V]) : 0.f);
    const float y = eb < V ? (has0 ? to_float(raw.first.v[eb < V ? eb : 0]) : 0.f) : (has1 ? to_float(raw.second.v[eb < V ? 0 : eb - V]) : 0.f);
    u.a.put(j, x), u.b.put(j, y);
  }
  return u;
}
template <typename T, int V, int kLayout>
__device__ __forceinline__ void store_unit(const Unit<V> &u, T *p, uint32_t c0, uint32_t c1, uint32_t head) {
  Pack<T, V> first, second;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (kLayout == B200_ROTARY_HALVES) {
      first.v[e] = from_float<T>(u.a.get(e)), second.v[e] = from_float<T>(u.b.get(e));
    } else {
      first.v[e] = from_float<T>((e & 1) ? u.b.get(e / 2) : u.a.get(e / 2));
      second.v[e] = from_float<T>(((e + V) & 1) ? u.b.get((e + V) / 2) : u.a.get((e + V) / 2));
    }
  }
  if (c0 < head) *reinterpret_cast<Pack<T, V> *>(p + c0) = first;
  if (c1 < head) *reinterpret_cast<Pack<T, V> *>(p + c1) = second;
}

// The group's sums of both, side by side.
template <int kLog2>
__device__ __forceinline__ void sums_over(float &v, float &w) {
#pragma unroll
  for (int o = 1; o < 1 << kLog2; o <<= 1) {
    const float x = __shfl_xor_sync(0xffffffffu, v, o), y = __shfl_xor_sync(0xffffffffu, w, o);
    v += x, w += y;
  }
}
__device__ __forceinline__ void group_sums(float &v, float &w, uint32_t lanes_log2) {
  switch (lanes_log2) {
    case 0: break;
    case 1: sums_over<1>(v, w); break;
    case 2: sums_over<2>(v, w); break;
    case 3: sums_over<3>(v, w); break;
    case 4: sums_over<4>(v, w); break;
    default: sums_over<5>(v, w); break;
  }
}

// kUnits: units per lane (heads are at most 256 elements, so single elements need four, pairs two).
template <int V> constexpr int kUnitsOf = V >= 4 ? 1 : (V == 2 ? 2 : 4);

template <typename T, int V, int kLayout, bool kNorm, bool kBack>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a) {
  pdl_enter();
  constexpr int kUnits = kUnitsOf<V>;
  constexpr bool kSums = kNorm && kBack;
  // Where sums are kept, registers leave room for three blocks on an SM, whose loads alone do not fill the memory's latency: the next row
  // is fetched into shared memory, where every thread has slots of its own.  (Into registers: two blocks, 199 us instead of 117.)
  constexpr bool kStaged = kSums && kUnits == 1 && V * sizeof(T) >= 8;
  constexpr uint32_t kStages = 2;   // (three or four: the same time)
  extern __shared__ float2 s_tab[];                                  // [token][V][pitch]
  __shared__ __align__(16) float s_sums[kSums ? kWarps * kMaxHead : (kNorm ? kMaxHead : 1)];   // the gain, and in the end the warps' sums
  __shared__ __align__(16) Pack<T, V> s_slots[kStaged ? kStages * 4 : 1][kThreads];

  const bool second = blockIdx.x >= a.blocks_q;
  const uint32_t block = second ? blockIdx.x - a.blocks_q : blockIdx.x, blocks = second ? gridDim.x - a.blocks_q : a.blocks_q;
  const uint32_t head0 = second ? a.heads_q : 0u, heads = second ? a.heads - a.heads_q : a.heads_q;
  const uint32_t split_log2 = second ? a.split_k_log2 : a.split_q_log2, split = 1u << split_log2;
  const uint32_t lanes = 1u << a.lanes_log2, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> a.lanes_log2;
  const uint32_t tile_tokens = (kThreads >> a.lanes_log2) >> split_log2, tiles = (a.tokens + tile_tokens - 1) / tile_tokens;
  const uint32_t my_tok = group >> split_log2, my_head = group & (split - 1), turns_of_heads = (heads + split - 1) >> split_log2;
  const uint32_t pairs = a.rot / 2, pitch = (pairs + V - 1) / V, tab_size = V * pitch;

  uint32_t c0[kUnits], c1[kUnits];
  bool turned[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    unit_at<V, kLayout>(lane + k * lanes, a.rot, c0[k], c1[k]);
    turned[k] = 2 * (lane + k * lanes) * V < a.rot;
  }
  Unit<V> gain[kNorm ? kUnits : 1], sums[kSums ? kUnits : 1];
  if constexpr (kNorm) {
    // Element by element, so that gains may begin anywhere in a buffer of parameters; every thread takes its own from here.
    static_assert(kMaxHead <= kThreads, "one element a thread");
    if (threadIdx.x < a.head) s_sums[threadIdx.x] = to_float(static_cast<const T *>(second ? a.gain_k : a.gain_q)[threadIdx.x]);
  }
  if constexpr (kSums) {
#pragma unroll
    for (int k = 0; k < kUnits; ++k) sums[k].a = sums[k].b = all_of<V>(0.f);
  }
  const float per_head = 1.f / static_cast<float>(a.head);

  for (uint32_t tile = block; tile < tiles; tile += blocks) {
    const uint32_t t0 = tile * tile_tokens, nt = min(tile_tokens, a.tokens - t0);
    if (tile != block) __syncthreads();   // the table's last readers are done
    for (uint32_t i = threadIdx.x; i < nt * pairs; i += kThreads) {
      const uint32_t t = i / pairs, p = i - t * pairs;
      const double pos = a.positions ? static_cast<double>(a.positions[t0 + t]) : static_cast<double>(t0 + t);
      constexpr double kTurn = 0.15915494309189533577, kTurnRest = -9.839338337591243477e-18;   // 1 / (2 pi) in two doubles
      const double freq = a.freqs[p], step = freq * kTurn, turns = pos * step;
      double part = turns - rint(turns);
      // far out a product's half bit is up to 2^-24 of a turn: what the two have rounded off (before 2^20 turns it is less than 2^-31)
      if (fabs(turns) > 1048576.0) part += ::fma(pos, step, -turns) + pos * (::fma(freq, kTurn, -step) + freq * kTurnRest);
      float sn, cs;
      sincospif(2.f * static_cast<float>(part), &sn, &cs);
      s_tab[t * tab_size + (p % V) * pitch + p / V] = make_float2(a.amplitude * cs, a.amplitude * (kBack ? -sn : sn));
    }
    if constexpr (kStaged) asm volatile("cp.async.wait_group 0;" ::: "memory");
    const bool live = my_tok < nt;
    const u64 t = t0 + my_tok, at = static_cast<u64>(head0 + my_head) * a.head, step = static_cast<u64>(a.head) << split_log2;
    const T *x = static_cast<const T *>(kBack && !kNorm ? a.g : a.x) + t * (kBack && !kNorm ? a.g_ld : a.x_ld) + at;
    const T *g = static_cast<const T *>(a.g) + t * a.g_ld + at;
    T *out = static_cast<T *>(a.y) + t * a.y_ld + at;
    Raw<T, V> raw[kUnits], raw_g[kSums ? kUnits : 1];
    auto fetch = [&](uint32_t i) {
      const uint32_t head = live && my_head + (i << split_log2) < heads ? a.head : 0u;
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        load_raw(raw[k], x, c0[k], c1[k], head);
        if constexpr (kSums) load_raw(raw_g[k], g, c0[k], c1[k], head);
      }
      x += step;
      if constexpr (kSums) g += step;
    };
    // the same into a stage's slots
    auto stage = [&](uint32_t i) {
      if constexpr (kStaged) {
        if (live && i < turns_of_heads && my_head + (i << split_log2) < heads) {
          auto copy = [&](uint32_t slot, const T *from) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(&s_slots[(i % kStages) * 4 + slot][threadIdx.x]))),
                         "l"(from), "n"(static_cast<int>(V * sizeof(T))) : "memory");
          };
          if (c0[0] < a.head) copy(0, x + c0[0]), copy(2, g + c0[0]);
          if (c1[0] < a.head) copy(1, x + c1[0]), copy(3, g + c1[0]);
        }
        x += step, g += step;
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
    };
    if constexpr (kStaged) {
#pragma unroll
      for (uint32_t i = 0; i + 1 < kStages; ++i) stage(i);
    } else {
      fetch(0);
    }
    __syncthreads();
    if constexpr (kNorm) {
      if (tile == block) {
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
          Raw<float, V> raw;
          load_raw(raw, s_sums, c0[k], c1[k], a.head);
          gain[k] = unit_of<float, V, kLayout>(raw, c0[k] < a.head, c1[k] < a.head);
        }
      }
    }
    Unit<V> cs[kUnits];   // a: cosine, b: sine
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      cs[k].a = all_of<V>(1.f), cs[k].b = all_of<V>(0.f);
      if (live && turned[k]) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float2 v = s_tab[my_tok * tab_size + j * pitch + lane + k * lanes];
          cs[k].a.put(j, v.x), cs[k].b.put(j, v.y);
        }
      }
    }
    auto turn = [&](Unit<V> &u, int k) {
      if (!turned[k]) return;
      const Lane<V> minus = all_of<V>(-1.f) * cs[k].b, a1 = fma(u.b, minus, u.a * cs[k].a);
      u.b = fma(u.a, cs[k].b, u.b * cs[k].a);
      u.a = a1;
    };
    for (uint32_t i = 0; i < turns_of_heads; ++i) {
      if constexpr (kStaged) {
        stage(i + kStages - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        const Pack<T, V> (*slots)[kThreads] = s_slots + (i % kStages) * 4;
        raw[0].first = slots[0][threadIdx.x], raw[0].second = slots[1][threadIdx.x];
        raw_g[0].first = slots[2][threadIdx.x], raw_g[0].second = slots[3][threadIdx.x];
      } else if (i > 0) {
        fetch(i);
      }
      const bool here = live && my_head + (i << split_log2) < heads;
      Unit<V> w[kUnits], gw[kSums ? kUnits : 1];
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        w[k] = unit_of<T, V, kLayout>(raw[k], here && c0[k] < a.head, here && c1[k] < a.head);
        if constexpr (kSums) gw[k] = unit_of<T, V, kLayout>(raw_g[k], here && c0[k] < a.head, here && c1[k] < a.head);
      }
      float ss = 0.f, dot = 0.f;
      if constexpr (kNorm) {
        Lane<V> sq = all_of<V>(0.f), dots = all_of<V>(0.f);
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
          sq = fma(w[k].b, w[k].b, fma(w[k].a, w[k].a, sq));
          if constexpr (kBack) {
            turn(gw[k], k);
            dots = fma(gw[k].b * gain[k].b, w[k].b, fma(gw[k].a * gain[k].a, w[k].a, dots));
          }
        }
        ss = sum_of(sq);
        if constexpr (kBack) dot = sum_of(dots);
        group_sums(ss, dot, a.lanes_log2);
      }
      if (here) {   // (without a row, an eps of 0 would make NaNs, which the sums keep)
        if constexpr (kNorm) {
          const float rs = rsqrtf(ss * per_head + a.eps);
          const Lane<V> rs_all = all_of<V>(rs);
          if constexpr (!kBack) {
#pragma unroll
            for (int k = 0; k < kUnits; ++k) w[k].a = w[k].a * (rs_all * gain[k].a), w[k].b = w[k].b * (rs_all * gain[k].b);
          } else {
            const Lane<V> minus_dot = all_of<V>(-per_head * rs * dot);
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
              w[k].a = w[k].a * rs_all, w[k].b = w[k].b * rs_all;          // n
              sums[k].a = fma(gw[k].a, w[k].a, sums[k].a), sums[k].b = fma(gw[k].b, w[k].b, sums[k].b);
              w[k].a = rs_all * fma(w[k].a, minus_dot, gw[k].a * gain[k].a), w[k].b = rs_all * fma(w[k].b, minus_dot, gw[k].b * gain[k].b);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
          if constexpr (!kSums) turn(w[k], k);
          if constexpr (kBack) {
            if (a.accumulate) {
              Raw<T, V> raw_old;
              load_raw(raw_old, static_cast<const T *>(out), c0[k], c1[k], a.head);
              const Unit<V> old = unit_of<T, V, kLayout>(raw_old, c0[k] < a.head, c1[k] < a.head);
              const Lane<V> one = all_of<V>(1.f);
              w[k].a = fma(old.a, one, w[k].a), w[k].b = fma(old.b, one, w[k].b);
            }
          }
          store_unit<T, V, kLayout>(w[k], out, c0[k], c1[k], a.head);
        }
      }
      out += step;
    }
  }

  if constexpr (kSums) {
    if (!a.partial) return;
    __syncthreads();   // the gain's last readers are done
    const uint32_t warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) {
        const bool is_b = kLayout == B200_ROTARY_HALVES ? e >= V : (e & 1);
        float v = is_b ? sums[k].b.get(kLayout == B200_ROTARY_HALVES ? e - V : e / 2) : sums[k].a.get(kLayout == B200_ROTARY_HALVES ? e : e / 2);
        for (uint32_t o = lanes; o < 32u; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        const uint32_t c = e < V ? c0[k] : c1[k], at = c + (e < V ? e : e - V);
        if ((threadIdx.x & 31u) < lanes && c < a.head) s_sums[warp * kMaxHead + at] = v;
      }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.head; i += kThreads) {
      float v = 0.f;
#pragma unroll
      for (unsigned wp = 0; wp < kWarps; ++wp) v += s_sums[wp * kMaxHead + i];
      a.partial[static_cast<u64>(blockIdx.x) * a.head + i] = v;
    }
  }
}

// ggain = (accumulate ? ggain : 0) + the blocks' rows, added in order by 32 lanes of threads and then those in order.
template <typename T>
__global__ void __launch_bounds__(1024) gain_sums_kernel(const float *partial, uint32_t rows_q, uint32_t rows, uint32_t head, T *gq, T *gk, int accumulate) {
  pdl_enter();
  __shared__ float s[32][33];
  const uint32_t col = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (col < 2 * head)
#pragma unroll 4
    for (uint32_t r = threadIdx.y + (col < head ? 0u : rows_q); r < (col < head ? rows_q : rows); r += 32)
      v += partial[static_cast<u64>(r) * head + (col < head ? col : col - head)];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y != 0 || col >= 2 * head) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) v += s[i][threadIdx.x];
  T *out = col < head ? gq : gk;
  const uint32_t at = col < head ? col : col - head;
  if (out) st(out, at, (accumulate ? ld(out, at) : 0.f) + v);
}

// The widest vectors that every address and extent allows.
template <typename T>
uint32_t vector_width(const RotaryArgs &a, int layout, int back, int norm) {
  uint32_t v = norm ? 4 : 16 / sizeof(T);   // (with norms eight halves a lane take so many registers that four are faster)
  auto fits = [&](uint32_t n) {
    auto ok = [&](const void *p, u64 ld) { return !p || (reinterpret_cast<uintptr_t>(p) % (n * sizeof(T)) == 0 && ld % n == 0); };
    if (!ok(a.y, a.y_ld) || ((!back || norm) && !ok(a.x, a.x_ld)) || (back && !ok(a.g, a.g_ld))) return false;
    return a.head % n == 0 && (layout == B200_ROTARY_PAIRS ? a.rot % (2 * n) == 0 : (a.rot / 2) % n == 0);
  };
  while (v > 1 && !fits(v)) v /= 2;
  return v;
}

template <typename T, int V, int kLayout, bool kNorm, bool kBack>
int launch_rotary(b200_ctx *ctx, cudaStream_t s, RotaryArgs a, uint32_t *rows_q) {
  const uint32_t turned = a.rot / 2 / V;
  a.units = kLayout == B200_ROTARY_HALVES ? turned + ((a.head - a.rot) / V + 1) / 2 : (a.head / V + 1) / 2;
  a.lanes_log2 = 0;
  while ((kUnitsOf<V> << a.lanes_log2) < static_cast<int>(a.units)) ++a.lanes_log2;
  const uint32_t groups_log2 = 8 - a.lanes_log2, sms = static_cast<uint32_t>(ctx->sm_count);
  static_assert(kThreads == 256, "2^8");
  if (!kNorm) a.heads_q = a.heads;
  const uint32_t heads_k = a.heads - a.heads_q;
  constexpr bool kSums = kNorm && kBack;
  // A group takes kHeadsEach heads of its token at least, one after the other, unless there are so few tokens that two blocks for
  // every SM need them apart.
  auto split_of = [&](uint32_t heads) {
    uint32_t split = 0;
    while (split < groups_log2 && ((heads >> (split + 1)) >= kHeadsEach ||
                                   ((heads >> split) > 1 && (static_cast<u64>(a.tokens) << split) >> groups_log2 < 2 * sms)))
      ++split;
    return split;
  };
  a.split_q_log2 = split_of(a.heads_q), a.split_k_log2 = split_of(heads_k);
  auto tiles_of = [&](uint32_t split) { return (a.tokens + (1u << (groups_log2 - split)) - 1) >> (groups_log2 - split); };
  a.blocks_q = a.heads_q ? tiles_of(a.split_q_log2) : 0u;
  uint32_t blocks_k = heads_k ? tiles_of(a.split_k_log2) : 0u;
  if (kSums) {   // as many as are resident at a time, shared out by heads
    const uint32_t room = std::min(kSumBlocks * sms, kMaxPartials);
    const uint32_t mine = std::max(1u, static_cast<uint32_t>(static_cast<u64>(room) * a.heads_q / a.heads));
    if (a.blocks_q) a.blocks_q = std::min(a.blocks_q, heads_k ? std::min(mine, room - 1) : room);
    blocks_k = std::min(blocks_k, room - a.blocks_q);
  }
  const uint32_t most = 1u << (groups_log2 - std::min(a.heads_q ? a.split_q_log2 : groups_log2, heads_k ? a.split_k_log2 : groups_log2));
  const size_t smem = static_cast<size_t>(most) * ((a.rot / 2 + V - 1) / V) * V * sizeof(float2);
  b200::launch(ctx, rotary_kernel<T, V, kLayout, kNorm, kBack>, dim3(a.blocks_q + blocks_k), dim3(kThreads), smem, s, 1u, a);
  *rows_q = a.blocks_q;
  return static_cast<int>(a.blocks_q + blocks_k);
}

template <typename T, int kLayout, bool kNorm, bool kBack>
int launch_rotary_v(b200_ctx *ctx, cudaStream_t s, const RotaryArgs &a, uint32_t *rows_q) {
  switch (vector_width<T>(a, kLayout, kBack, kNorm)) {
    case 8: if constexpr (sizeof(T) == 2 && !kNorm) return launch_rotary<T, 8, kLayout, kNorm, kBack>(ctx, s, a, rows_q);
    case 4: return launch_rotary<T, 4, kLayout, kNorm, kBack>(ctx, s, a, rows_q);
    case 2: return launch_rotary<T, 2, kLayout, kNorm, kBack>(ctx, s, a, rows_q);
    default: return launch_rotary<T, 1, kLayout, kNorm, kBack>(ctx, s, a, rows_q);
  }
}

template <typename T, bool kNorm, bool kBack>
int launch_rotary_l(b200_ctx *ctx, cudaStream_t s, const RotaryArgs &a, int layout, uint32_t *rows_q) {
  return layout == B200_ROTARY_HALVES ? launch_rotary_v<T, B200_ROTARY_HALVES, kNorm, kBack>(ctx, s, a, rows_q)
                                      : launch_rotary_v<T, B200_ROTARY_PAIRS, kNorm, kBack>(ctx, s, a, rows_q);
}

// What every entry point refuses; fills in dense strides.
int check(RotaryArgs *a, int layout, bool norm) {
  if (layout != B200_ROTARY_PAIRS && layout != B200_ROTARY_HALVES) return B200_ERR_INVALID_ARG;
  if (a->head == 0 || a->rot > a->head || a->rot % 2 != 0 || (a->rot != 0 && !a->freqs)) return B200_ERR_INVALID_ARG;
  if (a->head > kMaxHead) return B200_ERR_TOO_LARGE;
  if (static_cast<u64>(a->heads) * a->head > 0x7fffffffu || a->tokens > 0x7fffffffu) return B200_ERR_TOO_LARGE;
  const u64 dense = static_cast<u64>(a->heads) * a->head;
  for (u64 *ld : {&a->x_ld, &a->g_ld, &a->y_ld}) {
    if (*ld == 0) *ld = dense;
    if (*ld < dense) return B200_ERR_INVALID_ARG;
  }
  if (norm && a->heads_q > 0 && !a->gain_q) return B200_ERR_INVALID_ARG;
  if (norm && a->heads > a->heads_q && !a->gain_k) return B200_ERR_INVALID_ARG;
  return B200_OK;
}

// In place needs the same rows on both sides, and nothing to add to.
bool clash(const void *in, u64 in_ld, const void *out, u64 out_ld, int accumulate) { return in == out && (in_ld != out_ld || accumulate); }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200_rotary_frequencies(uint32_t rot, double base, int scaling, double factor, double original, double *freqs_host,
                            double *amplitude_host) {
  if (rot == 0 || rot % 2 != 0 || !freqs_host || !(base > 1.0) || !std::isfinite(base)) return B200_ERR_INVALID_ARG;
  if (scaling < B200_ROTARY_PLAIN || scaling > B200_ROTARY_BY_PARTS) return B200_ERR_INVALID_ARG;
  if (scaling != B200_ROTARY_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return B200_ERR_INVALID_ARG;
  if (scaling == B200_ROTARY_BY_PARTS && (!(original >= 1.0) || !std::isfinite(original))) return B200_ERR_INVALID_ARG;
  const double r = rot, pi2 = 6.283185307179586;
  double amplitude = 1.0, lo = 0.0, hi = 0.0;
  if (scaling == B200_ROTARY_BASE && rot > 2) base *= std::pow(factor, r / (r - 2.0));
  if (scaling == B200_ROTARY_BY_PARTS) {
    // the pair that turns n times in `original` positions: original base^(-2p/rot) = 2 pi n.  There need not be one: of a long context
    // all pairs turn more than once, and the blend ends behind the last.
    auto pair = [&](double n) { return r * std::log(original / (n * pi2)) / (2.0 * std::log(base)); };
    lo = std::floor(pair(32.0));
    hi = std::ceil(pair(1.0));
    amplitude = 1.0 + 0.1 * std::log(factor);
  }
  for (uint32_t p = 0; p < rot / 2; ++p) {
    double f = std::pow(base, -2.0 * p / r);
    if (scaling == B200_ROTARY_LINEAR) f /= factor;
    if (scaling == B200_ROTARY_BY_PARTS) {
      const double slow = std::min(std::max((p - lo) / (hi - lo), 0.0), 1.0);
      f = f / factor * slow + f * (1.0 - slow);
    }
    freqs_host[p] = f;
  }
  if (amplitude_host) *amplitude_host = amplitude;
  return B200_OK;
}

int b200_rotary_fw(b200_ctx *ctx, int mode, const void *x, void *y, uint32_t head, uint32_t heads, uint32_t tokens, uint64_t x_ld,
                   uint64_t y_ld, uint32_t rot, int layout, const double *freqs, float amplitude, const uint32_t *positions, void *stream) {
  B200_OPS_PROLOGUE(ctx);
  RotaryArgs a = {};
  a.x = x, a.y = y, a.x_ld = x_ld, a.y_ld = y_ld, a.head = head, a.heads = heads, a.heads_q = heads, a.tokens = tokens, a.rot = rot;
  a.freqs = freqs, a.positions = positions, a.amplitude = amplitude;
  if (const int rc = check(&a, layout, false)) return rc;
  if (heads == 0 || tokens == 0) return B200_OK;
  if (!x || !y || clash(x, a.x_ld, y, a.y_ld, 0)) return B200_ERR_INVALID_ARG;
  ProfScope prof(ctx, kProfElementwise, s);
  uint32_t rows_q = 0;
  B200_DISPATCH_MODE(mode, { (launch_rotary_l<T, false, false>(ctx, s, a, layout, &rows_q)); });
  B200_OPS_EPILOGUE(ctx);
}

int b200_rotary_bw(b200_ctx *ctx, int mode, const void *gy, void *gx, uint32_t head, uint32_t heads, uint32_t tokens, uint64_t gy_ld,
                   uint64_t gx_ld, uint32_t rot, int layout, const double *freqs, float amplitude, const uint32_t *positions, int accumulate,
                   void *stream) {
  B200_OPS_PROLOGUE(ctx);
  RotaryArgs a = {};
  a.g = gy, a.y = gx, a.g_ld = gy_ld, a.y_ld = gx_ld, a.head = head, a.heads = heads, a.heads_q = heads, a.tokens = tokens, a.rot = rot;
  a.freqs = freqs, a.positions = positions, a.amplitude = amplitude, a.accumulate = accumulate;
  if (const int rc = check(&a, layout, false)) return rc;
  if (heads == 0 || tokens == 0) return B200_OK;
  if (!gy || !gx || clash(gy, a.g_ld, gx, a.y_ld, accumulate)) return B200_ERR_INVALID_ARG;
  ProfScope prof(ctx, kProfElementwise, s);
  uint32_t rows_q = 0;
  B200_DISPATCH_MODE(mode, { (launch_rotary_l<T, false, true>(ctx, s, a, layout, &rows_q)); });
  B200_OPS_EPILOGUE(ctx);
}

int b200_norm_rotary_fw(b200_ctx *ctx, int mode, const void *x, const void *gain_q, const void *gain_k, void *y, uint32_t head,
                        uint32_t heads_q, uint32_t heads_k, uint32_t tokens, uint64_t x_ld, uint64_t y_ld, uint32_t rot, int layout,
                        const double *freqs, float amplitude, const uint32_t *positions, float eps, void *stream) {
  B200_OPS_PROLOGUE(ctx);
  RotaryArgs a = {};
  a.x = x, a.y = y, a.gain_q = gain_q, a.gain_k = gain_k, a.x_ld = x_ld, a.y_ld = y_ld, a.head = head, a.heads = heads_q + heads_k;
  a.heads_q = heads_q, a.tokens = tokens, a.rot = rot, a.freqs = freqs, a.positions = positions, a.amplitude = amplitude, a.eps = eps;
  if (a.heads < heads_q || !(eps >= 0.f)) return B200_ERR_INVALID_ARG;
  if (const int rc = check(&a, layout, true)) return rc;
  if (a.heads == 0 || tokens == 0) return B200_OK;
  if (!x || !y || clash(x, a.x_ld, y, a.y_ld, 0)) return B200_ERR_INVALID_ARG;
  ProfScope prof(ctx, kProfElementwise, s);
  uint32_t rows_q = 0;
  B200_DISPATCH_MODE(mode, { (launch_rotary_l<T, true, false>(ctx, s, a, layout, &rows_q)); });
  B200_OPS_EPILOGUE(ctx);
}

int b200_norm_rotary_bw(b200_ctx *ctx, int mode, const void *x, const void *gain_q, const void *gain_k, const void *gy, void *gx,
                        void *ggain_q, void *ggain_k, float *scratch, uint32_t head, uint32_t heads_q, uint32_t heads_k, uint32_t tokens,
                        uint64_t x_ld, uint64_t gy_ld, uint64_t gx_ld, uint32_t rot, int layout, const double *freqs, float amplitude,
                        const uint32_t *positions, float eps, int accumulate_x, int accumulate_gain, void *stream) {
  B200_OPS_PROLOGUE(ctx);
  RotaryArgs a = {};
  a.x = x, a.g = gy, a.y = gx, a.gain_q = gain_q, a.gain_k = gain_k, a.x_ld = x_ld, a.g_ld = gy_ld, a.y_ld = gx_ld, a.head = head;
  a.heads = heads_q + heads_k, a.heads_q = heads_q, a.tokens = tokens, a.rot = rot, a.freqs = freqs, a.positions = positions;
  a.amplitude = amplitude, a.eps = eps, a.accumulate = accumulate_x;
  if (a.heads < heads_q || !(eps >= 0.f)) return B200_ERR_INVALID_ARG;
  if (const int rc = check(&a, layout, true)) return rc;
  const bool sums = ggain_q || ggain_k, none = a.heads == 0 || tokens == 0;
  if (sums && !scratch) return B200_ERR_INVALID_ARG;
  if (!none && (!x || !gy || !gx || x == gx || clash(gy, a.g_ld, gx, a.y_ld, accumulate_x))) return B200_ERR_INVALID_ARG;
  if (none && (!sums || accumulate_gain)) return B200_OK;
  a.partial = sums ? scratch : nullptr;
  ProfScope prof(ctx, kProfElementwise, s);
  uint32_t rows_q = 0;
  B200_DISPATCH_MODE(mode, {
    const int rows = none ? 0 : launch_rotary_l<T, true, true>(ctx, s, a, layout, &rows_q);
    if (sums) {
      b200::launch(ctx, gain_sums_kernel<T>, dim3((2 * head + 31) / 32), dim3(32, 32), 0, s, 1u, scratch, rows_q, rows, head,
                   static_cast<T *>(ggain_q), static_cast<T *>(ggain_k), accumulate_gain);
      if (!none) ++ctx->launches;
    }
  });
  B200_OPS_EPILOGUE(ctx);
}

}  // extern "C"
