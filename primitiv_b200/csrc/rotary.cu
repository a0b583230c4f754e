// Rotary positions, and norms of queries and keys with the rotation in the same pass.
//
//   rotary        (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t),  t = position * freqs[pair]
//   norm_rotary   n = x r, r = 1 / sqrt(mean(x^2) + eps);  y = turned (n gain)
//   backward      g = gy turned back (t -> -t);  ggain += sum g n;  gx += r (g gain - n mean(g gain n))
//
// Bound by memory: one read and one write of every element (three with a backward norm).  A group of lanes
// (a power of two) holds one head of one token in registers, so the norm's sums are a few shuffles and nothing is
// read twice.  A lane's unit is the two vectors that turn with one another: in the HALVES layout they lie rot/2
// apart, in the PAIRS layout side by side.
//
// The cosines depend on the token alone.  A block takes a tile of tokens, forms their angles once, in shared memory,
// and every head reads them from there: with each head forming its own, 40 heads of 128 would cost 2.6 million
// 64-bit products and sines per 1024 tokens instead of 65 thousand.  An angle is formed in turns and reduced in 64 bits,
// so position 1000000 has the same error (2^-26 of a turn) as position 0; its sine and cosine are 32-bit.
//
// Gradients of gains are sums over every token and head.  Each thread keeps its elements' sums in registers over all
// the rows its block takes, a block writes one partial row and a second kernel adds the rows in order: no atomics, the
// same bits every run.
#include <algorithm>
#include <cmath>

#include "../../include/primitiv_b200_attention.h"
#include "ops_common.cuh"

namespace b200 {
namespace {

constexpr unsigned kThreads = 256;
constexpr unsigned kWarps = kThreads / 32;
constexpr uint32_t kMaxHead = 256;
constexpr uint32_t kMaxTile = 16;          // tokens per block
constexpr uint32_t kMaxPartials = B200_NORM_ROTARY_SCRATCH / (2 * kMaxHead);

struct RotaryArgs {
  const void *x, *g;        // forward: x; backward: g = gy, and x where there is a norm
  void *y;                  // y or gx
  const void *gain_q, *gain_k;
  float *partial;           // [block][q, k][head], or null
  const double *freqs;
  const uint32_t *positions;
  u64 x_ld, g_ld, y_ld;
  uint32_t head, heads, heads_q, tokens, rot;
  uint32_t units, lanes_log2, tile;   // units of a head; lanes of a group; tokens of a tile
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

// Elements 0 .. V-1 of w are the first vector, V .. 2V-1 the second.  `tab`: this token's row of the table.
template <int V, int kLayout>
__device__ __forceinline__ void turn(float (&w)[2 * V], uint32_t u, uint32_t rot, const float2 *tab, uint32_t pitch) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int ia = kLayout == B200_ROTARY_HALVES ? j : 2 * j, ib = kLayout == B200_ROTARY_HALVES ? j + V : 2 * j + 1;
    if (2 * (u * V + j) < rot) {
      const float2 cs = tab[j * pitch + u];
      const float a = w[ia], b = w[ib];
      w[ia] = a * cs.x - b * cs.y;
      w[ib] = b * cs.x + a * cs.y;
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void load_unit(float (&w)[2 * V], const T *p, uint32_t c0, uint32_t c1, uint32_t head) {
  Pack<T, V> a, b;
  const bool has0 = c0 < head, has1 = c1 < head;
  if (has0) a = *reinterpret_cast<const Pack<T, V> *>(p + c0);
  if (has1) b = *reinterpret_cast<const Pack<T, V> *>(p + c1);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    w[j] = has0 ? to_float(a.v[j]) : 0.f;
    w[V + j] = has1 ? to_float(b.v[j]) : 0.f;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_unit(const float (&w)[2 * V], T *p, uint32_t c0, uint32_t c1, uint32_t head) {
  Pack<T, V> a, b;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    a.v[j] = from_float<T>(w[j]);
    b.v[j] = from_float<T>(w[V + j]);
  }
  if (c0 < head) *reinterpret_cast<Pack<T, V> *>(p + c0) = a;
  if (c1 < head) *reinterpret_cast<Pack<T, V> *>(p + c1) = b;
}

__device__ __forceinline__ float group_sum(float v, uint32_t lanes) {
  for (uint32_t o = 1; o < lanes; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// kUnits: units per lane (heads are at most 256 elements, so single elements need four, pairs two).
// kRows: rows a lane has in flight.  One would leave HBM waiting: 16 Ki tokens of 40 heads of 128 halves.
template <typename T, int V, int kLayout, bool kNorm, bool kBack>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a) {
  pdl_enter();
  constexpr int kUnits = V >= 4 ? 1 : (V == 2 ? 2 : 4);
  constexpr int kRows = kUnits == 1 && !(kNorm && kBack) ? 2 : 1;
  extern __shared__ float2 s_tab[];                                  // [tile][V][pitch]
  __shared__ float s_gain[kNorm ? 2 * kMaxHead : 1];
  __shared__ float s_sums[kNorm && kBack ? kWarps * 2 * kMaxHead : 1];

  const uint32_t lanes = 1u << a.lanes_log2, lane = threadIdx.x & (lanes - 1), first_row = threadIdx.x >> a.lanes_log2;
  const uint32_t row_step = kThreads >> a.lanes_log2;
  const uint32_t pairs = a.rot / 2, pitch = (pairs + V - 1) / V, tab_size = V * pitch;
  const uint32_t tiles = (a.tokens + a.tile - 1) / a.tile;
  if constexpr (kNorm) {
    for (uint32_t i = threadIdx.x; i < 2 * a.head; i += kThreads) {
      const bool k = i >= a.head;
      const T *gain = static_cast<const T *>(k ? a.gain_k : a.gain_q);
      s_gain[i] = gain ? to_float(gain[k ? i - a.head : i]) : 0.f;
    }
  }
  float sums[kNorm && kBack ? 2 : 1][kUnits][2 * V];
  if constexpr (kNorm && kBack) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int k = 0; k < kUnits; ++k)
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) sums[s][k][j] = 0.f;
  }

  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const uint32_t t0 = tile * a.tile, nt = min(a.tile, a.tokens - t0);
    __syncthreads();   // the table's last readers are done
    for (uint32_t i = threadIdx.x; i < nt * pairs; i += kThreads) {
      const uint32_t t = i / pairs, p = i - t * pairs;
      const double pos = a.positions ? static_cast<double>(a.positions[t0 + t]) : static_cast<double>(t0 + t);
      const double turns = pos * (a.freqs[p] * 0.15915494309189533577);   // 1 / (2 pi)
      float sn, cs;
      sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn, &cs);
      s_tab[t * tab_size + (p % V) * pitch + p / V] = make_float2(a.amplitude * cs, a.amplitude * (kBack ? -sn : sn));
    }
    __syncthreads();
    const uint32_t rows = nt * a.heads, rounds = (rows + row_step - 1) / row_step;   // the same for every lane: shuffles below
    for (uint32_t round = 0; round < rounds; round += kRows) {
      float w[kRows][kUnits][2 * V], gw[kNorm && kBack ? kRows : 1][kUnits][2 * V];
      uint32_t tok[kRows], h[kRows];
      bool live[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const uint32_t row = first_row + (round + r) * row_step;
        live[r] = row < rows;
        tok[r] = live[r] ? row / a.heads : 0u;
        h[r] = live[r] ? row - tok[r] * a.heads : 0u;
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
          uint32_t c0, c1;
          unit_at<V, kLayout>(lane + k * lanes, a.rot, c0, c1);
          const uint32_t head = live[r] ? a.head : 0u;
          const u64 t = t0 + tok[r], at = static_cast<u64>(h[r]) * a.head;
          load_unit<T, V>(w[r][k], static_cast<const T *>(kBack && !kNorm ? a.g : a.x) + t * (kBack && !kNorm ? a.g_ld : a.x_ld) + at, c0, c1, head);
          if constexpr (kNorm && kBack) load_unit<T, V>(gw[r][k], static_cast<const T *>(a.g) + t * a.g_ld + at, c0, c1, head);
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float2 *tab = s_tab + tok[r] * tab_size;
        if constexpr (kNorm) {
          float ss = 0.f;
#pragma unroll
          for (int k = 0; k < kUnits; ++k)
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) ss += w[r][k][j] * w[r][k][j];
          ss = group_sum(ss, lanes);
          const float rs = 1.f / sqrtf(ss / static_cast<float>(a.head) + a.eps);
          const uint32_t is_k = h[r] >= a.heads_q ? 1u : 0u;
          const float *gain = s_gain + is_k * a.head;
          if constexpr (!kBack) {
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
              uint32_t c0, c1;
              unit_at<V, kLayout>(lane + k * lanes, a.rot, c0, c1);
#pragma unroll
              for (int j = 0; j < V; ++j) {
                w[r][k][j] *= rs * (c0 < a.head ? gain[c0 + j] : 0.f);
                w[r][k][V + j] *= rs * (c1 < a.head ? gain[c1 + j] : 0.f);
              }
            }
          } else {
            float dot = 0.f;
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
              uint32_t c0, c1;
              unit_at<V, kLayout>(lane + k * lanes, a.rot, c0, c1);
              turn<V, kLayout>(gw[r][k], lane + k * lanes, a.rot, tab, pitch);
#pragma unroll
              for (int j = 0; j < 2 * V; ++j) {
                w[r][k][j] *= rs;                                        // n
                const float gn = gw[r][k][j] * w[r][k][j];
                if (live[r]) sums[0][k][j] += is_k ? 0.f : gn, sums[1][k][j] += is_k ? gn : 0.f;
                const uint32_t c = j < V ? c0 : c1;
                gw[r][k][j] *= c < a.head ? gain[c + (j < V ? j : j - V)] : 0.f;
                dot += gw[r][k][j] * w[r][k][j];
              }
            }
            dot = group_sum(dot, lanes) / static_cast<float>(a.head);
#pragma unroll
            for (int k = 0; k < kUnits; ++k)
#pragma unroll
              for (int j = 0; j < 2 * V; ++j) w[r][k][j] = rs * (gw[r][k][j] - w[r][k][j] * dot);
          }
        }
        if (!live[r]) continue;
        T *out = static_cast<T *>(a.y) + static_cast<u64>(t0 + tok[r]) * a.y_ld + static_cast<u64>(h[r]) * a.head;
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
          uint32_t c0, c1;
          unit_at<V, kLayout>(lane + k * lanes, a.rot, c0, c1);
          if constexpr (!(kNorm && kBack)) turn<V, kLayout>(w[r][k], lane + k * lanes, a.rot, tab, pitch);
          if constexpr (kBack) {
            if (a.accumulate) {
              float old[2 * V];
              load_unit<T, V>(old, out, c0, c1, a.head);
#pragma unroll
              for (int j = 0; j < 2 * V; ++j) w[r][k][j] += old[j];
            }
          }
          store_unit<T, V>(w[r][k], out, c0, c1, a.head);
        }
      }
    }
  }

  if constexpr (kNorm && kBack) {
    if (!a.partial) return;
    const uint32_t warp = threadIdx.x >> 5;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        uint32_t c0, c1;
        unit_at<V, kLayout>(lane + k * lanes, a.rot, c0, c1);
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) {
          float v = sums[s][k][j];
          for (uint32_t o = lanes; o < 32u; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
          const uint32_t c = (j < V ? c0 : c1), at = c + (j < V ? j : j - V);
          if ((threadIdx.x & 31u) < lanes && c < a.head) s_sums[(warp * 2 + s) * kMaxHead + at] = v;
        }
      }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 2 * a.head; i += kThreads) {
      const uint32_t s = i >= a.head ? 1u : 0u, at = i - s * a.head;
      float v = 0.f;
#pragma unroll
      for (unsigned wp = 0; wp < kWarps; ++wp) v += s_sums[(wp * 2 + s) * kMaxHead + at];
      a.partial[(static_cast<u64>(blockIdx.x) * 2 + s) * a.head + at] = v;
    }
  }
}

// ggain = (accumulate ? ggain : 0) + the blocks' rows, added in order by 32 lanes of threads and then those in order.
template <typename T>
__global__ void __launch_bounds__(1024) gain_sums_kernel(const float *partial, uint32_t rows, uint32_t head, T *gq, T *gk, int accumulate) {
  pdl_enter();
  __shared__ float s[32][33];
  const uint32_t col = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (col < 2 * head)
#pragma unroll 4
    for (uint32_t r = threadIdx.y; r < rows; r += 32) v += partial[static_cast<u64>(r) * 2 * head + col];
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
  uint32_t v = 16 / sizeof(T);
  auto fits = [&](uint32_t n) {
    auto ok = [&](const void *p, u64 ld) { return !p || (reinterpret_cast<uintptr_t>(p) % (n * sizeof(T)) == 0 && ld % n == 0); };
    if (!ok(a.y, a.y_ld) || ((!back || norm) && !ok(a.x, a.x_ld)) || (back && !ok(a.g, a.g_ld))) return false;
    return a.head % n == 0 && (layout == B200_ROTARY_PAIRS || (a.rot / 2) % n == 0);
  };
  while (v > 1 && !fits(v)) v /= 2;
  return v;
}

template <typename T, int V, int kLayout, bool kNorm, bool kBack>
int launch_rotary(b200_ctx *ctx, cudaStream_t s, RotaryArgs a) {
  const uint32_t turned = a.rot / 2 / V;
  a.units = kLayout == B200_ROTARY_HALVES ? turned + ((a.head - a.rot) / V + 1) / 2 : (a.head / V + 1) / 2;
  constexpr int kUnits = V >= 4 ? 1 : (V == 2 ? 2 : 4);
  a.lanes_log2 = 0;
  while ((kUnits << a.lanes_log2) < static_cast<int>(a.units)) ++a.lanes_log2;
  const uint32_t at_once = kThreads >> a.lanes_log2;
  // Four rows a lane, but enough blocks for two on every SM first.
  const uint32_t sms = static_cast<uint32_t>(ctx->sm_count);
  a.tile = std::min(std::max(4 * at_once / a.heads, 1u), kMaxTile);
  while (a.tile > 1 && (a.tokens + a.tile - 1) / a.tile < 2 * sms) a.tile /= 2;
  const uint32_t tiles = (a.tokens + a.tile - 1) / a.tile;
  const uint32_t grid = kNorm && kBack ? std::min(tiles, std::min(3 * sms, kMaxPartials)) : tiles;
  const size_t smem = static_cast<size_t>(a.tile) * ((a.rot / 2 + V - 1) / V) * V * sizeof(float2);
  b200::launch(ctx, rotary_kernel<T, V, kLayout, kNorm, kBack>, dim3(grid), dim3(kThreads), smem, s, 1u, a);
  return static_cast<int>(grid);
}

template <typename T, int kLayout, bool kNorm, bool kBack>
int launch_rotary_v(b200_ctx *ctx, cudaStream_t s, const RotaryArgs &a) {
  switch (vector_width<T>(a, kLayout, kBack, kNorm)) {
    case 8: if constexpr (sizeof(T) == 2) return launch_rotary<T, 8, kLayout, kNorm, kBack>(ctx, s, a);
    case 4: return launch_rotary<T, 4, kLayout, kNorm, kBack>(ctx, s, a);
    case 2: return launch_rotary<T, 2, kLayout, kNorm, kBack>(ctx, s, a);
    default: return launch_rotary<T, 1, kLayout, kNorm, kBack>(ctx, s, a);
  }
}

template <typename T, bool kNorm, bool kBack>
int launch_rotary_l(b200_ctx *ctx, cudaStream_t s, const RotaryArgs &a, int layout) {
  return layout == B200_ROTARY_HALVES ? launch_rotary_v<T, B200_ROTARY_HALVES, kNorm, kBack>(ctx, s, a)
                                      : launch_rotary_v<T, B200_ROTARY_PAIRS, kNorm, kBack>(ctx, s, a);
}

// What every entry point refuses; fills in dense strides.
int check(RotaryArgs *a, int layout, bool norm) {
  if (layout != B200_ROTARY_PAIRS && layout != B200_ROTARY_HALVES) return B200_ERR_INVALID_ARG;
  if (a->head == 0 || a->rot > a->head || a->rot % 2 != 0 || (a->rot != 0 && !a->freqs)) return B200_ERR_INVALID_ARG;
  if (a->head > kMaxHead) return B200_ERR_TOO_LARGE;
  if (static_cast<u64>(a->heads) * a->head > 0xffffffffu / kMaxTile) return B200_ERR_TOO_LARGE;
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
    // the pair that turns n times in `original` positions: original base^(-2p/rot) = 2 pi n
    auto pair = [&](double n) { return r * std::log(original / (n * pi2)) / (2.0 * std::log(base)); };
    lo = std::max(std::floor(pair(32.0)), 0.0);
    hi = std::min(std::ceil(pair(1.0)), r / 2.0 - 1.0);
    amplitude = 1.0 + 0.1 * std::log(factor);
  }
  for (uint32_t p = 0; p < rot / 2; ++p) {
    double f = std::pow(base, -2.0 * p / r);
    if (scaling == B200_ROTARY_LINEAR) f /= factor;
    if (scaling == B200_ROTARY_BY_PARTS) {
      const double slow = std::min(std::max((p - lo) / std::max(hi - lo, 0.001), 0.0), 1.0);
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
  B200_DISPATCH_MODE(mode, { (launch_rotary_l<T, false, false>(ctx, s, a, layout)); });
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
  B200_DISPATCH_MODE(mode, { (launch_rotary_l<T, false, true>(ctx, s, a, layout)); });
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
  B200_DISPATCH_MODE(mode, { (launch_rotary_l<T, true, false>(ctx, s, a, layout)); });
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
  B200_DISPATCH_MODE(mode, {
    const int rows = none ? 0 : launch_rotary_l<T, true, true>(ctx, s, a, layout);
    if (sums) {
      b200::launch(ctx, gain_sums_kernel<T>, dim3((2 * head + 31) / 32), dim3(32, 32), 0, s, 1u, scratch, rows, head,
                   static_cast<T *>(ggain_q), static_cast<T *>(ggain_k), accumulate_gain);
      if (!none) ++ctx->launches;
    }
  });
  B200_OPS_EPILOGUE(ctx);
}

}  // extern "C"
