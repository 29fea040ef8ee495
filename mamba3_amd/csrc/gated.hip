// m3_gated_scan and m3_gated_scan_bwd: a gated linear recurrence with one FP32 state per channel.
//
//   given form:  h_t = a_t h_{t-1} + x_t,               a_t = exp(decay_t)
//   gate form:   h_t = a_t h_{t-1} + s_t q_t x_t,       a_t = exp(-rate p_t), s_t = sqrt(1 - a_t^2)
// with p_t = sigmoid(decay_t), q_t = sigmoid(gate_t).
//
// Forward, one token: one lane owns a channel (two where rows allow). Forward, more tokens: a
// workgroup takes a tile of 128 tokens x 128 channels, which stays in registers, so x, decay and
// gate are read once. Each of its 8 waves runs 16 tokens from a zero state, which gives the span's map
// h -> A h + H; the maps of the waves before give a wave its entry state, and the tokens are run
// again from there with one fma each. Tiles of one row are chained through memory: a tile publishes its own
// map, then looks back for the nearest state that is already known.
//
// The backward pass walks a channel's tokens from the end, tile by tile, recomputing each tile's
// states from the carry the forward pass left.
#include <hip/hip_runtime.h>

#include "m3_common.hpp"
#include "m3_host.hpp"

namespace m3 {
namespace {

constexpr int kTile = M3_GATED_TILE;
constexpr float kLog2e = 1.44269504088896340736f;

struct GatedGeom {
  const char *x, *r, *g;       // x, decay, gate: byte addresses
  const float* rate;
  const float* init;           // or null
  const int32_t* lengths;      // or null
  const uint8_t* reset;        // or null
  char* y;
  float* fin;
  float* carry;                // [tiles, B, C] or null
  int64_t x_b, r_b, g_b, y_b, init_b, fin_b, reset_b;  // batch strides (elements)
  int64_t x_t, r_t, g_t, y_t;                          // token strides
  int batch, length, width, tiles;
  // backward
  const char* dy;
  const float* dfin;           // or null
  char *dx, *dr, *dg;
  float* dinit;                // or null
  float* drate;                // [C]
  float* part;                 // partial sums of drate, [rows, C]
  float* scratch;              // [B, kTile, C]
  int64_t dy_b, dx_b, dr_b, dg_b, dfin_b, dinit_b;
  int64_t dy_t, dx_t, dr_t, dg_t;
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const char* p, int64_t i, float (&v)[VEC]) {
  typedef T tv __attribute__((ext_vector_type(VEC)));
  if constexpr (VEC == 1) {
    v[0] = to_f(reinterpret_cast<const T*>(p)[i]);
  } else {
    const tv t = *reinterpret_cast<const tv*>(reinterpret_cast<const T*>(p) + i);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = to_f(t[e]);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(char* p, int64_t i, const float (&v)[VEC]) {
  typedef T tv __attribute__((ext_vector_type(VEC)));
  if constexpr (VEC == 1) {
    reinterpret_cast<T*>(p)[i] = from_f<T>(v[0]);
  } else {
    tv t;
#pragma unroll
    for (int e = 0; e < VEC; ++e) t[e] = from_f<T>(v[e]);
    *reinterpret_cast<tv*>(reinterpret_cast<T*>(p) + i) = t;
  }
}

// Loads of a wave's span: its first token's address in a buffer descriptor, the token as a
// scalar offset and the channel as the lane's, so that no load needs a 64-bit address of its own.
template <typename T, int VEC>
struct Span {
  __amdgpu_buffer_rsrc_t rsrc;
  int stride;  // bytes between tokens
  int off;     // the lane's channel, in bytes
  __device__ __forceinline__ Span(const char* base, int64_t first, int64_t token_stride, int c)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(base + first * static_cast<int64_t>(sizeof(T))), static_cast<short>(0),
            0x7fffffff, 0x00020000)),
        stride(static_cast<int>(token_stride) * static_cast<int>(sizeof(T))),
        off(c * static_cast<int>(sizeof(T))) {}
  __device__ __forceinline__ auto load(int i) const {
    if constexpr (sizeof(T) * VEC == 8) {
      return __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, i * stride, 0);
    } else if constexpr (sizeof(T) * VEC == 4) {
      return __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, i * stride, 0);
    } else {
      return __builtin_amdgcn_raw_buffer_load_b16(rsrc, off, i * stride, 0);
    }
  }
};

// One token of one channel: its factor a and input b = w x, and what the gradients need.
struct Coef {
  float a, b, w;      // w = s q (1 in the given form)
  float p, q, pp, qq; // gates' sigmoids, p (1 - p), q (1 - q)
  float s, inv;       // sqrt(1 - a^2) and its reciprocal (0 where s is)
};

// 1 - exp(u) for u <= 0: the series of -expm1 near 0, where the difference would lose its digits
// (at -0.125 the first term left out is 4e-8 of the sum, the difference's error 5e-7).
__device__ __forceinline__ float one_minus_exp(float u, float e) {
  const float series =
      -u * fmaf(u, fmaf(u, fmaf(u, fmaf(u, 1.f / 120.f, 1.f / 24.f), 1.f / 6.f), 0.5f), 1.f);
  return u > -0.125f ? series : 1.f - e;
}

template <bool GATE>
__device__ __forceinline__ Coef coef(float x, float r, float g, float rate) {
  Coef c;
  if constexpr (!GATE) {
    c.a = __builtin_amdgcn_exp2f(r * kLog2e);
    c.b = x;
    c.w = 1.f;
  } else {
    // from exp(-|r|): both sigmoid and its complement keep their digits
    const float er = __builtin_amdgcn_exp2f(-fabsf(r) * kLog2e);
    const float hr = __builtin_amdgcn_rcpf(1.f + er);
    const float eg = __builtin_amdgcn_exp2f(-fabsf(g) * kLog2e);
    const float hg = __builtin_amdgcn_rcpf(1.f + eg);
    c.p = r < 0.f ? er * hr : hr;
    c.q = g < 0.f ? eg * hg : hg;
    c.pp = er * hr * hr;
    c.qq = eg * hg * hg;
    const float la = -rate * c.p;
    c.a = __builtin_amdgcn_exp2f(la * kLog2e);
    const float v = one_minus_exp(2.f * la, c.a * c.a);
    c.inv = fabsf(v) < 1e-37f ? 0.f : __builtin_amdgcn_rsqf(v);
    c.s = v * c.inv;
    c.w = c.s * c.q;
    c.b = c.w * x;
  }
  return c;
}

// The forward pass's share of it: the factor and the input.
template <bool GATE>
__device__ __forceinline__ void factor_input(float x, float r, float g, float rate, float& a,
                                             float& b) {
  if constexpr (!GATE) {
    a = __builtin_amdgcn_exp2f(r * kLog2e);
    b = x;
  } else {
    const float p = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(r * -kLog2e));
    const float q = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -kLog2e));
    a = __builtin_amdgcn_exp2f(rate * -kLog2e * p);
    const float v = one_minus_exp(rate * -2.f * p, a * a);
    b = __builtin_amdgcn_sqrtf(v) * q * x;
  }
}

__device__ __forceinline__ int row_length(const GatedGeom& g, int b) {
  return g.lengths == nullptr ? g.length : max(0, min(g.lengths[b], g.length));
}

// ----------------------------------------------------------------------------- chained tiles

// A span's map v -> A v + H. A < 0 marks a span that a reset cuts: what enters it is dropped, NaN
// and infinities too (a factor that merely underflows to 0 still passes NaN on).
__device__ __forceinline__ float fold(float a, float h, float v) {
  return a < 0.f ? h : fmaf(a, v, h);
}
__device__ __forceinline__ float join(float a, float b) {
  return a < 0.f || b < 0.f ? -1.f : a * b;
}

// What tiles tell each other: 32-bit states and 64-bit maps (H low, A high), each written and read as
// one relaxed atomic of device scope, with all bits set for "not yet" (a NaN of these bits is
// published as another). No fence and no flag beside the data is needed.
constexpr uint32_t kNotYet = 0xffffffffu;

__device__ __forceinline__ uint32_t word(float v) {
  const uint32_t u = __float_as_uint(v);
  return u == kNotYet ? 0x7fc00000u : u;
}

struct Chain {
  uint32_t* ticket;  // tiles started so far
  uint64_t* maps;    // [tiles, B, C]
  uint32_t* states;  // [tiles, B, C]: the state that leaves a tile
};

constexpr int kWindow = 4;           // tiles looked back over at once
constexpr int kSpins = 1 << 22;      // polls (about 1 us each) before a wait gives up with NaN

template <int VEC>
__device__ __forceinline__ void read_states(const uint32_t* p, uint32_t (&v)[VEC]) {
  if constexpr (VEC == 2) {
    const uint64_t u = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    v[0] = static_cast<uint32_t>(u);
    v[1] = static_cast<uint32_t>(u >> 32);
  } else {
    v[0] = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

template <int VEC>
__device__ __forceinline__ void write_states(uint32_t* p, const float (&v)[VEC]) {
  if constexpr (VEC == 2) {
    const uint64_t u = static_cast<uint64_t>(word(v[1])) << 32 | word(v[0]);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), u, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  } else {
    __hip_atomic_store(p, word(v[0]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// The state that enters link s of a chain (s >= 1), for the channels at `at`; `step` elements lie between links.
// Waits until, for every channel, one of the kWindow links before has published its state and
// all links after that one their maps. The state is carried forward over those maps by the very
// operation with which each link computes its own state, so it does not depend on which
// link was found. Every wait ends: links are started in ticket order, each waits for earlier ones
// only, and a running wave always gets to run; kSpins is there in case that is wrong.
template <int VEC>
__device__ __forceinline__ void look_back(const Chain& ch, int s, int64_t at, int64_t step,
                                          bool live, float (&v)[VEC]) {
  const int n = min(kWindow, s);
  for (int spin = 0;; ++spin) {
    uint32_t st[kWindow][VEC];
    uint64_t map[kWindow][VEC];
#pragma unroll
    for (int j = 0; j < kWindow; ++j) {
      const int64_t p = at + (s - 1 - min(j, n - 1)) * step;
      read_states<VEC>(ch.states + p, st[j]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        map[j][e] = __hip_atomic_load(ch.maps + p + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    bool all = true;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      bool have = false;
#pragma unroll
      for (int j = kWindow - 1; j >= 0; --j) {
        const uint32_t a = static_cast<uint32_t>(map[j][e] >> 32);
        if (st[j][e] != kNotYet) {
          v[e] = __uint_as_float(st[j][e]);
          have = true;
        } else {
          v[e] = fold(__uint_as_float(a), __uint_as_float(static_cast<uint32_t>(map[j][e])), v[e]);
          have = have && a != kNotYet;
        }
      }
      all = all && have;
    }
    if (__all(all || !live)) return;
    if (spin >= kSpins) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = __uint_as_float(0x7fc00000u);
      return;
    }
    __builtin_amdgcn_s_sleep(2);
  }
}

__global__ __launch_bounds__(256) void gated_chain_kernel(Chain ch, int64_t cells) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i == 0) *ch.ticket = 0;
  if (i >= cells) return;
  ch.maps[i] = ~uint64_t{0};
  ch.states[i] = kNotYet;
}

constexpr int kWaves = 8, kSpan = kTile / kWaves;  // a wave's tokens

template <typename T, bool GATE, int VEC, bool CHAIN>
__global__ __launch_bounds__(64 * kWaves, 4) void gated_tile_kernel(const GatedGeom g,
                                                                    const Chain ch) {
  constexpr int kCols = 64 * VEC;
  __shared__ float s_a[kWaves][kCols], s_h[kWaves][kCols], s_in[kCols];
  __shared__ unsigned s_ticket;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned id = blockIdx.x;
  if constexpr (CHAIN) {
    // tiles in the order in which workgroups start, so that none waits for one not yet started
    if (tid == 0) s_ticket = atomicAdd(ch.ticket, 1u);
    __syncthreads();
    id = __builtin_amdgcn_readfirstlane(s_ticket);
  }
  const unsigned groups = (g.width + kCols - 1) / kCols, cells = g.batch * groups;
  const int s = id / cells, b = id % cells / groups;
  const int c0 = (id % groups) * kCols + lane * VEC;
  const bool live = c0 < g.width;
  const int c = min(c0, g.width - VEC);  // lanes past the width read its last channels
  const int t0 = s * kTile + w * kSpan;
  const int n = max(0, min(row_length(g, b) - t0, kSpan));  // tokens of this wave
  const int64_t step = static_cast<int64_t>(g.batch) * g.width;
  const int64_t at = static_cast<int64_t>(b) * g.width + c;

  uint32_t early[VEC];
  if constexpr (CHAIN) {
    if (w == 0 && s > 0) read_states<VEC>(ch.states + at + (s - 1) * step, early);
  }
  float rate[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) rate[e] = GATE ? g.rate[c + e] : 0.f;
  uint64_t cut = 0;
  if (g.reset != nullptr) {
    cut = __ballot(lane < n && g.reset[b * g.reset_b + t0 + min(lane, max(n - 1, 0))] != 0);
  }

  float a[kSpan][VEC], h[kSpan][VEC];  // h: first the inputs
  float span_a[VEC], span_h[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) span_a[e] = 1.f, span_h[e] = 0.f;
  if (n > 0) {
    const Span<T, VEC> x(g.x, b * g.x_b + t0 * g.x_t, g.x_t, c);
    const Span<T, VEC> r(g.r, b * g.r_b + t0 * g.r_t, g.r_t, c);
    const Span<T, VEC> q(GATE ? g.g : g.x, b * g.g_b + t0 * g.g_t, g.g_t, c);
    typedef T tv __attribute__((ext_vector_type(VEC)));
    tv xv[kSpan], rv[kSpan], qv[kSpan];
#pragma unroll
    for (int i = 0; i < kSpan; ++i) {
      const int t = min(i, n - 1);
      xv[i] = __builtin_bit_cast(tv, x.load(t));
      rv[i] = __builtin_bit_cast(tv, r.load(t));
      if constexpr (GATE) qv[i] = __builtin_bit_cast(tv, q.load(t));
    }
#pragma unroll
    for (int i = 0; i < kSpan; ++i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        factor_input<GATE>(to_f(xv[i][e]), to_f(rv[i][e]), GATE ? to_f(qv[i][e]) : 0.f, rate[e],
                           a[i][e], h[i][e]);
      }
    }
    if (n < kSpan || cut != 0) {
#pragma unroll
      for (int i = 0; i < kSpan; ++i) {
        const bool past = i >= n, fresh = (cut >> i) & 1;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          a[i][e] = past ? 1.f : fresh ? -1.f : a[i][e];
          h[i][e] = past ? 0.f : h[i][e];
        }
      }
    }
    if (cut == 0) {
#pragma unroll
      for (int i = 0; i < kSpan; ++i) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          span_h[e] = fmaf(a[i][e], span_h[e], h[i][e]);
          span_a[e] *= a[i][e];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSpan; ++i) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          span_h[e] = fold(a[i][e], h[i][e], span_h[e]);
          span_a[e] = join(span_a[e], a[i][e]);
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    s_a[w][lane * VEC + e] = span_a[e];
    s_h[w][lane * VEC + e] = span_h[e];
  }
  __syncthreads();
  float v[VEC];  // the state that enters the tile, then the wave
  if (!CHAIN || s == 0) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = g.init != nullptr ? g.init[b * g.init_b + c + e] : 0.f;
  }
  if constexpr (CHAIN) {
    if (w == 0) {
      float ta[VEC], th[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        ta[e] = 1.f, th[e] = 0.f;
#pragma unroll
        for (int u = 0; u < kWaves; ++u) {
          const float ua = s_a[u][lane * VEC + e];
          th[e] = fold(ua, s_h[u][lane * VEC + e], th[e]);
          ta[e] = join(ta[e], ua);
        }
      }
      if (s > 0) {
        bool known = true;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          known = known && early[e] != kNotYet;
          v[e] = __uint_as_float(early[e]);
        }
        if (!__all(known || !live)) {
          if (live) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const uint64_t m = static_cast<uint64_t>(word(ta[e])) << 32 | __float_as_uint(th[e]);
              __hip_atomic_store(ch.maps + at + s * step + e, m, __ATOMIC_RELAXED,
                                 __HIP_MEMORY_SCOPE_AGENT);
            }
          }
          look_back<VEC>(ch, s, at, step, live, v);
        }
      }
      float out[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        out[e] = fold(ta[e], th[e], v[e]);
        s_in[lane * VEC + e] = v[e];
      }
      if (live) {
        if (s < g.tiles - 1 || g.carry != nullptr) write_states<VEC>(ch.states + at + s * step, out);
        if (s == g.tiles - 1) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) g.fin[b * g.fin_b + c + e] = out[e];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = s_in[lane * VEC + e];
  }
#pragma unroll
  for (int u = 0; u < kWaves; ++u) {
    if (u < w) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[e] = fold(s_a[u][lane * VEC + e], s_h[u][lane * VEC + e], v[e]);
      }
    }
  }
  const int rows = max(0, min(g.length - t0, kSpan));
  T* y = reinterpret_cast<T*>(g.y) + b * g.y_b + t0 * g.y_t;
  if (n == kSpan && cut == 0) {
#pragma unroll
    for (int i = 0; i < kSpan; ++i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = fmaf(a[i][e], v[e], h[i][e]);
      if (live) store_vec<T, VEC>(reinterpret_cast<char*>(y), i * g.y_t + c, v);
    }
  } else {
    const float zero[VEC] = {};
#pragma unroll
    for (int i = 0; i < kSpan; ++i) {
      if (i < n) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = fold(a[i][e], h[i][e], v[e]);
      }
      if (live && i < rows) {
        if (i < n) store_vec<T, VEC>(reinterpret_cast<char*>(y), i * g.y_t + c, v);
        else store_vec<T, VEC>(reinterpret_cast<char*>(y), i * g.y_t + c, zero);
      }
    }
  }
  if (!CHAIN && w == kWaves - 1 && live) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      g.fin[b * g.fin_b + c + e] = v[e];
      if (g.carry != nullptr) g.carry[at + e] = v[e];
    }
  }
}

// ----------------------------------------------------------------------------- token walk

template <typename T, bool GATE, int VEC>
__global__ __launch_bounds__(256) void gated_walk_kernel(const GatedGeom g) {
  const int lanes = g.width / VEC;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int b = static_cast<int>(id / lanes), c = static_cast<int>(id % lanes) * VEC;
  if (b >= g.batch) return;
  const int len = row_length(g, b);
  float rate[VEC], h[VEC], x[VEC], r[VEC], q[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    rate[e] = GATE ? g.rate[c + e] : 0.f;
    h[e] = g.init != nullptr ? g.init[b * g.init_b + c + e] : 0.f;
    q[e] = 0.f;
  }
  for (int t = 0; t < g.length; ++t) {
    float y[VEC];
    if (t < len) {
      load_vec<T, VEC>(g.x, b * g.x_b + t * g.x_t + c, x);
      load_vec<T, VEC>(g.r, b * g.r_b + t * g.r_t + c, r);
      if constexpr (GATE) load_vec<T, VEC>(g.g, b * g.g_b + t * g.g_t + c, q);
      const bool fresh = g.reset != nullptr && g.reset[b * g.reset_b + t] != 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const Coef k = coef<GATE>(x[e], r[e], q[e], rate[e]);
        h[e] = fresh ? k.b : fmaf(k.a, h[e], k.b);
        y[e] = h[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = 0.f;
    }
    store_vec<T, VEC>(g.y, b * g.y_b + t * g.y_t + c, y);
    if (g.carry != nullptr && (t % kTile == kTile - 1 || t == g.length - 1)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        g.carry[(static_cast<int64_t>(t / kTile) * g.batch + b) * g.width + c + e] = h[e];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) g.fin[b * g.fin_b + c + e] = h[e];
}

template <typename T, bool GATE>
__global__ __launch_bounds__(256) void gated_walk_bwd_kernel(const GatedGeom g) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int b = static_cast<int>(id / g.width), c = static_cast<int>(id % g.width);
  if (b >= g.batch) return;
  const int len = row_length(g, b);
  const float rate = GATE ? g.rate[c] : 0.f;
  float grad = g.dfin != nullptr ? g.dfin[b * g.dfin_b + c] : 0.f;  // a_{t+1} D_{t+1}
  float sum = 0.f;
  float x[1], r[1], q[1] = {0.f}, dy[1];
  for (int s = g.tiles - 1; s >= 0; --s) {
    const int t0 = s * kTile, t1 = min(g.length, t0 + kTile);
    float h = s > 0 ? g.carry[(static_cast<int64_t>(s - 1) * g.batch + b) * g.width + c]
                    : (g.init != nullptr ? g.init[b * g.init_b + c] : 0.f);
    for (int t = t0; t < t1; ++t) {
      const bool fresh = g.reset != nullptr && g.reset[b * g.reset_b + t] != 0;
      if (fresh && t < len) h = 0.f;
      g.scratch[(static_cast<int64_t>(b) * kTile + t - t0) * g.width + c] = h;
      if (t < len) {
        load_vec<T, 1>(g.x, b * g.x_b + t * g.x_t + c, x);
        load_vec<T, 1>(g.r, b * g.r_b + t * g.r_t + c, r);
        if constexpr (GATE) load_vec<T, 1>(g.g, b * g.g_b + t * g.g_t + c, q);
        const Coef k = coef<GATE>(x[0], r[0], q[0], rate);
        h = fmaf(k.a, h, k.b);
      }
    }
    for (int t = t1 - 1; t >= t0; --t) {
      float dx[1] = {0.f}, dr[1] = {0.f}, dg[1] = {0.f};
      if (t < len) {
        load_vec<T, 1>(g.x, b * g.x_b + t * g.x_t + c, x);
        load_vec<T, 1>(g.r, b * g.r_b + t * g.r_t + c, r);
        if constexpr (GATE) load_vec<T, 1>(g.g, b * g.g_b + t * g.g_t + c, q);
        load_vec<T, 1>(g.dy, b * g.dy_b + t * g.dy_t + c, dy);
        const Coef k = coef<GATE>(x[0], r[0], q[0], rate);
        const float before = g.scratch[(static_cast<int64_t>(b) * kTile + t - t0) * g.width + c];
        const float d = dy[0] + grad;
        dx[0] = d * k.w;
        if constexpr (GATE) {
          const float dlog = d * (k.a * before - k.q * x[0] * (k.a * k.a * k.inv));
          dr[0] = -rate * k.pp * dlog;
          dg[0] = d * x[0] * k.s * k.qq;
          sum -= k.p * dlog;
        } else {
          dr[0] = d * (k.a * before);
        }
        const bool fresh = g.reset != nullptr && g.reset[b * g.reset_b + t] != 0;
        grad = fresh ? 0.f : k.a * d;
      }
      store_vec<T, 1>(g.dx, b * g.dx_b + t * g.dx_t + c, dx);
      store_vec<T, 1>(g.dr, b * g.dr_b + t * g.dr_t + c, dr);
      if constexpr (GATE) store_vec<T, 1>(g.dg, b * g.dg_b + t * g.dg_t + c, dg);
    }
  }
  if (g.dinit != nullptr) g.dinit[b * g.dinit_b + c] = grad;
  if constexpr (GATE) g.part[static_cast<int64_t>(b) * g.width + c] = sum;
}

// drate[c] = the sum of rows of partial sums, in 64 bits (a cancelling sum over all tokens).
__global__ __launch_bounds__(256) void gated_rate_kernel(const float* part, float* drate, int rows,
                                                         int width) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= width) return;
  double sum = 0.0;
  for (int i = 0; i < rows; ++i) sum += part[static_cast<int64_t>(i) * width + c];
  drate[c] = static_cast<float>(sum);
}

// ----------------------------------------------------------------------------- host

int check_rows(const m3_tensor& t, const char* name, int dims, int64_t inner, bool required,
               int dtype) {
  return check_tensor(t, name, dims, inner, required, dtype);
}

int validate(const m3_gated_scan_args& a, bool backward) {
  if (a.batch < 0 || a.length < 0 || a.width < 0) {
    return fail(M3_EINVAL, "m3_gated_scan: negative dimensions");
  }
  if (!valid_dtype(a.dtype)) return fail(M3_EINVAL, "m3_gated_scan: invalid dtype %d", a.dtype);
  if (present(a.gate) != present(a.rate)) {
    return fail(M3_EINVAL, "m3_gated_scan: gate and rate are given together or not at all");
  }
  // a span's offsets are 32-bit, in bytes
  for (const m3_tensor* t : {&a.x, &a.decay, &a.gate, &a.out}) {
    if (t->ptr != nullptr && t->stride[1] > (1 << 24)) {
      return fail(M3_EUNSUPPORTED, "m3_gated_scan: tokens over 2^24 elements apart");
    }
  }
  // the lanes of a launch are counted in 32 bits
  if (static_cast<int64_t>(a.batch) * a.width >= INT32_MAX / 2) {
    return fail(M3_EUNSUPPORTED, "m3_gated_scan: batch * width %lld is above 2^30",
                static_cast<long long>(a.batch) * a.width);
  }
  const bool live = a.batch > 0 && a.length > 0 && a.width > 0;
  int rc;
  if ((rc = check_rows(a.x, "x", 3, a.width, live, a.dtype)) ||
      (rc = check_rows(a.decay, "decay", 3, a.width, live, a.dtype)) ||
      (rc = check_rows(a.gate, "gate", 3, a.width, false, a.dtype)) ||
      (rc = check_rows(a.rate, "rate", 1, a.width, false, M3_F32)) ||
      (rc = check_rows(a.initial_state, "initial_state", 2, a.width, false, M3_F32)) ||
      (rc = check_rows(a.carry, "carry", 3, a.width, false, M3_F32)) ||
      (!backward && ((rc = check_rows(a.out, "out", 3, a.width, live, a.dtype)) ||
                     (rc = check_rows(a.final_state, "final_state", 2, a.width, live, M3_F32))))) {
    return rc;
  }
  if (present(a.carry) && (a.carry.stride[1] != a.width ||
                           a.carry.stride[0] != static_cast<int64_t>(a.batch) * a.width)) {
    return fail(M3_EUNSUPPORTED, "m3_gated_scan: carry must be contiguous");
  }
  if (a.reset != nullptr && a.reset_stride < 0) {
    return fail(M3_EINVAL, "m3_gated_scan: negative reset stride");
  }
  return M3_OK;
}

GatedGeom geom(const m3_gated_scan_args& a) {
  GatedGeom g{};
  g.x = static_cast<const char*>(a.x.ptr);
  g.r = static_cast<const char*>(a.decay.ptr);
  g.g = static_cast<const char*>(a.gate.ptr);
  g.rate = static_cast<const float*>(a.rate.ptr);
  g.init = static_cast<const float*>(a.initial_state.ptr);
  g.lengths = a.lengths;
  g.reset = a.reset;
  g.y = static_cast<char*>(a.out.ptr);
  g.fin = static_cast<float*>(a.final_state.ptr);
  g.carry = static_cast<float*>(a.carry.ptr);
  g.x_b = a.x.stride[0], g.x_t = a.x.stride[1];
  g.r_b = a.decay.stride[0], g.r_t = a.decay.stride[1];
  g.g_b = a.gate.stride[0], g.g_t = a.gate.stride[1];
  g.y_b = a.out.stride[0], g.y_t = a.out.stride[1];
  g.init_b = a.initial_state.stride[0];
  g.fin_b = a.final_state.stride[0];
  g.reset_b = a.reset_stride;
  g.batch = a.batch, g.length = a.length, g.width = a.width;
  g.tiles = (a.length + kTile - 1) / kTile;
  return g;
}

// Whether rows of this tensor can be read two channels at a time.
bool paired(const m3_tensor& t, int dims) {
  if (t.ptr == nullptr) return true;
  if (reinterpret_cast<uintptr_t>(t.ptr) % (2 * elem_size(t.dtype)) != 0) return false;
  for (int i = 0; i + 1 < dims; ++i) {
    if (t.stride[i] % 2 != 0) return false;
  }
  return true;
}

// Workspace of a chained call: the ticket, the maps, and the states where no carry is asked for.
constexpr size_t kTicketBytes = 64;

size_t fwd_need(const m3_gated_scan_args& a) {
  if (a.length <= kTile || a.batch == 0 || a.width == 0) return 0;
  const size_t cells = static_cast<size_t>((a.length + kTile - 1) / kTile) * a.batch * a.width;
  return kTicketBytes + cells * (present(a.carry) ? 8 : 12);
}

template <typename T, bool GATE, int VEC>
int launch_tiles(const m3_gated_scan_args& a, const GatedGeom& g, hipStream_t stream) {
  const int cols = 64 * VEC;
  const int64_t count = static_cast<int64_t>((g.width + cols - 1) / cols) * g.batch * g.tiles;
  if (count > INT32_MAX) return fail(M3_EUNSUPPORTED, "m3_gated_scan: over 2^31 tiles");
  const dim3 grid(static_cast<unsigned>(count)), block(64 * kWaves);
  Chain ch{};
  if (g.tiles == 1) {
    hipLaunchKernelGGL((gated_tile_kernel<T, GATE, VEC, false>), grid, block, 0, stream, g, ch);
    return check_launch("m3_gated_scan");
  }
  const int64_t cells = static_cast<int64_t>(g.tiles) * g.batch * g.width;
  char* ws = static_cast<char*>(a.workspace);
  ch.ticket = reinterpret_cast<uint32_t*>(ws);
  ch.maps = reinterpret_cast<uint64_t*>(ws + kTicketBytes);
  ch.states = g.carry != nullptr ? reinterpret_cast<uint32_t*>(g.carry)
                                 : reinterpret_cast<uint32_t*>(ch.maps + cells);
  hipLaunchKernelGGL(gated_chain_kernel, dim3(static_cast<unsigned>((cells + 255) / 256)), dim3(256),
                     0, stream, ch, cells);
  const int rc = check_launch("m3_gated_scan");
  if (rc != M3_OK) return rc;
  hipLaunchKernelGGL((gated_tile_kernel<T, GATE, VEC, true>), grid, block, 0, stream, g, ch);
  return check_launch("m3_gated_scan");
}

template <typename T>
int launch_fwd(const m3_gated_scan_args& a, hipStream_t stream) {
  const GatedGeom g = geom(a);
  const bool gate = present(a.gate);
  const bool two = a.width % 2 == 0 && paired(a.x, 3) && paired(a.decay, 3) && paired(a.gate, 3) &&
                   paired(a.out, 3) && paired(a.carry, 1);
  if (a.length > 1) {
    if (gate) return two ? launch_tiles<T, true, 2>(a, g, stream) : launch_tiles<T, true, 1>(a, g, stream);
    return two ? launch_tiles<T, false, 2>(a, g, stream) : launch_tiles<T, false, 1>(a, g, stream);
  }
  const int64_t lanes = static_cast<int64_t>(a.batch) * (a.width / (two ? 2 : 1));
  const dim3 grid(static_cast<unsigned>((lanes + 255) / 256)), block(256);
  if (gate) {
    if (two) hipLaunchKernelGGL((gated_walk_kernel<T, true, 2>), grid, block, 0, stream, g);
    else hipLaunchKernelGGL((gated_walk_kernel<T, true, 1>), grid, block, 0, stream, g);
  } else {
    if (two) hipLaunchKernelGGL((gated_walk_kernel<T, false, 2>), grid, block, 0, stream, g);
    else hipLaunchKernelGGL((gated_walk_kernel<T, false, 1>), grid, block, 0, stream, g);
  }
  return check_launch("m3_gated_scan");
}

template <typename T>
int launch_bwd(const m3_gated_scan_bwd_args& a, hipStream_t stream) {
  GatedGeom g = geom(a.fwd);
  g.dy = static_cast<const char*>(a.dout.ptr);
  g.dfin = static_cast<const float*>(a.dfinal.ptr);
  g.dx = static_cast<char*>(a.dx.ptr);
  g.dr = static_cast<char*>(a.ddecay.ptr);
  g.dg = static_cast<char*>(a.dgate.ptr);
  g.drate = static_cast<float*>(a.drate.ptr);
  g.dinit = static_cast<float*>(a.dinitial.ptr);
  g.dy_b = a.dout.stride[0], g.dy_t = a.dout.stride[1];
  g.dx_b = a.dx.stride[0], g.dx_t = a.dx.stride[1];
  g.dr_b = a.ddecay.stride[0], g.dr_t = a.ddecay.stride[1];
  g.dg_b = a.dgate.stride[0], g.dg_t = a.dgate.stride[1];
  g.dfin_b = a.dfinal.stride[0];
  g.dinit_b = a.dinitial.stride[0];
  g.part = static_cast<float*>(a.fwd.workspace);
  g.scratch = g.part + static_cast<int64_t>(g.batch) * g.width;
  const int64_t lanes = static_cast<int64_t>(g.batch) * g.width;
  const dim3 grid(static_cast<unsigned>((lanes + 255) / 256)), block(256);
  if (present(a.fwd.gate)) {
    hipLaunchKernelGGL((gated_walk_bwd_kernel<T, true>), grid, block, 0, stream, g);
    const int rc = check_launch("m3_gated_scan_bwd");
    if (rc != M3_OK) return rc;
    hipLaunchKernelGGL(gated_rate_kernel, dim3((g.width + 255) / 256), block, 0, stream, g.part,
                       g.drate, g.batch, g.width);
  } else {
    hipLaunchKernelGGL((gated_walk_bwd_kernel<T, false>), grid, block, 0, stream, g);
  }
  return check_launch("m3_gated_scan_bwd");
}

bool nothing(const m3_gated_scan_args& a) { return a.batch == 0 || a.length == 0 || a.width == 0; }

size_t bwd_need(const m3_gated_scan_args& a) {
  return nothing(a) ? 0 : static_cast<size_t>(a.batch) * a.width * (1 + kTile) * 4;
}

int validate_bwd(const m3_gated_scan_bwd_args& a) {
  const m3_gated_scan_args& f = a.fwd;
  int rc;
  if ((rc = validate(f, true))) return rc;
  const bool live = !nothing(f), gate = present(f.gate);
  if ((rc = check_rows(a.dout, "dout", 3, f.width, live, f.dtype)) ||
      (rc = check_rows(a.dfinal, "dfinal", 2, f.width, false, M3_F32)) ||
      (rc = check_rows(a.dx, "dx", 3, f.width, live, f.dtype)) ||
      (rc = check_rows(a.ddecay, "ddecay", 3, f.width, live, f.dtype)) ||
      (rc = check_rows(a.dgate, "dgate", 3, f.width, live && gate, f.dtype)) ||
      (rc = check_rows(a.drate, "drate", 1, f.width, live && gate, M3_F32)) ||
      (rc = check_rows(a.dinitial, "dinitial", 2, f.width, false, M3_F32))) {
    return rc;
  }
  if (f.length > kTile && !present(f.carry) && live) {
    return fail(M3_EINVAL, "m3_gated_scan_bwd: more than %d tokens need the forward's carry", kTile);
  }
  return M3_OK;
}

}  // namespace
}  // namespace m3

extern "C" int m3_gated_scan_workspace_size(const m3_gated_scan_args* args, size_t* bytes) {
  using namespace m3;
  clear_error();
  if (args == nullptr || bytes == nullptr) return fail(M3_EINVAL, "m3_gated_scan: NULL args");
  const int rc = validate(*args, false);
  if (rc != M3_OK) return rc;
  *bytes = fwd_need(*args);
  return M3_OK;
}

extern "C" int m3_gated_scan(const m3_gated_scan_args* args, hipStream_t stream) {
  using namespace m3;
  clear_error();
  if (args == nullptr) return fail(M3_EINVAL, "m3_gated_scan: NULL args");
  const int rc = validate(*args, false);
  if (rc != M3_OK) return rc;
  if (nothing(*args)) return M3_OK;
  if (fwd_need(*args) > 0 && (args->workspace == nullptr || args->workspace_bytes < fwd_need(*args) ||
                              reinterpret_cast<uintptr_t>(args->workspace) % 8 != 0)) {
    return fail(M3_EWORKSPACE, "m3_gated_scan: workspace of %zu bytes, %zu needed (8-byte aligned)",
                args->workspace_bytes, fwd_need(*args));
  }
  switch (args->dtype) {
    case M3_F32: return launch_fwd<float>(*args, stream);
    case M3_BF16: return launch_fwd<__bf16>(*args, stream);
    default: return launch_fwd<_Float16>(*args, stream);
  }
}

extern "C" int m3_gated_scan_bwd_workspace_size(const m3_gated_scan_bwd_args* args, size_t* bytes) {
  using namespace m3;
  clear_error();
  if (args == nullptr || bytes == nullptr) return fail(M3_EINVAL, "m3_gated_scan_bwd: NULL args");
  const int rc = validate_bwd(*args);
  if (rc != M3_OK) return rc;
  *bytes = bwd_need(args->fwd);
  return M3_OK;
}

extern "C" int m3_gated_scan_bwd(const m3_gated_scan_bwd_args* args, hipStream_t stream) {
  using namespace m3;
  clear_error();
  if (args == nullptr) return fail(M3_EINVAL, "m3_gated_scan_bwd: NULL args");
  const int rc = validate_bwd(*args);
  if (rc != M3_OK) return rc;
  if (nothing(args->fwd)) return M3_OK;
  if (args->fwd.workspace == nullptr || args->fwd.workspace_bytes < bwd_need(args->fwd)) {
    return fail(M3_EWORKSPACE, "m3_gated_scan_bwd: workspace of %zu bytes, %zu needed",
                args->fwd.workspace_bytes, bwd_need(args->fwd));
  }
  switch (args->fwd.dtype) {
    case M3_F32: return launch_bwd<float>(*args, stream);
    case M3_BF16: return launch_bwd<__bf16>(*args, stream);
    default: return launch_bwd<_Float16>(*args, stream);
  }
}
