// m3_gated_scan and m3_gated_scan_bwd: a gated linear recurrence with one FP32 state per channel.
//
//   given form:  h_t = a_t h_{t-1} + x_t,               a_t = exp(decay_t)
//   gate form:   h_t = a_t h_{t-1} + s_t q_t x_t,       a_t = exp(-rate p_t), s_t = sqrt(1 - a_t^2)
// with p_t = sigmoid(decay_t), q_t = sigmoid(gate_t).
//
// What bounds it: memory, closely followed by the vector unit (33 instructions a token and channel forward
// in the gate form, 6 of them exponentials, reciprocals or roots at a quarter rate). So the inputs are read
// once and the transcendental work is done once.
//
// Forward, up to 16 tokens: one lane walks a channel's tokens (two channels where rows allow).
//
// Forward, more tokens: a workgroup takes a tile of 128 tokens x 128 channels (64 where rows are
// odd), which stays in registers. Each of its 8 waves runs 16 tokens from a zero state, which gives the
// span's map h -> A h + H; the maps of the waves before give a wave its entry state, and the tokens
// are run again from there with one fma each. Tiles of one row are chained through memory: a tile
// publishes its own map, then looks back for the nearest state that is already known. 16 tokens x 2
// channels a lane fill 116 of the 128 registers that leave two workgroups a CU; reading everything twice
// instead (maps first, outputs after) would move 14 bytes for every 8.
//
// Backward: tiles of 64 tokens (8 a wave: its inputs, factors and states fill the 128 registers), chained
// from the last, each with its states run again from the carry that the forward pass left, in
// place of 2 bytes a token and channel for the outputs, which are rounded.
//
// Measured in bf16, gate form (a large copy reaches 4.8 TB/s): 8 x 8192 x 2048 padded prompts 183 us
// (4.8 TB/s of what is read and written), one row of 65536 x 1536 179 us (4.5 TB/s), 1777 x 4096 20 us; forward
// and backward of 8 x 4096 x 2048 125 + 264 us (medians of a trace: 4.3 and 3.6 TB/s).
#include <hip/hip_runtime.h>

#include "m3_common.hpp"
#include "m3_host.hpp"

namespace m3 {
namespace {

constexpr int kTile = 128;             // tokens of a forward tile
constexpr int kLeap = M3_GATED_TILE;   // tokens between carried states; a backward tile
static_assert(kTile % kLeap == 0, "a forward tile leaves whole carries");
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
  float* part;                 // the tiles' shares of drate, [tiles, B, C]
  int64_t dy_b, dx_b, dr_b, dg_b, dfin_b, dinit_b;
  int64_t dy_t, dx_t, dr_t, dg_t;
};

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

// A wave's span of a tensor: its first token's address in a buffer descriptor, the token as a
// scalar offset and the channel as the lane's, so that no access needs a 64-bit address of its own.
// A lane past the width stores nowhere: past the extent.
template <typename T, int VEC>
struct Span {
  __amdgpu_buffer_rsrc_t rsrc;
  int stride;  // bytes between tokens
  unsigned off;  // the lane's channel, in bytes
  __device__ __forceinline__ Span(const char* base, int64_t first, int64_t token_stride, int c,
                                  bool live = true)
      : rsrc(__builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(base + first * static_cast<int64_t>(sizeof(T))), static_cast<short>(0),
            0x7fffffff, 0x00020000)),
        stride(static_cast<int>(token_stride) * static_cast<int>(sizeof(T))),
        off(live ? c * static_cast<unsigned>(sizeof(T)) : 0x80000000u) {}
  __device__ __forceinline__ void store(int i, const float (&v)[VEC]) const {
    typedef T tv __attribute__((ext_vector_type(VEC)));
    tv t;
#pragma unroll
    for (int e = 0; e < VEC; ++e) t[e] = from_f<T>(v[e]);
    if constexpr (sizeof(T) * VEC == 8) {
      typedef uint32_t u2 __attribute__((ext_vector_type(2)));
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, t), rsrc, off, i * stride, 0);
    } else if constexpr (sizeof(T) * VEC == 4) {
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, t), rsrc, off, i * stride, 0);
    } else {
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, t), rsrc, off, i * stride, 0);
    }
  }
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

// 1 - exp(u) for u <= 0: the series of -expm1 near 0, where the difference would lose its digits
// (at -0.125 the first term left out is 4e-8 of the sum, the difference's error 5e-7).
__device__ __forceinline__ float one_minus_exp(float u, float e) {
  const float series =
      -u * fmaf(u, fmaf(u, fmaf(u, fmaf(u, 1.f / 120.f, 1.f / 24.f), 1.f / 6.f), 0.5f), 1.f);
  return u > -0.125f ? series : 1.f - e;
}

__device__ __forceinline__ float sigmoid2(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -kLog2e));
}

// A sigmoid and its complement, both with all their digits: the complement is e / (1 + e), not a
// difference. WHOLE: from exp(-|x|), down to FP32's smallest values. Else (for 16-bit gradients, two instructions
// fewer) from e = exp(-x), whose infinity (x below -88) leaves open = 0 and shut = min(NaN, 1) = 1; a NaN
// x stays one in open, with which every use of shut is multiplied.
template <bool WHOLE>
struct Gate {
  float open, shut;
  __device__ __forceinline__ explicit Gate(float x) {
    if constexpr (WHOLE) {
      const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
      const float big = __builtin_amdgcn_rcpf(1.f + e), small = e * big;
      open = x < 0.f ? small : big;
      shut = x < 0.f ? big : small;
    } else {
      const float e = __builtin_amdgcn_exp2f(x * -kLog2e);
      open = __builtin_amdgcn_rcpf(1.f + e);
      shut = fminf(e * open, 1.f);
    }
  }
};

// The factor a of one token and channel, and s = sqrt(1 - a^2) (gate form).
template <bool GATE>
__device__ __forceinline__ void factor_root(float r, float rate, float& a, float& root) {
  if constexpr (!GATE) {
    a = __builtin_amdgcn_exp2f(r * kLog2e);
    root = 1.f;
  } else {
    const float p = sigmoid2(r);
    a = __builtin_amdgcn_exp2f(rate * -kLog2e * p);
    root = __builtin_amdgcn_sqrtf(one_minus_exp(rate * -2.f * p, a * a));
  }
}

// The factor and the input.
template <bool GATE>
__device__ __forceinline__ void factor_input(float x, float r, float g, float rate, float& a,
                                             float& b) {
  float root;
  factor_root<GATE>(r, rate, a, root);
  b = GATE ? root * sigmoid2(g) * x : x;
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
  uint32_t* tickets; // links started so far: of all chains (shared), or [chains]
  bool shared;
  uint64_t* maps;    // [tiles, B, C]
  uint32_t* states;  // [tiles, B, C]: the state that leaves a tile
};

constexpr int kWindow = 64;          // links looked back over
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

// The state that enters link s of a chain (s >= 1), for the channels at `at`; `step` elements lie
// between links. First the nearest link of the last kWindow whose states are published for all of the
// wave's channels, then the maps of the links after it, in order. A state is carried over a map by the
// very operation with which that link computes its own state, so the result does not depend on which
// link was found. A link that has its state at once publishes no map, so a map that is missing means
// another look at the states, never a wait for the map. Every wait ends: every link publishes its state once the
// links before it have; links are started in ticket order, and a running wave always gets to run. kSpins is
// there in case that is wrong. kStates and kMaps are read at once.
template <int VEC, int kStates, int kMaps>
__device__ __forceinline__ void look_back(const Chain& ch, int s, int64_t at, int64_t step,
                                          bool live, float (&v)[VEC]) {
  const int far = max(0, s - kWindow);
  for (int spin = 0; spin < kSpins; ++spin) {
    int found = -1;
    for (int near = s - 1; near >= far && found < 0; near -= kStates) {
      uint32_t st[kStates][VEC];
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        read_states<VEC>(ch.states + at + max(near - j, far) * step, st[j]);
      }
#pragma unroll
      for (int j = 0; j < kStates; ++j) {
        bool known = true;
#pragma unroll
        for (int e = 0; e < VEC; ++e) known = known && st[j][e] != kNotYet;
        if (found < 0 && near - j >= far && __all(known || !live)) {
          found = near - j;
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] = __uint_as_float(st[j][e]);
        }
      }
    }
    bool whole = found >= 0;
    for (int p = found + 1; p < s && whole; p += kMaps) {
      uint64_t map[kMaps][VEC];
#pragma unroll
      for (int j = 0; j < kMaps; ++j) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          map[j][e] = __hip_atomic_load(ch.maps + at + min(p + j, s - 1) * step + e, __ATOMIC_RELAXED,
                                        __HIP_MEMORY_SCOPE_AGENT);
        }
      }
      bool known = true;
#pragma unroll
      for (int j = 0; j < kMaps; ++j) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) known = known && (map[j][e] >> 32) != kNotYet;
      }
      whole = __all(known || !live);
#pragma unroll
      for (int j = 0; j < kMaps; ++j) {
        if (p + j < s) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            v[e] = fold(__uint_as_float(static_cast<uint32_t>(map[j][e] >> 32)),
                        __uint_as_float(static_cast<uint32_t>(map[j][e])), v[e]);
          }
        }
      }
    }
    if (whole) return;
    __builtin_amdgcn_s_sleep(2);
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) v[e] = __uint_as_float(0x7fc00000u);
}

__global__ __launch_bounds__(256) void gated_chain_kernel(Chain ch, int64_t cells, int chains) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < chains) ch.tickets[i] = 0;
  if (i >= cells) return;
  ch.maps[i] = ~uint64_t{0};
  ch.states[i] = kNotYet;
}

// The workgroup's chain and link: a chain's links in the order in which workgroups start, so that none
// waits for one that has not started. Both in scalar registers, where descriptors are made of them.
__device__ __forceinline__ int take_link(const Chain& ch, unsigned chains, unsigned& s_ticket,
                                         unsigned& chain) {
  const unsigned stride = ch.shared ? 0u : 1u;
  if (threadIdx.x == 0) s_ticket = atomicAdd(ch.tickets + stride * chain, 1u);
  __syncthreads();
  const unsigned id = __builtin_amdgcn_readfirstlane(s_ticket);
  chain = __builtin_amdgcn_readfirstlane(ch.shared ? id % chains : chain);
  return __builtin_amdgcn_readfirstlane(ch.shared ? id / chains : id);
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
  const unsigned groups = (g.width + kCols - 1) / kCols, chains = g.batch * groups;
  unsigned chain = blockIdx.x % chains;
  int s = 0;
  if constexpr (CHAIN) s = take_link(ch, chains, s_ticket, chain);
  const int b = chain / groups, c0 = (chain % groups) * kCols + lane * VEC;
  const bool live = c0 < g.width;
  const int c = min(c0, g.width - VEC);  // lanes past the width read its last channels
  const int t0 = s * kTile + w * kSpan;
  const int len = row_length(g, b), n = max(0, min(len - t0, kSpan));  // tokens of this wave
  const int64_t step = static_cast<int64_t>(g.batch) * g.width;
  const int64_t at = static_cast<int64_t>(b) * g.width + c;

  uint32_t early[VEC];
  if constexpr (CHAIN) {
    if (w == 0 && s > 0) read_states<VEC>(ch.states + at + (s - 1) * step, early);
  }
  // v: the state that enters the tile, then the wave; read before any wave can have written fin,
  // which may be the same memory
  float rate[VEC], v[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    rate[e] = GATE ? g.rate[c + e] : 0.f;
    if (!CHAIN || s == 0) v[e] = g.init != nullptr ? g.init[b * g.init_b + c + e] : 0.f;
  }
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
          look_back<VEC, 8, 8>(ch, s, at, step, live, v);
        }
      }
      float out[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        out[e] = fold(ta[e], th[e], v[e]);
        s_in[lane * VEC + e] = v[e];
      }
      if (live) {
        if (s < g.tiles - 1) write_states<VEC>(ch.states + at + s * step, out);
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
  const Span<T, VEC> y(g.y, b * g.y_b + t0 * g.y_t, g.y_t, c, live);
  if (n == kSpan && cut == 0) {
#pragma unroll
    for (int i = 0; i < kSpan; ++i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = fmaf(a[i][e], v[e], h[i][e]);
      y.store(i, v);
    }
  } else {
    const float zero[VEC] = {};
#pragma unroll
    for (int i = 0; i < kSpan; ++i) {
      if (i < n) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = fold(a[i][e], h[i][e], v[e]);
        y.store(i, v);
      } else if (i < rows) {
        y.store(i, zero);
      }
    }
  }
  // the final state is the last token's, as out has it before rounding
  if (live && (n > 0 ? t0 + n == len : len == 0 && s == 0 && w == 0)) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) g.fin[b * g.fin_b + c + e] = v[e];
  }
  constexpr int kPer = kLeap / kSpan;  // waves between carries
  const int leap = (s * kWaves + w) / kPer;
  if (g.carry != nullptr && live && w % kPer == kPer - 1 && leap * kLeap < g.length) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) g.carry[at + leap * step + e] = v[e];
  }
}

// ----------------------------------------------------------------------------- token walk

// kAtOnce: tokens whose loads are in flight together.
template <typename T, bool GATE, int VEC, int kAtOnce>
__global__ __launch_bounds__(256) void gated_walk_kernel(const GatedGeom g) {
  const int lanes = g.width / VEC;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int b = static_cast<int>(id / lanes), c = static_cast<int>(id % lanes) * VEC;
  if (b >= g.batch) return;
  const int len = row_length(g, b);
  float rate[VEC], h[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    rate[e] = GATE ? g.rate[c + e] : 0.f;
    h[e] = g.init != nullptr ? g.init[b * g.init_b + c + e] : 0.f;
  }
  typedef T tv __attribute__((ext_vector_type(VEC)));
  for (int t0 = 0; t0 < g.length; t0 += kAtOnce) {
    tv xv[kAtOnce], rv[kAtOnce], qv[kAtOnce];
    bool fresh[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t t = max(0, min(t0 + i, len - 1));
      xv[i] = *reinterpret_cast<const tv*>(reinterpret_cast<const T*>(g.x) + b * g.x_b + t * g.x_t + c);
      rv[i] = *reinterpret_cast<const tv*>(reinterpret_cast<const T*>(g.r) + b * g.r_b + t * g.r_t + c);
      if constexpr (GATE) {
        qv[i] = *reinterpret_cast<const tv*>(reinterpret_cast<const T*>(g.g) + b * g.g_b + t * g.g_t + c);
      }
      fresh[i] = g.reset != nullptr && g.reset[b * g.reset_b + t] != 0;
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (t0 + i < g.length) {
        float y[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float a, in;
          factor_input<GATE>(to_f(xv[i][e]), to_f(rv[i][e]), GATE ? to_f(qv[i][e]) : 0.f, rate[e], a, in);
          const float next = fresh[i] ? in : fmaf(a, h[e], in);
          h[e] = t0 + i < len ? next : h[e];
          y[e] = t0 + i < len ? h[e] : 0.f;
        }
        store_vec<T, VEC>(g.y, b * g.y_b + (t0 + i) * g.y_t + c, y);
      }
    }
  }
  if (g.carry != nullptr) {  // at most one tile
#pragma unroll
    for (int e = 0; e < VEC; ++e) g.carry[static_cast<int64_t>(b) * g.width + c + e] = h[e];
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) g.fin[b * g.fin_b + c + e] = h[e];
}

// ----------------------------------------------------------------------------- backward

constexpr int kBack = kLeap / kWaves;  // a wave's tokens

// v = 0 where bit i of `cut`, a scalar, is set: a branch (the asm keeps it one), for it seldom is.
template <int VEC>
__device__ __forceinline__ void drop_at(uint64_t cut, int i, float (&v)[VEC]) {
  if (cut >> i & 1) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      v[e] = 0.f;
      asm volatile("" : "+v"(v[e]));
    }
  }
}

// A tile of kLeap tokens x 64 VEC channels. The states before its tokens are run again from the
// carry the forward pass left, as a wave's map behind those of the waves before; the gradients
// e_{t-1} = a_t (dy_t + e_t) run the other way, their maps joined from the last wave to the first
// and from tile to tile in a chain that begins at the last. Both kinds of map are formed from one read
// of the inputs, kept as they came; the factor and s are kept too, the sigmoids formed again.
template <typename T, bool GATE, int VEC, bool CHAIN>
__global__ __launch_bounds__(64 * kWaves, 4) void gated_back_kernel(const GatedGeom g,
                                                                    const Chain ch) {
  constexpr int kCols = 64 * VEC;
  __shared__ float s_a[kWaves][kCols], s_h[kWaves][kCols], s_e[kWaves][kCols], s_in[kCols];
  __shared__ unsigned s_ticket;
  typedef T tv __attribute__((ext_vector_type(VEC)));
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned groups = (g.width + kCols - 1) / kCols, chains = g.batch * groups;
  unsigned chain = blockIdx.x % chains;
  int link = 0;
  if constexpr (CHAIN) link = take_link(ch, chains, s_ticket, chain);
  const int s = g.tiles - 1 - link;
  const int b = chain / groups, c0 = (chain % groups) * kCols + lane * VEC;
  const bool live = c0 < g.width;
  const int c = min(c0, g.width - VEC);
  const int t0 = s * kLeap + w * kBack;
  const int n = max(0, min(row_length(g, b) - t0, kBack));
  const int64_t step = static_cast<int64_t>(g.batch) * g.width;
  const int64_t at = static_cast<int64_t>(b) * g.width + c;

  uint32_t early[VEC];
  if constexpr (CHAIN) {
    if (w == 0 && link > 0) read_states<VEC>(ch.states + at + (link - 1) * step, early);
  }
  float rate[VEC], v[VEC];  // v: the state before the wave's tokens
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    rate[e] = GATE ? g.rate[c + e] : 0.f;
    v[e] = s > 0 ? g.carry[at + (s - 1) * step + e]
                 : (g.init != nullptr ? g.init[b * g.init_b + c + e] : 0.f);
  }
  uint64_t cut = 0;
  if (g.reset != nullptr) {
    cut = __ballot(lane < n && g.reset[b * g.reset_b + t0 + min(lane, max(n - 1, 0))] != 0);
  }

  tv xv[kBack], rv[kBack], qv[kBack], dv[kBack];
  float a[kBack][VEC], root[kBack][VEC], h[kBack][VEC];
  float span_a[VEC], span_h[VEC], span_e[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) span_a[e] = 1.f, span_h[e] = 0.f, span_e[e] = 0.f;
  if (n > 0) {
    const Span<T, VEC> x(g.x, b * g.x_b + t0 * g.x_t, g.x_t, c);
    const Span<T, VEC> r(g.r, b * g.r_b + t0 * g.r_t, g.r_t, c);
    const Span<T, VEC> q(GATE ? g.g : g.x, b * g.g_b + t0 * g.g_t, g.g_t, c);
    const Span<T, VEC> d(g.dy, b * g.dy_b + t0 * g.dy_t, g.dy_t, c);
#pragma unroll
    for (int i = 0; i < kBack; ++i) {
      const int t = min(i, n - 1);
      xv[i] = __builtin_bit_cast(tv, x.load(t));
      rv[i] = __builtin_bit_cast(tv, r.load(t));
      if constexpr (GATE) qv[i] = __builtin_bit_cast(tv, q.load(t));
      dv[i] = __builtin_bit_cast(tv, d.load(t));
    }
#pragma unroll
    for (int i = 0; i < kBack; ++i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        factor_root<GATE>(to_f(rv[i][e]), rate[e], a[i][e], root[i][e]);
        h[i][e] = to_f(xv[i][e]);
        if constexpr (GATE) h[i][e] *= root[i][e] * sigmoid2(to_f(qv[i][e]));
      }
    }
    if (n < kBack) {
#pragma unroll
      for (int i = 0; i < kBack; ++i) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          a[i][e] = i >= n ? 1.f : a[i][e];
          h[i][e] = i >= n ? 0.f : h[i][e];
          if (i >= n) dv[i][e] = from_f<T>(0.f);
        }
      }
    }
    if (cut == 0) {
#pragma unroll
      for (int i = 0; i < kBack; ++i) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          span_h[e] = fmaf(a[i][e], span_h[e], h[i][e]);
          span_a[e] *= a[i][e];
          const int k = kBack - 1 - i;
          span_e[e] = a[k][e] * (span_e[e] + to_f(dv[k][e]));
        }
      }
    } else {
      // a given decay at a reset token carries nothing, whatever it is (0 times infinity is NaN)
      if constexpr (!GATE) {
#pragma unroll
        for (int i = 0; i < kBack; ++i) drop_at(cut, i, a[i]);
      }
#pragma unroll
      for (int i = 0; i < kBack; ++i) {
        const int k = kBack - 1 - i;
        const bool fresh = (cut >> i) & 1, last = (cut >> k) & 1;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          span_h[e] = fresh ? h[i][e] : fmaf(a[i][e], span_h[e], h[i][e]);
          span_a[e] = -1.f;
          span_e[e] = last ? 0.f : a[k][e] * (span_e[e] + to_f(dv[k][e]));
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    s_a[w][lane * VEC + e] = span_a[e];
    s_h[w][lane * VEC + e] = span_h[e];
    s_e[w][lane * VEC + e] = span_e[e];
  }
  __syncthreads();
  float u[VEC];  // the gradient that enters the tile from behind, then the wave
  if (!CHAIN || link == 0) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) u[e] = g.dfin != nullptr ? g.dfin[b * g.dfin_b + c + e] : 0.f;
  }
  if (w == 0) {
    float ta[VEC], te[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      ta[e] = 1.f, te[e] = 0.f;
#pragma unroll
      for (int k = kWaves - 1; k >= 0; --k) {
        const float ka = s_a[k][lane * VEC + e];
        te[e] = fold(ka, s_e[k][lane * VEC + e], te[e]);
        ta[e] = join(ta[e], ka);
      }
    }
    if (CHAIN && link > 0) {
      bool known = true;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        known = known && early[e] != kNotYet;
        u[e] = __uint_as_float(early[e]);
      }
      if (!__all(known || !live)) {
        if (live) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const uint64_t m = static_cast<uint64_t>(word(ta[e])) << 32 | __float_as_uint(te[e]);
            __hip_atomic_store(ch.maps + at + link * step + e, m, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
          }
        }
        look_back<VEC, 4, 4>(ch, link, at, step, live, u);
      }
    }
    float out[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      out[e] = fold(ta[e], te[e], u[e]);
      if constexpr (CHAIN) s_in[lane * VEC + e] = u[e];
    }
    if (live) {
      if constexpr (CHAIN) {
        if (s > 0) write_states<VEC>(ch.states + at + link * step, out);
      }
      if (s == 0 && g.dinit != nullptr) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) g.dinit[b * g.dinit_b + c + e] = out[e];
      }
    }
  }
  // meanwhile the states before each token
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    if (k < w) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[e] = fold(s_a[k][lane * VEC + e], s_h[k][lane * VEC + e], v[e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kBack; ++i) {
    drop_at(cut, i, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float before = v[e];
      v[e] = fmaf(a[i][e], before, h[i][e]);
      h[i][e] = before;
    }
  }
  if constexpr (CHAIN) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) u[e] = s_in[lane * VEC + e];
  }
#pragma unroll
  for (int k = kWaves - 1; k >= 0; --k) {
    if (k > w) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        u[e] = fold(s_a[k][lane * VEC + e], s_e[k][lane * VEC + e], u[e]);
      }
    }
  }
  float sum[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
  const int rows = max(0, min(g.length - t0, kBack));
  const Span<T, VEC> sx(g.dx, b * g.dx_b + t0 * g.dx_t, g.dx_t, c, live);
  const Span<T, VEC> sr(g.dr, b * g.dr_b + t0 * g.dr_t, g.dr_t, c, live);
  const Span<T, VEC> sg(GATE ? g.dg : g.dx, b * g.dg_b + t0 * g.dg_t, g.dg_t, c, live);
#pragma unroll
  for (int k = 0; k < kBack; ++k) {
    const int i = kBack - 1 - k;
    float dx[VEC], dr[VEC], dg[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) dx[e] = 0.f, dr[e] = 0.f, dg[e] = 0.f;
    if (i < n) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = to_f(dv[i][e]) + u[e];
        if constexpr (GATE) {
          const float x = to_f(xv[i][e]);
          const Gate<sizeof(T) == 4> p(to_f(rv[i][e])), q(to_f(qv[i][e]));
          // a h - q x a^2 / s, with 1 / s = 0 where s is (its factor rate p vanishes faster)
          const float inv = root[i][e] == 0.f ? 0.f : __builtin_amdgcn_rcpf(root[i][e]);
          const float dlog = d * a[i][e] * (h[i][e] - q.open * x * (a[i][e] * inv));
          dx[e] = d * (root[i][e] * q.open);
          dg[e] = dx[e] * x * q.shut;
          dr[e] = -rate[e] * (p.open * p.shut) * dlog;
          sum[e] = fmaf(-p.open, dlog, sum[e]);
        } else {
          dx[e] = d;
          dr[e] = d * (a[i][e] * h[i][e]);
        }
        u[e] = a[i][e] * d;
      }
      drop_at(cut, i, u);
    }
    if (i < rows) {
      sx.store(i, dx);
      sr.store(i, dr);
      if constexpr (GATE) sg.store(i, dg);
    }
  }
  if constexpr (GATE) {
    __syncthreads();  // every wave is done with the maps
#pragma unroll
    for (int e = 0; e < VEC; ++e) s_a[w][lane * VEC + e] = sum[e];
    __syncthreads();
    if (w == 0 && live) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float total = 0.f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) total += s_a[k][lane * VEC + e];
        g.part[at + s * step + e] = total;
      }
    }
  }
}

// drate[c] = the sum of the tiles' shares, in 64 bits (a sum over all tokens that cancels), in a
// fixed order: 16 waves take every 16th row each.
__global__ __launch_bounds__(1024) void gated_rate_kernel(const float* part, float* drate,
                                                          int64_t rows, int width) {
  __shared__ double s_sum[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, at = min(c, width - 1);
  double sum = 0.0;
#pragma unroll 8
  for (int64_t i = w; i < rows; i += 16) sum += part[i * width + at];
  s_sum[w][lane] = sum;
  __syncthreads();
  if (w == 0 && c < width) {
#pragma unroll
    for (int k = 1; k < 16; ++k) sum += s_sum[k][lane];
    drate[c] = static_cast<float>(sum);
  }
}

// ----------------------------------------------------------------------------- host

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
  // more are over 2^23 tiles, and tiles and tokens are counted in 32 bits
  if (a.length > (1 << 30)) return fail(M3_EUNSUPPORTED, "m3_gated_scan: length above 2^30");
  if (a.width > (1 << 27)) return fail(M3_EUNSUPPORTED, "m3_gated_scan: width above 2^27");
  // the lanes of a launch are counted in 32 bits
  if (static_cast<int64_t>(a.batch) * a.width >= INT32_MAX / 2) {
    return fail(M3_EUNSUPPORTED, "m3_gated_scan: batch * width %lld is above 2^30",
                static_cast<long long>(a.batch) * a.width);
  }
  const bool live = a.batch > 0 && a.length > 0 && a.width > 0;
  int rc;
  if ((rc = check_tensor(a.x, "x", 3, a.width, live, a.dtype)) ||
      (rc = check_tensor(a.decay, "decay", 3, a.width, live, a.dtype)) ||
      (rc = check_tensor(a.gate, "gate", 3, a.width, false, a.dtype)) ||
      (rc = check_tensor(a.rate, "rate", 1, a.width, false, M3_F32)) ||
      (rc = check_tensor(a.initial_state, "initial_state", 2, a.width, false, M3_F32)) ||
      (rc = check_tensor(a.carry, "carry", 3, a.width, false, M3_F32)) ||
      (!backward && ((rc = check_tensor(a.out, "out", 3, a.width, live, a.dtype)) ||
                     (rc = check_tensor(a.final_state, "final_state", 2, a.width, live, M3_F32))))) {
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

// Up to here one lane walks a row's tokens: a tile would leave most of its waves without one.
constexpr int kWalk = 16;
static_assert(kWalk <= kLeap, "a walk leaves one carry");

// Workspace of a chained call: the tickets, the maps and the states.
int chains_of(int batch, int width) { return batch * ((width + 63) / 64); }  // at one channel a lane
size_t ticket_bytes(int batch, int width) {
  return (static_cast<size_t>(chains_of(batch, width)) * 4 + 63) / 64 * 64;
}

size_t fwd_need(const m3_gated_scan_args& a) {
  if (a.length <= kTile || a.batch == 0 || a.width == 0) return 0;
  const size_t cells = static_cast<size_t>((a.length + kTile - 1) / kTile) * a.batch * a.width;
  return ticket_bytes(a.batch, a.width) + cells * 12;
}

// One counter for all chains keeps a row's tiles together in time, which pays where they pass
// through the GPU many times over (8 x 8192 x 2048: 190 against 208 us); its increments take turns, which
// fewer tiles wait for (1777 x 4096: 25 against 23 us). The two meet at about 2,000 tiles.
constexpr int64_t kShared = 2048;

Chain chain(void* workspace, int64_t cells, size_t tickets, int64_t links) {
  char* ws = static_cast<char*>(workspace);
  uint64_t* maps = reinterpret_cast<uint64_t*>(ws + tickets);
  return Chain{reinterpret_cast<uint32_t*>(ws), links > kShared, maps,
               reinterpret_cast<uint32_t*>(maps + cells)};
}

constexpr int64_t kMostTiles = (int64_t{1} << 32) / (64 * kWaves) - 1;  // a grid has below 2^32 threads

template <typename T, bool GATE, int VEC>
int launch_tiles(const m3_gated_scan_args& a, const GatedGeom& g, hipStream_t stream) {
  const int cols = 64 * VEC;
  const int64_t count = static_cast<int64_t>((g.width + cols - 1) / cols) * g.batch * g.tiles;
  if (count > kMostTiles) return fail(M3_EUNSUPPORTED, "m3_gated_scan: over 2^23 tiles");
  const dim3 grid(static_cast<unsigned>(count)), block(64 * kWaves);
  if (g.tiles == 1) {
    hipLaunchKernelGGL((gated_tile_kernel<T, GATE, VEC, false>), grid, block, 0, stream, g,
                       Chain{});
    return check_launch("m3_gated_scan");
  }
  const int64_t cells = static_cast<int64_t>(g.tiles) * g.batch * g.width;
  const Chain ch = chain(a.workspace, cells, ticket_bytes(g.batch, g.width), count);
  hipLaunchKernelGGL(gated_chain_kernel, dim3(static_cast<unsigned>((cells + 255) / 256)), dim3(256),
                     0, stream, ch, cells, chains_of(g.batch, g.width));
  const int rc = check_launch("m3_gated_scan");
  if (rc != M3_OK) return rc;
  hipLaunchKernelGGL((gated_tile_kernel<T, GATE, VEC, true>), grid, block, 0, stream, g, ch);
  return check_launch("m3_gated_scan");
}

template <typename T, bool GATE, int VEC>
int launch_walk(const GatedGeom& g, hipStream_t stream) {
  const int64_t lanes = static_cast<int64_t>(g.batch) * (g.width / VEC);
  const dim3 grid(static_cast<unsigned>((lanes + 255) / 256)), block(256);
  if (g.length == 1) {
    hipLaunchKernelGGL((gated_walk_kernel<T, GATE, VEC, 1>), grid, block, 0, stream, g);
  } else {
    hipLaunchKernelGGL((gated_walk_kernel<T, GATE, VEC, 8>), grid, block, 0, stream, g);
  }
  return check_launch("m3_gated_scan");
}

template <typename T>
int launch_fwd(const m3_gated_scan_args& a, hipStream_t stream) {
  const GatedGeom g = geom(a);
  const bool gate = present(a.gate);
  const bool two = a.width % 2 == 0 && paired(a.x, 3) && paired(a.decay, 3) && paired(a.gate, 3) &&
                   paired(a.out, 3);
  if (a.length > kWalk) {
    if (gate) return two ? launch_tiles<T, true, 2>(a, g, stream) : launch_tiles<T, true, 1>(a, g, stream);
    return two ? launch_tiles<T, false, 2>(a, g, stream) : launch_tiles<T, false, 1>(a, g, stream);
  }
  if (gate) return two ? launch_walk<T, true, 2>(g, stream) : launch_walk<T, true, 1>(g, stream);
  return two ? launch_walk<T, false, 2>(g, stream) : launch_walk<T, false, 1>(g, stream);
}

template <typename T, bool GATE, int VEC>
int launch_back(const m3_gated_scan_bwd_args& a, GatedGeom& g, hipStream_t stream) {
  const int cols = 64 * VEC;
  const int64_t count = static_cast<int64_t>((g.width + cols - 1) / cols) * g.batch * g.tiles;
  if (count > kMostTiles) return fail(M3_EUNSUPPORTED, "m3_gated_scan_bwd: over 2^23 tiles");
  const dim3 grid(static_cast<unsigned>(count)), block(64 * kWaves);
  const int64_t cells = static_cast<int64_t>(g.tiles) * g.batch * g.width;
  const Chain ch = chain(a.fwd.workspace, cells, ticket_bytes(g.batch, g.width), count);
  g.part = reinterpret_cast<float*>(ch.states + cells);
  int rc;
  if (g.tiles == 1) {
    hipLaunchKernelGGL((gated_back_kernel<T, GATE, VEC, false>), grid, block, 0, stream, g, ch);
  } else {
    hipLaunchKernelGGL(gated_chain_kernel, dim3(static_cast<unsigned>((cells + 255) / 256)),
                       dim3(256), 0, stream, ch, cells, chains_of(g.batch, g.width));
    if ((rc = check_launch("m3_gated_scan_bwd"))) return rc;
    hipLaunchKernelGGL((gated_back_kernel<T, GATE, VEC, true>), grid, block, 0, stream, g, ch);
  }
  if ((rc = check_launch("m3_gated_scan_bwd")) || !GATE) return rc;
  hipLaunchKernelGGL(gated_rate_kernel, dim3((g.width + 63) / 64), dim3(1024), 0, stream, g.part,
                     g.drate, static_cast<int64_t>(g.tiles) * g.batch, g.width);
  return check_launch("m3_gated_scan_bwd");
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
  g.tiles = (g.length + kLeap - 1) / kLeap;
  // 16-bit channels in pairs; FP32 ones singly, whose rows a wave reads as widely
  if constexpr (sizeof(T) == 2) {
    if (g.width % 2 == 0 && paired(a.fwd.x, 3) && paired(a.fwd.decay, 3) && paired(a.fwd.gate, 3) &&
        paired(a.dout, 3) && paired(a.dx, 3) && paired(a.ddecay, 3) && paired(a.dgate, 3)) {
      return present(a.fwd.gate) ? launch_back<T, true, 2>(a, g, stream)
                                 : launch_back<T, false, 2>(a, g, stream);
    }
  }
  return present(a.fwd.gate) ? launch_back<T, true, 1>(a, g, stream)
                             : launch_back<T, false, 1>(a, g, stream);
}

bool nothing(const m3_gated_scan_args& a) { return a.batch == 0 || a.length == 0 || a.width == 0; }

size_t bwd_need(const m3_gated_scan_args& a) {
  if (nothing(a)) return 0;
  const size_t cells = static_cast<size_t>((a.length + kLeap - 1) / kLeap) * a.batch * a.width;
  return ticket_bytes(a.batch, a.width) + cells * 16;  // maps, states, shares of drate
}

int validate_bwd(const m3_gated_scan_bwd_args& a) {
  const m3_gated_scan_args& f = a.fwd;
  int rc;
  if ((rc = validate(f, true))) return rc;
  const bool live = !nothing(f), gate = present(f.gate);
  if ((rc = check_tensor(a.dout, "dout", 3, f.width, live, f.dtype)) ||
      (rc = check_tensor(a.dfinal, "dfinal", 2, f.width, false, M3_F32)) ||
      (rc = check_tensor(a.dx, "dx", 3, f.width, live, f.dtype)) ||
      (rc = check_tensor(a.ddecay, "ddecay", 3, f.width, live, f.dtype)) ||
      (rc = check_tensor(a.dgate, "dgate", 3, f.width, live && gate, f.dtype)) ||
      (rc = check_tensor(a.drate, "drate", 1, f.width, live && gate, M3_F32)) ||
      (rc = check_tensor(a.dinitial, "dinitial", 2, f.width, false, M3_F32))) {
    return rc;
  }
  for (const m3_tensor* t : {&a.dout, &a.dx, &a.ddecay, &a.dgate}) {
    if (t->ptr != nullptr && t->stride[1] > (1 << 24)) {
      return fail(M3_EUNSUPPORTED, "m3_gated_scan_bwd: tokens over 2^24 elements apart");
    }
  }
  if (f.length > kLeap && !present(f.carry) && live) {
    return fail(M3_EINVAL, "m3_gated_scan_bwd: more than %d tokens need the forward's carry", kLeap);
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
  if (args->fwd.workspace == nullptr || args->fwd.workspace_bytes < bwd_need(args->fwd) ||
      reinterpret_cast<uintptr_t>(args->fwd.workspace) % 8 != 0) {
    return fail(M3_EWORKSPACE, "m3_gated_scan_bwd: workspace of %zu bytes, %zu needed (8-byte aligned)",
                args->fwd.workspace_bytes, bwd_need(args->fwd));
  }
  switch (args->fwd.dtype) {
    case M3_F32: return launch_bwd<float>(*args, stream);
    case M3_BF16: return launch_bwd<__bf16>(*args, stream);
    default: return launch_bwd<_Float16>(*args, stream);
  }
}
