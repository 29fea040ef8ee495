// m3_linear4: out[M, N] = x'[M, K] * W[N, K]^T (+ residual), W = (q - z) * scale in 4-bit codes with a
// scale (and a zero) for every group of 32, 64 or 128 columns: the decode step's projections.
//
// A code goes into the mantissa of a 16-bit 16.0, which makes 16 + q exactly (a shift and an and-or
// for two codes), and that is the matrix operand. With A = sum (16 + q) x over a group and X = sum x,
// the group's share is scale * A - scale * (16 + z) * X: the scale and the zero meet FP32 sums, not the
// operands. X comes from one more matrix product, with ones.
//
// linear4_kernel (up to 16 rows of x; up to 32 a workgroup where there are few weight rows): a workgroup
// takes TN tiles of 16 weight rows and MT blocks of 16 operand rows: rows of x, or with the norm two for
// each, for its product with the norm's weight has more bits than one holds. Its waves take every WAVES-th tile of 128
// columns each, so no two read the same operand and the K loop has no barrier; their sums meet in
// LDS. A wave's next codes and x are on their way in registers while it multiplies; x goes through
// an LDS region of the wave's own, where it is normed, and comes back as the operand's columns. Bound by
// the weight's stream where it is long, else by the launch and one latency of memory: in graphs with
// cold weights 28672 x 8192 at 1 row 27.1 us (4.5 TB/s; a large copy reaches 4.8), 8672 x 2048 at 1 row 4.9
// us, 6.7 with the norm, 2048 x 4096 at 16 rows 5.5 us (512 x 512: 2.4 us). A second row for the norm costs nothing
// where matrix rows are idle (8672 x 2048 at 4 rows 6.9 us either way), else its instructions: 16 rows 10.6 us
// with whole products, 9.0 with rounded ones.
//
// linear4_wide_kernel (more rows of both): below.
#include <hip/hip_runtime.h>

#include "m3_common.hpp"
#include "m3_host.hpp"

namespace m3 {
namespace {

constexpr int kMaxRows = 256;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Two codes of a word at a time: nibbles j and j + 4 as the halves of a register.
template <typename T> struct Code;
template <> struct Code<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kOne = 0x41804180u, kMask = 0x00780078u;  // 16.0 twice
  static constexpr uint32_t kUnit = 0x3f803f80u;  // 1.0 twice
  static constexpr int kUp = 3;  // where a code's low bit is 1 of 16.0's 7 bits of mantissa
  static __device__ __forceinline__ f4 mma(v8 a, v8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Code<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kOne = 0x4c004c00u, kMask = 0x03c003c0u;
  static constexpr uint32_t kUnit = 0x3c003c00u;
  static constexpr int kUp = 6;
  static __device__ __forceinline__ f4 mma(v8 a, v8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// `sixteens` is Code<T>::kOne in a vector register (and-or takes one scalar, which the mask is).
template <typename T>
__device__ __forceinline__ typename Code<T>::v8 expand(uint32_t w, uint32_t sixteens) {
  u32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    constexpr int up = Code<T>::kUp;
    const uint32_t at = 4 * j > up ? w >> (4 * j - up) : w << (up - 4 * j);
    v[j] = (at & Code<T>::kMask) | sixteens;
  }
  return __builtin_bit_cast(typename Code<T>::v8, v);
}

struct Lin4Geom {
  const char* codes;
  const char* scales;
  const char* zeros;   // or null
  const char* x;       // [M, K]
  const char* nw;      // [K] or null
  const void* res;     // or null
  void* out;
  int64_t x_ld, r_ld, o_ld;
  int m, n, k, tk;     // tk: tiles of 128 columns
  int tiles;           // of 16 weight rows
  bool four;           // rows of out are 8-byte aligned
  float eps;
};

// Four scales of a group (16-bit, in two registers).
template <typename S>
__device__ __forceinline__ f4 scales4(u32x2 v) {
  f4 s;
  if constexpr (__is_same(S, __bf16)) {
    s = f4{__uint_as_float(v[0] << 16), __uint_as_float(v[0] & 0xffff0000u),
           __uint_as_float(v[1] << 16), __uint_as_float(v[1] & 0xffff0000u)};
  } else {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const h4 h = __builtin_bit_cast(h4, v);
    s = f4{static_cast<float>(h[0]), static_cast<float>(h[1]), static_cast<float>(h[2]),
           static_cast<float>(h[3])};
  }
  return s;
}

// -scale (16 + z) of four zeros in bytes.
__device__ __forceinline__ f4 shifts4(uint32_t z, f4 scale) {
  f4 v;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    v[r] = -(16.f + static_cast<float>((z >> (8 * r)) & 0xffu)) * scale[r];
  }
  return v;
}

// An offset past every extent, also with another added: the load gives 0. x spans less than 2^29 bytes, so
// 48 rows more (of over 16) add less than 3 x 2^29 and do not come round to 0. Offsets go into a load whole, none as the scalar offset, which the range check does not add.
constexpr unsigned kNowhere = 0x7fff0000u;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc4(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0),
                                           static_cast<int>(bytes), 0x00020000);
}

// Eight x values times the norm's weights, as a bf16 value and the bf16 remainder; the squares go to sq.
// The FP32 products are whole (8 + 8 or 11 + 11 bits). Two bf16 values hold those of bf16 rows whole and
// 16 or more bits of those of f16 rows (2^-17 of a term, against 2^-11 of the rounded result), over FP32's range:
// 1 / rms, which brings a row back into f16's, comes last.
template <typename T>
__device__ __forceinline__ void normed(u32x4 x, u32x4 weight, float& sq, u32x4& high, u32x4& low) {
  using V8 = typename Code<T>::v8;
  typename Code<__bf16>::v8 h, l;
  const V8 b = __builtin_bit_cast(V8, x), n = __builtin_bit_cast(V8, weight);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float xf = static_cast<float>(b[e]), p = xf * static_cast<float>(n[e]);
    sq = fmaf(xf, xf, sq);
    h[e] = static_cast<__bf16>(p);
    l[e] = static_cast<__bf16>(p - static_cast<float>(h[e]));
  }
  high = __builtin_bit_cast(u32x4, h);
  low = __builtin_bit_cast(u32x4, l);
}

// What feeds the matrix instructions: x itself, or with the norm two bf16 rows for each row of x, the
// remainders in the second half of a workgroup's rows. Their two sums are added at the end.
template <typename T, bool NORM> struct Operand { using type = T; };
template <typename T> struct Operand<T, true> { using type = __bf16; };

// Between a wave's writes of its own LDS region and its lanes' reads of one another's, and back: LDS
// operations of one wave complete in order, so only the compiler has to keep them so.
__device__ __forceinline__ void stage_turn() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A barrier for what lies in LDS: global loads stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

constexpr int kRowBytes = 256;  // an x row of a tile in LDS; chunk c of 16 bytes lies at c ^ (row & 15)

template <typename T, typename S, int GPT, int MT, int TN, int WAVES, bool NORM>
__global__ __launch_bounds__(64 * WAVES) void linear4_kernel(const Lin4Geom g) {
  using O = typename Operand<T, NORM>::type;
  using C = Code<O>;
  using V8 = typename C::v8;
  constexpr int kRows = 16 * MT / (NORM ? 2 : 1), kLoads = kRows / 4;  // rows of x
  constexpr int kStage = MT * 16 * kRowBytes, kSums = MT * TN * 256;
  constexpr int kLds = WAVES * (kStage > 4 * kSums ? kStage : 4 * kSums);
  __shared__ __attribute__((aligned(16))) char lds[kLds];
  __shared__ float s_sq[NORM ? WAVES : 1][kRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int tn = blockIdx.x * TN, m0 = blockIdx.y * kRows;
  char* const stage = lds + w * kStage;

  // what a tile of columns needs: codes, scales and zeros of TN tile rows, x rows 4 j + lg.
  u32x4 code[TN], xv[kLoads], nv;
  u32x2 sc[TN][GPT];
  uint32_t zr[TN][GPT];
  // reads past an extent give 0: tile rows past the last, x rows past M
  const int64_t tile0 = static_cast<int64_t>(tn) * g.tk, left = min(g.tiles - tn, TN) * g.tk;
  const __amdgpu_buffer_rsrc_t rc = rsrc4(g.codes + tile0 * 1024, left * 1024);
  const __amdgpu_buffer_rsrc_t rs = rsrc4(g.scales + tile0 * (GPT * 32), left * (GPT * 32));
  const bool has_zeros = g.zeros != nullptr;  // else 0 is read, and 8 meant
  const __amdgpu_buffer_rsrc_t rz = rsrc4(has_zeros ? g.zeros + tile0 * (GPT * 16) : g.codes,
                                          has_zeros ? left * (GPT * 16) : 0);
  const uint32_t eights = has_zeros ? 0u : 0x08080808u;
  const __amdgpu_buffer_rsrc_t rx = rsrc4(g.x, ((g.m - 1) * g.x_ld + g.k) * 2);
  const __amdgpu_buffer_rsrc_t rn = rsrc4(g.nw, NORM ? 2 * g.k : 0);
  const unsigned x_row = static_cast<unsigned>(g.x_ld) * 2;
  auto fetch = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int tile = j * g.tk + t;
      // non-temporal (aux bit 1): the codes are read once a call
      code[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                              rc, 1024 * tile + 16 * lane, 0, 2));
#pragma unroll
      for (int gi = 0; gi < GPT; ++gi) {
        const int at = (tile * GPT + gi) * 16;
        sc[j][gi] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(
                                                  rs, 2 * at + 8 * lg, 0, 0));
        zr[j][gi] = __builtin_amdgcn_raw_buffer_load_b32(rz, at + 4 * lg, 0, 0);
      }
    }
    const int k = 128 * t + 8 * l16;
    const unsigned at = k < g.k ? (m0 + lg) * x_row + 2 * k : kNowhere;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      if (kRows > 16 || j == 0 || 4 * j < g.m - m0) {
        xv[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                              rx, at + 4 * j * x_row, 0, 0));
      }
    }
    if constexpr (NORM) {
      nv = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rn, 2 * k, 0, 0));
    }
  };
  f4 total[TN][MT];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
#pragma unroll
    for (int m = 0; m < MT; ++m) total[j][m] = f4{0.f, 0.f, 0.f, 0.f};
  }
  float sq[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) sq[j] = 0.f;
  const V8 ones = __builtin_bit_cast(V8, u32x4{C::kUnit, C::kUnit, C::kUnit, C::kUnit});
  uint32_t sixteens = C::kOne;
  asm("" : "+v"(sixteens));

  if (w < g.tk) fetch(w);
  for (int t = w; t < g.tk; t += WAVES) {
    u32x4 q[TN];
    f4 s[TN][GPT], z[TN][GPT];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      q[j] = code[j];
#pragma unroll
      for (int gi = 0; gi < GPT; ++gi) {
        s[j][gi] = scales4<S>(sc[j][gi]);
        z[j][gi] = shifts4(zr[j][gi] | eights, s[j][gi]);
      }
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      if (kRows <= 16 && j > 0 && 4 * j >= g.m - m0) break;  // rows that are not there
      const auto put = [&](int row, u32x4 v) __attribute__((always_inline)) {
        *reinterpret_cast<u32x4*>(stage + row * kRowBytes + 16 * (l16 ^ (row & 15))) = v;
      };
      if constexpr (NORM) {
        u32x4 high, low;
        normed<T>(xv[j], nv, sq[j], high, low);
        put(4 * j + lg, high);
        put(kRows + 4 * j + lg, low);
      } else {
        put(4 * j + lg, xv[j]);
      }
    }
    if (t + WAVES < g.tk) fetch(t + WAVES);
    stage_turn();
#pragma unroll
    for (int gi = 0; gi < GPT; ++gi) {
      f4 acc[TN][MT], sum[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        sum[m] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[j][m] = f4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int i = gi * (4 / GPT); i < (gi + 1) * (4 / GPT); ++i) {
        V8 b[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          b[m] = *reinterpret_cast<const V8*>(stage + (16 * m + l16) * kRowBytes +
                                              16 * ((4 * i + lg) ^ l16));
          sum[m] = C::mma(ones, b[m], sum[m]);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const V8 a = expand<O>(q[j][i], sixteens);
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[j][m] = C::mma(a, b[m], acc[j][m]);
        }
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            total[j][m][r] = fmaf(z[j][gi][r], sum[m][r],
                                  fmaf(s[j][gi][r], acc[j][m][r], total[j][m][r]));
          }
        }
      }
    }
    stage_turn();
  }

  // lane holds weight rows 16 j + 4 lg + r, operand row 16 m + l16 (and, for the norm, the squares of x
  // rows 4 j + lg, over its columns)
  if constexpr (NORM) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      float v = sq[j];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) v += __shfl_xor(v, o);
      if (l16 == 0) s_sq[w][4 * j + lg] = v;
    }
  }
  __syncthreads();  // the stages become the waves' sums
  float* const sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int j = 0; j < TN; ++j) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sums[w * kSums + ((j * MT + m) * 4 + r) * 64 + lane] = total[j][m][r];
      }
    }
  }
  __syncthreads();
  for (int e = tid; e < kRows * 16 * TN; e += 64 * WAVES) {
    const int col = e % (16 * TN), row = e / (16 * TN);
    const int m = m0 + row, n = 16 * tn + col;
    if (m >= g.m || n >= g.n) continue;
    const int j = col >> 4, r = col & 3, ln = 16 * ((col >> 2) & 3) + (row & 15);
    const float* at = sums + ((j * MT + (row >> 4)) * 4 + r) * 64 + ln;
    float y = 0.f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) y += at[v * kSums];
    if constexpr (NORM) {
      constexpr int kLow = MT == 1 ? 8 : MT / 2 * 256;  // from a row's sum to its remainder's
#pragma unroll
      for (int v = 0; v < WAVES; ++v) y += at[v * kSums + kLow];
      float total_sq = 0.f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) total_sq += s_sq[v][row];
      y *= rsqrtf(total_sq / static_cast<float>(g.k) + g.eps);
    }
    if (g.res != nullptr) {
      y += static_cast<float>(static_cast<const T*>(g.res)[m * g.r_ld + n]);
    }
    static_cast<T*>(g.out)[m * g.o_ld + n] = static_cast<T>(y);
  }
}

// Many rows of x and many of W: a workgroup of four waves takes 64 operand rows (64 of x, or 32 with the
// norm: 8672 x 2048 at 64 rows then takes 19 us, 15.5 with rounded products) and 4 TN tiles of weight
// rows, TN for each wave, over all of K. A tile of x columns is staged once for the workgroup, in three
// LDS buffers; x comes from memory three tiles ahead of its use, the codes two. Wave w forms X of the next
// tile for x block w, and a group's sums begin at -(16 + z) X. KS = 2: two such teams, every other tile of
// columns each, for two waves a SIMD where one workgroup fills a CU.
// Bound by latency and issue together: 28672 x 8192 at 64 rows takes 54 to 59 us in graphs, with cold and
// with cached weights (2.1 TB/s of them, 530 TFLOP/s), and 50 timed call by call; with both kinds of load
// left out 49, with LDS reads, dequantising and scaling left out too 35, of which the matrix instructions
// are 18 and the rest barriers, staging and addresses (213 vector and 36 matrix instructions a tile of
// columns). Sums that begin at -(16 + z) X need no pass over X afterwards: 191 became 213 at groups of 128,
// which costs nothing there, and groups of 32 no longer spill (28672 x 4096 at 64 rows: 51 -> 40 us). Tried
// without gain: deeper rings, operands expanded or read a step earlier, set mixes of matrix and vector
// instructions, 4 tile rows a wave.
template <typename T, typename S, int GPT, int TN, int KS, bool NORM, bool ZEROS>
__global__ __launch_bounds__(256 * KS, 2) void linear4_wide_kernel(const Lin4Geom g) {
  using O = typename Operand<T, NORM>::type;
  using C = Code<O>;
  using V8 = typename C::v8;
  constexpr int MT = 4, kStage = MT * 16 * 256;  // a block of operand rows for each wave
  constexpr int kBlocks = MT / (NORM ? 2 : 1);   // of x rows
  constexpr int kAhead = 2;
  static_assert(KS <= 2 && 3 * kStage >= TN * MT * 4096, "the second team's sums fit its stages");
  __shared__ __attribute__((aligned(16))) char lds_all[KS][3 * kStage];
  __shared__ float s_x_all[KS][2][GPT][16 * MT], s_sq[NORM ? KS : 1][16 * kBlocks];
  const int team = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), tid = threadIdx.x & 255;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* const lds = lds_all[team];
  auto& s_x = s_x_all[team];
  const int l16 = lane & 15, lg = lane >> 4;
  const int tn = (blockIdx.x * 4 + w) * TN, m0 = blockIdx.y * (16 * kBlocks);

  // reads past an extent give 0: tile rows past the last, x rows past M
  const int64_t tile0 = static_cast<int64_t>(min(tn, g.tiles)) * g.tk;
  const int64_t left = max(0, min(g.tiles - tn, TN)) * g.tk;
  const __amdgpu_buffer_rsrc_t rc = rsrc4(g.codes + tile0 * 1024, left * 1024);
  const __amdgpu_buffer_rsrc_t rs = rsrc4(g.scales + tile0 * (GPT * 32), left * (GPT * 32));
  const __amdgpu_buffer_rsrc_t rz = rsrc4(ZEROS ? g.zeros + tile0 * (GPT * 16) : g.codes,
                                          ZEROS ? left * (GPT * 16) : 0);
  const __amdgpu_buffer_rsrc_t rx = rsrc4(g.x, ((g.m - 1) * g.x_ld + g.k) * 2);
  const __amdgpu_buffer_rsrc_t rn = rsrc4(g.nw, NORM ? 2 * g.k : 0);
  const unsigned x_row = static_cast<unsigned>(g.x_ld) * 2;
  const int row = tid >> 4, chunk = tid & 15;  // what this thread stages: rows 16 u + row

  u32x4 code[kAhead][TN], xv[kBlocks], nv;
  u32x2 sc[kAhead][TN][GPT];
  uint32_t zr[kAhead][TN][GPT];
  auto fetch_w = [&](int d, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      // tiles past K: nothing, which makes every product 0
      const unsigned tile = j * g.tk + t, none = t < g.tk ? 0u : kNowhere;
      code[d][j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                 rc, (none + 1024 * tile) + 16 * lane, 0, 2));
#pragma unroll
      for (int gi = 0; gi < GPT; ++gi) {
        const unsigned at = (tile * GPT + gi) * 16;
        sc[d][j][gi] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(
                                                     rs, (none + 2 * at) + 8 * lg, 0, 0));
        if constexpr (ZEROS) {
          zr[d][j][gi] = __builtin_amdgcn_raw_buffer_load_b32(rz, (none + at) + 4 * lg, 0, 0);
        }
      }
    }
  };
  auto fetch_x = [&](int t) __attribute__((always_inline)) {
    const int k = 128 * t + 8 * chunk;
    const unsigned at = k < g.k ? (m0 + row) * x_row + 2 * k : kNowhere;
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
      xv[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                            rx, at + 16 * u * x_row, 0, 0));
    }
    if constexpr (NORM) {
      nv = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rn, 2 * k, 0, 0));
    }
  };
  float sq[kBlocks];
  auto put_x = [&](int buffer) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
      u32x4* const to = reinterpret_cast<u32x4*>(lds + buffer + (16 * u + row) * 256 + 16 * (chunk ^ row));
      if constexpr (NORM) {
        normed<T>(xv[u], nv, sq[u], to[0], to[kBlocks * 256]);
      } else {
        *to = xv[u];
      }
    }
  };

  f4 total[TN][MT], acc[2][TN][MT], last[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    last[j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int m = 0; m < MT; ++m) total[j][m] = acc[0][j][m] = acc[1][j][m] = last[j];
  }
#pragma unroll
  for (int u = 0; u < kBlocks; ++u) sq[u] = 0.f;
  const V8 ones = __builtin_bit_cast(V8, u32x4{C::kUnit, C::kUnit, C::kUnit, C::kUnit});
  uint32_t sixteens = C::kOne;
  asm("" : "+v"(sixteens));
  // total += scale (A - (16 + z) X) of the group before
  auto settle = [&](int p) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          total[j][m][r] = fmaf(last[j][r], acc[p][j][m][r], total[j][m][r]);
        }
        asm volatile("" : "+v"(total[j][m]));  // here, not all after the loop
      }
    }
  };
  V8 b[2][MT];
  auto read = [&](int p, int buffer, int i) __attribute__((always_inline)) {
    // chunk c of a row lies at c ^ (row & 15): a read of 16 rows meets 16 bank groups
    const char* at = lds + buffer + l16 * 256 + 16 * ((4 * i + lg) ^ l16);
#pragma unroll
    for (int m = 0; m < MT; ++m) b[p][m] = *reinterpret_cast<const V8*>(at + 16 * m * 256);
  };
  // operand block w of a step: the wave's share of X
  auto own = [&](int buffer, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const V8*>(lds + buffer + (16 * w + l16) * 256 + 16 * ((4 * i + lg) ^ l16));
  };

  fetch_x(team);
#pragma unroll
  for (int d = 0; d < kAhead; ++d) fetch_w(d, team + KS * d);
  put_x(0);
  fetch_x(team + KS);
  put_x(kStage);
  fetch_x(team + 2 * KS);
  lds_barrier();
  constexpr int kPer = 4 / GPT;  // steps of a group
  f4 sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // X of the first tile
    if (i % kPer == 0) sum = f4{0.f, 0.f, 0.f, 0.f};
    sum = C::mma(ones, own(0, i), sum);
    if (i % kPer == kPer - 1) s_x[0][i / kPer][16 * w + l16] = sum[0];
  }
  lds_barrier();
  read(0, 0, 0);
  int here = 0, next = kStage, after = 2 * kStage;
  // Whole groups of kAhead tiles with no way out inside, so that the compiler's counts of loads in
  // flight stay exact; tiles past K add 0. A tile's x is put in place two tiles early, so its
  // operands can be read a step ahead also across a barrier. A group's sums are scaled while the next group's form.
  for (int t0 = team; t0 - team < g.tk; t0 += KS * kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      const int t = t0 + KS * d;
      put_x(after);
      fetch_x(t + 3 * KS);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int gi = i / kPer, p = (GPT * d + gi) & 1;
        float x[MT];
        if (i % kPer == 0) {
          // LDS answers in order, and the group's sums begin with these
#pragma unroll
          for (int m = 0; m < MT; ++m) x[m] = s_x[d & 1][gi][16 * m + l16];
          __builtin_amdgcn_sched_barrier(0);
        }
        read((i + 1) & 1, i < 3 ? here : next, (i + 1) & 3);
        const V8 share = own(next, i);
        if (i % kPer == 0) {
          sum = f4{0.f, 0.f, 0.f, 0.f};
          settle(p ^ 1);
          // a group's sums begin at -(16 + z) X
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            last[j] = scales4<S>(sc[d][j][gi]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                acc[p][j][m][r] = ZEROS
                    ? -(16.f + static_cast<float>((zr[d][j][gi] >> (8 * r)) & 0xffu)) * x[m]
                    : -24.f * x[m];
              }
            }
          }
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const V8 a = expand<O>(code[d][j][i], sixteens);
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[p][j][m] = C::mma(a, b[i & 1][m], acc[p][j][m]);
        }
        sum = C::mma(ones, share, sum);
        // X of the next tile, the same from four lanes
        if (i % kPer == kPer - 1) s_x[(d + 1) & 1][gi][16 * w + l16] = sum[0];
        __builtin_amdgcn_sched_barrier(0);
      }
      fetch_w(d, t + KS * kAhead);
      lds_barrier();
      const int free = here;
      here = next, next = after, after = free;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  settle((GPT * kAhead - 1) & 1);
  if constexpr (NORM) {
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
      float v = sq[u];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) v += __shfl_xor(v, o);
      if (chunk == 0) s_sq[team][16 * u + row] = v;
    }
  }
  if constexpr (KS == 2) {  // the second team's sums, through its own stages
    __syncthreads();
    f4* const sums = reinterpret_cast<f4*>(lds_all[KS - 1]);
    if (team == 1) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int m = 0; m < MT; ++m) sums[(j * MT + m) * 256 + tid] = total[j][m];
      }
    }
    __syncthreads();
    if (team == 1) return;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
      for (int m = 0; m < MT; ++m) total[j][m] += sums[(j * MT + m) * 256 + tid];
    }
  } else if constexpr (NORM) {
    __syncthreads();
  }
  // lane holds weight rows 16 j + 4 lg + r of the wave's, operand rows 16 m + l16
#pragma unroll
  for (int m = 0; m < kBlocks; ++m) {
    const int xr = m0 + 16 * m + l16;
    if (xr >= g.m) continue;
    float scale = 1.f;
    if constexpr (NORM) {
      float total_sq = s_sq[0][16 * m + l16];
      if constexpr (KS == 2) total_sq += s_sq[1][16 * m + l16];
      scale = rsqrtf(total_sq / static_cast<float>(g.k) + g.eps);
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = 16 * (tn + j) + 4 * lg;
      const T* res = g.res != nullptr ? static_cast<const T*>(g.res) + xr * g.r_ld + n : nullptr;
      T* out = static_cast<T*>(g.out) + xr * g.o_ld + n;
      typedef T t4 __attribute__((ext_vector_type(4)));
      t4 y;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = NORM ? (total[j][m][r] + total[j][(m + kBlocks) % MT][r]) * scale : total[j][m][r];
        if (res != nullptr && n + r < g.n) v += static_cast<float>(res[r]);
        y[r] = static_cast<T>(v);
      }
      if (g.four && n + 4 <= g.n) {
        *reinterpret_cast<t4*>(out) = y;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (n + r < g.n) out[r] = y[r];
        }
      }
    }
  }
}

bool apart(const char* a0, const char* a1, const char* b0, const char* b1) {
  return a1 <= b0 || b1 <= a0;
}

int validate(const m3_linear4_args& a) {
  if (a.m < 0 || a.n < 0 || a.k < 0) return fail(M3_EINVAL, "m3_linear4: negative dimensions");
  if (a.dtype != M3_BF16 && a.dtype != M3_F16) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: dtype %d, expected bf16 or f16", a.dtype);
  }
  if (a.scale_dtype != M3_BF16 && a.scale_dtype != M3_F16) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: scale dtype %d, expected bf16 or f16", a.scale_dtype);
  }
  if (a.group != 32 && a.group != 64 && a.group != 128) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: group %d, expected 32, 64 or 128", a.group);
  }
  if (a.m > kMaxRows) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: M = %lld > %d rows", static_cast<long long>(a.m),
                kMaxRows);
  }
  if (a.k % a.group != 0 || a.k > (1 << 20) || a.n > (1 << 27)) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: N = %lld, K = %lld: K must be a multiple of the group "
                "up to 2^20, N at most 2^27", static_cast<long long>(a.n),
                static_cast<long long>(a.k));
  }
  if (a.m == 0 || a.n == 0) return M3_OK;
  if (a.k == 0) return fail(M3_EUNSUPPORTED, "m3_linear4: K = 0");
  int rc;
  if ((rc = check_tensor(a.x, "x", 2, a.k, true, a.dtype)) ||
      (rc = check_tensor(a.norm_weight, "norm_weight", 1, a.k, false, a.dtype)) ||
      (rc = check_tensor(a.residual, "residual", 2, a.n, false, a.dtype)) ||
      (rc = check_tensor(a.out, "out", 2, a.n, true, a.dtype))) {
    return rc;
  }
  if (a.codes == nullptr || a.scales == nullptr) {
    return fail(M3_EINVAL, "m3_linear4: codes or scales are NULL");
  }
  const auto off = [](const void* p, int by) { return reinterpret_cast<uintptr_t>(p) % by != 0; };
  if (off(a.x.ptr, 16) || a.x.stride[0] % 8 != 0 || off(a.norm_weight.ptr, 16) ||
      off(a.codes, 16) || off(a.scales, 8) || off(a.zeros, 4)) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: x rows, norm_weight and codes must be 16-byte "
                "aligned, scales 8-byte, zeros 4-byte");
  }
  if (present(a.norm_weight) && !(a.norm_eps >= 0.f)) {
    return fail(M3_EINVAL, "m3_linear4: norm_eps must be >= 0");
  }
  // offsets within x, and within the tile rows of a workgroup, are 32-bit, in bytes
  if ((a.m - 1) * a.x.stride[0] + a.k >= (1 << 28)) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: x spans over 512 MB");
  }
  if (a.m > 1 && a.out.stride[0] < a.n) return fail(M3_EINVAL, "m3_linear4: rows of out overlap");
  const int64_t tiles = (a.n + 15) / 16 * ((a.k + 127) / 128), groups = tiles * (128 / a.group);
  const char* o0 = static_cast<const char*>(a.out.ptr);
  const char* o1 = o0 + ((a.m - 1) * a.out.stride[0] + a.n) * 2;
  const auto meets = [&](const void* p, int64_t bytes) {
    const char* p0 = static_cast<const char*>(p);
    return p != nullptr && !apart(o0, o1, p0, p0 + bytes);
  };
  if (meets(a.x.ptr, ((a.m - 1) * a.x.stride[0] + a.k) * 2) || meets(a.codes, tiles * 1024) ||
      meets(a.scales, groups * 32) || meets(a.zeros, groups * 16) || meets(a.norm_weight.ptr, a.k * 2)) {
    return fail(M3_EINVAL, "m3_linear4: out overlaps x, the weight or norm_weight");
  }
  const char* r0 = static_cast<const char*>(a.residual.ptr);
  const bool same = r0 == o0 && (a.m == 1 || a.residual.stride[0] == a.out.stride[0]);
  if (r0 != nullptr && !same && !apart(o0, o1, r0, r0 + ((a.m - 1) * a.residual.stride[0] + a.n) * 2)) {
    return fail(M3_EINVAL, "m3_linear4: out overlaps the residual without being it");
  }
  return M3_OK;
}

template <typename T, typename S, int GPT, int MT, int TN, int WAVES, bool NORM>
int launch_kernel(const Lin4Geom& g, hipStream_t stream) {
  constexpr int rows = 16 * MT / (NORM ? 2 : 1);
  const dim3 grid((g.tiles + TN - 1) / TN, (g.m + rows - 1) / rows), block(64 * WAVES);
  hipLaunchKernelGGL((linear4_kernel<T, S, GPT, MT, TN, WAVES, NORM>), grid, block, 0, stream, g);
  return check_launch("m3_linear4");
}

template <typename T, typename S, int GPT, int TN, int KS>
int launch_wide(const Lin4Geom& g, hipStream_t stream) {
  const bool norm = g.nw != nullptr, zeros = g.zeros != nullptr;
  const int rows = norm ? 32 : 64;
  const dim3 grid((g.tiles + 4 * TN - 1) / (4 * TN), (g.m + rows - 1) / rows), block(256 * KS);
  const auto kernel = norm ? (zeros ? linear4_wide_kernel<T, S, GPT, TN, KS, true, true>
                                    : linear4_wide_kernel<T, S, GPT, TN, KS, true, false>)
                           : (zeros ? linear4_wide_kernel<T, S, GPT, TN, KS, false, true>
                                    : linear4_wide_kernel<T, S, GPT, TN, KS, false, false>);
  hipLaunchKernelGGL(kernel, grid, block, 0, stream, g);
  return check_launch("m3_linear4");
}

// Up to 16 rows of x, by tile rows of W (us in graphs with cold weights; WAVES x TN):
//   few (2048 x 4096, 16 rows): 8 x 1 5.5, 4 x 1 7.9, 4 x 2 8.8, 4 x 4 10.8
//   542 (8672 x 2048), 1 row: 4 x 1 4.9, 4 x 2 5.4, 8 x 1 5.6; 16 rows: 6.4, 6.9, 7.6. With the norm, formed
//     once a workgroup, 4 x 2 6.6, 4 x 1 6.6, 8 x 1 7.4 at 1 row and 10.5, 11.1, 12.3 at 16, in two
//     workgroups of 8 rows; one of 16 rows takes 11.8
//   1792 (28672 x 8192), 16 rows: 4 x 4 30, 4 x 2 35, 4 x 1 46, 8 x 1 44; with the norm, the weight read once
//     for 16 rows, 49, and twice for 8 each 62. In groups of 32, whose scales fill the registers, 4 x 1 54, 8 x 1
//     53, 4 x 2 56, 4 x 4 76
// More rows: few tile rows keep the split over columns (2048 x 4096, 64 rows: 7.2 us in blocks of 32, 18 and
// more wide). Else the wide kernel in the form whose rounds of workgroups over the 256 CUs cost least: 65
// a round with 2 tile rows a wave, 44 with 1 (both one workgroup a CU), 87 for 512 workgroups of one team
// (two a CU): 28672 x 8192 at 64 rows 57 / 68 / 65 us, 16384 x 4096 27 / 20 / 26, 8672 x 2048 at 256 rows
// 31 / 31 / 23 and at 64 rows 16.5 / 11.8 / 14.7, with the norm 18.9 / 25.6 / 21.8; in groups of 32 28672 x 4096 at
// 64 rows 39 / 47 / 44. Between 384 and 1,023 tile rows at up to 32 rows of x the split over columns would be
// quicker (8672 x 2048: 8.6 at 17 rows and 9.7 at 32, against 10.8 and 11.0); it is slower with the norm (14.8 and
// 18.3 against 13.7 and 13.9) and from 64 rows on.
template <typename T, typename S, int GPT, bool NORM>
int launch_few(const Lin4Geom& g, hipStream_t stream) {
  if (g.tiles < 384) return launch_kernel<T, S, GPT, 1, 1, 8, NORM>(g, stream);
  if (g.tiles >= 1024) {
    constexpr int tn = GPT < 4 ? 4 : 1;
    if constexpr (NORM) {
      if (g.m > 8) return launch_kernel<T, S, GPT, 2, tn, 4, true>(g, stream);
    }
    return launch_kernel<T, S, GPT, 1, tn, 4, NORM>(g, stream);
  }
  return launch_kernel<T, S, GPT, 1, NORM && GPT < 4 ? 2 : 1, 4, NORM>(g, stream);
}

template <typename T, typename S, int GPT>
int launch_rows(const Lin4Geom& g, hipStream_t stream) {
  const bool norm = g.nw != nullptr;
  if (g.m <= 16) {
    return norm ? launch_few<T, S, GPT, true>(g, stream) : launch_few<T, S, GPT, false>(g, stream);
  }
  if (g.tiles < 384 && g.tiles * ((g.m + 63) / 64) < 512) {
    return norm ? launch_kernel<T, S, GPT, 2, 1, 8, true>(g, stream)
                : launch_kernel<T, S, GPT, 2, 1, 8, false>(g, stream);
  }
  const int blocks = norm ? (g.m + 31) / 32 : (g.m + 63) / 64;
  const int w1 = (g.tiles + 3) / 4 * blocks, w2 = (g.tiles + 7) / 8 * blocks;
  const int two = (w2 + 255) / 256 * 65, one = (w1 + 255) / 256 * 44, half = max(w1, 512) * 87 / 512;
  if (two <= one && two <= half) return launch_wide<T, S, GPT, 2, 2>(g, stream);
  return one <= half ? launch_wide<T, S, GPT, 1, 2>(g, stream)
                     : launch_wide<T, S, GPT, 1, 1>(g, stream);
}

template <typename T, typename S>
int launch_group(const Lin4Geom& g, int group, hipStream_t stream) {
  switch (group) {
    case 32: return launch_rows<T, S, 4>(g, stream);
    case 64: return launch_rows<T, S, 2>(g, stream);
    default: return launch_rows<T, S, 1>(g, stream);
  }
}

template <typename T>
int launch(const Lin4Geom& g, int scale_dtype, int group, hipStream_t stream) {
  return scale_dtype == M3_BF16 ? launch_group<T, __bf16>(g, group, stream)
                                : launch_group<T, _Float16>(g, group, stream);
}

}  // namespace
}  // namespace m3

extern "C" int m3_linear4(const m3_linear4_args* args, hipStream_t stream) {
  using namespace m3;
  clear_error();
  if (args == nullptr) return fail(M3_EINVAL, "m3_linear4: NULL args");
  const m3_linear4_args& a = *args;
  const int rc = validate(a);
  if (rc != M3_OK) return rc;
  if (a.m == 0 || a.n == 0) return M3_OK;
  const Lin4Geom g{static_cast<const char*>(a.codes), static_cast<const char*>(a.scales),
                   static_cast<const char*>(a.zeros), static_cast<const char*>(a.x.ptr),
                   static_cast<const char*>(a.norm_weight.ptr), a.residual.ptr, a.out.ptr,
                   a.x.stride[0], a.residual.stride[0], a.out.stride[0],
                   static_cast<int>(a.m), static_cast<int>(a.n), static_cast<int>(a.k),
                   static_cast<int>((a.k + 127) / 128), static_cast<int>((a.n + 15) / 16),
                   reinterpret_cast<uintptr_t>(a.out.ptr) % 8 == 0 && a.out.stride[0] % 4 == 0,
                   a.norm_eps};
  return a.dtype == M3_BF16 ? launch<__bf16>(g, a.scale_dtype, a.group, stream)
                            : launch<_Float16>(g, a.scale_dtype, a.group, stream);
}
