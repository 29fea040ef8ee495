// m3_linear4: out[M, N] = x'[M, K] * W[N, K]^T (+ residual), W = (q - z) * scale in 4-bit codes with a
// scale (and a zero) for every group of 32, 64 or 128 columns: the decode step's projections.
//
// A code goes into the mantissa of a 16-bit 16.0, which makes 16 + q exactly (a shift and an and-or
// for two codes), and that is the matrix operand. With A = sum (16 + q) x over a group and X = sum x,
// the group's share is scale * A - scale * (16 + z) * X: the scale and the zero meet FP32 sums, not the
// operands. X comes from one more matrix product, with ones.
//
// A workgroup takes TN tiles of 16 weight rows and up to MT blocks of 16 x rows. Its waves take every WAVES-th
// tile of 128 columns each, so no two read the same operand and the K loop has no barrier; their
// sums meet in LDS. A wave's next codes and x are on their way in registers while it multiplies; x goes
// through an LDS region of the wave's own, where it is normed, and comes back as the operand's columns.
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

template <typename T>
__device__ __forceinline__ typename Code<T>::v8 expand(uint32_t w) {
  u32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    constexpr int up = Code<T>::kUp;
    const uint32_t at = 4 * j > up ? w >> (4 * j - up) : w << (up - 4 * j);
    v[j] = (at & Code<T>::kMask) | Code<T>::kOne;
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

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc4(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0),
                                           static_cast<int>(bytes), 0x00020000);
}

// Between a wave's writes of its own LDS region and its lanes' reads of one another's, and back: LDS
// operations of one wave complete in order, so only the compiler has to keep them so.
__device__ __forceinline__ void stage_turn() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int kRowBytes = 256 + 16;  // an x row of a tile in LDS: 16 rows start in 16 bank groups

template <typename T, typename S, int GPT, int MT, int TN, int WAVES, bool NORM>
__global__ __launch_bounds__(64 * WAVES) void linear4_kernel(const Lin4Geom g) {
  using C = Code<T>;
  using V8 = typename C::v8;
  constexpr int kStage = MT * 16 * kRowBytes, kSums = MT * TN * 256;
  constexpr int kLds = WAVES * (kStage > 4 * kSums ? kStage : 4 * kSums);
  __shared__ __attribute__((aligned(16))) char lds[kLds];
  __shared__ float s_sq[NORM ? WAVES : 1][16 * MT];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int tn = blockIdx.x * TN, m0 = blockIdx.y * (16 * MT);
  const int loads = (min(g.m - m0, 16 * MT) + 3) / 4;  // four x rows of 256 bytes each
  char* const stage = lds + w * kStage;

  // what a tile of columns needs: codes, scales and zeros of TN tile rows, x rows 4 j + lg.
  u32x4 code[TN], xv[4 * MT], nv;
  u32x2 sc[TN][GPT];
  uint32_t zr[TN][GPT];
  // reads past an extent give 0: tile rows past the last, x rows past M
  const int64_t tile0 = static_cast<int64_t>(tn) * g.tk, left = min(g.tiles - tn, TN) * g.tk;
  const __amdgpu_buffer_rsrc_t rc = rsrc4(g.codes + tile0 * 1024, left * 1024);
  const __amdgpu_buffer_rsrc_t rs = rsrc4(g.scales + tile0 * (GPT * 32), left * (GPT * 32));
  const __amdgpu_buffer_rsrc_t rz =
      rsrc4(g.zeros + (g.zeros != nullptr ? tile0 * (GPT * 16) : 0), left * (GPT * 16));
  const __amdgpu_buffer_rsrc_t rx = rsrc4(g.x, ((g.m - 1) * g.x_ld + g.k) * 2);
  const __amdgpu_buffer_rsrc_t rn = rsrc4(g.nw, NORM ? 2 * g.k : 0);
  const int x_row = static_cast<int>(g.x_ld) * 2;
  auto fetch = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int tile = j * g.tk + t;
      // non-temporal (aux bit 1): the codes are read once a call
      code[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                              rc, 16 * lane, 1024 * tile, 2));
#pragma unroll
      for (int gi = 0; gi < GPT; ++gi) {
        const int at = (tile * GPT + gi) * 16;
        sc[j][gi] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(
                                                  rs, 8 * lg, 2 * at, 0));
        if (g.zeros != nullptr) {
          zr[j][gi] = __builtin_amdgcn_raw_buffer_load_b32(rz, 4 * lg, at, 0);
        }
      }
    }
    const int k = 2 * (128 * t + 8 * l16);  // columns past K: read, not used
#pragma unroll
    for (int j = 0; j < 4 * MT; ++j) {
      if (j < loads) {
        xv[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                              rx, lg * x_row + k, (m0 + 4 * j) * x_row, 0));
      }
    }
    if constexpr (NORM) {
      nv = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rn, k, 0, 0));
    }
  };
#pragma unroll
  for (int j = 0; j < TN; ++j) {
#pragma unroll
    for (int gi = 0; gi < GPT; ++gi) zr[j][gi] = 0x08080808u;
  }

  f4 total[TN][MT];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
#pragma unroll
    for (int m = 0; m < MT; ++m) total[j][m] = f4{0.f, 0.f, 0.f, 0.f};
  }
  float sq[4 * MT];
#pragma unroll
  for (int j = 0; j < 4 * MT; ++j) sq[j] = 0.f;
  const V8 ones = __builtin_bit_cast(V8, u32x4{C::kUnit, C::kUnit, C::kUnit, C::kUnit});

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
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          z[j][gi][r] = -(16.f + static_cast<float>((zr[j][gi] >> (8 * r)) & 0xffu)) * s[j][gi][r];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4 * MT; ++j) {
      if (j < loads) {
        u32x4 v = xv[j];
        if constexpr (NORM) {
          V8 b = __builtin_bit_cast(V8, v);
          const V8 n = __builtin_bit_cast(V8, nv);
          const bool in = 128 * t + 8 * l16 < g.k;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float xf = static_cast<float>(b[e]), xk = in ? xf : 0.f;
            sq[j] = fmaf(xk, xk, sq[j]);
            b[e] = static_cast<T>(xf * static_cast<float>(n[e]));
          }
          v = __builtin_bit_cast(u32x4, b);
        }
        *reinterpret_cast<u32x4*>(stage + (4 * j + lg) * kRowBytes + 16 * l16) = v;
      }
    }
    if (t + WAVES < g.tk) fetch(t + WAVES);
    stage_turn();
#pragma unroll
    for (int gi = 0; gi < GPT; ++gi) {
      if (128 * t + gi * (128 / GPT) < g.k) {
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
            b[m] = *reinterpret_cast<const V8*>(stage + (16 * m + l16) * kRowBytes + 64 * i + 16 * lg);
            sum[m] = C::mma(ones, b[m], sum[m]);
          }
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const V8 a = expand<T>(q[j][i]);
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
    }
    stage_turn();
  }

  // lane holds weight rows 16 j + 4 lg + r, x row 16 m + l16 (and, for the norm, the squares of x
  // rows 4 j + lg, over its columns)
  if constexpr (NORM) {
#pragma unroll
    for (int j = 0; j < 4 * MT; ++j) {
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
  for (int e = tid; e < kSums; e += 64 * WAVES) {
    const int col = e % (16 * TN), row = e / (16 * TN);
    const int m = m0 + row, n = 16 * tn + col;
    if (m >= g.m || n >= g.n) continue;
    const int j = col >> 4, r = col & 3, ln = 16 * ((col >> 2) & 3) + (row & 15);
    const float* at = sums + ((j * MT + (row >> 4)) * 4 + r) * 64 + ln;
    float y = 0.f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) y += at[v * kSums];
    if constexpr (NORM) {
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
  if (a.k % a.group != 0 || a.k > (1 << 20) || a.n > (1 << 28)) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: N = %lld, K = %lld: K must be a multiple of the group "
                "up to 2^20, N at most 2^28", static_cast<long long>(a.n),
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
  // offsets within x, and within the tile rows of a workgroup, are 32-bit, in bytes
  if ((a.m - 1) * a.x.stride[0] + a.k >= (1 << 29)) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: x spans over 1 GB");
  }
  if (a.m > 1 && a.out.stride[0] < a.n) return fail(M3_EINVAL, "m3_linear4: rows of out overlap");
  const int64_t tiles = (a.n + 15) / 16 * ((a.k + 127) / 128);
  const char* o0 = static_cast<const char*>(a.out.ptr);
  const char* o1 = o0 + ((a.m - 1) * a.out.stride[0] + a.n) * 2;
  const char* x0 = static_cast<const char*>(a.x.ptr);
  const char* c0 = static_cast<const char*>(a.codes);
  if (!apart(o0, o1, x0, x0 + ((a.m - 1) * a.x.stride[0] + a.k) * 2) ||
      !apart(o0, o1, c0, c0 + tiles * 1024)) {
    return fail(M3_EINVAL, "m3_linear4: out overlaps x or the weight");
  }
  return M3_OK;
}

template <typename T, typename S, int GPT, int MT, int TN, int WAVES>
int launch_kernel(const Lin4Geom& g, hipStream_t stream) {
  const dim3 grid((g.tiles + TN - 1) / TN, (g.m + 16 * MT - 1) / (16 * MT)), block(64 * WAVES);
  if (g.nw != nullptr) {
    hipLaunchKernelGGL((linear4_kernel<T, S, GPT, MT, TN, WAVES, true>), grid, block, 0, stream, g);
  } else {
    hipLaunchKernelGGL((linear4_kernel<T, S, GPT, MT, TN, WAVES, false>), grid, block, 0, stream, g);
  }
  return check_launch("m3_linear4");
}

template <typename T, typename S, int GPT>
int launch_rows(const Lin4Geom& g, hipStream_t stream) {
  if (g.m <= 16) {
    if (g.tiles < 256 && g.tk >= 32) return launch_kernel<T, S, GPT, 1, 1, 16>(g, stream);
    if (g.tiles < 1024) return launch_kernel<T, S, GPT, 1, 1, 8>(g, stream);
    return launch_kernel<T, S, GPT, 1, 2, 8>(g, stream);
  }
  if (g.m <= 32) {
    return g.tiles < 512 ? launch_kernel<T, S, GPT, 2, 1, 8>(g, stream)
                         : launch_kernel<T, S, GPT, 2, 2, 8>(g, stream);
  }
  return g.tiles < 512 ? launch_kernel<T, S, GPT, 4, 1, 8>(g, stream)
                       : launch_kernel<T, S, GPT, 4, 2, 8>(g, stream);
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
                   static_cast<int>((a.k + 127) / 128), static_cast<int>((a.n + 15) / 16), a.norm_eps};
  return a.dtype == M3_BF16 ? launch<__bf16>(g, a.scale_dtype, a.group, stream)
                            : launch<_Float16>(g, a.scale_dtype, a.group, stream);
}
