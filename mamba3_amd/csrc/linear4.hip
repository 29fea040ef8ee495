// m3_linear4: out[M, N] = x'[M, K] * W[N, K]^T (+ residual), W = (q - z) * scale in 4-bit codes with a
// scale (and a zero) for every group of 32, 64 or 128 columns: the decode step's projections.
//
// A code goes into the mantissa of a 16-bit 1.0, which makes 1 + q / 16 exactly (a shift and an
// and-or for two codes), and that is the matrix operand. With A = sum (1 + q / 16) x over a group and
// X = sum x, the group's share is scale * (16 A - (16 + z) X): the scale and the zero meet FP32
// sums, not the operands. X comes from one more matrix product, with ones.
//
// One workgroup takes 16 weight rows, its waves every WAVES-th tile of 128 columns; their sums
// meet in LDS.
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
  static constexpr uint32_t kOne = 0x3f803f80u, kMask = 0x00780078u;
  static constexpr int kUp = 3;  // the code's low bit: 1/16 in bf16's 7 bits of mantissa
  static __device__ __forceinline__ f4 mma(v8 a, v8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Code<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kOne = 0x3c003c00u, kMask = 0x03c003c0u;
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
  int scale_dtype;
  float eps;
};

template <typename T, int GPT, int WAVES, bool NORM>
__global__ __launch_bounds__(64 * WAVES) void linear4_kernel(const Lin4Geom g) {
  using C = Code<T>;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  const int tn = blockIdx.x, m0 = blockIdx.y * 16;
  const char* codes = g.codes + static_cast<int64_t>(tn) * g.tk * 1024 + lane * 16;
  const int64_t group0 = static_cast<int64_t>(tn) * g.tk * GPT;
  const char* xrow = g.x + static_cast<int64_t>(min(m0 + l16, g.m - 1)) * g.x_ld * 2;
  const typename C::v8 ones = expand<T>(0);
  f4 total = {0.f, 0.f, 0.f, 0.f};
  float ssq = 0.f;
  for (int t = w; t < g.tk; t += WAVES) {
    const u32x4 q = *reinterpret_cast<const u32x4*>(codes + static_cast<int64_t>(t) * 1024);
#pragma unroll
    for (int gi = 0; gi < GPT; ++gi) {
      if (128 * t + gi * (128 / GPT) >= g.k) break;
      f4 acc = {0.f, 0.f, 0.f, 0.f}, sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = gi * (4 / GPT); i < (gi + 1) * (4 / GPT); ++i) {
        const int k = 128 * t + 32 * i + 8 * lg;
        typename C::v8 b = *reinterpret_cast<const typename C::v8*>(xrow + 2 * k);
        if constexpr (NORM) {
          const typename C::v8 nv = *reinterpret_cast<const typename C::v8*>(g.nw + 2 * k);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float xf = static_cast<float>(b[e]);
            ssq = fmaf(xf, xf, ssq);
            b[e] = static_cast<T>(xf * static_cast<float>(nv[e]));
          }
        }
        acc = C::mma(expand<T>(q[i]), b, acc);
        sum = C::mma(ones, b, sum);
      }
      // rows 4 lg + r of the tile
      const int64_t at = (group0 + static_cast<int64_t>(t) * GPT + gi) * 16 + 4 * lg;
      const u32x2 sv = *reinterpret_cast<const u32x2*>(g.scales + 2 * at);
      const uint32_t zv = g.zeros != nullptr
                              ? *reinterpret_cast<const uint32_t*>(g.zeros + at) : 0x08080808u;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float s = decode_x((sv[r >> 1] >> (16 * (r & 1))) & 0xffffu, 0u, g.scale_dtype);
        const float z = static_cast<float>((zv >> (8 * r)) & 0xffu);
        total[r] = fmaf(s, fmaf(16.f, acc[r], -(16.f + z) * sum[r]), total[r]);
      }
    }
  }
  __shared__ float red[WAVES][4][64];
  __shared__ float red_ssq[WAVES][16];
#pragma unroll
  for (int r = 0; r < 4; ++r) red[w][r][lane] = total[r];
  if constexpr (NORM) {
    ssq += __shfl_xor(ssq, 16);
    ssq += __shfl_xor(ssq, 32);
    if (lg == 0) red_ssq[w][l16] = ssq;
  }
  __syncthreads();
  for (int e = tid; e < 256; e += 64 * WAVES) {
    const int r = e >> 6, ln = e & 63;
    const int m = m0 + (ln & 15), n = 16 * tn + 4 * (ln >> 4) + r;
    if (m >= g.m || n >= g.n) continue;
    float y = 0.f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) y += red[v][r][ln];
    if constexpr (NORM) {
      float sq = 0.f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) sq += red_ssq[v][ln & 15];
      y *= rsqrtf(sq / static_cast<float>(g.k) + g.eps);
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
  if (a.k % a.group != 0 || a.k > (1 << 24) || a.n > (1 << 28)) {
    return fail(M3_EUNSUPPORTED, "m3_linear4: N = %lld, K = %lld: K must be a multiple of the group "
                "up to 2^24, N at most 2^28", static_cast<long long>(a.n),
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

template <typename T, int GPT>
int launch_group(const Lin4Geom& g, hipStream_t stream) {
  constexpr int kWaves = 4;
  const dim3 grid((g.n + 15) / 16, (g.m + 15) / 16), block(64 * kWaves);
  if (g.nw != nullptr) {
    hipLaunchKernelGGL((linear4_kernel<T, GPT, kWaves, true>), grid, block, 0, stream, g);
  } else {
    hipLaunchKernelGGL((linear4_kernel<T, GPT, kWaves, false>), grid, block, 0, stream, g);
  }
  return check_launch("m3_linear4");
}

template <typename T>
int launch(const Lin4Geom& g, int group, hipStream_t stream) {
  switch (group) {
    case 32: return launch_group<T, 4>(g, stream);
    case 64: return launch_group<T, 2>(g, stream);
    default: return launch_group<T, 1>(g, stream);
  }
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
                   static_cast<int>((a.k + 127) / 128), a.scale_dtype, a.norm_eps};
  return a.dtype == M3_BF16 ? launch<__bf16>(g, a.group, stream)
                            : launch<_Float16>(g, a.group, stream);
}
