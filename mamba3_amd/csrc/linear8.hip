// m3_linear8: out[M, N] = (sum_k codes[m, k] q[n, k]) row_scale[m] scale[n] (+ residual), codes and q in 8
// bits, on the integer matrix instructions (16x16x64, twice bf16's rate): the projections of any number
// of rows.
//
// The sums are exact in 32 bits (K < 2^17), so their order is free and every kernel gives the same bits; each
// output then has three FP32 roundings and its own.
//
// The weight is an instruction's first operand: a lane of its result holds four consecutive columns n of one
// row m. The weight's tiles order their 64 rows so that two results side by side are eight columns, 16 bytes of
// a 16-bit output, and four lanes 64 bytes.
//
// linear8_rows_kernel (few rows): a workgroup takes 16 weight rows and 16 MT rows of codes; its waves
// take every WAVES-th tile of 64 columns, straight into registers, and their sums meet in LDS. Bound by the
// weight's stream, or the launch and one latency of memory.
//
// linear8_tile_kernel: a workgroup takes BM rows by BN columns and walks K in steps of 128. A step's
// codes and tiles go from memory into one of two LDS stages without passing through registers, while the other
// is multiplied; one barrier a step. Codes lie in LDS in rows of 128 bytes, whose eight pieces of 16 are
// exchanged by the row's low bits: eight lanes reading one column's pieces of eight rows meet all banks.
#include <hip/hip_runtime.h>

#include "m3_common.hpp"
#include "m3_host.hpp"

namespace m3 {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileBytes = 4096;  // 64 weight rows x 64 columns

struct Lin8Geom {
  const char* codes;
  const float* row_scales;
  const char* q;
  const float* scales;
  const void* res;  // or null
  void* out;
  int64_t c_ld, r_ld, o_ld;  // bytes; elements
  int64_t m;
  int n, k, tk;     // tk: tiles of 64 columns in a tile row of the weight
  int tiles;        // tile rows
};

// An offset past every extent, also with a whole row of tiles added.
constexpr unsigned kNowhere = 0x7fff0000u;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc8(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0),
                                           static_cast<int>(bytes), 0x00020000);
}

__device__ __forceinline__ i4 mma(i4 a, i4 b, i4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// The codes of up to `rows` rows from m0 on: all but the last one's end lies within the rows themselves.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t codes_rsrc(const Lin8Geom& g, int64_t m0, int rows) {
  const int64_t left = g.m - m0 < rows ? g.m - m0 : rows;
  return rsrc8(g.codes + m0 * g.c_ld, (left - 1) * g.c_ld + (g.k + 15) / 16 * 16);
}

// COUNT (4 or 8) consecutive outputs of one row from column n on.
template <typename T, int COUNT>
__device__ __forceinline__ void put(const Lin8Geom& g, int64_t m, int n, float rs, const i4* sums) {
  float v[COUNT];
#pragma unroll
  for (int e = 0; e < COUNT; e += 4) {
    const f4 sc = *reinterpret_cast<const f4*>(g.scales + n + e);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[e + r] = static_cast<float>(sums[e / 4][r]) * rs * sc[r];
  }
  const T* res = static_cast<const T*>(g.res) + m * g.r_ld + n;
  T* out = static_cast<T*>(g.out) + m * g.o_ld + n;
  T y[COUNT];
  if (n + COUNT <= g.n) {
    if (g.res != nullptr) {
      T t[COUNT];
      __builtin_memcpy(t, res, sizeof(t));
#pragma unroll
      for (int e = 0; e < COUNT; ++e) v[e] += to_f(t[e]);
    }
#pragma unroll
    for (int e = 0; e < COUNT; ++e) y[e] = from_f<T>(v[e]);
    __builtin_memcpy(out, y, sizeof(y));
  } else {
#pragma unroll
    for (int e = 0; e < COUNT; ++e) {
      if (n + e < g.n) out[e] = from_f<T>(g.res != nullptr ? v[e] + to_f(res[e]) : v[e]);
    }
  }
}

template <typename T, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void linear8_rows_kernel(const Lin8Geom g) {
  constexpr int kAhead = 4;  // tiles on their way at a time
  __shared__ i4 parts[WAVES][MT][64];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile = blockIdx.x >> 2, quarter = blockIdx.x & 3;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  const __amdgpu_buffer_rsrc_t rc = codes_rsrc(g, m0, 16 * MT);
  const __amdgpu_buffer_rsrc_t rq =
      rsrc8(g.q + static_cast<int64_t>(tile) * g.tk * kTileBytes, static_cast<int64_t>(g.tk) * kTileBytes);
  i4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = i4{0, 0, 0, 0};
  unsigned xoff[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    xoff[i] = m0 + 16 * i + l16 < g.m ? (16 * i + l16) * static_cast<unsigned>(g.c_ld) + 16 * lg : kNowhere;
  }
  const unsigned qoff = quarter * 1024 + lane * 16;
  const int tiles = (g.k + 63) / 64;
  for (int t0 = w; t0 < tiles; t0 += WAVES * kAhead) {
    i4 a[kAhead], b[kAhead][MT];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int t = t0 + u * WAVES;
      const bool live = t < tiles;
      a[u] = __builtin_bit_cast(i4, __builtin_amdgcn_raw_buffer_load_b128(
          rq, live ? qoff + t * kTileBytes : kNowhere, 0, 2));
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        b[u][i] = __builtin_bit_cast(i4, __builtin_amdgcn_raw_buffer_load_b128(
            rc, live ? xoff[i] + t * 64 : kNowhere, 0, 0));
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = mma(a[u], b[u][i], acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) parts[w][i][lane] = acc[i];
  __syncthreads();
  for (int i = w; i < MT; i += WAVES) {
    i4 sum = parts[0][i][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) sum += parts[v][i][lane];
    const int64_t m = m0 + 16 * i + l16;
    const int n = 64 * tile + 32 * (quarter >> 1) + 4 * (quarter & 1) + 8 * lg;
    if (m < g.m && n < g.n) put<T, 4>(g, m, n, g.row_scales[m], &sum);
  }
}

// The workgroup's tile. Workgroups go to the 8 XCDs in turn; each XCD takes a run of the tiles, in
// bands of `band` tiles along M, column by column, so that what runs on it at a time shares rows and columns in its
// L2.
struct Place {
  int64_t m;
  int n;
};
__device__ __forceinline__ Place place(unsigned id, unsigned tiles_m, unsigned tiles_n, unsigned band) {
  const unsigned all = tiles_m * tiles_n, each = all / 8, more = all % 8, xcd = id % 8;
  const unsigned at = xcd * each + min(xcd, more) + id / 8;
  const unsigned first = at / (band * tiles_n) * band, rest = at - first * tiles_n;
  const unsigned high = min(band, tiles_m - first);
  return Place{first + rest % high, static_cast<int>(rest / high)};
}

// Everything that is on its way into LDS has arrived, for all waves, and what they read was read.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, char* dst, unsigned off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16,
                                           static_cast<int>(off), 0, 0, 0);
}

// WM x WN waves, each 16 XI rows by 64 columns.
template <typename T, int WM, int WN, int XI>
__global__ __launch_bounds__(64 * WM * WN) void linear8_tile_kernel(const Lin8Geom g, unsigned tiles_m,
                                                                    unsigned tiles_n, unsigned band) {
  constexpr int kWaves = WM * WN, BM = 16 * XI * WM, BN = 64 * WN;
  constexpr int kStage = (BM + BN) * 128, kUnits = (BM + BN) / 8 / kWaves;
  static_assert((BM / 8) % kWaves == 0 && (BN / 8) % kWaves == 0, "units of one kind for all waves");
  __shared__ __attribute__((aligned(128))) char stages[2 * kStage];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), wm = w / WN, wn = w % WN;
  const Place at = place(blockIdx.x, tiles_m, tiles_n, band);
  const int64_t m0 = at.m * BM;
  const int tile0 = at.n * WN;  // the first of the workgroup's tile rows of the weight
  const int64_t row_bytes = static_cast<int64_t>(g.tk) * kTileBytes;
  const __amdgpu_buffer_rsrc_t rc = codes_rsrc(g, m0, BM);
  const __amdgpu_buffer_rsrc_t rq = rsrc8(g.q + tile0 * row_bytes, min(WN, g.tiles - tile0) * row_bytes);
  // unit u of the workgroup's loads is 1 KB: 8 rows of codes, or a quarter of a tile
  constexpr int kOfCodes = BM / 8 / kWaves;
  unsigned off[kUnits];
#pragma unroll
  for (int v = 0; v < kUnits; ++v) {
    if (v < kOfCodes) {
      const int r = 8 * (v * kWaves + w) + (lane >> 3);
      off[v] = m0 + r < g.m ? r * static_cast<unsigned>(g.c_ld) + 16 * ((lane & 7) ^ (lane >> 3)) : kNowhere;
    } else {
      const int u = (v - kOfCodes) * kWaves + w, tile = u >> 3;
      off[v] = tile0 + tile < g.tiles ? tile * static_cast<unsigned>(row_bytes) + (u & 7) * 1024 + lane * 16
                                      : kNowhere;
    }
  }
  const auto fetch = [&](char* stage) {
#pragma unroll
    for (int v = 0; v < kUnits; ++v) {
      char* const dst = stage + (v < kOfCodes ? v * kWaves + w : BM / 8 + (v - kOfCodes) * kWaves + w) * 1024;
      load_lds(v < kOfCodes ? rc : rq, dst, off[v]);
      off[v] += v < kOfCodes ? 128 : 2 * kTileBytes;
    }
  };
  i4 acc[4][XI];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int i = 0; i < XI; ++i) acc[j][i] = i4{0, 0, 0, 0};
  }
  const auto multiply = [&](const char* stage) {
    const char* const rows = stage + (16 * XI * wm + l16) * 128;
    const char* const tiles = stage + BM * 128 + wn * (2 * kTileBytes) + lane * 16;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      i4 a[4], b[XI];
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = *reinterpret_cast<const i4*>(tiles + kk * kTileBytes + j * 1024);
#pragma unroll
      for (int i = 0; i < XI; ++i) {
        b[i] = *reinterpret_cast<const i4*>(rows + i * 2048 + 16 * ((4 * kk + lg) ^ (l16 & 7)));
      }
#pragma unroll
      for (int i = 0; i < XI; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][i] = mma(a[j], b[i], acc[j][i]);
      }
    }
  };
  const int steps = g.tk / 2;
  fetch(stages);
  int now = 0;
#pragma unroll 1
  for (int s = 1; s < steps; ++s) {
    stage_barrier();
    fetch(stages + (kStage - now));
    multiply(stages + now);
    now = kStage - now;
  }
  stage_barrier();
  multiply(stages + now);
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int64_t m = m0 + 16 * XI * wm + 16 * i + l16;
    if (m >= g.m) continue;
    const float rs = g.row_scales[m];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = 64 * (tile0 + wn) + 32 * h + 8 * lg;
      const i4 pair[2] = {acc[2 * h][i], acc[2 * h + 1][i]};
      if (n < g.n) put<T, 8>(g, m, n, rs, pair);
    }
  }
}

template <typename T, int MT, int WAVES>
int launch_few(const Lin8Geom& g, hipStream_t stream) {
  const dim3 grid(4 * g.tiles, static_cast<unsigned>((g.m + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((linear8_rows_kernel<T, MT, WAVES>), grid, dim3(64 * WAVES), 0, stream, g);
  return check_launch("m3_linear8");
}

template <typename T, int WM, int WN, int XI>
int launch_tile(const Lin8Geom& g, hipStream_t stream) {
  constexpr int BM = 16 * XI * WM;
  const int64_t tm = (g.m + BM - 1) / BM, tn = (g.tiles + WN - 1) / WN;
  if (tm * tn >= INT32_MAX) return fail(M3_EUNSUPPORTED, "m3_linear8: too many tiles");
  hipLaunchKernelGGL((linear8_tile_kernel<T, WM, WN, XI>), dim3(static_cast<unsigned>(tm * tn)),
                     dim3(64 * WM * WN), 0, stream, g, static_cast<unsigned>(tm), static_cast<unsigned>(tn),
                     8u);
  return check_launch("m3_linear8");
}

template <typename T>
int launch8(const Lin8Geom& g, hipStream_t stream) {
  if (g.m <= 16) return launch_few<T, 1, 8>(g, stream);
  if (g.m <= 64) return launch_few<T, 4, 8>(g, stream);
  if ((g.m + 255) / 256 * ((g.tiles + 3) / 4) >= 256) return launch_tile<T, 2, 4, 8>(g, stream);
  return launch_tile<T, 2, 2, 4>(g, stream);
}

int validate(const m3_linear8_args& a) {
  if (a.m < 0 || a.n < 0 || a.k < 0) return fail(M3_EINVAL, "m3_linear8: negative dimensions");
  if (!valid_dtype(a.dtype)) return fail(M3_EINVAL, "m3_linear8: invalid dtype %d", a.dtype);
  if (a.m >= (1 << 30) || a.n > (1 << 27) || a.k > M3_LINEAR8_MAX_K) {
    return fail(M3_EUNSUPPORTED, "m3_linear8: M = %lld, N = %lld, K = %lld: below 2^30, at most 2^27, at "
                "most %d", static_cast<long long>(a.m), static_cast<long long>(a.n),
                static_cast<long long>(a.k), M3_LINEAR8_MAX_K);
  }
  if (a.m == 0 || a.n == 0) return M3_OK;
  if (a.k == 0) return fail(M3_EUNSUPPORTED, "m3_linear8: K = 0");
  int rc;
  if ((rc = check_tensor(a.residual, "residual", 2, a.n, false, a.dtype)) ||
      (rc = check_tensor(a.out, "out", 2, a.n, true, a.dtype))) {
    return rc;
  }
  if (a.codes == nullptr || a.row_scales == nullptr || a.q == nullptr || a.scales == nullptr) {
    return fail(M3_EINVAL, "m3_linear8: codes, q or scales are NULL");
  }
  const auto off = [](const void* p, int by) { return reinterpret_cast<uintptr_t>(p) % by != 0; };
  if (off(a.codes, 16) || a.codes_stride % 16 != 0 || off(a.q, 16) || off(a.scales, 16) ||
      off(a.row_scales, 4)) {
    return fail(M3_EUNSUPPORTED, "m3_linear8: rows of codes, q and scales must be 16-byte aligned, "
                "row_scales 4-byte");
  }
  // offsets within the rows of a workgroup (up to 256) are 32-bit
  if (a.codes_stride < a.k || a.codes_stride > (1 << 22)) {
    return fail(M3_EUNSUPPORTED, "m3_linear8: codes_stride %lld: at least K, at most 2^22",
                static_cast<long long>(a.codes_stride));
  }
  if (a.m > 1 && a.out.stride[0] < a.n) return fail(M3_EINVAL, "m3_linear8: rows of out overlap");
  const int64_t tiles = (a.n + 63) / 64, es = elem_size(a.dtype);
  const char* o0 = static_cast<const char*>(a.out.ptr);
  const char* o1 = o0 + ((a.m - 1) * a.out.stride[0] + a.n) * es;
  const auto meets = [&](const void* p, int64_t bytes) {
    const char* p0 = static_cast<const char*>(p);
    return p0 < o1 && o0 < p0 + bytes;
  };
  if (meets(a.codes, (a.m - 1) * a.codes_stride + a.k) || meets(a.row_scales, a.m * 4) ||
      meets(a.q, tiles * ((a.k + 127) / 128) * 2 * kTileBytes) || meets(a.scales, tiles * 256)) {
    return fail(M3_EINVAL, "m3_linear8: out overlaps codes, the weight or scales");
  }
  const bool same = a.residual.ptr == a.out.ptr && (a.m == 1 || a.residual.stride[0] == a.out.stride[0]);
  if (present(a.residual) && !same && meets(a.residual.ptr, ((a.m - 1) * a.residual.stride[0] + a.n) * es)) {
    return fail(M3_EINVAL, "m3_linear8: out overlaps the residual without being it");
  }
  return M3_OK;
}

}  // namespace
}  // namespace m3

extern "C" int m3_linear8(const m3_linear8_args* args, hipStream_t stream) {
  using namespace m3;
  clear_error();
  if (args == nullptr) return fail(M3_EINVAL, "m3_linear8: NULL args");
  const m3_linear8_args& a = *args;
  const int rc = validate(a);
  if (rc != M3_OK) return rc;
  if (a.m == 0 || a.n == 0) return M3_OK;
  const Lin8Geom g{reinterpret_cast<const char*>(a.codes), a.row_scales,
                   reinterpret_cast<const char*>(a.q), a.scales, a.residual.ptr, a.out.ptr,
                   a.codes_stride, a.residual.stride[0], a.out.stride[0], a.m, static_cast<int>(a.n),
                   static_cast<int>(a.k), static_cast<int>((a.k + 127) / 128 * 2),
                   static_cast<int>((a.n + 63) / 64)};
  switch (a.dtype) {
    case M3_F32: return launch8<float>(g, stream);
    case M3_BF16: return launch8<__bf16>(g, stream);
    default: return launch8<_Float16>(g, stream);
  }
}
