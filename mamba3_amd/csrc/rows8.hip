// m3_rows8: rows rounded to 8-bit codes with one FP32 scale each, alone or behind the residual add and
// RMSNorm of m3_rms_norm: the operand of m3_linear8.
//
//   s = x (+ add, rounded to x's dtype), p = s * w (or x), most = max |p|
//   code = rint(127 p / most),  scale = most / 127 * rsqrt(mean s^2 + eps)   (no norm: most / 127)
//
// The norm's factor is one positive number a row, so it is no part of the codes: they need no second
// reduction, and no rounding of the factor moves one of them.
//
// A code is the exact quotient's nearest integer, ties to even: half of the greatest value, 63.5 codes,
// is a value that 16-bit rows do hold. p times 127 / most in FP32 is off by less than 1e-4 codes; a quotient
// nearer than that to a half is settled by the sign of 254 |p| - (2 k + 1) most in FP64, which is
// exact. One element in 5,000 is.
//
// Bound by memory: the row stays in registers between the two passes over it (its maximum, its codes), so
// x, add, the sum and the codes each move once. Measured (a large copy reaches 5.0 to 5.5 TB/s): 65536 x 1024 FP32 with
// a bf16 add and the sum kept 138 to 145 us (5.35 to 5.1 TB/s of what moves), 16384 x 2048 bf16 the same way 43 to 47.5
// us (5.5 to 4.95), 32768 x 4096 without norm f16 76 us (5.3), bf16 77 to 97 (5.2 to 4.2), FP32 118 (5.7), one row of 2048
// 3.5 us. Rows over 8,192 wide do not fit and are walked twice: 8192 x 16384 bf16 107 us (3.8), of FP32 with a bf16
// add, norm and sum 358 (4.1).
//
// m3_rows8_values, what the rows stand for, likewise: 32768 x 4096 to FP32 104 us (6.4 TB/s).
#include <hip/hip_runtime.h>

#include "m3_common.hpp"
#include "m3_host.hpp"

namespace m3 {
namespace {

constexpr int kChunk = 8;  // elements a lane takes at a time: 8 bytes of codes

// Workgroups of 256 for so many: a launch has below 2^32 work-items along x.
inline dim3 grid_of(int64_t blocks) {
  constexpr int64_t most = 1 << 23;
  return dim3(static_cast<unsigned>(blocks < most ? blocks : most), static_cast<unsigned>((blocks + most - 1) / most));
}
__device__ __forceinline__ int64_t block_index() {
  return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
}

struct Rows8Geom {
  const char* x;
  const char* add;   // or null
  const void* w;     // or null: no norm
  char* sum;         // or null
  int8_t* codes;
  float* scales;
  int64_t x_ld, a_ld, s_ld, c_ld;  // elements (codes: bytes)
  int rows, dim, w_dtype;
  float eps;
};

// Eight elements from `at` on, at any alignment.
template <typename T>
__device__ __forceinline__ void load8(const void* row, int at, float (&v)[kChunk]) {
  T t[kChunk];
  __builtin_memcpy(t, static_cast<const T*>(row) + at, sizeof(t));
#pragma unroll
  for (int e = 0; e < kChunk; ++e) v[e] = to_f(t[e]);
}

// What a row's values tell: the sum of squares, the bits of the greatest magnitude (as integers they
// order infinities and NaN above all others), and for products of FP32 values, which FP32 does not hold,
// the greatest one in FP64.
template <bool WIDE>
struct Seen {
  float sq;
  uint32_t bits;
  double wide;
  __device__ __forceinline__ void look(float s, float w, float p) {
    sq = fmaf(s, s, sq);
    bits = max(bits, __float_as_uint(p) & 0x7fffffffu);
    if constexpr (WIDE) wide = fmax(wide, fabs(static_cast<double>(s) * static_cast<double>(w)));
  }
  __device__ __forceinline__ void join(const Seen& o) {
    sq += o.sq;
    bits = max(bits, o.bits);
    if constexpr (WIDE) wide = fmax(wide, o.wide);
  }
  template <int LANES>
  __device__ __forceinline__ void join_lanes() {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      Seen other;
      other.sq = __shfl_xor(sq, o);
      other.bits = __shfl_xor(bits, o);
      other.wide = WIDE ? __shfl_xor(wide, o) : 0.0;
      join(other);
    }
  }
};

// One row of the call.
template <typename T, typename TA, bool NORM, bool ADD>
struct Row {
  const T* x;
  const TA* add;
  T* sum;  // or null
  const Rows8Geom& g;
  __device__ __forceinline__ Row(const Rows8Geom& geom, int64_t row)
      : x(reinterpret_cast<const T*>(geom.x) + row * geom.x_ld),
        add(ADD ? reinterpret_cast<const TA*>(geom.add) + row * geom.a_ld : nullptr),
        sum(ADD && geom.sum != nullptr ? reinterpret_cast<T*>(geom.sum) + row * geom.s_ld : nullptr),
        g(geom) {}

  // s of eight elements, from x's and add's, and of one
  __device__ __forceinline__ void sums(const T (&v)[kChunk], const TA (&a)[kChunk], float (&s)[kChunk]) const {
#pragma unroll
    for (int e = 0; e < kChunk; ++e) s[e] = ADD ? rnd<T>(to_f(v[e]) + to_f(a[e])) : to_f(v[e]);
  }
  __device__ __forceinline__ void load(int at, T (&v)[kChunk], TA (&a)[kChunk]) const {
    __builtin_memcpy(v, x + at, sizeof(v));
    if constexpr (ADD) __builtin_memcpy(a, add + at, sizeof(a));
  }
  __device__ __forceinline__ float sum_at(int at) const {
    float s = to_f(x[at]);
    if constexpr (ADD) s = rnd<T>(s + to_f(add[at]));
    return s;
  }
  __device__ __forceinline__ void keep(int at, const float (&s)[kChunk]) const {
    if (ADD && sum != nullptr) {
      T t[kChunk];
#pragma unroll
      for (int e = 0; e < kChunk; ++e) t[e] = from_f<T>(s[e]);
      __builtin_memcpy(sum + at, t, sizeof(t));
    }
  }
  // s once more, where this lane has stored it: it may have taken x's place
  __device__ __forceinline__ float again(int at) const {
    return ADD && sum != nullptr ? to_f(sum[at]) : sum_at(at);
  }
  __device__ __forceinline__ void again8(int at, float (&s)[kChunk]) const {
    if (ADD && sum != nullptr) {
      load8<T>(sum, at, s);
    } else {
      T v[kChunk];
      TA a[kChunk];
      load(at, v, a);
      sums(v, a, s);
    }
  }

  // the norm's weight, rounded to the rows' dtype
  __device__ __forceinline__ void weights(int at, float (&w)[kChunk]) const {
    if constexpr (NORM) {
      if (g.w_dtype == M3_F32) {
        load8<float>(g.w, at, w);
      } else if (g.w_dtype == M3_BF16) {
        load8<__bf16>(g.w, at, w);
      } else {
        load8<_Float16>(g.w, at, w);
      }
#pragma unroll
      for (int e = 0; e < kChunk; ++e) w[e] = rnd<T>(w[e]);
    }
  }
  __device__ __forceinline__ float weight_at(int at) const {
    return NORM ? rnd<T>(ldx(g.w, g.w_dtype, at)) : 1.f;
  }
};

// The row's own constants for its codes.
struct Scaled {
  float up, inv;  // q = p * up * inv; `up` lifts rows whose 127 / most would be infinite
  double most;
  float scale;
};

template <bool NORM, bool WIDE>
__device__ __forceinline__ Scaled scaled(const Seen<WIDE>& seen, int dim, float eps) {
  const float most = __uint_as_float(seen.bits);
  const bool bad = seen.bits >= 0x7f800000u;  // an infinity or NaN
  const float up = most < 0x1p-100f ? 0x1p100f : 1.f;
  const float inv = bad || seen.bits == 0 ? 0.f : 127.f / (most * up);
  const float norm = NORM ? rsqrtf(seen.sq / static_cast<float>(dim) + eps) : 1.f;
  return Scaled{up, inv, WIDE ? seen.wide : static_cast<double>(most),
                bad ? __uint_as_float(0x7fc00000u) : most / 127.f * norm};
}

// The code of p, and whether it is too near to a half to be told in FP32. A row that holds an infinity
// or NaN has inv = 0, and codes of 0.
__device__ __forceinline__ int code8(float p, const Scaled& c, bool& close) {
  const float q = p * c.up * c.inv, n = rintf(q);
  close = fabsf(q - n) > 0.4999f;
  return c.inv == 0.f ? 0 : static_cast<int>(n);
}

// The code of s * w by the sign of 254 |s w| - (2 k + 1) most, where k and k + 1 are in question.
__device__ __forceinline__ int settle(float s, float w, const Scaled& c) {
  const float q = s * w * c.up * c.inv, k = floorf(fabsf(q));
  const double p = fabs(static_cast<double>(s) * static_cast<double>(w)), odd = 2.0 * k + 1.0;
  const double half = odd * c.most, rest = fma(odd, c.most, -half);
  const double over = fma(254.0, p, -half) - rest;
  const int n = static_cast<int>(k), up = over > 0.0 || (over == 0.0 && (n & 1) != 0);
  return q < 0.f ? -(n + up) : n + up;
}

// TPR threads (16, a wave or the workgroup of 256) take a row. A lane holds the p of CH chunks of eight and, for
// dim % 8, of one element more; CH = 0 walks longer rows twice instead. All loads of a lane's row are issued
// before the first is used, those of chunks past its end from its last one; the norm's weight is rounded once a
// workgroup, in LDS (each row on its own took 56 in place of 48 us for 16384 x 2048).
template <typename T, typename TA, bool NORM, bool ADD, int TPR, int CH>
__global__ __launch_bounds__(256) void rows8_kernel(const Rows8Geom g) {
  constexpr bool kWide = NORM && sizeof(T) == 4;
  const int tid = threadIdx.x, lane = tid % TPR;
  const int64_t r = block_index() * (256 / TPR) + tid / TPR;
  const bool live = r < g.rows;
  const Row<T, TA, NORM, ADD> row(g, live ? r : g.rows - 1);
  const int whole = g.dim / kChunk, rest = g.dim % kChunk, end = kChunk * whole + lane;
  Seen<kWide> seen = {0.f, 0u, 0.0};
  float p[CH > 0 ? CH : 1][kChunk], last = 0.f;
  const auto look8 = [&](const float (&w)[kChunk], float (&s)[kChunk]) {  // leaves p in s
#pragma unroll
    for (int e = 0; e < kChunk; ++e) {
      const float v = NORM ? s[e] * w[e] : s[e];
      seen.look(s[e], NORM ? w[e] : 1.f, v);
      s[e] = v;
    }
  };
  if constexpr (CH > 0) {
    __shared__ __attribute__((aligned(16))) float weight[NORM ? TPR * CH * kChunk : 4];
    T v[CH][kChunk];
    TA a[CH][kChunk];
    if (whole > 0) {
#pragma unroll
      for (int j = 0; j < CH; ++j) row.load(kChunk * min(lane + TPR * j, whole - 1), v[j], a[j]);
    }
    if constexpr (NORM) {
      if (whole > 0) {
        constexpr int kEach = (TPR * CH + 255) / 256;  // chunks of the weight a lane
        float w[kEach][kChunk];
#pragma unroll
        for (int u = 0; u < kEach; ++u) row.weights(kChunk * min(tid + 256 * u, whole - 1), w[u]);
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
          if (tid + 256 * u < whole) __builtin_memcpy(weight + kChunk * (tid + 256 * u), w[u], sizeof(w[u]));
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int at = kChunk * (lane + TPR * j);
      if (at < kChunk * whole) {
        float w[kChunk];
        if constexpr (NORM) __builtin_memcpy(w, weight + at, sizeof(w));
        row.sums(v[j], a[j], p[j]);
        if (live) row.keep(at, p[j]);
        look8(w, p[j]);
      }
    }
  } else {
    for (int c = lane; c < whole; c += TPR) {
      T v[kChunk];
      TA a[kChunk];
      float w[kChunk];
      row.load(kChunk * c, v, a);
      row.weights(kChunk * c, w);
      row.sums(v, a, p[0]);
      if (live) row.keep(kChunk * c, p[0]);
      look8(w, p[0]);
    }
  }
  if (lane < rest) {
    const float s = row.sum_at(end), w = row.weight_at(end);
    if (ADD && row.sum != nullptr && live) row.sum[end] = from_f<T>(s);
    last = s * w;
    seen.look(s, w, last);
  }
  seen.template join_lanes<TPR < 64 ? TPR : 64>();
  if constexpr (TPR > 64) {
    __shared__ Seen<kWide> parts[4];
    if ((tid & 63) == 0) parts[tid >> 6] = seen;
    __syncthreads();
    seen = parts[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) seen.join(parts[i]);
  }
  if (!live) return;
  const Scaled c = scaled<NORM, kWide>(seen, g.dim, g.eps);
  int8_t* const codes = g.codes + r * g.c_ld;
  const auto code_chunk = [&](int at, const float (&v)[kChunk]) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    u32x2 words = {0u, 0u};
    unsigned open = 0;  // the elements in question
#pragma unroll
    for (int e = 0; e < kChunk; ++e) {
      bool close;
      const int n = code8(v[e], c, close);
      words[e / 4] |= static_cast<uint32_t>(n & 0xff) << (8 * (e % 4));
      open |= close ? 1u << e : 0u;
    }
    *reinterpret_cast<u32x2*>(codes + at) = words;
    while (open != 0) {
      const int k = at + __builtin_ctz(open);
      open &= open - 1;
      codes[k] = static_cast<int8_t>(settle(row.again(k), row.weight_at(k), c));
    }
  };
  if constexpr (CH > 0) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if (lane + TPR * j < whole) code_chunk(kChunk * (lane + TPR * j), p[j]);
    }
  } else {
    for (int j = lane; j < whole; j += TPR) {
      float w[kChunk];
      row.again8(kChunk * j, p[0]);
      row.weights(kChunk * j, w);
#pragma unroll
      for (int e = 0; e < kChunk; ++e) p[0][e] = NORM ? p[0][e] * w[e] : p[0][e];
      code_chunk(kChunk * j, p[0]);
    }
  }
  if (lane < rest) {
    bool close;
    int n = code8(last, c, close);
    if (close) n = settle(row.again(end), row.weight_at(end), c);
    codes[end] = static_cast<int8_t>(n);
  }
  if (lane == 0) g.scales[r] = c.scale;
}

// code * scale in FP32, rounded to T: what the rows stand for. A lane writes 16 bytes; LANES lanes take a row.
template <typename T>
__global__ __launch_bounds__(256) void values8_kernel(const int8_t* codes, int64_t c_ld, const float* scales,
                                                      T* out, int64_t o_ld, int rows, int dim, int lanes_log2) {
  constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int64_t row = (block_index() << (8 - lanes_log2)) + (threadIdx.x >> lanes_log2);
  if (row >= rows) return;
  const float scale = scales[row];
  const int8_t* const from = codes + row * c_ld;
  T* const to = out + row * o_ld;
#pragma unroll 4
  for (int at = kPiece * lane; at < dim; at += kPiece * lanes) {
    if (at + kPiece <= dim) {
      int8_t c[kPiece];
      __builtin_memcpy(c, from + at, sizeof(c));
      T t[kPiece];
#pragma unroll
      for (int e = 0; e < kPiece; ++e) t[e] = from_f32<T>(static_cast<float>(c[e]) * scale);
      __builtin_memcpy(to + at, t, sizeof(t));
    } else {
      for (int e = at; e < dim; ++e) to[e] = from_f32<T>(static_cast<float>(from[e]) * scale);
    }
  }
}

template <typename T>
int launch_values(const m3_rows8_values_args& a, hipStream_t stream) {
  constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
  int log2 = 0;
  while (log2 < 8 && (kPiece << log2) < a.dim) ++log2;
  const int64_t per = 256 >> log2;
  hipLaunchKernelGGL(values8_kernel<T>, grid_of((a.rows + per - 1) / per), dim3(256), 0, stream, a.codes,
                     a.codes_stride, a.scales, static_cast<T*>(a.out.ptr), a.out.stride[0],
                     static_cast<int>(a.rows), static_cast<int>(a.dim), log2);
  return check_launch("m3_rows8_values");
}

template <typename T, typename TA, bool NORM, bool ADD, int TPR, int CH>
int launch_one(const Rows8Geom& g, hipStream_t stream) {
  constexpr int64_t rows = 256 / TPR;
  hipLaunchKernelGGL((rows8_kernel<T, TA, NORM, ADD, TPR, CH>), grid_of((g.rows + rows - 1) / rows), dim3(256), 0,
                     stream, g);
  return check_launch("m3_rows8");
}

template <typename T, typename TA, bool NORM, bool ADD>
int launch_dim(const Rows8Geom& g, hipStream_t stream) {
  const int chunks = (g.dim + kChunk - 1) / kChunk;
  if (chunks <= 16) return launch_one<T, TA, NORM, ADD, 16, 1>(g, stream);
  if (chunks <= 32) return launch_one<T, TA, NORM, ADD, 16, 2>(g, stream);
  if (chunks <= 64) return launch_one<T, TA, NORM, ADD, 64, 1>(g, stream);
  if (chunks <= 128) return launch_one<T, TA, NORM, ADD, 64, 2>(g, stream);
  if (chunks <= 256) return launch_one<T, TA, NORM, ADD, 64, 4>(g, stream);
  if (chunks <= 512) return launch_one<T, TA, NORM, ADD, 256, 2>(g, stream);
  if (chunks <= 1024) return launch_one<T, TA, NORM, ADD, 256, 4>(g, stream);
  return launch_one<T, TA, NORM, ADD, 256, 0>(g, stream);
}

template <typename T>
int launch_type(const Rows8Geom& g, int add_dtype, hipStream_t stream) {
  if (g.w == nullptr) return launch_dim<T, T, false, false>(g, stream);
  if (g.add == nullptr) return launch_dim<T, T, true, false>(g, stream);
  if constexpr (sizeof(T) == 4) {
    if (add_dtype == M3_BF16) return launch_dim<T, __bf16, true, true>(g, stream);
    if (add_dtype == M3_F16) return launch_dim<T, _Float16, true, true>(g, stream);
  }
  return launch_dim<T, T, true, true>(g, stream);
}

struct Range {
  const char *from, *to;
};

Range range(const m3_tensor& t, int64_t rows, int64_t dim) {
  const char* p = static_cast<const char*>(t.ptr);
  return {p, p == nullptr ? p : p + ((rows - 1) * t.stride[0] + dim) * elem_size(t.dtype)};
}

bool meets(const Range& a, const Range& b) {
  return a.from != nullptr && b.from != nullptr && a.from < b.to && b.from < a.to;
}

int check_sizes(const char* name, int64_t rows, int64_t dim) {
  if (rows < 0 || dim < 0) return fail(M3_EINVAL, "%s: negative dimensions", name);
  if (rows >= (1 << 30) || dim > M3_LINEAR8_MAX_K) {
    return fail(M3_EUNSUPPORTED, "%s: %lld rows of %lld: below 2^30, of at most %d", name,
                static_cast<long long>(rows), static_cast<long long>(dim), M3_LINEAR8_MAX_K);
  }
  if (rows != 0 && dim == 0) return fail(M3_EUNSUPPORTED, "%s: dim 0", name);
  return M3_OK;
}

int check_codes(const char* name, const int8_t* codes, int64_t stride, const float* scales, int64_t dim, int by) {
  if (codes == nullptr || scales == nullptr) return fail(M3_EINVAL, "%s: codes or scales are NULL", name);
  if (reinterpret_cast<uintptr_t>(codes) % by != 0 || stride % by != 0 ||
      reinterpret_cast<uintptr_t>(scales) % 4 != 0) {
    return fail(M3_EUNSUPPORTED, "%s: rows of codes must be %d-byte aligned, scales 4-byte", name, by);
  }
  if (stride < dim) return fail(M3_EINVAL, "%s: rows of codes overlap", name);
  return M3_OK;
}

int validate(const m3_rows8_args& a) {
  int rc;
  if ((rc = check_sizes("m3_rows8", a.rows, a.dim)) || a.rows == 0) return rc;
  if ((rc = check_tensor(a.x, "x", 2, a.dim, true, -1)) ||
      (rc = check_tensor(a.weight, "weight", 1, a.dim, false, -1)) ||
      (rc = check_tensor(a.add, "add", 2, a.dim, false, a.x.dtype == M3_F32 ? -1 : a.x.dtype)) ||
      (rc = check_tensor(a.sum_out, "sum_out", 2, a.dim, false, a.x.dtype))) {
    return rc;
  }
  if (present(a.add) && !present(a.weight)) return fail(M3_EINVAL, "m3_rows8: add needs weight");
  if (present(a.sum_out) && !present(a.add)) return fail(M3_EINVAL, "m3_rows8: sum_out needs add");
  if (present(a.weight) && !(a.eps >= 0.f)) return fail(M3_EINVAL, "m3_rows8: eps must be >= 0");
  if ((rc = check_codes("m3_rows8", a.codes, a.codes_stride, a.scales, a.dim, 16))) return rc;
  const int64_t whole = (a.dim + 15) / 16 * 16;
  if (a.rows > 1 && present(a.sum_out) && a.sum_out.stride[0] < a.dim) {
    return fail(M3_EINVAL, "m3_rows8: rows of sum_out overlap");
  }
  const char* c = reinterpret_cast<const char*>(a.codes);
  const char* f = reinterpret_cast<const char*>(a.scales);
  const Range x = range(a.x, a.rows, a.dim), add = range(a.add, a.rows, a.dim),
              w = range(a.weight, 1, a.dim), sum = range(a.sum_out, a.rows, a.dim),
              codes = {c, c + (a.rows - 1) * a.codes_stride + whole}, scales = {f, f + a.rows * 4};
  for (const Range* r : {&x, &add, &w, &sum}) {
    if (meets(*r, codes) || meets(*r, scales)) {
      return fail(M3_EINVAL, "m3_rows8: codes or scales overlap another tensor");
    }
  }
  if (meets(codes, scales)) return fail(M3_EINVAL, "m3_rows8: codes overlap scales");
  // s may take the place of x or of an add of its dtype: each element is read before it is written
  const auto in_place = [&](const m3_tensor& t) {
    return t.ptr == a.sum_out.ptr && t.dtype == a.sum_out.dtype &&
           (a.rows == 1 || t.stride[0] == a.sum_out.stride[0]);
  };
  if ((meets(sum, x) && !in_place(a.x)) || (meets(sum, add) && !in_place(a.add)) || meets(sum, w)) {
    return fail(M3_EINVAL, "m3_rows8: sum_out overlaps an input without being it");
  }
  return M3_OK;
}

int validate(const m3_rows8_values_args& a) {
  int rc;
  if ((rc = check_sizes("m3_rows8_values", a.rows, a.dim)) || a.rows == 0) return rc;
  if ((rc = check_codes("m3_rows8_values", a.codes, a.codes_stride, a.scales, a.dim, 1)) ||
      (rc = check_tensor(a.out, "out", 2, a.dim, true, -1))) {
    return rc;
  }
  if (a.rows > 1 && a.out.stride[0] < a.dim) return fail(M3_EINVAL, "m3_rows8_values: rows of out overlap");
  const char* c = reinterpret_cast<const char*>(a.codes);
  const char* f = reinterpret_cast<const char*>(a.scales);
  const Range out = range(a.out, a.rows, a.dim);
  if (meets(out, {c, c + (a.rows - 1) * a.codes_stride + a.dim}) || meets(out, {f, f + a.rows * 4})) {
    return fail(M3_EINVAL, "m3_rows8_values: out overlaps codes or scales");
  }
  return M3_OK;
}

}  // namespace
}  // namespace m3

extern "C" int m3_rows8_values(const m3_rows8_values_args* args, hipStream_t stream) {
  using namespace m3;
  clear_error();
  if (args == nullptr) return fail(M3_EINVAL, "m3_rows8_values: NULL args");
  const int rc = validate(*args);
  if (rc != M3_OK) return rc;
  if (args->rows == 0) return M3_OK;
  switch (args->out.dtype) {
    case M3_F32: return launch_values<float>(*args, stream);
    case M3_BF16: return launch_values<__bf16>(*args, stream);
    default: return launch_values<_Float16>(*args, stream);
  }
}

extern "C" int m3_rows8(const m3_rows8_args* args, hipStream_t stream) {
  using namespace m3;
  clear_error();
  if (args == nullptr) return fail(M3_EINVAL, "m3_rows8: NULL args");
  const m3_rows8_args& a = *args;
  const int rc = validate(a);
  if (rc != M3_OK) return rc;
  if (a.rows == 0) return M3_OK;
  const Rows8Geom g{static_cast<const char*>(a.x.ptr), static_cast<const char*>(a.add.ptr), a.weight.ptr,
                    static_cast<char*>(a.sum_out.ptr), a.codes, a.scales,
                    a.x.stride[0], a.add.stride[0], a.sum_out.stride[0], a.codes_stride,
                    static_cast<int>(a.rows), static_cast<int>(a.dim), a.weight.dtype, a.eps};
  switch (a.x.dtype) {
    case M3_F32: return launch_type<float>(g, a.add.dtype, stream);
    case M3_BF16: return launch_type<__bf16>(g, a.add.dtype, stream);
    default: return launch_type<_Float16>(g, a.add.dtype, stream);
  }
}
