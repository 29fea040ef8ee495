// m3_linear8: out[M, N] = (sum_k codes[m, k] q[n, k]) row_scale[m] scale[n] (+ residual), codes and q in 8
// bits, on the integer matrix instructions (16x16x64, twice bf16's rate): the projections of any number
// of rows.
//
// The sums are exact in 32 bits (K < 2^17), so their order is free and every kernel gives the same bits; each
// output then has three FP32 roundings (of the sum and of two products, the second one with the residual) and its own.
//
// The weight is an instruction's first operand: a lane of its result holds four consecutive columns n of one
// row m. The weight's tiles order their 64 rows so that two results side by side are eight columns, 16 bytes of
// a 16-bit output, and four lanes 64 bytes.
//
// linear8_rows_kernel (few rows, or little work): a workgroup's waves take every WAVES-th tile of 64
// columns, both operands straight into registers, and their sums meet in LDS. Bound by the weight's stream, or
// the launch and a few latencies of memory: 28672 x 8192 at 1 row 39.4 us (6 TB/s, in part from the last-level
// cache), 8672 x 2048 at 1 row 5.3 us, 2048 x 4096 at 16 rows 5.8 us.
//
// linear8_tile_kernel (the rest): below. Where K is long 8192 x 28672 x 8192 takes 1,300 to 1,360 us, 2.96 POP/s in
// the quickest: the matrix units are busy 77% of the cycles at 1.83 GHz, which is nearly the clock that products of such
// values alone, without a load, run at here (3.95 POP/s; 4.87 of zeros; a library's product of int8 2.30). Bound by
// what the units wait for in the other 23%. Where K is short (65536 x 4480 x 1024: 264 to 285 us, units busy 59%),
// also by what is written (587 MB) and the rounding of the outputs.
#include <hip/hip_runtime.h>

#include "m3_common.hpp"
#include "m3_host.hpp"

namespace m3 {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kCus = 256;
constexpr unsigned kBand = 8;  // tiles along M that an XCD takes before the next column
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
  bool aligned;     // rows of codes: 16-byte aligned, readable to the next multiple of 16
  bool whole;       // out and residual in 16 bytes at a time: aligned, N a multiple, a tile's offsets 32-bit
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

// The codes of the rows from m0 on, up to `rows` of them: the extent ends with the last one's codes, so that rows
// past M read 0. What a row reads past K, of the next row, meets zeros of the weight.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t codes_rsrc(const Lin8Geom& g, int64_t m0, int rows) {
  const int64_t left = g.m - m0 < rows ? g.m - m0 : rows;
  return rsrc8(g.codes + m0 * g.c_ld, (left - 1) * g.c_ld + (g.k + 15) / 16 * 16);
}

// COUNT values of a row of the residual from column n on; past its end 0.
template <typename T, int COUNT>
__device__ __forceinline__ void load_res(const T* row, int n, int end, float (&v)[COUNT]) {
  if (n + COUNT <= end) {
    T t[COUNT];
    __builtin_memcpy(t, row + n, sizeof(t));
#pragma unroll
    for (int e = 0; e < COUNT; ++e) v[e] = to_f(t[e]);
  } else {
#pragma unroll
    for (int e = 0; e < COUNT; ++e) v[e] = n + e < end ? to_f(row[n + e]) : 0.f;
  }
}

// An output before its rounding to T, the same operations in every kernel.
template <bool RES>
__device__ __forceinline__ float scaled(int sum, float rs, float sc, float res) {
  const float v = static_cast<float>(sum) * rs;
  return RES ? fmaf(v, sc, res) : v * sc;
}

// COUNT (4 or 8) consecutive outputs of one row from column n on, at any alignment.
template <typename T, int COUNT>
__device__ __forceinline__ void put(const Lin8Geom& g, int64_t m, int n, float rs, const i4* sums) {
  float res[COUNT];
  T y[COUNT];
  if (g.res != nullptr) load_res(static_cast<const T*>(g.res) + m * g.r_ld, n, g.n, res);
#pragma unroll
  for (int e = 0; e < COUNT; e += 4) {
    const f4 sc = *reinterpret_cast<const f4*>(g.scales + n + e);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int sum = sums[e / 4][r];
      y[e + r] = from_f32<T>(g.res != nullptr ? scaled<true>(sum, rs, sc[r], res[e + r])
                                              : scaled<false>(sum, rs, sc[r], 0.f));
    }
  }
  T* const out = static_cast<T*>(g.out) + m * g.o_ld + n;
  if (n + COUNT <= g.n) {
    __builtin_memcpy(out, y, sizeof(y));
  } else {
#pragma unroll
    for (int e = 0; e < COUNT; ++e) {
      if (n + e < g.n) out[e] = y[e];
    }
  }
}

// 16 codes at column `at` of row m, at any alignment. Those past the row's end meet zeros of the weight; past the last
// row's they are not read.
__device__ __forceinline__ i4 load_codes(const Lin8Geom& g, int64_t m, int at) {
  const char* p = g.codes + m * g.c_ld + at;
  const int64_t left = (g.m - 1 - m) * g.c_ld + g.k - at;
  i4 v = {0, 0, 0, 0};
  if (left >= 16) {
    __builtin_memcpy(&v, p, sizeof(v));
  } else {
    for (int e = 0; e < left; ++e) {
      v[e / 4] |= static_cast<int>(static_cast<uint32_t>(static_cast<uint8_t>(p[e])) << (8 * (e % 4)));
    }
  }
  return v;
}

// MT blocks of 16 rows by TN quarters of a tile's 64 columns of out (1 or 4); AHEAD tiles of K on their way at
// a time. Rows past M read 0. ONCE: no other workgroup reads these of the weight's rows, and they need not stay in
// the L2. ALIGNED: rows of codes are 16-byte aligned and readable to the next multiple of 16.
template <typename T, int MT, int TN, int WAVES, int AHEAD, bool ONCE, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES) void linear8_rows_kernel(const Lin8Geom g) {
  __shared__ i4 parts[WAVES][MT * TN][64];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile = blockIdx.x * TN >> 2, quarter = blockIdx.x * TN & 3;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  const __amdgpu_buffer_rsrc_t rc = codes_rsrc(g, m0, 16 * MT);
  const __amdgpu_buffer_rsrc_t rq =
      rsrc8(g.q + static_cast<int64_t>(tile) * g.tk * kTileBytes, static_cast<int64_t>(g.tk) * kTileBytes);
  i4 acc[TN][MT];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = i4{0, 0, 0, 0};
  }
  const unsigned xoff = l16 * static_cast<unsigned>(g.c_ld) + 16 * lg, xrow = 16 * static_cast<unsigned>(g.c_ld);
  const unsigned qoff = quarter * 1024 + lane * 16;
  const int tiles = (g.k + 63) / 64;
  // whether any lane's codes could lie past the last row's: then each asks
  const char* const from = g.codes + (m0 + l16) * g.c_ld + 16 * lg;
  const bool careful = (m0 + 16 * MT - 1) * g.c_ld + tiles * 64 > (g.m - 1) * g.c_ld + g.k;
  for (int t0 = w; t0 < tiles; t0 += WAVES * AHEAD) {
    i4 a[AHEAD][TN], b[AHEAD][MT];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int t = t0 + u * WAVES;
      const bool live = t < tiles;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        a[u][j] = __builtin_bit_cast(i4, __builtin_amdgcn_raw_buffer_load_b128(
            rq, live ? qoff + j * 1024 + t * kTileBytes : kNowhere, 0, ONCE ? 2 : 0));
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if constexpr (ALIGNED) {
          b[u][i] = __builtin_bit_cast(i4, __builtin_amdgcn_raw_buffer_load_b128(
              rc, live ? xoff + i * xrow + t * 64 : kNowhere, 0, 0));
        } else if (careful) {
          const int64_t m = m0 + 16 * i + l16;
          b[u][i] = live && m < g.m ? load_codes(g, m, t * 64 + 16 * lg) : i4{0, 0, 0, 0};
        } else {
          __builtin_memcpy(&b[u][i], from + (16 * i) * g.c_ld + min(t, tiles - 1) * 64, sizeof(i4));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[j][i] = mma(a[u][j], b[u][i], acc[j][i]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < TN; ++j) {
#pragma unroll
    for (int i = 0; i < MT; ++i) parts[w][i * TN + j][lane] = acc[j][i];
  }
  __syncthreads();
  constexpr int kWide = TN > 1 ? 2 : 1;
  for (int p = w; p < MT * TN / kWide; p += WAVES) {
    i4 sum[kWide];
#pragma unroll
    for (int e = 0; e < kWide; ++e) {
      sum[e] = parts[0][p * kWide + e][lane];
#pragma unroll
      for (int v = 1; v < WAVES; ++v) sum[e] += parts[v][p * kWide + e][lane];
    }
    const int i = p * kWide / TN, j = quarter + p * kWide % TN;
    const int64_t m = m0 + 16 * i + l16;
    const int n = 64 * tile + 32 * (j >> 1) + 4 * (j & 1) + 8 * lg;
    if (m < g.m && n < g.n) put<T, 4 * kWide>(g, m, n, g.row_scales[m], sum);
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

// Of what is on its way from memory all but the last LATER have arrived, for all waves, and what they read from
// LDS was read.
template <int LATER>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
}

__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, char* dst, unsigned off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16,
                                           static_cast<int>(off), 0, 0, 0);
}

// Neighbouring lanes hold rows 2 t (even lane) and 2 t + 1, two pieces of 16 bytes each that lie next to one another
// over four lanes. After the exchange `first` of both lanes is row 2 t and `second` row 2 t + 1, the even
// lane's their first pieces: a store then writes whole lines of 128 bytes. Stores of half lines reach 2.1 TB/s here,
// these 4 and more.
__device__ __forceinline__ void exchange(bool odd, u32x4& first, u32x4& second) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t got = __builtin_amdgcn_mov_dpp(odd ? first[e] : second[e], 0xb1, 0xf, 0xf, true);
    first[e] = odd ? got : first[e];
    second[e] = odd ? second[e] : got;
  }
}

// A piece of a row's outputs, at any alignment; the row ends at column `end`.
template <typename T>
__device__ __forceinline__ void store_piece(T* row, int n, int end, const u32x4& piece) {
  constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
  if (n + kPiece <= end) {
    __builtin_memcpy(row + n, &piece, sizeof(piece));
  } else {
    T t[kPiece];
    __builtin_memcpy(t, &piece, sizeof(t));
#pragma unroll
    for (int e = 0; e < kPiece; ++e) {
      if (n + e < end) row[n + e] = t[e];
    }
  }
}

// A workgroup of WM x WN waves, each 16 XI rows by 64 columns, takes tile after tile and walks K in steps of 128.
// A step's codes go from memory into one of two LDS stages without passing through registers, rows of 128
// bytes whose eight pieces of 16 are exchanged by the row's low bits: eight lanes that read one column's
// pieces of eight rows meet all banks. The weight's operands, which few waves share, come straight into
// registers: LDS then moves half as much. In each half of a step the products of one half are under way while
// the codes of the next are read and each operand of the weight is followed by the next step's; one barrier a
// step. The next tile's first step is on its way while a tile is written.
//
// WHOLE: out is written by every lane in 16 bytes at a time, what lies outside past the extent, so that the number
// of stores is known. Else rows may lie at any alignment and end within a piece.
//
// KS: groups of WM x WN waves that take every KS-th step of K, each with stages of its own; the others' sums
// go to the first through LDS. Such a workgroup takes one tile.
template <typename T, int WM, int WN, int XI, int KS, bool WHOLE, bool RES>
__global__ __launch_bounds__(64 * WM * WN * KS, 2) void linear8_tile_kernel(const Lin8Geom g, unsigned tiles_m,
                                                                         unsigned tiles_n, unsigned band) {
  constexpr int kWaves = WM * WN, BM = 16 * XI * WM, kStage = BM * 128, kUnits = BM / 8 / kWaves;
  constexpr int kSums = (KS - 1) * kWaves * 4 * XI * 1024, kLds = 2 * KS * kStage > kSums ? 2 * KS * kStage : kSums;
  static_assert(BM / 8 % kWaves == 0 && XI % 4 == 0, "whole units and reads for each wave");
  __shared__ __attribute__((aligned(128))) char lds[kLds];
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = KS == 1 ? 0 : wave / kWaves;
  const int w = KS == 1 ? wave : wave % kWaves, wm = w / WN, wn = w % WN;
  char* const stages = lds + part * 2 * kStage;
  const unsigned all = tiles_m * tiles_n;
  const int64_t row_bytes = static_cast<int64_t>(g.tk) * kTileBytes;
  const int all_steps = g.tk / 2, steps = (all_steps + KS - 1) / KS;

  // The codes' loads, units of 8 rows (1 KB), and where they have come to. Rows past M lie past the extent,
  // and so does everything after the last tile.
  __amdgpu_buffer_rsrc_t rc;
  unsigned coff, c_id = blockIdx.x;
  int c_step = 0;
  const unsigned unit = 8 * kWaves * static_cast<unsigned>(g.c_ld);
  const auto aim_codes = [&]() {
    const int64_t m0 = place(min(c_id, all - 1), tiles_m, tiles_n, band).m * BM;
    const int64_t left = g.m - m0 < BM ? g.m - m0 : BM;
    rc = rsrc8(g.codes + m0 * g.c_ld, c_id < all ? (left - 1) * g.c_ld + (g.k + 15) / 16 * 16 : 0);
    coff = (8 * w + (lane >> 3)) * static_cast<unsigned>(g.c_ld) + 16 * ((lane & 7) ^ (lane >> 3)) +
           128 * part;
  };
  const auto fetch = [&](int stage) {
#pragma unroll
    for (int v = 0; v < kUnits; ++v) load_lds(rc, stages + stage + (v * kWaves + w) * 1024, coff + v * unit);
    coff += 128 * KS;
    if (++c_step == steps) {
      c_step = 0;
      c_id += gridDim.x;
      aim_codes();
    }
  };

  // The same of the weight's operands; tile rows past N lie past the extent, and a step that a group has past
  // the last one does too: its products are 0.
  __amdgpu_buffer_rsrc_t rq;
  unsigned qoff, q_id = blockIdx.x;
  int q_step = 0;
  const auto aim_weight = [&]() {
    const int tile0 = place(min(q_id, all - 1), tiles_m, tiles_n, band).n * WN;
    rq = rsrc8(g.q + tile0 * row_bytes, q_id < all ? min(WN, g.tiles - tile0) * row_bytes : 0);
    qoff = part < all_steps ? (wn * static_cast<unsigned>(row_bytes) + 2 * kTileBytes * part) + lane * 16 : kNowhere;
  };
  const auto step_weight = [&]() {
    qoff += 2 * kTileBytes * KS;
    if (KS > 1 && (q_step + 1) * KS + part >= all_steps) qoff = kNowhere;
    if (++q_step == steps) {
      q_step = 0;
      q_id += gridDim.x;
      aim_weight();
    }
  };

  i4 acc[4][XI], a[2][4], b[2][XI];
  const auto weight = [&](int kk, int j) {
    a[kk][j] = __builtin_bit_cast(
        i4, __builtin_amdgcn_raw_buffer_load_b128(rq, qoff + (4 * kk + j) * 1024, 0, 0));
  };
  const char* const rows = stages + (16 * XI * wm + l16) * 128;
  const int piece[2] = {16 * (lg ^ (l16 & 7)), 16 * ((4 + lg) ^ (l16 & 7))};
  const auto read = [&](int stage, int kk, int i) {
    b[kk][i] = *reinterpret_cast<const i4*>(rows + stage + piece[kk] + i * 2048);
  };
  // half kk of a step; `stage` holds the half after it
  const auto half = [&](int kk, int stage) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < XI; ++i) acc[j][i] = mma(a[kk][j], b[kk][i], acc[j][i]);
      weight(kk, j);
#pragma unroll
      for (int i = 0; i < XI / 4; ++i) read(stage, 1 - kk, j * (XI / 4) + i);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < XI / 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // a read from LDS
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);  // products
      }
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // a load
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  aim_codes();
  aim_weight();
  fetch(0);
#pragma unroll
  for (int j = 0; j < 4; ++j) weight(0, j);
  stage_barrier<0>();
  int now = 0;
  fetch(kStage);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < 4; ++j) weight(1, j);
  step_weight();
  // loads and stores count down in the order of their issue: after a stage's fetch come the weight's 8 loads
  // in the two halves until it is needed, and at a tile's first step the stores of the tile before
  constexpr int kStores = (sizeof(T) == 4 ? 4 : 2) * XI;
  bool stored = false;
  for (unsigned id = blockIdx.x; id < all; id += gridDim.x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < XI; ++i) acc[j][i] = i4{0, 0, 0, 0};
    }
    // (once more after a tile before, whose last half has read them: they are not kept while it is written)
#pragma unroll
    for (int i = 0; i < XI; ++i) read(now, 0, i);
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      half(0, now);
      if (stored) {
        stored = false;
        stage_barrier<8 + kStores>();
      } else {
        stage_barrier<8>();
      }
      __builtin_amdgcn_sched_barrier(0);
      fetch(now);
      __builtin_amdgcn_sched_barrier(0);
      now = kStage - now;
      half(1, now);
      step_weight();
    }
    if constexpr (KS > 1) {
      i4* const sums = reinterpret_cast<i4*>(lds) + lane;
      stage_barrier<0>();  // of the fetches past the last step, too
      if (part > 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int i = 0; i < XI; ++i) sums[(((part - 1) * kWaves + w) * 4 * XI + j * XI + i) * 64] = acc[j][i];
        }
      }
      __syncthreads();
      if (part > 0) return;
#pragma unroll
      for (int u = 0; u < KS - 1; ++u) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int i = 0; i < XI; ++i) acc[j][i] += sums[((u * kWaves + w) * 4 * XI + j * XI + i) * 64];
        }
      }
    }
    const Place at = place(id, tiles_m, tiles_n, band);
    const int64_t m0 = at.m * BM;
    const int left = static_cast<int>(g.m - m0 < BM ? g.m - m0 : BM);  // rows
    const int m1 = 16 * XI * wm + l16, n0 = 64 * (at.n * WN + wn) + 8 * lg;
    // the scales before the first store: a wait for them waits for every store before them
    f4 sc[4];
    float rs[XI];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 32 * (j >> 1) + 4 * (j & 1);
      sc[j] = n < g.n ? *reinterpret_cast<const f4*>(g.scales + n) : f4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < XI; ++i) rs[i] = g.row_scales[m0 + min(m1 + 16 * i, left - 1)];
    T* const out = static_cast<T*>(g.out);
    __amdgpu_buffer_rsrc_t ro;
    if constexpr (WHOLE) {
      ro = rsrc8(out + m0 * g.o_ld, ((left - 1) * g.o_ld + g.n) * static_cast<int64_t>(sizeof(T)));
    }
    constexpr int kPiece = 16 / static_cast<int>(sizeof(T));  // elements
    const bool odd = (lane & 1) != 0;
    // out is not read again here: kept out of the L2 it leaves that to codes and weight (65536 x 4480 x 1024 294 -> 264
    // us, the next kernel that reads it 10 us more); the few outputs of tiles with K in parts gain nothing by it
    constexpr int kStream = KS == 1 ? 2 : 0;
    // the residual, as many blocks of rows at a time as the registers hold, before the stores of these
    constexpr int kBatch = RES && WHOLE ? 2 * XI / (8 / kPiece) / 4 : 1;
    u32x4 held[kBatch][2][8 / kPiece];
    __amdgpu_buffer_rsrc_t rr;
    unsigned from = 0, pitch_r = 0;
    if constexpr (RES && WHOLE) {
      rr = rsrc8(static_cast<const T*>(g.res) + m0 * g.r_ld,
                 ((left - 1) * g.r_ld + g.n) * static_cast<int64_t>(sizeof(T)));
      pitch_r = static_cast<unsigned>(g.r_ld) * static_cast<unsigned>(sizeof(T));
      from = m1 * pitch_r + n0 * static_cast<unsigned>(sizeof(T));
    }
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const int m = m1 + 16 * i;
      if constexpr (RES && WHOLE) {
        if (i % kBatch == 0) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int p = 0; p < 8 / kPiece; ++p) {
                held[u][h][p] = __builtin_amdgcn_raw_buffer_load_b128(
                    rr, from + 16 * (i + u) * pitch_r + 32 * h * static_cast<unsigned>(sizeof(T)) + 16 * p, 0, 0);
              }
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      u32x4 y[2][8 / kPiece];  // [half of the 64 columns][pieces of 16 bytes]
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
        T t[8];
        if constexpr (RES && WHOLE) {
          T r[8];
          __builtin_memcpy(r, held[i % kBatch][h], sizeof(r));
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = to_f(r[e]);
        } else if constexpr (RES) {
          load_res(static_cast<const T*>(g.res) + (m0 + min(m, left - 1)) * g.r_ld, n0 + 32 * h, g.n, v);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          t[e] = from_f32<T>(scaled<RES>(acc[2 * h + e / 4][i][e % 4], rs[i], sc[2 * h + e / 4][e % 4],
                                         RES ? v[e] : 0.f));
        }
        __builtin_memcpy(y[h], t, sizeof(t));
      }
#pragma unroll
      for (int p = 0; p < 8 / kPiece; ++p) {
        // 16 bits: the halves' pieces; FP32: the two of a half
        u32x4 first = y[kPiece == 4 ? p : 0][0], second = y[kPiece == 4 ? p : 1][8 / kPiece - 1];
        exchange(odd, first, second);
        const int n = kPiece == 4 ? n0 + 32 * p + (odd ? 4 : 0) : n0 + (odd ? 32 : 0), m2 = m - odd;
        if constexpr (WHOLE) {
          const unsigned pitch = static_cast<unsigned>(g.o_ld) * static_cast<unsigned>(sizeof(T));
          const unsigned to = m2 * pitch + n * static_cast<unsigned>(sizeof(T));
          __builtin_amdgcn_raw_buffer_store_b128(first, ro, n < g.n && m2 < left ? to : kNowhere, 0, kStream);
          __builtin_amdgcn_raw_buffer_store_b128(second, ro, n < g.n && m2 + 1 < left ? to + pitch : kNowhere, 0,
                                                 kStream);
        } else {
          T* const to = out + (m0 + m2) * g.o_ld;
          if (m2 < left) store_piece(to, n, g.n, first);
          if (m2 + 1 < left) store_piece(to + g.o_ld, n, g.n, second);
        }
      }
      // one block's addresses (and residual) at a time: more would not fit the registers
      if constexpr (!WHOLE) __builtin_amdgcn_sched_barrier(0);
    }
    stored = WHOLE;
  }
  // the fetches past the last tile write (zeros) to LDS, too: none is left behind
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <typename T, int MT, int TN, int WAVES, int AHEAD>
int launch_rows(const Lin8Geom& g, hipStream_t stream) {
  const dim3 grid(4 / TN * g.tiles, static_cast<unsigned>((g.m + 16 * MT - 1) / (16 * MT)));
  const auto kernel =
      g.aligned ? (grid.y == 1 ? linear8_rows_kernel<T, MT, TN, WAVES, AHEAD, true, true>
                               : linear8_rows_kernel<T, MT, TN, WAVES, AHEAD, false, true>)
                : (grid.y == 1 ? linear8_rows_kernel<T, MT, TN, WAVES, AHEAD, true, false>
                               : linear8_rows_kernel<T, MT, TN, WAVES, AHEAD, false, false>);
  hipLaunchKernelGGL(kernel, grid, dim3(64 * WAVES), 0, stream, g);
  return check_launch("m3_linear8");
}

// By a_cu workgroups on every CU, that take tile after tile; with groups of waves (KS > 1) by one a tile.
template <typename T, int WM, int WN, int XI, int KS>
int launch_tile(const Lin8Geom& g, int a_cu, hipStream_t stream) {
  constexpr int BM = 16 * XI * WM;
  const int64_t tm = (g.m + BM - 1) / BM, tn = (g.tiles + WN - 1) / WN, all = tm * tn;
  if (all >= 1 << 30) return fail(M3_EUNSUPPORTED, "m3_linear8: over 2^30 tiles of out");
  const unsigned grid = static_cast<unsigned>(KS > 1 || all < a_cu * kCus ? all : a_cu * kCus);
  const bool res = g.res != nullptr;
  const auto kernel = g.whole ? (res ? linear8_tile_kernel<T, WM, WN, XI, KS, true, true>
                                     : linear8_tile_kernel<T, WM, WN, XI, KS, true, false>)
                              : (res ? linear8_tile_kernel<T, WM, WN, XI, KS, false, true>
                                     : linear8_tile_kernel<T, WM, WN, XI, KS, false, false>);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * WM * WN * KS), 0, stream, g, static_cast<unsigned>(tm),
                     static_cast<unsigned>(tn), kBand);
  return check_launch("m3_linear8");
}

// Which kernel (us in graphs with cold weights, bf16; M x N x K):
//   16 x 16 of out a workgroup of 8 waves, while these are at most two a CU (64 x 2048 x 4096: 7.3, the next 8.3;
//     16 x 4480 x 1024: 3.9, 4.4), or three with up to 4 rows (4 x 8672 x 2048: 5.5, 5.9; 8 rows: 6.1, 6.0)
//   32 x 64, for up to 32 rows or 1.5 a CU (16 x 16384 x 4096: 12.4, the one before 21; 256 x 2048 x 4096: 10.1, the
//     next 13.9; 512 x 2048 x 4096, two a CU: 16.9, 16.0); one column of tiles, too, where the codes' alignment asks the
//     next ones for a copy of them (65536 x 64 x 1001: 31.6, 63.8; 65536 x 16 x 4095: 134, 200; two columns, 65536 x 128 x
//     4095: 264, 204)
//   64 x 128 with K in halves, for up to half a 128 x 256 tile a CU (1000 x 2048 x 4096: 16.6, 128 x 128 26.6;
//     2000 x 2048 x 4096: 26.1, 128 x 256 about 30; 512 x 8672 x 2048, 136 tiles: 21.2, 18.9)
//   128 x 256 by two workgroups a CU, whose outputs' rounding hides behind each other's products, or where K is long 128
//     x 512 by one, whose rounds cost 17 and 16, half a round of the first 12 (65536 x 4480 x 1024: 264, 274; 16384 x
//     8672 x 2048: 224, 237; 8192 x 28672 x 8192: 1,342, 1,300; 4000 x 2048 x 4096: 30.8, 42.8)
enum Form { kCells, kRows, kHalves, kMedium, kLarge };
Form form_of(int64_t m, int64_t tiles, int64_t k, bool aligned) {
  const int64_t cells = 4 * tiles * ((m + 15) / 16);
  if (cells <= 2 * kCus || (m <= 4 && cells <= 3 * kCus)) return kCells;
  if (m <= 32 || tiles * ((m + 31) / 32) <= 3 * kCus / 2) return kRows;
  // (a launch has 65,535 rows of workgroups)
  if (!aligned && tiles == 1 && (m + 31) / 32 < 1 << 16) return kRows;
  const int64_t tm = (m + 127) / 128, medium = tm * ((tiles + 3) / 4);
  if (medium <= kCus / 2) return kHalves;
  if (k <= 2048) return kMedium;
  const int64_t large = tm * ((tiles + 7) / 8), rest = medium % (2 * kCus);
  const int64_t one = (large + kCus - 1) / kCus * 16;
  const int64_t two = medium / (2 * kCus) * 17 + (rest == 0 ? 0 : rest <= kCus ? 12 : 17);
  return one <= two ? kLarge : kMedium;
}

template <typename T>
int launch8(const Lin8Geom& g, Form form, hipStream_t stream) {
  switch (form) {
    case kCells: return launch_rows<T, 1, 1, 8, 4>(g, stream);
    case kRows: return launch_rows<T, 2, 4, 8, 2>(g, stream);
    case kHalves: return launch_tile<T, 1, 2, 4, 2>(g, 1, stream);
    case kMedium: return launch_tile<T, 1, 4, 8, 1>(g, 2, stream);
    default: return launch_tile<T, 1, 8, 8, 1>(g, 1, stream);
  }
}

// Rows of codes at any alignment into rows of whole 16 bytes; what lies past a row's end becomes 0. A lane takes
// 16 bytes; 2^lanes_log2 lanes take a row.
__global__ __launch_bounds__(256) void pad8_kernel(const char* codes, int64_t c_ld, char* to, int64_t to_ld,
                                                   int64_t rows, int k, int lanes_log2) {
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int64_t block = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
  const int64_t row = (block << (8 - lanes_log2)) + (threadIdx.x >> lanes_log2);
  if (row >= rows) return;
  for (int at = 16 * lane; at < k; at += 16 * lanes) {
    const char* p = codes + row * c_ld + at;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (at + 16 <= k) {
      __builtin_memcpy(&v, p, sizeof(v));
    } else {
      for (int e = 0; e < k - at; ++e) {
        v[e / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(p[e])) << (8 * (e % 4));
      }
    }
    *reinterpret_cast<u32x4*>(to + row * to_ld + at) = v;
  }
}

int launch_pad(const Lin8Geom& g, char* to, int64_t to_ld, hipStream_t stream) {
  int log2 = 0;
  while (log2 < 8 && (16 << log2) < g.k) ++log2;
  const int64_t blocks = (g.m + (256 >> log2) - 1) / (256 >> log2), most = 1 << 23;
  const dim3 grid(static_cast<unsigned>(blocks < most ? blocks : most),
                  static_cast<unsigned>((blocks + most - 1) / most));
  hipLaunchKernelGGL(pad8_kernel, grid, dim3(256), 0, stream, g.codes, g.c_ld, to, to_ld, g.m, g.k, log2);
  return check_launch("m3_linear8 (codes)");
}

bool aligned(const m3_linear8_args& a) {
  return reinterpret_cast<uintptr_t>(a.codes) % 16 == 0 && (a.m == 1 || a.codes_stride % 16 == 0) &&
         (a.exact == 0 || a.k % 16 == 0);
}

// Bytes of the copy of the codes that the call needs.
size_t need(const m3_linear8_args& a) {
  if (a.m == 0 || a.n == 0 || aligned(a) || form_of(a.m, (a.n + 63) / 64, a.k, false) <= kRows) return 0;
  return static_cast<size_t>(a.m) * ((a.k + 15) / 16 * 16);
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
  if (off(a.q, 16) || off(a.scales, 16) || off(a.row_scales, 4)) {
    return fail(M3_EUNSUPPORTED, "m3_linear8: q and scales must be 16-byte aligned, row_scales 4-byte");
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
  const auto meets = [](const void* p, int64_t bytes, const char* from, const char* to) {
    const char* p0 = static_cast<const char*>(p);
    return p0 < to && from < p0 + bytes;
  };
  const int64_t codes = (a.m - 1) * a.codes_stride + a.k, q = tiles * ((a.k + 127) / 128) * 2 * kTileBytes;
  const int64_t residual = ((a.m - 1) * a.residual.stride[0] + a.n) * es;
  if (meets(a.codes, codes, o0, o1) || meets(a.row_scales, a.m * 4, o0, o1) || meets(a.q, q, o0, o1) ||
      meets(a.scales, tiles * 256, o0, o1)) {
    return fail(M3_EINVAL, "m3_linear8: out overlaps codes, the weight or scales");
  }
  if (const size_t bytes = need(a); a.workspace != nullptr && bytes != 0) {
    const char* const w0 = static_cast<const char*>(a.workspace);
    const char* const w1 = w0 + bytes;
    const char* const what = meets(a.codes, codes, w0, w1)                            ? "codes"
                             : meets(o0, o1 - o0, w0, w1)                             ? "out"
                             : meets(a.q, q, w0, w1)                                  ? "the weight"
                             : present(a.residual) && meets(a.residual.ptr, residual, w0, w1) ? "residual"
                             : meets(a.row_scales, a.m * 4, w0, w1) || meets(a.scales, tiles * 256, w0, w1)
                                 ? "scales"
                                 : nullptr;
    if (what != nullptr) return fail(M3_EINVAL, "m3_linear8: %s overlaps the workspace", what);
  }
  const bool same = a.residual.ptr == a.out.ptr && (a.m == 1 || a.residual.stride[0] == a.out.stride[0]);
  if (present(a.residual) && !same && meets(a.residual.ptr, residual, o0, o1)) {
    return fail(M3_EINVAL, "m3_linear8: out overlaps the residual without being it");
  }
  return M3_OK;
}

}  // namespace
}  // namespace m3

extern "C" int m3_linear8_workspace_size(const m3_linear8_args* args, size_t* bytes) {
  using namespace m3;
  clear_error();
  if (args == nullptr || bytes == nullptr) return fail(M3_EINVAL, "m3_linear8_workspace_size: NULL args");
  const int rc = validate(*args);
  if (rc != M3_OK) return rc;
  *bytes = need(*args);
  return M3_OK;
}

extern "C" int m3_linear8(const m3_linear8_args* args, hipStream_t stream) {
  using namespace m3;
  clear_error();
  if (args == nullptr) return fail(M3_EINVAL, "m3_linear8: NULL args");
  const m3_linear8_args& a = *args;
  int rc = validate(a);
  if (rc != M3_OK) return rc;
  if (a.m == 0 || a.n == 0) return M3_OK;
  const int64_t es = elem_size(a.dtype), pitch = a.out.stride[0] * es;
  const int64_t pitch_r = a.residual.stride[0] * es;
  const bool whole = reinterpret_cast<uintptr_t>(a.out.ptr) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(a.residual.ptr) % 16 == 0 && a.n * es % 16 == 0 &&
                     (a.m == 1 || (pitch % 16 == 0 && pitch < (1 << 23) && pitch_r % 16 == 0 &&
                                   pitch_r < (1 << 23)));
  Lin8Geom g{reinterpret_cast<const char*>(a.codes), a.row_scales,
             reinterpret_cast<const char*>(a.q), a.scales, a.residual.ptr, a.out.ptr,
             a.codes_stride, a.residual.stride[0], a.out.stride[0], a.m, static_cast<int>(a.n),
             static_cast<int>(a.k), static_cast<int>((a.k + 127) / 128 * 2),
             static_cast<int>((a.n + 63) / 64), aligned(a), whole};
  if (a.m == 1) g.c_ld = (a.k + 15) / 16 * 16;  // rows past the only one lie past the extent
  const Form form = form_of(a.m, g.tiles, a.k, g.aligned);
  if (const size_t bytes = need(a); bytes != 0) {
    if (a.workspace == nullptr || a.workspace_bytes < bytes || reinterpret_cast<uintptr_t>(a.workspace) % 16 != 0) {
      return fail(M3_EWORKSPACE, "m3_linear8: rows of codes at this alignment need a 16-byte aligned workspace of "
                  "%zu bytes", bytes);
    }
    const int64_t ld = (a.k + 15) / 16 * 16;
    char* const to = static_cast<char*>(a.workspace);
    if ((rc = launch_pad(g, to, ld, stream)) != M3_OK) return rc;
    g.codes = to;
    g.c_ld = ld;
    g.aligned = true;
  }
  switch (a.dtype) {
    case M3_F32: return launch8<float>(g, form, stream);
    case M3_BF16: return launch8<__bf16>(g, form, stream);
    default: return launch8<_Float16>(g, form, stream);
  }
}
