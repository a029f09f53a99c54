// MXFP4: the codec of tensors in blocks of 32 elements, and the grouped product
// of two MXFP4 operands on the scaled matrix instructions
// (v_mfma_scale_f32_32x32x64_f8f6f4, gfx950).
#include "mxfp4.h"

#include <algorithm>
#include <type_traits>

namespace mx {
namespace mxfp4 {
namespace {

constexpr int kUnroll = 4;  // groups of 8 elements per thread

// Groups of 8 elements in order of (row, group of the row): four consecutive ones
// are a block and meet in a quad of lanes, so that a wave reads runs of 1 KB (bf16) and
// writes runs of 256 bytes, and no block passes through LDS. Bound by memory: 64 x 1408
// x 2048 in bf16 93 us, 5.0 TB/s read and written, where a copy reaches 5.1.
template <bool BF16>
__global__ __launch_bounds__(256) void quantize_kernel(const void *x, int64_t rows, int64_t cols,
                                                       int64_t ldx, uint8_t *codes, uint8_t *scales) {
  const int64_t per_row = 4 * ((cols + kBlock - 1) / kBlock);
  const int64_t total = rows * per_row;
  const bool flat = ldx == cols && cols % kBlock == 0;
  auto row_of = [&](int64_t g) -> int64_t {
    return total <= 0xffffffffll ? static_cast<uint32_t>(g) / static_cast<uint32_t>(per_row)
                                 : g / per_row;
  };
  const int64_t g0 = static_cast<int64_t>(blockIdx.x) * (256 * kUnroll) + threadIdx.x;
  float v[kUnroll][8];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t g = g0 + 256 * u;
    if (g >= total) break;
    if (flat) {
      load8<BF16>(x, 8 * g, v[u]);
      continue;
    }
    const int64_t row = row_of(g), col = 8 * (g - row * per_row);
    if (col + 8 <= cols)
      load8<BF16>(x, row * ldx + col, v[u]);
    else
      load8_guarded<BF16>(x, row * ldx + col, static_cast<int>(max(min(cols - col, int64_t(8)), int64_t(0))), v[u]);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t g = g0 + 256 * u;
    if (g >= total) break;
    uint32_t scale;
    reinterpret_cast<uint32_t *>(codes)[g] = quantize8(v[u], scale);
    if ((g & 3) == 0) scales[g >> 2] = static_cast<uint8_t>(scale);
  }
}

// One group of 8 elements per thread and step, four steps under way. Bound by its
// writes: 64 x 1408 x 2048 to bf16 69 us (370 MB written, 5.4 TB/s, its codes in part
// from the cache that the quantisation before it filled).
template <bool BF16>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t *codes, const uint8_t *scales,
                                                         int64_t rows, int64_t cols, void *out) {
  const int64_t per_row = 4 * ((cols + kBlock - 1) / kBlock);
  const int64_t total = rows * per_row;
  const bool flat = cols % kBlock == 0;
  const int64_t g0 = static_cast<int64_t>(blockIdx.x) * (256 * kUnroll) + threadIdx.x;
  uint32_t c[kUnroll], e[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t g = g0 + 256 * u;
    if (g >= total) break;
    c[u] = reinterpret_cast<const uint32_t *>(codes)[g];
    e[u] = scales[g >> 2];
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t g = g0 + 256 * u;
    if (g >= total) break;
    int64_t at = 8 * g, left = 8;
    if (!flat) {
      const int64_t row = total <= 0xffffffffll
                              ? static_cast<uint32_t>(g) / static_cast<uint32_t>(per_row)
                              : g / per_row;
      const int64_t col = 8 * (g - row * per_row);
      at = row * cols + col;
      left = cols - col;
    }
    const float s = __uint_as_float(e[u] == 0 ? 0x00400000u : e[u] == 255 ? 0x7fc00000u : e[u] << 23);
    f32x2_t f[4];
    f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], s, 0);
    f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], s, 1);
    f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], s, 2);
    f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], s, 3);
    if constexpr (BF16) {
      uint16_t *o = static_cast<uint16_t *>(out) + at;
      u32x4 q;
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = pack_bf16x2(f[i][0], f[i][1]);
      if (left >= 8) {
        *reinterpret_cast<u32x4_any *>(o) = q;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) o[i] = static_cast<uint16_t>(q[i >> 1] >> (16 * (i & 1)));
      }
    } else {
      float *o = static_cast<float *>(out) + at;
      if (left >= 8) {
        reinterpret_cast<f32x4_any *>(o)[0] = f32x4{f[0][0], f[0][1], f[1][0], f[1][1]};
        reinterpret_cast<f32x4_any *>(o)[1] = f32x4{f[2][0], f[2][1], f[3][0], f[3][1]};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) o[i] = f[i >> 1][i & 1];
      }
    }
  }
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// ---------------------------------------------------------- grouped product
constexpr int kTall = 256, kShort = 128;  // rows of the product's tiles
constexpr int kStage = kTall * 64 + 128 * 64 + kTall * 4 + 128 * 4;  // bytes of an LDS stage
constexpr int kStep = 128;                // K columns of an LDS stage: 64 bytes of codes

// Workspace: a head of 256 bytes (int32 errors, tall tiles, short tiles), the tile
// lists, the rows' codes [ceil(K / 128)][S][64] and scales [ceil(K / 128)][S][4].
struct Layout {
  int64_t max_tall = 0, max_short = 0;
  size_t off_tall = 0, off_short = 0, off_codes = 0, off_scales = 0, bytes = 0;
};

Layout layout(int64_t rows, int experts, int64_t in_f) {
  Layout L;
  // A tall tile has more than kShort rows of its expert, a short one at least one.
  L.max_tall = rows / (kShort + 1);
  L.max_short = std::min<int64_t>(rows, experts);
  size_t off = 256;
  L.off_tall = off;
  off = align_up(off + sizeof(int4) * L.max_tall, 256);
  L.off_short = off;
  off = align_up(off + sizeof(int4) * L.max_short, 256);
  L.off_codes = off;
  off = align_up(off + ceil_div(in_f, kStep) * rows * 64, 256);
  L.off_scales = off;
  off = align_up(off + ceil_div(in_f, kStep) * rows * 4, 256);
  L.bytes = off;
  return L;
}

struct PlanOut {
  const void *offsets;
  bool wide;  // int64 offsets
  int64_t rows;
  int experts;
  int32_t *head;  // errors, tall tiles, short tiles
  int4 *tall, *rest;  // (expert, first row, rows, 0)
  int32_t *host_err;
};

// Inclusive sums over the 256 threads of a workgroup; `total` receives the last.
__device__ __forceinline__ int64_t scan256(int64_t v, int64_t *buf, int64_t &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(v, off, 64);
    v += lane >= off ? y : 0;
  }
  __syncthreads();  // the last use of buf
  if (lane == 63) buf[wave] = v;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    v += w < wave ? buf[w] : 0;
    total += buf[w];
  }
  return v;
}

// The tile list, by one workgroup: thread t takes the experts [t per, (t + 1) per).
// Counts are the differences of the row ends: an end below the one before it, or
// counts that do not add up, are errors, as in the plans of the other projections.
__device__ void plan_tiles(const PlanOut &P) {
  __shared__ int64_t buf[4];
  __shared__ int32_t n_err;
  if (threadIdx.x == 0) n_err = 0;
  const int per = (P.experts + 255) / 256;
  const int e0 = min(static_cast<int>(threadIdx.x) * per, P.experts), e1 = min(e0 + per, P.experts);
  auto end_of = [&](int e) -> int64_t {
    return P.wide ? static_cast<const int64_t *>(P.offsets)[e] : static_cast<const int32_t *>(P.offsets)[e];
  };
  int64_t rows = 0;
  int32_t bad = 0;
  auto count_of = [&](int e) -> int64_t {
    const int64_t c = end_of(e) - (e > 0 ? end_of(e - 1) : 0);
    return min(max(c, int64_t(0)), P.rows);
  };
  for (int e = e0; e < e1; ++e) {
    const int64_t c = end_of(e) - (e > 0 ? end_of(e - 1) : 0);
    bad += c < 0 || c > P.rows;
    rows += count_of(e);
  }
  int64_t all_rows;
  const int64_t start0 = scan256(rows, buf, all_rows) - rows;
  if (bad) atomicAdd(&n_err, bad);
  // Rows beyond P.rows are never touched, even if the ends disagree.
  auto each = [&](auto f) {
    int64_t start = start0;
    for (int e = e0; e < e1; ++e) {
      const int64_t end = start + count_of(e);
      const int64_t lo = min(start, P.rows), hi = min(end, P.rows);
      const int64_t tall = (hi - lo + kTall - kShort - 1) / kTall;
      f(e, lo, hi, tall, hi - lo > tall * kTall);
      start = end;
    }
  };
  int64_t tiles = 0, all_tiles;  // tall ones in the low half, short ones in the high half
  each([&](int, int64_t, int64_t, int64_t tall, bool rest) { tiles += tall + (static_cast<int64_t>(rest) << 32); });
  int64_t at = scan256(tiles, buf, all_tiles) - tiles;
  each([&](int e, int64_t lo, int64_t hi, int64_t tall, bool rest) {
    for (int64_t i = 0; i < tall; ++i)
      P.tall[(at & 0xffffffff) + i] = int4{e, static_cast<int>(lo + i * kTall),
                                           static_cast<int>(min(hi - lo - i * kTall, int64_t(kTall))), 0};
    if (rest) {
      P.rest[at >> 32] = int4{e, static_cast<int>(lo + tall * kTall), static_cast<int>(hi - lo - tall * kTall), 0};
      at += int64_t(1) << 32;
    }
    at += tall;
  });
  if (threadIdx.x == 0) {
    const int32_t errors = n_err + (all_rows != P.rows);
    P.head[0] = errors;
    P.head[1] = static_cast<int32_t>(all_tiles & 0xffffffff);
    P.head[2] = static_cast<int32_t>(all_tiles >> 32);
    if (P.host_err) __hip_atomic_store(P.host_err, errors, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
  }
}

// The rows' quantisation, codes and scales by 128 columns as the product reads them
// (zeros past K); the last workgroup forms the tile list meanwhile. A workgroup takes
// 64 rows of 128 columns: 16 lanes a row, so that reads are runs of 256 bytes (bf16)
// and a wave's writes of 4 neighbouring rows one run. 131072 x 2048: 131 us, 5.2 TB/s
// read and written; in order of the rows, with codes and scales of a row scattered over
// the tiles, 155.
template <bool BF16>
__global__ __launch_bounds__(256) void rows_kernel(const void *x, int64_t rows, int64_t cols, uint8_t *codes,
                                                   uint8_t *scales, PlanOut P) {
  if (blockIdx.x == gridDim.x - 1) {
    plan_tiles(P);
    return;
  }
  const int tiles = static_cast<int>((cols + kStep - 1) / kStep);
  // Runs of workgroups per XCD, the column tiles of the same rows side by side.
  const int64_t job = static_cast<int64_t>(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const int64_t group = job / tiles, tile = job - group * tiles;
  const int lane = threadIdx.x & 63, part = lane & 15;
  const int64_t row0 = group * 64 + 16 * (threadIdx.x >> 6) + (lane >> 4);
  const int64_t col = tile * kStep + 8 * part;
  float v[4][8];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t row = row0 + 4 * u;
    if (row < rows && col < cols) {
      load8<BF16>(x, row * cols + col, v[u]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t row = row0 + 4 * u;
    uint32_t scale;
    const uint32_t c = quantize8(v[u], scale);
    // The 16 lanes of a row's 4 blocks put their scales together.
    uint32_t w = scale << (8 * (part >> 2));
    w |= __builtin_amdgcn_mov_dpp(static_cast<int>(w), 0x141, 0xf, 0xf, true);  // mirrored half row
    w |= __builtin_amdgcn_mov_dpp(static_cast<int>(w), 0x140, 0xf, 0xf, true);  // mirrored row
    if (row >= rows) continue;
    reinterpret_cast<uint32_t *>(codes)[(tile * rows + row) * 16 + part] = c;
    if (part == 0) reinterpret_cast<uint32_t *>(scales)[tile * rows + row] = w;
  }
}

struct Product {
  const uint8_t *xc, *xs;  // [ceil(K/128)][S][64], [ceil(K/128)][S][4]
  const uint8_t *wc, *ws;  // [E, 4 ceil(K/128), N, 16], [E, ceil(K/128), N, 4]
  int64_t S, K, N;
  const int32_t *head;
  const int4 *tall, *rest;
  int n_tiles_n;
  void *out;
};

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef int i32x8 __attribute__((ext_vector_type(8)));

// 4-bit operands take the first four of the eight registers.
__device__ __forceinline__ i32x8 operand(u32x4 q) {
  return i32x8{static_cast<int>(q[0]), static_cast<int>(q[1]), static_cast<int>(q[2]),
               static_cast<int>(q[3]), 0, 0, 0, 0};
}

__device__ __forceinline__ void lds_dma16(const uint8_t *src, uint8_t *dst) {
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const void *>(src),
      reinterpret_cast<__attribute__((address_space(3))) void *>(reinterpret_cast<uintptr_t>(dst)), 16, 0, 0);
}

__device__ __forceinline__ void lds_dma4(const uint8_t *src, uint8_t *dst) {
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const void *>(src),
      reinterpret_cast<__attribute__((address_space(3))) void *>(reinterpret_cast<uintptr_t>(dst)), 4, 0, 0);
}

// A tile of up to 64 MB rows of an expert by 128 of its weight rows, by 4 waves with
// 32 MB x 64 outputs each: MB x 2 blocks of v_mfma_scale_f32_32x32x64_f8f6f4, the
// weights first (a lane's 4 consecutive values are 4 columns of an output row).
// K runs in stages of 128 columns (64 bytes of a row; rows of a stage side by side
// in memory, so that requests are of whole lines) through a ring of three in LDS, codes
// and scales filled by DMA two stages ahead: 76.5 KB, so two workgroups share a CU and
// cover each other's ends. 131072 rows, 2048 -> 1408, 64 experts: 270 us, 2.8 PFLOP/s
// (8192 cubed: 300 us, 3.7), with the clock at 1.8 to 1.95 GHz under this load. K is
// 16 stages here, so a tile's first loads and its results (0.37 GB in all) weigh as
// much as the products. Slower, or not worth their registers: scales read by row (a
// line per row: 462 us, most of it in the address units), two stages of 256 columns
// and one workgroup per CU (307), persistent tiles of 256 x 256 by 8 waves (258, and
// 281 for 8192 cubed, though they bring a quarter less to LDS). One kernel whose
// workgroups quantise 128 rows of up to 2048 columns into 136 KB of LDS and then take
// all columns of their expert against them reads and writes 0.29 GB less, but its
// workgroups run in step, one on a CU: 404 for both parts, as before.
template <bool BF16, int MB>
__device__ __forceinline__ void product_tile(const Product &p, int4 tile, int64_t n0, uint8_t *s0, uint8_t *s1,
                                             uint8_t *s2) {
  constexpr int NB = 2, WM = 32 * MB, WN = 64, BM = 2 * WM;
  constexpr int XD = BM / 64, WD = 2;  // DMA instructions of a wave per stage (16 rows each)
  // The weights' and the scales' places in a stage.
  constexpr int kW = BM * 64, kXS = kW + 128 * 64, kWS = kXS + BM * 4;
  static_assert(kWS + 512 <= kStage, "a stage holds the tile's columns");
  const int lane = threadIdx.x & 63, li = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wm = wave >> 1, wn = wave & 1;
  const int e = tile.x, m = tile.z;
  const int64_t row0 = tile.y;
  const int n = static_cast<int>(min(p.N - n0, int64_t(128)));
  const int KT = static_cast<int>((p.K + 127) / 128);
  const uint8_t *xc = p.xc + row0 * 64;
  const uint8_t *wc = p.wc + (static_cast<int64_t>(4 * e) * KT * p.N + n0) * 16;
  // The weights of a stage lie as in memory, block by block. 16-byte chunks of its rows
  // lie at chunk ^ (row >> 2 & 3): of 16 consecutive rows one chunk is in 16 different
  // slots of a 256-byte bank line. Rows past the tile's repeat its last one: their
  // products are not stored.
  const int chunk = 16 * ((lane & 3) ^ ((lane >> 4) & 3));
  uint32_t xo[XD], wo[WD];
#pragma unroll
  for (int i = 0; i < XD; ++i) xo[i] = 64 * min(16 * (4 * i + wave) + (lane >> 2), m - 1) + chunk;
#pragma unroll
  for (int i = 0; i < WD; ++i) wo[i] = 16 * min(64 * ((4 * i + wave) & 1) + lane, n - 1);
  // Scales: 4 bytes of a stage per row, 64 rows per DMA instruction (where there
  // are fewer rows than waves, two waves bring the same ones).
  const uint8_t *xs = p.xs + row0 * 4;
  const uint8_t *ws = p.ws + (static_cast<int64_t>(e) * KT * p.N + n0) * 4;
  const int xg = wave & (BM / 64 - 1), wg = wave & 1;
  const uint32_t xso = 4 * min(64 * xg + lane, m - 1), wso = 4 * min(64 * wg + lane, n - 1);
  auto load = [&](int k, uint8_t *s) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < XD; ++i) lds_dma16(xc + 64 * k * p.S + xo[i], s + (4 * i + wave) * 1024);
#pragma unroll
    for (int i = 0; i < WD; ++i)
      lds_dma16(wc + 16 * (4 * k + ((4 * i + wave) >> 1)) * p.N + wo[i], s + kW + (4 * i + wave) * 1024);
    lds_dma4(xs + (4 * k * p.S + xso), s + kXS + 256 * xg);
    lds_dma4(ws + (4 * k * p.N + wso), s + kWS + 256 * wg);
    __builtin_amdgcn_sched_barrier(0);
  };
  f32x16 acc[MB][NB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[mb][nb][q] = 0.0f;
  // Half h of a step's 64 columns: chunk 2 s + h, at the first one's place ^ (s << 5).
  const int place0 = li * 64 + ((h ^ ((li >> 2) & 3)) << 4);
  const int fx = wm * WM * 64 + place0, fw = kW + h * 2048 + (wn * WN + li) * 16;
  const int sxo = kXS + 4 * (wm * WM + li), swo = kWS + 4 * (wn * WN + li);
  auto step = [&](int k, const uint8_t *s, uint8_t *refill) __attribute__((always_inline)) {
    // The stage has landed once only the DMA of the one after it is under way, and
    // the reads of the one before it, which is refilled, are done (lgkmcnt(0)).
    if (k + 1 < KT)
      __builtin_amdgcn_s_waitcnt(0x0070 | (XD + WD + 2));
    else
      __builtin_amdgcn_s_waitcnt(0x0070);
    // (A fence would wait for all of the DMA.)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (k + 2 < KT) load(k + 2, refill);
    // Byte 0 of a shifted word: the scale of the lane's block of the first 64 columns;
    // byte 2: of the second. (Past K they are 2^-127 on both sides: products of at most
    // 36 * 2^-254, which vanish next to any fp32 number.)
    int sx[MB], sw[NB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
      sx[mb] = static_cast<int>(*reinterpret_cast<const uint32_t *>(s + sxo + 128 * mb) >> (8 * h));
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      sw[nb] = static_cast<int>(*reinterpret_cast<const uint32_t *>(s + swo + 128 * nb) >> (8 * h));
    u32x4 x[2][MB], w[2][NB];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) w[t][nb] = *reinterpret_cast<const u32x4 *>(s + fw + 4096 * t + 512 * nb);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) x[t][mb] = *reinterpret_cast<const u32x4 *>(s + (fx ^ (t << 5)) + 2048 * mb);
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        acc[mb][nb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w[0][nb]), operand(x[0][mb]),
                                                                      acc[mb][nb], 4, 4, 0, sw[nb], 0, sx[mb]);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        acc[mb][nb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(w[1][nb]), operand(x[1][mb]),
                                                                      acc[mb][nb], 4, 4, 2, sw[nb], 2, sx[mb]);
  };
  load(0, s0);
  if (KT > 1) load(1, s1);
  for (int k = 0;; k += 3) {
    step(k, s0, s2);
    if (k + 1 >= KT) break;
    step(k + 1, s1, s0);
    if (k + 2 >= KT) break;
    step(k + 2, s2, s1);
    if (k + 3 >= KT) break;
  }

  // Each wave turns 32 rows of its results over at a time in its part of a stage, so
  // that runs of 64 columns of a row are stored.
  constexpr int ES = BF16 ? 2 : 4, CH = WN * ES / 16;  // 16-byte chunks of a row
  __syncthreads();
  uint8_t *strip = (wave < 2 ? s0 : s1) + (wave & 1) * 8192;
  auto place = [&](int row, int c) { return row * (CH * 16) + ((c ^ (BF16 ? (row >> 1) & 7 : row & 15)) << 4); };
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x16 &v = acc[mb][nb];
        // Columns 32 nb + 8 g + 4 h .. + 3 of row li.
        if constexpr (BF16) {
          *reinterpret_cast<uint64_t *>(strip + place(li, 4 * nb + g) + 8 * h) =
              pack_bf16x2(v[4 * g], v[4 * g + 1]) |
              (static_cast<uint64_t>(pack_bf16x2(v[4 * g + 2], v[4 * g + 3])) << 32);
        } else {
          *reinterpret_cast<f32x4 *>(strip + place(li, 8 * nb + 2 * g + h)) =
              f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
        }
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    constexpr int RP = 64 / CH, IT = 32 / RP;  // rows per pass, passes
    u32x4 q[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) q[i] = *reinterpret_cast<const u32x4 *>(strip + place(RP * i + lane / CH, lane % CH));
    const int r0 = wm * WM + 32 * mb + lane / CH, col = wn * WN + (lane % CH) * (16 / ES);
    uint8_t *out = static_cast<uint8_t *>(p.out) + ((row0 + r0) * p.N + n0 + col) * ES;
    if (col < n) {
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if (r0 + RP * i < m) *reinterpret_cast<u32x4 *>(out + RP * i * p.N * ES) = q[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// Workgroups go to the 8 XCDs in turn; each XCD takes a run of the tall tiles and
// then a run of the short ones, column tiles of one row tile side by side, so that
// the rows of a tile and the weights of an expert are read through one L2.
template <bool BF16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void product_kernel(Product p) {
  __shared__ __attribute__((aligned(16))) uint8_t s0[kStage], s1[kStage], s2[kStage];
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  const int total_t = p.head[1] * p.n_tiles_n, total_s = p.head[2] * p.n_tiles_n;
  const int per_t = (total_t + 7) >> 3, per_s = (total_s + 7) >> 3;
  const bool tall = slot < per_t;
  const int logical = tall ? xcd * per_t + slot : xcd * per_s + slot - per_t;
  if (!tall && slot >= per_t + per_s) return;
  if (logical >= (tall ? total_t : total_s)) return;
  const int mt = logical / p.n_tiles_n;
  const int4 tile = (tall ? p.tall : p.rest)[mt];
  const int64_t n0 = static_cast<int64_t>(logical - mt * p.n_tiles_n) * 128;
  if (tall)
    product_tile<BF16, 4>(p, tile, n0, s0, s1, s2);
  else
    product_tile<BF16, 2>(p, tile, n0, s0, s1, s2);
}

bool dtype_ok(int d) { return d == MX_DTYPE_BF16 || d == MX_DTYPE_F32; }

int grid_ok(const char *name, int64_t blocks) {
  if (blocks > 0x7fffffff) {
    set_error("%s: too many elements for one launch", name);
    return MX_ERR_INVALID;
  }
  return MX_OK;
}

}  // namespace
}  // namespace mxfp4
}  // namespace mx

using namespace mx;
using namespace mx::mxfp4;

extern "C" int mx_mxfp4_quantize(const void *x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx,
                                 uint8_t *codes, uint8_t *scales, void *stream) {
  clear_error();
  const char *name = "mx_mxfp4_quantize";
  if (rows < 0 || cols <= 0 || ldx < cols || !dtype_ok(x_dtype)) {
    set_error("%s: need rows >= 0, cols >= 1, ldx >= cols and a bf16 or fp32 input", name);
    return MX_ERR_INVALID;
  }
  if (rows == 0) return MX_OK;
  if (!x || !codes || !scales || reinterpret_cast<uintptr_t>(codes) % 4 != 0) {
    set_error("%s: buffers must be non-null and codes 4-byte aligned", name);
    return MX_ERR_INVALID;
  }
  const int64_t blocks = ceil_div(rows * 4 * ceil_div(cols, kBlock), 256 * kUnroll);
  if (int rc = grid_ok(name, blocks)) return rc;
  const bool bf16 = x_dtype == MX_DTYPE_BF16;
  auto kernel = bf16 ? quantize_kernel<true> : quantize_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, as_stream(stream), x,
                     rows, cols, ldx, codes, scales);
  return check_launch(name);
}

extern "C" int mx_mxfp4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows,
                                   int64_t cols, void *out, int out_dtype, void *stream) {
  clear_error();
  const char *name = "mx_mxfp4_dequantize";
  if (rows < 0 || cols <= 0 || !dtype_ok(out_dtype)) {
    set_error("%s: need rows >= 0, cols >= 1 and a bf16 or fp32 output", name);
    return MX_ERR_INVALID;
  }
  if (rows == 0) return MX_OK;
  if (!codes || !scales || !out || reinterpret_cast<uintptr_t>(codes) % 4 != 0) {
    set_error("%s: buffers must be non-null and codes 4-byte aligned", name);
    return MX_ERR_INVALID;
  }
  const int64_t blocks = ceil_div(rows * 4 * ceil_div(cols, kBlock), 256 * kUnroll);
  if (int rc = grid_ok(name, blocks)) return rc;
  const bool bf16 = out_dtype == MX_DTYPE_BF16;
  auto kernel = bf16 ? dequantize_kernel<true> : dequantize_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, as_stream(stream),
                     codes, scales, rows, cols, out);
  return check_launch(name);
}

extern "C" size_t mx_mxfp4_grouped_linear_workspace_size(int64_t num_rows, int num_experts,
                                                         int64_t in_features) {
  if (num_rows < 0 || num_experts <= 0 || in_features <= 0) return 0;
  return layout(num_rows, num_experts, in_features).bytes;
}

extern "C" int mx_mxfp4_grouped_linear(const void *x, int x_dtype, const void *offsets, int offsets_64,
                                       int64_t num_rows, int num_experts, const mx_weight *w, void *out,
                                       int out_dtype, void *workspace, int32_t *host_err, void *stream) {
  clear_error();
  const char *name = "mx_mxfp4_grouped_linear";
  if (num_rows < 0 || num_rows >= (int64_t(1) << 31) || num_experts <= 0 ||
      num_experts > 8192) {
    set_error("%s: need 0 <= num_rows < 2^31 and num_experts in [1, 8192]", name);
    return MX_ERR_INVALID;
  }
  if (!dtype_ok(x_dtype) || !dtype_ok(out_dtype)) {
    set_error("%s: rows and output must be bf16 or fp32", name);
    return MX_ERR_INVALID;
  }
  if (!w || w->format != MX_FMT_MXFP4 || !w->data || !w->scale) {
    set_error("%s: needs an MX_FMT_MXFP4 weight with its scales", name);
    return MX_ERR_INVALID;
  }
  const int64_t K = w->in_features, N = w->out_features;
  if (K <= 0 || K % 64 != 0 || N <= 0 || N % 8 != 0) {
    set_error("%s: in_features must be a multiple of 64 and out_features of 8", name);
    return MX_ERR_INVALID;
  }
  if (num_rows == 0) return MX_OK;
  if (!x || !offsets || !out || !workspace) {
    set_error("%s: x, offsets, output and workspace must be non-null", name);
    return MX_ERR_INVALID;
  }
  if (!aligned16(w->data) || !aligned16(out) || !aligned16(workspace) ||
      reinterpret_cast<uintptr_t>(w->scale) % 4 != 0) {
    set_error("%s: weight codes, output and workspace must be 16-byte and weight scales 4-byte aligned", name);
    return MX_ERR_INVALID;
  }
  hipStream_t s = as_stream(stream);
  const Layout L = layout(num_rows, num_experts, K);
  char *base = static_cast<char *>(workspace);
  uint8_t *codes = reinterpret_cast<uint8_t *>(base + L.off_codes);
  uint8_t *scales = reinterpret_cast<uint8_t *>(base + L.off_scales);
  PlanOut P = {offsets, offsets_64 != 0, num_rows, num_experts, reinterpret_cast<int32_t *>(base),
               reinterpret_cast<int4 *>(base + L.off_tall), reinterpret_cast<int4 *>(base + L.off_short),
               host_err};
  const int64_t chunks = 8 * ceil_div(ceil_div(num_rows, 64) * ceil_div(K, kStep), 8);
  const int64_t n_tiles = ceil_div(N, 128);
  const int64_t grid = 8 * (ceil_div(L.max_tall * n_tiles, 8) + ceil_div(L.max_short * n_tiles, 8));
  if (int rc = grid_ok(name, std::max(chunks + 1, grid))) return rc;
  const bool bf16 = x_dtype == MX_DTYPE_BF16;
  auto rows_k = bf16 ? rows_kernel<true> : rows_kernel<false>;
  hipLaunchKernelGGL(rows_k, dim3(static_cast<unsigned>(chunks + 1)), dim3(256), 0, s, x, num_rows, K,
                     codes, scales, P);
  if (int rc = check_launch(name)) return rc;
  Product p = {codes, scales, static_cast<const uint8_t *>(w->data),
               static_cast<const uint8_t *>(w->scale), num_rows, K, N, P.head, P.tall, P.rest,
               static_cast<int>(n_tiles), out};
  auto product = out_dtype == MX_DTYPE_BF16 ? product_kernel<true> : product_kernel<false>;
  hipLaunchKernelGGL(product, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, p);
  return check_launch(name);
}
