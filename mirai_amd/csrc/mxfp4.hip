// MXFP4: the codec of tensors in blocks of 32 elements, and the grouped product
// of two MXFP4 operands on the scaled matrix instructions
// (v_mfma_scale_f32_32x32x64_f8f6f4, gfx950).
#include "mxfp4.h"

#include <algorithm>

namespace mx {
namespace mxfp4 {
namespace {

constexpr int kUnroll = 4;  // groups of 8 elements per thread

// Groups of 8 elements in order of (row, group of the row): four consecutive ones
// are a block and meet in a quad of lanes.
template <bool BF16>
__device__ __forceinline__ void quantize_groups(const void *x, int64_t rows, int64_t cols,
                                                int64_t ldx, bool vec, uint8_t *codes,
                                                uint8_t *scales, int64_t lds, int64_t chunk) {
  const int64_t per_row = 4 * ((cols + kBlock - 1) / kBlock);
  const int64_t total = rows * per_row;
  const bool flat = vec && ldx == cols && cols % kBlock == 0;
  auto row_of = [&](int64_t g) -> int64_t {
    return total <= 0xffffffffll ? static_cast<uint32_t>(g) / static_cast<uint32_t>(per_row)
                                 : g / per_row;
  };
  const int64_t g0 = chunk * (256 * kUnroll) + threadIdx.x;
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
    if (vec && col + 8 <= cols)
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
    if ((g & 3) == 0) {
      const int64_t b = g >> 2;
      scales[4 * lds == per_row ? b : b + row_of(g) * (lds - per_row / 4)] = static_cast<uint8_t>(scale);
    }
  }
}

template <bool BF16>
__global__ __launch_bounds__(256) void quantize_kernel(const void *x, int64_t rows, int64_t cols,
                                                       int64_t ldx, bool vec, uint8_t *codes,
                                                       uint8_t *scales) {
  quantize_groups<BF16>(x, rows, cols, ldx, vec, codes, scales, (cols + kBlock - 1) / kBlock, blockIdx.x);
}

// One group of 8 elements per thread and step.
template <bool BF16>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t *codes, const uint8_t *scales,
                                                         int64_t rows, int64_t cols, bool vec,
                                                         void *out) {
  const int64_t per_row = 4 * ((cols + kBlock - 1) / kBlock);
  const int64_t total = rows * per_row;
  const bool flat = vec && cols % kBlock == 0;
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
      if (vec && left >= 8) {
        *reinterpret_cast<u32x4 *>(o) = q;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) o[i] = static_cast<uint16_t>(q[i >> 1] >> (16 * (i & 1)));
      }
    } else {
      float *o = static_cast<float *>(out) + at;
      if (vec && left >= 8) {
        reinterpret_cast<f32x4 *>(o)[0] = f32x4{f[0][0], f[0][1], f[1][0], f[1][1]};
        reinterpret_cast<f32x4 *>(o)[1] = f32x4{f[2][0], f[2][1], f[3][0], f[3][1]};
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
constexpr int kStep = 256;                // K columns of an LDS stage: 128 bytes of codes

// Workspace: a head of 256 bytes (int32 errors, tall tiles, short tiles), the
// segment ends as the tiles use them, the tile lists, the rows' codes [S, K/2] and
// scales [S, ldxs].
struct Layout {
  int64_t max_tall = 0, max_short = 0, ldxs = 0;
  size_t off_ends = 0, off_tall = 0, off_short = 0, off_codes = 0, off_scales = 0, bytes = 0;
};

Layout layout(int64_t rows, int experts, int64_t in_f) {
  Layout L;
  // A tall tile has more than kShort rows of its expert, a short one at least one.
  L.max_tall = rows / (kShort + 1);
  L.max_short = std::min<int64_t>(rows, experts);
  L.ldxs = ceil_div(in_f, kStep) * (kStep / kBlock);
  size_t off = 256;
  L.off_ends = off;
  off = align_up(off + sizeof(int64_t) * experts, 256);
  L.off_tall = off;
  off = align_up(off + sizeof(int2) * L.max_tall, 256);
  L.off_short = off;
  off = align_up(off + sizeof(int2) * L.max_short, 256);
  L.off_codes = off;
  off = align_up(off + rows * (in_f / 2), 256);
  L.off_scales = off;
  off = align_up(off + rows * L.ldxs, 256);
  L.bytes = off;
  return L;
}

struct PlanOut {
  const void *offsets;
  bool wide;  // int64 offsets
  int64_t rows;
  int experts;
  int32_t *head;  // errors, tall tiles, short tiles
  int64_t *ends;
  int2 *tall, *rest;
  int32_t *host_err;
};

// Inclusive scan over the 256 threads of a workgroup.
template <class F>
__device__ __forceinline__ int64_t scan256(int64_t v, int64_t *buf, F op) {
  const int t = threadIdx.x;
  buf[t] = v;
  __syncthreads();
  for (int d = 1; d < 256; d <<= 1) {
    const int64_t o = t >= d ? buf[t - d] : buf[t];
    const bool use = t >= d;
    __syncthreads();
    if (use) buf[t] = op(o, buf[t]);
    __syncthreads();
  }
  const int64_t r = buf[t];
  __syncthreads();
  return r;
}

// The tile list of one workgroup: thread t takes the experts [t per, (t + 1) per).
// An expert's rows run from the largest end before it to its own end, both held
// within [0, rows].
__device__ void plan_tiles(const PlanOut &P) {
  __shared__ int64_t buf[256];
  const int per = (P.experts + 255) / 256;
  const int e0 = min(static_cast<int>(threadIdx.x) * per, P.experts), e1 = min(e0 + per, P.experts);
  auto raw = [&](int e) {
    return P.wide ? static_cast<const int64_t *>(P.offsets)[e]
                  : static_cast<int64_t>(static_cast<const int32_t *>(P.offsets)[e]);
  };
  auto held = [&](int64_t v) { return min(max(v, int64_t(0)), P.rows); };
  int64_t top = 0;
  for (int e = e0; e < e1; ++e) top = max(top, held(raw(e)));
  const int64_t upto = scan256(top, buf, [](int64_t a, int64_t b) { return max(a, b); });
  // The largest end before this thread's experts.
  buf[threadIdx.x] = upto;
  __syncthreads();
  const int64_t before = threadIdx.x ? buf[threadIdx.x - 1] : 0;
  const int64_t last = buf[255];
  __syncthreads();
  int64_t start = before, bad = 0;
  int64_t tiles = 0;  // tall ones in the low half, short ones in the high half
  auto tall_of = [](int64_t rows) { return (rows + kTall - kShort - 1) / kTall; };
  auto short_of = [&](int64_t rows) { return int64_t(rows > tall_of(rows) * kTall); };
  for (int e = e0; e < e1; ++e) {
    const int64_t r = raw(e), end = max(start, held(r));
    bad += r < start || r > P.rows;
    P.ends[e] = end;
    tiles += tall_of(end - start) + (short_of(end - start) << 32);
    start = end;
  }
  auto add = [](int64_t a, int64_t b) { return a + b; };
  const int64_t tiles_upto = scan256(tiles, buf, add);
  const int64_t bad_upto = scan256(bad, buf, add);
  int64_t at = tiles_upto - tiles;
  start = before;
  for (int e = e0; e < e1; ++e) {
    const int64_t end = max(start, held(raw(e)));
    int64_t n = tall_of(end - start);
    for (int64_t i = 0; i < n; ++i)
      P.tall[(at & 0xffffffff) + i] = int2{e, static_cast<int>(start + i * kTall)};
    if (short_of(end - start)) {
      P.rest[at >> 32] = int2{e, static_cast<int>(start + n * kTall)};
      at += int64_t(1) << 32;
    }
    at += n;
    start = end;
  }
  if (threadIdx.x == 255) {
    const int32_t errors = static_cast<int32_t>(bad_upto + (last != P.rows));
    P.head[0] = errors;
    P.head[1] = static_cast<int32_t>(tiles_upto & 0xffffffff);
    P.head[2] = static_cast<int32_t>(tiles_upto >> 32);
    if (P.host_err) __hip_atomic_store(P.host_err, errors, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
  }
}

// The rows' quantisation; the last workgroup forms the tile list meanwhile.
template <bool BF16>
__global__ __launch_bounds__(256) void rows_kernel(const void *x, int64_t rows, int64_t cols, bool vec,
                                                   uint8_t *codes, uint8_t *scales, int64_t lds,
                                                   PlanOut P) {
  if (blockIdx.x == gridDim.x - 1) {
    plan_tiles(P);
    return;
  }
  quantize_groups<BF16>(x, rows, cols, cols, vec, codes, scales, lds, blockIdx.x);
}

struct Product {
  const uint8_t *xc, *xs;  // [S, K/2], [S, ldxs]
  int64_t ldxs;
  const uint8_t *wc, *ws;  // [E, N, K/2], [E, N, K/32]
  int64_t K, N;
  const int32_t *head;
  const int64_t *ends;
  const int2 *tall, *rest;
  int n_tiles_n;
  void *out;
};

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Row key of a stage of 128-byte rows: the 16-byte chunks of 16 consecutive rows at
// one logical chunk lie in 16 different slots of a 256-byte bank line.
__device__ __forceinline__ int row_key(int row) { return ((row >> 1) ^ (row << 2)) & 7; }

__device__ __forceinline__ i32x8 fragment(const uint8_t *stage, int row, int chunk) {
  const u32x4 q = *reinterpret_cast<const u32x4 *>(stage + row * 128 + ((chunk ^ row_key(row)) << 4));
  return i32x8{static_cast<int>(q[0]), static_cast<int>(q[1]), static_cast<int>(q[2]),
               static_cast<int>(q[3]), 0, 0, 0, 0};
}

__device__ __forceinline__ void lds_dma16(const uint8_t *src, uint8_t *dst) {
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const void *>(src),
      reinterpret_cast<__attribute__((address_space(3))) void *>(reinterpret_cast<uintptr_t>(dst)), 16, 0, 0);
}

// One tile of up to BM rows x BN weight rows: 4 waves on a WGM x (4 / WGM) grid, each
// with MB x NB blocks of 32 x 32 (v_mfma_scale_f32_32x32x64_f8f6f4, the weights
// first: a lane's 4 consecutive values are 4 columns of an output row). K runs in
// stages of 256 columns through LDS, two stages, filled by DMA.
template <bool BF16, int BM, int BN, int WGM>
__device__ __forceinline__ void product_tile(const Product &p, int2 tile, int64_t n0, uint8_t *sX0, uint8_t *sX1,
                                             uint8_t *sW0, uint8_t *sW1) {
  constexpr int WGN = 4 / WGM, WM = BM / WGM, WN = BN / WGN, MB = WM / 32, NB = WN / 32;
  constexpr int XD = BM / 32, WD = BN / 32;  // DMA instructions of a wave per stage
  const int lane = threadIdx.x & 63, li = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wm = wave / WGN, wn = wave % WGN;
  const int e = tile.x;
  const int64_t row0 = tile.y;
  const int m = static_cast<int>(min(p.ends[e] - row0, static_cast<int64_t>(BM)));
  const int n = static_cast<int>(min(p.N - n0, static_cast<int64_t>(BN)));
  const int kb = static_cast<int>(p.K / 2);         // bytes of a row's codes
  const int last = static_cast<int>(p.K / kBlock) - 1;  // its last 16-byte chunk
  const uint8_t *xc = p.xc + row0 * kb;
  const uint8_t *wc = p.wc + (e * p.N + n0) * kb;
  // Rows past the tile's repeat its last one: their products are not stored.
  int xoff[XD], woff[WD], chunk[2];
#pragma unroll
  for (int i = 0; i < XD; ++i) xoff[i] = min((wave * XD + i) * 8 + (lane >> 3), m - 1) * kb;
#pragma unroll
  for (int i = 0; i < WD; ++i) woff[i] = min((wave * WD + i) * 8 + (lane >> 3), n - 1) * kb;
#pragma unroll
  for (int i = 0; i < 2; ++i) chunk[i] = (lane & 7) ^ row_key(8 * i + (lane >> 3));
  static_assert(XD % 2 == 0 && WD % 2 == 0, "a DMA's rows begin at an even multiple of 8 for even i");
  auto load = [&](int k, uint8_t *sX, uint8_t *sW) __attribute__((always_inline)) {
    // Chunks past K repeat the last one: the steps they belong to are left out.
    const int c[2] = {16 * min(8 * k + chunk[0], last), 16 * min(8 * k + chunk[1], last)};
#pragma unroll
    for (int i = 0; i < XD; ++i) lds_dma16(xc + (xoff[i] + c[i & 1]), sX + (wave * XD + i) * 1024);
#pragma unroll
    for (int i = 0; i < WD; ++i) lds_dma16(wc + (woff[i] + c[i & 1]), sW + (wave * WD + i) * 1024);
  };
  // Scales of the wave's rows: the 8 bytes of a stage per lane and block of 32 rows.
  struct __attribute__((packed, aligned(2))) Eight {
    uint64_t v;
  };
  const uint8_t *xs[MB], *ws[NB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) xs[mb] = p.xs + (row0 + min(wm * WM + 32 * mb + li, m - 1)) * p.ldxs;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
    ws[nb] = p.ws + (e * p.N + n0 + min(wn * WN + 32 * nb + li, n - 1)) * (p.K / kBlock);
  const int KT = static_cast<int>((p.K + kStep - 1) / kStep);
  const int tail = static_cast<int>(p.K % kStep) / 64;  // 64-column steps of a short last stage
  struct Scales {
    uint64_t x[MB], w[NB];
  };
  auto load_scales = [&](int k, Scales &s) __attribute__((always_inline)) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) s.x[mb] = *reinterpret_cast<const uint64_t *>(xs[mb] + 8 * k);
    if (tail != 0 && k == KT - 1) {
      // A weight row's scales end with it.
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const uint16_t *q = reinterpret_cast<const uint16_t *>(ws[nb] + 8 * k);
        uint64_t v = q[0];
        if (tail > 1) v |= static_cast<uint64_t>(q[1]) << 16;
        if (tail > 2) v |= static_cast<uint64_t>(q[2]) << 32;
        s.w[nb] = v;
      }
    } else {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s.w[nb] = reinterpret_cast<const Eight *>(ws[nb] + 8 * k)->v;
    }
  };
  f32x16 acc[MB][NB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[mb][nb][j] = 0.0f;

  auto step = [&](int k, const uint8_t *sX, const uint8_t *sW, uint8_t *nX, uint8_t *nW, const Scales &cur,
                  Scales &nxt) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this stage has landed
    __syncthreads();
    if (k + 1 < KT) {
      load(k + 1, nX, nW);
      load_scales(k + 1, nxt);
    }
    const int subs = k == KT - 1 && tail != 0 ? tail : 4;
    // Byte 0 of a half word pair: the lane's block of its first step; byte 2: of the second.
    int sx[2][MB], sw[2][NB];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) sx[i][mb] = static_cast<int>(static_cast<uint32_t>(cur.x[mb] >> (32 * i)) >> (8 * h));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) sw[i][nb] = static_cast<int>(static_cast<uint32_t>(cur.w[nb] >> (32 * i)) >> (8 * h));
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s >= subs) break;
      i32x8 x[MB], w[NB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) x[mb] = fragment(sX, wm * WM + 32 * mb + li, 2 * s + h);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) w[nb] = fragment(sW, wn * WN + 32 * nb + li, 2 * s + h);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          if (s & 1)
            acc[mb][nb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                w[nb], x[mb], acc[mb][nb], 4, 4, 2, sw[s >> 1][nb], 2, sx[s >> 1][mb]);
          else
            acc[mb][nb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                w[nb], x[mb], acc[mb][nb], 4, 4, 0, sw[s >> 1][nb], 0, sx[s >> 1][mb]);
    }
  };
  Scales s0, s1;
  load(0, sX0, sW0);
  load_scales(0, s0);
  int k = 0;
  for (; k + 1 < KT; k += 2) {
    step(k, sX0, sW0, sX1, sW1, s0, s1);
    step(k + 1, sX1, sW1, sX0, sW0, s1, s0);
  }
  if (k < KT) step(k, sX0, sW0, sX1, sW1, s0, s1);

  // Each wave turns 32 rows at a time over in its part of LDS, so that a row's
  // columns leave in runs of WN values.
  constexpr int ES = BF16 ? 2 : 4, CH = WN * ES / 16;  // 16-byte chunks of a row
  __syncthreads();
  uint8_t *strip = wave == 0 ? sX0 : wave == 1 ? sX1 : wave == 2 ? sW0 : sW1;
  auto place = [&](int row, int c) { return row * (CH * 16) + ((c ^ (row & (CH - 1))) << 4); };
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
#pragma unroll
    for (int i = 0; i < 32 * CH / 64; ++i) {
      const int row = (64 * i + lane) / CH, c = lane % CH;
      const int r = wm * WM + 32 * mb + row, col = wn * WN + c * (16 / ES);
      const u32x4 q = *reinterpret_cast<const u32x4 *>(strip + place(row, c));
      if (r < m && col < n)
        *reinterpret_cast<u32x4 *>(static_cast<uint8_t *>(p.out) + ((row0 + r) * p.N + n0 + col) * ES) = q;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// Workgroups go to the 8 XCDs in turn; each XCD takes a run of the tall tiles and
// then a run of the short ones, column tiles of one row tile side by side, so that
// the rows of a tile and the weights of an expert are read through one L2.
template <bool BF16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void product_kernel(Product p) {
  __shared__ __attribute__((aligned(16))) uint8_t sX0[kTall * 128], sX1[kTall * 128];
  __shared__ __attribute__((aligned(16))) uint8_t sW0[kTall * 128], sW1[kTall * 128];
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
  const int total_t = p.head[1] * p.n_tiles_n, total_s = p.head[2] * p.n_tiles_n;
  const int per_t = (total_t + 7) >> 3, per_s = (total_s + 7) >> 3;
  const bool tall = slot < per_t;
  const int logical = tall ? xcd * per_t + slot : xcd * per_s + slot - per_t;
  if (!tall && slot >= per_t + per_s) return;
  if (logical >= (tall ? total_t : total_s)) return;
  const int mt = logical / p.n_tiles_n;
  const int2 tile = (tall ? p.tall : p.rest)[mt];
  const int64_t n0 = static_cast<int64_t>(logical - mt * p.n_tiles_n) * 256;
  const bool half = p.N - n0 <= 128;
  if (tall) {
    if (half)
      product_tile<BF16, 256, 128, 2>(p, tile, n0, sX0, sX1, sW0, sW1);
    else
      product_tile<BF16, 256, 256, 2>(p, tile, n0, sX0, sX1, sW0, sW1);
  } else {
    if (half)
      product_tile<BF16, 128, 128, 2>(p, tile, n0, sX0, sX1, sW0, sW1);
    else
      product_tile<BF16, 128, 256, 2>(p, tile, n0, sX0, sX1, sW0, sW1);
  }
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
  const bool vec = aligned16(x) && (ldx * (bf16 ? 2 : 4)) % 16 == 0;
  auto kernel = bf16 ? quantize_kernel<true> : quantize_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, as_stream(stream), x,
                     rows, cols, ldx, vec, codes, scales);
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
  const bool vec = aligned16(out) && (cols * (bf16 ? 2 : 4)) % 16 == 0;
  auto kernel = bf16 ? dequantize_kernel<true> : dequantize_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, as_stream(stream),
                     codes, scales, rows, cols, vec, out);
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
  if (!aligned16(w->data) || !aligned16(out) || !aligned16(workspace)) {
    set_error("%s: weight codes, output and workspace must be 16-byte aligned", name);
    return MX_ERR_INVALID;
  }
  hipStream_t s = as_stream(stream);
  const Layout L = layout(num_rows, num_experts, K);
  char *base = static_cast<char *>(workspace);
  uint8_t *codes = reinterpret_cast<uint8_t *>(base + L.off_codes);
  uint8_t *scales = reinterpret_cast<uint8_t *>(base + L.off_scales);
  PlanOut P = {offsets, offsets_64 != 0, num_rows, num_experts, reinterpret_cast<int32_t *>(base),
               reinterpret_cast<int64_t *>(base + L.off_ends), reinterpret_cast<int2 *>(base + L.off_tall),
               reinterpret_cast<int2 *>(base + L.off_short), host_err};
  const int64_t chunks = ceil_div(num_rows * (K / 8), 256 * kUnroll);
  const int64_t n_tiles = ceil_div(N, 256);
  const int64_t grid = 8 * (ceil_div(L.max_tall * n_tiles, 8) + ceil_div(L.max_short * n_tiles, 8));
  if (int rc = grid_ok(name, std::max(chunks + 1, grid))) return rc;
  const bool bf16 = x_dtype == MX_DTYPE_BF16;
  auto rows_k = bf16 ? rows_kernel<true> : rows_kernel<false>;
  hipLaunchKernelGGL(rows_k, dim3(static_cast<unsigned>(chunks + 1)), dim3(256), 0, s, x, num_rows, K,
                     aligned16(x), codes, scales, L.ldxs, P);
  if (int rc = check_launch(name)) return rc;
  Product p = {codes, scales, L.ldxs, static_cast<const uint8_t *>(w->data),
               static_cast<const uint8_t *>(w->scale), K, N, P.head, P.ends, P.tall, P.rest,
               static_cast<int>(n_tiles), out};
  auto product = out_dtype == MX_DTYPE_BF16 ? product_kernel<true> : product_kernel<false>;
  hipLaunchKernelGGL(product, dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, p);
  return check_launch(name);
}
