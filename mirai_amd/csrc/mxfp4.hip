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
                                                uint8_t *scales, int64_t chunk) {
  const int64_t per_row = 4 * ((cols + kBlock - 1) / kBlock);
  const int64_t total = rows * per_row;
  const bool flat = vec && ldx == cols && cols % kBlock == 0;
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
    const int64_t row = total <= 0xffffffffll
                            ? static_cast<uint32_t>(g) / static_cast<uint32_t>(per_row)
                            : g / per_row;
    const int64_t col = 8 * (g - row * per_row);
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
    if ((g & 3) == 0) scales[g >> 2] = static_cast<uint8_t>(scale);
  }
}

template <bool BF16>
__global__ __launch_bounds__(256) void quantize_kernel(const void *x, int64_t rows, int64_t cols,
                                                       int64_t ldx, bool vec, uint8_t *codes,
                                                       uint8_t *scales) {
  quantize_groups<BF16>(x, rows, cols, ldx, vec, codes, scales, blockIdx.x);
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
constexpr int kTileRows = 32;

// Workspace: a head of 256 bytes (int32 errors, int32 tiles), the segment ends as
// the tiles use them, the tile list, the rows' codes and scales.
struct Layout {
  int64_t max_tiles = 0;
  size_t off_ends = 0, off_tiles = 0, off_codes = 0, off_scales = 0, bytes = 0;
};

Layout layout(int64_t rows, int experts, int64_t in_f) {
  Layout L;
  L.max_tiles = std::min(rows, rows / kTileRows + experts);
  size_t off = 256;
  L.off_ends = off;
  off = align_up(off + sizeof(int64_t) * experts, 256);
  L.off_tiles = off;
  off = align_up(off + sizeof(int2) * L.max_tiles, 256);
  L.off_codes = off;
  off = align_up(off + rows * (in_f / 2), 256);
  L.off_scales = off;
  off = align_up(off + rows * (in_f / kBlock), 256);
  L.bytes = off;
  return L;
}

struct PlanOut {
  const void *offsets;
  bool wide;  // int64 offsets
  int64_t rows;
  int experts;
  int32_t *head;  // errors, tiles
  int64_t *ends;
  int2 *tiles;
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
  int64_t start = before, tiles = 0, bad = 0;
  for (int e = e0; e < e1; ++e) {
    const int64_t r = raw(e), end = max(start, held(r));
    bad += r < start || r > P.rows;
    P.ends[e] = end;
    tiles += (end - start + kTileRows - 1) / kTileRows;
    start = end;
  }
  auto add = [](int64_t a, int64_t b) { return a + b; };
  const int64_t tiles_upto = scan256(tiles, buf, add);
  const int64_t bad_upto = scan256(bad, buf, add);
  int64_t at = tiles_upto - tiles;
  start = before;
  for (int e = e0; e < e1; ++e) {
    const int64_t end = max(start, held(raw(e)));
    for (int64_t r = start; r < end; r += kTileRows) P.tiles[at++] = int2{e, static_cast<int>(r)};
    start = end;
  }
  if (threadIdx.x == 255) {
    const int32_t errors = static_cast<int32_t>(bad_upto + (last != P.rows));
    P.head[0] = errors;
    P.head[1] = static_cast<int32_t>(tiles_upto);
    if (P.host_err) __hip_atomic_store(P.host_err, errors, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
  }
}

// The rows' quantisation; the last workgroup forms the tile list meanwhile.
template <bool BF16>
__global__ __launch_bounds__(256) void rows_kernel(const void *x, int64_t rows, int64_t cols, bool vec,
                                                   uint8_t *codes, uint8_t *scales, PlanOut P) {
  if (blockIdx.x == gridDim.x - 1) {
    plan_tiles(P);
    return;
  }
  quantize_groups<BF16>(x, rows, cols, cols, vec, codes, scales, blockIdx.x);
}

struct Product {
  const uint8_t *xc, *xs;  // [S, K/2], [S, K/32]
  const uint8_t *wc, *ws;  // [E, N, K/2], [E, N, K/32]
  int64_t K, N;
  const int32_t *head;
  const int64_t *ends;
  const int2 *tiles;
  int n_tiles_n;
  void *out;
};

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 operand(const uint8_t *p) {
  const u32x4 q = *reinterpret_cast<const u32x4 *>(p);
  return i32x8{static_cast<int>(q[0]), static_cast<int>(q[1]), static_cast<int>(q[2]),
               static_cast<int>(q[3]), 0, 0, 0, 0};
}

// Four columns of an output row from n0 on.
template <bool BF16>
__device__ __forceinline__ void store4(void *out, int64_t at, const float (&v)[4]) {
  if constexpr (BF16) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(out) + at) =
        u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  } else {
    *reinterpret_cast<f32x4 *>(static_cast<float *>(out) + at) = f32x4{v[0], v[1], v[2], v[3]};
  }
}

// A wave multiplies 32 weight rows with a tile of up to 32 token rows, straight
// from memory: lane l holds row l % 32 and, of each 64 columns, block l / 32.
template <bool BF16>
__global__ __launch_bounds__(256) void product_kernel(Product p) {
  const int total = p.head[1] * p.n_tiles_n;
  if (static_cast<int>(blockIdx.x) >= total) return;
  const int mt = blockIdx.x / p.n_tiles_n, nt = blockIdx.x - mt * p.n_tiles_n;
  const int2 tile = p.tiles[mt];
  const int lane = threadIdx.x & 63, li = lane & 31, h = lane >> 5;
  const int64_t n_base = static_cast<int64_t>(nt) * 128 + 32 * (threadIdx.x >> 6);
  if (n_base >= p.N) return;
  const int64_t end = p.ends[tile.x];
  // Rows past the segment and past N repeat the last one; their products are dropped.
  const int64_t xrow = min(tile.y + static_cast<int64_t>(li), end - 1);
  const int64_t wrow = tile.x * p.N + min(n_base + li, p.N - 1);
  const uint8_t *xc = p.xc + xrow * (p.K / 2) + 16 * h, *xs = p.xs + xrow * (p.K / kBlock) + h;
  const uint8_t *wc = p.wc + wrow * (p.K / 2) + 16 * h, *ws = p.ws + wrow * (p.K / kBlock) + h;
  f32x16 acc;
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.0f;
  for (int64_t k = 0; k < p.K / 64; ++k)
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(wc + 32 * k), operand(xc + 32 * k),
                                                          acc, 4, 4, 0, ws[2 * k], 0, xs[2 * k]);
  const int64_t r = tile.y + static_cast<int64_t>(li);
  if (r >= end) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int64_t n0 = n_base + 8 * g + 4 * h;
    const float v[4] = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
    if (n0 < p.N) store4<BF16>(p.out, r * p.N + n0, v);
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
               reinterpret_cast<int64_t *>(base + L.off_ends), reinterpret_cast<int2 *>(base + L.off_tiles),
               host_err};
  const int64_t chunks = ceil_div(num_rows * (K / 8), 256 * kUnroll);
  const int64_t n_tiles = ceil_div(N, 128);
  if (int rc = grid_ok(name, std::max(chunks + 1, L.max_tiles * n_tiles))) return rc;
  const bool bf16 = x_dtype == MX_DTYPE_BF16;
  auto rows_k = bf16 ? rows_kernel<true> : rows_kernel<false>;
  hipLaunchKernelGGL(rows_k, dim3(static_cast<unsigned>(chunks + 1)), dim3(256), 0, s, x, num_rows, K,
                     aligned16(x), codes, scales, P);
  if (int rc = check_launch(name)) return rc;
  Product p = {codes, scales, static_cast<const uint8_t *>(w->data), static_cast<const uint8_t *>(w->scale),
               K, N, P.head, P.ends, P.tiles, static_cast<int>(n_tiles), out};
  auto product = out_dtype == MX_DTYPE_BF16 ? product_kernel<true> : product_kernel<false>;
  hipLaunchKernelGGL(product, dim3(static_cast<unsigned>(L.max_tiles * n_tiles)), dim3(256), 0, s, p);
  return check_launch(name);
}
