// AdamW over many tensors per launch, moments in fp32 or in 8-bit blocks.
//
// A launch takes up to kMaxTensors tensors by value and cuts them into chunks of
// kChunk elements, one per workgroup: no table is uploaded, and a captured launch
// holds all that it needs. The step is one pass over p, g and the moments, so it is
// bound by memory: 28 bytes per element with fp32 tensors and moments, 16 with 8-bit
// moments. A thread has two runs of 8 elements under way, 16 lanes hold a block of the
// 8-bit moments. 255 M elements in 144 tensors (24 layers of 64 experts, rank 16), two
// launches: 1180 us with fp32 moments (6.0 TB/s), 720 to 860 with 8-bit ones (4.8 to
// 5.7), where a large copy reaches 5.1; 6 tensors of 49152 elements 5.2 us.
#include <math.h>

#include <algorithm>

#include "common.h"

namespace mx {
namespace adamw {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;     // consecutive elements of a thread
constexpr int kUnroll = 2;  // such runs per thread
constexpr int kChunk = kThreads * kVec * kUnroll;
constexpr int kBlock = 128;  // elements under one exponent: 16 lanes
constexpr int kMaxTensors = 88;

struct Tensor {
  void *p;
  const void *g;
  int64_t n, at;
  int32_t index, first_chunk;
};

// What a step's elements share.
struct Scalars {
  float step_size;  // lr / (1 - b1^t)
  float root;       // 1 / sqrt(1 - b2^t)
  float decay;      // 1 - lr wd
  uint32_t key;
};

struct Args {
  Tensor t[kMaxTensors];
  int count;
  float b1, c1, b2, c2, eps;  // c = 1 - b
  Scalars s;
  const Scalars *device;  // capturable: [index] instead of s
  void *m, *v;
  uint8_t *me, *ve;
};
static_assert(sizeof(Args) <= 4096, "kernel arguments");

__host__ __device__ inline uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x9E3779B9u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

__host__ __device__ inline Scalars scalars(double lr, double b1, double b2, double wd, int64_t step,
                                           uint32_t seed, uint32_t group) {
  Scalars s;
  s.step_size = static_cast<float>(lr / (1.0 - pow(b1, static_cast<double>(step))));
  s.root = static_cast<float>(1.0 / sqrt(1.0 - pow(b2, static_cast<double>(step))));
  s.decay = static_cast<float>(1.0 - lr * wd);
  s.key = mix(mix(seed) + static_cast<uint32_t>(step));
  if (group != 0) s.key = mix(s.key + group);
  return s;
}

// The tensor of a chunk: the last one whose first chunk is not past it. The lanes
// look at 64 tensors at a time.
__device__ __forceinline__ int tensor_of(const Args &a, int chunk) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int i = 0; i < a.count; i += 64) {
    const bool le = i + lane < a.count && a.t[i + lane < a.count ? i + lane : 0].first_chunk <= chunk;
    before += __popcll(__ballot(le));
  }
  return __builtin_amdgcn_readfirstlane(before - 1);
}

template <bool BF16>
__device__ __forceinline__ void load(const void *p, int64_t i, int n, float (&x)[kVec]) {
  if (n >= kVec) {
    if constexpr (BF16) {
      const u32x4 q = *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(q[j] << 16);
        x[2 * j + 1] = __uint_as_float(q[j] & 0xffff0000u);
      }
    } else {
      const f32x4_any *q = reinterpret_cast<const f32x4_any *>(static_cast<const float *>(p) + i);
      const f32x4 lo = q[0], hi = q[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = lo[j];
        x[j + 4] = hi[j];
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    if constexpr (BF16)
      x[j] = j < n ? bf16_bits_to_f32(static_cast<const uint16_t *>(p)[i + j]) : 0.0f;
    else
      x[j] = j < n ? static_cast<const float *>(p)[i + j] : 0.0f;
  }
}

template <bool BF16>
__device__ __forceinline__ void store(void *p, int64_t i, int n, const float (&x)[kVec]) {
  if (n >= kVec) {
    if constexpr (BF16) {
      *reinterpret_cast<u32x4_any *>(static_cast<uint16_t *>(p) + i) =
          u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                pack_bf16x2(x[6], x[7])};
    } else {
      f32x4_any *q = reinterpret_cast<f32x4_any *>(static_cast<float *>(p) + i);
      q[0] = f32x4{x[0], x[1], x[2], x[3]};
      q[1] = f32x4{x[4], x[5], x[6], x[7]};
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j)
    if (j < n) {
      if constexpr (BF16)
        static_cast<uint16_t *>(p)[i + j] = f32_to_bf16_bits(x[j]);
      else
        static_cast<float *>(p)[i + j] = x[j];
    }
}

// m', v' with every operation rounded, p' from them.
__device__ __forceinline__ void update(const Args &a, const Scalars &s, float g, float &p, float &m,
                                       float &v) {
#pragma clang fp contract(off)
  m = m * a.b1 + g * a.c1;
  v = v * a.b2 + (g * a.c2) * g;
  p = p * s.decay - s.step_size * (m / (sqrtf(v) * s.root + a.eps));
}

// ------------------------------------------------------- 8-bit block floats
// A code holds EB exponent and 3 fraction bits (below a sign, if any) of y = |x| /
// 2^E: y in [2^LOW, 2) with LOW = 2 - 2^EB, and eighths of 2^LOW below it.
template <int EB>
__device__ __forceinline__ float low_value() {
  return __uint_as_float(static_cast<uint32_t>(2 - (1 << EB) + 127) << 23);
}

template <int EB>
__device__ __forceinline__ float decode(uint32_t mag) {
  // Normal codes are the top bits of an fp32 number whose exponent runs from LOW on
  // for exponent 1; exponent 0 counts from 2^LOW, which is taken off again.
  constexpr uint32_t base = static_cast<uint32_t>(2 - (1 << EB) + 127) << 23;
  const bool sub = mag < 8;
  const float y = __uint_as_float((mag << 20) + base - (sub ? 0u : 1u << 23));
  return sub ? y - low_value<EB>() : y;
}

// y >= 0 with 16 random bits -> code: the 20 dropped fraction bits are rounded up
// with a probability of their value.
template <int EB>
__device__ __forceinline__ uint32_t encode(float y, uint32_t noise) {
  constexpr uint32_t base = static_cast<uint32_t>(2 - (1 << EB) + 127) << 3;
  const float low = low_value<EB>();
  const bool sub = y < low;
  const uint32_t bits = __float_as_uint(sub ? y + low : y) + (noise << 4);
  const uint32_t code = (bits >> 20) - base + (sub ? 0u : 8u);
  return min(code, (8u << EB) - 1u);
}

// Largest |x| bits over the 16 lanes of a block.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  auto step = [&](int o) { v = max(v, static_cast<uint32_t>(o)); };
  step(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xf, 0xf, true));   // lane ^ 1
  step(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xf, 0xf, true));   // lane ^ 2
  step(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xf, 0xf, true));  // mirrored half row
  step(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 0xf, 0xf, true));  // mirrored row
  return v;
}

// The stored exponent of a block from the bits of its largest magnitude.
__device__ __forceinline__ uint32_t block_exponent(uint32_t bits) {
  const uint32_t field = bits >> 23;
  return field == 255 ? 255 : min(max(field, 1u), 253u);
}
__device__ __forceinline__ float pow2(uint32_t field) { return __uint_as_float(field << 23); }
// 2^-E of a stored exponent in [1, 253].
__device__ __forceinline__ float inverse_pow2(uint32_t stored) { return pow2(254u - stored); }

template <int EB, bool SIGNED>
__device__ __forceinline__ void unpack(uint2 c, uint32_t e, float (&x)[kVec]) {
  const float s = e == 255 ? __uint_as_float(0x7fc00000u) : pow2(e);
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const uint32_t b = ((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 0xffu;
    const float y = decode<EB>(SIGNED ? b & 0x7fu : b) * s;
    x[j] = SIGNED && (b & 0x80u) ? -y : y;
  }
}

template <int EB, bool SIGNED>
__device__ __forceinline__ uint2 pack(const float (&x)[kVec], const uint32_t (&noise)[kVec], uint32_t e) {
  uint2 c = {0u, 0u};
  if (e == 255) return c;
  const float s = inverse_pow2(e);
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    uint32_t b = encode<EB>(fabsf(x[j]) * s, noise[j]);
    if (SIGNED) b |= (__float_as_uint(x[j]) >> 24) & 0x80u;
    (j < 4 ? c.x : c.y) |= b << (8 * (j & 3));
  }
  return c;
}

__device__ __forceinline__ uint32_t largest(const float (&x)[kVec]) {
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < kVec; ++j) a = max(a, __float_as_uint(x[j]) & 0x7fffffffu);
  return a;
}

template <bool BF16, bool STATE8>
__global__ __launch_bounds__(kThreads) void step_kernel(Args a) {
  const int ti = tensor_of(a, blockIdx.x);
  const Tensor t = a.t[ti];
  const Scalars s = a.device ? a.device[t.index] : a.s;
  const int64_t i0 = static_cast<int64_t>(static_cast<int>(blockIdx.x) - t.first_chunk) * kChunk +
                     kVec * static_cast<int64_t>(threadIdx.x);
  // The runs' places: whole blocks are taken, their elements past n as zeros.
  const int64_t padded = (t.n + kBlock - 1) / kBlock * kBlock;
  float p[kUnroll][kVec], g[kUnroll][kVec], m[kUnroll][kVec], v[kUnroll][kVec];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = i0 + u * (kThreads * kVec);
    if (i >= padded) break;
    const int n = static_cast<int>(max(min(t.n - i, int64_t(kVec)), int64_t(0)));
    load<BF16>(t.p, i, n, p[u]);
    load<BF16>(t.g, i, n, g[u]);
    const int64_t at = t.at + i;
    if constexpr (STATE8) {
      unpack<4, true>(*reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.m) + at),
                      a.me[at / kBlock], m[u]);
      unpack<5, false>(*reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(a.v) + at),
                       a.ve[at / kBlock], v[u]);
    } else {
      load<false>(a.m, at, kVec, m[u]);
      load<false>(a.v, at, kVec, v[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = i0 + u * (kThreads * kVec);
    if (i >= padded) break;
    const int n = static_cast<int>(max(min(t.n - i, int64_t(kVec)), int64_t(0)));
    const int64_t at = t.at + i;
#pragma unroll
    for (int j = 0; j < kVec; ++j) update(a, s, g[u][j], p[u][j], m[u][j], v[u][j]);
    store<BF16>(t.p, i, n, p[u]);
    if constexpr (STATE8) {
      // Padding stays zero.
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (j >= n) m[u][j] = v[u][j] = 0.0f;
      const uint32_t key = at >> 32 ? mix(s.key + static_cast<uint32_t>(at >> 32)) : s.key;
      uint32_t low[kVec], high[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const uint32_t r = mix(static_cast<uint32_t>(at) + j + key);
        low[j] = r & 0xffffu;
        high[j] = r >> 16;
      }
      const uint32_t me = block_exponent(max16(largest(m[u])));
      const uint32_t ve = block_exponent(max16(largest(v[u])));
      *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(a.m) + at) = pack<4, true>(m[u], low, me);
      *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(a.v) + at) = pack<5, false>(v[u], high, ve);
      if ((threadIdx.x & 15) == 0) {
        a.me[at / kBlock] = static_cast<uint8_t>(me);
        a.ve[at / kBlock] = static_cast<uint8_t>(ve);
      }
    } else {
      store<false>(a.m, at, kVec, m[u]);
      store<false>(a.v, at, kVec, v[u]);
    }
  }
}

struct AdvanceArgs {
  int64_t *steps;
  Scalars *out;
  const float *lr_ptr;
  double lr, b1, b2, wd;
  uint32_t seed, group;
  int count;
  int32_t index[512];
};

// Capturable steps: counts one more step of each tensor and leaves its scalars.
__global__ __launch_bounds__(256) void advance_kernel(AdvanceArgs a) {
  for (int i = threadIdx.x; i < a.count; i += 256) {
    const int k = a.index[i];
    const int64_t step = ++a.steps[k];
    const double lr = a.lr_ptr ? static_cast<double>(*a.lr_ptr) : a.lr;
    a.out[k] = scalars(lr, a.b1, a.b2, a.wd, step, a.seed, a.group);
  }
}

// The fp32 values of 8-bit moments: bound by its writes, 255 M elements 221 us (5.8
// TB/s).
template <int EB, bool SIGNED>
__global__ __launch_bounds__(256) void moments_kernel(const uint8_t *codes, const uint8_t *exponents,
                                                      int64_t runs, float *out) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (r >= runs) return;
  float x[kVec];
  unpack<EB, SIGNED>(reinterpret_cast<const uint2 *>(codes)[r], exponents[r / (kBlock / kVec)], x);
  store<false>(out, kVec * r, kVec, x);
}

bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int invalid(const char *what) {
  set_error("mx_adamw_step: %s", what);
  return MX_ERR_INVALID;
}

}  // namespace
}  // namespace adamw
}  // namespace mx

using namespace mx;
using namespace mx::adamw;

extern "C" int mx_adamw_step(const mx_adamw_tensor *tensors, int count, const mx_adamw_config *c,
                             void *stream) {
  clear_error();
  if (count < 0 || (count > 0 && !tensors) || !c) return invalid("tensors and configuration are missing");
  if (c->dtype != MX_DTYPE_BF16 && c->dtype != MX_DTYPE_F32) return invalid("tensors must be bf16 or fp32");
  if (c->state_bits != 32 && c->state_bits != 8) return invalid("state_bits must be 32 or 8");
  const bool state8 = c->state_bits == 8;
  if (!(c->beta1 >= 0.0 && c->beta1 < 1.0 && c->beta2 >= 0.0 && c->beta2 < 1.0) || !(c->eps >= 0.0))
    return invalid("betas must be in [0, 1) and eps not negative");
  if (!c->steps && c->step < 1) return invalid("steps count from 1");
  if (c->steps && !c->scalars) return invalid("device steps need their scalars");
  if (count == 0) return MX_OK;
  if (!c->exp_avg || !c->exp_avg_sq || (state8 && (!c->exp_avg_e || !c->exp_avg_sq_e)))
    return invalid("the moments are missing");
  if (!aligned(c->exp_avg, 16) || !aligned(c->exp_avg_sq, 16)) return invalid("moments must be 16-byte aligned");
  const size_t es = c->dtype == MX_DTYPE_BF16 ? 2 : 4;
  for (int i = 0; i < count; ++i) {
    const mx_adamw_tensor &t = tensors[i];
    if (t.n < 0 || t.at < 0 || t.at % kBlock != 0 || (t.n > 0 && (!t.p || !t.g)) ||
        !aligned(t.p, es) || !aligned(t.g, es) || t.index < 0 || t.index > 0x7fffffff)
      return invalid("a tensor needs its addresses, n >= 0 and a place that is a multiple of 128");
    if (t.n / kChunk >= 0x40000000) return invalid("a tensor is too large");
  }
  hipStream_t s = as_stream(stream);
  if (c->steps) {
    AdvanceArgs a = {c->steps, static_cast<Scalars *>(c->scalars), c->lr_ptr, c->lr, c->beta1, c->beta2,
                     c->weight_decay, c->seed, c->group, 0, {}};
    for (int i = 0; i < count; i += 512) {
      a.count = std::min(512, count - i);
      for (int j = 0; j < a.count; ++j) a.index[j] = static_cast<int32_t>(tensors[i + j].index);
      hipLaunchKernelGGL(advance_kernel, dim3(1), dim3(256), 0, s, a);
      if (int rc = check_launch("mx_adamw_step")) return rc;
    }
  }
  Args a = {};
  a.b1 = static_cast<float>(c->beta1);
  a.c1 = static_cast<float>(1.0 - c->beta1);
  a.b2 = static_cast<float>(c->beta2);
  a.c2 = static_cast<float>(1.0 - c->beta2);
  a.eps = static_cast<float>(c->eps);
  if (c->steps)
    a.device = static_cast<const Scalars *>(c->scalars);
  else
    a.s = scalars(c->lr, c->beta1, c->beta2, c->weight_decay, c->step, c->seed, c->group);
  a.m = c->exp_avg;
  a.v = c->exp_avg_sq;
  a.me = c->exp_avg_e;
  a.ve = c->exp_avg_sq_e;
  const bool bf16 = c->dtype == MX_DTYPE_BF16;
  auto kernel = bf16 ? (state8 ? step_kernel<true, true> : step_kernel<true, false>)
                     : (state8 ? step_kernel<false, true> : step_kernel<false, false>);
  for (int i = 0; i < count;) {
    a.count = 0;
    int64_t chunks = 0;
    for (; i < count && a.count < kMaxTensors; ++i) {
      const mx_adamw_tensor &t = tensors[i];
      const int64_t more = ceil_div(t.n, kChunk);
      if (more == 0) continue;
      if (chunks + more > 0x7fffffff) break;
      a.t[a.count++] = {t.p, t.g, t.n, t.at, static_cast<int32_t>(t.index), static_cast<int32_t>(chunks)};
      chunks += more;
    }
    if (a.count == 0) continue;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(chunks)), dim3(kThreads), 0, s, a);
    if (int rc = check_launch("mx_adamw_step")) return rc;
  }
  return MX_OK;
}

extern "C" int mx_adamw_moments(const uint8_t *codes, const uint8_t *exponents, int64_t n, int is_signed,
                                float *out, void *stream) {
  clear_error();
  if (n < 0 || n % kBlock != 0 || (n > 0 && (!codes || !exponents || !out)) || !aligned(codes, 8) ||
      !aligned(out, 16)) {
    set_error("mx_adamw_moments: need n a multiple of 128, non-null buffers, codes 8-byte and out "
              "16-byte aligned");
    return MX_ERR_INVALID;
  }
  if (n == 0) return MX_OK;
  const int64_t runs = n / kVec, blocks = ceil_div(runs, 256);
  if (blocks > 0x7fffffff) {
    set_error("mx_adamw_moments: too many elements for one launch");
    return MX_ERR_INVALID;
  }
  auto kernel = is_signed ? moments_kernel<4, true> : moments_kernel<5, false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, as_stream(stream), codes,
                     exponents, runs, out);
  return check_launch("mx_adamw_moments");
}
