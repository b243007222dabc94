// Activations held in 8 bits between the forward and the backward pass, and the
// GELU around them (gfx950).
//
// Blocks of 32 channels share a step 2^(floor(log2 m) - 6), m the block's largest
// magnitude; a channel is the nearest whole multiple of the step (half to even),
// at most 127, in int8, and the step's exponent is one byte (value 2^(byte -
// 127), 0 at least; 255 marks a block with an infinity or NaN, which stands for 32
// NaNs).  Division by a power of two is exact, so the held numbers do not depend
// on how they were computed; they differ from the activation by at most m / 128.
// A row's last block may be short.
//
//   gelu(u) = u Phi(u), from the exact u
//   gelu'(h) = Phi(h) + h phi(h), from the held h;  du = dy gelu'(h)
//
// The kernels move bytes: per 16-bit element 3 + 1/32 (pack, unpack), 5 + 1/32 (GELU,
// either way), 4 for the GELU alone, where no backward pass will read the 8 bits.  A
// thread has 8 channels, four threads a block: its largest magnitude takes two lane
// exchanges inside the quad.  16384 x 2048 bf16: 18 us to pack, 17 to
// unpack (5.6 and 6.0 TB/s; a copy reaches 5.2); the GELU of 16384 x 8192 110 to 140
// us forward, 120 to 150 backward (4.8 to 6.1 and 4.5 to 5.6 TB/s, by where its 700 MB
// meet the 256 MB of the last cache).  Past the caches a pass over both took 242 us
// instead of 249, but the training step of 12 layers that holds it 28.5 ms instead of
// 28.1: the products behind it find less of their inputs.
#include "saf_kernels.h"
#include "saf_rowio.h"

namespace saf {

namespace {

// Phi(u) and exp(-u^2 / 2): for a = |u| the tail Phi(-a) = exp(-a^2 / 2) t P(t),
// t = 1 / (1 + c a), P fitted to erfcx(a / sqrt 2) / (2 t) for its largest relative
// error over 0 <= a <= 14.5, so that small results far below zero keep their digits.
// 16-bit types: degree 5, 8.9e-6; evaluated in float32, where u^2 is rounded ahead of the
// exponential, 9.2e-6 up to a = 3, 1.1e-5 up to 8 and 1.4e-5 up to 13 (1/35 of half an
// fp16 step).
// float32: degree 8, 5.5e-8 with the coefficients as they are in float32; the tail is
// within 16 float32 roundings (2^-24) by their count, 6.2 at most in 400001 arguments
// down to -12.5, as what the square and the product lose is given back to the exponential
// (125 without).  With the library's erfc and exp in its place 16384 x 4096 float32 took
// 146 us forward and 166 backward, 113 and 112 so (5.4 TB/s).
template <bool EXACT>
__device__ inline float normal_cdf(float u, float& e) {
  if constexpr (EXACT) {
    constexpr float kHi = -0.7213475108146667f, kLo = -9.629815167500055e-09f;  // -log2(e) / 2
    const float a = fminf(fabsf(u), 20.f);  // behind it nothing is left, and the square stays finite
    const float s = a * a, x = s * kHi;
    const float rest = fmaf(s, kHi, -x) + fmaf(s, kLo, fmaf(a, a, -s) * kHi);
    e = fast_exp2(x);
    e = fmaf(e, rest * 0.6931471805599453f, e);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, a, 1.f));
    float h = -0.029157886281609535f;
    h = fmaf(h, t, 0.14403091371059418f);
    h = fmaf(h, t, -0.2558389902114868f);
    h = fmaf(h, t, 0.1593196988105774f);
    h = fmaf(h, t, -0.023212352767586708f);
    h = fmaf(h, t, 0.10555250197649002f);
    h = fmaf(h, t, 0.11982128769159317f);
    h = fmaf(h, t, 0.139863520860672f);
    h = fmaf(h, t, 0.139621302485466f);
    h *= t * e;
    return u < 0.f ? h : 1.f - h;
  } else {
    const float a = fabsf(u);
    e = fast_exp2(u * u * (-0.5f * kLog2e));
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.f));
    float h = -0.07670057564973831f;
    h = fmaf(h, t, 0.21484895050525665f);
    h = fmaf(h, t, -0.015597553923726082f);
    h = fmaf(h, t, 0.14347337186336517f);
    h = fmaf(h, t, 0.11392282694578171f);
    h = fmaf(h, t, 0.12005741894245148f);
    h *= t * e;
    return u < 0.f ? h : 1.f - h;
  }
}

template <typename T> constexpr bool kExact = sizeof(T) == 4;

// 2^(byte - 127) and its reciprocal
__device__ inline float step_of(uint32_t byte) { return byte ? __uint_as_float(byte << 23) : __uint_as_float(1u << 22); }
__device__ inline float per_step(uint32_t byte) { return __uint_as_float((254 - byte) << 23); }

template <int CTRL>
__device__ inline uint32_t quad_umax(uint32_t x) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
  return x > o ? x : o;
}

// The block's exponent byte and this thread's eight multiples; the four threads
// of a quad hold one block (channels past the row as zeros).
__device__ inline uint32_t pack8(const float (&f)[8], u32x2_any& q) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(f[e]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  top = quad_umax<0xb1>(top);
  top = quad_umax<0x4e>(top);
  const uint32_t ex = top >> 23;
  if (ex == 255) {
    q = 0;
    return 255;
  }
  const uint32_t byte = ex > 6 ? ex - 6 : 0;
  const float k = per_step(byte);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint32_t r = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = fminf(fmaxf(rintf(f[4 * w + e] * k), -127.f), 127.f);
      r |= ((uint32_t)(int)x & 0xffu) << (8 * e);
    }
    q[w] = r;
  }
  return byte;
}

__device__ inline void unpack8(const u32x2_any q, uint32_t byte, float (&f)[8]) {
  const float step = byte == 255 ? __uint_as_float(0x7fc00000u) : step_of(byte);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(q[e >> 2] >> (8 * (e & 3))) * step;
}

// Eight bytes of a row of C.
__device__ inline u32x2_any load_q8(const int8_t* row, int c, int C) {
  u32x2_any q = 0;
  if (c + 8 <= C) {
    q = *reinterpret_cast<const u32x2_any*>(row + c);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < C) q[e >> 2] |= (uint32_t)(uint8_t)row[c + e] << (8 * (e & 3));
  }
  return q;
}
__device__ inline void store_q8(int8_t* row, int c, int C, u32x2_any q) {
  if (c + 8 <= C) {
    *reinterpret_cast<u32x2_any*>(row + c) = q;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < C) row[c + e] = (int8_t)(q[e >> 2] >> (8 * (e & 3)));
  }
}

// Forward: x packed (KEEP), y = gelu(x) (GELU).
template <typename T, bool KEEP, bool GELU>
__global__ __launch_bounds__(256) void act_pack_kernel(const ActPackParams p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.units) return;  // units is a multiple of four: a quad leaves together
  const uint32_t row = p.per_row.div(i), k = i - row * p.per_row.d;
  const int c = 8 * (int)k, C = p.C;
  float f[8];
  load_row8(reinterpret_cast<const T*>(p.x) + (int64_t)row * p.x_rs, c, C, f);
  if constexpr (KEEP) {
    u32x2_any q;
    const uint32_t byte = pack8(f, q);
    store_q8(p.q + (int64_t)row * C, c, C, q);
    if ((k & 3) == 0) p.exp[(int64_t)row * (p.per_row.d >> 2) + (k >> 2)] = (uint8_t)byte;
  }
  if constexpr (GELU) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float g;
      f[e] *= normal_cdf<kExact<T>>(f[e], g);
    }
    store_row8(reinterpret_cast<T*>(p.y) + (int64_t)row * C, c, C, f);
  }
}

// What is held is at most the block's largest magnitude: no type overflows.
template <typename T>
__global__ __launch_bounds__(256) void act_unpack_kernel(const ActPackParams p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.units) return;
  const uint32_t row = p.per_row.div(i), k = i - row * p.per_row.d;
  const int c = 8 * (int)k, C = p.C;
  float f[8];
  unpack8(load_q8(p.q + (int64_t)row * C, c, C), p.exp[(int64_t)row * (p.per_row.d >> 2) + (k >> 2)], f);
  store_row8(reinterpret_cast<T*>(p.y) + (int64_t)row * p.y_rs, c, C, f);
}

// Backward of the GELU: dx = dy gelu'(h); with y also gelu(h), which the
// weight gradient of the layer after the activation multiplies.
template <typename T>
__global__ __launch_bounds__(256) void gelu_pack_bwd_kernel(const ActPackParams p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.units) return;
  const uint32_t row = p.per_row.div(i), k = i - row * p.per_row.d;
  const int c = 8 * (int)k, C = p.C;
  float h[8], d[8];
  unpack8(load_q8(p.q + (int64_t)row * C, c, C), p.exp[(int64_t)row * (p.per_row.d >> 2) + (k >> 2)], h);
  load_row8(reinterpret_cast<const T*>(p.x) + (int64_t)row * p.x_rs, c, C, d);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float g;
    const float cdf = normal_cdf<kExact<T>>(h[e], g);
    d[e] *= fmaf(h[e] * g, 0.3989422804014327f, cdf);
    h[e] *= cdf;
  }
  store_row8(reinterpret_cast<T*>(p.dx) + (int64_t)row * C, c, C, d);
  if (p.y) store_row8(reinterpret_cast<T*>(p.y) + (int64_t)row * p.y_rs, c, C, h);
}

template <typename T>
hipError_t launch_t(const ActPackParams& p, ActPackOp op, hipStream_t s) {
  const dim3 grid((p.units + 255) / 256), wg(256);
  switch (op) {
    case ActPackOp::kPack: hipLaunchKernelGGL((act_pack_kernel<T, true, false>), grid, wg, 0, s, p); break;
    case ActPackOp::kUnpack: hipLaunchKernelGGL((act_unpack_kernel<T>), grid, wg, 0, s, p); break;
    case ActPackOp::kGelu: hipLaunchKernelGGL((act_pack_kernel<T, true, true>), grid, wg, 0, s, p); break;
    case ActPackOp::kGeluOnly: hipLaunchKernelGGL((act_pack_kernel<T, false, true>), grid, wg, 0, s, p); break;
    case ActPackOp::kGeluBwd: hipLaunchKernelGGL((gelu_pack_bwd_kernel<T>), grid, wg, 0, s, p); break;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_act_pack(const ActPackParams& p, int dtype, ActPackOp op, hipStream_t s) {
  if (dtype == kBF16) return launch_t<__bf16>(p, op, s);
  if (dtype == kF16) return launch_t<_Float16>(p, op, s);
  return launch_t<float>(p, op, s);
}

}  // namespace saf
