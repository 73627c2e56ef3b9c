// Root-mean-square norm of rows for gfx950, with the residual's addition in front, an output
// gate behind and an output in Q8_0 blocks: the RmsNorm between the blocks of a layer
// (paramecia-model/src/quantized_nn.rs) and the gated norm behind the Gated-DeltaNet state
// update (LinearAttention, qwen3_next.rs:2900-4208).
//
//   h = residual + x (written back), y = h / sqrt(mean(h^2) + eps) * alpha [* silu(gate)]
//   Q8_0: per 32 values d = max|y| / 127, code = round(y / d), halves away from zero
//
// HBM-bound: each value is read once and each result written once. A group of kLanes lanes
// holds a whole row, kQuads quads of four values per lane, quad
// kLanes c + lane, so every access is 16 bytes a lane and a Q8_0 block is eight
// neighbouring lanes. A row has the fewest lanes that hold it in two quads each (eight from 2048
// values on), so that its sum crosses few lanes and its loads are in flight together. The row is in
// registers up to 8192 values; past that 1024 lanes leave 128 registers each, and part of it, of
// alpha and of the gate passes through scratch memory (248 to 380 bytes a lane): 513 rows of 20001
// with a gate 116 us, 1.1 TB/s. 4001 rows of 4096 with a gate 51 us, 3.9 TB/s; 8001 rows of
// 2048 with the residual, f32 and Q8_0 out: 50 us for 280 MB, 5.6 TB/s (more than a copy, as the
// residual is partly in the last-level cache); 32672 rows of 128 with a gate 11.7 us, 4.3 TB/s; one
// row 2.8 us, a launch. The mean and, for Q8_0, the row up to its rounding to 32 bits are
// computed in 64 bits: a code then does not depend on the order of a sum.
#include "pkv_internal.hpp"
#include "pkv_scalar.hpp"

namespace pkv {
namespace {

struct NormArgs {
  const float *x;
  float *residual;          // [rows][dim], updated; may be null
  const float *alpha;       // [dim]
  const float *gate;        // [rows][dim]; may be null
  float *out;               // [rows][dim]; may be null
  uint8_t *q8;              // [rows][blocks][34]; may be null
  int64_t rows, x_stride;
  int dim;
  double eps;
};

__device__ __forceinline__ double shfl_xor_d(double v, int m, int w) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __shfl_xor((int)(uint32_t)u, m, w), hi = __shfl_xor((int)(uint32_t)(u >> 32), m, w);
  return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}

template <bool kWide>
__device__ __forceinline__ void load4(const float *p, int e, int dim, float (&v)[4]) {
  if constexpr (kWide) {
    float4 f = {0.f, 0.f, 0.f, 0.f};
    if (e < dim) f = *reinterpret_cast<const float4 *>(p + e);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = e + i < dim ? p[e + i] : 0.0f;
  }
}
template <bool kWide>
__device__ __forceinline__ void store4(float *p, int e, int dim, const float (&v)[4]) {
  if constexpr (kWide) {
    if (e < dim) *reinterpret_cast<float4 *>(p + e) = float4{v[0], v[1], v[2], v[3]};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e + i < dim) p[e + i] = v[i];
  }
}

// kLanes lanes per row (16, 64, 256 or 1024), kQuads quads per lane.
template <int kLanes, int kQuads, bool kWide, bool kQ8>
__global__ __launch_bounds__(kLanes < 256 ? 256 : kLanes) void rms_norm_kernel(NormArgs a) {
  constexpr int kThreads = kLanes < 256 ? 256 : kLanes;
  constexpr int kRows = kThreads / kLanes;
  constexpr int kW = kLanes < 64 ? kLanes : 64;
  const int lane = threadIdx.x % kLanes;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kLanes;
  const bool live = row < a.rows;
  const int64_t at = (live ? row : 0) * a.dim;
  const int dim = live ? a.dim : 0;
  float h[kQuads][4], g[kQuads][4], al[kQuads][4];
  const float *x = a.x + (live ? row : 0) * a.x_stride;
#pragma unroll
  for (int c = 0; c < kQuads; ++c) load4<kWide>(x, 4 * (kLanes * c + lane), dim, h[c]);
  if (a.residual != nullptr) {
    float r[kQuads][4];
#pragma unroll
    for (int c = 0; c < kQuads; ++c) load4<kWide>(a.residual + at, 4 * (kLanes * c + lane), dim, r[c]);
#pragma unroll
    for (int c = 0; c < kQuads; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) h[c][i] += r[c][i];
  }
#pragma unroll
  for (int c = 0; c < kQuads; ++c) load4<kWide>(a.alpha, 4 * (kLanes * c + lane), dim, al[c]);
  if (a.gate != nullptr) {
#pragma unroll
    for (int c = 0; c < kQuads; ++c) load4<kWide>(a.gate + at, 4 * (kLanes * c + lane), dim, g[c]);
  }
  if (a.residual != nullptr) {
#pragma unroll
    for (int c = 0; c < kQuads; ++c) store4<kWide>(a.residual + at, 4 * (kLanes * c + lane), dim, h[c]);
  }
  double sum = 0.0;
#pragma unroll
  for (int c = 0; c < kQuads; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fma((double)h[c][i], (double)h[c][i], sum);
#pragma unroll
  for (int o = kW / 2; o > 0; o >>= 1) sum += shfl_xor_d(sum, o, kW);
  if constexpr (kLanes > 64) {
    __shared__ double part[kThreads / 64];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) sum += part[w];
  }
  const double inv = 1.0 / sqrt(sum / a.dim + a.eps);
  const int blocks = (a.dim + 31) / 32;
#pragma unroll
  for (int c = 0; c < kQuads; ++c) {
    const int e = 4 * (kLanes * c + lane);
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      double v = (double)h[c][i] * inv * (double)al[c][i];
      // In 64 bits for 8-bit rows, whose codes would otherwise follow the activation's rounding; f32
      // rows alone take 32 bits, off by 8 half steps at most (64 bits: 14.9 us for 11.4, 32672 rows of 128).
      if (a.gate != nullptr) {
        if constexpr (kQ8) {
          const double z = (double)g[c][i];
          v *= z / (1.0 + exp(-z));
        } else {
          v *= (double)(g[c][i] / (1.0f + expf(-g[c][i])));
        }
      }
      y[i] = (float)v;
    }
    if (a.out != nullptr) store4<kWide>(a.out + at, e, dim, y);
    if constexpr (kQ8) {
      // as the cache's Q8_0 quantizer: NaN is left out of the block's largest |y|
      int32_t key = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float z = e + i < dim ? y[i] : 0.0f;
        const int32_t k = z != z ? 0 : (int32_t)(f2u(z) & 0x7FFFFFFFu);
        key = k > key ? k : key;
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const int32_t k = __shfl_xor(key, o, 8);
        key = k > key ? k : key;
      }
      const float d = u2f((uint32_t)key) / 127.0f;
      const float id = d != 0.0f ? 1.0f / d : 0.0f;
      uint32_t w = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float z = e + i < dim ? y[i] : 0.0f;
        w |= (uint32_t)(uint8_t)rs_as_i8(__builtin_roundf(z * id)) << (8 * i);
      }
      if (live && (e >> 5) < blocks) {
        uint8_t *blk = a.q8 + (row * blocks + (e >> 5)) * 34;
        uint16_t *o = reinterpret_cast<uint16_t *>(blk + 2 + (e & 31));
        o[0] = (uint16_t)w;
        o[1] = (uint16_t)(w >> 16);
        if ((e & 31) == 0) *reinterpret_cast<uint16_t *>(blk) = f32_to_f16(d);
      }
    }
  }
}

template <int kLanes, int kQuads>
int launch(const NormArgs &a, bool wide, hipStream_t s) {
  constexpr int kThreads = kLanes < 256 ? 256 : kLanes, kRows = kThreads / kLanes;
  if (a.rows > INT32_MAX / kLanes)  // a launch holds fewer than 2^32 lanes; half of that is kept to
    return set_error(PKV_ERR_UNSUPPORTED, "rms norm: too many rows of this length for one call");
  const dim3 grid((unsigned)((a.rows + kRows - 1) / kRows)), t(kThreads);
  if (a.q8 != nullptr) {
    if (wide) hipLaunchKernelGGL((rms_norm_kernel<kLanes, kQuads, true, true>), grid, t, 0, s, a);
    else hipLaunchKernelGGL((rms_norm_kernel<kLanes, kQuads, false, true>), grid, t, 0, s, a);
  } else {
    if (wide) hipLaunchKernelGGL((rms_norm_kernel<kLanes, kQuads, true, false>), grid, t, 0, s, a);
    else hipLaunchKernelGGL((rms_norm_kernel<kLanes, kQuads, false, false>), grid, t, 0, s, a);
  }
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

}  // namespace

int launch_rms_norm(const float *x, int64_t x_stride, float *residual, const float *alpha,
                    const float *gate, float eps, float *out, uint8_t *q8, int64_t rows, int dim,
                    hipStream_t s) {
  const auto at16 = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool wide = dim % 4 == 0 && x_stride % 4 == 0 && at16(x) && at16(residual) && at16(alpha) &&
                    at16(gate) && at16(out);
  NormArgs a{x, residual, alpha, gate, out, q8, rows, x_stride, dim, (double)eps};
  if (dim <= 128) return launch<16, 2>(a, wide, s);
  if (dim <= 512) return launch<64, 2>(a, wide, s);
  if (dim <= 2048) return launch<256, 2>(a, wide, s);
  if (dim <= 8192) return launch<256, 8>(a, wide, s);
  if (dim <= 32768) return launch<1024, 8>(a, wide, s);
  return set_error(PKV_ERR_UNSUPPORTED, "rms norm: rows of at most 32768 values");
}

}  // namespace pkv
