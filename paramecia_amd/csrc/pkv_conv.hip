// Short causal convolution of a Gated-DeltaNet layer for gfx950, prompts and single tokens:
// the depthwise_conv1d role of paramecia-model/src/ops.rs:18-20 with the conv state of
// RecurrentState (qwen3_next.rs:683-700, 3455-3460) and the layer's SiLU.
//
// Per sequence b and channel c, with X = the K-1 kept inputs followed by the new ones:
//   y[t][c] = act(bias[c] + sum_j w[c][j] X[t + j][c]),  act(y) = y / (1 + exp(-y)) or y,
// and the kept inputs become the last K-1 of X up to the sequence's end.
//
// HBM-bound: 2 K flops for 8 bytes. A lane owns four neighbouring channels (16-byte
// accesses, a wave reads 1 KB of a token's row) and kTile tokens of them, whose inputs it
// holds in registers: K-1 inputs of the tile in front are read again, from L2 (3 of 16).
// 8001 tokens of 8192 channels, 4 taps: 104 us for 525 MB, 5.0 TB/s, as a large copy. Calls of up
// to 4 tokens take tiles of 4, whose registers hold whatever the kept inputs become (a tile of
// 16 reads them once more from memory, behind its weights): 16 sequences of one token 4.3 us.
#include "pkv_internal.hpp"

namespace pkv {
namespace {

struct ConvArgs {
  const float *x, *w, *bias;  // [b][n][c] by strides, [c][K], [c] or null
  float *state;               // [b][c][K - 1]
  const int *lens;            // [b] or null
  float *out;                 // [b][n][c]
  int64_t sb, st, n;
  int channels, silu;
};

__device__ __forceinline__ float activate(float y, int silu) {
  return silu ? y / (1.0f + expf(-y)) : y;
}

// kV channels per lane (4, or 1 where strides or alignment forbid 16-byte accesses). The
// lanes of the first tile also write the new state: no other tile reads the old one, as
// tiles hold at least K - 1 tokens.
template <int K, int kV, int kTile>
__global__ __launch_bounds__(256) void conv_kernel(ConvArgs a) {
  static_assert(kTile >= K - 1, "only the first tile may reach the state");
  const int c0 = (blockIdx.x * 256 + threadIdx.x) * kV;
  if (c0 >= a.channels) return;
  const int64_t b = blockIdx.z, t0 = (int64_t)blockIdx.y * kTile;
  int64_t end = a.n;
  if (a.lens != nullptr) {
    const int64_t l = a.lens[b];
    end = l < 0 ? 0 : (l < a.n ? l : a.n);
  }
  if (t0 >= end) return;  // an empty sequence keeps its state
  const float *x = a.x + b * a.sb + c0;
  auto load = [&](int64_t t, float (&v)[kV]) {
    if constexpr (kV == 4) {
      const float4 f = *reinterpret_cast<const float4 *>(x + t * a.st);
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      v[0] = x[t * a.st];
    }
  };
  float xv[kTile + K - 1][kV];  // inputs t0 - (K - 1) .. t0 + kTile - 1
  float *state = a.state + (b * a.channels + c0) * (K - 1);
  if (t0 == 0) {
#pragma unroll
    for (int i = 0; i < kV; ++i)
#pragma unroll
      for (int j = 0; j < K - 1; ++j) xv[j][i] = state[i * (K - 1) + j];
  } else {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) load(t0 - (K - 1) + j, xv[j]);
  }
#pragma unroll
  for (int t = 0; t < kTile; ++t) {
    if (t0 + t < end) {
      load(t0 + t, xv[K - 1 + t]);
    } else {
#pragma unroll
      for (int i = 0; i < kV; ++i) xv[K - 1 + t][i] = 0.0f;
    }
  }
  float w[kV][K], bias[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) w[i][j] = a.w[(int64_t)(c0 + i) * K + j];
    bias[i] = a.bias != nullptr ? a.bias[c0 + i] : 0.0f;
  }
  if (t0 == 0) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      const int64_t at = end + j;  // of kept inputs followed by new ones
      float v[kV];
      if (kTile > 4 && at >= K - 1) {
        load(at - (K - 1), v);
      } else {  // a prompt that the tile's registers hold, or one shorter than the kept inputs
        constexpr int kHeld = kTile > 4 ? K - 1 : K - 1 + kTile;
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          v[i] = 0.0f;
#pragma unroll
          for (int s = 0; s < kHeld; ++s) v[i] = at == s ? xv[s][i] : v[i];
        }
      }
#pragma unroll
      for (int i = 0; i < kV; ++i) state[i * (K - 1) + j] = v[i];
    }
  }
  float *out = a.out + b * a.n * a.channels + c0;
#pragma unroll
  for (int t = 0; t < kTile; ++t) {
    if (t0 + t >= end) break;
    float y[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      float s = bias[i];
#pragma unroll
      for (int j = 0; j < K; ++j) s = fmaf(w[i][j], xv[t + j][i], s);
      y[i] = activate(s, a.silu);
    }
    float *o = out + (t0 + t) * a.channels;
    if constexpr (kV == 4)
      *reinterpret_cast<float4 *>(o) = float4{y[0], y[1], y[2], y[3]};
    else
      o[0] = y[0];
  }
}

template <int K>
int launch(const ConvArgs &a, int batch, bool wide, hipStream_t s) {
  const int per_wg = wide ? 1024 : 256;
  const unsigned gx = (unsigned)((a.channels + per_wg - 1) / per_wg);
  constexpr int kTile = 16;
  const int64_t tiles = (a.n + kTile - 1) / kTile;
  if (a.n <= 4) {
    const dim3 grid(gx, 1, (unsigned)batch);
    if (wide) hipLaunchKernelGGL((conv_kernel<K, 4, 4>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((conv_kernel<K, 1, 4>), grid, dim3(256), 0, s, a);
  } else {
    if (tiles > 65535) return set_error(PKV_ERR_ARG, "causal conv: n must be <= 1048560");
    const dim3 grid(gx, (unsigned)tiles, (unsigned)batch);
    if (wide) hipLaunchKernelGGL((conv_kernel<K, 4, kTile>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((conv_kernel<K, 1, kTile>), grid, dim3(256), 0, s, a);
  }
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

}  // namespace

int launch_causal_conv(const float *x, int64_t stride_b, int64_t stride_t, const float *w,
                       const float *bias, float *state, const int *lens, float *out, int batch,
                       int64_t n, int channels, int taps, int silu, hipStream_t s) {
  if (batch > 65535) return set_error(PKV_ERR_ARG, "batch must be <= 65535");
  if (channels > 1 << 24) return set_error(PKV_ERR_ARG, "causal conv: at most 2^24 channels");
  const auto at16 = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool wide = channels % 4 == 0 && stride_b % 4 == 0 && stride_t % 4 == 0 && at16(x) && at16(out);
  ConvArgs a{x, w, bias, state, lens, out, stride_b, stride_t, n, channels, silu};
  switch (taps) {
    case 2: return launch<2>(a, batch, wide, s);
    case 3: return launch<3>(a, batch, wide, s);
    case 4: return launch<4>(a, batch, wide, s);
    default: return set_error(PKV_ERR_UNSUPPORTED, "causal conv: 2, 3 or 4 taps");
  }
}

}  // namespace pkv
