// The low-rank term that the output projection's kernels add to a row's outputs
// (pkv_lora.hip): B_a t with t = scale_a A_a x of the row's adapter a, in parts over the inputs.
// Include-only; every symbol has internal linkage.
#pragma once
#include "pkv_internal.hpp"
#include "pkv_scalar.hpp"

namespace pkv {
namespace {

// the row's adapter, -1 for none (an id past the adapters is none)
__device__ __forceinline__ int lora_adapter(const LoraTerm &l, int row) {
  const int id = l.ids[row];
  return id >= 0 && id < l.adapters ? id : -1;
}

__device__ __forceinline__ float lora_weight(const void *p, int type, int64_t i) {
  if (type == PKV_LORA_F32) return reinterpret_cast<const float *>(p)[i];
  const uint16_t h = reinterpret_cast<const uint16_t *>(p)[i];
  return type == PKV_LORA_BF16 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
}

// N weights i .. i + N - 1 (N 4 or 8, i a multiple of 4): 16-byte or 8-byte loads
template <int kType, int N>
__device__ __forceinline__ void lora_weights(const void *p, int64_t i, float (&w)[N]) {
  if constexpr (kType == PKV_LORA_F32) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const float4 f = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + i + 4 * j);
      w[4 * j] = f.x; w[4 * j + 1] = f.y; w[4 * j + 2] = f.z; w[4 * j + 3] = f.w;
    }
  } else {
    uint32_t u[N / 2];
    const uint16_t *h = reinterpret_cast<const uint16_t *>(p) + i;
    if constexpr (N == 8) {
      const uint4 f = *reinterpret_cast<const uint4 *>(h);
      u[0] = f.x; u[1] = f.y; u[2] = f.z; u[3] = f.w;
    } else {
      const uint2 f = *reinterpret_cast<const uint2 *>(h);
      u[0] = f.x; u[1] = f.y;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint16_t b = (uint16_t)(u[j >> 1] >> (16 * (j & 1)));
      w[j] = kType == PKV_LORA_BF16 ? bf16_to_f32(b) : (float)__builtin_bit_cast(_Float16, b);
    }
  }
}

// t[row][r]: its parts, four loads at a time
__device__ __forceinline__ float lora_t(const LoraTerm &l, int row, int r) {
  const float *p = l.t + (int64_t)row * l.rank + r;
  float t = p[0];
  int s = 1;
  for (; s + 4 <= l.S; s += 4) {
    const float a = p[s * l.plane], b = p[(s + 1) * l.plane];
    const float c = p[(s + 2) * l.plane], d = p[(s + 3) * l.plane];
    t += (a + b) + (c + d);
  }
  for (; s < l.S; ++s) t += p[s * l.plane];
  return t;
}

// One lane's share of (B t)[o] of a row: the caller sums over the wave. Up to 64 ranks, the
// lanes left over take some of the parts of t (with 16 parts of 16 ranks, four each).
__device__ __forceinline__ float lora_lane(const LoraTerm &l, int row, int o, int out_dim, int lane) {
  const int id = lora_adapter(l, row);
  if (id < 0) return 0.0f;
  const int64_t w0 = ((int64_t)id * out_dim + o) * l.rank;
  if (l.rank > 64) {
    float s = 0.0f;
    for (int r = lane; r < l.rank; r += 64)
      s = fmaf(lora_weight(l.b, l.type, w0 + r), lora_t(l, row, r), s);
    return s;
  }
  const int per = 64 / l.rank, s0 = lane / l.rank, r = lane - s0 * l.rank;
  if (s0 >= per || s0 >= l.S) return 0.0f;
  const float w = lora_weight(l.b, l.type, w0 + r);
  const float *p = l.t + (int64_t)row * l.rank + r;
  float t = 0.0f;
  int s = s0;
  for (; s + 3 * per < l.S; s += 4 * per) {
    const float a = p[s * l.plane], b = p[(s + per) * l.plane];
    const float c = p[(s + 2 * per) * l.plane], d = p[(s + 3 * per) * l.plane];
    t += (a + b) + (c + d);
  }
  for (; s < l.S; s += per) t += p[s * l.plane];
  return w * t;
}

// delta[tt][rt][i] = (B t) of tokens tok0 + 16 tt + 4 g + i and outputs col0 + 16 rt + lane % 16
// (g = lane / 16): v_mfma_f32_16x16x4_f32 with t as A and B's rows as B, four ranks a lane
// at a time, the loads of 32 ranks in flight together. The tokens' adapters are taken one
// after the other; a token keeps its own one's result by selection, so that nothing of
// another adapter (a NaN, say) reaches it. 4001 tokens of 2048 outputs, rank 64 in bf16: the
// projection's kernel takes 251 us with it and 222 without: f32 products (7 us of matrix time an
// adapter) behind two latencies that nothing is left to hide.
template <int kType, bool kVec, int kTT, int kRT>
__device__ void lora_tile_as(const LoraTerm &l, int tokens, int out_dim, int tok0, int col0,
                             int lane, float (&delta)[kTT][kRT][4]) {
  typedef float v4 __attribute__((ext_vector_type(4)));
  const int m = lane & 15, g = lane >> 4;
  int row[kTT], id[kTT];
  unsigned todo[kTT], any = 0;
#pragma unroll
  for (int tt = 0; tt < kTT; ++tt) {
    const int t = tok0 + 16 * tt + m;
    row[tt] = t < tokens ? t : tokens - 1;
    id[tt] = t < tokens ? lora_adapter(l, row[tt]) : -1;
    todo[tt] = (unsigned)(__ballot(id[tt] >= 0) & 0xFFFFu);
    any |= todo[tt];
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
      for (int i = 0; i < 4; ++i) delta[tt][rt][i] = 0.0f;
  }
  while (any != 0) {
    // the first adapter that a token still waits for
    int cur = -1;
#pragma unroll
    for (int tt = kTT - 1; tt >= 0; --tt)
      if (todo[tt] != 0) cur = __builtin_amdgcn_readlane(id[tt], __builtin_ctz(todo[tt]));
    unsigned mine[kTT];
    any = 0;
    v4 d[kTT][kRT];
#pragma unroll
    for (int tt = 0; tt < kTT; ++tt) {
      mine[tt] = (unsigned)(__ballot(id[tt] == cur) & 0xFFFFu);
      todo[tt] &= ~mine[tt];
      any |= todo[tt];
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt) d[tt][rt] = v4{0.f, 0.f, 0.f, 0.f};
    }
    for (int r0 = 0; r0 < l.rank; r0 += 32) {
      float a[2][kTT][4], w[2][kRT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = r0 + 16 * h + 4 * g;
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt) {
          const int col = col0 + 16 * rt + m;
          const int64_t at = ((int64_t)cur * out_dim + (col < out_dim ? col : out_dim - 1)) * l.rank;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[h][rt][i] = 0.0f;
          if constexpr (kVec) {
            if (r < l.rank) lora_weights<kType, 4>(l.b, at + r, w[h][rt]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (r + i < l.rank) w[h][rt][i] = lora_weight(l.b, kType, at + r + i);
          }
        }
#pragma unroll
        for (int tt = 0; tt < kTT; ++tt) {
          if constexpr (kVec) {
            const float *p = l.t + (int64_t)row[tt] * l.rank + (r < l.rank ? r : 0);
            float4 t = *reinterpret_cast<const float4 *>(p);
            for (int s = 1; s < l.S; ++s) {
              const float4 f = *reinterpret_cast<const float4 *>(p + s * l.plane);
              t.x += f.x; t.y += f.y; t.z += f.z; t.w += f.w;
            }
            const bool on = id[tt] == cur && r < l.rank;
            a[h][tt][0] = on ? t.x : 0.0f;
            a[h][tt][1] = on ? t.y : 0.0f;
            a[h][tt][2] = on ? t.z : 0.0f;
            a[h][tt][3] = on ? t.w : 0.0f;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float t = lora_t(l, row[tt], r + i < l.rank ? r + i : 0);
              a[h][tt][i] = id[tt] == cur && r + i < l.rank ? t : 0.0f;
            }
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
            for (int tt = 0; tt < kTT; ++tt)
              d[tt][rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[h][tt][i], w[h][rt][i], d[tt][rt], 0, 0, 0);
    }
#pragma unroll
    for (int tt = 0; tt < kTT; ++tt)
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          delta[tt][rt][i] = (mine[tt] >> (4 * g + i)) & 1 ? d[tt][rt][i] : delta[tt][rt][i];
  }
}
template <int kTT, int kRT>
__device__ __forceinline__ void lora_tile(const LoraTerm &l, int tokens, int out_dim, int tok0,
                                          int col0, int lane, float (&delta)[kTT][kRT][4]) {
  const bool vec = (l.rank & 3) == 0;
  if (l.type == PKV_LORA_F32) {
    if (vec) lora_tile_as<PKV_LORA_F32, true>(l, tokens, out_dim, tok0, col0, lane, delta);
    else lora_tile_as<PKV_LORA_F32, false>(l, tokens, out_dim, tok0, col0, lane, delta);
  } else if (l.type == PKV_LORA_F16) {
    if (vec) lora_tile_as<PKV_LORA_F16, true>(l, tokens, out_dim, tok0, col0, lane, delta);
    else lora_tile_as<PKV_LORA_F16, false>(l, tokens, out_dim, tok0, col0, lane, delta);
  } else {
    if (vec) lora_tile_as<PKV_LORA_BF16, true>(l, tokens, out_dim, tok0, col0, lane, delta);
    else lora_tile_as<PKV_LORA_BF16, false>(l, tokens, out_dim, tok0, col0, lane, delta);
  }
}

}  // namespace
}  // namespace pkv
