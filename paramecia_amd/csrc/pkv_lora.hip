// Low-rank adapters of many requests beside the gated output projection, gfx950
// (forward_with_scales_and_lora, paramecia-model/src/models/with_tracing.rs:253-300, around
// pkv_gated_oproj): for row m with adapter a = ids[m],
//   x = attn * sigmoid(gate), out[m] = W x + scale[a] * B_a (A_a x)
// and out[m] = W x where the row has none.
//
// The small product t = scale A x has a launch of its own (here), in front of the projection
// or between its two launches (the batched form, whose first one has gated the inputs); the
// projection's kernels add B t where they have a row's outputs in registers
// (pkv_lora.hpp): the per-token form in its dot product's sum, the batched form in its
// reduction over the splits or in its epilogue.
#include <algorithm>

#include "pkv_lora.hpp"

namespace pkv {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct ShrinkArgs {
  const float *attn, *gate;  // [rows][in]; gate may be null
  LoraSplit split;           // or the batched projection's operands of the same inputs
  const void *a;             // [adapters][rank][in]
  const float *scale;        // [adapters]
  const int *ids;            // [rows]
  float *t;                  // [S][rows][rank]
  unsigned *status;
  int rows, in_dim, rank, adapters, slice;  // slice: inputs per workgroup
};

__device__ __forceinline__ float fast_sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-g * 1.4426950408889634f));
}

// A workgroup takes 16 rows and a slice of the inputs, an eighth of it per wave, with
// v_mfma_f32_16x16x4_f32 (f32 products: 16 rows by 16 ranks, 4 inputs): lane (m, g) holds
// inputs 8 g .. 8 g + 7 of a 32-input step for row m of x and for rank m of A, and the eight
// MFMAs of a step take one of each. The rows' adapters are taken one after the other (in turn
// by gridDim.z workgroups), each for all 16 rows; a row keeps its own one's result. kC
// tiles of 16 ranks. kSplit: the inputs come, gated already, as the batched projection's
// fp16 pairs (hi + lo) 2^-e (half the bytes of x and gate, and written just before), and
// 16-bit weights take v_mfma_f32_16x16x32 as they are: F16 against hi and lo, BF16 against
// the three bf16 parts that hi + lo (22 bits) has. 4001 rows of 4096, three adapters of rank 64 in
// bf16: 41 us. Most of it is waiting for A from L2 (18 us are left without those loads):
// tiles of 32 or 64 rows, which halve them, more loads in flight and another order of the steps
// all took 41 to 49 us.
constexpr int kShrinkWaves = 8;
template <int kType, int kC, bool kSplit>
__global__ __launch_bounds__(64 * kShrinkWaves) void lora_shrink_kernel(ShrinkArgs a) {
  typedef float v4 __attribute__((ext_vector_type(4)));
  __shared__ v4 red[kShrinkWaves][kC][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m = lane & 15, g = lane >> 4;
  const int row0 = blockIdx.x * 16;
  const int row = row0 + m < a.rows ? row0 + m : a.rows - 1;
  int id = a.ids[row];
  if (id >= a.adapters) {
    if (blockIdx.y == 0 && blockIdx.z == 0 && tid < 16)
      __hip_atomic_fetch_or(a.status, kStatusAdapterId, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    id = -1;
  }
  if (row0 + m >= a.rows) id = -1;
  unsigned todo = (unsigned)(__ballot(id >= 0) & 0xFFFFu);
  const int k0 = blockIdx.y * a.slice + wave * (a.slice / kShrinkWaves) + 8 * g;
  const int steps = a.slice / (32 * kShrinkWaves);
  const int64_t x0 = (int64_t)row * a.in_dim + k0;
  const float4 *x4 = reinterpret_cast<const float4 *>(a.attn + x0);
  const float4 *g4 = a.gate == nullptr ? nullptr : reinterpret_cast<const float4 *>(a.gate + x0);
  const h8 *h4 = reinterpret_cast<const h8 *>(reinterpret_cast<const _Float16 *>(a.split.hi) + x0);
  const h8 *l4 = reinterpret_cast<const h8 *>(reinterpret_cast<const _Float16 *>(a.split.lo) + x0);
  for (int pass = 0; todo != 0; ++pass) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctz(todo));
    const unsigned mine = (unsigned)(__ballot(id == cur) & 0xFFFFu);
    todo &= ~mine;
    if (pass % gridDim.z != blockIdx.z) continue;
    v4 acc[kC];
    int64_t w0[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      acc[c] = v4{0.f, 0.f, 0.f, 0.f};
      const int r = 16 * c + m < a.rank ? 16 * c + m : a.rank - 1;
      w0[c] = ((int64_t)cur * a.rank + r) * a.in_dim + k0;
    }
    if constexpr (kSplit && kType != PKV_LORA_F32) {
      u4 wn[kC];
      h8 hn, ln;
      auto fetch = [&](int s) {
        hn = h4[4 * s];
        ln = l4[4 * s];
#pragma unroll
        for (int c = 0; c < kC; ++c)
          wn[c] = *reinterpret_cast<const u4 *>(reinterpret_cast<const uint16_t *>(a.a) + w0[c] + 32 * s);
      };
      fetch(0);
      for (int s = 0; s < steps; ++s) {
        const h8 hi = hn, lo = ln;
        u4 w[kC];
#pragma unroll
        for (int c = 0; c < kC; ++c) w[c] = wn[c];
        fetch(s + 1 < steps ? s + 1 : s);
        __builtin_amdgcn_sched_barrier(0);  // the loads stay in front of the products
        if constexpr (kType == PKV_LORA_F16) {
#pragma unroll
          for (int c = 0; c < kC; ++c)
            acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, __builtin_bit_cast(h8, w[c]), acc[c], 0, 0, 0);
#pragma unroll
          for (int c = 0; c < kC; ++c)
            acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, __builtin_bit_cast(h8, w[c]), acc[c], 0, 0, 0);
        } else {
          b8 part[3];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = (float)hi[i] + (float)lo[i];
            part[0][i] = (__bf16)x;
            const float y = x - (float)part[0][i];
            part[1][i] = (__bf16)y;
            part[2][i] = (__bf16)(y - (float)part[1][i]);
          }
#pragma unroll
          for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int c = 0; c < kC; ++c)
              acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(part[p], __builtin_bit_cast(b8, w[c]), acc[c], 0, 0, 0);
        }
      }
    } else {
      // the next step's inputs and weights are loaded while this one's products run
      float4 xn[2], gn[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      float wn[kC][8];
      h8 hn, ln;
      auto fetch = [&](int s) {
        if constexpr (kSplit) {
          hn = h4[4 * s];
          ln = l4[4 * s];
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            xn[h] = x4[8 * s + h];
            if (g4 != nullptr) gn[h] = g4[8 * s + h];
          }
        }
#pragma unroll
        for (int c = 0; c < kC; ++c) lora_weights<kType, 8>(a.a, w0[c] + 32 * s, wn[c]);
      };
      fetch(0);
      for (int s = 0; s < steps; ++s) {
        float x[8], w[kC][8];
        if constexpr (kSplit) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = (float)hn[i] + (float)ln[i];
        }
#pragma unroll
        for (int h = 0; h < (kSplit ? 0 : 2); ++h) {
          x[4 * h] = xn[h].x; x[4 * h + 1] = xn[h].y; x[4 * h + 2] = xn[h].z; x[4 * h + 3] = xn[h].w;
          if (g4 != nullptr) {
            x[4 * h] *= fast_sigmoid(gn[h].x);
            x[4 * h + 1] *= fast_sigmoid(gn[h].y);
            x[4 * h + 2] *= fast_sigmoid(gn[h].z);
            x[4 * h + 3] *= fast_sigmoid(gn[h].w);
          }
        }
#pragma unroll
        for (int c = 0; c < kC; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) w[c][i] = wn[c][i];
        fetch(s + 1 < steps ? s + 1 : s);
        __builtin_amdgcn_sched_barrier(0);  // the loads stay in front of the products
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int c = 0; c < kC; ++c)
            acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], w[c][i], acc[c], 0, 0, 0);
      }
    }
#pragma unroll
    for (int c = 0; c < kC; ++c) red[wave][c][lane] = acc[c];
    __syncthreads();
    const float scale = a.scale[cur];  // behind inv: their product may be too small to keep its bits
    for (int u = tid; u < 64 * kC; u += 64 * kShrinkWaves) {
      const int c = u >> 6, l = u & 63, r = 16 * c + (l & 15);
      v4 s = red[0][c][l];
#pragma unroll
      for (int w = 1; w < kShrinkWaves; ++w) s += red[w][c][l];
      if (r < a.rank) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = 4 * (l >> 4) + i;  // the row within the tile
          if ((mine >> n) & 1) {
            const float y = kSplit ? s[i] * a.split.inv[row0 + n] : s[i];
            a.t[((int64_t)blockIdx.y * a.rows + row0 + n) * a.rank + r] = y * scale;
          }
        }
      }
    }
    __syncthreads();  // the next adapter writes red again
  }
}

template <int kType, int kC>
void launch_shrink(const ShrinkArgs &a, const dim3 &grid, hipStream_t s) {
  const dim3 t(64 * kShrinkWaves);
  if (a.split.hi != nullptr) hipLaunchKernelGGL((lora_shrink_kernel<kType, kC, true>), grid, t, 0, s, a);
  else hipLaunchKernelGGL((lora_shrink_kernel<kType, kC, false>), grid, t, 0, s, a);
}
template <int kType>
void launch_shrink(const ShrinkArgs &a, const dim3 &grid, hipStream_t s) {
  if (a.rank <= 16) launch_shrink<kType, 1>(a, grid, s);
  else if (a.rank <= 32) launch_shrink<kType, 2>(a, grid, s);
  else if (a.rank <= 64) launch_shrink<kType, 4>(a, grid, s);
  else launch_shrink<kType, 8>(a, grid, s);
}

// The split of the inputs: workgroups for the 256 CUs twice over, at most one per 256 inputs
// (32 per wave): one row of 4096 inputs takes 16 (3.4 us), 4001 rows two.
int shrink_splits(int rows, int in_dim) {
  const int tiles = (rows + 15) / 16;
  int S = 1;
  while (S * 2 * tiles <= 512 && in_dim / (S * 2) >= 256) S *= 2;
  return S;
}
size_t t_bytes(int rows, int in_dim, int rank) {
  return ((size_t)shrink_splits(rows, in_dim) * rows * rank * 4 + 255) / 256 * 256;
}

}  // namespace

size_t oproj_lora_workspace(int w_type, int rows, int in_dim, int out_dim, int rank) {
  return t_bytes(rows, in_dim, rank) + oproj_workspace(w_type, rows, in_dim, out_dim);
}

int launch_oproj_lora(const float *attn, const float *gate, const uint8_t *w, int w_type,
                      const void *lora_a, const void *lora_b, int lora_type, int adapters,
                      int rank, const float *scale, const int *ids, float *out, int rows,
                      int in_dim, int out_dim, void *ws, size_t ws_bytes, hipStream_t s) {
  if (int rc = check_oproj(attn, gate, w, w_type, rows, in_dim, out_dim)) return rc;
  if (ws_bytes < oproj_lora_workspace(w_type, rows, in_dim, out_dim, rank))
    return set_error(PKV_ERR_ARG, "the workspace is smaller than pkv_gated_oproj_lora_workspace says");
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return set_error(PKV_ERR_ARG, "the workspace must be 256-byte aligned");
  const int S = shrink_splits(rows, in_dim);
  const size_t own = t_bytes(rows, in_dim, rank);
  const LoraTerm term{static_cast<const float *>(ws), lora_b, ids, lora_type, rank, adapters, S,
                      (int64_t)rows * rank, attn, gate, lora_a, scale, rows, in_dim};
  Workspace base;
  base.ptr = static_cast<uint8_t *>(ws) + own;
  base.bytes = ws_bytes - own;
  base.fixed = true;
  return oproj_any(attn, gate, w, w_type, out, rows, in_dim, out_dim, base, s, &term);
}

int launch_lora_shrink(const LoraTerm &l, const LoraSplit &split, hipStream_t s) {
  ShrinkArgs a{l.attn, l.gate, split, l.a, l.scale, l.ids, const_cast<float *>(l.t), nullptr,
               l.rows, l.in_dim, l.rank, l.adapters, l.in_dim / l.S};
  if (int rc = device_status_word(&a.status)) return rc;
  // a tile of 16 rows has as many adapters at most; few tiles take them side by side (24 rows
  // of 9 adapters: 5.1 us, one after the other 18.7)
  const int tiles = (a.rows + 15) / 16, most = std::min({a.rows, a.adapters, 16});
  const int Z = std::clamp(1024 / (tiles * l.S), 1, most);
  const dim3 grid((unsigned)tiles, (unsigned)l.S, (unsigned)Z);
  switch (l.type) {
    case PKV_LORA_F32: launch_shrink<PKV_LORA_F32>(a, grid, s); break;
    case PKV_LORA_F16: launch_shrink<PKV_LORA_F16>(a, grid, s); break;
    default: launch_shrink<PKV_LORA_BF16>(a, grid, s); break;
  }
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

}  // namespace pkv
