// Low-rank adapters of many requests beside the gated output projection, gfx950
// (forward_with_scales_and_lora, paramecia-model/src/models/with_tracing.rs:253-300, around
// pkv_gated_oproj): for row m with adapter a = ids[m],
//   x = attn * sigmoid(gate), out[m] = W x + scale[a] * B_a (A_a x)
// and out[m] = W x where the row has none. The small product t = scale A x comes first (t in
// the workspace), then the projection, then its sum with B t.
#include "pkv_internal.hpp"
#include "pkv_scalar.hpp"

namespace pkv {
namespace {

struct LoraArgs {
  const float *attn, *gate;  // [rows][in]; gate may be null
  const void *a, *b;         // [adapters][rank][in], [adapters][out][rank]
  const float *scale;        // [adapters]
  const int *ids;            // [rows]
  float *t;                  // [rows][rank]
  float *out;                // [rows][out]
  unsigned *status;
  int rows, in_dim, out_dim, rank, adapters;
};

enum : int { kF32 = 0, kF16 = 1, kBF16 = 2 };
template <int kType>
__device__ __forceinline__ float weight(const void *p, int64_t i) {
  if constexpr (kType == kF32) return reinterpret_cast<const float *>(p)[i];
  else if constexpr (kType == kF16) return f16_to_f32(reinterpret_cast<const uint16_t *>(p)[i]);
  else return bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[i]);
}

// the row's adapter, -1 for none; an id past the adapters flags the device status word
__device__ __forceinline__ int adapter_of(const LoraArgs &a, int row) {
  const int id = a.ids[row];
  if (id >= a.adapters) {
    if (threadIdx.x == 0)
      __hip_atomic_fetch_or(a.status, kStatusAdapterId, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return -1;
  }
  return id < 0 ? -1 : id;
}

// t[row][r]: a wave per rank of a row, lanes along the inputs.
template <int kType>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs a) {
  const int row = blockIdx.x, id = adapter_of(a, row);
  if (id < 0) return;
  const int lane = threadIdx.x & 63, r = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (r >= a.rank) return;
  const int64_t w0 = ((int64_t)id * a.rank + r) * a.in_dim, x0 = (int64_t)row * a.in_dim;
  float s = 0.0f;
  for (int i = lane; i < a.in_dim; i += 64) {
    float x = a.attn[x0 + i];
    if (a.gate != nullptr) x = x / (1.0f + expf(-a.gate[x0 + i]));
    s = fmaf(weight<kType>(a.a, w0 + i), x, s);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) a.t[(int64_t)row * a.rank + r] = s * a.scale[id];
}

// out[row][o] += B[o] . t[row]: a lane per output.
template <int kType>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a) {
  const int row = blockIdx.x, id = adapter_of(a, row);
  if (id < 0) return;
  const int o = blockIdx.y * 256 + threadIdx.x;
  if (o >= a.out_dim) return;
  const int64_t w0 = ((int64_t)id * a.out_dim + o) * a.rank;
  const float *t = a.t + (int64_t)row * a.rank;
  float s = 0.0f;
  for (int r = 0; r < a.rank; ++r) s = fmaf(weight<kType>(a.b, w0 + r), t[r], s);
  a.out[(int64_t)row * a.out_dim + o] += s;
}

template <int kType>
int launch_shrink(const LoraArgs &a, hipStream_t s) {
  const dim3 grid((unsigned)a.rows, (unsigned)((a.rank + 3) / 4));
  hipLaunchKernelGGL(lora_shrink_kernel<kType>, grid, dim3(256), 0, s, a);
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}
template <int kType>
int launch_expand(const LoraArgs &a, hipStream_t s) {
  const dim3 grid((unsigned)a.rows, (unsigned)((a.out_dim + 255) / 256));
  hipLaunchKernelGGL(lora_expand_kernel<kType>, grid, dim3(256), 0, s, a);
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

size_t t_bytes(int rows, int rank) { return ((size_t)rows * rank * 4 + 255) / 256 * 256; }

}  // namespace

size_t oproj_lora_workspace(int w_type, int rows, int in_dim, int out_dim, int rank) {
  return t_bytes(rows, rank) + oproj_workspace(w_type, rows, in_dim, out_dim);
}

int launch_oproj_lora(const float *attn, const float *gate, const uint8_t *w, int w_type,
                      const void *lora_a, const void *lora_b, int lora_type, int adapters,
                      int rank, const float *scale, const int *ids, float *out, int rows,
                      int in_dim, int out_dim, void *ws, size_t ws_bytes, hipStream_t s) {
  if (ws_bytes < oproj_lora_workspace(w_type, rows, in_dim, out_dim, rank))
    return set_error(PKV_ERR_ARG, "the workspace is smaller than pkv_gated_oproj_lora_workspace says");
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return set_error(PKV_ERR_ARG, "the workspace must be 256-byte aligned");
  LoraArgs a{attn, gate, lora_a, lora_b, scale, ids, static_cast<float *>(ws), out, nullptr,
             rows, in_dim, out_dim, rank, adapters};
  if (int rc = device_status_word(&a.status)) return rc;
  Workspace base;
  base.ptr = static_cast<uint8_t *>(ws) + t_bytes(rows, rank);
  base.bytes = ws_bytes - t_bytes(rows, rank);
  base.fixed = true;
  // the projection checks its own shapes and alignment before anything is enqueued
  if (int rc = oproj_any(attn, gate, w, w_type, out, rows, in_dim, out_dim, base, s)) return rc;
  int rc = lora_type == PKV_LORA_F32   ? launch_shrink<kF32>(a, s)
           : lora_type == PKV_LORA_F16 ? launch_shrink<kF16>(a, s)
                                       : launch_shrink<kBF16>(a, s);
  if (rc) return rc;
  return lora_type == PKV_LORA_F32   ? launch_expand<kF32>(a, s)
         : lora_type == PKV_LORA_F16 ? launch_expand<kF16>(a, s)
                                     : launch_expand<kBF16>(a, s);
}

}  // namespace pkv
