// Gated delta rule over the tokens of a prompt for gfx950: the prompt form of the
// Gated-DeltaNet state update (delta_net_chunked, paramecia-model/src/qwen3_next.rs:
// 3506-3731; one token: pkv_deltanet.hip).
//
// Per sequence b and value head h, with its key head h / (heads / k_heads) and the state
// S[i][j] (i: value channel, j: key channel), for t = 0 .. end - 1:
//   qn = q_t * scale / sqrt(|q_t|^2 + eps), kn = k_t / sqrt(|k_t|^2 + eps)
//   S *= exp(gate_t); u_i = (v_ti - S_i . kn) * sigmoid(beta_t); S_i += u_i kn; o_ti = S_i . qn
#include <type_traits>

#include "pkv_internal.hpp"

namespace pkv {
namespace {

struct ScanArgs {
  const float *q, *k, *v, *gate, *beta;
  int64_t qb, qt, kb, kt, vb, vt;  // batch and token strides in elements
  float *state, *gate_offset, *out;
  const int *lens;
  int64_t n;
  int heads, rep;  // rep: value heads per key head
  float scale, eps;
};

// Sum over the 16 lanes of a row (every lane receives it): DPP within rows of 16.
__device__ __forceinline__ float row16_sum(float x) {
  auto dpp = [](float v, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, v),
                                                                __builtin_bit_cast(int, v),
                                                                decltype(ctrl)::value, 0xF, 0xF,
                                                                false));
  };
  x += dpp(x, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  x += dpp(x, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  x += dpp(x, std::integral_constant<int, 0x141>{});  // row_half_mirror
  x += dpp(x, std::integral_constant<int, 0x140>{});  // row_mirror
  return x;
}

__device__ __forceinline__ int64_t valid_tokens(const int *lens, int64_t b, int64_t n) {
  if (lens == nullptr) return n;
  const int64_t l = lens[b];
  return l < 0 ? 0 : (l < n ? l : n);
}

// Token by token. A workgroup owns 16 rows S_i of one head, 16 lanes each (lane l holds the
// quads 4 l + 64 c of its row), and goes through the tokens kT at a time: its lanes
// normalise the next kT tokens' q and k into LDS while they are 16 lanes per token, then
// every row reads them back. Both products of a token are taken with the state in front of
// it (S_new . qn = exp(gate) S . qn + u (kn . qn)), so that their reductions run beside each
// other.
template <int kD, int kT>
__global__ __launch_bounds__(256) void scan_tokens_kernel(ScanArgs a) {
  constexpr int kQ = kD / 64;  // quads per lane
  __shared__ __attribute__((aligned(16))) float qs[2][kT][kD], ks[2][kT][kD];
  __shared__ float vs[2][kT][16];
  __shared__ float4 cs[2][kT];  // exp(gate), sigmoid(beta), kn . qn, gate
  const int tid = threadIdx.x, lane = tid & 15, r = tid >> 4;
  const int64_t b = blockIdx.z, h = blockIdx.y, hk = h / a.rep;
  const int64_t end = valid_tokens(a.lens, b, a.n);
  if (end == 0) return;
  const int row0 = blockIdx.x * 16;
  const float *q = a.q + b * a.qb + hk * kD + 4 * lane, *k = a.k + b * a.kb + hk * kD + 4 * lane;
  const float *v = a.v + b * a.vb + h * kD + row0;
  const float *gate = a.gate + b * a.n * a.heads + h, *beta = a.beta + b * a.n * a.heads + h;
  float *out = a.out + (b * a.n * a.heads + h) * kD + row0;
  float *state = a.state + ((b * a.heads + h) * kD + row0 + r) * kD + 4 * lane;

  float4 qv[kQ], kv[kQ];
  float vv = 0.0f, gv = 0.0f, bv = 0.0f;
  const bool stages = r < kT;  // kT tokens of 16 lanes
  auto fetch = [&](int64_t t0) {
    const int64_t t = t0 + r;
    const bool on = stages && t < end;
#pragma unroll
    for (int c = 0; c < kQ; ++c) {
      qv[c] = on ? *reinterpret_cast<const float4 *>(q + t * a.qt + 64 * c) : float4{0.f, 0.f, 0.f, 0.f};
      kv[c] = on ? *reinterpret_cast<const float4 *>(k + t * a.kt + 64 * c) : float4{0.f, 0.f, 0.f, 0.f};
    }
    vv = on ? v[t * a.vt + lane] : 0.0f;
    gv = on ? gate[t * a.heads] : 0.0f;
    bv = on ? beta[t * a.heads] : 0.0f;
  };
  auto stage = [&](int64_t t0, int buf) {
    float sq = 0.0f, sk = 0.0f, qk = 0.0f;
#pragma unroll
    for (int c = 0; c < kQ; ++c) {
      sq = fmaf(qv[c].x, qv[c].x, fmaf(qv[c].y, qv[c].y, fmaf(qv[c].z, qv[c].z, fmaf(qv[c].w, qv[c].w, sq))));
      sk = fmaf(kv[c].x, kv[c].x, fmaf(kv[c].y, kv[c].y, fmaf(kv[c].z, kv[c].z, fmaf(kv[c].w, kv[c].w, sk))));
    }
    sq = row16_sum(sq);
    sk = row16_sum(sk);
    const float iq = a.scale / __builtin_sqrtf(sq + a.eps), ik = 1.0f / __builtin_sqrtf(sk + a.eps);
    if (!stages) return;
#pragma unroll
    for (int c = 0; c < kQ; ++c) {
      const float4 x = {qv[c].x * iq, qv[c].y * iq, qv[c].z * iq, qv[c].w * iq};
      const float4 y = {kv[c].x * ik, kv[c].y * ik, kv[c].z * ik, kv[c].w * ik};
      qk = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, qk))));
      *reinterpret_cast<float4 *>(&qs[buf][r][4 * lane + 64 * c]) = x;
      *reinterpret_cast<float4 *>(&ks[buf][r][4 * lane + 64 * c]) = y;
    }
    qk = row16_sum(qk);
    vs[buf][r][lane] = vv;
    if (lane == 0) cs[buf][r] = float4{expf(gv), t0 + r < end ? 1.0f / (1.0f + expf(-bv)) : 0.0f, qk, gv};
  };

  float s[4 * kQ];
#pragma unroll
  for (int c = 0; c < kQ; ++c) {
    const float4 f = *reinterpret_cast<const float4 *>(state + 64 * c);
    s[4 * c] = f.x; s[4 * c + 1] = f.y; s[4 * c + 2] = f.z; s[4 * c + 3] = f.w;
  }
  double gates = 0.0;
  fetch(0);
  stage(0, 0);
  int buf = 0;
  for (int64_t t0 = 0; t0 < end; t0 += kT, buf ^= 1) {
    // one barrier a round: a wave writes buffer buf ^ 1 below only after every wave has
    // left the round before, which read it
    __syncthreads();
    if (t0 + kT < end) fetch(t0 + kT);
    float kept = 0.0f;
#pragma unroll 4
    for (int t = 0; t < kT; ++t) {
      const float4 c4 = cs[buf][t];
      const float vi = vs[buf][t][r];
      float kk[4 * kQ], dk[2] = {0.0f, 0.0f}, dq[2] = {0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < kQ; ++c) {
        const float4 x = *reinterpret_cast<const float4 *>(&qs[buf][t][4 * lane + 64 * c]);
        const float4 y = *reinterpret_cast<const float4 *>(&ks[buf][t][4 * lane + 64 * c]);
        kk[4 * c] = y.x; kk[4 * c + 1] = y.y; kk[4 * c + 2] = y.z; kk[4 * c + 3] = y.w;
        dk[0] = fmaf(s[4 * c + 1], y.y, fmaf(s[4 * c], y.x, dk[0]));
        dk[1] = fmaf(s[4 * c + 3], y.w, fmaf(s[4 * c + 2], y.z, dk[1]));
        dq[0] = fmaf(s[4 * c + 1], x.y, fmaf(s[4 * c], x.x, dq[0]));
        dq[1] = fmaf(s[4 * c + 3], x.w, fmaf(s[4 * c + 2], x.z, dq[1]));
      }
      const float sk = row16_sum(dk[0] + dk[1]), sq = row16_sum(dq[0] + dq[1]);
      const float u = (vi - c4.x * sk) * c4.y;
      const float o = fmaf(u, c4.z, c4.x * sq);
#pragma unroll
      for (int e = 0; e < 4 * kQ; ++e) s[e] = fmaf(u, kk[e], c4.x * s[e]);
      kept = lane == t ? o : kept;  // lane t keeps token t's output
      gates += (double)c4.w;
    }
    if (lane < kT && t0 + lane < end) out[(t0 + lane) * a.heads * kD + r] = kept;
    if (t0 + kT < end) stage(t0 + kT, buf ^ 1);
  }
#pragma unroll
  for (int c = 0; c < kQ; ++c)
    *reinterpret_cast<float4 *>(state + 64 * c) = float4{s[4 * c], s[4 * c + 1], s[4 * c + 2], s[4 * c + 3]};
  if (a.gate_offset != nullptr && blockIdx.x == 0 && tid == 0) {
    float *o = a.gate_offset + b * a.heads + h;
    *o = (float)((double)*o + gates);
  }
}

}  // namespace

size_t deltanet_prompt_workspace(int batch, int64_t n, int heads, int head_dim) {
  (void)batch, (void)n, (void)heads, (void)head_dim;
  return 0;
}

int launch_deltanet_prompt(const float *q, const float *k, const float *v, const int64_t *strides,
                           const float *gate, const float *beta, float *state, float *gate_offset,
                           const int *lens, float *out, int batch, int64_t n, int k_heads,
                           int heads, int head_dim, float scale, float eps, void *ws,
                           size_t ws_bytes, hipStream_t s) {
  for (const void *p : {(const void *)q, (const void *)k, (const void *)v, (const void *)state, (const void *)out})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0)
      return set_error(PKV_ERR_ARG, "q, k, v, state and out must be 16-byte aligned");
  for (int i = 0; i < 6; ++i)
    if (strides[i] % 4 != 0) return set_error(PKV_ERR_ARG, "q, k and v strides must be multiples of 4 elements");
  if (heads > 65535 || batch > 65535) return set_error(PKV_ERR_ARG, "heads and batch must be <= 65535");
  (void)ws, (void)ws_bytes;
  ScanArgs a{q, k, v, gate, beta, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5],
             state, gate_offset, out, lens, n, heads, heads / k_heads, scale, eps};
  const dim3 grid((unsigned)(head_dim / 16), (unsigned)heads, (unsigned)batch);
  switch (head_dim) {
    case 64: hipLaunchKernelGGL((scan_tokens_kernel<64, 16>), grid, dim3(256), 0, s, a); break;
    case 128: hipLaunchKernelGGL((scan_tokens_kernel<128, 16>), grid, dim3(256), 0, s, a); break;
    case 256: hipLaunchKernelGGL((scan_tokens_kernel<256, 8>), grid, dim3(256), 0, s, a); break;
    default:
      return set_error(PKV_ERR_UNSUPPORTED, "delta net prompt: head_dim must be 64, 128 or 256");
  }
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

}  // namespace pkv
