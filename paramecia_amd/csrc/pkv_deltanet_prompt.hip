// Gated delta rule over the tokens of a prompt for gfx950: the prompt form of the
// Gated-DeltaNet state update (delta_net_chunked, paramecia-model/src/qwen3_next.rs:
// 3506-3731; one token: pkv_deltanet.hip).
//
// Per sequence b and value head h, with its key head h / (heads / k_heads) and the state
// S[i][j] (i: value channel, j: key channel), for t = 0 .. end - 1:
//   qn = q_t * scale / sqrt(|q_t|^2 + eps), kn = k_t / sqrt(|k_t|^2 + eps)
//   S *= exp(gate_t); u_i = (v_ti - S_i . kn) * sigmoid(beta_t); S_i += u_i kn; o_ti = S_i . qn
//
// Short prompts go token by token (scan_tokens). Longer ones go by chunks of 64 tokens, in two
// launches a segment. With G_t the sum of a chunk's gates up to t, M = S^T in front of it
// and be = sigmoid(beta), the updates U (row t: u_t) of a chunk obey
//   (I + A) U = diag(be) (V - diag(e^G) K M),  A_ts = be_t e^(G_t - G_s) k_t . k_s  (s < t)
// so that, with T = (I + A)^-1 and P_ts = e^(G_t - G_s) q_t . k_s (s <= t),
//   R = diag(be) (V - diag(e^G) K M),  U = T R,
//   O = diag(e^G) Q M + P U,  M' = e^(G_63) M + K^T diag(e^(G_63 - G)) U.
// chunk_kernel makes T, P and the operands of K and Q for all chunks at once; state_kernel
// then walks each head's chunks, its state in registers. Products run on
// v_mfma_f32_16x16x32_f16 with every operand in two fp16 parts (22 bits; hi hi + hi lo + lo hi),
// which is exact to about f32: k, q, T and P are at most 1 in magnitude, and M, R and U are
// scaled by powers of two from bounds that hold while no gate is positive. A head with a
// positive gate, or a value that is not finite or past 2^90, goes token by token instead (a
// NaN then reaches the tokens behind it and no others, as there).
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
template <int kD>
struct TokenStage {
  static constexpr int kT = kD == 256 ? 8 : 16;
  float q[2][kT][kD], k[2][kT][kD];
  float4 c[2][kT];  // exp(gate), sigmoid(beta), kn . qn, gate
  float v[2][kT][16];
};

// Rows row0 .. row0 + 15 of head (b, h), tokens first .. end - 1.
template <int kD>
__device__ void scan_tokens(const ScanArgs &a, TokenStage<kD> &st, int64_t b, int64_t h, int row0,
                            int64_t first, int64_t end) {
  constexpr int kQ = kD / 64;  // quads per lane
  constexpr int kT = TokenStage<kD>::kT;
  const int tid = threadIdx.x, lane = tid & 15, r = tid >> 4;
  const int64_t hk = h / a.rep;
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
      *reinterpret_cast<float4 *>(&st.q[buf][r][4 * lane + 64 * c]) = x;
      *reinterpret_cast<float4 *>(&st.k[buf][r][4 * lane + 64 * c]) = y;
    }
    qk = row16_sum(qk);
    st.v[buf][r][lane] = vv;
    if (lane == 0) st.c[buf][r] = float4{expf(gv), t0 + r < end ? 1.0f / (1.0f + expf(-bv)) : 0.0f, qk, gv};
  };

  float s[4 * kQ];
#pragma unroll
  for (int c = 0; c < kQ; ++c) {
    const float4 f = *reinterpret_cast<const float4 *>(state + 64 * c);
    s[4 * c] = f.x; s[4 * c + 1] = f.y; s[4 * c + 2] = f.z; s[4 * c + 3] = f.w;
  }
  double gates = 0.0;
  fetch(first);
  stage(first, 0);
  int buf = 0;
  for (int64_t t0 = first; t0 < end; t0 += kT, buf ^= 1) {
    // one barrier a round: a wave writes buffer buf ^ 1 below only after every wave has
    // left the round before, which read it
    __syncthreads();
    if (t0 + kT < end) fetch(t0 + kT);
    float kept = 0.0f;
#pragma unroll 4
    for (int t = 0; t < kT; ++t) {
      const float4 c4 = st.c[buf][t];
      const float vi = st.v[buf][t][r];
      float kk[4 * kQ], dk[2] = {0.0f, 0.0f}, dq[2] = {0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < kQ; ++c) {
        const float4 x = *reinterpret_cast<const float4 *>(&st.q[buf][t][4 * lane + 64 * c]);
        const float4 y = *reinterpret_cast<const float4 *>(&st.k[buf][t][4 * lane + 64 * c]);
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
  if (a.gate_offset != nullptr && row0 == 0 && tid == 0) {
    float *o = a.gate_offset + b * a.heads + h;
    *o = (float)((double)*o + gates);
  }
}

template <int kD>
__global__ __launch_bounds__(256) void scan_tokens_kernel(ScanArgs a) {
  __shared__ __attribute__((aligned(16))) TokenStage<kD> st;
  const int64_t end = valid_tokens(a.lens, blockIdx.z, a.n);
  if (end > 0) scan_tokens<kD>(a, st, blockIdx.z, blockIdx.y, blockIdx.x * 16, 0, end);
}

// ---- by chunks
constexpr int kC = 64;           // tokens per chunk
constexpr float kUp = 1024.0f;   // scale of the fp16 parts of k, q, T and P (at most 1)
constexpr float kDown = 1.0f / 1024.0f;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// The empty asm pins x: where x is a product, the compiler otherwise rounds one use of hi from
// the exact product (v_fma_mixlo_f16) and another from its f32 value; now and then the two
// differ by a step of hi, which lo then does not make up for (a value off by 2^-12).
__device__ __forceinline__ void split(float x, _Float16 &hi, _Float16 &lo) {
  asm("" : "+v"(x));
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

// Workspace of a segment. An operand fragment is 16 rows by 32 k in two parts (hi, lo) of 64
// lanes x 16 bytes: lane (m, g) holds row m, k 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3,
// the order in which an MFMA's result tiles become the next one's B operand without moving
// between lanes. T and P are lower triangular: row tile w needs k step 1 (tokens 32 .. 63)
// from w = 2 on, six fragments.
struct ChunkWs {
  h8 *k, *q;       // [b][chunk][key head][row tile 4][d / 32][2][64]
  h8 *kt;          // [b][chunk][key head][d / 16][k step 2][2][64]: rows are key channels
  h8 *t, *p;       // [b][chunk][head][6][2][64]
  float *meta;     // [b][chunk][head][3][64]: be, e^G, e^(G_63 - G)
  double *gates;   // [b][chunk][head]: the chunk's sum
  unsigned *odd;   // [b][chunk][head]: this chunk needs the token path
};
constexpr size_t kFrag = 2 * 64;  // h8 per fragment
struct ChunkArgs {
  ScanArgs s;
  ChunkWs w;
  int64_t first;  // the segment's first token
  int chunks;     // of the segment
  int k_heads, batch;
};
__device__ __forceinline__ int tri(int w, int p) { return w < 2 ? w : 2 * w - 2 + p; }

// A chunk of one key head: normalised K and Q as fragments, their products, and for each of
// its value heads T and P. A wave owns 16 tokens, its lanes load q and k in fragment order;
// the waves take each other's K from LDS. T = (I + A)^-1 by blocks of 16, in f32: the
// diagonal blocks by forward substitution (16 lanes each, a column a lane), then T_ij = -T_ii
// sum_k A_ik T_kj down the block columns, a wave each, on v_mfma_f32_16x16x4_f32, whose result
// tiles are the next product's B operand as they are.
template <int kD>
__global__ __launch_bounds__(256) void chunk_kernel(ChunkArgs a) {
  constexpr int kS = kD / 32, kRow = kD + 8, kSq = 68;
  constexpr int kKB = 2 * kC * kRow * 2, kAB = 4 * kC * kSq * 4;
  __shared__ __attribute__((aligned(16))) char lds[kKB > kAB ? kKB : kAB];
  __shared__ double gam[2][kC];
  __shared__ float bet[2][kC];
  __shared__ unsigned bad;
  _Float16(*kh)[kC][kRow] = reinterpret_cast<_Float16(*)[kC][kRow]>(lds);  // [hi, lo][token][k]
  float(*am)[kC][kSq] = reinterpret_cast<float(*)[kC][kSq]>(lds);           // A of two heads, then P and T of both
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  const int64_t chunk = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int64_t t0 = a.first + chunk * kC;
  const int64_t left = valid_tokens(a.s.lens, b, a.s.n) - t0;
  if (left <= 0) return;
  if (tid == 0) bad = 0u;
  const int64_t slot = (b * a.chunks + chunk) * a.k_heads + hk;

  // ---- q and k of token t0 + 16 w + m
  h8 kf[kS][2], qf[kS][2];
  bool fine = true;
  {
    const bool on = 16 * w + m < left;
    const int64_t t = on ? t0 + 16 * w + m : t0;
    const float *src[2] = {a.s.k + b * a.s.kb + t * a.s.kt + hk * kD + 4 * g,
                           a.s.q + b * a.s.qb + t * a.s.qt + hk * kD + 4 * g};
    float x[2][kS][8];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float4 f = *reinterpret_cast<const float4 *>(src[u] + 32 * s + 16 * c);
          x[u][s][4 * c] = f.x; x[u][s][4 * c + 1] = f.y; x[u][s][4 * c + 2] = f.z; x[u][s][4 * c + 3] = f.w;
        }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float sq = 0.0f;
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[u][s][i] = on ? x[u][s][i] : 0.0f;
          sq = fmaf(x[u][s][i], x[u][s][i], sq);
        }
      sq += __shfl_xor(sq, 16);
      sq += __shfl_xor(sq, 32);
      const float up = on ? kUp / __builtin_sqrtf(sq + a.s.eps) : 0.0f;
      fine = fine && sq < 3.0e38f && up < 3.0e38f;  // false for NaN
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          _Float16 hi, lo;
          split(x[u][s][i] * up, hi, lo);
          (u == 0 ? kf : qf)[s][0][i] = hi;
          (u == 0 ? kf : qf)[s][1][i] = lo;
        }
    }
  }
  {
    h8 *ko = a.w.k + (slot * 4 + w) * kS * kFrag + lane, *qo = a.w.q + (slot * 4 + w) * kS * kFrag + lane;
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        ko[s * kFrag + 64 * u] = kf[s][u];
        qo[s * kFrag + 64 * u] = qf[s][u];
        *reinterpret_cast<h4 *>(&kh[u][16 * w + m][32 * s + 4 * g]) = __builtin_shufflevector(kf[s][u], kf[s][u], 0, 1, 2, 3);
        *reinterpret_cast<h4 *>(&kh[u][16 * w + m][32 * s + 16 + 4 * g]) = __builtin_shufflevector(kf[s][u], kf[s][u], 4, 5, 6, 7);
      }
  }
  __syncthreads();
  if (!fine) bad = 1u;
  // ---- k_t . k_s and q_t . k_s of the wave's tokens with tiles 0 .. w
  f4 kk[4], qk[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    kk[j] = qk[j] = f4{0.f, 0.f, 0.f, 0.f};
    if (j > w) continue;
    f4 kx = kk[j], qx = kk[j];
#pragma unroll
    for (int s = 0; s < kS; ++s) {
      h8 bf[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const h4 x = *reinterpret_cast<const h4 *>(&kh[u][16 * j + m][32 * s + 4 * g]);
        const h4 y = *reinterpret_cast<const h4 *>(&kh[u][16 * j + m][32 * s + 16 + 4 * g]);
        bf[u] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
      }
      kk[j] = mfma(kf[s][0], bf[0], kk[j]);
      qk[j] = mfma(qf[s][0], bf[0], qk[j]);
      kx = mfma(kf[s][1], bf[0], mfma(kf[s][0], bf[1], kx));
      qx = mfma(qf[s][1], bf[0], mfma(qf[s][0], bf[1], qx));
    }
    kk[j] = (kk[j] + kx) * (kDown * kDown);
    qk[j] = (qk[j] + qx) * (kDown * kDown);
  }
  // ---- K^T's fragments: rows are key channels 16 at + m, k the chunk's tokens
#pragma unroll
  for (int c = 0; c < kD / 64; ++c) {
    const int at = w * (kD / 64) + c;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        h8 f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = kh[u][32 * p + 16 * (i >> 2) + 4 * g + (i & 3)][16 * at + m];
        a.w.kt[((slot * (kD / 16) + at) * 2 + p) * kFrag + 64 * u + lane] = f;
      }
  }
  // ---- two value heads at a time
  for (int r0 = 0; r0 < a.s.rep; r0 += 2) {
    const int heads = a.s.rep - r0 < 2 ? a.s.rep - r0 : 2;
    const int64_t h0 = hk * a.s.rep + r0;
    const int64_t out = (b * a.chunks + chunk) * a.s.heads + h0;
    __syncthreads();  // kh, or the heads before, are done with; bad is set
    if (w < heads) {
      const bool on = lane < left;
      const int64_t at = (b * a.s.n + t0 + (on ? lane : 0)) * a.s.heads + h0 + w;
      const float gv = on ? a.s.gate[at] : 0.0f, bv = on ? a.s.beta[at] : 0.0f;
      const bool odd = !(gv <= 0.0f) || bv != bv;
      // e^-10000 is 0: a smaller gate does the same
      double G = (double)fmaxf(gv, -10000.0f), sum = on && !odd ? (double)gv : 0.0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(G, o);
        G += lane >= o ? up : 0.0;
        sum += __shfl_xor(sum, o);
      }
      const double last = __shfl(G, 63);
      const float be = on ? 1.0f / (1.0f + expf(-bv)) : 0.0f;
      gam[w][lane] = G;
      bet[w][lane] = be;
      float *meta = a.w.meta + (out + w) * 3 * kC + lane;
      meta[0] = be;
      meta[kC] = expf((float)G);
      meta[2 * kC] = expf((float)(last - G));
      const bool any = __ballot(odd) != 0;
      if (lane == 0) {
        a.w.gates[out + w] = sum;
        a.w.odd[out + w] = any || bad != 0u ? 1u : 0u;
      }
    }
    __syncthreads();
    for (int e = 0; e < heads; ++e) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j > (w | 1)) continue;  // a fragment covers two tiles
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = 16 * w + 4 * g + i, s = 16 * j + m;
          const float dec = s <= t ? expf((float)(gam[e][t] - gam[e][s])) : 0.0f;
          am[e][t][s] = s < t ? bet[e][t] * dec * kk[j][i] : 0.0f;
          am[2 + e][t][s] = s <= t ? dec * qk[j][i] : 0.0f;
        }
      }
    }
    __syncthreads();
    // the fragments of a lower triangular matrix's rows 16 w ..
    const auto put_rows = [&](const float(*x)[kSq], h8 *o) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        if (p > w >> 1) continue;
        h8 f[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const f4 y = *reinterpret_cast<const f4 *>(&x[16 * w + m][32 * p + 16 * c + 4 * g]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            _Float16 hi, lo;
            split(y[i] * kUp, hi, lo);
            f[0][4 * c + i] = hi;
            f[1][4 * c + i] = lo;
          }
        }
        o[tri(w, p) * kFrag + lane] = f[0];
        o[tri(w, p) * kFrag + 64 + lane] = f[1];
      }
    };
    for (int e = 0; e < heads; ++e) put_rows(am[2 + e], a.w.p + (out + e) * 6 * kFrag);
    if (w < heads) {  // lane m of block g: column m of its inverse
      float D[16];
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        float acc[4] = {t == m ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < t; s += 4) {
          const f4 x = *reinterpret_cast<const f4 *>(&am[w][16 * g + t][16 * g + s]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (s + i < t) acc[i] = fmaf(-x[i], D[s + i], acc[i]);
        }
        D[t] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
      }
#pragma unroll
      for (int t = 0; t < 16; ++t) am[w][16 * g + t][16 * g + m] = D[t];
    }
    __syncthreads();
    for (int e = 0; e < heads; ++e) {
      const int j = e == 0 ? w : 3 - w;  // long columns beside short ones
      f4 T[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < j) continue;
        if (i == j) {
#pragma unroll
          for (int c = 0; c < 4; ++c) T[i][c] = am[e][16 * j + 4 * g + c][16 * j + m];
        } else {
          f4 x = f4{0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
          for (int k = 0; k < i; ++k) {
            if (k < j) continue;
            const f4 row = *reinterpret_cast<const f4 *>(&am[e][16 * i + m][16 * k + 4 * g]);
#pragma unroll
            for (int c = 0; c < 4; ++c) x = __builtin_amdgcn_mfma_f32_16x16x4f32(row[c], T[k][c], x, 0, 0, 0);
          }
          const f4 row = *reinterpret_cast<const f4 *>(&am[e][16 * i + m][16 * i + 4 * g]);
#pragma unroll
          for (int c = 0; c < 4; ++c) y = __builtin_amdgcn_mfma_f32_16x16x4f32(row[c], x[c], y, 0, 0, 0);
          T[i] = -y;
        }
        // over P, whose zeros above the diagonal are T's too
#pragma unroll
        for (int c = 0; c < 4; ++c) am[2 + e][16 * i + 4 * g + c][16 * j + m] = T[i][c];
      }
    }
    __syncthreads();
    for (int e = 0; e < heads; ++e) put_rows(am[2 + e], a.w.t + (out + e) * 6 * kFrag);
  }
}

// Barrier that orders LDS only: loads of the next chunk stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
__device__ __forceinline__ uint32_t mag(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  const auto dpp = [](uint32_t v, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  x = umax(x, dpp(x, std::integral_constant<int, 0xB1>{}));
  x = umax(x, dpp(x, std::integral_constant<int, 0x4E>{}));
  x = umax(x, dpp(x, std::integral_constant<int, 0x141>{}));
  x = umax(x, dpp(x, std::integral_constant<int, 0x140>{}));
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = umax(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return umax(b[0], b[1]);
}
// The exponent that takes values up to `bound` (finite) below 2^15.
__device__ __forceinline__ int scale_exp(float bound) {
  const int e = 14 - ((int)(__builtin_bit_cast(uint32_t, bound) >> 23) - 127);
  return e > 100 ? 100 : e;
}
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

template <int kD>
union StateLds {
  struct {
    h8 m[kD / 32][2][64];   // the state's fragments
    h4 r[2][2][64][2], u[2][2][64][2], v[2][2][64][2];  // R, U and U e^(G_63 - G): [k step][part][lane][half]
    uint32_t top[4][2];     // largest |M| and |v| of each wave
    unsigned odd;
  } c;
  TokenStage<kD> t;
};

// The chunks of 16 value channels of one head, in order, by eight waves. Waves 0 - 3 carry the
// state: wave w owns key channels w d / 4 .. of it (f32, in an MFMA result's layout) and
// tokens 16 w .. of each chunk. Waves 4 - 7 make the outputs of the same tokens beside them, off
// the path from one chunk to the next. A wave loads its fragments of the next chunk (K and Q:
// of the one after, where the registers hold both) when a stage has just used them.
template <int kD>
__global__ __launch_bounds__(512) void state_kernel(ChunkArgs a) {
  constexpr int kS = kD / 32, kN = kD / 64;
  constexpr bool kDeep = kD <= 128;
  __shared__ __attribute__((aligned(16))) StateLds<kD> lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, w = wave & 3, m = lane & 15, g = lane >> 4;
  // the workgroups of a key head share an XCD and its L2 (workgroups go to the 8 XCDs in turn)
  const int groups = a.batch * a.k_heads, per = a.s.rep * (kD / 16);
  int grp, in;
  if (groups % 8 == 0) {
    const int id = blockIdx.x >> 3;
    grp = (id / per) * 8 + (blockIdx.x & 7);
    in = id % per;
  } else {
    grp = blockIdx.x / per;
    in = blockIdx.x % per;
  }
  const int64_t b = grp / a.k_heads, hk = grp % a.k_heads, h = hk * a.s.rep + in / (kD / 16);
  const int row0 = (in % (kD / 16)) * 16;
  int64_t end = valid_tokens(a.s.lens, b, a.s.n);
  const int64_t stop = a.first + (int64_t)a.chunks * kC;
  end = end < stop ? end : stop;
  if (end <= a.first) return;
  const int chunks = (int)((end - a.first + kC - 1) / kC);
  const int64_t kstep = (int64_t)a.k_heads * 4 * kS * kFrag, tstep = (int64_t)a.s.heads * 6 * kFrag;
  const int64_t key0 = b * a.chunks * a.k_heads + hk, val0 = b * a.chunks * a.s.heads + h;
  const float *meta = a.w.meta + val0 * 3 * kC + 16 * w + 4 * g;
  const int64_t mstep = (int64_t)a.s.heads * 3 * kC;
  const int64_t tok = a.first + 16 * w + 4 * g;  // the lane's first token of chunk 0

  if (tid == 0) lds.c.odd = 0u;
  __syncthreads();
  for (int c = tid; c < chunks; c += 512)
    if (a.w.odd[val0 + (int64_t)c * a.s.heads] != 0u) lds.c.odd = 1u;

  constexpr float kRoot = kD == 64 ? 8.1f : kD == 128 ? 11.4f : 16.1f;  // above sqrt(d)
  float mtop, vtop;
  bool odd;
  auto get_top = [&]() {
    const uint32_t x = umax(umax(lds.c.top[0][0], lds.c.top[1][0]), umax(lds.c.top[2][0], lds.c.top[3][0]));
    const uint32_t y = umax(umax(lds.c.top[0][1], lds.c.top[1][1]), umax(lds.c.top[2][1], lds.c.top[3][1]));
    mtop = __builtin_bit_cast(float, x);
    vtop = __builtin_bit_cast(float, y);
    odd = x > 0x6C800000u || y > 0x6C800000u;  // 2^90
  };
  // Scales of a chunk. R and U: the state's rows have norms up to sqrt(d) mtop, to which each
  // token adds vtop. The next state's, from this chunk's bounds: it is split before its
  // largest value is known to all waves.
  const auto exp_u = [&]() { return scale_exp(fmaf(65.0f, vtop, kRoot * mtop)); };
  const auto exp_m = [&]() { return scale_exp(fmaf(64.0f, vtop, kRoot * mtop)); };
  // four values' parts as half of a B fragment
  const auto put4 = [&](h4 (*to)[64][2], const f4 &x) {
    h4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      _Float16 p, q;
      split(x[i], p, q);
      hi[i] = p;
      lo[i] = q;
    }
    to[0][lane][w & 1] = hi;
    to[1][lane][w & 1] = lo;
  };
  const f4 zero = {0.f, 0.f, 0.f, 0.f};

  if (wave < 4) {
    const h8 *kw = a.w.k + (key0 * 4 + w) * kS * kFrag + lane;
    const h8 *ktw = a.w.kt + (key0 * (kD / 16) + w * kN) * 2 * kFrag + lane;
    const h8 *tw = a.w.t + (val0 * 6 + tri(w, 0)) * kFrag + lane;
    const float *vp = a.s.v + b * a.s.vb + tok * a.s.vt + h * kD + row0 + m;
    float *state = a.s.state + ((b * a.s.heads + h) * kD + row0 + m) * kD + w * (kD / 4) + 4 * g;
    h8 ka[kS][2], kb[kDeep ? kS : 1][2], ktf[kN][2][2], tf[2][2];
    f4 v, be, eg, ec;
    float whole;
    const auto load_k = [&](int c, h8 (*f)[2]) {
      const h8 *p = kw + (c < chunks ? c : chunks - 1) * kstep;
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) f[s][u] = p[s * kFrag + 64 * u];
    };
    const auto load_t = [&](int c) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (p <= w >> 1) tf[p][u] = tw[c * tstep + p * kFrag + 64 * u];
    };
    const auto load_kt = [&](int c) {
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int u = 0; u < 2; ++u) ktf[n][p][u] = ktw[c * kstep + (n * 2 + p) * kFrag + 64 * u];
    };
    const auto load_v = [&](int c, f4 &x) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] = tok + (int64_t)c * kC + i < end ? vp[((int64_t)c * kC + i) * a.s.vt] : 0.0f;
    };
    const auto load_meta = [&](int c, f4 &x, f4 &y, f4 &z, float &all) {
      const float *p = meta + c * mstep;
      x = *reinterpret_cast<const f4 *>(p);
      y = *reinterpret_cast<const f4 *>(p + kC);
      z = *reinterpret_cast<const f4 *>(p + 2 * kC);
      all = p[2 * kC - 1 - (16 * w + 4 * g)];  // e^(G_63)
    };
    load_meta(0, be, eg, ec, whole);
    load_v(0, v);
    load_k(0, ka);
    if constexpr (kDeep) load_k(1, kb);
    load_t(0);
    load_kt(0);
    f4 M[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) M[n] = *reinterpret_cast<const f4 *>(state + 16 * n);
    // largest |M| and |v| of the wave: as integers, so that a NaN is larger than everything
    const auto put_top = [&]() {
      uint32_t x = 0u, y = 0u;
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) x = umax(x, mag(M[n][i]));
#pragma unroll
      for (int i = 0; i < 4; ++i) y = umax(y, mag(v[i]));
      x = wave_max(x);
      y = wave_max(y);
      if (lane == 0) {
        lds.c.top[w][0] = x;
        lds.c.top[w][1] = y;
      }
    };
    const auto put_m = [&](float up) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        h4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          _Float16 x, y;
          split(M[n][i] * up, x, y);
          hi[i] = x;
          lo[i] = y;
        }
        const int at = w * kN + n;
        reinterpret_cast<h4 *>(&lds.c.m[at >> 1][0][lane])[at & 1] = hi;
        reinterpret_cast<h4 *>(&lds.c.m[at >> 1][1][lane])[at & 1] = lo;
      }
    };
    put_top();
    __syncthreads();
    get_top();
    odd = odd || lds.c.odd != 0u;
    int em = scale_exp(mtop);
    if (!odd) put_m(pow2(em));
    lds_barrier();

    const auto step = [&](int c, h8 (*kf)[2]) {
      const int next = c + 1 < chunks ? c + 1 : c;
      f4 vn, bn, gn, cn;
      float wn;
      load_meta(next, bn, gn, cn, wn);
      load_v(next, vn);
      const int eu = exp_u(), em1 = exp_m();
      // ---- R = be (V - e^G K M)
      f4 km = zero, kx = zero, ky = zero;
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        const h8 hi = lds.c.m[s][0][lane], lo = lds.c.m[s][1][lane];
        km = mfma(kf[s][0], hi, km);
        kx = mfma(kf[s][0], lo, kx);
        ky = mfma(kf[s][1], hi, ky);
      }
      load_k(c + (kDeep ? 2 : 1), kf);
      const float dm = kDown * pow2(-em), up = pow2(eu);
      f4 r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = (be[i] * up) * (v[i] - eg[i] * ((km[i] + (kx[i] + ky[i])) * dm));
      put4(lds.c.r[w >> 1], r);
      lds_barrier();
      // ---- U = T R, times 2^eu
      f4 u = zero, ux = zero, uy = zero;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        if (p > w >> 1) continue;
        const h8 hi = *reinterpret_cast<const h8 *>(lds.c.r[p][0][lane]), lo = *reinterpret_cast<const h8 *>(lds.c.r[p][1][lane]);
        u = mfma(tf[p][0], hi, u);
        ux = mfma(tf[p][0], lo, ux);
        uy = mfma(tf[p][1], hi, uy);
      }
      load_t(next);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = (u[i] + (ux[i] + uy[i])) * kDown;
      put4(lds.c.u[w >> 1], u);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] *= ec[i];
      put4(lds.c.v[w >> 1], u);
      lds_barrier();
      // ---- the next state
      f4 n0[kN], nx[kN], ny[kN];
#pragma unroll
      for (int n = 0; n < kN; ++n) n0[n] = nx[n] = ny[n] = zero;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const h8 hi = *reinterpret_cast<const h8 *>(lds.c.v[p][0][lane]), lo = *reinterpret_cast<const h8 *>(lds.c.v[p][1][lane]);
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          n0[n] = mfma(ktf[n][p][0], hi, n0[n]);
          nx[n] = mfma(ktf[n][p][0], lo, nx[n]);
          ny[n] = mfma(ktf[n][p][1], hi, ny[n]);
        }
      }
      load_kt(next);
      const float du = kDown * pow2(-eu);
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) M[n][i] = fmaf(M[n][i], whole, (n0[n][i] + (nx[n][i] + ny[n][i])) * du);
      put_m(pow2(em1));
      v = vn;
      be = bn;
      eg = gn;
      ec = cn;
      whole = wn;
      em = em1;
      put_top();
      lds_barrier();
      get_top();
    };
    if constexpr (kDeep) {
      for (int c = 0; c < chunks && !odd; c += 2) {
        step(c, ka);
        if (c + 1 < chunks && !odd) step(c + 1, kb);
      }
    } else {
      for (int c = 0; c < chunks && !odd; ++c) step(c, ka);
    }
    if (!odd) {
#pragma unroll
      for (int n = 0; n < kN; ++n) *reinterpret_cast<f4 *>(state + 16 * n) = M[n];
    }
  } else {
    const h8 *qw = a.w.q + (key0 * 4 + w) * kS * kFrag + lane;
    const h8 *pw = a.w.p + (val0 * 6 + tri(w, 0)) * kFrag + lane;
    float *op = a.s.out + ((b * a.s.n + tok) * a.s.heads + h) * kD + row0 + m;
    h8 qa[kS][2], qb[kDeep ? kS : 1][2], pf[2][2];
    f4 eg;
    const auto load_q = [&](int c, h8 (*f)[2]) {
      const h8 *p = qw + (c < chunks ? c : chunks - 1) * kstep;
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) f[s][u] = p[s * kFrag + 64 * u];
    };
    const auto load_p = [&](int c) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (p <= w >> 1) pf[p][u] = pw[c * tstep + p * kFrag + 64 * u];
    };
    eg = *reinterpret_cast<const f4 *>(meta + kC);
    load_q(0, qa);
    if constexpr (kDeep) load_q(1, qb);
    load_p(0);
    __syncthreads();
    get_top();
    odd = odd || lds.c.odd != 0u;
    int em = scale_exp(mtop);
    lds_barrier();

    const auto step = [&](int c, h8 (*qf)[2]) {
      const int next = c + 1 < chunks ? c + 1 : c;
      const f4 gn = *reinterpret_cast<const f4 *>(meta + next * mstep + kC);
      const int eu = exp_u(), em1 = exp_m();
      f4 qm = zero, qx = zero, qy = zero;
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        const h8 hi = lds.c.m[s][0][lane], lo = lds.c.m[s][1][lane];
        qm = mfma(qf[s][0], hi, qm);
        qx = mfma(qf[s][0], lo, qx);
        qy = mfma(qf[s][1], hi, qy);
      }
      load_q(c + (kDeep ? 2 : 1), qf);
      const float dm = kDown * pow2(-em) * a.s.scale, du = kDown * pow2(-eu) * a.s.scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) qm[i] = eg[i] * ((qm[i] + (qx[i] + qy[i])) * dm);
      lds_barrier();
      lds_barrier();
      f4 o = zero, ox = zero, oy = zero;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        if (p > w >> 1) continue;
        const h8 hi = *reinterpret_cast<const h8 *>(lds.c.u[p][0][lane]), lo = *reinterpret_cast<const h8 *>(lds.c.u[p][1][lane]);
        o = mfma(pf[p][0], hi, o);
        ox = mfma(pf[p][0], lo, ox);
        oy = mfma(pf[p][1], hi, oy);
      }
      load_p(next);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tok + (int64_t)c * kC + i < end)
          op[((int64_t)c * kC + i) * a.s.heads * kD] = fmaf(o[i] + (ox[i] + oy[i]), du, qm[i]);
      eg = gn;
      em = em1;
      lds_barrier();
      get_top();
    };
    if constexpr (kDeep) {
      for (int c = 0; c < chunks && !odd; c += 2) {
        step(c, qa);
        if (c + 1 < chunks && !odd) step(c + 1, qb);
      }
    } else {
      for (int c = 0; c < chunks && !odd; ++c) step(c, qa);
    }
  }
  if (odd) {
    __syncthreads();
    if (wave >= 4) return;  // a wave that has ended takes no part in the barriers below
    scan_tokens<kD>(a.s, lds.t, b, h, row0, a.first, end);
    return;
  }
  if (a.s.gate_offset != nullptr && row0 == 0 && tid == 0) {
    double sum = (double)a.s.gate_offset[b * a.s.heads + h];
    for (int c = 0; c < chunks; ++c) sum += a.w.gates[val0 + (int64_t)c * a.s.heads];
    a.s.gate_offset[b * a.s.heads + h] = (float)sum;
  }
}

// A segment's chunks, and where its workspace's parts lie.
constexpr int64_t kChunkedTokens = 48;          // prompts from here on go by chunks
constexpr size_t kSegmentBytes = (size_t)96 << 20;
struct SegmentPlan {
  int chunks = 0;  // 0: token by token
  size_t k = 0, q = 0, kt = 0, t = 0, p = 0, meta = 0, gates = 0, odd = 0, bytes = 0;
};
SegmentPlan plan_segment(int batch, int64_t n, int k_heads, int heads, int d) {
  SegmentPlan s;
  if (n < kChunkedTokens) return s;
  const size_t key = (size_t)kC * d * 4;  // one operand of a key head's chunk
  const size_t per = (size_t)batch * (k_heads * 3 * key + heads * (2 * 6 * kFrag * 16 + 3 * kC * 4 + 16));
  const int64_t all = (n + kC - 1) / kC, fit = (int64_t)(kSegmentBytes / per);
  const int64_t parts = (all + (fit < 1 ? 1 : fit) - 1) / (fit < 1 ? 1 : fit);
  s.chunks = (int)((all + parts - 1) / parts);  // segments of about one length
  const size_t keys = (size_t)batch * s.chunks * k_heads, vals = (size_t)batch * s.chunks * heads;
  s.q = keys * key;
  s.kt = 2 * s.q;
  s.t = 3 * s.q;
  s.p = s.t + vals * 6 * kFrag * 16;
  s.meta = s.p + vals * 6 * kFrag * 16;
  s.gates = s.meta + vals * 3 * kC * 4;
  s.odd = s.gates + vals * 8;
  s.bytes = s.odd + (vals * 4 + 15) / 16 * 16;
  return s;
}

template <int kD>
int launch(const ScanArgs &a, const SegmentPlan &plan, int batch, int k_heads, void *ws, hipStream_t s) {
  if (plan.chunks == 0) {
    const dim3 grid((unsigned)(kD / 16), (unsigned)a.heads, (unsigned)batch);
    hipLaunchKernelGGL((scan_tokens_kernel<kD>), grid, dim3(256), 0, s, a);
    PKV_HIP(hipGetLastError());
    return PKV_OK;
  }
  char *base = static_cast<char *>(ws);
  const ChunkWs w{reinterpret_cast<h8 *>(base), reinterpret_cast<h8 *>(base + plan.q),
                  reinterpret_cast<h8 *>(base + plan.kt), reinterpret_cast<h8 *>(base + plan.t),
                  reinterpret_cast<h8 *>(base + plan.p), reinterpret_cast<float *>(base + plan.meta),
                  reinterpret_cast<double *>(base + plan.gates), reinterpret_cast<unsigned *>(base + plan.odd)};
  const int64_t all = (a.n + kC - 1) / kC;
  for (int64_t c = 0; c < all; c += plan.chunks) {
    ChunkArgs ca{a, w, c * kC, (int)(all - c < plan.chunks ? all - c : plan.chunks), k_heads, batch};
    hipLaunchKernelGGL((chunk_kernel<kD>), dim3((unsigned)ca.chunks, (unsigned)k_heads, (unsigned)batch),
                       dim3(256), 0, s, ca);
    PKV_HIP(hipGetLastError());
    hipLaunchKernelGGL((state_kernel<kD>), dim3((unsigned)(batch * a.heads * (kD / 16))), dim3(512), 0, s, ca);
    PKV_HIP(hipGetLastError());
  }
  return PKV_OK;
}

}  // namespace

size_t deltanet_prompt_workspace(int batch, int64_t n, int k_heads, int heads, int head_dim) {
  return plan_segment(batch, n, k_heads, heads, head_dim).bytes;
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
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error(PKV_ERR_UNSUPPORTED, "delta net prompt: head_dim must be 64, 128 or 256");
  if (n > ((int64_t)1 << 30) || (int64_t)batch * heads > (1 << 24))
    return set_error(PKV_ERR_ARG, "n must be <= 2^30 and batch * heads <= 2^24");
  const SegmentPlan plan = plan_segment(batch, n, k_heads, heads, head_dim);
  if (ws_bytes < plan.bytes || (plan.bytes != 0 && ws == nullptr))
    return set_error(PKV_ERR_ARG, "the workspace is smaller than pkv_deltanet_prompt_workspace says");
  if (reinterpret_cast<uintptr_t>(ws) % 16 != 0)
    return set_error(PKV_ERR_ARG, "the workspace must be 16-byte aligned");
  ScanArgs a{q, k, v, gate, beta, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5],
             state, gate_offset, out, lens, n, heads, heads / k_heads, scale, eps};
  switch (head_dim) {
    case 64: return launch<64>(a, plan, batch, k_heads, ws, s);
    case 128: return launch<128>(a, plan, batch, k_heads, ws, s);
    default: return launch<256>(a, plan, batch, k_heads, ws, s);
  }
}

}  // namespace pkv
