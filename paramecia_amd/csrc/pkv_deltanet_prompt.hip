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
// then walks each head's chunks, its state in registers. Products run on 16-bit MFMA:
//   K, Q, M, W = diag(e^(G_63 - G)) U: two fp16 parts (22 bits; hi hi + hi lo + lo hi). K and Q are
//     at most 1. M and W are scaled, each value channel in each chunk by a power of two of its
//     own: what they are off by relative to a channel's largest is all that counts of them. With
//     N = |M_i| in front of the chunk and Y = max be_s e^(G_63 - G_s) |v_si|, both stay below
//     e^(G_63) N + 65 Y, as a token lengthens M_i by be |v| at most, and |u_s| <= be_s (|v_si| + |M_i|).
//   T, P, R, U: three bf16 parts (24 bits and f32's exponents; the six products down to 2^-16). A
//     token's values may be small beside those of tokens behind it, for which a common scale
//     would leave no bits.
// What an output or a state is off by is thus some roundings of the largest that the token's state
// can be, as token by token (a state that later tokens erase is held to that too); what decays
// by more than e^-87 within a chunk is held to 2^-126 of what it was. The bounds want gates that are
// not positive: a head with a positive gate, with a gate below -10000, with a key or query that
// normalisation leaves below 2^-8, or with a value or state that is not finite or past 2^90 goes
// token by token instead (a NaN then reaches the tokens behind it and no others, as there).
#include <algorithm>
#include <type_traits>

#include "pkv_q8_common.hpp"

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
// other. 5 tokens of 32 heads of 128: 5.0 us, mostly the 4 MB of state and two memory latencies;
// each token more 0.2 us, the chain from one state to the next.
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
    if (lane == 0) st.c[buf][r] = float4{expf(gv), 1.0f / (1.0f + expf(-bv)), qk, gv};
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
    const auto token = [&](int t) {
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
    };
    // the slots behind the end are left out: their q and k are of zero vectors (NaN with eps = 0),
    // and 0 times an infinite state is NaN
    const int slots = end - t0 < kT ? (int)(end - t0) : kT;
    int done = 0;
    for (; done + 4 <= slots; done += 4)
#pragma unroll
      for (int i = 0; i < 4; ++i) token(done + i);
    for (; done < slots; ++done) token(done);
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
constexpr int kMeta = 4 * kC + 4;
constexpr float kUp = 1024.0f;   // scale of the fp16 parts of k and q (at most 1)
constexpr float kDown = 1.0f / 1024.0f;

// The empty asm pins x: where x is a product, the compiler otherwise rounds one use of hi from
// the exact product (v_fma_mixlo_f16) and another from its f32 value; now and then the two
// differ by a step of hi, which lo then does not make up for (a value off by 2^-12).
__device__ __forceinline__ void split(float x, _Float16 &hi, _Float16 &lo) {
  asm("" : "+v"(x));
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f4 mfma32(b8 a, b8 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Two values as three bf16 parts each, together exact; a pair of parts a word.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&o)[3]) {
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    o[p] = __builtin_bit_cast(uint32_t, b2{(__bf16)x, (__bf16)y});
    x -= __builtin_bit_cast(float, o[p] << 16);
    y -= __builtin_bit_cast(float, o[p] & 0xFFFF0000u);
  }
}
// a b of three parts each, the sums by size
__device__ __forceinline__ void mfma3(const b8 (&a)[3], const b8 (&b)[3], f4 (&c)[3]) {
  c[0] = mfma32(a[0], b[0], c[0]);
  c[1] = mfma32(a[0], b[1], c[1]);
  c[2] = mfma32(a[0], b[2], c[2]);
  c[1] = mfma32(a[1], b[0], c[1]);
  c[2] = mfma32(a[1], b[1], c[2]);
  c[2] = mfma32(a[2], b[0], c[2]);
}

// Workspace of a segment. An operand fragment is 16 rows by 32 k in two or three parts of 64
// lanes x 16 bytes: lane (m, g) holds row m, k 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3,
// the order in which an MFMA's result tiles become the next one's B operand without moving
// between lanes. T and P are lower triangular: row tile w needs k step 1 (tokens 32 .. 63)
// from w = 2 on, six fragments.
struct ChunkWs {
  h8 *k, *q;       // [b][chunk][key head][row tile 4][d / 32][2][64]
  b8 *t, *p;       // [b][chunk][head][6][3][64]
  float *meta;     // [b][chunk][head][kMeta]: be, e^G, e^(G_63 - G) and be e^(G_63 - G) (not below
                   // 2^-126 where be is not) of its tokens; then e^(G_63)
  double *gates;   // [b][chunk][head]: the chunk's sum
  unsigned *odd;   // [b][chunk][head]: this chunk needs the token path
};
constexpr size_t kFrag = 2 * 64, kFrag3 = 3 * 64;  // units of 16 bytes per fragment
struct ChunkArgs {
  ScanArgs s;
  ChunkWs w;
  int64_t first;  // the segment's first token
  int chunks;     // of the segment
  int k_heads, batch;
  int parts;      // workgroups of chunk_kernel per key head: each has some of its value heads
};
__device__ __forceinline__ int tri(int w, int p) { return w < 2 ? w : 2 * w - 2 + p; }

__device__ __forceinline__ uint32_t mag(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ float as_f(uint32_t x) { return __builtin_bit_cast(float, x); }
// over the four lanes l % 16 apart (all of them receive it)
__device__ __forceinline__ uint32_t groups_max(uint32_t x) {
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = umax(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return umax(b[0], b[1]);
}
__device__ __forceinline__ double read_lane(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}
// Sums of x over the lanes up to each one, in 64 bits: DPP shifts within rows of 16 lanes
// (0 comes in), then the rows in front.
__device__ __forceinline__ double prefix64(float x) {
  double G = (double)x;
  const auto add = [&](auto ctrl) {
    const uint64_t u = __builtin_bit_cast(uint64_t, G);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, decltype(ctrl)::value, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), decltype(ctrl)::value, 0xF, 0xF, true);
    G += __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
  };
  add(std::integral_constant<int, 0x111>{});  // row_shr:1, 2, 4, 8
  add(std::integral_constant<int, 0x112>{});
  add(std::integral_constant<int, 0x114>{});
  add(std::integral_constant<int, 0x118>{});
  const double a = read_lane(G, 15), b = read_lane(G, 31), c = read_lane(G, 47);
  const int row = (threadIdx.x >> 4) & 3;
  return G + (row == 0 ? 0.0 : row == 1 ? a : row == 2 ? a + b : (a + b) + c);
}

// A chunk of one key head: normalised K and Q as fragments, their products, and for each of
// its value heads (of a part of them, where there are workgroups for it) T and P. A wave owns 16 tokens, its lanes load q and k in fragment order;
// the waves take each other's K from LDS (barriers order LDS only: the fragments' stores are
// not waited for). T = (I + A)^-1 by blocks of 16, in f32: the
// diagonal blocks by forward substitution (16 lanes each, a column a lane), then T_ij = -T_ii
// sum_k A_ik T_kj down the block columns, a wave each, on v_mfma_f32_16x16x4_f32, whose result
// tiles are the next product's B operand as they are. 63 chunks of 16 key heads of 128 with 32 value
// heads: 48 us for 139 MB written, two workgroups a CU (LDS). 8 chunks, a round of 256 workgroups with
// a value head each, 18 us: the chain of loads, norm, products, inverse and stores.
template <int kD>
__global__ __launch_bounds__(256) void chunk_kernel(ChunkArgs a) {
  constexpr int kS = kD / 32, kRow = kD + 8, kSq = 68;
  constexpr int kKB = 2 * kC * kRow * 2, kAB = 4 * kC * kSq * 4;
  __shared__ __attribute__((aligned(16))) char lds[kKB > kAB ? kKB : kAB];
  __shared__ float4 gam[2][kC];  // a token's sum of gates, base 2: whole number and rest; be
  __shared__ unsigned bad;
  _Float16(*kh)[kC][kRow] = reinterpret_cast<_Float16(*)[kC][kRow]>(lds);  // [hi, lo][token][k]
  float(*am)[kC][kSq] = reinterpret_cast<float(*)[kC][kSq]>(lds);           // A of two heads, then P and T of both
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  const int64_t chunk = blockIdx.x, hk = blockIdx.y / a.parts, b = blockIdx.z;
  const int part = blockIdx.y % a.parts, rep0 = a.s.rep * part / a.parts, rep1 = a.s.rep * (part + 1) / a.parts;
  const int64_t t0 = a.first + chunk * kC;
  const int64_t left = valid_tokens(a.s.lens, b, a.s.n) - t0;
  if (left <= 0) return;
  if (tid == 0) bad = 0u;
  // the gates of the first two value heads, a wave each, asked for before everything else
  float gv = 0.0f, bv = 0.0f;
  const auto load_gates = [&](int r) {
    const int64_t at = (b * a.s.n + t0 + lane) * a.s.heads + hk * a.s.rep + r + w;
    const bool on = w < 2 && r + w < rep1 && lane < left;
    gv = on ? a.s.gate[at] : 0.0f;
    bv = on ? a.s.beta[at] : 0.0f;
  };
  load_gates(rep0);
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
      bool any = false;
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[u][s][i] = on ? x[u][s][i] : 0.0f;
          any = any || x[u][s][i] != 0.0f;
          sq = fmaf(x[u][s][i], x[u][s][i], sq);
        }
      sq += __shfl_xor(sq, 16);
      sq += __shfl_xor(sq, 32);
      const float up = on ? kUp / __builtin_sqrtf(sq + a.s.eps) : 0.0f;
      // false for NaN; an all but vanishing vector would leave its fp16 parts without bits
      fine = fine && sq < 3.0e38f && up < 3.0e38f && (sq > 0x1p-16f * a.s.eps || !any);
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
#pragma unroll
  for (int s = 0; s < kS; ++s)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      *reinterpret_cast<h4 *>(&kh[u][16 * w + m][32 * s + 4 * g]) = __builtin_shufflevector(kf[s][u], kf[s][u], 0, 1, 2, 3);
      *reinterpret_cast<h4 *>(&kh[u][16 * w + m][32 * s + 16 + 4 * g]) = __builtin_shufflevector(kf[s][u], kf[s][u], 4, 5, 6, 7);
    }
  const auto put_kq = [&]() {
    if (part != 0) return;
    h8 *ko = a.w.k + (slot * 4 + w) * kS * kFrag + lane, *qo = a.w.q + (slot * 4 + w) * kS * kFrag + lane;
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        ko[s * kFrag + 64 * u] = kf[s][u];
        qo[s * kFrag + 64 * u] = qf[s][u];
      }
  };
  if constexpr (kD > 128) put_kq();  // two workgroups a CU have no registers to keep them
  lds_barrier();
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
      kk[j] = mfma32(kf[s][0], bf[0], kk[j]);
      qk[j] = mfma32(qf[s][0], bf[0], qk[j]);
      kx = mfma32(kf[s][1], bf[0], mfma32(kf[s][0], bf[1], kx));
      qx = mfma32(qf[s][1], bf[0], mfma32(qf[s][0], bf[1], qx));
    }
    kk[j] = (kk[j] + kx) * (kDown * kDown);
    qk[j] = (qk[j] + qx) * (kDown * kDown);
  }
  // ---- two value heads at a time
  for (int r0 = rep0; r0 < rep1; r0 += 2) {
    const int heads = rep1 - r0 < 2 ? rep1 - r0 : 2;
    const int64_t h0 = hk * a.s.rep + r0;
    const int64_t out = (b * a.chunks + chunk) * a.s.heads + h0;
    lds_barrier();  // kh, or the heads before, are done with; bad is set
    if (w < heads) {
      // e^-10000 is 0, but its sums would leave no bits for the others: the token path's
      const bool fit = gv <= 0.0f && gv >= -10000.0f && bv == bv;
      const double G = prefix64(gv), last = read_lane(G, 63);
      const float be = lane < left ? 1.0f / (1.0f + expf(-bv)) : 0.0f;
      // 2^(whole + rest): a sum rounded to f32 would cost its power up to 2^-18
      const double G2 = G * 1.4426950408889634, whole = __builtin_rint(G2);
      const int gi = (int)whole, li = __builtin_amdgcn_readlane(gi, 63);
      const float gf = (float)(G2 - whole), lf = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, gf), 63));
      gam[w][lane] = float4{__builtin_bit_cast(float, gi), gf, be, 0.0f};
      float *meta = a.w.meta + (out + w) * kMeta;
      const float ec = __builtin_ldexpf(__builtin_amdgcn_exp2f(lf - gf), li - gi);
      meta[lane] = be;
      meta[kC + lane] = __builtin_ldexpf(__builtin_amdgcn_exp2f(gf), gi);
      meta[2 * kC + lane] = ec;
      meta[3 * kC + lane] = fmaxf(be * ec, fminf(be, 0x1p-126f));
      if (lane < 4) meta[4 * kC + lane] = __builtin_ldexpf(__builtin_amdgcn_exp2f(lf), li);
      const bool all = __ballot(!fit) == 0;
      if (lane == 0) {
        a.w.gates[out + w] = last;
        a.w.odd[out + w] = all && bad == 0u ? 0u : 1u;
      }
    }
    lds_barrier();
    load_gates(r0 + 2);
    for (int e = 0; e < heads; ++e) {
      float4 row[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) row[i] = gam[e][16 * w + 4 * g + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j > (w | 1)) continue;  // a fragment covers two tiles
        const float4 col = gam[e][16 * j + m];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = 16 * w + 4 * g + i, s = 16 * j + m;
          const float dec = __builtin_ldexpf(__builtin_amdgcn_exp2f(row[i].y - col.y),
                                             __builtin_bit_cast(int, row[i].x) - __builtin_bit_cast(int, col.x));
          am[e][t][s] = s < t ? row[i].z * dec * kk[j][i] : 0.0f;
          am[2 + e][t][s] = s <= t ? dec * qk[j][i] : 0.0f;
        }
      }
    }
    if constexpr (kD <= 128)
      if (r0 == rep0) put_kq();  // in front of the products these stores cost 3 us of 48
    lds_barrier();
    // the fragments of a lower triangular matrix's rows 16 w ..
    const auto put_rows = [&](const float(*x)[kSq], b8 *o) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        if (p > w >> 1) continue;
        u4 f[3];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const f4 y = *reinterpret_cast<const f4 *>(&x[16 * w + m][32 * p + 16 * c + 4 * g]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t o3[3];
            split3(y[2 * i], y[2 * i + 1], o3);
#pragma unroll
            for (int u = 0; u < 3; ++u) f[u][2 * c + i] = o3[u];
          }
        }
#pragma unroll
        for (int u = 0; u < 3; ++u) o[tri(w, p) * kFrag3 + 64 * u + lane] = __builtin_bit_cast(b8, f[u]);
      }
    };
    for (int e = 0; e < heads; ++e) put_rows(am[2 + e], a.w.p + (out + e) * 6 * kFrag3);
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
    lds_barrier();
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
      }
      // over P, whose zeros above the diagonal are T's too
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < j) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c) am[2 + e][16 * i + 4 * g + c][16 * j + m] = T[i][c];
      }
    }
    lds_barrier();
    for (int e = 0; e < heads; ++e) put_rows(am[2 + e], a.w.t + (out + e) * 6 * kFrag3);
  }
}

// The exponent that takes values up to `bound` (finite) below 2^15.
__device__ __forceinline__ int scale_exp(float bound) {
  const int e = 14 - ((int)(__builtin_bit_cast(uint32_t, bound) >> 23) - 127);
  return e > 126 ? 126 : e;
}
// 1 / x of a power of two
__device__ __forceinline__ float inverse2(float x) { return as_f(0x7F000000u - __builtin_bit_cast(uint32_t, x)); }
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

template <int kD, int kNT>
union StateLds {
  struct {
    h8 m[kNT][kD / 32][2][64];  // the state's fragments
    // [k step][part][lane][half]: R and U, and U e^(G_63 - G), scaled
    uint2 r[kNT][2][3][64][2], u[kNT][2][3][64][2], v[kNT][2][2][64][2];
    h8 k[2][kC][kD / 8];  // K of the chunk, [part][token][.. in keys_at's order]
    uint4 n[kNT][16], y[kNT][16];  // [channel], a word of each wave: bits of its N and Y
    float scale[kNT][16];          // of U e^(G_63 - G) and of the state behind the chunk
    unsigned odd;
  } c;
  TokenStage<kD> t;
};

// One load at a wave-uniform address and a lane's byte offset.
template <typename T>
__device__ __forceinline__ T at(const void *base, uint32_t off) {
  return *reinterpret_cast<const T *>(static_cast<const char *>(base) + off);
}
// Element i of lane q of each four lanes to element q of lane i.
__device__ __forceinline__ f4 transpose4(f4 x) {
  const auto swap = [](float v, auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, true));
  };
  const bool q1 = threadIdx.x & 1, q2 = threadIdx.x & 2;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const float t = swap(q1 ? x[i] : x[i + 1], std::integral_constant<int, 0xB1>{});  // lane ^ 1
    x[i] = q1 ? t : x[i];
    x[i + 1] = q1 ? x[i + 1] : t;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float t = swap(q2 ? x[i] : x[i + 2], std::integral_constant<int, 0x4E>{});  // lane ^ 2
    x[i] = q2 ? t : x[i];
    x[i + 2] = q2 ? x[i + 2] : t;
  }
  return x;
}
// Four values (not MFMA results themselves: lo_pair is inline asm) as fp16 parts.
__device__ __forceinline__ void split4(const f4 &x, uint2 &hi, uint2 &lo) {
  float y[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("" : "+v"(y[i]));
  hi = uint2{as_u(h2{(_Float16)y[0], (_Float16)y[1]}), as_u(h2{(_Float16)y[2], (_Float16)y[3]})};
  lo = uint2{lo_pair(y[0], y[1], hi.x), lo_pair(y[2], y[3], hi.y)};
}

// K in LDS, from which K^T's fragments are read: eight channels (a lane's of a fragment) are 16
// bytes, whose place in a token's row is turned by the token, so that eight tokens' stores and
// sixteen lanes' loads of four tokens meet in a bank two at a time at most. (With places of 8 bytes
// nothing meets; a walk takes as long, with more registers.)
template <int kD>
__device__ __forceinline__ int keys_at(int token, int c) {
  return c ^ ((((token & 3) << 2) | ((token >> 2) & 3)) & (kD / 8 - 1));
}
// Four 16-bit values a lane, transposed within 16 lanes: they load four rows of 16, lane l the
// values 4 (l % 4) .. of row l / 4, and receive a column each.
__device__ __forceinline__ h4 load_columns(const _Float16 *p) {
  typedef __fp16 v4h __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4h lds_v4h;
  return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_v4h *)(p)));
}

// The chunks of 16 kNT value channels of one head, in order, by eight waves. Waves 0 - 3 carry the
// state: wave w owns key channels w d / 4 .. of it (f32, in an MFMA result's layout) and
// tokens 16 w .. of each chunk. Waves 4 - 7 make the outputs of the same tokens beside them, off
// the path from one chunk to the next. A wave
// loads its fragments of the next chunk (K and Q: of the one after, where the registers hold
// both) when a stage has used them, the state's waves once what others wait for is in LDS. K^T
// comes from the K that the state's waves hold anyway, through LDS.
// The scales are found by the outputs' waves: Y of the next chunk while the others make U, the
// scale itself beside their product Q M.
// 63 chunks of 32 heads of 128, 256 workgroups: 130 us, 2.06 a chunk: the three stages one
// behind the other, and the 104 KB of fragments that a CU takes from L2 beside them.
// (T, P, R and U in two fp16 parts with a scale per channel: 118 us, and wrong where a channel's tokens
// differ by more than 2^10. Y and the scale by the state's waves themselves: 140.)
template <int kD, int kNT>
__global__ __launch_bounds__(512) void state_kernel(ChunkArgs a) {
  constexpr int kS = kD / 32, kN = kD / 64;
  constexpr bool kDeep = kD <= 128;
  __shared__ __attribute__((aligned(16))) StateLds<kD, kNT> lds;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), w = wave & 3;
  // the workgroups of a key head share an XCD and its L2 (workgroups go to the 8 XCDs in turn)
  const int groups = a.batch * a.k_heads, per = a.s.rep * (kD / (16 * kNT));
  int grp, in;
  if (groups % 8 == 0) {
    const int id = blockIdx.x >> 3;
    grp = (id / per) * 8 + (blockIdx.x & 7);
    in = id % per;
  } else {
    grp = blockIdx.x / per;
    in = blockIdx.x % per;
  }
  const int64_t b = grp / a.k_heads, hk = grp % a.k_heads, h = hk * a.s.rep + in / (kD / (16 * kNT));
  const int row0 = (in % (kD / (16 * kNT))) * 16 * kNT;
  int64_t end = valid_tokens(a.s.lens, b, a.s.n);
  const int64_t stop = a.first + (int64_t)a.chunks * kC;
  end = end < stop ? end : stop;
  if (end <= a.first) return;
  const int tokens = (int)(end - a.first), chunks = (tokens + kC - 1) / kC;
  const int64_t kstep = (int64_t)a.k_heads * 4 * kS * kFrag, tstep = (int64_t)a.s.heads * 6 * kFrag3;
  const int64_t key0 = b * a.chunks * a.k_heads + hk, val0 = b * a.chunks * a.s.heads + h;
  const int64_t mstep = (int64_t)a.s.heads * kMeta;
  const float *meta = a.w.meta + val0 * kMeta;
  const float *v0 = a.s.v + b * a.s.vb + a.first * a.s.vt + h * kD + row0;
  const uint32_t moff = 4u * (uint32_t)(16 * w + 4 * g), foff = 16u * (uint32_t)lane;
  // v of token 16 w + 4 g + m % 4, channels 4 (m / 4) .. + 3 (one 16-byte load, 64-byte rows):
  // the transpose within each four lanes of the MFMA result's layout. Past the end the last
  // token's, whose weight there is 0.
  const auto load_v = [&](int c, f4 (&x)[kNT]) {
    const float *p = v0 + (int64_t)c * kC * a.s.vt;
    const int last = (tokens - c * kC < kC ? tokens - c * kC : kC) - 1;
    const int t = 16 * w + 4 * g + (m & 3) < last ? 16 * w + 4 * g + (m & 3) : last;
#pragma unroll
    for (int j = 0; j < kNT; ++j) x[j] = at<f4>(p + 16 * j, 4u * ((uint32_t)t * (uint32_t)a.s.vt + (uint32_t)(m & 12)));
  };

  if (tid == 0) lds.c.odd = 0u;
  __syncthreads();
  for (int c = tid; c < chunks; c += 512)
    if (a.w.odd[val0 + (int64_t)c * a.s.heads] != 0u) lds.c.odd = 1u;

  constexpr float kRoot = kD == 64 ? 8.1f : kD == 128 ? 11.4f : 16.1f;  // above sqrt(d)
  constexpr uint32_t kLargest = 0x6C800000u;  // 2^90; infinities and NaN are larger
  bool odd = false;
  uint32_t largest = 0u;  // magnitude of a value or of a state so far
  const auto all_done = [&]() {
    if (largest > kLargest) lds.c.odd = 1u;
    lds_barrier();
    odd = lds.c.odd != 0u;
  };
  const auto whole = [&](const uint4 &t) { return as_f(umax(umax(t.x, t.y), umax(t.z, t.w))); };
  const f4 zero = {0.f, 0.f, 0.f, 0.f};

  if (wave < 4) {
    const h8 *kw = a.w.k + (key0 * 4 + w) * kS * kFrag;
    const b8 *tw = a.w.t + (val0 * 6 + tri(w, 0)) * kFrag3;
    float *state = a.s.state + ((b * a.s.heads + h) * kD + row0 + m) * kD + w * (kD / 4) + 4 * g;
    h8 ka[kS][2], kb[kDeep ? kS : 1][2], ktf[kN][2][2];
    b8 tf[2][3];
    f4 v[kNT], be, eg, ec;
    float decay, sm[kNT];   // e^(G_63); the scale of the state's fragments
    const auto load_k = [&](int c, h8 (*f)[2]) {
      const h8 *p = kw + (c < chunks ? c : chunks - 1) * kstep;
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) f[s][u] = at<h8>(p + s * kFrag + 64 * u, foff);
    };
    const auto load_t = [&](int c) {
      const b8 *q = tw + c * tstep;
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int u = 0; u < 3; ++u)
          if (p <= w >> 1) tf[p][u] = at<b8>(q + p * kFrag3 + 64 * u, foff);
    };
    const auto put_k = [&](h8 (*f)[2]) {
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) lds.c.k[u][16 * w + m][keys_at<kD>(16 * w + m, 4 * s + g)] = f[s][u];
    };
    // K^T's fragments: rows are key channels w d / 4 + 16 n + m, k the chunk's tokens
    const auto get_kt = [&]() {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int at = w * kN + n;
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            h4 x[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int t = 32 * p + 16 * c + 4 * g + (m >> 2);
              x[c] = load_columns(reinterpret_cast<const _Float16 *>(&lds.c.k[u][t][keys_at<kD>(t, 4 * (at >> 1) + (m & 3))]) + 4 * (at & 1));
            }
            ktf[n][p][u] = __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7);
          }
      }
    };
    const auto load_meta = [&](int c, f4 &x, f4 &y, f4 &z, float &e) {
      const float *p = meta + c * mstep;
      x = at<f4>(p, moff);
      y = at<f4>(p + kC, moff);
      z = at<f4>(p + 2 * kC, moff);
      e = at<float>(p + 4 * kC, 0u);
    };
    load_meta(0, be, eg, ec, decay);
    load_v(0, v);
#pragma unroll
    for (int j = 0; j < kNT; ++j) v[j] = transpose4(v[j]);
    load_k(0, ka);
    if constexpr (kDeep) load_k(1, kb);
    load_t(0);
    f4 M[kNT][kN];
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int n = 0; n < kN; ++n) M[j][n] = *reinterpret_cast<const f4 *>(state + 16 * j * kD + 16 * n);
    const auto put_n = [&]() {  // the wave's part of max |M_i|
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        uint32_t x = 0u;
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) x = umax(x, mag(M[j][n][i]));
        largest = umax(largest, x);
        x = groups_max(x);
        if (g == 0) reinterpret_cast<uint32_t *>(&lds.c.n[j][m])[w] = x;
      }
    };
    put_n();
    const auto put_m = [&]() {
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          uint2 hi, lo;
          split4(M[j][n] * sm[j], hi, lo);
          const int k = w * kN + n;
          reinterpret_cast<uint2 *>(&lds.c.m[j][k >> 1][0][lane])[k & 1] = hi;
          reinterpret_cast<uint2 *>(&lds.c.m[j][k >> 1][1][lane])[k & 1] = lo;
        }
      }
    };
    const auto put3 = [&](uint2 (*to)[64][2], const f4 &x) {
      uint32_t a2[3], b2[3];
      split3(x[0], x[1], a2);
      split3(x[2], x[3], b2);
#pragma unroll
      for (int p = 0; p < 3; ++p) to[p][lane][w & 1] = uint2{a2[p], b2[p]};
    };
    __syncthreads();
    odd = lds.c.odd != 0u;
#pragma unroll
    for (int j = 0; j < kNT; ++j) sm[j] = pow2(scale_exp(whole(lds.c.n[j][m])));
    if (!odd) put_m();
    lds_barrier();

    const auto step = [&](int c, h8 (*kf)[2]) {
      const int next = c + 1 < chunks ? c + 1 : c;
      f4 bn, gn, cn, vn[kNT];
      float en;
      load_meta(next, bn, gn, cn, en);
      load_v(next, vn);
      // ---- R = be (V - e^G K M)
      f4 km[kNT], kx[kNT], ky[kNT];
#pragma unroll
      for (int j = 0; j < kNT; ++j) km[j] = kx[j] = ky[j] = zero;
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          const h8 hi = lds.c.m[j][s][0][lane], lo = lds.c.m[j][s][1][lane];
          km[j] = mfma32(kf[s][0], hi, km[j]);
          kx[j] = mfma32(kf[s][0], lo, kx[j]);
          ky[j] = mfma32(kf[s][1], hi, ky[j]);
        }
      put_k(kf);
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        f4 r;
        const float dm = kDown * inverse2(sm[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = be[i] * fmaf(-eg[i], (km[j][i] + (kx[j][i] + ky[j][i])) * dm, v[j][i]);
        put3(lds.c.r[j][w >> 1], r);
      }
      load_k(c + (kDeep ? 2 : 1), kf);
      lds_barrier();
      // ---- U = T R, and U e^(G_63 - G) at the scale that holds the next state too
      f4 u[kNT][3];
#pragma unroll
      for (int j = 0; j < kNT; ++j) u[j][0] = u[j][1] = u[j][2] = zero;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        if (p > w >> 1) continue;
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          b8 r[3];
#pragma unroll
          for (int i = 0; i < 3; ++i) r[i] = *reinterpret_cast<const b8 *>(lds.c.r[j][p][i][lane]);
          mfma3(tf[p], r, u[j]);
        }
      }
      get_kt();
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        sm[j] = lds.c.scale[j][m];
        const f4 x = u[j][0] + (u[j][1] + u[j][2]);
        uint2 hi, lo;
        split4(x * (ec * sm[j]), hi, lo);
        lds.c.v[j][w >> 1][0][lane][w & 1] = hi;
        lds.c.v[j][w >> 1][1][lane][w & 1] = lo;
        put3(lds.c.u[j][w >> 1], x);
      }
      if constexpr (kDeep) load_t(next);
      lds_barrier();
      // ---- the next state
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        const float dv = kDown * inverse2(sm[j]);
        f4 n0[kN], nx[kN], ny[kN];
#pragma unroll
        for (int n = 0; n < kN; ++n) n0[n] = nx[n] = ny[n] = zero;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const h8 hi = *reinterpret_cast<const h8 *>(lds.c.v[j][p][0][lane]), lo = *reinterpret_cast<const h8 *>(lds.c.v[j][p][1][lane]);
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            n0[n] = mfma32(ktf[n][p][0], hi, n0[n]);
            nx[n] = mfma32(ktf[n][p][0], lo, nx[n]);
            ny[n] = mfma32(ktf[n][p][1], hi, ny[n]);
          }
        }
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) M[j][n][i] = fmaf(M[j][n][i], decay, (n0[n][i] + (nx[n][i] + ny[n][i])) * dv);
      }
      put_m();
      put_n();
      if constexpr (!kDeep) load_t(next);
#pragma unroll
      for (int j = 0; j < kNT; ++j) v[j] = transpose4(vn[j]);
      be = bn;
      eg = gn;
      ec = cn;
      decay = en;
      lds_barrier();
    };
    if constexpr (kDeep) {
      for (int c = 0; c < chunks && !odd; c += 2) {
        step(c, ka);
        if (c + 1 < chunks) step(c + 1, kb);
      }
    } else {
      for (int c = 0; c < chunks && !odd; ++c) step(c, ka);
    }
    all_done();
    if (!odd) {
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int n = 0; n < kN; ++n) *reinterpret_cast<f4 *>(state + 16 * j * kD + 16 * n) = M[j][n];
    }
  } else {
    const h8 *qw = a.w.q + (key0 * 4 + w) * kS * kFrag;
    const b8 *pw = a.w.p + (val0 * 6 + tri(w, 0)) * kFrag3;
    const uint32_t row = (uint32_t)a.s.heads * kD * 4u;  // bytes between a token's outputs
    char *o0 = reinterpret_cast<char *>(a.s.out + ((b * a.s.n + a.first) * a.s.heads + h) * kD + row0);
    const uint32_t ooff = (uint32_t)(16 * w + 4 * g + (m & 3)) * row + 4u * (uint32_t)(m & 12);
    h8 qa[kS][2], qb[kDeep ? kS : 1][2];
    b8 pf[2][3];
    f4 eg;
    const auto load_q = [&](int c, h8 (*f)[2]) {
      const h8 *p = qw + (c < chunks ? c : chunks - 1) * kstep;
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) f[s][u] = at<h8>(p + s * kFrag + 64 * u, foff);
    };
    const auto load_p = [&](int c) {
      const b8 *q = pw + c * tstep;
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int u = 0; u < 3; ++u)
          if (p <= w >> 1) pf[p][u] = at<b8>(q + p * kFrag3 + 64 * u, foff);
    };
    f4 v[kNT], cy;  // of the chunk whose Y comes next
    float decay = at<float>(meta + 4 * kC, 0u), sm[kNT];
    const auto load_y = [&](int c) {
      load_v(c < chunks ? c : chunks - 1, v);
      cy = at<f4>(meta + (c < chunks ? c : chunks - 1) * mstep + 3 * kC, moff);
    };
    const auto put_y = [&]() {  // the wave's part of Y
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        const f4 x = transpose4(v[j]);
        uint32_t y = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y = umax(y, mag(cy[i] * x[i]));
          largest = umax(largest, mag(x[i]));
        }
        y = groups_max(y);
        if (g == 0) reinterpret_cast<uint32_t *>(&lds.c.y[j][m])[w] = y;
      }
    };
    eg = at<f4>(meta + kC, moff);
    load_y(0);
    load_q(0, qa);
    if constexpr (kDeep) load_q(1, qb);
    load_p(0);
    put_y();
    load_y(1);
    __syncthreads();
    odd = lds.c.odd != 0u;
#pragma unroll
    for (int j = 0; j < kNT; ++j) sm[j] = pow2(scale_exp(whole(lds.c.n[j][m])));
    lds_barrier();

    const auto step = [&](int c, h8 (*qf)[2]) {
      const int next = c + 1 < chunks ? c + 1 : c;
      const f4 gn = at<f4>(meta + next * mstep + kC, moff);
      const float dn = at<float>(meta + next * mstep + 4 * kC, 0u);
      f4 qm[kNT], qx[kNT], qy[kNT];
#pragma unroll
      for (int j = 0; j < kNT; ++j) qm[j] = qx[j] = qy[j] = zero;
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          const h8 hi = lds.c.m[j][s][0][lane], lo = lds.c.m[j][s][1][lane];
          qm[j] = mfma32(qf[s][0], hi, qm[j]);
          qx[j] = mfma32(qf[s][0], lo, qx[j]);
          qy[j] = mfma32(qf[s][1], hi, qy[j]);
        }
      load_q(c + (kDeep ? 2 : 1), qf);
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        const float dm = kDown * inverse2(sm[j]);
        sm[j] = pow2(scale_exp(fmaf(fmaxf(decay, 0x1p-126f) * kRoot, whole(lds.c.n[j][m]), 65.0f * whole(lds.c.y[j][m]))));
        if (w == 0 && g == 0) lds.c.scale[j][m] = sm[j];
#pragma unroll
        for (int i = 0; i < 4; ++i) qm[j][i] = eg[i] * ((qm[j][i] + (qx[j][i] + qy[j][i])) * dm);
      }
      decay = dn;
      lds_barrier();
      put_y();
      load_y(c + 2);
      lds_barrier();
      f4 o[kNT], o3[kNT][3];
#pragma unroll
      for (int j = 0; j < kNT; ++j) o3[j][0] = o3[j][1] = o3[j][2] = zero;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        if (p > w >> 1) continue;
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          b8 u[3];
#pragma unroll
          for (int i = 0; i < 3; ++i) u[i] = *reinterpret_cast<const b8 *>(lds.c.u[j][p][i][lane]);
          mfma3(pf[p], u, o3[j]);
        }
      }
      load_p(next);
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] = a.s.scale * (o3[j][0][i] + (o3[j][1][i] + o3[j][2][i]) + qm[j][i]);
      eg = gn;
      lds_barrier();
      // 64 bytes of each token's row, as load_v
#pragma unroll
      for (int j = 0; j < kNT; ++j) o[j] = transpose4(o[j]);
      if (16 * w + 4 * g + (m & 3) < tokens - c * kC)
#pragma unroll
        for (int j = 0; j < kNT; ++j) *reinterpret_cast<f4 *>(o0 + (int64_t)c * kC * row + 64 * j + ooff) = o[j];
    };
    if constexpr (kDeep) {
      for (int c = 0; c < chunks && !odd; c += 2) {
        step(c, qa);
        if (c + 1 < chunks) step(c + 1, qb);
      }
    } else {
      for (int c = 0; c < chunks && !odd; ++c) step(c, qa);
    }
    all_done();
  }
  if (odd) {
    __syncthreads();
    if (wave >= 4) return;  // a wave that has ended takes no part in the barriers below
#pragma unroll 1
    for (int j = 0; j < kNT; ++j) {
      scan_tokens<kD>(a.s, lds.t, b, h, row0 + 16 * j, a.first, end);
      __syncthreads();
    }
    return;
  }
  if (a.s.gate_offset != nullptr && row0 == 0 && wave == 0) {
    double sum = 0.0;  // the chunks' sums, 64 at a time, then across the lanes
    for (int c = lane; c < chunks; c += 64) sum += a.w.gates[val0 + (int64_t)c * a.s.heads];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    float *o = a.s.gate_offset + b * a.s.heads + h;
    if (lane == 0) *o = (float)((double)*o + sum);
  }
}

// A segment's chunks, and where its workspace's parts lie.
// Prompts go by chunks from 72 tokens on, from 48 where their heads fill the GPU more than
// twice (token by token a workgroup per 16 rows). us of the call, by tokens / by chunks, 32 heads
// of 128 over 16 key heads: one sequence 64 tokens 19.0 / 19.7, 72 20.8 / 21.4, 96 25.8 / 21.6; four 32 tokens
// 23.4 / 31.6, 48 33.0 / 31.8; twelve 32 tokens 54.1 / 60.5, 48 74.7 / 62.1. More value heads per key head
// change little: 20 over 4 key heads 72 tokens 20.5 / 21.8, 32 over 32 20.6 / 22.2. 16 heads of 256: 72 tokens
// 31.9 / 30.8; 32 of 64: 80 tokens 16.2 / 17.5, 96 18.8 / 17.6.
bool by_chunks(int batch, int64_t n, int heads, int d) {
  return n >= 72 || (n >= 48 && (int64_t)batch * heads * d > 8192);
}
// A segment's operands should stay in the 256 MB of last-level cache, but what a walk pays for
// each segment (its state, the last round of workgroups) should not weigh either. us by bytes of a
// segment 80 / 160 / 240 / 640 MB, 32 heads of 128: one sequence of 8001 tokens 345 / 334 / 334 / 394,
// of 40000 1815 / 1717 / 1957 / 1862; 14 of 1100 (2, 5, 6, 18 chunks a segment) 939 / 737 /
// 694 / 593; 28 of 2000 (1, 2, 3, 10 chunks) 4455 / 3327 / 2993 / 2277, 1 GB (16) 2100. A chunk of all
// sequences is a segment at least, whatever it takes (2.2 MB a sequence there).
constexpr size_t kSegmentBytes = (size_t)160 << 20, kSegmentMost = (size_t)1 << 30;
constexpr int64_t kSegmentChunks = 32;  // up to kSegmentMost
struct SegmentPlan {
  int chunks = 0;  // 0: token by token
  size_t q = 0, t = 0, p = 0, meta = 0, gates = 0, odd = 0, bytes = 0;
};
SegmentPlan plan_segment(int batch, int64_t n, int k_heads, int heads, int d) {
  SegmentPlan s;
  if (!by_chunks(batch, n, heads, d)) return s;
  const size_t key = (size_t)kC * d * 4;  // one operand of a key head's chunk
  const size_t per = (size_t)batch * (k_heads * 2 * key + heads * (2 * 6 * kFrag3 * 16 + kMeta * 4 + 16));
  const int64_t all = (n + kC - 1) / kC;
  const int64_t fit = std::max((int64_t)(kSegmentBytes / per), std::min((int64_t)(kSegmentMost / per), kSegmentChunks));
  const int64_t parts = (all + (fit < 1 ? 1 : fit) - 1) / (fit < 1 ? 1 : fit);
  s.chunks = (int)((all + parts - 1) / parts);  // segments of about one length
  const size_t keys = (size_t)batch * s.chunks * k_heads, vals = (size_t)batch * s.chunks * heads;
  s.q = keys * key;
  s.t = 2 * s.q;
  s.p = s.t + vals * 6 * kFrag3 * 16;
  s.meta = s.p + vals * 6 * kFrag3 * 16;
  s.gates = s.meta + vals * kMeta * 4;
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
                  reinterpret_cast<b8 *>(base + plan.t), reinterpret_cast<b8 *>(base + plan.p),
                  reinterpret_cast<float *>(base + plan.meta),
                  reinterpret_cast<double *>(base + plan.gates), reinterpret_cast<unsigned *>(base + plan.odd)};
  // 32 value channels a workgroup halve the fragments' loads, 16 give twice the workgroups: one
  // sequence of 8001 tokens (256 workgroups of 16) 330 us with 16, 445 with 32; two of 4000
  // 333 and 293, seven of 1100 403 and 329. Heads of 256 have no registers for 32.
  constexpr int kWide = kD <= 128 ? 2 : 1;
  const bool wide = kWide > 1 && (int64_t)batch * a.heads * (kD / 16) > 256;
  const int64_t all = (a.n + kC - 1) / kC;
  // A key head's value heads are shared out to workgroups while all of them have a CU of their
  // own: 509 tokens, 16 key and 32 value heads of 128: 41.2 to 39.7 us, 4 and 16 42.2 to 35.6 (past
  // 256, K and Q are worked out twice for nothing: 1000 tokens 53.0 either way).
  const int64_t groups = (int64_t)plan.chunks * k_heads * batch;
  const int parts = (int)std::clamp<int64_t>(256 / groups, 1, a.rep);
  for (int64_t c = 0; c < all; c += plan.chunks) {
    ChunkArgs ca{a, w, c * kC, (int)(all - c < plan.chunks ? all - c : plan.chunks), k_heads, batch, parts};
    hipLaunchKernelGGL((chunk_kernel<kD>), dim3((unsigned)ca.chunks, (unsigned)(k_heads * parts), (unsigned)batch),
                       dim3(256), 0, s, ca);
    PKV_HIP(hipGetLastError());
    const unsigned walks = (unsigned)(batch * a.heads * (kD / 16));
    if (wide)
      hipLaunchKernelGGL((state_kernel<kD, kWide>), dim3(walks / 2), dim3(512), 0, s, ca);
    else
      hipLaunchKernelGGL((state_kernel<kD, 1>), dim3(walks), dim3(512), 0, s, ca);
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
  if (n > ((int64_t)1 << 30) || (int64_t)batch * heads * head_dim > (1 << 26))  // walks of 512 lanes: below 2^32
    return set_error(PKV_ERR_ARG, "n must be <= 2^30 and batch * heads * head_dim <= 2^26");
  SegmentPlan plan = plan_segment(batch, n, k_heads, heads, head_dim);
  if (ws_bytes < plan.bytes || (plan.bytes != 0 && ws == nullptr))
    return set_error(PKV_ERR_ARG, "the workspace is smaller than pkv_deltanet_prompt_workspace says");
  if (reinterpret_cast<uintptr_t>(ws) % 16 != 0)
    return set_error(PKV_ERR_ARG, "the workspace must be 16-byte aligned");
  // a chunk's v and out are addressed by 32-bit byte offsets
  if (strides[5] >= 1 << 24 || (int64_t)heads * head_dim >= 1 << 24) plan.chunks = 0;
  ScanArgs a{q, k, v, gate, beta, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5],
             state, gate_offset, out, lens, n, heads, heads / k_heads, scale, eps};
  switch (head_dim) {
    case 64: return launch<64>(a, plan, batch, k_heads, ws, s);
    case 128: return launch<128>(a, plan, batch, k_heads, ws, s);
    default: return launch<256>(a, plan, batch, k_heads, ws, s);
  }
}

}  // namespace pkv
