// Drafted tokens against the target's probabilities, from given random numbers.
//
// The reference keeps the hooks that take a cache back behind rejected drafts
// (paramecia-model/src/qwen3_next.rs:2755-2762, 4291-4375) and the drafts' probabilities
// (compute_draft_probs, ops.rs:470-491); the acceptance between them runs here.
//
// Draft i is accepted while u_i q_i(x_i) < p_i(x_i). The token behind the accepted ones follows
// max(p - q, 0) of the first rejected draft's rows (p alone behind the last one): the lowest
// token whose running sum exceeds u_k times the whole sum. Probabilities are read as they are
// (f32); products, differences and sums are taken in 64 bits, since a sum's border decides on a
// token and a vocabulary's f32 sum is off by more than a token's probability.
//
// Bound: one or two rows of the vocabulary a sequence (0.6 MB each), and two dependent loads (the
// drafts, then their probabilities) in front of them. The first launch sums every 256 elements of the
// rows, a wave four such chunks at once; the second, a workgroup a sequence, finds the chunk among
// their sums and the token among its elements. MI355X, a vocabulary of 151936: one sequence of 5 drafts
// 4.2 + 3.8 us, 24 of them 6.0 + 5.0 (29 MB, 4.9 TB/s of the first launch); with the sums of one
// contiguous run a thread, uncoalesced, 26 us.
#include "pkv_internal.hpp"

namespace pkv {
namespace {

constexpr int kVThreads = 256, kVWaves = kVThreads / 64;
constexpr int kChunk = 256;  // elements: four a lane
constexpr int kWaveChunks = 4, kPart = kChunk * kWaveChunks * kVWaves;  // of a workgroup of the first launch

struct VerifyArgs {
  const float *target, *draft, *u;
  const int *drafts, *counts;
  int *tokens, *accepted;
  double *sums;  // [n][chunks]: of the rest
  int64_t target_row, draft_row;  // elements between rows
  int n, k, vocab, chunks;
};

// The first rejected draft of sequence b (its count if none is), the same in every lane.
__device__ __forceinline__ int first_rejected(const VerifyArgs &a, int b, int &count) {
  const int lane = threadIdx.x & 63;
  count = a.k;
  if (a.counts) {
    const int c = a.counts[b];
    count = c < 0 ? 0 : c > a.k ? a.k : c;
  }
  bool ok = false;
  if (lane < count) {
    const int x = a.drafts[(int64_t)b * a.k + lane];
    if (x >= 0 && x < a.vocab) {
      const double p = a.target[((int64_t)b * (a.k + 1) + lane) * a.target_row + x];
      const double q = a.draft ? a.draft[((int64_t)b * a.k + lane) * a.draft_row + x] : 1.0f;
      ok = (double)a.u[(int64_t)b * (a.k + 1) + lane] * q < p;
    }
  }
  const uint64_t taken = __ballot(ok);
  const int first = ~taken == 0ull ? 64 : __builtin_ctzll(~taken);
  return __builtin_amdgcn_readfirstlane(first < count ? first : count);
}

// What is left of the row behind the accepted drafts: p, less q where a draft was rejected.
struct Rest {
  const float *p, *q;
  int gone;  // the rejected token where the draft was sure of it, else -1
};
__device__ __forceinline__ Rest rest_of(const VerifyArgs &a, int b, int row, int count) {
  Rest r;
  const bool rejected = row < count;
  r.p = a.target + ((int64_t)b * (a.k + 1) + row) * a.target_row;
  r.q = rejected && a.draft ? a.draft + ((int64_t)b * a.k + row) * a.draft_row : nullptr;
  r.gone = rejected && !a.draft ? a.drafts[(int64_t)b * a.k + row] : -1;
  return r;
}
// The lane's four elements of a chunk (zeros behind the row's end); rows begin at any multiple of 4 bytes.
struct Four {
  float x[4];
} __attribute__((packed, aligned(4)));
__device__ __forceinline__ Four four(const float *row, int64_t first, int vocab) {
  Four f = {{0.0f, 0.0f, 0.0f, 0.0f}};
  if (first + 4 <= vocab) {
    f = *reinterpret_cast<const Four *>(row + first);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (first + i < vocab) f.x[i] = row[first + i];
  }
  return f;
}
// Their weights: max(p - q, 0), or p alone. (NaN is no probability: it weighs nothing.)
__device__ __forceinline__ void weigh(const Rest &r, int64_t first, const Four &p, const Four &q, double (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double d = (double)p.x[i] - (r.q ? (double)q.x[i] : first + i == r.gone ? 1.0 : 0.0);
    w[i] = d > 0.0 ? d : 0.0;
  }
}
__device__ __forceinline__ double wave_total(double x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ double wave_running(double x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double z = __shfl_up(x, o);
    if (lane >= o) x += z;
  }
  return x;
}

__global__ __launch_bounds__(kVThreads) void verify_sums_kernel(VerifyArgs a) {
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  int count;
  const int row = first_rejected(a, b, count);
  const Rest r = rest_of(a, b, row, count);
  const int chunk = ((int)blockIdx.x * kVWaves + (int)(threadIdx.x >> 6)) * kWaveChunks;
  Four p[kWaveChunks], q[kWaveChunks];
#pragma unroll
  for (int c = 0; c < kWaveChunks; ++c) p[c] = four(r.p, (int64_t)(chunk + c) * kChunk + 4 * lane, a.vocab);
  if (r.q) {
#pragma unroll
    for (int c = 0; c < kWaveChunks; ++c) q[c] = four(r.q, (int64_t)(chunk + c) * kChunk + 4 * lane, a.vocab);
  }
#pragma unroll
  for (int c = 0; c < kWaveChunks; ++c) {
    double w[4];
    weigh(r, (int64_t)(chunk + c) * kChunk + 4 * lane, p[c], q[c], w);
    const double sum = wave_total((w[0] + w[1]) + (w[2] + w[3]));
    if (lane == 0 && chunk + c < a.chunks) a.sums[(int64_t)b * a.chunks + chunk + c] = sum;
  }
}

// A row's running sums over a workgroup's threads, each with elements [first, end) of `count`,
// whose values value(i) gives: where the sum first passes u times the whole, or, where rounding or a u
// of one leaves none, the last with weight; -1 without any. `before`: the sum in front of it.
template <typename Value>
__device__ __forceinline__ int pick(int count, float u, Value value, double &bar, double &before) {
  __shared__ double s_sum[kVWaves], s_before[kVWaves + 1];
  __shared__ int s_first[kVWaves], s_last[kVWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (count + kVThreads - 1) / kVThreads;
  const int64_t at = (int64_t)tid * per;
  const int first = at < count ? (int)at : count, end = at + per < count ? (int)at + per : count;
  double sum = 0.0;
  for (int i = first; i < end; ++i) sum += value(i);
  const double run = wave_running(sum);
  if (lane == 63) s_sum[wave] = run;
  __syncthreads();
  double start = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kVWaves; ++w) {
    start += w < wave ? s_sum[w] : 0.0;
    all += s_sum[w];
  }
  bar = (double)u * all;
  double s = start + (run - sum), held = s;
  int hit = -1, last = -1;
  for (int i = first; i < end; ++i) {
    const double w = value(i);
    if (hit < 0 && w > 0.0) {
      if (s + w > bar) hit = i;
      last = i;
      held = s;
    }
    s += w;
  }
  const uint64_t hits = __ballot(hit >= 0), some = __ballot(last >= 0);
  const int from = hits ? __builtin_ctzll(hits) : some ? 63 - __builtin_clzll(some) : 0;
  const int mine = __shfl(hit >= 0 ? hit : last, from);
  const double mine_before = __shfl(held, from);
  if (lane == 0) {
    s_first[wave] = hits ? mine : -1;
    s_last[wave] = mine;
    s_before[wave] = mine_before;
  }
  __syncthreads();
  int got = -1;
  before = 0.0;
  for (int w = kVWaves - 1; w >= 0; --w)
    if (got < 0 && s_last[w] >= 0) got = s_last[w], before = s_before[w];
  for (int w = kVWaves - 1; w >= 0; --w)
    if (s_first[w] >= 0) got = s_first[w], before = s_before[w];
  return got;
}

__global__ __launch_bounds__(kVThreads) void verify_pick_kernel(VerifyArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  int count;
  const int row = first_rejected(a, b, count);
  const Rest r = rest_of(a, b, row, count);
  const float u = a.u[(int64_t)b * (a.k + 1) + a.k];
  const double *sums = a.sums + (int64_t)b * a.chunks;
  double bar, before;
  const int chunk = pick(a.chunks, u, [&](int i) { return sums[i]; }, bar, before);
  int token = -1;
  if (chunk >= 0) {
    const int64_t first = (int64_t)chunk * kChunk + 4 * lane;
    Four q = {{0.0f, 0.0f, 0.0f, 0.0f}};
    if (r.q) q = four(r.q, first, a.vocab);
    double w[4];
    weigh(r, first, four(r.p, first, a.vocab), q, w);
    const double own = (w[0] + w[1]) + (w[2] + w[3]);
    double s = before + (wave_running(own) - own);
    int hit = -1, last = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s += w[i];
      if (w[i] > 0.0) last = (int)first + i;
      if (hit < 0 && w[i] > 0.0 && s > bar) hit = (int)first + i;
    }
    const uint64_t hits = __ballot(hit >= 0), some = __ballot(last >= 0);
    token = hits ? __shfl(hit, __builtin_ctzll(hits)) : some ? __shfl(last, 63 - __builtin_clzll(some)) : -1;
  } else if (row < count) {
    // nothing is left where q is nowhere below p: p itself, element by element
    __syncthreads();
    token = pick(a.vocab, u, [&](int i) { return r.p[i] > 0.0f ? (double)r.p[i] : 0.0; }, bar, before);
  }
  if (tid <= a.k) {
    const int64_t o = (int64_t)b * (a.k + 1) + tid;
    a.tokens[o] = tid < row ? a.drafts[(int64_t)b * a.k + tid] : tid == row ? token : -1;
  }
  if (tid == 0) a.accepted[b] = row;
}

}  // namespace

size_t verify_drafts_workspace(int n, int vocab) { return (size_t)n * (((size_t)vocab + kChunk - 1) / kChunk) * sizeof(double); }

int launch_verify_drafts(const float *target, int64_t target_row, const float *draft,
                         int64_t draft_row, const int *drafts, const int *counts, const float *u,
                         int n, int k, int vocab, int *tokens, int *accepted, void *ws,
                         hipStream_t s) {
  VerifyArgs a;
  a.target = target;
  a.draft = draft;
  a.u = u;
  a.drafts = drafts;
  a.counts = counts;
  a.tokens = tokens;
  a.accepted = accepted;
  a.sums = static_cast<double *>(ws);
  a.target_row = target_row;
  a.draft_row = draft_row;
  a.n = n;
  a.k = k;
  a.vocab = vocab;
  a.chunks = (int)(((int64_t)vocab + kChunk - 1) / kChunk);
  hipLaunchKernelGGL(verify_sums_kernel, dim3((unsigned)(((int64_t)vocab + kPart - 1) / kPart), n), dim3(kVThreads), 0, s, a);
  hipLaunchKernelGGL(verify_pick_kernel, dim3(n), dim3(kVThreads), 0, s, a);
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

}  // namespace pkv
