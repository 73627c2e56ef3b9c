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
// Bound: one or two rows of the vocabulary a sequence (0.6 MB each), so a row is summed by
// kParts workgroups (the first launch); the second finds the part, then the token.
#include "pkv_internal.hpp"

namespace pkv {
namespace {

constexpr int kVThreads = 256, kVWaves = kVThreads / 64;
constexpr int kParts = 32;

struct VerifyArgs {
  const float *target, *draft, *u;
  const int *drafts, *counts;
  int *tokens, *accepted;
  double *sums;  // [n][kParts][2]: of the rest, of the row itself
  int64_t target_row, draft_row;  // elements between rows
  int n, k, vocab, run;  // run: elements that one thread of a part sums
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

// What is left of the row behind the accepted drafts: p, and q where a draft was rejected.
struct Rest {
  const float *p, *q;
  int gone;  // the rejected token where the draft was sure of it, else -1
  // (NaN is no probability: it weighs nothing)
  __device__ __forceinline__ double raw(float x) const { return x > 0.0f ? (double)x : 0.0; }
  __device__ __forceinline__ double at(int i, float x, float y) const {
    const double d = (double)x - (q ? (double)y : i == gone ? 1.0 : 0.0);
    return d > 0.0 ? d : 0.0;
  }
};
__device__ __forceinline__ Rest rest_of(const VerifyArgs &a, int b, int row, int count) {
  Rest r;
  const bool rejected = row < count;
  r.p = a.target + ((int64_t)b * (a.k + 1) + row) * a.target_row;
  r.q = rejected && a.draft ? a.draft + ((int64_t)b * a.k + row) * a.draft_row : nullptr;
  r.gone = rejected && !a.draft ? a.drafts[(int64_t)b * a.k + row] : -1;
  return r;
}

// f(i, p_i, q_i) for i in [first, end), in order, with kMost loads in flight.
template <typename F>
__device__ __forceinline__ void walk(const Rest &r, int first, int end, F f) {
  constexpr int kMost = 8;
  for (int i = first; i < end; i += kMost) {
    float x[kMost], y[kMost];
#pragma unroll
    for (int j = 0; j < kMost; ++j) x[j] = r.p[i + j < end ? i + j : end - 1];
#pragma unroll
    for (int j = 0; j < kMost; ++j) y[j] = r.q ? r.q[i + j < end ? i + j : end - 1] : 0.0f;
#pragma unroll
    for (int j = 0; j < kMost; ++j)
      if (i + j < end) f(i + j, x[j], y[j]);
  }
}

// Exclusive sum over the workgroup, and the sum.
__device__ __forceinline__ double scan_exclusive(double x, double *part, double &sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double z = __shfl_up(y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 63) part[wave] = y;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kVWaves; ++w) {
    before += w < wave ? part[w] : 0.0;
    all += part[w];
  }
  const double up = __shfl_up(y, 1);
  sum = all;
  return before + (lane ? up : 0.0);
}

__global__ __launch_bounds__(kVThreads) void verify_sums_kernel(VerifyArgs a) {
  __shared__ double part[kVWaves];
  const int b = blockIdx.y;
  int count;
  const int row = first_rejected(a, b, count);
  const Rest r = rest_of(a, b, row, count);
  const int64_t at = ((int64_t)blockIdx.x * kVThreads + threadIdx.x) * a.run;
  const int first = at < a.vocab ? (int)at : a.vocab;
  const int end = at + a.run < a.vocab ? (int)(at + a.run) : a.vocab;
  double rest = 0.0, raw = 0.0;
  walk(r, first, end, [&](int i, float x, float y) {
    rest += r.at(i, x, y);
    raw += r.raw(x);
  });
  double rests, raws;
  scan_exclusive(rest, part, rests);
  scan_exclusive(raw, part, raws);
  if (threadIdx.x == 0) {
    double *o = a.sums + ((int64_t)b * kParts + blockIdx.x) * 2;
    o[0] = rests;
    o[1] = raws;
  }
}

__global__ __launch_bounds__(kVThreads) void verify_pick_kernel(VerifyArgs a) {
  __shared__ double part[kVWaves];
  __shared__ int s_token;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  int count;
  const int row = first_rejected(a, b, count);
  const Rest r = rest_of(a, b, row, count);
  // the part whose running sum first exceeds u times the whole: every lane of a wave holds one
  double rest = lane < kParts ? a.sums[((int64_t)b * kParts + lane) * 2] : 0.0;
  const double raw = lane < kParts ? a.sums[((int64_t)b * kParts + lane) * 2 + 1] : 0.0;
  const bool left = __any(rest > 0.0);
  if (!left) rest = raw;  // nothing is left where p and q are the same: p itself
  double run = rest;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double z = __shfl_up(run, o);
    if (lane >= o) run += z;
  }
  const double bar = (double)a.u[(int64_t)b * (a.k + 1) + a.k] * __shfl(run, 63);
  // rounding, or a u of one, may leave no running sum above the bar: the last part with weight
  const uint64_t over = __ballot(lane < kParts && run > bar && rest > 0.0), some = __ballot(rest > 0.0);
  const int mine = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
  const double before = __shfl(run - rest, mine < 0 ? 0 : mine);
  if (tid == 0) s_token = -1;
  if (mine >= 0) {
    const int64_t at = ((int64_t)mine * kVThreads + tid) * a.run;
    const int first = at < a.vocab ? (int)at : a.vocab;
    const int end = at + a.run < a.vocab ? (int)(at + a.run) : a.vocab;
    double sum = 0.0, all;
    walk(r, first, end, [&](int i, float x, float y) { sum += left ? r.at(i, x, y) : r.raw(x); });
    const double s0 = before + scan_exclusive(sum, part, all);
    // the first thread whose own sums pass the bar; without one the last that has weight
    double s = s0;
    int token = -1, last = -1;
    walk(r, first, end, [&](int i, float x, float y) {
      const double w = left ? r.at(i, x, y) : r.raw(x);
      s += w;
      if (w > 0.0) last = i;
      if (token < 0 && w > 0.0 && s > bar) token = i;
    });
    __shared__ int s_first[kVWaves], s_last[kVWaves];
    const uint64_t hit = __ballot(token >= 0), any = __ballot(last >= 0);
    const int f = __shfl(token, hit ? __builtin_ctzll(hit) : 0), l = __shfl(last, any ? 63 - __builtin_clzll(any) : 0);
    if (lane == 0) {
      s_first[tid >> 6] = hit ? f : -1;
      s_last[tid >> 6] = any ? l : -1;
    }
    __syncthreads();
    if (tid == 0) {
      int t = -1;
      for (int w = 0; w < kVWaves; ++w)
        if (t < 0) t = s_first[w];
      for (int w = kVWaves - 1; w >= 0; --w)
        if (t < 0) t = s_last[w];
      s_token = t;
    }
  }
  __syncthreads();
  const int token = s_token;
  if (tid <= a.k) {
    const int64_t o = (int64_t)b * (a.k + 1) + tid;
    a.tokens[o] = tid < row ? a.drafts[(int64_t)b * a.k + tid] : tid == row ? token : -1;
  }
  if (tid == 0) a.accepted[b] = row;
}

}  // namespace

size_t verify_drafts_workspace(int n) { return (size_t)n * kParts * 2 * sizeof(double); }

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
  a.run = (vocab + kParts * kVThreads - 1) / (kParts * kVThreads);
  hipLaunchKernelGGL(verify_sums_kernel, dim3(kParts, n), dim3(kVThreads), 0, s, a);
  hipLaunchKernelGGL(verify_pick_kernel, dim3(n), dim3(kVThreads), 0, s, a);
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

}  // namespace pkv
