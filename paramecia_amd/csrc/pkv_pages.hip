// Pages of a paged cache handed out on the device: block tables and slot maps from request
// lengths, and the new rows of K and V rounded into their slots.
//
// Role: the bookkeeping of PreallocatedQuantizedKvCache (paramecia-model/src/qwen3_next.rs:
// 343-643: seq_len, truncate, append at seq_len) for many sequences that share pages, without
// the host: a step's launches are the same whatever the lengths are, so a captured step serves
// every later one.
#include "pkv_internal.hpp"
#include "pkv_scalar.hpp"

namespace pkv {
namespace {

// Tokens up to which the mapping workgroup writes the slots itself; more are left to a launch
// of their own (24 requests of 24 rows in all: with the launch 1.2 us more; of 1024 as long; of 4096 2.7
// less).
constexpr int64_t kMapTokensInline = 1024;
constexpr int kStartsInLds = 4096;

struct MapArgs {
  const int *lens, *add;
  int *tables, *held, *free_pages, *free_count;
  int64_t *slots;
  int *positions, *starts, *totals, *status;
  int64_t max_tokens;
  int n, max_pages, capacity, page_lg, fill;
};

struct Request {
  int64_t total;
  int lens, add, held, need, give, take;
  bool bad;
};
__device__ __forceinline__ Request request(const MapArgs &a, int b) {
  Request r = {0, 0, 0, 0, 0, 0, 0, false};
  if (b >= a.n) return r;
  r.lens = a.lens[b];
  r.add = a.add[b];
  r.held = a.held[b];
  r.total = (int64_t)r.lens + r.add;
  const int64_t need = (r.total + ((int64_t(1) << a.page_lg) - 1)) >> a.page_lg;
  r.bad = r.lens < 0 || r.add < 0 || r.held < 0 || r.held > a.max_pages || need > a.max_pages ||
          r.total > 0x7FFFFFFF;
  if (r.bad) return r;
  r.need = (int)need;
  r.give = r.held > r.need ? r.held - r.need : 0;
  r.take = r.need > r.held ? r.need - r.held : 0;
  return r;
}

// Pages given, pages taken and tokens added, summed together. (A table holds fewer than 2^31 pages
// in all; the tokens of a step that is refused may pass 32 bits.)
struct Sums {
  int give, take;
  int64_t add;
  __device__ __forceinline__ Sums operator+(const Sums &o) const { return {give + o.give, take + o.take, add + o.add}; }
  __device__ __forceinline__ Sums operator-(const Sums &o) const { return {give - o.give, take - o.take, add - o.add}; }
};
// Exclusive sums over the workgroup's threads, and the sums. part: an entry per wave.
template <int kThreads>
__device__ __forceinline__ Sums scan_exclusive(const Sums &x, Sums *part, Sums &sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Sums y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const Sums z = {__shfl_up(y.give, o), __shfl_up(y.take, o), __shfl_up(y.add, o)};
    if (lane >= o) y = y + z;
  }
  __syncthreads();  // the entries' previous readers are done
  if (lane == 63) part[wave] = y;
  __syncthreads();
  Sums before = {0, 0, 0};
  sum = {0, 0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) before = before + part[w];
    sum = sum + part[w];
  }
  return before + y - x;
}

// Token t of the step: its request is the last one whose start is not behind t.
template <typename Starts>
__device__ __forceinline__ void write_slot(const MapArgs &a, const Starts &starts, int64_t t) {
  const int64_t end = starts[a.n];
  int64_t slot = -1;
  int position = 0;
  if (t < end) {
    int lo = 0, hi = a.n;  // starts[lo] <= t < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= t) lo = mid;
      else hi = mid;
    }
    position = a.lens[lo] + (int)(t - starts[lo]);
    const int64_t page = a.tables[(int64_t)lo * a.max_pages + (position >> a.page_lg)];
    slot = (page << a.page_lg) + (position & ((1 << a.page_lg) - 1));
  }
  a.slots[t] = slot;
  a.positions[t] = position;
}

// One workgroup: the requests' needs and their sums, then (if the step fits) the pages that
// come back onto the free stack, request by request, then the pages taken from its top. A lane
// moves the few pages of its request; those of a request that moves more its whole wave, a lane a
// page. Bound: the chain of its loads and barriers (MI355X: 24 requests 4.0 us, 2.8 of it a launch;
// 300 with 8001 rows 7.1, and 3.5 for their slots). All three sums take one scan: with one each the
// kernel took 3.8 us more for 24 requests.
constexpr int kLanePages = 4;
template <int kThreads>
__global__ __launch_bounds__(kThreads) void pages_map_kernel(MapArgs a) {
  __shared__ Sums part[kThreads / 64];
  __shared__ int s_starts[kStartsInLds + 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const bool staged = a.n <= kStartsInLds;
  const int count = *a.free_count;
  const bool one = a.n <= kThreads;  // each thread keeps its request
  const Request mine = request(a, tid);
  Sums own = {0, 0, 0};
  bool bad = false;
  for (int b = tid; b < a.n; b += kThreads) {
    const Request r = b == tid ? mine : request(a, b);
    bad |= r.bad;
    own = own + Sums{r.give, r.take, r.bad ? 0 : r.add};
  }
  // a request that does not fit counts as more tokens than a step holds
  if (bad) own.add = a.max_tokens + 1;
  Sums all;
  const Sums first = scan_exclusive<kThreads>(own, part, all);
  const int64_t height = (int64_t)count + all.give;
  const bool valid = all.add <= a.max_tokens && count >= 0 && count <= a.capacity;
  // (pages that come back make the stack higher than its memory only if they were never its own)
  const bool ok = valid && all.take <= height && height <= a.capacity;
  if (tid == 0) {
    *a.status = ok ? PKV_OK : valid && all.take > height ? PKV_ERR_OVERFLOW : PKV_ERR_ARG;
    a.starts[a.n] = ok ? (int)all.add : 0;
    if (staged) s_starts[a.n] = ok ? (int)all.add : 0;
  }
  // the pages of the wave's requests: back onto the stack from `at` on, or off it down from `at`
  const auto move = [&](const Request &r, int b, int64_t at, bool back) {
    const int m = back ? r.give : r.take;
    int *row = a.tables + (int64_t)b * a.max_pages + (back ? r.need : r.held);
    if (m <= kLanePages) {
#pragma unroll
      for (int j = 0; j < kLanePages; ++j) {
        if (j >= m) continue;
        if (back) a.free_pages[at + j] = row[j];
        else row[j] = a.free_pages[at - j];
      }
    }
    uint64_t todo = __ballot(m > kLanePages);
    while (todo) {
      const int from = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int many = __shfl(m, from), head = __shfl(back ? r.need : r.held, from);
      const int64_t base = __shfl(at, from);
      int *of = a.tables + (int64_t)__shfl(b, from) * a.max_pages + head;
      for (int j = lane; j < many; j += 64) {
        if (back) a.free_pages[base + j] = of[j];
        else of[j] = a.free_pages[base - j];
      }
    }
  };
  if (!ok) {
    for (int b = tid; b < a.n; b += kThreads) {
      a.totals[b] = a.lens[b];
      a.starts[b] = 0;
      if (staged) s_starts[b] = 0;
    }
  } else {
    Sums run = {0, 0, 0};
    for (int b0 = 0; b0 < a.n; b0 += kThreads) {
      const int b = b0 + tid;
      const Request r = one ? mine : request(a, b);
      Sums at = first, sum = {0, 0, 0};
      if (!one) at = run + scan_exclusive<kThreads>({r.give, r.take, r.add}, part, sum);
      if (b < a.n) {
        a.totals[b] = (int)r.total;
        a.starts[b] = (int)at.add;
        if (staged) s_starts[b] = (int)at.add;
      }
      if (all.give) move(r, b, count + (int64_t)at.give, true);
      run = run + sum;
    }
    __syncthreads();  // what came back lies on the stack, and its height was read by all
    run = {0, 0, 0};
    for (int b0 = 0; b0 < a.n; b0 += kThreads) {
      const int b = b0 + tid;
      const Request r = one ? mine : request(a, b);
      Sums at = first, sum = {0, 0, 0};
      if (!one) at = run + scan_exclusive<kThreads>({r.give, r.take, r.add}, part, sum);
      if (all.take) move(r, b, height - 1 - at.take, false);
      if (b < a.n) a.held[b] = r.need;  // its only reader from here on is this thread
      run = run + sum;
    }
    if (tid == 0) *a.free_count = (int)(height - all.take);
  }
  if (!a.fill) return;
  __syncthreads();
  if (staged) {
    for (int64_t i = tid; i < a.max_tokens; i += kThreads) write_slot(a, s_starts, i);
  } else {
    for (int64_t i = tid; i < a.max_tokens; i += kThreads) write_slot(a, a.starts, i);
  }
}

__global__ __launch_bounds__(256) void pages_slots_kernel(MapArgs a) {
  __shared__ int s_starts[kStartsInLds + 1];
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (a.n <= kStartsInLds) {
    for (int b = threadIdx.x; b <= a.n; b += 256) s_starts[b] = a.starts[b];
    __syncthreads();
    if (t < a.max_tokens) write_slot(a, s_starts, t);
  } else if (t < a.max_tokens) {
    write_slot(a, a.starts, t);
  }
}

struct RowsArgs {
  const float *src[2];  // k, v: token t at t * stride
  int64_t stride[2];
  uint16_t *dst[2];
  const int64_t *slots;
  unsigned *status;
  int64_t n, n_slots;
  int width;  // elements of a token: heads x head_dim
};

template <bool kBf>
__device__ __forceinline__ uint32_t round2(float a, float b) {
  if constexpr (kBf) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b});
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
  }
}

// Eight elements a thread (16-byte loads and stores), or one where a row's width, stride or
// address allows no more. Bound: the bytes (MI355X: 8001 rows of 512 values of K and V in F16 9.1 us,
// 5.4 TB/s, part of it in the last-level cache; 24 rows 2.6 us, a launch).
template <bool kBf, int kPer>
__global__ __launch_bounds__(256) void pages_append_kernel(RowsArgs a, int per_row) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;  // (a launch holds fewer than 2^32)
  const uint32_t row = i / (uint32_t)per_row;
  const int64_t t = row;
  if (t >= a.n) return;
  const int e = (int)(i - row * (uint32_t)per_row) * kPer, p = blockIdx.y;
  const int64_t slot = a.slots[t];
  if (slot < 0) return;
  if (slot >= a.n_slots) {
    if (e == 0) atomicOr(a.status, kStatusSlot);
    return;
  }
  const float *x = a.src[p] + t * a.stride[p] + e;
  uint16_t *y = a.dst[p] + slot * a.width + e;
  if constexpr (kPer == 8) {
    const float4 u = reinterpret_cast<const float4 *>(x)[0], w = reinterpret_cast<const float4 *>(x)[1];
    *reinterpret_cast<uint4 *>(y) = uint4{round2<kBf>(u.x, u.y), round2<kBf>(u.z, u.w),
                                          round2<kBf>(w.x, w.y), round2<kBf>(w.z, w.w)};
  } else {
    *y = (uint16_t)round2<kBf>(*x, 0.0f);
  }
}

}  // namespace

int launch_pages_map(const int *lens, const int *add, int n, int *tables, int max_pages, int *held,
                     int *free_pages, int *free_count, int capacity, int page_tokens,
                     int64_t *slots, int *positions, int64_t max_tokens, int *starts, int *totals,
                     int *status, hipStream_t s) {
  MapArgs a;
  a.lens = lens;
  a.add = add;
  a.tables = tables;
  a.held = held;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.slots = slots;
  a.positions = positions;
  a.starts = starts;
  a.totals = totals;
  a.status = status;
  a.max_tokens = max_tokens;
  a.n = n;
  a.max_pages = max_pages;
  a.capacity = capacity;
  a.page_lg = __builtin_ctz((unsigned)page_tokens);
  a.fill = max_tokens <= kMapTokensInline;
  // a thread a request: fewer waves have shorter barriers (24 requests: with 1024 threads 2.1 us more)
  if (n <= 256)
    hipLaunchKernelGGL(pages_map_kernel<256>, dim3(1), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(pages_map_kernel<1024>, dim3(1), dim3(1024), 0, s, a);
  if (!a.fill)
    hipLaunchKernelGGL(pages_slots_kernel, dim3((unsigned)((max_tokens + 255) / 256)), dim3(256), 0, s, a);
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

int launch_pages_append(int quant, const float *k, const float *v, int64_t k_stride,
                        int64_t v_stride, const int64_t *slots, int64_t n, void *k_pages,
                        void *v_pages, int64_t n_slots, int width, hipStream_t s) {
  RowsArgs a;
  a.src[0] = k;
  a.src[1] = v;
  a.stride[0] = k_stride;
  a.stride[1] = v_stride;
  a.dst[0] = static_cast<uint16_t *>(k_pages);
  a.dst[1] = static_cast<uint16_t *>(v_pages);
  a.slots = slots;
  a.n = n;
  a.n_slots = n_slots;
  a.width = width;
  if (const int rc = device_status_word(&a.status)) return rc;
  const uintptr_t any = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                        reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages);
  const bool wide = width % 8 == 0 && k_stride % 4 == 0 && v_stride % 4 == 0 && any % 16 == 0;
  const int per_row = wide ? width / 8 : width;
  const dim3 grid((unsigned)((n * per_row + 255) / 256), 2), block(256);
  const bool bf = quant == PKV_QUANT_BF16;
  if (bf && wide) hipLaunchKernelGGL((pages_append_kernel<true, 8>), grid, block, 0, s, a, per_row);
  else if (bf) hipLaunchKernelGGL((pages_append_kernel<true, 1>), grid, block, 0, s, a, per_row);
  else if (wide) hipLaunchKernelGGL((pages_append_kernel<false, 8>), grid, block, 0, s, a, per_row);
  else hipLaunchKernelGGL((pages_append_kernel<false, 1>), grid, block, 0, s, a, per_row);
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

}  // namespace pkv
