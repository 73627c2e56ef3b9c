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

constexpr int kMapThreads = 1024, kMapWaves = kMapThreads / 64;
// Tokens up to which the mapping workgroup writes the slots itself; more are left to a launch
// of their own.
constexpr int64_t kMapTokensInline = 4096;
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

// Exclusive sum of x over the workgroup's threads, and the sum. part: one word per wave.
__device__ __forceinline__ int64_t scan_exclusive(int64_t x, int64_t *part, int64_t &sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t z = __shfl_up(y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();  // the words' previous readers are done
  if (lane == 63) part[wave] = y;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kMapWaves; ++w) {
    const int64_t p = part[w];
    before += w < wave ? p : 0;
    all += p;
  }
  sum = all;
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
// come back onto the free stack, request by request, then the pages taken from its top. A wave
// moves the pages of its requests one request at a time, a lane a page.
__global__ __launch_bounds__(kMapThreads) void pages_map_kernel(MapArgs a) {
  __shared__ int64_t part[kMapWaves];
  __shared__ int s_starts[kStartsInLds + 1];
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 63;
  const bool staged = a.n <= kStartsInLds;
  if (tid == 0) s_bad = 0;
  const int count = *a.free_count;
  const bool one = a.n <= kMapThreads;  // each thread keeps its request
  int64_t give = 0, take = 0, add = 0;
  Request mine = request(a, tid);
  bool bad = mine.bad;
  for (int b = tid; b < a.n; b += kMapThreads) {
    const Request r = b == tid ? mine : request(a, b);
    bad |= r.bad;
    give += r.give;
    take += r.take;
    add += r.add;
  }
  int64_t gives, takes, adds;
  const int64_t give0 = scan_exclusive(give, part, gives);
  if (bad) s_bad = 1;
  const int64_t take0 = scan_exclusive(take, part, takes);
  const int64_t add0 = scan_exclusive(add, part, adds);
  const int64_t height = (int64_t)count + gives;
  const bool valid = s_bad == 0 && adds <= a.max_tokens && count >= 0 && count <= a.capacity;
  // (pages that come back make the stack higher than its memory only if they were never its own)
  const bool fits = takes <= height && height <= a.capacity;
  const bool ok = valid && fits;
  if (tid == 0) {
    *a.status = ok ? PKV_OK : valid && takes > height ? PKV_ERR_OVERFLOW : PKV_ERR_ARG;
    a.starts[a.n] = ok ? (int)adds : 0;
    if (staged) s_starts[a.n] = ok ? (int)adds : 0;
    if (ok) *a.free_count = (int)(height - takes);
  }
  // what a wave's lanes' requests move, one after the other
  const auto move = [&](const Request &r, int b, int64_t at, bool back) {
    uint64_t todo = __ballot(back ? r.give > 0 : r.take > 0);
    while (todo) {
      const int from = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int m = __shfl(back ? r.give : r.take, from);
      const int first = __shfl(back ? r.need : r.held, from);
      const int64_t base = __shfl(at, from);
      int *row = a.tables + (int64_t)__shfl(b, from) * a.max_pages + first;
      for (int j = lane; j < m; j += 64) {
        if (back) a.free_pages[base + j] = row[j];
        else row[j] = a.free_pages[base - j];
      }
    }
  };
  if (!ok) {
    for (int b = tid; b < a.n; b += kMapThreads) {
      a.totals[b] = a.lens[b];
      a.starts[b] = 0;
      if (staged) s_starts[b] = 0;
    }
  } else {
    int64_t g = 0, s = 0;
    for (int b0 = 0; b0 < a.n; b0 += kMapThreads) {
      const int b = b0 + tid;
      const Request r = one ? mine : request(a, b);
      int64_t gat = give0, sat = add0, gs = 0, ss = 0;
      if (!one) {
        gat = g + scan_exclusive(r.give, part, gs);
        sat = s + scan_exclusive(r.add, part, ss);
      }
      if (b < a.n) {
        a.totals[b] = (int)r.total;
        a.starts[b] = (int)sat;
        if (staged) s_starts[b] = (int)sat;
      }
      if (gives) move(r, b, count + gat, true);
      g += gs;
      s += ss;
    }
    __syncthreads();  // what came back lies on the stack
    int64_t t = 0;
    for (int b0 = 0; b0 < a.n; b0 += kMapThreads) {
      const int b = b0 + tid;
      const Request r = one ? mine : request(a, b);
      int64_t tat = take0, ts = 0;
      if (!one) tat = t + scan_exclusive(r.take, part, ts);
      if (takes) move(r, b, height - 1 - tat, false);
      if (b < a.n) a.held[b] = r.need;  // its only reader from here on is this thread
      t += ts;
    }
  }
  if (!a.fill) return;
  __syncthreads();
  if (staged) {
    for (int64_t i = tid; i < a.max_tokens; i += kMapThreads) write_slot(a, s_starts, i);
  } else {
    for (int64_t i = tid; i < a.max_tokens; i += kMapThreads) write_slot(a, a.starts, i);
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
// address allows no more.
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
  hipLaunchKernelGGL(pages_map_kernel, dim3(1), dim3(kMapThreads), 0, s, a);
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
