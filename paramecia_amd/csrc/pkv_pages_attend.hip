// Attention over pages that block tables on the device name: the new tokens of many requests
// (one each, a few drafted ones, prompts) over their F16 or BF16 rows, with a window and some
// first tokens that stay visible, gfx950.
//
// Role: the SDPA of the reference's float cache (paramecia-model/src/qwen3_next.rs:2492-2605)
// for requests of any lengths in one step. Query i of a request of `len` keys and `new` queries
// sits at position p = len - new + i and sees key j iff j <= p and (no window, j > p - window,
// or j < sinks); scores are scaled, clamped to +-100 and soft-maxed; a query that sees nothing
// gives zeros. Lengths, tables and row counts are read on the device: the launches of a step do
// not depend on them, so a captured step serves every later one.
//
// Mathematics: with x_j = clamp(scale q.k_j) log2(e), one pass over the keys holds per row the running
// maximum m, l = sum 2^(x_j - m) and sum 2^(x_j - m) v_j in f32; a larger maximum rescales both. Parts
// of a row are kept as means, and join as those weighed with their share 2^(m_i - max m) l_i of the
// sum: BF16 values reach 3.4e38, whose mean f32 holds and whose sum it does not. The matrix cores
// take 16-bit operands, and K and V are 16-bit rows already, so that only q and the weights are
// rounded: they go in as sums of two fp16 parts (F16 pages) or three bf16 parts (BF16), 22 and 24
// bits, which costs two or three products for one and keeps a row within 2e-6 of 64-bit sums; one
// part alone is off by 2^-11 or 2^-8.
//
// Work: a tile is 16 to 128 rows of one request (row = token x query heads of a KV head, which share
// their keys); its keys are blocks of 32 (one page each), the sinks' blocks first, then the window's. The
// blocks of all tiles and KV heads lie in one line, which is cut into equal shares, one a workgroup,
// whatever the lengths are: 24 requests of 65 to 65536 keys end together. A share that holds a whole
// tile writes its rows of out; the parts of a tile that is cut meet in the join, a launch of their own.
//
// Bound: of few rows the bytes of the keys (2 rows of 16 bits a key and KV head); of prompts 4 head_dim
// flops a key and row, twice (F16) or three times (BF16), and what brings them their operands.
#include <algorithm>

#include "pkv_half_common.hpp"
#include "pkv_internal.hpp"

namespace pkv {
namespace {

struct Tile;
struct Count {
  int64_t units;  // of a head
  int tiles;
};
struct AttendArgs {
  const float *q;  // token t, head h at t * q_t + h * q_h
  int64_t q_t, q_h;
  const uint8_t *k, *v;  // page p at p * page_bytes
  int64_t page_bytes;
  const int *tables, *lens, *starts;
  float *out;
  Tile *tiles;      // [tile]
  int64_t *before;  // [tile + 1]: units of the tiles before it
  int *firsts;      // [share]: the tile that its first block is of
  Count *count;
  float *part;      // [2 workgroup + (not its first piece)][row][head_dim]: means
  float2 *ml;       // [..][row]: running max (log2 units), sum
  unsigned *status;
  int n, tokens, heads, kv_heads, group, page_lg, n_pages, max_pages, window, sinks, max_tiles, shares, start;
  float sl2;  // scale * log2(e)
};

struct Tile {
  int b, row0, rows, tok0;  // request, first row, rows, its first token in the step
  int p0, p1;               // positions of its first and last row's tokens
  int first;                // position of row 0's token of the request (may be below 0)
  int sink_blocks, lo, blocks;
  // a tile's place in the line: what its start costs, in blocks, and its blocks
  __device__ __forceinline__ int64_t units(int start) const { return blocks ? blocks + start : 0; }
  __device__ __forceinline__ int block(int i) const { return i < sink_blocks ? i : i - sink_blocks + lo; }
};

// Request b's queries [q0, q0 + new) and keys, as far as the step and the tables hold them.
__device__ __forceinline__ void request_of(const AttendArgs &a, int b, int &q0, int &fresh, int &len) {
  if (a.starts) {
    int s0 = a.starts[b], s1 = a.starts[b + 1];
    s0 = s0 < 0 ? 0 : s0 > a.tokens ? a.tokens : s0;
    s1 = s1 < s0 ? s0 : s1 > a.tokens ? a.tokens : s1;
    q0 = s0;
    fresh = s1 - s0;
  } else {
    q0 = b;
    fresh = 1;
  }
  const int64_t most = (int64_t)a.max_pages << a.page_lg;
  len = a.lens[b];
  len = len < 0 ? 0 : len > most ? (int)most : len;
}

// Tile i of request b, whose queries begin at q0 of the step.
__device__ __forceinline__ Tile tile_of(const AttendArgs &a, int b, int q0, int fresh, int len, int i, int rows_per_tile) {
  Tile t;
  t.tok0 = q0;
  const int all = fresh * a.group;
  t.b = b;
  t.row0 = i * rows_per_tile;
  t.rows = all - t.row0 < rows_per_tile ? all - t.row0 : rows_per_tile;
  t.first = len - fresh;
  t.sink_blocks = t.lo = t.blocks = 0;
  t.p0 = t.p1 = -1;
  if (t.rows <= 0) return t;
  t.p0 = t.first + t.row0 / a.group;
  t.p1 = t.first + (t.row0 + t.rows - 1) / a.group;
  if (t.p1 < 0) return t;
  const int from = t.p0 < 0 ? 0 : t.p0;
  if (a.window > 0 && from >= a.window) {
    t.lo = (from - a.window + 1) >> 5;
    const int s = (int)(((int64_t)a.sinks + 31) >> 5);
    t.sink_blocks = s < t.lo ? s : t.lo;
  }
  t.blocks = t.sink_blocks + (t.p1 >> 5) - t.lo + 1;
  return t;
}

__device__ __forceinline__ Tile tile_of(const AttendArgs &a, int b, int i, int rows_per_tile) {
  int q0, fresh, len;
  request_of(a, b, q0, fresh, len);
  return tile_of(a, b, q0, fresh, len, i, rows_per_tile);
}

// Whether the query at position p sees key j.
__device__ __forceinline__ bool sees(const AttendArgs &a, int p, int j) {
  return j <= p && (a.window <= 0 || j > p - a.window || j < a.sinks);
}

// The line of all units: KV head after KV head, tile after tile, of each its start and its blocks.
struct Line {
  int tiles, shares;
  int64_t per_head, all;
  int64_t each;  // units of a share; the first `more` have one more
  int more;
  __device__ __forceinline__ int64_t start(int w) const { return each * w + (w < more ? w : more); }
  // The share that holds unit u.
  __device__ __forceinline__ int share(int64_t u) const {
    const int64_t longer = (each + 1) * more;
    return (int)(u < longer ? quotient(u, each + 1) : more + quotient(u - longer, each));
  }
  __device__ __forceinline__ int head(int64_t u) const { return (int)quotient(u, per_head); }
  // x / y of numbers of at least 0, in 32 bits where they fit (a 64-bit quotient takes 500 cycles)
  static __device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
    return ((x | y) >> 32) == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
  }
};
__device__ __forceinline__ Line line_of(const AttendArgs &a, int tiles, int64_t per_head) {
  Line l;
  l.tiles = tiles;
  l.per_head = per_head;
  l.all = per_head * a.kv_heads;
  l.shares = l.all < a.shares ? (int)l.all : a.shares;
  l.each = l.shares ? Line::quotient(l.all, l.shares) : 0;
  l.more = (int)(l.all - l.each * l.shares);
  return l;
}
__device__ __forceinline__ Line line_of(const AttendArgs &a) {
  const Count c = *a.count;
  return line_of(a, c.tiles, c.units);
}
// The tile that holds unit u of a head (u below the head's units).
__device__ __forceinline__ int tile_at(const AttendArgs &a, int tiles, int64_t u) {
  int lo = 0, hi = tiles;  // before[lo] <= u < before[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.before[mid] <= u) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One workgroup: the tiles of all requests, the running count of their units, and the tile that
// each share begins in.
constexpr int kPlanThreads = 1024;
__device__ __forceinline__ int64_t plan_scan(int64_t x, int64_t *part, int64_t &sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t z = __shfl_up(y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 63) part[wave] = y;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    before += w < wave ? part[w] : 0;
    all += part[w];
  }
  sum = all;
  return before + y - x;
}

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(AttendArgs a, int rows_per_tile) {
  __shared__ int64_t part[kPlanThreads / 64];
  const int tid = threadIdx.x;
  int64_t tiles = 0;
  for (int b0 = 0; b0 < a.n; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int q0, fresh = 0, len;
    if (b < a.n) request_of(a, b, q0, fresh, len);
    const int mine = (int)(((int64_t)fresh * a.group + rows_per_tile - 1) / rows_per_tile);
    int64_t sum;
    const int64_t at = tiles + plan_scan(mine, part, sum);
    // a lane names the few tiles of its request; those of a longer one its whole wave
    const auto name = [&](int64_t t, int of, int i) {
      if (t < a.max_tiles) a.tiles[t].b = of, a.tiles[t].row0 = i;
    };
    if (mine <= 4)
      for (int i = 0; i < mine; ++i) name(at + i, b, i);
    uint64_t todo = __ballot(mine > 4);
    while (todo) {
      const int from = __builtin_ctzll(todo);
      todo &= todo - 1;
      const int many = __shfl(mine, from), of = __shfl(b, from);
      const int64_t base = __shfl(at, from);
      for (int i = tid & 63; i < many; i += 64) name(base + i, of, i);
    }
    tiles += sum;
  }
  // (starts that run backwards could name more tiles than the step has rows for)
  const int count = tiles < a.max_tiles ? (int)tiles : a.max_tiles;
  __syncthreads();
  int64_t blocks = 0;
  for (int t0 = 0; t0 < count; t0 += kPlanThreads) {
    const int t = t0 + tid;
    int64_t mine = 0;
    if (t < count) {
      const Tile x = tile_of(a, a.tiles[t].b, a.tiles[t].row0, rows_per_tile);
      a.tiles[t] = x;
      mine = x.units(a.start);
    }
    int64_t sum;
    const int64_t at = blocks + plan_scan(mine, part, sum);
    if (t < count) a.before[t] = at;
    blocks += sum;
  }
  if (tid == 0) {
    a.before[count] = blocks;
    *a.count = Count{blocks, count};
  }
  __syncthreads();
  const Line line = line_of(a, count, blocks);
  for (int w = tid; w < line.shares; w += kPlanThreads) a.firsts[w] = tile_at(a, count, line.start(w) - line.head(line.start(w)) * blocks);
}

// What the plan says, from memory, or worked out by the workgroup itself: a launch less where the
// requests are a wave's lanes.
constexpr int kHereTiles = 128;
struct HerePlan {
  int before[kHereTiles + 1], count;
  Tile tiles[kHereTiles];
};
// A value that is the same in all lanes, as a scalar.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ Tile uniform(const Tile &t) {
  return Tile{uniform(t.b), uniform(t.row0), uniform(t.rows), uniform(t.tok0), uniform(t.p0), uniform(t.p1),
              uniform(t.first), uniform(t.sink_blocks), uniform(t.lo), uniform(t.blocks)};
}
// Running sums of x over a wave's lanes.
__device__ __forceinline__ int wave_running(int x) {
  const auto add = [&](auto ctrl, auto rows) {
    return __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
  };
  using std::integral_constant;
  x += add(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});  // row_shr 1, 2, 4, 8
  x += add(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
  x += add(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
  x += add(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
  x += add(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // row_bcast 15, 31
  x += add(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});
  return x;
}
template <bool kHere>
struct Plan;
template <>
struct Plan<false> {
  Line line;
  struct Lds {};
  __device__ __forceinline__ void make(const AttendArgs &a, Lds &, int, int) { line = line_of(a); }
  __device__ __forceinline__ int64_t before(const AttendArgs &a, int x) const { return a.before[x]; }
  __device__ __forceinline__ Tile tile(const AttendArgs &a, int x) const { return a.tiles[x]; }
  __device__ __forceinline__ int first(const AttendArgs &a, int share) const { return a.firsts[share]; }
};
template <>
struct Plan<true> {
  Line line;
  using Lds = HerePlan;
  const HerePlan *lds;
  // n at most 64, max_tiles at most kHereTiles, a head's units below 2^31. The first workgroup leaves
  // the plan in memory, for the join.
  __device__ __forceinline__ void make(const AttendArgs &a, Lds &p, int rows_per_tile, int threads) {
    const int tid = threadIdx.x;
    if (tid < 64) {
      int q0 = 0, fresh = 0, len = 0;
      if (tid < a.n) request_of(a, tid, q0, fresh, len);
      const int mine = (fresh * a.group + rows_per_tile - 1) / rows_per_tile;
      if (!__any(mine > 1)) {  // a tile a request (of no rows, where it has none)
        const Tile x = tile_of(a, tid, q0, fresh, len, 0, rows_per_tile);
        if (tid < a.n) p.tiles[tid] = x;
        const int y = wave_running((int)x.units(a.start));
        p.before[tid + 1] = y;
        if (tid == 0) p.before[0] = 0, p.count = a.n;
      } else {
        const int to = wave_running(mine);
        const int count = uniform(__shfl(to, 63)) < a.max_tiles ? uniform(__shfl(to, 63)) : a.max_tiles;
        for (int i = 0; i < mine && to - mine + i < count; ++i)
          p.tiles[to - mine + i] = tile_of(a, tid, q0, fresh, len, i, rows_per_tile);
        int sum = 0;
        for (int t0 = 0; t0 < count; t0 += 64) {
          const int t = t0 + tid;
          const int y = sum + wave_running(t < count ? (int)p.tiles[t].units(a.start) : 0);
          if (t < count) p.before[t + 1] = y;
          sum = uniform(__shfl(y, 63));
        }
        if (tid == 0) p.before[0] = 0, p.count = count;
      }
    }
    __syncthreads();
    const int count = uniform(p.count);
    lds = &p;
    line = line_of(a, count, uniform(p.before[count]));
    if (blockIdx.x == 0) {
      for (int t = tid; t <= count; t += threads) a.before[t] = p.before[t];
      for (int t = tid; t < count; t += threads) a.tiles[t] = p.tiles[t];
      if (tid == 0) *a.count = Count{line.per_head, count};
    }
  }
  __device__ __forceinline__ int64_t before(const AttendArgs &, int x) const { return uniform(lds->before[x]); }
  __device__ __forceinline__ Tile tile(const AttendArgs &, int x) const { return uniform(lds->tiles[x]); }
  __device__ __forceinline__ int first(const AttendArgs &a, int share) const {
    const int64_t u = line.start(share) - line.head(line.start(share)) * line.per_head;
    int x = -1;  // tiles that begin at u or before it
    for (int t0 = 0; t0 < line.tiles; t0 += 64) {
      const int t = t0 + (int)(threadIdx.x & 63);
      x += __builtin_popcountll(__ballot(t < line.tiles && lds->before[t < line.tiles ? t : 0] <= u));
    }
    if (threadIdx.x == 0) a.firsts[share] = x;
    return x;
  }
};

// A block's rows of one KV head, in the plane of K and of V: `valid` rows from byte `at`, none
// where its page is none of the pool's.
struct Block {
  int64_t at;
  uint32_t span;  // bytes that may be read: loads behind them give zeros
  int valid;
};
// 64 entries of a request's table, a lane each: a scalar load a block would be waited for there and
// then, before the reads of LDS that share its counter.
struct Table {
  int first, held;
  __device__ __forceinline__ void look_at(const AttendArgs &a, int b, int page) {
    first = page;
    const int at = page + (int)(threadIdx.x & 63);
    held = at < a.max_pages ? a.tables[(int64_t)b * a.max_pages + at] : -1;
  }
};
__device__ __forceinline__ Block block_of(const AttendArgs &a, const Tile &t, Table &table, int h, int jb, int head_bytes) {
  Block r;
  const int j0 = jb << 5;
  const uint32_t row = (uint32_t)a.kv_heads * (uint32_t)head_bytes;
  const int nth = j0 >> a.page_lg;
  if ((uint32_t)(nth - table.first) >= 64u) table.look_at(a, t.b, nth);
  const int page = __builtin_amdgcn_readlane(table.held, nth - table.first);
  const bool ok = page >= 0 && page < a.n_pages;
  const int left = t.p1 + 1 - j0;
  r.valid = !ok ? 0 : left < kBlk ? left : kBlk;
  r.at = (ok ? (int64_t)page * a.page_bytes : 0) + (int64_t)(j0 & ((1 << a.page_lg) - 1)) * row + (int64_t)h * head_bytes;
  r.span = r.valid > 0 ? (uint32_t)(r.valid - 1) * row + (uint32_t)head_bytes : 0u;
  if (!ok && threadIdx.x == 0) atomicOr(a.status, kStatusPage);
  return r;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const uint8_t *plane, const Block &b) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(plane) + b.at, 0, b.span, 0x00020000);
}

// Row `row` of a tile over its blocks [i0, i1) in plain f32 products of the keys that it sees
// alone: for pieces that met infinities or NaN, where split operands and masked keys' zero
// weights would make more NaN than the formula does, or whose sums passed f32: acc is the mean, of BF16
// at every key, of F16 (whose sums f32 holds) behind the last: a running mean takes 15% longer. The lane
// owns kE elements; m in log2 units.
template <bool kBf, int kE>
__device__ __forceinline__ void plain_row(const AttendArgs &a, const Tile &t, int h, int row, int i0, int i1,
                                          int lane, float &m, float &l, float (&acc)[kE]) {
  constexpr int kD = 64 * kE;
  const int r = t.row0 + row, tok = r / a.group, p = t.first + tok;
  const float *q = a.q + (int64_t)(t.tok0 + tok) * a.q_t + (int64_t)(h * a.group + r % a.group) * a.q_h + lane * kE;
  float x[kE];
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    x[e] = q[e] * a.sl2;
    acc[e] = 0.0f;
  }
  const int64_t stride = (int64_t)a.kv_heads * kD;
  for (int i = i0; i < i1; ++i) {
    const int j0 = t.block(i) << 5;
    const int page = a.tables[(int64_t)t.b * a.max_pages + (j0 >> a.page_lg)];
    if (page < 0 || page >= a.n_pages) continue;
    const int64_t at = (int64_t)page * a.page_bytes + 2 * ((int64_t)(j0 & ((1 << a.page_lg) - 1)) * stride + (int64_t)h * kD + lane * kE);
    const uint16_t *k = reinterpret_cast<const uint16_t *>(a.k + at), *v = reinterpret_cast<const uint16_t *>(a.v + at);
    for (int j = 0; j < kBlk; ++j) {
      if (!sees(a, p, j0 + j)) continue;
      float dot = 0.0f;
#pragma unroll
      for (int e = 0; e < kE; ++e) dot += x[e] * half_value(k[j * stride + e], kBf);
      float s = wave_sum(dot);
      s = s > kClampL2 ? kClampL2 : s < -kClampL2 ? -kClampL2 : s;  // (NaN stays)
      const float mn = fmaxf(m, s == s ? s : -kClampL2);             // (a key that was seen)
      const float c = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(s - mn);
      const float before = l * c;
      l = before + w;
      const float by = kBf ? 1.0f / l : 1.0f, kept = kBf ? before * by : c, now = w * by;
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[e] = acc[e] * kept + now * half_value(v[j * stride + e], kBf);
      m = mn;
    }
  }
  if (!kBf && m != -INFINITY)
#pragma unroll
    for (int e = 0; e < kE; ++e) acc[e] /= l;
}

// Where a piece's rows go: out if it is the whole tile, else the share's slot, as means either way.
struct Sink {
  bool whole;
  int64_t slot;
};
__device__ __forceinline__ float *row_out(const AttendArgs &a, const Tile &t, int h, int row, int kD) {
  const int r = t.row0 + row;
  return a.out + ((int64_t)(t.tok0 + r / a.group) * a.heads + h * a.group + r % a.group) * kD;
}
template <bool kBf, int kE>
__device__ __forceinline__ void plain_store(const AttendArgs &a, const Tile &t, int h, int row, int i0, int i1, int lane,
                                            const Sink &to, int rows_per_tile) {
  constexpr int kD = 64 * kE;
  float m, l, acc[kE];
  plain_row<kBf, kE>(a, t, h, row, i0, i1, lane, m, l, acc);
  const int64_t at = to.slot * rows_per_tile + row;
  float *o = to.whole ? row_out(a, t, h, row, kD) : a.part + at * kD;
#pragma unroll
  for (int e = 0; e < kE; ++e) o[lane * kE + e] = acc[e];
  if (!to.whole && lane == 0) a.ml[at] = float2{m, l};
}

// The rows of tiles without a key that they see.
template <typename P>
__device__ __forceinline__ void zero_empty(const AttendArgs &a, const P &plan, int kD, int threads) {
  for (int x = blockIdx.x; x < plan.line.tiles; x += gridDim.x) {
    if (plan.before(a, x + 1) != plan.before(a, x)) continue;
    const Tile t = plan.tile(a, x);
    for (int h = 0; h < a.kv_heads; ++h)
      for (int i = threadIdx.x; i < t.rows * kD; i += threads) row_out(a, t, h, i / kD, kD)[i % kD] = 0.0f;
  }
}

// Queries as MFMA operands: q times scale and log2(e), as sums of 16-bit parts (F16 two, with
// a power of two per row that keeps both in fp16's range; BF16 three).
template <bool kBf>
constexpr int kParts = kBf ? 3 : 2;
template <bool kBf>
__device__ __forceinline__ void parts_of(float x0, float x1, uint32_t (&w)[kParts<kBf>]) {
  if constexpr (kBf) {
    w[0] = bf2(x0, x1);
    const float r0 = x0 - bf_lo(w[0]), r1 = x1 - bf_hi(w[0]);
    w[1] = bf2(r0, r1);
    w[2] = bf2(r0 - bf_lo(w[1]), r1 - bf_hi(w[1]));
  } else {
    const h2 h = {(_Float16)x0, (_Float16)x1};
    w[0] = as_u(h);
    w[1] = fp16_sub2(x0, x1, w[0]);
  }
}
// A row's elements 32 st + 8 g .. + 7 at q + 32 st: sent for, then taken times `by` (zeros unless
// `mine`). Of a long BF16 row the second half is sent for when the first is taken; F16 needs
// the row's largest magnitude first.
template <bool kBf, int kSteps>
struct Queries {
  static constexpr int kHold = kBf && kSteps > 4 ? 4 : kSteps;
  float4 x[kHold][2];
  __device__ __forceinline__ void load(const float *q) {
#pragma unroll
    for (int st = 0; st < kHold; ++st)
#pragma unroll
      for (int y = 0; y < 2; ++y) x[st][y] = *reinterpret_cast<const float4 *>(q + 32 * st + 4 * y);
  }
  __device__ __forceinline__ void split(const float *q, bool mine, float by, u4 (&qb)[kSteps][kParts<kBf>], float &back) {
    float f = 1.0f;
    back = 1.0f;
#pragma unroll
    for (int s0 = 0; s0 < kSteps; s0 += kHold) {
      if (s0 > 0) load(q + 32 * s0);
#pragma unroll
      for (int st = 0; st < kHold; ++st)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float4 &z = x[st][y];
          z.x = mine ? z.x * by : 0.0f, z.y = mine ? z.y * by : 0.0f, z.z = mine ? z.z * by : 0.0f, z.w = mine ? z.w * by : 0.0f;
        }
      if constexpr (!kBf) {  // a row's elements to [2^14, 2^15)
        float m = 0.0f;
#pragma unroll
        for (int st = 0; st < kHold; ++st)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            m = fmaxf(m, fmaxf(fmaxf(fabsf(x[st][y].x), fabsf(x[st][y].y)), fmaxf(fabsf(x[st][y].z), fabsf(x[st][y].w))));
        int e = (int)(f2u(xmax32(xmax16(m))) >> 23) - 127;
        e = e < -100 ? -100 : e > 100 ? 100 : e;
        f = __builtin_ldexpf(1.0f, 14 - e);
        back = __builtin_ldexpf(1.0f, e - 14);
      }
#pragma unroll
      for (int st = 0; st < kHold; ++st) {
        uint32_t w[4][kParts<kBf>];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          parts_of<kBf>(x[st][y].x * f, x[st][y].y * f, w[2 * y]);
          parts_of<kBf>(x[st][y].z * f, x[st][y].w * f, w[2 * y + 1]);
        }
#pragma unroll
        for (int p = 0; p < kParts<kBf>; ++p) qb[s0 + st][p] = u4{w[0][p], w[1][p], w[2][p], w[3][p]};
      }
      if (kHold < kSteps) __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// Of eight keys from j on, `valid` of them there, the i that the query at position p sees: i <= last,
// and i > above or i < below. (No key is seen where p < j: the other limits must only not overflow.)
struct Seen {
  int last, above, below;
};
__device__ __forceinline__ Seen seen_of(const AttendArgs &a, int p, int j, int valid) {
  const int x = p - j, y = valid - 1;
  return Seen{x < y ? x : y, a.window > 0 ? (x > 0 ? x : 0) - a.window : -1, a.sinks - j};
}

// A row's softmax, the lane's eight keys 8 g .. 8 g + 7 of a block of row n. Scores come in
// raw, as the MFMA gives them: a score in log2 units is one times `back`, a power of two.
template <bool kBf>
struct Row {
  static constexpr float kUp = kBf ? 1.0f : kPUp, kLazy = kBf ? kBf16Lazy : kF16Lazy;
  float m = -INFINITY, l = 0.0f;  // the running max, raised once a score passes it by kLazy; the sum
  // Masks and clamps c and raises the max: true if any row's was, and what was summed before
  // takes `alpha`. all: every key is seen, else those of `seen`. (NaN stays: it reaches the sum.)
  template <typename Which>
  __device__ __forceinline__ bool raise(float (&c)[8], float back, bool all, Which which, float &alpha) {
    float top = fmaxf(fmaxf(fmaxf(c[0], c[1]), fmaxf(c[2], c[3])), fmaxf(fmaxf(c[4], c[5]), fmaxf(c[6], c[7])));
    const float low = fminf(fminf(fminf(c[0], c[1]), fminf(c[2], c[3])), fminf(fminf(c[4], c[5]), fminf(c[6], c[7])));
    if (!all || __any(top * back > kClampL2 || low * back < -kClampL2)) {
      const float most = kClampL2 / back;
      const Seen s = which();
      top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool seen = (i <= s.last) & ((i > s.above) | (i < s.below));
        const float x = c[i] > most ? most : c[i] < -most ? -most : c[i];
        c[i] = seen ? x : -INFINITY;
        top = fmaxf(top, c[i]);
      }
    }
    top = xmax32(xmax16(top)) * back;
    const bool up = top > m + kLazy || (m == -INFINITY && top > -INFINITY);
    if (!__any(up)) return false;
    const float mn = up ? top : m;
    alpha = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= alpha;
    return true;
  }
  // The weights (times kUp) as MFMA operands.
  __device__ __forceinline__ void weights(const float (&c)[8], float back, u4 (&pb)[kParts<kBf>]) {
    const float base = m == -INFINITY ? 0.0f : m;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(fmaf(c[i], back, -base)) * kUp;
      l += p[i];
    }
    uint32_t w[4][kParts<kBf>];
#pragma unroll
    for (int i = 0; i < 4; ++i) parts_of<kBf>(p[2 * i], p[2 * i + 1], w[i]);
#pragma unroll
    for (int x = 0; x < kParts<kBf>; ++x) pb[x] = u4{w[0][x], w[1][x], w[2][x], w[3][x]};
  }
  __device__ __forceinline__ float sum() const {  // of the row's four lanes
    float x = l;
    x += __shfl_xor(x, 16);
    x += __shfl_xor(x, 32);
    return x * (1.0f / kUp);
  }
};
// Every query of positions p0 .. p1 (p0 below 0: some see nothing) sees all keys j0 .. j0 + 31.
__device__ __forceinline__ bool all_seen(const AttendArgs &a, int p0, int p1, int j0) {
  return (j0 + 31 <= p0) & ((a.window <= 0) | ((int64_t)j0 + a.window > p1) | (j0 + 31 < a.sinks));
}

// ---- up to 16 kRT rows a tile, for one token and a few.
// Measured (MI355X, the kernel alone; 16 query heads over 2 KV heads of 256): 24 tokens of 297000 BF16
// keys in all 113 us, 5.4 TB/s of keys (a copy of 2 GiB: 4.8); one token of 131073 BF16 keys 46 us, 5.8
// TB/s; one of 1025 F16 keys 7.2 us, four dependent trips to memory (lengths, table, rows, sums of the
// line); 16 x 5 drafted tokens, F16, a window of 4096: 30 us, 16 of it the keys' bytes, the rest each
// workgroup's plan, its 40 rows of queries and its parts' rows. Straight into registers since a block's
// rows serve one tile only (by way of LDS 24 tokens took a fifth longer).
// A workgroup of kD / 64 waves: wave w takes
// elements 64 w .. of all 32 keys of a block for the scores, and columns 64 w .. of V. Rows go from
// memory straight into registers as MFMA operands, a block ahead; the waves' partial scores meet
// in LDS, one barrier a block, and of a single row tile every wave runs the softmax itself. Of two and
// three each tile's softmax is one wave's, which hands the weights on behind a second barrier (80
// drafted tokens: 30 us, 35 where every wave ran all three).
//   scores (transposed, A = K): lane (r, g) holds 8 elements of key 8 (r / 4) + 4 t + r % 4 for
//   tile t, so that the result (row n, keys 8 g + 4 t + i) is the weights' operand as it is;
//   out (transposed, A = V): lane (m, g) holds columns 4 m + j (tile j) of keys 8 g .. + 7, pairs
//   of keys joined by v_perm; the result is columns 16 g + 4 i + j of row n.
constexpr int kScoreRow = 36;  // floats, 32 keys and a pad that spreads rows over banks

template <bool kBf, int kD, int kRT, bool kHere>
__global__ __launch_bounds__(kD, 2) void few_kernel(AttendArgs a) {
  constexpr int kW = kD / 64, kRows = 16 * kRT, kP = kParts<kBf>;
  // Of several row tiles each wave runs the softmax of its own and hands the weights on
  constexpr bool kOwn = kRT > 1 && kW > 1;
  __shared__ __attribute__((aligned(16))) float sc[kOwn ? 1 : 2][kW][kRows][kScoreRow];
  __shared__ u4 s_weights[kOwn ? kRT : 1][kP][64];
  __shared__ float s_alpha[kRT][16], s_l[kRT][16];
  __shared__ uint32_t s_bad;
  __shared__ typename Plan<kHere>::Lds s_plan;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Plan<kHere> plan;
  plan.make(a, s_plan, kRows, kD);
  const Line line = plan.line;
  zero_empty(a, plan, kD, kD);
  const int share = blockIdx.x;
  if (share >= line.shares) return;
  int64_t u = line.start(share);
  const int64_t u0 = u, end = line.start(share + 1);
  if (tid == 0) s_bad = 0u;
  int turn = 0;
  const uint32_t stride = (uint32_t)a.kv_heads * 2u * kD;
  int x = plan.first(a, share), h = line.head(u);
  for (; u < end; ++x) {
    if (x == line.tiles) x = 0, ++h;
    const Tile t = plan.tile(a, x);
    if (t.blocks == 0) continue;
    const int64_t tile0 = h * line.per_head + plan.before(a, x), behind = tile0 + t.units(a.start);
    const Sink to = {u <= tile0 + a.start && end >= behind, 2 * (int64_t)share + (u > u0 ? 1 : 0)};
    const int i0 = u <= tile0 + a.start ? 0 : (int)(u - tile0) - a.start;
    const int i1 = end >= behind ? t.blocks : (int)(end - tile0) - a.start;
    u = behind;
    if (i1 <= i0) continue;  // the share ends within the tile's start

    u4 kw[2][2];
    uint2 vw[8];
    int valid;
    const auto load_k = [&](const Block &b) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t off = (uint32_t)(8 * (n >> 2) + 4 * y + (n & 3)) * stride + 128u * wave + 16u * g;
#pragma unroll
        for (int st = 0; st < 2; ++st) kw[y][st] = row_load<u4>(rsrc_of(a.k, b), off + 64 * st);
      }
    };
    const auto load_v = [&](const Block &b) {
#pragma unroll
      for (int k = 0; k < 8; ++k) vw[k] = row_load<uint2>(rsrc_of(a.v, b), (uint32_t)(8 * g + k) * stride + 128u * wave + 8u * n);
    };
    Table table;
    table.look_at(a, t.b, (t.block(i0) << 5) >> a.page_lg);
    Queries<kBf, 2> qs[kRT];
    const float *qp[kRT];
    bool mine[kRT];
    int pos[kRT];
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
      mine[rt] = 16 * rt + n < t.rows;
      const int r = t.row0 + (mine[rt] ? 16 * rt + n : 0), tok = r / a.group;
      pos[rt] = mine[rt] ? t.first + tok : -1;
      qp[rt] = a.q + (int64_t)(t.tok0 + tok) * a.q_t + (int64_t)(h * a.group + r % a.group) * a.q_h + 64 * wave + 8 * g;
      qs[rt].load(qp[rt]);
    }
    Block blk = block_of(a, t, table, h, t.block(i0), 2 * kD);
    valid = blk.valid;
    load_k(blk);
    load_v(blk);

    u4 qb[kRT][2][kP];
    float back[kRT];
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) qs[rt].split(qp[rt], mine[rt], a.sl2, qb[rt], back[rt]);
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 acc[kRT][4];
    Row<kBf> row[kRT];
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[rt][j] = zero;
    for (int i = i0; i < i1; ++i, turn ^= 1) {
      const int j0 = t.block(i) << 5;
      const bool more = i + 1 < i1;
      float(*all_sc)[kRows][kScoreRow] = sc[kOwn ? 0 : turn];
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          f4 z = zero;
#pragma unroll
          for (int p = kP - 1; p >= 0; --p)
#pragma unroll
            for (int st = 0; st < 2; ++st) z = half_mfma<kBf>(kw[y][st], qb[rt][st][p], z);
          *reinterpret_cast<float4 *>(&all_sc[wave][16 * rt + n][8 * g + 4 * y]) =
              float4{z[0] * back[rt], z[1] * back[rt], z[2] * back[rt], z[3] * back[rt]};
        }
      // V's columns as operands; the next block's rows are sent for
      u4 A[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = j < 2 ? __builtin_amdgcn_perm(vw[2 * k + 1].x, vw[2 * k].x, sel)
                       : __builtin_amdgcn_perm(vw[2 * k + 1].y, vw[2 * k].y, sel);
        A[j] = u4{w[0], w[1], w[2], w[3]};
      }
      const int now_valid = valid;
      if (more) {
        blk = block_of(a, t, table, h, t.block(i + 1), 2 * kD);
        valid = blk.valid;
        load_k(blk);
        load_v(blk);
      }
      lds_barrier();
      const bool all = (now_valid == kBlk) & (t.rows == kRows) & all_seen(a, t.p0, t.p1, j0);
      const auto raise = [&](int rt, float (&c)[8], float &alpha) {
#pragma unroll
        for (int w = 0; w < kW; ++w)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float4 f = *reinterpret_cast<const float4 *>(&all_sc[w][16 * rt + n][8 * g + 4 * y]);
            c[4 * y] = w ? c[4 * y] + f.x : f.x;
            c[4 * y + 1] = w ? c[4 * y + 1] + f.y : f.y;
            c[4 * y + 2] = w ? c[4 * y + 2] + f.z : f.z;
            c[4 * y + 3] = w ? c[4 * y + 3] + f.w : f.w;
          }
        return row[rt].raise(c, 1.0f, all, [&] { return seen_of(a, pos[rt], j0 + 8 * g, now_valid - 8 * g); }, alpha);
      };
      const auto rescale = [&](int rt, float alpha) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[rt][j][e] *= alpha;
      };
      const auto add = [&](int rt, const u4 (&pb)[kP]) {
#pragma unroll
        for (int p = kP - 1; p >= 0; --p)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[rt][j] = half_mfma<kBf>(A[j], pb[p], acc[rt][j]);
      };
      if constexpr (kOwn) {
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt) {
          if (rt % kW != wave) continue;
          u4 pb[kP];
          float c[8], alpha = 1.0f;
          raise(rt, c, alpha);
          row[rt].weights(c, 1.0f, pb);
#pragma unroll
          for (int p = 0; p < kP; ++p) s_weights[rt][p][lane] = pb[p];
          if (g == 0) s_alpha[rt][n] = alpha;
        }
        lds_barrier();  // (the next scores are written behind it, the next weights behind the barrier after)
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt) {
          u4 pb[kP];
#pragma unroll
          for (int p = 0; p < kP; ++p) pb[p] = s_weights[rt][p][lane];
          const float alpha = s_alpha[rt][n];
          if (__any(alpha != 1.0f)) rescale(rt, alpha);
          add(rt, pb);
        }
      } else {
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt) {
          float c[8], alpha = 1.0f;
          if (raise(rt, c, alpha)) rescale(rt, alpha);
          u4 pb[kP];
          row[rt].weights(c, 1.0f, pb);
          add(rt, pb);
        }
      }
    }
    // ---- the piece's rows
    float l[kRT];
    bool bad = false;
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
      if (!kOwn || rt % kW == wave) {
        l[rt] = row[rt].sum();
        bad |= !(l[rt] < INFINITY);
        if (kOwn && g == 0) s_l[rt][n] = l[rt];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[rt][j][e] *= 1.0f / Row<kBf>::kUp;
          bad |= !(fabsf(acc[rt][j][e]) < INFINITY);
        }
    }
    if (bad) s_bad = 1u;
    __syncthreads();
    const bool redo = s_bad != 0u;
    __syncthreads();
    if (redo) {
      for (int y = wave; y < t.rows; y += kW) plain_store<kBf, kW>(a, t, h, y, i0, i1, lane, to, kRows);
      if (tid == 0) s_bad = 0u;
    } else {
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt) {
        const int y = 16 * rt + n;
        if (y >= t.rows) continue;
        if (kOwn) l[rt] = s_l[rt][n];
        const int64_t at = to.slot * kRows + y;
        float *o = (to.whole ? row_out(a, t, h, y, kD) : a.part + at * kD) + 64 * wave + 16 * g;
        const float f = l[rt] > 0.0f ? 1.0f / l[rt] : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          reinterpret_cast<float4 *>(o)[e] = float4{acc[rt][0][e] * f, acc[rt][1][e] * f, acc[rt][2][e] * f, acc[rt][3][e] * f};
        if (!to.whole && wave == (kOwn ? rt % kW : 0) && g == 0) a.ml[at] = float2{row[rt].m, l[rt]};
      }
    }
  }
}

// ---- tiles of 16 kW rows, 16 a wave, for prompts.
// Measured (MI355X, a call less its plan and join; 16 query heads over 2 KV heads of 256): 512 new tokens
// over 16896 BF16 keys 320 us, 1.31 PFLOP/s of products in three parts (a library product of 8192^3 in
// BF16: 1.14); 8001 tokens of F16 in a window of 1024 behind 4 first keys 260 us, 0.84 PFLOP/s of the keys
// seen in two parts. Bound, by copies of this kernel that leave a part out: no one part. Of the BF16
// chunk's time the softmax is 10%, the reads of LDS 16, the loads into it 5, and products, barriers and
// the tiles' starts what is left; a block takes 2.0 us in F16, 0.9 of them the products at the matrix
// cores' full rate. A tile's start and end (queries, first blocks, rows of out) take 13 us with nothing
// beside them, one workgroup a CU: a quarter of the 8001 tokens in a window, whose softmax is 5% and loads
// 7. Of head_dim 128 and 64 the softmax is 18 and 28%. 16 rows a wave: 32, with half the reads of LDS, need
// more than 256 registers beside the sums of 256 columns (one wave a SIMD: three times as long), and
// where they fit (head_dim 128) gain 4% in F16 and nothing in BF16.
// Blocks' rows of K and V go from memory into LDS ahead of their use; every wave runs its rows from there:
//   scores (transposed, A = K) with keys in the order of few_kernel; out (transposed, A = V): V's
//   columns come by transposing reads; the result is columns 16 c + 4 g + i of row n.
// Pieces of 16 bytes of a row are turned by the row, so that the 16 rows which a quarter of a wave
// reads at once lie on different banks; V's by 32 bytes, for the 8 rows of a transposing read.
template <int kD>
__device__ __forceinline__ int k_piece(int key, int c) {
  const int r = ((key >> 3) << 2) | (key & 3);
  if constexpr (kD == 64) return c ^ ((r >> 1) & 7);
  else return c ^ r;
}
template <int kD>
__device__ __forceinline__ int v_piece(int key, int c) {
  if constexpr (kD == 64) return c ^ ((((key >> 1) & 1) | ((key >> 3 & 1) << 1)) << 1);
  else return c ^ (((key & 3) | ((key >> 3 & 1) << 2)) << 1);
}
__device__ __forceinline__ uint2 load_columns(const uint16_t *p) {
  typedef __fp16 v4h __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4h lds_v4h;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_v4h *)(p)));
}

// One load of 16 bytes a lane from r + off into LDS from byte `at` (wave-uniform) on, in the lanes'
// order. In asm, since the compiler would wait for it in front of every later read of LDS: the
// kernel waits itself (fetched) before the barrier behind which the data is read.
__device__ __forceinline__ void fetch_rows(uint32_t at, uint32_t off, u4s r) {
  const uint32_t m = __builtin_amdgcn_readfirstlane(at);
  uint32_t saved;
  asm volatile(
      "s_nop 4\n\t"  // SGPRs written by vector instructions: 5 wait states before the load reads them
      "s_mov_b32 %[sv], m0\n\t"
      "s_mov_b32 m0, %[m]\n\ts_nop 0\n\t"
      "buffer_load_dwordx4 %[o], %[r], 0 offen lds\n\t"
      "s_mov_b32 m0, %[sv]"
      : [sv] "=&s"(saved)
      : [m] "s"(m), [o] "v"(off), [r] "s"(r)
      : "memory");
}
// All but the newest `kLeft` loads of this wave have landed.
template <int kLeft>
__device__ __forceinline__ void fetched() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLeft) : "memory");
}
// The lane, from the hardware again rather than from a register.
__device__ __forceinline__ int this_lane() {
  int ones = -1;
  asm volatile("" : "+v"(ones));
  return __builtin_amdgcn_mbcnt_hi(ones, __builtin_amdgcn_mbcnt_lo(ones, 0));
}
// Vector and scalar arithmetic may move across, reads of LDS and matrix products may not.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0x406); }

template <bool kBf, int kD, int kW>
__global__ __launch_bounds__(64 * kW, kD == 256 ? 2 : kD == 128 ? 3 : 4) void many_kernel(AttendArgs a) {
  constexpr int kThreads = 64 * kW, kRows = 16 * kW, kSteps = kD / 32, kCols = kD / 16, kP = kParts<kBf>;
  constexpr int kMoves = 4 * kD / kThreads;  // 16-byte pieces of K, and of V, that a thread moves
  // Blocks of K and of V in LDS. Four: two between barriers, the two behind them on their way. Rows
  // of 256 bytes take three, one and one or two, so that three workgroups fit a CU's LDS (8001 tokens in a
  // window, 32 heads of 128: with four 31% longer; of 256, 16 heads: one by one 4% longer than by pairs),
  // and BF16 rows of 512 bytes, whose registers a pair's second block exceeds (512 tokens over 16896
  // keys: by pairs 1% longer).
  constexpr bool kPairs = kD == 64 || (kD == 256 && !kBf);
  constexpr int kRing = kPairs ? 4 : 3;
  __shared__ __attribute__((aligned(1024))) uint16_t lk[kRing][kBlk * kD], lv[kRing][kBlk * kD];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Plan<false> plan;
  Plan<false>::Lds none;
  plan.make(a, none, kRows, kThreads);
  const Line line = plan.line;
  zero_empty(a, plan, kD, kThreads);
  // neighbouring shares read the same keys: they go to the same XCD (workgroups go to the 8 in turn)
  const int per_xcd = (line.shares + 7) / 8, share = ((int)blockIdx.x % 8) * per_xcd + (int)blockIdx.x / 8;
  if ((int)blockIdx.x / 8 >= per_xcd || share >= line.shares) return;
  int64_t u = line.start(share);
  const int64_t u0 = u, end = line.start(share + 1);
  const uint32_t stride = (uint32_t)a.kv_heads * 2u * kD;
  const int row0 = 16 * wave;  // the wave's first row of a tile
  // where the pieces that the thread moves come from: of a key's row the one that belongs where it lands
  uint32_t koff[kMoves], voff[kMoves];
#pragma unroll
  for (int j = 0; j < kMoves; ++j) {
    const int p = j * kThreads + tid, key = p / (kD / 8), c = p % (kD / 8);
    koff[j] = (uint32_t)key * stride + 16u * (uint32_t)k_piece<kD>(key, c);
    voff[j] = (uint32_t)key * stride + 16u * (uint32_t)v_piece<kD>(key, c);
  }
  // Where the lane reads: K's pieces 4 st + g of key 8 (n / 4) + n % 4 (the other keys are four rows on),
  // V's row n / 4 of keys 8 g .. + 3 in tile cc of 16 columns (keys + 4 four rows on). Pieces are turned
  // by an exclusive or of their low bits, so four steps and eight tiles on the place is 256 bytes on.
  // BF16 rows of 512 bytes leave no registers for twelve places: they are worked out again in each
  // block from the lane's two. (What the compiler puts into scratch memory instead comes back
  // behind the loads of LDS: 8001 tokens 2.5 times as long. Fifteen values still lie there, of which a
  // block with masks reads two and one block in three another.)
  constexpr bool kAgain = kBf && kD == 256;
  constexpr int kK = kAgain ? 1 : kSteps < 4 ? kSteps : 4, kV = kAgain ? 1 : kCols < 8 ? kCols : 8;
  const auto k_place = [](int st) {
    const int ln = kAgain ? this_lane() : (int)(threadIdx.x & 63), m = ln & 15, key = 8 * (m >> 2) + (m & 3);
    return key * kD + 8 * k_piece<kD>(key, 4 * st + (ln >> 4));
  };
  const auto v_place = [](int cc) {
    const int ln = kAgain ? this_lane() : (int)(threadIdx.x & 63), m = ln & 15, key = 8 * (ln >> 4) + (m >> 2);
    return key * kD + 8 * v_piece<kD>(key, 2 * cc + ((m & 3) >> 1)) + 4 * (m & 1);
  };
  int k_held[kK], v_held[kV];
  if constexpr (!kAgain) {
#pragma unroll
    for (int st = 0; st < kK; ++st) k_held[st] = k_place(st);
#pragma unroll
    for (int cc = 0; cc < kV; ++cc) v_held[cc] = v_place(cc);
  }
  int x = plan.first(a, share), h = line.head(u);
  for (; u < end; ++x) {
    if (x == line.tiles) x = 0, ++h;
    const Tile t = plan.tile(a, x);
    if (t.blocks == 0) continue;
    const int64_t tile0 = h * line.per_head + plan.before(a, x), behind = tile0 + t.units(a.start);
    const Sink to = {u <= tile0 + a.start && end >= behind, 2 * (int64_t)share + (u > u0 ? 1 : 0)};
    const int i0 = u <= tile0 + a.start ? 0 : (int)(u - tile0) - a.start;
    const int i1 = end >= behind ? t.blocks : (int)(end - tile0) - a.start;
    u = behind;
    if (i1 <= i0) continue;  // the share ends within the tile's start

    // a block's rows into LDS; rows behind its valid ones are the last one again (never seen)
    const auto fetch = [&](const uint8_t *plane, const Block &b, const uint32_t (&off)[kMoves], uint16_t *to_lds) {
      const u4s r = make_rsrc(plane + b.at, b.span);
      const uint32_t base = (uint32_t)(size_t)((PKV_LDS void *)to_lds) + 1024u * (uint32_t)wave;
      uint32_t o[kMoves];
#pragma unroll
      for (int j = 0; j < kMoves; ++j) o[j] = off[j];
      if (b.valid < kBlk) {
#pragma unroll
        for (int j = 0; j < kMoves; ++j) {
          const int over = (j * kThreads + tid) / (kD / 8) - (b.valid > 0 ? b.valid - 1 : 0);
          o[j] -= over > 0 ? (uint32_t)over * stride : 0u;
        }
      }
#pragma unroll
      for (int j = 0; j < kMoves; ++j) fetch_rows(base + 1024u * kW * (uint32_t)j, o[j], r);
    };
    Table table;
    table.look_at(a, t.b, (t.block(i0) << 5) >> a.page_lg);
    const int y = row0 + n;
    const bool mine = y < t.rows;
    const int r = t.row0 + (mine ? y : 0), tok = r / a.group, pos = mine ? t.first + tok : -1;
    const float *q = a.q + (int64_t)(t.tok0 + tok) * a.q_t + (int64_t)(h * a.group + r % a.group) * a.q_h + 8 * g;
    Queries<kBf, kSteps> qs;
    qs.load(q);
    // (behind the piece's end: the last block again, which nobody looks at)
    const auto block = [&](int i) { return block_of(a, t, table, h, t.block(i < i1 ? i : i1 - 1), 2 * kD); };
    lds_barrier();  // what was sent for behind the last piece's end has landed
    Block b0 = block(i0), b1 = block(i0 + 1);
    fetch(a.k, b0, koff, lk[0]);
    fetch(a.v, b0, voff, lv[0]);
    fetch(a.k, b1, koff, lk[1]);
    fetch(a.v, b1, voff, lv[1]);

    u4 qb[kSteps][kP];
    float back;
    qs.split(q, mine, a.sl2, qb, back);
    // the wave's rows' positions
    const int w1 = t.rows < row0 + 16 ? t.rows : row0 + 16;  // behind its last row
    const bool some = row0 < w1, full = w1 == row0 + 16;
    const int wp0 = some ? t.first + (t.row0 + row0) / a.group : -1;
    const int wp1 = some ? t.first + (t.row0 + w1 - 1) / a.group : -1;
    __builtin_amdgcn_sched_barrier(0);  // (the sums take the registers that the queries came through)
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 acc[kCols];
    Row<kBf> row;
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[c] = zero;
    f4 sc[2];
    // operands come from LDS kAhead reads ahead of the products that take them (two: 512 tokens over
    // 16896 BF16 keys 6% longer; six and eight: the same within 1%)
    constexpr int kAhead = 4;
    const auto scores = [&](const uint16_t *kb) {
      constexpr int kReads = 2 * kSteps;
      const int own = kAgain ? k_place(0) : 0;
      const auto read = [&](int i) {
        const int st = i >> 1, at = kAgain ? own ^ (32 * st) : k_held[st % kK] + st / kK * 128;
        return *reinterpret_cast<const u4 *>(kb + at + (i & 1) * 4 * kD);
      };
      u4 A[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) A[i] = read(i);
      keep_order();
      sc[0] = sc[1] = zero;
#pragma unroll
      for (int i = 0; i < kReads; i += 2) {  // (both key tiles in turn: a sum waits for its last product)
#pragma unroll
        for (int p = kP - 1; p >= 0; --p)
#pragma unroll
          for (int z = 0; z < 2; ++z) sc[z] = half_mfma<kBf>(A[(i + z) % kAhead], qb[i >> 1][p], sc[z]);
        keep_order();
#pragma unroll
        for (int z = 0; z < 2; ++z)
          if (i + z + kAhead < kReads) A[(i + z) % kAhead] = read(i + z + kAhead);
        keep_order();
      }
    };

    fetched<kPairs ? 0 : 2 * kMoves>();  // the first blocks, or the first
    lds_barrier();
    const auto step = [&](int i, int valid, auto slot) {
      constexpr int at = decltype(slot)::value;
      const int j0 = t.block(i) << 5;
      scores(lk[at]);
      float c[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = sc[e >> 2][e & 3];
      const bool all = (valid == kBlk) & full & all_seen(a, wp0, wp1, j0);
      float alpha = 1.0f;
      if (row.raise(c, back, all, [&] { return seen_of(a, pos, j0 + 8 * g, valid - 8 * g); }, alpha))
#pragma unroll
        for (int cc = 0; cc < kCols; ++cc)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[cc][e] *= alpha;
      u4 pb[kP];
      row.weights(c, back, pb);
      // lane n of each 16: four values of row n / 4 of keys 8 g .. + 3, then of + 4 .. + 7
      const int own = kAgain ? v_place(0) : 0;
      const auto read = [&](int cc) {
        const uint16_t *vp = lv[at] + (kAgain ? own ^ (16 * cc) : v_held[cc % kV] + cc / kV * 128);
        const uint2 lo = load_columns(vp), hi = load_columns(vp + 4 * kD);
        return u4{lo.x, lo.y, hi.x, hi.y};
      };
      u4 A[kAhead];
#pragma unroll
      for (int cc = 0; cc < kAhead; ++cc) A[cc] = read(cc);
      keep_order();
#pragma unroll
      for (int cc = 0; cc < kCols; cc += 2) {
#pragma unroll
        for (int p = kP - 1; p >= 0; --p)
#pragma unroll
          for (int z = 0; z < 2; ++z) acc[cc + z] = half_mfma<kBf>(A[(cc + z) % kAhead], pb[p], acc[cc + z]);
        keep_order();
#pragma unroll
        for (int z = 0; z < 2; ++z)
          if (cc + z + kAhead < kCols) A[(cc + z) % kAhead] = read(cc + z + kAhead);
        keep_order();
      }
    };
    if constexpr (kPairs) {
      const auto pair = [&](int i, auto which) {
        constexpr int at = 2 * decltype(which)::value, other = 2 - at;
        const Block b2 = block(i + 2), b3 = block(i + 3);
        fetch(a.k, b2, koff, lk[other]);
        fetch(a.v, b2, voff, lv[other]);
        fetch(a.k, b3, koff, lk[other + 1]);
        fetch(a.v, b3, voff, lv[other + 1]);
        step(i, b0.valid, std::integral_constant<int, at>{});
        if (i + 1 < i1) step(i + 1, b1.valid, std::integral_constant<int, at + 1>{});
        fetched<0>();
        lds_barrier();
        b0 = b2;
        b1 = b3;
      };
      for (int i = i0; i < i1; i += 4) {
        pair(i, std::integral_constant<int, 0>{});
        if (i + 2 < i1) pair(i + 2, std::integral_constant<int, 1>{});
      }
    } else {
      const auto one = [&](int i, auto which) {
        constexpr int at = decltype(which)::value, other = (at + 2) % 3;
        const Block b2 = block(i + 2);
        fetch(a.k, b2, koff, lk[other]);
        fetch(a.v, b2, voff, lv[other]);
        step(i, b0.valid, std::integral_constant<int, at>{});
        fetched<2 * kMoves>();  // all but what was just sent for
        lds_barrier();
        b0 = b1;
        b1 = b2;
      };
      for (int i = i0; i < i1; i += 3) {
        one(i, std::integral_constant<int, 0>{});
        if (i + 1 < i1) one(i + 1, std::integral_constant<int, 1>{});
        if (i + 2 < i1) one(i + 2, std::integral_constant<int, 2>{});
      }
    }
    fetched<0>();  // (what was sent for behind the end lands before LDS is used again)
    const float l = row.sum();
    bool bad = !(l < INFINITY);
#pragma unroll
    for (int cc = 0; cc < kCols; ++cc)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[cc][e] *= 1.0f / Row<kBf>::kUp;
        bad |= !(fabsf(acc[cc][e]) < INFINITY);
      }
    if (__any(bad)) {
      for (int z = row0; z < w1; ++z) plain_store<kBf, kD / 64>(a, t, h, z, i0, i1, lane, to, kRows);
    } else if (mine) {
      const int64_t at = to.slot * kRows + y;
      float *o = (to.whole ? row_out(a, t, h, y, kD) : a.part + at * kD) + 4 * g;
      const float f = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
      for (int cc = 0; cc < kCols; ++cc)
        *reinterpret_cast<float4 *>(o + 16 * cc) = float4{acc[cc][0] * f, acc[cc][1] * f, acc[cc][2] * f, acc[cc][3] * f};
      if (!to.whole && g == 0) a.ml[at] = float2{row.m, l};
    }
  }
}

// ---- the parts of a tile that was cut, joined (5 us where one token's 1025 keys lie in 64 parts, 7 for 24
// requests, 8 for 131073 keys in 512 parts, 24 behind 8001 prompt tokens: 53 MB read, 26 written). Bound: two
// trips to memory and a launch, or the parts' bytes. A wave a row, or kAcross waves a row of a tile
// of many parts. The parts' maxima and sums come side by side, a lane a part; then their rows, four
// in flight. By tile where there are fewer tiles than cuts, else by cut: the first cut inside a
// tile joins it.
template <int kE>
__device__ __forceinline__ void load_elems(const float *p, float (&x)[kE]) {
  if constexpr (kE == 4) {
    const float4 f = *reinterpret_cast<const float4 *>(p);
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
  } else if constexpr (kE == 2) {
    const float2 f = *reinterpret_cast<const float2 *>(p);
    x[0] = f.x, x[1] = f.y;
  } else {
    x[0] = *p;
  }
}
// Parts [i0, i1) of a row, their mean: slot(i) is where part i's row is.
template <int kE, typename Slot>
__device__ __forceinline__ void join_parts(const AttendArgs &a, Slot slot, int i0, int i1, int lane, float &m, float &l,
                                           float (&acc)[kE]) {
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int e = 0; e < kE; ++e) acc[e] = 0.0f;
  for (int b = i0; b < i1; b += 64) {
    const int count = i1 - b < 64 ? i1 - b : 64;
    const float2 ml = lane < count ? a.ml[slot(b + lane)] : float2{-INFINITY, 0.0f};
    float x[4][kE];
    const auto load = [&](int i) {
#pragma unroll
      for (int y = 0; y < 4; ++y)
        load_elems<kE>(a.part + slot(b + (i + y < count ? i + y : count - 1)) * (64 * kE) + lane * kE, x[y]);
    };
    load(0);
    float top = xmax32(xmax16(ml.x));
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (top == -INFINITY) continue;
    const float mn = fmaxf(m, top), c = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    const float before = l * c, own = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mn) * ml.y;
    // (a part that saw nothing wrote zeros: a weight of 0 takes it out)
    l = before + wave_sum(own);
    const float by = 1.0f / l, w = own * by;
#pragma unroll
    for (int e = 0; e < kE; ++e) acc[e] *= before * by;
    m = mn;
    for (int i = 0; i < count; i += 4) {
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if (i + y >= count) break;  // (the last part again, which may hold infinities)
        const float f = __shfl(w, i + y);
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[e] += f * x[y][e];
      }
      if (i + 4 < count) load(i + 4);
    }
  }
}

template <int kD, int kAcross>
__global__ __launch_bounds__(kAcross > 1 ? 64 * kAcross : 256) void join_kernel(AttendArgs a, int rows_per_tile, int by_cut) {
  constexpr int kE = kD / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Line line = line_of(a);
  // (what the plan says of the tile is asked for together, whether there is such a tile or not)
  const int cut = (int)blockIdx.x + 1;
  if (by_cut && cut >= line.shares) return;
  const int x = by_cut ? a.firsts[cut] : (int)blockIdx.x / a.kv_heads;
  const int64_t before = a.before[x], behind = a.before[x + 1];
  const Tile t = a.tiles[x];
  int h, w0;  // w0: the share that holds the tile's first block
  if (by_cut) {
    const int64_t u = line.start(cut);
    h = line.head(u);
    const int64_t first = h * line.per_head + before + a.start;
    if (u <= first || (cut > 1 && line.start(cut - 1) > first)) return;
    w0 = cut - 1;
  } else {
    h = (int)blockIdx.x % a.kv_heads;
    if (x >= line.tiles || behind == before) return;
    w0 = line.share(h * line.per_head + before + a.start);
  }
  const int64_t tile0 = h * line.per_head + before, last = h * line.per_head + behind;
  if (line.start(w0 + 1) >= last) return;  // not cut
  const int pieces = line.share(last - 1) - w0 + 1, odd = line.start(w0) < tile0 ? 1 : 0;
  const int row = kAcross > 1 ? (int)blockIdx.y : (int)blockIdx.y * 4 + wave;
  if (row >= t.rows) return;
  const auto slot = [&](int i) { return (2 * (int64_t)(w0 + i) + (i == 0 ? odd : 0)) * rows_per_tile + row; };
  float m, l, acc[kE];
  if constexpr (kAcross == 1) {
    join_parts<kE>(a, slot, 0, pieces, lane, m, l, acc);
    float *o = row_out(a, t, h, row, kD) + lane * kE;
#pragma unroll
    for (int e = 0; e < kE; ++e) o[e] = acc[e];
  } else {
    __shared__ float part[kAcross][kD], s_m[kAcross], s_l[kAcross];
    const int per = (pieces + kAcross - 1) / kAcross;
    const int i0 = wave * per < pieces ? wave * per : pieces, i1 = i0 + per < pieces ? i0 + per : pieces;
    join_parts<kE>(a, slot, i0, i1, lane, m, l, acc);
#pragma unroll
    for (int e = 0; e < kE; ++e) part[wave][lane * kE + e] = acc[e];
    if (lane == 0) {
      s_m[wave] = m;
      s_l[wave] = l;
    }
    __syncthreads();
    if (threadIdx.x >= kD) return;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kAcross; ++i) top = fmaxf(top, s_m[i]);
    float w[kAcross], all = 0.0f, mean = 0.0f;
#pragma unroll
    for (int i = 0; i < kAcross; ++i) {
      w[i] = s_m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[i] - top) * s_l[i];
      all += w[i];
    }
    const float by = top == -INFINITY ? 0.0f : 1.0f / all;
#pragma unroll
    for (int i = 0; i < kAcross; ++i) mean += part[i][threadIdx.x] * (w[i] * by);
    row_out(a, t, h, row, kD)[threadIdx.x] = mean;
  }
}

// Rows a tile holds, the workgroups that share the blocks (as many as the chip runs at once), and how
// many blocks a tile's start costs: 2 of a few rows, 6 of a prompt's (start, queries, first loads and
// stores take 13 us, a block 2; 4 and 8 made 8001 tokens in a window 3% slower).
// Tiles of few rows for requests of up to 48 rows on average: 80 drafted tokens of 40 rows each
// take 38 us in tiles of 48 and 53 in the prompts' tiles. The average is the step's, its rows of no request
// among them, since lengths are not known here: one token of 65536 keys in a step of 9 rows or more takes
// 67 us instead of 36, a chunk of 512 tokens over 4608 keys beside 23 tokens 184, in two calls 169.
// Three waves a SIMD hold 16 rows of head_dim 64 and 128 (24 requests of 64: a quarter less than by two),
// two anything else.
struct Shape {
  int rows, shares, start;
  bool prompts() const { return start == 6; }
};
constexpr int kFewRows[] = {16, 32, 48};
Shape few_shape(int rows, int head_dim) {
  return Shape{rows, (rows == 16 && head_dim < 256 ? 768 : 512) * 256 / head_dim, 2};
}
Shape prompt_shape(int head_dim) {
  return head_dim == 64 ? Shape{64, 1024, 6} : head_dim == 128 ? Shape{64, 768, 6} : Shape{128, 256, 6};
}
// rows: of the whole step, tokens x query heads of a KV head
Shape shape_of(int n, int64_t rows, int head_dim) {
  for (const int r : kFewRows)
    if (rows <= r * (int64_t)n) return few_shape(r, head_dim);
  return prompt_shape(head_dim);
}
struct Layout {
  size_t tiles, before, firsts, count, ml, part, all;
  int max_tiles;
};
Layout layout_of(const Shape &sh, int n, int64_t rows, int head_dim) {
  Layout l;
  const auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  l.max_tiles = (int)(n + rows / sh.rows);
  l.tiles = 0;
  l.before = up((size_t)l.max_tiles * sizeof(Tile));
  l.firsts = l.before + up(((size_t)l.max_tiles + 1) * sizeof(int64_t));
  l.count = l.firsts + up((size_t)sh.shares * sizeof(int));
  l.ml = l.count + 256;
  l.part = l.ml + up((size_t)2 * sh.shares * sh.rows * sizeof(float2));
  l.all = l.part + (size_t)2 * sh.shares * sh.rows * head_dim * sizeof(float);
  return l;
}

template <int kD>
void join(AttendArgs &a, const Shape &sh, hipStream_t s) {
  const int64_t tiles = (int64_t)a.max_tiles * a.kv_heads;
  const int by_cut = tiles > sh.shares;
  const unsigned x = by_cut ? (unsigned)sh.shares : (unsigned)tiles;
  // by the parts a tile has on average, waves a row. What the others cost: 131073 keys in 256 parts a tile
  // (16) 15 us more with four, 79 with one; 8 requests of 3000 keys (32 parts, 16) 5 and 26; 80 drafted
  // tokens (9 parts, four) 9 us more with 16, 5 with one; 8001 prompt tokens (one or two parts, one) 226
  // with 16, 50 with four
  if (tiles * 16 <= sh.shares)
    hipLaunchKernelGGL((join_kernel<kD, 16>), dim3(x, sh.rows), dim3(1024), 0, s, a, sh.rows, by_cut);
  else if (tiles * 4 <= sh.shares)
    hipLaunchKernelGGL((join_kernel<kD, 4>), dim3(x, sh.rows), dim3(256), 0, s, a, sh.rows, by_cut);
  else
    hipLaunchKernelGGL((join_kernel<kD, 1>), dim3(x, sh.rows / 4), dim3(256), 0, s, a, sh.rows, by_cut);
}
template <bool kBf, int kD, bool kHere>
void few(AttendArgs &a, const Shape &sh, hipStream_t s) {
  const dim3 grid(sh.shares), block(kD);
  if (sh.rows == 16) hipLaunchKernelGGL((few_kernel<kBf, kD, 1, kHere>), grid, block, 0, s, a);
  else if (sh.rows == 32) hipLaunchKernelGGL((few_kernel<kBf, kD, 2, kHere>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((few_kernel<kBf, kD, 3, kHere>), grid, block, 0, s, a);
  join<kD>(a, sh, s);
}
template <bool kBf, int kD>
int go(AttendArgs &a, const Shape &sh, hipStream_t s) {
  // a head's units at most, as 32-bit sums of the workgroup's own plan
  const int64_t most = (int64_t)a.max_tiles * ((((int64_t)a.max_pages << a.page_lg) >> 5) + sh.start + 1);
  if (!sh.prompts() && a.n <= 64 && a.max_tiles <= kHereTiles && most < ((int64_t)1 << 31)) {
    few<kBf, kD, true>(a, sh, s);
  } else {
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, sh.rows);
    if (!sh.prompts()) {
      few<kBf, kD, false>(a, sh, s);
    } else {
      hipLaunchKernelGGL((many_kernel<kBf, kD, (kD > 128 ? 8 : 4)>), dim3(sh.shares), dim3(kD > 128 ? 512 : 256), 0, s, a);
      join<kD>(a, sh, s);
    }
  }
  PKV_HIP(hipGetLastError());
  return PKV_OK;
}

}  // namespace

// What any step of up to n requests and `tokens` tokens needs, so that a buffer for the largest step holds
// the smaller ones: tiles of fewer rows have more shares and may need more (head_dim 64, 24 requests, 8
// heads of a KV head: 52 MB for 144 tokens, 35 for 8192).
size_t pages_attend_workspace(int n, int64_t tokens, int heads, int kv_heads, int head_dim) {
  const int64_t rows = tokens * (heads / kv_heads);
  size_t most = 0;
  int64_t below = 0;  // one request of more rows takes the shape at hand, or a later one
  for (const int r : kFewRows) {
    const int64_t own = rows < r * (int64_t)n ? rows : r * (int64_t)n;  // as many as it is for
    if (rows > below) most = std::max(most, layout_of(few_shape(r, head_dim), n, own, head_dim).all);
    below = r;
  }
  return rows > below ? std::max(most, layout_of(prompt_shape(head_dim), n, rows, head_dim).all) : most;
}

int launch_pages_attend(const PagesAttend &p, void *ws, hipStream_t s) {
  const int group = p.heads / p.kv_heads;
  const Shape sh = shape_of(p.n, p.tokens * group, p.head_dim);
  const Layout l = layout_of(sh, p.n, p.tokens * group, p.head_dim);
  uint8_t *w = static_cast<uint8_t *>(ws);
  AttendArgs a;
  a.q = p.q;
  a.q_t = p.q_t;
  a.q_h = p.q_h;
  a.k = static_cast<const uint8_t *>(p.k_pages);
  a.v = static_cast<const uint8_t *>(p.v_pages);
  a.page_bytes = (int64_t)p.page_tokens * p.kv_heads * p.head_dim * 2;
  a.tables = p.tables;
  a.lens = p.lens;
  a.starts = p.starts;
  a.out = p.out;
  a.tiles = reinterpret_cast<Tile *>(w + l.tiles);
  a.before = reinterpret_cast<int64_t *>(w + l.before);
  a.firsts = reinterpret_cast<int *>(w + l.firsts);
  a.count = reinterpret_cast<Count *>(w + l.count);
  a.ml = reinterpret_cast<float2 *>(w + l.ml);
  a.part = reinterpret_cast<float *>(w + l.part);
  a.n = p.n;
  a.tokens = (int)p.tokens;
  a.heads = p.heads;
  a.kv_heads = p.kv_heads;
  a.group = group;
  a.page_lg = __builtin_ctz((unsigned)p.page_tokens);
  a.n_pages = p.n_pages;
  a.max_pages = p.max_pages;
  a.window = p.window;
  a.sinks = p.sinks;
  a.max_tiles = l.max_tiles;
  a.shares = sh.shares;
  a.start = sh.start;
  a.sl2 = p.scale * kLog2e;
  if (const int rc = device_status_word(&a.status)) return rc;
  const bool bf = p.quant == PKV_QUANT_BF16;
  if (p.head_dim == 64) return bf ? go<true, 64>(a, sh, s) : go<false, 64>(a, sh, s);
  if (p.head_dim == 128) return bf ? go<true, 128>(a, sh, s) : go<false, 128>(a, sh, s);
  return bf ? go<true, 256>(a, sh, s) : go<false, 256>(a, sh, s);
}

}  // namespace pkv
