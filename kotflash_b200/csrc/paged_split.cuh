// What the paged decode kernels share (16-bit and 8-bit pools): the list of
// tiles and its split over the blocks, the partials of units that were cut, and
// their join.
#pragma once
#include <math.h>

#include "kf_host.h"
#include "kf_sm100.cuh"

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kBlocksPerSm = 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// What both kernels and the join need to know of a call.
struct PagedWork {
  uint16_t* o;             // [B][Hq][D]
  float* lse;              // may be null
  const int32_t* table;
  const int32_t* lengths;
  float* part_o;           // [blocks][2][rows of a unit][D]
  float* part_lse;         // [blocks][2][rows of a unit], log2
  int4* joins;             // by unit if join_units, else by block: (request, KV head and row block, first
                           // block, last block) of a unit that was cut, or x = -1
  int32_t* status;         // set when a bounded wait expires (may be null)
  int64_t table_stride;
  int B, Hq, Hkv, G, D, row_blocks;
  uint32_t max_pages;
  uint32_t capacity;       // tokens a table row can hold
  uint32_t page_size, num_pages;
  uint32_t page_mul, page_shift;  // x / page_size = x page_mul >> page_shift for x < 2^31
  bool join_units;
};

__device__ __forceinline__ uint32_t visible(const PagedWork& a, int b) {
  const int32_t n = a.lengths[b];
  return n <= 0 ? 0u : min((uint32_t)n, a.capacity);
}

// A tile and its position in the list: tile `t` of the `tiles` of the unit
// (request b, KV head h, row block rb).  A unit takes tiles + 1 positions: its
// end (joining the teams, writing, the next unit's Q) costs about what a tile
// does, 1.0 us where a tile takes 1.4, so a position counts as much.
template <int TILE>
struct Cursor {
  int b, h, rb;
  uint32_t t, tiles, keys, pos;
  bool whole;  // the table holds all of the request's positions

  __device__ __forceinline__ void set_request(const PagedWork& a, int request) { set_request(a, request, a.lengths[request]); }
  __device__ __forceinline__ void set_request(const PagedWork& a, int request, int32_t length) {
    b = request;
    whole = length <= 0 || (uint32_t)length <= a.capacity;
    keys = length <= 0 ? 0u : min((uint32_t)length, a.capacity);
    tiles = (keys + TILE - 1) / TILE;
  }
  __device__ __forceinline__ bool unit_ends() const { return t + 1 == tiles; }
  // whether another tile follows before position `end`
  __device__ __forceinline__ bool more(uint32_t end) const { return pos + (unit_ends() ? 2 : 1) < end; }
  // to that tile
  __device__ __forceinline__ void next(const PagedWork& a) {
    ++pos;
    if (++t < tiles) return;
    ++pos;
    t = 0;
    if (++rb < a.row_blocks) return;
    rb = 0;
    if (++h < a.Hkv) return;
    h = 0;
    do {
      set_request(a, b + 1);
    } while (tiles == 0 && b + 1 < a.B);
  }
};

// A block's share of the list of tiles: positions [begin, end), the first of
// them in the units of request `first`, whose units begin at position
// `before` * units.  `total`: positions of all requests, per unit.
struct Share {
  uint32_t begin, end, even, longer, total, before;
  int first;
  int32_t length;                      // of request `first`
};
struct ShareScratch {  // shared memory
  uint32_t warp_tiles[kWarps];
  int first;
  uint32_t before;
  int32_t length;
};

// By a prefix sum over the requests' lengths (fewer than 2^31 positions, see
// the host's check).  False where there are more blocks than positions.
template <int TILE>
__device__ __forceinline__ bool find_share(const PagedWork& a, ShareScratch& scratch, Share& s) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int units = a.Hkv * a.row_blocks;  // per request
  const int per = (a.B + kThreads - 1) / kThreads;  // requests per thread, contiguous
  const int b_lo = min(tid * per, a.B), b_hi = min(b_lo + per, a.B);
  uint32_t mine = 0;
  auto positions = [&](int b) {        // of one unit of request b
    const uint32_t keys = visible(a, b);
    return keys == 0 ? 0u : (keys + TILE - 1) / TILE + 1;
  };
  for (int b = b_lo; b < b_hi; ++b) mine += positions(b);
  uint32_t upto = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += y;
  }
  if (lane == 31) scratch.warp_tiles[warp] = upto;
  __syncthreads();
  s.total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += scratch.warp_tiles[w];
    s.total += scratch.warp_tiles[w];
  }
  const uint32_t list = s.total * units;
  const uint32_t shares = min(gridDim.x, list), me = blockIdx.x;
  if (me >= shares) return false;
  // shares differ by one position at most, the longer ones first
  s.even = list / shares;
  s.longer = list - s.even * shares;
  s.begin = me * s.even + min(me, s.longer);
  s.end = s.begin + s.even + (me < s.longer ? 1 : 0);
  if (s.begin >= (upto - mine) * units && s.begin < upto * units) {  // exactly one thread
    uint32_t sum = upto - mine;
    int b = b_lo;
    while (true) {
      const uint32_t here = positions(b);
      if (s.begin < (sum + here) * units) break;
      sum += here;
      ++b;
    }
    scratch.first = b;
    scratch.before = sum;
    scratch.length = a.lengths[b];
  }
  __syncthreads();
  s.first = scratch.first;
  s.before = scratch.before;
  s.length = scratch.length;
  return true;
}

// The first tile of a share; false where it holds only the end of a unit.
template <int TILE>
__device__ __forceinline__ bool first_tile(const PagedWork& a, const Share& s, Cursor<TILE>& work) {
  work.set_request(a, s.first, s.length);
  const uint32_t at = s.begin - s.before * (a.Hkv * a.row_blocks);  // inside the request's units
  const int hr = (int)(at / (work.tiles + 1));
  work.t = at - hr * (work.tiles + 1);
  work.h = hr / a.row_blocks;
  work.rb = hr - work.h * a.row_blocks;
  work.pos = s.begin;
  if (work.t < work.tiles) return true;
  // it begins with a unit's end: the first tile is the next unit's
  if (s.begin + 1 >= s.end) return false;
  --work.t;
  --work.pos;
  work.next(a);
  return true;
}

// The share that position `pos` lies in.
__device__ __forceinline__ uint32_t share_of(const Share& s, uint32_t pos) {
  const uint32_t in_longer = s.longer * (s.even + 1);
  return pos < in_longer ? pos / (s.even + 1) : s.longer + (pos - in_longer) / s.even;
}

// Requests without a visible position are nobody's unit.
__device__ __forceinline__ void clear_empty(const PagedWork& a) {
  const int tid = threadIdx.x, units = a.Hkv * a.row_blocks;
  for (int b = (int)blockIdx.x; b < a.B; b += gridDim.x) {
    if (visible(a, b) != 0) continue;
    for (int i = tid; i < a.Hq * (a.D / 8); i += kThreads) {
      const int h = i / (a.D / 8), c = i % (a.D / 8);
      *reinterpret_cast<uint4*>(a.o + ((int64_t)b * a.Hq + h) * a.D + c * 8) = make_uint4(0, 0, 0, 0);
    }
    if (a.lse)
      for (int h = tid; h < a.Hq; h += kThreads) a.lse[(int64_t)b * a.Hq + h] = -INFINITY;
    if (a.join_units)
      for (int u = tid; u < units; u += kThreads) a.joins[b * units + u].x = -1;
  }
}

// 16 bytes of zeros to shared memory where `pred` (without a branch).
__device__ __forceinline__ void clear16(uint32_t at, bool pred) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p st.shared.v4.b32 [%0], {%2, %2, %2, %2};\n\t}" ::"r"(at),
               "r"((uint32_t)pred), "r"(0)
               : "memory");
}

// 1 / x to one unit in the last place.  x is a sum of weights: wherever a row
// sees anything finite 1 or more in a 16-bit cache, between 2^-49 and 2^75
// times the number of keys over an 8-bit one (kf::kMaxExponent), so neither x
// nor 1 / x is subnormal, which the instruction takes for 0.
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// Barrier of a team's warps that returns the AND of their `pred`, so that all
// of them go on alike.
template <int RG>
__device__ __forceinline__ bool team_and(int team, bool pred) {
  if constexpr (RG == 1)
    return __all_sync(0xffffffffu, pred);
  else if constexpr (RG == kWarps)
    return __syncthreads_and(pred);
  else
    return kf::named_bar_and(1 + team, RG * 32, pred);
}

// Joins the partials of a unit that was cut: slot 1 of its first share, slot 0
// of the shares up to its last.  A group of D / 4 lanes takes one row, alone
// or, where a unit has many partials, with `split` - 1 others that take every
// split-th partial; each partial is read once, with a running maximum, and the
// groups' results meet in shared memory.
constexpr int kJoinThreads = 256;
constexpr int kJoinBatch = 8;  // partials a group has in flight (4: 0.3 to 0.5 us more on calls of 12 to 50 us)

template <bool BF16>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedWork a, int rows, int split) {
  kf::griddep_wait();
  kf::griddep_launch_dependents();
  const int4 unit = a.joins[blockIdx.x];
  if (unit.x < 0) return;
  const int h = unit.y / a.row_blocks, rb = unit.y - h * a.row_blocks;
  const int count = unit.w - unit.z + 1;
  __shared__ float4 acc_s[kJoinThreads];
  __shared__ float m_s[kJoinThreads / 4], l_s[kJoinThreads / 4];
  const int lanes = a.D / 4, per_block = kJoinThreads / lanes / split;  // rows of a block
  const int g = threadIdx.x / lanes, c = threadIdx.x % lanes;
  const int part = g % split, r = blockIdx.y * per_block + g / split;
  const bool mine = g < per_block * split && r < min(rows, a.G - rb * rows);
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (mine) {
    for (int j0 = part; j0 < count; j0 += split * kJoinBatch) {
      float lse[kJoinBatch];
      float4 o[kJoinBatch];
#pragma unroll
      for (int x = 0; x < kJoinBatch; ++x) {
        const int j = j0 + x * split;
        lse[x] = -INFINITY;
        o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j < count) {
          const int64_t row = (((int64_t)unit.z + j) * 2 + (j == 0 ? 1 : 0)) * rows + r;
          lse[x] = a.part_lse[row];
          o[x] = *reinterpret_cast<const float4*>(a.part_o + row * a.D + c * 4);
        }
      }
      float top = m;
#pragma unroll
      for (int x = 0; x < kJoinBatch; ++x) top = fmaxf(top, lse[x]);
      const float mu = top == -INFINITY ? 0.f : top;
      const float old = kf::ex2(m - mu);
      l *= old;
      acc.x *= old;
      acc.y *= old;
      acc.z *= old;
      acc.w *= old;
#pragma unroll
      for (int x = 0; x < kJoinBatch; ++x) {
        const float w = kf::ex2(lse[x] - mu);
        l += w;
        acc.x += w * o[x].x;
        acc.y += w * o[x].y;
        acc.z += w * o[x].z;
        acc.w += w * o[x].w;
      }
      m = top;
    }
  }
  if (split > 1) {
    acc_s[threadIdx.x] = acc;
    if (mine && c == 0) {
      m_s[g] = m;
      l_s[g] = l;
    }
    __syncthreads();
    if (mine && part == 0) {
      float top = m;
      for (int i = 1; i < split; ++i) top = fmaxf(top, m_s[g + i]);
      const float mu = top == -INFINITY ? 0.f : top;
      const float old = kf::ex2(m - mu);
      l *= old;
      acc.x *= old;
      acc.y *= old;
      acc.z *= old;
      acc.w *= old;
      for (int i = 1; i < split; ++i) {
        const float w = kf::ex2(m_s[g + i] - mu);
        const float4 x = acc_s[threadIdx.x + i * lanes];
        l += w * l_s[g + i];
        acc.x += w * x.x;
        acc.y += w * x.y;
        acc.z += w * x.z;
        acc.w += w * x.w;
      }
      m = top;
    }
  }
  if (!mine || part != 0) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int head = h * a.G + rb * rows + r;
  *reinterpret_cast<uint2*>(a.o + ((int64_t)unit.x * a.Hq + head) * a.D + c * 4) =
      make_uint2(kf::pack2<BF16>(acc.x * inv, acc.y * inv), kf::pack2<BF16>(acc.z * inv, acc.w * inv));
  if (a.lse && c == 0) a.lse[(int64_t)unit.x * a.Hq + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Query rows of a unit for G rows per KV head, and the variant that has them.
inline int unit_rows(int64_t G) { return G <= 8 ? 8 : G <= 16 ? 16 : G <= 32 ? 32 : 64; }

inline size_t workspace_need(int blocks, int rows, int64_t D) {
  return 256 + (size_t)blocks * (16 + (size_t)2 * rows * 4 + (size_t)2 * rows * D * 4);
}

// The sizes of a call, the grid and where its partials lie.  `tile`: keys of a
// tile, `rows`: query rows of a unit.  One wave of blocks, or fewer when the
// tables cannot hold that many tiles.  A unit of one tile is never cut, so
// nothing is left to join (*most == 1).
inline int plan_work(const char* what, PagedWork& a, int64_t max_pages, int rows, int64_t tile, int blocks_per_sm,
                     void* workspace, uint64_t workspace_bytes, int64_t* blocks_out, int64_t* most_out) {
  a.row_blocks = (a.G + rows - 1) / rows;
  const int64_t capacity = max_pages * a.page_size;
  a.capacity = (uint32_t)(capacity < 0x7fffffffLL ? capacity : 0x7fffffffLL);
  a.max_pages = (uint32_t)max_pages;
  kf::division(a.page_size, &a.page_mul, &a.page_shift);
  const int64_t most = (a.capacity + tile - 1) / tile;
  const int64_t units = (int64_t)a.B * a.Hkv * a.row_blocks;
  int64_t blocks = (int64_t)kf::sm_count_current_device() * blocks_per_sm;
  if (units * (most + 1) > 0x7fffffffLL) return kf::set_error(KF_ERR_UNSUPPORTED, "%s: tensors too large", what);
  if (most == 1 && units < blocks) blocks = units;
  if (units * (most + 1) < blocks) blocks = units * (most + 1);
  a.part_o = nullptr;
  a.part_lse = nullptr;
  a.joins = nullptr;
  a.join_units = false;
  if (most > 1) {
    const size_t need = workspace_need((int)blocks, rows, a.D);
    if (!workspace || workspace_bytes < need)
      return kf::set_error(KF_ERR_WORKSPACE, "%s: workspace needs %zu bytes", what, need);
    uintptr_t base = (reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255);
    a.joins = reinterpret_cast<int4*>(base);
    a.part_o = reinterpret_cast<float*>(a.joins + blocks);
    a.part_lse = a.part_o + (size_t)blocks * 2 * rows * a.D;
    a.join_units = units < blocks;  // whichever list is shorter
  }
  *blocks_out = blocks;
  *most_out = most;
  return KF_OK;
}

// The join of what the blocks left.  Groups that share a row: as many as leave
// each about one batch of the partials that a unit has on average (2 where
// units outnumber the blocks).
inline int launch_join(const char* what, const PagedWork& a, bool bf16, int rows, int64_t blocks, cudaStream_t st) {
  const int64_t units = (int64_t)a.B * a.Hkv * a.row_blocks;
  const int groups = kJoinThreads / (a.D / 4);
  const int64_t partials = a.join_units ? blocks / units + 1 : 2;
  int split = 1;
  while (split * kJoinBatch < partials && split * 2 <= groups) split *= 2;
  const int per_block = groups / split, row_count = a.G < rows ? a.G : rows;
  const dim3 grid((unsigned)(a.join_units ? units : blocks), (unsigned)((row_count + per_block - 1) / per_block));
  return bf16 ? kf::launch_dependent(paged_join_kernel<true>, grid, dim3(kJoinThreads), 0, st, what, a, rows, split)
              : kf::launch_dependent(paged_join_kernel<false>, grid, dim3(kJoinThreads), 0, st, what, a, rows, split);
}

}  // namespace
