// K6: the paged KV cache's own kernels: append of K/V rows to their slots,
// and the block tables and slot maps made from request lengths.
//
// A pool of pages [pages, Hkv, page_size, D] holds the K (and V) rows of all
// requests; position p of request b is row p % page_size of page
// block_table[b][p / page_size], and its slot is page * page_size + p %
// page_size.  The pages that no request owns are a stack, free_pages[0 ..
// free_count).
#include <cooperative_groups.h>

#include <type_traits>

#include "kf_host.h"
#include "kf_sm100.cuh"

namespace cg = cooperative_groups;

namespace {

// ---------------------------------------------------------------- append
// Pure data movement: 2 x Hkv x D elements read and written per token, no
// arithmetic, so HBM (or, for one token per request, latency) bounds it: 16384
// tokens of 8 x 128 take 22.7 us, 90% of the measured copy rate.  A thread
// keeps one 16-byte column of a token's Hkv * D elements and walks
// over tokens, so the division that finds (head, column) is done once; U
// tokens are loaded before the first is stored.
constexpr int kAppendThreads = 256;

struct AppendArgs {
  const uint16_t* src_k;
  const uint16_t* src_v;
  uint16_t* dst_k;
  uint16_t* dst_v;
  const int64_t* slots;
  int64_t sk[4], sv[4], dk[4], dv[4];
  int64_t num_slots;
  uint32_t T, S;            // tokens in all, and per batch entry
  uint32_t per_token;       // vectors of one token (Hkv * D / VEC)
  uint32_t per_head;        // vectors of one head (D / VEC)
  uint32_t page_size;
  uint32_t block_tokens;    // tokens side by side in a block (0: a block walks one token's vectors)
};

template <int VEC>
__device__ __forceinline__ void move_token(const AppendArgs& a, int64_t slot, uint32_t t, uint32_t vec, bool load,
                                           uint4 (&val)[2]) {
  using E = typename std::conditional<VEC == 8, uint4, uint16_t>::type;
  const uint32_t h = vec / a.per_head, d = (vec - h * a.per_head) * VEC;
  if (load) {
    const uint32_t n = a.S == a.T ? 0 : t / a.S, s = t - n * a.S;
    const E* pk = reinterpret_cast<const E*>(a.src_k + n * a.sk[0] + h * a.sk[1] + s * a.sk[2] + d * a.sk[3]);
    const E* pv = reinterpret_cast<const E*>(a.src_v + n * a.sv[0] + h * a.sv[1] + s * a.sv[2] + d * a.sv[3]);
    if constexpr (VEC == 8) {
      // through L2: the predecessor may have written these while this kernel was
      // alive, so not non-coherently (16384 tokens: 22.9 us as with non-coherent
      // loads, 24.3 with loads that look in L1 first)
      val[0] = __ldcg(pk);
      val[1] = __ldcg(pv);
    } else {
      val[0].x = *pk;
      val[1].x = *pv;
    }
  } else {
    // slots of a pool fit 32 bits unless it holds over 2^32 tokens
    const bool small = a.num_slots <= 0xffffffffLL;
    const int64_t page = small ? (int64_t)((uint32_t)slot / a.page_size) : slot / a.page_size;
    const int64_t r = slot - page * a.page_size;
    E* pk = reinterpret_cast<E*>(a.dst_k + page * a.dk[0] + h * a.dk[1] + r * a.dk[2] + d * a.dk[3]);
    E* pv = reinterpret_cast<E*>(a.dst_v + page * a.dv[0] + h * a.dv[1] + r * a.dv[2] + d * a.dv[3]);
    if constexpr (VEC == 8) {
      *pk = val[0];
      *pv = val[1];
    } else {
      *pk = (uint16_t)val[0].x;
      *pv = (uint16_t)val[1].x;
    }
  }
}

template <int VEC, int U>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendArgs a) {
  kf::griddep_wait();
  kf::griddep_launch_dependents();
  const uint32_t side = a.block_tokens ? a.block_tokens : 1;
  const uint32_t local = a.block_tokens ? threadIdx.x / a.per_token : 0;
  if (local >= side) return;
  const uint32_t vec0 = threadIdx.x - local * (a.block_tokens ? a.per_token : 0);
  const uint64_t step = (uint64_t)gridDim.x * side * U;
  for (uint64_t base = (uint64_t)blockIdx.x * side * U; base < a.T; base += step) {
    int64_t slot[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t t = base + u * side + local;
      slot[u] = t < a.T ? a.slots[t] : -1;
      if (slot[u] >= a.num_slots) slot[u] = -1;  // no such slot: the token is not stored
    }
    for (uint32_t vec = vec0; vec < a.per_token; vec += kAppendThreads) {
      uint4 val[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (slot[u] >= 0) move_token<VEC>(a, slot[u], (uint32_t)(base + u * side + local), vec, true, val[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (slot[u] >= 0) move_token<VEC>(a, slot[u], (uint32_t)(base + u * side + local), vec, false, val[u]);
    }
  }
}

bool vec_ok(const kf_tensor4* t) {
  if (!kf::aligned16(t->ptr) || t->stride[3] != 1) return false;
  for (int i = 0; i < 3; ++i)
    if (t->size[i] > 1 && (t->stride[i] % 8) != 0) return false;
  return true;
}

// ---------------------------------------------------------------- tables
// Both kernels below are prefix sums over requests followed by independent
// writes; they move a few bytes per token and page, so latency bounds them.
// They run as ONE cluster of up to 8 blocks: every block scans all requests
// itself (reading 8 bytes per request is cheaper than a second launch), takes
// its share of the writes, and the cluster barrier lets block 0 replace the
// lengths and the stack count in place once nobody reads the old ones.
// Blocks of kSmall threads, whose barriers and scans are quicker, for what one
// such block passes over once or a few times (256 single tokens: 3.5 us with
// 512 threads, 3.6 with 256, 4.3 with 1024), else of kLarge (122377 prompt
// tokens: 14.4 us with 512 threads, 12.0 with 1024).
constexpr int kSmall = 512, kLarge = 1024;
constexpr int kMaxCluster = 8;
constexpr int64_t kMaxRequests = 16384;  // 12 bytes of shared memory each

// x / page_size for x < 2^31
struct PageDiv {
  uint32_t size, mul, shift;
  __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (uint32_t)(((uint64_t)x * mul) >> shift); }
  __device__ __forceinline__ uint32_t pages(uint32_t tokens) const {  // rounded up
    const uint32_t q = (*this)(tokens);
    return q + (q * size != tokens);
  }
};

__device__ __forceinline__ int32_t saturate(int64_t x) { return x > 0x7fffffff ? 0x7fffffff : (int32_t)x; }

// Inclusive sums of x and y over the block's threads; every thread also gets
// the block's totals.  `part` is reused by the next call.
template <int THREADS>
__device__ __forceinline__ void block_scan(int64_t& x, int64_t& y, int64_t (*part)[2], int64_t& x_total,
                                           int64_t& y_total) {
  constexpr int WARPS = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, (long long)x, off), v = __shfl_up_sync(0xffffffffu, (long long)y, off);
    if (lane >= off) {
      x += u;
      y += v;
    }
  }
  __syncthreads();  // the previous call's readers are done with part
  if (lane == 31) {
    part[warp][0] = x;
    part[warp][1] = y;
  }
  __syncthreads();
  // every warp sums the warps' totals itself: lane w holds warp w's
  int64_t u = lane < WARPS ? part[lane][0] : 0, v = lane < WARPS ? part[lane][1] : 0;
#pragma unroll
  for (int off = 1; off < WARPS; off <<= 1) {
    const int64_t p = __shfl_up_sync(0xffffffffu, (long long)u, off), q = __shfl_up_sync(0xffffffffu, (long long)v, off);
    if (lane >= off) {
      u += p;
      v += q;
    }
  }
  x_total = __shfl_sync(0xffffffffu, (long long)u, WARPS - 1);
  y_total = __shfl_sync(0xffffffffu, (long long)v, WARPS - 1);
  const int64_t x_before = __shfl_sync(0xffffffffu, (long long)u, warp > 0 ? warp - 1 : 0);
  const int64_t y_before = __shfl_sync(0xffffffffu, (long long)v, warp > 0 ? warp - 1 : 0);
  if (warp > 0) {
    x += x_before;
    y += y_before;
  }
}

// Largest i in [0, n) with v[i] <= x (v is nondecreasing and v[0] <= x).
__device__ __forceinline__ int last_at_most(const int32_t* v, int n, int64_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct ReserveArgs {
  const int32_t* lengths;
  const int32_t* added;
  int32_t* table;
  const int32_t* free_pages;
  const int32_t* free_count;
  int64_t* slots;
  int32_t* starts;
  int32_t* lengths_out;
  int32_t* free_count_out;
  int64_t table_stride;
  int64_t T;
  PageDiv div;
  uint32_t padded;  // 0: tokens request after request; else the slots of each request
  int B;
  uint32_t max_pages, num_pages;
};

// need_b = ceil((len_b + new_b) / page) - ceil(len_b / page), 0 where the
// request would outgrow its table row (or its padded slots); upto = inclusive
// sum of need.  A request is granted when it fits, upto_b <= free_count (or
// it needs no page) and its packed slots end within num_tokens (or it has no
// token); the granted requests that need pages are then a prefix, since both
// sums only grow, so request b takes the stack entries free_count - 1 -
// (upto_b - need_b) - j.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) paged_reserve_kernel(const ReserveArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* starts = sm;               // [B + 1] first token of each request
  int32_t* first = sm + a.B + 1;      // [B] pages taken by the requests before it
  int32_t* held = first + a.B;        // [B] its length so far, or -1 where it is refused
  __shared__ int64_t part[THREADS / 32][2];
  __shared__ int taken_s;
  kf::griddep_wait();
  kf::griddep_launch_dependents();
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  const unsigned rank = blockIdx.x, blocks = gridDim.x;  // the grid is one cluster
  if (tid == 0) taken_s = 0;
  int32_t count = *a.free_count;
  count = count < 0 ? 0 : (uint32_t)count > a.num_pages ? (int32_t)a.num_pages : count;

  int64_t tokens = 0, pages = 0;  // of the requests of earlier rounds
  for (int base = 0; base < a.B; base += THREADS) {
    const int b = base + tid;
    uint32_t len = 0, add = 0;
    if (b < a.B) {
      len = (uint32_t)max(a.lengths[b], 0);
      add = (uint32_t)max(a.added[b], 0);
    }
    const uint32_t end = len + add;  // below 2^32
    const uint32_t before = a.div.pages(len), after = end <= 0x7fffffffu ? a.div.pages(end) : 0xffffffffu;
    const bool fits = after <= a.max_pages && (a.padded == 0 || add <= a.padded);
    const int64_t need = fits ? after - before : 0;
    int64_t add_upto = add, upto = need, add_total, need_total;
    block_scan<THREADS>(add_upto, upto, part, add_total, need_total);
    add_upto += tokens;
    upto += pages;
    if (b < a.B) {
      const bool slotted = a.padded != 0 || add == 0 || add_upto <= a.T;
      const bool granted = fits && slotted && (need == 0 || upto <= count);
      starts[b] = saturate(a.padded ? (int64_t)b * a.padded : add_upto - add);
      first[b] = saturate(upto - need);
      held[b] = granted ? (int32_t)len : -1;
      if (granted && need > 0) atomicMax(&taken_s, (int)upto);  // a maximum: the order does not matter
    }
    tokens += add_total;
    pages += need_total;
  }
  if (tid == 0) starts[a.B] = saturate(a.padded ? (int64_t)a.B * a.padded : tokens);
  __syncthreads();
  const int taken = taken_s;

  // page j of request b, a new one or one that it holds
  auto page_at = [&](int b, uint32_t before, uint32_t j) -> int64_t {
    const int32_t p = j < before ? a.table[b * a.table_stride + j]
                                 : a.free_pages[count - 1 - (first[b] + (int32_t)(j - before))];
    return (uint32_t)p < a.num_pages ? (int64_t)p * a.div.size : -1;
  };
  // Slots.  A thread takes `run` consecutive tokens: one, so that a step of
  // single tokens is one pass of independent lookups, or four where there are
  // more tokens than threads; along a run it moves from row to row and looks
  // a page up only where one begins.
  const int64_t threads = (int64_t)blocks * THREADS;
  const int run = a.T > threads ? 4 : 1;
  for (int64_t t0 = ((int64_t)rank * THREADS + tid) * run; t0 < a.T; t0 += threads * run) {
    int64_t slot[4];
    int b = last_at_most(starts, a.B, t0);
    int64_t base = -1;
    int32_t next = starts[b], stop = 0;  // the run's request ends before token `next`, its new tokens before `stop`
    uint32_t before = 0, j = 0, r = 0;
    bool inside = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      slot[e] = -1;
      if (e >= run) continue;
      const int64_t t = t0 + e;
      if (!inside || t >= next) {  // the first token of the run, or of another request
        while (b + 1 < a.B && starts[b + 1] <= t) ++b;
        next = b + 1 < a.B ? starts[b + 1] : 0x7fffffff;
        stop = held[b] < 0 ? 0 : a.padded ? starts[b] + max(a.added[b], 0) : starts[b + 1];
        inside = true;
        if (t < stop) {
          const uint32_t pos = (uint32_t)held[b] + (uint32_t)(t - starts[b]);
          before = a.div.pages((uint32_t)held[b]);
          j = a.div(pos);
          r = pos - j * a.div.size;
          base = page_at(b, before, j);
        }
      } else if (t < stop && ++r == a.div.size) {
        r = 0;
        base = page_at(b, before, ++j);
      }
      if (t < stop && base >= 0) slot[e] = base + r;
    }
    if (run == 1) {
      a.slots[t0] = slot[0];
    } else if (t0 + 4 <= a.T) {
      longlong2* dst = reinterpret_cast<longlong2*>(a.slots + t0);
      dst[0] = make_longlong2(slot[0], slot[1]);
      dst[1] = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (t0 + e < a.T) a.slots[t0 + e] = slot[e];
    }
  }
  // New entries of the block table: stack entry count - 1 - p is the p-th page
  // taken.  From the far end of the threads, which a short list of tokens
  // leaves free.
  for (int64_t p = threads - 1 - ((int64_t)rank * THREADS + tid); p < taken; p += threads) {
    const int b = last_at_most(first, a.B, p);
    a.table[b * a.table_stride + a.div.pages((uint32_t)held[b]) + (p - first[b])] = a.free_pages[count - 1 - p];
  }
  // lengths_out and free_count_out may be lengths and free_count themselves
  cluster.sync();
  if (rank == 0) {
    for (int b = tid; b < a.B; b += THREADS) {
      const int32_t len = held[b];
      a.lengths_out[b] = len < 0 ? max(a.lengths[b], 0) : len + max(a.added[b], 0);
    }
    for (int b = tid; b <= a.B; b += THREADS) a.starts[b] = starts[b];
    if (tid == 0) *a.free_count_out = count - taken;
  }
}

struct ReleaseArgs {
  const int32_t* lengths;
  const uint8_t* finished;
  const int32_t* table;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* lengths_out;
  int32_t* free_count_out;
  int64_t table_stride;
  PageDiv div;
  int B;
  uint32_t max_pages, num_pages;
};

// One warp per request: count the row's valid entries (a row may hold -1 where
// a page was given up earlier), then, after a prefix sum over requests, write
// them to the stack in order.  The counts reach every block through
// distributed shared memory.  The first kKept * 32 entries of a warp's first
// request stay in registers from the count to the write.
constexpr int kKept = 16;

template <int THREADS>
__global__ void __launch_bounds__(THREADS) paged_release_kernel(const ReleaseArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* counts = sm;  // [B] valid pages of each request, then their exclusive sum
  __shared__ int64_t part[THREADS / 32][2];
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();  // this block has started: its shared memory may be written
  kf::griddep_wait();
  kf::griddep_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned rank = blockIdx.x, blocks = gridDim.x;
  int32_t count = *a.free_count;
  count = count < 0 ? 0 : (uint32_t)count > a.num_pages ? (int32_t)a.num_pages : count;

  auto row_pages = [&](int b) -> uint32_t {
    const int32_t len = a.lengths[b];
    return a.finished[b] ? min(a.div.pages((uint32_t)max(len, 0)), a.max_pages) : 0;
  };
  const int b0 = (int)rank * (THREADS / 32) + warp;  // this warp's first request
  uint32_t kept[kKept];
  bool waited = false;
  for (int b = b0; b < a.B; b += blocks * (THREADS / 32)) {
    const uint32_t n = row_pages(b);
    const int32_t* row = a.table + b * a.table_stride;
    int c = 0;
    uint32_t j = lane;
    if (b == b0) {
#pragma unroll
      for (int k = 0; k < kKept; ++k) kept[k] = j + k * 32 < n ? (uint32_t)row[j + k * 32] : 0xffffffffu;
#pragma unroll
      for (int k = 0; k < kKept; ++k) c += kept[k] < a.num_pages;
      j += kKept * 32;
    }
#pragma unroll 8
    for (; j < n; j += 32) c += (uint32_t)row[j] < a.num_pages;
    c = __reduce_add_sync(0xffffffffu, c);
    if (!waited) cluster.barrier_wait();
    waited = true;
    if (lane < (int)blocks) cluster.map_shared_rank(counts, lane)[b] = c;
  }
  if (!waited) cluster.barrier_wait();
  cluster.sync();
  int64_t total = 0;
  for (int base = 0; base < a.B; base += THREADS) {
    const int b = base + tid;
    const int32_t c = b < a.B ? counts[b] : 0;
    int64_t upto = c, none = 0, round, unused;
    block_scan<THREADS>(upto, none, part, round, unused);
    if (b < a.B) counts[b] = saturate(total + upto - c);
    total += round;
  }
  __syncthreads();
  for (int b = b0; b < a.B; b += blocks * (THREADS / 32)) {
    const uint32_t n = row_pages(b);
    const int32_t* row = a.table + b * a.table_stride;
    int64_t at = (int64_t)count + counts[b];
    auto push = [&](uint32_t page) {
      const bool valid = page < a.num_pages;
      const unsigned mask = __ballot_sync(0xffffffffu, valid);
      const int64_t to = at + __popc(mask & ((1u << lane) - 1));
      if (valid && to < a.num_pages) a.free_pages[to] = (int32_t)page;  // a stack that is full keeps what it has
      at += __popc(mask);
    };
    uint32_t j0 = 0;
    if (b == b0) {
#pragma unroll
      for (int k = 0; k < kKept; ++k)
        if (k * 32 < n) push(kept[k]);
      j0 = kKept * 32;
    }
    for (; j0 < n; j0 += 128) {
      uint32_t page[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t j = j0 + k * 32 + lane;
        page[k] = j < n ? (uint32_t)row[j] : 0xffffffffu;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) push(page[k]);
    }
  }
  cluster.sync();
  if (rank == 0) {
    for (int b = tid; b < a.B; b += THREADS) a.lengths_out[b] = a.finished[b] ? 0 : max(a.lengths[b], 0);
    if (tid == 0) *a.free_count_out = (int32_t)min((int64_t)a.num_pages, count + total);
  }
}

int check_tables(const char* what, const kf_page_tables& t) {
  using kf::set_error;
  if (!t.lengths || !t.block_table || !t.free_pages || !t.free_count || !t.lengths_out || !t.free_count_out)
    return set_error(KF_ERR_INVALID, "%s: null data pointer", what);
  if (t.B <= 0 || t.max_pages <= 0 || t.num_pages <= 0)
    return set_error(KF_ERR_INVALID, "%s: requests, table columns and pages must be non-zero", what);
  if (t.page_size <= 0 || t.page_size > (1 << 20))
    return set_error(KF_ERR_INVALID, "%s: page_size must be in [1, 2^20]", what);
  if (t.B > 1 && t.table_stride < t.max_pages)
    return set_error(KF_ERR_INVALID, "%s: block table rows overlap", what);
  if (t.B > kMaxRequests)
    return set_error(KF_ERR_UNSUPPORTED, "%s: at most %lld requests", what, (long long)kMaxRequests);
  if (t.max_pages > 0x7fffffffLL || t.num_pages > 0x7fffffffLL)
    return set_error(KF_ERR_UNSUPPORTED, "%s: too many pages", what);
  return KF_OK;
}

// Dynamic shared memory of the two kernels.
constexpr size_t reserve_smem(int64_t B) { return (size_t)(3 * B + 1) * 4; }
constexpr size_t release_smem(int64_t B) { return (size_t)B * 4; }

// Without this a block gets 48 KB, its static arrays (up to 528 bytes)
// included.  The limit is raised to the kernel's largest size, `most`, never to
// that of one call: calls of other threads may lie between this and the launch.
template <typename... KArgs>
int raise_smem(void (*kern)(KArgs...), size_t smem, size_t most, const char* what) {
  if (smem > 47 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess) {
    (void)cudaGetLastError();
    return kf::set_error(KF_ERR_CUDA, "%s: cannot reserve %zu bytes of shared memory", what, most);
  }
  return KF_OK;
}

PageDiv page_div(int64_t page_size) {
  PageDiv d;
  d.size = (uint32_t)page_size;
  kf::division(page_size, &d.mul, &d.shift);
  return d;
}

unsigned cluster_for(int64_t units, int64_t per_block) {
  int64_t n = (units + per_block - 1) / per_block;
  if (n <= 1) return 1;
  if (n <= 2) return 2;
  if (n <= 4) return 4;
  return kMaxCluster;
}

}  // namespace

extern "C" int kf_paged_append(const kf_paged_append_args* args) {
  using kf::set_error;
  if (!args) return set_error(KF_ERR_INVALID, "kf_paged_append: null arguments");
  const kf_tensor4 *k_pages = &args->k_pages, *v_pages = &args->v_pages, *new_k = &args->new_k, *new_v = &args->new_v;
  const int64_t dtype = args->dtype;
  if (dtype != KF_F16 && dtype != KF_BF16)
    return set_error(KF_ERR_INVALID, "kf_paged_append: dtype must be fp16 or bf16");
  for (int i = 0; i < 4; ++i) {
    if (k_pages->size[i] != v_pages->size[i])
      return set_error(KF_ERR_INVALID, "kf_paged_append: K/V page shapes must match");
    if (new_k->size[i] != new_v->size[i])
      return set_error(KF_ERR_INVALID, "kf_paged_append: new K/V shapes must match");
  }
  const int64_t N = new_k->size[0], H = new_k->size[1], S = new_k->size[2], D = new_k->size[3];
  if (H != k_pages->size[1] || D != k_pages->size[3])
    return set_error(KF_ERR_INVALID, "kf_paged_append: new K/V heads and head_dim must match the pages");
  if (N <= 0 || H <= 0 || S <= 0 || D <= 0 || k_pages->size[0] <= 0 || k_pages->size[2] <= 0)
    return set_error(KF_ERR_INVALID, "kf_paged_append: dimensions must be non-zero");
  if (N > 0x7fffffffLL || S > 0x7fffffffLL || N * S > 0x7fffffffLL || H > 0x7fffffffLL || D > 0x7fffffffLL ||
      H * D > 0x7fffffffLL || k_pages->size[2] > (1 << 20))
    return set_error(KF_ERR_UNSUPPORTED, "kf_paged_append: tensors too large");
  if (!k_pages->ptr || !v_pages->ptr || !new_k->ptr || !new_v->ptr || !args->slots)
    return set_error(KF_ERR_INVALID, "kf_paged_append: null data pointer");
  kf::DeviceGuard guard(k_pages->ptr);
  if (guard.status()) return guard.status();

  AppendArgs a;
  a.src_k = static_cast<const uint16_t*>(new_k->ptr);
  a.src_v = static_cast<const uint16_t*>(new_v->ptr);
  a.dst_k = static_cast<uint16_t*>(k_pages->ptr);
  a.dst_v = static_cast<uint16_t*>(v_pages->ptr);
  a.slots = args->slots;
  for (int i = 0; i < 4; ++i) {
    a.sk[i] = new_k->stride[i];
    a.sv[i] = new_v->stride[i];
    a.dk[i] = k_pages->stride[i];
    a.dv[i] = v_pages->stride[i];
  }
  const bool vec = D % 8 == 0 && vec_ok(k_pages) && vec_ok(v_pages) && vec_ok(new_k) && vec_ok(new_v);
  a.num_slots = k_pages->size[0] * k_pages->size[2];
  a.T = (uint32_t)(N * S);
  a.S = (uint32_t)S;
  a.per_head = (uint32_t)(vec ? D / 8 : D);
  a.per_token = (uint32_t)H * a.per_head;
  a.page_size = (uint32_t)k_pages->size[2];
  a.block_tokens = a.per_token <= kAppendThreads ? kAppendThreads / a.per_token : 0;
  const int64_t side = a.block_tokens ? a.block_tokens : 1;
  const int64_t sms = kf::sm_count_current_device();
  cudaStream_t st = static_cast<cudaStream_t>(args->stream);
  auto go = [&](auto kern, int64_t per_block) {
    int64_t blocks = (a.T + per_block - 1) / per_block;
    if (blocks > sms * 64) blocks = sms * 64;
    return kf::launch_dependent(kern, dim3((unsigned)blocks), dim3(kAppendThreads), 0, st, "kf_paged_append", a);
  };
  if (!vec) return go(paged_append_kernel<1, 1>, side);
  // Four tokens a thread in flight once that still leaves three blocks per SM
  // (4096 tokens of 8 x 128: 7.1 us with one, 6.5 with four; 20000 of 1 x 128:
  // 4.2 with one, 5.4 with four).
  return a.T >= side * 4 * sms * 3 ? go(paged_append_kernel<8, 4>, side * 4) : go(paged_append_kernel<8, 1>, side);
}

extern "C" int kf_paged_reserve(const kf_paged_reserve_args* args) {
  using kf::set_error;
  const char* what = "kf_paged_reserve";
  if (!args) return set_error(KF_ERR_INVALID, "%s: null arguments", what);
  const kf_page_tables& t = args->tables;
  int rc = check_tables(what, t);
  if (rc != KF_OK) return rc;
  const int64_t num_tokens = args->num_tokens, per_request = args->tokens_per_request;
  if (num_tokens < 0 || num_tokens > 0x7fffffffLL)
    return set_error(KF_ERR_INVALID, "%s: num_tokens must be in [0, 2^31)", what);
  if (per_request < 0 || (per_request > 0 && (per_request > num_tokens || per_request * t.B != num_tokens)))
    return set_error(KF_ERR_INVALID, "%s: num_tokens must be tokens_per_request for each request", what);
  if (!args->new_lengths || !args->starts || (num_tokens > 0 && !args->slots))
    return set_error(KF_ERR_INVALID, "%s: null data pointer", what);
  if (num_tokens > 0 && !kf::aligned16(args->slots))
    return set_error(KF_ERR_INVALID, "%s: slots must be 16-byte aligned", what);
  kf::DeviceGuard guard(t.lengths);
  if (guard.status()) return guard.status();
  ReserveArgs a;
  a.lengths = t.lengths;
  a.added = args->new_lengths;
  a.table = t.block_table;
  a.free_pages = t.free_pages;
  a.free_count = t.free_count;
  a.slots = args->slots;
  a.starts = args->starts;
  a.lengths_out = t.lengths_out;
  a.free_count_out = t.free_count_out;
  a.table_stride = t.table_stride;
  a.T = num_tokens;
  a.padded = (uint32_t)per_request;
  a.B = (int)t.B;
  a.max_pages = (uint32_t)t.max_pages;
  a.div = page_div(t.page_size);
  a.num_pages = (uint32_t)t.num_pages;
  const size_t smem = reserve_smem(t.B);
  const bool large = t.B > kSmall || num_tokens > 4 * kSmall;
  const unsigned cluster = large ? cluster_for(num_tokens, kLarge * 4) : 1;
  auto kern = large ? paged_reserve_kernel<kLarge> : paged_reserve_kernel<kSmall>;
  rc = raise_smem(kern, smem, reserve_smem(kMaxRequests), what);
  if (rc != KF_OK) return rc;
  return kf::launch_dependent_cluster(kern, cluster, dim3(cluster), dim3(large ? kLarge : kSmall), smem,
                                      static_cast<cudaStream_t>(t.stream), what, a);
}

extern "C" int kf_paged_release(const kf_paged_release_args* args) {
  const char* what = "kf_paged_release";
  if (!args) return kf::set_error(KF_ERR_INVALID, "%s: null arguments", what);
  const kf_page_tables& t = args->tables;
  int rc = check_tables(what, t);
  if (rc != KF_OK) return rc;
  if (!args->finished) return kf::set_error(KF_ERR_INVALID, "%s: null data pointer", what);
  kf::DeviceGuard guard(t.lengths);
  if (guard.status()) return guard.status();
  ReleaseArgs a;
  a.lengths = t.lengths;
  a.finished = args->finished;
  a.table = t.block_table;
  a.free_pages = t.free_pages;
  a.free_count = t.free_count;
  a.lengths_out = t.lengths_out;
  a.free_count_out = t.free_count_out;
  a.table_stride = t.table_stride;
  a.B = (int)t.B;
  a.max_pages = (uint32_t)t.max_pages;
  a.div = page_div(t.page_size);
  a.num_pages = (uint32_t)t.num_pages;
  const size_t smem = release_smem(t.B);
  const bool large = t.B > kSmall / 32;  // a warp per request
  const unsigned cluster = large ? cluster_for(t.B, kLarge / 32) : 1;
  auto kern = large ? paged_release_kernel<kLarge> : paged_release_kernel<kSmall>;
  rc = raise_smem(kern, smem, release_smem(kMaxRequests), what);
  if (rc != KF_OK) return rc;
  return kf::launch_dependent_cluster(kern, cluster, dim3(cluster), dim3(large ? kLarge : kSmall), smem,
                                      static_cast<cudaStream_t>(t.stream), what, a);
}
