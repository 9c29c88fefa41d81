// K8: rows of K and V into 8-bit pools of pages, and back.
//
// Storing reads 2 bytes and writes 1 per element of K and V, reading back the
// reverse, with a few operations between, so HBM bounds both.  A row (one
// token, one head) belongs to a group of 1 to 8 lanes with two pieces of 8
// values each; the largest magnitude goes round the group by shuffles, as
// 16-bit patterns, two at a time.
#include <type_traits>

#include "paged8.cuh"

namespace {

constexpr int kThreads = 128;

struct Rows8Args {
  uint16_t* rows[2];       // K and V: the source of a store, the destination of a load
  uint8_t* pages[2];
  uint8_t* scales[2];
  const int64_t* slots;
  int64_t rs[2][3], ps[2][3], ss[2][2];
  int64_t num_slots;
  uint32_t T, S, heads;    // tokens in all, and per batch entry
  uint32_t page_size, page_mul, page_shift;
  int chunks;              // D / 8
  int block_shift;         // log2 of the tokens of a scale
  // Blocks of several tokens: the tokens of a window, and thread blocks in front
  // that take the runs that do not fill their block (0: all take both).
  uint32_t window, front;
};

// Page and row of a slot; slots of a pool fit 31 bits unless it holds over 2^31 tokens.
__device__ __forceinline__ int64_t page_of(const Rows8Args& a, int64_t slot, uint32_t& row) {
  const int64_t page = a.num_slots <= 0x7fffffffLL ? (int64_t)(((uint64_t)(uint32_t)slot * a.page_mul) >> a.page_shift)
                                                   : slot / a.page_size;
  row = (uint32_t)(slot - page * a.page_size);
  return page;
}

__device__ __forceinline__ uint16_t* row_at(const Rows8Args& a, int w, uint32_t t, uint32_t h) {
  const uint32_t n = a.S == a.T ? 0 : t / a.S, s = t - n * a.S;
  return a.rows[w] + n * a.rs[w][0] + h * a.rs[w][1] + s * a.rs[w][2];
}

// ---------------------------------------------------------------- a scale for each row
// GROUP lanes share a row; lane c takes its 8-column pieces c and c + GROUP,
// so that every access of a warp covers whole sectors (16384 tokens 17.1 us;
// with pieces 2 c and 2 c + 1 and one 16-byte store 17.9).  One row of K and of V
// a thread: with two, fewer threads fit (18.9).
template <bool INT8, bool BF16, int GROUP>
__global__ void __launch_bounds__(kThreads) append8_kernel(const Rows8Args a) {
  kf::griddep_wait();
  kf::griddep_launch_dependents();
  const int c = threadIdx.x % GROUP;
  const uint32_t r = blockIdx.x * (kThreads / GROUP) + threadIdx.x / GROUP;
  const uint32_t token = r / a.heads, head = r - token * a.heads;
  int64_t slot = r < a.T * a.heads ? __ldcg(reinterpret_cast<const long long*>(a.slots) + token) : -1;
  if (slot >= a.num_slots) slot = -1;  // no such slot: the token is not stored
  uint4 val[2][2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint4* from = reinterpret_cast<const uint4*>(row_at(a, w, token, head)) + c;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      val[w][i] = make_uint4(0, 0, 0, 0);
      if (slot >= 0 && c + i * GROUP < a.chunks) val[w][i] = __ldcg(from + i * GROUP);
    }
  }
  uint32_t row;
  const int64_t page = page_of(a, slot < 0 ? 0 : slot, row);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint32_t m = kf::max_magnitudes(kf::magnitudes(val[w][0]), kf::magnitudes(val[w][1]));
#pragma unroll
    for (int off = 1; off < GROUP; off <<= 1) m = kf::max_magnitudes(m, __shfl_xor_sync(0xffffffffu, m, off));
    const int e = kf::scale_exponent<INT8>(kf::largest<BF16>(m));
    const bool nan = e > kf::kMaxExponent;
    const float by = nan ? 0.f : kf::power2(-e);
    uint8_t* to = a.pages[w] + page * a.ps[w][0] + head * a.ps[w][1] + row * a.ps[w][2] + c * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint2 codes = kf::encode8<INT8, BF16>(val[w][i], by);
      if (slot >= 0 && c + i * GROUP < a.chunks)
        *reinterpret_cast<uint2*>(to + i * GROUP * 8) = nan ? make_uint2(0, 0) : codes;
    }
    if (slot >= 0 && c == 0) a.scales[w][page * a.ss[w][0] + head * a.ss[w][1] + row] = (uint8_t)kf::scale_byte(e);
  }
}

// ---------------------------------------------------------------- a scale for several rows
// The tokens of a call that go to one block of rows determine its scale
// together: by their largest magnitude and, if the block has rows before the
// first of them, by its scale; if that grows, the rows before are rounded
// again.  Tokens that follow one another into a block are a run.  A warp
// takes one head of K or V of the runs that begin in a window of tokens, one
// after another, the warps of a thread block those of one window: `block`
// tokens or, in short calls, as few as one wave of thread blocks allows.
//
// Three trips to memory bound it (slots, rows with the old scale, stores), so
// slots are read once and, of blocks up to 16 tokens, rows too and kept.  (With
// slots and rows read twice 4096 tokens took 13.7 us.)  A run that does not
// fill its block may have others beside it: the warps look through all slots
// for them, once for up to 32 runs, and the first of several runs takes all of
// them, in loops that read slots and rows again.  In long calls, where most
// runs are whole blocks, thread blocks in front take those that are not, so
// that the look overlaps the rest (4096 tokens in 11 runs 10.4 us, 11.6 with
// all alike and 9.2 without a look; 16384 in 8 runs 28.5, 32 and 24.6; 1003 in
// 3 runs 6.3, 6.1 and 5.1).  Single tokens would wait for one another there
// (4096 of them 137 us, 82 with all alike), but calls of so many are rare; short
// calls, which they are mostly, take small windows (64 of them 4.4 us, 24 in
// windows of 16).
constexpr int kKept = 16;        // rows of a run that a warp keeps
constexpr int kWindowWarps = 4;  // of a thread block
constexpr int kWindowsPerSm = 7;
constexpr uint32_t kLong = 2048;  // tokens of a call with thread blocks for runs that do not fill their block
constexpr int kLook = 16;        // slots that a thread has in flight when it looks through them

// The runs of `partial` that have tokens of their block before and behind
// them, as far as this thread's slots say.  (Not inlined: it would take the
// registers that let seven thread blocks share an SM.)
__device__ __noinline__ uint2 look_through(const int64_t* slots, uint32_t T, int64_t num_slots, int shift, const uint32_t* run_block,
                                           const uint32_t* run_end, uint64_t base, uint32_t partial) {
  uint32_t earlier = 0, later = 0;
  for (uint32_t at = threadIdx.x; at < T; at += kLook * blockDim.x) {
    uint32_t block[kLook];
#pragma unroll
    for (int x = 0; x < kLook; ++x) {
      const uint32_t t = at + x * blockDim.x;
      const int64_t s = t < T ? __ldcg(reinterpret_cast<const long long*>(slots) + t) : -1;
      block[x] = s >= 0 && s < num_slots ? (uint32_t)(s >> shift) : 0xffffffffu;
    }
    for (uint32_t left = partial; left; left &= left - 1) {
      const int i = __ffs(left) - 1;
      const uint32_t own = run_block[i], begin = (uint32_t)base + i, end = run_end[i];
#pragma unroll
      for (int x = 0; x < kLook; ++x) {
        const uint32_t t = at + x * blockDim.x;
        if (block[x] == own && t < begin) earlier |= 1u << i;
        if (block[x] == own && t >= end) later |= 1u << i;
      }
    }
  }
  return make_uint2(earlier, later);
}

template <bool INT8, bool BF16>
__global__ void __launch_bounds__(kWindowWarps * 32, kWindowsPerSm) append8_blocks_kernel(const Rows8Args a) {
  constexpr int GROUP = 8, SIDE = 32 / GROUP;  // lanes of a row, rows side by side
  kf::griddep_wait();
  kf::griddep_launch_dependents();
  const int lane = threadIdx.x & 31, c = lane % GROUP, g = lane / GROUP;
  const uint32_t size = 1u << a.block_shift;
  const uint32_t parts = (2 * a.heads + kWindowWarps - 1) / kWindowWarps;  // thread blocks of a window
  const bool partly = blockIdx.x < a.front, wholly = !partly && a.front > 0;
  const uint32_t at = blockIdx.x - (wholly ? a.front : 0), turn = at / parts, hw = (at - turn * parts) * kWindowWarps + (threadIdx.x >> 5);
  const bool active = hw < 2 * a.heads;  // a warp without a head helps to look through the slots
  const uint32_t h = hw >> 1;
  const int w = hw & 1;
  const uint32_t window = partly ? max(size, 32u) : a.window;
  const uint64_t from = (uint64_t)turn * window, until = min(from + window, (uint64_t)a.T);
  auto slot_at = [&](uint64_t t) { return t < a.T ? __ldcg(reinterpret_cast<const long long*>(a.slots) + t) : -1; };
  // Blocks by their number in the pool (which memory holds fewer than 2^32 - 1 of, see the host's check).
  auto block_of = [&](int64_t s) { return s >= 0 && s < a.num_slots ? (uint32_t)(s >> a.block_shift) : 0xffffffffu; };
  __shared__ uint32_t run_block[32];     // of the runs of these 32 slots, by the lane of their first
  __shared__ uint32_t run_end[32], earlier_s, later_s;
  // Windows of up to 16 tokens see with 32 slots where their runs end.  What
  // the loop branches on is alike in all warps.
  for (uint64_t base = from; base < until; base += 32) {
    const int64_t s = slot_at(base + lane);
    int64_t before = __shfl_up_sync(0xffffffffu, (long long)s, 1);
    if (lane == 0) before = base > 0 ? slot_at(base - 1) : -2;
    const bool follows = before == s - 1 && before >> a.block_shift == s >> a.block_shift;
    const uint32_t runs_on = __ballot_sync(0xffffffffu, follows);
    const bool leads = base + lane < until && s >= 0 && s < a.num_slots && !follows;
    // Tokens of the run that this lane leads: in these slots ...
    uint32_t tokens = lane == 31 ? 1 : __ffs(~(runs_on >> (lane + 1)));
    const uint32_t goes_on = __ballot_sync(0xffffffffu, leads && lane + tokens == 32);
    if (goes_on) {                             // ... and, of one, behind them
      const int who = __ffs(goes_on) - 1;
      const int64_t s0 = __shfl_sync(0xffffffffu, (long long)s, who);
      const uint32_t room = size - (uint32_t)(s0 & (size - 1));
      uint32_t n = 32 - who;
      for (uint32_t more = 32; more == 32 && n < room;) {
        const uint32_t i = n + lane;
        const uint32_t in = __ballot_sync(0xffffffffu, i < room && slot_at(base + who + i) == s0 + (int64_t)i);
        more = in == 0xffffffffu ? 32 : __ffs(~in) - 1;
        n += more;
      }
      if (lane == who) tokens = n;
    }
    uint32_t leaders = __ballot_sync(0xffffffffu, leads), several = 0;
    const uint32_t partial = __ballot_sync(0xffffffffu, leads && tokens < size);
    if (partly) leaders &= partial;
    if (wholly) leaders &= ~partial;
    if (partial && !wholly) {
      __syncthreads();                         // the masks of the slots before have been read
      if (threadIdx.x < 32) {
        run_block[lane] = block_of(s);
        run_end[lane] = (uint32_t)base + lane + tokens;
        if (lane == 0) earlier_s = later_s = 0;
      }
      __syncthreads();
      const uint2 found = look_through(a.slots, a.T, a.num_slots, a.block_shift, run_block, run_end, base, partial);
      const uint32_t earlier = found.x, later = found.y;
      if (earlier) atomicOr(&earlier_s, earlier);
      if (later) atomicOr(&later_s, later);
      __syncthreads();
      leaders &= ~earlier_s;                   // taken with the first of them
      several = later_s;
    }
    if (!active) continue;
    for (; leaders; leaders &= leaders - 1) {
      const int who = __ffs(leaders) - 1;
      const uint32_t t0 = (uint32_t)base + who, n = __shfl_sync(0xffffffffu, tokens, who);
      const int64_t s0 = __shfl_sync(0xffffffffu, (long long)s, who);
      const uint32_t inside = (uint32_t)(s0 & (size - 1));
      const bool with_others = (several >> who) & 1;
      uint32_t row;
      const int64_t page = page_of(a, s0, row);
      // the block's first row
      uint8_t* codes = a.pages[w] + page * a.ps[w][0] + h * a.ps[w][1] + (int64_t)(row - inside) * a.ps[w][2];
      uint8_t* scale = a.scales[w] + page * a.ss[w][0] + h * a.ss[w][1] + (row >> a.block_shift);
      const uint32_t old = inside > 0 ? __ldcg(scale) : 0;
      auto source = [&](uint32_t i, int x) {
        return i < n && c + x * GROUP < a.chunks
                   ? __ldcg(reinterpret_cast<const uint4*>(row_at(a, w, t0 + i, h)) + c + x * GROUP)
                   : make_uint4(0, 0, 0, 0);
      };
      uint4 kept[kKept / SIDE][2];
#pragma unroll
      for (int k = 0; k < kKept / SIDE; ++k)
#pragma unroll
        for (int x = 0; x < 2; ++x) kept[k][x] = source(k * SIDE + g, x);
      uint32_t m = 0, first = inside;
#pragma unroll
      for (int k = 0; k < kKept / SIDE; ++k)
#pragma unroll
        for (int x = 0; x < 2; ++x) m = kf::max_magnitudes(m, kf::magnitudes(kept[k][x]));
#pragma unroll 4
      for (uint32_t i = kKept + g; i < n; i += SIDE)
#pragma unroll
        for (int x = 0; x < 2; ++x) m = kf::max_magnitudes(m, kf::magnitudes(source(i, x)));
      // act(row of the block, piece of a token's row) for the tokens of the block behind the first run
      auto others = [&](auto act) {
        for (uint64_t at = (uint64_t)t0 + n; at < a.T; at += 32) {
          const int64_t mine = slot_at(at + lane);
          uint32_t in = __ballot_sync(0xffffffffu, mine >> a.block_shift == s0 >> a.block_shift);
          for (; in; in &= in - 1) {
            const uint32_t to = (uint32_t)__shfl_sync(0xffffffffu, (long long)mine, __ffs(in) - 1) & (size - 1);
            const uint16_t* src = row_at(a, w, (uint32_t)at + __ffs(in) - 1, h);
            act(to, lane < a.chunks ? __ldcg(reinterpret_cast<const uint4*>(src) + lane) : make_uint4(0, 0, 0, 0));
          }
        }
      };
      if (with_others)
        others([&](uint32_t to, uint4 value) {
          first = min(first, to);
          m = kf::max_magnitudes(m, kf::magnitudes(value));
        });
      // (lanes may have left the loop apart from one another)
      __syncwarp();
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) m = kf::max_magnitudes(m, __shfl_xor_sync(0xffffffffu, m, off));
      int e = kf::scale_exponent<INT8>(kf::largest<BF16>(m));
      bool nan = e > kf::kMaxExponent;
      if (first > 0) {
        const int was = kf::scale_of_byte(old);
        nan |= old == kf::kNanScale;
        e = max(e, was);
        if (nan || e > was) {
          const float shift = nan ? 0.f : kf::power2(was - e);
          for (uint32_t i = g; i < first; i += SIDE)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if (c + x * GROUP >= a.chunks) continue;
              uint2* at = reinterpret_cast<uint2*>(codes + (int64_t)i * a.ps[w][2] + (c + x * GROUP) * 8);
              const uint2 y = __ldcg(at);
              float p[4], q[4];
              kf::decode4<INT8>(y.x, p);
              kf::decode4<INT8>(y.y, q);
              *at = nan ? make_uint2(0, 0)
                        : make_uint2(kf::encode4<INT8>(p[0] * shift, p[1] * shift, p[2] * shift, p[3] * shift),
                                     kf::encode4<INT8>(q[0] * shift, q[1] * shift, q[2] * shift, q[3] * shift));
            }
        }
      }
      const float by = nan ? 0.f : kf::power2(-e);
      auto put = [&](uint32_t to, int piece, uint4 value) {
        const uint2 y = kf::encode8<INT8, BF16>(value, by);
        if (piece < a.chunks)
          *reinterpret_cast<uint2*>(codes + (int64_t)to * a.ps[w][2] + piece * 8) = nan ? make_uint2(0, 0) : y;
      };
#pragma unroll
      for (int k = 0; k < kKept / SIDE; ++k)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (k * SIDE + g < n) put(inside + k * SIDE + g, c + x * GROUP, kept[k][x]);
#pragma unroll 4
      for (uint32_t i = kKept + g; i < n; i += SIDE)
#pragma unroll
        for (int x = 0; x < 2; ++x) put(inside + i, c + x * GROUP, source(i, x));
      __syncwarp();  // every lane has read the old scale
      if (with_others) others([&](uint32_t to, uint4 value) { put(to, lane, value); });
      if (lane == 0) *scale = (uint8_t)(nan ? kf::kNanScale : kf::scale_byte(e));
    }
  }
}

// ---------------------------------------------------------------- reading back
// As append8_kernel, with the tokens of a head side by side: they are
// neighbours in the page and in the output (16384 tokens 15.7 us; with 16 codes
// and two stores a lane, which cover half of each sector, 22.1).
template <bool INT8, bool BF16, int GROUP>
__global__ void __launch_bounds__(kThreads) read8_kernel(const Rows8Args a) {
  kf::griddep_wait();
  kf::griddep_launch_dependents();
  const int c = threadIdx.x % GROUP;
  const uint32_t r = blockIdx.x * (kThreads / GROUP) + threadIdx.x / GROUP;
  if (r >= a.T * a.heads) return;
  const uint32_t head = r / a.T, token = r - head * a.T;
  int64_t slot = __ldcg(reinterpret_cast<const long long*>(a.slots) + token);
  if (slot >= a.num_slots) slot = -1;
  uint32_t row;
  const int64_t page = page_of(a, slot < 0 ? 0 : slot, row);
  uint2 codes[2][2];
  uint32_t scale[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint8_t* from = a.pages[w] + page * a.ps[w][0] + head * a.ps[w][1] + row * a.ps[w][2] + c * 8;
    scale[w] = 127;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      codes[w][i] = make_uint2(0, 0);  // rows without a slot read as 0
      if (slot >= 0 && c + i * GROUP < a.chunks) codes[w][i] = __ldcg(reinterpret_cast<const uint2*>(from + i * GROUP * 8));
    }
    if (slot >= 0) scale[w] = __ldcg(a.scales[w] + page * a.ss[w][0] + head * a.ss[w][1] + (row >> a.block_shift));
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const float by = scale[w] == kf::kNanScale ? __uint_as_float(0x7fc00000u) : kf::power2(kf::scale_of_byte(scale[w]));
    uint4* to = reinterpret_cast<uint4*>(row_at(a, w, token, head)) + c;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float p[4], q[4];
      kf::decode4<INT8>(codes[w][i].x, p);
      kf::decode4<INT8>(codes[w][i].y, q);
      if (c + i * GROUP < a.chunks)
        to[i * GROUP] = make_uint4(kf::pack2<BF16>(p[0] * by, p[1] * by), kf::pack2<BF16>(p[2] * by, p[3] * by),
                                   kf::pack2<BF16>(q[0] * by, q[1] * by), kf::pack2<BF16>(q[2] * by, q[3] * by));
    }
  }
}

bool rows16(const kf_tensor4& t) {
  if (!kf::aligned16(t.ptr) || t.stride[3] != 1) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size[i] > 1 && t.stride[i] % 8 != 0) return false;
  return true;
}

// Arguments that a store and a load share: a cache, two tensors of rows, slots.
int set_up(const char* what, const kf_paged8_cache& cache, const kf_tensor4& k, const kf_tensor4& v, const int64_t* slots,
           int64_t dtype, Rows8Args* a) {
  using kf::set_error;
  if (dtype != KF_F16 && dtype != KF_BF16) return set_error(KF_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  const int rc = kf::check_cache8(what, cache);
  if (rc != KF_OK) return rc;
  for (int i = 0; i < 4; ++i)
    if (k.size[i] != v.size[i]) return set_error(KF_ERR_INVALID, "%s: the shapes of the K and V rows must match", what);
  const int64_t N = k.size[0], H = k.size[1], S = k.size[2], D = k.size[3];
  if (H != cache.k_pages.size[1] || D != cache.k_pages.size[3])
    return set_error(KF_ERR_INVALID, "%s: heads and head_dim of the rows must match the pages", what);
  if (N <= 0 || S <= 0) return set_error(KF_ERR_INVALID, "%s: dimensions must be non-zero", what);
  if (N > 0x7fffffffLL || S > 0x7fffffffLL || N * S > 0x7fffffffLL || N * S * H > 0x0fffffffLL)
    return set_error(KF_ERR_UNSUPPORTED, "%s: tensors too large", what);
  if (!k.ptr || !v.ptr || !slots) return set_error(KF_ERR_INVALID, "%s: null data pointer", what);
  if (!rows16(k) || !rows16(v))
    return set_error(KF_ERR_INVALID, "%s: K/V rows must be contiguous and 16-byte aligned", what);
  a->rows[0] = static_cast<uint16_t*>(k.ptr);
  a->rows[1] = static_cast<uint16_t*>(v.ptr);
  a->pages[0] = static_cast<uint8_t*>(cache.k_pages.ptr);
  a->pages[1] = static_cast<uint8_t*>(cache.v_pages.ptr);
  a->scales[0] = cache.k_scales;
  a->scales[1] = cache.v_scales;
  a->slots = slots;
  for (int i = 0; i < 3; ++i) {
    a->rs[0][i] = k.stride[i];
    a->rs[1][i] = v.stride[i];
    a->ps[0][i] = cache.k_pages.stride[i];
    a->ps[1][i] = cache.v_pages.stride[i];
  }
  for (int i = 0; i < 2; ++i) {
    a->ss[0][i] = cache.k_scale_strides[i];
    a->ss[1][i] = cache.v_scale_strides[i];
  }
  const int64_t page_size = cache.k_pages.size[2];
  a->num_slots = cache.k_pages.size[0] * page_size;
  a->T = (uint32_t)(N * S);
  a->S = (uint32_t)S;
  a->heads = (uint32_t)H;
  a->page_size = (uint32_t)page_size;
  kf::division(page_size, &a->page_mul, &a->page_shift);
  a->chunks = (int)(D / 8);
  a->block_shift = 0;
  while (((int64_t)1 << a->block_shift) < cache.scale_block) ++a->block_shift;
  return KF_OK;
}

template <int N>
using Number = std::integral_constant<int, N>;

// Launches kernel(lanes of a row) over all rows.
template <typename Kernel>
int launch_rows(const char* what, const Rows8Args& a, cudaStream_t st, Kernel kernel) {
  const uint64_t rows = (uint64_t)a.T * a.heads;
  auto go = [&](auto group) {
    const uint64_t per_block = kThreads / group;
    return kf::launch_dependent(kernel(group), dim3((unsigned)((rows + per_block - 1) / per_block)), dim3(kThreads), 0, st,
                                what, a);
  };
  if (a.chunks <= 2) return go(Number<1>());
  if (a.chunks <= 4) return go(Number<2>());
  if (a.chunks <= 8) return go(Number<4>());
  return go(Number<8>());
}

template <bool INT8, bool BF16>
int launch_append(Rows8Args& a, cudaStream_t st) {
  const char* what = "kf_paged8_append";
  if (a.block_shift > 0) {
    const uint32_t size = 1u << a.block_shift, parts = (2 * a.heads + kWindowWarps - 1) / kWindowWarps;
    auto blocks_of = [&](uint32_t window) { return ((uint64_t)a.T + window - 1) / window * parts; };
    a.window = size;
    a.front = 0;
    if (a.T >= kLong)
      a.front = (uint32_t)blocks_of(size < 32 ? 32 : size);
    else
      while (a.window > 1 && blocks_of(a.window / 2) <= (uint64_t)kWindowsPerSm * kf::sm_count_current_device()) a.window /= 2;
    const unsigned blocks = (unsigned)(a.front + blocks_of(a.window));
    return kf::launch_dependent(append8_blocks_kernel<INT8, BF16>, dim3(blocks), dim3(kWindowWarps * 32), 0, st, what, a);
  }
  return launch_rows(what, a, st, [](auto group) { return append8_kernel<INT8, BF16, group>; });
}

template <bool INT8, bool BF16>
int launch_read(const Rows8Args& a, cudaStream_t st) {
  return launch_rows("kf_paged8_read", a, st, [](auto group) { return read8_kernel<INT8, BF16, group>; });
}

}  // namespace

namespace kf {

int check_cache8(const char* what, const kf_paged8_cache& c) {
  const kf_tensor4 &k = c.k_pages, &v = c.v_pages;
  if (c.format != KF_E4M3 && c.format != KF_INT8)
    return set_error(KF_ERR_INVALID, "%s: pages must be e4m3 or int8", what);
  for (int i = 0; i < 4; ++i)
    if (k.size[i] != v.size[i]) return set_error(KF_ERR_INVALID, "%s: K/V page shapes must match", what);
  const int64_t D = k.size[3], page_size = k.size[2], block = c.scale_block;
  if (k.size[0] <= 0 || k.size[1] <= 0 || page_size <= 0)
    return set_error(KF_ERR_INVALID, "%s: dimensions must be non-zero", what);
  if (D < 16 || D > 128 || D % 8 != 0)
    return set_error(KF_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 in [16, 128]", what);
  if (page_size > (1 << 20) || k.size[0] > 0x7fffffffLL || k.size[1] > (1 << 16))
    return set_error(KF_ERR_UNSUPPORTED, "%s: tensors too large", what);
  if (block <= 0 || block > 128 || (block & (block - 1)) || page_size % block)
    return set_error(KF_ERR_INVALID, "%s: the tokens of a scale must be a power of two up to 128 that divides page_size", what);
  for (const kf_tensor4* t : {&k, &v}) {
    bool good = aligned16(t->ptr) && t->stride[3] == 1;
    for (int i = 0; i < 3; ++i)
      if (t->size[i] > 1 && (t->stride[i] % 16 != 0 || t->stride[i] <= 0)) good = false;
    if (!good) return set_error(KF_ERR_INVALID, "%s: pages need a contiguous last dim and 16-byte aligned rows", what);
  }
  if (!k.ptr || !v.ptr || !c.k_scales || !c.v_scales) return set_error(KF_ERR_INVALID, "%s: null data pointer", what);
  return KF_OK;
}

}  // namespace kf

extern "C" int kf_paged8_append(const kf_paged8_append_args* args) {
  const char* what = "kf_paged8_append";
  if (!args) return kf::set_error(KF_ERR_INVALID, "%s: null arguments", what);
  Rows8Args a;
  const int rc = set_up(what, args->cache, args->new_k, args->new_v, args->slots, args->dtype, &a);
  if (rc != KF_OK) return rc;
  if (a.block_shift > 0 && (a.num_slots >> a.block_shift) >= 0xffffffffLL)  // (twice what memory holds)
    return kf::set_error(KF_ERR_UNSUPPORTED, "%s: tensors too large", what);
  kf::DeviceGuard guard(args->cache.k_pages.ptr);
  if (guard.status()) return guard.status();
  cudaStream_t st = static_cast<cudaStream_t>(args->stream);
  if (args->cache.format == KF_INT8)
    return args->dtype == KF_BF16 ? launch_append<true, true>(a, st) : launch_append<true, false>(a, st);
  return args->dtype == KF_BF16 ? launch_append<false, true>(a, st) : launch_append<false, false>(a, st);
}

extern "C" int kf_paged8_read(const kf_paged8_read_args* args) {
  const char* what = "kf_paged8_read";
  if (!args) return kf::set_error(KF_ERR_INVALID, "%s: null arguments", what);
  Rows8Args a;
  const int rc = set_up(what, args->cache, args->k_out, args->v_out, args->slots, args->dtype, &a);
  if (rc != KF_OK) return rc;
  kf::DeviceGuard guard(args->cache.k_pages.ptr);
  if (guard.status()) return guard.status();
  cudaStream_t st = static_cast<cudaStream_t>(args->stream);
  if (args->cache.format == KF_INT8)
    return args->dtype == KF_BF16 ? launch_read<true, true>(a, st) : launch_read<true, false>(a, st);
  return args->dtype == KF_BF16 ? launch_read<false, true>(a, st) : launch_read<false, false>(a, st);
}
