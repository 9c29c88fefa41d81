// K9: attention of one new token per request over an 8-bit paged K/V cache,
// split over the cache's length and joined, with an optional fused append.
//
// With codes k^, v^ and the scales' exponents e, f of position j, and x_j =
// scale q.k^_j 2^e_j in base 2:
//   l = sum 2^x_j,  O = sum 2^(x_j + f_j) v^_j / l,  LSE = ln l.
// Weights 2^(x_j + f_j - m) carry V's scale as a part of the exponent, with m
// a running reference of x_j + f_j: whatever the scales, the key that adds
// most to O has a weight at the top of fp16's range.  So codes enter the
// products as they are, exact in fp16, and K's scale is one factor of a score.
// l is summed in 32 bits, as 2^(x_j - m) from an exponential of its own: a key
// with a small V can lie far below m and weigh more than all others.  The key
// at the reference has x - m >= 11 - 60 and no key x - m > 15 + 60, so l lies
// between 2^-49 and 2^75 times the number of keys, and what is lost below
// 2^-126 is less than 2^-77 of it per key.
//
// Every K/V row is read once for G query rows, 2 D bytes for 4 G D flops, so
// HBM bounds it up to about 16 rows per KV head; at half the bytes of a 16-bit
// cache, the latency of a step and the conversions are the next bound.
//
// The split over blocks, teams and rings is paged_decode.cu's (see there and
// paged_split.cuh).  What differs, for a team of warps:
// - A step takes 32 keys of the longest rows, 64 or 128 of shorter ones: half of
//   a microsecond of a step does not depend on its keys (32 requests of 8192
//   keys, D = 64, with two blocks to an SM: 69 us with 32 a step, 56 with 64).
// - One TMA load brings a box of keys of both K and V where the two pools have
//   the same strides: the pair is a dimension of the tensor map, as long as the
//   distance of the pools.  (A load takes a lane about 66 cycles to issue.)
// - K is loaded by ldmatrix as pairs of bytes: a lane gets columns 4 c .. 4 c +
//   3 of a key, which after conversion are the columns that a lane holds for k
//   = 2 c, 2 c + 1 and 2 c + 8, 2 c + 9, so Q is loaded in that order.  V comes
//   through the 8-bit transposing ldmatrix: a lane gets keys 4 c .. 4 c + 3 of
//   a column, and rows of K are taken in the order that makes P^T match.
// - Q of bf16 is brought to fp16 by a power of two per row: exact for elements
//   down to 2^-30 of the row's largest, off by 2^-39 of it below.
// - Scales are read by the lane that looks a key's page up, a step after its
//   page, and kept as (2^e, f) beside the ring.
#pragma once
#include <float.h>

#include <type_traits>

#include "paged8.cuh"
#include "paged_split.cuh"

namespace {

struct Paged8Args : PagedWork {
  const uint16_t* q;
  uint8_t* k;              // written only by the fused append
  uint8_t* v;
  uint8_t* ks_;            // scales
  uint8_t* vs_;
  const uint16_t* nk;      // null: no fused append
  const uint16_t* nv;
  const int64_t* slots;    // of the new rows; < 0: this request has none
  int64_t qs[2], ks[3], vs[3], nks[2], nvs[2];
  int64_t kss[2], vss[2];  // strides of the scales
  int block_shift;         // log2 of the tokens of a scale
  int box;                 // keys of a TMA box
  int group;               // keys whose K rows and then V rows lie together in a tile: 16 or more, box or more
  int k_plane, v_plane;    // 0 and 1, or 1 and 0: which of the two lies first
  bool paired;             // one load brings both
  float scale_log2;        // scale log2(e)
};

// Blocks per SM.  Three where registers allow it without a spill and the
// conversions and the latency of a step, not HBM, set the pace (D = 64: 32
// requests of 8192 keys 57 -> 52 us, two of 100000 with 32 heads 45.6 -> 41.4);
// two for longer rows, where three ask for more than HBM gives and end far
// apart (D = 128: 86.5 -> 109), and shorter ones, whose 128 keys a step want
// the registers (D = 32, with weights in one part: 42 -> 52).
constexpr int blocks_per_sm(int steps, int rows) { return steps == 4 && rows == 8 ? 3 : 2; }

// Variants: KD = 16-column chunks of the head dim; LINES: pages are brought as
// lines of 128 bytes, keys lie KD * 16 bytes apart (otherwise KD is 8, each row
// has a line of the tile, comes in chunks of 16 bytes, and the chunks are counted
// at run time); NT = 8-row tiles of query
// rows per warp; RG = warps of a team.
template <int KD, int NT, int RG>
struct Cfg8 {
  static constexpr int KW = KD <= 3 ? 128 : KD <= 6 ? 64 : 32;  // keys a team takes of a tile
  static constexpr int TEAMS = kWarps / RG;
  static constexpr int TILE = TEAMS * KW;
  static constexpr int ROWS = NT * 8 * RG;                   // query rows of a unit
  static constexpr int PITCH = KD * 16;                      // bytes from key to key
  static constexpr int STAGE = KW * PITCH * 2;               // K and V rows
  static constexpr int BLOCKS = blocks_per_sm(KD, ROWS);
  static constexpr int FIT = 196608 / BLOCKS / (TEAMS * STAGE);  // of 192 KB of ring per SM
  static constexpr int MOST = KD == 1 ? 4 : 8;                // (six of the shortest rows do not fit with their scales)
  static constexpr int STAGES = FIT < MOST ? FIT : MOST;
  static constexpr int SHALLOW = STAGES / 3 > 1 ? STAGES / 3 : 1;
  static constexpr bool SWIZZLE = KD == 2 || KD == 4 || KD == 8;
  static constexpr int HANDED = KD * 4 * 32;                 // floats of a warp's O^T of one row tile
  static constexpr int SCALES = TEAMS * STAGES * KW * 8;     // bytes
  // All of it is dynamic, with the ring, which wants to begin on 1024 bytes, in front.
  struct Tail {
    uint64_t full[TEAMS][STAGES];
    uint32_t seen[TEAMS][STAGES][KW / 32];                   // visible keys of each stage
    uint32_t nan[TEAMS][STAGES][KW / 32];                    // keys whose V has the scale NaN
    ShareScratch scratch;
    int abort_any;
  };
  static constexpr int SMEM =
      TEAMS * STAGES * STAGE + SCALES + (TEAMS > 1 ? 2 * HANDED + kWarps * NT * 32 : 0) * 4 + (int)sizeof(Tail);
};

// A tile holds keys as a page does, one behind the other, brought as lines of
// 128 bytes whatever a row's length: a TMA load of rows takes a cycle for each
// row and each sector of 32 bytes that it touches, which rows of 64 to 96 bytes
// pay more for than for HBM.  Where a row's chunks of 16 bytes are even in
// number the lines are swizzled; where they are odd, keys lie on different
// banks as they are (and six chunks apart, on pairs of them).
template <bool SWIZZLE>
__device__ __forceinline__ uint32_t swizzled(uint32_t at) {
  return SWIZZLE ? at ^ ((at >> 3) & 0x70u) : at;
}

// The key of a 16-key part that stands in place x of a product.  V's fragments
// hold keys 4 c .. 4 c + 3 of a lane, so K's two 8 x 8 parts take places {0, 1,
// 4, 5, ..} and {2, 3, 6, 7, ..}; with this order of keys both those and eight
// places in a row lie on different banks.
__device__ __forceinline__ int key_of(int x) { return x ^ ((x >> 2) & 2); }

// x4 over two 16 x 16 matrices of bytes, transposed: lane l gets of each
// column l / 4 (then l / 4 + 8) rows 4 (l % 4) .. + 3.
__device__ __forceinline__ void ldmatrix_trans_b8(uint32_t (&r)[4], uint32_t saddr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(saddr));
}

// A scale, and the rest of its line of 128 bytes to L2: the other heads of the
// page, which other blocks ask for at about the same time.
__device__ __forceinline__ uint32_t load_scale(const uint8_t* p) {
  uint32_t x;
  asm volatile("ld.global.cg.L2::128B.u8 %0, [%1];" : "=r"(x) : "l"(p));
  return x;
}

template <bool INT8, bool BF16, int KD, bool LINES, int NT, int RG>
__global__ void __launch_bounds__(kThreads, (Cfg8<KD, NT, RG>::BLOCKS))
paged8_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const Paged8Args a) {
  using C = Cfg8<KD, NT, RG>;
  constexpr int KW = C::KW, STAGES = C::STAGES, TILE = C::TILE;
  constexpr int H = KW / 16;           // 16-key parts of a step
  constexpr int LOOKS = KW / 32;       // keys that a lane looks up
  constexpr int PAIRS = (KD + 1) / 2;  // pairs of chunks
  // Weights lie between 2^BELOW and 2^LIMIT at the row's largest x + f, the
  // top of fp16's range: its 11 bits hold down to 2^-25 of the largest, and
  // what is lost below is at most 2^-36 of it.
  constexpr float BELOW = 11.f, LIMIT = 15.f;
  extern __shared__ __align__(1024) uint8_t smem[];
  typename C::Tail& tail = *reinterpret_cast<typename C::Tail*>(smem + C::SMEM - sizeof(typename C::Tail));
  auto& full = tail.full;
  auto& seen_s = tail.seen;
  auto& nan_s = tail.nan;
  int& abort_any = tail.abort_any;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int team = warp / RG, rg = warp % RG;
  const int units = a.Hkv * a.row_blocks;  // per request
  uint8_t* ring = smem + team * STAGES * C::STAGE;
  float2* scales = reinterpret_cast<float2*>(smem + C::TEAMS * STAGES * C::STAGE) + team * STAGES * KW;  // (2^e, f)
  float* handed = reinterpret_cast<float*>(smem + C::TEAMS * STAGES * C::STAGE + C::SCALES);  // [2][KD][lane][4]
  float* ml = handed + 2 * C::HANDED;  // [warp][NT][4 lanes][2 rows](m, l, NaN if V has one, -)

  if (tid == 0) {
    for (int i = 0; i < C::TEAMS * STAGES; ++i) kf::mbar_init(&full[0][0] + i, LINES ? 1 : 32);
    kf::fence_barrier_init();
    abort_any = 0;
    if constexpr (LINES) {
      kf::tma_prefetch_desc(&map_k);
      kf::tma_prefetch_desc(&map_v);
    }
  }
  // The chain lengths -> table -> K/V starts cold: hints while the previous
  // kernel still runs.
  {
    const uint32_t line = blockIdx.x * kThreads + tid;  // of 32 entries
    if (line * 32 < (uint32_t)a.B) prefetch_l2(a.lengths + line * 32);
    const uint32_t lines_per_row = (a.max_pages + 31) / 32, b = line / lines_per_row;
    if (b < (uint32_t)a.B) prefetch_l2(a.table + b * a.table_stride + (line - b * lines_per_row) * 32);
    const uint32_t request = line / a.Hq;
    if (request < (uint32_t)a.B)
      kf::prefetch_l2_bulk(a.q + request * a.qs[0] + (line - request * a.Hq) * a.qs[1], a.D * 2);
  }
  constexpr int PITCH = C::PITCH;
  const int chunks = LINES ? KD : (a.D + 15) / 16;
  // Where key r's chunk c lies in a stage: groups of keys, K rows and then V
  // rows (or V rows first) of each.
  const uint32_t k_base = (uint32_t)(a.k_plane * a.group * PITCH), v_base = (uint32_t)(a.v_plane * a.group * PITCH);
  auto place = [&](int r, int c, uint32_t base) {
    const int inside = r & (a.group - 1);
    return swizzled<C::SWIZZLE>(base + (uint32_t)((2 * r - inside) * PITCH + c * 16));
  };
  // Offsets of a lane's ldmatrix rows, by pair of chunks; a missing second
  // chunk repeats the first.
  uint32_t k_off[PAIRS], v_off[PAIRS];
#pragma unroll
  for (int x = 0; x < PAIRS; ++x) {
    const int i = lane & 7, c = min(2 * x + (lane >> 4), chunks - 1);
    k_off[x] = place(key_of(4 * (i >> 1) + (i & 1) + ((lane >> 3) & 1) * 2), c, k_base);
    v_off[x] = place(key_of(lane & 15), c, v_base);
  }
  // From a 16-key part to the next, the one after and the fourth; in lines of
  // four keys a step of 512 bytes swizzles the other way about.
  const uint32_t step1 = (a.group > 16 ? 16 : 32) * PITCH, step2 = (a.group > 32 ? 32 : 64) * PITCH,
                 step4 = (a.group > 64 ? 64 : 128) * PITCH;
  const uint32_t flip = C::SWIZZLE && PITCH == 32 && a.group > 16 ? 64u : 0u;
  auto part = [&](uint32_t off, int h) {
    return (PITCH == 32 && (h & 1) ? off ^ flip : off) + (h & 1 ? step1 : 0) + (h & 2 ? step2 : 0) + (h & 4 ? step4 : 0);
  };
  // Half a chunk at the end of a row: what lies behind it can be a code of NaN,
  // which Q's zeros do not silence.
  const uint32_t edge = (a.D & 8) && (lane & 3) >= 2 ? 0u : 0xffffffffu;
  kf::griddep_wait();
  kf::griddep_launch_dependents();

  const uint32_t me = blockIdx.x;
  const bool join_blocks = a.joins && !a.join_units;
  Share share;
  Cursor<TILE> load, work;
  if (!find_share<TILE>(a, tail.scratch, share) || !first_tile(a, share, work)) {
    if (tid == 0 && join_blocks) a.joins[me].x = -1;
    clear_empty(a);
    return;
  }
  const uint32_t end = share.end;
  load = work;

  // ---- loads: a lane looks up keys lane, lane + 32, .. of the team's share of a tile
  struct Place {
    uint32_t page[LOOKS], row[LOOKS];
    int h;
  };
  // K/V rows leave L2 first, to the scales' lines: 32 requests of 8192 keys
  // 86.8 us, 94.4 without.  Where rows are read again it makes no difference (the
  // same with 7168 of them in pages that all share 85.1 and 85.3; 8 requests of
  // 32768 keys with 72 query rows per KV head, in two row blocks, 219 and 219).
  const uint64_t once = kf::l2_evict_first();
  auto look_up = [&]() {
    Place p;
    p.h = load.h;
#pragma unroll
    for (int i = 0; i < LOOKS; ++i) {
      const uint32_t key = load.t * TILE + team * KW + i * 32 + lane;
      const uint32_t pg = (uint32_t)(((uint64_t)key * a.page_mul) >> a.page_shift);
      p.row[i] = key - pg * a.page_size;
      p.page[i] = key < load.keys ? (uint32_t)a.table[load.b * a.table_stride + pg] : 0xffffffffu;
    }
    return p;
  };
  struct Scale {
    uint32_t k[LOOKS], v[LOOKS];       // bytes; 256: no such key
  };
  auto issue = [&](int stage, const Place& p, Scale& s) {
    uint32_t seen[LOOKS], boxes = 0;
    bool starts[LOOKS];
#pragma unroll
    for (int i = 0; i < LOOKS; ++i) {
      const bool valid = p.page[i] < a.num_pages;
      seen[i] = __ballot_sync(0xffffffffu, valid);
      starts[i] = valid && ((i * 32 + lane) & (a.box - 1)) == 0;
      boxes += __popc(__ballot_sync(0xffffffffu, starts[i]));
    }
    uint64_t* bar = &full[team][stage];
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < LOOKS; ++i) seen_s[team][stage][i] = seen[i];
      if constexpr (LINES) kf::mbar_arrive_expect_tx(bar, boxes * (uint32_t)(a.box * PITCH * 2));
    }
    __syncwarp();
    if constexpr (!LINES) {
      // The rows' own chunks, with no byte besides; neighbouring lanes take those
      // of one row (a row per lane: half of each sector at a time).
      const int64_t k_at = p.page[0] * a.ks[0] + p.h * a.ks[1] + p.row[0] * a.ks[2];
      const int64_t v_at = p.page[0] * a.vs[0] + p.h * a.vs[1] + p.row[0] * a.vs[2];
      const uint32_t st = kf::smem_u32(ring + stage * C::STAGE), per_row = (65536 + chunks - 1) / chunks;
#pragma unroll 2
      for (int i = 0; i < chunks; ++i) {
        const uint32_t x = i * 32 + lane, r = x * per_row >> 16, c = x - r * chunks;  // of 32 chunks: exact
        const int64_t k = __shfl_sync(0xffffffffu, (long long)k_at, r), v = __shfl_sync(0xffffffffu, (long long)v_at, r);
        if ((seen[0] >> r) & 1) {
          kf::cp_async16(st + place(r, c, k_base), a.k + k + c * 16);
          kf::cp_async16(st + place(r, c, v_base), a.v + v + c * 16);
        }
      }
      kf::cp_async_mbar_arrive(bar);   // of each lane, once its copies are there
    }
#pragma unroll
    for (int i = 0; i < LOOKS; ++i) {
      if (LINES && starts[i]) {
        const int r = i * 32 + lane, inside = r & (a.group - 1);
        uint8_t* st = ring + stage * C::STAGE + (2 * r - inside) * PITCH;
        const int line = (int)(p.row[i] * (uint32_t)KD >> 3);
        if (a.paired) {
          kf::tma_load_5d_once(st, &map_k, bar, 0, line, 0, p.h, p.page[i], once);
        } else {
          kf::tma_load_5d_once(st + k_base, &map_k, bar, 0, line, 0, p.h, p.page[i], once);
          kf::tma_load_5d_once(st + v_base, &map_v, bar, 0, line, 0, p.h, p.page[i], once);
        }
      }
      s.k[i] = s.v[i] = 256;
      if (p.page[i] < a.num_pages) {
        const uint32_t r = p.row[i] >> a.block_shift;
        s.k[i] = load_scale(a.ks_ + p.page[i] * a.kss[0] + p.h * a.kss[1] + r);
        s.v[i] = load_scale(a.vs_ + p.page[i] * a.vss[0] + p.h * a.vss[1] + r);
      }
    }
  };
  // the scales of a tile that was issued a step before, to where its readers find them
  auto keep = [&](int stage, const Scale& s) {
#pragma unroll
    for (int i = 0; i < LOOKS; ++i) {
      const float k = s.k[i] == kf::kNanScale ? NAN : kf::power2(kf::scale_of_byte(s.k[i]));
      const float f = s.v[i] >= kf::kNanScale ? 0.f : (float)kf::scale_of_byte(s.v[i]);
      scales[stage * KW + i * 32 + lane] = make_float2(k, f);
      const uint32_t nan = __ballot_sync(0xffffffffu, s.v[i] == kf::kNanScale);
      if (lane == 0) nan_s[team][stage][i] = nan;
    }
  };

  // (an index within KD for what odd numbers of chunks do not use)
  constexpr auto last = [](int x) { return x < KD ? x : KD - 1; };

  // ---- state of the unit being worked on
  uint32_t qb[NT][KD][2];              // Q^T as B fragments
  // rows 2 (lane % 4) + {0, 1} of each row tile: the factor of a product, the
  // reference m of the weights 2^(x + f - m), the sum of 2^(x - m), and m as it
  // enters the exponent (0 for -inf)
  float factor[NT][2], m_run[NT][2], l_run[NT][2], mu[NT][2];
  float ot[NT][KD][4];                 // O^T
  bool v_nan = false;
  // The loads of the unit's Q, issued early.  start_unit() follows where the
  // unit begins.
  auto load_q = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = work.rb * C::ROWS + rg * NT * 8 + nt * 8 + (lane >> 2);
      const uint16_t* src = a.q + work.b * a.qs[0] + (int64_t)(work.h * a.G + row) * a.qs[1] + 4 * (lane & 3);
#pragma unroll
      for (int x = 0; x < KD; ++x) {
        qb[nt][x][0] = qb[nt][x][1] = 0u;
        if (row < a.G && x * 16 + 4 * (lane & 3) < a.D)
          asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(qb[nt][x][0]), "=r"(qb[nt][x][1]) : "l"(src + x * 16));
      }
    }
  };
  auto start_unit = [&]() {
    v_nan = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float back = 1.f;                // of row lane / 4: what its factor makes up for
      if constexpr (BF16) {
        uint32_t m = 0;
#pragma unroll
        for (int x = 0; x < KD; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) m = kf::max_magnitudes(m, qb[nt][x][e] & 0x7fff7fffu);
        m = kf::max_magnitudes(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = kf::max_magnitudes(m, __shfl_xor_sync(0xffffffffu, m, 2));
        // largest element to [2^14, 2^15), as far as a power of two in 32 bits does it
        const int up = 14 - max((int)(max(m & 0xffffu, m >> 16) >> 7) - 127, -100);
        const float by = kf::power2(up);
        back = kf::power2(-up);
#pragma unroll
        for (int x = 0; x < KD; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 y = kf::unpack2<true>(qb[nt][x][e]);
            qb[nt][x][e] = kf::pack2<false>(y.x * by, y.y * by);
          }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        factor[nt][j] = a.scale_log2 * __shfl_sync(0xffffffffu, back, 8 * (lane & 3) + 4 * j);
        m_run[nt][j] = -INFINITY;
        l_run[nt][j] = mu[nt][j] = 0.f;
      }
#pragma unroll
      for (int x = 0; x < KD; ++x) ot[nt][x][0] = ot[nt][x][1] = ot[nt][x][2] = ot[nt][x][3] = 0.f;
    }
  };

  load_q();
  // Tiles loaded ahead of the one in use: all of the ring where units are short
  // and drain it at each end, and where shares are long (32 requests of 8192
  // keys 86.8 us, 89.1 with a third of it); else a third, since whoever comes
  // first in a short call would take the others' bandwidth (8 requests of 4200
  // keys 19.6 us, 20.3 with all of it).
  const int depth = share.even < 32 && share.total >= 10u * a.B ? C::SHALLOW : STAGES - 1;
  // The first warp of a team loads.  To begin with it looks up the pages of the
  // whole ring at once, then always one step ahead of their use.
  bool more = rg == 0;                 // whether the load cursor stands on a tile that is not loaded yet
  int issued = 0, late = -1;           // `late`: stage whose scales are on their way
  Place ahead;
  Scale coming, got[STAGES - 1];
  if (rg == 0) {
    Place first[STAGES - 1];
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      if (more && s < depth) {
        first[s] = look_up();
        issued = s + 1;
        more = load.more(end);
        if (more) load.next(a);
      }
    }
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
      if (s < issued) issue(s, first[s], got[s]);
    if (more) ahead = look_up();
  }
  uint32_t unit_t0 = work.t;           // first tile of the unit in this share
  if (tid == 0 && join_blocks) a.joins[me].x = -1;
  clear_empty(a);
  start_unit();
  if (rg == 0) {
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
      if (s < issued) keep(s, got[s]);
  }

  int stage = 0, fill = depth;
  uint32_t parity = 0;
  bool alive = true;                   // false once a wait of this block has expired
  for (bool going = true; going;) {
    // scales that were asked for a step ago; their stage's last readers left it before it was issued
    if (rg == 0 && late >= 0) keep(late, coming);
    late = -1;
    bool landed = kf::mbar_try_wait(&full[team][stage], parity);
    if (!landed) landed = alive && !*(volatile int*)&abort_any && kf::mbar_wait(&full[team][stage], parity, a.status);
    // One outcome for the team: no lane reaches a collective instruction alone.
    // The barrier also says that the team has left stage i - 1.
    __syncwarp();
    alive = team_and<RG>(team, alive && landed);
    if (!alive && lane == 0) *(volatile int*)&abort_any = 1;
    uint32_t seen[LOOKS], any = 0, all = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < LOOKS; ++i) {
      seen[i] = alive ? seen_s[team][stage][i] : 0u;
      any |= seen[i];
      all &= seen[i];
    }
    auto sees = [&](uint32_t key) {
      uint32_t word = seen[0];
#pragma unroll
      for (int i = 1; i < LOOKS; ++i) word = key >> 5 == i ? seen[i] : word;
      return ((word >> (key & 31)) & 1) != 0;
    };
    if (rg == 0 && alive && more) {
      issue(fill, ahead, coming);
      late = fill;
      ++issued;
      more = load.more(end);
      if (more) {
        load.next(a);
        ahead = look_up();
      }
    }

    uint8_t* tile = ring + stage * C::STAGE;
    const uint32_t key0 = work.t * TILE + team * KW;
    if (any != 0 && (all != 0xffffffffu || (a.nk && key0 + KW >= work.keys))) {
      // The end of a request or pages without a table entry.  Rows that nobody
      // sees hold anything: their scores are replaced below, their V rows must
      // be zero (a code can be NaN).  A new row takes its place here and goes
      // to its page, in 8 bits.
#pragma unroll
      for (int x = rg; x < KW / 4; x += RG) {
        const int r = 4 * x + (lane >> 3);
        clear16(kf::smem_u32(tile) + place(r, lane & 7, v_base), (lane & 7) * 16 < PITCH && !sees(r));
      }
      const uint32_t r = work.keys - 1 - key0;  // the newest position, unless the table is too short for it
      if (a.nk && r < (uint32_t)KW && sees(r) && work.whole && a.slots[work.b] >= 0 && rg == 0) {
        const int c = lane & 15;       // 8 columns of K (lanes 0 to 15) or V
        const bool is_v = lane >= 16;
        const uint32_t pg = (uint32_t)(((uint64_t)(key0 + r) * a.page_mul) >> a.page_shift);
        const int64_t page = a.table[work.b * a.table_stride + pg], row = key0 + r - pg * a.page_size;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (c < a.D / 8)
          x = __ldcg(reinterpret_cast<const uint4*>(is_v ? a.nv + work.b * a.nvs[0] + work.h * a.nvs[1]
                                                         : a.nk + work.b * a.nks[0] + work.h * a.nks[1]) + c);
        uint32_t m = kf::magnitudes(x);
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) m = kf::max_magnitudes(m, __shfl_xor_sync(0xffffffffu, m, off));
        const int e = kf::scale_exponent<INT8>(kf::largest<BF16>(m));
        const bool nan = e > kf::kMaxExponent;
        const float by = nan ? 0.f : kf::power2(-e);
        uint2 codes = kf::encode8<INT8, BF16>(x, by);
        if (nan) codes = make_uint2(0, 0);
        if (c < a.D / 8) {
          *reinterpret_cast<uint2*>(tile + place((int)r, c >> 1, is_v ? v_base : k_base) + (c & 1) * 8) = codes;
          if (work.rb == 0)
            *reinterpret_cast<uint2*>(is_v ? a.v + page * a.vs[0] + work.h * a.vs[1] + row * a.vs[2] + c * 8
                                           : a.k + page * a.ks[0] + work.h * a.ks[1] + row * a.ks[2] + c * 8) = codes;
        }
        if (c == 0) {
          float* at = reinterpret_cast<float*>(scales + stage * KW + r) + (is_v ? 1 : 0);
          *at = is_v ? (nan ? 0.f : (float)e) : (nan ? NAN : kf::power2(e));
          if (work.rb == 0)
            (is_v ? a.vs_ + page * a.vss[0] + work.h * a.vss[1] : a.ks_ + page * a.kss[0] + work.h * a.kss[1])[row] =
                (uint8_t)kf::scale_byte(e);
        }
        // what the slot's byte said before does not count, what the new row says does
        const uint32_t v_is_nan = __shfl_sync(0xffffffffu, (uint32_t)nan, 16);
        if (lane == 0) {
          uint32_t& word = nan_s[team][stage][r >> 5];
          word = (word & ~(1u << (r & 31))) | (v_is_nan << (r & 31));
        }
      }
      kf::fence_proxy_async_smem();    // before a later load into this stage
      __syncwarp();                    // (the vote of a team of one warp orders no memory)
      team_and<RG>(team, true);
    }
    if (any != 0) {
#pragma unroll
      for (int i = 0; i < LOOKS; ++i) v_nan |= nan_s[team][stage][i] != 0;
      const uint32_t st = kf::smem_u32(tile);
      // S^T (keys x rows)
      float cc[H][NT][4];
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) cc[h][nt][0] = cc[h][nt][1] = cc[h][nt][2] = cc[h][nt][3] = 0.f;
#pragma unroll
      for (int x = 0; x < PAIRS; ++x) {
        if (!LINES && 2 * x >= chunks) continue;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          uint32_t w[4], f[2][4];
          kf::ldmatrix_x4(w, st + part(k_off[x], h));
          if (2 * x + 1 == chunks) w[0] &= edge, w[1] &= edge;
          if (2 * x + 2 == chunks) w[2] &= edge, w[3] &= edge;
          kf::decode4<INT8>(w[0], f[0][0], f[0][2]);
          kf::decode4<INT8>(w[1], f[0][1], f[0][3]);
          kf::decode4<INT8>(w[2], f[1][0], f[1][2]);
          kf::decode4<INT8>(w[3], f[1][1], f[1][3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) kf::mma_16816<false>(cc[h][nt], f[0], qb[nt][2 * x][0], qb[nt][2 * x][1]);
          if (2 * x + 1 < chunks) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              kf::mma_16816<false>(cc[h][nt], f[1], qb[nt][last(2 * x + 1)][0], qb[nt][last(2 * x + 1)][1]);
          }
        }
      }
      // Scores with V's exponent: places 16 h + 4 (g / 2) + g % 2 (+ 2 for the
      // second pair of a fragment), g = lane / 4, of rows 2 (lane % 4) + {0, 1}.
      const int g = lane >> 2;
      const int own_key[2] = {key_of(4 * (g >> 1) + (g & 1)), key_of(4 * (g >> 1) + (g & 1) + 2)};
      float own_f[H][2];
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int key = h * 16 + own_key[y];
          const float2 s = scales[stage * KW + key];
          own_f[h][y] = s.y;
          const uint64_t sx = kf::f2(s.x, s.x), sy = kf::f2(s.y, s.y);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint64_t v = kf::f2(cc[h][nt][2 * y], cc[h][nt][2 * y + 1]);
            v = kf::mul2(v, sx);
            kf::f2_split(kf::fma2(v, kf::f2(factor[nt][0], factor[nt][1]), sy), cc[h][nt][2 * y], cc[h][nt][2 * y + 1]);
          }
        }
      if (all != 0xffffffffu) {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            if (!((seen[h >> 1] >> ((h & 1) * 16 + own_key[y])) & 1)) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) cc[h][nt][2 * y] = cc[h][nt][2 * y + 1] = -INFINITY;
            }
      }
      // The reference of a row follows its maximum only when a score passes it
      // by LIMIT.
      bool raise = false;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[nt][j] = fmaxf(cc[0][nt][j], cc[0][nt][2 + j]);
#pragma unroll
          for (int h = 1; h < H; ++h) top[nt][j] = kf::fmax3(top[nt][j], cc[h][nt][j], cc[h][nt][2 + j]);
          raise |= top[nt][j] - m_run[nt][j] > LIMIT;
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float t = top[nt][j];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, off));
            const float m_new = fmaxf(m_run[nt][j], t - BELOW);
            mu[nt][j] = m_new == -INFINITY ? 0.f : m_new;
            const float old = kf::ex2(m_run[nt][j] - mu[nt][j]);
            // (in two halves: where m leaps, `old` can be 0 and a sum of keys with small values not)
            const float half = kf::ex2(0.5f * (m_run[nt][j] - mu[nt][j]));
            m_run[nt][j] = m_new;
            l_run[nt][j] = l_run[nt][j] * half * half;
#pragma unroll
            for (int dm = 0; dm < KD; ++dm) {
              ot[nt][dm][j] *= old;
              ot[nt][dm][2 + j] *= old;
            }
          }
      }
      // Weights in two parts of fp16, 11 bits each: cut, and what was cut off.
      // One part alone is off by 2^-11: 1.5 times the error of an fp16 O, an
      // eighth of a bf16 O's rounding (64 ragged requests in bf16 86.5 us instead
      // of 88.7, 16 query rows per KV head 105 instead of 117).
      uint32_t pb[H][NT][2], pl[H][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint64_t sum2 = 0;             // of the step: fewer roundings against a large l
        const uint64_t mu2 = kf::f2(mu[nt][0], mu[nt][1]);
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float p[2], w[2], x[2];
            const uint64_t over = kf::sub2(kf::f2(cc[h][nt][2 * y], cc[h][nt][2 * y + 1]), mu2);
            kf::f2_split(over, w[0], w[1]);
            kf::f2_split(kf::sub2(over, kf::f2(own_f[h][y], own_f[h][y])), x[0], x[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              w[j] = kf::ex2(w[j]);
              p[j] = __uint_as_float(__float_as_uint(w[j]) & 0xffffe000u);
            }
            sum2 = kf::add2(sum2, kf::f2(kf::ex2(x[0]), kf::ex2(x[1])));
            pl[h][nt][y] = kf::movmatrix_trans(kf::pack2<false>(w[0] - p[0], w[1] - p[1]));
            pb[h][nt][y] = kf::movmatrix_trans(kf::pack2<false>(p[0], p[1]));
          }
        float sum[2];
        kf::f2_split(sum2, sum[0], sum[1]);
        l_run[nt][0] += sum[0];
        l_run[nt][1] += sum[1];
      }
      // O^T (head dim x rows) += V^T P^T.  The products of a step are summed
      // from zero and then added, as an MMA cuts each of its products off where
      // its accumulator's digits end.
#pragma unroll
      for (int x = 0; x < PAIRS; ++x) {
        if (!LINES && 2 * x >= chunks) continue;
        float step[2][NT][4];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) step[e][nt][0] = step[e][nt][1] = step[e][nt][2] = step[e][nt][3] = 0.f;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          uint32_t w[4], f[2][4];
          ldmatrix_trans_b8(w, st + part(v_off[x], h));
          kf::decode4<INT8>(w[0], f[0][0], f[0][2]);
          kf::decode4<INT8>(w[1], f[0][1], f[0][3]);
          kf::decode4<INT8>(w[2], f[1][0], f[1][2]);
          kf::decode4<INT8>(w[3], f[1][1], f[1][3]);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (2 * x + e < chunks) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                kf::mma_16816<false>(step[e][nt], f[e], pb[h][nt][0], pb[h][nt][1]);
                kf::mma_16816<false>(step[e][nt], f[e], pl[h][nt][0], pl[h][nt][1]);
              }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4 && 2 * x + e < KD; i += 2)
              kf::f2_split(kf::add2(kf::f2(ot[nt][last(2 * x + e)][i], ot[nt][last(2 * x + e)][i + 1]),
                                    kf::f2(step[e][nt][i], step[e][nt][i + 1])),
                           ot[nt][last(2 * x + e)][i], ot[nt][last(2 * x + e)][i + 1]);
      }
    }
    if (++stage == STAGES) {
      stage = 0;
      parity ^= 1;
    }
    if (++fill == STAGES) fill = 0;

    const bool unit_done = work.unit_ends();
    going = work.more(end);
    if (!unit_done && going) {
      ++work.t;
      ++work.pos;
      continue;
    }
    // ---- join the teams and write the unit's rows (or its partial)
    const int b = work.b, h = work.h, rb = work.rb;
    if (unit_t0 == 0 && tid == 0 && (a.join_units || !unit_done)) {
      // a unit that begins here and goes on ends in the share of its last tile
      const int hr = h * a.row_blocks + rb;
      const uint32_t last = share_of(share, work.pos + (work.tiles - 1 - work.t));
      a.joins[a.join_units ? (int64_t)b * units + hr : (int64_t)me] =
          unit_done ? make_int4(-1, 0, 0, 0) : make_int4(b, hr, (int)me, (int)last);
    }
    if (going) {
      work.next(a);
      load_q();  // of the next unit: it arrives during what follows
    }
    const bool direct = unit_t0 == 0 && unit_done;
    const int64_t slot = (int64_t)me * 2 + (unit_t0 > 0 ? 0 : 1);  // 0: began in an earlier share, 1: begins here
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], off);
        if (!alive) l_run[nt][j] = m_run[nt][j] = NAN;  // a lost load shows in the result
      }
    const float spoiled = v_nan ? NAN : 0.f;        // O, not the LSE
    // Each warp scales its O^T to the rows' common reference and sum; then the
    // upper half of the teams hand theirs over, lane by lane as they hold it,
    // and the lower half add, until team 0 has the sum.
    if constexpr (C::TEAMS > 1) {
      if (lane < 4) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            *reinterpret_cast<float4*>(ml + (((warp * NT + nt) * 4 + lane) * 2 + j) * 4) =
                make_float4(m_run[nt][j], l_run[nt][j], spoiled, 0.f);
      }
      __syncthreads();
    }
    float lse2[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float by[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float ref = m_run[nt][j], sum = l_run[nt][j], held = spoiled, own = 1.f;
        if constexpr (C::TEAMS > 1) {
          // By the teams' sums: a reference of their m can lie past all of l.
          float4 x[C::TEAMS];
          ref = -INFINITY;
#pragma unroll
          for (int t = 0; t < C::TEAMS; ++t) {
            x[t] = *reinterpret_cast<const float4*>(ml + ((((t * RG + rg) * NT + nt) * 4 + (lane & 3)) * 2 + j) * 4);
            ref = fmaxf(ref, x[t].x + __log2f(x[t].y));
          }
          ref = ref == -INFINITY ? 0.f : ceilf(ref);
          sum = 0.f;
#pragma unroll
          for (int t = 0; t < C::TEAMS; ++t) {
            sum += kf::ex2(x[t].x - ref) * x[t].y;
            held += x[t].z;
          }
          own = kf::ex2(m_run[nt][j] - ref);
        }
        by[j] = sum + held == 0.f ? 0.f : own * reciprocal(sum + held);
        if (team == 0) lse2[nt][j] = sum == 0.f ? -INFINITY : ref + log2f(sum);
      }
#pragma unroll
      for (int dm = 0; dm < KD; ++dm) {
        ot[nt][dm][0] *= by[0];
        ot[nt][dm][1] *= by[1];
        ot[nt][dm][2] *= by[0];
        ot[nt][dm][3] *= by[1];
      }
    }
    const int valid_rows = min(C::ROWS, a.G - rb * C::ROWS);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // handed[0]: to team 0, handed[1]: to team 1 and then from it.  Team t's
      // writes follow its reads of that buffer; the next unit's first barrier
      // keeps its writes behind team 0's last reads.
#pragma unroll
      for (int step = C::TEAMS / 2; step >= 1; step /= 2) {
        if (RG == 1 && nt > 0 && step == 2) __syncthreads();  // team 0 has read the row tile before
        if (RG == 2 && nt > 0) __syncthreads();
        if (team >= step && team < 2 * step) {
          float* to = handed + (RG == 2 ? rg : step == 2 ? team - 2 : 1) * C::HANDED;
#pragma unroll
          for (int dm = 0; dm < KD; ++dm)
            *reinterpret_cast<float4*>(to + (dm * 32 + lane) * 4) =
                make_float4(ot[nt][dm][0], ot[nt][dm][1], ot[nt][dm][2], ot[nt][dm][3]);
        }
        __syncthreads();
        if (team < step) {
          const float* from = handed + (RG == 2 ? rg : step == 2 ? team : 1) * C::HANDED;
#pragma unroll
          for (int dm = 0; dm < KD; ++dm) {
            const float4 x = *reinterpret_cast<const float4*>(from + (dm * 32 + lane) * 4);
            ot[nt][dm][0] += x.x;
            ot[nt][dm][1] += x.y;
            ot[nt][dm][2] += x.z;
            ot[nt][dm][3] += x.w;
          }
        }
      }
      if (team != 0) continue;
      // rows of the unit: 8-row tile rg * NT + nt; O^T holds columns dm * 16 +
      // lane / 4 (+ 8) of rows 2 (lane % 4) + {0, 1}
      const int row0 = (rg * NT + nt) * 8;
      if (direct) {
        // 8 x 8 blocks transposed: row lane / 4, columns 2 (lane % 4) + {0, 1}
        const int r = row0 + (lane >> 2), head = h * a.G + rb * C::ROWS + r;
        uint16_t* out = a.o + ((int64_t)b * a.Hq + head) * a.D + 2 * (lane & 3);
#pragma unroll
        for (int dm = 0; dm < KD; ++dm)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float lo = ot[nt][dm][2 * e], hi = ot[nt][dm][2 * e + 1];
            const uint32_t x = kf::movmatrix_trans(kf::pack2<BF16>(lo, hi));
            if (r < valid_rows && dm * 16 + e * 8 < a.D) *reinterpret_cast<uint32_t*>(out + dm * 16 + e * 8) = x;
          }
        if (a.lse && lane < 4) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (row0 + 2 * lane + j < valid_rows)
              a.lse[(int64_t)b * a.Hq + h * a.G + rb * C::ROWS + row0 + 2 * lane + j] = lse2[nt][j] * kLn2;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = row0 + 2 * (lane & 3) + j;
          if (r >= valid_rows) continue;
          float* out = a.part_o + (slot * C::ROWS + r) * a.D + (lane >> 2);
#pragma unroll
          for (int dm = 0; dm < KD; ++dm)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (dm * 16 + e * 8 < a.D) out[dm * 16 + e * 8] = ot[nt][dm][2 * e + j];
          if (lane < 4) a.part_lse[slot * C::ROWS + r] = lse2[nt][j];
        }
      }
    }
    if (going) {
      start_unit();
      unit_t0 = 0;
    }
  }
  // after a failed wait, let the loads still in flight land (bounded) before leaving
  if (!alive && rg == 0 && lane == 0)
    for (int s = 0; s < STAGES; ++s) {
      const int used = issued / STAGES + (s < issued % STAGES ? 1 : 0);
      if (used > 0) kf::mbar_wait(&full[team][s], (uint32_t)(used - 1) & 1, nullptr, 100000000ull);
    }
}

// How the rows of a pool lie in a tile, and the variant that takes them.  Pages
// whose boxes of keys are whole lines of 128 bytes come by TMA, and rows of 128
// bytes in any case; other pages (shorter rows with gaps, sizes with few factors
// of two) by cp.async.  A TMA box of such rows is wider than they are, and a load of two
// planes of such boxes with its promotion to 256 bytes in L2 asks for blocks up
// to 20 KB off the box, past the end of the pool's memory.
struct Layout {
  int steps, box;
  bool lines;    // pages are brought as lines of 128 bytes
};

Layout layout_of(int64_t D, const kf_tensor4& k, const kf_tensor4& v) {
  Layout l;
  const int64_t page_size = k.size[2];
  const int chunks = (int)((D + 15) / 16), pitch = chunks * 16, keys = chunks <= 3 ? 128 : chunks <= 6 ? 64 : 32;
  l.box = keys;                        // keys that never cross a page
  while (page_size % l.box) l.box /= 2;
  l.lines = pitch * l.box % 128 == 0 &&
            (pitch == 128 || page_size == 1 || (k.stride[2] == pitch && v.stride[2] == pitch));
  l.steps = l.lines ? chunks : 8;
  if (!l.lines && l.box > 32) l.box = 32;
  return l;
}

template <int KD>
int tile_keys_of(int rows) {
  return rows == 8    ? Cfg8<KD, 1, 1>::TILE
         : rows == 16 ? Cfg8<KD, 2, 1>::TILE
         : rows == 32 ? Cfg8<KD, 2, 2>::TILE
                      : Cfg8<KD, 2, 4>::TILE;
}
int tile_keys(int steps, int rows) {
  return steps <= 3 ? tile_keys_of<3>(rows) : steps <= 6 ? tile_keys_of<6>(rows) : tile_keys_of<8>(rows);
}

template <bool INT8, bool BF16, int KD, bool LINES, int NT, int RG>
int launch_variant(const Paged8Args& a, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t st) {
  using C = Cfg8<KD, NT, RG>;
  static_assert(C::STAGES >= 2, "the ring needs two stages");
  static_assert(C::STAGE % 1024 == 0, "stages begin where a swizzle does");
  // an SM has 228 KB, of which each block takes 1 KB besides its own
  static_assert(C::SMEM <= (228 / C::BLOCKS - 1) * 1024, "the blocks of an SM");
  auto kern = paged8_decode_kernel<INT8, BF16, KD, LINES, NT, RG>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) {
    (void)cudaGetLastError();
    return kf::set_error(KF_ERR_CUDA, "kf_paged8_decode: cannot reserve %d bytes of shared memory", C::SMEM);
  }
  return kf::launch_dependent(kern, dim3((unsigned)blocks), dim3(kThreads), C::SMEM, st, "kf_paged8_decode", mk, mv, a);
}

template <bool INT8, bool BF16, int KD, bool LINES>
int dispatch_rows(const Paged8Args& a, const CUtensorMap& mk, const CUtensorMap& mv, int rows, int blocks,
                  cudaStream_t st) {
  switch (rows) {  // unit_rows()'s
    case 8: return launch_variant<INT8, BF16, KD, LINES, 1, 1>(a, mk, mv, blocks, st);
    case 16: return launch_variant<INT8, BF16, KD, LINES, 2, 1>(a, mk, mv, blocks, st);
    case 32: return launch_variant<INT8, BF16, KD, LINES, 2, 2>(a, mk, mv, blocks, st);
    default: return launch_variant<INT8, BF16, KD, LINES, 2, 4>(a, mk, mv, blocks, st);
  }
}

template <bool INT8, bool BF16>
int dispatch(const kf::Paged8Launch& l) {
  const Paged8Args& a = *static_cast<const Paged8Args*>(l.args);
  auto go = [&](auto steps, auto lines) {
    return dispatch_rows<INT8, BF16, steps, lines>(a, *l.map_k, *l.map_v, l.rows, l.blocks, l.stream);
  };
  constexpr std::true_type lines;
  if (!l.lines) return go(std::integral_constant<int, 8>(), std::false_type());
  switch (l.steps) {
    case 1: return go(std::integral_constant<int, 1>(), lines);
    case 2: return go(std::integral_constant<int, 2>(), lines);
    case 3: return go(std::integral_constant<int, 3>(), lines);
    case 4: return go(std::integral_constant<int, 4>(), lines);
    case 5: return go(std::integral_constant<int, 5>(), lines);
    case 6: return go(std::integral_constant<int, 6>(), lines);
    case 7: return go(std::integral_constant<int, 7>(), lines);
    default: return go(std::integral_constant<int, 8>(), lines);
  }
}

}  // namespace
