// K5: attention of one new token per request over a paged K/V cache, split
// over the cache's length and joined, with an optional fused append of that
// token's own K/V row.
//
// For request b, query head h (of KV head h / G) and the visible positions j
// (j < lengths[b] whose page is in the pool), with x_j = scale q.k_j:
//   m = max x_j,  l = sum e^(x_j - m),  O = sum e^(x_j - m) v_j / l,
//   LSE = m + ln l;  no visible position: O = 0, LSE = -inf.
// Every K/V row is read once for G query rows (4 G D flops per 4 D bytes at
// 16 bits), so HBM bounds it up to a few dozen rows per KV head.
//
// Work split.  A unit is (request, KV head, block of query rows); its keys
// are cut into tiles.  All tiles of the call, unit after unit with a position
// for the unit's end, form one list that is dealt out in equal contiguous
// shares to a grid that fills the GPU once.  Each block finds its share from the lengths by a prefix sum, so
// ragged batches are balanced without the host knowing a length (no
// synchronisation, and a captured graph follows the lengths).  A unit that
// lies inside one share is finished there; one cut by a share's end leaves
// fp32 partials (normalised O, log2 LSE) in at most two slots per block and
// is joined by a second kernel.
//
// Inside a block four warps take different keys of each tile (or, with more
// than 16 rows per KV head, 2 or 4 warps form a team that shares keys and
// splits the rows).  Each team streams its own keys through its own ring of
// shared-memory stages by TMA, so teams never wait for one another inside a
// unit; the ring runs ahead across unit boundaries.  A tensor map over the
// pool turns (page, head, row) into addresses, whatever the cache's strides:
// a lane looks up the page of one key, and the lanes at the start of a box of
// gcd(page_size, 16) rows, which never crosses a page, load it.  The products
// are taken transposed on warp MMAs (S^T = K Q^T, O^T = V^T P^T): keys and
// head-dim fill the m = 16 side and up to 8 query rows the n = 8 side, so
// few rows waste little.
#include <float.h>
#include <math.h>

#include "paged_split.cuh"

namespace {

struct PagedArgs : PagedWork {
  const uint16_t* q;
  uint16_t* k;             // written only by the fused append
  uint16_t* v;
  const uint16_t* nk;      // null: no fused append
  const uint16_t* nv;
  const int64_t* slots;    // of the new rows; < 0: this request has none
  int64_t qs[2], ks[3], vs[3], nks[2], nvs[2];
  int box, box_ops;        // rows of a TMA box, and loads that bring its columns
  int box_bytes;           // of K and V together
  int width;               // 16-byte chunks of a panel's rows (8, 4 or 2), or 0: dense rows (see tile_offset)
  int block_bytes, row_bytes;  // from 16 rows of a tile to the next, and between rows as boxes of fewer start
  bool shallow;            // long units are loaded a third of the ring ahead instead of all of it
  float scale_log2;        // |scale| log2(e), at least the smallest number
  uint32_t q_sign;         // flips the signs of two elements of Q where scale is negative
};

// Variants: KD = 16-column steps of the padded head dim (4, 6 or 8); FULL: D is
// KD * 16; NT = 8-row tiles of query rows per warp; RG = warps of a team (row
// groups).
template <int KD, int NT, int RG>
struct Cfg {
  static constexpr int DP = KD * 16;
  static constexpr int KW = (KD > 6 && RG == 1) ? 16 : 32;  // keys a team takes of a tile
  static constexpr int TEAMS = kWarps / RG;
  static constexpr int TILE = TEAMS * KW;                    // keys of a tile
  static constexpr int ROWS = NT * 8 * RG;                   // query rows of a unit
  static constexpr int STAGE = KW * DP * 2 * 2;              // bytes: K rows, then V rows
  static constexpr int STAGES = 98304 / (TEAMS * STAGE);     // 96 KB of ring per block, two blocks per SM
  static constexpr int SHALLOW = STAGES / 3 > 1 ? STAGES / 3 : 1;  // stages loaded ahead for long units, at least one
  static constexpr int HANDED = KD * 4 * 32;                 // floats of a warp's O^T of one row tile
  static constexpr int SMEM = 1024 + TEAMS * STAGES * STAGE + (TEAMS > 1 ? 2 * HANDED + kWarps * NT * 16 : 0) * 4;
};

// Offset of 16-byte chunk c of row r in a K or V tile as TMA writes it: blocks
// of 16 rows, in a block the panels of `width` chunks one after another, in a
// panel row after row with the chunks swizzled, so that the 8 rows an ldmatrix
// reads lie on different banks.  Panels are as wide as divides D (64, 32 or 16
// columns), since a panel wider than what is left of a row fetches the columns
// beyond it as well (D = 72 in 64-column panels: 638 MB through L2 for 302 MB).
// An odd number of chunks per row (72, 104) needs neither panels nor a
// swizzle: width 0, rows one after another.  Boxes of fewer than 16 rows
// (page sizes that 16 does not divide) bring one panel at a time, so they
// keep 64-column panels; dense rows can still be boxes of 8.
__device__ __forceinline__ uint32_t tile_at(int r, int c, int width, int block_bytes) {
  if (width == 0) return (uint32_t)((r >> 4) * block_bytes + (r & 15) * (block_bytes >> 4) + c * 16);
  const int log = width == 8 ? 3 : width == 4 ? 2 : 1, x = r >> (3 - log);
  return (uint32_t)((r >> 4) * block_bytes + (c >> log) * 256 * width + (r & 15) * 16 * width +
                    (((c ^ x) & (width - 1)) << 4));
}

template <bool BF16, int KD, bool FULL, int NT, int RG>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const PagedArgs a) {
  using C = Cfg<KD, NT, RG>;
  constexpr int KW = C::KW, STAGES = C::STAGES, TILE = C::TILE;
  constexpr int H = KW / 16;           // 16-key halves of a step
  constexpr int K_BYTES = KW * C::DP * 2;
  constexpr uint32_t ALL = KW == 32 ? 0xffffffffu : 0xffffu;
  // The reference m of a row's weights 2^(x - m) lies BELOW under a maximum of
  // the row and is raised once a score passes it by LIMIT.  bf16 holds small
  // weights as well as large ones.  fp16's two parts end at 2^-24 whatever the
  // weight, so weights use the top of its range: 2^11 at the maximum, 2^15 at
  // most, and the parts end at 2^-35 of the row's largest weight or lower.
  // (With the maximum as the reference 32768 keys 2^25 below one that leads
  // were lost from O and counted in the sum: 8e-4 of O.)
  constexpr float BELOW = BF16 ? 0.f : 11.f, LIMIT = BF16 ? 8.f : 15.f;
  constexpr float LEAST = BF16 ? FLT_MIN : 1.f / (1 << 24);  // of a part of a weight
  extern __shared__ uint8_t smem_raw[];
  // (an offset, not a rounded address: the compiler keeps seeing shared memory)
  uint8_t* smem = smem_raw + (-kf::smem_u32(smem_raw) & 1023u);
  __shared__ ShareScratch scratch;
  __shared__ __align__(8) uint64_t full[C::TEAMS][STAGES];
  __shared__ uint32_t seen_s[C::TEAMS][STAGES];  // visible keys of each stage
  __shared__ int abort_any;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int team = warp / RG, rg = warp % RG;
  const int units = a.Hkv * a.row_blocks;  // per request
  uint8_t* ring = smem + team * STAGES * C::STAGE;
  float* handed = reinterpret_cast<float*>(smem + C::TEAMS * STAGES * C::STAGE);  // [2][KD][lane][4]
  float* ml = handed + 2 * C::HANDED;                                             // [warp][NT * 8 rows][m, l]

  if (tid == 0) {
    for (int i = 0; i < C::TEAMS * STAGES; ++i) kf::mbar_init(&full[0][0] + i, 1);
    kf::fence_barrier_init();
    abort_any = 0;
    kf::tma_prefetch_desc(&map_k);
    kf::tma_prefetch_desc(&map_v);
  }
  // The chain lengths -> table -> K/V starts cold: bring the lengths and, over
  // all blocks, the first part of the table to L2 while the previous kernel
  // still runs (hints only: L2 stays coherent with what that kernel writes).
  {
    const uint32_t line = blockIdx.x * kThreads + tid;  // of 32 entries
    if (line * 32 < (uint32_t)a.B) prefetch_l2(a.lengths + line * 32);
    const uint32_t lines_per_row = (a.max_pages + 31) / 32, b = line / lines_per_row;
    if (b < (uint32_t)a.B) prefetch_l2(a.table + b * a.table_stride + (line - b * lines_per_row) * 32);
    const uint32_t request = line / a.Hq;
    if (request < (uint32_t)a.B)
      kf::prefetch_l2_bulk(a.q + request * a.qs[0] + (line - request * a.Hq) * a.qs[1], a.D * 2);
  }
  // where things lie in a tile
  const int block_bytes = FULL ? KD * 512 : a.block_bytes;
  auto tile_offset = [&](int r, int c) { return tile_at(r, c, FULL ? 8 : a.width, block_bytes); };
  // what a lane clears of an unseen row: the row's pitch, and this lane's chunk (swizzle aside) or -1
  const int row_pitch = FULL ? 128 : a.width ? a.width * 16 : block_bytes >> 4;
  const int zero_chunk = (lane & 15) < (block_bytes >> 8) ? (int)tile_offset(0, lane & 15) : -1;
  // offsets of a lane's ldmatrix rows in a K or V tile, by 16-column step (mod
  // 4 in panels); in a dense tile a step's missing second half repeats its first
  constexpr int OFFSETS = FULL ? 4 : KD;
  uint32_t k_off[OFFSETS], v_off[OFFSETS];
#pragma unroll
  for (int x = 0; x < OFFSETS; ++x) {
    const int last = FULL ? KD * 2 - 1 : a.D / 8 - 1;
    k_off[x] = tile_offset(lane & 15, min(2 * x + (lane >> 4), last));
    v_off[x] = tile_offset((lane & 7) + ((lane >> 4) << 3), min(2 * x + ((lane >> 3) & 1), last));
  }
  // (The kernel may have been alive while its predecessor wrote the lengths,
  // tables, Q or slots, so none of them is read through the non-coherent path.)
  kf::griddep_wait();
  kf::griddep_launch_dependents();

  const uint32_t me = blockIdx.x;
  const bool join_blocks = a.joins && !a.join_units;
  Share share;
  Cursor<TILE> load, work;
  if (!find_share<TILE>(a, scratch, share) || !first_tile(a, share, work)) {
    if (tid == 0 && join_blocks) a.joins[me].x = -1;
    clear_empty(a);
    return;
  }
  const uint32_t end = share.end;
  load = work;

  // ---- loads: lane r (of KW) looks up key r of the team's share of a tile
  struct Place {
    uint32_t page, row;
    int h;
  };
  auto look_up = [&]() {
    const uint32_t key = load.t * TILE + team * KW + (KW == 32 ? lane : (lane & 15));
    const uint32_t pg = (uint32_t)(((uint64_t)key * a.page_mul) >> a.page_shift);
    Place p;
    p.row = key - pg * a.page_size;
    p.page = key < load.keys ? (uint32_t)a.table[load.b * a.table_stride + pg] : 0xffffffffu;
    p.h = load.h;
    return p;
  };
  auto issue = [&](int stage, const Place& p) {
    const bool valid = p.page < a.num_pages;
    const uint32_t seen = __ballot_sync(0xffffffffu, valid) & ALL;
    const bool starts_box = valid && lane < KW && (lane & (a.box - 1)) == 0;
    const uint32_t boxes = __ballot_sync(0xffffffffu, starts_box);
    uint64_t* bar = &full[team][stage];
    if (lane == 0) {
      seen_s[team][stage] = seen;
      kf::mbar_arrive_expect_tx(bar, (uint32_t)(__popc(boxes) * a.box_bytes));
    }
    __syncwarp();
    if (starts_box) {
      uint8_t* st = ring + stage * C::STAGE + (lane >> 4) * block_bytes + (lane & 15) * a.row_bytes;
      kf::tma_load_5d(st, &map_k, bar, 0, p.row, 0, p.h, p.page);
      kf::tma_load_5d(st + K_BYTES, &map_v, bar, 0, p.row, 0, p.h, p.page);
      if (KD == 8 && a.box_ops == 2) {  // the second 64-column panel
        kf::tma_load_5d(st + 2048, &map_k, bar, 64, p.row, 0, p.h, p.page);
        kf::tma_load_5d(st + K_BYTES + 2048, &map_v, bar, 64, p.row, 0, p.h, p.page);
      }
    }
  };

  // ---- state of the unit being worked on
  uint32_t qb[NT][KD][2];              // Q^T as B fragments
  // rows 2 (lane % 4) + {0, 1} of each row tile: the reference of the weights
  // 2^(x - m), their sum, and m again as it enters the exponent (0 for -inf)
  float m_run[NT][2], l_run[NT][2], mu[NT][2];
  float ot[NT][KD][4];                 // O^T
  auto at = [&](const uint32_t (&off)[OFFSETS], int step, int h) -> uint32_t {
    if constexpr (FULL)
      return off[step & 3] + (step >> 2) * 2048 + h * (KD * 512);
    else
      return off[step] + h * block_bytes;
  };
  // The loads of the unit's Q, issued where they are written: early, since they
  // queue behind the K/V loads in flight.  start_unit() follows where the unit
  // begins.
  auto load_q = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = work.rb * C::ROWS + rg * NT * 8 + nt * 8 + (lane >> 2);
      const uint16_t* src = a.q + work.b * a.qs[0] + (int64_t)(work.h * a.G + row) * a.qs[1] + 2 * (lane & 3);
#pragma unroll
      for (int kk = 0; kk < KD; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qb[nt][kk][e] = 0u;
          if (row < a.G && kk * 16 + e * 8 < a.D)
            asm volatile("ld.global.b32 %0, [%1];" : "=r"(qb[nt][kk][e]) : "l"(src + kk * 16 + e * 8));
        }
    }
  };
  auto start_unit = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int kk = 0; kk < KD; ++kk) {
        qb[nt][kk][0] ^= a.q_sign;
        qb[nt][kk][1] ^= a.q_sign;
        ot[nt][kk][0] = ot[nt][kk][1] = ot[nt][kk][2] = ot[nt][kk][3] = 0.f;
      }
      m_run[nt][0] = m_run[nt][1] = -INFINITY;
      l_run[nt][0] = l_run[nt][1] = mu[nt][0] = mu[nt][1] = 0.f;
    }
  };

  load_q();
  // Tiles loaded ahead of the one in use.  Short units drain the ring at each
  // end and want all of it; for the rest a third, 64 KB per SM, is what HBM
  // needs, and more only queues: blocks then get unequal shares of the
  // bandwidth and end far apart.  Whole ring against a third, D = 128: 8192
  // keys 171.5 and 165.6 us, 600 to 1000 keys 72.8 and 72.9, 200 to 600 keys
  // 72.3 and 74.5, so long starts at 10 tiles; D = 64, 8192 keys: 91.9 and 87.4.
  const int depth = a.shallow && share.total >= 10u * a.B ? C::SHALLOW : STAGES - 1;
  // The first warp of a team loads.  To begin with it looks up the pages of the
  // whole ring at once, then always one step ahead of their use.
  int issued = 0;
  bool more = rg == 0;                 // whether the load cursor stands on a tile that is not loaded yet
  Place ahead;
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
      if (s < issued) issue(s, first[s]);
    if (more) ahead = look_up();
  }
  uint32_t unit_t0 = work.t;           // first tile of the unit in this share
  if (tid == 0 && join_blocks) a.joins[me].x = -1;
  clear_empty(a);
  start_unit();

  int stage = 0, fill = depth;
  uint32_t parity = 0;
  bool alive = true;                   // false once a wait of this block has expired
  for (bool going = true; going;) {
    // One outcome for the team: no lane reaches a collective instruction alone.
    // The barrier also says that the team has left stage i - 1.
    uint32_t seen = RG == 1 ? seen_s[team][stage] : 0u;  // (this warp's own word: read before the wait)
    bool landed = kf::mbar_try_wait(&full[team][stage], parity);
    if (!landed) landed = alive && !*(volatile int*)&abort_any && kf::mbar_wait(&full[team][stage], parity, a.status);
    alive = team_and<RG>(team, alive && landed);
    if (!alive && lane == 0) *(volatile int*)&abort_any = 1;
    if (RG > 1) seen = seen_s[team][stage];
    if (!alive) seen = 0;
    if (rg == 0 && alive && more) {
      issue(fill, ahead);
      ++issued;
      more = load.more(end);
      if (more) {
        load.next(a);
        ahead = look_up();
      }
    }

    uint8_t* kt = ring + stage * C::STAGE;
    uint8_t* vt = kt + K_BYTES;
    const uint32_t key0 = work.t * TILE + team * KW;
    if (seen != 0 && (seen != ALL || (a.nk && key0 + KW >= work.keys))) {
      // The end of a request or pages without a table entry.  Rows that nobody
      // sees hold anything: their scores are replaced below, their V rows must
      // be zero.  A new row takes its place here and goes to its page.
      // (Two rows at a time, a lane per chunk; whole rows, so that the swizzle
      // does not matter.  Every short unit comes here and its other teams wait:
      // 300 to 500 cycles, where a loop over rows and chunks took 800 to 2500;
      // 1808 units of 22 to 45 positions went from 31.7 to 20.6 us.)
#pragma unroll
      for (int x = rg; x < KW / 2; x += RG) {
        const int r = 2 * x + (lane >> 4);
        clear16(kf::smem_u32(vt) + (r >> 4) * block_bytes + (r & 15) * row_pitch + zero_chunk,
                zero_chunk >= 0 && !((seen >> r) & 1));
      }
      const uint32_t r = work.keys - 1 - key0;  // the newest position, unless the table is too short for it
      if (a.nk && r < (uint32_t)KW && ((seen >> r) & 1) && work.whole && a.slots[work.b] >= 0) {
        const int c = lane & 15;
        if (rg == 0 && c < a.D / 8) {
          const uint32_t pg = (uint32_t)(((uint64_t)(key0 + r) * a.page_mul) >> a.page_shift);
          const int64_t page = a.table[work.b * a.table_stride + pg], row = key0 + r - pg * a.page_size;
          const uint16_t* src = lane < 16 ? a.nk + work.b * a.nks[0] + work.h * a.nks[1]
                                          : a.nv + work.b * a.nvs[0] + work.h * a.nvs[1];
          uint16_t* dst = lane < 16 ? a.k + page * a.ks[0] + work.h * a.ks[1] + row * a.ks[2]
                                    : a.v + page * a.vs[0] + work.h * a.vs[1] + row * a.vs[2];
          const uint4 x = reinterpret_cast<const uint4*>(src)[c];
          *reinterpret_cast<uint4*>((lane < 16 ? kt : vt) + tile_offset(r, c)) = x;
          if (work.rb == 0) reinterpret_cast<uint4*>(dst)[c] = x;
        }
      }
      kf::fence_proxy_async_smem();    // before a later load into this stage
      __syncwarp();                    // (the vote of a team of one warp orders no memory)
      team_and<RG>(team, true);
    }
    if (seen != 0) {
      const uint32_t sk = kf::smem_u32(kt), sv = kf::smem_u32(vt);
      // S^T (keys x rows).  Operands are loaded four at a time ahead of their
      // products, and a lone chain of products is cut in two: with two warps
      // per scheduler the latency of a step is what short shares wait for.
      constexpr int CHAINS = H * NT == 1 ? 2 : 1;
      float cc[CHAINS][H][NT][4];
#pragma unroll
      for (int x = 0; x < CHAINS; ++x)
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) cc[x][h][nt][0] = cc[x][h][nt][1] = cc[x][h][nt][2] = cc[x][h][nt][3] = 0.f;
      constexpr int KG = H == 1 ? 4 : 2;
#pragma unroll
      for (int k0 = 0; k0 < KD; k0 += KG) {
        uint32_t ka[KG][H][4];
#pragma unroll
        for (int x = 0; x < KG && k0 + x < KD; ++x)
#pragma unroll
          for (int h = 0; h < H; ++h)
            if (FULL || (k0 + x) * 16 < a.D) kf::ldmatrix_x4(ka[x][h], sk + at(k_off, k0 + x, h));
#pragma unroll
        for (int x = 0; x < KG && k0 + x < KD; ++x) {
          if (FULL || (k0 + x) * 16 + 8 < a.D) {
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                kf::mma_16816<BF16>(cc[x % CHAINS][h][nt], ka[x][h], qb[nt][k0 + x][0], qb[nt][k0 + x][1]);
          } else if ((k0 + x) * 16 < a.D) {
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                kf::mma_1688<BF16>(cc[x % CHAINS][h][nt], ka[x][h][0], ka[x][h][1], qb[nt][k0 + x][0]);
          }
        }
      }
      float (&c)[H][NT][4] = cc[0];
      if constexpr (CHAINS == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[0][0][e] += cc[1][0][0][e];
      }
      // rows 2 (lane % 4) + {0, 1}; keys 16 h + lane / 4 (c0, c1) and + 8 (c2, c3)
      if (seen != ALL) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const uint32_t bits = seen >> (h * 16 + (lane >> 2));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[h][nt][e] = (bits & (e < 2 ? 1u : 256u)) ? c[h][nt][e] : -INFINITY;
        }
      }
      // The reference of a row follows its maximum only when a score passes it
      // by LIMIT: most steps need no exchange between lanes (the softmax of a
      // step: 295 -> 194 cycles of 1770 with one row tile, 558 -> 257 of
      // 2280 with two).  The test computes what the exponent will be, so no
      // weight exceeds 2^LIMIT however large the scores.
      bool raise = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = fmaxf(c[0][nt][j], c[0][nt][2 + j]);
          if constexpr (H == 2) top = kf::fmax3(top, c[H - 1][nt][j], c[H - 1][nt][2 + j]);
          raise |= fmaf(top, a.scale_log2, -m_run[nt][j]) > LIMIT;
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = fmaxf(c[0][nt][j], c[0][nt][2 + j]);
            if constexpr (H == 2) top = kf::fmax3(top, c[H - 1][nt][j], c[H - 1][nt][2 + j]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const float m_new = fmaxf(m_run[nt][j], fmaf(top, a.scale_log2, -BELOW));
            mu[nt][j] = m_new == -INFINITY ? 0.f : m_new;
            const float old = kf::ex2(m_run[nt][j] - mu[nt][j]);
            m_run[nt][j] = m_new;
            l_run[nt][j] *= old;
#pragma unroll
            for (int dm = 0; dm < KD; ++dm) {
              ot[nt][dm][j] *= old;
              ot[nt][dm][2 + j] *= old;
            }
          }
      }
      uint32_t pb[H][NT][2], pl[H][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float sum[2] = {0.f, 0.f};  // of the step: fewer roundings against a large l
#pragma unroll
        for (int h = 0; h < H; ++h) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = kf::ex2(fmaf(c[h][nt][e], a.scale_log2, -mu[nt][e & 1]));
            sum[e & 1] += p[e];
          }
          // P as the next smaller 16-bit value plus the 16-bit rest: two
          // products hold a weight to 2^-16 of itself (bf16), or to 2^-21 of
          // itself and 2^-34 of the row's largest (fp16).  Both parts are
          // positive whatever the weight, so that an infinity in V stays one
          // (0 times it would be NaN); the V of masked keys is 0.
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float w0 = fmaxf(p[2 * x], 2 * LEAST), w1 = fmaxf(p[2 * x + 1], 2 * LEAST);
            const uint32_t hi = kf::pack2_below<BF16>(w0, w1);
            const float2 back = kf::unpack2<BF16>(hi);
            pb[h][nt][x] = kf::movmatrix_trans(hi);
            pl[h][nt][x] = kf::movmatrix_trans(kf::pack2<BF16>(fmaxf(w0 - back.x, LEAST), fmaxf(w1 - back.y, LEAST)));
          }
        }
        l_run[nt][0] += sum[0];
        l_run[nt][1] += sum[1];
      }
      // O^T (head dim x rows) += V^T P^T, the two parts of P apart from one
      // another so that no product waits for the one before it.  The products
      // of a step are summed from zero and then added: an MMA cuts each of its
      // products off where its accumulator's digits end, which lost 4e-3 of O
      // on 131072 keys beside one that leads by 2^23.5.  (It costs nothing up to
      // 8 rows per KV head, 56.2 -> 58.8 us at 32: 32 requests of 16384 keys.)
      constexpr int VG = NT == 1 ? 4 : 2;
#pragma unroll
      for (int d0 = 0; d0 < KD; d0 += VG) {
        float step[VG][NT][4];
#pragma unroll
        for (int x = 0; x < VG; ++x)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) step[x][nt][0] = step[x][nt][1] = step[x][nt][2] = step[x][nt][3] = 0.f;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          uint32_t va[VG][4];
#pragma unroll
          for (int x = 0; x < VG && d0 + x < KD; ++x)
            if (FULL || (d0 + x) * 16 < a.D) kf::ldmatrix_x4_trans(va[x], sv + at(v_off, d0 + x, h));
#pragma unroll
          for (int x = 0; x < VG && d0 + x < KD; ++x)
            if (FULL || (d0 + x) * 16 < a.D) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) kf::mma_16816<BF16>(step[x][nt], va[x], pb[h][nt][0], pb[h][nt][1]);
            }
#pragma unroll
          for (int x = 0; x < VG && d0 + x < KD; ++x)
            if (FULL || (d0 + x) * 16 < a.D) {
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) kf::mma_16816<BF16>(step[x][nt], va[x], pl[h][nt][0], pl[h][nt][1]);
            }
        }
#pragma unroll
        for (int x = 0; x < VG && d0 + x < KD; ++x)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) ot[nt][d0 + x][e] += step[x][nt][e];
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
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], off);
    if (!alive) {  // a lost load shows in the result
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) l_run[nt][0] = l_run[nt][1] = m_run[nt][0] = m_run[nt][1] = NAN;
    }
    // Each warp scales its O^T to the rows' common reference and sum; then the
    // upper half of the teams hand theirs over, lane by lane as they hold it,
    // and the lower half add, until team 0 has the sum.  (Rows gathered from
    // all teams through a transposed buffer, with the weights worked out by
    // every reader: 63 instead of 57 us for 64 query heads on one KV head.)
    if constexpr (C::TEAMS > 1) {
      if (lane < 4) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          *reinterpret_cast<float4*>(ml + (warp * NT + nt) * 16 + lane * 4) =
              make_float4(m_run[nt][0], l_run[nt][0], m_run[nt][1], l_run[nt][1]);
      }
      __syncthreads();
    }
    float lse2[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top[2] = {m_run[nt][0], m_run[nt][1]}, sum[2] = {l_run[nt][0], l_run[nt][1]}, own[2] = {1.f, 1.f};
      if constexpr (C::TEAMS > 1) {
        float4 x[C::TEAMS];
#pragma unroll
        for (int t = 0; t < C::TEAMS; ++t) {
          x[t] = *reinterpret_cast<const float4*>(ml + ((t * RG + rg) * NT + nt) * 16 + (lane & 3) * 4);
          top[0] = fmaxf(top[0], x[t].x);
          top[1] = fmaxf(top[1], x[t].z);
        }
        const float ref[2] = {top[0] == -INFINITY ? 0.f : top[0], top[1] == -INFINITY ? 0.f : top[1]};
        sum[0] = sum[1] = 0.f;
#pragma unroll
        for (int t = 0; t < C::TEAMS; ++t) {
          sum[0] += kf::ex2(x[t].x - ref[0]) * x[t].y;
          sum[1] += kf::ex2(x[t].z - ref[1]) * x[t].w;
        }
        own[0] = kf::ex2(m_run[nt][0] - ref[0]);
        own[1] = kf::ex2(m_run[nt][1] - ref[1]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        own[j] = sum[j] == 0.f ? 0.f : own[j] * reciprocal(sum[j]);
        if (team == 0) lse2[nt][j] = sum[j] == 0.f ? -INFINITY : top[j] + log2f(sum[j]);
      }
#pragma unroll
      for (int dm = 0; dm < KD; ++dm) {
        ot[nt][dm][0] *= own[0];
        ot[nt][dm][1] *= own[1];
        ot[nt][dm][2] *= own[0];
        ot[nt][dm][3] *= own[1];
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
            const uint32_t x = kf::movmatrix_trans(kf::pack2<BF16>(ot[nt][dm][2 * e], ot[nt][dm][2 * e + 1]));
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

// KD of the variant for a head dim.
int head_steps(int64_t D, bool wide) { return D <= 64 ? 4 : D <= 96 && !wide ? 6 : 8; }

// Keys per tile of the variant.
template <int KD>
int tile_keys_of(int rows) {
  return rows == 8    ? Cfg<KD, 1, 1>::TILE
         : rows == 16 ? Cfg<KD, 2, 1>::TILE
         : rows == 32 ? Cfg<KD, 2, 2>::TILE
                      : Cfg<KD, 2, 4>::TILE;
}
int tile_keys(int steps, int rows) {
  return steps == 4 ? tile_keys_of<4>(rows) : steps == 6 ? tile_keys_of<6>(rows) : tile_keys_of<8>(rows);
}

template <bool BF16, int KD, bool FULL, int NT, int RG>
int launch_variant(const PagedArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t st) {
  using C = Cfg<KD, NT, RG>;
  static_assert(C::STAGES >= 2, "the ring needs two stages");
  auto kern = paged_decode_kernel<BF16, KD, FULL, NT, RG>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) {
    (void)cudaGetLastError();
    return kf::set_error(KF_ERR_CUDA, "kf_paged_decode: cannot reserve %d bytes of shared memory", C::SMEM);
  }
  return kf::launch_dependent(kern, dim3((unsigned)blocks), dim3(kThreads), C::SMEM, st, "kf_paged_decode", mk, mv, a);
}

template <bool BF16, int KD, bool FULL>
int dispatch_rows(const PagedArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int rows, int blocks,
                  cudaStream_t st) {
  static_assert(Cfg<KD, 1, 1>::ROWS == 8 && Cfg<KD, 2, 1>::ROWS == 16 && Cfg<KD, 2, 2>::ROWS == 32 &&
                    Cfg<KD, 2, 4>::ROWS == 64,
                "the cases are unit_rows()'s");
  switch (rows) {
    case 8: return launch_variant<BF16, KD, FULL, 1, 1>(a, mk, mv, blocks, st);
    case 16: return launch_variant<BF16, KD, FULL, 2, 1>(a, mk, mv, blocks, st);
    case 32: return launch_variant<BF16, KD, FULL, 2, 2>(a, mk, mv, blocks, st);
    default: return launch_variant<BF16, KD, FULL, 2, 4>(a, mk, mv, blocks, st);
  }
}

bool rows16(const kf_tensor4* t, int dims) {
  if (!kf::aligned16(t->ptr) || t->stride[3] != 1) return false;
  for (int i = 0; i < dims; ++i)
    if (t->size[i] > 1 && t->stride[i] % 8 != 0) return false;
  return true;
}

}  // namespace

extern "C" size_t kf_paged_decode_workspace_bytes(int64_t Hq, int64_t Hkv, int64_t D, int sm_count) {
  if (Hq <= 0 || Hkv <= 0 || D <= 0 || sm_count <= 0) return 0;
  return workspace_need(sm_count * kBlocksPerSm, unit_rows(Hq / Hkv), D);
}

extern "C" int kf_paged_decode(const kf_paged_decode_args* args) {
  using kf::set_error;
  const char* what = "kf_paged_decode";
  if (!args) return set_error(KF_ERR_INVALID, "%s: null arguments", what);
  const kf_tensor4 *q = &args->q, *k_pages = &args->k_pages, *v_pages = &args->v_pages;
  const kf_tensor4 *new_k = &args->new_k, *new_v = &args->new_v;
  const int64_t dtype = args->dtype, max_pages = args->max_pages;
  if (dtype != KF_F16 && dtype != KF_BF16) return set_error(KF_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  const int64_t B = q->size[0], Hq = q->size[1], D = q->size[3];
  const int64_t pages = k_pages->size[0], Hkv = k_pages->size[1], page_size = k_pages->size[2];
  for (int i = 0; i < 4; ++i)
    if (k_pages->size[i] != v_pages->size[i])
      return set_error(KF_ERR_INVALID, "%s: K/V page shapes must match", what);
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || pages <= 0 || page_size <= 0 || max_pages <= 0)
    return set_error(KF_ERR_INVALID, "%s: dimensions must be non-zero", what);
  if (q->size[2] != 1) return set_error(KF_ERR_INVALID, "%s: Q must hold one token per request", what);
  if (k_pages->size[3] != D) return set_error(KF_ERR_INVALID, "%s: Q/K/V head dimensions must match", what);
  if (Hq % Hkv != 0)
    return set_error(KF_ERR_INVALID, "%s: num_query_heads must be divisible by num_kv_heads", what);
  if (D < 16 || D > 128 || D % 8 != 0)
    return set_error(KF_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 in [16, 128]", what);
  if (page_size > (1 << 20) || pages > 0x7fffffffLL || max_pages > 0x7fffffffLL || B > (1 << 20) || Hq > (1 << 16))
    return set_error(KF_ERR_UNSUPPORTED, "%s: tensors too large", what);
  if (!rows16(q, 2) || !rows16(k_pages, 3) || !rows16(v_pages, 3) ||
      !kf::aligned16(args->o))
    return set_error(KF_ERR_INVALID, "%s: tensors need a contiguous last dim and 16-byte aligned rows", what);
  if (!q->ptr || !k_pages->ptr || !v_pages->ptr || !args->o || !args->block_table || !args->lengths)
    return set_error(KF_ERR_INVALID, "%s: null data pointer", what);
  if (!isfinite((float)args->scale * kLog2e))
    return set_error(KF_ERR_INVALID, "%s: scale must be finite in single precision", what);
  const bool fused = new_k->ptr || new_v->ptr || args->slots;
  if (fused) {
    if (!new_k->ptr || !new_v->ptr || !args->slots)
      return set_error(KF_ERR_INVALID, "%s: new_k, new_v and slots go together", what);
    for (int i = 0; i < 4; ++i)
      if (new_v->size[i] != new_k->size[i])
        return set_error(KF_ERR_INVALID, "%s: new K and V shapes must match", what);
    if (new_k->size[0] != B || new_k->size[1] != Hkv || new_k->size[2] != 1 || new_k->size[3] != D)
      return set_error(KF_ERR_INVALID, "%s: new K/V must be [B, Hkv, 1, D]", what);
    if (!rows16(new_k, 2) || !rows16(new_v, 2))
      return set_error(KF_ERR_INVALID, "%s: new K/V rows must be 16-byte aligned", what);
  }
  kf::DeviceGuard guard(q->ptr);
  if (guard.status()) return guard.status();

  const int rows = unit_rows(Hq / Hkv);
  PagedArgs a;
  a.q = static_cast<const uint16_t*>(q->ptr);
  a.k = static_cast<uint16_t*>(k_pages->ptr);
  a.v = static_cast<uint16_t*>(v_pages->ptr);
  a.nk = fused ? static_cast<const uint16_t*>(new_k->ptr) : nullptr;
  a.nv = fused ? static_cast<const uint16_t*>(new_v->ptr) : nullptr;
  a.slots = args->slots;
  a.o = static_cast<uint16_t*>(args->o);
  a.lse = args->lse;
  a.table = args->block_table;
  a.lengths = args->lengths;
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = q->stride[i];
    a.nks[i] = fused ? new_k->stride[i] : 0;
    a.nvs[i] = fused ? new_v->stride[i] : 0;
  }
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = k_pages->stride[i];
    a.vs[i] = v_pages->stride[i];
  }
  a.table_stride = args->table_stride;
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.D = (int)D;
  a.page_size = (uint32_t)page_size;
  a.num_pages = (uint32_t)pages;
  a.status = args->status;
  // Boxes of 16 rows (32 where one panel or no swizzle holds a row) never cross
  // a page nor a team's keys; smaller ones where 16 does not divide the pages.
  const bool full = D == 64 || D == 128, odd = D % 16 != 0;
  a.box = D == 64 || odd ? (D <= 96 || rows > 16 ? 32 : 16) : 16;
  while (page_size % a.box) a.box /= 2;
  if (full || a.box < (odd ? 8 : 16)) {
    a.width = 8;
  } else {
    a.width = odd ? 0 : D % 32 == 0 ? 4 : 2;
  }
  const bool wide = a.width == 8;
  const int cols = wide ? 64 : a.width ? a.width * 8 : (int)D;
  // boxes of 16 rows bring all panels at once
  const int panels = wide ? (D == 128 && a.box == 16 ? 2 : 1) : (int)D / cols;
  a.box_ops = wide && D > 64 && panels == 1 ? 2 : 1;
  a.block_bytes = wide ? (D <= 64 ? 2048 : 4096) : (int)D * 32;
  a.row_bytes = wide ? 128 : (int)D * 2;
  a.box_bytes = a.box * (a.block_bytes / 16) * 2;
  // The other head dims keep the ring full: below 64 HBM is not the only bound
  // (32 requests of 8192 keys, D = 16: 65.7 us with the whole ring, 65.9 with a
  // third, D = 40: 69.5 and 70.7), 72 to 96 have two stages, of which one is
  // ahead either way, and 104 shows nothing (141 to 153 us with either).
  a.shallow = full;

  // A negative scale is taken as -q and a positive one, so that the largest
  // product is the largest score; 0 as a scale that no product survives (the
  // largest number times this is 5e-7), so that a masked -inf stays -inf.
  a.scale_log2 = fmaxf(fabsf((float)args->scale) * kLog2e, FLT_TRUE_MIN);
  a.q_sign = args->scale < 0 ? 0x80008000u : 0u;

  const int steps = head_steps(D, wide);
  int64_t blocks, most;
  int rc = plan_work(what, a, max_pages, rows, tile_keys(steps, rows), kBlocksPerSm, args->workspace,
                     args->workspace_bytes, &blocks, &most);
  if (rc != KF_OK) return rc;
  CUtensorMap mk, mv;
  rc = kf::encode_tmap_pages(&mk, k_pages, cols, a.box, panels, a.width != 0);
  if (rc != KF_OK) return rc;
  rc = kf::encode_tmap_pages(&mv, v_pages, cols, a.box, panels, a.width != 0);
  if (rc != KF_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(args->stream);
  const bool bf16 = dtype == KF_BF16;
  if (D == 64)
    rc = bf16 ? dispatch_rows<true, 4, true>(a, mk, mv, rows, (int)blocks, st)
              : dispatch_rows<false, 4, true>(a, mk, mv, rows, (int)blocks, st);
  else if (D == 128)
    rc = bf16 ? dispatch_rows<true, 8, true>(a, mk, mv, rows, (int)blocks, st)
              : dispatch_rows<false, 8, true>(a, mk, mv, rows, (int)blocks, st);
  else if (steps == 4)
    rc = bf16 ? dispatch_rows<true, 4, false>(a, mk, mv, rows, (int)blocks, st)
              : dispatch_rows<false, 4, false>(a, mk, mv, rows, (int)blocks, st);
  else if (steps == 6)
    rc = bf16 ? dispatch_rows<true, 6, false>(a, mk, mv, rows, (int)blocks, st)
              : dispatch_rows<false, 6, false>(a, mk, mv, rows, (int)blocks, st);
  else
    rc = bf16 ? dispatch_rows<true, 8, false>(a, mk, mv, rows, (int)blocks, st)
              : dispatch_rows<false, 8, false>(a, mk, mv, rows, (int)blocks, st);
  if (rc != KF_OK || most == 1) return rc;
  return launch_join(what, a, bf16, rows, blocks, st);
}
