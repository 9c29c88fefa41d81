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
// are cut into tiles.  All tiles of the call, unit after unit, form one list
// that is dealt out in equal contiguous shares to a grid that fills the GPU
// once.  Each block finds its share from the lengths by a prefix sum, so
// ragged batches are balanced without the host knowing a length (no
// synchronisation, and a captured graph follows the lengths).  A unit that
// lies inside one share is finished there; one cut by a share's end leaves
// fp32 partials (normalised O, log2 LSE) in at most two slots per block and
// is joined by a second kernel.
//
// Inside a block four warps take different keys of each tile (or, with more
// than 16 rows per KV head, 2 or 4 warps form a team that shares keys and
// splits the rows).  Each team streams its own keys through its own ring of
// shared-memory stages with 16-byte cp.async gathers: a lane resolves the
// page of one key, the addresses go round by shuffles, so pages of any size
// and any cache strides take one path, and teams never wait for one another
// inside a unit.  The ring runs ahead across unit boundaries.  The products
// are taken transposed on warp MMAs (S^T = K Q^T, O^T = V^T P^T): keys and
// head-dim fill the m = 16 side and up to 8 query rows the n = 8 side, so
// few rows waste little.
#include <math.h>

#include "kf_host.h"
#include "kf_sm100.cuh"

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kBlocksPerSm = 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PagedArgs {
  const uint16_t* q;
  uint16_t* k;             // written only by the fused append
  uint16_t* v;
  const uint16_t* nk;      // null: no fused append
  const uint16_t* nv;
  const int64_t* slots;    // of the new rows; < 0: this request has none
  uint16_t* o;
  float* lse;              // may be null
  const int32_t* table;
  const int32_t* lengths;
  float* part_o;           // [blocks][2][rows of a unit][D]
  float* part_lse;         // [blocks][2][rows of a unit], log2
  int4* joins;             // [blocks]: (request, KV head and row block, last block of the unit, -) or x = -1
  int64_t qs[2], ks[3], vs[3], nks[2], nvs[2], os[2];
  int64_t table_stride;
  int B, Hq, Hkv, G, D, row_blocks;
  uint32_t capacity;       // tokens a table row can hold
  uint32_t page_size, num_pages;
  float scale_log2;
};

// Variants: NP = 64-column panels of the padded head dim; NT = 8-row tiles of
// query rows per warp; RG = warps of a team (row groups).
template <int NP, int NT, int RG>
struct Cfg {
  static constexpr int DP = NP * 64;
  static constexpr int KW = (NP == 2 && RG == 1) ? 16 : 32;  // keys a team takes of a tile
  static constexpr int TEAMS = kWarps / RG;
  static constexpr int TILE = TEAMS * KW;                    // keys of a tile
  static constexpr int ROWS = NT * 8 * RG;                   // query rows of a unit
  static constexpr int STAGE = KW * DP * 2 * 2;              // bytes: K rows, then V rows
  static constexpr int STAGES = 98304 / (TEAMS * STAGE);     // 96 KB of ring per block, two blocks per SM
  static constexpr int PASS = 64 / NT < DP ? 64 / NT : DP;   // head-dim columns joined per pass of the epilogue
  static constexpr int OSTRIDE = PASS + 4;                   // keeps the four row pairs of a store on separate banks
  static constexpr int SMEM = TEAMS * STAGES * STAGE + kWarps * NT * 8 * OSTRIDE * 4 + kWarps * NT * 8 * 2 * 4;
};

__device__ __forceinline__ uint32_t swz(int row, int chunk, int row_bytes) {
  return (uint32_t)(row * row_bytes + ((((chunk & 7) ^ (row & 7)) | (chunk & ~7)) << 4));
}

__device__ __forceinline__ uint32_t visible(const PagedArgs& a, int b) {
  const int32_t n = a.lengths[b];
  return n <= 0 ? 0u : min((uint32_t)n, a.capacity);
}

// Position in the list of tiles: tile `t` of the `tiles` of unit (b, hr).
template <int TILE>
struct Cursor {
  int b, hr;
  uint32_t t, tiles, keys;

  __device__ __forceinline__ void set_request(const PagedArgs& a, int request) {
    b = request;
    keys = visible(a, b);
    tiles = (keys + TILE - 1) / TILE;
  }
  // true when the next tile belongs to another unit
  __device__ __forceinline__ bool next(const PagedArgs& a, int units) {
    if (++t < tiles) return false;
    t = 0;
    if (++hr == units) {
      hr = 0;
      do {
        set_request(a, b + 1);
      } while (tiles == 0 && b + 1 < a.B);
    }
    return true;
  }
};

template <int RG>
__device__ __forceinline__ void team_sync(int team) {
  if constexpr (RG == 1)
    __syncwarp();
  else if constexpr (RG == kWarps)
    __syncthreads();
  else
    kf::named_bar_sync(1 + team, RG * 32);
}

__device__ __forceinline__ uint64_t shfl64(uint64_t x, int src) {
  return __shfl_sync(0xffffffffu, (unsigned long long)x, src);
}

template <bool BF16, int NP, int NT, int RG>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) paged_decode_kernel(const PagedArgs a) {
  using C = Cfg<NP, NT, RG>;
  constexpr int DP = C::DP, KW = C::KW, STAGES = C::STAGES, TILE = C::TILE;
  constexpr int H = KW / 16;           // 16-key halves of a step
  constexpr int ROW_BYTES = DP * 2;
  constexpr int CHUNKS = DP / 8;       // 16-byte chunks of a row
  constexpr int K_BYTES = KW * ROW_BYTES;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t warp_tiles[kWarps];
  __shared__ int first_request;
  __shared__ int64_t first_before;     // tiles of the requests before it
  __shared__ uint32_t seen_s[C::TEAMS][STAGES];  // visible keys of each stage

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int team = warp / RG, rg = warp % RG;
  const int units = a.Hkv * a.row_blocks;  // per request
  uint8_t* ring = smem + team * STAGES * C::STAGE;
  float* obuf = reinterpret_cast<float*>(smem + C::TEAMS * STAGES * C::STAGE);  // [warp][NT * 8][OSTRIDE]
  float* ml = obuf + kWarps * NT * 8 * C::OSTRIDE;                              // [warp][NT * 8][2]

  // columns [D, DP) of every stage stay zero: they add nothing to K Q^T
  if (a.D < DP) {
    const int pad = CHUNKS - a.D / 8;
    constexpr int ALL = C::TEAMS * STAGES * 2 * KW;  // K and V rows of all rings
    for (int i = tid; i < ALL * pad; i += kThreads) {
      const int r = i / pad, c = a.D / 8 + i % pad;
      *reinterpret_cast<uint4*>(smem + (r / KW) * K_BYTES + swz(r % KW, c, ROW_BYTES)) = make_uint4(0, 0, 0, 0);
    }
  }
  kf::griddep_wait();
  kf::griddep_launch_dependents();

  // ---- this block's share of the list of tiles
  const int per = (a.B + kThreads - 1) / kThreads;  // requests per thread, contiguous
  const int b_lo = min(tid * per, a.B), b_hi = min(b_lo + per, a.B);
  int64_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += (visible(a, b) + TILE - 1) / TILE;
  int64_t upto = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, (long long)upto, off);
    if (lane >= off) upto += y;
  }
  if (lane == 31) warp_tiles[warp] = upto;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += warp_tiles[w];
    total += warp_tiles[w];
  }
  const int64_t list = total * units;
  const int64_t shares = min((int64_t)gridDim.x, list);
  const int64_t me = blockIdx.x;

  // requests without a visible position are nobody's unit
  for (int64_t b = me; b < a.B; b += gridDim.x) {
    if (visible(a, (int)b) != 0) continue;
    for (int i = tid; i < a.Hq * (a.D / 8); i += kThreads) {
      const int h = i / (a.D / 8), c = i % (a.D / 8);
      *reinterpret_cast<uint4*>(a.o + b * a.os[0] + h * a.os[1] + c * 8) = make_uint4(0, 0, 0, 0);
    }
    if (a.lse)
      for (int h = tid; h < a.Hq; h += kThreads) a.lse[b * a.Hq + h] = -INFINITY;
  }
  if (me >= shares) {
    if (tid == 0 && a.joins) a.joins[me].x = -1;
    return;
  }
  const int64_t begin = me * list / shares;
  const int n = (int)((me + 1) * list / shares - begin);
  {
    const int64_t before = (upto - mine) * units;
    if (begin >= before && begin < upto * units) {  // exactly one thread
      int64_t sum = upto - mine;
      int b = b_lo;
      while (true) {
        const int64_t tiles = (visible(a, b) + TILE - 1) / TILE;
        if (begin < (sum + tiles) * units) break;
        sum += tiles;
        ++b;
      }
      first_request = b;
      first_before = sum;
    }
  }
  __syncthreads();

  Cursor<TILE> load, work;
  work.set_request(a, first_request);
  {
    const int64_t at = begin - first_before * units;  // inside the request's tiles x units
    work.hr = (int)(at / work.tiles);
    work.t = (uint32_t)(at - (int64_t)work.hr * work.tiles);
  }
  load = work;

  // ---- loads: lane r (of KW) resolves key r of the team's share of the tile
  int32_t next_page;       // of the tile the load cursor stands on, loaded one step ahead
  uint32_t next_row;
  bool next_in;
  auto look_up = [&]() {
    const uint32_t key = load.t * TILE + team * KW + (KW == 32 ? lane : (lane & 15));
    next_in = key < load.keys;
    const uint32_t pg = next_in ? key / a.page_size : 0;
    next_row = key - pg * a.page_size;
    next_page = next_in ? __ldg(a.table + load.b * a.table_stride + pg) : -1;
  };
  auto issue = [&](int stage) {
    const int h = load.hr / a.row_blocks, rb = load.hr - h * a.row_blocks;
    const bool valid = next_in && (uint32_t)next_page < a.num_pages;
    const uint32_t seen = __ballot_sync(0xffffffffu, valid) & (KW == 32 ? 0xffffffffu : 0xffffu);
    uint64_t row_k = 0, row_v = 0;
    if (valid) {
      row_k = reinterpret_cast<uint64_t>(a.k + next_page * a.ks[0] + h * a.ks[1] + next_row * a.ks[2]);
      row_v = reinterpret_cast<uint64_t>(a.v + next_page * a.vs[0] + h * a.vs[1] + next_row * a.vs[2]);
    }
    if (a.nk) {
      // the newest position comes from the caller's row, and one warp stores it
      const uint32_t r = (uint32_t)a.lengths[load.b] - 1 - (load.t * TILE + team * KW);
      if (r < (uint32_t)KW && ((seen >> r) & 1) && a.slots[load.b] >= 0) {
        const uint64_t src_k = reinterpret_cast<uint64_t>(a.nk + load.b * a.nks[0] + h * a.nks[1]);
        const uint64_t src_v = reinterpret_cast<uint64_t>(a.nv + load.b * a.nvs[0] + h * a.nvs[1]);
        const uint64_t dst_k = shfl64(row_k, r), dst_v = shfl64(row_v, r);
        if (rb == 0 && rg == 0 && (lane & 15) < a.D / 8) {
          const uint4* src = reinterpret_cast<const uint4*>(lane < 16 ? src_k : src_v) + (lane & 15);
          uint4* dst = reinterpret_cast<uint4*>(lane < 16 ? dst_k : dst_v) + (lane & 15);
          *dst = *src;
        }
        if ((uint32_t)(KW == 32 ? lane : (lane & 15)) == r) {
          row_k = src_k;
          row_v = src_v;
        }
      }
    }
    uint8_t* st = ring + stage * C::STAGE;
#pragma unroll
    for (int i = 0; i < KW * CHUNKS / (32 * RG); ++i) {
      const int idx = i * 32 * RG + rg * 32 + lane;
      const int r = idx / CHUNKS, c = idx % CHUNKS;
      const uint64_t sk = shfl64(row_k, r), sv = shfl64(row_v, r);
      const bool ok = (seen >> r) & 1;
      if (c * 8 < a.D) {
        const uint32_t at = swz(r, c, ROW_BYTES);
        kf::cp_async16(st + at, reinterpret_cast<const uint4*>(ok ? sk : (uint64_t)a.k) + (ok ? c : 0), ok);
        kf::cp_async16(st + K_BYTES + at, reinterpret_cast<const uint4*>(ok ? sv : (uint64_t)a.v) + (ok ? c : 0), ok);
      }
    }
    if (rg == 0 && lane == 0) seen_s[team][stage] = seen;
  };

  // ---- state of the unit being worked on
  uint32_t qb[NT][DP / 16][2];         // Q^T as B fragments
  float m_run[NT][2], l_run[NT][2];    // rows 2 (lane % 4) + {0, 1} of each row tile
  float ot[NT][DP / 16][4];            // O^T
  auto start_unit = [&]() {
    const int h = work.hr / a.row_blocks, rb = work.hr - h * a.row_blocks;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = rb * C::ROWS + rg * NT * 8 + nt * 8 + (lane >> 2);
      const uint16_t* src = a.q + work.b * a.qs[0] + (int64_t)(h * a.G + row) * a.qs[1] + 2 * (lane & 3);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qb[nt][kk][e] = (row < a.G && kk * 16 + e * 8 < a.D)
                              ? __ldg(reinterpret_cast<const uint32_t*>(src + kk * 16 + e * 8)) : 0u;
        ot[nt][kk][0] = ot[nt][kk][1] = ot[nt][kk][2] = ot[nt][kk][3] = 0.f;
      }
      m_run[nt][0] = m_run[nt][1] = -INFINITY;
      l_run[nt][0] = l_run[nt][1] = 0.f;
    }
  };

  look_up();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (s < n) {
      issue(s);
      if (s + 1 < n) {
        load.next(a, units);
        look_up();
      }
    }
    kf::cp_async_commit();
  }
  start_unit();
  uint32_t unit_t0 = work.t;           // first tile of the unit in this share
  if (tid == 0 && a.joins) a.joins[me].x = -1;

  int stage = 0, fill = STAGES - 1;
  for (int i = 0; i < n; ++i) {
    kf::cp_async_wait<STAGES - 2>();
    team_sync<RG>(team);               // stage i has landed for the team, stage i - 1 is free
    if (i + STAGES - 1 < n) {
      issue(fill);
      if (i + STAGES < n) {
        load.next(a, units);
        look_up();
      }
    }
    kf::cp_async_commit();

    const uint32_t seen = seen_s[team][stage];
    if (seen != 0) {
      const uint32_t sk = kf::smem_u32(ring + stage * C::STAGE), sv = sk + K_BYTES;
      // S^T (keys x rows)
      float c[H][NT][4];
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[h][nt][0] = c[h][nt][1] = c[h][nt][2] = c[h][nt][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          uint32_t ka[4];
          kf::ldmatrix_x4(ka, sk + swz(h * 16 + (lane & 15), 2 * kk + (lane >> 4), ROW_BYTES));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) kf::mma_16816<BF16>(c[h][nt], ka, qb[nt][kk][0], qb[nt][kk][1]);
        }
      uint32_t pb[H][NT][2], pl[H][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // rows 2 (lane % 4) + {0, 1}; keys 16 h + lane / 4 (c0, c1) and + 8 (c2, c3)
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const uint32_t bits = seen >> (h * 16 + (lane >> 2));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            c[h][nt][e] = (bits & (e < 2 ? 1u : 256u)) ? c[h][nt][e] * a.scale_log2 : -INFINITY;
          mx[0] = kf::fmax3(mx[0], c[h][nt][0], c[h][nt][2]);
          mx[1] = kf::fmax3(mx[1], c[h][nt][1], c[h][nt][3]);
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
        }
        float alpha[2], mu[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float m_new = fmaxf(m_run[nt][j], mx[j]);
          mu[j] = m_new == -INFINITY ? 0.f : m_new;
          alpha[j] = kf::ex2(m_run[nt][j] - mu[j]);
          m_run[nt][j] = m_new;
        }
        float ls[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < H; ++h) {
          float p[4], r[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = kf::ex2(c[h][nt][e] - mu[e & 1]);
            ls[e & 1] += p[e];
          }
          // P as a 16-bit value plus the 16-bit rest: two products keep the
          // weights at about fp32 accuracy, as a plain fp32 softmax has them
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t hi = kf::pack2<BF16>(p[2 * x], p[2 * x + 1]);
            const float2 back = kf::unpack2<BF16>(hi);
            r[2 * x] = p[2 * x] - back.x;
            r[2 * x + 1] = p[2 * x + 1] - back.y;
            pb[h][nt][x] = kf::movmatrix_trans(hi);
            pl[h][nt][x] = kf::movmatrix_trans(kf::pack2<BF16>(r[2 * x], r[2 * x + 1]));
          }
        }
        l_run[nt][0] = l_run[nt][0] * alpha[0] + ls[0];
        l_run[nt][1] = l_run[nt][1] * alpha[1] + ls[1];
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
          for (int dm = 0; dm < DP / 16; ++dm) {
            ot[nt][dm][0] *= alpha[0];
            ot[nt][dm][1] *= alpha[1];
            ot[nt][dm][2] *= alpha[0];
            ot[nt][dm][3] *= alpha[1];
          }
        }
      }
      // O^T (head dim x rows) += V^T P^T
#pragma unroll
      for (int dm = 0; dm < DP / 16; ++dm)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          uint32_t va[4];
          kf::ldmatrix_x4_trans(va, sv + swz(h * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * dm + ((lane >> 3) & 1),
                                             ROW_BYTES));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            kf::mma_16816<BF16>(ot[nt][dm], va, pb[h][nt][0], pb[h][nt][1]);
            kf::mma_16816<BF16>(ot[nt][dm], va, pl[h][nt][0], pl[h][nt][1]);
          }
        }
    }
    if (++stage == STAGES) stage = 0;
    if (++fill == STAGES) fill = 0;

    const bool unit_done = work.t + 1 == work.tiles;
    if (!unit_done && i + 1 < n) {
      ++work.t;
      continue;
    }
    // ---- join the teams and write the unit's rows (or its partial)
    const int h = work.hr / a.row_blocks, rb = work.hr - h * a.row_blocks;
    const bool direct = unit_t0 == 0 && unit_done;
    const int64_t slot = me * 2 + (unit_t0 > 0 ? 0 : 1);  // 0: began in an earlier share, 1: begins here
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], off);
#pragma unroll
    for (int pass = 0; pass < DP / C::PASS; ++pass) {
      __syncthreads();  // the buffer's readers of the pass (or unit) before are done
      if (pass == 0 && lane < 4) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            ml[(warp * NT * 8 + nt * 8 + 2 * lane + j) * 2 + 0] = m_run[nt][j];
            ml[(warp * NT * 8 + nt * 8 + 2 * lane + j) * 2 + 1] = l_run[nt][j];
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float* row = obuf + (warp * NT * 8 + nt * 8 + 2 * (lane & 3) + j) * C::OSTRIDE;
#pragma unroll
          for (int x = 0; x < C::PASS / 16; ++x) {
            const int dm = pass * (C::PASS / 16) + x;
            row[x * 16 + (lane >> 2)] = ot[nt][dm][j];
            row[x * 16 + (lane >> 2) + 8] = ot[nt][dm][2 + j];
          }
        }
      __syncthreads();
      const int valid_rows = min(C::ROWS, a.G - rb * C::ROWS);
      for (int idx = tid; idx < valid_rows * (C::PASS / 4); idx += kThreads) {
        const int r = idx / (C::PASS / 4), col = (idx % (C::PASS / 4)) * 4;
        const int d = pass * C::PASS + col;
        if (d >= a.D) continue;
        const int group = r / (NT * 8), in = r % (NT * 8);
        float M = -INFINITY;
#pragma unroll
        for (int t = 0; t < C::TEAMS; ++t) M = fmaxf(M, ml[((t * RG + group) * NT * 8 + in) * 2]);
        float L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < C::TEAMS; ++t) {
          const int w = (t * RG + group) * NT * 8 + in;
          const float wt = M == -INFINITY ? 0.f : kf::ex2(ml[w * 2] - M);
          L += wt * ml[w * 2 + 1];
          const float4 x = *reinterpret_cast<const float4*>(obuf + w * C::OSTRIDE + col);
          acc[0] += wt * x.x;
          acc[1] += wt * x.y;
          acc[2] += wt * x.z;
          acc[3] += wt * x.w;
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const float lse2 = L == 0.f ? -INFINITY : M + log2f(L);
        const int head = h * a.G + rb * C::ROWS + r;
        if (direct) {
          *reinterpret_cast<uint2*>(a.o + work.b * a.os[0] + head * a.os[1] + d) =
              make_uint2(kf::pack2<BF16>(acc[0] * inv, acc[1] * inv), kf::pack2<BF16>(acc[2] * inv, acc[3] * inv));
          if (a.lse && d == 0) a.lse[(int64_t)work.b * a.Hq + head] = lse2 * kLn2;
        } else {
          *reinterpret_cast<float4*>(a.part_o + (slot * C::ROWS + r) * a.D + d) =
              make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
          if (d == 0) a.part_lse[slot * C::ROWS + r] = lse2;
        }
      }
    }
    if (!direct && unit_t0 == 0 && tid == 0) {
      // begins here and goes on: the share that holds list position p is ((p + 1) shares - 1) / list
      const int64_t last_tile = begin + i + (work.tiles - 1 - work.t);
      a.joins[me] = make_int4(work.b, work.hr, (int)(((last_tile + 1) * shares - 1) / list), 0);
    }
    if (i + 1 < n) {
      work.next(a, units);
      start_unit();
      unit_t0 = 0;
    }
  }
}

// Joins the partials of the unit that begins in share blockIdx.x and goes on:
// slot 1 of that share, slot 0 of the shares up to the unit's last.  One row
// per block; groups of D / 4 lanes take every groups-th partial with a
// running maximum, so each partial is read once and in any number.
constexpr int kJoinThreads = 256;
constexpr int kJoinBatch = 4;  // partials a group has in flight

template <bool BF16>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedArgs a, int rows) {
  kf::griddep_wait();
  kf::griddep_launch_dependents();
  const int4 unit = a.joins[blockIdx.x];
  if (unit.x < 0) return;
  const int h = unit.y / a.row_blocks, rb = unit.y - h * a.row_blocks;
  const int r = blockIdx.y;
  if (r >= a.G - rb * rows) return;
  const int count = unit.z - (int)blockIdx.x + 1;
  __shared__ float4 acc_s[kJoinThreads];
  __shared__ float m_s[kJoinThreads / 4], l_s[kJoinThreads / 4];
  const int lanes = a.D / 4, groups = kJoinThreads / lanes;
  const int g = threadIdx.x / lanes, c = threadIdx.x % lanes;
  if (g < groups) {
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = g; j0 < count; j0 += groups * kJoinBatch) {
      float lse[kJoinBatch];
      float4 o[kJoinBatch];
#pragma unroll
      for (int x = 0; x < kJoinBatch; ++x) {
        const int j = j0 + x * groups;
        lse[x] = -INFINITY;
        o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j < count) {
          const int64_t row = (((int64_t)blockIdx.x + j) * 2 + (j == 0 ? 1 : 0)) * rows + r;
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
    acc_s[threadIdx.x] = acc;
    if (c == 0) {
      m_s[g] = m;
      l_s[g] = l;
    }
  }
  __syncthreads();
  if (g != 0) return;
  float M = -INFINITY;
  for (int i = 0; i < groups; ++i) M = fmaxf(M, m_s[i]);
  const float mu = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < groups; ++i) {
    const float w = kf::ex2(m_s[i] - mu);
    const float4 x = acc_s[i * lanes + c];
    L += w * l_s[i];
    acc.x += w * x.x;
    acc.y += w * x.y;
    acc.z += w * x.z;
    acc.w += w * x.w;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int head = h * a.G + rb * rows + r;
  *reinterpret_cast<uint2*>(a.o + unit.x * a.os[0] + head * a.os[1] + c * 4) =
      make_uint2(kf::pack2<BF16>(acc.x * inv, acc.y * inv), kf::pack2<BF16>(acc.z * inv, acc.w * inv));
  if (a.lse && c == 0) a.lse[(int64_t)unit.x * a.Hq + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// Query rows of a unit for G rows per KV head, and the variant that has them.
int unit_rows(int64_t G) { return G <= 8 ? 8 : G <= 16 ? 16 : G <= 32 ? 32 : 64; }

// Keys per tile of the variant (Cfg::TILE).
int tile_keys(int64_t D, int rows) { return rows <= 16 ? (D <= 64 ? 128 : 64) : rows == 32 ? 64 : 32; }

size_t workspace_need(int blocks, int rows, int64_t D) {
  return 256 + (size_t)blocks * (16 + (size_t)2 * rows * 4 + (size_t)2 * rows * D * 4);
}

template <bool BF16, int NP, int NT, int RG>
int launch_variant(const PagedArgs& a, int blocks, cudaStream_t st) {
  using C = Cfg<NP, NT, RG>;
  static_assert(C::STAGES >= 3, "the ring needs three stages");
  auto kern = paged_decode_kernel<BF16, NP, NT, RG>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) {
    (void)cudaGetLastError();
    return kf::set_error(KF_ERR_CUDA, "kf_paged_decode: cannot reserve %d bytes of shared memory", C::SMEM);
  }
  return kf::launch_dependent(kern, dim3((unsigned)blocks), dim3(kThreads), C::SMEM, st, "kf_paged_decode", a);
}

template <bool BF16, int NP>
int dispatch_rows(const PagedArgs& a, int rows, int blocks, cudaStream_t st) {
  switch (rows) {
    case 8: return launch_variant<BF16, NP, 1, 1>(a, blocks, st);
    case 16: return launch_variant<BF16, NP, 2, 1>(a, blocks, st);
    case 32: return launch_variant<BF16, NP, 2, 2>(a, blocks, st);
    default: return launch_variant<BF16, NP, 2, 4>(a, blocks, st);
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

extern "C" int kf_paged_decode(const kf_tensor4* q, const kf_tensor4* k_pages, const kf_tensor4* v_pages,
                               const int32_t* block_table, int64_t max_pages, int64_t table_stride,
                               const int32_t* lengths, const kf_tensor4* new_k, const kf_tensor4* new_v,
                               const int64_t* slots, const kf_tensor4* o, float* lse, int dtype, float scale, void* workspace,
                               size_t workspace_bytes, void* stream) {
  using kf::set_error;
  const char* what = "kf_paged_decode";
  if (!q || !k_pages || !v_pages || !o) return set_error(KF_ERR_INVALID, "%s: null tensor descriptor", what);
  if (dtype != KF_F16 && dtype != KF_BF16) return set_error(KF_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  const int64_t B = q->size[0], Hq = q->size[1], D = q->size[3];
  const int64_t pages = k_pages->size[0], Hkv = k_pages->size[1], page_size = k_pages->size[2];
  for (int i = 0; i < 4; ++i) {
    if (k_pages->size[i] != v_pages->size[i])
      return set_error(KF_ERR_INVALID, "%s: K/V page shapes must match", what);
    if (o->size[i] != q->size[i]) return set_error(KF_ERR_INVALID, "%s: O must have Q's shape", what);
  }
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
  if (!rows16(q, 2) || !rows16(k_pages, 3) || !rows16(v_pages, 3) || !rows16(o, 2))
    return set_error(KF_ERR_INVALID, "%s: tensors need a contiguous last dim and 16-byte aligned rows", what);
  if (!q->ptr || !k_pages->ptr || !v_pages->ptr || !o->ptr || !block_table || !lengths)
    return set_error(KF_ERR_INVALID, "%s: null data pointer", what);
  const bool fused = new_k != nullptr || new_v != nullptr;
  if (fused) {
    if (!new_k || !new_v) return set_error(KF_ERR_INVALID, "%s: new_k and new_v go together", what);
    for (int i = 0; i < 4; ++i)
      if (new_v->size[i] != new_k->size[i])
        return set_error(KF_ERR_INVALID, "%s: new K and V shapes must match", what);
    if (new_k->size[0] != B || new_k->size[1] != Hkv || new_k->size[2] != 1 || new_k->size[3] != D)
      return set_error(KF_ERR_INVALID, "%s: new K/V must be [B, Hkv, 1, D]", what);
    if (!rows16(new_k, 2) || !rows16(new_v, 2))
      return set_error(KF_ERR_INVALID, "%s: new K/V rows must be 16-byte aligned", what);
    if (!new_k->ptr || !new_v->ptr || !slots) return set_error(KF_ERR_INVALID, "%s: null data pointer", what);
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
  a.slots = slots;
  a.o = static_cast<uint16_t*>(o->ptr);
  a.lse = lse;
  a.table = block_table;
  a.lengths = lengths;
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = q->stride[i];
    a.os[i] = o->stride[i];
    a.nks[i] = fused ? new_k->stride[i] : 0;
    a.nvs[i] = fused ? new_v->stride[i] : 0;
  }
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = k_pages->stride[i];
    a.vs[i] = v_pages->stride[i];
  }
  a.table_stride = table_stride;
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.D = (int)D;
  a.row_blocks = (a.G + rows - 1) / rows;
  const int64_t capacity = max_pages * page_size;
  a.capacity = (uint32_t)(capacity < 0x7fffffffLL ? capacity : 0x7fffffffLL);
  a.page_size = (uint32_t)page_size;
  a.num_pages = (uint32_t)pages;
  a.scale_log2 = scale * kLog2e;

  // One wave of blocks, or fewer when the tables cannot hold that many tiles.
  // A unit of one tile is never cut, so nothing is left to join.
  const int64_t tile = tile_keys(D, rows), most = (a.capacity + tile - 1) / tile;
  const int64_t units = B * Hkv * a.row_blocks;
  int64_t blocks = (int64_t)kf::sm_count_current_device() * kBlocksPerSm;
  if (units * most > (int64_t)1 << 38) return set_error(KF_ERR_UNSUPPORTED, "%s: tensors too large", what);
  if (units * most < blocks) blocks = units * most;
  a.part_o = nullptr;
  a.part_lse = nullptr;
  a.joins = nullptr;
  if (most > 1) {
    const size_t need = workspace_need((int)blocks, rows, D);
    if (!workspace || workspace_bytes < need)
      return set_error(KF_ERR_WORKSPACE, "%s: workspace needs %zu bytes", what, need);
    uintptr_t base = (reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255);
    a.joins = reinterpret_cast<int4*>(base);
    a.part_o = reinterpret_cast<float*>(a.joins + blocks);
    a.part_lse = a.part_o + (size_t)blocks * 2 * rows * D;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = dtype == KF_BF16;
  int rc;
  if (D <= 64)
    rc = bf16 ? dispatch_rows<true, 1>(a, rows, (int)blocks, st) : dispatch_rows<false, 1>(a, rows, (int)blocks, st);
  else
    rc = bf16 ? dispatch_rows<true, 2>(a, rows, (int)blocks, st) : dispatch_rows<false, 2>(a, rows, (int)blocks, st);
  if (rc != KF_OK || most == 1) return rc;
  const dim3 grid((unsigned)blocks, (unsigned)(a.G < rows ? a.G : rows));
  return bf16 ? kf::launch_dependent(paged_join_kernel<true>, grid, dim3(kJoinThreads), 0, st, what, a, rows)
              : kf::launch_dependent(paged_join_kernel<false>, grid, dim3(kJoinThreads), 0, st, what, a, rows);
}
