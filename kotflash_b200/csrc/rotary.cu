// K7: rotary positions.  Column pairs (a, b) of every head of Q and K are
// turned by the angle t = position * frequency of the pair:
//   a' = (a cos t - b sin t) m,  b' = (b cos t + a sin t) m,
// the columns behind the rotated ones pass unchanged.  The gradient is the
// same with -t.  Pairs are column i with i + R / 2, or 2 i with 2 i + 1.
//
// Every element is read and written once (4 bytes for 3 flops), so HBM
// bounds it: 4 x 4096 tokens of 32 and 8 heads of 128 columns take 53.4 us, 96%
// of the measured copy rate.  cos and sin depend on the token and the pair
// only: a thread keeps those of its pairs in registers and takes four heads,
// which it asks for before it works the angles out.  (Angles shared by a block
// through shared memory, all heads of a few tokens per block: 64 to 90 us, the
// barriers cost more than the angles.)
//
// Frequencies become whole numbers of 2^-64 turns, so a product with the
// position modulo 2^64 is the angle modulo a turn, with no reduction to make;
// its upper half, 2^-32 turns, goes to cos_sin().  A double holds a frequency
// in turns to 2^-52 of itself after its roundings, so an angle of A turns is
// off by A 2^-52 turns besides: below the 2^-23 of cos_sin() up to 2^26 turns,
// which is as far as the same product in doubles goes (a frequency of 1 at
// position 2^28; at 2^31 it is off by 2^-21 radians).
#include <math.h>

#include <type_traits>

#include "kf_host.h"
#include "kf_sm100.cuh"

namespace {

constexpr int kThreads = 128;
constexpr int kHeads = 4;  // of a thread, at most

struct RotaryArgs {
  const uint16_t* x[2];    // Q and K
  uint16_t* y[2];
  int64_t xs[2][3], ys[2][3];
  const void* positions;
  int64_t ps[2];
  const double* frequencies;
  uint32_t tokens, S;      // in all, and per batch entry
  uint32_t items;          // threads per token
  uint32_t turning;        // of them, those with rotated columns
  int heads[2], chunk;     // of Q and K; heads of a block
  int R;
  bool wide;               // positions are 64-bit
  float magnitude, sign;
};

template <int VEC>
struct Vec {
  using type = typename std::conditional<VEC == 8, uint4,
               typename std::conditional<VEC == 4, uint2, typename std::conditional<VEC == 2, uint32_t, uint16_t>::type>::type>::type;
};

// VEC 16-bit values.  Loads go through L2: the predecessor may have written
// them while this kernel was alive.
template <int VEC>
struct Block {
  uint32_t w[VEC > 1 ? VEC / 2 : 1];
  __device__ __forceinline__ void load(const uint16_t* p) {
    using T = typename Vec<VEC>::type;
    const T v = __ldcg(reinterpret_cast<const T*>(p));
    if constexpr (VEC == 8) {
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (VEC == 4) {
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = v;
    }
  }
  __device__ __forceinline__ void store(uint16_t* p) const {
    if constexpr (VEC == 8)
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (VEC == 4)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (VEC == 2)
      *reinterpret_cast<uint32_t*>(p) = w[0];
    else
      *p = (uint16_t)w[0];
  }
};

// cos and sin of `turn` / 2^32 turns.  The quarter nearest to it leaves t in
// +-pi / 4, for which sin t = t + t z (a1 + a2 z + a3 z^2) and cos t = 1 + z (b1 +
// b2 z + b3 z^2), z = t^2, with coefficients fitted to the least largest error
// on that interval (by iterated reweighted least squares): 2^-29 and 2^-24.9.
// With the roundings of t and of the sums both are off by 2^-23 at most.
__device__ __forceinline__ void cos_sin(uint32_t turn, float& c, float& s) {
  const uint32_t quarter = turn + 0x20000000u;
  const float t = (float)(int32_t)((quarter & 0x3fffffffu) - 0x20000000u) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float z = t * t;
  float x = fmaf(fmaf(fmaf(-0.00019495567673f, z, 0.00833197812420f), z, -0.16666650659734f) * z, t, t);
  float y = fmaf(fmaf(fmaf(-0.00135977654526f, z, 0.04165629045595f), z, -0.49999894718539f), z, 1.f);
  if (quarter & 0x40000000u) {  // t + pi / 2
    const float w = x;
    x = y;
    y = -w;
  }
  const uint32_t half = quarter & 0x80000000u;  // t + pi
  c = __uint_as_float(__float_as_uint(y) ^ half);
  s = __uint_as_float(__float_as_uint(x) ^ half);
}

// HALVES: a thread turns columns j .. j + VEC - 1 with those R / 2 behind
// them; else columns j .. j + VEC - 1 hold its pairs (VEC = 1: j and j + 1,
// one value at a time).
template <int VEC, bool HALVES, bool BF16>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  constexpr int PAIRS = HALVES ? VEC : VEC > 1 ? VEC / 2 : 1;
  constexpr bool TWO = HALVES || VEC == 1;   // two loads per head
  // Frequencies in 2^-64 turns.  From shared memory: read by every thread through
  // L2 they are one line that all SMs ask for (4 x 4096 tokens: 110 us).
  extern __shared__ uint64_t turns_s[];
  kf::griddep_wait();
  kf::griddep_launch_dependents();
  for (int i = threadIdx.x; i < a.R / 2; i += kThreads) {
    const double turns = __ldcg(a.frequencies + i) * 0.15915494309189535;
    turns_s[i] = __double2ull_rz((turns - floor(turns)) * 18446744073709551616.0);
  }
  const uint32_t index = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t token = index / a.items, item = index - token * a.items;
  const bool here = token < a.tokens;
  const uint32_t n = token / a.S, s = token - n * a.S;
  const int h0 = blockIdx.y * a.chunk, h1 = here ? min(h0 + a.chunk, a.heads[0] + a.heads[1]) : h0;
  const bool turns = item < a.turning;
  // columns of this thread: j, and `other` for the second load of a pair
  const int j = turns ? (int)item * (HALVES ? VEC : 2 * PAIRS) : a.R + (int)(item - a.turning) * VEC;
  const int other = HALVES ? j + a.R / 2 : j + 1;

  auto at = [&](const int64_t (&st)[2][3], int h) {
    const int which = h >= a.heads[0];
    return (int64_t)n * st[which][0] + (int64_t)(h - (which ? a.heads[0] : 0)) * st[which][1] + (int64_t)s * st[which][2];
  };
  Block<VEC> u[kHeads], v[kHeads];
  auto load = [&](int h, int x) {
    const uint16_t* p = a.x[h >= a.heads[0]] + at(a.xs, h);
    u[x].load(p + j);
    if (TWO && turns) v[x].load(p + other);
  };
  // the heads' values travel while the angles are worked out
#pragma unroll
  for (int x = 0; x < kHeads; ++x)
    if (h0 + x < h1) load(h0 + x, x);

  float c[PAIRS], d[PAIRS];
  __syncthreads();
  if (here && turns) {
    const int64_t where = (int64_t)n * a.ps[0] + (int64_t)s * a.ps[1];
    const int64_t position = a.wide ? __ldcg(static_cast<const long long*>(a.positions) + where)
                                    : __ldcg(static_cast<const int*>(a.positions) + where);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      cos_sin((uint32_t)((uint64_t)position * turns_s[(HALVES ? j : j / 2) + i] >> 32), c[i], d[i]);
      c[i] *= a.magnitude;
      d[i] *= a.magnitude * a.sign;
    }
  }
#pragma unroll
  for (int x = 0; x < kHeads; ++x) {
    if (h0 + x >= h1) continue;
    uint16_t* p = a.y[h0 + x >= a.heads[0]] + at(a.ys, h0 + x);
    if (turns) {
      if constexpr (HALVES && VEC > 1) {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const float2 r = kf::unpack2<BF16>(u[x].w[i]), q = kf::unpack2<BF16>(v[x].w[i]);
          u[x].w[i] = kf::pack2<BF16>(r.x * c[2 * i] - q.x * d[2 * i], r.y * c[2 * i + 1] - q.y * d[2 * i + 1]);
          v[x].w[i] = kf::pack2<BF16>(q.x * c[2 * i] + r.x * d[2 * i], q.y * c[2 * i + 1] + r.y * d[2 * i + 1]);
        }
      } else if constexpr (!HALVES && VEC > 1) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          const float2 r = kf::unpack2<BF16>(u[x].w[i]);
          u[x].w[i] = kf::pack2<BF16>(r.x * c[i] - r.y * d[i], r.y * c[i] + r.x * d[i]);
        }
      } else {
        const float r = kf::unpack2<BF16>(u[x].w[0]).x, q = kf::unpack2<BF16>(v[x].w[0]).x;
        u[x].w[0] = kf::pack2<BF16>(r * c[0] - q * d[0], 0.f);
        v[x].w[0] = kf::pack2<BF16>(q * c[0] + r * d[0], 0.f);
      }
    }
    u[x].store(p + j);
    if (TWO && turns) v[x].store(p + other);
  }
}

// Whether rows of `t` can be moved in pieces of `vec` values.
bool fits(const kf_tensor4& t, int vec) {
  if (reinterpret_cast<uintptr_t>(t.ptr) % (2 * vec)) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size[i] > 1 && t.stride[i] % vec) return false;
  return true;
}

template <int VEC, bool HALVES>
int launch(RotaryArgs& a, int D, bool bf16, cudaStream_t st) {
  const char* what = "kf_rotary";
  a.turning = HALVES ? a.R / 2 / VEC : a.R / (VEC > 1 ? VEC : 2);
  a.items = a.turning + (D - a.R) / VEC;
  const int64_t threads = (int64_t)a.tokens * a.items, heads = a.heads[0] + a.heads[1];
  if (threads > 0x7fffffffLL - kThreads) return kf::set_error(KF_ERR_UNSUPPORTED, "%s: too many tokens", what);
  const int64_t blocks = (threads + kThreads - 1) / kThreads;
  // Heads of a thread: four, all in flight at once, are what still shares the
  // angles (4 x 4096 tokens of 40 heads: 53.4 us; with more in turns of four, and
  // the registers for the next turn, 60 for eight and 67 for fourteen); fewer where that leaves SMs without a block (64 tokens: 2.3 us
  // with one, 2.8 with four).
  a.chunk = kHeads;
  while (a.chunk > 1 && blocks * ((heads + a.chunk - 1) / a.chunk) < kf::sm_count_current_device() * 2) a.chunk /= 2;
  const dim3 grid((unsigned)blocks, (unsigned)((heads + a.chunk - 1) / a.chunk));
  const size_t smem = (size_t)a.R / 2 * sizeof(uint64_t);
  return bf16 ? kf::launch_dependent(rotary_kernel<VEC, HALVES, true>, grid, dim3(kThreads), smem, st, what, a)
              : kf::launch_dependent(rotary_kernel<VEC, HALVES, false>, grid, dim3(kThreads), smem, st, what, a);
}

}  // namespace

extern "C" int kf_rotary(const kf_rotary_args* args) {
  using kf::set_error;
  const char* what = "kf_rotary";
  if (!args) return set_error(KF_ERR_INVALID, "%s: null arguments", what);
  if (args->dtype != KF_F16 && args->dtype != KF_BF16)
    return set_error(KF_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  const kf_tensor4 &q = args->q, &k = args->k;
  const bool second = k.ptr || args->k_out.ptr;
  const int64_t B = q.size[0], S = q.size[2], D = q.size[3], R = args->rotated;
  if (B <= 0 || q.size[1] <= 0 || S <= 0 || D <= 0 || (second && k.size[1] <= 0))
    return set_error(KF_ERR_INVALID, "%s: dimensions must be non-zero", what);
  if (second && (k.size[0] != B || k.size[2] != S || k.size[3] != D))
    return set_error(KF_ERR_INVALID, "%s: Q and K must agree in batch, tokens and head_dim", what);
  for (int i = 0; i < 4; ++i)
    if (args->q_out.size[i] != q.size[i] || (second && args->k_out.size[i] != k.size[i]))
      return set_error(KF_ERR_INVALID, "%s: output shapes must be the inputs'", what);
  if (R <= 0 || R > D || R % 2)
    return set_error(KF_ERR_INVALID, "%s: the rotated columns must be even, at least 2 and at most head_dim", what);
  if (B > 0x7fffffffLL || S > 0x7fffffffLL || B * S > 0x7fffffffLL || D > 4096 || q.size[1] > (1 << 16) ||
      (second && k.size[1] > (1 << 16)))
    return set_error(KF_ERR_UNSUPPORTED, "%s: tensors too large", what);
  if (args->position_bits != 32 && args->position_bits != 64)
    return set_error(KF_ERR_INVALID, "%s: positions must have 32 or 64 bits", what);
  if (!q.ptr || !args->q_out.ptr || (second && (!k.ptr || !args->k_out.ptr)) || !args->positions || !args->frequencies)
    return set_error(KF_ERR_INVALID, "%s: null data pointer", what);
  if (!isfinite((float)args->magnitude)) return set_error(KF_ERR_INVALID, "%s: magnitude must be finite", what);
  const kf_tensor4* all[4] = {&q, &args->q_out, second ? &k : &q, second ? &args->k_out : &q};
  for (const kf_tensor4* t : all)
    if (t->stride[3] != 1 && D > 1) return set_error(KF_ERR_INVALID, "%s: tensors need a contiguous last dim", what);
  kf::DeviceGuard guard(q.ptr);
  if (guard.status()) return guard.status();

  RotaryArgs a;
  const kf_tensor4 *in[2] = {&q, second ? &k : &q}, *out[2] = {&args->q_out, second ? &args->k_out : &args->q_out};
  for (int w = 0; w < 2; ++w) {
    a.x[w] = static_cast<const uint16_t*>(in[w]->ptr);
    a.y[w] = static_cast<uint16_t*>(out[w]->ptr);
    a.heads[w] = w == 0 || second ? (int)in[w]->size[1] : 0;
    for (int i = 0; i < 3; ++i) {
      a.xs[w][i] = in[w]->stride[i];
      a.ys[w][i] = out[w]->stride[i];
    }
  }
  a.positions = args->positions;
  a.ps[0] = args->position_strides[0];
  a.ps[1] = args->position_strides[1];
  a.wide = args->position_bits == 64;
  a.frequencies = args->frequencies;
  a.tokens = (uint32_t)(B * S);
  a.S = (uint32_t)S;
  a.R = (int)R;
  a.magnitude = (float)args->magnitude;
  a.sign = args->inverse ? -1.f : 1.f;
  // The widest pieces that alignment and the column counts allow.
  int vec = 8;
  const int64_t unit = args->interleaved ? R : R / 2;
  while (vec > 1 && (unit % vec || D % vec || !fits(*all[0], vec) || !fits(*all[1], vec) || !fits(*all[2], vec) ||
                     !fits(*all[3], vec)))
    vec /= 2;
  cudaStream_t st = static_cast<cudaStream_t>(args->stream);
  const bool bf16 = args->dtype == KF_BF16;
  if (args->interleaved)
    return vec == 8   ? launch<8, false>(a, (int)D, bf16, st)
           : vec == 4 ? launch<4, false>(a, (int)D, bf16, st)
           : vec == 2 ? launch<2, false>(a, (int)D, bf16, st)
                      : launch<1, false>(a, (int)D, bf16, st);
  return vec == 8   ? launch<8, true>(a, (int)D, bf16, st)
         : vec == 4 ? launch<4, true>(a, (int)D, bf16, st)
         : vec == 2 ? launch<2, true>(a, (int)D, bf16, st)
                    : launch<1, true>(a, (int)D, bf16, st);
}
