// Rotary positions with several axes, alone or behind a norm over the channels of a head, on queries and keys in one launch:
//
//   y = (x - mean) / sqrt(var + eps) w + b   (layer),   x / sqrt(mean(x^2) + eps) w   (rms),   x   (none)
//   out_c = cos(a_c) y_c -/+ sin(a_c) y_partner(c),   a_c = 2 pi turns_c position[axis of c]
//
// and backward, g = dout turned by -a:   dw = sum g xh, db = sum g, dx = rstd (g w - mean(g w) - xh mean(g w xh)), the means of the layer norm alone.
//
// Bound by memory: a head's channels are read once and written once (x and dy in the backward pass), and mean and variance are computed again rather than kept.
// A group of lanes has the channels of a head and goes over the heads of a token; what comes next, of whichever token, is copied to shared memory meanwhile.  A lane
// has four pairs of channels, both of each, so that it turns them without its neighbours: two runs of four channels (halves of a band), or eight side by side
// (neighbours).  (Eight side by side in either case, and partners fetched from their lanes: 37080 tokens, 16 heads of 128 with norms, both ways, 188 us where this took
// 175 then; 16200 tokens, 16 heads of 48 62 / 54.)  Angles are computed once for a token's heads, in 64 bits down to the fraction of a turn (the angle of position 100000 in 32 bits would be off by 4e-3).  Statistics, sums and gradients of
// weights are fp32; blocks leave one row of partial sums each, added up in a fixed order by a second launch.
#include "rotary.cuh"

#include <algorithm>

#include "fused_ops.cuh"
#include "gelu.cuh"
#include "gemm_tcgen05.cuh"
#include "launch.cuh"
#include "vec8.cuh"

namespace mk {

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
// Steps of heads in the ring: two on their way beside the one that is computed.  us, two / three / four, rotation of 16200 tokens, 24 heads of 64, both ways, 52 / 42 /
// 41; 37080 tokens, 16 heads of 128 with norms, 154 / 150 / 153.  (The next heads in registers, and none of the next token's: 44, 166.)
constexpr int STAGES = 3;

struct KernelParams {
  RotShape s;
  int chunks[2];           // of a token's heads: divisors
  int blocks0;             // blocks of part 0
  int blocks;
  float* sums;             // [2: dw, db][blocks][D]
};

// Sums of N values over the LANES lanes of a group (powers of two), in all of them.  While there are several, a step of the butterfly gives half of them away:
// 15 exchanges for eight values over eight lanes where 24 were.
template <int LANES, int N>
__device__ __forceinline__ void group_sum(float (&a)[N]) {
  const int l = threadIdx.x & 31;
  int o = LANES / 2;
#pragma unroll
  for (int n = N; n > 1 && o > 0; n >>= 1, o >>= 1) {
    const bool upper = (l & o) != 0;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float mine = upper ? a[i + n / 2] : a[i], other = upper ? a[i] : a[i + n / 2];
      a[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
    }
  }
#pragma unroll
  for (; o > 0; o >>= 1) a[0] += __shfl_xor_sync(0xffffffffu, a[0], o);
  // the values i KEPT .. of them are now with the lanes i EACH .. of the group
  constexpr int EACH = N < LANES ? LANES / N : 1, KEPT = N > LANES ? N / LANES : 1;
  float part[KEPT];
#pragma unroll
  for (int i = 0; i < KEPT; ++i) part[i] = a[i];
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = __shfl_sync(0xffffffffu, part[i % KEPT], (l & ~(LANES - 1)) + i / KEPT * EACH);
}

__device__ __forceinline__ double position_of(const void* at, int type, long long i) {
  switch (type) {
    case ROT_POS_I32: return static_cast<double>(static_cast<const int*>(at)[i]);
    case ROT_POS_I64: return static_cast<double>(static_cast<const long long*>(at)[i]);
    case ROT_POS_F32: return static_cast<double>(static_cast<const float*>(at)[i]);
    default: return static_cast<const double*>(at)[i];
  }
}

// Sines and cosines of two angles in turns.  For bf16 from polynomials (the first terms of the series) of what is left, at most half of a quarter, after whole
// quarters are taken off in 64 bits: the first terms left out are 4e-7 of the sine and 2e-8 of the cosine.  Their error is one of the value, also next to a multiple
// of a quarter, where that of the special function unit, 2^-21 of one, is much of such a value (its sine of position 355 at one radian each, 3e-5, rounded to bf16: 0.7 %;
// of 2e-6 9 %, of 2e-7 all of it).
template <typename T>
__device__ __forceinline__ void sines_cosines(double v0, double v1, float (&sine)[2], float (&cosine)[2]) {
  const double t[2] = {v0 - rint(v0), v1 - rint(v1)};
  if constexpr (sizeof(T) == 2) {
    uint32_t q[2];
    float r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double nearest = 6755399441055744.0, n = fma(t[i], 4.0, nearest);      // 1.5 2^52: the sum's last bits are those of the nearest whole number
      q[i] = static_cast<uint32_t>(__double2loint(n));
      r[i] = static_cast<float>(fma(t[i], 4.0, nearest - n));
    }
    auto both = [](float v) { return f2_pack(v, v); };
    const f32x2 a = f2_mul(f2_pack(r[0], r[1]), both(1.5707963267948966f)), a2 = f2_mul(a, a);
    const f32x2 s = f2_fma(f2_mul(a, a2), f2_fma(f2_fma(both(-1.f / 5040.f), a2, both(1.f / 120.f)), a2, both(-1.f / 6.f)), a);
    const f32x2 c = f2_fma(f2_fma(f2_fma(f2_fma(both(1.f / 40320.f), a2, both(-1.f / 720.f)), a2, both(1.f / 24.f)), a2, both(-0.5f)), a2, both(1.f));
    float ss[2], cc[2];
    f2_unpack(s, ss[0], ss[1]);
    f2_unpack(c, cc[0], cc[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x = q[i] & 1 ? cc[i] : ss[i], y = q[i] & 1 ? ss[i] : cc[i];
      sine[i] = __uint_as_float(__float_as_uint(x) ^ (q[i] & 2) << 30);
      cosine[i] = __uint_as_float(__float_as_uint(y) ^ ((q[i] + 1) & 2) << 30);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) sincospif(2.f * static_cast<float>(t[i]), &sine[i], &cosine[i]);
  }
}

// Pair i of a head: its channels, its axis (-1: not turned; the channels behind the bands are paired up as they come)
struct Pair {
  int lo, hi, axis;
};
__device__ __forceinline__ Pair pair_of(const RotShape& s, int i, bool positions) {
  int start = 0;
  if (positions)
    for (int a = 0; a < s.axes; ++a) {
      const int half = s.band[a] >> 1, in = i - (start >> 1);
      if (in >= 0 && in < half) return s.interleaved ? Pair{start + 2 * in, start + 2 * in + 1, a} : Pair{start + in, start + half + in, a};
      start += 2 * half;
    }
  return {2 * i, 2 * i + 1, -1};
}

// How a lane's four pairs lie in memory: RUN 0: eight channels side by side, pairs are neighbours; 4: first and second channels in runs of four; 2: in runs of
// two, those of the first two pairs, then those of the others; 1: anyhow
template <int RUN>
struct Place {
  int at[RUN == 0 ? 1 : RUN == 4 ? 2 : RUN == 2 ? 4 : 8];
};
// The channels of four pairs as they come from memory; first and second ones as two values each
template <typename T, int RUN>
struct Channels {
  Vec8<T> raw;
  __device__ __forceinline__ void load(const T* p, const Place<RUN>& place) {
    if constexpr (RUN == 0) {
      raw.load(p);
    } else if constexpr (RUN == 4 && sizeof(T) == 2) {
      const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + place.at[1]);
      raw.v = make_uint4(a.x, a.y, b.x, b.y);
    } else if constexpr (RUN == 4) {
      raw.a = *reinterpret_cast<const float4*>(p);
      raw.b = *reinterpret_cast<const float4*>(p + place.at[1]);
    } else if constexpr (RUN == 2 && sizeof(T) == 2) {
      auto two = [&](int i) { return *reinterpret_cast<const uint32_t*>(p + place.at[i]); };
      raw.v = make_uint4(two(0), two(2), two(1), two(3));
    } else if constexpr (RUN == 2) {
      auto two = [&](int i) { return *reinterpret_cast<const float2*>(p + place.at[i]); };
      const float2 a = two(0), b = two(2), c = two(1), d = two(3);
      raw.a = make_float4(a.x, a.y, b.x, b.y);
      raw.b = make_float4(c.x, c.y, d.x, d.y);
    } else {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = value_of(p[place.at[i]]);
      raw.set(v);
    }
  }
  __device__ __forceinline__ void store(T* p, const Place<RUN>& place) const {
    if constexpr (RUN == 0) {
      raw.store(p);
    } else if constexpr (RUN == 4 && sizeof(T) == 2) {
      *reinterpret_cast<uint2*>(p) = make_uint2(raw.v.x, raw.v.y);
      *reinterpret_cast<uint2*>(p + place.at[1]) = make_uint2(raw.v.z, raw.v.w);
    } else if constexpr (RUN == 4) {
      *reinterpret_cast<float4*>(p) = raw.a;
      *reinterpret_cast<float4*>(p + place.at[1]) = raw.b;
    } else if constexpr (RUN == 2 && sizeof(T) == 2) {
      auto two = [&](int i) { return reinterpret_cast<uint32_t*>(p + place.at[i]); };
      *two(0) = raw.v.x, *two(2) = raw.v.y, *two(1) = raw.v.z, *two(3) = raw.v.w;
    } else if constexpr (RUN == 2) {
      auto two = [&](int i) { return reinterpret_cast<float2*>(p + place.at[i]); };
      *two(0) = make_float2(raw.a.x, raw.a.y), *two(2) = make_float2(raw.a.z, raw.a.w);
      *two(1) = make_float2(raw.b.x, raw.b.y), *two(3) = make_float2(raw.b.z, raw.b.w);
    } else {
      float v[8];
      raw.get(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) p[place.at[i]] = rounded<T>(v[i]);
    }
  }
  // (raw: RUN 0 pair by pair, else the first channels, then the second ones)
  __device__ __forceinline__ void get(f32x2 (&lo)[2], f32x2 (&hi)[2]) const {
    float v[8];
    raw.get(v);
    if constexpr (RUN == 0) {
      lo[0] = f2_pack(v[0], v[2]), lo[1] = f2_pack(v[4], v[6]), hi[0] = f2_pack(v[1], v[3]), hi[1] = f2_pack(v[5], v[7]);
    } else {
      lo[0] = f2_pack(v[0], v[1]), lo[1] = f2_pack(v[2], v[3]), hi[0] = f2_pack(v[4], v[5]), hi[1] = f2_pack(v[6], v[7]);
    }
  }
  __device__ __forceinline__ void set(const f32x2 (&lo)[2], const f32x2 (&hi)[2]) {
    float a[4], b[4];
    f2_unpack(lo[0], a[0], a[1]), f2_unpack(lo[1], a[2], a[3]), f2_unpack(hi[0], b[0], b[1]), f2_unpack(hi[1], b[2], b[3]);
    const float pairs[8] = {a[0], b[0], a[1], b[1], a[2], b[2], a[3], b[3]}, runs[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    raw.set(RUN == 0 ? pairs : runs);
  }
};
// Eight values to shared memory, zeros where not `in`, as a copy that goes on beside the thread
template <typename T>
__device__ __forceinline__ void copy8(T* to, const T* from, bool in) {
  const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
#pragma unroll
  for (uint32_t i = 0; i < sizeof(T) / 2; ++i)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + 16 * i), "l"(reinterpret_cast<const uint8_t*>(from) + 16 * i), "r"(in ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ f32x2 both(float v) { return f2_pack(v, v); }
__device__ __forceinline__ float sum_of(const f32x2 (&a)[2], const f32x2 (&b)[2]) {
  float x, y;
  f2_unpack(f2_add(f2_add(a[0], a[1]), f2_add(b[0], b[1])), x, y);
  return x + y;
}
// sum of a c + b d
__device__ __forceinline__ float sum_of_products(const f32x2 (&a)[2], const f32x2 (&b)[2], const f32x2 (&c)[2], const f32x2 (&d)[2]) {
  float x, y;
  f2_unpack(f2_fma(a[0], c[0], f2_fma(a[1], c[1], f2_fma(b[0], d[0], f2_mul(b[1], d[1])))), x, y);
  return x + y;
}
// Turns pairs by (cos, sin); `alone`: a bit for each that is not turned, and has nothing to do with its partner, whatever it holds
__device__ __forceinline__ void turn(f32x2 (&lo)[2], f32x2 (&hi)[2], const f32x2 (&cs)[2], const f32x2 (&sn)[2], const f32x2 (&neg)[2], bool plain, uint32_t alone) {
  f32x2 a[2] = {lo[0], lo[1]}, b[2] = {hi[0], hi[1]};
  if (plain) {      // (some of a head's channels are not turned)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x, y;
      f2_unpack(a[i], x, y);
      a[i] = f2_pack(alone >> 2 * i & 1 ? 0.f : x, alone >> (2 * i + 1) & 1 ? 0.f : y);
      f2_unpack(b[i], x, y);
      b[i] = f2_pack(alone >> 2 * i & 1 ? 0.f : x, alone >> (2 * i + 1) & 1 ? 0.f : y);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    lo[i] = f2_fma(cs[i], lo[i], f2_mul(neg[i], b[i]));
    hi[i] = f2_fma(cs[i], hi[i], f2_mul(sn[i], a[i]));
  }
}

// T: type of the tensors; LANES x 8 channels of a head at most; BACK: gradients; RUN: see `Place`; R: heads at a time
template <typename T, int LANES, int NORM, bool BACK, int RUN, int R, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) rotary_kernel(const __grid_constant__ KernelParams p) {
  constexpr int GROUPS = 32 / LANES, ROW = LANES * 8;
  constexpr bool NORMED = NORM != ROT_NORM_NONE, READ_X = NORMED || !BACK, SUMS = BACK && NORMED, LAYER = NORM == ROT_NORM_LAYER;
  const RotShape& s = p.s;
  constexpr int VALUES = READ_X && BACK ? 2 : 1;
  __shared__ __align__(16) double turns[ROW / 2];      // of every pair per unit of position
  extern __shared__ __align__(16) uint8_t ring_raw[];  // [STAGES][VALUES][R][WARPS][32 x 8]: steps that are on their way
  T* const ring = reinterpret_cast<T*>(ring_raw);
  const int which = blockIdx.x < static_cast<unsigned>(p.blocks0) ? 0 : 1;
  const RotPart& part = s.part[which];
  const T *x = static_cast<const T*>(part.x.ptr), *dy = static_cast<const T*>(part.dy.ptr);
  const float *w_at = part.w, *b_at = part.b;
  const void* positions = s.positions;
  chain_begin(true, x, dy, w_at, b_at, positions);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LANES, l = lane % LANES, D = s.D;
  const bool mine = l * 8 < D;                         // (lanes behind the last channel have zeros)
  Place<RUN> place;
  uint32_t alone = 0, axes = 0;                        // of the lane's pairs: whether they are not turned, their axes (a byte each)
  auto pair = [&](int i) { return pair_of(s, mine ? 4 * l + i : i, positions != nullptr); };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Pair q = pair(i);
    axes |= static_cast<uint32_t>(max(q.axis, 0)) << 8 * i;
    if (q.axis < 0) alone |= 1u << i;
    if constexpr (RUN == 1) place.at[i] = q.lo, place.at[4 + i] = q.hi;
    // (what is not turned: pairs side by side are two runs as well)
    if constexpr (RUN == 2)
      if (i % 2 == 0) place.at[i] = q.lo, place.at[i + 1] = q.axis < 0 ? q.lo + 2 : q.hi;
  }
  if constexpr (RUN == 4) {      // (what is not turned: four channels, and four more)
    place.at[0] = alone ? (mine ? 8 * l : 0) : pair(0).lo;
    place.at[1] = alone ? 4 : pair(0).hi - pair(0).lo;
  }
  if constexpr (RUN == 0) place.at[0] = mine ? 8 * l : 0;
  constexpr bool APART = RUN == 1 || RUN == 2;         // a lane's channels, here and there in a head
  const int offset = APART ? 0 : place.at[0];
  // channels of the pairs: first ones, then second ones
  auto channel = [&](int i) {
    if constexpr (RUN == 0) return place.at[0] + 2 * (i & 3) + (i >> 2);
    else if constexpr (RUN == 4) return place.at[0] + (i & 3) + (i < 4 ? 0 : place.at[1]);
    else if constexpr (RUN == 2) return place.at[(i & 2) + (i >> 2)] + (i & 1);
    else return place.at[i];
  };
  int rotated = 0;
  if (positions)
    for (int a = 0; a < s.axes; ++a) rotated += s.band[a];
  const bool plain = rotated < D;
  for (int i = threadIdx.x; i < ROW / 2; i += THREADS) turns[i] = 2 * i < rotated ? s.turns[i] : 0.0;
  __syncthreads();
  f32x2 w_lo[2], w_hi[2], b_lo[2], b_hi[2], dw_lo[2], dw_hi[2], db_lo[2], db_hi[2];
  if constexpr (NORMED) {
    float w[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = w_at ? w_at[channel(i)] : 1.f;
      b[i] = b_at ? b_at[channel(i)] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w_lo[i] = f2_pack(w[2 * i], w[2 * i + 1]), w_hi[i] = f2_pack(w[4 + 2 * i], w[5 + 2 * i]);
      b_lo[i] = f2_pack(b[2 * i], b[2 * i + 1]), b_hi[i] = f2_pack(b[4 + 2 * i], b[5 + 2 * i]);
      dw_lo[i] = dw_hi[i] = db_lo[i] = db_hi[i] = 0ull;
    }
  }
  const int limit = BACK && s.limit ? min(max(*s.limit, 0), s.N) : s.N;
  const float inv = 1.f / static_cast<float>(D);
  const int chunks = p.chunks[which], per_chunk = part.heads / chunks;
  const unsigned units = limit > 0 ? static_cast<unsigned>(s.B) * s.N * chunks : 0u;      // (below 2^31)
  const int block = which ? blockIdx.x - p.blocks0 : blockIdx.x, blocks = which ? p.blocks - p.blocks0 : p.blocks0;
  const unsigned step = static_cast<unsigned>(blocks) * WARPS * GROUPS;
  // A unit: its sample, token and first head; whether the group has something to do there
  struct Unit {
    int bat, n, h0;
    bool live;
  };
  auto unit_of = [&](unsigned first) {
    // (a group behind the last unit or the limit goes along with zeros)
    const unsigned u = min(first + group, units - 1), t = chunks == 1 ? u : u / chunks;
    Unit a;
    a.h0 = static_cast<int>(u - t * chunks) * per_chunk;
    a.bat = s.B == 1 ? 0 : static_cast<int>(t / s.N);
    a.n = static_cast<int>(t - static_cast<unsigned>(a.bat) * s.N);
    a.live = mine && first + group < units && (!BACK || a.n < limit);
    return a;
  };
  auto start_of = [&](const RotTensor& t, const Unit& u) { return u.bat * t.batch + u.n * t.token + u.h0 * t.head; };
  // Steps are fetched STAGES - 1 ahead, whatever unit they are of: all lanes of a warp fetch eight channels side by side and read their pairs behind the wait
  const unsigned begin = (static_cast<unsigned>(block) * WARPS + warp) * GROUPS;
  unsigned ahead = begin;
  int ahead_k = 0, ahead_stage = 0;
  bool ahead_live = false;
  const T *x_from = nullptr, *d_from = nullptr;
  auto slot = [&](int stage, int value, int q) { return ring + (((stage * VALUES + value) * R + q) * WARPS + warp) * (32 * 8); };
  auto enter = [&](const Unit& u) {
    ahead_live = u.live;
    if constexpr (READ_X) x_from = x + start_of(part.x, u) + (mine ? 8 * l : 0);
    if constexpr (BACK) d_from = dy + start_of(part.dy, u) + (mine ? 8 * l : 0);
  };
  auto fetch = [&] {
    if (ahead < units) {
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const bool in = ahead_live && (q == 0 || ahead_k + q < per_chunk);
        if constexpr (READ_X) {
          copy8(slot(ahead_stage, 0, q) + lane * 8, in ? x_from : x, in);
          x_from += part.x.head;
        }
        if constexpr (BACK) {
          copy8(slot(ahead_stage, VALUES - 1, q) + lane * 8, in ? d_from : dy, in);
          d_from += part.dy.head;
        }
      }
      ahead_k += R;
      if (ahead_k >= per_chunk) {
        ahead_k = 0;
        ahead += step;
        if (ahead < units) enter(unit_of(ahead));
      }
      ahead_stage = ahead_stage + 1 == STAGES ? 0 : ahead_stage + 1;
    }
    copies_commit();
  };
  Unit next{};
  if (begin < units) {
    next = unit_of(begin);
    enter(next);
  }
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch();
  int stage = 0;
  // (positions of the next unit are on their way, too)
  double at[RUN == 4 ? 1 : 4] = {};
  auto fetch_positions = [&](const Unit& u) {
    if (!positions) return;
    const long long from = u.bat * s.position_batch + 1ll * u.n * s.axes;
#pragma unroll
    for (int i = 0; i < (RUN == 4 ? 1 : 4); ++i)      // (zeros that go along stay zeros, in the sums too, whatever stands behind the limit)
      at[i] = !SUMS || u.live ? position_of(positions, s.position_type, from + (axes >> 8 * i & 255)) : 0.0;
  };
  if (begin < units) fetch_positions(next);
  // (the groups of a warp go through the loop together)
  for (unsigned first = begin; first < units; first += step) {
    const Unit unit = next;
    const bool live = unit.live;
    T* o_at = static_cast<T*>(part.out.ptr) + start_of(part.out, unit) + offset;

    // angles of the lane's pairs
    f32x2 cs[2], sn[2], neg[2];
    {
      float c[4] = {1.f, 1.f, 1.f, 1.f}, d[4] = {0.f, 0.f, 0.f, 0.f};
      if (positions) {
        const bool back = BACK != (s.inverse != 0);
        auto angle = [&](int i) { return at[RUN == 4 ? 0 : i] * turns[4 * l + i]; };
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          float sine[2], cosine[2];
          sines_cosines<T>(angle(i), angle(i + 1), sine, cosine);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            c[i + k] = cosine[k];
            d[i + k] = back ? -sine[k] : sine[k];
          }
        }
      }
      if (plain) {      // (whatever position there is)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          c[i] = alone >> i & 1 ? 1.f : c[i];
          d[i] = alone >> i & 1 ? 0.f : d[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        cs[i] = f2_pack(c[2 * i], c[2 * i + 1]);
        sn[i] = f2_pack(d[2 * i], d[2 * i + 1]);
        neg[i] = f2_pack(-d[2 * i], -d[2 * i + 1]);
      }
    }

    if (first + step < units) {
      next = unit_of(first + step);
      fetch_positions(next);
    }
    // (all groups of the warp make as many turns)
    for (int k = 0; k < per_chunk; k += R) {
      copies_wait<STAGES - 2>();
      __syncwarp();      // (what other lanes fetched is here, and they have read what the next step is fetched to)
      fetch();
      Channels<T, RUN> now[READ_X ? R : 1], now_d[BACK ? R : 1];
#pragma unroll
      for (int q = 0; q < R; ++q) {
        if constexpr (READ_X) now[q].load(slot(stage, 0, q) + group * ROW + offset, place);
        if constexpr (BACK) now_d[q].load(slot(stage, VALUES - 1, q) + group * ROW + offset, place);
        if (NORMED && !mine) {
          now[q].raw.clear();
          if constexpr (BACK) now_d[q].raw.clear();
        }
      }
      const int used = stage;
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      auto put = [&](int q, const f32x2 (&lo)[2], const f32x2 (&hi)[2]) {
        Channels<T, RUN> out;
        out.set(lo, hi);
        const bool in = live && (q == 0 || k + q < per_chunk);
        if constexpr (APART) {      // (eight channels side by side to a lane again, by way of the slot that all have read)
          T* const at = slot(used, 0, q);
          __syncwarp();
          if (mine) out.store(at + group * ROW, place);
          __syncwarp();
          if (in) {
            Vec8<T> v;
            v.load(at + lane * 8);
            v.store(o_at + 8 * l);
          }
        } else {
          if (in) out.store(o_at, place);
        }
        o_at += part.out.head;
      };
      if constexpr (!NORMED) {
#pragma unroll
        for (int q = 0; q < R; ++q) {
          f32x2 lo[2], hi[2];
          if constexpr (BACK) now_d[q].get(lo, hi);
          else now[q].get(lo, hi);
          turn(lo, hi, cs, sn, neg, plain, alone);
          put(q, lo, hi);
        }
      } else {
        // Sums of a head: of the deviations from a value near the mean (that of the first lane's channels: the variance loses little to their own mean) and of their
        // squares; backward, of g w and its products with them
        constexpr int EACH = (LAYER ? 2 : 1) * (BACK ? 2 : 1);
        f32x2 lo[R][2], hi[R][2], g_lo[BACK ? R : 1][2], g_hi[BACK ? R : 1][2];
        float sums[R * EACH];
#pragma unroll
        for (int q = 0; q < R; ++q) {
          now[q].get(lo[q], hi[q]);
          if constexpr (LAYER) {
            const float pivot = __shfl_sync(0xffffffffu, sum_of(lo[q], hi[q]) * 0.125f, lane & ~(LANES - 1));
            const f32x2 off = both(mine ? -pivot : 0.f);
#pragma unroll
            for (int i = 0; i < 2; ++i) lo[q][i] = f2_add(lo[q][i], off), hi[q][i] = f2_add(hi[q][i], off);
            sums[q * EACH + (BACK ? 2 : 1)] = sum_of(lo[q], hi[q]);
          }
          sums[q * EACH] = sum_of_products(lo[q], hi[q], lo[q], hi[q]);
          if constexpr (BACK) {
            now_d[q].get(g_lo[q], g_hi[q]);
            turn(g_lo[q], g_hi[q], cs, sn, neg, plain, alone);
            f32x2 e_lo[2], e_hi[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              db_lo[i] = f2_add(db_lo[i], g_lo[q][i]), db_hi[i] = f2_add(db_hi[i], g_hi[q][i]);
              e_lo[i] = f2_mul(g_lo[q][i], w_lo[i]), e_hi[i] = f2_mul(g_hi[q][i], w_hi[i]);
            }
            sums[q * EACH + 1] = sum_of_products(e_lo, e_hi, lo[q], hi[q]);
            if constexpr (LAYER) sums[q * EACH + 3] = sum_of(e_lo, e_hi);
          }
        }
        group_sum<LANES>(sums);
#pragma unroll
        for (int q = 0; q < R; ++q) {
          const float mean = LAYER ? sums[q * EACH + (BACK ? 2 : 1)] * inv : 0.f;      // of the deviations
          // (a variance that rounding has left below zero is none; NaN stays NaN, which a maximum would make a zero of)
          const float var = fmaf(sums[q * EACH], inv, -mean * mean);
          float rstd = rsqrtf((var < 0.f ? 0.f : var) + s.eps);
          // (what goes along with zeros has no deviation, and the reciprocal is infinite without eps)
          if (BACK && !(live && (q == 0 || k + q < per_chunk))) rstd = 0.f;
          const f32x2 r2 = both(rstd), m2 = both(-mean);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (LAYER) lo[q][i] = f2_add(lo[q][i], m2), hi[q][i] = f2_add(hi[q][i], m2);
            lo[q][i] = f2_mul(lo[q][i], r2), hi[q][i] = f2_mul(hi[q][i], r2);
          }
          if constexpr (!BACK) {
#pragma unroll
            for (int i = 0; i < 2; ++i) lo[q][i] = f2_fma(lo[q][i], w_lo[i], b_lo[i]), hi[q][i] = f2_fma(hi[q][i], w_hi[i], b_hi[i]);
            turn(lo[q], hi[q], cs, sn, neg, plain, alone);
          } else {
            const float over = LAYER ? sums[q * EACH + 3] * inv : 0.f;                  // mean of g w
            const float along = rstd * fmaf(sums[q * EACH + 1], inv, -mean * over);     // and of g w xh
            const f32x2 o2 = both(-over), a2 = both(-along);
            auto slope = [&](f32x2 xh, f32x2 g, f32x2 w) {
              f32x2 e = f2_mul(g, w);
              if (LAYER) e = f2_add(e, o2);
              return f2_mul(f2_fma(xh, a2, e), r2);
            };
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              dw_lo[i] = f2_fma(g_lo[q][i], lo[q][i], dw_lo[i]), dw_hi[i] = f2_fma(g_hi[q][i], hi[q][i], dw_hi[i]);
              lo[q][i] = slope(lo[q][i], g_lo[q][i], w_lo[i]), hi[q][i] = slope(hi[q][i], g_hi[q][i], w_hi[i]);
            }
          }
          put(q, lo[q], hi[q]);
        }
      }
    }
  }
  if constexpr (SUMS) {
    if (!p.sums) return;
    // the groups of a warp, then the warps one after the other
    __shared__ float cols[2][ROW];
    float fw[8], fb[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f2_unpack(dw_lo[i], fw[2 * i], fw[2 * i + 1]), f2_unpack(dw_hi[i], fw[4 + 2 * i], fw[5 + 2 * i]);
      f2_unpack(db_lo[i], fb[2 * i], fb[2 * i + 1]), f2_unpack(db_hi[i], fb[4 + 2 * i], fb[5 + 2 * i]);
    }
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        fw[i] += __shfl_xor_sync(0xffffffffu, fw[i], o);
        fb[i] += __shfl_xor_sync(0xffffffffu, fb[i], o);
      }
    for (int k = 0; k < WARPS; ++k) {
      if (warp == k && group == 0 && mine) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          cols[0][channel(i)] = (k ? cols[0][channel(i)] : 0.f) + fw[i];
          cols[1][channel(i)] = (k ? cols[1][channel(i)] : 0.f) + fb[i];
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * D; c += THREADS) {
      const int j = c >= D;
      p.sums[(1ll * j * p.blocks + blockIdx.x) * D + (c - j * D)] = cols[j][c - j * D];
    }
  }
}

// Adds up the blocks' rows: blockIdx.x 32 channels, blockIdx.y the sum (dw, db), blockIdx.z the part
__global__ void __launch_bounds__(1024) rotary_sums_kernel(const __grid_constant__ KernelParams p) {
  __shared__ float sh[32][33];
  const float* sums = p.sums;
  chain_begin(true, sums);
  const int which = blockIdx.z, j = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5, D = p.s.D;
  const int lo = which ? p.blocks0 : 0, hi = which ? p.blocks : p.blocks0;
  float a = 0.f;
  if (c < D)
    for (int i = lo + r; i < hi; i += 32) a += sums[(1ll * j * p.blocks + i) * D + c];
  sh[r][threadIdx.x & 31] = a;
  __syncthreads();
  if (r == 0) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) a += sh[i][threadIdx.x];
    float* const to = j ? p.s.part[which].db : p.s.part[which].dw;
    if (c < D && to) to[c] = a;
  }
}

// (four lanes for heads of 32 and less: rotation of 50000 tokens, one head of 8, 11.7 us, of eight lanes 18.1; norms of 129600, 4 heads of 16, 30 / 55)
int lanes_of(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// Blocks and shares of heads.  A unit is a token with all heads of a part, so that its angles are computed once; with fewer units than threads that the device
// holds, heads are shared out, four at least to a unit.
constexpr int LEAST_HEADS = 4;
// Blocks to an SM and heads at a time (bf16; half of them in fp32).  us by (heads, blocks): rotation of 16200 tokens, 24 heads of 64, (4, 3) 18.4, (2, 4) 18.3, (6, 2)
// 19.4, (6, 3) 20.1, (2, 5) 25.0, 15.2 of it memory; 9113 tokens, 20 heads of 96, both ways, (4, 3) 39.7, (2, 4) 42.2, (6, 2) 45.4; with norms, 37080 tokens, 16
// heads of 128, (4, 2) 59.6, (2, 3) 61.9, (2, 2) 62.7, (4, 3), which spills, 74.4 (memory 46.5); their gradients (2, 2) 90, (1, 3) 113 (memory 69.7).
constexpr int blocks_per_sm(int norm) { return norm == ROT_NORM_NONE ? 3 : 2; }
constexpr int heads_at_a_time(int norm, bool back, bool half) { return (norm != ROT_NORM_NONE && back ? 2 : 4) / (half ? 1 : 2); }
void plan(KernelParams& k) {
  const RotShape& s = k.s;
  const int per_block = WARPS * (32 / lanes_of(s.D));
  const long long most = 1ll * blocks_per_sm(s.norm) * sm_count(), tokens = 1ll * s.B * s.N;
  int heads = 0;
  for (int i = 0; i < s.parts; ++i) heads += s.part[i].heads;
  long long blocks[2] = {0, 0};
  for (int i = 0; i < 2; ++i) {
    k.chunks[i] = 1;
    if (i >= s.parts) continue;
    const int h = s.part[i].heads;
    const long long share = std::max<long long>(1, most * h / heads);        // blocks of this part in one wave
    const long long wanted = (share * per_block + tokens - 1) / tokens;
    k.chunks[i] = static_cast<int>(std::max<long long>(1, std::min<long long>(wanted, (h + LEAST_HEADS - 1) / LEAST_HEADS)));
    while (h % k.chunks[i]) ++k.chunks[i];
    blocks[i] = std::min<long long>(share, (tokens * k.chunks[i] + per_block - 1) / per_block);
  }
  k.blocks0 = static_cast<int>(blocks[0]);
  k.blocks = static_cast<int>(blocks[0] + blocks[1]);
}

bool shape_ok(const RotShape& s, bool back) {
  if (s.parts < 1 || s.parts > 2 || s.B < 1 || s.N < 1 || s.D < 8 || s.D > ROT_WIDTH || s.D % 8 || s.axes < 0 || s.axes > ROT_AXES) return false;
  int rotated = 0;
  for (int a = 0; a < s.axes; ++a) {
    if (s.band[a] < 2 || s.band[a] % 2) return false;
    rotated += s.band[a];
  }
  if (rotated > s.D || (s.positions && s.axes < 1)) return false;
  auto bad = [](const RotTensor& t) { return !t.ptr || (reinterpret_cast<uintptr_t>(t.ptr) & 15) || ((t.token | t.head | t.batch) & 7); };
  for (int i = 0; i < s.parts; ++i) {
    const RotPart& q = s.part[i];
    if (q.heads < 1 || 1ll * s.B * s.N * q.heads >= (1ll << 31) - (1ll << 24) || bad(q.out) || (back && bad(q.dy)) || ((!back || s.norm) && bad(q.x)) || (q.dw != nullptr) != (q.db != nullptr)) return false;
  }
  return true;
}

// See `Place`.  Pairs of halves whose bands have a multiple of four of them lie in runs of four, of two in runs of two.  (Rotation of
// 16200 tokens, 24 heads of 64, two bands of 20: one by one 41 us, runs of two 26.)
int run_of(const RotShape& s) {
  if (!s.positions || s.interleaved) return 0;
  int run = 4;
  for (int a = 0; a < s.axes; ++a) run = std::min(run, s.band[a] % 8 == 0 ? 4 : s.band[a] % 4 == 0 ? 2 : 1);
  return run;
}

template <typename T, int LANES, int NORM, bool BACK>
cudaError_t by_run(const KernelParams& k, cudaStream_t s) {
  constexpr int R = heads_at_a_time(NORM, BACK, sizeof(T) == 2), BLOCKS = blocks_per_sm(NORM);
  static std::atomic<uint64_t> devices[4];
  constexpr int BYTES = STAGES * (NORM != ROT_NORM_NONE && BACK ? 2 : 1) * R * THREADS * 8 * static_cast<int>(sizeof(T));
  auto go = [&](auto* kernel, std::atomic<uint64_t>& of) {
    const cudaError_t e = allow_shared_memory(of, reinterpret_cast<const void*>(kernel), BYTES);
    return e != cudaSuccess ? e : launch_chained(kernel, dim3(k.blocks), dim3(THREADS), BYTES, s, 1, true, k);
  };
  switch (run_of(k.s)) {
    case 0: return go(rotary_kernel<T, LANES, NORM, BACK, 0, R, BLOCKS>, devices[0]);
    case 4: return go(rotary_kernel<T, LANES, NORM, BACK, 4, R, BLOCKS>, devices[1]);
    case 2: return go(rotary_kernel<T, LANES, NORM, BACK, 2, R, BLOCKS>, devices[2]);
    default: return go(rotary_kernel<T, LANES, NORM, BACK, 1, R, BLOCKS>, devices[3]);
  }
}
template <typename T, int LANES, bool BACK>
cudaError_t by_norm(const KernelParams& k, cudaStream_t s) {
  switch (k.s.norm) {
    case ROT_NORM_NONE: return by_run<T, LANES, ROT_NORM_NONE, BACK>(k, s);
    case ROT_NORM_LAYER: return by_run<T, LANES, ROT_NORM_LAYER, BACK>(k, s);
    default: return by_run<T, LANES, ROT_NORM_RMS, BACK>(k, s);
  }
}
template <typename T, bool BACK>
cudaError_t by_width(const KernelParams& k, cudaStream_t s) {
  switch (lanes_of(k.s.D)) {
    case 4: return by_norm<T, 4, BACK>(k, s);
    case 8: return by_norm<T, 8, BACK>(k, s);
    case 16: return by_norm<T, 16, BACK>(k, s);
    default: return by_norm<T, 32, BACK>(k, s);
  }
}

}  // namespace

cudaError_t rotary_fwd(const RotShape& p, cudaStream_t s) {
  if (!shape_ok(p, false)) return cudaErrorInvalidValue;
  KernelParams k{};
  k.s = p;
  plan(k);
  return p.f32 ? by_width<float, false>(k, s) : by_width<__nv_bfloat16, false>(k, s);
}

long long rotary_scratch(const RotShape& p) {
  KernelParams k{};
  k.s = p;
  plan(k);
  return 2ll * k.blocks * p.D;
}

cudaError_t rotary_bwd(const RotShape& p, float* sums, int* launches, cudaStream_t s) {
  *launches = 0;
  if (!shape_ok(p, true)) return cudaErrorInvalidValue;
  KernelParams k{};
  k.s = p;
  plan(k);
  bool asked = false;
  for (int i = 0; i < p.parts; ++i) asked = asked || p.part[i].dw;
  if (asked && (!p.norm || !sums)) return cudaErrorInvalidValue;
  k.sums = asked ? sums : nullptr;
  *launches = 1;
  const cudaError_t e = p.f32 ? by_width<float, true>(k, s) : by_width<__nv_bfloat16, true>(k, s);
  if (e != cudaSuccess || !asked) return e;
  ++*launches;
  return launch_chained(rotary_sums_kernel, dim3((p.D + 31) / 32, 2, p.parts), dim3(1024), 0, s, 1, true, k);
}

}  // namespace mk
