// Rotary positions with several axes, alone or behind a norm over the channels of a head, on queries and keys in one launch:
//
//   y = (x - mean) / sqrt(var + eps) w + b   (layer),   x / sqrt(mean(x^2) + eps) w   (rms),   x   (none)
//   out_c = cos(a_c) y_c -/+ sin(a_c) y_partner(c),   a_c = 2 pi turns_c position[axis of c]
//
// and backward, g = dout turned by -a:   dw = sum g xh, db = sum g, dx = rstd (g w - mean(g w) - xh mean(g w xh)), the means of the layer norm alone.
//
// Bound by memory: a head's channels are read once and written once (x and dy in the backward pass), and mean and variance are computed again rather than kept.
// A group of lanes has the channels of a head, eight to a lane, and goes over the heads of a token: the angles of a token are computed once, in 64 bits down to
// the fraction of a turn (the angle of position 100000 in 32 bits would be off by 4e-3), sine and cosine of that fraction in 32 bits, and stay in registers with the
// weights.  The partner's channels come through shared memory as they are in memory.  Statistics, sums and gradients of weights are fp32; blocks leave one row of
// partial sums each, added up in a fixed order by a second launch.
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

struct KernelParams {
  RotShape s;
  int chunks[2];           // of a token's heads
  int blocks0;             // blocks of part 0
  int blocks;
  float* sums;             // [2: dw, db][blocks][D]
};

// Sums of N values (a power of two) over the LANES lanes of a group, in all of them.  While there are several, a step of the butterfly gives half of them away:
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
  static_assert(N <= LANES, "a value to a lane at least");
  // value i is now with the lanes whose upper bits (below LANES) are i's
  constexpr int EACH = LANES / N;
  const float part = a[0];
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = __shfl_sync(0xffffffffu, part, (l & ~(LANES - 1)) + i * EACH);
}

__device__ __forceinline__ double position_of(const void* at, int type, long long i) {
  switch (type) {
    case ROT_POS_I32: return static_cast<double>(static_cast<const int*>(at)[i]);
    case ROT_POS_I64: return static_cast<double>(static_cast<const long long*>(at)[i]);
    case ROT_POS_F32: return static_cast<double>(static_cast<const float*>(at)[i]);
    default: return static_cast<const double*>(at)[i];
  }
}

// Of a fraction of a turn, at most half of one.  For bf16 the special function unit's, which are off by 2^-20 (a step of bf16 is 2^-7 of the value; 16200 tokens, 24
// heads of 64, SINUS us with the library's).
template <typename T>
__device__ __forceinline__ void sine_cosine(float turn, float& sine, float& cosine) {
  if constexpr (sizeof(T) == 2) {
    const float angle = turn * 6.283185307179586f;
    sine = __sinf(angle);
    cosine = __cosf(angle);
  } else {
    sincospif(2.f * turn, &sine, &cosine);
  }
}

// The channel that c is turned with; c itself where it is not
__device__ __forceinline__ int partner_of(const RotShape& s, int c) {
  int start = 0;
  for (int a = 0; a < s.axes; ++a) {
    const int half = s.band[a] >> 1, in = c - start;
    if (in >= 0 && in < 2 * half) return s.interleaved ? c ^ 1 : in < half ? c + half : c - half;
    start += 2 * half;
  }
  return c;
}

// Eight values as four pairs
__device__ __forceinline__ void pairs_of(const Vec8<__nv_bfloat16>& raw, f32x2 (&f)[4]) {
  const uint32_t u[4] = {raw.v.x, raw.v.y, raw.v.z, raw.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f2_pack(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
}
__device__ __forceinline__ void pairs_of(const Vec8<float>& raw, f32x2 (&f)[4]) {
  f[0] = f2_pack(raw.a.x, raw.a.y), f[1] = f2_pack(raw.a.z, raw.a.w), f[2] = f2_pack(raw.b.x, raw.b.y), f[3] = f2_pack(raw.b.z, raw.b.w);
}
template <typename T>
__device__ __forceinline__ Vec8<T> rounded_pairs(const f32x2 (&f)[4]) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_unpack(f[i], v[2 * i], v[2 * i + 1]);
  Vec8<T> raw;
  raw.set(v);
  return raw;
}
__device__ __forceinline__ float sum_of(const f32x2 (&f)[4]) {
  float a, b;
  f2_unpack(f2_add(f2_add(f[0], f[1]), f2_add(f[2], f[3])), a, b);
  return a + b;
}
__device__ __forceinline__ float sum_of_products(const f32x2 (&f)[4], const f32x2 (&g)[4]) {
  float a, b;
  f2_unpack(f2_add(f2_fma(f[0], g[0], f2_mul(f[1], g[1])), f2_fma(f[2], g[2], f2_mul(f[3], g[3]))), a, b);
  return a + b;
}

// What a lane's channels are turned with.  RUN 4: partners stand side by side in runs of four channels at least; 1: wherever; 0: neighbours
template <typename T, int RUN>
__device__ __forceinline__ void partners(const T* row, const int (&at)[RUN == 4 ? 2 : 8], const f32x2 (&own)[4], f32x2 (&f)[4]) {
  if constexpr (RUN == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      f2_unpack(own[i], a, b);
      f[i] = f2_pack(b, a);
    }
  } else if constexpr (RUN == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = f2_pack(value_of(row[at[2 * i]]), value_of(row[at[2 * i + 1]]));
  } else {
    Vec8<T> raw;
    if constexpr (sizeof(T) == 2) {
      const uint2 a = *reinterpret_cast<const uint2*>(row + at[0]), b = *reinterpret_cast<const uint2*>(row + at[1]);
      raw.v = make_uint4(a.x, a.y, b.x, b.y);
    } else {
      raw.a = *reinterpret_cast<const float4*>(row + at[0]);
      raw.b = *reinterpret_cast<const float4*>(row + at[1]);
    }
    pairs_of(raw, f);
  }
}

// T: type of the tensors; LANES x 8 channels of a head at most; BACK: gradients; RUN: see `partners`; R: heads at a time
template <typename T, int LANES, int NORM, bool BACK, int RUN, int R, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) rotary_kernel(const __grid_constant__ KernelParams p) {
  constexpr int GROUPS = 32 / LANES, ROW = LANES * 8;
  constexpr bool XCHG = RUN > 0, NORMED = NORM != ROT_NORM_NONE, READ_X = NORMED || !BACK, SUMS = BACK && NORMED, LAYER = NORM == ROT_NORM_LAYER;
  const RotShape& s = p.s;
  __shared__ __align__(16) T rows[XCHG ? WARPS * R * GROUPS * ROW : 8];
  __shared__ __align__(16) float2 angles[WARPS * GROUPS * ROW];      // cos and signed sin of every channel
  __shared__ double turns[ROW / 2];                                  // of every pair, and (axis, its channels)
  __shared__ int places[ROW / 2];
  __shared__ float params[NORMED ? 2 : 1][NORMED ? ROW : 1];
  const int which = blockIdx.x < static_cast<unsigned>(p.blocks0) ? 0 : 1;
  const RotPart& part = s.part[which];
  const T *x = static_cast<const T*>(part.x.ptr), *dy = static_cast<const T*>(part.dy.ptr);
  const float *w_at = part.w, *b_at = part.b;
  const void* positions = s.positions;
  chain_begin(true, x, dy, w_at, b_at, positions);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LANES, l = lane % LANES, c0 = l * 8, D = s.D;
  const bool mine = c0 < D;                  // (lanes behind the last channel have zeros)
  T* const my_rows = rows + (XCHG ? (warp * GROUPS + group) * R * ROW : 0);
  float2* const my_angles = angles + (warp * GROUPS + group) * ROW;
  int at[RUN == 4 ? 2 : 8], pairs = 0;
#pragma unroll
  for (int i = 0; i < (RUN == 4 ? 2 : 8); ++i) at[i] = RUN == 0 ? 0 : partner_of(s, c0 + i * (RUN == 4 ? 4 : 1));
  if (positions) {
    int start = 0;
    for (int a = 0; a < s.axes; ++a) {
      const int half = s.band[a] >> 1;
      for (int i = threadIdx.x; i < half; i += THREADS) {
        const int lo = start + (RUN == 0 ? 2 * i : i), hi = lo + (RUN == 0 ? 1 : half);
        turns[pairs + i] = s.turns[pairs + i];
        places[pairs + i] = a << 16 | lo << 8 | hi;
      }
      pairs += half;
      start += 2 * half;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) my_angles[c0 + i] = make_float2(1.f, 0.f);
  if constexpr (NORMED) {
    for (int c = threadIdx.x; c < ROW; c += THREADS) {
      params[0][c] = c < D ? (w_at ? w_at[c] : 1.f) : 0.f;
      params[1][c] = c < D && b_at ? b_at[c] : 0.f;
    }
  }
  __syncthreads();
  // channels that are not turned have no partner (whatever it holds)
  const int alone = 2 * pairs - c0;
  auto turned = [&](f32x2 (&y)[4]) {
    if (alone >= 8) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = 2 * i < alone ? y[i] : 0ull;      // (bands are even)
  };
  f32x2 w[4], dw[4], db[4];
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = f2_pack(params[0][c0 + 2 * i], params[0][c0 + 2 * i + 1]);
      dw[i] = db[i] = 0ull;
    }
  }
  const int limit = BACK && s.limit ? *s.limit : s.N;
  const float inv = 1.f / static_cast<float>(D);
  const int chunks = p.chunks[which], per_chunk = (part.heads + chunks - 1) / chunks;
  const unsigned units = static_cast<unsigned>(s.B) * s.N * chunks;      // (below 2^31)
  const int block = which ? blockIdx.x - p.blocks0 : blockIdx.x, blocks = which ? p.blocks - p.blocks0 : p.blocks0;
  const unsigned step = static_cast<unsigned>(blocks) * WARPS * GROUPS;
  // (the groups of a warp go through the loop together)
  for (unsigned first = (static_cast<unsigned>(block) * WARPS + warp) * GROUPS; first < units; first += step) {
    const unsigned u = min(first + group, units - 1), t = chunks == 1 ? u : u / chunks;
    const int chunk = static_cast<int>(u - t * chunks), bat = s.B == 1 ? 0 : static_cast<int>(t / s.N), n = static_cast<int>(t - static_cast<unsigned>(bat) * s.N);
    const int h0 = chunk * per_chunk;
    const int count = mine && first + group < units && (!BACK || n < limit) ? min(part.heads - h0, per_chunk) : 0;      // heads that this lane has a part of
    const T* x_at = READ_X ? x + bat * part.x.batch + n * part.x.token + h0 * part.x.head + c0 : nullptr;
    const T* d_at = BACK ? dy + bat * part.dy.batch + n * part.dy.token + h0 * part.dy.head + c0 : nullptr;
    T* o_at = static_cast<T*>(part.out.ptr) + bat * part.out.batch + n * part.out.token + h0 * part.out.head + c0;

    Vec8<T> vx[READ_X ? R : 1], vd[BACK ? R : 1];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if constexpr (READ_X) vx[q].clear();
      if constexpr (BACK) vd[q].clear();
    }
    auto fetch = [&](int k) {
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const bool in = k + q < count;
        if constexpr (READ_X) {
          if (in) vx[q].load(x_at);
          x_at += part.x.head;
        }
        if constexpr (BACK) {
          if (in) vd[q].load(d_at);
          else vd[q].clear();      // (they would be added to the sums)
          d_at += part.dy.head;
        }
      }
    };
    fetch(0);

    // angles of the token
    if (positions) {
      __syncwarp();
      const long long from = bat * s.position_batch + 1ll * n * s.axes;
      int place[4];
      double turn[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {      // (at most half of a lane's eight channels)
        const int i = l + j * LANES;
        place[j] = i < pairs ? places[i] : 0;
        turn[j] = i < pairs ? position_of(positions, s.position_type, from + (place[j] >> 16)) * turns[i] : 0.0;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float sine, cosine;
        sine_cosine<T>(static_cast<float>(turn[j] - rint(turn[j])), sine, cosine);
        if (BACK != (s.inverse != 0)) sine = -sine;
        if (l + j * LANES < pairs) {
          my_angles[place[j] >> 8 & 255] = make_float2(cosine, -sine);
          my_angles[place[j] & 255] = make_float2(cosine, sine);
        }
      }
      __syncwarp();
    }
    f32x2 cs[4], sn[4], add[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 a = *reinterpret_cast<const float4*>(my_angles + c0 + 2 * i);
      cs[i] = f2_pack(a.x, a.z);
      sn[i] = f2_pack(a.y, a.w);
    }
    // forward: out = rstd ((x - mean) (cos w) + (x' - mean) (sin w')) + (cos b + sin b')
    if constexpr (NORMED && !BACK) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        auto mate = [&](int c) { return RUN == 0 ? (pairs > 0 ? c ^ 1 : c) : RUN == 4 ? at[(c - c0) / 4] + (c - c0) % 4 : at[c - c0]; };
        const int c = c0 + 2 * i, m0 = mate(c), m1 = mate(c + 1);
        add[i] = f2_fma(cs[i], f2_pack(params[1][c], params[1][c + 1]), f2_mul(sn[i], f2_pack(params[1][m0], params[1][m1])));
        cs[i] = f2_mul(cs[i], f2_pack(params[0][c], params[0][c + 1]));
        sn[i] = f2_mul(sn[i], f2_pack(params[0][m0], params[0][m1]));
      }
    }

    // (all groups of the warp make as many turns)
    for (int k = 0; k < per_chunk; k += R) {
      Vec8<T> now[READ_X ? R : 1], now_d[BACK ? R : 1];
#pragma unroll
      for (int q = 0; q < R; ++q) {
        if constexpr (READ_X) now[q] = vx[q];
        if constexpr (BACK) now_d[q] = vd[q];
      }
      if constexpr (XCHG) {
        __syncwarp();
#pragma unroll
        for (int q = 0; q < R; ++q) {
          if constexpr (BACK) now_d[q].store(my_rows + q * ROW + c0);
          else now[q].store(my_rows + q * ROW + c0);
        }
        __syncwarp();
      }
      if (k + R < per_chunk) fetch(k + R);
      auto put = [&](int q, const f32x2 (&v)[4]) {
        if (k + q < count) rounded_pairs<T>(v).store(o_at);
        o_at += part.out.head;
      };
      if constexpr (!NORMED) {
#pragma unroll
        for (int q = 0; q < R; ++q) {
          f32x2 v[4], y[4];
          if constexpr (BACK) pairs_of(now_d[q], v);
          else pairs_of(now[q], v);
          partners<T, RUN>(my_rows + q * ROW, at, v, y);
          turned(y);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = f2_fma(cs[i], v[i], f2_mul(sn[i], y[i]));
          put(q, v);
        }
      } else {
        // Sums of a head: of the deviations from a value near the mean (that of its first eight channels: the variance loses little to their own mean) and of their
        // squares; backward, of g w and its products with them
        constexpr int EACH = (LAYER ? 2 : 1) * (BACK ? 2 : 1);
        f32x2 v[R][4], g[BACK ? R : 1][4];
        float sums[R * EACH], pivot[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
          pairs_of(now[q], v[q]);
          if constexpr (LAYER) {
            pivot[q] = __shfl_sync(0xffffffffu, sum_of(v[q]) * 0.125f, lane & ~(LANES - 1));
            const f32x2 off = f2_pack(mine ? -pivot[q] : 0.f, mine ? -pivot[q] : 0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[q][i] = f2_add(v[q][i], off);
          } else {
            pivot[q] = 0.f;
          }
          if constexpr (BACK) {
            f32x2 y[4];
            pairs_of(now_d[q], g[q]);
            partners<T, RUN>(my_rows + q * ROW, at, g[q], y);
            turned(y);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              g[q][i] = f2_fma(cs[i], g[q][i], f2_mul(sn[i], y[i]));
              db[i] = f2_add(db[i], g[q][i]);
              y[i] = f2_mul(g[q][i], w[i]);
            }
            sums[q * EACH + 1] = sum_of_products(y, v[q]);
            if constexpr (LAYER) sums[q * EACH + 3] = sum_of(y);
          }
          sums[q * EACH] = sum_of_products(v[q], v[q]);
          if constexpr (LAYER) sums[q * EACH + (BACK ? 2 : 1)] = sum_of(v[q]);
        }
        group_sum<LANES>(sums);
#pragma unroll
        for (int q = 0; q < R; ++q) {
          const float mean = LAYER ? sums[q * EACH + (BACK ? 2 : 1)] * inv : 0.f;      // of the deviations
          const float rstd = rsqrtf(fmaxf(fmaf(sums[q * EACH], inv, -mean * mean), 0.f) + s.eps);
          const f32x2 r2 = f2_pack(rstd, rstd), m2 = f2_pack(-mean, -mean);
          if constexpr (!BACK) {
            f32x2 y[4], o[4];
            if constexpr (RUN == 0) {
              partners<T, RUN>(my_rows, at, v[q], y);
            } else {
              partners<T, RUN>(my_rows + q * ROW, at, v[q], y);
              if constexpr (LAYER) {
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = f2_add(y[i], f2_pack(-pivot[q], -pivot[q]));
              }
            }
            turned(y);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (LAYER) o[i] = f2_fma(r2, f2_fma(cs[i], f2_add(v[q][i], m2), f2_mul(sn[i], f2_add(y[i], m2))), add[i]);
              else o[i] = f2_fma(r2, f2_fma(cs[i], v[q][i], f2_mul(sn[i], y[i])), add[i]);
            }
            put(q, o);
          } else {
            const float over = LAYER ? sums[q * EACH + 3] * inv : 0.f;                  // mean of g w
            const float along = rstd * fmaf(sums[q * EACH + 1], inv, -mean * over);     // and of g w xh
            const f32x2 o2 = f2_pack(-over, -over), a2 = f2_pack(-along, -along);
            f32x2 o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const f32x2 xh = f2_mul(LAYER ? f2_add(v[q][i], m2) : v[q][i], r2);
              dw[i] = f2_fma(g[q][i], xh, dw[i]);
              f32x2 e = f2_mul(g[q][i], w[i]);
              if (LAYER) e = f2_add(e, o2);
              o[i] = f2_mul(f2_fma(xh, a2, e), r2);
            }
            put(q, o);
          }
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
    for (int i = 0; i < 4; ++i) {
      f2_unpack(dw[i], fw[2 * i], fw[2 * i + 1]);
      f2_unpack(db[i], fb[2 * i], fb[2 * i + 1]);
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
          cols[0][c0 + i] = (k ? cols[0][c0 + i] : 0.f) + fw[i];
          cols[1][c0 + i] = (k ? cols[1][c0 + i] : 0.f) + fb[i];
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

int lanes_of(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// Blocks and shares of heads.  A unit is a token with all of its heads, so that its angles are computed once; with fewer units than threads that the device holds,
// heads are shared out, four at least to a unit.
constexpr int LEAST_HEADS = 4;
constexpr int blocks_per_sm(int norm, bool back) { return norm == ROT_NORM_NONE ? 3 : back ? 2 : 3; }
void plan(KernelParams& k, bool back) {
  const RotShape& s = k.s;
  const int per_block = WARPS * (32 / lanes_of(s.D));
  const long long most = 1ll * blocks_per_sm(s.norm, back) * sm_count(), tokens = 1ll * s.B * s.N;
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

// Channels that have their partners side by side: see `partners`
int run_of(const RotShape& s) {
  if (!s.positions || s.interleaved) return 0;
  int all = 0, at = 0;
  for (int a = 0; a < s.axes; ++a) {
    all |= at | (s.band[a] >> 1);
    at += s.band[a];
  }
  return (all | at) % 4 == 0 ? 4 : 1;
}

template <typename T, int LANES, int NORM, bool BACK>
cudaError_t by_run(const KernelParams& k, cudaStream_t s) {
  constexpr int R = NORM == ROT_NORM_NONE ? (sizeof(T) == 2 ? 4 : 2) : (sizeof(T) == 2 ? 2 : 1), BLOCKS = blocks_per_sm(NORM, BACK);
  auto go = [&](auto* kernel) { return launch_chained(kernel, dim3(k.blocks), dim3(THREADS), 0, s, 1, true, k); };
  switch (run_of(k.s)) {
    case 0: return go(rotary_kernel<T, LANES, NORM, BACK, 0, R, BLOCKS>);
    case 4: return go(rotary_kernel<T, LANES, NORM, BACK, 4, R, BLOCKS>);
    default: return go(rotary_kernel<T, LANES, NORM, BACK, 1, R, BLOCKS>);
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
  plan(k, false);
  return p.f32 ? by_width<float, false>(k, s) : by_width<__nv_bfloat16, false>(k, s);
}

long long rotary_scratch(const RotShape& p) {
  KernelParams k{};
  k.s = p;
  plan(k, true);
  return 2ll * k.blocks * p.D;
}

cudaError_t rotary_bwd(const RotShape& p, float* sums, int* launches, cudaStream_t s) {
  *launches = 0;
  if (!shape_ok(p, true)) return cudaErrorInvalidValue;
  KernelParams k{};
  k.s = p;
  plan(k, true);
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
