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

// Sum over the LANES lanes of a group, in all of them
template <int LANES, int N>
__device__ __forceinline__ void group_sum(float (&a)[N]) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] += __shfl_xor_sync(0xffffffffu, a[i], o);
}

__device__ __forceinline__ double position_of(const void* at, int type, long long i) {
  switch (type) {
    case ROT_POS_I32: return static_cast<double>(static_cast<const int*>(at)[i]);
    case ROT_POS_I64: return static_cast<double>(static_cast<const long long*>(at)[i]);
    case ROT_POS_F32: return static_cast<double>(static_cast<const float*>(at)[i]);
    default: return static_cast<const double*>(at)[i];
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

// A lane's channels have their partners in runs of four channels, wherever, or (RUN 1) one by one; RUN 0: neighbours
template <typename T, int RUN>
__device__ __forceinline__ void partners(const T* row, const int (&at)[RUN == 4 ? 2 : 8], const float (&own)[8], float (&f)[8]) {
  if constexpr (RUN == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = own[i ^ 1];
  } else if constexpr (RUN == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = value_of(row[at[i]]);
  } else if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint2 u = *reinterpret_cast<const uint2*>(row + at[i]);
      f[4 * i] = __uint_as_float(u.x << 16);
      f[4 * i + 1] = __uint_as_float(u.x & 0xffff0000u);
      f[4 * i + 2] = __uint_as_float(u.y << 16);
      f[4 * i + 3] = __uint_as_float(u.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(row + at[i]);
      f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
    }
  }
}

// Mean (layer norm) and 1 / sqrt(var + eps) of R heads, whose channels a group has
template <int LANES, int NORM, int R>
__device__ __forceinline__ void statistics(const float (&v)[R][8], bool mine, float inv, float eps, float (&mean)[R], float (&rstd)[R]) {
  if constexpr (NORM == ROT_NORM_LAYER) {
    float a[R], dev[2 * R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      a[q] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[q] += v[q][i];
    }
    group_sum<LANES>(a);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = a[q] * inv;
      dev[2 * q] = dev[2 * q + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = mine ? v[q][i] - mean[q] : 0.f;
        dev[2 * q] += d;
        dev[2 * q + 1] = fmaf(d, d, dev[2 * q + 1]);
      }
    }
    group_sum<LANES>(dev);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      // (deviations from the rounded mean; their own mean puts it right)
      const float left = dev[2 * q] * inv;
      mean[q] += left;
      rstd[q] = 1.f / sqrtf(fmaxf(fmaf(dev[2 * q + 1], inv, -left * left), 0.f) + eps);
    }
  } else {
    float a[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      a[q] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[q] = fmaf(v[q][i], v[q][i], a[q]);
    }
    group_sum<LANES>(a);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      mean[q] = 0.f;
      rstd[q] = 1.f / sqrtf(fmaf(a[q], inv, eps));
    }
  }
}

// T: type of the tensors; LANES x 8 channels of a head at most; BACK: gradients; RUN: see `partners`; R: heads at a time
template <typename T, int LANES, int NORM, bool BACK, int RUN, int R, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) rotary_kernel(const __grid_constant__ KernelParams p) {
  constexpr int GROUPS = 32 / LANES, ROW = LANES * 8;
  constexpr bool XCHG = RUN > 0, NORMED = NORM != ROT_NORM_NONE, READ_X = NORMED || !BACK, SUMS = BACK && NORMED;
  const RotShape& s = p.s;
  __shared__ __align__(16) T rows[XCHG ? WARPS * R * GROUPS * ROW : 8];
  __shared__ __align__(16) float2 angles[WARPS * GROUPS * ROW];      // cos and signed sin of every channel
  __shared__ float params[NORMED ? 2 : 1][NORMED ? ROT_WIDTH : 1];
  const int which = blockIdx.x < static_cast<unsigned>(p.blocks0) ? 0 : 1;
  const RotPart& part = s.part[which];
  const T *x = static_cast<const T*>(part.x.ptr), *dy = static_cast<const T*>(part.dy.ptr);
  const float *w_at = part.w, *b_at = part.b;
  const void* positions = s.positions;
  chain_begin(true, x, dy, w_at, b_at, positions);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LANES, l = lane % LANES, c0 = l * 8, D = s.D;
  const bool mine = c0 < D;                  // (lanes behind the last channel)
  T* const my_rows = rows + (XCHG ? (warp * GROUPS + group) * R * ROW : 0);
  float2* const my_angles = angles + (warp * GROUPS + group) * ROW;
  int at[RUN == 4 ? 2 : 8], pairs = 0;
#pragma unroll
  for (int i = 0; i < (RUN == 4 ? 2 : 8); ++i) at[i] = RUN == 0 ? 0 : partner_of(s, c0 + i * (RUN == 4 ? 4 : 1));
  if (positions)
    for (int a = 0; a < s.axes; ++a) pairs += s.band[a] >> 1;
#pragma unroll
  for (int i = 0; i < 8; ++i) my_angles[c0 + i] = make_float2(1.f, 0.f);
  // channels that are not turned have no partner (whatever it holds)
  const int alone = 2 * pairs - c0;
  auto turned = [&](float (&y)[8]) {
    if (alone >= 8) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = i < alone ? y[i] : 0.f;
  };
  if constexpr (NORMED) {
    for (int c = threadIdx.x; c < D; c += THREADS) {
      params[0][c] = w_at ? w_at[c] : 1.f;
      params[1][c] = b_at ? b_at[c] : 0.f;
    }
    __syncthreads();
  }
  float w[8], dw[8], db[8];
  if constexpr (SUMS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = mine ? params[0][c0 + i] : 0.f;
      dw[i] = db[i] = 0.f;
    }
  }
  const int limit = BACK && s.limit ? *s.limit : s.N;
  const float inv = 1.f / static_cast<float>(D);
  const int chunks = p.chunks[which], per_chunk = (part.heads + chunks - 1) / chunks;
  const long long units = 1ll * s.B * s.N * chunks;
  const int block = which ? blockIdx.x - p.blocks0 : blockIdx.x, blocks = which ? p.blocks - p.blocks0 : p.blocks0;
  const long long step = 1ll * blocks * WARPS * GROUPS;
  // (the groups of a warp go through the loop together)
  for (long long first = (1ll * block * WARPS + warp) * GROUPS; first < units; first += step) {
    const long long u = first + group, t = u < units ? u / chunks : 0;
    const int chunk = u < units ? static_cast<int>(u - t * chunks) : 0, bat = static_cast<int>(t / s.N), n = static_cast<int>(t - 1ll * bat * s.N);
    const bool here = u < units && (!BACK || n < limit);
    const int h0 = chunk * per_chunk, h1 = here ? min(part.heads, h0 + per_chunk) : h0;
    const T* const x_at = READ_X ? x + bat * part.x.batch + n * part.x.token + c0 : nullptr;
    const T* const d_at = BACK ? dy + bat * part.dy.batch + n * part.dy.token + c0 : nullptr;
    T* const o_at = static_cast<T*>(part.out.ptr) + bat * part.out.batch + n * part.out.token + c0;

    Vec8<T> vx[READ_X ? R : 1], vd[BACK ? R : 1];
    auto fetch = [&](int h) {
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const bool in = mine && h + q < h1;
        if constexpr (READ_X) {
          if (in) vx[q].load(x_at + (h + q) * part.x.head);
          else vx[q].clear();
        }
        if constexpr (BACK) {
          if (in) vd[q].load(d_at + (h + q) * part.dy.head);
          else vd[q].clear();
        }
      }
    };
    fetch(h0);

    // angles of the token
    if (positions) {
      __syncwarp();
      for (int i = l; i < pairs; i += LANES) {
        int a = 0, start = 0, half = s.band[0] >> 1, in = i;
        while (in >= half) {
          in -= half;
          start += 2 * half;
          half = s.band[++a] >> 1;
        }
        const double turns = position_of(positions, s.position_type, bat * s.position_batch + 1ll * n * s.axes + a) * s.turns[i];
        float sine, cosine;
        sincospif(2.f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
        if (BACK != (s.inverse != 0)) sine = -sine;
        const int lo = start + (RUN == 0 ? 2 * in : in), hi = lo + (RUN == 0 ? 1 : half);
        my_angles[lo] = make_float2(cosine, -sine);
        my_angles[hi] = make_float2(cosine, sine);
      }
      __syncwarp();
    }
    float cs[8], sn[8], add[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 a = my_angles[c0 + i];
      cs[i] = a.x;
      sn[i] = a.y;
    }
    // forward: out = rstd ((x - mean) (cos w) + (x' - mean) (sin w')) + (cos b + sin b')
    if constexpr (NORMED && !BACK) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = RUN == 0 ? (pairs > 0 ? (c0 + i) ^ 1 : c0 + i) : RUN == 4 ? at[i / 4] + i % 4 : at[i];
        add[i] = mine ? fmaf(cs[i], params[1][c0 + i], sn[i] * params[1][c]) : 0.f;
        cs[i] *= mine ? params[0][c0 + i] : 0.f;
        sn[i] *= mine ? params[0][c] : 0.f;
      }
    }

    // (all groups of the warp make as many turns)
    for (int k = 0; k < per_chunk; k += R) {
      const int h = h0 + k;
      Vec8<T> now[R], now_d[BACK ? R : 1];
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
      if (k + R < per_chunk) fetch(h + R);
      if constexpr (!NORMED) {
#pragma unroll
        for (int q = 0; q < R; ++q) {
          float v[8], y[8];
          if constexpr (BACK) now_d[q].get(v);
          else now[q].get(v);
          partners<T, RUN>(my_rows + q * ROW, at, v, y);
          turned(y);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = fmaf(cs[i], v[i], sn[i] * y[i]);
          Vec8<T> out;
          out.set(v);
          if (mine && h + q < h1) out.store(o_at + (h + q) * part.out.head);
        }
      } else {
        float v[R][8], mean[R], rstd[R];
#pragma unroll
        for (int q = 0; q < R; ++q) now[q].get(v[q]);
        statistics<LANES, NORM, R>(v, mine, inv, s.eps, mean, rstd);
        if constexpr (!BACK) {
#pragma unroll
          for (int q = 0; q < R; ++q) {
            float y[8], o[8];
            partners<T, RUN>(my_rows + q * ROW, at, v[q], y);
            turned(y);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              o[i] = NORM == ROT_NORM_RMS ? fmaf(rstd[q], fmaf(cs[i], v[q][i], sn[i] * y[i]), add[i])
                                          : fmaf(rstd[q], fmaf(cs[i], v[q][i] - mean[q], sn[i] * (y[i] - mean[q])), add[i]);
            Vec8<T> out;
            out.set(o);
            if (mine && h + q < h1) out.store(o_at + (h + q) * part.out.head);
          }
        } else {
          float g[R][8], a[2 * R];
#pragma unroll
          for (int q = 0; q < R; ++q) {
            float y[8];
            now_d[q].get(g[q]);
            partners<T, RUN>(my_rows + q * ROW, at, g[q], y);
            turned(y);
            a[2 * q] = a[2 * q + 1] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float gi = fmaf(cs[i], g[q][i], sn[i] * y[i]);
              v[q][i] = (v[q][i] - mean[q]) * rstd[q];
              dw[i] = fmaf(gi, v[q][i], dw[i]);
              db[i] += gi;
              y[i] = gi * w[i];
              a[2 * q] += y[i];
              a[2 * q + 1] = fmaf(y[i], v[q][i], a[2 * q + 1]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) g[q][i] = y[i];
          }
          group_sum<LANES>(a);
#pragma unroll
          for (int q = 0; q < R; ++q) {
            const float m0 = NORM == ROT_NORM_LAYER ? a[2 * q] * inv : 0.f, m1 = a[2 * q + 1] * inv;
#pragma unroll
            for (int i = 0; i < 8; ++i) g[q][i] = rstd[q] * (g[q][i] - m0 - v[q][i] * m1);
            Vec8<T> out;
            out.set(g[q]);
            if (mine && h + q < h1) out.store(o_at + (h + q) * part.out.head);
          }
        }
      }
    }
  }
  if constexpr (SUMS) {
    if (!p.sums) return;
    // the groups of a warp, then the warps one after the other
    __shared__ float cols[2][ROT_WIDTH];
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
        db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
      }
    for (int k = 0; k < WARPS; ++k) {
      if (warp == k && group == 0 && mine) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          cols[0][c0 + i] = (k ? cols[0][c0 + i] : 0.f) + dw[i];
          cols[1][c0 + i] = (k ? cols[1][c0 + i] : 0.f) + db[i];
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
    if (q.heads < 1 || bad(q.out) || (back && bad(q.dy)) || ((!back || s.norm) && bad(q.x)) || (q.dw != nullptr) != (q.db != nullptr)) return false;
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
