// Layer norm over the last dimension of tokens:
//
//   mean = sum x / C,  var = sum (x - mean)^2 / C,  xh = (x - mean) / sqrt(var + eps),  y = xh w + b
//   g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// One read and one write of memory a row: a group of G threads holds its row in registers, so that the variance is a second sum over
// registers of deviations (E[x^2] - E[x]^2 loses everything where |mean| >> spread), and the next row is on its way while the sums go
// through the shuffles.  Groups are 8 or 16 threads for short rows, a warp up to 1024 channels, the block above.  The backward pass keeps
// its columns' sums of dy xh and dy in registers over all its rows; blocks leave one row of partial sums each, which a second launch
// adds up in a fixed order.  All sums are fp32; outputs are rounded once.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "fused_ops.cuh"
#include "gemm_tcgen05.cuh"
#include "launch.cuh"
#include "layer_norm.cuh"

namespace mk {

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

// VEC elements of T as they come from memory
template <typename T, int VEC>
struct Raw;
template <>
struct Raw<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    v = make_uint4(u[0], u[1], u[2], u[3]);
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = v; }
};
template <>
struct Raw<float, 8> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    a = make_float4(f[0], f[1], f[2], f[3]);
    b = make_float4(f[4], f[5], f[6], f[7]);
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
};
template <>
struct Raw<__nv_bfloat16, 1> {
  __nv_bfloat16 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = __ldg(p); }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = __bfloat162float(v); }
  __device__ __forceinline__ void set(const float (&f)[1]) { v = __float2bfloat16(f[0]); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *p = v; }
};
template <>
struct Raw<float, 1> {
  float v;
  __device__ __forceinline__ void load(const float* p) { v = __ldg(p); }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = v; }
  __device__ __forceinline__ void set(const float (&f)[1]) { v = f[0]; }
  __device__ __forceinline__ void store(float* p) const { *p = v; }
};

// Sums of N values over the G threads of a group, in all of them.  `sh` (G = THREADS): N * WARPS floats, another set for each of the sums that
// follow one another between two uses of the same.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&a)[N], float* sh) {
  constexpr int W = G < 32 ? G : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] += __shfl_xor_sync(0xffffffffu, a[i], o);
  if constexpr (G > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) sh[i * WARPS + warp] = a[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      a[i] = 0.f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) a[i] += sh[i * WARPS + k];
    }
  }
}

__device__ __forceinline__ long long row_offset(long long r, long long inner, long long so, long long si) {
  const unsigned long long q = (static_cast<unsigned long long>(r) >> 32) == 0 && (static_cast<unsigned long long>(inner) >> 32) == 0
                                   ? static_cast<uint32_t>(r) / static_cast<uint32_t>(inner)
                                   : static_cast<unsigned long long>(r) / static_cast<unsigned long long>(inner);
  const long long o = static_cast<long long>(q);
  return o * so + (r - o * inner) * si;
}

// TR: type of the tensor that is added first (void: none)
template <typename TI, typename TO, typename TR, int VEC, int G, int NV>
__global__ void __launch_bounds__(THREADS) ln_fwd_kernel(LnForward p) {
  constexpr bool ADD = !std::is_void<TR>::value;
  using Res = typename std::conditional<ADD, TR, TI>::type;
  constexpr int GROUPS = THREADS / G, PER_WARP = G < 32 ? 32 / G : 1;
  __shared__ float sh[3 * WARPS];
  const TI* x = static_cast<const TI*>(p.x);
  const Res* res = static_cast<const Res*>(p.r);
  const float *w = p.w, *b = p.b;
  chain_begin(true, x, res, w, b);
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const long long step = static_cast<long long>(gridDim.x) * GROUPS;
  // a warp's groups go through the loop together
  long long first = static_cast<long long>(blockIdx.x) * GROUPS + group / PER_WARP * PER_WARP;
  const int mine = group % PER_WARP;
  const float inv = 1.f / static_cast<float>(p.C);

  Raw<TI, VEC> next[NV];
  Raw<Res, VEC> next_r[ADD ? NV : 1];
  auto fetch = [&](long long r) {
    if (r >= p.rows) return;
    const TI* const from = x + row_offset(r, p.inner, p.outer_stride, p.inner_stride);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * G) * VEC;
      if (c < p.C) {
        next[i].load(from + c);
        if constexpr (ADD) next_r[i].load(res + r * p.C + c);
      }
    }
  };
  fetch(first + mine);
  for (; first < p.rows; first += step) {
    const long long r = first + mine;
    const bool here = r < p.rows;
    float v[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * G) * VEC;
      if (here && c < p.C) {
        next[i].get(v[i]);
        if constexpr (ADD) {
          float a[VEC];
          next_r[i].get(a);
#pragma unroll
          for (int j = 0; j < VEC; ++j) a[j] += v[i][j];
          Raw<TI, VEC> sum;
          sum.set(a);
          sum.store(static_cast<TI*>(p.s) + r * p.C + c);
          sum.get(v[i]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
      }
    }
    fetch(r + step);
    float total[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) total[0] += v[i][j];
    group_sum<G>(total, sh);
    const float near = total[0] * inv;
    // Deviations from the rounded mean; their own mean puts it right (a row of one value comes out as zeros)
    float a[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((lane + i * G) * VEC < p.C) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[i][j] -= near;
          a[0] += v[i][j];
          a[1] = fmaf(v[i][j], v[i][j], a[1]);
        }
      }
    }
    group_sum<G>(a, sh + WARPS);
    const float left = a[0] * inv, rstd = 1.f / sqrtf(fmaxf(fmaf(a[1], inv, -left * left), 0.f) + p.eps);
    if (!here) continue;
    if (lane == 0 && p.stats) p.stats[r] = make_float2(near + left, rstd);
    TO* const to = static_cast<TO*>(p.y) + r * p.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * G) * VEC;
      if (c < p.C) {
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = (v[i][j] - left) * rstd;
        if (w) {
          Raw<float, VEC> q;
          float a[VEC];
          q.load(w + c);
          q.get(a);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] *= a[j];
        }
        if (b) {
          Raw<float, VEC> q;
          float a[VEC];
          q.load(b + c);
          q.get(a);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] += a[j];
        }
        Raw<TO, VEC> out;
        out.set(f);
        out.store(to + c);
      }
    }
  }
}

template <typename TI, typename TO, int VEC, int G, int NV>
__global__ void __launch_bounds__(THREADS) ln_bwd_kernel(LnBackward p) {
  constexpr int GROUPS = THREADS / G, PER_WARP = G < 32 ? 32 / G : 1;
  extern __shared__ float cols[];            // [2][C]: the block's sums
  __shared__ float sh[2][2 * WARPS];
  const TI *x = static_cast<const TI*>(p.x), *ds = static_cast<const TI*>(p.ds);
  const TO* dy = static_cast<const TO*>(p.dy);
  const float* w = p.w;
  const float2* stats = p.stats;
  chain_begin(true, x, ds, dy, w, stats);
  const int lane = threadIdx.x % G, group = threadIdx.x / G;
  const long long step = static_cast<long long>(gridDim.x) * GROUPS;
  long long first = static_cast<long long>(blockIdx.x) * GROUPS + group / PER_WARP * PER_WARP;
  const int mine = group % PER_WARP;
  const float inv = 1.f / static_cast<float>(p.C);
  float aw[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) aw[i][j] = ab[i][j] = 0.f;

  Raw<TI, VEC> nx[NV];
  Raw<TO, VEC> ny[NV];
  float2 nst;
  auto fetch = [&](long long r) {
    if (r >= p.rows) return;
    nst = __ldg(stats + r);
    const TI* const from = x + row_offset(r, p.inner, p.outer_stride, p.inner_stride);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * G) * VEC;
      if (c < p.C) {
        nx[i].load(from + c);
        ny[i].load(dy + r * p.C + c);
      }
    }
  };
  fetch(first + mine);
  for (int turn = 0; first < p.rows; first += step, turn ^= 1) {
    const long long r = first + mine;
    const bool here = r < p.rows;
    float xh[NV][VEC], g[NV][VEC];
    const float mean = nst.x, rstd = nst.y;
    float a[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * G) * VEC;
      if (here && c < p.C) {
        nx[i].get(xh[i]);
        ny[i].get(g[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          xh[i][j] = (xh[i][j] - mean) * rstd;
          aw[i][j] = fmaf(g[i][j], xh[i][j], aw[i][j]);
          ab[i][j] += g[i][j];
        }
        if (w) {
          Raw<float, VEC> q;
          float f[VEC];
          q.load(w + c);
          q.get(f);
#pragma unroll
          for (int j = 0; j < VEC; ++j) g[i][j] *= f[j];
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          a[0] += g[i][j];
          a[1] = fmaf(g[i][j], xh[i][j], a[1]);
        }
      }
    }
    fetch(r + step);
    group_sum<G>(a, sh[turn]);
    if (!here) continue;
    const float m0 = a[0] * inv, m1 = a[1] * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * G) * VEC;
      if (c < p.C) {
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = rstd * (g[i][j] - m0 - xh[i][j] * m1);
        if (ds) {
          Raw<TI, VEC> q;
          float e[VEC];
          q.load(ds + r * p.C + c);
          q.get(e);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] += e[j];
        }
        Raw<TI, VEC> out;
        out.set(f);
        out.store(static_cast<TI*>(p.dx) + r * p.C + c);
        if (sizeof(TI) == 4 && p.dr) {
          Raw<__nv_bfloat16, VEC> half;
          half.set(f);
          half.store(static_cast<__nv_bfloat16*>(p.dr) + r * p.C + c);
        }
      }
    }
  }
  if (!p.dw) return;
  // the groups of a warp, then the warps one after the other
  if constexpr (G < 32) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          aw[i][j] += __shfl_xor_sync(0xffffffffu, aw[i][j], o);
          ab[i][j] += __shfl_xor_sync(0xffffffffu, ab[i][j], o);
        }
  }
  float* const out_w = gridDim.x == 1 ? p.dw : p.part + static_cast<long long>(blockIdx.x) * p.C;
  float* const out_b = gridDim.x == 1 ? p.db : p.part + (static_cast<long long>(gridDim.x) + blockIdx.x) * p.C;
  if constexpr (G <= 32) {
    for (int k = 0; k < WARPS; ++k) {
      if ((threadIdx.x >> 5) == k && mine == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (lane + i * G) * VEC;
          if (c < p.C) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              cols[c + j] = (k ? cols[c + j] : 0.f) + aw[i][j];
              cols[p.C + c + j] = (k ? cols[p.C + c + j] : 0.f) + ab[i][j];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < p.C; c += THREADS) {
      out_w[c] = cols[c];
      out_b[c] = cols[p.C + c];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (lane + i * G) * VEC;
      if (c < p.C) {
        Raw<float, VEC> q;
        q.set(aw[i]);
        q.store(out_w + c);
        q.set(ab[i]);
        q.store(out_b + c);
      }
    }
  }
}

// threads of a row, and blocks
int ln_group(int C, bool vec) {
  if (C > 1024) return THREADS;
  if (vec && C <= 64) return 8;
  if (vec && C <= 128) return 16;
  return 32;
}
unsigned ln_blocks(long long rows, int C, bool vec, int per_sm) {
  const long long groups = THREADS / ln_group(C, vec);
  return static_cast<unsigned>(std::max<long long>(1, std::min<long long>((rows + groups - 1) / groups, 1ll * per_sm * sm_count())));
}
constexpr int FWD_PER_SM = 4, BWD_PER_SM = 2;

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename TI, typename TO, int VEC, int G, int NV>
cudaError_t launch(const LnForward& p, cudaStream_t s) {
  const unsigned grid = ln_blocks(p.rows, p.C, VEC > 1, FWD_PER_SM);
  auto go = [&](auto* kernel) { return launch_chained(kernel, dim3(grid), dim3(THREADS), 0, s, 1, true, p); };
  if (!p.r) return go(ln_fwd_kernel<TI, TO, void, VEC, G, NV>);
  if constexpr (sizeof(TI) == 4)
    if (!p.r_f32) return go(ln_fwd_kernel<TI, TO, __nv_bfloat16, VEC, G, NV>);
  return go(ln_fwd_kernel<TI, TO, TI, VEC, G, NV>);
}
template <typename TI, typename TO, int VEC, int G, int NV>
cudaError_t launch(const LnBackward& p, cudaStream_t s) {
  const unsigned grid = ln_blocks(p.rows, p.C, VEC > 1, BWD_PER_SM);
  return launch_chained(ln_bwd_kernel<TI, TO, VEC, G, NV>, dim3(grid), dim3(THREADS), G <= 32 ? 8 * p.C : 0, s, 1, true, p);
}

template <typename TI, typename TO, typename P>
cudaError_t by_size(const P& p, bool vec, cudaStream_t s) {
  const int C = p.C;
  if (vec) {
    if (C <= 64) return launch<TI, TO, 8, 8, 1>(p, s);
    if (C <= 128) return launch<TI, TO, 8, 16, 1>(p, s);
    if (C <= 256) return launch<TI, TO, 8, 32, 1>(p, s);
    if (C <= 512) return launch<TI, TO, 8, 32, 2>(p, s);
    if (C <= 768) return launch<TI, TO, 8, 32, 3>(p, s);
    if (C <= 1024) return launch<TI, TO, 8, 32, 4>(p, s);
    if (C <= 2048) return launch<TI, TO, 8, THREADS, 1>(p, s);
    return launch<TI, TO, 8, THREADS, 4>(p, s);
  }
  if (C <= 256) return launch<TI, TO, 1, 32, 8>(p, s);
  if (C <= 512) return launch<TI, TO, 1, 32, 16>(p, s);
  if (C <= 1024) return launch<TI, TO, 1, 32, 32>(p, s);
  return launch<TI, TO, 1, THREADS, 32>(p, s);
}
template <typename P>
cudaError_t by_type(const P& p, bool vec, cudaStream_t s) {
  if (p.x_f32) return p.y_f32 ? by_size<float, float>(p, vec, s) : by_size<float, __nv_bfloat16>(p, vec, s);
  return p.y_f32 ? by_size<__nv_bfloat16, float>(p, vec, s) : by_size<__nv_bfloat16, __nv_bfloat16>(p, vec, s);
}

}  // namespace

cudaError_t layer_norm_fwd(const LnForward& p, cudaStream_t s) {
  if (p.rows <= 0) return cudaSuccess;
  if (p.C <= 0 || p.C > LN_CHANNELS || p.inner <= 0 || (p.r != nullptr) != (p.s != nullptr) || (p.r && p.r_f32 && !p.x_f32))
    return cudaErrorInvalidValue;
  // whole 16-byte vectors in every tensor
  const bool vec = p.C % 8 == 0 && p.outer_stride % 8 == 0 && p.inner_stride % 8 == 0 && aligned(p.x) && aligned(p.r) && aligned(p.s) && aligned(p.y) &&
                   aligned(p.w) && aligned(p.b);
  return by_type(p, vec, s);
}

long long layer_norm_scratch(long long rows, int C) {
  // (as many blocks as either form of the kernel may take)
  const long long n = std::max(ln_blocks(rows, C, true, BWD_PER_SM), ln_blocks(rows, C, false, BWD_PER_SM));
  return n > 1 ? 2 * n * C : 0;
}

cudaError_t layer_norm_bwd(const LnBackward& p, int* launches, cudaStream_t s) {
  *launches = 0;
  if (p.C <= 0 || p.C > LN_CHANNELS || p.inner <= 0 || (p.dw != nullptr) != (p.db != nullptr)) return cudaErrorInvalidValue;
  if (p.rows <= 0) return cudaSuccess;
  const bool vec = p.C % 8 == 0 && p.outer_stride % 8 == 0 && p.inner_stride % 8 == 0 && aligned(p.x) && aligned(p.dy) && aligned(p.ds) &&
                   aligned(p.dx) && aligned(p.dr) && aligned(p.w) && aligned(p.dw) && aligned(p.db) && aligned(p.part);
  const unsigned blocks = ln_blocks(p.rows, p.C, vec, BWD_PER_SM);
  if (p.dw && blocks > 1 && !p.part) return cudaErrorInvalidValue;
  ++*launches;
  const cudaError_t e = by_type(p, vec, s);
  if (e != cudaSuccess || !p.dw || blocks == 1) return e;
  ++*launches;
  const int n = static_cast<int>(blocks);
  return colsum_add_slabs(RowSlabs{p.part, p.dw, n, p.C, 1}, RowSlabs{p.part + static_cast<long long>(n) * p.C, p.db, n, p.C, 1}, s);
}

}  // namespace mk
