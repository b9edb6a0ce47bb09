// Layer norm over the last dimension of tokens:
//
//   mean = sum x / C,  var = sum (x - mean)^2 / C,  xh = (x - mean) / sqrt(var + eps),  y = xh w + b
//   g = dy w,  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
//
// One read and one write of memory a row.  A thread has eight neighbouring channels (16 bytes of bf16; four single ones where rows are not whole
// vectors) for all rows that its group goes over, so that weights and the sums of dy xh and dy stay in registers; groups are 8 or 16 threads for
// short rows, else as many warps as a row needs.  A group takes ROWS rows at a time, whose sums share shuffles and barriers, with the next ones on
// their way.  The variance is a second sum over registers of deviations (E[x^2] - E[x]^2 loses everything where |mean| >> spread).  In the backward
// pass blocks leave one row of partial sums each, which a second launch adds up in a fixed order.  All sums are fp32; outputs are rounded once.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "fused_ops.cuh"
#include "gelu.cuh"
#include "gemm_tcgen05.cuh"
#include "launch.cuh"
#include "layer_norm.cuh"

namespace mk {

namespace {

constexpr int THREADS = 256, MOST_WARPS = THREADS / 32;

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

// The threads of one row: SUB of a warp (8, 16), or whole warps (SUB = 32), `warps` of them
template <int SUB>
struct Group {
  int size, lane, index, per_block, warps;
  __device__ __forceinline__ explicit Group(int w) : warps(SUB < 32 ? 1 : w) {
    size = SUB < 32 ? SUB : 32 * warps;
    lane = threadIdx.x % size;
    index = threadIdx.x / size;
    per_block = blockDim.x / size;
  }
  // Sums of N values (a power of two) over the group, in all of its threads.  While there are several, a step of the butterfly gives half of them away
  // instead of adding up all: 9 exchanges for eight values in a warp where 40 were.  `sh`: N * MOST_WARPS floats, 16-byte aligned, another set for each of
  // the sums that follow one another between two uses of the same.
  template <int N>
  __device__ __forceinline__ void sum(float (&a)[N], float* sh) const {
    const int l = threadIdx.x & 31;
    int o = SUB / 2;
#pragma unroll
    for (int n = N; n > 1; n >>= 1, o >>= 1) {
      const bool upper = (l & o) != 0;
#pragma unroll
      for (int i = 0; i < n / 2; ++i) {
        const float mine = upper ? a[i + n / 2] : a[i], other = upper ? a[i] : a[i + n / 2];
        a[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
      }
    }
#pragma unroll
    for (; o > 0; o >>= 1) a[0] += __shfl_xor_sync(0xffffffffu, a[0], o);
    // value i is now with the lanes whose upper bits (below SUB) are i's
    constexpr int EACH = SUB / N;
    const float part = a[0];
    if (SUB < 32 || warps == 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) a[i] = __shfl_sync(0xffffffffu, part, (l & ~(SUB - 1)) + i * EACH);
      return;
    }
    float* const all = sh + index * warps * N;
    if (l % EACH == 0) all[(lane >> 5) * N + l / EACH] = part;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + index), "r"(size) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = 0.f;
    for (int k = 0; k < warps; ++k) {
      if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(all + k * N + i);
          a[i] += v.x, a[i + 1] += v.y, a[i + 2] += v.z, a[i + 3] += v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] += all[k * N + i];
      }
    }
  }
};

__device__ __forceinline__ long long row_offset(long long r, long long rows, long long inner, long long so, long long si) {
  if (inner >= rows) return r * si;
  const unsigned long long q = (static_cast<unsigned long long>(r) >> 32) == 0 && (static_cast<unsigned long long>(inner) >> 32) == 0
                                   ? static_cast<uint32_t>(r) / static_cast<uint32_t>(inner)
                                   : static_cast<unsigned long long>(r) / static_cast<unsigned long long>(inner);
  const long long o = static_cast<long long>(q);
  return o * so + (r - o * inner) * si;
}

__device__ __forceinline__ float sum_of(f32x2 v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

// A thread's NV vectors of VEC channels, of which the i-th begins at channel (lane + i size) VEC, as PAIRS pairs of values
template <int VEC, int NV>
struct Cols {
  static constexpr int PAIRS = VEC * NV / 2;
  static_assert(VEC == 8 || NV % 2 == 0, "whole pairs");
};
template <typename T, int VEC, int NV>
__device__ __forceinline__ void unpack(const Raw<T, VEC> (&raw)[NV], f32x2 (&v)[Cols<VEC, NV>::PAIRS]) {
  float f[VEC * NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float e[VEC];
    raw[i].get(e);
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[i * VEC + j] = e[j];
  }
#pragma unroll
  for (int k = 0; k < Cols<VEC, NV>::PAIRS; ++k) v[k] = f2_pack(f[2 * k], f[2 * k + 1]);
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void pack(const f32x2 (&v)[Cols<VEC, NV>::PAIRS], Raw<T, VEC> (&raw)[NV]) {
  float f[VEC * NV];
#pragma unroll
  for (int k = 0; k < Cols<VEC, NV>::PAIRS; ++k) f2_unpack(v[k], f[2 * k], f[2 * k + 1]);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float e[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = f[i * VEC + j];
    raw[i].set(e);
  }
}
// zeros where a vector is behind the last channel
template <int VEC, int NV>
__device__ __forceinline__ void keep(f32x2 (&v)[Cols<VEC, NV>::PAIRS], int lane, int size, int C) {
  if (VEC == 8) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((lane + i * size) * VEC >= C)
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) v[i * (VEC / 2) + k] = 0ull;
  } else {
#pragma unroll
    for (int k = 0; k < Cols<VEC, NV>::PAIRS; ++k) {
      float a, b;
      f2_unpack(v[k], a, b);
      v[k] = f2_pack(lane + 2 * k * size < C ? a : 0.f, lane + (2 * k + 1) * size < C ? b : 0.f);
    }
  }
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void load_row(const T* from, Raw<T, VEC> (&raw)[NV], int lane, int size, int C) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + i * size) * VEC;
    if (c < C) raw[i].load(from + c);
  }
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void store_row(T* to, const Raw<T, VEC> (&raw)[NV], int lane, int size, int C) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (lane + i * size) * VEC;
    if (c < C) raw[i].store(to + c);
  }
}

// Weights or biases, in fp32 or bf16; of long rows in fp32 (with both types in the kernel the registers do not hold 32 values a thread: 3000 x 4099 in fp32,
// forward, 45 us where this takes 41)
template <int VEC, int NV>
__device__ __forceinline__ void load_params(const void* from, bool f32, f32x2 (&v)[Cols<VEC, NV>::PAIRS], int lane, int size, int C) {
  if (VEC * NV > 8 || f32) {
    Raw<float, VEC> raw[NV];
    load_row(static_cast<const float*>(from), raw, lane, size, C);
    unpack(raw, v);
  } else {
    Raw<__nv_bfloat16, VEC> raw[NV];
    load_row(static_cast<const __nv_bfloat16*>(from), raw, lane, size, C);
    unpack(raw, v);
  }
}
__device__ __forceinline__ void store_param(void* to, bool f32, int c, float v) {
  if (f32) static_cast<float*>(to)[c] = v;
  else static_cast<__nv_bfloat16*>(to)[c] = __float2bfloat16(v);
}

// TR: type of the tensor that is added first (void: none)
template <typename TI, typename TO, typename TR, int VEC, int NV, int SUB, int ROWS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) ln_fwd_kernel(LnForward p, int warps) {
  constexpr bool ADD = !std::is_void<TR>::value;
  using Res = typename std::conditional<ADD, TR, TI>::type;
  constexpr int P = Cols<VEC, NV>::PAIRS;
  __shared__ __align__(16) float sh[3 * ROWS * MOST_WARPS];
  const TI* x = static_cast<const TI*>(p.x);
  const Res* res = static_cast<const Res*>(p.r);
  const void *w = p.w, *b = p.b;
  chain_begin(true, x, res, w, b);
  const Group<SUB> g(warps);
  const int C = p.C;
  const float inv = 1.f / static_cast<float>(C);
  f32x2 wv[P], bv[P];
#pragma unroll
  for (int k = 0; k < P; ++k) {
    wv[k] = f2_pack(1.f, 1.f);
    bv[k] = 0ull;
  }
  if (w) load_params<VEC, NV>(w, p.w_f32, wv, g.lane, g.size, C);
  if (b) load_params<VEC, NV>(b, p.b_f32, bv, g.lane, g.size, C);
  const long long step = static_cast<long long>(gridDim.x) * g.per_block * ROWS;
  // (the groups of a warp go through the loop together)
  const int per_warp = SUB < 32 ? 32 / SUB : 1;
  const int mine = SUB < 32 ? g.index % per_warp : 0;
  long long first = (static_cast<long long>(blockIdx.x) * g.per_block + (g.index - mine)) * ROWS;

  Raw<TI, VEC> next[ROWS][NV];
  Raw<Res, VEC> next_r[ADD ? ROWS : 1][NV];
  auto fetch = [&](long long r0) {
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const long long r = r0 + q;
      if (r >= p.rows) return;
      load_row(x + row_offset(r, p.rows, p.inner, p.outer_stride, p.inner_stride), next[q], g.lane, g.size, C);
      if constexpr (ADD) load_row(res + r * C, next_r[q], g.lane, g.size, C);
    }
  };
  fetch(first + mine * ROWS);
  for (; first < p.rows; first += step) {
    const long long r0 = first + mine * ROWS;
    f32x2 v[ROWS][P];
    float total[ROWS];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      unpack(next[q], v[q]);
      if constexpr (ADD) {
        f32x2 a[P];
        unpack(next_r[q], a);
#pragma unroll
        for (int k = 0; k < P; ++k) a[k] = f2_add(a[k], v[q][k]);
        Raw<TI, VEC> sum[NV];
        pack(a, sum);
        if (r0 + q < p.rows) store_row(static_cast<TI*>(p.s) + (r0 + q) * C, sum, g.lane, g.size, C);
        unpack(sum, v[q]);
      }
      keep<VEC, NV>(v[q], g.lane, g.size, C);
      f32x2 t = v[q][0];
#pragma unroll
      for (int k = 1; k < P; ++k) t = f2_add(t, v[q][k]);
      total[q] = sum_of(t);
    }
    fetch(r0 + step);
    g.sum(total, sh);
    // Deviations from the rounded mean; their own mean puts it right (a row of one value comes out as zeros)
    float dev[2 * ROWS];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const float near = total[q] * inv;
      const f32x2 n2 = f2_pack(-near, -near);
      f32x2 s = 0ull, s2 = 0ull;
#pragma unroll
      for (int k = 0; k < P; ++k) v[q][k] = f2_add(v[q][k], n2);
      keep<VEC, NV>(v[q], g.lane, g.size, C);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        s = f2_add(s, v[q][k]);
        s2 = f2_fma(v[q][k], v[q][k], s2);
      }
      dev[2 * q] = sum_of(s);
      dev[2 * q + 1] = sum_of(s2);
    }
    g.sum(dev, sh + ROWS * MOST_WARPS);
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const long long r = r0 + q;
      if (r >= p.rows) break;
      const float left = dev[2 * q] * inv, rstd = 1.f / sqrtf(fmaxf(fmaf(dev[2 * q + 1], inv, -left * left), 0.f) + p.eps);
      if (g.lane == 0 && p.stats) p.stats[r] = make_float2(fmaf(total[q], inv, left), rstd);
      const f32x2 l2 = f2_pack(-left, -left), r2 = f2_pack(rstd, rstd);
#pragma unroll
      for (int k = 0; k < P; ++k) v[q][k] = f2_fma(f2_mul(f2_add(v[q][k], l2), r2), wv[k], bv[k]);
      Raw<TO, VEC> out[NV];
      pack(v[q], out);
      store_row(static_cast<TO*>(p.y) + r * C, out, g.lane, g.size, C);
    }
  }
}

// ADD: there is a gradient of the sum in front
template <typename TI, typename TO, bool ADD, int VEC, int NV, int SUB, int ROWS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) ln_bwd_kernel(LnBackward p, int warps) {
  constexpr int P = Cols<VEC, NV>::PAIRS;
  extern __shared__ float cols[];            // [2][C]: the block's sums
  __shared__ __align__(16) float sh[2][2 * ROWS * MOST_WARPS];
  const TI *x = static_cast<const TI*>(p.x), *ds = static_cast<const TI*>(p.ds);
  const TO* dy = static_cast<const TO*>(p.dy);
  const void* w = p.w;
  const float2* stats = p.stats;
  chain_begin(true, x, ds, dy, w, stats);
  const Group<SUB> g(warps);
  const int C = p.C;
  const float inv = 1.f / static_cast<float>(C);
  f32x2 wv[P], aw[P], ab[P];
#pragma unroll
  for (int k = 0; k < P; ++k) {
    wv[k] = f2_pack(1.f, 1.f);
    aw[k] = ab[k] = 0ull;
  }
  if (w) {
    load_params<VEC, NV>(w, p.w_f32, wv, g.lane, g.size, C);
    keep<VEC, NV>(wv, g.lane, g.size, C);
  }
  const long long step = static_cast<long long>(gridDim.x) * g.per_block * ROWS;
  const int per_warp = SUB < 32 ? 32 / SUB : 1;
  const int mine = SUB < 32 ? g.index % per_warp : 0;
  long long first = (static_cast<long long>(blockIdx.x) * g.per_block + (g.index - mine)) * ROWS;

  Raw<TI, VEC> nx[ROWS][NV], nd[ADD ? ROWS : 1][NV];
  Raw<TO, VEC> ny[ROWS][NV];
  float2 nst[ROWS];
  auto fetch = [&](long long r0) {
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const long long r = r0 + q;
      if (r >= p.rows) return;
      nst[q] = __ldg(stats + r);
      load_row(x + row_offset(r, p.rows, p.inner, p.outer_stride, p.inner_stride), nx[q], g.lane, g.size, C);
      load_row(dy + r * C, ny[q], g.lane, g.size, C);
      if constexpr (ADD) load_row(ds + r * C, nd[q], g.lane, g.size, C);
    }
  };
  fetch(first + mine * ROWS);
  for (int turn = 0; first < p.rows; first += step, turn ^= 1) {
    const long long r0 = first + mine * ROWS;
    f32x2 xh[ROWS][P], gr[ROWS][P];
    Raw<TI, VEC> d[ADD ? ROWS : 1][NV];
    float rstd[ROWS], a[2 * ROWS];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const bool here = r0 + q < p.rows;
      unpack(nx[q], xh[q]);
      unpack(ny[q], gr[q]);
      rstd[q] = nst[q].y;
      if constexpr (ADD) {
#pragma unroll
        for (int i = 0; i < NV; ++i) d[q][i] = nd[q][i];
      }
      const f32x2 m2 = f2_pack(-nst[q].x, -nst[q].x), r2 = f2_pack(nst[q].y, nst[q].y);
#pragma unroll
      for (int k = 0; k < P; ++k) xh[q][k] = f2_mul(f2_add(xh[q][k], m2), r2);
      keep<VEC, NV>(xh[q], g.lane, g.size, here ? C : 0);
      keep<VEC, NV>(gr[q], g.lane, g.size, here ? C : 0);
      f32x2 s0 = 0ull, s1 = 0ull;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        aw[k] = f2_fma(gr[q][k], xh[q][k], aw[k]);
        ab[k] = f2_add(ab[k], gr[q][k]);
        gr[q][k] = f2_mul(gr[q][k], wv[k]);
        s0 = f2_add(s0, gr[q][k]);
        s1 = f2_fma(gr[q][k], xh[q][k], s1);
      }
      a[2 * q] = sum_of(s0);
      a[2 * q + 1] = sum_of(s1);
    }
    fetch(r0 + step);
    g.sum(a, sh[turn]);
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const long long r = r0 + q;
      if (r >= p.rows) break;
      const float m0 = -a[2 * q] * inv, m1 = -a[2 * q + 1] * inv;
      const f32x2 m02 = f2_pack(m0, m0), m12 = f2_pack(m1, m1), r2 = f2_pack(rstd[q], rstd[q]);
#pragma unroll
      for (int k = 0; k < P; ++k) gr[q][k] = f2_mul(f2_fma(xh[q][k], m12, f2_add(gr[q][k], m02)), r2);
      if constexpr (ADD) {
        f32x2 e[P];
        unpack(d[q], e);
#pragma unroll
        for (int k = 0; k < P; ++k) gr[q][k] = f2_add(gr[q][k], e[k]);
      }
      Raw<TI, VEC> out[NV];
      pack(gr[q], out);
      store_row(static_cast<TI*>(p.dx) + r * C, out, g.lane, g.size, C);
      if (sizeof(TI) == 4 && p.dr) {
        Raw<__nv_bfloat16, VEC> half[NV];
        pack(gr[q], half);
        store_row(static_cast<__nv_bfloat16*>(p.dr) + r * C, half, g.lane, g.size, C);
      }
    }
  }
  if (!p.dw) return;
  // the groups of a warp, then those of the block one after the other
  float fw[2 * P], fb[2 * P];
#pragma unroll
  for (int k = 0; k < P; ++k) {
    f2_unpack(aw[k], fw[2 * k], fw[2 * k + 1]);
    f2_unpack(ab[k], fb[2 * k], fb[2 * k + 1]);
  }
  if (SUB < 32) {
#pragma unroll
    for (int o = SUB; o < 32; o <<= 1)
#pragma unroll
      for (int k = 0; k < 2 * P; ++k) {
        fw[k] += __shfl_xor_sync(0xffffffffu, fw[k], o);
        fb[k] += __shfl_xor_sync(0xffffffffu, fb[k], o);
      }
  }
  const int sets = SUB < 32 ? blockDim.x / 32 : g.per_block, set = SUB < 32 ? threadIdx.x / 32 : g.index;
  for (int t = 0; t < sets; ++t) {
    if (set == t && mine == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (g.lane + i * g.size) * VEC;
        if (c < C) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            cols[c + j] = (t ? cols[c + j] : 0.f) + fw[i * VEC + j];
            cols[C + c + j] = (t ? cols[C + c + j] : 0.f) + fb[i * VEC + j];
          }
        }
      }
    }
    __syncthreads();
  }
  if (gridDim.x == 1) {
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
      store_param(p.dw, p.dw_f32, c, cols[c]);
      store_param(p.db, p.db_f32, c, cols[C + c]);
    }
    return;
  }
  float* const out_w = p.part + static_cast<long long>(blockIdx.x) * C;
  float* const out_b = p.part + (static_cast<long long>(gridDim.x) + blockIdx.x) * C;
  for (int c = threadIdx.x; c < C; c += blockDim.x) {
    out_w[c] = cols[c];
    out_b[c] = cols[C + c];
  }
}

// How a row is spread: warps of a group (0: a part of a warp), threads of a block, rows that it takes at a time; blocks to an SM, rows of a group.  What
// carries it is that several rows share shuffles and barriers.  us by (blocks, rows): forward, 74160 x 1024 bf16, (3, 2) 71, (2, 4) 63 (DRAM 46; every value through
// all steps of the butterfly 70); 129600 x 48 7.7, 8.1; 16471 x 387 fp32 18.4, 16.1.  Forward and backward of the first (3, 1) 174, (2, 2) 157, (1, 4) 165 (DRAM
// 116).  (A warp to a row, its weights read again for every row: 71 and 212; 16471 x 387 74.  Rows through a ring of cp.async, (2, 4) 77 and (4, 2) 86: more bytes on
// their way are not what is missing.  Forward, a scheduler issues in 64 % of the cycles, and its warps wait for fixed latencies, shuffles and one another, hardly for
// memory.)  Behind a sum one row at a time: 16200 x 768 (4, 1) 21.0, (3, 2) 23.3 (DRAM 15).
// Registers: what stays in them is more than there is in some forms.  Backward behind a sum in fp32, two rows at a time at 128 registers, 120 to 200 bytes a thread are
// spilled (16200 x 768, both passes 93 us, DRAM 61); rows of more than 1024 channels that are no whole vectors, behind a sum, 770 to 850.
constexpr int FWD_BLOCKS = 2, BWD_BLOCKS = 2;
constexpr int WIDE = 2048, RAGGED = LN_HALF_PARAMS;      // most channels of eight warps with one vector, or four single values, a thread
struct Spread {
  int warps, threads, rows;
};
Spread spread(int C, bool vec, int rows_at_a_time) {
  if (vec && C <= 128) return {0, THREADS, THREADS / (C <= 64 ? 8 : 16) * rows_at_a_time};
  const int per_warp = vec ? (C <= WIDE ? 256 : 1024) : (C <= RAGGED ? 128 : 1024);
  const int warps = (C + per_warp - 1) / per_warp, groups = MOST_WARPS / warps;
  return {warps, 32 * warps * groups, groups * (C <= (vec ? WIDE : RAGGED) ? rows_at_a_time : 1)};
}
unsigned blocks_of(long long rows, const Spread& s, int per_sm) {
  return static_cast<unsigned>(std::max<long long>(1, std::min<long long>((rows + s.rows - 1) / s.rows, 1ll * per_sm * sm_count())));
}
constexpr int FWD_ROWS = 4, BWD_ROWS = 2;
constexpr int FWD_ADD_BLOCKS = 4;      // one row at a time where two tensors are read

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename TI, typename TO, int VEC, int NV, int SUB>
cudaError_t launch(const LnForward& p, cudaStream_t s) {
  constexpr bool BIG = VEC * NV > 8;
  auto go = [&](auto* kernel, int rows, int blocks) {
    const Spread q = spread(p.C, VEC > 1, rows);
    return launch_chained(kernel, dim3(blocks_of(p.rows, q, blocks)), dim3(q.threads), 0, s, 1, true, p, q.warps);
  };
  constexpr int ROWS = BIG ? 1 : FWD_ROWS, BLOCKS = BIG ? 1 : FWD_BLOCKS, ADD_BLOCKS = BIG ? 1 : FWD_ADD_BLOCKS;
  if (!p.r) return go(ln_fwd_kernel<TI, TO, void, VEC, NV, SUB, ROWS, BLOCKS>, FWD_ROWS, FWD_BLOCKS);
  if constexpr (sizeof(TI) == 4)
    if (!p.r_f32) return go(ln_fwd_kernel<TI, TO, __nv_bfloat16, VEC, NV, SUB, 1, ADD_BLOCKS>, 1, FWD_ADD_BLOCKS);
  return go(ln_fwd_kernel<TI, TO, TI, VEC, NV, SUB, 1, ADD_BLOCKS>, 1, FWD_ADD_BLOCKS);
}
template <typename TI, typename TO, int VEC, int NV, int SUB>
cudaError_t launch(const LnBackward& p, cudaStream_t s) {
  constexpr bool BIG = VEC * NV > 8;
  constexpr int ROWS = BIG ? 1 : BWD_ROWS, BLOCKS = BIG ? 1 : BWD_BLOCKS;
  const Spread q = spread(p.C, VEC > 1, BWD_ROWS);
  auto go = [&](auto* kernel, std::atomic<uint64_t>& devices) {
    const cudaError_t e = BIG ? allow_shared_memory(devices, reinterpret_cast<const void*>(kernel), 8 * LN_CHANNELS) : cudaSuccess;
    if (e != cudaSuccess) return e;
    return launch_chained(kernel, dim3(blocks_of(p.rows, q, BWD_BLOCKS)), dim3(q.threads), 8 * p.C, s, 1, true, p, q.warps);
  };
  static std::atomic<uint64_t> with, without;
  return p.ds ? go(ln_bwd_kernel<TI, TO, true, VEC, NV, SUB, ROWS, BLOCKS>, with) : go(ln_bwd_kernel<TI, TO, false, VEC, NV, SUB, ROWS, BLOCKS>, without);
}

template <typename TI, typename TO, typename P>
cudaError_t by_size(const P& p, bool vec, cudaStream_t s) {
  const int C = p.C;
  if (vec) {
    if (C <= 64) return launch<TI, TO, 8, 1, 8>(p, s);
    if (C <= 128) return launch<TI, TO, 8, 1, 16>(p, s);
    if (C <= WIDE) return launch<TI, TO, 8, 1, 32>(p, s);
    return launch<TI, TO, 8, 4, 32>(p, s);
  }
  if (C <= RAGGED) return launch<TI, TO, 1, 4, 32>(p, s);
  return launch<TI, TO, 1, 32, 32>(p, s);
}
template <typename P>
cudaError_t by_type(const P& p, bool vec, cudaStream_t s) {
  if (p.x_f32) return p.y_f32 ? by_size<float, float>(p, vec, s) : by_size<float, __nv_bfloat16>(p, vec, s);
  return p.y_f32 ? by_size<__nv_bfloat16, float>(p, vec, s) : by_size<__nv_bfloat16, __nv_bfloat16>(p, vec, s);
}

}  // namespace

cudaError_t layer_norm_fwd(const LnForward& p, cudaStream_t s) {
  if (p.rows <= 0) return cudaSuccess;
  if (p.C <= 0 || p.C > LN_CHANNELS || p.inner <= 0 || (p.r != nullptr) != (p.s != nullptr) || (p.r && p.r_f32 && !p.x_f32) ||
      (p.C > LN_HALF_PARAMS && ((p.w && !p.w_f32) || (p.b && !p.b_f32))))
    return cudaErrorInvalidValue;
  // whole 16-byte vectors in every tensor
  const bool vec = p.C % 8 == 0 && p.outer_stride % 8 == 0 && p.inner_stride % 8 == 0 && aligned(p.x) && aligned(p.r) && aligned(p.s) && aligned(p.y) &&
                   aligned(p.w) && aligned(p.b);
  return by_type(p, vec, s);
}

long long layer_norm_scratch(long long rows, int C) {
  // (as many blocks as either form of the kernel may take)
  const long long n = std::max(blocks_of(rows, spread(C, C % 8 == 0, BWD_ROWS), BWD_BLOCKS), blocks_of(rows, spread(C, false, BWD_ROWS), BWD_BLOCKS));
  return n > 1 ? 2 * n * C : 0;
}

cudaError_t layer_norm_bwd(const LnBackward& p, int* launches, cudaStream_t s) {
  *launches = 0;
  if (p.C <= 0 || p.C > LN_CHANNELS || p.inner <= 0 || (p.dw != nullptr) != (p.db != nullptr) || (p.C > LN_HALF_PARAMS && p.w && !p.w_f32))
    return cudaErrorInvalidValue;
  if (p.rows <= 0) return cudaSuccess;
  const bool vec = p.C % 8 == 0 && p.outer_stride % 8 == 0 && p.inner_stride % 8 == 0 && aligned(p.x) && aligned(p.dy) && aligned(p.ds) &&
                   aligned(p.dx) && aligned(p.dr) && aligned(p.w) && aligned(p.dw) && aligned(p.db) && aligned(p.part);
  const unsigned blocks = blocks_of(p.rows, spread(p.C, vec, BWD_ROWS), BWD_BLOCKS);
  if (p.dw && blocks > 1 && !p.part) return cudaErrorInvalidValue;
  ++*launches;
  const cudaError_t e = by_type(p, vec, s);
  if (e != cudaSuccess || !p.dw || blocks == 1) return e;
  ++*launches;
  const int n = static_cast<int>(blocks);
  return colsum_add_slabs(RowSlabs{p.part, p.dw, n, p.C, 1, !p.dw_f32}, RowSlabs{p.part + static_cast<long long>(n) * p.C, p.db, n, p.C, 1, !p.db_f32}, s);
}

}  // namespace mk
