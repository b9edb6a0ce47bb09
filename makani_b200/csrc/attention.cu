// Softmax attention on the tensor cores, with S = scale Q K^T:
//
//   forward    P = exp(S - max), O = P V / sum P, L = max + log sum P                           (one pass over the keys, running max and sum)
//   backward   P = exp(S - L), dV = P^T dO, dS = P (dO V^T - delta), dQ = scale dS K, dK = scale dS^T Q,  delta = sum_d O dO
//
// Exponentials are powers of two of (scale log2 e) S: one special-function instruction each, but for a quarter of those of the backward pass, which are a
// polynomial on the FMA pipe (`ex2_poly`).  Products take bf16 operands and add in fp32 (tensor memory); P and dS are rounded to bf16 as operands of the
// second products (half a step, 2^-8 of each weight at most, as the rounding of the outputs), sums, maxima and L stay in fp32.
//
// Warps: 0 loads tiles (TMA), 1 (and 3, narrow heads forward) issues products, 2 (and 3, dK and dV) loads statistics and clears rows that belong to another
// sequence, those from 4 on compute on rows in tensor memory, a thread a row or a part of one.  Every wait is bounded; on expiry the kernel records a
// code in *err and drains.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "attention.cuh"
#include "fused_ops.cuh"
#include "launch.cuh"
#include "tcgen05.cuh"
#include "gelu.cuh"

namespace mk {

namespace {

constexpr int TILE = 128;                        // keys (or queries) of a tile
constexpr int BOX = TILE * 128;                  // bytes of 64 channels of a tile
constexpr int THREADS = 384;
constexpr int COMPUTE_WARP = 4;                  // first of eight
constexpr float LOG2E = 1.4426950408889634f;

// fp32 accumulator, bf16 operands
constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((TILE >> 4) << 24);
__device__ __forceinline__ constexpr uint32_t idesc_n(int n) { return IDESC | (static_cast<uint32_t>(n >> 3) << 17); }
constexpr uint32_t B_MN = 1u << 16;      // second operand with its rows contiguous

// first operand from tensor memory: a lane a row, two bf16 to a column
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 db;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accum)
      : "memory");
}

// A wait that is mostly over when it begins
__device__ __forceinline__ bool mbar_wait_soon(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred P1;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 P1, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P1;\n\t"
      "}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok || mbar_wait(bar, parity);
}

#define MK_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define MK_RW8(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7])
#define MK_RD8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
// 32 columns of the thread's lane: request, and the wait for all requests
__device__ __forceinline__ void tmem_req32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : MK_R8(v, 0), MK_R8(v, 8), MK_R8(v, 16), MK_R8(v, 24)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait32(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : MK_RW8(v, 0), MK_RW8(v, 8), MK_RW8(v, 16), MK_RW8(v, 24)::"memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31};" ::MK_RD8(v, 0),
      MK_RD8(v, 8), MK_RD8(v, 16), MK_RD8(v, 24), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::MK_RD8(v, 0),
               MK_RD8(v, 8), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::MK_RD8(v, 0), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Registers of a warp group: all of them together stay within the THREADS * 168 of the launch
constexpr int FEW_REGS = 80, MANY_REGS = 208;
static_assert(128 * FEW_REGS + 256 * MANY_REGS <= THREADS * 168);
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// Two branches that begin with this stay two: merged, whole tiles pay for the comparisons of those at an edge (4 instructions an element)
template <bool EDGE>
__device__ __forceinline__ void apart() { asm volatile("" ::"n"(EDGE ? 1 : 0)); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The greater of x and `least`, NaN if x is NaN
__device__ __forceinline__ float at_least(float x, float least) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(least));
  return y;
}
// 2^x of two values with fp32 arithmetic, for a share of a tile's exponentials: the special function unit takes 1024 cycles for 128 x 128 of them, while the
// FMA pipe has time.  x = n + f with n the integer next to it (1.5 2^23 added and taken away), 2^f from a polynomial (Remez exchange for the least
// relative error on |f| <= 1/2: 2.7e-6 in fp32), times 2^n made of n's bits.  Below -126 it stays at 2^-126.  NaN comes out as NaN (through the product:
// n added to the exponent's bits would make a number of it): a row whose scores have no finite sum has L = NaN, and shows it in every gradient.
__device__ __forceinline__ void ex2_poly(float& a, float& b) {
  const float nearest = 12582912.f;
  const f32x2 x = f2_pack(at_least(a, -126.f), at_least(b, -126.f));
  const f32x2 t = f2_add(x, f2_pack(nearest, nearest));
  const f32x2 n = f2_add(t, f2_pack(-nearest, -nearest));
  const f32x2 f = f2_fma(n, f2_pack(-1.f, -1.f), x);
  f32x2 y = f2_fma(f, f2_pack(0.009570102207362652f, 0.009570102207362652f), f2_pack(0.05591785907745361f, 0.05591785907745361f));
  y = f2_fma(y, f, f2_pack(0.240247443318367f, 0.240247443318367f));
  y = f2_fma(y, f, f2_pack(0.6931217908859253f, 0.6931217908859253f));
  y = f2_fma(y, f, f2_pack(0.9999992847442627f, 0.9999992847442627f));
  float ta, tb;
  f2_unpack(t, ta, tb);
  constexpr uint32_t one = 0x3f800000u;
  f2_unpack(f2_mul(y, f2_pack(__uint_as_float((__float_as_uint(ta) << 23) + one), __uint_as_float((__float_as_uint(tb) << 23) + one))), a, b);
}
// Pair `i` of a row: POLY of every eight on the FMA pipe
template <int POLY>
__device__ __forceinline__ void ex2_pair(int i, float& a, float& b) {
  if ((i * POLY) % 8 < POLY) {
    ex2_poly(a, b);
  } else {
    a = ex2(a);
    b = ex2(b);
  }
}
// The greatest (of what is no NaN) of N values; three at a time where the warp has nothing else to wait for (8192 causal tokens, 16 heads of 128: 284 us
// with, 266 without; 16200 tokens, 8 heads of 48: 723 with, 728 without)
template <bool THREE, int N>
__device__ __forceinline__ float max_of(const uint32_t (&v)[N]) {
  if constexpr (!THREE) {
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __uint_as_float(v[i]);
#pragma unroll
    for (int c = 4; c < N; ++c) m[c & 3] = fmaxf(m[c & 3], __uint_as_float(v[c]));
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  } else {
    float m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = __uint_as_float(v[i]);
#pragma unroll
    for (int c = 8; c + 15 < N; c += 16)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        asm("max.f32 %0, %0, %1, %2;" : "+f"(m[i]) : "f"(__uint_as_float(v[c + 2 * i])), "f"(__uint_as_float(v[c + 2 * i + 1])));
#pragma unroll
    for (int c = 8 + (N - 8) / 16 * 16; c < N; ++c) m[c & 7] = fmaxf(m[c & 7], __uint_as_float(v[c]));
    return fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), fmaxf(fmaxf(m[4], m[5]), fmaxf(m[6], m[7])));
  }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ------------------------------------------------------------------------------------------ sequences and tiles

// What a CTA works on: rows r0 .. of a sequence of `len` tokens that begins at token `lo` of batch `b`
struct Work {
  int b, h, lo, len, r0;
  bool padding;            // rows behind the last sequence
};

// Tiles of `rows` rows.  Sequence s has the slots from offsets[s] / rows + s on: as many as it can need without knowing the others' lengths, so
// that a slot finds its sequence by a search over the offsets.  At most one slot of a sequence has no rows.
struct Slots {
  int B, N, H, rows, slots;
  int order;               // of the CTAs: 0: the tiles of one head follow one another; causal, long rows first: 1: last tiles first, 2: first tiles first; through a
                           // window (`find_work_of_head`) always one of these
  const int* offsets;
  int sequences;
};

__device__ __forceinline__ int clamp_offset(int v, int n) { return min(max(v, 0), n); }

// The sequence and the rows of a slot, all lanes of a warp; false: nothing to do
__device__ __forceinline__ bool find_rows(const Slots& g, const int* offsets, int slot, Work& w) {
  w.padding = false;
  if (!offsets) {
    w.lo = 0;
    w.len = g.N;
    w.r0 = slot * g.rows;
    return w.r0 < w.len;
  }
  // (the first sequence begins with the first token)
  auto begin = [&](int s) { return s == 0 ? 0 : clamp_offset(__ldg(offsets + s), g.N); };
  // the last sequence whose first slot is not behind this one, 32 ways at a time
  int lo = 0, hi = g.sequences + 1;                    // it is in [lo, hi); `sequences` stands for the rows behind the last one
  const int lane = threadIdx.x & 31;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const bool ok = at < hi && (at == lo || begin(at) / g.rows + at <= slot);
    const uint32_t m = __ballot_sync(0xffffffffu, ok);
    const int best = 31 - __clz(m);
    lo = lo + best * step;
    hi = min(hi, lo + step);
  }
  w.padding = lo == g.sequences;
  w.lo = begin(lo);
  w.len = (w.padding ? g.N : max(begin(lo + 1), w.lo)) - w.lo;
  w.r0 = (slot - (w.lo / g.rows + lo)) * g.rows;
  return w.r0 >= 0 && w.r0 < w.len;
}
__device__ __forceinline__ bool find_work(const Slots& g, const int* offsets, uint32_t block, Work& w) {
  int slot;
  if (g.order) {
    w.h = static_cast<int>(block % g.H);
    const uint32_t rest = block / g.H;
    slot = static_cast<int>(rest % g.slots);
    if (g.order == 1) slot = g.slots - 1 - slot;
    w.b = static_cast<int>(rest / g.slots);
  } else {
    slot = static_cast<int>(block % g.slots);
    const uint32_t rest = block / g.slots;
    w.h = static_cast<int>(rest % g.H);
    w.b = static_cast<int>(rest / g.H);
  }
  return find_rows(g, offsets, slot, w);
}
// Through a window, heads along x, and the tiles of the batches one behind the other along y and z: a CTA does not begin with divisions that wait for one another, and
// long and short ones, in the middle and at the ends of a sequence, come in the same order for all heads (with the tiles of one head behind the other 9472 tokens, 8 heads
// of 64, 4000 to either side took 226 us forward, 727 both ways, where this takes 184 and 641; 16204 tokens, 12 heads of 64, 720 to either side 159 / 149, 588 / 578;
// the middle of all heads first, their ends last 182, 645; 153, 593).  `unit` comes in as the place along y and z and goes out as what `find_work` takes (order 0).
__device__ __forceinline__ uint32_t place_in_head() { return blockIdx.z * gridDim.y + blockIdx.y; }
__device__ __forceinline__ bool find_work_of_head(const Slots& g, const int* offsets, uint32_t& unit, Work& w) {
  const uint32_t b = g.B == 1 ? 0u : unit / g.slots;
  int slot = static_cast<int>(unit - b * g.slots);
  w = Work{};
  if (b >= static_cast<uint32_t>(g.B) || slot >= g.slots) return false;      // (y times z is more than there are)
  if (g.order == 1) slot = g.slots - 1 - slot;
  w.h = static_cast<int>(blockIdx.x);
  w.b = static_cast<int>(b);
  unit = (b * g.H + w.h) * g.slots + slot;
  return find_rows(g, offsets, slot, w);
}

// Clears the rows from `valid` on of a tile of `boxes` boxes (a warp): they belong to another sequence, and what stands there, NaN perhaps, would
// be multiplied by zero weights.
__device__ __forceinline__ void clear_rows(uint8_t* tile, int boxes, int valid) {
  const int lane = threadIdx.x & 31;
  for (int b = 0; b < boxes; ++b)
    for (int i = valid * 8 + lane; i < TILE * 8; i += 32) *reinterpret_cast<uint4*>(tile + b * BOX + i * 16) = make_uint4(0, 0, 0, 0);
  fence_async_smem();
  __syncwarp();
}

// A wait behind `n` tiles (a warp): the bound of one wait for every 64 of them, as the others' waits are bounded tile by tile
__device__ __forceinline__ bool wait_long(uint32_t bar, uint32_t parity, int n) {
  for (int i = 0; i <= n; i += 64)
    if (__all_sync(0xffffffffu, mbar_wait(bar, parity))) return true;
  return false;
}

struct TileParams {
  Slots grid;
  int D, DP;               // channels of a head, and rounded up to 16
  int group;               // heads of q that share one of k and v
  int causal;
  float scale, scale_log2;
  int* err;
};

// ------------------------------------------------------------------------------------------ windows
//
// Token i sees key j if i - left <= j <= i + right, or j < sinks (and j <= i where causal).  Tiles of keys outside are not visited: a tile of queries goes
// over those of its window and those with sinks.  Instances of the kernels without WIN are what they are without windows.

struct Window {
  int causal, left, right, sinks;      // right is 0 where causal
};

// Tiles of keys that a CTA goes over, in order: `front` from `lo` on, those with sinks, and the rest of the window.  Of two query tiles the first sees
// those up to end[0], and the second those from start on (its window begins a tile later), up to end[1]; what else one of them does not see it hides.
struct KeyTiles {
  int lo = 0, front = 0, sinks = 0, start = 0, end[2] = {0, 0};
  __device__ __forceinline__ int operator()(int j) const { return j < front ? lo + j : j < front + sinks ? j - front : lo + j - sinks; }
};
__device__ __forceinline__ int last_seen(const Window& p, int i, int len) { return p.causal || i >= len ? min(i, len - 1) : p.right < len - 1 - i ? i + p.right : len - 1; }
__device__ __forceinline__ KeyTiles key_tiles(const Window& p, int r0, int rows, int len) {
  KeyTiles k;
  if (rows <= 0) return k;
  const bool two = rows > TILE;
  const int last[2] = {r0 + min(rows, TILE) - 1, r0 + rows - 1};
  const int lo0 = max(r0 - p.left, 0) / TILE, lo1 = max(r0 + TILE - p.left, 0) / TILE;
  const int hi0 = last_seen(p, last[0], len) / TILE + 1, hi1 = last_seen(p, last[1], len) / TILE + 1;
  k.sinks = (min(p.sinks, p.causal ? last[1] + 1 : len) + TILE - 1) / TILE;
  if (k.sinks > 0 && lo0 <= k.sinks) {      // they meet
    k.end[0] = max(hi0, k.sinks);
    k.end[1] = two ? max(hi1, k.sinks) : 0;
    k.sinks = 0;
    return k;
  }
  k.lo = lo0;
  k.front = k.start = two ? lo1 - lo0 : 0;
  k.end[0] = hi0 - lo0 + k.sinks;
  k.end[1] = two ? hi1 - lo0 + k.sinks : 0;
  return k;
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
template <bool WIN, typename P>
__device__ __forceinline__ KeyTiles window_keys(const P& p, const Work& w, int rows) {
  if constexpr (WIN) return key_tiles(p.win, w.r0, w.padding ? 0 : rows, w.len);
  else return KeyTiles();
}
// The keys from k0 on that token i sees, as columns: from `from` to `to`, and those below `sinks`
struct SeenKeys {
  int from, to, sinks;
  __device__ __forceinline__ SeenKeys(const Window& p, int i, int len, int k0)
      : from(i - p.left - k0), to(last_seen(p, i, len) + 1 - k0), sinks(min(p.sinks, p.causal ? min(i + 1, len) : len) - k0) {}
  // of the 32 columns from c0 on
  __device__ __forceinline__ uint32_t bits(int c0) const { return (low_bits(to - c0) & ~low_bits(from - c0)) | low_bits(sinks - c0); }
};
// Tiles of a CTA's list that are seen as a whole, as a range (tiles with sinks count for none: they may always be looked at)
struct Whole {
  int from = 0;
  uint32_t n = 0;
  __device__ __forceinline__ bool operator()(int j) const { return static_cast<uint32_t>(j - from) < n; }
};
__device__ __forceinline__ int tiles_over(int n) { return n <= 0 ? 0 : (n + TILE - 1) / TILE; }
// Of keys, by each of the 128 tokens from `first` on
__device__ __forceinline__ Whole whole_keys(const Window& p, const KeyTiles& k, int first, int len) {
  const int from = max(tiles_over(first + TILE - 1 - p.left) - k.lo, k.front), to = (last_seen(p, first, len) + 1) / TILE - k.lo;
  return {from + k.sinks, static_cast<uint32_t>(max(to - from, 0))};
}
// Of queries, by which all 128 keys from r0 on are seen: tiles behind `first`
__device__ __forceinline__ Whole whole_queries(const Window& p, int r0, int len, int first) {
  const bool sinks = r0 + TILE <= p.sinks;
  const int from = max(sinks && !p.causal ? 0 : tiles_over(r0 + TILE - 1 - p.right), first);
  const int to = sinks || p.left >= len - 1 - r0 ? len / TILE : (r0 + p.left + 1) / TILE;
  return {from - first, static_cast<uint32_t>(max(to - from, 0))};
}

// 16 (or the first 8) fp32 values as bf16
__device__ __forceinline__ void store16(const uint32_t (&v)[16], __nv_bfloat16* to, bool all) {
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = pack_bf16(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
  reinterpret_cast<uint4*>(to)[0] = make_uint4(h[0], h[1], h[2], h[3]);
  if (all) reinterpret_cast<uint4*>(to)[1] = make_uint4(h[4], h[5], h[6], h[7]);
}
// The first D columns of an accumulator's row, times f, as bf16: those from `first` on in steps of `step` (multiples of 16)
__device__ __forceinline__ void store_row(uint32_t taddr, int D, float f, __nv_bfloat16* to, bool here, int first = 0, int step = 16) {
  for (int c = first; c < D; c += step) {
    uint32_t v[16];
    tmem_ld16(taddr + c, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
    if (here) store16(v, to + c, c + 8 < D);
  }
}
// The same for o, with what its rounding leaves out beside it (`rest`, if there is one): delta = sum o d_o from o alone, off by half a step of every
// o, made the gradients of queries and keys of short sequences half as much less exact again (128 tokens, 8 channels: 2.6e-3 of their size, 2.3e-3
// with it)
__device__ __forceinline__ void store_output(uint32_t taddr, int D, float f, __nv_bfloat16* to, __nv_bfloat16* rest, bool here) {
  for (int c = 0; c < D; c += 16) {
    uint32_t v[16];
    tmem_ld16(taddr + c, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
    if (here) store16(v, to + c, c + 8 < D);
    if (rest && here) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) - __bfloat162float(__float2bfloat16(__uint_as_float(v[i]))));
      store16(v, rest + c, c + 8 < D);
    }
  }
}
// Eight bf16 of eight fp32 values
__device__ __forceinline__ uint4 pack8(const uint32_t* v) {
  return make_uint4(pack_bf16(__uint_as_float(v[0]), __uint_as_float(v[1])), pack_bf16(__uint_as_float(v[2]), __uint_as_float(v[3])),
                    pack_bf16(__uint_as_float(v[4]), __uint_as_float(v[5])), pack_bf16(__uint_as_float(v[6]), __uint_as_float(v[7])));
}
// The same through shared memory (`stage`: 32 rows of PITCH bytes), so that lanes side by side write what lies side by side.  `to`: of the warp's first row, `rows` of
// which are here, `stride` elements apart.
template <int PITCH>
__device__ __forceinline__ void stage_output(uint32_t taddr, int D, float f, uint8_t* stage, __nv_bfloat16* to, __nv_bfloat16* rest, long long stride, int rows) {
  const int lane = threadIdx.x & 31, chunks = D / 8;
  const uint32_t by_chunks = 65536u / chunks + 1;      // i / chunks = i by_chunks >> 16 for i below 32 x 16
  auto at = [&](int row, int c) { return reinterpret_cast<uint4*>(stage + row * PITCH + ((c ^ (row & 7)) << 4)); };
  for (int pass = 0; pass < (rest ? 2 : 1); ++pass) {
    for (int c = 0; c < D; c += 16) {
      uint32_t v[16];
      tmem_ld16(taddr + c, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float o = __uint_as_float(v[i]) * f;
        v[i] = __float_as_uint(pass ? o - __bfloat162float(__float2bfloat16(o)) : o);
      }
      *at(lane, c / 8) = pack8(v);
      if (c + 8 < D) *at(lane, c / 8 + 1) = pack8(v + 8);
    }
    __syncwarp();
    __nv_bfloat16* const out = pass ? rest : to;
    for (int i = lane; i < rows * chunks; i += 32) {
      const int row = static_cast<int>(i * by_chunks >> 16), c = i - row * chunks;
      *reinterpret_cast<uint4*>(out + row * stride + c * 8) = *at(row, c);
    }
    __syncwarp();
  }
}
// Columns c0 to c1 (whole eights, 8 CHUNKS of them at most) of an accumulator's rows, times f, as bf16, through shared memory in the same way (`stage`: 32 rows of CHUNKS x 16 bytes)
template <int CHUNKS>
__device__ __forceinline__ void stage_rows(uint32_t taddr, int c0, int c1, float f, uint8_t* stage, __nv_bfloat16* to, long long stride, int rows) {
  const int lane = threadIdx.x & 31;
  auto at = [&](int row, int c) { return reinterpret_cast<uint4*>(stage + (row * CHUNKS + (c ^ ((row * CHUNKS >> 3) & (CHUNKS - 1)))) * 16); };
#pragma unroll
  for (int c = 0; c < 8 * CHUNKS; c += 16) {
    if (c0 + c >= c1) break;
    uint32_t v[16];
    tmem_ld16(taddr + c0 + c, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
    *at(lane, c / 8) = pack8(v);
    *at(lane, c / 8 + 1) = pack8(v + 8);      // (behind the last column perhaps)
  }
  __syncwarp();
#pragma unroll
  for (int i = lane; i < 32 * CHUNKS; i += 32) {
    const int row = i / CHUNKS, c = i % CHUNKS;
    if (row < rows && c0 + c * 8 < c1) *reinterpret_cast<uint4*>(to + row * stride + c0 + c * 8) = *at(row, c);
  }
}
// CTAs that are split over what they go along: those from `whole` on, into `parts`
struct Parts {
  uint32_t whole;
  int parts;               // 0: none is split
};
// What this CTA has of it: its unit, its part (-1: all of it), tiles in front of its own and number of its own.  Without SPLIT it has all of its unit: the
// kernels of the gradients are built both ways, since the part that may begin in the middle costs a whole one 3 % (dQ) and 1 % (dK, dV).
template <bool SPLIT>
struct ShareOf {
  uint32_t unit;
  int part, first, n;
  __device__ __forceinline__ explicit ShareOf(const Parts& s) : ShareOf(s, blockIdx.x) {}
  __device__ __forceinline__ ShareOf(const Parts& s, uint32_t block) : unit(block), part(-1) {
    if (SPLIT && s.parts > 0 && block >= s.whole) {
      unit = s.whole + (block - s.whole) / s.parts;
      part = static_cast<int>((block - s.whole) % s.parts);
    }
  }
  __device__ __forceinline__ void along(const Parts& s, int tiles) {
    first = !SPLIT || part < 0 ? 0 : static_cast<int>(static_cast<long long>(tiles) * part / s.parts);
    n = (!SPLIT || part < 0 ? tiles : static_cast<int>(static_cast<long long>(tiles) * (part + 1) / s.parts)) - first;
  }
  // row of a buffer [unit - whole][part][rows]
  __device__ __forceinline__ long long row(const Parts& s, int rows, int r) const {
    return (static_cast<long long>(unit - s.whole) * s.parts + part) * rows + r;
  }
};
using Share = ShareOf<true>;
// An accumulator's row as it is, the first D columns, from `first` on in steps of `step`
__device__ __forceinline__ void store_part(uint32_t taddr, int D, float* to, bool here, int first = 0, int step = 8) {
  for (int c = first; c < D; c += step) {
    uint32_t v[8];
    tmem_ld8(taddr + c, v);
    if (here) {
      reinterpret_cast<uint4*>(to + c)[0] = make_uint4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<uint4*>(to + c)[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
  }
}
__device__ __forceinline__ void zero_row(int D, __nv_bfloat16* to) {
  for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(to + c) = make_uint4(0, 0, 0, 0);
}

template <uint32_t COLS>
__device__ __forceinline__ void tmem_alloc(volatile uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t*>(slot))), "r"(COLS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <uint32_t COLS>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
}

// ------------------------------------------------------------------------------------------ forward

// O is rescaled where the maximum has grown by more than a factor of 2^8 since: the weights then reach 256 instead of 1, with the same relative
// rounding, and nearly all tiles leave O alone.  (That the maximum may lag behind by a bounded factor is known from published work on attention for this chip.)
constexpr float MAX_GROWTH = 8.f;

// A row of the running softmax: what its weights are relative to (times scale), and their sum
struct Row {
  float m = -INFINITY;
  f32x2 sum[2] = {0ull, 0ull};

  // Whether the scores of a tile ask for a new maximum; `f`: what sums, and O, are multiplied by then.  Row by row: what a row holds does not depend
  // on its neighbours.
  __device__ __forceinline__ bool grows(float top) const { return top > m + MAX_GROWTH; }
  __device__ __forceinline__ float grow(float top) {
    const float up = grows(top) ? top : m, f = up == m ? 1.f : ex2(m - up);
    m = up;
    sum[0] = f2_mul(sum[0], f2_pack(f, f));
    sum[1] = f2_mul(sum[1], f2_pack(f, f));
    return f;
  }
  __device__ __forceinline__ float total() const {
    float a, b;
    f2_unpack(f2_add(sum[0], sum[1]), a, b);
    return a + b;
  }
  // 128 scores -> weights 2^(scale S - m), as bf16 in the first half of them.  (A share of the exponentials on the FMA pipe, which helps the backward
  // pass, is slower here: 16200 tokens, 8 heads of 48: 750 us without, 860 - 930 with an eighth to three eighths of them.)
  __device__ __forceinline__ void weights(uint32_t (&v)[TILE], float scale) {
    // (a row that has seen nothing but -inf has no maximum yet, and weights of 0)
    const float from = m == -INFINITY ? 0.f : -m;
    const f32x2 scale2 = f2_pack(scale, scale), from2 = f2_pack(from, from);
#pragma unroll
    for (int c = 0; c < TILE; c += 2) {
      float a, b;
      f2_unpack(f2_fma(f2_pack(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, from2), a, b);
      a = ex2(a);
      b = ex2(b);
      sum[(c >> 1) & 1] = f2_add(sum[(c >> 1) & 1], f2_pack(a, b));
      v[c / 2] = pack_bf16(a, b);
    }
  }
  // The same; `none`: a bit for each 32 columns whose weights are 0 without a look
  __device__ __forceinline__ void weights(uint32_t (&v)[TILE], float scale, uint32_t none) {
    const float from = m == -INFINITY ? 0.f : -m;
    const f32x2 scale2 = f2_pack(scale, scale), from2 = f2_pack(from, from);
#pragma unroll
    for (int c0 = 0; c0 < TILE; c0 += 32) {
      if (none >> (c0 / 32) & 1) {
#pragma unroll
        for (int c = 0; c < 16; ++c) v[c0 / 2 + c] = 0u;
        continue;
      }
#pragma unroll
      for (int c = c0; c < c0 + 32; c += 2) {
        float a, b;
        f2_unpack(f2_fma(f2_pack(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, from2), a, b);
        a = ex2(a);
        b = ex2(b);
        sum[(c >> 1) & 1] = f2_add(sum[(c >> 1) & 1], f2_pack(a, b));
        v[c / 2] = pack_bf16(a, b);
      }
    }
  }
};
__device__ __forceinline__ void load_scores(uint32_t s_at, uint32_t (&v)[TILE]) {
#pragma unroll
  for (int c = 0; c < TILE; c += 32) tmem_req32(s_at + c, v + c);
#pragma unroll
  for (int c = 0; c < TILE; c += 32) tmem_wait32(v + c);
}
// what is hidden is -inf, and its weight 0
__device__ __forceinline__ void hide_scores(uint32_t (&v)[TILE], int seen) {
#pragma unroll
  for (int c = 0; c < TILE; ++c)
    if (c >= seen) v[c] = 0xff800000u;
}
// The same through a window, 32 columns at a time; a bit for each of those that no row of the warp sees
__device__ __forceinline__ uint32_t hide_scores(uint32_t (&v)[TILE], const SeenKeys& seen) {
  uint32_t none = 0;
#pragma unroll
  for (int c = 0; c < TILE; c += 32) {
    const uint32_t m = seen.bits(c);
    if (__all_sync(0xffffffffu, m == 0xffffffffu)) continue;
    if (!__any_sync(0xffffffffu, m != 0)) none |= 1u << (c / 32);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (!(m >> i & 1)) v[c + i] = 0xff800000u;
  }
  return none;
}
__device__ __forceinline__ void store_weights(uint32_t p_at, const uint32_t (&v)[TILE]) {
  tmem_st32(p_at, v);
  tmem_st32(p_at + 32, v + 32);
  tmem_st_wait();
}
// O of a row times f
__device__ __forceinline__ void scale_row(uint32_t o_at, int cols, float f) {
#pragma unroll 1
  for (int c = 0; c < cols; c += 8) {
    uint32_t a[8];
    tmem_ld8(o_at + c, a);
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = __float_as_uint(__uint_as_float(a[k]) * f);
    tmem_st8(o_at + c, a);
  }
}

// S in tensor memory (128 columns a query tile) is replaced by P in its first half; O has 128 columns beside it.  Two query tiles share every tile of keys
// and values, so that the products of one run beside the exponentials of the other; with one (short sequences) two CTAs share an SM instead, each
// with half of its tensor memory, and one's start and end run beside the other's work.
template <int DB, int QT>
struct Fwd {
  static constexpr int STAGES = QT == 2 ? 2 : 3 - DB, TILE_BYTES = DB * BOX, WARPS = COMPUTE_WARP + 4 * QT, THREADS_ = 32 * WARPS;
  static constexpr int K_AT = QT * TILE_BYTES, V_AT = K_AT + STAGES * TILE_BYTES, BAR_AT = V_AT + STAGES * TILE_BYTES;
  static constexpr int BARS = 4 * STAGES + 7;
  static constexpr int SMEM = BAR_AT + 8 * BARS + 16 + 1024;
  static constexpr uint32_t COLS = 256 * QT, O_AT = 128 * QT;
  // registers: within the launch's, 168 or (two CTAs) 128 a thread (for which the compiler spills 36 to 52 bytes in each of the forward kernels)
  static constexpr int FEW = QT == 2 ? FEW_REGS : 56, MANY = QT == 2 ? MANY_REGS : 200;
  static_assert(SMEM * (3 - QT) <= SMEM_LIMIT && 128 * FEW + 128 * QT * MANY <= THREADS_ * (QT == 2 ? 168 : 128));
};
constexpr uint32_t S_COLS = 128;
// Of the pairs of query tiles, those from `whole` on are split over the keys into `parts` CTAs each, which leave O (not divided) and maximum and sum of every
// row for the kernel that joins them
struct Split : Parts {
  float* o;                // [pair - whole][part][2 TILE][D]
  float2* ml;              // [pair - whole][part][2 TILE]
};

struct FwdParams {
  TileParams t;
  Split split;
  __nv_bfloat16 *o, *o_rest;
  float* lse;
};
// What a kernel has of `P`: with a window, that as well.  (In the parameters of all of them it makes the compiler arrange the registers of those without another
// way: 16200 tokens, 8 heads of 48, 677 us instead of 643.)
template <typename P>
struct Windowed : P {
  Window win;
};
template <typename P, bool WIN>
using With = typename std::conditional<WIN, Windowed<P>, P>::type;

template <int DB, int QT, bool WIN>
__global__ void __launch_bounds__(Fwd<DB, QT>::THREADS_, 3 - QT)
attn_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const With<FwdParams, WIN> p) {
  using L = Fwd<DB, QT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t base = raw_addr + pad, bars = base + L::BAR_AT;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 8u * (L::STAGES + s); };
  auto v_full = [&](int s) { return bars + 8u * (2 * L::STAGES + s); };
  auto v_empty = [&](int s) { return bars + 8u * (3 * L::STAGES + s); };
  const uint32_t q_full = bars + 8u * (4 * L::STAGES), v_fixed = q_full + 8u;
  auto s_full = [&](int t) { return v_fixed + 8u + 8u * t; };
  auto p_ready = [&](int t) { return v_fixed + 24u + 8u * t; };
  const uint32_t v_fix = v_fixed + 40u;
  volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_raw + pad + L::BAR_AT + 8 * L::BARS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    mbar_init(q_full, 1);
    mbar_init(v_fixed, 1);
    mbar_init(v_fix, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(p_ready(t), 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  // (two to an SM: not before the kernel in front has given its tensor memory back, which it may want to take on an SM that this one shares)
  if (QT == 2 && warp == 1) tmem_alloc<L::COLS>(tmem_slot);
  const int* offsets = p.t.grid.offsets;
  chain_begin(true, offsets);
  if (QT == 1 && warp == 1) tmem_alloc<L::COLS>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  Work w;
  Share share(p.split, WIN ? place_in_head() : blockIdx.x);
  const bool any = WIN ? find_work_of_head(p.t.grid, offsets, share.unit, w) : find_work(p.t.grid, offsets, share.unit, w);
  const int rows = any ? min(w.len - w.r0, QT * TILE) : 0;
  const bool causal = p.t.causal != 0;
  auto tiles_of = [&](int t) {      // of keys, that the queries of tile t see
    if (w.padding || rows <= t * TILE) return 0;
    const int last = causal ? w.r0 + min(rows, (t + 1) * TILE) - 1 : w.len - 1;
    return last / TILE + 1;
  };
  const KeyTiles keys = window_keys<WIN>(p, w, rows);
  int n0 = WIN ? keys.end[0] : tiles_of(0), n1 = WIN ? keys.end[1] : tiles_of(1);
  share.along(p.split, max(n0, n1));
  const int n = share.n, j0 = share.first;
  if (share.part >= 0) {      // (not causal: both see the same keys)
    n0 = n0 > 0 ? n : 0;
    n1 = n1 > 0 ? n : 0;
  }
  auto tile = [=](int j) {
    if constexpr (WIN) return keys(j);
    else return j0 + j;
  };
  // keys of the last tile that belong to the sequence, where other tokens follow it
  const int tail = w.len - tile(n - 1) * TILE;
  const bool fix = n > 0 && tail < TILE && w.lo + w.len < p.t.grid.N;

  if (warp < COMPUTE_WARP) {
    regs_down<L::FEW>();
    if (warp == 0) {
    // ------------------------------------------------------------------ tiles
    if (n > 0 && elect_one()) {
      const int hk = w.h / p.t.group;
      mbar_expect_tx(q_full, (n1 > 0 ? 2 : 1) * L::TILE_BYTES);
      for (int t = 0; t < (n1 > 0 ? 2 : 1); ++t)
        for (int b = 0; b < DB; ++b) tma_load_4d(base + t * L::TILE_BYTES + b * BOX, &map_q, q_full, b * 64, w.lo + w.r0 + t * TILE, w.h, w.b);
      int s = 0;
      uint32_t ph = 0;
      for (int j = 0; j < n; ++j) {
        if (!mbar_wait(k_empty(s), ph ^ 1u)) {
          atomicExch(p.t.err, 80);
          break;
        }
        mbar_expect_tx(k_full(s), L::TILE_BYTES);
        for (int b = 0; b < DB; ++b) tma_load_4d(base + L::K_AT + s * L::TILE_BYTES + b * BOX, &map_k, k_full(s), b * 64, w.lo + tile(j) * TILE, hk, w.b);
        if (!mbar_wait(v_empty(s), ph ^ 1u)) {
          atomicExch(p.t.err, 80);
          break;
        }
        mbar_expect_tx(v_full(s), L::TILE_BYTES);
        for (int b = 0; b < DB; ++b) tma_load_4d(base + L::V_AT + s * L::TILE_BYTES + b * BOX, &map_v, v_full(s), b * 64, w.lo + tile(j) * TILE, hk, w.b);
        if (++s == L::STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ products
    if (n > 0 && elect_one()) {
      const uint32_t hi = desc_hi(1024);
      const uint32_t q_lo = desc_lo(base, 16), k_lo = desc_lo(base + L::K_AT, 16), v_lo = desc_lo(base + L::V_AT, BOX);
      const uint32_t id_s = idesc_n(TILE), id_o = idesc_n(p.t.DP) | B_MN;
      const int ksteps = p.t.DP >> 4;
      auto scores = [&](int t, int s) {
        const uint32_t a = q_lo + t * (L::TILE_BYTES >> 4), b = k_lo + s * (L::TILE_BYTES >> 4);
        for (int i = 0; i < ksteps; ++i) {
          const uint32_t at = (i >> 2) * (BOX >> 4) + (i & 3) * 2;
          tc_mma<2, 1>(tmem + t * S_COLS, a + at, hi, b + at, hi, id_s, i > 0);
        }
        tc_commit(s_full(t));
      };
      bool ok = mbar_wait(q_full, 0) && mbar_wait(k_full(0), 0);
      if (!ok) atomicExch(p.t.err, 81);
      if (ok) {
        tc_fence_after();
        if (n0 > 0) scores(0, 0);
        if (n1 > 0 && keys.start == 0) scores(1, 0);
        tc_commit(k_empty(0));
      }
      int s = 0;
      uint32_t ph = 0;
      for (int j = 0; j < n && ok; ++j) {
        const int sn = s + 1 == L::STAGES ? 0 : s + 1;
        const uint32_t phn = sn == 0 ? ph ^ 1u : ph;
        ok = mbar_wait(v_full(s), ph);
        if (ok && fix && j == n - 1) {
          mbar_arrive(v_fix);
          ok = mbar_wait(v_fixed, 0);
        }
        if (ok && j + 1 < n) ok = mbar_wait(k_full(sn), phn);
        if (!ok) {
          atomicExch(p.t.err, 82);
          break;
        }
        tc_fence_after();
        for (int t = 0; t < 2 && ok; ++t) {
          const int nt = t == 0 ? n0 : n1, start = !WIN || t == 0 ? 0 : keys.start;
          if (j >= nt) continue;
          if (WIN && j < start) {      // (the first is the next one)
            scores(t, sn);
            continue;
          }
          if (!mbar_wait(p_ready(t), (j - start) & 1)) {
            atomicExch(p.t.err, 83);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t b = v_lo + s * (L::TILE_BYTES >> 4);
#pragma unroll
          for (int i = 0; i < TILE / 16; ++i)
            mma_ts(tmem + L::O_AT + t * ATTN_WIDTH, tmem + t * S_COLS + i * 8, b + i * (2048 >> 4), hi, id_o, j > start || i > 0);
          // (in order behind the products above: S takes the place of P)
          if (j + 1 < nt) scores(t, sn);
          else tc_commit(s_full(t));
        }
        tc_commit(v_empty(s));
        if (j + 1 < n) tc_commit(k_empty(sn));
        s = sn;
        ph = phn;
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ rows of the next sequence
    // (at the word of warp 1, which has seen the tile arrive)
    if (fix && wait_long(v_fix, 0, n)) {
      clear_rows(smem_raw + pad + L::V_AT + (n - 1) % L::STAGES * L::TILE_BYTES, DB, tail);
      if (lane == 0) mbar_arrive(v_fixed);
    }
    }
  } else {
    regs_up<L::MANY>();
    // ------------------------------------------------------------------ softmax
    const int t = (warp - COMPUTE_WARP) >> 2, row = t * TILE + (warp & 3) * 32 + lane, nt = t == 0 ? n0 : n1;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * S_COLS, o_at = tmem + lanes + L::O_AT + t * ATTN_WIDTH;
    const float scale = p.t.scale_log2;
    const bool here = row < rows;
    Row r;
    bool ok = true;
    const int start = !WIN || t == 0 ? 0 : keys.start;
    Whole whole;
    if constexpr (WIN) whole = whole_keys(p.win, keys, w.r0 + t * TILE, w.len);
    for (int j = start; j < nt; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(s_full(t), (j - start) & 1));
      if (!ok) break;
      tc_fence_after();
      uint32_t v[TILE];
      load_scores(s_at, v);
      auto grow = [&] {
        const float top = max_of<false>(v) * scale;
        if (__any_sync(0xffffffffu, r.grows(top))) {
          // (the scores of tile j are behind the products of tile j - 1: O is complete up to there)
          const float f = r.grow(top);
          if (j > start) scale_row(o_at, p.t.DP, f);
        }
      };
      if constexpr (WIN) {
        // (two ways from here on: on one for whole tiles and others, 16128 tokens, 8 heads of 48 with a window over nearly all took 925 us where there are 720 without it
        // and 791 like this)
        if (whole(j)) {
          apart<false>();
          grow();
          r.weights(v, scale);
        } else {
          apart<true>();
          const uint32_t none = hide_scores(v, SeenKeys(p.win, w.r0 + row, w.len, tile(j) * TILE));
          grow();
          r.weights(v, scale, none);
        }
      } else {
        const int k0 = tile(j) * TILE;
        if (k0 + TILE > w.len || (causal && k0 + TILE - 1 > w.r0 + t * TILE)) hide_scores(v, (causal ? min(w.len, w.r0 + row + 1) : w.len) - k0);
        grow();
        r.weights(v, scale);
      }
      store_weights(s_at, v);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready(t));
    }
    if (nt > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(s_full(t), (nt - start) & 1));
    if (!ok && lane == 0) atomicExch(p.t.err, 84);
    const long long token = static_cast<long long>(w.b) * p.t.grid.N + w.lo + w.r0 + row;
    __nv_bfloat16* const to = p.o + (token * p.t.grid.H + w.h) * p.t.D;
    if (nt > 0 && ok) {
      tc_fence_after();
      const float total = r.total();
      if (share.part >= 0) {
        const long long at = share.row(p.split, 2 * TILE, row);
        store_part(o_at, p.t.D, p.split.o + at * p.t.D, here);
        if (here) p.split.ml[at] = make_float2(r.m, total);
      } else {
        if constexpr (WIN) {
          __nv_bfloat16* const first = to - static_cast<long long>(lane) * p.t.grid.H * p.t.D;      // (the warp's first row)
          stage_output<DB * 128>(o_at, p.t.D, 1.f / total, smem_raw + pad + t * L::TILE_BYTES + (warp & 3) * (L::TILE_BYTES / 4), first,
                                 p.o_rest ? p.o_rest + (first - p.o) : nullptr, 1ll * p.t.grid.H * p.t.D, min(rows - row + lane, 32));
        } else {
          store_output(o_at, p.t.D, 1.f / total, to, p.o_rest ? p.o_rest + (to - p.o) : nullptr, here);
        }
        if (here && p.lse)
          p.lse[(static_cast<long long>(w.b) * p.t.grid.H + w.h) * p.t.grid.N + w.lo + w.r0 + row] = r.m + __log2f(total);
      }
    } else if (here && w.padding) {
      zero_row(p.t.D, to);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<L::COLS>(tmem);
  }
}

// Heads of up to 64 channels: tensor memory has room for S, P and O of both query tiles side by side (128, 64 and 64 columns), so that the next scores are
// on their way as soon as the last have been read, and no warp waits for products.  Through windows also with one query tile and two CTAs to an SM (16128 tokens, 8
// heads of 48, 704 to either side: 102 us where the kernel above takes 113).
template <int QT>
struct FwdNarrow {
  static constexpr int STAGES = 2 * QT, THREADS_ = 32 * (COMPUTE_WARP + 4 * QT);
  static constexpr int K_AT = QT * BOX, V_AT = K_AT + STAGES * BOX, BAR_AT = V_AT + STAGES * BOX;
  static constexpr int BARS = 4 * STAGES + 11;
  static constexpr int SMEM = BAR_AT + 8 * BARS + 16 + 1024;
  static constexpr uint32_t COLS = 256 * QT, P_AT = 128 * QT, O_AT = 192 * QT;
  static constexpr int FEW = Fwd<1, QT>::FEW, MANY = Fwd<1, QT>::MANY;
  static_assert(SMEM * (3 - QT) <= SMEM_LIMIT);
};

template <int QT, bool WIN>
__global__ void __launch_bounds__(FwdNarrow<QT>::THREADS_, 3 - QT)
attn_fwd_narrow_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const With<FwdParams, WIN> p) {
  using L = FwdNarrow<QT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t base = raw_addr + pad, bars = base + L::BAR_AT;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 8u * (L::STAGES + s); };
  auto v_full = [&](int s) { return bars + 8u * (2 * L::STAGES + s); };
  auto v_empty = [&](int s) { return bars + 8u * (3 * L::STAGES + s); };
  const uint32_t q_full = bars + 8u * (4 * L::STAGES), v_fix = q_full + 8u, v_fixed = q_full + 16u;
  auto s_full = [&](int t) { return q_full + 24u + 32u * t; };
  auto s_read = [&](int t) { return q_full + 32u + 32u * t; };
  auto p_ready = [&](int t) { return q_full + 40u + 32u * t; };
  auto o_done = [&](int t) { return q_full + 48u + 32u * t; };
  volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_raw + pad + L::BAR_AT + 8 * L::BARS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(k_empty(s), QT);
      mbar_init(v_empty(s), QT);
    }
    mbar_init(q_full, 1);
    mbar_init(v_fix, QT);
    mbar_init(v_fixed, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(s_read(t), 4);
      mbar_init(p_ready(t), 4);
      mbar_init(o_done(t), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (QT == 2 && warp == 1) tmem_alloc<L::COLS>(tmem_slot);
  const int* offsets = p.t.grid.offsets;
  chain_begin(true, offsets);
  if (QT == 1 && warp == 1) tmem_alloc<L::COLS>(tmem_slot);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  Work w;
  Share share(p.split, WIN ? place_in_head() : blockIdx.x);
  const bool any = WIN ? find_work_of_head(p.t.grid, offsets, share.unit, w) : find_work(p.t.grid, offsets, share.unit, w);
  const int rows = any ? min(w.len - w.r0, QT * TILE) : 0;
  const bool causal = p.t.causal != 0;
  auto tiles_of = [&](int t) {      // of keys, that the queries of tile t see
    if (w.padding || rows <= t * TILE) return 0;
    const int last = causal ? w.r0 + min(rows, (t + 1) * TILE) - 1 : w.len - 1;
    return last / TILE + 1;
  };
  const KeyTiles keys = window_keys<WIN>(p, w, rows);
  int n0 = WIN ? keys.end[0] : tiles_of(0), n1 = WIN ? keys.end[1] : tiles_of(1);
  share.along(p.split, max(n0, n1));
  const int n = share.n, j0 = share.first;
  if (share.part >= 0) {      // (not causal: both see the same keys)
    n0 = n0 > 0 ? n : 0;
    n1 = n1 > 0 ? n : 0;
  }
  auto tile = [=](int j) {
    if constexpr (WIN) return keys(j);
    else return j0 + j;
  };
  const int tail = w.len - tile(n - 1) * TILE;
  const bool fix = n > 0 && tail < TILE && w.lo + w.len < p.t.grid.N;

  if (warp < COMPUTE_WARP) {
    regs_down<L::FEW>();
    if (warp == 0) {
      // ---------------------------------------------------------------- tiles
      if (n > 0 && elect_one()) {
        const int hk = w.h / p.t.group, nq = rows > TILE ? 2 : 1;
        mbar_expect_tx(q_full, nq * BOX);
        for (int t = 0; t < nq; ++t) tma_load_4d(base + t * BOX, &map_q, q_full, 0, w.lo + w.r0 + t * TILE, w.h, w.b);
        int s = 0;
        uint32_t ph = 0;
        for (int j = 0; j < n; ++j) {
          if (!mbar_wait(k_empty(s), ph ^ 1u)) {
            atomicExch(p.t.err, 80);
            break;
          }
          mbar_expect_tx(k_full(s), BOX);
          tma_load_4d(base + L::K_AT + s * BOX, &map_k, k_full(s), 0, w.lo + tile(j) * TILE, hk, w.b);
          if (!mbar_wait(v_empty(s), ph ^ 1u)) {
            atomicExch(p.t.err, 80);
            break;
          }
          mbar_expect_tx(v_full(s), BOX);
          tma_load_4d(base + L::V_AT + s * BOX, &map_v, v_full(s), 0, w.lo + tile(j) * TILE, hk, w.b);
          if (++s == L::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    } else if (QT == 2 ? (warp & 1) != 0 : warp == 1) {
      // ---------------------------------------------------------------- products, a warp for either query tile
      if (n > 0 && elect_one()) {
        const int t = warp >> 1, nt = t == 0 ? n0 : n1, start = !WIN || t == 0 ? 0 : keys.start;
        const uint32_t hi = desc_hi(1024);
        const uint32_t q_lo = desc_lo(base + t * BOX, 16), k_lo = desc_lo(base + L::K_AT, 16), v_lo = desc_lo(base + L::V_AT, BOX);
        const uint32_t id_s = idesc_n(TILE), id_o = idesc_n(p.t.DP) | B_MN, o = tmem + L::O_AT + t * 64, a = tmem + L::P_AT + t * 64;
        const int ksteps = p.t.DP >> 4;
        auto scores = [&](int s) {
          const uint32_t b = k_lo + s * (BOX >> 4);
          for (int k = 0; k < ksteps; ++k) tc_mma<2, 1>(tmem + t * S_COLS, q_lo + 2 * k, hi, b + 2 * k, hi, id_s, k > 0);
          tc_commit(s_full(t));
        };
        bool ok = mbar_wait(q_full, 0) && mbar_wait(k_full(0), 0);
        if (!ok) atomicExch(p.t.err, 81);
        if (ok) {
          tc_fence_after();
          if (nt > 0 && start == 0) scores(0);
          tc_commit(k_empty(0));
        }
        int s = 0;
        uint32_t ph = 0;
        for (int j = 0; j < n && ok; ++j) {
          const int sn = s + 1 == L::STAGES ? 0 : s + 1;
          const uint32_t phn = sn == 0 ? ph ^ 1u : ph;
          // (a tile that this warp has no use for is given back as soon as it is there)
          if (j + 1 < n) {
            ok = mbar_wait(k_full(sn), phn) && (j + 1 >= nt || j < start || mbar_wait(s_read(t), (j - start) & 1));
            if (!ok) {
              atomicExch(p.t.err, 82);
              break;
            }
            tc_fence_after();
            if (j + 1 < nt) scores(sn);
            tc_commit(k_empty(sn));
          }
          ok = mbar_wait(v_full(s), ph);
          if (ok && fix && j == n - 1) {
            mbar_arrive(v_fix);
            ok = mbar_wait(v_fixed, 0);
          }
          if (ok && j >= start && j < nt) ok = mbar_wait(p_ready(t), (j - start) & 1);
          if (!ok) {
            atomicExch(p.t.err, 83);
            break;
          }
          tc_fence_after();
          if (j >= start && j < nt) {
            const uint32_t b = v_lo + s * (BOX >> 4);
#pragma unroll
            for (int k = 0; k < TILE / 16; ++k) mma_ts(o, a + k * 8, b + k * (2048 >> 4), hi, id_o, j > start || k > 0);
            tc_commit(o_done(t));
          }
          tc_commit(v_empty(s));
          s = sn;
          ph = phn;
        }
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- rows of the next sequence, at the word of the warps that multiply
      if (fix && wait_long(v_fix, 0, n)) {
        clear_rows(smem_raw + pad + L::V_AT + (n - 1) % L::STAGES * BOX, 1, tail);
        if (lane == 0) mbar_arrive(v_fixed);
      }
    }
  } else {
    regs_up<L::MANY>();
    // ------------------------------------------------------------------ softmax
    const int t = (warp - COMPUTE_WARP) >> 2, row = t * TILE + (warp & 3) * 32 + lane, nt = t == 0 ? n0 : n1;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + t * S_COLS, p_at = tmem + lanes + L::P_AT + t * 64, o_at = tmem + lanes + L::O_AT + t * 64;
    const float scale = p.t.scale_log2;
    const bool here = row < rows;
    Row r;
    bool ok = true;
    const int start = !WIN || t == 0 ? 0 : keys.start;
    Whole whole;
    if constexpr (WIN) whole = whole_keys(p.win, keys, w.r0 + t * TILE, w.len);
    for (int j = start; j < nt; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait_soon(s_full(t), (j - start) & 1));
      if (!ok) break;
      tc_fence_after();
      uint32_t v[TILE];
      load_scores(s_at, v);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read(t));
      auto grow = [&] {
        const float top = max_of<true>(v) * scale;
        if (__any_sync(0xffffffffu, r.grows(top))) {
          const float f = r.grow(top);
          if (j > start) {
            ok = __all_sync(0xffffffffu, mbar_wait(o_done(t), (j - start - 1) & 1));
            if (!ok) return;
            tc_fence_after();
            scale_row(o_at, p.t.DP, f);
          }
        }
      };
      if constexpr (WIN) {
        // (two ways from here on, as above)
        if (whole(j)) {
          apart<false>();
          grow();
          r.weights(v, scale);
        } else {
          apart<true>();
          const uint32_t none = hide_scores(v, SeenKeys(p.win, w.r0 + row, w.len, tile(j) * TILE));
          grow();
          r.weights(v, scale, none);
        }
      } else {
        const int k0 = tile(j) * TILE;
        if (k0 + TILE > w.len || (causal && k0 + TILE - 1 > w.r0 + t * TILE)) hide_scores(v, (causal ? min(w.len, w.r0 + row + 1) : w.len) - k0);
        grow();
        r.weights(v, scale);
      }
      if (!ok) break;
      if (j > start) {
        ok = __all_sync(0xffffffffu, mbar_wait_soon(o_done(t), (j - start - 1) & 1));
        if (!ok) break;
        tc_fence_after();
      }
      store_weights(p_at, v);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready(t));
    }
    if (nt > 0 && ok) ok = __all_sync(0xffffffffu, mbar_wait(o_done(t), (nt - start - 1) & 1));
    if (!ok && lane == 0) atomicExch(p.t.err, 84);
    const long long token = static_cast<long long>(w.b) * p.t.grid.N + w.lo + w.r0 + row;
    __nv_bfloat16* const to = p.o + (token * p.t.grid.H + w.h) * p.t.D;
    if (nt > 0 && ok) {
      tc_fence_after();
      const float total = r.total();
      if (share.part >= 0) {
        const long long at = share.row(p.split, 2 * TILE, row);
        store_part(o_at, p.t.D, p.split.o + at * p.t.D, here);
        if (here) p.split.ml[at] = make_float2(r.m, total);
      } else {
        if constexpr (WIN) {
          __nv_bfloat16* const first = to - static_cast<long long>(lane) * p.t.grid.H * p.t.D;      // (the warp's first row)
          stage_output<128>(o_at, p.t.D, 1.f / total, smem_raw + pad + t * BOX + (warp & 3) * (BOX / 4), first, p.o_rest ? p.o_rest + (first - p.o) : nullptr,
                            1ll * p.t.grid.H * p.t.D, min(rows - row + lane, 32));
        } else {
          store_output(o_at, p.t.D, 1.f / total, to, p.o_rest ? p.o_rest + (to - p.o) : nullptr, here);
        }
        if (here && p.lse) p.lse[(static_cast<long long>(w.b) * p.t.grid.H + w.h) * p.t.grid.N + w.lo + w.r0 + row] = r.m + __log2f(total);
      }
    } else if (here && w.padding) {
      zero_row(p.t.D, to);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<L::COLS>(tmem);
  }
}

// Joins the parts of the pairs of tiles that were split: a warp a row
__global__ void __launch_bounds__(256) attn_join_kernel(FwdParams p) {
  const Split& s = p.split;
  const float* parts_o = s.o;
  const float2* parts_ml = s.ml;
  chain_begin(true, parts_o, parts_ml);
  const int lane = threadIdx.x & 31;
  const uint32_t at = blockIdx.x * 8 + (threadIdx.x >> 5), pair = at / (2 * TILE);
  const int row = static_cast<int>(at % (2 * TILE));
  Work w;
  if (!find_work(p.t.grid, nullptr, s.whole + pair, w) || w.r0 + row >= w.len) return;
  const long long first = static_cast<long long>(pair) * s.parts * (2 * TILE) + row;
  float top = -INFINITY, total = 0.f;
  for (int k = 0; k < s.parts; ++k) top = fmaxf(top, __ldg(&parts_ml[first + k * 2 * TILE].x));
  if (top == -INFINITY) top = 0.f;
  const int c = lane * 4;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < s.parts; ++k) {
    const long long from = first + k * 2 * TILE;
    const float2 ml = __ldg(parts_ml + from);
    const float f = ex2(ml.x - top);
    total = fmaf(ml.y, f, total);
    if (c < p.t.D) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(parts_o + from * p.t.D + c));
      o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
    }
  }
  const long long token = static_cast<long long>(w.b) * p.t.grid.N + w.r0 + row, to = (token * p.t.grid.H + w.h) * p.t.D + c;
  if (c < p.t.D) {
    const float f = 1.f / total;
    o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
    const uint2 h = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
    *reinterpret_cast<uint2*>(p.o + to) = h;
    if (p.o_rest)
      *reinterpret_cast<uint2*>(p.o_rest + to) =
          make_uint2(pack_bf16(o.x - __uint_as_float(h.x << 16), o.y - __uint_as_float(h.x & 0xffff0000u)),
                     pack_bf16(o.z - __uint_as_float(h.y << 16), o.w - __uint_as_float(h.y & 0xffff0000u)));
  }
  if (lane == 0 && p.lse) p.lse[(static_cast<long long>(w.b) * p.t.grid.H + w.h) * p.t.grid.N + w.r0 + row] = top + __log2f(total);
}

// ------------------------------------------------------------------------------------------ backward

// Sixteen computing warps: a thread has a row and 32 columns of a tile of scores and of the products dO V^T, P = 2^(scale S - L) and dS = P (dP - delta)
// of them replace the scores as operands of the next products.  (With eight warps of 64 columns the two warps of a scheduler waited for the same
// things at the same time: 128 x 128 keys by queries of 64 channels in 2645 and 3300 cycles for dQ and dK, dV, where the exponentials take 1024.)
constexpr int BWD_WARPS = 16, BWD_THREADS = 32 * (COMPUTE_WARP + BWD_WARPS), BWD_COLS = 32;
constexpr int BWD_FEW_REGS = 96, BWD_MANY_REGS = 96;
static_assert(BWD_COLS * BWD_WARPS / 4 == TILE && 128 * BWD_FEW_REGS + 512 * BWD_MANY_REGS <= BWD_THREADS * 96);
constexpr int BWD_POLY = 2;      // of eight pairs of exponentials, those on the FMA pipe
// 16 of the 128 rows of the operand that stands in `at`
__device__ __forceinline__ uint32_t operand_cols(uint32_t at, int i) { return at + BWD_COLS * (i >> 1) + 8u * (i & 1); }

// P of 32 columns, from S in v; statistics (-L, -delta) of a row, or of the columns in shared memory.  `seen(c)`: with EDGE, whether column c counts.
template <bool EDGE, typename Neg, typename Seen>
__device__ __forceinline__ void weights_of(uint32_t (&v)[BWD_COLS], f32x2 scale2, Neg neg, Seen seen) {
  apart<EDGE>();
#pragma unroll
  for (int c = 0; c < BWD_COLS; c += 2) {
    float a, b;
    f2_unpack(f2_fma(f2_pack(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, neg(c)), a, b);
    ex2_pair<BWD_POLY>(c / 2, a, b);
    if (EDGE) {
      a = seen(c) ? a : 0.f;
      b = seen(c + 1) ? b : 0.f;
    }
    v[c] = __float_as_uint(a);
    v[c + 1] = __float_as_uint(b);
  }
  // (here, and not where they are used, behind the wait for the products)
  asm volatile("" : MK_RW8(v, 0), MK_RW8(v, 8), MK_RW8(v, 16), MK_RW8(v, 24));
}
template <bool EDGE, typename Neg, typename Seen>
__device__ __forceinline__ void slopes_of(const uint32_t (&v)[BWD_COLS], const uint32_t (&d)[BWD_COLS], uint32_t (&packed)[BWD_COLS / 2], Neg neg, Seen seen) {
#pragma unroll
  for (int c = 0; c < BWD_COLS; c += 2) {
    if (c == 0) apart<EDGE>();
    float a, b;
    f2_unpack(f2_mul(f2_add(f2_pack(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), neg(c)), f2_pack(__uint_as_float(v[c]), __uint_as_float(v[c + 1]))), a,
              b);
    if (EDGE) {      // (what is not seen may be NaN)
      a = seen(c) ? a : 0.f;
      b = seen(c + 1) ? b : 0.f;
    }
    packed[c / 2] = pack_bf16(a, b);
  }
}

// Gradient of the queries.  A CTA has 128 queries of a head and goes over the keys.  S has two buffers, so that the products of the next tile are there when the
// warps come to them.  delta is computed on the way and written for the second kernel (CTAs that share queries write the same).
template <int DB>
struct Dq {
  static constexpr int STAGES = DB == 1 ? 4 : 2, TILE_BYTES = DB * BOX;
  static constexpr int K_AT = 2 * TILE_BYTES, V_AT = K_AT + STAGES * TILE_BYTES, BAR_AT = V_AT + STAGES * TILE_BYTES;
  static constexpr int BARS = 4 * STAGES + 8;
  static constexpr int DELTA_AT = BAR_AT + (8 * BARS + 16 + 15) / 16 * 16, SMEM = DELTA_AT + 4 * TILE + 1024;
  static_assert(SMEM <= SMEM_LIMIT);
};
constexpr uint32_t DQ_DP = 256, DQ_ACC = 384;

struct DqParams {
  TileParams t;
  Parts split;             // over the keys
  float* sums;             // [unit - whole][part][TILE][D]
  const __nv_bfloat16 *o, *o_rest, *d_o;
  const float* lse;
  float* delta;
  AttnTensor dq;
};

// delta of the rows of a tile, eight rows to a computing warp, into shared memory and p.delta.  A row is read by lanes side by side: by the thread that computes on it, a
// warp's load touches 32 lines, and the four threads of a row read it four times: 12000 cycles, a quarter of what a CTA with 13 tiles of keys took.
template <int DB>
__device__ __forceinline__ void row_deltas(const DqParams& p, const Work& w, int rows, int warp, const __nv_bfloat16* out, const __nv_bfloat16* rest,
                                           const __nv_bfloat16* d_out, float* deltas) {
  constexpr int LANES = 8 * DB, AT_ONCE = 32 / LANES, TURNS = TILE / BWD_WARPS / AT_ONCE;
  const int lane = threadIdx.x & 31, c = (lane % LANES) * 8;
  const long long token = static_cast<long long>(w.b) * p.t.grid.N + w.lo + w.r0;
  uint4 u[TURNS], r[TURNS], v[TURNS];
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const int row = warp * (TILE / BWD_WARPS) + i * AT_ONCE + lane / LANES;
    u[i] = r[i] = v[i] = make_uint4(0, 0, 0, 0);
    if (row < rows && c < p.t.D) {
      const long long at = ((token + row) * p.t.grid.H + w.h) * p.t.D + c;
      u[i] = __ldg(reinterpret_cast<const uint4*>(out + at));
      r[i] = __ldg(reinterpret_cast<const uint4*>(rest + at));
      v[i] = __ldg(reinterpret_cast<const uint4*>(d_out + at));
    }
  }
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const uint32_t us[4] = {u[i].x, u[i].y, u[i].z, u[i].w}, rs[4] = {r[i].x, r[i].y, r[i].z, r[i].w}, vs[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    float delta = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      delta = fmaf(__uint_as_float(us[k] << 16) + __uint_as_float(rs[k] << 16), __uint_as_float(vs[k] << 16), delta);
      delta = fmaf(__uint_as_float(us[k] & 0xffff0000u) + __uint_as_float(rs[k] & 0xffff0000u), __uint_as_float(vs[k] & 0xffff0000u), delta);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) delta += __shfl_xor_sync(0xffffffffu, delta, o);
    const int row = warp * (TILE / BWD_WARPS) + i * AT_ONCE + lane / LANES;
    if (row < rows && lane % LANES == 0) {
      deltas[row] = delta;
      p.delta[(static_cast<long long>(w.b) * p.t.grid.H + w.h) * p.t.grid.N + w.lo + w.r0 + row] = delta;
    }
  }
}

template <int DB, bool SPLIT, bool WIN>
__global__ void __launch_bounds__(BWD_THREADS, 1)
attn_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const __grid_constant__ CUtensorMap map_do, const With<DqParams, WIN> p) {
  using L = Dq<DB>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t base = raw_addr + pad, bars = base + L::BAR_AT;
  auto k_full = [&](int s) { return bars + 8u * s; };
  auto k_empty = [&](int s) { return bars + 8u * (L::STAGES + s); };
  auto v_full = [&](int s) { return bars + 8u * (2 * L::STAGES + s); };
  auto v_empty = [&](int s) { return bars + 8u * (3 * L::STAGES + s); };
  const uint32_t q_full = bars + 8u * (4 * L::STAGES), k_fixed = q_full + 8u, dp_full = q_full + 16u, ds_ready = q_full + 24u, dq_full = q_full + 32u;
  auto s_full = [&](int b) { return q_full + 40u + 8u * b; };
  const uint32_t k_fix = q_full + 56u;
  volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_raw + pad + L::BAR_AT + 8 * L::BARS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 4 * L::STAGES; ++s) mbar_init(bars + 8u * s, 1);
    mbar_init(q_full, 1);
    mbar_init(k_fixed, 1);
    mbar_init(k_fix, 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, BWD_WARPS);
    mbar_init(dq_full, 1);
    mbar_init(s_full(0), 1);
    mbar_init(s_full(1), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == 1) tmem_alloc<512>(tmem_slot);
  const int* offsets = p.t.grid.offsets;
  const __nv_bfloat16 *out = p.o, *rest = p.o_rest, *d_out = p.d_o;
  const float* lse = p.lse;
  chain_begin(true, offsets, out, rest, d_out, lse);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  Work w;
  ShareOf<SPLIT> share(p.split, WIN ? place_in_head() : blockIdx.x);
  const bool any = WIN ? find_work_of_head(p.t.grid, offsets, share.unit, w) : find_work(p.t.grid, offsets, share.unit, w);
  const int rows = any ? min(w.len - w.r0, TILE) : 0;
  const bool causal = p.t.causal != 0;
  const KeyTiles keys = window_keys<WIN>(p, w, rows);
  share.along(p.split, WIN ? keys.end[0] : rows == 0 || w.padding ? 0 : (causal ? w.r0 + rows - 1 : w.len - 1) / TILE + 1);
  const int n = share.n, j0 = share.first;
  auto tile = [=](int j) {
    if constexpr (WIN) return keys(j);
    else return j0 + j;
  };
  const int tail = w.len - tile(n - 1) * TILE;
  const bool fix = n > 0 && tail < TILE && w.lo + w.len < p.t.grid.N;

  if (warp < COMPUTE_WARP) {
    regs_down<BWD_FEW_REGS>();
    if (warp == 0) {
      // ---------------------------------------------------------------- tiles
      if (n > 0 && elect_one()) {
        const int hk = w.h / p.t.group;
        mbar_expect_tx(q_full, 2 * L::TILE_BYTES);
        for (int b = 0; b < DB; ++b) {
          tma_load_4d(base + b * BOX, &map_q, q_full, b * 64, w.lo + w.r0, w.h, w.b);
          tma_load_4d(base + L::TILE_BYTES + b * BOX, &map_do, q_full, b * 64, w.lo + w.r0, w.h, w.b);
        }
        int s = 0;
        uint32_t ph = 0;
        for (int j = 0; j < n; ++j) {
          if (!mbar_wait(k_empty(s), ph ^ 1u)) {
            atomicExch(p.t.err, 85);
            break;
          }
          mbar_expect_tx(k_full(s), L::TILE_BYTES);
          for (int b = 0; b < DB; ++b) tma_load_4d(base + L::K_AT + s * L::TILE_BYTES + b * BOX, &map_k, k_full(s), b * 64, w.lo + tile(j) * TILE, hk, w.b);
          if (!mbar_wait(v_empty(s), ph ^ 1u)) {
            atomicExch(p.t.err, 85);
            break;
          }
          mbar_expect_tx(v_full(s), L::TILE_BYTES);
          for (int b = 0; b < DB; ++b) tma_load_4d(base + L::V_AT + s * L::TILE_BYTES + b * BOX, &map_v, v_full(s), b * 64, w.lo + tile(j) * TILE, hk, w.b);
          if (++s == L::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- products
      if (n > 0 && elect_one()) {
        const uint32_t hi = desc_hi(1024);
        const uint32_t q_lo = desc_lo(base, 16), do_lo = desc_lo(base + L::TILE_BYTES, 16), k_lo = desc_lo(base + L::K_AT, 16),
                       v_lo = desc_lo(base + L::V_AT, 16), km_lo = desc_lo(base + L::K_AT, BOX);
        const uint32_t id_s = idesc_n(TILE), id_q = idesc_n(p.t.DP) | B_MN;
        const int ksteps = p.t.DP >> 4;
        auto over_channels = [&](uint32_t d, uint32_t a, uint32_t b) {
          for (int i = 0; i < ksteps; ++i) {
            const uint32_t at = (i >> 2) * (BOX >> 4) + (i & 3) * 2;
            tc_mma<2, 1>(d, a + at, hi, b + at, hi, id_s, i > 0);
          }
        };
        bool ok = mbar_wait(q_full, 0) && mbar_wait(k_full(0), 0);
        if (!ok) atomicExch(p.t.err, 86);
        if (ok) {
          tc_fence_after();
          over_channels(tmem, q_lo, k_lo);
          tc_commit(s_full(0));
        }
        int s = 0;
        uint32_t ph = 0;
        for (int j = 0; j < n && ok; ++j) {
          const int sn = s + 1 == L::STAGES ? 0 : s + 1;
          const uint32_t phn = sn == 0 ? ph ^ 1u : ph;
          const uint32_t at = s * (L::TILE_BYTES >> 4);
          if (!mbar_wait(v_full(s), ph)) {
            atomicExch(p.t.err, 87);
            break;
          }
          tc_fence_after();
          over_channels(tmem + DQ_DP, do_lo, v_lo + at);
          tc_commit(dp_full);
          tc_commit(v_empty(s));
          if (j + 1 < n) {
            // (the other buffer of S has been read: dS of tile j - 1 was ready)
            if (!mbar_wait(k_full(sn), phn)) {
              atomicExch(p.t.err, 87);
              break;
            }
            tc_fence_after();
            over_channels(tmem + ((j + 1) & 1) * S_COLS, q_lo, k_lo + sn * (L::TILE_BYTES >> 4));
            tc_commit(s_full((j + 1) & 1));
          }
          const bool clear = fix && j == n - 1;
          if (clear) mbar_arrive(k_fix);
          ok = (!clear || mbar_wait(k_fixed, 0)) && mbar_wait(ds_ready, j & 1);
          if (!ok) {
            atomicExch(p.t.err, 88);
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < TILE / 16; ++i)
            mma_ts(tmem + DQ_ACC, operand_cols(tmem + DQ_DP, i), km_lo + at + i * (2048 >> 4), hi, id_q, j > 0 || i > 0);
          tc_commit(k_empty(s));
          s = sn;
          ph = phn;
        }
        if (ok) tc_commit(dq_full);
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- keys of the next sequence
      if (fix && wait_long(k_fix, 0, n)) {
        clear_rows(smem_raw + pad + L::K_AT + (n - 1) % L::STAGES * L::TILE_BYTES, DB, tail);
        if (lane == 0) mbar_arrive(k_fixed);
      }
    }
  } else {
    regs_up<BWD_MANY_REGS>();
    // ------------------------------------------------------------------ P and dS
    const int x = (warp - COMPUTE_WARP) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool here = row < rows;
    const long long token = static_cast<long long>(w.b) * p.t.grid.N + w.lo + w.r0 + row;
    const long long stat = (static_cast<long long>(w.b) * p.t.grid.H + w.h) * p.t.grid.N + w.lo + w.r0 + row;
    float l = 0.f, delta = 0.f;
    if (here && n > 0) {
      l = __ldg(lse + stat);
      const long long at = (token * p.t.grid.H + w.h) * p.t.D;
      for (int c = 0; !WIN && c < p.t.D; c += 8) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(out + at + c)), r = __ldg(reinterpret_cast<const uint4*>(rest + at + c)),
                    v = __ldg(reinterpret_cast<const uint4*>(d_out + at + c));
        const uint32_t us[4] = {u.x, u.y, u.z, u.w}, rs[4] = {r.x, r.y, r.z, r.w}, vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          delta = fmaf(__uint_as_float(us[i] << 16) + __uint_as_float(rs[i] << 16), __uint_as_float(vs[i] << 16), delta);
          delta = fmaf(__uint_as_float(us[i] & 0xffff0000u) + __uint_as_float(rs[i] & 0xffff0000u), __uint_as_float(vs[i] & 0xffff0000u), delta);
        }
      }
      if (!WIN && x == 0) p.delta[stat] = delta;
    }
    if constexpr (WIN) {
      float* const deltas = reinterpret_cast<float*>(smem_raw + pad + L::DELTA_AT);
      if (n > 0) row_deltas<DB>(p, w, rows, warp - COMPUTE_WARP, out, rest, d_out, deltas);
      asm volatile("bar.sync 1, %0;" ::"n"(32 * BWD_WARPS) : "memory");
      delta = here ? deltas[row] : 0.f;
    }
    const float scale = p.t.scale_log2;
    const f32x2 scale2 = f2_pack(scale, scale), l2 = f2_pack(-l, -l), delta2 = f2_pack(-delta, -delta);
    Whole whole;
    if constexpr (WIN) whole = whole_keys(p.win, keys, w.r0, w.len);
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait_soon(s_full(j & 1), (j >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      uint32_t v[BWD_COLS];
      const uint32_t s_at = tmem + lanes + (j & 1) * S_COLS + x * BWD_COLS, dp_at = tmem + lanes + DQ_DP + x * BWD_COLS;
      tmem_req32(s_at, v);
      const int k0 = tile(j) * TILE + x * BWD_COLS;
      bool edge = k0 + BWD_COLS > w.len || (causal && k0 + BWD_COLS - 1 > w.r0), none = false;
      const int below = (causal ? min(w.len, w.r0 + row + 1) : w.len) - k0;
      uint32_t bits = 0xffffffffu;
      if constexpr (WIN) {
        edge = !whole(j);
        if (edge) {
          bits = SeenKeys(p.win, w.r0 + row, w.len, k0).bits(0);
          none = !__any_sync(0xffffffffu, bits != 0);
        }
      }
      auto seen = [&](int c) { return WIN ? (bits >> c & 1) != 0 : c < below; };
      tmem_wait32(v);
      if (!WIN || !none) weights_of<false>(v, scale2, [&](int) { return l2; }, seen);
      ok = __all_sync(0xffffffffu, mbar_wait_soon(dp_full, j & 1));
      if (!ok) break;
      tc_fence_after();
      uint32_t d[BWD_COLS], packed[BWD_COLS / 2];
      tmem_req32(dp_at, d);
      tmem_wait32(d);
      if (edge) slopes_of<true>(v, d, packed, [&](int) { return delta2; }, seen);
      else slopes_of<false>(v, d, packed, [&](int) { return delta2; }, seen);
      tmem_st16(dp_at, packed);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_ready);
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(dq_full, 0));
    if (!ok && lane == 0) atomicExch(p.t.err, 89);
    __nv_bfloat16* const to = p.dq.ptr + w.b * p.dq.batch + (w.lo + w.r0 + row) * p.dq.token + w.h * p.dq.head;
    if (n > 0 && ok) {
      tc_fence_after();
      if (SPLIT && share.part >= 0) store_part(tmem + lanes + DQ_ACC, p.t.D, p.sums + share.row(p.split, TILE, row) * p.t.D, here, x * 8, 32);
      else if constexpr (WIN)      // (a row to a thread, each of its stores touches 32 lines a warp)
        stage_rows<4 * DB / 2>(tmem + lanes + DQ_ACC, x * 16 * DB, min(p.t.D, (x + 1) * 16 * DB), p.t.scale, smem_raw + pad + L::K_AT + (warp - COMPUTE_WARP) * 1024 * DB,
                               to - static_cast<long long>(lane) * p.dq.token, p.dq.token, min(rows - row + lane, 32));
      else store_row(tmem + lanes + DQ_ACC, p.t.D, p.t.scale, to, here, x * 16, 64);
    } else if (here && w.padding && x == 0) {
      zero_row(p.t.D, to);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<512>(tmem);
  }
}

// Gradients of keys and values.  A CTA has 128 keys of a head and goes over the queries of all heads that share it, so that nothing is added up
// afterwards but what `key_parts` splits.  Scores are transposed (a thread's row is a key), so that P and dS come out of tensor memory as the first operands of the
// products with dO and Q.  Heads of up to 64 channels: two buffers of S, the next tile's scores run in front of the products that wait for the
// warps; above, tensor memory is full with one, and they run behind the first of these.
template <int DB>
struct Dkv {
  static constexpr int STAGES = DB == 1 ? 3 : 2, TILE_BYTES = DB * BOX, S_BUFS = DB == 1 ? 2 : 1;
  static constexpr int STAGE_AT = 2 * TILE_BYTES, STAGE = 2 * TILE_BYTES, STAT_AT = STAGE_AT + STAGES * STAGE, STAT = 2 * TILE * 4;
  static constexpr int BAR_AT = STAT_AT + STAGES * STAT, BARS = 4 * STAGES + 10;
  static constexpr int SMEM = BAR_AT + 8 * BARS + 16 + 1024;
  static constexpr uint32_t DP_AT = S_BUFS * S_COLS, DV_AT = DP_AT + S_COLS, DK_AT = DV_AT + DB * 64;
  static_assert(SMEM <= SMEM_LIMIT && DK_AT + DB * 64 == 512);
};

// Windows: tiles with sinks are seen by all queries of their sequence, and go apart.  The `first` CTAs of a head have them: (sequence, tile, part) in as many parts,
// along queries and heads, as have two tiles of queries each; they leave sums, by units (sequence, head, tile).  The others have the rest.
struct SinkTiles {
  int parts, tiles;        // parts 0: nothing goes apart
  uint32_t units, first;
  __host__ __device__ int parts_of(int total) const {      // that have something to do
    const int most = total / 2 > 1 ? total / 2 : 1;
    return parts < most ? parts : most;
  }
};
// Queries of `len` that see the keys r0 .. of a tile: tiles of them from `first` on
struct QueryTiles {
  int first, n;
  __device__ __forceinline__ QueryTiles(const Window& p, int r0, int rows, int len) {
    const bool sinks = r0 < p.sinks;
    const int lo = p.causal ? r0 : sinks ? 0 : max(r0 - p.right, 0), key = r0 + rows - 1;
    const int hi = sinks || p.left >= len - 1 - key ? len - 1 : key + p.left;
    first = lo / TILE;
    n = rows > 0 ? hi / TILE + 1 - first : 0;
  }
};
__device__ __forceinline__ bool place_sinks(const Slots& g, const int* offsets, int sequence, int head, int tile, Work& w) {
  w.h = head;
  w.b = offsets ? 0 : sequence;
  w.lo = offsets && sequence > 0 ? clamp_offset(__ldg(offsets + sequence), g.N) : 0;
  w.len = offsets ? max(clamp_offset(__ldg(offsets + sequence + 1), g.N) - w.lo, 0) : g.N;
  w.r0 = tile * TILE;
  w.padding = false;
  return w.r0 < w.len;
}

struct DkvParams {
  TileParams t;
  Parts split;             // over the queries
  float *dk_sums, *dv_sums;
  int heads_q;
  const float *lse, *delta;
  AttnTensor dk, dv;
};
struct DkvWindowParams : DkvParams {
  SinkTiles sinks;
};
template <bool WIN>
using DkvWith = typename std::conditional<WIN, Windowed<DkvWindowParams>, DkvParams>::type;

template <int DB, bool SPLIT, bool WIN>
__global__ void __launch_bounds__(BWD_THREADS, 1)
attn_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ CUtensorMap map_do, const DkvWith<WIN> p) {
  using L = Dkv<DB>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t base = raw_addr + pad, bars = base + L::BAR_AT;
  auto q_full = [&](int s) { return bars + 8u * s; };
  auto do_full = [&](int s) { return bars + 8u * (L::STAGES + s); };
  auto empty = [&](int s) { return bars + 8u * (2 * L::STAGES + s); };
  auto stat_full = [&](int s) { return bars + 8u * (3 * L::STAGES + s); };
  const uint32_t kv_full = bars + 8u * (4 * L::STAGES), fixed = kv_full + 8u, fix_bar = kv_full + 16u, ds_ready = kv_full + 24u,
                 dp_full = kv_full + 32u, acc_full = kv_full + 40u;
  auto s_full = [&](int b) { return kv_full + 48u + 8u * b; };
  // (one for either buffer of S: where the next scores are there early, a warp with little to do may be done with them before others are with these)
  auto p_ready = [&](int b) { return kv_full + 64u + 8u * b; };
  volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_raw + pad + L::BAR_AT + 8 * L::BARS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 4 * L::STAGES; ++s) mbar_init(bars + 8u * s, 1);
    mbar_init(kv_full, 1);
    mbar_init(fixed, 1);
    mbar_init(fix_bar, 1);
    mbar_init(p_ready(0), BWD_WARPS);
    mbar_init(p_ready(1), BWD_WARPS);
    mbar_init(ds_ready, BWD_WARPS);
    mbar_init(dp_full, 1);
    mbar_init(acc_full, 1);
    mbar_init(s_full(0), 1);
    mbar_init(s_full(1), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == 1) tmem_alloc<512>(tmem_slot);
  const int* offsets = p.t.grid.offsets;
  const float *lse = p.lse, *delta = p.delta;
  chain_begin(true, offsets, lse, delta);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  Work w;
  ShareOf<SPLIT> share(p.split, WIN ? place_in_head() : blockIdx.x);
  bool any, apart = false;
  if constexpr (WIN && SPLIT) {
    const uint32_t place = place_in_head();
    apart = place < p.sinks.first;
    if (apart) {
      const uint32_t r = place / p.sinks.parts, sequence = r / p.sinks.tiles, tile = r - sequence * p.sinks.tiles;
      share.unit = (sequence * p.t.grid.H + blockIdx.x) * p.sinks.tiles + tile;
      share.part = static_cast<int>(place - r * p.sinks.parts);
      any = place_sinks(p.t.grid, offsets, static_cast<int>(sequence), static_cast<int>(blockIdx.x), static_cast<int>(tile), w);
    } else {
      share = ShareOf<SPLIT>(p.split, place - p.sinks.first);
      any = find_work_of_head(p.t.grid, offsets, share.unit, w) && !(p.sinks.first > 0 && !w.padding && w.r0 < p.win.sinks);
    }
  } else if constexpr (WIN) {
    any = find_work_of_head(p.t.grid, offsets, share.unit, w);
  } else {
    any = find_work(p.t.grid, offsets, share.unit, w);
  }
  const int rows = any ? min(w.len - w.r0, TILE) : 0;
  const bool causal = p.t.causal != 0;
  // tiles of queries, from the first that sees one of these keys, of one head after the other
  int q_first = causal ? w.r0 / TILE : 0, q_tiles = rows == 0 || w.padding ? 0 : (w.len + TILE - 1) / TILE - q_first;
  if constexpr (WIN) {
    const QueryTiles queries(p.win, w.r0, w.padding ? 0 : rows, w.len);
    q_first = queries.first;
    q_tiles = queries.n;
  }
  if (!apart) share.along(p.split, q_tiles * p.t.group);
  if constexpr (WIN && SPLIT) {
    if (apart) {
      const int total = q_tiles * p.t.group, parts = p.sinks.parts_of(total);
      share.first = share.part < parts ? static_cast<int>(static_cast<long long>(total) * share.part / parts) : 0;
      share.n = share.part < parts ? static_cast<int>(static_cast<long long>(total) * (share.part + 1) / parts) - share.first : 0;
    }
  }
  // first tile of queries and head of this CTA
  const int n = share.n, t0 = q_tiles > 0 ? share.first % q_tiles : 0, g0 = q_tiles > 0 ? share.first / q_tiles : 0, h0 = w.h * p.t.group;
  const int tail = w.len - (q_first + q_tiles - 1) * TILE;
  const bool fix = n > 0 && tail < TILE && w.lo + w.len < p.t.grid.N;

  if (warp < COMPUTE_WARP) {
    regs_down<BWD_FEW_REGS>();
    if (warp == 0) {
      // ---------------------------------------------------------------- tiles
      if (n > 0 && elect_one()) {
        mbar_expect_tx(kv_full, 2 * L::TILE_BYTES);
        for (int b = 0; b < DB; ++b) {
          tma_load_4d(base + b * BOX, &map_k, kv_full, b * 64, w.lo + w.r0, w.h, w.b);
          tma_load_4d(base + L::TILE_BYTES + b * BOX, &map_v, kv_full, b * 64, w.lo + w.r0, w.h, w.b);
        }
        int s = 0, t = t0, g = g0;
        uint32_t ph = 0;
        for (int j = 0; j < n; ++j) {
          if (!mbar_wait(empty(s), ph ^ 1u)) {
            atomicExch(p.t.err, 90);
            break;
          }
          const uint32_t at = base + L::STAGE_AT + s * L::STAGE;
          const int q0 = w.lo + (q_first + t) * TILE;
          mbar_expect_tx(q_full(s), L::TILE_BYTES);
          for (int b = 0; b < DB; ++b) tma_load_4d(at + b * BOX, &map_q, q_full(s), b * 64, q0, h0 + g, w.b);
          mbar_expect_tx(do_full(s), L::TILE_BYTES);
          for (int b = 0; b < DB; ++b) tma_load_4d(at + L::TILE_BYTES + b * BOX, &map_do, do_full(s), b * 64, q0, h0 + g, w.b);
          if (++t == q_tiles) {
            t = 0;
            ++g;
          }
          if (++s == L::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- products
      if (n > 0 && elect_one()) {
        const uint32_t hi = desc_hi(1024);
        const uint32_t k_lo = desc_lo(base, 16), v_lo = desc_lo(base + L::TILE_BYTES, 16), q_lo = desc_lo(base + L::STAGE_AT, 16),
                       qm_lo = desc_lo(base + L::STAGE_AT, BOX);
        const uint32_t id_s = idesc_n(TILE), id_d = idesc_n(p.t.DP) | B_MN;
        constexpr uint32_t DO = L::TILE_BYTES >> 4;
        const int ksteps = p.t.DP >> 4;
        auto over_channels = [&](uint32_t d, uint32_t a, uint32_t b) {
          for (int i = 0; i < ksteps; ++i) {
            const uint32_t at = (i >> 2) * (BOX >> 4) + (i & 3) * 2;
            tc_mma<2, 1>(d, a + at, hi, b + at, hi, id_s, i > 0);
          }
        };
        auto over_queries = [&](uint32_t d, uint32_t a, uint32_t b, uint32_t accum) {
#pragma unroll
          for (int i = 0; i < TILE / 16; ++i) mma_ts(d, operand_cols(a, i), b + i * (2048 >> 4), hi, id_d, accum | (i > 0));
        };
        bool ok = mbar_wait(kv_full, 0) && mbar_wait(q_full(0), 0) && mbar_wait(do_full(0), 0);
        if (!ok) atomicExch(p.t.err, 91);
        if (ok) {
          tc_fence_after();
          over_channels(tmem, k_lo, q_lo);
          tc_commit(s_full(0));
          over_channels(tmem + L::DP_AT, v_lo, q_lo + DO);
          tc_commit(dp_full);
        }
        int s = 0, t = t0, g = g0;
        uint32_t ph = 0;
        for (int j = 0; j < n && ok; ++j) {
          const int sn = s + 1 == L::STAGES ? 0 : s + 1;
          const uint32_t phn = sn == 0 ? ph ^ 1u : ph;
          const uint32_t at = s * (L::STAGE >> 4), atn = sn * (L::STAGE >> 4);
          const int buf = L::S_BUFS == 2 ? j & 1 : 0, bufn = L::S_BUFS == 2 ? (j + 1) & 1 : 0;
          auto next_scores = [&] {
            if (j + 1 == n) return true;
            if (!mbar_wait(q_full(sn), phn)) {
              atomicExch(p.t.err, 91);
              return false;
            }
            tc_fence_after();
            over_channels(tmem + bufn * S_COLS, k_lo, q_lo + atn);
            tc_commit(s_full(bufn));
            return true;
          };
          if (L::S_BUFS == 2) ok = next_scores();
          if (!ok) break;
          const bool clear = fix && t == q_tiles - 1;
          if (clear) mbar_arrive(fix_bar);
          ok = (!clear || mbar_wait(fixed, (g - g0) & 1)) && mbar_wait(p_ready(buf), L::S_BUFS == 2 ? (j >> 1) & 1 : j & 1);
          if (!ok) {
            atomicExch(p.t.err, 92);
            break;
          }
          tc_fence_after();
          over_queries(tmem + L::DV_AT, tmem + buf * S_COLS, qm_lo + at + DO, j > 0);
          if (L::S_BUFS == 1) ok = next_scores();
          if (!ok) break;
          if (!mbar_wait(ds_ready, j & 1)) {
            atomicExch(p.t.err, 92);
            ok = false;
            break;
          }
          tc_fence_after();
          over_queries(tmem + L::DK_AT, tmem + L::DP_AT, qm_lo + at, j > 0);
          tc_commit(empty(s));
          if (j + 1 < n) {
            if (!mbar_wait(do_full(sn), phn)) {
              atomicExch(p.t.err, 91);
              ok = false;
              break;
            }
            tc_fence_after();
            over_channels(tmem + L::DP_AT, v_lo, q_lo + atn + DO);
            tc_commit(dp_full);
          }
          if (++t == q_tiles) {
            t = 0;
            ++g;
          }
          s = sn;
          ph = phn;
        }
        if (ok) tc_commit(acc_full);
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- L and delta of the queries
      int s = 0, t = t0, g = g0;
      uint32_t ph = 0;
      for (int j = 0; j < n; ++j) {
        if (!__all_sync(0xffffffffu, mbar_wait(empty(s), ph ^ 1u))) {
          if (lane == 0) atomicExch(p.t.err, 90);
          break;
        }
        float* const to = reinterpret_cast<float*>(smem_raw + pad + L::STAT_AT + s * L::STAT);
        const int q0 = (q_first + t) * TILE;
        const long long from = (static_cast<long long>(w.b) * p.heads_q + h0 + g) * p.t.grid.N + w.lo + q0;
#pragma unroll
        for (int i = 0; i < TILE; i += 32) {
          const bool in = q0 + i + lane < w.len;
          to[i + lane] = in ? -__ldg(lse + from + i + lane) : 0.f;
          to[TILE + i + lane] = in ? -__ldg(delta + from + i + lane) : 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(stat_full(s));
        if (++t == q_tiles) {
          t = 0;
          ++g;
        }
        if (++s == L::STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
    } else if (fix) {
      // ---------------------------------------------------------------- queries of the next sequence
      // (a part of a tile with sinks may begin in the middle of a head's queries)
      const int before = WIN ? t0 : 0;
      for (int g = 0; g < (before + n) / q_tiles; ++g) {
        if (!wait_long(fix_bar, g & 1, q_tiles)) break;
        clear_rows(smem_raw + pad + L::STAGE_AT + (g * q_tiles + q_tiles - 1 - before) % L::STAGES * L::STAGE, 2 * DB, tail);
        if (lane == 0) mbar_arrive(fixed);
      }
    }
  } else {
    regs_up<BWD_MANY_REGS>();
    // ------------------------------------------------------------------ P and dS, transposed
    const int x = (warp - COMPUTE_WARP) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const bool here = row < rows;
    const f32x2 scale2 = f2_pack(p.t.scale_log2, p.t.scale_log2);
    Whole whole;
    if constexpr (WIN) whole = whole_queries(p.win, w.r0, w.len, q_first);
    bool ok = true;
    int s = 0, t = t0;
    uint32_t ph = 0;
    for (int j = 0; j < n; ++j) {
      const int buf = L::S_BUFS == 2 ? j & 1 : 0;
      ok = __all_sync(0xffffffffu, mbar_wait_soon(stat_full(s), ph) && mbar_wait_soon(s_full(buf), L::S_BUFS == 2 ? (j >> 1) & 1 : j & 1));
      if (!ok) break;
      tc_fence_after();
      const float* const stats = reinterpret_cast<const float*>(smem_raw + pad + L::STAT_AT + s * L::STAT) + x * BWD_COLS;
      const int q0 = (q_first + t) * TILE + x * BWD_COLS;
      // the queries that see this key are the columns from `from` to `to`
      bool edge = q0 + BWD_COLS > w.len || (causal && q0 < w.r0 + TILE - 1);
      int from = causal ? w.r0 + row - q0 : 0, to = w.len - q0;
      uint32_t bits = 0xffffffffu;
      bool none = false;
      if constexpr (WIN) {
        edge = !whole(t);
        if (edge) {
          const int key = w.r0 + row;
          if (key >= p.win.sinks) {
            if (!causal) from = key - p.win.right - q0;
            if (p.win.left < w.len - 1 - key) to = key + p.win.left + 1 - q0;
          }
          bits = low_bits(to) & ~low_bits(from);
          none = !__any_sync(0xffffffffu, bits != 0);
        }
      }
      auto seen = [&](int c) { return WIN ? (bits >> c & 1) != 0 : c >= from && c < to; };
      auto neg_l = [&](int c) { return *reinterpret_cast<const f32x2*>(stats + c); };
      auto neg_delta = [&](int c) { return *reinterpret_cast<const f32x2*>(stats + TILE + c); };
      uint32_t v[BWD_COLS], packed[BWD_COLS / 2];
      const uint32_t s_at = tmem + lanes + buf * S_COLS + x * BWD_COLS, dp_at = tmem + lanes + L::DP_AT + x * BWD_COLS;
      tmem_req32(s_at, v);
      tmem_wait32(v);
      if (WIN && none) {
#pragma unroll
        for (int c = 0; c < BWD_COLS; ++c) v[c] = 0u;
      } else if (edge) {
        weights_of<true>(v, scale2, neg_l, seen);
      } else {
        weights_of<false>(v, scale2, neg_l, seen);
      }
#pragma unroll
      for (int c = 0; c < BWD_COLS; c += 2) packed[c / 2] = pack_bf16(__uint_as_float(v[c]), __uint_as_float(v[c + 1]));
      tmem_st16(s_at, packed);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready(buf));
      ok = __all_sync(0xffffffffu, mbar_wait_soon(dp_full, j & 1));
      if (!ok) break;
      tc_fence_after();
      uint32_t d[BWD_COLS];
      tmem_req32(dp_at, d);
      tmem_wait32(d);
      if (edge) slopes_of<true>(v, d, packed, neg_delta, seen);
      else slopes_of<false>(v, d, packed, neg_delta, seen);
      tmem_st16(dp_at, packed);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_ready);
      if (++t == q_tiles) t = 0;
      if (++s == L::STAGES) {
        s = 0;
        ph ^= 1u;
      }
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0));
    if (!ok && lane == 0) atomicExch(p.t.err, 93);
    // half of the warps store either
    const bool values = x < 2;
    const AttnTensor& d = values ? p.dv : p.dk;
    __nv_bfloat16* const to = d.ptr + w.b * d.batch + (w.lo + w.r0 + row) * d.token + w.h * d.head;
    if (n > 0 && ok) {
      tc_fence_after();
      const uint32_t acc = tmem + lanes + (values ? L::DV_AT : L::DK_AT);
      if (SPLIT && share.part >= 0) {
        long long at;
        if constexpr (WIN) at = apart ? (static_cast<long long>(share.unit) * p.sinks.parts + share.part) * TILE + row : share.row(p.split, TILE, row);
        else at = share.row(p.split, TILE, row);
        store_part(acc, p.t.D, (values ? p.dv_sums : p.dk_sums) + at * p.t.D, here, (x & 1) * 8, 16);
      }
      else if constexpr (WIN)
        stage_rows<4 * DB>(acc, (x & 1) * 32 * DB, min(p.t.D, ((x & 1) + 1) * 32 * DB), values ? 1.f : p.t.scale,
                           smem_raw + pad + L::STAGE_AT + (warp - COMPUTE_WARP) * 2048 * DB, to - static_cast<long long>(lane) * d.token, d.token,
                           min(rows - row + lane, 32));
      else store_row(acc, p.t.D, values ? 1.f : p.t.scale, to, here, (x & 1) * 16, 32);
    } else if (here && w.padding && (x & 1) == 0) {
      zero_row(p.t.D, to);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_free<512>(tmem);
  }
}

// Adds up the parts of the units that were split, times a factor: a warp a row; blockIdx.y chooses among two tensors
struct Sums {
  const float* parts[2];
  AttnTensor out[2];
  float factor[2];
};
__global__ void __launch_bounds__(256) attn_sum_kernel(Slots grid, Parts split, Sums p, int D) {
  const float* parts = p.parts[blockIdx.y];
  const int* offsets = grid.offsets;
  chain_begin(true, parts, offsets);
  const int lane = threadIdx.x & 31, c = lane * 4;
  const uint32_t at = blockIdx.x * 8 + (threadIdx.x >> 5), unit = at / TILE;
  const int row = static_cast<int>(at % TILE);
  Work w;
  if (!find_work(grid, offsets, split.whole + unit, w) || w.padding || w.r0 + row >= w.len || c >= D) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < split.parts; ++k) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(parts + ((static_cast<long long>(unit) * split.parts + k) * TILE + row) * D + c));
    a = make_float4(a.x + v.x, a.y + v.y, a.z + v.z, a.w + v.w);
  }
  const float f = p.factor[blockIdx.y];
  const AttnTensor& o = p.out[blockIdx.y];
  *reinterpret_cast<uint2*>(o.ptr + w.b * o.batch + (w.lo + w.r0 + row) * o.token + w.h * o.head + c) =
      make_uint2(pack_bf16(a.x * f, a.y * f), pack_bf16(a.z * f, a.w * f));
}

// The same for tiles with sinks that went apart
__global__ void __launch_bounds__(256) attn_sink_sum_kernel(TileParams t, Window win, SinkTiles s, Sums p) {
  const float* parts = p.parts[blockIdx.y];
  const int* offsets = t.grid.offsets;
  chain_begin(true, parts, offsets);
  const int lane = threadIdx.x & 31, c = lane * 4;
  const uint32_t at = blockIdx.x * 8 + (threadIdx.x >> 5), unit = at / TILE;
  const int row = static_cast<int>(at % TILE);
  Work w;
  const uint32_t rest = unit / s.tiles, sequence = rest / t.grid.H;
  if (!place_sinks(t.grid, offsets, static_cast<int>(sequence), static_cast<int>(rest - sequence * t.grid.H), static_cast<int>(unit - rest * s.tiles), w) ||
      w.r0 + row >= w.len || c >= t.D)
    return;
  const int n = s.parts_of(QueryTiles(win, w.r0, min(w.len - w.r0, TILE), w.len).n * t.group);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < n; ++k) {
    const float4 v = __ldcg(reinterpret_cast<const float4*>(parts + ((static_cast<long long>(unit) * s.parts + k) * TILE + row) * t.D + c));
    a = make_float4(a.x + v.x, a.y + v.y, a.z + v.z, a.w + v.w);
  }
  const float f = p.factor[blockIdx.y];
  const AttnTensor& o = p.out[blockIdx.y];
  *reinterpret_cast<uint2*>(o.ptr + w.b * o.batch + (w.lo + w.r0 + row) * o.token + w.h * o.head + c) =
      make_uint2(pack_bf16(a.x * f, a.y * f), pack_bf16(a.z * f, a.w * f));
}

// ------------------------------------------------------------------------------------------ host

bool map_of(CUtensorMap* map, const AttnTensor& t, const AttnShape& p, int heads) {
  GemmOperand op;
  op.ptr = t.ptr;
  op.rows = p.N;
  op.mn_major = 0;
  op.ld = t.token;
  op.zs_lo = t.head;
  op.zs_hi = t.batch;
  return make_map(map, op, p.D, 2, heads, p.B, TILE);
}

Slots slots_of(const AttnShape& p, int heads, int rows, int causal_order) {
  Slots g;
  g.B = p.B;
  g.N = p.N;
  g.H = heads;
  g.rows = rows;
  g.order = p.causal ? causal_order : p.window ? 2 : 0;
  g.slots = p.offsets ? p.N / rows + p.sequences + 1 : (p.N + rows - 1) / rows;
  g.offsets = p.offsets;
  g.sequences = p.sequences;
  return g;
}
long long blocks_of(const Slots& g) { return 1ll * g.slots * g.H * g.B; }

bool shape_ok(const AttnShape& p) {
  return p.B > 0 && p.N > 0 && p.H > 0 && p.Hk > 0 && p.H % p.Hk == 0 && p.D > 0 && p.D % 8 == 0 && p.D <= ATTN_WIDTH && p.scale > 0.f &&
         (!p.offsets || (p.B == 1 && p.sequences >= 0)) &&
         (!p.window || (p.left >= 0 && p.left <= p.N && p.right >= 0 && p.right <= p.N && p.sinks >= 0 && p.sinks <= p.N)) && blocks_of(slots_of(p, p.H, TILE, 1)) < (1ll << 31);
}

TileParams tile_params(const AttnShape& p, const Slots& g, int* err) {
  TileParams t;
  t.grid = g;
  t.D = p.D;
  t.DP = (p.D + 15) / 16 * 16;
  t.group = p.H / p.Hk;
  t.causal = p.causal;
  t.scale = p.scale;
  t.scale_log2 = p.scale * LOG2E;
  t.err = err;
  return t;
}

Window window_of(const AttnShape& p) { return {p.causal, p.left, p.causal ? 0 : p.right, p.window ? p.sinks : 0}; }

// One query tile to a CTA, two CTAs to an SM, where sequences are short and CTAs of two tiles would take the SMs more than once.  us, two tiles / one, heads of
// 64 (batch x tokens x heads): 64 x 128 x 8 19.3 / 11.6, 64 x 200 x 8 32.7 / 27.9, 32 x 384 x 8 33.7 / 27.1, 16 x 512 x 8 23.4 / 22.5, 8 x 768 x 8 28.9 / 26.1, 8 x
// 1024 x 8 35.7 / 36.5, 2 x 4096 x 8 104 / 121; fitting at once 16 x 128 x 8 5.4 / 6.2, 16 x 256 x 8 8.7 / 8.5.  Heads of 96: 64 x 128 x 8 23.4 / 16.3, 32 x 384 x 8
// 41.6 / 35.4, 16 x 512 x 8 27.7 / 28.3, 8 x 768 x 8 34.0 / 34.9; packed, 41 sequences of 7001 tokens 52.7 / 45.6.  (Lengths of packed sequences are on the
// device: their mean is known.)
int mean_length(const AttnShape& p) { return p.offsets ? p.N / std::max(1, p.sequences) : p.N; }
// Tiles that one tile sees through a window, a sequence permitting: one at least (with more sequences than tokens the mean length is none)
int window_tiles(const AttnShape& p) {
  const long long span = 1ll * p.left + (p.causal ? 0 : p.right) + TILE;
  return static_cast<int>(std::max<long long>(1, std::min<long long>((span + TILE - 1) / TILE + 1, (mean_length(p) + TILE - 1) / TILE)));
}
// Through a window: up to 17 tiles, where start and end of a CTA are a quarter of it, and where CTAs of two tiles would leave half of the SMs idle.  us by tokens to
// either side, two tiles / one: 16128 tokens, 8 heads of 48 192 58 / 54, 704 115 / 102, 960 143 / 125; of 128 704 150 / 144, 960 180 / 177, 1472 238 / 240, 3008 402 /
// 430; 1 head of 64 300 20.5 / 16.9, 2000 63 / 48, 8000 206 / 160; 4000 tokens, 4 of 64 500 24.2 / 19.5.
constexpr int ONE_TILE_WINDOW = 17;
bool one_tile_pays(const AttnShape& p) {
  const long long blocks = blocks_of(slots_of(p, p.H, 2 * TILE, 1));
  if (p.window) return 2 * blocks <= sm_count() || window_tiles(p) <= ONE_TILE_WINDOW;
  return mean_length(p) <= (p.D <= 64 ? 768 : 448) && blocks > sm_count();
}
// CTAs of one length that would be a last wave of their own, or that are fewer than the SMs, are split over the keys so that they fill them, where that saves more
// than joining them costs: tiles of keys, of some 0.7 us.  us, whole / split: 16200 tokens, 8 heads of 48 720 / 641, 12 of 64 1086 / 955, 8 of 128 943 / 847; 5000
// tokens, 8 heads of 64 124 / 83; 2048 tokens 30.2 / 26.4; 1536 23.8 / 20.2.
// The gradients' tiles of queries and of keys in the same way, over the keys and over the queries; heads of more than 64 from 12 tiles on, for what the parts
// weigh.  us, forward and backward, whole / split: 5000 tokens, 8 heads of 64 365 / 320; 2432 139 / 119; 2048, 4 heads 67.1 / 66.5, 1 head 62 / 49; 1536, 6 heads
// with 2 of keys 84 / 58; 2560, 8 heads of 128 209 / 181; 16200, 12 of 64 (at the power limit) 3787 / 3734.  8 tiles saved, wide heads: 1536 tokens, 4 heads of 128
// 82 / 86, 2 x 1536, 2 of 96 75 / 81.
constexpr int MIN_SAVED = 8, MIN_SAVED_WIDE = 12;
Parts parts_of(const AttnShape& p, const Slots& g, int tiles, int min_saved) {
  if (p.offsets || p.causal || p.window) return {0, 0};      // (not of one length)
  const long long units = blocks_of(g), sms = sm_count(), last = units % sms;
  if (last == 0) return {0, 0};
  const long long parts = std::min<long long>(sms / last, std::max(1, tiles / 4));
  if (parts < 2 || tiles - tiles / parts < min_saved) return {0, 0};
  return {static_cast<uint32_t>(units - last), static_cast<int>(parts)};
}
long long blocks_of(const Slots& g, const Parts& s) {
  const long long units = blocks_of(g);
  return s.parts > 0 ? s.whole + (units - s.whole) * s.parts : units;
}
// rows of the buffers of parts
long long part_rows(const Slots& g, const Parts& s) { return s.parts > 0 ? (blocks_of(g) - s.whole) * s.parts * g.rows : 0; }
int tiles_of(const AttnShape& p) { return (p.N + TILE - 1) / TILE; }
Parts forward_parts(const AttnShape& p) { return one_tile_pays(p) ? Parts{0, 0} : parts_of(p, slots_of(p, p.H, 2 * TILE, 1), tiles_of(p), MIN_SAVED); }
Parts query_parts(const AttnShape& p, const Slots& g) { return parts_of(p, g, tiles_of(p), p.D <= 64 ? MIN_SAVED : MIN_SAVED_WIDE); }
// Where lengths differ: over the heads that share keys, if CTAs are for two thirds of the SMs at most (in all of them, then).  us, forward and backward, causal,
// whole / split, 64 channels: 1024 tokens, 8 heads on 2 78 / 56; 2048, 16 on 4 141 / 106; 2000 in 4 sequences 126 / 104; 1000 in 2, 8 on 1 77 / 47; 128 channels, 2048, 8
// on 2 188 / 117; with more CTAs 4000 in 3, 8 on 4 111 / 120; 9113 in 7, 16 on 4 479 / 501.
Parts key_parts(const AttnShape& p, const Slots& g) {
  const int group = p.H / p.Hk, min_saved = p.D <= 64 ? MIN_SAVED : MIN_SAVED_WIDE;
  if (!p.offsets && !p.causal && !p.window) return parts_of(p, g, tiles_of(p) * group, min_saved);
  const long long units = blocks_of(g), sms = sm_count();
  if (3 * units > 2 * sms) return {0, 0};
  int parts = static_cast<int>(std::min<long long>(group, 3 * sms / units));
  while (group % parts) --parts;
  const int tiles = (p.window ? window_tiles(p) : (mean_length(p) + TILE - 1) / TILE) * group;
  if (parts < 2 || tiles - tiles / parts < min_saved) return {0, 0};
  return {0, parts};
}
// Tiles with sinks have all queries of a sequence where others have a window's: parts of about that length, in two waves at most
SinkTiles sink_tiles(const AttnShape& p) {
  if (!p.window || p.sinks <= 0) return {0, 1, 0, 0};
  const int tiles = (p.sinks + TILE - 1) / TILE, along = tiles_of(p), each = window_tiles(p);
  const long long rows = 1ll * (p.offsets ? p.sequences : p.B) * tiles, units = rows * p.Hk;
  if (units == 0) return {0, 1, 0, 0};
  const long long parts = std::min<long long>((along + each - 1) / each, 2ll * sm_count() / units);
  if (parts < 2) return {0, 1, 0, 0};
  return {static_cast<int>(parts), tiles, static_cast<uint32_t>(units), static_cast<uint32_t>(rows * parts)};
}
long long sink_rows(const SinkTiles& s) { return 1ll * s.units * s.parts * TILE; }

// CTAs along x; through a window heads along x, and behind `first` CTAs each their own along y and, where these are many, z
template <bool WIN>
dim3 grid_of(const Slots& g, const Parts& s, uint32_t first) {
  if (!WIN) return dim3(static_cast<unsigned>(blocks_of(g, s)));
  const long long each = first + 1ll * g.slots * g.B * std::max(1, s.parts), z = (each + 65534) / 65535;
  return dim3(static_cast<unsigned>(g.H), static_cast<unsigned>((each + z - 1) / z), static_cast<unsigned>(z));
}
template <typename Params>
cudaError_t launch(void (*kernel)(CUtensorMap, CUtensorMap, CUtensorMap, Params), std::atomic<uint64_t>& devices, int threads, int smem, const CUtensorMap& q,
                   const CUtensorMap& k, const CUtensorMap& v, const Params& p, cudaStream_t s) {
  const cudaError_t e = allow_shared_memory(devices, reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  return launch_chained(kernel, grid_of<!std::is_same<Params, FwdParams>::value>(p.t.grid, p.split, 0), dim3(threads), smem, s, 1, true, q, k, v, p);
}
template <bool WIN>
cudaError_t launch_fwd(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const With<FwdParams, WIN>& p, bool one_tile, cudaStream_t s) {
  static std::atomic<uint64_t> devices[4];
  if (one_tile) {
    if constexpr (WIN) {
      if (p.t.D <= 64) return launch(attn_fwd_narrow_kernel<1, true>, devices[0], FwdNarrow<1>::THREADS_, FwdNarrow<1>::SMEM, q, k, v, p, s);
    } else {
      if (p.t.D <= 64) return launch(attn_fwd_kernel<1, 1, false>, devices[0], Fwd<1, 1>::THREADS_, Fwd<1, 1>::SMEM, q, k, v, p, s);
    }
    return launch(attn_fwd_kernel<2, 1, WIN>, devices[1], Fwd<2, 1>::THREADS_, Fwd<2, 1>::SMEM, q, k, v, p, s);
  }
  if (p.t.D <= 64) return launch(attn_fwd_narrow_kernel<2, WIN>, devices[2], THREADS, FwdNarrow<2>::SMEM, q, k, v, p, s);
  return launch(attn_fwd_kernel<2, 2, WIN>, devices[3], Fwd<2, 2>::THREADS_, Fwd<2, 2>::SMEM, q, k, v, p, s);
}
template <int DB, bool SPLIT, bool WIN>
cudaError_t launch_dq(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& g, const With<DqParams, WIN>& p, cudaStream_t s) {
  static std::atomic<uint64_t> devices;
  const cudaError_t e = allow_shared_memory(devices, reinterpret_cast<const void*>(&attn_dq_kernel<DB, SPLIT, WIN>), Dq<DB>::SMEM);
  if (e != cudaSuccess) return e;
  return launch_chained(attn_dq_kernel<DB, SPLIT, WIN>, grid_of<WIN>(p.t.grid, p.split, 0), dim3(BWD_THREADS), Dq<DB>::SMEM, s, 1, true, q, k, v, g, p);
}
template <int DB, bool SPLIT, bool WIN>
cudaError_t launch_dkv(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& g, const DkvWith<WIN>& p, cudaStream_t s) {
  static std::atomic<uint64_t> devices;
  const cudaError_t e = allow_shared_memory(devices, reinterpret_cast<const void*>(&attn_dkv_kernel<DB, SPLIT, WIN>), Dkv<DB>::SMEM);
  if (e != cudaSuccess) return e;
  uint32_t first = 0;
  if constexpr (WIN) first = p.sinks.first;
  return launch_chained(attn_dkv_kernel<DB, SPLIT, WIN>, grid_of<WIN>(p.t.grid, p.split, first), dim3(BWD_THREADS), Dkv<DB>::SMEM, s, 1, true, q, k, v, g, p);
}
template <int DB>
cudaError_t launch_dq(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& g, const Windowed<DqParams>& p, bool window,
                      cudaStream_t s) {
  if (window) return launch_dq<DB, false, true>(q, k, v, g, p, s);
  return p.split.parts > 0 ? launch_dq<DB, true, false>(q, k, v, g, p, s) : launch_dq<DB, false, false>(q, k, v, g, p, s);
}
template <int DB>
cudaError_t launch_dkv(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& g, const DkvWith<true>& p, bool window,
                       cudaStream_t s) {
  const bool split = p.split.parts > 0 || p.sinks.parts > 0;
  if (window) return split ? launch_dkv<DB, true, true>(q, k, v, g, p, s) : launch_dkv<DB, false, true>(q, k, v, g, p, s);
  return split ? launch_dkv<DB, true, false>(q, k, v, g, p, s) : launch_dkv<DB, false, false>(q, k, v, g, p, s);
}

}  // namespace

long long attention_scratch(const AttnShape& p) {
  return shape_ok(p) ? part_rows(slots_of(p, p.H, 2 * TILE, 1), forward_parts(p)) * (p.D + 2) : 0;
}

cudaError_t attention_fwd(const AttnShape& p, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, __nv_bfloat16* o, __nv_bfloat16* o_rest,
                          float* lse, float* scratch, int* launches, int* err, cudaStream_t s) {
  if (!shape_ok(p) || ((reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(o_rest) | reinterpret_cast<uintptr_t>(scratch)) & 15) ||
      (o_rest != nullptr) != (lse != nullptr))
    return cudaErrorInvalidValue;
  bind_context(s);
  CUtensorMap mq, mk_, mv;
  if (!map_of(&mq, q, p, p.H) || !map_of(&mk_, k, p, p.Hk) || !map_of(&mv, v, p, p.Hk)) return cudaErrorInvalidValue;
  Windowed<FwdParams> f;
  const bool one_tile = one_tile_pays(p);
  f.t = tile_params(p, slots_of(p, p.H, one_tile ? TILE : 2 * TILE, 1), err);
  static_cast<Parts&>(f.split) = scratch ? forward_parts(p) : Parts{0, 0};
  f.split.o = scratch;
  const long long rows = part_rows(f.t.grid, f.split);
  f.split.ml = reinterpret_cast<float2*>(scratch + rows * p.D);
  f.o = o;
  f.o_rest = o_rest;
  f.lse = lse;
  f.win = window_of(p);
  *launches = 1;
  const cudaError_t e = p.window ? launch_fwd<true>(mq, mk_, mv, f, one_tile, s) : launch_fwd<false>(mq, mk_, mv, f, one_tile, s);
  if (e != cudaSuccess || f.split.parts == 0) return e;
  ++*launches;
  return launch_chained(attn_join_kernel, dim3(static_cast<unsigned>(rows / f.split.parts / 8)), dim3(256), 0, s, 1, true, static_cast<const FwdParams&>(f));
}

long long attention_bwd_scratch(const AttnShape& p) {
  if (!shape_ok(p)) return 0;
  const Slots q = slots_of(p, p.H, TILE, 1), k = slots_of(p, p.Hk, TILE, 2);
  const SinkTiles sinks = sink_tiles(p);
  if (sinks.parts > 0) return 2 * sink_rows(sinks) * p.D;
  return std::max(part_rows(q, query_parts(p, q)), 2 * part_rows(k, key_parts(p, k))) * p.D;
}

cudaError_t attention_bwd(const AttnShape& p, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, const __nv_bfloat16* o,
                          const __nv_bfloat16* o_rest, const __nv_bfloat16* d_o, const float* lse, float* delta, const AttnTensor& dq,
                          const AttnTensor& dk, const AttnTensor& dv, float* scratch, int* launches, int* err, cudaStream_t s) {
  auto off = [](const void* at) { return (reinterpret_cast<uintptr_t>(at) & 15) != 0; };
  auto bad = [&](const AttnTensor& t) { return off(t.ptr) || ((t.token | t.head | t.batch) & 7); };
  if (!shape_ok(p) || off(o) || off(o_rest) || off(d_o) || off(scratch) || bad(dq) || bad(dk) || bad(dv)) return cudaErrorInvalidValue;
  bind_context(s);
  const AttnTensor g{const_cast<__nv_bfloat16*>(d_o), 1ll * p.H * p.D, p.D, 1ll * p.N * p.H * p.D};
  CUtensorMap mq, mk_, mv, mg;
  if (!map_of(&mq, q, p, p.H) || !map_of(&mk_, k, p, p.Hk) || !map_of(&mv, v, p, p.Hk) || !map_of(&mg, g, p, p.H)) return cudaErrorInvalidValue;
  Windowed<DqParams> a;
  a.t = tile_params(p, slots_of(p, p.H, TILE, 1), err);
  a.o = o;
  a.o_rest = o_rest;
  a.d_o = d_o;
  a.lse = lse;
  a.delta = delta;
  a.dq = dq;
  a.win = window_of(p);
  DkvWith<true> b;
  b.t = tile_params(p, slots_of(p, p.Hk, TILE, 2), err);
  b.heads_q = p.H;
  b.lse = lse;
  b.delta = delta;
  b.dk = dk;
  b.dv = dv;
  b.win = a.win;
  a.split = scratch ? query_parts(p, a.t.grid) : Parts{0, 0};
  a.sums = scratch;
  b.sinks = scratch ? sink_tiles(p) : SinkTiles{0, 1, 0, 0};
  b.split = scratch && b.sinks.parts == 0 ? key_parts(p, b.t.grid) : Parts{0, 0};
  const long long rows_q = part_rows(a.t.grid, a.split), rows_k = part_rows(b.t.grid, b.split);
  // (the parts of dQ have been added up where those of dK and dV begin)
  b.dv_sums = scratch;
  b.dk_sums = scratch + (b.sinks.parts > 0 ? sink_rows(b.sinks) : rows_k) * p.D;
  *launches = 1;
  const bool window = p.window != 0;
  cudaError_t e = p.D <= 64 ? launch_dq<1>(mq, mk_, mv, mg, a, window, s) : launch_dq<2>(mq, mk_, mv, mg, a, window, s);
  if (e == cudaSuccess && rows_q > 0) {
    ++*launches;
    const Sums sums{{a.sums, nullptr}, {dq, dq}, {p.scale, 0.f}};
    e = launch_chained(attn_sum_kernel, dim3(static_cast<unsigned>(rows_q / a.split.parts / 8)), dim3(256), 0, s, 1, true, a.t.grid, a.split, sums, p.D);
  }
  if (e != cudaSuccess) return e;
  ++*launches;
  e = p.D <= 64 ? launch_dkv<1>(mq, mk_, mv, mg, b, window, s) : launch_dkv<2>(mq, mk_, mv, mg, b, window, s);
  const Sums sums{{b.dv_sums, b.dk_sums}, {dv, dk}, {1.f, p.scale}};
  if (e == cudaSuccess && b.sinks.parts > 0) {
    ++*launches;
    e = launch_chained(attn_sink_sum_kernel, dim3(static_cast<unsigned>(b.sinks.units * (TILE / 8)), 2), dim3(256), 0, s, 1, true, b.t, b.win, b.sinks, sums);
  }
  if (e == cudaSuccess && rows_k > 0) {
    ++*launches;
    Slots units = b.t.grid;
    if (p.window) units.order = 0;      // (see `find_work_of_head`)
    e = launch_chained(attn_sum_kernel, dim3(static_cast<unsigned>(rows_k / b.split.parts / 8), 2), dim3(256), 0, s, 1, true, units, b.split, sums, p.D);
  }
  return e;
}

}  // namespace mk
