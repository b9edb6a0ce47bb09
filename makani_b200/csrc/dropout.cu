// Dropout whose mask is a function of a key, the number of the call and the element, and is made again in the backward pass instead of being kept:
//
//   out_i = keep_i x_i / (1 - p) (+ r_i),   keep_i = word_i >= p 2^32
//
// word_i is word i % 4 of the Philox4x32 generator with ten rounds (Salmon, Moraes, Dror and Shaw, 2011): a bijection of a 128-bit counter, here (number of the
// call, i / 4) with 64 bits each, under a 64-bit key.  A round is two 32 x 32 bit products and four exclusive ors.  All 32 bits are compared, so that p is met to
// 2^-32.  An element that is dropped is zero whatever x holds.
//
// What bounds it: in bf16 the products of 32 x 32 bits, 20 for four words.  Counters of 8 x 16200 x 768 elements: the pipe that has them is busy in 72 % of the
// cycles, that of the exclusive ors and comparisons in 53 %, a scheduler issues in 65 %, and of the 11 cycles that a warp takes for an instruction it waits
// 2.9 for a busy pipe and 3.1 for other warps.  16200 x 768 take 16.8 us, memory 7.6: 1519 CTAs are 2.6 waves (four to an SM), and with start and end SMs have nothing to do
// for a quarter of the time.  With fp32 beside it memory: 64800 x 768 with an fp32 residual, forward, 498 MB, of which 443 reach memory and the rest stays in L2,
// in 74.8 us.
#include "dropout.cuh"

#include <type_traits>

#include "launch.cuh"
#include "vec8.cuh"

namespace mk {

namespace {

constexpr int THREADS = 256;
// Vectors a thread from MANY elements on.  us, bf16, 16200 x 768 elements and 64800 x 768 with an fp32 residual: one 19.5, 74.9; two 18.0, 95.8; four 16.7, 74.4;
// eight 20.5, 104.  (4M elements: 8.0, two 7.5; 2M one 5.2.)
constexpr int LONG = 4;
static_assert((LONG & (LONG - 1)) == 0 && (THREADS & (THREADS - 1)) == 0);
constexpr long long MANY = 1ll << 22;

constexpr uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u, W0 = 0x9E3779B9u, W1 = 0xBB67AE85u;
__device__ __forceinline__ uint64_t wide(uint32_t a, uint32_t b) { return static_cast<uint64_t>(a) * b; }
__device__ __forceinline__ uint32_t high(uint64_t v) { return static_cast<uint32_t>(v >> 32); }

// The generator for the blocks i / 4 of a CTA: they differ in their lower 32 bits alone (a CTA's number of them is a power of two), so that one of two products of
// the first round and of the second are the same for all.
struct Generator {
  uint32_t k0, k1, c1, c3a, c1b, high_b;
  __device__ __forceinline__ Generator(uint64_t key, uint64_t number, uint32_t block_high)
      : k0(static_cast<uint32_t>(key)), k1(high(key)), c1(high(number)) {
    const uint64_t p0 = wide(static_cast<uint32_t>(number), M0);
    c3a = static_cast<uint32_t>(p0);
    const uint64_t p1 = wide(high(p0) ^ block_high ^ k1, M1);
    c1b = static_cast<uint32_t>(p1);
    high_b = high(p1);
  }
  __device__ __forceinline__ void words(uint32_t block, uint32_t (&w)[4]) const {
    const uint64_t a = wide(block, M1);                                                // first round
    const uint64_t b = wide(high(a) ^ c1 ^ k0, M0);                                    // second
    uint32_t c0 = high_b ^ static_cast<uint32_t>(a) ^ (k0 + W0), c_1 = c1b, c2 = high(b) ^ c3a ^ (k1 + W1), c3 = static_cast<uint32_t>(b);
#pragma unroll
    for (uint32_t i = 2; i < 10; ++i) {
      const uint64_t p0 = wide(c0, M0), p1 = wide(c2, M1);
      c0 = high(p1) ^ c_1 ^ (k0 + i * W0);
      c_1 = static_cast<uint32_t>(p1);
      c2 = high(p0) ^ c3 ^ (k1 + i * W1);
      c3 = static_cast<uint32_t>(p0);
    }
    w[0] = c0, w[1] = c_1, w[2] = c2, w[3] = c3;
  }
};

// VEC: whole vectors of eight; else one element after the other.  A thread has the eight elements of each of TURNS vectors, a block's width apart, so that the
// keys of the rounds are made once for them; their loads go out together.
template <typename TX, typename TR, typename TO, bool VEC, int TURNS>
__global__ void __launch_bounds__(THREADS) dropout_kernel(DropParams p) {
  constexpr bool ADD = !std::is_void<TR>::value;
  using Res = typename std::conditional<ADD, TR, TX>::type;
  const TX* x = static_cast<const TX*>(p.x);
  const Res* res = static_cast<const Res*>(p.r);
  const int64_t *key_at = p.source.key_at, *offset_at = p.source.offset_at;
  chain_begin(true, x, res, key_at, offset_at);
  const long long begin = static_cast<long long>(blockIdx.x) * (TURNS * THREADS * 8) + threadIdx.x * 8;
  Vec8<TX> a[TURNS];
  Vec8<Res> r[ADD ? TURNS : 1];
  if constexpr (VEC) {
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
      const long long first = begin + t * (THREADS * 8);
      if (first + 8 <= p.n) {
        a[t].load(x + first);
        if constexpr (ADD) r[t].load(res + first);
      }
    }
  }
  const uint64_t key = key_at ? static_cast<uint64_t>(*key_at) : p.source.key;
  const uint64_t number = ((offset_at ? static_cast<uint64_t>(*offset_at) : 0ull) + p.source.more) >> p.source.shift;
  if (begin == 0 && p.source.kept) {
    p.source.kept[0] = static_cast<int64_t>(key);
    p.source.kept[1] = static_cast<int64_t>(number);
  }
  const Generator generator(key, number, static_cast<uint32_t>(static_cast<uint64_t>(begin) >> 34));
#pragma unroll
  for (int t = 0; t < TURNS; ++t) {
    const long long first = begin + t * (THREADS * 8);
    if (first >= p.n) return;
    const bool whole = VEC && first + 8 <= p.n;
    const int count = static_cast<int>(p.n - first < 8 ? p.n - first : 8);
    float v[8], add[8];
    if (whole) {
      a[t].get(v);
      if constexpr (ADD) r[t].get(add);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = i < count ? value_of(x[first + i]) : 0.f;
        if constexpr (ADD) add[i] = i < count ? value_of(res[first + i]) : 0.f;
      }
    }
    const uint32_t block = static_cast<uint32_t>(static_cast<uint64_t>(first) >> 2);
    uint32_t w[2][4];
    generator.words(block, w[0]);
    generator.words(block + 1, w[1]);
    float out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool keep = w[i >> 2][i & 3] > p.last;
      if constexpr (ADD) out[i] = keep ? fmaf(v[i], p.factor, add[i]) : add[i];
      else out[i] = keep ? v[i] * p.factor : 0.f;
    }
    TO* const to = static_cast<TO*>(p.out) + first;
    __nv_bfloat16* const copy = p.copy ? static_cast<__nv_bfloat16*>(p.copy) + first : nullptr;
    if (whole) {
      Vec8<TO> o;
      o.set(out);
      o.store(to);
      if (copy) {
        Vec8<__nv_bfloat16> h;
        h.set(v);
        h.store(copy);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < count) {
          to[i] = rounded<TO>(out[i]);
          if (copy) copy[i] = __float2bfloat16(v[i]);
        }
    }
  }
}

template <typename TX, typename TR, typename TO>
cudaError_t launch(const DropParams& p, bool vec, cudaStream_t s) {
  auto go = [&](auto* kernel, int turns) {
    const long long each = 8ll * THREADS * turns, blocks = (p.n + each - 1) / each;
    if (blocks >= (1ll << 31)) return cudaErrorInvalidValue;
    return launch_chained(kernel, dim3(static_cast<unsigned>(blocks)), dim3(THREADS), 0, s, 1, true, p);
  };
  if (!vec) return go(dropout_kernel<TX, TR, TO, false, 1>, 1);
  return p.n >= MANY ? go(dropout_kernel<TX, TR, TO, true, LONG>, LONG) : go(dropout_kernel<TX, TR, TO, true, 1>, 1);
}

}  // namespace

cudaError_t dropout(const DropParams& p, cudaStream_t s) {
  if (p.n <= 0) return cudaSuccess;
  auto off = [](const void* at) { return (reinterpret_cast<uintptr_t>(at) & 15) != 0; };
  const bool vec = !off(p.x) && !off(p.r) && !off(p.out) && !off(p.copy);
  using H = __nv_bfloat16;
  if (!p.r) {
    if (p.x_f32) return p.out_f32 ? launch<float, void, float>(p, vec, s) : launch<float, void, H>(p, vec, s);
    return p.out_f32 ? cudaErrorInvalidValue : launch<H, void, H>(p, vec, s);
  }
  if (p.out_f32 != (p.x_f32 | p.r_f32)) return cudaErrorInvalidValue;
  if (p.x_f32) return p.r_f32 ? launch<float, float, float>(p, vec, s) : launch<float, H, float>(p, vec, s);
  return p.r_f32 ? launch<H, float, float>(p, vec, s) : launch<H, H, H>(p, vec, s);
}

}  // namespace mk
