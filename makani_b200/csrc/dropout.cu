// Dropout whose mask is a function of a key, the number of the call and the element, and is made again in the backward pass instead of being kept:
//
//   out_i = keep_i x_i / (1 - p) (+ r_i),   keep_i = word_i >= p 2^32
//
// word_i is word i % 4 of the Philox4x32 generator with ten rounds (Salmon, Moraes, Dror and Shaw, 2011): a bijection of a 128-bit counter, here (number of the
// call, i / 4) with 64 bits each, under a 64-bit key.  A round is two 32 x 32 bit products and four exclusive ors; 40 instructions or so for the words of four
// elements.  All 32 bits are compared, so that p is met to 2^-32.  An element that is dropped is zero whatever x holds.
#include "dropout.cuh"

#include <type_traits>

#include "launch.cuh"
#include "vec8.cuh"

namespace mk {

namespace {

constexpr int THREADS = 256;
constexpr int LONG = 4;                    // vectors a thread from MANY elements on
constexpr long long MANY = 1ll << 22;

__device__ __forceinline__ void philox(uint64_t key, uint64_t number, uint64_t block, uint32_t (&w)[4]) {
  uint32_t c0 = static_cast<uint32_t>(number), c1 = static_cast<uint32_t>(number >> 32), c2 = static_cast<uint32_t>(block),
           c3 = static_cast<uint32_t>(block >> 32), k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u, p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0, w[1] = c1, w[2] = c2, w[3] = c3;
}

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
    const uint64_t block = static_cast<uint64_t>(first) >> 2;
    uint32_t w[2][4];
    philox(key, number, block, w[0]);
    philox(key, number, block + 1, w[1]);
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
