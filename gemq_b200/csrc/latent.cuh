// What the latent attention kernels share: 16-bit types, and where the rows of a sequence lie.
#pragma once

#include "ptx.cuh"

namespace gemq {
namespace latent {

constexpr int kRope = 64;  // rotated part of a key
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T> struct Pair;  // two 16-bit numbers in a word
template <> struct Pair<__half> {
  static constexpr int kBf16 = 0;
  static __device__ __forceinline__ float2 f(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static __device__ __forceinline__ uint32_t r(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Pair<__nv_bfloat16> {
  static constexpr int kBf16 = 1;
  static __device__ __forceinline__ float2 f(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }
  static __device__ __forceinline__ uint32_t r(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

inline bool rank_ok(int rank) { return rank >= 128 && rank <= 512 && rank % 128 == 0; }
inline bool page_ok(int page_size) { return page_size == 16 || page_size == 32 || (page_size > 0 && page_size % 64 == 0); }

// A length as the device has it, within its table; one that is not is reported.
__device__ __forceinline__ int clamp_length(int n, int pitch, int page_size, int* err) {
  const long long most = static_cast<long long>(pitch) * page_size;
  if (n >= 0 && n <= most) return n;
  atomicExch(err, GEMQ_LATENT_BAD_LENGTH);
  return n < 0 ? 0 : static_cast<int>(most);
}

// Whether n + 1 offsets rise from 0 to at most `most`.  By one thread of the launch, to report; each use is clamped by itself.
__device__ __forceinline__ bool offsets_ok(const int* v, int n, int most) {
  int last = 0;
  bool ok = v[0] == 0;
  for (int i = 1; i <= n; ++i) {
    ok = ok && v[i] >= last && v[i] <= most;
    last = v[i];
  }
  return ok;
}

// A wait that runs out (about a second) is reported and ends all waits of the CTA.
__device__ __forceinline__ void wait_here(uint32_t bar, uint32_t parity, int* abort, int* err) {
  for (int i = 0; i < (1 << 16); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20000)
        : "memory");
    if (ok || *reinterpret_cast<volatile int*>(abort)) return;
  }
  *reinterpret_cast<volatile int*>(abort) = 1;
  atomicExch(err, GEMQ_LATENT_WAIT);
}
// Out of line where it can be: the waits are many, and a launch that runs for 10 us spends half of its time on instructions that are not in
// the cache yet.  (CALL: not in code that has asked for more registers, where a call cannot be allocated.)
static __device__ __noinline__ void wait_on(uint32_t bar, uint32_t parity, int* abort, int* err) { wait_here(bar, parity, abort, err); }
template <bool CALL = false>
__device__ __forceinline__ void wait_for(unsigned long long* bar, uint32_t parity, int* abort, int* err) {
  if (mbar_test_wait(bar, parity)) return;
  if (CALL) wait_on(smem_u32(bar), parity, abort, err);
  else wait_here(smem_u32(bar), parity, abort, err);
}

// Division of a 32-bit n >= 0 by a number of the launch (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994): with l = ceil(log2 d) the multiplier floor(2^32 (2^l - d) / d) + 1 and 2^32 above it
// give n / d after a shift by l, the sum halved on the way so that it fits.
struct Div {
  uint32_t mul;
  int half, shift;
  __device__ __forceinline__ int operator()(int n) const {
    const uint32_t q = __umulhi(mul, static_cast<uint32_t>(n));
    return static_cast<int>((((static_cast<uint32_t>(n) - q) >> half) + q) >> shift);
  }
};
inline Div div_by(uint32_t d) {  // d > 0
  int l = 0;
  while ((1ull << l) < d) ++l;
  return {static_cast<uint32_t>(((1ull << l) - d) * (1ull << 32) / d + 1), l > 0 ? 1 : 0, l > 0 ? l - 1 : 0};
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two numbers, eight of them: an infinity or a NaN among them.
template <typename T>
__device__ __forceinline__ bool has_nonfinite(uint32_t w) {
  constexpr uint32_t kExp = Pair<T>::kBf16 ? 0x7f80u : 0x7c00u;
  return (w & kExp) == kExp || ((w >> 16) & kExp) == kExp;
}
template <typename T>
__device__ __forceinline__ bool has_nonfinite(uint4 v) {
  return has_nonfinite<T>(v.x) || has_nonfinite<T>(v.y) || has_nonfinite<T>(v.z) || has_nonfinite<T>(v.w);
}
// A map is a launch parameter: its first use finds it in the cache.
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<unsigned long long>(map)) : "memory");
}
// The same in all lanes, and known to be so: what the TMA and MMA instructions take stays in uniform registers.
__device__ __forceinline__ int uniform(int v) { return static_cast<int>(__reduce_or_sync(0xffffffffu, static_cast<unsigned>(v))); }

}  // namespace latent
}  // namespace gemq
