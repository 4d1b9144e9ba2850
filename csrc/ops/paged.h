// What the paged 8-bit serving kernels share: the page geometry, e4m3 codes and small wave helpers.
//
// A page holds 64 tokens of one kv head: K as [64 tokens][D] codes, V as [D][64 tokens] codes (so that both
// operands of the attention's matrix instructions are 16-byte loads), one power-of-two scale each for K and V.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace paged {

typedef uint16_t bf16_t;

constexpr int PAGE = 64;
constexpr int MAX_ROWS = 1024;           // requests of one call: every workgroup scans them in registers and LDS
constexpr int EMIN = -110, EMAX = 119;   // exponents of a scale: 2^EMIN * 2^-9 is a normal bf16, 448 * 2^EMAX is finite
constexpr uint8_t CODE_NAN = 0x7f;

__device__ __forceinline__ float bf2f(bf16_t x) { return __uint_as_float(((uint32_t)x) << 16); }

// two floats to bf16, round to nearest even, NaN stays NaN: one instruction
__device__ __forceinline__ uint32_t pack2bf(float a, float b) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
  return __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)a, (__bf16)b});
}

__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
  f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
  f[4] = __uint_as_float(v.z << 16); f[5] = __uint_as_float(v.z & 0xffff0000u);
  f[6] = __uint_as_float(v.w << 16); f[7] = __uint_as_float(v.w & 0xffff0000u);
}

// four floats (|x| <= 448 or NaN) -> four e4m3 codes, round to nearest even
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// the smallest e in [EMIN, EMAX] with amax <= 448 * 2^e (448 = 0.875 * 2^9); amax finite, >= 0
__device__ __forceinline__ int scale_exp(float amax) {
  if (!(amax > 0.f)) return EMIN;
  const uint32_t u = __float_as_uint(amax);
  const int x = (int)(u >> 23) - 126;                  // amax = f * 2^x, f in [0.5, 1) (subnormal amax: below EMIN anyway)
  const int e = x - 9 + ((u & 0x7fffffu) > 0x600000u);  // f > 0.875
  return min(max(e, EMIN), EMAX);
}
// a scale as the append makes them: a power of two, 2^EMIN to 2^EMAX
__device__ __forceinline__ bool is_scale(float s) {
  const uint32_t u = __float_as_uint(s);
  return (u & 0x7fffffu) == 0 && u - ((uint32_t)(EMIN + 127) << 23) <= (uint32_t)(EMAX - EMIN) << 23;
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// inclusive sum over the workgroup's NT threads (a multiple of 64); red: NT / 64 entries of shared memory.
// Ends with every thread past its last read of red.
template <int NT, class T>
__device__ __forceinline__ T block_scan(T v, T* red, T* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  if (lane == 63) red[w] = v;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    if (i < w) before += red[i];
    all += red[i];
  }
  __syncthreads();
  *total = all;
  return v + before;
}

// the first index in [0, n) with a[index] > x (n if none); a ascending
__device__ __forceinline__ int upper_bound(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

}  // namespace paged
