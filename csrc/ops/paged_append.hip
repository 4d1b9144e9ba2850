// QK-norm + RoPE over a ragged batch of tokens, and the append of their K/V to 8-bit pages.
//
//   q, k: y = x * rsqrt(mean(x^2) + eps) * w over each head, then for i < D/2 the pair (y_i, y_{i+D/2}) turned by
//         pos * theta^(-2i/D).  The angle is taken in turns as a 64-bit fixed-point fraction: turns_i =
//         round(2^64 theta^(-2i/D) / 2pi), and pos * turns_i mod 2^64 is the fraction of a turn to within
//         pos * 2^-65, at any position, with three integer products and no 64-bit floats.
//   k, v: codes e4m3(x / s), one scale s = 2^e for K and one for V of each page and head, e the smallest with
//         max |x| <= 448 * 2^e over the page's live tokens (at least EMIN).  A power of two costs e4m3 at most one
//         bit of range at the small end and no precision; when a later token raises it, the older codes are
//         multiplied by 2^(old - new), which is exact but for subnormal codes.
//
// A token-head whose K or V is not finite is stored as NaN in K and zero in V: every query that sees it then gives
// NaN through its score, and a query that does not see it cannot be reached through 0 * NaN in the product with V.
//
// Bound: HBM (the rows once in, q and the codes once out).  Two kinds of workgroups in one launch:
//   * K/V: one for each kv head and run of up to `window` tokens.  It takes every segment (consecutive slots of one
//     page) that starts in its run, whole: the page's scale needs all of the segment's values, which 256 threads hold
//     in registers (64 tokens x D values of K and of V), so nothing is read twice;
//   * q: one for each token; a thread keeps its 8 sines and cosines for all heads.
#include "paged.h"

using namespace paged;

namespace {

constexpr int NT = 256;

template <int D>
struct Head {
  static constexpr int LANES = D / 8;          // lanes of one head row, 8 values each
  static constexpr int ROWS = NT / LANES;      // head rows at once
};

// sines and cosines of the 8 pairs that lane `l` of a head row works on
template <int D>
__device__ __forceinline__ void angles(int pos, const unsigned long long* __restrict__ turns, int l, float* c, float* s) {
  const int i0 = (l * 8) % (D / 2);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned long long f = (unsigned long long)(long long)pos * turns[i0 + e];
    // the fraction's top 32 bits as a signed half-turn count in [-1, 1): off by 2^-25 of a turn at most
    sincospif((float)(int)(unsigned)(f >> 32) * 0x1p-31f, &s[e], &c[e]);
  }
}

// RMS norm and rotation of one head row spread over its lanes
template <int D>
__device__ __forceinline__ void norm_rope(float* x, const float* w, const float* c, const float* s, int l, float eps) {
  constexpr int LANES = Head<D>::LANES;
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor(ss, o, 64);
  const float inv = rsqrtf(ss * (1.f / D) + eps);
  const float sign = l < LANES / 2 ? -1.f : 1.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * w[e];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = __shfl_xor(x[e], LANES / 2, 64);
    x[e] = x[e] * c[e] + sign * (y * s[e]);
  }
}

__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float f) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  return to_codes(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}

// writes the bytes of `w` whose key (4 * first + i) lies in [lo, hi)
__device__ __forceinline__ void store_keys(uint8_t* row, int first, uint32_t w, int lo, int hi) {
  const int k = 4 * first;
  if (k >= lo && k + 4 <= hi) {
    *reinterpret_cast<uint32_t*>(row + k) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k + i >= lo && k + i < hi) row[k + i] = (uint8_t)(w >> (8 * i));
  }
}

template <int D>
__global__ void __launch_bounds__(NT)
append_kernel(const bf16_t* __restrict__ qkv, long long ld, const bf16_t* __restrict__ qw, const bf16_t* __restrict__ kw,
              const int* __restrict__ positions, const int* __restrict__ slots,
              const unsigned long long* __restrict__ turns, bf16_t* __restrict__ q_out, uint8_t* __restrict__ kc,
              uint8_t* __restrict__ vc, float* __restrict__ kscale, float* __restrict__ vscale, int N, int Hq, int Hkv,
              int pages, int window, int nkv, float eps) {
  constexpr int LANES = Head<D>::LANES, ROWS = Head<D>::ROWS, PASS = PAGE / ROWS;
  __shared__ float red[2][NT / 64];
  __shared__ uint32_t vt[D][PAGE / 4 + 1];       // V codes turned: [dim][key], one word of padding against conflicts
  const int t = threadIdx.x, l = t % LANES, g = t / LANES;
  float w[8], c[8], s[8], x[8];

  if ((int)blockIdx.x >= nkv) {                  // ---- q heads of one token
    const int i = blockIdx.x - nkv;
    angles<D>(positions[i], turns, l, c, s);
    unpack8(*reinterpret_cast<const uint4*>(qw + 8 * l), w);
    const bf16_t* row = qkv + (size_t)i * ld;
    for (int h = g; h < (Hq + ROWS - 1) / ROWS * ROWS; h += ROWS) {   // whole waves: the lanes exchange values
      const bool live = h < Hq;
      unpack8(*reinterpret_cast<const uint4*>(row + (size_t)min(h, Hq - 1) * D + 8 * l), x);
      norm_rope<D>(x, w, c, s, l, eps);
      if (live)
        *reinterpret_cast<uint4*>(q_out + ((size_t)i * Hq + h) * D + 8 * l) =
            make_uint4(pack2bf(x[0], x[1]), pack2bf(x[2], x[3]), pack2bf(x[4], x[5]), pack2bf(x[6], x[7]));
    }
    return;
  }

  // ---- K/V of one kv head: the segments that start in tokens [i0, i0 + window)
  const int hk = blockIdx.x % Hkv, i0 = (int)(blockIdx.x / Hkv) * window;
  const int lane = t & 63;
  const long long limit = (long long)pages * PAGE;
  for (int i = i0; i < min(i0 + window, N); ++i) {
    const int slot = slots[i];
    if (slot < 0 || slot >= limit) continue;
    const int off = slot % PAGE;
    if (off != 0 && i > 0 && slots[i - 1] == slot - 1) continue;      // inside a segment
    // its length: tokens whose slots go on in the page
    const bool more = lane + off < PAGE && i + lane < N && slots[min(i + lane, N - 1)] == slot + lane;
    const unsigned long long run = __ballot(more);
    const int cnt = run == ~0ull ? 64 : __ffsll((long long)~run) - 1;
    const size_t ph = (size_t)(slot / PAGE) * Hkv + hk;

    float kf[PASS][8], vf[PASS][8], ka = 0.f, va = 0.f;
    unpack8(*reinterpret_cast<const uint4*>(kw + 8 * l), w);
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      const int j = p * ROWS + g;
      const int tok = i + min(j, cnt - 1);
      const bf16_t* row = qkv + (size_t)tok * ld + ((size_t)Hq + hk) * D + 8 * l;
      unpack8(*reinterpret_cast<const uint4*>(row), kf[p]);
      unpack8(*reinterpret_cast<const uint4*>(row + (size_t)Hkv * D), vf[p]);
      angles<D>(positions[tok], turns, l, c, s);
      norm_rope<D>(kf[p], w, c, s, l, eps);
      float kmax = 0.f, vmax = 0.f;
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        kmax = fmaxf(kmax, fabsf(kf[p][e]));
        vmax = fmaxf(vmax, fabsf(vf[p][e]));
        bad |= !(fabsf(kf[p][e]) < INFINITY) || !(fabsf(vf[p][e]) < INFINITY);
      }
      // any lane of the head row
      const unsigned long long b = __ballot(bad) >> (lane / LANES * LANES) & ((1ull << LANES) - 1);
      if (b != 0) {
        kmax = vmax = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) kf[p][e] = NAN, vf[p][e] = 0.f;
      }
      ka = fmaxf(ka, kmax);
      va = fmaxf(va, vmax);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      ka = fmaxf(ka, __shfl_xor(ka, o, 64));
      va = fmaxf(va, __shfl_xor(va, o, 64));
    }
    if (lane == 0) red[0][t >> 6] = ka, red[1][t >> 6] = va;
    __syncthreads();
    ka = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    va = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
    float ks = exp2i(scale_exp(ka)), vs = exp2i(scale_exp(va));
    float kr = 1.f, vr = 1.f;                    // what the older codes are multiplied by
    if (off > 0) {
      const float ko = kscale[ph], vo = vscale[ph];
      if (ko > ks) ks = ko;
      if (vo > vs) vs = vo;
      kr = ko / ks;
      vr = vo / vs;
    }
    __syncthreads();                             // every thread has the old scales and the maxima
    if (t == 0) kscale[ph] = ks, vscale[ph] = vs;
    const float ki = 1.f / ks, vi = 1.f / vs;    // powers of two: exact
    uint8_t* kp = kc + ph * PAGE * D;
    uint8_t* vp = vc + ph * PAGE * D;
    if (kr != 1.f) {
      for (int x4 = t; x4 < off * (D / 4); x4 += NT) {
        uint32_t* at = reinterpret_cast<uint32_t*>(kp) + x4;
        *at = rescale4(*at, kr);
      }
    }
    if (vr != 1.f) {
      for (int x4 = t; x4 < D * (PAGE / 4); x4 += NT) {
        uint8_t* row = vp + (size_t)(x4 / (PAGE / 4)) * PAGE;
        const int first = x4 % (PAGE / 4);
        if (4 * first < off) store_keys(row, first, rescale4(reinterpret_cast<uint32_t*>(row)[first], vr), 0, off);
      }
    }
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      const int j = p * ROWS + g;
      if (j < cnt) {
        const auto fit = [](float y, float inv) { return fminf(fmaxf(y * inv, -448.f), 448.f); };
        float a[8];
        const bool nan = kf[p][0] != kf[p][0];   // the whole head row or none of it
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = fit(kf[p][e], ki);
        uint2 code = make_uint2(to_codes(a[0], a[1], a[2], a[3]), to_codes(a[4], a[5], a[6], a[7]));
        if (nan) code = make_uint2(CODE_NAN * 0x01010101u, CODE_NAN * 0x01010101u);
        *reinterpret_cast<uint2*>(kp + (size_t)(off + j) * D + 8 * l) = code;
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = fit(vf[p][e], vi);
        const uint32_t lo = to_codes(a[0], a[1], a[2], a[3]), hi = to_codes(a[4], a[5], a[6], a[7]);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          reinterpret_cast<uint8_t*>(vt[8 * l + e])[off + j] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
      }
    }
    __syncthreads();
    for (int x4 = t; x4 < D * (PAGE / 4); x4 += NT) {
      const int dim = x4 / (PAGE / 4), first = x4 % (PAGE / 4);
      if (4 * first + 4 > off && 4 * first < off + cnt)
        store_keys(vp + (size_t)dim * PAGE, first, vt[dim][first], off, off + cnt);
    }
    __syncthreads();                             // vt and red are free for the next segment
  }
}

}  // namespace

extern "C" {

int mivgpu_paged_qk_norm_rope_kv(const void* qkv, long long ld, const void* qw, const void* kw, const int* positions,
                                 const int* slots, const void* turns, void* q_out, void* kc, void* vc, float* kscale,
                                 float* vscale, int N, int Hq, int Hkv, int head_dim, int pages, float eps,
                                 hipStream_t s) {
  if (N < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || pages <= 0 || (long long)pages * PAGE > INT_MAX) return -1;
  if (ld < (long long)(Hq + 2 * Hkv) * head_dim || ld % 8) return -1;
  if (N == 0) return 0;
  // A decode step has a segment for each token: a workgroup for each.  In a long batch most tokens lie inside a
  // segment: runs of 16 keep the workgroups that find nothing few.
  const int window = N <= 1024 ? 1 : 16;
  const long long nkv = (long long)((N + window - 1) / window) * Hkv;
  if (nkv + N > INT_MAX) return -1;
  const dim3 grid((unsigned)(nkv + N));
#define MIVGPU_APPEND(DD)                                                                                            \
  hipLaunchKernelGGL(append_kernel<DD>, grid, dim3(NT), 0, s, (const bf16_t*)qkv, ld, (const bf16_t*)qw,             \
                     (const bf16_t*)kw, positions, slots, (const unsigned long long*)turns, (bf16_t*)q_out,          \
                     (uint8_t*)kc, (uint8_t*)vc, kscale, vscale, N, Hq, Hkv, pages, window, (int)nkv, eps)
  if (head_dim == 128) MIVGPU_APPEND(128);
  else if (head_dim == 64) MIVGPU_APPEND(64);
  else return -1;
#undef MIVGPU_APPEND
  return (int)hipGetLastError();
}

}  // extern "C"
