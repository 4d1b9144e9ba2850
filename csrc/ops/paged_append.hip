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
//   * K/V: some for each kv head and window of 256 tokens, which the segments (consecutive slots of one page) that
//     start there are dealt out to.  A segment is taken whole: the page's scale needs all of its values, which 256
//     threads hold in registers (64 tokens x D values of K and of V), so nothing is read twice; one within 16 slots, a
//     decoding request's token above all, is a single wave's, without a barrier.  A thread has 8 dimensions of 4 (D =
//     128) or 2 neighbouring slots, so that its V codes are whole words of V's rows [D][64];
//   * q: waves of one token each; a lane keeps its 8 sines and cosines for the heads that it walks through.
// Sines and cosines are the hardware's, which take turns: off by 2^-22.9 at most over [-1/2, 1/2] (all multiples of
// 2^-22 measured), 40 instructions less than the library's for each of 8 angles.
#include "paged.h"

using namespace paged;

namespace {

constexpr int NT = 256;
constexpr int GROUP = 16;                        // slots of a wave, aligned
// Tokens whose segments are dealt out together, and the fewest workgroups for them
constexpr int WINDOW = 256, EACH = 4, LIST = WINDOW / EACH;

template <int D>
struct Head {
  static constexpr int LANES = D / 8;          // lanes of one head row, 8 values each
  static constexpr int ROWS = NT / LANES;      // head rows at once
};

// The 8 pairs that lane `l` of a head row works on: their angles as fractions of a turn, times 2^64 ...
template <int D>
__device__ __forceinline__ void fractions(int pos, const unsigned long long* __restrict__ turns, int l, unsigned long long* f) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (unsigned long long)(long long)pos * turns[(l * 8) % (D / 2) + e];
}
// ... and their cosines and sines
__device__ __forceinline__ void angles(const unsigned long long* f, float* c, float* s) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    // the fraction's top 32 bits, signed: turns in [-1/2, 1/2), off by 2^-26 at most as a float
    const float x = (float)(int)(unsigned)(f[e] >> 32) * 0x1p-32f;
    s[e] = __builtin_amdgcn_sinf(x);
    c[e] = __builtin_amdgcn_cosf(x);
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

// writes the bytes of `w` whose slot (first + i) lies in [lo, hi); BYTES of them, aligned
template <int BYTES>
__device__ __forceinline__ void store_slots(uint8_t* row, int first, uint32_t w, int lo, int hi) {
  if (first >= lo && first + BYTES <= hi) {
    if (BYTES == 4) *reinterpret_cast<uint32_t*>(row + first) = w;
    else *reinterpret_cast<uint16_t*>(row + first) = (uint16_t)w;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES; ++i)
      if (first + i >= lo && first + i < hi) row[first + i] = (uint8_t)(w >> (8 * i));
  }
}

// One segment (consecutive slots of one page, from token i on) of one kv head: by the whole workgroup, or by one wave
// where it lies in one group of the wave's 16 slots.
template <int D>
struct Append {
  const bf16_t* __restrict__ qkv;
  long long ld;
  const bf16_t* __restrict__ kw;
  const int *__restrict__ positions, *__restrict__ slots;
  const unsigned long long* __restrict__ turns;
  uint8_t *__restrict__ kc, *__restrict__ vc;
  float *__restrict__ kscale, *__restrict__ vscale;
  int N, Hq, Hkv;
  float eps;

  template <bool WAVE>
  __device__ __forceinline__ void segment(int i, int hk, float (*red)[NT / 64]) const {
    constexpr int LANES = Head<D>::LANES, ROWS = Head<D>::ROWS, PASS = PAGE / ROWS;
    static_assert(64 / LANES * PASS == GROUP, "a wave's slots");
    const int t = threadIdx.x, lane = t & 63, l = t % LANES;
    const int slot = slots[i], off = slot % PAGE;
    // its length: tokens whose slots go on in the page
    const bool more = lane + off < PAGE && i + lane < N && slots[min(i + lane, N - 1)] == slot + lane;
    const unsigned long long run = __ballot(more);
    const int cnt = run == ~0ull ? 64 : __ffsll((long long)~run) - 1, end = off + cnt;
    const size_t ph = (size_t)(slot / PAGE) * Hkv + hk;
    const float ko = off > 0 ? kscale[ph] : 0.f, vo = off > 0 ? vscale[ph] : 0.f;
    const int wslot = WAVE ? off & ~(GROUP - 1) : (t & ~63) / LANES * PASS;  // the wave's slots: GROUP from here
    const int slot0 = wslot + lane / LANES * PASS;                           // of the thread's PASS slots

    float w[8], c[8], s[8];
    float kf[PASS][8], ka = 0.f, va = 0.f;
    uint4 vin[PASS];
    unsigned bads = 0;                           // of the thread's slots: not finite
    const bool busy = WAVE || (wslot < end && wslot + GROUP > off);
    if (busy) {
      uint4 kin[PASS];
      int pos[PASS];
#pragma unroll
      for (int p = 0; p < PASS; ++p) {           // slots outside the segment repeat one of its tokens
        const int tok = i + min(max(slot0 + p - off, 0), cnt - 1);
        const bf16_t* row = qkv + (size_t)tok * ld + ((size_t)Hq + hk) * D + 8 * l;
        kin[p] = *reinterpret_cast<const uint4*>(row);
        vin[p] = *reinterpret_cast<const uint4*>(row + (size_t)Hkv * D);
        pos[p] = positions[tok];
      }
      unpack8(*reinterpret_cast<const uint4*>(kw + 8 * l), w);
      unsigned long long f[8];
      fractions<D>(pos[0], turns, l, f);
#pragma unroll
      for (int p = 0; p < PASS; ++p) {
        unpack8(kin[p], kf[p]);
        float vf[8];
        unpack8(vin[p], vf);
        if (p > 0) fractions<D>(pos[p], turns, l, f);
        angles(f, c, s);
        norm_rope<D>(kf[p], w, c, s, l, eps);
        float kmax = 0.f, vmax = 0.f;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          kmax = fmaxf(kmax, fabsf(kf[p][e]));
          vmax = fmaxf(vmax, fabsf(vf[e]));
          bad |= !(fabsf(kf[p][e]) < INFINITY) || !(fabsf(vf[e]) < INFINITY);
        }
        // any lane of the head row
        const unsigned long long b = __ballot(bad) >> (lane / LANES * LANES) & ((1ull << LANES) - 1);
        if (b != 0) {
          kmax = vmax = 0.f;
          bads |= 1u << p;
        }
        ka = fmaxf(ka, kmax);
        va = fmaxf(va, vmax);
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        ka = fmaxf(ka, __shfl_xor(ka, o, 64));
        va = fmaxf(va, __shfl_xor(va, o, 64));
      }
    }
    if (!WAVE) {
      if (lane == 0) red[0][t >> 6] = ka, red[1][t >> 6] = va;
      __syncthreads();                           // and every thread has the old scales
      ka = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
      va = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
    }
    const int me = WAVE ? lane : t, all = WAVE ? 64 : NT;
    float ks = exp2i(scale_exp(ka)), vs = exp2i(scale_exp(va));
    float kr = 1.f, vr = 1.f;                    // what the older codes are multiplied by
    if (off > 0) {
      if (ko > ks) ks = ko;
      if (vo > vs) vs = vo;
      kr = ko / ks;
      vr = vo / vs;
    }
    if (me == 0) kscale[ph] = ks, vscale[ph] = vs;
    const float ki = 1.f / ks, vi = 1.f / vs;    // powers of two: exact
    uint8_t* kp = kc + ph * PAGE * D;
    uint8_t* vp = vc + ph * PAGE * D;
    if (kr != 1.f) {
      for (int x4 = me; x4 < off * (D / 4); x4 += all) {
        uint32_t* at = reinterpret_cast<uint32_t*>(kp) + x4;
        *at = rescale4(*at, kr);
      }
    }
    if (vr != 1.f) {
      for (int x4 = me; x4 < D * (PAGE / 4); x4 += all) {
        uint8_t* row = vp + (size_t)(x4 / (PAGE / 4)) * PAGE;
        const int first = x4 % (PAGE / 4) * 4;
        if (first < off) store_slots<4>(row, first, rescale4(*reinterpret_cast<uint32_t*>(row + first), vr), 0, off);
      }
    }
    if (busy) {
      const auto fit = [](float y, float inv) { return fminf(fmaxf(y * inv, -448.f), 448.f); };
#pragma unroll
      for (int p = 0; p < PASS; ++p) {
        if (slot0 + p < off || slot0 + p >= end) continue;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fit(kf[p][e], ki);
        uint2 code = make_uint2(to_codes(y[0], y[1], y[2], y[3]), to_codes(y[4], y[5], y[6], y[7]));
        if (bads >> p & 1) code = make_uint2(CODE_NAN * 0x01010101u, CODE_NAN * 0x01010101u);
        *reinterpret_cast<uint2*>(kp + (size_t)(slot0 + p) * D + 8 * l) = code;
      }
#pragma unroll
      for (int p = 0; p < PASS; ++p)
        if (bads >> p & 1) vin[p] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        auto code = [&](int p) {
          const uint32_t x = e < 2 ? vin[p].x : e < 4 ? vin[p].y : e < 6 ? vin[p].z : vin[p].w;
          return fit(__uint_as_float((e & 1) ? x & 0xffff0000u : x << 16), vi);
        };
        store_slots<PASS>(vp + (size_t)(8 * l + e) * PAGE, slot0, to_codes(code(0), code(1), code(PASS - 2), code(PASS - 1)), off, end);
      }
    }
    if (!WAVE) __syncthreads();                  // red is free for the next segment
  }
};

template <int D>
__global__ void __launch_bounds__(NT, 3)
append_kernel(const bf16_t* __restrict__ qkv, long long ld, const bf16_t* __restrict__ qw, const bf16_t* __restrict__ kw,
              const int* __restrict__ positions, const int* __restrict__ slots,
              const unsigned long long* __restrict__ turns, bf16_t* __restrict__ q_out, uint8_t* __restrict__ kc,
              uint8_t* __restrict__ vc, float* __restrict__ kscale, float* __restrict__ vscale, int N, int Hq, int Hkv,
              int pages, int each, unsigned share, int spread, float eps) {
  constexpr int LANES = Head<D>::LANES, WROWS = 64 / LANES;
  __shared__ float red[2][NT / 64];
  __shared__ int sums[NT / 64], found[2][LIST];
  const int t = threadIdx.x, lane = t & 63, l = t % LANES;

  // The two kinds take turns, so that the K/V workgroups' latencies lie beside the q workgroups' traffic (8192 tokens: 50
  // us against 76 with the K/V ones first).  kv: K/V workgroups before this one; share: their part of all, times 2^32
  const unsigned me = blockIdx.x;
  const int kv = (int)__umulhi(me, share);
  if ((int)__umulhi(me + 1, share) == kv) {      // ---- q: a wave has every spread-th group of WROWS heads of a token
    const int x = ((int)me - kv) * (NT / 64) + (t >> 6), i = x / spread;
    if (i >= N) return;
    const bf16_t* row = qkv + (size_t)i * ld + 8 * l;
    bf16_t* to = q_out + (size_t)i * Hq * D + 8 * l;
    float w[8], c[8], s[8];
    unpack8(*reinterpret_cast<const uint4*>(qw + 8 * l), w);
    {
      unsigned long long f[8];
      fractions<D>(positions[i], turns, l, f);
      angles(f, c, s);
    }
    constexpr int AHEAD = 4;                     // heads on their way
    const int step = WROWS * spread;
    for (int h0 = x % spread * WROWS + lane / LANES; h0 < Hq + WROWS; h0 += AHEAD * step) {   // whole waves
      uint4 in[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) in[j] = *reinterpret_cast<const uint4*>(row + (size_t)min(h0 + j * step, Hq - 1) * D);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        float y[8];
        unpack8(in[j], y);
        norm_rope<D>(y, w, c, s, l, eps);
        if (h0 + j * step < Hq)
          *reinterpret_cast<uint4*>(to + (size_t)(h0 + j * step) * D) =
              make_uint4(pack2bf(y[0], y[1]), pack2bf(y[2], y[3]), pack2bf(y[4], y[5]), pack2bf(y[6], y[7]));
      }
    }
    return;
  }

  // ---- K/V of one kv head: the window's segments, dealt out to its `each` workgroups, the short ones to their waves.
  // Every workgroup goes through the window's slots: a few KB.
  const int hk = kv % Hkv, mine = kv / Hkv % each, i0 = kv / Hkv / each * WINDOW, n = min(WINDOW, N - i0);
  const long long limit = (long long)pages * PAGE;
  const Append<D> to = {qkv, ld, kw, positions, slots, turns, kc, vc, kscale, vscale, N, Hq, Hkv, eps};
  // 0: token i (slot `slot`, behind `before`) starts no segment; 1: one within a group of a wave's slots; 2: a longer one
  auto ahead = [&](int slot) { return GROUP - (slot & (GROUP - 1)); };
  auto kind = [&](int i, int slot, int before, int next) {
    if (i >= N || slot < 0 || slot >= limit || (slot % PAGE != 0 && i > 0 && before == slot - 1)) return 0;
    const int left = ahead(slot);
    return slot % PAGE + left < PAGE && i + left < N && next == slot + left ? 2 : 1;
  };
  if (n <= each) {                               // a token each
    const int i = i0 + mine;
    if (mine >= n) return;                       // the next window's, or none
    const int slot = slots[i], k = kind(i, slot, slots[max(i - 1, 0)], slots[min(i + ahead(slot), N - 1)]);
    if (k == 2) to.template segment<false>(i, hk, red);
    if (k == 1 && t < 64) to.template segment<true>(i, hk, red);
    return;
  }
  // A thread for each token.  Both kinds' numbers in one word
  static_assert(WINDOW == NT, "a token a thread");
  int k = 0;
  {
    const int i = min(i0 + t, N - 1), slot = slots[i], before = slots[max(i - 1, 0)];
    if (t < n) k = kind(i, slot, before, slots[min(i + ahead(slot), N - 1)]);
  }
  const int one = k == 1 ? 1 : k == 2 ? 1 << 16 : 0;
  int all;
  const int at = block_scan<NT>(one, sums, &all) - one, no = k == 1 ? at & 0xffff : at >> 16;
  if (k != 0 && no % each == mine) found[k - 1][no / each] = i0 + t;
  __syncthreads();
  const int shorts = all & 0xffff, longs = all >> 16;
  for (int x = 0; x * each + mine < longs; ++x)
    to.template segment<false>(__builtin_amdgcn_readfirstlane(found[1][x]), hk, red);
  for (int x = t >> 6; x * each + mine < shorts; x += NT / 64)
    to.template segment<true>(__builtin_amdgcn_readfirstlane(found[0][x]), hk, red);
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
  // Segments: up to one a token in a decode step, one for 64 in a prompt, and any mixture.  Few tokens have a workgroup
  // each, more are dealt out to about 1024 (768 are resident): 1024 decoding requests 30 us, 8192 tokens of a prompt 39,
  // 4000 beside 1000 decoding requests 57 (the same buffers again and again).  With a run of 1, 16 or 64 tokens a
  // workgroup, its segments one by one, the first take 65, 80 and 284, the second 88, 47 and 39, the third 104, 84 and
  // 300; with windows of 8192 tokens 32, 59 and 58.
  const int windows = (N + WINDOW - 1) / WINDOW, resident = (1024 + windows * Hkv - 1) / (windows * Hkv);
  const int most = resident < EACH ? EACH : resident > WINDOW ? WINDOW : resident, each = N < most ? N : most;
  const long long nkv = (long long)windows * each * Hkv;
  // q: from 1024 tokens on there are waves enough, fewer spread their heads over two (8 tokens 6.4 us against 6.8, 512 of
  // a prompt 9.0 against 9.9; but 4096 25.8 against 24.5, and over four waves 29)
  const int groups = (Hq * head_dim / 8 + 63) / 64;
  const int spread = N >= 1024 || groups < 2 ? 1 : 2;
  const long long nq = ((long long)N * spread + NT / 64 - 1) / (NT / 64);
  if (nkv + nq > INT_MAX || (long long)N * spread > INT_MAX) return -1;
  const dim3 grid((unsigned)(nkv + nq));
  // rounded up: share * all >> 32 is nkv, and one more K/V workgroup at most from one workgroup to the next (nq > 0)
  const unsigned share = (unsigned)((((unsigned long long)nkv << 32) + (nkv + nq) - 1) / (nkv + nq));
#define MIVGPU_APPEND(DD)                                                                                            \
  hipLaunchKernelGGL(append_kernel<DD>, grid, dim3(NT), 0, s, (const bf16_t*)qkv, ld, (const bf16_t*)qw,             \
                     (const bf16_t*)kw, positions, slots, (const unsigned long long*)turns, (bf16_t*)q_out,          \
                     (uint8_t*)kc, (uint8_t*)vc, kscale, vscale, N, Hq, Hkv, pages, each, share, spread, eps)
  if (head_dim == 128) MIVGPU_APPEND(128);
  else if (head_dim == 64) MIVGPU_APPEND(64);
  else return -1;
#undef MIVGPU_APPEND
  return (int)hipGetLastError();
}

}  // extern "C"
