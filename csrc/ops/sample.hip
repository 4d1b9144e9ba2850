// A token for each row of bf16 logits: temperature, top-k, top-p, min-p, from a given random number.
//
// Order the row's tokens by larger logit, then by lower index.  With w_i = exp((l_i - l_max) / T):
//   keep the first k; of these the smallest prefix whose w sum to at least p times theirs; of these the ones with
//   w >= min_p (their probability is at least min_p times the likeliest's); the answer is the first kept token whose
//   running sum of w exceeds u times the sum of the kept.
// Every rule keeps a prefix of the order, so only the multiset of values matters until the last step, and a bf16
// logit has at most 2^16 values: a histogram over all of them, held in 128 KB of LDS, is a counting sort of the row.
// The answer is a rank; the rank is a value and a place among the equal values; a last look at the row finds it.
//
// No exponential is taken for a token.  A thread owns 64 neighbouring values; within them they are equally spaced
// (128 bf16 values share an exponent), so their weights are a geometric series: two exp in 64 bits and 64 products,
// off by 64 * 2^-53 at most.  With the counts and weights before each thread's values in LDS, every rule is a search:
// the thread by two ballots, its 64 values by a scan over a wave's lanes.  All waves make the same searches, so none
// waits for another.  All sums are 64-bit and in one fixed order: the same inputs give the same token.
//
// Bound: the LDS atomics of the count (about 10 cycles for 64 tokens) and the row's way through one CU, twice.  A
// workgroup of 1024 threads takes a row, so up to 256 rows take the time of one.
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

typedef uint16_t bf16_t;

constexpr int NT = 1024, WAVES = NT / 64;
constexpr int BINS = 65536, PER = BINS / NT;      // values of a thread
constexpr int WORDS = BINS / 2;                   // two 16-bit counters a word
constexpr int CHUNK = 32768;                      // tokens after which counters over 32767 are carried out
constexpr int CARRIES = 128;                      // carried counts of 32768: rows of up to CARRIES * CHUNK tokens

// Bins: 0 for the largest value, 65535 for the smallest.  Positive values x (and +NaN first) are bins 0x7fff - x, negative
// ones stand as they are: +inf is bin 0x7f, +0 0x7fff, -0 0x8000 (its count is moved to +0's), -inf 0xff80.
constexpr int BIN_INF = 0x7f, BIN_ZERO = 0x7fff, BIN_MINUS_ZERO = 0x8000, BIN_MINUS_INF = 0xff80;

// two tokens at once
__device__ __forceinline__ uint32_t bins_of(uint32_t x) {
  const uint32_t neg = (x >> 15) & 0x00010001u;
  return x ^ (0x7fff7fffu - ((neg << 15) - neg));
}
__device__ __forceinline__ float value_of(int bin) {
  return __uint_as_float((uint32_t)(bin < 0x8000 ? 0x7fff - bin : bin) << 16);
}

// the row in aligned vectors of 8: vector v holds tokens 8v - lead .. 8v - lead + 7, those outside [0, V) are not ours
struct Row {
  const uint4* at;
  int lead, V, vecs;
  __device__ Row(const bf16_t* p, int V_) : V(V_) {
    lead = (int)(((uintptr_t)p & 15) / 2);
    at = reinterpret_cast<const uint4*>((uintptr_t)p & ~(uintptr_t)15);
    vecs = (V + lead + 7) / 8;
  }
  // bit e: token e of vector v is ours
  __device__ uint32_t ours(int v) const {
    const int lo = max(lead - 8 * v, 0), hi = min(V + lead - 8 * v, 8);
    return (0xffu >> (8 - hi)) & (0xffu << lo);
  }
};
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <class T>
__device__ __forceinline__ T lane_scan(T v) {      // inclusive, over a wave
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(v, o, 64);
    if ((int)(threadIdx.x & 63) >= o) v += y;
  }
  return v;
}

struct Shared {
  double red_d[WAVES];
  int red_i[WAVES];
  int first;                   // the largest value's bin
  int nan;                     // whether there is a NaN, then its lowest index
  int carries, carry[CARRIES + 2];
  int in_wave[WAVES];
  int before_c[NT + 1];        // tokens of the values before each thread's
  double before_w[NT];         // their weight
};

// the last thread whose entry is below x (or equal to it, where `equal`); -1 if none.  The entries ascend.
template <class T>
__device__ __forceinline__ int last_below(const T* a, T x, bool equal) {
  const int lane = threadIdx.x & 63;
  T y = a[lane * (NT / 64)];
  const int seg = __popcll(__ballot(y < x || (equal && y == x))) - 1;
  if (seg < 0) return -1;
  y = a[seg * (NT / 64) + (lane & (NT / 64 - 1))];
  return seg * (NT / 64) + __popcll(__ballot(y < x || (equal && y == x)) & ((1ull << (NT / 64)) - 1)) - 1;
}

__global__ void __launch_bounds__(NT)
sample_kernel(const bf16_t* __restrict__ logits, long long ld, int V, const float* __restrict__ uniform,
              const float* __restrict__ temperature, const int* __restrict__ top_k, const float* __restrict__ top_p,
              const float* __restrict__ min_p, int64_t* __restrict__ tokens, float* __restrict__ probs) {
  extern __shared__ __attribute__((aligned(16))) uint32_t hist[];
  __shared__ Shared sh;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, b = blockIdx.x;
  const Row row(logits + (size_t)b * ld, V);
  float T = temperature != nullptr ? temperature[b] : 1.f;
  int k = top_k != nullptr ? top_k[b] : 0;
  double p = top_p != nullptr ? (double)top_p[b] : 1.0;
  double mp = min_p != nullptr ? (double)min_p[b] : 0.0;
  if (!(T > 0.f)) T = 1.f, k = 1, p = 1.0, mp = 0.0;          // greedy
  const double u = uniform[b] < 0.f ? 0.0 : (double)uniform[b];

  for (int i = t; i < WORDS / 4; i += NT) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  if (t == 0) {
    sh.first = BINS;
    sh.nan = 0;
    sh.carries = 0;
  }
  __syncthreads();

  // ---- count
  for (int v0 = 0; v0 < row.vecs; v0 += CHUNK / 8) {
    if (v0 > 0) {
      __syncthreads();
      for (int i = t; i < WORDS / 4; i += NT) {
        const uint4 x = reinterpret_cast<uint4*>(hist)[i];
        if ((x.x | x.y | x.z | x.w) & 0x80008000u) {
          uint32_t* h = &hist[4 * i];
          for (int j = 0; j < 4; ++j)
            for (int c = 0; c < 2; ++c)
              if (h[j] & (0x8000u << (16 * c))) {
                h[j] -= 0x8000u << (16 * c);
                sh.carry[atomicAdd(&sh.carries, 1)] = 2 * (4 * i + j) + c;
              }
        }
      }
      __syncthreads();
    }
    const int v1 = min(v0 + CHUNK / 8, row.vecs);
    for (int v = v0 + t; v < v1; v += NT) {
      const uint4 x = row.at[v];
      const uint32_t ours = row.ours(v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = bins_of(word_of(x, i)), lo = two & 0xffffu, hi = two >> 16;
        // masked tokens (-inf) are not counted: they may be most of the row, and on one address
        if (lo != (uint32_t)BIN_MINUS_INF && (ours == 0xffu || (ours >> (2 * i) & 1))) atomicAdd(&hist[lo >> 1], (lo & 1) ? 0x10000u : 1u);
        if (hi != (uint32_t)BIN_MINUS_INF && (ours == 0xffu || (ours >> (2 * i + 1) & 1))) atomicAdd(&hist[hi >> 1], (hi & 1) ? 0x10000u : 1u);
      }
    }
  }
  __syncthreads();
  if (t == 0) {
    uint32_t c = (hist[BIN_ZERO >> 1] >> 16) + (hist[BIN_MINUS_ZERO >> 1] & 0xffffu);
    for (int j = 0; j < sh.carries; ++j)
      if (sh.carry[j] == BIN_MINUS_ZERO) sh.carry[j] = BIN_ZERO;
    for (; c > 0xffffu; c -= CHUNK) sh.carry[sh.carries++] = BIN_ZERO;
    hist[BIN_ZERO >> 1] = (hist[BIN_ZERO >> 1] & 0xffffu) | (c << 16);
    hist[BIN_MINUS_ZERO >> 1] &= 0xffff0000u;
  }
  __syncthreads();

  // ---- the weight of each thread's 64 values
  const int ncarry = sh.carries;
  const int bin0 = t * PER;
  uint32_t cnt2[PER / 2];
  int mine = BINS;
  {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < PER / 8; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(hist)[t * (PER / 8) + i];
      cnt2[4 * i] = x.x, cnt2[4 * i + 1] = x.y, cnt2[4 * i + 2] = x.z, cnt2[4 * i + 3] = x.w;
      any |= x.x | x.y | x.z | x.w;
    }
    if (any) {
#pragma unroll
      for (int i = PER / 2 - 1; i >= 0; --i) {
        if (cnt2[i] >> 16) mine = bin0 + 2 * i + 1;
        if (cnt2[i] & 0xffffu) mine = bin0 + 2 * i;
      }
    }
    for (int j = 0; j < ncarry; ++j)
      if (sh.carry[j] / PER == t) mine = min(mine, sh.carry[j]);
    // NaN: before +inf, or behind -inf (which is not counted)
    if (mine < BIN_INF || (mine < BINS && bin0 >= BIN_MINUS_INF)) sh.nan = 1;
  }
  int best = mine;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, 64));
  if (lane == 0 && best < BINS) atomicMin(&sh.first, best);
  __syncthreads();
  const int first = sh.first;
  if (sh.nan || first == BINS) {       // a NaN counts as the maximum; a row without any token gives -1
    const bool some = sh.nan;
    __syncthreads();
    if (t == 0) sh.nan = INT_MAX;
    __syncthreads();
    if (some) {
      for (int v = t; v < row.vecs; v += NT) {
        const uint4 x = row.at[v];
        const uint32_t ours = row.ours(v);
        for (int e = 0; e < 8; ++e)
          if ((ours >> e & 1) && ((word_of(x, e >> 1) >> (16 * (e & 1))) & 0x7fffu) > 0x7f80u) atomicMin(&sh.nan, 8 * v + e - row.lead);
      }
    }
    __syncthreads();
    if (t == 0) {
      tokens[b] = some ? sh.nan : -1;
      probs[b] = some ? NAN : 0.f;
    }
    return;
  }
  const float vmax = value_of(first);
  const double rT = (double)T;
  // exp((value - max) / T); the largest value's is 1 whatever T and the value are
  auto weight = [&](int bin) {
    if (bin == first) return 1.0;
    return isfinite(vmax) ? exp(((double)value_of(bin) - (double)vmax) / rT) : 0.0;
  };
  int C = 0;
  double S = 0.0;
  if (mine < BINS) {
    // from the first value at or below the maximum: w0 * ratio^i.  Neighbours are equally spaced (subnormals too); the
    // thread that holds +inf has no other value to weigh
    const int i0 = max(first - bin0, 0);
    const double ratio = bin0 > BIN_INF ? exp(((double)value_of(bin0 + PER - 1) - (double)value_of(bin0 + PER - 2)) / rT) : 0.0;
    double wt = weight(bin0 + i0);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (int)((cnt2[i >> 1] >> (16 * (i & 1))) & 0xffffu);
      C += c;
      S += (double)c * wt;                       // nothing is counted above the maximum
      if (i >= i0) wt *= ratio;
    }
    for (int j = 0; j < ncarry; ++j)
      if (sh.carry[j] / PER == t) {
        C += CHUNK;
        S += CHUNK * weight(sh.carry[j]);
      }
  }
  {
    const int ci = lane_scan(C);
    const double si = lane_scan(S);
    if (lane == 63) sh.red_i[w] = ci, sh.red_d[w] = si;
    __syncthreads();
    int c0 = 0;
    double s0 = 0.0;
    for (int i = 0; i < w; ++i) {
      c0 += sh.red_i[i];
      s0 += sh.red_d[i];
    }
    // lane 0 starts exactly at the sum of the waves before it, so that the entries ascend
    const int cp = __shfl_up(ci, 1, 64);
    const double sp = __shfl_up(si, 1, 64);
    sh.before_c[t] = c0 + (lane > 0 ? cp : 0);
    sh.before_w[t] = s0 + (lane > 0 ? sp : 0.0);
    if (t == NT - 1) sh.before_c[NT] = c0 + ci;
    __syncthreads();
  }

  // ---- from here on every wave does the same.  A thread's values in a wave's lanes: count, weight, what is before
  auto count_of = [&](int bin) {
    int c = (int)((hist[bin >> 1] >> (16 * (bin & 1))) & 0xffffu);
    for (int j = 0; j < ncarry; ++j) c += sh.carry[j] == bin ? CHUNK : 0;
    return c;
  };
  auto all_lanes = [&](double x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
  };
  // weight of the first n >= 1 tokens in order
  auto weight_to = [&](int n) {
    const int thr = last_below(sh.before_c, n, false), bin = thr * PER + lane;
    const int c = count_of(bin), m = min(max(n - sh.before_c[thr] - (lane_scan(c) - c), 0), c);
    return sh.before_w[thr] + all_lanes(m > 0 ? m * weight(bin) : 0.0);
  };
  const int total = sh.before_c[NT];
  int keep = k > 0 ? min(k, total) : total;
  if (p < 1.0) {
    // tokens that have less than p of the first keep's weight before them
    const double pz = p * weight_to(keep);
    const int thr = last_below(sh.before_w, pz, false);
    int n = 1;
    if (thr >= 0) {
      const int bin = thr * PER + lane, c = count_of(bin);
      const double wt = c > 0 ? weight(bin) : 0.0, cw = c * wt, before = sh.before_w[thr] + (lane_scan(cw) - cw);
      int m = 0;
      if (c > 0 && before < pz) m = wt > 0.0 ? (int)min((double)c, ceil((pz - before) / wt)) : c;
      n = sh.before_c[thr];
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o, 64);
      n += m;
    }
    keep = max(1, min(keep, n));
  }
  if (mp > 0.0) {
    // tokens of a weight of at least min_p: weights fall along the bins, so look at every 1024th, then every 64th of
    // those, then each
    auto heavy = [&](int bin) { return bin <= first || weight(bin) >= mp; };
    const int seg = max(__popcll(__ballot(heavy(lane * (BINS / 64)))) - 1, 0);
    const int sub = max(__popcll(__ballot(lane < BINS / 64 / PER && heavy(seg * (BINS / 64) + lane * PER))) - 1, 0);
    const int thr = seg * (BINS / 64 / PER) + sub;
    int m = heavy(thr * PER + lane) ? count_of(thr * PER + lane) : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o, 64);
    keep = max(1, min(keep, sh.before_c[thr] + m));
  }
  const double z = weight_to(keep), target = u * z;
  int bin = 0, place = 0, in_bin = 0;
  double prob = 0.0;
  {
    // the thread whose weights reach past the target; for u at or past 1 (or a NaN) the last kept token's
    int thr = target < z ? max(last_below(sh.before_w, target, true), 0) : last_below(sh.before_c, keep, false);
    for (;; --thr) {       // a thread without a kept token of any weight only at the ends of rounding: the one before
      const int x = thr * PER + lane, c = count_of(x), ci = lane_scan(c) - c;
      const int m = min(max(keep - sh.before_c[thr] - ci, 0), c);
      const double wt = m > 0 ? weight(x) : 0.0, mw = m * wt, before = sh.before_w[thr] + (lane_scan(mw) - mw);
      const unsigned long long some = __ballot(wt > 0.0), hit = __ballot(wt > 0.0 && before + mw > target);
      if (some == 0 && thr > 0) continue;
      const int who = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
      const int j = hit ? min(max((int)floor((target - before) / wt), 0), m - 1) : m - 1;
      bin = thr * PER + who;
      place = __shfl(j, who, 64);
      in_bin = __shfl(c, who, 64);
      prob = __shfl(wt, who, 64) / z;
      break;
    }
  }

  // ---- the token: number `place` among those of the value, by index
  // a value's tokens are the halves of its bits; of a zero, of its bits without the sign
  const uint32_t want = bin < 0x8000 ? 0x7fffu - bin : bin, pattern = want | (want << 16);
  const uint32_t keepbits = bin == BIN_ZERO ? 0x7fff7fffu : 0xffffffffu;
  auto matches = [&](int v) {
    const uint4 x = row.at[v];
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t d = (word_of(x, i) & keepbits) ^ pattern;
      mask |= ((d & 0xffffu) == 0 ? 1u << (2 * i) : 0) | ((d >> 16) == 0 ? 2u << (2 * i) : 0);
    }
    return mask & row.ours(v);
  };
  if (in_bin == 1) {                             // the only one: whoever meets it
    for (int v = t; v < row.vecs; v += NT) {
      const uint32_t mask = matches(v);
      if (mask) {
        tokens[b] = 8ll * v + (__ffs((int)mask) - 1) - row.lead;
        probs[b] = (float)prob;
      }
    }
    return;
  }
  const int share = (row.vecs + WAVES - 1) / WAVES, v0 = w * share, v1 = min(v0 + share, row.vecs);
  int n = 0;
  for (int v = v0 + lane; v < v1; v += 64) n += __popc(matches(v));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if (lane == 0) sh.in_wave[w] = n;
  __syncthreads();
  for (int i = 0; i < w; ++i) place -= sh.in_wave[i];
  if (place < 0 || place >= n) return;           // not this wave
  for (int vb = v0; vb < v1; vb += 64) {
    const int v = vb + lane;
    const uint32_t mask = v < v1 ? matches(v) : 0;
    const int c = __popc(mask), x = lane_scan(c), all = __shfl(x, 63, 64);
    if (place < all) {
      int left = place - (x - c);
      if (left >= 0 && left < c) {
        uint32_t mk = mask;
        while (left-- > 0) mk &= mk - 1;
        tokens[b] = 8ll * v + (__ffs((int)mk) - 1) - row.lead;
        probs[b] = (float)prob;
      }
      return;
    }
    place -= all;
  }
}

}  // namespace

extern "C" {

int mivgpu_sample(const void* logits, long long ld, int V, int B, const float* uniform, const float* temperature,
                  const int* top_k, const float* top_p, const float* min_p, int64_t* tokens, float* probs,
                  hipStream_t s) {
  if (B <= 0 || V <= 0 || V > CARRIES * CHUNK || (B > 1 && ld < V)) return -1;
  constexpr int lds = WORDS * 4;
  const hipError_t e = hipFuncSetAttribute((const void*)sample_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(sample_kernel, dim3(B), dim3(NT), lds, s, (const bf16_t*)logits, ld, V, uniform, temperature, top_k,
                     top_p, min_p, tokens, probs);
  return (int)hipGetLastError();
}

}  // extern "C"
