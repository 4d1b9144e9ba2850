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
// off by 64 * 2^-53 at most.  All sums are 64-bit and in one fixed order: the same inputs give the same token.
//
// Bound: HBM for many rows (2 bytes a token), the row's way through one CU for few.  A workgroup of 1024 threads
// takes a row.
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

typedef uint16_t bf16_t;

constexpr int NT = 1024, WAVES = NT / 64;
constexpr int BINS = 65536, PER = BINS / NT;      // values of a thread
constexpr int WORDS = BINS / 2;                   // two 16-bit counters a word
constexpr int CHUNK = 32768;                      // tokens after which counters over 32767 are carried out
constexpr int CARRIES = 128;                      // carried counts of 32768: rows of up to CARRIES * CHUNK tokens

// 0 for the largest value (all NaN first), 65535 for the smallest; -0 and +0 alike
__device__ __forceinline__ uint32_t bin_of(uint32_t x) {
  if (x == 0x8000u) x = 0;
  return 0xffffu - ((x & 0x8000u) ? (~x & 0xffffu) : (x | 0x8000u));
}
__device__ __forceinline__ float value_of(int bin) {
  const uint32_t o = 0xffffu - (uint32_t)bin;
  return __uint_as_float(((o & 0x8000u) ? (o & 0x7fffu) : (~o & 0xffffu)) << 16);
}
constexpr int BIN_INF = 0xffff - 0xff80;          // of +inf; the bins before it are NaN

// the row in aligned vectors of 8: vector v holds tokens 8v - lead .. 8v - lead + 7, those outside [0, V) are not ours
struct Row {
  const uint4* at;
  int lead, V, vecs;
  __device__ Row(const bf16_t* p, int V_) : V(V_) {
    lead = (int)(((uintptr_t)p & 15) / 2);
    at = reinterpret_cast<const uint4*>((uintptr_t)p & ~(uintptr_t)15);
    vecs = (V + lead + 7) / 8;
  }
};
__device__ __forceinline__ uint32_t half_of(const uint4& v, int e) {
  const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
  return (e & 1) ? w >> 16 : w & 0xffffu;
}

// exclusive sums over the workgroup
template <class T>
__device__ __forceinline__ T scan_before(T v, T* red, T* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  T x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) red[w] = x;
  __syncthreads();
  T before = 0, all = 0;
  for (int i = 0; i < WAVES; ++i) {
    if (i < w) before += red[i];
    all += red[i];
  }
  __syncthreads();
  *total = all;
  // lane 0 starts exactly at the sum of the waves before it
  const T mine = __shfl_up(x, 1, 64);
  return before + (lane > 0 ? mine : 0);
}

struct Shared {
  double red_d[WAVES];
  int red_i[WAVES];
  int first;                   // the largest value's bin
  int nan;                     // lowest index of a NaN
  int carries, carry[CARRIES];
  int rank_p, rank_m, rank, last;
  double zk, z;
  int bin, place;              // the answer: a value and which of its tokens
  double prob;
  int in_wave[WAVES];
};

__global__ void __launch_bounds__(NT)
sample_kernel(const bf16_t* __restrict__ logits, long long ld, int V, const float* __restrict__ uniform,
              const float* __restrict__ temperature, const int* __restrict__ top_k, const float* __restrict__ top_p,
              const float* __restrict__ min_p, int64_t* __restrict__ tokens, float* __restrict__ probs) {
  extern __shared__ __attribute__((aligned(16))) uint32_t hist[];
  __shared__ Shared sh;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, b = blockIdx.x;
  const Row row(logits + (size_t)b * ld, V);

  for (int i = t; i < WORDS / 4; i += NT) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
  if (t == 0) {
    sh.first = BINS;
    sh.nan = INT_MAX;
    sh.carries = 0;
    sh.rank_p = sh.rank_m = sh.rank = INT_MAX;
    sh.last = -1;
    sh.bin = -1;
  }
  __syncthreads();

  // ---- count
  for (int v0 = 0; v0 < row.vecs; v0 += CHUNK / 8) {
    if (v0 > 0) {
      __syncthreads();
      for (int i = t; i < WORDS / 4; i += NT) {
        uint4 x = reinterpret_cast<uint4*>(hist)[i];
        if ((x.x | x.y | x.z | x.w) & 0x80008000u) {
          uint32_t* h = &hist[4 * i];
          for (int j = 0; j < 4; ++j)
            for (int k = 0; k < 2; ++k)
              if (h[j] & (0x8000u << (16 * k))) {
                h[j] -= 0x8000u << (16 * k);
                sh.carry[atomicAdd(&sh.carries, 1)] = 2 * (4 * i + j) + k;
              }
        }
      }
      __syncthreads();
    }
    const int v1 = min(v0 + CHUNK / 8, row.vecs);
    for (int v = v0 + t; v < v1; v += NT) {
      const uint4 x = row.at[v];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = 8 * v + e - row.lead;
        const uint32_t y = half_of(x, e);
        if (i < 0 || i >= V || y == 0xff80u) continue;        // -inf: a masked token
        if ((y & 0x7fffu) > 0x7f80u) {
          atomicMin(&sh.nan, i);
          continue;
        }
        const uint32_t bin = bin_of(y);
        atomicAdd(&hist[bin >> 1], 1u << (16 * (bin & 1)));
      }
    }
  }
  __syncthreads();

  // ---- a thread's 64 values
  uint32_t cnt2[PER / 2];
#pragma unroll
  for (int i = 0; i < PER / 8; ++i) {
    const uint4 x = reinterpret_cast<const uint4*>(hist)[t * (PER / 8) + i];
    cnt2[4 * i] = x.x, cnt2[4 * i + 1] = x.y, cnt2[4 * i + 2] = x.z, cnt2[4 * i + 3] = x.w;
  }
  auto count = [&](int i) {      // of value t * PER + i
    int c = (int)((cnt2[i >> 1] >> (16 * (i & 1))) & 0xffffu);
    return c;
  };
  const int ncarry = sh.carries;
  auto carried = [&](int bin) {  // rare
    int c = 0;
    for (int j = 0; j < ncarry; ++j) c += sh.carry[j] == bin ? CHUNK : 0;
    return c;
  };
  auto full = [&](int i) { return count(i) + (ncarry ? carried(t * PER + i) : 0); };

  int mine = BINS;
#pragma unroll
  for (int i = PER - 1; i >= 0; --i)
    if (count(i)) mine = t * PER + i;
  for (int j = 0; j < ncarry; ++j)
    if (sh.carry[j] / PER == t) mine = min(mine, sh.carry[j]);
  if (mine < BINS) atomicMin(&sh.first, mine);
  __syncthreads();
  const int first = sh.first;
  const int nan = sh.nan;
  if (nan < V || first == BINS) {      // a NaN counts as the maximum; a row without any token gives -1
    if (t == 0) {
      tokens[b] = nan < V ? nan : -1;
      probs[b] = nan < V ? NAN : 0.f;
    }
    return;
  }
  const float vmax = value_of(first);
  float T = temperature != nullptr ? temperature[b] : 1.f;
  int k = top_k != nullptr ? top_k[b] : 0;
  double p = top_p != nullptr ? (double)top_p[b] : 1.0;
  double mp = min_p != nullptr ? (double)min_p[b] : 0.0;
  if (!(T > 0.f)) T = 1.f, k = 1, p = 1.0, mp = 0.0;          // greedy
  const double u = (double)uniform[b];

  // weights of the thread's values from its first one at or below the maximum: w0 * ratio^i
  const int i0 = min(max(first - t * PER, 0), PER);
  double w0 = 0.0, ratio = 0.0;
  if (mine < BINS) {
    const int bin0 = t * PER + i0;
    if (bin0 == first) w0 = 1.0;
    else if (isfinite(vmax)) w0 = exp(((double)value_of(bin0) - (double)vmax) / (double)T);
    // two neighbours inside the thread's values (a subnormal step is one too); the thread that holds +inf has no
    // other finite value
    const int lo = t * PER + PER - 1;
    if (t * PER > BIN_INF) ratio = exp(((double)value_of(lo) - (double)value_of(lo - 1)) / (double)T);
  }
  int C = 0;
  double S = 0.0;
  {
    double wt = w0;
    for (int i = i0; i < PER; ++i) {
      const int c = full(i);
      C += c;
      S += c * wt;
      wt *= ratio;
    }
  }
  int ctotal;
  double stotal;
  const int c0 = scan_before(C, sh.red_i, &ctotal);
  const double s0 = scan_before(S, sh.red_d, &stotal);
  const int kk = k > 0 ? min(k, ctotal) : ctotal;

  // weight of the first `n` tokens in order, known to the thread that holds token n - 1
  auto weight_to = [&](int n, double* to) {
    if (n > c0 && n <= c0 + C) {
      int left = n - c0;
      double x = s0, wt = w0;
      for (int i = i0; i < PER && left > 0; ++i) {
        const int c = min(full(i), left);
        x += c * wt;
        left -= c;
        wt *= ratio;
      }
      *to = x;
    }
  };
  weight_to(kk, &sh.zk);
  __syncthreads();
  const double pz = p * sh.zk;
  if (C > 0) {
    // how many tokens have less than p of the mass before them, and how many a weight of at least min_p
    int np = INT_MAX, nm = INT_MAX, c = c0;
    double x = s0, wt = w0;
    for (int i = i0; i < PER; ++i) {
      const int f = full(i);
      if (f > 0) {
        if (p < 1.0 && np == INT_MAX) {
          if (!(x < pz)) np = c;
          else if (wt > 0.0) {
            const double m = ceil((pz - x) / wt);
            if (m < (double)f) np = c + (int)m;
          }
        }
        if (wt < mp && nm == INT_MAX) nm = c;
        c += f;
        x += f * wt;
      }
      wt *= ratio;
    }
    if (np != INT_MAX) atomicMin(&sh.rank_p, np);
    if (nm != INT_MAX) atomicMin(&sh.rank_m, nm);
  }
  __syncthreads();
  const int keep = max(1, min(kk, min(sh.rank_p, sh.rank_m)));
  weight_to(keep, &sh.z);
  __syncthreads();
  const double z = sh.z, target = u * z;
  int at = -1;                     // the thread's candidate: value, place
  int place = 0;
  if (C > 0 && c0 < keep) {
    int c = c0, last = -1;
    double x = s0, wt = w0;
    for (int i = i0; i < PER && c < keep; ++i) {
      const int f = min(full(i), keep - c);
      if (f > 0 && wt > 0.0) {
        if (at < 0 && x + f * wt > target) {
          at = i;
          place = min(max((int)floor((target - x) / wt), 0), f - 1);
          atomicMin(&sh.rank, c + place);
        }
        last = c + f - 1;
      }
      c += f;
      x += f * wt;
      wt *= ratio;
    }
    if (last >= 0) atomicMax(&sh.last, last);
  }
  __syncthreads();
  // u at or past 1, or a NaN: the last kept token that has a weight
  const int rank = sh.rank != INT_MAX ? sh.rank : sh.last;
  if (rank >= c0 && rank < c0 + C) {
    int c = c0;
    double wt = w0;
    for (int i = i0; i < PER; ++i) {
      const int f = full(i);
      if (rank < c + f) {
        sh.bin = t * PER + i;
        sh.place = rank - c;
        sh.prob = wt / z;
        break;
      }
      c += f;
      wt *= ratio;
    }
  }
  __syncthreads();

  // ---- the token: number `place` among those of the value, by index
  const uint32_t want = (uint32_t)sh.bin;
  const int share = (row.vecs + WAVES - 1) / WAVES, v0 = w * share, v1 = min(v0 + share, row.vecs);
  auto matches = [&](int v) {
    const uint4 x = row.at[v];
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = 8 * v + e - row.lead;
      const uint32_t y = half_of(x, e);
      if (i >= 0 && i < V && bin_of(y) == want) mask |= 1u << e;
    }
    return mask;
  };
  int n = 0;
  for (int v = v0 + lane; v < v1; v += 64) n += __popc(matches(v));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  if (lane == 0) sh.in_wave[w] = n;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < w; ++i) before += sh.in_wave[i];
  place = sh.place - before;
  if (place < 0 || place >= n) return;           // not this wave
  for (int vb = v0; vb < v1; vb += 64) {
    const int v = vb + lane;
    const uint32_t mask = v < v1 ? matches(v) : 0;
    int c = __popc(mask), x = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    const int all = __shfl(x, 63, 64);
    if (place < all) {
      int left = place - (x - c);
      if (left >= 0 && left < c) {
        uint32_t mk = mask;
        while (left-- > 0) mk &= mk - 1;
        tokens[b] = 8ll * v + (__ffs((int)mk) - 1) - row.lead;
        probs[b] = (float)sh.prob;
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
