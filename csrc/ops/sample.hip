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
// No exponential is taken for a token: only for the values of the 64-value units that hold any, a unit in the lanes of
// a wave.  With the counts and weights before each unit in LDS, every rule is a search: the unit by two ballots, the
// value by a scan over the lanes.  All waves make the same searches, so none waits for another.  Weights and sums are
// 64-bit and in one fixed order: the same inputs give the same token.
//
// Bound: the LDS atomics of the count (14 of 29 us; 64 lanes on random banks, 14 cycles an instruction) and a chain of
// latencies.  A workgroup of 1024 threads takes a row, so up to 256 rows take little more than one: 30 us for 1 row of
// 152k tokens, 35 for 32 of mixed settings, 40 for 256.  Measured and left out: the row kept in registers (1 row 37 us
// against 30) -- the loops unrolled for it run from cold instruction lines; few rows counted by eight workgroups each,
// whose counts the last to arrive adds up (1 row 29.4 us against 29.5, 32 rows 37 against 35) -- leaving the counts,
// arriving and reading them takes what the shorter count saves.
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

typedef uint16_t bf16_t;

constexpr int NT = 1024, WAVES = NT / 64;
constexpr int BINS = 65536, UNITS = BINS / 64;
constexpr int WORDS = BINS / 2;                   // two 16-bit counters a word
constexpr int CARRY = 32768;                      // what is carried out of a counter
constexpr int CARRIES = 128;                      // carried counts: rows of up to CARRIES * CARRY tokens
constexpr int BATCH = 4;                          // vectors a thread loads at once: CARRY tokens of a workgroup
static_assert(BATCH * 8 * NT == CARRY, "a batch of tokens fits a counter of at most 32767 more");

// Bins: 0 for the largest value, 65535 for the smallest.  Positive values x (and +NaN first) are bins 0x7fff - x,
// negative ones (sign bit set) x - 1, so that both zeros are bin 0x7fff.
constexpr int BIN_INF = 0x7f, BIN_MINUS_INF = 0xff7f;   // behind it: -NaN

typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
typedef __attribute__((ext_vector_type(2))) int16_t i16x2;

// two tokens at once
__device__ __forceinline__ uint32_t bins_of(uint32_t x) {
  const uint32_t neg = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, x) >> (int16_t)15);   // 0xffff or 0
  const u16x2 y = __builtin_bit_cast(u16x2, x ^ (0x7fff7fffu & ~neg)) + __builtin_bit_cast(u16x2, neg);
  return __builtin_bit_cast(uint32_t, y);
}
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ float value_of(int bin) { return __uint_as_float((uint32_t)(bin < 0x8000 ? 0x7fff - bin : bin + 1) << 16); }

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// The row in aligned vectors of 8: vector v holds tokens 8v - lead .. 8v - lead + 7.  A wave has a run of them, 64 a
// turn, so that the tokens' order is that of the waves, turns, lanes.
struct Row {
  const uint4* at;
  int lead, V, vecs, from;     // from: the wave's first vector
  __device__ Row(const bf16_t* p, int V_, int turns, int w) : V(V_) {
    lead = (int)(((uintptr_t)p & 15) / 2);
    at = reinterpret_cast<const uint4*>((uintptr_t)p & ~(uintptr_t)15);
    vecs = (V + lead + 7) / 8;
    from = w * turns * 64;
  }
  // bins that a workgroup sees, those read as masked among them
  __device__ int seen(int turns) const { return WAVES * turns * 64 * 8; }
  // all 64 vectors of the turn lie in the row
  __device__ bool whole(int turn) const { return 8 * (from + 64 * turn) >= lead && 8 * (from + 64 * turn + 64) <= V + lead; }
  __device__ int vec(int turn) const { return from + 64 * turn + (int)(threadIdx.x & 63); }
  __device__ __forceinline__ uint4 load(int turn) const { return at[min(vec(turn), vecs - 1)]; }
  // the lane's first vectors, asked for ahead of a look at the row
  struct Batch { uint4 v[BATCH]; };
  __device__ __forceinline__ Batch first() const {
    Batch y;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) y.v[j] = load(j);
    return y;
  }
  // f(bins of the lane's vector, turn) for all turns, the next batch on its way; before(batch) ahead of each
  template <class F, class G>
  __device__ __forceinline__ void each(const Batch& begin, int turns, F f, G before) const {
    uint4 x[BATCH], y[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) y[j] = begin.v[j];
    for (int i = 0; i < turns; i += BATCH) {
#pragma unroll
      for (int j = 0; j < BATCH; ++j) x[j] = y[j];
      if (i + BATCH < turns) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) y[j] = load(i + BATCH + j);
      }
      before(i / BATCH);
#pragma unroll
      for (int j = 0; j < BATCH; ++j)
        if (i + j < turns) f(bins(x[j], i + j), i + j);
    }
  }
  template <class F>
  __device__ __forceinline__ void each(const Batch& begin, int turns, F f) const { each(begin, turns, f, [](int) {}); }
  template <class F>
  __device__ __forceinline__ void each(int turns, F f) const { each(first(), turns, f); }
  // bins of a turn's vector; what is not the row's reads as masked
  __device__ __forceinline__ uint4 bins(uint4 x, int turn) const {
    x = make_uint4(bins_of(x.x), bins_of(x.y), bins_of(x.z), bins_of(x.w));
    if (!whole(turn)) {
      auto pair = [&](uint32_t d, int e) {
        const int i = 8 * vec(turn) + e - lead;
        if (i < 0 || i >= V) d = (d & 0xffff0000u) | (uint32_t)BIN_MINUS_INF;
        if (i + 1 < 0 || i + 1 >= V) d = (d & 0xffffu) | ((uint32_t)BIN_MINUS_INF << 16);
        return d;
      };
      x = make_uint4(pair(x.x, 0), pair(x.y, 2), pair(x.z, 4), pair(x.w, 6));
    }
    return x;
  }
};

// inclusive sums over a wave's lanes, without LDS: row shifts, then the rows' ends broadcast
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = (uint32_t)moved<CTRL, ROWS>((int)(uint32_t)b), hi = (uint32_t)moved<CTRL, ROWS>((int)(b >> 32));
  return __builtin_bit_cast(double, (unsigned long long)lo | ((unsigned long long)hi << 32));
}
template <class T>
__device__ __forceinline__ T lane_scan(T v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ int lane_of(int v, int i) { return __builtin_amdgcn_readlane(v, i); }
__device__ __forceinline__ double lane_of(double v, int i) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = (uint32_t)lane_of((int)(uint32_t)b, i), hi = (uint32_t)lane_of((int)(b >> 32), i);
  return __builtin_bit_cast(double, (unsigned long long)lo | ((unsigned long long)hi << 32));
}
template <class T>
__device__ __forceinline__ T lane_sum(T v) { return lane_of(lane_scan(v), 63); }

struct Shared {
  double red_d[WAVES];
  int red_i[WAVES];
  int first, last;               // the largest and smallest value's bin (greedy rows), the largest one's unit (others)
  int nan;
  int counted, masked;           // tokens in the counters, and those that are -inf
  int index;                     // lowest index of what is looked for
  int carries, carry[CARRIES];
  int found[WAVES];
  int before_c[UNITS + 1];       // a unit's tokens, then the tokens before it
  double before_w[UNITS + 1];    // their weight
};

// the last unit whose entry is below x (or equal to it, where `equal`); -1 if none.  The entries ascend.
template <class T>
__device__ __forceinline__ int last_below(const T* a, T x, bool equal) {
  const int lane = threadIdx.x & 63;
  T y = a[lane * (UNITS / 64)];
  const int seg = __popcll(__ballot(y < x || (equal && y == x))) - 1;
  if (seg < 0) return -1;
  y = a[seg * (UNITS / 64) + (lane & (UNITS / 64 - 1))];
  return seg * (UNITS / 64) + __popcll(__ballot(y < x || (equal && y == x)) & ((1ull << (UNITS / 64)) - 1)) - 1;
}

__global__ void __launch_bounds__(NT)
sample_kernel(const bf16_t* __restrict__ logits, long long ld, int V, int turns, const float* __restrict__ uniform,
              const float* __restrict__ temperature, const int* __restrict__ top_k, const float* __restrict__ top_p,
              const float* __restrict__ min_p, int64_t* __restrict__ tokens, float* __restrict__ probs) {
  extern __shared__ __attribute__((aligned(16))) uint32_t hist[];
  __shared__ Shared sh;
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), b = blockIdx.x;
  const Row row(logits + (size_t)b * ld, V, turns, w);
  Row::Batch begin = row.first();
  const float T = temperature != nullptr ? temperature[b] : 1.f;
  if (t == 0) {
    sh.first = BINS;
    sh.last = -1;
    sh.index = INT_MAX;
  }

  // every token that `wanted` says: the lowest index is the answer; none: -1
  auto lowest = [&](auto wanted, float prob) {
    int at = INT_MAX;
    row.each(turns, [&](const uint4& x, int i) {
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (wanted((word_of(x, e >> 1) >> (16 * (e & 1))) & 0xffffu)) at = min(at, 8 * row.vec(i) + e - row.lead);
    });
    if (at != INT_MAX) atomicMin(&sh.index, at);
    __syncthreads();
    if (t == 0) {
      tokens[b] = sh.index != INT_MAX ? sh.index : -1;
      probs[b] = sh.index != INT_MAX ? prob : 0.f;
    }
  };
  // a NaN counts as the maximum
  auto is_nan = [](uint32_t bin) { return bin < (uint32_t)BIN_INF || bin > (uint32_t)BIN_MINUS_INF; };

  if (!(T > 0.f)) {                // greedy
    uint32_t lo = 0xffffffffu, hi = 0;
    row.each(begin, turns, [&](const uint4& x, int) {
      lo = min2(lo, min2(min2(x.x, x.y), min2(x.z, x.w)));
      hi = max2(hi, max2(max2(x.x, x.y), max2(x.z, x.w)));
    });
    int first = (int)min(lo & 0xffffu, lo >> 16), last = (int)max(hi & 0xffffu, hi >> 16);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      first = min(first, __shfl_xor(first, o, 64));
      last = max(last, __shfl_xor(last, o, 64));
    }
    __syncthreads();
    if (lane == 0) {
      atomicMin(&sh.first, first);
      atomicMax(&sh.last, last);
    }
    __syncthreads();
    first = sh.first;
    if (first < BIN_INF || sh.last > BIN_MINUS_INF) lowest(is_nan, NAN);
    else lowest([&](uint32_t bin) { return bin == (uint32_t)first && bin != (uint32_t)BIN_MINUS_INF; }, 1.f);
    return;
  }

  const int k = top_k != nullptr ? top_k[b] : 0;
  const double p = top_p != nullptr ? (double)top_p[b] : 1.0;
  const double mp = min_p != nullptr ? (double)min_p[b] : 0.0;
  const double u = uniform[b] < 0.f ? 0.0 : (double)uniform[b];
  const double rT = 1.0 / (double)T;    // one division a row: off by 2^-53 of the exponent
  int first = 0, ncarry = 0;
  float vmax = 0.f;
  // exp((value - max) / T); the largest value's is 1 whatever T and the value are
  auto weight = [&](int bin) {
    if (bin == first) return 1.0;
    return isfinite(vmax) ? exp(((double)value_of(bin) - (double)vmax) * rT) : 0.0;
  };
  auto count_of = [&](int bin) {
    int c = (int)((hist[bin >> 1] >> (16 * (bin & 1))) & 0xffffu);
    for (int j = 0; j < ncarry; ++j) c += sh.carry[j] == bin ? CARRY : 0;
    return c;
  };

  // Count, and the units' sums.  A value that more than 65535 tokens have overflows its counter, and then the counts
  // add up to less than the tokens (a carry into the word's other counter makes up for 1 of 65536): the row is counted
  // again, this time with full counters carried out as it goes.
  for (int careful = 0;; ++careful) {
    for (int i = t; i < WORDS / 4; i += NT) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
    sh.before_w[t] = 0.0;
    if (t == 0) {
      sh.first = BINS;
      sh.nan = 0;
      sh.counted = sh.masked = 0;
      sh.carries = 0;
    }
    __syncthreads();
    auto add = [&](uint32_t bin) { atomicAdd(&hist[bin >> 1], 1u + (bin & 1) * 0xffffu); };
    int masked = 0;
    row.each(
        begin, turns,
        [&](const uint4& x, int) {
          const uint32_t top = max2(max2(x.x, x.y), max2(x.z, x.w));
          const bool some = (top & 0xffffu) >= (uint32_t)BIN_MINUS_INF || (top >> 16) >= (uint32_t)BIN_MINUS_INF;
          if (!__ballot(some)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              add(word_of(x, j) & 0xffffu);
              add(word_of(x, j) >> 16);
            }
          } else {
            // masked tokens are not counted: they may be most of the row, and all on one address
            for (int j = 0; j < 8; ++j) {
              const uint32_t bin = (word_of(x, j >> 1) >> (16 * (j & 1))) & 0xffffu;
              if (bin != (uint32_t)BIN_MINUS_INF) add(bin);
              else ++masked;
            }
          }
        },
        [&](int batch) {
          if (!careful || batch == 0) return;
          __syncthreads();
          for (int i = t; i < WORDS; i += NT)
            for (int c = 0; c < 2; ++c)
              if (hist[i] & (0x8000u << (16 * c))) {
                hist[i] -= 0x8000u << (16 * c);
                sh.carry[atomicAdd(&sh.carries, 1)] = 2 * i + c;
              }
          __syncthreads();
        });
    masked = lane_sum(masked);
    if (lane == 0 && masked) atomicAdd(&sh.masked, masked);
    __syncthreads();

    // Unit u is wave u mod WAVES's.  Which hold anything: a lane looks at one, its eight vectors from a place of its own
    // on, so that the lanes of a read lie on different banks
    ncarry = __builtin_amdgcn_readfirstlane(sh.carries);
    const int mine = lane * WAVES + w;
    int cs = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(hist)[mine * 8 + ((i + lane) & 7)];
#pragma unroll
      for (int j = 0; j < 4; ++j) cs += (int)((word_of(x, j) & 0xffffu) + (word_of(x, j) >> 16));
    }
    for (int j = 0; j < ncarry; ++j) cs += sh.carry[j] / 64 == mine ? CARRY : 0;
    sh.before_c[mine] = cs;
    unsigned long long left = __ballot(cs != 0);
    const int sum = lane_sum(cs);
    if (left && lane == 0) {
      atomicMin(&sh.first, __builtin_ctzll(left) * WAVES + w);
      atomicAdd(&sh.counted, sum);
    }
    if (cs != 0 && mine * 64 > BIN_MINUS_INF) sh.nan = 1;
    __syncthreads();
    if (!careful && sh.counted != row.seen(turns) - sh.masked) {
      __syncthreads();
      continue;
    }
    first = sh.first;
    if (first == BINS) {                         // no token
      if (t == 0) tokens[b] = -1, probs[b] = 0.f;
      return;
    }
    first = first * 64 + __builtin_ctzll(__ballot(count_of(first * 64 + lane) != 0));
    if (first < BIN_INF || sh.nan) {
      lowest(is_nan, NAN);
      return;
    }
    vmax = value_of(first);
    for (; left != 0; left &= left - 1) {
      const int unit = __builtin_ctzll(left) * WAVES + w, bin = unit * 64 + lane;
      const int c = count_of(bin);
      const double ws = lane_sum(c > 0 ? c * weight(bin) : 0.0);
      if (lane == 0) sh.before_w[unit] = ws;
    }
    __syncthreads();
    const int c = sh.before_c[t], ci = lane_scan(c);
    const double s = sh.before_w[t], si = lane_scan(s);
    if (lane == 63) sh.red_i[w] = ci, sh.red_d[w] = si;
    __syncthreads();
    int cb = 0;
    double sb = 0.0;
    for (int i = 0; i < w; ++i) {
      cb += sh.red_i[i];
      sb += sh.red_d[i];
    }
    // an entry is the sum up to the lane before, a wave's first the sum of the waves before, so that they ascend
    const int cp = __shfl_up(ci, 1, 64);
    const double sp = __shfl_up(si, 1, 64);
    sh.before_c[t] = cb + (lane > 0 ? cp : 0);
    sh.before_w[t] = sb + (lane > 0 ? sp : 0.0);
    if (t == NT - 1) sh.before_c[UNITS] = cb + ci, sh.before_w[UNITS] = sb + si;
    __syncthreads();
    break;
  }

  // ---- from here on every wave does the same
  begin = row.first();                           // for the last look
  const int total = sh.before_c[UNITS];
  // weight of the first n >= 1 tokens in order
  auto weight_to = [&](int n) {
    if (n == total) return sh.before_w[UNITS];
    const int unit = last_below(sh.before_c, n, false), bin = unit * 64 + lane;
    const int c = count_of(bin), m = min(max(n - sh.before_c[unit] - (lane_scan(c) - c), 0), c);
    return sh.before_w[unit] + lane_sum(m > 0 ? m * weight(bin) : 0.0);
  };
  int keep = k > 0 ? min(k, total) : total;
  if (p < 1.0) {
    // tokens that have less than p of the first keep's weight before them
    const double pz = p * weight_to(keep);
    const int unit = last_below(sh.before_w, pz, false);
    int n = 1;
    if (unit >= 0) {
      const int bin = unit * 64 + lane, c = count_of(bin);
      const double wt = c > 0 ? weight(bin) : 0.0, cw = c * wt, before = sh.before_w[unit] + (lane_scan(cw) - cw);
      int m = 0;
      if (c > 0 && before < pz) m = wt > 0.0 ? (int)min((double)c, ceil((pz - before) / wt)) : c;
      n = sh.before_c[unit] + lane_sum(m);
    }
    keep = max(1, min(keep, n));
  }
  if (mp > 1.0) {
    keep = 1;                                    // no weight reaches it, the largest neither
  } else if (mp > 0.0) {
    // tokens of a weight of at least min_p: weights fall along the bins, so look at every 1024th, then every 64th of
    // those, then each
    auto heavy = [&](int bin) { return bin <= first || weight(bin) >= mp; };
    const int seg = max(__popcll(__ballot(heavy(lane * (BINS / 64)))) - 1, 0);
    const int sub = max(__popcll(__ballot(lane < UNITS / 64 && heavy(seg * (BINS / 64) + lane * 64))) - 1, 0);
    const int unit = seg * (UNITS / 64) + sub;
    const int m = lane_sum(heavy(unit * 64 + lane) ? count_of(unit * 64 + lane) : 0);
    keep = max(1, min(keep, sh.before_c[unit] + m));
  }
  const double z = weight_to(keep), target = u * z;
  int bin = 0, place = 0, in_bin = 0;
  double prob = 0.0;
  // the unit whose weights reach past the target; for u at or past 1 (or a NaN) the last kept token's
  for (int unit = target < z ? last_below(sh.before_w, target, true) : last_below(sh.before_c, keep, false);; --unit) {
    const int x = unit * 64 + lane, c = count_of(x), ci = lane_scan(c) - c;
    const int m = min(max(keep - sh.before_c[unit] - ci, 0), c);
    const double wt = m > 0 ? weight(x) : 0.0, mw = m * wt, before = sh.before_w[unit] + (lane_scan(mw) - mw);
    const unsigned long long some = __ballot(wt > 0.0), hit = __ballot(wt > 0.0 && before + mw > target);
    // no kept token of any weight only at the ends of rounding: the unit before.  The first token is kept and weighs 1
    if (some == 0) continue;
    const int who = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
    const int j = hit ? min(max((int)floor((target - before) / wt), 0), m - 1) : m - 1;
    bin = unit * 64 + who;
    place = lane_of(j, who);
    in_bin = lane_of(c, who);
    prob = lane_of(wt, who) / z;
    break;
  }

  // ---- the token: number `place` among those of the value, by index
  const uint32_t pattern = (uint32_t)bin * 0x10001u;
  auto answer = [&](int turn, int e) {
    tokens[b] = 8ll * row.vec(turn) + e - row.lead;
    probs[b] = (float)prob;
  };
  auto matches = [&](const uint4& x) {           // a bit for each token of a vector
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t d = word_of(x, i) ^ pattern;
      mask |= ((d & 0xffffu) == 0 ? 1u << (2 * i) : 0) | ((d >> 16) == 0 ? 2u << (2 * i) : 0);
    }
    return mask;
  };
  int n = 0;
  row.each(begin, turns, [&](const uint4& x, int i) {
    uint32_t far = 0x00010001u;                  // 0 in a half where some token matches
#pragma unroll
    for (int j = 0; j < 4; ++j) far = min2(far, word_of(x, j) ^ pattern);
    if (far != 0x00010001u) {
      const uint32_t mask = matches(x);
      if (in_bin == 1) answer(i, __ffs((int)mask) - 1);      // the only one: whoever has it
      n += (int)__popc(mask);
    }
  });
  if (in_bin == 1) return;
  n = lane_sum(n);
  if (lane == 0) sh.found[w] = n;
  __syncthreads();
  for (int i = 0; i < w; ++i) place -= sh.found[i];
  if (place < 0 || place >= n) return;           // not this wave
  row.each(turns, [&](const uint4& x, int i) {
    const uint32_t mask = matches(x);
    const int c = (int)__popc(mask), s = lane_scan(c);
    int left = place - (s - c);
    if (left >= 0 && left < c) {
      uint32_t mk = mask;
      while (left-- > 0) mk &= mk - 1;
      answer(i, __ffs((int)mk) - 1);
    }
    place -= lane_of(s, 63);                     // below 0 behind the answer: no turn matches again
  });
}

}  // namespace

extern "C" {

int mivgpu_sample(const void* logits, long long ld, int V, int B, const float* uniform, const float* temperature,
                  const int* top_k, const float* top_p, const float* min_p, int64_t* tokens, float* probs,
                  hipStream_t s) {
  if (B <= 0 || V <= 0 || V > CARRIES * CARRY || (B > 1 && ld < V)) return -1;
  constexpr int lds = WORDS * 4;
  const int turns = ((V + 7 + 7) / 8 + NT - 1) / NT;        // wherever the row starts
  const hipError_t e = hipFuncSetAttribute((const void*)sample_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(sample_kernel, dim3(B), dim3(NT), lds, s, (const bf16_t*)logits, ld, V, turns, uniform, temperature,
                     top_k, top_p, min_p, tokens, probs);
  return (int)hipGetLastError();
}

}  // extern "C"
