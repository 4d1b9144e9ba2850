// Attention of a ragged batch of tokens over 8-bit K/V pages (paged.h: layout and scales).
//
// Request b owns the q rows cu[b] .. cu[b+1] (n of them) and kv_lens[b] = L keys; its row i sits at position
// L - n + i and sees the keys up to there.  A row that sees no key gives zeros.
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale (q_i . k_j) - m_i)
// in one pass over the pages with the running maximum m and sum (fp32).
//
// The rows of one kv head's G query heads are flattened (row = token * G + head) and cut into tiles: of 16 rows where
// a request brings few of them (short_rows: decode, a few tokens), of 256 in the others (chunks, prompts).  Both
// kinds of workgroups are in one launch, so that the short ones' waits for memory lie beside the long ones' products (a
// chunk of 855 tokens beside seven decoding requests: 80 us; in a launch each 90).
// A tile's pages are split over as many workgroups as keep the chip evenly busy: every workgroup scans the requests'
// lengths (at most 1024: a few a lane) and takes its share of all tiles' pages, so that one long request among short
// ones is cut into more parts and nothing is planned on the host.  The parts of a tile leave their (m, l, O) in the
// workspace, and the last one to arrive (a counter that it sets back to zero) joins them in the order of the parts, so
// that a call's bits do not depend on who that is.
//
// Tiles of 16: the waves of a workgroup take its pages in turn and join in LDS.  Per page of 64 keys a wave computes,
// with 16x16x32 bf16 MFMAs,
//   S^T (64 keys x 16 rows) = K . Q^T        4 tiles of 16 keys: tile t's row 4a + c is key 16a + 4t + c, so that
//                                            lane (row r, quarter a) ends with the 16 consecutive keys 16a .. 16a+15;
//   O^T (D x 16 rows) += V^T . P^T           whose operands want exactly that: 8 consecutive keys a lane and k-step.
// P never leaves its lane.  e4m3 codes become bf16 with their page's scale in one instruction for two values
// (exact: a code has 4 significant bits and the scale is a power of two).  P is rounded to bf16 (half a step of the
// output's type, before a sum that averages it); scores, m, l and O stay in fp32.
#include "paged.h"
#include <type_traits>

using namespace paged;

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

typedef __attribute__((ext_vector_type(16))) float f32x16_t;

// short requests
constexpr int TILE = 16, SWAVES = 4;     // waves of a workgroup (where the launch has long ones too, as many as those)
constexpr int MAX_PARTS = 256;           // of a tile: their (m, l) take 32 KB of LDS
constexpr int JOIN = 64;                 // head dimensions that the waves join at once
// long requests
constexpr int LNT = 512, LWAVES = 8, LTILE = 32 * LWAVES;
constexpr int LMIN_CHUNK = 8;

// The most rows of a request that go in short tiles.  A short tile is soon done but reads its pages for 16 rows, a long
// one takes 2 to 3 times as long for up to 256; calls of few rows have CUs over for short ones.  32 / 8 heads, 4096 keys
// before the new ones, us short / long: 1 request of 64 rows 13 / 26, of 256 27 / 50; 4 of 64 28 / 29, of 128 31 / 35;
// 16 of 64 56 / 87, of 128 109 / 87; 64 of 32 134 / 175, of 64 228 / 178.
constexpr int FEW_ROWS = 512, MANY_ROWS = 4096;
constexpr int short_rows(long long rows) {
  return rows <= FEW_ROWS ? FEW_ROWS : rows < MANY_ROWS ? 64 : 32;
}

// A call aims at as many workgroups as are resident (of the short ones two a CU, one beside long ones; of the long ones
// one), over all kv heads, and with that bounds the slots of the workspace: with t parts aimed at a kv head a
// split tile of np pages gets at most np / chunk + 1 <= 2 np / chunk parts, which add up to at most 2 t.
constexpr int MAX_CUS = 256, MAX_HKV = 256;
// (Beside long ones there is LDS for one, also with D = 64.  Aiming at two, 16 decoding requests of 4096 keys beside a
// chunk of 1000, 8 / 8 heads of 64: 49 us instead of 42; 20 of 30 to 8000 beside 512, 32 / 4 heads: 25.3 and 23.)
constexpr int short_resident(bool longs) { return longs ? 1 : 2; }
constexpr int SHORT_SLOTS = 2 * 2 * MAX_CUS, LONG_SLOTS = 2 * MAX_CUS;

// 8 codes -> 8 bf16, times 2^e
__device__ __forceinline__ bf16x8_t widen(uint32_t lo, uint32_t hi, float s) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// bytes of a word whose key (k0 + i) is below `live`
__device__ __forceinline__ uint32_t live_bytes(int k0, int live) {
  const int n = min(max(live - k0, 0), 4);
  return n == 4 ? ~0u : (1u << (8 * n)) - 1u;
}

// waits for a loaded operand here.  Without it the compiler waits wherever a loop uses the operand, there for the loads
// that the loop itself has on their way
__device__ __forceinline__ void arrived(bf16x8_t& x) {
  typedef __attribute__((ext_vector_type(4))) int i32x4_t;
  i32x4_t y = __builtin_bit_cast(i32x4_t, x);
  asm volatile("" : "+v"(y));
  x = __builtin_bit_cast(bf16x8_t, y);
}

// two floats to and from memory that workgroups on other XCDs share within a launch
__device__ __forceinline__ void put2(float* at, float x, float y) {
  const unsigned long long v = (unsigned long long)__float_as_uint(x) | ((unsigned long long)__float_as_uint(y) << 32);
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(at), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* at) {
  const unsigned long long v =
      __hip_atomic_load(reinterpret_cast<const unsigned long long*>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// The widening takes a scale's exponent only.  A page with a scale that is no power of two (or outside the append's range)
// reads as NaN in K: rows that see it give NaN, not values that are up to twice too small.
__device__ __forceinline__ void check_scales(float& ks, float& vs) {
  const bool good = is_scale(ks) && is_scale(vs);
  ks = good ? ks : __uint_as_float(0x7fc00000u);
  vs = good ? vs : 1.f;
}

// a row's four values of head dimension d .. d+3; a row that saw no key (l = 0) gives zeros
__device__ __forceinline__ void store_row(bf16_t* out, f32x4_t o, float l, int row, int tok0, int G, int Hq, int hk, int D,
                                          int d) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bf16_t* at = out + ((size_t)(tok0 + row / G) * Hq + (size_t)hk * G + row % G) * D + d;
  *reinterpret_cast<uint2*>(at) = make_uint2(pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv));
}

// which request, tile of its rows and part of that tile's pages a workgroup takes, from its index among all parts
struct Share {
  int b, tile, part, ns;     // ns: parts of the tile; 0: nothing left for this workgroup
  int slot;                  // of the tile's first part, among the split tiles' parts
};

// inclusive sum over the wave's lanes, without LDS (row shifts, then the rows' ends broadcast)
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// Every wave scans all requests of more than `above` and at most `upto` rows by itself, 64 at once, in registers: no
// barrier, and one round of loads.  Workgroup 0 takes the last part of all: in a prompt the tiles at the end have the
// most keys, and the longest work should start first.  The caller sees to it that the sums fit 31 bits (and
// no more is added to them).
// Joining the parts of a short tile takes about 0.1 us a part, a page for each of its waves 1.5: at most sqrt(2 pages)
// parts (one request of 131072 keys, 16 / 1 heads: 31 us against 53 with 256 parts; of 32768 20 against 23).
template <int ROWS, int SMALLEST>
__device__ __forceinline__ Share find_share(const int* __restrict__ cu, const int* __restrict__ kv_lens, int N, int B, int W,
                                            int G, int target, int above, int upto, int me, int Hkv, unsigned grid) {
  constexpr int PER = MAX_ROWS / 64;
  const int lane = threadIdx.x & 63;
  int tiles[PER], np[PER], sum = 0, some = 0;    // of requests 64 x + lane
  {
    int from[PER], to[PER];
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      if (64 * x >= B) break;
      const int b = min(64 * x + lane, B - 1);
      from[x] = cu[b];
      to[x] = cu[b + 1];
      np[x] = kv_lens[b];
    }
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      if (64 * x >= B) break;
      const int rows = max(min(to[x], N) - min(max(from[x], 0), N), 0) * G;
      const bool ours = 64 * x + lane < B && rows > above && rows <= upto;
      tiles[x] = ours ? (rows + ROWS - 1) / ROWS : 0;
      np[x] = (min(max(np[x], 0), W * PAGE) + PAGE - 1) / PAGE;
      sum += tiles[x] * np[x];
      some += tiles[x];
    }
  }
  const int total = __builtin_amdgcn_readlane(wave_scan(sum), 63);
  // a tile's last part is mostly smaller than a chunk: leave a workgroup for each, so that all parts are resident at once
  const int goal = max(target - __builtin_amdgcn_readlane(wave_scan(some), 63), (target + 1) / 2);
  const int chunk = max((total - 1) / goal + 1, SMALLEST);
  int all = 0;
#pragma unroll
  for (int x = 0; x < PER; ++x) {
    if (64 * x >= B) break;
    const int most = ROWS == TILE ? min(MAX_PARTS, (int)__builtin_amdgcn_sqrtf(2.f * (float)np[x])) : MAX_PARTS;
    np[x] = max(min((np[x] - 1) / chunk + 1, most), 1);                  // from here on: parts of a tile
    all += tiles[x] * np[x];
  }
  all = __builtin_amdgcn_readlane(wave_scan(all), 63);
  me = all - 1 - me;
  Share sh = {0, 0, 0, 0, 0};
  // requests that overlap may have more parts than the launch: then none is worked on, so that none waits in a counter
  if (me < 0 || (long long)all * Hkv > grid) return sh;
  int before = 0, split = 0;                     // parts of the requests before, and those of split tiles
#pragma unroll
  for (int x = 0; x < PER; ++x) {
    if (64 * x >= B) break;
    const int ns = np[x], n = tiles[x] * ns, end = before + wave_scan(n);
    const int cut = ns > 1 ? n : 0, slot = split + wave_scan(cut) - cut;
    const unsigned long long owner = __ballot(me >= end - n && me < end);
    if (owner != 0) {
      const int who = __ffsll((long long)owner) - 1, at = me - __builtin_amdgcn_readlane(end - n, who);
      sh.b = 64 * x + who;
      sh.ns = __builtin_amdgcn_readlane(ns, who);
      sh.tile = at / sh.ns;
      sh.part = at % sh.ns;
      sh.slot = __builtin_amdgcn_readlane(slot, who) + sh.tile * sh.ns;
      // split tiles have at most `goal` whole chunks and one part more each: never past the workspace
      if (sh.ns > 1 && (sh.slot < 0 || sh.slot + sh.ns > 2 * target)) sh.ns = 0;
      break;
    }
    before = __builtin_amdgcn_readlane(end, 63);
    split = __builtin_amdgcn_readlane(slot + cut, 63);
  }
  return sh;
}

// What both kinds of workgroups are called with
struct Call {
  const bf16_t* __restrict__ q;
  const uint8_t *__restrict__ kc, *__restrict__ vc;
  const float *__restrict__ kscale, *__restrict__ vscale;
  const int *__restrict__ table, *__restrict__ cu, *__restrict__ kv_lens;
  bf16_t* __restrict__ out;
  int N, B, W, Hq, Hkv, pages, upto;     // upto: the most rows of a request that short tiles take
  float scale_log2;
};
// Of one kind: its workspace, the parts it aims at for each kv head, and its workgroups
struct Work {
  int* __restrict__ counters;
  float *__restrict__ part_ml, *__restrict__ part_o;
  int target;
  unsigned grid;
};
#define MIVGPU_PATTN_ARGS                                                                                             \
  const bf16_t* __restrict__ q = c.q;                                                                                 \
  const uint8_t *__restrict__ kc = c.kc, *__restrict__ vc = c.vc;                                                     \
  const float *__restrict__ kscale = c.kscale, *__restrict__ vscale = c.vscale;                                       \
  const int *__restrict__ table = c.table, *__restrict__ cu = c.cu, *__restrict__ kv_lens = c.kv_lens;                \
  bf16_t* __restrict__ out = c.out;                                                                                   \
  int* __restrict__ counters = k.counters;                                                                            \
  float *__restrict__ part_ml = k.part_ml, *__restrict__ part_o = k.part_o;                                           \
  const int N = c.N, B = c.B, W = c.W, Hq = c.Hq, Hkv = c.Hkv, pages = c.pages, target = k.target;                    \
  const float scale_log2 = c.scale_log2

template <int D, int WAVES>
struct ShortLds {
  float m[WAVES][TILE], l[WAVES][TILE];
  int last;
  // the waves' O; later the (m, l) of a tile's parts and what groups of threads make of them
  static constexpr int O_BYTES = WAVES * TILE * (JOIN + 4) * 4, JOIN_BYTES = MAX_PARTS * TILE * 8 + WAVES * 64 * 20;
  __attribute__((aligned(16))) char raw[O_BYTES > JOIN_BYTES ? O_BYTES : JOIN_BYTES];
};

// upto: as in Call, or all
template <int D, int WAVES>
__device__ __forceinline__ void short_part(const Call& c, const Work& k, int upto, unsigned block, ShortLds<D, WAVES>& lds) {
  MIVGPU_PATTN_ARGS;
  constexpr int NT = 64 * WAVES;
  constexpr int KU = D / 64;              // 16-byte chunks of a K row per lane
  constexpr int DT = D / 16;              // output tiles
  auto& s_m = lds.m;
  auto& s_l = lds.l;
  auto& s_raw = lds.raw;
  int& s_last = lds.last;
  float(*s_o)[TILE][JOIN + 4] = reinterpret_cast<float(*)[TILE][JOIN + 4]>(s_raw);
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 15, a = lane >> 4;
  const int G = Hq / Hkv, hk = block % Hkv;
  const Share sh = find_share<TILE, WAVES>(cu, kv_lens, N, B, W, G, target, 0, upto, block / Hkv, Hkv, k.grid);
  if (sh.ns == 0) return;
  const int b = sh.b, row0 = sh.tile * TILE, ns = sh.ns;
  const int tok0 = min(max(cu[b], 0), N), n = min(cu[b + 1], N) - tok0, rows = n * G;
  const int L = min(max(kv_lens[b], 0), W * PAGE);

  // keys that this lane's row sees, and the most that a row of the tile sees
  const int row = row0 + r;
  const int vis = row < rows ? max(L - n + row / G + 1, 0) : 0;
  const int last = min(row0 + TILE, rows) - 1;
  const int most = max(L - n + last / G + 1, 0);
  const int least = max(L - n + row0 / G + 1, 0);

  // Q^T operand: lane (r, a) holds dims 16 (a + 4u) + 8 half .. + 8 of its row, as the K chunks come
  bf16x8_t qf[KU][2];
  {
    const int rr = min(row, rows - 1);
    const bf16_t* qp = q + ((size_t)(tok0 + rr / G) * Hq + (size_t)hk * G + rr % G) * D;
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) qf[u][h] = *reinterpret_cast<const bf16x8_t*>(qp + 16 * (a + 4 * u) + 8 * h);
  }

  f32x4_t o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  const int npages = (most + PAGE - 1) / PAGE;
  const int p0 = (int)((long long)npages * sh.part / ns), p1 = (int)((long long)npages * (sh.part + 1) / ns);
  const int turns = p1 - p0 > w ? (p1 - p0 - w + WAVES - 1) / WAVES : 0;   // pages of this wave
  int ids = 0;                                    // lane i: one of the wave's next 64 pages, and its scales
  float kss = 0.f, vss = 0.f;
  uint4 kr[4][KU], vr[DT];
  struct Page {
    size_t ph;
    bool bad;                                     // not a page of the cache: its keys count as masked
  };
  auto page_at = [&](int turn) {
    if ((turn & 63) == 0) {
      ids = table[(size_t)b * W + min(p0 + w + (turn + lane) * WAVES, npages - 1)];
      const size_t at = (size_t)(ids < 0 || ids >= pages ? 0 : ids) * Hkv + hk;
      kss = kscale[at];
      vss = vscale[at];
    }
    const int id = __builtin_amdgcn_readlane(ids, turn & 63);
    Page x;
    x.bad = id < 0 || id >= pages;
    x.ph = (size_t)(x.bad ? 0 : id) * Hkv + hk;
    return x;
  };
  auto load_k = [&](size_t ph) {
    const uint8_t* kp = kc + ph * PAGE * D + (size_t)(16 * (r >> 2) + (r & 3)) * D + 16 * a;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int u = 0; u < KU; ++u) kr[tt][u] = *reinterpret_cast<const uint4*>(kp + 4 * tt * D + 64 * u);
  };
  auto load_v = [&](size_t ph) {
    const uint8_t* vp = vc + ph * PAGE * D + (size_t)r * PAGE + 16 * a;
#pragma unroll
    for (int i = 0; i < DT; ++i) vr[i] = *reinterpret_cast<const uint4*>(vp + 16 * i * PAGE);
  };
  // K and V of a page are in registers before their turn: the next page's K is on its way from the moment that the
  // scores have read this one's, its V from the moment that the output has
  Page cur{}, next{};
  if (turns > 0) {
    cur = page_at(0);
    load_k(cur.ph);
    load_v(cur.ph);
  }
  for (int turn = 0; turn < turns; ++turn) {
    if ((turn & 63) == 0) check_scales(kss, vss);   // not where they are loaded: K and V need not wait for them
    const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kss), turn & 63));
    const float vs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vss), turn & 63));
    f32x4_t s[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      s[tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const uint4 c = kr[tt][u];
        s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(c.x, c.y, ks), qf[u][0], s[tt], 0, 0, 0);
        s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(c.z, c.w, ks), qf[u][1], s[tt], 0, 0, 0);
      }
    }
    if (turn + 1 < turns) {
      next = page_at(turn + 1);
      load_k(next.ph);
    }
    const int key0 = (p0 + w + turn * WAVES) * PAGE;
    const int live = cur.bad ? 0 : L - key0;      // keys of the page that were written
    if (cur.bad || key0 + PAGE > least) {
      const int seen = cur.bad ? 0 : vis - key0;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * a + 4 * tt + i >= seen) s[tt][i] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[tt][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mnew = fmaxf(m, mx * scale_log2);
    const float base = mnew == -INFINITY ? 0.f : mnew;    // nothing seen yet: every p is exp2(-inf) = 0
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    m = mnew;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] *= alpha;
    bf16x8_t pf[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[2 * h + j / 4][j & 3], scale_log2, -base));
        l += e;
        pf[h][j] = (__bf16)e;
      }
    if (live < PAGE) {                            // slots never written may hold any code, NaN too
      const uint32_t m0 = live_bytes(16 * a, live), m1 = live_bytes(16 * a + 4, live), m2 = live_bytes(16 * a + 8, live),
                     m3 = live_bytes(16 * a + 12, live);
#pragma unroll
      for (int i = 0; i < DT; ++i) vr[i].x &= m0, vr[i].y &= m1, vr[i].z &= m2, vr[i].w &= m3;
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const uint4 c = vr[i];
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(c.x, c.y, vs), pf[0], o[i], 0, 0, 0);
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(c.z, c.w, vs), pf[1], o[i], 0, 0, 0);
    }
    if (turn + 1 < turns) load_v(next.ph);
    cur = next;
  }

  // join the waves
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (a == 0) s_m[w][r] = m, s_l[w][r] = l;
  const size_t slot0 = (size_t)sh.slot * Hkv + hk, slot_step = Hkv;     // the tile's parts in the workspace
  const size_t slot = slot0 + sh.part * slot_step;
  const int filled = min(TILE, rows - row0);
#pragma unroll
  for (int j = 0; j < D / JOIN; ++j) {
    if (j > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < JOIN / 16; ++i)
      if (r < filled) *reinterpret_cast<f32x4_t*>(&s_o[w][r][16 * i + 4 * a]) = o[JOIN / 16 * j + i];
    __syncthreads();
    const int rr = t / (JOIN / 4), d = t % (JOIN / 4) * 4;             // a thread's row and four dimensions
    if (rr < filled) {
      float mm = -INFINITY;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) mm = fmaxf(mm, s_m[i][rr]);
      const float base = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      f32x4_t oo = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        const float f = __builtin_amdgcn_exp2f(s_m[i][rr] - base);
        ll += s_l[i][rr] * f;
        oo += *reinterpret_cast<const f32x4_t*>(&s_o[i][rr][d]) * f;
      }
      if (ns == 1) {
        store_row(out, oo, ll, row0 + rr, tok0, G, Hq, hk, D, JOIN * j + d);
      } else {
        put2(part_o + (slot * TILE + rr) * D + JOIN * j + d, oo[0], oo[1]);
        put2(part_o + (slot * TILE + rr) * D + JOIN * j + d + 2, oo[2], oo[3]);
        if (j == 0 && d == 0) put2(part_ml + (slot * TILE + rr) * 2, mm, ll);
      }
    }
  }
  if (ns == 1) return;

  // The last part of the tile to arrive joins them all.  The parts are stored and loaded past the XCDs' own caches
  // (put2 / get2); each wave waits for its stores before the workgroup counts itself.  A release fence here instead
  // writes back the whole of the XCD's L2 for every part: 110 us against 20 for 32 rows of 1024 keys.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (t == 0) s_last = __hip_atomic_fetch_add(&counters[slot0], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == ns - 1;
  __syncthreads();
  if (!s_last) return;
  if (t == 0) __hip_atomic_store(&counters[slot0], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // Four values a thread; few rows leave threads over, and each of `groups` takes every groups-th part.  The first parts'
  // O are on their way while all (m, l) come into LDS.
  float2* ml = reinterpret_cast<float2*>(s_raw);                      // [part][row]
  float* joined = reinterpret_cast<float*>(s_raw + MAX_PARTS * TILE * 8);   // [thread][4 values, l]
  const int units = filled * (D / 4), groups = max(NT / units, 1);
  for (int u0 = 0; u0 < units; u0 += NT) {        // more than once for four waves and many rows only
    const int group = (u0 + t) / units, unit = u0 + t - group * units, rr = unit / (D / 4), d = unit % (D / 4) * 4;
    constexpr int AHEAD = 8;                      // loads in flight
    float2 x01[AHEAD], x23[AHEAD];
    auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const float* src = part_o + ((slot0 + min(i0 + j * groups, ns - 1) * slot_step) * TILE + rr) * D + d;
        x01[j] = get2(src);
        x23[j] = get2(src + 2);
      }
    };
    if (group < groups) load(group);
    if (u0 == 0) {
      for (int x = t; x < ns * filled; x += NT) {
        const int i = x / filled, row = x % filled;
        ml[i * TILE + row] = get2(part_ml + ((slot0 + i * slot_step) * TILE + row) * 2);
      }
      __syncthreads();
    }
    if (group < groups) {
      float mm = -INFINITY;
      for (int i = 0; i < ns; ++i) mm = fmaxf(mm, ml[i * TILE + rr].x);
      const float base = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      f32x4_t oo = f32x4_t{0.f, 0.f, 0.f, 0.f};
      for (int i0 = group; i0 < ns; i0 += groups * AHEAD) {
        if (i0 != group) load(i0);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const int i = i0 + j * groups;
          if (i < ns) {
            const float2 e = ml[i * TILE + rr];
            const float f = __builtin_amdgcn_exp2f(e.x - base);
            ll += e.y * f;
            oo += f32x4_t{x01[j].x, x01[j].y, x23[j].x, x23[j].y} * f;
          }
        }
      }
      if (groups == 1) {
        store_row(out, oo, ll, row0 + rr, tok0, G, Hq, hk, D, d);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) joined[t * 5 + j] = oo[j];
        joined[t * 5 + 4] = ll;
      }
    }
  }
  if (groups == 1) return;
  __syncthreads();
  if (t < units) {
    float ll = 0.f;
    f32x4_t oo = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < groups; ++g) {
      const float* from = joined + (g * units + t) * 5;
      oo += f32x4_t{from[0], from[1], from[2], from[3]};
      ll += from[4];
    }
    store_row(out, oo, ll, row0 + t / (D / 4), tok0, G, Hq, hk, D, t % (D / 4) * 4);
  }
}

// ------------------------------------------------------------------------------------------------ long requests --
// Eight waves of 32 rows share every page: its codes become bf16 once, on their way from registers (a 16-byte load
// of K and of V a thread) to LDS.  LDS has room for four pages: between the two pages that are worked on, the next two
// are stored and the loads of the two after those sent off; one barrier for two pages.  Per page a wave computes, with
// 32x32x16 bf16 MFMAs,
//   S^T (2 x 32 keys x 32 rows) = K . Q^T     lane (row r, half h) holds the keys (i & 3) + 8 (i >> 2) + 4 h of each 32;
//   O^T (D x 32 rows) += V^T . P^T            eight registers of S^T are the operand of a k-step of 16 keys: keys
//                                             {0-3, 8-11} + 4 h; V's 16 keys are stored in two chunks in that order.
// LDS rows are permuted by 16-byte chunks (chunk ^ row; V's, two rows to the banks, chunk ^ row / 2) so that the lanes
// of a read cover all banks.
// The output and sum are rescaled only where a row's maximum grew by more than 8 (in log2): the p stay below 2^8,
// which neither bf16 nor the sums mind.
// Measured on an 8192-token prompt, 32 / 8 heads: 514 us, 1070 TFLOP/s; with the stores before the barrier instead of
// between the pages 525, a barrier a page 568, the buffers picked at run time 551.  The matrix units are busy half of
// the time and the vector units the other half, one after the other, at a clock of 1.9 to 2.1 GHz of the card's 2.4.
// That is no limit of the card: in a probe, matrix instructions of one wave and vector ones of another on a SIMD do
// overlap (0.242 and 0.237 ms alone, 0.305 together).  Nothing tried here made the loop do so: operands read three steps
// ahead 511, the next page's scores beside this one's exponentials in a wave 528, the two waves of a SIMD half a page
// apart, one's matrix instructions beside the other's exponentials, two barriers a page 653 (614 without the offset), four
// waves of 64 rows, which halve the LDS reads, with the next page's scores beside this one's exponentials 792.  Less work
// gains time: without the stores and loads it would be 396.
template <int D>
__device__ __forceinline__ int k_at(int row, int ch) { return row * D + ((ch ^ (row & (D / 8 - 1))) << 3); }
__device__ __forceinline__ int v_at(int dim, int ch) { return dim * PAGE + ((ch ^ ((dim >> 1) & 7)) << 3); }

template <int D>
__device__ __forceinline__ void long_part(const Call& c, const Work& k, unsigned block, bf16_t (&s_k)[4][PAGE * D],
                                          bf16_t (&s_v)[4][PAGE * D]) {
  MIVGPU_PATTN_ARGS;
  constexpr int KS = D / 16, DC = D / 32;              // k-steps of the scores, 32-wide blocks of the output
  constexpr int CHUNKS = PAGE * D / 16;                // 16-byte chunks of codes in a page, each of K and V
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 31, h = lane >> 5;
  // kv head = workgroup mod Hkv: with 8 of them each XCD's L2 serves one head's pages
  const int G = Hq / Hkv, hk = block % Hkv;
  const Share sh =
      find_share<LTILE, LMIN_CHUNK>(cu, kv_lens, N, B, W, G, target, c.upto, INT_MAX, block / Hkv, Hkv, k.grid);
  if (sh.ns == 0) return;
  const int b = sh.b, ns = sh.ns, tile0 = sh.tile * LTILE, row0 = tile0 + 32 * w;
  const int tok0 = min(max(cu[b], 0), N), n = min(cu[b + 1], N) - tok0, rows = n * G;
  const int L = min(max(kv_lens[b], 0), W * PAGE);
  const int row = min(row0 + r, rows - 1);             // rows behind the last repeat it
  const int vis = max(L - n + row / G + 1, 0);
  const int least = max(L - n + min(row0, rows - 1) / G + 1, 0), most = max(L - n + min(row0 + 31, rows - 1) / G + 1, 0);
  const int tile_most = max(L - n + min(tile0 + LTILE - 1, rows - 1) / G + 1, 0);
  const bool idle = row0 >= rows;

  bf16x8_t qf[KS];
  {
    const bf16_t* qp = q + ((size_t)(tok0 + row / G) * Hq + (size_t)hk * G + row % G) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const bf16x8_t*>(qp + 16 * s);
#pragma unroll
    for (int s = 0; s < KS; ++s) arrived(qf[s]);
  }
  f32x16_t o[DC];
#pragma unroll
  for (int dc = 0; dc < DC; ++dc)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dc][i] = 0.f;
  float m = -INFINITY, l = 0.f;

  const int npages = (min(tile_most, L) + PAGE - 1) / PAGE;
  const int p0 = (int)((long long)npages * sh.part / ns), p1 = (int)((long long)npages * (sh.part + 1) / ns);
  int ids = 0;                                         // lane i: one of the next 64 pages, and its scales
  float kss = 0.f, vss = 0.f;
  uint4 kr[2], vr[2];                                  // the next two pages' codes, and what goes with them
  float ks[2], vs[2];
  bool bad[2] = {false, false};                        // not a page of the cache: its keys count as masked
  auto fetch = [&](int z, int p) __attribute__((always_inline)) {
    const int at = (p - p0) & 63;
    if (at == 0) {
      ids = table[(size_t)b * W + min(p + lane, npages - 1)];
      const size_t x = (size_t)(ids < 0 || ids >= pages ? 0 : ids) * Hkv + hk;
      kss = kscale[x];
      vss = vscale[x];
      // arrived: a wait here, every 64 pages, not behind the branch, where it would be for the codes on their way too
      asm volatile("" : "+v"(ids), "+v"(kss), "+v"(vss));
      check_scales(kss, vss);
    }
    const int id = __builtin_amdgcn_readlane(ids, at);
    ks[z] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kss), at));
    vs[z] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vss), at));
    bad[z] = id < 0 || id >= pages;
    const size_t ph = ((size_t)(bad[z] ? 0 : id) * Hkv + hk) * (PAGE * D);
    if (t < CHUNKS) {
      kr[z] = *reinterpret_cast<const uint4*>(kc + ph + 16 * t);
      vr[z] = *reinterpret_cast<const uint4*>(vc + ph + 16 * t);
    }
  };
  auto stage = [&](int z, int buf, int p) __attribute__((always_inline)) {
    if (t < CHUNKS) {
      const int kt = t / (D / 16), kch = t % (D / 16) * 2;
      *reinterpret_cast<bf16x8_t*>(&s_k[buf][k_at<D>(kt, kch)]) = widen(kr[z].x, kr[z].y, ks[z]);
      *reinterpret_cast<bf16x8_t*>(&s_k[buf][k_at<D>(kt, kch + 1)]) = widen(kr[z].z, kr[z].w, ks[z]);
      const int dim = t / (PAGE / 16), qk = t % (PAGE / 16), live = bad[z] ? 0 : L - p * PAGE;
      uint4& v = vr[z];
      if (live < PAGE) {                               // slots never written may hold any code, NaN too
        v.x &= live_bytes(16 * qk, live);
        v.y &= live_bytes(16 * qk + 4, live);
        v.z &= live_bytes(16 * qk + 8, live);
        v.w &= live_bytes(16 * qk + 12, live);
      }
      *reinterpret_cast<bf16x8_t*>(&s_v[buf][v_at(dim, 2 * qk)]) = widen(v.x, v.z, vs[z]);
      *reinterpret_cast<bf16x8_t*>(&s_v[buf][v_at(dim, 2 * qk + 1)]) = widen(v.y, v.w, vs[z]);
    }
  };

  auto page = [&](int p, int buf, bool masked) __attribute__((always_inline)) {
    const int key0 = p * PAGE;
    if (!idle && key0 < most) {
      const bf16_t* sk = s_k[buf];
      const bf16_t* sv = s_v[buf];
      f32x16_t s0, s1;
#pragma unroll
      for (int i = 0; i < 16; ++i) s0[i] = 0.f, s1[i] = 0.f;
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(&sk[k_at<D>(r, 2 * st + h)]), qf[st], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(&sk[k_at<D>(32 + r, 2 * st + h)]), qf[st], s1, 0, 0, 0);
      }
      if (masked || key0 + PAGE > least) {
        const int seen = (masked ? 0 : vis - key0) - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if ((i & 3) + 8 * (i >> 2) >= seen) s0[i] = -INFINITY;
          if ((i & 3) + 8 * (i >> 2) + 32 >= seen) s1[i] = -INFINITY;
        }
      }
      float mx = s0[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s0[i]);
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s1[i]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mt = mx * scale_log2;
      if (__ballot(mt > m + 8.f)) {
        const float mnew = fmaxf(m, mt);
        const float alpha = __builtin_amdgcn_exp2f(m - (mnew == -INFINITY ? 0.f : mnew));
        m = mnew;
        l *= alpha;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[dc][i] *= alpha;
      }
      const float base = m == -INFINITY ? 0.f : m;     // nothing seen yet: every p is exp2(-inf) = 0
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s0[i] = __builtin_amdgcn_exp2f(fmaf(s0[i], scale_log2, -base));
        sum += s0[i];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s1[i] = __builtin_amdgcn_exp2f(fmaf(s1[i], scale_log2, -base));
        sum += s1[i];
      }
      l += sum;
      auto pv = [&](const f32x16_t& s, int u) __attribute__((always_inline)) {        // k-step u of the page's four
        bf16x8_t pf;
#pragma unroll
        for (int j = 0; j < 8; ++j) pf[j] = (__bf16)s[8 * (u & 1) + j];
#pragma unroll
        for (int dc = 0; dc < DC; ++dc)
          o[dc] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8_t*>(&sv[v_at(32 * dc + r, 2 * u + h)]), pf, o[dc], 0, 0, 0);
      };
      pv(s0, 0);
      pv(s0, 1);
      pv(s1, 2);
      pv(s1, 3);
    }
  };
  auto fetch_two = [&](int p) __attribute__((always_inline)) {
    if (p < p1) fetch(0, p);
    if (p + 1 < p1) fetch(1, p + 1);
  };
  auto stage_two = [&](int p, int buf) __attribute__((always_inline)) {
    if (p < p1) stage(0, buf, p);
    if (p + 1 < p1) stage(1, buf + 1, p + 1);
  };
  bool now[2];
  if (p0 < p1) {
    fetch_two(p0);
    stage_two(p0, 0);
  }
  now[0] = bad[0], now[1] = bad[1];
  fetch_two(p0 + 2);
  __syncthreads();
  auto two = [&](int p, auto buf) __attribute__((always_inline)) {
    constexpr int B0 = decltype(buf)::value;
    page(p, B0, now[0]);
    const bool second = now[1];
    if (p + 2 < p1) {
      stage_two(p + 2, B0 ^ 2);
      now[0] = bad[0], now[1] = bad[1];
      fetch_two(p + 4);
    }
    if (p + 1 < p1) page(p + 1, B0 + 1, second);
    __syncthreads();
  };
  for (int p = p0; p < p1; p += 4) {
    two(p, std::integral_constant<int, 0>());
    if (p + 2 < p1) two(p + 2, std::integral_constant<int, 2>());
  }

  // Parts of a tile: a wave's rows are joined with the same wave's of the other parts, without the rest of the
  // workgroup.  All but the last to arrive leave (m, l) and O, in the order of their registers, and count themselves
  // done; the last has its own at hand and waits for the others, which are past their arrival and wait for nothing.  It
  // adds the parts in their order, whoever came last.  (Two parts of 39 pages each a tile, 32 / 8 heads: 90 us; with all
  // parts stored in rows of the output, counted once a workgroup and read again 113.  The short requests in a launch of
  // their own in both.)
  if (idle) return;
  l += __shfl_xor(l, 32, 64);
  if (ns > 1) {
    const size_t slot0 = (size_t)sh.slot * Hkv + hk;
    const auto at = [&](int part) { return (slot0 + (size_t)part * Hkv) * (LNT / 64) + w; };
    int *arrived_at = counters + at(0), *done_at = counters + at(1), came = 0;
    if (lane == 0) came = __hip_atomic_fetch_add(arrived_at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__builtin_amdgcn_readfirstlane(came) != ns - 1) {
      float* to = part_o + (at(sh.part) * (D / 4) * 64 + lane) * 2;
#pragma unroll
      for (int dc = 0; dc < DC; ++dc)
#pragma unroll
        for (int i = 0; i < 16; i += 2) put2(to + (8 * dc + i / 2) * 128, o[dc][i], o[dc][i + 1]);
      if (h == 0) put2(part_ml + (at(sh.part) * 32 + r) * 2, m, l);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // as in attn_kernel
      if (lane == 0) __hip_atomic_fetch_add(done_at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return;
    }
    while (__builtin_amdgcn_readfirstlane(__hip_atomic_load(done_at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) != ns - 1)
      __builtin_amdgcn_s_sleep(1);
    asm volatile("" ::: "memory");
    if (lane == 0) {
      __hip_atomic_store(arrived_at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(done_at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    float top = m;
    for (int i = 0; i < ns; ++i)
      if (i != sh.part) top = fmaxf(top, get2(part_ml + (at(i) * 32 + r) * 2).x);
    const float base = top == -INFINITY ? 0.f : top;
    f32x16_t mine[DC];
    float ll = 0.f;
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) {
      mine[dc] = o[dc];
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dc][i] = 0.f;
    }
    for (int i = 0; i < ns; ++i) {
      f32x16_t x[DC];
      float2 e = {m, l};
      if (i != sh.part) {
        e = get2(part_ml + (at(i) * 32 + r) * 2);
        const float* from = part_o + (at(i) * (D / 4) * 64 + lane) * 2;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc)
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float2 y = get2(from + (8 * dc + j / 2) * 128);
            x[dc][j] = y.x;
            x[dc][j + 1] = y.y;
          }
      } else {
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) x[dc] = mine[dc];
      }
      const float f = __builtin_amdgcn_exp2f(e.x - base);
      ll += e.y * f;
#pragma unroll
      for (int dc = 0; dc < DC; ++dc)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[dc][j] += x[dc][j] * f;
    }
    l = ll;
  }
  // lane (r, h) holds dims 32 dc + 8 j + 4 h .. + 4 of its row
  if (row0 + r < rows) {
#pragma unroll
    for (int dc = 0; dc < DC; ++dc)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        store_row(out, f32x4_t{o[dc][4 * j], o[dc][4 * j + 1], o[dc][4 * j + 2], o[dc][4 * j + 3]}, l, row, tok0, G, Hq, hk,
                  D, 32 * dc + 8 * j + 4 * h);
  }
}

#undef MIVGPU_PATTN_ARGS

// All rows in short tiles.  Four waves, two workgroups a CU (or more), against eight, one: 1024 requests of 256 keys, 32 /
// 8 heads, 205 us and 364, 32 of 1000 15.1 and 15.8, 64 of 16 to 4000 50 and 44.
template <int D>
__global__ void __launch_bounds__(64 * SWAVES, D == 64 ? 4 : 2) attn_kernel(const Call c, const Work k) {
  __shared__ ShortLds<D, SWAVES> lds;
  short_part<D, SWAVES>(c, k, INT_MAX, blockIdx.x, lds);
}
// The long requests' workgroups, then the short ones': these start where the first leave a CU
template <int D>
__global__ void __launch_bounds__(LNT, 2) attn_both_kernel(const Call c, const Work longs, const Work shorts) {
  typedef ShortLds<D, LWAVES> Lds;
  __shared__ __attribute__((aligned(16))) bf16_t s_k[4][PAGE * D], s_v[4][PAGE * D];
  if (blockIdx.x < longs.grid) {
    long_part<D>(c, longs, blockIdx.x, s_k, s_v);
  } else if constexpr (sizeof(Lds) <= sizeof(s_k)) {
    short_part<D, LWAVES>(c, shorts, c.upto, blockIdx.x - longs.grid, *reinterpret_cast<Lds*>(s_k));
  } else {
    __shared__ Lds lds;
    short_part<D, LWAVES>(c, shorts, c.upto, blockIdx.x - longs.grid, lds);
  }
}

}  // namespace

extern "C" {

int mivgpu_ops_visible_cus();
static int all_cus() {
  static const int n = mivgpu_ops_visible_cus();
  return n < MAX_CUS ? n : MAX_CUS;
}

// The workspace, for any head size: counters (zero before the first call, left zero), then (m, l) and O of the short
// and, where a call has more than FEW_ROWS rows, of the long tiles' parts.
constexpr long long ZEROED = SHORT_SLOTS + LONG_SLOTS * (LNT / 64);
constexpr long long SHORT_FLOATS = (long long)SHORT_SLOTS * TILE * (2 + 128);
constexpr long long LONG_FLOATS = (long long)LONG_SLOTS * LTILE * (2 + 128);

long long mivgpu_paged_attention_work(int N, int Hq, int Hkv, long long* zeroed) {
  if (N < 0 || Hq <= 0 || Hkv <= 0 || Hkv > MAX_HKV || Hq % Hkv) return -1;
  *zeroed = ZEROED;
  return ZEROED + SHORT_FLOATS + ((long long)N * (Hq / Hkv) > FEW_ROWS ? LONG_FLOATS : 0);
}

// Short workgroups that a call counts on for each CU, and in *fit how many of the kernel's the current GPU's CUs hold
int mivgpu_paged_attention_resident(int head_dim, int longs, int* fit) {
  const void* both = head_dim == 64 ? (const void*)attn_both_kernel<64> : (const void*)attn_both_kernel<128>;
  const void* alone = head_dim == 64 ? (const void*)attn_kernel<64> : (const void*)attn_kernel<128>;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(fit, longs ? both : alone, longs ? LNT : 64 * SWAVES, 0) != hipSuccess)
    return -1;
  return short_resident(longs != 0);
}

// max_new: the most new tokens of a request, or negative if not known
int mivgpu_paged_attention(const void* q, const void* kc, const void* vc, const float* kscale, const float* vscale,
                           const int* table, const int* cu, const int* kv_lens, void* out, float* work, long long floats,
                           int N, int B, int W, int Hq, int Hkv, int head_dim, int pages, int max_new, float scale,
                           hipStream_t s) {
  if (N < 0 || B <= 0 || B > MAX_ROWS || W <= 0 || (long long)W * PAGE > INT_MAX || Hq <= 0 || Hkv <= 0 ||
      Hkv > MAX_HKV || Hq % Hkv || pages <= 0 || (long long)N * (Hq / Hkv) > INT_MAX / 2 ||
      (head_dim != 64 && head_dim != 128))
    return -1;
  if (N == 0) return 0;
  const int G = Hq / Hkv;
  const long long rows = (long long)N * G, some = N < B ? N : B;
  // All rows through the short kernel where no request is long; then it also takes one that is longer than it was
  // said to be.
  const int upto = short_rows(rows);
  const bool longs = rows > upto && (max_new < 0 || (long long)max_new * G > upto);
  if (work == nullptr || floats < ZEROED + SHORT_FLOATS + (longs ? LONG_FLOATS : 0)) return -2;
  // Parts: no more than the tiles there can be and `target` on top (each part but a tile's last is a whole chunk), nor
  // than all chunks of all tiles
  auto grid_of = [&](long long tiles, int target, int chunk) {
    const long long all = tiles * ((W + chunk - 1) / chunk), most = tiles + target;
    return all < most ? all : most;
  };
  const int ltarget = all_cus() / Hkv > 1 ? all_cus() / Hkv : 1;
  long long tiles = rows / TILE + some, each = (long long)N * ((G + TILE - 1) / TILE);
  if (tiles > each) tiles = each;          // a token adds no more tiles than its own rows fill
  if (longs && tiles > some * (upto / TILE)) tiles = some * (upto / TILE);
  // beside long ones short workgroups have eight waves, alone four
  const int waves = longs ? LWAVES : SWAVES, resident = short_resident(longs) * all_cus();
  const int target = resident / Hkv > 1 ? resident / Hkv : 1;
  const long long few = rows / (upto + 1), ltiles = rows / LTILE + (few < some ? few : some);
  const long long parts = grid_of(tiles, target, waves) * Hkv, lparts = grid_of(ltiles, ltarget, LMIN_CHUNK) * Hkv;
  if (tiles * W > INT_MAX || (longs && ltiles * W > INT_MAX) || parts > INT_MAX || lparts > INT_MAX) return -1;
  if (longs && parts + lparts > INT_MAX) return -1;
  const Call c = {(const bf16_t*)q, (const uint8_t*)kc, (const uint8_t*)vc, kscale, vscale, table, cu, kv_lens,
                  (bf16_t*)out, N, B, W, Hq, Hkv, pages, upto, scale * 1.4426950408889634f};
  const Work shorts = {(int*)work, work + ZEROED, work + ZEROED + SHORT_SLOTS * TILE * 2, target, (unsigned)parts};
  float* lml = work + ZEROED + SHORT_FLOATS;
  const Work more = {(int*)work + SHORT_SLOTS, lml, lml + LONG_SLOTS * LTILE * 2, ltarget, (unsigned)lparts};
#define MIVGPU_PATTN(DD)                                                                                              \
  do {                                                                                                                \
    if (longs)                                                                                                        \
      hipLaunchKernelGGL(attn_both_kernel<DD>, dim3((unsigned)(lparts + parts)), dim3(LNT), 0, s, c, more, shorts);   \
    else                                                                                                              \
      hipLaunchKernelGGL(attn_kernel<DD>, dim3((unsigned)parts), dim3(64 * SWAVES), 0, s, c, shorts);                 \
  } while (0)
  if (head_dim == 128) MIVGPU_PATTN(128);
  else MIVGPU_PATTN(64);
#undef MIVGPU_PATTN
  return (int)hipGetLastError();
}

}  // extern "C"
