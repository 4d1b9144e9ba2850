// Attention of a ragged batch of tokens over 8-bit K/V pages (paged.h: layout and scales).
//
// Request b owns the q rows cu[b] .. cu[b+1] (n of them) and kv_lens[b] = L keys; its row i sits at position
// L - n + i and sees the keys up to there.  A row that sees no key gives zeros.
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale (q_i . k_j) - m_i)
// in one pass over the pages with the running maximum m and sum (fp32).
//
// The rows of one kv head's G query heads are flattened (row = token * G + head) and cut into tiles of 16.  A tile's
// pages are split over as many workgroups as keep the chip evenly busy: every workgroup scans the requests' lengths
// (at most 1024: a few a thread) and takes its share of all tiles' pages, so that one long request among short ones
// is cut into more parts and nothing is planned on the host.  In a workgroup four waves take every fourth page and
// join their (m, l, O) in LDS; the parts of a tile leave theirs in the workspace, and the last one to arrive (a
// counter that it sets back to zero) joins them in the order of the parts.  Per page of 64 keys a wave
// computes, with 16x16x32 bf16 MFMAs,
//   S^T (64 keys x 16 rows) = K . Q^T        4 tiles of 16 keys: tile t's row 4a + c is key 16a + 4t + c, so that
//                                            lane (row r, quarter a) ends with the 16 consecutive keys 16a .. 16a+15;
//   O^T (D x 16 rows) += V^T . P^T           whose operands want exactly that: 8 consecutive keys a lane and k-step.
// P never leaves its lane.  e4m3 codes become bf16 with their page's scale in one instruction for two values
// (exact: a code has 4 significant bits and the scale is a power of two).  P is rounded to bf16 (half a step of the
// output's type, before a sum that averages it); scores, m, l and O stay in fp32.
#include "paged.h"

using namespace paged;

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

constexpr int NT = 256, WAVES = 4, TILE = 16;
constexpr int MIN_CHUNK = WAVES;         // pages of a part: at least one for each wave

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

// a row's four values of head dimension d .. d+3; a row that saw no key (l = 0) gives zeros
__device__ __forceinline__ void store_row(bf16_t* out, f32x4_t o, float l, int row, int tok0, int G, int Hq, int hk, int D,
                                          int d) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bf16_t* at = out + ((size_t)(tok0 + row / G) * Hq + (size_t)hk * G + row % G) * D + d;
  *reinterpret_cast<uint2*>(at) = make_uint2(pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv));
}

template <int D>
__global__ void __launch_bounds__(NT)
attn_kernel(const bf16_t* __restrict__ q, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
            const float* __restrict__ kscale, const float* __restrict__ vscale, const int* __restrict__ table,
            const int* __restrict__ cu, const int* __restrict__ kv_lens, bf16_t* __restrict__ out,
            int* __restrict__ counters, float* __restrict__ part_ml, float* __restrict__ part_o, int N, int B, int W,
            int Hq, int Hkv, int pages, int target, float scale_log2) {
  constexpr int KU = D / 64;              // 16-byte chunks of a K row per lane
  constexpr int DT = D / 16;              // output tiles
  __shared__ long long red[WAVES];
  __shared__ int s_b, s_tile, s_part, s_ns, s_first;
  __shared__ float s_m[WAVES][TILE], s_l[WAVES][TILE];
  __shared__ __attribute__((aligned(16))) float s_o[WAVES][TILE][D + 4];
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 15, a = lane >> 4;
  const int G = Hq / Hkv, hk = blockIdx.y;

  // which request, tile and part: the workgroup's index among all tiles' parts
  {
    constexpr int PER = MAX_ROWS / NT;
    int tiles[PER], np[PER];
    long long sum = 0, all;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = t * PER + i;
      tiles[i] = np[i] = 0;
      if (b < B) {
        const int n = max(min(cu[b + 1], N) - min(max(cu[b], 0), N), 0);
        tiles[i] = (n * G + TILE - 1) / TILE;
        np[i] = (min(max(kv_lens[b], 0), W * PAGE) + PAGE - 1) / PAGE;
      }
      sum += (long long)tiles[i] * np[i];
    }
    block_scan<NT>(sum, red, &all);
    const int chunk = (int)max((all + target - 1) / target, (long long)MIN_CHUNK);
    sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      np[i] = max((np[i] + chunk - 1) / chunk, 1);       // now parts of a tile
      sum += (long long)tiles[i] * np[i];
    }
    long long at = block_scan<NT>(sum, red, &all) - sum;
    if ((long long)blockIdx.x >= all) return;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const long long mine = (long long)tiles[i] * np[i];
      if (blockIdx.x >= at && blockIdx.x < at + mine) {
        const int x = (int)(blockIdx.x - at);
        s_b = t * PER + i;
        s_tile = x / np[i];
        s_part = x % np[i];
        s_ns = np[i];
        s_first = (int)blockIdx.x - s_part;
      }
      at += mine;
    }
    __syncthreads();
  }
  const int b = s_b, row0 = s_tile * TILE, ns = s_ns, first = s_first;
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
  const int p0 = (int)((long long)npages * s_part / ns), p1 = (int)((long long)npages * (s_part + 1) / ns);
  for (int p = p0 + w; p < p1; p += WAVES) {
    int page = table[(size_t)b * W + p];
    const bool bad = page < 0 || page >= pages;   // its keys count as masked
    page = bad ? 0 : page;
    const size_t ph = (size_t)page * Hkv + hk;
    const uint8_t* kp = kc + ph * PAGE * D;
    const uint8_t* vp = vc + ph * PAGE * D;
    const float ks = kscale[ph], vs = vscale[ph];

    f32x4_t s[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      s[tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      const uint8_t* kr = kp + (size_t)(16 * (r >> 2) + 4 * tt + (r & 3)) * D;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const uint4 c = *reinterpret_cast<const uint4*>(kr + 16 * (a + 4 * u));
        s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(c.x, c.y, ks), qf[u][0], s[tt], 0, 0, 0);
        s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(c.z, c.w, ks), qf[u][1], s[tt], 0, 0, 0);
      }
    }
    const int key0 = p * PAGE;
    const int live = bad ? 0 : L - key0;          // keys of the page that were written
    if (bad || key0 + PAGE > least) {
      const int seen = bad ? 0 : vis - key0;
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
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      uint4 c = *reinterpret_cast<const uint4*>(vp + (size_t)(16 * i + r) * PAGE + 16 * a);
      if (live < PAGE) {                          // slots never written may hold any code, NaN too
        c.x &= live_bytes(16 * a, live);
        c.y &= live_bytes(16 * a + 4, live);
        c.z &= live_bytes(16 * a + 8, live);
        c.w &= live_bytes(16 * a + 12, live);
      }
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(c.x, c.y, vs), pf[0], o[i], 0, 0, 0);
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(c.z, c.w, vs), pf[1], o[i], 0, 0, 0);
    }
  }

  // join the waves
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (a == 0) s_m[w][r] = m, s_l[w][r] = l;
#pragma unroll
  for (int i = 0; i < DT; ++i) *reinterpret_cast<f32x4_t*>(&s_o[w][r][16 * i + 4 * a]) = o[i];
  __syncthreads();
  const size_t slot0 = (size_t)first * Hkv + hk, slot_step = Hkv;     // the tile's parts in the workspace
  const size_t slot = slot0 + s_part * slot_step;
  for (int x = t; x < TILE * (D / 4); x += NT) {
    const int rr = x / (D / 4), d = x % (D / 4) * 4;
    if (row0 + rr >= rows) continue;
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
      store_row(out, oo, ll, row0 + rr, tok0, G, Hq, hk, D, d);
    } else {
      put2(part_o + (slot * TILE + rr) * D + d, oo[0], oo[1]);
      put2(part_o + (slot * TILE + rr) * D + d + 2, oo[2], oo[3]);
      if (d == 0) put2(part_ml + (slot * TILE + rr) * 2, mm, ll);
    }
  }
  if (ns == 1) return;

  // The last part of the tile to arrive joins them all.  The parts are stored and loaded past the XCDs' own caches
  // (put2 / get2); each wave waits for its stores before the workgroup counts itself.  A release fence here instead
  // writes back the whole of the XCD's L2 for every part: 110 us against 20 for 32 rows of 1024 keys.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (t == 0) s_tile = __hip_atomic_fetch_add(&counters[slot0], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_tile != ns - 1) return;
  if (t == 0) __hip_atomic_store(&counters[slot0], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int x = t; x < TILE * (D / 4); x += NT) {
    const int rr = x / (D / 4), d = x % (D / 4) * 4;
    if (row0 + rr >= rows) continue;
    float mm = -INFINITY;
    for (int i = 0; i < ns; ++i) mm = fmaxf(mm, get2(part_ml + ((slot0 + i * slot_step) * TILE + rr) * 2).x);
    const float base = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    f32x4_t oo = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < ns; ++i) {
      const size_t at = (slot0 + i * slot_step) * TILE + rr;
      const float2 ml = get2(part_ml + at * 2), x01 = get2(part_o + at * D + d), x23 = get2(part_o + at * D + d + 2);
      const float f = __builtin_amdgcn_exp2f(ml.x - base);
      ll += ml.y * f;
      oo += f32x4_t{x01.x, x01.y, x23.x, x23.y} * f;
    }
    store_row(out, oo, ll, row0 + rr, tok0, G, Hq, hk, D, d);
  }
}

// No more tiles than this, whatever the lengths; parts: `target` more, as each part but a tile's last is a full chunk.
long long most_tiles(long long N, int B, int G) { return N * G / TILE + (N < B ? N : B); }

}  // namespace

extern "C" {

// Parts of a call (grid and workspace slots per kv head) for N tokens of B requests on a GPU of `cus` CUs.
static long long most_parts(long long N, int B, int G, int Hkv, int cus, int* target) {
  *target = (4 * cus + Hkv - 1) / Hkv;     // four workgroups fit a CU
  return most_tiles(N, B, G) + *target;
}

int mivgpu_ops_visible_cus();
static int all_cus() {
  static const int n = mivgpu_ops_visible_cus();
  return n;
}

// counters (ints, zero before the first call, left zero), then (m, l) and O of the parts; in floats
long long mivgpu_paged_attention_work(int N, int B, int Hq, int Hkv, int head_dim, long long* zeroed) {
  if (N < 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return -1;
  int target;
  const long long parts = most_parts(N, B, Hq / Hkv, Hkv, all_cus(), &target) * Hkv;
  *zeroed = (parts + 3) / 4 * 4;
  return *zeroed + parts * TILE * (2 + head_dim);
}

int mivgpu_paged_attention(const void* q, const void* kc, const void* vc, const float* kscale, const float* vscale,
                           const int* table, const int* cu, const int* kv_lens, void* out, float* work, long long floats,
                           int N, int B, int W, int Hq, int Hkv, int head_dim, int pages, float scale, hipStream_t s) {
  if (N < 0 || B <= 0 || B > MAX_ROWS || W <= 0 || (long long)W * PAGE > INT_MAX || Hq <= 0 || Hkv <= 0 || Hq % Hkv ||
      Hkv > 65535 || pages <= 0 || (long long)N * (Hq / Hkv) > INT_MAX / 2)
    return -1;
  if (N == 0) return 0;
  const int G = Hq / Hkv;
  long long zeroed;
  const long long need = mivgpu_paged_attention_work(N, B, Hq, Hkv, head_dim, &zeroed);
  if (work == nullptr || floats < need) return -2;
  int target;
  const long long parts = most_parts(N, B, G, Hkv, all_cus(), &target);
  if (parts > INT_MAX) return -1;
  float* ml = work + zeroed;
  float* po = ml + parts * Hkv * TILE * 2;
  const dim3 grid((unsigned)parts, Hkv);
  const float sl2 = scale * 1.4426950408889634f;
#define MIVGPU_PATTN(DD)                                                                                              \
  hipLaunchKernelGGL(attn_kernel<DD>, grid, dim3(NT), 0, s, (const bf16_t*)q, (const uint8_t*)kc, (const uint8_t*)vc, \
                     kscale, vscale, table, cu, kv_lens, (bf16_t*)out, (int*)work, ml, po, N, B, W, Hq, Hkv, pages,   \
                     target, sl2)
  if (head_dim == 128) MIVGPU_PATTN(128);
  else if (head_dim == 64) MIVGPU_PATTN(64);
  else return -1;
#undef MIVGPU_PATTN
  return (int)hipGetLastError();
}

}  // extern "C"
