// Attention over the paged 8-bit KV cache on sm_100a: the form for few query rows (a decode step).
//
// Query row (token t of sequence s, head h) stands at position p = start[s] + t and sees key j of its
// own sequence when j <= p and (no window, or j > p - window, or j < sinks):
//   o = sum_j softmax_j(q . k_j s_k(page of j) scale) v_j s_v(page of j)
// with k_j, v_j the cache's integers. A row that sees nothing (an idle slot, window 0 without sinks)
// is zero.
//
// k_paged_token: at most 16 rows share a KV head's keys (its query heads times the new tokens), so the
// bound is the cache's bytes from HBM. The visible keys of all (sequence, KV head) units, in tiles of 64,
// form one line that is cut into equal parts, one per resident CTA: any raggedness is balanced, and a
// unit that lies in several parts is joined by the last CTA to finish it, in key order, so the bits do
// not depend on which that is. A unit is kUnitCost tiles longer than its keys, for its queries, its four
// warps' sums and its output: with equal numbers of tiles the CTAs with many short units ended last (32
// sequences of 1 to 8192, 32 heads on 8: 71.7 us; with 3, 5 and 8 tiles a unit 59.4, 59.2 and 58.5; 16
// sequences with 4 drafts each 32.4, 27.5, 26.7 and 27.3). Per CTA one warp fetches pages (TMA, 128-byte swizzle, a ring of 16 KiB
// stages, page ids and scales eight tiles ahead) and four warps compute, 16 keys of a tile each:
//   S^T = K Q^T and O^T = V^T P^T as mma m16n8k16 in fp16 with float32 sums. The integers are exact in
//   fp16 (a byte permute and one subtraction a pair); a query row is scaled by a power of two that puts
//   its largest value at 2^14, which keeps 11 bits of everything within 2^-28 of it; the page scales and
//   1/sqrt(d) multiply the float32 sums. Keys lie on the M side, so the conversion serves every query
//   row, and the order of dims and keys inside a fragment is chosen so that a thread reads 16-byte runs
//   (conflict-free under the swizzle) and no shuffle moves K or V; P is transposed by movmatrix.
//   Weights are 2^(score - m) s_v 2^(m - v), with m 7 below the row's maximum when it was last looked at and v as far
//   below its largest score + log2 s_v; both are raised only when a key passes one by 15, so most tiles neither reduce
//   over lanes nor rescale. They stay below 2^15, inside fp16, which keeps 11 bits of those down to 2^-21 of the row's
//   largest contribution, however far apart the pages' scales are (2^-14 without the 7).
//
// Measured on B200 (a graph of calls): one sequence of 131071 tokens, 32 heads on 8: 58 us, 4.6 TB/s; 32
// sequences of up to 8192: 59 us, 4.8 TB/s; 64 with a window of 1024: 40 us, 3.2 TB/s. A share's first tile comes
// 6 us after the launch (metadata, pages, scales, the copy), and a unit's end takes 3 to 5 us (four warps' sums,
// the part's write, the count, the join), which three CTAs an SM hide in part.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <mutex>
#include <set>
#include <utility>

#include "det_math.cuh"
#include "paged.cuh"
#include "uwc_host.h"

namespace {

using namespace paged;

constexpr int kWarps = 4;                    // consumer warps
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kTile = 64;                    // keys per stage
constexpr int kGroups = kTile / 16;          // 16-key groups: one warp's share, always inside one page
constexpr int kStageBytes = 2 * kTile * kHd; // keys, then values
constexpr float kHeadroom = 7.f, kRaise = 8.f;   // log2: of the largest weight when m and v are set; by which a later one may pass it
constexpr float kLow = 116.f;                // v is no lower than m by more: 2^(m - v) is finite, 2^(v - m) not 0
constexpr int kBatch = 8;                    // tiles whose page ids and scales are fetched at once
constexpr int kUnitCost = 5;                 // what a unit costs beside its tiles, in tiles
constexpr int kMinTiles = 4;                 // the least tiles of a CTA's share of the line (a join costs about as much)

// rows: 8 NT. Stages and CTAs per SM: about 200 KB of loads in flight on an SM either way.
template <int NT>
struct TokenCfg {
  static constexpr int kStages = NT == 1 ? 4 : 5;
  static constexpr int kCtas = NT == 1 ? 3 : 2;
  static constexpr int kCombine = 2 * 8 * NT * kHd * 4;            // two warps' O
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kCombine;
};

struct TokenArgs {
  AttnArgs a;
  float* part_o;           // (2 grid, 8 NT, 128): a CTA's two partial units, unnormalized
  float2* part_ml;         // (2 grid, 8 NT): m (log2), sum
  uint32_t* counters;      // (grid): finished parts of the unit that starts in this CTA; left zero
  int withhold;            // 1: every other CTA copies no pages (a test's hook), so that its waits run out
};

// A sequence's tiles: one pass over the keys for all its new tokens.
struct Unit : Keys<kTile> {
  Span sp;
  __device__ __forceinline__ Unit(const AttnArgs& a, const Span& s) : Keys<kTile>(a, s, 0, s.n - 1), sp(s) {
    if (s.n <= 0) total = 0;
  }
  __device__ __forceinline__ int cost() const { return total > 0 ? kUnitCost + total : 0; }   // its length on the line
};
__device__ __forceinline__ Unit unit_of(const AttnArgs& a, int s) { return Unit(a, span_of(a.b, a.c.ps, s)); }

// This CTA's part of the line: `count` steps from step `at` of KV head `head` of sequence `seq` on. A unit's steps
// are kUnitCost for itself, then one a tile.
struct Part {
  int seq, head, at;
  uint32_t per;                    // steps of a part (2^32 of them would be days of work)
  long long count;
};
// Every warp finds it for itself: lanes take sequences, two passes (the sum, then the place).
__device__ __forceinline__ Part find_part(const AttnArgs& a) {
  const int lane = threadIdx.x & 31, S = a.b.seqs;
  long long sum = 0;
  int most = 0;
#pragma unroll 1
  for (int s = lane; s < S; s += 32) {
    const int t = unit_of(a, s).cost();
    sum += t;
    most = max(most, t);
  }
  sum = warp_sumll(sum);
  most = __reduce_max_sync(0xffffffffu, most);
  Part p = {};
  sum *= a.c.Hkv;
  p.per = (uint32_t)max((sum + gridDim.x - 1) / gridDim.x, (long long)min(kMinTiles + kUnitCost, most));
  const long long first = (long long)p.per * blockIdx.x;
  p.count = min((long long)p.per, sum - first);
  if (p.count <= 0) return p;
  long long before = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < S; s0 += 32) {
    const long long t = s0 + lane < S ? (long long)unit_of(a, s0 + lane).cost() * a.c.Hkv : 0;
    long long inc = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + inc > first);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const long long at = first - (before + __shfl_sync(0xffffffffu, inc - t, l));
      const int steps = (int)(__shfl_sync(0xffffffffu, t, l) / a.c.Hkv);
      p.seq = s0 + l;
      p.head = (int)(at / steps);
      p.at = (int)(at % steps);
      return p;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  p.count = 0;
  return p;
}

// ---- fragments
__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, const uint32_t* b, const float* c) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

template <typename T, int NT>
__global__ void __launch_bounds__(kThreads, TokenCfg<NT>::kCtas)
    k_paged_token(const TokenArgs ta, const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV) {
  using Cfg = TokenCfg<NT>;
  constexpr int ST = Cfg::kStages, R = 8 * NT;
  const AttnArgs& a = ta.a;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>(((uintptr_t)sm_raw + 1023) & ~(uintptr_t)1023);
  float* comb = reinterpret_cast<float*>(sm + ST * kStageBytes);
  __shared__ uint64_t full[ST], empty[ST];
  __shared__ float2 s_scale[ST][kGroups];
  __shared__ int s_seen[ST][kGroups];
  __shared__ float s_m[kWarps][R], s_l[kWarps][R];
  __shared__ int s_abort, s_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < ST; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    s_abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&mapK);
    tma_prefetch_desc(&mapV);
  }
  if (blockIdx.x == 0 && warp == kWarps)
#pragma unroll 1
    for (int s = lane; s < a.b.seqs; s += 32)
      if (span_of(a.b, a.c.ps, s).bad) set_status(a.status, UWC_DEV_RANGE);
  const Part part = find_part(a);
  __syncthreads();
  if (part.count <= 0) return;
  const int Hkv = a.c.Hkv, G = a.H / Hkv, ps = a.c.ps;

  if (warp == kWarps) {
    // ---------------------------------------------------------------- the fetching warp
    const int box = min(ps, kTile), per_box = box / 16;      // keys, 16-key groups a TMA box
    const int grp = lane & (kGroups - 1);
    int it = 0;
    int s = part.seq, h = part.head, u0 = part.at;
    long long left = part.count;
#pragma unroll 1
    while (left > 0) {
      const Unit k = unit_of(a, s);
#pragma unroll 1
      for (; h < Hkv && left > 0; h++, u0 = 0) {
        const int u1 = (int)min((long long)k.cost(), u0 + left), t0 = max(u0 - kUnitCost, 0), end = u1 - kUnitCost;
        // page ids and scales of eight tiles, one 16-key group a lane
        auto fetch = [&](int tb, int& page, float2& sc, int& j0) {
          const int i = tb + lane / kGroups;
          j0 = k.key(i) + 16 * grp;
          page = -1;
          sc = make_float2(0.f, 0.f);
          if (i < end && k.seen(j0, 16)) {
            page = page_at(a.b, a.c, s, j0 >> a.c.lg);
            if (page < 0) set_status(a.status, UWC_DEV_RANGE);
            else sc = make_float2(a.c.sk[(size_t)page * Hkv + h], a.c.sv[(size_t)page * Hkv + h]);
          }
        };
        int page = -1, j0 = 0, npage = -1, nj0 = 0;
        float2 sc = make_float2(0.f, 0.f), nsc = sc;
        if (end > t0) fetch(t0, page, sc, j0);
#pragma unroll 1
        for (int tb = t0; tb < end; tb += kBatch) {
          if (tb + kBatch < end) fetch(tb + kBatch, npage, nsc, nj0);
#pragma unroll 1
          for (int i = 0; i < kBatch && tb + i < end; i++, it++) {
            const int st = it % ST;
            const uint32_t use = (uint32_t)(it / ST);
            // A wait that ran out in another warp counts here too: its stage was given back without its copies, so
            // the barrier's phase is not over and takes no second arrival.
            if (use > 0 && (!__all_sync(0xffffffffu, mbar_wait(&empty[st], (use - 1) & 1, &s_abort, a.status)) ||
                            __any_sync(0xffffffffu, *static_cast<volatile int*>(&s_abort)))) {
              // give up: let the copies in flight land (bounded), then leave
#pragma unroll 1
              for (int x = max(0, it - ST); x < it; x++)
#pragma unroll 1
                for (int n = 0; n < (1 << 16) && !mbar_try_wait(&full[x % ST], (uint32_t)(x / ST) & 1); n++) {
                }
              return;
            }
            const bool mine = lane / kGroups == i;
            if (mine) {
              s_scale[st][grp] = sc;
              s_seen[st][grp] = page >= 0;
            }
            // a box is fetched when one of its groups is seen; its lanes agree on the page
            const unsigned seen = __ballot_sync(0xffffffffu, mine && page >= 0) >> (i * kGroups);
            const unsigned in_box = ((1u << per_box) - 1) << (grp / per_box * per_box);
            const bool issue = mine && grp % per_box == 0 && (seen & in_box);
            const int from = __ffs(seen & in_box) - 1;
            const int bpage = __shfl_sync(0xffffffffu, page, from >= 0 ? i * kGroups + from : lane);
            const int boxes = __popc(__ballot_sync(0xffffffffu, issue));
            __syncwarp();
            if (elect_one()) mbar_expect_tx(&full[st], (uint32_t)(boxes * 2 * box * kHd));
            __syncwarp();
            if (issue && !(ta.withhold & blockIdx.x & 1)) {
              const int y = (bpage * Hkv + h) * ps + (j0 & (ps - 1));
              uint8_t* dst = sm + st * kStageBytes + grp * 16 * kHd;
              tma_load_2d(dst, &mapK, &full[st], 0, y);
              tma_load_2d(dst + kTile * kHd, &mapV, &full[st], 0, y);
            }
          }
          page = npage;
          sc = nsc;
          j0 = nj0;
        }
        left -= u1 - u0;
      }
      s++;
      h = 0;
      u0 = 0;
#pragma unroll 1
      while (left > 0 && s < a.b.seqs && unit_of(a, s).total == 0) s++;
      if (s >= a.b.seqs) break;
    }
    return;
  }

  // ------------------------------------------------------------------ the computing warps
  const int g = lane >> 2, t = lane & 3;
  const uint32_t sm0 = smem_u32(sm);
  // byte offsets of this thread's 16-byte runs inside a stage
  const uint32_t koff0 = (16 * warp + g) * kHd + (((2 * t) ^ g) << 4), koff1 = (16 * warp + g) * kHd + (((2 * t + 1) ^ g) << 4);
  const uint32_t voff0 = kTile * kHd + (16 * warp + 2 * t) * kHd + ((g ^ (2 * t)) << 4);
  const uint32_t voff1 = kTile * kHd + (16 * warp + 2 * t + 1) * kHd + ((g ^ (2 * t + 1)) << 4);
  int it = 0;
  int s = part.seq, h = part.head, u0 = part.at;
  long long left = part.count;
#pragma unroll 1
  while (left > 0) {
    const Unit k = unit_of(a, s);
    const int rows = k.sp.n * G;
#pragma unroll 1
    for (; h < Hkv && left > 0; h++, u0 = 0) {
      const int u1 = (int)min((long long)k.cost(), u0 + left), t0 = max(u0 - kUnitCost, 0), end = u1 - kUnitCost;
      left -= u1 - u0;
      if (end <= t0) continue;                           // none of its tiles
      // ---- this unit's queries: row r = token r / G, head r % G; thread (g, t) has dims 32 t .. of rows g + 8 n
      uint32_t qf[NT][8][2];
      float qmul[NT][2];
      int qpos[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const int r = g + 8 * n;
        float x[32], mx = 0.f;
        if (r < rows) {
          const T* q = reinterpret_cast<const T*>(a.q) + (long long)(k.sp.row0 + r / G) * a.q_tok + (long long)(h * G + r % G) * a.q_head + 32 * t;
          const uint4* qv = reinterpret_cast<const uint4*>(q);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint4 w = __ldg(qv + i);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float2 f = two_f(u[j], T());
              x[8 * i + 2 * j] = f.x;
              x[8 * i + 2 * j + 1] = f.y;
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i++) x[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 32; i++) mx = fmaxf(mx, fabsf(x[i]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = row_exponent(mx);
        const float up = pow2i(e);
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const __half2 hh = __floats2half2_rn(x[4 * i + 2 * j] * up, x[4 * i + 2 * j + 1] * up);
            qf[n][i][j] = *reinterpret_cast<const uint32_t*>(&hh);
          }
        // scores have the rows as columns: this thread's are 2 t and 2 t + 1 (+ 8 n)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const int ec = __shfl_sync(0xffffffffu, e, (2 * t + c) * 4);
          const int rc = 8 * n + 2 * t + c;
          qmul[n][c] = a.scale * kLog2OfE * pow2i(-ec);
          qpos[n][c] = rc < rows ? k.sp.start + rc / G : -1;
        }
      }
      float m[NT][2], v[NT][2], unit[NT][2], l[NT][2], o[NT][8][4];   // unit: 2^(m - v)
#pragma unroll
      for (int n = 0; n < NT; n++) {
        m[n][0] = m[n][1] = v[n][0] = v[n][1] = kNoMax;
        l[n][0] = l[n][1] = unit[n][0] = unit[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) o[n][i][j] = 0.f;
      }
      // ---- the tiles
#pragma unroll 1
      for (int i = t0; i < end; i++, it++) {
        const int st = it % ST;
        // after a wait that ran out the warps run through their schedule without computing
        const bool there = __all_sync(0xffffffffu, mbar_wait(&full[st], (uint32_t)(it / ST) & 1, &s_abort, a.status));
        const int j0 = k.key(i) + 16 * warp;
        if (there && s_seen[st][warp]) {
          const float2 sc = s_scale[st][warp];
          const float lv = __log2f(fabsf(sc.y));
          const uint32_t base = sm0 + st * kStageBytes;
          uint4 kw[4];
          kw[0] = lds128(base + koff0);
          kw[1] = lds128(base + koff1);
          kw[2] = lds128(base + koff0 + 8 * kHd);
          kw[3] = lds128(base + koff1 + 8 * kHd);
          float sa[NT][4];
#pragma unroll
          for (int n = 0; n < NT; n++) sa[n][0] = sa[n][1] = sa[n][2] = sa[n][3] = 0.f;
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const uint32_t lo[4] = {kw[c].x, kw[c].y, kw[c].z, kw[c].w};
            const uint32_t hi[4] = {kw[2 + c].x, kw[2 + c].y, kw[2 + c].z, kw[2 + c].w};
#pragma unroll
            for (int w = 0; w < 4; w++) {
              const uint32_t x = lo[w] ^ 0x80808080u, y = hi[w] ^ 0x80808080u;
              const uint32_t af[4] = {i8_half2(x, 0x4140), i8_half2(y, 0x4140), i8_half2(x, 0x4342), i8_half2(y, 0x4342)};
#pragma unroll
              for (int n = 0; n < NT; n++) mma_f16(sa[n], af, qf[n][4 * c + w], sa[n]);
            }
          }
          uint4 vw[4];
          vw[0] = lds128(base + voff0);
          vw[1] = lds128(base + voff1);
          vw[2] = lds128(base + voff0 + 8 * kHd);
          vw[3] = lds128(base + voff1 + 8 * kHd);
          // ---- scores (log2): keys j0 + g (sa 0, 1) and j0 + g + 8 (sa 2, 3)
          bool over = false;
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
              const float f = qmul[n][c] * sc.x;
              sa[n][c] *= f;
              sa[n][2 + c] *= f;
            }
          if (!k.full(a, j0, 16)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
              for (int x = 0; x < 4; x++) {
                const int j = j0 + g + 8 * (x >> 1), p = qpos[n][x & 1];
                if (!sees(a, p, j)) sa[n][x] = -INFINITY;
              }
          }
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int x = 0; x < 4; x++) over |= sa[n][x] > fminf(m[n][x & 1], v[n][x & 1] - lv) + (kHeadroom + kRaise);
          if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
              for (int c = 0; c < 2; c++) {
                float x = fmaxf(sa[n][c], sa[n][2 + c]);
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                x -= kHeadroom;
                const float m2 = fmaxf(x, m[n][c]), v2 = fmaxf(fmaxf(x + lv, v[n][c]), m2 - kLow);
                const float f = exp2_fast(v[n][c] - v2);
                l[n][c] *= exp2_fast(m[n][c] - m2);
                m[n][c] = m2;
                v[n][c] = v2;
                unit[n][c] = exp2_fast(m2 - v2);
#pragma unroll
                for (int d = 0; d < 8; d++) {
                  o[n][d][c] *= f;
                  o[n][d][2 + c] *= f;
                }
              }
          }
          uint32_t pf[NT][2];
#pragma unroll
          for (int n = 0; n < NT; n++) {
            // (a page that a row does not see may make its factor infinite: the row's weights there are 0)
            const float by[2] = {fminf(sc.y * unit[n][0], FLT_MAX), fminf(sc.y * unit[n][1], FLT_MAX)};
#pragma unroll
            for (int x = 0; x < 4; x++) {
              sa[n][x] = exp2_fast(sa[n][x] - m[n][x & 1]);
              l[n][x & 1] += sa[n][x];
              sa[n][x] *= by[x & 1];
            }
            const __half2 p0 = __floats2half2_rn(sa[n][0], sa[n][1]), p1 = __floats2half2_rn(sa[n][2], sa[n][3]);
            pf[n][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&p0));
            pf[n][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&p1));
          }
          // ---- O^T += V^T P^T: dims 16 g + 2 i and 16 g + 2 i + 1 are rows g and g + 8 of product i
          const uint32_t r0[4] = {vw[0].x, vw[0].y, vw[0].z, vw[0].w}, r1[4] = {vw[1].x, vw[1].y, vw[1].z, vw[1].w};
          const uint32_t r2[4] = {vw[2].x, vw[2].y, vw[2].z, vw[2].w}, r3[4] = {vw[3].x, vw[3].y, vw[3].z, vw[3].w};
#pragma unroll
          for (int w = 0; w < 4; w++) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
              const uint32_t sel = y ? 0x7362 : 0x5140;
              const uint32_t u = __byte_perm(r0[w], r1[w], sel) ^ 0x80808080u, v = __byte_perm(r2[w], r3[w], sel) ^ 0x80808080u;
              const uint32_t af[4] = {i8_half2(u, 0x4140), i8_half2(u, 0x4342), i8_half2(v, 0x4140), i8_half2(v, 0x4342)};
#pragma unroll
              for (int n = 0; n < NT; n++) mma_f16(o[n][2 * w + y], af, pf[n], o[n][2 * w + y]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
      }
      // ---- the four warps' parts of the unit
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float x = l[n][c];
          x += __shfl_xor_sync(0xffffffffu, x, 4);
          x += __shfl_xor_sync(0xffffffffu, x, 8);
          x += __shfl_xor_sync(0xffffffffu, x, 16);
          l[n][c] = x;
          if (g == 0) {
            s_m[warp][8 * n + 2 * t + c] = m[n][c];
            s_l[warp][8 * n + 2 * t + c] = x;
          }
        }
      named_bar_sync(1, kWarps * 32);
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const int r = 8 * n + 2 * t + c;
          float M = s_m[0][r];
#pragma unroll
          for (int w = 1; w < kWarps; w++) M = fmaxf(M, s_m[w][r]);
          float L = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; w++) L += s_l[w][r] * exp2_fast(s_m[w][r] - M);
          const float f = exp2_fast(v[n][c] - M);        // to the units of M
          m[n][c] = M;
          l[n][c] = L;
#pragma unroll
          for (int d = 0; d < 8; d++) {
            o[n][d][c] *= f;
            o[n][d][2 + c] *= f;
          }
        }
      // warps 2, 3 onto 0, 1, then 1 onto 0; row r's dims 16 g .. 16 g + 15 lie in 16 values of a thread
      auto put = [&](float* dst) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int c = 0; c < 2; c++)
#pragma unroll
            for (int d = 0; d < 8; d++)
              reinterpret_cast<float2*>(dst + (8 * n + 2 * t + c) * kHd + 16 * g)[(d + t + 4 * c) & 7] = make_float2(o[n][d][c], o[n][d][2 + c]);
      };
      auto add = [&](const float* src) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int c = 0; c < 2; c++)
#pragma unroll
            for (int d = 0; d < 8; d++) {
              const float2 x = reinterpret_cast<const float2*>(src + (8 * n + 2 * t + c) * kHd + 16 * g)[(d + t + 4 * c) & 7];
              o[n][d][c] += x.x;
              o[n][d][2 + c] += x.y;
            }
      };
      // onto warp 0, one warp after the other (a rolled loop: a CTA comes here once or twice, and straight-line
      // code would be fetched for as long as it runs)
#pragma unroll 1
      for (int w = 1; w <= kWarps; w++) {
        if (warp == w) put(comb + (w & 1) * R * kHd);
        if (warp == 0 && w > 1) add(comb + ((w - 1) & 1) * R * kHd);
        named_bar_sync(1, kWarps * 32);
      }
      const bool whole = t0 == 0 && end == k.total;
      // parts of this unit lie in CTAs b0 .. b1: its tiles before t0 in those before this one, `per` steps each,
      // those from `end` on in those after it
      const int b0 = blockIdx.x - (t0 > 0 ? (uint32_t)(t0 - 1) / part.per + 1 : 0);
      const int b1 = blockIdx.x + (end < k.total ? (uint32_t)(k.total - end - 1) / part.per + 1 : 0);
      if (warp == 0) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const int r = 8 * n + 2 * t + c;
            if (r >= rows) continue;
            if (whole) {
              const float inv = l[n][c] == 0.f ? 0.f : 1.f / l[n][c];
              T* out = reinterpret_cast<T*>(a.out) + ((size_t)(k.sp.row0 + r / G) * a.H + h * G + r % G) * kHd + 16 * g;
              float x[16];
#pragma unroll
              for (int d = 0; d < 8; d++) {
                x[2 * d] = o[n][d][c] * inv;
                x[2 * d + 1] = o[n][d][2 + c] * inv;
              }
              uint32_t w[8];
#pragma unroll
              for (int d = 0; d < 8; d++) w[d] = pack2(x[2 * d], x[2 * d + 1], T());
              reinterpret_cast<uint4*>(out)[0] = make_uint4(w[0], w[1], w[2], w[3]);
              reinterpret_cast<uint4*>(out)[1] = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
              const size_t slot = (size_t)(2 * blockIdx.x + (t0 == 0)) * R + r;
              float4* po = reinterpret_cast<float4*>(ta.part_o + slot * kHd + 16 * g);
#pragma unroll
              for (int d = 0; d < 4; d++)
                po[d] = make_float4(o[n][2 * d][c], o[n][2 * d][2 + c], o[n][2 * d + 1][c], o[n][2 * d + 1][2 + c]);
              if (g == 0) ta.part_ml[slot] = make_float2(m[n][c], l[n][c]);
            }
          }
        if (!whole) {
          // the last of this unit's CTAs to get here joins its parts
          __threadfence();
          __syncwarp();
          if (lane == 0) {
            const uint32_t done = atomicAdd(&ta.counters[b0], 1u);
            s_last = done == (uint32_t)(b1 - b0);
            if (s_last) ta.counters[b0] = 0;
            __threadfence();
          }
        }
      }
      if (!whole) {
        named_bar_sync(1, kWarps * 32);
        if (s_last) {
          __threadfence();
#pragma unroll 1
          for (int r = warp; r < rows; r += kWarps) {
            auto slot = [&](int b) { return (size_t)(2 * b + (b == b0)) * R + r; };
            float M = kNoMax, L = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            // one pass, eight parts' loads in flight (a part past b1 loads b1's again and counts nothing)
#pragma unroll 1
            for (int b = b0; b <= b1; b += 8) {
              float2 ml[8];
              float4 x[8];
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const size_t at = slot(min(b + i, b1));
                ml[i] = __ldcg(&ta.part_ml[at]);
                x[i] = __ldcg(reinterpret_cast<const float4*>(ta.part_o + at * kHd) + lane);
              }
              float M2 = M;
#pragma unroll
              for (int i = 0; i < 8; i++) M2 = fmaxf(M2, ml[i].x);
              const float down = exp2_fast(M - M2);
              M = M2;
              L *= down;
              acc.x *= down;
              acc.y *= down;
              acc.z *= down;
              acc.w *= down;
#pragma unroll
              for (int i = 0; i < 8; i++)
                if (b + i <= b1) {
                  const float f = exp2_fast(ml[i].x - M);
                  L = fmaf(ml[i].y, f, L);
                  acc.x = fmaf(x[i].x, f, acc.x);
                  acc.y = fmaf(x[i].y, f, acc.y);
                  acc.z = fmaf(x[i].z, f, acc.z);
                  acc.w = fmaf(x[i].w, f, acc.w);
                }
            }
            const float inv = L == 0.f ? 0.f : 1.f / L;
            T* out = reinterpret_cast<T*>(a.out) + ((size_t)(k.sp.row0 + r / G) * a.H + h * G + r % G) * kHd + 4 * lane;
            *reinterpret_cast<uint2*>(out) = make_uint2(pack2(acc.x * inv, acc.y * inv, T()), pack2(acc.z * inv, acc.w * inv, T()));
          }
        }
      }
    }
    s++;
    h = 0;
    u0 = 0;
#pragma unroll 1
    while (left > 0 && s < a.b.seqs && unit_of(a, s).total == 0) s++;
    if (s >= a.b.seqs) break;
  }
}

}  // namespace

int uwc_paged_allow_smem(const void* kernel, int bytes) {
  static std::mutex mu;
  static std::set<std::pair<int, const void*>> done;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({dev, kernel})) return UWC_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return UWC_ERR_CUDA;
  }
  done.insert({dev, kernel});
  return UWC_OK;
}

namespace {

// Rows of a KV head up to which the few-row form runs: what two tiles of eight columns hold. Against the 256-row form at
// 9 to 16 rows (4 heads a KV head): 16 sequences of up to 3001 with 4 new tokens 27 us and 44, 64 of up to 8192 164 and 281,
// one of 8192 25 and 55.
constexpr int kFewRows = 16;
constexpr int kMaxGrid = 1024;                      // counters of a workspace
constexpr uint64_t kCounterBytes = kMaxGrid * 4;

// CTAs of the few-row form: what the device holds at once, or one per tile where there are fewer.
template <int NT>
int token_grid(int seqs, int max_new, int max_len, int Hkv, int window, int sinks) {
  long long keys = max_len;
  if (window >= 0) keys = std::min(keys, (long long)window + max_new + 2 * kTile + std::min(sinks, max_len) + kTile);
  const long long tiles = std::max(1ll, (keys + kTile - 1) / kTile);
  const long long slots = std::min(kMaxGrid, uwc_num_sms() * TokenCfg<NT>::kCtas);
  return (int)std::max(1ll, std::min(slots, tiles * seqs * Hkv));
}
template <int NT>
uint64_t token_workspace(int grid) {
  return kCounterBytes + (uint64_t)grid * 2 * 8 * NT * (kHd * 4 + 8);
}

template <typename T, int NT>
int launch_token(const AttnArgs& a, int max_len, uint8_t* ws, cudaStream_t st) {
  CUtensorMap mk, mv;
  const uint64_t rows = (uint64_t)a.c.pages * a.c.Hkv * a.c.ps;
  const int box = std::min(a.c.ps, kTile);
  int rc = uwc_make_tmap_2d(&mk, a.c.k, rows, kHd, kHd, box, kHd);
  if (rc == UWC_OK) rc = uwc_make_tmap_2d(&mv, a.c.v, rows, kHd, kHd, box, kHd);
  if (rc == UWC_OK) rc = uwc_paged_allow_smem((const void*)k_paged_token<T, NT>, TokenCfg<NT>::kSmem);
  if (rc != UWC_OK) return rc;
  const int grid = token_grid<NT>(a.b.seqs, a.b.max_new, max_len, a.c.Hkv, a.window, a.sinks);
  TokenArgs ta;
  ta.a = a;
  ta.counters = reinterpret_cast<uint32_t*>(ws);
  ta.part_o = reinterpret_cast<float*>(ws + kCounterBytes);
  ta.part_ml = reinterpret_cast<float2*>(ta.part_o + (size_t)grid * 2 * 8 * NT * kHd);
  ta.withhold = uwc_withhold();
  k_paged_token<T, NT><<<grid, kThreads, TokenCfg<NT>::kSmem, st>>>(ta, mk, mv);
  uwc_count_launch();
  return uwc_launch_status();
}

}  // namespace

extern "C" uint64_t uwc_paged_attention_workspace_bytes(int seqs, int max_new, int max_len, int H, int Hkv, int window,
                                                        int sinks) {
  if (seqs < 1 || max_new < 1 || max_len < 0 || Hkv < 1 || H < Hkv) return 0;
  const long long rows = (long long)max_new * (H / Hkv);
  if (rows <= 8) return token_workspace<1>(token_grid<1>(seqs, max_new, max_len, Hkv, window, sinks));
  if (rows <= kFewRows) return token_workspace<2>(token_grid<2>(seqs, max_new, max_len, Hkv, window, sinks));
  return uwc_paged_tile_workspace(seqs, max_new, max_len, H, Hkv, window, sinks);
}

extern "C" int uwc_paged_attention(const int8_t* kc, const float* sk, const int8_t* vc, const float* sv, int pages,
                                   int page_size, int Hkv, const int* table, const int* start, const int* cu, int seqs,
                                   int width, int rows, int max_new, int max_len, int dtype, const void* q,
                                   long long q_tok, long long q_head, void* out, int H, float scale, int window,
                                   int sinks, void* workspace, uint64_t workspace_bytes, void* stream) {
  AttnArgs a = {};
  a.c = Cache{const_cast<int8_t*>(kc), const_cast<float*>(sk), const_cast<int8_t*>(vc), const_cast<float*>(sv), pages,
              page_size, Hkv, 0};
  a.b = Seqs{table, start, cu, seqs, width, rows, max_new};
  const int rc = uwc_paged_check(&a.c, &a.b);
  if (rc != UWC_OK) return rc;
  if ((rows && (!q || !out)) || (dtype != UWC_T_BF16 && dtype != UWC_T_F16)) return UWC_ERR_ARG;
  if (!std::isfinite(scale)) return UWC_ERR_ARG;
  if (H < 1 || H % Hkv || max_len < 0 || sinks < 0) return UWC_ERR_SHAPE;
  if ((long long)max_new * (H / Hkv) > (1ll << 30)) return UWC_ERR_SHAPE;   // a sequence's rows are counted in int
  if (((uintptr_t)q | (uintptr_t)out) & 15 || q_tok < 0 || q_head < 0 || q_tok % 8 || q_head % 8) return UWC_ERR_ALIGN;
  UWC_CHECK_DEVICE();
  if (seqs == 0 || rows == 0 || max_new == 0) return UWC_OK;
  a.q = q;
  a.q_tok = q_tok;
  a.q_head = q_head;
  a.out = out;
  a.H = H;
  a.window = window < 0 ? -1 : window;
  a.sinks = sinks;
  a.scale = scale;
  a.status = uwc_status_ptr();
  if (workspace_bytes < uwc_paged_attention_workspace_bytes(seqs, max_new, max_len, H, Hkv, a.window, sinks) || !workspace)
    return UWC_ERR_SCRATCH;
  if ((uintptr_t)workspace & 15) return UWC_ERR_ALIGN;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const cudaStream_t st = (cudaStream_t)stream;
  const long long group = (long long)max_new * (H / Hkv);
  if (group > kFewRows) return uwc_paged_tile_launch(&a, dtype, max_len, ws, st);
  if (group <= 8)
    return dtype == UWC_T_BF16 ? launch_token<__nv_bfloat16, 1>(a, max_len, ws, st) : launch_token<__half, 1>(a, max_len, ws, st);
  return dtype == UWC_T_BF16 ? launch_token<__nv_bfloat16, 2>(a, max_len, ws, st) : launch_token<__half, 2>(a, max_len, ws, st);
}
