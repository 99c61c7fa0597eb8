// Attention over the paged 8-bit KV cache on sm_100a: the form for many query rows (prompts, chunks,
// wide groups of heads). The formula and the masks are paged_attn.cu's.
//
// k_paged_tile: an item is 256 rows of one (sequence, KV head) -- its tokens times the query heads of the
// group, token-major, so every head of the group uses a key tile once -- as two 128-row tiles. The bound is
// the tensor core (S = Q K^T and O = P V, tcgen05 kind::f16) against the exponentials (one each score).
// Roles of a CTA (one per SM, 13 warps):
//   warps 0-3, 4-7   the softmax of the first and second 128 rows, a row a thread: scores from TMEM, the
//                    running maximum and sum in float32 registers, weights back to TMEM as fp16 over the
//                    scores that they came from. They also turn the queries to fp16 and write the output.
//   warps 8-11       pages to operands: 128 keys of int8 from HBM through registers to fp16 in shared memory
//                    (the integers are exact; a byte permute and a subtraction a pair), two stages each for
//                    keys and values, so no scale is multiplied in: the key scale multiplies the score, the
//                    value scale (over a reference that follows its size) the weight, both a page's constant.
//   warp 12          one thread issues the products: while one row tile is in its softmax the other's run.
// O stays in TMEM; it is rescaled only when a row's maximum grew by more than 2^4 (so a weight is
// below 1024 * 2^4 * 2 in fp16, and keeps its 11 bits down to 2^-24 of the reference) or the tile's largest value
// scale left [1/64, 2] of the reference; both are rare after an item's first tile.
// Items lie on one line of key tiles, cut into equal parts, one per SM, as in the few-row form; an item in
// several parts is joined by the last of them in key order.
#include <algorithm>

#include "det_math.cuh"
#include "paged.cuh"
#include "uwc_host.h"

namespace {

using namespace paged;

constexpr int kRows = 128;                   // rows of a softmax warpgroup
constexpr int kTile = 128;                   // keys per tile
constexpr int kGroups = kTile / 16;          // 16-key groups, each inside one page
constexpr int kThreads = 13 * 32;
constexpr int kHalf = kTile * 128;           // bytes of 128 rows x 64 dims of fp16 (one swizzled block)
constexpr int kOperand = 2 * kHalf;          // a 128 x 128 fp16 operand
constexpr int kScaleRing = 4;
constexpr int kSeqs = 1024;                  // sequences whose span and tiles are kept in shared memory
constexpr int kSmem = 1024 + 6 * kOperand + kSeqs * 24;   // two query tiles, two stages of keys, two of values
constexpr int kMinTiles = 4;                 // a CTA's least share of the line
constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
constexpr uint32_t kIdescO = kIdescS | (1u << 16);   // values are stored key by key: B is MN-major
constexpr float kRaise = 4.f;                // log2 by which a score may pass the running maximum
constexpr float kWeightUnit = 1024.f;         // the fp16 weight of p = 1 at the reference scale

struct TileArgs {
  AttnArgs a;
  float* part_o;           // (2 grid, 256, 128): a CTA's two partial items, unnormalized
  float2* part_ml;         // (2 grid, 256): running maximum (log2), sum
  uint32_t* counters;      // (grid, 2): finished parts of the item that starts in this CTA; left zero
};

// 256 rows of one (sequence, KV head): tokens t0 .. t1 have rows in it.
struct Item : Keys<kTile> {
  __device__ __forceinline__ Item(const AttnArgs& a, const Span& sp, int G, int blk)
      : Keys<kTile>(a, sp, 2 * kRows * blk / G, min(sp.n - 1, (2 * kRows * blk + 2 * kRows - 1) / G)) {}
};

// The batch as a CTA's roles see it: spans and tiles (of one KV head) of the first kSeqs sequences in
// shared memory, of any further ones from global memory.
struct Batch {
  const AttnArgs& a;
  int G;
  int4* span_;             // row0, n, start, idle
  long long* tiles_;
  __device__ __forceinline__ Span span(int s) const {
    if (s >= kSeqs) return span_of(a.b, a.c.ps, s);
    const int4 x = span_[s];
    return Span{x.x, x.y, x.z, x.w != 0, false};
  }
  __device__ __forceinline__ int blocks(const Span& z) const { return (int)(((long long)z.n * G + 2 * kRows - 1) / (2 * kRows)); }
  // all lanes of a warp together
  __device__ __forceinline__ long long count(const Span& z) const {
    const int nb = blocks(z);
    long long t = 0;
    for (int b = threadIdx.x & 31; b < nb; b += 32) t += Item(a, z, G, b).total;
    return warp_sumll(t);
  }
  __device__ __forceinline__ long long tiles(int s) const { return s < kSeqs ? tiles_[s] : count(span(s)); }
  __device__ __forceinline__ void load() {
    const int n = min(a.b.seqs, kSeqs);
    for (int s = threadIdx.x; s < n; s += kThreads) {
      const Span z = span_of(a.b, a.c.ps, s);
      if (z.bad && blockIdx.x == 0) set_status(a.status, UWC_DEV_RANGE);
      span_[s] = make_int4(z.row0, z.n, z.start, z.idle);
    }
    if (blockIdx.x == 0)
      for (int s = kSeqs + threadIdx.x; s < a.b.seqs; s += kThreads)
        if (span_of(a.b, a.c.ps, s).bad) set_status(a.status, UWC_DEV_RANGE);
    __syncthreads();
    for (int s = threadIdx.x / 32; s < n; s += kThreads / 32) {
      const long long t = count(span(s));
      if ((threadIdx.x & 31) == 0) tiles_[s] = t;
    }
  }
};

// A CTA's walk along the line: pieces (sequence, KV head, block, tiles t0 .. t1 - 1). Every warp walks for
// itself, all lanes together.
struct Walk {
  const Batch& q;
  const AttnArgs& a;
  int G, s, h, blk, blks;
  int t0, t1, total;       // this piece's tiles, the item's
  long long at, left, per; // the line's tile that t0 is; tiles of this CTA from t0 on
  Span sp;

  __device__ __forceinline__ Walk(const Batch& batch) : q(batch), a(batch.a), G(batch.G) {
    const int lane = threadIdx.x & 31, S = a.b.seqs, kept = min(S, kSeqs);
    long long sum = 0;
    for (int i = lane; i < kept; i += 32) sum += q.tiles(i);
    sum = warp_sumll(sum);
    for (int i = kept; i < S; i++) sum += q.tiles(i);
    sum *= a.c.Hkv;
    per = max((sum + gridDim.x - 1) / gridDim.x, (long long)kMinTiles);
    at = per * blockIdx.x;
    left = min(per, sum - at);
    if (left <= 0) return;
    // the sequence, then the block, that tile `at` lies in
    long long rest = at;
    for (s = 0; s < S; s++) {
      const long long one = q.tiles(s);
      if (rest >= one * a.c.Hkv) {
        rest -= one * a.c.Hkv;
        continue;
      }
      sp = q.span(s);
      blks = q.blocks(sp);
      h = (int)(rest / one);
      rest %= one;
      for (int b0 = 0; b0 < blks; b0 += 32) {
        const int t = b0 + lane < blks ? Item(a, sp, G, b0 + lane).total : 0;
        int inc = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, inc > rest);
        if (hit) {
          const int l = __ffs(hit) - 1;
          blk = b0 + l;
          t0 = (int)(rest - __shfl_sync(0xffffffffu, inc - t, l));
          break;
        }
        rest -= __shfl_sync(0xffffffffu, inc, 31);
      }
      break;
    }
    piece();
  }
  __device__ __forceinline__ void piece() {
    total = Item(a, sp, G, blk).total;
    t1 = (int)min((long long)total, t0 + left);
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next() {
    at += t1 - t0;
    left -= t1 - t0;
    if (left <= 0) return;
    t0 = 0;
    if (++blk == blks) {
      blk = 0;
      if (++h == a.c.Hkv) {
        h = 0;
        do {
          sp = q.span(++s);
          blks = q.blocks(sp);
        } while (blks == 0 && s + 1 < a.b.seqs);
      }
    }
    piece();
  }
  __device__ __forceinline__ int rows(int w) const { return min(kRows, max(0, sp.n * G - 2 * kRows * blk - kRows * w)); }
  // the CTAs that the item's parts lie in
  __device__ __forceinline__ int first_cta() const { return (int)((at - t0) / per); }
  __device__ __forceinline__ int last_cta() const { return (int)((at - t0 + total - 1) / per); }
};

// ---- tcgen05
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t saddr) {
  // MN-major operand, 128-byte swizzle: 64 dims a 128-byte row, 8-key atoms 1024 bytes apart (SBO), the
  // next 64 dims one block on (LBO)
  uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(kHalf >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

struct Bars {
  uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2], wg[2], fin;
};

// Ends the role when a wait ran out (the status is set, the other roles follow by the abort flag).
#define TILE_WAIT(bar, parity) \
  if (!__all_sync(0xffffffffu, mbar_wait(&(bar), (parity), &s_abort, a.status))) goto done

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) k_paged_tile(const TileArgs ta) {
  const AttnArgs& a = ta.a;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>(((uintptr_t)sm_raw + 1023) & ~(uintptr_t)1023);
  __shared__ Bars bar;
  __shared__ float2 s_scale[kScaleRing][kGroups];   // key scale (-1: no key of the group is seen), value scale
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_last[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t smQ = smem_u32(sm), smK = smQ + 2 * kOperand, smV = smK + 2 * kOperand;
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&bar.q_full[i], kRows);
      mbar_init(&bar.k_full[i], 128);
      mbar_init(&bar.k_empty[i], 1);
      mbar_init(&bar.v_full[i], 128);
      mbar_init(&bar.v_empty[i], 1);
      mbar_init(&bar.s_full[i], 2);
      mbar_init(&bar.p_full[i], kRows);
      mbar_init(&bar.o_done[i], 1);
      mbar_init(&bar.wg[i], kRows);
    }
    mbar_init(&bar.fin, 1);
    s_abort = 0;
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  Batch batch{a, a.H / a.c.Hkv, reinterpret_cast<int4*>(sm + 6 * kOperand),
              reinterpret_cast<long long*>(sm + 6 * kOperand + kSeqs * 16)};
  batch.load();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int Hkv = a.c.Hkv, ps = a.c.ps;

  if (warp < 8) {
    // ------------------------------------------------------------------ softmax, a row a thread
    const int w = warp >> 2, r = tid & (kRows - 1);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + w * 128, tO = tmem + lanes + 256 + w * 128;
    uint32_t it = 0, all = 0, wgp = 0;             // this warpgroup's tiles, every tile, its barrier's phases
    for (Walk k(batch); k.more(); k.next()) {
      const int rows = k.rows(w);
      if (rows == 0) {                             // only w = 1: the second tile of a short block
        all += k.t1 - k.t0;
        continue;
      }
      const int row = 2 * kRows * k.blk + kRows * w + r, t = row / k.G, hh = k.h * k.G + row % k.G;
      const bool live = r < rows;
      const int pos = live && !k.sp.idle ? k.sp.start + t : -1;
      const Item key(a, k.sp, k.G, k.blk);
      // ---- the query row as fp16 (its largest value at 2^14), into the swizzled operand
      float qmul;
      {
        uint4 x[16];
        const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (long long)(k.sp.row0 + t) * a.q_tok +
                                                        (long long)hh * a.q_head);
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = live ? __ldg(q + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float2 f = two_f(u[j], T());
            mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        const int e = row_exponent(mx);
        const float up = a.scale < 0.f ? -pow2i(e) : pow2i(e);   // a negative scale goes with the query
        qmul = fabsf(a.scale) * kLog2OfE * pow2i(-e);
#pragma unroll
        for (int i = 0; i < 16; i++) {
          uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float2 f = two_f(u[j], T());
            u[j] = pack2(f.x * up, f.y * up, __half());
          }
          sts128(smQ + w * kOperand + (i >> 3) * kHalf + r * 128 + (((i & 7) ^ (r & 7)) << 4), make_uint4(u[0], u[1], u[2], u[3]));
        }
      }
      fence_async_smem();
      mbar_arrive(&bar.q_full[w]);
      // positions of this warpgroup's first and last row bound where its masks are needed
      const int pa = k.sp.idle ? -1 : k.sp.start + (2 * kRows * k.blk + kRows * w) / k.G;
      const int pb = k.sp.idle ? -1 : k.sp.start + (2 * kRows * k.blk + kRows * w + rows - 1) / k.G;
      float m = kNoMax, l = 0.f, ref = 0.f;
      for (int i = k.t0; i < k.t1; i++, it++, all++) {
        const int j0 = key.key(i);
        TILE_WAIT(bar.s_full[w], it & 1);
        tc_fence_after();
        const float2* sc = s_scale[all % kScaleRing];
        bool seen = true;
        float f[kGroups], vs = 0.f;
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
          const float2 x = sc[g];
          seen &= x.x >= 0.f;
          f[g] = fmaxf(x.x * qmul, 1e-37f);        // not 0: a hidden score stays -inf
          vs = fmaxf(vs, x.y);
        }
        const bool masked = !seen || !(j0 + kTile - 1 <= pa && (a.window < 0 || j0 > pb - a.window || j0 + kTile <= a.sinks));
        auto load = [&](int c, uint32_t* s) {      // 64 scores of this row, hidden ones -inf
          tmem_ld_32x32b_x32(tS + 64 * c, s);
          tmem_ld_32x32b_x32(tS + 64 * c + 32, s + 32);
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int x = 0; x < 64; x++) {
              const int j = j0 + 64 * c + x;
              if (!sees(a, pos, j) || sc[4 * c + x / 16].x < 0.f) s[x] = 0xff800000u;
            }
          }
        };
        uint32_t s[64];
        float mx = kNoMax;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          load(c, s);
#pragma unroll
          for (int g = 0; g < 4; g++) {
            float x = __uint_as_float(s[16 * g]);
#pragma unroll
            for (int y = 1; y < 16; y++) x = fmaxf(x, __uint_as_float(s[16 * g + y]));
            mx = fmaxf(mx, x * f[4 * c + g]);
          }
        }
        // ---- raise the maximum or the value reference, and bring O along (its products must be done)
        const bool raise = mx > m + kRaise, refer = vs > 2.f * ref || (vs > 0.f && vs < ref * (1.f / 64.f));
        if (__any_sync(0xffffffffu, raise || refer)) {
          const float m2 = fmaxf(m, mx), ref2 = refer ? vs : ref;
          const float down = exp2_fast(m - m2);
          const float by = ref2 > 0.f ? down * __fdividef(ref, ref2) : down;
          l *= down;
          m = m2;
          ref = ref2;
          if (i > k.t0) {
            TILE_WAIT(bar.o_done[w], (it - 1) & 1);
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 4; c++) {
              tmem_ld_32x32b_x32(tO + 32 * c, s);
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 32; x++) s[x] = __float_as_uint(__uint_as_float(s[x]) * by);
              tmem_st_32x32b_x32(tO + 32 * c, s);
            }
          }
        }
        // ---- weights: p = 2^(score - m); the row sum keeps p, the product gets p s_v / ref in fp16
        const float unit = ref > 0.f ? __fdividef(kWeightUnit, ref) : 0.f;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          load(c, s);
          uint32_t p[32];
#pragma unroll
          for (int g = 0; g < 4; g++) {
            const float fg = f[4 * c + g], wg = sc[4 * c + g].y * unit;
#pragma unroll
            for (int y = 0; y < 8; y++) {
              const float x0 = exp2_fast(fmaf(__uint_as_float(s[16 * g + 2 * y]), fg, -m));
              const float x1 = exp2_fast(fmaf(__uint_as_float(s[16 * g + 2 * y + 1]), fg, -m));
              l += x0 + x1;
              p[8 * g + y] = pack2(x0 * wg, x1 * wg, __half());
            }
          }
          tmem_st_32x32b_x16(tS + 32 * c, p);
          tmem_st_32x32b_x16(tS + 32 * c + 16, p + 16);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bar.p_full[w]);
      }
      // ---- the item's (or the part's) result
      TILE_WAIT(bar.o_done[w], (it - 1) & 1);
      tc_fence_after();
      const bool whole = k.t0 == 0 && k.t1 == k.total;
      const float back = ref * (1.f / kWeightUnit);
      T* out = reinterpret_cast<T*>(a.out) + ((size_t)(k.sp.row0 + t) * a.H + hh) * kHd;
      if (whole) {
        const float inv = l == 0.f ? 0.f : back / l;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          uint32_t s[32];
          tmem_ld_32x32b_x32(tO + 32 * c, s);
          tmem_wait_ld();
          if (live) {
#pragma unroll
            for (int x = 0; x < 4; x++) {
              uint32_t u[4];
#pragma unroll
              for (int y = 0; y < 4; y++)
                u[y] = pack2(__uint_as_float(s[8 * x + 2 * y]) * inv, __uint_as_float(s[8 * x + 2 * y + 1]) * inv, T());
              reinterpret_cast<uint4*>(out + 32 * c)[x] = make_uint4(u[0], u[1], u[2], u[3]);
            }
          }
        }
        tc_fence_before();
        continue;
      }
      const int b0 = k.first_cta(), b1 = k.last_cta();
      {
        const size_t slot = ((size_t)(2 * blockIdx.x + (k.t0 == 0)) * 2 + w) * kRows + r;
#pragma unroll
        for (int c = 0; c < 4; c++) {
          uint32_t s[32];
          tmem_ld_32x32b_x32(tO + 32 * c, s);
          tmem_wait_ld();
          if (live) {
            float4* po = reinterpret_cast<float4*>(ta.part_o + slot * kHd + 32 * c);
#pragma unroll
            for (int x = 0; x < 8; x++)
              po[x] = make_float4(__uint_as_float(s[4 * x]) * back, __uint_as_float(s[4 * x + 1]) * back,
                                  __uint_as_float(s[4 * x + 2]) * back, __uint_as_float(s[4 * x + 3]) * back);
          }
        }
        if (live) ta.part_ml[slot] = make_float2(m, l);
        tc_fence_before();
      }
      __threadfence();
      mbar_arrive(&bar.wg[w]);
      TILE_WAIT(bar.wg[w], wgp & 1);
      wgp++;
      if (r == 0) {
        const uint32_t n = atomicAdd(&ta.counters[2 * b0 + w], 1u);
        s_last[w] = n == (uint32_t)(b1 - b0);
        if (s_last[w]) ta.counters[2 * b0 + w] = 0;
        __threadfence();
      }
      mbar_arrive(&bar.wg[w]);
      TILE_WAIT(bar.wg[w], wgp & 1);
      wgp++;
      if (s_last[w] && live) {
        __threadfence();
        auto slot = [&](int b) { return ((size_t)(2 * b + (b == b0)) * 2 + w) * kRows + r; };
        float M = kNoMax, L = 0.f;
        for (int b = b0; b <= b1; b++) M = fmaxf(M, __ldcg(&ta.part_ml[slot(b)]).x);
        for (int b = b0; b <= b1; b++) {
          const float2 ml = __ldcg(&ta.part_ml[slot(b)]);
          L = fmaf(ml.y, exp2_fast(ml.x - M), L);
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
        for (int c = 0; c < 16; c++) {
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
          for (int b = b0; b <= b1; b++) {
            const float f = exp2_fast(__ldcg(&ta.part_ml[slot(b)]).x - M);
            const float4* po = reinterpret_cast<const float4*>(ta.part_o + slot(b) * kHd) + 2 * c;
            const float4 u = __ldcg(po), v = __ldcg(po + 1);
            x = make_float4(fmaf(u.x, f, x.x), fmaf(u.y, f, x.y), fmaf(u.z, f, x.z), fmaf(u.w, f, x.w));
            y = make_float4(fmaf(v.x, f, y.x), fmaf(v.y, f, y.y), fmaf(v.z, f, y.z), fmaf(v.w, f, y.w));
          }
          reinterpret_cast<uint4*>(out)[c] = make_uint4(pack2(x.x * inv, x.y * inv, T()), pack2(x.z * inv, x.w * inv, T()),
                                                        pack2(y.x * inv, y.y * inv, T()), pack2(y.z * inv, y.w * inv, T()));
        }
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ pages to operands
    const int ct = tid - 256, row = ct >> 3, c = ct & 7;        // key row % 16, 16 dims from 16 c on
    const uint32_t half = (uint32_t)(c >> 2) * kHalf, c16 = (c & 3) * 2;
    uint32_t it = 0;
    for (Walk k(batch); k.more(); k.next()) {
      const Item key(a, k.sp, k.G, k.blk);
      // lane g < 8 of each warp looks up 16-key group g of a tile
      auto page_of = [&](int i) {
        const int j = key.key(i) + 16 * lane;
        int page = -1;
        if (lane < kGroups && i < k.t1 && key.seen(j, 16)) {
          page = page_at(a.b, a.c, k.s, j / ps);
          if (page < 0) set_status(a.status, UWC_DEV_RANGE);
        }
        return page;
      };
      auto fetch = [&](const int8_t* data, int page, int j0, uint4* x) {
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
          const int pg = __shfl_sync(0xffffffffu, page, g);
          x[g] = make_uint4(0, 0, 0, 0);
          if (pg >= 0)
            x[g] = __ldg(reinterpret_cast<const uint4*>(data + (((size_t)pg * Hkv + k.h) * ps + (j0 + 16 * g) % ps + row) * kHd) + c);
        }
      };
      auto store = [&](uint32_t base, const uint4* x) {
#pragma unroll
        for (int g = 0; g < kGroups; g++) {
          const uint32_t u[4] = {x[g].x ^ 0x80808080u, x[g].y ^ 0x80808080u, x[g].z ^ 0x80808080u, x[g].w ^ 0x80808080u};
          const uint4 lo = make_uint4(i8_half2(u[0], 0x4140), i8_half2(u[0], 0x4342), i8_half2(u[1], 0x4140), i8_half2(u[1], 0x4342));
          const uint4 hi = make_uint4(i8_half2(u[2], 0x4140), i8_half2(u[2], 0x4342), i8_half2(u[3], 0x4140), i8_half2(u[3], 0x4342));
          const uint32_t at = base + half + (16 * g + row) * 128;
          const uint32_t a0 = at + ((c16 ^ (row & 7)) << 4), a1 = at + (((c16 + 1) ^ (row & 7)) << 4);
          // the two blocks' threads write opposite halves of a row pair at a time: no bank conflict
          const bool swap = c >= 4;
          sts128(swap ? a1 : a0, swap ? hi : lo);
          sts128(swap ? a0 : a1, swap ? lo : hi);
        }
      };
      uint4 x[kGroups], y[kGroups];
      int page = page_of(k.t0);
      fetch(a.c.k, page, key.key(k.t0), x);
      for (int i = k.t0; i < k.t1; i++, it++) {
        const int st = it & 1;
        const uint32_t use = it >> 1;
        const int j0 = key.key(i), npage = i + 1 < k.t1 ? page_of(i + 1) : -1;
        float2 sc = make_float2(-1.f, 0.f);
        if (ct < kGroups && page >= 0) {
          const size_t ph = (size_t)page * Hkv + k.h;
          sc = make_float2(__ldg(a.c.sk + ph), __ldg(a.c.sv + ph));
        }
        fetch(a.c.v, page, j0, y);
        if (use > 0) TILE_WAIT(bar.k_empty[st], (use - 1) & 1);
        store(smK + st * kOperand, x);
        if (ct < kGroups) s_scale[it % kScaleRing][ct] = sc;
        fence_async_smem();
        mbar_arrive(&bar.k_full[st]);
        if (i + 1 < k.t1) fetch(a.c.k, npage, key.key(i + 1), x);
        if (use > 0) TILE_WAIT(bar.v_empty[st], (use - 1) & 1);
        store(smV + st * kOperand, y);
        fence_async_smem();
        mbar_arrive(&bar.v_full[st]);
        page = npage;
      }
    }
  } else {
    // ------------------------------------------------------------------ the products
    uint32_t it = 0, items[2] = {0, 0}, n1 = 0;   // tiles; items of each row tile; tiles of the second row tile
    for (Walk k(batch); k.more(); k.next()) {
      const int nw = k.rows(1) > 0 ? 2 : 1;
      const uint32_t itw[2] = {it, n1};           // each row tile's own count of tiles (its barriers' phases)
      const int T1 = k.t1 - k.t0;
      auto scores = [&](int st, int w) {
#pragma unroll
        for (int x = 0; x < 8; x++) {
          const uint32_t off = (x >> 2) * kHalf + (x & 3) * 32;
          mma_ss(tmem + w * 128, sdesc_sw128(smQ + w * kOperand + off), sdesc_sw128(smK + st * kOperand + off), kIdescS, x > 0);
        }
      };
      // the first tile's scores
      TILE_WAIT(bar.k_full[it & 1], (it >> 1) & 1);
      for (int w = 0; w < nw; w++) {
        TILE_WAIT(bar.q_full[w], items[w] & 1);
        tc_fence_after();
        if (elect_one()) {
          scores(it & 1, w);
          mbar_arrive(&bar.s_full[w]);
          mma_commit(&bar.s_full[w]);
          if (w == nw - 1) mma_commit(&bar.k_empty[it & 1]);
        }
        __syncwarp();
      }
      for (int j = 0; j < T1; j++, it++) {
        const uint32_t st = it & 1, nx = it + 1;
        for (int w = 0; w < nw; w++) {
          if (w == 0) TILE_WAIT(bar.v_full[st], (it >> 1) & 1);
          TILE_WAIT(bar.p_full[w], (itw[w] + j) & 1);
          if (w == 0 && j + 1 < T1) TILE_WAIT(bar.k_full[nx & 1], (nx >> 1) & 1);
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int x = 0; x < 8; x++)
              mma_ts(tmem + 256 + w * 128, tmem + w * 128 + x * 8, sdesc_mn(smV + st * kOperand + x * 2048), kIdescO, j > 0 || x > 0);
            mma_commit(&bar.o_done[w]);
            if (w == nw - 1) mma_commit(&bar.v_empty[st]);
            if (j + 1 < T1) {
              scores(nx & 1, w);
              mbar_arrive(&bar.s_full[w]);
              mma_commit(&bar.s_full[w]);
              if (w == nw - 1) mma_commit(&bar.k_empty[nx & 1]);
            }
          }
          __syncwarp();
        }
      }
      items[0]++;
      if (nw == 2) {
        items[1]++;
        n1 += T1;
      }
    }
  }
done:
  __syncwarp();
  if (warp == 12) {
    // every product that was issued has landed before the tensor memory goes (bounded, as every wait)
    if (elect_one()) mma_commit(&bar.fin);
    __syncwarp();
    for (int n = 0; n < (1 << 20) && !mbar_try_wait(&bar.fin, 0); n++) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

int tile_grid(int seqs, int max_new, int max_len, int H, int Hkv, int window, int sinks) {
  long long keys = max_len;
  if (window >= 0) keys = std::min(keys, (long long)window + max_new + 3ll * kTile + std::min(sinks, max_len));
  const long long blocks = ((long long)max_new * (H / Hkv) + 2 * kRows - 1) / (2 * kRows);
  const long long tiles = std::max(1ll, (keys + kTile - 1) / kTile);
  const double all = (double)blocks * tiles * seqs * Hkv;
  return (int)std::max(1.0, std::min((double)std::min(uwc_num_sms(), 512), all));
}

constexpr uint64_t kCounterBytes = 4096;

}  // namespace

uint64_t uwc_paged_tile_workspace(int seqs, int max_new, int max_len, int H, int Hkv, int window, int sinks) {
  const uint64_t grid = tile_grid(seqs, max_new, max_len, H, Hkv, window, sinks);
  return kCounterBytes + grid * 2 * 2 * kRows * (kHd * 4 + 8);
}

int uwc_paged_tile_launch(const AttnArgs* a, int dtype, int max_len, void* workspace, cudaStream_t stream) {
  const int grid = tile_grid(a->b.seqs, a->b.max_new, max_len, a->H, a->c.Hkv, a->window, a->sinks);
  TileArgs ta;
  ta.a = *a;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  ta.counters = reinterpret_cast<uint32_t*>(ws);
  ta.part_o = reinterpret_cast<float*>(ws + kCounterBytes);
  ta.part_ml = reinterpret_cast<float2*>(ta.part_o + (size_t)grid * 4 * kRows * kHd);
  const void* fn = dtype == UWC_T_BF16 ? (const void*)k_paged_tile<__nv_bfloat16> : (const void*)k_paged_tile<__half>;
  const int rc = uwc_paged_allow_smem(fn, kSmem);
  if (rc != UWC_OK) return rc;
  if (dtype == UWC_T_BF16) k_paged_tile<__nv_bfloat16><<<grid, kThreads, kSmem, stream>>>(ta);
  else k_paged_tile<__half><<<grid, kThreads, kSmem, stream>>>(ta);
  uwc_count_launch();
  return uwc_launch_status();
}
