// The paged 8-bit KV cache on sm_100a: new tokens in, values back out.
//
//   k_paged_append   rotates the new keys (and the queries) and stores keys and values as int8 with
//                    one scale for each (page, KV head). With x a page's new values in float32 and
//                    s0 the scale of the tokens that it already holds (0 where it holds none),
//                      s = max(s0, fdiv(max|x|, 127)),  q(x) = clamp(rint(fdiv(x, s)), +-127),
//                    and an old token's q becomes rint(fdiv(fmul(q, s0), s)) when s > s0. Every step
//                    is one IEEE operation, the rotation too (fadd(fmul(x, cos), fmul(rot(x), sin))),
//                    so a cache is the same bit for bit wherever and in whatever batch it was written,
//                    and appending a sequence's newest tokens again changes nothing. A call sets the sequence's
//                    end: tokens that its last page held past it are not brought to a scale that grows or starts anew.
//   k_paged_gather   cached tokens back as 16- or 32-bit values.
//
// Both are bound by HBM at prompt sizes and by latency at decode sizes. Measured on B200 (a graph of calls): 8
// prompts of 2048, 16 + 2 x 8 heads, 63 us (3.7 TB/s: about 20 instructions a value, twice over the rows) and 20 us
// to read it back; a token each of 64 sequences, 32 + 2 x 8 heads, 4.8 us.
#include <algorithm>
#include <cfloat>

#include "det_math.cuh"
#include "paged.cuh"
#include "uwc_host.h"

namespace {

using paged::Cache;
using paged::kHd;
using paged::page_at;
using paged::Seqs;
using paged::Span;
using paged::span_of;

constexpr int kThreads = 256;
constexpr int kQHeads = 2;       // query heads that share a thread's rotation values

// Eight 16-bit values as float32, and back.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4 w, float* f) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 x = paged::two_f(u[i], T());
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
  using paged::pack2;
  return make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()), pack2(f[4], f[5], T()), pack2(f[6], f[7], T()));
}

struct Rows {              // token rows of heads: element (n, h, d) at n * tok + h * head + d
  const void* p;
  long long tok, head;
};

struct AppendArgs {
  Cache c;
  Seqs b;
  Rows k, v, q;
  void* q_out;             // (rows, H, 128)
  int H, max_pos, most;    // most: pages that one sequence's new tokens may touch
  const float *cos, *sin;  // (max_pos, 128)
  const float *q_norm, *k_norm;
  float eps;
  uint32_t* status;
};

// A token head lies in eight lanes: lane c of them holds dims 8 c .. 8 c + 7 (lo) and their rotation
// partners 64 + 8 c .. (hi).
struct Raw {
  uint4 lo, hi;
};
template <typename T>
__device__ __forceinline__ Raw load_raw(const Rows& r, long long row, int h, int c) {
  const T* p = reinterpret_cast<const T*>(r.p) + row * r.tok + h * r.head + 8 * c;
  return Raw{*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(p + 64)};
}

// det_rmsnorm over the head (exact fixed-point sum of 128 squares, runtime/detrt/core.py:151-159); all
// lanes of a warp together
__device__ __forceinline__ void norm_head(const float* __restrict__ w, float eps, int c, float* lo, float* hi) {
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) mx = fmaxf(mx, fmaxf(__fmul_rn(lo[i], lo[i]), __fmul_rn(hi[i], hi[i])));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  int e;
  frexpf(mx, &e);
  const int sh = min(max((62 - 7) - e, -1000), 1000);
  long long a = 0;
#pragma unroll
  for (int i = 0; i < 8; i++)
    a += __double2ll_rn((double)__fmul_rn(lo[i], lo[i]) * pow2d(sh)) +
         __double2ll_rn((double)__fmul_rn(hi[i], hi[i]) * pow2d(sh));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  const float ss = __double2float_rn(__ll2double_rn(a) * pow2d(-sh));
  const float rr = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.0f / kHd), eps)));
#pragma unroll
  for (int i = 0; i < 8; i++) {
    lo[i] = __fmul_rn(__fmul_rn(lo[i], rr), __ldg(w + 8 * c + i));
    hi[i] = __fmul_rn(__fmul_rn(hi[i], rr), __ldg(w + 64 + 8 * c + i));
  }
}

// The rotation values of four dims of a lane (half 0: its first four) and of their partners, and the
// rotation of those: rows `pos` of the tables.
struct Turn4 {
  float4 cl, ch, sl, sh;
};
__device__ __forceinline__ Turn4 load_turn(const float* cos, const float* sin, int pos, int c, int half) {
  const float4* a = reinterpret_cast<const float4*>(cos + (size_t)pos * kHd) + 2 * c + half;
  const float4* b = reinterpret_cast<const float4*>(sin + (size_t)pos * kHd) + 2 * c + half;
  return Turn4{__ldg(a), __ldg(a + 16), __ldg(b), __ldg(b + 16)};
}
__device__ __forceinline__ void rotate4(const Turn4& t, float* lo, float* hi) {
  const float cl[4] = {t.cl.x, t.cl.y, t.cl.z, t.cl.w}, ch[4] = {t.ch.x, t.ch.y, t.ch.z, t.ch.w};
  const float sl[4] = {t.sl.x, t.sl.y, t.sl.z, t.sl.w}, sh[4] = {t.sh.x, t.sh.y, t.sh.z, t.sh.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float x = lo[i], y = hi[i];
    lo[i] = __fadd_rn(__fmul_rn(x, cl[i]), __fmul_rn(-y, sl[i]));
    hi[i] = __fadd_rn(__fmul_rn(y, ch[i]), __fmul_rn(x, sh[i]));
  }
}

// A value's part in its page's scale: its magnitude, 0 for infinities and NaN (stored as +-127 and 0).
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= FLT_MAX ? a : 0.f;
}
// Four values as clamp(rint(fdiv(x, s)), least, 127), NaN as 0. least: -127 for new values; -128 for held ones, whose
// integers a caller may have written.
__device__ __forceinline__ uint32_t quant4_exact(float4 x4, float s, float least) {
  const float x[4] = {x4.x, x4.y, x4.z, x4.w};
  uint32_t o = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float v = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), least), 127.f) : 0.f;
    const int q = x[i] == x[i] ? (int)v : 0;
    o |= (uint32_t)(q & 255) << (8 * i);
  }
  return o;
}
// The same without the divisions (half of the kernel's instructions) where that cannot change a bit: inv is
// 1 / s, so x inv is within 1e-4 of the quotient (|quotient| <= 128), and both round to the same integer
// unless it lies that near to a half. 1.5 2^23 + x inv has the integer in its low byte. Infinities, NaN and
// an infinite inv leave a NaN, which fails the test too.
__device__ __forceinline__ uint32_t quant4(const float* x, float s, float inv, float least = -127.f) {
  constexpr float kMagic = 12582912.f;
  uint32_t t[4];
  float off = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float z = fmaf(x[i], inv, kMagic);
    t[i] = __float_as_uint(z);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(off) : "f"(fabsf(fmaf(x[i], inv, kMagic - z))));
  }
  if (!(off < 0.4999f)) return quant4_exact(make_float4(x[0], x[1], x[2], x[3]), s, least);
  return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}
__device__ __forceinline__ float inverse(float s) { return s > 1e-30f ? __frcp_rn(s) : __int_as_float(0x7f800000); }

// One row of queries: unit u is (row, kQHeads query heads) of eight lanes, four units a warp.
template <typename T, bool NORM>
__device__ __forceinline__ void query_unit(const AppendArgs& a, long long u, int c) {
  const int groups = (a.H + kQHeads - 1) / kQHeads;
  const int row = (int)(u / groups), h0 = (int)(u % groups) * kQHeads;
  const bool in = row < a.b.rows;
  int pos = -1;
  bool covered = false;
  Raw raw[kQHeads];
#pragma unroll
  for (int i = 0; i < kQHeads; i++) {
    raw[i] = Raw{};
    if (in && h0 + i < a.H && !(NORM && a.q_norm)) raw[i] = load_raw<T>(a.q, row, h0 + i, c);
  }
  if (in) {
    // the sequence whose span holds this row: the last with cu[s] <= row
    int s = 0;
    for (int n = a.b.seqs; n > 1;) {
      const int half = n >> 1;
      if (__ldg(a.b.cu + s + half) <= row) s += half;
      n -= half;
    }
    const Span sp = span_of(a.b, a.c.ps, s);
    const int t = row - sp.row0;
    covered = t >= 0 && t < sp.n;
    if (covered && !sp.idle) {
      pos = sp.start + t;
      if (pos >= a.max_pos) {
        set_status(a.status, UWC_DEV_RANGE);
        pos = -1;
      }
    }
  }
  T* out = reinterpret_cast<T*>(a.q_out) + ((size_t)row * a.H + h0) * kHd + 8 * c;
  if (NORM && a.q_norm) {
#pragma unroll 1
    for (int i = 0; i < kQHeads; i++) {
      float lo[8], hi[8];
      Raw x = {};
      if (in && h0 + i < a.H) x = load_raw<T>(a.q, row, h0 + i, c);
      unpack8<T>(x.lo, lo);
      unpack8<T>(x.hi, hi);
      norm_head(a.q_norm, a.eps, c, lo, hi);
      if (pos >= 0)
#pragma unroll
        for (int k = 0; k < 2; k++) rotate4(load_turn(a.cos, a.sin, pos, c, k), lo + 4 * k, hi + 4 * k);
      if (covered && h0 + i < a.H) {
        *reinterpret_cast<uint4*>(out + i * kHd) = pos >= 0 ? pack8<T>(lo) : make_uint4(0, 0, 0, 0);   // an idle slot's rows are zero
        *reinterpret_cast<uint4*>(out + i * kHd + 64) = pos >= 0 ? pack8<T>(hi) : make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  // in place, four dims of all its heads at a time: the rotation values are read once
  if (pos >= 0) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const Turn4 t = load_turn(a.cos, a.sin, pos, c, k);
#pragma unroll
      for (int i = 0; i < kQHeads; i++) {
        uint32_t* lw = reinterpret_cast<uint32_t*>(&raw[i].lo) + 2 * k;
        uint32_t* hw = reinterpret_cast<uint32_t*>(&raw[i].hi) + 2 * k;
        const float2 l0 = paged::two_f(lw[0], T()), l1 = paged::two_f(lw[1], T());
        const float2 h0_ = paged::two_f(hw[0], T()), h1 = paged::two_f(hw[1], T());
        float lo[4] = {l0.x, l0.y, l1.x, l1.y}, hi[4] = {h0_.x, h0_.y, h1.x, h1.y};
        rotate4(t, lo, hi);
        lw[0] = paged::pack2(lo[0], lo[1], T());
        lw[1] = paged::pack2(lo[2], lo[3], T());
        hw[0] = paged::pack2(hi[0], hi[1], T());
        hw[1] = paged::pack2(hi[2], hi[3], T());
      }
    }
  }
  if (covered)
#pragma unroll
    for (int i = 0; i < kQHeads; i++)
      if (h0 + i < a.H) {
        *reinterpret_cast<uint4*>(out + i * kHd) = pos >= 0 ? raw[i].lo : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(out + i * kHd + 64) = pos >= 0 ? raw[i].hi : make_uint4(0, 0, 0, 0);
      }
}

// A page's part in a call: unit (sequence, touched page, HP KV heads, keys or values).
struct PageUnit {
  int p0, p1, base, row0, h;   // positions p0 .. p1 - 1 are written; row of position p: row0 + p; first head
  bool is_k;
  int8_t* data;                // the page's (page_size, 128) of the head
  float* scale;
};
template <int HP = 1>
__device__ __forceinline__ bool page_unit(const AppendArgs& a, long long unit, bool leader, PageUnit& u) {
  const int parts = (a.c.Hkv + HP - 1) / HP;
  u.is_k = (unit & 1) == 0;
  u.h = (int)((unit >> 1) % parts) * HP;
  const int sj = (int)((unit >> 1) / parts), s = sj / a.most, j = sj - s * a.most;
  const Span sp = span_of(a.b, a.c.ps, s);
  if (sp.bad && j == 0 && leader) set_status(a.status, UWC_DEV_RANGE);
  if (sp.idle || sp.n <= 0) return false;
  const int ps = a.c.ps, slot = (sp.start >> a.c.lg) + j;
  u.base = slot * ps;
  u.p0 = max(sp.start, u.base);
  u.p1 = min(sp.start + sp.n, u.base + ps);        // positions written here
  if (u.p0 >= u.p1) return false;
  u.row0 = sp.row0 - sp.start;
  const int page = page_at(a.b, a.c, s, slot);
  if (page < 0 || (u.is_k && u.p1 > a.max_pos)) {
    if (leader) set_status(a.status, UWC_DEV_RANGE);
    return false;
  }
  const size_t ph = (size_t)page * a.c.Hkv + u.h;
  u.scale = (u.is_k ? a.c.sk : a.c.sv) + ph;
  u.data = (u.is_k ? a.c.k : a.c.v) + ph * ps * kHd;
  return true;
}

// A lane's 16 values of the row at position p, rotated where they are a key's.
template <typename T, bool NORM>
__device__ __forceinline__ void row_values(const AppendArgs& a, const PageUnit& u, const Raw& raw, int p, bool live, int c,
                                           float* lo, float* hi) {
  unpack8<T>(raw.lo, lo);
  unpack8<T>(raw.hi, hi);
  if (!u.is_k) return;
  if (NORM && a.k_norm) norm_head(a.k_norm, a.eps, c, lo, hi);
  if (!live) return;
#pragma unroll
  for (int i = 0; i < 2; i++) rotate4(load_turn(a.cos, a.sin, p, c, i), lo + 4 * i, hi + 4 * i);
}
__device__ __forceinline__ float row_max(const float* lo, const float* hi) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) m = fmaxf(m, fmaxf(finite_abs(lo[i]), finite_abs(hi[i])));
  return m;
}
__device__ __forceinline__ void store_row(const PageUnit& u, int p, int c, const float* lo, const float* hi, float s, float inv) {
  int8_t* d = u.data + (size_t)(p - u.base) * kHd + 8 * c;
  *reinterpret_cast<uint2*>(d) = make_uint2(quant4(lo, s, inv), quant4(lo + 4, s, inv));
  *reinterpret_cast<uint2*>(d + 64) = make_uint2(quant4(hi, s, inv), quant4(hi + 4, s, inv));
}
// The tokens that the page already holds, brought from scale s0 to a grown one: n threads, 16 values a step.
__device__ __forceinline__ void requantize(const PageUnit& u, float s0, float s, float inv, int tid, int n) {
  uint4* d = reinterpret_cast<uint4*>(u.data);
#pragma unroll 4
  for (int w = tid; w < (u.p0 - u.base) * (kHd / 16); w += n) {
    const uint4 x = d[w];
    uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = __fmul_rn((float)(int8_t)(y[k] >> (8 * i)), s0);
      y[k] = quant4(f, s, inv, -128.f);
    }
    d[w] = make_uint4(y[0], y[1], y[2], y[3]);
  }
}

// Four of a lane's low and of its high values.
template <typename T>
__device__ __forceinline__ void unpack4(const Raw& r, int k, float* lo, float* hi) {
  const uint32_t* l = reinterpret_cast<const uint32_t*>(&r.lo) + 2 * k;
  const uint32_t* h = reinterpret_cast<const uint32_t*>(&r.hi) + 2 * k;
  const float2 a = paged::two_f(l[0], T()), b = paged::two_f(l[1], T()), c = paged::two_f(h[0], T()), d = paged::two_f(h[1], T());
  lo[0] = a.x, lo[1] = a.y, lo[2] = b.x, lo[3] = b.y;
  hi[0] = c.x, hi[1] = c.y, hi[2] = d.x, hi[3] = d.y;
}

// Prompts: one CTA a page unit of HP heads, its rows in NP passes of TH / 8. All rows' loads are issued first
// and stay packed (16 bits); without a norm a key is rotated twice, for the maximum and for its quantization,
// which costs less than the registers that would hold it (80 for pages of 64 and 128, three CTAs an SM; 64 for
// pages of 16 and 32, four). What bounds it is latency at that occupancy: a CTA loads, waits for its maximum,
// stores and leaves, nothing of which overlaps inside it. Of 8 prompts of 2048's 63 us the schedulers issue in 55 %
// of the cycles, with a third of the warps resident and DRAM at 38 %. Two heads share the rotation values, which are
// four times a key's bytes (13 x up to 777 tokens of 12 + 2 x 4 heads, pages of 16: 13.2 us instead of 15.2). Pages
// of 16 have CTAs of half the size: half of 256 threads had no row. A norm takes a head's 128 values at once and runs
// in both passes: 135 us with norms where it is 62 without.
template <typename T, int NP, int TH, int HP, bool NORM>
__global__ void __launch_bounds__(TH, (NORM ? 2 : NP * HP == 4 ? 3 : 4) * kThreads / TH) k_paged_append(const AppendArgs a) {
  const int tid = threadIdx.x, c = tid & 7, r8 = tid >> 3;
  const long long units = (long long)a.b.seqs * a.most * ((a.c.Hkv + HP - 1) / HP) * 2;
  if (blockIdx.x >= units) {
    query_unit<T, NORM>(a, (blockIdx.x - units) * (TH / 8) + r8, c);
    return;
  }
  PageUnit u;
  if (!page_unit<HP>(a, blockIdx.x, tid == 0, u)) return;
  const int heads = min(HP, a.c.Hkv - u.h);
  float s0[HP];
  Raw raw[NP][HP];
#pragma unroll
  for (int g = 0; g < HP; g++) s0[g] = u.p0 > u.base && g < heads ? u.scale[g] : 0.f;
#pragma unroll
  for (int n = 0; n < NP; n++) {
    const int p = u.base + n * (TH / 8) + r8;
#pragma unroll
    for (int g = 0; g < HP; g++) {
      raw[n][g] = Raw{};
      if (p >= u.p0 && p < u.p1 && g < heads) raw[n][g] = load_raw<T>(u.is_k ? a.k : a.v, u.row0 + p, u.h + g, c);
    }
  }
  // a row's values, four low and four high dims of a head at a time
  auto each = [&](int n, auto&& f) {
    const int p = u.base + n * (TH / 8) + r8;
    const bool live = p >= u.p0 && p < u.p1;
    if (NORM) {
      float lo[8], hi[8];
      row_values<T, NORM>(a, u, raw[n][0], p, live, c, lo, hi);
      if (live)
#pragma unroll
        for (int k = 0; k < 2; k++) f(0, k, lo + 4 * k, hi + 4 * k);
    } else if (live) {
#pragma unroll
      for (int k = 0; k < 2; k++) {
        Turn4 t;
        if (u.is_k) t = load_turn(a.cos, a.sin, p, c, k);
#pragma unroll
        for (int g = 0; g < HP; g++) {
          float lo[4], hi[4];
          unpack4<T>(raw[n][g], k, lo, hi);
          if (u.is_k) rotate4(t, lo, hi);
          f(g, k, lo, hi);
        }
      }
    }
  };
  // the largest magnitudes (a maximum passes NaN over); infinities do not count, and are rare
  float amax[HP], sn[HP], inv[HP];
#pragma unroll
  for (int g = 0; g < HP; g++) amax[g] = 0.f;
#pragma unroll
  for (int n = 0; n < NP; n++)
    each(n, [&](int g, int, const float* lo, const float* hi) {
#pragma unroll
      for (int i = 0; i < 4; i++) amax[g] = fmaxf(amax[g], fmaxf(fabsf(lo[i]), fabsf(hi[i])));
    });
  __shared__ float red[HP][TH / 32];
  bool infinite = false;
#pragma unroll
  for (int g = 0; g < HP; g++) {
    amax[g] = block_maxf<TH>(amax[g], red[g]);
    infinite |= amax[g] > FLT_MAX;
  }
  if (infinite) {
    __syncthreads();                               // red is used again
#pragma unroll
    for (int g = 0; g < HP; g++) amax[g] = 0.f;
#pragma unroll
    for (int n = 0; n < NP; n++)
      each(n, [&](int g, int, const float* lo, const float* hi) {
#pragma unroll
        for (int i = 0; i < 4; i++) amax[g] = fmaxf(amax[g], fmaxf(finite_abs(lo[i]), finite_abs(hi[i])));
      });
#pragma unroll
    for (int g = 0; g < HP; g++) amax[g] = block_maxf<TH>(amax[g], red[g]);
  }
#pragma unroll
  for (int g = 0; g < HP; g++) {
    sn[g] = fmaxf(s0[g], __fdiv_rn(amax[g], 127.0f));
    inv[g] = inverse(sn[g]);
  }
  const size_t head = (size_t)a.c.ps * kHd;
#pragma unroll
  for (int n = 0; n < NP; n++) {
    int8_t* d = u.data + (size_t)(n * (TH / 8) + r8) * kHd + 8 * c;
    each(n, [&](int g, int k, const float* lo, const float* hi) {
      if (g < heads) {
        *reinterpret_cast<uint32_t*>(d + g * head + 4 * k) = quant4(lo, sn[g], inv[g]);
        *reinterpret_cast<uint32_t*>(d + g * head + 4 * k + 64) = quant4(hi, sn[g], inv[g]);
      }
    });
  }
#pragma unroll
  for (int g = 0; g < HP; g++)
    if (g < heads) {
      PageUnit v = u;
      v.data += g * head;
      if (u.p0 > u.base && sn[g] > s0[g]) requantize(v, s0[g], sn[g], inv[g], tid, TH);
      if (tid == 0) u.scale[g] = sn[g];   // after block_maxf's barriers: every thread has read s0
    }
}

// Decode steps (at most kFewNew new tokens a sequence): one warp a page unit, so that a batch's units are
// all resident at once and none waits at a barrier. Eight is what two rows a lane hold; against the page kernel (32 + 2 x 8
// heads): 64 sequences with 1 new token 4.6 us and 8.7 (pages of 64; of 16: 4.2 and 5.3), with 4 4.9 and 8.8, with 8
// 6.7 and 9.7 (6.2 either way); with norms 5.7 and 17 for 1 token.
constexpr int kFewNew = 8;
constexpr int kFewThreads = 128;
template <typename T, bool NORM>
__global__ void __launch_bounds__(kFewThreads) k_paged_append_few(const AppendArgs a) {
  const int lane = threadIdx.x & 31, c = lane & 7, r4 = lane >> 3;
  const long long units = (long long)a.b.seqs * a.most * a.c.Hkv * 2;
  const long long unit = (long long)blockIdx.x * (kFewThreads / 32) + threadIdx.x / 32;
  if (unit >= units) {
    if (a.q.p) query_unit<T, NORM>(a, (unit - units) * 4 + r4, c);
    return;
  }
  PageUnit u;
  if (!page_unit(a, unit, lane == 0, u)) return;
  const float s0 = u.p0 > u.base ? *u.scale : 0.f;
  constexpr int NP = kFewNew / 4;
  float lo[NP][8], hi[NP][8], amax = 0.f;
#pragma unroll
  for (int n = 0; n < NP; n++) {
    const int p = u.p0 + 4 * n + r4;
    const bool live = p < u.p1;
    Raw raw = {};
    if (live) raw = load_raw<T>(u.is_k ? a.k : a.v, u.row0 + p, u.h, c);
    row_values<T, NORM>(a, u, raw, p, live, c, lo[n], hi[n]);
    if (live) amax = fmaxf(amax, row_max(lo[n], hi[n]));
  }
  amax = warp_maxf(amax);
  const float sn = fmaxf(s0, __fdiv_rn(amax, 127.0f)), inv = inverse(sn);
#pragma unroll
  for (int n = 0; n < NP; n++) {
    const int p = u.p0 + 4 * n + r4;
    if (p < u.p1) store_row(u, p, c, lo[n], hi[n], sn, inv);
  }
  if (u.p0 > u.base && sn > s0) requantize(u, s0, sn, inv, lane, 32);
  __syncwarp();
  if (lane == 0) *u.scale = sn;
}

struct GatherArgs {
  Cache c;
  Seqs b;                  // start: first position to read; cu: rows of the output
  void *k, *v;             // (rows, Hkv, 128)
  uint32_t* status;
};

__device__ __forceinline__ void store8(__nv_bfloat16* o, const float* f) { *reinterpret_cast<uint4*>(o) = pack8<__nv_bfloat16>(f); }
__device__ __forceinline__ void store8(__half* o, const float* f) { *reinterpret_cast<uint4*>(o) = pack8<__half>(f); }
__device__ __forceinline__ void store8(float* o, const float* f) {
  reinterpret_cast<float4*>(o)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(o)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// 16 lanes a (token, KV head), eight dims each, keys and values both.
template <typename O>
__global__ void __launch_bounds__(kThreads) k_paged_gather(const GatherArgs a) {
  const int s = blockIdx.y;
  const Span sp = span_of(a.b, a.c.ps, s);
  if (sp.bad && blockIdx.x == 0 && threadIdx.x == 0) set_status(a.status, UWC_DEV_RANGE);
  const long long u = (long long)blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4);
  const int t = (int)(u / a.c.Hkv), h = (int)(u - (long long)t * a.c.Hkv), c = threadIdx.x & 15;
  if (t >= sp.n) return;
  const int pos = sp.start + t, ps = a.c.ps;
  const int page = sp.idle ? -1 : page_at(a.b, a.c, s, pos >> a.c.lg);
  if (page < 0 && !sp.idle) set_status(a.status, UWC_DEV_RANGE);
  const size_t out = ((size_t)(sp.row0 + t) * a.c.Hkv + h) * kHd + 8 * c;
  uint2 w[2] = {make_uint2(0, 0), make_uint2(0, 0)};
  float sc[2] = {0.f, 0.f};
  if (page >= 0) {
    const size_t ph = (size_t)page * a.c.Hkv + h, at = (ph * ps + (pos & (ps - 1))) * kHd + 8 * c;
    w[0] = *reinterpret_cast<const uint2*>(a.c.k + at);
    w[1] = *reinterpret_cast<const uint2*>(a.c.v + at);
    sc[0] = a.c.sk[ph];
    sc[1] = a.c.sv[ph];
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = __fmul_rn((float)(int8_t)((e < 4 ? w[i].x : w[i].y) >> (8 * (e & 3))), sc[i]);
    store8(reinterpret_cast<O*>(i ? a.v : a.k) + out, f);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

// The checks that every paged call shares: UWC_OK, or why not.
int uwc_paged_check(Cache* cache, const Seqs* seqs) {
  Cache& c = *cache;
  const Seqs& b = *seqs;
  if (!c.k || !c.sk || !c.v || !c.sv || (b.seqs && (!b.table || !b.start || !b.cu))) return UWC_ERR_ARG;
  if (c.pages < 1 || c.Hkv < 1 || (c.ps != 16 && c.ps != 32 && c.ps != 64 && c.ps != 128)) return UWC_ERR_SHAPE;
  if (b.seqs < 0 || b.seqs > 65535 || b.width < 1 || b.rows < 0 || b.max_new < 0) return UWC_ERR_SHAPE;
  if ((long long)b.width * c.ps > (1ll << 30) || b.rows > (1 << 30)) return UWC_ERR_SHAPE;
  if ((long long)c.pages * c.Hkv * c.ps > 0x7fffffffll) return UWC_ERR_SHAPE;   // 256 GB of keys
  if (!aligned16(c.k) || !aligned16(c.v)) return UWC_ERR_ALIGN;
  c.lg = c.ps == 16 ? 4 : c.ps == 32 ? 5 : c.ps == 64 ? 6 : 7;
  return UWC_OK;
}

namespace {

bool row_strides_ok(long long tok, long long head) { return tok >= 0 && head >= 0 && tok % 8 == 0 && head % 8 == 0; }

template <typename T, int NP, int TH, int HP, bool NORM>
int launch_pages(const AppendArgs& a, cudaStream_t st) {
  const long long units = (long long)a.b.seqs * a.most * ((a.c.Hkv + HP - 1) / HP) * 2;
  const long long queries = a.q.p ? (long long)a.b.rows * ((a.H + kQHeads - 1) / kQHeads) : 0;
  const long long grid = units + (queries * 8 + TH - 1) / TH;
  if (grid > 0x7fffffffll) return UWC_ERR_SHAPE;
  k_paged_append<T, NP, TH, HP, NORM><<<(unsigned)grid, TH, 0, st>>>(a);
  uwc_count_launch();
  return uwc_launch_status();
}
template <typename T, bool NORM>
int launch_append(const AppendArgs& a, cudaStream_t st) {
  if (a.b.max_new <= kFewNew) {
    const long long units = (long long)a.b.seqs * a.most * a.c.Hkv * 2;
    const long long queries = a.q.p ? (long long)a.b.rows * ((a.H + kQHeads - 1) / kQHeads) : 0;
    const long long per = kFewThreads / 32, grid = (units + (queries + 3) / 4 + per - 1) / per;
    if (grid > 0x7fffffffll) return UWC_ERR_SHAPE;
    k_paged_append_few<T, NORM><<<(unsigned)grid, kFewThreads, 0, st>>>(a);
    uwc_count_launch();
    return uwc_launch_status();
  }
  constexpr int HP = NORM ? 1 : 2;                 // a norm holds a whole head's values
  if (a.c.ps == 128) return launch_pages<T, 4, kThreads, 1, NORM>(a, st);
  if (a.c.ps == 64) return launch_pages<T, 2, kThreads, HP, NORM>(a, st);
  if (a.c.ps == 32) return launch_pages<T, 1, kThreads, HP, NORM>(a, st);
  return launch_pages<T, 1, kThreads / 2, HP, NORM>(a, st);
}

}  // namespace

extern "C" int uwc_paged_append(int8_t* kc, float* sk, int8_t* vc, float* sv, int pages, int page_size, int Hkv,
                                const int* table, const int* start, const int* cu, int seqs, int width, int rows,
                                int max_new, int dtype, const void* k, long long k_tok, long long k_head,
                                const void* v, long long v_tok, long long v_head, const void* q, long long q_tok,
                                long long q_head, void* q_out, int H, const float* cos, const float* sin, int max_pos,
                                const float* q_norm, const float* k_norm, double eps, void* stream) {
  AppendArgs a = {};
  a.c = Cache{kc, sk, vc, sv, pages, page_size, Hkv, 0};
  a.b = Seqs{table, start, cu, seqs, width, rows, max_new};
  const int rc = uwc_paged_check(&a.c, &a.b);
  if (rc != UWC_OK) return rc;
  if ((rows && (!k || !v)) || !cos || !sin || (dtype != UWC_T_BF16 && dtype != UWC_T_F16) || (q && !q_out)) return UWC_ERR_ARG;
  if (max_pos < 1 || (q && H < 1)) return UWC_ERR_SHAPE;
  if (!aligned16(k) || !aligned16(v) || !aligned16(cos) || !aligned16(sin) || !row_strides_ok(k_tok, k_head) ||
      !row_strides_ok(v_tok, v_head))
    return UWC_ERR_ALIGN;
  if (q && (!aligned16(q) || !aligned16(q_out) || !row_strides_ok(q_tok, q_head))) return UWC_ERR_ALIGN;
  UWC_CHECK_DEVICE();
  if (seqs == 0 || rows == 0 || max_new == 0) return UWC_OK;
  a.k = Rows{k, k_tok, k_head};
  a.v = Rows{v, v_tok, v_head};
  a.q = Rows{q, q_tok, q_head};
  a.q_out = q_out;
  a.H = H;
  a.max_pos = max_pos;
  a.most = (int)std::min(((long long)max_new + page_size - 2) / page_size + 1, (long long)width);
  a.cos = cos;
  a.sin = sin;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = (float)eps;
  a.status = uwc_status_ptr();
  const cudaStream_t st = (cudaStream_t)stream;
  const bool norm = q_norm || k_norm;
  if (dtype == UWC_T_BF16) return norm ? launch_append<__nv_bfloat16, true>(a, st) : launch_append<__nv_bfloat16, false>(a, st);
  return norm ? launch_append<__half, true>(a, st) : launch_append<__half, false>(a, st);
}

extern "C" int uwc_paged_gather(const int8_t* kc, const float* sk, const int8_t* vc, const float* sv, int pages,
                                int page_size, int Hkv, const int* table, const int* first, const int* cu, int seqs,
                                int width, int rows, int max_rows, int dtype, void* k, void* v, void* stream) {
  GatherArgs a = {};
  a.c = Cache{const_cast<int8_t*>(kc), const_cast<float*>(sk), const_cast<int8_t*>(vc), const_cast<float*>(sv), pages,
              page_size, Hkv, 0};
  a.b = Seqs{table, first, cu, seqs, width, rows, max_rows};
  const int rc = uwc_paged_check(&a.c, &a.b);
  if (rc != UWC_OK) return rc;
  if ((rows && (!k || !v)) || (dtype != UWC_T_BF16 && dtype != UWC_T_F16 && dtype != UWC_T_F32)) return UWC_ERR_ARG;
  if (!aligned16(k) || !aligned16(v)) return UWC_ERR_ALIGN;
  UWC_CHECK_DEVICE();
  if (seqs == 0 || rows == 0 || max_rows == 0) return UWC_OK;
  const long long per = ((long long)max_rows * Hkv * 16 + kThreads - 1) / kThreads;
  if (per > 0x7fffffffll) return UWC_ERR_SHAPE;
  a.k = k;
  a.v = v;
  a.status = uwc_status_ptr();
  const dim3 grid((unsigned)per, (unsigned)seqs);
  const cudaStream_t st = (cudaStream_t)stream;
  if (dtype == UWC_T_BF16) k_paged_gather<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a);
  else if (dtype == UWC_T_F16) k_paged_gather<__half><<<grid, kThreads, 0, st>>>(a);
  else k_paged_gather<float><<<grid, kThreads, 0, st>>>(a);
  uwc_count_launch();
  return uwc_launch_status();
}
