// The paged 8-bit KV cache on sm_100a: new tokens in, values back out.
//
//   k_paged_append   rotates the new keys (and the queries) and stores keys and values as int8 with
//                    one scale for each (page, KV head). With x a page's new values in float32 and
//                    s0 the scale of the tokens that it already holds (0 where it holds none),
//                      s = max(s0, fdiv(max|x|, 127)),  q(x) = clamp(rint(fdiv(x, s)), +-127),
//                    and an old token's q becomes rint(fdiv(fmul(q, s0), s)) when s > s0. Every step
//                    is one IEEE operation, the rotation too (fadd(fmul(x, cos), fmul(rot(x), sin))),
//                    so a cache is the same bit for bit wherever and in whatever batch it was written,
//                    and appending the same tokens again changes nothing.
//   k_paged_gather   cached tokens back as 16- or 32-bit values.
//
// Both are bound by HBM at prompt sizes and by latency at decode sizes.
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
constexpr int kQHeads = 4;       // query heads that share a thread's rotation values

// Eight 16-bit values as float32.
__device__ __forceinline__ void unpack8(const uint4 w, float* f, __nv_bfloat16) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const uint4 w, float* f, __half) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
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

// A token head lies in eight threads: thread c of them holds dims 8 c .. 8 c + 7 (lo) and their
// rotation partners 64 + 8 c .. (hi).
template <typename T>
__device__ __forceinline__ void load_head(const Rows& r, long long row, int h, int c, float* lo, float* hi) {
  const T* p = reinterpret_cast<const T*>(r.p) + row * r.tok + h * r.head + 8 * c;
  unpack8(*reinterpret_cast<const uint4*>(p), lo, T());
  unpack8(*reinterpret_cast<const uint4*>(p + 64), hi, T());
}

// det_rmsnorm over the head (exact fixed-point sum of 128 squares, runtime/detrt/core.py:151-159)
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

struct Turn {              // one token's rotation values for a thread's dims
  float4 v[8];             // cos lo, cos hi, sin lo, sin hi (two float4 each)
};
__device__ __forceinline__ Turn load_turn(const float* cos, const float* sin, int pos, int c) {
  Turn t;
  const float4* a = reinterpret_cast<const float4*>(cos + (size_t)pos * kHd) + 2 * c;
  const float4* b = reinterpret_cast<const float4*>(sin + (size_t)pos * kHd) + 2 * c;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    t.v[i] = __ldg(a + i);
    t.v[2 + i] = __ldg(a + 16 + i);
    t.v[4 + i] = __ldg(b + i);
    t.v[6 + i] = __ldg(b + 16 + i);
  }
  return t;
}
__device__ __forceinline__ void rotate(const Turn& t, float* lo, float* hi) {
  const float* f = reinterpret_cast<const float*>(t.v);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float x = lo[i], y = hi[i];
    lo[i] = __fadd_rn(__fmul_rn(x, f[i]), __fmul_rn(-y, f[16 + i]));
    hi[i] = __fadd_rn(__fmul_rn(y, f[8 + i]), __fmul_rn(x, f[24 + i]));
  }
}

// A value's part in its page's scale: its magnitude, 0 for infinities and NaN (stored as +-127 and 0).
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= FLT_MAX ? a : 0.f;
}
__device__ __forceinline__ uint32_t quant4(const float* x, float s) {
  uint32_t o = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float v = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -127.f), 127.f) : 0.f;
    const int q = x[i] == x[i] ? (int)v : 0;
    o |= (uint32_t)(q & 255) << (8 * i);
  }
  return o;
}

// Page units: one CTA for the new tokens of one (sequence, touched page, KV head) and of keys or
// values. The page's new rows stay in registers between their maximum and their quantization (NP
// passes of 32 token rows). Query units: 32 (token, four query heads) a CTA.
template <typename T, int NP>
__global__ void __launch_bounds__(kThreads) k_paged_append(const AppendArgs a) {
  const int tid = threadIdx.x, c = tid & 7, r8 = tid >> 3;
  const long long units = (long long)a.b.seqs * a.most * a.c.Hkv * 2;
  if (blockIdx.x >= units) {
    // ---- queries
    const int groups = (a.H + kQHeads - 1) / kQHeads;
    const long long u = (blockIdx.x - units) * (kThreads / 8) + r8;
    const int row = (int)(u / groups), h0 = (int)(u % groups) * kQHeads;
    const bool in = row < a.b.rows;
    int pos = -1;
    bool covered = false;
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
    // (all threads stay for the norm's shuffles)
    Turn tn = {};
    if (pos >= 0) tn = load_turn(a.cos, a.sin, pos, c);
#pragma unroll
    for (int i = 0; i < kQHeads; i++) {
      const int h = h0 + i;
      float lo[8] = {}, hi[8] = {};
      if (pos >= 0 && h < a.H) load_head<T>(a.q, row, h, c, lo, hi);
      if (a.q_norm) norm_head(a.q_norm, a.eps, c, lo, hi);
      if (pos >= 0) rotate(tn, lo, hi);
      else
#pragma unroll
        for (int j = 0; j < 8; j++) lo[j] = hi[j] = 0.f;
      if (covered && h < a.H) {
        T* o = reinterpret_cast<T*>(a.q_out) + ((size_t)row * a.H + h) * kHd + 8 * c;
        *reinterpret_cast<uint4*>(o) = pack8<T>(lo);
        *reinterpret_cast<uint4*>(o + 64) = pack8<T>(hi);
      }
    }
    return;
  }
  // ---- keys and values
  const int unit = blockIdx.x;
  const bool is_k = (unit & 1) == 0;
  const int h = (unit >> 1) % a.c.Hkv, sj = (unit >> 1) / a.c.Hkv;
  const int s = sj / a.most, j = sj % a.most;
  const Span sp = span_of(a.b, a.c.ps, s);
  if (sp.bad && j == 0 && tid == 0) set_status(a.status, UWC_DEV_RANGE);
  if (sp.idle || sp.n <= 0) return;
  const int ps = a.c.ps, slot = (sp.start >> a.c.lg) + j, base = slot * ps;
  const int p0 = max(sp.start, base), p1 = min(sp.start + sp.n, base + ps);   // positions written here
  if (p0 >= p1) return;
  const int page = page_at(a.b, a.c, s, slot);
  if (page < 0 || (is_k && p1 > a.max_pos)) {
    if (tid == 0) set_status(a.status, UWC_DEV_RANGE);
    return;
  }
  const size_t ph = (size_t)page * a.c.Hkv + h;
  float* scale = (is_k ? a.c.sk : a.c.sv) + ph;
  int8_t* data = (is_k ? a.c.k : a.c.v) + ph * ps * kHd;
  const float s0 = p0 > base ? *scale : 0.f;
  float lo[NP][8], hi[NP][8], amax = 0.f;
#pragma unroll
  for (int n = 0; n < NP; n++) {
    const int p = base + n * 32 + r8;
    const bool live = p >= p0 && p < p1;
#pragma unroll
    for (int i = 0; i < 8; i++) lo[n][i] = hi[n][i] = 0.f;
    if (live) load_head<T>(is_k ? a.k : a.v, sp.row0 + (p - sp.start), h, c, lo[n], hi[n]);
    if (is_k) {
      if (a.k_norm) norm_head(a.k_norm, a.eps, c, lo[n], hi[n]);
      if (live) rotate(load_turn(a.cos, a.sin, p, c), lo[n], hi[n]);
    }
    if (live)
#pragma unroll
      for (int i = 0; i < 8; i++) amax = fmaxf(amax, fmaxf(finite_abs(lo[n][i]), finite_abs(hi[n][i])));
  }
  __shared__ float red[kThreads / 32];
  amax = block_maxf<kThreads>(amax, red);
  const float sn = fmaxf(s0, __fdiv_rn(amax, 127.0f));
#pragma unroll
  for (int n = 0; n < NP; n++) {
    const int p = base + n * 32 + r8;
    if (p < p0 || p >= p1) continue;
    int8_t* d = data + (size_t)(p - base) * kHd + 8 * c;
    *reinterpret_cast<uint2*>(d) = make_uint2(quant4(lo[n], sn), quant4(lo[n] + 4, sn));
    *reinterpret_cast<uint2*>(d + 64) = make_uint2(quant4(hi[n], sn), quant4(hi[n] + 4, sn));
  }
  if (p0 > base && sn > s0) {
    // the tokens that the page already holds, brought to the grown scale
    for (int w = tid; w < (p0 - base) * (kHd / 4); w += kThreads) {
      uint32_t* d = reinterpret_cast<uint32_t*>(data) + w;
      const uint32_t x = *d;
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = __fmul_rn((float)(int8_t)(x >> (8 * i)), s0);
      *d = quant4(f, sn);
    }
  }
  if (tid == 0) *scale = sn;   // after block_maxf's barriers: every thread has read s0
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

// Eight threads a (token, KV head), 16 dims each; 32 of them a CTA, keys and values both.
template <typename O>
__global__ void __launch_bounds__(kThreads) k_paged_gather(const GatherArgs a) {
  const int s = blockIdx.y;
  const Span sp = span_of(a.b, a.c.ps, s);
  if (sp.bad && blockIdx.x == 0 && threadIdx.x == 0) set_status(a.status, UWC_DEV_RANGE);
  const long long u = (long long)blockIdx.x * (kThreads / 8) + (threadIdx.x >> 3);
  const int t = (int)(u / a.c.Hkv), h = (int)(u % a.c.Hkv), c = threadIdx.x & 7;
  if (t >= sp.n) return;
  const int pos = sp.start + t, ps = a.c.ps;
  const int page = sp.idle ? -1 : page_at(a.b, a.c, s, pos >> a.c.lg);
  if (page < 0 && !sp.idle) set_status(a.status, UWC_DEV_RANGE);
  const size_t out = ((size_t)(sp.row0 + t) * a.c.Hkv + h) * kHd + 16 * c;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    uint4 w = make_uint4(0, 0, 0, 0);
    float sc = 0.f;
    if (page >= 0) {
      const size_t ph = (size_t)page * a.c.Hkv + h;
      w = *reinterpret_cast<const uint4*>((i ? a.c.v : a.c.k) + (ph * ps + (pos & (ps - 1))) * kHd + 16 * c);
      sc = (i ? a.c.sv : a.c.sk)[ph];
    }
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    float f[16];
#pragma unroll
    for (int e = 0; e < 16; e++) f[e] = __fmul_rn((float)(int8_t)(x[e >> 2] >> (8 * (e & 3))), sc);
    O* o = reinterpret_cast<O*>(i ? a.v : a.k) + out;
    store8(o, f);
    store8(o + 8, f + 8);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

// The checks that every paged call shares: UWC_OK, or why not.
int uwc_paged_check(Cache* cache, const Seqs* seqs) {
  Cache& c = *cache;
  const Seqs& b = *seqs;
  if (!c.k || !c.sk || !c.v || !c.sv || !b.table || !b.start || !b.cu) return UWC_ERR_ARG;
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

template <typename T>
int launch_append(const AppendArgs& a, long long grid, cudaStream_t st) {
  switch (a.c.ps) {
    case 128: k_paged_append<T, 4><<<(unsigned)grid, kThreads, 0, st>>>(a); break;
    case 64: k_paged_append<T, 2><<<(unsigned)grid, kThreads, 0, st>>>(a); break;
    default: k_paged_append<T, 1><<<(unsigned)grid, kThreads, 0, st>>>(a); break;
  }
  uwc_count_launch();
  return uwc_launch_status();
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
  if (!k || !v || !cos || !sin || (dtype != UWC_T_BF16 && dtype != UWC_T_F16) || (q && !q_out)) return UWC_ERR_ARG;
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
  a.most = min((max_new + page_size - 2) / page_size + 1, width);
  a.cos = cos;
  a.sin = sin;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = (float)eps;
  a.status = uwc_status_ptr();
  long long grid = (long long)seqs * a.most * Hkv * 2;
  if (q) grid += ((long long)rows * ((H + kQHeads - 1) / kQHeads) * 8 + kThreads - 1) / kThreads;
  if (grid > 0x7fffffffll) return UWC_ERR_SHAPE;
  const cudaStream_t st = (cudaStream_t)stream;
  return dtype == UWC_T_BF16 ? launch_append<__nv_bfloat16>(a, grid, st) : launch_append<__half>(a, grid, st);
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
  if (!k || !v || (dtype != UWC_T_BF16 && dtype != UWC_T_F16 && dtype != UWC_T_F32)) return UWC_ERR_ARG;
  if (!aligned16(k) || !aligned16(v)) return UWC_ERR_ALIGN;
  UWC_CHECK_DEVICE();
  if (seqs == 0 || rows == 0 || max_rows == 0) return UWC_OK;
  const long long per = ((long long)max_rows * Hkv * 8 + kThreads - 1) / kThreads;
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
