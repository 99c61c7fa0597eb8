// Attention over the paged 8-bit KV cache on sm_100a.
//
// Query row (token t of sequence s, head h) stands at position p = start[s] + t and sees key j of its
// own sequence when j <= p and (no window, or j > p - window, or j < sinks):
//   o = sum_j softmax_j(q . k_j s_k(page of j) scale) v_j s_v(page of j)
// with k_j, v_j the cache's integers. A row that sees nothing (an idle slot, window 0 without sinks)
// is zero.
#include <cfloat>

#include "paged.cuh"
#include "uwc_host.h"

namespace {

using paged::Cache;
using paged::kHd;
using paged::page_at;
using paged::Seqs;
using paged::Span;
using paged::span_of;

struct AttnArgs {
  Cache c;
  Seqs b;
  const void* q;           // element (n, h, d) at n * q_tok + h * q_head + d
  long long q_tok, q_head;
  void* out;               // (rows, H, 128)
  int H, window, sinks;    // window < 0: none
  float scale;
  uint32_t* status;
};

__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// One warp a (token, query head), one key a step, four dims a lane: the online softmax in registers.
template <typename T>
__global__ void __launch_bounds__(128) k_paged_attention(const AttnArgs a) {
  const int s = blockIdx.y, lane = threadIdx.x & 31;
  const Span sp = span_of(a.b, a.c.ps, s);
  if (sp.bad && blockIdx.x == 0 && threadIdx.x == 0) set_status(a.status, UWC_DEV_RANGE);
  const long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(u / a.H), h = (int)(u % a.H), g = h / (a.H / a.c.Hkv);
  if (t >= sp.n) return;
  const size_t row = (size_t)(sp.row0 + t);
  const T* q = reinterpret_cast<const T*>(a.q) + row * a.q_tok + h * a.q_head + 4 * lane;
  float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) qv[i] = to_f(q[i]) * a.scale;
  const int p = sp.start + t;
  const int lo = a.window < 0 ? 0 : max(0, p - a.window + 1);
  for (int j = 0; !sp.idle && j <= p; j++) {
    if (j < lo && j >= a.sinks) {
      j = lo - 1;
      continue;
    }
    const int page = page_at(a.b, a.c, s, j / a.c.ps);
    if (page < 0) {
      set_status(a.status, UWC_DEV_RANGE);
      continue;
    }
    const size_t ph = (size_t)page * a.c.Hkv + g, at = (ph * a.c.ps + j % a.c.ps) * kHd + 4 * lane;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(a.c.k + at);
    const uint32_t vw = *reinterpret_cast<const uint32_t*>(a.c.v + at);
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) d += qv[i] * (float)(int8_t)(kw >> (8 * i));
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
    d *= a.c.sk[ph];
    const float m2 = fmaxf(m, d), f = m2 == -INFINITY ? 1.f : expf(m - m2), w = d == -INFINITY ? 0.f : expf(d - m2);
    const float wv = w * a.c.sv[ph];
    l = l * f + w;
    m = m2;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = o[i] * f + wv * (float)(int8_t)(vw >> (8 * i));
  }
  const float r = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
  T* out = reinterpret_cast<T*>(a.out) + (row * a.H + h) * kHd + 4 * lane;
#pragma unroll
  for (int i = 0; i < 4; i++) out[i] = from_f<T>(o[i] * r);
}

}  // namespace

extern "C" uint64_t uwc_paged_attention_workspace_bytes(int seqs, int max_new, int max_len, int H, int Hkv, int window,
                                                        int sinks) {
  return 0;
}

extern "C" int uwc_paged_attention(const int8_t* kc, const float* sk, const int8_t* vc, const float* sv, int pages,
                                   int page_size, int Hkv, const int* table, const int* start, const int* cu, int seqs,
                                   int width, int rows, int max_new, int max_len, int dtype, const void* q,
                                   long long q_tok, long long q_head, void* out, int H, float scale, int window,
                                   int sinks, void* workspace, uint64_t workspace_bytes, void* stream) {
  AttnArgs a = {};
  a.c = Cache{const_cast<int8_t*>(kc), const_cast<float*>(sk), const_cast<int8_t*>(vc), const_cast<float*>(sv), pages,
              page_size, Hkv};
  a.b = Seqs{table, start, cu, seqs, width, rows, max_new};
  const int rc = uwc_paged_check(&a.c, &a.b);
  if (rc != UWC_OK) return rc;
  if (!q || !out || (dtype != UWC_T_BF16 && dtype != UWC_T_F16)) return UWC_ERR_ARG;
  if (H < 1 || H % Hkv || max_len < 0 || sinks < 0) return UWC_ERR_SHAPE;
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
  const dim3 grid((unsigned)(((long long)max_new * H + 3) / 4), (unsigned)seqs);
  if (dtype == UWC_T_BF16) k_paged_attention<__nv_bfloat16><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
  else k_paged_attention<__half><<<grid, 128, 0, (cudaStream_t)stream>>>(a);
  uwc_count_launch();
  return uwc_launch_status();
}
