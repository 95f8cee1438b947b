// g4_paged_attn.cu -- attention of new tokens over paged, quantised keys and values.
#include <cuda_runtime.h>
#include <math.h>

#include "g4_device.cuh"
#include "g4_kernels.cuh"
#include "g4_paged.cuh"

namespace g4 {

// One warp per (row, head), one position at a time, f32 throughout. With V = scale * code the
// running maximum is that of score + ln(scale), so that the greatest weight p * scale of a row is
// always 1, however far the scales lie apart.
__device__ __forceinline__ float paged_code(const Pool &p, const uint8_t *base, long long row, int d) {
  if (p.fmt == G4_PAGE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(base)[row * p.hd + d]);
  const uint8_t c = base[row * p.hd + d];
  if (p.fmt == G4_PAGE_INT8) return (float)(int8_t)c;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

__global__ void __launch_bounds__(128) k_paged_attention(const PagedAttn a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.y;
  const SeqSpan s = seq_span(a, b);
  const long long item = (long long)blockIdx.x * 4 + warp;
  const int i = (int)(item / a.heads), h = (int)(item % a.heads);
  if (i >= s.n) return;
  const Pool &p = a.pool;
  const int kvh = h / a.group, hd = p.hd;
  float q[16], o[16];
  const long long qo = (long long)(s.row + i) * a.q_stride + (long long)h * hd;
  for (int j = 0; j < hd / 32; j++) {
    const int d = j * 32 + lane;
    q[j] = a.type == G4_F32 ? ((const float *)a.q)[qo + d] : __bfloat162float(((const __nv_bfloat16 *)a.q)[qo + d]);
    o[j] = 0.0f;
  }
  int lo, hi;
  row_range(a, s.pos + i, s.kv, lo, hi);
  float m = -INFINITY, l = 0.0f;
  for (int t = lo; t < hi; t++) {
    const int page = a.table[(long long)b * a.table_stride + t / p.page_size];
    if (page < 0 || page >= p.n_pages) {
      if (lane == 0) paged_raise(a.err, G4_PAGED_BAD_PAGE);
      continue;
    }
    const long long row = ((long long)page * p.kv_heads + kvh) * p.page_size + t % p.page_size;
    float dot = 0.0f;
    for (int j = 0; j < hd / 32; j++) dot = fmaf(q[j], paged_code(p, p.k, row, j * 32 + lane), dot);
    dot = warp_sum_bfly(dot) * a.scale * (p.ks ? p.ks[row] : 1.0f);
    const float vs = p.vs ? p.vs[row] : 1.0f;
    const float mn = fmaxf(m, dot + logf(fmaxf(vs, 0x1p-100f))), r = expf(m - mn), w = expf(dot - mn);
    l = l * r + w;
    for (int j = 0; j < hd / 32; j++) o[j] = fmaf(w * vs, paged_code(p, p.v, row, j * 32 + lane), o[j] * r);
    m = mn;
  }
  const long long oo = (long long)(s.row + i) * a.o_stride + (long long)h * hd;
  for (int j = 0; j < hd / 32; j++) {
    const float v = l > 0.0f ? o[j] / l : 0.0f;
    const int d = j * 32 + lane;
    if (a.type == G4_F32)
      ((float *)a.out)[oo + d] = v;
    else
      ((__nv_bfloat16 *)a.out)[oo + d] = __float2bfloat16_rn(v);
  }
  if (lane == 0 && a.lse) a.lse[(long long)(s.row + i) * a.heads + h] = m + logf(l);
}

size_t paged_attention_partials(const PagedAttn &) { return 0; }

cudaError_t launch_paged_attention(const PagedAttn &a, cudaStream_t st) {
  const dim3 grid((unsigned)(((long long)a.max_q * a.heads + 3) / 4), (unsigned)a.batch);
  return launch_k(k_paged_attention, grid, dim3(128), 0, st, false, a);
}

}  // namespace g4
