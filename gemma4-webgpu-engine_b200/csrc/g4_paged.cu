// g4_paged.cu -- the paged, quantised KV cache: rows quantised as they are written, rows read
// back, and the C entries of the paged-cache operators (include/g4.h).
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "g4_device.cuh"
#include "g4_kernels.cuh"
#include "g4_paged.cuh"

void g4_internal_set_error(const char *msg);

namespace g4 {

static __device__ int g4_paged_error;

// The flags' address per device; a lookup that fails is not remembered.
int *paged_error_flags() {
  static std::atomic<int *> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return nullptr;
  int *p = dev < 64 ? known[dev].load(std::memory_order_acquire) : nullptr;
  if (p) return p;
  void *q = nullptr;
  if (cudaGetSymbolAddress(&q, g4_paged_error) != cudaSuccess) return nullptr;
  if (dev < 64) known[dev].store((int *)q, std::memory_order_release);
  return (int *)q;
}

// ------------------------------------------------------------------------------ store, read
// A row of head_dim values is shared by head_dim / 8 lanes of a warp (two chunks of eight a lane
// at 512): 16 bytes of bf16 or 32 of f32 in, 8 bytes of codes out, so a warp's accesses cover
// whole sectors and the row's greatest magnitude is a few shuffles. K and V rows of a (token,
// head) go through the same lanes, their loads in flight together. Bound by HBM: each value is
// read once and written once.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float *p) {
    a = *reinterpret_cast<const float4 *>(p);
    b = *reinterpret_cast<const float4 *>(p + 4);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  static __device__ __forceinline__ void put(float *p, const float (&x)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  }
};
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&h);
}
template <>
struct Eight<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) { a = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void put(__nv_bfloat16 *p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]),
                                               pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  }
};

// Codes of eight values (scale s, 0 or NaN: codes 0): that of the correctly rounded quotient x / s. The
// divisions bind the kernel by instructions (82% of issue slots); multiplying by the reciprocal and
// dividing only next to the middle between two codes lost, as bf16 rows lie there often (16,389 x 8 x 128
// stored and read back: e4m3 57 us against 51).
template <int FMT>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float s) {
  uint32_t w[2] = {0, 0};
  if (!(s > 0.0f)) return make_uint2(0, 0);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float a = __fdiv_rn(x[i], s), b = __fdiv_rn(x[i + 1], s);
    uint32_t two;
    if (FMT == G4_PAGE_INT8) {
      const int ca = (int)fminf(fmaxf(rintf(a), -127.0f), 127.0f);
      const int cb = (int)fminf(fmaxf(rintf(b), -127.0f), 127.0f);
      two = (uint32_t)(ca & 0xff) | ((uint32_t)(cb & 0xff) << 8);
    } else {
      two = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    }
    w[i >> 2] |= two << (8 * (i & 2));
  }
  return make_uint2(w[0], w[1]);
}
template <int FMT>
__device__ __forceinline__ void decode8(uint2 c, float s, float (&x)[8]) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint32_t two = (w[i >> 2] >> (8 * (i & 2))) & 0xffffu;
    if (FMT == G4_PAGE_INT8) {
      x[i] = __fmul_rn((float)(int8_t)(two & 0xff), s);
      x[i + 1] = __fmul_rn((float)(int8_t)(two >> 8), s);
    } else {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
      x[i] = __fmul_rn(f.x, s);
      x[i + 1] = __fmul_rn(f.y, s);
    }
  }
}

// kRowItems: (token, head) pairs a thread has in flight, 2 where the call fills the SMs several times over
// (40,001 x 8 x 128 read back: 44 us against 53), else 1 (129 x 512: 2.9 us against 4.5).
template <typename T, int FMT, int HD, int kRowItems>
__global__ void __launch_bounds__(256)
    k_page_store(const Pool p, const T *__restrict__ k, const T *__restrict__ v, long long k_stride,
                 long long v_stride, int tokens, const int32_t *__restrict__ slots) {
  constexpr int LR = HD / 8 < 32 ? HD / 8 : 32;   // lanes per row
  constexpr int CH = HD / 8 / LR;                 // chunks of eight per lane
  constexpr int IPB = 256 / LR;                   // items a block takes side by side
  const int l = threadIdx.x % LR;
  const long long items = (long long)tokens * p.kv_heads;
  Eight<T> in[kRowItems][2][CH];
  int slot[kRowItems], head[kRowItems];
#pragma unroll
  for (int n = 0; n < kRowItems; n++) {
    const long long item = ((long long)blockIdx.x * kRowItems + n) * IPB + threadIdx.x / LR;
    const bool live = item < items;
    const int tok = live ? (int)(item / p.kv_heads) : 0;
    head[n] = live ? (int)(item - (long long)tok * p.kv_heads) : 0;
    slot[n] = live ? slots[tok] : -1;
    // (The rows are there whatever the slot: their loads do not wait for it.)
#pragma unroll
    for (int c = 0; c < CH; c++) {
      in[n][0][c].load(k + tok * k_stride + head[n] * HD + (c * LR + l) * 8);
      in[n][1][c].load(v + tok * v_stride + head[n] * HD + (c * LR + l) * 8);
    }
  }
#pragma unroll
  for (int n = 0; n < kRowItems; n++) {
    if (slot[n] >= p.n_pages * p.page_size) {
      if (l == 0) paged_raise(&g4_paged_error, G4_PAGED_BAD_PAGE);
      slot[n] = -1;
    }
    const bool on = slot[n] >= 0;
    const int page = on ? slot[n] / p.page_size : 0, off = on ? slot[n] - page * p.page_size : 0;
    const long long row = ((long long)page * p.kv_heads + head[n]) * p.page_size + off;
#pragma unroll
    for (int w = 0; w < 2; w++) {
      uint8_t *const base = w ? p.v : p.k;
      if (FMT == G4_PAGE_BF16) {
        if (on) {
#pragma unroll
          for (int c = 0; c < CH; c++) {
            float x[8];
            in[n][w][c].get(x);
            Eight<__nv_bfloat16>::put(reinterpret_cast<__nv_bfloat16 *>(base) + row * HD + (c * LR + l) * 8, x);
          }
        }
        continue;
      }
      // The greatest magnitude over the row: magnitudes order as their bits do, infinities and NaN last.
      uint32_t most = 0;
#pragma unroll
      for (int c = 0; c < CH; c++) {
        float x[8];
        in[n][w][c].get(x);
#pragma unroll
        for (int i = 0; i < 8; i++) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
      }
#pragma unroll
      for (int m = 1; m < LR; m <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, m));
      const float top = __uint_as_float(min(most, 0x7f800000u));
      float s = __fdiv_rn(top, FMT == G4_PAGE_INT8 ? 127.0f : 448.0f);
      if (s == __int_as_float(0x7f800000)) s = __int_as_float(0x7fffffff);
      if (on) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
          float x[8];
          in[n][w][c].get(x);
          *reinterpret_cast<uint2 *>(base + row * HD + (c * LR + l) * 8) = encode8<FMT>(x, s);
        }
        if (l == 0) (w ? p.vs : p.ks)[row] = s;
      }
    }
  }
}

template <typename T, int FMT, int HD, int kRowItems>
__global__ void __launch_bounds__(256)
    k_page_read(const Pool p, T *__restrict__ k, T *__restrict__ v, long long k_stride, long long v_stride,
                int tokens, const int32_t *__restrict__ slots) {
  constexpr int LR = HD / 8 < 32 ? HD / 8 : 32;
  constexpr int CH = HD / 8 / LR;
  constexpr int IPB = 256 / LR;
  const int l = threadIdx.x % LR;
  const long long items = (long long)tokens * p.kv_heads;
  using Code = typename std::conditional<FMT == G4_PAGE_BF16, uint4, uint2>::type;   // eight of them
  constexpr int ES = FMT == G4_PAGE_BF16 ? 2 : 1;
  Code in[kRowItems][2][CH];
  float s[kRowItems][2];
  int tok[kRowItems], head[kRowItems];
#pragma unroll
  for (int n = 0; n < kRowItems; n++) {
    const long long item = ((long long)blockIdx.x * kRowItems + n) * IPB + threadIdx.x / LR;
    tok[n] = item < items ? (int)(item / p.kv_heads) : -1;
    head[n] = item < items ? (int)(item - (long long)tok[n] * p.kv_heads) : 0;
    int slot = tok[n] >= 0 ? slots[tok[n]] : -1;
    if (slot >= p.n_pages * p.page_size) {
      if (l == 0) paged_raise(&g4_paged_error, G4_PAGED_BAD_PAGE);
      slot = -1;
    }
    const bool on = slot >= 0;
    const int page = on ? slot / p.page_size : 0, off = on ? slot - page * p.page_size : 0;
    const long long row = ((long long)page * p.kv_heads + head[n]) * p.page_size + off;
#pragma unroll
    for (int w = 0; w < 2; w++) {
#pragma unroll
      for (int c = 0; c < CH; c++) {
        in[n][w][c] = Code{};
        if (on) in[n][w][c] = *reinterpret_cast<const Code *>((w ? p.v : p.k) + (row * HD + (c * LR + l) * 8) * ES);
      }
      s[n][w] = 0.0f;
      if (on && FMT != G4_PAGE_BF16) s[n][w] = (w ? p.vs : p.ks)[row];
    }
  }
#pragma unroll
  for (int n = 0; n < kRowItems; n++) {
    if (tok[n] < 0) continue;
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int c = 0; c < CH; c++) {
        float x[8];
        if constexpr (FMT == G4_PAGE_BF16) {
          Eight<__nv_bfloat16> e;
          e.a = in[n][w][c];
          e.get(x);
        } else {
          decode8<FMT>(in[n][w][c], s[n][w], x);
        }
        Eight<T>::put((w ? v + tok[n] * v_stride : k + tok[n] * k_stride) + head[n] * HD + (c * LR + l) * 8, x);
      }
  }
}

template <typename T, int FMT>
cudaError_t launch_rows(const Pool &p, bool store, void *k, void *v, long long ks, long long vs, int tokens,
                        const int32_t *slots, cudaStream_t st) {
  const int lanes = p.hd / 8 < 32 ? p.hd / 8 : 32;
  const long long items = (long long)tokens * p.kv_heads, side = 256 / lanes;
  const int n = items > side * 148 * 8 * 2 ? 2 : 1;
  const dim3 grid((unsigned)((items + side * n - 1) / (side * n))), block(256);
  T *tk = (T *)k, *tv = (T *)v;
  auto go = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    if (store)
      return launch_k(n == 2 ? k_page_store<T, FMT, HD, 2> : k_page_store<T, FMT, HD, 1>, grid, block, 0, st, false, p, (const T *)tk,
                      (const T *)tv, ks, vs, tokens, slots);
    return launch_k(n == 2 ? k_page_read<T, FMT, HD, 2> : k_page_read<T, FMT, HD, 1>, grid, block, 0, st, false, p, tk, tv, ks, vs, tokens, slots);
  };
  switch (p.hd) {
    case 64: return go(std::integral_constant<int, 64>{});
    case 128: return go(std::integral_constant<int, 128>{});
    case 256: return go(std::integral_constant<int, 256>{});
    default: return go(std::integral_constant<int, 512>{});
  }
}
template <typename T>
cudaError_t launch_rows_fmt(const Pool &p, bool store, void *k, void *v, long long ks, long long vs,
                            int tokens, const int32_t *slots, cudaStream_t st) {
  switch (p.fmt) {
    case G4_PAGE_BF16: return launch_rows<T, G4_PAGE_BF16>(p, store, k, v, ks, vs, tokens, slots, st);
    case G4_PAGE_INT8: return launch_rows<T, G4_PAGE_INT8>(p, store, k, v, ks, vs, tokens, slots, st);
    default: return launch_rows<T, G4_PAGE_E4M3>(p, store, k, v, ks, vs, tokens, slots, st);
  }
}

}  // namespace g4

// ------------------------------------------------------------------------------ C entries
namespace {

int set_error(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g4_internal_set_error(buf);
  return code;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int check_pool(const char *who, const g4_page_pool *s, g4::Pool *p) {
  if (!s || !s->k || !s->v) return set_error(G4_ERR_INVALID, "%s: null pool or pages", who);
  if (s->format < G4_PAGE_BF16 || s->format > G4_PAGE_E4M3) return set_error(G4_ERR_INVALID, "%s: page format %d", who, s->format);
  if (s->head_dim != 64 && s->head_dim != 128 && s->head_dim != 256 && s->head_dim != 512)
    return set_error(G4_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128, 256 or 512)", who, s->head_dim);
  if (s->page_size < 16 || s->page_size > 1024 || s->page_size % 16)
    return set_error(G4_ERR_INVALID, "%s: page_size %d is not a multiple of 16 up to 1024", who, s->page_size);
  if (s->n_pages < 1 || s->kv_heads < 1 || s->kv_heads > 65535 || (long long)s->n_pages * s->page_size >= (1ll << 31))
    return set_error(G4_ERR_INVALID, "%s: %d pages of %d, %d KV heads", who, s->n_pages, s->page_size, s->kv_heads);
  const bool scaled = s->format != G4_PAGE_BF16;
  if (scaled && (!s->k_scale || !s->v_scale)) return set_error(G4_ERR_INVALID, "%s: 8-bit pages need their scales", who);
  if (!aligned16(s->k) || !aligned16(s->v) || (scaled && (!aligned16(s->k_scale) || !aligned16(s->v_scale))))
    return set_error(G4_ERR_INVALID, "%s: pages and scales are 16-byte aligned", who);
  *p = {(uint8_t *)s->k, (uint8_t *)s->v, s->k_scale, s->v_scale, s->n_pages, s->page_size, s->kv_heads, s->head_dim, s->format};
  return G4_OK;
}

// Rows of `width` contiguous elements `stride` apart at p: 16-byte accesses need all three to agree.
int check_rows(const char *who, const char *what, const void *p, int type, long long stride, long long width) {
  const int per16 = type == G4_F32 ? 4 : 8;
  if (!aligned16(p) || stride % per16) return set_error(G4_ERR_INVALID, "%s: %s rows are 16-byte aligned", who, what);
  if (stride < width) return set_error(G4_ERR_INVALID, "%s: %s rows of %lld elements lie %lld apart", who, what, width, stride);
  return G4_OK;
}

int check_launch(const char *who, cudaError_t e) {
  if (e == cudaSuccess) return G4_OK;
  return set_error(G4_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

int move_rows(const char *who, bool store, const g4_page_pool *pool, void *k, void *v, int32_t type, int64_t k_stride,
              int64_t v_stride, int32_t tokens, const int32_t *slots, void *stream) {
  g4::Pool p;
  if (int rc = check_pool(who, pool, &p)) return rc;
  if (!k || !v || !slots) return set_error(G4_ERR_INVALID, "%s: null pointer", who);
  if (type != G4_F32 && type != G4_BF16) return set_error(G4_ERR_INVALID, "%s: type %d", who, type);
  if (tokens < 0) return set_error(G4_ERR_INVALID, "%s: %d tokens", who, tokens);
  const long long width = (long long)p.kv_heads * p.hd;
  if (int rc = check_rows(who, "k", k, type, k_stride, width)) return rc;
  if (int rc = check_rows(who, "v", v, type, v_stride, width)) return rc;
  if (tokens == 0) return G4_OK;
  if ((long long)tokens * p.kv_heads >= (1ll << 35)) return set_error(G4_ERR_UNSUPPORTED, "%s: %d tokens of %d heads", who, tokens, p.kv_heads);
  cudaStream_t st = (cudaStream_t)stream;
  return check_launch(who, type == G4_F32
                               ? g4::launch_rows_fmt<float>(p, store, k, v, k_stride, v_stride, tokens, slots, st)
                               : g4::launch_rows_fmt<__nv_bfloat16>(p, store, k, v, k_stride, v_stride, tokens, slots, st));
}

int check_attention(const char *who, const g4_page_pool *pool, int32_t type, int32_t heads, int32_t rows,
                    int32_t batch, int32_t max_q, int32_t max_kv, int32_t window, g4::PagedAttn *a) {
  memset(a, 0, sizeof(*a));
  if (int rc = check_pool(who, pool, &a->pool)) return rc;
  if (type != G4_F32 && type != G4_BF16) return set_error(G4_ERR_INVALID, "%s: type %d", who, type);
  if (heads < 1 || heads % a->pool.kv_heads || heads / a->pool.kv_heads > 128)
    return set_error(G4_ERR_INVALID, "%s: %d query heads over %d KV heads (a multiple, at most 128 times)", who, heads, a->pool.kv_heads);
  if (rows < 0 || batch < 0 || max_q < 0 || max_kv < 0 || window < 0)
    return set_error(G4_ERR_INVALID, "%s: rows %d, batch %d, max_q %d, max_kv %d, window %d", who, rows, batch, max_q, max_kv, window);
  if ((long long)rows * heads >= (1ll << 30) || batch > 65535 || max_kv > (1 << 30))
    return set_error(G4_ERR_UNSUPPORTED, "%s: rows %d x %d heads (fewer than 2^30), batch %d (at most 65535), max_kv %d (2^30)", who, rows, heads, batch, max_kv);
  // A sequence's tiles (16 positions x up to 32 rows) are counted in 32 bits.
  const long long q_rows = (long long)(max_q < rows ? max_q : rows) * (heads / a->pool.kv_heads);
  if ((type == G4_F32 || max_kv > (1 << 24) || q_rows <= 32) && ((long long)max_kv / 16 + 32) * (q_rows / 32 + 1) >= (1ll << 31))
    return set_error(G4_ERR_UNSUPPORTED, "%s: %lld rows over %d positions in one sequence", who, q_rows, max_kv);
  a->type = type;
  a->heads = heads;
  a->group = heads / a->pool.kv_heads;
  a->rows = rows;
  a->batch = batch;
  a->max_q = max_q < rows ? max_q : rows;
  a->max_kv = max_kv;
  a->window = window;
  return G4_OK;
}

}  // namespace

extern "C" int g4_op_page_store(const g4_page_pool *pool, const void *k, const void *v, int32_t type,
                                int64_t k_stride, int64_t v_stride, int32_t tokens, const int32_t *slots, void *stream) {
  return move_rows("g4_op_page_store", true, pool, const_cast<void *>(k), const_cast<void *>(v), type, k_stride, v_stride, tokens, slots, stream);
}

extern "C" int g4_op_page_read(const g4_page_pool *pool, const int32_t *slots, int32_t tokens, int32_t type,
                               void *k_out, void *v_out, int64_t k_stride, int64_t v_stride, void *stream) {
  return move_rows("g4_op_page_read", false, pool, k_out, v_out, type, k_stride, v_stride, tokens, slots, stream);
}

extern "C" int g4_op_paged_attention_workspace(const g4_page_pool *pool, int32_t type, int32_t heads, int32_t rows,
                                               int32_t batch, int32_t max_q, int32_t max_kv, int32_t window, uint64_t *bytes) {
  const char *who = "g4_op_paged_attention_workspace";
  g4::PagedAttn a;
  if (!bytes) return set_error(G4_ERR_INVALID, "%s: null pointer", who);
  if (int rc = check_attention(who, pool, type, heads, rows, batch, max_q, max_kv, window, &a)) return rc;
  *bytes = g4::kPagedHeader + g4::paged_attention_partials(a);
  return G4_OK;
}

extern "C" int g4_op_paged_attention(const g4_page_pool *pool, const void *q, int64_t q_stride, void *out,
                                     int64_t out_stride, float *lse, int32_t type, int32_t heads, int32_t rows,
                                     int32_t batch, const int32_t *q_begin, const int32_t *q_pos,
                                     const int32_t *kv_len, const int32_t *page_table, int32_t table_stride,
                                     int32_t max_q, int32_t max_kv, int32_t window, float scale,
                                     void *workspace, uint64_t workspace_bytes, void *stream) {
  const char *who = "g4_op_paged_attention";
  g4::PagedAttn a;
  if (int rc = check_attention(who, pool, type, heads, rows, batch, max_q, max_kv, window, &a)) return rc;
  if (rows == 0 || batch == 0 || max_q == 0) return G4_OK;
  if (!q || !out || !q_begin || !q_pos || !kv_len || !page_table || !workspace) return set_error(G4_ERR_INVALID, "%s: null pointer", who);
  const long long width = (long long)heads * a.pool.hd;
  if (int rc = check_rows(who, "q", q, type, q_stride, width)) return rc;
  if (int rc = check_rows(who, "out", out, type, out_stride, width)) return rc;
  if ((long long)table_stride * a.pool.page_size < max_kv)
    return set_error(G4_ERR_INVALID, "%s: page tables of %d pages of %d hold fewer than max_kv %d positions", who, table_stride, a.pool.page_size, max_kv);
  if (!isfinite(scale)) return set_error(G4_ERR_INVALID, "%s: scale is not finite", who);
  const size_t need = g4::kPagedHeader + g4::paged_attention_partials(a);
  if (workspace_bytes < need || ((uintptr_t)workspace & 255))
    return set_error(G4_ERR_INVALID, "%s: needs a workspace of %llu bytes, 256-byte aligned; got %llu", who, (unsigned long long)need, (unsigned long long)workspace_bytes);
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.q_stride = q_stride;
  a.o_stride = out_stride;
  a.q_begin = q_begin;
  a.q_pos = q_pos;
  a.kv_len = kv_len;
  a.table = page_table;
  a.table_stride = table_stride;
  a.scale = scale;
  a.count = (uint32_t *)workspace;
  a.part = (float *)((char *)workspace + g4::kPagedHeader);
  a.err = g4::paged_error_flags();
  if (!a.err) return set_error(G4_ERR_CUDA, "%s: cannot resolve the device's error flags", who);
  return check_launch(who, g4::launch_paged_attention(a, (cudaStream_t)stream));
}

static int check_drafts(const char *who, int32_t vocab, int32_t rows, int32_t batch, int32_t max_drafts) {
  if (vocab < 1 || rows < 0 || batch < 0 || max_drafts < 0)
    return set_error(G4_ERR_INVALID, "%s: vocab %d, rows %d, batch %d, max_drafts %d", who, vocab, rows, batch, max_drafts);
  if (max_drafts > g4::kMaxDrafts || batch > 65535)
    return set_error(G4_ERR_UNSUPPORTED, "%s: max_drafts %d (at most %d), batch %d (65535)", who, max_drafts, g4::kMaxDrafts, batch);
  return G4_OK;
}

extern "C" int g4_op_verify_drafts_workspace(int32_t vocab, int32_t rows, int32_t batch, int32_t max_drafts, uint64_t *bytes) {
  const char *who = "g4_op_verify_drafts_workspace";
  if (!bytes) return set_error(G4_ERR_INVALID, "%s: null pointer", who);
  if (int rc = check_drafts(who, vocab, rows, batch, max_drafts)) return rc;
  *bytes = g4::kPagedHeader + g4::verify_drafts_partials(vocab, rows, batch, max_drafts);
  return G4_OK;
}

extern "C" int g4_op_verify_drafts(const void *logits, int64_t ld, int32_t type, int32_t vocab, int32_t rows,
                                   int32_t batch, const int32_t *row_begin, const int32_t *drafts,
                                   const float *draft_probs, int64_t ld_probs, const float *uniforms,
                                   const float *gumbel, int64_t ld_gumbel, const float *temperature,
                                   int32_t max_drafts, int32_t *tokens, float *logprobs, int32_t *counts,
                                   void *workspace, uint64_t workspace_bytes, void *stream) {
  const char *who = "g4_op_verify_drafts";
  if (int rc = check_drafts(who, vocab, rows, batch, max_drafts)) return rc;
  if (type != G4_F32 && type != G4_BF16) return set_error(G4_ERR_INVALID, "%s: type %d", who, type);
  if (batch == 0) return G4_OK;
  if (!row_begin || !gumbel || !temperature || !tokens || !logprobs || !counts || !workspace || (rows && (!logits || !drafts || !uniforms)))
    return set_error(G4_ERR_INVALID, "%s: null pointer", who);
  if (ld < vocab || ld_gumbel < vocab || (draft_probs && ld_probs < vocab))
    return set_error(G4_ERR_INVALID, "%s: rows of %d lie %lld / %lld / %lld apart", who, vocab, (long long)ld, (long long)ld_gumbel, (long long)ld_probs);
  if (((uintptr_t)logits & (type == G4_F32 ? 3 : 1)) || (((uintptr_t)gumbel | (uintptr_t)draft_probs) & 3))
    return set_error(G4_ERR_INVALID, "%s: a pointer is not aligned to its type", who);
  const size_t need = g4::kPagedHeader + g4::verify_drafts_partials(vocab, rows, batch, max_drafts);
  if (workspace_bytes < need || ((uintptr_t)workspace & 255))
    return set_error(G4_ERR_INVALID, "%s: needs a workspace of %llu bytes, 256-byte aligned; got %llu", who, (unsigned long long)need, (unsigned long long)workspace_bytes);
  g4::DraftArgs a;
  memset(&a, 0, sizeof(a));
  a.logits = logits;
  a.ld = ld;
  a.type = type;
  a.vocab = vocab;
  a.rows = rows;
  a.batch = batch;
  a.row_begin = row_begin;
  a.drafts = drafts;
  a.probs = draft_probs;
  a.ld_probs = ld_probs;
  a.uniforms = uniforms;
  a.gumbel = gumbel;
  a.ld_gumbel = ld_gumbel;
  a.temperature = temperature;
  a.max_drafts = max_drafts;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.counts = counts;
  a.count = (uint32_t *)workspace;
  a.part = (g4::DraftPart *)((char *)workspace + g4::kPagedHeader);
  a.err = g4::paged_error_flags();
  if (!a.err) return set_error(G4_ERR_CUDA, "%s: cannot resolve the device's error flags", who);
  return check_launch(who, g4::launch_verify_drafts(a, (cudaStream_t)stream));
}

extern "C" int g4_op_paged_errors(int32_t *flags) {
  if (!flags) return set_error(G4_ERR_INVALID, "g4_op_paged_errors: null pointer");
  int v = 0, zero = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g4::g4_paged_error, sizeof(v));
  if (e == cudaSuccess && v) e = cudaMemcpyToSymbol(g4::g4_paged_error, &zero, sizeof(zero));
  if (e != cudaSuccess) return set_error(G4_ERR_CUDA, "g4_op_paged_errors: %s", cudaGetErrorString(e));
  *flags = v;
  return G4_OK;
}
