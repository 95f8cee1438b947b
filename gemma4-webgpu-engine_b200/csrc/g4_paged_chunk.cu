// g4_paged_chunk.cu -- attention of chunks of new tokens over paged, quantised keys and values, on
// tcgen05.
//
// The mathematics is g4_paged_attn.cu's (codes exact in the products, scales applied in f32 to the
// scores and the weights, running maximum of score + ln vscale). A chunk's work is two products,
// 4 rows positions head_dim operations, so the tensor cores bound it and everything else is laid
// out to run beside them:
//  - A block owns 128 rows (queries x the heads that share a KV head), M of the products, and walks
//    the context in blocks of 128 positions. S = Q K^T and O += P V accumulate in tensor memory:
//    two S buffers of 128 columns and O of 256 fill its 512 columns. P goes back into the columns
//    of its S as f16 (bf16 pages: bf16) and is the second product's A operand from there.
//  - K and V pass through one ring of 16 KB slots, each [128 positions][64 dimensions] 16-bit in
//    the 128-byte swizzle: K-major B operand of the first product, and the same bytes are the
//    MN-major B operand of the second, so both are written alike. Eight producer warps gather the
//    pages' rows: 8-bit codes through registers (six slots in flight), widened to f16; bf16 rows by
//    asynchronous copies.
//  - One thread issues the products in the order S(j), O(j - 1), so the softmax of block j runs
//    under the products of its neighbours.
//  - Softmax: one thread a row. The maximum is stale by up to a factor of 2^1.9 (weights stay
//    below f16's greatest number); only when a row outgrows it are its warp's O rows rescaled.
// head_dim 512: O would fill tensor memory alone, so two blocks compute the scores each and take
// half of V's dimensions (1.5 times the operations).
#include <cuda_runtime.h>
#include <math.h>

#include "g4_device.cuh"
#include "g4_kernels.cuh"
#include "g4_paged.cuh"

namespace g4 {

namespace {

constexpr int kProducers = 256, kSoftmax = 128;
constexpr int kThreads = kSoftmax + kProducers + 32;
constexpr int BN = 128;            // positions per block
constexpr int SLOT = BN * 128;     // bytes of a slot
constexpr int NSC = 4;             // buffers of a block's scales
constexpr float kL2e = 1.44269504088896341f, kLn2f = 0.693147180559945309f;

template <int FMT, int HD>
struct ChunkShape {
  static constexpr bool HALF = FMT != G4_PAGE_BF16;
  static constexpr int KC = HD / 64;                    // K slots of a block
  static constexpr int OD = HD < 256 ? HD : 256;        // dimensions of O a block accumulates
  static constexpr int VC = OD / 64;                    // V slots of a block
  static constexpr int NS = HD == 512 ? 5 : 9;          // ring slots
  static constexpr int AHEAD = HD == 512 ? 4 : 6;       // slots in flight ahead of the ring's writes
  static constexpr int Q_BYTES = KC * SLOT;
  static constexpr int SC_OFF = Q_BYTES + NS * SLOT;    // [NSC][3][BN] floats: ks, vs, log2 vs
  static constexpr int BAR_OFF = SC_OFF + NSC * 3 * BN * 4;
  // full[NS], empty[NS], s_full[2], p_ready[2], pv_done, sc_full[NSC], sc_free[NSC], end
  static constexpr int BARS = 2 * NS + 2 + 2 + 1 + 2 * NSC + 1;
  static constexpr int SMEM = BAR_OFF + BARS * 8 + 64 + 1024;
};

__device__ __forceinline__ float cex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float crescale(float l, float d) {
  const float h = cex2(0.5f * d);
  return (l * h) * h;
}
__device__ __forceinline__ void arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A whole warp's bounded wait: all lanes agree on its result.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle, 8-row groups 1024 bytes apart. It serves both
// uses of a slot: K-major (rows are N, 64 K elements a row) and MN-major (rows are K, 64 N
// elements a row).
__device__ __forceinline__ uint64_t slot_desc(const void *p) {
  const uint32_t a = smem_u32(p);
  return (uint64_t)((a >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor, kind::f16: D f32, A and B f16 or bf16, M 128, N n, B MN-major or not.
constexpr uint32_t idesc_f16(bool half, int n, bool b_mn) {
  return (1u << 4) | (half ? 0u : (1u << 7) | (1u << 10)) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tld32(uint32_t at, float (&r)[32]) {
  uint32_t *u = reinterpret_cast<uint32_t *>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(at));
}
__device__ __forceinline__ void tld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tst_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tst16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tst32(uint32_t at, const float (&f)[32]) {
  const uint32_t *r = reinterpret_cast<const uint32_t *>(f);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(at)
      : "memory");
}

// Two f32 operations in one instruction.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 un2(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

template <bool HALF>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if (HALF) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Four codes as two f16 pairs, exactly (g4_paged_attn.cu).
template <int FMT>
__device__ __forceinline__ uint2 widen4(uint32_t w) {
  if (FMT == G4_PAGE_INT8) {
    const uint32_t x = w ^ 0x80808080u, magic = 0x64646464u;
    const uint32_t a = __byte_perm(x, magic, 0x4140), b = __byte_perm(x, magic, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const __half2 c = __hsub2(*reinterpret_cast<const __half2 *>(&a), off);
    const __half2 d = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&c), *reinterpret_cast<const uint32_t *>(&d));
  }
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffff), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
  return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// The ring's order of slots: K(0), then K(j), V(j - 1) for each further block, then V(last).
struct Walk {
  int j, c;       // block, slot of it
  bool v;
  int nb, kc, vc;
  __device__ __forceinline__ Walk(int nb_, int kc_, int vc_) : j(0), c(0), v(false), nb(nb_), kc(kc_), vc(vc_) {}
  __device__ __forceinline__ void next() {
    c++;
    if (!v && c == kc) {
      c = 0;
      if (j == 0) {
        if (nb == 1)
          v = true;
        else
          j = 1;
      } else {
        v = true;
        j--;
      }
    } else if (v && c == vc) {
      c = 0;
      if (j == nb - 1) {
        j = nb;   // done
      } else if (j == nb - 2) {
        j = nb - 1;   // V of the last block follows V of the one before it
      } else {
        j += 2;
        v = false;
      }
    }
  }
};

struct RowTile {
  int row0, rows;      // first token of the tile, rows (tokens x group) that exist
  int tlo, thi;        // positions some row sees
  int all_lo, all_hi;  // positions every row sees
};

// Block (row tile x half of V, KV head, sequence).
template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_paged_chunk(const PagedAttn a) {
  using S = ChunkShape<FMT, HD>;
  constexpr bool HALF = S::HALF;
  constexpr int NH = HD / S::OD;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int tpt = 128 / a.group;   // tokens per tile
  const int b = blockIdx.z, kvh = blockIdx.y, half = blockIdx.x % NH;
  const SeqSpan s = seq_span(a, b);
  const int tiles = (s.n + tpt - 1) / tpt;
  // The last rows see the most positions: they start first.
  const int tile = tiles - 1 - (int)(blockIdx.x / NH);
  if (tile < 0) return;
  RowTile rt;
  rt.row0 = tile * tpt;
  const int tokens = min(tpt, s.n - rt.row0);
  rt.rows = tokens * a.group;
  row_range(a, s.pos + rt.row0, s.kv, rt.tlo, rt.all_hi);
  row_range(a, s.pos + rt.row0 + tokens - 1, s.kv, rt.all_lo, rt.thi);
  const int j0 = rt.tlo / BN, nb = rt.thi > rt.tlo ? (rt.thi + BN - 1) / BN - j0 : 0;

  extern __shared__ __align__(1024) uint8_t csm_raw[];
  uint8_t *csm = csm_raw + ((1024 - (smem_u32(csm_raw) & 1023)) & 1023);
  float *sc = reinterpret_cast<float *>(csm + S::SC_OFF);
  uint64_t *full = reinterpret_cast<uint64_t *>(csm + S::BAR_OFF);
  uint64_t *empty = full + S::NS, *s_full = empty + S::NS, *p_ready = s_full + 2, *pv_done = p_ready + 2;
  uint64_t *sc_full = pv_done + 1, *sc_free = sc_full + NSC, *end = sc_free + NSC;
  uint32_t *tslot = reinterpret_cast<uint32_t *>(end + 1);
  int *failed = reinterpret_cast<int *>(tslot + 1);
  __shared__ uint32_t bad_v[4][4];   // bf16 pages: positions of boundary blocks whose V is not finite
  __shared__ float q_scale[128];
  auto slot = [&](int i) { return csm + S::Q_BYTES + i * SLOT; };
  const Pool &p = a.pool;

  if (t == 0) {
    for (int i = 0; i < S::NS; i++) {
      mbar_init(&full[i], kProducers / 32);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], kSoftmax / 32);
    }
    mbar_init(pv_done, 1);
    for (int i = 0; i < NSC; i++) {
      mbar_init(&sc_full[i], 4);
      mbar_init(&sc_free[i], kSoftmax / 32);
    }
    mbar_init(end, 1);
    mbar_fence_init();
    *failed = 0;
  }
  if (t < 16) (&bad_v[0][0])[t] = 0;
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // ---- Q into K-major slots, one warp a row, four rows of loads in flight. 8-bit pages: f16 scaled
  // by a power of two per row, so that the row's greatest value lies in 2^8 .. 2^9.
  if (warp < 12) {
    constexpr int LD = HD == 512 ? 2 : 1, ACT = HD / 8 < 32 ? HD / 8 : 32;
    for (int r0 = warp; r0 < 128; r0 += 48) {
      uint4 in[4][LD];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int r = r0 + 12 * k;
#pragma unroll
        for (int i = 0; i < LD; i++) {
          in[k][i] = make_uint4(0, 0, 0, 0);
          if (r < rt.rows && lane < ACT)
            in[k][i] = *reinterpret_cast<const uint4 *>(
                reinterpret_cast<const __nv_bfloat16 *>(a.q) + (long long)(s.row + rt.row0 + r / a.group) * a.q_stride +
                (long long)(kvh * a.group + r % a.group) * HD + 8 * lane + 256 * i);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int r = r0 + 12 * k;
        if (r >= 128) break;
        int e = 0;
        if (HALF) {
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < LD; i++) {
            const uint32_t w[4] = {in[k][i].x, in[k][i].y, in[k][i].z, in[k][i].w};
#pragma unroll
            for (int z = 0; z < 4; z++) top = max(top, max(w[z] & 0x7f80u, (w[z] >> 16) & 0x7f80u));
          }
          top = __reduce_max_sync(0xffffffffu, top);
          // Exponent of the greatest; infinities and NaN stay what they are at any power of two.
          e = (int)(top >> 7) - 127;
          e = e < -110 ? -110 : (e > 127 ? 0 : e);
        }
        const float f = __uint_as_float((uint32_t)(127 + 8 - e) << 23);
#pragma unroll
        for (int i = 0; i < LD; i++) {
          uint4 o = in[k][i];
          if (HALF) {
            uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int z = 0; z < 4; z++)
              w[z] = pack16<true>(__uint_as_float(w[z] << 16) * f, __uint_as_float(w[z] & 0xffff0000u) * f);
            o = make_uint4(w[0], w[1], w[2], w[3]);
          }
          const int d = 8 * lane + 256 * i;
          if (lane < ACT)
            *reinterpret_cast<uint4 *>(csm + (d >> 6) * SLOT + r * 128 + ((((d >> 3) & 7) ^ (r & 7)) << 4)) = o;
        }
        if (lane == 0) q_scale[r] = a.scale * kL2e * (HALF ? __uint_as_float((uint32_t)(127 - 8 + e) << 23) : 1.0f);
      }
    }
    fence_async();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tslot;
  const uint32_t t_s[2] = {tmem, tmem + 128}, t_o = tmem + 256;

  if (warp >= 4 && warp < 12) {
    // ============================================================ producers
    const int pt = t - kSoftmax;
    constexpr int RPT = HALF ? 2 : 4;                  // rows of a slot a thread moves 16 bytes of
    constexpr int STEP = HALF ? 64 : 32;
    const int r0 = HALF ? pt >> 2 : pt >> 3, x = HALF ? pt & 3 : pt & 7;
    const int32_t *table = a.table + (long long)b * a.table_stride;
    // Row of the pool that holds position pos (for this KV head), -1 for none.
    auto page_of = [&](int pos) -> int {
      if (pos < rt.tlo || pos >= rt.thi) return -2;
      const int pg = table[pos / p.page_size];
      return pg;
    };
    auto row_of = [&](int pos, int pg) -> long long {
      if (pg == -2) return -1;
      if (pg < 0 || pg >= p.n_pages) {
        paged_raise(a.err, G4_PAGED_BAD_PAGE);
        return -1;
      }
      return ((long long)pg * p.kv_heads + kvh) * p.page_size + pos % p.page_size;
    };
    long long cur[RPT], prev[RPT];
    int pg[RPT];
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      cur[i] = prev[i] = -1;
      pg[i] = nb > 0 ? page_of(j0 * BN + r0 + STEP * i) : -2;
    }
    // This thread's position for the scales (the first four warps), one block ahead.
    const bool scaler = pt < BN;
    float nks = 0.0f, nvs = -1.0f;
    int npg = -2;
    auto load_scale = [&](int j, int page) {
      const int pos = (j0 + j) * BN + pt;
      const long long row = row_of(pos, page);
      nks = 0.0f;
      nvs = -1.0f;   // not a scale: no row may see this position
      if (row >= 0) {
        nks = HALF ? __ldg(p.ks + row) : 1.0f;
        nvs = HALF ? __ldg(p.vs + row) : 1.0f;
      }
    };
    if (scaler && nb > 0) {
      load_scale(0, page_of(j0 * BN + pt));
      npg = nb > 1 ? page_of((j0 + 1) * BN + pt) : -2;
    }
    constexpr int A = S::AHEAD;
    uint4 st[HALF ? A : 1][RPT];
    Walk ld(nb, S::KC, S::VC), put(nb, S::KC, S::VC);
    bool ok = true;

    // Loads of the slot `ld` stands at, into register stage k (8 bit) or ring slot n (16 bit).
    auto load = [&](uint4 (&d)[RPT], int n) {
      if (!ld.v && ld.c == 0) {
#pragma unroll
        for (int i = 0; i < RPT; i++) {
          prev[i] = cur[i];
          cur[i] = row_of((j0 + ld.j) * BN + r0 + STEP * i, pg[i]);
          pg[i] = ld.j + 1 < nb ? page_of((j0 + ld.j + 1) * BN + r0 + STEP * i) : -2;
        }
      }
      const bool latest = ld.j == nb - 1;   // V of the last block: no K moved `cur` on
      const uint8_t *base = ld.v ? p.v : p.k;
      const int ch = ld.v ? half * S::VC + ld.c : ld.c;
#pragma unroll
      for (int i = 0; i < RPT; i++) {
        const long long row = ld.v && !latest ? prev[i] : cur[i];
        if (HALF) {
          d[i] = make_uint4(0, 0, 0, 0);
          if (row >= 0) d[i] = __ldg(reinterpret_cast<const uint4 *>(base + row * HD + ch * 64 + x * 16));
        } else {
          const int r = r0 + STEP * i;
          uint8_t *dst = slot(n) + r * 128 + ((x ^ (r & 7)) << 4);
          if (row >= 0)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)),
                         "l"(base + (row * HD + ch * 64) * 2 + x * 16)
                         : "memory");
          else
            *reinterpret_cast<uint4 *>(dst) = make_uint4(0, 0, 0, 0);
        }
      }
      ld.next();
    };
    // Hands slot n over (writing it first from the register stage at 8 bits).
    auto hand = [&](const uint4 (&d)[RPT], int n) {
      if constexpr (HALF) {
#pragma unroll
        for (int i = 0; i < RPT; i++) {
          const int r = r0 + STEP * i;
          const uint2 w0 = widen4<FMT>(d[i].x), w1 = widen4<FMT>(d[i].y), w2 = widen4<FMT>(d[i].z), w3 = widen4<FMT>(d[i].w);
          uint8_t *row = slot(n) + r * 128;
          *reinterpret_cast<uint4 *>(row + (((2 * x) ^ (r & 7)) << 4)) = make_uint4(w0.x, w0.y, w1.x, w1.y);
          *reinterpret_cast<uint4 *>(row + (((2 * x + 1) ^ (r & 7)) << 4)) = make_uint4(w2.x, w2.y, w3.x, w3.y);
        }
      } else if (put.v) {
        // Blocks that some row sees only in part: a weight of 0 must not meet an infinity or a NaN.
        const int pos0 = (j0 + put.j) * BN;
        if (pos0 < rt.all_lo || pos0 + BN > rt.all_hi) {
#pragma unroll
          for (int i = 0; i < RPT; i++) {
            const int r = r0 + STEP * i;
            uint4 *at = reinterpret_cast<uint4 *>(slot(n) + r * 128 + ((x ^ (r & 7)) << 4));
            uint32_t w[4] = {at->x, at->y, at->z, at->w};
            bool bad = false;
#pragma unroll
            for (int z = 0; z < 4; z++) {
              if ((w[z] & 0x7f80u) == 0x7f80u) {
                w[z] &= 0xffff0000u;
                bad = true;
              }
              if ((w[z] & 0x7f800000u) == 0x7f800000u) {
                w[z] &= 0xffffu;
                bad = true;
              }
            }
            if (bad) {
              *at = make_uint4(w[0], w[1], w[2], w[3]);
              atomicOr(&bad_v[put.j < 2 ? put.j : 2 + (nb - 1 - put.j)][r >> 5], 1u << (r & 31));
            }
          }
        }
      }
      fence_async();
      __syncwarp();
      if (lane == 0) arrive(&full[n]);
      if (!put.v && put.c == 0 && scaler) {
        // The block's scales, and the next block's on their way.
        const int k = put.j % NSC;
        if (put.j >= NSC && !warp_wait(&sc_free[k], (uint32_t)((put.j / NSC - 1) & 1))) ok = false;
        float *f = sc + k * 3 * BN;
        f[pt] = nks;
        f[BN + pt] = nvs;
        f[2 * BN + pt] = HALF ? __log2f(fmaxf(nvs, 0x1p-100f)) : 0.0f;
        __syncwarp();
        if (lane == 0) arrive(&sc_full[k]);
        if (put.j + 1 < nb) {
          load_scale(put.j + 1, npg);
          npg = put.j + 2 < nb ? page_of((j0 + put.j + 2) * BN + pt) : -2;
        }
      }
      put.next();
    };

    const int total = nb * (S::KC + S::VC);
    if constexpr (HALF) {
#pragma unroll
      for (int k = 0; k < A; k++)
        if (k < total) load(st[k], 0);
      for (int n = 0; n < total && ok; n += A) {
#pragma unroll
        for (int k = 0; k < A; k++) {
          const int i = n + k;
          if (i >= total) break;
          const int sl = i % S::NS;
          if (i >= S::NS && !warp_wait(&empty[sl], (uint32_t)((i / S::NS - 1) & 1))) {
            ok = false;
            break;
          }
          hand(st[k], sl);
          if (i + A < total) load(st[k], 0);
        }
      }
    } else {
      // Slot i + A - 1 is requested before slot i is handed over: A groups in flight at most.
      uint4 none[RPT];
      for (int i = 0; i < total + A - 1 && ok; i++) {
        if (i < total) {
          const int sl = i % S::NS;
          if (i >= S::NS && !warp_wait(&empty[sl], (uint32_t)((i / S::NS - 1) & 1))) {
            ok = false;
            break;
          }
          load(none, sl);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (i >= A - 1) {
          asm volatile("cp.async.wait_group %0;" ::"n"(A - 1) : "memory");
          hand(none, (i - (A - 1)) % S::NS);
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    if (!ok) {
      *failed = 1;
      paged_raise(a.err, G4_PAGED_TIMEOUT);
    }
  } else if (warp == 12) {
    // ============================================================ products
    if (lane == 0) {
      constexpr uint32_t IS = idesc_f16(HALF, BN, false), IO = idesc_f16(HALF, 64, true);
      int n = 0;
      bool ok = true;
      auto scores = [&](int j) {
        if (j >= 2 && !mbar_wait(pv_done, (uint32_t)(j & 1))) return false;   // O(j - 2) has read P from these columns
        for (int c = 0; c < S::KC; c++, n++) {
          const int sl = n % S::NS;
          if (!mbar_wait(&full[sl], (uint32_t)((n / S::NS) & 1))) return false;
          fence_after();
          const uint64_t ad = slot_desc(csm + c * SLOT), bd = slot_desc(slot(sl));
#pragma unroll
          for (int k = 0; k < 4; k++) mma_ss(t_s[j & 1], ad + 2 * k, bd + 2 * k, IS, (c | k) != 0);
          commit(&empty[sl]);
        }
        commit(&s_full[j & 1]);
        return true;
      };
      auto outputs = [&](int j) {
        if (!mbar_wait(&p_ready[j & 1], (uint32_t)((j >> 1) & 1))) return false;
        for (int c = 0; c < S::VC; c++, n++) {
          const int sl = n % S::NS;
          if (!mbar_wait(&full[sl], (uint32_t)((n / S::NS) & 1))) return false;
          fence_after();
          const uint64_t bd = slot_desc(slot(sl));
#pragma unroll
          for (int k = 0; k < BN / 16; k++) mma_ts(t_o + 64 * c, t_s[j & 1] + 8 * k, bd + 128 * k, IO, (j | k) != 0);
          commit(&empty[sl]);
        }
        commit(pv_done);
        return true;
      };
      for (int j = 0; j < nb && ok; j++) {
        ok = scores(j);
        if (ok && j >= 1) ok = outputs(j - 1);
      }
      if (ok && nb > 0) ok = outputs(nb - 1);
      if (!ok) {
        *failed = 1;
        paged_raise(a.err, G4_PAGED_TIMEOUT);
      }
      // Everything issued has ended before tensor memory and the slots are given up.
      commit(end);
      if (!mbar_wait(end, 0)) paged_raise(a.err, G4_PAGED_TIMEOUT);
    }
    __syncwarp();
  }
  float m = -INFINITY, l = 0.0f;
  int lo = 0, hi = 0;
  const float bits = HALF ? 14.0f : 0.0f;
  const uint32_t lane_base = (uint32_t)(32 * warp) << 16;
  if (warp < 4) {
    // ============================================================ softmax: thread t is row t
    const float qf = q_scale[t];
    if (t < rt.rows) row_range(a, s.pos + rt.row0 + t / a.group, s.kv, lo, hi);
    bool ok = true;
    for (int j = 0; j < nb && ok; j++) {
      const int k = j % NSC, pos0 = (j0 + j) * BN;
      ok = warp_wait(&sc_full[k], (uint32_t)((j / NSC) & 1)) && warp_wait(&s_full[j & 1], (uint32_t)((j >> 1) & 1));
      if (!ok) break;
      fence_after();
      const float4 *ks = reinterpret_cast<const float4 *>(sc + k * 3 * BN), *vs = ks + BN / 4, *lv = vs + BN / 4;
      const uint32_t at = t_s[j & 1] + lane_base;
      // Scales within a factor of 2^8 of each other (and every page there): one bound serves them.
      const float4 mine = lv[lane];
      const float4 mv = vs[lane];
      float lmax = fmaxf(fmaxf(mine.x, mine.y), fmaxf(mine.z, mine.w)), lmin = fminf(fminf(mine.x, mine.y), fminf(mine.z, mine.w));
      float vmin = fminf(fminf(mv.x, mv.y), fminf(mv.z, mv.w));
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        if (HALF) {
          lmax = fmaxf(lmax, __shfl_xor_sync(0xffffffffu, lmax, d));
          lmin = fminf(lmin, __shfl_xor_sync(0xffffffffu, lmin, d));
        }
        vmin = fminf(vmin, __shfl_xor_sync(0xffffffffu, vmin, d));
      }
      const bool plain = pos0 >= rt.all_lo && pos0 + BN <= rt.all_hi && !(vmin < 0.0f) && lmax - lmin <= 8.0f;
      float top = -INFINITY;
      float sv[32];
      if (plain) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
          tld32(at + 32 * c, sv);
          tld_wait();
#pragma unroll
          for (int i = 0; i < 8; i++) {
            if (HALF) {
              const float4 f = ks[8 * c + i];
              const float2 u = un2(mul2(f2(sv[4 * i], sv[4 * i + 1]), f2(f.x, f.y)));
              const float2 w = un2(mul2(f2(sv[4 * i + 2], sv[4 * i + 3]), f2(f.z, f.w)));
              // A negative scale turns the order round.
              top = qf >= 0.0f ? max3(top, u.x, u.y) : max3(top, -u.x, -u.y);
              top = qf >= 0.0f ? max3(top, w.x, w.y) : max3(top, -w.x, -w.y);
            } else {
              const float sg = qf >= 0.0f ? 1.0f : -1.0f;
              top = max3(top, sg * sv[4 * i], sg * sv[4 * i + 1]);
              top = max3(top, sg * sv[4 * i + 2], sg * sv[4 * i + 3]);
            }
          }
        }
        top = top * fabsf(qf) + (HALF ? lmax : 0.0f);
      } else {
#pragma unroll 1
        for (int c = 0; c < 4; c++) {
          tld32(at + 32 * c, sv);
          tld_wait();
#pragma unroll
          for (int i = 0; i < 32; i++) {
            const int q = 32 * c + i, pos = pos0 + q;
            const float v = reinterpret_cast<const float *>(vs)[q];
            const float z = sv[i] * reinterpret_cast<const float *>(ks)[q] * qf + reinterpret_cast<const float *>(lv)[q];
            if (pos >= lo && pos < hi && !(v < 0.0f)) top = fmaxf(top, z);
          }
        }
      }
      // The maximum moves only when a row outgrows it by more than 2^1.9.
      const bool grow = top > m + 1.9f || (m == -INFINITY && top > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? cex2(m - top) : 1.0f;
        if (grow) {
          l = m == -INFINITY ? 0.0f : crescale(l, m - top);
          m = top;
        }
        if (j > 0) {
          ok = warp_wait(pv_done, (uint32_t)((j - 1) & 1));
          if (!ok) break;
          fence_after();
#pragma unroll 1
          for (int c = 0; c < S::OD / 32; c++) {
            float o[32];
            tld32(t_o + lane_base + 32 * c, o);
            tld_wait();
#pragma unroll
            for (int i = 0; i < 32; i++) o[i] *= f;
            tst32(t_o + lane_base + 32 * c, o);
          }
          tst_wait();
        }
      }
      const float r = m == -INFINITY ? 0.0f : m - bits;
      F2 sum = f2(0.0f, 0.0f);
      if (plain) {
        const F2 q2 = f2(qf, qf), r2 = f2(-r, -r);
#pragma unroll
        for (int c = 0; c < 4; c++) {
          tld32(at + 32 * c, sv);
          tld_wait();
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            F2 z0 = f2(sv[4 * i], sv[4 * i + 1]), z1 = f2(sv[4 * i + 2], sv[4 * i + 3]);
            if (HALF) {
              const float4 f = ks[8 * c + i];
              z0 = mul2(z0, f2(f.x, f.y));
              z1 = mul2(z1, f2(f.z, f.w));
            }
            const float2 y0 = un2(fma2(z0, q2, r2)), y1 = un2(fma2(z1, q2, r2));
            F2 p0 = f2(cex2(y0.x), cex2(y0.y)), p1 = f2(cex2(y1.x), cex2(y1.y));
            sum = add2(sum, p0);
            sum = add2(sum, p1);
            if (HALF) {
              const float4 f = vs[8 * c + i];
              p0 = mul2(p0, f2(f.x, f.y));
              p1 = mul2(p1, f2(f.z, f.w));
            }
            const float2 w0 = un2(p0), w1 = un2(p1);
            pk[2 * i] = pack16<HALF>(w0.x, w0.y);
            pk[2 * i + 1] = pack16<HALF>(w1.x, w1.y);
          }
          tst16(at + 16 * c, pk);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < 4; c++) {
          tld32(at + 32 * c, sv);
          tld_wait();
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i++) {
            const int q = 32 * c + i, pos = pos0 + q;
            const float v = reinterpret_cast<const float *>(vs)[q];
            const bool see = pos >= lo && pos < hi && !(v < 0.0f);
            const float z = sv[i] * reinterpret_cast<const float *>(ks)[q] * qf;
            const float e = see ? cex2(z - r) : 0.0f;
            sum = add2(sum, f2(e, 0.0f));
            sv[i] = see ? e * v : 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 16; i++) pk[i] = pack16<HALF>(sv[2 * i], sv[2 * i + 1]);
          tst16(at + 16 * c, pk);
        }
      }
      const float2 two = un2(sum);
      l += two.x + two.y;
      tst_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) {
        arrive(&p_ready[j & 1]);
        arrive(&sc_free[k]);
      }
    }
    if (!ok) {
      *failed = 1;
      paged_raise(a.err, G4_PAGED_TIMEOUT);
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp < 4 && !*failed) {
    // ============================================================ the rows out
    const int i = rt.row0 + t / a.group, h = kvh * a.group + t % a.group;
    if (!HALF && nb > 0 && t < rt.rows) {
      // A row that sees a value which is not finite is not either.
#pragma unroll 1
      for (int k = 0; k < 16; k++) {
        uint32_t w = bad_v[k >> 2][k & 3];
        const int j = (k >> 2) < 2 ? (k >> 2) : nb - 1 - ((k >> 2) - 2);
        while (w) {
          const int pos = (j0 + j) * BN + 32 * (k & 3) + __ffs((int)w) - 1;
          if (pos >= lo && pos < hi) l = __int_as_float(0x7fffffff);
          w &= w - 1;
        }
      }
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const bool live = t < rt.rows;
    __nv_bfloat16 *out = reinterpret_cast<__nv_bfloat16 *>(a.out) + (long long)(s.row + i) * a.o_stride + (long long)h * HD + half * S::OD;
#pragma unroll 1
    for (int c = 0; c < S::OD / 32; c++) {
      float o[32];
      if (nb > 0) {
        tld32(t_o + lane_base + 32 * c, o);
        tld_wait();
      } else {
#pragma unroll
        for (int k = 0; k < 32; k++) o[k] = 0.0f;
      }
      if (live) {
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          uint32_t w[4];
#pragma unroll
          for (int z = 0; z < 4; z++) {
            // (An O row whose weights were all 0 is 0.)
            w[z] = pack16<false>(o[k + 2 * z] * inv, o[k + 2 * z + 1] * inv);
          }
          *reinterpret_cast<uint4 *>(out + 32 * c + k) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    if (live && a.lse && half == 0)
      a.lse[(long long)(s.row + i) * a.heads + h] = m == -INFINITY ? -INFINITY : (m - bits + log2f(l)) * kLn2f;
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

}  // namespace

template <int FMT, int HD>
static cudaError_t launch_chunk_hd(const PagedAttn &a, cudaStream_t st) {
  using S = ChunkShape<FMT, HD>;
  static DeviceOnce once;
  cudaError_t e = cudaSuccess;
  once([&] { e = cudaFuncSetAttribute(k_paged_chunk<FMT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); });
  if (e != cudaSuccess) return e;
  const int tpt = 128 / a.group, tiles = (a.max_q + tpt - 1) / tpt;
  const dim3 grid((unsigned)(tiles * (HD / S::OD)), a.pool.kv_heads, a.batch);
  return launch_k(k_paged_chunk<FMT, HD>, grid, dim3(kThreads), S::SMEM, st, false, a);
}
template <int FMT>
static cudaError_t launch_chunk(const PagedAttn &a, cudaStream_t st) {
  switch (a.pool.hd) {
    case 64: return launch_chunk_hd<FMT, 64>(a, st);
    case 128: return launch_chunk_hd<FMT, 128>(a, st);
    case 256: return launch_chunk_hd<FMT, 256>(a, st);
    default: return launch_chunk_hd<FMT, 512>(a, st);
  }
}
cudaError_t launch_paged_chunk(const PagedAttn &a, cudaStream_t st) {
  switch (a.pool.fmt) {
    case G4_PAGE_BF16: return launch_chunk<G4_PAGE_BF16>(a, st);
    case G4_PAGE_INT8: return launch_chunk<G4_PAGE_INT8>(a, st);
    default: return launch_chunk<G4_PAGE_E4M3>(a, st);
  }
}

}  // namespace g4
