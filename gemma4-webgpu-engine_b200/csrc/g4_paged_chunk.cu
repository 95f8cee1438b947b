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
//  - K and V pass through one ring of 16 KB slots of 64-dimension columns in the 128-byte swizzle.
//    A K slot is one column of 128 positions, K-major B operand; a V slot is all columns of 128 / 64
//    / 32 positions (head_dim 64 / 128 / 256), MN-major B operand with all of O's dimensions as N: a
//    product of N 64 costs 112 cycles, not the 32 of its share (head_dim 256 by columns took 3,600
//    cycles a block for O, 8 products of N 256 are 1,024). Both are written alike. Six producer warps gather the
//    pages' rows, each a slot of its own: 8-bit codes through registers, the next slot's requested
//    as this one's are widened to f16, bf16 rows by TMA. A scout warp reads the
//    page table and the scales blocks ahead.
//  - One thread issues the products in the order S(j), O(j - 1), so the softmax of block j runs
//    under the products of its neighbours.
//  - Softmax: two threads a row, 64 positions of a block each, held in registers from the scores to
//    the weights. The maximum is stale by up to a factor of 2^2.9; only when a row outgrows it are its
//    warp's O rows rescaled (1,000 to 4,000 cycles). Weights are scaled by 2^13, so they stay below
//    f16's greatest number and are held to 2^-38 of the row's greatest; a staler maximum would cost
//    that.
// head_dim 512: O would fill tensor memory alone, so two blocks compute the scores each and take
// half of V's dimensions (1.5 times the operations).
#include <cuda_runtime.h>
#include <math.h>

#include "g4_device.cuh"
#include "g4_kernels.cuh"
#include "g4_paged.cuh"

namespace g4 {

namespace {

// Warps by role: softmax, producers, the scout, the products.
constexpr int kSoftWarps = 8, kProdWarps = 6;
constexpr int kScout = kSoftWarps + kProdWarps, kMma = kScout + 1;
constexpr int kThreads = 32 * (kMma + 1);
constexpr int BN = 128;            // positions per block
constexpr int SLOT = BN * 128;     // bytes of a slot
constexpr int NSC = 8;             // buffers of what the scout found out about a block
constexpr float kL2e = 1.44269504088896341f, kLn2f = 0.693147180559945309f;

// A block of positions as the scout leaves it: their scales (vs < 0: no page there), log2 of the V
// scales, the byte offset of each 16 positions' rows in the pool (the pool's first where there is no
// page: read, never used), the greatest log2, and whether one bound serves all (every page there, scales within 2^8 of each other).
struct __align__(16) BlockInfo {
  float ks[BN], vs[BN], lv[BN];
  long long at[BN / 16];
  float lmax;
  int even;
  int pad[2];
};

template <int FMT, int HD>
struct ChunkShape {
  static constexpr bool HALF = FMT != G4_PAGE_BF16;
  static constexpr int KC = HD / 64;                    // K slots of a block
  static constexpr int OD = HD < 256 ? HD : 256;        // dimensions of O a block accumulates
  static constexpr int VC = OD / 64;                    // V slots of a block
  static constexpr int TV = BN / VC;                    // positions of a V slot
  static constexpr int NS = HD == 512 ? 4 : 8;          // ring slots
  static constexpr int G = VC;                          // consecutive slots the issue loop is unrolled over
  static_assert(NS % G == 0 && KC % G == 0, "groups of slots stay whole around the ring");
  // Producer warps: warp w fills slots w, w + PW, ... A slot's rounds are told apart by one parity bit, so
  // whoever waits for a round must know that the one before it has begun: slots are consumed in
  // order, and with PW <= NS the warp's own last slot was filled after that one's consumption.
  static constexpr int PW = HD == 512 ? 4 : kProdWarps;
  static_assert(PW <= NS, "see PW");
  static constexpr int Q_BYTES = KC * SLOT;
  static constexpr int SC_OFF = Q_BYTES + NS * SLOT;
  static constexpr int BAR_OFF = SC_OFF + NSC * (int)sizeof(BlockInfo);
  // full[NS], empty[NS], s_full[2], p_ready[2], pv_done, info_full[NSC], info_free[NSC], end
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
__device__ __forceinline__ bool elect() {
  uint32_t on;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(on));
  return on != 0;
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
// A copy of 16 rows of the pool, 128 bytes of each from byte x, into the 128-byte swizzle (bf16 pages).
__device__ __forceinline__ void tma_rows(void *dst, const CUtensorMap *map, int x, int row, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(smem_u32(bar))
      : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle, 8-row groups 1024 bytes apart. It serves both
// uses of a slot: K-major (rows are N, 64 K elements a row) and MN-major (rows are K, 64 N
// elements a row, columns `column` bytes apart).
__device__ __forceinline__ uint64_t slot_desc(const void *p, uint32_t column = 16) {
  const uint32_t a = smem_u32(p);
  return (uint64_t)((a >> 4) & 0x3FFF) | ((uint64_t)(column >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
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
__device__ __forceinline__ void tld16(uint32_t at, float (&r)[16]) {
  uint32_t *u = reinterpret_cast<uint32_t *>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

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
template <int KC, int VC>
struct SlotAt {
  int j, c;
  bool v;
  __device__ __forceinline__ SlotAt(int i, int nb) {
    if (i < KC) {
      j = 0;
      c = i;
      v = false;
      return;
    }
    const int q = (i - KC) / (KC + VC), r = (i - KC) % (KC + VC);
    v = q + 1 == nb || r >= KC;
    j = v ? q : q + 1;
    c = v && q + 1 < nb ? r - KC : r;
  }
};

struct RowTile {
  int row0, rows;      // first token of the tile, rows (tokens x group) that exist
  int tlo, thi;        // positions some row sees
  int all_lo, all_hi;  // positions every row sees
};

// Block (row tile x half of V, KV head, sequence).
template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_paged_chunk(const PagedAttn a, const __grid_constant__ CUtensorMap map_k,
                                                          const __grid_constant__ CUtensorMap map_v) {
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
  BlockInfo *info = reinterpret_cast<BlockInfo *>(csm + S::SC_OFF);
  uint64_t *full = reinterpret_cast<uint64_t *>(csm + S::BAR_OFF);
  uint64_t *empty = full + S::NS, *s_full = empty + S::NS, *p_ready = s_full + 2, *pv_done = p_ready + 2;
  uint64_t *info_full = pv_done + 1, *info_free = info_full + NSC, *end = info_free + NSC;
  uint32_t *tslot = reinterpret_cast<uint32_t *>(end + 1);
  int *failed = reinterpret_cast<int *>(tslot + 1);
  __shared__ uint64_t own_bar[S::PW];
  __shared__ uint32_t bad_v[4][4];   // bf16 pages: positions of boundary blocks whose V is not finite
  __shared__ float q_scale[128], row_top[2][2][128];
  auto slot = [&](int i) { return csm + S::Q_BYTES + i * SLOT; };
  const Pool &p = a.pool;

  if (t == 0) {
    for (int i = 0; i < S::NS; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], kSoftWarps);
    }
    mbar_init(pv_done, 1);
    for (int i = 0; i < NSC; i++) {
      mbar_init(&info_full[i], 1);
      mbar_init(&info_free[i], kSoftWarps + S::VC);
    }
    mbar_init(end, 1);
    for (int i = 0; i < S::PW; i++) mbar_init(&own_bar[i], 1);
    mbar_fence_init();
    *failed = 0;
  }
  if (t < 16) (&bad_v[0][0])[t] = 0;
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // ---- Q into K-major slots, one warp a row, four rows of loads in flight. 8-bit pages: f16 scaled
  // by a power of two per row, so that the row's greatest value lies in 2^8 .. 2^9.
  {
    const uint32_t flip = __float_as_uint(a.scale) & 0x80000000u;   // a negative scale turns Q round: row factors are >= 0
    constexpr int LD = HD == 512 ? 2 : 1, ACT = HD / 8 < 32 ? HD / 8 : 32;
    for (int r0 = warp; r0 < 128; r0 += 64) {
      uint4 in[4][LD];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int r = r0 + 16 * k;
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
        const int r = r0 + 16 * k;
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
        const float f = __uint_as_float((uint32_t)(127 + 8 - e) << 23 | flip);
#pragma unroll
        for (int i = 0; i < LD; i++) {
          uint4 o = in[k][i];
          if (!HALF) {
            const uint32_t two = flip | flip >> 16;
            o = make_uint4(o.x ^ two, o.y ^ two, o.z ^ two, o.w ^ two);
          } else {
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
        if (lane == 0) q_scale[r] = fabsf(a.scale) * kL2e * (HALF ? __uint_as_float((uint32_t)(127 - 8 + e) << 23) : 1.0f);
      }
    }
    fence_async();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tslot;
  const uint32_t t_s[2] = {tmem, tmem + 128}, t_o = tmem + 256;

  if (warp >= kSoftWarps && warp < kSoftWarps + S::PW) {
    // ============================================================ producers
    constexpr int ROW = HALF ? HD : 2 * HD;   // bytes of a position
    const int total = nb * (S::KC + S::VC), w = warp - kSoftWarps;
    bool ok = true;
    // The block's rows are known, or a wait gave up.
    auto known = [&](const SlotAt<S::KC, S::VC> &at) {
      return warp_wait(&info_full[at.j % NSC], (uint32_t)((at.j / NSC) & 1));
    };
    // This warp's last use of a V slot's rows.
    auto used = [&](const SlotAt<S::KC, S::VC> &at) {
      __syncwarp();
      if (at.v && lane == 0) arrive(&info_free[at.j % NSC]);
    };
    auto slot_free = [&](int i) { return i < S::NS || warp_wait(&empty[i % S::NS], (uint32_t)((i / S::NS - 1) & 1)); };
    auto edge = [&](int j) {
      const int pos0 = (j0 + j) * BN;
      return pos0 < rt.all_lo || pos0 + BN > rt.all_hi;
    };
    // A block some of whose positions some row may not see, or that lacks a page; and whether a position
    // of it is there for any row.
    auto odd_block = [&](int j) { return edge(j) || !info[j % NSC].even; };
    auto seen = [&](int j, int q) {
      const int pos = (j0 + j) * BN + q;
      return pos >= rt.tlo && pos < rt.thi && !(info[j % NSC].vs[q] < 0.0f);
    };
    if constexpr (HALF) {
      // Piece k of a lane: 16 codes of row 8 k + lane / 4 of the slot's columns laid end to end.
      const int rr = lane >> 2, x = lane & 3;
      uint4 d[16];
      // Where pieces 2 k and 2 k + 1 start. (Read together, before the stores to shared memory that they
      // may not pass.)
      long long rows[8];
      auto find = [&](const SlotAt<S::KC, S::VC> &at) {
        const long long *src = info[at.j % NSC].at;
        constexpr int T = S::TV / 16;
#pragma unroll
        for (int k = 0; k < 8; k++) rows[k] = src[at.v ? at.c * T + k % T : k] + (at.v ? 64 * (k / T) : 0);
      };
      auto load = [&](const uint8_t *base, int k) {
        return __ldg(reinterpret_cast<const uint4 *>(base + rows[k >> 1] + (k & 1) * 8 * ROW));
      };
      // e4m3 codes of V at positions that no row sees may be NaN, which a weight of 0 would not hide:
      // the pieces of a slot to set to zero.
      auto unseen = [&](const SlotAt<S::KC, S::VC> &at) -> uint32_t {
        uint32_t m = 0;
        if (FMT == G4_PAGE_E4M3 && at.v && odd_block(at.j)) {
          for (int k = 0; k < 16; k++)
            if (!seen(at.j, at.c * S::TV + 8 * (k % (S::TV / 8)) + rr)) m |= 1u << k;
        }
        return m;
      };
      uint32_t zero = 0;
      auto base_of = [&](const SlotAt<S::KC, S::VC> &at) {
        return (at.v ? p.v + half * S::OD : p.k + at.c * 64) + rr * ROW + x * 16;
      };
      const uint32_t o0 = rr * 128 + (((2 * x) ^ rr) << 4), o1 = o0 ^ 16;
      if (w < total) {
        const SlotAt<S::KC, S::VC> at(w, nb);
        ok = known(at);
        if (ok) {
          const uint8_t *base = base_of(at);
          find(at);
          zero = unseen(at);
#pragma unroll
          for (int k = 0; k < 16; k++) d[k] = load(base, k);
          used(at);
        }
      }
#pragma unroll 1
      for (int i = w; i < total && ok; i += S::PW) {
        const bool more = i + S::PW < total;
        const SlotAt<S::KC, S::VC> next(more ? i + S::PW : i, nb);
        ok = slot_free(i) && (!more || known(next));
        if (!ok) break;
        const uint8_t *base = base_of(next);
        if (FMT == G4_PAGE_E4M3 && zero) {
#pragma unroll
          for (int k = 0; k < 16; k++)
            if ((zero >> k) & 1) d[k] = make_uint4(0, 0, 0, 0);
        }
        zero = more ? unseen(next) : 0;
        uint8_t *to = slot(i % S::NS);
        find(next);
#pragma unroll
        for (int k = 0; k < 16; k++) {
          const uint2 w0 = widen4<FMT>(d[k].x), w1 = widen4<FMT>(d[k].y), w2 = widen4<FMT>(d[k].z), w3 = widen4<FMT>(d[k].w);
          *reinterpret_cast<uint4 *>(to + o0 + k * 1024) = make_uint4(w0.x, w0.y, w1.x, w1.y);
          *reinterpret_cast<uint4 *>(to + o1 + k * 1024) = make_uint4(w2.x, w2.y, w3.x, w3.y);
          if (more) d[k] = load(base, k);
        }
        fence_async();
        __syncwarp();
        if (lane == 0) arrive(&full[i % S::NS]);
        if (more) used(next);
      }
    } else {
      // Eight copies of 16 rows x 64 dimensions, swizzled on the way, a lane each. They count on the
      // slot's barrier; where V has to be looked over first, on the warp's own.
      uint64_t *const own = &own_bar[w];
      uint32_t turn = 0;
      int asked = w;   // the slot after the last one asked for
#pragma unroll 1
      for (int i = w; i < total; i += S::PW) {
        const SlotAt<S::KC, S::VC> at(i, nb);
        ok = known(at) && slot_free(i);
        if (!ok) break;
        const int sl = i % S::NS;
        const bool partly = at.v && odd_block(at.j);
        uint64_t *const bar = partly ? own : &full[sl];
        if (lane == 0) mbar_expect_tx(bar, SLOT);
        __syncwarp();
        if (lane < 8) {
          constexpr int T = S::TV / 16;   // tiles of a V slot's column
          const int tile = at.v ? at.c * T + lane % T : lane, col = at.v ? half * S::VC + lane / T : at.c;
          tma_rows(slot(sl) + lane * 2048, at.v ? &map_v : &map_k, col * 128, (int)(info[at.j % NSC].at[tile] / ROW), bar);
        }
        asked = i + S::PW;
        if (partly) {
          ok = warp_wait(own, turn);
          turn ^= 1;
          if (!ok) break;
          // A weight of 0 must not meet an infinity or a NaN: positions no row sees become 0, and so do
          // values that are not finite in a block that some row sees only in part (rows that see them
          // are told by bad_v).
          const int rr = lane >> 3, x = lane & 7;
          const bool cut = edge(at.j);
#pragma unroll 1
          for (int k = 0; k < 32; k++) {
            const int r = 4 * k + rr, pos = at.c * S::TV + 4 * (k % (S::TV / 4)) + rr;
            uint4 *q = reinterpret_cast<uint4 *>(slot(sl) + r * 128 + ((x ^ (r & 7)) << 4));
            uint32_t u[4] = {q->x, q->y, q->z, q->w};
            const bool gone = !seen(at.j, pos);
            bool bad = false;
#pragma unroll
            for (int z = 0; z < 4; z++) {
              if ((u[z] & 0x7f80u) == 0x7f80u) {
                u[z] &= 0xffff0000u;
                bad = true;
              }
              if ((u[z] & 0x7f800000u) == 0x7f800000u) {
                u[z] &= 0xffffu;
                bad = true;
              }
            }
            if (gone)
              *q = make_uint4(0, 0, 0, 0);
            else if (bad && cut) {
              *q = make_uint4(u[0], u[1], u[2], u[3]);
              atomicOr(&bad_v[at.j < 2 ? at.j : 2 + (nb - 1 - at.j)][pos >> 5], 1u << (pos & 31));
            }
          }
          fence_async();
          __syncwarp();
          if (lane == 0) arrive(&full[sl]);
        }
        used(at);
      }
      // Every copy asked for has landed before the block can end: those of the ring's last round are
      // waited for here (a slot filled again since is of a round that its barrier no longer tells).
      for (int i = asked - S::PW; i >= w && i >= total - S::NS; i -= S::PW) warp_wait(&full[i % S::NS], (uint32_t)((i / S::NS) & 1));
    }
    if (!ok) {
      *failed = 1;
      paged_raise(a.err, G4_PAGED_TIMEOUT);
    }
  } else if (warp == kScout) {
    // ============================================================ the scout: lane l positions 4 l .. + 3
    const int32_t *table = a.table + (long long)b * a.table_stride;
    // The page of this lane's 16 positions, -2 where no row sees any of them.
    auto page_of = [&](int j) -> int {
      const int pos = (j0 + j) * BN + (lane >> 2) * 16;
      return j < nb && pos + 16 > rt.tlo && pos < rt.thi ? table[pos / p.page_size] : -2;
    };
    int page = page_of(0), next = page_of(1);
    bool ok = true;
    for (int j = 0; j < nb; j++) {
      const int k = j % NSC, pos = (j0 + j) * BN + (lane >> 2) * 16;
      long long row = -1;
      if (page >= 0 && page < p.n_pages)
        row = ((long long)page * p.kv_heads + kvh) * p.page_size + pos % p.page_size;
      else if (page != -2)
        paged_raise(a.err, G4_PAGED_BAD_PAGE);
      page = next;
      next = page_of(j + 2);
      const float none = row >= 0 ? 1.0f : -1.0f;
      float4 ks = make_float4(1, 1, 1, 1), vs = make_float4(none, none, none, none);
      if (HALF && row >= 0) {
        ks = __ldg(reinterpret_cast<const float4 *>(p.ks + row + (lane & 3) * 4));
        vs = __ldg(reinterpret_cast<const float4 *>(p.vs + row + (lane & 3) * 4));
      }
      float4 lv = make_float4(0, 0, 0, 0);
      if (HALF)
        lv = make_float4(__log2f(fmaxf(vs.x, 0x1p-100f)), __log2f(fmaxf(vs.y, 0x1p-100f)), __log2f(fmaxf(vs.z, 0x1p-100f)),
                         __log2f(fmaxf(vs.w, 0x1p-100f)));
      float hi_ = fmaxf(fmaxf(lv.x, lv.y), fmaxf(lv.z, lv.w)), lo_ = fminf(fminf(lv.x, lv.y), fminf(lv.z, lv.w));
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        hi_ = fmaxf(hi_, __shfl_xor_sync(0xffffffffu, hi_, d));
        lo_ = fminf(lo_, __shfl_xor_sync(0xffffffffu, lo_, d));
      }
      const bool even = __all_sync(0xffffffffu, row >= 0) && hi_ - lo_ <= 8.0f;
      if (j >= NSC) ok = warp_wait(&info_free[k], (uint32_t)((j / NSC - 1) & 1));
      if (!ok) break;
      BlockInfo &f = info[k];
      reinterpret_cast<float4 *>(f.ks)[lane] = ks;
      reinterpret_cast<float4 *>(f.vs)[lane] = vs;
      reinterpret_cast<float4 *>(f.lv)[lane] = lv;
      if ((lane & 3) == 0) f.at[lane >> 2] = row >= 0 ? row * (HALF ? HD : 2 * HD) : 0;
      if (lane == 0) {
        f.lmax = hi_;
        f.even = even;
      }
      __syncwarp();
      if (lane == 0) arrive(&info_full[k]);
    }
    if (!ok) {
      *failed = 1;
      paged_raise(a.err, G4_PAGED_TIMEOUT);
    }
  } else if (warp == kMma) {
    // ============================================================ products
    // One thread, and the slots of a group unrolled: an issue waits until the products before it are
    // nearly done, so whatever stands between two issues is lost. (Per block of head_dim 256, whose
    // products are 2,056 cycles: 2,326 like this, 3,490 with the slots in a loop, 4,490 with the whole
    // warp waiting and electing at each.)
    if (elect()) {
      constexpr uint32_t IS = idesc_f16(HALF, BN, false), IO = idesc_f16(HALF, S::OD, true);
      const uint64_t q0 = slot_desc(csm), k0 = slot_desc(slot(0)), v0 = slot_desc(slot(0), S::TV * 128);
      int at = 0;             // the ring's group at hand, in slots, and its round
      uint32_t round = 0;
      bool bad = false;       // a wait gave up: the rest is issued without waiting, and not used
      auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (!mbar_try_wait(bar, parity) && !bad) bad = !mbar_wait(bar, parity);
      };
      auto advance = [&] {
        at += S::G;
        if (at == S::NS) {
          at = 0;
          round ^= 1;
        }
      };
      auto scores = [&](int j) {
        const uint32_t d = t_s[j & 1];
        if (j >= 2) wait(pv_done, (uint32_t)(j & 1));   // O(j - 2) has read P from these columns
#pragma unroll
        for (int h = 0; h < S::KC / S::G; h++) {
          const uint64_t kd = k0 + at * (SLOT >> 4);
#pragma unroll
          for (int c = 0; c < S::G; c++) {
            wait(&full[at + c], round);
            fence_after();
#pragma unroll
            for (int k = 0; k < 4; k++)
              mma_ss(d, q0 + (h * S::G + c) * (SLOT >> 4) + 2 * k, kd + c * (SLOT >> 4) + 2 * k, IS, (h | c | k) != 0);
            commit(&empty[at + c]);
          }
          advance();
        }
        commit(&s_full[j & 1]);
      };
      auto outputs = [&](int j) {
        const uint32_t d = t_s[j & 1];
        const uint64_t vd = v0 + at * (SLOT >> 4);
        wait(&p_ready[j & 1], (uint32_t)((j >> 1) & 1));
#pragma unroll
        for (int c = 0; c < S::VC; c++) {
          wait(&full[at + c], round);
          fence_after();
#pragma unroll
          for (int k = 0; k < S::TV / 16; k++) {
            const int q = c * (S::TV / 16) + k;   // P of positions 64 .. lies over their S, from column 64
            mma_ts(t_o, d + 8 * q + (q >= 4 ? 32 : 0), vd + c * (SLOT >> 4) + 128 * k, IO, (j | q) != 0);
          }
          commit(&empty[at + c]);
        }
        advance();
        commit(pv_done);
      };
#pragma unroll 1
      for (int j = 0; j <= nb; j++) {
        if (j < nb) scores(j);
        if (j >= 1) outputs(j - 1);
      }
      // Everything issued has ended before tensor memory and the slots are given up.
      commit(end);
      if (!mbar_wait(end, 0)) bad = true;
      if (bad) {
        *failed = 1;
        paged_raise(a.err, G4_PAGED_TIMEOUT);
      }
    }
    __syncwarp();
  }
  float m = -INFINITY, l = 0.0f;
  int lo = 0, hi = 0;
  const float bits = HALF ? 13.0f : 0.0f;
  const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
  const int row = 32 * (warp & 3) + lane, ch = (warp >> 2) & 1;   // softmax: thread's row, its half of the columns
  if (warp < kSoftWarps) {
    // ============================================================ softmax
    const float qf = q_scale[row];
    if (row < rt.rows) row_range(a, s.pos + rt.row0 + row / a.group, s.kv, lo, hi);
    bool ok = true;
#pragma unroll 1
    for (int j = 0; j < nb; j++) {
      const int k = j % NSC, pos0 = (j0 + j) * BN + 64 * ch;
      const auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };
      if (ok) {
        const uint32_t pi = (uint32_t)((j / NSC) & 1), ps = (uint32_t)((j >> 1) & 1);
        ok = __all_sync(0xffffffffu, mbar_try_wait(&info_full[k], pi) && mbar_try_wait(&s_full[j & 1], ps)) ||
             (warp_wait(&info_full[k], pi) && warp_wait(&s_full[j & 1], ps));
      }
      if (!ok) {   // the other half's warp still counts on this one's barriers
        pair_sync();
        continue;
      }
      fence_after();
      const BlockInfo &f = info[k];
      const float4 *ks = reinterpret_cast<const float4 *>(f.ks + 64 * ch), *vs = reinterpret_cast<const float4 *>(f.vs + 64 * ch);
      const uint32_t at = t_s[j & 1] + lane_base + 64 * ch;
      const bool plain = (j0 + j) * BN >= rt.all_lo && (j0 + j + 1) * BN <= rt.all_hi && f.even;
      float z[2][32];
      tld32(at, z[0]);
      tld32(at + 32, z[1]);
      tld_wait();
      // The scores in units of log2, less the row's factor in the plain case.
      float top = -INFINITY;
      if (plain) {
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            if (HALF) {
              const float4 c = ks[8 * h + i / 4];
              const float2 u = un2(mul2(f2(z[h][i], z[h][i + 1]), f2(c.x, c.y)));
              const float2 w = un2(mul2(f2(z[h][i + 2], z[h][i + 3]), f2(c.z, c.w)));
              z[h][i] = u.x;
              z[h][i + 1] = u.y;
              z[h][i + 2] = w.x;
              z[h][i + 3] = w.y;
            }
            tops[0 + (i & 4) / 2] = max3(tops[0 + (i & 4) / 2], z[h][i], z[h][i + 1]);
            tops[1 + (i & 4) / 2] = max3(tops[1 + (i & 4) / 2], z[h][i + 2], z[h][i + 3]);
          }
        top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]) * qf + (HALF ? f.lmax : 0.0f);
      } else {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int i = 0; i < 32; i++) {
            const int q = 64 * ch + 32 * h + i, pos = pos0 + 32 * h + i;
            const bool see = pos >= lo && pos < hi && !(f.vs[q] < 0.0f);
            z[h][i] = see ? z[h][i] * f.ks[q] * qf : -INFINITY;
            if (see) top = fmaxf(top, z[h][i] + f.lv[q]);
          }
      }
      // With the other half of the columns.
      row_top[j & 1][ch][row] = top;
      pair_sync();
      top = fmaxf(top, row_top[j & 1][ch ^ 1][row]);
      // The maximum moves only when a row outgrows it by more than 2^2.9.
      const bool grow = top > m + 2.9f;
      if (__any_sync(0xffffffffu, grow)) {
        const float e = grow ? cex2(m - top) : 1.0f;
        if (grow) {
          l = m == -INFINITY ? 0.0f : crescale(l, m - top);
          m = top;
        }
        if (j > 0) {
          ok = warp_wait(pv_done, (uint32_t)((j - 1) & 1));
          if (!ok) continue;
          fence_after();
#pragma unroll 1
          for (int c = 0; c < S::OD / 32; c++) {
            const uint32_t oc = t_o + lane_base + ch * (S::OD / 2) + 16 * c;
            float o[16];
            tld16(oc, o);
            tld_wait();
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] *= e;
            tst16(oc, reinterpret_cast<const uint32_t(&)[16]>(o));
          }
        }
      }
      const float r = m == -INFINITY ? 0.0f : m - bits;
      F2 sum = f2(0.0f, 0.0f), sum1 = sum;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        uint32_t pk[16];
        if (plain) {
          const F2 q2 = f2(qf, qf), r2 = f2(-r, -r);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float2 y0 = un2(fma2(f2(z[h][i], z[h][i + 1]), q2, r2)), y1 = un2(fma2(f2(z[h][i + 2], z[h][i + 3]), q2, r2));
            F2 p0 = f2(cex2(y0.x), cex2(y0.y)), p1 = f2(cex2(y1.x), cex2(y1.y));
            sum = add2(sum, p0);
            sum1 = add2(sum1, p1);
            if (HALF) {
              const float4 c = vs[8 * h + i / 4];
              p0 = mul2(p0, f2(c.x, c.y));
              p1 = mul2(p1, f2(c.z, c.w));
            }
            const float2 w0 = un2(p0), w1 = un2(p1);
            pk[i / 2] = pack16<HALF>(w0.x, w0.y);
            pk[i / 2 + 1] = pack16<HALF>(w1.x, w1.y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 v = *reinterpret_cast<const float2 *>(f.vs + 64 * ch + 32 * h + i);
            const float e0 = cex2(z[h][i] - r), e1 = cex2(z[h][i + 1] - r);
            sum = add2(sum, f2(e0, e1));
            pk[i / 2] = pack16<HALF>(z[h][i] == -INFINITY ? 0.0f : e0 * v.x, z[h][i + 1] == -INFINITY ? 0.0f : e1 * v.y);
          }
        }
        tst16(at + 16 * h, pk);
      }
      const float2 two = un2(add2(sum, sum1));
      l += two.x + two.y;
      tst_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) {
        arrive(&p_ready[j & 1]);
        arrive(&info_free[k]);
      }
    }
    if (!ok) {
      *failed = 1;
      paged_raise(a.err, G4_PAGED_TIMEOUT);
    }
    // The row's sum over both halves of the columns (after the last maximum was read).
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
    row_top[0][ch][row] = l;
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
    l += row_top[0][ch ^ 1][row];
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp < kSoftWarps && !*failed) {
    // ============================================================ the rows out
    const int i = rt.row0 + row / a.group, h = kvh * a.group + row % a.group;
    const bool live = row < rt.rows;
    if (!HALF && nb > 0 && live) {
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
    __nv_bfloat16 *out = reinterpret_cast<__nv_bfloat16 *>(a.out) + (long long)(s.row + i) * a.o_stride + (long long)h * HD + half * S::OD + ch * (S::OD / 2);
#pragma unroll 1
    for (int c = 0; c < S::OD / 64; c++) {
      float o[32];
      if (nb > 0) {
        tld32(t_o + lane_base + ch * (S::OD / 2) + 32 * c, o);
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
          for (int q = 0; q < 4; q++) w[q] = pack16<false>(o[k + 2 * q] * inv, o[k + 2 * q + 1] * inv);
          *reinterpret_cast<uint4 *>(out + 32 * c + k) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    if (live && a.lse && half == 0 && ch == 0)
      a.lse[(long long)(s.row + i) * a.heads + h] = m == -INFINITY ? -INFINITY : (m - bits + log2f(l)) * kLn2f;
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == kMma) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
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
  CUtensorMap map_k = {}, map_v = {};
  if (!S::HALF) {
    // Rows of the pool as bytes; head_dim 64 or more of them stay far below 2^31.
    const uint64_t rows = (uint64_t)a.pool.n_pages * a.pool.kv_heads * a.pool.page_size;
    if (rows >= 1ull << 31 || make_tmap_u8(&map_k, a.pool.k, 2 * HD, rows, 2 * HD, 128, 16, true) ||
        make_tmap_u8(&map_v, a.pool.v, 2 * HD, rows, 2 * HD, 128, 16, true))
      return cudaErrorInvalidValue;
  }
  return launch_k(k_paged_chunk<FMT, HD>, grid, dim3(kThreads), S::SMEM, st, false, a, map_k, map_v);
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
