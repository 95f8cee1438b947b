// g4_paged_attn.cu -- attention of few new tokens (decode steps, verify passes) over paged,
// quantised keys and values.
//
// For the rows (query, head) that share a KV head, with codes K, V and scales ks, vs per position:
//   s_t = scale ks_t (q . K_t),  p_t = exp(s_t - M),  o = sum_t p_t vs_t V_t / sum_t p_t.
// M is the running maximum of s_t + ln vs_t, not of s_t: the greatest p_t vs_t is then 1 and the
// products' 16-bit weights keep their precision however far the scales lie apart; the sum of p_t
// is f32. What bounds the kernel is reading the codes once from HBM (1 byte a value at 8 bits), so
// everything else has to stay out of the loads' way:
//  - The 16 positions of a tile lie side by side in their page (a KV head's rows are contiguous), so
//    one bulk copy brings all of K's rows, one V's, two the scales. Each group of warps keeps a ring
//    of such units in flight; nothing but the copy engine waits for memory.
//  - Codes go from shared memory into the registers of the matrix products as they lie. The sums over
//    head_dim and over positions may run in any order: for S^T = K Q^T (16 positions x 8 rows) lane
//    (g, c) takes 16 bytes of positions g and g + 8 as its part of four K steps, for O^T = V^T P^T (16
//    dimensions x 8 rows) 16 bytes of positions 2c, 2c + 1, 2c + 8, 2c + 9, two dimensions a step. 8-bit
//    codes become f16 exactly in about an instruction each; Q is laid out to match, once.
//  - Eight rows fill the N of the products, so a group of 8 heads wastes none of it, and one
//    8 x 8 transpose in registers turns S^T's layout into P^T's.
//  - f32 rows: q and p vs are carried in two f16 parts (8-bit codes; 22 bits together) or three
//    bf16 parts (bf16 pages), one product each, all accumulated in f32.
// The work is one list: every (sequence, KV head, 8 RT rows) with its tiles, end to end. Each of a fixed
// number of blocks, as many as the SMs hold at once, takes an equal share of the list, so ragged
// lengths cost nothing (64 contexts of 128 .. 4,096 positions at head_dim 512: 68 us with a grid of
// equal splits, of which half the slots were empty and the rest worked in two rounds). A block's
// share may begin or end inside a context; such parts are joined by the last of 16 neighbours to
// finish, and those by the last of them (one block would read 2.4 MB alone for 148 parts of
// head_dim 512).
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "g4_device.cuh"
#include "g4_kernels.cuh"
#include "g4_paged.cuh"

namespace g4 {

constexpr int kDecWarps = 4;
// The list's units (plan_decode): what beginning a context costs, in tiles (64 x 4,096 at head_dim 256 47 us
// at 6, 45 at 12; 64 ragged at head_dim 512 67 at 1, 53 at 12 and 52 at 16), and the least share of a
// block, in tiles a warp (1 x 2,000: 18 us at 3, 19 at 5, 24 at 8).
constexpr int kBeginTiles = 16, kLeastTiles = 3;
constexpr int kRingKb = 96;          // of an SM's shared memory in rings
constexpr int kJoin = 16;            // partials one block joins
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kWeightBits = 14.0f; // 8-bit codes: weights are scaled by 2^14, clear of f16's subnormals

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// l 2^d for d <= 0. l may be as large as 2^114 (positions whose V scale is next to nothing), so that
// 2^d alone could underflow where the product does not.
__device__ __forceinline__ float rescale(float l, float d) {
  const float h = ex2(0.5f * d);
  return (l * h) * h;
}
template <bool HALF>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }

// Four codes in memory order as two f16 pairs. int8: u = code + 128 as the low byte of 1024 + u
// (exponent bits 0x64), less 1152: exact. e4m3 values are f16 values.
template <int FMT>
__device__ __forceinline__ void codes4(uint32_t w, uint32_t &lo, uint32_t &hi) {
  if (FMT == G4_PAGE_INT8) {
    const uint32_t x = w ^ 0x80808080u, magic = 0x64646464u;
    const uint32_t a = __byte_perm(x, magic, 0x4140), b = __byte_perm(x, magic, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));   // 1152
    lo = half2_bits(__hsub2(*reinterpret_cast<const __half2 *>(&a), off));
    hi = half2_bits(__hsub2(*reinterpret_cast<const __half2 *>(&b), off));
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffff), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    lo = *reinterpret_cast<const uint32_t *>(&a);
    hi = *reinterpret_cast<const uint32_t *>(&b);
  }
}

// v as parts of HALF (f16) or bf16, greatest first; their sum is v to 11 NP (or 8 NP) bits.
template <bool HALF, int NP>
__device__ __forceinline__ void split2(float v0, float v1, uint32_t (&out)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; i++) {
    if (HALF) {
      const __half2 h = __floats2half2_rn(v0, v1);
      out[i] = half2_bits(h);
      if (i + 1 < NP) {
        const float2 f = __half22float2(h);
        v0 = __fsub_rn(v0, f.x);
        v1 = __fsub_rn(v1, f.y);
      }
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v0, v1);
      out[i] = *reinterpret_cast<const uint32_t *>(&h);
      if (i + 1 < NP) {
        v0 = __fsub_rn(v0, __low2float(h));
        v1 = __fsub_rn(v1, __high2float(h));
      }
    }
  }
}

// Blocks an SM holds by registers.
constexpr int most_blocks(int hd) { return hd == 512 ? 2 : (hd == 256 ? 3 : 4); }

template <int FMT, int HD, int NP, int RT>
struct DecShape {
  static constexpr bool HALF = FMT != G4_PAGE_BF16;
  static constexpr int ES = HALF ? 1 : 2;              // bytes of a code
  static constexpr int ROW = HD * ES;                  // bytes of a position
  static constexpr bool NARROW = ROW == 64;            // V loads of 8 bytes instead of 16
  static constexpr int KSTEPS = HD / 16;
  static constexpr int TG = kDecWarps / RT;            // groups of warps, a ring each
  static constexpr int UNIT = 16 * ROW + (HALF ? 128 : 0);   // K's (with both scales) or V's 16 positions
  static constexpr int Q_BYTES = RT * NP * KSTEPS * 32 * 8;
  // Blocks on an SM: as many as the registers allow (O takes HD / 4 of them) with three units a ring.
  // (228 KB of shared memory an SM, 1 KB a block the system's; the arrays besides Q and ring.)
  static constexpr int ring_depth(int occ) {
    return ((occ == 1 ? 227 : 228 / occ - 1) * 1024 - 1536 - (kJoin + 1) * 8 * RT * 4 - Q_BYTES) / (TG * UNIT);
  }
  static constexpr int MOST = most_blocks(HD);
  static constexpr int OCC = ring_depth(MOST) >= 2 ? MOST : (ring_depth(2) >= 2 ? 2 : 1);
  // Deep enough for the bytes that HBM needs in flight and no deeper: the queue before the memory is
  // what every other load of the block waits in.
  static constexpr int WANT = kRingKb * 1024 / (OCC * TG * UNIT), CAP = ring_depth(OCC) > 8 ? 8 : ring_depth(OCC);
  static constexpr int D = WANT < 2 ? 2 : (WANT > CAP ? CAP : WANT);
  static_assert(D >= 2, "a ring holds K and V of a tile");
  static constexpr int RING = TG * D * UNIT, JOIN = TG * 8 * RT * (HD + 2) * 4;
  static constexpr int SMEM = Q_BYTES + RING > JOIN ? Q_BYTES + RING : JOIN;
};

// The join of `np` partials of `rows` rows (o [rows][HD], then m [rows], l [rows]), the first at `first`,
// the others `stride` floats apart from `rest` on: every thread takes part; result rows go to out and
// lse, or to another partial (`to`, which may be the first: each thread reads an element of all before
// it writes it).
template <int HD>
__device__ __forceinline__ void join_partials(const PagedAttn &a, const float *first, const float *rest, long long stride, int np, int rows,
                                              float *to, const SeqSpan &s, int kvh, int row0, float bits, float *fsh) {
  // fsh: [np][rows] factors, then [rows] l. Sixteen lanes a row, a partial each.
  const int t = threadIdx.x, nt = blockDim.x;
  auto part = [&](int i) { return i == 0 ? first : rest + (i - 1) * stride; };
  static_assert(kJoin == 16, "half a warp a row");
  for (int x = t; x < rows * kJoin; x += nt) {
    const int r = x / kJoin, i = x % kJoin;
    float m = -INFINITY, l = 0.0f;
    if (i < np) {
      m = __ldcg(part(i) + rows * HD + r);
      l = __ldcg(part(i) + rows * HD + rows + r);
    }
    float M = m;
#pragma unroll
    for (int d = 1; d < kJoin; d <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    if (i < np) fsh[i * rows + r] = M == -INFINITY ? 0.0f : ex2(m - M);
    l = i < np ? rescale(l, M == -INFINITY ? 0.0f : m - M) : 0.0f;
#pragma unroll
    for (int d = 1; d < kJoin; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    if (i != 0) continue;
    fsh[np * rows + r] = l;
    const int rr = row0 + r, j = rr / a.group;
    if (to) {
      to[rows * HD + r] = M;
      to[rows * HD + rows + r] = l;
    } else if (a.lse && j < s.n) {
      a.lse[(long long)(s.row + j) * a.heads + kvh * a.group + rr % a.group] =
          M == -INFINITY ? -INFINITY : (M - bits + log2f(l)) * kLn2;
    }
  }
  __syncthreads();
  for (int e = t; e < rows * (HD / 4); e += nt) {
    const int r = e / (HD / 4), d = e % (HD / 4) * 4, rr = row0 + r, i = rr / a.group;
    if (!to && i >= s.n) continue;
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int k0 = 0; k0 < kJoin; k0 += 8) {
      if (k0 >= np) break;
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; k++)
        v[k] = k0 + k < np ? __ldcg(reinterpret_cast<const float4 *>(part(k0 + k) + r * HD + d)) : make_float4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float f = k0 + k < np ? fsh[(k0 + k) * rows + r] : 0.0f;
        o.x = fmaf(f, v[k].x, o.x);
        o.y = fmaf(f, v[k].y, o.y);
        o.z = fmaf(f, v[k].z, o.z);
        o.w = fmaf(f, v[k].w, o.w);
      }
    }
    if (to) {
      *reinterpret_cast<float4 *>(to + r * HD + d) = o;
      continue;
    }
    const float l = fsh[np * rows + r], inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const long long at = (long long)(s.row + i) * a.o_stride + (long long)(kvh * a.group + rr % a.group) * HD + d;
    if (a.type == G4_F32) {
      *reinterpret_cast<float4 *>((float *)a.out + at) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    } else {
      const __nv_bfloat162 u = __floats2bfloat162_rn(o.x * inv, o.y * inv), v = __floats2bfloat162_rn(o.z * inv, o.w * inv);
      *reinterpret_cast<uint2 *>((__nv_bfloat16 *)a.out + at) =
          make_uint2(*reinterpret_cast<const uint32_t *>(&u), *reinterpret_cast<const uint32_t *>(&v));
    }
  }
}

// RT warps share each tile of positions, one row tile of 8 each; 4 / RT tiles are worked on side by side.
template <int FMT, int HD, int NP, int RT>
__global__ void __launch_bounds__(kDecWarps * 32, DecShape<FMT, HD, NP, RT>::OCC) k_paged_decode(const PagedAttn a) {
  using S = DecShape<FMT, HD, NP, RT>;
  constexpr bool HALF = S::HALF;
  constexpr int TG = S::TG, ROWS = 8 * RT, D = S::D, NT = kDecWarps * 32;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, c = lane & 3;
  const int rt = warp % RT, tg = warp / RT;
  const Pool &p = a.pool;
  const int per_page = p.page_size >> 4;

  extern __shared__ __align__(128) uint8_t dsm[];   // Q, then the groups' rings; at the end the groups' partials
  uint8_t *const ring = dsm + S::Q_BYTES + tg * D * S::UNIT;
  __shared__ uint64_t full_[TG][D], empty_[TG][D];
  __shared__ int has_[TG][D];   // whether the unit's page exists
  __shared__ float q_scale[ROWS];
  __shared__ int row_lo[ROWS], row_hi[ROWS];
  __shared__ float fsh[(kJoin + 1) * ROWS];
  __shared__ int sum_sh[kDecWarps + 4];
  uint64_t *const full = full_[tg], *const empty = empty_[tg];
  volatile int *const has = has_[tg];
  if (t == 0) {
    for (int i = 0; i < TG * D; i++) {
      mbar_init(&full_[0][i], 1);
      mbar_init(&empty_[0][i], RT);
    }
    mbar_fence_init();
  }

  // ---- the list. Tiles of row group rg of sequence s from its first one, and before them a.begin_tiles
  // that stand for what beginning it costs (a second part of a block's share costs as much as so many
  // tiles; where nothing is seen they are all there is, and zeros are written).
  auto tiles_of = [&](const SeqSpan &s, int rg, int &first) {
    const int R = s.n * a.group, r0 = rg * ROWS;
    if (r0 >= R) return 0;
    int lo, hi, tmp;
    row_range(a, s.pos + r0 / a.group, s.kv, lo, tmp);
    row_range(a, s.pos + (min(r0 + ROWS, R) - 1) / a.group, s.kv, tmp, hi);
    first = lo >> 4;
    return (hi > lo ? ((hi + 15) >> 4) - first : 0) + a.begin_tiles;
  };
  // All row groups' tiles of a sequence for one KV head, by the whole warp.
  auto all_groups = [&](const SeqSpan &s) {
    int n = 0, first;
    if (a.row_groups == 1) return tiles_of(s, 0, first);
    for (int rg = lane; rg < a.row_groups; rg += 32) n += tiles_of(s, rg, first);
    return __reduce_add_sync(0xffffffffu, n);
  };
  // All tiles of sequence b, by one thread.
  auto seq_tiles = [&](int b, bool report) -> long long {
    const SeqSpan s = seq_span(a, b, report);
    int n = 0, first;
    for (int rg = 0; rg < a.row_groups; rg++) n += tiles_of(s, rg, first);
    return (long long)n * p.kv_heads;
  };
  // Thread t holds the tiles of its share of the sequences; the block's scan gives where each begins.
  const int per = (a.batch + NT - 1) / NT;
  long long mine_sum = 0;
  if (a.row_groups < 8) {
    for (int i = 0; i < per; i++) {
      const int b = t * per + i;
      if (b < a.batch) mine_sum += seq_tiles(b, blockIdx.x == 0);
    }
  } else {   // (a chunk of f32 rows has hundreds: a sequence at a time, 32 groups at once)
    for (int b = warp * 32 * per; b < min(a.batch, (warp + 1) * 32 * per); b++) {
      const int n = all_groups(seq_span(a, b, blockIdx.x == 0 && lane == 0));
      if (lane == b / per - warp * 32) mine_sum += (long long)n * p.kv_heads;
    }
  }
  long long incl = mine_sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  __shared__ long long warp_sum[kDecWarps];
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  long long before = incl - mine_sum, total = 0;
#pragma unroll
  for (int w = 0; w < kDecWarps; w++) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const long long share = max((total + gridDim.x - 1) / gridDim.x, (long long)a.split_tiles);
  long long at = share * blockIdx.x;
  const long long end = min(total, at + share);
  if (at >= end) return;
  // The sequence this block begins in, and where its tiles begin.
  __shared__ long long seq_at_sh;
  if (before <= at && at < before + mine_sum) {
    long long x = before;
    int b = t * per;
    for (; per > 1; b++) {
      const long long n = seq_tiles(b, false);
      if (at < x + n) break;
      x += n;
    }
    sum_sh[0] = b;
    seq_at_sh = x;
  }
  __syncthreads();
  int b = sum_sh[0];
  long long seq_at = seq_at_sh;
  int ubase = 0;   // units of the ring used by the parts before

  bool bad = false;   // a wait gave up: go on without waiting (the call is reported as not complete)
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (!bad && !mbar_wait(bar, parity)) bad = true;
  };
  auto lds16 = [](const uint8_t *at) { return *reinterpret_cast<const uint4 *>(at); };
  uint2 *const qs = reinterpret_cast<uint2 *>(dsm);   // [RT][NP][KSTEPS][32]
  const uint2 *const qw = qs + (size_t)rt * NP * S::KSTEPS * 32 + lane;

#pragma unroll 1
  while (at < end) {
    // ---- the part at hand: KV head and row group of sequence b, its tiles tile0 .. tile1 - 1.
    const SeqSpan s = seq_span(a, b, false);
    int kvh = 0, rg = 0, first = 0, tiles;
    long long item_at = seq_at;
    {
      const int all = all_groups(s);
      if (at >= seq_at + (long long)all * p.kv_heads) {   // this sequence is done
        seq_at += (long long)all * p.kv_heads;
        b++;
        continue;
      }
      kvh = (int)((at - seq_at) / all);
      item_at += (long long)kvh * all;
      if (a.row_groups > 1) {
        // The row group that `at` lies in: a scan of 32 at a time.
        int off = (int)(at - item_at), unused;
        for (int r0 = 0;; r0 += 32) {
          const int n = r0 + lane < a.row_groups ? tiles_of(s, r0 + lane, unused) : 0;
          int upto = n;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
          }
          const unsigned past = __ballot_sync(0xffffffffu, off < upto);
          if (past) {
            const int l = __ffs((int)past) - 1;
            rg = r0 + l;
            item_at += __shfl_sync(0xffffffffu, upto - n, l);
            break;
          }
          const int sum = __shfl_sync(0xffffffffu, upto, 31);
          off -= sum;
          item_at += sum;
        }
      }
      tiles = tiles_of(s, rg, first);
    }
    const int R = s.n * a.group, row0 = rg * ROWS;
    const int from = (int)(at - item_at), count = (int)min((long long)tiles - from, end - at);
    // The share may end among the tiles that stand for the beginning: then there is nothing to do here.
    const int begin = a.begin_tiles, real = tiles - begin;
    const int tile0 = first + max(from - begin, 0), tile1 = first + max(from + count - begin, 0);
    if (real > 0 && tile1 == tile0) {
      at += count;
      continue;
    }
    const bool complete = tile1 - tile0 == real;

    // ---- this group's tiles: tile0 + tg + TG n; its first warp asks for them.
    const int mine = tile1 - tile0 - tg > 0 ? (tile1 - tile0 - tg + TG - 1) / TG : 0;
    const int32_t *table = a.table + (long long)b * a.table_stride;
    // Lane i of the first warp holds where the rows of the i-th of 32 tiles from pages_at on lie in the
    // pool (-1: no such page), so that asking for one is a shuffle and the copies.
    long long rows = -1;
    int pages_at = 0;
    auto fetch_pages = [&](int n) {
      const int k = n + lane;
      rows = -1;
      if (k < mine) {
        const int tile = tile0 + tg + TG * k, of = tile / per_page;
        const int page = table[of];
        if (page < 0 || page >= p.n_pages)
          paged_raise(a.err, G4_PAGED_BAD_PAGE);
        else
          rows = ((long long)page * p.kv_heads + kvh) * p.page_size + (tile - of * per_page) * 16;
      }
      pages_at = n;
    };
    if (rt == 0 && mine > 0) fetch_pages(0);

    // ---- Q: its loads go out before the first positions are asked for. One warp a row, two rows at a
    // time; a lane takes four dimensions of each 128.
    constexpr int QC = (HD + 127) / 128;
    float4 qv[2][QC];
    auto load_q = [&](int r, float4 (&v)[QC]) {
      const int rr = row0 + r, i = rr / a.group;
#pragma unroll
      for (int j = 0; j < QC; j++) {
        const int d = 128 * j + 4 * lane;
        v[j] = make_float4(0, 0, 0, 0);
        if (rr < R && d < HD) {
          const long long from = (long long)(s.row + i) * a.q_stride + (long long)(kvh * a.group + rr % a.group) * HD + d;
          if (a.type == G4_F32) {
            v[j] = *reinterpret_cast<const float4 *>((const float *)a.q + from);
          } else {
            const uint2 u = *reinterpret_cast<const uint2 *>((const __nv_bfloat16 *)a.q + from);
            v[j] = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                               __uint_as_float(u.y & 0xffff0000u));
          }
        }
      }
    };
    load_q(warp, qv[0]);
    load_q(warp + kDecWarps, qv[1]);

    // Unit u of the group (K of tile u / 2, or V) into slot sl, by its whole first warp.
    auto request = [&](int u, int sl) {
      const int n = u >> 1;
      if (n >= mine) return;
      if (n - pages_at >= 32) fetch_pages(n);
      const long long row = __shfl_sync(0xffffffffu, rows, n - pages_at);
      if (lane != 0) return;
      has[sl] = row >= 0;
      if (row < 0) {
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&full[sl])) : "memory");
        return;
      }
      uint8_t *to = ring + sl * S::UNIT;
      const bool is_v = u & 1;
      mbar_expect_tx(&full[sl], 16 * S::ROW + (HALF && !is_v ? 128 : 0));
      bulk_g2s(to, (is_v ? p.v : p.k) + row * S::ROW, 16 * S::ROW, &full[sl]);
      if (HALF && !is_v) {
        bulk_g2s(to + 16 * S::ROW, p.ks + row, 64, &full[sl]);
        bulk_g2s(to + 16 * S::ROW + 64, p.vs + row, 64, &full[sl]);
      }
    };
    const int sl0 = ubase % D;   // the first unit's slot
    if (rt == 0)
      for (int u = 0; u < D; u++) request(u, sl0 + u < D ? sl0 + u : sl0 + u - D);

    // Q into fragment order: for K step k of row tile r lane (g, c) holds four consecutive dimensions of
    // row g. 8-bit pages: f16 parts, scaled by a power of two that takes the row's greatest to 2^8 .. 2^9.
#pragma unroll 1
    for (int r0 = warp; r0 < ROWS; r0 += 2 * kDecWarps) {
      if (r0 > warp) {
        load_q(r0, qv[0]);
        load_q(r0 + kDecWarps, qv[1]);
      }
#pragma unroll
      for (int z = 0; z < 2; z++) {
        const int r = r0 + z * kDecWarps;
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < QC; j++)
          top = fmaxf(fmaxf(fmaxf(top, fabsf(qv[z][j].x)), fmaxf(fabsf(qv[z][j].y), fabsf(qv[z][j].z))), fabsf(qv[z][j].w));
        int e = 0;
        if (HALF) {
          // (Magnitudes order as their bits do.) Infinities and NaN stay what they are at any scale.
          e = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23) - 127;
          e = e < -110 ? -110 : (e > 127 ? 0 : e);
        }
        const float f = HALF ? __uint_as_float((uint32_t)(127 + 8 - e) << 23) : 1.0f;
#pragma unroll
        for (int j = 0; j < QC; j++) {
          const int d = 128 * j + 4 * lane;
          uint32_t p01[NP], p23[NP];
          split2<HALF, NP>(qv[z][j].x * f, qv[z][j].y * f, p01);
          split2<HALF, NP>(qv[z][j].z * f, qv[z][j].w * f, p23);
          // 8 bit: d = 64 m + 16 c + 4 j, step 4 m + j; 16 bit: d = 32 m + 8 c + 4 j, step 2 m + j.
          const int step = HALF ? (d >> 6) * 4 + ((d >> 2) & 3) : (d >> 5) * 2 + ((d >> 2) & 1);
          const int cc = HALF ? (d >> 4) & 3 : (d >> 3) & 3;
          if (d < HD && r < ROWS) {
#pragma unroll
            for (int k = 0; k < NP; k++)
              qs[(((r >> 3) * NP + k) * S::KSTEPS + step) * 32 + (r & 7) * 4 + cc] = make_uint2(p01[k], p23[k]);
          }
        }
        if (lane == 0 && r < ROWS) {
          q_scale[r] = a.scale * kLog2e * (HALF ? __uint_as_float((uint32_t)(127 - 8 + e) << 23) : 1.0f);
          int x0 = 0, x1 = 0;
          if (row0 + r < R) row_range(a, s.pos + (row0 + r) / a.group, s.kv, x0, x1);
          row_lo[r] = x0;
          row_hi[r] = x1;
        }
      }
    }
    __syncthreads();

    const float qf0 = q_scale[rt * 8 + 2 * c], qf1 = q_scale[rt * 8 + 2 * c + 1];
    const int lo0 = row_lo[rt * 8 + 2 * c], hi0 = row_hi[rt * 8 + 2 * c];
    const int lo1 = row_lo[rt * 8 + 2 * c + 1], hi1 = row_hi[rt * 8 + 2 * c + 1];
    // Positions that every row of this warp sees need no mask.
    const int rv = min(8, R - row0 - rt * 8);   // rows of this warp's tile that exist
    int all_lo = 0, all_hi = 0;
    if (rv > 0) {
      all_lo = row_lo[rt * 8 + rv - 1];
      all_hi = row_hi[rt * 8];
    }

    float o[HD / 16][4];
#pragma unroll
    for (int i = 0; i < HD / 16; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

    // This warp is done with unit u in slot sl; the first warp of the group asks for the unit that takes its
    // place.
    auto release = [&](int u, int sl, uint32_t round) {
      __syncwarp();
      if (RT > 1) {
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&empty[sl])) : "memory");
        if (rt == 0 && (u + D) >> 1 < mine) wait(&empty[sl], round);
        __syncwarp();
      }
      if (rt == 0) request(u + D, sl);
    };
    int sl = sl0;                                       // the ring's slot at hand and its round
    uint32_t round = (uint32_t)(ubase / D) & 1;
    auto advance = [&] {
      if (++sl == D) {
        sl = 0;
        round ^= 1;
      }
    };

#pragma unroll 1
    for (int n = 0; n < mine; n++) {
      const int pos0 = (tile0 + tg + TG * n) * 16;
      wait(&full[sl], round);
      const bool on = has[sl];
      float sc[4][4] = {};
      float ks0 = 1.0f, ks1 = 1.0f, w0 = 1.0f, w1 = 1.0f;
      const uint8_t *unit = ring + sl * S::UNIT;
      if (on) {
        const uint8_t *kp = unit + g * S::ROW + c * 16;
        if (HALF) {
          const float *f = reinterpret_cast<const float *>(unit + 16 * S::ROW);
          ks0 = f[g];
          ks1 = f[g + 8];
          w0 = f[16 + g];
          w1 = f[24 + g];
        }
        constexpr int ST = HALF ? 4 : 2;
#pragma unroll 2
        for (int m = 0; m < S::ROW / 64; m++) {
          const uint4 x = lds16(kp + 64 * m), y = lds16(kp + 64 * m + 8 * S::ROW);
          const uint32_t r0[4] = {x.x, x.y, x.z, x.w}, r1[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int j = 0; j < ST; j++) {
            uint32_t a0, a1, a2, a3;
            if constexpr (HALF) {
              codes4<FMT>(r0[j], a0, a2);
              codes4<FMT>(r1[j], a1, a3);
            } else {
              a0 = r0[2 * j];
              a2 = r0[2 * j + 1];
              a1 = r1[2 * j];
              a3 = r1[2 * j + 1];
            }
#pragma unroll
            for (int k = 0; k < NP; k++) {
              const uint2 bq = qw[(k * S::KSTEPS + m * ST + j) * 32];
              mma16816<HALF>(sc[(m * ST + j) & 3], a0, a1, a2, a3, bq.x, bq.y);
            }
          }
        }
      }
      release(2 * n, sl, round);
      advance();
      // ---- softmax of the tile: sums 0, 1 are position g of rows 2c, 2c + 1; 2, 3 position g + 8.
      float sa[4];
#pragma unroll
      for (int i = 0; i < 4; i++) sa[i] = (sc[0][i] + sc[1][i]) + (sc[2][i] + sc[3][i]);
      float s0 = sa[0] * (ks0 * qf0), s1 = sa[1] * (ks0 * qf1), s2 = sa[2] * (ks1 * qf0), s3 = sa[3] * (ks1 * qf1);
      bool see0 = on, see1 = on, see2 = on, see3 = on;
      const bool whole = on && pos0 >= all_lo && pos0 + 16 <= all_hi;
      uint32_t dead = 0;   // positions that no row of the warp sees
      if (!whole && on) {
        const int t0 = pos0 + g, t1 = t0 + 8;
        see0 = t0 >= lo0 && t0 < hi0;
        see1 = t0 >= lo1 && t0 < hi1;
        see2 = t1 >= lo0 && t1 < hi0;
        see3 = t1 >= lo1 && t1 < hi1;
        const unsigned live0 = __ballot_sync(0xffffffffu, see0 || see1), live1 = __ballot_sync(0xffffffffu, see2 || see3);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (!((live0 >> (4 * i)) & 0xf)) dead |= 1u << i;
          if (!((live1 >> (4 * i)) & 0xf)) dead |= 1u << (i + 8);
        }
      }
      const float g0 = HALF ? __log2f(fmaxf(w0, 0x1p-100f)) : 0.0f, g1 = HALF ? __log2f(fmaxf(w1, 0x1p-100f)) : 0.0f;
      s0 = see0 ? s0 : -INFINITY;
      s1 = see1 ? s1 : -INFINITY;
      s2 = see2 ? s2 : -INFINITY;
      s3 = see3 ? s3 : -INFINITY;
      float n0 = fmaxf(s0 + g0, s2 + g1), n1 = fmaxf(s1 + g0, s3 + g1);
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
      }
      n0 = fmaxf(n0, m0);
      n1 = fmaxf(n1, m1);
      if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
        const float f0 = n0 > m0 ? ex2(m0 - n0) : 1.0f, f1 = n1 > m1 ? ex2(m1 - n1) : 1.0f;
        l0 = n0 > m0 ? rescale(l0, m0 - n0) : l0;
        l1 = n1 > m1 ? rescale(l1, m1 - n1) : l1;
#pragma unroll
        for (int i = 0; i < HD / 16; i++) {
          o[i][0] *= f0;
          o[i][1] *= f1;
          o[i][2] *= f0;
          o[i][3] *= f1;
        }
        m0 = n0;
        m1 = n1;
      }
      uint32_t pw[2][NP];
      {
        const float bits = HALF ? kWeightBits : 0.0f;
        const float r0 = m0 == -INFINITY ? 0.0f : m0 - bits, r1 = m1 == -INFINITY ? 0.0f : m1 - bits;
        const float p0 = ex2(s0 - r0), p1 = ex2(s1 - r1), p2 = ex2(s2 - r0), p3 = ex2(s3 - r1);
        l0 += p0 + p2;
        l1 += p1 + p3;
        uint32_t x[NP], y[NP];
        split2<HALF, NP>(see0 ? p0 * w0 : 0.0f, see1 ? p1 * w0 : 0.0f, x);
        split2<HALF, NP>(see2 ? p2 * w1 : 0.0f, see3 ? p3 * w1 : 0.0f, y);
#pragma unroll
        for (int k = 0; k < NP; k++) {
          pw[0][k] = transpose8x8(x[k]);
          pw[1][k] = transpose8x8(y[k]);
        }
      }
      wait(&full[sl], round);
      if (on) {
        const uint8_t *vp = ring + sl * S::UNIT + 2 * c * S::ROW + g * (S::NARROW ? 8 : 16);
        uint32_t odd = 0;   // bf16 pages: this lane met a value that is not finite at its i-th position
        constexpr int MM = S::NARROW ? 1 : S::ROW / 128;
#pragma unroll
        for (int mm = 0; mm < MM; mm++) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint8_t *at = vp + ((i & 1) + (i >> 1) * 8) * S::ROW + mm * 128;
            if (S::NARROW) {
              const uint2 w = *reinterpret_cast<const uint2 *>(at);
              v[i] = make_uint4(w.x, w.y, 0, 0);
            } else {
              v[i] = lds16(at);
            }
          }
          if (FMT != G4_PAGE_INT8 && !whole) {
            // What no row sees may be anything, and 0 times an infinity or a NaN is NaN. e4m3 codes of
            // stored rows are finite; in bf16 pages a row may see a position that another does not.
#pragma unroll
            for (int i = 0; i < 4; i++) {
              if ((dead >> (2 * c + (i & 1) + (i >> 1) * 8)) & 1) v[i] = make_uint4(0, 0, 0, 0);
              if constexpr (!HALF) {
                uint32_t z[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                  if ((z[k] & 0x7f80u) == 0x7f80u) {
                    z[k] &= 0xffff0000u;
                    odd |= 1u << i;
                  }
                  if ((z[k] & 0x7f800000u) == 0x7f800000u) {
                    z[k] &= 0xffffu;
                    odd |= 1u << i;
                  }
                }
                v[i] = make_uint4(z[0], z[1], z[2], z[3]);
              }
            }
          }
          const uint32_t vw[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w}, {v[1].x, v[1].y, v[1].z, v[1].w},
                                     {v[2].x, v[2].y, v[2].z, v[2].w}, {v[3].x, v[3].y, v[3].z, v[3].w}};
          constexpr int WORDS = S::NARROW ? 2 : 4;
          const int ob = mm * (HALF ? 8 : 4);
#pragma unroll
          for (int j = 0; j < WORDS; j++) {
            if constexpr (HALF) {
              // Four dimensions of the pairs (2c, 2c + 1) and (2c + 8, 2c + 9).
              uint32_t e[2][4];
#pragma unroll
              for (int h = 0; h < 2; h++) {
                const uint32_t t0 = __byte_perm(vw[2 * h][j], vw[2 * h + 1][j], 0x5140);
                const uint32_t t1 = __byte_perm(vw[2 * h][j], vw[2 * h + 1][j], 0x7362);
                codes4<FMT>(t0, e[h][0], e[h][1]);
                codes4<FMT>(t1, e[h][2], e[h][3]);
              }
#pragma unroll
              for (int i = 0; i < 2; i++)
#pragma unroll
                for (int k = 0; k < NP; k++)
                  mma16816<HALF>(o[ob + 2 * j + i], e[0][2 * i], e[0][2 * i + 1], e[1][2 * i], e[1][2 * i + 1], pw[0][k], pw[1][k]);
            } else {
              const uint32_t a0 = __byte_perm(vw[0][j], vw[1][j], 0x5410), a1 = __byte_perm(vw[0][j], vw[1][j], 0x7632);
              const uint32_t a2 = __byte_perm(vw[2][j], vw[3][j], 0x5410), a3 = __byte_perm(vw[2][j], vw[3][j], 0x7632);
#pragma unroll
              for (int k = 0; k < NP; k++) mma16816<HALF>(o[ob + j], a0, a1, a2, a3, pw[0][k], pw[1][k]);
            }
          }
        }
        if (!HALF && __any_sync(0xffffffffu, odd != 0)) {
          // Rows that see such a position are not finite.
          uint32_t lanes[4];
#pragma unroll
          for (int i = 0; i < 4; i++) lanes[i] = __ballot_sync(0xffffffffu, (odd >> i) & 1);
          const uint32_t of = 0x11111111u << (g >> 1);
          const bool b0 = ((g & 1) ? lanes[1] : lanes[0]) & of, b1 = ((g & 1) ? lanes[3] : lanes[2]) & of;
          const float nan = __int_as_float(0x7fffffff);
          if ((b0 && see0) || (b1 && see2)) l0 = nan;
          if ((b0 && see1) || (b1 && see3)) l1 = nan;
        }
      }
      release(2 * n + 1, sl, round);
      advance();
    }
    if (bad) {
      paged_raise(a.err, G4_PAGED_TIMEOUT);
      // What was asked for has landed, or a second limit has passed, before the ring is given up.
      for (int u = 2 * mine > D ? 2 * mine - D : 0; u < 2 * mine; u++) mbar_wait(&full[(ubase + u) % D], (uint32_t)(((ubase + u) / D) & 1));
    }

    // ---- join the token groups through shared memory (over Q), then write out or leave a partial.
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    __syncthreads();
    // Partials [TG]: o [ROWS][HD], m [ROWS], l [ROWS].
    constexpr int PART = ROWS * (HD + 2);
    float *sm = reinterpret_cast<float *>(dsm) + tg * PART;
#pragma unroll
    for (int q = 0; q < HD / 16; q++) {
      // Accumulator q: dimensions 16 g + 2 j of a 128-byte column (8 bit; 8 g + 2 j narrow or at 16 bits) and the next.
      constexpr int PER = S::NARROW ? 4 : (HALF ? 8 : 4);
      const int chunk = q / PER, j = q % PER;
      const int d = chunk * (HALF && !S::NARROW ? 128 : 64) + g * (HALF && !S::NARROW ? 16 : 8) + 2 * j;
      *reinterpret_cast<float2 *>(sm + (rt * 8 + 2 * c) * HD + d) = make_float2(o[q][0], o[q][2]);
      *reinterpret_cast<float2 *>(sm + (rt * 8 + 2 * c + 1) * HD + d) = make_float2(o[q][1], o[q][3]);
    }
    if (g == 0) {
      sm[ROWS * HD + rt * 8 + 2 * c] = m0;
      sm[ROWS * HD + rt * 8 + 2 * c + 1] = m1;
      sm[ROWS * HD + ROWS + rt * 8 + 2 * c] = l0;
      sm[ROWS * HD + ROWS + rt * 8 + 2 * c + 1] = l1;
    }
    __syncthreads();
    const float bits = HALF ? kWeightBits : 0.0f;
    // Partial slots: 2 i for a part that block i begins inside of, 2 i + 1 for one it begins and leaves.
    const int c_first = (int)((item_at + begin) / share), c_last = (int)((item_at + tiles - 1) / share), me = blockIdx.x;
    auto slot_of = [&](int i) { return i == c_first ? 2 * i + 1 : 2 * i; };
    float *mine_part = complete ? nullptr : a.part + (long long)slot_of(me) * PART;
    {
      // The same join as between blocks, its partials in shared memory.
      const float *sp = reinterpret_cast<const float *>(dsm);
      for (int r = t; r < ROWS; r += kDecWarps * 32) {
        float M = -INFINITY, l = 0.0f;
        for (int i = 0; i < TG; i++) M = fmaxf(M, sp[i * PART + ROWS * HD + r]);
        for (int i = 0; i < TG; i++) {
          const float m = sp[i * PART + ROWS * HD + r];
          fsh[i * ROWS + r] = M == -INFINITY ? 0.0f : ex2(m - M);
          l += rescale(sp[i * PART + ROWS * HD + ROWS + r], M == -INFINITY ? 0.0f : m - M);
        }
        fsh[TG * ROWS + r] = l;
        const int rr = row0 + r, i = rr / a.group;
        if (mine_part) {
          mine_part[ROWS * HD + r] = M;
          mine_part[ROWS * HD + ROWS + r] = l;
        } else if (a.lse && rr < R) {
          a.lse[(long long)(s.row + i) * a.heads + kvh * a.group + rr % a.group] =
              M == -INFINITY ? -INFINITY : (M - bits + log2f(l)) * kLn2;
        }
      }
      __syncthreads();
      for (int e = t; e < ROWS * (HD / 4); e += kDecWarps * 32) {
        const int r = e / (HD / 4), d = e % (HD / 4) * 4, rr = row0 + r, i = rr / a.group;
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < TG; k++) {
          const float f = fsh[k * ROWS + r];
          const float4 z = *reinterpret_cast<const float4 *>(sp + k * PART + r * HD + d);
          v.x = fmaf(f, z.x, v.x);
          v.y = fmaf(f, z.y, v.y);
          v.z = fmaf(f, z.z, v.z);
          v.w = fmaf(f, z.w, v.w);
        }
        if (mine_part) {
          *reinterpret_cast<float4 *>(mine_part + r * HD + d) = v;
          continue;
        }
        if (rr >= R) continue;
        const float l = fsh[TG * ROWS + r], inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const long long at = (long long)(s.row + i) * a.o_stride + (long long)(kvh * a.group + rr % a.group) * HD + d;
        if (a.type == G4_F32) {
          *reinterpret_cast<float4 *>((float *)a.out + at) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        } else {
          *reinterpret_cast<uint2 *>((__nv_bfloat16 *)a.out + at) = make_uint2(
              [&] { const __nv_bfloat162 h = __floats2bfloat162_rn(v.x * inv, v.y * inv); return *reinterpret_cast<const uint32_t *>(&h); }(),
              [&] { const __nv_bfloat162 h = __floats2bfloat162_rn(v.z * inv, v.w * inv); return *reinterpret_cast<const uint32_t *>(&h); }());
        }
      }
    }
    if (!complete) {
      // ---- the last of each kJoin neighbours joins them; the last of those the whole.
      const int parts = c_last - c_first + 1, groups = (parts + kJoin - 1) / kJoin, grp = (me - c_first) / kJoin;
      const int g0 = c_first + grp * kJoin, in_group = min(kJoin, parts - grp * kJoin);
      uint32_t *group_count = a.count + 2 * slot_of(g0), *all_count = a.count + 2 * slot_of(c_first) + 1;
      __syncthreads();
      if (t == 0) {
        __threadfence();   // (orders what the barrier has ordered before it)
        const bool last = atomicAdd(group_count, 1u) == (unsigned)in_group - 1;
        __threadfence();
        if (last) *group_count = 0;
        sum_sh[1] = last;
      }
      __syncthreads();
      if (sum_sh[1]) {
        // Slots of a group's members are 2 PART apart from the second on; the first one's place differs.
        float *base = a.part + (long long)slot_of(g0) * PART;
        join_partials<HD>(a, base, in_group > 1 ? a.part + (long long)slot_of(g0 + 1) * PART : nullptr, 2ll * PART, in_group, ROWS,
                          groups > 1 ? base : nullptr, s, kvh, row0, bits, fsh);
        if (groups > 1) {
          __syncthreads();
          if (t == 0) {
            __threadfence();
            const bool last = atomicAdd(all_count, 1u) == (unsigned)groups - 1;
            __threadfence();
            if (last) *all_count = 0;
            sum_sh[2] = last;
          }
          __syncthreads();
          if (sum_sh[2]) {
            join_partials<HD>(a, a.part + (long long)slot_of(c_first) * PART, a.part + (long long)slot_of(c_first + kJoin) * PART,
                              2ll * kJoin * PART, groups, ROWS, nullptr, s, kvh, row0, bits, fsh);
          }
        }
      }
    }
    ubase += 2 * mine;
    at += count;
    if (at < end) {
      // The next part's positions come over what this one's partials took up.
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------------------ launch
// Whether the chunk kernel takes the call. Its blocks own 128 rows and walk their context alone, so its time
// is that walk (about 2.4 us a block of 128 positions at head_dim 256, and 10) times its rounds over the
// SMs; here the list is spread over all SMs but costs the more the more rows it has (about 45 us and
// 6.5 ns a tile of 16 positions x 32 rows). Both in us, from (B x new tokens of 8 heads over a
// context: chunk, here) 64 x 8 over 2,000: 56, 142; 64 x 3: 55, 84; 16 x 8: 51, 63; 1 x 8 over 8,000: 153, 54;
// 1 x 32: 155, 74; 8 x 32: 156, 234. Up to 16 rows the padding of a 128-row tile does not pay; f32 rows need
// products in parts, which only the kernel here carries.
static bool chunk_path(const PagedAttn &a) {
  const long long rows = (long long)a.max_q * a.group;
  if (a.type != G4_BF16 || rows <= 16) return false;
  const int hd = a.pool.hd, tokens = 128 / a.group;
  const double walk = hd == 512 ? 1.45 : (hd == 256 ? 1.0 : (hd == 128 ? 0.8 : 0.7));
  const double tile = hd == 512 ? 2.0 : (hd == 256 ? 1.0 : (hd == 128 ? 0.75 : 0.65));
  double span = a.max_kv;
  if (a.window > 0) span = std::min(span, (double)a.window + std::min(a.max_q, tokens));
  const long long heads = (long long)a.batch * a.pool.kv_heads;
  const long long blocks = heads * ((a.max_q + tokens - 1) / tokens) * (hd == 512 ? 2 : 1);
  const double chunk = (double)((blocks + 147) / 148) * (10.0 + 2.4 * walk * (span / 128 + 1));
  const double list = 45.0 + 0.0065 * tile * (double)(heads * ((rows + 31) / 32)) * (span / 16);
  return chunk < list;
}

// Row tiles per block: 1 for a group's 8 rows, up to 4 (each reads the positions again, from L1).
static int decode_rt(const PagedAttn &a) {
  const long long R = (long long)a.max_q * a.group;
  return R <= 8 ? 1 : (R <= 16 ? 2 : 4);
}

static_assert(4 * 148 * 4 <= kPagedCounters, "two counters a partial, two partials a block");

static void plan_decode(PagedAttn &a) {
  const int rt = decode_rt(a), rows = 8 * rt;
  a.row_groups = (int)(((long long)a.max_q * a.group + rows - 1) / rows);
  a.split_tiles = kLeastTiles * kDecWarps / rt;
  // (One context alone: no share holds a second beginning.)
  a.begin_tiles = (long long)a.batch * a.pool.kv_heads * a.row_groups == 1 ? 1 : kBeginTiles;
}

size_t paged_attention_partials(const PagedAttn &args) {
  PagedAttn a = args;
  if (a.max_q < 1 || a.batch < 1 || chunk_path(a)) return 0;
  return (size_t)2 * 148 * most_blocks(a.pool.hd) * (8 * decode_rt(a)) * (a.pool.hd + 2) * sizeof(float);
}

template <int FMT, int HD, int NP, int RT>
static cudaError_t launch_decode_rt(const PagedAttn &a, cudaStream_t st) {
  using S = DecShape<FMT, HD, NP, RT>;
  constexpr int SMEM = S::SMEM;
  static DeviceOnce once;
  cudaError_t e = cudaSuccess;
  once([&] { e = cudaFuncSetAttribute(k_paged_decode<FMT, HD, NP, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); });
  if (e != cudaSuccess) return e;
  // As many blocks as the SMs hold at once, or as there can be shares.
  long long span = a.max_kv;
  if (a.window > 0) span = std::min<long long>(span, (long long)a.window + (8 * RT + a.group - 1) / a.group + 16);
  const long long most = (long long)a.batch * a.pool.kv_heads * a.row_groups * std::max<long long>(1, (span + 15) / 16);
  const long long blocks = std::min<long long>((most + a.split_tiles - 1) / a.split_tiles, 148 * S::OCC);
  return launch_k(k_paged_decode<FMT, HD, NP, RT>, dim3((unsigned)blocks), dim3(kDecWarps * 32), SMEM, st, false, a);
}
template <int FMT, int HD, int NP>
static cudaError_t launch_decode_np(const PagedAttn &a, cudaStream_t st) {
  switch (decode_rt(a)) {
    case 1: return launch_decode_rt<FMT, HD, NP, 1>(a, st);
    case 2: return launch_decode_rt<FMT, HD, NP, 2>(a, st);
    default: return launch_decode_rt<FMT, HD, NP, 4>(a, st);
  }
}
template <int FMT, int HD>
static cudaError_t launch_decode_hd(const PagedAttn &a, cudaStream_t st) {
  if (a.type == G4_BF16) return launch_decode_np<FMT, HD, 1>(a, st);
  return launch_decode_np<FMT, HD, FMT == G4_PAGE_BF16 ? 3 : 2>(a, st);
}
template <int FMT>
static cudaError_t launch_decode(const PagedAttn &a, cudaStream_t st) {
  switch (a.pool.hd) {
    case 64: return launch_decode_hd<FMT, 64>(a, st);
    case 128: return launch_decode_hd<FMT, 128>(a, st);
    case 256: return launch_decode_hd<FMT, 256>(a, st);
    default: return launch_decode_hd<FMT, 512>(a, st);
  }
}

cudaError_t launch_paged_attention(const PagedAttn &args, cudaStream_t st) {
  PagedAttn a = args;
  if (chunk_path(a)) return launch_paged_chunk(a, st);
  plan_decode(a);
  switch (a.pool.fmt) {
    case G4_PAGE_BF16: return launch_decode<G4_PAGE_BF16>(a, st);
    case G4_PAGE_INT8: return launch_decode<G4_PAGE_INT8>(a, st);
    default: return launch_decode<G4_PAGE_E4M3>(a, st);
  }
}

}  // namespace g4
