// g4_drafts.cu -- verification of drafted tokens against the target model's probabilities.
//
// With x = logits / T a draft d stands when u w < p[d] = exp(x[d] - lse), lse = m + ln sum exp(x -
// m): one pass over the row gives m and the sum. The greatest x are counted and only the others summed:
// where one token has nearly all of p, ln p is -ln(1 + r) of a small r, and r keeps its digits. The token that follows is a race of exponential
// clocks, argmax(ln weight + gumbel): with a certain drafter the weights of a refused row are p
// without d, so ln weight is x itself up to a constant and the same pass over the row finds the
// winner; no second pass and no cumulative sums, whose rounding would decide the token. Only a
// drafter with probabilities needs the finished lse first (weights max(p - q, 0)): a second kernel
// reads that one row of each sequence again.
// Bound by HBM: the logits are read once.
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "g4_device.cuh"
#include "g4_kernels.cuh"
#include "g4_paged.cuh"

namespace g4 {

constexpr int kDraftThreads = 256;
constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Race {
  float key;
  int idx;
  // The greater key; the lower token on equal ones. A NaN key is never the greater one.
  __device__ __forceinline__ void add(float k, int i) {
    if (k > key || (k == key && i < idx)) {
      key = k;
      idx = i;
    }
  }
};

struct RowSum {
  float m, n, r;
  __device__ __forceinline__ void add(float om, float on, float orr) {
    if (om == m) {
      n += on;
      r += orr;
      return;
    }
    const bool up = om > m;
    const float hi = up ? om : m, lo = up ? m : om;
    // (A NaN on either side stays in the sum.)
    const float f = lo == -INFINITY ? 0.0f : ex2((lo - hi) * kLog2e);
    r = up ? fmaf(n + r, f, orr) : fmaf(on + orr, f, r);
    n = up ? on : n;
    m = hi;
  }
  // ln of the whole sum.
  __device__ __forceinline__ float ln() const { return n == 1.0f ? log1pf(r) : logf(n + r); }
};

constexpr DraftPart kNone = {-INFINITY, 0.0f, 0.0f, -INFINITY, 0x7fffffff, {0, 0, 0}};

__device__ __forceinline__ DraftPart warp_join(DraftPart v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, v.m, d), on = __shfl_xor_sync(0xffffffffu, v.n, d);
    const float orr = __shfl_xor_sync(0xffffffffu, v.r, d), ok = __shfl_xor_sync(0xffffffffu, v.key, d);
    const int oi = __shfl_xor_sync(0xffffffffu, v.idx, d);
    RowSum r{v.m, v.n, v.r};
    r.add(om, on, orr);
    Race c{v.key, v.idx};
    c.add(ok, oi);
    v = {r.m, r.n, r.r, c.key, c.idx, {0, 0, 0}};
  }
  return v;
}
// The block's sum; every thread of warp 0 receives it.
__device__ __forceinline__ DraftPart block_join(DraftPart v, DraftPart *sh) {
  v = warp_join(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = threadIdx.x < kDraftThreads / 32 ? sh[threadIdx.x] : kNone;
    v = warp_join(v);
  }
  return v;
}

template <typename T>
__device__ __forceinline__ float logit_at(const DraftArgs &a, long long row, int t) {
  const T *p = reinterpret_cast<const T *>(a.logits) + row * a.ld + t;
  if constexpr (sizeof(T) == 4)
    return *p;
  else
    return __bfloat162float(*p);
}

// Four consecutive elements at p: one load where p is aligned to them, else four.
template <typename T, bool WIDE>
__device__ __forceinline__ void load4(const T *p, float (&x)[4]) {
  if constexpr (!WIDE) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if constexpr (sizeof(T) == 4)
        x[e] = __ldg(p + e);
      else
        x[e] = __bfloat162float(p[e]);
    }
  } else if constexpr (sizeof(T) == 4) {
    const float4 v = __ldg(reinterpret_cast<const float4 *>(p));
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
    x[0] = __uint_as_float(v.x << 16);
    x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16);
    x[3] = __uint_as_float(v.y & 0xffff0000u);
  }
}
// Elements before the first one that is aligned to four.
template <typename T>
__device__ __forceinline__ int before4(const T *p) {
  return (int)((-(intptr_t)p & (4 * sizeof(T) - 1)) / sizeof(T));
}

struct SeqRows {
  int row, n;
};
__device__ __forceinline__ SeqRows seq_rows(const DraftArgs &a, int b, bool report) {
  const int b0 = a.row_begin[b], b1 = a.row_begin[b + 1];
  SeqRows s;
  s.row = min(max(b0, 0), a.rows);
  const int end = min(max(b1, s.row), a.rows);
  s.n = min(end - s.row, a.max_drafts + 1);
  if (report && (b0 < 0 || b1 < b0 || b1 > a.rows || end - s.row > s.n)) paged_raise(a.err, G4_PAGED_BAD_LENGTH);
  return s;
}

// What the scan leaves for the remainder's race: the row that emits (-1: done), its place, its greatest x
// and ln sum exp(x - m).
struct DraftState {
  int row, at;
  float m, ln;
};

// Block (split, j, b): split's share of sequence b's row j. The sequence's last block to finish
// joins the shares and decides. Shares begin where the row's logits are aligned to four, so these always
// come four a load; NW: so does the noise.
template <typename T, bool NW>
__global__ void __launch_bounds__(kDraftThreads) k_draft_scan(const DraftArgs a, DraftState *state) {
  const int b = blockIdx.z, j = blockIdx.y, split = blockIdx.x, t = threadIdx.x;
  const SeqRows sr = seq_rows(a, b, j == 0 && split == 0 && t == 0);
  const int width = a.max_drafts + 1;
  if (sr.n == 0) {
    if (j == 0 && split == 0) {
      for (int i = t; i < width; i += kDraftThreads) {
        a.tokens[(long long)b * width + i] = -1;
        a.logprobs[(long long)b * width + i] = 0.0f;
      }
      if (t == 0) {
        a.counts[b] = 0;
        state[b].row = -1;
      }
    }
    return;
  }
  if (j >= sr.n) return;
  __shared__ DraftPart sh[kDraftThreads / 32];
  __shared__ bool last_block;
  const float temp = a.temperature[b];
  const bool greedy = temp == 0.0f, final_row = j == sr.n - 1;
  const float inv = greedy ? 1.0f : __fdiv_rn(1.0f, temp);
  const long long row = sr.row + j;
  // A refused draft of a certain drafter is left out of its row's race; with probabilities the
  // race of a drafted row is the second kernel's.
  const int left_out = !greedy && !final_row && !a.probs ? a.drafts[row] : -1;
  const bool race = greedy || final_row || !a.probs, noisy = race && !greedy;
  const T *src = reinterpret_cast<const T *>(a.logits) + row * a.ld;
  const float *noise = a.gumbel + (long long)b * a.ld_gumbel;
  RowSum sum{-INFINITY, 0.0f, 0.0f};
  Race best{-INFINITY, 0x7fffffff};
  const int head = before4(src);   // tokens before the first share's first load
  const int c0 = split * a.chunk + head, c1 = min(a.vocab, c0 + a.chunk);
  constexpr int STEP = kDraftThreads * 4;
  // One pass of 16 tokens a thread, 32 where only the logits are read: the loads in flight. FULL: all of them are there and none is left out.
  auto pass = [&](auto full_, auto race_, auto noisy_, int i0) {
    constexpr bool FULL = decltype(full_)::value, RACE = decltype(race_)::value, NOISY = decltype(noisy_)::value;
    constexpr int U = NOISY ? 4 : 8;
    float x[U][4], g[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * STEP;
      if (FULL || i + 4 <= c1) {
        load4<T, true>(src + i, x[u]);
        if (NOISY) load4<float, NW>(noise + i, g[u]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[u][e] = i + e < c1 ? logit_at<T>(a, row, i + e) : -INFINITY;
          g[u][e] = NOISY && i + e < c1 ? noise[i + e] : 0.0f;
        }
      }
    }
    float top = sum.m;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        x[u][e] = __fmul_rn(x[u][e], inv);
        top = fmaxf(top, x[u][e]);
      }
    // (A row of nothing but -inf so far: ref 0, and every term is 0.)
    const float ref = top == -INFINITY ? 0.0f : top;
    float n = sum.n, s0 = sum.r, s1 = 0.0f;
    if (top != sum.m) {
      s0 = sum.m == -INFINITY ? s0 : (n + s0) * ex2((sum.m - ref) * kLog2e);
      n = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float p = ex2((x[u][e] - ref) * kLog2e);
        const bool is_top = x[u][e] == top;
        n += is_top ? 1.0f : 0.0f;
        (e & 1 ? s1 : s0) += is_top ? 0.0f : p;
        if (RACE) {
          const int i = i0 + u * STEP + e;
          const float key = NOISY ? __fadd_rn(x[u][e], g[u][e]) : x[u][e];
          if (key > best.key && (FULL || i != left_out)) best = {key, i};
        }
      }
    sum = {top, n, s0 + s1};
  };
  auto passes = [&](auto race_, auto noisy_) {
    if (split == 0 && t < head && t < a.vocab) {
      const float x = __fmul_rn(logit_at<T>(a, row, t), inv);
      const float key = decltype(noisy_)::value ? __fadd_rn(x, noise[t]) : x;
      // (A NaN makes the row's sum one, as in the passes.)
      sum = x != x ? RowSum{-INFINITY, 0.0f, x} : RowSum{x, 1.0f, 0.0f};
      if (decltype(race_)::value && key > best.key && t != left_out) best = {key, t};
    }
    constexpr int U = decltype(noisy_)::value ? 4 : 8;
    for (int b0 = c0; b0 < c1; b0 += STEP * U) {
      const int i0 = b0 + t * 4;
      if (b0 + STEP * U <= c1 && (left_out < b0 || left_out >= b0 + STEP * U))
        pass(std::true_type{}, race_, noisy_, i0);
      else
        pass(std::false_type{}, race_, noisy_, i0);
    }
  };
  if (noisy)
    passes(std::true_type{}, std::true_type{});
  else if (race)
    passes(std::true_type{}, std::false_type{});
  else
    passes(std::false_type{}, std::false_type{});
  DraftPart v = block_join({sum.m, sum.n, sum.r, best.key, best.idx, {0, 0, 0}}, sh);
  DraftPart *parts = a.part + ((long long)b * width + j) * a.splits;
  if (t == 0) {
    parts[split] = v;
    __threadfence();
    last_block = atomicAdd(a.count + b, 1u) == (unsigned)(sr.n * a.splits) - 1;
  }
  __syncthreads();
  if (!last_block) return;
  __threadfence();

  // Every row's sums, one warp a row; then the first draft that does not stand.
  __shared__ float row_m[kMaxDrafts + 1], row_ln[kMaxDrafts + 1], lp[kMaxDrafts + 1];
  __shared__ int chosen[kMaxDrafts + 1];
  __shared__ bool stands[kMaxDrafts + 1];
  const int warp = t >> 5, lane = t & 31;
  for (int r = warp; r < sr.n; r += kDraftThreads / 32) {
    const DraftPart *rp = a.part + ((long long)b * width + r) * a.splits;
    DraftPart w = kNone;
    for (int s = lane; s < a.splits; s += 32) {
      const float4 f = __ldcg(reinterpret_cast<const float4 *>(rp + s));
      RowSum rs{w.m, w.n, w.r};
      rs.add(f.x, f.y, f.z);
      Race c{w.key, w.idx};
      c.add(f.w, __ldcg(&rp[s].idx));
      w = {rs.m, rs.n, rs.r, c.key, c.idx, {0, 0, 0}};
    }
    w = warp_join(w);
    if (lane == 0) {
      const float ln = RowSum{w.m, w.n, w.r}.ln();
      const int pick = w.idx == 0x7fffffff ? 0 : w.idx;
      bool ok = false;
      float lpd = 0.0f;
      if (r < sr.n - 1) {
        const int d = a.drafts[sr.row + r];
        if (d >= 0 && d < a.vocab) {
          lpd = (__fmul_rn(logit_at<T>(a, sr.row + r, d), inv) - w.m) - ln;
          if (greedy) {
            ok = d == pick;
          } else {
            const float q = a.probs ? a.probs[(sr.row + r) * a.ld_probs + d] : 1.0f;
            ok = __fmul_rn(a.uniforms[sr.row + r], q) < expf(lpd);
          }
        }
      }
      stands[r] = ok;
      chosen[r] = pick;
      lp[r] = lpd;
      row_m[r] = w.m;
      row_ln[r] = ln;
      // ln p of the row's winner, for the row that emits it.
      if (!ok) lp[r] = (__fmul_rn(logit_at<T>(a, sr.row + r, pick), inv) - w.m) - ln;
    }
  }
  __syncthreads();
  __shared__ int stop;
  if (t == 0) {
    int r = 0;
    while (r < sr.n - 1 && stands[r]) r++;
    stop = r;
    a.count[b] = 0;
    a.counts[b] = r + 1;
    const bool rest = a.probs && !greedy && r < sr.n - 1;
    state[b] = {rest ? sr.row + r : -1, r, row_m[r], row_ln[r]};
  }
  __syncthreads();
  for (int i = t; i < width; i += kDraftThreads) {
    a.tokens[(long long)b * width + i] = i < stop ? a.drafts[sr.row + i] : (i == stop ? chosen[i] : -1);
    a.logprobs[(long long)b * width + i] = i <= stop ? lp[i] : 0.0f;
  }
}

// The remainder's race over the refused row of each sequence whose drafter gave probabilities:
// ln max(p - q, 0) + gumbel, and x + gumbel for the case that no remainder is left.
template <typename T, bool NW>
__global__ void __launch_bounds__(kDraftThreads) k_draft_rest(const DraftArgs a, const DraftState *state) {
  const int b = blockIdx.y, split = blockIdx.x, t = threadIdx.x;
  const DraftState st = state[b];
  if (st.row < 0) return;
  __shared__ DraftPart sh[kDraftThreads / 32];
  __shared__ bool last_block;
  const float temp = a.temperature[b], inv = __fdiv_rn(1.0f, temp);
  const T *src = reinterpret_cast<const T *>(a.logits) + (long long)st.row * a.ld;
  const float *noise = a.gumbel + (long long)b * a.ld_gumbel;
  const float *probs = a.probs + (long long)st.row * a.ld_probs;
  Race rest{-INFINITY, 0x7fffffff}, plain{-INFINITY, 0x7fffffff};
  const int head = before4(src), c0 = split * a.chunk + head, c1 = min(a.vocab, c0 + a.chunk);
  float bar = -INFINITY;   // a key of this warp's: what is below it is out
  auto race = [&](int i, float x, float g, float q) {
    const float xs = __fmul_rn(x, inv), lp = __fsub_rn(__fsub_rn(xs, st.m), st.ln), key = __fadd_rn(xs, g);
    if (key > plain.key) plain = {key, i};
    // What is left is at most p, so ln left + gumbel at most ln p + gumbel (and 1e-3 covers what the
    // functions' rounding adds): nearly every token is out of the race without either function.
    if (__fadd_rn(lp, g) + fmaf(fabsf(xs), 1e-6f, 1e-3f) > bar) {
      const float left = __fsub_rn(expf(lp), q);
      if (left > 0.0f) {
        const float k = __fadd_rn(logf(left), g);
        if (k > rest.key) rest = {k, i};
      }
    }
  };
  if (split == 0 && t < head && t < a.vocab) race(t, logit_at<T>(a, st.row, t), noise[t], probs[t]);
  constexpr int U = 2, STEP = kDraftThreads * 4;
  for (int b0 = c0; b0 < c1; b0 += STEP * U) {
    const int i0 = b0 + t * 4;
    float x[U][4], g[U][4], q[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = i0 + u * STEP;
      if (i + 4 <= c1) {
        load4<T, true>(src + i, x[u]);
        load4<float, NW>(noise + i, g[u]);
        load4<float, NW>(probs + i, q[u]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const bool in = i + e < c1;
          x[u][e] = in ? logit_at<T>(a, st.row, i + e) : -INFINITY;
          g[u][e] = in ? noise[i + e] : 0.0f;
          q[u][e] = in ? probs[i + e] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        race(i0 + u * STEP + e, x[u][e], g[u][e], q[u][e]);
        if (e == 0) {
          bar = rest.key;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) bar = fmaxf(bar, __shfl_xor_sync(0xffffffffu, bar, d));
        }
      }
  }
  const DraftPart r = block_join({-INFINITY, 0.0f, 0.0f, rest.key, rest.idx, {0, 0, 0}}, sh);
  __syncthreads();
  const DraftPart p = block_join({-INFINITY, 0.0f, 0.0f, plain.key, plain.idx, {0, 0, 0}}, sh);
  DraftPart *parts = a.part + (long long)b * a.splits;
  if (t == 0) {
    parts[split] = {p.key, __int_as_float(p.idx), r.key, __int_as_float(r.idx), 0, {0, 0, 0}};
    __threadfence();
    last_block = atomicAdd(a.count + b, 1u) == (unsigned)a.splits - 1;
  }
  __syncthreads();
  if (!last_block || t >= 32) return;
  __threadfence();
  rest = {-INFINITY, 0x7fffffff};
  plain = {-INFINITY, 0x7fffffff};
  for (int s = t; s < a.splits; s += 32) {
    const float4 f = __ldcg(reinterpret_cast<const float4 *>(parts + s));
    plain.add(f.x, __float_as_int(f.y));
    rest.add(f.z, __float_as_int(f.w));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float rk = __shfl_xor_sync(0xffffffffu, rest.key, d), pk = __shfl_xor_sync(0xffffffffu, plain.key, d);
    const int ri = __shfl_xor_sync(0xffffffffu, rest.idx, d), pi = __shfl_xor_sync(0xffffffffu, plain.idx, d);
    rest.add(rk, ri);
    plain.add(pk, pi);
  }
  if (t == 0) {
    const int pick = rest.idx != 0x7fffffff ? rest.idx : (plain.idx != 0x7fffffff ? plain.idx : 0);
    const long long at = (long long)b * (a.max_drafts + 1) + st.at;
    a.count[b] = 0;
    a.tokens[at] = pick;
    a.logprobs[at] = __fsub_rn(__fsub_rn(__fmul_rn(logit_at<T>(a, st.row, pick), inv), st.m), st.ln);
  }
}

// Tokens a block scans: as many as let `rows` rows fill the SMs once (4 blocks each; a block costs a few
// microseconds besides its loads: 144 rows of 262,144 took 29 us in one round, 34 and 40 in two and
// four), at least 2048, in steps of 1024.
static int draft_chunk(int vocab, int rows) {
  const int splits = std::max(1, 4 * 148 / std::max(rows, 1));
  return std::max(2048, ((vocab + splits - 1) / splits + 1023) / 1024 * 1024);
}

// Few sequences have such a row, so its shares are small: one pass of a block.
constexpr int kRestChunk = 2048;

size_t verify_drafts_partials(int vocab, int rows, int batch, int max_drafts) {
  const int chunk = draft_chunk(vocab, rows), splits = (vocab + chunk - 1) / chunk;
  const int rest_splits = (vocab + kRestChunk - 1) / kRestChunk;
  const size_t scan = (size_t)(max_drafts + 1) * splits;
  return (size_t)batch * std::max(scan, (size_t)rest_splits) * sizeof(DraftPart) + (size_t)batch * sizeof(DraftState);
}

template <typename T, bool NW>
static cudaError_t launch_drafts(const DraftArgs &a, DraftState *state, cudaStream_t st) {
  const dim3 block(kDraftThreads);
  cudaError_t e = launch_k(k_draft_scan<T, NW>, dim3(a.splits, a.max_drafts + 1, a.batch), block, 0, st, false, a, state);
  if (e == cudaSuccess && a.probs) {
    DraftArgs r = a;   // one row a sequence at most: shares of its own size
    r.chunk = kRestChunk;
    r.splits = (a.vocab + r.chunk - 1) / r.chunk;
    e = launch_k(k_draft_rest<T, NW>, dim3(r.splits, a.batch), block, 0, st, false, r, state);
  }
  return e;
}

cudaError_t launch_verify_drafts(const DraftArgs &args, cudaStream_t st) {
  DraftArgs a = args;
  a.chunk = draft_chunk(a.vocab, a.rows);
  a.splits = (a.vocab + a.chunk - 1) / a.chunk;
  DraftState *state = reinterpret_cast<DraftState *>(
      (char *)a.part + verify_drafts_partials(a.vocab, a.rows, a.batch, a.max_drafts) - (size_t)a.batch * sizeof(DraftState));
  // Noise and probabilities come four a load where they lie in step with the logits: every row of all of
  // them on its boundary.
  const uintptr_t at = (uintptr_t)a.gumbel | (a.probs ? (uintptr_t)a.probs : 0);
  const bool wide = a.ld % 4 == 0 && a.ld_gumbel % 4 == 0 && (!a.probs || a.ld_probs % 4 == 0) && !(at & 15) &&
                    !((uintptr_t)a.logits & (a.type == G4_F32 ? 15 : 7));
  if (a.type == G4_F32) return wide ? launch_drafts<float, true>(a, state, st) : launch_drafts<float, false>(a, state, st);
  return wide ? launch_drafts<__nv_bfloat16, true>(a, state, st) : launch_drafts<__nv_bfloat16, false>(a, state, st);
}

}  // namespace g4
