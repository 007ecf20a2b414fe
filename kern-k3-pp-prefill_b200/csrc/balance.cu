// The router's training side: the load-balance loss with its per-sequence expert counts, and the gradient of the
// router logits (from the loss and from the combine weights of the top-k).
//
// With s = sigmoid(S) (the top-k's scores), z_t = sum_e s_te + 1e-20 and p_te = s_te / z_t, over the counted rows
// of sequence b (inside [seq[b], seq[b+1]) and not masked out): n_b rows, c_be picks of expert e, P_be = sum p_te,
//   loss = alpha / B' * sum_b sum_e (E c_be / (K n_b)) (P_be / n_b),    B' = sequences with a counted row.
// The counts are constants of the gradient, so with f_be = alpha dloss E c_be / (B' K n_b^2)
//   dS_te += (f_be - sum_j f_bj p_tj) s_te (1 - s_te) / z_t,
// and from the weights w_k = rs s_k / den, den = sum_k s_k + 1e-20, of a row's picks
//   dS_{t, idx_k} += rs / den (g_k - sum_j g_j s_j / den) s_k (1 - s_k),    g = dloss/dw.
// No counterpart in the reference: it serves only.
//
// Measured on a B200, 8192 x 896 logits, top-8, 16 sequences: loss and counts 17.2 us (11.8 us at 2048 rows, 5 of them the
// join; 22 MB more cost 5 us; reading them takes 3.4), gradient of both terms 16.9 us into one buffer, 19-21 us into a new
// one a call (4 us a round of 16 rows an SM behind 6 us of prologue and first rows; a copy of the same 59 MB takes 10.3 us),
// of the weight term alone 10.0 us.
// Both passes read S once.  Sums run in a fixed order (no floating-point atomics), so equal inputs give equal
// bytes.  A score is 1 / (1 + exp(-S)) by one exponential and one reciprocal instruction, the rounding of the exponential's
// argument put right: within 2^-20 of itself from S = -87 on, 0 further down.
#pragma once
#include "common.cuh"

namespace k3 {

namespace bal {
constexpr int JOIN_WARPS = 32;   // of a block of the join, at most
constexpr int JOIN_BLOCKS = 8 * 148;
constexpr int ROW_WARPS = 16;    // of a block that walks rows
constexpr int FLUSH = 256;       // rows a warp sums in f32
constexpr int PICKS = 16;        // K at most
// Row slots a warp: as many as fit, four at most.  One block an SM where a row is long, two where it is short.
__host__ __device__ constexpr int slots(int nv) { return nv <= 5 ? 4 : nv <= 7 ? 3 : 2; }
__host__ __device__ constexpr int blocks_per_sm(int nv) { return nv <= 2 ? 2 : 1; }
__host__ __device__ constexpr int slot_floats(int nv) { return 128 * nv + 2 * PICKS; }
__host__ __device__ constexpr int ring_bytes(int nv) { return ROW_WARPS * slots(nv) * slot_floats(nv) * 4; }
__host__ __device__ constexpr int rows_smem(int nv) {
  return ring_bytes(nv) + (ROW_WARPS / 2) * 128 * nv * 4 + 128 * nv * 8 + 128 * nv * 4;
}
__host__ __device__ constexpr int grad_smem(int nv) { return ring_bytes(nv) + 2 * 128 * nv * 4; }
constexpr float TINY = 1e-20f;  // the top-k's guard of its own sum
constexpr int COLS = 32;        // experts a block of the second pass
constexpr int WIDE = 16;        // partial rows that a lone warp adds up, at most
}  // namespace bal

struct RouterRows {
  const float* S;          // [T, lds]
  long long lds;
  const int* idx;          // [T, K]
  const int* seq;          // [B + 1] or null: one sequence of all T rows
  const uint8_t* mask;     // [T] or null
  int T, E, K, B;
  int vec;                 // S rows may be read 16 bytes at a time
};

// A warp's finder of sequences: up to 128 offsets stay in its registers, four a lane, so that a row's sequence is a count
// of the offsets up to it; of more, a binary search, which neighbouring rows of one sequence share.
struct SeqFinder {
  const int* seq;
  int B, lo, hi;       // rows outside [lo, hi) lie in none
  int mine[4];
  int b, end;          // the last answer, good up to row `end`
  __device__ __forceinline__ void init(const RouterRows& in, int lane) {
    seq = in.seq;
    B = in.B;
    lo = 0;
    hi = in.T;
    b = -1;
    end = -1;
    if (seq == nullptr) return;
    lo = max(seq[0], 0);
    hi = min(seq[B], in.T);
#pragma unroll
    for (int i = 0; i < 4; ++i) mine[i] = i * 32 + lane < B && B <= 128 ? seq[i * 32 + lane] : 0x7fffffff;
  }
  // the sequence of row t, the last b with seq[b] <= t, or -1; every lane of the warp asks for the same row
  __device__ __forceinline__ int operator()(int t) {
    if (t < lo || t >= hi) return -1;
    if (seq == nullptr) return 0;
    if (B <= 128) {
      int n = __popc(__ballot_sync(0xffffffffu, mine[0] <= t));
      if (B > 32) {
#pragma unroll
        for (int i = 1; i < 4; ++i) n += __popc(__ballot_sync(0xffffffffu, mine[i] <= t));
      }
      return max(n - 1, 0);
    }
    if (b >= 0 && t >= seq[b] && t < end) return b;
    if (b >= 0 && b + 2 <= B && t >= end && t < seq[b + 2]) {
      ++b;  // the next one: sequences are short and follow one another
    } else {
      int x = 0, y = B - 1;
      while (x < y) {
        const int m = (x + y + 1) >> 1;
        if (seq[m] <= t) x = m;
        else y = m - 1;
      }
      b = x;
    }
    end = seq[b + 1];
    return b;
  }
};

// A row on its way through shared memory: the logits, the picks, the gradients of their weights.  Each warp keeps a few
// rows in flight by cp.async, which takes no registers and leaves nothing to spin on.  A lane's experts are 4 consecutive
// ones in each group of 128, (j * 32 + lane) * 4 + i, and it copies what it will read; experts past E stay at -inf.
template <int NV>
struct RowRing {
  float* base;
  int lane;
  __device__ __forceinline__ float* slot(int i) const { return base + (i % bal::slots(NV)) * bal::slot_floats(NV); }
  __device__ __forceinline__ void init(float* smem, int warp, int lane_, int E) {
    lane = lane_;
    base = smem + warp * bal::slots(NV) * bal::slot_floats(NV);
    for (int s = 0; s < bal::slots(NV); ++s)
      for (int c = E / 4 * 4 + lane; c < 128 * NV; c += 32) slot(s)[c] = -INFINITY;
    __syncwarp();
  }
  // start row t's copy into slot i (t < 0: an empty group, so that the groups count up with the rows)
  __device__ __forceinline__ void fetch(const RouterRows& in, int i, int t, bool logits, bool picks, const float* dwts) {
    if (t >= 0) {
      float* d = slot(i);
      const u32 s = smem_u32(d);
      const float* row = in.S + t * in.lds;
      if (logits) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int c = (j * 32 + lane) * 4;
          if (in.vec && c + 4 <= in.E) {
            cp_async16(s + c * 4, row + c);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (c + k < in.E) cp_async4(s + (c + k) * 4, row + c + k);
          }
        }
      }
      if (picks && lane < in.K) {
        cp_async4(s + (128 * NV + lane) * 4, in.idx + (long long)t * in.K + lane);
        if (dwts) cp_async4(s + (128 * NV + bal::PICKS + lane) * 4, dwts + (long long)t * in.K + lane);
      }
    }
    cp_async_commit();
  }
  // wait until the oldest of the copies in flight is there (slots - 1 younger ones may be on their way)
  __device__ __forceinline__ void wait() const {
    cp_async_wait_group<bal::slots(NV) - 1>();
    __syncwarp();
  }
};

// With e = exp(-x) the score is 1 / (1 + e) and its slope e / (1 + e)^2, without cancellation at either end; two at a time,
// four multifunction instructions a pair.  The exponential's argument is put right but for ln 2's low part (with it the
// gradient of 65536 x 896 logits takes 103 us, without 92.7, with the argument left as rounded 90.4).  Logits are clamped to +-FAR for it (NaN stays): from there on the score is 1 with
// slope 0, or below the smallest normal f32 and 0, infinities among them.
constexpr float FAR = 88.f;
__device__ __forceinline__ float clamp_logit(float x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-FAR));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(FAR));
  return x;
}
__device__ __forceinline__ u64 exp_neg2(u64 x) {
  const float2 v = f32x2_get(x);
  return exp_f32x2<false>(f32x2(-clamp_logit(v.x), -clamp_logit(v.y)));
}
__device__ __forceinline__ u64 score2(u64 e) {
  const float2 v = f32x2_get(add_f32x2(e, f32x2(1.f, 1.f)));
  return f32x2(rcp_ftz(v.x), rcp_ftz(v.y));
}
__device__ __forceinline__ u64 slope2(u64 score, u64 e) { return mul_f32x2(mul_f32x2(e, score), score); }
// 1 / x of a sum: the instruction and one step of Newton's iteration
__device__ __forceinline__ float reciprocal(float x) {
  const float r = rcp_ftz(x);
  return __fmaf_rn(r, __fmaf_rn(-x, r, 1.f), r);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// the sums of N values each over the warp, side by side
template <int N>
__device__ __forceinline__ void warp_sums(float (&v)[N]) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
}

// ---------------------------------------------------------------- forward
// First pass: a block takes `chunk` consecutive rows, a warp every sixteenth of them, each lane summing its experts' p in
// registers.  At the end of a sequence, or of the block's rows, the warps' sums are added in order and stored as one
// partial row; where a sequence goes on for longer, every 16 * FLUSH rows they go into a sum in double, so that no f32 sum
// has more than FLUSH rows however many there are (one sum over the 14000 rows a warp takes of 64 million was off by
// 1e-4; up to 600 thousand rows nothing is flushed).  Block i and sequence b meet in slot i + b: along the rows either i or
// b goes up, so no two pairs share a slot and nothing needs zeroing.
struct BalanceScratch {
  float* prob;   // [slots, E]
  int* count;    // [slots, E]
  int* rows;     // [slots]
  float2* term;  // [blocks of the second pass]: sum of terms, sequences with a counted row
  u32* done;
};

// Second pass: a team (a warp, where few of the first pass's blocks meet the average sequence, or a block) adds up 32
// experts of one sequence over the blocks that met it, its warps side by side and joined in order, then the next such group
// of its share; the last block of all adds up the loss.  A warp that meets a long sequence among short or empty ones (a
// batch padded to a fixed number of offsets) leaves it to its whole block; the groups of a sequence go to blocks in turn, so
// that a block has one of them.
struct BalanceOut {
  float alpha;
  int* counts;   // [B, E]
  float* prob;   // [B, E]
  int* rows;     // [B]
  float* loss;
};
template <bool WARP_TEAM>
__global__ void __launch_bounds__(32 * bal::JOIN_WARPS)
    balance_join_kernel(RouterRows in, BalanceScratch w, int chunk, BalanceOut out) {
  using namespace bal;
  __shared__ float s_p[JOIN_WARPS][COLS];
  __shared__ int s_c[JOIN_WARPS][COLS], s_n[JOIN_WARPS];
  __shared__ int s_wide[WARP_TEAM ? JOIN_WARPS : 1][4];  // i0, i1 (-1: not wide), sequence and group of a warp's unit
  __shared__ int s_last;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = (in.E + COLS - 1) / COLS;
  const int lo = in.seq ? max(in.seq[0], 0) : 0, hi = in.seq ? min(in.seq[in.B], in.T) : in.T;
  const long long units = (long long)in.B * groups, turn = (long long)gridDim.x * (WARP_TEAM ? warps : 1);
  float terms = 0.f;
  int full = 0;  // sequences with a counted row
  bool waited = false;
  for (long long base = 0; base + blockIdx.x < units; base += turn) {
    const long long unit = base + blockIdx.x + (WARP_TEAM ? (long long)gridDim.x * warp : 0);
    const bool mine = !WARP_TEAM || unit < units;
    const int b = mine ? (int)(unit / groups) : 0, g = (int)(unit % groups), e = g * COLS + lane;
    const int s0 = in.seq ? max(lo, in.seq[b]) : lo, s1 = in.seq ? min(hi, in.seq[b + 1]) : hi;
    // the first pass's blocks that met the sequence
    const int i0 = s0 / chunk, i1 = mine && s0 < s1 ? (s1 - 1) / chunk : -1;
    const bool wide = !WARP_TEAM || i1 - i0 >= WIDE;
    // its partial rows (the first pass lets this one start after its own wait: the offsets are there before)
    if (!waited) grid_wait_previous();
    waited = true;
    float p = 0.f;
    int c = 0, n = 0;
    if (!WARP_TEAM || !wide) {
#pragma unroll 5
      for (int i = i0 + (WARP_TEAM ? 0 : warp); i <= i1; i += WARP_TEAM ? 1 : warps) {
        const long long slot = (long long)i + b;
        if (e < in.E) {
          p += w.prob[slot * in.E + e];
          c += w.count[slot * in.E + e];
        }
        n += w.rows[slot];
      }
    }
    if (!WARP_TEAM) {
      __syncthreads();  // the group before has been read
      s_p[warp][lane] = p;
      s_c[warp][lane] = c;
      if (lane == 0) s_n[warp] = n;
      __syncthreads();
      for (int k = 1; warp == 0 && k < warps; ++k) {
        p += s_p[k][lane];
        c += s_c[k][lane];
        n += s_n[k];
      }
    } else if (__syncthreads_or(wide)) {
      if (lane == 0) {
        s_wide[warp][0] = wide ? i0 : 0;
        s_wide[warp][1] = wide ? i1 : -1;
        s_wide[warp][2] = b;
        s_wide[warp][3] = g;
      }
      __syncthreads();
      for (int k = 0; k < warps; ++k) {
        const int j1 = s_wide[k][1], bk = s_wide[k][2], ek = s_wide[k][3] * COLS + lane;
        if (j1 < 0) continue;
        float pk = 0.f;
        int ck = 0, nk = 0;
#pragma unroll 5
        for (int i = s_wide[k][0] + warp; i <= j1; i += warps) {
          const long long slot = (long long)i + bk;
          if (ek < in.E) {
            pk += w.prob[slot * in.E + ek];
            ck += w.count[slot * in.E + ek];
          }
          nk += w.rows[slot];
        }
        s_p[warp][lane] = pk;
        s_c[warp][lane] = ck;
        if (lane == 0) s_n[warp] = nk;
        __syncthreads();
        for (int j = 0; warp == k && j < warps; ++j) {
          p += s_p[j][lane];
          c += s_c[j][lane];
          n += s_n[j];
        }
        __syncthreads();
      }
    }
    if (WARP_TEAM ? mine : warp == 0) {
      float term = 0.f;
      if (e < in.E) {
        out.counts[(long long)b * in.E + e] = c;
        out.prob[(long long)b * in.E + e] = p;
        if (n > 0) term = ((float)in.E * (float)c / ((float)in.K * (float)n)) * (p / (float)n);
      }
      terms += term;
      if (g == 0) {
        full += n > 0;
        if (lane == 0) out.rows[b] = n;
      }
    }
  }
  if (!waited) grid_wait_previous();
  terms = warp_sum(terms);
  __syncthreads();
  if (lane == 0) {
    s_p[warp][0] = terms;
    s_c[warp][0] = full;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < warps; ++k) {
      terms += s_p[k][0];
      full += s_c[k][0];
    }
    w.term[blockIdx.x] = make_float2(terms, __int_as_float(full));
    // releases this thread's store above and acquires those of the blocks that counted before
    u32 before;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(w.done) : "memory");
    s_last = before == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  terms = 0.f;
  full = 0;
  for (int i = threadIdx.x; i < gridDim.x; i += blockDim.x) {
    const float2 t = __ldcg(&w.term[i]);
    terms += t.x;
    full += __float_as_int(t.y);
  }
  terms = warp_sum(terms);
  full = __reduce_add_sync(0xffffffffu, full);
  if (lane == 0) {
    s_p[warp][1] = terms;
    s_c[warp][1] = full;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < warps; ++k) {
      terms += s_p[k][1];
      full += s_c[k][1];
    }
    *out.loss = out.alpha * terms / (float)max(full, 1);
  }
}

template <int NV>
__global__ void __launch_bounds__(32 * bal::ROW_WARPS, bal::blocks_per_sm(NV))
    balance_rows_kernel(RouterRows in, BalanceScratch w, int chunk) {
  using namespace bal;
  constexpr int N = 2 * NV;  // pairs of experts a lane
  extern __shared__ __align__(16) float ring_smem[];
  float* s_acc = ring_smem + ring_bytes(NV) / 4;                                 // [ROW_WARPS / 2][128 NV]
  double* s_long = reinterpret_cast<double*>(s_acc + ROW_WARPS / 2 * 128 * NV);  // [128 NV]
  int* s_hist = reinterpret_cast<int*>(s_long + 128 * NV);                       // [128 NV]
  __shared__ int s_rows[ROW_WARPS];
  grid_wait_previous();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r0 = blockIdx.x * chunk, r1 = min(in.T, r0 + chunk);
  if (blockIdx.x == 0 && threadIdx.x == 0) *w.done = 0u;
  RowRing<NV> ring;
  ring.init(ring_smem, warp, lane, in.E);
  int t = r0 + warp, at = 0;  // the warp's next row, in slot `at`
  auto ahead = [&](int i) {
    const int u = t + i * ROW_WARPS;
    return u < r1 ? u : -1;
  };
  for (int i = 0; i < slots(NV) - 1; ++i) ring.fetch(in, i, ahead(i), true, true, nullptr);
  SeqFinder find;
  find.init(in, lane);
  int r = max(r0, find.lo);
  const int last = min(r1, find.hi);
  while (r < last) {
    const int b = find(r), end = in.seq ? min(last, in.seq[b + 1]) : last;
    if (end <= r) break;  // offsets that go down: nothing more is counted
    int n = 0;
    for (int e = threadIdx.x; e < in.E; e += 32 * ROW_WARPS) s_hist[e] = 0;
    __syncthreads();
    for (int from = r, stop; from < end; from = stop) {
      stop = min(end, from + ROW_WARPS * FLUSH);
      u64 acc[N];
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = f32x2(0.f, 0.f);
      for (; t < stop; t += ROW_WARPS, ++at) {
        ring.fetch(in, at + slots(NV) - 1, ahead(slots(NV) - 1), true, true, nullptr);
        ring.wait();
        if (t < r || (in.mask && in.mask[t] == 0)) continue;
        ++n;
        const float* row = ring.slot(at);
        u64 z2 = f32x2(0.f, 0.f), s[N];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(row + (j * 32 + lane) * 4);
          s[2 * j] = score2(exp_neg2(v.x));
          s[2 * j + 1] = score2(exp_neg2(v.y));
          z2 = add_f32x2(z2, add_f32x2(s[2 * j], s[2 * j + 1]));
        }
        const float2 z = f32x2_get(z2);
        if (lane < in.K) {
          const int e = reinterpret_cast<const int*>(row + 128 * NV)[lane];
          if (e >= 0 && e < in.E) atomicAdd(&s_hist[e], 1);
        }
        const float inv = reciprocal(warp_sum(z.x + z.y) + TINY);
        const u64 inv2 = f32x2(inv, inv);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fma_f32x2(s[i], inv2, acc[i]);
        __syncwarp();  // every lane has read the slot that the next fetch fills
      }
      // the upper half of the warps, then the lower half onto them
      float* mine = s_acc + warp % (ROW_WARPS / 2) * 128 * NV;
      if (warp >= ROW_WARPS / 2) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          *reinterpret_cast<ulonglong2*>(mine + (j * 32 + lane) * 4) = make_ulonglong2(acc[2 * j], acc[2 * j + 1]);
      }
      if (lane == 0) s_rows[warp] = n;
      __syncthreads();
      if (warp < ROW_WARPS / 2) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          ulonglong2* q = reinterpret_cast<ulonglong2*>(mine + (j * 32 + lane) * 4);
          const ulonglong2 o = *q;
          *q = make_ulonglong2(add_f32x2(o.x, acc[2 * j]), add_f32x2(o.y, acc[2 * j + 1]));
        }
      }
      __syncthreads();
      const long long slot = (long long)blockIdx.x + b;
      for (int e = threadIdx.x; e < in.E; e += 32 * ROW_WARPS) {
        float p = 0.f;
#pragma unroll
        for (int k = 0; k < ROW_WARPS / 2; ++k) p += s_acc[k * 128 * NV + e];
        if (from > r || stop < end) {
          const double sum = (from > r ? s_long[e] : 0.0) + p;
          s_long[e] = sum;
          p = (float)sum;
        }
        if (stop < end) continue;
        w.prob[slot * in.E + e] = p;
        w.count[slot * in.E + e] = s_hist[e];
      }
      if (stop == end && threadIdx.x == 0) {
        int total = 0;
        for (int k = 0; k < ROW_WARPS; ++k) total += s_rows[k];
        w.rows[slot] = total;
      }
      __syncthreads();
    }
    r = end;
  }
  cp_async_wait_all();
}

// ---------------------------------------------------------------- backward
struct RouteBackward {
  float alpha;
  const int* counts;    // [B, E] or null: no balance term
  const int* rows;      // [B]
  const float* dloss;   // [1] or null (1)
  const float* dwts;    // [T, K] or null: no weight term
  const bf16* rs;       // [1]
  void* dS;             // [T, ldd] f32 or bf16
  long long ldd;
  int bf16_out;
  int vec_out;          // rows may be stored 4 elements at a time
};

// A block takes consecutive rows, a warp every sixteenth.  The coefficients f of the sequences that the block's first and
// last rows are in lie in shared memory; rows of others, where sequences are short, read their counts.  The weight term
// touches K experts of a row: the lanes that hold the picks store those elements' sums after the row.
template <int NV>
__global__ void __launch_bounds__(32 * bal::ROW_WARPS, bal::blocks_per_sm(NV))
    route_backward_kernel(RouterRows in, RouteBackward q, int chunk) {
  using namespace bal;
  constexpr int N = 2 * NV;  // pairs of experts a lane
  constexpr int PER = (128 * NV + 32 * ROW_WARPS - 1) / (32 * ROW_WARPS);
  extern __shared__ __align__(16) float ring_smem[];
  float* s_f = ring_smem + ring_bytes(NV) / 4;  // [2][128 NV]
  __shared__ int s_full[ROW_WARPS];
  grid_wait_previous();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r0 = blockIdx.x * chunk, r1 = min(in.T, r0 + chunk);
  RowRing<NV> ring;
  ring.init(ring_smem, warp, lane, in.E);
  int t = r0 + warp, at = 0;
  const bool balance = q.counts != nullptr, weights = q.dwts != nullptr;
  auto ahead = [&](int i) {
    const int u = t + i * ROW_WARPS;
    return u < r1 ? u : -1;
  };
  for (int i = 0; i < slots(NV) - 1; ++i) ring.fetch(in, i, ahead(i), balance, weights, q.dwts);
  SeqFinder find;
  find.init(in, lane);
  int b0 = -1, b1 = -1;
  float scale = 0.f;  // alpha dloss E / (B' K)
  if (balance) {
    int full = 0;
    for (int i = threadIdx.x; i < in.B; i += 32 * ROW_WARPS) full += q.rows[i] > 0;
    const float dloss = q.dloss ? *q.dloss : 1.0f;
    b0 = find(r0);
    b1 = find(r1 - 1);
    int c0[PER], c1[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * 32 * ROW_WARPS + threadIdx.x;
      c0[i] = b0 >= 0 && e < in.E ? q.counts[(long long)b0 * in.E + e] : 0;
      c1[i] = b1 >= 0 && e < in.E ? q.counts[(long long)b1 * in.E + e] : 0;
    }
    const int n0 = b0 >= 0 ? q.rows[b0] : 0, n1 = b1 >= 0 ? q.rows[b1] : 0;
    full = __reduce_add_sync(0xffffffffu, full);
    if (lane == 0) s_full[warp] = full;
    __syncthreads();
    full = 0;
    for (int k = 0; k < ROW_WARPS; ++k) full += s_full[k];
    scale = q.alpha * dloss * ((float)in.E / ((float)max(full, 1) * (float)in.K));
    const float k0 = n0 > 0 ? scale / (float)n0 / (float)n0 : 0.f, k1 = n1 > 0 ? scale / (float)n1 / (float)n1 : 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * 32 * ROW_WARPS + threadIdx.x;
      if (e < 128 * NV) {
        s_f[e] = k0 * (float)c0[i];
        s_f[128 * NV + e] = k1 * (float)c1[i];
      }
    }
    __syncthreads();
  }
  const float rs = weights ? __bfloat162float(q.rs[0]) : 0.f;
  const bool vec_counts = in.E % 4 == 0 && reinterpret_cast<uintptr_t>(q.counts) % 16 == 0;
  for (; t < r1; t += ROW_WARPS, ++at) {
    ring.fetch(in, at + slots(NV) - 1, ahead(slots(NV) - 1), balance, weights, q.dwts);
    ring.wait();
    const float* row = ring.slot(at);
    const int b = balance && !(in.mask && in.mask[t] == 0) ? find(t) : -1;
    const bool term = b >= 0;
    // the lane's pick: its logit, score and slope, and the gradient of its weight
    int e = -1;
    float g = 0.f, pick = 0.f, pick_slope = 0.f;
    u32 peers = 0;
    if (weights) {
      float x = 0.f;
      if (lane < in.K) {
        e = reinterpret_cast<const int*>(row + 128 * NV)[lane];
        if (e < 0 || e >= in.E) e = -1;
        if (e >= 0) {
          x = balance ? row[e] : in.S[t * in.lds + e];
          g = row[128 * NV + PICKS + lane];
        }
      }
      const u64 ex = exp_neg2(f32x2(x, x)), sc = score2(ex);
      pick = e >= 0 ? f32x2_get(sc).x : 0.f;
      pick_slope = f32x2_get(slope2(sc, ex)).x;
      peers = __match_any_sync(0xffffffffu, e);
    }
    u64 d[N], slope[N];
    float k = 0.f;
    const int* cb = nullptr;  // the counts of a sequence other than the block's first and last
    const float* sf = b == b0 ? s_f : s_f + 128 * NV;
    float sums[4] = {0.f, 0.f, pick, g * pick};  // of scores, f scores; of the picks' scores, and with their gradients
    if (term) {
      u64 z2 = f32x2(0.f, 0.f), m2 = z2;
      if (b != b0 && b != b1) {
        const int n = q.rows[b];
        k = n > 0 ? scale / (float)n / (float)n : 0.f;
        cb = q.counts + (long long)b * in.E;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * 32 + lane) * 4;
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(row + c);
        const u64 e0 = exp_neg2(v.x), e1 = exp_neg2(v.y), s0 = score2(e0), s1 = score2(e1);
        z2 = add_f32x2(z2, add_f32x2(s0, s1));
        slope[2 * j] = slope2(s0, e0);
        slope[2 * j + 1] = slope2(s1, e1);
        ulonglong2 f;
        if (cb == nullptr) {
          f = *reinterpret_cast<const ulonglong2*>(sf + c);
        } else {
          int4 n = make_int4(0, 0, 0, 0);
          if (vec_counts) {
            if (c < in.E) n = *reinterpret_cast<const int4*>(cb + c);
          } else {
            n.x = c < in.E ? cb[c] : 0;
            n.y = c + 1 < in.E ? cb[c + 1] : 0;
            n.z = c + 2 < in.E ? cb[c + 2] : 0;
            n.w = c + 3 < in.E ? cb[c + 3] : 0;
          }
          f = make_ulonglong2(f32x2(k * (float)n.x, k * (float)n.y), f32x2(k * (float)n.z, k * (float)n.w));
        }
        m2 = fma_f32x2(f.x, s0, fma_f32x2(f.y, s1, m2));
        d[2 * j] = f.x;
        d[2 * j + 1] = f.y;
      }
      const float2 z = f32x2_get(z2), m = f32x2_get(m2);
      sums[0] = z.x + z.y;
      sums[1] = m.x + m.y;
    }
    warp_sums(sums);
    const float inv = reciprocal(sums[0] + TINY), m = sums[1] * inv;
    if (term) {
      const u64 minus = f32x2(-m, -m), inv2 = f32x2(inv, inv);
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = mul_f32x2(add_f32x2(d[i], minus), mul_f32x2(slope[i], inv2));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = 0ull;
    }
    // the pick's element: the sum of both terms, stored over the balance term alone
    float total = 0.f;
    if (weights) {
      const float den = reciprocal(sums[2] + TINY);
      const float mine = rs * den * (g - sums[3] * den) * pick_slope;
      const float f = !term || e < 0 ? 0.f : cb == nullptr ? sf[e] : k * (float)cb[e];
      const float base = term ? (f - m) * (pick_slope * inv) : 0.f;
      total = base + mine;
      // an expert named twice gets both parts, added in pick order
      if (!__all_sync(0xffffffffu, e < 0 || (peers & (peers - 1)) == 0)) {
        total = base;
        for (int i = 0; i < in.K; ++i) {
          const float other = __shfl_sync(0xffffffffu, mine, i);
          if (peers >> i & 1) total += other;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * 32 + lane) * 4;
      const float2 x = f32x2_get(d[2 * j]), y = f32x2_get(d[2 * j + 1]);
      const float v[4] = {x.x, x.y, y.x, y.y};
      if (q.bf16_out) {
        bf16* o = reinterpret_cast<bf16*>(q.dS) + t * q.ldd + c;
        if (q.vec_out && c + 4 <= in.E) {
          *reinterpret_cast<uint2*>(o) = make_uint2(f2_to_bf16x2(v[0], v[1]), f2_to_bf16x2(v[2], v[3]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + i < in.E) o[i] = __float2bfloat16_rn(v[i]);
        }
      } else {
        float* o = reinterpret_cast<float*>(q.dS) + t * q.ldd + c;
        if (q.vec_out && c + 4 <= in.E) {
          *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + i < in.E) o[i] = v[i];
        }
      }
    }
    __syncwarp();  // the row's stores are ordered before the picks', and its slot has been read
    if (e >= 0) {
      if (q.bf16_out) reinterpret_cast<bf16*>(q.dS)[t * q.ldd + e] = __float2bfloat16_rn(total);
      else reinterpret_cast<float*>(q.dS)[t * q.ldd + e] = total;
    }
  }
  cp_async_wait_all();
}

}  // namespace k3
