// Products in 8-bit integers (W8A8): the quantiser that gives every token (or weight channel) one scale, and
//   out[t, c] = sx[t] * sw[c] * sum_k q[t, k] w[c, k]
// on the tensor cores' integer path (tcgen05.mma kind::i8, int32 accumulators in TMEM), dense or grouped by expert
// over the routing tables.  The int32 sums are exact (|q w| <= 2^14, fewer than 2^17 terms), so the result does not
// depend on how the reduction is split.  No counterpart in the reference, whose experts are MXFP4.
#pragma once
#include "common.cuh"
#include "gemm.cu"

namespace k3 {

// ============================================================ quantiser
// amax = the row's largest magnitude, scale = amax / 127, q = round-half-even(127 x / amax): the rounding of the real
// quotient, not of a float product.
// bf16: with 127 / amax bracketed, 2^-21 of it above and below, one FMA each (1.5 * 2^23 + x inv) rounds the quotient seen
// from either side.  The quotient of two 8-bit mantissas is a half exactly or at least 2^-17 of itself from one, so the two
// integers are equal, or the neighbours of an exact half: then the even one is it, bit arithmetic on pairs, no branch (ties
// are common: rows whose maximum has few mantissa bits have them by the hundred).
// f32, and the gate's values (f32 too: their quotients come as near to a half as 2^-24): one FMA, and the elements whose
// x inv is within 1e-5 of a half (inv moves the quotient by 7.6e-6 at most) compare 254 |x| with (2k + 1) amax, both exact
// in double.
// A row with an infinity or a NaN has scale NaN and q = 0, so every result it enters is NaN; a zero row scale 0, q = 0.
// HBM-bound: a row is read once and kept in registers (bf16 as it came) between the maximum and the codes; what counts
// beside the bytes is the instructions an element, about 7, and blocks enough an SM.  Measured: 8192 x 7168 bf16 29.0 us
// (6.1 TB/s), f32 47.6 us (6.2 TB/s), gated 8192 x 2 x 2048 SwiGLU 19.5 us (4.3 TB/s: instructions, about 2 an element more
// than its exponential without the correction, 18.7 us), SiTU 38.6 us (two tanhf an element).
enum { I8_BF16 = 0, I8_F32 = 1, I8_GATED = 2 };

struct QuantRows {
  const void* x;       // bf16 or f32 [rows, ldx]; gated: bf16 [rows, gate | up]
  long long ldx;
  long long rows;
  int cols;
  int vec;             // rows may be read 16 bytes at a time
  int act;             // gated: 0 SwiGLU, 1 SiTU
  int8_t* q;           // [.., ldq]
  long long ldq;
  float* scale;
  // where row r goes: row r; or with exp2perm, rows exp2perm[r * K + k] >= 0 and (meta[2] >= 0) row meta[2] + r
  const int* exp2perm;
  int K;
  // which rows are real (null: all): r < cta_limit[r / 128], r / 128 < meta[0]
  const int* cta_limit;
  const int* meta;
  int max_ctas;
  long long cap_rows;  // output rows
};

// act(g) * u of two elements, bf16 pairs; the sigmoid by one exponential and one reciprocal instruction, within 2^-21 of
// its value.  Gates are clamped to +-88 for it: below, the sigmoid is under the smallest normal f32 and 0 here (g = -inf:
// 0 * -inf, a NaN, as for any row that holds an infinity).
__device__ __forceinline__ float2 gate_of(u32 gate, u32 up, int act) {
  u32 y = gate ^ 0x80008000u;  // -g
  asm("min.bf16x2 %0, %0, %1;" : "+r"(y) : "r"(0x42b042b0u));
  asm("max.bf16x2 %0, %0, %1;" : "+r"(y) : "r"(0xc2b0c2b0u));
  const float2 ny = bf16x2_to_f2(y), g = bf16x2_to_f2(gate), u = bf16x2_to_f2(up);
  const float2 d = f32x2_get(add_f32x2(exp_f32x2(f32x2(ny.x, ny.y)), f32x2(1.f, 1.f)));
  const u64 sg = f32x2(rcp_ftz(d.x), rcp_ftz(d.y));
  if (act == 0) return f32x2_get(mul_f32x2(mul_f32x2(f32x2(g.x, g.y), sg), f32x2(u.x, u.y)));
  const u64 a = f32x2(4.f * tanhf(0.25f * g.x), 4.f * tanhf(0.25f * g.y));
  return f32x2_get(mul_f32x2(mul_f32x2(a, sg), f32x2(25.f * tanhf(0.04f * u.x), 25.f * tanhf(0.04f * u.y))));
}

// 8 consecutive elements of a row as they are kept: bf16 pairs, or f32
template <int SRC>
struct Kept {
  u32 w[SRC == I8_BF16 ? 4 : 8];
  __device__ __forceinline__ float operator[](int i) const {
    if (SRC == I8_BF16) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    return __uint_as_float(w[SRC == I8_BF16 ? i >> 1 : i]);
  }
};

// 8 bf16 from s; not WHOLE: one at a time, zero past `left`
template <bool WHOLE>
__device__ __forceinline__ uint4 load_bf16x8(const bf16* s, int left) {
  if (WHOLE) return *reinterpret_cast<const uint4*>(s);
  u32 h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = i < left ? (u32)__bfloat16_as_ushort(s[i]) : 0u;
  return make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
}

// elements c .. c + 7 of a row that starts at x
template <int SRC, bool WHOLE>
__device__ __forceinline__ void load8(const QuantRows& p, const void* x, int c, Kept<SRC>& v) {
  constexpr int M = SRC == I8_BF16 ? 4 : 8;
  const int left = p.cols - c;
  if (SRC == I8_F32) {
    const u32* s = reinterpret_cast<const u32*>(x) + c;
    if (WHOLE) {
      const uint4 a = reinterpret_cast<const uint4*>(s)[0], b = reinterpret_cast<const uint4*>(s)[1];
      const u32 w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v.w[i % M] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v.w[i % M] = i < left ? s[i] : 0u;
    }
    return;
  }
  const bf16* s = reinterpret_cast<const bf16*>(x) + c;
  const uint4 a = load_bf16x8<WHOLE>(s, left);
  const u32 g[4] = {a.x, a.y, a.z, a.w};
  if (SRC == I8_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = g[i];
    return;
  }
  const uint4 b = load_bf16x8<WHOLE>(s + p.cols, left);
  const u32 u[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 h = gate_of(g[i], u[i], p.act);
    v.w[(2 * i) % M] = __float_as_uint(h.x);
    v.w[(2 * i + 1) % M] = __float_as_uint(h.y);
  }
}

// The running maximum of magnitudes as ordered bits (a NaN above an infinity above all numbers): bf16 pairs as two
// 16-bit halves, f32 whole.
template <int SRC>
__device__ __forceinline__ u32 max_bits(u32 m, const Kept<SRC>& v) {
  if (SRC == I8_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("max.s16x2 %0, %0, %1;" : "+r"(m) : "r"(v.w[i] & 0x7fff7fffu));
  } else {
    float f = __uint_as_float(m);
#pragma unroll
    for (int i = 0; i < (SRC == I8_BF16 ? 4 : 8); ++i)
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(f) : "f"(fabsf(__uint_as_float(v.w[i]))));
    m = __float_as_uint(f);
  }
  return m;
}

struct RowScale {
  float amax, pre, inv;  // pre: a power of two that keeps 127 / amax finite; inv 0: a row of zeros, or with no number
};
template <int SRC>
__device__ __forceinline__ RowScale row_scale(u32 amax_bits) {
  RowScale s;
  s.amax = __uint_as_float(amax_bits);
  s.pre = s.inv = 0.f;
  if (amax_bits < 0x7f800000u && amax_bits != 0u) {
    s.pre = s.amax < 0x1p-60f ? 0x1p64f : s.amax > 0x1p60f ? 0x1p-64f : 1.f;
    s.inv = SRC == I8_BF16 ? 127.f * rcp_ftz(s.amax * s.pre) : __fdiv_rn(127.f, s.amax * s.pre);
  }
  return s;
}
__device__ __forceinline__ float scale_of(const RowScale& s) {
  return __float_as_uint(s.amax) >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __fdiv_rn(s.amax, 127.f);
}
// Rows at the ends of the range: the kept elements times `pre` (exact, but for those far too small to have a code), or
// zeros where there is no scale.  Every other row skips this.
template <int SRC>
__device__ __forceinline__ void settle8(const RowScale& s, Kept<SRC>& v) {
  if (SRC == I8_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v.w[i] = s.inv == 0.f ? 0u : f2_to_bf16x2(v[2 * i] * s.pre, v[2 * i + 1] * s.pre);
  } else {
#pragma unroll
    for (int i = 0; i < (SRC == I8_BF16 ? 4 : 8); ++i) v.w[i] = s.inv == 0.f ? 0u : __float_as_uint(v[i] * s.pre);
  }
}

// the code of an element whose quotient lies near k + 1/2 in magnitude
__device__ __forceinline__ int code_near_half(float x, int k, float amax) {
  const double a = 254.0 * fabs((double)x), h = (double)(2 * k + 1) * (double)amax;
  const int m = a > h || (a == h && (k & 1)) ? k + 1 : k;
  return x < 0.f ? -m : m;
}

template <int SRC>
__device__ __forceinline__ uint2 encode8(const RowScale& s, const Kept<SRC>& v) {
  if (SRC == I8_BF16) {
    constexpr float ROUND = 12582912.f + 256.f;  // the integer, plus 256, in the low 16 bits
    const float above = s.inv * (1.f + 0x1p-21f), below = s.inv * (1.f - 0x1p-21f);
    const u64 up = f32x2(above, above), down = f32x2(below, below), round = f32x2(ROUND, ROUND);
    u32 k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u64 x = f32x2(v[2 * i], v[2 * i + 1]);
      const float2 a = f32x2_get(fma_f32x2(x, up, round)), b = f32x2_get(fma_f32x2(x, down, round));
      // two elements' integers in the halves of a word; their sum is odd where the two roundings differ, and half of it
      // rounded up to even is the code
      const u32 sum = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x5410) +
                      __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x5410);
      const u32 half = sum >> 1;
      k[i] = half + (sum & half & 0x00010001u);
    }
    return make_uint2(__byte_perm(k[0], k[1], 0x6420), __byte_perm(k[2], k[3], 0x6420));
  }
  constexpr float ROUND = 12582912.f;  // 1.5 * 2^23: the integer sits in the low bits
  constexpr float NEAR = 0.5f - 1e-5f;
  const u64 inv = f32x2(s.inv, s.inv), round = f32x2(ROUND, ROUND), minus = f32x2(-1.f, -1.f);
  u32 k[8];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u64 x = f32x2(v[2 * i], v[2 * i + 1]), t = fma_f32x2(x, inv, round);
    const float2 n = f32x2_get(t), d = f32x2_get(fma_f32x2(x, inv, fma_f32x2(t, minus, round)));  // d: x inv - its integer
    far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
    k[2 * i] = __float_as_uint(n.x);
    k[2 * i + 1] = __float_as_uint(n.y);
  }
  if (far > NEAR) {  // one group in some thousands
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float n = __uint_as_float(k[i]) - ROUND, d = __fmaf_rn(v[i], s.inv, -n);
      // |quotient| = |n| + d (with n's sign), and the integer below it
      if (fabsf(d) > NEAR)
        k[i] = (u32)code_near_half(v[i], (int)fabsf(n) - (n != 0.f && (d < 0.f) == (n > 0.f) ? 1 : 0), s.amax * s.pre);
    }
  }
  const u32 a = __byte_perm(k[0], k[1], 0x0040), b = __byte_perm(k[2], k[3], 0x0040);
  const u32 c = __byte_perm(k[4], k[5], 0x0040), d = __byte_perm(k[6], k[7], 0x0040);
  return make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410));
}
template <bool WHOLE>
__device__ __forceinline__ void put8(int8_t* dst, int left, uint2 w) {
  if (WHOLE || left >= 8) {
    *reinterpret_cast<uint2*>(dst) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) dst[i] = (int8_t)((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
  }
}

// LANES threads a row (a warp of a block of 256, or a block), NV groups of 8 elements a thread kept in registers;
// NV = 0: rows too long for that are read a second time (from L2).  MINB blocks an SM: enough loads in flight.  WHOLE:
// rows are read 16 bytes at a time and end with a group (else an element at a time).
template <int SRC, int LANES, int NV, int MINB, bool WHOLE>
__global__ void __launch_bounds__(LANES > 32 ? LANES : 256, MINB) quant_int8_kernel(QuantRows p) {
  __shared__ u32 s_max[2][LANES > 32 ? LANES / 32 : 1];
  constexpr int PER = LANES > 32 ? 1 : 8;
  constexpr int STEP = LANES * 8;
  constexpr int KEPT = NV > 0 ? NV : 1;
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  grid_wait_previous();
  grid_launch_dependents();
  long long first = (long long)blockIdx.x * PER + sub, last = p.rows, next = (long long)gridDim.x * PER;
  if (p.cta_limit) {  // sixteen blocks a tile of 128 rows, over its real ones
    const int c = blockIdx.x >> 4;
    if (c >= min(p.meta[0], p.max_ctas)) return;
    first = c * 128ll + (blockIdx.x & 15) * PER + sub;
    last = min(last, min((long long)p.cta_limit[c], c * 128ll + 128));
    next = 16 * PER;
  }
  const int shared_row = p.exp2perm ? p.meta[2] : -1;
  const long long row_bytes = p.ldx * (SRC == I8_F32 ? 4 : 2);
  int buf = 0;
  for (long long r = first; r < last; r += next) {
    // lane k of a warp holds the row's k-th target, loaded ahead of its elements
    int target = -1;
    if (p.exp2perm) {
      const int k = lane & 31;
      if (k < p.K) target = p.exp2perm[r * p.K + k];
      else if (k == p.K && shared_row >= 0) target = shared_row + (int)r;
    }
    const char* x = reinterpret_cast<const char*>(p.x) + r * row_bytes;
    u32 m = 0;
    Kept<SRC> v[KEPT];
    if (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = j * STEP + lane * 8;
#pragma unroll
        for (int i = 0; i < (SRC == I8_BF16 ? 4 : 8); ++i) v[j].w[i] = 0u;
        if (c < p.cols) load8<SRC, WHOLE>(p, x, c, v[j]);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) m = max_bits<SRC>(m, v[j]);
    } else {
      for (int c = lane * 8; c < p.cols; c += STEP) {
        load8<SRC, WHOLE>(p, x, c, v[0]);
        m = max_bits<SRC>(m, v[0]);
      }
    }
    if (SRC == I8_BF16) m = max(m << 16, m & 0xffff0000u);
    m = __reduce_max_sync(0xffffffffu, m);
    if (LANES > 32) {
      if ((threadIdx.x & 31) == 0) s_max[buf][threadIdx.x >> 5] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < LANES / 32; ++i) m = max(m, s_max[buf][i]);
      buf ^= 1;  // the next row's maxima go to the other half: one barrier a row
    }
    const RowScale s = row_scale<SRC>(m);
    const bool rare = s.pre != 1.f;
    if (NV > 0 && rare) {
#pragma unroll
      for (int j = 0; j < NV; ++j) settle8<SRC>(s, v[j]);
    }
    if (NV > 0 && !p.exp2perm) {
      int8_t* dst = p.q + r * p.ldq;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = j * STEP + lane * 8;
        if (c < p.cols) put8<WHOLE>(dst + c, p.cols - c, encode8<SRC>(s, v[j]));
      }
      if (lane == 0) p.scale[r] = scale_of(s);
      continue;
    }
    if (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const uint2 w = encode8<SRC>(s, v[j]);  // past the row's end: zeros, kept and not stored
        v[j].w[0] = w.x;
        v[j].w[1] = w.y;
      }
    }
    const int targets = p.exp2perm ? p.K + 1 : 1;
    for (int k = 0; k < targets; ++k) {
      const long long o = p.exp2perm ? (long long)__shfl_sync(0xffffffffu, target, k) : r;
      if (o < 0 || o >= p.cap_rows) continue;
      int8_t* dst = p.q + o * p.ldq;
      if (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int c = j * STEP + lane * 8;
          if (c < p.cols) put8<WHOLE>(dst + c, p.cols - c, make_uint2(v[j].w[0], v[j].w[1]));
        }
      } else {
        for (int c = lane * 8; c < p.cols; c += STEP) {
          load8<SRC, WHOLE>(p, x, c, v[0]);
          if (rare) settle8<SRC>(s, v[0]);
          put8<WHOLE>(dst + c, p.cols - c, encode8<SRC>(s, v[0]));
        }
      }
      if (lane == 0) p.scale[o] = scale_of(s);
    }
  }
}

// ============================================================ products
// Tiles.  The MMA's M is 128 weight channels and its N the tokens (16 to 256 in steps of 16), so that a decode batch
// or an expert's few rows cost what they are and not 128 rows: the weights, which bound those shapes, stream through
// at full rate.  A stage is 128 K bytes (one swizzle atom) of both operands in an mbarrier ring; rows and K past the
// ends are zero-filled by the loads.  Roles: warp 0 lane 0 issues the TMA boxes, warp 1 lane 0 the MMAs
// into one of two TMEM accumulators, the other warps scale and store the other.  Every wait is bounded and reports.
//
// Where there is work enough (PAIR) two blocks share a unit of 256 channels x up to 256 tokens (cta_group::2): each
// loads its 128 channels and half of the tokens, the even block issues M = 256 MMAs over both blocks' shared memory, and
// each drains its own channels.  One block alone would write and read 96 KB of shared memory for the 512 MMA cycles of a
// stage, more than its 128 bytes a cycle; a pair halves the tokens' part.
//
// Measured: 8192 x 7168 -> 4096 143 us (3.36 POP/s, tensor pipe 84% active) against 160 us on single blocks; called without
// a pause both run into the 1000 W cap (1.38 GHz, 162 us).  112 experts, 8192 picks, 2048 -> 7168: 278 us (6.4 TB/s).
//
// With few units a cluster of `splits` blocks shares one unit, each a part of K; the parts' int32 sums meet in shared
// memory (each block adds every split-th token of all blocks' tiles through the cluster), so a decode step keeps all
// SMs loading weights without a workspace or a second launch (one token, 7168 -> 4096: 18.4 us on one part, 12.9 on two,
// 10.9 on four; 5 us of it are fixed, the weights come at 5.2 TB/s).
namespace i8 {
constexpr int BM = 128;                  // weight channels a unit
constexpr int BK = 128;                  // K bytes a stage
constexpr int W_BYTES = BM * BK;
constexpr int RING_BYTES = 192 * 1024;
constexpr int MAX_STAGES = 10;
constexpr int EPI_WARPS = 16;            // four a TMEM sub-partition
constexpr int EPI_STEP = EPI_WARPS / 4 * 16;  // tokens they take in a turn
constexpr int EPI_SCALES = 256 / (EPI_WARPS / 4);  // tokens of a warp
constexpr int BAR_BYTES = 256;
constexpr int SMEM_BYTES = RING_BYTES + 1024 /*align*/ + BAR_BYTES + EPI_WARPS * EPI_SCALES * 4 /*token scales*/;
constexpr int WARPS = 2 + EPI_WARPS;
constexpr int THREADS = 32 * WARPS;
}  // namespace i8

struct Int8Params {
  const float* sx;         // [T] (grouped: permuted rows)
  const float* sw;         // [experts * N]
  void* out;               // [T, ldo] of the kernel's OUT
  long long ldo;
  int T;                   // token rows (dense)
  int N;                   // weight channels (an expert)
  int kstages;
  int bn;                  // token rows a unit, a multiple of 16
  int xbox;                // rows of the token map's box
  int n_tiles;             // ceil(N / 128)
  int t_tiles;             // dense: ceil(T / bn)
  int stages, stage_bytes;
  u32 tmem_cols;
  int splits;              // blocks of a cluster sharing a unit
  const int* cta_batch;    // grouped: the routing tables (null: dense)
  const int* cta_limit;
  const int* meta;
  int n_experts, max_ctas, cap_rows;
  u32* err;
};

struct Int8Unit {
  int valid, e, row0, n, ch0;
};
template <bool PAIR>
__device__ __forceinline__ Int8Unit int8_unit(const Int8Params& p, int u, int rank) {
  Int8Unit w;
  const int c = u / p.n_tiles;
  w.ch0 = PAIR ? (u % p.n_tiles) * 2 * i8::BM + rank * i8::BM : (u % p.n_tiles) * i8::BM;
  if (p.cta_batch) {
    w.e = p.cta_batch[c];
    w.row0 = c * 128;
    w.n = p.cta_limit[c] - w.row0;
    w.valid = w.e >= 0 && w.e < p.n_experts && w.n > 0 && w.n <= 128 && w.row0 + 128 <= p.cap_rows;
  } else {
    w.e = 0;
    w.row0 = c * p.bn;
    w.n = min(p.bn, p.T - w.row0);
    w.valid = 1;
  }
  return w;
}

// kind::i8 instruction descriptor: s32 accumulator, signed A and B, both K-major, M x N
__device__ __forceinline__ u32 i8_idesc(int m, int n) {
  return 2u << 4 | 1u << 7 | 1u << 10 | (u32)(n >> 3) << 17 | (u32)(m >> 4) << 24;
}
__device__ __forceinline__ void i8_mma_pair(u32 d_tmem, u64 adesc, u64 bdesc, u32 idesc, u32 accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void i8_mma(u32 d_tmem, u64 adesc, u64 bdesc, u32 idesc, u32 accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void i8_ld16(u32 taddr, u32 (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ int4 ld_cluster_v4(u32 saddr, u32 rank) {
  int4 v;
  asm volatile(
      "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %4, %5;\n ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [a];\n}\n"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "r"(saddr), "r"(rank)
      : "memory");
  return v;
}

// out = fl(fl(fl(acc) * sx) * sw), rounded once more to bf16
__device__ __forceinline__ void int8_put(float* d, u32 acc, float sx, float sw) { *d = __int2float_rn((int)acc) * sx * sw; }
__device__ __forceinline__ void int8_put(bf16* d, u32 acc, float sx, float sw) {
  *d = __float2bfloat16_rn(__int2float_rn((int)acc) * sx * sw);
}
// two tokens of one channel, at d and d + step
__device__ __forceinline__ float2 int8_pair(u32 a0, u32 a1, u64 sx, u64 sw) {
  return f32x2_get(mul_f32x2(mul_f32x2(f32x2(__int2float_rn((int)a0), __int2float_rn((int)a1)), sx), sw));
}
__device__ __forceinline__ void int8_put2(float* d, long long step, u32 a0, u32 a1, u64 sx, u64 sw) {
  const float2 v = int8_pair(a0, a1, sx, sw);
  d[0] = v.x;
  d[step] = v.y;
}
__device__ __forceinline__ void int8_put2(bf16* d, long long step, u32 a0, u32 a1, u64 sx, u64 sw) {
  const float2 v = int8_pair(a0, a1, sx, sw);
  const u32 h = f2_to_bf16x2(v.x, v.y);
  unsigned short* o = reinterpret_cast<unsigned short*>(d);
  o[0] = (unsigned short)h;
  o[step] = (unsigned short)(h >> 16);
}

template <typename OUT, bool PAIR>
__global__ void __launch_bounds__(i8::THREADS, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, Int8Params p) {
  using namespace i8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  u64* bars = reinterpret_cast<u64*>(smem + RING_BYTES);
  u64* full = bars;                          // [MAX_STAGES]
  u64* empty = bars + MAX_STAGES;            // [MAX_STAGES]
  u64* acc_full = bars + 2 * MAX_STAGES;     // [2]
  u64* acc_empty = bars + 2 * MAX_STAGES + 2;  // [2]
  u64* drain = bars + 2 * MAX_STAGES + 4;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * MAX_STAGES + 5);
  u32* tmem_slot = reinterpret_cast<u32*>(bars + 2 * MAX_STAGES + 6);
  float* scales = reinterpret_cast<float*>(smem + RING_BYTES + BAR_BYTES);  // [EPI_WARPS][EPI_SCALES]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, p.tmem_cols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, p.tmem_cols);
      tmem_relinquish();
    }
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], PAIR ? 2 * EPI_WARPS : EPI_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmX);
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // the other block's barriers are there
  tc_fence_after();
  const u32 tmem_base = *tmem_slot;
  // the block's part of K (all of it without a cluster)
  const int rank = PAIR || p.splits > 1 ? (int)cluster_rank() : 0;
  const int k0 = PAIR ? 0 : (int)((long long)rank * p.kstages / p.splits);
  const int k1 = PAIR ? p.kstages : (int)((long long)(rank + 1) * p.kstages / p.splits);
  const int share = PAIR ? 2 : p.splits;  // blocks a unit
  const int first = blockIdx.x / share, stride = gridDim.x / share;
  grid_wait_previous();  // the rows (and whatever else an earlier kernel writes) are there from here on
  const int units = (p.cta_batch ? min(p.meta[0], p.max_ctas) : p.t_tiles) * p.n_tiles;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer
      int stage = 0;
      u32 phase = 0;
      u32 armed = 0;  // fills issued; stage s holds the last of them with index = s mod stages
      for (int u = first; u < units && !*abort_flag; u += stride) {
        const Int8Unit w = int8_unit<PAIR>(p, u, rank);
        if (!w.valid) {
          report_error(p.err, ERR_BAD_TABLE, 0xD00u);
          continue;
        }
        const int boxes = PAIR ? 1 : (w.n + p.xbox - 1) / p.xbox;
        // PAIR: both blocks' loads complete on the even block's barrier, which expects them all
        const u32 tx = (u32)(W_BYTES + boxes * p.xbox * BK) * (PAIR ? 2u : 1u);
        const int wrow = w.e * p.N + w.ch0;
        const int xrow = w.row0 + (PAIR ? rank * (((w.n + 31) & ~31) / 2) : 0);
        for (int ks = k0; ks < k1; ++ks) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.err, 0xD10u)) break;
          uint8_t* st = smem + stage * p.stage_bytes;
          if (PAIR) {
            if (rank == 0) {
              mbar_arrive_expect_tx(&full[stage], tx);
              ++armed;
            }
            const u32 bar = cluster_addr(&full[stage], 0);
            tma_load_2d_pair(st, &tmW, bar, ks * BK, wrow);
            tma_load_2d_pair(st + W_BYTES, &tmX, bar, ks * BK, xrow);
          } else {
            mbar_arrive_expect_tx(&full[stage], tx);
            ++armed;
            tma_load_2d(st, &tmW, &full[stage], ks * BK, wrow);
            for (int i = 0; i < boxes; ++i)
              tma_load_2d(st + W_BYTES + i * p.xbox * BK, &tmX, &full[stage], ks * BK, xrow + i * p.xbox);
          }
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // every fill has landed before the block may exit (PAIR: before either may, behind the cluster barrier below)
      for (u32 s = 0; s < (u32)p.stages && s < armed; ++s)
        mbar_wait(&full[s], ((armed - 1 - s) / (u32)p.stages) & 1u, nullptr, p.err, 0xD20u, 100000000ull);
    }
  } else if (warp == 1) {
    if (lane == 0 && (!PAIR || rank == 0)) {
      // ------------------------------------------------ MMA issuer
      int stage = 0, buf = 0;
      u32 phase = 0;
      u32 acc_phase = 0;  // bit b: accumulator b's parity
      bool issued = false;
      for (int u = first; u < units && !*abort_flag; u += stride) {
        const Int8Unit w = int8_unit<PAIR>(p, u, rank);
        if (!w.valid) continue;
        if (!mbar_wait(&acc_empty[buf], ((acc_phase >> buf) & 1u) ^ 1u, abort_flag, p.err, 0xD30u)) break;
        tc_fence_after();
        const u32 idesc = PAIR ? i8_idesc(2 * BM, (w.n + 31) & ~31) : i8_idesc(BM, (w.n + 15) & ~15);
        const u32 d = tmem_base + (u32)(buf * p.bn);
        bool ok = true;
        for (int ks = k0; ks < k1; ++ks) {
          if (!mbar_wait(&full[stage], phase, abort_flag, p.err, 0xD40u)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const u32 st = smem_u32(smem + stage * p.stage_bytes);
#pragma unroll
          for (int kk = 0; kk < BK / 32; ++kk) {
            const u64 a = sdesc_k_sw128(st + kk * 32), b = sdesc_k_sw128(st + W_BYTES + kk * 32);
            if (PAIR) i8_mma_pair(d, a, b, idesc, ks != k0 || kk != 0);
            else i8_mma(d, a, b, idesc, ks != k0 || kk != 0);
          }
          if (PAIR) tc_commit_pair(&empty[stage]);
          else tc_commit(&empty[stage]);
          issued = true;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (PAIR) tc_commit_pair(&acc_full[buf]);
        else tc_commit(&acc_full[buf]);
        acc_phase ^= 1u << buf;
        buf ^= 1;
      }
      if (issued) {
        if (PAIR) tc_commit_pair(drain);
        else tc_commit(drain);
        mbar_wait(drain, 0, nullptr, p.err, 0xD50u, 100000000ull);
      }
    }
  } else {
    // ------------------------------------------------ epilogue (warps 2 on): a lane is a channel, columns are tokens;
    // the warps of a sub-partition take 16 tokens in turn, the next 16 on their way while these are scaled and stored
    // (a token's 32 channels a warp store).  The tokens' scales come by broadcast from shared memory.
    const int sub = warp & 3, turn = (warp - 2) >> 2;
    const u32 lane_base = (u32)(sub * 32) << 16;
    int* red = reinterpret_cast<int*>(smem);
    float* sxs = scales + (warp - 2) * EPI_SCALES;  // this warp's tokens: 16 of every EPI_STEP
    const long long row_step = p.ldo;
    u32 acc_phase = 0;
    int buf = 0;
    for (int u = first; u < units && !*abort_flag; u += stride) {
      const Int8Unit w = int8_unit<PAIR>(p, u, rank);
      if (!w.valid) continue;
      const int ch = w.ch0 + sub * 32 + lane;
      const float swc = ch < p.N ? p.sw[(long long)w.e * p.N + ch] : 0.f;
      for (int i = lane; i < EPI_SCALES; i += 32) {
        const int t = (i >> 4) * EPI_STEP + turn * 16 + (i & 15);
        sxs[i] = t < w.n ? p.sx[w.row0 + t] : 0.f;
      }
      __syncwarp();
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (acc_phase >> buf) & 1u, abort_flag, p.err, 0xD60u))) break;
      tc_fence_after();
      const u32 acc = tmem_base + lane_base + (u32)(buf * p.bn);
      int c = turn * 16;
      u32 v[16];
      if (c < w.n) i8_ld16(acc + (u32)c, v);
      OUT* dst = reinterpret_cast<OUT*>(p.out) + ((long long)w.row0 + c) * row_step + ch;
      const float* sx = sxs;
      const bool whole = w.ch0 + BM <= p.N;
#pragma unroll 1
      for (; c < w.n; c += EPI_STEP, dst += EPI_STEP * row_step, sx += 16) {
        tmem_wait_ld();
        u32 x[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = v[j];
        if (c + EPI_STEP < w.n) i8_ld16(acc + (u32)(c + EPI_STEP), v);
        if (!PAIR && p.splits > 1) {
#pragma unroll
          for (int j = 0; j < 16; ++j) red[(c + j) * BM + sub * 32 + lane] = (int)x[j];
        } else if (whole && c + 16 <= w.n) {
          OUT* d = dst;
          const u64 sw2 = f32x2(swc, swc);
#pragma unroll
          for (int j = 0; j < 16; j += 4, d += 4 * row_step) {
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(sx + j);
            int8_put2(d, row_step, x[j], x[j + 1], q.x, sw2);
            int8_put2(d + 2 * row_step, row_step, x[j + 2], x[j + 3], q.y, sw2);
          }
        } else {
          OUT* d = dst;
#pragma unroll
          for (int j = 0; j < 16; ++j, d += row_step)
            if (ch < p.N && c + j < w.n) int8_put(d, x[j], sx[j], swc);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(cluster_addr(&acc_empty[buf], 0));
        else mbar_arrive(&acc_empty[buf]);
      }
      acc_phase ^= 1u << buf;
      buf ^= 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // neither block's shared memory, barriers or accumulators are in use any more
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, p.tmem_cols);
    else tmem_dealloc(tmem_base, p.tmem_cols);
  }
  if (!PAIR && p.splits > 1) {
    // one unit a cluster: the parts of K meet
    const Int8Unit w = int8_unit<PAIR>(p, first, rank);
    const u32 red = smem_u32(smem);
    const int ch = w.ch0 + lane * 4;
    float sw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sw[i] = ch + i < p.N ? p.sw[ch + i] : 0.f;
    cluster_sync();
    for (int t = warp * p.splits + rank; t < w.n; t += WARPS * p.splits) {
      const float s = p.sx[w.row0 + t];
      int4 b[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < p.splits) b[r] = ld_cluster_v4(red + (u32)(t * BM + lane * 4) * 4, (u32)r);
      int q[4] = {0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < p.splits) {
          q[0] += b[r].x;
          q[1] += b[r].y;
          q[2] += b[r].z;
          q[3] += b[r].w;
        }
      OUT* dst = reinterpret_cast<OUT*>(p.out) + ((long long)w.row0 + t) * p.ldo + ch;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (ch + i < p.N) int8_put(dst + i, (u32)q[i], s, sw[i]);
    }
    cluster_sync();  // no block leaves while another reads its part
  }
}

}  // namespace k3
