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
// quotient, not of a float product.  y = x * (127 / amax) is within 2e-5 of it, which settles every element but those
// within 1e-4 of a half; these compare 254 |x| with (2k + 1) amax, both exact in double.
// A row with an infinity or a NaN has scale NaN and q = 0, so every result it enters is NaN; a zero row scale 0, q = 0.
// HBM-bound: a row is read once and kept in registers between the maximum and the codes.
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

// 16 consecutive elements of a row as f32, zero past `cols`
template <int SRC>
__device__ __forceinline__ void load16(const QuantRows& p, long long r, int c, float (&v)[16]) {
  if (SRC == I8_F32) {
    const float* s = reinterpret_cast<const float*>(p.x) + r * p.ldx + c;
    if (p.vec && c + 16 <= p.cols) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = reinterpret_cast<const float4*>(s)[i];
        v[4 * i] = f.x;
        v[4 * i + 1] = f.y;
        v[4 * i + 2] = f.z;
        v[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = c + i < p.cols ? s[i] : 0.f;
    }
    return;
  }
  const bf16* s = reinterpret_cast<const bf16*>(p.x) + r * p.ldx + c;
  if (p.vec && c + 16 <= p.cols) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 a = reinterpret_cast<const uint4*>(s)[i];
      const u32 w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = bf16x2_to_f2(w[k]);
        v[8 * i + 2 * k] = f.x;
        v[8 * i + 2 * k + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c + i < p.cols ? __bfloat162float(s[i]) : 0.f;
  }
  if (SRC == I8_GATED) {
    const bf16* u = s + p.cols;
    if (p.vec && c + 16 <= p.cols) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 a = reinterpret_cast<const uint4*>(u)[i];
        const u32 w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = bf16x2_to_f2(w[k]);
          v[8 * i + 2 * k] = gated_act(v[8 * i + 2 * k], f.x, p.act);
          v[8 * i + 2 * k + 1] = gated_act(v[8 * i + 2 * k + 1], f.y, p.act);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (c + i < p.cols) v[i] = gated_act(v[i], __bfloat162float(u[i]), p.act);
    }
  }
}

// the code of an element whose quotient lies near a half: y its float quotient
__device__ __noinline__ int code_near_half(float x, float y, float amax) {
  const int k = (int)fabsf(y);
  const double a = 254.0 * fabs((double)x), h = (double)(2 * k + 1) * (double)amax;
  const int m = a > h || (a == h && (k & 1)) ? k + 1 : k;
  return x < 0.f ? -m : m;
}

// bytes lo .. hi of four codes
__device__ __forceinline__ u32 pack_s8(int a, int b, int c, int d) {
  u32 r;
  asm("{\n .reg .b32 t;\n cvt.pack.sat.s8.s32.b32 t, %4, %3, 0;\n cvt.pack.sat.s8.s32.b32 %0, %2, %1, t;\n}\n"
      : "=r"(r)
      : "r"(a), "r"(b), "r"(c), "r"(d));
  return r;
}

struct RowScale {
  float amax, pre, inv, scale;  // pre: a power of two that keeps 127 / amax finite
};
__device__ __forceinline__ RowScale row_scale(u32 amax_bits) {
  RowScale s;
  s.amax = __uint_as_float(amax_bits);
  if (amax_bits >= 0x7f800000u) {
    s.pre = s.inv = 0.f;
    s.scale = __uint_as_float(0x7fc00000u);
  } else if (amax_bits == 0u) {
    s.pre = s.inv = s.scale = 0.f;
  } else {
    s.pre = s.amax < 0x1p-60f ? 0x1p64f : s.amax > 0x1p60f ? 0x1p-64f : 1.f;
    s.inv = __fdiv_rn(127.f, s.amax * s.pre);
    s.scale = __fdiv_rn(s.amax, 127.f);
  }
  return s;
}

__device__ __forceinline__ uint4 encode16(const RowScale& s, const float (&v)[16]) {
  int k[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float y = (v[i] * s.pre) * s.inv, n = rintf(y);
    k[i] = s.inv == 0.f ? 0 : (int)n;  // a non-finite row: 0
    if (fabsf(fabsf(y - n) - 0.5f) < 1e-4f) k[i] = code_near_half(v[i], y, s.amax);
  }
  return make_uint4(pack_s8(k[0], k[1], k[2], k[3]), pack_s8(k[4], k[5], k[6], k[7]),
                    pack_s8(k[8], k[9], k[10], k[11]), pack_s8(k[12], k[13], k[14], k[15]));
}
__device__ __forceinline__ void put16(int8_t* dst, int left, uint4 w) {
  if (left >= 16) {
    *reinterpret_cast<uint4*>(dst) = w;
  } else {
    const u32 b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < left) dst[i] = (int8_t)(b[i >> 2] >> (8 * (i & 3)));
  }
}

// LANES threads a row (a warp, or the block of 256), NV groups of 16 elements a thread kept in registers; NV = 0: rows
// too long for that are read a second time (from L2).
template <int SRC, int LANES, int NV>
__global__ void __launch_bounds__(256) quant_int8_kernel(QuantRows p) {
  __shared__ u32 s_max[2][8];
  constexpr int PER = 256 / LANES;
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const int step = LANES * 16;
  const int nne = p.meta && p.cta_limit ? min(p.meta[0], p.max_ctas) : 0;
  int buf = 0;
  for (long long r = (long long)blockIdx.x * PER + sub; r < p.rows; r += (long long)gridDim.x * PER) {
    if (p.cta_limit && ((r >> 7) >= nne || r >= p.cta_limit[r >> 7])) continue;  // the row's LANES threads together
    u32 m = 0;
    float v[NV > 0 ? NV : 1][16];
    if (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = j * step + lane * 16;
        if (c < p.cols) {
          load16<SRC>(p, r, c, v[j]);
#pragma unroll
          for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[j][i]) & 0x7fffffffu);
        }
      }
    } else {
      for (int c = lane * 16; c < p.cols; c += step) {
        load16<SRC>(p, r, c, v[0]);
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[0][i]) & 0x7fffffffu);
      }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (LANES > 32) {
      if ((threadIdx.x & 31) == 0) s_max[buf][threadIdx.x >> 5] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, s_max[buf][i]);
      buf ^= 1;  // the next row's maxima go to the other half: one barrier a row
    }
    const RowScale s = row_scale(m);
    const int targets = p.exp2perm ? p.K + 1 : 1;
    uint4 w[NV > 0 ? NV : 1];
    if (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * step + lane * 16 < p.cols) w[j] = encode16(s, v[j]);
    }
    for (int k = 0; k < targets; ++k) {
      long long o = r;
      if (p.exp2perm) {
        if (k < p.K) o = p.exp2perm[r * p.K + k];
        else o = p.meta[2] >= 0 ? p.meta[2] + r : -1;
      }
      if (o < 0 || o >= p.cap_rows) continue;
      int8_t* dst = p.q + o * p.ldq;
      if (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int c = j * step + lane * 16;
          if (c < p.cols) put16(dst + c, p.cols - c, w[j]);
        }
      } else {
        for (int c = lane * 16; c < p.cols; c += step) {
          load16<SRC>(p, r, c, v[0]);
          w[0] = encode16(s, v[0]);
          put16(dst + c, p.cols - c, w[0]);
        }
      }
      if (lane == 0) p.scale[o] = s.scale;
    }
  }
}

// ============================================================ products
// Tiles.  The MMA's M is 128 weight channels and its N the tokens (16 to 256 in steps of 16), so that a decode batch
// or an expert's few rows cost what they are and not 128 rows: the weights, which bound those shapes, stream through
// at full rate.  A stage is 128 K bytes (one swizzle atom) of both operands in an mbarrier ring; rows and K past the
// ends are zero-filled by the loads.  Roles (320 threads): warp 0 lane 0 issues the TMA boxes, warp 1 lane 0 the MMAs
// into one of two TMEM accumulators, warps 2-9 scale and store the other.  Every wait is bounded and reports.
//
// With few units a cluster of `splits` blocks shares one unit, each a part of K; the parts' int32 sums meet in shared
// memory (each block adds every split-th token of all blocks' tiles through the cluster), so a decode step keeps all
// SMs loading weights without a workspace or a second launch.
namespace i8 {
constexpr int BM = 128;                  // weight channels a unit
constexpr int BK = 128;                  // K bytes a stage
constexpr int W_BYTES = BM * BK;
constexpr int RING_BYTES = 192 * 1024;
constexpr int MAX_STAGES = 10;
constexpr int SMEM_BYTES = RING_BYTES + 1024 + 512;
constexpr int EPI_WARPS = 8;
constexpr int WARPS = 2 + EPI_WARPS;
constexpr int THREADS = 32 * WARPS;
}  // namespace i8

struct Int8Params {
  const float* sx;         // [T] (grouped: permuted rows)
  const float* sw;         // [experts * N]
  void* out;               // [T, ldo] bf16 or f32
  long long ldo;
  int f32_out;
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
__device__ __forceinline__ Int8Unit int8_unit(const Int8Params& p, int u) {
  Int8Unit w;
  const int c = u / p.n_tiles;
  w.ch0 = (u % p.n_tiles) * i8::BM;
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
__device__ __forceinline__ u32 cluster_rank() {
  u32 r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
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

__device__ __forceinline__ void int8_store(const Int8Params& p, long long row, int ch, float v) {
  if (p.f32_out) reinterpret_cast<float*>(p.out)[row * p.ldo + ch] = v;
  else reinterpret_cast<bf16*>(p.out)[row * p.ldo + ch] = __float2bfloat16_rn(v);
}

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

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 1) {
    tmem_alloc(tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], EPI_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmX);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const u32 tmem_base = *tmem_slot;
  const int units = (p.cta_batch ? min(p.meta[0], p.max_ctas) : p.t_tiles) * p.n_tiles;
  // the block's part of K (all of it without a cluster)
  const int rank = p.splits > 1 ? (int)cluster_rank() : 0;
  const int k0 = (int)((long long)rank * p.kstages / p.splits);
  const int k1 = (int)((long long)(rank + 1) * p.kstages / p.splits);
  const int first = blockIdx.x / p.splits, stride = gridDim.x / p.splits;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer
      int stage = 0;
      u32 phase = 0;
      u32 armed = 0;  // fills issued; stage s holds the last of them with index = s mod stages
      for (int u = first; u < units && !*abort_flag; u += stride) {
        const Int8Unit w = int8_unit(p, u);
        if (!w.valid) {
          report_error(p.err, ERR_BAD_TABLE, 0xD00u);
          continue;
        }
        const int boxes = (w.n + p.xbox - 1) / p.xbox;
        const u32 tx = (u32)(W_BYTES + boxes * p.xbox * BK);
        const int wrow = w.e * p.N + w.ch0;
        for (int ks = k0; ks < k1; ++ks) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.err, 0xD10u)) break;
          uint8_t* st = smem + stage * p.stage_bytes;
          mbar_arrive_expect_tx(&full[stage], tx);
          ++armed;
          tma_load_2d(st, &tmW, &full[stage], ks * BK, wrow);
          for (int i = 0; i < boxes; ++i)
            tma_load_2d(st + W_BYTES + i * p.xbox * BK, &tmX, &full[stage], ks * BK, w.row0 + i * p.xbox);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // every fill has landed before the block may exit
      for (u32 s = 0; s < (u32)p.stages && s < armed; ++s)
        mbar_wait(&full[s], ((armed - 1 - s) / (u32)p.stages) & 1u, nullptr, p.err, 0xD20u, 100000000ull);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ------------------------------------------------ MMA issuer
      int stage = 0, buf = 0;
      u32 phase = 0;
      u32 acc_phase[2] = {0u, 0u};
      bool issued = false;
      for (int u = first; u < units && !*abort_flag; u += stride) {
        const Int8Unit w = int8_unit(p, u);
        if (!w.valid) continue;
        if (!mbar_wait(&acc_empty[buf], acc_phase[buf] ^ 1u, abort_flag, p.err, 0xD30u)) break;
        tc_fence_after();
        const u32 idesc = i8_idesc(BM, (w.n + 15) & ~15);
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
          for (int kk = 0; kk < BK / 32; ++kk)
            i8_mma(d, sdesc_k_sw128(st + kk * 32), sdesc_k_sw128(st + W_BYTES + kk * 32), idesc,
                   ks != k0 || kk != 0);
          tc_commit(&empty[stage]);
          issued = true;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit(&acc_full[buf]);
        acc_phase[buf] ^= 1u;
        buf ^= 1;
      }
      if (issued) {
        tc_commit(drain);
        mbar_wait(drain, 0, nullptr, p.err, 0xD50u, 100000000ull);
      }
    }
  } else {
    // ------------------------------------------------ epilogue (warps 2..9): a lane is a channel, columns are tokens;
    // the two warps of a sub-partition take 16 tokens in turn
    const int sub = warp & 3;
    const u32 lane_base = (u32)(sub * 32) << 16;
    int* red = reinterpret_cast<int*>(smem);
    u32 acc_phase[2] = {0u, 0u};
    int buf = 0;
    for (int u = first; u < units && !*abort_flag; u += stride) {
      const Int8Unit w = int8_unit(p, u);
      if (!w.valid) continue;
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], acc_phase[buf], abort_flag, p.err, 0xD60u))) break;
      tc_fence_after();
      const int ch = w.ch0 + sub * 32 + lane;
      const float swc = ch < p.N ? p.sw[(long long)w.e * p.N + ch] : 0.f;
      for (int c = ((warp - 2) >> 2) * 16; c < w.n; c += 32) {
        u32 v[16];
        i8_ld16(tmem_base + lane_base + (u32)(buf * p.bn + c), v);
        const float sx = lane < 16 && c + lane < w.n ? p.sx[w.row0 + c + lane] : 0.f;
        tmem_wait_ld();
        if (p.splits > 1) {
#pragma unroll
          for (int j = 0; j < 16; ++j) red[(c + j) * BM + sub * 32 + lane] = (int)v[j];
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float s = __shfl_sync(0xffffffffu, sx, j);
            if (ch < p.N && c + j < w.n)
              int8_store(p, (long long)w.row0 + c + j, ch, __int2float_rn((int)v[j]) * s * swc);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
      acc_phase[buf] ^= 1u;
      buf ^= 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, p.tmem_cols);
  }
  if (p.splits > 1) {
    // one unit a cluster: the parts of K meet
    const Int8Unit w = int8_unit(p, first);
    const u32 red = smem_u32(smem);
    cluster_sync();
    for (int t = warp * p.splits + rank; t < w.n; t += WARPS * p.splits) {
      int4 a = make_int4(0, 0, 0, 0);
      for (int r = 0; r < p.splits; ++r) {
        const int4 b = ld_cluster_v4(red + (u32)(t * BM + lane * 4) * 4, (u32)r);
        a.x += b.x;
        a.y += b.y;
        a.z += b.z;
        a.w += b.w;
      }
      const int ch = w.ch0 + lane * 4;
      const float s = p.sx[w.row0 + t];
      const int q[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (ch + i < p.N) int8_store(p, (long long)w.row0 + t, ch + i, __int2float_rn(q[i]) * s * p.sw[ch + i]);
    }
    cluster_sync();  // no block leaves while another reads its part
  }
}

}  // namespace k3
