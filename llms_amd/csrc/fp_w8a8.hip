// fp_w8a8.hip — projections in 8-bit integers: weights with a scale for each output,
// activations with one for each token.
//
//   top[m]  = max_k |x[m][k]|
//   c[m][k] = rne(127 x[m][k] / top[m]),  sx[m] = top[m] / 127
//   y[m][n] = sx[m] sw[n] sum_k c[m][k] q[n][k]
//
// The sum is an exact int32 (|sum| <= 127^2 K, K <= 2^17), so no order of it and no split
// of k changes a result. It is rounded to fp32, multiplied by the two scales and, once,
// rounded to bf16 (gate-up: silu(g) u of the fp32 values). A token with an infinity or a
// NaN has the scale NaN, and so has every output of it.
//
// Codes without a division per element: with r = 127 / top rounded up to fp32, c is x r rounded
// to a whole number in one fma. The quotient 127 x / top of two bf16 is a tie of that rounding or at least
// 2^-17 of itself away from one (254 a - (2 c + 1) b 2^d is a whole number, a and b under 256), and
// x r is off by 2^-23 of itself: only ties matter. 127 divides 254 a, so it divides 2 c + 1 (then c + 1/2
// is 63.5, whose even neighbour, 64, the excess of r leads to as well) or b (then top is 254
// times a power of two, r exact and the tie rounded as one).
//
//   - w8a8_prep_kernel: tokens into codes in the workspace, rows of whole 128 (zeros behind K).
//   - w8a8_rows_kernel: up to 16 tokens, 32 on narrow weights with long rows.
//   - w8a8_general_kernel: more tokens, weight rows of any alignment.
#include "fp_common.h"
#include "fp_launch.h"
#include "fp_norm.h"

namespace fp {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 128;  // inputs of a k-step: one cache line of a weight row

// D(16x16, int32) += A(16x64) * B(64x16): lane l supplies row (A) and column (B) l % 16, 16
// consecutive k of the 64 from 16 (l / 16) on; D lane l holds rows 4 (l / 16) + r, column l % 16.
__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// Between MFMAs and the first reads of their sums, where branches lie between them: the
// wait states in so many instructions, which the compiler counts along straight code only. (The empty
// statements keep the products before and the reads behind.)
template <int N>
__device__ __forceinline__ void settle(i32x4 (&acc)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(acc[i]));
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(acc[i]));
}

// ---- tokens into codes --------------------------------------------------------

// What turns a token's values into codes, c = rne(x up r), and the token's scale. r is
// 127 / (top up) rounded up: up to 2^-23 of it too much (see the file's head). up is 1 but
// for tops so small that r would not be finite.
struct RowCode {
  float up, r, s;
};
// top: max |x| as the bits of a bf16 without its sign (an infinity or a NaN: 0x7f80 or more)
__device__ __forceinline__ RowCode row_code(uint32_t top) {
  const float t = __uint_as_float(top << 16);
  if (top >= 0x7f80u) return {1.f, 0.f, __uint_as_float(0x7fc00000u)};
  const float up = top < (7u << 7) ? 0x1p66f : 1.f;  // tops under 2^-120
  float r = top ? 127.f / (t * up) : 0.f;
  if (fmaf(r, t * up, -127.f) < 0.f && top) r = __uint_as_float(__float_as_uint(r) + 1);
  return {up, r, t / 127.f};
}
// The code in the low byte (the others: anything).
__device__ __forceinline__ uint32_t code_of(float x, float r) {
  return __float_as_uint(fmaf(x, r, 12582912.f));  // 1.5 2^23: rne into the low bits
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                               0x05040100u);
}
// Eight packed bf16 as eight codes.
__device__ __forceinline__ u32x2 codes8(u32x4 v, RowCode c) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) x[2 * j] = __uint_as_float(v[j] << 16), x[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
  if (c.up != 1.f) {  // one branch for the whole workgroup
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= c.up;
  }
  uint32_t b[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = code_of(x[e], c.r);
  return u32x2{pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7])};
}
// The larger of top and the eight magnitudes.
__device__ __forceinline__ uint32_t top8(u32x4 v, uint32_t top) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = v[j] & 0x7fffu, hi = (v[j] >> 16) & 0x7fffu;
    const uint32_t m = lo > hi ? lo : hi;
    top = top > m ? top : m;
  }
  return top;
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
  return v > o ? v : o;
}
// Max over a wave (the steps of wave_sum).
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<0x140>(dpp_max<0x141>(dpp_max<0x4e>(dpp_max<0xb1>(v))));
  uint32_t m = 0;
#pragma unroll
  for (int l = 0; l < kWave; l += 16) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)v, l);
    m = m > o ? m : o;
  }
  return m;
}
// Max over a workgroup of NT threads. red: NT / 64 words of LDS.
template <int NT>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / kWave; ++w) v = v > red[w] ? v : red[w];
  return v;
}
__device__ __forceinline__ float sumsq8(u32x4 v, float s) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float lo = bf16_bits_to_f32(v[j] & 0xffffu), hi = bf16_bits_to_f32(v[j] >> 16);
    s += __fmul_rn(lo, lo);
    s += __fmul_rn(hi, hi);
  }
  return s;
}

// One token per workgroup. NV > 0: its chunks of eight in registers (K <= 2048 NV), else read
// three times. NORM: of RMSNorm(x) (rounded to bf16 as the norm kernels do). Bound by memory: 4096 tokens of 4096.
template <int NV, bool NORM>
__global__ __launch_bounds__(256) void w8a8_prep_kernel(W8A8Args a) {
  __shared__ float fred[4];
  __shared__ uint32_t ured[4];
  const int64_t m = blockIdx.x;
  const uint16_t* row = a.x + m * a.ldx;
  int8_t* out = a.xq + m * a.Kp;
  const int64_t K = a.K;
  if constexpr (NV > 0) {
    u32x4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t k = ((int64_t)threadIdx.x + 256 * i) * 8;
      v[i] = k < K ? load_bf16x8<false>(row, k, K) : u32x4{0u, 0u, 0u, 0u};
    }
    if constexpr (NORM) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) s = sumsq8(v[i], s);
      const float r = rms_scale(block_sum<256>(s, fred), K, a.eps);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int64_t k = ((int64_t)threadIdx.x + 256 * i) * 8;
        if (k < K) v[i] = norm_bf16x8(v[i], load_bf16x8<false>(a.gamma, k, K), r);
      }
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) top = top8(v[i], top);
    const RowCode c = row_code(block_max<256>(top, ured));
    if (threadIdx.x == 0) a.sx[m] = c.s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t k = ((int64_t)threadIdx.x + 256 * i) * 8;
      if (k < a.Kp) *reinterpret_cast<u32x2*>(out + k) = codes8(v[i], c);
    }
  } else {
    float r = 1.f;
    if constexpr (NORM) {
      float s = 0.f;
      for (int64_t k = (int64_t)threadIdx.x * 8; k < K; k += 2048) s = sumsq8(load_bf16x8<false>(row, k, K), s);
      r = rms_scale(block_sum<256>(s, fred), K, a.eps);
    }
    const auto chunk = [&](int64_t k) -> u32x4 {
      u32x4 v = load_bf16x8<false>(row, k, K);
      if constexpr (NORM) v = norm_bf16x8(v, load_bf16x8<false>(a.gamma, k, K), r);
      return v;
    };
    uint32_t top = 0;
    for (int64_t k = (int64_t)threadIdx.x * 8; k < K; k += 2048) top = top8(chunk(k), top);
    const RowCode c = row_code(block_max<256>(top, ured));
    if (threadIdx.x == 0) a.sx[m] = c.s;
    for (int64_t k = (int64_t)threadIdx.x * 8; k < a.Kp; k += 2048)
      *reinterpret_cast<u32x2*>(out + k) = codes8(k < K ? chunk(k) : u32x4{0u, 0u, 0u, 0u}, c);
  }
}

// ---- epilogue --------------------------------------------------------------------

// One output of its sums: s and, for gate-up, of the up weight.
__device__ __forceinline__ float scaled(int s, float sw, float sx) { return (float)s * sw * sx; }

// ---- weights -----------------------------------------------------------------------

constexpr uint32_t kOut = 0x7ffffff0u;  // a buffer offset past every buffer: reads 0, and nothing of memory

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, int64_t bytes) {
  constexpr int kRsrcFlags = 0x00020000;  // raw buffer, 32-bit data format
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, kRsrcFlags);
}

// Weight rows from row n0 on as a buffer: what lies behind a row's end meets codes of zero, behind the
// weight's end it reads as zero. Rows off a 4-byte boundary are read from the boundary before,
// one dword more, and shifted: a load of 16 bytes at any address takes twice the time (9700 x 2541 at
// 5 tokens 22.0 us, at an even stride of 2548 10.7).
struct WeightRows {
  const int8_t* base;  // ALIGNED: row n0; else the boundary before it
  int64_t bytes;
  template <bool ALIGNED>
  __device__ __forceinline__ static WeightRows at(const int8_t* q, int64_t ld, int64_t n0, int64_t N, int64_t K) {
    const int8_t* p = q + n0 * ld;
    int64_t b = (N - 1 - n0) * ld + K;
    if constexpr (!ALIGNED) {
      const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(p) & 3);
      p -= d;
      b += d;
    }
    b = (b + 3) & ~(int64_t)3;  // (a dword that the range ends inside of would read as zero)
    const int64_t far = kOut;
    return {p, b < far ? b : far};
  }
};
// Sixteen bytes that lie `sh` bytes behind v's first, with the dword behind v.
__device__ __forceinline__ u32x4 shifted(u32x4 v, uint32_t next, uint32_t sh) {
  return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], sh), __builtin_amdgcn_alignbyte(v[2], v[1], sh),
               __builtin_amdgcn_alignbyte(v[3], v[2], sh), __builtin_amdgcn_alignbyte(next, v[3], sh)};
}
// The first dword of the next lane (of 16).
__device__ __forceinline__ uint32_t next_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x101, 0xf, 0xf, false);  // row_shl:1
}

// ---- few tokens ---------------------------------------------------------------------
//
// Bound by the weights' stream. The product's 16 A rows are R = 16 / C weight rows times C pieces of
// their k, its 16 B columns TOK = 16 / C tokens times the same pieces: of the sums, those where row and
// column have one piece count, and their sum over the pieces is the output. So C lanes in turn read one
// row's bytes (64 C of a row per instruction, in 16-byte chunks g C + c by lane group g and piece c), as
// the address unit wants them: with one row per lane (C = 1) it takes a request per lane. C is the
// largest that leaves columns for the tokens.
//
// A workgroup has 16 weight rows (gate-up: 8 of each): its four waves split them, 2 R rows each as two
// blocks, and what is left of the waves splits k. A wave has S steps in flight; every load is
// issued without a branch (past the end through an empty buffer), so that their count is known and
// none waits for another.
// QM > 0: the codes of up to QM tokens are made here, by every workgroup, into LDS, while the first
// weights are in flight (NV chunks of eight per thread and token); else they are read from the
// workspace (L2) as the weights are.
template <int C, bool GATEUP, bool ALIGNED, int QM, int NV, int TG = 1>
__global__ __launch_bounds__(256, 3) void w8a8_rows_kernel(W8A8Args a) {
  constexpr int S = 4, R = 16 / C, TOK = 16 / C;
  constexpr int WR = 8 / R, WK = 4 / WR;  // waves over rows and over k
  constexpr int KS = 64 * C;              // a row's bytes per step
  constexpr int TS = KS + 16 * C;         // a token's in LDS: the tokens' chunks fall on distinct banks
  static_assert(QM <= TOK && 8 % R == 0 && WR * WK == 4, "tokens and waves");
  extern __shared__ __attribute__((aligned(1024))) char lds[];  // QM: [steps][TOK][TS] codes
  __shared__ int red[TG][4][2][R][16];  // [group][wave][block][row][column]
  __shared__ float fred[QM ? QM : 1][4];
  __shared__ uint32_t ured[QM ? QM : 1][4];
  __shared__ float ssx[TOK * TG];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wr = wave / WK, wk = wave % WK;
  const int li = lane & 15, grp = lane >> 4, c = li % C, g = li / C;  // g: row of a block, or token
  const int nk = (int)((a.K + KS - 1) / KS);
  const int64_t n0 = (int64_t)blockIdx.x * (GATEUP ? 8 : 16);  // first output
  const int at = (grp * C + c) * 16;

  // this lane's row of each block: its offset from the workgroup's first row
  const WeightRows rows[2] = {WeightRows::at<ALIGNED>(a.q0, a.ldq0, n0, a.N, a.K),
                              GATEUP ? WeightRows::at<ALIGNED>(a.q1, a.ldq1, n0, a.N, a.K) : WeightRows{}};
  uint32_t off[2], sh[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int w = GATEUP ? i : 0;
    int64_t n = (GATEUP ? wr : 2 * wr + i) * R + g;
    if (n0 + n >= a.N) n = a.N - 1 - n0;  // not stored
    const int8_t* p = (w ? a.q1 : a.q0) + (n0 + n) * (w ? a.ldq1 : a.ldq0) + at;
    sh[i] = ALIGNED ? 0 : (uint32_t)(reinterpret_cast<uintptr_t>(p) & 3);
    off[i] = (uint32_t)(p - sh[i] - rows[w].base);
  }
  // QM = 0: this lane's codes (tokens past the last: its codes, in columns that are not stored)
  uint32_t xoff[TG];
#pragma unroll
  for (int p = 0; p < TG; ++p) xoff[p] = (uint32_t)((p * TOK + g < a.M ? p * TOK + g : a.M - 1) * a.Kp) + at;
  struct Chunk {
    u32x4 v;
    uint32_t next;  // (unaligned rows: of the last of a run of chunks, else the next lane has it)
  };
  const auto load1 = [&](Chunk (&v)[2], u32x4 (&x)[TG], int k) {
    const uint32_t o = k < nk ? (uint32_t)k * KS : 0u;
    if constexpr (QM == 0) {
#pragma unroll
      for (int p = 0; p < TG; ++p)
        x[p] = __builtin_amdgcn_raw_buffer_load_b128(make_rsrc(a.xq, k < nk ? a.M * a.Kp : 0), xoff[p], o, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const WeightRows& w = rows[GATEUP ? i : 0];
      const auto r = make_rsrc(w.base, k < nk ? w.bytes : 0);
      // (the step is in the lanes' offset, which every description of the range check has in it)
      v[i].v = __builtin_amdgcn_raw_buffer_load_b128(r, off[i] + o, 0, 2);  // non-temporal
      if constexpr (!ALIGNED)
        v[i].next = __builtin_amdgcn_raw_buffer_load_b32(r, c == C - 1 ? off[i] + o + 16 : kOut, 0, 0);
    }
  };
  const auto weight = [&](const Chunk& v, int i) -> u32x4 {
    if constexpr (ALIGNED) return v.v;
    const uint32_t n = next_lane(v.v[0]);
    return shifted(v.v, c == C - 1 ? v.next : n, sh[i]);
  };
  Chunk v[S][2];
  u32x4 xv[S][TG];
  // The tokens' loads (and the norm weight's) go out before the weights': loads return in order.
  // Whole chunks (K is a multiple of 8 here), those past the end from the row's start and not used.
  u32x4 x[QM ? QM : 1][NV], gm[NV];
  if constexpr (QM > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t k = ((int64_t)threadIdx.x + 256 * i) * 8, at_k = k < a.K ? k : 0;
#pragma unroll
      for (int m = 0; m < QM; ++m) x[m][i] = ld16_any(a.x + (m < a.M ? m : 0) * a.ldx + at_k);
      gm[i] = ld16_any((a.gamma ? a.gamma : a.x) + at_k);
    }
  }
#pragma unroll
  for (int u = 0; u < S; ++u) load1(v[u], xv[u], wk + WK * u);

  if constexpr (QM > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (((int)threadIdx.x + 256 * i) * 8 >= a.K)
#pragma unroll
        for (int m = 0; m < QM; ++m) x[m][i] = u32x4{0u, 0u, 0u, 0u};
    if (a.gamma) {
#pragma unroll
      for (int m = 0; m < QM; ++m) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) s = sumsq8(x[m][i], s);
        s = wave_sum(s);
        if (lane == 0) fred[m][wave] = s;
      }
      __syncthreads();
      float r[QM];
#pragma unroll
      for (int m = 0; m < QM; ++m) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) t += fred[m][w];
        r[m] = rms_scale(t, a.K, a.eps);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int m = 0; m < QM; ++m) {
          x[m][i] = norm_bf16x8(x[m][i], gm[i], r[m]);
          if (((int)threadIdx.x + 256 * i) * 8 >= a.K) x[m][i] = u32x4{0u, 0u, 0u, 0u};  // (0 inf)
        }
    }
#pragma unroll
    for (int m = 0; m < QM; ++m) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) top = top8(x[m][i], top);
      top = wave_max(top);
      if (lane == 0) ured[m][wave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < QM; ++m) {
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = top > ured[m][w] ? top : ured[m][w];
      const RowCode rc = row_code((uint32_t)__builtin_amdgcn_readfirstlane((int)top));
      if (threadIdx.x == 0) ssx[m] = rc.s;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = (int)(threadIdx.x + 256 * i) * 8;
        if (k < nk * KS) *reinterpret_cast<u32x2*>(lds + (k / KS * QM + m) * TS + k % KS) = codes8(x[m][i], rc);
      }
    }
  } else {
    if (threadIdx.x < TOK * TG) ssx[threadIdx.x] = (int)threadIdx.x < a.M ? a.sx[threadIdx.x] : 0.f;
  }
  __syncthreads();

  i32x4 acc[2 * TG];
#pragma unroll
  for (int i = 0; i < 2 * TG; ++i) acc[i] = i32x4{0, 0, 0, 0};
  for (int t = 0; WK * t < nk; t += S) {
#pragma unroll
    for (int u = 0; u < S; ++u) {
      const int k = wk + WK * (t + u);
      if constexpr (QM > 0) {
        const int m = g < QM ? g : 0;
        xv[u][0] = *reinterpret_cast<const u32x4*>(lds + ((k < nk ? k : 0) * QM + m) * TS + at);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32x4 w = weight(v[u][i], i);
#pragma unroll
        for (int p = 0; p < TG; ++p) acc[2 * p + i] = mfma_i8(w, xv[u][p], acc[2 * p + i]);
      }
      load1(v[u], xv[u], k + WK * S);
    }
  }
  settle(acc);

  // Lane (grp, li) holds the products of rows 4 grp .. + 3 with column li: of those, row g' C + c of
  // the column's own piece c, where it is among them.
#pragma unroll
  for (int i = 0; i < 2 * TG; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if ((4 * grp + r) % C == c) red[i / 2][wave][i % 2][(4 * grp + r) / C][li] = acc[i][r];
  __syncthreads();
  const int nout = GATEUP ? 8 : 16;
  for (int i = threadIdx.x; i < nout * TOK * TG; i += 256) {
    const int o = i % nout, m = i / nout;
    const int64_t n = n0 + o;
    if (m >= a.M || n >= a.N) continue;
    const int w0 = GATEUP ? o / R : o / (2 * R), blk = GATEUP ? 0 : (o / R) % 2;
    int s0 = 0, s1 = 0;
#pragma unroll
    for (int w = 0; w < WK; ++w)
#pragma unroll
      for (int p = 0; p < C; ++p) {
        const int col = m % TOK * C + p;
        s0 += red[m / TOK][w0 * WK + w][blk][o % R][col];
        if constexpr (GATEUP) s1 += red[m / TOK][w0 * WK + w][1][o % R][col];
      }
    float y = scaled(s0, a.s0[n], ssx[m]);
    if constexpr (GATEUP) y = silu_mul(y, scaled(s1, a.s1[n], ssx[m]));
    a.y[m * a.ldy + n] = (uint16_t)f32_to_bf16_bits(y);
  }
}

// ---- more tokens, any alignment -----------------------------------------------------
//
// Tiles of BN weight rows x BM tokens, k-steps of 128, four waves of BN / 2 x BM / 2. Operands
// go through registers into LDS (rows of any alignment cannot take the direct way), the next step's
// loads in flight while one is computed. 16-byte chunk c of row r lies at c ^ (r & 7): the eight
// rows that a fragment read touches at once are on distinct banks.
// Bound by the way through registers (two stages of them; four are slower, 36 us against 33). 64 weight rows and
// 128 tokens (us, 128 x 64 | 128 x 128 | this: 9700 x 2541 at 64 tokens 22 | 26 | 19, at 300 31 | 29 | 27, at 2000
// 132 | 95 | 108; 2600 x 4097 at 300 31 | 37 | 26); with a column tile's workgroups spread over the XCDs 36 at 300.
template <int BN, int BM, bool GATEUP>
__global__ __launch_bounds__(256, 2) void w8a8_general_kernel(W8A8Args a) {
  constexpr int FN = BN / 32, FM = BM / 32;       // MFMA blocks per wave
  constexpr int NW = BN * 8 / 256, NX = BM * 8 / 256;  // chunks per thread and step
  constexpr int COLS = GATEUP ? BN / 2 : BN;
  static_assert(!GATEUP || FN % 2 == 0, "whole pairs of gate and up blocks per wave");
  __shared__ __attribute__((aligned(1024))) char sW[2][BN * kStep];
  __shared__ __attribute__((aligned(1024))) char sX[2][BM * kStep];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wn = wave >> 1, wm = wave & 1, li = lane & 15, grp = lane >> 4;
  const int64_t m0 = (int64_t)(blockIdx.x / 8) * BM, c0 = ((int64_t)blockIdx.y * 8 + blockIdx.x % 8) * COLS;
  if (c0 >= a.N) return;
  const int nk = (int)((a.K + 2 * kStep - 1) / (2 * kStep)) * 2;  // an even count: codes of zero behind K

  const WeightRows rows[2] = {WeightRows::at<false>(a.q0, a.ldq0, c0, a.N, a.K),
                              GATEUP ? WeightRows::at<false>(a.q1, a.ldq1, c0, a.N, a.K) : WeightRows{}};
  uint32_t woff[NW], sh[NW];
  const int8_t* xb[NX];
  const int ch = threadIdx.x % 8;
  const auto is_up = [&](int i) { return GATEUP && ((wave * 8 + 32 * i) & 16) != 0; };  // of the wave's eight rows
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int r = threadIdx.x / 8 + 32 * i;
    const bool up = is_up(i);
    int64_t n = GATEUP ? c0 + (r / 32) * 16 + r % 16 : c0 + r;
    if (n >= a.N) n = a.N - 1;  // not stored
    const int8_t* p = (up ? a.q1 : a.q0) + n * (up ? a.ldq1 : a.ldq0) + ch * 16;
    sh[i] = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 3);
    woff[i] = (uint32_t)(p - sh[i] - (up ? rows[1].base : rows[0].base));
  }
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    int64_t m = m0 + threadIdx.x / 8 + 32 * i;
    if (m >= a.M) m = a.M - 1;
    xb[i] = a.xq + m * a.Kp + ch * 16;
  }
  struct Step {
    u32x4 w[NW], x[NX];
    uint32_t next[NW];  // of a row's last chunk (of the others the next lane has it)
  };
  const auto load = [&](Step& v, int k) {  // (past the last step: at its place, and not used)
    k = k < nk ? k : nk - 1;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const auto r = make_rsrc(is_up(i) ? rows[1].base : rows[0].base, is_up(i) ? rows[1].bytes : rows[0].bytes);
      const uint32_t o = woff[i] + (uint32_t)k * kStep;  // (in the lanes' offset: the range check)
      v.w[i] = __builtin_amdgcn_raw_buffer_load_b128(r, o, 0, 0);
      v.next[i] = __builtin_amdgcn_raw_buffer_load_b32(r, ch == 7 ? o + 16 : kOut, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NX; ++i) v.x[i] = ld16(xb[i] + (int64_t)k * kStep);
  };
  const auto store = [&](Step& v, int st) {
    const int r = threadIdx.x / 8, o = (ch ^ (r & 7)) * 16;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const uint32_t n = next_lane(v.w[i][0]);
      *reinterpret_cast<u32x4*>(sW[st] + (r + 32 * i) * kStep + o) = shifted(v.w[i], ch == 7 ? v.next[i] : n, sh[i]);
    }
#pragma unroll
    for (int i = 0; i < NX; ++i) *reinterpret_cast<u32x4*>(sX[st] + (r + 32 * i) * kStep + o) = v.x[i];
  };
  i32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  const int ra = wn * (BN / 2) + li, rb = wm * (BM / 2) + li;
  const auto compute = [&](int st) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 fa[FN], fb[FM];
#pragma unroll
      for (int i = 0; i < FN; ++i)
        fa[i] = *reinterpret_cast<const u32x4*>(sW[st] + (ra + 16 * i) * kStep + (((4 * h + grp) ^ (ra & 7)) * 16));
#pragma unroll
      for (int j = 0; j < FM; ++j)
        fb[j] = *reinterpret_cast<const u32x4*>(sX[st] + (rb + 16 * j) * kStep + (((4 * h + grp) ^ (rb & 7)) * 16));
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = mfma_i8(fa[i], fb[j], acc[i][j]);
    }
  };
  // step k from LDS stage k % 2, step k + 1 in registers, step k + 2's loads in flight
  Step v0, v1;
  load(v0, 0);
  load(v1, 1);
  store(v0, 0);
  __syncthreads();
  for (int k = 0; k < nk; k += 2) {
    load(v0, k + 2);
    compute(0);
    store(v1, 1);
    __syncthreads();
    load(v1, k + 3);
    compute(1);
    store(v0, 0);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < FN; ++i) settle(acc[i]);
  // every scale before the first store: a load between stores and branches would be waited for by itself
  f32x4 sw[FN];
  float sx[FM];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    const int64_t n = c0 + (GATEUP ? wn * (COLS / 2) + (i / 2) * 16 : wn * (BN / 2) + i * 16) + 4 * grp;
#pragma unroll
    for (int r = 0; r < 4; ++r) sw[i][r] = (GATEUP && (i & 1) ? a.s1 : a.s0)[n + r < a.N ? n + r : a.N - 1];
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int64_t m = m0 + wm * (BM / 2) + 16 * j + li;
    sx[j] = a.sx[m < a.M ? m : a.M - 1];
  }
  const bool y8 = a.ldy % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 7) == 0;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int64_t m = m0 + wm * (BM / 2) + 16 * j + li;
#pragma unroll
    for (int i = 0; i < FN; i += GATEUP ? 2 : 1) {
      const int64_t n = c0 + (GATEUP ? wn * (COLS / 2) + (i / 2) * 16 : wn * (BN / 2) + i * 16) + 4 * grp;
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[r] = scaled(acc[i][j][r], sw[i][r], sx[j]);
        if constexpr (GATEUP) y[r] = silu_mul(y[r], scaled(acc[i + 1][j][r], sw[i + 1][r], sx[j]));
      }
      if (m >= a.M || n >= a.N) continue;
      uint16_t* p = a.y + m * a.ldy + n;
      const u32x2 h = {pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
      if (y8 && n + 3 < a.N) {
        *reinterpret_cast<u32x2*>(p) = h;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < a.N) p[r] = (uint16_t)(h[r / 2] >> (16 * (r & 1)));
      }
    }
  }
}

template <bool NORM>
int launch_prep(const W8A8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)a.M), block(256);
  if (a.Kp <= 2048) hipLaunchKernelGGL((w8a8_prep_kernel<1, NORM>), grid, block, 0, s, a);
  else if (a.Kp <= 4096) hipLaunchKernelGGL((w8a8_prep_kernel<2, NORM>), grid, block, 0, s, a);
  else if (a.Kp <= 10240) hipLaunchKernelGGL((w8a8_prep_kernel<5, NORM>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((w8a8_prep_kernel<0, NORM>), grid, block, 0, s, a);
  return (int)hipGetLastError();
}

template <bool GATEUP>
int launch_general(const W8A8Args& a, hipStream_t s) {
  constexpr int BN = 64, BM = 128;
  // (a column tile's workgroups are eight apart: on one XCD, whose cache then has its weights once)
  const int64_t cols = GATEUP ? BN / 2 : BN;
  const dim3 grid((unsigned)((a.M + BM - 1) / BM * 8), (unsigned)((a.N + 8 * cols - 1) / (8 * cols)));
  hipLaunchKernelGGL((w8a8_general_kernel<BN, BM, GATEUP>), grid, dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

// The kernel for few tokens, and whether it makes the codes itself.
// Up to 16 tokens; up to 32 with few outputs and a long k, where the tiles take a split of k (us, this
// kernel / the tiles at 17 and 32 tokens: 4B down 14.3, 16.5 / 17.3, 18.1, 8B down 18.6, 22.3 / 23.6, 24.6, 4B o
// 9.7, 10.4 / 12.0, 12.7; but 8B QKV 13.1, 14.8 / 15.7, 14.9, 4B gate-up 22.2, 24.1 / 18.9, 19.1).
inline bool rows_take(int64_t M, int64_t N, int64_t K, bool gateup) {
  return M <= 16 || (M <= 32 && K >= 4096 && N * (gateup ? 2 : 1) <= 4096);
}

inline bool rows_quantise(int64_t M, int64_t K) { return K % 8 == 0 && ((M == 1 && K <= 12288) || (M <= 4 && K <= 4096)); }

template <int C, bool GATEUP, bool ALIGNED, int QM, int NV, int TG = 1>
int launch_rows_cfg(const W8A8Args& a, hipStream_t s) {
  constexpr int64_t KS = 64 * C, TS = KS + 16 * C, per = GATEUP ? 8 : 16;
  hipLaunchKernelGGL((w8a8_rows_kernel<C, GATEUP, ALIGNED, QM, NV, TG>), dim3((unsigned)((a.N + per - 1) / per)), dim3(256),
                     (size_t)((a.K + KS - 1) / KS * QM * TS), s, a);
  return (int)hipGetLastError();
}
template <bool GATEUP, bool ALIGNED>
int launch_rows_al(const W8A8Args& a, hipStream_t s) {
  if (rows_quantise(a.M, a.K)) {
    if (a.M == 1 && a.K <= 4096) return launch_rows_cfg<8, GATEUP, ALIGNED, 1, 2>(a, s);
    if (a.M == 1) return launch_rows_cfg<8, GATEUP, ALIGNED, 1, 6>(a, s);
    if (a.M == 2) return launch_rows_cfg<8, GATEUP, ALIGNED, 2, 2>(a, s);
    return launch_rows_cfg<4, GATEUP, ALIGNED, 4, 2>(a, s);
  }
  if (a.M <= 2) return launch_rows_cfg<8, GATEUP, ALIGNED, 0, 1>(a, s);
  if (a.M <= 4) return launch_rows_cfg<4, GATEUP, ALIGNED, 0, 1>(a, s);
  if (a.M <= 8) return launch_rows_cfg<2, GATEUP, ALIGNED, 0, 1>(a, s);
  if (a.M <= 16) return launch_rows_cfg<2, GATEUP, ALIGNED, 0, 1, 2>(a, s);
  return launch_rows_cfg<2, GATEUP, ALIGNED, 0, 1, 4>(a, s);
}
template <bool GATEUP>
int launch_rows(const W8A8Args& a, bool aligned, hipStream_t s) {
  return aligned ? launch_rows_al<GATEUP, true>(a, s) : launch_rows_al<GATEUP, false>(a, s);
}

inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
// Codes of a token with zeros behind: whole steps of every kernel.
inline int64_t padded(int64_t K) { return (K + 4 * kStep - 1) / (4 * kStep) * (4 * kStep); }
// Whether the prefill tiles take a call: sizes of every operand within their 32-bit offsets.
inline bool tiles_supported(int64_t M, int64_t N, int64_t Kp, int64_t ldq) {
  constexpr int64_t kLim = (int64_t)1 << 31;
  return (N + 256) * ldq < kLim && (M + 256) * Kp < kLim;
}

}  // namespace

int64_t w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K, bool gateup) {
  (void)N, (void)gateup;
  if (rows_quantise(M, K)) return 0;
  // (a weight's row stride and alignment may rule the tiles out: the partials' room is then unused)
  return up256(M * padded(K)) + up256(M * 4) +
         (rows_take(M, N, K, gateup) ? 0 : i8_workspace_bytes(M, N, padded(K), gateup));
}

int launch_w8a8(W8A8Args a, bool gateup, bool aligned, void* ws, hipStream_t s) {
  a.Kp = padded(a.K);
  a.xq = (int8_t*)ws;
  a.sx = (float*)((char*)ws + up256(a.M * a.Kp));
  const bool rows = rows_take(a.M, a.N, a.K, gateup);
  if (rows && rows_quantise(a.M, a.K))
    return gateup ? launch_rows<true>(a, aligned, s) : launch_rows<false>(a, aligned, s);
  const int e = a.gamma ? launch_prep<true>(a, s) : launch_prep<false>(a, s);
  if (e) return e;
  if (rows) return gateup ? launch_rows<true>(a, aligned, s) : launch_rows<false>(a, aligned, s);
  const int64_t ldq = gateup && a.ldq1 > a.ldq0 ? a.ldq1 : a.ldq0;
  if (aligned && tiles_supported(a.M, a.N, a.Kp, ldq)) {
    I8Args t{};
    t.x = (const uint16_t*)a.xq, t.ldx = a.Kp / 2;
    t.w0 = a.q0, t.ldw0 = a.ldq0 / 2, t.w1 = gateup ? a.q1 : nullptr, t.ldw1 = a.ldq1 / 2;
    t.s0 = a.s0, t.s1 = a.s1, t.y = a.y, t.ldy = a.ldy;
    t.M = a.M, t.N = a.N, t.K = a.Kp / 2;
    t.sx = a.sx, t.wbytes = (a.K + 3) & ~(int64_t)3;
    t.ws = (float*)((char*)a.sx + up256(a.M * 4));
    return launch_i8(t, gateup, s);
  }
  return gateup ? launch_general<true>(a, s) : launch_general<false>(a, s);
}

}  // namespace fp
