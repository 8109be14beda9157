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
// Codes without a division per element: the quotient of two bf16 times 127 is a tie of
// rounding or at least 2^-17 of itself away from one (254 a - (2 c + 1) b 2^d is a whole number, a
// and b under 256). x times the rounded 127 / top is within 2^-23, and rounding that to 18
// significant bits moves it by up to 2^-19: a tie comes out exactly, nothing else crosses one.
//
//   - w8a8_prep_kernel: tokens into codes in the workspace, rows of whole 128 (zeros behind K).
//   - w8a8_rows_kernel: up to 16 tokens.
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

// ---- tokens into codes --------------------------------------------------------

// What turns a token's values into codes: c = rne(x up r) with up a power of two that
// keeps 127 / (top up) finite, and the token's scale.
struct RowCode {
  float up, r, s;
};
// top: max |x| as the bits of a bf16 without its sign (an infinity or a NaN: 0x7f80 or more)
__device__ __forceinline__ RowCode row_code(uint32_t top) {
  const float t = __uint_as_float(top << 16);
  if (top >= 0x7f80u) return {0.f, 0.f, __uint_as_float(0x7fc00000u)};
  const float up = top < (67u << 7) ? 0x1p66f : 1.f;  // tops under 2^-60
  return {up, top ? 127.f / (t * up) : 0.f, t / 127.f};
}
// The code in the low byte (the others: anything).
__device__ __forceinline__ uint32_t code_of(float x, RowCode c) {
  const float t = x * c.up * c.r;
  const float snapped = __uint_as_float((__float_as_uint(t) + 0x10u) & ~0x1fu);
  return __float_as_uint(snapped + 12582912.f);  // 1.5 2^23: rne into the low bits
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                               0x05040100u);
}
// Eight packed bf16 as eight codes.
__device__ __forceinline__ u32x2 codes8(u32x4 v, RowCode c) {
  uint32_t b[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    b[2 * j] = code_of(__uint_as_float(v[j] << 16), c);
    b[2 * j + 1] = code_of(__uint_as_float(v[j] & 0xffff0000u), c);
  }
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
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, off);
    v = v > o ? v : o;
  }
  return v;
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
__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.f + __expf(-g)) * u; }

// ---- weights -----------------------------------------------------------------------

// Sixteen bytes shifted down by d bytes (d >= 16: anything).
__device__ __forceinline__ u32x4 bytes_down(u32x4 v, uint32_t d) {
  if (d & 8) v[0] = v[2], v[1] = v[3];
  if (d & 4) v[0] = v[1], v[1] = v[2], v[2] = v[3];
  return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], d), __builtin_amdgcn_alignbyte(v[2], v[1], d),
               __builtin_amdgcn_alignbyte(v[3], v[2], d), v[3] >> (8 * (d & 3))};
}

// Sixteen bytes at offset off of a weight of `last` + 16 bytes, at any alignment: what lies past
// the row meets codes of zero, so only the weight's last byte must not be passed. There the
// load moves back and its bytes down.
__device__ __forceinline__ u32x4 ld_weight(const int8_t* w, int64_t off, int64_t last) {
  if (__builtin_expect(off <= last, 1)) return ld16_any(w + off);
  const int64_t d = off - last;
  return d < 16 ? bytes_down(ld16_any(w + last), (uint32_t)d) : u32x4{0u, 0u, 0u, 0u};
}

// ---- more tokens, any alignment -----------------------------------------------------
//
// Tiles of BN weight rows x BM tokens, k-steps of 128, four waves of BN / 2 x BM / 2. Operands
// go through registers into LDS (rows of any alignment cannot take the direct way), the next step's
// loads in flight while one is computed. 16-byte chunk c of row r lies at c ^ (r & 7): the eight
// rows that a fragment read touches at once are on distinct banks.
template <int BN, int BM, bool GATEUP>
__global__ __launch_bounds__(256) void w8a8_general_kernel(W8A8Args a) {
  constexpr int FN = BN / 32, FM = BM / 32;       // MFMA blocks per wave
  constexpr int NW = BN * 8 / 256, NX = BM * 8 / 256;  // chunks per thread and step
  constexpr int COLS = GATEUP ? BN / 2 : BN;
  static_assert(!GATEUP || FN % 2 == 0, "whole pairs of gate and up blocks per wave");
  __shared__ __attribute__((aligned(1024))) char sW[2][BN * kStep];
  __shared__ __attribute__((aligned(1024))) char sX[2][BM * kStep];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wn = wave >> 1, wm = wave & 1, li = lane & 15, grp = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.x * BM, c0 = (int64_t)blockIdx.y * COLS;
  const int nk = (int)(a.Kp / kStep);

  const int8_t* wb[NW];
  int64_t woff[NW], wlast[NW];
  const int8_t* xb[NX];
  const int ch = threadIdx.x % 8;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int r = threadIdx.x / 8 + 32 * i;
    const bool up = GATEUP && ((r / 16) & 1);
    int64_t n = GATEUP ? c0 + (r / 32) * 16 + r % 16 : c0 + r;
    if (n >= a.N) n = a.N - 1;  // not stored
    const int64_t ld = up ? a.ldq1 : a.ldq0;
    wb[i] = up ? a.q1 : a.q0;
    woff[i] = n * ld + ch * 16;
    wlast[i] = (a.N - 1) * ld + a.K - 16;
  }
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    int64_t m = m0 + threadIdx.x / 8 + 32 * i;
    if (m >= a.M) m = a.M - 1;
    xb[i] = a.xq + m * a.Kp + ch * 16;
  }
  u32x4 vw[NW], vx[NX];
  const auto load = [&](int k) {
#pragma unroll
    for (int i = 0; i < NW; ++i) vw[i] = ld_weight(wb[i], woff[i] + (int64_t)k * kStep, wlast[i]);
#pragma unroll
    for (int i = 0; i < NX; ++i) vx[i] = ld16(xb[i] + (int64_t)k * kStep);
  };
  const auto store = [&](int st) {
    const int r = threadIdx.x / 8, o = (ch ^ (r & 7)) * 16;
#pragma unroll
    for (int i = 0; i < NW; ++i) *reinterpret_cast<u32x4*>(sW[st] + (r + 32 * i) * kStep + o) = vw[i];
#pragma unroll
    for (int i = 0; i < NX; ++i) *reinterpret_cast<u32x4*>(sX[st] + (r + 32 * i) * kStep + o) = vx[i];
  };
  i32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  const int ra = wn * (BN / 2) + li, rb = wm * (BM / 2) + li;
  load(0);
  store(0);
  __syncthreads();
  for (int k = 0; k < nk; ++k) {
    const int st = k & 1;
    if (k + 1 < nk) load(k + 1);
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
    if (k + 1 < nk) store(st ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int64_t m = m0 + wm * (BM / 2) + 16 * j + li;
    if (m >= a.M) continue;
    const float sx = a.sx[m];
#pragma unroll
    for (int i = 0; i < FN; i += GATEUP ? 2 : 1) {
      const int64_t n0 = c0 + (GATEUP ? wn * (COLS / 2) + (i / 2) * 16 : wn * (BN / 2) + i * 16) + 4 * grp;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t n = n0 + r;
        if (n >= a.N) break;
        float y = scaled(acc[i][j][r], a.s0[n], sx);
        if constexpr (GATEUP) y = silu_mul(y, scaled(acc[i + 1][j][r], a.s1[n], sx));
        a.y[m * a.ldy + n] = (uint16_t)f32_to_bf16_bits(y);
      }
    }
  }
}

// Weights of fewer than 16 bytes, which the kernels above could not load from.
template <bool GATEUP>
__global__ __launch_bounds__(64) void w8a8_small_kernel(W8A8Args a) {
  const int64_t i = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (i >= a.M * a.N) return;
  const int64_t m = i / a.N, n = i - m * a.N;
  int g = 0, u = 0;
  for (int64_t k = 0; k < a.K; ++k) {
    const int c = a.xq[m * a.Kp + k];
    g += c * a.q0[n * a.ldq0 + k];
    if constexpr (GATEUP) u += c * a.q1[n * a.ldq1 + k];
  }
  float y = scaled(g, a.s0[n], a.sx[m]);
  if constexpr (GATEUP) y = silu_mul(y, scaled(u, a.s1[n], a.sx[m]));
  a.y[m * a.ldy + n] = (uint16_t)f32_to_bf16_bits(y);
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
  constexpr int BN = 128, BM = 128;
  const int64_t least = (a.N - 1) * (GATEUP && a.ldq1 < a.ldq0 ? a.ldq1 : a.ldq0) + a.K;
  if (least < 16) {
    hipLaunchKernelGGL(w8a8_small_kernel<GATEUP>, dim3((unsigned)((a.M * a.N + 63) / 64)), dim3(64), 0, s, a);
  } else {
    const int64_t cols = GATEUP ? BN / 2 : BN;
    const dim3 grid((unsigned)((a.M + BM - 1) / BM), (unsigned)((a.N + cols - 1) / cols));
    hipLaunchKernelGGL((w8a8_general_kernel<BN, BM, GATEUP>), grid, dim3(256), 0, s, a);
  }
  return (int)hipGetLastError();
}

inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }
inline int64_t padded(int64_t K) { return (K + kStep - 1) / kStep * kStep; }

}  // namespace

int64_t w8a8_workspace_bytes(int64_t M, int64_t N, int64_t K, bool gateup) {
  (void)N, (void)gateup;
  return up256(M * padded(K)) + up256(M * 4);
}

int launch_w8a8(W8A8Args a, bool gateup, bool aligned, void* ws, hipStream_t s) {
  (void)aligned;
  a.Kp = padded(a.K);
  a.xq = (int8_t*)ws;
  a.sx = (float*)((char*)ws + up256(a.M * a.Kp));
  int e = a.gamma ? launch_prep<true>(a, s) : launch_prep<false>(a, s);
  if (e) return e;
  return gateup ? launch_general<true>(a, s) : launch_general<false>(a, s);
}

}  // namespace fp
