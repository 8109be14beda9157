// fp_w4.hip — projections on 4-bit weights with a scale for each group of K.
//
//   s[n][g] = max |w| / 7 over the group, rounded to five significant bits (bf16)
//   q[n][k] = rne(w / s) in -7 .. 7, held as q + 8; byte j of a row: inputs 2j
//             (low half) and 2j + 1
//   y[m][n] = sum_g s[n][g] sum_{k in g} q[n][k] x[m][k]
//
// Five bits of scale and three of code fit the eight of a bf16: q s is exact there,
// so a product on the dequantised weights is the same sum.
//
// w4_rows_kernel (M <= 64): x is the A operand of v_mfma_f32_16x16x32_bf16, the
// codes the B operand: a lane's accumulators belong to one weight row (column lane %
// 16), so its group's scale is one register. Codes become bf16 without a conversion:
// (w & 0x000f000f) | 0x43004300 holds two codes as 128 + (q + 8) exactly; the 136
// too much is taken out by one MFMA per 32 k on a constant B of -136, which starts
// the group's sum and is shared by the column blocks of a wave. A lane's 16 bytes are
// 32 consecutive k of its row; a 4 x 4 transpose of dwords between the four lane groups
// (v_permlane32_swap, v_permlane16_swap) turns them into four operands of 32
// consecutive k each, so any group of 32, 64 or 128 is whole MFMAs. The nibbles of a
// dword come out as k 0 4 1 5 2 6 3 7: x is put into that order on the way in.
//
// Larger calls write the dequantised weights to the workspace and run the bf16 tiles.
#include "fp_common.h"
#include "fp_launch.h"

namespace fp {

namespace {

constexpr uint32_t kOut = 0x7ffffff0u;  // a buffer offset past every buffer: reads 0

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, int64_t bytes) {
  constexpr int kRsrcFlags = 0x00020000;  // raw buffer, 32-bit data format
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, kRsrcFlags);
}

// Eight bf16 into the order of a code dword's nibble pairs: k 0 4 1 5 2 6 3 7.
__device__ __forceinline__ u32x4 nibble_order(u32x4 v) {
  return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
               __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// Eight codes as bf16 128 + (q + 8), in that order.
__device__ __forceinline__ u32x4 codes_bf16(uint32_t w) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
  return v;
}

// Register d of lane group g <-> register g of lane group d.
__device__ __forceinline__ u32x4 transpose_groups(u32x4 v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4{c[0], c[1], d[0], d[1]};
}

// RT blocks of 16 rows of x, NC blocks of 16 weight rows (gate-up: gate and up in
// turn), W waves that take every W-th slab of 128 k, PF slabs in flight per wave.
// ALIGNED: 16-byte aligned weight rows, read through a buffer whose end returns
// zeros, so that every load is issued without a branch (a branch would make the
// compiler wait for all of them); else ordinary loads at any address.
template <int RT, int NC, int GS, bool GATEUP, bool ALIGNED, int W, int PF>
__global__ __launch_bounds__(W * 64) void w4_rows_kernel(W4Args a) {
  constexpr int NG = 128 / GS, FPG = 4 / NG;  // groups of a slab, MFMAs of a group
  constexpr int NB = GATEUP ? NC / 2 : NC;    // 16-column blocks of the output
  __shared__ __attribute__((aligned(16))) f32x4 red[W][RT * NC][64];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, grp = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NB);
  const int slabs = (int)((a.K + 127) / 128), groups = (int)((a.K + GS - 1) / GS);
  const int rowb = (int)((a.K + 1) / 2);  // bytes of a weight row

  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, ((a.M - 1) * a.ldx + (a.K + 7) / 8 * 8) * 2);
  uint32_t xoff[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int64_t m = rt * 16 + li < a.M ? rt * 16 + li : a.M - 1;
    xoff[rt] = (uint32_t)(m * a.ldx * 2) + 16 * grp;
  }
  // each column block's weight and scale rows, through buffers that start at it
  const uint8_t* qb[NC];
  __amdgpu_buffer_rsrc_t qr[NC], sr[NC];
  uint32_t qoff[NC], soff[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const bool up = GATEUP && (c & 1);
    const int64_t r0 = n0 + (GATEUP ? c / 2 : c) * 16;
    const int64_t first = r0 < a.N ? r0 : a.N - 1;
    const int rows = a.N - first < 16 ? (int)(a.N - first) : 16;
    const int row = li < rows ? li : rows - 1;
    const int64_t ldq = up ? a.ldq1 : a.ldq0, lds = up ? a.lds1 : a.lds0;
    qb[c] = (up ? a.q1 : a.q0) + first * ldq;
    qoff[c] = (uint32_t)(row * ldq) + 16 * grp;
    // a whole last chunk of 16 bytes: it lies in one page with its first byte
    qr[c] = make_rsrc(qb[c], (rows - 1) * ldq + (rowb + 15) / 16 * 16);
    sr[c] = make_rsrc((up ? a.s1 : a.s0) + first * lds, ((rows - 1) * lds + groups) * 2);
    soff[c] = (uint32_t)(row * lds * 2);
  }

  u32x4 wq[PF][NC], xf[PF][RT][4];
  uint32_t sc[PF][NC][NG];
  auto load = [&](int p, int slab) {
    const bool in = slab < slabs;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if constexpr (ALIGNED) {
        wq[p][c] = __builtin_amdgcn_raw_buffer_load_b128(qr[c], in ? qoff[c] + slab * 64 : kOut, 0, 0);
      } else {
        wq[p][c] = u32x4{0u, 0u, 0u, 0u};
        const int b = slab * 64 + 16 * grp;
        const uint8_t* src = qb[c] + (qoff[c] - 16 * grp) + b;
        if (b + 16 <= rowb) {
          wq[p][c] = ld16_any(src);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (b + e < rowb) wq[p][c][e / 4] |= (uint32_t)src[e] << (8 * (e % 4));
        }
      }
#pragma unroll
      for (int g = 0; g < NG; ++g)
        sc[p][c][g] = __builtin_amdgcn_raw_buffer_load_b16(
            sr[c], slab * NG + g < groups ? soff[c] + (slab * NG + g) * 2 : kOut, 0, 0);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int f = 0; f < 4; ++f)  // k of the slab: 32 f + 8 grp + ..
        xf[p][rt][f] = __builtin_amdgcn_raw_buffer_load_b128(
            xr, slab * 128 + 32 * f + 8 * grp < a.K ? xoff[rt] + slab * 256 + 64 * f : kOut, 0, 0);
  };

  f32x4 acc[RT][NC];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[rt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr uint32_t kNeg136 = 0xc308c308u;
  const u32x4 bias = {kNeg136, kNeg136, kNeg136, kNeg136};
  auto compute = [&](int p) {
    f32x4 off[RT][NG];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int f = 0; f < 4; ++f) xf[p][rt][f] = nibble_order(xf[p][rt][f]);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        off[rt][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < FPG; ++f) off[rt][g] = mfma16(xf[p][rt][g * FPG + f], bias, off[rt][g]);
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const u32x4 t = transpose_groups(wq[p][c]);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 part[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) part[rt] = off[rt][g];
#pragma unroll
        for (int f = 0; f < FPG; ++f) {
          const u32x4 w = codes_bf16(t[g * FPG + f]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) part[rt] = mfma16(xf[p][rt][g * FPG + f], w, part[rt]);
        }
        const float s = bf16_bits_to_f32(sc[p][c][g]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[rt][c][r] = fmaf(s, part[rt][r], acc[rt][c][r]);
      }
    }
  };

#pragma unroll
  for (int p = 0; p < PF; ++p) load(p, wave + p * W);
  for (int i = wave; i < slabs; i += W * PF) {
#pragma unroll
    for (int p = 0; p < PF; ++p) {
      if (i + p * W >= slabs) break;
      compute(p);
      load(p, i + (p + PF) * W);
    }
  }

  // the waves' sums in wave order, then the epilogue
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int c = 0; c < NC; ++c) red[wave][rt * NC + c][lane] = acc[rt][c];
  __syncthreads();
  auto total = [&](int t) {
    f32x4 v = red[0][t][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += red[w][t][lane];
    return v;
  };
  for (int t = wave; t < RT * NB; t += W) {
    const int rt = t / NB, b = t - rt * NB;
    const int64_t n = n0 + b * 16 + li;
    f32x4 v, u;
    if constexpr (GATEUP) {
      v = total(rt * NC + 2 * b);
      u = total(rt * NC + 2 * b + 1);
    } else {
      v = total(rt * NC + b);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t m = rt * 16 + 4 * grp + r;
      if (m >= a.M || n >= a.N) continue;
      a.y[m * a.ldy + n] = (uint16_t)(GATEUP ? gate_up_silu_bits(v[r], u[r]) : f32_to_bf16_bits(v[r]));
    }
  }
}

// Weights out of their codes: out [N][Kp] bf16, zero from K on. A thread's 32 k are
// one group's at most.
__global__ __launch_bounds__(256) void w4_dequantize_kernel(const uint8_t* q, int64_t ldq,
                                                            const uint16_t* s, int64_t lds, int gs,
                                                            uint16_t* out, int64_t N, int64_t K,
                                                            int64_t Kp) {
  const int64_t cols = Kp / 32, item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= N * cols) return;
  const int64_t n = item / cols, k0 = (item - n * cols) * 32;
  const uint8_t* src = q + n * ldq + k0 / 2;
  u32x4 w = {0u, 0u, 0u, 0u};
  if (k0 + 32 <= K) {
    w = ld16_any(src);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (k0 + 2 * e < K) w[e / 4] |= (uint32_t)src[e] << (8 * (e % 4));
  }
  const float f = k0 < K ? bf16_bits_to_f32(s[n * lds + k0 / gs]) : 0.f;
  const float off = -8.f * f;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t k = k0 + 8 * d + 2 * i;
      const float lo = fmaf((float)((w[d] >> (8 * i)) & 15u), f, off);
      const float hi = fmaf((float)((w[d] >> (8 * i + 4)) & 15u), f, off);
      o[i] = pack_bf16x2(k < K ? lo : 0.f, k + 1 < K ? hi : 0.f);
    }
    *reinterpret_cast<u32x4*>(out + n * Kp + k0 + 8 * d) = o;
  }
}

// x rows [M][K] as [M][Kp], zero from K on.
__global__ __launch_bounds__(256) void w4_pad_kernel(const uint16_t* x, int64_t ldx, uint16_t* out,
                                                     int64_t M, int64_t K, int64_t Kp) {
  const int64_t cols = Kp / 8, item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= M * cols) return;
  const int64_t m = item / cols, k = (item - m * cols) * 8;
  const u32x4 v = k < K ? load_bf16x8<false>(x + m * ldx, k, K) : u32x4{0u, 0u, 0u, 0u};
  *reinterpret_cast<u32x4*>(out + m * Kp + k) = v;
}

// One group per GS / 8 lanes, eight weights each (group sizes 32, 64, 128: 4, 8, 16
// lanes of one 16-lane row).
template <int GS>
__global__ __launch_bounds__(256) void w4_quantize_kernel(const uint16_t* w, int64_t ldw, uint8_t* q,
                                                          int64_t ldq, uint16_t* s, int64_t lds,
                                                          int64_t N, int64_t K) {
  const int64_t groups = (K + GS - 1) / GS, cols = groups * (GS / 8);
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool live = item < N * cols;  // lanes past the end stay for the exchanges
  const int64_t n = live ? item / cols : N - 1, k = live ? (item - n * cols) * 8 : 0;
  const u32x4 v = k < K ? load_bf16x8<false>(w + n * ldw, k, K) : u32x4{0u, 0u, 0u, 0u};
  float x[8], top = 0.f;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = bf16_bits_to_f32(e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xffffu);
    top = fmaxf(top, fabsf(x[e]));
    bad |= !(fabsf(x[e]) < INFINITY);
  }
  if (bad) top = INFINITY;  // an infinity or a NaN
  top = fmaxf(top, dpp_f32<0xb1>(top));
  top = fmaxf(top, dpp_f32<0x4e>(top));
  if constexpr (GS >= 64) top = fmaxf(top, dpp_f32<0x141>(top));
  if constexpr (GS >= 128) top = fmaxf(top, dpp_f32<0x140>(top));
  // five significant bits, ties to even; nothing under the normal numbers
  const uint32_t b = __float_as_uint(top / 7.0f);
  uint32_t sb = (b + 0x3ffffu + ((b >> 19) & 1u)) & 0xfff80000u;
  if (sb < 0x00800000u) sb = 0;
  if (!(top < INFINITY)) sb = 0x7fc00000u;
  const float scale = __uint_as_float(sb);
  if (!live) return;
  if (k % GS == 0) s[n * lds + k / GS] = (uint16_t)(sb >> 16);
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float c = scale > 0.f ? fminf(fmaxf(rintf(x[e] / scale), -7.f), 7.f) : 0.f;
    word |= (uint32_t)((int)c + 8) << (4 * e);
  }
  uint8_t* dst = q + n * ldq + k / 2;
  if (k + 8 <= K) {
    __builtin_memcpy(dst, &word, 4);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k + 2 * e < K) dst[e] = (uint8_t)(word >> (8 * e));
  }
}

template <int RT, int NC, int GS, bool GATEUP, bool ALIGNED>
int launch_rows_g(const W4Args& a, hipStream_t s) {
  constexpr int NB = GATEUP ? NC / 2 : NC;
  constexpr int PF = RT == 1 ? 4 : 2;
  const dim3 grid((unsigned)((a.N + 16 * NB - 1) / (16 * NB)));
  if (RT * NC <= 4 && a.K > 4096)
    hipLaunchKernelGGL((w4_rows_kernel<RT, NC, GS, GATEUP, ALIGNED, 8, PF>), grid, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((w4_rows_kernel<RT, NC, GS, GATEUP, ALIGNED, 4, PF>), grid, dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

template <int GS, bool GATEUP, bool ALIGNED>
int launch_rows_m(const W4Args& a, hipStream_t s) {
  constexpr int NC1 = GATEUP ? 2 : 1;
  if (a.M <= 16) return launch_rows_g<1, NC1, GS, GATEUP, ALIGNED>(a, s);
  if (a.M <= 32) return launch_rows_g<2, 2, GS, GATEUP, ALIGNED>(a, s);
  return launch_rows_g<4, 4, GS, GATEUP, ALIGNED>(a, s);
}

template <bool GATEUP, bool ALIGNED>
int launch_rows_gs(const W4Args& a, hipStream_t s) {
  if (a.group == 128) return launch_rows_m<128, GATEUP, ALIGNED>(a, s);
  if (a.group == 64) return launch_rows_m<64, GATEUP, ALIGNED>(a, s);
  return launch_rows_m<32, GATEUP, ALIGNED>(a, s);
}

}  // namespace

int launch_w4_rows(const W4Args& a, bool gateup, bool aligned, hipStream_t s) {
  if (gateup) return aligned ? launch_rows_gs<true, true>(a, s) : launch_rows_gs<true, false>(a, s);
  return aligned ? launch_rows_gs<false, true>(a, s) : launch_rows_gs<false, false>(a, s);
}

int launch_w4_dequantize(const uint8_t* q, int64_t ldq, const uint16_t* sc, int64_t lds, int group,
                         uint16_t* out, int64_t N, int64_t K, int64_t Kp, hipStream_t s) {
  const int64_t items = N * (Kp / 32);
  hipLaunchKernelGGL(w4_dequantize_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, q,
                     ldq, sc, lds, group, out, N, K, Kp);
  return (int)hipGetLastError();
}

int launch_w4_pad(const uint16_t* x, int64_t ldx, uint16_t* out, int64_t M, int64_t K, int64_t Kp,
                  hipStream_t s) {
  const int64_t items = M * (Kp / 8);
  hipLaunchKernelGGL(w4_pad_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, x, ldx,
                     out, M, K, Kp);
  return (int)hipGetLastError();
}

int launch_w4_quantize(const uint16_t* w, int64_t ldw, uint8_t* q, int64_t ldq, uint16_t* sc,
                       int64_t lds, int64_t N, int64_t K, int group, hipStream_t s) {
  const int64_t items = N * ((K + group - 1) / group) * (group / 8);
  const dim3 grid((unsigned)((items + 255) / 256)), block(256);
  if (group == 32) hipLaunchKernelGGL(w4_quantize_kernel<32>, grid, block, 0, s, w, ldw, q, ldq, sc, lds, N, K);
  else if (group == 64) hipLaunchKernelGGL(w4_quantize_kernel<64>, grid, block, 0, s, w, ldw, q, ldq, sc, lds, N, K);
  else hipLaunchKernelGGL(w4_quantize_kernel<128>, grid, block, 0, s, w, ldw, q, ldq, sc, lds, N, K);
  return (int)hipGetLastError();
}

}  // namespace fp
