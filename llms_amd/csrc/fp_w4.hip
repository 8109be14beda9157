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
// x is the A operand of v_mfma_f32_16x16x32_bf16, the codes the B operand: a lane's
// accumulators belong to one weight row (column lane % 16), so its group's scale is one
// register. Codes become bf16 without a conversion: (w >> s & 0x00780078) | 0x41804180
// holds two codes as 16 + (q + 8) exactly. The 24 too much times the group's sum
// of x is what the group's sum starts from: sums of up to 31 |x|, where products of codes alone
// have 7 |x|, so fp32 rounds a group's sum at up to four times their size (with the codes
// in the low bits, as 128 + (q + 8), twenty times: an input of 1e5 then cost outputs that
// do not use it as much as their rounding), and a group's inputs have to stay under 2^123
// together. The nibbles of a dword come out as k 0 4 1 5
// 2 6 3 7: x is put into that order on its way into LDS. A lane's 16 bytes are 32
// consecutive k of its row, so with groups of 128 the four operands of a slab of 128
// k are its dwords as they come; with groups of 64 or 32 a 4 x 4 transpose of dwords between
// the four lane groups (v_permlane32_swap, v_permlane16_swap) makes them four
// operands of 32 consecutive k, so that a group is whole MFMAs.
//
//   - w4_row_kernel: few rows. The waves of a workgroup split k; x (all of it) goes into
//     LDS once, behind the first weight loads.
//   - w4_tiles_kernel: more rows. The waves split the columns and share slabs of x, which
//     w4_prep_kernel lays out as they will lie in LDS; weights go straight into
//     registers, four slabs ahead. k may be split over workgroups (fp32 partials,
//     summed in order by w4_reduce_kernel).
#include "fp_common.h"
#include "fp_launch.h"

#include <type_traits>

namespace fp {

namespace {

constexpr float kOff = -24.f;  // what codes_bf16 has too much, taken off

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

// Eight codes as bf16 16 + (q + 8), in that order; high is 0x41804180 in a vector
// register that the compiler cannot see through: it then masks and sets a pair in one
// instruction, which may read one scalar register only (with two constants it takes two).
__device__ __forceinline__ u32x4 codes_bf16(uint32_t w, uint32_t high) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((i == 0 ? w << 3 : w >> (4 * i - 3)) & 0x00780078u) | high;
  return v;
}
__device__ __forceinline__ uint32_t code_high() {
  uint32_t v;
  asm("v_mov_b32 %0, 0x41804180" : "=v"(v));
  return v;
}

// Eight codes as the bf16 values code * s, in that order (exact: eight bits at most).
__device__ __forceinline__ u32x4 values_bf16(uint32_t w, float s, float n8s) {
  const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = (i & 1 ? odd : even) >> (8 * (i / 2));
    const float lo = fmaf((float)(b & 0xffu), s, n8s), hi = fmaf((float)((b >> 16) & 0xffu), s, n8s);
    v[i] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
  }
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

// Sixteen bytes shifted down by d bytes (d >= 16: anything).
__device__ __forceinline__ u32x4 bytes_down(u32x4 v, uint32_t d) {
  if (d & 8) v[0] = v[2], v[1] = v[3];
  if (d & 4) v[0] = v[1], v[1] = v[2], v[2] = v[3];
  return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], d), __builtin_amdgcn_alignbyte(v[2], v[1], d),
               __builtin_amdgcn_alignbyte(v[3], v[2], d), v[3] >> (8 * (d & 3))};
}

// The weight rows of a wave's NC column blocks (gate-up: gate and up in turn), 16 bytes
// per lane and slab. What lies past K meets zeros of x: any codes do there.
// ALIGNED: 16-byte aligned rows, read through buffers whose end returns zeros.
// Else ordinary loads at any address, moved back where they would pass the weight's last
// byte and put right when they are used (fix; a weight has at least 16 bytes). Every load is issued without a
// branch: at one the compiler would wait for all that are in flight.
template <int NC, bool GATEUP, bool ALIGNED>
struct Weights {
  const uint8_t* base[NC];
  __amdgpu_buffer_rsrc_t rsrc[NC];
  uint32_t off[NC];   // of the lane's row from base
  uint32_t last[NC];  // the last offset with 16 bytes of the weight behind it
  int safe[NC];       // slabs that lie within the weight for all of the block's rows

  // n0: the first output column of the wave's blocks
  __device__ __forceinline__ void init(const W4Args& a, int64_t n0, int li, int grp) {
    const int rowb = (int)((a.K + 1) / 2);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const bool up = GATEUP && (c & 1);
      const int64_t r0 = n0 + (GATEUP ? c / 2 : c) * 16, first = r0 < a.N ? r0 : a.N - 1;
      const int rows = a.N - first < 16 ? (int)(a.N - first) : 16;
      const int row = li < rows ? li : rows - 1;
      const int64_t ldq = up ? a.ldq1 : a.ldq0;
      base[c] = (up ? a.q1 : a.q0) + first * ldq;
      off[c] = (uint32_t)(row * ldq) + 16 * grp;
      if constexpr (ALIGNED) {
        // with the whole last 16 bytes: they lie in one page with their first
        rsrc[c] = make_rsrc(base[c], (rows - 1) * ldq + (rowb + 15) / 16 * 16);
      } else {
        const int64_t left = (a.N - first - 1) * ldq + rowb;  // bytes from base on
        last[c] = left - 16 < 0x7fffffff ? (uint32_t)(left - 16) : 0x7fffffffu;
        const int64_t whole = ((a.N - first - rows) * ldq + rowb) / 64;
        safe[c] = whole < (1 << 30) ? (int)whole : 1 << 30;
      }
    }
  }
  __device__ __forceinline__ u32x4 load(int c, int slab, int slabs) const {
    if constexpr (ALIGNED)
      return __builtin_amdgcn_raw_buffer_load_b128(rsrc[c], slab < slabs ? off[c] + slab * 64 : kOut, 0, 0);
    const uint32_t at = slab < slabs ? off[c] + slab * 64 : 0;
    // last counts down from base where the block holds the weight's last bytes alone
    const int32_t to = (int32_t)at < (int32_t)last[c] ? (int32_t)at : (int32_t)last[c];
    return ld16_any(base[c] + to);
  }
  __device__ __forceinline__ u32x4 fix(int c, u32x4 w, int slab) const {
    if constexpr (ALIGNED) return w;
    if (__builtin_expect(slab < safe[c], 1)) return w;
    const int32_t over = (int32_t)(off[c] + slab * 64) - (int32_t)last[c];
    return over > 0 ? bytes_down(w, (uint32_t)over) : w;
  }
};

// The scales of the same rows: a slab's in one load (without a branch, as the weights'),
// moved back at the row's end and shifted when they are used (past the last group: 0, where the codes meet zeros).
template <int NC, int GS, bool GATEUP>
struct Scales {
  static constexpr int NG = 128 / GS;
  // 32 bits where that is enough: a wider one is widened, and so waited for, at its load
  using Raw = std::conditional_t<NG == 4, uint64_t, uint32_t>;
  const uint16_t* row[NC];
  int groups, last;

  __device__ __forceinline__ void init(const W4Args& a, int64_t n0, int li) {
    groups = (int)((a.K + GS - 1) / GS);
    last = groups > NG ? groups - NG : 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const bool up = GATEUP && (c & 1);
      const int64_t n = n0 + (GATEUP ? c / 2 : c) * 16 + li;
      row[c] = (up ? a.s1 : a.s0) + (n < a.N ? n : a.N - 1) * (up ? a.lds1 : a.lds0);
    }
  }
  __device__ __forceinline__ Raw load(int c, int slab) const {
    const int at = slab * NG < last ? slab * NG : last;
    if constexpr (NG == 1) return row[c][at];
    uint32_t v[2] = {0u, 0u};
    __builtin_memcpy(v, row[c] + at, 2 * NG);  // rows of fewer have been widened
    if constexpr (NG == 4) return v[0] | ((uint64_t)v[1] << 32);
    else return v[0];
  }
  __device__ __forceinline__ Raw fix(Raw s, int slab) const {
    return NG > 1 && slab * NG > last ? s >> (16 * (slab * NG - last)) : s;
  }
  static __device__ __forceinline__ float at(Raw s, int g) {
    return __uint_as_float((uint32_t)(s >> (16 * g)) << 16);
  }
};

// Where chunk cc (8 k) of a slab's 128 goes as an A operand: MFMA f, lane group g.
template <int GS>
__device__ __forceinline__ int frag_of(int cc) { return GS == 128 ? cc & 3 : cc >> 2; }
template <int GS>
__device__ __forceinline__ int grp_of(int cc) { return GS == 128 ? cc >> 2 : cc & 3; }
// Sum of v over the GS / 8 consecutive lanes of a group's chunks.
template <int GS>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp_f32<0xb1>(v);
  v += dpp_f32<0x4e>(v);
  if constexpr (GS >= 64) v += dpp_f32<0x141>(v);
  if constexpr (GS >= 128) v += dpp_f32<0x140>(v);
  return v;
}
__device__ __forceinline__ float sum8(u32x4 v) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s += __uint_as_float(v[i] << 16) + __uint_as_float(v[i] & 0xffff0000u);
  return s;
}

// y of a 16 x 16 block: rows m0 + r, column n; g and u are rounded once, as their product.
template <bool GATEUP>
__device__ __forceinline__ void store_block(const W4Args& a, f32x4 v, f32x4 u, int64_t m0, int64_t n) {
  if (n >= a.N) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (m0 + r >= a.M) continue;
    const float y = GATEUP ? __fdividef(v[r], 1.0f + __expf(-v[r])) * u[r] : v[r];
    a.y[(m0 + r) * a.ldy + n] = (uint16_t)f32_to_bf16_bits(y);
  }
}

// M <= 16 rows with room for x in LDS. W waves split the slabs of k in contiguous
// ranges; each has SB slabs of weights in one half of its registers while it
// multiplies the other half's. (Larger batches and a staging loop unrolled further are
// slower: a launch runs the code once, so its instructions come from memory.) Scales go
// through LDS too: two bytes a row and slab read where they are needed cost as many
// lines as the weights do. One row of 2560 x 2 x 9728 (groups of 128) 10 us, 2.6 TB/s of
// packed weights from HBM, 10240 x 2 x 9728 30 us, 3.4 TB/s; below a few us of work the launch and x's
// way into LDS bound it, above the loads that two workgroups of a CU keep in flight.
template <int NC, int GS, bool GATEUP, bool ALIGNED, int W>
__global__ __launch_bounds__(W * 64) void w4_row_kernel(W4Args a) {
  constexpr int NG = 128 / GS, FPG = 4 / NG;  // groups of a slab, MFMAs of a group
  constexpr int NB = GATEUP ? NC / 2 : NC;    // 16-column blocks of the output
  constexpr int SB = 2, NT = W * 64;
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, grp = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NB);
  const int M = (int)a.M, slabs = (int)((a.K + 127) / 128);
  const int kp = slabs * 128, ldx = kp * 2 + 16;  // LDS row of x, off the banks of the next
  // LDS: x rows, kOff sum x [group][16], scales [group][16 NC]; the waves' sums at the end
  char* sx = lds;
  float* sb = reinterpret_cast<float*>(lds + M * ldx);
  float* ss = sb + slabs * NG * 16;

  const int per = (slabs + W - 1) / W;
  const int lo = wave * per, hi = lo + per < slabs ? lo + per : slabs;
  const int chunks = M * (kp / 8);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, ((a.M - 1) * a.ldx + a.K) * 2);
  const bool vec = a.K % 8 == 0 && a.ldx % 8 == 0 && ((uintptr_t)a.x & 15) == 0;  // uniform
  auto load_x = [&](int i) -> u32x4 {
    const int r = i / (kp / 8), k = (i - r * (kp / 8)) * 8;
    const uint32_t off = (uint32_t)((r * (int)a.ldx + k) * 2);
    return __builtin_amdgcn_raw_buffer_load_b128(xr, i < chunks && k < a.K ? off : kOut, 0, 0);
  };
  auto load_x_any = [&](int i) -> u32x4 {  // any alignment, any K
    const int r = i / (kp / 8), k = (i - r * (kp / 8)) * 8;
    const uint32_t off = (uint32_t)((r * (int)a.ldx + k) * 2);
    uint32_t h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      h[e] = __builtin_amdgcn_raw_buffer_load_b16(xr, i < chunks && k + e < a.K ? off + 2 * e : kOut, 0, 0);
    return u32x4{h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16)};
  };
  auto store_x = [&](int i, u32x4 v) {
    const int r = i / (kp / 8), c = i - r * (kp / 8);
    const float s = group_sum<GS>(sum8(v));
    if (i >= chunks) return;
    *reinterpret_cast<u32x4*>(sx + r * ldx + c * 16) = nibble_order(v);
    if (c % (GS / 8) == 0) sb[c / (GS / 8) * 16 + r] = kOff * s;
  };
  // scales: along a row's groups from lane to lane (loaded where they are used, each of the
  // 16 rows of a wave's load would cost as much as 64 bytes of weights)
  const int n_sc = slabs * NG * 16 * NC;
  const int sc_rows = a.N - n0 < 16 * NB ? (int)(a.N - n0) : 16 * NB, groups = (int)((a.K + GS - 1) / GS);
  const __amdgpu_buffer_rsrc_t s0 = make_rsrc(a.s0 + n0 * a.lds0, ((sc_rows - 1) * a.lds0 + groups) * 2);
  const __amdgpu_buffer_rsrc_t s1 =
      GATEUP ? make_rsrc(a.s1 + n0 * a.lds1, ((sc_rows - 1) * a.lds1 + groups) * 2) : s0;
  auto load_s = [&](int i) -> uint32_t {
    const int row = i / (slabs * NG), g = i - row * (slabs * NG);
    const int c = row / 16, n = (GATEUP ? c / 2 : c) * 16 + (row & 15);
    const bool in = i < n_sc && g < groups && n < sc_rows, up = GATEUP && (c & 1);
    uint32_t s = __builtin_amdgcn_raw_buffer_load_b16(s0, in && !up ? (uint32_t)((n * (int)a.lds0 + g) * 2) : kOut, 0, 0);
    if constexpr (GATEUP)
      s |= __builtin_amdgcn_raw_buffer_load_b16(s1, in && up ? (uint32_t)((n * (int)a.lds1 + g) * 2) : kOut, 0, 0);
    return s;
  };
  auto store_s = [&](int i, uint32_t s) {
    const int row = i / (slabs * NG), g = i - row * (slabs * NG);
    if (i < n_sc) ss[g * (16 * NC) + row] = bf16_bits_to_f32(s);
  };
  constexpr int SN = 3;
  uint32_t sv[SN];
#pragma unroll
  for (int n = 0; n < SN; ++n) sv[n] = load_s(n * NT + tid);
  // the first of x before the first weights: its LDS stores wait for it alone
  const u32x4 x0 = load_x(vec ? tid : chunks), x1 = load_x(vec ? NT + tid : chunks);
  Weights<NC, GATEUP, ALIGNED> wt;
  wt.init(a, n0, li, grp);
  u32x4 wq[2][SB][NC];
  auto load_w = [&](int h, int slab) {
#pragma unroll
    for (int p = 0; p < SB; ++p)
#pragma unroll
      for (int c = 0; c < NC; ++c) wq[h][p][c] = wt.load(c, slab + p < hi ? slab + p : slabs, slabs);
  };
  load_w(0, lo);
  load_w(1, lo + SB);
  for (int i = tid; i < slabs * NG * 16; i += NT)
    if ((i & 15) >= M) sb[i] = 0.f;  // rows that are not there
#pragma unroll
  for (int n = 0; n < SN; ++n) store_s(n * NT + tid, sv[n]);
#pragma unroll 1
  for (int i = SN * NT; i < n_sc; i += 4 * NT) {
    uint32_t v[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) v[n] = load_s(i + n * NT + tid);
#pragma unroll
    for (int n = 0; n < 4; ++n) store_s(i + n * NT + tid, v[n]);
  }
  // (whole workgroups, for the lane exchanges of the sums)
  if (vec) {
    store_x(tid, x0);
    store_x(NT + tid, x1);
#pragma unroll 1
    for (int i = 2 * NT; i < chunks; i += 4 * NT) {
      u32x4 v[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) v[n] = load_x(i + n * NT + tid);
#pragma unroll
      for (int n = 0; n < 4; ++n) store_x(i + n * NT + tid, v[n]);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < chunks; i += NT) store_x(i + tid, load_x_any(i + tid));
  }
  __syncthreads();

  const uint32_t high = code_high();
  f32x4 acc[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const char* xrow = sx + (li < M ? li : M - 1) * ldx;
  auto compute = [&](int h, int slab) {
#pragma unroll
    for (int p = 0; p < SB; ++p) {
      const int at = slab + p;
      if (at >= hi) break;
      // (before the MFMAs: at a branch between one and the use of its result the compiler
      // has left out the wait for it)
      u32x4 t[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        t[c] = wt.fix(c, wq[h][p][c], at);
        if constexpr (GS != 128) t[c] = transpose_groups(t[c]);
      }
      u32x4 xf[4];
#pragma unroll
      for (int f = 0; f < 4; ++f)
        xf[f] = *reinterpret_cast<const u32x4*>(xrow + at * 256 + (GS == 128 ? 64 * grp + 16 * f : 64 * f + 16 * grp));
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const f32x4 b = *reinterpret_cast<const f32x4*>(sb + (at * NG + g) * 16 + 4 * grp);
        f32x4 part[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) part[c] = b;
#pragma unroll
        for (int f = 0; f < FPG; ++f)
#pragma unroll
          for (int c = 0; c < NC; ++c)
            part[c] = mfma16(xf[g * FPG + f], codes_bf16(t[c][g * FPG + f], high), part[c]);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float s = ss[(at * NG + g) * (16 * NC) + c * 16 + li];
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[c][r] = fmaf(s, part[c][r], acc[c][r]);
        }
      }
    }
  };
  for (int at = lo; at < hi; at += 2 * SB) {
    compute(0, at);
    load_w(0, at + 2 * SB);
    compute(1, at + SB);
    load_w(1, at + 3 * SB);
  }

  // the waves' sums in wave order, then the epilogue
  __syncthreads();  // x and the scales have been read
  f32x4(*red)[NC][64] = reinterpret_cast<f32x4(*)[NC][64]>(lds);
#pragma unroll
  for (int c = 0; c < NC; ++c) red[wave][c][lane] = acc[c];
  __syncthreads();
  auto total = [&](int t) {
    f32x4 v = red[0][t][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += red[w][t][lane];
    return v;
  };
  for (int b = wave; b < NB; b += W) {
    const f32x4 v = total(GATEUP ? 2 * b : b);
    store_block<GATEUP>(a, v, GATEUP ? total(2 * b + 1) : v, 4 * grp, n0 + b * 16 + li);
  }
}

// ---- more rows --------------------------------------------------------------
//
// A panel of 16 RT rows of x is laid out slab by slab as it lies in LDS: for each block of
// 16 rows and each of the slab's four operands the 64 lanes' 16 bytes, then kOff
// sum x as [group of the slab][row].
//
// 64 rows of 4096 x 2 x 12288 take 31 us here, 4 us in prep and 5 in the reduction (350
// TFLOP/s; 384 workgroups of sixteen slabs each, whose barrier a slab is what is left);
// 1024 rows of 2560 x 2 x 9728 125 us, 2048 235 (870 TFLOP/s; 770 with groups of 32, whose codes are
// scaled before the product). The weights are expanded by each panel of rows anew, eight
// blocks of 16 rows to a wave at most: the vector unit beside the matrix core bounds it.
constexpr int panel_bytes(int rt) { return rt * 4096 + 4 * rt * 64; }

template <int GS>
__global__ __launch_bounds__(256) void w4_prep_kernel(const uint16_t* x, int64_t ldx, char* out, int64_t M,
                                                      int64_t K, int slabs, int rt) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t cols = (int64_t)slabs * 16, rows = (M + 16 * rt - 1) / (16 * rt) * (16 * rt);
  if (item >= rows * cols) return;  // a multiple of 16: whole 16-lane rows leave together
  const int64_t m = item / cols, c = item - m * cols, k = c * 8;
  u32x4 v = {0u, 0u, 0u, 0u};
  if (m < M && k < K) v = load_bf16x8<false>(x + m * ldx, k, K);
  const float s = group_sum<GS>(sum8(v));
  const int64_t panel = m / (16 * rt);
  const int r = (int)(m - panel * (16 * rt)), slab = (int)(c / 16), cc = (int)(c % 16);
  char* p = out + (panel * slabs + slab) * panel_bytes(rt);
  *reinterpret_cast<u32x4*>(p + ((r / 16) * 4 + frag_of<GS>(cc)) * 1024 + (grp_of<GS>(cc) * 16 + r % 16) * 16) =
      nibble_order(v);
  if (cc % (GS / 8) == 0) reinterpret_cast<float*>(p + rt * 4096)[cc / (GS / 8) * (16 * rt) + r] = kOff * s;
}

template <int RT, int NC, int GS, bool GATEUP, bool ALIGNED, int W>
__global__ __launch_bounds__(W * 64, 2) void w4_tiles_kernel(W4Args a) {
  constexpr int NG = 128 / GS, FPG = 4 / NG;
  constexpr int NB = GATEUP ? NC / 2 : NC;
  constexpr int PF = RT == 8 ? 2 : 4, NT = W * 64, PB = panel_bytes(RT);
  constexpr int XN = (PB / 16 + NT - 1) / NT;  // 16-byte chunks of a slab per thread
  // Scaling a group's sums costs RT x 4 multiply-adds of each column block, scaling its
  // codes 23 instructions of each dword: with many rows and small groups the latter, which
  // also needs no second set of sums (exact either way).
  constexpr bool DEQ = RT == 8 && GS < 128;
  __shared__ __attribute__((aligned(16))) char sx[2][PB];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, grp = lane >> 4;
  const int64_t n0 = ((int64_t)blockIdx.y * W + wave) * (16 * NB);
  const int slabs = (int)((a.K + 127) / 128);
  const int per = (slabs + a.splits - 1) / a.splits;
  const int lo = (int)blockIdx.z * per, hi = lo + per < slabs ? lo + per : slabs;
  Weights<NC, GATEUP, ALIGNED> wt;
  wt.init(a, n0, li, grp);
  Scales<NC, GS, GATEUP> sl;
  sl.init(a, n0, li);

  const u32x4* xp = reinterpret_cast<const u32x4*>(a.panels + (int64_t)blockIdx.x * slabs * PB);
  u32x4 xv[XN];
  auto load_x = [&](int slab) {
    const u32x4* src = xp + (int64_t)(slab < hi ? slab : hi - 1) * (PB / 16);
#pragma unroll
    for (int n = 0; n < XN; ++n) {
      const int i = n * NT + tid;
      xv[n] = src[i < PB / 16 ? i : PB / 16 - 1];
    }
  };
  auto store_x = [&](char* dst) {
#pragma unroll
    for (int n = 0; n < XN; ++n) {
      const int i = n * NT + tid;
      if (PB / 16 % NT == 0 || i < PB / 16) reinterpret_cast<u32x4*>(dst)[i] = xv[n];
    }
  };
  u32x4 wq[PF][NC];
  typename Scales<NC, GS, GATEUP>::Raw sc[PF][NC];
  auto load_w = [&](int p, int slab) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      wq[p][c] = wt.load(c, slab < hi ? slab : slabs, slabs);
      sc[p][c] = sl.load(c, slab);
    }
  };

  const uint32_t high = code_high();
  f32x4 acc[RT][NC];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[rt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const char* x, int p, int slab) {
    u32x4 t[NC];
    typename Scales<NC, GS, GATEUP>::Raw s4[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const u32x4 w = wt.fix(c, wq[p][c], slab);
      t[c] = GS == 128 ? w : transpose_groups(w);
      s4[c] = sl.fix(sc[p][c], slab);
    }
    if constexpr (DEQ) {
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        u32x4 w[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float s = sl.at(s4[c], f / FPG);
          w[c] = values_bf16(t[c][f], s, -8.f * s);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const u32x4 xf = *reinterpret_cast<const u32x4*>(x + (rt * 4 + f) * 1024 + lane * 16);
#pragma unroll
          for (int c = 0; c < NC; ++c) acc[rt][c] = mfma16(xf, w[c], acc[rt][c]);
        }
      }
      return;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4 part[RT][NC];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const f32x4 b = *reinterpret_cast<const f32x4*>(x + RT * 4096 + (g * (16 * RT) + rt * 16 + 4 * grp) * 4);
#pragma unroll
        for (int c = 0; c < NC; ++c) part[rt][c] = b;
      }
#pragma unroll
      for (int f = 0; f < FPG; ++f) {
        u32x4 w[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) w[c] = codes_bf16(t[c][g * FPG + f], high);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const u32x4 xf = *reinterpret_cast<const u32x4*>(x + (rt * 4 + g * FPG + f) * 1024 + lane * 16);
#pragma unroll
          for (int c = 0; c < NC; ++c) part[rt][c] = mfma16(xf, w[c], part[rt][c]);
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float s = sl.at(s4[c], g);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[rt][c][r] = fmaf(s, part[rt][c][r], acc[rt][c][r]);
      }
      // one group's sums at a time: several would not fit the registers
      if constexpr (NG > 1 && RT == 4) __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (lo < hi) {
    load_x(lo);
#pragma unroll
    for (int p = 0; p < PF - 1; ++p) load_w(p, lo + p);
    store_x(sx[0]);
    load_x(lo + 1);
    // in the loop's order: x with no weights behind it here would have the compiler wait for
    // the weights in flight once in PF slabs
    load_w(PF - 1, lo + PF - 1);
    __syncthreads();
    for (int i = lo; i < hi; i += PF) {
#pragma unroll
      for (int p = 0; p < PF; ++p) {
        const int slab = i + p;
        if (slab >= hi) break;
        store_x(sx[(p + 1) & 1]);  // slab + 1, loaded a slab ago; read last before the barrier
        load_x(slab + 2);
        compute(sx[p & 1], p, slab);
        load_w(p, slab + PF);
        __syncthreads();
      }
    }
  }

#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int64_t m = ((int64_t)blockIdx.x * RT + rt) * 16 + 4 * grp, n = n0 + b * 16 + li;
      if (a.splits == 1) {
        store_block<GATEUP>(a, acc[rt][GATEUP ? 2 * b : b], acc[rt][GATEUP ? 2 * b + 1 : b], m, n);
      } else if (n < a.N) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (m + r >= a.M) continue;
          const int64_t at = ((int64_t)blockIdx.z * a.M + m + r) * a.N + n;
          if constexpr (GATEUP)
            reinterpret_cast<f32x2*>(a.part)[at] = f32x2{acc[rt][2 * b][r], acc[rt][2 * b + 1][r]};
          else a.part[at] = acc[rt][b][r];
        }
      }
    }
}

// Rows of rowb bytes as rows of `to`, zeros behind them: for a weight of under 16 bytes (the
// kernels load 16 at a time) and for scales of less than a slab's groups.
__global__ __launch_bounds__(256) void w4_widen_kernel(const uint8_t* q, int64_t ld, uint8_t* out, int64_t rows,
                                                       int64_t rowb, int to) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * to) return;
  const int64_t r = i / to, c = i - r * to;
  out[i] = c < rowb ? q[r * ld + c] : 0;
}

template <bool GATEUP>
__global__ __launch_bounds__(256) void w4_reduce_kernel(W4Args a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, total = a.M * a.N;
  if (i >= total) return;
  float v = 0.f, u = 0.f;
  for (int z = 0; z < a.splits; ++z) {
    if constexpr (GATEUP) {
      const f32x2 p = reinterpret_cast<const f32x2*>(a.part)[z * total + i];
      v += p.x, u += p.y;
    } else {
      v += a.part[z * total + i];
    }
  }
  const float y = GATEUP ? __fdividef(v, 1.0f + __expf(-v)) * u : v;
  a.y[i / a.N * a.ldy + i % a.N] = (uint16_t)f32_to_bf16_bits(y);
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

// How a call runs: w4_row_kernel, or w4_tiles_kernel on panels of 16 rt rows with
// column workgroups of `waves` waves and k in `splits` ranges.
struct W4Plan {
  bool row;
  int nc, waves, rt, splits;
};

// Workspace of a weight that may have under 16 bytes (rows apart only make it longer).
int64_t wide_bytes(int64_t N, int64_t K) { return N * ((K + 1) / 2) < 16 ? 512 : 0; }
// ... and of the scales of two weights of at most three groups.
int64_t scale_bytes(int64_t N, int64_t K) { return K <= 96 ? (N * 16 + 255) / 256 * 256 : 0; }

int64_t row_lds(int64_t M, int64_t K, int nc, int group) {
  const int64_t slabs = (K + 127) / 128;
  return M * (slabs * 256 + 16) + slabs * (128 / group) * 64 * (1 + nc);
}

W4Plan w4_plan(int64_t M, int64_t N, int64_t K, int group, bool gateup) {
  W4Plan p{};
  const int64_t slabs = (K + 127) / 128;
  p.nc = gateup ? 2 : 1;
  p.waves = slabs > 24 ? 8 : 4;
  p.splits = 1;
  // Two workgroups of the row kernel per CU, or the one that a CU gets at most: 5 rows of
  // 9728 x 2560 10.6 us against 16.8 on the tiles (prep, k split in 8, reduce); with one of
  // several at a time the tiles win, 16 rows of 2560 x 2 x 9728 18 us against 28.
  const int64_t lds = row_lds(M, K, p.nc, group);
  p.row = M <= 16 && (lds <= kW4RowLds / 2 || (lds <= kW4RowLds && (N + 15) / 16 <= 256));
  if (p.row) return p;
  p.nc = 2;
  p.rt = M <= 16 ? 1 : M <= 32 ? 2 : M <= 64 ? 4 : 8;
  p.waves = 4;
  const int64_t cols = gateup ? N : (N + 1) / 2;  // outputs, or pairs of column blocks
  const int64_t panels = (M + 16 * p.rt - 1) / (16 * p.rt);
  const int64_t groups = (cols + 63) / 64 * panels;
  // k split while the grid leaves CUs idle, ranges of at least eight slabs
  while (p.splits < 16 && groups * p.splits * 2 <= 512 && slabs / (p.splits * 2) >= 8) p.splits *= 2;
  return p;
}

template <int GS, bool GATEUP, bool ALIGNED>
int launch_row(const W4Args& a, const W4Plan& p, hipStream_t s) {
  constexpr int NC = GATEUP ? 2 : 1, NB = 1;
  const dim3 grid((unsigned)((a.N + 16 * NB - 1) / (16 * NB)));
  int64_t lds = row_lds(a.M, a.K, NC, GS);
  const int64_t red = (int64_t)p.waves * NC * 1024;
  if (lds < red) lds = red;
  if (p.waves == 8) hipLaunchKernelGGL((w4_row_kernel<NC, GS, GATEUP, ALIGNED, 8>), grid, dim3(512), (size_t)lds, s, a);
  else hipLaunchKernelGGL((w4_row_kernel<NC, GS, GATEUP, ALIGNED, 4>), grid, dim3(256), (size_t)lds, s, a);
  return (int)hipGetLastError();
}

template <int GS, bool GATEUP, bool ALIGNED>
int launch_tiles(const W4Args& a, const W4Plan& p, hipStream_t s) {
  const int64_t cols = GATEUP ? 64 : 128, panels = (a.M + 16 * p.rt - 1) / (16 * p.rt);
  const dim3 grid((unsigned)panels, (unsigned)((a.N + cols - 1) / cols), (unsigned)p.splits), block(256);
  if (p.rt == 1) hipLaunchKernelGGL((w4_tiles_kernel<1, 2, GS, GATEUP, ALIGNED, 4>), grid, block, 0, s, a);
  else if (p.rt == 2) hipLaunchKernelGGL((w4_tiles_kernel<2, 2, GS, GATEUP, ALIGNED, 4>), grid, block, 0, s, a);
  else if (p.rt == 4) hipLaunchKernelGGL((w4_tiles_kernel<4, 2, GS, GATEUP, ALIGNED, 4>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((w4_tiles_kernel<8, 2, GS, GATEUP, ALIGNED, 4>), grid, block, 0, s, a);
  int e = (int)hipGetLastError();
  if (e || p.splits == 1) return e;
  hipLaunchKernelGGL(w4_reduce_kernel<GATEUP>, dim3((unsigned)((a.M * a.N + 255) / 256)), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

int widen(const uint8_t* q, int64_t ld, uint8_t* out, int64_t rows, int64_t rowb, int to, hipStream_t s) {
  hipLaunchKernelGGL(w4_widen_kernel, dim3((unsigned)((rows * to + 255) / 256)), dim3(256), 0, s, q, ld, out, rows,
                     rowb, to);
  return (int)hipGetLastError();
}

template <int GS>
int launch_gs(W4Args a, const W4Plan& p, bool gateup, bool aligned, char* ws, hipStream_t s) {
  const int64_t rowb = (a.K + 1) / 2;
  if (!aligned && ((a.N - 1) * a.ldq0 + rowb < 16 || (gateup && (a.N - 1) * a.ldq1 + rowb < 16))) {
    uint8_t* wide = (uint8_t*)ws;  // N <= 15 rows, twice
    int e = widen(a.q0, a.ldq0, wide, a.N, rowb, 16, s);
    if (!e && gateup) e = widen(a.q1, a.ldq1, wide + 256, a.N, rowb, 16, s);
    if (e) return e;
    a.q0 = wide, a.ldq0 = 16;
    if (gateup) a.q1 = wide + 256, a.ldq1 = 16;
    aligned = true;
  }
  ws += wide_bytes(a.N, a.K);
  if (p.row) {
    if (gateup) return aligned ? launch_row<GS, true, true>(a, p, s) : launch_row<GS, true, false>(a, p, s);
    return aligned ? launch_row<GS, false, true>(a, p, s) : launch_row<GS, false, false>(a, p, s);
  }
  const int64_t slabs = (a.K + 127) / 128, rows = (a.M + 16 * p.rt - 1) / (16 * p.rt) * (16 * p.rt);
  const int64_t groups = (a.K + GS - 1) / GS, most = 128 / GS;
  if (groups < most) {
    uint8_t* wide = (uint8_t*)ws;
    const int64_t one = a.N * most * 2;
    int e = widen((const uint8_t*)a.s0, a.lds0 * 2, wide, a.N, groups * 2, (int)most * 2, s);
    if (!e && gateup) e = widen((const uint8_t*)a.s1, a.lds1 * 2, wide + one, a.N, groups * 2, (int)most * 2, s);
    if (e) return e;
    a.s0 = (const uint16_t*)wide, a.lds0 = most;
    if (gateup) a.s1 = (const uint16_t*)(wide + one), a.lds1 = most;
  }
  ws += scale_bytes(a.N, a.K);
  a.panels = ws;
  a.part = (float*)(ws + rows / (16 * p.rt) * slabs * panel_bytes(p.rt));
  a.splits = p.splits;
  hipLaunchKernelGGL(w4_prep_kernel<GS>, dim3((unsigned)((rows * slabs * 16 + 255) / 256)), dim3(256), 0, s, a.x,
                     a.ldx, ws, a.M, a.K, (int)slabs, p.rt);
  const int e = (int)hipGetLastError();
  if (e) return e;
  if (gateup) return aligned ? launch_tiles<GS, true, true>(a, p, s) : launch_tiles<GS, true, false>(a, p, s);
  return aligned ? launch_tiles<GS, false, true>(a, p, s) : launch_tiles<GS, false, false>(a, p, s);
}

}  // namespace

int64_t w4_workspace_bytes(int64_t M, int64_t N, int64_t K, bool gateup) {
  int64_t most = 0;
  for (int group = 32; group <= 128; group *= 2) {
    const W4Plan p = w4_plan(M, N, K, group, gateup);
    if (p.row) continue;
    int64_t b = (M + 16 * p.rt - 1) / (16 * p.rt) * ((K + 127) / 128) * panel_bytes(p.rt) + scale_bytes(N, K);
    if (p.splits > 1) b += p.splits * M * N * (gateup ? 8 : 4);
    most = most > b ? most : b;
  }
  return most + wide_bytes(N, K);
}

int launch_w4(const W4Args& a, bool gateup, bool aligned, void* ws, hipStream_t s) {
  const W4Plan p = w4_plan(a.M, a.N, a.K, a.group, gateup);
  if (a.group == 128) return launch_gs<128>(a, p, gateup, aligned, (char*)ws, s);
  if (a.group == 64) return launch_gs<64>(a, p, gateup, aligned, (char*)ws, s);
  return launch_gs<32>(a, p, gateup, aligned, (char*)ws, s);
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
