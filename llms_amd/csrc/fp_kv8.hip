// fp_kv8.hip — a key/value cache in 8 bits with one scale for each block of 64
// tokens and head, and causal attention over it.
//
//   top = max |x| over a block's 64 x D finite entries,  s = top / 127
//   code = rne(127 x / top);  the block's value is code * s
//
// Only whole blocks are packed, from their bf16 tokens, when the last token
// arrives; the tokens of the unfinished block stay in bf16 in a ring of two blocks per
// head (`tail`, `tail_block` says which block a slot holds), so what the cache
// holds does not depend on how its tokens were cut into calls. A call that goes back
// within the ring finds its bf16 tokens there; further back, the block's codes are
// expanded into the ring first. Keys are held [64][D], values [D][64] (codes and
// ring): a value column then is 16 contiguous bytes per lane of a V^T operand.
// Code -128 stands for an entry that was not finite; a block with one has its scale
// negated, so that only such blocks pay for the check. The ring holds such entries as NaN too.
//
//   - kv8_write_kernel: a workgroup per touched block and kv head; QK-norm and RoPE of
//     the new keys on the way where the caller asks (and of q, in more workgroups).
//   - kv8_rows_kernel (T * group <= 64 query rows per kv head) and kv8_tiles_kernel
//     (prompts): S^T = K Q^T and O^T = V^T P^T as in fp_attn.hip. Tile n of a block
//     takes keys 16 (i / 4) + 4 n + i % 4 as rows i, so that a lane's accumulators of
//     the four tiles are keys 16 g .. 16 g + 15 of its lane group g: the order of the 16
//     bytes it loads of a V row.
//   - kv8_combine_kernel: sums a split's partials in split order.
//
// Precision: codes are exact in bf16 (keys) and fp16 (values), scores exact products
// summed in fp32 and scaled after the sum, softmax and its sum in fp32. p enters the
// matrix core in fp16 (2^-12 of itself, an eighth of the output's rounding): the codes
// carry no more than 8 bits, so the parts that fp_attn.hip adds would be lost on
// them. fp16 has its full 11 bits from 2^-14 on only, and a row of one large p and many
// tiny ones is common (a first token that most heads look at): so p goes in times
// 2^kLift, up to 2^15 with what kRise leaves it, and the value codes times 2^-kLift, both
// exact. p keeps 2^-12 of itself down to 2^-28 of a row's largest in kv8_rows_kernel, 2^-24
// in kv8_tiles_kernel; below, what is lost is 2^-39 and 2^-35 of that largest. A block's
// product is scaled by s_v in fp32. The unfinished block's values are bf16, and stay it (in
// fp16 a large value would take the bits of the small ones beside it): p is taken in two
// bf16 parts there.
#include "fp_common.h"
#include "fp_launch.h"
#include "fp_rope.h"

#include <type_traits>

namespace fp {

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

constexpr int kBlk = 64;
constexpr int kKv8MaxSplit = 64;  // one lane per split in kv8_combine_kernel
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRise = 5.f;  // kv8_tiles_kernel: log2 of the largest p
// p's factor in fp16, as a power of two, and so that of the codes: the largest p times it
// is 2^14 and 2^15 (fp16 ends at 65504), a code of 1 by it no less than 2^-14
constexpr int kLiftRows = 14, kLiftTiles = 10;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ f32x4 mfma16h(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, int64_t bytes) {
  constexpr int kRsrcFlags = 0x00020000;  // raw buffer, 32-bit data format
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, kRsrcFlags);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, f16x2{(_Float16)lo, (_Float16)hi});
}
// max / sum over the four lane groups that share a row column.
__device__ __forceinline__ float col_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Four codes of a dword as bf16 (BAD: -128 as NaN).
template <bool BAD>
__device__ __forceinline__ u32x2 codes4_bf16(uint32_t w) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = (float)(int8_t)(w >> (8 * i));
    if (BAD && f[i] == -128.f) f[i] = __uint_as_float(0x7fc00000u);
  }
  // the low halves are zero: every code has at most 8 significant bits
  return u32x2{__builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u),
               __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u)};
}
template <bool BAD>
__device__ __forceinline__ u32x4 codes8_bf16(uint32_t a, uint32_t b) {
  const u32x2 lo = codes4_bf16<BAD>(a), hi = codes4_bf16<BAD>(b);
  return u32x4{lo.x, lo.y, hi.x, hi.y};
}
// Four codes times 2^-LIFT as fp16: 1024 + (code + 128) is exact, and so is 1152 less.
template <bool BAD, int LIFT>
__device__ __forceinline__ u32x2 codes4_f16(uint32_t w) {
  constexpr float kDown = 1.f / (1 << LIFT);
  constexpr uint32_t kBad = 0xd800u - (LIFT << 10);  // -128 times 2^-LIFT
  const uint32_t u = w ^ 0x80808080u;
  u32x2 v;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t biased = __builtin_amdgcn_perm(0x64646464u, u, i ? 0x04030402u : 0x04010400u);
    const f16x2 h = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, biased), f16x2{(_Float16)kDown, (_Float16)kDown},
                                              f16x2{(_Float16)(-1152.f * kDown), (_Float16)(-1152.f * kDown)});
    uint32_t w2 = __builtin_bit_cast(uint32_t, h);
    if constexpr (BAD) {
      if ((w2 & 0xffffu) == kBad) w2 = (w2 & 0xffff0000u) | 0x7e00u;
      if ((w2 >> 16) == kBad) w2 = (w2 & 0xffffu) | 0x7e000000u;
    }
    v[i] = w2;
  }
  return v;
}
template <bool BAD, int LIFT>
__device__ __forceinline__ u32x4 codes8_f16(uint32_t a, uint32_t b) {
  const u32x2 lo = codes4_f16<BAD, LIFT>(a), hi = codes4_f16<BAD, LIFT>(b);
  return u32x4{lo.x, lo.y, hi.x, hi.y};
}
// Eight codes at scale s as bf16 values (what a block going back into the ring holds).
__device__ __forceinline__ u32x4 expand8(u32x2 w, float s) {
  const float a = fabsf(s);
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = (int8_t)(w[i / 2] >> (16 * (i & 1) + 8 * e));
      v[e] = c == -128 ? __uint_as_float(0x7fc00000u) : (float)c * a;
    }
    o[i] = pack_bf16x2(v[0], v[1]);
  }
  return o;
}

// Where one sequence's new tokens go, within 32 bits.
struct Span {
  int first;   // position of token 0
  int tokens;  // of this call
  int beg, end;  // positions written: those within the cache
};
__device__ __forceinline__ Span span_of(const Kv8Args& a, int b) {
  constexpr int64_t kFar = 1 << 30;
  const int64_t p = a.pos_dev ? a.pos_dev[b * a.pos_stride] : a.pos;
  int64_t n = a.lengths ? a.lengths[b] : a.T;
  n = n < 0 ? 0 : n > a.T ? a.T : n;
  Span s;
  s.first = (int)(p < -kFar ? -kFar : p > kFar ? kFar : p);
  s.tokens = (int)n;
  s.beg = s.first < 0 ? 0 : s.first;
  s.end = s.first + s.tokens < a.S ? s.first + s.tokens : a.S;
  if (s.end < s.beg) s.end = s.beg;
  return s;
}

// ---- write ------------------------------------------------------------------

// 17 blocks of 8 heads take 15 us, 16 sequences of 4000 tokens (8000 blocks) 132 us, 3 TB/s: the
// exact division of each entry and the turning of the values bound a block; one token of
// 16 sequences, without a block to pack, 3-5 us.
constexpr int kVRow = kBlk + 8;  // LDS row of a value column, padded against bank conflicts

template <int D>
struct WriteLds {
  uint16_t k[kBlk * D];
  uint16_t v[D * kVRow];
  float top[2][4];
  int bad[2][4];
};

// The largest finite |x| of eight bf16, and whether one is not finite.
__device__ __forceinline__ void top8(u32x4 v, float& top, int& bad) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float f = fabsf(__uint_as_float(e ? v[i] & 0xffff0000u : v[i] << 16));
      if (f < INFINITY) top = fmaxf(top, f);
      else bad = 1;
    }
}
__device__ __forceinline__ u32x2 code8(u32x4 v, float top) {
  u32x2 o = {0u, 0u};
  const float down = top > 1.f ? 0x1p-7f : 1.f;  // 127 f stays finite
  const float div = top * down;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float f = __uint_as_float(e ? v[i] & 0xffff0000u : v[i] << 16);
      // 127 f is exact: a tie of the quotient is seen as one
      const int c = !(fabsf(f) < INFINITY) ? -128 : top > 0.f ? (int)rintf(127.f * (f * down) / div) : 0;
      o[i / 2] |= (uint32_t)(uint8_t)(int8_t)c << (16 * (i & 1) + 8 * e);
    }
  return o;
}

// Two bf16 with an infinity as a NaN: an exponent of ones gets a bit in its fraction.
__device__ __forceinline__ uint32_t inf_to_nan(uint32_t w) {
  return w | ((((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 9);
}
__device__ __forceinline__ u32x2 inf_to_nan(u32x2 w) { return u32x2{inf_to_nan(w.x), inf_to_nan(w.y)}; }

template <int D>
__global__ __launch_bounds__(256) void kv8_write_kernel(Kv8Args a) {
  constexpr int LPH = D / 8, RPP = 256 / LPH;  // lanes per row, rows per pass
  __shared__ __attribute__((aligned(16))) WriteLds<D> sm;
  const int tid = threadIdx.x, j = tid % LPH;

  if ((int64_t)blockIdx.x >= (int64_t)a.B * a.Hk * a.touch) {  // q heads
    const int64_t items = (int64_t)a.B * a.T * a.Hq;
    int64_t item = ((int64_t)blockIdx.x - (int64_t)a.B * a.Hk * a.touch) * RPP + tid / LPH;
    const bool live = item < items;  // dead lanes stay for the cross-lane sums
    if (!live) item = items - 1;
    const int64_t m = item / a.Hq, h = item - m * a.Hq, t = m % a.T;
    const uint16_t* src = a.q + m * a.ldq + h * D;
    u32x2 lo = *reinterpret_cast<const u32x2*>(src + 4 * j);
    u32x2 hi = *reinterpret_cast<const u32x2*>(src + D / 2 + 4 * j);
    norm_rope_row<D>(lo, hi, a.gq, a.epsq, a.cos + t * a.ldc, a.sin + t * a.lds, j);
    if (!live) return;
    uint16_t* dst = a.qn + item * D;
    *reinterpret_cast<u32x2*>(dst + 4 * j) = lo;
    *reinterpret_cast<u32x2*>(dst + D / 2 + 4 * j) = hi;
    return;
  }

  const int bh = blockIdx.x / a.touch, b = bh / a.Hk, h = bh - b * a.Hk;
  const Span s = span_of(a, b);
  if (s.beg >= s.end) return;
  const int fb = s.beg / kBlk, lb = (s.end - 1) / kBlk;  // blocks touched
  const int blk = fb + (int)(blockIdx.x - (int64_t)bh * a.touch);
  if (blk > lb) return;
  const int row0 = blk == fb ? s.beg - fb * kBlk : 0;
  const int row1 = blk == lb ? s.end - lb * kBlk : kBlk;
  const int slot = blk & 1;
  const bool complete = row1 == kBlk, in_tail = blk >= lb - 1, have_old = row0 > 0;
  // Of the last two blocks, which stay in bf16, the one in the slot that the first
  // block's old rows are read from is stored by that block's workgroup, after it has
  // read them.
  const bool old_first = s.beg % kBlk != 0 && fb < lb - 1;
  const int after = ((lb ^ fb) & 1) ? lb - 1 : lb;  // of {lb - 1, lb}, the one in fb's slot
  const bool tag_ok = have_old && a.tail_block[bh * 2 + slot] == blk;
  const int64_t at = (int64_t)bh * a.NB + blk;
  int8_t* kc = a.k_codes + at * (kBlk * D);
  int8_t* vc = a.v_codes + at * (kBlk * D);
  auto tail_k = [&](int sl) { return a.k_tail + ((int64_t)bh * 2 + sl) * (kBlk * D); };
  auto tail_v = [&](int sl) { return a.v_tail + ((int64_t)bh * 2 + sl) * (kBlk * D); };

  // rows r0 .. r1-1 of block w: into the ring, or into LDS
  auto put = [&](int w, int r0, int r1, bool ring) {
    constexpr int NP = kBlk / RPP;
    uint16_t* tk = tail_k(w & 1);
    uint16_t* tv = tail_v(w & 1);
    u32x2 lo[NP], hi[NP], v0[NP], v1[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {  // every row's loads before the first store
      const int r = r0 + tid / LPH + p * RPP;
      if (r >= r1) continue;
      const int64_t m = (int64_t)b * a.T + (w * kBlk + r - s.first);
      const uint16_t* ks = a.k + m * a.ldk + (int64_t)h * D;
      const uint16_t* vs = a.v + m * a.ldv + (int64_t)h * D;
      lo[p] = *reinterpret_cast<const u32x2*>(ks + 4 * j);
      hi[p] = *reinterpret_cast<const u32x2*>(ks + D / 2 + 4 * j);
      v0[p] = *reinterpret_cast<const u32x2*>(vs + 8 * j);
      v1[p] = *reinterpret_cast<const u32x2*>(vs + 8 * j + 4);
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int r = r0 + tid / LPH + p * RPP, t = w * kBlk + r - s.first;
      if (r >= r1) continue;
      if (a.cos) norm_rope_row<D>(lo[p], hi[p], a.gk, a.epsk, a.cos + t * a.ldc, a.sin + t * a.lds, j);
      if (w >= lb - 1)  // a block that goes into the ring
        lo[p] = inf_to_nan(lo[p]), hi[p] = inf_to_nan(hi[p]), v0[p] = inf_to_nan(v0[p]), v1[p] = inf_to_nan(v1[p]);
      const uint32_t vv[4] = {v0[p].x, v0[p].y, v1[p].x, v1[p].y};
      if (ring) {
        *reinterpret_cast<u32x2*>(tk + r * D + 4 * j) = lo[p];
        *reinterpret_cast<u32x2*>(tk + r * D + D / 2 + 4 * j) = hi[p];
#pragma unroll
        for (int e = 0; e < 8; ++e) tv[(8 * j + e) * kBlk + r] = (uint16_t)(vv[e / 2] >> (16 * (e & 1)));
      } else {
        *reinterpret_cast<u32x2*>(sm.k + r * D + 4 * j) = lo[p];
        *reinterpret_cast<u32x2*>(sm.k + r * D + D / 2 + 4 * j) = hi[p];
#pragma unroll
        for (int e = 0; e < 8; ++e) sm.v[(8 * j + e) * kVRow + r] = (uint16_t)(vv[e / 2] >> (16 * (e & 1)));
      }
    }
  };

  // LDS rows 0 .. n-1 into a slot of the ring (of a value column's last eight, anything
  // behind them)
  auto keep = [&](int sl, int n) {
    for (int i = tid; i < n * (D / 8); i += 256)
      reinterpret_cast<u32x4*>(tail_k(sl))[i] = reinterpret_cast<const u32x4*>(sm.k)[i];
    const int nc = (n + 7) / 8;
    for (int i = tid; i < D * nc; i += 256) {
      const int d = i / nc, c = (i % nc) * 8;
      *reinterpret_cast<u32x4*>(tail_v(sl) + d * kBlk + c) = *reinterpret_cast<const u32x4*>(sm.v + d * kVRow + c);
    }
  };

  const bool mine = !(old_first && blk == after);  // whether this workgroup stores its block's ring
  if (!complete && !mine) return;
  const bool assemble = complete || (have_old && !tag_ok);
  // most calls of one token: nothing but its rows; more than a few of them as single
  // elements of the value columns cost more than the way through LDS
  if (!assemble && (have_old || row1 < 8)) {
    put(blk, row0, row1, true);
    if (!have_old && tid == 0) a.tail_block[bh * 2 + slot] = blk;
    return;
  }
  if (have_old) {
    const float ksc = a.k_scale[at], vsc = a.v_scale[at];
    for (int i = tid; i < row0 * (D / 8); i += 256) {
      const int r = i / (D / 8), c = (i % (D / 8)) * 8;
      *reinterpret_cast<u32x4*>(sm.k + r * D + c) =
          tag_ok ? ld16(tail_k(slot) + r * D + c) : expand8(*reinterpret_cast<const u32x2*>(kc + r * D + c), ksc);
    }
    const int nc = (row0 + 7) / 8;
    for (int i = tid; i < D * nc; i += 256) {
      const int d = i / nc, c = (i % nc) * 8;
      *reinterpret_cast<u32x4*>(sm.v + d * kVRow + c) =
          tag_ok ? ld16(tail_v(slot) + d * kBlk + c) : expand8(*reinterpret_cast<const u32x2*>(vc + d * kBlk + c), vsc);
    }
  }
  __syncthreads();  // the old rows' last chunk reaches into the new rows
  put(blk, row0, row1, false);
  __syncthreads();
  if (in_tail && mine) {  // the whole block: its old rows may not be in the ring
    keep(slot, row1);
    if (tid == 0) a.tail_block[bh * 2 + slot] = blk;
  }
  if (!complete) return;

  constexpr int NC = kBlk * D / 8 / 256;  // chunks of 8 per thread
  u32x4 kx[NC], vx[NC];
  float top[2] = {0.f, 0.f};
  int bad[2] = {0, 0};
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int i = n * 256 + tid;
    kx[n] = reinterpret_cast<const u32x4*>(sm.k)[i];
    vx[n] = *reinterpret_cast<const u32x4*>(sm.v + (i / 8) * kVRow + (i % 8) * 8);
    top8(kx[n], top[0], bad[0]);
    top8(vx[n], top[1], bad[1]);
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) top[w] = fmaxf(top[w], __shfl_xor(top[w], off));
    bad[w] = __any(bad[w]);
    if ((tid & 63) == 0) sm.top[w][tid >> 6] = top[w], sm.bad[w][tid >> 6] = bad[w];
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    top[w] = fmaxf(fmaxf(sm.top[w][0], sm.top[w][1]), fmaxf(sm.top[w][2], sm.top[w][3]));
    bad[w] = sm.bad[w][0] | sm.bad[w][1] | sm.bad[w][2] | sm.bad[w][3];
  }
  if (tid == 0) {
    const float ks = top[0] / 127.f, vs = top[1] / 127.f;
    a.k_scale[at] = bad[0] ? -ks : ks;  // -0 counts as negative
    a.v_scale[at] = bad[1] ? -vs : vs;
  }
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int i = n * 256 + tid;
    reinterpret_cast<u32x2*>(kc)[i] = code8(kx[n], top[0]);
    reinterpret_cast<u32x2*>(vc)[i] = code8(vx[n], top[1]);
  }
  if (old_first && blk == fb) {  // `after`, behind the old rows and the packed block
    const int n = after == lb ? s.end - lb * kBlk : kBlk;
    put(after, 0, n, false);
    __syncthreads();
    keep(slot, n);
    if (tid == 0) a.tail_block[bh * 2 + slot] = after;
  }
}

// The values of positions pos .. pos + T - 1 of sequences that end there, in fp32:
// a workgroup per 16 (D 128) or 32 tokens of a kv head.
template <int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8Args a, float* ko, float* vo) {
  constexpr int LPH = D / 8, RPP = 256 / LPH;
  const int groups = (a.T + RPP - 1) / RPP;
  const int bh = blockIdx.x / groups, b = bh / a.Hk, h = bh - b * a.Hk;
  const int t = (int)(blockIdx.x - (int64_t)bh * groups) * RPP + threadIdx.x / LPH, j = threadIdx.x % LPH;
  if (t >= a.T) return;
  const Span s = span_of(a, b);
  const int p = s.first + t;
  float kv[8] = {}, vv[8] = {};
  if (p >= s.beg && p < s.end) {
    const int blk = p / kBlk, r = p % kBlk, slot = blk & 1;
    const int64_t at = (int64_t)bh * a.NB + blk, tl = ((int64_t)bh * 2 + slot) * (kBlk * D);
    if (blk == s.end / kBlk && a.tail_block[bh * 2 + slot] == blk) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        kv[e] = bf16_bits_to_f32(a.k_tail[tl + r * D + 8 * j + e]);
        vv[e] = bf16_bits_to_f32(a.v_tail[tl + (8 * j + e) * kBlk + r]);
      }
    } else {
      const float ks = fabsf(a.k_scale[at]), vs = fabsf(a.v_scale[at]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int kc = a.k_codes[at * (kBlk * D) + r * D + 8 * j + e];
        const int vc = a.v_codes[at * (kBlk * D) + (8 * j + e) * kBlk + r];
        kv[e] = kc == -128 ? __uint_as_float(0x7fc00000u) : (float)kc * ks;
        vv[e] = vc == -128 ? __uint_as_float(0x7fc00000u) : (float)vc * vs;
      }
    }
  }
  const int64_t o = (((int64_t)b * a.T + t) * a.Hk + h) * D + 8 * j;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    reinterpret_cast<f32x4*>(ko + o)[e] = f32x4{kv[4 * e], kv[4 * e + 1], kv[4 * e + 2], kv[4 * e + 3]};
    reinterpret_cast<f32x4*>(vo + o)[e] = f32x4{vv[4 * e], vv[4 * e + 1], vv[4 * e + 2], vv[4 * e + 3]};
  }
}

// ---- attention --------------------------------------------------------------

// Last key that query row rr (token rr / G) sees; -1: none (a token past the
// sequence's own, or at a position outside the cache).
__device__ __forceinline__ int last_key(const Span& s, int t) {
  const int p = s.first + t;
  return t < s.tokens && p >= s.beg && p < s.end ? p : -1;
}

// One softmax step over the 16 keys that a lane holds of each of its row columns:
// scores x (in units of log 2) to probabilities times 2^kLiftRows, m and l (of such
// probabilities) updated; returns what the row's earlier sums are multiplied by.
__device__ __forceinline__ float softmax_step(f32x4 (&x)[4], float& mx, float& sum) {
  float m = -INFINITY;
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) m = fmaxf(m, x[n][r]);
  const float mn = fmaxf(mx, col_max(m));
  const float base = mn == -INFINITY ? 0.f : mn;
  const float al = exp2_fast(mx - base), lift = base - kLiftRows;
  mx = mn;
  float l = 0.f;
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[n][r] = exp2_fast(x[n][r] - lift);
      l += x[n][r];
    }
  sum = sum * al + l;
  return al;
}
// Its probabilities as the two B operands of 32 keys.
__device__ __forceinline__ void p_operands(const f32x4 (&x)[4], u32x4 (&pf)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    pf[i] = u32x4{pack_f16x2(x[2 * i][0], x[2 * i][1]), pack_f16x2(x[2 * i][2], x[2 * i][3]),
                  pack_f16x2(x[2 * i + 1][0], x[2 * i + 1][1]), pack_f16x2(x[2 * i + 1][2], x[2 * i + 1][3])};
}

__device__ __forceinline__ int64_t part_row(const Kv8Args& a, int split, int bh, int64_t rr) {
  return ((int64_t)split * a.B * a.Hk + bh) * ((int64_t)a.T * (a.Hq / a.Hk)) + rr;
}

// ... and as those of their bf16 values (times 2^-LIFT) and of what is left: p to 2^-17 of itself.
template <int LIFT>
__device__ __forceinline__ void p_operands_bf16(const f32x4 (&x)[4], u32x4 (&hi)[2], u32x4 (&lo)[2]) {
  constexpr float kDown = 1.f / (1 << LIFT);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = x[2 * i + w / 2][2 * (w & 1)] * kDown, b = x[2 * i + w / 2][2 * (w & 1) + 1] * kDown;
      const uint32_t h = pack_bf16x2(a, b);
      hi[i][w] = h;
      lo[i][w] = pack_bf16x2(a - __uint_as_float(h << 16), b - __uint_as_float(h & 0xffff0000u));
    }
}

// Decode and verify. A workgroup takes one kv head of one sequence, 16 * RT query
// rows (token t, group head g at row t * G + g) and one contiguous range of blocks;
// its four waves take blocks w, w + 4, ... of the range straight into registers (buffers
// that end with the last whole block return zeros past it, so loads are issued without a
// branch) and merge their softmax
// states through LDS in wave order. 16 sequences of 4000 tokens, 32 heads over 8: 23.5 us
// and 4 us to combine, 4.3 TB/s of codes (RT 1: two workgroups per CU); five tokens at 65001:
// 36 us, 3.7 TB/s (RT 2: one workgroup per CU, 109 registers would spill at two); one token
// at 333: 7.5 us, of which most is the way to the first scores and through the merge.
template <int D, int RT>
__global__ __launch_bounds__(256, RT == 1 ? 2 : 1) void kv8_rows_kernel(Kv8Args a) {
  constexpr int NW = 4, DK = D / 32, DT = D / 16, KU = D / 64;
  __shared__ __attribute__((aligned(16))) float sO[NW][16 * RT][D + 4];
  __shared__ float sM[NW][16 * RT], sL[NW][16 * RT];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, grp = lane >> 4;
  const int G = a.Hq / a.Hk, rows = a.T * G;
  const int bh = blockIdx.y, b = bh / a.Hk, kh = bh - b * a.Hk;
  const int row0 = blockIdx.z * 16 * RT;
  const Span s = span_of(a, b);
  const int end = s.beg < s.end ? s.end : 0;  // no live row: no keys
  const int nc = (end + kBlk - 1) / kBlk, full = end / kBlk;
  const int per = (nc + a.nsplit - 1) / a.nsplit;
  const int c_lo = (int)blockIdx.x * per, c_hi = c_lo + per < nc ? c_lo + per : nc;
  const int f_hi = c_hi < full ? c_hi : full;  // whole blocks of the range

  // q of this lane's row columns, in the order of the keys' 16-byte loads: step
  // 2u + h holds elements 64 u + 16 grp + 8 h ..
  u32x4 qf[RT][DK];
  int lim[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int rr = row0 + rt * 16 + li;
    if (rr >= rows) rr = rows - 1;
    const int t = rr / G, h = kh * G + (rr - t * G);
    lim[rt] = last_key(s, t);
    const uint16_t* qp = a.qsrc + ((int64_t)b * a.T + t) * a.ldqs + (int64_t)h * D + 16 * grp;
#pragma unroll
    for (int i = 0; i < DK; ++i) qf[rt][i] = ld16_any(qp + 64 * (i / 2) + 8 * (i & 1));
  }

  const int64_t at = (int64_t)bh * a.NB;
  const __amdgpu_buffer_rsrc_t kr = make_rsrc(a.k_codes + at * (kBlk * D), (int64_t)full * (kBlk * D));
  const __amdgpu_buffer_rsrc_t vr = make_rsrc(a.v_codes + at * (kBlk * D), (int64_t)full * (kBlk * D));
  const __amdgpu_buffer_rsrc_t ksr = make_rsrc(a.k_scale + at, (int64_t)full * 4);
  const __amdgpu_buffer_rsrc_t vsr = make_rsrc(a.v_scale + at, (int64_t)full * 4);
  const uint32_t koff = (uint32_t)((16 * (li >> 2) + (li & 3)) * D + 16 * grp);
  const uint32_t voff = (uint32_t)(li * kBlk + 16 * grp);

  const float sc = kLog2e / sqrtf((float)D);
  f32x4 o[DT][RT];
  float mx[RT], sum[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    mx[rt] = -INFINITY;
    sum[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // one block's codes: a block's keys come in behind the last one's values and its values
  // behind its scores, each into the registers that have just been used, its scales before
  u32x4 xk[4][KU], xv[DT];
  float ks, vs, ks_next, vs_next;
  auto load_s = [&](int c) __attribute__((always_inline)) {
    const uint32_t sb = c < f_hi ? (uint32_t)c * 4 : 0x7fff0000u;
    ks_next = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ksr, sb, 0, 0));
    vs_next = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(vsr, sb, 0, 0));
  };
  auto load_k = [&](int c) __attribute__((always_inline)) {
    const uint32_t base = c < f_hi ? (uint32_t)c * (kBlk * D) : 0x7fff0000u;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int u = 0; u < KU; ++u)
        xk[n][u] = __builtin_amdgcn_raw_buffer_load_b128(kr, base + koff + 4 * n * D + 64 * u, 0, 0);
  };
  auto load_v = [&](int c) __attribute__((always_inline)) {
    const uint32_t base = c < f_hi ? (uint32_t)c * (kBlk * D) : 0x7fff0000u;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      xv[dt] = __builtin_amdgcn_raw_buffer_load_b128(vr, base + voff + dt * 16 * kBlk, 0, 0);
  };
  // scores of block c at factor f to probabilities of row column rt; what o is multiplied by
  auto softmax = [&](const f32x4 (&x)[4][RT], int rt, int c, float f, f32x4 (&y)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        y[n][r] = c * kBlk + 16 * grp + 4 * n + r <= lim[rt] ? x[n][rt][r] * f : -INFINITY;
    return softmax_step(y, mx[rt], sum[rt]);
  };
  auto compute = [&](int c, auto bad) __attribute__((always_inline)) {
    constexpr bool BAD = decltype(bad)::value;
    f32x4 y[4][RT];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) y[n][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 kf = codes8_bf16<BAD>(xk[n][u][2 * h], xk[n][u][2 * h + 1]);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) y[n][rt] = mfma16(kf, qf[rt][2 * u + h], y[n][rt]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_k(c + NW);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 pf[RT][2];
    float al[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      f32x4 p[4];
      al[rt] = softmax(y, rt, c, fabsf(ks) * sc, p);
      p_operands(p, pf[rt]);
    }
    const float f = fabsf(vs);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const u32x4 v0 = codes8_f16<BAD, kLiftRows>(xv[dt][0], xv[dt][1]);
      const u32x4 v1 = codes8_f16<BAD, kLiftRows>(xv[dt][2], xv[dt][3]);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x4 pv = mfma16h(v0, pf[rt][0], f32x4{0.f, 0.f, 0.f, 0.f});
        pv = mfma16h(v1, pf[rt][1], pv);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[dt][rt][r] = fmaf(pv[r], f, o[dt][rt][r] * al[rt]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_v(c + NW);
    __builtin_amdgcn_sched_barrier(0);
  };

  load_s(c_lo + wave);
  load_k(c_lo + wave);
  load_v(c_lo + wave);
  // q has arrived (a load pending at the loop's entry would be waited for in every round)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int i = 0; i < DK; ++i) asm volatile("" : "+v"(qf[rt][i]));
  for (int c = c_lo + wave; c < f_hi; c += NW) {
    ks = ks_next, vs = vs_next;
    load_s(c + NW);
    const uint32_t sign = (__float_as_uint(ks) | __float_as_uint(vs)) >> 31;
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(sign), 0)) compute(c, std::true_type{});
    else compute(c, std::false_type{});
  }

  // the unfinished block, from the ring: the wave whose turn it is
  if (full < c_hi && c_lo <= full && ((full - c_lo) & (NW - 1)) == wave) {
    const int64_t tl = ((int64_t)bh * 2 + (full & 1)) * (kBlk * D);
    const uint16_t* kt = a.k_tail + tl;
    const uint16_t* vt = a.v_tail + tl;
    u32x4 k[4][DK], v[DT][2];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < DK; ++i) k[n][i] = ld16(kt + koff + 4 * n * D + 64 * (i / 2) + 8 * (i & 1));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 2; ++i) v[dt][i] = ld16(vt + voff + dt * 16 * kBlk + 8 * i);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 y[4][RT];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) y[n][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DK; ++i)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) y[n][rt] = mfma16(k[n][i], qf[rt][i], y[n][rt]);
    }
    u32x4 hi[RT][2], lo[RT][2], live[2];
    float al[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      f32x4 p[4];
      al[rt] = softmax(y, rt, full, sc, p);
      p_operands_bf16<kLiftRows>(p, hi[rt], lo[rt]);
    }
    const int left = end - full * kBlk - 16 * grp;  // of the lane group's 16 keys
#pragma unroll
    for (int i = 0; i < 2; ++i)  // the ring holds anything past the last key
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int key = 8 * i + 2 * w;
        live[i][w] = key + 1 < left ? ~0u : key < left ? 0xffffu : 0u;
      }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const u32x4 v0 = v[dt][0] & live[0], v1 = v[dt][1] & live[1];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x4 pv = mfma16(v0, hi[rt][0], f32x4{0.f, 0.f, 0.f, 0.f});
        pv = mfma16(v1, hi[rt][1], pv);
        pv = mfma16(v0, lo[rt][0], pv);
        pv = mfma16(v1, lo[rt][1], pv);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[dt][rt][r] = fmaf(o[dt][rt][r], al[rt], pv[r]);
      }
    }
  }

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float l = col_sum(sum[rt]) * (1.f / (1 << kLiftRows));
    if (grp == 0) {
      sM[wave][rt * 16 + li] = mx[rt];
      sL[wave][rt * 16 + li] = l;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<f32x4*>(&sO[wave][rt * 16 + li][dt * 16 + 4 * grp]) = o[dt][rt];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * RT * (D / 4); i += NW * 64) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4, rr = row0 + r;
    if (rr >= rows) continue;
    float m = sM[0][r];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, sM[w][r]);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float e = exp2_fast(sM[w][r] - base);
      l += e * sL[w][r];
      v += *reinterpret_cast<const f32x4*>(&sO[w][r][d]) * e;
    }
    if (a.nsplit > 1) {
      const int64_t pr = part_row(a, blockIdx.x, bh, rr);
      *reinterpret_cast<f32x4*>(a.part + pr * D + d) = v;
      if (d == 0) *reinterpret_cast<f32x2*>(a.stat + pr * 2) = f32x2{m, l};
    } else {
      const int t = rr / G, h = kh * G + (rr - t * G);
      if (l == 0.f) v = f32x4{0.f, 0.f, 0.f, 0.f}, l = 1.f;  // a row that sees no key
      *reinterpret_cast<u32x2*>(a.y + (((int64_t)b * a.T + t) * a.Hq + h) * D + d) =
          u32x2{pack_bf16x2(v[0] / l, v[1] / l), pack_bf16x2(v[2] / l, v[3] / l)};
    }
  }
}

// Prompts. A workgroup takes one kv head of one sequence and 64 query rows (wave w rows
// 16 w ..), and walks its blocks: codes into registers one block ahead, then converted once
// for the four waves into LDS (keys bf16, values fp16, both double-buffered), one
// barrier per block. p is taken relative to a maximum that is moved only when the running
// one has passed it by kRise (fp16 and the sums have room), so that a block seldom
// rescales o. 128 rows to a workgroup of four waves halve the conversions and the LDS reads but
// leave the registers no room: 8192 tokens of 16 heads 617 us against 580.
// 1000 tokens at 1037, 32 heads: 65 us, 390 TFLOP/s; 2048 at 30000, 16 heads: 877 us with its
// write, 590 TFLOP/s: bound by the vector unit (softmax and conversions) beside the matrix core.
template <int D>
__global__ __launch_bounds__(256, 2) void kv8_tiles_kernel(Kv8Args a, int n_rt) {
  constexpr int DK = D / 32, DT = D / 16;
  constexpr int NL = kBlk * D / 16 / 256;  // 16-code chunks per thread
  constexpr int CH = D / 8;                // 16-byte chunks of a key row in LDS
  constexpr uint32_t SZ = kBlk * D * 2;
  __shared__ __attribute__((aligned(16))) char sm[4 * SZ];  // keys, keys, values, values

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, grp = lane >> 4;
  const int G = a.Hq / a.Hk, rows = a.T * G;
  const int bh = blockIdx.y, b = bh / a.Hk, kh = bh - b * a.Hk;
  // the tiles with the most keys first; where the whole grid is resident at once (two
  // workgroups per CU) its second half goes the other way, so that a CU's two make up for each other
  const bool back = (int64_t)gridDim.x * gridDim.y * gridDim.z <= 512 && 2 * blockIdx.y >= gridDim.y;
  const int tile = back ? (int)blockIdx.x : n_rt - 1 - (int)blockIdx.x;
  const int row0 = tile * 64 + wave * 16;
  const Span s = span_of(a, b);
  const int end = s.beg < s.end ? s.end : 0;
  const int full = end / kBlk;
  // keys this workgroup's last row sees
  int last = (tile + 1) * 64 - 1;
  if (last >= rows) last = rows - 1;
  const int64_t seen = (int64_t)s.first + last / G + 1;
  const int kend = seen < 0 ? 0 : seen < end ? (int)seen : end;
  const int nt = (kend + kBlk - 1) / kBlk;
  const int per = (nt + a.nsplit - 1) / a.nsplit;
  const int t_lo = (int)blockIdx.z * per, t_hi = t_lo + per < nt ? t_lo + per : nt;

  const int rr = row0 + li < rows ? row0 + li : rows - 1;
  const int tq = rr / G, hq = kh * G + (rr - tq * G), lim = last_key(s, tq);
  const uint16_t* qp = a.qsrc + ((int64_t)b * a.T + tq) * a.ldqs + (int64_t)hq * D + 8 * grp;
  u32x4 qf[DK];
#pragma unroll
  for (int i = 0; i < DK; ++i) qf[i] = ld16_any(qp + 32 * i);
  // the least and the largest last key of the wave's rows
  int lo = lim, hi = lim;
#pragma unroll
  for (int off = 1; off < 16; off <<= 1) {
    const int x = __shfl_xor(lo, off), y = __shfl_xor(hi, off);
    lo = x < lo ? x : lo;
    hi = y > hi ? y : hi;
  }
  const int lim_lo = __builtin_amdgcn_readfirstlane(lo), lim_hi = __builtin_amdgcn_readfirstlane(hi);

  const int64_t at = (int64_t)bh * a.NB;
  // LDS places: key row r's chunk c at c ^ (4 (r / 16) + r % 4) (16 rows that a read
  // takes together differ there), value row d's chunk at c ^ (d % 8)
  auto k_at = [](int r, int c) { return (uint32_t)(r * (D * 2) + ((c ^ (((r >> 4) * 4 + (r & 3)) & (CH - 1))) * 16)); };
  auto v_at = [](int d, int c) { return (uint32_t)(d * (kBlk * 2) + ((c ^ (d & 7)) * 16)); };
  // where this lane reads (tile n of the keys 4 n rows on, value block dt 16 dt rows on) and
  // puts its codes (the second half of 16 codes one chunk on: 16 off by an exclusive or)
  uint32_t k_rd[DK], v_rd[2], k_wr[NL];
#pragma unroll
  for (int i = 0; i < DK; ++i) k_rd[i] = k_at(16 * (li >> 2) + (li & 3), 4 * i + grp);
#pragma unroll
  for (int i = 0; i < 2; ++i) v_rd[i] = v_at(li, 2 * grp + i);
#pragma unroll
  for (int n = 0; n < NL; ++n) k_wr[n] = k_at((n * 256 + tid) / (D / 16), (n * 256 + tid) % (D / 16) * 2);
  const uint32_t v_wr = v_at(tid / 4, tid % 4 * 2);  // 64 n rows on
  u32x4 kx[NL], vx[NL];
  float ksc = 0.f, vsc = 0.f, ks_next = 0.f, vs_next = 0.f;
  auto load = [&](int kt) __attribute__((always_inline)) {
    if (kt >= full) return;
    ks_next = a.k_scale[at + kt], vs_next = a.v_scale[at + kt];
    const u32x4* kc = reinterpret_cast<const u32x4*>(a.k_codes + (at + kt) * (kBlk * D));
    const u32x4* vc = reinterpret_cast<const u32x4*>(a.v_codes + (at + kt) * (kBlk * D));
#pragma unroll
    for (int n = 0; n < NL; ++n) kx[n] = kc[n * 256 + tid], vx[n] = vc[n * 256 + tid];
  };
  auto st = [&](uint32_t at, u32x4 x) { *reinterpret_cast<u32x4*>(sm + at) = x; };
  auto put = [&](uint32_t k, uint32_t v, auto bad) __attribute__((always_inline)) {
    constexpr bool BAD = decltype(bad)::value;
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      st(k + k_wr[n], codes8_bf16<BAD>(kx[n][0], kx[n][1]));
      st(k + (k_wr[n] ^ 16), codes8_bf16<BAD>(kx[n][2], kx[n][3]));
      st(v + v_wr + n * (64 * kBlk * 2), codes8_f16<BAD, kLiftTiles>(vx[n][0], vx[n][1]));
      st(v + (v_wr ^ 16) + n * (64 * kBlk * 2), codes8_f16<BAD, kLiftTiles>(vx[n][2], vx[n][3]));
    }
  };
  // block kt (loaded before, if whole) into LDS; its scales into ks, vs
  auto store = [&](uint32_t k, uint32_t v, int kt, float& ks, float& vs) __attribute__((always_inline)) {
    if (kt < full) {
      // not before here: the compiler would pull the conversions' shifts up to the loads
      // and wait for them there
#pragma unroll
      for (int n = 0; n < NL; ++n) asm volatile("" : "+v"(kx[n]), "+v"(vx[n]));
      const float k0 = ks_next, v0 = vs_next;
      const uint32_t sign = (__float_as_uint(k0) | __float_as_uint(v0)) >> 31;
      if (__builtin_expect(__builtin_amdgcn_readfirstlane(sign), 0)) put(k, v, std::true_type{});
      else put(k, v, std::false_type{});
      ks = fabsf(k0), vs = fabsf(v0);
      return;
    }
    const int64_t tl = ((int64_t)bh * 2 + (full & 1)) * (kBlk * D);
    constexpr int NT = kBlk * D / 8 / 256;
    const int n_rows = end - full * kBlk;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int i = n * 256 + tid;
      st(k + k_at(i / CH, i % CH), ld16(a.k_tail + tl + i * 8));
      u32x4 vv = ld16(a.v_tail + tl + i * 8);
#pragma unroll
      for (int w = 0; w < 4; ++w) {  // the ring holds anything past the last key
        const int key = (i % 8) * 8 + 2 * w;
        if (key >= n_rows) vv[w] = 0u;
        else if (key + 1 >= n_rows) vv[w] &= 0xffffu;
      }
      st(v + v_at(i / 8, i % 8), vv);
    }
    ks = 1.f, vs = 1.f;
  };

  const float sc = kLog2e / sqrtf((float)D);
  f32x4 o[DT], sum = {0.f, 0.f, 0.f, 0.f};  // sum: of p, four equal rows of ones (by 2^kLift) times p
  float mx = -INFINITY;  // what p is relative to: at most kRise under the running maximum
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto step = [&](uint32_t k, uint32_t v, int kt, float ks, float vs, auto tail) __attribute__((always_inline)) {
    if (kt * kBlk > lim_hi) return;  // every key hidden from every row
    f32x4 x[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      x[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DK; ++i) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(sm + (k + k_rd[i]) + 4 * n * (D * 2));
        x[n] = mfma16(kf, qf[i], x[n]);
      }
    }
    // the values' reads go out behind the scores, ahead of the softmax
    u32x4 vf[DT][2];
    auto read_v = [&](int dt) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) vf[dt][i] = *reinterpret_cast<const u32x4*>(sm + (v + v_rd[i]) + dt * 16 * (kBlk * 2));
    };
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) read_v(dt);
    __builtin_amdgcn_sched_barrier(0);
    const float f = ks * sc;
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < 4; ++n) x[n] *= f;
    if (kt * kBlk + kBlk - 1 > lim_lo) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[n][r] = kt * kBlk + 16 * grp + 4 * n + r <= lim ? x[n][r] : -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, x[n][r]);
    top = col_max(top);
    const bool rise = top > mx + kRise;
    if (__ballot(rise)) {
      const float to = rise ? top : mx;
      const float al = exp2_fast(mx - (to == -INFINITY ? 0.f : to));
      mx = to;
      sum *= al;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= al;
    }
    const float lift = (mx == -INFINITY ? 0.f : mx) - kLiftTiles;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[n][r] = exp2_fast(x[n][r] - lift);
    if constexpr (decltype(tail)::value) {  // bf16 values
      u32x4 ph[2], pl[2];
      p_operands_bf16<kLiftTiles>(x, ph, pl);
      constexpr u32x4 kOnes = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
      for (int i = 0; i < 2; ++i) sum = mfma16(kOnes, pl[i], mfma16(kOnes, ph[i], sum));
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 2; ++i) o[dt] = mfma16(vf[dt][i], pl[i], mfma16(vf[dt][i], ph[i], o[dt]));
      return;
    }
    u32x4 pf[2];
    p_operands(x, pf);
    constexpr uint32_t kOne = (0x3c00u - (kLiftTiles << 10)) * 0x10001u;  // 2^-kLiftTiles, as the codes have it
    constexpr u32x4 kOnes = {kOne, kOne, kOne, kOne};
#pragma unroll
    for (int i = 0; i < 2; ++i) sum = mfma16h(kOnes, pf[i], sum);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      f32x4 pv = mfma16h(vf[dt][0], pf[0], f32x4{0.f, 0.f, 0.f, 0.f});
      pv = mfma16h(vf[dt][1], pf[1], pv);
#pragma unroll
      for (int r = 0; r < 4; ++r) o[dt][r] = fmaf(pv[r], vs, o[dt][r]);
    }
  };

  // q has arrived: a load pending at the loop's entry would have the compiler wait, in
  // every round, for the loads of the next block too
#pragma unroll
  for (int i = 0; i < DK; ++i) asm volatile("" : "+v"(qf[i]));
  if (t_lo < t_hi) {
    load(t_lo);
    store(0, 2 * SZ, t_lo, ksc, vsc);
    __syncthreads();
    const int f_hi = t_hi < full ? t_hi : full;
    uint32_t u = 0;
    for (int kt = t_lo; kt < f_hi; ++kt, u ^= SZ) {
      const bool more = kt + 1 < t_hi;
      if (more) load(kt + 1);
      step(u, 2 * SZ + u, kt, ksc, vsc, std::false_type{});
      if (more) {
        store(u ^ SZ, 2 * SZ + (u ^ SZ), kt + 1, ksc, vsc);
        __syncthreads();
      }
    }
    if (f_hi < t_hi) step(u, 2 * SZ + u, full, 1.f, 1.f, std::true_type{});
  }

  if (row0 + li >= rows) return;
  const float l = sum[0];
  if (a.nsplit > 1) {
    const int64_t pr = part_row(a, blockIdx.z, bh, rr);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(a.part + pr * D + dt * 16 + 4 * grp) = o[dt];
    if (grp == 0) *reinterpret_cast<f32x2*>(a.stat + pr * 2) = f32x2{mx, l};
    return;
  }
  const bool none = l == 0.f;  // a row that sees no key
  uint16_t* yp = a.y + (((int64_t)b * a.T + tq) * a.Hq + hq) * D + 4 * grp;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    *reinterpret_cast<u32x2*>(yp + dt * 16) =
        none ? u32x2{0u, 0u} : u32x2{pack_bf16x2(o[dt][0] / l, o[dt][1] / l), pack_bf16x2(o[dt][2] / l, o[dt][3] / l)};
}

// One output row per workgroup: lane s of each wave holds split s's statistics; each
// group of D / 4 threads sums every NG-th split's partials, then the groups in order.
template <int D>
__global__ __launch_bounds__(256) void kv8_combine_kernel(Kv8Args a) {
  constexpr int LPR = D / 4, NG = 256 / LPR;
  __shared__ __attribute__((aligned(16))) f32x4 part[NG][LPR];
  const int rows = a.T * (a.Hq / a.Hk);
  const int64_t total = (int64_t)a.B * a.Hk * rows, i = blockIdx.x;
  const int lane = threadIdx.x & 63, grp = threadIdx.x / LPR, q = threadIdx.x % LPR;
  const bool has = lane < a.nsplit;
  f32x2 st = {-INFINITY, 0.f};
  if (has) st = *reinterpret_cast<const f32x2*>(a.stat + (lane * total + i) * 2);
  float m = st.x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off));
  const float base = m == -INFINITY ? 0.f : m;
  const float e = has ? exp2_fast(st.x - base) : 0.f;
  float l = wave_sum(has ? e * st.y : 0.f);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int n = 0; n < kKv8MaxSplit / NG; ++n) {
    const int s = n * NG + grp;
    const float w = __shfl(e, s);  // every lane takes part in the exchange
    if (s < a.nsplit) v += *reinterpret_cast<const f32x4*>(a.part + (s * total + i) * D + q * 4) * w;
  }
  part[grp][q] = v;
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int g = 1; g < NG; ++g) v += part[g][q];
  if (l == 0.f) v = f32x4{0.f, 0.f, 0.f, 0.f}, l = 1.f;  // a row that sees no key
  const int bh = (int)(i / rows), b = bh / a.Hk, kh = bh - b * a.Hk;
  const int rr = (int)(i - (int64_t)bh * rows), G = a.Hq / a.Hk;
  const int t = rr / G, h = kh * G + (rr - t * G);
  *reinterpret_cast<u32x2*>(a.y + (((int64_t)b * a.T + t) * a.Hq + h) * D + q * 4) =
      u32x2{pack_bf16x2(v[0] / l, v[1] / l), pack_bf16x2(v[2] / l, v[3] / l)};
}

// The attention kernel's shape for a call that may see `keys` keys.
struct Kv8Plan {
  bool rows;   // kv8_rows_kernel (else kv8_tiles_kernel)
  int rt;      // 16-row blocks per wave (rows)
  int n_rt;    // row groups (rows) or row tiles
  int nsplit;  // key ranges
};
constexpr int kKv8RowsMax = 64;   // query rows per kv head of kv8_rows_kernel
constexpr int kKv8Groups = 512;   // workgroups a call aims at (two per CU)

Kv8Plan kv8_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t keys) {
  Kv8Plan p;
  const int64_t rows = T * (Hq / Hk);
  p.rows = rows <= kKv8RowsMax;
  if (p.rows) {
    p.rt = rows <= 16 ? 1 : 2;
    p.n_rt = (int)((rows + 16 * p.rt - 1) / (16 * p.rt));
  } else {
    p.rt = 1;
    p.n_rt = (int)((rows + 63) / 64);
  }
  // no range shorter than two blocks for each wave, or eight tiles: one token at 333 keys
  // 7.5 us in one range against 10.8 and 3.8 to combine in two
  const int64_t groups = B * Hk * p.n_rt, most = (keys + 8 * kBlk - 1) / (8 * kBlk);
  int64_t ns = (p.rows && p.rt == 2 ? kKv8Groups / 2 : kKv8Groups) / groups;
  ns = ns < most ? ns : most;
  ns = ns < kKv8MaxSplit ? ns : kKv8MaxSplit;
  p.nsplit = (int)(ns < 1 ? 1 : ns);
  return p;
}

inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

template <int D>
int launch_write_d(const Kv8Args& a, bool with_q, hipStream_t s) {
  constexpr int RPP = 256 / (D / 8);
  int64_t groups = (int64_t)a.B * a.Hk * a.touch;
  if (with_q) groups += ((int64_t)a.B * a.T * a.Hq + RPP - 1) / RPP;
  hipLaunchKernelGGL(kv8_write_kernel<D>, dim3((unsigned)groups), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

template <int D>
int launch_kv8_d(Kv8Args a, int64_t keys, hipStream_t s) {
  int e = launch_write_d<D>(a, a.cos != nullptr, s);
  if (e) return e;
  const Kv8Plan p = kv8_plan(a.B, a.T, a.Hq, a.Hk, keys);
  const unsigned bh = (unsigned)(a.B * a.Hk);
  if (p.rows) {
    const dim3 grid((unsigned)p.nsplit, bh, (unsigned)p.n_rt);
    if (p.rt == 1) hipLaunchKernelGGL((kv8_rows_kernel<D, 1>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv8_rows_kernel<D, 2>), grid, dim3(256), 0, s, a);
  } else {
    const dim3 grid((unsigned)p.n_rt, bh, (unsigned)p.nsplit);
    hipLaunchKernelGGL(kv8_tiles_kernel<D>, grid, dim3(256), 0, s, a, p.n_rt);
  }
  e = (int)hipGetLastError();
  if (e || p.nsplit == 1) return e;
  hipLaunchKernelGGL(kv8_combine_kernel<D>, dim3((unsigned)((int64_t)a.B * a.T * a.Hq)), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

// Blocks that T new tokens can touch.
inline int touched(int64_t T) { return (int)((T + 2 * kBlk - 2) / kBlk); }

}  // namespace

int64_t kv8_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t keys, bool rope) {
  const Kv8Plan p = kv8_plan(B, T, Hq, Hk, keys);
  const int64_t rows = B * T * Hq;
  int64_t b = rope ? up256(rows * D * 2) : 0;
  if (p.nsplit > 1) b += up256(rows * p.nsplit * 8) + rows * p.nsplit * D * 4;
  return b;
}

int launch_kv8_attention(Kv8Args a, int64_t D, int64_t keys, void* ws, hipStream_t s) {
  const Kv8Plan p = kv8_plan(a.B, a.T, a.Hq, a.Hk, keys);
  const int64_t rows = (int64_t)a.B * a.T * a.Hq;
  char* w = (char*)ws;
  a.qn = (uint16_t*)w;  // q normalised and rotated
  if (a.cos) w += up256(rows * D * 2);
  a.stat = (float*)w;
  if (p.nsplit > 1) w += up256(rows * p.nsplit * 8);
  a.part = (float*)w;
  a.nsplit = p.nsplit;
  a.touch = touched(a.T);
  a.qsrc = a.cos ? a.qn : a.q;
  a.ldqs = a.cos ? (int64_t)a.Hq * D : a.ldq;
  return D == 128 ? launch_kv8_d<128>(a, keys, s) : launch_kv8_d<64>(a, keys, s);
}

int launch_kv8_write(Kv8Args a, int64_t D, hipStream_t s) {
  a.touch = touched(a.T);
  return D == 128 ? launch_write_d<128>(a, false, s) : launch_write_d<64>(a, false, s);
}

int launch_kv8_read(Kv8Args a, int64_t D, float* k, float* v, hipStream_t s) {
  const int rpp = D == 128 ? 16 : 32;
  const dim3 grid((unsigned)((int64_t)a.B * a.Hk * ((a.T + rpp - 1) / rpp)));
  if (D == 128) hipLaunchKernelGGL(kv8_read_kernel<128>, grid, dim3(256), 0, s, a, k, v);
  else hipLaunchKernelGGL(kv8_read_kernel<64>, grid, dim3(256), 0, s, a, k, v);
  return (int)hipGetLastError();
}

}  // namespace fp
