// fp_seg.hip — attention over a cache of two parts: a fixed part (the first F positions) and an
// own part (the positions from F on, all of them or the last W in a ring).
//
//   y_p = sum_j w_j v_j,  w = softmax_j(q_p . k_j / sqrt(D))  over
//         j < F, j <= p   and   F <= j <= p, p - W < j
//
// With one fixed part for the whole batch this is attention of sequences that continue one text
// (its keys are read once for all of them); with a fixed part of a few first tokens for each sequence and
// a ring it is attention with a sliding window and sinks.
//
//   - seg_rows_kernel (few rows per kv head) and seg_tiles_kernel (many): a work item is a group of
//     query rows of one kv head and a range of the key blocks that they see, fixed ones first. Rows are
//     one sequence's (tokens x heads of the group), or, for a shared fixed part alone, those
//     of all sequences. An item of all of its rows' keys writes the output, else partial sums.
//   - seg_prep_kernel, before seg_tiles_kernel: normalises and rotates q and k (or takes them as they are), writes
//     the new keys and values into the cache. (seg_rows_kernel's items do their own: a launch less.)
//   - seg_combine_kernel: sums the partials of a row in order.
//
// Products as in fp_attn.hip: S^T = K Q^T, so a row's scores lie in one lane column and are the B
// operand of O^T = V^T P^T as they come. Softmax in fp32 with the maximum followed in steps: p is taken
// about a reference that is raised (and the sums scaled) when a score passes it by 2^kLift. p enters the
// matrix core in two bf16 parts (off by 2^-17 of each, so that a row's error is its output's rounding), whatever
// the call's size. The sums of p come from the matrix core too, with a row of ones, so they are of p as it enters.
//
// An entry that a row does not see has no part in it, whatever it holds. An infinity or a NaN among
// the values would (0 inf): the sums show it, and then the item is done again with such entries taken
// out of the products and counted for the rows that see them, which become NaN.
#include "fp_common.h"
#include "fp_launch.h"
#include "fp_rope.h"

#include <type_traits>

namespace fp {

namespace {

// f(0), f(1), .. f(N - 1) with constants, so that what they index stays in registers.
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<N, I + 1>(f);
  }
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLift = 6.f;
constexpr int kParts = 2;       // bf16 parts of p
constexpr int kMaxPlanes = 64;  // one lane per plane in seg_combine_kernel

constexpr int vmcnt_imm(int v) { return (v & 15) | (7 << 4) | (15 << 8) | ((v >> 4) << 14); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, int bytes) {
  constexpr int kRsrcFlags = 0x00020000;  // raw buffer, 32-bit data format
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, kRsrcFlags);
}
// 16 bytes per lane from the buffer at voff into LDS at dst + 16 * lane; past its end zeros.
__device__ __forceinline__ void load_lds16(const void* base, int nbytes, lds_ptr_t dst, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(base, nbytes), dst, 16, voff, 0, 0, 0);
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Position of sequence b's first token (one far outside any cache stays outside, in 32 bits).
__device__ __forceinline__ int first_pos(const SegArgs& a, int b) {
  constexpr int64_t kFar = 1 << 30;
  const int64_t p = a.pos_dev ? a.pos_dev[b * a.pos_stride] : a.pos;
  return (int)(p < -kFar ? -kFar : p > kFar ? kFar : p);
}
__device__ __forceinline__ int count(const SegArgs& a, int b) {
  if (!a.lengths) return a.T;
  const int64_t n = a.lengths[b];
  return (int)(n < 0 ? 0 : n > a.T ? a.T : n);
}
// Whether position p is one that the cache takes.
__device__ __forceinline__ bool in_cache(const SegArgs& a, int p) {
  return a.ring ? p >= 0 && p < (1 << 30) : p >= a.F && p - a.F < a.S;
}

// ---- new tokens -------------------------------------------------------------------

// A new token's key or value of one head to its place, by LPH = D / 8 lanes (lane j; fp_rope.h).
template <int D>
__device__ __forceinline__ void put_new(const SegArgs& a, int b, int kh, int t, int p, bool value, int j) {
  const uint16_t* src = value ? a.v + b * a.svb + t * a.svt + (int64_t)kh * D : a.k + b * a.skb + t * a.skt + (int64_t)kh * D;
  u32x2 lo = *reinterpret_cast<const u32x2*>(src + 4 * j);
  u32x2 hi = *reinterpret_cast<const u32x2*>(src + D / 2 + 4 * j);
  if (a.cos && !value)
    norm_rope_row<D>(lo, hi, a.gk, a.epsk, a.cos + b * a.scb + t * a.sct, a.sin + b * a.ssb + t * a.sst, j);
  const int u = p - a.F;
  uint16_t* dst;
  if (u < 0) dst = (value ? a.fv : a.fk) + b * a.sfb + kh * a.sfh + (int64_t)p * a.sfs;
  else dst = (value ? a.ov : a.ok) + b * a.sob + kh * a.soh + (int64_t)(a.ring ? u % a.S : u) * a.sos;
  *reinterpret_cast<u32x2*>(dst + 4 * j) = lo;
  *reinterpret_cast<u32x2*>(dst + D / 2 + 4 * j) = hi;
}

// Every new token's, and with queries the rotated q. (Lanes past the last row leave together with the others of
// their row.)
template <int D>
__global__ __launch_bounds__(256) void seg_prep_kernel(SegArgs a) {
  constexpr int LPH = D / 8;
  const int qh = a.qn ? a.Hq : 0, heads = qh + 2 * a.Hk;
  const int64_t item = (int64_t)blockIdx.x * (256 / LPH) + threadIdx.x / LPH;
  if (item >= (int64_t)a.B * a.T * heads) return;
  const int j = threadIdx.x % LPH;
  const int64_t m = item / heads;
  const int h = (int)(item - m * heads), b = (int)(m / a.T), t = (int)(m - (int64_t)b * a.T);
  if (h >= qh) {
    const int p = first_pos(a, b) + t, hk = h - qh;
    if (t < count(a, b) && in_cache(a, p)) put_new<D>(a, b, hk < a.Hk ? hk : hk - a.Hk, t, p, hk >= a.Hk, j);
    return;
  }
  const uint16_t* src = a.q + b * a.sqb + t * a.sqt + (int64_t)h * D;
  uint16_t* dst = a.qn + (m * a.Hq + h) * D;
  u32x2 lo = *reinterpret_cast<const u32x2*>(src + 4 * j);
  u32x2 hi = *reinterpret_cast<const u32x2*>(src + D / 2 + 4 * j);
  norm_rope_row<D>(lo, hi, a.gq, a.epsq, a.cos + b * a.scb + t * a.sct, a.sin + b * a.ssb + t * a.sst, j);
  *reinterpret_cast<u32x2*>(dst + 4 * j) = lo;
  *reinterpret_cast<u32x2*>(dst + D / 2 + 4 * j) = hi;
}

// ---- shared pieces of the two attention kernels ---------------------------------------

// Whether any of the eight bf16 is an infinity or a NaN.
__device__ __forceinline__ bool nonfinite8(u32x4 v) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= ((v[i] & 0x7fff7fffu) + 0x00800080u);
  return (any & 0x80008000u) != 0;
}
// v with those entries zero, and bad with a one in their places and zeros elsewhere.
__device__ __forceinline__ void take_nonfinite8(u32x4& v, u32x4& bad) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t at = (((v[i] & 0x7fff7fffu) + 0x00800080u) & 0x80008000u) >> 15;  // 1 in each half
    v[i] &= ~(at * 0xffffu);
    bad[i] = at * 0x3f80u;  // bf16 1
  }
}

// Where 16-byte chunk c of key (value) row r lies in the row's D * 2 bytes of LDS: at c ^ swk (swv). Half a
// wave's lanes of one read then meet every bank once: 16 rows of a chunk of the keys, 8 rows of a pair of
// chunks of the values. (With c ^ r for both, two rows of each pair met: half of the LDS cycles were conflicts.)
template <int D>
__device__ __forceinline__ int swk(int r) {
  return D == 128 ? r & 15 : (r >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int swv(int r) {
  return D == 128 ? (r & 7) * 2 : ((r >> 1) & 3) * 2;
}

// A operand of V^T for d block dt and keys {4g .. 4g+3, 16 + 4g ..} of 32 V rows in LDS.
template <int D>
__device__ __forceinline__ u32x4 read_vt(const char* rows, int dt, int li, int grp) {
  const int key = 4 * grp + (li >> 2), c = 2 * dt + ((li & 3) >> 1), half = (li & 1) * 8;
  u32x4 out;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int r = key + 16 * s;
    const char* p = rows + r * (D * 2) + ((c ^ swv<D>(r)) * 16) + half;
    const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)p));
    out[2 * s] = w.x;
    out[2 * s + 1] = w.y;
  }
  return out;
}

// max over the four lane groups that share a row column
__device__ __forceinline__ float col_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

// Eight probabilities (keys 4g .. 4g+3 and 16 + 4g ..) as PARTS bf16 B operands.
template <int PARTS>
__device__ __forceinline__ void split_p(const f32x4& p0, const f32x4& p1, u32x4 (&f)[PARTS]) {
  const float p[8] = {p0[0], p0[1], p0[2], p0[3], p1[0], p1[1], p1[2], p1[3]};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = p[2 * i], y = p[2 * i + 1];
#pragma unroll
    for (int c = 0; c < PARTS; ++c) {
      const uint32_t h = cvt_bf16x2(x, y);
      f[c][i] = h;
      if (c + 1 < PARTS) {
        x -= __uint_as_float(h << 16);  // exact
        y -= __uint_as_float(h & 0xffff0000u);
      }
    }
  }
}

// One query row: which of its kv head's rows it is, and the keys it sees of each part (none: hi < lo).
struct RowKeys {
  int hi_f, lo_o, hi_o;
};
__device__ __forceinline__ RowKeys row_keys(const SegArgs& a, int p) {
  RowKeys r;
  const int u = p - a.F;
  r.hi_f = p < a.F ? p : a.F - 1;
  r.lo_o = a.W > 0 && u - a.W + 1 > 0 ? u - a.W + 1 : 0;
  r.hi_o = a.ring || u < a.S ? u : a.S - 1;
  return r;
}

// A work item: rows row0 .. of kv head kh, of sequence b or (packed) of all, and key blocks
// lo .. hi - 1 of: nf blocks of the fixed part, then the own part's from c0 on.
struct Item {
  int b, kh, row0, rows;  // rows: of the kv head in all
  int nf, c0, lo, hi;
  int ring, at;           // blocks of the ring (or more than there are), and the place of block c0 in it
  int plane;              // of the partial sums
  bool packed;
};
// The position of the token of row r.
__device__ __forceinline__ int row_pos(const SegArgs& a, const Item& it, int r, int p0) {
  return p0 + (it.packed ? 0 : r / (a.Hq / a.Hk));
}

// Blocks of KB keys for rows row0 .. row0 + n - 1, cut into nsplit ranges, of which this is the s-th.
template <int KB>
__device__ __forceinline__ void item_keys(const SegArgs& a, Item& it, int n, bool fixed, bool own, int s, int nsplit) {
  int total = 0;
  it.nf = it.c0 = 0;
  if (it.packed) {
    it.nf = (a.F + KB - 1) / KB;
    total = it.nf;
  } else {
    const int G = a.Hq / a.Hk, p0 = first_pos(a, it.b);
    int last = it.row0 + n - 1;
    if (last >= it.rows) last = it.rows - 1;
    // (rows past the sequence's tokens need no keys)
    const int live = count(a, it.b) * G - 1;
    if (last > live) last = live;
    if (last >= it.row0) {
      const RowKeys f = row_keys(a, p0 + it.row0 / G), l = row_keys(a, p0 + last / G);
      if (fixed && l.hi_f >= 0) it.nf = l.hi_f / KB + 1;
      total = it.nf;
      if (own && l.hi_o >= f.lo_o) {
        it.c0 = f.lo_o / KB;
        total += l.hi_o / KB + 1 - it.c0;
      }
    }
  }
  it.ring = a.ring ? a.S / KB : 1 << 30;
  it.at = it.c0 % it.ring;
  const int per = (total + nsplit - 1) / nsplit;
  it.lo = s * per;
  it.hi = it.lo + per < total ? it.lo + per : total;
}

// Where block c lies in its part. (An item's own blocks span the ring at most, and one more.)
__device__ __forceinline__ int place(const Item& it, int c) {
  if (c < it.nf) return c;
  const int x = it.at + c - it.nf;
  return x < it.ring ? x : x - it.ring;
}

// The block of an item's own sequence that position p is in (-1: before those that it has).
template <int KB>
__device__ __forceinline__ int new_block(const SegArgs& a, const Item& it, int p) {
  const int u = p - a.F;
  if (u < 0) return p < 0 || it.nf == 0 ? -1 : p / KB;
  return u / KB < it.c0 ? -1 : it.nf + u / KB - it.c0;
}

// q row r of an item (clamped; rows past the last are not stored).
__device__ __forceinline__ const uint16_t* q_row(const SegArgs& a, const Item& it, int r, int D) {
  if (r >= it.rows) r = it.rows - 1;
  const int G = a.Hq / a.Hk, n = r / G, h = it.kh * G + (r - n * G);
  const int b = it.packed ? n / a.T : it.b, t = it.packed ? n - b * a.T : n;
  return a.qsrc + b * a.sqsb + t * a.sqst + (int64_t)h * D;
}

// Where a row's partial sums lie.
__device__ __forceinline__ int64_t part_row(const SegArgs& a, const Item& it, int r) {
  const int G = a.Hq / a.Hk;
  return ((int64_t)it.plane * a.Hk + it.kh) * ((int64_t)a.B * a.T * G) + (it.packed ? 0 : (int64_t)it.b * a.T * G) + r;
}

// Whether row r (of one sequence) is of a token that there is, in the cache.
__device__ __forceinline__ bool row_live(const SegArgs& a, const Item& it, int r) {
  const int t = r / (a.Hq / a.Hk);
  return t < count(a, it.b) && in_cache(a, first_pos(a, it.b) + t);
}
// The output of a row that has all of its keys: four elements from d on.
__device__ __forceinline__ void store_row(const SegArgs& a, const Item& it, int r, int d, int D, f32x4 v, float l,
                                          bool live) {
  const int G = a.Hq / a.Hk, t = r / G, h = it.kh * G + (r - t * G);
  const float s = 1.f / l;
  u32x2 o = {0u, 0u};
  if (live) o = u32x2{pack_bf16x2(v[0] * s, v[1] * s), pack_bf16x2(v[2] * s, v[3] * s)};
  *reinterpret_cast<u32x2*>(a.y + it.b * a.syb + (int64_t)t * a.Hq * D + (int64_t)h * D + d) = o;
}

// The softmax state of RT row blocks in a wave: accumulators of O^T, sums of p, references.
template <int D, int RT>
struct State {
  f32x4 o[D / 16][RT];
  f32x4 sum[RT];
  float mx[RT];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      mx[rt] = -INFINITY;
      sum[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) o[dt][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  // Raises the references where the scores s (NB blocks of 16 keys) pass them.
  template <int NB>
  __device__ __forceinline__ void follow(const f32x4 (&s)[RT][NB], float sc) {
    float m[RT];
    bool up = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -INFINITY;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) m[rt] = fmaxf(m[rt], s[rt][n][r]);
      up |= m[rt] * sc > mx[rt] + kLift;
    }
    if (__any(up)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float mn = fmaxf(mx[rt], col_max(m[rt]) * sc);
        // The factor in two halves: the sums may be up to 2^127 about the old reference, so one below 2^-126,
        // which v_exp_f32 gives as 0, can still leave them a part of the row.
        const float al = mn == -INFINITY ? 1.f : exp2_fast(0.5f * (mx[rt] - mn));
        mx[rt] = mn;
        sum[rt] = sum[rt] * al * al;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[dt][rt] = o[dt][rt] * al * al;
      }
    }
  }
  // Whether an infinity or a NaN is in any sum.
  __device__ __forceinline__ bool nonfinite() const {
    float t = 0.f;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) t = fmaf(sum[rt][0], 0.f, t);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) t = fmaf(o[dt][rt][r], 0.f, t);  // 0 inf: NaN
    return t != t;
  }
};

__device__ __forceinline__ u32x4 ones8() { return u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}; }

// ---- few rows ------------------------------------------------------------------------
//
// Bound by the cache's bytes. 16 query rows; the four waves take 32-key blocks w, w + 4, ... of the
// item's range, each with the next block's keys in registers and values in its own LDS buffer while it
// computes; their states are merged through LDS in wave order.
// Items: first those of the shared fixed part (grid: n_split1 ranges x row groups x kv heads), then of each
// sequence (ranges x row groups x kv heads x sequences). An item normalises and rotates its queries (into LDS)
// and its new keys itself (into the cache: those in its range, which a token's own row always sees, so
// every one is in some item's; two items of one write the same).
template <int D>
__global__ __launch_bounds__(256, 2) void seg_rows_kernel(SegArgs a, SegPlan pl) {
  constexpr int NW = 4, KB = 32, PARTS = kParts;
  constexpr int DK = D / 32, DT = D / 16;      // k-steps of q.k, d blocks of p.V
  constexpr int RPI = 1024 / (D * 2);          // V rows per load instruction
  constexpr int NV = KB / RPI, NK = 2 * DK;    // V and K load instructions per block
  constexpr int CH = D / 8;                    // 16-byte chunks per row
  __shared__ __attribute__((aligned(1024))) char sV0[NW][KB * D * 2];
  __shared__ __attribute__((aligned(1024))) char sV1[NW][KB * D * 2];
  __shared__ __attribute__((aligned(1024))) char sQ[16 * D * 2];
  __shared__ float sM[NW][16], sL[NW][16];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int li = lane & 15, grp = lane >> 4;
  const int G = a.Hq / a.Hk;
  Item it;
  int id = blockIdx.x;
  it.packed = id < pl.items1;
  if (!it.packed) id -= pl.items1;
  it.kh = id % a.Hk;
  id /= a.Hk;
  if (it.packed) {
    it.b = 0;
    it.rows = a.B * a.T * G;
    const int n = (it.rows + 15) / 16;
    it.row0 = id % n * 16;
    it.plane = id / n;
    item_keys<KB>(a, it, 16, true, false, it.plane, pl.split1);
  } else {
    it.b = id % a.B;
    id /= a.B;
    it.rows = a.T * G;
    const int n = (it.rows + 15) / 16;
    it.row0 = id % n * 16;
    it.plane = pl.split1 + id / n;
    item_keys<KB>(a, it, 16, !pl.shared, true, id / n, pl.split2);
  }

  const int p0 = it.packed ? a.F : first_pos(a, it.b), r0 = it.row0 + li;
  const RowKeys rk = row_keys(a, row_pos(a, it, r0 < it.rows ? r0 : it.rows - 1, p0));

  const uint16_t* const kb[2] = {a.fk + it.b * a.sfb + it.kh * a.sfh, a.ok + it.b * a.sob + it.kh * a.soh};
  const uint16_t* const vb[2] = {a.fv + it.b * a.sfb + it.kh * a.sfh, a.ov + it.b * a.sob + it.kh * a.soh};
  const int bytes[2] = {a.F > 0 ? (int)(((int64_t)(a.F - 1) * a.sfs + D) * 2) : 0,
                        (int)(((int64_t)(a.S - 1) * a.sos + D) * 2)};
  const uint32_t step[2] = {(uint32_t)(a.sfs * 2), (uint32_t)(a.sos * 2)};
  const int vr = lane / CH;
  auto issue = [&](u32x4 (&kf)[2][DK], char* sv, int c) {
    const int own = c < it.nf ? 0 : 1;
    const int blk = place(it, c);
    const uint32_t st = step[own];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int r = n * RPI + vr;
      load_lds16(vb[own], bytes[own], (lds_ptr_t)(sv + n * 1024),
                 (uint32_t)(blk * KB + r) * st + (uint32_t)(((lane % CH) ^ swv<D>(r)) * 16));
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < DK; ++i)
        kf[kt][i] = __builtin_amdgcn_raw_buffer_load_b128(make_rsrc(kb[own], bytes[own]),
                                                          (uint32_t)(blk * KB + 16 * kt + li) * st + 16 * grp + 64 * i, 0, 0);
  };

  // new keys are in the range (uniform; conservative: from the first token's block to the last's)
  const int n_new = it.packed ? 0 : count(a, it.b);
  const bool fresh = n_new > 0 && it.lo < it.hi && new_block<KB>(a, it, p0) < it.hi &&
                     new_block<KB>(a, it, p0 + n_new - 1) >= it.lo;
  constexpr int LPH = D / 8;
  const int hr = threadIdx.x / LPH, hj = threadIdx.x % LPH;
  for (int r = hr; r < 16; r += 256 / LPH) {
    const int rc = it.row0 + r < it.rows ? it.row0 + r : it.rows - 1, n = rc / G;
    const int b = it.packed ? n / a.T : it.b, t = it.packed ? n - b * a.T : n;
    const uint16_t* src = a.q + b * a.sqb + t * a.sqt + (int64_t)(it.kh * G + rc - n * G) * D;
    u32x2 lo = *reinterpret_cast<const u32x2*>(src + 4 * hj);
    u32x2 hi = *reinterpret_cast<const u32x2*>(src + D / 2 + 4 * hj);
    if (a.cos)
      norm_rope_row<D>(lo, hi, a.gq, a.epsq, a.cos + b * a.scb + t * a.sct, a.sin + b * a.ssb + t * a.sst, hj);
    char* const dst = sQ + r * (D * 2) + (hj & 1) * 8;
    *reinterpret_cast<u32x2*>(dst + (((hj >> 1) ^ swk<D>(r)) * 16)) = lo;
    *reinterpret_cast<u32x2*>(dst + (((D / 16 + (hj >> 1)) ^ swk<D>(r)) * 16)) = hi;
  }
  if (fresh) {
    for (int i = hr; i < 2 * n_new; i += 256 / LPH) {
      const int t = i >> 1, c = new_block<KB>(a, it, p0 + t);
      if (!in_cache(a, p0 + t) || c < it.lo || c >= it.hi) continue;
      put_new<D>(a, it.b, it.kh, t, p0 + t, (i & 1) != 0, hj);
    }
  }
  __syncthreads();  // (the keys: read by this workgroup after their writes)
  u32x4 qf[DK];
#pragma unroll
  for (int i = 0; i < DK; ++i)
    qf[i] = *reinterpret_cast<const u32x4*>(sQ + li * (D * 2) + (((4 * i + grp) ^ swk<D>(li)) * 16));

  const float sc = kLog2e / sqrtf((float)D);
  State<D, 1> S;
  auto compute = [&](u32x4 (&kf)[2][DK], const char* sv, int c, bool careful) {
    const int own = c < it.nf ? 0 : 1;
    const int first = own ? (it.c0 + c - it.nf) * KB : c * KB;
    const int lo = own ? rk.lo_o : 0, hi = own ? rk.hi_o : rk.hi_f;
    f32x4 s[1][2], one[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[0][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DK; ++i) s[0][kt] = mfma16(kf[kt][i], qf[i], s[0][kt]);
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = first + kt * 16 + 4 * grp + r;
        const bool hidden = i < lo || i > hi;
        if (hidden) s[0][kt][r] = -INFINITY;
        one[kt][r] = hidden ? 0.f : 1.f;
      }
    u32x4 pf[PARTS], seen[1];
    if (careful) split_p<1>(one[0], one[1], seen);
    S.follow(s, sc);
    const float base = S.mx[0] == -INFINITY ? 0.f : S.mx[0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[0][kt][r] = exp2_fast(fmaf(s[0][kt][r], sc, -base));
    split_p<PARTS>(s[0][0], s[0][1], pf);
#pragma unroll
    for (int c2 = 0; c2 < PARTS; ++c2) S.sum[0] = mfma16(ones8(), pf[c2], S.sum[0]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      u32x4 vt = read_vt<D>(sv, dt, li, grp);
      if (careful) {
        u32x4 bad;
        take_nonfinite8(vt, bad);
        const f32x4 n = mfma16(bad, seen[0], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n[r] > 0.f) S.o[dt][0][r] = __uint_as_float(0x7fc00000u);
      }
#pragma unroll
      for (int c2 = 0; c2 < PARTS; ++c2) S.o[dt][0] = mfma16(vt, pf[c2], S.o[dt][0]);
    }
  };

  // block it.lo + wave + 4 i of this wave, the next one's loads in flight
  auto pass = [&](bool careful) {
    S.clear();
    u32x4 k0[2][DK], k1[2][DK];
    int c = it.lo + wave;
    if (c < it.hi) issue(k0, sV0[wave], c);
    while (c < it.hi) {
      if (c + NW < it.hi) {
        issue(k1, sV1[wave], c + NW);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(NK + NV));
      } else {
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      }
      compute(k0, sV0[wave], c, careful);
      c += NW;
      if (c >= it.hi) break;
      if (c + NW < it.hi) {
        issue(k0, sV0[wave], c + NW);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(NK + NV));
      } else {
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      }
      compute(k1, sV1[wave], c, careful);
      c += NW;
    }
  };
  pass(false);
  if (__any(S.nonfinite())) pass(true);

  // Merge the waves' states in wave order. A wave's row sums go over its own first V buffer (free now), 16-byte
  // chunk q of row r at q ^ r, so 16 rows' stores spread over the banks.
  static_assert(16 * D * 4 == KB * D * 2, "the sums fit the V buffer");
  auto slot = [&](int w, int r, int q) -> f32x4* {
    return reinterpret_cast<f32x4*>(sV0[w] + r * (D * 4) + ((q ^ r) * 16));
  };
  if (grp == 0) {
    sM[wave][li] = S.mx[0];
    sL[wave][li] = S.sum[0][0];
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) *slot(wave, li, dt * 4 + grp) = S.o[dt][0];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * (D / 4); i += NW * kWave) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4, rr = it.row0 + r;
    if (rr >= it.rows) continue;
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
      v += *slot(w, r, d / 4) * e;
    }
    if (pl.planes > 1) {
      const int64_t pr = part_row(a, it, rr);
      *reinterpret_cast<f32x4*>(a.part + pr * D + d) = v;
      if (d == 0) *reinterpret_cast<f32x2*>(a.stat + pr * 2) = f32x2{m, l};
    } else {
      store_row(a, it, rr, d, D, v, l, row_live(a, it, rr));
    }
  }
}

// ---- many rows -----------------------------------------------------------------------
//
// Four waves of 16 RT query rows each share 64-key tiles of keys and values in LDS, the next tile's
// loads in flight while one is computed.
// Items: ranges x row tiles (of one sequence, or of all where only a shared fixed part is read) with the kv
// head fastest, so that one XCD runs a head's tiles.
template <int D, int RT>
__global__ __launch_bounds__(256, RT > 2 ? 1 : 2) void seg_tiles_kernel(SegArgs a, SegPlan pl) {
  constexpr int NW = 4, KB = 64, PARTS = kParts;
  constexpr int DK = D / 32, DT = D / 16;
  constexpr int RPI = 1024 / (D * 2);          // rows per load instruction
  constexpr int NL = KB / RPI / NW;            // load instructions per wave of a tile's keys
  constexpr int CH = D / 8;
  __shared__ __attribute__((aligned(1024))) char sK0[KB * D * 2];
  __shared__ __attribute__((aligned(1024))) char sK1[KB * D * 2];
  __shared__ __attribute__((aligned(1024))) char sV0[KB * D * 2];
  __shared__ __attribute__((aligned(1024))) char sV1[KB * D * 2];
  __shared__ int sBad[NW];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int li = lane & 15, grp = lane >> 4;
  const int G = a.Hq / a.Hk;
  Item it;
  it.kh = blockIdx.x % a.Hk;
  const int64_t g = blockIdx.x / a.Hk, n1 = pl.items1 / a.Hk, n = n1 + pl.items2 / a.Hk;
  int id = (int)(g * n1 / n);
  it.packed = (g + 1) * n1 / n > id;
  it.b = 0;
  if (!it.packed) {
    id = (int)g - id;
    it.b = id % a.B;
    id /= a.B;
  }
  it.rows = (it.packed ? a.B : 1) * a.T * G;
  constexpr int ROWS = NW * 16 * RT;
  const int n_rt = (it.rows + ROWS - 1) / ROWS;
  int rtile, range;
  if (it.packed) {
    // (ranges fastest: the workgroups of a CU are then of several row tiles, and a last one with few rows
    // leaves the matrix cores to the others; 160 rows of 50001 keys: 61 -> 57 us)
    range = it.plane = id % pl.split1;
    rtile = id / pl.split1;
  } else {
    rtile = n_rt - 1 - id % n_rt;  // the later tokens of a prompt see more
    range = id / n_rt;
    it.plane = pl.split1 + range;
  }
  it.row0 = rtile * ROWS;
  item_keys<KB>(a, it, ROWS, it.packed || !pl.shared, !it.packed, range, it.packed ? pl.split1 : pl.split2);
  const int row0 = it.row0 + wave * 16 * RT;  // this wave's first row
  // A wave without a row of a token loads its share of the tiles only.
  const bool idle = row0 >= (it.packed ? it.rows : count(a, it.b) * G);

  u32x4 qf[RT][DK];
  RowKeys rk[RT];
  const int p0 = it.packed ? a.F : first_pos(a, it.b);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + li;
    rk[rt] = row_keys(a, row_pos(a, it, r < it.rows ? r : it.rows - 1, p0));
    const uint16_t* qp = q_row(a, it, r, D) + 8 * grp;
#pragma unroll
    for (int i = 0; i < DK; ++i) qf[rt][i] = ld16(qp + 32 * i);
  }
  // of the wave's first and last row (uniform)
  const RowKeys first = row_keys(a, row_pos(a, it, row0 < it.rows ? row0 : it.rows - 1, p0));
  const int row1 = row0 + 16 * RT - 1;
  const RowKeys last = row_keys(a, row_pos(a, it, row1 < it.rows ? row1 : it.rows - 1, p0));

  const uint16_t *const fk = a.fk + it.b * a.sfb + it.kh * a.sfh, *const ok = a.ok + it.b * a.sob + it.kh * a.soh;
  const uint16_t *const fv = a.fv + it.b * a.sfb + it.kh * a.sfh, *const ov = a.ov + it.b * a.sob + it.kh * a.soh;
  const int bytes[2] = {a.F > 0 ? (int)(((int64_t)(a.F - 1) * a.sfs + D) * 2) : 0,
                        (int)(((int64_t)(a.S - 1) * a.sos + D) * 2)};
  const uint32_t step[2] = {(uint32_t)(a.sfs * 2), (uint32_t)(a.sos * 2)};
  // this lane's row of a tile's first load instruction, and its chunks of keys and of values in each
  const uint32_t row = (uint32_t)(wave * NL * RPI + lane / CH);
  uint32_t chk[NL], chv[NL];
#pragma unroll
  for (int n = 0; n < NL; ++n) {
    const int r = (int)row + n * RPI;
    chk[n] = (uint32_t)(((lane % CH) ^ swk<D>(r)) * 16);
    chv[n] = (uint32_t)(((lane % CH) ^ swv<D>(r)) * 16);
  }
  // each tile's rows through a buffer that starts at the tile and ends with the part's last row, so
  // that the lane offset alone tells whether a row is past it
  struct Tile {
    const char* p;
    int bytes;
    uint32_t step;  // a row's bytes
  };
  auto tile_of = [&](const uint16_t* fix, const uint16_t* own, int c) __attribute__((always_inline)) -> Tile {
    const bool o = c >= it.nf;
    const uint32_t st = o ? step[1] : step[0];
    const int skip = (int)((uint32_t)(place(it, c) * KB) * st);
    return {(const char*)(o ? own : fix) + skip, c < it.hi ? (o ? bytes[1] : bytes[0]) - skip : 0, st};  // past the item's: nothing
  };
  auto issue = [&](const Tile& t, char* dst, int n, uint32_t ch) __attribute__((always_inline)) {
    load_lds16(t.p, t.bytes, (lds_ptr_t)(dst + (wave * NL + n) * 1024), row * t.step + (uint32_t)(n * RPI) * t.step + ch);
  };

  const float sc = kLog2e / sqrtf((float)D);
  State<D, RT> S;
  bool ready = false;
  // A bare barrier (__syncthreads' fence would wait for every load in flight); what was read from LDS before
  // it has been used.
  auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // The operands of 16 keys (block n of a tile), and of the values for four d blocks of 32 keys: each lot
  // is read from LDS while the products of the one before run.
  auto read_k = [&](u32x4 (&f)[DK], const char* sk, int n) __attribute__((always_inline)) {
    const int r = n * 16 + li;
#pragma unroll
    for (int i = 0; i < DK; ++i)
      f[i] = *reinterpret_cast<const u32x4*>(sk + r * (D * 2) + (((4 * i + grp) ^ swk<D>(r)) * 16));
  };
  constexpr int VB = DT / 4;  // lots of a half tile's values
  auto read_v = [&](u32x4 (&f)[4], const char* sv, int b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = read_vt<D>(sv + b / VB * 32 * D * 2, b % VB * 4 + i, li, grp);
  };
  // Tile c of keys sk and values sv. Loads go out one at a time between the products (in one burst they
  // would hold the wave's other instructions back): the next values (into nv) with the scores, as the values
  // before these are done with then, and the keys after the next (into sk) with the values' products. So each
  // has more than a tile's time to land in two stages; every step issues the same loads (past the item's
  // end of nothing), so that the count in flight is known.
  auto tile = [&](char* sk, const char* sv, char* nv, int c, bool careful) __attribute__((always_inline)) {
    // these keys have landed (behind them: the values, the next keys), and every wave is done with the
    // values before these
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * NL));
    barrier();
    const Tile tk = tile_of(fk, ok, c + 2), tv = tile_of(fv, ov, c + 1);
    f32x4 s[RT][4];
    u32x4 kf[2][DK];
    read_k(kf[0], sk, 0);
    each<4>([&](auto N) __attribute__((always_inline)) {
      constexpr int n = decltype(N)::value;
      if constexpr (n < 3) read_k(kf[(n + 1) & 1], sk, n + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DK; ++i)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][n] = mfma16(kf[n & 1][i], qf[rt][i], s[rt][n]);
#pragma unroll
      for (int i = n * NL / 4; i < (n + 1) * NL / 4; ++i) {
        issue(tv, nv, i, chv[i]);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    const int own = c < it.nf ? 0 : 1;
    const int at = own ? (it.c0 + c - it.nf) * KB : c * KB;
    // whether a row of this wave does not see some key (uniform)
    const bool mask = at + KB - 1 > (own ? first.hi_o : first.hi_f) || (own && at < last.lo_o);
    u32x4 seen[RT][2], pf[RT][2][PARTS];
    const auto softmax = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float base = S.mx[rt] == -INFINITY ? 0.f : S.mx[rt];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) s[rt][n][r] = exp2_fast(fmaf(s[rt][n][r], sc, -base));
          if (n & 1) split_p<PARTS>(s[rt][n - 1], s[rt][n], pf[rt][n / 2]);
        }
      }
    };
    // A row's reference comes from the first tiles that it sees keys of. After one that all of the wave's rows
    // see whole, and that has given each a reference, only the careful pass follows it: exponents then may reach
    // 2^127 (floating point, so p is no less exact for that), and past it the sums are infinite and the item is
    // done again.
    // (The two ways have their own softmax, and the empty statement keeps them apart: where they meet before it
    // the scores are moved twice, 64 instructions a tile.)
    if (careful || mask || !ready) {
      if (mask || careful) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const int lo = own ? rk[rt].lo_o : 0, hi = own ? rk[rt].hi_o : rk[rt].hi_f;
          f32x4 one[4];
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int i = at + n * 16 + 4 * grp + r;
              const bool hidden = i < lo || i > hi;
              if (hidden) s[rt][n][r] = -INFINITY;
              one[n][r] = hidden ? 0.f : 1.f;
            }
          if (careful)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              u32x4 f[1];
              split_p<1>(one[2 * n], one[2 * n + 1], f);
              seen[rt][n] = f[0];
            }
        }
      }
      S.follow(s, sc);
      if (!mask) {  // (scores of the negative infinity alone give no reference)
        bool all = true;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) all &= S.mx[rt] > -INFINITY;
        ready = __all(all);
      }
      softmax();
    } else {
      softmax();
      asm volatile("");
    }
    // these values have landed (behind them: the next keys and values), and every wave is done with the keys
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * NL));
    barrier();
    u32x4 vf[2][4];
    read_v(vf[0], sv, 0);
    __builtin_amdgcn_sched_barrier(0);
    each<2 * VB>([&](auto B) __attribute__((always_inline)) {
      constexpr int b = decltype(B)::value, n = b / VB;
      if constexpr (b + 1 < 2 * VB) read_v(vf[(b + 1) & 1], sv, b + 1);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (b % VB == 0) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int c2 = 0; c2 < PARTS; ++c2) S.sum[rt] = mfma16(ones8(), pf[rt][n][c2], S.sum[rt]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int dt = b % VB * 4 + i;
        u32x4 vt = vf[b & 1][i];
        if (careful) {
          u32x4 bad;
          take_nonfinite8(vt, bad);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const f32x4 k = mfma16(bad, seen[rt][n], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (k[r] > 0.f) S.o[dt][rt][r] = __uint_as_float(0x7fc00000u);
          }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int c2 = 0; c2 < PARTS; ++c2) S.o[dt][rt] = mfma16(vt, pf[rt][n][c2], S.o[dt][rt]);
      }
#pragma unroll
      for (int i = b * NL / (2 * VB); i < (b + 1) * NL / (2 * VB); ++i) issue(tk, sk, i, chk[i]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // (The compiler waits for every load at the top of a loop with some in flight: so four tiles a round.)
  auto pass = [&](auto CAREFUL) __attribute__((always_inline)) {
    constexpr bool careful = decltype(CAREFUL)::value;
    constexpr int U = careful ? 2 : 4;
    S.clear();
    ready = false;
    if (it.lo >= it.hi) return;
    const Tile k0 = tile_of(fk, ok, it.lo), v0 = tile_of(fv, ov, it.lo), k1 = tile_of(fk, ok, it.lo + 1);
#pragma unroll
    for (int n = 0; n < NL; ++n) issue(k0, sK0, n, chk[n]);
#pragma unroll
    for (int n = 0; n < NL; ++n) issue(v0, sV0, n, chv[n]);
#pragma unroll
    for (int n = 0; n < NL; ++n) issue(k1, sK1, n, chk[n]);
    if (idle) {
      for (int c = it.lo; c < it.hi; ++c) {
        const bool odd = (c - it.lo) & 1;
        const Tile tk = tile_of(fk, ok, c + 2), tv = tile_of(fv, ov, c + 1);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * NL));
        barrier();
#pragma unroll
        for (int n = 0; n < NL; ++n) issue(tv, odd ? sV0 : sV1, n, chv[n]);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * NL));
        barrier();
#pragma unroll
        for (int n = 0; n < NL; ++n) issue(tk, odd ? sK1 : sK0, n, chk[n]);
      }
    } else for (int c = it.lo; c < it.hi; c += U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = c + u;
        if (k >= it.hi) break;
        if (u & 1) tile(sK1, sV1, sV0, k, careful);
        else tile(sK0, sV0, sV1, k, careful);
      }
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __syncthreads();  // (a second pass writes the first stages)
  };
  pass(std::false_type{});
  const int any = __any(S.nonfinite()) ? 1 : 0;
  if (lane == 0) sBad[wave] = any;
  __syncthreads();
  int bad = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) bad |= sBad[w];
  if (bad) {  // (the tiles are shared: all waves or none)
    pass(std::true_type{});
  }

  int lj = li;
  asm volatile("" : "+v"(lj));  // (so that no address of this is kept from before the tiles)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + lj;
    if (r >= it.rows) continue;
    const float l = S.sum[rt][0];
    if (pl.planes > 1) {
      const int64_t pr = part_row(a, it, r);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<f32x4*>(a.part + pr * D + dt * 16 + 4 * grp) = S.o[dt][rt];
      if (grp == 0) *reinterpret_cast<f32x2*>(a.stat + pr * 2) = f32x2{S.mx[rt], l};
    } else {
      const bool live = row_live(a, it, r);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) store_row(a, it, r, dt * 16 + 4 * grp, D, S.o[dt][rt], l, live);
    }
  }
}

// One output row per workgroup: lane s of each wave holds plane s's statistics (at most 64), so the
// weights take one load and a few lane exchanges; each group of D / 4 threads sums every NG-th plane's
// partials (loaded before the weights are known: one trip to memory) and the groups' sums are added in
// group order. MP: a bound of the planes.
template <int D, int MP>
__global__ __launch_bounds__(256) void seg_combine_kernel(SegArgs a, int planes) {
  constexpr int LPR = D / 4, NG = 256 / LPR, N = (MP + NG - 1) / NG;
  __shared__ __attribute__((aligned(16))) f32x4 part[NG][LPR];
  const int G = a.Hq / a.Hk;
  const int64_t rows = (int64_t)a.B * a.T * G, total = rows * a.Hk, i = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1), grp = threadIdx.x / LPR, q = threadIdx.x % LPR;
  const f32x2 st = *reinterpret_cast<const f32x2*>(a.stat + ((lane < planes ? lane : 0) * total + i) * 2);
  f32x4 p[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int s = n * NG + grp;
    p[n] = *reinterpret_cast<const f32x4*>(a.part + ((s < planes ? s : 0) * total + i) * D + q * 4);
  }
  const int kh = (int)(i / rows);
  const int64_t r = i - (int64_t)kh * rows, t = r / G;
  Item it;
  it.kh = kh;
  it.b = (int)(t / a.T);
  const int rr = (int)(r - (int64_t)it.b * a.T * G);
  const bool live = row_live(a, it, rr);
  // A plane's sums may be up to 2^127 about its reference, so the base is above all of the planes' sums, not
  // their references alone, and the factors are applied in halves (e, twice): so neither does a large sum about a low
  // reference fall out (below 2^-126 v_exp_f32 gives 0), nor do several pass the largest number together.
  float m = lane < planes ? st.x + (float)__builtin_amdgcn_frexp_expf(st.y) : -INFINITY;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) m = fmaxf(m, __shfl_xor(m, off));
  const float base = m == -INFINITY ? 0.f : m;
  const float e = lane < planes ? exp2_fast(0.5f * (st.x - base)) : 0.f;
  const float l = wave_sum(lane < planes ? st.y * e * e : 0.f);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int s = n * NG + grp;
    const float w = __shfl(e, s < kWave ? s : 0);  // every lane takes part in the exchange
    if (s < planes) v += p[n] * w * w;
  }
  part[grp][q] = v;
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int g = 1; g < NG; ++g) v += part[g][q];
  store_row(a, it, rr, q * 4, D, v, l, live);
}

// ---- plan ---------------------------------------------------------------------------

constexpr int kGroups = 512;  // workgroups that a call aims at: two per CU
// Rows of a sequence and kv head up to which a shared text is read once for all sequences (us, for all | each by
// itself, heads of 128: 32 sequences of 20 rows of 9000 positions 61 | 162, 8 of 32 rows 40 | 51, 8 of 40 rows 41 | 40,
// 8 of 64 rows 50 | 46). It does not weigh the text's length: past what the second level of cache holds more rows
// can gain (8 of 64 rows of 25000 90 | 92, of 50000 151 | 166, but 32 of 64 rows of 50000 729 | 620), and with many
// rows of a short one packing loses (32 of 32 rows of 2000 48 | 42).
constexpr int64_t kPackedMax = 32;
// Query rows per kv head that seg_rows_kernel takes, in groups of 16 that each read the keys: one group; two of up to
// 4 M elements of keys and while all of their workgroups run at once; up to four of up to 1536 keys in all,
// which the second level of cache then holds (us, it | seg_tiles_kernel, windows and heads of 128: 16 rows of 16 x 4096
// keys 49 | 52; 20 rows of 1024 9.5 | 14, of 4 x 4096 21.7 | 22.4, of 8 x 4096 31.9 | 31.9, of 12 x 4096 58 | 43, of
// 16 x 4096 57 | 53, of 64 x 300 34 | 25, heads of 64: of 32 x 1024 19 | 27; 64 rows of 1000 11 | 16.5, 36 of 2000
// 13 | 16, of 4 x 2000 19.5 | 19.0; a shared text: 20 rows of 1000 9.8 | 13.4, of 9000 20.1 | 18.4, of 50000 41 | 41).
constexpr int64_t kRowsOne = 16, kRowsMax = 32, kRowsShort = 64, kKeys = 1 << 22, kShort = 1536;

// keys: how many a token may see of its own part.
SegPlan seg_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t F, int64_t keys, bool shared) {
  SegPlan p{};
  const int64_t rows = T * (Hq / Hk), all = B * rows;
  // Ranges of at least 128 keys (a block for each wave) or four tiles: shorter ones cost more in partial sums than
  // the waiting that they save (us: 20 rows of 4 x 1024 keys in 128s 14 | 64s 15; 64 rows of 4000 in 256s
  // 18 | 128s 20 | 512s 20).
  const auto cut = [](int64_t n, int64_t keys, int64_t least) {
    const int64_t v = kGroups / n, most = (keys + least - 1) / least;
    return (int)(v < 1 ? 1 : v > most ? most : v);
  };
  p.shared = shared && F > 0 && rows <= kPackedMax;
  const int64_t most = p.shared ? all : rows;
  const int64_t in_all = p.shared ? F : B * (F + keys), heads = p.shared ? Hk : B * Hk;
  const bool few = most <= kRowsOne || (most <= kRowsMax && in_all * D <= kKeys && 2 * heads <= kGroups) ||
                   (most <= kRowsShort && in_all <= kShort);
  // Two row blocks a wave read the tiles half as often from LDS; one makes twice the workgroups, and is taken
  // while they all run at once (us, two | one, a window of 2048: 2000 tokens of 8 kv heads 104 | 120, 1000 tokens
  // 97 | 64; 256 packed rows 73 | 78, 128 52 | 52, 160 59 | 57).
  // Up to 64 rows one is all that there is (128 sequences of 36 rows on a window of 300: 51 | 43).
  if (!few) p.tiles = most > 64 && (p.shared || B * Hk * ((rows + 63) / 64) > kGroups) ? 2 : 1;
  const int64_t unit = p.tiles ? 64 * p.tiles : 16, least = p.tiles ? 256 : 128;
  const int64_t n2 = B * Hk * ((rows + unit - 1) / unit);
  p.split2 = cut(n2, p.shared ? keys : F + keys, least);
  if (p.shared) {
    const int64_t n1 = Hk * ((all + unit - 1) / unit);
    p.split1 = cut(n1, F, least);
    if (p.split2 > 8) p.split2 = 8;
    if (p.split1 > kMaxPlanes - 8) p.split1 = kMaxPlanes - 8;
    p.items1 = (int)(n1 * p.split1);
  }
  if (p.split2 > kMaxPlanes) p.split2 = kMaxPlanes;
  p.items2 = (int)(n2 * p.split2);
  p.planes = p.split1 + p.split2;
  return p;
}

inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

template <int D>
int launch_prep(const SegArgs& a, hipStream_t s) {
  const int64_t heads = (int64_t)a.B * a.T * ((a.qn ? a.Hq : 0) + 2 * a.Hk), per = 256 / (D / 8);
  hipLaunchKernelGGL(seg_prep_kernel<D>, dim3((unsigned)((heads + per - 1) / per)), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

template <int D>
int launch_attend(const SegArgs& a, const SegPlan& p, hipStream_t s) {
  int e = 0;
  const dim3 items((unsigned)(p.items1 + p.items2));
  if (p.tiles == 0) hipLaunchKernelGGL((seg_rows_kernel<D>), items, dim3(256), 0, s, a, p);
  else if (p.tiles == 2) hipLaunchKernelGGL((seg_tiles_kernel<D, 2>), items, dim3(256), 0, s, a, p);
  else hipLaunchKernelGGL((seg_tiles_kernel<D, 1>), items, dim3(256), 0, s, a, p);
  e = (int)hipGetLastError();
  if (e) return e;
  if (p.planes > 1) {
    const dim3 grid((unsigned)((int64_t)a.B * a.T * a.Hq));
    if (p.planes <= 16) hipLaunchKernelGGL((seg_combine_kernel<D, 16>), grid, dim3(256), 0, s, a, p.planes);
    else hipLaunchKernelGGL((seg_combine_kernel<D, kMaxPlanes>), grid, dim3(256), 0, s, a, p.planes);
    e = (int)hipGetLastError();
  }
  return e;
}

}  // namespace

int64_t seg_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t F, int64_t keys, bool shared,
                            bool rope) {
  const SegPlan p = seg_plan(B, T, Hq, Hk, D, F, keys, shared);
  const int64_t rows = B * T * Hq;
  int64_t b = rope && p.tiles ? up256(rows * D * 2) : 0;
  if (p.planes > 1) b += up256(rows * p.planes * 8) + rows * p.planes * D * 4;
  return b;
}

int launch_seg_write(const SegArgs& a, int64_t D, hipStream_t s) {
  return D == 128 ? launch_prep<128>(a, s) : launch_prep<64>(a, s);
}

int launch_seg_attention(SegArgs a, int64_t D, int64_t keys, bool shared, void* ws, hipStream_t s) {
  const SegPlan p = seg_plan(a.B, a.T, a.Hq, a.Hk, D, a.F, keys, shared);
  const int64_t rows = (int64_t)a.B * a.T * a.Hq;
  char* w = (char*)ws;
  a.qsrc = a.q, a.sqsb = a.sqb, a.sqst = a.sqt;
  if (p.tiles && a.cos) {
    a.qn = (uint16_t*)w;
    a.qsrc = a.qn, a.sqst = (int64_t)a.Hq * D, a.sqsb = a.T * a.sqst;
    w += up256(rows * D * 2);
  }
  a.stat = (float*)w;
  if (p.planes > 1) w += up256(rows * p.planes * 8);
  a.part = (float*)w;
  if (p.tiles) {  // (seg_rows_kernel does its own)
    const int e = launch_seg_write(a, D, s);
    if (e) return e;
  }
  return D == 128 ? launch_attend<128>(a, p, s) : launch_attend<64>(a, p, s);
}

}  // namespace fp
