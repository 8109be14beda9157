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
//   - seg_prep_kernel: normalises and rotates q and k (or takes them as they are), writes the new
//     keys and values into the cache.
//   - seg_rows_kernel (few rows per kv head) and seg_tiles_kernel (many): a work item is a group of
//     query rows of one kv head and a range of the key blocks that they see, fixed ones first. Rows are
//     one sequence's (tokens x heads of the group), or, for a shared fixed part alone, those
//     of all sequences. An item of all of its rows' keys writes the output, else partial sums.
//   - seg_combine_kernel: sums the partials of a row in order.
//
// Products as in fp_attn.hip: S^T = K Q^T, so a row's scores lie in one lane column and are the B
// operand of O^T = V^T P^T as they come. Softmax in fp32 with the maximum followed in steps: p is taken
// about a reference that is raised (and the sums scaled) when a score passes it by 2^kLift. The
// sums of p come from the matrix core too, with a row of ones, so they are of p as it enters: in one bf16 part
// (seg_tiles_kernel where it is bound by the products: 2^-9 of each p, no more than the rounding of the
// values' own sums to bf16 costs) or two (2^-17; where keys are what bounds, they cost nothing).
//
// An entry that a row does not see has no part in it, whatever it holds. An infinity or a NaN among
// the values would (0 inf): the sums show it, and then the item is done again with such entries taken
// out of the products and counted for the rows that see them, which become NaN.
#include "fp_common.h"
#include "fp_launch.h"
#include "fp_rope.h"

namespace fp {

namespace {

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLift = 6.f;
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

// One head row per LPH = D / 8 lanes (fp_rope.h). Without cos: k and v only, as they are.
template <int D>
__global__ __launch_bounds__(256) void seg_prep_kernel(SegArgs a) {
  constexpr int LPH = D / 8;
  const int qh = a.cos ? a.Hq : 0, heads = qh + 2 * a.Hk;
  const int64_t items = (int64_t)a.B * a.T * heads;
  int64_t item = (int64_t)blockIdx.x * (256 / LPH) + threadIdx.x / LPH;
  const bool live = item < items;  // dead lanes stay for the cross-lane sums
  if (!live) item = items - 1;
  const int j = threadIdx.x % LPH;
  const int64_t m = item / heads;
  const int h = (int)(item - m * heads), b = (int)(m / a.T), t = (int)(m - (int64_t)b * a.T);
  const bool isq = h < qh, isk = !isq && h < qh + a.Hk;
  const int hk = isk ? h - qh : h - qh - a.Hk;
  const uint16_t* src = isq   ? a.q + b * a.sqb + t * a.sqt + (int64_t)h * D
                        : isk ? a.k + b * a.skb + t * a.skt + (int64_t)hk * D
                              : a.v + b * a.svb + t * a.svt + (int64_t)hk * D;
  u32x2 lo = *reinterpret_cast<const u32x2*>(src + 4 * j);
  u32x2 hi = *reinterpret_cast<const u32x2*>(src + D / 2 + 4 * j);
  if (a.cos && (isq || isk))
    norm_rope_row<D>(lo, hi, isq ? a.gq : a.gk, isq ? a.epsq : a.epsk, a.cos + b * a.scb + t * a.sct,
                     a.sin + b * a.ssb + t * a.sst, j);
  uint16_t* dst;
  if (isq) {
    dst = a.qn + (m * a.Hq + h) * D;
  } else {
    const int p = first_pos(a, b) + t, u = p - a.F;
    if (t >= count(a, b) || !in_cache(a, p)) return;
    if (u < 0) dst = (isk ? a.fk : a.fv) + b * a.sfb + hk * a.sfh + (int64_t)p * a.sfs;
    else dst = (isk ? a.ok : a.ov) + b * a.sob + hk * a.soh + (int64_t)(a.ring ? u % a.S : u) * a.sos;
  }
  if (!live) return;
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

// A operand of V^T for d block dt and keys {4g .. 4g+3, 16 + 4g ..} of 32 V rows in LDS (row
// stride D * 2 bytes, 16-byte chunk c of row r at c ^ (r & (D / 8 - 1))).
template <int D>
__device__ __forceinline__ u32x4 read_vt(const char* rows, int dt, int li, int grp) {
  constexpr int CM = D / 8 - 1;
  const int key = 4 * grp + (li >> 2), c = 2 * dt + ((li & 3) >> 1), half = (li & 1) * 8;
  u32x4 out;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int r = key + 16 * s;
    const char* p = rows + r * (D * 2) + ((c ^ (r & CM)) * 16) + half;
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
  const int per = (total + nsplit - 1) / nsplit;
  it.lo = s * per;
  it.hi = it.lo + per < total ? it.lo + per : total;
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
  // Scores s (NB blocks of 16 keys) of row block rt into probabilities about the reference.
  template <int NB>
  __device__ __forceinline__ void softmax(f32x4 (&s)[NB], int rt, float sc) {
    float m = -INFINITY;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, s[n][r]);
    if (__any(m * sc > mx[rt] + kLift)) {
      const float mn = fmaxf(mx[rt], col_max(m) * sc);
      const float al = mn == -INFINITY ? 1.f : exp2_fast(mx[rt] - mn);
      mx[rt] = mn;
      sum[rt] *= al;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) o[dt][rt] *= al;
    }
    const float base = mx[rt] == -INFINITY ? 0.f : mx[rt];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[n][r] = exp2_fast(fmaf(s[n][r], sc, -base));
  }
  // Whether an infinity or a NaN is in any sum (of values: rows' own scores leave theirs in sum as well).
  __device__ __forceinline__ bool nonfinite() const {
    float t = 0.f;
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
// Bound by the cache's bytes. 16 RT query rows; the four waves take 32-key blocks w, w + 4, ... of the
// item's range, each with the next block's keys in registers and values in its own LDS buffer while it
// computes; their states are merged through LDS in wave order.
// Items: first those of the shared fixed part (grid: n_split1 ranges x row groups x kv heads), then of each
// sequence (ranges x row groups x kv heads x sequences).
template <int D, int RT>
__global__ __launch_bounds__(256, RT == 1 ? 2 : 1) void seg_rows_kernel(SegArgs a, SegPlan pl) {
  constexpr int NW = 4, KB = 32, PARTS = 2;
  constexpr int DK = D / 32, DT = D / 16;      // k-steps of q.k, d blocks of p.V
  constexpr int RPI = 1024 / (D * 2);          // V rows per load instruction
  constexpr int NV = KB / RPI, NK = 2 * DK;    // V and K load instructions per block
  constexpr int CH = D / 8;                    // 16-byte chunks per row
  __shared__ __attribute__((aligned(1024))) char sV0[NW][KB * D * 2];
  __shared__ __attribute__((aligned(1024))) char sV1[NW][KB * D * 2];
  __shared__ float sM[NW][16 * RT], sL[NW][16 * RT];
  __shared__ int sBad[NW];

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
    const int n = (it.rows + 16 * RT - 1) / (16 * RT);
    it.row0 = id % n * 16 * RT;
    it.plane = id / n;
    item_keys<KB>(a, it, 16 * RT, true, false, it.plane, pl.split1);
  } else {
    it.b = id % a.B;
    id /= a.B;
    it.rows = a.T * G;
    const int n = (it.rows + 16 * RT - 1) / (16 * RT);
    it.row0 = id % n * 16 * RT;
    it.plane = pl.split1 + id / n;
    item_keys<KB>(a, it, 16 * RT, !pl.shared, true, id / n, pl.split2);
  }

  u32x4 qf[RT][DK];
  RowKeys rk[RT];
  const int p0 = it.packed ? a.F : first_pos(a, it.b);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = it.row0 + rt * 16 + li;
    rk[rt] = row_keys(a, row_pos(a, it, r < it.rows ? r : it.rows - 1, p0));
    const uint16_t* qp = q_row(a, it, r, D) + 8 * grp;
#pragma unroll
    for (int i = 0; i < DK; ++i) qf[rt][i] = ld16(qp + 32 * i);
  }

  const uint16_t* const kb[2] = {a.fk + it.b * a.sfb + it.kh * a.sfh, a.ok + it.b * a.sob + it.kh * a.soh};
  const uint16_t* const vb[2] = {a.fv + it.b * a.sfb + it.kh * a.sfh, a.ov + it.b * a.sob + it.kh * a.soh};
  const int bytes[2] = {a.F > 0 ? (int)(((int64_t)(a.F - 1) * a.sfs + D) * 2) : 0,
                        (int)(((int64_t)(a.S - 1) * a.sos + D) * 2)};
  const uint32_t step[2] = {(uint32_t)(a.sfs * 2), (uint32_t)(a.sos * 2)};
  const int vr = lane / CH, ring = a.ring ? a.S / KB : 1 << 30;
  auto issue = [&](u32x4 (&kf)[2][DK], char* sv, int c) {
    const int own = c < it.nf ? 0 : 1;
    const int blk = own ? (it.c0 + c - it.nf) % ring : c;
    const uint32_t st = step[own];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int r = n * RPI + vr;
      load_lds16(vb[own], bytes[own], (lds_ptr_t)(sv + n * 1024),
                 (uint32_t)(blk * KB + r) * st + (uint32_t)(((lane % CH) ^ (r & (CH - 1))) * 16));
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < DK; ++i)
        kf[kt][i] = __builtin_amdgcn_raw_buffer_load_b128(make_rsrc(kb[own], bytes[own]),
                                                          (uint32_t)(blk * KB + 16 * kt + li) * st + 16 * grp + 64 * i, 0, 0);
  };

  const float sc = kLog2e / sqrtf((float)D);
  State<D, RT> S;
  auto compute = [&](u32x4 (&kf)[2][DK], const char* sv, int c, bool careful) {
    const int own = c < it.nf ? 0 : 1;
    const int first = own ? (it.c0 + c - it.nf) * KB : c * KB;
    f32x4 s[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        s[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < DK; ++i) s[rt][kt] = mfma16(kf[kt][i], qf[rt][i], s[rt][kt]);
      }
    u32x4 pf[RT][PARTS], seen[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int lo = own ? rk[rt].lo_o : 0, hi = own ? rk[rt].hi_o : rk[rt].hi_f;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = first + kt * 16 + 4 * grp + r;
          if (i < lo || i > hi) s[rt][kt][r] = -INFINITY;
        }
      if (careful) {
        f32x4 t[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = first + kt * 16 + 4 * grp + r;
            t[kt][r] = i < lo || i > hi ? 0.f : 1.f;
          }
        u32x4 f[1];
        split_p<1>(t[0], t[1], f);
        seen[rt] = f[0];
      }
      S.softmax(s[rt], rt, sc);
      split_p<PARTS>(s[rt][0], s[rt][1], pf[rt]);
#pragma unroll
      for (int c2 = 0; c2 < PARTS; ++c2) S.sum[rt] = mfma16(ones8(), pf[rt][c2], S.sum[rt]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      u32x4 vt = read_vt<D>(sv, dt, li, grp);
      if (careful) {
        u32x4 bad;
        take_nonfinite8(vt, bad);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const f32x4 n = mfma16(bad, seen[rt], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n[r] > 0.f) S.o[dt][rt][r] = __uint_as_float(0x7fc00000u);
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int c2 = 0; c2 < PARTS; ++c2) S.o[dt][rt] = mfma16(vt, pf[rt][c2], S.o[dt][rt]);
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

  // Merge the waves' states in wave order. Row block rt's sums go over the wave's own V buffer rt
  // (free now), 16-byte chunk q of row r at q ^ r, so 16 rows' stores spread over the banks.
  static_assert(RT <= 2 && 16 * D * 4 == KB * D * 2, "row sums fit the V buffers");
  auto slot = [&](int w, int r, int q) -> f32x4* {
    char* base = r < 16 ? sV0[w] : sV1[w];
    return reinterpret_cast<f32x4*>(base + (r & 15) * (D * 4) + ((q ^ (r & 15)) * 16));
  };
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (grp == 0) {
      sM[wave][rt * 16 + li] = S.mx[rt];
      sL[wave][rt * 16 + li] = S.sum[rt][0];
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *slot(wave, rt * 16 + li, dt * 4 + grp) = S.o[dt][rt];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * RT * (D / 4); i += NW * kWave) {
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
template <int D, int RT, int PARTS>
__global__ __launch_bounds__(256, 2) void seg_tiles_kernel(SegArgs a, SegPlan pl) {
  constexpr int NW = 4, KB = 64;
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
  int id = blockIdx.x;
  it.kh = id % a.Hk;
  id /= a.Hk;
  it.packed = pl.items1 > 0;
  it.b = 0;
  if (!it.packed) {
    it.b = id % a.B;
    id /= a.B;
  }
  it.rows = (it.packed ? a.B : 1) * a.T * G;
  const int n_rt = (it.rows + 64 * RT - 1) / (64 * RT);
  const int tile = n_rt - 1 - id % n_rt;  // (the later tokens of a prompt see more)
  it.plane = id / n_rt;
  it.row0 = tile * 64 * RT;
  item_keys<KB>(a, it, 64 * RT, true, !it.packed, it.plane, it.packed ? pl.split1 : pl.split2);
  const int row0 = it.row0 + wave * 16 * RT;  // this wave's first row

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

  const uint16_t* const kb[2] = {a.fk + it.b * a.sfb + it.kh * a.sfh, a.ok + it.b * a.sob + it.kh * a.soh};
  const uint16_t* const vb[2] = {a.fv + it.b * a.sfb + it.kh * a.sfh, a.ov + it.b * a.sob + it.kh * a.soh};
  const int bytes[2] = {a.F > 0 ? (int)(((int64_t)(a.F - 1) * a.sfs + D) * 2) : 0,
                        (int)(((int64_t)(a.S - 1) * a.sos + D) * 2)};
  const int ring = a.ring ? a.S / KB : 1 << 30;
  uint32_t off[2][NL];
#pragma unroll
  for (int n = 0; n < NL; ++n) {
    const int r = (wave * NL + n) * RPI + lane / CH;
    const uint32_t ch = (uint32_t)(((lane % CH) ^ (r & (CH - 1))) * 16);
    off[0][n] = (uint32_t)r * (uint32_t)(a.sfs * 2) + ch;
    off[1][n] = (uint32_t)r * (uint32_t)(a.sos * 2) + ch;
  }
  // each tile's rows through a buffer that starts at the tile and ends with the part's last row, so
  // that the lane offset alone tells whether a row is past it
  auto issue = [&](char* sk, char* sv, int c) {
    const int own = c < it.nf ? 0 : 1;
    const int blk = own ? (it.c0 + c - it.nf) % ring : c;
    const int skip = (int)((uint32_t)(blk * KB) * (uint32_t)((own ? a.sos : a.sfs) * 2));
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const uint32_t o = own ? off[1][n] : off[0][n];
      load_lds16((const char*)kb[own] + skip, bytes[own] - skip, (lds_ptr_t)(sk + (wave * NL + n) * 1024), o);
      load_lds16((const char*)vb[own] + skip, bytes[own] - skip, (lds_ptr_t)(sv + (wave * NL + n) * 1024), o);
    }
  };

  const float sc = kLog2e / sqrtf((float)D);
  State<D, RT> S;
  auto compute = [&](const char* sk, const char* sv, int c, bool careful) {
    const int own = c < it.nf ? 0 : 1;
    const int at = own ? (it.c0 + c - it.nf) * KB : c * KB;
    // every key hidden from every row of this wave, or none from any (uniform)
    if (at > (own ? last.hi_o : last.hi_f) || (own && at + KB - 1 < first.lo_o)) return;
    const bool mask = at + KB - 1 > (own ? first.hi_o : first.hi_f) || (own && at < last.lo_o);
    f32x4 s[RT][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DK; ++i) {
        const int r = n * 16 + li;
        const u32x4 kf =
            *reinterpret_cast<const u32x4*>(sk + r * (D * 2) + (((4 * i + grp) ^ (r & (CH - 1))) * 16));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][n] = mfma16(kf, qf[rt][i], s[rt][n]);
      }
    }
    u32x4 pf[RT][2][PARTS], seen[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int lo = own ? rk[rt].lo_o : 0, hi = own ? rk[rt].hi_o : rk[rt].hi_f;
      if (mask) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = at + n * 16 + 4 * grp + r;
            if (i < lo || i > hi) s[rt][n][r] = -INFINITY;
          }
      }
      if (careful) {
        f32x4 t[4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = at + n * 16 + 4 * grp + r;
            t[n][r] = i < lo || i > hi ? 0.f : 1.f;
          }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          u32x4 f[1];
          split_p<1>(t[2 * n], t[2 * n + 1], f);
          seen[rt][n] = f[0];
        }
      }
      S.softmax(s[rt], rt, sc);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        split_p<PARTS>(s[rt][2 * n], s[rt][2 * n + 1], pf[rt][n]);
#pragma unroll
        for (int c2 = 0; c2 < PARTS; ++c2) S.sum[rt] = mfma16(ones8(), pf[rt][n][c2], S.sum[rt]);
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        u32x4 vt = read_vt<D>(sv + n * 32 * D * 2, dt, li, grp);
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
  };
  auto pass = [&](bool careful) {
    S.clear();
    if (it.lo >= it.hi) return;
    issue(sK0, sV0, it.lo);
    for (int c = it.lo; c < it.hi; c += 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = c + u;
        if (k >= it.hi) break;
        // tile k has landed, and every wave is done with the one before
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        __syncthreads();
        if (k + 1 < it.hi) issue(u ? sK0 : sK1, u ? sV0 : sV1, k + 1);
        compute(u ? sK1 : sK0, u ? sV1 : sV0, k, careful);
      }
    }
  };
  pass(false);
  const int any = __any(S.nonfinite()) ? 1 : 0;
  if (lane == 0) sBad[wave] = any;
  __syncthreads();
  if (sBad[0] | sBad[1] | sBad[2] | sBad[3]) {  // (the tiles are shared: all waves or none)
    pass(true);
  }

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + rt * 16 + li;
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
// weights take one load and a few lane exchanges; then each group of D / 4 threads sums every NG-th
// plane's partials and the groups' sums are added in group order.
template <int D>
__global__ __launch_bounds__(256) void seg_combine_kernel(SegArgs a, int planes) {
  constexpr int LPR = D / 4, NG = 256 / LPR;
  __shared__ __attribute__((aligned(16))) f32x4 part[NG][LPR];
  const int G = a.Hq / a.Hk;
  const int64_t rows = (int64_t)a.B * a.T * G, total = rows * a.Hk, i = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1), grp = threadIdx.x / LPR, q = threadIdx.x % LPR;
  const bool has = lane < planes;
  f32x2 st = {-INFINITY, 0.f};
  if (has) st = *reinterpret_cast<const f32x2*>(a.stat + (lane * total + i) * 2);
  float m = st.x;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) m = fmaxf(m, __shfl_xor(m, off));
  const float base = m == -INFINITY ? 0.f : m;
  const float e = has ? exp2_fast(st.x - base) : 0.f;
  const float l = wave_sum(has ? e * st.y : 0.f);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int n = 0; n < kMaxPlanes / NG; ++n) {
    const int s = n * NG + grp;
    const float w = __shfl(e, s);  // every lane takes part in the exchange
    if (s < planes) v += *reinterpret_cast<const f32x4*>(a.part + (s * total + i) * D + q * 4) * w;
  }
  part[grp][q] = v;
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int g = 1; g < NG; ++g) v += part[g][q];
  const int kh = (int)(i / rows);
  const int64_t r = i - (int64_t)kh * rows, n = r / G;
  Item it;
  it.kh = kh;
  it.b = (int)(n / a.T);
  const int rr = (int)(r - (int64_t)it.b * a.T * G);
  store_row(a, it, rr, q * 4, D, v, l, row_live(a, it, rr));
}

// ---- plan ---------------------------------------------------------------------------

constexpr int kGroups = 512;    // workgroups that a call aims at (two per CU)
constexpr int64_t kRowsMax = 64;  // query rows per kv head of seg_rows_kernel

// keys: how many a token may see of its own part.
SegPlan seg_plan(int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t F, int64_t keys, bool shared) {
  SegPlan p{};
  const int64_t G = Hq / Hk, rows = T * G;
  const auto clamp = [](int64_t v, int64_t hi) { return v < 1 ? 1 : v > hi ? hi : v; };
  p.shared = shared && F > 0 && rows <= kRowsMax;
  if (p.shared) {
    // the fixed part's rows are all sequences', in ranges of at least 128 keys (rows) or four tiles
    const int64_t all = B * rows;
    p.tiles1 = all > 32 ? (all > 64 ? 2 : 1) : 0;  // row blocks per wave; 0: seg_rows_kernel
    p.rt = rows > 16 || (!p.tiles1 && all > 16) ? 2 : 1;
    const int64_t unit1 = p.tiles1 ? 64 * p.tiles1 : 16 * p.rt, n1 = (all + unit1 - 1) / unit1 * Hk;
    const int64_t least = p.tiles1 ? 256 : 128;
    p.split1 = (int)clamp(kGroups / n1, (F + least - 1) / least);
    const int64_t n2 = B * Hk * ((rows + 16 * p.rt - 1) / (16 * p.rt));
    p.split2 = (int)clamp(kGroups / n2, (keys + 127) / 128);
    if (p.split1 > kMaxPlanes - 8) p.split1 = kMaxPlanes - 8;
    if (p.split2 > 8) p.split2 = 8;
    p.items1 = (int)(n1 * p.split1);
    p.items2 = (int)(n2 * p.split2);
    p.planes = p.split1 + p.split2;
    return p;
  }
  const int64_t all = F + keys;
  if (rows <= kRowsMax) {
    p.rt = rows <= 16 ? 1 : 2;
    const int64_t n = B * Hk * ((rows + 16 * p.rt - 1) / (16 * p.rt));
    p.split2 = (int)clamp(clamp(kGroups / n, (all + 127) / 128), kMaxPlanes);
    p.items2 = (int)(n * p.split2);
  } else {
    p.tiles2 = B * Hk * ((rows + 127) / 128) >= kGroups ? 2 : 1;
    const int64_t n = B * Hk * ((rows + 64 * p.tiles2 - 1) / (64 * p.tiles2));
    p.split2 = (int)clamp(clamp(kGroups / n, (all + 255) / 256), kMaxPlanes);
    p.items2 = (int)(n * p.split2);
  }
  p.planes = p.split2;
  return p;
}

inline int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

template <int D>
int launch_prep(const SegArgs& a, hipStream_t s) {
  const int64_t heads = (int64_t)a.B * a.T * ((a.cos ? a.Hq : 0) + 2 * a.Hk), per = 256 / (D / 8);
  hipLaunchKernelGGL(seg_prep_kernel<D>, dim3((unsigned)((heads + per - 1) / per)), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

template <int D>
int launch_attend(const SegArgs& a, const SegPlan& p, hipStream_t s) {
  int e = 0;
  SegPlan r = p;
  if (p.tiles1 || p.tiles2) {
    const dim3 grid((unsigned)(p.tiles1 ? p.items1 : p.items2));
    if (p.tiles1 == 1) hipLaunchKernelGGL((seg_tiles_kernel<D, 1, 2>), grid, dim3(256), 0, s, a, p);
    else if (p.tiles1 == 2) hipLaunchKernelGGL((seg_tiles_kernel<D, 2, 2>), grid, dim3(256), 0, s, a, p);
    else if (p.tiles2 == 1) hipLaunchKernelGGL((seg_tiles_kernel<D, 1, 1>), grid, dim3(256), 0, s, a, p);
    else hipLaunchKernelGGL((seg_tiles_kernel<D, 2, 1>), grid, dim3(256), 0, s, a, p);
    e = (int)hipGetLastError();
    if (e) return e;
    r.items1 = 0;
  }
  if (!p.tiles2) {
    const dim3 grid((unsigned)(r.items1 + r.items2));
    if (p.rt == 1) hipLaunchKernelGGL((seg_rows_kernel<D, 1>), grid, dim3(256), 0, s, a, r);
    else hipLaunchKernelGGL((seg_rows_kernel<D, 2>), grid, dim3(256), 0, s, a, r);
    e = (int)hipGetLastError();
    if (e) return e;
  }
  if (p.planes > 1) {
    hipLaunchKernelGGL(seg_combine_kernel<D>, dim3((unsigned)((int64_t)a.B * a.T * a.Hq)), dim3(256), 0, s, a, p.planes);
    e = (int)hipGetLastError();
  }
  return e;
}

}  // namespace

int64_t seg_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t F, int64_t keys, bool shared,
                            bool rope) {
  const SegPlan p = seg_plan(B, T, Hq, Hk, F, keys, shared);
  const int64_t rows = B * T * Hq;
  int64_t b = rope ? up256(rows * D * 2) : 0;
  if (p.planes > 1) b += up256(rows * p.planes * 8) + rows * p.planes * D * 4;
  return b;
}

int launch_seg_write(const SegArgs& a, int64_t D, hipStream_t s) {
  return D == 128 ? launch_prep<128>(a, s) : launch_prep<64>(a, s);
}

int launch_seg_attention(SegArgs a, int64_t D, int64_t keys, bool shared, void* ws, hipStream_t s) {
  const SegPlan p = seg_plan(a.B, a.T, a.Hq, a.Hk, a.F, keys, shared);
  const int64_t rows = (int64_t)a.B * a.T * a.Hq;
  char* w = (char*)ws;
  a.qsrc = a.q, a.sqsb = a.sqb, a.sqst = a.sqt;
  if (a.cos) {
    a.qn = (uint16_t*)w;
    a.qsrc = a.qn, a.sqst = (int64_t)a.Hq * D, a.sqsb = a.T * a.sqst;
    w += up256(rows * D * 2);
  }
  a.stat = (float*)w;
  if (p.planes > 1) w += up256(rows * p.planes * 8);
  a.part = (float*)w;
  const int e = launch_seg_write(a, D, s);
  if (e) return e;
  return D == 128 ? launch_attend<128>(a, p, s) : launch_attend<64>(a, p, s);
}

}  // namespace fp
