// fp_logprob.hip — log-probabilities of given tokens, the entropy and the most
// likely tokens of every row of logits, in one pass over the logits.
//
//   m = max x,  l = sum e^(x-m),  u = sum (x-m) e^(x-m)
//   logprob(t) = x_t - m - log l,   entropy = log l - u / l
//
// u is summed about the maximum, not about zero, so that the entropy of a row far
// from zero does not cancel. The top k are by value, ties to the lowest token.
//
//   - logprob_part_kernel: a workgroup holds one piece of a row in registers (up to
//     256 E elements, all loads in flight at once): its maximum, then its sums and
//     its own top k. Threshold: the k-th largest of the maxima of 64 groups of
//     threads (at least k elements reach it, few more do); the elements that reach
//     it go to LDS and are ranked by counting. Where too many do (a row of equal
//     values) or the sums hold a NaN, k rounds of a workgroup-wide maximum instead.
//   - logprob_join_kernel: one wave per row merges the pieces' sums and sorted lists.
// A row of one piece needs no second launch. Everything is summed in a fixed order.
// 2048 rows of 151936 bf16 logits take 131 us in a graph of such calls (a piece of 64 elements
// per thread, five waves per SIMD), 6 of them to join, 4.8 TB/s: about nine vector operations
// per element keep pace with the loads. One row with its top 20 takes 6 and 5.6 us: launches and the serial
// search, not the 0.3 MB.
//
// A key is (order-preserving bits of the value, ~token): unique, larger is better.
// Key 0 is no element. NaN logits come before +inf.
#include "fp_common.h"
#include "fp_launch.h"

namespace fp {

namespace {

constexpr int kTopCap = 1024;  // candidates that are ranked by counting
constexpr int kTopMax = 64;    // top_k: one lane each in logprob_join_kernel
constexpr int kMaxPieces = 64; // one lane each in logprob_join_kernel

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_f32<0xb1>(v));
  v = fmaxf(v, dpp_f32<0x4e>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
  v = fmaxf(v, dpp_f32<0x140>(v));
  return fmaxf(fmaxf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 0)),
                     __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16))),
               fmaxf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 32)),
                     __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 48))));
}

// The largest of three that is a number (fmaxf would first quiet each operand).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float v;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(v) : "v"(a), "v"(b), "v"(c));
  return v;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
  return v > o ? v : o;
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = dpp_umax<0xb1>(v);
  v = dpp_umax<0x4e>(v);
  v = dpp_umax<0x141>(v);
  v = dpp_umax<0x140>(v);
  const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 0);
  const uint32_t b = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 32);
  const uint32_t d = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
  const uint32_t ab = a > b ? a : b, cd = c > d ? c : d;
  return ab > cd ? ab : cd;
}
__device__ __forceinline__ uint64_t wave_umax64(uint64_t v) {
  const uint32_t hi = wave_umax((uint32_t)(v >> 32));
  const uint32_t lo = wave_umax((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return ((uint64_t)hi << 32) | lo;
}

// Order-preserving bits of a float (-0 as +0; NaN above everything).
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xfffffffeu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  if (o == 0xfffffffeu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t top_key(float x, uint32_t i) {
  return ((uint64_t)ordered(x) << 32) | (uint32_t)~i;
}

// One logit of a row, by its type (DT: 0 bf16, 1 fp16, 2 fp32).
template <int DT>
__device__ __forceinline__ float logit(const void* row, int64_t i) {
  if constexpr (DT == 0) return bf16_bits_to_f32(((const uint16_t*)row)[i]);
  if constexpr (DT == 1) return (float)((const _Float16*)row)[i];
  return ((const float*)row)[i];
}

// Eight logits in registers.
template <int DT>
struct Eight {
  u32x4 w[DT == 2 ? 2 : 1];
  __device__ __forceinline__ float at(int e) const {
    if constexpr (DT == 0)
      return __uint_as_float(e & 1 ? w[0][e / 2] & 0xffff0000u : w[0][e / 2] << 16);
    if constexpr (DT == 1)
      return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[0][e / 2] >> (16 * (e & 1))));
    return __uint_as_float(w[e / 4][e & 3]);
  }
  // elements i .. i+7 of a row, all of them before `end` or none: -inf
  __device__ __forceinline__ void load_whole(const void* row, int64_t i, int64_t end) {
    constexpr int size = DT == 2 ? 4 : 2;
    constexpr uint32_t none = DT == 0 ? 0xff80ff80u : DT == 1 ? 0xfc00fc00u : 0xff800000u;
    const bool has = i < end;
    const char* p = (const char*)row + (has ? i : end - 8) * size;
#pragma unroll
    for (int q = 0; q < (DT == 2 ? 2 : 1); ++q) {
      w[q] = ld16_any(p + 16 * q);
#pragma unroll
      for (int c = 0; c < 4; ++c) w[q][c] = has ? w[q][c] : none;
    }
  }
  // elements i .. i+7 of a row, -inf from `end` on
  __device__ __forceinline__ void load(const void* row, int64_t i, int64_t end) {
    constexpr int size = DT == 2 ? 4 : 2;
    if (__builtin_expect(i + 8 <= end, 1)) {
      const char* p = (const char*)row + i * size;
      w[0] = ld16_any(p);
      if constexpr (DT == 2) w[1] = ld16_any(p + 16);
      return;
    }
    constexpr uint32_t none = DT == 0 ? 0xff80u : DT == 1 ? 0xfc00u : 0xff800000u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (DT == 2) {
        w[e / 4][e & 3] = i + e < end ? ((const uint32_t*)row)[i + e] : none;
      } else {
        const uint32_t h = i + e < end ? (uint32_t)((const uint16_t*)row)[i + e] : none;
        w[0][e / 2] = e & 1 ? w[0][e / 2] | (h << 16) : h;
      }
    }
  }
};

// What a row's sums say about its token and about lane r's top entry.
template <int DT>
__device__ __forceinline__ void write_row(const LogprobArgs& a, int64_t row, float m, float l,
                                          float u) {
  const float log_l = logf(l);
  const int64_t t = a.tokens[row];
  float lp = 0.f;  // a negative token: none is asked for
  if (t >= a.V) lp = __uint_as_float(0x7fc00000u);
  else if (t >= 0)
    lp = logit<DT>((const char*)a.x + row * a.ld * (DT == 2 ? 4 : 2), t) - m - log_l;
  a.logprob[row] = lp;
  a.entropy[row] = log_l - u / l;
}
__device__ __forceinline__ void write_top(const LogprobArgs& a, int64_t row, int r, uint64_t key,
                                          float m, float l) {
  a.top_ids[row * a.k + r] = (int64_t)(uint32_t)~(uint32_t)key;
  a.top_logprobs[row * a.k + r] = from_ordered((uint32_t)(key >> 32)) - m - logf(l);
}

template <int DT, int E, bool TOP>
__global__ __launch_bounds__(256) void logprob_part_kernel(LogprobArgs a) {
  constexpr int NV = E / 8;
  __shared__ float sMax[64];
  __shared__ float sL[4], sU[4];
  __shared__ int sCount;
  __shared__ uint64_t sKey[TOP ? kTopCap : 1];
  __shared__ uint64_t sBest[4];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / a.pieces;
  const int piece = (int)(blockIdx.x - row * a.pieces);
  const int64_t i0 = (int64_t)piece * a.per;
  const int64_t end = i0 + a.per < a.V ? i0 + a.per : a.V;
  const void* x = (const char*)a.x + row * a.ld * (DT == 2 ? 4 : 2);

  Eight<DT> v[NV];
  if ((end - i0) % 8 == 0) {  // whole chunks: no branch between the loads
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j].load_whole(x, i0 + (int64_t)(j * 256 + tid) * 8, end);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j].load(x, i0 + (int64_t)(j * 256 + tid) * 8, end);
  }
  if (TOP && tid == 0) sCount = 0;

  float vm[NV], tm = -INFINITY;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    vm[j] = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; e += 2) vm[j] = max3(vm[j], v[j].at(e), v[j].at(e + 1));
    tm = fmaxf(tm, vm[j]);
  }
  tm = fmaxf(tm, dpp_f32<0xb1>(tm));
  tm = fmaxf(tm, dpp_f32<0x4e>(tm));
  if ((lane & 3) == 0) sMax[tid >> 2] = tm;
  __syncthreads();
  const float gm = sMax[lane];
  const float m = wave_max(gm);

  float l = 0.f, u = 0.f;
  const float base = m == -INFINITY ? 0.f : m;
  if (fabsf(base) < 0x1p20f) {
    // exponents (x - base) log2 e by one operation each, about c = fl(base log2 e); what c is
    // off by (d, up to half a step of c: 2^-4 here, far beyond exp2's range for a mask of
    // -1e10) goes into the sums afterwards
    constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
    const float c = base * kLog2e, d = -fmaf(base, kLog2e, -c);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float z = fmaf(v[j].at(e), kLog2e, -c);
        const float p = __builtin_amdgcn_exp2f(z);
        l += p;
        u = fmaf(fmaxf(z, -1e4f), p, u);  // 0 where z is -inf
      }
    const float r = __builtin_amdgcn_exp2f(d);
    u = fmaf(d, l, u) * (r * kLn2);
    l *= r;
  } else {  // (a maximum of +inf gives NaN)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float z = v[j].at(e) - base;
        const float p = __builtin_amdgcn_exp2f(z * 1.4426950408889634f);
        l += p;
        u += fmaxf(z, -1e4f) * p;
      }
  }
  l = wave_sum(l);
  u = wave_sum(u);
  if (lane == 0) sL[wave] = l, sU[wave] = u;

  if constexpr (TOP) {
    // the 16 high bits of the k-th largest group maximum: at least k elements reach it
    const uint32_t go = ordered(gm) >> 16;
    uint32_t tau = 0;
#pragma unroll
    for (int b = 15; b >= 0; --b) {
      const uint32_t t = tau | (1u << b);
      if (__popcll(__ballot(go >= t)) >= a.k) tau = t;
    }
    // at or under -inf every element of the piece is a candidate
    const bool all = tau <= 0x7fu;
    const float cut = all ? -INFINITY : from_ordered(tau << 16);
    auto offer = [&](const Eight<DT>& c, int64_t i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = c.at(e);
        if (!(f >= cut) || i + e >= end) continue;
        const int at = atomicAdd(&sCount, 1);
        if (at < kTopCap) sKey[at] = top_key(f, (uint32_t)(i + e));
      }
    };
    if constexpr (E == 16) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (vm[j] >= cut) offer(v[j], i0 + (int64_t)(j * 256 + tid) * 8);
    } else {  // read again: kept in registers, the logits would leave two waves per SIMD (206 us)
      uint32_t some = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) some |= (uint32_t)(vm[j] >= cut) << j;
      for (; some; some &= some - 1) {
        const int64_t i = i0 + (int64_t)(__builtin_ctz(some) * 256 + tid) * 8;
        Eight<DT> c;
        c.load(x, i, end);
        offer(c, i);
      }
    }
  }
  __syncthreads();
  l = (sL[0] + sL[1]) + (sL[2] + sL[3]);
  u = (sU[0] + sU[1]) + (sU[2] + sU[3]);
  if (a.pieces > 1) {
    if (tid == 0) reinterpret_cast<f32x4*>(a.stat)[blockIdx.x] = f32x4{m, l, u, 0.f};
  } else if (tid == 0) {
    write_row<DT>(a, row, m, l, u);
  }
  if constexpr (!TOP) return;

  auto put = [&](int r, uint64_t key) {
    if (a.pieces > 1) a.keys[(int64_t)blockIdx.x * a.k + r] = key;
    else write_top(a, row, r, key, m, l);
  };
  const int n = sCount;
  if (n <= kTopCap && l == l) {
    for (int c = tid; c < n; c += 256) {
      const uint64_t key = sKey[c];
      int rank = 0;
#pragma unroll 4
      for (int o = 0; o < n; ++o) rank += sKey[o] > key;
      if (rank < a.k) put(rank, key);
    }
    for (int r = n + tid; r < a.k; r += 256) put(r, 0);  // a piece of fewer than k elements
    return;
  }
  uint64_t last = ~0ull;
  for (int r = 0; r < a.k; ++r) {
    uint64_t best = 0;
#pragma unroll 2
    for (int64_t i = i0 + tid * 8; i < end; i += 2048) {
      Eight<DT> c;
      c.load(x, i, end);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint64_t key = i + e < end ? top_key(c.at(e), (uint32_t)(i + e)) : 0;
        if (key < last && key > best) best = key;
      }
    }
    best = wave_umax64(best);
    __syncthreads();  // sBest of the last round has been read
    if (lane == 0) sBest[wave] = best;
    __syncthreads();
    best = sBest[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) best = best > sBest[w] ? best : sBest[w];
    if (tid == 0) put(r, best);
    last = best;
  }
}

// One wave per row: lane s holds piece s's sums and the head of its sorted list;
// k rounds take the largest head.
template <int DT>
__global__ __launch_bounds__(64) void logprob_join_kernel(LogprobArgs a) {
  extern __shared__ uint64_t list[];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const bool has = lane < a.pieces;
  const int n_keys = a.pieces * a.k;
  const uint64_t* keys = a.keys + row * n_keys;
  for (int i0 = 0; i0 < n_keys; i0 += 512) {  // eight loads in flight (one at a time: 7.2 us for 760, against 5.6)
    uint64_t key[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * 64 + lane;
      key[j] = keys[i < n_keys ? i : 0];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * 64 + lane;
      if (i < n_keys) list[i] = key[j];
    }
  }
  f32x4 st = {-INFINITY, 0.f, 0.f, 0.f};
  if (has) st = reinterpret_cast<const f32x4*>(a.stat)[row * a.pieces + lane];
  const float m = wave_max(st[0]);
  // a piece of nothing but -inf adds nothing (its e is 0, its distance kept finite)
  const float d = fmaxf(st[0] - (m == -INFINITY ? 0.f : m), -1e4f);
  const float e = has ? __builtin_amdgcn_exp2f(d * 1.4426950408889634f) : 0.f;
  const float l = wave_sum(e * st[1]);
  const float u = wave_sum(e * (st[2] + d * st[1]));
  if (lane == 0) write_row<DT>(a, row, m, l, u);
  if (a.k == 0) return;
  __syncthreads();
  uint64_t head = has ? list[lane * a.k] : 0, mine = 0;
  int next = 1;
  for (int r = 0; r < a.k; ++r) {
    const uint64_t best = wave_umax64(head);
    if (lane == r) mine = best;
    if (head == best) {
      head = next < a.k && has ? list[lane * a.k + next] : 0;
      ++next;
    }
  }
  if (lane < a.k) write_top(a, row, lane, mine, m, l);
}

// Pieces of a row: registers hold up to 64 elements of a thread; rows are cut finer
// (down to 16) while the call has fewer than 512 workgroups, two per CU.
struct LogprobPlan {
  int e;        // elements per thread
  int pieces;
  int64_t per;  // elements per piece, a multiple of 8
};
LogprobPlan logprob_plan(int64_t M, int64_t V) {
  LogprobPlan p;
  p.e = 64;
  if (M * ((V + 256 * 64 - 1) / (256 * 64)) < 512 && V <= kMaxPieces * 256 * 16) p.e = 16;
  p.pieces = (int)((V + 256 * p.e - 1) / (256 * p.e));
  p.per = ((V + p.pieces - 1) / p.pieces + 7) / 8 * 8;
  p.pieces = (int)((V + p.per - 1) / p.per);
  return p;
}

template <int DT, int E>
int launch_part(const LogprobArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.M * a.pieces)), block(256);
  if (a.k) hipLaunchKernelGGL((logprob_part_kernel<DT, E, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((logprob_part_kernel<DT, E, false>), grid, block, 0, s, a);
  return (int)hipGetLastError();
}

template <int DT>
int launch_dt(LogprobArgs a, const LogprobPlan& p, hipStream_t s) {
  const int rc = p.e == 64 ? launch_part<DT, 64>(a, s) : launch_part<DT, 16>(a, s);
  if (rc || a.pieces == 1) return rc;
  hipLaunchKernelGGL(logprob_join_kernel<DT>, dim3((unsigned)a.M), dim3(64),
                     (size_t)(a.pieces * a.k * 8), s, a);
  return (int)hipGetLastError();
}

}  // namespace

bool logprob_supported(int64_t M, int64_t V, int64_t k) {
  if (M < 1 || V < 1 || V > (int64_t)kMaxPieces * 256 * 64 || k < 0 || k > kTopMax || k > V)
    return false;
  // grids of at most 2^32 threads
  return M <= (int64_t)1 << 24 && M * logprob_plan(M, V).pieces <= (int64_t)1 << 23;
}

int64_t logprob_workspace_bytes(int64_t M, int64_t V, int64_t k) {
  const LogprobPlan p = logprob_plan(M, V);
  return p.pieces > 1 ? M * p.pieces * (16 + 8 * k) : 0;
}

int launch_logprobs(LogprobArgs a, int dtype, void* ws, hipStream_t s) {
  const LogprobPlan p = logprob_plan(a.M, a.V);
  a.pieces = p.pieces;
  a.per = p.per;
  a.stat = (float*)ws;
  a.keys = (uint64_t*)((char*)ws + a.M * p.pieces * 16);
  return dtype == 0 ? launch_dt<0>(a, p, s) : dtype == 1 ? launch_dt<1>(a, p, s) : launch_dt<2>(a, p, s);
}

}  // namespace fp
