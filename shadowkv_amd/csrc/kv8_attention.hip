// Attention over an 8-bit KV cache (the format of kv8.hip): the new tokens of each sequence, its last ones, over
// the cached keys and values that they see.
//
//   out[b, t, hq] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b, hq, t] . k_j),  k_j = ks * code, v_j = vs * code
//
// over the keys j <= p of the query's position p = length_b - n_b + t, with a window w only those with j > p - w
// or j < sinks. A query that sees nothing, or is padding (t >= n_b), gets zeros. Codes become bf16 (exactly) on
// their way into the matrix cores; a key block's scale multiplies its scores and a value block's scale its
// probabilities, so no dequantised row is ever formed. Scores, probabilities and sums are fp32; a probability
// enters the product with the values as two bf16 parts (16 significant bits, an error of 2^-16 where the output's
// one rounding is 2^-9).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "skv_common.h"

namespace {

using skv::u32x4;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kD = 128;
constexpr int kNoWindow = 1 << 30;

struct Args {
  const uint16_t* q;
  int64_t q_sb, q_sh, q_st;
  const uint8_t* k8;
  const uint8_t* v8;
  int64_t c_sb, c_sh, c_ss;
  const float* ks;
  const float* vs;
  int64_t s_sb, s_sh;
  const int32_t* lengths;
  const int32_t* counts;
  uint16_t* out;  // [B, T, Hq, 128]
  float* ws_o;
  float* ws_ml;
  int B, H, G, T, cap, block_shift, window, sinks;
  float scale_log2e;  // of the scale's magnitude
  bool negative;      // whether the scale is: the queries' sign is turned instead
  int target;   // one token: workgroups to aim for
  int splits;   // many: shares of a row tile's keys
  int rtiles;   // many: row tiles of a (sequence, kv head)
};

__device__ __forceinline__ int length_of(const Args& a, int b) { return min(max(a.lengths[b], 0), a.cap); }
__device__ __forceinline__ int count_of(const Args& a, int b) {
  return a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
}

// The groups of 2^shift keys that hold a key seen by a query at a position in [pmin, pmax]: the first `first`,
// and those behind the next `skip`; `total` in all.
struct Groups {
  int first, skip, total;
  __device__ __forceinline__ int at(int i) const { return i < first ? i : i + skip; }
};
__device__ __forceinline__ Groups groups_seen(int pmin, int pmax, int window, int sinks, int shift) {
  if (pmax < 0) return {0, 0, 0};
  const int end = (pmax >> shift) + 1;
  const int lo = max(0, max(pmin, 0) - window + 1);
  const int s = (min(sinks, lo) + (1 << shift) - 1) >> shift, w = lo >> shift;
  if (w <= s) return {end, 0, end};
  return {s, w - s, end - (w - s)};
}

__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) {
  return j <= p && (j > p - window || j < sinks);
}

// A scale at a wave-uniform place, through the scalar unit (nothing writes the scales while these kernels run).
__device__ __forceinline__ float scale_at(const float* scales, int block) {
  return *reinterpret_cast<const __attribute__((address_space(4))) float*>(reinterpret_cast<uintptr_t>(scales + block));
}

// A key block's factor of its scores, in units of log2: positive, so that a hidden key's -inf stays one.
__device__ __forceinline__ float key_factor(float scale, float scale_log2e) {
  const float f = scale * scale_log2e;
  return f < 1.17549435e-38f ? 1.17549435e-38f : f;  // (NaN stays NaN)
}

__device__ __forceinline__ bf16x8 bf16_of(uint32_t a, uint32_t b) {
  u32x4 o;
  o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false));
  o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true));
  o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, false));
  o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, true));
  return __builtin_bit_cast(bf16x8, o);
}

// Eight tokens' codes of four dims, a token's in w[i], as the bf16 of each dim's eight tokens in turn: o[dim].
__device__ __forceinline__ void transpose_bf16(const uint32_t (&w)[8], u32x4 (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05010400u);  // dims 0 and 1 of the pair
    const uint32_t hi = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07030602u);  // dims 2 and 3
    o[0][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
    o[1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
    o[2][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
    o[3][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
  }
}

// The same as f16 of code * factor (a power of two).
__device__ __forceinline__ void transpose_f16(const uint32_t (&w)[8], float factor, u32x4 (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05010400u);
    const uint32_t hi = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07030602u);
    o[0][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, factor, false));
    o[1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, factor, true));
    o[2][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, factor, false));
    o[3][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, factor, true));
  }
}

// Two fp32 as two bf16 parts each: part[0] cut off, part[1] what that leaves, rounded.
__device__ __forceinline__ void two_parts(float x0, float x1, uint32_t& first, uint32_t& second) {
  const uint32_t a0 = __float_as_uint(x0), a1 = __float_as_uint(x1);
  first = __builtin_amdgcn_perm(a1, a0, 0x07060302u);
  second = skv::f2bf2(x0 - __uint_as_float(a0 & 0xffff0000u), x1 - __uint_as_float(a1 & 0xffff0000u));
}

__device__ __forceinline__ float max_of_rows(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
  s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float sum_of_rows(float x) {
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// ------------------------------------------------------------------------------------------------
// One new token a sequence, at most 16 query heads to a kv head.
//
// Bound: HBM, 256 bytes a key. The sequences' keys are cut into chunks of equal length, however different the
// sequences are (planned on the device from the lengths, so that a captured call follows them), each a workgroup
// of four waves that take its groups of 32 keys in turn, straight from memory into registers: S^T = K Q^T on
// v_mfma_f32_16x16x32_bf16 (a query head a column) leaves a lane with 8 keys' scores of one head, which is the
// second operand of O^T = V^T P^T, whose first is the lane's 8 tokens of one dim: neither probabilities nor
// values cross lanes.
constexpr int kGroup = 32;
constexpr int kGroupShift = 5;
constexpr int kMinGroups = 8;   // a chunk's groups of 32 keys, at least
constexpr int kTarget = 1024;   // chunks to aim for: four workgroups to a CU
constexpr int kOutLd = kD + 4;

struct Chunk {
  int b, index, groups;  // sequence, which of its chunks, groups of a chunk
};

__device__ __forceinline__ Groups token_groups(const Args& a, int b) {
  const int p = length_of(a, b) - 1;
  return groups_seen(count_of(a, b) ? p : -1, count_of(a, b) ? p : -1, a.window, a.sinks, kGroupShift);
}

// The chunk length, wave-uniform: the sequences' groups dealt over the workgroups to aim for.
__device__ __forceinline__ int chunk_groups(const Args& a, int lane) {
  int64_t total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int t = b0 + lane < a.B ? token_groups(a, b0 + lane).total : 0;
    total += __builtin_amdgcn_readlane(skv::wave_inclusive_scan(t), 63);
  }
  return static_cast<int>(max(static_cast<int64_t>(kMinGroups), (total * a.H + a.target - 1) / a.target));
}

// Chunk i of all sequences' (false past the last).
__device__ __forceinline__ bool find_chunk(const Args& a, int i, int lane, Chunk& c) {
  c.groups = chunk_groups(a, lane);
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int n = b0 + lane < a.B ? (token_groups(a, b0 + lane).total + c.groups - 1) / c.groups : 0;
    const int incl = before + skv::wave_inclusive_scan(n);
    const uint64_t hit = __ballot(i < incl && i >= incl - n);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      c.b = b0 + l;
      c.index = i - __builtin_amdgcn_readlane(incl - n, l);
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

__global__ void __launch_bounds__(256) token_kernel(Args a) {
  __shared__ float o_lds[4][16][kOutLd];
  __shared__ float m_lds[4][16], l_lds[4][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = blockIdx.x / a.H, h = blockIdx.x - slot * a.H;
  Chunk c;
  if (!find_chunk(a, slot, lane, c)) return;  // workgroup-uniform
  const int b = c.b, G = a.G;
  const int len = length_of(a, b), p = len - 1;
  const Groups seen = token_groups(a, b);
  const int i0 = c.index * c.groups, i1 = min(i0 + c.groups, seen.total);
  const int li = lane & 15, grp = lane >> 4;

  // Q as the B operand: lane (li, grp) holds head li, in step s dims 64 (s / 2) + 16 grp + 8 (s % 2) and on.
  bf16x8 qf[4];
  {
    const uint16_t* q = a.q + b * a.q_sb + (h * G + min(li, G - 1)) * a.q_sh + 16 * grp;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      qf[s] = __builtin_bit_cast(bf16x8, skv::load16_or_zero(q + 64 * (s >> 1) + 8 * (s & 1), li < G) ^
                                             (a.negative ? 0x80008000u : 0u));
  }
  const uint8_t* kh = a.k8 + b * a.c_sb + h * a.c_sh + 16 * grp;
  const uint8_t* vh = a.v8 + b * a.c_sb + h * a.c_sh + 8 * li;
  const float* ksh = a.ks + b * a.s_sb + h * a.s_sh;
  const float* vsh = a.vs + b * a.s_sb + h * a.s_sh;

  f32x4 o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // the head's reference, in units of log2; this lane's share of its sum

  u32x4 kr[2][2];
  u32x2 vr[8];
  float kc[2], vc[2];
  auto load = [&](int i) __attribute__((always_inline)) {
    const int j0 = seen.at(i) * kGroup;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t* row = kh + static_cast<int64_t>(min(j0 + 16 * u + li, p)) * a.c_ss;
      kr[u][0] = *reinterpret_cast<const u32x4*>(row);
      kr[u][1] = *reinterpret_cast<const u32x4*>(row + 64);
      const int blk = min(j0 + 16 * u, p) >> a.block_shift;
      kc[u] = ksh[blk];
      vc[u] = vsh[blk];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        vr[4 * u + r] = *reinterpret_cast<const u32x2*>(
            vh + static_cast<int64_t>(min(j0 + 16 * u + 4 * grp + r, p)) * a.c_ss);
  };

  for (int i = i0 + wave; i < i1; i += 4) {
    load(i);
    const int j0 = seen.at(i) * kGroup;
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < 4; ++st)
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            bf16_of(kr[u][st >> 1][2 * (st & 1)], kr[u][st >> 1][2 * (st & 1) + 1]), qf[st], s[u], 0, 0, 0);
      const float f = key_factor(kc[u], a.scale_log2e);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[u][r] *= f;
    }
    // wave-uniform: a group at an end of what the token sees. Hidden values may be anything: zero codes.
    if (j0 + kGroup > len || (j0 < len - a.window && j0 + kGroup > a.sinks)) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!sees(p, j0 + 16 * u + 4 * grp + r, a.window, a.sinks)) {
            s[u][r] = -INFINITY;
            vr[4 * u + r] = u32x2{0u, 0u};
          }
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = max_of_rows(mx);
    if (__any(mx > m)) {  // wave-uniform
      const float mn = fmaxf(m, mx);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= f;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    u32x4 part[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(s[u][r] - ref), p1 = __builtin_amdgcn_exp2f(s[u][r + 1] - ref);
        l += p0 + p1;
        uint32_t first, second;
        two_parts(p0 * vc[u], p1 * vc[u], first, second);
        part[0][2 * u + r / 2] = first;
        part[1][2 * u + r / 2] = second;
      }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t w[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) w[t] = vr[t][half];
      u32x4 vf[4];
      transpose_bf16(w, vf);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          o[4 * half + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, vf[e]), __builtin_bit_cast(bf16x8, part[x]), o[4 * half + e], 0, 0, 0);
    }
  }

  // The waves' parts: lane (li, grp) holds head li's dims 8 (4 grp + r) + e.
  l = sum_of_rows(l);
  if (grp == 0) {
    m_lds[wave][li] = m;
    l_lds[wave][li] = l;
  }
  if (li < G) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<f32x4*>(&o_lds[wave][li][8 * (4 * grp + r) + e]) =
            f32x4{o[e][r], o[e + 1][r], o[e + 2][r], o[e + 3][r]};
  }
  __syncthreads();
  const int64_t row0 = (static_cast<int64_t>(slot) * a.H + h) * G;
  for (int i = threadIdx.x; i < G * 32; i += 256) {
    const int g = i >> 5, d = 4 * (i & 31);
    float top = m_lds[0][g];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, m_lds[w][g]);
    const float ref = top == -INFINITY ? 0.f : top;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    float ls = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(m_lds[w][g] - ref);
      ls += f * l_lds[w][g];
      sum += f * *reinterpret_cast<const f32x4*>(&o_lds[w][g][d]);
    }
    *reinterpret_cast<f32x4*>(a.ws_o + (row0 + g) * kD + d) = sum;
    if (d == 0) {
      a.ws_ml[2 * (row0 + g)] = top;
      a.ws_ml[2 * (row0 + g) + 1] = ls;
    }
  }
}

// Joins n partial results (m, l, o), part i at index first + i * stride, into one row: 256 threads, 32 lanes of
// four dims by 8 parts at a time. Every wave of it sees the same maximum and sum.
__device__ __forceinline__ void join_parts(const float* ws_o, const float* ws_ml, int64_t first, int64_t stride, int n,
                                           uint16_t* out, f32x4 (&acc_lds)[8][32]) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  for (int i = lane; i < n; i += 64) m = fmaxf(m, ws_ml[2 * (first + i * stride)]);
  m = skv::wave_max_dpp(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int i = lane; i < n; i += 64)
    l += ws_ml[2 * (first + i * stride) + 1] * __builtin_amdgcn_exp2f(ws_ml[2 * (first + i * stride)] - ref);
  l = skv::wave_sum_dpp(l);
  const int d = threadIdx.x & 31, s = threadIdx.x >> 5;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = s; i < n; i += 8) {
    const int64_t at = first + i * stride;
    acc += __builtin_amdgcn_exp2f(ws_ml[2 * at] - ref) * *reinterpret_cast<const f32x4*>(ws_o + at * kD + 4 * d);
  }
  acc_lds[s][d] = acc;
  __syncthreads();
  if (threadIdx.x < 32) {
#pragma unroll
    for (int i = 1; i < 8; ++i) acc += acc_lds[i][d];
    const float inv = l == 0.f ? 0.f : 1.f / l;  // (nothing seen: zeros)
    *reinterpret_cast<u32x2*>(out + 4 * d) = {skv::f2bf2(acc[0] * inv, acc[1] * inv),
                                              skv::f2bf2(acc[2] * inv, acc[3] * inv)};
  }
}

__global__ void __launch_bounds__(256) token_join_kernel(Args a) {
  __shared__ f32x4 acc_lds[8][32];
  const int lane = threadIdx.x & 63;
  const int Hq = a.H * a.G;
  const int b = blockIdx.x / Hq, hq = blockIdx.x - b * Hq;
  const int h = hq / a.G, g = hq - h * a.G;
  const int each = chunk_groups(a, lane);
  int before = 0;
  for (int b0 = 0; b0 < b; b0 += 64) {
    const int n = b0 + lane < b ? (token_groups(a, b0 + lane).total + each - 1) / each : 0;
    before += __builtin_amdgcn_readlane(skv::wave_inclusive_scan(n), 63);
  }
  const int n = (token_groups(a, b).total + each - 1) / each;
  join_parts(a.ws_o, a.ws_ml, (static_cast<int64_t>(before) * a.H + h) * a.G + g, static_cast<int64_t>(a.H) * a.G, n,
             a.out + static_cast<int64_t>(blockIdx.x) * kD, acc_lds);
}

// ------------------------------------------------------------------------------------------------
// Several new tokens a sequence, or more than 16 query heads to a kv head.
//
// Bound: the matrix cores (with few rows, HBM). The rows of a kv head are its queries' heads together, row
// t * G + g, so that a tile of keys serves all of them. A workgroup of four waves owns 128 rows (32 a wave, a row
// a lane) and walks the tiles of 64 keys that any of them sees, or a share of them where there are too few rows to
// fill the chip. Keys and values are read once a tile, turned into bf16 (the values transposed) by the threads
// that read them, and shared through LDS, the next tile on its way meanwhile.
constexpr int kTile = 64;
constexpr int kTileShift = 6;
constexpr int kRowsWave = 32;
constexpr int kRowsTile = 4 * kRowsWave;

// 16-byte chunk c (8 dims) of key row r of a tile in LDS, and chunk (group of 16 keys, half of its order, dim).
__device__ __forceinline__ int k_at(int r, int c) { return r * 16 + (c ^ (r & 15)); }
__device__ __forceinline__ int v_at(int gk, int half, int d) { return gk * 256 + half * 128 + (d ^ ((d >> 3) & 7)); }

__device__ __forceinline__ u32x4 load4(const uint8_t* p) { return *reinterpret_cast<const u32x4*>(p); }

// 0x80 in each byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Powers of two by which the value blocks of a workgroup may differ for f16 to hold their values exactly, and the
// one that the largest block's codes are raised by: 448 * 2^7 is just below f16's largest, 2^-9 * 2^(7 - 12) its
// smallest normal value.
constexpr int kSpread = 12;
constexpr int kRaise = 7;
// A probability is at most 2^(kRaise + kSlack), below f16's largest: kSlack is how far a score may pass the reference.
constexpr float kSlack = 8.f;

__global__ void __launch_bounds__(256, 2) rows_kernel(Args a) {
  __shared__ u32x4 kt[2][kTile * 16], vt[2][kTile * 16];
  // Values that are NaN, by (buffer, wave that carries them): whether there are any, and each dim's keys as bits.
  __shared__ int odd_lds[2][2];
  __shared__ uint32_t odd_keys[2][2][kD];
  __shared__ int vexp[3];  // largest and smallest exponent of the value blocks' scales, whether one is no power of two
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 31, half = lane >> 5;
  int i = blockIdx.x;
  const int BH = a.B * a.H;
  const int bh = i % BH;
  i /= BH;
  const int split = i % a.splits;
  const int rt = a.rtiles - 1 - i / a.splits;  // the longest first
  const int b = bh / a.H, h = bh - b * a.H;
  const int G = a.G, R = a.T * G;
  const int len = length_of(a, b), n = count_of(a, b);
  const int r0 = rt * kRowsTile;
  const int p0 = len - n;  // the position of the first new token
  // The rows' positions; those of padding see nothing.
  const int t_last = min(n - 1, (r0 + kRowsTile - 1) / G);
  const int pmin = p0 + r0 / G, pmax = r0 / G < n ? p0 + t_last : -1;
  const Groups seen = groups_seen(pmin, pmax, a.window, a.sinks, kTileShift);
  const int each = (seen.total + a.splits - 1) / a.splits;
  const int i0 = min(split * each, seen.total), i1 = min(i0 + each, seen.total);

  const int row = r0 + wave * kRowsWave + li;
  const int t = min(row, R - 1) / G, g = min(row, R - 1) - t * G;
  const int p = row < R && t < n ? p0 + t : -1;
  // the wave's positions (wave-uniform): rows past the last or of padding do not widen them
  const int wr = r0 + wave * kRowsWave;
  const int wmin = p0 + wr / G, wmax = wr / G < n ? p0 + min(n - 1, (wr + kRowsWave - 1) / G) : -1;
  const bool whole = wr + kRowsWave <= R && (wr + kRowsWave - 1) / G < n;  // every row of the wave is a query

  u32x4 qf[8];
  {
    const uint16_t* q = a.q + b * a.q_sb + (h * G + g) * a.q_sh + t * a.q_st + 8 * half;
#pragma unroll
    for (int s = 0; s < 8; ++s) qf[s] = *reinterpret_cast<const u32x4*>(q + 16 * s);
    if (a.negative)
#pragma unroll
      for (int s = 0; s < 8; ++s) qf[s] ^= 0x80008000u;
  }
  const uint8_t* kh = a.k8 + b * a.c_sb + h * a.c_sh;
  const uint8_t* vh = a.v8 + b * a.c_sb + h * a.c_sh;
  const float* ksh = a.ks + b * a.s_sb + h * a.s_sh;
  const float* vsh = a.vs + b * a.s_sb + h * a.s_sh;

  // Waves 0 and 1 carry the keys (a thread 64 bytes of a row), waves 2 and 3 the values (a thread 8 dims of the 8
  // tokens of a half group, the keys' order in the scores' registers).
  const int x = threadIdx.x & 127;
  const int krow = x >> 1, kpart = x & 1;
  const int vgk = x >> 5, vhalf = (x >> 4) & 1, vc = x & 15;
  // Row offsets of the thread in a tile; rows behind the sequence's end are out of the buffer's bounds and come as
  // zeros, whatever lies there.
  const int stride = static_cast<int>(a.c_ss);
  const int mine = wave < 2 ? krow * stride + 64 * kpart : (16 * vgk + 4 * vhalf) * stride + 8 * vc;
  u32x4 held[4];
  float kf[4], kn[4];  // this tile's and the next one's key factors
  auto fetch = [&](int tile) __attribute__((always_inline)) {
    const int64_t j0 = static_cast<int64_t>(tile) * kTile;
    const int bytes = min(len - tile * kTile - 1, kTile - 1) * stride + kD;
    constexpr int kDw3 = 0x00020000;  // buffer resource word 3 (gfx9)
    if (wave < 2) {
      const __amdgpu_buffer_rsrc_t src =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(kh + j0 * a.c_ss), 0, bytes, kDw3);
#pragma unroll
      for (int c = 0; c < 4; ++c) held[c] = __builtin_amdgcn_raw_buffer_load_b128(src, mine, 16 * c, 0);
    } else {
      const __amdgpu_buffer_rsrc_t src =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(vh + j0 * a.c_ss), 0, bytes, kDw3);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(src, mine, ((e & 3) + 8 * (e >> 2)) * stride, 0);
        held[e >> 1][2 * (e & 1)] = w[0];
        held[e >> 1][2 * (e & 1) + 1] = w[1];
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      kn[q] = key_factor(scale_at(ksh, min(tile * kTile + 16 * q, len - 1) >> a.block_shift), a.scale_log2e);
  };
  auto place = [&](auto f16, float factor, int buf) __attribute__((always_inline)) {
    if (wave < 2) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        kt[buf][k_at(krow, 8 * kpart + 2 * c)] = __builtin_bit_cast(u32x4, bf16_of(held[c][0], held[c][1]));
        kt[buf][k_at(krow, 8 * kpart + 2 * c + 1)] = __builtin_bit_cast(u32x4, bf16_of(held[c][2], held[c][3]));
      }
    } else {
      bool any = false;
      if constexpr (!decltype(f16)::value) {
        uint32_t odd = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= nan_bytes(held[c][e]);
        any = __any(odd != 0);
        if (lane == 0) odd_lds[buf][wave - 2] = any;
      }
      if (any) {  // wave-uniform: their keys are noted, and they enter the products as zeros
        uint32_t* keys = odd_keys[buf][wave - 2];
        keys[lane] = 0u;
        keys[lane + 64] = 0u;
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t f = nan_bytes(held[c][e]);
            const int t = 2 * c + (e >> 1);  // the token, in the order of the registers
            const int key = 16 * (vgk & 1) + 4 * vhalf + (t & 3) + 8 * (t >> 2);
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (f & (0x80u << (8 * y))) atomicOr(&keys[8 * vc + 4 * (e & 1) + y], 1u << key);
            held[c][e] &= ~((f >> 7) * 0xffu);
          }
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = held[e >> 1][2 * (e & 1) + hf];
        u32x4 o[4];
        if constexpr (decltype(f16)::value) transpose_f16(w, factor, o);
        else transpose_bf16(w, o);
#pragma unroll
        for (int e = 0; e < 4; ++e) vt[buf][v_at(vgk, vhalf, 8 * vc + 4 * hf + e)] = o[e];
      }
    }
  };

  f32x16 o[4];
  float m, l;
  uint64_t odd = 0;  // this lane's output dims that a value seen by its row makes NaN, bit 16 d + r

  auto compute = [&](auto f16, int tile, int buf) __attribute__((always_inline)) {
    constexpr bool kF16 = decltype(f16)::value;
    const int k0 = tile * kTile;
    // wave-uniform: nothing of the tile is seen
    if (k0 > wmax || (k0 + kTile <= wmin - a.window + 1 && k0 >= a.sinks)) return;
    f32x16 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, kt[buf][k_at(32 * u + li, 2 * c + half)]), __builtin_bit_cast(bf16x8, qf[c]),
            s[u], 0, 0, 0);
    // Registers 8 i to 8 i + 7 of s[u] hold 8 of the keys 32 u + 16 i to 32 u + 16 i + 15, which share a block.
    const bool all = whole && k0 + kTile - 1 <= wmin && (k0 > wmax - a.window || k0 + kTile <= a.sinks);
    if (!all) {  // wave-uniform
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!sees(p, k0 + 32 * u + 8 * (r / 4) + 4 * half + (r % 4), a.window, a.sinks)) s[u][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float y = s[q >> 1][8 * (q & 1)];
#pragma unroll
      for (int r = 1; r < 8; ++r) y = fmaxf(y, s[q >> 1][8 * (q & 1) + r]);
      mx = fmaxf(mx, y * kf[q]);
    }
    {
      const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
      mx = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
    }
    // The reference moves only when a score passes it by 2^kSlack: the ratio of the sums does not depend on it.
    if (__any(mx > m + kSlack)) {  // wave-uniform
      const float mn = fmaxf(m, mx);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
    }
    const float ref = (m == -INFINITY ? 0.f : m) - static_cast<float>(kRaise);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], kf[2 * u + (r >> 3)], -ref));
        l += s[u][r];
      }
    if (!kF16 && (odd_lds[buf][0] | odd_lds[buf][1])) {  // the same for all waves
      // A value that is NaN makes the sums of the rows that see its key NaN, and no others (in the product it
      // would: a hidden key's zero times NaN).
      for (int hw = 0; hw < 2; ++hw) {
        if (!odd_lds[buf][hw]) continue;
        uint32_t vis = 0;
        for (int j = 0; j < 32; ++j) vis |= sees(p, k0 + 32 * hw + j, a.window, a.sinks) ? 1u << j : 0u;
        for (int d = 0; d < 64; ++d)
          if (odd_keys[buf][hw][32 * (d >> 4) + 8 * ((d & 15) >> 2) + 4 * half + (d & 3)] & vis) odd |= 1ull << d;
      }
    }
#pragma unroll
    for (int gk = 0; gk < 4; ++gk) {
      u32x4 vf[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) vf[d] = vt[buf][v_at(gk, half, 32 * d + li)];
      if constexpr (kF16) {
        u32x4 part;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          part[e] = __builtin_bit_cast(
              uint32_t, __builtin_convertvector(f32x2{s[gk >> 1][8 * (gk & 1) + 2 * e],
                                                      s[gk >> 1][8 * (gk & 1) + 2 * e + 1]}, f16x2));
#pragma unroll
        for (int d = 0; d < 4; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, vf[d]),
                                                        __builtin_bit_cast(f16x8, part), o[d], 0, 0, 0);
      } else {
        __builtin_amdgcn_sched_barrier(0);  // (one group's operands at a time: registers)
        const float vsc = scale_at(vsh, min(k0 + 16 * gk, len - 1) >> a.block_shift);
        u32x4 part[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t first, second;
          two_parts(s[gk >> 1][8 * (gk & 1) + 2 * e] * vsc, s[gk >> 1][8 * (gk & 1) + 2 * e + 1] * vsc, first, second);
          part[0][e] = first;
          part[1][e] = second;
        }
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int d = 0; d < 4; ++d)
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vf[d]),
                                                           __builtin_bit_cast(bf16x8, part[y]), o[d], 0, 0, 0);
      }
    }
  };

  // Whether f16 holds this workgroup's values: blocks of scales that are powers of two and near one another (those
  // at the smallest, 2^-126, are zeros beside any other).
  if (threadIdx.x < 3) vexp[threadIdx.x] = threadIdx.x == 0 ? 1 : threadIdx.x == 1 ? 255 : 0;
  __syncthreads();
  for (int i = 4 * i0 + threadIdx.x; i < 4 * i1; i += 256) {
    const uint32_t v = __float_as_uint(vsh[min(seen.at(i >> 2) * kTile + 16 * (i & 3), len - 1) >> a.block_shift]);
    const int e = static_cast<int>(v >> 23);
    if (v > 0x00800000u) {
      atomicMax(&vexp[0], e);
      atomicMin(&vexp[1], e);
      if (v & 0x807fffffu) vexp[2] = 1;
    }
  }
  __syncthreads();
  const int vtop = vexp[0];
  const bool fits = !vexp[2] && vtop < 255 && vtop - vexp[1] <= kSpread;  // the same for all
  auto walk = [&](auto f16) __attribute__((always_inline)) {
    // The factor of the wave's value blocks: a group of 16 keys a half wave.
    auto factor = [&](int tile) __attribute__((always_inline)) {
      const uint32_t v = __float_as_uint(vsh[min(tile * kTile + 16 * vgk, len - 1) >> a.block_shift]);
      return __uint_as_float(static_cast<uint32_t>(max(static_cast<int>(v >> 23) - vtop + 127 + kRaise, 1)) << 23);
    };
    float next = 1.f;
    fetch(seen.at(i0));
    if constexpr (decltype(f16)::value) next = factor(seen.at(i0));
    place(f16, next, 0);
    for (int i = i0; i < i1; ++i) {
      const int buf = (i - i0) & 1;
      // Tile i is in buf, and every wave is past tile i - 1 in the other one.
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 4; ++q) kf[q] = kn[q];
      if (i + 1 < i1) {
        fetch(seen.at(i + 1));
        if constexpr (decltype(f16)::value) next = factor(seen.at(i + 1));
      }
      compute(f16, seen.at(i), buf);
      if (i + 1 < i1) place(f16, next, buf ^ 1);
    }
  };
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    m = -INFINITY;
    l = 0.f;
  };
  clear();
  float back = 1.f;  // what the values' sums are multiplied with in the end
  if (i0 < i1) {     // workgroup-uniform
    bool exact = fits;
    if (fits) {
      walk(std::true_type{});
      back = __builtin_ldexpf(1.f, vtop - 127 - kRaise);
      // NaN anywhere: a value may have reached rows that do not see it.
      bool odd = false;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd |= o[d][r] != o[d][r];
      exact = !__syncthreads_or(odd);
    }
    if (!exact) {
      clear();
      back = 1.f;
      walk(std::false_type{});
    }
  }

  {
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(w[0]) + __uint_as_float(w[1]);
  }
  if (row >= R) return;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = (odd >> (16 * d + r)) & 1 ? __builtin_nanf("") : o[d][r] * back;
  if (a.splits == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // (nothing seen: zeros)
    uint16_t* dst = a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H * G + h * G + g) * kD + 4 * half;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<u32x2*>(dst + 32 * d + 8 * r) = {skv::f2bf2(o[d][4 * r] * inv, o[d][4 * r + 1] * inv),
                                                           skv::f2bf2(o[d][4 * r + 2] * inv, o[d][4 * r + 3] * inv)};
    return;
  }
  const int64_t at = (static_cast<int64_t>(bh) * R + row) * a.splits + split;
  if (half == 0) {
    a.ws_ml[2 * at] = m;
    a.ws_ml[2 * at + 1] = l;
  }
  float* dst = a.ws_o + at * kD + 4 * half;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * r) =
          f32x4{o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]};
}

__global__ void __launch_bounds__(256) rows_join_kernel(Args a) {
  __shared__ f32x4 acc_lds[8][32];
  const int R = a.T * a.G, bh = blockIdx.x / R, row = blockIdx.x - bh * R;
  const int b = bh / a.H, h = bh - b * a.H, t = row / a.G, g = row - t * a.G;
  join_parts(a.ws_o, a.ws_ml, static_cast<int64_t>(blockIdx.x) * a.splits, 1, a.splits,
             a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H * a.G + h * a.G + g) * kD, acc_lds);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// How a call is cut up, from its sizes alone (the lengths are on the device).
struct Plan {
  bool token;
  int64_t grid;
  int splits, rtiles;
  int64_t parts;  // partial rows of 128 + 2 floats
};

Plan plan_of(int B, int H, int G, int T, int cap, int window, int sinks) {
  Plan p{};
  p.token = T == 1 && G <= 16;
  // groups that a query can see: both ends of a window may lie inside one
  const int64_t keys = window ? std::min<int64_t>(cap, static_cast<int64_t>(window) + T - 1 + sinks) : cap;
  if (p.token) {
    const int64_t groups = std::min<int64_t>((static_cast<int64_t>(cap) + kGroup - 1) / kGroup,
                                             (keys + kGroup - 1) / kGroup + 2);
    const int64_t each = (groups + kMinGroups - 1) / kMinGroups;
    const int64_t slots = std::min<int64_t>(B * each, (kTarget + H - 1) / H + B);
    p.grid = slots * H;
    p.parts = p.grid * G;
    p.splits = 1;
    return p;
  }
  const int64_t R = static_cast<int64_t>(T) * G;
  p.rtiles = static_cast<int>((R + kRowsTile - 1) / kRowsTile);
  const int64_t wgs = static_cast<int64_t>(B) * H * p.rtiles;
  const int64_t tiles = (keys + kTile - 1) / kTile;
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((512 + wgs - 1) / wgs, tiles / 4)));
  p.grid = wgs * p.splits;
  p.parts = p.splits > 1 ? static_cast<int64_t>(B) * H * R * p.splits : 0;
  return p;
}

bool sizes_ok(int B, int H, int Hq, int T, int cap, int window, int sinks) {
  return B >= 1 && H >= 1 && Hq >= H && Hq % H == 0 && T >= 1 && cap >= 1 && window >= 0 && sinks >= 0 &&
         static_cast<int64_t>(B) * Hq * T < (int64_t{1} << 30) && cap <= (1 << 30);
}

}  // namespace

extern "C" int64_t skv_kv8_attn_workspace_bytes(int batch_size, int q_heads, int kv_heads, int rows, int cap,
                                                int window, int sinks) {
  if (!sizes_ok(batch_size, kv_heads, q_heads, rows, cap, window, sinks)) return 0;
  return plan_of(batch_size, kv_heads, q_heads / kv_heads, rows, cap, window, sinks).parts * (kD + 2) * 4;
}

extern "C" int skv_kv8_attn(const uint16_t* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
                            const uint8_t* k8, const uint8_t* v8, int64_t c_stride_b, int64_t c_stride_h,
                            int64_t c_stride_s, const float* k_scale, const float* v_scale, int64_t s_stride_b,
                            int64_t s_stride_h, const int32_t* lengths, const int32_t* counts, int batch_size,
                            int q_heads, int kv_heads, int rows, int cap, int block, float scale, int window, int sinks,
                            uint16_t* out, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "kv8_attn";
  if (!q || !k8 || !v8 || !k_scale || !v_scale || !lengths || !out) {
    skv_set_error("%s: null pointer", what);
    return SKV_EINVAL;
  }
  if (!sizes_ok(batch_size, kv_heads, q_heads, rows, cap, window, sinks)) {
    skv_set_error("%s: batch=%d q_heads=%d kv_heads=%d rows=%d cap=%d window=%d sinks=%d", what, batch_size, q_heads,
                  kv_heads, rows, cap, window, sinks);
    return SKV_EINVAL;
  }
  if (block != 16 && block != 32 && block != 64 && block != 128) {
    skv_set_error("%s: block=%d (16, 32, 64 or 128 tokens)", what, block);
    return SKV_EUNSUPPORTED;
  }
  if (!aligned(q, 16) || !aligned(k8, 16) || !aligned(v8, 16) || !aligned(out, 16) || !aligned(k_scale, 4) ||
      !aligned(v_scale, 4) || q_stride_b % 8 || q_stride_h % 8 || q_stride_t % 8 || c_stride_b % 16 ||
      c_stride_h % 16 || c_stride_s % 16) {
    skv_set_error("%s: rows of q, of the caches and of out must be 16-byte aligned", what);
    return SKV_EINVAL;
  }
  if (cap == 1) c_stride_s = kD;  // (of no meaning)
  if (c_stride_s < kD || c_stride_s > (1 << 24)) {
    skv_set_error("%s: tokens %lld bytes apart (128 to 2^24)", what, (long long)c_stride_s);
    return SKV_EUNSUPPORTED;
  }
  const Plan p = plan_of(batch_size, kv_heads, q_heads / kv_heads, rows, cap, window, sinks);
  const int64_t need = p.parts * (kD + 2) * 4;
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) {
    skv_set_error("%s: workspace of %lld bytes (%lld needed, 16-byte aligned)", what, (long long)workspace_bytes,
                  (long long)need);
    return SKV_EINVAL;
  }
  if (p.grid > (int64_t{1} << 30)) {
    skv_set_error("%s: batch=%d q_heads=%d rows=%d", what, batch_size, q_heads, rows);
    return SKV_EUNSUPPORTED;
  }
  int shift = 4;
  while ((1 << shift) < block) ++shift;
  float* ws_o = static_cast<float*>(workspace);
  Args a{q, q_stride_b, q_stride_h, q_stride_t, k8, v8, c_stride_b, c_stride_h, c_stride_s, k_scale, v_scale,
         s_stride_b, s_stride_h, lengths, counts, out, ws_o, ws_o ? ws_o + p.parts * kD : nullptr, batch_size,
         kv_heads, q_heads / kv_heads, rows, cap, shift, window ? std::min(window, kNoWindow) : kNoWindow, sinks,
         std::fabs(scale) * 1.44269504088896340736f, scale < 0.f, kTarget, p.splits, p.rtiles};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 g(static_cast<unsigned>(p.grid)), t(256);
  if (p.token) {
    hipLaunchKernelGGL(token_kernel, g, t, 0, s, a);
    hipLaunchKernelGGL(token_join_kernel, dim3(batch_size * q_heads), t, 0, s, a);
  } else {
    hipLaunchKernelGGL(rows_kernel, g, t, 0, s, a);
    if (p.splits > 1) hipLaunchKernelGGL(rows_join_kernel, dim3(batch_size * q_heads * rows), t, 0, s, a);
  }
  return skv_check_launch(what);
}
