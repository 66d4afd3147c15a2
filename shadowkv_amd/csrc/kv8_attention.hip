// Attention over an 8-bit KV cache (the format of kv8.hip): the new tokens of each sequence, its last ones, over
// the cached keys and values that they see.
//
//   out[b, t, hq] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b, hq, t] . k_j),  k_j = ks * code, v_j = vs * code
//
// over the keys j <= p of the query's position p = length_b - n_b + t, with a window w only those with j > p - w
// or j < sinks. A query that sees nothing (p < 0), or is padding (t >= n_b), gets zeros. Codes become bf16 (exactly) on
// their way into the matrix cores; a key block's scale multiplies its scores and a value block's scale its
// probabilities, so no dequantised row is ever formed. Scores, probabilities and sums are fp32. A probability
// enters the product with the values as two bf16 parts (16 significant bits, an error of 2^-16 where the output's
// one rounding is 2^-8); with many rows, where the matrix cores are the bound, as one f16 (11 bits, 2^-11, and the
// sum that divides the result takes the same rounded ones), wherever f16 holds the values exactly.
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
  int target;   // few rows: workgroups to aim for
  int splits;   // more: shares of a row tile's keys
  int rtiles;   // more: row tiles of a (sequence, kv head)
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
  __device__ __forceinline__ int index(int group) const {  // of the first group at or behind `group`
    return group < first ? group : max(first, group - skip);
  }
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

// Dims 2 y and 2 y + 1 of the same, tokens 2 i and 2 i + 1, as f16 of code * factor (a power of two).
__device__ __forceinline__ void f16_pair(uint32_t even, uint32_t odd, float factor, int y, int i, u32x4& o0,
                                         u32x4& o1) {
  const uint32_t w = __builtin_amdgcn_perm(odd, even, y ? 0x07030602u : 0x05010400u);
  o0[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, factor, false));
  o1[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, factor, true));
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
// Few rows: up to 32 of a kv head's query heads and new tokens together (row t * G + g).
//
// Bound: HBM, 256 bytes a key. The sequences' keys are cut into chunks of equal length, however different the sequences
// are (planned on the device from the lengths, so that a captured call follows them), each a workgroup of four waves
// that take its groups of 32 keys in turn, straight from memory into registers: S^T = K Q^T on v_mfma_f32_16x16x32_bf16
// (a row of the queries a column) leaves a lane with 8 keys' scores of one row, which is the second operand of O^T =
// V^T P^T, whose first is the lane's 8 tokens of one dim: neither probabilities nor values cross lanes. Measured
// (MI355X, 4 query heads on each of 8 kv heads, both launches): 8 sequences of 122880 tokens 306 us, 6.6 TB/s; 24
// windows of 8192 keys and 64 sinks 74 us, 5.3 TB/s; 5 tokens each of 4 sequences of up to 30011 41 us, 3.8 TB/s (two
// tiles of rows leave two waves a SIMD to hide the loads' latency).
constexpr int kGroup = 32;
constexpr int kGroupShift = 5;
constexpr int kMinGroups = 8;   // a chunk's groups of 32 keys, at least
// Chunks to aim for: four workgroups to a CU, twice that for up to 8 rows, whose partial results cost little (24
// windows of 8256 keys, 4 rows: 80 -> 73 us; 16 rows, 4 sequences of 262143: 99 -> 111).
constexpr int target_chunks(int64_t rows) { return rows <= 8 ? 2048 : 1024; }
constexpr int kOutLd = kD + 4;
// Groups that a sequence's rows can see (by the capacity and the window) up to which one workgroup of 16 waves (8 for
// two tiles of rows) takes them all, in one launch, rather than chunks and a join: a window of 1024 keys with sinks,
// its ends inside a group, or twice that where the sequences fill half of the chip (MI355X, us in a graph, 4 query
// heads on each of 8 kv heads, chunks / whole: 1 sequence of 512 keys 10.0 / 7.6, 1024 9.9 / 10.1 and a launch less
// from the host, 2048 10.0 / 15.8; 24 sequences of 1024 16.4 / 11.8, 2048 26.1 / 20.2).
constexpr int whole_groups(int tiles, int64_t rows_of_kv) { return (rows_of_kv >= 128 ? 72 : 36) / tiles; }

struct Chunk {
  int b, index, groups;  // sequence, which of its chunks, groups of a chunk
};

__device__ __forceinline__ Groups few_groups(const Args& a, int b) {
  const int len = length_of(a, b), n = count_of(a, b);
  return groups_seen(len - n, n ? len - 1 : -1, a.window, a.sinks, kGroupShift);
}

// The chunk length, wave-uniform: the sequences' groups dealt over the workgroups to aim for.
__device__ __forceinline__ int chunk_groups(const Args& a, int lane) {
  int64_t total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int t = b0 + lane < a.B ? few_groups(a, b0 + lane).total : 0;
    total += skv::wave_total(t);  // (64 sequences of 2^30 tokens have 2^31 groups)
  }
  return static_cast<int>(min(max(static_cast<int64_t>(kMinGroups), (total * a.H + a.target - 1) / a.target),
                              static_cast<int64_t>(1 << 30)));
}

// Chunk i of all sequences' (false past the last).
__device__ __forceinline__ bool find_chunk(const Args& a, int i, int lane, Chunk& c) {
  c.groups = chunk_groups(a, lane);
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int n = b0 + lane < a.B ? (few_groups(a, b0 + lane).total + c.groups - 1) / c.groups : 0;
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

// 0x80 in each byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// kTiles: of 16 rows. kWhole: a workgroup of more waves takes all that a sequence's rows see, and writes its result.
constexpr int few_threads(int tiles, bool whole) { return 64 * (whole ? 16 / tiles : 4); }

template <int kTiles, bool kWhole>
__global__ void __launch_bounds__(few_threads(kTiles, kWhole), kTiles == 1 ? 4 : 2) few_kernel(Args a) {
  constexpr int kWaves = few_threads(kTiles, kWhole) / 64;
  __shared__ float o_lds[kWaves][16][kOutLd];
  __shared__ float m_lds[kWaves][16], l_lds[kWaves][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = blockIdx.x / a.H, h = blockIdx.x - slot * a.H;
  Chunk c{slot, 0, 1 << 30};
  if (!kWhole && !find_chunk(a, slot, lane, c)) return;  // workgroup-uniform
  const int b = c.b, G = a.G, R = G * a.T;
  const int len = length_of(a, b), n = count_of(a, b);
  const int pmin = len - n, pmax = len - 1;
  const Groups seen = few_groups(a, b);
  const int i0 = kWhole ? 0 : c.index * c.groups, i1 = kWhole ? seen.total : min(i0 + c.groups, seen.total);
  const int li = lane & 15, grp = lane >> 4;

  // Q as the B operand: lane (li, grp) holds row li of a tile, in step s dims 64 (s / 2) + 16 grp + 8 (s % 2) and on.
  // Rows past the last, and of padding, ride along with the last query (padding's own memory, which may hold anything,
  // is not read), and give nothing in the end.
  bf16x8 qf[kTiles][4];
  int p[kTiles];
#pragma unroll
  for (int y = 0; y < kTiles; ++y) {
    const int row = min(16 * y + li, R - 1), t = row / G;
    p[y] = t < n ? pmin + t : pmax;
    const uint16_t* q = a.q + b * a.q_sb + (h * G + row - t * G) * a.q_sh + min(t, max(n - 1, 0)) * a.q_st + 16 * grp;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      qf[y][s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(q + 64 * (s >> 1) + 8 * (s & 1)) ^
                                                (a.negative ? 0x80008000u : 0u));
  }
  const uint8_t* kh = a.k8 + b * a.c_sb + h * a.c_sh + 16 * grp;
  const uint8_t* vh = a.v8 + b * a.c_sb + h * a.c_sh + 8 * li;
  const float* ksh = a.ks + b * a.s_sb + h * a.s_sh;
  const float* vsh = a.vs + b * a.s_sb + h * a.s_sh;

  f32x4 o[kTiles][8];
  float m[kTiles], l[kTiles];  // the row's reference, in units of log2; this lane's share of its sum
#pragma unroll
  for (int y = 0; y < kTiles; ++y) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[y][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[y] = -INFINITY;
    l[y] = 0.f;
  }

  u32x4 kr[2][2];
  u32x2 vr[8];
  float kc[2], vc[2];
  auto load_keys = [&](int i, u32x4 (&k)[2][2], float (&c)[2]) __attribute__((always_inline)) {
    const int j0 = seen.at(i) * kGroup;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t* row = kh + static_cast<int64_t>(min(j0 + 16 * u + li, pmax)) * a.c_ss;
      k[u][0] = *reinterpret_cast<const u32x4*>(row);
      k[u][1] = *reinterpret_cast<const u32x4*>(row + 64);
      c[u] = ksh[min(j0 + 16 * u, pmax) >> a.block_shift];
    }
  };
  auto load_values = [&](int i) __attribute__((always_inline)) {
    const int j0 = seen.at(i) * kGroup;
#pragma unroll
    for (int u = 0; u < 2; ++u) vc[u] = vsh[min(j0 + 16 * u, pmax) >> a.block_shift];
    // (values, whole rows of each line a load, with the streaming hint: 8 sequences of 122880 tokens 340 -> 317 us;
    // keys, half of a line a load, gain nothing from it)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        vr[4 * u + r] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(
            vh + static_cast<int64_t>(min(j0 + 16 * u + 4 * grp + r, pmax)) * a.c_ss));
  };

  // With two tiles of rows there are but two waves a SIMD, and registers for the next group's keys (5 drafted tokens of
  // 4 sequences: 43 -> 41 us; its values too: 44).
  constexpr bool kAhead = kTiles == 2;
  u32x4 kn[2][2];
  float kcn[2];
  if (kAhead && i0 + wave < i1) load_keys(i0 + wave, kn, kcn);
  for (int i = i0 + wave; i < i1; i += kWaves) {
    if constexpr (kAhead) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        kr[u][0] = kn[u][0];
        kr[u][1] = kn[u][1];
        kc[u] = kcn[u];
      }
    } else load_keys(i, kr, kc);
    load_values(i);
    if (kAhead) load_keys(min(i + kWaves, i1 - 1), kn, kcn);
    const int j0 = seen.at(i) * kGroup;
    f32x4 s[kTiles][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float f = key_factor(kc[u], a.scale_log2e);
#pragma unroll
      for (int y = 0; y < kTiles; ++y) s[y][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const bf16x8 kf = bf16_of(kr[u][st >> 1][2 * (st & 1)], kr[u][st >> 1][2 * (st & 1) + 1]);
#pragma unroll
        for (int y = 0; y < kTiles; ++y)
          s[y][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[y][st], s[y][u], 0, 0, 0);
      }
#pragma unroll
      for (int y = 0; y < kTiles; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[y][u][r] *= f;
    }
    float vf[kTiles][2];  // the value blocks' factors
#pragma unroll
    for (int y = 0; y < kTiles; ++y)
#pragma unroll
      for (int u = 0; u < 2; ++u) vf[y][u] = vc[u];
    // wave-uniform: a group at an end of what a row sees
    if (j0 + kGroup > pmin + 1 || (j0 <= pmax - a.window && j0 + kGroup > a.sinks)) {
      uint32_t odd = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        bool some[kTiles] = {};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = j0 + 16 * u + 4 * grp + r;
#pragma unroll
          for (int y = 0; y < kTiles; ++y) {
            const bool yes = sees(p[y], j, a.window, a.sinks);
            s[y][u][r] = yes ? s[y][u][r] : -INFINITY;
            some[y] |= yes;
          }
          // a value that no row sees may be anything: zero codes
          u32x2& w = vr[4 * u + r];
          if (!(j <= pmax && (j > pmin - a.window || j < a.sinks))) w = u32x2{0u, 0u};
          odd |= nan_bytes(w[0]) | nan_bytes(w[1]);
        }
#pragma unroll
        for (int y = 0; y < kTiles; ++y) vf[y][u] = some[y] ? vf[y][u] : 0.f;  // (so may its scale)
      }
      if (n > 1 && __any(odd != 0)) {  // wave-uniform
        // A value that is NaN makes the sums of the rows that see its key NaN, and no others (in the product it
        // would: a hidden key's zero times NaN): how many such keys a row sees is a product of its own.
        uint32_t ones[2][8];
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t f = nan_bytes(vr[t][x]) >> 7;
            ones[x][t] = f * 0x38u;  // 1
            vr[t][x] &= ~(f * 0xffu);
          }
#pragma unroll
        for (int y = 0; y < kTiles; ++y) {
          u32x4 vis;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + 16 * (e >> 1) + 4 * grp + 2 * (e & 1);
            vis[e] = (sees(p[y], j, a.window, a.sinks) ? 0x3f80u : 0u) |
                     (sees(p[y], j + 1, a.window, a.sinks) ? 0x3f800000u : 0u);
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            u32x4 is[4];
            transpose_bf16(ones[x], is);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f32x4 count = {0.f, 0.f, 0.f, 0.f};
              count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, is[e]),
                                                              __builtin_bit_cast(bf16x8, vis), count, 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (count[r] > 0.f) o[y][4 * x + e][r] = __builtin_nanf("");
            }
          }
        }
      }
    }
    u32x4 part[kTiles][2];
#pragma unroll
    for (int y = 0; y < kTiles; ++y) {
      float mx = fmaxf(fmaxf(fmaxf(s[y][0][0], s[y][0][1]), fmaxf(s[y][0][2], s[y][0][3])),
                       fmaxf(fmaxf(s[y][1][0], s[y][1][1]), fmaxf(s[y][1][2], s[y][1][3])));
      mx = max_of_rows(mx);
      if (__any(mx > m[y])) {  // wave-uniform
        const float mn = fmaxf(m[y], mx);
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[y] - mn);
        m[y] = mn;
        l[y] *= f;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[y][e] *= f;
      }
      const float ref = m[y] == -INFINITY ? 0.f : m[y];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const float p0 = __builtin_amdgcn_exp2f(s[y][u][r] - ref);
          const float p1 = __builtin_amdgcn_exp2f(s[y][u][r + 1] - ref);
          l[y] += p0 + p1;
          uint32_t first, second;
          two_parts(p0 * vf[y][u], p1 * vf[y][u], first, second);
          part[y][0][2 * u + r / 2] = first;
          part[y][1][2 * u + r / 2] = second;
        }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t w[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) w[t] = vr[t][half];
      u32x4 vt[4];
      transpose_bf16(w, vt);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < kTiles; ++y)
            o[y][4 * half + e] =
                __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vt[e]),
                                                        __builtin_bit_cast(bf16x8, part[y][x]), o[y][4 * half + e], 0,
                                                        0, 0);
    }
  }

  // The waves' parts: lane (li, grp) holds row li's dims 8 (4 grp + r) + e.
  const int64_t row0 = (static_cast<int64_t>(slot) * a.H + h) * R;
#pragma unroll
  for (int y = 0; y < kTiles; ++y) {
    const float ls = sum_of_rows(l[y]);
    const int rows = min(16, R - 16 * y);
    if (y) __syncthreads();
    if (grp == 0) {
      m_lds[wave][li] = m[y];
      l_lds[wave][li] = ls;
    }
    if (li < rows) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<f32x4*>(&o_lds[wave][li][8 * (4 * grp + r) + e]) =
              f32x4{o[y][e][r], o[y][e + 1][r], o[y][e + 2][r], o[y][e + 3][r]};
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * 32; i += 64 * kWaves) {
      const int g = i >> 5, d = 4 * (i & 31), row = 16 * y + g;
      const bool query = row / G < n && pmin + row / G >= 0;  // (else padding, or it sees nothing: zeros)
      float top = m_lds[0][g];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_lds[w][g]);
      const float ref = top == -INFINITY ? 0.f : top;
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float lsum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(m_lds[w][g] - ref);
        lsum += f * l_lds[w][g];
        sum += f * *reinterpret_cast<const f32x4*>(&o_lds[w][g][d]);
      }
      if constexpr (kWhole) {
        const float inv = 1.f / lsum;
        const u32x2 out = {skv::f2bf2(sum[0] * inv, sum[1] * inv), skv::f2bf2(sum[2] * inv, sum[3] * inv)};
        const int t = row / G;
        const int64_t at = (static_cast<int64_t>(b) * a.T + t) * a.H * G + h * G + row - t * G;
        *reinterpret_cast<u32x2*>(a.out + at * kD + d) = query ? out : u32x2{0u, 0u};
        continue;
      }
      *reinterpret_cast<f32x4*>(a.ws_o + (row0 + row) * kD + d) = query ? sum : f32x4{0.f, 0.f, 0.f, 0.f};
      if (d == 0) {
        a.ws_ml[2 * (row0 + row)] = query ? top : -INFINITY;
        a.ws_ml[2 * (row0 + row) + 1] = query ? lsum : 0.f;
      }
    }
  }
}

// Joins n partial results (m, l, o), part i at index first + i * stride, into the row of sequence b's query t: 256
// threads, 32 lanes of four dims by 8 parts at a time. Every wave of it sees the same maximum and sum.
__device__ __forceinline__ void join_parts(const Args& a, int b, int t, int64_t first, int64_t stride, int n,
                                           uint16_t* out, f32x4 (&acc_lds)[8][32]) {
  const float* ws_o = a.ws_o;
  const float* ws_ml = a.ws_ml;
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
    const int count = count_of(a, b);
    const bool query = t < count && length_of(a, b) - count + t >= 0;  // (else padding, or it sees nothing: zeros)
    const float inv = 1.f / l;
    const u32x2 row = {skv::f2bf2(acc[0] * inv, acc[1] * inv), skv::f2bf2(acc[2] * inv, acc[3] * inv)};
    *reinterpret_cast<u32x2*>(out + 4 * d) = query ? row : u32x2{0u, 0u};
  }
}

__global__ void __launch_bounds__(256) few_join_kernel(Args a) {
  __shared__ f32x4 acc_lds[8][32];
  const int lane = threadIdx.x & 63;
  const int Hq = a.H * a.G, bt = blockIdx.x / Hq, hq = blockIdx.x - bt * Hq;
  const int b = bt / a.T, t = bt - b * a.T, h = hq / a.G, g = hq - h * a.G;
  const int each = chunk_groups(a, lane);
  int before = 0;
  for (int b0 = 0; b0 < b; b0 += 64) {
    const int n = b0 + lane < b ? (few_groups(a, b0 + lane).total + each - 1) / each : 0;
    before += __builtin_amdgcn_readlane(skv::wave_inclusive_scan(n), 63);
  }
  const int n = (few_groups(a, b).total + each - 1) / each;
  const int64_t R = static_cast<int64_t>(a.T) * a.G;
  join_parts(a, b, t, (static_cast<int64_t>(before) * a.H + h) * R + t * a.G + g, a.H * R, n,
             a.out + static_cast<int64_t>(blockIdx.x) * kD, acc_lds);
}

// ------------------------------------------------------------------------------------------------
// More rows.
//
// Bound: the matrix cores (with few rows, HBM). The rows of a kv head are its queries' heads together, row t * G + g,
// so that a tile of keys serves all of them. A workgroup of four waves (eight) owns 128 (256) rows, 32 a wave, a row a
// lane, and walks the tiles of 64 keys that any of them sees, or a share of them where there are too few rows to fill
// the chip. Keys and values are read once a tile, turned into 16 bits (the values transposed) by the threads that read
// them, and shared through LDS, the next tile on its way meanwhile. Measured (MI355X): 8192 causal tokens of 32 heads
// over 8, 547 us, 1.00 PFLOP/s where a large bf16 GEMM has 1.22 (533 to 557 from machine to machine), 1003 us where the
// values take the form in 16 bits; 2048 tokens behind up to 31285 others, 16 heads on each of 2 kv heads, a window of
// 8192, two sequences, 532 us, 0.91 PFLOP/s. Counters (the prompt): the matrix cores are busy in 46% of the cycles, the
// vector units in 47%, LDS in 32%, at a clock of 1.9 of 2.4 GHz: the power is the limit, and vector work that hides
// behind the matrix instructions only in part.
constexpr int kTile = 64;
constexpr int kTileShift = 6;
constexpr int kRowsWave = 32;

// 16-byte chunk c (8 dims) of key row r of a tile in LDS, and chunk (group of 16 keys, half of its order, dim).
__device__ __forceinline__ int k_at(int r, int c) { return r * 16 + (c ^ (r & 15)); }
__device__ __forceinline__ int v_at(int gk, int half, int d) { return gk * 256 + half * 128 + (d ^ ((d >> 3) & 7)); }

// The largest of eight, four instructions (fmaxf would first quiet each operand that comes from a matrix instruction).
// Not right behind the one that makes them: the compiler does not see what this waits for.
__device__ __forceinline__ float max8(const f32x16& v, int r) {
  float o;
  asm("v_max3_f32 %0, %1, %2, %3\n\tv_max3_f32 %0, %0, %4, %5\n\tv_max3_f32 %0, %0, %6, %7\n\tv_max_f32 %0, %0, %8"
      : "=&v"(o)
      : "v"(v[r]), "v"(v[r + 1]), "v"(v[r + 2]), "v"(v[r + 3]), "v"(v[r + 4]), "v"(v[r + 5]), "v"(v[r + 6]),
        "v"(v[r + 7]));
  return o;
}

// A barrier for what goes through LDS: loads from memory stay on their way.
__device__ __forceinline__ void barrier_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Powers of two by which the value blocks of a workgroup may differ for f16 to hold their values exactly, and the
// one that the largest block's codes are raised by: 448 * 2^7 is just below f16's largest, 2^-9 * 2^(7 - 12) its
// smallest normal value.
constexpr int kSpread = 12;
constexpr int kRaise = 7;
// A probability is at most 2^(kRaise + kSlack), below f16's largest: kSlack is how far a score may pass the reference.
constexpr float kSlack = 8.f;

// kWaves: 4, two workgroups to a CU, or 8, one.
template <int kWaves>
__global__ void __launch_bounds__(64 * kWaves, 2) rows_kernel(Args a) {
  constexpr int kRowsTile = kWaves * kRowsWave;
  constexpr int kKeyLoads = 8 / kWaves;   // of 16 bytes of a key's row that a thread carries
  constexpr int kValueDims = 16 / kWaves;  // that it carries of the values of 8 tokens
  __shared__ u32x4 kt[2][kTile * 16], vt[2][kTile * 16];
  // Values that are NaN, by (buffer, wave that carries them): whether there are any, and each dim's keys as bits.
  __shared__ int odd_lds[2][kWaves];
  __shared__ uint32_t odd_keys[2][kWaves][kD];
  __shared__ int vexp[3];  // largest and smallest exponent of the value blocks' scales, whether one is no power of two
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int i = blockIdx.x;
  const int BH = a.B * a.H;
  int bh = i % BH;
  i /= BH;
  // Consecutive workgroups go to the XCDs in turn: one (sequence, kv head) stays with its XCDs, whose L2 holds its
  // keys, while the chip takes on one set of workgroups; for the next set the sequences, whose work differs, change
  // places (1024 tokens of each of four sequences of 2000 to 8000: 412 us without, 388 so, 398 at every tile; two
  // pieces of 2048 under a window: 476, 481, 510; sequences of one length lose 1%).
  bh = (bh / a.H + static_cast<int>(static_cast<int64_t>(i) * BH / (2048 / kWaves))) % a.B * a.H + bh % a.H;
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

  // Row li of the wave: query t, head g of the kv head's. Those past the last row, and of padding, ride along with the
  // last query (padding's own memory, which may hold anything, is not read), and give nothing in the end.
  struct Row {
    int row, t, g;
    bool query;
  };
  auto row_of = [&](int li) __attribute__((always_inline)) {
    Row x;
    x.row = r0 + wave * kRowsWave + li;
    x.t = min(x.row, R - 1) / G;
    x.g = min(x.row, R - 1) - x.t * G;
    x.query = x.row < R && x.t < n;
    return x;
  };
  // A wave of rows past the last, or of padding: it carries its share of the tiles, and no more.
  const bool idle = r0 + wave * kRowsWave >= min(R, n * G);
  u32x4 qf[8];
  {
    const Row x = row_of(threadIdx.x & 31);
    const uint16_t* q = a.q + b * a.q_sb + (h * G + x.g) * a.q_sh + min(x.t, max(n - 1, 0)) * a.q_st + 8 * (lane >> 5);
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

  // A thread carries 32 bytes of a key row (of 8 waves 16), and four dims (two) of the values of 8 tokens: half of a
  // group of 16, in the order of the keys in the scores' registers; a group is a wave's (two waves', a half each). Rows
  // behind the sequence's end are out of the buffer's bounds and come as zeros, whatever lies there.
  const int stride = static_cast<int>(a.c_ss);
  struct Lane {
    int li, half, krow, kpart, kmine, vmine, vhalf, vdim;
  };
  const int vgroup = kWaves == 4 ? wave : wave >> 1;
  // (made anew where a walk begins, from a thread id that the compiler takes for another one: what hangs on it would
  // else be held in registers from walk to walk)
  auto own_lane = [&]() __attribute__((always_inline)) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    Lane x;
    x.li = tid & 31;
    x.half = (tid >> 5) & 1;
    x.krow = tid / kWaves;
    x.kpart = tid % kWaves;
    x.kmine = x.krow * stride + 16 * kKeyLoads * x.kpart;
    x.vhalf = kWaves == 4 ? x.half : wave & 1;
    x.vdim = kValueDims * (kWaves == 4 ? x.li : tid & 63);
    x.vmine = (16 * vgroup + 4 * x.vhalf) * stride + x.vdim;
    return x;
  };
  constexpr int kDw3 = 0x00020000;  // buffer resource word 3 (gfx9)
  auto tile_rows = [&](const uint8_t* base, int tile) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(base + static_cast<int64_t>(tile) * kTile * a.c_ss), 0,
        min(len - tile * kTile - 1, kTile - 1) * stride + kD, kDw3);
  };
  u32x4 kheld[kKeyLoads];
  uint32_t vheld[8];
  auto fetch_keys = [&](const Lane& x, __amdgpu_buffer_rsrc_t src) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < kKeyLoads; ++c) kheld[c] = __builtin_amdgcn_raw_buffer_load_b128(src, x.kmine, 16 * c, 0);
  };
  // (a buffer's bounds are checked against the vector offset alone: a row's place in its group goes there wherever the
  // sequence may end inside the tile)
  auto fetch_values = [&](auto whole, const Lane& x, __amdgpu_buffer_rsrc_t src) __attribute__((always_inline)) {
    constexpr bool kCut = !decltype(whole)::value;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = ((e & 3) + 8 * (e >> 2)) * stride;
      const int vector = kCut ? x.vmine + at : x.vmine, scalar = kCut ? 0 : at;
      if constexpr (kWaves == 4) vheld[e] = __builtin_amdgcn_raw_buffer_load_b32(src, vector, scalar, 0);
      else vheld[e] = __builtin_amdgcn_raw_buffer_load_b16(src, vector, scalar, 0);
    }
  };
  auto place_chunk = [&](const Lane& x, int buf, int c) __attribute__((always_inline)) {
    kt[buf][k_at(x.krow, 2 * kKeyLoads * x.kpart + c)] =
        __builtin_bit_cast(u32x4, bf16_of(kheld[c >> 1][2 * (c & 1)], kheld[c >> 1][2 * (c & 1) + 1]));
  };
  auto place_keys = [&](const Lane& x, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 2 * kKeyLoads; ++c) place_chunk(x, buf, c);
  };
  auto put_value = [&](const Lane& x, const u32x4& o, int buf, int e) __attribute__((always_inline)) {
    vt[buf][v_at(vgroup, x.vhalf, x.vdim + e)] = o;
  };
  // The block of a tile's group of 16 keys.
  auto block_of = [&](int tile, int group) __attribute__((always_inline)) {
    return min(tile * kTile + 16 * group, len - 1) >> a.block_shift;
  };
  auto key_scales = [&](int tile, float (&ks)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) ks[q] = scale_at(ksh, block_of(tile, q));
  };

  f32x16 o[4];
  float m, l;
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    m = -INFINITY;
    l = 0.f;
  };
  // S^T of a tile: registers 8 i to 8 i + 7 of s[u] hold 8 of the keys 32 u + 16 i to 32 u + 16 i + 15, a block's.
  auto scores = [&](const Lane& x, int buf, f32x16 (&s)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, kt[buf][k_at(32 * u + x.li, 2 * c + x.half)]), __builtin_bit_cast(bf16x8, qf[c]),
            s[u], 0, 0, 0);
      if (c & 1) __builtin_amdgcn_sched_barrier(0);  // (a few operands at a time: registers)
    }
  };
  auto hide = [&](const Lane& x, int p, int tile, f32x16 (&s)[2]) __attribute__((always_inline)) {
    const int first = tile * kTile + 4 * x.half;  // key c of the lane: first + c
    const int last = p - first, behind = p - a.window - first, sink = a.sinks - first;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int c = 32 * u + 8 * (r / 4) + (r % 4);
        s[u][r] = (c <= last) & ((c > behind) | (c < sink)) ? s[u][r] : -INFINITY;
      }
  };
  auto largest_half = [&](float mx) __attribute__((always_inline)) {  // with the row's other lane
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
  };
  auto largest = [&](const f32x16 (&s)[2]) __attribute__((always_inline)) {
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[u][r]);
    return largest_half(mx);
  };
  // The reference moves only when a score passes it by 2^kSlack: the ratio of the sums does not depend on it.
  auto refer = [&](float mx) __attribute__((always_inline)) {
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
    return (m == -INFINITY ? 0.f : m) - static_cast<float>(kRaise);
  };

  // Whether f16 holds this workgroup's values: blocks of scales that are powers of two and near one another (those
  // at the smallest, 2^-126, are zeros beside any other).
  if (threadIdx.x < 3) vexp[threadIdx.x] = threadIdx.x == 0 ? 1 : threadIdx.x == 1 ? 255 : 0;
  __syncthreads();
  for (int i = 4 * i0 + threadIdx.x; i < 4 * i1; i += 64 * kWaves) {
    const uint32_t v = __float_as_uint(vsh[block_of(seen.at(i >> 2), i & 3)]);
    const int e = static_cast<int>(v >> 23);
    if (v > 0x00800000u) {
      atomicMax(&vexp[0], e);
      atomicMin(&vexp[1], e);
      if (v & 0x807fffffu) vexp[2] = 1;
    }
  }
  __syncthreads();
  const int vtop = __builtin_amdgcn_readfirstlane(vexp[0]);
  const bool fits = !__builtin_amdgcn_readfirstlane(vexp[2]) && vtop < 255 &&
                    vtop - __builtin_amdgcn_readfirstlane(vexp[1]) <= kSpread;  // the same for all

  // A value block's factor on its way to f16.
  auto value_factor = [&](float scale) __attribute__((always_inline)) {
    const uint32_t v = __float_as_uint(scale);
    return __uint_as_float(static_cast<uint32_t>(max(static_cast<int>(v >> 23) - vtop + 127 + kRaise, 1)) << 23);
  };

  // Part y of the values, in f16: two tokens' pairs of two dims.
  auto place_pairs = [&](const Lane& x, int buf, int y, float factor, u32x4 (&o)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 2 * (y & 1); e < 2 * (y & 1) + 2; ++e)
      f16_pair(vheld[2 * e], vheld[2 * e + 1], factor, y >> 1, e, o[0], o[1]);
    if (y & 1)
#pragma unroll
      for (int z = 0; z < 2; ++z) put_value(x, o[z], buf, 2 * (y >> 1) + z);
  };
  auto place_f16 = [&](const Lane& x, int tile, int buf) __attribute__((always_inline)) {
    u32x4 o[2];
    const float factor = value_factor(scale_at(vsh, block_of(tile, vgroup)));
#pragma unroll
    for (int y = 0; y < kValueDims; ++y) place_pairs(x, buf, y, factor, o);
  };

  // Tiles that every row sees whole, values and probabilities in f16, one product. Tile i's probabilities and their
  // product are taken while tile i + 1's scores are, tile i + 2's keys and i + 1's values go to LDS and the next ones
  // are on their way: one barrier a tile, and vector work beside every matrix instruction. The order is written down
  // slice by slice (a scheduler of its own would read all operands first, and spill).
  auto walk_whole = [&](int from, int to) __attribute__((always_inline)) {
    __syncthreads();  // every wave is past the tiles before these
    const Lane g = own_lane();
    int kbase = k_at(g.li, g.half);
    const int end = to - 1;  // (tiles one behind the other, none cut off by the sequence's end)
    const uint64_t tile_bytes = static_cast<uint64_t>(kTile) * stride;
    auto whole_rows = [&](const uint8_t* base, int tile) __attribute__((always_inline)) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base + min(tile, end) * tile_bytes), 0,
                                               (kTile - 1) * stride + kD, kDw3);
    };
    // The factors of a tile's groups of 16 keys in a lane each: the keys' in lanes 0 to 3, the values' in 4 to 7. Of
    // tiles i and i + 1, and the scales of i + 2.
    float factors[2], scales;
    const float* own_scales = g.li & 4 ? vsh : ksh;
    auto fetch_scales = [&](int tile) __attribute__((always_inline)) {
      return own_scales[(min(tile, end) * kTile + 16 * (g.li & 3)) >> a.block_shift];
    };
    auto factors_of = [&](float scale) __attribute__((always_inline)) {
      const float k = key_factor(scale, a.scale_log2e), v = value_factor(scale);
      return g.li & 4 ? v : k;
    };
    auto lane_factor = [&](float held, int which) __attribute__((always_inline)) {
      return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(held), which));
    };
    auto next_factors = [&](int i) __attribute__((always_inline)) {
      factors[0] = factors[1];
      factors[1] = factors_of(scales);
      scales = fetch_scales(i + 3);
    };
    // One tile: its scores in s, the next one's into sn (past the last, the last one's again). Keys i are in kt[par],
    // values in vt[par]. 32 slices of a matrix instruction each (16 of the next scores, 16 of this product), its
    // operand read from LDS three slices before.
    auto step = [&](auto par_, int i, f32x16 (&s)[2], f32x16 (&sn)[2]) __attribute__((always_inline)) {
      constexpr int par = decltype(par_)::value;
      // Every wave is past tile i - 1's values and tile i's keys; tile i's values and tile i + 1's keys are in place.
      barrier_lds();
      asm volatile("" : "+v"(kbase));  // (its eight forms are made anew each time: registers)
      u32x4 f[4];
      auto operand = [&](int j) __attribute__((always_inline)) {
        if (j < 16) f[j & 3] = kt[par ^ 1][512 * (j & 1) + (kbase ^ (j & 14))];  // k_at(32 u + li, 2 c + half)
        else f[j & 3] = vt[par][v_at((j - 16) >> 2, g.half, 32 * (j & 3) + g.li)];
      };
#pragma unroll
      for (int j = 0; j < 3; ++j) operand(j);
      float kf[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) kf[q] = lane_factor(factors[0], q);
      const float factor = lane_factor(factors[1], 4 + vgroup);
      float mx = -INFINITY, ref = 0.f;
      auto largest_of = [&](int q) __attribute__((always_inline)) {
        mx = fmaxf(mx, max8(s[q >> 1], 8 * (q & 1)) * kf[q]);
      };
      u32x4 part[4];
      auto probabilities = [&](int gk, int e) __attribute__((always_inline)) {
        const float x0 = __builtin_amdgcn_exp2f(fmaf(s[gk >> 1][8 * (gk & 1) + 2 * e], kf[gk], -ref));
        const float x1 = __builtin_amdgcn_exp2f(fmaf(s[gk >> 1][8 * (gk & 1) + 2 * e + 1], kf[gk], -ref));
        const f16x2 x = __builtin_convertvector(f32x2{x0, x1}, f16x2);
        l = __builtin_amdgcn_fdot2(x, f16x2{1, 1}, l, false);  // (the sum of what the product takes)
        part[gk][e] = __builtin_bit_cast(uint32_t, x);
      };
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) sn[u][r] = 0.f;
      u32x4 x[2];
      largest_of(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        if (j < 29) operand(j + 3);
        if (j < 16)
          sn[j & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[j & 3]),
                                                              __builtin_bit_cast(bf16x8, qf[j >> 1]), sn[j & 1], 0, 0,
                                                              0);
        else
          o[j & 3] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, f[j & 3]),
                                                            __builtin_bit_cast(f16x8, part[(j - 16) >> 2]), o[j & 3], 0,
                                                            0, 0);
        asm volatile("s_nop 0");  // (a slot for the SIMD's other wave: 544 -> 540 us; two: 545)
        // (vector work, evenly: the maximum and the reference, 16 pairs of probabilities, each before the product that
        // takes it, and between those the tiles on their way)
        constexpr int kPair[32] = {-1, -1, -1, -1, 0, 1, -1, 2, 3, -1, 4, 5, -1, 6, 7, -1,
                                   8, 9, -1, 10, 11, -1, 12, 13, -1, 14, 15, -1, -1, -1, -1, -1};
        if (j < 3) largest_of(j + 1);
        else if (j == 3) ref = refer(largest_half(mx));
        else if (kPair[j] >= 0) probabilities(kPair[j] >> 2, kPair[j] & 3);
        else if (j <= 15 && j % 3 == 0 && j / 3 - 2 < 2 * kKeyLoads) place_chunk(g, par, j / 3 - 2);
        else if (j == 18) fetch_keys(g, whole_rows(kh, i + 3));
        else if (j == 21 || j == 24) place_pairs(g, par ^ 1, j / 3 - 7, factor, x);
        else if ((j == 27 || j == 28) && kValueDims == 4) place_pairs(g, par ^ 1, j - 25, factor, x);
        else if (j == 29) fetch_values(std::true_type{}, g, whole_rows(vh, i + 2));
        else if (j == 30) next_factors(i);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    fetch_keys(g, whole_rows(kh, from));
    fetch_values(std::true_type{}, g, whole_rows(vh, from));
    place_keys(g, 0);
    place_f16(g, from, 0);
    __builtin_amdgcn_sched_barrier(0);
    fetch_keys(g, whole_rows(kh, from + 1));
    place_keys(g, 1);
    __builtin_amdgcn_sched_barrier(0);
    fetch_keys(g, whole_rows(kh, from + 2));
    fetch_values(std::true_type{}, g, whole_rows(vh, from + 1));
    __syncthreads();
    factors[0] = factors_of(fetch_scales(from));
    factors[1] = factors_of(fetch_scales(from + 1));
    scales = fetch_scales(from + 2);
    if (idle) {  // wave-uniform
      for (int i = from; i <= end; ++i) {
        barrier_lds();
        const int par = (i - from) & 1;
        const float factor = lane_factor(factors[1], 4 + vgroup);
        u32x4 x[2];
#pragma unroll
        for (int c = 0; c < 2 * kKeyLoads; ++c) place_chunk(g, par, c);
#pragma unroll
        for (int y = 0; y < kValueDims; ++y) place_pairs(g, par ^ 1, y, factor, x);
        fetch_keys(g, whole_rows(kh, i + 3));
        fetch_values(std::true_type{}, g, whole_rows(vh, i + 2));
        next_factors(i);
      }
      return;
    }
    f32x16 sa[2], sb[2];
    scores(g, 0, sa);
    asm volatile("s_nop 15\n\ts_nop 7" : "+v"(sa[0]), "+v"(sa[1]));  // (their first reader is max8's asm)
    for (int i = from;;) {
      step(std::integral_constant<int, 0>{}, i, sa, sb);
      if (++i > end) break;
      step(std::integral_constant<int, 1>{}, i, sb, sa);
      if (++i > end) break;
    }
  };

  // Any tiles, one after the other: f16 as above, or for any values bf16, two parts of a probability times its block's
  // scale, and NaN kept to the rows that see them.
  uint64_t odd = 0;  // this lane's output dims that a value seen by its row makes NaN, bit 16 d + r
  auto place_any = [&](const Lane& x, int buf) __attribute__((always_inline)) {
    uint32_t some = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) some |= nan_bytes(vheld[e]);
    const bool any = __any(some != 0);
    if (lane == 0) odd_lds[buf][wave] = any;
    if (any) {  // wave-uniform: their keys are noted, and they enter the products as zeros
      uint32_t* keys = odd_keys[buf][wave];
      keys[lane] = 0u;
      keys[lane + 64] = 0u;
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t f = nan_bytes(vheld[e]);
#pragma unroll
        for (int y = 0; y < kValueDims; ++y)
          if (f & (0x80u << (8 * y))) atomicOr(&keys[x.vdim + y], 1u << (4 * x.vhalf + (e & 3) + 8 * (e >> 2)));
        vheld[e] &= ~((f >> 7) * 0xffu);
      }
    }
    u32x4 o4[4];
    transpose_bf16(vheld, o4);
#pragma unroll
    for (int e = 0; e < kValueDims; ++e) put_value(x, o4[e], buf, e);
  };
  auto walk = [&](auto f16, int from, int to) __attribute__((always_inline)) {
    constexpr bool kF16 = decltype(f16)::value;
    if (from >= to) return;  // workgroup-uniform
    const Lane g = own_lane();
    const Row mine = row_of(g.li);
    const int p = mine.query ? p0 + mine.t : pmax;
    __syncthreads();  // every wave is past the tiles before these
    fetch_keys(g, tile_rows(kh, seen.at(from)));
    fetch_values(std::false_type{}, g, tile_rows(vh, seen.at(from)));
    for (int i = from; i < to; ++i) {
      const int buf = (i - from) & 1, tile = seen.at(i);
      place_keys(g, buf);
      if constexpr (kF16) place_f16(g, tile, buf);
      else place_any(g, buf);
      __syncthreads();  // (and every wave is past the tile before last, whose place the next one takes)
      if (i + 1 < to) {
        fetch_keys(g, tile_rows(kh, seen.at(i + 1)));
        fetch_values(std::false_type{}, g, tile_rows(vh, seen.at(i + 1)));
      }
      if (idle) continue;  // wave-uniform
      f32x16 s[2];
      float kf[4];
      scores(g, buf, s);
      key_scales(tile, kf);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float f = key_factor(kf[q], a.scale_log2e);
#pragma unroll
        for (int r = 0; r < 8; ++r) s[q >> 1][8 * (q & 1) + r] *= f;
      }
      hide(g, p, tile, s);  // (behind the factors: a hidden block's scale may be anything)
      const float ref = refer(largest(s));
      if constexpr (!kF16) {
        for (int q = 0; q < kWaves; ++q) {
          // A value that is NaN makes the sums of the rows that see its key NaN, and no others (in the product it
          // would: a hidden key's zero times NaN).
          if (!odd_lds[buf][q]) continue;  // the same for all
          const int first = tile * kTile + 16 * (q / (kWaves / 4));
          uint32_t vis = 0;
          for (int j = 0; j < 16; ++j) vis |= sees(p, first + j, a.window, a.sinks) ? 1u << j : 0u;
          for (int d = 0; d < 64; ++d)
            if (odd_keys[buf][q][32 * (d >> 4) + 8 * ((d & 15) >> 2) + 4 * g.half + (d & 3)] & vis) odd |= 1ull << d;
        }
      }
#pragma unroll
      for (int gk = 0; gk < 4; ++gk) {
        __builtin_amdgcn_sched_barrier(0);  // (one group's operands at a time: registers)
        float vsc = kF16 ? 1.f : scale_at(vsh, block_of(tile, gk));
        if (!kF16 && !(__builtin_fabsf(vsc) < INFINITY)) {  // wave-uniform
          // It reaches the rows that see a key of its block, whatever their probabilities, and no others.
          bool some = false;
          for (int e = 0; e < 8; ++e)
            some |= sees(p, tile * kTile + 16 * gk + 4 * g.half + (e & 3) + 8 * (e >> 2), a.window, a.sinks);
          vsc = some ? vsc : 0.f;
        }
        u32x4 part[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = __builtin_amdgcn_exp2f(s[gk >> 1][8 * (gk & 1) + 2 * e] - ref);
          const float x1 = __builtin_amdgcn_exp2f(s[gk >> 1][8 * (gk & 1) + 2 * e + 1] - ref);
          if constexpr (kF16) {
            const f16x2 x = __builtin_convertvector(f32x2{x0, x1}, f16x2);
            l = __builtin_amdgcn_fdot2(x, f16x2{1, 1}, l, false);  // (the sum of what the product takes)
            part[0][e] = __builtin_bit_cast(uint32_t, x);
          } else {
            l += x0 + x1;
            uint32_t first, second;
            two_parts(x0 * vsc, x1 * vsc, first, second);
            part[0][e] = first;
            part[1][e] = second;
          }
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const u32x4 vf = vt[buf][v_at(gk, g.half, 32 * d + g.li)];
          if constexpr (kF16) {
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, vf),
                                                          __builtin_bit_cast(f16x8, part[0]), o[d], 0, 0, 0);
          } else {
#pragma unroll
            for (int y = 0; y < 2; ++y)
              o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vf),
                                                             __builtin_bit_cast(bf16x8, part[y]), o[d], 0, 0, 0);
          }
        }
      }
    }
  };

  // Of the tiles that are seen, i0 to i1 - 1, those that every row sees whole and that lie one behind the other: j0 to
  // j1 - 1.
  const int low = a.window < kNoWindow ? max(0, pmax - a.window + kTile) >> kTileShift : 0;
  const int j0 = min(max(seen.index(low), i0), i1), j1 = min(max(seen.index((pmin + 1) >> kTileShift), j0), i1);
  clear();
  float back = 1.f;  // what the values' sums are multiplied with in the end
  if (i0 < i1) {     // workgroup-uniform
    bool exact = fits;
    if (fits) {
      walk(std::true_type{}, i0, j0);
      if (j0 < j1) walk_whole(seen.at(j0), seen.at(j0) + j1 - j0);
      walk(std::true_type{}, j1, i1);
      back = __builtin_ldexpf(1.f, vtop - 127 - kRaise);
      // NaN anywhere: a value may have reached rows that do not see it. A sum without end: scores past 2^24, whose
      // product with the factor, rounded for the reference and not for the exponential, differs by more than f16 holds.
      bool odd_sum = l == INFINITY;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd_sum |= o[d][r] != o[d][r];
      exact = !__syncthreads_or(odd_sum);
    }
    if (!exact) {
      clear();
      back = 1.f;
      walk(std::false_type{}, i0, i1);
    }
  }

  {
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(w[0]) + __uint_as_float(w[1]);
  }
  const Lane g = own_lane();
  const Row x = row_of(g.li);
  if (x.row >= R) return;
  if (!x.query) l = 0.f;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float v = (odd >> (16 * d + r)) & 1 ? __builtin_nanf("") : o[d][r] * back;
      o[d][r] = x.query ? v : 0.f;
    }
  if (a.splits == 1) {
    const float inv = x.query && p0 + x.t >= 0 ? 1.f / l : 0.f;  // (padding, or it sees nothing: zeros)
    uint16_t* dst = a.out + ((static_cast<int64_t>(b) * a.T + x.t) * a.H * G + h * G + x.g) * kD + 4 * g.half;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<u32x2*>(dst + 32 * d + 8 * r) = {skv::f2bf2(o[d][4 * r] * inv, o[d][4 * r + 1] * inv),
                                                           skv::f2bf2(o[d][4 * r + 2] * inv, o[d][4 * r + 3] * inv)};
    return;
  }
  const int64_t at = (static_cast<int64_t>(bh) * R + x.row) * a.splits + split;
  if (g.half == 0) {
    a.ws_ml[2 * at] = x.query ? m : -INFINITY;
    a.ws_ml[2 * at + 1] = l;
  }
  float* dst = a.ws_o + at * kD + 4 * g.half;
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
  join_parts(a, b, t, static_cast<int64_t>(blockIdx.x) * a.splits, 1, a.splits,
             a.out + ((static_cast<int64_t>(b) * a.T + t) * a.H * a.G + h * a.G + g) * kD, acc_lds);
}

constexpr int64_t kMaxThreads = int64_t{1} << 32;  // of a launch

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// How a call is cut up, from its sizes alone (the lengths are on the device).
struct Plan {
  int tiles;   // few rows: tiles of 16; 0 for more
  bool whole;  // few rows: one workgroup a (sequence, kv head)
  int64_t grid;
  int waves;   // more: of a workgroup
  int splits, rtiles;
  int64_t parts;  // partial rows of 128 + 2 floats
};

// Tiles of 64 keys from which workgroups of 8 waves take the rows, if more than 128 and enough for every CU: a thread
// then turns half as many codes into 16 bits, but a tile's barrier holds a whole CU, and a CU without a second
// workgroup waits for the longest (MI355X, us on the device, 4 waves / 8; 4 query heads on each of 8 kv heads: 2000
// tokens of a prompt 57 / 65, 4096 164 / 154, 16384 2116 / 2064, 4 sequences' 100 tokens on 30000 keys 250 / 235; three
// ragged prompts of 4000 on 4 heads, 192 workgroups of 8, 90 / 111; with up to 128 rows the added waves have none: 9
// tokens of 4 sequences on 30000 67 / 84. It loses where 192 workgroups have the same work each: 24 sequences' 64
// tokens on 16000 keys 518 / 477, but on 667 to 16000 352 / 422).
constexpr int kLongTiles = 40;

// Shares of a row tile's keys, of at least 4 tiles, where the workgroups alone would leave part of the chip idle: as
// many as make the walk and the join together shortest. A share's partial rows, written and read, cost 1 KB each, and
// the join 5 us. A workgroup walks a tile in 1.2 us alone on its CU and in 2.0 beside another: taken as 1.1, which
// leaves one share where two would only put workgroups beside one another (1000 tokens on 2000 keys 51 us, with 1.2 in
// two shares 74). Measured (MI355X, us on the device, one share / as many as fit / these; 4 query heads on each of 8 kv
// heads): 64 tokens on 8000 keys 156 / 34 / 36, on 2000 50 / 24 / 24; a prompt of 1000 tokens 32 / 57 / 32, of 500 21 /
// 39 / 21; 471 on 100315 1915 / 809 / 832. It errs where two shares just fill the chip: seven sequences' 520 tokens on
// 3064 keys, 7 heads on one, 71 / 81 / 81.
int shares(int64_t tiles, int64_t wgs, int64_t resident, double rows) {
  const double walk = 1.1 * static_cast<double>(tiles), each = 2e-4 * rows;
  const int64_t most = std::min<int64_t>(resident / wgs, tiles / 4);
  const int64_t n = std::min<int64_t>(most, static_cast<int64_t>(std::sqrt(walk / each)));
  return n > 1 && walk / static_cast<double>(n) + 5. + each * static_cast<double>(n) < walk ? static_cast<int>(n) : 1;
}

Plan plan_of(int B, int H, int G, int T, int cap, int window, int sinks) {
  Plan p{};
  const int64_t R = static_cast<int64_t>(T) * G;
  p.tiles = R <= 32 ? static_cast<int>((R + 15) / 16) : 0;
  // groups that a query can see: both ends of a window may lie inside one
  const int64_t keys = window ? std::min<int64_t>(cap, static_cast<int64_t>(window) + T - 1 + sinks) : cap;
  if (p.tiles) {
    const int64_t groups = std::min<int64_t>((static_cast<int64_t>(cap) + kGroup - 1) / kGroup,
                                             (keys + kGroup - 1) / kGroup + 2);
    p.whole = groups <= whole_groups(p.tiles, static_cast<int64_t>(B) * H);
    if (p.whole) {
      p.grid = static_cast<int64_t>(B) * H;
      return p;
    }
    const int64_t each = (groups + kMinGroups - 1) / kMinGroups;
    const int64_t slots = std::min<int64_t>(B * each, (target_chunks(R) + H - 1) / H + B);
    p.grid = slots * H;
    p.parts = p.grid * R;
    p.splits = 1;
    return p;
  }
  const int64_t tiles = (keys + kTile - 1) / kTile;
  int64_t wgs = 0;
  for (p.waves = R > 4 * kRowsWave && tiles >= kLongTiles ? 8 : 4;; p.waves = 4) {
    const int64_t tile = p.waves * kRowsWave, resident = 2048 / p.waves;  // workgroups at once on the chip's 256 CUs
    p.rtiles = static_cast<int>((R + tile - 1) / tile);
    wgs = static_cast<int64_t>(B) * H * p.rtiles;
    p.splits = shares(tiles, wgs, resident, static_cast<double>(B) * H * R);
    if (p.waves == 4 || wgs * p.splits >= resident) break;
  }
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
  const int threads = p.whole ? few_threads(p.tiles, true) : p.tiles ? 256 : 64 * p.waves;
  const int64_t join = p.parts ? static_cast<int64_t>(batch_size) * q_heads * rows : 0;  // workgroups of it
  if (p.grid * threads >= kMaxThreads || join * 256 >= kMaxThreads) {
    skv_set_error("%s: batch=%d q_heads=%d rows=%d", what, batch_size, q_heads, rows);
    return SKV_EUNSUPPORTED;
  }
  int shift = 4;
  while ((1 << shift) < block) ++shift;
  float* ws_o = static_cast<float*>(workspace);
  Args a{q, q_stride_b, q_stride_h, q_stride_t, k8, v8, c_stride_b, c_stride_h, c_stride_s, k_scale, v_scale,
         s_stride_b, s_stride_h, lengths, counts, out, ws_o, ws_o ? ws_o + p.parts * kD : nullptr, batch_size,
         kv_heads, q_heads / kv_heads, rows, cap, shift, window ? std::min(window, kNoWindow) : kNoWindow, sinks,
         std::fabs(scale) * 1.44269504088896340736f, scale < 0.f,
         target_chunks(static_cast<int64_t>(rows) * (q_heads / kv_heads)), p.splits, p.rtiles};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 g(static_cast<unsigned>(p.grid)), t(256);
  if (p.whole) {
    if (p.tiles == 1) hipLaunchKernelGGL((few_kernel<1, true>), g, dim3(threads), 0, s, a);
    else hipLaunchKernelGGL((few_kernel<2, true>), g, dim3(threads), 0, s, a);
  } else if (p.tiles) {
    if (p.tiles == 1) hipLaunchKernelGGL((few_kernel<1, false>), g, t, 0, s, a);
    else hipLaunchKernelGGL((few_kernel<2, false>), g, t, 0, s, a);
    hipLaunchKernelGGL(few_join_kernel, dim3(static_cast<unsigned>(join)), t, 0, s, a);
  } else {
    if (p.waves == 4) hipLaunchKernelGGL(rows_kernel<4>, g, dim3(threads), 0, s, a);
    else hipLaunchKernelGGL(rows_kernel<8>, g, dim3(threads), 0, s, a);
    if (p.splits > 1) hipLaunchKernelGGL(rows_join_kernel, dim3(static_cast<unsigned>(join)), t, 0, s, a);
  }
  return skv_check_launch(what);
}
