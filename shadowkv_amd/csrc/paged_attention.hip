// Causal attention of packed rows: of a step's new tokens, the last ones of their sequences, over keys and values in
// pages (paged), or of whole prompts over their own (packed).
//
//   out[row, hq] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[row, hq] . k_j)
//
// over the keys j <= p of the query's position p = len_b - n_b + t, with a window w only those with j > p - w; keys of a
// page that does not exist are not seen. A query that sees nothing, and a row of no sequence, gets zeros. Scores, sums and
// maxima are fp32, keys and values bf16 as they lie in memory.
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "skv_common.h"

namespace {

using skv::u32x4;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kD = 128;
constexpr int kNoWindow = 1 << 30;

struct Args {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_sp, k_sh, k_st;  // of a page (paged), a head, a token
  int64_t v_sp, v_sh, v_st;  // (paged: the same)
  const int32_t* table;
  int64_t t_stride;
  const int32_t* lengths;
  const int32_t* cu;  // null: one row a sequence
  uint16_t* out;      // [N, H * G, 128]
  float* few_o;       // partial results of the few-row form: [slots * H * R, 128], and their maxima and sums
  float* few_ml;
  float* rows_o;  // of the other: [split items, 128 rows, 128]
  float* rows_ml;
  int N, B, H, G, cap, pages, shift, window;
  int max_new, few_max;  // new tokens of a sequence: of any, of one that the few-row form takes
  int R, target;         // the few-row form's rows of a chunk, and workgroups to aim for
  int splits;            // whether row tiles may be cut into shares
  int64_t parts;         // cut row tiles' shares that there is room for
  float scale_log2e;     // of the scale's magnitude
  bool negative;         // whether the scale is: the queries' sign is turned instead
};

// A wave-uniform word through the scalar unit (nothing writes tables and lengths while these kernels run).
__device__ __forceinline__ int32_t scalar_at(const int32_t* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

struct Seq {
  int first, n, len;  // its rows, its tokens (0 for one with more rows than was said: they see nothing)
};
template <bool kPaged>
__device__ __forceinline__ Seq seq_of(const Args& a, int b) {
  Seq s;
  s.first = b;
  s.n = 1;
  if (a.cu) {
    s.first = min(max(a.cu[b], 0), a.N);
    s.n = min(max(a.cu[b + 1], s.first), a.N) - s.first;
  }
  if constexpr (kPaged) s.len = s.n > a.max_new ? 0 : min(max(a.lengths[b], 0), a.cap);
  else s.len = s.n;
  return s;
}

__device__ __forceinline__ bool sees(int p, int j, int window) { return j <= p && j > p - window; }

__device__ __forceinline__ bool valid_page(const Args& a, int32_t id) {
  return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.pages);
}

// Two fp32 as two bf16 parts each: the first cut off, the second what that leaves, rounded.
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

// x plus a pair of bf16, in one instruction.
__device__ __forceinline__ float add_pair(uint32_t pair, float x) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, 0x3f803f80u), x,
                                         false);
}

// x * f, f at most 1: an infinity stays one, also where f has become zero.
__device__ __forceinline__ f32x4 lowered(f32x4 x, float f) {
#pragma unroll
  for (int r = 0; r < 4; ++r) x[r] = __builtin_fabsf(x[r]) == INFINITY ? x[r] : x[r] * f;
  return x;
}

// x * scale - ref, the product rounded as the reference's was.
__device__ __forceinline__ float behind(float x, float scale, float ref) {
#pragma clang fp contract(off)
  const float y = x * scale;
  return y - ref;
}

// Of a bf16 pair: 1.0 where a value is NaN or the infinity of this sign.
__device__ __forceinline__ uint32_t endless(uint32_t w, uint32_t sign) {
  uint32_t out = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t x = (w >> (16 * e)) & 0xffffu;
    if ((x & 0x7fffu) > 0x7f80u || x == (0x7f80u | sign)) out |= 0x3f80u << (16 * e);
  }
  return out;
}
__device__ __forceinline__ bool any_endless(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {  // those as zeros
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
  return w;
}
// Of eight tokens' rows of eight dims, dim e's eight tokens in turn.
template <typename Rows>
__device__ __forceinline__ u32x4 dims_of(const Rows& w, int e) {
  u32x4 o;
#pragma unroll
  for (int t = 0; t < 4; ++t)
    o[t] = __builtin_amdgcn_perm(w[2 * t + 1][e >> 1], w[2 * t][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
  return o;
}

// Rows [from, to) as zeros, workgroup i of n. All threads.
__device__ __forceinline__ void clear_rows(const Args& a, int from, int to, int i, int n) {
  const int64_t words = static_cast<int64_t>(a.H) * a.G * kD / 8;  // of 16 bytes, a row's
  u32x4* out = reinterpret_cast<u32x4*>(a.out);
  for (int r = from + i; r < to; r += n)
    for (int64_t w = threadIdx.x; w < words; w += blockDim.x) out[r * words + w] = u32x4{0u, 0u, 0u, 0u};
}

// ------------------------------------------------------------------------------------------------
// Few rows over pages: up to 32 of a kv head's query heads and new tokens together (row t * G + g).
//
// Bound: HBM, 512 bytes a key. The sequences' keys are cut into chunks of equal length, however different the sequences
// are (planned on the device from the lengths, so that a captured call follows them), each a workgroup of four waves
// that take its groups of 32 keys in turn, straight from memory into registers: S^T = K Q^T on v_mfma_f32_16x16x32_bf16
// (a row of the queries a column) leaves a lane with 8 keys' scores of one row, which is the second operand of O^T =
// V^T P^T, whose first is the lane's 8 tokens of one dim: neither probabilities nor values cross lanes. A probability
// enters as two bf16 parts (16 significant bits; the matrix cores have the time). 16 keys in a row lie in one page, whose
// number is a scalar load ahead of theirs. Measured (MI355X, 4 query heads on each of 8 kv heads, with the join): 16
// sequences of up to 122880 tokens 688 us, 6.2 TB/s where reads reach 6.45; 1 to 5 drafted tokens of 6 of up to 30011 in
// pages of 16 tokens 98 us, 4.4 TB/s (up to 20 rows: two tiles for every sequence of the call, two waves a SIMD).
constexpr int kGroup = 32;
constexpr int kGroupShift = 5;
constexpr int kMinGroups = 8;  // a chunk's groups, at least
constexpr int kOutLd = kD + 4;
// Chunks to aim for: two workgroups for each that the chip holds at once, since sequences of different lengths end in
// shorter chunks, and with one each the last of them run alone (4 query heads on each of 8 kv heads, behind a fill of 1 GB,
// 768 / 1024 / 1536 / 2304 chunks: 16 sequences of 7680 to 122880 keys 944 / 890 / 892 / 886 us, 32 of up to 30000 180 / 172 /
// 170 / 171, 16 of 65000 725 / 729 / 729 / 736; two tiles, 512 / 768 / 1024 / 1536: 6 of up to 30011 keys 164 / 153 / 156 /
// 148, 24 of up to 8000 164 / 151 / 156 / 152).
constexpr int target_chunks(int rows) { return rows <= 16 ? 1536 : 1024; }
// Groups that a sequence's rows can see (by the table's width and the window) up to which one workgroup of 8 waves takes
// them all, in one launch: what a CU reads by itself while the chip has room, twice that where sequences and kv heads fill
// half of it (us on the device, chunks and a join / whole: one sequence of 512 keys 11.3 / 8.6, of 1024 11.4 / 13.3, 24 of
// 1024 25 / 20, of 2048 40 / 34).
constexpr int whole_groups(int tiles, int64_t rows_of_kv) { return (rows_of_kv >= 128 ? 72 : 24) / tiles; }

struct Span {
  int first, total;  // groups (tiles) of keys that a range of positions sees
};
__device__ __forceinline__ Span seen_by(int pmin, int pmax, int window, int shift) {
  if (pmax < 0) return {0, 0};
  const int lo = max(0, max(pmin, 0) - window + 1) >> shift;
  return {lo, (pmax >> shift) + 1 - lo};
}
__device__ __forceinline__ Span few_groups(const Args& a, const Seq& s) {
  const bool mine = s.n > 0 && s.n <= a.few_max;
  return seen_by(s.len - s.n, mine ? s.len - 1 : -1, a.window, kGroupShift);
}

struct Chunk {
  int index, count, groups;  // which of its sequence's chunks, how many that has, groups of each
};

__device__ __forceinline__ Seq seq_or_none(const Args& a, int b) { return b < a.B ? seq_of<true>(a, b) : Seq{0, 0, 0}; }

// The chunk length, wave-uniform: the sequences' groups dealt over the workgroups to aim for. total0: the lane's
// sequence's, of the first 64.
__device__ __forceinline__ int chunk_groups(const Args& a, int lane, int total0) {
  int64_t total = skv::wave_total(total0);  // (64 sequences of 2^30 tokens have 2^31 groups)
  for (int b0 = 64; b0 < a.B; b0 += 64) total += skv::wave_total(few_groups(a, seq_or_none(a, b0 + lane)).total);
  // (at most what no sequence has)
  return static_cast<int>(min(max(static_cast<int64_t>(kMinGroups), (total * a.H + a.target - 1) / a.target),
                              static_cast<int64_t>(1 << 30)));
}

__device__ __forceinline__ Seq lane_seq(const Seq& s, int l) {
  return Seq{__builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.n, l),
             __builtin_amdgcn_readlane(s.len, l)};
}

// Chunk i of all sequences' and its sequence (false past the last).
__device__ __forceinline__ bool find_chunk(const Args& a, int i, int lane, Chunk& c, int& b, Seq& seq) {
  Seq s = seq_or_none(a, lane);
  int groups = few_groups(a, s).total;
  c.groups = chunk_groups(a, lane, groups);
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    if (b0) {
      s = seq_or_none(a, b0 + lane);
      groups = few_groups(a, s).total;
    }
    const int n = (groups + c.groups - 1) / c.groups;
    const int incl = before + skv::wave_inclusive_scan(n);
    const uint64_t hit = __ballot(i < incl && i >= incl - n);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      b = b0 + l;
      seq = lane_seq(s, l);
      c.count = __builtin_amdgcn_readlane(n, l);
      c.index = i - __builtin_amdgcn_readlane(incl - n, l);
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// kTiles: of 16 rows. kWhole: a workgroup of more waves takes all that a sequence's rows see.
constexpr int few_threads(bool whole) { return 64 * (whole ? 8 : 4); }

template <int kTiles, bool kWhole>
__global__ void __launch_bounds__(few_threads(kWhole), !kWhole && kTiles == 1 ? 3 : 2)
    few_kernel(Args a, bool zeros) {
  constexpr int kWaves = few_threads(kWhole) / 64;
  __shared__ float o_lds[kWaves][16][kOutLd];
  __shared__ float m_lds[kWaves][16], l_lds[kWaves][16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (zeros && a.cu) {  // rows of no sequence, and of sequences with more than was said
    clear_rows(a, 0, min(max(a.cu[0], 0), a.N), blockIdx.x, gridDim.x);
    clear_rows(a, min(max(a.cu[a.B], 0), a.N), a.N, blockIdx.x, gridDim.x);
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int rows = b0 + lane < a.B ? seq_of<true>(a, b0 + lane).n : 0;
      for (uint64_t more = __ballot(rows > a.max_new); more; more &= more - 1) {
        const Seq s = seq_of<true>(a, b0 + __builtin_ctzll(more));
        clear_rows(a, s.first, s.first + s.n, blockIdx.x, gridDim.x);
      }
    }
  }
  const int slot = blockIdx.x / a.H, h = blockIdx.x - slot * a.H;
  Chunk c{0, 1, 1 << 30};
  int b = slot;
  Seq seq;
  if constexpr (kWhole) {
    const Seq x = seq_of<true>(a, b);
    seq = lane_seq(x, 0);
  } else if (!find_chunk(a, slot, lane, c, b, seq)) {  // workgroup-uniform
    return;
  }
  const int G = a.G, len = seq.len, n = seq.n, first = seq.first;
  if (n < 1 || n > a.few_max) return;  // workgroup-uniform
  const int R = n * G;
  const int pmin = len - n, pmax = len - 1;
  const Span seen = few_groups(a, seq);
  const int i0 = kWhole ? 0 : c.index * c.groups, i1 = kWhole ? seen.total : min(i0 + c.groups, seen.total);
  const int li = lane & 15, grp = lane >> 4;

  // Q as the B operand: lane (li, grp) holds row li of a tile, in step s dims 32 s + 8 grp and on. Rows past the last
  // ride along with it and give nothing in the end.
  bf16x8 qf[kTiles][4];
  int p[kTiles];
#pragma unroll
  for (int y = 0; y < kTiles; ++y) {
    const int row = min(16 * y + li, R - 1), t = row / G;
    p[y] = pmin + t;
    const uint16_t* q = a.q + static_cast<int64_t>(first + t) * a.q_st + (h * G + row - t * G) * a.q_sh + 8 * grp;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      qf[y][s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(q + 32 * s) ^
                                                (a.negative ? 0x80008000u : 0u));
  }
  const uint16_t* kh = a.k + h * a.k_sh + 8 * grp;
  const uint16_t* vh = a.v + h * a.k_sh + 8 * li;
  const int32_t* table = a.table + b * a.t_stride;
  const int in_page = (1 << a.shift) - 1;

  f32x4 o[kTiles][8];
  float m[kTiles], l[kTiles];  // the row's reference, in units of log2; this lane's share of its sum
  bool some[kTiles];           // whether it sees a key

  // The pages of a group's two halves (those of the last key for a half behind it).
  auto pages_of = [&](int i, int32_t (&id)[2]) __attribute__((always_inline)) {
    const int j0 = (seen.first + i) * kGroup;
#pragma unroll
    for (int u = 0; u < 2; ++u) id[u] = scalar_at(table + (min(j0 + 16 * u, pmax) >> a.shift));
  };
  // A group's keys and values, the lane's part. Rows behind the sequence's last are that one again.
  u32x4 kr[2][4], vr[8];
  int32_t next[2] = {0, 0};
  // A value that is no number turns what it is multiplied with into NaN, a hidden key's zero too: where NaN comes out,
  // the wave walks again and takes such values out of the products.
  for (bool careful = false;; careful = true) {
#pragma unroll
    for (int y = 0; y < kTiles; ++y) {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[y][e] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[y] = -INFINITY;
      l[y] = 0.f;
      some[y] = false;
    }
    if (i0 + wave < i1) pages_of(i0 + wave, next);
    for (int i = i0 + wave; i < i1; i += kWaves) {
      const int j0 = (seen.first + i) * kGroup;
      const bool exists[2] = {valid_page(a, next[0]), valid_page(a, next[1])};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint16_t* row = kh + static_cast<int64_t>(exists[u] ? next[u] : 0) * a.k_sp +
                              (min(j0 + 16 * u + li, pmax) & in_page) * a.k_st;
#pragma unroll
        for (int s = 0; s < 4; ++s) kr[u][s] = *reinterpret_cast<const u32x4*>(row + 32 * s);
      }
      // (values, whole lines a load, with the streaming hint: 24 sequences of 4096 tokens 88 -> 70 us; keys, half of a
      // line a load, gain nothing from it)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          vr[4 * u + r] = skv::load_nt(reinterpret_cast<const u32x4*>(
              vh + static_cast<int64_t>(exists[u] ? next[u] : 0) * a.k_sp +
              (min(j0 + 16 * u + 4 * grp + r, pmax) & in_page) * a.k_st));
      pages_of(min(i + kWaves, i1 - 1), next);
      f32x4 s[kTiles][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int y = 0; y < kTiles; ++y) s[y][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
          for (int y = 0; y < kTiles; ++y)
            s[y][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[u][st]), qf[y][st], s[y][u], 0,
                                                              0, 0);
#pragma unroll
        for (int y = 0; y < kTiles; ++y)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[y][u][r] *= a.scale_log2e;
      }
      // wave-uniform: a group at an end of what a row sees, or without a page
      if (j0 + kGroup > pmin + 1 || j0 <= pmax - a.window || !exists[0] || !exists[1]) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = j0 + 16 * u + 4 * grp + r;
#pragma unroll
            for (int y = 0; y < kTiles; ++y) {
              const bool yes = exists[u] && sees(p[y], j, a.window);
              s[y][u][r] = yes ? s[y][u][r] : -INFINITY;
              some[y] |= yes;
            }
            // a value that no row sees may be anything
            u32x4& w = vr[4 * u + r];
            if (!(exists[u] && j <= pmax && j > pmin - a.window)) w = u32x4{0u, 0u, 0u, 0u};
          }
      } else {
#pragma unroll
        for (int y = 0; y < kTiles; ++y) some[y] = true;
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
          for (int e = 0; e < 8; ++e) o[y][e] = lowered(o[y][e], f);
        }
        const float ref = m[y] == -INFINITY ? 0.f : m[y];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            const float p0 = __builtin_amdgcn_exp2f(s[y][u][r] - ref);
            const float p1 = __builtin_amdgcn_exp2f(s[y][u][r + 1] - ref);
            l[y] += p0 + p1;
            uint32_t hi, lo;
            two_parts(p0, p1, hi, lo);
            part[y][0][2 * u + r / 2] = hi;
            part[y][1][2 * u + r / 2] = lo;
          }
      }
      bool odd = false;
      if (careful)
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) odd |= any_endless(vr[t][x]);
      if (__any(odd)) {  // wave-uniform
        // It makes the sums of the rows that see its key the same, and no others: how many such keys a row sees is a
        // product of its own, for each sign.
        u32x4 vis[kTiles];
#pragma unroll
        for (int y = 0; y < kTiles; ++y)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + 16 * (e >> 1) + 4 * grp + 2 * (e & 1);
            vis[y][e] = (exists[e >> 1] && sees(p[y], j, a.window) ? 0x3f80u : 0u) |
                        (exists[e >> 1] && sees(p[y], j + 1, a.window) ? 0x3f800000u : 0u);
          }
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers)
            u32x4 is = dims_of(vr, e);
#pragma unroll
            for (int t = 0; t < 4; ++t) is[t] = endless(is[t], z ? 0x8000u : 0u);
#pragma unroll
            for (int y = 0; y < kTiles; ++y) {
              f32x4 count = {0.f, 0.f, 0.f, 0.f};
              count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, is),
                                                              __builtin_bit_cast(bf16x8, vis[y]), count, 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (count[r] > 0.f) o[y][e][r] += z ? -INFINITY : INFINITY;  // (both: NaN)
            }
          }
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) vr[t][x] = finite_part(vr[t][x]);
      }
      // Output tile e: dims 8 li + e.
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const u32x4 vt = dims_of(vr, e);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < kTiles; ++y)
            o[y][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vt),
                                                              __builtin_bit_cast(bf16x8, part[y][x]), o[y][e], 0, 0, 0);
      }
    }
    bool nan = false;
#pragma unroll
    for (int y = 0; y < kTiles; ++y)
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) nan |= o[y][e][r] != o[y][e][r];
    if (careful || !__any(nan)) break;  // wave-uniform
  }

  // The waves' parts: lane (li, grp) holds row li's dims 8 (4 grp + r) + e.
  const bool final_ = kWhole || c.count == 1;
  const int64_t row0 = (static_cast<int64_t>(slot) * a.H + h) * a.R;
#pragma unroll
  for (int y = 0; y < kTiles; ++y) {
    // (all that a row sees at -inf: its sum is 0 / 0)
    const float any = sum_of_rows(some[y] ? 1.f : 0.f);
    float ls = sum_of_rows(l[y]);
    if (any > 0.f && m[y] == -INFINITY) ls = __builtin_nanf("");
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
      float top = m_lds[0][g];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_lds[w][g]);
      const float ref = top == -INFINITY ? 0.f : top;
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float lsum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        // (a wave that saw only -inf, beside one that saw more, adds nothing)
        const float f = __builtin_amdgcn_exp2f(m_lds[w][g] - ref);
        const float lw = top > -INFINITY && m_lds[w][g] == -INFINITY ? 0.f : l_lds[w][g];
        lsum += f * lw;
        sum += lowered(*reinterpret_cast<const f32x4*>(&o_lds[w][g][d]), f);
      }
      if (final_) {
        // (a sum of zero: it sees nothing)
        const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
        const u32x2 out = {skv::f2bf2(sum[0] * inv, sum[1] * inv), skv::f2bf2(sum[2] * inv, sum[3] * inv)};
        const int t = row / G;
        const int64_t at = static_cast<int64_t>(first + t) * a.H * G + h * G + row - t * G;
        *reinterpret_cast<u32x2*>(a.out + at * kD + d) = out;
        continue;
      }
      *reinterpret_cast<f32x4*>(a.few_o + (row0 + row) * kD + d) = sum;
      if (d == 0) {
        a.few_ml[2 * (row0 + row)] = top;
        a.few_ml[2 * (row0 + row) + 1] = lsum;
      }
    }
  }
}

// Joins n partial results (m, l, o), part i at index first + i * stride, into a row of the output: 256 threads, 32
// lanes of four dims by 8 parts at a time. Every wave of it sees the same maximum and sum.
__device__ __forceinline__ void join_parts(const float* ws_o, const float* ws_ml, int64_t first, int64_t stride, int n,
                                           uint16_t* out, f32x4 (&acc_lds)[8][32]) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY;
  for (int i = lane; i < n; i += 64) m = fmaxf(m, ws_ml[2 * (first + i * stride)]);
  m = skv::wave_max_dpp(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int i = lane; i < n; i += 64) {
    const float mi = ws_ml[2 * (first + i * stride)], li = ws_ml[2 * (first + i * stride) + 1];
    l += m > -INFINITY && mi == -INFINITY ? 0.f : li * __builtin_amdgcn_exp2f(mi == -INFINITY ? 0.f : mi - ref);
  }
  l = skv::wave_sum_dpp(l);
  const int d = threadIdx.x & 31, s = threadIdx.x >> 5;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = s; i < n; i += 8) {
    const int64_t at = first + i * stride;
    acc += lowered(*reinterpret_cast<const f32x4*>(ws_o + at * kD + 4 * d), __builtin_amdgcn_exp2f(ws_ml[2 * at] - ref));
  }
  acc_lds[s][d] = acc;
  __syncthreads();
  if (threadIdx.x < 32) {
#pragma unroll
    for (int i = 1; i < 8; ++i) acc += acc_lds[i][d];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<u32x2*>(out + 4 * d) =
        u32x2{skv::f2bf2(acc[0] * inv, acc[1] * inv), skv::f2bf2(acc[2] * inv, acc[3] * inv)};
  }
}

// Workgroup (b, row of at most R, h).
__device__ __forceinline__ void few_join(const Args& a, f32x4 (&acc_lds)[8][32]) {
  const int lane = threadIdx.x & 63;
  const int h = blockIdx.x % a.H, br = blockIdx.x / a.H, b = br / a.R, row = br - b * a.R;
  const Seq mine = seq_or_none(a, lane);
  const Seq s = b < 64 ? lane_seq(mine, b) : seq_of<true>(a, b);
  if (s.n < 1 || s.n > a.few_max || row >= s.n * a.G) return;  // workgroup-uniform
  const int groups = few_groups(a, mine).total;
  const int each = chunk_groups(a, lane, groups);
  const int n = (few_groups(a, s).total + each - 1) / each;
  if (n == 1) return;  // few_kernel's own
  int before = 0;
  for (int b0 = 0; b0 < b; b0 += 64) {
    const int all = b0 ? few_groups(a, seq_or_none(a, b0 + lane)).total : groups;
    const int c = b0 + lane < b ? (all + each - 1) / each : 0;
    before += __builtin_amdgcn_readlane(skv::wave_inclusive_scan(c), 63);
  }
  const int t = row / a.G, g = row - t * a.G;
  join_parts(a.few_o, a.few_ml, (static_cast<int64_t>(before) * a.H + h) * a.R + row, static_cast<int64_t>(a.H) * a.R, n,
             a.out + (static_cast<int64_t>(s.first + t) * a.H * a.G + h * a.G + g) * kD, acc_lds);
}
__global__ void __launch_bounds__(256) few_join_kernel(Args a) {
  __shared__ f32x4 acc_lds[8][32];
  few_join(a, acc_lds);
}

// ------------------------------------------------------------------------------------------------
// Any rows.
//
// Bound: the matrix cores. The rows of a kv head are its queries' heads together, row t * G + g, so that a tile of keys
// serves all of them. A workgroup of four waves owns 128 rows, 32 a wave, a row a lane, and walks the tiles of 64 keys
// that any of them sees, or a share of them where a sequence's tiles are many beside what the chip has to do (planned on
// the device: a decoded token beside prompts, a few prompts). Tiles come straight from memory into LDS, two of each ahead.
// S^T = K Q^T on v_mfma_f32_32x32x16_bf16 leaves a lane with 32 keys' scores of one row, in the order of which the
// values' operand is read from LDS with the transposing loads: O^T = V^T P^T.
//
// Measured (MI355X, where a large bf16 GEMM has 1.41 PFLOP/s): two prompts of 16001 and 10000 tokens, 16 query heads on each
// of 2 kv heads, 2600 us, 1.12 PFLOP/s; 8 of 4096 down to 1400, 4 on each of 8, 575 to 610, 0.90 to 0.95; 2048 tokens
// behind 58000 in pages 2400, 1.08. Counters (the first, before rows went through LDS): the matrix cores are busy in 55% of
// the cycles, the vector units in 39%, no bank conflicts, at a clock of 1.84 of 2.4 GHz; with zeros in Q, K and V the same
// call takes three quarters of the time: the power is the limit, and what is not computed or moved counts for more than
// what is hidden.
//
// A probability enters its product rounded to bf16, and the sum that divides the result takes the same rounded ones. A
// rounding is 2^-9 of the probability (2^-8 at worst) either way, so that the output's error is that of a mean over the
// keys of terms of 2^-9, beside the 2^-9 of its own rounding; a second bf16 part would cost half as many matrix
// instructions again.
constexpr int kTile = 64;
constexpr int kTileShift = 6;
constexpr int kRowsWave = 32;
constexpr int kTileWords = kTile * kD * 2 / 16;  // 16-byte chunks
constexpr int kMinTiles = 4;  // a share's tiles, at least: less is a workgroup's beginning and end
// Tiles that shares have to save a walk: a join's launch, and the partial rows' way out and back (1 KB a row and share).
constexpr int kShareGain = 8;
constexpr float kGainRows = 4600.f;  // rows for one tile more, for each share
constexpr int resident(int tile_rows) { return 65536 / tile_rows; }  // workgroups at once
constexpr float kSlack = 8.f;  // how far (in log2) the reference is set above the largest score

// What a sequence is for the rows kernel: its row tiles, the tiles of keys that the last of them sees (the most), and the
// first.
struct Work {
  int rts, tiles, least;
};
template <bool kPaged, int kRowsTile>
__device__ __forceinline__ Work work_of(const Args& a, const Seq& s) {
  if (s.n <= a.few_max) return {0, 0, 0};
  const int rts = (s.n * a.G + kRowsTile - 1) / kRowsTile;  // (below 2^30 rows)
  const int all = (s.len + kTile - 1) >> kTileShift;
  if (a.window < kNoWindow) {  // each as many, but where the sequence begins
    const int most = min(all, (a.window + (kRowsTile - 1) / a.G + 1 + 2 * kTile - 2) >> kTileShift);
    return {rts, most, most};
  }
  const int last = s.len - s.n + min(s.n - 1, (kRowsTile - 1) / a.G);  // the first row tile's last position
  return {rts, all, last < 0 ? 0 : (last >> kTileShift) + 1};
}

// How row tiles are cut into shares of at most `tiles` tiles of keys: one that sees fewer than `cut` is one share. Row
// tiles see more the later they are, so that those of as many shares lie together.
struct Share {
  int tiles, cut;
};
template <int kRowsTile>
struct Cut {
  const Args& a;
  Seq s;
  Work w;
  Share share;
  __device__ __forceinline__ int shares_of(int tiles) const {
    if (tiles < share.cut) return 1;
    return static_cast<int>((static_cast<uint32_t>(tiles) + share.tiles - 1) / static_cast<uint32_t>(share.tiles));
  }
  // Row tiles that see at most t tiles of keys (no window).
  __device__ __forceinline__ int upto(int t) const {
    const int64_t x = static_cast<int64_t>(t) * kTile - (s.len - s.n);  // tokens of them that see no more
    return x <= 0 ? 0 : x >= s.n ? w.rts : min(w.rts, static_cast<int>(x) * a.G / kRowsTile);
  }
  __device__ __forceinline__ bool even() const { return a.window < kNoWindow || shares_of(w.tiles) == 1; }
  __device__ __forceinline__ int whole() const {  // row tiles that are not cut
    return even() ? shares_of(w.tiles) == 1 ? w.rts : 0 : upto(share.cut - 1);
  }
  // Row tiles of k > 1 shares: from() to upto().
  __device__ __forceinline__ int below(int k, int uncut) const { return max(uncut, upto(k * share.tiles)); }
  __device__ __forceinline__ int least() const { return max(2, shares_of(w.least)); }
  // All shares, and of them those of row tiles that are cut.
  __device__ __forceinline__ void count(int& items, int& parts) const {
    const int uncut = whole();
    if (even()) {
      items = w.rts * shares_of(w.tiles);
    } else {
      items = uncut;
      int before = uncut;
      for (int k = least(), most = shares_of(w.tiles); k <= most; ++k) {
        const int end = k == most ? w.rts : below(k, uncut);
        items += k * (end - before);
        before = end;
      }
    }
    parts = items - uncut;
  }
  // Share i of all, the last row tile's first; returns the row tile.
  __device__ __forceinline__ int find(int i, int& split, int& splits) const {
    int end = w.rts;
    const int uncut = whole();
    splits = shares_of(w.tiles);
    if (!even())
      for (const int low = least(); splits >= low; --splits) {
        const int begin = splits == low ? uncut : below(splits - 1, uncut);
        if (i < splits * (end - begin)) break;
        i -= splits * (end - begin);
        end = begin;
        if (splits == low) {
          splits = 1;
          break;
        }
      }
    const uint32_t tile = static_cast<uint32_t>(i) / static_cast<uint32_t>(splits);
    split = i - static_cast<int>(tile) * splits;
    return end - 1 - static_cast<int>(tile);
  }
  // Row tile rt's first share, and how many it has.
  __device__ __forceinline__ int place(int rt, int& splits) const {
    int end = w.rts, i = 0;
    const int uncut = whole();
    splits = shares_of(w.tiles);
    if (!even())
      for (const int low = least(); splits > low; --splits) {
        const int begin = below(splits - 1, uncut);
        if (rt >= begin) break;
        i += splits * (end - begin);
        end = begin;
      }
    return i + splits * (end - 1 - rt);
  }
};

// The shares, wave-uniform: all row tiles' tiles dealt over the workgroups that the chip holds at once; a little longer
// where there are few row tiles and their shares would need a second round of workgroups (19 row tiles of 1917 tiles in 14
// shares, 266 for 256 workgroups). s, w: the lane's sequence's, of the first 64.
// The join makes the same plan again: every step of it is rounded by itself, so that no compiler's choice of fused ones in
// either kernel tells them apart.
template <bool kPaged, int kRowsTile>
__device__ __forceinline__ Share share_tiles(const Args& a, int lane, const Seq& s, const Work& w) {
#pragma clang fp contract(off)
  // (few tiles: the way past the rest, which costs the smallest calls 3 us)
  if (!a.splits || (a.B <= 64 && !__any(w.tiles >= kMinTiles + kShareGain))) return {1, 1 << 30};
  constexpr float kAtOnce = resident(kRowsTile);
  float total = 0.f, rts = 0.f;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    Work y = b0 ? Work{0, 0, 0} : w;
    if (b0 && b0 + lane < a.B) y = work_of<kPaged, kRowsTile>(a, seq_of<kPaged>(a, b0 + lane));
    total += skv::wave_sum_dpp(static_cast<float>(y.rts) * 0.5f * static_cast<float>(y.tiles + y.least));
    rts += skv::wave_sum_dpp(static_cast<float>(y.rts));
  }
  rts *= static_cast<float>(a.H);
  // Shares of n tiles for one walk of t: worth it where t - n is above kShareGain + r t / n.
  const float r = rts * kRowsTile / kGainRows;
  const auto shares = [&](float n) __attribute__((always_inline)) {
#pragma clang fp contract(off)
    n = fminf(ceilf(fmaxf(fmaxf(n, kMinTiles), 2.f * r)), 1e9f);
    return Share{static_cast<int>(n), static_cast<int>(fminf(ceilf((n + kShareGain) / (1.f - r / n)), 1e9f))};
  };
  Share share = shares(total * static_cast<float>(a.H) / kAtOnce);
  if (rts * 2.f > kAtOnce) return share;
  for (int turn = 0; turn < 2; ++turn) {
    float items = 0.f;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      Seq x = b0 ? Seq{0, 0, 0} : s;
      Work y = b0 ? Work{0, 0, 0} : w;
      if (b0 && b0 + lane < a.B) {
        x = seq_of<kPaged>(a, b0 + lane);
        y = work_of<kPaged, kRowsTile>(a, x);
      }
      int n, parts;
      Cut<kRowsTile>{a, x, y, share}.count(n, parts);
      items += skv::wave_sum_dpp(static_cast<float>(n));
    }
    const float over = items * static_cast<float>(a.H) / kAtOnce;
    if (over <= 1.f) break;
    share = shares(static_cast<float>(share.tiles) * over);
  }
  return share;
}

struct Item {
  int b, rt, split, splits;
  int part;  // its index among those of cut row tiles, of one kv head
  Seq seq;
  int begin, end;  // the rows of all sequences
};
// Item i of all sequences' (false past the last). Row tiles from a sequence's last on, the longest.
template <bool kPaged, int kRowsTile>
__device__ __forceinline__ bool find_item(const Args& a, int i, int lane, Item& it) {
  Seq s{0, 0, 0};
  Work w{0, 0, 0};
  if (lane < a.B) {
    s = seq_of<kPaged>(a, lane);
    w = work_of<kPaged, kRowsTile>(a, s);
  }
  const Share share = share_tiles<kPaged, kRowsTile>(a, lane, s, w);
  it.begin = __builtin_amdgcn_readlane(s.first, 0);
  it.end = a.B <= 64 ? __builtin_amdgcn_readlane(s.first + s.n, a.B - 1)
                     : a.cu ? min(max(scalar_at(a.cu + a.B), 0), a.N) : a.N;
  int before = 0, parts = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    if (b0) {
      s = Seq{0, 0, 0};
      w = Work{0, 0, 0};
      if (b0 + lane < a.B) {
        s = seq_of<kPaged>(a, b0 + lane);
        w = work_of<kPaged, kRowsTile>(a, s);
      }
    }
    int n = w.rts, cut = 0;
    if (__any(w.tiles >= share.cut)) Cut<kRowsTile>{a, s, w, share}.count(n, cut);  // (else none is cut)
    const int incl = before + skv::wave_inclusive_scan(n);
    const int incl_parts = parts + skv::wave_inclusive_scan(cut);
    const uint64_t hit = __ballot(i < incl && i >= incl - n);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int at = i - __builtin_amdgcn_readlane(incl - n, l);
      it.b = b0 + l;
      it.seq = lane_seq(s, l);
      const Work mine{__builtin_amdgcn_readlane(w.rts, l), __builtin_amdgcn_readlane(w.tiles, l),
                      __builtin_amdgcn_readlane(w.least, l)};
      it.rt = mine.rts - 1 - at;
      it.split = 0;
      it.splits = 1;
      if (mine.tiles >= share.cut) it.rt = Cut<kRowsTile>{a, it.seq, mine, share}.find(at, it.split, it.splits);
      it.part = __builtin_amdgcn_readlane(incl_parts - cut, l) + at;  // (those that are cut come first)
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
    parts = __builtin_amdgcn_readlane(incl_parts, 63);
  }
  return false;
}

__device__ __forceinline__ void load_lds(const void* src, u32x4* dst) {  // lane l's 16 bytes go to dst + l
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// 16-byte chunk c (8 dims) of key row r of a tile in LDS, and of value row r: both spread over the banks, the keys' for
// loads of a chunk from each of 32 rows, the values' for transposing loads of two from each of 4.
__device__ __forceinline__ int k_at(int r, int c) { return r * 16 + (c ^ (r & 15)); }
__device__ __forceinline__ int v_at(int r, int c) { return r * 16 + (c ^ (4 * (r & 3))); }

// kWaves: 4, two workgroups to a CU, or 8, one.
template <bool kPaged, int kWaves>
__global__ void __launch_bounds__(64 * kWaves, 2) rows_kernel(Args a) {
  constexpr int kRowsTile = kWaves * kRowsWave;
  constexpr int kCarry = kTile / kWaves;  // a tile's rows that a wave carries
  __shared__ u32x4 ka[kTileWords], kb[kTileWords], va[kTileWords], vb[kTileWords];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.x % a.H;
  Item it;
  if (!find_item<kPaged, kRowsTile>(a, blockIdx.x / a.H, lane, it)) {  // workgroup-uniform
    clear_rows(a, 0, it.begin, blockIdx.x, gridDim.x);
    clear_rows(a, it.end, a.N, blockIdx.x, gridDim.x);
    return;
  }
  if (it.splits > 1 && static_cast<int64_t>(it.part + 1) * a.H > a.parts) return;  // (places that fall)
  const int b = it.b, G = a.G, len = it.seq.len, n = it.seq.n, first = it.seq.first;
  const int R = n * G;
  const int r0 = it.rt * kRowsTile;
  const int p0 = len - n;  // the position of the first new token
  const int pmin = p0 + r0 / G;
  const int pmax = p0 + min(n - 1, (r0 + kRowsTile - 1) / G);
  const Span seen = seen_by(pmin, pmax, a.window, kTileShift);
  const int each = (seen.total + it.splits - 1) / it.splits;
  const int t0 = seen.first + min(it.split * each, seen.total);
  const int t1 = min(t0 + each, seen.first + seen.total);

  // Row li of the wave: token t, head g of the kv head's. Those past the last ride along with it and give nothing.
  struct Row {
    int li, half, t, g;
    bool query;
  };
  // (made anew where it is needed, from a thread id that the compiler takes for another one: what hangs on it would else
  // be held in registers)
  auto own_row = [&]() __attribute__((always_inline)) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    Row x;
    x.li = tid & 31;
    x.half = (tid >> 5) & 1;
    const int row = r0 + wave * kRowsWave + x.li, at = min(row, R - 1);
    x.query = row < R;
    x.t = at / G;
    x.g = at - x.t * G;
    return x;
  };
  const int li = lane & 31, half = lane >> 5;
  const int wave0 = r0 + wave * kRowsWave;
  const bool idle = wave0 >= R;  // a wave of rows past the last: it carries its share of the tiles, and no more
  const int wmin = p0 + wave0 / G;  // the wave's positions
  const int wmax = p0 + min(n - 1, (wave0 + kRowsWave - 1) / G);
  // A wave carries kCarry of a tile's rows, 4 at a time; they lie in one page. Rows behind the sequence's last key are that
  // one again: what lies there may be anything, or nothing.
  const int k_st = static_cast<int>(a.k_st), v_st = kPaged ? k_st : static_cast<int>(a.v_st);
  const uint16_t* kh = a.k + h * a.k_sh;
  const uint16_t* vh = a.v + h * (kPaged ? a.k_sh : a.v_sh);
  const int32_t* table = kPaged ? a.table + b * a.t_stride : nullptr;
  const int in_page = (1 << a.shift) - 1;
  auto page_of = [&](int tile) __attribute__((always_inline)) {  // of the wave's rows
    return kPaged ? scalar_at(table + (min(tile * kTile + kCarry * wave, len - 1) >> a.shift)) : 0;
  };
  // A wave's rows of a tile that lies whole in the sequence.
  auto place = [&](const uint16_t* head, int st, int tile, int32_t id) __attribute__((always_inline)) {
    const int j0 = tile * kTile + kCarry * wave;
    if constexpr (kPaged) head += (valid_page(a, id) ? id : 0) * a.k_sp + static_cast<int64_t>(j0 & in_page) * st;
    else head += static_cast<int64_t>(first + j0) * st;
    return reinterpret_cast<const char*>(head);
  };
  auto load_tile = [&](const uint16_t* head, int st, int spread, int tile, int32_t id, u32x4* dst)
                       __attribute__((always_inline)) {
    const int j0 = tile * kTile + kCarry * wave;  // the wave's first key
    const int from = min(j0, len - 1);
    const uint16_t* base;
    if constexpr (kPaged)
      base = head + (valid_page(a, id) ? id : 0) * a.k_sp + static_cast<int64_t>(from & in_page) * st;
    else base = head + static_cast<int64_t>(first + from) * st;
    const int most = len - 1 - from;  // rows there, but one
    int l_ = lane;
    asm volatile("" : "+v"(l_));  // (what hangs on it is made anew each time: registers)
#pragma unroll
    for (int i = 0; i < kCarry / 4; ++i) {
      const int r = 4 * i + (l_ >> 4);
      const int c = spread ? (l_ & 15) ^ ((kCarry * wave + r) & 15) : (l_ & 15) ^ (4 * (r & 3));
      load_lds(base + min(r, most) * st + 8 * c, dst + (wave * kCarry + 4 * i) * 16);
    }
  };
  auto load_keys = [&](int tile, int32_t id, u32x4* dst) __attribute__((always_inline)) {
    load_tile(kh, k_st, 1, tile, id, dst);
  };
  auto load_values = [&](int tile, int32_t id, u32x4* dst) __attribute__((always_inline)) {
    load_tile(vh, v_st, 0, tile, id, dst);
  };

  if (t0 < t1) {  // workgroup-uniform: the first tile is on its way
    const int32_t id = page_of(t0);
    load_keys(t0, id, ka);
    load_values(t0, id, va);
  }
  // Q, read a row (16 lanes) at a time and turned into the B operand in the wave's share of LDS (chunk c of row r at c ^
  // (r & 15)): lane (li, half) holds row li's chunks 2 s + half.
  u32x4 qf[8];
  int p;  // the row's position
  {
    const Row x = own_row();
    p = p0 + x.t;
    u32x4 held[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 4), t = __shfl(x.t, r), g = min(r0 + wave * kRowsWave + r, R - 1) - t * G;
      held[i] = *reinterpret_cast<const u32x4*>(a.q + static_cast<int64_t>(first + t) * a.q_st + (h * G + g) * a.q_sh +
                                                8 * (lane & 15));
      if (a.negative) held[i] ^= 0x80008000u;
    }
    u32x4* own = (wave < 4 ? kb : vb) + (wave & 3) * 256;
#pragma unroll
    for (int turn = 0; turn < 2; ++turn) {  // (16 rows at a time: the first tile comes into the other half of LDS)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * i + (lane >> 4);
        own[r * 16 + ((lane & 15) ^ r)] = held[4 * turn + i];
      }
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const u32x4 w = own[(li & 15) * 16 + ((2 * s + half) ^ (li & 15))];
        qf[s] = turn == 0 || li >> 4 ? w : qf[s];
      }
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    }
  }

  f32x16 o[4];
  float m, l;
  bool some = false;  // whether the row sees a key
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    m = -INFINITY;
    l = 0.f;
  };
  int kbase = k_at(li, half);
  auto scores = [&](const u32x4* kt, f32x16 (&s)[2]) __attribute__((always_inline)) {
    asm volatile("" : "+v"(kbase));  // (its eight forms are made anew each time: registers)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, kt[512 * u + (kbase ^ (2 * c))]), __builtin_bit_cast(bf16x8, qf[c]), s[u], 0,
            0, 0);
      if (c & 1) __builtin_amdgcn_sched_barrier(0);  // (a few operands at a time: registers)
    }
  };
  // keys: bit i, whether the tile's keys 16 i to 16 i + 15 have a page.
  auto hide = [&](int tile, uint32_t keys, f32x16 (&s)[2]) __attribute__((always_inline)) {
    const int from = tile * kTile + 4 * half;  // key c of the lane: from + c
    const int last = p - from, behind = p - a.window - from;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int c = 32 * u + 8 * (r / 4) + (r % 4);
        const bool yes = (c <= last) & (c > behind) & ((keys >> (2 * u + r / 8)) & 1);
        s[u][r] = yes ? s[u][r] : -INFINITY;
        some |= yes;
      }
  };
  auto cut_off = [&](int tile) __attribute__((always_inline)) {  // wave-uniform
    return tile * kTile + kTile - 1 > wmin || tile * kTile <= wmax - a.window;
  };
  auto largest_half = [&](float mx) __attribute__((always_inline)) {  // with the row's other lane
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(w[0]), __uint_as_float(w[1]));
  };
  auto largest = [&](const f32x16 (&s)[2]) __attribute__((always_inline)) {  // NaN where there is one
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = __builtin_elementwise_maximum(mx, s[u][r]);
    return largest_half(mx);
  };
  // The reference moves only when a score passes it, to kSlack above that: the ratio of the sums does not depend on it, and
  // no probability is above one.
  auto refer = [&](float mx) __attribute__((always_inline)) {
    if (__any(mx > m)) {  // wave-uniform
      const float mn = fmaxf(m, mx + kSlack);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
    }
    return m == -INFINITY ? 0.f : m;
  };
  // Where the lane's transposing loads of a group's first half begin, for the four tiles of 32 dims: bytes.
  int vlane[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
    vlane[d] = 16 * v_at(4 * half + ((lane & 15) >> 2), 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) +
               8 * (lane & 1);
  auto value_operand = [&](const u32x4* vt, int gk, int d) __attribute__((always_inline)) {
    const auto at = (const __attribute__((address_space(3))) char*)vt + vlane[d] + 16 * gk * 256;
    u32x4 f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const auto w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                   (__attribute__((address_space(3))) s16x4*)(at + 8 * s * 256)));
      f[2 * s] = w[0];
      f[2 * s + 1] = w[1];
    }
    return f;
  };
  auto probabilities = [&](const f32x16 (&s)[2], int gk, float ref, u32x4& part) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x0 = __builtin_amdgcn_exp2f(fmaf(s[gk >> 1][8 * (gk & 1) + 2 * e], a.scale_log2e, -ref));
      const float x1 = __builtin_amdgcn_exp2f(fmaf(s[gk >> 1][8 * (gk & 1) + 2 * e + 1], a.scale_log2e, -ref));
      part[e] = skv::f2bf2(x0, x1);
      l = add_pair(part[e], l);
    }
  };
  // The lane's places in a wave's rows of a tile, in bytes from the first: keys (4 i in them), values.
  uint32_t k_off[kCarry / 4], v_off;
  {
    const int r = lane >> 4, c = lane & 15;
#pragma unroll
    for (int i = 0; i < kCarry / 4; ++i)
      k_off[i] = 2u * ((4 * i + r) * static_cast<uint32_t>(k_st) + 8 * (c ^ ((kCarry * wave + 4 * i + r) & 15)));
    v_off = 2u * (r * static_cast<uint32_t>(v_st) + 8 * (c ^ (4 * r)));
  }
  // Tiles that every row sees whole, in a pipeline: a tile's probabilities and their product are taken while the next
  // one's scores are and the keys after that and the next values are on their way: one barrier a tile, and vector work
  // beside every matrix instruction. The order is written down slice by slice (a scheduler of its own would read all
  // operands first, and spill).
  // The tile behind them is in place then, in ka and va if their number is even.
  auto walk_whole = [&](int from, int to) __attribute__((always_inline)) {
    const int end = t1 - 1;
    int32_t id1, id2;  // the pages of tiles i + 1 and i + 2
    auto fetch_keys = [&](int tile, int32_t id, u32x4* dst) __attribute__((always_inline)) {
      const char* base = place(kh, k_st, tile, id);
#pragma unroll
      for (int i = 0; i < kCarry / 4; ++i) load_lds(base + k_off[i], dst + (wave * kCarry + 4 * i) * 16);
    };
    auto fetch_values = [&](int tile, int32_t id, u32x4* dst) __attribute__((always_inline)) {
      const char* base = place(vh, v_st, tile, id);
#pragma unroll
      for (int i = 0; i < kCarry / 4; ++i)
        load_lds(base + 8 * i * static_cast<int64_t>(v_st) + v_off, dst + (wave * kCarry + 4 * i) * 16);
    };
    // Keys i + 2 and values i + 1 (past the last, the last one's again, which the sequence may end in).
    auto fetch_next = [&](int tile, u32x4* kd, u32x4* vd) __attribute__((always_inline)) {
      if (tile + 2 < end) {
        fetch_keys(tile + 2, id2, kd);
        fetch_values(tile + 1, id1, vd);
      } else {
        load_keys(min(tile + 2, end), id2, kd);
        load_values(min(tile + 1, end), id1, vd);
      }
      id1 = id2;
      id2 = page_of(min(tile + 3, end));
    };
    // One tile: its scores in s, the next one's into sn (past the last, the last one's again). Keys i + 1 are in kt,
    // values i in vt; keys i + 2 go to kd and values i + 1 to vd.
    auto step = [&](int tile, f32x16 (&s)[2], f32x16 (&sn)[2], const u32x4* kt, const u32x4* vt, u32x4* kd, u32x4* vd)
                    __attribute__((always_inline)) {
      // Keys i + 1 and values i are in place, and every wave is past keys i and values i - 1.
      skv::drain_and_barrier();
      asm volatile("" : "+v"(kbase));
      u32x4 f[4];
      auto operand = [&](int j) __attribute__((always_inline)) {
        if (j < 16) f[j & 3] = kt[512 * (j & 1) + (kbase ^ (j & 14))];  // k_at(32 u + li, 2 c + half)
        else f[j & 3] = value_operand(vt, (j - 16) >> 2, j & 3);
      };
#pragma unroll
      for (int j = 0; j < 3; ++j) operand(j);
      fetch_next(tile, kd, vd);
      float mx = -INFINITY, ref = 0.f;
      u32x4 part[4];
      auto pair = [&](int k) __attribute__((always_inline)) {
        const int gk = k >> 2, e = k & 3;
        const float x0 = __builtin_amdgcn_exp2f(fmaf(s[gk >> 1][8 * (gk & 1) + 2 * e], a.scale_log2e, -ref));
        const float x1 = __builtin_amdgcn_exp2f(fmaf(s[gk >> 1][8 * (gk & 1) + 2 * e + 1], a.scale_log2e, -ref));
        part[gk][e] = skv::f2bf2(x0, x1);
        l = add_pair(part[gk][e], l);
      };
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) sn[u][r] = 0.f;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        if (j < 29) operand(j + 3);
        if (j < 16)
          sn[j & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[j & 3]),
                                                              __builtin_bit_cast(bf16x8, qf[j >> 1]), sn[j & 1], 0, 0,
                                                              0);
        else
          o[j & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[j & 3]),
                                                             __builtin_bit_cast(bf16x8, part[(j - 16) >> 2]), o[j & 3],
                                                             0, 0, 0);
        // (vector work, evenly: the maximum and the reference, 16 pairs of probabilities, each before the product that
        // takes it)
        constexpr int kPair[32] = {-1, -1, -1, -1, 0, -1, 1, -1, 2, 3, -1, 4, 5, -1, 6, 7,
                                   8, 9, -1, 10, 11, -1, 12, 13, -1, 14, 15, -1, -1, -1, -1, -1};
        if (j < 4) {
#pragma unroll
          for (int r = 0; r < 8; ++r) mx = __builtin_elementwise_maximum(mx, s[j >> 1][8 * (j & 1) + r]);
          if (j == 3) ref = refer(largest_half(mx) * a.scale_log2e);
        } else if (kPair[j] >= 0) {
          pair(kPair[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    id1 = page_of(min(from + 1, end));
    id2 = page_of(min(from + 2, end));
    load_keys(min(from + 1, end), id1, kb);
    some = true;
    skv::drain_and_barrier();
    if (idle) {  // wave-uniform
      for (int i = from; i < to; ++i) {
        const bool odd = (i - from) & 1;
        skv::drain_and_barrier();
        fetch_next(i, odd ? kb : ka, odd ? va : vb);
      }
      return;
    }
    f32x16 sa[2], sb[2];
    scores(ka, sa);
    for (int i = from;;) {
      step(i, sa, sb, kb, va, ka, vb);
      if (++i >= to) break;
      step(i, sb, sa, ka, vb, kb, va);
      if (++i >= to) break;
    }
  };
  // Any tiles, one after the other, the next one on its way; the first one is, too: to kb and vb where odd.
  auto walk = [&](int from, int to, bool odd) __attribute__((always_inline)) {
    if (from >= to) return;  // workgroup-uniform
    auto step = [&](int tile, const u32x4* kt, const u32x4* vt, u32x4* kd, u32x4* vd) __attribute__((always_inline)) {
      skv::drain_and_barrier();
      if (tile + 1 < to) {
        const int32_t id = page_of(tile + 1);
        load_keys(tile + 1, id, kd);
        load_values(tile + 1, id, vd);
      }
      if (idle) return;
      f32x16 s[2];
      scores(kt, s);
      if (cut_off(tile)) hide(tile, 15u, s);
      else some = true;
      const float ref = refer(largest(s) * a.scale_log2e);
#pragma unroll
      for (int gk = 0; gk < 4; ++gk) {
        __builtin_amdgcn_sched_barrier(0);  // (one group's operands at a time: registers)
        u32x4 part;
        probabilities(s, gk, ref, part);
#pragma unroll
        for (int d = 0; d < 4; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, value_operand(vt, gk, d)),
                                                         __builtin_bit_cast(bf16x8, part), o[d], 0, 0, 0);
      }
    };
    for (int tile = from;;) {
      if (!odd) {
        step(tile, ka, va, kb, vb);
        if (++tile >= to) break;
      }
      odd = false;
      step(tile, kb, vb, ka, va);
      if (++tile >= to) break;
    }
  };

  // One tile after the other, whatever the values and the table hold: a value that is no number reaches the rows that
  // see its key, and no others; keys without a page are seen by none.
  uint64_t pos = 0, neg = 0;  // this lane's outputs that an infinity, or NaN, reaches: bit 16 d + r
  auto walk_any = [&]() __attribute__((always_inline)) {
    uint32_t* odd = reinterpret_cast<uint32_t*>(kb);  // [sign][half of the tile's keys][dim]: keys as bits
    for (int tile = t0; tile < t1; ++tile) {
      __syncthreads();  // every wave is past the tile before
      const int32_t id = page_of(tile);
      load_keys(tile, id, ka);
      load_values(tile, id, va);
      uint32_t keys = 15u;
      if constexpr (kPaged) {
        keys = 0;
        for (int i = 0; i < 4; ++i)
          if (valid_page(a, scalar_at(table + (min(tile * kTile + 16 * i, len - 1) >> a.shift)))) keys |= 1u << i;
      }
      skv::drain_and_barrier();
      if (threadIdx.x < 256) {
        const int d = threadIdx.x & (kD - 1), side = threadIdx.x >> 7;
        uint16_t* column = reinterpret_cast<uint16_t*>(va);
        uint32_t up = 0, down = 0;
        for (int j = 0; j < 32; ++j) {
          uint16_t& x = column[8 * v_at(32 * side + j, d >> 3) + (d & 7)];
          if ((x & 0x7f80u) != 0x7f80u) continue;
          if (x != 0xff80u) up |= 1u << j;
          if (x != 0x7f80u) down |= 1u << j;
          x = 0;
        }
        odd[side * kD + d] = up;
        odd[(2 + side) * kD + d] = down;
      }
      __syncthreads();
      if (idle) continue;
      f32x16 s[2];
      scores(ka, s);
      hide(tile, keys, s);
      const float ref = refer(largest(s) * a.scale_log2e);
      uint32_t seen_keys[2] = {0, 0};
      for (int j = 0; j < kTile; ++j)
        if (sees(p, tile * kTile + j, a.window) && ((keys >> (j >> 4)) & 1)) seen_keys[j >> 5] |= 1u << (j & 31);
      for (int d = 0; d < 64; ++d) {
        const int dim = 32 * (d >> 4) + 8 * ((d & 15) >> 2) + 4 * half + (d & 3);
        if ((odd[dim] & seen_keys[0]) | (odd[kD + dim] & seen_keys[1])) pos |= 1ull << d;
        if ((odd[2 * kD + dim] & seen_keys[0]) | (odd[3 * kD + dim] & seen_keys[1])) neg |= 1ull << d;
      }
#pragma unroll
      for (int gk = 0; gk < 4; ++gk) {
        __builtin_amdgcn_sched_barrier(0);  // (one group's operands at a time: registers)
        u32x4 part;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = __builtin_amdgcn_exp2f(behind(s[gk >> 1][8 * (gk & 1) + 2 * e], a.scale_log2e, ref));
          const float x1 = __builtin_amdgcn_exp2f(behind(s[gk >> 1][8 * (gk & 1) + 2 * e + 1], a.scale_log2e, ref));
          part[e] = skv::f2bf2(x0, x1);
          l = add_pair(part[e], l);
        }
#pragma unroll
        for (int d = 0; d < 4; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, value_operand(va, gk, d)),
                                                         __builtin_bit_cast(bf16x8, part), o[d], 0, 0, 0);
      }
    }
  };

  clear();
  if (t0 < t1) {  // workgroup-uniform
    bool missing = false;
    if constexpr (!kPaged) __syncthreads();  // every wave is past its queries in LDS
    if constexpr (kPaged) {
      const int e0 = (t0 * kTile) >> a.shift, e1 = min(t1 * kTile - 1, len - 1) >> a.shift;
      for (int e = e0 + static_cast<int>(threadIdx.x); e <= e1; e += 64 * kWaves) missing |= !valid_page(a, table[e]);
      missing = __syncthreads_or(missing);
    }
    bool any = missing;
    if (!any) {
      // Of the tiles that are seen, those that every row sees whole: w0 to w1 - 1.
      const int w0 = min(max(a.window < kNoWindow ? max(0, pmax - a.window + kTile) >> kTileShift : 0, t0), t1);
      const int w1 = min((pmin + 1) >> kTileShift, t1);
      const bool whole = w1 > w0;
      bool odd_place = false;
#pragma nounroll
      for (int end = 0; end < 2; ++end) {  // (one walk for both ends)
        if (end && whole) {
          if (t0 < w0) {
            skv::drain_and_barrier();  // every wave is past the tiles before, whose loads have come
            const int32_t id = page_of(w0);
            load_keys(w0, id, ka);
            load_values(w0, id, va);
          }
          walk_whole(w0, w1);
          odd_place = (w1 - w0) & 1;
        }
        walk(end ? whole ? w1 : t1 : t0, end || !whole ? t1 : w0, odd_place);
      }
      // NaN anywhere: a value may have reached rows that do not see it.
      // Scores past 2^24: the reference's product with the scale is rounded, the exponential's is not.
      bool odd = !(l < INFINITY) || (m != -INFINITY && fabsf(m) > 16777216.f);
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd |= o[d][r] != o[d][r];
      any = __syncthreads_or(odd);
    }
    if (any) {
      clear();
      some = false;
      skv::drain_and_barrier();
      walk_any();
    }
  }

  {
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(w[0]) + __uint_as_float(w[1]);
    const auto y = __builtin_amdgcn_permlane32_swap(some, some, false, false);
    if ((y[0] | y[1]) && m == -INFINITY) l = __builtin_nanf("");  // (all that it sees at -inf: its sum is 0 / 0)
  }
  // (read again: the arguments that only the end needs would be held in registers)
  auto again = (const __attribute__((address_space(4))) Args*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(again));
  const Row x = own_row();
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool up = (pos >> (16 * d + r)) & 1, down = (neg >> (16 * d + r)) & 1;
      if (up || down) o[d][r] = up && down ? __builtin_nanf("") : up ? INFINITY : -INFINITY;
    }
  // Out through LDS, a row (16 lanes) at a time: as bf16, or for the join in fp32, 64 dims after the others.
  skv::drain_and_barrier();  // (a pipeline's last loads may be on their way)
  u32x4* own = (wave < 2 ? ka : wave < 4 ? kb : wave < 6 ? va : vb) + (wave & 1) * 512;
  if (it.splits == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // (a sum of zero: it sees nothing)
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        reinterpret_cast<u32x2*>(own + x.li * 16 + ((4 * d + r) ^ (x.li & 15)))[x.half] =
            u32x2{skv::f2bf2(o[d][4 * r] * inv, o[d][4 * r + 1] * inv),
                  skv::f2bf2(o[d][4 * r + 2] * inv, o[d][4 * r + 3] * inv)};
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    uint16_t* out = again->out;
    const int Hq = a.H * G;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 4), at = r0 + wave * kRowsWave + r, t = __shfl(x.t, r);
      if (at < R)
        // (fewer than 2^30 rows of all heads)
        *reinterpret_cast<u32x4*>(out + (static_cast<int64_t>((first + t) * Hq + h * G + at - t * G) * kD +
                                         8 * (lane & 15))) = own[r * 16 + ((lane & 15) ^ (r & 15))];
    }
  } else {
    const int64_t from = (static_cast<int64_t>(it.part) * a.H + h) * kRowsTile + wave * kRowsWave;
    if (x.query && x.half == 0) {
      again->rows_ml[2 * (from + x.li)] = m;
      again->rows_ml[2 * (from + x.li) + 1] = l;
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
#pragma unroll
      for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x16& w = o[2 * side + d];
          own[x.li * 16 + ((8 * d + 2 * r + x.half) ^ (x.li & 15))] =
              __builtin_bit_cast(u32x4, f32x4{w[4 * r], w[4 * r + 1], w[4 * r + 2], w[4 * r + 3]});
        }
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 4);
        if (r0 + wave * kRowsWave + r < R)
          *reinterpret_cast<u32x4*>(again->rows_o + (from + r) * kD + 64 * side + 4 * (lane & 15)) =
              own[r * 16 + ((lane & 15) ^ (r & 15))];
      }
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    }
  }
  clear_rows(a, 0, it.begin, blockIdx.x, gridDim.x);
  clear_rows(a, it.end, a.N, blockIdx.x, gridDim.x);
}

// The cut row tiles' rows: 8 of them a workgroup at a time, 32 lanes of four dims each, or one with many parts; before
// them, with few_wgs workgroups, the few-row form's.
constexpr int kManyParts = 16;
template <bool kPaged, int kRowsTile>
__global__ void __launch_bounds__(256) rows_join_kernel(Args a, int few_wgs) {
  __shared__ f32x4 acc_lds[8][32];
  if constexpr (kPaged) {
    if (static_cast<int>(blockIdx.x) < few_wgs) {  // workgroup-uniform
      few_join(a, acc_lds);
      return;
    }
  }
  const int lane = threadIdx.x & 63;
  Seq s{0, 0, 0};
  Work w{0, 0, 0};
  if (lane < a.B) {
    s = seq_of<kPaged>(a, lane);
    w = work_of<kPaged, kRowsTile>(a, s);
  }
  const Share share = share_tiles<kPaged, kRowsTile>(a, lane, s, w);
  int before = 0;     // units before these
  int64_t parts = 0;  // cut row tiles' shares before these, of one kv head
  int unit = static_cast<int>(blockIdx.x) - few_wgs;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    if (b0) {
      s = Seq{0, 0, 0};
      w = Work{0, 0, 0};
      if (b0 + lane < a.B) {
        s = seq_of<kPaged>(a, b0 + lane);
        w = work_of<kPaged, kRowsTile>(a, s);
      }
    }
    int shares, cuts = 0;
    if (__any(w.tiles >= share.cut)) Cut<kRowsTile>{a, s, w, share}.count(shares, cuts);
    for (uint64_t cut = __ballot(cuts > 0); cut; cut &= cut - 1) {
      const int x = __builtin_ctzll(cut);
      const Cut<kRowsTile> c{a, lane_seq(s, x),
                             Work{__builtin_amdgcn_readlane(w.rts, x), __builtin_amdgcn_readlane(w.tiles, x),
                                  __builtin_amdgcn_readlane(w.least, x)},
                             share};
      const int row0 = c.whole() * kRowsTile;  // the rows behind are cut
      const int rows = (c.s.n * a.G - row0) * a.H;
      const bool many = c.shares_of(c.w.least) > kManyParts;
      const int units = many ? rows : (rows + 7) / 8;
      for (; unit < before + units; unit += static_cast<int>(gridDim.x) - few_wgs) {
        const int at = many ? unit - before : 8 * (unit - before) + static_cast<int>(threadIdx.x >> 5);
        if (at >= rows) continue;
        const int row = row0 + at / a.H, h = at % a.H;
        const int rt = row / kRowsTile, t = row / a.G;
        int splits;
        const int64_t part = parts + c.place(rt, splits);
        if ((part + splits) * a.H > a.parts) continue;
        const int64_t from = (part * a.H + h) * kRowsTile + row - rt * kRowsTile;
        const int64_t stride = static_cast<int64_t>(a.H) * kRowsTile;
        uint16_t* out = a.out + (static_cast<int64_t>(c.s.first + t) * a.H * a.G + h * a.G + row - t * a.G) * kD;
        if (many) {
          __syncthreads();  // (acc_lds)
          join_parts(a.rows_o, a.rows_ml, from, stride, splits, out, acc_lds);
          continue;
        }
        const int d = 4 * (threadIdx.x & 31);
        float m = -INFINITY, l = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < splits; ++i) m = fmaxf(m, a.rows_ml[2 * (from + i * stride)]);
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 4
        for (int i = 0; i < splits; ++i) {
          const int64_t p = from + i * stride;
          const float mi = a.rows_ml[2 * p], li = a.rows_ml[2 * p + 1];
          l += m > -INFINITY && mi == -INFINITY ? 0.f : li * __builtin_amdgcn_exp2f(mi == -INFINITY ? 0.f : mi - ref);
          acc += lowered(*reinterpret_cast<const f32x4*>(a.rows_o + p * kD + d), __builtin_amdgcn_exp2f(mi - ref));
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<u32x2*>(out + d) =
            u32x2{skv::f2bf2(acc[0] * inv, acc[1] * inv), skv::f2bf2(acc[2] * inv, acc[3] * inv)};
      }
      before += units;
      parts += __builtin_amdgcn_readlane(cuts, x);
    }
  }
}

constexpr int64_t kMaxThreads = int64_t{1} << 32;  // of a launch

// The scale's magnitude in units of log2: positive, so that a hidden key's -inf stays one, and as small as that can be, so
// that a scale of zero makes 2^-21 of the largest product.
float log2_scale(float scale) {
  return std::max(std::fabs(scale) * 1.44269504088896340736f, std::numeric_limits<float>::denorm_min());
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// How a call is cut up, from its sizes alone (the lengths are on the device).
struct Plan {
  int few_max = 0;   // new tokens of a sequence up to which the few-row form takes it
  int tiles = 0;     // its tiles of 16 rows
  bool whole = false;
  int R = 0;         // its rows of a chunk
  int64_t few_grid = 0, few_parts = 0, few_join = 0;
  int waves = 0;     // of the other's workgroups; 0: it has nothing to do
  bool splits = false;
  int64_t rows_grid = 0, rows_parts = 0, rows_join = 0;
  int64_t bytes() const { return (few_parts + rows_parts) * (kD + 2) * 4; }
};

// Waves of a workgroup: 8 where rows see many keys, so that a tile's way from memory serves 256 rows (and each CU's one
// workgroup hides less of what surrounds its walk), and there are rows enough; else 4. Measured (MI355X, us on the device,
// 4 waves / 8, 4 query heads on each of 8 kv heads, prompts packed): 64 of 256 tokens 138 / 159, 16 of 1024 221 / 220, 8 of
// 2048 331 / 325, 4 of 4096 560 / 545, one of 8192 530 / 500, of 2048 59 / 64 (256 workgroups of 8).
int waves_of(int64_t rows, int64_t most, int64_t keys) {
  return most >= 256 && (keys >= 4096 ? rows >= 16384 : keys >= 1024 && rows >= 131072) ? 8 : 4;
}

Plan plan_of(bool paged, int64_t N, int64_t B, int H, int G, int max_new, int64_t cap, int window) {
  Plan p;
  max_new = static_cast<int>(std::min<int64_t>(max_new, N));
  const int64_t keys = window ? std::min<int64_t>(cap, static_cast<int64_t>(window) + max_new - 1) : cap;
  const bool all_few = paged && static_cast<int64_t>(max_new) * G <= 32;
  // One sequence beside whose rows there are no others has one form, and so have tables of a few tiles: one launch, no join
  // (up to 25 new tokens of each of 24 sequences of up to 473: 32 -> 25 us). Single tokens and drafts among them then take
  // bf16 probabilities, as the pieces beside them do: 2^-9 of the values' mean magnitude beside the 2^-9 of the output's own
  // rounding, where the few-row form has 2^-17. The others': up to 16 rows, one tile.
  if (all_few) p.few_max = max_new;
  else if (paged && B > 1 && cap >= (kMinTiles + kShareGain) * kTile) p.few_max = 16 / G;
  if (p.few_max) {
    p.R = p.few_max * G;
    p.tiles = p.R <= 16 ? 1 : 2;
    // groups that a query can see: both ends of a window may lie inside one
    const int64_t groups = std::min<int64_t>((cap + kGroup - 1) / kGroup, (keys + kGroup - 1) / kGroup + 2);
    p.whole = all_few && groups <= whole_groups(p.tiles, B * H);
    if (p.whole) {
      p.few_grid = B * H;
    } else {
      const int64_t each = (groups + kMinGroups - 1) / kMinGroups;
      const int64_t slots = std::min<int64_t>(B * each, (target_chunks(p.R) + H - 1) / H + B);
      p.few_grid = slots * H;
      p.few_parts = p.few_grid * p.R;
      p.few_join = B * H * p.R;
    }
  }
  if (!all_few) {
    p.waves = waves_of(N * G * H, static_cast<int64_t>(max_new) * G, paged ? keys : std::min(keys, N / B));
    const int tile_rows = p.waves * kRowsWave, at_once = resident(tile_rows);
    const int64_t items = static_cast<int64_t>(H) * (N * G / tile_rows + std::min(B, N));
    const int64_t tiles = (cap + kTile - 1) / kTile;
    // Prompts that fill the chip by their row tiles are not cut.
    p.splits = tiles >= kMinTiles + kShareGain && (paged || items < 2 * at_once);
    p.rows_grid = items + (p.splits ? 2 * at_once : 0);
    if (p.splits) {
      const int64_t cut = std::min<int64_t>(4 * at_once, items * ((tiles + kMinTiles - 1) / kMinTiles));
      // (what is cut has more tiles than a share, so that its shares are at most twice the workgroups that the chip holds;
      // as many again for what the plan rounds: a share without a place would leave its rows)
      p.rows_parts = (cut + H) * tile_rows;
      p.rows_join = std::min<int64_t>(2048, N * G * H);
    }
  }
  return p;
}

bool sizes_ok(int N, int B, int Hq, int H, int max_new, int window) {
  return N >= 1 && B >= 1 && H >= 1 && Hq >= H && Hq % H == 0 && max_new >= 1 && window >= 0 && B <= (1 << 24) &&
         static_cast<int64_t>(N) * Hq < (int64_t{1} << 30);
}

template <bool kPaged>
int launch(const char* what, Args a, const Plan& p, void* workspace, int64_t workspace_bytes, hipStream_t s) {
  const int64_t need = p.bytes();
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) {
    skv_set_error("%s: workspace of %lld bytes (%lld needed, 16-byte aligned)", what, (long long)workspace_bytes,
                  (long long)need);
    return SKV_EINVAL;
  }
  const int threads = p.few_max ? few_threads(p.whole) : 0;
  if (p.few_grid * threads >= kMaxThreads || (p.few_join + p.rows_join) * 256 >= kMaxThreads ||
      p.rows_grid * 64 * p.waves >= kMaxThreads) {
    skv_set_error("%s: batch=%d rows=%d q_heads=%d", what, a.B, a.N, a.H * a.G);
    return SKV_EUNSUPPORTED;
  }
  a.few_max = p.few_max;
  a.R = p.R;
  a.target = target_chunks(p.R);
  a.splits = p.splits;
  a.parts = p.waves ? p.rows_parts / (p.waves * kRowsWave) : 0;
  a.few_o = static_cast<float*>(workspace);
  a.rows_o = a.few_o ? a.few_o + p.few_parts * kD : nullptr;
  a.few_ml = a.rows_o ? a.rows_o + p.rows_parts * kD : nullptr;
  a.rows_ml = a.few_ml ? a.few_ml + p.few_parts * 2 : nullptr;
  if constexpr (kPaged) {
    if (p.few_max) {
      const dim3 g(static_cast<unsigned>(p.few_grid)), t(threads);
      if (p.whole) {
        if (p.tiles == 1) hipLaunchKernelGGL((few_kernel<1, true>), g, t, 0, s, a, true);
        else hipLaunchKernelGGL((few_kernel<2, true>), g, t, 0, s, a, true);
      } else {
        if (p.tiles == 1) hipLaunchKernelGGL((few_kernel<1, false>), g, t, 0, s, a, !p.waves);
        else hipLaunchKernelGGL((few_kernel<2, false>), g, t, 0, s, a, !p.waves);
        if (!p.splits) hipLaunchKernelGGL(few_join_kernel, dim3(static_cast<unsigned>(p.few_join)), dim3(256), 0, s, a);
      }
    }
  }
  const dim3 g(static_cast<unsigned>(p.rows_grid)), t(64 * p.waves);
  const dim3 join(static_cast<unsigned>(p.few_join + p.rows_join));
  const int few_wgs = static_cast<int>(p.few_join);
  if (p.waves == 4) {
    hipLaunchKernelGGL((rows_kernel<kPaged, 4>), g, t, 0, s, a);
    if (p.splits) hipLaunchKernelGGL((rows_join_kernel<kPaged, 128>), join, dim3(256), 0, s, a, few_wgs);
  } else if (p.waves == 8) {
    hipLaunchKernelGGL((rows_kernel<kPaged, 8>), g, t, 0, s, a);
    if (p.splits) hipLaunchKernelGGL((rows_join_kernel<kPaged, 256>), join, dim3(256), 0, s, a, few_wgs);
  }
  return skv_check_launch(what);
}

}  // namespace

extern "C" int64_t skv_paged_attn_workspace_bytes(int rows, int batch_size, int q_heads, int kv_heads, int max_new,
                                                  int width, int page, int window) {
  if (!sizes_ok(rows, batch_size, q_heads, kv_heads, max_new, window) || width < 1 || page < 1) return 0;
  return plan_of(true, rows, batch_size, kv_heads, q_heads / kv_heads, max_new, static_cast<int64_t>(width) * page,
                 window)
      .bytes();
}

extern "C" int skv_paged_attn(const uint16_t* q, int64_t q_stride_t, int64_t q_stride_h, const uint16_t* k_pages,
                              const uint16_t* v_pages, int64_t p_stride_p, int64_t p_stride_h, int64_t p_stride_s,
                              int pages, int page, const int32_t* table, int64_t table_stride, int width,
                              const int32_t* lengths, const int32_t* cu, int rows, int batch_size, int q_heads,
                              int kv_heads, int max_new, float scale, int window, uint16_t* out, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const char* what = "paged_attn";
  if (!q || !k_pages || !v_pages || !table || !lengths || !out) {
    skv_set_error("%s: null pointer", what);
    return SKV_EINVAL;
  }
  int shift = 4;
  while (shift < 8 && (1 << shift) < page) ++shift;
  if (page != 1 << shift) {
    skv_set_error("%s: page=%d (16, 32, 64, 128 or 256 tokens)", what, page);
    return SKV_EUNSUPPORTED;
  }
  if (!sizes_ok(rows, batch_size, q_heads, kv_heads, max_new, window) || width < 1 || pages < 1 ||
      static_cast<int64_t>(width) * page > (1 << 30) || (batch_size > 1 && table_stride < 0) ||
      (!cu && rows != batch_size)) {
    skv_set_error("%s: rows=%d batch=%d q_heads=%d kv_heads=%d max_new=%d window=%d pages=%d width=%d", what, rows,
                  batch_size, q_heads, kv_heads, max_new, window, pages, width);
    return SKV_EINVAL;
  }
  if (!std::isfinite(log2_scale(scale))) {
    skv_set_error("%s: scale=%g", what, static_cast<double>(scale));
    return SKV_EINVAL;
  }
  if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 16) ||
      ((q_stride_t | q_stride_h | p_stride_p | p_stride_h | p_stride_s) & 7)) {
    skv_set_error("%s: rows of q, of the pages and of out must be 16-byte aligned", what);
    return SKV_EINVAL;
  }
  if (p_stride_s < 0 || p_stride_s > (1 << 24)) {
    skv_set_error("%s: tokens %lld elements apart (at most 2^24)", what, (long long)p_stride_s);
    return SKV_EUNSUPPORTED;
  }
  const int cap = width * page;
  const Plan p = plan_of(true, rows, batch_size, kv_heads, q_heads / kv_heads, cu ? max_new : 1, cap, window);
  Args a{};
  a.q = q;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k = k_pages;
  a.v = v_pages;
  a.k_sp = a.v_sp = p_stride_p;
  a.k_sh = a.v_sh = p_stride_h;
  a.k_st = a.v_st = p_stride_s;
  a.table = table;
  a.t_stride = table_stride;
  a.lengths = lengths;
  a.cu = cu;
  a.out = out;
  a.N = rows;
  a.B = batch_size;
  a.H = kv_heads;
  a.G = q_heads / kv_heads;
  a.cap = cap;
  a.pages = pages;
  a.shift = shift;
  a.window = window ? std::min(window, kNoWindow) : kNoWindow;
  a.max_new = cu ? std::min(max_new, rows) : 1;
  a.scale_log2e = log2_scale(scale);
  a.negative = scale < 0.f;
  return launch<true>(what, a, p, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int64_t skv_packed_attn_workspace_bytes(int rows, int batch_size, int q_heads, int kv_heads, int window) {
  if (!sizes_ok(rows, batch_size, q_heads, kv_heads, rows, window)) return 0;
  return plan_of(false, rows, batch_size, kv_heads, q_heads / kv_heads, rows, rows, window).bytes();
}

extern "C" int skv_packed_attn(const uint16_t* q, int64_t q_stride_t, int64_t q_stride_h, const uint16_t* k,
                               int64_t k_stride_t, int64_t k_stride_h, const uint16_t* v, int64_t v_stride_t,
                               int64_t v_stride_h, const int32_t* cu, int rows, int batch_size, int q_heads,
                               int kv_heads, float scale, int window, uint16_t* out, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  const char* what = "packed_attn";
  if (!q || !k || !v || !cu || !out) {
    skv_set_error("%s: null pointer", what);
    return SKV_EINVAL;
  }
  if (!sizes_ok(rows, batch_size, q_heads, kv_heads, rows, window)) {
    skv_set_error("%s: rows=%d batch=%d q_heads=%d kv_heads=%d window=%d", what, rows, batch_size, q_heads, kv_heads,
                  window);
    return SKV_EINVAL;
  }
  if (!std::isfinite(log2_scale(scale))) {
    skv_set_error("%s: scale=%g", what, static_cast<double>(scale));
    return SKV_EINVAL;
  }
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) ||
      ((q_stride_t | q_stride_h | k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7)) {
    skv_set_error("%s: rows of q, k, v and out must be 16-byte aligned", what);
    return SKV_EINVAL;
  }
  if (k_stride_t < 0 || k_stride_t > (1 << 24) || v_stride_t < 0 || v_stride_t > (1 << 24)) {
    skv_set_error("%s: tokens of k or v %lld or %lld elements apart (at most 2^24)", what, (long long)k_stride_t,
                  (long long)v_stride_t);
    return SKV_EUNSUPPORTED;
  }
  const Plan p = plan_of(false, rows, batch_size, kv_heads, q_heads / kv_heads, rows, rows, window);
  Args a{};
  a.q = q;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k = k;
  a.v = v;
  a.k_sh = k_stride_h;
  a.v_sh = v_stride_h;
  a.k_st = k_stride_t;
  a.v_st = v_stride_t;
  a.cu = cu;
  a.out = out;
  a.N = rows;
  a.B = batch_size;
  a.H = kv_heads;
  a.G = q_heads / kv_heads;
  a.cap = rows;
  a.pages = 1;
  a.window = window ? std::min(window, kNoWindow) : kNoWindow;
  a.max_new = rows;
  a.scale_log2e = log2_scale(scale);
  a.negative = scale < 0.f;
  return launch<false>(what, a, p, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}
