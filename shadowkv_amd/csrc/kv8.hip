// The 8-bit KV cache: tokens quantised as they are written, cached rows read back.
//
// A cache of keys or values is e4m3 codes [B, H, cap, 128] and one fp32 scale per block of tokens and head;
// a value is code * scale. A written scale is a power of two, the smallest 2^e (e >= -126) under which the
// block's largest finite magnitude is at most 448 (e4m3's largest): the format floats, so a power of two costs
// none of its 4 significant bits, code * scale is exact in bf16, and rows encoded again under a larger scale
// change only where they become subnormal.
//
// Bound: HBM bytes (written rows 2 + 1 per element, read rows 1 + 2); a decoded token is a launch. Measured (MI355X, 8
// heads): 122880 tokens written in 140 us, 5.4 TB/s (a large copy has 4.7); 100003 rows read in 63, 4.9 TB/s; a
// token of each of 8 sequences written in 4.4 on the device (10.8 a call from Python).
#include "skv_common.h"

namespace {

using skv::u32x4;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kD = 128;
constexpr int kThreads = 256;
constexpr int kRowsPass = kThreads / 16;  // rows that a workgroup writes at once, 16 lanes of 8 elements each

struct WriteArgs {
  const uint16_t* x[2];  // keys, values
  int64_t x_sb[2], x_sh[2], x_st[2];
  uint8_t* codes[2];
  float* scale[2];
  int64_t c_sb, c_sh, c_ss, s_sb, s_sh;
  const int32_t* start;
  const int32_t* counts;
  int H, T, cap, blocks;  // blocks: that T rows can touch
};

// 2^e as fp32 for the largest finite magnitude amax (bf16 bits): the smallest with amax <= 448 * 2^e. Its
// exponent field is amax's less 8, one more where the fraction passes 1.75 = 448 / 256.
__device__ __forceinline__ float scale_for(uint32_t amax) {
  const int e = static_cast<int>(amax >> 7) - 8 + ((amax & 127u) > 96u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}

// Eight fp32 as e4m3 codes, to nearest even; what is not finite as NaN.
__device__ __forceinline__ u32x2 encode8(const float (&f)[8]) {
  u32x2 o;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float g[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = f[4 * w + e];
      g[e] = __builtin_fabsf(x) < INFINITY ? x : __builtin_nanf("");
    }
    int d = __builtin_amdgcn_cvt_pk_fp8_f32(g[0], g[1], 0, false);
    o[w] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(g[2], g[3], d, true));
  }
  return o;
}

__device__ __forceinline__ void decode4(uint32_t w, float* f) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
}

// A workgroup owns one block of one sequence, head and cache (keys or values), so that a block's scale has
// one writer: no atomics, the same result in any order. Heads run fastest over the grid: the rows of a
// projection's output hold the heads side by side.
template <int kPasses>  // block / 16
__global__ void __launch_bounds__(kThreads) write_kernel(WriteArgs a) {
  constexpr int kBlock = kPasses * kRowsPass;
  __shared__ uint32_t part[kThreads / 64];
  int i = blockIdx.x;
  const int h = i % a.H;
  i /= a.H;
  const int w = i % a.blocks;
  i /= a.blocks;
  const int which = i & 1, b = i >> 1;
  const int64_t st = a.start[b];
  const int64_t n = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  const int64_t end = min(st + n, static_cast<int64_t>(a.cap));
  if (st < 0) return;
  const int64_t lo = (st / kBlock + w) * kBlock;  // the block's first position
  if (lo >= end || st >= end) return;             // workgroup-uniform

  const int row = threadIdx.x >> 4, c = threadIdx.x & 15;
  const uint16_t* x = a.x[which] + b * a.x_sb[which] + h * a.x_sh[which] + 8 * c;
  u32x4 v[kPasses];
  bool fresh[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int64_t at = lo + p * kRowsPass + row;
    fresh[p] = at >= st && at < end;
    v[p] = skv::load16_or_zero(x + (min(max(at, st), end - 1) - st) * a.x_st[which], fresh[p]);
  }
  uint32_t top = 0;
#pragma unroll
  for (int p = 0; p < kPasses; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t l = v[p][e] & 0x7fffu, u = (v[p][e] >> 16) & 0x7fffu;
      top = max(top, l < 0x7f80u ? l : 0u);
      top = max(top, u < 0x7f80u ? u : 0u);
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, 64)));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max(max(part[0], part[1]), max(part[2], part[3]));

  float* sp = a.scale[which] + b * a.s_sb + h * a.s_sh + lo / kBlock;
  const bool begun = lo < st;  // older rows share the block and its scale
  const float was = begun ? *sp : 0.f;
  const float s = fmaxf(was, scale_for(top));
  const float inv = 1.f / s;
  // (uniform; of a held scale that no write made: the product with the reciprocal would miss ties)
  const bool divide = (__float_as_uint(s) & 0x7fffffu) != 0;
  const bool again = begun && was < s;
  const float ratio = was * inv;
  uint8_t* dst = a.codes[which] + b * a.c_sb + h * a.c_sh + 8 * c;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int64_t at = lo + p * kRowsPass + row;
    u32x2* d = reinterpret_cast<u32x2*>(dst + at * a.c_ss);
    float f[8];
    if (fresh[p]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = skv::bf_lo(v[p][e]) * inv;
        f[2 * e + 1] = skv::bf_hi(v[p][e]) * inv;
      }
      if (divide)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[2 * e] = skv::bf_lo(v[p][e]) / s;
          f[2 * e + 1] = skv::bf_hi(v[p][e]) / s;
        }
      *d = encode8(f);
    } else if (again && at < st) {
      const u32x2 old = *d;
      decode4(old[0], f);
      decode4(old[1], f + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= ratio;
      *d = encode8(f);
    }
  }
  __syncthreads();  // every thread has read the block's old scale
  if (threadIdx.x == 0) *sp = s;
}

struct ReadArgs {
  const uint8_t* codes;
  const float* scale;
  int64_t c_sb, c_sh, c_ss, s_sb, s_sh;
  const int64_t* ids;  // [B, H, chunks] or null
  uint16_t* out;       // [B, H, rows, 128]
  int64_t start;
  int H, cap, block, chunk, chunks, rows, groups;  // chunks: that begin inside the cache
};

constexpr int kReadRows = 128;  // rows of a workgroup, 8 lanes of 16 elements each, 4 in flight a thread

__global__ void __launch_bounds__(kThreads) read_kernel(ReadArgs a) {
  const int bh = blockIdx.x / a.groups, grp = blockIdx.x - bh * a.groups;
  const int b = bh / a.H, h = bh - b * a.H;
  const uint8_t* src = a.codes + b * a.c_sb + h * a.c_sh;
  const float* sc = a.scale + b * a.s_sb + h * a.s_sh;
  const int c = threadIdx.x & 7;
  constexpr int kEach = kReadRows * 8 / kThreads;
  u32x4 v[kEach];
  float s[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int r = min(grp * kReadRows + i * (kThreads / 8) + static_cast<int>(threadIdx.x >> 3), a.rows - 1);
    int64_t at = a.start + r;
    bool ok = true;
    if (a.ids) {
      const int64_t id = a.ids[static_cast<int64_t>(bh) * (a.rows / a.chunk) + r / a.chunk];
      ok = id >= 0 && id < a.chunks;
      at = (ok ? id : 0) * a.chunk + r % a.chunk;
    }
    ok = ok && at < a.cap;
    if (!ok) at = 0;
    v[i] = skv::load16_or_zero(src + at * a.c_ss + 16 * c, ok);
    s[i] = sc[at / a.block];
    if (!ok) s[i] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int r = grp * kReadRows + i * (kThreads / 8) + static_cast<int>(threadIdx.x >> 3);
    if (r >= a.rows) continue;
    u32x4 o[2];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float f[4];
      decode4(v[i][w], f);
      o[w >> 1][2 * (w & 1)] = skv::f2bf2(f[0] * s[i], f[1] * s[i]);
      o[w >> 1][2 * (w & 1) + 1] = skv::f2bf2(f[2] * s[i], f[3] * s[i]);
    }
    u32x4* d = reinterpret_cast<u32x4*>(a.out + (static_cast<int64_t>(bh) * a.rows + r) * kD + 16 * c);
    d[0] = o[0];
    d[1] = o[1];
  }
}

constexpr int64_t kMaxThreads = int64_t{1} << 32;  // of a launch
constexpr int kMaxTokens = 1 << 30;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool block_ok(int block) { return block == 16 || block == 32 || block == 64 || block == 128; }

}  // namespace

extern "C" int skv_kv8_write(const uint16_t* k, int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_t,
                             const uint16_t* v, int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_t, uint8_t* k8,
                             uint8_t* v8, int64_t c_stride_b, int64_t c_stride_h, int64_t c_stride_s, float* k_scale,
                             float* v_scale, int64_t s_stride_b, int64_t s_stride_h, const int32_t* start,
                             const int32_t* counts, int batch_size, int heads, int rows, int cap, int block,
                             void* stream) {
  const char* what = "kv8_write";
  if (!k || !v || !k8 || !v8 || !k_scale || !v_scale || !start) {
    skv_set_error("%s: null pointer", what);
    return SKV_EINVAL;
  }
  if (batch_size < 1 || heads < 1 || rows < 1 || rows > kMaxTokens || cap < 1 || cap > kMaxTokens) {
    skv_set_error("%s: batch=%d heads=%d rows=%d cap=%d", what, batch_size, heads, rows, cap);
    return SKV_EINVAL;
  }
  if (!block_ok(block)) {
    skv_set_error("%s: block=%d (16, 32, 64 or 128 tokens)", what, block);
    return SKV_EUNSUPPORTED;
  }
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(k8, 16) || !aligned(v8, 16) || !aligned(k_scale, 4) ||
      !aligned(v_scale, 4) || k_stride_b % 8 || k_stride_h % 8 || k_stride_t % 8 || v_stride_b % 8 ||
      v_stride_h % 8 || v_stride_t % 8 || c_stride_b % 16 || c_stride_h % 16 || c_stride_s % 16) {
    skv_set_error("%s: rows of k, v and the caches must be 16-byte aligned", what);
    return SKV_EINVAL;
  }
  const int64_t blocks = (static_cast<int64_t>(rows) + block - 2) / block + 1;
  const int64_t grid = blocks * heads * batch_size * 2;
  if (grid * kThreads >= kMaxThreads) {
    skv_set_error("%s: batch=%d heads=%d rows=%d", what, batch_size, heads, rows);
    return SKV_EUNSUPPORTED;
  }
  WriteArgs a{{k, v}, {k_stride_b, v_stride_b}, {k_stride_h, v_stride_h}, {k_stride_t, v_stride_t}, {k8, v8},
              {k_scale, v_scale}, c_stride_b, c_stride_h, c_stride_s, s_stride_b, s_stride_h, start, counts, heads,
              rows, cap, static_cast<int>(blocks)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 g(static_cast<unsigned>(grid)), t(kThreads);
  switch (block) {
    case 16: hipLaunchKernelGGL(write_kernel<1>, g, t, 0, s, a); break;
    case 32: hipLaunchKernelGGL(write_kernel<2>, g, t, 0, s, a); break;
    case 64: hipLaunchKernelGGL(write_kernel<4>, g, t, 0, s, a); break;
    default: hipLaunchKernelGGL(write_kernel<8>, g, t, 0, s, a); break;
  }
  return skv_check_launch(what);
}

extern "C" int skv_kv8_read(const uint8_t* codes, int64_t c_stride_b, int64_t c_stride_h, int64_t c_stride_s,
                            const float* scale, int64_t s_stride_b, int64_t s_stride_h, const int64_t* chunk_ids,
                            int chunk_size, int64_t start, uint16_t* out, int batch_size, int heads, int rows, int cap,
                            int block, void* stream) {
  const char* what = "kv8_read";
  if (!codes || !scale || !out) {
    skv_set_error("%s: null pointer", what);
    return SKV_EINVAL;
  }
  if (batch_size < 1 || heads < 1 || rows < 1 || rows > kMaxTokens || cap < 1 || cap > kMaxTokens || start < 0 ||
      (chunk_ids ? chunk_size < 1 || rows % chunk_size || start : start > cap - rows)) {
    skv_set_error("%s: batch=%d heads=%d start=%lld rows=%d chunk=%d cap=%d", what, batch_size, heads,
                  (long long)start, rows, chunk_size, cap);
    return SKV_EINVAL;
  }
  if (!block_ok(block)) {
    skv_set_error("%s: block=%d (16, 32, 64 or 128 tokens)", what, block);
    return SKV_EUNSUPPORTED;
  }
  if (!aligned(codes, 16) || !aligned(scale, 4) || !aligned(out, 16) || c_stride_b % 16 || c_stride_h % 16 ||
      c_stride_s % 16) {
    skv_set_error("%s: rows of the cache and of out must be 16-byte aligned", what);
    return SKV_EINVAL;
  }
  const int64_t groups = (static_cast<int64_t>(rows) + kReadRows - 1) / kReadRows;
  const int64_t grid = groups * heads * batch_size;
  if (grid * kThreads >= kMaxThreads) {
    skv_set_error("%s: batch=%d heads=%d rows=%d", what, batch_size, heads, rows);
    return SKV_EUNSUPPORTED;
  }
  const int chunk = chunk_ids ? chunk_size : 1;
  ReadArgs a{codes, scale, c_stride_b, c_stride_h, c_stride_s, s_stride_b, s_stride_h, chunk_ids, out, start, heads,
             cap, block, chunk, static_cast<int>((static_cast<int64_t>(cap) + chunk - 1) / chunk), rows,
             static_cast<int>(groups)};
  hipLaunchKernelGGL(read_kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  return skv_check_launch(what);
}
