// Pages of a KV cache: which sequence holds which, where a step's tokens go, and the write of their rows.
//
// The free pages are a stack, the lowest sequence's first new page on its top: with need_b pages for sequence b and upto_b
// = need_0 + .. + need_b, page i of them is free[count - 1 - (upto_b - need_b + i)]. Both sums (tokens, pages) are scans
// over the sequences that stop at a bound (min(a + b, bound) is associative, so that no sum overflows), and what follows is
// flat: a new page, or a token, finds its sequence by bisection in LDS. Giving back counts the same way, so that a step's
// pages return to where they were.
//
// Bound: latency (a chain of loads, two scans, a bisection), one launch of one workgroup; the slots of many rows take a
// second one over the chip. Measured (MI355X, us on the device): one token of each of 64 sequences 4.1, given back 2.4;
// pieces of 256 sequences, 48146 tokens in pages of 16, 11.4 in two launches, given back 7.3.
#include "skv_common.h"

namespace {

using skv::u32x4;

constexpr int kD = 128;
constexpr int kSeqs = 1024;  // sequences at a time, a thread each

struct Pages {
  int32_t* table;
  int64_t stride;
  int width;
  int32_t* held;
  int32_t* free_pages;
  int cap;
  int32_t* free_count;
  int B, shift;
};

// Inclusive scan over the workgroup of min(a + b, bound); bound < 2^31, v <= bound. *total: the last one's.
__device__ __forceinline__ uint32_t scan_to(uint32_t v, uint32_t bound, uint32_t (&part)[kSeqs / 64], uint32_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(v, o);
    if (lane >= o) v = min(v + u, bound);
  }
  __syncthreads();  // (part may still be read)
  if (lane == 63) part[wave] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSeqs / 64; ++w) {
    if (w == wave) before = all;
    all = min(all + part[w], bound);
  }
  *total = all;
  return min(before + v, bound);
}

// The first i in [0, n) with x < ends[i] (ends never fall; x is below the last one's).
__device__ __forceinline__ int find(const uint32_t* ends, int n, uint32_t x) {
  int lo = 0;
  for (int len = n; len > 0;) {
    const int h = len >> 1;
    if (ends[lo + h] <= x) {
      lo += h + 1;
      len -= h + 1;
    } else {
      len = h;
    }
  }
  return min(lo, n - 1);
}

__device__ __forceinline__ int32_t slot_of(int32_t page, int at, int shift) {
  const int64_t slot = (static_cast<int64_t>(page) << shift) + (at & ((1 << shift) - 1));
  return page >= 0 && slot < (int64_t{1} << 31) ? static_cast<int32_t>(slot) : -1;
}

__device__ __forceinline__ int pages_of(int tokens, int shift) {
  return static_cast<int>((static_cast<int64_t>(tokens) + (1 << shift) - 1) >> shift);
}

// kSlots: the slots too (else slots_kernel, behind it).
template <bool kSlots>
__global__ void __launch_bounds__(kSeqs) reserve_kernel(Pages g, const int32_t* lengths, const int32_t* counts,
                                                        int rows, int32_t* cu, int32_t* totals, int32_t* slots) {
  __shared__ uint32_t part[kSeqs / 64];
  __shared__ uint32_t row_end[kSeqs], page_end[kSeqs];
  __shared__ int32_t first[kSeqs];  // pages held before, then the position of the first new token, -1: not served
  __shared__ uint32_t taken_lds;
  const int tid = threadIdx.x;
  const int count = min(max(g.free_count[0], 0), g.cap);
  const uint32_t row_bound = static_cast<uint32_t>(rows) + 1, page_bound = static_cast<uint32_t>(count) + 1;
  uint32_t rows_before = 0, pages_before = 0, taken = 0;
  if (tid == 0) {
    cu[0] = 0;
    taken_lds = 0;
  }
  for (int b0 = 0; b0 < g.B; b0 += kSeqs) {
    const int b = b0 + tid, n = min(g.B - b0, kSeqs);
    const bool is = b < g.B;
    const int len = is ? lengths[b] : 0, have = is ? min(max(g.held[b], 0), g.width) : 0;
    const uint32_t want = is ? static_cast<uint32_t>(max(counts[b], 0)) : 0u;
    uint32_t total;
    const uint32_t mine = min(want, row_bound);
    const uint32_t end = min(rows_before + scan_to(mine, row_bound, part, &total), row_bound);
    const bool fits = is && len >= 0 && (want == 0 || end < row_bound) &&  // (where the rows fit, want == mine)
                      static_cast<int64_t>(len) + want <= static_cast<int64_t>(g.width) << g.shift;
    const int last = min(rows, static_cast<int>(end));
    const uint32_t need =
        fits && want
            ? min(static_cast<uint32_t>(max(0, pages_of(len + static_cast<int>(want), g.shift) - have)), page_bound)
            : 0u;
    const int row0 = min(rows, static_cast<int>(rows_before));
    rows_before = min(rows_before + total, row_bound);
    const uint32_t upto = min(pages_before + scan_to(need, page_bound, part, &total), page_bound);
    pages_before = min(pages_before + total, page_bound);
    const bool served = fits && (need == 0 || upto <= static_cast<uint32_t>(count));
    if (is) {
      cu[b + 1] = last;
      totals[b] = served ? len + static_cast<int>(want) : 0;
      if (served && need) {
        g.held[b] = have + static_cast<int>(need);
        atomicMax(&taken_lds, upto);
      }
    }
    row_end[tid] = static_cast<uint32_t>(last);
    page_end[tid] = upto;
    first[tid] = have;
    __syncthreads();
    const uint32_t upto_taken = taken_lds;  // (those that are refused for pages come last)
    for (uint32_t i = taken + tid; i < upto_taken; i += kSeqs) {
      const int s = find(page_end, n, i);
      const uint32_t begin = s ? page_end[s - 1] : taken;
      g.table[(b0 + s) * g.stride + first[s] + (i - begin)] = g.free_pages[count - 1 - static_cast<int>(i)];
    }
    taken = upto_taken;
    if constexpr (kSlots) {
      __syncthreads();
      first[tid] = served ? len : -1;
      __syncthreads();
      const int row1 = static_cast<int>(row_end[n - 1]);
      for (int r = row0 + tid; r < row1; r += kSeqs) {
        const int s = find(row_end, n, static_cast<uint32_t>(r));
        const int begin = s ? static_cast<int>(row_end[s - 1]) : row0;
        const int at = first[s] + r - begin;
        slots[r] = first[s] >= 0 ? slot_of(g.table[(b0 + s) * g.stride + (at >> g.shift)], at, g.shift) : -1;
      }
    }
    __syncthreads();
  }
  if constexpr (kSlots)
    for (int r = min(rows, static_cast<int>(rows_before)) + tid; r < rows; r += kSeqs) slots[r] = -1;
  if (tid == 0 && taken) g.free_count[0] = count - static_cast<int>(taken);
}

// The slot of each row, from what reserve_kernel left.
__global__ void __launch_bounds__(256) slots_kernel(Pages g, const int32_t* cu, const int32_t* totals, int rows,
                                                    int32_t* slots) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= rows) return;
  if (r >= cu[g.B]) {
    slots[r] = -1;
    return;
  }
  int lo = 0, hi = g.B - 1;  // the first b with r < cu[b + 1]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > r) hi = mid;
    else lo = mid + 1;
  }
  const int total = totals[lo], at = total - cu[lo + 1] + r;
  slots[r] = total > 0 ? slot_of(g.table[lo * g.stride + (at >> g.shift)], at, g.shift) : -1;
}

// From the last sequence's last page to the first one's first, which comes to lie on top. Entries below zero are no pages:
// they are cleared and not given back.
__global__ void __launch_bounds__(kSeqs) release_kernel(Pages g, int32_t* lengths, const int32_t* keep) {
  __shared__ uint32_t part[kSeqs / 64];
  __shared__ uint32_t page_end[kSeqs];
  __shared__ int32_t first[kSeqs];
  constexpr uint32_t kBound = 0x7fffffffu;
  constexpr int kEach = 4;  // entries a thread and scan (some 4800 pages: 7.3 us; one 8.0, eight 9.4)
  const int tid = threadIdx.x;
  const int count = min(max(g.free_count[0], 0), g.cap);
  int64_t top = count;
  for (int b0 = (g.B - 1) / kSeqs * kSeqs; b0 >= 0; b0 -= kSeqs) {
    const int b = b0 + tid, n = min(g.B - b0, kSeqs);
    const bool is = b < g.B;
    const int k = is ? keep[b] : -1, left = is ? min(max(lengths[b], 0), k) : 0;
    const int have = is ? min(max(g.held[b], 0), g.width) : 0;
    const int stay = k < 0 ? have : min(have, pages_of(left, g.shift));
    uint32_t total;
    page_end[tid] = scan_to(static_cast<uint32_t>(have - stay), kBound, part, &total);
    first[tid] = stay;
    if (k >= 0) {
      lengths[b] = left;
      if (stay < have) g.held[b] = stay;
    }
    __syncthreads();
    for (int64_t end = total; end > 0; end -= kEach * kSeqs) {
      int32_t* entry[kEach];
      int32_t id[kEach];
      uint32_t mine = 0, pages;
      const int64_t last = end - 1 - kEach * tid;
      int s = last < 0 ? 0 : find(page_end, n, static_cast<uint32_t>(last));
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int64_t i = last - e;
        while (s && i < page_end[s - 1]) --s;
        entry[e] = i < 0 ? nullptr : g.table + (b0 + s) * g.stride + first[s] + (i - (s ? page_end[s - 1] : 0));
      }
#pragma unroll
      for (int e = 0; e < kEach; ++e) id[e] = entry[e] ? *entry[e] : -1;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (entry[e]) *entry[e] = -1;
        mine += id[e] >= 0;
      }
      int64_t to = top + scan_to(mine, kBound, part, &pages) - mine;
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (id[e] >= 0) {
          if (to < g.cap) g.free_pages[to] = id[e];
          ++to;
        }
      top += pages;
    }
  }
  if (tid == 0 && top > count) g.free_count[0] = static_cast<int>(min(top, static_cast<int64_t>(g.cap)));
}

struct WriteArgs {
  const uint16_t* k;
  int64_t k_st, k_sh;
  const uint16_t* v;
  int64_t v_st, v_sh;
  uint16_t* k_pages;
  uint16_t* v_pages;
  int64_t p_sp, p_sh, p_ss;
  const int32_t* slots;
  int64_t n;  // rows * heads * 16
  int heads, shift;
  int64_t slots_end;
};

// Bound: HBM, 1 KB a token and head. 16 bytes of a key and of its value a thread: no more of them is needed in flight
// (22362 tokens of 8 heads, 181 MB, 38 us from memory: 4.8 TB/s, where a large copy has 5.1).
__global__ void __launch_bounds__(256) write_kernel(WriteArgs a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.n) return;
  const uint32_t rh = static_cast<uint32_t>(i >> 4), c = 8 * (static_cast<uint32_t>(i) & 15);
  const uint32_t r = rh / static_cast<uint32_t>(a.heads), h = rh - r * static_cast<uint32_t>(a.heads);
  const int32_t slot = a.slots[r];
  if (slot < 0 || slot >= a.slots_end) return;
  const int64_t to = (slot >> a.shift) * a.p_sp + h * a.p_sh + (slot & ((1 << a.shift) - 1)) * a.p_ss + c;
  const u32x4 k = *reinterpret_cast<const u32x4*>(a.k + r * a.k_st + h * a.k_sh + c);
  const u32x4 v = *reinterpret_cast<const u32x4*>(a.v + r * a.v_st + h * a.v_sh + c);
  *reinterpret_cast<u32x4*>(a.k_pages + to) = k;
  *reinterpret_cast<u32x4*>(a.v_pages + to) = v;
}

int shift_of(int page) {  // of 16, 32, 64, 128 and 256; -1 for others
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

// Rows up to which the one workgroup that plans a step writes its slots too (256 sequences, 4096 rows: 7.0 us on the
// device and 11.0 a call, with a second launch 7.3 and 13.9).
constexpr int kOneLaunchRows = 4096;

int check_pages(const char* what, const Pages& g, int page) {
  if (!g.table || !g.held || !g.free_pages || !g.free_count) {
    skv_set_error("%s: null pointer", what);
    return SKV_EINVAL;
  }
  if (g.shift < 0) {
    skv_set_error("%s: page=%d (16, 32, 64, 128 or 256 tokens)", what, page);
    return SKV_EUNSUPPORTED;
  }
  if (g.B < 1 || g.width < 1 || static_cast<int64_t>(g.width) * page > (1 << 30) || g.cap < 1 || g.cap > (1 << 30) ||
      (g.B > 1 && g.stride < g.width)) {
    skv_set_error("%s: batch=%d width=%d (stride %lld) free=%d", what, g.B, g.width, (long long)g.stride, g.cap);
    return SKV_EINVAL;
  }
  return SKV_OK;
}

}  // namespace

extern "C" int skv_paged_reserve(const int32_t* lengths, const int32_t* counts, int32_t* table, int64_t table_stride,
                                 int width, int32_t* held, const int32_t* free_pages, int free_cap, int32_t* free_count,
                                 int batch_size, int rows, int page, int32_t* cu, int32_t* totals, int32_t* slots,
                                 void* stream) {
  const char* what = "paged_reserve";
  const Pages g{table, table_stride, width, held, const_cast<int32_t*>(free_pages), free_cap, free_count, batch_size,
                shift_of(page)};
  if (const int rc = check_pages(what, g, page)) return rc;
  if (!lengths || !counts || !cu || !totals || (rows > 0 && !slots)) {
    skv_set_error("%s: null pointer", what);
    return SKV_EINVAL;
  }
  if (rows < 0 || rows > (1 << 30)) {
    skv_set_error("%s: rows=%d", what, rows);
    return SKV_EINVAL;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows <= kOneLaunchRows) {
    hipLaunchKernelGGL(reserve_kernel<true>, dim3(1), dim3(kSeqs), 0, s, g, lengths, counts, rows, cu, totals, slots);
  } else {
    hipLaunchKernelGGL(reserve_kernel<false>, dim3(1), dim3(kSeqs), 0, s, g, lengths, counts, rows, cu, totals, slots);
    hipLaunchKernelGGL(slots_kernel, dim3((rows + 255) / 256), dim3(256), 0, s, g, cu, totals, rows, slots);
  }
  return skv_check_launch(what);
}

extern "C" int skv_paged_release(int32_t* lengths, const int32_t* keep, int32_t* table, int64_t table_stride, int width,
                                 int32_t* held, int32_t* free_pages, int free_cap, int32_t* free_count, int batch_size,
                                 int page, void* stream) {
  const char* what = "paged_release";
  const Pages g{table, table_stride, width, held, free_pages, free_cap, free_count, batch_size, shift_of(page)};
  if (const int rc = check_pages(what, g, page)) return rc;
  if (!lengths || !keep) {
    skv_set_error("%s: null pointer", what);
    return SKV_EINVAL;
  }
  hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kSeqs), 0, static_cast<hipStream_t>(stream), g, lengths, keep);
  return skv_check_launch(what);
}

extern "C" int skv_paged_write(const uint16_t* k, int64_t k_stride_t, int64_t k_stride_h, const uint16_t* v,
                               int64_t v_stride_t, int64_t v_stride_h, uint16_t* k_pages, uint16_t* v_pages,
                               int64_t p_stride_p, int64_t p_stride_h, int64_t p_stride_s, const int32_t* slots,
                               int rows, int heads, int pages, int page, void* stream) {
  const char* what = "paged_write";
  if (!k || !v || !k_pages || !v_pages || !slots) {
    skv_set_error("%s: null pointer", what);
    return SKV_EINVAL;
  }
  const int shift = shift_of(page);
  if (shift < 0) {
    skv_set_error("%s: page=%d (16, 32, 64, 128 or 256 tokens)", what, page);
    return SKV_EUNSUPPORTED;
  }
  const int64_t n = static_cast<int64_t>(rows) * heads * 16;
  if (rows < 1 || heads < 1 || heads > 65535 || pages < 1 ||
      (static_cast<int64_t>(pages) << shift) > (int64_t{1} << 31) || n >= (int64_t{1} << 32)) {
    skv_set_error("%s: rows=%d heads=%d pages=%d page=%d", what, rows, heads, pages, page);
    return SKV_EINVAL;
  }
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_pages) |
        reinterpret_cast<uintptr_t>(v_pages)) & 15) ||
      ((k_stride_t | k_stride_h | v_stride_t | v_stride_h | p_stride_p | p_stride_h | p_stride_s) & 7)) {
    skv_set_error("%s: rows must be 16-byte aligned", what);
    return SKV_EINVAL;
  }
  WriteArgs a{k, k_stride_t, k_stride_h, v, v_stride_t, v_stride_h, k_pages, v_pages, p_stride_p, p_stride_h,
              p_stride_s, slots, n, heads, shift, static_cast<int64_t>(pages) << shift};
  hipLaunchKernelGGL(write_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  return skv_check_launch(what);
}
