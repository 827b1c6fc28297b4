// The paged key-value cache's bookkeeping (decode.h): block tables and slot
// maps from request lengths, the rows of new tokens into their slots, and the
// states of beams that changed places.
#include <hip/hip_runtime.h>
#include <cstdint>
#include "decode.h"

namespace commeff {
namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ extend
// With e_i the tokens asked for (negative: none) and c(x) = ceil(x / page):
//   start_i = sum_{j<i} e_j,  need_i = c(len_i + e_i) - c(len_i),
// sequence i is served if its counts are sound, its table row and the output
// rows are long enough and the pool holds the pages that it and all sequences
// before it need; its pages are pool[used + sum_{j<i} need_j ..].  Row r of
// sequence i is token p = len_i + r - start_i, slot table[i][p / page] * page
// + p % page.  A few hundred KB at most: bound by latency, that is by the
// launch, two scans and the chain row -> sequence -> page.  So one workgroup
// does all of it with the sequences' plan in LDS; only batches too large for
// that (kFused) leave the rows to a second launch over the whole chip.
constexpr int kScan = 1024, kEach = 4;  // threads of the scan, sequences a thread takes at once
constexpr int kFused = 8192;            // sequences and rows of a single launch

// inclusive scan of min(a + b, cap) over the block, values <= cap <= 2^30 + 1;
// `total`: all of it
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t cap, uint32_t* lds, uint32_t* total) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(v, o, 64);
    if (lane >= o) v = min(u + v, cap);
  }
  __syncthreads();  // (lds is free again)
  if (lane == 63) lds[w] = v;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kScan / 64; ++i) {
    if (i == w) before = all;
    all = min(all + lds[i], cap);
  }
  *total = all;
  return min(before + v, cap);
}

struct KvPlan {  // of the sequences: LDS, or global memory
  int32_t *start, *base, *first;
};

// row r: its slot, position and sequence, and the table entry where it opens a page
__device__ __forceinline__ void extend_row(const KvExtendArgs& a, const KvPlan& p, int r) {
  int lo = 0, hi = a.n;  // the first sequence that ends past r
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.start[mid + 1] > r) hi = mid;
    else lo = mid + 1;
  }
  int64_t slot = -1;
  int pos = 0;
  if (lo < a.n) {
    const int len = p.base[lo];
    if (len >= 0) {
      pos = len + r - p.start[lo];
      const int pi = static_cast<uint32_t>(pos) / static_cast<uint32_t>(a.page);
      const int have = static_cast<uint32_t>(len + a.page - 1) / static_cast<uint32_t>(a.page);
      int32_t* row = a.table + lo * a.table_ld;
      int64_t id;
      if (pi < have) {
        id = row[pi];
      } else {
        id = a.pool[p.first[lo] + pi - have];
        if (pos == pi * a.page) row[pi] = static_cast<int32_t>(id);
      }
      if (id >= 0) slot = id * a.page + (pos - pi * a.page);
    }
  }
  a.slots[r] = slot;
  a.pos[r] = pos;
  a.seq[r] = lo < a.n ? lo : -1;
}

template <bool FUSED>
__global__ void __launch_bounds__(kScan) kv_extend_kernel(KvExtendArgs a) {
  extern __shared__ int32_t s_plan[];  // FUSED: start [n + 1] | base [n] | first [n]
  __shared__ uint32_t lds[kScan / 64];
  __shared__ int s_got, s_miss;
  const int tid = threadIdx.x;
  KvPlan p = {a.start, a.base, a.first};
  if constexpr (FUSED) p = {s_plan, s_plan + a.n + 1, s_plan + 2 * a.n + 1};
  if (tid == 0) s_got = s_miss = 0;
  const int used = a.used[0];
  const uint32_t avail = used < 0 || used > a.pool_n ? 0u : static_cast<uint32_t>(a.pool_n - used);
  const uint32_t rows = static_cast<uint32_t>(a.rows), page = static_cast<uint32_t>(a.page);
  uint32_t rows_before = 0, need_before = 0;  // saturated at rows + 1 and avail + 1
  int got = 0, miss = 0;
  for (int i0 = 0; i0 < a.n; i0 += kScan * kEach) {
    const int i = i0 + tid * kEach;
    int len[kEach], fresh[kEach];
    uint32_t end[kEach], upto[kEach], need[kEach], total;
    bool fits[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      len[k] = i + k < a.n ? a.lens[i + k] : 0;
      fresh[k] = i + k < a.n ? a.fresh[i + k] : 0;
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k)
      end[k] = min((k ? end[k - 1] : 0u) + min(static_cast<uint32_t>(max(fresh[k], 0)), rows + 1), rows + 1);
    const uint32_t rb = rows_before;
    uint32_t mine = end[kEach - 1];
    uint32_t incl = block_scan(mine, rows + 1, lds, &total);
    // (what lies before this thread: the scan without its own, which saturation forbids to subtract)
    uint32_t prev = __shfl_up(incl, 1, 64);
    if ((tid & 63) == 0) {
      prev = 0;
      for (int w = 0; w < (tid >> 6); ++w) prev = min(prev + lds[w], rows + 1);
    }
    prev = min(rb + prev, rows + 1);
    rows_before = min(rb + total, rows + 1);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const uint32_t begin = k ? min(prev + end[k - 1], rows + 1) : prev, e = min(prev + end[k], rows + 1);
      fits[k] = i + k < a.n && fresh[k] >= 0 && len[k] >= 0 && e <= rows &&
                static_cast<int64_t>(len[k]) + fresh[k] <= static_cast<int64_t>(a.width) * a.page;
      need[k] = 0;
      if (fits[k])
        need[k] = (static_cast<uint32_t>(len[k] + fresh[k]) + page - 1) / page -
                  (static_cast<uint32_t>(len[k]) + page - 1) / page;
      upto[k] = min((k ? upto[k - 1] : 0u) + min(need[k], avail + 1), avail + 1);
      if (i + k < a.n) {
        p.start[i + k] = static_cast<int32_t>(min(begin, rows));
        if constexpr (FUSED) a.start[i + k] = static_cast<int32_t>(min(begin, rows));
      }
    }
    const uint32_t nb = need_before;
    mine = upto[kEach - 1];
    incl = block_scan(mine, avail + 1, lds, &total);
    prev = __shfl_up(incl, 1, 64);
    if ((tid & 63) == 0) {
      prev = 0;
      for (int w = 0; w < (tid >> 6); ++w) prev = min(prev + lds[w], avail + 1);
    }
    prev = min(nb + prev, avail + 1);
    need_before = min(nb + total, avail + 1);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (i + k >= a.n) break;
      const uint32_t u = min(prev + upto[k], avail + 1);
      const bool served = fits[k] && (need[k] == 0 || u <= avail);
      p.base[i + k] = served ? len[k] : -1;
      p.first[i + k] = served ? used + static_cast<int>(u - need[k]) : 0;
      a.lens_out[i + k] = served ? len[k] + fresh[k] : len[k];
      if (served && need[k]) got = static_cast<int>(u);  // (the last one served has them all before it)
      miss += !served;
    }
  }
  __syncthreads();  // s_got and s_miss are set, `used` was read
  if (got) atomicMax(&s_got, got);
  if (miss) atomicAdd(&s_miss, miss);
  if (tid == 0) {
    const int32_t last = static_cast<int32_t>(min(rows_before, rows));
    p.start[a.n] = last;
    if constexpr (FUSED) a.start[a.n] = last;
  }
  __syncthreads();
  if (tid == 0) {
    a.used_out[0] = used + s_got;
    a.missed[0] = s_miss;
  }
  if constexpr (FUSED)
    for (int r = tid; r < a.rows; r += kScan) extend_row(a, p, r);
}

__global__ void __launch_bounds__(256) kv_extend_rows_kernel(KvExtendArgs a) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < a.rows) extend_row(a, KvPlan{a.start, a.base, a.first}, r);
}

// ------------------------------------------------------------------- write
template <typename U>
__global__ void __launch_bounds__(256) kv_write_kernel(KvWriteArgs a) {
  const int per = a.row_bytes / static_cast<int>(sizeof(U));  // units of a head's row
  const int64_t all = a.rows * a.heads * per;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
    const int64_t r = i / (a.heads * per);
    const int x = static_cast<int>(i - r * (a.heads * per));
    const int h = x / per, u = x - h * per;
    const int64_t slot = a.slots[r];
    if (slot < 0 || slot >= a.pages * a.page) continue;
    const int64_t pg = slot / a.page, off = slot - pg * a.page;
    *(reinterpret_cast<U*>(a.kc + pg * a.kc_page + h * a.kc_head + off * a.kc_tok) + u) =
        *(reinterpret_cast<const U*>(a.k + r * a.k_row + h * a.k_head) + u);
    *(reinterpret_cast<U*>(a.vc + pg * a.vc_page + h * a.vc_head + off * a.vc_tok) + u) =
        *(reinterpret_cast<const U*>(a.v + r * a.v_row + h * a.v_head) + u);
  }
}

// ----------------------------------------------------------------- reorder
// Beam j of a request takes the history of beam parent[j]: the ids of its full
// pages (shared from then on) and the content of its part-filled page, which
// goes into the page that beam j itself holds there.  One thread owns a piece
// (a table column, or 16 bytes of a token's row of one layer) of ALL the
// request's beams: it loads every moved beam's source before it stores, so
// the beams may change places in any way, in place, without a second buffer.
template <typename U, int JM>
__global__ void __launch_bounds__(256) beam_reorder_kernel(BeamReorderArgs a) {
  const int b = blockIdx.x, J = a.beams, tid = threadIdx.x;
  __shared__ int s_par[JM], s_len[JM], s_tail[JM];
  const int64_t n0 = static_cast<int64_t>(b) * J;
  if (tid < J) {
    const int64_t p = a.parent[n0 + tid];
    const int len = a.lens[n0 + tid];
    const int full = len < 0 ? -1 : len / a.page;
    const bool part = len > 0 && len % a.page != 0;
    s_par[tid] = p >= 0 && p < J ? static_cast<int>(p) : -1;
    s_len[tid] = len >= 0 && full + (part ? 1 : 0) <= a.width ? len : -1;
    s_tail[tid] = part && full < a.width ? a.table[(n0 + tid) * a.table_ld + full] : -1;
  }
  __syncthreads();
  if (tid < J) {
    // beams that cannot move as asked stay as they are
    const int p = s_par[tid], len = s_len[tid];
    bool ok = p >= 0 && p != tid && len > 0 && s_len[p] == len;
    if (ok && len % a.page != 0)
      ok = s_tail[tid] >= 0 && s_tail[tid] < a.pages && s_tail[p] >= 0 && s_tail[p] < a.pages;
    if (!ok) s_par[tid] = -1;  // (each thread reads other beams' s_len and s_tail only)
  }
  __syncthreads();
  const int64_t step = static_cast<int64_t>(gridDim.y) * 256;
  const int64_t me = blockIdx.y * 256ll + tid;
  for (int64_t c = me; c < a.width; c += step) {
    int32_t v[JM];
#pragma unroll
    for (int j = 0; j < JM; ++j)
      if (j < J && s_par[j] >= 0 && c < s_len[j] / a.page) v[j] = a.table[(n0 + s_par[j]) * a.table_ld + c];
#pragma unroll
    for (int j = 0; j < JM; ++j)
      if (j < J && s_par[j] >= 0 && c < s_len[j] / a.page) a.table[(n0 + j) * a.table_ld + c] = v[j];
  }
  int most = 0;
  for (int j = 0; j < J; ++j)
    if (s_par[j] >= 0) most = max(most, s_len[j] % a.page);
  if (most == 0) return;
  const int per = a.row_bytes / static_cast<int>(sizeof(U));
  const int64_t all = 2ll * a.layers * a.heads * most * per;
  for (int64_t i = me; i < all; i += step) {
    int64_t x = i;
    const int u = static_cast<int>(x % per);
    x /= per;
    const int t = static_cast<int>(x % most);
    x /= most;
    const int h = static_cast<int>(x % a.heads);
    x /= a.heads;
    unsigned char* plane = a.kv + (x >> 1) * a.s_layer + (x & 1) * a.s_kv + h * a.s_head + t * a.s_tok;
    U v[JM];
#pragma unroll
    for (int j = 0; j < JM; ++j)
      if (j < J && s_par[j] >= 0 && t < s_len[j] % a.page)
        v[j] = *(reinterpret_cast<const U*>(plane + s_tail[s_par[j]] * a.s_page) + u);
#pragma unroll
    for (int j = 0; j < JM; ++j)
      if (j < J && s_par[j] >= 0 && t < s_len[j] % a.page)
        *(reinterpret_cast<U*>(plane + s_tail[j] * a.s_page) + u) = v[j];
  }
}

template <typename U>
void reorder_unit(const BeamReorderArgs& a, hipStream_t stream) {
  const int64_t units = 2ll * a.layers * a.heads * a.page * (a.row_bytes / static_cast<int>(sizeof(U)));
  int64_t gy = (units / 2 + 255) / 256;
  gy = gy < 1 ? 1 : gy > 1024 ? 1024 : gy;
  const dim3 grid(static_cast<uint32_t>(a.requests), static_cast<uint32_t>(gy));
  if (a.beams <= 8) COMMEFF_LAUNCH((beam_reorder_kernel<U, 8>), grid, dim3(256), 0, stream, a);
  else COMMEFF_LAUNCH((beam_reorder_kernel<U, kReorderMaxBeams>), grid, dim3(256), 0, stream, a);
}

}  // namespace

void launch_kv_extend(const KvExtendArgs& a, hipStream_t stream) {
  if (a.n <= kFused && a.rows <= kFused) {
    const uint32_t lds = static_cast<uint32_t>(3 * a.n + 1) * 4;
    if (lds > 48 * 1024) {
      static bool attr = false;
      if (!attr) {
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kv_extend_kernel<true>),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, (3 * kFused + 1) * 4);
        attr = true;
      }
    }
    COMMEFF_LAUNCH(kv_extend_kernel<true>, dim3(1), dim3(kScan), lds, stream, a);
    return;
  }
  COMMEFF_LAUNCH(kv_extend_kernel<false>, dim3(1), dim3(kScan), 0, stream, a);
  if (a.rows > 0)
    COMMEFF_LAUNCH(kv_extend_rows_kernel, dim3(static_cast<uint32_t>((a.rows + 255) / 256)), dim3(256), 0, stream, a);
}

void launch_kv_write(const KvWriteArgs& a, hipStream_t stream) {
  if (a.rows == 0) return;
  const int64_t all = a.rows * a.heads * (a.row_bytes / a.unit);
  int64_t blocks = (all + 255) / 256;
  if (blocks > 65536) blocks = 65536;
  const dim3 grid(static_cast<uint32_t>(blocks));
  if (a.unit == 16) COMMEFF_LAUNCH(kv_write_kernel<v4u>, grid, dim3(256), 0, stream, a);
  else if (a.unit == 4) COMMEFF_LAUNCH(kv_write_kernel<uint32_t>, grid, dim3(256), 0, stream, a);
  else COMMEFF_LAUNCH(kv_write_kernel<uint16_t>, grid, dim3(256), 0, stream, a);
}

void launch_beam_reorder(const BeamReorderArgs& a, hipStream_t stream) {
  if (a.requests == 0 || a.beams < 2) return;  // (one beam: its own parent)
  if (a.unit == 16) reorder_unit<v4u>(a, stream);
  else if (a.unit == 4) reorder_unit<uint32_t>(a, stream);
  else reorder_unit<uint16_t>(a, stream);
}

}  // namespace commeff
