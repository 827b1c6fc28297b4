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
// that (kFused) leave the rows to a second launch over the whole chip.  16
// prompts of up to 500 tokens 7.5 us (an empty launch 1.4, the scans 2.8, the
// rows 2.9), one token for 4,096 sequences 11.1.  Against the two launches:
// 1,024 sequences 7.9 to 10.0 us, 4,096 11.2 to 15.0, 8,192 19.3 to 21.6; 1,000
// with 8 rows each 11.5 either way.
constexpr int kScan = 1024, kEach = 4;  // threads of the scan, sequences a thread takes at once
constexpr int kFused = 8192;            // sequences and rows of a single launch

// exclusive scan of min(a + b, cap) over the block, values <= cap <= 2^30 + 1;
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
  v = __shfl_up(v, 1, 64);
  return lane == 0 ? before : min(before + v, cap);
}

struct KvPlan {  // of the sequences: LDS, or global memory
  int32_t *start, *base, *first;
};

// rows r0 .. r0 + 3: slot, position, sequence, and the table entry where one
// opens a page.  One search for the four: the later rows mostly belong to the
// same sequence or the next (4,096 rows on one CU are bound by instructions).
__device__ __forceinline__ void extend_rows(const KvExtendArgs& a, const KvPlan& p, int r0) {
  if (r0 >= a.rows) return;
  int i = 0;  // the sequences that end at or before the row: start[i] <= r for i <= that many
  auto search = [&](int r) {
    i = 0;
    for (int s = a.search; s > 0; s >>= 1)
      if (i + s <= a.n && p.start[i + s] <= r) i += s;
  };
  search(r0);
  int seq[4], pos[4], off[4], id[4];
  const int32_t* src[4];
  int32_t* dst[4];
  int end = i < a.n ? p.start[i + 1] : 0x7fffffff, len = -1, begin = 0, have = 0;
  const int32_t* taken = nullptr;
  int32_t* row = nullptr;
  bool enter = true;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + k;
    if (r >= end && r < a.rows) {
      ++i;
      end = i < a.n ? p.start[i + 1] : 0x7fffffff;
      if (r >= end) {  // (empty sequences between)
        search(r);
        end = i < a.n ? p.start[i + 1] : 0x7fffffff;
      }
      enter = true;
    }
    if (enter) {
      enter = false;
      len = i < a.n ? p.base[i] : -1;
      if (len >= 0) {
        begin = p.start[i];
        have = a.by_page.of(len + a.page - 1);
        row = a.table + i * a.table_ld;
        taken = a.pool + p.first[i];
      }
    }
    seq[k] = i < a.n ? i : -1;
    src[k] = nullptr;
    dst[k] = nullptr;
    pos[k] = off[k] = 0;
    if (len >= 0 && r < a.rows) {
      pos[k] = len + r - begin;
      const int pi = a.by_page.of(pos[k]);
      off[k] = pos[k] - pi * a.page;
      src[k] = pi < have ? row + pi : taken + (pi - have);
      if (pi >= have && off[k] == 0) dst[k] = row + pi;
    }
  }
  int64_t slot[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) id[k] = src[k] ? *src[k] : -1;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (dst[k]) *dst[k] = id[k];
    slot[k] = id[k] < 0 ? -1 : static_cast<int64_t>(id[k]) * a.page + off[k];
  }
  if (r0 + 4 <= a.rows) {  // (the outputs start at multiples of 16 bytes)
    *reinterpret_cast<longlong2*>(a.slots + r0) = longlong2{slot[0], slot[1]};
    *reinterpret_cast<longlong2*>(a.slots + r0 + 2) = longlong2{slot[2], slot[3]};
    *reinterpret_cast<int4*>(a.pos + r0) = int4{pos[0], pos[1], pos[2], pos[3]};
    *reinterpret_cast<int4*>(a.seq + r0) = int4{seq[0], seq[1], seq[2], seq[3]};
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r0 + k < a.rows) a.slots[r0 + k] = slot[k], a.pos[r0 + k] = pos[k], a.seq[r0 + k] = seq[k];
  }
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
  const uint32_t rows = static_cast<uint32_t>(a.rows);
  uint32_t rows_before = 0, need_before = 0;  // saturated at rows + 1 and avail + 1
  int got = 0, miss = 0;
  for (int i0 = 0; i0 < a.n; i0 += kScan * kEach) {
    const int i = i0 + tid * kEach;
    int len[kEach], fresh[kEach];
    uint32_t end[kEach], upto[kEach], need[kEach], total;
    bool fits[kEach];
    if (a.wide && i + kEach <= a.n) {
      const int4 l = *reinterpret_cast<const int4*>(a.lens + i), f = *reinterpret_cast<const int4*>(a.fresh + i);
      len[0] = l.x, len[1] = l.y, len[2] = l.z, len[3] = l.w;
      fresh[0] = f.x, fresh[1] = f.y, fresh[2] = f.z, fresh[3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        len[k] = i + k < a.n ? a.lens[i + k] : 0;
        fresh[k] = i + k < a.n ? a.fresh[i + k] : 0;
      }
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k)
      end[k] = min((k ? end[k - 1] : 0u) + min(static_cast<uint32_t>(max(fresh[k], 0)), rows + 1), rows + 1);
    const uint32_t rb = rows_before;
    uint32_t prev = min(rb + block_scan(end[kEach - 1], rows + 1, lds, &total), rows + 1);
    rows_before = min(rb + total, rows + 1);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const uint32_t begin = k ? min(prev + end[k - 1], rows + 1) : prev, e = min(prev + end[k], rows + 1);
      fits[k] = i + k < a.n && fresh[k] >= 0 && len[k] >= 0 && e <= rows &&
                static_cast<int64_t>(len[k]) + fresh[k] <= static_cast<int64_t>(a.width) * a.page;
      need[k] = 0;
      if (fits[k])
        need[k] = a.by_page.of(len[k] + fresh[k] + a.page - 1) - a.by_page.of(len[k] + a.page - 1);
      upto[k] = min((k ? upto[k - 1] : 0u) + min(need[k], avail + 1), avail + 1);
      if (i + k < a.n) {
        p.start[i + k] = static_cast<int32_t>(min(begin, rows));
        if constexpr (FUSED) a.start[i + k] = static_cast<int32_t>(min(begin, rows));
      }
    }
    const uint32_t nb = need_before;
    prev = min(nb + block_scan(upto[kEach - 1], avail + 1, lds, &total), avail + 1);
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
    for (int r = tid * 4; r < a.rows; r += 4 * kScan) extend_rows(a, p, r);
}

__global__ void __launch_bounds__(256) kv_extend_rows_kernel(KvExtendArgs a) {
  extend_rows(a, KvPlan{a.start, a.base, a.first}, (blockIdx.x * 256 + threadIdx.x) * 4);
}

// ------------------------------------------------------------------- write
// A copy, bound by HBM.  A workgroup takes a.chunk rows, a thread every 256th
// of their pieces (16 bytes where all addresses allow it).  Stores that are not
// kept in the caches leave them to the loads: 65,536 rows of 8 x 128 bf16 97
// against 105 us, 5.5 TB/s.
template <typename U>
__global__ void __launch_bounds__(256) kv_write_kernel(KvWriteArgs a) {
  const int64_t r0 = blockIdx.x * static_cast<int64_t>(a.chunk);
  const int rows = static_cast<int>(min(static_cast<int64_t>(a.chunk), a.rows - r0));
  const int per = static_cast<int>(a.by_unit.d), row = per * a.heads;  // pieces of a head's row, of a row
  for (int x = threadIdx.x; x < rows * row; x += 256) {
    const int hr = a.by_unit.of(x), u = x - hr * per;
    const int ri = a.by_heads.of(hr), h = hr - ri * a.heads;
    const int64_t r = r0 + ri, slot = a.slots[r];
    if (slot < 0 || slot >= a.pages * a.page) continue;
    const int pg = a.by_page.of(static_cast<int>(slot));  // (pages x page < 2^31)
    const int64_t off = slot - static_cast<int64_t>(pg) * a.page;
    const U k = *(reinterpret_cast<const U*>(a.k + r * a.k_row + h * a.k_head) + u);
    const U v = *(reinterpret_cast<const U*>(a.v + r * a.v_row + h * a.v_head) + u);
    __builtin_nontemporal_store(k, reinterpret_cast<U*>(a.kc + pg * a.kc_page + h * a.kc_head + off * a.kc_tok) + u);
    __builtin_nontemporal_store(v, reinterpret_cast<U*>(a.vc + pg * a.vc_page + h * a.vc_head + off * a.vc_tok) + u);
  }
}

// ----------------------------------------------------------------- reorder
// Beam j of a request takes the history of beam parent[j]: the ids of its full
// pages (shared from then on) and the content of its part-filled page, which
// goes into the page that beam j itself holds there.  One thread owns a piece
// (a table column, or 16 bytes of a token's row of one layer) of ALL the
// request's beams: it loads every moved beam's source before it stores, so
// the beams may change places in any way, in place, without a second buffer.
// A copy, bound by HBM: the workgroups that run at a time belong to few requests
// and sweep their pages in one direction (requests in turn instead: 72 against
// 67 us for 64 x 8 beams), stores past the caches (64 us).
template <typename U, int JM>
__global__ void __launch_bounds__(256) beam_reorder_kernel(BeamReorderArgs a) {
  const int b = blockIdx.y, J = a.beams, tid = threadIdx.x;
  __shared__ int s_len[JM], s_tail[JM], s_par[JM];
  __shared__ int s_from[JM], s_full[JM], s_rest[JM];  // the parent's part-filled page, and what to take (0: nothing)
  const int64_t n0 = static_cast<int64_t>(b) * J;
  int len = 0, full = 0, rest = 0;
  if (tid < J) {
    len = a.lens[n0 + tid];
    full = len < 0 ? 0 : a.by_page.of(len), rest = len < 0 ? 0 : len - full * a.page;
    const int64_t p = a.parent[n0 + tid];
    s_par[tid] = p >= 0 && p < J ? static_cast<int>(p) : -1;
    s_len[tid] = len >= 0 && full + (rest ? 1 : 0) <= a.width ? len : -1;
    s_tail[tid] = rest && full < a.width ? a.table[(n0 + tid) * a.table_ld + full] : -1;
  }
  __syncthreads();
  if (tid < J) {
    // beams that cannot move as asked stay as they are
    const int p = s_par[tid];
    bool ok = p >= 0 && p != tid && s_len[tid] > 0 && s_len[p] == len;
    if (ok && rest)
      ok = s_tail[tid] >= 0 && s_tail[tid] < a.pages && s_tail[p] >= 0 && s_tail[p] < a.pages;
    s_from[tid] = ok ? s_tail[p] : 0;
    s_full[tid] = ok ? full : 0;
    s_rest[tid] = ok ? rest : 0;
  }
  __syncthreads();
  for (int c = blockIdx.x * 256 + tid; c < a.width; c += gridDim.x * 256) {
    int32_t v[JM];
#pragma unroll
    for (int j = 0; j < JM; ++j)
      if (j < J && c < s_full[j]) v[j] = a.table[(n0 + s_par[j]) * a.table_ld + c];
#pragma unroll
    for (int j = 0; j < JM; ++j)
      if (j < J && c < s_full[j]) a.table[(n0 + j) * a.table_ld + c] = v[j];
  }
  int most = 0;
  for (int j = 0; j < J; ++j) most = max(most, s_rest[j]);
  if (most == 0) return;
  // every (layer, k or v, head) plane's part-filled page, piece after piece
  const int d = most * static_cast<int>(a.by_unit.d);
  const FastDiv by_plane = {static_cast<uint32_t>(d), 0xffffffffu / static_cast<uint32_t>(d) + 1};
  const int64_t all = 2ll * a.layers * a.heads * d;  // (below 2^31)
  for (int64_t x = blockIdx.x * 256ll + tid; x < all; x += gridDim.x * 256ll) {
    const int pl = by_plane.of(static_cast<int>(x)), i = static_cast<int>(x) - pl * d;
    const int t = a.by_unit.of(i), u = i - t * static_cast<int>(a.by_unit.d);
    const int lk = a.by_heads.of(pl), h = pl - lk * a.heads;
    unsigned char* at = a.kv + (lk >> 1) * a.s_layer + (lk & 1) * a.s_kv + h * a.s_head + t * a.s_tok;
    U v[JM];
#pragma unroll
    for (int j = 0; j < JM; ++j)
      if (j < J && t < s_rest[j]) v[j] = *(reinterpret_cast<const U*>(at + s_from[j] * a.s_page) + u);
#pragma unroll
    for (int j = 0; j < JM; ++j)
      if (j < J && t < s_rest[j])
        __builtin_nontemporal_store(v[j], reinterpret_cast<U*>(at + s_tail[j] * a.s_page) + u);
  }
}

template <typename U>
void reorder_unit(const BeamReorderArgs& a, int gy, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(gy), static_cast<uint32_t>(a.requests));
  if (a.beams <= 4) COMMEFF_LAUNCH((beam_reorder_kernel<U, 4>), grid, dim3(256), 0, stream, a);
  else if (a.beams <= 8) COMMEFF_LAUNCH((beam_reorder_kernel<U, 8>), grid, dim3(256), 0, stream, a);
  else if (a.beams <= 16) COMMEFF_LAUNCH((beam_reorder_kernel<U, 16>), grid, dim3(256), 0, stream, a);
  else COMMEFF_LAUNCH((beam_reorder_kernel<U, kReorderMaxBeams>), grid, dim3(256), 0, stream, a);
}

}  // namespace

bool kv_extend_fused(const KvExtendArgs& a) { return a.n <= kFused && a.rows <= kFused; }

void launch_kv_extend(KvExtendArgs a, hipStream_t stream) {
  a.by_page = fast_div(a.page);
  a.search = 1;
  while (2ll * a.search <= a.n) a.search *= 2;
  a.wide = ((reinterpret_cast<uintptr_t>(a.lens) | reinterpret_cast<uintptr_t>(a.fresh)) & 15) == 0;
  if (kv_extend_fused(a)) {
    const uint32_t lds = static_cast<uint32_t>(3 * a.n + 1) * 4;
    if (lds > 65536 - 1024)  // (of the current device: set wherever it is needed)
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kv_extend_kernel<true>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (3 * kFused + 1) * 4);
    COMMEFF_LAUNCH(kv_extend_kernel<true>, dim3(1), dim3(kScan), lds, stream, a);
    return;
  }
  COMMEFF_LAUNCH(kv_extend_kernel<false>, dim3(1), dim3(kScan), 0, stream, a);
  if (a.rows > 0)
    COMMEFF_LAUNCH(kv_extend_rows_kernel, dim3(static_cast<uint32_t>((a.rows + 1023) / 1024)), dim3(256), 0, stream, a);
}

void launch_kv_write(KvWriteArgs a, hipStream_t stream) {
  if (a.rows == 0) return;
  const int row = a.heads * (a.row_bytes / a.unit);
  a.by_unit = fast_div(a.row_bytes / a.unit);
  a.by_heads = fast_div(a.heads);
  a.by_page = fast_div(a.page);
  a.chunk = row >= 512 ? 1 : 512 / row;  // two pieces a thread, or one row
  const dim3 grid(static_cast<uint32_t>((a.rows + a.chunk - 1) / a.chunk));
  if (a.unit == 16) COMMEFF_LAUNCH(kv_write_kernel<v4u>, grid, dim3(256), 0, stream, a);
  else if (a.unit == 4) COMMEFF_LAUNCH(kv_write_kernel<uint32_t>, grid, dim3(256), 0, stream, a);
  else COMMEFF_LAUNCH(kv_write_kernel<uint16_t>, grid, dim3(256), 0, stream, a);
}

void launch_beam_reorder(BeamReorderArgs a, hipStream_t stream) {
  if (a.requests == 0 || a.beams < 2) return;  // (one beam: its own parent)
  a.by_page = fast_div(a.page);
  a.by_heads = fast_div(a.heads);
  a.by_unit = fast_div(a.row_bytes / a.unit);
  // two pieces a thread where the pages are all but full
  int64_t gy = (2ll * a.layers * a.heads * a.page * (a.row_bytes / a.unit) + 511) / 512;
  gy = gy < 1 ? 1 : gy > 1024 ? 1024 : gy;
  if (a.unit == 16) reorder_unit<v4u>(a, static_cast<int>(gy), stream);
  else if (a.unit == 4) reorder_unit<uint32_t>(a, static_cast<int>(gy), stream);
  else reorder_unit<uint16_t>(a, static_cast<int>(gy), stream);
}

}  // namespace commeff
