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
// inclusive scan over a 1,024-thread block (16 waves); `total` is its sum
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* lds, int64_t* total) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  __syncthreads();  // (lds is free again)
  if (lane == 63) lds[w] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (i < w) before += lds[i];
    all += lds[i];
  }
  *total = all;
  return v + before;
}

// With e_i the tokens asked for (negative: none) and c(x) = ceil(x / page):
//   start_i = sum_{j<i} e_j,  need_i = c(len_i + e_i) - c(len_i),
// sequence i is served if its counts are sound, its table row and the output
// rows are long enough and the pool holds the pages that it and all sequences
// before it need; its pages are pool[used + sum_{j<i} need_j ..].  Row r of
// sequence i is token p = len_i + r - start_i, slot table[i][p / page] * page
// + p % page.  One workgroup: two scans over the sequences, then the rows.
__global__ void __launch_bounds__(1024) kv_extend_kernel(KvExtendArgs a) {
  __shared__ int64_t lds[16];
  const int tid = threadIdx.x;
  const int64_t used = a.used[0];
  const int64_t avail = used < 0 ? 0 : (a.pool_n > used ? a.pool_n - used : 0);
  int64_t rows_before = 0, need_before = 0, got = 0, miss = 0;
  for (int i0 = 0; i0 < a.n; i0 += 1024) {
    const int i = i0 + tid;
    const bool in = i < a.n;
    const int64_t len = in ? a.lens[i] : 0, fresh = in ? a.fresh[i] : 0;
    int64_t total;
    const int64_t add = fresh > 0 ? fresh : 0;
    const int64_t end = rows_before + block_scan(add, lds, &total);
    rows_before += total;
    const bool fits = in && fresh >= 0 && len >= 0 && end <= a.rows &&
                      len + fresh <= static_cast<int64_t>(a.width) * a.page;
    const int64_t need = fits ? (len + fresh + a.page - 1) / a.page - (len + a.page - 1) / a.page : 0;
    const int64_t upto = need_before + block_scan(need, lds, &total);
    need_before += total;
    const bool served = fits && (need == 0 || upto <= avail);
    if (in) {
      a.start[i] = static_cast<int32_t>(end - add < a.rows ? end - add : a.rows);
      if (i == a.n - 1) a.start[a.n] = static_cast<int32_t>(end < a.rows ? end : a.rows);
      a.base[i] = served ? static_cast<int32_t>(len) : -1;
      a.first[i] = static_cast<int32_t>(used + (served ? upto - need : 0));
      a.lens_out[i] = static_cast<int32_t>(served ? len + fresh : len);
    }
    block_scan(served ? need : 0, lds, &total);
    got += total;
    block_scan(in && !served ? 1 : 0, lds, &total);
    miss += total;
  }
  if (a.n == 0 && tid == 0) a.start[0] = 0;
  __syncthreads();  // start, base and first of every sequence are written; used was read
  if (tid == 0) {
    a.used_out[0] = static_cast<int32_t>(used + got);
    a.missed[0] = static_cast<int32_t>(miss);
  }
  for (int r = tid; r < a.rows; r += 1024) {
    int lo = 0, hi = a.n;  // the first sequence that ends past r
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.start[mid + 1] > r) hi = mid;
      else lo = mid + 1;
    }
    int64_t slot = -1;
    int pos = 0;
    if (lo < a.n) {
      const int len = a.base[lo];
      if (len >= 0) {
        pos = len + r - a.start[lo];
        const int pi = pos / a.page, have = (len + a.page - 1) / a.page;
        int32_t* row = a.table + static_cast<int64_t>(lo) * a.table_ld;
        int64_t id;
        if (pi < have) {
          id = row[pi];
        } else {
          id = a.pool[a.first[lo] + pi - have];
          if (pos == pi * a.page) row[pi] = static_cast<int32_t>(id);
        }
        if (id >= 0) slot = id * a.page + (pos - pi * a.page);
      }
    }
    a.slots[r] = slot;
    a.pos[r] = pos;
    a.seq[r] = lo < a.n ? lo : -1;
  }
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
  COMMEFF_LAUNCH(kv_extend_kernel, dim3(1), dim3(1024), 0, stream, a);
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
