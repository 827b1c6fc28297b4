// Generation from a paged key-value cache: what the bindings (decode_ops.cpp)
// pass to the kernels of kvcache.hip, paged_attention.hip and beam.hip.
//
// A cache of one layer is k, v [pages, kv heads, page size, head dim]: a slot
// s names row (s / page size, ., s % page size).  table [sequences, width]
// int32 names each sequence's pages in order, lens [sequences] int32 counts
// its tokens.  A page id outside [0, pages) is never followed.
#pragma once
#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#else
#include <hip/hip_runtime_api.h>
#endif
#include <cstdint>
#include "launch.h"

namespace commeff {

enum DecodeType { kBf16 = 0, kF16 = 1, kF32 = 2 };

// x / d for 0 <= x < 2^31 by a product: umulhi(x, 2^32 / d + 1) is the quotient
// or one more (it adds at most x / 2^32 to x / d)
struct FastDiv {
  uint32_t d, m;
#ifdef __HIPCC__
  __device__ __forceinline__ int of(int x) const {
    uint32_t q = __umulhi(static_cast<uint32_t>(x), m);
    q -= q * d > static_cast<uint32_t>(x);
    return d == 1 ? x : static_cast<int>(q);
  }
#endif
};
inline FastDiv fast_div(int64_t d) {
  return {static_cast<uint32_t>(d < 1 ? 1 : d), d <= 1 ? 0u : static_cast<uint32_t>((1ull << 32) / d + 1)};
}

constexpr int kBeamMaxKeep = 64;     // candidates of one beam_select request
constexpr int kBeamMaxBeams = 1024;
constexpr int kBeamWaves = 4;        // of a workgroup of its first kernel
constexpr int kReorderMaxBeams = 32;

struct KvExtendArgs {
  int32_t* table;
  int64_t table_ld;
  const int32_t* lens;
  const int32_t* fresh;  // tokens to add, one count a sequence
  const int32_t* pool;   // free page ids from pool[used] on
  const int32_t* used;
  int64_t* slots;        // [rows]
  int32_t *pos, *seq;    // [rows]
  int32_t* start;        // [n + 1]
  int32_t* missed;       // [1]
  int32_t *lens_out, *used_out;  // may be lens / used
  int32_t *base, *first;         // scratch [n] unless fused: length before, or -1; first pool index
  int n, width, page, rows, pool_n;
  int search, wide;  // launch_kv_extend: the first step of a search, 16-byte loads
  FastDiv by_page;
};

struct KvWriteArgs {
  const unsigned char *k, *v;
  unsigned char *kc, *vc;
  const int64_t* slots;
  int64_t k_row, k_head, v_row, v_head;                    // bytes
  int64_t kc_page, kc_head, kc_tok, vc_page, vc_head, vc_tok;  // bytes
  int64_t rows, pages;
  int heads, page, row_bytes;  // row_bytes: one head's
  int unit;                    // bytes moved at once: 16, 4 or 2
  int chunk;                   // launch_kv_write
  FastDiv by_unit, by_heads, by_page;
};

struct BeamReorderArgs {
  const int64_t* parent;  // [requests, beams]
  int32_t* table;         // [requests * beams, width]
  int64_t table_ld;
  const int32_t* lens;    // [requests * beams]
  unsigned char* kv;      // [layers, 2, pages, heads, page, dim]
  int64_t s_layer, s_kv, s_page, s_head, s_tok;  // bytes
  int64_t pages;
  int requests, beams, width, layers, heads, page, row_bytes, unit;
  FastDiv by_page, by_heads, by_unit;  // launch_beam_reorder
};

struct PagedAttnArgs {
  const void* q;
  const void *k, *v;  // the new token's rows, or null
  void *kc, *vc;
  const int32_t* table;
  const int32_t* lens;
  void* out;
  float* part;  // split > 1: [n, heads, split] x (max, sum, head dim values)
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;         // elements
  int64_t kc_page, kc_head, kc_tok, vc_page, vc_head, vc_tok;  // elements
  int64_t table_ld, pages;
  int n, heads, kv_heads, dim, width, page;
  float scale;
  int split, waves, group;  // plan_paged_attention
  FastDiv by_heads, by_n, by_kv, by_tiles, by_split, by_page;
};

struct BeamSelectArgs {
  const void* logits;
  const float* scores;      // [requests, beams]
  const uint8_t* finished;  // [requests, beams] or null
  float* out_scores;        // [requests, keep]
  int64_t *out_parent, *out_token;
  unsigned long long* cand;  // workspace [requests * beams, parts, keep]
  double* stat;              // workspace [requests * beams, parts, kBeamWaves, 2]
  int64_t s_request, s_beam;  // elements
  int64_t eos;
  int requests, beams, vocab, keep, parts;
  int tight, type;                       // launch_beam_select
  double near;
  FastDiv by_beams, by_parts, by_lists;
};

bool kv_extend_fused(const KvExtendArgs& a);  // one launch, the plan in LDS
void launch_kv_extend(KvExtendArgs a, hipStream_t stream);
void launch_kv_write(KvWriteArgs a, hipStream_t stream);
void launch_beam_reorder(BeamReorderArgs a, hipStream_t stream);
void launch_paged_attention(const PagedAttnArgs& a, DecodeType t, hipStream_t stream);
// fills in the split and the divisors; longest: a hint of the longest sequence
void plan_paged_attention(PagedAttnArgs& a, DecodeType t, int64_t longest);
void launch_beam_select(BeamSelectArgs a, DecodeType t, hipStream_t stream);
int beam_select_parts(int vocab, DecodeType t);

}  // namespace commeff
