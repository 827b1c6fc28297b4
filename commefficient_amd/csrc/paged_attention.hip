// One new token of every sequence against its paged keys and values:
//   o[n, h] = sum_t softmax_t(scale q[n, h] . k[n, t, h / group]) v[n, t, h / group],
// t < lens[n], the keys read through table[n].  When the new token's own k, v
// rows are given they stand for position lens[n] - 1 and are stored into that
// slot by the same launch.  Rows without tokens, or with every score -inf, are
// 0; a row that meets a page
// id outside the cache, or is longer than its table row, is NaN and nothing
// is read or written through that id.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <cstdint>
#include "decode.h"

namespace commeff {
namespace {

template <DecodeType T>
struct Elem;
template <>
struct Elem<kBf16> {
  typedef uint16_t t;
  static __device__ __forceinline__ float load(t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
  static __device__ __forceinline__ t store(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
  }
};
template <>
struct Elem<kF16> {
  typedef uint16_t t;
  static __device__ __forceinline__ float load(t x) { return static_cast<float>(__builtin_bit_cast(_Float16, x)); }
  static __device__ __forceinline__ t store(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  }
};
template <>
struct Elem<kF32> {
  typedef float t;
  static __device__ __forceinline__ float load(t x) { return x; }
  static __device__ __forceinline__ t store(float f) { return f; }
};

// a workgroup per (sequence, query head), a wave per token, a lane per column
template <DecodeType T>
__global__ void __launch_bounds__(256) paged_attn_kernel(PagedAttnArgs a) {
  typedef Elem<T> E;
  typedef typename E::t S;
  const int n = blockIdx.x / a.heads, h = blockIdx.x - n * a.heads;
  const int kh = h / (a.heads / a.kv_heads);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int len = a.lens[n];
  S* out = static_cast<S*>(a.out) + (static_cast<int64_t>(n) * a.heads + h) * a.dim;
  if (len <= 0) {
    for (int d = tid; d < a.dim; d += 256) out[d] = E::store(0.f);
    return;
  }
  bool bad = len > static_cast<int64_t>(a.width) * a.page;
  const int32_t* row = a.table + n * a.table_ld;
  const S* q = static_cast<const S*>(a.q) + n * a.q_row + h * a.q_head;
  const S* kn = a.k ? static_cast<const S*>(a.k) + n * a.k_row + kh * a.k_head : nullptr;
  const S* vn = a.v ? static_cast<const S*>(a.v) + n * a.v_row + kh * a.v_head : nullptr;
  S* kc = static_cast<S*>(a.kc) + kh * a.kc_head;
  S* vc = static_cast<S*>(a.vc) + kh * a.vc_head;
  constexpr int MD = 4;  // 64-column pieces of a head of at most 256
  float qv[MD], acc[MD];
#pragma unroll
  for (int i = 0; i < MD; ++i) {
    const int d = lane + 64 * i;
    qv[i] = d < a.dim ? E::load(q[d]) * a.scale : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  if (!bad) {
    for (int t = w; t < len; t += 4) {
      const int64_t id = row[t / a.page];
      if (id < 0 || id >= a.pages) {
        bad = true;  // (the new token is stored all the same, through its own page)
        continue;
      }
      const int64_t off = t % a.page;
      const bool fresh = kn && t == len - 1;
      S* kslot = kc + id * a.kc_page + off * a.kc_tok;
      S* vslot = vc + id * a.vc_page + off * a.vc_tok;
      const S* kr = fresh ? kn : kslot;
      const S* vr = fresh ? vn : vslot;
      float x = 0.f, v[MD];
#pragma unroll
      for (int i = 0; i < MD; ++i) {
        const int d = lane + 64 * i;
        v[i] = 0.f;
        if (d < a.dim) {
          x += qv[i] * E::load(kr[d]);
          v[i] = E::load(vr[d]);
          if (fresh && h % (a.heads / a.kv_heads) == 0) {
            kslot[d] = kr[d];
            vslot[d] = vr[d];
          }
        }
      }
      for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
      const float mn = fmaxf(m, x), at = mn == -INFINITY ? 0.f : mn;  // (all scores -inf: weights 0)
      const float c = __expf(m - at), p = __expf(x - at);
      m = mn;
      l = l * c + p;
#pragma unroll
      for (int i = 0; i < MD; ++i) acc[i] = acc[i] * c + p * v[i];
    }
  }
  __shared__ float sm[4], sl[4], so[4][256];
  if (lane == 0) {
    sm[w] = m;
    sl[w] = bad ? NAN : l;
  }
#pragma unroll
  for (int i = 0; i < MD; ++i) so[w][lane + 64 * i] = acc[i];
  __syncthreads();
  const float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  for (int d = tid; d < a.dim; d += 256) {
    float num = 0.f, den = 0.f;
    for (int i = 0; i < 4; ++i) {
      const float c = sm[i] == -INFINITY ? 0.f : __expf(sm[i] - mm);
      num += c * so[i][d];
      den += sl[i] != sl[i] ? NAN : c * sl[i];
    }
    out[d] = E::store(den == 0.f ? 0.f : num / den);
  }
}

}  // namespace

int paged_attention_split(int, int, int, int64_t) { return 1; }

void launch_paged_attention(const PagedAttnArgs& a, DecodeType t, hipStream_t stream) {
  if (a.n == 0) return;
  const dim3 grid(static_cast<uint32_t>(a.n) * a.heads);
  if (t == kBf16) COMMEFF_LAUNCH(paged_attn_kernel<kBf16>, grid, dim3(256), 0, stream, a);
  else if (t == kF16) COMMEFF_LAUNCH(paged_attn_kernel<kF16>, grid, dim3(256), 0, stream, a);
  else COMMEFF_LAUNCH(paged_attn_kernel<kF32>, grid, dim3(256), 0, stream, a);
}

}  // namespace commeff
