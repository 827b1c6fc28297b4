// Beam search's selection: of the beams x vocabulary continuations of a
// request, the `keep` best by
//   score(j, v) = scores[j] + x[j, v] - log sum_u exp x[j, u],
// equal scores by the lower j, then the lower v.  A finished beam goes on with
// `eos` alone, at its own score.  A beam has no continuation where its score
// or its log-sum-exp is not finite (a NaN or +inf logit, no logit above -inf),
// nor has a token whose logit is -inf; places that nothing is left for hold
// (-inf, 0, 0).
//
// Two launches, bound by reading the logits once.  Within a row a score is
// monotone in the logit, so the first kernel ranks raw logits and never forms
// a score: a workgroup holds up to 8,192 of a row's logits in registers, takes
// their maximum, the sum of exponentials beside it and the `keep` best of
// them.  The second turns what is left of a request (beams x parts x keep)
// into scores, in 64 bits: candidates of different beams may lie closer than
// fp32 tells apart.
//
// The best of many by a threshold: of the 64 lanes of a wave, at least `keep`
// hold an element that is no less than the keep-th largest of the lanes' own
// maxima, so nothing below that (the largest such of the waves) can be among
// the `keep` best.  It is found by bits with a ballot a bit, some 2 keep to 4
// keep elements pass, and those are ranked by counting.  Where more than kList
// pass (thousands of equal logits) `keep` rounds of an argmax take over.
#include <hip/hip_runtime.h>
#include <cstdint>
#include "conv_common.h"
#include "decode.h"

namespace commeff {
namespace {

constexpr int kThreads = 256;
constexpr int kRow = 32;     // logits a thread holds
constexpr int kList = 1024;  // candidates that are ranked by counting

typedef unsigned long long u64;

template <DecodeType T>
__device__ __forceinline__ float to_float(uint32_t bits) {  // of one element
  if constexpr (T == kBf16) return bf2f(bits);
  else if constexpr (T == kF16) return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
  else return __uint_as_float(bits);
}

// unsigned integers in the order of the floats (+0 and -0 made one before)
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u ^ (u >> 31 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ u64 ordered(double x) {
  const u64 u = __builtin_bit_cast(u64, x);
  return u ^ (u >> 63 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double unordered(u64 u) {
  return __builtin_bit_cast(double, u ^ (u >> 63 ? 1ull << 63 : ~0ull));
}
constexpr uint32_t kNone = 0x007fffffu;  // ordered(-inf): no candidate

// a bound that at least `keep` lanes' values reach (0 where fewer than `keep`
// lanes have any): the keep-th largest, or less by bits that do not matter
__device__ __forceinline__ uint32_t wave_bound(uint32_t x, int keep) {
  uint32_t bound = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = bound | 1u << bit;
    const int n = __popcll(__ballot(x >= c));
    if (n >= keep) bound = c;
    if (n == keep) break;
  }
  return bound;
}

// (value, index) pairs; the greater value first, then the lower index
struct Best {
  u64 value, index;
};
__device__ __forceinline__ bool before(const Best& a, const Best& b) {
  return a.value > b.value || (a.value == b.value && a.index < b.index);
}
__device__ __forceinline__ Best block_best(Best x, Best* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const Best y = {__shfl_xor(x.value, o, 64), __shfl_xor(x.index, o, 64)};
    if (before(y, x)) x = y;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  x = lds[0];
#pragma unroll
  for (int i = 1; i < kThreads / 64; ++i)
    if (before(lds[i], x)) x = lds[i];
  return x;
}

// part `blockIdx.x` of row `blockIdx.y`: (maximum, sum of exponentials beside
// it) into stat, the best `keep` as ordered(logit) << 32 | ~index into cand, in
// their order, 0 where there are fewer
template <DecodeType T>
__global__ void __launch_bounds__(kThreads) beam_rows_kernel(BeamSelectArgs a) {
  constexpr int EB = T == kF32 ? 4 : 2, GE = 16 / EB, GT = kRow / GE;  // elements of 16 bytes, those of a thread
  __shared__ float s_f[4];
  __shared__ double s_d[4];
  __shared__ uint32_t s_u[4];
  __shared__ u64 s_list[kList];
  __shared__ Best s_best[4];
  __shared__ int s_n;
  const int row = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const float score = a.scores[row];
  if ((a.finished && a.finished[row]) || !(fabsf(score) < INFINITY)) return;  // the logits do not matter
  const unsigned char* p = static_cast<const unsigned char*>(a.logits) +
                           (row / a.beams * a.s_request + row % a.beams * a.s_beam) * EB;
  // 16-byte pieces counted from the multiple of 16 at or before the row's start
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) / EB;
  const int pieces = (skew + a.vocab + GE - 1) / GE;
  const int per = (pieces + a.parts - 1) / a.parts, end = min(pieces, (part + 1) * per);
  float x[kRow];
#pragma unroll
  for (int i = 0; i < GT; ++i) {
    const int pc = part * per + i * kThreads + tid;
    const int v0 = pc * GE - skew;
    if (pc < end && v0 >= 0 && v0 + GE <= a.vocab) {
      const v4u u = *reinterpret_cast<const v4u*>(p + static_cast<int64_t>(v0) * EB);
#pragma unroll
      for (int e = 0; e < GE; ++e)
        x[i * GE + e] = to_float<T>(EB == 4 ? u[e % 4] : (u[e / 2] >> (16 * (e & 1))) & 0xffffu);
    } else {
#pragma unroll
      for (int e = 0; e < GE; ++e) {
        x[i * GE + e] = -INFINITY;
        if (pc < end && v0 + e >= 0 && v0 + e < a.vocab) {
          if constexpr (EB == 4) x[i * GE + e] = reinterpret_cast<const float*>(p)[v0 + e];
          else x[i * GE + e] = to_float<T>(reinterpret_cast<const uint16_t*>(p)[v0 + e]);
        }
      }
    }
  }
  float most = -INFINITY;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < kRow; ++i) {
    x[i] += 0.f;  // -0 is +0
    odd |= !(x[i] < INFINITY);
    most = fmaxf(most, x[i]);
  }
  uint32_t bound = wave_bound(ordered(most), a.keep);
  float m = most;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if (__any(odd)) m = INFINITY;
  if (lane == 0) s_f[w] = m, s_u[w] = bound;
  if (tid == 0) s_n = 0;
  __syncthreads();
  m = fmaxf(fmaxf(s_f[0], s_f[1]), fmaxf(s_f[2], s_f[3]));
  bound = max(max(max(s_u[0], s_u[1]), max(s_u[2], s_u[3])), kNone + 1);
  double* stat = a.stat + (static_cast<int64_t>(row) * a.parts + part) * 2;
  u64* cand = a.cand + (static_cast<int64_t>(row) * a.parts + part) * a.keep;
  if (!(fabsf(m) < INFINITY)) {  // nothing above -inf, or no row at all
    if (tid == 0) stat[0] = m, stat[1] = 0.0;
    for (int k = tid; k < a.keep; k += kThreads) cand[k] = 0;
    return;
  }
  // the difference first: its rounding is that of a small number
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kRow; ++i) sum += __builtin_amdgcn_exp2f((x[i] - m) * 1.44269504088896340736f);
  double all = sum;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o, 64);
  if (lane == 0) s_d[w] = all;
  auto key = [&](int i) {
    const int v = (part * per + i / GE * kThreads + tid) * GE - skew + i % GE;
    return static_cast<u64>(ordered(x[i])) << 32 | (0xffffffffu - static_cast<uint32_t>(v));
  };
  if (ordered(most) >= bound) {
#pragma unroll
    for (int i = 0; i < kRow; ++i)
      if (ordered(x[i]) >= bound) {
        const int at = atomicAdd(&s_n, 1);  // (any order: the list is ranked)
        if (at < kList) s_list[at] = key(i);
      }
  }
  __syncthreads();
  if (tid == 0) stat[0] = m, stat[1] = s_d[0] + s_d[1] + s_d[2] + s_d[3];
  const int n = s_n;
  if (n <= kList) {
    for (int c = tid; c < n; c += kThreads) {
      const u64 mine = s_list[c];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += s_list[i] > mine;
      if (rank < a.keep) cand[rank] = mine;
    }
    for (int k = n + tid; k < a.keep; k += kThreads) cand[k] = 0;
    return;
  }
  u64 last = ~0ull;
  for (int k = 0; k < a.keep; ++k) {
    Best b = {0, 0};
#pragma unroll
    for (int i = 0; i < kRow; ++i) {
      const u64 c = key(i);
      if (ordered(x[i]) > kNone && c < last && c > b.value) b.value = c;
    }
    b = block_best(b, s_best);
    last = b.value;
    if (tid == 0) cand[k] = last;
  }
}

// a request's beams: their log-sum-exp, the scores of what the parts kept, and
// the best of them
__global__ void __launch_bounds__(kThreads) beam_join_kernel(BeamSelectArgs a) {
  __shared__ Best s_list[kList];
  __shared__ Best s_best[4];
  __shared__ uint32_t s_u[4];
  __shared__ int s_n;
  extern __shared__ __attribute__((aligned(16))) double s_lse[];  // [beams], +inf: no continuation by its logits
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row0 = static_cast<int64_t>(b) * a.beams;
  auto ends = [&](int j) { return a.finished && a.finished[row0 + j]; };
  for (int j = tid; j < a.beams; j += kThreads) {
    const double* stat = a.stat + (row0 + j) * a.parts * 2;
    double lse = INFINITY;
    if (!ends(j) && fabsf(a.scores[row0 + j]) < INFINITY) {
      double m = -INFINITY;
      for (int i = 0; i < a.parts; ++i) m = fmax(m, stat[2 * i]);
      if (fabs(m) < INFINITY) {
        double sum = 0.0;
        for (int i = 0; i < a.parts; ++i) sum += stat[2 * i + 1] * exp(stat[2 * i] - m);
        lse = m + log(sum);
      }
    }
    s_lse[j] = lse;
  }
  if (tid == 0) s_n = 0;
  __syncthreads();
  const int per = a.parts * a.keep;
  const int64_t all = static_cast<int64_t>(a.beams) * per;
  // candidate c: the (c / lists)-th of list c % lists, so that a wave's lanes see the lists' heads
  const int lists = a.beams * a.parts;
  auto score = [&](int64_t c) {  // value 0: none
    const int rank = static_cast<int>(c / lists), list = static_cast<int>(c - static_cast<int64_t>(rank) * lists);
    const int j = list / a.parts, part = list - j * a.parts;
    const double s = a.scores[row0 + j];
    if (ends(j)) {
      if (rank != 0 || part != 0 || !(fabs(s) < INFINITY)) return Best{0, 0};
      return Best{ordered(s + 0.0), static_cast<u64>(j) * a.vocab + a.eos};
    }
    if (s_lse[j] == INFINITY) return Best{0, 0};
    const u64 k = a.cand[(row0 + j) * per + part * a.keep + rank];
    if (k == 0) return Best{0, 0};
    const double x = s + (unordered(static_cast<uint32_t>(k >> 32)) - s_lse[j]);
    return Best{ordered(x + 0.0), static_cast<u64>(j) * a.vocab + (0xffffffffu - static_cast<uint32_t>(k))};
  };
  uint32_t most = 0;  // the upper halves do for a bound
  for (int64_t c = tid; c < all; c += kThreads) most = max(most, static_cast<uint32_t>(score(c).value >> 32));
  uint32_t bound = wave_bound(most, a.keep);
  if (lane == 0) s_u[w] = bound;
  __syncthreads();
  bound = max(max(s_u[0], s_u[1]), max(max(s_u[2], s_u[3]), 1u));
  for (int64_t c = tid; c < all; c += kThreads) {
    const Best x = score(c);
    if (static_cast<uint32_t>(x.value >> 32) >= bound) {
      const int at = atomicAdd(&s_n, 1);  // (any order: the list is ranked)
      if (at < kList) s_list[at] = x;
    }
  }
  __syncthreads();
  const int n = s_n;
  auto put = [&](int k, const Best& x, bool some) {
    const int64_t at = static_cast<int64_t>(b) * a.keep + k;
    a.out_scores[at] = some ? static_cast<float>(unordered(x.value)) : -INFINITY;
    a.out_parent[at] = some ? static_cast<int64_t>(x.index / a.vocab) : 0;
    a.out_token[at] = some ? static_cast<int64_t>(x.index % a.vocab) : 0;
  };
  if (n <= kList) {
    for (int c = tid; c < n; c += kThreads) {
      const Best mine = s_list[c];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += before(s_list[i], mine);
      if (rank < a.keep) put(rank, mine, true);
    }
    for (int k = n + tid; k < a.keep; k += kThreads) put(k, Best{0, 0}, false);
    return;
  }
  Best last = {~0ull, 0};
  for (int k = 0; k < a.keep; ++k) {
    Best x = {0, ~0ull};
    for (int64_t c = tid; c < all; c += kThreads) {
      const Best y = score(c);
      if (before(last, y) && before(y, x)) x = y;
    }
    x = block_best(x, s_best);
    last = x;
    if (tid == 0) put(k, x, x.value != 0);
  }
}

template <DecodeType T>
void launch_type(const BeamSelectArgs& a, hipStream_t stream) {
  COMMEFF_LAUNCH(beam_rows_kernel<T>, dim3(static_cast<uint32_t>(a.parts), static_cast<uint32_t>(a.requests * a.beams)),
                 dim3(kThreads), 0, stream, a);
}

}  // namespace

// equal parts of at most 8,192 logits, whatever the row's alignment adds
int beam_select_parts(int vocab, DecodeType t) {
  const int ge = t == kF32 ? 4 : 8, most = kThreads * kRow / ge;
  return ((vocab + ge - 1) / ge + 1 + most - 1) / most;
}

void launch_beam_select(const BeamSelectArgs& a, DecodeType t, hipStream_t stream) {
  if (a.requests == 0) return;
  if (t == kBf16) launch_type<kBf16>(a, stream);
  else if (t == kF16) launch_type<kF16>(a, stream);
  else launch_type<kF32>(a, stream);
  COMMEFF_LAUNCH(beam_join_kernel, dim3(static_cast<uint32_t>(a.requests)), dim3(kThreads),
                 static_cast<uint32_t>(a.beams) * 8, stream, a);
}

}  // namespace commeff
