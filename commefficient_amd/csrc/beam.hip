// Beam search's selection: of the beams x vocabulary continuations of a
// request, the `keep` best by
//   score(j, v) = scores[j] + x[j, v] - log sum_u exp x[j, u],
// equal scores by the lower j, then the lower v.  A finished beam goes on with
// `eos` alone, at its own score.  A beam has no continuation where its score
// or its log-sum-exp is not finite (a NaN or +inf logit, no logit above -inf),
// nor has a token whose logit is -inf; places that nothing is left for hold
// (-inf, 0, 0).
#include <hip/hip_runtime.h>
#include <cstdint>
#include "decode.h"

namespace commeff {
namespace {

template <DecodeType T>
__device__ __forceinline__ float ldx(const void* p, int64_t i);
template <>
__device__ __forceinline__ float ldx<kBf16>(const void* p, int64_t i) {
  return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
}
template <>
__device__ __forceinline__ float ldx<kF16>(const void* p, int64_t i) {
  return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<const uint16_t*>(p)[i]));
}
template <>
__device__ __forceinline__ float ldx<kF32>(const void* p, int64_t i) {
  return static_cast<const float*>(p)[i];
}

// one workgroup per request: the beams' log-sum-exp, then `keep` rounds of an
// argmax over every continuation that is behind the last one taken
template <DecodeType T>
__global__ void __launch_bounds__(256) beam_select_kernel(BeamSelectArgs a) {
  __shared__ double s_val[256];
  __shared__ int64_t s_idx[256];
  __shared__ float s_f[256];
  extern __shared__ double s_lse[];  // [beams]
  const int b = blockIdx.x, tid = threadIdx.x;
  for (int j = 0; j < a.beams; ++j) {
    const int64_t at = b * a.s_request + j * a.s_beam;
    float m = -INFINITY;
    bool odd = false;
    for (int v = tid; v < a.vocab; v += 256) {
      const float x = ldx<T>(a.logits, at + v);
      odd |= x != x || x == INFINITY;
      m = fmaxf(m, x);
    }
    s_f[tid] = odd ? INFINITY : m;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
      if (tid < o) s_f[tid] = fmaxf(s_f[tid], s_f[tid + o]);
      __syncthreads();
    }
    m = s_f[0];
    double sum = 0.0;
    if (m > -INFINITY && m < INFINITY)
      for (int v = tid; v < a.vocab; v += 256) sum += expf(ldx<T>(a.logits, at + v) - m);
    s_val[tid] = sum;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
      if (tid < o) s_val[tid] += s_val[tid + o];
      __syncthreads();
    }
    if (tid == 0) s_lse[j] = m > -INFINITY && m < INFINITY ? m + log(s_val[0]) : INFINITY;
    __syncthreads();
  }
  double last = INFINITY;
  int64_t last_i = -1;
  const int64_t all = static_cast<int64_t>(a.beams) * a.vocab;
  for (int k = 0; k < a.keep; ++k) {
    double best = -INFINITY;
    int64_t best_i = -1;
    for (int j = 0; j < a.beams; ++j) {
      const double s = a.scores[b * a.beams + j];
      if (!(s > -INFINITY && s < INFINITY)) continue;
      const bool fin = a.finished && a.finished[b * a.beams + j];
      if (!fin && s_lse[j] == INFINITY) continue;
      const int64_t at = b * a.s_request + j * a.s_beam;
      for (int v = tid; v < a.vocab; v += 256) {
        if (fin && v != a.eos) continue;
        const double x = fin ? s : s + (ldx<T>(a.logits, at + v) - s_lse[j]);
        const int64_t i = static_cast<int64_t>(j) * a.vocab + v;
        const bool behind = x < last || (x == last && i > last_i);
        if (behind && x > best) {  // (a thread's own i only grow)
          best = x;
          best_i = i;
        }
      }
    }
    s_val[tid] = best;
    s_idx[tid] = best_i < 0 ? all : best_i;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
      if (tid < o && (s_val[tid + o] > s_val[tid] || (s_val[tid + o] == s_val[tid] && s_idx[tid + o] < s_idx[tid]))) {
        s_val[tid] = s_val[tid + o];
        s_idx[tid] = s_idx[tid + o];
      }
      __syncthreads();
    }
    last = s_val[0];
    last_i = s_idx[0];
    __syncthreads();
    if (tid == 0) {
      const bool some = last > -INFINITY;
      a.out_scores[b * a.keep + k] = static_cast<float>(last);
      a.out_parent[b * a.keep + k] = some ? last_i / a.vocab : 0;
      a.out_token[b * a.keep + k] = some ? last_i % a.vocab : 0;
    }
  }
}

}  // namespace

int beam_select_parts(int) { return 1; }

void launch_beam_select(const BeamSelectArgs& a, DecodeType t, hipStream_t stream) {
  if (a.requests == 0 || a.keep == 0) return;
  const dim3 grid(static_cast<uint32_t>(a.requests));
  const uint32_t lds = static_cast<uint32_t>(a.beams) * 8;
  if (t == kBf16) COMMEFF_LAUNCH(beam_select_kernel<kBf16>, grid, dim3(256), lds, stream, a);
  else if (t == kF16) COMMEFF_LAUNCH(beam_select_kernel<kF16>, grid, dim3(256), lds, stream, a);
  else COMMEFF_LAUNCH(beam_select_kernel<kF32>, grid, dim3(256), lds, stream, a);
}

}  // namespace commeff
