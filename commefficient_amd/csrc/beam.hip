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
// a score: a workgroup holds up to 16,384 of a row's logits (8,192
// in fp32) in registers, takes
// their maximum, the sum of exponentials beside it and the `keep` best of
// them.  The second turns what is left of a request (beams x parts x keep)
// into scores.
//
// Candidates of different beams are in the order of 64 bits.  Scores are formed in
// 64 bits, but the sums' exponentials are the hardware's: a term beside its wave's
// maximum m is off by 2^-24 x (1 for x - m, 1.25 for its product with log2 e) |x - m|,
// 2^-23 for exp2 (1.42 x 2^-24 at most, measured) and 3 x 2^-24 for the fp32 sum of a
// 16-byte piece; everything above that is in 64 bits.  The mean of |x - m| under the
// softmax is at most log(vocabulary) (entropy), so a log-sum-exp is off by at most
// 2^-24 (5 + 2.25 log(vocabulary)).  Where two candidates of different beams, one of
// them among the `keep` best, are closer than twice that (one request of 8 beams and 16
// places in a thousand), the join sums those beams' rows again in 64 bits, by index, so
// that equal rows give equal sums wherever they lie, and chooses anew: 17 us a row of
// 50,262 logits, which other requests do not wait for.
//
// The best of many by a threshold: of the 64 lanes of a wave, at least `keep`
// hold an element that is no less than the keep-th largest of the lanes' own
// maxima, so nothing below that (the largest such of the waves) can be among
// the `keep` best.  It is found by bits with a ballot a bit, some 2 keep to 4
// keep elements pass, and those are ranked by counting.  Where more than the
// lists hold pass (thousands of equal logits; `keep` near 64, where the bound is the
// least of a wave's lanes) `keep` rounds of an argmax take over: 16 rows of 50,262
// logits 450 us for 64 places.
#include <hip/hip_runtime.h>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include "conv_common.h"
#include "decode.h"

namespace commeff {
namespace {

constexpr int kThreads = 256;
static_assert(kBeamWaves == kThreads / 64, "a sum of every wave");
constexpr int kPieces = 8;   // 16-byte pieces of a row that a thread holds
constexpr int kList = 256;   // candidates of a wave that are ranked by counting
constexpr int kJoinList = 1024;  // .. of the join

constexpr float kLog2e = 1.44269504088896340736f;

typedef unsigned long long u64;

template <DecodeType T>
__device__ __forceinline__ float to_float(uint32_t bits) {  // of one element
  if constexpr (T == kBf16) return bf2f(bits);
  else if constexpr (T == kF16) return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
  else return __uint_as_float(bits);
}

template <DecodeType T>
constexpr uint32_t kLow = T == kBf16 ? 0xff80ff80u : T == kF16 ? 0xfc00fc00u : 0xff800000u;  // -inf

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

// 64 x 8 rows of 50,262 bf16 logits, a quarter of them at their end: 18 us for
// 39 MB, bound by the chain of its phases (loads, maxima, search, exponentials,
// list, ranks), which all parts walk at about the same time: nearly the whole grid
// is resident at once; four rows 7 us.
// Part `blockIdx.x` of row `blockIdx.y`: every wave's (maximum, sum of exponentials
// beside it) into stat, the best `keep` as ordered(logit) << 32 | ~index into cand, in
// their order, 0 where there are fewer
template <DecodeType T>
__global__ void __launch_bounds__(kThreads) beam_rows_kernel(BeamSelectArgs a) {
  constexpr int EB = T == kF32 ? 4 : 2, GE = 16 / EB;  // elements of 16 bytes
  __shared__ uint32_t s_u[4];
  __shared__ u64 s_list[4][kList];
  __shared__ Best s_best[4];
  __shared__ int s_n[4];
  __shared__ uint32_t s_v[64];
  const int row = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const float score = a.scores[row];
  if ((a.finished && a.finished[row]) || !(fabsf(score) < INFINITY)) return;  // the logits do not matter
  const int64_t req = a.by_beams.of(row);
  const unsigned char* p = static_cast<const unsigned char*>(a.logits) +
                           (req * a.s_request + (row - req * a.beams) * a.s_beam) * EB;
  // 16-byte pieces counted from the multiple of 16 at or before the row's start
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) / EB;
  const int pieces = (skew + a.vocab + GE - 1) / GE;
  const int per = a.by_parts.of(pieces + a.parts - 1), end = min(pieces, (part + 1) * per);
  // pieces by thread; where they are too few for a bound, over all waves: their
  // lists then hold every element
  const int mine_pc = part * per + (per < a.keep ? lane * 4 + w : tid);
  v4u u[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int pc = mine_pc + i * kThreads;
    const int v0 = pc * GE - skew;
    u[i] = v4u{kLow<T>, kLow<T>, kLow<T>, kLow<T>};
    if (pc < end && v0 >= 0 && v0 + GE <= a.vocab) {
      u[i] = *reinterpret_cast<const v4u*>(p + static_cast<int64_t>(v0) * EB);
    } else if (pc < end) {  // the row's ends: element by element
#pragma unroll
      for (int e = 0; e < GE; ++e)
        if (v0 + e >= 0 && v0 + e < a.vocab) {
          if constexpr (EB == 4) u[i][e] = reinterpret_cast<const uint32_t*>(p)[v0 + e];
          else u[i][e / 2] = (u[i][e / 2] & (0xffffu << (16 * (1 - (e & 1))))) |
                             static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[v0 + e]) << (16 * (e & 1));
        }
    }
  }
  auto at = [&](int i, int e) {  // element e of piece i
    return to_float<T>(EB == 4 ? u[i][e % 4] : (u[i][e / 2] >> (16 * (e & 1))) & 0xffffu);
  };
  float top[kPieces];
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    top[i] = at(i, 0);
#pragma unroll
    for (int e = 1; e < GE; ++e) top[i] = fmaxf(top[i], at(i, e));
    most = fmaxf(most, top[i]);
  }
  // (unpacked again for each use: held, the numbers would cost half the waves)
  auto anew = [&] {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) asm volatile("" : "+v"(u[i]));
  };
  anew();
  uint32_t bound = wave_bound(ordered(most + 0.f), a.keep);
  float m = most;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  // the exponentials beside the wave's own maximum; the difference first, so
  // that its rounding is that of a small number.  NaN (+inf - inf too) stays.
  const float beside = fmaxf(m, -FLT_MAX);
  double all = 0.0;
#pragma unroll
  for (int i = 0; i < kPieces; ++i)
    if (i * kThreads < per) {  // (a whole piece of the workgroup: rows shorter than its registers)
      float x[GE];
#pragma unroll
      for (int e = 0; e < GE; ++e) x[e] = __builtin_amdgcn_exp2f((at(i, e) - beside) * kLog2e);
#pragma unroll
      for (int o = 1; o < GE; o *= 2)
#pragma unroll
        for (int e = 0; e < GE; e += 2 * o) x[e] += x[e + o];
      all += x[0];
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o, 64);
  if (lane == 0) {  // (a NaN: no row at all)
    double* stat = a.stat + ((static_cast<int64_t>(row) * a.parts + part) * kBeamWaves + w) * 2;
    stat[0] = all != all ? INFINITY : m, stat[1] = all;
    s_u[w] = bound;
  }
  if (a.tight) {  // the waves' best lanes together: a bound for all four
    const u64 mask = __ballot(ordered(most + 0.f) >= bound);
    const int c = __popcll(mask & ((1ull << lane) - 1));
    if (lane < 16 && lane >= __popcll(mask)) s_v[w * 16 + lane] = 0;
    if ((mask >> lane & 1) && c < 16) s_v[w * 16 + c] = ordered(most + 0.f);
  }
  __syncthreads();
  bound = max(max(max(s_u[0], s_u[1]), max(s_u[2], s_u[3])), kNone + 1);
  if (a.tight) bound = max(bound, wave_bound(s_v[lane], a.keep));
  u64* cand = a.cand + (static_cast<int64_t>(row) * a.parts + part) * a.keep;
  auto key = [](float x, int v) {  // (-0 is +0)
    return static_cast<u64>(ordered(x + 0.f)) << 32 | (0xffffffffu - static_cast<uint32_t>(v));
  };
  anew();
  const float least = unordered(bound);  // (from -FLT_MAX on: a number)
  int mine = 0;  // of the wave's list
#pragma unroll
  for (int i = 0; i < kPieces; ++i)
    if (__any(top[i] >= least)) {
#pragma unroll
      for (int e = 0; e < GE; ++e) {
        const bool in = at(i, e) >= least;
        const u64 mask = __ballot(in);
        if (mask == 0) continue;
        const int c = mine + __popcll(mask & ((1ull << lane) - 1));
        if (in && c < kList) s_list[w][c] = key(at(i, e), (mine_pc + i * kThreads) * GE - skew + e);
        mine += __popcll(mask);
      }
    }
  if (lane == 0) s_n[w] = mine;
  __syncthreads();
  const int most_n = max(max(s_n[0], s_n[1]), max(s_n[2], s_n[3])), n = s_n[0] + s_n[1] + s_n[2] + s_n[3];
  if (most_n <= kList) {
    // four lanes a candidate, each against every fourth one of all lists
    for (int c = tid >> 2; c < n; c += kThreads / 4) {
      int l = 0, i0 = c;
      while (i0 >= s_n[l]) i0 -= s_n[l++];
      const u64 k = s_list[l][i0];
      int rank = 0;
      for (int q = 0; q < 4; ++q) {
        const int nq = s_n[q];
#pragma unroll 4
        for (int i = tid & 3; i < nq; i += 4) rank += s_list[q][i] > k;
      }
      rank += __shfl_xor(rank, 1, 64);
      rank += __shfl_xor(rank, 2, 64);
      if ((tid & 3) == 0 && rank < a.keep) cand[rank] = k;
    }
    for (int k = n + tid; k < a.keep; k += kThreads) cand[k] = 0;
    return;
  }
  u64 last = ~0ull;  // (the row again from the cache: rare, and no registers for it)
  for (int k = 0; k < a.keep; ++k) {
    Best b = {0, 0};
    for (int pc = part * per + tid; pc < end; pc += kThreads)
      for (int v = max(pc * GE - skew, 0); v < min((pc + 1) * GE - skew, a.vocab); ++v) {
        float x;
        if constexpr (EB == 4) x = reinterpret_cast<const float*>(p)[v];
        else x = to_float<T>(reinterpret_cast<const uint16_t*>(p)[v]);
        const u64 c = key(x, v);
        if (x > -INFINITY && c < last && c > b.value) b.value = c;
      }
    b = block_best(b, s_best);
    last = b.value;
    if (tid == 0) cand[k] = last;
  }
}

// exp(x), x <= 0, from -700 on e^-700: 2^n e^r with n next to x / log 2 (the low bits of a sum that holds
// no fraction), |r| < 0.35 and e^r its series to 4e-18; off by some 1e-15
__device__ __forceinline__ double exp64(double x) {
  constexpr double kLog2 = 0.69314718055994530942, kHi = 0x1.62e42fefap-1;  // (the upper part of log(2))
  constexpr double kWhole = 0x1.8p52;
  x = fmax(x, -700.0);
  constexpr double kTerm[14] = {1.0, 1.0, 0.5, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320,
                                1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800, 1.0 / 479001600, 1.0 / 6227020800.0};
  const double sum = fma(x, 1.0 / kLog2, kWhole), n = sum - kWhole;
  const double r = fma(n, -(kLog2 - kHi), fma(n, -kHi, x));
  double e = kTerm[13];
#pragma unroll
  for (int i = 12; i >= 0; --i) e = fma(e, r, kTerm[i]);
  const u64 up = static_cast<u64>(static_cast<uint32_t>(__builtin_bit_cast(u64, sum))) << 52;
  return __builtin_bit_cast(double, __builtin_bit_cast(u64, e) + up);  // (2^n into the exponent)
}

// a thread's part of a row's sum of exp(x - m): every 256th 16 bytes from the row's first
// element on, whatever its alignment; seven loads on their way under the eighth's terms
template <DecodeType T>
__device__ __forceinline__ double row_sum(const BeamSelectArgs& a, int64_t at, double m) {
  constexpr int EB = T == kF32 ? 4 : 2, GE = 16 / EB, kAhead = 8;
  const unsigned char* p = static_cast<const unsigned char*>(a.logits) + at * EB;
  const int full = a.vocab / GE, tid = threadIdx.x;
  auto load = [&](int i) {
    v4u u = {kLow<T>, kLow<T>, kLow<T>, kLow<T>};
    if (i < full) __builtin_memcpy(&u, p + static_cast<int64_t>(i) * 16, 16);
    return u;
  };
  v4u u[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) u[i] = load(tid + i * kThreads);
  double sum = 0.0;
  for (int i = tid; i < full; i += kThreads) {
    const v4u now = u[0];
#pragma unroll
    for (int k = 0; k + 1 < kAhead; ++k) u[k] = u[k + 1];
    u[kAhead - 1] = load(i + kAhead * kThreads);
#pragma unroll
    for (int e = 0; e < GE; ++e)
      sum += exp64(to_float<T>(EB == 4 ? now[e % 4] : (now[e / 2] >> (16 * (e & 1))) & 0xffffu) - m);
  }
  const int v = full * GE + tid;
  if (v < a.vocab) {
    uint32_t x = 0;
    __builtin_memcpy(&x, p + static_cast<int64_t>(v) * EB, EB);
    sum += exp64(to_float<T>(x) - m);
  }
  return sum;
}

// a request's beams: their log-sum-exp, the scores of what the parts kept, and
// the best of them.  Bound by latency (one request of 4 beams 4.7 us, 64 of 8
// beams 7.5): the first candidates are on their way while the sums are joined
// (a wave a beam), and stay in registers.
__global__ void __launch_bounds__(kThreads) beam_join_kernel(BeamSelectArgs a) {
  constexpr int kHeld = 4;  // candidates a thread holds
  __shared__ Best s_list[kJoinList], s_sorted[kJoinList];
  __shared__ Best s_best[4];
  __shared__ double s_sum[4];
  __shared__ uint32_t s_u[2][4];
  __shared__ uint32_t s_again[kBeamMaxBeams / 32];  // a bit a beam: its sum in 64 bits
  __shared__ int s_n, s_near;
  extern __shared__ __attribute__((aligned(16))) double s_lse[];  // [beams], +inf: no continuation by its logits
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row0 = static_cast<int64_t>(b) * a.beams;
  auto ends = [&](int j) { return a.finished && a.finished[row0 + j]; };
  auto alive = [&](int j) { return !ends(j) && fabsf(a.scores[row0 + j]) < INFINITY; };
  // candidate c: the (c / lists)-th of list c % lists, so that a wave's lanes see the lists' heads
  const int lists = a.beams * a.parts, all = lists * a.keep, stats = a.parts * kBeamWaves;
  auto place = [&](int c, int& rank, int& list, int& j) {
    rank = a.by_lists.of(c);
    list = c - rank * lists;
    j = a.by_parts.of(list);
  };
  auto fetch = [&](int c) {
    int rank, list, j;
    place(c, rank, list, j);
    return a.cand[(row0 * a.parts + list) * a.keep + rank];  // (of a beam that has none: not looked at)
  };
  u64 held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = tid + i * kThreads < all ? fetch(tid + i * kThreads) : 0;
  double size = 0.0;  // of what a score is formed from
  for (int j = w; j < a.beams; j += kThreads / 64) {
    double lse = INFINITY;
    const double* stat = a.stat + (row0 + j) * stats * 2;
    double m = -INFINITY, sum = 0.0;
    for (int i = lane; i < stats; i += 64) m = fmax(m, stat[2 * i]);
    if (alive(j)) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m = fmax(m, __shfl_xor(m, o, 64));
      if (fabs(m) < INFINITY) {
        for (int i = lane; i < stats; i += 64)
          if (stat[2 * i + 1] > 0.0) sum += stat[2 * i + 1] * exp(stat[2 * i] - m);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        lse = m + log(sum);
        size = fmax(size, fabs(lse) + fabsf(a.scores[row0 + j]));
      }
    }
    if (lane == 0) s_lse[j] = lse;
  }
  if (lane == 0) s_sum[w] = size;
  if (tid < kBeamMaxBeams / 32) s_again[tid] = 0;
  if (tid == 0) s_n = s_near = 0;
  __syncthreads();
  // closer than this: the order is not certain (64-bit roundings of large scores, too)
  const double near = a.near + 0x1p-50 * fmax(fmax(s_sum[0], s_sum[1]), fmax(s_sum[2], s_sum[3]));
  auto score = [&](int c, u64 k) {  // value 0: none; index: beam << 32 | token
    int rank, list, j;
    place(c, rank, list, j);
    const double s = a.scores[row0 + j];
    const u64 beam = static_cast<u64>(j) << 32;
    if (ends(j)) {
      if (rank != 0 || list != j * a.parts || !(fabs(s) < INFINITY)) return Best{0, 0};
      return Best{ordered(s + 0.0), beam | static_cast<u64>(a.eos)};
    }
    if (k == 0 || s_lse[j] == INFINITY) return Best{0, 0};
    const double x = s + (unordered(static_cast<uint32_t>(k >> 32)) - s_lse[j]);
    return Best{ordered(x + 0.0), beam | (0xffffffffu - static_cast<uint32_t>(k))};
  };
  auto put = [&](int k, const Best& x, bool some) {
    const int64_t at = static_cast<int64_t>(b) * a.keep + k;
    a.out_scores[at] = some ? static_cast<float>(unordered(x.value)) : -INFINITY;
    a.out_parent[at] = some ? static_cast<int64_t>(x.index >> 32) : 0;
    a.out_token[at] = some ? static_cast<int64_t>(x.index & 0xffffffffu) : 0;
  };
  Best mine[kHeld];
  uint32_t most = 0;  // the upper halves do for a bound
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    mine[i] = tid + i * kThreads < all ? score(tid + i * kThreads, held[i]) : Best{0, 0};
    most = max(most, static_cast<uint32_t>(mine[i].value >> 32));
  }
  for (int c = tid + kHeld * kThreads; c < all; c += kThreads)
    most = max(most, static_cast<uint32_t>(score(c, fetch(c)).value >> 32));
  // the upper half of the keep-th largest of all candidates (or less by bits that do not
  // matter), by bits
  auto counted = [&] {
    uint32_t bound = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = bound | 1u << bit;
      int n = 0;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) n += __popcll(__ballot(static_cast<uint32_t>(mine[i].value >> 32) >= c));
      for (int i = kHeld * kThreads; i < all; i += kThreads)
        n += __popcll(__ballot(i + tid < all && static_cast<uint32_t>(score(i + tid, fetch(i + tid)).value >> 32) >= c));
      if (lane == 0) s_u[bit & 1][w] = n;
      __syncthreads();  // (the other half is read until the next one)
      n = s_u[bit & 1][0] + s_u[bit & 1][1] + s_u[bit & 1][2] + s_u[bit & 1][3];
      if (n >= a.keep) bound = c;
      if (n == a.keep) break;
    }
    return bound;
  };
  int n = 0;
  auto pass = [&](const Best& x, uint32_t bound) {
    if (static_cast<uint32_t>(x.value >> 32) >= bound) {
      const int at = atomicAdd(&s_n, 1);  // (any order: the list is ranked)
      if (at < kJoinList) s_list[at] = x;
    }
  };
  auto make_list = [&](uint32_t bound) {
    // (down to what may belong above it; up to 0x000fffff no number's upper half)
    if (bound > 0x000fffffu) {
      const double x = unordered(static_cast<u64>(bound) << 32);
      bound = static_cast<uint32_t>(ordered(x - near - 0x1p-50 * fabs(x)) >> 32);
    }
    bound = max(bound, 1u);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) pass(mine[i], bound);
    for (int c = tid + kHeld * kThreads; c < all; c += kThreads) pass(score(c, fetch(c)), bound);
    __syncthreads();
    n = s_n;
  };
  const bool held_all = all <= kHeld * kThreads;
  if (a.keep <= 32 || !held_all) {
    const uint32_t bound = wave_bound(most, a.keep);
    if (lane == 0) s_u[0][w] = bound;
    __syncthreads();
    make_list(max(max(s_u[0][0], s_u[0][1]), max(s_u[0][2], s_u[0][3])));
  } else {
    // many places: counted, so that few more than those are left to rank (8 requests of 16
    // beams, 64 places: 16 against 131 us; for up to 32 the search costs what it saves)
    make_list(counted());
  }
  if (n > kJoinList && !held_all) {
    // .. and where the list does not hold what the waves' bound lets pass (16 beams of
    // 50,262, 64 places: 92 against 400 us)
    __syncthreads();
    if (tid == 0) s_n = 0;
    make_list(counted());  // (barriers in it)
  }
  auto rank_list = [&] {
    for (int c = tid >> 2; c < n; c += kThreads / 4) {
      const Best x = s_list[c];
      int rank = 0;
#pragma unroll 4
      for (int i = tid & 3; i < n; i += 4) rank += before(s_list[i], x);
      rank += __shfl_xor(rank, 1, 64);
      rank += __shfl_xor(rank, 2, 64);
      if ((tid & 3) == 0) s_sorted[rank] = x;
    }
    __syncthreads();
    for (int k = tid; k < a.keep; k += kThreads) put(k, k < n ? s_sorted[k] : Best{0, 0}, k < n);
  };
  if (n <= kJoinList) {
    rank_list();
    // Neighbours of different beams, one of them kept (or no further from the last
    // one kept): any two that are close have such neighbours between them.
    for (int i = tid; i + 1 < n; i += kThreads) {
      const int jx = static_cast<int>(s_sorted[i].index >> 32), jy = static_cast<int>(s_sorted[i + 1].index >> 32);
      if (jx == jy) continue;
      const double v = unordered(s_sorted[min(i, a.keep - 1)].value), u = unordered(s_sorted[i + 1].value);
      if (v - u <= near + 0x1p-50 * fabs(v)) {
        s_near = 1;
        atomicOr(&s_again[jx >> 5], 1u << (jx & 31));
        atomicOr(&s_again[jy >> 5], 1u << (jy & 31));
      }
    }
    __syncthreads();
    if (s_near == 0) return;
  } else if (a.beams > 1 && tid < kBeamMaxBeams / 32) {
    s_again[tid] = ~0u;
  }
  __syncthreads();
  // Rare: those beams' sums in 64 bits, and the list by them
  for (int j = 0; j < a.beams; ++j) {
    if (!(s_again[j >> 5] >> (j & 31) & 1) || !alive(j) || s_lse[j] == INFINITY) continue;
    double m = -INFINITY;
    for (int i = 0; i < stats; ++i) m = fmax(m, a.stat[((row0 + j) * stats + i) * 2]);
    const int64_t at = b * a.s_request + j * a.s_beam;
    double sum = 0.0;
    if (a.type == kF32) sum = row_sum<kF32>(a, at, m);
    else if (a.type == kBf16) sum = row_sum<kBf16>(a, at, m);
    else sum = row_sum<kF16>(a, at, m);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) s_sum[w] = sum;
    __syncthreads();
    if (tid == 0) s_lse[j] = m + log(s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]);
    __syncthreads();
  }
  if (n <= kJoinList) {
    for (int c = tid; c < n; c += kThreads) {
      const int j = static_cast<int>(s_list[c].index >> 32);
      if (ends(j)) continue;
      const int64_t at = b * a.s_request + j * a.s_beam + static_cast<int64_t>(s_list[c].index & 0xffffffffu);
      float x;
      if (a.type == kF32) x = static_cast<const float*>(a.logits)[at];
      else if (a.type == kBf16) x = to_float<kBf16>(static_cast<const uint16_t*>(a.logits)[at]);
      else x = to_float<kF16>(static_cast<const uint16_t*>(a.logits)[at]);
      s_list[c].value = ordered(a.scores[row0 + j] + (x - s_lse[j]) + 0.0);
    }
    __syncthreads();
    rank_list();
    return;
  }
  Best last = {~0ull, 0};
  for (int k = 0; k < a.keep; ++k) {
    Best x = {0, ~0ull};
    for (int c = tid; c < all; c += kThreads) {
      const Best y = score(c, fetch(c));
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

// equal parts of at most 2,048 pieces, whatever the row's alignment adds
int beam_select_parts(int vocab, DecodeType t) {
  const int ge = t == kF32 ? 4 : 8, most = kThreads * kPieces;
  return ((vocab + ge - 1) / ge + 1 + most - 1) / most;
}

void launch_beam_select(BeamSelectArgs a, DecodeType t, hipStream_t stream) {
  if (a.requests == 0) return;
  // a tighter bound costs a search more and saves passing elements: worth it
  // where throughput counts (64 x 8 beams 25.9 against 28.5 us), not for few
  // workgroups (1 x 4 beams 11.7 against 11.6); its table holds 16 of a wave
  a.tight = a.keep <= 16 && static_cast<int64_t>(a.requests) * a.beams * a.parts >= 512;
  a.type = t;
  a.near = 2.0 * 0x1p-24 * (5.0 + 2.25 * std::log(static_cast<double>(a.vocab)));
  a.by_beams = fast_div(a.beams);
  a.by_parts = fast_div(a.parts);
  a.by_lists = fast_div(static_cast<int64_t>(a.beams) * a.parts);
  if (t == kBf16) launch_type<kBf16>(a, stream);
  else if (t == kF16) launch_type<kF16>(a, stream);
  else launch_type<kF32>(a, stream);
  COMMEFF_LAUNCH(beam_join_kernel, dim3(static_cast<uint32_t>(a.requests)), dim3(kThreads),
                 static_cast<uint32_t>(a.beams) * 8, stream, a);
}

}  // namespace commeff
