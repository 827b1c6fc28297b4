// One new token of every sequence against its paged keys and values:
//   o[n, h] = sum_t softmax_t(scale q[n, h] . k[n, t, h / group]) v[n, t, h / group],
// t < lens[n], the keys read through table[n].  When the new token's own k, v
// rows are given they stand for position lens[n] - 1 and are stored into that
// slot by the same launch.  Rows without tokens, or with every score -inf, are
// 0; a row that meets a page id outside the cache, or is longer than its table
// row, is NaN and nothing is read or written through that id.
//
// Every key and value is read once for all `group` query heads that share it
// and used for 4 x group operations a number: bound by HBM, so the kernel is
// built around its loads.  A wave takes 32 tokens at a time of one (sequence,
// cache head); the group's heads (up to 16, the rest of the columns idle: the
// MFMA time is under a tenth of the loads' even so) are the columns of both
// products, computed transposed:
//   S^T [token, head] = K Q^T,   O^T [column, head] += V^T P^T.
// The MFMA's row order is free as long as both sides agree, and is chosen so
// that nothing moves between lanes:
//   * row m of key set s (s = 0, 1) is token 8 (m / 4) + 4 s + m % 4, so that
//     lane l's eight scores are tokens 8 (l / 16) .. + 7 of head l % 16: the
//     very operand layout that the second product wants for P^T;
//   * a lane loads 8 tokens x head_dim / 16 columns of V and transposes them
//     within its own registers (v_perm_b32) into rows of V^T.
// So K and V go from memory to the matrix cores without LDS.  Weights are fed
// as two 16-bit pieces (a rounding and its remainder: 2^-16 of a weight for
// bf16, 2^-22 for fp16), sums and maxima stay in fp32; fp32 caches use the
// fp32 MFMA.  A wave whose sums come out infinite or NaN takes its tiles a second
// time, so that an infinite value meets its weight once and not in two pieces.
// The running maximum is only raised when some score exceeds it by kSlack (in
// powers of two), which a wave votes on: the cross-lane maximum and the rescaling
// of O run a few times a sequence, not once a tile.
// Reached: 8 sequences of up to 65,536 tokens, 32 heads over 8 of 128, bf16:
// 1.21 GB at 4.9 to 5.0 TB/s; 128 x 8 heads of 128, up to 1,024 tokens: 271 MB at 4.6;
// 64 x 12 of 64: 103 MB in 27 us (a copy of as much 21); one short reply 6.5.
#include <hip/hip_runtime.h>
#include <cfloat>
#include <cstdint>
#include "conv_common.h"
#include "decode.h"

namespace commeff {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kTile = 32;       // tokens a wave takes at a time
constexpr int kMaxSplit = 64;   // parts of a sequence

template <bool B>
struct Flag {
  static constexpr bool value = B;
};

template <DecodeType T>
struct Elem;
template <>
struct Elem<kBf16> {
  typedef uint16_t t;
  static constexpr float kSlack = 8.f, kLift = 0.f;
  static constexpr uint32_t kExp = 0x7f80u, kUlp = 0x0080u;  // an exponent's bits, the lowest of them
  static __device__ __forceinline__ t store(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
  static __device__ __forceinline__ float load(t x) { return bf2f(x); }
  static __device__ __forceinline__ f32x4_t mfma(v4u a, v4u b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                   c, 0, 0, 0);
  }
};
template <>
struct Elem<kF16> {
  typedef uint16_t t;
  // weights reach 2^(1 + 12) < 65,504 and the smallest kept piece is 2^-24 / 2^12
  static constexpr float kSlack = 1.f, kLift = 12.f;
  static constexpr uint32_t kExp = 0x7c00u, kUlp = 0x0400u;
  static __device__ __forceinline__ t store(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  }
  static __device__ __forceinline__ float load(t x) { return static_cast<float>(__builtin_bit_cast(_Float16, x)); }
  static __device__ __forceinline__ f32x4_t mfma(v4u a, v4u b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                  0, 0, 0);
  }
};
template <>
struct Elem<kF32> {
  typedef float t;
  static constexpr float kSlack = 8.f, kLift = 0.f;
  static __device__ __forceinline__ t store(float f) { return f; }
};

// Waves a SIMD holds at least, by a token's row in bytes.  Many waves with one
// tile each in flight beat fewer that load the next tile under the products:
// 64 x 12 heads of 64 bf16, up to 1,024 tokens, 27.3 against 29.6 us.
constexpr int min_waves(int type, int dim, int few) {
  const int row = dim * (type == kF32 ? 4 : 2);
  return row <= (few == 1 ? 256 : 128) ? 4 : row <= 256 ? 3 : 2;
}

// what a lane holds of 32 tokens: dwords of K rows and of V columns
template <DecodeType T, int HD>
struct Tile {
  static constexpr int E = T == kF32 ? 4 : 2;      // bytes an element
  static constexpr int KL = HD * E / 64;           // 16-byte pieces a K row leaves to a lane
  static constexpr int NC = HD / 16;               // V columns a lane holds
  static constexpr int CH = NC * E > 16 ? 16 / E : NC;  // .. of them in one load
  // Rows of more than 256 bytes do not fit the registers of two waves a SIMD
  // at once: V comes in NP parts of columns, each on its way under the product
  // of the last, K of the widest a key set at a time, and Q waits in LDS.
  static constexpr int NP = HD * E > 256 ? HD * E / 256 : 1, NV = NC / NP;
  v4u k[NP > 2 ? 1 : 2][KL];
  uint32_t v[NP > 1 ? 2 : 1][8][NV * E / 4];
};
// column j of lane row m (of 16)
template <DecodeType T, int HD>
__device__ __forceinline__ int v_col(int m, int j) {
  constexpr int CH = Tile<T, HD>::CH;
  return (j / CH) * (16 * CH) + m * CH + j % CH;
}

// What of a lane's V pieces is infinite or NaN, times the weights' first pieces, into o; the
// pieces keep the rest.  One dword (two columns) after the other: no registers for all.
template <DecodeType T, int N>
__device__ __forceinline__ void take_odd(uint32_t (&v)[8][N], v4u hi, f32x4_t* o) {
  typedef Elem<T> E;
#pragma unroll
  for (int c = 0; c < N; ++c) {
    uint32_t odd[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      asm volatile("" : "+v"(v[i][c]));
      // (an exponent of all ones and one more: the half's sign bit)
      odd[i] = v[i][c] & ((((v[i][c] & (E::kExp * 0x10001u)) + E::kUlp * 0x10001u) >> 15 & 0x10001u) * 0xffffu);
      v[i][c] ^= odd[i];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      v4u vt;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        vt[i] = __builtin_amdgcn_perm(odd[2 * i + 1], odd[2 * i], j ? 0x07060302u : 0x05040100u);
      o[2 * c + j] = E::mfma(vt, hi, o[2 * c + j]);
    }
  }
}

// FEW > 0 (fp32, groups of FEW = 1 or 2 heads): the products on the
// vector units, head by head.  The fp32 MFMA works on 16 columns whatever the
// group needs, 8,192 cycles for 32 tokens of 256 columns against 1,100 a head
// here (4 sequences x 4 heads of 256, 600 tokens, 27.8 against 47.9 us; 33 x 12 of
// 64, up to 777 tokens, 22.1 against 28.0).  A lane then has the scores
// of tokens m16 of both key sets, summed over the lanes g, and its columns'
// sums of tokens 8 g .. + 7, joined at the end.
template <DecodeType T, int HD, int W, int FEW>
__global__ void __launch_bounds__(W * 64, min_waves(T, HD, FEW)) paged_attn_kernel(PagedAttnArgs a) {
  typedef Elem<T> E;
  typedef typename E::t S;
  typedef Tile<T, HD> Regs;
  constexpr int NC = Regs::NC, KL = Regs::KL, CH = Regs::CH, EB = Regs::E, NP = Regs::NP, NV = Regs::NV;
  extern __shared__ __attribute__((aligned(16))) float lds[];  // (Q) | W x min(group, 16) x (HD + 2)

  // On one XCD, at about the same time: the parts of a group of more than 16
  // heads, which read the same rows (16 x 8 heads, groups of 20, 4,096 tokens
  // 33.9 against 37.5 us), and neighbours in the batch (the beams of a request share pages).
  int id = xcd_remap(blockIdx.x, gridDim.x);
  int rest = a.by_tiles.of(id);
  const int gt = id - rest * static_cast<int>(a.by_tiles.d);
  id = rest;
  rest = a.by_n.of(id);
  const int n = id - rest * a.n, sp = a.by_kv.of(rest), kh = rest - sp * a.kv_heads;
  const int cols = min(16, a.group - 16 * gt);  // query heads of this workgroup
  const int h0 = kh * a.group + 16 * gt;

  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m16 = lane & 15, g = lane >> 4;
  const int32_t* row = a.table + n * a.table_ld;
  const int len = a.lens[n];
  // the first tile's page ids do not wait for the length where its place does not depend on it
  int early = 0;
  if (a.split == 1) {
    const int pg = a.by_page.of(w * kTile + (lane & 31));
    early = pg < a.width ? row[pg] : 0;
  }
  bool bad = len > static_cast<int64_t>(a.width) * a.page;
  const int all = len > 0 && !bad ? (len + kTile - 1) / kTile : 0;  // tiles of the sequence
  const int per = a.split == 1 ? all : a.by_split.of(all + a.split - 1);
  const int t_end = min(all, (sp + 1) * per);
  if (sp > 0 && sp * per >= all) return;  // (the join knows)

  const S* kn = a.k ? static_cast<const S*>(a.k) + n * a.k_row + kh * a.k_head : nullptr;
  const S* vn = a.k ? static_cast<const S*>(a.v) + n * a.v_row + kh * a.v_head : nullptr;
  S* const kc = static_cast<S*>(a.kc) + kh * a.kc_head;
  S* const vc = static_cast<S*>(a.vc) + kh * a.vc_head;

  // Tokens behind the last one read the last one's page instead: their scores
  // are masked and their V pieces cleared before the product.
  const int last = len - 1;
  const bool by8 = (a.page & 7) == 0;  // eight aligned tokens lie in one page
  auto sound = [&](int pid) {  // a page outside the cache is not followed
    const bool ok = pid >= 0 && pid < a.pages;
    bad |= !ok;
    return ok ? pid : 0;
  };
  auto look = [&](int tile) {  // the page of token lane % 32 of a tile
    return sound(row[a.by_page.of(min(tile * kTile + (lane & 31), last))]);
  };
  const S *kr[2], *vr[8];  // the lane's K and V rows of a tile
  auto point = [&](int tile, int ids) {
    const int base = tile * kTile;
    const bool fresh = kn && base + kTile > last;  // the tile with the new token
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = min(8 * (m16 >> 2) + 4 * s + (m16 & 3), last - base), tok = base + at;
      kr[s] = kc + __shfl(ids, at, 64) * a.kc_page + (tok - a.by_page.of(tok) * a.page) * a.kc_tok;
    }
    if (by8) {
      const int at = min(8 * g, (last - base) & ~7), tok = base + at;
      vr[0] = vc + __shfl(ids, at, 64) * a.vc_page + (tok - a.by_page.of(tok) * a.page) * a.vc_tok;
#pragma unroll
      for (int i = 1; i < 8; ++i) vr[i] = vr[i - 1] + a.vc_tok;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = min(8 * g + i, last - base), tok = base + at;
        vr[i] = vc + __shfl(ids, at, 64) * a.vc_page + (tok - a.by_page.of(tok) * a.page) * a.vc_tok;
      }
    }
    if (fresh) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (base + 8 * (m16 >> 2) + 4 * s + (m16 & 3) == last) kr[s] = kn;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (base + 8 * g + i == last) vr[i] = vn;
    }
  };
  auto load_k = [&](v4u(&k)[KL], int s) {
#pragma unroll
    for (int i = 0; i < KL; ++i) k[i] = *reinterpret_cast<const v4u*>(kr[s] + i * (64 / EB) + g * (16 / EB));
  };
  auto load_v = [&](uint32_t(&v)[8][NV * EB / 4], int part) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int c = 0; c < NV / CH; ++c) {
        const S* src = vr[i] + v_col<T, HD>(m16, part * NV + c * CH);
        uint32_t* dst = &v[i][c * CH * EB / 4];
        if constexpr (CH * EB == 16) {
          const v4u u = *reinterpret_cast<const v4u*>(src);
          dst[0] = u[0], dst[1] = u[1], dst[2] = u[2], dst[3] = u[3];
        } else if constexpr (CH * EB == 8) {
          const v2u u = *reinterpret_cast<const v2u*>(src);
          dst[0] = u[0], dst[1] = u[1];
        } else {
          dst[0] = *reinterpret_cast<const uint32_t*>(src);
        }
      }
    }
  };

  // Q^T: lane l holds head l % 16, the columns that it holds of a K row
  v4u* const lq = reinterpret_cast<v4u*>(lds);  // [KL][64], where it does not stay in registers
  v4u q[NP > 1 || FEW > 0 ? 1 : KL];
  auto q_of = [&](int i) {
    if (m16 >= cols) return v4u{0u, 0u, 0u, 0u};
    return *reinterpret_cast<const v4u*>(static_cast<const S*>(a.q) + n * a.q_row + (h0 + m16) * a.q_head +
                                         i * (64 / EB) + g * (16 / EB));
  };
  if constexpr (FEW > 0) {  // [FEW][KL][4 lanes g]
    for (int x = tid; x < FEW * KL * 4; x += W * 64) {
      const int h = x / (KL * 4), i = x / 4 % KL;
      v4u u = {0u, 0u, 0u, 0u};
      if (h < cols)
        u = *reinterpret_cast<const v4u*>(static_cast<const S*>(a.q) + n * a.q_row + (h0 + h) * a.q_head +
                                          i * (64 / EB) + x % 4 * (16 / EB));
      lq[x] = u;
    }
    __syncthreads();
  } else if constexpr (NP > 1) {
    for (int i = w; i < KL; i += W) lq[i * 64 + lane] = q_of(i);
    __syncthreads();
  } else {
#pragma unroll
    for (int i = 0; i < KL; ++i) q[i] = q_of(i);
  }
  const float scale = a.scale * 1.44269504088896340736f;  // scores in powers of two
  float top = -FLT_MAX, sum = 0.f;                        // of head l % 16; sum: this lane's tokens
  f32x4_t o[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  auto scores = [&](const v4u(&k)[KL]) {
    f32x4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      v4u qi;
      if constexpr (NP > 1) qi = lq[i * 64 + lane];
      else qi = q[i];
      if constexpr (T == kF32) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[i][e]), __uint_as_float(qi[e]), c, 0, 0, 0);
      } else {
        c = E::mfma(k[i], qi, c);
      }
    }
    return c;
  };
  // `flag`, careful: infinite and NaN values enter beside the first piece of their weight alone (0
  // where the weight is: 0 x inf is NaN, as in fp32), the finite ones as ever.  The second,
  // which may be 0 or negative, would make an infinity NaN.
  auto compute = [&](int tile, int& ids, int next, auto flag) {
    constexpr bool careful = decltype(flag)::value;
    Regs r;
    const int first = tile * kTile + 8 * g;
    f32x4_t s4[2];
    load_k(r.k[0], 0);
    if constexpr (NP <= 2) load_k(r.k[1], 1);
    load_v(r.v[0], 0);
    if (next >= 0) ids = look(next);  // (under this tile's loads)
    s4[0] = scores(r.k[0]);
    if constexpr (NP > 2) {
      load_k(r.k[0], 1);
      s4[1] = scores(r.k[0]);
    } else {
      s4[1] = scores(r.k[1]);
    }
    if constexpr (NP > 1) load_v(r.v[1], 1);
    float x[8], most = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = s4[i >> 2][i & 3] * scale;
      if (first + i >= len) x[i] = -INFINITY;
      most = fmaxf(most, x[i]);
    }
    if (__any(m16 < cols && most > top + E::kSlack)) {
      most = fmaxf(most, __shfl_xor(most, 16, 64));
      most = fmaxf(most, __shfl_xor(most, 32, 64));
      const float now = fmaxf(top, most), c = __builtin_amdgcn_exp2f(top - now);
      top = now;
      sum *= c;
#pragma unroll
      for (int j = 0; j < NC; ++j) o[j] *= c;
    }
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(x[i] - top + E::kLift);
      sum += p[i];
    }
    v4u hi, lo;
    if constexpr (T != kF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u0 = E::store(p[2 * i]), u1 = E::store(p[2 * i + 1]);
        hi[i] = u0 | u1 << 16;
        lo[i] = E::store(p[2 * i] - E::load(u0)) | static_cast<uint32_t>(E::store(p[2 * i + 1] - E::load(u1))) << 16;
        if constexpr (T == kF16 && careful)  // (2^-36 of the largest for weights too small for fp16)
          hi[i] |= (u0 == 0 && p[2 * i] != 0.f ? 1u : 0u) | (u1 == 0 && p[2 * i + 1] != 0.f ? 0x10000u : 0u);
      }
    }
#pragma unroll
    for (int part = 0; part < NP; ++part) {
      auto& v = r.v[part & (NP > 1 ? 1 : 0)];
      if (tile * kTile + kTile > len) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (first + i >= len) {
#pragma unroll
            for (int c = 0; c < NV * EB / 4; ++c) v[i][c] = 0u;
          }
      }
      if constexpr (T != kF32 && careful) take_odd<T>(v, hi, o + part * NV);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        f32x4_t& oj = o[part * NV + j];
        if constexpr (T == kF32) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            oj = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[i][j]), p[i], oj, 0, 0, 0);
        } else {
          v4u vt;  // row j of V^T: the lane's eight tokens
#pragma unroll
          for (int i = 0; i < 4; ++i)
            vt[i] = __builtin_amdgcn_perm(v[2 * i + 1][j >> 1], v[2 * i][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
          oj = E::mfma(vt, hi, oj);
          oj = E::mfma(vt, lo, oj);
        }
      }
      if (NP > 1 && part + 2 < NP) load_v(v, part + 2);
    }
  };

  // the same, head by head
  constexpr int NF = FEW > 0 ? FEW : 1;
  float ftop[NF], fsum[NF], fo[NF][FEW > 0 ? NC : 1];
#pragma unroll
  for (int h = 0; h < NF; ++h) {
    ftop[h] = -FLT_MAX;
    fsum[h] = 0.f;
#pragma unroll
    for (int j = 0; j < (FEW > 0 ? NC : 1); ++j) fo[h][j] = 0.f;
  }
  auto compute_few = [&](int tile, int& ids, int next) {
    Regs r;
    const int base = tile * kTile, first = base + 8 * g;
    float x[NF][2];
    load_k(r.k[0], 0);
    if constexpr (NP <= 2) load_k(r.k[1], 1);
    load_v(r.v[0], 0);
    if (next >= 0) ids = look(next);
    auto dot = [&](const v4u(&k)[KL], int s) {
#pragma unroll
      for (int h = 0; h < NF; ++h) {
        float c0 = 0.f, c1 = 0.f;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const v4u u = lq[(h * KL + i) * 4 + g];
          c0 = fmaf(__uint_as_float(k[i][0]), __uint_as_float(u[0]), c0);
          c1 = fmaf(__uint_as_float(k[i][1]), __uint_as_float(u[1]), c1);
          c0 = fmaf(__uint_as_float(k[i][2]), __uint_as_float(u[2]), c0);
          c1 = fmaf(__uint_as_float(k[i][3]), __uint_as_float(u[3]), c1);
        }
        c0 += c1;
        c0 += __shfl_xor(c0, 16, 64);
        c0 += __shfl_xor(c0, 32, 64);
        x[h][s] = base + 8 * (m16 >> 2) + 4 * s + (m16 & 3) < len ? c0 * scale : -INFINITY;
      }
    };
    dot(r.k[0], 0);
    if constexpr (NP > 2) {
      load_k(r.k[0], 1);
      dot(r.k[0], 1);
    } else {
      dot(r.k[1], 1);
    }
    if constexpr (NP > 1) load_v(r.v[1], 1);
    float p[NF][8];
#pragma unroll
    for (int h = 0; h < NF; ++h) {
      float most = fmaxf(x[h][0], x[h][1]);
      if (__any(most > ftop[h] + E::kSlack)) {
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) most = fmaxf(most, __shfl_xor(most, d, 64));
        const float now = fmaxf(ftop[h], most), c = __builtin_amdgcn_exp2f(ftop[h] - now);
        ftop[h] = now;
        fsum[h] *= c;
#pragma unroll
        for (int j = 0; j < (FEW > 0 ? NC : 1); ++j) fo[h][j] *= c;
      }
      const float p0 = __builtin_amdgcn_exp2f(x[h][0] - ftop[h]), p1 = __builtin_amdgcn_exp2f(x[h][1] - ftop[h]);
      fsum[h] += p0 + p1;
#pragma unroll
      for (int i = 0; i < 8; ++i) p[h][i] = __shfl(i < 4 ? p0 : p1, 4 * g + (i & 3), 64);
    }
#pragma unroll
    for (int part = 0; part < NP; ++part) {
      auto& v = r.v[part & (NP > 1 ? 1 : 0)];
      if (base + kTile > len) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (first + i >= len) {
#pragma unroll
            for (int c = 0; c < NV * EB / 4; ++c) v[i][c] = 0u;
          }
      }
#pragma unroll
      for (int h = 0; h < NF; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < NV; ++j)
            fo[h][part * NV + j] = fmaf(p[h][i], __uint_as_float(v[i][j]), fo[h][part * NV + j]);
      if (NP > 1 && part + 2 < NP) load_v(v, part + 2);
    }
  };

  const int t0 = sp * per + w;
  auto sweep = [&](auto flag) {
    int ids = a.split == 1 ? sound(t0 * kTile + (lane & 31) <= last ? early : 0) : look(t0);
    for (int t = t0; t < t_end; t += W) {
      point(t, ids);
      if constexpr (FEW > 0) compute_few(t, ids, t + W < t_end ? t + W : -1);
      else compute(t, ids, t + W < t_end ? t + W : -1, flag);
    }
  };
  if (t0 < t_end) {
    sweep(Flag<false>{});
    if constexpr (T != kF32) {
      // Once more, carefully, where a sum is not finite: rare, and a test of every value would
      // cost the others 4 % (64 x 12 heads of 64: 28.0 against 26.7 us).
      float z[4] = {0.f, 0.f, 0.f, 0.f};  // 0, or NaN
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = fmaf(o[j][r], 0.f, z[r]);
      const float odd = (z[0] + z[1]) + (z[2] + z[3]);
      if (__any(m16 < cols && odd != 0.f)) {
        top = -FLT_MAX, sum = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        sweep(Flag<true>{});
      }
    }
  }

  // the new row into its slot, by the workgroup that holds the last token
  if (kn && len > 0 && gt == 0 && len <= static_cast<int64_t>(a.width) * a.page && t_end == all && w == W - 1) {
    const int pg = a.by_page.of(last), pid = row[pg];
    if (pid >= 0 && pid < a.pages) {
      const int64_t off = last - pg * a.page;
      for (int c = lane; c < HD * EB / 16; c += 64) {
        reinterpret_cast<v4u*>(kc + pid * a.kc_page + off * a.kc_tok)[c] = reinterpret_cast<const v4u*>(kn)[c];
        reinterpret_cast<v4u*>(vc + pid * a.vc_page + off * a.vc_tok)[c] = reinterpret_cast<const v4u*>(vn)[c];
      }
    }
  }

  constexpr int kQ = FEW > 0 ? FEW * KL * 16 : NP > 1 ? KL * 256 : 0;  // (launch_one)
  float* const lw = lds + kQ;              // [W][cols][HD]
  float* const lo = lw + w * cols * HD;
  float* const lms = lw + W * cols * HD;   // [W][cols] maxima, then sums
  const bool any_bad = __any(bad);
  if constexpr (FEW > 0) {
#pragma unroll
    for (int h = 0; h < NF; ++h) {
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) fsum[h] += __shfl_xor(fsum[h], d, 64);
      if (h < cols && lane == 0) {
        lms[w * cols + h] = ftop[h];
        lms[(W + w) * cols + h] = any_bad ? NAN : fsum[h];
      }
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        float c = fo[h][j];
        c += __shfl_xor(c, 16, 64);
        c += __shfl_xor(c, 32, 64);
        if (h < cols && g == 0) lo[h * HD + v_col<T, HD>(m16, j)] = c;
      }
    }
  } else {
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (any_bad) sum = NAN;
    if (m16 < cols) {
      if (g == 0) {
        lms[w * cols + m16] = top;
        lms[(W + w) * cols + m16] = sum;
      }
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) lo[m16 * HD + v_col<T, HD>(4 * g + r, j)] = o[j][r];
    }
  }
  __syncthreads();
  for (int x = tid; x < cols * HD; x += W * 64) {
    const int c = x / HD, d = x - c * HD;
    float mm = lms[c];
#pragma unroll
    for (int i = 1; i < W; ++i) mm = fmaxf(mm, lms[i * cols + c]);
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float f = exp2f(lms[i * cols + c] - mm);
      num += f * lw[i * cols * HD + x];
      den += f * lms[(W + i) * cols + c];
    }
    const int64_t at = static_cast<int64_t>(n) * a.heads + h0 + c;
    if (a.split == 1) {
      static_cast<S*>(a.out)[at * HD + d] = E::store(den == 0.f ? 0.f : num / den);
    } else {
      float* part = a.part + (at * a.split + sp) * (HD + 2);
      part[d] = num;
      if (d == 0) part[HD] = mm, part[HD + 1] = den;
    }
  }
}

// the parts of a split sequence: 256 threads, 256 / dim of them to a column
template <DecodeType T>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(PagedAttnArgs a) {
  typedef Elem<T> E;
  __shared__ float s_w[256], s_num[256], s_top[4], s_den[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int at = blockIdx.x, n = a.by_heads.of(at);
  const int len = a.lens[n];
  const bool over = len > static_cast<int64_t>(a.width) * a.page;
  const int all = len > 0 && !over ? (len + kTile - 1) / kTile : 0;
  const int per = a.by_split.of(all + a.split - 1);
  int parts = 1;  // those that some workgroup wrote
  if (per > 0) parts = (all + per - 1) / per;
  const float* part = a.part + static_cast<int64_t>(at) * a.split * (a.dim + 2);
  float top = -FLT_MAX, den = 0.f;
  if (tid < parts) top = part[tid * (a.dim + 2) + a.dim], den = part[tid * (a.dim + 2) + a.dim + 1];
  float m = top;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if (lane == 0) s_top[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  const float f = exp2f(top - m);
  s_w[tid] = f;
  den *= f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o, 64);
  if (lane == 0) s_den[w] = den;
  __syncthreads();
  const int d = tid & (a.dim - 1), step = 256 / a.dim;
  float num = 0.f;
#pragma unroll 8
  for (int i = tid / a.dim; i < parts; i += step) num += s_w[i] * part[i * (a.dim + 2) + d];
  s_num[tid] = num;
  __syncthreads();
  if (tid < a.dim) {
    for (int i = 1; i < step; ++i) num += s_num[tid + i * a.dim];
    den = s_den[0] + s_den[1] + s_den[2] + s_den[3];
    static_cast<typename E::t*>(a.out)[static_cast<int64_t>(at) * a.dim + d] = E::store(den == 0.f ? 0.f : num / den);
  }
}

template <DecodeType T, int HD, int W, int FEW>
void launch_one(const PagedAttnArgs& a, hipStream_t stream) {
  const int group = a.heads / a.kv_heads, cols = group < 16 ? group : 16;
  typedef Tile<T, HD> Regs;
  const uint32_t lds = static_cast<uint32_t>(W * cols * (HD + 2) * 4 + (FEW > 0 ? FEW * Regs::KL * 64 : Regs::NP > 1 ? Regs::KL * 1024 : 0));
  if (lds > 65536)  // (of the current device: set wherever it is needed)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(paged_attn_kernel<T, HD, W, FEW>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
  const uint32_t blocks = static_cast<uint32_t>(a.n) * a.kv_heads * ((group + 15) / 16) * a.split;
  COMMEFF_LAUNCH((paged_attn_kernel<T, HD, W, FEW>), dim3(blocks), dim3(W * 64), lds, stream, a);
  if (a.split > 1)
    COMMEFF_LAUNCH(paged_attn_join_kernel<T>, dim3(static_cast<uint32_t>(a.n) * a.heads), dim3(256), 0, stream, a);
}

template <DecodeType T, int HD, int W>
void launch_group(const PagedAttnArgs& a, hipStream_t stream) {
  if constexpr (T == kF32) {
    if (a.group == 1) return launch_one<T, HD, W, 1>(a, stream);
    // (256 columns: the registers of two waves a SIMD leave 20 bytes a lane of one head in
    // scratch, more of a second one, and 124 to 128 of the MFMA form)
    if constexpr (HD <= 128) {
      if (a.group == 2) return launch_one<T, HD, W, 2>(a, stream);
    }
  }
  launch_one<T, HD, W, 0>(a, stream);
}

template <DecodeType T, int HD>
void launch_dim(const PagedAttnArgs& a, hipStream_t stream) {
  if constexpr (HD * Tile<T, HD>::E <= 256) {
    if (a.waves == 8) return launch_group<T, HD, 8>(a, stream);
  }
  if (a.waves == 1) return launch_group<T, HD, 1>(a, stream);
  launch_group<T, HD, 4>(a, stream);
}

template <DecodeType T>
void launch_type(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.dim == 32) launch_dim<T, 32>(a, stream);
  else if (a.dim == 64) launch_dim<T, 64>(a, stream);
  else if (a.dim == 128) launch_dim<T, 128>(a, stream);
  else launch_dim<T, 256>(a, stream);
}

}  // namespace

// Waves a workgroup and parts a sequence.  A workgroup serves one (sequence,
// cache head, 16 query heads), its waves take the sequence's tiles in turn: 8
// of them; 4 where sequences are short (64 x 12 heads of up to 256 tokens 10.7
// against 12.0 us) or rows fill the registers; 1 for one or two tiles, or for
// up to four where the batch fills the chip even so (250 x 12 heads, 32 tokens
// 7.3 against 12.4 us, 128 tokens 14.0 against 16.4; 64 x 12 heads, 128 tokens
// 9.7 against 7.6).  Where there are fewer than 1,024 workgroups, a sequence of
// 6 or more tiles a wave is split so that two are left: 1 x 12 heads, 4,096
// tokens 11.5 against 29.7 us, 8 x 8 heads, 65,536 tokens 245 against 776;
// below that the second launch costs more than it saves (16 x 12 heads, 1,024
// tokens 15.5 against 11.9).
void plan_paged_attention(PagedAttnArgs& a, DecodeType t, int64_t longest) {
  const int group = a.heads / a.kv_heads;
  const int64_t groups = static_cast<int64_t>(a.n) * a.kv_heads * ((group + 15) / 16);
  const int64_t tiles = (longest + kTile - 1) / kTile;
  a.waves = tiles <= 2 || (tiles <= 4 && groups >= 2048) ? 1 : tiles > 8 && a.dim * (t == kF32 ? 4 : 2) <= 256 ? 8 : 4;
  // (a launch has less than 2^32 threads; sequences x heads are at most 2^24)
  while (groups * a.waves * 64 >= 1ll << 32) a.waves = a.waves == 8 ? 4 : 1;
  int64_t split = 1;
  if (groups > 0 && tiles >= 6 * a.waves) split = (1024 + groups - 1) / groups;
  const int64_t most = tiles / (2 * a.waves);
  split = split > most ? most : split;
  a.split = static_cast<int>(split < 1 ? 1 : split > kMaxSplit ? kMaxSplit : split);
  a.group = group;
  a.by_heads = fast_div(a.heads);
  a.by_n = fast_div(a.n);
  a.by_kv = fast_div(a.kv_heads);
  a.by_tiles = fast_div((group + 15) / 16);
  a.by_split = fast_div(a.split);
  a.by_page = fast_div(a.page);
}

void launch_paged_attention(const PagedAttnArgs& a, DecodeType t, hipStream_t stream) {
  if (a.n == 0) return;
  if (t == kBf16) launch_type<kBf16>(a, stream);
  else if (t == kF16) launch_type<kF16>(a, stream);
  else launch_type<kF32>(a, stream);
}

}  // namespace commeff
