// torch.ops.commeff registrations of generation from a paged key-value cache
// (ops/decode.py): the argument checks that the CPU and HIP sides share, the
// CPU kernels (plain loops, sums in 64 bits) and the launches of kvcache.hip,
// paged_attention.hip and beam.hip.
#include <ATen/ATen.h>
#include <ATen/Dispatch.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>
#include <vector>

#include "decode.h"

namespace commeff {
namespace {

using OptTensor = c10::optional<at::Tensor>;

hipStream_t stream_now() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void same_device(const at::Tensor& t, const at::Tensor& ref, const char* op, const char* name) {
  TORCH_CHECK(t.device() == ref.device(), op, ": ", name, " is on ", t.device(), ", not on ", ref.device());
}

void check_i32(const at::Tensor& t, int64_t n, const at::Tensor& ref, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && (n < 0 || t.numel() == n), op,
              ": ", name, " must be contiguous int32 [", n < 0 ? std::string("any") : std::to_string(n), "], not ",
              t.scalar_type(), " ", t.sizes());
  same_device(t, ref, op, name);
}

void check_table(const at::Tensor& t, const char* op) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) &&
                  (t.size(0) <= 1 || t.stride(0) >= t.size(1)),
              op, ": table must be int32 [sequences, width] with unit column stride and rows of their own, not ",
              t.scalar_type(), " ", t.sizes(), " with strides ", t.strides());
}

void check_page(int64_t page, int64_t width, const char* op) {
  TORCH_CHECK(page >= 1 && page <= (1 << 20), op, ": a page holds 1 to 2^20 tokens, not ", page);
  TORCH_CHECK(width * page <= (1ll << 30), op, ": a table row covers at most 2^30 tokens, not ", width, " x ", page);
}

DecodeType decode_type(const at::Tensor& t, const char* op, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return kBf16;
    case at::kHalf: return kF16;
    case at::kFloat: return kF32;
    default: TORCH_CHECK(false, op, ": ", name, " must be bfloat16, float16 or float32, not ", t.scalar_type());
  }
}

void no_grad(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), op, ": ", name,
              " requires a gradient, and this operator has none: call it under torch.no_grad()");
}

// Whether every element has an address of its own (up to 6 dimensions): each dimension's
// steps are longer than all that the dimensions of shorter ones span.
bool own_addresses(const at::Tensor& t) {
  std::pair<int64_t, int64_t> dims[6];  // (stride, size), the shortest strides first
  int n = 0;
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) <= 1) continue;
    int at = n++;
    for (; at > 0 && dims[at - 1].first > t.stride(d); --at) dims[at] = dims[at - 1];
    dims[at] = {t.stride(d), t.size(d)};
  }
  int64_t span = 0;  // the furthest element so far
  for (int i = 0; i < n; ++i) {
    if (dims[i].first <= span) return false;
    span += dims[i].first * (dims[i].second - 1);
  }
  return true;
}

// [pages, kv heads, page, dim], any strides but a unit one over dim; a cache that is
// written has an address for every element
void check_cache(const at::Tensor& c, bool written, const char* op, const char* name) {
  TORCH_CHECK(c.dim() == 4 && c.size(1) >= 1 && c.size(2) >= 1 && c.size(3) >= 1, op, ": ", name,
              " must be [pages, kv heads, page size, head dim], not ", c.sizes());
  TORCH_CHECK(c.size(3) == 1 || c.stride(3) == 1, op, ": ", name, " needs a unit stride over the head's columns");
  for (int d = 0; d < 3; ++d)
    TORCH_CHECK(c.size(d) <= 1 || c.numel() == 0 || c.stride(d) > 0, op, ": ", name, " is an expanded view");
  TORCH_CHECK(!written || c.numel() == 0 || own_addresses(c), op, ": ", name, " overlaps itself: strides ", c.strides(),
              " of ", c.sizes());
}

void check_pair(const at::Tensor& kc, const at::Tensor& vc, bool written, const char* op) {
  check_cache(kc, written, op, "the key cache");
  check_cache(vc, written, op, "the value cache");
  TORCH_CHECK(kc.sizes() == vc.sizes() && kc.scalar_type() == vc.scalar_type(), op,
              ": key and value cache differ: ", kc.scalar_type(), " ", kc.sizes(), " and ", vc.scalar_type(), " ",
              vc.sizes());
  same_device(vc, kc, op, "the value cache");
}

// [rows, kv heads, dim] beside a cache
void check_rows(const at::Tensor& x, int64_t rows, const at::Tensor& cache, const char* op, const char* name) {
  TORCH_CHECK(x.dim() == 3 && (rows < 0 || x.size(0) == rows) && x.size(1) == cache.size(1) &&
                  x.size(2) == cache.size(3) && x.scalar_type() == cache.scalar_type(),
              op, ": ", name, " must be [rows, ", cache.size(1), ", ", cache.size(3), "] in the cache's type, not ",
              x.scalar_type(), " ", x.sizes());
  same_device(x, cache, op, name);
  no_grad(x, op, name);
}

bool aligned16(const at::Tensor& t, int dims) {
  const int64_t e = t.element_size();
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int d = 0; d < dims; ++d)
    if (t.size(d) > 1 && t.stride(d) * e % 16 != 0) return false;
  return true;
}

// rows whose head columns are contiguous (a copy where they are not)
at::Tensor unit_rows(const at::Tensor& x) {
  return x.size(2) == 1 || x.stride(2) == 1 ? x : x.contiguous();
}

// contiguous `size` elements of `buf` from `at` on: a narrow() without the
// dispatcher, which would be half of such a call's host time
at::Tensor piece_of(const at::Tensor& buf, int64_t at, at::IntArrayRef size) {
  auto t = c10::make_intrusive<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), buf.dtype());
  t->set_storage_offset(at);
  t->set_sizes_contiguous(size);
  return at::Tensor(std::move(t));
}

// ------------------------------------------------------------------ extend
std::vector<at::Tensor> extend_outputs(at::Tensor& table, at::Tensor& lens, const at::Tensor& fresh,
                                       const at::Tensor& pool, at::Tensor& used, int64_t page, int64_t rows,
                                       bool in_place) {
  const char* op = "kv_extend";
  check_table(table, op);
  const int64_t n = table.size(0);
  check_page(page, table.size(1), op);
  check_i32(lens, n, table, op, "lens");
  check_i32(fresh, n, table, op, "new");
  check_i32(pool, -1, table, op, "pool");
  check_i32(used, 1, table, op, "used");
  TORCH_CHECK(rows >= 0 && rows <= (1ll << 30), op, ": rows must be in [0, 2^30], not ", rows);
  TORCH_CHECK(n <= (1ll << 30) && pool.numel() <= (1ll << 30), op, ": at most 2^30 sequences and pages");
  auto i32 = lens.options();
  // slots [rows] | one allocation: pos [rows], seq [rows], start [n + 1], missed (, lens [n], used)
  const int64_t all = 2 * (rows + 3) + n + 1 + 3 + 4 + (in_place ? 0 : n + 3 + 4);
  const auto buf = at::empty({all}, i32);
  int64_t at = 0;
  auto piece = [&](int64_t size) {
    auto t = piece_of(buf, at, {size});
    at += (size + 3) / 4 * 4;  // (each at a multiple of 16 bytes)
    return t;
  };
  std::vector<at::Tensor> out;
  out.reserve(7);
  out.push_back(at::empty({rows}, i32.dtype(at::kLong)));
  for (int64_t size : {rows, rows, n + 1, static_cast<int64_t>(1)}) out.push_back(piece(size));
  if (!in_place) {
    out.push_back(piece(n));
    out.push_back(piece(1));
  }
  return out;
}

std::vector<at::Tensor> kv_extend_hip(at::Tensor table, at::Tensor lens, const at::Tensor& fresh,
                                      const at::Tensor& pool, at::Tensor used, int64_t page, int64_t rows,
                                      bool in_place) {
  c10::hip::HIPGuardMasqueradingAsCUDA guard(table.device());
  auto out = extend_outputs(table, lens, fresh, pool, used, page, rows, in_place);
  const int64_t n = table.size(0);
  at::Tensor work;
  KvExtendArgs a;
  a.table = table.data_ptr<int32_t>();
  a.table_ld = table.stride(0);
  a.lens = lens.data_ptr<int32_t>();
  a.fresh = fresh.data_ptr<int32_t>();
  a.pool = pool.data_ptr<int32_t>();
  a.used = used.data_ptr<int32_t>();
  a.slots = out[0].data_ptr<int64_t>();
  a.pos = out[1].data_ptr<int32_t>();
  a.seq = out[2].data_ptr<int32_t>();
  a.start = out[3].data_ptr<int32_t>();
  a.missed = out[4].data_ptr<int32_t>();
  a.lens_out = (in_place ? lens : out[5]).data_ptr<int32_t>();
  a.used_out = (in_place ? used : out[6]).data_ptr<int32_t>();
  a.base = a.first = nullptr;
  a.n = static_cast<int>(n);
  a.width = static_cast<int>(table.size(1));
  a.page = static_cast<int>(page);
  a.rows = static_cast<int>(rows);
  a.pool_n = static_cast<int>(pool.numel());
  if (!kv_extend_fused(a)) {
    work = at::empty({2 * n}, lens.options());
    a.base = work.data_ptr<int32_t>();
    a.first = a.base + n;
  }
  launch_kv_extend(a, stream_now());
  return out;
}

std::vector<at::Tensor> kv_extend_cpu(at::Tensor table, at::Tensor lens, const at::Tensor& fresh,
                                      const at::Tensor& pool, at::Tensor used, int64_t page, int64_t rows,
                                      bool in_place) {
  auto out = extend_outputs(table, lens, fresh, pool, used, page, rows, in_place);
  const int64_t n = table.size(0), width = table.size(1), taken = used.data_ptr<int32_t>()[0];
  const int64_t avail = taken < 0 ? 0 : std::max<int64_t>(0, pool.numel() - taken);
  int64_t* slots = out[0].data_ptr<int64_t>();
  int32_t *pos = out[1].data_ptr<int32_t>(), *seq = out[2].data_ptr<int32_t>(), *start = out[3].data_ptr<int32_t>();
  std::fill(slots, slots + rows, -1);
  std::fill(pos, pos + rows, 0);
  std::fill(seq, seq + rows, -1);
  int64_t row = 0, upto = 0, got = 0, missed = 0;
  auto pages_of = [page](int64_t x) { return (x + page - 1) / page; };
  for (int64_t i = 0; i < n; ++i) {
    const int64_t len = lens.data_ptr<int32_t>()[i], more = fresh.data_ptr<int32_t>()[i];
    const int64_t add = std::max<int64_t>(0, more), end = row + add;
    start[i] = static_cast<int32_t>(std::min(row, rows));
    const bool fits = more >= 0 && len >= 0 && end <= rows && len + more <= width * page;
    const int64_t need = fits ? pages_of(len + more) - pages_of(len) : 0;
    const int64_t first = taken + upto;
    upto += need;
    const bool served = fits && (need == 0 || upto <= avail);
    int32_t* ids = table.data_ptr<int32_t>() + i * table.stride(0);
    if (served) {
      for (int64_t c = 0; c < need; ++c) ids[pages_of(len) + c] = pool.data_ptr<int32_t>()[first + c];
      got += need;
    } else {
      ++missed;
    }
    for (int64_t r = row; r < std::min(end, rows); ++r) {
      seq[r] = static_cast<int32_t>(i);
      if (!served) continue;
      const int64_t p = len + r - row;
      pos[r] = static_cast<int32_t>(p);
      if (ids[p / page] >= 0) slots[r] = static_cast<int64_t>(ids[p / page]) * page + p % page;
    }
    (in_place ? lens : out[5]).data_ptr<int32_t>()[i] = static_cast<int32_t>(served ? len + more : len);
    row = end;
  }
  start[n] = static_cast<int32_t>(std::min(row, rows));
  (in_place ? used : out[6]).data_ptr<int32_t>()[0] = static_cast<int32_t>(taken + got);
  out[4].data_ptr<int32_t>()[0] = static_cast<int32_t>(missed);
  return out;
}

// ------------------------------------------------------------------- write
void check_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& kc, const at::Tensor& vc,
                 const at::Tensor& slots) {
  const char* op = "kv_write";
  decode_type(kc, op, "the key cache");
  check_pair(kc, vc, true, op);
  check_page(kc.size(2), 0, op);
  TORCH_CHECK(kc.size(0) * kc.size(2) < (1ll << 31), op, ": the caches must hold less than 2^31 slots, not ",
              kc.size(0), " pages of ", kc.size(2));
  TORCH_CHECK(kc.numel() == 0 || kc.data_ptr() != vc.data_ptr(), op, ": key and value cache are the same");
  check_rows(k, -1, kc, op, "k");
  TORCH_CHECK(k.size(0) < (1ll << 31) && k.size(1) * k.size(2) <= (1ll << 24), op, ": rows too many or too long: ",
              k.sizes());
  check_rows(v, k.size(0), vc, op, "v");
  TORCH_CHECK(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous() &&
                  slots.numel() == k.size(0),
              op, ": slots must be contiguous int64 [", k.size(0), "], not ", slots.scalar_type(), " ", slots.sizes());
  same_device(slots, kc, op, "slots");
}

void kv_write_hip(const at::Tensor& k_, const at::Tensor& v_, at::Tensor kc, at::Tensor vc, const at::Tensor& slots) {
  c10::hip::HIPGuardMasqueradingAsCUDA guard(kc.device());
  check_write(k_, v_, kc, vc, slots);
  const auto k = unit_rows(k_), v = unit_rows(v_);
  const int64_t e = kc.element_size();
  KvWriteArgs a;
  a.k = static_cast<const unsigned char*>(k.data_ptr());
  a.v = static_cast<const unsigned char*>(v.data_ptr());
  a.kc = static_cast<unsigned char*>(kc.data_ptr());
  a.vc = static_cast<unsigned char*>(vc.data_ptr());
  a.slots = slots.data_ptr<int64_t>();
  a.k_row = k.stride(0) * e, a.k_head = k.stride(1) * e;
  a.v_row = v.stride(0) * e, a.v_head = v.stride(1) * e;
  a.kc_page = kc.stride(0) * e, a.kc_head = kc.stride(1) * e, a.kc_tok = kc.stride(2) * e;
  a.vc_page = vc.stride(0) * e, a.vc_head = vc.stride(1) * e, a.vc_tok = vc.stride(2) * e;
  a.rows = k.size(0);
  a.pages = kc.size(0);
  a.heads = static_cast<int>(kc.size(1));
  a.page = static_cast<int>(kc.size(2));
  a.row_bytes = static_cast<int>(kc.size(3) * e);
  a.unit = a.row_bytes % 16 == 0 && aligned16(k, 2) && aligned16(v, 2) && aligned16(kc, 3) && aligned16(vc, 3)
               ? 16
               : static_cast<int>(e);
  launch_kv_write(a, stream_now());
}

void kv_write_cpu(const at::Tensor& k, const at::Tensor& v, at::Tensor kc, at::Tensor vc, const at::Tensor& slots) {
  check_write(k, v, kc, vc, slots);
  const int64_t page = kc.size(2);
  for (int64_t r = 0; r < slots.numel(); ++r) {
    const int64_t s = slots.data_ptr<int64_t>()[r];
    if (s < 0 || s >= kc.size(0) * page) continue;
    kc.select(0, s / page).select(1, s % page).copy_(k.select(0, r));
    vc.select(0, s / page).select(1, s % page).copy_(v.select(0, r));
  }
}

// ----------------------------------------------------------------- reorder
void check_reorder(const at::Tensor& parent, const at::Tensor& table, const at::Tensor& lens, const at::Tensor& kv) {
  const char* op = "beam_reorder";
  check_table(table, op);
  TORCH_CHECK(parent.scalar_type() == at::kLong && parent.dim() == 2 && parent.is_contiguous() &&
                  parent.numel() == table.size(0),
              op, ": parent must be contiguous int64 [requests, beams] over the table's ", table.size(0),
              " sequences, not ", parent.scalar_type(), " ", parent.sizes());
  TORCH_CHECK(parent.size(0) <= 65535, op, ": at most 65,535 requests, not ", parent.size(0));
  TORCH_CHECK(parent.size(1) <= kReorderMaxBeams, op, ": at most ", kReorderMaxBeams, " beams, not ", parent.size(1));
  same_device(parent, table, op, "parent");
  check_i32(lens, table.size(0), table, op, "lens");
  decode_type(kv, op, "kv");
  TORCH_CHECK(kv.dim() == 6 && kv.size(1) == 2 && kv.size(3) >= 1 && kv.size(4) >= 1 && kv.size(5) >= 1 &&
                  (kv.size(5) == 1 || kv.stride(5) == 1),
              op, ": kv must be [layers, 2, pages, kv heads, page size, head dim] with a unit column stride, not ",
              kv.sizes());
  for (int d = 0; d < 5; ++d)
    TORCH_CHECK(kv.size(d) <= 1 || kv.stride(d) > 0, op, ": kv is an expanded view");
  TORCH_CHECK(kv.numel() == 0 || own_addresses(kv), op, ": kv overlaps itself: strides ", kv.strides(), " of ",
              kv.sizes());
  same_device(kv, table, op, "kv");
  check_page(kv.size(4), table.size(1), op);
  TORCH_CHECK(2 * kv.size(0) * kv.size(3) * kv.size(4) * kv.size(5) < (1ll << 31), op,
              ": a page of all layers holds less than 2^31 numbers, not ", kv.sizes());
}

void beam_reorder_hip(const at::Tensor& parent, at::Tensor table, const at::Tensor& lens, at::Tensor kv) {
  c10::hip::HIPGuardMasqueradingAsCUDA guard(table.device());
  check_reorder(parent, table, lens, kv);
  const int64_t e = kv.element_size();
  BeamReorderArgs a;
  a.parent = parent.data_ptr<int64_t>();
  a.table = table.data_ptr<int32_t>();
  a.table_ld = table.stride(0);
  a.lens = lens.data_ptr<int32_t>();
  a.kv = static_cast<unsigned char*>(kv.data_ptr());
  a.s_layer = kv.stride(0) * e, a.s_kv = kv.stride(1) * e, a.s_page = kv.stride(2) * e;
  a.s_head = kv.stride(3) * e, a.s_tok = kv.stride(4) * e;
  a.pages = kv.size(2);
  a.requests = static_cast<int>(parent.size(0));
  a.beams = static_cast<int>(parent.size(1));
  a.width = static_cast<int>(table.size(1));
  a.layers = static_cast<int>(kv.size(0));
  a.heads = static_cast<int>(kv.size(3));
  a.page = static_cast<int>(kv.size(4));
  a.row_bytes = static_cast<int>(kv.size(5) * e);
  a.unit = a.row_bytes % 16 == 0 && aligned16(kv, 5) ? 16 : static_cast<int>(e);
  launch_beam_reorder(a, stream_now());
}

void beam_reorder_cpu(const at::Tensor& parent, at::Tensor table, const at::Tensor& lens, at::Tensor kv) {
  check_reorder(parent, table, lens, kv);
  const int64_t B = parent.size(0), J = parent.size(1), page = kv.size(4), pages = kv.size(2), width = table.size(1);
  const int32_t* len = lens.data_ptr<int32_t>();
  for (int64_t b = 0; b < B; ++b) {
    const auto old = table.narrow(0, b * J, J).clone();
    std::vector<at::Tensor> part(J);
    for (int pass = 0; pass < 2; ++pass) {
      for (int64_t j = 0; j < J; ++j) {
        const int64_t p = parent.data_ptr<int64_t>()[b * J + j], n = b * J + j;
        if (p < 0 || p >= J || p == j) continue;
        const int64_t ln = len[n], full = ln / page, rest = ln % page;
        if (ln <= 0 || ln != len[b * J + p] || full + (rest != 0) > width) continue;
        const int32_t* mine = old.data_ptr<int32_t>() + j * width;
        const int32_t* from = old.data_ptr<int32_t>() + p * width;
        if (rest && (mine[full] < 0 || mine[full] >= pages || from[full] < 0 || from[full] >= pages)) continue;
        if (pass == 0) {
          if (rest) part[j] = kv.select(2, from[full]).narrow(3, 0, rest).clone();
        } else {
          if (rest) kv.select(2, mine[full]).narrow(3, 0, rest).copy_(part[j]);
          std::copy(from, from + full, table.data_ptr<int32_t>() + n * table.stride(0));
        }
      }
    }
  }
}

// --------------------------------------------------------------- attention
void check_attention(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& table,
                     const at::Tensor& lens, const OptTensor& k, const OptTensor& v) {
  const char* op = "paged_attention";
  decode_type(kc, op, "the key cache");
  check_pair(kc, vc, given(k), op);
  const int64_t hd = kc.size(3);
  TORCH_CHECK(hd == 32 || hd == 64 || hd == 128 || hd == 256, op, ": head dim 32, 64, 128 or 256, not ", hd);
  TORCH_CHECK(q.dim() == 3 && q.scalar_type() == kc.scalar_type() && q.size(2) == hd && q.size(1) >= 1 &&
                  q.size(1) % kc.size(1) == 0,
              op, ": q must be [sequences, heads, ", hd, "] in the cache's type, its heads a multiple of the cache's ",
              kc.size(1), ", not ", q.scalar_type(), " ", q.sizes());
  same_device(q, kc, op, "q");
  no_grad(q, op, "q");
  check_table(table, op);
  TORCH_CHECK(table.size(0) == q.size(0), op, ": table has ", table.size(0), " rows for ", q.size(0), " sequences");
  same_device(table, kc, op, "table");
  check_i32(lens, q.size(0), kc, op, "lens");
  check_page(kc.size(2), table.size(1), op);
  TORCH_CHECK(kc.size(0) >= 1 && kc.size(0) * kc.size(2) < (1ll << 31), op,
              ": the caches must hold 1 to 2^31 - 1 slots, not ", kc.size(0), " pages of ", kc.size(2));
  TORCH_CHECK(q.size(0) * q.size(1) <= (1ll << 24), op, ": at most 2^24 sequences x heads");
  TORCH_CHECK(given(k) == given(v), op, ": k and v come together");
  if (given(k)) {
    TORCH_CHECK(kc.data_ptr() != vc.data_ptr(), op, ": key and value cache are the same");
    check_rows(*k, q.size(0), kc, op, "k");
    check_rows(*v, q.size(0), vc, op, "v");
  }
}

at::Tensor paged_attention_hip(const at::Tensor& q_, at::Tensor kc, at::Tensor vc, const at::Tensor& table,
                               const at::Tensor& lens, const OptTensor& k, const OptTensor& v,
                               c10::optional<double> scale, c10::optional<int64_t> longest) {
  c10::hip::HIPGuardMasqueradingAsCUDA guard(kc.device());
  check_attention(q_, kc, vc, table, lens, k, v);
  TORCH_CHECK(aligned16(kc, 3) && aligned16(vc, 3),
              "paged_attention: the caches' pages, heads and slots must start at multiples of 16 bytes");
  auto rows16 = [](const at::Tensor& t) {
    const auto u = unit_rows(t);
    return aligned16(u, 2) ? u : u.clone(at::MemoryFormat::Contiguous);
  };
  const auto q = rows16(q_);
  PagedAttnArgs a;
  at::Tensor kn, vn;
  a.k = a.v = nullptr;
  a.k_row = a.k_head = a.v_row = a.v_head = 0;
  if (given(k)) {
    kn = rows16(*k), vn = rows16(*v);
    a.k = kn.data_ptr(), a.v = vn.data_ptr();
    a.k_row = kn.stride(0), a.k_head = kn.stride(1);
    a.v_row = vn.stride(0), a.v_head = vn.stride(1);
  }
  auto out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  a.q = q.data_ptr();
  a.q_row = q.stride(0), a.q_head = q.stride(1);
  a.kc = kc.data_ptr(), a.vc = vc.data_ptr();
  a.kc_page = kc.stride(0), a.kc_head = kc.stride(1), a.kc_tok = kc.stride(2);
  a.vc_page = vc.stride(0), a.vc_head = vc.stride(1), a.vc_tok = vc.stride(2);
  a.table = table.data_ptr<int32_t>();
  a.table_ld = table.stride(0);
  a.lens = lens.data_ptr<int32_t>();
  a.out = out.data_ptr();
  a.n = static_cast<int>(q.size(0));
  a.heads = static_cast<int>(q.size(1));
  a.kv_heads = static_cast<int>(kc.size(1));
  a.dim = static_cast<int>(q.size(2));
  a.width = static_cast<int>(table.size(1));
  a.page = static_cast<int>(kc.size(2));
  a.pages = kc.size(0);
  a.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(a.dim)));
  const int64_t most = std::min<int64_t>(longest.has_value() ? std::max<int64_t>(1, *longest) : (1ll << 30),
                                         static_cast<int64_t>(a.width) * a.page);
  const DecodeType type = decode_type(kc, "paged_attention", "the key cache");
  plan_paged_attention(a, type, most);
  a.part = nullptr;
  at::Tensor part;
  if (a.split > 1) {
    part = at::empty({static_cast<int64_t>(a.n) * a.heads * a.split * (a.dim + 2)}, q.options().dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  launch_paged_attention(a, type, stream_now());
  return out;
}

template <typename S>
void paged_attention_loops(const at::Tensor& q, at::Tensor& kc, at::Tensor& vc, const at::Tensor& table,
                           const at::Tensor& lens, const at::Tensor* k, const at::Tensor* v, double scale,
                           at::Tensor& out) {
  const int64_t n = q.size(0), heads = q.size(1), hd = q.size(2), kh = kc.size(1), page = kc.size(2);
  const auto qa = q.accessor<S, 3>();
  auto ka = kc.accessor<S, 4>(), va = vc.accessor<S, 4>();
  auto oa = out.accessor<S, 3>();
  const auto ta = table.accessor<int32_t, 2>();
  for (int64_t i = 0; i < n; ++i) {
    const int64_t len = lens.data_ptr<int32_t>()[i];
    if (len <= 0) {
      out.select(0, i).zero_();
      continue;
    }
    bool bad = len > table.size(1) * page;
    for (int64_t c = 0; !bad && c < (len + page - 1) / page; ++c) bad = ta[i][c] < 0 || ta[i][c] >= kc.size(0);
    const int64_t last = len - 1;
    if (k && !(len > table.size(1) * page) && ta[i][last / page] >= 0 && ta[i][last / page] < kc.size(0)) {
      kc.select(0, ta[i][last / page]).select(1, last % page).copy_(k->select(0, i));
      vc.select(0, ta[i][last / page]).select(1, last % page).copy_(v->select(0, i));
    }
    if (bad) {
      out.select(0, i).fill_(std::numeric_limits<float>::quiet_NaN());
      continue;
    }
    std::vector<double> p(len), o(hd);
    for (int64_t h = 0; h < heads; ++h) {
      const int64_t g = h / (heads / kh);
      double m = -std::numeric_limits<double>::infinity(), l = 0;
      for (int64_t t = 0; t < len; ++t) {
        double x = 0;
        for (int64_t d = 0; d < hd; ++d)
          x += static_cast<double>(static_cast<float>(qa[i][h][d])) *
               static_cast<float>(ka[ta[i][t / page]][g][t % page][d]);
        p[t] = x * scale;
        m = std::max(m, p[t]);
      }
      std::fill(o.begin(), o.end(), 0.0);
      for (int64_t t = 0; t < len; ++t) {
        const double w = std::exp(p[t] - (m > -std::numeric_limits<double>::infinity() ? m : 0.0));
        l += w;
        for (int64_t d = 0; d < hd; ++d) o[d] += w * static_cast<float>(va[ta[i][t / page]][g][t % page][d]);
      }
      for (int64_t d = 0; d < hd; ++d) oa[i][h][d] = static_cast<S>(static_cast<float>(l == 0 ? 0.0 : o[d] / l));
    }
  }
}

at::Tensor paged_attention_cpu(const at::Tensor& q, at::Tensor kc, at::Tensor vc, const at::Tensor& table,
                               const at::Tensor& lens, const OptTensor& k, const OptTensor& v,
                               c10::optional<double> scale, c10::optional<int64_t> /*longest*/) {
  check_attention(q, kc, vc, table, lens, k, v);
  auto out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(2)));
  AT_DISPATCH_FLOATING_TYPES_AND2(at::kBFloat16, at::kHalf, q.scalar_type(), "paged_attention", [&] {
    paged_attention_loops<scalar_t>(q, kc, vc, table, lens, given(k) ? &*k : nullptr, given(v) ? &*v : nullptr, s,
                                    out);
  });
  return out;
}

// ------------------------------------------------------------------ select
void check_select(const at::Tensor& logits, const at::Tensor& scores, int64_t keep, const OptTensor& finished,
                  int64_t eos) {
  const char* op = "beam_select";
  decode_type(logits, op, "logits");
  TORCH_CHECK(logits.dim() == 3 && logits.size(1) >= 1 && logits.size(2) >= 1, op,
              ": logits must be [requests, beams, vocabulary], not ", logits.sizes());
  TORCH_CHECK(logits.size(1) * logits.size(2) <= (1ll << 31) - (1 << 16), op,
              ": beams x vocabulary must be at most 2^31 - 2^16, not ", logits.size(1), " x ", logits.size(2));
  TORCH_CHECK(logits.size(1) <= kBeamMaxBeams && logits.size(0) * logits.size(1) <= 65535, op,
              ": at most 1,024 beams and 65,535 rows, not ", logits.size(0), " x ", logits.size(1));
  no_grad(logits, op, "logits");
  TORCH_CHECK(scores.scalar_type() == at::kFloat && scores.dim() == 2 && scores.is_contiguous() &&
                  scores.size(0) == logits.size(0) && scores.size(1) == logits.size(1),
              op, ": scores must be contiguous float32 [", logits.size(0), ", ", logits.size(1), "], not ",
              scores.scalar_type(), " ", scores.sizes());
  same_device(scores, logits, op, "scores");
  TORCH_CHECK(keep >= 1 && keep <= kBeamMaxKeep, op, ": keep must be in [1, ", kBeamMaxKeep, "], not ", keep);
  if (given(finished)) {
    TORCH_CHECK(finished->scalar_type() == at::kBool && finished->is_contiguous() &&
                    finished->sizes() == scores.sizes(),
                op, ": finished must be contiguous bool ", scores.sizes(), ", not ", finished->scalar_type(), " ",
                finished->sizes());
    same_device(*finished, logits, op, "finished");
    TORCH_CHECK(eos >= 0 && eos < logits.size(2), op, ": finished beams need eos in [0, ", logits.size(2), "), not ",
                eos);
  }
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> select_outputs(const at::Tensor& scores, int64_t keep) {
  const int64_t b = scores.size(0);
  const auto ids = at::empty({2 * b * keep}, scores.options().dtype(at::kLong));
  return {at::empty({b, keep}, scores.options()), piece_of(ids, 0, {b, keep}), piece_of(ids, b * keep, {b, keep})};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> beam_select_hip(const at::Tensor& logits, const at::Tensor& scores,
                                                               int64_t keep, const OptTensor& finished, int64_t eos) {
  c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
  check_select(logits, scores, keep, finished, eos);
  const auto x = logits.size(2) == 1 || logits.stride(2) == 1 ? logits : logits.contiguous();
  auto out = select_outputs(scores, keep);
  BeamSelectArgs a;
  a.logits = x.data_ptr();
  a.scores = scores.data_ptr<float>();
  a.finished = given(finished) ? reinterpret_cast<const uint8_t*>(finished->data_ptr<bool>()) : nullptr;
  a.out_scores = std::get<0>(out).data_ptr<float>();
  a.out_parent = std::get<1>(out).data_ptr<int64_t>();
  a.out_token = std::get<2>(out).data_ptr<int64_t>();
  a.s_request = x.stride(0), a.s_beam = x.stride(1);
  a.eos = eos;
  a.requests = static_cast<int>(x.size(0));
  a.beams = static_cast<int>(x.size(1));
  a.vocab = static_cast<int>(x.size(2));
  a.keep = static_cast<int>(keep);
  const DecodeType type = decode_type(x, "beam_select", "logits");
  a.parts = beam_select_parts(a.vocab, type);
  const int64_t lists = scores.numel() * a.parts;
  TORCH_CHECK(x.size(1) * a.parts * keep < (1ll << 31), "beam_select: too many beams for this vocabulary");
  auto work = at::empty({lists * (keep + 2 * kBeamWaves)}, scores.options().dtype(at::kLong));
  a.cand = reinterpret_cast<unsigned long long*>(work.data_ptr<int64_t>());
  a.stat = reinterpret_cast<double*>(a.cand + lists * keep);
  launch_beam_select(a, type, stream_now());
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> beam_select_cpu(const at::Tensor& logits, const at::Tensor& scores,
                                                               int64_t keep, const OptTensor& finished, int64_t eos) {
  check_select(logits, scores, keep, finished, eos);
  auto out = select_outputs(scores, keep);
  const int64_t B = logits.size(0), J = logits.size(1), V = logits.size(2);
  const double inf = std::numeric_limits<double>::infinity();
  for (int64_t b = 0; b < B; ++b) {
    std::vector<std::pair<double, int64_t>> c;  // (-score, flat index): the smallest first
    for (int64_t j = 0; j < J; ++j) {
      const double s = scores.data_ptr<float>()[b * J + j];
      if (!std::isfinite(s)) continue;
      if (given(finished) && finished->data_ptr<bool>()[b * J + j]) {
        c.emplace_back(-s, j * V + eos);
        continue;
      }
      const auto row = logits.select(0, b).select(0, j).to(at::kDouble).contiguous();
      const double* x = row.data_ptr<double>();
      double m = -inf, sum = 0;
      bool odd = false;
      for (int64_t v = 0; v < V; ++v) {
        odd = odd || std::isnan(x[v]) || x[v] == inf;
        m = std::max(m, x[v]);
      }
      if (odd || m == -inf) continue;
      for (int64_t v = 0; v < V; ++v) sum += std::exp(x[v] - m);
      const double lse = m + std::log(sum);
      for (int64_t v = 0; v < V; ++v)
        if (x[v] > -inf) c.emplace_back(-(s + (x[v] - lse)), j * V + v);
    }
    const int64_t some = std::min<int64_t>(keep, c.size());
    std::partial_sort(c.begin(), c.begin() + some, c.end());
    for (int64_t i = 0; i < keep; ++i) {
      std::get<0>(out).data_ptr<float>()[b * keep + i] = static_cast<float>(i < some ? -c[i].first : -inf);
      std::get<1>(out).data_ptr<int64_t>()[b * keep + i] = i < some ? c[i].second / V : 0;
      std::get<2>(out).data_ptr<int64_t>()[b * keep + i] = i < some ? c[i].second % V : 0;
    }
  }
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(commeff, m) {
  m.def("kv_extend(Tensor(a!) table, Tensor(b!) lens, Tensor fresh, Tensor pool, Tensor(c!) used, int page, "
        "int rows, bool in_place) -> Tensor[]");
  m.def("kv_write(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots) -> ()");
  m.def("beam_reorder(Tensor parent, Tensor(a!) table, Tensor lens, Tensor(b!) kv) -> ()");
  m.def("paged_attention(Tensor q, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor table, Tensor lens, Tensor? k, "
        "Tensor? v, float? scale, int? longest) -> Tensor");
  m.def("beam_select(Tensor logits, Tensor scores, int keep, Tensor? finished, int eos) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(commeff, CPU, m) {
  m.impl("kv_extend", &kv_extend_cpu);
  m.impl("kv_write", &kv_write_cpu);
  m.impl("beam_reorder", &beam_reorder_cpu);
  m.impl("paged_attention", &paged_attention_cpu);
  m.impl("beam_select", &beam_select_cpu);
}

TORCH_LIBRARY_IMPL(commeff, CUDA, m) {
  m.impl("kv_extend", &kv_extend_hip);
  m.impl("kv_write", &kv_write_hip);
  m.impl("beam_reorder", &beam_reorder_hip);
  m.impl("paged_attention", &paged_attention_hip);
  m.impl("beam_select", &beam_select_hip);
}

}  // namespace commeff
