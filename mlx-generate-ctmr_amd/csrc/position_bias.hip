// The plan of places that a position bias reads, and the checks of its descriptor.
#include "position_bias.hpp"

#include <algorithm>

namespace ctmr {
namespace attn {

int bias_steps(const ctmr_buckets_desc* b) {
  int columns = 0;
  for (int a = 0; a < b->axes; ++a) columns += b->extents[a];
  return columns <= 48 ? 3 : columns <= 64 ? 4 : columns <= 96 ? 6 : 8;
}

namespace {

int check_plan(const ctmr_buckets_desc* b) {
  if (!b) return fail(CTMR_E_INVALID, "null descriptor");
  if (b->query_items <= 0 || b->key_items <= 0 || b->lq <= 0 || b->lk <= 0)
    return fail(CTMR_E_INVALID, "non-positive dimension");
  if (b->axes < 1 || b->axes > 4) return fail(CTMR_E_INVALID, "places have one to four axes");
  int columns = 0;
  for (int a = 0; a < b->axes; ++a) {
    if (b->extents[a] < 1 || b->extents[a] > kColumns) return fail(CTMR_E_INVALID, "extents must be 1 to 128");
    columns += b->extents[a];
  }
  if (columns > kColumns) return fail(CTMR_E_UNSUPPORTED, "extents must add up to 128 at most");
  if (b->table_rows < 1 || b->table_rows > (1 << 16)) return fail(CTMR_E_INVALID, "the table has 1 to 65536 rows");
  if ((int64_t)b->query_items * b->lq > (1ll << 28) || (int64_t)b->key_items * b->lk > (1ll << 28))
    return fail(CTMR_E_UNSUPPORTED, "too many rows");
  return CTMR_OK;
}

struct Parts {
  int64_t rows, query_columns, key_columns, query_places, key_places, query_hot, key_hot, bytes;
};

// Where a plan's parts start.  One-hot rows of equal sides are the same.
Parts parts_of(const ctmr_buckets_desc* b) {
  Parts p = {};
  const int64_t width = bias_steps(b) * 32, q = (int64_t)b->query_items * b->lq, k = (int64_t)b->key_items * b->lk;
  auto take = [&](int64_t size) {
    const int64_t at = p.bytes;
    p.bytes += round_up(size, 256);
    return at;
  };
  p.rows = take(kNumbers * 4);
  p.query_columns = take(kColumns * 4);
  p.key_columns = take(kColumns * 4);
  p.query_places = take(q * 4);
  p.query_hot = take(q * width);
  p.key_places = b->same ? p.query_places : take(k * 4);
  p.key_hot = b->same ? p.query_hot : take(k * width);
  return p;
}

struct PlanArgs {
  const int* positions[2];  // (items, rows, axes)
  unsigned* places[2];
  __bf16* hot[2];
  int64_t rows[2];
  int* table;
  int axes, extents[4], width;
  unsigned short of[kDistances];  // the table's row of each distance's number
};

// blockIdx.y: the side; a thread makes a row's place and its one-hot row in pieces of eight columns.  The first
// workgroup also lays out the tables.
__global__ __launch_bounds__(256) void places_kernel(PlanArgs a) {
  const int side = blockIdx.y;
  if (side == 0 && blockIdx.x == 0) {
    for (int n = threadIdx.x; n < kNumbers; n += 256) a.table[n] = -1;
    __syncthreads();
    int number = 0, column = 0;
    for (int x = 0; x < a.axes; ++x) {
      const int extent = a.extents[x];
      for (int n = threadIdx.x; n < 2 * extent - 1; n += 256) a.table[number + n] = a.of[number + n];
      // from a query row at place 0 to column c's: its coordinate; from there to a key at place 0: less it
      for (int c = threadIdx.x; c < extent; c += 256) {
        a.table[kNumbers + column + c] = x << 16 | (number + extent - 1 + c);
        a.table[kNumbers + kColumns + column + c] = x << 16 | (number + extent - 1 - c);
      }
      number += 2 * extent - 1;
      column += extent;
    }
    // numbers that no distance has, whichever place is added or taken
    for (int c = column + threadIdx.x; c < kColumns; c += 256) {
      a.table[kNumbers + c] = kNumbers - 1;
      a.table[kNumbers + kColumns + c] = kNumbers - kColumns;
    }
  }
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows[side]) return;
  unsigned places = 0u;
  int columns[4], start = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    columns[x] = -1;
    if (x >= a.axes) continue;
    const int place = max(0, min(a.positions[side][row * a.axes + x], a.extents[x] - 1));
    places |= (unsigned)place << (8 * x);
    columns[x] = start + place;
    start += a.extents[x];
  }
  a.places[side][row] = places;
  for (int c = 0; c < a.width; c += 8) {
    Vec<unsigned short, 8> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      bool hot = false;
#pragma unroll
      for (int x = 0; x < 4; ++x) hot |= columns[x] == c + e;
      v[e] = hot ? 0x3f80 : 0;  // 1 in bf16
    }
    *reinterpret_cast<Vec<unsigned short, 8>*>(a.hot[side] + row * a.width + c) = v;
  }
}

}  // namespace

int check_buckets(const ctmr_masked_attention_desc* d, const ctmr_buckets_desc* b) {
  const int rc = check_plan(b);
  if (rc) return rc;
  if (b->lq != d->lq || b->lk != d->lk || (b->query_items != 1 && b->query_items != d->n) ||
      (b->key_items != 1 && b->key_items != d->n))
    return fail(CTMR_E_INVALID, "the places are of other rows");
  if (!valid_elem(b->table_elem)) return fail(CTMR_E_INVALID, "bad element type");
  if ((d->softcap > 0.f ? d->softcap : d->scale) < 0x1p-20f)  // so that what hides a pair is below every score
    return fail(CTMR_E_UNSUPPORTED, "scores too small for a position bias");
  return CTMR_OK;
}

Bias make_bias(const ctmr_masked_attention_desc* d, const ctmr_buckets_desc* b, const void* plan, const void* table) {
  const Parts p = parts_of(b);
  const char* base = static_cast<const char*>(plan);
  Bias r = {};
  r.rows = reinterpret_cast<const int*>(base + p.rows);
  r.query_columns = reinterpret_cast<const int*>(base + p.query_columns);
  r.key_columns = reinterpret_cast<const int*>(base + p.key_columns);
  r.query_places = reinterpret_cast<const unsigned*>(base + p.query_places);
  r.key_places = reinterpret_cast<const unsigned*>(base + p.key_places);
  r.query_hot = reinterpret_cast<const __bf16*>(base + p.query_hot);
  r.key_hot = reinterpret_cast<const __bf16*>(base + p.key_hot);
  r.query_item = b->query_items > 1 ? b->lq : 0;
  r.key_item = b->key_items > 1 ? b->lk : 0;
  r.table = table, r.elem = b->table_elem, r.table_rows = b->table_rows, r.axes = b->axes;
  int column = 0, number = 0;
  for (int a = 0; a < b->axes; ++a) {
    r.extents[a] = b->extents[a], r.first_column[a] = column, r.first_number[a] = number;
    column += b->extents[a], number += 2 * b->extents[a] - 1;
  }
  return r;
}

}  // namespace attn
}  // namespace ctmr

using namespace ctmr;
using namespace ctmr::attn;

extern "C" {

int64_t ctmr_buckets_bytes(const ctmr_buckets_desc* b) {
  const int rc = check_plan(b);
  if (rc) return rc;
  if (b->same && (b->lq != b->lk || b->query_items != b->key_items)) return fail(CTMR_E_INVALID, "sides differ in size");
  return parts_of(b).bytes;
}

int ctmr_buckets(const ctmr_buckets_desc* b, const int32_t* query_places, const int32_t* key_places, const int32_t* rows,
                 void* plan, size_t plan_bytes, void* stream) {
  const int64_t need = ctmr_buckets_bytes(b);
  if (need < 0) return (int)need;
  if (!query_places || (!key_places && !b->same) || !rows || !plan) return fail(CTMR_E_INVALID, "null pointer");
  if ((int64_t)plan_bytes < need || ((uintptr_t)plan & 15) != 0)
    return fail(CTMR_E_WORKSPACE, "plan of places too small or not on a 16-byte boundary");
  PlanArgs a = {};
  int numbers = 0;
  for (int x = 0; x < b->axes; ++x) numbers += 2 * b->extents[x] - 1;
  for (int n = 0; n < numbers; ++n) {
    if (rows[n] < 0 || rows[n] >= b->table_rows) return fail(CTMR_E_INVALID, "a row that the table does not have");
    a.of[n] = (unsigned short)rows[n];
  }
  const Parts p = parts_of(b);
  char* base = static_cast<char*>(plan);
  a.positions[0] = query_places, a.positions[1] = key_places;
  a.places[0] = reinterpret_cast<unsigned*>(base + p.query_places);
  a.places[1] = reinterpret_cast<unsigned*>(base + p.key_places);
  a.hot[0] = reinterpret_cast<__bf16*>(base + p.query_hot), a.hot[1] = reinterpret_cast<__bf16*>(base + p.key_hot);
  a.rows[0] = (int64_t)b->query_items * b->lq, a.rows[1] = b->same ? 0 : (int64_t)b->key_items * b->lk;
  a.table = reinterpret_cast<int*>(base + p.rows);
  a.axes = b->axes, a.width = 16 * bias_steps(b);
  std::copy(b->extents, b->extents + 4, a.extents);
  static_assert(kNumbers * 4 % 256 == 0 && kColumns * 4 % 256 == 0, "the tables lie one behind the other");
  hipLaunchKernelGGL(places_kernel, dim3((unsigned)ceil_div(std::max(a.rows[0], a.rows[1]), 256), b->same ? 1 : 2), dim3(256),
                     0, (hipStream_t)stream, a);
  return check_launch("places");
}

}  // extern "C"
