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

// The axes in two pairs, the pairing with the fewest values.
struct Pairs {
  int axis[kAxes], extent[kAxes];  // extent 1: no axis
  int values[2];
};
Pairs pairs_of(const ctmr_buckets_desc* b) {
  static const int kPairings[3][kAxes] = {{0, 1, 2, 3}, {0, 2, 1, 3}, {0, 3, 1, 2}};
  Pairs best = {};
  for (const auto& pairing : kPairings) {
    Pairs p;
    for (int i = 0; i < kAxes; ++i) {
      p.axis[i] = pairing[i] < b->axes ? pairing[i] : -1;
      p.extent[i] = p.axis[i] < 0 ? 1 : b->extents[p.axis[i]];
    }
    for (int i = 0; i < 2; ++i) p.values[i] = (2 * p.extent[2 * i] - 1) * (2 * p.extent[2 * i + 1] - 1);
    if (!best.values[0] || p.values[0] + p.values[1] < best.values[0] + best.values[1]) best = p;
  }
  return best;
}

struct Parts {
  int64_t rows, query_codes, key_codes, query_places, key_places, hot, bytes;
};

int64_t room_of(int rows) { return round_up(rows, kTile); }

// Where a plan's parts start.
Parts parts_of(const ctmr_buckets_desc* b) {
  Parts p = {};
  const int64_t q = b->query_items * room_of(b->lq), k = b->key_items * room_of(b->lk);
  auto take = [&](int64_t size) {
    const int64_t at = p.bytes;
    p.bytes += round_up(size, 256);
    return at;
  };
  p.rows = take(kDistances * 4);
  p.query_codes = take(q * 4);
  p.key_codes = take(k * 4);
  p.query_places = take(q * 4);
  p.key_places = take(k * 4);
  p.hot = take((int64_t)b->key_items * b->lk * bias_steps(b) * 32);
  return p;
}

struct PlanArgs {
  const int* positions[2];  // of rows and keys: (items, rows, axes)
  unsigned *codes[2], *places[2];
  int64_t count[2];  // words of all items
  int rows[2], room[2];
  __bf16* hot;
  int* table;
  int axes, extents[kAxes], width;
  Pairs pairs;
  unsigned short of[kDistances];  // the table's row of each distance's number
  int numbers;
};

// blockIdx.y: rows or keys; a thread makes the words of one of them, and a key's one-hot row.  The first workgroup also lays
// out the table's rows.
__global__ __launch_bounds__(256) void places_kernel(PlanArgs a) {
  const int side = blockIdx.y;
  if (side == 0 && blockIdx.x == 0)
    for (int n = threadIdx.x; n < kDistances; n += 256) a.table[n] = n < a.numbers ? a.of[n] : -1;
  const int64_t word = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (word >= a.count[side]) return;
  const int64_t item = word / a.room[side];
  const int i = (int)(word - item * a.room[side]);
  const bool real = i < a.rows[side];
  unsigned places = 0u;
  int place[kAxes], columns[kAxes], start = 0;
#pragma unroll
  for (int x = 0; x < kAxes; ++x) {
    place[x] = 0;
    columns[x] = -1;
    if (x >= a.axes) continue;
    if (real) place[x] = max(0, min(a.positions[side][(item * a.rows[side] + i) * a.axes + x], a.extents[x] - 1));
    places |= (unsigned)place[x] << (8 * x);
    columns[x] = start + place[x];
    start += a.extents[x];
  }
  // Bytes of a pair's value: a row's from its far end, so that no difference is negative; the second pair's are behind.
  unsigned code = 0u;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    unsigned at = 0u;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = 2 * p + e, axis = a.pairs.axis[n], extent = a.pairs.extent[n];
      int x = 0;
#pragma unroll
      for (int y = 0; y < kAxes; ++y) x = axis == y ? place[y] : x;
      at = at * (2 * extent - 1) + x + (side == 0 ? extent - 1 : 0);
    }
    if (p == 1 && side == 0) at += a.pairs.values[0];
    code |= at * 4 << (16 * p);
  }
  a.codes[side][word] = code;
  a.places[side][word] = places;
  if (side == 0 || !real) return;
  for (int c = 0; c < a.width; c += 8) {
    Vec<unsigned short, 8> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      bool hot = false;
#pragma unroll
      for (int x = 0; x < kAxes; ++x) hot |= columns[x] == c + e;
      v[e] = hot ? 0x3f80 : 0;  // 1 in bf16
    }
    *reinterpret_cast<Vec<unsigned short, 8>*>(a.hot + (item * a.rows[1] + i) * a.width + c) = v;
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
  auto words = [&](int64_t at) { return reinterpret_cast<const unsigned*>(base + at); };
  r.query_codes = words(p.query_codes), r.key_codes = words(p.key_codes);
  r.query_places = words(p.query_places), r.key_places = words(p.key_places);
  r.key_hot = reinterpret_cast<const __bf16*>(base + p.hot);
  r.query_item = b->query_items > 1 ? room_of(b->lq) : 0;
  r.key_item = b->key_items > 1 ? room_of(b->lk) : 0;
  r.hot_item = b->key_items > 1 ? b->lk : 0;
  r.table = table, r.elem = b->table_elem, r.table_rows = b->table_rows, r.axes = b->axes;
  int column = 0, number = 0;
  for (int a = 0; a < b->axes; ++a) {
    r.extents[a] = b->extents[a], r.first_column[a] = column, r.first_number[a] = number;
    r.reach |= (unsigned)(b->extents[a] - 1) << (8 * a);
    column += b->extents[a], number += 2 * b->extents[a] - 1;
  }
  const Pairs pairs = pairs_of(b);
  for (int i = 0; i < kAxes; ++i) {
    r.pair_extents[i] = pairs.extent[i];
    r.pair_number[i] = pairs.axis[i] < 0 ? -1 : r.first_number[pairs.axis[i]];
  }
  r.values = pairs.values[0] + pairs.values[1];
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
  for (int x = 0; x < b->axes; ++x) a.numbers += 2 * b->extents[x] - 1;
  for (int n = 0; n < a.numbers; ++n) {
    if (rows[n] < 0 || rows[n] >= b->table_rows) return fail(CTMR_E_INVALID, "a row that the table does not have");
    a.of[n] = (unsigned short)rows[n];
  }
  const Parts p = parts_of(b);
  char* base = static_cast<char*>(plan);
  auto words = [&](int64_t at) { return reinterpret_cast<unsigned*>(base + at); };
  a.positions[0] = query_places, a.positions[1] = b->same ? query_places : key_places;
  a.codes[0] = words(p.query_codes), a.codes[1] = words(p.key_codes);
  a.places[0] = words(p.query_places), a.places[1] = words(p.key_places);
  a.rows[0] = b->lq, a.rows[1] = b->lk;
  a.room[0] = (int)room_of(b->lq), a.room[1] = (int)room_of(b->lk);
  a.count[0] = (int64_t)b->query_items * a.room[0], a.count[1] = (int64_t)b->key_items * a.room[1];
  a.hot = reinterpret_cast<__bf16*>(base + p.hot);
  a.table = reinterpret_cast<int*>(base + p.rows);
  a.axes = b->axes, a.width = 16 * bias_steps(b), a.pairs = pairs_of(b);
  std::copy(b->extents, b->extents + kAxes, a.extents);
  hipLaunchKernelGGL(places_kernel, dim3((unsigned)ceil_div(std::max(a.count[0], a.count[1]), 256), 2), dim3(256), 0,
                     (hipStream_t)stream, a);
  return check_launch("places");
}

}  // extern "C"
