// Masked attention's entry points, and the documents' plan: which tiles of one side
// the rows of the other meet.  The kernels are in masked_attention_forward.hpp.
#include "masked_attention_forward.hpp"

#include <climits>

namespace ctmr {
namespace attn {
namespace {

// --------------------------------------------------------------------------
// documents: ids of each side, ranges of its tiles and their hulls on the other
// --------------------------------------------------------------------------
struct DocArgs {
  const int* from[2];
  int* ids[2];
  DocTile* tiles[2];
  int4* hull[2];
  int* mixed[2];
  int rows[2], stride[2], count[2], grains[2];
};

// One wave per tile: blockIdx = (tile, item, side).
__global__ __launch_bounds__(kTile) void document_tiles_kernel(DocArgs a) {
  const int side = blockIdx.z, b = blockIdx.y, tile = blockIdx.x, lane = threadIdx.x;
  if (tile >= a.count[side]) return;
  const int i = tile * kTile + lane;
  const bool real = i < a.rows[side];
  const int id = real ? max(a.from[side][(int64_t)b * a.rows[side] + i], -1) : -1;
  a.ids[side][(int64_t)b * a.stride[side] + i] = id;
  int least = real ? id : INT_MAX, most = id, least_id = id >= 0 ? id : INT_MAX;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    least = min(least, __shfl_xor(least, m));
    most = max(most, __shfl_xor(most, m));
    least_id = min(least_id, __shfl_xor(least_id, m));
  }
  if (lane == 0) a.tiles[side][(int64_t)b * a.count[side] + tile] = DocTile{least, most, least_id, 0};
}

// Tiles of a side [x, y) that may hold ids least .. most, and the first run [z, w) of tiles that hold only the one
// id, for least = most >= 0.
__device__ __forceinline__ int4 document_run(const DocArgs& a, int side, int b, int lane, int least, int most) {
  const DocTile* tiles = a.tiles[side] + (int64_t)b * a.count[side];
  const int count = a.count[side];
  const bool one = least == most;
  int4 run = {INT_MAX, 0, INT_MAX, 0};
  if (most < 0 || least > most) return run;
  for (int o = lane; o < count; o += kTile) {
    const DocTile tile = tiles[o];
    if (least <= tile.most && tile.least_id <= most) {
      run.x = min(run.x, o);
      run.y = max(run.y, o + 1);
    }
    if (one && tile.least == least && tile.most == least) run.z = min(run.z, o);
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    run.x = min(run.x, __shfl_xor(run.x, m));
    run.y = max(run.y, __shfl_xor(run.y, m));
    run.z = min(run.z, __shfl_xor(run.z, m));
  }
  int end = run.z == INT_MAX ? 0 : count;
  for (int o = lane; o < end; o += kTile)
    if (o > run.z && (tiles[o].least != least || tiles[o].most != least)) end = min(end, o);
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) end = min(end, __shfl_xor(end, m));
  run.w = end;
  return run;
}

// One wave per kGrain rows: blockIdx = (grain, item, side).
__global__ __launch_bounds__(kTile) void document_hulls_kernel(DocArgs a) {
  const int side = blockIdx.z, b = blockIdx.y, grain = blockIdx.x, lane = threadIdx.x;
  if (grain >= a.grains[side]) return;
  if (grain % 4 == 0) {
    const int* ids = a.ids[side] + (int64_t)b * a.stride[side];
    bool other = false;
#pragma unroll
    for (int r = lane; r < kBlockRows; r += kTile) {
      const int row = grain * kGrain + r;
      other |= row < a.rows[side] && ids[row] != ids[grain * kGrain];
    }
    other = __any(other);
    if (lane == 0) a.mixed[side][(int64_t)b * ((a.grains[side] + 3) / 4) + grain / 4] = other;
  }
  const int i = grain * kGrain + lane % kGrain;
  const int id = i < a.rows[side] ? a.ids[side][(int64_t)b * a.stride[side] + i] : -1;
  // The first row's document, and the range of the other rows' ids, padding aside: which tiles may hold them, and
  // the first run of tiles that hold nothing else.
  const int first = __shfl(id, 0);
  int least = id >= 0 && id != first ? id : INT_MAX, most = id != first ? id : -1;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    least = min(least, __shfl_xor(least, m));
    most = max(most, __shfl_xor(most, m));
  }
  const bool padded = __any(i < a.rows[side] && id < 0 && first >= 0);
  const int4 own = document_run(a, 1 - side, b, lane, first, first);
  int4 rest = document_run(a, 1 - side, b, lane, least, most);
  if (padded) rest.z = INT_MAX, rest.w = 0;  // the padding goes with the other documents and sees none of their tiles
  if (lane == 0) {
    int4* hull = a.hull[side] + 3 * ((int64_t)b * a.grains[side] + grain);
    hull[0] = own;
    hull[1] = rest;
    // padding among the rows is as good as another document that no tile holds, so no tile is whole for the rest
    hull[2] = least <= most ? int4{padded ? -1 : least, most, 0, 0} : padded ? int4{-1, -1, 0, 0} : int4{1, 0, 0, 0};
  }
}

}  // namespace

int padded(int head_dim) { return head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : 128; }

static Side side_of(int rows, const int* ids, const void* tiles, const void* hull, const int* mixed) {
  Side s = {};
  s.ids = ids;
  s.tiles = static_cast<const DocTile*>(tiles);
  s.hull = static_cast<const int4*>(hull);
  s.mixed = mixed;
  s.count = (int)ceil_div(rows, kTile);
  s.stride = s.count * kTile;
  s.grains = (int)ceil_div(rows, kGrain);
  return s;
}

// A plan's parts: ids of both sides, tiles of both, hulls of both.
static void plan_parts(int32_t n, int32_t lq, int32_t lk, char* base, Side& q, Side& k, int64_t* bytes) {
  const int64_t nq = ceil_div(lq, kTile), nk = ceil_div(lk, kTile);
  int64_t at = 0;
  auto take = [&](int64_t size) {
    const int64_t here = at;
    at += size;
    return base ? base + here : nullptr;
  };
  const int* qi = (const int*)take(n * nq * kTile * 4);
  const int* ki = (const int*)take(n * nk * kTile * 4);
  const void* qt = take(n * nq * (int64_t)sizeof(DocTile));
  const void* kt = take(n * nk * (int64_t)sizeof(DocTile));
  const void* qh = take(n * ceil_div(lq, kGrain) * 48);
  const void* kh = take(n * ceil_div(lk, kGrain) * 48);
  const int* qm = (const int*)take(n * ceil_div(lq, kBlockRows) * 4);
  const int* km = (const int*)take(n * ceil_div(lk, kBlockRows) * 4);
  q = side_of(lq, qi, qt, qh, qm);
  k = side_of(lk, ki, kt, kh, km);
  if (bytes) *bytes = at;
}

int check_desc(const ctmr_masked_attention_desc* d) {
  if (!d) return fail(CTMR_E_INVALID, "null descriptor");
  if (d->n <= 0 || d->lq <= 0 || d->lk <= 0 || d->q_heads <= 0 || d->k_heads <= 0)
    return fail(CTMR_E_INVALID, "non-positive dimension");
  if (d->q_heads % d->k_heads != 0) return fail(CTMR_E_INVALID, "query heads must be a multiple of key heads");
  if (!valid_elem(d->elem)) return fail(CTMR_E_INVALID, "bad element type");
  if (d->head_dim <= 0 || d->head_dim % 8 != 0 || d->head_dim > 128)
    return fail(CTMR_E_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128");
  if (!(d->scale > 0.f) || !(d->scale < INFINITY) || !(d->softcap >= 0.f) || !(d->softcap < INFINITY))
    return fail(CTMR_E_INVALID, "scale must be positive, softcap not negative, both finite");
  if (d->softcap > 0.f && !(d->scale / d->softcap < 1e30f))
    return fail(CTMR_E_INVALID, "softcap too small for the scale");
  if (d->softcap > 1e30f || (d->softcap > 0.f && d->scale / d->softcap < 1e-30f))  // fp32 ends not far above
    return fail(CTMR_E_INVALID, "softcap too large for the scale");
  if (d->lq > (1 << 28) || d->lk > (1 << 28) ||
      (int64_t)d->n * d->q_heads * ceil_div(std::max(d->lq, d->lk), kTile) > (1ll << 23))  // 2^32 threads
    return fail(CTMR_E_UNSUPPORTED, "too many rows");
  int rc = check_strides(d, d->q_strides, d->lq);
  if (!rc) rc = check_strides(d, d->k_strides, d->lk);
  return rc ? rc : check_strides(d, d->v_strides, d->lk);
}

// Rows may not overlap: the kernels take what lies past the last one as out of range.
int check_strides(const ctmr_masked_attention_desc* d, const int64_t* s, int rows) {
  const int bytes = elem_bytes(d->elem);
  if (s[0] < 0 || s[1] < 0 || s[2] < 0 || (s[0] | s[1] | s[2]) * bytes % 16 != 0)
    return fail(CTMR_E_INVALID, "strides must be multiples of 16 bytes and not negative");
  if (rows > 1 && s[2] < d->head_dim) return fail(CTMR_E_INVALID, "rows overlap");
  if (s[2] * bytes > (1ll << 30) / kTile - 4096) return fail(CTMR_E_UNSUPPORTED, "row stride too large");
  return CTMR_OK;
}

int64_t row_stride(const int64_t* s, int rows, int head_dim) { return rows > 1 ? s[2] : head_dim; }

int check_call(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v, const void* plan,
               const void* out, const void* rest, const void* workspace, size_t workspace_bytes, int64_t need) {
  if (!q || !k || !v || !out) return fail(CTMR_E_INVALID, "null pointer");
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)rest | (uintptr_t)plan) & 15) !=
      0)
    return fail(CTMR_E_INVALID, "q, k, v, out, rest and the document plan must start on 16-byte boundaries");
  if ((d->out_strides[0] | d->out_strides[1] | d->out_strides[2]) % 4 != 0)
    return fail(CTMR_E_INVALID, "strides of out must be multiples of 4 values");
  if (need > 0 && ((int64_t)workspace_bytes < need || !workspace || ((uintptr_t)workspace & 15) != 0)) {
    set_error("attention workspace: %zu bytes given, %lld needed on a 16-byte boundary", workspace_bytes,
              (long long)need);
    return CTMR_E_WORKSPACE;
  }
  return CTMR_OK;
}

Args make_args(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v, const float* slopes,
               const int32_t* prefixes, const void* plan) {
  Args a = {};
  a.q = q, a.k = k, a.v = v, a.slopes = slopes, a.prefixes = prefixes;
  a.n = d->n, a.lq = d->lq, a.lk = d->lk, a.hq = d->q_heads, a.hk = d->k_heads, a.group = d->q_heads / d->k_heads;
  a.d = d->head_dim, a.prefixed = d->prefixed != 0, a.prefix = d->prefix, a.scale = d->scale, a.cap = d->softcap;
  a.qb = d->q_strides[0], a.qh = d->q_strides[1], a.ql = row_stride(d->q_strides, d->lq, d->head_dim);
  a.kb = d->k_strides[0], a.kh = d->k_strides[1], a.kl = row_stride(d->k_strides, d->lk, d->head_dim);
  a.vb = d->v_strides[0], a.vh = d->v_strides[1], a.vl = row_stride(d->v_strides, d->lk, d->head_dim);
  a.splits = 1;
  if (plan) plan_parts(d->n, d->lq, d->lk, (char*)plan, a.qdoc, a.kdoc, nullptr);
  return a;
}

}  // namespace attn
}  // namespace ctmr

using namespace ctmr;
using namespace ctmr::attn;

extern "C" {

int64_t ctmr_documents_bytes(int32_t n, int32_t lq, int32_t lk) {
  if (n <= 0 || lq <= 0 || lk <= 0) return fail(CTMR_E_INVALID, "non-positive dimension");
  if (n > 65535 || lq > (1 << 28) || lk > (1 << 28)) return fail(CTMR_E_UNSUPPORTED, "too many rows");
  Side q, k;
  int64_t bytes = 0;
  plan_parts(n, lq, lk, nullptr, q, k, &bytes);
  return bytes;
}

int ctmr_documents(int32_t n, int32_t lq, int32_t lk, const int32_t* query_ids, const int32_t* key_ids, void* plan,
                   size_t plan_bytes, void* stream) {
  const int64_t need = ctmr_documents_bytes(n, lq, lk);
  if (need < 0) return (int)need;
  if (!query_ids || !key_ids || !plan) return fail(CTMR_E_INVALID, "null pointer");
  if ((int64_t)plan_bytes < need || ((uintptr_t)plan & 15) != 0)
    return fail(CTMR_E_WORKSPACE, "document plan too small or not on a 16-byte boundary");
  Side q, k;
  plan_parts(n, lq, lk, (char*)plan, q, k, nullptr);
  DocArgs a = {};
  a.from[0] = query_ids, a.from[1] = key_ids;
  const Side* sides[2] = {&q, &k};
  const int rows[2] = {lq, lk};
  for (int s = 0; s < 2; ++s) {
    a.ids[s] = const_cast<int*>(sides[s]->ids);
    a.tiles[s] = const_cast<DocTile*>(sides[s]->tiles);
    a.hull[s] = const_cast<int4*>(sides[s]->hull);
    a.mixed[s] = const_cast<int*>(sides[s]->mixed);
    a.rows[s] = rows[s], a.stride[s] = sides[s]->stride, a.count[s] = sides[s]->count;
    a.grains[s] = sides[s]->grains;
  }
  const dim3 grid(std::max(a.count[0], a.count[1]), n, 2);
  hipLaunchKernelGGL(document_tiles_kernel, grid, dim3(kTile), 0, (hipStream_t)stream, a);
  const int rc = check_launch("document_tiles");
  if (rc) return rc;
  hipLaunchKernelGGL(document_hulls_kernel, dim3(std::max(a.grains[0], a.grains[1]), n, 2), dim3(kTile), 0,
                     (hipStream_t)stream, a);
  return check_launch("document_hulls");
}

int64_t ctmr_masked_attention_workspace_bytes(const ctmr_masked_attention_desc* d) {
  const int rc = check_desc(d);
  if (rc) return rc;
  const int64_t splits = split_count(d);
  return splits == 1 ? 0 : splits * d->n * d->q_heads * d->lq * (padded(d->head_dim) + 2) * 4;
}

int ctmr_masked_attention(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v,
                          const float* slopes, const int32_t* prefixes, const void* plan, void* out, void* rest,
                          float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t need = ctmr_masked_attention_workspace_bytes(d);
  if (need < 0) return (int)need;
  const int rc = check_call(d, q, k, v, plan, out, rest, workspace, workspace_bytes, need);
  if (rc) return rc;
  Args a = make_args(d, q, k, v, slopes, prefixes, plan);
  a.out = out, a.rest = rest, a.lse = lse, a.part = (float*)workspace, a.splits = split_count(d);
  a.ob = d->out_strides[0], a.oh = d->out_strides[1], a.ol = d->out_strides[2];
  const bool few = few_rows(d);
  const BiasOf<0> none;
  hipStream_t st = (hipStream_t)stream;
#define CTMR_ATTENTION_CASE(T)                          \
  switch (padded(d->head_dim)) {                        \
    case 32: return launch<T, 32>(a, none, few, st);    \
    case 64: return launch<T, 64>(a, none, few, st);    \
    default: return launch<T, 128>(a, none, few, st);   \
  }
  if (d->elem == CTMR_ELEM_F32) CTMR_ATTENTION_CASE(float)
  if (d->elem == CTMR_ELEM_BF16) CTMR_ATTENTION_CASE(__bf16)
  CTMR_ATTENTION_CASE(_Float16)
#undef CTMR_ATTENTION_CASE
}

}  // extern "C"
