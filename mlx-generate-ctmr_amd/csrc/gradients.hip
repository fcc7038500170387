// The global norm of a list of gradients, their scaling by a factor on the
// device, and AdamW steps of a list of parameters, in fp32, bf16 and fp16.
//
//   norm = scale sqrt(sum g^2),  factor = scale min(1, most / (norm + 1e-6))
//   g' = factor g
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   w -= lr decay w + lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
// with w the parameter, or its fp32 copy where the parameter has 16 bits and gets
// the copy rounded, and t its own steps: all of the list's but those it had no
// gradient in.  Squares are added in fp64, which none of the types' values
// leave; moments, copies and all arithmetic of the step are fp32.
//
// The tensors of a list are passed in the kernels' arguments, so a launch takes up
// to kMost of them and nothing is copied to the device.  A workgroup works on a
// chunk of one tensor; it finds it by the chunks before each.  Sums have one order,
// set by the sizes alone.
//
// Bound by memory: the norm reads each gradient once, the scaling reads and writes
// it, a step moves 28 bytes an fp32 parameter.  240 tensors of 24 blocks of 1024 channels,
// fp32 (403 MB): the norm 52 + 26 us (5.1 TB/s; 79 + 27 behind a step's writes), its end
// 5, the scaling 79 + 48 (22 where the norm is below the limit), the steps 158 + 185 + 186
// (2.8 GB at 5.3 TB/s).  Short lists are bound by the host: 160 tensors of 16 blocks of 301
// channels, fp16, 105 us for 18 of kernels.
// (Chunks of four times as many values, each workgroup's own or in turns, take the 22 us
// to 13 and 9 but the 127 to 129 and 138, and steps to 540.)
#include "elements.hpp"

#include <algorithm>
#include <cmath>

namespace ctmr {
namespace {

constexpr int kThreads = 256;

// 16 bytes of values at any address that a value may have: the hardware's vector loads and stores take it.
template <typename T>
using Wide = T __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));

struct Entry {
  void* data;
  int64_t count;
  int first;  // chunk of the launch
  int elem;
};
constexpr int kMost = 160;  // entries that fit the 4 KB of a kernel's arguments
struct List {
  Entry entry[kMost];
  int64_t chunk;
  int entries;
};

// The entry of a chunk: the last that starts at it or before.
template <typename L>
__device__ __forceinline__ int entry_of(const L& list, int chunk) {
  int lo = 0, hi = list.entries - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (list.entry[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// A workgroup's sum, for its first thread.
template <int WAVES>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[WAVES];
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) total += part[w];
  return total;
}

template <typename T>
__device__ __forceinline__ double square_sum(const T* p, int64_t count) {
  constexpr int kWide = 16 / sizeof(T), kAhead = 4;  // loads on their way at once
  const int64_t wide = count / kWide, rounds = wide / (kAhead * kThreads) * kAhead * kThreads;
  double sum = 0.0;
  auto add = [&](const Wide<T>& v) {
#pragma unroll
    for (int e = 0; e < kWide; ++e) {
      const double x = (double)(float)v[e];
      sum = fma(x, x, sum);
    }
  };
  for (int64_t i = threadIdx.x; i < rounds; i += kAhead * kThreads) {
    Wide<T> v[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) v[a] = reinterpret_cast<const Wide<T>*>(p)[i + a * kThreads];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) add(v[a]);
  }
  for (int64_t i = rounds + threadIdx.x; i < wide; i += kThreads) add(reinterpret_cast<const Wide<T>*>(p)[i]);
  for (int64_t i = wide * kWide + threadIdx.x; i < count; i += kThreads) {
    const double x = (double)(float)p[i];
    sum = fma(x, x, sum);
  }
  return sum;
}

__global__ __launch_bounds__(kThreads) void square_sums_kernel(List list, double* sums) {
  const Entry& e = list.entry[entry_of(list, blockIdx.x)];
  const int64_t at = (blockIdx.x - e.first) * list.chunk, count = min(list.chunk, e.count - at);
  double sum;
  if (e.elem == CTMR_ELEM_F32) sum = square_sum(static_cast<const float*>(e.data) + at, count);
  else if (e.elem == CTMR_ELEM_BF16) sum = square_sum(static_cast<const __bf16*>(e.data) + at, count);
  else sum = square_sum(static_cast<const _Float16*>(e.data) + at, count);
  sum = block_sum<kThreads / 64>(sum);
  if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// What a step reads: the norm and the factor first, as ctmr_gradient_norm leaves them.
struct Control {
  float norm, factor;
  float lr_decay, go;  // lr decay, whether there is a step
};

// Without a limit the norm, which may be infinite or NaN, has no part in it.
__device__ __forceinline__ float clip_factor(float norm, float scale, float most) {
  const float f = most / (norm + 1e-6f);
  return most == INFINITY ? scale : scale * (f > 1.0f ? 1.0f : f);  // a NaN stays
}

__global__ __launch_bounds__(1024) void finish_norm_kernel(const double* sums, int count, float scale, float most,
                                                           float* out) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += 1024) sum += sums[i];
  sum = block_sum<16>(sum);
  if (threadIdx.x == 0) {
    out[0] = (float)(sqrt(sum) * fabs((double)scale));
    out[1] = clip_factor(out[0], scale, most);
  }
}

// What the bias corrections make of a parameter's steps.
struct Correction {
  float rate, root;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

// The control of a step from the norm (count 0: none is taken) and the steps so far, and the corrections of each of
// `parameters`, a thread each; `missed`: the steps that they had no part in, or null.
__global__ __launch_bounds__(1024) void begin_step_kernel(const double* sums, int count, ctmr_adamw_desc d, const float* lr,
                                                          int64_t* steps, int parameters, const int64_t* missed,
                                                          Control* control, Correction* corrections, float* norm) {
  const int64_t before = steps[0];  // the first thread writes it after the barrier
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += 1024) sum += sums[i];
  sum = block_sum<16>(sum);
  Control c;
  c.norm = (float)(sqrt(sum) * fabs((double)d.scale));
  c.factor = count > 0 ? clip_factor(c.norm, d.scale, d.most) : d.scale;
  const bool go = !d.skip || fabsf(c.norm) < INFINITY;
  const int64_t now = before + (go ? 1 : 0);
  const double rate = lr ? (double)lr[0] : d.lr;
  for (int i = threadIdx.x; i < parameters; i += 1024) {
    const double t = (double)max(now - (missed ? missed[i] : (int64_t)0), (int64_t)1);
    corrections[i] = {(float)(rate / (1.0 - pow(d.beta1, t))), (float)(1.0 / sqrt(1.0 - pow(d.beta2, t)))};
  }
  if (threadIdx.x != 0) return;
  if (go) steps[0] = now;
  c.lr_decay = (float)(rate * d.decay);
  c.go = go ? 1.f : 0.f;
  *control = c;
  if (norm) norm[0] = c.norm;
}

// Counts a step as missed for parameters that had no gradient, if it is taken.
constexpr int kMostNumbers = 960;
struct Numbers {
  int number[kMostNumbers];
  int count;
};
__global__ __launch_bounds__(kThreads) void count_missed_kernel(Numbers list, const Control* control, int64_t* missed) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i < list.count && control->go != 0.f) ++missed[list.number[i]];
}

template <typename T>
__device__ __forceinline__ void scale_values(T* p, int64_t count, float factor) {
  constexpr int kWide = 16 / sizeof(T);
  const int64_t wide = count / kWide;
  for (int64_t i = threadIdx.x; i < wide; i += kThreads) {
    Wide<T> v = reinterpret_cast<Wide<T>*>(p)[i];
#pragma unroll
    for (int e = 0; e < kWide; ++e) v[e] = (T)((float)v[e] * factor);
    reinterpret_cast<Wide<T>*>(p)[i] = v;
  }
  for (int64_t i = wide * kWide + threadIdx.x; i < count; i += kThreads) p[i] = (T)((float)p[i] * factor);
}

// With sums (`count` of them, a thread each at most) a workgroup makes the factor itself, and the first one leaves norm
// and factor in `out`: a launch less where the launches are what a call takes.
struct Sums {
  const double* sums;
  int count;
  float most;
  float* out;
};

__global__ __launch_bounds__(kThreads) void scale_kernel(List list, const float* factor, Sums sums) {
  const Entry& e = list.entry[entry_of(list, blockIdx.x)];
  const int64_t at = (blockIdx.x - e.first) * list.chunk, count = min(list.chunk, e.count - at);
  float f;
  if (sums.sums) {
    const double sum = block_sum<kThreads / 64>((int)threadIdx.x < sums.count ? sums.sums[threadIdx.x] : 0.0);
    const float norm = (float)sqrt(sum);
    f = clip_factor(norm, 1.0f, sums.most);
    if (blockIdx.x == 0 && threadIdx.x == 0 && sums.out) sums.out[0] = norm, sums.out[1] = f;
  } else {
    f = factor[0];
  }
  if (f == 1.0f) return;  // nothing would change
  if (e.elem == CTMR_ELEM_F32) scale_values(static_cast<float*>(e.data) + at, count, f);
  else if (e.elem == CTMR_ELEM_BF16) scale_values(static_cast<__bf16*>(e.data) + at, count, f);
  else scale_values(static_cast<_Float16*>(e.data) + at, count, f);
}

struct StepEntry {
  void* parameter;
  const void* gradient;
  int64_t count;
  int64_t start, master;  // of its moments and its fp32 copy
  int first;
  unsigned elem : 2, number : 30;  // its correction's
};
constexpr int kMostSteps = 80;
struct StepList {
  StepEntry entry[kMostSteps];
  float *m, *v, *master;
  const Control* control;
  const Correction* corrections;
  float beta1, beta2, eps;
  float rest1, rest2;  // 1 - beta
  int64_t chunk;
  int entries;
};

struct StepRule {
  float factor, lr_decay, rate, root, beta1, beta2, rest1, rest2, eps;
  __device__ __forceinline__ void operator()(float g, float& m, float& v, float& w) const {
    g *= factor;
    m = fmaf(beta1, m, rest1 * g);
    v = fmaf(beta2, v, rest2 * g * g);
    const float by = fmaf(sqrtf(v), root, eps);
    w -= fmaf(lr_decay, w, rate * (m / by));
  }
};

// The moments and copies start on 16 bytes, four values at a time; T's values where they are.
template <typename T>
__device__ __forceinline__ void step_values(const StepRule& rule, T* p, const T* g, float* m, float* v, float* master,
                                            int64_t count) {
  typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  typedef Vec<float, 4> F4;
  const int64_t wide = count / 4;
  for (int64_t i = threadIdx.x; i < wide; i += kThreads) {
    const T4 g4 = reinterpret_cast<const T4*>(g)[i];
    F4 m4 = reinterpret_cast<const F4*>(m)[i], v4 = reinterpret_cast<const F4*>(v)[i];
    F4 w4;
    if constexpr (sizeof(T) == 2) w4 = reinterpret_cast<const F4*>(master)[i];
    else w4 = reinterpret_cast<const T4*>(p)[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float me = m4[e], ve = v4[e], we = w4[e];
      rule((float)g4[e], me, ve, we);
      m4[e] = me, v4[e] = ve, w4[e] = we;
    }
    reinterpret_cast<F4*>(m)[i] = m4;
    reinterpret_cast<F4*>(v)[i] = v4;
    if constexpr (sizeof(T) == 2) reinterpret_cast<F4*>(master)[i] = w4;
    reinterpret_cast<T4*>(p)[i] = __builtin_convertvector(w4, Vec<T, 4>);
  }
  for (int64_t i = wide * 4 + threadIdx.x; i < count; i += kThreads) {
    float w = sizeof(T) == 2 ? master[i] : (float)p[i];
    rule((float)g[i], m[i], v[i], w);
    if constexpr (sizeof(T) == 2) master[i] = w;
    p[i] = (T)w;
  }
}

__global__ __launch_bounds__(kThreads) void adamw_kernel(StepList list) {
  const StepEntry& e = list.entry[entry_of(list, blockIdx.x)];
  const int64_t at = (blockIdx.x - e.first) * list.chunk, count = min(list.chunk, e.count - at);
  const Control c = *list.control;
  if (c.go == 0.f) return;
  const Correction by = list.corrections[e.number];
  const StepRule rule = {c.factor, c.lr_decay, by.rate, by.root, list.beta1, list.beta2, list.rest1, list.rest2, list.eps};
  float *m = list.m + e.start + at, *v = list.v + e.start + at;
  float* master = list.master ? list.master + e.master + at : nullptr;
  auto step = [&](auto* p, const auto* g) { step_values(rule, p + at, g + at, m, v, master, count); };
  if (e.elem == CTMR_ELEM_F32) step(static_cast<float*>(e.parameter), static_cast<const float*>(e.gradient));
  else if (e.elem == CTMR_ELEM_BF16) step(static_cast<__bf16*>(e.parameter), static_cast<const __bf16*>(e.gradient));
  else step(static_cast<_Float16*>(e.parameter), static_cast<const _Float16*>(e.gradient));
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------
constexpr int64_t kChunk = 4096;     // values of a chunk that is written
constexpr int64_t kSumsWanted = 2048;  // chunks of a norm, about

int64_t total_of(int count, const int64_t* sizes) {
  int64_t total = 0;
  for (int i = 0; i < count; ++i) total += sizes[i];
  return total;
}

// Values of a chunk whose squares one workgroup adds.
int64_t sum_chunk(int64_t total) { return round_up(std::max<int64_t>(ceil_div(total, kSumsWanted), 1), kChunk); }

int64_t chunks_of(int count, const int64_t* sizes, int64_t chunk) {
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) chunks += ceil_div(sizes[i], chunk);
  return chunks;
}

int check_list(int count, const void* const* tensors, const int64_t* sizes, const int32_t* elems) {
  if (count < 0 || (count > 0 && (!sizes || !elems || !tensors))) return fail(CTMR_E_INVALID, "null list");
  int64_t total = 0;
  for (int i = 0; i < count; ++i) {
    if (sizes[i] < 0) return fail(CTMR_E_INVALID, "negative size");
    if (!valid_elem(elems[i])) return fail(CTMR_E_INVALID, "bad element type");
    if (sizes[i] > 0 && !tensors[i]) return fail(CTMR_E_INVALID, "null tensor");
    if ((uintptr_t)tensors[i] % elem_bytes(elems[i]) != 0) return fail(CTMR_E_INVALID, "tensor off its type's grid");
    if (sizes[i] > (1ll << 40) || (total += sizes[i]) > (1ll << 40)) return fail(CTMR_E_UNSUPPORTED, "too many values");
  }
  // Chunks, of kThreads threads each, are counted in 32 bits.
  if (chunks_of(count, sizes, kChunk) > (1ll << 23)) return fail(CTMR_E_UNSUPPORTED, "too many values");
  return CTMR_OK;
}

// Launches `go(list, chunks)` for every kMost tensors that hold values.
template <typename F>
int for_lists(int count, void* const* tensors, const int64_t* sizes, const int32_t* elems, int64_t chunk, F go) {
  List list;
  list.chunk = chunk;
  int i = 0;
  while (i < count) {
    int chunks = 0;
    for (list.entries = 0; i < count && list.entries < kMost; ++i) {
      if (sizes[i] == 0) continue;
      list.entry[list.entries++] = {tensors[i], sizes[i], chunks, elems[i]};
      chunks += (int)ceil_div(sizes[i], chunk);
    }
    if (list.entries == 0) break;
    const int rc = go(list, chunks);
    if (rc) return rc;
  }
  return CTMR_OK;
}

// The sums of squares of all chunks; `count` of them.
int square_sums(int tensors, const void* const* data, const int64_t* sizes, const int32_t* elems, double* sums, int* count,
                hipStream_t st) {
  *count = 0;
  return for_lists(tensors, const_cast<void* const*>(data), sizes, elems,
                   sum_chunk(total_of(tensors, sizes)), [&](const List& list, int chunks) {
                     hipLaunchKernelGGL(square_sums_kernel, dim3(chunks), dim3(kThreads), 0, st, list, sums + *count);
                     *count += chunks;
                     return check_launch("square_sums");
                   });
}

int check_workspace(const void* ws, size_t bytes, int64_t need) {
  if (ws && (int64_t)bytes >= need && ((uintptr_t)ws & 15) == 0) return CTMR_OK;
  set_error("workspace of a list: %zu bytes given, %lld needed on a 16-byte boundary", bytes, (long long)need);
  return CTMR_E_WORKSPACE;
}

constexpr int64_t kControlBytes = 64;
constexpr int64_t kCorrectionAt = 32;  // of all parameters' where they have the same steps
static_assert(sizeof(Control) <= kCorrectionAt && kCorrectionAt + sizeof(Correction) <= kControlBytes && sizeof(List) + sizeof(Sums) + 16 <= 4096 && sizeof(StepList) <= 4096 &&
                  sizeof(Numbers) + 16 <= 4096,
              "argument sizes");
constexpr int kMostParameters = 1 << 24;

// The steps of `parameters` parameters, `count` of which have a gradient: entry i of the lists is number numbers[i], in
// order (null: i).  missed or null: all have the same steps.
int adamw(const ctmr_adamw_desc* d, int count, void* const* data, const void* const* gradients, const int64_t* sizes,
          const int32_t* elems, const int64_t* starts, const int64_t* master_starts, float* exp_avg, float* exp_avg_sq,
          float* master, int64_t* steps, int parameters, const int32_t* numbers, int64_t* missed, const float* lr, float* norm,
          void* workspace, size_t workspace_bytes, int64_t need, hipStream_t st) {
  int rc = check_list(count, data, sizes, elems);
  if (!rc) rc = check_list(count, gradients, sizes, elems);
  if (rc) return rc;
  if (!(d->beta1 >= 0.0 && d->beta1 < 1.0 && d->beta2 >= 0.0 && d->beta2 < 1.0) || !(d->eps >= 0.0) ||
      !(d->decay >= 0.0) || !(d->most > 0.f) || std::isnan(d->scale) || !(d->lr >= 0.0))
    return fail(CTMR_E_INVALID, "bad step: betas in [0, 1), eps, decay and lr not negative, most positive");
  if (!steps || (count > 0 && (!starts || !exp_avg || !exp_avg_sq))) return fail(CTMR_E_INVALID, "null pointer");
  bool half = false;
  for (int i = 0; i < count; ++i) {
    half |= elems[i] != CTMR_ELEM_F32;
    if (starts[i] < 0 || starts[i] % 4 != 0) return fail(CTMR_E_INVALID, "starts must be multiples of 4");
    if (numbers && (numbers[i] >= parameters || numbers[i] < (i > 0 ? numbers[i - 1] + 1 : 0)))
      return fail(CTMR_E_INVALID, "numbers must rise and be below the parameters'");
  }
  if (half && (!master || !master_starts)) return fail(CTMR_E_INVALID, "16-bit parameters need an fp32 copy");
  for (int i = 0; half && i < count; ++i)
    if (elems[i] != CTMR_ELEM_F32 && (master_starts[i] < 0 || master_starts[i] % 4 != 0))
      return fail(CTMR_E_INVALID, "starts must be multiples of 4");
  if ((((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq | (uintptr_t)master) & 15) != 0)
    return fail(CTMR_E_INVALID, "moments and copies must start on 16-byte boundaries");
  rc = check_workspace(workspace, workspace_bytes, need);
  if (rc) return rc;
  Control* control = static_cast<Control*>(workspace);
  double* sums = reinterpret_cast<double*>((char*)workspace + kControlBytes);
  Correction* corrections = reinterpret_cast<Correction*>(
      (char*)workspace + (missed ? ctmr_gradients_workspace_bytes(count, sizes) : kCorrectionAt));
  int sums_taken = 0;
  if (d->most < INFINITY || d->skip || norm) {
    rc = square_sums(count, gradients, sizes, elems, sums, &sums_taken, st);
    if (rc) return rc;
  }
  hipLaunchKernelGGL(begin_step_kernel, dim3(1), dim3(1024), 0, st, sums, sums_taken, *d, lr, steps, missed ? parameters : 1,
                     missed, control, corrections, norm);
  rc = check_launch("begin_step");
  if (rc) return rc;
  StepList list;
  list.m = exp_avg, list.v = exp_avg_sq, list.master = master, list.control = control, list.corrections = corrections;
  list.beta1 = (float)d->beta1, list.beta2 = (float)d->beta2, list.eps = (float)d->eps;
  list.rest1 = (float)(1.0 - d->beta1), list.rest2 = (float)(1.0 - d->beta2), list.chunk = kChunk;
  int i = 0;
  while (i < count) {
    int chunks = 0;
    for (list.entries = 0; i < count && list.entries < kMostSteps; ++i) {
      if (sizes[i] == 0) continue;
      StepEntry& e = list.entry[list.entries++];
      e.parameter = data[i], e.gradient = gradients[i], e.count = sizes[i], e.start = starts[i];
      e.master = elems[i] != CTMR_ELEM_F32 ? master_starts[i] : 0;
      e.first = chunks, e.elem = (unsigned)elems[i], e.number = (unsigned)(!missed ? 0 : numbers ? numbers[i] : i);
      chunks += (int)ceil_div(sizes[i], kChunk);
    }
    if (list.entries == 0) break;
    hipLaunchKernelGGL(adamw_kernel, dim3(chunks), dim3(kThreads), 0, st, list);
    rc = check_launch("adamw");
    if (rc) return rc;
  }
  if (!missed || count == parameters) return CTMR_OK;
  Numbers absent;
  for (int number = 0, at = 0; number < parameters;) {
    for (absent.count = 0; number < parameters && absent.count < kMostNumbers; ++number) {
      if (at < count && (numbers ? numbers[at] : at) == number) ++at;
      else absent.number[absent.count++] = number;
    }
    if (absent.count == 0) break;
    hipLaunchKernelGGL(count_missed_kernel, dim3((unsigned)ceil_div(absent.count, kThreads)), dim3(kThreads), 0, st, absent,
                       control, missed);
    rc = check_launch("count_missed");
    if (rc) return rc;
  }
  return CTMR_OK;
}

}  // namespace
}  // namespace ctmr

using namespace ctmr;

extern "C" {

int64_t ctmr_gradients_workspace_bytes(int32_t count, const int64_t* sizes) {
  if (count < 0 || (count > 0 && !sizes)) return fail(CTMR_E_INVALID, "null list");
  for (int i = 0; i < count; ++i) {
    if (sizes[i] < 0) return fail(CTMR_E_INVALID, "negative size");
    if (sizes[i] > (1ll << 40)) return fail(CTMR_E_UNSUPPORTED, "too many values");
  }
  return kControlBytes + round_up(chunks_of(count, sizes, sum_chunk(total_of(count, sizes))) * 8, 16);
}

int ctmr_gradient_norm(int32_t count, const void* const* gradients, const int64_t* sizes, const int32_t* elems,
                       float scale, float most, float* norm_factor, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_list(count, gradients, sizes, elems);
  if (rc) return rc;
  if (!norm_factor) return fail(CTMR_E_INVALID, "null pointer");
  if (!(most > 0.f) || std::isnan(scale)) return fail(CTMR_E_INVALID, "most must be positive");
  rc = check_workspace(workspace, workspace_bytes, ctmr_gradients_workspace_bytes(count, sizes));
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  double* sums = reinterpret_cast<double*>((char*)workspace + kControlBytes);
  int chunks = 0;
  rc = square_sums(count, gradients, sizes, elems, sums, &chunks, st);
  if (rc) return rc;
  hipLaunchKernelGGL(finish_norm_kernel, dim3(1), dim3(1024), 0, st, sums, chunks, scale, most, norm_factor);
  return check_launch("finish_norm");
}

int ctmr_scale_tensors(int32_t count, void* const* tensors, const int64_t* sizes, const int32_t* elems,
                       const float* factor, void* stream) {
  const int rc = check_list(count, tensors, sizes, elems);
  if (rc) return rc;
  if (!factor) return fail(CTMR_E_INVALID, "null pointer");
  return for_lists(count, tensors, sizes, elems, kChunk, [&](const List& list, int chunks) {
    hipLaunchKernelGGL(scale_kernel, dim3(chunks), dim3(kThreads), 0, (hipStream_t)stream, list, factor, Sums{});
    return check_launch("scale_tensors");
  });
}

int ctmr_clip_gradients(int32_t count, void* const* gradients, const int64_t* sizes, const int32_t* elems, float most,
                        float* norm_factor, void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t need = ctmr_gradients_workspace_bytes(count, sizes);
  if (need < 0) return (int)need;
  // Up to as many sums as a workgroup has threads, each workgroup adds them by itself: two launches instead of three, 26 us
  // for 30 with 10 tensors of 64 channels, bf16; with more of them each would add too many.
  const int64_t chunks = chunks_of(count, sizes, sum_chunk(total_of(count, sizes)));
  if (chunks == 0 || chunks > kThreads) {
    const int rc = ctmr_gradient_norm(count, gradients, sizes, elems, 1.0f, most, norm_factor, workspace, workspace_bytes,
                                      stream);
    return rc ? rc : ctmr_scale_tensors(count, gradients, sizes, elems, norm_factor + 1, stream);
  }
  int rc = check_list(count, gradients, sizes, elems);
  if (rc) return rc;
  if (!norm_factor) return fail(CTMR_E_INVALID, "null pointer");
  if (!(most > 0.f)) return fail(CTMR_E_INVALID, "most must be positive");
  rc = check_workspace(workspace, workspace_bytes, need);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  Sums sums = {reinterpret_cast<double*>((char*)workspace + kControlBytes), 0, most, norm_factor};
  rc = square_sums(count, gradients, sizes, elems, const_cast<double*>(sums.sums), &sums.count, st);
  if (rc) return rc;
  return for_lists(count, gradients, sizes, elems, kChunk, [&](const List& list, int blocks) {
    hipLaunchKernelGGL(scale_kernel, dim3(blocks), dim3(kThreads), 0, st, list, nullptr, sums);
    sums.out = nullptr;
    return check_launch("clip_gradients");
  });
}

int64_t ctmr_adamw_workspace_bytes(int32_t count, const int64_t* sizes, int32_t parameters) {
  const int64_t bytes = ctmr_gradients_workspace_bytes(count, sizes);
  if (bytes < 0) return bytes;
  if (parameters < count) return fail(CTMR_E_INVALID, "more gradients than parameters");
  if (parameters > kMostParameters) return fail(CTMR_E_UNSUPPORTED, "too many parameters");
  return bytes + round_up(parameters * (int64_t)sizeof(Correction), 16);
}

int ctmr_adamw(const ctmr_adamw_desc* d, int32_t count, void* const* parameters, const void* const* gradients,
               const int64_t* sizes, const int32_t* elems, const int64_t* starts, const int64_t* master_starts,
               float* exp_avg, float* exp_avg_sq, float* master, int64_t* steps, const float* lr, float* norm,
               void* workspace, size_t workspace_bytes, void* stream) {
  if (!d) return fail(CTMR_E_INVALID, "null descriptor");
  const int64_t need = ctmr_gradients_workspace_bytes(count, sizes);
  if (need < 0) return (int)need;
  return adamw(d, count, parameters, gradients, sizes, elems, starts, master_starts, exp_avg, exp_avg_sq, master, steps, count,
               nullptr, nullptr, lr, norm, workspace, workspace_bytes, need, (hipStream_t)stream);
}

int ctmr_adamw_counted(const ctmr_adamw_desc* d, int32_t count, void* const* data, const void* const* gradients,
                       const int64_t* sizes, const int32_t* elems, const int64_t* starts, const int64_t* master_starts,
                       float* exp_avg, float* exp_avg_sq, float* master, int64_t* steps, int32_t parameters,
                       const int32_t* numbers, int64_t* missed, const float* lr, float* norm, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (!d) return fail(CTMR_E_INVALID, "null descriptor");
  const int64_t need = ctmr_adamw_workspace_bytes(count, sizes, parameters);
  if (need < 0) return (int)need;
  if (!missed && parameters > 0) return fail(CTMR_E_INVALID, "null pointer");
  return adamw(d, count, data, gradients, sizes, elems, starts, master_starts, exp_avg, exp_avg_sq, master, steps, parameters,
               numbers, missed, lr, norm, workspace, workspace_bytes, need, (hipStream_t)stream);
}

}  // extern "C"
