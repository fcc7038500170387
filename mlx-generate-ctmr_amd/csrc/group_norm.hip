// Group norm with an optional SiLU over channels-last rows, forward and
// backward, on fp32, bf16 and fp16 activations.
//
// x is (n, s, c): s voxels of c channels, a group is c / groups neighbouring
// channels over all voxels of a batch item, M = s * c / groups values.
//   mean = sum x / M, rstd = (sum (x - mean)^2 / M + eps)^-1/2
//   xhat = (x - mean) rstd, z = gamma xhat + beta, y = z or z sigmoid(z)
// and with dz = dy y'(z)
//   dbeta_c = sum dz, dgamma_c = sum dz xhat          (over voxels and items)
//   dx = rstd (gamma dz - A - xhat B),  A = sum_c gamma_c dbeta_nc / M,
//                                       B = sum_c gamma_c dgamma_nc / M.
// Both directions are per-channel sums followed by an element-wise pass, bound
// by HBM: x is read twice (the second time from the 256 MB memory-side cache
// where it fits), in the backward pass dy too.  Sums are fp64, but for 32 rows at a
// time in fp32, of x less the thread's first value: E[x^2] - mean^2 then keeps the
// variance of a channel whose mean is a thousand times its spread.  Rows whose squares
// leave fp32's range are added again in fp64.  The mean is kept as two floats (hi + lo),
// so x - mean is exact to fp32 also there.
// Measured: 80x128x128 voxels of 64 channels, bf16: forward 103 us, backward 194 (3.3
// and 2.6 TB/s of the bytes that both passes would need at least, 4.7 a copy);
// 45x90x117 of 128, fp16: 74 and 129 of values that the cache holds, 95 forward of
// others; 2 x 8x8x4 of 512, bf16 (small form): 12 and 17, the launches' time.
//
// Two forms:
//  * small (gn_small_*): a group's values stay in the registers of one
//    workgroup between the sums and the element-wise pass: one launch (two
//    backward with several items, whose dgamma are added in order by the second).
//  * large: partial sums per (item, chunk of voxels, channel), a fixed-order
//    reduction per group, the element-wise pass: three launches each way.
// No atomics: every sum has an order given by the shape.
#include "elements.hpp"

#include <algorithm>
#include <type_traits>

namespace ctmr {
namespace {

constexpr int kThreads = 256;
constexpr int kSmallThreads = 512;
constexpr int kSmallBytes = 64;  // bytes of values a thread of the small form holds

struct Mean {  // saved per (item, group)
  float hi, lo, rstd, unused;
};

struct NormArgs {
  const void* x;
  const void* dy;
  const void* gamma;
  const void* beta;
  void* y;          // y forward, dx backward
  Mean* saved;
  double* part;     // (n, chunks, c, 2)
  float* coef;      // (n, groups, 2): A, B
  double* sums;     // small backward, n > 1: (n, c, 2)
  void* dgamma;
  void* dbeta;
  int64_t s;
  int64_t chunk;    // voxels of a chunk
  int n, c, groups, cpg, chunks, cols;  // cols: channel vectors
  int ptype, silu;
  float eps;
};

__device__ __forceinline__ Mean finish(double sum, double sq, double count, float eps) {
  const double mean = sum / count;
  const double var = sq / count - mean * mean;
  Mean m;
  m.hi = (float)mean;
  m.lo = (float)(mean - (double)m.hi);
  m.rstd = (float)(1.0 / sqrt((var > 0.0 || var != var ? var : 0.0) + (double)eps));
  m.unused = 0.f;
  return m;
}

__device__ __forceinline__ float xhat_of(float x, const Mean& m) { return ((x - m.hi) - m.lo) * m.rstd; }

// dy y'(z)
__device__ __forceinline__ float through_silu(float dy, float z) {
  const float sig = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z));
  return dy * (sig * fmaf(z, 1.0f - sig, 1.0f));
}

// Sums W values of the `rows` threads of each of `cols` columns (thread = row * cols
// + col, others idle) that lie in LDS, value k of a thread at k * rows * cols +
// thread; the threads of row 0 get the result.  The tree's shape depends on rows only.
template <int W>
__device__ __forceinline__ void sum_rows(double (&v)[W], double* lds, int col, int row, int rows, int cols,
                                         bool active) {
  const int stride = cols * rows;
  int left = rows;
  while (left > 1) {
    const int half = (left + 1) >> 1;
    __syncthreads();
    if (active && row < left - half)
#pragma unroll
      for (int k = 0; k < W; ++k) lds[k * stride + row * cols + col] += lds[k * stride + (row + half) * cols + col];
    left = half;
  }
  __syncthreads();
  if (active && row == 0)
#pragma unroll
    for (int k = 0; k < W; ++k) v[k] = lds[k * stride + col];
}

template <int W>
__device__ __forceinline__ void reduce_rows(double (&v)[W], double* lds, int col, int row, int rows, int cols,
                                            bool active) {
  if (active)
#pragma unroll
    for (int k = 0; k < W; ++k) lds[k * cols * rows + row * cols + col] = v[k];
  sum_rows<W>(v, lds, col, row, rows, cols, active);
}

// Per-channel sums of a chunk: x and x^2, or backward dz and dz xhat.  A thread sums kBatch rows in fp32 before they
// join its fp64 sums: with three fp64 operations a value the backward sums took 99 us for 80x128x128 voxels of 64
// channels in bf16, bound by them, not by memory.  Forward the fp32 sums are of x - x0, x0 the thread's first value of
// the channel, so that they lose nothing to a mean far above the spread.
constexpr int kBatch = 32;

// Whether fp32 lost a batch's squares: an overflow (spreads past 1.8e19, and NaN, which fp64 does not mend either), or
// with an eps that is nothing beside them an underflow.  Never of fp16's range.
template <typename T, int V>
__device__ __forceinline__ bool outside_fp32(const Vec<float, V>& q, float eps) {
  if constexpr (std::is_same_v<T, _Float16>) return false;
  const float least = eps < 1e-18f ? 0x1p-90f : -1.0f;  // 32 squares, each off by 2^-150 at most
  bool lost = false;
#pragma unroll
  for (int k = 0; k < V; ++k) lost |= !(q[k] < INFINITY) || q[k] < least;
  return lost;
}

// Such a batch again, in fp64 throughout.
template <typename T, int V>
__device__ __forceinline__ void add_wide(double* acc, int slots, const T* x, int64_t step, int batch, Vec<float, V> x0) {
#pragma unroll 1
  for (int r = 0; r < batch; ++r) {
    const Vec<float, V> v = load_as_float<T, V>(x + r * step);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const double d = (double)v[k] - (double)x0[k];
      acc[k * slots] += d;
      acc[(V + k) * slots] += d * d;
    }
  }
}

// The fp64 sums wait in LDS, where they are added up at the end.
template <typename T, int V, bool BACKWARD>
__global__ __launch_bounds__(kThreads, BACKWARD ? 4 : 5) void gn_sums_kernel(NormArgs a) {
  __shared__ double lds[2 * V * kThreads];
  const int b = blockIdx.y;
  const int col0 = blockIdx.z * kThreads;
  const int cols = min(a.cols - col0, kThreads), rows = kThreads / cols;
  const int col = threadIdx.x % cols, row = threadIdx.x / cols;
  const bool active = row < rows;
  const int c0 = (col0 + col) * V;
  const int slots = rows * cols;
  double* acc = lds + threadIdx.x;
  if (active) {
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) acc[k * slots] = 0.0;
    const int64_t first = (int64_t)blockIdx.x * a.chunk + row, last = min((int64_t)(blockIdx.x + 1) * a.chunk, a.s);
    const int64_t step = (int64_t)rows * a.c;
    const T* x = static_cast<const T*>(a.x) + ((int64_t)b * a.s + first) * a.c + c0;
    int left = first < last ? (int)((last - first + rows - 1) / rows) : 0;
    const int count = left;
    if constexpr (!BACKWARD) {
      Vec<float, V> x0 = Vec<float, V>(0.f);
      if (left > 0) x0 = load_as_float<T, V>(x);
      while (left > 0) {
        Vec<float, V> p = Vec<float, V>(0.f), q = Vec<float, V>(0.f);
        const int batch = min(left, kBatch);
#pragma unroll 8
        for (int r = 0; r < batch; ++r) {
          const Vec<float, V> d = load_as_float<T, V>(x) - x0;
          x += step;
          p += d;
#pragma unroll
          for (int k = 0; k < V; ++k) q[k] = fmaf(d[k], d[k], q[k]);
        }
        left -= batch;
        if (__builtin_expect(outside_fp32<T, V>(q, a.eps), 0)) {
          add_wide<T, V>(acc, slots, x - batch * step, step, batch, x0);
          continue;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
          acc[k * slots] += (double)p[k];
          acc[(V + k) * slots] += (double)q[k];
        }
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {  // sums of x and x^2 again
        const double base = (double)x0[k], sum = acc[k * slots], all = fma((double)count, base, sum);
        acc[k * slots] = all;
        acc[(V + k) * slots] += base * (sum + all);
      }
    } else {
      const T* dy = static_cast<const T*>(a.dy) + ((int64_t)b * a.s + first) * a.c + c0;
      Mean m[V];
      float gamma[V], beta[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        m[k] = a.saved[b * a.groups + (c0 + k) / a.cpg];
        gamma[k] = load_param(a.gamma, a.ptype, c0 + k);
        beta[k] = load_param(a.beta, a.ptype, c0 + k);
      }
      while (left > 0) {
        Vec<float, V> p = Vec<float, V>(0.f), q = Vec<float, V>(0.f);
        const int batch = min(left, kBatch);
#pragma unroll(16 / V < 4 ? 16 / V : 4)
        for (int r = 0; r < batch; ++r) {
          const Vec<float, V> v = load_as_float<T, V>(x), g = load_as_float<T, V>(dy);
          x += step;
          dy += step;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float xh = xhat_of(v[k], m[k]);
            const float dz = a.silu ? through_silu(g[k], fmaf(gamma[k], xh, beta[k])) : g[k];
            p[k] += dz;
            q[k] = fmaf(dz, xh, q[k]);
          }
        }
        left -= batch;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          acc[k * slots] += (double)p[k];
          acc[(V + k) * slots] += (double)q[k];
        }
      }
    }
  }
  double sums[2 * V];
  sum_rows<2 * V>(sums, lds, col, row, rows, cols, active);
  if (active && row == 0) {
    double* out = a.part + (((int64_t)b * a.chunks + blockIdx.x) * a.c + c0) * 2;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      out[2 * k] = sums[k];
      out[2 * k + 1] = sums[V + k];
    }
  }
}

// A workgroup's sum of a pair, in a fixed order; every thread gets it.
__device__ __forceinline__ void block_sum2(double& p, double& q, double* lds, int threads) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    p += __shfl_xor(p, m);
    q += __shfl_xor(q, m);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    lds[2 * (threadIdx.x >> 6)] = p;
    lds[2 * (threadIdx.x >> 6) + 1] = q;
  }
  __syncthreads();
  p = q = 0.0;
  for (int w = 0; w < threads / 64; ++w) {
    p += lds[2 * w];
    q += lds[2 * w + 1];
  }
}

// (mean, rstd) of a group from its channels' partials: blockIdx = (group, item).
constexpr int kWide = 256;
__global__ __launch_bounds__(kWide) void gn_mean_kernel(NormArgs a) {
  __shared__ double lds[2 * kWide / 64];
  const int g = blockIdx.x, b = blockIdx.y;
  double p = 0.0, q = 0.0;
  const double* part = a.part + ((int64_t)b * a.chunks * a.c + (int64_t)g * a.cpg) * 2;
#pragma unroll 4
  for (int i = threadIdx.x; i < a.chunks * a.cpg; i += kWide) {
    const double2 v = *reinterpret_cast<const double2*>(part + ((int64_t)(i / a.cpg) * a.c + i % a.cpg) * 2);
    p += v.x;
    q += v.y;
  }
  block_sum2(p, q, lds, kWide);
  if (threadIdx.x == 0) a.saved[b * a.groups + g] = finish(p, q, (double)a.s * a.cpg, a.eps);
}

// One workgroup a group: for each item the sums of its channels over the chunks, which give A and B; over the items
// (in order) dgamma and dbeta.
__global__ __launch_bounds__(kWide) void gn_params_kernel(NormArgs a) {
  __shared__ double lds[2 * kWide];
  const int g = blockIdx.x;
  const int cols = min(a.cpg, kWide), rows = kWide / cols;
  const int col = threadIdx.x % cols, row = threadIdx.x / cols;
  const bool active = row < rows;
  const double count = (double)a.s * a.cpg;
  for (int c0 = 0; c0 < a.cpg; c0 += cols) {  // more channels than threads: block by block
    const int c = g * a.cpg + c0 + col;
    const bool real = active && c0 + col < a.cpg;
    double beta = 0.0, gamma = 0.0;
    const double weight = real ? (double)load_param(a.gamma, a.ptype, c) : 0.0;
    for (int b = 0; b < a.n; ++b) {
      double v[2] = {0.0, 0.0};
      if (real) {
        const double* part = a.part + ((int64_t)b * a.chunks * a.c + c) * 2;
#pragma unroll 4
        for (int i = row; i < a.chunks; i += rows) {
          const double2 d = *reinterpret_cast<const double2*>(part + (int64_t)i * a.c * 2);
          v[0] += d.x;
          v[1] += d.y;
        }
      }
      __syncthreads();  // the last item's sums are read
      reduce_rows<2>(v, lds, col, row, rows, cols, active);
      const bool first = active && row == 0;
      beta += first ? v[0] : 0.0;
      gamma += first ? v[1] : 0.0;
      double p = first ? weight * v[0] : 0.0, q = first ? weight * v[1] : 0.0;
      __syncthreads();
      block_sum2(p, q, lds, kWide);
      if (threadIdx.x == 0) {
        float* coef = a.coef + 2 * ((int64_t)b * a.groups + g);
        coef[0] = (c0 ? coef[0] : 0.f) + (float)(p / count);
        coef[1] = (c0 ? coef[1] : 0.f) + (float)(q / count);
      }
    }
    if (real && row == 0 && a.dgamma) {
      store_param(a.dbeta, a.ptype, c, (float)beta);
      store_param(a.dgamma, a.ptype, c, (float)gamma);
    }
  }
}

// The small form's dgamma and dbeta: items added in order.
__global__ __launch_bounds__(kThreads) void gn_small_params_kernel(NormArgs a) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.c) return;
  double p = 0.0, q = 0.0;
#pragma unroll 4
  for (int b = 0; b < a.n; ++b) {
    const double2 v = *reinterpret_cast<const double2*>(a.sums + ((int64_t)b * a.c + i) * 2);
    p += v.x;
    q += v.y;
  }
  store_param(a.dbeta, a.ptype, i, (float)p);
  store_param(a.dgamma, a.ptype, i, (float)q);
}

// The element-wise pass.  The chunks run from the last to the first: what the
// sums' pass read last is what the caches still hold.
template <typename T, int V, bool BACKWARD>
__global__ __launch_bounds__(kThreads) void gn_apply_kernel(NormArgs a) {
  const int b = blockIdx.y;
  const int col0 = blockIdx.z * kThreads;
  const int cols = min(a.cols - col0, kThreads), rows = kThreads / cols;
  const int col = threadIdx.x % cols, row = threadIdx.x / cols;
  if (row >= rows) return;
  const int c0 = (col0 + col) * V;
  const int64_t first = (int64_t)(gridDim.x - 1 - blockIdx.x) * a.chunk, last = min(first + a.chunk, a.s);
  const int64_t base = (int64_t)b * a.s * a.c + c0;
  const T* x = static_cast<const T*>(a.x) + base;
  T* y = static_cast<T*>(a.y) + base;
  Mean m[V];
  float gamma[V], beta[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    m[k] = a.saved[b * a.groups + (c0 + k) / a.cpg];
    gamma[k] = load_param(a.gamma, a.ptype, c0 + k);
    beta[k] = load_param(a.beta, a.ptype, c0 + k);
  }
  if constexpr (!BACKWARD) {
#pragma unroll 4
    for (int64_t r = first + row; r < last; r += rows) {
      Vec<float, V> v = load_as_float<T, V>(x + r * a.c);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float z = fmaf(gamma[k], xhat_of(v[k], m[k]), beta[k]);
        v[k] = a.silu ? silu_f(z) : z;
      }
      store_rounded<T, V>(y + r * a.c, v);
    }
  } else {
    const T* dy = static_cast<const T*>(a.dy) + base;
    float ca[V], cb[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int g = b * a.groups + (c0 + k) / a.cpg;
      ca[k] = a.coef[2 * g];
      cb[k] = a.coef[2 * g + 1];
    }
#pragma unroll 2
    for (int64_t r = first + row; r < last; r += rows) {
      Vec<float, V> v = load_as_float<T, V>(x + r * a.c);
      const Vec<float, V> g = load_as_float<T, V>(dy + r * a.c);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float xh = xhat_of(v[k], m[k]);
        const float dz = a.silu ? through_silu(g[k], fmaf(gamma[k], xh, beta[k])) : g[k];
        v[k] = m[k].rstd * (fmaf(gamma[k], dz, -ca[k]) - xh * cb[k]);
      }
      store_rounded<T, V>(y + r * a.c, v);
    }
  }
}

// The small form: blockIdx = (group, item).  A thread holds kSmallBytes of the
// vectors of one channel column, as they lie in memory.
template <typename T, int V, bool BACKWARD>
__global__ __launch_bounds__(kSmallThreads) void gn_small_kernel(NormArgs a) {
  constexpr int kVecs = kSmallBytes / (int)sizeof(T) / V;
  __shared__ double lds[BACKWARD ? 2 * V * kSmallThreads : 2 * kSmallThreads / 64];
  __shared__ float both[2];
  const int g = blockIdx.x, b = blockIdx.y;
  const int cols = a.cpg / V, rows = kSmallThreads / cols;
  const int col = threadIdx.x % cols, row = threadIdx.x / cols;
  const bool active = row < rows;
  const int c0 = g * a.cpg + col * V;
  const int64_t base = (int64_t)b * a.s * a.c + c0;
  const T* x = static_cast<const T*>(a.x) + base;
  T* y = static_cast<T*>(a.y) + base;
  Vec<T, V> held[kVecs];
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int r = row + i * rows;
    held[i] = Vec<T, V>(0);  // rows past the end add nothing to the sums
    if (active && r < a.s) held[i] = *reinterpret_cast<const Vec<T, V>*>(x + (int64_t)r * a.c);
  }
  if constexpr (!BACKWARD) {
    double p = 0.0, q = 0.0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const double d = (double)(float)held[i][k];
        p += d;
        q = fma(d, d, q);
      }
    block_sum2(p, q, lds, kSmallThreads);
    const Mean m = finish(p, q, (double)a.s * a.cpg, a.eps);
    if (threadIdx.x == 0) a.saved[b * a.groups + g] = m;
    if (!active) return;
    float gamma[V], beta[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      gamma[k] = load_param(a.gamma, a.ptype, c0 + k);
      beta[k] = load_param(a.beta, a.ptype, c0 + k);
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int r = row + i * rows;
      if (r < a.s) {
        Vec<float, V> v;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float z = fmaf(gamma[k], xhat_of((float)held[i][k], m), beta[k]);
          v[k] = a.silu ? silu_f(z) : z;
        }
        store_rounded<T, V>(y + (int64_t)r * a.c, v);
      }
    }
  } else {
    const T* dy = static_cast<const T*>(a.dy) + base;
    const Mean m = a.saved[b * a.groups + g];
    float gamma[V], beta[V];
    double acc[2 * V];
    Vec<T, V> grad[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int r = row + i * rows;
      grad[i] = Vec<T, V>(0);
      if (active && r < a.s) grad[i] = *reinterpret_cast<const Vec<T, V>*>(dy + (int64_t)r * a.c);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      gamma[k] = active ? load_param(a.gamma, a.ptype, c0 + k) : 0.f;
      beta[k] = active ? load_param(a.beta, a.ptype, c0 + k) : 0.f;
      acc[k] = acc[V + k] = 0.0;
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float xh = xhat_of((float)held[i][k], m);
        const float dv = (float)grad[i][k];
        const float dz = a.silu ? through_silu(dv, fmaf(gamma[k], xh, beta[k])) : dv;
        acc[k] += (double)dz;
        acc[V + k] = fma((double)dz, (double)xh, acc[V + k]);
      }
    reduce_rows<2 * V>(acc, lds, col, row, rows, cols, active);
    // the group's A and B: the columns' sums weighted by gamma, added in order by one thread
    __syncthreads();
    if (active && row == 0) {
      double p = 0.0, q = 0.0;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (a.sums) {
          a.sums[((int64_t)b * a.c + c0 + k) * 2] = acc[k];
          a.sums[((int64_t)b * a.c + c0 + k) * 2 + 1] = acc[V + k];
        } else if (a.dgamma) {
          store_param(a.dbeta, a.ptype, c0 + k, (float)acc[k]);
          store_param(a.dgamma, a.ptype, c0 + k, (float)acc[V + k]);
        }
        p += (double)gamma[k] * acc[k];
        q += (double)gamma[k] * acc[V + k];
      }
      lds[2 * col] = p;
      lds[2 * col + 1] = q;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      double p = 0.0, q = 0.0;
      for (int k = 0; k < cols; ++k) {
        p += lds[2 * k];
        q += lds[2 * k + 1];
      }
      const double count = (double)a.s * a.cpg;
      both[0] = (float)(p / count);
      both[1] = (float)(q / count);
    }
    __syncthreads();
    if (!active || !a.y) return;
    const float ca = both[0], cb = both[1];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int r = row + i * rows;
      if (r < a.s) {
        Vec<float, V> v;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float xh = xhat_of((float)held[i][k], m);
          const float dv = (float)grad[i][k];
          const float dz = a.silu ? through_silu(dv, fmaf(gamma[k], xh, beta[k])) : dv;
          v[k] = m.rstd * (fmaf(gamma[k], dz, -ca) - xh * cb);
        }
        store_rounded<T, V>(y + (int64_t)r * a.c, v);
      }
    }
  }
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------
// Whether a group's values fit the registers of a workgroup.  Depends on shape and
// type only: kSmallThreads / cpg rows of single values at a time are the least that
// any vector width takes.
bool small_form(int64_t s, int cpg, int elem) {
  if (cpg > kSmallThreads / 4) return false;
  const int64_t rows = kSmallThreads / cpg;  // of single values: the narrowest column
  return s <= rows * (kSmallBytes / elem_bytes(elem));
}

// Voxels of a chunk: about 1024 chunks over all items, four workgroups a CU, at least 32 KB of values each, so that a
// chunk's 16 bytes a channel of partials stay a few percent of it.  With 2048, 80x128x128 voxels of 64 channels, bf16,
// took 115 us forward where 1024 take 103, and 182 backward where 1024 take 193; 45x90x117 of 128, fp16, 88 for 74 and
// 143 for 129.
int64_t chunk_voxels(int n, int64_t s, int c, int bytes) {
  const int64_t fill = ceil_div(s * n, 1024);
  const int64_t least = std::max<int64_t>(ceil_div(32768, (int64_t)c * bytes), 64);
  return std::min(s, std::max(fill, least));
}

int norm_check(int32_t n, int64_t s, int32_t c, int32_t groups, int32_t elem, int32_t ptype) {
  if (n <= 0 || s <= 0 || c <= 0 || groups <= 0) return fail(CTMR_E_INVALID, "non-positive dimension");
  if (c % groups != 0) return fail(CTMR_E_INVALID, "channels must be divisible by groups");
  if (!valid_elem(elem) || !valid_elem(ptype)) return fail(CTMR_E_INVALID, "bad element type");
  if (n > 65535 || groups > 65535 || c > (1 << 20) || s > (1ll << 40) / c)
    return fail(CTMR_E_UNSUPPORTED, "volume too large for the group norm");
  return CTMR_OK;
}

struct NormSpace {  // byte offsets in the workspace
  int64_t part = 0, coef = 0, total = 0;
};

NormSpace norm_space(int32_t n, int64_t s, int32_t c, int32_t groups, int32_t elem, bool backward) {
  NormSpace w;
  if (small_form(s, c / groups, elem)) {
    w.total = backward && n > 1 ? (int64_t)n * c * 16 : 0;
    return w;
  }
  const int64_t chunks = ceil_div(s, chunk_voxels(n, s, c, elem_bytes(elem)));
  w.coef = (int64_t)n * chunks * c * 16;
  w.total = w.coef + (backward ? (int64_t)n * groups * 8 : 0);
  return w;
}

// The widest vector (16 bytes at most) that divides the channels it may not cross and the addresses.
int vector_width(int elem, int channels, int c, uintptr_t addresses) {
  const int bytes = elem_bytes(elem);
  for (int v = 16 / bytes; v > 1; v >>= 1)
    if (channels % v == 0 && c % v == 0 && addresses % (uintptr_t)(v * bytes) == 0) return v;
  return 1;
}

template <typename T, int V, bool BACKWARD>
int launch(NormArgs a, bool small, hipStream_t st) {
  if (small) {
    hipLaunchKernelGGL((gn_small_kernel<T, V, BACKWARD>), dim3(a.groups, a.n), dim3(kSmallThreads), 0, st, a);
    const int rc = check_launch("gn_small");
    if (rc || !BACKWARD || !a.sums || !a.dgamma) return rc;
    hipLaunchKernelGGL(gn_small_params_kernel, dim3((unsigned)ceil_div(a.c, kThreads)), dim3(kThreads), 0, st, a);
    return check_launch("gn_small_params");
  }
  a.cols = a.c / V;
  const dim3 grid(a.chunks, a.n, (unsigned)ceil_div(a.cols, kThreads));
  hipLaunchKernelGGL((gn_sums_kernel<T, V, BACKWARD>), grid, dim3(kThreads), 0, st, a);
  int rc = check_launch("gn_sums");
  if (rc) return rc;
  if constexpr (!BACKWARD)
    hipLaunchKernelGGL(gn_mean_kernel, dim3(a.groups, a.n), dim3(kWide), 0, st, a);
  else
    hipLaunchKernelGGL(gn_params_kernel, dim3(a.groups), dim3(kWide), 0, st, a);
  rc = check_launch("gn_reduce");
  if (rc || !a.y) return rc;
  hipLaunchKernelGGL((gn_apply_kernel<T, V, BACKWARD>), grid, dim3(kThreads), 0, st, a);
  return check_launch("gn_apply");
}

template <bool BACKWARD>
int dispatch(NormArgs a, int elem, hipStream_t st) {
  const bool small = small_form(a.s, a.cpg, elem);
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy;
  const int v = vector_width(elem, small ? a.cpg : a.c, a.c, at);
#define CTMR_NORM_CASE(T, W) \
  case W:                    \
    return launch<T, W, BACKWARD>(a, small, st);
  if (elem == CTMR_ELEM_F32) switch (v) {
      CTMR_NORM_CASE(float, 4) CTMR_NORM_CASE(float, 2) CTMR_NORM_CASE(float, 1)
    }
  else if (elem == CTMR_ELEM_BF16) switch (v) {
      CTMR_NORM_CASE(__bf16, 8) CTMR_NORM_CASE(__bf16, 4) CTMR_NORM_CASE(__bf16, 2) CTMR_NORM_CASE(__bf16, 1)
    }
  else switch (v) {
      CTMR_NORM_CASE(_Float16, 8) CTMR_NORM_CASE(_Float16, 4) CTMR_NORM_CASE(_Float16, 2) CTMR_NORM_CASE(_Float16, 1)
    }
#undef CTMR_NORM_CASE
  return fail(CTMR_E_INVALID, "bad element type");
}

NormArgs norm_args(int32_t n, int64_t s, int32_t c, int32_t groups, int32_t elem, int32_t ptype, int32_t silu) {
  NormArgs a = {};
  a.n = n;
  a.s = s;
  a.c = c;
  a.groups = groups;
  a.cpg = c / groups;
  a.chunk = chunk_voxels(n, s, c, elem_bytes(elem));
  a.chunks = (int)ceil_div(s, a.chunk);
  a.ptype = ptype;
  a.silu = silu != 0;
  return a;
}

int space_check(int64_t need, const void* workspace, size_t bytes) {
  if ((int64_t)bytes < need || (need > 0 && (!workspace || ((uintptr_t)workspace & 15) != 0))) {
    set_error("group-norm workspace: %zu bytes given, %lld needed on a 16-byte boundary", bytes, (long long)need);
    return CTMR_E_WORKSPACE;
  }
  return CTMR_OK;
}

}  // namespace
}  // namespace ctmr

using namespace ctmr;

extern "C" {

int64_t ctmr_norm_workspace_bytes(int32_t n, int64_t s, int32_t c, int32_t groups, int32_t elem, int32_t backward) {
  const int rc = norm_check(n, s, c, groups, elem, CTMR_ELEM_F32);
  return rc ? rc : norm_space(n, s, c, groups, elem, backward != 0).total;
}

int ctmr_norm_forward(int32_t n, int64_t s, int32_t c, int32_t groups, float eps, int32_t elem, const void* x,
                      int32_t param_elem, const void* gamma, const void* beta, int32_t silu, void* y, float* saved,
                      void* workspace, size_t workspace_bytes, void* stream) {
  int rc = norm_check(n, s, c, groups, elem, param_elem);
  if (rc) return rc;
  if (!x || !gamma || !beta || !y || !saved) return fail(CTMR_E_INVALID, "null pointer");
  if (((uintptr_t)saved & 15) != 0) return fail(CTMR_E_INVALID, "saved must be 16-byte aligned");
  rc = space_check(norm_space(n, s, c, groups, elem, false).total, workspace, workspace_bytes);
  if (rc) return rc;
  NormArgs a = norm_args(n, s, c, groups, elem, param_elem, silu);
  a.x = x;
  a.gamma = gamma;
  a.beta = beta;
  a.y = y;
  a.saved = (Mean*)saved;
  a.part = (double*)workspace;
  a.eps = eps;
  return dispatch<false>(a, elem, (hipStream_t)stream);
}

int ctmr_norm_backward(int32_t n, int64_t s, int32_t c, int32_t groups, int32_t elem, const void* x, const void* dy,
                       int32_t param_elem, const void* gamma, const void* beta, int32_t silu, const float* saved,
                       void* dx, void* dgamma, void* dbeta, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = norm_check(n, s, c, groups, elem, param_elem);
  if (rc) return rc;
  if (!x || !dy || !gamma || !beta || !saved) return fail(CTMR_E_INVALID, "null pointer");
  if ((dgamma == nullptr) != (dbeta == nullptr)) return fail(CTMR_E_INVALID, "dgamma and dbeta go together");
  if (((uintptr_t)saved & 15) != 0) return fail(CTMR_E_INVALID, "saved must be 16-byte aligned");
  const NormSpace w = norm_space(n, s, c, groups, elem, true);
  rc = space_check(w.total, workspace, workspace_bytes);
  if (rc) return rc;
  if (!dx && !dgamma) return CTMR_OK;
  NormArgs a = norm_args(n, s, c, groups, elem, param_elem, silu);
  a.x = x;
  a.dy = dy;
  a.gamma = gamma;
  a.beta = beta;
  a.y = dx;
  a.saved = (Mean*)const_cast<float*>(saved);
  a.dgamma = dgamma;
  a.dbeta = dbeta;
  char* base = (char*)workspace;
  if (small_form(s, a.cpg, elem)) {
    a.sums = n > 1 ? (double*)base : nullptr;
  } else {
    a.part = (double*)(base + w.part);
    a.coef = (float*)(base + w.coef);
  }
  return dispatch<true>(a, elem, (hipStream_t)stream);
}

}  // extern "C"
