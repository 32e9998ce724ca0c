// The global gradient norm over many tensors, clipping by it, and the Adam step that takes the clipped gradient (the reference's loop steps
// torch.optim.Adam without clipping, vddp.py:1481, 1629-1633; recurrent encoders are trained with it).
//
//   norm = scale * sqrt(sum_i g_i^2),   c = min(1, max_norm / (norm + 1e-6)),   g_i <- c g_i   or   Adam on  c * scale * g_i
//
// All three are bound by memory: the norm reads every gradient once (4 or 2 bytes a value), clipping in place reads and writes it -- and does neither
// where c = 1 --, the Adam step moves 28 bytes a value in fp32 and takes c from device memory, so that clipping costs it no pass of its own.
//
// Tensors come as a HOST array of jobs that travels in the kernel arguments: gradients move from step to step, and a table in device memory would need a copy at
// each (which a captured norm or clipping would replay from stale host memory; the optimizer step is not captured, and could do with one).  4 KiB of arguments hold NORM_JOBS / ADAM_JOBS tensors a launch.  The tensors of a launch
// are laid end to end in chunks of CHUNK values; every workgroup takes an equal run of chunks, so one large matrix and hundreds of short vectors
// balance alike, and the number of partial sums is bounded by the grid and not by the number of values.
//
// Sums are held in 64 bits from the first square on: 1e8 squares lose nothing, and a square of a finite fp32 value never overflows, so an infinite sum
// says that a gradient is infinite (or NaN) and nothing else.  Partial sums are written one per workgroup and added in a fixed order: no atomics,
// the same bits every time.
#include <algorithm>
#include <new>
#include <vector>
#include "vmm_common.h"
#include "../../include/vmm_kernels.h"

namespace {

constexpr int CHUNK = 4096;        // values: 256 threads x 16 values, four 16-byte loads in flight per thread in fp32
constexpr int NORM_JOBS = 176;     // 20 bytes each
constexpr int ADAM_JOBS = 80;      // 44 bytes each
constexpr int MAX_BLOCKS = 2048;   // eight workgroups of 256 threads per CU: every wave slot of the 256 CUs

struct GradTable {
  void* g[NORM_JOBS];
  unsigned long long n_type[NORM_JOBS];  // values << 2 | type
  unsigned first[NORM_JOBS];             // first chunk
  int jobs;
  unsigned chunks;
};
struct AdamTable {
  float* p[ADAM_JOBS];
  const void* g[ADAM_JOBS];
  float* m[ADAM_JOBS];
  float* v[ADAM_JOBS];
  unsigned long long n_type[ADAM_JOBS];
  unsigned first[ADAM_JOBS];
  int jobs;
  unsigned chunks;
};
static_assert(sizeof(GradTable) < 3700 && sizeof(AdamTable) < 3700, "kernel arguments are limited to 4 KiB");

// the last job whose first chunk is <= c (jobs hold one chunk at least)
template <typename T>
__device__ __forceinline__ int job_of(const T& t, unsigned c) {
  int lo = 0, hi = t.jobs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int TYPE> struct Elem;
template <> struct Elem<0> { typedef float T; static __device__ float up(T x) { return x; } static __device__ T down(float x) { return x; } };
template <> struct Elem<1> { typedef __bf16 T; static __device__ float up(T x) { return (float)x; } static __device__ T down(float x) { return (T)x; } };
template <> struct Elem<2> { typedef _Float16 T; static __device__ float up(T x) { return (float)x; } static __device__ T down(float x) { return (T)x; } };

template <typename T> struct Vec16 { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)))); };

template <int TYPE>
__device__ __forceinline__ double chunk_square_sum(const void* base, long long at, long long n) {
  typedef typename Elem<TYPE>::T T;
  const T* g = (const T*)base + at;
  const int left = (int)(n - at < CHUNK ? n - at : CHUNK);
  double s0 = 0.0, s1 = 0.0;
  constexpr int W = 16 / sizeof(T), STEP = 256 * W;
  if (((uintptr_t)g & 15) == 0 && left == CHUNK) {
    typedef typename Vec16<T>::type V;
    V r[CHUNK / STEP];
#pragma unroll
    for (int k = 0; k < CHUNK / STEP; ++k) r[k] = *reinterpret_cast<const V*>(g + k * STEP + threadIdx.x * W);
#pragma unroll
    for (int k = 0; k < CHUNK / STEP; ++k)
#pragma unroll
      for (int j = 0; j < W; j += 2) {
        const double a = (double)Elem<TYPE>::up(r[k][j]), b = (double)Elem<TYPE>::up(r[k][j + 1]);
        s0 = fma(a, a, s0);
        s1 = fma(b, b, s1);
      }
  } else {
    for (int i = threadIdx.x; i < left; i += 256) {
      const double a = (double)Elem<TYPE>::up(g[i]);
      s0 = fma(a, a, s0);
    }
  }
  return s0 + s1;
}

__device__ __forceinline__ double block_sum(double s) {
  __shared__ double part[4];
  s = wave_sum_d(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  return (part[0] + part[1]) + (part[2] + part[3]);
}

__global__ __launch_bounds__(256) void grad_square_kernel(const GradTable t, double* __restrict__ partial) {
  const unsigned c0 = (unsigned)((unsigned long long)t.chunks * blockIdx.x / gridDim.x);
  const unsigned c1 = (unsigned)((unsigned long long)t.chunks * (blockIdx.x + 1) / gridDim.x);
  double s = 0.0;
  if (c0 < c1) {
    int j = job_of(t, c0);
    for (unsigned c = c0; c < c1; ++c) {
      while (j + 1 < t.jobs && t.first[j + 1] <= c) ++j;
      const unsigned long long nt = t.n_type[j];
      const long long n = (long long)(nt >> 2), at = (long long)(c - t.first[j]) * CHUNK;
      switch (nt & 3) {
        case 0: s += chunk_square_sum<0>(t.g[j], at, n); break;
        case 1: s += chunk_square_sum<1>(t.g[j], at, n); break;
        default: s += chunk_square_sum<2>(t.g[j], at, n); break;
      }
    }
  }
  s = block_sum(s);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// out[0] = the norm of scale * g, out[1] = the factor that clips it; a non-finite sum sets the loss scaler's found_inf
__global__ __launch_bounds__(256) void grad_norm_finish_kernel(const double* __restrict__ partial, int n, float scale, float max_norm, float* __restrict__ scaler,
                                                               float* __restrict__ out) {
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 256) s += partial[i];
  s = block_sum(s);
  if (threadIdx.x == 0) {
    const double unscale = scaler ? (double)scale / (double)scaler[0] : (double)scale;
    const double norm = sqrt(s) * fabs(unscale);
    const double c = (double)max_norm / (norm + 1e-6);
    out[0] = (float)norm;
    out[1] = max_norm > 0.f ? (float)(c < 1.0 || c != c ? c : 1.0) : 1.0f;  // (a NaN norm makes a NaN factor)
    if (scaler && !(s - s == 0.0)) scaler[2] = 1.0f;
  }
}

template <int TYPE>
__device__ __forceinline__ void chunk_scale(void* base, long long at, long long n, float c) {
  typedef typename Elem<TYPE>::T T;
  T* g = (T*)base + at;
  const int left = (int)(n - at < CHUNK ? n - at : CHUNK);
  constexpr int W = 16 / sizeof(T), STEP = 256 * W;
  if (((uintptr_t)g & 15) == 0 && left == CHUNK) {
    typedef typename Vec16<T>::type V;
    V r[CHUNK / STEP];
#pragma unroll
    for (int k = 0; k < CHUNK / STEP; ++k) r[k] = *reinterpret_cast<const V*>(g + k * STEP + threadIdx.x * W);
#pragma unroll
    for (int k = 0; k < CHUNK / STEP; ++k) {
#pragma unroll
      for (int j = 0; j < W; ++j) r[k][j] = Elem<TYPE>::down(Elem<TYPE>::up(r[k][j]) * c);
      *reinterpret_cast<V*>(g + k * STEP + threadIdx.x * W) = r[k];
    }
  } else {
    for (int i = threadIdx.x; i < left; i += 256) g[i] = Elem<TYPE>::down(Elem<TYPE>::up(g[i]) * c);
  }
}

__global__ __launch_bounds__(256) void grad_clip_kernel(const GradTable t, const float* __restrict__ clip) {
  const float c = clip[1];
  if (c == 1.0f) return;  // within the bound: multiplying by one would read and write everything for nothing
  const unsigned c0 = (unsigned)((unsigned long long)t.chunks * blockIdx.x / gridDim.x);
  const unsigned c1 = (unsigned)((unsigned long long)t.chunks * (blockIdx.x + 1) / gridDim.x);
  if (c0 >= c1) return;
  int j = job_of(t, c0);
  for (unsigned k = c0; k < c1; ++k) {
    while (j + 1 < t.jobs && t.first[j + 1] <= k) ++j;
    const unsigned long long nt = t.n_type[j];
    const long long n = (long long)(nt >> 2), at = (long long)(k - t.first[j]) * CHUNK;
    switch (nt & 3) {
      case 0: chunk_scale<0>(t.g[j], at, n, c); break;
      case 1: chunk_scale<1>(t.g[j], at, n, c); break;
      default: chunk_scale<2>(t.g[j], at, n, c); break;
    }
  }
}

struct AdamScalars { float beta1, rest1, beta2, rest2, eps, step_size, bc2_sqrt, scale; };  // rest = 1 - beta, rounded once

__device__ __forceinline__ void adam_one(float& p, float g, float& m, float& v, const AdamScalars& a) {
  g *= a.scale;
  m = a.beta1 * m + a.rest1 * g;
  v = a.beta2 * v + a.rest2 * g * g;
  p = p - a.step_size * (m / (sqrtf(v) / a.bc2_sqrt + a.eps));
}

template <int TYPE>
__device__ __forceinline__ void chunk_adam(float* p, const void* base, float* m, float* v, long long at, long long n, const AdamScalars& a) {
  typedef typename Elem<TYPE>::T T;
  const T* g = (const T*)base + at;
  p += at; m += at; v += at;
  const int left = (int)(n - at < CHUNK ? n - at : CHUNK);
  typedef T G4 __attribute__((ext_vector_type(4)));
  const bool wide = ((((uintptr_t)p | (uintptr_t)m | (uintptr_t)v) & 15) | ((uintptr_t)g & (4 * sizeof(T) - 1))) == 0;
  if (wide && left == CHUNK) {
#pragma unroll 2
    for (int k = 0; k < CHUNK / 1024; ++k) {
      const int i = k * 1024 + threadIdx.x * 4;
      f32x4 pp = *reinterpret_cast<const f32x4*>(p + i), mm = *reinterpret_cast<const f32x4*>(m + i), vv = *reinterpret_cast<const f32x4*>(v + i);
      const G4 gg = *reinterpret_cast<const G4*>(g + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = pp[j], y = mm[j], z = vv[j];
        adam_one(x, Elem<TYPE>::up(gg[j]), y, z, a);
        pp[j] = x; mm[j] = y; vv[j] = z;
      }
      *reinterpret_cast<f32x4*>(m + i) = mm;
      *reinterpret_cast<f32x4*>(v + i) = vv;
      *reinterpret_cast<f32x4*>(p + i) = pp;
    }
  } else {
    for (int i = threadIdx.x; i < left; i += 256) {
      float x = p[i], y = m[i], z = v[i];
      adam_one(x, Elem<TYPE>::up(g[i]), y, z, a);
      m[i] = y; v[i] = z; p[i] = x;
    }
  }
}

__global__ __launch_bounds__(256) void adam_clipped_kernel(const AdamTable t, AdamScalars a, double lr, double beta1, double beta2,
                                                           const float* __restrict__ clip, const float* __restrict__ scaler) {
  a.scale *= clip[1];
  if (scaler) {
    if (scaler[2] != 0.f) return;  // an overflowed step: weights and moments stay as they are
    const double step = (double)scaler[4] + 1.0;  // the steps that were taken, which the host does not know
    a.step_size = (float)(lr / (1.0 - pow(beta1, step)));
    a.bc2_sqrt = (float)sqrt(1.0 - pow(beta2, step));
    a.scale /= scaler[0];
  }
  const unsigned c0 = (unsigned)((unsigned long long)t.chunks * blockIdx.x / gridDim.x);
  const unsigned c1 = (unsigned)((unsigned long long)t.chunks * (blockIdx.x + 1) / gridDim.x);
  if (c0 >= c1) return;
  int j = job_of(t, c0);
  for (unsigned k = c0; k < c1; ++k) {
    while (j + 1 < t.jobs && t.first[j + 1] <= k) ++j;
    const unsigned long long nt = t.n_type[j];
    const long long n = (long long)(nt >> 2), at = (long long)(k - t.first[j]) * CHUNK;
    switch (nt & 3) {
      case 0: chunk_adam<0>(t.p[j], t.g[j], t.m[j], t.v[j], at, n, a); break;
      case 1: chunk_adam<1>(t.p[j], t.g[j], t.m[j], t.v[j], at, n, a); break;
      default: chunk_adam<2>(t.p[j], t.g[j], t.m[j], t.v[j], at, n, a); break;
    }
  }
}

inline int elem_size(int type) { return type == 0 ? 4 : 2; }

inline bool bad_job(const void* g, int64_t n, int type) {
  return n < 0 || n > (1LL << 40) || type < 0 || type > 2 || (n > 0 && (!g || ((uintptr_t)g & (elem_size(type) - 1))));
}

inline int blocks_for(unsigned chunks) { return (int)(chunks < (unsigned)MAX_BLOCKS ? chunks : (unsigned)MAX_BLOCKS); }

// how many jobs from `i` on go into one launch: at most `most` non-empty ones, and less than 2^32 chunks
template <typename Job, typename Put>
int fill(const Job* jobs, int njobs, int i, int most, unsigned& chunks, int& used, Put put) {
  unsigned long long c = 0;
  used = 0;
  for (; i < njobs; ++i) {
    if (jobs[i].n == 0) continue;
    const unsigned long long more = (unsigned long long)(jobs[i].n + CHUNK - 1) / CHUNK;
    if (used == most || c + more > 0xffffffffull) break;
    put(used++, jobs[i], (unsigned)c);
    c += more;
  }
  chunks = (unsigned)c;
  return i;
}

int fill_grads(GradTable& t, const vmm_grad_job* jobs, int njobs, int i) {
  return fill(jobs, njobs, i, NORM_JOBS, t.chunks, t.jobs, [&](int k, const vmm_grad_job& jb, unsigned first) {
    t.g[k] = jb.g;
    t.n_type[k] = (unsigned long long)jb.n << 2 | (unsigned)jb.type;
    t.first[k] = first;
  });
}

// Ranges that are written may meet no other range of the call: a value scaled twice, or not, as the workgroups fall.  Usually they ascend already
// (slices of one buffer); only otherwise are they sorted.
struct Range { uintptr_t lo, hi; bool written; };
int overlapping(std::vector<Range>& r) {
  const auto meets = [](const std::vector<Range>& v) {
    uintptr_t any = 0, wrote = 0;  // ends of the furthest range so far, of any kind and written
    for (const Range& x : v) {
      if ((x.written && x.lo < any) || x.lo < wrote) return true;
      any = std::max(any, x.hi);
      if (x.written) wrote = std::max(wrote, x.hi);
    }
    return false;
  };
  if (!std::is_sorted(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; }))
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  return meets(r) ? 1 : 0;
}

}  // namespace

extern "C" int64_t vmm_grad_norm_workspace(const vmm_grad_job* jobs, int32_t njobs) {
  if (njobs < 0 || (njobs > 0 && !jobs)) return -1;
  for (int i = 0; i < njobs; ++i)
    if (bad_job(jobs[i].g, jobs[i].n, jobs[i].type)) return -1;
  int64_t blocks = 0;
  GradTable t;
  for (int i = 0; i < njobs;) {
    i = fill_grads(t, jobs, njobs, i);
    blocks += blocks_for(t.chunks);
  }
  return 8 * std::max<int64_t>(blocks, 1);
}

extern "C" int vmm_grad_norm(const vmm_grad_job* jobs, int32_t njobs, float scale, float max_norm, float* scaler_state, void* workspace, float* out,
                             vmm_stream_t stream) {
  if (njobs < 0 || (njobs > 0 && !jobs) || !workspace || ((uintptr_t)workspace & 7) || !out) return -1;
  for (int i = 0; i < njobs; ++i)
    if (bad_job(jobs[i].g, jobs[i].n, jobs[i].type)) return -1;
  double* partial = (double*)workspace;
  int64_t n = 0;
  GradTable t;
  for (int i = 0; i < njobs;) {
    i = fill_grads(t, jobs, njobs, i);
    const int blocks = blocks_for(t.chunks);
    if (!blocks) continue;
    hipLaunchKernelGGL(grad_square_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, t, partial + n);
    VMM_LAUNCH_CHECK();
    n += blocks;
  }
  hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, partial, (int)n, scale, max_norm, scaler_state, out);
  VMM_LAUNCH_CHECK();
  return 0;
}

extern "C" int vmm_grad_clip(const vmm_grad_job* jobs, int32_t njobs, const float* clip, vmm_stream_t stream) {
  if (njobs < 0 || (njobs > 0 && !jobs) || !clip) return -1;
  try {
    std::vector<Range> r;
    r.reserve(njobs);
    for (int i = 0; i < njobs; ++i) {
      if (bad_job(jobs[i].g, jobs[i].n, jobs[i].type)) return -1;
      const uintptr_t lo = (uintptr_t)jobs[i].g;
      if (jobs[i].n) r.push_back({lo, lo + (uintptr_t)jobs[i].n * elem_size(jobs[i].type), true});
    }
    if (overlapping(r)) return -2;
  } catch (const std::bad_alloc&) {
    return -12;
  }
  GradTable t;
  for (int i = 0; i < njobs;) {
    i = fill_grads(t, jobs, njobs, i);
    if (!t.chunks) continue;
    hipLaunchKernelGGL(grad_clip_kernel, dim3(blocks_for(t.chunks)), dim3(256), 0, (hipStream_t)stream, t, clip);
    VMM_LAUNCH_CHECK();
  }
  return 0;
}

extern "C" int vmm_adam_step_clipped(const vmm_clip_adam_job* jobs, int32_t njobs, double lr, double beta1, double beta2, double eps, int64_t step,
                                     float grad_scale, const float* clip, const float* scaler_state, vmm_stream_t stream) {
  if (njobs < 0 || (njobs > 0 && !jobs) || !clip || (!scaler_state && step < 1)) return -1;
  try {
    std::vector<Range> r;
    r.reserve(4 * (size_t)njobs);
    for (int k = 0; k < 4; ++k)  // list by list: each usually ascends
      for (int i = 0; i < njobs; ++i) {
        const vmm_clip_adam_job& jb = jobs[i];
        if (k == 0 && (bad_job(jb.g, jb.n, jb.type) || (jb.n > 0 && (!jb.p || !jb.m || !jb.v || (((uintptr_t)jb.p | (uintptr_t)jb.m | (uintptr_t)jb.v) & 3))))) return -1;
        if (!jb.n) continue;
        const uintptr_t lo = k == 0 ? (uintptr_t)jb.p : k == 1 ? (uintptr_t)jb.m : k == 2 ? (uintptr_t)jb.v : (uintptr_t)jb.g;
        r.push_back({lo, lo + (uintptr_t)jb.n * (k == 3 ? elem_size(jb.type) : 4), k != 3});
      }
    if (overlapping(r)) return -2;
  } catch (const std::bad_alloc&) {
    return -12;
  }
  // (1 - beta in 64 bits: 1 - 0.999f is off by 1e-5 of itself)
  AdamScalars a = {(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, 0.f, 1.f, grad_scale};
  if (!scaler_state) {
    a.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
    a.bc2_sqrt = (float)sqrt(1.0 - pow(beta2, (double)step));
  }
  AdamTable t;
  for (int i = 0; i < njobs;) {
    i = fill(jobs, njobs, i, ADAM_JOBS, t.chunks, t.jobs, [&](int k, const vmm_clip_adam_job& jb, unsigned first) {
      t.p[k] = jb.p; t.g[k] = jb.g; t.m[k] = jb.m; t.v[k] = jb.v;
      t.n_type[k] = (unsigned long long)jb.n << 2 | (unsigned)jb.type;
      t.first[k] = first;
    });
    if (!t.chunks) continue;
    hipLaunchKernelGGL(adam_clipped_kernel, dim3(blocks_for(t.chunks)), dim3(256), 0, (hipStream_t)stream, t, a, lr, beta1, beta2, clip, scaler_state);
    VMM_LAUNCH_CHECK();
  }
  return 0;
}
