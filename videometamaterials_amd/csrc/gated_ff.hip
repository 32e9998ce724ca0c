// Gated feed-forward product and its backward pass (the channel mixing of the recurrent load-history encoder, beside the GRU of vddp.py:546-549):
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u
//   dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dbg = sum_m dg,  dbu = sum_m du
//
// Four matrix products of 2 M K F operations in the forward and backward each but for one half: 4 M K F forward, 8 M K F backward.
#include "vmm_common.h"
#include "../../include/vmm_kernels.h"

namespace {

template <int TYPE> struct Elem;
template <> struct Elem<0> { typedef float T; static constexpr int PLANES = 3; };
template <> struct Elem<1> { typedef __bf16 T; static constexpr int PLANES = 1; };
template <> struct Elem<2> { typedef _Float16 T; static constexpr int PLANES = 1; };

template <int TYPE>
__device__ __forceinline__ f32x16 mfma(const uint4& a, const uint4& b, f32x16 c) {
  if constexpr (TYPE == 2) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vmm_f16x8, a), __builtin_bit_cast(vmm_f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vmm_bf16x8, a), __builtin_bit_cast(vmm_bf16x8, b), c, 0, 0, 0);
}

// One operand of a product: `rows` x `red` (the reduced index); value (r, k) at p[r ld + k], or p[k ld + r] where COL.
struct Operand { const void* p; long long ld, rows, red; };

// A fp32 value as three bf16 parts, x = h + m + l without a remainder: 24 bits of significand are 3 x 8.
__device__ __forceinline__ void thirds(float x, unsigned short& h, unsigned short& m, unsigned short& l) {
  const unsigned a = __float_as_uint(x) & 0xffff0000u;
  const float r = x - __uint_as_float(a);
  const unsigned b = __float_as_uint(r) & 0xffff0000u;
  const float s = r - __uint_as_float(b);
  h = a >> 16; m = b >> 16; l = __float_as_uint(s) >> 16;
}

constexpr int BM = 128, BK = 32, LDK = BK + 8;  // tile rows, reduced indexes of a step, row pitch in LDS (two-byte values)

// tile[plane][r][k] <- rows r0 .. r0 + ROWS, reduced k0 .. k0 + BK; zero outside
template <int TYPE, bool COL, int ROWS>
__device__ __forceinline__ void stage(const Operand& o, long long r0, long long k0, unsigned short* tile) {
  typedef typename Elem<TYPE>::T T;
  const T* p = (const T*)o.p;
  for (int c = threadIdx.x; c < ROWS * BK / 8; c += 256) {
    const int r = COL ? (c % (ROWS / 8)) * 8 : c / (BK / 8), k = COL ? c / (ROWS / 8) : (c % (BK / 8)) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int rr = COL ? r + j : r, kk = COL ? k : k + j;
      const long long gr = r0 + rr, gk = k0 + kk;
      const bool in = gr < o.rows && gk < o.red;
      const T v = in ? p[COL ? gk * o.ld + gr : gr * o.ld + gk] : (T)0.f;
      unsigned short* t = tile + rr * LDK + kk;
      if constexpr (TYPE == 0) thirds(v, t[0], t[ROWS * LDK], t[2 * ROWS * LDK]);
      else t[0] = __builtin_bit_cast(unsigned short, v);
    }
  }
}

// acc[mt][nt] += A-tile (rows wm ..) * B-tile (rows wn ..) over BK
template <int TYPE, int MT, int NT, int AROWS, int BROWS>
__device__ __forceinline__ void multiply(const unsigned short* ta, const unsigned short* tb, int wm, int wn, f32x16 (&acc)[MT][NT]) {
  constexpr int P = Elem<TYPE>::PLANES;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int ks = 0; ks < BK / 16; ++ks) {
    uint4 a[MT][P], b[NT][P];
    const int k = ks * 16 + (lane >> 5) * 8;
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int i = 0; i < MT; ++i) a[i][p] = *reinterpret_cast<const uint4*>(ta + (p * AROWS + wm + i * 32 + (lane & 31)) * LDK + k);
#pragma unroll
      for (int i = 0; i < NT; ++i) b[i][p] = *reinterpret_cast<const uint4*>(tb + (p * BROWS + wn + i * 32 + (lane & 31)) * LDK + k);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if constexpr (P == 3) {  // the products of the parts down to 2^-16 of the largest, small ones first; what is left out is below 2^-22
          acc[i][j] = mfma<TYPE>(a[i][2], b[j][0], acc[i][j]);
          acc[i][j] = mfma<TYPE>(a[i][0], b[j][2], acc[i][j]);
          acc[i][j] = mfma<TYPE>(a[i][1], b[j][1], acc[i][j]);
          acc[i][j] = mfma<TYPE>(a[i][1], b[j][0], acc[i][j]);
          acc[i][j] = mfma<TYPE>(a[i][0], b[j][1], acc[i][j]);
        }
        acc[i][j] = mfma<TYPE>(a[i][0], b[j][0], acc[i][j]);
      }
  }
}

__device__ __forceinline__ float act_of(float g, int act) { return act == 0 ? g / (1.0f + expf(-g)) : 0.5f * g * (1.0f + erff(g * 0.70710678118654752f)); }
__device__ __forceinline__ void act_both(float g, int act, float& a, float& slope) {
  if (act == 0) {
    const float p = 1.0f / (1.0f + expf(-g));
    a = g * p;
    slope = p * (1.0f + g * (1.0f - p));
  } else {
    const float p = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    a = g * p;
    slope = p + g * expf(-0.5f * g * g) * 0.39894228040143268f;
  }
}

// row of accumulator register r of a 32 x 32 tile (its column is the lane's lower five bits)
__device__ __forceinline__ int acc_row(int r) { return (r >> 2) * 8 + ((threadIdx.x & 63) >> 5) * 4 + (r & 3); }

// ---- forward: 128 rows x 64 columns of both projections a workgroup; each of 2 x 2 waves holds the same 64 x 32 of g and u, so that the activation and
// the product need no exchange
template <int TYPE>
__global__ __launch_bounds__(256) void ff_fwd_kernel(const vmm_gated_ff_desc d) {
  typedef typename Elem<TYPE>::T T;
  constexpr int P = Elem<TYPE>::PLANES, BF = 64;
  __shared__ __attribute__((aligned(16))) unsigned short ta[P * BM * LDK], tg[P * BF * LDK], tu[P * BF * LDK];
  const long long m0 = (long long)blockIdx.x * BM;
  const int f0 = blockIdx.y * BF;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = (wave & 1) * 64, wf = (wave >> 1) * 32;
  const Operand x = {d.x, d.ldx, d.M, d.K}, wg = {d.w_gate, d.K, d.F, d.K}, wu = {d.w_up, d.K, d.F, d.K};
  f32x16 g[2][1] = {}, u[2][1] = {};
  for (int k0 = 0; k0 < d.K; k0 += BK) {
    stage<TYPE, false, BM>(x, m0, k0, ta);
    stage<TYPE, false, BF>(wg, f0, k0, tg);
    stage<TYPE, false, BF>(wu, f0, k0, tu);
    __syncthreads();
    multiply<TYPE, 2, 1, BM, BF>(ta, tg, wm, wf, g);
    multiply<TYPE, 2, 1, BM, BF>(ta, tu, wm, wf, u);
    __syncthreads();
  }
  const int f = f0 + wf + (lane & 31);
  if (f >= d.F) return;
  const float bg = d.b_gate ? (float)((const T*)d.b_gate)[f] : 0.f, bu = d.b_up ? (float)((const T*)d.b_up)[f] : 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const long long m = m0 + wm + i * 32 + acc_row(r);
      if (m >= d.M) continue;
      const float gv = g[i][0][r] + bg, uv = u[i][0][r] + bu;
      ((T*)d.h)[m * d.ldh + f] = (T)(act_of(gv, d.act) * uv);
      if (d.g_pre) {
        d.g_pre[m * d.F + f] = gv;
        d.u_pre[m * d.F + f] = uv;
      }
    }
}

// ---- backward, first: dg and du (rounded to the type, as operands) and the partial column sums of a run of rows
constexpr int ROW_RUN = 64;
template <int TYPE>
__global__ __launch_bounds__(256) void ff_dact_kernel(const vmm_gated_ff_desc d, void* dg_, void* du_, float* __restrict__ sums) {
  typedef typename Elem<TYPE>::T T;
  const int f = blockIdx.x * 256 + threadIdx.x;
  if (f >= d.F) return;
  T* dg = (T*)dg_;
  T* du = (T*)du_;
  float sg = 0.f, su = 0.f;
  const long long m1 = min((long long)d.M, (long long)(blockIdx.y + 1) * ROW_RUN);
  for (long long m = (long long)blockIdx.y * ROW_RUN; m < m1; ++m) {
    const float dh = (float)((const T*)d.dh)[m * d.lddh + f];
    float a, slope;
    act_both(d.g_pre[m * d.F + f], d.act, a, slope);
    const float vg = dh * d.u_pre[m * d.F + f] * slope, vu = dh * a;
    dg[m * d.F + f] = (T)vg;
    du[m * d.F + f] = (T)vu;
    sg += vg;
    su += vu;
  }
  if (sums) {
    sums[(long long)blockIdx.y * 2 * d.F + f] = sg;
    sums[(long long)blockIdx.y * 2 * d.F + d.F + f] = su;
  }
}
template <int TYPE>
__global__ __launch_bounds__(256) void ff_dbias_kernel(const vmm_gated_ff_desc d, const float* __restrict__ sums, int runs) {
  typedef typename Elem<TYPE>::T T;
  const int f = blockIdx.x * 256 + threadIdx.x;
  if (f >= 2 * d.F) return;
  float s = 0.f;
  for (int r = 0; r < runs; ++r) s += sums[(long long)r * 2 * d.F + f];
  if (f < d.F) { if (d.db_gate) ((T*)d.db_gate)[f] = (T)s; }
  else if (d.db_up) ((T*)d.db_up)[f - d.F] = (T)s;
}

// ---- backward products: out[i][j] = sum over the parts and k of A(i, k) B(j, k)
struct Product { Operand a[2], b[2]; int parts; void* out[2]; long long ldo; };
template <int TYPE, bool ACOL>
__global__ __launch_bounds__(256) void ff_product_kernel(const Product p) {
  typedef typename Elem<TYPE>::T T;
  constexpr int P = Elem<TYPE>::PLANES;
  __shared__ __attribute__((aligned(16))) unsigned short ta[P * BM * LDK], tb[P * BM * LDK];
  const long long m0 = (long long)blockIdx.x * BM, n0 = (long long)blockIdx.y * BM;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
  f32x16 acc[2][2] = {};
  const int z = blockIdx.z;  // with one part, z picks the product
  for (int part = 0; part < p.parts; ++part) {
    const Operand a = p.a[z + part], b = p.b[z + part];
    for (long long k0 = 0; k0 < a.red; k0 += BK) {
      stage<TYPE, ACOL, BM>(a, m0, k0, ta);
      stage<TYPE, true, BM>(b, n0, k0, tb);
      __syncthreads();
      multiply<TYPE, 2, 2, BM, BM>(ta, tb, wm, wn, acc);
      __syncthreads();
    }
  }
  const long long M = p.a[z].rows, N = p.b[z].rows;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const long long m = m0 + wm + i * 32 + acc_row(r), n = n0 + wn + j * 32 + (lane & 31);
        if (m < M && n < N) ((T*)p.out[z])[m * p.ldo + n] = (T)acc[i][j][r];
      }
}

inline int esize(int type) { return type == 0 ? 4 : 2; }
inline long long up16(long long n) { return (n + 15) / 16 * 16; }

bool bad_ff(const vmm_gated_ff_desc* d) {
  return !d || d->M < 0 || d->K < 1 || d->F < 1 || d->M >= (1LL << 31) || d->type < 0 || d->type > 2 || d->act < 0 || d->act > 1;
}
struct Layout { long long dg, du, sums, bytes; int runs; };
Layout layout(const vmm_gated_ff_desc* d) {
  Layout l;
  l.runs = (int)((d->M + ROW_RUN - 1) / ROW_RUN);
  l.dg = 0;
  l.du = up16(d->M * d->F * esize(d->type));
  l.sums = 2 * l.du;
  l.bytes = l.sums + up16(8LL * l.runs * d->F);
  return l;
}

template <int TYPE>
int forward(const vmm_gated_ff_desc* d, hipStream_t s) {
  hipLaunchKernelGGL(ff_fwd_kernel<TYPE>, dim3(cdiv(d->M, BM), cdiv(d->F, 64)), dim3(256), 0, s, *d);
  VMM_LAUNCH_CHECK();
  return 0;
}

template <int TYPE>
int backward(const vmm_gated_ff_desc* d, hipStream_t s) {
  const Layout l = layout(d);
  char* w = (char*)d->workspace;
  const bool bias = d->db_gate || d->db_up;
  float* sums = bias ? (float*)(w + l.sums) : nullptr;
  if (d->M > 0) {
    hipLaunchKernelGGL(ff_dact_kernel<TYPE>, dim3(cdiv(d->F, 256), l.runs), dim3(256), 0, s, *d, (void*)(w + l.dg), (void*)(w + l.du), sums);
    VMM_LAUNCH_CHECK();
  }
  if (bias) {
    hipLaunchKernelGGL(ff_dbias_kernel<TYPE>, dim3(cdiv(2LL * d->F, 256)), dim3(256), 0, s, *d, (const float*)sums, l.runs);
    VMM_LAUNCH_CHECK();
  }
  if (d->dx && d->M > 0) {
    const Product p = {{{w + l.dg, d->F, d->M, d->F}, {w + l.du, d->F, d->M, d->F}}, {{d->w_gate, d->K, d->K, d->F}, {d->w_up, d->K, d->K, d->F}}, 2, {d->dx, nullptr}, d->lddx};
    hipLaunchKernelGGL((ff_product_kernel<TYPE, false>), dim3(cdiv(d->M, BM), cdiv(d->K, BM), 1), dim3(256), 0, s, p);
    VMM_LAUNCH_CHECK();
  }
  if (d->dw_gate) {
    const Operand x = {d->x, d->ldx, d->K, d->M};
    const Product p = {{{w + l.dg, d->F, d->F, d->M}, {w + l.du, d->F, d->F, d->M}}, {x, x}, 1, {d->dw_gate, d->dw_up}, d->K};
    hipLaunchKernelGGL((ff_product_kernel<TYPE, true>), dim3(cdiv(d->F, BM), cdiv(d->K, BM), 2), dim3(256), 0, s, p);
    VMM_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace

extern "C" int64_t vmm_gated_ff_workspace(const vmm_gated_ff_desc* d, int32_t backward) {
  if (bad_ff(d)) return -1;
  return backward ? layout(d).bytes : 0;
}

extern "C" int vmm_gated_ff(const vmm_gated_ff_desc* d, vmm_stream_t stream) {
  if (bad_ff(d)) return -1;
  if (d->M == 0) return 0;
  if (!d->x || !d->w_gate || !d->w_up || !d->h || !d->g_pre != !d->u_pre) return -1;
  hipStream_t s = (hipStream_t)stream;
  return d->type == 0 ? forward<0>(d, s) : d->type == 1 ? forward<1>(d, s) : forward<2>(d, s);
}

extern "C" int vmm_gated_ff_bwd(const vmm_gated_ff_desc* d, vmm_stream_t stream) {
  if (bad_ff(d)) return -1;
  if (!d->dw_gate != !d->dw_up) return -1;
  if (d->M > 0 && (!d->x || !d->w_gate || !d->w_up || !d->dh || !d->g_pre || !d->u_pre)) return -1;
  if (vmm_gated_ff_workspace(d, 1) > 0 && (!d->workspace || ((uintptr_t)d->workspace & 15))) return -1;
  hipStream_t s = (hipStream_t)stream;
  return d->type == 0 ? backward<0>(d, s) : d->type == 1 ? backward<1>(d, s) : backward<2>(d, s);
}
