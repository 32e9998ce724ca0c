// Gated feed-forward product and its backward pass (the channel mixing of the recurrent load-history encoder, beside the GRU of vddp.py:546-549):
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u
//   dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dbg = sum_m dg,  dbu = sum_m du
//
// Matrix products bound it: 4 M K F operations forward, 8 M K F backward.  All of them are one kernel, out(i, j) = sum_k A(i, k) B(j, k) over 16-bit
// operands with fp32 sums, whose operands may be stored with either index contiguous; a product may be the sum of several parts.
//   forward   A = x, B = rows of Wg and Wu side by side in one tile: a wave holds the same places of g and u, so activation and product need no exchange
//   dx        A = dg, B = Wg (stored [k][j]), then the part of du and Wu
//   dW        A = dg (stored [k][i]), B = x (stored [k][j]);  gate and up side by side in the grid
// fp32 operands are split into three bf16 parts without a remainder (24 = 3 x 8 bits), each rounded to nearest, so the second is below 2^-8 and the third below 2^-17
// of the value's power of two; a product is the sum of the six products of parts that reach 2^-17 of it, small ones first.  What is left out, second times third
// both ways, is below 2^-24 and of either sign (the matrix unit itself floors an accumulator that is smaller than a product to the sum's last place).
// The last bit of a value from 2^-110 on is 2^-133 at the least, the smallest bf16 number; smaller values are rounded to a multiple of it.  That is six matrix passes at 16 times the rate of fp32 ones.
//
// A tile step is 64 reduced indexes.  It goes from memory to LDS directly (buffer loads with an LDS destination: no registers, and what lies
// outside the operand arrives as zero), into the one of two buffers that the matrix instructions do not read.  Such a load fills 1 KiB of LDS in lane order,
// so the banks are spread by which 16 bytes each lane FETCHES: row-contiguous operands swap 16-byte pieces by bits 1..3 of the row (16 lanes read 16
// rows at once, and rows two apart start at the same bank), column-contiguous ones by the lower two bits of k (read back with the transposing 8-byte reads).
#include <algorithm>
#include "vmm_common.h"
#include "../../include/vmm_kernels.h"

namespace {

typedef unsigned short u16;
typedef __attribute__((address_space(3))) void lds_void;

template <int TYPE> struct Elem;
template <> struct Elem<0> { typedef float T; static constexpr int PLANES = 3; };
template <> struct Elem<1> { typedef __bf16 T; static constexpr int PLANES = 1; };
template <> struct Elem<2> { typedef _Float16 T; static constexpr int PLANES = 1; };

template <bool HALF>
__device__ __forceinline__ f32x16 mfma(const uint4& a, const uint4& b, f32x16 c) {
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(vmm_f16x8, a), __builtin_bit_cast(vmm_f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(vmm_bf16x8, a), __builtin_bit_cast(vmm_bf16x8, b), c, 0, 0, 0);
}

constexpr int BK = 64;          // reduced indexes of a step
constexpr int MAX_PARTS = 12;   // dx in fp32: two products of six parts

// One product (or two of one shape, dWg and dWu).  A: rows x red, B: cols x red; strides in values, multiples of 8 at 16-byte aligned addresses.
struct Gemm {
  const u16* a[MAX_PARTS];
  const u16* b[MAX_PARTS];
  const u16* b2[6];                 // forward: the parts of Wu
  long long lda, ldb, rows, cols, red;
  int parts, splits;                // the reduced length (of all parts) is cut into `splits` runs
  long long tiles_m, tiles_n;
  void* out[2]; long long ldo;      // one run
  bool pairs;                       // rows of `out` and their length are even: results of 16 bits can leave in pairs
  float* partial;                   // several: [product][run][rows][cols], forward [run][2][rows][cols]
  // forward
  const void* b_gate; const void* b_up; float* g_pre; float* u_pre; int act;
};

// a value that is the same in every lane, in a scalar register: integer divisions leave theirs in vector registers, and a buffer descriptor made from
// such values would be re-read lane by lane
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const u16* uniform(const u16* p) {
  const unsigned long long v = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
  return (const u16*)((unsigned long long)hi << 32 | lo);
}

// e^-m, m >= 0.  In 16 bits the hardware's 2^p of the rounded p = -m log2(e) does; fp32 corrects for what the rounding has lost, up to m 2^-25 of the result.
template <int TYPE>
__device__ __forceinline__ float exp_minus(float m) {
  if constexpr (TYPE == 0) {
    m = m > 104.f ? 104.f : m;  // (zero from there on; an infinite one would leave inf - inf below)
    const float p = m * -1.44269502162933349609375f;
    float t = fmaf(m, -1.44269502162933349609375f, -p);
    t = fmaf(m, -1.925963033500011e-08f, t);
    const float e = __builtin_amdgcn_exp2f(p);
    return fmaf(e, t * 0.6931471805599453f, e);
  } else {
    return __builtin_amdgcn_exp2f(m * -1.44269502162933349609375f);
  }
}
// The activation's factor P (a = g P) and its derivative P + g P'.
//   silu: P = sigmoid(g) from e^-|g|, P' = P (1 - P)
//   gelu: P = Phi(g), the normal distribution: Phi(-|g|) = e^(-g^2/2) erfcx(|g| / sqrt 2) / 2, whose last two factors are a polynomial in
//         t = 1 / (1 + |g| / sqrt 8), fitted for the least relative error over |g| <= 13.4 (5.4e-8 with its coefficients in fp32; 3.2e-7 as evaluated); P' = e^(-g^2/2) / sqrt(2 pi)
// (erff and the exact division took half of the epilogue: 512 x 256 x 128 values, 13 us a tile)
template <int TYPE, int ACT, bool SLOPE>
__device__ __forceinline__ float act_parts(float g, float& slope) {
  const float m = fabsf(g);
  if constexpr (ACT == 0) {
    const float e = exp_minus<TYPE>(m), r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r, p = g < 0.f ? er : r;
    if constexpr (SLOPE) slope = p * fmaf(g, g < 0.f ? r : er, 1.0f);
    return g * p;
  } else {
    const float t = __builtin_amdgcn_rcpf(fmaf(m, 0.35355339059327376f, 1.0f)), e = exp_minus<TYPE>(0.5f * g * g);
    float q = -0.029445331543684006f;
    q = fmaf(q, t, 0.14185069501399994f);
    q = fmaf(q, t, -0.2426912486553192f);
    q = fmaf(q, t, 0.1379883736371994f);
    q = fmaf(q, t, -0.012588338926434517f);
    q = fmaf(q, t, 0.10103470087051392f);
    q = fmaf(q, t, 0.12163055688142776f);
    q = fmaf(q, t, 0.1411767303943634f);
    q = fmaf(q, t, 0.14104384183883667f);
    q *= t * e;
    const float p = g < 0.f ? q : 1.0f - q;
    if constexpr (SLOPE) slope = fmaf(g * e, 0.3989422804014327f, p);
    return g * p;
  }
}
template <int TYPE, int ACT>
__device__ __forceinline__ float act_of(float g) {
  float slope;
  return act_parts<TYPE, ACT, false>(g, slope);
}

// row of accumulator register r of a 32 x 32 tile (its column is the lane's lower five bits)
__device__ __forceinline__ int acc_row(int r) { return (r >> 2) * 8 + ((threadIdx.x & 63) >> 5) * 4 + (r & 3); }

// A 32 x 32 tile of results to rows of T from row m, column n on (the same for all lanes: the address of a row is, and the lane's part is 32 bits).
// One value after the other (the empty asm): computed side by side they would need more registers than there are and the steps' loop would spill.
// PAIRS: even rows and columns, so that lanes exchange a value for each two and 16-bit results leave two at a time.
template <typename T, typename F>
__device__ __forceinline__ void put_tile(T* out, long long ldo, long long rows, long long cols, long long m, long long n, bool pairs, F value) {
  const int lane = threadIdx.x & 63, col = lane & 31, row0 = (lane >> 5) * 4;
  const int rows_left = (int)min(rows - m, 32LL) - row0, cols_left = (int)min(cols - n, 32LL);
  char* base = (char*)(out + m * ldo + n);
  const long long pitch = ldo * (long long)sizeof(T);
  if constexpr (sizeof(T) == 2) {
    if (pairs) {
      typedef T T2 __attribute__((ext_vector_type(2)));
      typedef float f32x2_t __attribute__((ext_vector_type(2)));
      const int odd = col & 1;
      const unsigned off = (unsigned)((row0 + odd) * (int)pitch) + (col & ~1) * 2;
      if (col < cols_left) {
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          float v0 = value(r), v1 = value(r + 1);
          asm volatile("" : "+v"(v0), "+v"(v1)::"memory");
          const float other = lane_xor(odd ? v0 : v1, 0);
          const f32x2_t v = {odd ? other : v0, odd ? v1 : other};
          const int at = (r >> 2) * 8 + (r & 3);
          if (at + odd < rows_left) *reinterpret_cast<T2*>(base + at * pitch + off) = __builtin_convertvector(v, T2);
        }
      }
      return;
    }
  }
  const unsigned off = (unsigned)(row0 * (int)pitch) + col * (unsigned)sizeof(T);
  if (col < cols_left) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int at = (r >> 2) * 8 + (r & 3);
      float v = value(r);
      asm volatile("" : "+v"(v)::"memory");
      if (at < rows_left) *reinterpret_cast<T*>(base + at * pitch + off) = (T)v;
    }
  }
}

// ---- one operand's tile of R rows.  Every wave issues R / 8 / WAVES loads of 1 KiB.
template <bool COL, int R, int WAVES>
struct Loader {
  static constexpr int LOADS = R / 8 / WAVES;
  static_assert(LOADS % 2 == 0, "a wave's loads start at an even row of pieces");
  unsigned off[LOADS];  // byte offset of this lane's 16 bytes from the tile's first value
  int kc;               // row-contiguous: first k of the lane's piece in even loads; in odd ones it is 32 away
  long long ld, left;
  // r0: first row of the tile of the `rows`; FOLD: rows 32..63 of every 64 are rows 0..31 of the same 32 in a second matrix
  template <bool FOLD>
  __device__ __forceinline__ void init(long long r0, long long rows, long long ld_) {
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    ld = ld_;
    left = rows - r0;
    kc = ((lane & 7) ^ (lane >> 4)) * 8;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int piece = (wave * LOADS + i) * 64 + lane;  // of 16 bytes, in LDS order
      if constexpr (COL) {
        const int k = piece / (R / 8), c = (piece % (R / 8)) ^ ((k & 3) << 2);
        off[i] = c * 8 < left ? (unsigned)(k * ld * 2 + c * 16) : 0xfffffff0u;
      } else {
        int r = piece / 8;
        if constexpr (FOLD) r = (r >> 6) * 32 + (r & 31);
        off[i] = r < left ? (unsigned)(r * ld * 2 + (kc ^ (i & 1) * 32) * 2) : 0xfffffff0u;
      }
    }
  }
  // p: the tile's first value; k0: reduced index of the step, of `red`
  __device__ __forceinline__ void load(const u16* p, long long k0, long long red, u16* tile, int i) const {
    const long long rest = red - k0;
    const u16* base = p + (COL ? k0 * ld : k0);
    const unsigned size = COL ? (unsigned)((rest < BK ? rest : BK) * ld * 2) : 0xfffffff0u;  // (rows outside have an offset that no size reaches)
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<u16*>(base), 0, (int)size, 0x00027000);
    const int wave = uniform(threadIdx.x >> 6);
    unsigned o = off[i];
    if (!COL && (kc ^ (i & 1) * 32) >= rest) o = 0xfffffff0u;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(tile + (wave * LOADS + i) * 512), 16, o, 0, 0, 0);
  }
};

// fragment of 32 rows from r0 on, reduced indexes ks * 16 ..
template <bool COL, int R>
__device__ __forceinline__ uint4 fragment(const u16* tile, int r0, int ks) {
  const int lane = threadIdx.x & 63;
  if constexpr (COL) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    const int i = lane & 15, k = ks * 16 + (lane >> 5) * 8 + (i >> 2), r = r0 + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
    const u16* at = tile + k * R + (((r >> 3) ^ ((i >> 2) << 2)) << 3) + (r & 7);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 4 * R));
    const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
    return make_uint4(l.x, l.y, h.x, h.y);
  } else {
    const int r = r0 + (lane & 31), c = (ks * 2 + (lane >> 5)) ^ ((r >> 1) & 7);
    return *reinterpret_cast<const uint4*>(tile + r * BK + c * 8);
  }
}

// ---- out = A B^T.  BIG: 256 x 256 tiles, 8 waves of 128 x 64; else 128 x 128 tiles, 4 waves of 64 x 64.
template <int TYPE, bool ACOL, bool BCOL, bool GATED, bool BIG>
__global__ __launch_bounds__(BIG ? 512 : 256, BIG ? 2 : 2) void ff_gemm_kernel(const Gemm q) {
  typedef typename Elem<TYPE>::T T;
  constexpr bool HALF = TYPE == 2;
  constexpr int R = BIG ? 256 : 128, WAVES = BIG ? 8 : 4, WM = BIG ? 128 : 64, MT = WM / 32;
  __shared__ __attribute__((aligned(16))) u16 a0[R * BK], b0[R * BK], a1[R * BK], b1[R * BK];
  // Consecutive workgroups go to different XCDs: each XCD gets a run of tiles that are neighbours, 8 rows of tiles at a time, and finds its operands
  // in its own L2.
  const unsigned tiles = (unsigned)(q.tiles_m * q.tiles_n), per = (tiles + 7) / 8, t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (t >= tiles) return;
  const unsigned in_all = 8 * (unsigned)q.tiles_n, band = t / in_all, bm = min(8u, (unsigned)q.tiles_m - band * 8), in_band = t - band * in_all;
  long long m0 = (long long)uniform(band * 8 + in_band % bm) * R, n0 = (long long)uniform(in_band / bm) * (GATED ? R / 2 : R);
  const int run = uniform(blockIdx.y % q.splits), prod = uniform(blockIdx.y / q.splits);
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = BIG ? (wave & 1) * 128 : (wave & 1) * 64, wn = (wave >> 1) * 64;

  Loader<ACOL, R, WAVES> la;
  Loader<BCOL, R, WAVES> lb;
  la.template init<false>(m0, q.rows, q.lda);
  lb.template init<GATED>(n0, q.cols, q.ldb);
  const int steps = (int)((q.red + BK - 1) / BK), units = steps * q.parts;
  const int u0 = uniform((int)((long long)units * run / q.splits)), u1 = uniform((int)((long long)units * (run + 1) / q.splits));
  int part = uniform(u0 / max(steps, 1)), step = u0 - part * steps;
  const long long ao = ACOL ? m0 : m0 * q.lda, bo = BCOL ? n0 : n0 * q.ldb;
  auto fetch = [&](u16* ta, u16* tb) {
    const u16* pa = q.a[prod * q.parts + part] + ao;
    const u16* pb = q.b[prod * q.parts + part] + bo;
    const long long k0 = (long long)step * BK;
#pragma unroll
    for (int i = 0; i < la.LOADS; ++i) la.load(pa, k0, q.red, ta, i);
#pragma unroll
    for (int i = 0; i < lb.LOADS; ++i) {
      const u16* p = pb;
      if constexpr (GATED) {
        const int row = (wave * lb.LOADS + i) * 8;  // of the tile: eight rows a load
        if (row & 32) p = q.b2[part] + bo;
      }
      lb.load(p, k0, q.red, tb, i);
    }
    if (++step == steps) { step = 0; ++part; }
  };
  f32x16 acc[MT][2] = {};
  auto compute = [&](const u16* ta, const u16* tb) {
#pragma unroll
    for (int ks = 0; ks < BK / 16; ++ks) {
      uint4 a[MT], b[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) b[j] = fragment<BCOL, R>(tb, wn + j * 32, ks);
#pragma unroll
      for (int i = 0; i < MT; ++i) a[i] = fragment<ACOL, R>(ta, wm + i * 32, ks);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma<HALF>(a[i], b[j], acc[i][j]);
    }
  };
  // At each barrier this wave's loads of the step have landed, and every wave's behind it; nobody reads the other buffer any more.
  int u = u0;
  if (u < u1) fetch(a0, b0);
  for (; u + 1 < u1; u += 2) {
    __syncthreads();
    fetch(a1, b1);
    compute(a0, b0);
    __syncthreads();
    if (u + 2 < u1) fetch(a0, b0);
    compute(a1, b1);
  }
  if (u < u1) {
    __syncthreads();
    compute(a0, b0);
  }

  // (what follows starts from values that exist only here: worked out ahead of the steps, its addresses would take the registers of the operands)
  int here = 0;
  asm volatile("" : "+s"(here));
  m0 += here;
  n0 += here;
  if constexpr (GATED) {
    const long long fn = n0 + wn / 2, f = fn + (lane & 31);
    if (q.splits > 1) {
      float* pg = q.partial + (long long)run * 2 * q.rows * q.cols;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          put_tile(pg + j * q.rows * q.cols, q.cols, q.rows, q.cols, m0 + wm + i * 32, fn, false, [&](int r) { return acc[i][j][r]; });
      return;
    }
    const float bg = q.b_gate && f < q.cols ? (float)((const T*)q.b_gate)[f] : 0.f, bu = q.b_up && f < q.cols ? (float)((const T*)q.b_up)[f] : 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (q.g_pre) {
        put_tile(q.g_pre, q.cols, q.rows, q.cols, m0 + wm + i * 32, fn, false, [&](int r) { return acc[i][0][r] + bg; });
        put_tile(q.u_pre, q.cols, q.rows, q.cols, m0 + wm + i * 32, fn, false, [&](int r) { return acc[i][1][r] + bu; });
      }
      T* h = (T*)q.out[0];
      if (q.act == 0) put_tile(h, q.ldo, q.rows, q.cols, m0 + wm + i * 32, fn, q.pairs, [&](int r) { return act_of<TYPE, 0>(acc[i][0][r] + bg) * (acc[i][1][r] + bu); });
      else put_tile(h, q.ldo, q.rows, q.cols, m0 + wm + i * 32, fn, q.pairs, [&](int r) { return act_of<TYPE, 1>(acc[i][0][r] + bg) * (acc[i][1][r] + bu); });
    }
  } else {
    float* part_out = q.partial + (long long)blockIdx.y * q.rows * q.cols;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (q.splits > 1) put_tile(part_out, q.cols, q.rows, q.cols, m0 + wm + i * 32, n0 + wn + j * 32, false, [&](int r) { return acc[i][j][r]; });
        else put_tile((T*)q.out[prod], q.ldo, q.rows, q.cols, m0 + wm + i * 32, n0 + wn + j * 32, q.pairs, [&](int r) { return acc[i][j][r]; });
      }
  }
}

// ---- the runs of a split product, added in order
template <int TYPE>
__global__ __launch_bounds__(256) void ff_join_kernel(const Gemm q) {
  typedef typename Elem<TYPE>::T T;
  const long long n = q.rows * q.cols, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const float* p = q.partial + (long long)blockIdx.y * q.splits * n + i;
  float s = 0.f;
  for (int r = 0; r < q.splits; ++r) s += p[r * n];
  ((T*)q.out[blockIdx.y])[i / q.cols * q.ldo + i % q.cols] = (T)s;
}
template <int TYPE>
__global__ __launch_bounds__(256) void ff_join_gated_kernel(const Gemm q) {
  typedef typename Elem<TYPE>::T T;
  const long long n = q.rows * q.cols, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long long m = i / q.cols, f = i % q.cols;
  float g = 0.f, u = 0.f;
  for (int r = 0; r < q.splits; ++r) {
    g += q.partial[2 * r * n + i];
    u += q.partial[(2 * r + 1) * n + i];
  }
  g += q.b_gate ? (float)((const T*)q.b_gate)[f] : 0.f;
  u += q.b_up ? (float)((const T*)q.b_up)[f] : 0.f;
  ((T*)q.out[0])[m * q.ldo + f] = (T)((q.act == 0 ? act_of<TYPE, 0>(g) : act_of<TYPE, 1>(g)) * u);
  if (q.g_pre) { q.g_pre[i] = g; q.u_pre[i] = u; }
}

// ---- operands: three bf16 parts of fp32 values, or 16-bit values whose rows are not made of whole 16-byte pieces, laid out with padded rows
struct Layin { const void* src[3]; u16* dst[3]; long long rows[3], ld[3]; int cols, pitch; };

__device__ __forceinline__ unsigned near16(float x) { return (unsigned)__builtin_bit_cast(u16, (__bf16)x) << 16; }  // bits of the nearest bf16 as fp32
__device__ __forceinline__ void thirds(float x, u16& h, u16& m, u16& l) {
  unsigned a = near16(x);
  if ((a & 0x7fffffffu) == 0x7f800000u) a = __float_as_uint(x) & 0xffff0000u;  // (a finite value next to the largest is cut: rounded up it would be infinite)
  const float r = x - __uint_as_float(a);
  const unsigned b = near16(r);
  const float s = r - __uint_as_float(b);
  h = a >> 16; m = b >> 16; l = near16(s) >> 16;
}
template <int TYPE>
__device__ __forceinline__ void put(u16* p, long long plane, float v) {
  if constexpr (TYPE == 0) thirds(v, p[0], p[plane], p[2 * plane]);
  else *p = __builtin_bit_cast(u16, (typename Elem<TYPE>::T)v);
}

template <int TYPE>
__global__ __launch_bounds__(256) void ff_layin_kernel(const Layin a) {
  typedef typename Elem<TYPE>::T T;
  const int z = blockIdx.y;
  const long long n = a.rows[z] * a.pitch;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long r = i / a.pitch;
    const int c = (int)(i - r * a.pitch);
    const T v = c < a.cols ? ((const T*)a.src[z])[r * a.ld[z] + c] : (T)0.f;
    put<TYPE>(a.dst[z] + i, n, (float)v);
  }
}

// ---- backward, first: dg and du as operands (rounded to the type, or split) and the column sums of a run of rows.  64 lanes of 4 columns x 4 rows.
// In 16 bits dg and du have one rounding before the products, as any 16-bit operand has, so dx and dW are off by two roundings, this one and their own: sqrt 2
// times the error of their own alone (2.9e-4 against 2.1e-4 in fp16, 2.3e-3 against 1.7e-3 in bf16, of the result's norm).  Two parts of each would be without
// it and cost the backward's matrix work a second time (8 M K F of the 12 M K F operations of a training pass).
template <int TYPE, bool WIDE>
__global__ __launch_bounds__(256) void ff_dact_kernel(const vmm_gated_ff_desc d, u16* dg, u16* du, int pitch, int run, float* __restrict__ sums) {
  typedef typename Elem<TYPE>::T T;
  typedef T T4 __attribute__((ext_vector_type(4)));
  typedef u16 U4 __attribute__((ext_vector_type(4)));
  __shared__ float part[4][2][256];
  const int lane = threadIdx.x & 63, row = threadIdx.x >> 6, f = (blockIdx.x * 64 + lane) * 4;
  const long long plane = d.M * pitch, m1 = min((long long)d.M, (long long)(blockIdx.y + 1) * run);
  float sg[4] = {}, su[4] = {};
  if (f < pitch) {
#pragma unroll 4
    for (long long m = (long long)blockIdx.y * run + row; m < m1; m += 4) {
      float g[4], u[4], dh[4];
      const T* hp = (const T*)d.dh + m * d.lddh + f;
      const float *gp = d.g_pre + m * d.F + f, *up = d.u_pre + m * d.F + f;
      if constexpr (WIDE) {
        T4 hv = {};
        f32x4 gv = {}, uv = {};
        if (f < d.F) {
          hv = *reinterpret_cast<const T4*>(hp);
          gv = *reinterpret_cast<const f32x4*>(gp);
          uv = *reinterpret_cast<const f32x4*>(up);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) { dh[j] = (float)hv[j]; g[j] = gv[j]; u[j] = uv[j]; }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool in = f + j < d.F;
          dh[j] = in ? (float)hp[j] : 0.f;
          g[j] = in ? gp[j] : 0.f;
          u[j] = in ? up[j] : 0.f;
        }
      }
      u16 og[3][4], ou[3][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a, slope;
        if (d.act == 0) a = act_parts<TYPE, 0, true>(g[j], slope);
        else a = act_parts<TYPE, 1, true>(g[j], slope);
        const float vg = dh[j] * u[j] * slope, vu = dh[j] * a;
        sg[j] += vg;
        su[j] += vu;
        put<TYPE>(&og[0][j], 4, vg);
        put<TYPE>(&ou[0][j], 4, vu);
      }
#pragma unroll
      for (int p = 0; p < Elem<TYPE>::PLANES; ++p) {
        *reinterpret_cast<U4*>(dg + p * plane + m * pitch + f) = U4{og[p][0], og[p][1], og[p][2], og[p][3]};
        *reinterpret_cast<U4*>(du + p * plane + m * pitch + f) = U4{ou[p][0], ou[p][1], ou[p][2], ou[p][3]};
      }
    }
  }
  if (!sums) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    part[row][0][lane * 4 + j] = sg[j];
    part[row][1][lane * 4 + j] = su[j];
  }
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < d.F) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      sums[((long long)blockIdx.y * 2 + k) * d.F + c] = (part[0][k][threadIdx.x] + part[1][k][threadIdx.x]) + (part[2][k][threadIdx.x] + part[3][k][threadIdx.x]);
  }
}
// 32 columns x 8 lanes that share the runs
template <int TYPE>
__global__ __launch_bounds__(256) void ff_dbias_kernel(const vmm_gated_ff_desc d, const float* __restrict__ sums, int runs) {
  typedef typename Elem<TYPE>::T T;
  __shared__ float part[8][32];
  const int col = threadIdx.x & 31, share = threadIdx.x >> 5;
  const long long f = (long long)blockIdx.x * 32 + col;
  float s = 0.f;
  if (f < 2LL * d.F) {
#pragma unroll 4
    for (int r = share; r < runs; r += 8) s += sums[(long long)r * 2 * d.F + f];
  }
  part[share][col] = s;
  __syncthreads();
  if (share == 0 && f < 2LL * d.F) {
    for (int k = 1; k < 8; ++k) s += part[k][col];
    if (f < d.F) { if (d.db_gate) ((T*)d.db_gate)[f] = (T)s; }
    else if (d.db_up) ((T*)d.db_up)[f - d.F] = (T)s;
  }
}

// ---- host side

inline int esize(int type) { return type == 0 ? 4 : 2; }
inline long long up(long long n, long long to) { return (n + to - 1) / to * to; }

inline long long cdiv64(long long a, long long b) { return (a + b - 1) / b; }
bool bad_ld(int64_t ld) { return ld < 0 || ld >= (1 << 22); }
bool bad_ff(const vmm_gated_ff_desc* d) {
  // (K, F < 2^22: a tile of 256 rows is addressed with 32-bit byte offsets)
  if (!d || d->M < 0 || d->K < 1 || d->F < 1 || d->K >= (1 << 22) || d->F >= (1 << 22) || d->M >= (1LL << 31) || d->type < 0 || d->type > 2 || d->act < 0 ||
      d->act > 1 || bad_ld(d->ldx) || bad_ld(d->ldh) || bad_ld(d->lddh) || bad_ld(d->lddx))
    return true;
  const auto too_many = [](long long rows, long long cols) { return cdiv64(rows, 256) * cdiv64(cols, 256) >= (1LL << 23) - 8; };  // a launch has less than 2^32 threads
  return too_many(d->M, 2LL * d->F) || too_many(d->M, d->K) || too_many(d->F, d->K);
}

// The tiles and runs of a product.  Big tiles read LDS 0.75 times per matrix instruction slot where small ones read it as often as it can be read; they
// are taken where they fill the card (M x K x F of 8192 x 2048 x 8192, bf16, keeping the products: 590 us, small 759; the weight gradients of 1024 x 1024 x
// 4096, 128 big tiles: 61 us, small 33).  Products whose tiles do not put two workgroups on every CU are cut along their reduced length, by four steps a
// run at the least (4 x 1024 x 4096 forward: 10.5 us, whole 16.7; dx of 3996 x 1000 x 4096: 136 with the activation's 46, whole 173; a sum that is
// short for its size loses the time of the join: the weight gradients of 2048 x 1024 x 2048 46, whole 41).
struct Shape { bool big; int splits; };
Shape shape_of(long long rows, long long cols, bool gated, long long units, int products) {
  const auto tiles = [&](long long r) { return std::max(cdiv64(rows, r) * cdiv64(cols * (gated ? 2 : 1), r) * products, 1LL); };  // (no rows: nothing is launched)
  Shape s;
  s.big = tiles(256) >= 192;
  const long long t = tiles(s.big ? 256 : 128) * (s.big ? 2 : 1);
  long long n = 1;
  if (t < 512) n = (512 + t / 2) / t;
  if (n > units / 4) n = units / 4;
  if (n > 64) n = 64;
  s.splits = (int)(n < 1 ? 1 : n);
  return s;
}
inline long long units_of(long long red, int parts) { return (red + BK - 1) / BK * parts; }

struct Layout {
  bool lay;                 // operands are laid out in the workspace
  int planes, kp, fp, runs, run;
  long long x, wg, wu, dg, du, sums, partial, bytes;
  Shape fwd, dx, dw;
};
// x as an operand where it is: whole 16-byte pieces
bool whole(const void* p, long long ld, int cols, int type) { return type != 0 && ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld >= cols; }

Layout layout(const vmm_gated_ff_desc* d, bool backward) {
  Layout l;
  l.planes = d->type == 0 ? 3 : 1;
  const int parts = d->type == 0 ? 6 : 1;
  l.kp = (int)up(d->K, 8);
  l.fp = (int)up(d->F, 8);
  l.lay = !(d->K % 8 == 0 && whole(d->x, d->ldx, d->K, d->type) && whole(d->w_gate, d->K, d->K, d->type) && whole(d->w_up, d->K, d->K, d->type));
  long long at = 0;
  const auto take = [&](long long bytes) { const long long o = at; at += up(bytes, 256); return o; };
  l.x = l.lay ? take(2LL * l.planes * d->M * l.kp) : 0;
  l.wg = l.lay ? take(2LL * l.planes * d->F * l.kp) : 0;
  l.wu = l.lay ? take(2LL * l.planes * d->F * l.kp) : 0;
  l.fwd = shape_of(d->M, d->F, true, units_of(d->K, parts), 1);
  l.dx = shape_of(d->M, d->K, false, units_of(d->F, 2 * parts), 1);
  l.dw = shape_of(d->F, d->K, false, units_of(d->M, parts), 2);
  if (backward) {
    l.dg = take(2LL * l.planes * d->M * l.fp);
    l.du = take(2LL * l.planes * d->M * l.fp);
    // runs of rows for the activation's backward: four workgroups a CU, 64 rows a run at the most unless the runs became too many
    const long long columns = (l.fp + 255) / 256, share = up(std::max(cdiv64(d->M * columns, 1024), 1LL), 4);
    l.run = (int)(share < 64 ? share : d->M <= 64 * 1024 ? 64 : up((d->M + 1023) / 1024, 4));
    l.runs = (int)((d->M + l.run - 1) / l.run);
    l.sums = take(8LL * l.runs * d->F);
    const long long px = l.dx.splits > 1 && d->dx ? 4LL * l.dx.splits * d->M * d->K : 0, pw = l.dw.splits > 1 && d->dw_gate ? 8LL * l.dw.splits * d->F * d->K : 0;
    l.partial = take(px > pw ? px : pw);
  } else {
    l.partial = take(l.fwd.splits > 1 ? 8LL * l.fwd.splits * d->M * d->F : 0);
  }
  l.bytes = at;
  return l;
}

bool room(const vmm_gated_ff_desc* d, bool backward) {
  const long long bytes = layout(d, backward).bytes;
  return bytes == 0 || (d->workspace && ((uintptr_t)d->workspace & 15) == 0 && d->workspace_bytes >= bytes);
}

template <int TYPE, bool ACOL, bool BCOL, bool GATED>
int product(Gemm& q, const Shape& sh, int products, hipStream_t s) {
  const int r = sh.big ? 256 : 128;
  q.splits = sh.splits;
  q.tiles_m = (q.rows + r - 1) / r;
  q.tiles_n = (q.cols * (GATED ? 2 : 1) + r - 1) / r;
  q.pairs = q.cols % 2 == 0 && q.ldo % 2 == 0 && (((uintptr_t)q.out[0] | (uintptr_t)q.out[1]) & 3) == 0;
  const long long blocks = (q.tiles_m * q.tiles_n + 7) / 8 * 8;
  if (cdiv64(q.red, BK) * q.parts >= (1LL << 30)) return -1;
  const dim3 grid((unsigned)blocks, products * q.splits);
  if (sh.big) hipLaunchKernelGGL((ff_gemm_kernel<TYPE, ACOL, BCOL, GATED, true>), grid, dim3(512), 0, s, q);
  else hipLaunchKernelGGL((ff_gemm_kernel<TYPE, ACOL, BCOL, GATED, false>), grid, dim3(256), 0, s, q);
  VMM_LAUNCH_CHECK();
  if (q.splits > 1) {
    const long long n = cdiv64(q.rows * q.cols, 256);  // (less than 512 tiles of 128 x 128, or nothing would be split)
    if constexpr (GATED) hipLaunchKernelGGL(ff_join_gated_kernel<TYPE>, dim3((unsigned)n), dim3(256), 0, s, q);
    else hipLaunchKernelGGL(ff_join_kernel<TYPE>, dim3((unsigned)n, products), dim3(256), 0, s, q);
    VMM_LAUNCH_CHECK();
  }
  return 0;
}

// which parts of A and B a product is made of, small ones first
constexpr int PART_A[6] = {2, 0, 1, 1, 0, 0}, PART_B[6] = {0, 2, 1, 0, 1, 0};
template <int TYPE> int parts_of(int i, bool of_a) { return TYPE == 0 ? (of_a ? PART_A[i] : PART_B[i]) : 0; }

struct Operands { const u16 *x, *wg, *wu; long long ldx, ldw, xplane, wplane; };
template <int TYPE>
int operands(const vmm_gated_ff_desc* d, const Layout& l, Operands& o, hipStream_t s) {
  char* w = (char*)d->workspace;
  if (!l.lay) {
    o = {(const u16*)d->x, (const u16*)d->w_gate, (const u16*)d->w_up, d->ldx, d->K, 0, 0};
    return 0;
  }
  o = {(const u16*)(w + l.x), (const u16*)(w + l.wg), (const u16*)(w + l.wu), l.kp, l.kp, d->M * l.kp, (long long)d->F * l.kp};
  const Layin a = {{d->x, d->w_gate, d->w_up}, {(u16*)(w + l.x), (u16*)(w + l.wg), (u16*)(w + l.wu)}, {d->M, d->F, d->F}, {d->ldx, d->K, d->K}, d->K, l.kp};
  const long long most = (d->M > d->F ? d->M : d->F) * (long long)l.kp;
  hipLaunchKernelGGL(ff_layin_kernel<TYPE>, dim3((unsigned)std::min(cdiv64(most, 256), 4096LL), 3), dim3(256), 0, s, a);
  VMM_LAUNCH_CHECK();
  return 0;
}

template <int TYPE>
int forward(const vmm_gated_ff_desc* d, hipStream_t s) {
  constexpr int NP = TYPE == 0 ? 6 : 1;
  const Layout l = layout(d, false);
  Operands o;
  if (const int e = operands<TYPE>(d, l, o, s)) return e;
  Gemm q = {};
  for (int i = 0; i < NP; ++i) {
    q.a[i] = o.x + parts_of<TYPE>(i, true) * o.xplane;
    q.b[i] = o.wg + parts_of<TYPE>(i, false) * o.wplane;
    q.b2[i] = o.wu + parts_of<TYPE>(i, false) * o.wplane;
  }
  q.lda = o.ldx; q.ldb = o.ldw; q.rows = d->M; q.cols = d->F; q.red = d->K; q.parts = NP;
  q.out[0] = d->h; q.ldo = d->ldh;
  q.partial = (float*)((char*)d->workspace + l.partial);
  q.b_gate = d->b_gate; q.b_up = d->b_up; q.g_pre = d->g_pre; q.u_pre = d->u_pre; q.act = d->act;
  return product<TYPE, false, false, true>(q, l.fwd, 1, s);
}

template <int TYPE>
int backward(const vmm_gated_ff_desc* d, hipStream_t s) {
  constexpr int NP = TYPE == 0 ? 6 : 1;
  const Layout l = layout(d, true);
  char* w = (char*)d->workspace;
  const bool bias = d->db_gate || d->db_up;
  float* sums = bias ? (float*)(w + l.sums) : nullptr;
  u16 *dg = (u16*)(w + l.dg), *du = (u16*)(w + l.du);
  if (d->M > 0) {
    const bool wide = d->F % 4 == 0 && d->lddh % 4 == 0 && ((uintptr_t)d->dh & (4 * esize(d->type) - 1)) == 0 && (((uintptr_t)d->g_pre | (uintptr_t)d->u_pre) & 15) == 0;
    const dim3 grid(cdiv(l.fp, 256), l.runs);
    if (wide) hipLaunchKernelGGL((ff_dact_kernel<TYPE, true>), grid, dim3(256), 0, s, *d, dg, du, l.fp, l.run, sums);
    else hipLaunchKernelGGL((ff_dact_kernel<TYPE, false>), grid, dim3(256), 0, s, *d, dg, du, l.fp, l.run, sums);
    VMM_LAUNCH_CHECK();
  }
  if (bias) {
    hipLaunchKernelGGL(ff_dbias_kernel<TYPE>, dim3(cdiv(2LL * d->F, 32)), dim3(256), 0, s, *d, (const float*)sums, l.runs);
    VMM_LAUNCH_CHECK();
  }
  if (!(d->dx && d->M > 0) && !d->dw_gate) return 0;
  Operands o = {};
  if (d->M > 0) {  // (without rows nothing is read, neither x nor weights need be there, and the weights' gradients are zero)
    if (const int e = operands<TYPE>(d, l, o, s)) return e;
  }
  const long long plane = d->M * l.fp;
  if (d->dx && d->M > 0) {
    Gemm q = {};
    for (int i = 0; i < NP; ++i) {
      q.a[2 * i] = dg + parts_of<TYPE>(i, true) * plane;
      q.b[2 * i] = o.wg + parts_of<TYPE>(i, false) * o.wplane;
      q.a[2 * i + 1] = du + parts_of<TYPE>(i, true) * plane;
      q.b[2 * i + 1] = o.wu + parts_of<TYPE>(i, false) * o.wplane;
    }
    q.lda = l.fp; q.ldb = o.ldw; q.rows = d->M; q.cols = d->K; q.red = d->F; q.parts = 2 * NP;
    q.out[0] = d->dx; q.ldo = d->lddx;
    q.partial = (float*)(w + l.partial);
    if (const int e = product<TYPE, false, true, false>(q, l.dx, 1, s)) return e;
  }
  if (d->dw_gate) {
    Gemm q = {};
    for (int i = 0; i < NP; ++i) {
      q.a[i] = dg + parts_of<TYPE>(i, true) * plane;
      q.a[NP + i] = du + parts_of<TYPE>(i, true) * plane;
      q.b[i] = q.b[NP + i] = o.x + parts_of<TYPE>(i, false) * o.xplane;
    }
    q.lda = l.fp; q.ldb = o.ldx; q.rows = d->F; q.cols = d->K; q.red = d->M; q.parts = NP;
    q.out[0] = d->dw_gate; q.out[1] = d->dw_up; q.ldo = d->K;
    q.partial = (float*)(w + l.partial);
    if (const int e = product<TYPE, true, true, false>(q, l.dw, 2, s)) return e;
  }
  return 0;
}

}  // namespace

extern "C" int64_t vmm_gated_ff_workspace(const vmm_gated_ff_desc* d, int32_t backward) {
  if (bad_ff(d)) return -1;
  return layout(d, backward != 0).bytes;
}

extern "C" int vmm_gated_ff(const vmm_gated_ff_desc* d, vmm_stream_t stream) {
  if (bad_ff(d)) return -1;
  if (d->M == 0) return 0;
  if (!d->x || !d->w_gate || !d->w_up || !d->h || !d->g_pre != !d->u_pre) return -1;
  if (!room(d, false)) return -1;
  hipStream_t s = (hipStream_t)stream;
  return d->type == 0 ? forward<0>(d, s) : d->type == 1 ? forward<1>(d, s) : forward<2>(d, s);
}

extern "C" int vmm_gated_ff_bwd(const vmm_gated_ff_desc* d, vmm_stream_t stream) {
  if (bad_ff(d)) return -1;
  if (!d->dw_gate != !d->dw_up) return -1;
  if (d->M > 0 && (!d->x || !d->w_gate || !d->w_up || !d->dh || !d->g_pre || !d->u_pre)) return -1;
  if (!room(d, true)) return -1;
  hipStream_t s = (hipStream_t)stream;
  return d->type == 0 ? backward<0>(d, s) : d->type == 1 ? backward<1>(d, s) : backward<2>(d, s);
}
