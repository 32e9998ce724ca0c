// Gated linear recurrence over time and its backward pass (an encoder layer beside the GRU of cond_att_GRU, vddp.py:546-549):
//
//   f_t = sigmoid(g_t),   h_t = f_t h_(t-1) + (1 - f_t) x_t,   y_t = h_t
//   dh_t = dy_t + f_(t+1) dh_(t+1),   dx_t = dh_t (1 - f_t),   dg_t = dh_t (h_(t-1) - x_t) f_t (1 - f_t),   dh0 = f_1 dh_1
//
// A step is the map h -> P h + Q with (P, Q) = (f, (1 - f) x), and maps compose: (P2, Q2) o (P1, Q1) = (P2 P1, P2 Q1 + Q2).  So time is cut into pieces
// whose maps are formed side by side and then joined in order; the backward runs the same machine from the right with c_t = f_t (dy_t + c_(t+1)).
//
// What bounds it: memory.  Forward reads x and gate once and writes y (3 values a step), backward reads x, gate, dy and writes dx, dgate (5).  Nothing
// is read twice: a tile stays in registers while its carry arrives.
//   thread   4 adjacent channels x TS steps; f and (1 - f) x in registers
//   wave     16 channel groups x 4 segments of time; joined with lane exchanges
//   block    4 waves = 16 segments: a tile of 64 channels x 16 TS steps; wave totals joined through LDS
//   grid     tiles along time pass the state on through memory: a tile first publishes its own map, then takes the state at the start of its group of
//            GROUP tiles and the maps published since, and joins them in order.  The last tile of a group publishes the state behind it.  The order in
//            which maps are joined is fixed by their places, not by who came first, so the result has the same bits every time.
// A tile waits for earlier tiles only.  Tiles are handed out by a counter in that order, so whoever holds the earliest unfinished one is working on it
// with all it needs published: every wait ends, however workgroups are placed.  A published value is one 64-bit (map) or 32-bit (state) word that is
// written whole and is not EMPTY, so it needs no flag and no fence.
#include "vmm_common.h"
#include "../../include/vmm_kernels.h"

namespace {

constexpr unsigned EMPTY = 0xffffffffu;  // what the workspace is filled with: a NaN that publish() never writes
constexpr int V = 4;                     // channels of a thread
constexpr int CG = 16;                   // channel groups of a tile: rows of 128 bytes in 16 bits, 256 in fp32
constexpr int STATE_STEP = 64;           // steps between the states that the forward keeps: the backward's tile

template <int TYPE> struct Elem;
template <> struct Elem<0> { typedef float T; typedef uint4 W; static constexpr unsigned PAD = 0x42D00000u; };
template <> struct Elem<1> { typedef __bf16 T; typedef uint2 W; static constexpr unsigned PAD = 0x42D042D0u; };
template <> struct Elem<2> { typedef _Float16 T; typedef uint2 W; static constexpr unsigned PAD = 0x56805680u; };
// PAD: gates of 104.  sigmoid(104) is 1 in fp32, so a padded step (x = 0) is the identity map, and its 1 - f is below the smallest normal number.

// V values side by side, kept as loaded until they are used
template <int TYPE> struct Raw {
  typedef typename Elem<TYPE>::W W;
  W u;
  __device__ __forceinline__ float get(int j) const {
    if constexpr (TYPE == 0) {
      const unsigned w[4] = {u.x, u.y, u.z, u.w};
      return __uint_as_float(w[j]);
    } else {
      const unsigned w = j < 2 ? u.x : u.y;
      if constexpr (TYPE == 1) return __uint_as_float((j & 1) ? (w & 0xffff0000u) : (w << 16));
      else return (float)__builtin_bit_cast(_Float16, (unsigned short)((j & 1) ? (w >> 16) : (w & 0xffffu)));
    }
  }
};
template <int TYPE>
__device__ __forceinline__ typename Elem<TYPE>::W pack(const float* v) {
  if constexpr (TYPE == 0) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else {
    typedef typename Elem<TYPE>::T T2 __attribute__((ext_vector_type(2)));
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t lo = {v[0], v[1]}, hi = {v[2], v[3]};
    return make_uint2(__builtin_bit_cast(unsigned, __builtin_convertvector(lo, T2)), __builtin_bit_cast(unsigned, __builtin_convertvector(hi, T2)));
  }
}
template <int TYPE>
__device__ __forceinline__ typename Elem<TYPE>::W fill_word(unsigned w) {
  if constexpr (TYPE == 0) return make_uint4(w, w, w, w);
  else return make_uint2(w, w);
}

// Where a thread's V channels are: side by side where accesses of four values are possible (WIDE), else 16 apart, so that the 16 lanes of a row still
// read 16 neighbours.
template <int TYPE, bool WIDE>
struct Place {
  typedef typename Elem<TYPE>::T T;
  typedef typename Elem<TYPE>::W W;
  int d0, D;
  __device__ __forceinline__ Place(int tile, int cg, int D_) : d0(tile * CG * V + (WIDE ? cg * V : cg)), D(D_) {}
  __device__ __forceinline__ int channel(int j) const { return WIDE ? d0 + j : d0 + j * CG; }
  __device__ __forceinline__ bool has(int j) const { return WIDE ? d0 < D : d0 + j * CG < D; }
  // row: the address of channel 0 of a step
  __device__ __forceinline__ W load(const T* row, unsigned pad) const {
    if constexpr (WIDE) {
      W r = fill_word<TYPE>(pad);
      if (d0 < D) r = *reinterpret_cast<const W*>(row + d0);
      return r;
    } else {
      unsigned w[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        w[j] = pad;
        if (has(j)) {
          if constexpr (TYPE == 0) w[j] = __builtin_bit_cast(unsigned, row[channel(j)]);
          else w[j] = __builtin_bit_cast(unsigned short, row[channel(j)]);
        }
      }
      if constexpr (TYPE == 0) return make_uint4(w[0], w[1], w[2], w[3]);
      else return make_uint2((w[0] & 0xffffu) | (w[1] << 16), (w[2] & 0xffffu) | (w[3] << 16));
    }
  }
  __device__ __forceinline__ void store(T* row, const float* v) const {
    if constexpr (WIDE) {
      if (d0 < D) *reinterpret_cast<W*>(row + d0) = pack<TYPE>(v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (has(j)) row[channel(j)] = (T)v[j];
    }
  }
  __device__ __forceinline__ void load_state(const float* s, float* v) const {  // s: channel 0 of a row of fp32 states
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = has(j) ? s[channel(j)] : 0.f;
  }
  __device__ __forceinline__ void store_state(float* s, const float* v) const {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (has(j)) s[channel(j)] = v[j];
  }
};

// f = sigmoid(g) and i = 1 - f = sigmoid(-g), each to a few ulp of itself: e = exp(-g) = 2^p 2^t with p = -g log2(e) rounded and t what the rounding
// left, f = 1 / (1 + e), i = e f.  Beyond +-104 / -87 both are constant in fp32; NaN passes.
__device__ __forceinline__ void gate_of(float g, float& f, float& i) {
  g = g < -87.f ? -87.f : g;
  g = g > 104.f ? 104.f : g;
  const float p = g * -1.44269502162933349609375f;
  float t = fmaf(g, -1.44269502162933349609375f, -p);
  t = fmaf(g, -1.925963033500011e-08f, t);
  float e = __builtin_amdgcn_exp2f(p);
  e = fmaf(e, t * 0.6931471805599453f, e);
  f = __builtin_amdgcn_rcpf(1.0f + e);
  i = e * f;
}

__device__ __forceinline__ unsigned word_of(float v) {
  const unsigned u = __float_as_uint(v);
  return u == EMPTY ? 0x7fc00000u : u;
}
__device__ __forceinline__ void publish_map(unsigned long long* at, float p, float q) {
  __hip_atomic_store(at, (unsigned long long)word_of(q) << 32 | word_of(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish_state(unsigned* at, float h) { __hip_atomic_store(at, word_of(h), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ unsigned long long peek(const unsigned long long* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ unsigned peek(const unsigned* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct ScanArgs {
  vmm_gated_scan_desc d;
  unsigned* counter;             // the next tile
  unsigned long long* maps;      // [tile along time][B][D]
  unsigned* states;              // [group][B][D]
  int tiles;                     // channel tiles
  unsigned chunks, total;        // tiles along time, and in all
};

constexpr int GROUP = 16;

// the map of the segments before (FORWARD) or behind this one inside its wave, and the wave's own map, from the segment's (p, q)
template <bool FORWARD>
__device__ __forceinline__ void wave_join(float* p, float* q, float* pe, float* qe) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    pe[j] = 1.f; qe[j] = 0.f;
#pragma unroll
    for (int bit = 4; bit <= 5; ++bit) {
      const bool upper = threadIdx.x & (1u << bit);
      const bool later = upper == FORWARD;  // this side's map is applied after the other's
      const float pp = lane_xor(p[j], bit), qq = lane_xor(q[j], bit);
      if (later) {  // (its exclusive part follows everything of the other side)
        qe[j] = fmaf(pe[j], qq, qe[j]);
        pe[j] *= pp;
      }
      const float first_q = later ? qq : q[j], then_p = later ? p[j] : pp, then_q = later ? q[j] : qq;
      q[j] = fmaf(then_p, first_q, then_q);
      p[j] *= pp;
    }
  }
}

// The state in front of tile `c` (c counts in the direction of the walk), from the state at its group's start and the maps since.
// Sixteen rows of lanes fetch one map each, so the waits for a group's maps are one wait; joined by every wave for itself.
template <int TYPE, bool WIDE>
__device__ __forceinline__ void carry_in(const ScanArgs& a, const Place<TYPE, WIDE>& at, unsigned c, int b, const float* start, float (*got)[CG][2 * V],
                                         float* h) {
  const int cg = threadIdx.x & 15, row = threadIdx.x >> 4;
  const unsigned base = c / GROUP * GROUP, mine = base + row;
  const long long BD = (long long)a.d.B * a.d.D, bd = (long long)b * a.d.D;
  if (mine < c) {
    const unsigned long long* m = a.maps + mine * BD + bd;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      unsigned long long w = 0;
      if (at.has(j)) {
        while ((unsigned)(w = peek(m + at.channel(j))) == EMPTY) __builtin_amdgcn_s_sleep(1);
      }
      got[row][cg][2 * j] = __uint_as_float((unsigned)w);
      got[row][cg][2 * j + 1] = __uint_as_float((unsigned)(w >> 32));
    }
  } else if (row == GROUP - 1) {  // c - base is 15 at most: this row has no map to fetch
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float v = start[j];
      if (base > 0 && at.has(j)) {
        const unsigned* s = a.states + (base / GROUP - 1) * BD + bd + at.channel(j);
        unsigned w;
        while ((w = peek(s)) == EMPTY) __builtin_amdgcn_s_sleep(1);
        v = __uint_as_float(w);
      }
      got[row][cg][j] = v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) h[j] = got[GROUP - 1][cg][j];
  for (unsigned k = 0; k < c - base; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = fmaf(got[k][cg][2 * j], h[j], got[k][cg][2 * j + 1]);
}

template <int TYPE, bool WIDE, int TS>
__global__ __launch_bounds__(256, 3) void scan_fwd_kernel(const ScanArgs a) {
  typedef typename Elem<TYPE>::T T;
  constexpr int TILE = 16 * TS;
  __shared__ float wave_map[4][CG][2 * V];
  __shared__ float got[16][CG][2 * V];
  __shared__ unsigned next_tile;
  const vmm_gated_scan_desc& d = a.d;
  const int cg = threadIdx.x & 15, seg = threadIdx.x >> 4, wave = threadIdx.x >> 6;
  const long long BD = (long long)d.B * d.D;
  unsigned tile = blockIdx.x;
  if (a.chunks > 1) {
    if (threadIdx.x == 0) next_tile = atomicAdd(a.counter, 1u);
    __syncthreads();
    tile = next_tile;
  }
  while (tile < a.total) {
    const unsigned per = (unsigned)d.B * a.tiles;
    const unsigned c = tile / per, bt = tile % per;
    const int b = bt / a.tiles;
    const Place<TYPE, WIDE> at(bt % a.tiles, cg, d.D);
    const long long len = d.lengths ? max(0LL, min((long long)d.lengths[b], (long long)d.L)) : (long long)d.L;
    const long long t0 = (long long)c * TILE + seg * TS;
    const T* xr = (const T*)d.x + b * d.x_batch + t0 * d.x_row;
    const T* gr = (const T*)d.gate + b * d.gate_batch + t0 * d.gate_row;
    Raw<TYPE> x[TS], g[TS];
    if (t0 + TS <= len) {
#pragma unroll
      for (int k = 0; k < TS; ++k) { x[k].u = at.load(xr + k * d.x_row, 0u); g[k].u = at.load(gr + k * d.gate_row, Elem<TYPE>::PAD); }
    } else {
#pragma unroll
      for (int k = 0; k < TS; ++k) {
        x[k].u = fill_word<TYPE>(0u);
        g[k].u = fill_word<TYPE>(Elem<TYPE>::PAD);
        if (t0 + k < len) { x[k].u = at.load(xr + k * d.x_row, 0u); g[k].u = at.load(gr + k * d.gate_row, Elem<TYPE>::PAD); }
      }
    }
    unsigned ahead = 0;
    if (a.chunks > 1 && threadIdx.x == 0) ahead = atomicAdd(a.counter, 1u);
    float start[V];
#pragma unroll
    for (int j = 0; j < V; ++j) start[j] = 0.f;
    if (c < GROUP && d.h0) at.load_state(d.h0 + (long long)b * d.D, start);

    float f[TS][V], q[TS][V], P[V], Q[V], pe[V], qe[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { P[j] = 1.f; Q[j] = 0.f; }
#pragma unroll
    for (int k = 0; k < TS; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float i;
        gate_of(g[k].get(j), f[k][j], i);
        q[k][j] = i * x[k].get(j);
        P[j] *= f[k][j];
        Q[j] = fmaf(f[k][j], Q[j], q[k][j]);
      }
    wave_join<true>(P, Q, pe, qe);
    if ((threadIdx.x & 48) == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) { wave_map[wave][cg][2 * j] = P[j]; wave_map[wave][cg][2 * j + 1] = Q[j]; }
    }
    __syncthreads();
    float pw[V], qw[V];  // the waves before this one
#pragma unroll
    for (int j = 0; j < V; ++j) { pw[j] = 1.f; qw[j] = 0.f; }
    for (int w = 0; w < wave; ++w)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float p1 = wave_map[w][cg][2 * j], q1 = wave_map[w][cg][2 * j + 1];
        pw[j] *= p1;
        qw[j] = fmaf(p1, qw[j], q1);
      }
    if (a.chunks > 1) {
      if (threadIdx.x == 0) next_tile = ahead;
      if (seg == 15 && c + 1 < a.chunks && c % GROUP != GROUP - 1) {
        unsigned long long* m = a.maps + c * BD + (long long)b * d.D;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (at.has(j)) publish_map(m + at.channel(j), P[j] * pw[j], fmaf(P[j], qw[j], Q[j]));
      }
      carry_in<TYPE, WIDE>(a, at, c, b, start, got, start);
    }
    float h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = fmaf(pe[j], fmaf(pw[j], start[j], qw[j]), qe[j]);
    if (d.states && (seg * TS) % STATE_STEP == 0) {
      const long long s = (long long)c * (TILE / STATE_STEP) + seg * TS / STATE_STEP;
      if (s * STATE_STEP < d.L) at.store_state(d.states + s * BD + (long long)b * d.D, h);
    }
    T* yr = (T*)d.y + b * d.y_batch + t0 * d.y_row;
#pragma unroll
    for (int k = 0; k < TS; ++k) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[j] = fmaf(f[k][j], h[j], q[k][j]);
        o[j] = t0 + k < len ? h[j] : 0.f;
      }
      if (t0 + k < d.L) at.store(yr + k * d.y_row, o);
    }
    if (seg == 15) {
      if (c + 1 == a.chunks) {
        if (d.h_last) at.store_state(d.h_last + (long long)b * d.D, h);
      } else if (c % GROUP == GROUP - 1) {
        unsigned* s = a.states + c / GROUP * BD + (long long)b * d.D;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (at.has(j)) publish_state(s + at.channel(j), h[j]);
      }
    }
    if (a.chunks == 1) break;
    tile = next_tile;  // (written before carry_in's barrier; written again behind the next tile's first one)
  }
}

template <int TYPE, bool WIDE, int TS>
__global__ __launch_bounds__(256, 3) void scan_bwd_kernel(const ScanArgs a) {
  typedef typename Elem<TYPE>::T T;
  constexpr int TILE = 16 * TS;
  static_assert(TILE == STATE_STEP, "a tile starts from the state that the forward kept");
  __shared__ float wave_map[2][4][CG][2 * V];
  __shared__ float got[16][CG][2 * V];
  __shared__ unsigned next_tile;
  const vmm_gated_scan_desc& d = a.d;
  const int cg = threadIdx.x & 15, seg = threadIdx.x >> 4, wave = threadIdx.x >> 6;
  const long long BD = (long long)d.B * d.D;
  unsigned tile = blockIdx.x;
  if (a.chunks > 1) {
    if (threadIdx.x == 0) next_tile = atomicAdd(a.counter, 1u);
    __syncthreads();
    tile = next_tile;
  }
  while (tile < a.total) {
    const unsigned per = (unsigned)d.B * a.tiles;
    const unsigned r = tile / per, bt = tile % per, c = a.chunks - 1 - r;  // r counts from the end of time
    const int b = bt / a.tiles;
    const long long bd = (long long)b * d.D;
    const Place<TYPE, WIDE> at(bt % a.tiles, cg, d.D);
    const long long len = d.lengths ? max(0LL, min((long long)d.lengths[b], (long long)d.L)) : (long long)d.L;
    const long long t0 = (long long)c * TILE + seg * TS;
    const T* xr = (const T*)d.x + b * d.x_batch + t0 * d.x_row;
    const T* gr = (const T*)d.gate + b * d.gate_batch + t0 * d.gate_row;
    const T* yr = (const T*)d.dy + b * d.dy_batch + t0 * d.dy_row;
    Raw<TYPE> x[TS], g[TS], dy[TS];
#pragma unroll
    for (int k = 0; k < TS; ++k) {
      x[k].u = dy[k].u = fill_word<TYPE>(0u);
      g[k].u = fill_word<TYPE>(Elem<TYPE>::PAD);
      if (t0 + k < len) {
        x[k].u = at.load(xr + k * d.x_row, 0u);
        g[k].u = at.load(gr + k * d.gate_row, Elem<TYPE>::PAD);
        if (d.dy) dy[k].u = at.load(yr + k * d.dy_row, 0u);
      }
    }
    unsigned ahead = 0;
    if (a.chunks > 1 && threadIdx.x == 0) ahead = atomicAdd(a.counter, 1u);
    float h[V], start[V];
    at.load_state(d.states + c * BD + bd, h);
#pragma unroll
    for (int j = 0; j < V; ++j) start[j] = 0.f;
    if (r < GROUP && d.dh_last) at.load_state(d.dh_last + bd, start);

    float f[TS][V], i[TS][V], P[V], Q[V], R[V], pf[V], qf[V], pb[V], rb[V], P2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { P[j] = 1.f; Q[j] = 0.f; R[j] = 0.f; }
#pragma unroll
    for (int k = 0; k < TS; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        gate_of(g[k].get(j), f[k][j], i[k][j]);
        P[j] *= f[k][j];
        Q[j] = fmaf(f[k][j], Q[j], i[k][j] * x[k].get(j));
      }
#pragma unroll
    for (int k = TS - 1; k >= 0; --k)
#pragma unroll
      for (int j = 0; j < V; ++j) R[j] = f[k][j] * (dy[k].get(j) + R[j]);
#pragma unroll
    for (int j = 0; j < V; ++j) P2[j] = P[j];
    wave_join<true>(P, Q, pf, qf);
    wave_join<false>(P2, R, pb, rb);
    if ((threadIdx.x & 48) == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        wave_map[0][wave][cg][2 * j] = P[j]; wave_map[0][wave][cg][2 * j + 1] = Q[j];
        wave_map[1][wave][cg][2 * j] = P2[j]; wave_map[1][wave][cg][2 * j + 1] = R[j];
      }
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w)  // the state in front of this wave
#pragma unroll
      for (int j = 0; j < V; ++j) h[j] = fmaf(wave_map[0][w][cg][2 * j], h[j], wave_map[0][w][cg][2 * j + 1]);
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = fmaf(pf[j], h[j], qf[j]);
    float pw[V], rw[V];  // the waves behind this one
#pragma unroll
    for (int j = 0; j < V; ++j) { pw[j] = 1.f; rw[j] = 0.f; }
    for (int w = 3; w > wave; --w)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float p1 = wave_map[1][w][cg][2 * j], r1 = wave_map[1][w][cg][2 * j + 1];
        pw[j] *= p1;
        rw[j] = fmaf(p1, rw[j], r1);
      }
    if (a.chunks > 1) {
      if (threadIdx.x == 0) next_tile = ahead;
      if (seg == 0 && r + 1 < a.chunks && r % GROUP != GROUP - 1) {
        unsigned long long* m = a.maps + r * BD + bd;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (at.has(j)) publish_map(m + at.channel(j), P2[j] * pw[j], fmaf(P2[j], rw[j], R[j]));
      }
      carry_in<TYPE, WIDE>(a, at, r, b, start, got, start);
    }
    float back[V];  // c_(t+1) of the segment's last step
#pragma unroll
    for (int j = 0; j < V; ++j) back[j] = fmaf(pb[j], fmaf(pw[j], start[j], rw[j]), rb[j]);
    // h_(t-1) - x_t, forwards; it takes the place of x
    float hx[TS][V];
#pragma unroll
    for (int k = 0; k < TS; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xv = x[k].get(j);
        hx[k][j] = h[j] - xv;
        h[j] = fmaf(f[k][j], h[j], i[k][j] * xv);
      }
    T* xo = (T*)d.dx + b * d.dx_batch + t0 * d.dx_row;
    T* go = (T*)d.dgate + b * d.dgate_batch + t0 * d.dgate_row;
#pragma unroll
    for (int k = TS - 1; k >= 0; --k) {
      float ox[V], og[V];
      const bool live = t0 + k < len;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float dh = dy[k].get(j) + back[j], di = dh * i[k][j];
        ox[j] = live ? di : 0.f;
        og[j] = live ? di * f[k][j] * hx[k][j] : 0.f;
        back[j] = f[k][j] * dh;
      }
      if (t0 + k < d.L) {
        if (d.dx) at.store(xo + k * d.dx_row, ox);
        if (d.dgate) at.store(go + k * d.dgate_row, og);
      }
    }
    if (seg == 0) {
      if (c == 0) {
        if (d.dh0) at.store_state(d.dh0 + bd, back);
      } else if (r % GROUP == GROUP - 1) {
        unsigned* s = a.states + r / GROUP * BD + bd;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (at.has(j)) publish_state(s + at.channel(j), back[j]);
      }
    }
    if (a.chunks == 1) break;
    tile = next_tile;
  }
}

__global__ __launch_bounds__(256) void scan_clear_kernel(unsigned* counter, uint4* p, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i == 0) *counter = 0u;
  if (i < n) p[i] = make_uint4(EMPTY, EMPTY, EMPTY, EMPTY);
}

constexpr int FWD_TS = 8, BWD_TS = 4;

inline int esize(int type) { return type == 0 ? 4 : 2; }

bool bad_scan(const vmm_gated_scan_desc* d) {
  return !d || d->B < 0 || d->D < 0 || d->L < 0 || d->L >= (1LL << 31) || d->type < 0 || d->type > 2 || (int64_t)d->B * d->D >= (1LL << 31);
}
struct Layout { unsigned chunks; long long maps, states; };  // counts of words
Layout layout(const vmm_gated_scan_desc* d, bool backward) {
  const int tile = 16 * (backward ? BWD_TS : FWD_TS);
  Layout l;
  l.chunks = (unsigned)((d->L + tile - 1) / tile);
  const long long BD = (long long)d->B * d->D;
  l.maps = l.chunks > 1 ? l.chunks * BD : 0;
  l.states = l.chunks > 1 ? (l.chunks / GROUP + 1) * BD : 0;
  return l;
}
inline long long up16(long long n) { return (n + 15) / 16 * 16; }

// accesses of four values to rows of D: addresses, strides and D itself have to allow them
bool wide(const void* p, int64_t batch, int64_t row, int D, int type) {
  return !p || (((uintptr_t)p & (V * esize(type) - 1)) == 0 && batch % V == 0 && row % V == 0 && D % V == 0);
}

template <bool FWD, int TYPE>
void launch(const ScanArgs& a, bool w, int blocks, hipStream_t s) {
  if constexpr (FWD) {
    if (w) hipLaunchKernelGGL((scan_fwd_kernel<TYPE, true, FWD_TS>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((scan_fwd_kernel<TYPE, false, FWD_TS>), dim3(blocks), dim3(256), 0, s, a);
  } else {
    if (w) hipLaunchKernelGGL((scan_bwd_kernel<TYPE, true, BWD_TS>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((scan_bwd_kernel<TYPE, false, BWD_TS>), dim3(blocks), dim3(256), 0, s, a);
  }
}

template <bool FWD>
int scan(const vmm_gated_scan_desc* d, hipStream_t s) {
  const Layout l = layout(d, !FWD);
  ScanArgs a;
  a.d = *d;
  a.tiles = (d->D + CG * V - 1) / (CG * V);
  a.chunks = l.chunks;
  const unsigned long long total = (unsigned long long)l.chunks * d->B * a.tiles;
  if (total >= 0xff000000ull) return -1;  // (the counter runs past it by the number of workgroups)
  a.total = (unsigned)total;
  int blocks = (int)total;
  if (l.chunks > 1) {
    if (!d->workspace || ((uintptr_t)d->workspace & 15)) return -1;
    a.counter = (unsigned*)d->workspace;
    a.maps = (unsigned long long*)((char*)d->workspace + 16);
    a.states = (unsigned*)((char*)d->workspace + 16 + up16(8 * l.maps));
    const long long n = (up16(8 * l.maps) + up16(4 * l.states)) / 16;
    hipLaunchKernelGGL(scan_clear_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a.counter, (uint4*)a.maps, n);
    VMM_LAUNCH_CHECK();
    blocks = (int)min(total, 1024ull);  // at least what the card holds at once; each takes tiles until none is left
  }
  const bool w = wide(d->x, d->x_batch, d->x_row, d->D, d->type) && wide(d->gate, d->gate_batch, d->gate_row, d->D, d->type) &&
                 (FWD ? wide(d->y, d->y_batch, d->y_row, d->D, d->type)
                      : wide(d->dy, d->dy_batch, d->dy_row, d->D, d->type) && wide(d->dx, d->dx_batch, d->dx_row, d->D, d->type) &&
                            wide(d->dgate, d->dgate_batch, d->dgate_row, d->D, d->type));
  if (d->type == 0) launch<FWD, 0>(a, w, blocks, s);
  else if (d->type == 1) launch<FWD, 1>(a, w, blocks, s);
  else launch<FWD, 2>(a, w, blocks, s);
  VMM_LAUNCH_CHECK();
  return 0;
}

// no steps: the state passes through, and so does its gradient
__global__ __launch_bounds__(256) void scan_pass_kernel(const float* __restrict__ from, float* __restrict__ to, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.f;
}
int pass(const float* from, float* to, long long n, hipStream_t s) {
  if (!to || n == 0) return 0;
  hipLaunchKernelGGL(scan_pass_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, from, to, n);
  VMM_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" int64_t vmm_gated_scan_states(const vmm_gated_scan_desc* d) {
  if (bad_scan(d)) return -1;
  return (d->L + STATE_STEP - 1) / STATE_STEP * d->B * d->D;
}

extern "C" int64_t vmm_gated_scan_workspace(const vmm_gated_scan_desc* d, int32_t backward) {
  if (bad_scan(d)) return -1;
  const Layout l = layout(d, backward != 0);
  return l.chunks > 1 ? 16 + up16(8 * l.maps) + up16(4 * l.states) : 0;
}

extern "C" int vmm_gated_scan(const vmm_gated_scan_desc* d, vmm_stream_t stream) {
  if (bad_scan(d)) return -1;
  const long long BD = (long long)d->B * d->D;
  if (BD == 0) return 0;
  if (d->L == 0) return pass(d->h0, d->h_last, BD, (hipStream_t)stream);
  if (!d->x || !d->gate || !d->y) return -1;
  return scan<true>(d, (hipStream_t)stream);
}

extern "C" int vmm_gated_scan_bwd(const vmm_gated_scan_desc* d, vmm_stream_t stream) {
  if (bad_scan(d)) return -1;
  const long long BD = (long long)d->B * d->D;
  if (BD == 0) return 0;
  if (d->L == 0) return pass(d->dh_last, d->dh0, BD, (hipStream_t)stream);
  if (!d->x || !d->gate || !d->states) return -1;
  return scan<false>(d, (hipStream_t)stream);
}
