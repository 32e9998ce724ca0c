// Gated linear recurrence over time and its backward pass (an encoder layer beside the GRU of cond_att_GRU, vddp.py:546-549):
//
//   f_t = sigmoid(g_t),   h_t = f_t h_(t-1) + (1 - f_t) x_t,   y_t = h_t
//   dh_t = dy_t + f_(t+1) dh_(t+1),   dx_t = dh_t (1 - f_t),   dg_t = dh_t (h_(t-1) - x_t) f_t (1 - f_t),   dh0 = f_1 dh_1
//
// A step is the map h -> P h + Q with (P, Q) = (f, (1 - f) x), and maps compose: (P2, Q2) o (P1, Q1) = (P2 P1, P2 Q1 + Q2).  So time is cut into units of
// 64 steps.  The backward runs the same machine from the end of time with c_t = f_t (dy_t + c_(t+1)), whose maps are (f, f dy).
//   1. maps     every unit's map, and that of every 16 units (a group)                       reads x and gate (backward: gate and dy)
//   2. states   the state in front of every unit: maps of the groups before, then of the units before inside the group
//   3. apply    every unit by itself from that state                                         reads x and gate, writes y
// A sequence of one unit needs the last alone.  Where there are more than 256 groups, the state in front of every 256th (an anchor) is formed first, so
// that step 2 goes through 255 groups at the most.  Which maps are joined in which order depends on the sizes alone: the same bits every time.
//
// What bounds it: memory and instructions alike.  3 values a step move forward and 5 backward, plus 2 for the maps, which the third step finds in the 256 MB
// of last-level cache for the most part: it walks time from the end, where step 1 has read last.  65536 steps of 1024 channels in bf16 take 57 + 8 + 70 us: the
// maps read at a copy's 4.8 TB/s; the 402 MB that have to move once are 83 us of it.  Each value costs some thirty instructions, so whatever can be
// decided for a whole unit is (see `unit`).  Passing states from workgroup to workgroup inside one launch would read all of it once, and was
// built first; workgroups then poll each other's results past the caches, and the same took 192 us (228 us with groups and tiles of 128 steps; 370 us with tiles of 64).
#include <type_traits>
#include "vmm_common.h"
#include "../../include/vmm_kernels.h"

namespace {

constexpr int V = 4;                     // channels of a thread
constexpr int CG = 16;                   // channel groups of a tile: rows of 128 bytes in 16 bits, 256 in fp32
constexpr int UNIT = 64;                 // steps of a unit of time
constexpr int GROUP = 16;                // units of a group
constexpr int ANCHOR = 256;              // groups between anchors

template <int TYPE> struct Elem;
template <> struct Elem<0> { typedef float T; typedef uint4 W; static constexpr unsigned PAD = 0x42D00000u; };
template <> struct Elem<1> { typedef __bf16 T; typedef uint2 W; static constexpr unsigned PAD = 0x42D042D0u; };
template <> struct Elem<2> { typedef _Float16 T; typedef uint2 W; static constexpr unsigned PAD = 0x56805680u; };
// PAD: gates of 104.  sigmoid(104) is 1 in fp32, so a padded step (x = 0) is the identity map.

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

// A thread's V channels inside a tile: side by side where accesses of four values are possible (WIDE), else 16 apart, so that the 16 lanes of a row
// still read 16 neighbours.  Rows are addressed as a place that is the same for all lanes plus a 32-bit lane offset.
template <int TYPE, bool WIDE>
struct Place {
  typedef typename Elem<TYPE>::T T;
  typedef typename Elem<TYPE>::W W;
  int d0, D;  // D: channels from the tile's first one on
  __device__ __forceinline__ Place(int cg, int D_) : d0(WIDE ? cg * V : cg), D(D_) {}
  __device__ __forceinline__ int channel(int j) const { return WIDE ? d0 + j : d0 + j * CG; }
  __device__ __forceinline__ bool has(int j) const { return WIDE ? d0 < D : d0 + j * CG < D; }
  // row: the address of the tile's first channel, off: of the lane's own beyond it, in bytes
  __device__ __forceinline__ W load(const char* row, unsigned off, unsigned pad) const {
    if constexpr (WIDE) {
      W r = fill_word<TYPE>(pad);
      if (d0 < D) r = *reinterpret_cast<const W*>(row + off);
      return r;
    } else {
      unsigned w[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        w[j] = pad;
        if (has(j)) {
          const T* p = reinterpret_cast<const T*>(row + off) + j * CG;
          if constexpr (TYPE == 0) w[j] = __builtin_bit_cast(unsigned, *p);
          else w[j] = __builtin_bit_cast(unsigned short, *p);
        }
      }
      if constexpr (TYPE == 0) return make_uint4(w[0], w[1], w[2], w[3]);
      else return make_uint2((w[0] & 0xffffu) | (w[1] << 16), (w[2] & 0xffffu) | (w[3] << 16));
    }
  }
  __device__ __forceinline__ void store(char* row, unsigned off, const float* v) const {
    if constexpr (WIDE) {
      if (d0 < D) *reinterpret_cast<W*>(row + off) = pack<TYPE>(v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (has(j)) (reinterpret_cast<T*>(row + off))[j * CG] = (T)v[j];
    }
  }
  __device__ __forceinline__ void load_state(const float* s, float* v) const {  // s: the tile's first channel in a row of fp32 states
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = has(j) ? s[channel(j)] : 0.f;
  }
  __device__ __forceinline__ void store_state(float* s, const float* v) const {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (has(j)) s[channel(j)] = v[j];
  }
};

// a value that is the same in every lane, in a scalar register
__device__ __forceinline__ unsigned uniform(unsigned v) { return __builtin_amdgcn_readfirstlane(v); }

// f = sigmoid(g) and i = 1 - f = sigmoid(-g), each accurate in itself: dgate and dh0 are proportional to f, and f is multiplied with itself over a whole memory.  The smaller
// of the two is e / (1 + e) with e = e^-|g|, the larger 1 minus that, which has one rounding (the error of a reciprocal would add up over a memory).
// 16 bits: i = 1 / (1 + e^g) serves either way, zero and infinite e^g too; f = 1 - i where the gate is open and e^g i where it is closed, where 1 - i has lost it
// (by a sixth at g = -15, all of it from -17 on).
// fp32: exp is corrected for what rounding p = -|g| log2(e) has lost, up to |g| 2^-25 of e.  NaN passes in both.
template <int TYPE>
__device__ __forceinline__ void gate_of(float g, float& f, float& i) {
  if constexpr (TYPE == 0) {
    float m = fabsf(g);
    m = m > 104.f ? 104.f : m;  // (exp is zero from there on; an infinite one would leave inf - inf below)
    const float p = m * -1.44269502162933349609375f;
    float t = fmaf(m, -1.44269502162933349609375f, -p);
    t = fmaf(m, -1.925963033500011e-08f, t);
    float e = __builtin_amdgcn_exp2f(p);
    e = fmaf(e, t * 0.6931471805599453f, e);
    const float small = e * __builtin_amdgcn_rcpf(1.0f + e), large = 1.0f - small;
    f = g < 0.f ? small : large;
    i = g < 0.f ? large : small;
  } else {
    const float e = __builtin_amdgcn_exp2f(g * 1.44269502162933349609375f);
    i = __builtin_amdgcn_rcpf(1.0f + e);
    f = g < 0.f ? e * i : 1.0f - i;
  }
}

struct ScanArgs {
  vmm_gated_scan_desc d;
  int tiles;           // of 64 channels
  unsigned units, groups;
  bool runs;           // whether an XCD's workgroups are neighbours
  float2* maps;        // [unit][B][D]; units and groups count in the direction of the walk
  float2* group_maps;  // [group][B][D]
  float* anchors;      // [group / 256][B][D]
  float* states;       // [unit][B][D]: the state in front of each (forward: the caller's, where it keeps them)
};

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
      qe[j] = later ? fmaf(pe[j], qq, qe[j]) : qe[j];  // (its exclusive part follows everything of the other side)
      pe[j] = later ? pe[j] * pp : pe[j];
      const float first_q = later ? qq : q[j], then_p = later ? p[j] : pp, then_q = later ? q[j] : qq;
      q[j] = fmaf(then_p, first_q, then_q);
      p[j] *= pp;
    }
  }
}

// Consecutive workgroups go to different XCDs.  Where rows do not start on cache lines, each XCD gets a run of the work instead, so that tiles beside each
// other share the lines at their borders in one L2: 4093 steps of 8 x 1000 channels in bf16 take 27 / 35 / 27 / 68 us for forward maps and application,
// backward maps and application where the plain order takes 34 / 48 / 33 / 86; rows that do (65536 x 1024) 57 / 70 us in the plain order and
// 61 / 71 in runs.  The grid is eight runs; numbers from `work` on are nobody's.
__device__ __forceinline__ unsigned number(const ScanArgs& a, unsigned work) {
  return a.runs ? (blockIdx.x & 7) * ((work + 7) / 8) + (blockIdx.x >> 3) : blockIdx.x;
}

// both directions at once, whose maps have their factor in common: (p, q) forwards, (p, r) backwards
__device__ __forceinline__ void wave_join_both(float* p, float* q, float* r, float* pf, float* qf, float* pb, float* rb) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    pf[j] = pb[j] = 1.f; qf[j] = rb[j] = 0.f;
#pragma unroll
    for (int bit = 4; bit <= 5; ++bit) {
      const bool upper = threadIdx.x & (1u << bit);
      const float pp = lane_xor(p[j], bit), qq = lane_xor(q[j], bit), rr = lane_xor(r[j], bit);
      qf[j] = upper ? fmaf(pf[j], qq, qf[j]) : qf[j];
      pf[j] = upper ? pf[j] * pp : pf[j];
      rb[j] = upper ? rb[j] : fmaf(pb[j], rr, rb[j]);
      pb[j] = upper ? pb[j] : pb[j] * pp;
      q[j] = upper ? fmaf(p[j], qq, q[j]) : fmaf(pp, q[j], qq);
      r[j] = upper ? fmaf(pp, r[j], rr) : fmaf(p[j], rr, r[j]);
      p[j] *= pp;
    }
  }
}

// ---- step 1.  A workgroup makes the maps of a group: a wave a unit, a lane 4 channels and a quarter of its steps, four at a time with the next ones on
// their way (eight at a time need more registers than 16 waves have, and took a sixth longer).
// Forward from x and gate, BACK from dy and gate.
template <int TYPE, bool WIDE, bool BACK>
__global__ __launch_bounds__(1024) void scan_map_kernel(const ScanArgs a) {
  constexpr int STEPS = UNIT / 4, BATCH = 4, BATCHES = STEPS / BATCH;
  __shared__ float2 join[GROUP][CG][V];
  const vmm_gated_scan_desc& d = a.d;
  const int cg = threadIdx.x & 15, quarter = (threadIdx.x >> 4) & 3, wave = uniform(threadIdx.x >> 6);
  const unsigned id = number(a, a.groups * d.B * a.tiles);
  if (id >= a.groups * d.B * a.tiles) return;
  const unsigned rest = uniform(id / a.tiles), tile = id - rest * a.tiles, group = uniform(rest / d.B), b = rest - group * d.B;
  const int columns = d.D - (int)tile * CG * V;
  const unsigned u = group * GROUP + wave;  // in the direction of the walk
  const bool exists = u < a.units;
  const long long first = (long long)(BACK ? a.units - 1 - u : u) * UNIT;
  long long len = d.L;
  if (d.lengths) len = max(0LL, min((long long)d.lengths[b], len));
  const long long es = sizeof(typename Elem<TYPE>::T), bd = (long long)b * d.D + (long long)tile * CG * V;
  const void* xv = BACK ? d.dy : d.x;
  const int64_t xb = BACK ? d.dy_batch : d.x_batch, xs = BACK ? d.dy_row : d.x_row;
  const auto row = [&](const void* p, int64_t batch, int64_t step, int k) {
    return (const char*)p + (b * batch + (first + k) * step + (long long)tile * CG * V) * es;
  };
  const bool has_x = !BACK || d.dy;
  const auto unit = [&](auto whole) {
    constexpr bool ALL = decltype(whole)::value;
    const Place<TYPE, WIDE> at(cg, ALL ? CG * V : columns);
    const int live = ALL ? UNIT : exists ? (int)min(max(len - first, 0LL), (long long)UNIT) - quarter * STEPS : 0;
    const unsigned xl = (quarter * STEPS * (unsigned)xs + at.d0) * (unsigned)es, gl = (quarter * STEPS * (unsigned)d.gate_row + at.d0) * (unsigned)es;
    Raw<TYPE> x[BATCH], g[BATCH];
    auto load = [&](int k0) {
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        x[k].u = fill_word<TYPE>(0u);
        g[k].u = fill_word<TYPE>(Elem<TYPE>::PAD);
        if (k0 + k < live) {
          if (has_x) x[k].u = at.load(row(xv, xb, xs, k0 + k), xl, 0u);
          g[k].u = at.load(row(d.gate, d.gate_batch, d.gate_row, k0 + k), gl, Elem<TYPE>::PAD);
        }
      }
    };
    float P[V], Q[V], pe[V], qe[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { P[j] = 1.f; Q[j] = 0.f; }
    if (ALL || (exists && len > first)) {
      load(BACK ? STEPS - BATCH : 0);
#pragma unroll
      for (int n = 0; n < BATCHES; ++n) {
        float f[BATCH][V], q[BATCH][V];
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float i;
            gate_of<TYPE>(g[k].get(j), f[k][j], i);
            q[k][j] = BACK ? x[k].get(j) : i * x[k].get(j);
          }
        if (n + 1 < BATCHES) load((BACK ? BATCHES - 2 - n : n + 1) * BATCH);
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
          const int k = BACK ? BATCH - 1 - s : s;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            Q[j] = BACK ? f[k][j] * (q[k][j] + Q[j]) : fmaf(f[k][j], Q[j], q[k][j]);
            P[j] *= f[k][j];
          }
        }
      }
    }
    wave_join<!BACK>(P, Q, pe, qe);
    if (quarter == 0) {
      float2* m = a.maps + (long long)u * d.B * d.D + bd;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        join[wave][cg][j] = make_float2(P[j], Q[j]);
        if (exists && at.has(j)) m[at.channel(j)] = make_float2(P[j], Q[j]);
      }
    }
    __syncthreads();
    if (threadIdx.x < 16) {
      float2* gm = a.group_maps + (long long)group * d.B * d.D + bd;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float p = 1.f, q = 0.f;
        for (int r = 0; r < GROUP; ++r) {  // (units that do not exist left the identity)
          const float2 w = join[r][cg][j];
          p *= w.x;
          q = fmaf(w.x, q, w.y);
        }
        if (at.has(j)) gm[at.channel(j)] = make_float2(p, q);
      }
    }
  };
  // Nearly every group is whole (all steps within the length, all channels there), and works without masks, paddings and their moves: 85 -> 69 us for the
  // application and 59 -> 56 for the maps of 65536 x 1024 (with closed gates exact, 70 and 57).  (A third form, for units behind a sequence's end, gained nothing.)
  if (columns >= CG * V && (group + 1) * GROUP <= a.units && len >= (BACK ? a.units - group * GROUP : (group + 1) * GROUP) * (long long)UNIT && has_x) unit(std::true_type{});
  else unit(std::false_type{});
}

// ---- step 2.  16 lanes of 4 channels x 16 rows a workgroup, as above; channels side by side (maps and states are the kernels' own: always aligned to
// their type, which is all that is asked for here).

// h = the maps [from, to) applied to h: each row joins a sixteenth of them, and every row then applies the sixteen
__device__ __forceinline__ void apply_range(const float2* maps, long long BD, unsigned from, unsigned to, const bool* has, const int* channel, float2 (*join)[CG][V],
                                            float* h) {
  const int cg = threadIdx.x & 15, row = threadIdx.x >> 4;
  const unsigned n = to - from, r0 = from + n * row / 16, r1 = from + n * (row + 1) / 16;
  float p[V], q[V];
#pragma unroll
  for (int j = 0; j < V; ++j) { p[j] = 1.f; q[j] = 0.f; }
#pragma unroll 4
  for (unsigned r = r0; r < r1; ++r)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 w = has[j] ? maps[r * BD + channel[j]] : make_float2(1.f, 0.f);
      p[j] *= w.x;
      q[j] = fmaf(w.x, q[j], w.y);
    }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) join[row][cg][j] = make_float2(p[j], q[j]);
  __syncthreads();
  for (int r = 0; r < 16; ++r)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 w = join[r][cg][j];
      h[j] = fmaf(w.x, h[j], w.y);
    }
}

__global__ __launch_bounds__(256) void scan_anchor_kernel(const ScanArgs a, const float* start) {
  __shared__ float2 join[16][CG][V];
  const int cg = threadIdx.x & 15, row = threadIdx.x >> 4, tile = blockIdx.x % a.tiles, b = blockIdx.x / a.tiles;
  const long long BD = (long long)a.d.B * a.d.D, bd = (long long)b * a.d.D;
  bool has[V];
  int channel[V];
  float h[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    channel[j] = (tile * CG + cg) * V + j;
    has[j] = channel[j] < a.d.D;
    h[j] = start && has[j] ? start[bd + channel[j]] : 0.f;
  }
  for (unsigned k = 1; k * ANCHOR < a.groups; ++k) {
    apply_range(a.group_maps + bd, BD, (k - 1) * ANCHOR, k * ANCHOR, has, channel, join, h);
    if (row == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (has[j]) a.anchors[(k - 1) * BD + bd + channel[j]] = h[j];
    }
  }
}

__global__ __launch_bounds__(256) void scan_states_kernel(const ScanArgs a, const float* start) {
  __shared__ float2 join[16][CG][V];
  const int cg = threadIdx.x & 15, row = threadIdx.x >> 4;
  const unsigned tile = blockIdx.x % a.tiles, rest = blockIdx.x / a.tiles, b = rest % a.d.B, group = rest / a.d.B, anchor = group / ANCHOR;
  const long long BD = (long long)a.d.B * a.d.D, bd = (long long)b * a.d.D;
  const unsigned u = group * GROUP + row;
  bool has[V];
  int channel[V];
  float h[V];
  float2 own[V];
  const float* from = anchor ? a.anchors + (anchor - 1) * BD : start;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    channel[j] = (tile * CG + cg) * V + j;
    has[j] = channel[j] < (unsigned)a.d.D;
    h[j] = from && has[j] ? from[bd + channel[j]] : 0.f;
    own[j] = u < a.units && has[j] ? a.maps[u * BD + bd + channel[j]] : make_float2(1.f, 0.f);
  }
  apply_range(a.group_maps + bd, BD, anchor * ANCHOR, group, has, channel, join, h);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < V; ++j) join[row][cg][j] = own[j];
  __syncthreads();
  for (int r = 0; r < row; ++r)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 w = join[r][cg][j];
      h[j] = fmaf(w.x, h[j], w.y);
    }
  if (u < a.units) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (has[j]) a.states[u * BD + bd + channel[j]] = h[j];
  }
}

// ---- step 3.  A workgroup takes a unit into registers: 16 segments of 4 steps, joined with lane exchanges inside a wave and through LDS between the four
// waves, so that a short sequence does not wait step by step.
template <int TYPE, bool WIDE>
__global__ __launch_bounds__(256, 5) void scan_fwd_kernel(const ScanArgs a) {
  constexpr int TS = UNIT / 16;
  __shared__ float2 wave_map[4][CG][V];
  const vmm_gated_scan_desc& d = a.d;
  const int cg = threadIdx.x & 15, seg = threadIdx.x >> 4, wave = threadIdx.x >> 6;
  const unsigned id = number(a, a.units * d.B * a.tiles);
  if (id >= a.units * d.B * a.tiles) return;
  const unsigned rest = uniform(id / a.tiles), tile = id - rest * a.tiles, turn = uniform(rest / d.B), b = rest - turn * d.B;
  const unsigned u = a.units - 1 - turn;  // from the end of time, where the maps were read last
  const long long first = (long long)u * UNIT;
  const int columns = d.D - (int)tile * CG * V;
  long long len = d.L;
  if (d.lengths) len = max(0LL, min((long long)d.lengths[b], len));
  const long long es = sizeof(typename Elem<TYPE>::T), bd = (long long)b * d.D + (long long)tile * CG * V;
  const auto row = [&](auto* p, int64_t batch, int64_t step, int k) { return p + (b * batch + (first + k) * step + (long long)tile * CG * V) * es; };
  const auto unit = [&](auto whole) {
    constexpr bool ALL = decltype(whole)::value;
    const Place<TYPE, WIDE> at(cg, ALL ? CG * V : columns);
    const int live = ALL ? UNIT : (int)min(max(len - first, 0LL), (long long)UNIT) - seg * TS, there = ALL ? UNIT : (int)min(d.L - first, (int64_t)UNIT) - seg * TS;
    const auto lane = [&](int64_t step) { return (seg * TS * (unsigned)step + at.d0) * (unsigned)es; };
    Raw<TYPE> x[TS], g[TS];
    const unsigned xl = lane(d.x_row), gl = lane(d.gate_row);
#pragma unroll
    for (int k = 0; k < TS; ++k) {
      x[k].u = fill_word<TYPE>(0u);
      g[k].u = fill_word<TYPE>(Elem<TYPE>::PAD);
      if (k < live) {
        x[k].u = at.load(row((const char*)d.x, d.x_batch, d.x_row, k), xl, 0u);
        g[k].u = at.load(row((const char*)d.gate, d.gate_batch, d.gate_row, k), gl, Elem<TYPE>::PAD);
      }
    }
    float h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = 0.f;
    if (a.units > 1) at.load_state(a.states + (long long)u * d.B * d.D + bd, h);
    else if (d.h0) at.load_state(d.h0 + bd, h);
    if (a.units == 1 && d.states && seg == 0) at.store_state(d.states + bd, h);  // (step 2 would have left it)

    float f[TS][V], q[TS][V], P[V], Q[V], pe[V], qe[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { P[j] = 1.f; Q[j] = 0.f; }
#pragma unroll
    for (int k = 0; k < TS; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float i;
        gate_of<TYPE>(g[k].get(j), f[k][j], i);
        q[k][j] = i * x[k].get(j);
        P[j] *= f[k][j];
        Q[j] = fmaf(f[k][j], Q[j], q[k][j]);
      }
    wave_join<true>(P, Q, pe, qe);
    if ((threadIdx.x & 48) == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) wave_map[wave][cg][j] = make_float2(P[j], Q[j]);
    }
    __syncthreads();  // (and every wave has read h0, which h_last may be)
    for (int w = 0; w < wave; ++w)
#pragma unroll
      for (int j = 0; j < V; ++j) h[j] = fmaf(wave_map[w][cg][j].x, h[j], wave_map[w][cg][j].y);
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = fmaf(pe[j], h[j], qe[j]);
    const unsigned yl = lane(d.y_row);
#pragma unroll
    for (int k = 0; k < TS; ++k) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[j] = fmaf(f[k][j], h[j], q[k][j]);
        o[j] = k < live ? h[j] : 0.f;
      }
      if (k < there) at.store(row((char*)d.y, d.y_batch, d.y_row, k), yl, o);
    }
    if (seg == 15 && u + 1 == a.units && d.h_last) at.store_state(d.h_last + bd, h);
  };
  if (columns >= CG * V && len - first >= UNIT) unit(std::true_type{});  // (as for the maps)
  else unit(std::false_type{});
}

// backward: h has to be known forwards and c backwards, so the segments are joined in both directions.  Three workgroups a CU: for four, 28 registers would
// have to go to scratch (8 x 4093 x 1000 bf16: 105 us, here 68).
template <int TYPE, bool WIDE>
__global__ __launch_bounds__(256, 3) void scan_bwd_kernel(const ScanArgs a) {
  constexpr int TS = UNIT / 16;
  __shared__ float2 wave_map[4][CG][V];
  __shared__ float wave_back[4][CG][V];
  const vmm_gated_scan_desc& d = a.d;
  const int cg = threadIdx.x & 15, seg = threadIdx.x >> 4, wave = threadIdx.x >> 6;
  const long long BD = (long long)d.B * d.D;
  const unsigned id = number(a, a.units * d.B * a.tiles);
  if (id >= a.units * d.B * a.tiles) return;
  const unsigned rest = uniform(id / a.tiles), tile = id - rest * a.tiles, u = uniform(rest / d.B), b = rest - u * d.B;
  const unsigned v = a.units - 1 - u;  // from the start of time (where the maps were read last), and in the direction of the walk
  const long long first = (long long)u * UNIT;
  const int columns = d.D - (int)tile * CG * V;
  long long len = d.L;
  if (d.lengths) len = max(0LL, min((long long)d.lengths[b], len));
  const long long es = sizeof(typename Elem<TYPE>::T), bd = (long long)b * d.D + (long long)tile * CG * V;
  const auto row = [&](auto* p, int64_t batch, int64_t step, int k) { return p + (b * batch + (first + k) * step + (long long)tile * CG * V) * es; };
  const auto unit = [&](auto whole) {
    constexpr bool ALL = decltype(whole)::value;
    const Place<TYPE, WIDE> at(cg, ALL ? CG * V : columns);
    const int live = ALL ? UNIT : (int)min(max(len - first, 0LL), (long long)UNIT) - seg * TS, there = ALL ? UNIT : (int)min(d.L - first, (int64_t)UNIT) - seg * TS;
    const auto lane = [&](int64_t step) { return (seg * TS * (unsigned)step + at.d0) * (unsigned)es; };
    Raw<TYPE> x[TS], g[TS], dy[TS];
    const unsigned xl = lane(d.x_row), gl = lane(d.gate_row), yl = lane(d.dy_row);
#pragma unroll
    for (int k = 0; k < TS; ++k) {
      x[k].u = dy[k].u = fill_word<TYPE>(0u);
      g[k].u = fill_word<TYPE>(Elem<TYPE>::PAD);
      if (k < live) {
        x[k].u = at.load(row((const char*)d.x, d.x_batch, d.x_row, k), xl, 0u);
        g[k].u = at.load(row((const char*)d.gate, d.gate_batch, d.gate_row, k), gl, Elem<TYPE>::PAD);
        if (d.dy) dy[k].u = at.load(row((const char*)d.dy, d.dy_batch, d.dy_row, k), yl, 0u);
      }
    }
    float h[V], back[V];
    at.load_state(d.states + u * BD + bd, h);
#pragma unroll
    for (int j = 0; j < V; ++j) back[j] = 0.f;
    if (a.units > 1) at.load_state(a.states + v * BD + bd, back);
    else if (d.dh_last) at.load_state(d.dh_last + bd, back);

    float f[TS][V], i[TS][V], P[V], Q[V], R[V], pf[V], qf[V], pb[V], rb[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { P[j] = 1.f; Q[j] = 0.f; R[j] = 0.f; }
#pragma unroll
    for (int k = 0; k < TS; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        gate_of<TYPE>(g[k].get(j), f[k][j], i[k][j]);
        P[j] *= f[k][j];
        Q[j] = fmaf(f[k][j], Q[j], i[k][j] * x[k].get(j));
      }
#pragma unroll
    for (int k = TS - 1; k >= 0; --k)
#pragma unroll
      for (int j = 0; j < V; ++j) R[j] = f[k][j] * (dy[k].get(j) + R[j]);
    wave_join_both(P, Q, R, pf, qf, pb, rb);
    if ((threadIdx.x & 48) == 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        wave_map[wave][cg][j] = make_float2(P[j], Q[j]);
        wave_back[wave][cg][j] = R[j];
      }
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w)  // the state in front of this wave
#pragma unroll
      for (int j = 0; j < V; ++j) h[j] = fmaf(wave_map[w][cg][j].x, h[j], wave_map[w][cg][j].y);
    for (int w = 3; w > wave; --w)  // and what the waves behind it hand on
#pragma unroll
      for (int j = 0; j < V; ++j) back[j] = fmaf(wave_map[w][cg][j].x, back[j], wave_back[w][cg][j]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      h[j] = fmaf(pf[j], h[j], qf[j]);
      back[j] = fmaf(pb[j], back[j], rb[j]);  // c_(t+1) of the segment's last step
    }
    float hx[TS][V];  // h_(t-1) - x_t, forwards
#pragma unroll
    for (int k = 0; k < TS; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xv = x[k].get(j);
        hx[k][j] = h[j] - xv;
        h[j] = fmaf(f[k][j], h[j], i[k][j] * xv);
      }
    const unsigned xo = lane(d.dx_row), go = lane(d.dgate_row);
#pragma unroll
    for (int k = TS - 1; k >= 0; --k) {
      float ox[V], og[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float dh = dy[k].get(j) + back[j], di = dh * i[k][j];
        ox[j] = k < live ? di : 0.f;
        og[j] = k < live ? di * f[k][j] * hx[k][j] : 0.f;
        back[j] = f[k][j] * dh;
      }
      if (k < there) {
        if (d.dx) at.store(row((char*)d.dx, d.dx_batch, d.dx_row, k), xo, ox);
        if (d.dgate) at.store(row((char*)d.dgate, d.dgate_batch, d.dgate_row, k), go, og);
      }
    }
    if (seg == 0 && u == 0 && d.dh0) at.store_state(d.dh0 + bd, back);
  };
  if (columns >= CG * V && len - first >= UNIT) unit(std::true_type{});
  else unit(std::false_type{});
}

inline int esize(int type) { return type == 0 ? 4 : 2; }
inline unsigned up8(unsigned n) { return (n + 7) / 8 * 8; }
inline long long up16(long long n) { return (n + 15) / 16 * 16; }

bool bad_rows(int64_t row) { return row < 0 || row >= (1LL << 23); }  // 64 rows are addressed with 32-bit byte offsets
bool bad_scan(const vmm_gated_scan_desc* d) {
  if (!d || d->B < 0 || d->D < 0 || d->L < 0 || d->L >= (1LL << 31) || d->type < 0 || d->type > 2 || (int64_t)d->B * d->D >= (1LL << 31) ||
         bad_rows(d->x_row) || bad_rows(d->gate_row) || bad_rows(d->y_row) || bad_rows(d->dy_row) || bad_rows(d->dx_row) || bad_rows(d->dgate_row))
    return true;
  // a launch has less than 2^32 threads: 256 a unit, 1024 a group
  const long long chains = (long long)d->B * ((d->D + CG * V - 1) / (CG * V)), units = (d->L + UNIT - 1) / UNIT;
  return chains * units > (1LL << 24) - 8 || (units > 1 && chains * ((units + GROUP - 1) / GROUP) > (1LL << 22) - 8);
}

struct Layout { unsigned units, groups; long long group_maps, anchors, states, bytes; };
Layout layout(const vmm_gated_scan_desc* d, bool backward) {
  Layout l = {};
  l.units = (unsigned)((d->L + UNIT - 1) / UNIT);
  l.groups = (l.units + GROUP - 1) / GROUP;
  if (l.units < 2) return l;
  const long long BD = (long long)d->B * d->D;
  l.group_maps = up16(8 * BD * l.units);
  l.anchors = l.group_maps + up16(8 * BD * l.groups);
  l.states = l.anchors + up16(4 * BD * ((l.groups - 1) / ANCHOR));
  l.bytes = l.states + (backward || !d->states ? up16(4 * BD * l.units) : 0);
  return l;
}

// accesses of four values to rows of D: addresses, strides and D itself have to allow them
bool wide(const void* p, int64_t batch, int64_t row, int D, int type) {
  return !p || (((uintptr_t)p & (V * esize(type) - 1)) == 0 && batch % V == 0 && row % V == 0 && D % V == 0);
}

template <int TYPE, bool WIDE>
int run(const ScanArgs& a, bool forward, hipStream_t s) {
  const unsigned chains = (unsigned)a.d.B * a.tiles;
  if (a.units > 1) {
    const float* start = forward ? a.d.h0 : a.d.dh_last;
    const unsigned blocks = chains * a.groups;
    if (forward) hipLaunchKernelGGL((scan_map_kernel<TYPE, WIDE, false>), dim3(up8(blocks)), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((scan_map_kernel<TYPE, WIDE, true>), dim3(up8(blocks)), dim3(1024), 0, s, a);
    VMM_LAUNCH_CHECK();
    if (a.groups > ANCHOR) {
      hipLaunchKernelGGL(scan_anchor_kernel, dim3(chains), dim3(256), 0, s, a, start);
      VMM_LAUNCH_CHECK();
    }
    hipLaunchKernelGGL(scan_states_kernel, dim3(blocks), dim3(256), 0, s, a, start);
    VMM_LAUNCH_CHECK();
  }
  if (forward) hipLaunchKernelGGL((scan_fwd_kernel<TYPE, WIDE>), dim3(up8(chains * a.units)), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((scan_bwd_kernel<TYPE, WIDE>), dim3(up8(chains * a.units)), dim3(256), 0, s, a);
  VMM_LAUNCH_CHECK();
  return 0;
}

int scan(const vmm_gated_scan_desc* d, bool forward, hipStream_t s) {
  const Layout l = layout(d, !forward);
  if (l.bytes > 0 && (!d->workspace || ((uintptr_t)d->workspace & 15) || d->workspace_bytes < l.bytes)) return -1;
  ScanArgs a = {};
  a.d = *d;
  a.tiles = (d->D + CG * V - 1) / (CG * V);
  a.units = l.units;
  a.groups = l.groups;
  a.runs = (d->x_row * esize(d->type)) % 128 != 0 || (d->gate_row * esize(d->type)) % 128 != 0;
  char* w = (char*)d->workspace;
  a.maps = (float2*)w;
  a.group_maps = (float2*)(w + l.group_maps);
  a.anchors = (float*)(w + l.anchors);
  a.states = forward && d->states ? d->states : (float*)(w + l.states);
  const auto ok = [&](const void* p, int64_t batch, int64_t row) { return wide(p, batch, row, d->D, d->type); };
  const bool w4 = ok(d->x, d->x_batch, d->x_row) && ok(d->gate, d->gate_batch, d->gate_row) &&
                  (forward ? ok(d->y, d->y_batch, d->y_row)
                           : ok(d->dy, d->dy_batch, d->dy_row) && ok(d->dx, d->dx_batch, d->dx_row) && ok(d->dgate, d->dgate_batch, d->dgate_row));
  switch (d->type * 2 + (w4 ? 1 : 0)) {
    case 0: return run<0, false>(a, forward, s);
    case 1: return run<0, true>(a, forward, s);
    case 2: return run<1, false>(a, forward, s);
    case 3: return run<1, true>(a, forward, s);
    case 4: return run<2, false>(a, forward, s);
    default: return run<2, true>(a, forward, s);
  }
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
  return (d->L + UNIT - 1) / UNIT * d->B * d->D;
}

extern "C" int64_t vmm_gated_scan_workspace(const vmm_gated_scan_desc* d, int32_t backward) {
  if (bad_scan(d)) return -1;
  return layout(d, backward != 0).bytes;
}

extern "C" int vmm_gated_scan(const vmm_gated_scan_desc* d, vmm_stream_t stream) {
  if (bad_scan(d)) return -1;
  const long long BD = (long long)d->B * d->D;
  if (BD == 0) return 0;
  if (d->L == 0) return pass(d->h0, d->h_last, BD, (hipStream_t)stream);
  if (!d->x || !d->gate || !d->y) return -1;
  return scan(d, true, (hipStream_t)stream);
}

extern "C" int vmm_gated_scan_bwd(const vmm_gated_scan_desc* d, vmm_stream_t stream) {
  if (bad_scan(d)) return -1;
  const long long BD = (long long)d->B * d->D;
  if (BD == 0) return 0;
  if (d->L == 0) return pass(d->dh_last, d->dh0, BD, (hipStream_t)stream);
  if (!d->x || !d->gate || !d->states) return -1;
  return scan(d, false, (hipStream_t)stream);
}
