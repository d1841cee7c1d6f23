// The norms before and after a residual branch with its gate and scale, forward and backward.
//
//   rms(u) = u / sqrt(mean(u^2) + eps)
//   n = rms(b) post (or b),  h = x + scale gate n,  y = rms(h) pre
//   backward, from dh and dy: a = dy pre, hh = rms(h), rh = 1 / sqrt(mean(h^2) + eps)
//     dx = dh + rh (a - hh mean(a hh)),  dpre = sum_rows dy hh,  dgate = sum scale dx n
//     c = scale gate post, bh = rms(b): dpost = sum_rows scale gate dx bh,
//     db = rb (c dx - bh mean(c dx bh))
//
// Memory bound: the forward reads x and b and writes h and y, the backward reads dh, dy, h and b
// and writes dx and db. A row is held in registers by a team of NT threads, CH words of 8 columns
// each, so it is read once. mean(c dx bh) is linear in mean(a hh):
//   sum c bh (dh + rh a) - mean(a hh) sum c bh rh hh,
// so the backward reduces three sums behind one barrier instead of two after another.
// A team walks over a run of consecutive rows with the next row's loads issued before this
// row's sums. Runs end where a gate's group of rows ends or hold whole groups, so the gate of a
// group and its gradient stay in registers; gradients of shared parameters are written as one
// partial row a run (or wave) and added in a fixed order by a second kernel.
//
// Measured at 6 10^7 values, both streams and branch (bf16 and bf16; fp32 and fp32), a gate a sequence: forward
// 106-110 us and 199-224 us from 64 to 4096 columns (4.4-4.8 TB/s; 768 in bf16 123 us, a quarter of its lanes idle and the sums
// in 64 bits shown), backward with all gradients 156-164 us and 300-325 us (4.4-4.8 TB/s). Without a branch: forward 47-48 us
// (768: 61) and 103-115, backward 82-89 us (768: 104) and 152-161 (4.1-5.1 TB/s; 768 in bf16 3.5-3.9).
#include <algorithm>
#include <type_traits>

#include "pd_common.hpp"

namespace pd {
namespace {

constexpr int RN_MAX_D = 16384;  // largest row held in registers
// Rows whose squares leave fp32 are squared again: those past its end times RN_WIDE, and times RN_NEAR those below
// RN_LEAST, where squares are subnormal or nothing and eps does not hide it.
constexpr float RN_WIDE = 0x1p-80f, RN_NEAR = 0x1p80f, RN_LEAST = 0x1p-90f;

// 8 columns of a row as they are stored, loaded at any element's boundary (the hardware takes 16
// bytes as one access).
struct __attribute__((packed, aligned(2))) RnHalf8 {
  uint32_t v[4];
};
struct __attribute__((packed, aligned(4))) RnFloat4 {
  uint32_t v[4];
};
template <typename T>
struct RnWord {
  uint32_t v[sizeof(T) * 2];
  __device__ inline float operator[](int e) const {
    if constexpr (sizeof(T) == 2) return __uint_as_float((e & 1) ? v[e >> 1] & 0xFFFF0000u : v[e >> 1] << 16);
    else return __uint_as_float(v[e]);
  }
};
// Columns from d on are zero. `row` NULL: all are. The last columns of a row are a branch of their own: as the other
// side of the first one, lanes past the row would enter it, and the wait before its writes ends the loads ahead.
template <typename T>
__device__ inline RnWord<T> rn_load(const T* __restrict__ row, int col, int d) {
  RnWord<T> w;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) * 2); ++i) w.v[i] = 0u;
  if (!row) return w;
  if (col + 8 <= d) {
    if constexpr (sizeof(T) == 2) {
      const RnHalf8 p = *(const RnHalf8*)(row + col);
#pragma unroll
      for (int i = 0; i < 4; ++i) w.v[i] = p.v[i];
    } else {
      const RnFloat4 p = *(const RnFloat4*)(row + col), q = *(const RnFloat4*)(row + col + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) w.v[i] = p.v[i], w.v[4 + i] = q.v[i];
    }
  }
  if (col < d && col + 8 > d) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < d) {
        if constexpr (sizeof(T) == 2) w.v[e >> 1] |= (uint32_t)((const uint16_t*)row)[col + e] << (16 * (e & 1));
        else w.v[e] = ((const uint32_t*)row)[col + e];
      }
  }
  return w;
}
template <typename T>
__device__ inline void rn_store(T* __restrict__ row, int col, int d, const float (&v)[8]) {
  if (col + 8 <= d) {
    if constexpr (sizeof(T) == 2) {
      *(RnHalf8*)(row + col) = RnHalf8{{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                        pack_bf16x2(v[6], v[7])}};
    } else {
#pragma unroll
      for (int k = 0; k < 8; k += 4)
        *(RnFloat4*)(row + col + k) = RnFloat4{{__float_as_uint(v[k]), __float_as_uint(v[k + 1]),
                                                __float_as_uint(v[k + 2]), __float_as_uint(v[k + 3])}};
    }
  } else if (col < d) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < d) store_f<T>(row, col + e, v[e]);
  }
}

// The gate: kind 0 none, 1 one row of `gate` for each of `groups` runs of rows, 2 one for each row.
struct RnGate {
  const void* p;
  int bf16, kind;
  int64_t groups;
};
__device__ inline void rn_gate(const RnGate& g, int64_t group, int d, int col, float scale, float (&v)[8]) {
  if (g.kind == 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = scale;
  } else if (g.bf16) {
    const RnWord<bf16_t> w = rn_load<bf16_t>((const bf16_t*)g.p + group * d, col, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = scale * w[e];
  } else {
    const RnWord<float> w = rn_load<float>((const float*)g.p + group * d, col, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = scale * w[e];
  }
}

// Runs of rows: of `groups` groups of `per_group` rows each, either `slices` runs a group, or
// (slices 0) `run_groups` whole groups a run.
struct RnRuns {
  int64_t groups, per_group, slices, run_groups, runs;
  __host__ __device__ void rows(int64_t run, int64_t& lo, int64_t& hi) const {
    if (slices) {
      const int64_t g = run / slices, per = (per_group + slices - 1) / slices, at = (run % slices) * per;
      lo = g * per_group + (at < per_group ? at : per_group);
      hi = g * per_group + (at + per < per_group ? at + per : per_group);
    } else {
      lo = run * run_groups * per_group;
      const int64_t end = groups * per_group, to = lo + run_groups * per_group;
      hi = to < end ? to : end;
      if (lo > hi) lo = hi;
    }
  }
};

constexpr int rn_threads(int nt) { return nt <= 64 ? 256 : nt; }

// Sums over a team's threads; the other buffer of `part` is rewritten behind the next barrier.
template <int NT, int K>
__device__ inline void rn_sum(float (&s)[K], float (*part)[K], int tid) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int off = (NT < 64 ? NT : 64) / 2; off > 0; off >>= 1) s[k] += __shfl_xor(s[k], off, 64);
  if constexpr (NT > 64) {
    if ((tid & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) part[tid >> 6][k] = s[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k] += part[i][k];
  }
}

// 1 / sqrt(mean(u^2) + eps) of a row held in u.
template <int NT, int CH>
__device__ inline float rn_rstd(const float (&u)[CH][8], float d, float eps, float (*part)[1], int tid) {
  constexpr int NW = NT > 64 ? NT / 64 : 1;
  float s[1] = {0.f};
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[0] = fmaf(u[c][e], u[c][e], s[0]);
  rn_sum<NT, 1>(s, part, tid);
  const bool wide = s[0] == INFINITY;  // the same way for the team's threads
  if (!wide && !(fmaf(eps, d, s[0]) < RN_LEAST)) return 1.f / sqrtf(s[0] / d + eps);
  const float by = wide ? RN_WIDE : RN_NEAR;
  s[0] = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[0] = fmaf(u[c][e] * by, u[c][e] * by, s[0]);
  if constexpr (NT > 64) __syncthreads();
  rn_sum<NT, 1>(s, part + NW, tid);
  if constexpr (NT > 64) __syncthreads();
  return by / sqrtf(s[0] / d + eps * by * by);
}

// The same in 64 bits, from fp32 sums of two squares (each of bf16 values is exact): 1 neighbour of the right bf16 in
// 10^7 values of a stream, where fp32 sums of eight left 9 in 3.6 10^6, at the same time; squares in 64 bits leave none and
// cost the forward a quarter (4096 columns 106 -> 130 us). The root is fp32's with a Newton step.
template <int NT, int CH>
__device__ inline double rn_rstd_d(const float (&u)[CH][8], int d, float eps, double* part, float (*part_f)[1], int tid) {
  double t = 0.0;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const float lo = fmaf(u[c][e], u[c][e], u[c][e + 1] * u[c][e + 1]), hi = fmaf(u[c][e + 2], u[c][e + 2], u[c][e + 3] * u[c][e + 3]);
      t += (double)lo + (double)hi;
    }
#pragma unroll
  for (int off = (NT < 64 ? NT : 64) / 2; off > 0; off >>= 1) t += __shfl_xor(t, off, 64);
  if constexpr (NT > 64) {
    if ((tid & 63) == 0) part[tid >> 6] = t;
    __syncthreads();
    t = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) t += part[i];
  }
  // the same way for the team's threads
  if (!(t < (double)__FLT_MAX__ && t + (double)eps * d >= (double)RN_LEAST)) {
    if constexpr (NT > 64) __syncthreads();
    return (double)rn_rstd<NT, CH>(u, (float)d, eps, part_f, tid);
  }
  const double ms = t / (double)d + (double)eps;
  if (!(ms > 1e-30 && ms < 1e30)) return 1.0 / sqrt(ms);
  const double r = (double)(1.f / sqrtf((float)ms));
  return r * (1.5 - 0.5 * ms * r * r);
}
// To bf16 by way of fp32, as a cast does: the compiler may take the two conversions as one.
__device__ inline float rn_bf16(double v) {
  float f = (float)v;
  asm volatile("" : "+v"(f));
  return bf16_to_f32(f32_to_bf16(f));
}

struct RnFwd {
  const void *x, *b;  // b NULL: h = x, not written
  const float *post, *pre;
  int post_norm;
  float weight_offset, scale, eps;
  RnGate gate;
  void *h, *y;
  float* stats;  // [rows, 2]: 1 / rms of b (1 without its norm) and of h
  int d;
  RnRuns runs;
};

template <int CH>
__device__ inline void rn_param(const float* __restrict__ w, float off, int tid, int nt, int d, float (&v)[CH][8]) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = 8 * (tid + c * nt);
    const RnWord<float> p = rn_load<float>(w, col, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[c][e] = w ? p[e] + off : 1.f;
  }
}

template <typename TX, typename TB, int NT, int CH>
__global__ __launch_bounds__(rn_threads(NT)) void k_rn_fwd(RnFwd a) {
  constexpr int NW = NT > 64 ? NT / 64 : 1, TEAMS = rn_threads(NT) / NT;
  __shared__ float part[4][2 * NW][1];
  __shared__ double part_d[2][NW];
  const int tid = threadIdx.x % NT, d = a.d;
  const int64_t run = (int64_t)blockIdx.x * TEAMS + threadIdx.x / NT;
  if (run >= a.runs.runs) return;  // whole teams; with NT > 64 none
  int64_t lo, hi;
  a.runs.rows(run, lo, hi);
  const TX* x = (const TX*)a.x;
  const TB* b = (const TB*)a.b;
  // A bf16 stream is formed in 64 bits and rounded from there: y and the gradients go on from what
  // is stored, and a neighbour of the right bf16 would move them by far more than their own roundings (in
  // fp32 99 of 3.6 10^6 values were one).
  constexpr bool ONCE = sizeof(TX) == 2;
  constexpr bool AHEAD = NT < 1024;  // the next row's loads before this row's sums, where registers are left for it
  typedef std::conditional_t<ONCE, double, float> TF;
  float pre[CH][8], post[CH][8];
  TF factor[CH][8];  // scale gate post
  rn_param<CH>(a.pre, a.weight_offset, tid, NT, d, pre);
  rn_param<CH>(a.post, a.weight_offset, tid, NT, d, post);
  const int64_t per = a.gate.kind == 2 ? 1 : a.runs.per_group;
  int64_t left = 0;  // rows until the gate changes
  RnWord<TX> xc[CH], xn[CH];
  RnWord<TB> bc[CH], bn[CH];
  auto load = [&](int64_t r, RnWord<TX>(&xw)[CH], RnWord<TB>(&bw)[CH]) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = 8 * (tid + c * NT);
      xw[c] = rn_load<TX>(x + r * d, col, d);
      bw[c] = rn_load<TB>(b ? b + r * d : nullptr, col, d);
    }
  };
  if (lo < hi) load(lo, xc, bc);
  for (int64_t r = lo, it = 0; r < hi; ++r, it ^= 1) {
    if constexpr (AHEAD) {
      if (r + 1 < hi) load(r + 1, xn, bn);
    } else if (r > lo) load(r, xc, bc);
    if (left == 0) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float g[8];
        rn_gate(a.gate, r / per, d, 8 * (tid + c * NT), 1.f, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) factor[c][e] = (TF)a.scale * (TF)g[e] * (TF)post[c][e];
      }
      left = per - r % per;
    }
    --left;
    float u[CH][8];
    TF rb = (TF)1;
    if (b) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) u[c][e] = bc[c][e];
      if (a.post_norm) {
        if constexpr (ONCE) rb = rn_rstd_d<NT, CH>(u, d, a.eps, part_d[it], part[2 * it], tid);
        else rb = rn_rstd<NT, CH>(u, (float)d, a.eps, part[2 * it], tid);
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (ONCE) u[c][e] = rn_bf16(fma(factor[c][e] * rb, (double)u[c][e], (double)xc[c][e]));
          else u[c][e] = fmaf(factor[c][e], u[c][e] * rb, xc[c][e]);
        }
        rn_store<TX>((TX*)a.h + r * d, 8 * (tid + c * NT), d, u[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) u[c][e] = xc[c][e];
    }
    const float rh = rn_rstd<NT, CH>(u, (float)d, a.eps, part[2 * it + 1], tid);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[c][e] = u[c][e] * rh * pre[c][e];
      rn_store<TB>((TB*)a.y + r * d, 8 * (tid + c * NT), d, u[c]);
    }
    if (a.stats && tid == 0) *(float2*)(a.stats + 2 * r) = make_float2((float)rb, rh);
    if constexpr (AHEAD) {
#pragma unroll
      for (int c = 0; c < CH; ++c) xc[c] = xn[c], bc[c] = bn[c];
    }
  }
}

struct RnBwd {
  const void *h, *b, *dh, *dy;  // b, dh, dy NULL: none
  const float *post, *pre;
  int post_norm;
  float weight_offset, scale;
  RnGate gate;
  const float* stats;
  void *dx, *db;     // NULL: not wanted
  float* dpar;       // [slots][2][d]: partial dpost and dpre (NULL: neither is wanted)
  void* dgate;       // gate's type, where a run holds whole groups of it (or it has a row for each)
  float* dgate_part; // [runs][d] otherwise
  float* means;      // [rows]: mean(a hh) for k_rn_cols
  int d;
  RnRuns runs;
};

// SUMS: the gradients of gate and weights with it (else k_rn_cols's).
template <typename TX, typename TB, int NT, int CH, bool SUMS>
__global__ __launch_bounds__(rn_threads(NT)) void k_rn_bwd(RnBwd a) {
  constexpr int NW = NT > 64 ? NT / 64 : 1, TEAMS = rn_threads(NT) / NT;
  __shared__ float part[2][NW][3];
  const int tid = threadIdx.x % NT, d = a.d;
  const int64_t run = (int64_t)blockIdx.x * TEAMS + threadIdx.x / NT;
  int64_t lo = 0, hi = 0;
  if (run < a.runs.runs) a.runs.rows(run, lo, hi);
  const TX *h = (const TX*)a.h, *dh = (const TX*)a.dh;
  const TB *b = (const TB*)a.b, *dy = (const TB*)a.dy;
  float pre[CH][8], post[CH][8], gate[CH][8], dpre[CH][8], dpost[CH][8], dgate[CH][8];
  rn_param<CH>(a.pre, a.weight_offset, tid, NT, d, pre);
  rn_param<CH>(a.post, a.weight_offset, tid, NT, d, post);
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) dpre[c][e] = dpost[c][e] = dgate[c][e] = 0.f;
  const int64_t per = a.gate.kind == 2 ? 1 : a.runs.per_group;
  const bool want_gate = a.dgate || a.dgate_part;
  const float invd = 1.f / (float)d;
  int64_t left = 0;
  RnWord<TX> hc[CH], hn[CH], gc[CH], gn[CH];  // h and dh
  RnWord<TB> bc[CH], bn[CH], yc[CH], yn[CH];  // b and dy
  float2 st = make_float2(1.f, 1.f), stn = st;
  auto load = [&](int64_t r, RnWord<TX>(&hw)[CH], RnWord<TX>(&gw)[CH], RnWord<TB>(&bw)[CH], RnWord<TB>(&yw)[CH],
                  float2& s) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = 8 * (tid + c * NT);
      hw[c] = rn_load<TX>(h + r * d, col, d);
      gw[c] = rn_load<TX>(dh ? dh + r * d : nullptr, col, d);
      bw[c] = rn_load<TB>(b ? b + r * d : nullptr, col, d);
      yw[c] = rn_load<TB>(dy ? dy + r * d : nullptr, col, d);
    }
    s = *(const float2*)(a.stats + 2 * r);
  };
  if (lo < hi) load(lo, hc, gc, bc, yc, st);
  for (int64_t r = lo, it = 0; r < hi; ++r, it ^= 1) {
    if constexpr (SUMS) {
      if (r + 1 < hi) load(r + 1, hn, gn, bn, yn, stn);
    } else if (r > lo) load(r, hc, gc, bc, yc, st);
    if (left == 0) {
#pragma unroll
      for (int c = 0; c < CH; ++c) rn_gate(a.gate, r / per, d, 8 * (tid + c * NT), a.scale, gate[c]);
      left = per - r % per;
    }
    --left;
    const float rb = a.post_norm ? st.x : 1.f, rh = st.y;
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float hh = hc[c][e] * rh, ga = yc[c][e] * pre[c][e], cb = gate[c][e] * post[c][e] * (bc[c][e] * rb);
        s[0] = fmaf(ga, hh, s[0]);
        s[1] = fmaf(cb, fmaf(rh, ga, gc[c][e]), s[1]);
        s[2] = fmaf(cb, rh * hh, s[2]);
        if constexpr (SUMS) dpre[c][e] = fmaf(yc[c][e], hh, dpre[c][e]);
      }
    rn_sum<NT, 3>(s, part[it], tid);
    const float m1 = s[0] * invd, m2 = a.post_norm ? (s[1] - m1 * s[2]) * invd : 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = 8 * (tid + c * NT);
      float dx[8], db[8], dg[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float hh = hc[c][e] * rh, bh = bc[c][e] * rb;
        dx[e] = fmaf(rh, fmaf(-hh, m1, yc[c][e] * pre[c][e]), gc[c][e]);
        const float dn = gate[c][e] * dx[e];
        if constexpr (SUMS) {
          dpost[c][e] = fmaf(dn, bh, dpost[c][e]);
          dg[e] = a.scale * dx[e] * (bh * post[c][e]);
        }
        db[e] = rb * fmaf(-bh, m2, dn * post[c][e]);
      }
      if (a.dx) rn_store<TX>((TX*)a.dx + r * d, col, d, dx);
      if (a.db) rn_store<TB>((TB*)a.db + r * d, col, d, db);
      if (SUMS && want_gate) {
#pragma unroll
        for (int e = 0; e < 8; ++e) dgate[c][e] += dg[e];
        if (left == 0 && !a.dgate_part) {
          if (a.gate.bf16) rn_store<bf16_t>((bf16_t*)a.dgate + r / per * d, col, d, dgate[c]);
          else rn_store<float>((float*)a.dgate + r / per * d, col, d, dgate[c]);
#pragma unroll
          for (int e = 0; e < 8; ++e) dgate[c][e] = 0.f;
        }
      }
    }
    if (!SUMS && a.means && tid == 0) a.means[r] = m1;
    if constexpr (SUMS) {
#pragma unroll
      for (int c = 0; c < CH; ++c) hc[c] = hn[c], gc[c] = gn[c], bc[c] = bn[c], yc[c] = yn[c];
      st = stn;
    }
  }
  if constexpr (!SUMS) return;
  if (a.dgate_part && run < a.runs.runs) {
#pragma unroll
    for (int c = 0; c < CH; ++c) rn_store<float>(a.dgate_part + run * d, 8 * (tid + c * NT), d, dgate[c]);
  }
  if (!a.dpar) return;
  // teams that share a wave are added over it; one partial row a wave, or a team of several
  const int64_t slot = NT <= 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if constexpr (NT < 64) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int off = 32; off >= NT; off >>= 1) {
          dpost[c][e] += __shfl_xor(dpost[c][e], off, 64);
          dpre[c][e] += __shfl_xor(dpre[c][e], off, 64);
        }
    }
    if ((threadIdx.x & 63) < NT || NT > 64) {
      rn_store<float>(a.dpar + slot * 2 * d, 8 * (tid + c * NT), d, dpost[c]);
      rn_store<float>(a.dpar + slot * 2 * d + d, 8 * (tid + c * NT), d, dpre[c]);
    }
  }
}

// The gradients of gate and weights of rows wider than k_rn_bwd has registers for beside its own: a block takes
// 2048 columns of a run and forms dx again from the row's mean. It reads the row's four inputs a second time; with the
// sums held by k_rn_bwd, in scratch then, both took 399 us at 8192 columns and 1177 us at 16384 (6 10^7 values in
// bf16), apart 278 and 542 us.
template <typename TX, typename TB>
__global__ __launch_bounds__(256) void k_rn_cols(RnBwd a) {
  const int d = a.d, col = 8 * ((int)blockIdx.x * 256 + (int)threadIdx.x);
  if (col >= d) return;
  const int64_t run = blockIdx.y;
  int64_t lo, hi;
  a.runs.rows(run, lo, hi);
  const TX *h = (const TX*)a.h, *dh = (const TX*)a.dh;
  const TB *b = (const TB*)a.b, *dy = (const TB*)a.dy;
  const RnWord<float> pw = rn_load<float>(a.pre, col, d), qw = rn_load<float>(a.post, col, d);
  float gate[8], dpre[8], dpost[8], dgate[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dpre[e] = dpost[e] = dgate[e] = 0.f;
  const int64_t per = a.gate.kind == 2 ? 1 : a.runs.per_group;
  const bool want_gate = a.dgate || a.dgate_part;
  int64_t left = 0;
  for (int64_t r = lo; r < hi; ++r) {
    const RnWord<TX> hw = rn_load<TX>(h + r * d, col, d), gw = rn_load<TX>(dh ? dh + r * d : nullptr, col, d);
    const RnWord<TB> bw = rn_load<TB>(b ? b + r * d : nullptr, col, d), yw = rn_load<TB>(dy ? dy + r * d : nullptr, col, d);
    const float2 st = *(const float2*)(a.stats + 2 * r);
    const float m1 = a.means[r], rb = a.post_norm ? st.x : 1.f, rh = st.y;
    if (left == 0) {
      rn_gate(a.gate, r / per, d, col, a.scale, gate);
      left = per - r % per;
    }
    --left;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float pre = a.pre ? pw[e] + a.weight_offset : 1.f, post = a.post ? qw[e] + a.weight_offset : 1.f;
      const float hh = hw[e] * rh, bh = bw[e] * rb, dx = fmaf(rh, fmaf(-hh, m1, yw[e] * pre), gw[e]);
      dpre[e] = fmaf(yw[e], hh, dpre[e]);
      dpost[e] = fmaf(gate[e] * dx, bh, dpost[e]);
      dgate[e] = fmaf(a.scale * dx, bh * post, dgate[e]);
    }
    if (want_gate && left == 0 && !a.dgate_part) {
      if (a.gate.bf16) rn_store<bf16_t>((bf16_t*)a.dgate + r / per * d, col, d, dgate);
      else rn_store<float>((float*)a.dgate + r / per * d, col, d, dgate);
#pragma unroll
      for (int e = 0; e < 8; ++e) dgate[e] = 0.f;
    }
  }
  if (a.dgate_part) rn_store<float>(a.dgate_part + run * d, col, d, dgate);
  if (!a.dpar) return;
  rn_store<float>(a.dpar + run * 2 * d, col, d, dpost);
  rn_store<float>(a.dpar + run * 2 * d + d, col, d, dpre);
}

// Sums of n partial rows of `cols` values in a fixed order: a block's 16 waves take a slice of the rows
// each, 64 columns. A job for the parameters (columns dpost | dpre) and one for each group of the gate. (16 columns
// by 64 slices a block, the gates' few partials among them: 16 us at d = 4096 with 16 gates.)
struct RnSums {
  const float* par;
  int64_t par_n;
  float *dpost, *dpre;
  const float* gate;
  int64_t gate_n;
  void* dgate;
  int gate_bf16;
  int64_t d;
};
__global__ __launch_bounds__(1024) void k_rn_sums(RnSums a) {
  __shared__ float red[16][64];
  const int c = threadIdx.x & 63, sl = threadIdx.x >> 6;
  const bool gates = a.gate && (int64_t)blockIdx.y >= (a.par ? 1 : 0);
  const int64_t group = (int64_t)blockIdx.y - (a.par ? 1 : 0);
  const int64_t cols = gates ? a.d : 2 * a.d, n = gates ? a.gate_n : a.par_n;
  if ((int64_t)blockIdx.x * 64 >= cols) return;
  const int64_t col = (int64_t)blockIdx.x * 64 + c;
  const int64_t per = (n + 15) / 16, lo = sl * per < n ? sl * per : n;
  const int64_t hi = col < cols ? (lo + per < n ? lo + per : n) : lo;
  const float* p = (gates ? a.gate + group * n * cols : a.par) + col;
  float s = 0.f;
  for (int64_t i = lo; i < hi; i += 16) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = i + j < hi ? p[(i + j) * cols] : 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s += v[j];
  }
  red[sl][c] = s;
  __syncthreads();
  if (sl || col >= cols) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += red[i][c];
  if (gates) {
    if (a.gate_bf16) store_f<bf16_t>((bf16_t*)a.dgate, group * a.d + col, s);
    else ((float*)a.dgate)[group * a.d + col] = s;
  } else {
    float* out = col < a.d ? a.dpost : a.dpre;
    if (out) out[col < a.d ? col : col - a.d] = s;
  }
}

// The team a row is held by: the fewest threads that cover it.
template <typename F>
void rn_form(int64_t d, F&& f) {
  using std::integral_constant;
  const integral_constant<int, 1> one;
  const integral_constant<int, 2> two;
  if (d <= 64) f(integral_constant<int, 8>{}, one);
  else if (d <= 128) f(integral_constant<int, 16>{}, one);
  else if (d <= 256) f(integral_constant<int, 32>{}, one);
  else if (d <= 512) f(integral_constant<int, 64>{}, one);
  else if (d <= 1024) f(integral_constant<int, 128>{}, one);
  else if (d <= 2048) f(integral_constant<int, 256>{}, one);
  else if (d <= 4096) f(integral_constant<int, 512>{}, one);
  else if (d <= 8192) f(integral_constant<int, 512>{}, two);
  else f(integral_constant<int, 1024>{}, two);
}

constexpr int64_t RN_THREADS = 256 * 1024;
constexpr int64_t RN_SUMS_D = 4096;  // widest rows whose sums k_rn_bwd holds
constexpr int64_t RN_COL_RUNS = 256;

// Runs for so many teams.
RnRuns rn_team_runs(int64_t rows, int64_t groups, int64_t teams) {
  RnRuns r;
  r.groups = groups, r.per_group = rows / groups;
  if (teams >= groups) {
    r.slices = std::min(teams / groups, r.per_group);
    r.slices = cdiv(r.per_group, cdiv(r.per_group, r.slices));  // none of them empty
    r.run_groups = 0;
    r.runs = groups * r.slices;
  } else {
    r.slices = 0;
    r.run_groups = cdiv(groups, teams);
    r.runs = cdiv(groups, r.run_groups);
  }
  return r;
}
// The runs of a launch of at most `threads` threads (or a block a CU).
RnRuns rn_runs(int64_t rows, int64_t groups, int64_t d, int64_t threads) {
  int64_t teams = 1;
  rn_form(d, [&](auto nt, auto) {
    constexpr int NT = decltype(nt)::value;
    teams = std::max<int64_t>(threads / NT, 256);
  });
  return rn_team_runs(rows, groups, teams);
}

template <typename F>
void rn_types(int xdt, int bdt, F&& f) {
  if (xdt == PD_DTYPE_BF16) f((bf16_t*)nullptr, (bf16_t*)nullptr);
  else if (bdt == PD_DTYPE_BF16) f((float*)nullptr, (bf16_t*)nullptr);
  else f((float*)nullptr, (float*)nullptr);
}

int rn_check(const char* what, int x_dtype, int b_dtype, int64_t rows, int64_t d, int post_norm, const void* post_weight,
             const void* gate, int gate_dtype, int64_t groups, float scale) {
  if ((x_dtype != PD_DTYPE_F32 && x_dtype != PD_DTYPE_BF16) || (b_dtype != PD_DTYPE_F32 && b_dtype != PD_DTYPE_BF16) ||
      (x_dtype == PD_DTYPE_BF16 && b_dtype == PD_DTYPE_F32))
    return fail(PD_EUNSUPPORTED, std::string(what) + ": stream and branch are bf16, fp32, or an fp32 stream with a bf16 branch");
  if (rows < 0 || d <= 0) return fail(PD_EINVAL, std::string(what) + ": rows >= 0 and d >= 1");
  if (rows > 0x7FFFFFFF || d > RN_MAX_D) return fail(PD_EUNSUPPORTED, std::string(what) + ": rows or d too large");
  if (gate && gate_dtype != PD_DTYPE_F32 && gate_dtype != PD_DTYPE_BF16)
    return fail(PD_EUNSUPPORTED, std::string(what) + ": the gate is fp32 or bf16");
  if (!post_norm && post_weight) return fail(PD_EINVAL, std::string(what) + ": a weight of a norm that is not there");
  if (rows && gate && (groups <= 0 || rows % groups))
    return fail(PD_EINVAL, std::string(what) + ": the gate's rows divide the rows");
  if (!std::isfinite(scale)) return fail(PD_EINVAL, std::string(what) + ": scale must be finite");
  return PD_OK;
}

RnGate rn_make_gate(const void* gate, int dtype, int64_t groups, int64_t rows) {
  // one row for all rows is a group too, also where there is only one row
  return RnGate{gate, dtype == PD_DTYPE_BF16, !gate ? 0 : groups == rows && rows > 1 ? 2 : 1, groups};
}
// Groups that runs have to keep apart.
int64_t rn_groups(const RnGate& g) { return g.kind == 1 ? g.groups : 1; }

struct RnPlan {
  RnRuns runs, col_runs;
  int64_t slots;
  bool cols, gate_part;
  size_t par_bytes, gate_bytes, total;
};
RnPlan rn_plan(int64_t rows, int64_t d, int64_t groups, bool params, bool dgate, bool full_gate) {
  RnPlan P;
  if (full_gate) groups = 1;
  P.cols = d > RN_SUMS_D && (params || dgate);
  P.runs = rn_runs(rows, groups, d, RN_THREADS / 2);
  P.col_runs = rn_team_runs(rows, groups, RN_COL_RUNS);
  int64_t blocks = 0;
  rn_form(d, [&](auto nt, auto) {
    constexpr int NT = decltype(nt)::value;
    blocks = cdiv(P.runs.runs, rn_threads(NT) / NT);
    P.slots = NT <= 64 ? blocks * 4 : blocks;
  });
  const RnRuns& sums = P.cols ? P.col_runs : P.runs;
  if (P.cols) P.slots = sums.runs;
  P.gate_part = dgate && !full_gate && sums.slices > 1;
  P.par_bytes = params ? ((size_t)P.slots * 2 * d * 4 + 255) & ~(size_t)255 : 0;
  P.gate_bytes = P.gate_part ? ((size_t)sums.runs * d * 4 + 255) & ~(size_t)255 : 0;
  P.total = P.par_bytes + P.gate_bytes + (P.cols ? (size_t)rows * 4 : 0);
  return P;
}

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" {

int pd_residual_norm_fwd(const void* x, int x_dtype, const void* branch, int branch_dtype, int64_t rows, int64_t d,
                         int post_norm, const float* post_weight, const void* gate, int gate_dtype,
                         int64_t gate_rows, float scale, const float* pre_weight, float weight_offset, float eps,
                         void* stream_out, void* y, float* stats, void* stream) {
  const char* what = "pd_residual_norm_fwd";
  if (int rc = rn_check(what, x_dtype, branch_dtype, rows, d, post_norm, post_weight, gate, gate_dtype, gate_rows, scale)) return rc;
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(PD_EINVAL, std::string(what) + ": eps must be finite and >= 0");
  if (rows && (!x || !y || (branch && !stream_out))) return fail(PD_EINVAL, std::string(what) + ": null pointer");
  if (!rows) return PD_OK;
  RnFwd a{x, branch, post_weight, pre_weight, post_norm, weight_offset, scale, eps,
          rn_make_gate(branch ? gate : nullptr, gate_dtype, gate_rows, rows), stream_out, y, stats, (int)d, {}};
  a.runs = rn_runs(rows, rn_groups(a.gate), d, RN_THREADS);
  rn_types(x_dtype, branch_dtype, [&](auto tx, auto tb) {
    typedef std::remove_pointer_t<decltype(tx)> TX;
    typedef std::remove_pointer_t<decltype(tb)> TB;
    rn_form(d, [&](auto nt, auto ch) {
      constexpr int NT = decltype(nt)::value, CH = decltype(ch)::value;
      hipLaunchKernelGGL((k_rn_fwd<TX, TB, NT, CH>), dim3((unsigned)cdiv(a.runs.runs, rn_threads(NT) / NT)),
                         dim3(rn_threads(NT)), 0, (hipStream_t)stream, a);
    });
  });
  return check_launch(what);
}

size_t pd_residual_norm_bwd_workspace_size(int64_t rows, int64_t d, int64_t gate_rows, int want_weights,
                                           int want_gate) {
  if (rows <= 0 || d <= 0 || d > RN_MAX_D || (gate_rows > 0 && rows % gate_rows)) return 0;
  const bool full = gate_rows == rows && rows > 1;
  return rn_plan(rows, d, gate_rows > 0 ? gate_rows : 1, want_weights, want_gate && gate_rows > 0, full).total;
}

int pd_residual_norm_bwd(const void* stream_out, int x_dtype, const void* branch, int branch_dtype, int64_t rows,
                         int64_t d, int post_norm, const float* post_weight, const void* gate, int gate_dtype,
                         int64_t gate_rows, float scale, const float* pre_weight, float weight_offset,
                         const float* stats, const void* d_stream, const void* d_y, void* d_x, void* d_branch,
                         float* d_post, void* d_gate, float* d_pre, void* workspace, size_t workspace_bytes,
                         void* stream) {
  const char* what = "pd_residual_norm_bwd";
  if (int rc = rn_check(what, x_dtype, branch_dtype, rows, d, post_norm, post_weight, gate, gate_dtype, gate_rows, scale)) return rc;
  if (rows && (!stream_out || !stats)) return fail(PD_EINVAL, std::string(what) + ": null pointer");
  if ((d_branch || d_post || d_gate) && rows && !branch) return fail(PD_EINVAL, std::string(what) + ": gradients of a branch that is not there");
  if (d_gate && !gate) return fail(PD_EINVAL, std::string(what) + ": the gradient of a gate that is not there");
  const bool params = d_post || d_pre;
  hipStream_t s = (hipStream_t)stream;
  if (!rows) {  // sums over no rows
    if (params) {
      const RnSums z{(const float*)(d_post ? d_post : d_pre), 0, d_post, d_pre, nullptr, 0, nullptr, 0, d};
      hipLaunchKernelGGL(k_rn_sums, dim3((unsigned)cdiv(2 * d, 64)), dim3(1024), 0, s, z);
    }
    return check_launch(what);
  }
  RnBwd a{stream_out, branch, d_stream, d_y, post_weight, pre_weight, post_norm, weight_offset, scale,
          rn_make_gate(branch ? gate : nullptr, gate_dtype, gate_rows, rows), stats, d_x, d_branch, nullptr, d_gate, nullptr,
          nullptr, (int)d, {}};
  const RnPlan P = rn_plan(rows, d, rn_groups(a.gate), params, d_gate != nullptr, a.gate.kind == 2);
  if (P.total && (!workspace || workspace_bytes < P.total)) return fail(PD_EWORKSPACE, std::string(what) + ": workspace");
  a.runs = P.runs;
  if (params) a.dpar = (float*)workspace;
  if (P.gate_part) a.dgate_part = (float*)((char*)workspace + P.par_bytes), a.dgate = nullptr;
  if (P.cols) a.means = (float*)((char*)workspace + P.par_bytes + P.gate_bytes);
  rn_types(x_dtype, branch_dtype, [&](auto tx, auto tb) {
    typedef std::remove_pointer_t<decltype(tx)> TX;
    typedef std::remove_pointer_t<decltype(tb)> TB;
    rn_form(d, [&](auto nt, auto ch) {
      constexpr int NT = decltype(nt)::value, CH = decltype(ch)::value;
      hipLaunchKernelGGL((k_rn_bwd<TX, TB, NT, CH, (NT * CH * 8 <= RN_SUMS_D)>),
                         dim3((unsigned)cdiv(a.runs.runs, rn_threads(NT) / NT)), dim3(rn_threads(NT)), 0, s, a);
    });
    if (P.cols) {
      a.runs = P.col_runs;
      hipLaunchKernelGGL((k_rn_cols<TX, TB>), dim3((unsigned)cdiv(d, 2048), (unsigned)P.col_runs.runs), dim3(256), 0, s, a);
    }
  });
  if (params || P.gate_part) {
    const RnSums z{a.dpar, P.slots, d_post, d_pre, a.dgate_part, (P.cols ? P.col_runs : P.runs).slices, d_gate, gate_dtype == PD_DTYPE_BF16, d};
    hipLaunchKernelGGL(k_rn_sums, dim3((unsigned)cdiv(params ? 2 * d : d, 64),
                                       (unsigned)((params ? 1 : 0) + (P.gate_part ? P.runs.groups : 0))),
                       dim3(1024), 0, s, z);
  }
  return check_launch(what);
}

}  // extern "C"
