// Layer norm over the last axis, forward and backward, with the reduction of the weight's
// and bias's gradients.
//
//   mean = sum(x) / d, var = sum((x - mean)^2) / d, rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd, y = xh w + b
//   backward, a = dy w: dx = rstd (a - mean(a) - xh mean(a xh)), dw = sum_rows dy xh,
//   db = sum_rows dy
//
// Memory bound: the forward reads x and writes y, the backward reads x and dy and writes dx.
// A row is held in registers by NT threads of E elements each, so it is read once; blocks
// walk over rows with the next row's loads issued before this row's reductions. A wave's
// residuals around its own mean give the variance and the mean's own rounding; waves are
// joined relative to the first one's mean (the base), and the mean is kept as base + delta
// (stats: base, delta, rstd), so an offset far above the spread costs no digits and a row
// takes one barrier. Weight and bias gradients are summed over a block's rows in registers (columns
// are fixed per thread), written as one partial row per block and added in block order by a
// second kernel: results are the same on every run.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "pd_common.hpp"

namespace pd {
namespace {

constexpr int LN_MAX_D = 16384;   // largest row held in registers
// Most threads of a launch that walks over rows: forward 16384 x 4096 bf16 67 us with half as
// many, 52, 53 with twice as many (60000 x 512 37, 25, 24). Where each block leaves a row of partial gradients and rows
// are long, half of that (backward 93 us, 105 with all; 30000 x 1024 41, 50; but 60000 x 512
// 43, 38).
constexpr int LN_THREADS = 256 * 1024;
constexpr int LN_GRAD_THREADS = 256 * 512;
constexpr int LN_GRAD_ALL_D = 512;

// Distances from the mean past 2^63 have squares past fp32: a row whose variance is infinite
// takes them again times this (sums of x itself end at 3.4 10^38).
constexpr float LN_WIDE = 0x1p-80f;
__device__ inline float ln_wide_rstd(float sum, float d, float eps) {
  return LN_WIDE / sqrtf(sum / d + eps * LN_WIDE * LN_WIDE);
}

struct LnStat {
  float base, delta, rstd;  // mean = base + delta
};

// 16 bytes of a row, at any element's boundary (the hardware takes them as one access), and
// kept packed in registers.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) LnWord {
  uint32_t v[4];
  __device__ inline float operator[](int e) const {
    if constexpr (sizeof(T) == 2) return __uint_as_float((e & 1) ? v[e >> 1] & 0xFFFF0000u : v[e >> 1] << 16);
    else return __uint_as_float(v[e]);
  }
};

// This thread's columns: word c covers columns VEC (tid + c NT) .. + VEC where those are
// below d, and threads 0, 1, .. have one column each behind the last whole word.
template <typename T, int NT, int CH>
__device__ inline void ln_load(const T* __restrict__ row, int tid, int d, LnWord<T> (&p)[CH], float& pt) {
  constexpr int VEC = 16 / sizeof(T);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = VEC * (tid + c * NT);
    if (col + VEC <= d) p[c] = *(const LnWord<T>*)(row + col);
    else p[c] = LnWord<T>{};
  }
  if (tid < d % VEC) pt = load_f<T>(row, d - d % VEC + tid);
}
template <typename T>
__device__ inline void ln_store(T* __restrict__ row, const float* v) {
  LnWord<T> p;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 2) p.v[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
    else p.v[e] = __float_as_uint(v[e]);
  }
  *(LnWord<T>*)row = p;
}
template <int VEC, int NT, int CH>
__device__ inline void ln_load_param(const float* __restrict__ w, float none, int tid, int d, float (&v)[CH * VEC],
                                     float& vt) {
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = VEC * (tid + c * NT);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[c * VEC + e] = w && col + VEC <= d ? w[col + e] : none;
  }
  vt = w && tid < d % VEC ? w[d - d % VEC + tid] : none;
}
// Sum over the NT threads of a row, or over the wave where a row has more.
template <int NT>
__device__ inline float ln_sum(float v) {
#pragma unroll
  for (int off = (NT < 64 ? NT : 64) / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Columns below d that wave w of the row holds (the row's all threads where it has one).
template <int VEC, int NT, int CH>
__device__ inline int ln_wave_count(int w, int d) {
  if (NT <= 64) return d;
  int n = 0;
#pragma unroll
  for (int c = 0; c < CH; ++c) n += min(max(d / VEC - (64 * w + c * NT), 0), 64) * VEC;
  return n + (w == 0 ? d % VEC : 0);
}
constexpr int ln_threads(int nt) { return nt <= 64 ? 256 : nt; }

// Forward. Grid: row groups; a block holds RPB rows at a time (NT <= 64: rows share waves or
// have one each, with no barrier). At the rate of a copy: 16384 x 4096 bf16 52 us, 5.1 TB/s.
template <typename T, int NT, int E>
__global__ __launch_bounds__(ln_threads(NT)) void k_ln_fwd(const T* __restrict__ x, int64_t rows, int d,
                                                           const float* __restrict__ w, const float* __restrict__ b,
                                                           float eps, T* __restrict__ y, LnStat* __restrict__ stats) {
  constexpr int VEC = 16 / sizeof(T), CH = E / VEC, RPB = ln_threads(NT) / NT, NW = NT <= 64 ? 1 : NT / 64;
  __shared__ float4 part[2][NW];
  __shared__ float again[NW];
  const int tid = threadIdx.x % NT, wv = tid >> 6, lane = threadIdx.x & 63;
  int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / NT;
  const int64_t step = (int64_t)gridDim.x * RPB;
  if (NT <= 64 && r >= rows) return;
  const bool tail = tid < d % VEC;
  float wr[E], br[E], wt, bt;
  ln_load_param<VEC, NT, CH>(w, 1.f, tid, d, wr, wt);
  ln_load_param<VEC, NT, CH>(b, 0.f, tid, d, br, bt);
  LnWord<T> cur[CH], nxt[CH];
  float vt = 0.f, nt = 0.f;
  ln_load<T, NT, CH>(x + r * d, tid, d, cur, vt);
  const int nw = ln_wave_count<VEC, NT, CH>(wv, d);
  for (int it = 0; r < rows; r += step, it ^= 1) {
    if (r + step < rows) ln_load<T, NT, CH>(x + (r + step) * d, tid, d, nxt, nt);
    float v[E], s = vt;
#pragma unroll
    for (int i = 0; i < E; ++i) s += v[i] = cur[i / VEC][i % VEC];
    s = ln_sum<NT>(s);
    float base = nw ? s / (float)nw : 0.f, res = tail ? vt - base : 0.f, q = res * res;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (VEC * (tid + (i / VEC) * NT) + VEC <= d) {
        const float t = v[i] - base;
        res += t;
        q = fmaf(t, t, q);
      }
    }
    q = ln_sum<NT>(q);
    res = ln_sum<NT>(res);
    float delta, var;
    if constexpr (NT <= 64) {
      delta = res / (float)d;
      var = fmaxf(q / (float)d - delta * delta, 0.f);
    } else {
      if (lane == 0) part[it][wv] = make_float4(base, res, q, (float)nw);
      __syncthreads();  // the other buffer is rewritten behind the next row's barrier
      base = part[it][0].x;
      delta = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) delta += fmaf(part[it][i].w, part[it][i].x - base, part[it][i].y);
      delta /= (float)d;
      float Q = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) {  // sum (t - u)^2 = q - 2 u res + n u^2, u = (base - own) + delta
        const float4 p = part[it][i];
        const float u = (base - p.x) + delta;
        if (p.w > 0.f) Q += p.z + u * fmaf(p.w, u, -2.f * p.y);
      }
      var = fmaxf(Q / (float)d, 0.f);
    }
    float rstd = 1.f / sqrtf(var + eps);
    if (var == INFINITY) {  // the same for the row's threads
      float t = tail ? ((vt - base) - delta) * LN_WIDE : 0.f, wide = t * t;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (VEC * (tid + (i / VEC) * NT) + VEC <= d) t = ((v[i] - base) - delta) * LN_WIDE, wide = fmaf(t, t, wide);
      wide = ln_sum<NT>(wide);
      if constexpr (NT > 64) {
        if (lane == 0) again[wv] = wide;
        __syncthreads();  // written anew behind a later row's barrier
        wide = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) wide += again[i];
      }
      rstd = ln_wide_rstd(wide, (float)d, eps);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = VEC * (tid + c * NT);
      if (col + VEC > d) continue;
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int i = c * VEC + e;
        o[e] = fmaf(((v[i] - base) - delta) * rstd, wr[i], br[i]);
      }
      ln_store<T>(y + r * d + col, o);
    }
    if (tail) store_f<T>(y + r * d, d - d % VEC + tid, fmaf(((vt - base) - delta) * rstd, wt, bt));
    if (stats && tid == 0) stats[r] = LnStat{base, delta, rstd};
#pragma unroll
    for (int c = 0; c < CH; ++c) cur[c] = nxt[c];
    vt = nt;
  }
}

// Backward. dwdb [gridDim.x][2][d]: each block's sums of dy xh and dy over its rows (NULL:
// not wanted). 16384 x 4096 bf16: 78 us without them, 5.2 TB/s; 93 with them and their
// reduction, where the sums' registers leave a CU fewer rows in flight.
template <typename T, int NT, int E>
__global__ __launch_bounds__(ln_threads(NT)) void k_ln_bwd(const T* __restrict__ x, const T* __restrict__ dy,
                                                           int64_t rows, int d, const float* __restrict__ w,
                                                           const LnStat* __restrict__ stats, T* __restrict__ dx,
                                                           float* __restrict__ dwdb) {
  constexpr int VEC = 16 / sizeof(T), CH = E / VEC, RPB = ln_threads(NT) / NT, NW = NT <= 64 ? 1 : NT / 64;
  __shared__ float2 part[2][NW];
  extern __shared__ float cols[];  // [2][d] where NT <= 64 and gradients are wanted
  const int tid = threadIdx.x % NT, wv = tid >> 6, lane = threadIdx.x & 63;
  int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / NT;
  const int64_t step = (int64_t)gridDim.x * RPB;
  const bool tail = tid < d % VEC;
  float wr[E], wt;
  ln_load_param<VEC, NT, CH>(w, 1.f, tid, d, wr, wt);
  float dw[E], db[E], dwt = 0.f, dbt = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) dw[i] = db[i] = 0.f;
  LnWord<T> cx[CH], cg[CH], nx[CH], ng[CH];
  float xt = 0.f, gt = 0.f, nxt = 0.f, ngt = 0.f;
  LnStat st = {}, nst = {};
  if (r < rows) {
    ln_load<T, NT, CH>(x + r * d, tid, d, cx, xt);
    ln_load<T, NT, CH>(dy + r * d, tid, d, cg, gt);
    st = stats[r];
  }
  const float invd = 1.f / (float)d;
  for (int it = 0; r < rows; r += step, it ^= 1) {
    if (r + step < rows) {
      ln_load<T, NT, CH>(x + (r + step) * d, tid, d, nx, nxt);
      ln_load<T, NT, CH>(dy + (r + step) * d, tid, d, ng, ngt);
      nst = stats[r + step];
    }
    const float xht = ((xt - st.base) - st.delta) * st.rstd, at = gt * wt;
    float s1 = 0.f, s2 = 0.f;
    if (tail) {
      s1 = at, s2 = at * xht;
      dwt = fmaf(gt, xht, dwt);
      dbt += gt;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float g = cg[i / VEC][i % VEC];
      const float xh = ((cx[i / VEC][i % VEC] - st.base) - st.delta) * st.rstd;
      if (VEC * (tid + (i / VEC) * NT) + VEC <= d) {
        const float a = g * wr[i];
        s1 += a;
        s2 = fmaf(a, xh, s2);
        dw[i] = fmaf(g, xh, dw[i]);
        db[i] += g;
      }
    }
    if (dx) {
      s1 = ln_sum<NT>(s1);
      s2 = ln_sum<NT>(s2);
      if constexpr (NT > 64) {
        if (lane == 0) part[it][wv] = make_float2(s1, s2);
        __syncthreads();
        s1 = s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) s1 += part[it][i].x, s2 += part[it][i].y;
      }
      const float m1 = s1 * invd, m2 = s2 * invd;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = VEC * (tid + c * NT);
        if (col + VEC > d) continue;
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int i = c * VEC + e;
          const float xh = ((cx[c][e] - st.base) - st.delta) * st.rstd;
          o[e] = st.rstd * (cg[c][e] * wr[i] - m1 - xh * m2);
        }
        ln_store<T>(dx + r * d + col, o);
      }
      if (tail) store_f<T>(dx + r * d, d - d % VEC + tid, st.rstd * (at - m1 - xht * m2));
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) cx[c] = nx[c], cg[c] = ng[c];
    xt = nxt, gt = ngt;
    st = nst;
  }
  if (!dwdb) return;
  float* dst = dwdb + (int64_t)blockIdx.x * 2 * d;
  if constexpr (NT <= 64) {  // the rows that share a wave, then the four waves' sums in order
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int off = 32; off >= NT; off >>= 1) dw[i] += __shfl_xor(dw[i], off, 64), db[i] += __shfl_xor(db[i], off, 64);
#pragma unroll
    for (int off = 32; off >= NT; off >>= 1) dwt += __shfl_xor(dwt, off, 64), dbt += __shfl_xor(dbt, off, 64);
    for (int wave = 0; wave < 4; ++wave) {
      if ((int)(threadIdx.x >> 6) == wave && lane < NT) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int word = VEC * (tid + (i / VEC) * NT), col = word + i % VEC;
          if (word + VEC <= d) {
            cols[col] = wave ? cols[col] + dw[i] : dw[i];
            cols[d + col] = wave ? cols[d + col] + db[i] : db[i];
          }
        }
        if (tail) {
          const int col = d - d % VEC + tid;
          cols[col] = wave ? cols[col] + dwt : dwt;
          cols[d + col] = wave ? cols[d + col] + dbt : dbt;
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * d; i += 256) dst[i] = cols[i];
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int word = VEC * (tid + (i / VEC) * NT), col = word + i % VEC;
      if (word + VEC <= d) dst[col] = dw[i], dst[d + col] = db[i];
    }
    if (tail) dst[d - d % VEC + tid] = dwt, dst[d + d - d % VEC + tid] = dbt;
  }
}

// dw, db = the partial rows [n][2][d] added in a fixed order: 16 columns by 64 slices of the
// rows per block, a slice's loads in batches of 8. n = 0 (no rows) gives zeros.
__global__ __launch_bounds__(1024) void k_ln_cols(const float* __restrict__ part, int n, int64_t d,
                                                  float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float red[16][17];
  const int c = threadIdx.x & 15, sl = threadIdx.x >> 4, wv = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 16 + c;
  const int per = (n + 63) / 64, lo = min(sl * per, n), hi = col < 2 * d ? min(lo + per, n) : lo;
  const float* p = part + col;
  float s = 0.f;
  for (int i = lo; i < hi; i += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < hi ? p[(i + j) * 2 * d] : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += v[j];
  }
  s += __shfl_xor(s, 16, 64);
  s += __shfl_xor(s, 32, 64);
  if ((threadIdx.x & 63) < 16) red[wv][c] = s;
  __syncthreads();
  if (threadIdx.x >= 16 || col >= 2 * d) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += red[i][c];
  float* out = col < d ? dw : db;
  if (out) out[col < d ? col : col - d] = s;
}

// ---------------------------------------------------------------- rows beyond the registers
// One block of 1024 threads per row; the row is read again for each of its passes.
__device__ inline float2 block_sum2(float a, float b, float2* red) {
  a = wave_sum(a), b = wave_sum(b);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(a, b);
  __syncthreads();
  a = b = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) a += red[i].x, b += red[i].y;
  return make_float2(a, b);
}

template <typename T>
__global__ __launch_bounds__(1024) void k_ln_fwd_long(const T* __restrict__ x, int64_t d, const float* __restrict__ w,
                                                      const float* __restrict__ b, float eps, T* __restrict__ y,
                                                      LnStat* __restrict__ stats) {
  __shared__ float2 red[16];
  const T* row = x + (int64_t)blockIdx.x * d;
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < d; i += 1024) s += load_f<T>(row, i);
  const float base = block_sum2(s, 0.f, red).x / (float)d;
  float q = 0.f, res = 0.f;
  for (int64_t i = threadIdx.x; i < d; i += 1024) {
    const float t = load_f<T>(row, i) - base;
    res += t;
    q = fmaf(t, t, q);
  }
  const float2 rq = block_sum2(res, q, red);
  const float delta = rq.x / (float)d;
  const float var = fmaxf(rq.y / (float)d - delta * delta, 0.f);
  float rstd = 1.f / sqrtf(var + eps);
  if (var == INFINITY) {
    float wide = 0.f;
    for (int64_t i = threadIdx.x; i < d; i += 1024) {
      const float t = ((load_f<T>(row, i) - base) - delta) * LN_WIDE;
      wide = fmaf(t, t, wide);
    }
    rstd = ln_wide_rstd(block_sum2(wide, 0.f, red).x, (float)d, eps);
  }
  for (int64_t i = threadIdx.x; i < d; i += 1024)
    store_f<T>(y + (int64_t)blockIdx.x * d, i,
               fmaf(((load_f<T>(row, i) - base) - delta) * rstd, w ? w[i] : 1.f, b ? b[i] : 0.f));
  if (stats && threadIdx.x == 0) stats[blockIdx.x] = LnStat{base, delta, rstd};
}

template <typename T>
__global__ __launch_bounds__(1024) void k_ln_dx_long(const T* __restrict__ x, const T* __restrict__ dy, int64_t d,
                                                     const float* __restrict__ w, const LnStat* __restrict__ stats,
                                                     T* __restrict__ dx) {
  __shared__ float2 red[16];
  const int64_t r = blockIdx.x;
  const LnStat st = stats[r];
  float s1 = 0.f, s2 = 0.f;
  for (int64_t i = threadIdx.x; i < d; i += 1024) {
    const float a = load_f<T>(dy + r * d, i) * (w ? w[i] : 1.f);
    s1 += a;
    s2 = fmaf(a, ((load_f<T>(x + r * d, i) - st.base) - st.delta) * st.rstd, s2);
  }
  const float2 s = block_sum2(s1, s2, red);
  const float m1 = s.x / (float)d, m2 = s.y / (float)d;
  for (int64_t i = threadIdx.x; i < d; i += 1024) {
    const float a = load_f<T>(dy + r * d, i) * (w ? w[i] : 1.f);
    store_f<T>(dx + r * d, i, st.rstd * (a - m1 - ((load_f<T>(x + r * d, i) - st.base) - st.delta) * st.rstd * m2));
  }
}

// Columns 256 blockIdx.x .. of slice blockIdx.y of the rows, into partial row blockIdx.y.
template <typename T>
__global__ __launch_bounds__(256) void k_ln_dw_long(const T* __restrict__ x, const T* __restrict__ dy, int64_t rows,
                                                    int64_t d, const LnStat* __restrict__ stats,
                                                    float* __restrict__ dwdb) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y, lo = per * blockIdx.y;
  const int64_t hi = lo + per < rows ? lo + per : rows;
  if (col >= d) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = lo; r < hi; ++r) {
    const float g = load_f<T>(dy, r * d + col);
    const LnStat st = stats[r];
    dw = fmaf(g, ((load_f<T>(x, r * d + col) - st.base) - st.delta) * st.rstd, dw);
    db += g;
  }
  dwdb[(int64_t)blockIdx.y * 2 * d + col] = dw;
  dwdb[(int64_t)blockIdx.y * 2 * d + d + col] = db;
}

constexpr int LN_LONG_SLICES = 16;

// Threads and elements a row is held in: the smallest of the built forms that covers d (a row
// in twice the threads, half of them idle: forward, backward of 16384 x 4096 bf16 52, 93 ->
// 90, 134 us; 100000 x 256 22, 32 -> 38, 43; one even case, the backward of 8192 x 8192: 106,
// 104). fp32 rows above 8192 spill 39 of the backward's registers and 7 of the forward's.
// F is called with (NT, E) as integral constants.
template <typename F>
void ln_form(int64_t d, F&& f) {
  using std::integral_constant;
  auto form = [&](auto nt) {
    constexpr int NT = decltype(nt)::value;
    f(nt, integral_constant<int, NT <= 64 ? 8 : 16>{});
  };
  if (d <= 64) form(integral_constant<int, 8>{});
  else if (d <= 128) form(integral_constant<int, 16>{});
  else if (d <= 256) form(integral_constant<int, 32>{});
  else if (d <= 512) form(integral_constant<int, 64>{});
  else if (d <= 1024) f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
  else if (d <= 2048) form(integral_constant<int, 128>{});
  else if (d <= 4096) form(integral_constant<int, 256>{});
  else if (d <= 8192) form(integral_constant<int, 512>{});
  else form(integral_constant<int, 1024>{});
}

// Blocks of a launch that walks over rows: `threads` threads in all at most, or a block a CU.
int64_t ln_blocks(int64_t rows, int64_t d, int64_t threads) {
  int64_t n = 0;
  ln_form(d, [&](auto nt, auto) {
    constexpr int NT = decltype(nt)::value;
    n = std::min(cdiv(rows, ln_threads(NT) / NT), std::max<int64_t>(threads / ln_threads(NT), 256));
  });
  return n;
}
int64_t ln_partials(int64_t rows, int64_t d) {
  if (d > LN_MAX_D) return rows < LN_LONG_SLICES ? rows : LN_LONG_SLICES;
  return ln_blocks(rows, d, d <= LN_GRAD_ALL_D ? LN_THREADS : LN_GRAD_THREADS);
}

int ln_check(const char* what, int dtype, int64_t rows, int64_t d, std::initializer_list<const void*> needed) {
  if (dtype != PD_DTYPE_F32 && dtype != PD_DTYPE_BF16)
    return fail(PD_EUNSUPPORTED, std::string(what) + ": dtype must be fp32 or bf16");
  if (rows < 0 || d <= 0) return fail(PD_EINVAL, std::string(what) + ": rows >= 0 and d >= 1");
  if (rows > 0x7FFFFFFF || d > 0x7FFFFFFF / 2) return fail(PD_EUNSUPPORTED, std::string(what) + ": rows or d too large");
  if (rows)
    for (const void* p : needed)
      if (!p) return fail(PD_EINVAL, std::string(what) + ": null pointer");
  return PD_OK;
}

template <typename T>
void ln_fwd(const T* x, int64_t rows, int64_t d, const float* w, const float* b, float eps, T* y, LnStat* stats,
            hipStream_t s) {
  if (d > LN_MAX_D) {
    hipLaunchKernelGGL(k_ln_fwd_long<T>, dim3((unsigned)rows), dim3(1024), 0, s, x, d, w, b, eps, y, stats);
    return;
  }
  const unsigned grid = (unsigned)ln_blocks(rows, d, LN_THREADS);
  ln_form(d, [&](auto nt, auto e) {
    constexpr int NT = decltype(nt)::value, E = decltype(e)::value;
    hipLaunchKernelGGL((k_ln_fwd<T, NT, E>), dim3(grid), dim3(ln_threads(NT)), 0, s, x, rows, (int)d, w, b, eps, y, stats);
  });
}

template <typename T>
void ln_bwd(const T* x, const T* dy, int64_t rows, int64_t d, const float* w, const LnStat* stats, T* dx, float* part,
            hipStream_t s) {
  if (d > LN_MAX_D) {
    if (dx) hipLaunchKernelGGL(k_ln_dx_long<T>, dim3((unsigned)rows), dim3(1024), 0, s, x, dy, d, w, stats, dx);
    if (part)
      hipLaunchKernelGGL(k_ln_dw_long<T>, dim3((unsigned)cdiv(d, 256), (unsigned)ln_partials(rows, d)), dim3(256), 0, s,
                         x, dy, rows, d, stats, part);
    return;
  }
  const unsigned grid = (unsigned)(part ? ln_partials(rows, d) : ln_blocks(rows, d, LN_THREADS));
  ln_form(d, [&](auto nt, auto e) {
    constexpr int NT = decltype(nt)::value, E = decltype(e)::value;
    const size_t lds = NT <= 64 && part ? (size_t)2 * d * sizeof(float) : 0;
    hipLaunchKernelGGL((k_ln_bwd<T, NT, E>), dim3(grid), dim3(ln_threads(NT)), lds, s, x, dy, rows, (int)d, w, stats, dx,
                       part);
  });
}

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" {

int pd_layer_norm_fwd(const void* x, int dtype, int64_t rows, int64_t d, const float* weight, const float* bias,
                      float eps, void* y, float* stats, void* stream) {
  if (int rc = ln_check("pd_layer_norm_fwd", dtype, rows, d, {x, y})) return rc;
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(PD_EINVAL, "pd_layer_norm_fwd: eps must be finite and >= 0");
  if (!rows) return PD_OK;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PD_DTYPE_F32) ln_fwd<float>((const float*)x, rows, d, weight, bias, eps, (float*)y, (LnStat*)stats, s);
  else ln_fwd<bf16_t>((const bf16_t*)x, rows, d, weight, bias, eps, (bf16_t*)y, (LnStat*)stats, s);
  return check_launch("pd_layer_norm_fwd");
}

size_t pd_layer_norm_bwd_workspace_size(int64_t rows, int64_t d) {
  if (rows <= 0 || d <= 0) return 0;
  return (size_t)ln_partials(rows, d) * 2 * (size_t)d * sizeof(float);
}

int pd_layer_norm_bwd(const void* x, const void* d_y, int dtype, int64_t rows, int64_t d, const float* weight,
                      const float* stats, void* d_x, float* d_weight, float* d_bias, void* workspace,
                      size_t workspace_bytes, void* stream) {
  if (int rc = ln_check("pd_layer_norm_bwd", dtype, rows, d, {x, d_y, stats})) return rc;
  const bool params = d_weight || d_bias;
  if (params && rows && (!workspace || workspace_bytes < pd_layer_norm_bwd_workspace_size(rows, d)))
    return fail(PD_EWORKSPACE, "pd_layer_norm_bwd: workspace");
  hipStream_t s = (hipStream_t)stream;
  float* part = params ? (float*)workspace : nullptr;
  if (rows && (d_x || params)) {
    if (dtype == PD_DTYPE_F32)
      ln_bwd<float>((const float*)x, (const float*)d_y, rows, d, weight, (const LnStat*)stats, (float*)d_x, part, s);
    else
      ln_bwd<bf16_t>((const bf16_t*)x, (const bf16_t*)d_y, rows, d, weight, (const LnStat*)stats, (bf16_t*)d_x, part, s);
  }
  if (params)
    hipLaunchKernelGGL(k_ln_cols, dim3((unsigned)cdiv(2 * d, 16)), dim3(1024), 0, s, part,
                       rows ? (int)ln_partials(rows, d) : 0, d, d_weight, d_bias);
  return check_launch("pd_layer_norm_bwd");
}

}  // extern "C"
