// Routing of rows to experts by scores: softmax or sigmoid, a bias that only the choice sees,
// limited groups, the k best, weights renormalised or not; and the logits' gradient.
//
//   s = softmax(x) or 1 / (1 + e^-x),  key = s + bias
//   group score = the sum of its two best keys; the top_groups best groups stay
//   idx = the k best keys of those, best first, the lower index first among equals
//   w = scale s[idx] (/ sum s[idx]);   renormalised sigmoids as softmax(log s[idx]), so that small
//   ones do not underflow together
//
// The choice is that of 64-bit scores. A row is held by a team of NT lanes, 8 (or 16) experts a lane, and
// each round takes the team's largest key. Keys are 32-bit words whose order is that of fp32
// scores, with the expert's place in its lane in the low bits; a second look is needed only where
// neighbours among the chosen (or the best of the rest) are closer than fp32 tells apart, and such a
// row is chosen again from 64-bit scores. Without bias and groups the logits' own order decides:
// exact in 32 bits, and for bf16 logits the word holds the whole index, so equal logits need no second look.
// Bound by the rounds' vector instructions rather than by memory: several rows share a wave. Measured: 131072 x 128, 8
// chosen by softmax, fp32: forward 48 us (70 with words compared one by one and every close row chosen again; reading
// the logits is 14), backward 28 (4.8 TB/s); 8192 x 256, sigmoid with bias, 4 of 8 groups, bf16: 28 and 8.4.
#include <algorithm>
#include <cmath>

#include "pd_common.hpp"

namespace pd {
namespace {

constexpr int RT_MAX_E = 1024, RT_MAX_K = 64, RT_MAX_GROUPS = 64;
constexpr int64_t RT_MAX_T = (((int64_t)1 << 24) - 1) * 4;  // a launch has fewer than 2^32 threads; the widest rows are four to a block

struct RtArgs {
  const void* x;
  int64_t T;
  int E, k;
  int sigmoid;
  const float* bias;
  int groups, top_groups;
  int renorm;
  float scale;
  float* w;
  int32_t* idx;
};

// 8 logits at any element's boundary.
struct __attribute__((packed, aligned(2))) RtHalf8 {
  uint16_t v[8];
};
struct __attribute__((packed, aligned(4))) RtFloat4 {
  float v[4];
};
template <typename T, int J>
__device__ inline void rt_load(const T* __restrict__ row, int e0, int E, float (&x)[J]) {
#pragma unroll
  for (int c = 0; c < J; c += 8) {
    if (e0 + c + 8 <= E) {
      if constexpr (sizeof(T) == 2) {
        const RtHalf8 h = *(const RtHalf8*)(row + e0 + c);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[c + i] = bf16_to_f32(h.v[i]);
      } else {
        const RtFloat4 a = *(const RtFloat4*)(row + e0 + c), b = *(const RtFloat4*)(row + e0 + c + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[c + i] = a.v[i], x[c + 4 + i] = b.v[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[c + i] = e0 + c + i < E ? load_f<T>(row, e0 + c + i) : -INFINITY;
    }
  }
}

// ---------------------------------------------------------------- over a team's NT lanes
template <int CTRL>
__device__ inline uint32_t rt_dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
// Folds v over the team with f, a commutative and associative step; every lane gets the result.
template <int NT, typename F>
__device__ inline uint32_t rt_fold(uint32_t v, F&& f) {
  static_assert(NT == 8 || NT == 16 || NT == 32 || NT == 64, "team");
  v = f(v, rt_dpp<0xB1>(v));   // lanes 1, 0, 3, 2 of a quad
  v = f(v, rt_dpp<0x4E>(v));   // 2, 3, 0, 1
  v = f(v, rt_dpp<0x141>(v));  // the other quad of 8 lanes
  if constexpr (NT > 8) v = f(v, rt_dpp<0x140>(v));  // the other 8 of 16
  if constexpr (NT > 16) {  // each 16 lanes beside the next 16, then each 32
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(p[0], p[1]);
  }
  if constexpr (NT > 32) {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = f(p[0], p[1]);
  }
  return v;
}
template <int NT>
__device__ inline uint32_t rt_max_u(uint32_t v) {
  return rt_fold<NT>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int NT>
__device__ inline uint32_t rt_add_u(uint32_t v) {
  return rt_fold<NT>(v, [](uint32_t a, uint32_t b) { return a + b; });
}
template <int NT>
__device__ inline float rt_max(float v) {
  return __uint_as_float(rt_fold<NT>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
template <int NT>
__device__ inline float rt_add(float v) {
  return __uint_as_float(rt_fold<NT>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
template <int NT>
__device__ inline double rt_add_d(double v) {
#pragma unroll
  for (int off = NT / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// LDS between the lanes of one wave: what was written before is seen behind it.
__device__ inline void rt_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Words in the order of floats (both zeros the same); 0 is below all.
__device__ inline uint32_t rt_order(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ inline float rt_unorder(uint32_t u) {
  return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

template <int NT, typename D>
__device__ inline D rt_least(D v) {
#pragma unroll
  for (int off = NT / 2; off > 0; off >>= 1) {
    const D o = __shfl_xor(v, off, 64);
    v = o < v ? o : v;
  }
  return v;
}

// The groups that stay, as bits: the lanes' keys go through LDS and lane g takes the two best of
// group g. A masked expert (key -inf) adds nothing. `low` and `high`: the score of the last group
// that stays and of the first that does not (-inf: none).
template <int NT, int J, typename D>
__device__ inline uint64_t rt_groups(const RtArgs& a, const D (&key)[J], D* lds, int lane, D& low, D& high) {
  constexpr int Q = (RT_MAX_GROUPS + NT - 1) / NT;
#pragma unroll
  for (int j = 0; j < J; ++j) lds[lane * J + j] = key[j];
  rt_wave_sync();
  const int size = a.E / a.groups;
  D score[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int g = lane + q * NT;
    D b1 = (D)-INFINITY, b2 = (D)-INFINITY;
    if (g < a.groups)
      for (int i = 0; i < size; ++i) {
        const D v = lds[g * size + i];
        if (v > b1) b2 = b1, b1 = v;
        else if (v > b2) b2 = v;
      }
    score[q] = b2 > (D)-INFINITY ? b1 + b2 : b1;
  }
  rt_wave_sync();
#pragma unroll
  for (int q = 0; q < Q; ++q)
    if (lane + q * NT < a.groups) lds[lane + q * NT] = score[q];
  rt_wave_sync();
  uint32_t lo = 0, hi = 0;  // the bits of this lane's groups
  low = (D)INFINITY, high = (D)INFINITY;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int g = lane + q * NT;
    if (g < a.groups) {
      int rank = 0;
      for (int o = 0; o < a.groups; ++o) {
        const D other = lds[o];
        rank += other > score[q] || (other == score[q] && o < g);
      }
      if (rank < a.top_groups) {
        if (g < 32) lo |= 1u << g;
        else hi |= 1u << (g - 32);
        low = score[q] < low ? score[q] : low;
      } else {
        high = -score[q] < high ? -score[q] : high;
      }
    }
  }
  rt_wave_sync();
  low = rt_least<NT, D>(low);
  high = -rt_least<NT, D>(high);
  auto either = [](uint32_t x, uint32_t y) { return x | y; };
  lo = rt_fold<NT>(lo, either);
  if (a.groups > 32) hi = rt_fold<NT>(hi, either);
  return ((uint64_t)hi << 32) | lo;
}

// The choice from 64-bit scores of the row's logits xs (in LDS): indices into won[r].y.
template <int NT, int J>
__device__ __noinline__ void rt_choose_wide(const RtArgs& a, const float* xs, int lane, double* lds, uint2* won) {
  double key[J];
  float x[J];
#pragma unroll
  for (int j = 0; j < J; ++j) x[j] = xs[lane * J + j];
  const bool raw = !a.bias && a.groups == 1;
  if (!raw && !a.sigmoid) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; ++j) m = fmaxf(m, x[j]);
    m = rt_max<NT>(m);
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) s += key[j] = x[j] == -INFINITY ? 0.0 : exp((double)x[j] - (double)m);
    s = rt_add_d<NT>(s);
#pragma unroll
    for (int j = 0; j < J; ++j) key[j] /= s;
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = lane * J + j;
    double v = raw ? (double)x[j] : a.sigmoid ? 1.0 / (1.0 + exp(-(double)x[j])) : key[j];
    if (a.bias && e < a.E) v += (double)a.bias[e];
    if (v != v) v = INFINITY;  // a NaN is chosen: it shows in the weights
    key[j] = x[j] == -INFINITY ? -INFINITY : v;
  }
  uint32_t gone = 0;  // experts chosen, behind the last, or of groups that do not stay
#pragma unroll
  for (int j = 0; j < J; ++j) gone |= (uint32_t)(lane * J + j >= a.E) << j;
  if (a.groups > 1) {
    double low, high;
    const uint64_t stay = rt_groups<NT, J, double>(a, key, lds, lane, low, high);
    const int size = a.E / a.groups;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (lane * J + j < a.E) gone |= (uint32_t)(!((stay >> ((lane * J + j) / size)) & 1)) << j;
  }
  for (int r = 0; r < a.k; ++r) {
    double best = 0.0;
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (!((gone >> j) & 1) && (at == 0x7FFFFFFF || key[j] > best)) best = key[j], at = lane * J + j;
#pragma unroll
    for (int off = NT / 2; off > 0; off >>= 1) {
      const double v = __shfl_xor(best, off, 64);
      const int o = __shfl_xor(at, off, 64);
      if (o != 0x7FFFFFFF && (at == 0x7FFFFFFF || v > best || (v == best && o < at))) best = v, at = o;
    }
    if (at / J == lane) gone |= 1u << (at % J);
    if (lane == 0) won[r].y = (uint32_t)at;
  }
}

// The order of n candidates won[i] (words and their lanes' first experts) by the scores that rt_choose_wide compares: the
// k best of them into won[r].y. Each lane ranks its candidates against all.
template <int NT, int J>
__device__ __noinline__ void rt_rank_wide(const RtArgs& a, const float* xs, int lane, int n, double* lds, uint2* won) {
  double m = 0.0, total = 1.0;
  const bool raw = !a.bias && a.groups == 1;
  if (!raw && !a.sigmoid) {
    float top = -INFINITY;
    for (int j = 0; j < J; ++j) top = fmaxf(top, xs[lane * J + j]);
    m = (double)rt_max<NT>(top);
    total = 0.0;
    for (int j = 0; j < J; ++j) total += exp((double)xs[lane * J + j] - m);
    total = rt_add_d<NT>(total);
  }
  int32_t* order = (int32_t*)(lds + RT_MAX_K);
  for (int i = lane; i < n; i += NT) {
    const int e = (int)(won[i].y + (J - 1 - (won[i].x & (J - 1))));
    const double v = (double)xs[e];
    // scores, not logits: those of unequal logits may be equal, and the lower index is first then
    double key = raw ? v : a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - m) / total;
    if (a.bias) key += (double)a.bias[e];
    lds[i] = v == -INFINITY ? v : key;  // masked, whatever its bias
    won[i].y = (uint32_t)e;
  }
  rt_wave_sync();
  for (int i = lane; i < n; i += NT) {
    const double mine = lds[i];
    const uint32_t e = won[i].y;
    int rank = 0;
    for (int o = 0; o < n; ++o) {
      const double other = lds[o];
      rank += other > mine || (other == mine && won[o].y < e);
    }
    order[rank] = (int32_t)e;
  }
  rt_wave_sync();
  for (int r = lane; r < a.k; r += NT) won[r].y = (uint32_t)order[r];
}

__device__ inline void rt_swap(uint32_t& a, uint32_t& b) {  // the larger first
  const uint32_t hi = a > b ? a : b, lo = a > b ? b : a;
  a = hi, b = lo;
}
// A lane's words in falling order (Batcher's odd-even merge network).
template <int J>
__device__ inline void rt_sort(uint32_t (&v)[J]) {
#pragma unroll
  for (int p = 1; p < J; p *= 2)
#pragma unroll
    for (int k = p; k > 0; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < J; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < J && (i + j) / (2 * p) == (i + j + k) / (2 * p)) rt_swap(v[i + j], v[i + j + k]);
}

// Whether the lane's group stays, where each lane's experts are of one group and a group has a
// power of two of lanes: the two best keys are merged over its lanes.
template <int NT, int J>
__device__ inline bool rt_lane_group(const RtArgs& a, const float (&key)[J], float* lds, int lane, float& low, float& high) {
  const int lanes = a.E / a.groups / J, mine = lane / lanes;
  float b1 = key[0], b2 = -INFINITY;
#pragma unroll
  for (int j = 1; j < J; ++j) {
    b2 = fmaxf(b2, fminf(b1, key[j]));
    b1 = fmaxf(b1, key[j]);
  }
  for (int off = 1; off < lanes; off *= 2) {
    const float o1 = __shfl_xor(b1, off, 64), o2 = __shfl_xor(b2, off, 64);
    b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
    b1 = fmaxf(b1, o1);
  }
  const float score = b2 > -INFINITY ? b1 + b2 : b1;
  const bool in = mine < a.groups;
  if (in) lds[mine] = score;
  rt_wave_sync();
  int rank = 0;
  for (int o = 0; o < a.groups; ++o) {
    const float other = lds[o];
    rank += other > score || (other == score && o < mine);
  }
  rt_wave_sync();
  const bool stays = in && rank < a.top_groups;
  low = -rt_max<NT>(stays ? -score : -INFINITY);
  high = rt_max<NT>(in && !stays ? score : -INFINITY);
  return stays;
}

template <typename T, int NT, int J>
__global__ __launch_bounds__(256, J > 8 ? 4 : 8) void k_rt_fwd(RtArgs a) {
  constexpr int TEAMS = 256 / NT, SPAN = NT * J < RT_MAX_GROUPS ? RT_MAX_GROUPS : NT * J;
  constexpr uint32_t LOW = J - 1;
  constexpr bool WHOLE = sizeof(T) == 2;  // whether a word without bias and groups holds the index
  __shared__ float rows[TEAMS][SPAN];
  __shared__ double wides[4][SPAN + RT_MAX_K / 2];        // one a wave: its teams take the second look in turn
  __shared__ uint2 wons[TEAMS][RT_MAX_K];  // words chosen and their lanes' first expert
  const int lane = threadIdx.x % NT, team = threadIdx.x / NT;
  const int64_t row = (int64_t)blockIdx.x * TEAMS + team;
  if (row >= a.T) return;  // whole teams; nothing below waits for the block
  const T* xr = (const T*)a.x + row * a.E;
  const int e0 = lane * J;
  float* xs = rows[team];
  uint2* won = wons[team];
  float x[J];
  rt_load<T, J>(xr, e0, a.E, x);
  const bool raw = !a.bias && a.groups == 1;
  bool again = false;
  uint32_t key[J];
  float smax = 1.f, m = -INFINITY, total = 0.f;
  if (!a.sigmoid) {
#pragma unroll
    for (int j = 0; j < J; ++j) m = fmaxf(m, x[j]);
    m = rt_max<NT>(m);
#pragma unroll
    for (int j = 0; j < J; ++j) total += __expf(x[j] - m);
    total = rt_add<NT>(total);
  }
  if (raw) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if constexpr (WHOLE) {
        const uint32_t u = x[j] != x[j] ? 0xFFFF0000u : rt_order(x[j]) & 0xFFFF0000u;
        key[j] = u | (uint32_t)(0xFFFF - (e0 + j));
      } else {
        key[j] = (rt_order(x[j]) & ~LOW) | (LOW - j);
        again |= x[j] != x[j];
      }
    }
  } else {
    float s[J];
    if (a.sigmoid) {
#pragma unroll
      for (int j = 0; j < J; ++j) s[j] = __builtin_amdgcn_rcpf(1.f + __expf(-x[j]));
    } else {
      smax = 1.f / total;
#pragma unroll
      for (int j = 0; j < J; ++j) s[j] = __expf(x[j] - m) * smax;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (a.bias && e0 + j < a.E) s[j] += a.bias[e0 + j];
      again |= !(fabsf(s[j]) < INFINITY);
      if (x[j] == -INFINITY) s[j] = -INFINITY;
    }
    const int size = a.E / a.groups;
    uint32_t stay = ~0u;  // bits of the lane's experts
    if (a.groups > 1) {
      float low, high;
      const int lanes = size / J;
      if (size % J == 0 && (lanes & (lanes - 1)) == 0) {
        stay = rt_lane_group<NT, J>(a, s, xs, lane, low, high) ? ~0u : 0u;
      } else {
        const uint64_t groups = rt_groups<NT, J, float>(a, s, xs, lane, low, high);
        stay = 0u;
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (e0 + j < a.E) stay |= (uint32_t)((groups >> ((e0 + j) / size)) & 1) << j;
      }
      again |= high > -INFINITY && !(low - high > 3e-6f * smax + 5e-7f * fmaxf(fabsf(low), fabsf(high)));
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      key[j] = s[j] == -INFINITY ? LOW + 1u : rt_order(s[j]);
      key[j] = (stay >> j) & 1 ? (key[j] & ~LOW) | (LOW - j) : 0u;
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (e0 + j >= a.E) key[j] = 0u;
  rt_sort<J>(key);
  uint32_t wins = 0;
  for (int r = 0; r < a.k; ++r) {
    const uint32_t M = rt_max_u<NT>(key[0]);
    if (key[0] == M) {
      won[r] = make_uint2(M, (uint32_t)e0);
      ++wins;
#pragma unroll
      for (int j = 0; j + 1 < J; ++j) key[j] = key[j + 1];
      key[J - 1] = 0u;
    }
  }
  uint32_t rest = rt_max_u<NT>(key[0]);
#pragma unroll
  for (int j = 0; j < J; ++j) xs[e0 + j] = x[j];  // the row's logits beside the choice
  rt_wave_sync();
  bool ranked = false;  // whether won[r].y is the choice itself
  if (!(raw && WHOLE)) {
    // whether 64 bits may order two words the other way round
    auto close = [&](uint32_t hi, uint32_t lo) {
      if (raw) return (hi & ~LOW) == (lo & ~LOW);
      if (lo <= LOW + 1u + LOW) return lo != 0u && hi <= LOW + 1u + LOW;  // masked: equal to its like, behind all others
      const float f = rt_unorder(hi & ~LOW), g = rt_unorder(lo & ~LOW);
      return !(f - g > 1.5e-6f * smax + (J * 1.2e-7f + 5e-7f) * fmaxf(fabsf(f), fabsf(g)));
    };
    // the rest that may belong to the k best joins them
    int n = a.k;
    const uint32_t last = won[a.k - 1].x;
    while (rest && close(last, rest)) {
      if (n == RT_MAX_K) {
        again = true;
        break;
      }
      if (key[0] == rest) {
        won[n] = make_uint2(rest, (uint32_t)e0);
        ++wins;
#pragma unroll
        for (int j = 0; j + 1 < J; ++j) key[j] = key[j + 1];
        key[J - 1] = 0u;
      }
      ++n;
      rest = rt_max_u<NT>(key[0]);
    }
    rt_wave_sync();
    bool look = n > a.k;
    for (int r = lane; r + 1 < a.k; r += NT) look |= close(won[r].x, won[r + 1].x);
    again |= rt_add_u<NT>(wins) != (uint32_t)n;
    const uint32_t flags = rt_fold<NT>((again ? 2u : 0u) | (look ? 1u : 0u), [](uint32_t p, uint32_t q) { return p | q; });
    ranked = flags != 0u;
    if (__ballot(ranked)) {
      for (int t = 0; t < 64 / NT; ++t) {
        if (ranked && team % (64 / NT) == t) {
          if (flags & 2u) rt_choose_wide<NT, J>(a, xs, lane, wides[threadIdx.x >> 6], won);
          else rt_rank_wide<NT, J>(a, xs, lane, n, wides[threadIdx.x >> 6], won);
        }
        rt_wave_sync();
      }
    }
  }
  auto chosen = [&](int r) {
    const uint2 w = won[r];
    return ranked ? (int)w.y : raw && WHOLE ? (int)(0xFFFFu - (w.x & 0xFFFFu)) : (int)(w.y + (LOW - (w.x & LOW)));
  };
  float* wout = a.w + row * a.k;
  int32_t* iout = a.idx + row * a.k;
  uint32_t live = 0;  // whether one is not masked
  if (a.sigmoid) {
    float sum = 0.f;
    uint32_t faint = 0;  // a score that leaves fp32, whose weight may not
    for (int r = lane; r < a.k; r += NT) {
      const int e = chosen(r);
      const float s = 1.f / (1.f + expf(-xs[e]));
      won[r] = make_uint2(__float_as_uint(s), (uint32_t)e);
      sum += s;
      faint |= s < 0x1p-100f && xs[e] != -INFINITY;
    }
    float by = a.scale;
    if (a.renorm) {
      sum = rt_add<NT>(sum);
      faint = rt_fold<NT>(faint, [](uint32_t p, uint32_t q) { return p | q; });
      if (sum < 0x1p-60f || faint) {  // the same for the team: by their logarithms
        float lmax = -INFINITY, total = 0.f;
        for (int r = lane; r < a.k; r += NT) {
          const float v = xs[won[r].y], l = fminf(v, 0.f) - log1pf(expf(-fabsf(v)));
          won[r].x = __float_as_uint(l);
          live |= v != -INFINITY;
          lmax = fmaxf(lmax, l);
        }
        lmax = rt_max<NT>(lmax);
        for (int r = lane; r < a.k; r += NT) {
          const float e = expf(__uint_as_float(won[r].x) - lmax);
          won[r].x = __float_as_uint(e);
          total += e;
        }
        total = rt_add<NT>(total);
        if (!rt_fold<NT>(live, [](uint32_t p, uint32_t q) { return p | q; })) {  // all are masked
          for (int r = lane; r < a.k; r += NT) won[r].x = 0u;
          total = 1.f;
        }
        sum = total;
      }
      by /= sum;
    }
    for (int r = lane; r < a.k; r += NT) {
      wout[r] = __uint_as_float(won[r].x) * by;
      iout[r] = (int32_t)won[r].y;
    }
    return;
  }
  float by = a.scale;
  if (a.renorm) {  // over the chosen: from the largest of them on
    if (total != total) by = NAN;  // a row that holds a NaN has no softmax, whatever is chosen of it
    m = -INFINITY;
    for (int r = lane; r < a.k; r += NT) {
      const int e = chosen(r);
      const float v = xs[e];
      won[r] = make_uint2(__float_as_uint(v), (uint32_t)e);
      live |= v != -INFINITY;
      m = fmaxf(m, v);
    }
    m = rt_max<NT>(m);
    total = 0.f;
    for (int r = lane; r < a.k; r += NT) {
      const float e = expf(__uint_as_float(won[r].x) - m);
      won[r].x = __float_as_uint(e);
      total += e;
    }
    total = rt_add<NT>(total);
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j) live |= x[j] != -INFINITY;
    for (int r = lane; r < a.k; r += NT) {
      const int e = chosen(r);
      won[r] = make_uint2(__float_as_uint(expf(xs[e] - m)), (uint32_t)e);
    }
  }
  const bool none = !rt_fold<NT>(live, [](uint32_t p, uint32_t q) { return p | q; });  // all are masked
  by /= total;
  for (int r = lane; r < a.k; r += NT) {
    wout[r] = none ? 0.f : __uint_as_float(won[r].x) * by;
    iout[r] = (int32_t)won[r].y;
  }
}

struct RtBwd {
  const void* x;
  int64_t T;
  int E, k, sigmoid, renorm;
  float scale;
  const int32_t* idx;
  const float* g;
  void* dx;
};

// d_logits from the weights' gradient g: with G = sum g w / scale over the chosen,
//   renormalised: d = w (g - G), times 1 - s for sigmoids;  sigmoid: scale g s (1 - s);
//   softmax: w g at the chosen, less s times sum g w everywhere.
template <typename T, int NT, int J>
__global__ __launch_bounds__(256) void k_rt_bwd(RtBwd a) {
  constexpr int TEAMS = 256 / NT;
  __shared__ float rows[TEAMS][NT * J];
  const int lane = threadIdx.x % NT, team = threadIdx.x / NT;
  const int64_t row = (int64_t)blockIdx.x * TEAMS + team;
  if (row >= a.T) return;
  const T* xr = (const T*)a.x + row * a.E;
  const int32_t* idx = a.idx + row * a.k;
  const float* g = a.g + row * a.k;
  float* d = rows[team];
  const int e0 = lane * J;
  float x[J], m = -INFINITY, total = 0.f, lmax = -INFINITY;
  const bool dense = !a.sigmoid && !a.renorm;
  uint32_t live = 0;  // whether one is not masked
  auto logit = [&](int r, int& e) {  // an index outside [0, E) is nowhere
    e = idx[r];
    if ((uint32_t)e >= (uint32_t)a.E) e = -1;
    return e < 0 ? -INFINITY : load_f<T>(xr, e);
  };
  auto lscore = [&](float v) { return a.sigmoid ? fminf(v, 0.f) - log1pf(expf(-fabsf(v))) : v; };
  if (dense) {
    rt_load<T, J>(xr, e0, a.E, x);
#pragma unroll
    for (int j = 0; j < J; ++j) m = fmaxf(m, x[j]), live |= x[j] != -INFINITY;
    m = rt_max<NT>(m);
#pragma unroll
    for (int j = 0; j < J; ++j) total += x[j] = expf(x[j] - m);
    total = rt_add<NT>(total);
    lmax = m;
  } else if (a.renorm) {
    int e;
    for (int r = lane; r < a.k; r += NT) {
      const float v = logit(r, e);
      live |= v != -INFINITY;
      lmax = fmaxf(lmax, lscore(v));
    }
    lmax = rt_max<NT>(lmax);
    for (int r = lane; r < a.k; r += NT) total += expf(lscore(logit(r, e)) - lmax);
    total = rt_add<NT>(total);
  }
  const bool none = (a.renorm || dense) && !rt_fold<NT>(live, [](uint32_t p, uint32_t q) { return p | q; });
  float G = 0.f;
  if (a.renorm || dense) {
    for (int r = lane; r < a.k; r += NT) {
      int e;
      const float v = logit(r, e);
      if (e >= 0 && !none) G += g[r] * (expf(lscore(v) - lmax) / total);
    }
    G = rt_add<NT>(G);
  }
#pragma unroll
  for (int j = 0; j < J; ++j) d[e0 + j] = dense && !none ? -(x[j] / total) * G * a.scale : 0.f;
  rt_wave_sync();
  for (int r = lane; r < a.k; r += NT) {
    int e;
    const float v = logit(r, e);
    if (e < 0 || none) continue;
    float c;
    if (a.renorm) {
      c = expf(lscore(v) - lmax) / total * (g[r] - G) * a.scale;
      if (a.sigmoid) c *= 1.f / (1.f + expf(v));
    } else if (a.sigmoid) {
      const float t = expf(-fabsf(v));  // s (1 - s) = t / (1 + t)^2
      c = g[r] * a.scale * (t / ((1.f + t) * (1.f + t)));
    } else {
      c = expf(v - m) / total * g[r] * a.scale;
    }
    atomicAdd(&d[e], c);  // a caller's row may hold an index twice
  }
  rt_wave_sync();
  T* out = (T*)a.dx + row * a.E;
#pragma unroll
  for (int c = 0; c < J; c += 8) {
    if (e0 + c + 8 <= a.E) {
      if constexpr (sizeof(T) == 2) {
        RtHalf8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) h.v[i] = f32_to_bf16(d[e0 + c + i]);
        *(RtHalf8*)(out + e0 + c) = h;
      } else {
        RtFloat4 p, q;
#pragma unroll
        for (int i = 0; i < 4; ++i) p.v[i] = d[e0 + c + i], q.v[i] = d[e0 + c + 4 + i];
        *(RtFloat4*)(out + e0 + c) = p;
        *(RtFloat4*)(out + e0 + c + 4) = q;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e0 + c + i < a.E) store_f<T>(out, e0 + c + i, d[e0 + c + i]);
    }
  }
}

// Lanes a row takes.
template <typename F>
void rt_form(int E, F&& f) {
  using std::integral_constant;
  const integral_constant<int, 8> eight;
  if (E <= 64) f(integral_constant<int, 8>{}, eight);
  else if (E <= 128) f(integral_constant<int, 16>{}, eight);
  else if (E <= 256) f(integral_constant<int, 32>{}, eight);
  else if (E <= 512) f(integral_constant<int, 64>{}, eight);
  else f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

int rt_check(const char* what, int dtype, int64_t T, int E, int k, float scale) {
  if (dtype != PD_DTYPE_F32 && dtype != PD_DTYPE_BF16)
    return fail(PD_EUNSUPPORTED, std::string(what) + ": logits are fp32 or bf16");
  if (T < 0 || E < 1 || k < 1 || k > E) return fail(PD_EINVAL, std::string(what) + ": T >= 0 and 1 <= k <= E");
  if (E > RT_MAX_E || k > RT_MAX_K || T > RT_MAX_T)
    return fail(PD_EUNSUPPORTED, std::string(what) + ": up to 1024 experts, 64 of them chosen, and 2^26 - 4 rows");
  if (!std::isfinite(scale)) return fail(PD_EINVAL, std::string(what) + ": scale must be finite");
  return PD_OK;
}

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" {

int pd_route_scores_fwd(const void* logits, int dtype, int64_t T, int E, int k, int sigmoid, const float* bias,
                        int n_groups, int top_groups, int renormalize, float scale, float* weights, int32_t* top_idx,
                        void* stream) {
  const char* what = "pd_route_scores_fwd";
  if (int rc = rt_check(what, dtype, T, E, k, scale)) return rc;
  if (n_groups < 1 || n_groups > RT_MAX_GROUPS || E % n_groups || top_groups < 1 || top_groups > n_groups ||
      k > E / n_groups * top_groups)
    return fail(PD_EINVAL, std::string(what) + ": up to 64 groups of equal size, of which those that stay hold k experts");
  if (T && (!logits || !weights || !top_idx)) return fail(PD_EINVAL, std::string(what) + ": null pointer");
  if (!T) return PD_OK;
  if (top_groups == n_groups) n_groups = top_groups = 1;  // all of them stay
  const RtArgs a{logits, T, E, k, sigmoid, bias, n_groups, top_groups, renormalize, scale, weights, top_idx};
  rt_form(E, [&](auto nt, auto j) {
    constexpr int NT = decltype(nt)::value, J = decltype(j)::value;
    const dim3 grid((unsigned)cdiv(T, 256 / NT));
    if (dtype == PD_DTYPE_BF16) hipLaunchKernelGGL((k_rt_fwd<bf16_t, NT, J>), grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((k_rt_fwd<float, NT, J>), grid, dim3(256), 0, (hipStream_t)stream, a);
  });
  return check_launch(what);
}

int pd_route_scores_bwd(const void* logits, int dtype, int64_t T, int E, int k, int sigmoid, int renormalize,
                        float scale, const int32_t* top_idx, const float* d_weights, void* d_logits, void* stream) {
  const char* what = "pd_route_scores_bwd";
  if (int rc = rt_check(what, dtype, T, E, k, scale)) return rc;
  if (T && (!logits || !top_idx || !d_weights || !d_logits)) return fail(PD_EINVAL, std::string(what) + ": null pointer");
  if (!T) return PD_OK;
  const RtBwd a{logits, T, E, k, sigmoid, renormalize, scale, top_idx, d_weights, d_logits};
  rt_form(E, [&](auto nt, auto j) {
    constexpr int NT = decltype(nt)::value, J = decltype(j)::value;
    const dim3 grid((unsigned)cdiv(T, 256 / NT));
    if (dtype == PD_DTYPE_BF16) hipLaunchKernelGGL((k_rt_bwd<bf16_t, NT, J>), grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((k_rt_bwd<float, NT, J>), grid, dim3(256), 0, (hipStream_t)stream, a);
  });
  return check_launch(what);
}

}  // extern "C"
