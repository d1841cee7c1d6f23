// KL from a teacher's top logits to a row of full logits, and its gradient.
//
//   q = softmax(z / tau) over the vocabulary; p over the k listed entries: softmax(t / tau)
//   over them, or, with the teacher's logsumexp, exp(t / tau - lse) and the mass they leave,
//   p_r = 1 - sum p, on all other entries together
//   kl = sum_j p_j (log p_j - log q_{i_j}) [+ p_r (log p_r - log q_r)], q_r = sum_{v not listed} q_v
//   with P = sum p + p_r and s = the row's weight / tau:
//   dz_v = s (P q_v - sum_{i_j = v} p_j)             listed v
//   dz_v = s e^{z_v / tau} / S_r (P q_r - p_r)         other v, S_r = sum_{v not listed} e^{z_v / tau}
//
// Memory bound: the logits are read once and the gradient written once. A block holds a row
// in registers (NT threads, U words of 16 bytes each), so its sums, its loss and its gradient
// come from the one read; longer rows are read a second time for the gradient. Blocks walk
// over rows: as the last pass over a row is done with a word, the same registers take the
// next row's, so loads and stores go on under the arithmetic of a row.
//
// Each listed entry belongs to a thread, which reads its logit and writes its gradient. A bit
// per vocabulary entry in LDS tells the row's threads where they are: there the registers
// take -inf, and the passes go over whole words with no test of an element (with tests a
// word with a listed entry cost its wave every pass twice: 8192 x 50277, 64 listed, 547 us).
// The elements behind a row's last whole word are one thread's each. So q_r is a sum and never a difference. Repeated indices
// add their p and count once in q.
//
// The loss is a small difference of logarithms: a second kernel forms p, the logarithms and
// the loss of a row in 64 bits from the row's maxima and sums (32-bit, their exponents with
// log2(e) / tau in two parts). In the first kernel that arithmetic took the registers that
// hold the row. The 32-bit sums leave a loss off by up to a few 1e-7 whatever its size. The
// gradient's rest is 64-bit too (what the listed leave of 1), its other terms are 32-bit: the
// exponents of the entries not listed take log2(e) / tau in one part, off by 2^-23 of their
// size, which is below a gradient's other roundings up to exponents of some tens.
#include <float.h>
#include <type_traits>

#include "pd_common.hpp"

namespace pd {
namespace {

constexpr double REST_MIN = 1.0 / (1 << 20);  // a rest below this is the rounding of its inputs: none
constexpr int KL_MAX_K = 1024;
constexpr int KL_LIST_NT = 256;  // forms of up to so many threads keep the listed logits for the loss
constexpr int64_t KL_MAX_V = 1 << 19;  // 64 KiB of bits

struct TopKLArgs {
  const void* z;
  int64_t rows;
  int V;
  const void* top;
  int top_dtype;
  const void* idx;
  int idx64;
  int k;
  const float* lse;
  double tau;
  float c, c_lo;  // log2(e) / tau, rounded down, and the positive rest of it
  float itau;
  const float* weight;
  float* kl;
  void* grad;
  struct KLRow* row;  // [rows] (NULL: no loss is wanted)
  float* listed;      // [rows, k] the listed logits, for the loss (forms of few threads)
};

// 16 bytes of a row, at any element's boundary (the hardware takes them as one access).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) KLWord {
  uint32_t v[4];
};
template <typename T>
__device__ inline float kl_elem(const uint4& w, int e) {
  const uint32_t u = (&w.x)[sizeof(T) == 2 ? e >> 1 : e];
  if constexpr (sizeof(T) == 2) return __uint_as_float((e & 1) ? u & 0xFFFF0000u : u << 16);
  else return __uint_as_float(u);
}
template <typename T>
__device__ inline float kl_f(T v) {
  if constexpr (sizeof(T) == 2) return bf16_to_f32(v);
  else return v;
}
__device__ inline float kl_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// Keeps the row packed between its passes: the compiler would carry a pass's unpacked
// values over to the next, twice the registers.
__device__ inline void kl_keep(uint4& w) { asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w)); }

// -inf in every element of a word.
template <typename T>
__device__ inline uint4 kl_none() {
  const uint32_t n = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
  return make_uint4(n, n, n, n);
}
template <typename T>
__device__ inline uint4 kl_load(const T* p) {
  const KLWord<T> x = *(const KLWord<T>*)p;
  return make_uint4(x.v[0], x.v[1], x.v[2], x.v[3]);
}

// What a row's loss takes from its logits: maximum and sum e^{(z - m) / tau} of the others
// and of the listed entries, and how many entries are listed.
struct KLRow {
  float mt, st, mp, sp;
  int listed, pad[3];
};

template <int G>
__device__ inline double kl_group_sum(double v) {
  for (int off = G / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// kl of a row, G lanes each. LIST: the listed logits come from the first kernel, in order; read
// again from the rows they are a line of memory each (100000 x 1000, 32 listed, with the
// gradient 202 us in place of 262). Where rows are long there are fewer of them, and keeping
// the list costs the first kernel more (1500 x 32000 fp32, the loss alone: 50 us, 47 without).
// With 16 lanes a wave takes the last step's logarithms for four rows at once; up to 4096
// rows, where that would leave SIMDs without a wave, a row has a wave (2048 rows of 128
// listed 9 us, 13 with 16 lanes; 8192 rows of 64 from the rows 23.4 us with 16, 24.7 with a
// wave).
template <typename T, int G, bool LIST>
__global__ __launch_bounds__(256) void k_top_kl_loss(TopKLArgs a) {
  const int lane = threadIdx.x % G;
  const int64_t r = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (r >= a.rows) return;
  const KLRow R = a.row[r];
  const double itau = 1.0 / a.tau;
  auto entry = [&](int e, int64_t& v, double& t) -> bool {
    v = a.idx64 ? ((const int64_t*)a.idx)[r * a.k + e] : ((const int32_t*)a.idx)[r * a.k + e];
    t = (double)(a.top_dtype == PD_DTYPE_F32 ? ((const float*)a.top)[r * a.k + e]
                                             : bf16_to_f32(((const bf16_t*)a.top)[r * a.k + e])) / a.tau;
    return v >= 0 && v < a.V;
  };
  int64_t v;
  double t, norm = 0.0, valid = 0.0;
  if (a.lse) {
    norm = (double)a.lse[r];
  } else {  // log of the teacher's partition sum
    double mx = -INFINITY, s = 0.0;
    for (int e = lane; e < a.k; e += G)
      if (entry(e, v, t)) mx = fmax(mx, t), valid += 1.0;
    for (int off = G / 2; off > 0; off >>= 1) mx = fmax(mx, __shfl_xor(mx, off, 64));
    for (int e = lane; e < a.k; e += G)
      if (entry(e, v, t)) s += exp(t - mx);
    norm = mx + log(kl_group_sum<G>(s));
    valid = kl_group_sum<G>(valid);
  }
  double sum_p = 0.0, plogp = 0.0, pz = 0.0;
  for (int e = lane; e < a.k; e += G)
    if (entry(e, v, t)) {
      const double l = t - norm, p = exp(l);
      sum_p += p;
      if (p != 0.0) plogp += p * l, pz += p * (double)(LIST ? a.listed[r * a.k + e] : load_f<T>((const T*)a.z + r * a.V, v));
    }
  sum_p = kl_group_sum<G>(sum_p);
  plogp = kl_group_sum<G>(plogp);
  pz = kl_group_sum<G>(pz);
  if (lane) return;
  const double M = fmax((double)R.mt, (double)R.mp);
  const double S = (double)R.st * exp(((double)R.mt - M) * itau) + (double)R.sp * exp(((double)R.mp - M) * itau);
  const double log_s = log(S);  // logsumexp of the row = M / tau + log_s
  double kl = plogp - pz * itau + sum_p * (M * itau + log_s);
  if (a.lse) {
    double rest = 1.0 - sum_p;
    if (rest < REST_MIN || R.listed == a.V) rest = 0.0;  // a NaN stays one
    if (rest != 0.0) kl += rest * (log(rest) - ((double)R.mt - M) * itau - log((double)R.st) + log_s);
  } else if (valid == 0.0) {
    kl = 0.0;  // no teacher, no loss
  }
  a.kl[r] = (float)kl;
}

// Entries of the list a thread takes: forms of few threads are used for short lists only.
constexpr int kl_entries(int nt) { return nt >= 256 ? KL_MAX_K / nt : 4; }
// REG: the row fits NT * U words and stays in registers between the two passes. What bounds it
// is a row's chain of passes (maximum, sum, gradient, with a reduction between each two) at
// two rows a CU where rows are long: 8192 x 50277 bf16, 64 listed, the gradient 430 us,
// 3.8 TB/s, the loss another 19; 1500 x 32000 fp32 93 us, 4.1 TB/s (calls one behind another).
// At 128 registers a thread 16 words spill 27 of them with the gradient and 16 to 20 without
// (20 to 22 and 12 to 16 in 1024 threads), 256 threads of 8 words 13 and 2, the streaming form
// 5 to 10 with the gradient; the others none or 2.
template <typename T, int NT, int U, bool REG, bool GRAD>
__global__ __launch_bounds__(NT, 4) void k_top_kl(TopKLArgs a) {
#pragma clang fp contract(off)  // the same sums with and without the gradient
  constexpr int VEC = 16 / sizeof(T), NW = NT / 64, KT = kl_entries(NT);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float4 red_f[2][NW];
  __shared__ float2 red_n[2][NW];  // listed entries, all entries
  __shared__ double red_p[2][NW];
  __shared__ float red_0[2][NW];
  __shared__ int repeated[2];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int V = a.V, words = V / VEC, tail = V % VEC, groups = REG ? 1 : (words + NT * U - 1) / (NT * U);
  static_assert(NT >= VEC, "a thread for each element of the tail");
  uint32_t* bits = (uint32_t*)lds;
  int* vlist = (int*)(bits + (V + 31) / 32);
  float* plist = (float*)(vlist + a.k);
  for (int i = tid; i < (V + 31) / 32; i += NT) bits[i] = 0;
  if (tid < 2) repeated[tid] = 0;

  uint4 w[U];
  auto load = [&](int64_t r, int g) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (g * U + u) * NT + tid;
      w[u] = i < words ? kl_load<T>((const T*)a.z + r * V + i * VEC) : kl_none<T>();
    }
  };
  float ztail = -INFINITY;  // this thread's element behind the last whole word
  auto load_tail = [&](int64_t r) {
    if (tid < tail) ztail = kl_f<T>(((const T*)a.z)[r * V + words * VEC + tid]);
  };
  // What a row takes besides its logits is loaded ahead: the list two rows (the listed
  // logits' addresses come out of it), the listed logits and the row's scalars one.
  int nidx[KT], vi[KT];  // -1: absent
  float ntop[KT], zj[KT], pj[KT], lse_r = 0.f, weight_r = 1.f;
  auto load_top = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      const int e = tid + j * NT;
      nidx[j] = -1;
      if (e < a.k) {
        const int64_t v = a.idx64 ? ((const int64_t*)a.idx)[r * a.k + e] : ((const int32_t*)a.idx)[r * a.k + e];
        nidx[j] = v >= 0 && v < V ? (int)v : -1;
        ntop[j] = a.top_dtype == PD_DTYPE_F32 ? ((const float*)a.top)[r * a.k + e]
                                              : bf16_to_f32(((const bf16_t*)a.top)[r * a.k + e]);
      }
    }
  };
  // e^{d / tau}, d <= 0 (-inf: 0), its exponent in two parts: one of 32 bits is off by the
  // same 2^-24 for every entry, which the loss would show.
  auto scaled = [&](float d) { return kl_exp2(fmaf(d, a.c, d * a.c_lo)); };
  // Puts -inf in the listed elements of the words in registers.
  auto hide = [&](int g, int at) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (g * U + u) * NT + at;
      uint32_t h = 0;
      if (i < words) {
        if constexpr (VEC == 8) h = ((const uint8_t*)bits)[i];
        else h = ((const uint8_t*)bits)[i >> 1] >> (4 * (i & 1)) & 15u;
      }
      if (h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t& x = (&w[u].x)[e];
          if constexpr (VEC == 8) {
            if (h >> (2 * e) & 1) x = (x & 0xFFFF0000u) | 0xFF80u;
            if (h >> (2 * e + 1) & 1) x = (x & 0xFFFFu) | 0xFF800000u;
          } else {
            if (h >> e & 1) x = 0xFF800000u;
          }
        }
      }
    }
  };

  auto load_listed = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      vi[j] = nidx[j];
      pj[j] = ntop[j];
      zj[j] = vi[j] >= 0 ? kl_f<T>(((const T*)a.z)[r * V + vi[j]]) : 0.f;
    }
    if (a.lse) lse_r = a.lse[r];
    if (GRAD && a.weight) weight_r = a.weight[r];
  };

  int64_t r = blockIdx.x;
  load_top(r);
  load_listed(r);
  if (r + gridDim.x < a.rows) load_top(r + gridDim.x);
  load(r, 0);
  load_tail(r);
  __syncthreads();
  for (int it = 0; r < a.rows; r += gridDim.x, ++it) {
    const int par = it & 1;
    const int64_t nr = r + gridDim.x;
    // the thread's place in a row, as new for each row: addresses formed once for all rows
    // take the registers that hold one
    int at = tid;
    asm volatile("" : "+v"(at));

    // ---- the listed entries: bits, own logits, p
    uint32_t own = 0;  // bit j: this thread's entry j is there, and the first with its index
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      if (vi[j] >= 0) {
        own |= 1u << j;
        const uint32_t b = 1u << (vi[j] & 31);
        if (atomicOr(&bits[vi[j] >> 5], b) & b) repeated[par] = 1;
      }
    }
    const bool has_top = wv * 64 < a.k;  // whether the wave has an entry (k > NT: every wave)
    double sum_p = 0.0;
    if (a.lse) {  // in 64 bits: the rest is what they leave of 1
      if (has_top) {
        const double lse = (double)lse_r, itau = 1.0 / a.tau;
#pragma unroll
        for (int j = 0; j < KT; ++j)
          if (own >> j & 1) {
            asm volatile("" : "+v"(pj[j]));  // one after the other: side by side they take the row's registers
            const double p = exp((double)pj[j] * itau - lse);
            pj[j] = (float)p;
            asm volatile("" : "+v"(pj[j]));
            sum_p += p;
          }
        sum_p = wave_sum_d(sum_p);
      }
    } else {
      float mx = -INFINITY, sum = 0.f;
#pragma unroll
      for (int j = 0; j < KT; ++j)
        if (own >> j & 1) mx = fmaxf(mx, pj[j]);
      mx = wave_max(mx);
      if (a.k > 64) {  // more than one wave's entries
        if (lane == 0) red_0[0][wv] = mx;
        __syncthreads();
        for (int i = 0; i < NW; ++i) mx = fmaxf(mx, red_0[0][i]);
      }
      if (has_top) {
#pragma unroll
        for (int j = 0; j < KT; ++j)
          if (own >> j & 1) {
            pj[j] = scaled(pj[j] - mx);
            sum += pj[j];
          }
        sum = wave_sum(sum);
      }
      if (a.k > 64) {
        if (lane == 0) red_0[1][wv] = sum;
        __syncthreads();
        sum = 0.f;
        for (int i = 0; i < NW; ++i) sum += red_0[1][i];
      }
      const float norm = 1.f / sum;
#pragma unroll
      for (int j = 0; j < KT; ++j) pj[j] *= norm;
      sum_p = wv == 0 ? 1.0 : 0.0;
    }
    const float valid_w = has_top ? wave_sum((float)__popc(own)) : 0.f;
    __syncthreads();  // the bits are set
    if (repeated[par]) {  // the first of equal indices takes the others' p, in list order
#pragma unroll
      for (int j = 0; j < KT; ++j)
        if (tid + j * NT < a.k) vlist[tid + j * NT] = vi[j], plist[tid + j * NT] = pj[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < KT; ++j)
        if (own >> j & 1) {
          float p = 0.f;
          for (int e = 0; e < a.k; ++e)
            if (vlist[e] == vi[j]) {
              if (e < tid + j * NT) own &= ~(1u << j);
              p += plist[e];
            }
          pj[j] = p;
        }
    }

    // ---- one pass over the row: the others' and the listed entries' maxima and sums
    float mt = -FLT_MAX, st = 0.f;
    for (int g = 0; g < groups; ++g) {
      if (!REG && (g || it)) load(r, g);
      hide(g, at);
      float m = mt;
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = fmaxf(m, kl_elem<T>(w[u], e));
        kl_keep(w[u]);
      }
      st *= scaled(mt - m);
      mt = m;
      asm volatile("" : "+v"(at));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += scaled(kl_elem<T>(w[u], e) - m);
        st += s;
        asm volatile("" : "+v"(st));
        kl_keep(w[u]);
        const int i = u * NT + at;
        if (REG && !GRAD && nr < a.rows && i < words) w[u] = kl_load<T>((const T*)a.z + nr * V + i * VEC);
      }
    }
    const float zt = ztail;
    bool mine = false;  // the tail's element is there and not listed
    if (tid < tail) {
      mine = !(bits[(words * VEC + tid) >> 5] >> ((words * VEC + tid) & 31) & 1);
      if (mine) {
        const float m = fmaxf(mt, zt);
        st = st * scaled(mt - m) + scaled(zt - m);
        mt = m;
      }
    }
    if (nr < a.rows) load_tail(nr);
    float mp = -FLT_MAX, sp = 0.f, listed = 0.f;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float x = __shfl_xor(mt, off, 64), m = fmaxf(mt, x);
      st *= scaled(mt - m);
      mt = m;
      st += __shfl_xor(st, off, 64);
    }
    if (has_top) {
#pragma unroll
      for (int j = 0; j < KT; ++j)
        if (own >> j & 1) mp = fmaxf(mp, zj[j]);
      mp = wave_max(mp);
#pragma unroll
      for (int j = 0; j < KT; ++j)
        if (own >> j & 1) {
          sp += scaled(zj[j] - mp);
        }
      sp = wave_sum(sp);
      listed = wave_sum((float)__popc(own));
    }
    if (lane == 0) {
      red_f[par][wv] = make_float4(mt, st, mp, sp);
      red_n[par][wv] = make_float2(listed, valid_w);
      red_p[par][wv] = sum_p;
    }
    __syncthreads();
    // every wave joins the waves' sums: lane i the one of wave i
    const float4 f = red_f[par][lane & (NW - 1)];
    const float2 n2 = red_n[par][lane & (NW - 1)];
    mt = f.x, mp = f.z, listed = n2.x, sum_p = red_p[par][lane & (NW - 1)];
    float valid = n2.y;
#pragma unroll
    for (int off = NW / 2; off > 0; off >>= 1) mt = fmaxf(mt, __shfl_xor(mt, off, 64)), mp = fmaxf(mp, __shfl_xor(mp, off, 64));
    st = f.y * scaled(f.x - mt);
    sp = f.w * scaled(f.z - mp);
#pragma unroll
    for (int off = NW / 2; off > 0; off >>= 1) {
      st += __shfl_xor(st, off, 64);
      sp += __shfl_xor(sp, off, 64);
      sum_p += __shfl_xor(sum_p, off, 64);
      listed += __shfl_xor(listed, off, 64);
      valid += __shfl_xor(valid, off, 64);
    }
    if (tid == 0) {
      if (a.row) a.row[r] = KLRow{mt, st, mp, sp, (int)listed, {0, 0, 0}};
      repeated[par ^ 1] = 0;  // for the next row; this row's has been read
    }

    if (NT <= KL_LIST_NT && a.row) {
#pragma unroll
      for (int j = 0; j < KT; ++j)
        if (vi[j] >= 0) a.listed[r * a.k + at + j * NT] = zj[j];  // repeated entries too
    }

    // ---- the gradient
    if constexpr (GRAD) {
      const float M = fmaxf(mt, mp), wt = scaled(mt - M), S = st * wt + sp * scaled(mp - M);
      double left = 0.0;
      if (a.lse) {
        left = 1.0 - sum_p;
        if (left < REST_MIN || listed == (float)V) left = 0.0;
      }
      const float s = weight_r * a.itau, P = (float)(sum_p + left), rest = (float)left;
      const float At = st > 0.f || st != st ? s * (P * (st * wt / S) - rest) / st : 0.f, As = s * P / S;
      const bool skip = s == 0.f || (valid == 0.f && !a.lse);  // unweighted, or without a teacher: zeros
      T* grow = (T*)a.grad + r * V;
      asm volatile("" : "+v"(at));
      for (int g = groups - 1; g >= 0; --g) {  // the last group is still in registers
        if (!REG && g != groups - 1) {
          load(r, g);
          hide(g, at);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = (g * U + u) * NT + at;
          if (i >= words) continue;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (!skip) {
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = kl_exp2((kl_elem<T>(w[u], e) - mt) * a.c) * At;
            kl_keep(w[u]);
            if constexpr (VEC == 8)
              x = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]),
                             pack_bf16x2(o[6], o[7]));
            else
              x = make_uint4(__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
          }
          *(KLWord<T>*)(grow + i * VEC) = KLWord<T>{{x.x, x.y, x.z, x.w}};
          if (REG && nr < a.rows) w[u] = kl_load<T>((const T*)a.z + nr * V + i * VEC);
        }
      }
      if (mine) store_f<T>(grow, words * VEC + tid, skip ? 0.f : kl_exp2((zt - mt) * a.c) * At);
      // the words' stores are in memory before the listed entries' own
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
#pragma unroll
      for (int j = 0; j < KT; ++j)
        if (own >> j & 1) store_f<T>(grow, vi[j], skip ? 0.f : scaled(zj[j] - M) * As - s * pj[j]);
    }
    if (!GRAD) __syncthreads();  // the bits have been read
#pragma unroll
    for (int j = 0; j < KT; ++j)
      if (vi[j] >= 0) bits[vi[j] >> 5] = 0;
    if (nr < a.rows) load_listed(nr);
    if (nr + gridDim.x < a.rows) load_top(nr + gridDim.x);
    __syncthreads();
  }
}

template <typename T, bool GRAD>
int top_kl_launch(const TopKLArgs& a, hipStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t words = a.V / VEC;
  const size_t lds = (size_t)cdiv(a.V, 32) * 4 + (size_t)a.k * 8;
  // Blocks that walk over the rows: as many as the GPU holds of a form at once.
  auto go = [&](auto kernel, int nt, int64_t held) -> int {
    if (lds > 48 * 1024 &&
        hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024) != hipSuccess)
      return fail(PD_ELAUNCH, "pd_top_kl: shared memory");
    hipLaunchKernelGGL(kernel, dim3((unsigned)(a.rows < held ? a.rows : held)), dim3(nt), lds, s, a);
    auto loss = [&](auto wave, auto list) {
      constexpr int G = wave ? 64 : 16;
      hipLaunchKernelGGL((k_top_kl_loss<T, G, list>), dim3((unsigned)cdiv(a.rows, 256 / G)), dim3(256), 0, s, a);
    };
    const std::true_type yes;
    const std::false_type no;
    if (a.kl) {
      if (a.rows <= 4096) nt <= KL_LIST_NT ? loss(yes, yes) : loss(yes, no);
      else nt <= KL_LIST_NT ? loss(no, yes) : loss(no, no);
    }
    return check_launch("pd_top_kl");
  };
  // The smallest form that holds the row (and, with one wave, its list): loss and gradient in
  // the next two, and the streaming one: 100000 x 1000 bf16 291, 343, 895, 3628 us; 8192 x
  // 16000 135, 193, 245, 343; 4096 x 50277 217, 319, streaming 295. The widest is even with the
  // streaming one (2048 x 131000: 284 and 288) and reads a row once. 512 threads of 16 words
  // with one block a CU, two, more: 289, 229, 231 us at 4096 x 50277. The loss alone, in this
  // form, the next one and the streaming one: 100000 x 1000 bf16 159, 225, 2878 us; 8192 x
  // 16000 86, 141, 272; 8192 x 50277 245, 422, 393; 1500 x 32000 fp32 51, 66, 60; 2048 x 131072
  // bf16 153, streaming 167.
  if (a.k <= 256 && words <= 64 * 2) return go(k_top_kl<T, 64, 2, true, GRAD>, 64, 256 * 16);
  if (a.k <= 256 && words <= 64 * 8) return go(k_top_kl<T, 64, 8, true, GRAD>, 64, 256 * 16);
  if (words <= 256 * 8) return go(k_top_kl<T, 256, 8, true, GRAD>, 256, 256 * 8);
  if (words <= 512 * 8) return go(k_top_kl<T, 512, 8, true, GRAD>, 512, 256 * 4);
  if (words <= 512 * 16) return go(k_top_kl<T, 512, 16, true, GRAD>, 512, 256 * 2);
  if (words <= 1024 * 16) return go(k_top_kl<T, 1024, 16, true, GRAD>, 1024, 256);
  return go(k_top_kl<T, 1024, 8, false, GRAD>, 1024, 256 * 2);
}

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" {

size_t pd_top_kl_workspace_size(int64_t rows, int k) {
  return rows > 0 && k > 0 ? (size_t)rows * (sizeof(KLRow) + (size_t)k * sizeof(float)) : 0;
}

int pd_top_kl(const void* z, int dtype, int64_t rows, int64_t vocab, const void* top, int top_dtype, const void* idx,
              int idx_bits, int k, const float* clean_lse, double temperature, const float* row_weight, float* kl,
              void* grad, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != PD_DTYPE_F32 && dtype != PD_DTYPE_BF16) return fail(PD_EUNSUPPORTED, "pd_top_kl: logits are fp32 or bf16");
  if (top_dtype != PD_DTYPE_F32 && top_dtype != PD_DTYPE_BF16)
    return fail(PD_EUNSUPPORTED, "pd_top_kl: top logits are fp32 or bf16");
  if (idx_bits != 32 && idx_bits != 64) return fail(PD_EUNSUPPORTED, "pd_top_kl: indices are 32- or 64-bit");
  if (rows < 0 || vocab <= 0 || k <= 0) return fail(PD_EINVAL, "pd_top_kl: rows >= 0, vocab >= 1 and k >= 1");
  if (rows > 0x7FFFFFFF || vocab > KL_MAX_V || k > KL_MAX_K)
    return fail(PD_EUNSUPPORTED, "pd_top_kl: at most 2^31 - 1 rows, 2^19 logits a row and 1024 listed");
  if (!(temperature > 0.f) || !std::isfinite(temperature))
    return fail(PD_EINVAL, "pd_top_kl: temperature must be positive and finite");
  if (!rows) return PD_OK;
  if (!z || !top || !idx || (!kl && !grad)) return fail(PD_EINVAL, "pd_top_kl: null pointer");
  if (kl && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < pd_top_kl_workspace_size(rows, k)))
    return fail(PD_EWORKSPACE, "pd_top_kl: workspace");
  const double c = 1.4426950408889634074 / temperature, itau = 1.0 / temperature;
  float c_hi = (float)c;
  if ((double)c_hi >= c) c_hi = std::nextafter(c_hi, 0.f);
  const TopKLArgs a = {z, rows, (int)vocab, top, top_dtype, idx, idx_bits == 64, k, clean_lse, temperature, c_hi,
                       (float)(c - (double)c_hi), (float)itau, row_weight, kl,
                       grad, kl ? (KLRow*)workspace : nullptr, kl ? (float*)((KLRow*)workspace + rows) : nullptr};
  if (!std::isfinite(a.c) || !(a.c_lo > 0.f) || !std::isfinite(a.itau)) return fail(PD_EINVAL, "pd_top_kl: temperature is out of range");
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PD_DTYPE_F32) return grad ? top_kl_launch<float, true>(a, s) : top_kl_launch<float, false>(a, s);
  return grad ? top_kl_launch<bf16_t, true>(a, s) : top_kl_launch<bf16_t, false>(a, s);
}

}  // extern "C"
