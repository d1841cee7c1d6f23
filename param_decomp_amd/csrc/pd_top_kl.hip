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
// Memory bound: the logits are read once and the gradient written once. One block per row
// holds the row in registers (NT threads, U loads of 16 bytes each), so its sums, its loss
// and its gradient come from the one read; longer rows are read a second time for the
// gradient. Listed entries are kept out of the other entries' sum and given their own, by
// a bit per vocabulary entry in LDS (one byte read per 16-byte load), so q_r is a sum and
// never a difference; a listed entry finds its p through a small hash table, also in LDS.
// Repeated indices add their p and count once in q. Rows start at any 2-byte (4-byte)
// boundary: loads and stores are whole aligned 16-byte words but for a row's first and last.
// The scalars of a row (p, logarithms, the loss) are formed in 64 bits, since the loss is
// a small difference of them; the sums of exponentials are 32-bit.
#include <float.h>

#include "pd_common.hpp"

namespace pd {
namespace {

constexpr double REST_MIN = 1.0 / (1 << 20);  // a rest below this is the rounding of its inputs: none
constexpr int KL_MAX_K = 1024;
constexpr int64_t KL_MAX_V = 1 << 19;  // 64 KiB of bits

struct TopKLArgs {
  const void* z;
  int64_t V;
  const void* top;
  int top_dtype;
  const void* idx;
  int idx64;
  int k;
  const float* lse;
  float tau;
  const float* weight;
  float* kl;
  void* grad;
  int slots;  // hash slots, a power of two, at least 2 k
  int vec_out;  // grad's rows are aligned as the logits' are
};

template <typename T>
__device__ inline float kl_elem(const uint4& w, int e) {
  const uint32_t u = (&w.x)[sizeof(T) == 2 ? e >> 1 : e];
  if constexpr (sizeof(T) == 2) return __uint_as_float((e & 1) ? u & 0xFFFF0000u : u << 16);
  else return __uint_as_float(u);
}

// The word of VEC elements from element v0 on (v0 < 0 or past V in a row's first and last).
template <typename T, int VEC>
__device__ inline uint4 kl_load(const T* __restrict__ row, int v0, int V) {
  if (v0 >= 0 && v0 + VEC <= V) return *(const uint4*)(row + v0);
  T e[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) e[i] = v0 + i >= 0 && v0 + i < V ? row[v0 + i] : T(0);
  uint4 w;
  if constexpr (VEC == 8)
    w = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                   e[6] | (uint32_t)e[7] << 16);
  else
    w = make_uint4(__float_as_uint(e[0]), __float_as_uint(e[1]), __float_as_uint(e[2]), __float_as_uint(e[3]));
  return w;
}

// Bits of a word's elements inside the row.
template <int VEC>
__device__ inline uint32_t kl_inside(int v0, int V) {
  if (v0 >= 0 && v0 + VEC <= V) return (1u << VEC) - 1;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VEC; ++i) m |= (v0 + i >= 0 && v0 + i < V ? 1u : 0u) << i;
  return m;
}

struct MaxSum {
  float m, s;  // s = sum e^{(z - m) / tau}; m = -FLT_MAX and s = 0 where nothing counts
};
__device__ inline MaxSum ms_join(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * exp2f((a.m - m) * c) + b.s * exp2f((b.m - m) * c)};
}

__device__ inline uint32_t kl_hash(uint32_t v, int mask) { return (v * 2654435761u >> 12) & mask; }
__device__ inline int kl_find(const int* key, int mask, int v) {
  uint32_t h = kl_hash(v, mask);
  while (key[h] != v) h = (h + 1) & mask;  // v is in the table
  return h;
}

// REG: the row fits NT * U words and stays in registers between the two passes.
template <typename T, int NT, int U, bool REG>
__global__ __launch_bounds__(NT) void k_top_kl(TopKLArgs a) {
  constexpr int VEC = 16 / sizeof(T), NW = NT / 64;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ double red_d[NW][3];
  __shared__ float red_f[NW][4];
  __shared__ int2 red_n[NW];  // entries with an index of their own, entries
  __shared__ float fin[6];  // M_t, A_t (others' factor), M, P s / S, s
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t r = blockIdx.x;
  const int V = (int)a.V;
  const T* row = (const T*)a.z + r * a.V;
  const int lead = (int)(((uintptr_t)row & 15) / sizeof(T));  // words start at element -lead
  const int words = (V + lead + VEC - 1) / VEC;
  const int groups = REG ? 1 : (words + NT * U - 1) / (NT * U);
  uint4 w[U];
  auto load = [&](int g) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (g * U + u) * NT + tid;
      w[u] = i < words ? kl_load<T, VEC>(row, i * VEC - lead, V) : make_uint4(0, 0, 0, 0);
    }
  };
  load(0);

  // ---- the listed entries: bits, hash table, p
  int* key = (int*)lds;                       // [slots] vocabulary index or -1
  int* own = key + a.slots;                   // [slots] the first entry with that index
  float* pslot = (float*)(own + a.slots);     // [slots]
  uint32_t* bits = (uint32_t*)(pslot + a.slots);
  const int bit_words = (words * VEC + 31) / 32;
  for (int i = tid; i < bit_words; i += NT) bits[i] = 0;
  for (int i = tid; i < a.slots; i += NT) key[i] = -1, own[i] = 0x7FFFFFFF, pslot[i] = 0.f;
  constexpr int KT = (KL_MAX_K + NT - 1) / NT;
  int vi[KT];
  double lp[KT];  // t / tau, then log p
  double mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < KT; ++j) {
    const int e = tid + j * NT;
    vi[j] = -1;
    lp[j] = -INFINITY;
    if (e < a.k) {
      const int64_t v = a.idx64 ? ((const int64_t*)a.idx)[r * a.k + e] : ((const int32_t*)a.idx)[r * a.k + e];
      if (v >= 0 && v < a.V) {
        vi[j] = (int)v;
        const float t = a.top_dtype == PD_DTYPE_F32 ? ((const float*)a.top)[r * a.k + e]
                                                    : bf16_to_f32(((const bf16_t*)a.top)[r * a.k + e]);
        lp[j] = (double)t / (double)a.tau;
        mx = t != t ? (double)NAN : fmax(mx, lp[j]);
      }
    }
  }
  __syncthreads();
  int uniq = 0;
#pragma unroll
  for (int j = 0; j < KT; ++j)
    if (vi[j] >= 0) {
      const uint32_t b = (uint32_t)(vi[j] + lead);
      if (!(atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1)) ++uniq;
      uint32_t h = kl_hash(vi[j], a.slots - 1);
      for (;;) {  // at most k <= slots / 2 keys: a free slot is met
        const int was = atomicCAS(&key[h], -1, vi[j]);
        if (was == -1 || was == vi[j]) break;
        h = (h + 1) & (a.slots - 1);
      }
      atomicMin(&own[h], tid + j * NT);
    }
  double norm;  // log of the teacher's partition sum
  if (a.lse) {
    norm = (double)a.lse[r];
  } else {
    for (int off = 32; off > 0; off >>= 1) mx = fmax(mx, __shfl_xor(mx, off, 64));
    if (lane == 0) red_d[wv][0] = mx;
    __syncthreads();
    mx = red_d[0][0];
    for (int i = 1; i < NW; ++i) mx = fmax(mx, red_d[i][0]);
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < KT; ++j)
      if (vi[j] >= 0) s += exp(lp[j] - mx);
    s = wave_sum_d(s);
    if (lane == 0) red_d[wv][1] = s;
    __syncthreads();
    s = 0.0;
    for (int i = 0; i < NW; ++i) s += red_d[i][1];
    norm = mx + log(s);
  }
  double sum_p = 0.0, sum_plogp = 0.0;
  float pj[KT];
#pragma unroll
  for (int j = 0; j < KT; ++j) {
    pj[j] = 0.f;
    if (vi[j] >= 0) {
      const double l = lp[j] - norm, p = exp(l);
      pj[j] = (float)p;
      sum_p += p;
      if (p != 0.0) sum_plogp += p * l;
    }
  }
  int valid = 0;
#pragma unroll
  for (int j = 0; j < KT; ++j) valid += vi[j] >= 0;
  uniq = (int)wave_sum((float)uniq);
  valid = (int)wave_sum((float)valid);
  if (lane == 0) red_n[wv] = make_int2(uniq, valid);
  __syncthreads();
  int n_uniq = 0, n_valid = 0;
  for (int i = 0; i < NW; ++i) n_uniq += red_n[i].x, n_valid += red_n[i].y;
  if (n_valid == n_uniq) {
#pragma unroll
    for (int j = 0; j < KT; ++j)
      if (vi[j] >= 0) pslot[kl_find(key, a.slots - 1, vi[j])] = pj[j];
  } else {
    // an index listed more than once: its first entry adds the others' p in list order
    float* plist = (float*)own;  // rewritten below once every owner is known
    bool first[KT];
    int slot[KT];
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      slot[j] = vi[j] >= 0 ? kl_find(key, a.slots - 1, vi[j]) : -1;
      first[j] = slot[j] >= 0 && own[slot[j]] == tid + j * NT;
    }
    __syncthreads();
    int* vlist = (int*)own + a.slots / 2;
#pragma unroll
    for (int j = 0; j < KT; ++j)
      if (tid + j * NT < a.k) plist[tid + j * NT] = pj[j], vlist[tid + j * NT] = vi[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < KT; ++j)
      if (first[j]) {
        float p = 0.f;
        for (int e = tid + j * NT; e < a.k; ++e)
          if (vlist[e] == vi[j]) p += plist[e];
        pslot[slot[j]] = p;
      }
  }
  __syncthreads();

  // ---- one pass over the row: the others' and the listed entries' maxima and sums, and
  // sum_j p_j z_{i_j}
  const float c = 1.4426950408889634f / a.tau;
  MaxSum mt = {-FLT_MAX, 0.f}, mp = {-FLT_MAX, 0.f};
  double pz = 0.0;
  for (int g = 0; g < groups; ++g) {
    if (g) load(g);
    float m = mt.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (g * U + u) * NT + tid;
      if (i >= words) continue;
      const uint32_t in = kl_inside<VEC>(i * VEC - lead, V);
      const uint32_t hit = VEC == 8 ? ((const uint8_t*)bits)[i] : ((const uint8_t*)bits)[i >> 1] >> (4 * (i & 1)) & 15u;
      if (hit == 0 && in == (1u << VEC) - 1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = fmaxf(m, kl_elem<T>(w[u], e));
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (in & ~hit & (1u << e)) m = fmaxf(m, kl_elem<T>(w[u], e));
      }
    }
    mt.s *= exp2f((mt.m - m) * c);
    mt.m = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (g * U + u) * NT + tid;
      if (i >= words) continue;
      const uint32_t in = kl_inside<VEC>(i * VEC - lead, V);
      const uint32_t hit = VEC == 8 ? ((const uint8_t*)bits)[i] : ((const uint8_t*)bits)[i >> 1] >> (4 * (i & 1)) & 15u;
      if (hit == 0 && in == (1u << VEC) - 1) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += __builtin_amdgcn_exp2f((kl_elem<T>(w[u], e) - m) * c);
        mt.s += s;
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float z = kl_elem<T>(w[u], e);
          if (in & ~hit & (1u << e)) mt.s += __builtin_amdgcn_exp2f((z - m) * c);
          if (hit & (1u << e)) {
            mp = ms_join(mp, {z == z ? fmaxf(z, -FLT_MAX) : 0.f, z == -INFINITY ? 0.f : (z == z ? 1.f : NAN)}, c);
            const float p = pslot[kl_find(key, a.slots - 1, i * VEC - lead + e)];
            if (p != 0.f) pz += (double)p * (double)z;
          }
        }
      }
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    mt = ms_join(mt, {__shfl_xor(mt.m, off, 64), __shfl_xor(mt.s, off, 64)}, c);
    mp = ms_join(mp, {__shfl_xor(mp.m, off, 64), __shfl_xor(mp.s, off, 64)}, c);
  }
  sum_p = wave_sum_d(sum_p);
  sum_plogp = wave_sum_d(sum_plogp);
  pz = wave_sum_d(pz);
  if (lane == 0) {
    red_d[wv][0] = sum_p, red_d[wv][1] = sum_plogp, red_d[wv][2] = pz;
    red_f[wv][0] = mt.m, red_f[wv][1] = mt.s, red_f[wv][2] = mp.m, red_f[wv][3] = mp.s;
  }
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < NW; ++i) {
      sum_p += red_d[i][0], sum_plogp += red_d[i][1], pz += red_d[i][2];
      mt = ms_join(mt, {red_f[i][0], red_f[i][1]}, c);
      mp = ms_join(mp, {red_f[i][2], red_f[i][3]}, c);
    }
    const double itau = 1.0 / (double)a.tau;
    const float M = fmaxf(mt.m, mp.m);
    const double wt = exp(((double)mt.m - (double)M) * itau);
    const double S = (double)mt.s * wt + (double)mp.s * exp(((double)mp.m - (double)M) * itau);
    double rest = 0.0;
    if (a.lse) {
      rest = 1.0 - sum_p;
      if (rest < REST_MIN || n_uniq == V) rest = 0.0;  // a NaN stays one
    }
    const double P = sum_p + rest;
    const double log_s = log(S);  // logsumexp = M / tau + log_s
    double kl = sum_plogp - pz * itau + sum_p * ((double)M * itau + log_s);
    if (rest != 0.0) kl += rest * (log(rest) - ((double)mt.m - (double)M) * itau - log((double)mt.s) + log_s);
    if (n_valid == 0 && !a.lse) kl = 0.0;  // no teacher, no loss
    if (a.kl) a.kl[r] = (float)kl;
    const double s = (a.weight ? (double)a.weight[r] : 1.0) * itau;
    fin[0] = mt.m;
    fin[1] = mt.s > 0.f || mt.s != mt.s ? (float)(s * (P * (double)mt.s * wt / S - rest) / (double)mt.s) : 0.f;
    fin[2] = M;
    fin[3] = (float)(s * P / S);
    fin[4] = (float)s;
  }
  if (!a.grad) return;
  __syncthreads();
  const float Mt = fin[0], At = fin[1], M = fin[2], As = fin[3], s = fin[4];
  T* grow = (T*)a.grad + r * a.V;
  const bool skip = s == 0.f || (n_valid == 0 && !a.lse);  // unweighted, or without a teacher: zeros
  for (int g = groups - 1; g >= 0; --g) {  // the last group is still in registers
    if (!REG && g != groups - 1) load(g);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (g * U + u) * NT + tid;
      if (i >= words) continue;
      const int v0 = i * VEC - lead;
      const uint32_t in = kl_inside<VEC>(v0, V);
      const uint32_t hit = VEC == 8 ? ((const uint8_t*)bits)[i] : ((const uint8_t*)bits)[i >> 1] >> (4 * (i & 1)) & 15u;
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = __builtin_amdgcn_exp2f((kl_elem<T>(w[u], e) - Mt) * c) * At;
      if (hit) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (hit & (1u << e))
            o[e] = __builtin_amdgcn_exp2f((kl_elem<T>(w[u], e) - M) * c) * As -
                   s * pslot[kl_find(key, a.slots - 1, v0 + e)];
      }
      if (skip) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = 0.f;
      }
      if (a.vec_out && in == (1u << VEC) - 1) {
        if constexpr (VEC == 8)
          *(uint4*)(grow + v0) = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]),
                                            pack_bf16x2(o[6], o[7]));
        else
          *(float4*)(grow + v0) = make_float4(o[0], o[1], o[2], o[3]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (in & (1u << e)) store_f<T>(grow, v0 + e, o[e]);
      }
    }
  }
}

template <typename T>
int top_kl_launch(TopKLArgs a, int64_t rows, hipStream_t s) {
  constexpr int VEC = 16 / sizeof(T);
  a.vec_out = (((uintptr_t)a.z ^ (uintptr_t)a.grad) & 15) == 0;
  a.slots = 64;
  while (a.slots < 2 * a.k) a.slots *= 2;
  const int64_t words = (a.V + 2 * (VEC - 1)) / VEC;  // at most, over the rows' alignments
  const size_t lds = (size_t)a.slots * 12 + (size_t)cdiv(words * VEC, 32) * 4 + 16;
  auto go = [&](auto kernel, int nt) -> int {
    if (lds > 48 * 1024 &&
        hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 112 * 1024) != hipSuccess)
      return fail(PD_ELAUNCH, "pd_top_kl: shared memory");
    hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(nt), lds, s, a);
    return check_launch("pd_top_kl");
  };
  if (words <= 128 * 4) return go(k_top_kl<T, 128, 4, true>, 128);
  if (words <= 256 * 8) return go(k_top_kl<T, 256, 8, true>, 256);
  if (words <= 512 * 16) return go(k_top_kl<T, 512, 16, true>, 512);
  if (words <= 1024 * 16) return go(k_top_kl<T, 1024, 16, true>, 1024);
  return go(k_top_kl<T, 1024, 16, false>, 1024);
}

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" {

int pd_top_kl(const void* z, int dtype, int64_t rows, int64_t vocab, const void* top, int top_dtype, const void* idx,
              int idx_bits, int k, const float* clean_lse, float temperature, const float* row_weight, float* kl,
              void* grad, void* stream) {
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
  const TopKLArgs a = {z, vocab, top, top_dtype, idx, idx_bits == 64, k, clean_lse, temperature, row_weight, kl, grad, 0, 0};
  hipStream_t s = (hipStream_t)stream;
  return dtype == PD_DTYPE_F32 ? top_kl_launch<float>(a, rows, s) : top_kl_launch<bf16_t>(a, rows, s);
}

}  // extern "C"
