// Causal attention over packed sequences with grouped heads, forward and backward.
//
// The rows of q [N, H, D], k and v [N, KV, D] are tokens; sequence s is rows
// [offsets[s], offsets[s+1]) and row i of it, for a query head h and its key head
// h / (H / KV), with s_ij = scale q_i . k_j over start <= j <= i:
//   L_i = log sum_j e^{s_ij}, p_ij = e^{s_ij - L_i}, o_i = sum_j p_ij v_j
//   backward, D_i = do_i . o_i and dp_ij = do_i . v_j: ds_ij = scale p_ij (dp_ij - D_i),
//   dq_i = sum_j ds_ij k_j, dk_j = sum_{h of the group} sum_i ds_ij q_i,
//   dv_j = sum_{h of the group} sum_i p_ij do_i
//
// Tiles are cut from the token axis, not from the sequences: a query tile meets the keys
// from the first of its rows' sequence starts to its last row, and a row's mask is
// start <= j <= i with a start of its own. So a launch's grid needs only N (no lengths on
// the host), and many short sequences share a tile instead of filling one each.
//
// One pass with a running maximum and sum per row (32 bits), exponentials in base 2. The
// matrix products run on MFMA 32x32 tiles (bf16 32x32x16, fp32 32x32x2), operands written
// mfma(X, Y): lane 32 hh + r supplies row r of X and of Y at k = 8 hh .. + 8 of a 16-wide
// slice, and receives out[Y row r][X row 8 g + 4 hh + e] in accumulator register 4 g + e.
// With the queries as Y a lane holds one query row's scores, its softmax needs one
// exchange between the wave's halves, and the accumulator's registers are, slice by slice,
// the Y operand of the next product; its X partner (channels as rows, positions as k) is
// read transposed from the row-major LDS image. P and dS are rounded to bf16 as operands
// where the inputs are bf16 (as they would be if stored in the inputs' type) and stay fp32
// otherwise; sums and statistics are fp32.
#include <type_traits>

#include "pd_gemm_dtl.hpp"

namespace pd {
namespace {

typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned at_u32x4;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short at_i16x4;
typedef __attribute__((address_space(3))) at_i16x4* at_lds_i16x4;

constexpr int AT_THREADS = 256;  // 4 waves of 32 rows
constexpr int AT_ROWS = 128;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float AT_NONE = -1e38f;  // a row's maximum before its first key (base-2 units)

struct AttnArgs {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int N, H, KV, D;
  const int32_t* off;
  int S;
  float scale, c2;  // c2 = scale log2 e
  int fill;         // rows of no sequence: 1 zeros, 0 left as they are
  void* out;        // [N, H, D]
  float* stats;     // [H, N]: L_i / ln 2
  const void* d_out;
  float* rowdot;  // [H, N]: D_i
  void *dq, *dk, *dv;
};

// ---------------------------------------------------------------- operand fragments
template <typename T>
struct Op;

template <>
struct Op<bf16_t> {
  typedef bf16x8 Frag;
  static __device__ inline Frag zero() { return Frag{}; }
  static __device__ inline Frag load(const bf16_t* p) { return *(const Frag*)p; }
  static __device__ inline f32x16 mma(const Frag& x, const Frag& y, f32x16 acc) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, acc, 0, 0, 0);
  }
  static __device__ inline Frag pack(const float* v) {
    return (Frag)(at_u32x4){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                            pack_bf16x2(v[6], v[7])};
  }
  static __device__ inline float dot(const Frag& a, const Frag& b, float s) {
    const at_u32x4 x = (at_u32x4)a, y = (at_u32x4)b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), s);
      s = fmaf(__uint_as_float(x[i] & 0xFFFF0000u), __uint_as_float(y[i] & 0xFFFF0000u), s);
    }
    return s;
  }
  static __device__ inline void store4(bf16_t* p, float a, float b, float c, float d) {
    *(uint2*)p = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
  }
};

template <>
struct Op<float> {
  struct Frag {
    float v[8];
  };
  static __device__ inline Frag zero() { return Frag{}; }
  static __device__ inline Frag load(const float* p) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    return Frag{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  }
  static __device__ inline f32x16 mma(const Frag& x, const Frag& y, f32x16 acc) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x.v[j], y.v[j], acc, 0, 0, 0);
    return acc;
  }
  static __device__ inline Frag pack(const float* v) {
    return Frag{{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}};
  }
  static __device__ inline float dot(const Frag& a, const Frag& b, float s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(a.v[i], b.v[i], s);
    return s;
  }
  static __device__ inline void store4(float* p, float a, float b, float c, float d) {
    *(float4*)p = make_float4(a, b, c, d);
  }
};

// ---------------------------------------------------------------- LDS images
// Row-major image of rows of DP elements in 16-byte chunks, chunk c of row R at physical
// chunk c ^ swz(R). Reads are conflict-free: 16 consecutive rows at one chunk (row
// fragments: swz is a permutation over them, over the even and the odd rows where a row is
// 128 bytes), 4 consecutive rows at 4 consecutive chunks (the transposing bf16 reads) and
// rows p and p + 4 at 8 consecutive chunks (the fp32 transposed reads).
template <typename T, int DP>
struct Img {
  static constexpr int ROWB = DP * (int)sizeof(T), CHUNKS = ROWB / 16, EPC = 16 / (int)sizeof(T);
  static __device__ inline int swz(int R) {
    if constexpr (sizeof(T) == 4) return ((R & 4) << 1) | (R & 3) | ((R >> 1) & 4);
    else if constexpr (ROWB == 128) return (((R >> 1) & 1) << 2) | ((R >> 2) & 3);
    else return ((R & 3) << 2) | ((R >> 2) & 3);
  }
  static __device__ inline int off(int R, int c) { return R * ROWB + ((c ^ swz(R)) << 4); }
  // Fragment of row R, elements 16 s + 8 hh .. + 8.
  static __device__ inline typename Op<T>::Frag rows(const char* img, int R, int s, int hh) {
    if constexpr (sizeof(T) == 2) {
      return *(const bf16x8*)(img + off(R, 2 * s + hh));
    } else {
      const float4 a = *(const float4*)(img + off(R, 4 * s + 2 * hh));
      const float4 b = *(const float4*)(img + off(R, 4 * s + 2 * hh + 1));
      return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    }
  }
  // Transposed partner of accumulator registers 8 kk .. 8 kk + 7 over image rows
  // R0 .. R0 + 31: channel 32 cb + (lane & 31) at rows R0 + 16 kk + 8 (i >> 2) + 4 hh + (i & 3).
  static __device__ inline typename Op<T>::Frag cols(const char* img, int R0, int kk, int cb, int lane) {
    if constexpr (sizeof(T) == 2) {
      const int G = lane >> 4, e = (lane >> 2) & 3, a = lane & 3;
      const int c = 4 * cb + 2 * (G & 1) + (a >> 1);
      const int R = R0 + 16 * kk + 4 * (G >> 1) + e;
      const at_i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_i16x4)(img + off(R, c) + 8 * (a & 1)));
      const at_i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_i16x4)(img + off(R + 8, c) + 8 * (a & 1)));
      return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    } else {
      const int r = lane & 31, hh = lane >> 5, c = 8 * cb + (r >> 2);
      typename Op<T>::Frag f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int R = R0 + 16 * kk + 8 * (i >> 2) + 4 * hh + (i & 3);
        f.v[i] = *(const float*)(img + off(R, c) + 4 * (r & 3));
      }
      return f;
    }
  }
};

// Rows of one operand on their way from memory into an image of ROWS rows: each thread
// carries ROWS * CHUNKS / 256 chunks. Row j of the image is row `first + j` of the operand,
// held inside [lo, hi] (a row beyond them repeats the edge: masked where it is used);
// columns from D on are zeros.
template <typename T, int DP, int ROWS>
struct Stage {
  static constexpr int CH = Img<T, DP>::CHUNKS, PER = ROWS * CH / AT_THREADS;
  static_assert(PER * AT_THREADS == ROWS * CH, "whole chunks per thread");
  uint4 w[PER];
  __device__ inline void load(const T* base, int64_t stride, int first, int lo, int hi, int D, int tid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = tid + i * AT_THREADS, c = at % CH;
      const int row = min(max(first + at / CH, lo), hi);
      w[i] = c * Img<T, DP>::EPC < D ? *(const uint4*)(base + row * stride + c * Img<T, DP>::EPC)
                                     : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ inline void store(char* img, int tid) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = tid + i * AT_THREADS;
      *(uint4*)(img + Img<T, DP>::off(at / CH, at % CH)) = w[i];
    }
  }
};

// Fragments of one row of an operand in memory (zeros from column D on).
template <typename T, int DP>
__device__ inline void at_row(const T* row, int D, int hh, typename Op<T>::Frag (&f)[DP / 16]) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) f[s] = 16 * s + 8 * hh < D ? Op<T>::load(row + 16 * s + 8 * hh) : Op<T>::zero();
}

// Key (or query) position inside a 32-row block that accumulator register i holds.
__device__ inline int at_pos(int i, int hh) { return 8 * (i >> 2) + 4 * hh + (i & 3); }
__device__ inline float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// First and one-past-last row of the sequence that holds `row`, or {row + 1, row} where
// none does. The search stays inside offsets[0 .. S] whatever they hold, and the range
// inside [0, N) and around the row.
__device__ inline void at_sequence(const int32_t* __restrict__ off, int S, int N, int row, int& start, int& end) {
  start = row + 1, end = row;
  if (row >= N || S <= 0) return;
  int a = 0, b = S + 1;  // offsets below a are <= row, from b on are > row
  while (a < b) {
    const int m = (a + b) >> 1;
    if (off[m] <= row) a = m + 1;
    else b = m;
  }
  if (a == 0 || a > S) return;
  start = min(max(off[a - 1], 0), row);
  end = min(max(off[a], row + 1), N);
}

// Smallest and largest of a value over a wave's 32 rows.
__device__ inline int at_wave_min(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ inline int at_wave_max(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

template <typename T>
__device__ inline float at_f(T v) {
  if constexpr (sizeof(T) == 2) return bf16_to_f32(v);
  else return v;
}
template <typename T>
__device__ inline float at_dot(const T* a, const T* b, int D) {
  float s = 0.f;
  for (int c = 0; c < D; c += 8) s = Op<T>::dot(Op<T>::load(a + c), Op<T>::load(b + c), s);
  return s;
}

// ---------------------------------------------------------------- rows next to a NaN
// A masked entry's weight is 0 in a tile's product, and 0 times a NaN or an infinity of a
// row that the mask hides would be a NaN. So a wave that finds a NaN in a row's result forms
// that row again here from the rows its mask allows alone: the same definition, one row per
// wave. Rows with a NaN of their own get it again.
template <typename T>
__device__ __attribute__((noinline)) void at_fwd_row(const AttnArgs* a, int h, int row, int start, int lane) {
  const int D = a->D, hk = h / (a->H / a->KV);
  const T* q = (const T*)a->q + row * a->q_row + h * a->q_head;
  const T* k = (const T*)a->k + hk * a->k_head;
  const T* v = (const T*)a->v + hk * a->v_head;
  float m = AT_NONE, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = start; j0 <= row; j0 += 64) {
    const int j = j0 + lane;
    const float s = j <= row ? at_dot<T>(q, k + j * a->k_row, D) * a->c2 : -INFINITY;
    const float mn = fmaxf(m, wave_max(s)), al = at_exp2(m - mn), p = j <= row ? at_exp2(s - mn) : 0.f;
    m = mn;
    l = l * al + wave_sum(p);
    o0 *= al, o1 *= al;
    for (int i = 0; i < 64 && j0 + i <= row; ++i) {
      const float w = __shfl(p, i, 64);
      const T* vr = v + (j0 + i) * a->v_row;
      if (lane < D) o0 = fmaf(w, at_f<T>(vr[lane]), o0);
      if (lane + 64 < D) o1 = fmaf(w, at_f<T>(vr[lane + 64]), o1);
    }
  }
  T* o = (T*)a->out + ((int64_t)row * a->H + h) * D;
  if (lane < D) store_f<T>(o, lane, o0 / l);
  if (lane + 64 < D) store_f<T>(o, lane + 64, o1 / l);
  if (a->stats && lane == 0) a->stats[(int64_t)h * a->N + row] = m + log2f(l);
}

template <typename T>
__device__ __attribute__((noinline)) void at_dq_row(const AttnArgs* a, int h, int row, int start, int lane) {
  const int D = a->D, hk = h / (a->H / a->KV);
  const T* q = (const T*)a->q + row * a->q_row + h * a->q_head;
  const T* g = (const T*)a->d_out + ((int64_t)row * a->H + h) * D;
  const T* k = (const T*)a->k + hk * a->k_head;
  const T* v = (const T*)a->v + hk * a->v_head;
  const float L = a->stats[(int64_t)h * a->N + row];
  const float dot = at_dot<T>(g, (const T*)a->out + ((int64_t)row * a->H + h) * D, D);
  float o0 = 0.f, o1 = 0.f;
  for (int j0 = start; j0 <= row; j0 += 64) {
    const int j = j0 + lane;
    float ds = 0.f;
    if (j <= row)
      ds = at_exp2(at_dot<T>(q, k + j * a->k_row, D) * a->c2 - L) * (at_dot<T>(g, v + j * a->v_row, D) - dot) * a->scale;
    for (int i = 0; i < 64 && j0 + i <= row; ++i) {
      const float w = __shfl(ds, i, 64);
      const T* kr = k + (j0 + i) * a->k_row;
      if (lane < D) o0 = fmaf(w, at_f<T>(kr[lane]), o0);
      if (lane + 64 < D) o1 = fmaf(w, at_f<T>(kr[lane + 64]), o1);
    }
  }
  T* o = (T*)a->dq + ((int64_t)row * a->H + h) * D;
  if (lane < D) store_f<T>(o, lane, o0);
  if (lane + 64 < D) store_f<T>(o, lane + 64, o1);
}

template <typename T>
__device__ __attribute__((noinline)) void at_dkv_row(const AttnArgs* a, int hk, int row, int end, int lane) {
  const int D = a->D, rep = a->H / a->KV;
  const T* k = (const T*)a->k + row * a->k_row + hk * a->k_head;
  const T* v = (const T*)a->v + row * a->v_row + hk * a->v_head;
  float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
  for (int h = hk * rep; h < (hk + 1) * rep; ++h)
    for (int i0 = row; i0 < end; i0 += 64) {
      const int i = i0 + lane;
      float p = 0.f, ds = 0.f;
      if (i < end) {
        const T* q = (const T*)a->q + i * a->q_row + h * a->q_head;
        const T* g = (const T*)a->d_out + ((int64_t)i * a->H + h) * D;
        p = at_exp2(at_dot<T>(q, k, D) * a->c2 - a->stats[(int64_t)h * a->N + i]);
        ds = p * (at_dot<T>(g, v, D) - a->rowdot[(int64_t)h * a->N + i]) * a->scale;
      }
      for (int t = 0; t < 64 && i0 + t < end; ++t) {
        const float wp = __shfl(p, t, 64), ws = __shfl(ds, t, 64);
        const T* q = (const T*)a->q + (i0 + t) * a->q_row + h * a->q_head;
        const T* g = (const T*)a->d_out + ((int64_t)(i0 + t) * a->H + h) * D;
        if (lane < D) k0 = fmaf(ws, at_f<T>(q[lane]), k0), v0 = fmaf(wp, at_f<T>(g[lane]), v0);
        if (lane + 64 < D) k1 = fmaf(ws, at_f<T>(q[lane + 64]), k1), v1 = fmaf(wp, at_f<T>(g[lane + 64]), v1);
      }
    }
  T* dk = (T*)a->dk + ((int64_t)row * a->KV + hk) * D;
  T* dv = (T*)a->dv + ((int64_t)row * a->KV + hk) * D;
  if (lane < D) store_f<T>(dk, lane, k0), store_f<T>(dv, lane, v0);
  if (lane + 64 < D) store_f<T>(dk, lane + 64, k1), store_f<T>(dv, lane + 64, v1);
}

// The kernel's own arguments, where they lie (a copy of them would live in scratch).
__device__ inline const AttnArgs* at_args() { return (const AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr(); }

// Query tile and head of a block: the heads of one key head on one XCD (blocks go round
// the 8 XCDs in turn), tiles with the most keys behind a long sequence's start first.
__device__ inline void at_query_tile(const AttnArgs& a, int& h, int& q0) {
  const int nt = (a.N + AT_ROWS - 1) / AT_ROWS, rep = a.H / a.KV;
  const int id = blockIdx.x, x = id % a.H;
  h = (x % a.KV) * rep + x / a.KV;
  q0 = (nt - 1 - id / a.H) * AT_ROWS;
}

// ---------------------------------------------------------------- forward
// Grid: query tiles x heads. Keys come through LDS BK rows at a time, the next tile's loads
// in flight during this one's products.
template <typename T, int DP, int BK>
__global__ __launch_bounds__(AT_THREADS, 2) void k_attn_fwd(AttnArgs a) {
  typedef Img<T, DP> I;
  typedef typename Op<T>::Frag Frag;
  constexpr int NS = DP / 16, NB = BK / 32, NC = DP / 32;
  __shared__ __attribute__((aligned(1024))) char Kl[BK * I::ROWB];
  __shared__ __attribute__((aligned(1024))) char Vl[BK * I::ROWB];
  __shared__ int ends[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r = lane & 31, hh = lane >> 5;
  int h, q0;
  at_query_tile(a, h, q0);
  const int hk = h / (a.H / a.KV), row = q0 + 32 * w + r;
  const T* kb = (const T*)a.k + hk * a.k_head;
  const T* vb = (const T*)a.v + hk * a.v_head;
  Frag qf[NS];
  at_row<T, DP>((const T*)a.q + (int64_t)min(row, a.N - 1) * a.q_row + h * a.q_head, a.D, hh, qf);
  int start, end;
  at_sequence(a.off, a.S, a.N, row, start, end);
  const bool in = start <= row;
  const int lo = at_wave_min(in ? start : 0x7FFFFFFF), hi = at_wave_max(in ? row + 1 : -1);
  const int inner_lo = at_wave_max(in ? start : -1);
  const bool whole = __all(in);
  if (lane == 0) ends[0][w] = lo, ends[1][w] = hi;
  __syncthreads();
  const int blo = min(min(ends[0][0], ends[0][1]), min(ends[0][2], ends[0][3]));
  const int bhi = max(max(ends[1][0], ends[1][1]), max(ends[1][2], ends[1][3]));

  float m = AT_NONE, l = 0.f;
  f32x16 o[NC] = {};
  Stage<T, DP, BK> sk, sv;
  if (blo < bhi) {
    sk.load(kb, a.k_row, blo, blo, bhi - 1, a.D, tid);
    sv.load(vb, a.v_row, blo, blo, bhi - 1, a.D, tid);
  }
  for (int j0 = blo; j0 < bhi; j0 += BK) {
    __syncthreads();
    sk.store(Kl, tid);
    sv.store(Vl, tid);
    __syncthreads();
    if (j0 + BK < bhi) {
      sk.load(kb, a.k_row, j0 + BK, blo, bhi - 1, a.D, tid);
      sv.load(vb, a.v_row, j0 + BK, blo, bhi - 1, a.D, tid);
    }
    if (j0 >= hi || j0 + BK <= lo) continue;
    f32x16 sc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      sc[b] = f32x16{};
#pragma unroll
      for (int s = 0; s < NS; ++s) sc[b] = Op<T>::mma(I::rows(Kl, 32 * b + r, s, hh), qf[s], sc[b]);
    }
    // scores in base-2 units; masked ones are -inf whatever their keys hold
    const bool inner = whole && j0 >= inner_lo && j0 + BK <= q0 + 32 * w + 1;
    float mt = -INFINITY;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float t = sc[b][i] * a.c2;
        if (!inner) {
          const int j = j0 + 32 * b + at_pos(i, hh);
          t = j >= start && j <= row ? t : -INFINITY;
        }
        sc[b][i] = t;
        mt = fmaxf(mt, t);
      }
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    if (__any(mt > m)) {
      const float mn = fmaxf(m, mt), al = at_exp2(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[c][i] *= al;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = at_exp2(sc[b][i] - m);
        l += p[i];
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const Frag pf = Op<T>::pack(p + 8 * kk);
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c] = Op<T>::mma(I::cols(Vl, 32 * b, kk, c, lane), pf, o[c]);
      }
    }
  }
  l += __shfl_xor(l, 32, 64);
  const float il = in ? 1.f / l : 0.f;
  float sum = 0.f;  // NaN where any of the row's outputs is
  if (row < a.N && (in || a.fill)) {
    T* orow = (T*)a.out + ((int64_t)row * a.H + h) * a.D;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int ch = 32 * c + 8 * g + 4 * hh;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = in ? o[c][4 * g + e] * il : 0.f;
          sum = fmaf(v[e], 0.f, sum);
        }
        if (ch < a.D) Op<T>::store4(orow + ch, v[0], v[1], v[2], v[3]);
      }
    if (in && a.stats && hh == 0) a.stats[(int64_t)h * a.N + row] = m + log2f(l);
  }
  // infinities count too: 0 times one is a NaN in another row's product
  unsigned long long bad = __ballot(in && sum != 0.f);
  bad = (bad | bad >> 32) & 0xFFFFFFFFull;
  while (bad) {
    const int i = __builtin_ctzll(bad);
    bad &= bad - 1;
    at_fwd_row<T>(at_args(), h, q0 + 32 * w + i, __shfl(start, i, 64), lane);
  }
}

// ---------------------------------------------------------------- backward: queries
// dq, and D_i for the key side. Tiles and waves as the forward's.
template <typename T, int DP, int BK>
__global__ __launch_bounds__(AT_THREADS, 2) void k_attn_dq(AttnArgs a) {
  typedef Img<T, DP> I;
  typedef typename Op<T>::Frag Frag;
  constexpr int NS = DP / 16, NB = BK / 32, NC = DP / 32;
  __shared__ __attribute__((aligned(1024))) char Kl[BK * I::ROWB];
  __shared__ __attribute__((aligned(1024))) char Vl[BK * I::ROWB];
  __shared__ int ends[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r = lane & 31, hh = lane >> 5;
  int h, q0;
  at_query_tile(a, h, q0);
  const int hk = h / (a.H / a.KV), row = q0 + 32 * w + r, rc = min(row, a.N - 1);
  const T* kb = (const T*)a.k + hk * a.k_head;
  const T* vb = (const T*)a.v + hk * a.v_head;
  Frag qf[NS], gf[NS];
  at_row<T, DP>((const T*)a.q + (int64_t)rc * a.q_row + h * a.q_head, a.D, hh, qf);
  at_row<T, DP>((const T*)a.d_out + ((int64_t)rc * a.H + h) * a.D, a.D, hh, gf);
  int start, end;
  at_sequence(a.off, a.S, a.N, row, start, end);
  const bool in = start <= row;
  const int lo = at_wave_min(in ? start : 0x7FFFFFFF), hi = at_wave_max(in ? row + 1 : -1);
  const int inner_lo = at_wave_max(in ? start : -1);
  const bool whole = __all(in);
  if (lane == 0) ends[0][w] = lo, ends[1][w] = hi;
  float dot = 0.f, L = 0.f;
  if (in) {
    Frag of[NS];
    at_row<T, DP>((const T*)a.out + ((int64_t)rc * a.H + h) * a.D, a.D, hh, of);
#pragma unroll
    for (int s = 0; s < NS; ++s) dot = Op<T>::dot(gf[s], of[s], dot);
    L = a.stats[(int64_t)h * a.N + row];
  }
  dot += __shfl_xor(dot, 32, 64);
  if (in && hh == 0) a.rowdot[(int64_t)h * a.N + row] = dot;
  __syncthreads();
  const int blo = min(min(ends[0][0], ends[0][1]), min(ends[0][2], ends[0][3]));
  const int bhi = max(max(ends[1][0], ends[1][1]), max(ends[1][2], ends[1][3]));

  f32x16 dq[NC] = {};
  Stage<T, DP, BK> sk, sv;
  if (blo < bhi) {
    sk.load(kb, a.k_row, blo, blo, bhi - 1, a.D, tid);
    sv.load(vb, a.v_row, blo, blo, bhi - 1, a.D, tid);
  }
  for (int j0 = blo; j0 < bhi; j0 += BK) {
    __syncthreads();
    sk.store(Kl, tid);
    sv.store(Vl, tid);
    __syncthreads();
    if (j0 + BK < bhi) {
      sk.load(kb, a.k_row, j0 + BK, blo, bhi - 1, a.D, tid);
      sv.load(vb, a.v_row, j0 + BK, blo, bhi - 1, a.D, tid);
    }
    if (j0 >= hi || j0 + BK <= lo) continue;
    const bool inner = whole && j0 >= inner_lo && j0 + BK <= q0 + 32 * w + 1;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f32x16 sc = {}, dp = {};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        sc = Op<T>::mma(I::rows(Kl, 32 * b + r, s, hh), qf[s], sc);
        dp = Op<T>::mma(I::rows(Vl, 32 * b + r, s, hh), gf[s], dp);
      }
      float ds[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        ds[i] = at_exp2(fmaf(sc[i], a.c2, -L)) * (dp[i] - dot);
        if (!inner) {
          const int j = j0 + 32 * b + at_pos(i, hh);
          ds[i] = j >= start && j <= row ? ds[i] : 0.f;
        }
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const Frag sf = Op<T>::pack(ds + 8 * kk);
#pragma unroll
        for (int c = 0; c < NC; ++c) dq[c] = Op<T>::mma(I::cols(Kl, 32 * b, kk, c, lane), sf, dq[c]);
      }
    }
  }
  float sum = 0.f;
  if (row < a.N && (in || a.fill)) {
    T* orow = (T*)a.dq + ((int64_t)row * a.H + h) * a.D;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int ch = 32 * c + 8 * g + 4 * hh;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = in ? dq[c][4 * g + e] * a.scale : 0.f;
          sum = fmaf(v[e], 0.f, sum);
        }
        if (ch < a.D) Op<T>::store4(orow + ch, v[0], v[1], v[2], v[3]);
      }
  }
  unsigned long long bad = __ballot(in && sum != 0.f);
  bad = (bad | bad >> 32) & 0xFFFFFFFFull;
  while (bad) {
    const int i = __builtin_ctzll(bad);
    bad &= bad - 1;
    at_dq_row<T>(at_args(), h, q0 + 32 * w + i, __shfl(start, i, 64), lane);
  }
}

// ---------------------------------------------------------------- backward: keys
// dk and dv of a tile of 128 keys and one key head: every query head of the group, and the
// queries from the tile's first row to the last row of its rows' sequences, BQ at a time.
// The accumulators hold dk^T and dv^T (a lane one key row); shared key heads are summed
// here, in head order, so the result is the same on every run. Grid: key tiles x key heads,
// the tiles with the most queries (a long sequence's first) first.
template <typename T, int DP, int BQ>
__global__ __launch_bounds__(AT_THREADS, 1) void k_attn_dkv(AttnArgs a) {
  typedef Img<T, DP> I;
  typedef typename Op<T>::Frag Frag;
  constexpr int NS = DP / 16, NB = BQ / 32, NC = DP / 32;
  __shared__ __attribute__((aligned(1024))) char Ql[BQ * I::ROWB];
  __shared__ __attribute__((aligned(1024))) char Gl[BQ * I::ROWB];
  __shared__ __attribute__((aligned(16))) float qs[2][BQ];  // L and D of the staged queries
  __shared__ int ends[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, r = lane & 31, hh = lane >> 5;
  const int hk = blockIdx.x % a.KV, k0 = blockIdx.x / a.KV * AT_ROWS, rep = a.H / a.KV;
  const int row = k0 + 32 * w + r, rc = min(row, a.N - 1);
  Frag kf[NS], vf[NS];
  at_row<T, DP>((const T*)a.k + (int64_t)rc * a.k_row + hk * a.k_head, a.D, hh, kf);
  at_row<T, DP>((const T*)a.v + (int64_t)rc * a.v_row + hk * a.v_head, a.D, hh, vf);
  int start, end;
  at_sequence(a.off, a.S, a.N, row, start, end);
  const bool in = start <= row;
  const int lo = at_wave_min(in ? row : 0x7FFFFFFF), hi = at_wave_max(in ? end : -1);
  const int inner_hi = at_wave_min(in ? end : 0x7FFFFFFF);  // smallest end of the wave's rows
  const bool whole = __all(in);
  if (lane == 0) ends[w] = hi;
  // the block's first row in a sequence: rows of none come before the first sequence or
  // behind the last, so it is the tile's first row or the first sequence's
  const int blo = max(k0, a.S > 0 ? max(a.off[0], 0) : 0);
  __syncthreads();
  const int bhi = max(max(ends[0], ends[1]), max(ends[2], ends[3]));

  f32x16 dk[NC] = {}, dv[NC] = {};
  Stage<T, DP, BQ> sq, sg;
  float st = 0.f;  // L (threads below BQ) or D (the next BQ) of one staged query
  const int nq = blo < bhi ? (bhi - blo + BQ - 1) / BQ : 0, total = nq * rep;
  auto load = [&](int t) {
    const int h = hk * rep + t / nq, i0 = blo + t % nq * BQ;
    sq.load((const T*)a.q + h * a.q_head, a.q_row, i0, blo, bhi - 1, a.D, tid);
    sg.load((const T*)a.d_out + (int64_t)h * a.D, (int64_t)a.H * a.D, i0, blo, bhi - 1, a.D, tid);
    const int64_t at = (int64_t)h * a.N + min(i0 + tid % BQ, bhi - 1);
    if (tid < 2 * BQ) st = tid < BQ ? a.stats[at] : a.rowdot[at];
  };
  if (total) load(0);
  for (int t = 0; t < total; ++t) {
    const int i0 = blo + t % nq * BQ;
    __syncthreads();
    sq.store(Ql, tid);
    sg.store(Gl, tid);
    if (tid < 2 * BQ) qs[tid / BQ][tid % BQ] = st;
    __syncthreads();
    if (t + 1 < total) load(t + 1);
    if (i0 >= hi || i0 + BQ <= lo) continue;
    const bool inner = whole && i0 >= k0 + 32 * w + 31 && i0 + BQ <= inner_hi;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f32x16 sc = {}, dp = {};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        sc = Op<T>::mma(I::rows(Ql, 32 * b + r, s, hh), kf[s], sc);
        dp = Op<T>::mma(I::rows(Gl, 32 * b + r, s, hh), vf[s], dp);
      }
      float p[16], ds[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 L = *(const float4*)&qs[0][32 * b + 8 * g + 4 * hh];
        const float4 Dt = *(const float4*)&qs[1][32 * b + 8 * g + 4 * hh];
        const float Lv[4] = {L.x, L.y, L.z, L.w}, Dv[4] = {Dt.x, Dt.y, Dt.z, Dt.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * g + e;
          p[i] = at_exp2(fmaf(sc[i], a.c2, -Lv[e]));
          ds[i] = p[i] * (dp[i] - Dv[e]);
          if (!inner) {
            const int qi = i0 + 32 * b + at_pos(i, hh);
            const bool ok = qi >= row && qi < end;
            p[i] = ok ? p[i] : 0.f;
            ds[i] = ok ? ds[i] : 0.f;
          }
        }
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const Frag pf = Op<T>::pack(p + 8 * kk), sf = Op<T>::pack(ds + 8 * kk);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          dv[c] = Op<T>::mma(I::cols(Gl, 32 * b, kk, c, lane), pf, dv[c]);
          dk[c] = Op<T>::mma(I::cols(Ql, 32 * b, kk, c, lane), sf, dk[c]);
        }
      }
    }
  }
  float sum = 0.f;
  if (row < a.N && (in || a.fill)) {
    T* krow = (T*)a.dk + ((int64_t)row * a.KV + hk) * a.D;
    T* vrow = (T*)a.dv + ((int64_t)row * a.KV + hk) * a.D;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int ch = 32 * c + 8 * g + 4 * hh;
        float x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = in ? dk[c][4 * g + e] * a.scale : 0.f;
          y[e] = in ? dv[c][4 * g + e] : 0.f;
          sum = fmaf(x[e], 0.f, fmaf(y[e], 0.f, sum));
        }
        if (ch < a.D) {
          Op<T>::store4(krow + ch, x[0], x[1], x[2], x[3]);
          Op<T>::store4(vrow + ch, y[0], y[1], y[2], y[3]);
        }
      }
  }
  unsigned long long bad = __ballot(in && sum != 0.f);
  bad = (bad | bad >> 32) & 0xFFFFFFFFull;
  while (bad) {
    const int i = __builtin_ctzll(bad);
    bad &= bad - 1;
    at_dkv_row<T>(at_args(), hk, k0 + 32 * w + i, __shfl(end, i, 64), lane);
  }
}

// ---------------------------------------------------------------- host side
int at_check(const char* what, int dtype, int64_t rows, int H, int KV, int D, const int32_t* off, int64_t n_seq,
             float scale, const int64_t* strides, const void* const* tensors, int n_tensors) {
  const std::string w(what);
  if (dtype != PD_DTYPE_F32 && dtype != PD_DTYPE_BF16) return fail(PD_EUNSUPPORTED, w + ": dtype must be fp32 or bf16");
  if (rows < 0 || n_seq < 0) return fail(PD_EINVAL, w + ": rows and sequences must be >= 0");
  if (H <= 0 || KV <= 0 || H % KV) return fail(PD_EINVAL, w + ": n_head must be a multiple of n_kv_head");
  if (D <= 0 || D % 8 || D > 128) return fail(PD_EUNSUPPORTED, w + ": head_dim must be a multiple of 8 up to 128");
  if (rows > (1 << 30) || n_seq > (1 << 30) || cdiv(rows, AT_ROWS) * H > 0x7FFFFFFF)
    return fail(PD_EUNSUPPORTED, w + ": rows too many");
  if (!std::isfinite(scale)) return fail(PD_EINVAL, w + ": scale must be finite");
  if (!rows) return PD_OK;
  if (!off) return fail(PD_EINVAL, w + ": null offsets");
  const int per = dtype == PD_DTYPE_F32 ? 4 : 8;
  for (int i = 0; i < 6; ++i)
    if (strides[i] % per) return fail(PD_EUNSUPPORTED, w + ": strides must be whole 16-byte words");
  for (int i = 0; i < n_tensors; ++i) {
    if (!tensors[i]) return fail(PD_EINVAL, w + ": null pointer");
    if ((uintptr_t)tensors[i] & 15) return fail(PD_EUNSUPPORTED, w + ": tensors must be 16-byte aligned");
  }
  return PD_OK;
}

// F(T, DP, rows a stage of LDS holds): 64 rows, 32 where a row is 512 bytes.
template <typename F>
void at_form(int dtype, int D, F&& f) {
  using std::integral_constant;
  if (dtype == PD_DTYPE_BF16) {
    if (D <= 64) f(bf16_t(0), integral_constant<int, 64>{}, integral_constant<int, 64>{});
    else f(bf16_t(0), integral_constant<int, 128>{}, integral_constant<int, 64>{});
  } else {
    if (D <= 64) f(0.f, integral_constant<int, 64>{}, integral_constant<int, 64>{});
    else f(0.f, integral_constant<int, 128>{}, integral_constant<int, 32>{});
  }
}

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" {

int pd_packed_attention_fwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                            const void* v, int64_t v_row, int64_t v_head, int dtype, int64_t rows, int n_head,
                            int n_kv_head, int head_dim, const int32_t* offsets, int64_t n_seq, float scale, int fill,
                            void* out, float* stats, void* stream) {
  const int64_t st[6] = {q_row, q_head, k_row, k_head, v_row, v_head};
  const void* ts[4] = {q, k, v, out};
  if (int rc = at_check("pd_packed_attention_fwd", dtype, rows, n_head, n_kv_head, head_dim, offsets, n_seq, scale, st, ts, 4))
    return rc;
  if (!rows) return PD_OK;
  AttnArgs a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
  a.N = (int)rows, a.H = n_head, a.KV = n_kv_head, a.D = head_dim, a.off = offsets, a.S = (int)n_seq;
  a.scale = scale, a.c2 = scale * LOG2E, a.fill = fill != 0, a.out = out, a.stats = stats;
  const unsigned grid = (unsigned)(cdiv(rows, AT_ROWS) * n_head);
  at_form(dtype, head_dim, [&](auto t, auto dp, auto bk) {
    hipLaunchKernelGGL((k_attn_fwd<decltype(t), decltype(dp)::value, decltype(bk)::value>), dim3(grid), dim3(AT_THREADS), 0,
                       (hipStream_t)stream, a);
  });
  return check_launch("pd_packed_attention_fwd");
}

size_t pd_packed_attention_bwd_workspace_size(int64_t rows, int n_head) {
  return rows > 0 && n_head > 0 ? (size_t)rows * n_head * sizeof(float) : 0;
}

int pd_packed_attention_bwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                            const void* v, int64_t v_row, int64_t v_head, int dtype, int64_t rows, int n_head,
                            int n_kv_head, int head_dim, const int32_t* offsets, int64_t n_seq, float scale, int fill,
                            const void* out, const float* stats, const void* d_out, void* dq, void* dk, void* dv,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t st[6] = {q_row, q_head, k_row, k_head, v_row, v_head};
  const void* ts[8] = {q, k, v, out, d_out, dq, dk, dv};
  if (int rc = at_check("pd_packed_attention_bwd", dtype, rows, n_head, n_kv_head, head_dim, offsets, n_seq, scale, st, ts, 8))
    return rc;
  if (!rows) return PD_OK;
  if (!stats) return fail(PD_EINVAL, "pd_packed_attention_bwd: null stats");
  if (!workspace || ((uintptr_t)workspace & 15) ||
      workspace_bytes < pd_packed_attention_bwd_workspace_size(rows, n_head))
    return fail(PD_EWORKSPACE, "pd_packed_attention_bwd: workspace");
  AttnArgs a = {};
  a.q = q, a.k = k, a.v = v;
  a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
  a.N = (int)rows, a.H = n_head, a.KV = n_kv_head, a.D = head_dim, a.off = offsets, a.S = (int)n_seq;
  a.scale = scale, a.c2 = scale * LOG2E, a.fill = fill != 0;
  a.out = const_cast<void*>(out), a.stats = const_cast<float*>(stats);
  a.d_out = d_out, a.dq = dq, a.dk = dk, a.dv = dv, a.rowdot = (float*)workspace;
  hipStream_t s = (hipStream_t)stream;
  at_form(dtype, head_dim, [&](auto t, auto dp, auto bk) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value, BK = decltype(bk)::value;
    hipLaunchKernelGGL((k_attn_dq<T, DP, BK>), dim3((unsigned)(cdiv(rows, AT_ROWS) * n_head)), dim3(AT_THREADS), 0, s, a);
    hipLaunchKernelGGL((k_attn_dkv<T, DP, BK>), dim3((unsigned)(cdiv(rows, AT_ROWS) * n_kv_head)), dim3(AT_THREADS), 0, s, a);
  });
  return check_launch("pd_packed_attention_bwd");
}

}  // extern "C"
