// Causal attention over packed sequences with grouped heads, forward and backward.
//
// The rows of q [N, H, D], k and v [N, KV, D] are tokens; sequence s is rows
// [offsets[s], offsets[s+1]) and row i of it, for a query head h and its key head
// h / (H / KV), with s_ij = scale q_i . k_j over start <= j <= i:
//   p_ij = e^{s_ij} / sum_j e^{s_ij}, o_i = sum_j p_ij v_j
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
// where the inputs are bf16 (as they would be if stored in the inputs' type: the products then
// run at the bf16 rate, 7 times the fp32 one's) and stay fp32 otherwise; sums and statistics are
// fp32. Against 64 bits a bf16 result is off by 2.0 10^-3 of its norm forward and 2.4 10^-3 with
// its gradients, where rounding the results alone is 1.5 to 1.7 10^-3.
//
// A row keeps two statistics for the backward: a reference score m_i = q_i . k_j of one of its
// keys and the log of its sum relative to that. p = 2^{c2 (q . k - m) - log}: the difference
// of two scores is exact where they are close, whatever their size. (From the log of the sum
// itself, one fp32 number, p is off by 2^-24 of the scores' size: a row's only key got weights
// of 0.96 to 1.04 at scores of 10^6 and 0 at 10^30.)
#include <algorithm>
#include <type_traits>
#include <utility>

#include "pd_gemm_dtl.hpp"

namespace pd {
namespace {

typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned at_u32x4;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short at_i16x4;
typedef __attribute__((address_space(3))) at_i16x4* at_lds_i16x4;

constexpr int AT_THREADS = 256;  // 4 waves
constexpr int AT_ROWS = 128;     // rows of a block whose waves own 32 each
constexpr int AT_SPLIT = 32;     // rows of a block whose waves share them
constexpr float LOG2E = 1.4426950408889634f;
constexpr float AT_SLACK = 8.f;    // a row is rescaled once its maximum has grown past 2^this

struct AttnArgs {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int N, H, KV, D;
  const int32_t* off;
  int S;
  // Scores take the scale's sign (flip: the sign bits of a word of q or k that change with it)
  // and exponents take them times c2 = |scale| log2 e, or fp32's smallest number where that is 0.
  float scale, c2;
  uint32_t flip;
  int fill;         // rows of no sequence: 1 zeros, 0 left as they are
  void* out;        // [N, H, D]
  void* rest;       // bf16 [N, H, D]: what rounding took off out (NULL: not kept; fp32: none)
  float* stats;     // [H, N] m_i, a score of row i, then [H, N] log2 sum_j 2^{c2 (score ij - m_i)}
  const void* d_out;
  float* rowdot;  // [H, N]: D_i
  void *dq, *dk, *dv;
  float* part;  // [hs][2][N, KV, D]: dk and dv over a share of a group's heads (hs > 1)
  int hs;       // shares
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
  // Accumulator registers 8 kk .. 8 kk + 7 as an operand.
  static __device__ inline Frag pack(const f32x16& v, int kk) {
    return (Frag)(at_u32x4){pack_bf16x2(v[8 * kk], v[8 * kk + 1]), pack_bf16x2(v[8 * kk + 2], v[8 * kk + 3]),
                            pack_bf16x2(v[8 * kk + 4], v[8 * kk + 5]), pack_bf16x2(v[8 * kk + 6], v[8 * kk + 7])};
  }
  static __device__ inline void flip(Frag& a, uint32_t signs) {
    at_u32x4 x = (at_u32x4)a;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] ^= signs;
    a = (Frag)x;
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
  static __device__ inline Frag pack(const f32x16& v, int kk) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = v[8 * kk + i];
    return f;
  }
  static __device__ inline void flip(Frag& a, uint32_t signs) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a.v[i] = __uint_as_float(__float_as_uint(a.v[i]) ^ signs);
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
  // bytes a row takes: a power of two (rows of 96 elements leave a quarter of it unused)
  static constexpr int ROWB = (DP <= 64 ? 64 : 128) * (int)sizeof(T), EPC = 16 / (int)sizeof(T);
  static __device__ inline int swz(int R) {
    if constexpr (sizeof(T) == 4) return ((R & 4) << 1) | (R & 3) | ((R >> 1) & 4);
    else if constexpr (ROWB == 128) return (((R >> 1) & 1) << 2) | ((R >> 2) & 3);
    else return ((R & 3) << 2) | ((R >> 2) & 3);
  }
  static __device__ inline int off(int R, int c) { return R * ROWB + ((c ^ swz(R)) << 4); }
  // Fragment of row R, elements 16 s + 8 hh .. + 8.
  static __device__ inline typename Op<T>::Frag rows(const char* img, int R, int s, int hh) {
    if constexpr (sizeof(T) == 2) {
      return *(const bf16x8*)(img + (off(R, hh) ^ s << 5));
    } else {
      const float4 a = *(const float4*)(img + (off(R, 2 * hh) ^ s << 6));
      const float4 b = *(const float4*)(img + (off(R, 2 * hh + 1) ^ s << 6));
      return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    }
  }
  // Transposed partner of accumulator registers 8 kk .. 8 kk + 7 over image rows
  // R0 .. R0 + 31: channel 32 cb + (lane & 31) at rows R0 + 16 kk + 8 (i >> 2) + 4 hh + (i & 3).
  static __device__ inline typename Op<T>::Frag cols(const char* img, int R0, int kk, int cb, int lane) {
    if constexpr (sizeof(T) == 2) {
      const int G = lane >> 4, e = (lane >> 2) & 3, a = lane & 3;
      const int at = off(4 * (G >> 1) + e, 2 * (G & 1) + (a >> 1)) + 8 * (a & 1) ^ cb << 6;
      const char* p = img + (R0 + 16 * kk) * ROWB;  // the swizzle is the same 16 rows on, and 8 rows on at ^ 32
      const at_i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_i16x4)(p + at));
      const at_i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_i16x4)(p + 8 * ROWB + (at ^ 32)));
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

// Rows of one operand into an image of ROWS rows by buffer loads straight to LDS, 1 KB an
// instruction, shared by NW waves. Lane l of a load writes 16 bytes at 16 l, so it fetches
// the chunk that the swizzle puts there. The descriptor ends behind row `hi`: later rows,
// and columns from D on (lanes with an offset no descriptor reaches), arrive as zeros.
template <typename T, int DP, int ROWS, int NW>
struct Loader {
  typedef Img<T, DP> I;
  static constexpr int RPI = 1024 / I::ROWB, NI = ROWS / RPI / NW;
  static_assert(NI * NW * RPI == ROWS, "whole loads per wave");
  uint32_t voff[NI];
  __device__ inline void init(int64_t stride, int D, int wave, int lane) {
    constexpr int C = I::ROWB / 16;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int R = (wave + NW * i) * RPI + lane / C, c = (lane % C) ^ I::swz(R);
      voff[i] = c * I::EPC < D ? (uint32_t)(R * stride * (int64_t)sizeof(T)) + 16 * c : 0x80000000u;
    }
  }
  // Image row 0 is row `first` (first <= hi) of the operand at `base`. (The host pass does
  // not know the descriptor's type: a body it parsed would leave the kernels without stubs.)
  __device__ inline void issue(const T* base, int64_t stride, int first, int hi, int D, char* img, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)
    const int bytes = (min(hi - first, ROWS - 1) * (int)stride + D) * (int)sizeof(T);  // a row is 8 MiB at most
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base + first * stride), (short)0,
                                                        bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < NI; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_t*)(img + (wave + NW * i) * 1024), 16, voff[i], 0, 0, 0);
#endif
  }
};

// Waits for this wave's LDS reads, so that loads issued next may overwrite what they read.
__device__ inline void at_lds_free() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
}
// Waits until at most `left` of the wave's loads are in flight.
template <int LEFT>
__device__ inline void at_landed(bool more) {
  asm volatile("" ::: "memory");
  if (more) wait_vmcnt<LEFT>();
  else wait_vmcnt<0>();
  asm volatile("" ::: "memory");
}
// Every wave's loads have landed and every wave's LDS reads are done.
__device__ inline void at_exchange() {
  asm volatile("" ::: "memory");
  wait_loads_and_lds<0>();
  lds_barrier();
}

// Fragments of one row of an operand in memory (zeros from column D on).
template <typename T, int DP>
__device__ inline void at_row(const T* row, int D, int hh, typename Op<T>::Frag (&f)[DP / 16]) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) f[s] = 16 * s + 8 * hh < D ? Op<T>::load(row + 16 * s + 8 * hh) : Op<T>::zero();
}

// Gives a row's scores the scale's sign, forward and backward in the same operands (a product
// of -q is not always the negative of q's to the bit), so that c2 is positive.
template <typename T, int NS>
__device__ inline void at_sign(const AttnArgs& a, typename Op<T>::Frag (&f)[NS]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) Op<T>::flip(f[s], a.flip);
}

// Lane i's value of each row of 16 lanes, in all of them.
template <int I>
__device__ inline float at_of(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + I, 0xf, 0xf, true));  // row_newbcast
}
template <typename F, int... I>
__device__ __forceinline__ void at_each(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
// Key (or query) position inside a 32-row block that accumulator register i holds.
__device__ inline int at_pos(int i, int hh) { return 8 * (i >> 2) + 4 * hh + (i & 3); }
// The lane again, as a value that nothing was formed from yet: LDS addresses of a loop are
// formed from it in each turn, where kept over the loop they take registers from the tiles.
__device__ inline int at_fresh(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}
__device__ inline float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// a b as a number of its own, joined with no addition: in exponents relative to a reference a b
// its rounding is one factor for all of a row's weights, as long as every use has the same.
__device__ inline float at_mul(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// The offsets in LDS, every step-th of them where there are more than the table holds: one
// round trip to memory for a block, where a search in memory takes one for each halving.
struct SeqTable {
  static constexpr int SIZE = 1024;
  int* tab;
  const int32_t* off;
  int S, N, step, n;
  __device__ inline SeqTable(const AttnArgs& a, int* lds, int tid) : tab(lds), off(a.off), S(a.S), N(a.N) {
    step = (S + SIZE) / SIZE;
    n = S / step + 1;
    for (int i = tid; i < n; i += AT_THREADS) tab[i] = off[i * step];
  }
  // After a barrier: first and one-past-last row of the sequence that holds `row`, or
  // {row + 1, row} where none does. The search stays inside offsets[0 .. S] whatever they
  // hold, and the range inside [0, N) and around the row.
  __device__ inline void find(int row, int& start, int& end) const {
    start = row + 1, end = row;
    int a = 0, b = n;  // entries below a are <= row, from b on are > row
    while (a < b) {
      const int m = (a + b) >> 1;
      if (tab[m] <= row) a = m + 1;
      else b = m;
    }
    if (a == 0 || row >= N) return;
    int at = (a - 1) * step, next;
    if (step == 1) {
      if (at >= S) return;
      start = tab[at], next = tab[at + 1];
    } else {
      for (int hi = min(at + step, S + 1); at + 1 < hi;) {  // off[at] <= row, off[hi] > row
        const int m = (at + hi) >> 1;
        if (off[m] <= row) at = m;
        else hi = m;
      }
      if (at >= S) return;
      start = off[at], next = off[at + 1];
    }
    start = min(max(start, 0), row);
    end = min(max(next, row + 1), N);
  }
};

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

// The larger of a lane's value and its partner's in the wave's other half.
__device__ inline float at_halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// ---------------------------------------------------------------- rows next to a NaN
// A masked entry's weight is 0 in a tile's product, and 0 times a NaN or an infinity of a
// row that the mask hides would be a NaN. So a wave that finds a NaN in a row's result forms
// that row again here from the rows its mask allows alone: the same definition, one row per
// wave, which is slow. Rows whose NaN or infinity is their own keep the tile's result: their
// statistics and the rows they see tell, mostly the first one looked at, and a batch that has
// diverged runs at about its normal speed. Rows of large scores come here too: their weights
// are formed from differences of scores, where a tile's take c2 s - round(c2 m).

// Products of y, its signs flipped by `signs`, with rows j0 .. j0 + 31 of an operand (those
// behind `last` read as row `last`), by the tiles' instructions and in their order, so scores
// are the tiles' own bits: register i is row j0 + at_pos(i, hh), the same in a half's 32 lanes.
template <typename T>
__device__ inline f32x16 at_products(const T* x, int64_t stride, int j0, int last, const T* y, uint32_t signs, int D,
                                     int lane) {
  const T* row = x + min(j0 + (lane & 31), last) * stride;
  f32x16 s = {};
#pragma unroll 1
  for (int c0 = 0; c0 < D; c0 += 64) {  // four slices' loads before their products
    typename Op<T>::Frag xs[4], ys[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + 16 * i + 8 * (lane >> 5);
      xs[i] = Op<T>::load(row + min(c, D - 8)), ys[i] = Op<T>::load(y + min(c, D - 8));
      if (c >= D) xs[i] = ys[i] = Op<T>::zero();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      Op<T>::flip(ys[i], signs);
      s = Op<T>::mma(xs[i], ys[i], s);
    }
  }
  return s;
}
// Adds w times each of the rows j0 .. min(j0 + 31, last) to channels lane and lane + 64; w as
// at_products gives it, 0 behind `last` (that row is read there again: one that is seen).
template <typename T>
__device__ inline void at_add_rows(const T* x, int64_t stride, int j0, int last, const f32x16& w, int D, int lane,
                                   float& o0, float& o1) {
  const bool hh = lane >> 5;
  const int c0 = min(lane, D - 1), c1 = min(lane + 64, D - 1);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float other = __shfl_xor(w[i], 32, 64), ws[2] = {hh ? other : w[i], hh ? w[i] : other};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const T* r = x + min(j0 + at_pos(i, e), last) * stride;
      o0 = fmaf(ws[e], at_f<T>(r[c0]), o0);
      o1 = fmaf(ws[e], at_f<T>(r[c1]), o1);
    }
  }
}

template <typename T>
__device__ __forceinline__ void at_fwd_row(const AttnArgs* a, int h, int row, int start, int lane) {
  const int D = a->D, hk = h / (a->H / a->KV), hh = lane >> 5;
  const T* q = (const T*)a->q + row * a->q_row + h * a->q_head;
  const T* k = (const T*)a->k + hk * a->k_head;
  const T* v = (const T*)a->v + hk * a->v_head;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = start; j0 <= row; j0 += 32) {
    f32x16 s = at_products<T>(k, a->k_row, j0, row, q, a->flip, D, lane);
    float mt = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = j0 + at_pos(i, hh) <= row ? s[i] : -INFINITY;
      mt = fmaxf(mt, s[i]);
    }
    const float mn = fmaxf(m, at_halves_max(mt)), al = m == mn ? 1.f : at_exp2((m - mn) * a->c2);
#pragma unroll
    for (int i = 0; i < 16; ++i) {  // (before the first finite score mn is -inf too)
      s[i] = s[i] == -INFINITY ? 0.f : at_exp2((s[i] - mn) * a->c2);
      sum += s[i];
    }
    const float before = l * al;
    m = mn;
    l = before + (sum + __shfl_xor(sum, 32, 64));
    // o is the result over the keys so far, so that values up to fp32's end add up to no more
    const float inv = l == 0.f ? 0.f : 1.f / l, kept = before * inv;
    o0 *= kept, o1 *= kept;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] *= inv;
    at_add_rows<T>(v, a->v_row, j0, row, s, D, lane, o0, o1);
  }
  if (l == 0.f) o0 = o1 = NAN;  // no finite score
  T* o = (T*)a->out + ((int64_t)row * a->H + h) * D;
  if (lane < D) store_f<T>(o, lane, o0);
  if (lane + 64 < D) store_f<T>(o, lane + 64, o1);
  if constexpr (sizeof(T) == 2) {
    T* rest = (T*)a->rest + ((int64_t)row * a->H + h) * D;
    if (a->rest && lane < D) store_f<T>(rest, lane, o0 - at_f<T>(o[lane]));
    if (a->rest && lane + 64 < D) store_f<T>(rest, lane + 64, o1 - at_f<T>(o[lane + 64]));
  }
  if (a->stats && lane == 0) {
    a->stats[(int64_t)h * a->N + row] = m;
    a->stats[((int64_t)a->H + h) * a->N + row] = log2f(l);
  }
}

template <typename T>
__device__ __forceinline__ void at_dq_row(const AttnArgs* a, int h, int row, int start, int lane) {
  const int D = a->D, hk = h / (a->H / a->KV), hh = lane >> 5;
  const T* q = (const T*)a->q + row * a->q_row + h * a->q_head;
  const T* g = (const T*)a->d_out + ((int64_t)row * a->H + h) * D;
  const T* k = (const T*)a->k + hk * a->k_head;
  const T* v = (const T*)a->v + hk * a->v_head;
  const float m = a->stats[(int64_t)h * a->N + row], ll = a->stats[((int64_t)a->H + h) * a->N + row];
  float dot = at_dot<T>(g, (const T*)a->out + ((int64_t)row * a->H + h) * D, D);
  if (sizeof(T) == 2) dot += at_dot<T>(g, (const T*)a->rest + ((int64_t)row * a->H + h) * D, D);
  float o0 = 0.f, o1 = 0.f;
  for (int j0 = start; j0 <= row; j0 += 32) {
    f32x16 ds = at_products<T>(k, a->k_row, j0, row, q, a->flip, D, lane);
    const f32x16 dp = at_products<T>(v, a->v_row, j0, row, g, 0, D, lane);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      ds[i] = j0 + at_pos(i, hh) <= row ? at_exp2(fmaf(ds[i] - m, a->c2, -ll)) * (dp[i] - dot) : 0.f;
    at_add_rows<T>(k, a->k_row, j0, row, ds, D, lane, o0, o1);
  }
  T* o = (T*)a->dq + ((int64_t)row * a->H + h) * D;
  if (lane < D) store_f<T>(o, lane, o0 * a->scale);
  if (lane + 64 < D) store_f<T>(o, lane + 64, o1 * a->scale);
}

template <typename T>
__device__ __forceinline__ void at_dkv_row(const AttnArgs* a, int hk, int share, int row, int end,
                                                         int lane) {
  const int D = a->D, rep = a->H / a->KV, nh = rep / a->hs, h0 = hk * rep + share * nh, hh = lane >> 5;
  const T* k = (const T*)a->k + row * a->k_row + hk * a->k_head;
  const T* v = (const T*)a->v + row * a->v_row + hk * a->v_head;
  float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
  for (int h = h0; h < h0 + nh; ++h) {
    const T* q = (const T*)a->q + h * a->q_head;
    const T* g = (const T*)a->d_out + (int64_t)h * D;
    const int64_t g_row = (int64_t)a->H * D, st = (int64_t)h * a->N, logs = (int64_t)a->H * a->N;
    for (int i0 = row; i0 < end; i0 += 32) {
      f32x16 p = at_products<T>(q, a->q_row, i0, end - 1, k, a->flip, D, lane);
      f32x16 ds = at_products<T>(g, g_row, i0, end - 1, v, 0, D, lane);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = i0 + at_pos(i, hh);
        const int64_t at = st + min(j, end - 1);
        p[i] = j < end ? at_exp2(fmaf(p[i] - a->stats[at], a->c2, -a->stats[logs + at])) : 0.f;
        ds[i] = j < end ? p[i] * (ds[i] - a->rowdot[at]) : 0.f;
      }
      at_add_rows<T>(q, a->q_row, i0, end - 1, ds, D, lane, k0, k1);
      at_add_rows<T>(g, g_row, i0, end - 1, p, D, lane, v0, v1);
    }
  }
  k0 *= a->scale, k1 *= a->scale;
  const int64_t at = ((int64_t)row * a->KV + hk) * D, plane = (int64_t)a->N * a->KV * D;
  if (a->hs > 1) {
    float* pk = a->part + 2 * share * plane + at;
    float* pv = pk + plane;
    if (lane < D) pk[lane] = k0, pv[lane] = v0;
    if (lane + 64 < D) pk[lane + 64] = k1, pv[lane + 64] = v1;
    return;
  }
  T* dk = (T*)a->dk + at;
  T* dv = (T*)a->dv + at;
  if (lane < D) store_f<T>(dk, lane, k0), store_f<T>(dv, lane, v0);
  if (lane + 64 < D) store_f<T>(dk, lane + 64, k1), store_f<T>(dv, lane + 64, v1);
}

__device__ inline bool at_odd(float x) { return !(fabsf(x) < INFINITY); }

// Whether the values of the channels lane and lane + 64 of a row are not finite.
template <typename T>
__device__ inline void at_odd_channels(const T* row, int D, int lane, bool& o0, bool& o1) {
  o0 = lane < D && at_odd(at_f<T>(row[min(lane, D - 1)]));
  o1 = lane + 64 < D && at_odd(at_f<T>(row[min(lane + 64, D - 1)]));
}

// Forms the wave's rows again that are marked in `far`, and those marked in `bad` whose NaN or
// infinity is not their own: a NaN in the query, in a key or (by channel, and infinities too)
// in a value that the row sees. `nan`: rows whose sum of weights is a NaN, which a key can have
// caused. Behind the rows' stores.
template <typename T>
__device__ __forceinline__ void at_fwd_again(const AttnArgs* a, int h, int row0, unsigned bad, unsigned nan, unsigned far,
                                             int start, int lane) {
  if (!(bad | far)) return;
  __threadfence_block();
  const int D = a->D, hk = h / (a->H / a->KV);
  const T* q = (const T*)a->q + h * a->q_head;
  const T* k = (const T*)a->k + hk * a->k_head;
  const T* v = (const T*)a->v + hk * a->v_head;
  const T* out = (const T*)a->out + ((int64_t)row0 * a->H + h) * D;
  const int64_t o_row = (int64_t)a->H * D;
  int k_from = -1, kf = 0;          // the first key row of sequence `k_from` with a NaN
  int v_from = -1, f0 = 0, f1 = 0;  // the first value rows of `v_from` that are not finite, by channel
  for (unsigned left = bad | far; left; left &= left - 1) {
    const int i = __builtin_ctz(left), row = row0 + i, first = __shfl(start, i, 64);
    if (!(far >> i & 1) && nan >> i & 1) {
      bool o0, o1;
      at_odd_channels<T>(q + row * a->q_row, D, lane, o0, o1);
      if (__any(o0 || o1)) continue;
      if (first != k_from) {
        k_from = first, kf = 0x7FFFFFFF;
        const int last = min(row0 + 31, a->N - 1);
        for (int j0 = first; j0 <= last && kf == 0x7FFFFFFF; j0 += 8) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const T* r = k + min(j0 + e, last) * a->k_row;
            const float x = at_f<T>(r[min(lane, D - 1)]), y = at_f<T>(r[min(lane + 64, D - 1)]);
            if (__any(x != x || y != y)) kf = min(kf, min(j0 + e, last));
          }
        }
      }
      if (kf <= row) continue;
    } else if (!(far >> i & 1)) {
      bool o0, o1;
      at_odd_channels<T>(out + i * o_row, D, lane, o0, o1);
      if (first != v_from) {
        v_from = first;
        bool n0 = false, n1 = false;  // channels that a row of the sequence asks for
        int last = row;
        for (unsigned more = left & bad & ~nan; more; more &= more - 1) {
          const int e = __builtin_ctz(more);
          if (__shfl(start, e, 64) != first) break;
          bool p0, p1;
          at_odd_channels<T>(out + e * o_row, D, lane, p0, p1);
          n0 |= p0, n1 |= p1;
          last = row0 + e;
        }
        f0 = n0 ? 0x7FFFFFFF : -1, f1 = n1 ? 0x7FFFFFFF : -1;
        for (int j0 = first; j0 <= last && __any(max(f0, f1) == 0x7FFFFFFF); j0 += 8) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            bool p0, p1;
            at_odd_channels<T>(v + min(j0 + e, last) * a->v_row, D, lane, p0, p1);
            if (p0) f0 = min(f0, min(j0 + e, last));
            if (p1) f1 = min(f1, min(j0 + e, last));
          }
        }
      }
      if (!__any((o0 && f0 > row) || (o1 && f1 > row))) continue;
    }
    at_fwd_row<T>(a, h, row, first, lane);
  }
}

// Forms the wave's key rows again that are marked in `bad`, but for those whose NaN or
// infinity is their own: a query that sees the row has no weights (both gradients are NaN
// then), or no finite D (dk is) and, for dv, a cotangent without a finite value in each of its
// channels. `end`: of the lane's row's sequence.
template <typename T>
__device__ __forceinline__ void at_dkv_again(const AttnArgs* a, int hk, int share, int row0, unsigned bad, int end,
                                             int lane) {
  if (!bad) return;
  __threadfence_block();
  const int D = a->D, rep = a->H / a->KV, nh = rep / a->hs, h0 = hk * rep + share * nh;
  const int64_t logs = (int64_t)a->H * a->N, plane = (int64_t)a->N * a->KV * D;
  auto channels = [&](int row, bool dv, bool& o0, bool& o1) {
    const int64_t at = ((int64_t)row * a->KV + hk) * D;
    if (a->hs > 1) at_odd_channels<float>(a->part + (2 * share + dv) * plane + at, D, lane, o0, o1);
    else at_odd_channels<T>((const T*)(dv ? a->dv : a->dk) + at, D, lane, o0, o1);
  };
  int to = -1, last_w = -1, last_d = -1, g0 = -1, g1 = -1;  // last such queries of the sequence that ends at `to`
  bool scanned = false;
  for (; bad; bad &= bad - 1) {
    const int i = __builtin_ctz(bad), row = row0 + i, e = __shfl(end, i, 64);
    if (e != to) {
      to = e, last_w = last_d = g0 = g1 = -1, scanned = false;
      for (int h = h0; h < h0 + nh; ++h)
        for (int q0 = (e - 1) & ~63, w = -1, d = -1; q0 + 63 >= row && w < 0; q0 -= 64) {
          const int q = q0 + lane;
          const int64_t at = (int64_t)h * a->N + min(q, e - 1);
          const bool in = q >= row && q < e;
          const unsigned long long bw = __ballot(in && (at_odd(a->stats[at]) || at_odd(a->stats[logs + at])));
          const unsigned long long bd = __ballot(in && at_odd(a->rowdot[at]));
          if (bw) w = q0 + 63 - __builtin_clzll(bw);
          if (bd && d < 0) d = q0 + 63 - __builtin_clzll(bd);
          last_w = max(last_w, w), last_d = max(last_d, d);
        }
    }
    if (last_w >= row) continue;
    bool o0, o1;
    if (last_d >= row) {
      channels(row, true, o0, o1);
      if (!__any(o0 || o1)) continue;
      if (!scanned) {  // the last cotangents without a finite value, by channel, for the rows left
        scanned = true;
        bool n0 = o0, n1 = o1;
        for (unsigned more = bad & (bad - 1); more; more &= more - 1) {
          const int x = __builtin_ctz(more);
          if (__shfl(end, x, 64) != e) break;
          bool p0, p1;
          channels(row0 + x, true, p0, p1);
          n0 |= p0, n1 |= p1;
        }
        for (int h = h0; h < h0 + nh; ++h)
          for (int q0 = last_d & ~63; q0 + 63 >= row && __any((n0 && g0 < 0) || (n1 && g1 < 0)); q0 -= 64) {
            const int q = q0 + lane;
            for (unsigned long long m = __ballot(q >= row && q < e && at_odd(a->rowdot[(int64_t)h * a->N + min(q, e - 1)])); m;) {
              const int x = 63 - __builtin_clzll(m);
              m ^= 1ull << x;
              bool p0, p1;
              at_odd_channels<T>((const T*)a->d_out + ((int64_t)(q0 + x) * a->H + h) * D, D, lane, p0, p1);
              if (p0) g0 = max(g0, q0 + x);
              if (p1) g1 = max(g1, q0 + x);
              if (!__any((n0 && g0 < 0) || (n1 && g1 < 0))) break;
            }
          }
      }
      if (!__any((o0 && g0 < row) || (o1 && g1 < row))) continue;
    }
    at_dkv_row<T>(a, hk, share, row, e, lane);
  }
}

// The kernel's own arguments, where they lie (a copy of them would live in scratch).
__device__ inline const AttnArgs* at_args() { return (const AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr(); }

// The order of a grid's blocks, `per` of them (heads) to a tile of ROWS rows. Blocks go to the
// CUs in turn, id mod 256, so with the tiles in order of their work, most first, and the
// first 256 turned around (by eights: the 8 XCDs keep their heads), the longest blocks share
// a CU with the shortest ones, or with none, and where they do not all fit at once the short
// ones come last. Every block forms the order itself from the offsets: thread t a key
// of tile t (its work in units of 32 rows, then t), and its rank. Up to 256 blocks a CU holds
// one and no order is better than another; beyond 256 tiles the ranks would cost more than
// the order gives, and there the tiles at the sequences' long side simply come first.
// Starts with a barrier behind which the table is whole.
template <int ROWS, bool QUERIES>
__device__ inline void at_order(const AttnArgs& a, const SeqTable& table, int (&keys)[260], int per, int tid, int& x,
                                int& first) {
  const int nt = (a.N + ROWS - 1) / ROWS, total = nt * per, id = blockIdx.x;
  __syncthreads();
  if (nt > 256 || total <= 256) {
    x = id % per;
    first = (QUERIES ? nt - 1 - id / per : id / per) * ROWS;
    return;
  }
  int c = id & 255;
  const int round = id - c;
  if (round == 0) c = (248 - (c & 248)) | (c & 7);
  const int want = (round + c) / per;
  x = (round + c) % per;
  int mine = -1;
  if (tid < nt) {
    const int lo = tid * ROWS, hi = min(lo + ROWS, a.N);
    int start, end, work = 0;
    table.find(QUERIES ? lo : hi - 1, start, end);
    if (start < end) work = QUERIES ? hi - start : end - lo;
    mine = (work + 31) >> 5 << 8 | tid;
  }
  keys[tid] = mine;
  __syncthreads();
  int rank = 0;
#pragma unroll 4
  for (int j = 0; j < nt; j += 4) {
    const int4 k = *(const int4*)&keys[j];
    rank += (k.x > mine) + (k.y > mine) + (k.z > mine) + (k.w > mine);
  }
  if (tid < nt && rank == want) keys[256] = tid;
  __syncthreads();
  first = __builtin_amdgcn_readfirstlane(keys[256]) * ROWS;
}

// Query tile and head of a block: the heads of one key head on one XCD.
template <int ROWS>
__device__ inline void at_query_tile(const AttnArgs& a, const SeqTable& table, int (&keys)[260], int tid, int& h, int& q0) {
  int x;
  at_order<ROWS, true>(a, table, keys, a.H, tid, x, q0);
  h = x % a.KV * (a.H / a.KV) + x / a.KV;
}

// The positions that a lane's row sees: `width` of them from `first` on (none: width 0).
struct Span {
  int first, width;
  __device__ inline bool sees(int j) const { return (unsigned)(j - first) < (unsigned)width; }
  // Whether any lane of the wave sees a part of [j, j + n). Where none does, a lane sees all
  // of it, or it is `hidden` from it: one value, a row's infinite log or no maximum, hides it,
  // where a part takes a comparison an entry. A wave that holds a sequence's end and the next
  // one's start meets such blocks from the one's start on.
  __device__ inline bool some(int j, int n, bool& hidden) const {
    const int b = j - first;
    hidden = b + n <= 0 || b >= width;
    return !__all(hidden || (b >= 0 && b + n <= width));
  }
};

// A lane's query row, the keys it sees, and the keys its wave meets.
struct Rows {
  int row, start;  // start: of the row's sequence, behind the row where it has none
  bool in;         // the row is in a sequence
  int lo, hi;      // keys the wave meets: [lo, hi)
  Span sees;
  __device__ inline void init(const SeqTable& t, int r) {
    int end;
    row = r;
    t.find(row, start, end);
    in = start <= row;
    lo = at_wave_min(in ? start : 0x7FFFFFFF);
    hi = at_wave_max(in ? row + 1 : -1);
    sees = {start, in ? row + 1 - start : 0};
  }
};

// Keys the block's four waves meet.
__device__ inline void at_block_range(int lo, int hi, int lane, int w, int (&ends)[2][4], int& blo, int& bhi) {
  if (lane == 0) ends[0][w] = lo, ends[1][w] = hi;
  __syncthreads();
  blo = __builtin_amdgcn_readfirstlane(min(min(ends[0][0], ends[0][1]), min(ends[0][2], ends[0][3])));
  bhi = __builtin_amdgcn_readfirstlane(max(max(ends[1][0], ends[1][1]), max(ends[1][2], ends[1][3])));
}

// Stores a lane's row from its accumulators (times f; zeros where the row has no sequence)
// and tells whether a value is a NaN or infinite.
template <typename T, int NC>
__device__ inline bool at_store_row(T* orow, T* rest, const f32x16 (&o)[NC], float f, bool in, int D, int hh) {
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int ch = 32 * c + 8 * g + 4 * hh;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = in ? o[c][4 * g + e] * f : 0.f;
        sum = fmaf(v[e], 0.f, sum);
      }
      if (ch < D) {
        Op<T>::store4(orow + ch, v[0], v[1], v[2], v[3]);
        if constexpr (sizeof(T) == 2)
          if (rest) {
            float l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) l[e] = v[e] - bf16_to_f32(f32_to_bf16(v[e]));
            Op<T>::store4(rest + ch, l[0], l[1], l[2], l[3]);
          }
      }
    }
  return in && sum != 0.f;
}

// What rounding took off m c2 in the exponents of a row's weights. Beyond AT_FAR the weights
// lose digits to it, and from 2^31 on all of them: such a row (scores of 5 10^7 and more) is
// formed again from differences.
constexpr float AT_FAR = 4.f;
__device__ inline float at_rounded_off(float m, float c2) { return fmaf(m, c2, -at_mul(m, c2)); }

// Row stats of one query: the reference score and the log of the sum.
__device__ inline void at_store_stats(const AttnArgs& a, int h, int row, float m, float l) {
  const int64_t at = (int64_t)h * a.N + row;
  a.stats[at] = m;
  a.stats[(int64_t)a.H * a.N + at] = log2f(l) - at_rounded_off(m, a.c2);
}

// ---------------------------------------------------------------- forward
// One row block's online softmax over a tile of NB key blocks: scores sc (raw, masked ones
// -inf) to weights in place, the running reference m (raw, -inf before the row's first finite
// score: that one is taken whatever its size), the lane's own part of the sum l, and the
// accumulators rescaled where a maximum has grown by more than the slack: weights stay below
// 2^8 and a tile without growth costs no pass over the accumulators.
template <int NB, int NC>
__device__ __forceinline__ void at_softmax(f32x16 (&sc)[NB], bool hidden, float& m, float& l, f32x16 (&o)[NC],
                                           float c2) {
  // four chains of maxima and of sums: one would be a wait for each of its steps
  float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i & 3] = fmaxf(x[i & 3], sc[b][i]);
  const float mt = hidden ? -INFINITY : at_halves_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
  if (__any((mt - m) * c2 > AT_SLACK)) {
    const float mn = fmaxf(m, mt), al = m == mn ? 1.f : at_exp2(at_mul(m, c2) - at_mul(mn, c2));
    m = mn;
    l *= al;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[c][i] *= al;
  }
  const float mc = hidden || m == -INFINITY ? -INFINITY : -at_mul(m, c2);  // -inf: weights 0
  float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      sc[b][i] = at_exp2(fmaf(sc[b][i], c2, mc));
      y[i & 3] += sc[b][i];
    }
  l += (y[0] + y[1]) + (y[2] + y[3]);
}

// Two LDS buffers that loads and reads alternate between. They are two variables, and the
// loops run two tiles a turn, so that the compiler can tell a load into one from a read of
// the other: where it cannot, it waits for every load in flight before the read.
#define AT_TWO_BUFFERS(bytes)                                   \
  __shared__ __attribute__((aligned(1024))) char ldsA[bytes]; \
  __shared__ __attribute__((aligned(1024))) char ldsB[bytes]

// A block of 128 query rows, 32 a wave. Grid: query tiles x heads. Keys and values come
// through LDS BK rows at a time in two buffers: one barrier a tile, behind it the next
// tile's loads go out and have this tile's products to land. The matrix cores and, in
// between, a tile's exponentials bound long sequences (16384 tokens, 16/4 heads of 128:
// 1025 us, 1070 TFLOP/s; 8192 tokens, 32/8 heads, the longest sequence 5003: 290 us), the
// longest tile's dependent chain of them short ones (0.85 us for 64 keys of D = 64 in a block
// that is alone on its CU; 8192 tokens in ten sequences of up to 2048, 12 heads: 44 us).
// fp32 rows of more than 96 channels spill 36 registers at two waves a SIMD.
template <typename T, int DP>
struct FwdCfg {
  static constexpr int BK = Img<T, DP>::ROWB == 512 ? 32 : 64, TILE = BK * Img<T, DP>::ROWB;
};
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, 2) void k_attn_fwd(AttnArgs a) {
  typedef Img<T, DP> I;
  typedef typename Op<T>::Frag Frag;
  constexpr int BK = FwdCfg<T, DP>::BK, TILE = FwdCfg<T, DP>::TILE, NS = DP / 16, NB = BK / 32, NC = DP / 32;
  AT_TWO_BUFFERS(2 * TILE);
  __shared__ int ends[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hh = lane >> 5;
  __shared__ int seq[SeqTable::SIZE];
  __shared__ __attribute__((aligned(16))) int keys[260];
  const SeqTable table(a, seq, tid);
  int h, q0;
  at_query_tile<AT_ROWS>(a, table, keys, tid, h, q0);
  const int hk = h / (a.H / a.KV), row0 = q0 + 32 * w;
  const T* kb = (const T*)a.k + hk * a.k_head;
  const T* vb = (const T*)a.v + hk * a.v_head;
  Frag qf[NS];
  at_row<T, DP>((const T*)a.q + (int64_t)min(row0 + r, a.N - 1) * a.q_row + h * a.q_head, a.D, hh, qf);
  at_sign<T>(a, qf);
  const float c2 = a.c2;
  Rows R;
  R.init(table, row0 + r);
  int blo, bhi;
  at_block_range(R.lo, R.hi, lane, w, ends, blo, bhi);
  Loader<T, DP, BK, 4> lk, lv;
  lk.init(a.k_row, a.D, w, lane);
  lv.init(a.v_row, a.D, w, lane);
  float m = -INFINITY, l = 0.f;
  f32x16 o[NC] = {};
  auto issue = [&](int j0, char* img) {
    lk.issue(kb, a.k_row, j0, bhi - 1, a.D, img, w);
    lv.issue(vb, a.v_row, j0, bhi - 1, a.D, img + TILE, w);
  };
  auto tile = [&](int j0, const char* Kl, char* next) {
    at_exchange();
    if (j0 + BK < bhi) issue(j0 + BK, next);
    if (j0 >= R.hi || j0 + BK <= R.lo) return;
    const char* Vl = Kl + TILE;
    f32x16 sc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      sc[b] = f32x16{};
#pragma unroll
      for (int s = 0; s < NS; ++s) sc[b] = Op<T>::mma(I::rows(Kl, 32 * b + r, s, hh), qf[s], sc[b]);
    }
    bool hidden;
    if (R.sees.some(j0, BK, hidden)) {  // hidden scores are -inf whatever their keys hold
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[b][i] = R.sees.sees(j0 + 32 * b + at_pos(i, hh)) ? sc[b][i] : -INFINITY;
    }
    at_softmax<NB, NC>(sc, hidden, m, l, o, c2);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const Frag pf = Op<T>::pack(sc[b], kk);
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c] = Op<T>::mma(I::cols(Vl, 32 * b, kk, c, lane), pf, o[c]);
      }
  };
  if (blo < bhi) issue(blo, ldsA);
  for (int j0 = blo; j0 < bhi; j0 += 2 * BK) {
    tile(j0, ldsA, ldsB);
    if (j0 + BK < bhi) tile(j0 + BK, ldsB, ldsA);
  }
  l += __shfl_xor(l, 32, 64);
  bool odd = false, far = false;
  if (R.row < a.N && (R.in || a.fill)) {
    const int64_t at = ((int64_t)R.row * a.H + h) * a.D;
    odd = at_store_row<T, NC>((T*)a.out + at, a.rest ? (T*)a.rest + at : nullptr, o, 1.f / l, R.in, a.D, hh);
    if (R.in && a.stats && hh == 0) at_store_stats(a, h, R.row, m, l);
    odd = odd && !(l == 0.f && m == -INFINITY);  // no finite score: NaN it is
    far = R.in && fabsf(at_rounded_off(m, c2)) > AT_FAR;
  }
  // infinities count too: 0 times one is a NaN in another row's product
  const unsigned long long bad = __ballot(odd);
  at_fwd_again<T>(at_args(), h, row0, (unsigned)(bad | bad >> 32), (unsigned)__ballot(l != l), (unsigned)__ballot(far),
                  R.start, lane);
}

// fp32 rows of four waves for a join, two waves in each of two LDS regions: value v of row r
// at chunk (v / 4) ^ (r & 15).
template <int DP>
struct Join {
  static constexpr int SHARE = 32 * (DP <= 64 ? 64 : 128) * 4;
  char *a, *b;
  __device__ inline float4* at(int w, int r, int ch) const {
    return (float4*)((w < 2 ? a : b) + (w & 1) * SHARE + ((r * (DP <= 64 ? 16 : 32) + ((ch >> 2) ^ (r & 15))) << 4));
  }
  // Writes a wave's accumulators into its share, times f.
  __device__ inline void put(int w, int r, int hh, const f32x16 (&o)[DP / 32], float f) const {
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *at(w, r, 32 * c + 8 * g + 4 * hh) =
            make_float4(o[c][4 * g] * f, o[c][4 * g + 1] * f, o[c][4 * g + 2] * f, o[c][4 * g + 3] * f);
  }
  // The four waves' values ch .. ch + 3 of row r, added in wave order.
  __device__ inline float4 sum(int r, int ch) const {
    float4 s = *at(0, r, ch);
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 v = *at(w, r, ch);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    return s;
  }
};
// Marks rows with a NaN or an infinity among the values this thread stored of row r
// (the 8 threads of a row are neighbours).
__device__ inline unsigned at_join_odd(float sum, bool in) {
  const unsigned long long b = __ballot(in && sum != 0.f);
  unsigned rows = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) rows |= (b >> (8 * i) & 0xFF ? 1u : 0u) << i;
  return rows;  // of the wave's 8 rows
}

// The same for grids too small to fill the GPU: a block of 32 query rows whose four waves
// take every fourth block of 32 keys each, through LDS of their own (no barrier in the
// loop: a block's keys come in while the last one's weights are used, its values while its
// scores are formed), and join their sums at the end.
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, 1) void k_attn_fwd_split(AttnArgs a) {
  typedef Img<T, DP> I;
  typedef typename Op<T>::Frag Frag;
  constexpr int TILE = 32 * I::ROWB, NS = DP / 16, NC = DP / 32;
  typedef Loader<T, DP, 32, 1> Ld;
  static_assert(4 * TILE >= 2 * Join<DP>::SHARE, "a region holds two waves' rows");
  AT_TWO_BUFFERS(4 * TILE);  // the waves' keys, and their values
  __shared__ float ml[2][4][32];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hh = lane >> 5;
  __shared__ int seq[SeqTable::SIZE];
  __shared__ __attribute__((aligned(16))) int keys[260];
  const SeqTable table(a, seq, tid);
  int h, q0;
  at_query_tile<AT_SPLIT>(a, table, keys, tid, h, q0);
  const int hk = h / (a.H / a.KV);
  const T* kb = (const T*)a.k + hk * a.k_head;
  const T* vb = (const T*)a.v + hk * a.v_head;
  Frag qf[NS];
  at_row<T, DP>((const T*)a.q + (int64_t)min(q0 + r, a.N - 1) * a.q_row + h * a.q_head, a.D, hh, qf);
  at_sign<T>(a, qf);
  const float c2 = a.c2;
  Rows R;
  R.init(table, q0 + r);
  Ld lk, lv;
  lk.init(a.k_row, a.D, 0, lane);
  lv.init(a.v_row, a.D, 0, lane);
  char* Kl = ldsA + w * TILE;
  char* Vl = ldsB + w * TILE;
  float m = -INFINITY, l = 0.f;
  f32x16 o[NC] = {};
  int j0 = R.lo < R.hi ? R.lo + 32 * w : R.hi;
  if (j0 < R.hi) {
    lk.issue(kb, a.k_row, j0, R.hi - 1, a.D, Kl, 0);
    lv.issue(vb, a.v_row, j0, R.hi - 1, a.D, Vl, 0);
  }
  for (; j0 < R.hi; j0 += 128) {
    const bool more = j0 + 128 < R.hi;
    at_landed<Ld::NI>(true);  // the keys; the values may still be on their way
    f32x16 sc[1] = {};
#pragma unroll
    for (int s = 0; s < NS; ++s) sc[0] = Op<T>::mma(I::rows(Kl, r, s, hh), qf[s], sc[0]);
    at_lds_free();
    if (more) lk.issue(kb, a.k_row, j0 + 128, R.hi - 1, a.D, Kl, 0);
    bool hidden;
    if (R.sees.some(j0, 32, hidden)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[0][i] = R.sees.sees(j0 + at_pos(i, hh)) ? sc[0][i] : -INFINITY;
    }
    at_softmax<1, NC>(sc, hidden, m, l, o, c2);
    at_landed<Ld::NI>(more);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const Frag pf = Op<T>::pack(sc[0], kk);
#pragma unroll
      for (int c = 0; c < NC; ++c) o[c] = Op<T>::mma(I::cols(Vl, 0, kk, c, lane), pf, o[c]);
    }
    at_lds_free();
    if (more) lv.issue(vb, a.v_row, j0 + 128, R.hi - 1, a.D, Vl, 0);
  }
  l += __shfl_xor(l, 32, 64);
  if (hh == 0) ml[0][w][r] = m, ml[1][w][r] = l;
  __syncthreads();
  // (a row without a finite score has no reference: NaN, as its softmax is, or no sequence)
  const float M = fmaxf(fmaxf(ml[0][0][r], ml[0][1][r]), fmaxf(ml[0][2][r], ml[0][3][r]));
  float sum_l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum_l += ml[1][i][r] * at_exp2(at_mul(ml[0][i][r], c2) - at_mul(M, c2));
  const Join<DP> join = {ldsA, ldsB};
  join.put(w, r, hh, o, at_exp2(at_mul(m, c2) - at_mul(M, c2)) / sum_l);
  if (w == 0 && hh == 0 && R.in && a.stats) at_store_stats(a, h, R.row, M, sum_l);
  __syncthreads();
  const unsigned long long far = __ballot(R.in && fabsf(at_rounded_off(M, c2)) > AT_FAR);
  const unsigned long long nan = __ballot(sum_l != sum_l);
  const int rr = tid >> 3, row = q0 + rr;
  const int start = __shfl(R.start, rr, 64);
  const bool in = start <= row;
  float odd = 0.f;
  if (row < a.N && (in || a.fill)) {
    const int64_t at = ((int64_t)row * a.H + h) * a.D;
#pragma unroll
    for (int q = 0; q < DP / 32; ++q) {
      const int ch = 4 * ((tid & 7) + 8 * q);
      float4 v = join.sum(rr, ch);
      if (!in) v = make_float4(0.f, 0.f, 0.f, 0.f);
      odd = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, fmaf(v.w, 0.f, odd))));
      if (ch >= a.D) continue;
      Op<T>::store4((T*)a.out + at + ch, v.x, v.y, v.z, v.w);
      if constexpr (sizeof(T) == 2)
        if (a.rest)
          Op<T>::store4((T*)a.rest + at + ch, v.x - bf16_to_f32(f32_to_bf16(v.x)), v.y - bf16_to_f32(f32_to_bf16(v.y)),
                        v.z - bf16_to_f32(f32_to_bf16(v.z)), v.w - bf16_to_f32(f32_to_bf16(v.w)));
    }
  }
  const unsigned rows = 0xFFu << (8 * w);
  at_fwd_again<T>(at_args(), h, q0, at_join_odd(odd, in) << (8 * w), (unsigned)nan, (unsigned)far & rows, R.start, lane);
}

// ---------------------------------------------------------------- backward: queries
// The row's operands: q and do fragments, its statistics, and D = do . out from the stored out
// and what rounding took off it (from the rounded out alone, D's error weighs on every key of
// a row alike and was the largest of dq's), written for the key side.
template <typename T, int DP>
struct QueryRow {
  typename Op<T>::Frag q[DP / 16], g[DP / 16];
  float m, ll, dot = 0.f;
  __device__ inline void load(const AttnArgs& a, int h, int row, int hh) {
    const int rc = min(row, a.N - 1);
    const int64_t at = ((int64_t)rc * a.H + h) * a.D, st = (int64_t)h * a.N + rc;
    m = a.stats[st], ll = a.stats[(int64_t)a.H * a.N + st];
    at_row<T, DP>((const T*)a.d_out + at, a.D, hh, g);
    typename Op<T>::Frag o[DP / 16];
    at_row<T, DP>((const T*)a.out + at, a.D, hh, o);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) dot = Op<T>::dot(g[s], o[s], dot);
    if constexpr (sizeof(T) == 2) {
      at_row<T, DP>((const T*)a.rest + at, a.D, hh, o);
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) dot = Op<T>::dot(g[s], o[s], dot);
    }
    at_row<T, DP>((const T*)a.q + (int64_t)rc * a.q_row + h * a.q_head, a.D, hh, q);
    at_sign<T>(a, q);
    dot += __shfl_xor(dot, 32, 64);
  }
  // The row has no weights or no finite D: no channel of its dq is finite.
  __device__ inline bool odd() const { return at_odd(m) || at_odd(ll) || at_odd(dot); }
};

// ds / scale of one block (images of its 32 keys and values at row R0), and dq += ds k.
template <typename T, int DP>
__device__ __forceinline__ void at_dq_block(const char* Kl, const char* Vl, int R0, int j0, const Rows& R,
                                   const QueryRow<T, DP>& Q, float c2, int lane, f32x16 (&dq)[DP / 32]) {
  typedef Img<T, DP> I;
  const int r = lane & 31, hh = lane >> 5;
  f32x16 sc = {}, dp = {};
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    sc = Op<T>::mma(I::rows(Kl, R0 + r, s, hh), Q.q[s], sc);
    dp = Op<T>::mma(I::rows(Vl, R0 + r, s, hh), Q.g[s], dp);
  }
  bool hidden;
  const bool some = R.sees.some(j0, 32, hidden);
  const float ll = hidden ? INFINITY : Q.ll;
#pragma unroll
  for (int i = 0; i < 16; ++i) sc[i] = at_exp2(fmaf(sc[i] - Q.m, c2, -ll)) * (dp[i] - Q.dot);
  if (some) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = R.sees.sees(j0 + at_pos(i, hh)) ? sc[i] : 0.f;
  }
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    const typename Op<T>::Frag sf = Op<T>::pack(sc, kk);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) dq[c] = Op<T>::mma(I::cols(Kl, R0, kk, c, lane), sf, dq[c]);
  }
}

// dq, and D_i for the key side. Tiles, waves and bounds as the forward's (8192 tokens, 32/8
// heads of 128: 385 us, 970 TFLOP/s over its three products; ten sequences, 12 heads of 64:
// 51 us, the first 10 of them for the rows of q, do, out and its rest). fp32 rows of more than
// 64 channels take one wave a SIMD: with two, 100 values spilled (D = 128: 972 -> 620 us).
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, sizeof(T) == 4 && DP > 64 ? 1 : 2) void k_attn_dq(AttnArgs a) {
  constexpr int BK = FwdCfg<T, DP>::BK, TILE = FwdCfg<T, DP>::TILE, NC = DP / 32;
  AT_TWO_BUFFERS(2 * TILE);
  __shared__ int ends[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hh = lane >> 5;
  __shared__ int seq[SeqTable::SIZE];
  __shared__ __attribute__((aligned(16))) int keys[260];
  const SeqTable table(a, seq, tid);
  int h, q0;
  at_query_tile<AT_ROWS>(a, table, keys, tid, h, q0);
  const int hk = h / (a.H / a.KV), row0 = q0 + 32 * w;
  const T* kb = (const T*)a.k + hk * a.k_head;
  const T* vb = (const T*)a.v + hk * a.v_head;
  QueryRow<T, DP> Q;
  Q.load(a, h, row0 + r, hh);
  Rows R;
  R.init(table, row0 + r);
  if (R.in && hh == 0) a.rowdot[(int64_t)h * a.N + R.row] = Q.dot;
  int blo, bhi;
  at_block_range(R.lo, R.hi, lane, w, ends, blo, bhi);
  Loader<T, DP, BK, 4> lk, lv;
  lk.init(a.k_row, a.D, w, lane);
  lv.init(a.v_row, a.D, w, lane);
  f32x16 dq[NC] = {};
  auto issue = [&](int j0, char* img) {
    lk.issue(kb, a.k_row, j0, bhi - 1, a.D, img, w);
    lv.issue(vb, a.v_row, j0, bhi - 1, a.D, img + TILE, w);
  };
  auto tile = [&](int j0, const char* Kl, char* next) {
    at_exchange();
    if (j0 + BK < bhi) issue(j0 + BK, next);
    if (j0 >= R.hi || j0 + BK <= R.lo) return;
#pragma unroll
    for (int b = 0; b < BK / 32; ++b)
      at_dq_block<T, DP>(Kl, Kl + TILE, 32 * b, j0 + 32 * b, R, Q, a.c2, lane, dq);
  };
  if (blo < bhi) issue(blo, ldsA);
  for (int j0 = blo; j0 < bhi; j0 += 2 * BK) {
    tile(j0, ldsA, ldsB);
    if (j0 + BK < bhi) tile(j0 + BK, ldsB, ldsA);
  }
  bool odd = false;
  if (R.row < a.N && (R.in || a.fill))
    odd = at_store_row<T, NC>((T*)a.dq + ((int64_t)R.row * a.H + h) * a.D, nullptr, dq, a.scale, R.in, a.D, hh);
  unsigned long long bad = __ballot(odd && !Q.odd());
  bad = (bad | bad >> 32) & 0xFFFFFFFFull;
  while (bad) {
    const int i = __builtin_ctzll(bad);
    bad &= bad - 1;
    at_dq_row<T>(at_args(), h, row0 + i, __shfl(R.start, i, 64), lane);
  }
}

// The form for small grids, as the forward's, but a block's keys are read to the end of it:
// with bf16 the next block has a buffer of its own, with fp32 it is loaded behind this one
// (its products take eight times as long, the loads' latency is small beside them).
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, 1) void k_attn_dq_split(AttnArgs a) {
  typedef Img<T, DP> I;
  constexpr int TILE = 32 * I::ROWB, NC = DP / 32, NBUF = sizeof(T) == 2 ? 2 : 1;
  typedef Loader<T, DP, 32, 1> Ld;
  constexpr int MINE = 2 * TILE;
  static_assert(4 * MINE >= 4 * Join<DP>::SHARE, "a buffer holds the waves' rows");
  AT_TWO_BUFFERS(4 * MINE);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hh = lane >> 5;
  __shared__ int seq[SeqTable::SIZE];
  __shared__ __attribute__((aligned(16))) int keys[260];
  const SeqTable table(a, seq, tid);
  int h, q0;
  at_query_tile<AT_SPLIT>(a, table, keys, tid, h, q0);
  const int hk = h / (a.H / a.KV);
  const T* kb = (const T*)a.k + hk * a.k_head;
  const T* vb = (const T*)a.v + hk * a.v_head;
  QueryRow<T, DP> Q;
  Q.load(a, h, q0 + r, hh);
  Rows R;
  R.init(table, q0 + r);
  if (R.in && hh == 0 && w == 0) a.rowdot[(int64_t)h * a.N + R.row] = Q.dot;
  Ld lk, lv;
  lk.init(a.k_row, a.D, 0, lane);
  lv.init(a.v_row, a.D, 0, lane);
  f32x16 dq[NC] = {};
  auto issue = [&](int j, char* img) {
    lk.issue(kb, a.k_row, j, R.hi - 1, a.D, img, 0);
    lv.issue(vb, a.v_row, j, R.hi - 1, a.D, img + TILE, 0);
  };
  auto block = [&](int j0, char* Kl, char* next) {
    const bool more = j0 + 128 < R.hi;
    if (NBUF == 2 && more) issue(j0 + 128, next);  // its last reads were waited for
    at_landed<2 * Ld::NI>(NBUF == 2 && more);
    at_dq_block<T, DP>(Kl, Kl + TILE, 0, j0, R, Q, a.c2, lane, dq);
    at_lds_free();
    if (NBUF == 1 && more) issue(j0 + 128, next);
  };
  char* mineA = ldsA + w * MINE;
  char* mineB = NBUF == 2 ? ldsB + w * MINE : mineA;
  const int first = R.lo < R.hi ? R.lo + 32 * w : R.hi;
  if (first < R.hi) issue(first, mineA);
  for (int j0 = first; j0 < R.hi; j0 += 256) {
    block(j0, mineA, mineB);
    if (j0 + 128 < R.hi) block(j0 + 128, mineB, mineA);
  }
  __syncthreads();
  const Join<DP> join = {ldsA, ldsA + 2 * Join<DP>::SHARE};
  join.put(w, r, hh, dq, a.scale);
  __syncthreads();
  const int rr = tid >> 3, row = q0 + rr;
  const bool in = __shfl(R.start, rr, 64) <= row;
  float odd = 0.f;
  if (row < a.N && (in || a.fill)) {
#pragma unroll
    for (int q = 0; q < DP / 32; ++q) {
      const int ch = 4 * ((tid & 7) + 8 * q);
      float4 v = join.sum(rr, ch);
      if (!in) v = make_float4(0.f, 0.f, 0.f, 0.f);
      odd = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, fmaf(v.w, 0.f, odd))));
      if (ch < a.D) Op<T>::store4((T*)a.dq + ((int64_t)row * a.H + h) * a.D + ch, v.x, v.y, v.z, v.w);
    }
  }
  const unsigned own = (unsigned)__ballot(Q.odd());
  for (unsigned bad = at_join_odd(odd, in) & ~(own >> (8 * w)); bad; bad &= bad - 1) {
    const int i = 8 * w + __builtin_ctz(bad);
    at_dq_row<T>(at_args(), h, q0 + i, __shfl(R.start, i, 64), lane);
  }
}

// ---------------------------------------------------------------- backward: keys
// A lane's key row, the queries that see it, and the queries that its wave meets.
struct Keys {
  Span seen;   // from the row itself to the end of its sequence
  int lo, hi;  // queries the wave meets: [lo, hi)
  __device__ inline int row() const { return seen.first; }
  __device__ inline int end() const { return seen.first + seen.width; }
  __device__ inline bool in() const { return seen.width > 0; }
  __device__ inline void init(const SeqTable& t, int r) {
    int start, end;
    t.find(r, start, end);
    seen = {r, end - r};
    lo = at_wave_min(in() ? r : 0x7FFFFFFF);
    hi = at_wave_max(in() ? end : -1);
  }
};

// One block of 32 queries (images at Ql, Gl; in qs their logs of sums, infinite ones for lanes
// that the queries do not see, and pairs of references and D): dv += p do, dk += ds / scale q.
// vf(s) gives fragment s of the lane's value row.
template <typename T, int DP, typename VF>
__device__ __forceinline__ void at_dkv_block(const char* Ql, const char* Gl, const float (*qs)[32], int i0,
                                    const Keys& K, const typename Op<T>::Frag (&kf)[DP / 16], VF&& vf, float c2,
                                    int lane, f32x16 (&dk)[DP / 32], f32x16 (&dv)[DP / 32]) {
  typedef Img<T, DP> I;
  typedef typename Op<T>::Frag Frag;
  if constexpr (sizeof(T) == 2) lane = at_fresh(lane);  // (fp32 has room, and more addresses)
  const int r = lane & 31, hh = lane >> 5;
  f32x16 p = {}, ds = {};
  // lane 32 hh + i and 16 lanes on: the reference and D of the query in accumulator register i.
  // One value a lane, handed to the others by the subtractions themselves: read from LDS as the
  // logs are, four words a lane, they took a tenth of the reads that bound this product (8192
  // tokens, 32/8 heads of 128: 565 -> 540 us).
  const float2 mD = ((const float2*)qs[2])[lane & 47];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    p = Op<T>::mma(I::rows(Ql, r, s, hh), kf[s], p);
    ds = Op<T>::mma(I::rows(Gl, r, s, hh), vf(s), ds);
  }
  bool hidden;
  const bool some = K.seen.some(i0, 32, hidden);
  const float* ql = qs[hidden ? 1 : 0];
  at_each([&](auto group) {
    constexpr int g = decltype(group)::value;
    const float4 l = *(const float4*)&ql[8 * g + 4 * hh];
    const float lv[4] = {l.x, l.y, l.z, l.w};
    at_each([&](auto reg) {
      constexpr int e = decltype(reg)::value, i = 4 * g + e;
      p[i] = at_exp2(fmaf(p[i] - at_of<i>(mD.x), c2, -lv[e]));
      ds[i] = p[i] * (ds[i] - at_of<i>(mD.y));
    }, std::make_integer_sequence<int, 4>{});
  }, std::make_integer_sequence<int, 4>{});
  if (some) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool ok = K.seen.sees(i0 + at_pos(i, hh));
      p[i] = ok ? p[i] : 0.f;
      ds[i] = ok ? ds[i] : 0.f;
    }
  }
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    const Frag pf = Op<T>::pack(p, kk), sf = Op<T>::pack(ds, kk);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
      dv[c] = Op<T>::mma(I::cols(Gl, 0, kk, c, lane), pf, dv[c]);
      dk[c] = Op<T>::mma(I::cols(Ql, 0, kk, c, lane), sf, dk[c]);
    }
  }
}

// Key tile, key head and share of its query heads of a block.
struct KeyTile {
  int hk, k0, share, h0, nh;
  template <int ROWS>
  __device__ inline void init(const AttnArgs& a, const SeqTable& table, int (&keys)[260], int tid) {
    const int rep = a.H / a.KV;
    int x;
    at_order<ROWS, false>(a, table, keys, a.KV * a.hs, tid, x, k0);
    hk = x % a.KV;
    share = x / a.KV;
    nh = rep / a.hs;
    h0 = hk * rep + share * nh;
  }
};

// Statistics and D of one query, for thread q of a block of 32.
struct QueryStats {
  float ll, D, m;
  __device__ inline void load(const AttnArgs& a, int h, int row) {
    const int64_t at = (int64_t)h * a.N + row;
    m = a.stats[at], ll = a.stats[at + (int64_t)a.H * a.N], D = a.rowdot[at];
  }
  __device__ inline void store(float (*qs)[32], int q) const {
    qs[0][q] = ll, qs[1][q] = INFINITY;
    // at_pos(i, hh) = q at slot 32 hh + i: the pair of lane 32 hh + i
    ((float2*)qs[2])[(q & 4) << 3 | (q >> 1 & 12) | (q & 3)] = make_float2(m, D);
  }
};

// Stores a lane's dk and dv rows, or its share's fp32 sums.
template <typename T, int DP>
__device__ inline bool at_store_keys(const AttnArgs& a, const KeyTile& t, const Keys& K, const f32x16 (&dk)[DP / 32],
                                     const f32x16 (&dv)[DP / 32], int hh) {
  if (K.row() >= a.N) return false;
  const int64_t at = ((int64_t)K.row() * a.KV + t.hk) * a.D;
  if (a.hs > 1) {
    if (!K.in()) return false;  // the sum over shares knows
    const int64_t plane = (int64_t)a.N * a.KV * a.D;
    float* pk = a.part + 2 * t.share * plane + at;
    const bool x = at_store_row<float, DP / 32>(pk, nullptr, dk, a.scale, true, a.D, hh);
    const bool y = at_store_row<float, DP / 32>(pk + plane, nullptr, dv, 1.f, true, a.D, hh);
    return x || y;
  }
  if (!K.in() && !a.fill) return false;
  const bool x = at_store_row<T, DP / 32>((T*)a.dk + at, nullptr, dk, a.scale, K.in(), a.D, hh);
  const bool y = at_store_row<T, DP / 32>((T*)a.dv + at, nullptr, dv, 1.f, K.in(), a.D, hh);
  return x || y;
}

// dk and dv of a tile of 128 keys, 32 a wave, over a share of its group's query heads: the
// queries from the tile's first row to the end of its rows' sequences, 32 at a time in two
// buffers. The accumulators hold dk^T and dv^T (a lane one key row); heads are added in
// order, so the result is the same on every run. The keys' fragments stay in registers and
// the values' in LDS: with both in registers a wave takes more than 256 and a SIMD holds
// one, with nothing beside it while it waits. LDS reads bound it beside the matrix cores: a
// wave reads 40 KB for its 32 products of a block at D = 128 (8192 tokens, 32/8 heads: 540 us,
// 920 TFLOP/s; ten sequences, 12 heads of 64: 66 us). D = 64 keeps to three waves a SIMD: 66 us,
// and 16 sequences of 512 29, where two took 68 and 36.
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, sizeof(T) == 2 ? (DP == 64 ? 3 : 2) : 1) void k_attn_dkv(AttnArgs a) {
  typedef Img<T, DP> I;
  typedef typename Op<T>::Frag Frag;
  constexpr int TILE = 32 * I::ROWB, NS = DP / 16, NC = DP / 32;
  constexpr int VLDS = sizeof(T) == 2 ? AT_ROWS * I::ROWB : 16;
  AT_TWO_BUFFERS(2 * TILE);
  __shared__ __attribute__((aligned(1024))) char Vl[VLDS];
  __shared__ __attribute__((aligned(16))) float qs[2][5][32];
  __shared__ int ends[2][4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hh = lane >> 5;
  __shared__ int seq[SeqTable::SIZE];
  __shared__ __attribute__((aligned(16))) int keys[260];
  const SeqTable table(a, seq, tid);
  KeyTile t;
  t.init<AT_ROWS>(a, table, keys, tid);
  const int row0 = t.k0 + 32 * w, rc = min(row0 + r, a.N - 1);
  if constexpr (sizeof(T) == 2) {
    Loader<T, DP, AT_ROWS, 4> lv;
    lv.init(a.v_row, a.D, w, lane);
    lv.issue((const T*)a.v + t.hk * a.v_head, a.v_row, t.k0, a.N - 1, a.D, Vl, w);
  }
  Keys K;
  K.init(table, row0 + r);
  int blo, bhi;
  at_block_range(K.lo, K.hi, lane, w, ends, blo, bhi);
  Frag kf[NS], vf[sizeof(T) == 2 ? 1 : NS];
  at_row<T, DP>((const T*)a.k + (int64_t)rc * a.k_row + t.hk * a.k_head, a.D, hh, kf);
  at_sign<T>(a, kf);
  if constexpr (sizeof(T) == 4)
    at_row<T, DP>((const T*)a.v + (int64_t)rc * a.v_row + t.hk * a.v_head, a.D, hh, vf);
  auto value = [&](int s) -> Frag {
    if constexpr (sizeof(T) == 2) return I::rows(Vl, 32 * w + r, s, hh);
    else return vf[s];
  };
  Loader<T, DP, 32, 4> lq, lg;
  lq.init(a.q_row, a.D, w, lane);
  lg.init((int64_t)a.H * a.D, a.D, w, lane);
  const int nq = blo < bhi ? (bhi - blo + 31) / 32 : 0, total = nq * t.nh;
  QueryStats st;
  int nh = t.h0, ni = blo;  // the next block to load
  auto issue = [&](char* img) {
    lq.issue((const T*)a.q + nh * a.q_head, a.q_row, ni, bhi - 1, a.D, img, w);
    lg.issue((const T*)a.d_out + (int64_t)nh * a.D, (int64_t)a.H * a.D, ni, bhi - 1, a.D, img + TILE, w);
    if (tid < 32) st.load(a, nh, min(ni + tid, bhi - 1));
    ni += 32;
    if (ni >= bhi) ni = blo, ++nh;
  };
  f32x16 dk[NC] = {}, dv[NC] = {};
  if (total) issue(ldsA);
  int i0 = blo;
  auto block = [&](int n, const char* Ql, char* next) {
    if (tid < 32) st.store(qs[n & 1], tid);
    at_exchange();
    if (n + 1 < total) issue(next);
    if (i0 < K.hi && i0 + 32 > K.lo)
      at_dkv_block<T, DP>(Ql, Ql + TILE, qs[n & 1], i0, K, kf, value, a.c2, lane, dk, dv);
    i0 += 32;
    if (i0 >= bhi) i0 = blo;
  };
  for (int n = 0; n < total; n += 2) {
    block(n, ldsA, ldsB);
    if (n + 1 < total) block(n + 1, ldsB, ldsA);
  }
  const unsigned long long bad = __ballot(at_store_keys<T, DP>(a, t, K, dk, dv, hh));
  at_dkv_again<T>(at_args(), t.hk, t.share, row0, (unsigned)(bad | bad >> 32), K.end(), lane);
}

// The form for small grids: a block of 32 keys whose four waves take every fourth block of
// 32 queries (over the share's heads), and join their sums at the end.
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, 1) void k_attn_dkv_split(AttnArgs a) {
  typedef Img<T, DP> I;
  typedef typename Op<T>::Frag Frag;
  constexpr int TILE = 32 * I::ROWB, NS = DP / 16, NC = DP / 32, NBUF = sizeof(T) == 2 ? 2 : 1;
  typedef Loader<T, DP, 32, 1> Ld;
  constexpr int MINE = 2 * TILE;
  AT_TWO_BUFFERS(4 * MINE);
  __shared__ __attribute__((aligned(16))) float qs[4][5][32];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hh = lane >> 5;
  __shared__ int seq[SeqTable::SIZE];
  __shared__ __attribute__((aligned(16))) int keys[260];
  const SeqTable table(a, seq, tid);
  KeyTile t;
  t.init<AT_SPLIT>(a, table, keys, tid);
  const int rc = min(t.k0 + r, a.N - 1);
  Frag kf[NS], vf[NS];
  at_row<T, DP>((const T*)a.k + (int64_t)rc * a.k_row + t.hk * a.k_head, a.D, hh, kf);
  at_sign<T>(a, kf);
  at_row<T, DP>((const T*)a.v + (int64_t)rc * a.v_row + t.hk * a.v_head, a.D, hh, vf);
  auto value = [&](int s) -> const Frag& { return vf[s]; };
  Keys K;
  K.init(table, t.k0 + r);
  Ld lq, lg;
  lq.init(a.q_row, a.D, 0, lane);
  lg.init((int64_t)a.H * a.D, a.D, 0, lane);
  const int nq = K.lo < K.hi ? (K.hi - K.lo + 31) / 32 : 0, total = nq * t.nh;
  QueryStats st;
  auto issue = [&](int n, char* img) {
    const int h = t.h0 + n / nq, i = K.lo + n % nq * 32;
    lq.issue((const T*)a.q + h * a.q_head, a.q_row, i, K.hi - 1, a.D, img, 0);
    lg.issue((const T*)a.d_out + (int64_t)h * a.D, (int64_t)a.H * a.D, i, K.hi - 1, a.D, img + TILE, 0);
    if (lane < 32) st.load(a, h, min(i + lane, K.hi - 1));
  };
  f32x16 dk[NC] = {}, dv[NC] = {};
  auto block = [&](int n, const char* Ql, char* next) {
    const int i0 = K.lo + n % nq * 32;
    const bool more = n + 4 < total;
    if (lane < 32) st.store(qs[w], lane);
    at_landed<0>(false);
    if (NBUF == 2 && more) issue(n + 4, next);
    at_dkv_block<T, DP>(Ql, Ql + TILE, qs[w], i0, K, kf, value, a.c2, lane, dk, dv);
    at_lds_free();
    if (NBUF == 1 && more) issue(n + 4, next);
  };
  char* mineA = ldsA + w * MINE;
  char* mineB = NBUF == 2 ? ldsB + w * MINE : mineA;
  if (w < total) issue(w, mineA);
  for (int n = w; n < total; n += 8) {
    block(n, mineA, mineB);
    if (n + 4 < total) block(n + 4, mineB, mineA);
  }
  // dk, then dv, through the same LDS
  const Join<DP> join = {ldsA, ldsA + 2 * Join<DP>::SHARE};
  float odd = 0.f;
  const int rr = tid >> 3, row = t.k0 + rr;
  const bool in = __shfl(K.seen.width, rr, 64) > 0;
  const int64_t at = ((int64_t)row * a.KV + t.hk) * a.D, plane = (int64_t)a.N * a.KV * a.D;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    join.put(w, r, hh, which ? dv : dk, which ? 1.f : a.scale);
    __syncthreads();
    if (row < a.N && (in || (a.fill && a.hs == 1))) {
#pragma unroll
      for (int q = 0; q < DP / 32; ++q) {
        const int ch = 4 * ((tid & 7) + 8 * q);
        float4 v = join.sum(rr, ch);
        if (!in) v = make_float4(0.f, 0.f, 0.f, 0.f);
        odd = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, fmaf(v.w, 0.f, odd))));
        if (ch >= a.D) continue;
        if (a.hs > 1) *(float4*)(a.part + (2 * t.share + which) * plane + at + ch) = v;
        else Op<T>::store4((T*)(which ? a.dv : a.dk) + at + ch, v.x, v.y, v.z, v.w);
      }
    }
  }
  at_dkv_again<T>(at_args(), t.hk, t.share, t.k0, at_join_odd(odd, in) << (8 * w), K.end(), lane);
}

// dk and dv as the shares' sums in share order; rows of no sequence as `fill` says. One
// thread per four values, at the rate of a copy (four shares of 8192 tokens, 8 heads of 128:
// 54 us, 5.6 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_sum(AttnArgs a) {
  const int64_t plane = (int64_t)a.N * a.KV * a.D;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  __shared__ int seq[SeqTable::SIZE];
  const SeqTable table(a, seq, threadIdx.x);
  __syncthreads();
  if (i >= 2 * plane) return;
  const int which = i >= plane;
  const int64_t at = i - which * plane;
  int start, end;
  table.find((int)(at / ((int64_t)a.KV * a.D)), start, end);
  const bool in = end > start;
  if (!in && !a.fill) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (in)
    for (int h = 0; h < a.hs; ++h) {
      const float4 v = *(const float4*)(a.part + (2 * h + which) * plane + at);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  Op<T>::store4((T*)(which ? a.dv : a.dk) + at, s.x, s.y, s.z, s.w);
}

// ---------------------------------------------------------------- host side
int at_check(const char* what, int dtype, int64_t rows, int H, int KV, int D, const int32_t* off, int64_t n_seq,
             float scale, const int64_t* strides, const void* const* tensors, int n_tensors) {
  const std::string w(what);
  if (dtype != PD_DTYPE_F32 && dtype != PD_DTYPE_BF16) return fail(PD_EUNSUPPORTED, w + ": dtype must be fp32 or bf16");
  if (rows < 0 || n_seq < 0) return fail(PD_EINVAL, w + ": rows and sequences must be >= 0");
  if (H <= 0 || KV <= 0 || H % KV) return fail(PD_EINVAL, w + ": n_head must be a multiple of n_kv_head");
  if (D <= 0 || D % 8 || D > 128) return fail(PD_EUNSUPPORTED, w + ": head_dim must be a multiple of 8 up to 128");
  if (rows > (1 << 30) || n_seq > (1 << 30) || cdiv(rows, AT_SPLIT) * H > 0x7FFFFFFF)
    return fail(PD_EUNSUPPORTED, w + ": rows too many");
  if (!std::isfinite(scale * LOG2E)) return fail(PD_EINVAL, w + ": scale (times log2 e, as the kernels take it) must be finite");
  if (!rows) return PD_OK;
  if (!off) return fail(PD_EINVAL, w + ": null offsets");
  const int per = dtype == PD_DTYPE_F32 ? 4 : 8;
  for (int i = 0; i < 6; ++i)
    if (strides[i] % per) return fail(PD_EUNSUPPORTED, w + ": strides must be whole 16-byte words");
  for (int i = 0; i < 6; i += 2)  // a tile's 128 rows within a 31-bit offset
    if (strides[i] < 0 || strides[i] * (per == 4 ? 4 : 2) > (1 << 23))
      return fail(PD_EUNSUPPORTED, w + ": row strides of at most 8 MiB");
  if ((int64_t)H * D * (per == 4 ? 4 : 2) > (1 << 23)) return fail(PD_EUNSUPPORTED, w + ": rows of at most 8 MiB");
  for (int i = 0; i < n_tensors; ++i) {
    if (!tensors[i]) return fail(PD_EINVAL, w + ": null pointer");
    if ((uintptr_t)tensors[i] & 15) return fail(PD_EUNSUPPORTED, w + ": tensors must be 16-byte aligned");
  }
  return PD_OK;
}

// F(T, DP): the widths the kernels are built for.
template <typename F>
void at_form(int dtype, int D, F&& f) {
  using std::integral_constant;
  auto width = [&](auto t) {
    if (D <= 64) f(t, integral_constant<int, 64>{});
    else if (D <= 96) f(t, integral_constant<int, 96>{});
    else f(t, integral_constant<int, 128>{});
  };
  if (dtype == PD_DTYPE_BF16) width(bf16_t(0));
  else width(0.f);
}

// Blocks of 128 rows below which the 32-row forms run: one a CU (bf16, 4096 tokens in four
// sequences, 12 heads: D = 64 forward, dq, dk/dv 36, 44, 59 us against 34, 49, 83 split;
// D = 128 47, 61, 90 against 57, 112, 129; 2048 tokens, 192 blocks, D = 64: 25, 30, 41 against
// 17, 26, 35). For queries in fp32, whose products take eight times as long, the finer tiles
// gain up to two a CU (D = 64: 4096 tokens, 12 heads forward, dq 141, 198 us against 115, 162;
// 8192 tokens 240, 344 against 264, 370; the key side is even at 4096 tokens: 263 against
// 233, D = 128 497 against 600).
constexpr int64_t AT_FULL = 256;

bool at_query_split(int64_t rows, int H, int dtype) {
  return cdiv(rows, AT_ROWS) * H < (dtype == PD_DTYPE_BF16 ? AT_FULL : 2 * AT_FULL);
}

// Shares of a group's heads and the tile of the key side: as few shares as fill the GPU
// eight times with 128-key tiles, else one head a share, else 32-key tiles whose waves share
// the queries, two blocks a CU.
struct KeyPlan {
  int hs;
  bool split;
};
KeyPlan at_key_plan(int64_t rows, int H, int KV) {
  const int rep = H / KV;
  for (int hs = 1; hs <= rep; ++hs)
    if (rep % hs == 0 && cdiv(rows, AT_ROWS) * KV * hs >= 8 * AT_FULL) return {hs, false};
  if (cdiv(rows, AT_ROWS) * KV * rep >= AT_FULL) return {rep, false};
  for (int hs = 1; hs <= rep; ++hs)
    if (rep % hs == 0 && cdiv(rows, AT_SPLIT) * KV * hs >= 2 * AT_FULL) return {hs, true};
  return {rep, true};
}

void at_fill_args(AttnArgs& a, const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                  const void* v, int64_t v_row, int64_t v_head, int64_t rows, int H, int KV, int D, const int32_t* off,
                  int64_t n_seq, float scale, int fill, int dtype) {
  a.q = q, a.k = k, a.v = v;
  a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
  a.N = (int)rows, a.H = H, a.KV = KV, a.D = D, a.off = off, a.S = (int)n_seq;
  a.scale = scale, a.c2 = std::max(std::fabs(scale * LOG2E), 0x1p-149f);
  a.flip = scale >= 0.f ? 0u : dtype == PD_DTYPE_BF16 ? 0x80008000u : 0x80000000u;
  a.fill = fill != 0, a.hs = 1;
}

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" {

int pd_packed_attention_fwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                            const void* v, int64_t v_row, int64_t v_head, int dtype, int64_t rows, int n_head,
                            int n_kv_head, int head_dim, const int32_t* offsets, int64_t n_seq, float scale, int fill,
                            void* out, void* out_rest, float* stats, void* stream) {
  const int64_t st[6] = {q_row, q_head, k_row, k_head, v_row, v_head};
  const void* ts[4] = {q, k, v, out};
  if (int rc = at_check("pd_packed_attention_fwd", dtype, rows, n_head, n_kv_head, head_dim, offsets, n_seq, scale, st, ts, 4))
    return rc;
  if (!rows) return PD_OK;
  if (dtype == PD_DTYPE_F32 && out_rest) return fail(PD_EINVAL, "pd_packed_attention_fwd: out_rest goes with bf16");
  if ((uintptr_t)out_rest & 15) return fail(PD_EUNSUPPORTED, "pd_packed_attention_fwd: tensors must be 16-byte aligned");
  AttnArgs a = {};
  at_fill_args(a, q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, rows, n_head, n_kv_head, head_dim, offsets, n_seq,
               scale, fill, dtype);
  a.out = out, a.rest = out_rest, a.stats = stats;
  const bool split = at_query_split(rows, n_head, dtype);
  const unsigned grid = (unsigned)(cdiv(rows, split ? AT_SPLIT : AT_ROWS) * n_head);
  at_form(dtype, head_dim, [&](auto t, auto dp) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value;
    if (split) hipLaunchKernelGGL((k_attn_fwd_split<T, DP>), dim3(grid), dim3(AT_THREADS), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((k_attn_fwd<T, DP>), dim3(grid), dim3(AT_THREADS), 0, (hipStream_t)stream, a);
  });
  return check_launch("pd_packed_attention_fwd");
}

size_t pd_packed_attention_bwd_workspace_size(int64_t rows, int n_head, int n_kv_head, int head_dim) {
  if (rows <= 0 || n_head <= 0 || n_kv_head <= 0 || head_dim <= 0 || n_head % n_kv_head) return 0;
  const int hs = at_key_plan(rows, n_head, n_kv_head).hs;
  const size_t dots = (size_t)cdiv(rows * n_head, 4) * 16;
  return dots + (hs > 1 ? (size_t)hs * 2 * rows * n_kv_head * head_dim * sizeof(float) : 0);
}

int pd_packed_attention_bwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                            const void* v, int64_t v_row, int64_t v_head, int dtype, int64_t rows, int n_head,
                            int n_kv_head, int head_dim, const int32_t* offsets, int64_t n_seq, float scale, int fill,
                            const void* out, const void* out_rest, const float* stats, const void* d_out, void* dq,
                            void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t st[6] = {q_row, q_head, k_row, k_head, v_row, v_head};
  const void* ts[8] = {q, k, v, out, d_out, dq, dk, dv};
  if (int rc = at_check("pd_packed_attention_bwd", dtype, rows, n_head, n_kv_head, head_dim, offsets, n_seq, scale, st, ts, 8))
    return rc;
  if (!rows) return PD_OK;
  if (!stats || (dtype == PD_DTYPE_BF16 && !out_rest))
    return fail(PD_EINVAL, "pd_packed_attention_bwd: the forward's stats (and out_rest with bf16) are needed");
  if (dtype == PD_DTYPE_F32 && out_rest) return fail(PD_EINVAL, "pd_packed_attention_bwd: out_rest goes with bf16");
  if ((uintptr_t)out_rest & 15) return fail(PD_EUNSUPPORTED, "pd_packed_attention_bwd: tensors must be 16-byte aligned");
  if (!workspace || ((uintptr_t)workspace & 15) ||
      workspace_bytes < pd_packed_attention_bwd_workspace_size(rows, n_head, n_kv_head, head_dim))
    return fail(PD_EWORKSPACE, "pd_packed_attention_bwd: workspace");
  AttnArgs a = {};
  at_fill_args(a, q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, rows, n_head, n_kv_head, head_dim, offsets, n_seq,
               scale, fill, dtype);
  a.out = const_cast<void*>(out), a.rest = const_cast<void*>(out_rest), a.stats = const_cast<float*>(stats);
  a.d_out = d_out, a.dq = dq, a.dk = dk, a.dv = dv, a.rowdot = (float*)workspace;
  const KeyPlan plan = at_key_plan(rows, n_head, n_kv_head);
  a.hs = plan.hs;
  a.part = (float*)((char*)workspace + (size_t)cdiv(rows * n_head, 4) * 16);
  hipStream_t s = (hipStream_t)stream;
  const bool split = at_query_split(rows, n_head, dtype);
  const dim3 block(AT_THREADS), gq((unsigned)(cdiv(rows, split ? AT_SPLIT : AT_ROWS) * n_head)),
      gk((unsigned)(cdiv(rows, plan.split ? AT_SPLIT : AT_ROWS) * n_kv_head * plan.hs)),
      gs((unsigned)cdiv(2 * rows * n_kv_head * head_dim, 1024));
  at_form(dtype, head_dim, [&](auto t, auto dp) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value;
    if (split) hipLaunchKernelGGL((k_attn_dq_split<T, DP>), gq, block, 0, s, a);
    else hipLaunchKernelGGL((k_attn_dq<T, DP>), gq, block, 0, s, a);
    if (plan.split) hipLaunchKernelGGL((k_attn_dkv_split<T, DP>), gk, block, 0, s, a);
    else hipLaunchKernelGGL((k_attn_dkv<T, DP>), gk, block, 0, s, a);
    if (plan.hs > 1) hipLaunchKernelGGL((k_attn_dkv_sum<T>), gs, block, 0, s, a);
  });
  return check_launch("pd_packed_attention_bwd");
}

}  // extern "C"
