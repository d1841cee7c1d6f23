// Softmax cross entropy over a vocabulary, from activations and head, and its gradients. The loss keeps no logits;
// its gradients form them again, or take what a loss kept for them.
//
//   z = act head^T, loss_i = log(sum_v e^{z_iv}) - z_i,t_i
//   G = g (softmax(z) - 1_t), d_act = G head, d_head = G^T act
//
// Bound by the matrix cores: 2 N d V operations forward, and backward 2 N d V to form the logits
// again and 2 N d V for each gradient. bf16: the forward's product keeps each tile's maximum and
// sum for every row and the target's logit, and a second kernel merges tiles in a fixed order; the
// logits stay in registers. The backward goes over the vocabulary in pieces of which G (bf16) fits
// CE_PIECE bytes of workspace: one product whose epilogue writes G, then both gradients from it.
// The softmax is formed from the row's maximum and the sum of the others relative to it, kept apart: the log of the sum
// alone would round a probability near one to 1e-6, and a sum that holds the maximum's 1 what is one less it.
//
// Where a chunk of positions' softmax fits CE_KEPT it is kept in 16 bits instead (EpiCEKeep; fp32: the logits, EpiCEKeepF), 6 N d V
// in all: in one call for weights known beforehand, where G takes its place, or from the loss to its gradients (pd_streamed_ce_kept_*),
// where G is as large again. bf16, loss and both gradients: 8192 x 768 over 50277 2790 us with the logits formed again (1.1 GB beside
// inputs), 2590 kept (2.0 GB; product and epilogue 835, apply 360, d_act 662 and its slabs' sum 36, d_head 713); three quarters of
// 4096 x 4096 over 131072 11.1 and 8.9 ms (2700, 300, 2900, 2900: 1.14 PFLOP/s).
// fp32, 903 of 1003 x 1000 over 32003: 1515 us formed again, 1190 kept (product 423, apply 39, d_act 421, d_head 393).
//
// Positions whose target lies outside the vocabulary do not count (nor, backward, those of weight
// zero): their rows are left out of a dense copy of the activations, so they cost no products and
// what they hold reaches nothing. How many count only the device knows: grids cover all positions
// and the products read the count (MODE_COUNTED).
//
// fp32: the matrix cores take bf16 at sixteen times fp32's rate, so each operand enters as three bf16 parts
// (8 + 8 + 8 bits: exact) and a product as the six products of parts that reach 2^-24 of it, with fp32 sums. The
// parts are formed between a tile's loads and LDS (k_gemm_parts).
#include <algorithm>
#include <cmath>

#include "pd_gemm_dtl.hpp"

namespace pd {
namespace {

constexpr size_t CE_PIECE = (size_t)1024 << 20;
// The one-call form keeps a chunk of positions' softmax (16 bits) below this, the end of a product's
// operands.
constexpr size_t CE_KEPT = ((size_t)1 << 31) - ((size_t)1 << 22);
constexpr int CE_SPAN = 64;
constexpr float LOG2E = 1.4426950408889634f;

struct CETargets {
  const void* p;
  int bits;
  int64_t ignore, V;
  // the target of position i, or -1 where it does not count
  __device__ inline int at(int64_t i) const {
    const int64_t t = bits == 64 ? ((const int64_t*)p)[i] : ((const int32_t*)p)[i];
    return t == ignore || t < 0 || t >= V ? -1 : (int)t;
  }
};

// rows[0 .. count) = the positions that count, in order; pos[i] = position i's place among them or
// -1. With `loss` those that do not get loss 0 and, with `stats`, statistics (0, 0). One block, about 1 us for 1024 positions.
__global__ __launch_bounds__(1024) void k_ce_compact(CETargets t, const float* __restrict__ g, int64_t N,
                                                     int32_t* __restrict__ rows, int32_t* __restrict__ pos,
                                                     int32_t* __restrict__ count, float* __restrict__ loss,
                                                     float2* __restrict__ stats) {
  __shared__ int32_t part[2][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t base = 0;
  for (int64_t i0 = 0, it = 0; i0 < N; i0 += 1024, it ^= 1) {
    const int64_t i = i0 + threadIdx.x;
    const bool on = i < N && t.at(i) >= 0 && !(g && g[i] == 0.f);
    const unsigned long long hit = __ballot(on);
    if (lane == 0) part[it][wave] = __popcll(hit);
    __syncthreads();
    int32_t before = base, total = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += part[it][w];
      total += part[it][w];
    }
    base += total;
    const int32_t at = before + __popcll(hit & ((1ull << lane) - 1));
    if (on) rows[at] = (int32_t)i;
    if (i < N) {
      if (pos) pos[i] = on ? at : -1;
      if (loss && !on) {
        loss[i] = 0.f;
        if (stats) stats[i] = make_float2(0.f, 0.f);
      }
    }
  }
  if (threadIdx.x == 0) *count = base;
}

// dst[r] = src[rows[r]] for r < count, n words of T a row.
template <typename T>
__global__ __launch_bounds__(256) void k_ce_gather(const T* __restrict__ src, int64_t n, const int32_t* __restrict__ rows,
                                                   const int32_t* __restrict__ count, T* __restrict__ dst) {
  const int64_t total = *count * n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / n;
    dst[i] = src[(int64_t)rows[r] * n + (i - r * n)];
  }
}
void ce_gather(bool half, const void* src, int64_t N, int64_t d, const int32_t* rows, const int32_t* count, void* dst,
               hipStream_t s) {
  const int64_t n = half ? d / 8 : d;
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(N * n, 256), 4096));
  if (half) hipLaunchKernelGGL(k_ce_gather<uint4>, grid, dim3(256), 0, s, (const uint4*)src, n, rows, count, (uint4*)dst);
  else hipLaunchKernelGGL(k_ce_gather<float>, grid, dim3(256), 0, s, (const float*)src, n, rows, count, (float*)dst);
}

// d_act[i] = the sum over `slabs` of the row of position i, of the positions whose place is in
// [first, first + R); zeros where it does not count.
template <typename T>
__global__ __launch_bounds__(256) void k_ce_scatter(const float* __restrict__ part, int slabs, int64_t stride,
                                                    int64_t N, int64_t d, const int32_t* __restrict__ pos,
                                                    int64_t first, int64_t R,
                                                    T* __restrict__ d_act) {
  const bool vec = d % 4 == 0;  // bf16: d is a multiple of 8
  const int64_t q = vec ? d / 4 : d, total = N * q;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / q, c = (i - r * q) * (vec ? 4 : 1);
    const int64_t at = pos[r] < 0 ? -1 : pos[r] - first;
    if (at < 0 ? pos[r] >= 0 : at >= R) continue;  // another chunk's
    if (vec) {
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at >= 0)
        for (int k = 0; k < slabs; ++k) {
          const float4 v = *(const float4*)(part + k * stride + at * d + c);
          s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
      if constexpr (sizeof(T) == 2) *(uint2*)(d_act + r * d + c) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
      else *(float4*)(d_act + r * d + c) = s;
    } else {
      float s = 0.f;
      if (at >= 0)
        for (int k = 0; k < slabs; ++k) s += part[k * stride + at * d + c];
      store_f<T>(d_act, r * d + c, s);
    }
  }
}

__device__ inline float ce_exp(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// Of two sets of columns: (maximum m, sum of e^{z - m} less the maximum's own 1); (-inf, -1) is none.
__device__ inline void ce_merge(float2& o, float2 q) {
  const bool first = o.x >= q.x;
  const float2 hi = first ? o : q, lo = first ? q : o;
  o = make_float2(hi.x, hi.y + (lo.y + 1.f) * (lo.x == hi.x ? 1.f : expf(lo.x - hi.x)));
}

// Forward epilogue: each row's maximum and the others' sum over the tile's columns, to part[row][tile], and
// the target's logit. A lane holds 16 columns of 32 in its row, its neighbour 32 lanes on the others.
template <class CFG>
struct EpiCEStats {
  static constexpr int LDS_BYTES = CFG::WN * CFG::BM * 8;
  struct Args {
    float2* part;
    int64_t n_tiles;
    float* target;           // [M]
    const int32_t* rows;     // NULL: row r is position r
    CETargets t;
    int64_t first = 0;       // the piece's first column of the vocabulary (whole tiles)
  };
  template <class, typename>
  __device__ static void run(const GemmArgs& p, const Args& a, const TileJob& t, int wm, int wn, int tid,
                             f32x16 (&z)[CFG::TM][CFG::TN], char* smem) {
    if (t.n0 + CFG::BN <= p.N) run_t<true>(p, a, t, wm, wn, tid, z, smem);
    else run_t<false>(p, a, t, wm, wn, tid, z, smem);
  }
  template <bool FULL>
  __device__ static void run_t(const GemmArgs& p, const Args& a, const TileJob& t, int wm, int wn, int tid,
                               f32x16 (&z)[CFG::TM][CFG::TN], char* smem) {
    const int lane = tid & 63;
    float2* red = (float2*)smem;  // [WN][BM]
    lds_write_barrier();          // the k loop's stage buffers are free
#pragma unroll
    for (int i = 0; i < CFG::TM; ++i) {
      const int rl = wm * CFG::WTM + i * 32 + (lane & 31);
      float m, r;
      row_stats<FULL>(p, a, t, t.m0 + rl, t.n0 + wn * CFG::WTN + 4 * (lane >> 5), z[i], m, r);
      if (lane < 32) red[wn * CFG::BM + rl] = make_float2(m, r);
    }
    lds_write_barrier();
    store(a, t, tid, red);
  }
  // A row's maximum m and the others' sum r over the wave's columns (`first`: the lane's first one); z becomes
  // e^{z - m}, and the target's logit is kept. r leaves the maximum's 1 out from the start: added to it, a rest below
  // 2^-24 would be lost. Entries equal to 1 are counted by what their fractions lack of the sum.
  template <bool FULL>
  __device__ static void row_stats(const GemmArgs& p, const Args& a, const TileJob& t, int64_t row, int64_t first,
                                   f32x16 (&z)[CFG::TN], float& m, float& r) {
    int want = -1;  // the target's place in this lane's columns
    if (row < t.M) want = a.t.at(a.rows ? a.rows[row] : row);
    want = want < 0 ? -1 : want - (int)(a.first + first);
    m = -INFINITY;
#pragma unroll
    for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int c = j * 32 + 8 * (v >> 2) + (v & 3);
        if (FULL || first + c < p.N) {
          m = fmaxf(m, z[j][v]);
          if (want == c) a.target[row] = z[j][v];
        }
      }
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    float s = 0.f, f = 0.f;
    if (m > -INFINITY) {  // columns there are, and numbers in them
#pragma unroll
      for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int c = j * 32 + 8 * (v >> 2) + (v & 3);
          z[j][v] = ce_exp(z[j][v] - m);
          if (FULL || first + c < p.N) s += z[j][v], f += __builtin_amdgcn_fractf(z[j][v]);
        }
    } else {  // no columns, or NaN and -inf throughout: -inf is no part of the sum, a NaN shows
#pragma unroll
      for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int c = j * 32 + 8 * (v >> 2) + (v & 3);
          z[j][v] = z[j][v] == -INFINITY ? 0.f : z[j][v];
          if (FULL || first + c < p.N) s += z[j][v];
        }
    }
    s += __shfl_xor(s, 32, 64);
    f += __shfl_xor(f, 32, 64);
    r = f + (rintf(s - f) - 1.f);
  }
  __device__ static void store(const Args& a, const TileJob& t, int tid, const float2* red) {
    for (int r = tid; r < CFG::BM; r += CFG::NT) {
      if (t.m0 + r >= t.M) continue;
      float2 o = red[r];
#pragma unroll
      for (int w = 1; w < CFG::WN; ++w) ce_merge(o, red[w * CFG::BM + r]);
      a.part[(t.m0 + r) * a.n_tiles + (a.first + t.n0) / CFG::BN] = o;
    }
  }
};

// Backward epilogue: G[row, col] = g (e^{z - m} / s - [col = t]) in bf16, through a row-major LDS
// image so that its lines are written whole. Columns from N up to ldg's multiple of 8 are zeros.
template <class CFG>
struct EpiCEGrad {
  static constexpr int RSB = CFG::BN * 2 + 16;  // LDS bytes per image row
  static constexpr int LDS_BYTES = CFG::BM * RSB;
  struct Args {
    const float2* stats;
    const float* g;
    const int32_t* rows;
    CETargets t;
    int64_t first;  // the piece's first column of the vocabulary
    bf16_t* G;
    int64_t ldg;
  };
  template <class, typename>
  __device__ static void run(const GemmArgs& p, const Args& a, const TileJob& t, int wm, int wn, int tid,
                             f32x16 (&z)[CFG::TM][CFG::TN], char* smem) {
    if (t.n0 + CFG::BN <= p.N) run_t<true>(p, a, t, wm, wn, tid, z, smem);
    else run_t<false>(p, a, t, wm, wn, tid, z, smem);
  }
  template <bool FULL>
  __device__ static void run_t(const GemmArgs& p, const Args& a, const TileJob& t, int wm, int wn, int tid,
                               f32x16 (&z)[CFG::TM][CFG::TN], char* smem) {
    const int lane = tid & 63;
    lds_write_barrier();  // the k loop's stage buffers are free
#pragma unroll
    for (int i = 0; i < CFG::TM; ++i) {
      const int rl = wm * CFG::WTM + i * 32 + (lane & 31);
      const int64_t row = t.m0 + rl, r = a.rows[row < t.M ? row : t.m0];
      const float2 st = a.stats[r];
      const float gs = a.g[r] / (1.f + st.y);
      const int want = a.t.at(r) - (int)(a.first + t.n0) - (wn * CFG::WTN + 4 * (lane >> 5));
#pragma unroll
      for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = j * 32 + 8 * q;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = ce_exp(z[i][j][4 * q + e] - st.x);
            v[e] = (want == c + e ? (x - 1.f) - st.y : x) * gs;  // p - 1 from the others' sum: p may be near 1
            if (!FULL && t.n0 + wn * CFG::WTN + 4 * (lane >> 5) + c + e >= p.N) v[e] = 0.f;
          }
          *(uint2*)(smem + rl * RSB + (wn * CFG::WTN + c + 4 * (lane >> 5)) * 2) =
              make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        }
    }
    lds_write_barrier();
    constexpr int CPR = CFG::BN / 8, RPP = CFG::NT / CPR;
    static_assert(CFG::NT % CPR == 0 && CFG::BM % RPP == 0, "store passes");
    const int cc = tid % CPR;
    const int64_t col = t.n0 + cc * 8;
    for (int r = tid / CPR; r < CFG::BM; r += RPP)
      if (t.m0 + r < t.M && col < p.N)
        *(uint4*)(a.G + (t.m0 + r) * a.ldg + col) = *(const uint4*)(smem + r * RSB + cc * 16);
  }
};

// Epilogue of the one-call form: a row's maximum m and the others' sum over each wave's CE_SPAN columns, and
// 2^15 e^{z - m} in fp16: 11 bits down to 2^-29 of that maximum, 2^-39 at least. (One maximum for the
// tile would have all its accumulators wait for the others': 66 of them spilled.)
template <class CFG>
struct EpiCEKeep {
  static constexpr int RSB = CFG::BN * 2 + 16, IMAGE = CFG::BM * RSB;
  static constexpr int LDS_BYTES = IMAGE + CFG::WN * CFG::BM * 8;
  struct Args {
    typename EpiCEStats<CFG>::Args st;
    uint16_t* E;
    int64_t ld;
  };
  template <class, typename>
  __device__ static void run(const GemmArgs& p, const Args& a, const TileJob& t, int wm, int wn, int tid,
                             f32x16 (&z)[CFG::TM][CFG::TN], char* smem) {
    if (t.n0 + CFG::BN <= p.N) run_t<true>(p, a, t, wm, wn, tid, z, smem);
    else run_t<false>(p, a, t, wm, wn, tid, z, smem);
  }
  template <bool FULL>
  __device__ static void run_t(const GemmArgs& p, const Args& a, const TileJob& t, int wm, int wn, int tid,
                               f32x16 (&z)[CFG::TM][CFG::TN], char* smem) {
    const int lane = tid & 63;
    const int64_t first = t.n0 + wn * CFG::WTN + 4 * (lane >> 5);  // the lane's first column
    float2* red = (float2*)(smem + IMAGE);                         // [BM][WN]
    lds_write_barrier();  // the k loop's stage buffers are free
#pragma unroll
    for (int i = 0; i < CFG::TM; ++i) {
      const int rl = wm * CFG::WTM + i * 32 + (lane & 31);
      float m, r;
      EpiCEStats<CFG>::template row_stats<FULL>(p, a.st, t, t.m0 + rl, first, z[i], m, r);
      if (lane < 32) red[rl * CFG::WN + wn] = make_float2(m, r);
#pragma unroll
      for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = j * 32 + 8 * q;
          uint16_t v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = FULL || first + c + e < p.N ? __builtin_bit_cast(uint16_t, (_Float16)(z[i][j][4 * q + e] * 32768.f)) : 0;
          *(uint2*)(smem + rl * RSB + (wn * CFG::WTN + c + 4 * (lane >> 5)) * 2) =
              make_uint2(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16);
        }
    }
    lds_write_barrier();
    static_assert(CFG::WTN == CE_SPAN, "a wave's columns");
    const int64_t sub = t.n0 / CE_SPAN;
    for (int i = tid; i < CFG::BM * CFG::WN; i += CFG::NT) {
      const int r = i / CFG::WN, w = i % CFG::WN;
      if (t.m0 + r < t.M && sub + w < a.st.n_tiles) a.st.part[(t.m0 + r) * a.st.n_tiles + sub + w] = red[i];
    }
    constexpr int CPR = CFG::BN / 8, RPP = CFG::NT / CPR;
    const int cc = tid % CPR;
    const int64_t col = t.n0 + cc * 8;
    for (int r = tid / CPR; r < CFG::BM; r += RPP)
      if (t.m0 + r < t.M && col < p.N) *(uint4*)(a.E + (t.m0 + r) * a.ld + col) = *(const uint4*)(smem + r * RSB + cc * 16);
  }
};

// loss and statistics of the positions that count: one wave a row, the tiles' partials in a fixed order.
__global__ __launch_bounds__(256) void k_ce_merge(const float2* __restrict__ part, const float* __restrict__ target,
                                                  int64_t N, int64_t n_tiles, const int32_t* __restrict__ rows,
                                                  const int32_t* __restrict__ count, CETargets t,
                                                  float* __restrict__ loss, float2* __restrict__ stats,
                                                  float2* __restrict__ row_stats) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (count ? (int64_t)*count : N)) return;
  float2 o = make_float2(-INFINITY, -1.f);
  for (int64_t i = lane; i < n_tiles; i += 64) ce_merge(o, part[row * n_tiles + i]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) ce_merge(o, make_float2(__shfl_xor(o.x, off, 64), __shfl_xor(o.y, off, 64)));
  if (lane == 0) {
    const int64_t r = rows ? rows[row] : row;
    const bool on = t.at(r) >= 0;
    loss[r] = on ? (o.x - target[row]) + log1pf(o.y) : 0.f;
    if (stats) stats[r] = on ? o : make_float2(0.f, 0.f);
    if (row_stats) row_stats[row] = o;
  }
}

// counts[c] = how many of count rows are in chunk c of R.
__global__ void k_ce_counts(const int32_t* __restrict__ count, int64_t R, int chunks, int32_t* __restrict__ counts) {
  for (int c = threadIdx.x; c < chunks; c += 64) {
    const int64_t left = (int64_t)*count - c * R;
    counts[c] = (int32_t)(left < 0 ? 0 : (left < R ? left : R));
  }
}
// G = g (softmax - 1_t) in bf16 from what EpiCEKeep kept (E; G may be its memory): the values of each CE_SPAN
// columns times e^{their m - m} g / s. A position of weight zero gets zeros whatever it holds, and so
// does its row of the activations: d_head's product has 0 times it. Blocks: a row, 8192 columns of it.
__global__ __launch_bounds__(256) void k_ce_apply(const uint16_t* E, uint16_t* G, int64_t ld, int64_t cols, const float2* __restrict__ part,
                                                  int64_t n_tiles, const float2* __restrict__ st,
                                                  const float* __restrict__ target, const int32_t* __restrict__ rows,
                                                  const int32_t* __restrict__ count, CETargets t, const float* __restrict__ g,
                                                  uint4* __restrict__ act, int64_t words) {
  const int64_t row = blockIdx.x;
  if (row >= *count) return;
  const int64_t r = rows[row], want = t.at(r);
  const float2 o = st[row];
  const float gr = g[r], gs = gr / (1.f + o.y), by = gs * 0x1p-15f;
  const float hit = ((ce_exp(target[row] - o.x) - 1.f) - o.y) * gs;  // p - 1 from the others' sum: p may be near 1
  if (gr == 0.f && blockIdx.y == 0)
    for (int64_t c = threadIdx.x; c < words; c += 256) act[row * words + c] = make_uint4(0u, 0u, 0u, 0u);
  const uint16_t* e = E + row * ld;
  const int64_t c0 = (int64_t)blockIdx.y * 8192 + threadIdx.x * 8;
  uint4 w[4];
  float f[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t c = c0 + k * 2048;
    if (c >= cols) continue;
    w[k] = *(const uint4*)(e + c);
    f[k] = ce_exp(part[row * n_tiles + c / CE_SPAN].x - o.x) * by;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t c = c0 + k * 2048;
    if (c >= cols) continue;
    const uint32_t in[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
    uint32_t out[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float lo = (float)__builtin_bit_cast(_Float16, (uint16_t)in[q]) * f[k];
      float hi = (float)__builtin_bit_cast(_Float16, (uint16_t)(in[q] >> 16)) * f[k];
      if (c + 2 * q == want) lo = hit;
      if (c + 2 * q + 1 == want) hi = hit;
      out[q] = gr == 0.f ? 0u : pack_bf16x2(lo, hi);
    }
    *(uint4*)(G + row * ld + c) = make_uint4(out[0], out[1], out[2], out[3]);
  }
}
__global__ __launch_bounds__(256) void k_ce_round(const float4* __restrict__ src, int64_t n, uint2* __restrict__ dst) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const float4 v = src[i];
    dst[i] = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  }
}

// ---------------------------------------------------------------- fp32 as parts of bf16
// EpiCEGrad with G in fp32, straight from the registers.
template <class CFG>
struct EpiCEGradF {
  static constexpr int LDS_BYTES = 0;
  struct Args {
    const float2* stats;
    const float* g;
    const int32_t* rows;
    CETargets t;
    int64_t first;
    float* G;
    int64_t ldg;  // a multiple of 4
  };
  template <class, typename>
  __device__ static void run(const GemmArgs& p, const Args& a, const TileJob& t, int wm, int wn, int tid,
                             f32x16 (&z)[CFG::TM][CFG::TN], char*) {
    const int lane = tid & 63;
#pragma unroll
    for (int i = 0; i < CFG::TM; ++i) {
      const int64_t row = t.m0 + wm * CFG::WTM + i * 32 + (lane & 31);
      if (row >= t.M) continue;
      const int64_t r = a.rows[row];
      const float2 st = a.stats[r];
      const float gs = a.g[r] / (1.f + st.y);
      const int64_t first = t.n0 + wn * CFG::WTN + 4 * (lane >> 5);
      const int want = a.t.at(r) - (int)(a.first + first);
#pragma unroll
      for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = j * 32 + 8 * q;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = expf(z[i][j][4 * q + e] - st.x);
            v[e] = (want == c + e ? (x - 1.f) - st.y : x) * gs;
          }
          float* dst = a.G + row * a.ldg + first + c;
          if (first + c + 3 < p.N) {
            *(float4*)dst = make_float4(v[0], v[1], v[2], v[3]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (first + c + e < p.N) dst[e] = v[e];
          }
        }
    }
  }
};

// EpiCEStats that writes the logits too, in fp32.
template <class CFG>
struct EpiCEKeepF {
  static constexpr int LDS_BYTES = EpiCEStats<CFG>::LDS_BYTES;
  struct Args {
    typename EpiCEStats<CFG>::Args st;
    float* Z;
    int64_t ld;  // a multiple of 4
  };
  template <class TJ, typename TC>
  __device__ static void run(const GemmArgs& p, const Args& a, const TileJob& t, int wm, int wn, int tid,
                             f32x16 (&z)[CFG::TM][CFG::TN], char* smem) {
    const int lane = tid & 63;
    const int64_t first = t.n0 + wn * CFG::WTN + 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < CFG::TM; ++i) {
      const int64_t row = t.m0 + wm * CFG::WTM + i * 32 + (lane & 31);
      if (row >= t.M) continue;
#pragma unroll
      for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = j * 32 + 8 * q;
          float* dst = a.Z + row * a.ld + first + c;
          if (first + c + 3 < p.N) {
            *(float4*)dst = make_float4(z[i][j][4 * q], z[i][j][4 * q + 1], z[i][j][4 * q + 2], z[i][j][4 * q + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (first + c + e < p.N) dst[e] = z[i][j][4 * q + e];
          }
        }
    }
    EpiCEStats<CFG>::template run<TJ, TC>(p, a.st, t, wm, wn, tid, z, smem);
  }
};

// EpiCEGradF from the logits kept: G (which may be their memory) in fp32. Blocks: a row, 4096 columns of it.
__global__ __launch_bounds__(256) void k_ce_apply_f32(const float* Z, float* G, int64_t ld, int64_t V, const float2* __restrict__ st,
                                                      const int32_t* __restrict__ rows, const int32_t* __restrict__ count,
                                                      CETargets t, const float* __restrict__ g, float* __restrict__ act, int64_t d) {
  const int64_t row = blockIdx.x;
  if (row >= *count) return;
  const int64_t r = rows[row], want = t.at(r);
  const float2 o = st[row];
  const float gr = g[r], gs = gr / (1.f + o.y);
  if (gr == 0.f && blockIdx.y == 0)
    for (int64_t c = threadIdx.x; c < d; c += 256) act[row * d + c] = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t c = (int64_t)blockIdx.y * 4096 + k * 1024 + threadIdx.x * 4;
    if (c >= V) continue;
    float v[4];  // the row's pitch is a multiple of 4, what lies behind V is not read again
    const float4 z = *(const float4*)(Z + row * ld + c);
    v[0] = z.x, v[1] = z.y, v[2] = z.z, v[3] = z.w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = expf(v[e] - o.x);
      v[e] = gr == 0.f ? 0.f : (want == c + e ? (x - 1.f) - o.y : x) * gs;
    }
    *(float4*)(G + row * ld + c) = make_float4(v[0], v[1], v[2], v[3]);
  }
}

struct __attribute__((packed, aligned(4))) CEWord {  // at any element's boundary
  float v[4];
};
typedef float ce_f8 __attribute__((ext_vector_type(8)));
// 8 floats from p on; EDGE: those from `left` on are zeros (none is read).
template <bool EDGE>
__device__ inline ce_f8 ce_load8(const float* __restrict__ p, int64_t left) {
  ce_f8 v;
  if (!EDGE || left >= 8) {
    const CEWord a = *(const CEWord*)p, b = *(const CEWord*)(p + 4);
    v = ce_f8{a.v[0], a.v[1], a.v[2], a.v[3], b.v[0], b.v[1], b.v[2], b.v[3]};
  } else {
    v = (ce_f8)0.f;
    if (left > 0) v[0] = p[0];
    if (left > 1) v[1] = p[1];
    if (left > 2) v[2] = p[2];
    if (left > 3) v[3] = p[3];
    if (left > 4) v[4] = p[4];
    if (left > 5) v[5] = p[5];
    if (left > 6) v[6] = p[6];
  }
  return v;
}
// Word u of a thread's share of an operand's stage: 8 values of a tile of R rows from `first` on (below `end`) and
// 64 k from k0 on (below kend). K-major: row i / 8, chunk i % 8 of its k; MN-major: k-row i / (R / 8), chunk i % (R / 8).
template <bool MN, int R, int NT, bool EDGE>
__device__ inline ce_f8 ce_word(const float* __restrict__ base, int64_t ld, int64_t first, int64_t end, int64_t k0,
                                int64_t kend, int u, int tid) {
  const int i = tid + u * NT;
  const int64_t x = first + (MN ? i % (R / 8) * 8 : i / 8), k = k0 + (MN ? i / (R / 8) : i % 8 * 8);
  const int64_t left = EDGE && (x >= end || k >= kend) ? 0 : MN ? end - x : kend - k;
  return ce_load8<EDGE>(base + (EDGE && left <= 0 ? 0 : MN ? k * ld + x : x * ld + k), left);
}
template <bool MN, int R, int NT>
__device__ inline char* ce_place(char* region, int u, int tid) {
  const int i = tid + u * NT, row = MN ? i / (R / 8) : i / 8, c = MN ? i % (R / 8) : i % 8;
  return region + (MN ? row * 2 * R + ((c ^ (4 * (row & 3))) << 4) : row * 128 + ((c ^ dtl_swz(row)) << 4));
}
// The three parts of 8 values, to the same place of each plane.
__device__ inline void ce_parts8(char* at, int plane, ce_f8 v) {
  uint32_t p[3][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float a = v[2 * k], b = v[2 * k + 1];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      p[i][k] = pack_bf16x2(a, b);
      a -= __uint_as_float(p[i][k] << 16);
      b -= __uint_as_float(p[i][k] & 0xFFFF0000u);
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) *(uint4*)(at + i * plane) = make_uint4(p[i][0], p[i][1], p[i][2], p[i][3]);
}

// C = op(A) op(B) as k_gemm_dtl gives it (the same tiles, LDS layout and epilogues), of fp32 operands (p.A and p.B
// point to floats, lda and ldb count them) at any alignment. A stage of 64 k is loaded into registers while the
// one before is multiplied, and goes to LDS as three planes of parts. Bound by what lies between the stages' two barriers: forming
// and writing the parts (6 vector instructions a value) beside the fragments' reads.
template <class CFG, int MODE, class EPI, bool AMN, bool BMN>
__global__ __launch_bounds__(CFG::NT) void k_gemm_parts(GemmArgs p, typename EPI::Args ea) {
  constexpr int BM = CFG::BM, BN = CFG::BN, TM = CFG::TM, TN = CFG::TN, PLANE = CFG::STAGE_BYTES;
  constexpr int AW = BM * 8 / CFG::NT, BW = BN * 8 / CFG::NT;  // 8-value words of a thread
  static_assert(BM * 8 % CFG::NT == 0 && BN * 8 % CFG::NT == 0, "whole words");
  constexpr int LDS = 3 * PLANE > EPI::LDS_BYTES ? 3 * PLANE : EPI::LDS_BYTES;
  __shared__ __attribute__((aligned(1024))) char smem[LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int wm = wave / CFG::WN, wn = wave % CFG::WN;
  TileJob t;
  if (!map_tile<BM, BN, MODE, float>(p, lane, t)) return;
  const float *A = (const float*)p.A, *B = (const float*)p.B;
  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
  ce_f8 wa[AW], wb[BW];
  const bool whole = t.m0 + BM <= t.M && t.n0 + BN <= p.N;
  auto load = [&](int64_t k0) {
    if (whole && k0 + 64 <= t.kend) {
#pragma unroll
      for (int u = 0; u < AW; ++u) wa[u] = ce_word<AMN, BM, CFG::NT, false>(A, p.lda, t.m0, t.M, k0, t.kend, u, tid);
#pragma unroll
      for (int u = 0; u < BW; ++u) wb[u] = ce_word<BMN, BN, CFG::NT, false>(B, p.ldb, t.n0, p.N, k0, t.kend, u, tid);
    } else {
#pragma unroll
      for (int u = 0; u < AW; ++u) wa[u] = ce_word<AMN, BM, CFG::NT, true>(A, p.lda, t.m0, t.M, k0, t.kend, u, tid);
#pragma unroll
      for (int u = 0; u < BW; ++u) wb[u] = ce_word<BMN, BN, CFG::NT, true>(B, p.ldb, t.n0, p.N, k0, t.kend, u, tid);
    }
  };
  auto store = [&]() {
#pragma unroll
    for (int u = 0; u < AW; ++u) ce_parts8(ce_place<AMN, BM, CFG::NT>(smem, u, tid), PLANE, wa[u]);
#pragma unroll
    for (int u = 0; u < BW; ++u) ce_parts8(ce_place<BMN, BN, CFG::NT>(smem + BM * CFG::ROWB, u, tid), PLANE, wb[u]);
  };
  const FragOffs<CFG, AMN, BMN> fo(wm, wn, lane);
  if (t.kbeg < t.kend) load(t.kbeg);
  for (int64_t k0 = t.kbeg; k0 < t.kend; k0 += 64) {
    __syncthreads();  // the last stage's fragments have been read
    store();
    __syncthreads();
    if (k0 + 64 < t.kend) load(k0 + 64);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      Frags<CFG> f[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) read_frags<CFG>(smem + i * PLANE, fo, lane, kk, f[i]);
      // the small ones first
      dtl_mfma<CFG>(f[2].a, f[0].b, acc);
      dtl_mfma<CFG>(f[0].a, f[2].b, acc);
      dtl_mfma<CFG>(f[1].a, f[1].b, acc);
      dtl_mfma<CFG>(f[1].a, f[0].b, acc);
      dtl_mfma<CFG>(f[0].a, f[1].b, acc);
      dtl_mfma<CFG>(f[0].a, f[0].b, acc);
    }
  }
  EPI::template run<CFG, float>(p, ea, t, wm, wn, tid, acc, smem);
}

// ---------------------------------------------------------------- plans and launches
typedef CfgDtl CfgSmall;
typedef CfgDtlBig CfgBig;

// Rows of the head that one product takes: its operands end at 2 GiB (whole tiles, and the rows that a last stage of
// an operand stored along the other axis may reach).
int64_t ce_head_rows(int64_t d) { return (0x7FFFFFFF / (2 * d) - 128) & ~(int64_t)255; }

// Row pitch of G: whole 128-byte lines, an odd number of them (rows a power of two apart are in the same
// memory channels).
int64_t ce_pitch(int64_t cols) { return (tiles_up(cols, 64) | 1) * 64; }

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// Positions from which the forward leaves out those that do not count: one row of tiles saves nothing.
constexpr int64_t CE_COMPACT = 128;

struct CEFwdPlan {
  bool compact, big;
  int64_t n_tiles;
  int32_t *rows, *count;
  float* target;
  float2 *part;
  void* act;
  size_t total;
};
bool ce_big(int64_t N, int64_t V) { return big_rounds(tiles_up(N, 256) * tiles_up(V, 256), tiles_up(N, 128) * tiles_up(V, 128), SHARED_ROUND); }

CEFwdPlan ce_fwd_plan(int dtype, int64_t N, int64_t d, int64_t V, char* base) {
  CEFwdPlan P{};
  size_t off = 0;
  auto take = [&](size_t bytes) { char* p = base + off; off += up256(bytes); return p; };
  P.target = (float*)take((size_t)N * 4);
  P.big = dtype == PD_DTYPE_BF16 && ce_big(N, V);
  P.n_tiles = tiles_up(V, P.big ? 256 : 128);
  P.part = (float2*)take((size_t)N * P.n_tiles * 8);
  P.compact = N > CE_COMPACT;
  if (P.compact) {
    P.count = (int32_t*)take(4);
    P.rows = (int32_t*)take((size_t)N * 4);
    P.act = take((size_t)N * d * (dtype == PD_DTYPE_BF16 ? 2 : 4));
  }
  P.total = off;
  return P;
}

struct CEBwdPlan {
  bool big, big_act, big_head;
  int64_t cw, ld;  // columns of a piece, G's row pitch
  int splits;
  int64_t slice;
  int32_t *rows, *pos, *count;
  void* act;
  void* G;
  float* part;  // [splits][N][d]
  size_t total;
};
// Tiles and slices of the contraction of d_act = G head (N x d over cw columns a piece): its few tiles
// fill the chip only in slices, each of which leaves an fp32 slab to write and read. The rounds are
// those of all positions and, with a quarter of the weight, those where a part of them counts, which is not known here:
// as many as its tiles fill and half a round for the last. us of 1 / 4 / 5 / 8 slices of 256x256 tiles, the slabs' sum with
// them: 8192 x 768 over 50277 columns 1484 / 920 / 806 / 772, three fifths of it 1454 / 507 / 696 / 548 (8 are taken);
// 4096 x 4096 over 131072 3952 / 4048 / 4096 / 4196, three quarters of it 3818 / 3169 / 3301 / 3288 (4 are).
void ce_dact_form(int64_t N, int64_t d, int64_t cw, int64_t V, bool half, bool& big, int& splits) {
  double best = 1e30;
  for (int b = 0; b < (half ? 2 : 1); ++b)
    for (int sp = 1; sp <= 64 && (sp == 1 || cw / sp >= 1024); ++sp) {
      // 256x256 or two 128x128 a CU; fp32 one of 256x128 or 128x128
      const int64_t tm = half ? (b ? 256 : 128) : (N > 128 ? 256 : 128), tn = b ? 256 : 128, round = b || !half ? 256 : 512;
      const int64_t tiles = tiles_up(N, tm) * tiles_up(d, tn) * sp;
      const double rounds = 0.75 * (double)tiles_up(tiles, round) + 0.25 * std::max(1.0, (double)tiles / (double)round + 0.5);
      const double per_round = 2.0 * tm * tn * round * ((double)V / sp) / (b ? 1.2e15 : half ? 1.0e15 : 1.7e14);
      const double slabs = (double)sp * N * d * 4 * 2 * cdiv(V, cw) / 4e12;
      const double time = rounds * per_round + slabs;
      if (time < best) best = time, big = b, splits = sp;
    }
}

CEBwdPlan ce_bwd_plan(int dtype, int64_t N, int64_t d, int64_t V, bool dact, char* base) {
  CEBwdPlan P{};
  size_t off = 0;
  auto take = [&](size_t bytes) { char* p = base + off; off += up256(bytes); return p; };
  P.count = (int32_t*)take(4);
  P.rows = (int32_t*)take((size_t)N * 4);
  P.pos = (int32_t*)take((size_t)N * 4);
  const int64_t V8 = (V + 7) & ~(int64_t)7;
  const bool half = dtype == PD_DTYPE_BF16;
  const size_t esz = half ? 2 : 4;
  P.cw = std::min<int64_t>(V8, std::max<int64_t>(256, (int64_t)(CE_PIECE / ((size_t)N * esz)) & ~(int64_t)255));
  if (half) P.cw = std::min(P.cw, ce_head_rows(d));
  P.ld = ce_pitch(P.cw);
  P.act = take((size_t)N * d * esz);
  P.G = take((size_t)N * P.ld * esz);
  P.splits = 1;
  if (dact) ce_dact_form(N, d, P.cw, V, half, P.big_act, P.splits);
  P.slice = tiles_up(tiles_up(P.cw, P.splits), 64) * 64;
  P.big = half && ce_big(N, P.cw);
  P.big_head = half && big_tiles(P.cw, d, N);
  if (dact) P.part = (float*)take((size_t)P.splits * N * d * 4);
  P.total = off;
  return P;
}

// The form that keeps the softmax: what the gradients take from the loss (`kept`), and the memory of either.
struct CEOnePlan {
  int64_t R, ld, n_tiles;  // positions of a chunk, E's row, partials of a row
  int chunks, splits;
  bool big, big_act, big_head;
  int64_t slice;
  int32_t *rows, *pos, *count, *counts;
  bool half;
  void *act, *E, *G;  // E: bf16 the softmax in 16 bits, fp32 the logits
  float2 *part, *stats;
  float *target, *slabs, *head;
  size_t kept, work;
};
// A head that one product takes and a softmax whose shortest chunk is below CE_KEPT; else the
// two calls, one after the other.
bool ce_one_form(int dtype, int64_t d, int64_t V) {
  const bool half = dtype == PD_DTYPE_BF16;
  return (!half || V <= ce_head_rows(d)) && (size_t)(256 + 128) * ce_pitch(V) * (half ? 2 : 4) < CE_KEPT;
}
CEOnePlan ce_one_plan(int dtype, int64_t N, int64_t d, int64_t V, bool dact, bool dhead, bool apart, char* kept, char* work) {
  CEOnePlan P{};
  size_t off = 0;
  char* base = kept;
  auto take = [&](size_t bytes) { char* p = base + off; off += up256(bytes); return p; };
  P.half = dtype == PD_DTYPE_BF16;
  const size_t esz = P.half ? 2 : 4;
  P.ld = ce_pitch(V);
  P.R = std::min<int64_t>(N, std::max<int64_t>(256, (int64_t)(CE_KEPT / ((size_t)P.ld * esz)) - 128) & ~(int64_t)255);
  P.chunks = (int)cdiv(N, P.R);
  P.big = P.half && ce_big(P.R, V);
  P.n_tiles = tiles_up(V, P.half ? CE_SPAN : 128);
  P.big_head = P.half && big_tiles(V, d, P.R);
  P.count = (int32_t*)take(4);
  P.counts = (int32_t*)take((size_t)P.chunks * 4);
  P.rows = (int32_t*)take((size_t)N * 4);
  P.pos = (int32_t*)take((size_t)N * 4);
  P.E = take((size_t)P.R * P.ld * esz);
  P.part = (float2*)take((size_t)P.R * P.n_tiles * 8);
  P.stats = (float2*)take((size_t)P.R * 8);
  P.target = (float*)take((size_t)P.R * 4);
  P.kept = off;
  base = work, off = 0;
  P.act = take((size_t)N * d * esz);
  P.G = apart && (dact || dhead) ? take((size_t)P.R * P.ld * esz) : P.E;
  P.splits = 1;
  if (dact) {
    ce_dact_form(P.R, d, V, V, P.half, P.big_act, P.splits);
    P.slabs = (float*)take((size_t)P.splits * P.R * d * 4);
  }
  P.slice = tiles_up(tiles_up(V, P.splits), 64) * 64;
  if (P.half && dhead && P.chunks > 1) P.head = (float*)take((size_t)V * d * 4);
  P.work = off;
  return P;
}

template <class CFG, typename TC, int MODE, class EPI, bool AMN, bool BMN>
void ce_launch(const GemmArgs& a, const typename EPI::Args& ea, int slices, bool edge, hipStream_t s) {
  const dim3 grid((unsigned)tiles_up(a.N, CFG::BN), (unsigned)tiles_up(a.M, CFG::BM), (unsigned)slices);
  if (edge) hipLaunchKernelGGL((k_gemm_dtl<CFG, TC, MODE, true, EPI, AMN, BMN>), grid, dim3(CFG::NT), 0, s, a, ea);
  else hipLaunchKernelGGL((k_gemm_dtl<CFG, TC, MODE, false, EPI, AMN, BMN>), grid, dim3(CFG::NT), 0, s, a, ea);
}

// 256 x 128 tiles from the second row of 128 x 128 ones on: 12 fragments read for 24 MFMAs of a wave in place of 9
// for 12. 1003 x 1000 over 32003: the four products 512, 459, 452, 416 -> 392, 393, 375, 367 us, 170 TFLOP/s of the
// product itself (fp32 MFMAs end at 157).
typedef DtlCfg<256, 128, 4, 2, false> CfgParts;
template <class CFG, int MODE, class EPI, bool AMN, bool BMN>
void ce_launch_parts(const GemmArgs& a, const typename EPI::Args& ea, int slices, hipStream_t s) {
  const dim3 grid((unsigned)tiles_up(a.N, CFG::BN), (unsigned)tiles_up(a.M, CFG::BM), (unsigned)slices);
  hipLaunchKernelGGL((k_gemm_parts<CFG, MODE, EPI, AMN, BMN>), grid, dim3(CFG::NT), 0, s, a, ea);
}
template <int MODE, template <class> class EPI, bool AMN, bool BMN, class... Args>
void ce_launch_f32(const GemmArgs& a, int slices, hipStream_t s, Args... args) {
  if (a.M > 128) ce_launch_parts<CfgParts, MODE, EPI<CfgParts>, AMN, BMN>(a, {args...}, slices, s);
  else ce_launch_parts<CfgSmall, MODE, EPI<CfgSmall>, AMN, BMN>(a, {args...}, slices, s);
}
template <class>
using EpiCEStore = EpiStore;

int ce_check(const char* what, int dtype, int64_t N, int64_t d, int64_t V, const void* act, const void* head,
             const void* targets, int bits) {
  if (dtype != PD_DTYPE_F32 && dtype != PD_DTYPE_BF16)
    return fail(PD_EUNSUPPORTED, std::string(what) + ": dtype must be fp32 or bf16");
  if (N < 0 || d <= 0 || V <= 0) return fail(PD_EINVAL, std::string(what) + ": N >= 0, d >= 1 and V >= 1");
  if (bits != 32 && bits != 64) return fail(PD_EINVAL, std::string(what) + ": targets are int32 or int64");
  if (N && (!act || !head || !targets)) return fail(PD_EINVAL, std::string(what) + ": null pointer");
  if (dtype == PD_DTYPE_BF16) {
    if (d % 8) return fail(PD_EUNSUPPORTED, std::string(what) + ": bf16 needs d to be a multiple of 8");
    if (N && (((uintptr_t)act | (uintptr_t)head) & 15)) return fail(PD_EINVAL, std::string(what) + ": 16-byte aligned tensors");
    if (!dtl_fits_mn(N, d) || d > 1 << 20)
      return fail(PD_EUNSUPPORTED, std::string(what) + ": activations of 2 GiB or more");
  }
  if (tiles_up(N, 128) > 65535 || tiles_up(V, 128) > 65535 || N > (int64_t)1 << 21)
    return fail(PD_EUNSUPPORTED, std::string(what) + ": too large");
  return PD_OK;
}

// The logits of chunk c: softmax kept, loss and statistics.
void ce_one_loss(const CEOnePlan& P, int c, int64_t N, int64_t d, int64_t V, const void* head, const CETargets& t,
                 float* loss, hipStream_t s) {
  const int64_t R = P.R, M = std::min(R, N - c * R);
  const int32_t *rows = P.rows + c * R, *count = P.counts + c;
  const bool edge = d % 64 != 0;
  const bf16_t* a_c = (const bf16_t*)((const char*)P.act + c * R * d * (P.half ? 2 : 4));
  const GemmArgs a{M, V, d, a_c, d, (const bf16_t*)head, d, nullptr, 0, 1.f, 0.f, count, 0, 0, 0, cdiv(d, 64) * 64,
                   nullptr, nullptr, nullptr};
  if (!P.half) {
    if (M > 128) ce_launch_parts<CfgParts, MODE_COUNTED, EpiCEKeepF<CfgParts>, false, false>(a, {{P.part, P.n_tiles, P.target, rows, t}, (float*)P.E, P.ld}, 1, s);
    else ce_launch_parts<CfgSmall, MODE_COUNTED, EpiCEKeepF<CfgSmall>, false, false>(a, {{P.part, P.n_tiles, P.target, rows, t}, (float*)P.E, P.ld}, 1, s);
  } else if (P.big) {
    ce_launch<CfgBig, float, MODE_COUNTED, EpiCEKeep<CfgBig>, false, false>(
        a, {{P.part, P.n_tiles, P.target, rows, t}, (uint16_t*)P.E, P.ld}, 1, edge, s);
  } else {
    ce_launch<CfgSmall, float, MODE_COUNTED, EpiCEKeep<CfgSmall>, false, false>(
        a, {{P.part, P.n_tiles, P.target, rows, t}, (uint16_t*)P.E, P.ld}, 1, edge, s);
  }
  hipLaunchKernelGGL(k_ce_merge, dim3((unsigned)cdiv(M, 4)), dim3(256), 0, s, P.part, P.target, M, P.n_tiles, rows, count, t,
                     loss, nullptr, P.stats);
}
// Its gradients.
void ce_one_grads(const CEOnePlan& P, int c, int64_t N, int64_t d, int64_t V, const void* head, const CETargets& t,
                  const float* g, void* d_act, void* d_head, hipStream_t s) {
  const int64_t R = P.R, M = std::min(R, N - c * R);
  const int32_t *rows = P.rows + c * R, *count = P.counts + c;
  char* a_c = (char*)P.act + c * R * d * (P.half ? 2 : 4);
  if (P.half)
    hipLaunchKernelGGL(k_ce_apply, dim3((unsigned)M, (unsigned)cdiv(V, 8192)), dim3(256), 0, s, (const uint16_t*)P.E,
                       (uint16_t*)P.G, P.ld, (V + 7) & ~(int64_t)7, P.part, P.n_tiles, P.stats, P.target, rows, count, t, g,
                       (uint4*)a_c, d / 8);
  else
    hipLaunchKernelGGL(k_ce_apply_f32, dim3((unsigned)M, (unsigned)cdiv(V, 4096)), dim3(256), 0, s, (const float*)P.E,
                       (float*)P.G, P.ld, V, P.stats, rows, count, t, g, (float*)a_c, d);
  const bf16_t* G = (const bf16_t*)P.G;  // k_gemm_parts takes its operands so
  if (d_act) {
    const GemmArgs b{M, d, V, G, P.ld, (const bf16_t*)head, d, P.slabs, d, 1.f, 0.f, count, 0, 0, R * d, P.slice, nullptr, nullptr, nullptr};
    const dim3 grid((unsigned)std::min<int64_t>(cdiv(P.half ? N * d / 4 : N * d, 256), 8192));
    if (!P.half) {
      ce_launch_f32<MODE_COUNTED, EpiCEStore, false, true>(b, P.splits, s);
      hipLaunchKernelGGL(k_ce_scatter<float>, grid, dim3(256), 0, s, P.slabs, P.splits, R * d, N, d, P.pos, c * R, R, (float*)d_act);
    } else {
      if (P.big_act) ce_launch<CfgBig, float, MODE_COUNTED, EpiStore, false, true>(b, {}, P.splits, V % 64 != 0, s);
      else ce_launch<CfgSmall, float, MODE_COUNTED, EpiStore, false, true>(b, {}, P.splits, V % 64 != 0, s);
      hipLaunchKernelGGL(k_ce_scatter<bf16_t>, grid, dim3(256), 0, s, P.slabs, P.splits, R * d, N, d, P.pos, c * R, R, (bf16_t*)d_act);
    }
  }
  if (d_head) {
    const bool sum = P.half && P.chunks > 1;  // bf16 chunks are added in fp32
    const GemmArgs b{V, d, M, G, P.ld, (const bf16_t*)a_c, d, sum ? (void*)P.head : d_head, d, 1.f, c ? 1.f : 0.f, count, 0, 0, 0, 0,
                     nullptr, nullptr, nullptr};
    if (!P.half) {
      ce_launch_f32<MODE_COUNTED_K, EpiCEStore, true, true>(b, 1, s);
    } else if (sum) {
      if (P.big_head) ce_launch<CfgBig, float, MODE_COUNTED_K, EpiStore, true, true>(b, {}, 1, true, s);
      else ce_launch<CfgSmall, float, MODE_COUNTED_K, EpiStore, true, true>(b, {}, 1, true, s);
    } else {
      if (P.big_head) ce_launch<CfgBig, bf16_t, MODE_COUNTED_K, EpiStore, true, true>(b, {}, 1, true, s);
      else ce_launch<CfgSmall, bf16_t, MODE_COUNTED_K, EpiStore, true, true>(b, {}, 1, true, s);
    }
  }
}

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" {

size_t pd_streamed_ce_fwd_workspace_size(int dtype, int64_t N, int64_t d, int64_t V) {
  if (N <= 0 || d <= 0 || V <= 0) return 0;
  return ce_fwd_plan(dtype, N, d, V, nullptr).total;
}

int pd_streamed_ce_fwd(int dtype, int64_t N, int64_t d, int64_t V, const void* act, const void* head,
                       const void* targets, int target_bits, int64_t ignore_index, float* loss, float* stats,
                       void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "pd_streamed_ce_fwd";
  if (int rc = ce_check(what, dtype, N, d, V, act, head, targets, target_bits)) return rc;
  if (!N) return PD_OK;
  if (!loss) return fail(PD_EINVAL, std::string(what) + ": loss required");
  const CEFwdPlan P = ce_fwd_plan(dtype, N, d, V, (char*)workspace);
  if (!workspace || workspace_bytes < P.total) return fail(PD_EWORKSPACE, std::string(what) + ": workspace");
  hipStream_t s = (hipStream_t)stream;
  const CETargets t{targets, target_bits, ignore_index, V};
  const bool half = dtype == PD_DTYPE_BF16;
  GemmArgs a{N, V, d, (const bf16_t*)act, d, (const bf16_t*)head, d, nullptr, 0, 1.f, 0.f, nullptr, 0, 0, 0, cdiv(d, 64) * 64,
             nullptr, nullptr, nullptr};
  if (P.compact) {
    hipLaunchKernelGGL(k_ce_compact, dim3(1), dim3(1024), 0, s, t, nullptr, N, P.rows, nullptr, P.count, loss, (float2*)stats);
    ce_gather(half, act, N, d, P.rows, P.count, P.act, s);
    a.A = (const bf16_t*)P.act;
    a.offsets = P.count;
  }
  if (!half) ce_launch_f32<MODE_COUNTED, EpiCEStats, false, false>(a, 1, s, P.part, P.n_tiles, P.target, (const int32_t*)P.rows, t);
  for (int64_t c = 0, most = ce_head_rows(d); half && c < V; c += most) {
    a.N = std::min(most, V - c);
    a.B = (const bf16_t*)head + c * d;
    if (P.big)
      ce_launch<CfgBig, float, MODE_COUNTED, EpiCEStats<CfgBig>, false, false>(a, {P.part, P.n_tiles, P.target, P.rows, t, c}, 1,
                                                                               d % 64 != 0, s);
    else
      ce_launch<CfgSmall, float, MODE_COUNTED, EpiCEStats<CfgSmall>, false, false>(
          a, {P.part, P.n_tiles, P.target, P.rows, t, c}, 1, d % 64 != 0, s);
  }
  hipLaunchKernelGGL(k_ce_merge, dim3((unsigned)cdiv(N, 4)), dim3(256), 0, s, P.part, P.target, N, P.n_tiles, P.rows, P.count, t,
                     loss, (float2*)stats, nullptr);
  return check_launch(what);
}

size_t pd_streamed_ce_bwd_workspace_size(int dtype, int64_t N, int64_t d, int64_t V, int want_dact) {
  if (N <= 0 || d <= 0 || V <= 0) return 0;
  return ce_bwd_plan(dtype, N, d, V, want_dact, nullptr).total;
}

int pd_streamed_ce_bwd(int dtype, int64_t N, int64_t d, int64_t V, const void* act, const void* head,
                       const void* targets, int target_bits, int64_t ignore_index, const float* stats, const float* g,
                       void* d_act, void* d_head, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "pd_streamed_ce_bwd";
  if (int rc = ce_check(what, dtype, N, d, V, act, head, targets, target_bits)) return rc;
  if (!d_act && !d_head) return PD_OK;
  if (!N) return fail(PD_EINVAL, std::string(what) + ": no positions");
  if (!stats || !g) return fail(PD_EINVAL, std::string(what) + ": stats and g required");
  const CEBwdPlan P = ce_bwd_plan(dtype, N, d, V, d_act != nullptr, (char*)workspace);
  if (!workspace || workspace_bytes < P.total) return fail(PD_EWORKSPACE, std::string(what) + ": workspace");
  hipStream_t s = (hipStream_t)stream;
  const CETargets t{targets, target_bits, ignore_index, V};
  hipLaunchKernelGGL(k_ce_compact, dim3(1), dim3(1024), 0, s, t, g, N, P.rows, P.pos, P.count, nullptr, nullptr);
  if (dtype == PD_DTYPE_BF16) {
    bf16_t *act_c = (bf16_t*)P.act, *G = (bf16_t*)P.G;
    ce_gather(true, act, N, d, P.rows, P.count, act_c, s);
    for (int64_t c = 0; c < V; c += P.cw) {
      const int64_t w = std::min(P.cw, V - c);
      const bf16_t* h = (const bf16_t*)head + c * d;
      GemmArgs a{N, w, d, act_c, d, h, d, nullptr, 0, 1.f, 0.f, P.count, 0, 0, 0, cdiv(d, 64) * 64, nullptr, nullptr, nullptr};
      if (P.big)
        ce_launch<CfgBig, float, MODE_COUNTED, EpiCEGrad<CfgBig>, false, false>(
            a, {(const float2*)stats, g, P.rows, t, c, G, P.ld}, 1, d % 64 != 0, s);
      else
        ce_launch<CfgSmall, float, MODE_COUNTED, EpiCEGrad<CfgSmall>, false, false>(
            a, {(const float2*)stats, g, P.rows, t, c, G, P.ld}, 1, d % 64 != 0, s);
      if (d_act) {  // slabs [splits][N][d] += G [count, w] head [w, d], a slice of w each
        GemmArgs b{N, d, w, G, P.ld, h, d, P.part, d, 1.f, c ? 1.f : 0.f, P.count, 0, 0, N * d, P.slice, nullptr, nullptr, nullptr};
        if (P.big_act) ce_launch<CfgBig, float, MODE_COUNTED, EpiStore, false, true>(b, {}, P.splits, w % 64 != 0, s);
        else ce_launch<CfgSmall, float, MODE_COUNTED, EpiStore, false, true>(b, {}, P.splits, w % 64 != 0, s);
      }
      if (d_head) {  // [w, d] = G^T act over the positions that count
        GemmArgs b{w, d, N, G, P.ld, act_c, d, (bf16_t*)d_head + c * d, d, 1.f, 0.f, P.count, 0, 0, 0, 0, nullptr, nullptr, nullptr};
        if (P.big_head) ce_launch<CfgBig, bf16_t, MODE_COUNTED_K, EpiStore, true, true>(b, {}, 1, true, s);
        else ce_launch<CfgSmall, bf16_t, MODE_COUNTED_K, EpiStore, true, true>(b, {}, 1, true, s);
      }
    }
    if (d_act)
      hipLaunchKernelGGL(k_ce_scatter<bf16_t>, dim3((unsigned)std::min<int64_t>(cdiv(N * d / 4, 256), 8192)), dim3(256), 0, s,
                         P.part, P.splits, N * d, N, d, P.pos, (int64_t)0, N, (bf16_t*)d_act);
    return check_launch(what);
  }
  float *act_c = (float*)P.act, *G = (float*)P.G;
  ce_gather(false, act, N, d, P.rows, P.count, act_c, s);
  auto as = [](const float* p) { return (const bf16_t*)p; };  // as k_gemm_parts takes its operands
  for (int64_t c = 0; c < V; c += P.cw) {
    const int64_t w = std::min(P.cw, V - c);
    const float* h = (const float*)head + c * d;
    const GemmArgs a{N, w, d, as(act_c), d, as(h), d, nullptr, 0, 1.f, 0.f, P.count, 0, 0, 0, cdiv(d, 64) * 64, nullptr, nullptr, nullptr};
    ce_launch_f32<MODE_COUNTED, EpiCEGradF, false, false>(a, 1, s, (const float2*)stats, g, (const int32_t*)P.rows, t, c, G, P.ld);
    if (d_act) {
      const GemmArgs b{N, d, w, as(G), P.ld, as(h), d, P.part, d, 1.f, c ? 1.f : 0.f, P.count, 0, 0, N * d, P.slice, nullptr, nullptr, nullptr};
      ce_launch_f32<MODE_COUNTED, EpiCEStore, false, true>(b, P.splits, s);
    }
    if (d_head) {
      const GemmArgs b{w, d, N, as(G), P.ld, as(act_c), d, (float*)d_head + c * d, d, 1.f, 0.f, P.count, 0, 0, 0, 0, nullptr, nullptr, nullptr};
      ce_launch_f32<MODE_COUNTED_K, EpiCEStore, true, true>(b, 1, s);
    }
  }
  if (d_act)
    hipLaunchKernelGGL(k_ce_scatter<float>, dim3((unsigned)std::min<int64_t>(cdiv(N * d, 256), 8192)), dim3(256), 0, s, P.part,
                       P.splits, N * d, N, d, P.pos, (int64_t)0, N, (float*)d_act);
  return check_launch(what);
}

size_t pd_streamed_ce_train_workspace_size(int dtype, int64_t N, int64_t d, int64_t V, int want_dact, int want_dhead) {
  if (N <= 0 || d <= 0 || V <= 0) return 0;
  if (ce_one_form(dtype, d, V)) {
    const CEOnePlan P = ce_one_plan(dtype, N, d, V, want_dact, want_dhead, false, nullptr, nullptr);
    return P.kept + P.work;
  }
  return up256((size_t)N * 8) + std::max(ce_fwd_plan(dtype, N, d, V, nullptr).total,
                                         ce_bwd_plan(dtype, N, d, V, want_dact, nullptr).total);
}

int pd_streamed_ce_train(int dtype, int64_t N, int64_t d, int64_t V, const void* act, const void* head,
                         const void* targets, int target_bits, int64_t ignore_index, const float* g, float* loss,
                         void* d_act, void* d_head, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "pd_streamed_ce_train";
  if (int rc = ce_check(what, dtype, N, d, V, act, head, targets, target_bits)) return rc;
  if (!N || !g || !loss || (!d_act && !d_head)) return fail(PD_EINVAL, std::string(what) + ": positions, g, loss and a gradient required");
  const size_t need = pd_streamed_ce_train_workspace_size(dtype, N, d, V, d_act != nullptr, d_head != nullptr);
  if (!workspace || workspace_bytes < need) return fail(PD_EWORKSPACE, std::string(what) + ": workspace");
  hipStream_t s = (hipStream_t)stream;
  if (!ce_one_form(dtype, d, V)) {
    float* stats = (float*)workspace;
    char* ws = (char*)workspace + up256((size_t)N * 8);
    const size_t left = workspace_bytes - up256((size_t)N * 8);
    if (int rc = pd_streamed_ce_fwd(dtype, N, d, V, act, head, targets, target_bits, ignore_index, loss, stats, ws, left, stream))
      return rc;
    return pd_streamed_ce_bwd(dtype, N, d, V, act, head, targets, target_bits, ignore_index, stats, g, d_act, d_head, ws, left,
                              stream);
  }
  const size_t kept = ce_one_plan(dtype, N, d, V, false, false, false, nullptr, nullptr).kept;
  const CEOnePlan P = ce_one_plan(dtype, N, d, V, d_act != nullptr, d_head != nullptr, false, (char*)workspace, (char*)workspace + kept);
  if (P.half && !dtl_fits_mn(P.R, P.ld)) return fail(PD_EUNSUPPORTED, std::string(what) + ": too large");
  const CETargets t{targets, target_bits, ignore_index, V};
  hipLaunchKernelGGL(k_ce_compact, dim3(1), dim3(1024), 0, s, t, nullptr, N, P.rows, P.pos, P.count, loss, nullptr);
  ce_gather(P.half, act, N, d, P.rows, P.count, P.act, s);
  hipLaunchKernelGGL(k_ce_counts, dim3(1), dim3(64), 0, s, P.count, P.R, P.chunks, P.counts);
  for (int c = 0; c < P.chunks; ++c) {
    ce_one_loss(P, c, N, d, V, head, t, loss, s);
    ce_one_grads(P, c, N, d, V, head, t, g, d_act, d_head, s);
  }
  if (P.half && d_head && P.chunks > 1)
    hipLaunchKernelGGL(k_ce_round, dim3((unsigned)std::min<int64_t>(cdiv(V * d / 4, 256), 16384)), dim3(256), 0, s,
                       (const float4*)P.head, V * d / 4, (uint2*)d_head);
  return check_launch(what);
}

size_t pd_streamed_ce_kept_size(int dtype, int64_t N, int64_t d, int64_t V) {
  if (N <= 0 || d <= 0 || V <= 0 || !ce_one_form(dtype, d, V)) return 0;
  const CEOnePlan P = ce_one_plan(dtype, N, d, V, false, false, true, nullptr, nullptr);
  return P.chunks == 1 && (!P.half || dtl_fits_mn(P.R, P.ld)) ? P.kept : 0;
}

size_t pd_streamed_ce_kept_workspace_size(int dtype, int64_t N, int64_t d, int64_t V, int want_dact, int want_dhead) {
  if (!pd_streamed_ce_kept_size(dtype, N, d, V)) return 0;
  return ce_one_plan(dtype, N, d, V, want_dact, want_dhead, true, nullptr, nullptr).work;
}

int pd_streamed_ce_kept_fwd(int dtype, int64_t N, int64_t d, int64_t V, const void* act, const void* head,
                            const void* targets, int target_bits, int64_t ignore_index, float* loss, void* kept,
                            size_t kept_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "pd_streamed_ce_kept_fwd";
  if (int rc = ce_check(what, dtype, N, d, V, act, head, targets, target_bits)) return rc;
  if (!N || !loss) return fail(PD_EINVAL, std::string(what) + ": positions and loss required");
  const size_t need = pd_streamed_ce_kept_size(dtype, N, d, V);
  if (!need) return fail(PD_EUNSUPPORTED, std::string(what) + ": nothing is kept at this size");
  const CEOnePlan P = ce_one_plan(dtype, N, d, V, false, false, true, (char*)kept, (char*)workspace);
  if (!kept || kept_bytes < need || !workspace || workspace_bytes < P.work)
    return fail(PD_EWORKSPACE, std::string(what) + ": workspace");
  hipStream_t s = (hipStream_t)stream;
  const CETargets t{targets, target_bits, ignore_index, V};
  hipLaunchKernelGGL(k_ce_compact, dim3(1), dim3(1024), 0, s, t, nullptr, N, P.rows, P.pos, P.count, loss, nullptr);
  ce_gather(P.half, act, N, d, P.rows, P.count, P.act, s);
  hipLaunchKernelGGL(k_ce_counts, dim3(1), dim3(64), 0, s, P.count, P.R, P.chunks, P.counts);
  ce_one_loss(P, 0, N, d, V, head, t, loss, s);
  return check_launch(what);
}

int pd_streamed_ce_kept_bwd(int dtype, int64_t N, int64_t d, int64_t V, const void* act, const void* head,
                            const void* targets, int target_bits, int64_t ignore_index, const void* kept,
                            size_t kept_bytes, const float* g, void* d_act, void* d_head, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const char* what = "pd_streamed_ce_kept_bwd";
  if (int rc = ce_check(what, dtype, N, d, V, act, head, targets, target_bits)) return rc;
  if (!d_act && !d_head) return PD_OK;
  if (!N || !g) return fail(PD_EINVAL, std::string(what) + ": positions and g required");
  const size_t need = pd_streamed_ce_kept_size(dtype, N, d, V);
  if (!need) return fail(PD_EUNSUPPORTED, std::string(what) + ": nothing is kept at this size");
  const CEOnePlan P = ce_one_plan(dtype, N, d, V, d_act != nullptr, d_head != nullptr, true, (char*)const_cast<void*>(kept),
                                  (char*)workspace);
  if (!kept || kept_bytes < need || !workspace || workspace_bytes < P.work)
    return fail(PD_EWORKSPACE, std::string(what) + ": workspace");
  hipStream_t s = (hipStream_t)stream;
  const CETargets t{targets, target_bits, ignore_index, V};
  ce_gather(P.half, act, N, d, P.rows, P.count, P.act, s);
  ce_one_grads(P, 0, N, d, V, head, t, g, d_act, d_head, s);
  return check_launch(what);
}

}  // extern "C"
