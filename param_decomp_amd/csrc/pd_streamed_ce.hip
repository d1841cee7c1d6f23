// Softmax cross entropy over a vocabulary whose logits are never kept, and its gradients.
//
//   z = act head^T, loss_i = log(sum_v e^{z_iv}) - z_i,t_i
//   G = g (softmax(z) - 1_t), d_act = G head, d_head = G^T act
//
// Bound by the matrix cores: 2 N d V operations forward, and backward 2 N d V to form the logits
// again and 2 N d V for each gradient. bf16: the forward's product keeps each tile's maximum and
// sum for every row and the target's logit, and a second kernel merges tiles in a fixed order; the
// logits stay in registers. The backward goes over the vocabulary in pieces of which G (bf16) fits
// CE_PIECE bytes of workspace: one product whose epilogue writes G, then both gradients from it.
// The softmax is formed from the row's maximum and sum, kept apart: the log of the sum alone would
// round a probability near one to 1e-6.
//
// Positions whose target lies outside the vocabulary do not count (nor, backward, those of weight
// zero): their rows are left out of a dense copy of the activations, so they cost no products and
// what they hold reaches nothing. How many count only the device knows: grids cover all positions
// and the products read the count (MODE_COUNTED).
//
// fp32 runs pieces of logits through pd_gemm and passes over them.
#include <algorithm>
#include <cmath>

#include "pd_gemm_dtl.hpp"

namespace pd {
namespace {

constexpr size_t CE_PIECE = (size_t)512 << 20;
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
// -1. With `loss` those that do not get loss 0 and statistics (0, 1). One block.
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
        stats[i] = make_float2(0.f, 1.f);
      }
    }
  }
  if (threadIdx.x == 0) *count = base;
}

// dst[r] = src[rows[r]] for r < count (words of 16 bytes, n a row); ZERO: zeros for the rest.
template <bool ZERO>
__global__ __launch_bounds__(256) void k_ce_gather(const uint4* __restrict__ src, int64_t N, int64_t n,
                                                   const int32_t* __restrict__ rows, const int32_t* __restrict__ count,
                                                   uint4* __restrict__ dst) {
  const int64_t held = *count, total = (ZERO ? N : held) * n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / n;
    dst[i] = r < held ? src[(int64_t)rows[r] * n + i % n] : make_uint4(0u, 0u, 0u, 0u);
  }
}
__global__ __launch_bounds__(256) void k_ce_gather_f32(const float* __restrict__ src, int64_t N, int64_t d,
                                                       const int32_t* __restrict__ rows,
                                                       const int32_t* __restrict__ count, float* __restrict__ dst) {
  const int64_t held = *count;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < N * d; i += (int64_t)gridDim.x * 256)
    dst[i] = i / d < held ? src[(int64_t)rows[i / d] * d + i % d] : 0.f;
}

// d_act[i] = the sum over `slabs` of the row of position i, zeros where it does not count.
template <typename T>
__global__ __launch_bounds__(256) void k_ce_scatter(const float* __restrict__ part, int slabs, int64_t stride,
                                                    int64_t N, int64_t d, const int32_t* __restrict__ pos,
                                                    T* __restrict__ d_act) {
  const int64_t q = d / 4;  // bf16: d is a multiple of 8
  const bool vec = d % 4 == 0;
  const int64_t total = vec ? N * q : N * d;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = vec ? i / q : i / d, at = pos[r];
    if (vec) {
      const int64_t c = i % q * 4;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at >= 0)
        for (int k = 0; k < slabs; ++k) {
          const float4 v = *(const float4*)(part + k * stride + at * d + c);
          s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
      if constexpr (sizeof(T) == 2) *(uint2*)(d_act + r * d + c) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
      else *(float4*)(d_act + r * d + c) = s;
    } else {
      const int64_t c = i % d;
      float s = 0.f;
      if (at >= 0)
        for (int k = 0; k < slabs; ++k) s += part[k * stride + at * d + c];
      store_f<T>(d_act, r * d + c, s);
    }
  }
}

__device__ inline float ce_exp(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// (maximum, sum relative to it) of two sets of columns; (-inf, 0) is none.
__device__ inline void ce_merge(float2& o, float2 q) {
  const float m = fmaxf(o.x, q.x);
  o.y = o.y * (o.x == m ? 1.f : expf(o.x - m)) + q.y * (q.x == m ? 1.f : expf(q.x - m));
  o.x = m;
}

// Forward epilogue: each row's maximum and sum over the tile's columns, to part[row][tile], and
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
    const int lane = tid & 63, rl = lane & 31;
    float2* red = (float2*)smem;  // [WN][BM]
    lds_write_barrier();          // the k loop's stage buffers are free
#pragma unroll
    for (int i = 0; i < CFG::TM; ++i) {
      const int64_t row = t.m0 + wm * CFG::WTM + i * 32 + rl;
      int want = -1;  // the target's place in this lane's columns
      if (row < t.M) want = a.t.at(a.rows ? a.rows[row] : row);
      if (want >= 0) want -= (int)t.n0 + wn * CFG::WTN + 4 * (lane >> 5);
      float m = -INFINITY, s = 0.f;
#pragma unroll
      for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int c = j * 32 + 8 * (v >> 2) + (v & 3);
          const float x = z[i][j][v];
          if (FULL || t.n0 + wn * CFG::WTN + 4 * (lane >> 5) + c < p.N) {
            m = fmaxf(m, x);
            if (want == c) a.target[row] = x;
          }
        }
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      if (m > -INFINITY) {  // columns there are, and numbers in them
#pragma unroll
        for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int c = j * 32 + 8 * (v >> 2) + (v & 3);
            if (FULL || t.n0 + wn * CFG::WTN + 4 * (lane >> 5) + c < p.N) s += ce_exp(z[i][j][v] - m);
          }
      } else if (t.n0 + wn * CFG::WTN < p.N) {
        s = NAN;  // NaN or -inf throughout: no softmax
      }
      s += __shfl_xor(s, 32, 64);
      if (lane < 32) red[wn * CFG::BM + wm * CFG::WTM + i * 32 + rl] = make_float2(m, s);
    }
    lds_write_barrier();
    for (int r = tid; r < CFG::BM; r += CFG::NT) {
      if (t.m0 + r >= t.M) continue;
      float2 o = red[r];
#pragma unroll
      for (int w = 1; w < CFG::WN; ++w) ce_merge(o, red[w * CFG::BM + r]);
      a.part[(t.m0 + r) * a.n_tiles + t.n0 / CFG::BN] = o;
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
      const float g = a.g[r], gs = g / st.y;
      const int want = a.t.at(r) - (int)(a.first + t.n0) - (wn * CFG::WTN + 4 * (lane >> 5));
#pragma unroll
      for (int j = 0; j < CFG::TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = j * 32 + 8 * q;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = ce_exp(z[i][j][4 * q + e] - st.x) * gs;
            if (want == c + e) v[e] -= g;
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

// loss and statistics of the positions that count: one wave a row, the tiles' partials in a fixed order.
__global__ __launch_bounds__(256) void k_ce_merge(const float2* __restrict__ part, const float* __restrict__ target,
                                                  int64_t N, int64_t n_tiles, const int32_t* __restrict__ rows,
                                                  const int32_t* __restrict__ count, CETargets t,
                                                  float* __restrict__ loss, float2* __restrict__ stats) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (count ? (int64_t)*count : N)) return;
  float2 o = make_float2(-INFINITY, 0.f);
  for (int64_t i = lane; i < n_tiles; i += 64) ce_merge(o, part[row * n_tiles + i]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) ce_merge(o, make_float2(__shfl_xor(o.x, off, 64), __shfl_xor(o.y, off, 64)));
  if (lane == 0) {
    const int64_t r = rows ? rows[row] : row;
    const bool on = t.at(r) >= 0;
    loss[r] = on ? (o.x - target[row]) + logf(o.y) : 0.f;
    if (stats) stats[r] = on ? o : make_float2(0.f, 1.f);
  }
}

// ---------------------------------------------------------------- fp32: pieces of logits in memory
// Row r's maximum and sum over the piece's w columns, added to those of the pieces before.
__global__ __launch_bounds__(256) void k_ce_piece_stats(const float* __restrict__ z, int64_t w, int64_t ld,
                                                        int64_t first, CETargets t, float2* __restrict__ run,
                                                        float* __restrict__ target) {
  __shared__ float red[4];
  __shared__ float2 both[4];
  const int64_t r = blockIdx.x;
  const float* row = z + r * ld;
  float m = -INFINITY, s = 0.f;
  for (int64_t v = threadIdx.x; v < w; v += 256) m = fmaxf(m, row[v]);
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  for (int64_t v = threadIdx.x; v < w; v += 256) s += m > -INFINITY ? expf(row[v] - m) : NAN;
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) both[threadIdx.x >> 6] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x) return;
  float2 o = make_float2(m, (both[0].y + both[1].y) + (both[2].y + both[3].y));
  if (first) {
    float2 old = run[r];
    ce_merge(old, o);
    o = old;
  }
  run[r] = o;
  const int64_t want = (int64_t)t.at(r) - first;
  if (want >= 0 && want < w) target[r] = row[want];
}
// z -> G in place for the rows that count, zeros for the others.
__global__ __launch_bounds__(256) void k_ce_piece_grad(float* __restrict__ z, int64_t w, int64_t ld, int64_t first,
                                                       CETargets t, const float2* __restrict__ stats,
                                                       const float* __restrict__ g, const int32_t* __restrict__ rows,
                                                       const int32_t* __restrict__ count) {
  const int64_t r = blockIdx.x;
  float* row = z + r * ld;
  const bool on = r < *count;
  const int64_t i = on ? rows[r] : 0;
  const float2 st = on ? stats[i] : make_float2(0.f, 1.f);
  const float gi = on ? g[i] : 0.f, gs = gi / st.y;
  const int64_t want = (int64_t)t.at(i) - first;
  for (int64_t v = threadIdx.x; v < w; v += 256) {
    float x = on ? expf(row[v] - st.x) * gs : 0.f;
    if (v == want) x -= gi;
    row[v] = x;
  }
}

// ---------------------------------------------------------------- plans and launches
typedef CfgDtl CfgSmall;
typedef CfgDtlBig CfgBig;

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// Positions from which the forward leaves out those that do not count: one row of tiles saves nothing.
constexpr int64_t CE_COMPACT = 128;

struct CEFwdPlan {
  bool compact, big;
  int64_t n_tiles, cw;
  int32_t *rows, *count;
  float* target;
  float2 *part;
  bf16_t* act;
  float* z;
  size_t total;
};
bool ce_big(int64_t N, int64_t V) { return big_rounds(tiles_up(N, 256) * tiles_up(V, 256), tiles_up(N, 128) * tiles_up(V, 128), SHARED_ROUND); }

CEFwdPlan ce_fwd_plan(int dtype, int64_t N, int64_t d, int64_t V, char* base) {
  CEFwdPlan P{};
  size_t off = 0;
  auto take = [&](size_t bytes) { char* p = base + off; off += up256(bytes); return p; };
  P.target = (float*)take((size_t)N * 4);
  if (dtype == PD_DTYPE_BF16) {
    P.compact = N > CE_COMPACT;
    P.big = ce_big(N, V);
    P.n_tiles = tiles_up(V, P.big ? 256 : 128);
    P.part = (float2*)take((size_t)N * P.n_tiles * 8);
    if (P.compact) {
      P.count = (int32_t*)take(4);
      P.rows = (int32_t*)take((size_t)N * 4);
      P.act = (bf16_t*)take((size_t)N * d * 2);
    }
  } else {
    P.cw = std::min<int64_t>(V, std::max<int64_t>(64, (int64_t)(CE_PIECE / ((size_t)N * 4)) & ~(int64_t)63));
    P.part = (float2*)take((size_t)N * 8);
    P.z = (float*)take((size_t)N * P.cw * 4);
  }
  P.total = off;
  return P;
}

struct CEBwdPlan {
  bool big, big_act, big_head;
  int64_t cw;  // columns of a piece
  int splits;
  int64_t slice;
  int32_t *rows, *pos, *count;
  void* act;
  void* G;
  float* part;  // [splits][N][d]
  size_t total;
};
CEBwdPlan ce_bwd_plan(int dtype, int64_t N, int64_t d, int64_t V, bool dact, char* base) {
  CEBwdPlan P{};
  size_t off = 0;
  auto take = [&](size_t bytes) { char* p = base + off; off += up256(bytes); return p; };
  const size_t esz = dtype == PD_DTYPE_BF16 ? 2 : 4;
  P.cw = std::min<int64_t>((V + 7) & ~(int64_t)7, std::max<int64_t>(256, (int64_t)(CE_PIECE / ((size_t)N * esz)) & ~(int64_t)255));
  P.big = ce_big(N, P.cw);
  P.big_act = big_tiles(N, d, P.cw);
  P.big_head = big_tiles(P.cw, d, N);
  P.count = (int32_t*)take(4);
  P.rows = (int32_t*)take((size_t)N * 4);
  P.pos = (int32_t*)take((size_t)N * 4);
  P.act = take((size_t)N * d * esz);
  P.G = take((size_t)N * P.cw * esz);
  P.splits = 1;
  if (dact) {
    if (dtype == PD_DTYPE_BF16) {
      // the fewest slices of the contraction (each at least 1024 deep) that fill whole rounds to 90%
      const int64_t t = P.big_act ? 256 : 128, round = P.big_act ? 256 : 512;
      const int64_t tiles = tiles_up(N, t) * tiles_up(d, t);
      double best = 0.0;
      for (int sp = 1; sp <= 8 && (sp == 1 || P.cw / sp >= 1024); ++sp) {
        const double eff = (double)(tiles * sp) / (double)(tiles_up(tiles * sp, round) * round);
        if (eff > best + 1e-9) best = eff, P.splits = sp;
        if (eff >= 0.9) break;
      }
    }
    P.part = (float*)take((size_t)P.splits * N * d * 4);
  }
  P.slice = tiles_up(tiles_up(P.cw, P.splits), 64) * 64;
  P.total = off;
  return P;
}

template <class CFG, typename TC, int MODE, class EPI, bool AMN, bool BMN>
void ce_launch(const GemmArgs& a, const typename EPI::Args& ea, int slices, bool edge, hipStream_t s) {
  const dim3 grid((unsigned)tiles_up(a.N, CFG::BN), (unsigned)tiles_up(a.M, CFG::BM), (unsigned)slices);
  if (edge) hipLaunchKernelGGL((k_gemm_dtl<CFG, TC, MODE, true, EPI, AMN, BMN>), grid, dim3(CFG::NT), 0, s, a, ea);
  else hipLaunchKernelGGL((k_gemm_dtl<CFG, TC, MODE, false, EPI, AMN, BMN>), grid, dim3(CFG::NT), 0, s, a, ea);
}

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
    if (!dtl_fits(N, d, V, d) || !dtl_fits_mn(V, d) || !dtl_fits_mn(N, d))
      return fail(PD_EUNSUPPORTED, std::string(what) + ": operands of 2 GiB or more");
  }
  if (tiles_up(N, 128) > 65535 || tiles_up(V, 128) > 65535 || N > (int64_t)1 << 21)
    return fail(PD_EUNSUPPORTED, std::string(what) + ": too large");
  return PD_OK;
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
  if (dtype == PD_DTYPE_BF16) {
    GemmArgs a{N, V, d, (const bf16_t*)act, d, (const bf16_t*)head, d, nullptr, 0, 1.f, 0.f, nullptr, 0, 0, 0, d,
               nullptr, nullptr, nullptr};
    a.strideA = cdiv(d, 64) * 64;  // one slice
    if (P.compact) {
      hipLaunchKernelGGL(k_ce_compact, dim3(1), dim3(1024), 0, s, t, nullptr, N, P.rows, nullptr, P.count, loss,
                         (float2*)stats);
      hipLaunchKernelGGL(k_ce_gather<false>, dim3((unsigned)std::min<int64_t>(cdiv(N * d / 8, 256), 4096)), dim3(256), 0, s,
                         (const uint4*)act, N, d / 8, P.rows, P.count, (uint4*)P.act);
      a.A = P.act;
      a.offsets = P.count;
    }
    if (P.big)
      ce_launch<CfgBig, float, MODE_COUNTED, EpiCEStats<CfgBig>, false, false>(a, {P.part, P.n_tiles, P.target, P.rows, t}, 1,
                                                                               d % 64 != 0, s);
    else
      ce_launch<CfgSmall, float, MODE_COUNTED, EpiCEStats<CfgSmall>, false, false>(a, {P.part, P.n_tiles, P.target, P.rows, t},
                                                                                   1, d % 64 != 0, s);
    hipLaunchKernelGGL(k_ce_merge, dim3((unsigned)cdiv(N, 4)), dim3(256), 0, s, P.part, P.target, N, P.n_tiles, P.rows,
                       P.count, t, loss, (float2*)stats);
    return check_launch(what);
  }
  for (int64_t c = 0; c < V; c += P.cw) {
    const int64_t w = std::min(P.cw, V - c);
    if (int rc = pd_gemm(PD_DTYPE_F32, N, w, d, act, d, 0, (const float*)head + c * d, d, 1, P.z, P.cw, PD_DTYPE_F32, 1.f,
                         0.f, stream))
      return rc;
    hipLaunchKernelGGL(k_ce_piece_stats, dim3((unsigned)N), dim3(256), 0, s, P.z, w, P.cw, c, t, P.part, P.target);
  }
  hipLaunchKernelGGL(k_ce_merge, dim3((unsigned)cdiv(N, 4)), dim3(256), 0, s, P.part, P.target, N, (int64_t)1, nullptr,
                     nullptr, t, loss, (float2*)stats);
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
    hipLaunchKernelGGL(k_ce_gather<false>, dim3((unsigned)std::min<int64_t>(cdiv(N * d / 8, 256), 4096)), dim3(256), 0, s,
                       (const uint4*)act, N, d / 8, P.rows, P.count, (uint4*)act_c);
    for (int64_t c = 0; c < V; c += P.cw) {
      const int64_t w = std::min(P.cw, V - c);
      const bf16_t* h = (const bf16_t*)head + c * d;
      GemmArgs a{N, w, d, act_c, d, h, d, nullptr, 0, 1.f, 0.f, P.count, 0, 0, 0, cdiv(d, 64) * 64, nullptr, nullptr, nullptr};
      if (P.big)
        ce_launch<CfgBig, float, MODE_COUNTED, EpiCEGrad<CfgBig>, false, false>(
            a, {(const float2*)stats, g, P.rows, t, c, G, P.cw}, 1, d % 64 != 0, s);
      else
        ce_launch<CfgSmall, float, MODE_COUNTED, EpiCEGrad<CfgSmall>, false, false>(
            a, {(const float2*)stats, g, P.rows, t, c, G, P.cw}, 1, d % 64 != 0, s);
      if (d_act) {  // slabs [splits][N][d] += G [count, w] head [w, d], a slice of w each
        GemmArgs b{N, d, w, G, P.cw, h, d, P.part, d, 1.f, c ? 1.f : 0.f, P.count, 0, 0, N * d, P.slice, nullptr, nullptr, nullptr};
        if (P.big_act) ce_launch<CfgBig, float, MODE_COUNTED, EpiStore, false, true>(b, {}, P.splits, w % 64 != 0, s);
        else ce_launch<CfgSmall, float, MODE_COUNTED, EpiStore, false, true>(b, {}, P.splits, w % 64 != 0, s);
      }
      if (d_head) {  // [w, d] = G^T act over the positions that count
        GemmArgs b{w, d, N, G, P.cw, act_c, d, (bf16_t*)d_head + c * d, d, 1.f, 0.f, P.count, 0, 0, 0, 0, nullptr, nullptr, nullptr};
        if (P.big_head) ce_launch<CfgBig, bf16_t, MODE_COUNTED_K, EpiStore, true, true>(b, {}, 1, true, s);
        else ce_launch<CfgSmall, bf16_t, MODE_COUNTED_K, EpiStore, true, true>(b, {}, 1, true, s);
      }
    }
    if (d_act)
      hipLaunchKernelGGL(k_ce_scatter<bf16_t>, dim3((unsigned)std::min<int64_t>(cdiv(N * d / 4, 256), 8192)), dim3(256), 0, s,
                         P.part, P.splits, N * d, N, d, P.pos, (bf16_t*)d_act);
    return check_launch(what);
  }
  float *act_c = (float*)P.act, *G = (float*)P.G;
  hipLaunchKernelGGL(k_ce_gather_f32, dim3((unsigned)std::min<int64_t>(cdiv(N * d, 256), 4096)), dim3(256), 0, s,
                     (const float*)act, N, d, P.rows, P.count, act_c);
  for (int64_t c = 0; c < V; c += P.cw) {
    const int64_t w = std::min(P.cw, V - c);
    const float* h = (const float*)head + c * d;
    int rc = pd_gemm(PD_DTYPE_F32, N, w, d, act_c, d, 0, h, d, 1, G, P.cw, PD_DTYPE_F32, 1.f, 0.f, stream);
    if (rc) return rc;
    hipLaunchKernelGGL(k_ce_piece_grad, dim3((unsigned)N), dim3(256), 0, s, G, w, P.cw, c, t, (const float2*)stats, g, P.rows,
                       P.count);
    if (d_act && (rc = pd_gemm(PD_DTYPE_F32, N, d, w, G, P.cw, 0, h, d, 0, P.part, d, PD_DTYPE_F32, 1.f, c ? 1.f : 0.f, stream)))
      return rc;
    if (d_head && (rc = pd_gemm(PD_DTYPE_F32, w, d, N, G, P.cw, 1, act_c, d, 0, (float*)d_head + c * d, d, PD_DTYPE_F32, 1.f,
                                0.f, stream)))
      return rc;
  }
  if (d_act)
    hipLaunchKernelGGL(k_ce_scatter<float>, dim3((unsigned)std::min<int64_t>(cdiv(N * d, 256), 8192)), dim3(256), 0, s, P.part,
                       1, N * d, N, d, P.pos, (float*)d_act);
  return check_launch(what);
}

}  // extern "C"
