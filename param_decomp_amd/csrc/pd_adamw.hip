// AdamW over many tensors in one pass, with states in 32 bits or in 8.
//
//   m' = m + (1 - beta1) (g - m),  v' = v + (1 - beta2) (g^2 - v),  t = step + 1
//   p' = p - lr (decay p + m' / (1 - beta1^t) / (sqrt(v' / (1 - beta2^t)) + eps))
//
// Memory bound: a value takes 28 bytes with fp32 states (p, m and v read and written, g read),
// 14 with 8-bit states and bf16 gradients, 2 more for a bf16 copy of p'. One launch covers up to
// ADAMW_TENSORS tensors, whose pointers travel in the kernel's arguments: nothing is copied to
// the device beforehand and a captured graph holds them. The step count lives in device memory
// and is advanced by the last block of the last launch, so a replayed graph goes on counting.
//
// 8-bit states: m and r = sqrt(v) as e4m3 codes with one fp32 scale (largest magnitude / 448) for
// 256 values, which one wave holds, four a lane. v changes by a thousandth of itself a step, far
// below half a code, so codes are rounded up with the probability of the fraction (16 random bits
// each: the two halves of a Threefry word of the value's index and the step). A root that is not
// zero keeps the smallest code rather than zero, where the step m / (r + eps) would grow past
// measure. The update itself uses m' and v' before rounding.
//
// Measured: 1.51 10^8 values in 48 tensors, fp32 states and copies, 890 us (5.1 TB/s); 2.64 10^8 in 24, 8-bit states,
// bf16 gradients and copies, 885-905 us (4.7-4.8 TB/s); a large copy moves 4.84.
#include <algorithm>
#include <cmath>

#include "pd_common.hpp"

namespace pd {
namespace {

constexpr int ADAMW_TENSORS = 48;  // in one launch: 3.9 KB of its 4 KB of arguments
constexpr int64_t ADAMW_BLOCKS = (1 << 24) - 1;  // of a launch: 2^32 threads less one
constexpr int QB = 256;            // values that share a scale
constexpr float FP8_TOP = 448.f;

struct AdamWTensor {
  float* p;
  const void* g;
  void* m;
  void* v;
  float* m_scale;  // NULL: fp32 states
  float* v_scale;
  bf16_t* copy;
  int64_t n;
  int64_t base;  // of its values' indices in the random draw (a multiple of QB)
  int32_t first;  // block of the launch
  int32_t g_bf16;
};
struct AdamWArgs {
  AdamWTensor t[ADAMW_TENSORS];
  int32_t* step;
  uint32_t* ticket;  // NULL: not the last launch
  const float* lr_dev;
  const float* grad_scale;
  double log_b1, log_b2;
  float lr, a1, a2, eps, decay;  // a = 1 - beta
  uint32_t k0, k1;
  int32_t n_tensors, chunk;
};
static_assert(sizeof(AdamWArgs) <= 4096, "kernel arguments");

struct AdamWRates {
  float a1, a2, size, root, eps, decay, gs;  // size = lr / c1, root = 1 / sqrt(c2), decay = lr times it
  uint32_t k0, k1;
};

// Words at any element's boundary (the hardware takes them as one access).
struct __attribute__((packed, aligned(4))) F4 {
  float v[4];
};
struct __attribute__((packed, aligned(2))) H4 {
  uint16_t v[4];
};
struct __attribute__((packed, aligned(1))) B4 {
  uint8_t v[4];
};

// Four values of a lane: p, g, and the states as they are kept.
template <bool Q8>
struct AdamWFour {
  float p[4], g[4];
  float m[4], v[4];  // fp32 states
  uint32_t mq, vq;   // codes, lowest first
  float ms, vs;
};

template <bool Q8, bool GB, bool FULL>
__device__ inline AdamWFour<Q8> adamw_load(const AdamWTensor& t, int64_t i, int64_t block) {
  AdamWFour<Q8> w;
  const int left = FULL ? 4 : (int)(t.n - i < 0 ? 0 : (t.n - i < 4 ? t.n - i : 4));
  if (FULL) {
    const F4 p = *(const F4*)(t.p + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) w.p[e] = p.v[e];
    if constexpr (GB) {
      const H4 g = *(const H4*)((const uint16_t*)t.g + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) w.g[e] = bf16_to_f32(g.v[e]);
    } else {
      const F4 g = *(const F4*)((const float*)t.g + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) w.g[e] = g.v[e];
    }
    if constexpr (Q8) {
      w.mq = __builtin_bit_cast(uint32_t, *(const B4*)((const uint8_t*)t.m + i));
      w.vq = __builtin_bit_cast(uint32_t, *(const B4*)((const uint8_t*)t.v + i));
    } else {
      const F4 m = *(const F4*)((const float*)t.m + i), v = *(const F4*)((const float*)t.v + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) w.m[e] = m.v[e], w.v[e] = v.v[e];
    }
  } else {
    w.mq = w.vq = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = e < left;
      w.p[e] = in ? t.p[i + e] : 0.f;
      w.g[e] = !in ? 0.f : GB ? bf16_to_f32(((const bf16_t*)t.g)[i + e]) : ((const float*)t.g)[i + e];
      if constexpr (Q8) {
        if (in) w.mq |= (uint32_t)((const uint8_t*)t.m)[i + e] << (8 * e);
        if (in) w.vq |= (uint32_t)((const uint8_t*)t.v)[i + e] << (8 * e);
      } else {
        w.m[e] = in ? ((const float*)t.m)[i + e] : 0.f;
        w.v[e] = in ? ((const float*)t.v)[i + e] : 0.f;
      }
    }
  }
  if constexpr (Q8) w.ms = t.m_scale[block], w.vs = t.v_scale[block];
  return w;
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// Values rounded to fp32 before they are used (not inside an fma): the state is what it stands for.
__device__ inline void fp8_decode(uint32_t w, float scale, float (&x)[4]) {
#pragma clang fp contract(off)
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0] * scale, x[1] = lo[1] * scale, x[2] = hi[0] * scale, x[3] = hi[1] * scale;
}

__device__ inline bool finite_f(float x) { return fabsf(x) < INFINITY; }

// x's magnitude times `inv` as an e4m3 value, rounded up with the probability of its fraction
// (`r`: 16 random bits); FLOOR: not to zero. A value that is not finite becomes NaN.
template <bool FLOOR>
__device__ inline float fp8_round(float x, float inv, uint32_t r) {
  const float a = fminf(fabsf(x) * inv, FP8_TOP);
  const float normal = __uint_as_float((__float_as_uint(a) + (r << 4)) & 0xFFF00000u);
  const float small = floorf(fmaf(a, 512.f, (float)r * 0x1p-16f)) * 0x1p-9f;
  float q = a >= 0x1p-6f ? normal : small;
  if (FLOOR) q = a > 0.f ? fmaxf(q, 0x1p-9f) : q;
  return finite_f(x) ? copysignf(q, x) : NAN;
}

__device__ inline uint32_t fp8_pack(const float (&q)[4]) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}

// g^2 - v with both roundings: what rounds to a code is then the same in plain arithmetic.
__device__ inline float square_less(float g, float v) {
#pragma clang fp contract(off)
  const float s = g * g;
  return s - v;
}

template <bool Q8, bool FULL>
__device__ inline void adamw_finish(const AdamWTensor& t, const AdamWRates& h, int64_t i, int64_t block,
                                    AdamWFour<Q8>& w) {
  float m[4], v[4], root[4], p[4];
  if constexpr (Q8) {
    fp8_decode(w.mq, w.ms, m);
    fp8_decode(w.vq, w.vs, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = w.m[e], v[e] = w.v[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float g = w.g[e] * h.gs;
    m[e] = fmaf(h.a1, g - m[e], m[e]);
    v[e] = fmaf(h.a2, square_less(g, v[e]), v[e]);
    root[e] = sqrtf(v[e]);  // the hardware's own reads subnormal numbers as zero, and the step would be m / eps
    // taken off with the update: 1 - lr decay would round what lies below 2^-24 away
    p[e] = w.p[e] - fmaf(h.decay, w.p[e], m[e] * h.size * __builtin_amdgcn_rcpf(fmaf(root[e], h.root, h.eps)));
  }
  const int left = FULL ? 4 : (int)(t.n - i < 0 ? 0 : (t.n - i < 4 ? t.n - i : 4));
  if (FULL) {
    *(F4*)(t.p + i) = F4{p[0], p[1], p[2], p[3]};
    if (t.copy) {
      const uint32_t lo = pack_bf16x2(p[0], p[1]), hi = pack_bf16x2(p[2], p[3]);
      *(H4*)(t.copy + i) = H4{(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) {
        t.p[i + e] = p[e];
        if (t.copy) t.copy[i + e] = f32_to_bf16(p[e]);
      }
  }
  if constexpr (Q8) {
    float mt = 0.f, vt = 0.f;  // largest finite magnitudes of the wave's 256 values
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mt = fmaxf(mt, finite_f(m[e]) ? fabsf(m[e]) : 0.f);
      vt = fmaxf(vt, finite_f(root[e]) ? root[e] : 0.f);
    }
    mt = wave_max(mt);
    vt = wave_max(vt);
    const float mi = 1.f / fmaxf(mt, 0x1p-100f) * FP8_TOP, vi = 1.f / fmaxf(vt, 0x1p-100f) * FP8_TOP;
    const uint64_t pair = (uint64_t)(t.base + i) >> 1;
    uint32_t r[4];
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      r[e] = (uint32_t)((pair + e / 2) >> 32), r[e + 1] = (uint32_t)(pair + e / 2);
      threefry2x32(h.k0, h.k1, r[e], r[e + 1]);
    }
    float mq[4], vq[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mq[e] = fp8_round<false>(m[e], mi, r[e] & 0xFFFFu);
      vq[e] = fp8_round<true>(root[e], vi, r[e] >> 16);
    }
    const uint32_t mw = fp8_pack(mq), vw = fp8_pack(vq);
    if (FULL) {
      *(B4*)((uint8_t*)t.m + i) = __builtin_bit_cast(B4, mw);
      *(B4*)((uint8_t*)t.v + i) = __builtin_bit_cast(B4, vw);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) ((uint8_t*)t.m)[i + e] = (uint8_t)(mw >> (8 * e)), ((uint8_t*)t.v)[i + e] = (uint8_t)(vw >> (8 * e));
    }
    if ((threadIdx.x & 63) == 0) {
      t.m_scale[block] = mt * (1.f / FP8_TOP);
      t.v_scale[block] = vt * (1.f / FP8_TOP);
    }
  } else if (FULL) {
    *(F4*)((float*)t.m + i) = F4{m[0], m[1], m[2], m[3]};
    *(F4*)((float*)t.v + i) = F4{v[0], v[1], v[2], v[3]};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) ((float*)t.m)[i + e] = m[e], ((float*)t.v)[i + e] = v[e];
  }
}

// Values [lo, hi) of a tensor (lo a multiple of 4 QB), a wave's 256 at a time, two such blocks'
// loads in flight.
template <bool Q8, bool GB>
__device__ inline void adamw_span(const AdamWTensor& t, const AdamWRates& h, int64_t lo, int64_t hi) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int64_t b = lo + wave * QB; b < hi; b += 8 * QB) {
    const int64_t c = b + 4 * QB;
    if (c < hi && c + QB <= t.n) {
      AdamWFour<Q8> x = adamw_load<Q8, GB, true>(t, b + 4 * lane, b / QB);
      AdamWFour<Q8> y = adamw_load<Q8, GB, true>(t, c + 4 * lane, c / QB);
      adamw_finish<Q8, true>(t, h, b + 4 * lane, b / QB, x);
      adamw_finish<Q8, true>(t, h, c + 4 * lane, c / QB, y);
    } else {
      for (int64_t a = b; a <= c && a < hi; a += 4 * QB) {
        if (a + QB <= t.n) {
          AdamWFour<Q8> x = adamw_load<Q8, GB, true>(t, a + 4 * lane, a / QB);
          adamw_finish<Q8, true>(t, h, a + 4 * lane, a / QB, x);
        } else {
          AdamWFour<Q8> x = adamw_load<Q8, GB, false>(t, a + 4 * lane, a / QB);
          adamw_finish<Q8, false>(t, h, a + 4 * lane, a / QB, x);
        }
      }
    }
  }
}

__global__ __launch_bounds__(256) void k_adamw(AdamWArgs a) {
  const int lane = threadIdx.x & 63;
  // the tensor whose blocks hold this one
  const int first = lane < a.n_tensors ? a.t[lane].first : 0x7FFFFFFF;
  const int at = __builtin_amdgcn_readfirstlane(__popcll(__ballot(first <= (int)blockIdx.x)) - 1);
  const AdamWTensor t = a.t[at];
  const int32_t step = *a.step + 1;
  AdamWRates h;
  h.a1 = a.a1, h.a2 = a.a2, h.eps = a.eps;
  const float lr = a.lr_dev ? *a.lr_dev : a.lr;
  h.gs = a.grad_scale ? *a.grad_scale : 1.f;
  h.size = lr / -expm1f((float)((double)step * a.log_b1));
  h.root = 1.f / sqrtf(-expm1f((float)((double)step * a.log_b2)));
  h.decay = lr * a.decay;
  h.k0 = 0u, h.k1 = (uint32_t)step;
  threefry2x32(a.k0, a.k1, h.k0, h.k1);
  const int64_t lo = (int64_t)((int)blockIdx.x - t.first) * a.chunk;
  const int64_t hi = lo + a.chunk < t.n ? lo + a.chunk : t.n;
  if (t.m_scale) {
    if (t.g_bf16) adamw_span<true, true>(t, h, lo, hi);
    else adamw_span<true, false>(t, h, lo, hi);
  } else {
    if (t.g_bf16) adamw_span<false, true>(t, h, lo, hi);
    else adamw_span<false, false>(t, h, lo, hi);
  }
  if (!a.ticket) return;
  __syncthreads();  // every wave has read the step
  if (threadIdx.x == 0 && atomicAdd(a.ticket, 1u) == gridDim.x - 1) {
    *a.ticket = 0u;
    *a.step = step;
  }
}

__global__ void k_adamw_count(int32_t* step) { *step += 1; }

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" int pd_adamw_step(int n_tensors, const int64_t* sizes, void* const* p, const void* const* grads,
                             const int32_t* grad_dtypes, void* const* m, void* const* v, void* const* m_scale,
                             void* const* v_scale, void* const* copies, int32_t* step, uint32_t* ticket, double lr,
                             const float* lr_dev, const float* grad_scale, double beta1, double beta2, double eps,
                             double weight_decay, uint32_t k0, uint32_t k1, void* stream) {
  const char* what = "pd_adamw_step";
  if (n_tensors < 0 || (n_tensors && (!sizes || !p || !grads || !grad_dtypes || !m || !v)) || !step || !ticket)
    return fail(PD_EINVAL, std::string(what) + ": null argument");
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0))
    return fail(PD_EINVAL, std::string(what) + ": betas must be in [0, 1)");
  // below the smallest normal number its reciprocal is infinite, and a value without gradient would become NaN
  if (!std::isfinite((float)eps) || !((float)eps >= 0x1p-126f))
    return fail(PD_EINVAL, std::string(what) + ": eps must be at least 2^-126 and finite");
  if (!std::isfinite(lr) || !std::isfinite(weight_decay))
    return fail(PD_EINVAL, std::string(what) + ": lr and weight_decay must be finite");
  int64_t total = 0, base = 0;
  for (int i = 0; i < n_tensors; ++i) {
    if (sizes[i] < 0 || sizes[i] > (int64_t)1 << 37) return fail(PD_EINVAL, std::string(what) + ": size of a tensor");
    if (!sizes[i] || !grads[i]) continue;
    const void *ms = m_scale ? m_scale[i] : nullptr, *vs = v_scale ? v_scale[i] : nullptr;
    if (!p[i] || !m[i] || !v[i] || !ms != !vs) return fail(PD_EINVAL, std::string(what) + ": null pointer");
    if (grad_dtypes[i] != PD_DTYPE_F32 && grad_dtypes[i] != PD_DTYPE_BF16)
      return fail(PD_EUNSUPPORTED, std::string(what) + ": gradients are fp32 or bf16");
    total += sizes[i];
  }
  // Blocks of 1024 values (small sets: as many CUs as there are blocks) up to 16384, where a block's
  // own start is hidden.
  const int64_t per = std::min<int64_t>(std::max<int64_t>(cdiv(total, 2048), 1024), 16384);
  const int64_t chunk = cdiv(per, 1024) * 1024;
  hipStream_t s = (hipStream_t)stream;
  AdamWArgs a;
  a.step = step;
  a.lr_dev = lr_dev, a.grad_scale = grad_scale;
  a.log_b1 = std::log(beta1), a.log_b2 = std::log(beta2);
  a.lr = (float)lr, a.a1 = (float)(1.0 - beta1), a.a2 = (float)(1.0 - beta2);
  a.eps = (float)eps, a.decay = (float)weight_decay;
  a.k0 = k0, a.k1 = k1;
  a.chunk = (int32_t)chunk;
  a.n_tensors = 0;
  int64_t blocks = 0;
  bool counted = false;
  auto launch = [&](bool last) {
    if (!a.n_tensors) return;
    a.ticket = last ? ticket : nullptr;
    hipLaunchKernelGGL(k_adamw, dim3((unsigned)blocks), dim3(256), 0, s, a);
    a.n_tensors = 0;
    blocks = 0;
    counted = last;
  };
  int last = -1;
  for (int i = 0; i < n_tensors; ++i)
    if (sizes[i] && grads[i]) last = i;
  for (int i = 0; i < n_tensors; ++i) {
    const int64_t n = sizes[i], here = base;
    base += cdiv(n, QB) * QB;
    if (!n || !grads[i]) continue;
    const int64_t need = cdiv(n, chunk);
    if (a.n_tensors == ADAMW_TENSORS || (a.n_tensors && blocks + need > ADAMW_BLOCKS)) launch(false);
    AdamWTensor& t = a.t[a.n_tensors++];
    t.p = (float*)p[i], t.g = grads[i], t.m = m[i], t.v = v[i];
    t.m_scale = m_scale ? (float*)m_scale[i] : nullptr, t.v_scale = v_scale ? (float*)v_scale[i] : nullptr;
    t.copy = copies ? (bf16_t*)copies[i] : nullptr;
    t.n = n, t.base = here, t.first = (int32_t)blocks, t.g_bf16 = grad_dtypes[i] == PD_DTYPE_BF16;
    blocks += need;
    if (i == last) launch(true);
  }
  if (!counted) hipLaunchKernelGGL(k_adamw_count, dim3(1), dim3(1), 0, s, step);
  return check_launch(what);
}
