// dgnn_adamw.hip -- one AdamW step over many tensors (dgnn_adamw, include/dgnn_train.h).
//
// Per element the step reads p, g and two moments and writes p and the moments: there is nothing to reuse, so the kernel
// is one pass at the memory's rate and everything else is arranged around that. All tensors of a call are cut into chunks
// of 1024 to 4096 elements; a workgroup finds its tensor by bisection in a table that travels in the kernel's arguments (no
// upload, nothing to keep alive, and a captured graph keeps its own copy), 64 tensors a launch. Values that are touched once
// are loaded and stored past the caches' usual order of replacement (200 M fp32 elements: 1031 us without, 928 us with).
//
// 256 elements are the unit that shares a scale where moments are 8 bits wide. 16, 32 or 64 lanes own such a block: quad j
// of lane l of L is elements 4 (L j + l) .. + 3, so every load of 4 elements is contiguous over the lanes, and the block's
// maximum is a few exchanges among them.
//
// Measured on 200 M elements (bytes read and written): fp32 5.4 to 6.0 TB/s; 16-bit parameters with 32-bit moments 762 us, 5.8
// TB/s, with a master copy 1060 us, 5.7; 8-bit moments with a master copy 6.1 TB/s, without 4.4 (bf16) to 5.9 (fp32); a large
// copy reaches 4.75.
//
// Compiled without contraction: each operation is rounded once, in the order the header states, so results do not depend
// on how the compiler fuses.

#include "dgnn_internal.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>

namespace {

constexpr int kBlock = 256;        // elements that share a scale
constexpr int kTable = 64;         // tensors a launch: 64 * 48 B of kernel arguments stay under 4 KiB

struct Entry {
  void* param;
  const void* grad;
  int64_t numel;
  uint32_t start;                  // in blocks of 256
  float decay, rate, root;
  uint32_t turn;
  int32_t index;
};

struct Table {
  int32_t count;
  uint32_t chunks;                 // of all tensors
  uint32_t first[kTable];          // first chunk of each tensor
  Entry t[kTable];
};

struct State {
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  float* master;
  const float* factors;
  float b1, c1, b2, c2, eps;       // c = 1 - b
};

template <typename T> struct Quad { using V = T __attribute__((ext_vector_type(4), aligned(sizeof(T)))); };
typedef float f4 __attribute__((ext_vector_type(4)));

// Elements a lane takes; a workgroup takes 256 times as many. 32-bit moments are bound by memory alone and want many loads in
// flight (200 M fp32 elements: 16 928 us, 8 969 us). 8-bit ones are bound by the arithmetic as well and want waves, so few
// registers (bf16 with a master copy, 200 M elements: 16 996 us, 8 652 us, 4 598 us); without a master copy there is less to
// load and more of the rest, which 8 share better (16 616 us, 8 458 us, 4 488 us).
constexpr int each(bool bits8, bool master) { return !bits8 ? 16 : master ? 4 : 8; }

template <typename T> __device__ __forceinline__ float widen(T x) { return (float)x; }

// the largest |x| as bits: NaN above infinity above every finite value, so a value that is not finite is not lost
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int LANES> __device__ __forceinline__ uint32_t max_over(uint32_t a) {
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) {
    const uint32_t b = (uint32_t)__shfl_xor((int)a, d, LANES);
    a = a > b ? a : b;
  }
  return a;
}

// s floor(|x| / s + u) with the sign of x, s the e4m3 step at |x|
__device__ __forceinline__ float at_step(float x, float u) {
  uint32_t e = magnitude(x) & 0x7f800000u;
  e = e > (121u << 23) ? e : (121u << 23);
  const float s = __uint_as_float(e - (3u << 23));
  const float inv = __uint_as_float((257u << 23) - e);                     // 1 / s, exact
  return copysignf(floorf(fabsf(x) * inv + u) * s, x);
}

__device__ __forceinline__ float dither(uint32_t h) { return (float)(h >> 16) * 0x1p-16f; }

// The same for |x| >= 2^-6 or x = 0, in three integer operations: |x| / s has 3 bits before the 20 that the addition of
// the 16 bits of u carries into, and where the sum reaches the next power of two its floor is that power either way.
__device__ __forceinline__ float at_step_above(float x, uint32_t h) {
  return __uint_as_float((__float_as_uint(x) + ((h >> 16) << 4)) & 0xfff00000u);
}

// sqrt(x) rounded to nearest for x = 0 and 2^-96 <= x < inf: x rsq(x) is within 2 ulp, its residual is exact in an fma, and
// one correction by it rounds right (every float of the range was compared with sqrtf). 6 operations where sqrtf, which has
// to scale small arguments, takes 16.
__device__ __forceinline__ float root_above(float x) {
  const float y = __builtin_amdgcn_rsqf(fmaxf(x, 0x1p-126f));
  const float g = x * y;
  return __builtin_fmaf(__builtin_fmaf(-g, g, x), 0.5f * y, g);
}

constexpr uint32_t kMAlong = 0x6A09E667u, kMAhead = 0x9E3779B9u, kRAlong = 0x3C6EF372u, kRAhead = 0xBB67AE85u;

template <typename T, bool MASTER, bool BITS8>
__global__ __launch_bounds__(256) void adamw_kernel(const Table tab, const State st) {
  using V4 = typename Quad<T>::V;
  constexpr int EACH = each(BITS8, MASTER), LANES = kBlock / EACH;                          // elements of a lane, lanes of a block
  int lo = 0, hi = tab.count - 1;
  const uint32_t chunk = blockIdx.y * gridDim.x + blockIdx.x;
  if (chunk >= tab.chunks) return;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  const Entry& e = tab.t[lo];
  const int64_t numel = e.numel;
  T* const p = (T*)e.param;
  const T* const g = (const T*)e.grad;
  float rate = e.rate, root_c = e.root;
  uint32_t turn = e.turn;
  if (st.factors) {
    const float* f = st.factors + 4 * (int64_t)e.index;
    rate = f[0]; root_c = f[1]; turn = __float_as_uint(f[2]);
  }
  const int lane = threadIdx.x % LANES, blk = threadIdx.x / LANES;
  const int64_t at = (int64_t)(chunk - tab.first[lo]) * (256 * EACH) + blk * kBlock;      // this block's first element
  if (at >= numel) return;                                                          // whole blocks
  const int64_t sat = (int64_t)e.start * kBlock + at;                               // and its place in the state
  const bool whole = at + kBlock <= numel;
  const int left = whole ? kBlock : (int)(numel - at);

  float pw[EACH], gw[EACH], m[EACH], v[EACH];                                               // v holds the root where BITS8
#pragma unroll
  for (int j = 0; j < EACH / 4; ++j) {
    const int q = 4 * (LANES * j + lane);
    if (whole) {
      const V4 gv = __builtin_nontemporal_load(reinterpret_cast<const V4*>(g + at + q));
#pragma unroll
      for (int i = 0; i < 4; ++i) gw[4 * j + i] = widen(gv[i]);
      const V4 pv = __builtin_nontemporal_load(reinterpret_cast<const V4*>(p + at + q));
#pragma unroll
      for (int i = 0; i < 4; ++i) pw[4 * j + i] = widen(pv[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        gw[4 * j + i] = q + i < left ? widen(g[at + q + i]) : 0.f;
        pw[4 * j + i] = q + i < left ? widen(p[at + q + i]) : 0.f;
      }
    }
    if constexpr (MASTER) {
      const f4 wide = __builtin_nontemporal_load(reinterpret_cast<const f4*>(st.master + sat + q));
#pragma unroll
      for (int i = 0; i < 4; ++i)                                                   // else p was written by somebody else
        if (__float_as_uint(widen((T)wide[i])) == __float_as_uint(pw[4 * j + i])) pw[4 * j + i] = wide[i];
    }
    if constexpr (BITS8) {
      const uint32_t mc = *reinterpret_cast<const uint32_t*>((const uint8_t*)st.m + sat + q);
      const uint32_t vc = *reinterpret_cast<const uint32_t*>((const uint8_t*)st.v + sat + q);
      m[4 * j + 0] = __builtin_amdgcn_cvt_f32_fp8((int)mc, 0);
      m[4 * j + 1] = __builtin_amdgcn_cvt_f32_fp8((int)mc, 1);
      m[4 * j + 2] = __builtin_amdgcn_cvt_f32_fp8((int)mc, 2);
      m[4 * j + 3] = __builtin_amdgcn_cvt_f32_fp8((int)mc, 3);
      v[4 * j + 0] = __builtin_amdgcn_cvt_f32_fp8((int)vc, 0);
      v[4 * j + 1] = __builtin_amdgcn_cvt_f32_fp8((int)vc, 1);
      v[4 * j + 2] = __builtin_amdgcn_cvt_f32_fp8((int)vc, 2);
      v[4 * j + 3] = __builtin_amdgcn_cvt_f32_fp8((int)vc, 3);
    } else {
      const f4 mv = __builtin_nontemporal_load(reinterpret_cast<const f4*>((const float*)st.m + sat + q));
      const f4 vv = __builtin_nontemporal_load(reinterpret_cast<const f4*>((const float*)st.v + sat + q));
#pragma unroll
      for (int i = 0; i < 4; ++i) { m[4 * j + i] = mv[i]; v[4 * j + i] = vv[i]; }
    }
  }

  const int64_t b = sat / kBlock;
  float ms = 0.f, vs = 0.f;
  if constexpr (BITS8) { ms = st.m_scale[b]; vs = st.v_scale[b]; }
  uint32_t mtop = 0, vtop = 0, low = 0xffffffffu, high = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    float mi = m[i], vi = v[i];
    const float gi = gw[i];
    if constexpr (BITS8) {
      mi = mi * ms;
      const float r = vi * vs;
      vi = r * r;
    }
    m[i] = mi * st.b1 + gi * st.c1;
    v[i] = vi * st.b2 + (gi * gi) * st.c2;
    if constexpr (BITS8) {
      low = min(low, __float_as_uint(v[i]) - 1);                                    // zero wraps round to the top
      high = max(high, __float_as_uint(v[i]));
    }
  }
  if constexpr (BITS8) {
    if (__any(low < 0x0f800000u - 1 || high >= 0x7f800000u)) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) v[i] = sqrtf(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < EACH; ++i) v[i] = root_above(v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const float r = BITS8 ? v[i] : sqrtf(v[i]);
    const float step = m[i] / (r * root_c + st.eps);
    pw[i] = pw[i] * e.decay - step * rate;
    if constexpr (BITS8) {
      if (whole || 4 * (LANES * (i >> 2) + lane) + (i & 3) < left) {
        mtop = max(mtop, magnitude(m[i]));
        vtop = max(vtop, magnitude(r));
      }
    }
  }

  if constexpr (BITS8) {
    mtop = max(max_over<LANES>(mtop), __float_as_uint(0x1p-100f));
    vtop = max(max_over<LANES>(vtop), __float_as_uint(0x1p-100f));
    const float mt = __uint_as_float(mtop), vt = __uint_as_float(vtop);
    const float minv = 448.f / mt, vinv = 448.f / vt;
    if (lane == 0) { st.m_scale[b] = mt * (1.f / 448.f); st.v_scale[b] = vt * (1.f / 448.f); }
    const uint32_t hm = (uint32_t)(at + 4 * lane) * kMAlong + turn * kMAhead;
    const uint32_t hr = (uint32_t)(at + 4 * lane) * kRAlong + turn * kRAhead;
    low = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      m[i] = m[i] * minv;
      v[i] = v[i] * vinv;
      low = min(low, (__float_as_uint(m[i]) << 1) - 2);                             // without the sign
      low = min(low, (__float_as_uint(v[i]) << 1) - 2);
    }
    // A value below 2^-6 of the codes' 448 is one in 10^4 of normally distributed ones, so most waves have none
    if (__any(low < (0x3c800000u << 1) - 2 || mtop >= 0x7f800000u || vtop >= 0x7f800000u)) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const uint32_t k = 4 * LANES * (i >> 2) + (i & 3);
        m[i] = at_step(m[i], dither(hm + k * kMAlong));
        const float c = at_step(v[i], dither(hr + k * kRAlong));
        v[i] = v[i] > 0.f && c < 0x1p-9f ? 0x1p-9f : c;
      }
    } else {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const uint32_t k = 4 * LANES * (i >> 2) + (i & 3);
        m[i] = at_step_above(m[i], hm + k * kMAlong);
        v[i] = at_step_above(v[i], hr + k * kRAlong);
      }
    }
  }

#pragma unroll
  for (int j = 0; j < EACH / 4; ++j) {
    const int q = 4 * (LANES * j + lane);
    if (whole) {
      V4 pv;
#pragma unroll
      for (int i = 0; i < 4; ++i) pv[i] = (T)pw[4 * j + i];
      __builtin_nontemporal_store(pv, reinterpret_cast<V4*>(p + at + q));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (q + i < left) p[at + q + i] = (T)pw[4 * j + i];
    }
    if constexpr (MASTER) {
      f4 pv;
#pragma unroll
      for (int i = 0; i < 4; ++i) pv[i] = whole || q + i < left ? pw[4 * j + i] : 0.f;
      __builtin_nontemporal_store(pv, reinterpret_cast<f4*>(st.master + sat + q));
    }
    if constexpr (BITS8) {
      int mc = __builtin_amdgcn_cvt_pk_fp8_f32(m[4 * j], m[4 * j + 1], 0, false);
      mc = __builtin_amdgcn_cvt_pk_fp8_f32(m[4 * j + 2], m[4 * j + 3], mc, true);
      int vc = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j], v[4 * j + 1], 0, false);
      vc = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j + 2], v[4 * j + 3], vc, true);
      *reinterpret_cast<int*>((uint8_t*)st.m + sat + q) = mc;
      *reinterpret_cast<int*>((uint8_t*)st.v + sat + q) = vc;
    } else {
      f4 mv, vv;
#pragma unroll
      for (int i = 0; i < 4; ++i) { mv[i] = m[4 * j + i]; vv[i] = v[4 * j + i]; }
      __builtin_nontemporal_store(mv, reinterpret_cast<f4*>((float*)st.m + sat + q));
      __builtin_nontemporal_store(vv, reinterpret_cast<f4*>((float*)st.v + sat + q));
    }
  }
}

// Advances the device's step counters and derives what depends on them (one lane a tensor).
__global__ __launch_bounds__(64) void adamw_tick_kernel(const Table tab, int64_t* steps, float* factors, double lr, double b1, double b2) {
  const int i = threadIdx.x;
  if (i >= tab.count) return;
  const int64_t at = tab.t[i].index;
  const int64_t t = steps[at] + 1;
  steps[at] = t;
  float* f = factors + 4 * at;
  f[0] = (float)(lr / (1.0 - pow(b1, (double)t)));
  f[1] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
  f[2] = __uint_as_float((uint32_t)t);
}

template <typename T>
void launch(const Table& tab, const State& st, bool master, bool bits8, hipStream_t s) {
  constexpr uint32_t row = 1 << 23;                      // a grid holds fewer than 2^32 lanes along a side
  const dim3 g(tab.chunks < row ? tab.chunks : row, (tab.chunks + row - 1) / row), b(256);
  if (bits8) {
    if (master) hipLaunchKernelGGL((adamw_kernel<T, true, true>), g, b, 0, s, tab, st);
    else hipLaunchKernelGGL((adamw_kernel<T, false, true>), g, b, 0, s, tab, st);
  } else {
    if (master) hipLaunchKernelGGL((adamw_kernel<T, true, false>), g, b, 0, s, tab, st);
    else hipLaunchKernelGGL((adamw_kernel<T, false, false>), g, b, 0, s, tab, st);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int dgnn_adamw(const struct dgnn_adamw_tensor* tensors, int32_t count, int32_t dtype, int32_t state_bits,
                          const struct dgnn_adamw_state* state, double lr, double beta1, double beta2, double eps, void* stream) {
  if (count < 0 || (count > 0 && !tensors) || !state) return dgnn_fail(DGNN_E_BADARG, "adamw: bad argument%s");
  if (dtype != DGNN_F32 && dtype != DGNN_BF16 && dtype != DGNN_F16) return dgnn_fail(DGNN_E_BADARG, "adamw: unknown type%s (%lld)", "", dtype);
  if (state_bits != 32 && state_bits != 8) return dgnn_fail(DGNN_E_BADARG, "adamw: moments have 32 or 8 bits%s (got %lld)", "", state_bits);
  if (!(lr >= 0) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0)) return dgnn_fail(DGNN_E_BADARG, "adamw: lr, beta or eps out of range%s");
  if (count == 0) return DGNN_OK;
  int32_t filled = 0;
  for (int32_t i = 0; i < count; ++i) filled += tensors[i].numel > 0;
  if (filled && (!state->exp_avg || !state->exp_avg_sq || (state_bits == 8 && (!state->exp_avg_scale || !state->exp_avg_sq_scale))))
    return dgnn_fail(DGNN_E_BADARG, "adamw: null state buffer%s");
  if (!aligned16(state->exp_avg) || !aligned16(state->exp_avg_sq) || !aligned16(state->master))
    return dgnn_fail(DGNN_E_BADARG, "adamw: state buffers must be 16-byte aligned%s");
  if (!state->steps != !state->factors) return dgnn_fail(DGNN_E_BADARG, "adamw: steps and factors go together%s");
  const uintptr_t esz = dtype == DGNN_F32 ? 4 : 2;
  for (int32_t i = 0; i < count; ++i) {
    const struct dgnn_adamw_tensor& t = tensors[i];
    if (t.numel < 0 || t.numel > (1LL << 38) || t.start < 0 || t.start % kBlock || t.start > (1LL << 39))
      return dgnn_fail(DGNN_E_BADARG, "adamw: bad size or start of tensor%s %lld", "", i);
    if (t.numel > 0 && (!t.param || !t.grad || (uintptr_t)t.param % esz || (uintptr_t)t.grad % esz))
      return dgnn_fail(DGNN_E_BADARG, "adamw: null or misaligned pointer of tensor%s %lld", "", i);
    if (state->steps && t.index < 0) return dgnn_fail(DGNN_E_BADARG, "adamw: negative index of tensor%s %lld", "", i);
  }
  hipStream_t s = (hipStream_t)stream;
  const State st{state->exp_avg, state->exp_avg_sq, state->exp_avg_scale, state->exp_avg_sq_scale, state->master, state->factors,
                 (float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
  const int64_t chunk = 256 * each(state_bits == 8, state->master != nullptr);
  constexpr int64_t most = 1 << 30;                      // chunks a launch
  for (int32_t i = 0; i < count;) {
    Table tab;
    tab.count = 0;
    tab.chunks = 0;
    int64_t chunks = 0;
    while (i < count && tab.count < kTable) {
      const struct dgnn_adamw_tensor& t = tensors[i];
      const int64_t need = (t.numel + chunk - 1) / chunk;
      if (chunks + need > most && tab.count) break;
      if (need || state->steps) {                        // an empty tensor still counts its steps
        tab.first[tab.count] = (uint32_t)chunks;
        tab.t[tab.count++] = Entry{t.param, t.grad, t.numel, (uint32_t)(t.start / kBlock), t.decay, t.rate, t.root, t.turn, t.index};
        chunks += need;
      }
      ++i;
    }
    if (tab.count == 0) break;
    if (state->steps) {
      hipLaunchKernelGGL(adamw_tick_kernel, dim3(1), dim3(64), 0, s, tab, state->steps, state->factors, lr, beta1, beta2);
      DGNN_LAUNCHED();
    }
    if (chunks == 0) continue;
    tab.chunks = (uint32_t)chunks;
    if (dtype == DGNN_F32) launch<float>(tab, st, state->master != nullptr, state_bits == 8, s);
    else if (dtype == DGNN_BF16) launch<__bf16>(tab, st, state->master != nullptr, state_bits == 8, s);
    else launch<_Float16>(tab, st, state->master != nullptr, state_bits == 8, s);
    DGNN_LAUNCHED();
  }
  return DGNN_OK;
}
