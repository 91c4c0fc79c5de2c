// dgnn_gemm.h -- the matrix product behind dgnn_linear_*: C[M x N] = A[M x K] B[K x N] on the matrix cores with the layer's
// epilogue. Compiled once per element type (dgnn_gemm_f32.hip, dgnn_gemm_bf16.hip, dgnn_gemm_f16.hip).
//
// Each operand comes in one of two layouts: "along" keeps the contraction contiguous in memory (x and P in x W and P W^T, W in
// P W^T), "across" keeps the other dimension contiguous (W in x W, both operands of x^T P). Either way a tile is staged in
// LDS as 16-byte chunks of 8 consecutive contraction elements of one row (or column), chunk-major: what one lane hands to
// v_mfma_f32_32x32x16 is one ds_read_b128, and 32 lanes read 512 consecutive bytes. "Across" tiles are turned in registers: a
// lane loads 8 contraction rows of a few columns and writes one chunk per column.
//
// fp32 operands: gfx950 has no wide fp32 matrix instruction (its 32-bit rate is a sixteenth of bf16's), so an fp32 value is
// split into three bf16 pieces a = a1 + a2 + a3, each the rounding of what the ones before leave (8 bits each, 24 in all, so
// the split is exact up to 2^-25 |a|), and the six products of at least 2^-16 relative size are summed in the fp32
// accumulators: a1 b1 + a1 b2 + a2 b1 + a2 b2 + a1 b3 + a3 b1. What is left out is at most 2^-24 |a| |b| a term, as much as
// one fp32 rounding. Values under 2^-109 lose bits (their last pieces are below bf16's smallest number): absolute
// errors of 2^-134 |b|. An infinity's pieces are not finite and would give NaN where fp32 gives infinity, so a tile of 32 x 32
// outputs with some that are not finite is multiplied again by fp32's own matrix instruction (again() below), whose infinities
// and NaN are those of fp32 operations; only the outputs that are not finite take its values.
#pragma once
#include "dgnn_internal.h"

#include <type_traits>

namespace dgnn {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

struct Gemm {
  const void* a;
  const void* b;
  int64_t lda, ldb;
  bool a_along, b_along;
  int64_t M, N, K;
  // epilogue: c = act(acc + bias) + residual; save receives acc + bias in fp32 (or, for relu, a bit per value that is > 0): in 16
  // bits its rounding would be the largest error of the gradients' column sums
  const void* bias;
  const void* residual;
  int64_t ld_residual;
  void* c;
  int64_t ldc;
  void* save;
  int64_t ld_save;
  int act;
  float* partial;          // slices x M x N when slices > 1 (x 2 N with `pieces`, however many slices)
  int slices;
  bool pieces;             // b is M rows of 2 N values, each second N what rounding left of the first: c = a (first + second)
  int64_t slice_k;         // contraction elements a slice takes, a multiple of 32 (of 64 by tiles)
  char* image;             // room for W's image where the product runs on rows_kernel, else null
  hipStream_t stream;
};

// The normal distribution's density e = exp(-t^2/2) (times sqrt(2 pi)) and tail Phi(-|t|), for results of 16 bits: the tail is
// e u P(u), u = 1 / (1 + 0.36 |t|), P fitted to a relative error below 1e-6 over |t| <= 14, beyond which both are 0 in
// fp32 -- 2^-9 is what a result's rounding is off by. 15 operations where erff and expf take some 60.
__device__ __forceinline__ void normal_tail(float t, float& e, float& tail) {
  const float u = __builtin_amdgcn_rcpf(fmaf(0.36f, fabsf(t), 1.f));
  e = __builtin_amdgcn_exp2f(t * t * -0.72134752044448170f);
  float q = 0.04706796788f;
  q = fmaf(q, u, -0.1798049046f);
  q = fmaf(q, u, 0.1810091365f);
  q = fmaf(q, u, 0.02651105193f);
  q = fmaf(q, u, 0.1397333685f);
  q = fmaf(q, u, 0.1417698558f);
  q = fmaf(q, u, 0.1437132311f);
  tail = e * u * q;
}

template <typename T> __device__ __forceinline__ float sigmoid_of(float t) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t * -1.4426950408889634f));
  else return 1.f / (1.f + expf(-t));
}

template <typename T> __device__ __forceinline__ float act_of(int act, float t) {
  switch (act) {
    case ACT_RELU: return t <= 0.f ? 0.f : t;
    case ACT_GELU:
      if constexpr (sizeof(T) == 2) {
        float e, tail;
        normal_tail(t, e, tail);
        return t * (t < 0.f ? tail : 1.f - tail);
      } else {
        return 0.5f * t * (1.f + erff(t * 0.70710678118654752f));
      }
    case ACT_SILU: return sizeof(T) == 2 ? t * sigmoid_of<T>(t) : t / (1.f + expf(-t));
    default: return t;
  }
}

// f(0), f(1), ... f(N - 1) with constant arguments: register arrays that f indexes stay in registers whatever its size
template <int I, int N, typename F> __device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    each<I + 1, N>(f);
  }
}

template <typename T> struct Unit;          // W: elements of a 16-byte load
template <> struct Unit<float> { static constexpr int W = 4, PLANES = 3, BK = 32; };
template <> struct Unit<__bf16> { static constexpr int W = 8, PLANES = 1, BK = 64; };
template <> struct Unit<_Float16> { static constexpr int W = 8, PLANES = 1, BK = 64; };

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// 16 bytes at an address that is only element-aligned
template <typename T> __device__ __forceinline__ u4 load16(const T* p) {
  if constexpr (sizeof(T) == 4) return *reinterpret_cast<const u4_at4*>(p);
  else return *reinterpret_cast<const u4_at2*>(p);
}

// W elements of which only the first `n` (0..W) exist; the others are zero
template <typename T> __device__ __forceinline__ u4 load_some(const T* p, int64_t n) {
  constexpr int W = Unit<T>::W;
  union { u4 v; T e[W]; } r;
  r.v = u4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < W; ++i)
    if (i < n) r.e[i] = p[i];
  return r.v;
}

// W elements of which only the first `n` exist where reading all of them is safe (what lies behind a row's end is the next row)
template <typename T> __device__ __forceinline__ u4 load_masked(const T* p, int64_t n) {
  u4 v = load16(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) v[i] = i < n ? v[i] : 0u;
    else v[i] = 2 * i + 1 < n ? v[i] : 2 * i < n ? v[i] & 0xffffu : 0u;
  }
  return v;
}

__device__ __forceinline__ uint32_t pack_bf(float x, float y) {
  union { bf2 h; uint32_t u; } r;
  r.h = __builtin_convertvector(f2{x, y}, bf2);
  return r.u;
}

// 8 fp32 values -> 3 chunks of 8 bf16: their exact sum is the value to 24 bits
__device__ __forceinline__ void split8(const float (&v)[8], u4 (&out)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = v[2 * i], y = v[2 * i + 1];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t h = pack_bf(x, y);
      out[p][i] = h;
      if (p < 2) { x -= __uint_as_float(h << 16); y -= __uint_as_float(h & 0xffff0000u); }
    }
  }
}

// One operand's tile: ROWS rows (or columns) by BK contraction elements, fetched by THREADS lanes into registers and stored
// to LDS as PLANES x BK/8 chunk columns.
template <typename T, bool ALONG, int ROWS, int THREADS> struct Tile {
  static constexpr int W = Unit<T>::W, BK = Unit<T>::BK, PL = Unit<T>::PLANES, CH = BK / 8;
  static constexpr int COLUMN = ROWS * 16 + 32;               // bytes of a chunk column; the 32 spread chunk columns over banks
  static constexpr int BYTES = PL * CH * COLUMN;
  static constexpr int UNITS = ALONG ? ROWS * CH : (ROWS / W) * CH;
  static constexpr int PER = (UNITS + THREADS - 1) / THREADS;
  static constexpr int QUADS = ALONG ? 8 / W : 8;             // 16-byte loads of a unit
  u4 r[PER][QUADS];

  // chunks of neighbouring rows lie side by side; the exchange inside groups of 8 spreads the writes of turned tiles,
  // whose lanes are W rows apart, over the banks
  static __device__ __forceinline__ int place(int row) { return row ^ ((row >> 4) & 7); }

  // `kall`: the whole contraction, kend the slice's. Loads may run over a row's end wherever another row follows: rows (or
  // columns) past the operand's give sums that nobody keeps, contraction elements past kend are made zero.
  __device__ __forceinline__ void fetch(const T* base, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int64_t kend, int64_t kall, int tid) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int id = tid + u * THREADS;
      if (UNITS % THREADS != 0 && id >= UNITS) break;
      if constexpr (ALONG) {
        int64_t row = row0 + id / CH;
        row = row < rows ? row : rows - 1;
        const T* p = base + row * ld + k0 + 8 * (id % CH);
        const int64_t left = kend - k0 - 8 * (id % CH);
        if (left >= 8) {
#pragma unroll
          for (int q = 0; q < QUADS; ++q) r[u][q] = load16(p + q * W);
        } else if (left > 0 && row + 1 < rows && ld >= 8) {
#pragma unroll
          for (int q = 0; q < QUADS; ++q) r[u][q] = load_masked(p + q * W, left - q * W);
        } else {
#pragma unroll
          for (int q = 0; q < QUADS; ++q) r[u][q] = load_some(p + q * W, left - q * W);
        }
      } else {
        const int64_t k = k0 + 8 * (id / (ROWS / W));
        int64_t col = row0 + (id % (ROWS / W)) * W;
        if (k0 + BK <= kend && k0 + BK < kall && ld >= W) {
          col = col < rows ? col : row0;
          const T* p = base + k * ld + col;
#pragma unroll
          for (int q = 0; q < 8; ++q) r[u][q] = load16(p + q * ld);
        } else {
          const T* p = base + k * ld + col;
          const int64_t left = rows - col;
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            if (k + q >= kend) r[u][q] = u4{0, 0, 0, 0};
            else if (left >= W) r[u][q] = load16(p + q * ld);
            else r[u][q] = load_some(p + q * ld, left);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void store(char* lds, int tid) const {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int id = tid + u * THREADS;
      if (UNITS % THREADS != 0 && id >= UNITS) break;
      if constexpr (ALONG) {
        char* at = lds + (id % CH) * COLUMN + place(id / CH) * 16;
        if constexpr (PL == 3) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[u][i / 4][i % 4]);
          u4 h[3];
          split8(v, h);
#pragma unroll
          for (int p = 0; p < 3; ++p) *reinterpret_cast<u4*>(at + p * CH * COLUMN) = h[p];
        } else {
          *reinterpret_cast<u4*>(at) = r[u][0];
        }
      } else {
        const int row = (id % (ROWS / W)) * W;
        char* col = lds + (id / (ROWS / W)) * COLUMN;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          char* at = col + place(row + w) * 16;
          if constexpr (PL == 3) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[u][i][w]);
            u4 h[3];
            split8(v, h);
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<u4*>(at + p * CH * COLUMN) = h[p];
          } else {
            u4 h;
#pragma unroll
            for (int i = 0; i < 4; ++i)                       // half w of rows 2i and 2i + 1
              h[i] = __builtin_amdgcn_perm(r[u][2 * i + 1][w / 2], r[u][2 * i][w / 2], w % 2 ? 0x07060302u : 0x05040100u);
            *reinterpret_cast<u4*>(at) = h;
          }
        }
      }
    }
  }
};

__device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c, __bf16) {
  union { u4 u; bf8 h; } x, y;
  x.u = a; y.u = b;
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.h, y.h, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c, float) { return mfma(a, b, c, __bf16()); }
__device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c, _Float16) {
  union { u4 u; h8 h; } x, y;
  x.u = a; y.u = b;
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, y.h, c, 0, 0, 0);
}

// sums that are not finite: 0 if there are none, else NaN
__device__ __forceinline__ float unsound(const f16v& acc) {
  float seen = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) seen = fmaf(acc[e], 0.f, seen);
  return seen;
}

// Those of a wave's 32 x 32 sums that are not finite, once more, from `t`: D[m][n] += sum over k of a(m, k) b(n, k), a lane's
// a(lane % 32, k) at a + k ak and b(lane % 32, k) at b + k bk. All lanes take part. A step of two of the contraction takes 64
// cycles, 2.7 times the six bf16 products, and its operands come from memory one by one: with every value NaN 232965 x 602 x 256
// takes 2509 us (finite 522), 4096 x 256 x 256 84 (18.6); with one infinity in the latter's x 74. (A chain of multiply-adds by
// the lane that holds a sum: 1935 and 1584.)
__device__ __forceinline__ void again(f16v& acc, f16v t, const float* a, int64_t ak, const float* b, int64_t bk, int64_t k0, int64_t kend) {
  constexpr int U = 4;                                         // loads of each operand in flight
  const int64_t mine = U * ((threadIdx.x & 63) >> 5);
  a += (k0 + mine) * ak;
  b += (k0 + mine) * bk;
#pragma unroll 1
  for (int64_t left = kend - k0; left > 0; left -= 2 * U) {
    float x[U], y[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const bool in = mine + i < left;
      x[i] = in ? a[i * ak] : 0.f;
      y[i] = in ? b[i * bk] : 0.f;
    }
    a += 2 * U * ak;
    b += 2 * U * bk;
#pragma unroll
    for (int i = 0; i < U; ++i) t = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], t, 0, 0, 0);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = fabsf(acc[e]) < __builtin_huge_valf() ? acc[e] : t[e];
}

template <typename T> struct Four { typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T) == 4 ? 4 : 2))); };

// `have` (0..4) elements at p; the others are zero
template <typename T> __device__ __forceinline__ void load4(const T* p, int have, float (&v)[4]) {
  if (have == 4) {
    const typename Four<T>::type q = *reinterpret_cast<const typename Four<T>::type*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)q[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < have ? (float)p[i] : 0.f;
  }
}

template <typename T> __device__ __forceinline__ void store4(T* p, int have, const float (&v)[4]) {
  if (have == 4) {
    typename Four<T>::type q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = (T)v[i];
    *reinterpret_cast<typename Four<T>::type*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < have) p[i] = (T)v[i];
  }
}

// What 4 neighbouring sums of a row become: bias, saved slope data, activation, residual, one rounding. Lanes of a wave hold
// neighbouring fours (8 lanes make relu's word of 32 bits), `have` of the 4 exist (0: none, but the lane still takes part).
template <typename T>
__device__ __forceinline__ void finish(const Gemm& g, int64_t row, int64_t col, int have, float (&v)[4], const float (&bias)[4], const float (&res)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] += bias[i];
  if (g.save && g.act == ACT_RELU) {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) bits |= (i < have && !(v[i] <= 0.f) ? 1u : 0u) << i;
    const int lane = threadIdx.x & 7;
    bits <<= 4 * lane;
    bits |= __shfl_xor(bits, 1);
    bits |= __shfl_xor(bits, 2);
    bits |= __shfl_xor(bits, 4);
    if (lane == 0 && have > 0) ((uint32_t*)g.save)[row * g.ld_save + col / 32] = bits;
  } else if (g.save) {
    store4((float*)g.save + row * g.ld_save + col, have, v);
  }
  switch (g.act) {
    case ACT_NONE: break;
    case ACT_RELU:
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = act_of<T>(ACT_RELU, v[i]);
      break;
    case ACT_GELU:
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = act_of<T>(ACT_GELU, v[i]);
      break;
    default:
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = act_of<T>(ACT_SILU, v[i]);
  }
  if (g.residual) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += res[i];
  }
  store4((T*)g.c + row * g.ldc + col, have, v);
}

// Lanes of a wave exchange values through LDS: what was written before is there for what is read behind, whichever lane's it is.
// The wave's LDS operations run in order, so this is an order for the compiler and no instruction.
__device__ __forceinline__ void lanes_meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wave's TM x TN tiles of 32 x 32 from its accumulators to memory, 32 rows at a time through its own part of LDS: the
// matrix cores leave a column's rows in a lane, memory wants a row's columns side by side (16 bytes of fp32 a lane). The
// residual's rows are fetched before the turn, so that nothing waits for them one by one.
template <typename T, int TM, int TN, bool AA, bool BA>
__device__ __forceinline__ void epilogue(const Gemm& g, f16v (&acc)[TM][TN], float* room, int64_t row0, int64_t col0, int64_t k0, int64_t kend) {
  constexpr int PITCH = TN * 32 + 4, LANES = TN * 8, STEP = 64 / LANES, TURNS = 32 / STEP;
  const int lane = threadIdx.x & 63;
  const int64_t col = col0 + (lane % LANES) * 4;
  const int have_n = g.N - col >= 4 ? 4 : (g.N > col ? (int)(g.N - col) : 0);
  const bool whole = g.slices == 1 && !g.pieces;
  float bias[4] = {0.f, 0.f, 0.f, 0.f};
  if (whole && g.bias) load4((const T*)g.bias + col, have_n, bias);
  if constexpr (Unit<T>::PLANES == 3) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int64_t m = row0 + i * 32 + (lane & 31), n = col0 + j * 32 + (lane & 31);          // past the ends the last ones stand in
        if (!__ballot(n < g.N && !(unsound(acc[i][j]) == 0.f))) continue;
        const int64_t mi = m < g.M ? m : g.M - 1, ni = n < g.N ? n : g.N - 1;
        again(acc[i][j], f16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0}, (const T*)g.a + (AA ? mi * g.lda : mi), AA ? 1 : g.lda,
              (const T*)g.b + (BA ? ni * g.ldb : ni), BA ? 1 : g.ldb, k0, kend);
      }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t first = row0 + i * 32 + lane / LANES;
    float res[TURNS][4];
    if (whole && g.residual) {
#pragma unroll
      for (int q = 0; q < TURNS; ++q) {
        const int64_t row = first + q * STEP;
        load4((const T*)g.residual + row * g.ld_residual + col, row < g.M ? have_n : 0, res[q]);
      }
    }
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e)              // element e of a lane: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32
        room[(8 * (e / 4) + 4 * (lane >> 5) + e % 4) * PITCH + j * 32 + (lane & 31)] = acc[i][j][e];
    lanes_meet();
#pragma unroll
    for (int q = 0; q < TURNS; ++q) {
      const int64_t row = first + q * STEP;
      const int have = row < g.M ? have_n : 0;
      const float4 t = *reinterpret_cast<const float4*>(room + (lane / LANES + q * STEP) * PITCH + (lane % LANES) * 4);
      float v[4] = {t.x, t.y, t.z, t.w};
      if (whole) finish<T>(g, row, col, have, v, bias, res[q]);
      else store4(g.partial + ((int64_t)blockIdx.y * g.M + row) * g.N + col, have, v);
    }
    lanes_meet();                               // the next 32 rows take the same room
  }
}

// The product by tiles: while a stage is multiplied from one LDS buffer, the next one is on its way to registers and is then
// written to the other. For weight gradients, for outputs too small for rows_kernel and for what is cut into slices. Bound by
// LDS: a wave's 64 x 64 take a 16-byte read for each matrix instruction, and turned operands are written there 16 bytes a lane.
// bf16 8192 x 1024 x 4096 (x^T p) 117 us, 590 TFLOP/s, where a large library product reaches 1138; fp32 232965 x 256 x 256 222 us,
// 137 TFLOP/s (library 153); 2708 x 1433 x 16 fp32 13 us, which is latency: 22 row tiles, 12 slices, a join.
template <typename T, bool AA, bool BA, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void gemm_kernel(const Gemm g) {
  constexpr int THREADS = WM * WN * 64, BK = Unit<T>::BK, PL = Unit<T>::PLANES;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  using TA = Tile<T, AA, BM, THREADS>;
  using TB = Tile<T, BA, BN, THREADS>;
  __shared__ __attribute__((aligned(16))) char lds[2][TA::BYTES + TB::BYTES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave % WM, wn = wave / WM;
  const int64_t tiles_n = (g.N + BN - 1) / BN;
  const int64_t row0 = (int64_t)(blockIdx.x / tiles_n) * BM, col0 = (int64_t)(blockIdx.x % tiles_n) * BN;
  const int64_t k0 = (int64_t)blockIdx.y * g.slice_k;
  const int64_t kend = k0 + g.slice_k < g.K ? k0 + g.slice_k : g.K;
  const T* a = (const T*)g.a;
  const T* b = (const T*)g.b;

  f16v acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

  TA ta;
  TB tb;
  if (k0 < kend) {
    ta.fetch(a, g.lda, row0, g.M, k0, kend, g.K, tid);
    tb.fetch(b, g.ldb, col0, g.N, k0, kend, g.K, tid);
    ta.store(lds[0], tid);
    tb.store(lds[0] + TA::BYTES, tid);
  }
  __syncthreads();
  int buf = 0;
  for (int64_t k = k0; k < kend; k += BK) {
    const bool more = k + BK < kend;
    if (more) {
      ta.fetch(a, g.lda, row0, g.M, k + BK, kend, g.K, tid);
      tb.fetch(b, g.ldb, col0, g.N, k + BK, kend, g.K, tid);
    }
    const char* la = lds[buf];
    const char* lb = lds[buf] + TA::BYTES;
#pragma unroll
    for (int s = 0; s < BK / 16; ++s) {
      const int chunk = 2 * s + (lane >> 5);
      u4 fa[TM][PL], fb[TN][PL];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int p = 0; p < PL; ++p)
          fa[i][p] = *reinterpret_cast<const u4*>(la + (p * (BK / 8) + chunk) * TA::COLUMN + TA::place((wm * TM + i) * 32 + (lane & 31)) * 16);
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int p = 0; p < PL; ++p)
          fb[j][p] = *reinterpret_cast<const u4*>(lb + (p * (BK / 8) + chunk) * TB::COLUMN + TB::place((wn * TN + j) * 32 + (lane & 31)) * 16);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if constexpr (PL == 3) {                             // small products first
            acc[i][j] = mfma(fa[i][2], fb[j][0], acc[i][j], T());
            acc[i][j] = mfma(fa[i][0], fb[j][2], acc[i][j], T());
            acc[i][j] = mfma(fa[i][1], fb[j][1], acc[i][j], T());
            acc[i][j] = mfma(fa[i][1], fb[j][0], acc[i][j], T());
            acc[i][j] = mfma(fa[i][0], fb[j][1], acc[i][j], T());
          }
          acc[i][j] = mfma(fa[i][0], fb[j][0], acc[i][j], T());
        }
    }
    if (more) {
      ta.store(lds[buf ^ 1], tid);
      tb.store(lds[buf ^ 1] + TA::BYTES, tid);
    }
    __syncthreads();
    buf ^= 1;
  }

  static_assert(WM * WN * 32 * (TN * 32 + 4) * 4 <= 2 * (TA::BYTES + TB::BYTES), "the epilogue's rows fit the tiles' LDS");
  epilogue<T, TM, TN, AA, BA>(g, acc, reinterpret_cast<float*>(&lds[0][0]) + wave * 32 * (TN * 32 + 4), row0 + wm * TM * 32,
                              col0 + wn * TN * 32, k0, kend);
}

// Joins the slices of a product that was cut along its contraction and finishes it, in 64 bits: PARTS lanes to a four of
// columns, each adding every PARTS-th slice with up to 8 loads in flight; the PARTS sums meet in their order. Up to 8 slices
// one lane has them all in flight by itself (1024 x 4096 bf16 from 2: 30 us with 8 lanes, 11 with one); with more, as
// small outputs have them, 8 lanes shorten the chain. A row takes a multiple of 8 fours, so that relu's bits are whole words.
template <typename T, int PARTS>
__global__ __launch_bounds__(256) void gemm_join_kernel(const Gemm g) {
  constexpr int FOURS = 256 / PARTS;
  __shared__ double sums[PARTS > 1 ? PARTS : 1][PARTS > 1 ? FOURS : 1][4];
  const int four = threadIdx.x % FOURS, part = threadIdx.x / FOURS;
  const int64_t wide = (g.N + 31) / 32 * 8;
  const int64_t at = (int64_t)blockIdx.x * FOURS + four;
  const int64_t row = at / wide, col = at % wide * 4;
  const int have = row < g.M && col < g.N ? (g.N - col >= 4 ? 4 : (int)(g.N - col)) : 0;
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  if (have) {
    const float* p = g.partial + row * g.N + col;
    const int64_t step = g.M * g.N;
    for (int s = part; s < g.slices; s += 8 * PARTS) {
      float t[8][4];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s + PARTS * u < g.slices) load4(p + (s + PARTS * u) * step, have, t[u]);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s + PARTS * u < g.slices) {
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] += t[u][i];
        }
    }
  }
  if constexpr (PARTS > 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[part][four][i] = sum[i];
    __syncthreads();
    if (part) return;
  }
  float bias[4] = {0.f, 0.f, 0.f, 0.f}, res[4] = {0.f, 0.f, 0.f, 0.f};
  if (have && g.bias) load4((const T*)g.bias + col, have, bias);
  if (have && g.residual) load4((const T*)g.residual + row * g.ld_residual + col, have, res);
  if constexpr (PARTS > 1) {
#pragma unroll
    for (int k = 1; k < PARTS; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += sums[k][four][i];
  }
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)sum[i];
  finish<T>(g, row, col, have, v, bias, res);
}

// The same for a product whose right operand came in two pieces: a four of columns adds its own sums and those of the second
// pieces, N columns on. Where that is not finite the first pieces' sums alone stand, which are the product with p rounded to
// 16 bits: an infinity times two pieces of opposite signs would be NaN.
template <typename T>
__global__ __launch_bounds__(256) void pieces_join_kernel(const Gemm g) {
  constexpr int PARTS = 8, FOURS = 256 / PARTS;
  __shared__ double sums[PARTS][FOURS][8];
  const int four = threadIdx.x % FOURS, part = threadIdx.x / FOURS;
  const int64_t wide = (g.N + 3) / 4, at = (int64_t)blockIdx.x * FOURS + four, row = at / wide, col = at % wide * 4;
  const int have = row < g.M ? (g.N - col >= 4 ? 4 : (int)(g.N - col)) : 0;
  double sum[8] = {0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
  if (have) {
    const float* p = g.partial + row * 2 * g.N + col;
    const int64_t step = g.M * 2 * g.N;
    for (int s = part; s < g.slices; s += 4 * PARTS) {
      float t[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (s + PARTS * u < g.slices) {
          float first[4], second[4];
          load4(p + (s + PARTS * u) * step, have, first);
          load4(p + (s + PARTS * u) * step + g.N, have, second);
#pragma unroll
          for (int i = 0; i < 4; ++i) { t[u][i] = first[i]; t[u][4 + i] = second[i]; }
        }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (s + PARTS * u < g.slices) {
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[i] += t[u][i];
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[part][four][i] = sum[i];
  __syncthreads();
  if (part || !have) return;
#pragma unroll
  for (int k = 1; k < PARTS; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += sums[k][four][i];
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double both = sum[i] + sum[4 + i];
    v[i] = (float)(fabs(both) < __builtin_huge_val() ? both : sum[i]);
  }
  store4((T*)g.c + row * g.ldc + col, have, v);
}

template <typename T> void join(const Gemm& g) {
  const int64_t fours = g.M * ((g.N + 31) / 32 * 8);
  if (g.slices <= 8) hipLaunchKernelGGL((gemm_join_kernel<T, 1>), dim3((uint32_t)((fours + 255) / 256)), dim3(256), 0, g.stream, g);
  else hipLaunchKernelGGL((gemm_join_kernel<T, 8>), dim3((uint32_t)((fours + 31) / 32)), dim3(256), 0, g.stream, g);
}

// ---------------------------------------------------------------------------------------
// Many rows (forward and input gradient of whole graphs or batches). W is laid out first, once a call: zero-padded chunks in the
// order in which a workgroup's stages read them (split into its three pieces where T is float), so that a stage is one
// contiguous copy into LDS and the main kernel spends no instruction on W's layout or split. A's rows are not shared by
// waves -- a wave owns 32 rows and all BN columns -- so they go from memory straight to the lanes that multiply them, and an
// element is split once. The product is taken transposed, W^T's piece as the first operand: a lane then holds one row's
// columns in fours and writes them itself, without a turn through LDS.
// ---------------------------------------------------------------------------------------
template <typename T> struct Rows;                          // BK: contraction elements a stage
template <> struct Rows<float> { static constexpr int BK = 32; };
template <> struct Rows<__bf16> { static constexpr int BK = 64; };
template <> struct Rows<_Float16> { static constexpr int BK = 64; };

struct Layout {
  const void* w;
  int64_t ld, N, K;
  bool along;
  int64_t ktiles, ntiles;
  char* image;              // [ntiles][ktiles][PLANES][BK / 8][BN] chunks
};

template <typename T, int BN>
__global__ __launch_bounds__(256) void lay_out_kernel(const Layout g) {
  constexpr int CH = Rows<T>::BK / 8, PL = Unit<T>::PLANES;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;         // chunk (column tile, stage, chunk, column)
  const int64_t n = at % BN, c = at / BN % CH, kt = at / BN / CH % g.ktiles, nt = at / BN / CH / g.ktiles;
  if (nt >= g.ntiles) return;
  const int64_t col = nt * BN + n, k = (kt * CH + c) * 8;
  const T* w = (const T*)g.w + (g.along ? col * g.ld + k : k * g.ld + col);
  const int64_t step = g.along ? 1 : g.ld;
  T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = col < g.N && k + i < g.K ? w[i * step] : (T)0.f;
  u4* out = reinterpret_cast<u4*>(g.image) + ((nt * g.ktiles + kt) * PL * CH + c) * BN + n;
  if constexpr (PL == 3) {
    float f[8];
    u4 h[3];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
    split8(f, h);
#pragma unroll
    for (int p = 0; p < 3; ++p) out[(int64_t)p * CH * BN] = h[p];
  } else {
    union { T e[8]; u4 u; } r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.e[i] = v[i];
    *out = r.u;
  }
}

// 8 consecutive elements of a row, `left` of which exist; `over`: a load may run over the row's end
template <typename T> struct Eight { u4 q[8 / Unit<T>::W]; };
template <typename T> __device__ __forceinline__ void load8(const T* p, int64_t left, bool over, Eight<T>& v) {
  constexpr int W = Unit<T>::W;
  if (left >= 8) {
#pragma unroll
    for (int i = 0; i < 8 / W; ++i) v.q[i] = load16(p + i * W);
  } else if (left > 0 && over) {
#pragma unroll
    for (int i = 0; i < 8 / W; ++i) v.q[i] = load_masked(p + i * W, left - i * W);
  } else {
#pragma unroll
    for (int i = 0; i < 8 / W; ++i) v.q[i] = load_some(p + i * W, left - i * W);
  }
}

// A lane of a transposed tile holds its row's columns 8 q + 4 half .. + 3, q = 0..3. Memory takes them as 16 bytes a lane:
// fp32 fours as they are; two fours of 16-bit values after the halves of the wave have exchanged them, so that a lane of the
// lower half has columns 16 u .. + 7 and its partner columns 16 u + 8 .. + 15 (u = 0, 1).
template <typename T> struct Out16;
template <typename T> struct Out : Out16<T> {};
template <> struct Out<float> {
  static constexpr int PIECES = 4, WIDE = 4;                  // 16-byte pieces of a tile's row a lane, elements in one
  static __device__ __forceinline__ int column(int piece, int half) { return 8 * piece + 4 * half; }
  static __device__ __forceinline__ void pack(const float (&v)[16], u4 (&out)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) out[q][i] = __float_as_uint(v[4 * q + i]);
  }
  static __device__ __forceinline__ void unpack(const u4 (&in)[4], float (&v)[16]) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * q + i] = __uint_as_float(in[q][i]);
  }
};
template <typename T> struct Out16 {
  static constexpr int PIECES = 2, WIDE = 8;
  static __device__ __forceinline__ int column(int piece, int half) { return 16 * piece + 8 * half; }
  static __device__ __forceinline__ void exchange(uint32_t& a, uint32_t& b) {       // a's upper half and b's lower half
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const u2 r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  }
  static __device__ __forceinline__ void pack(const float (&v)[16], u4 (&out)[2]) {
    union { T e[16]; uint32_t u[8]; } r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r.e[i] = (T)v[i];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int d = 0; d < 2; ++d) exchange(r.u[4 * u + d], r.u[4 * u + 2 + d]);
#pragma unroll
      for (int d = 0; d < 2; ++d) { out[u][d] = r.u[4 * u + d]; out[u][2 + d] = r.u[4 * u + 2 + d]; }
    }
  }
  static __device__ __forceinline__ void unpack(const u4 (&in)[2], float (&v)[16]) {
    union { T e[16]; uint32_t u[8]; } r;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        r.u[4 * u + d] = in[u][d];
        r.u[4 * u + 2 + d] = in[u][2 + d];
        exchange(r.u[4 * u + d], r.u[4 * u + 2 + d]);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = (float)r.e[i];
  }
};

// the first `have` elements of a 16-byte piece at p
template <typename T> __device__ __forceinline__ void store_piece(T* p, int have, u4 v) {
  constexpr int W = Unit<T>::W;
  if (have >= W) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<u4_at4*>(p) = v;
    else *reinterpret_cast<u4_at2*>(p) = v;
  } else {
    union { u4 u; T e[W]; } r;
    r.u = v;
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < have) p[i] = r.e[i];
  }
}
template <typename T> __device__ __forceinline__ u4 load_piece(const T* p, int have) {
  return have >= Unit<T>::W ? load16(p) : load_some(p, have);
}

// A lane's columns of its row: saved slope data, activation, residual, one rounding. `res` holds the residual's pieces.
template <typename T, int TN, int ACT>
__device__ __forceinline__ void rows_out(const Gemm& g, const f16v (&acc)[TN], const u4 (&res)[TN][Out<T>::PIECES], int64_t row, int64_t col0, int half, bool in) {
  constexpr int PIECES = Out<T>::PIECES, WIDE = Out<T>::WIDE;
  T* const c = (T*)g.c + row * g.ldc;
  each<0, TN>([&](auto j) __attribute__((always_inline)) {
    const int64_t base = col0 + j * 32, left = in ? g.N - base : 0;
    auto have = [&](int piece) __attribute__((always_inline)) {
      const int64_t n = left - Out<T>::column(piece, half);
      return n >= WIDE ? WIDE : n > 0 ? (int)n : 0;
    };
    float v[16];
    u4 out[PIECES];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = acc[j][e];
    if (ACT != ACT_NONE && g.save) {
      if constexpr (ACT == ACT_RELU) {
        uint32_t bits = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int n = 8 * (e / 4) + 4 * half + e % 4;
          bits |= (n < left && !(v[e] <= 0.f) ? 1u : 0u) << n;
        }
        bits |= __shfl_xor(bits, 32);
        if (half == 0 && left > 0) ((uint32_t*)g.save)[row * g.ld_save + (col0 / 32 + j)] = bits;
      } else {
        u4 wide[4];
        Out<float>::pack(v, wide);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t n = left - Out<float>::column(q, half);
          store_piece((float*)g.save + row * g.ld_save + base + Out<float>::column(q, half), n >= 4 ? 4 : n > 0 ? (int)n : 0, wide[q]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = act_of<T>(ACT, v[e]);
    if (g.residual) {
      float r[16];
      Out<T>::unpack(res[j], r);
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] += r[e];
    }
    Out<T>::pack(v, out);
#pragma unroll
    for (int q = 0; q < PIECES; ++q) store_piece(c + base + Out<T>::column(q, half), have(q), out[q]);
  });
}

// What a wave of rows_kernel does for a block of rows: TN column tiles of 32 rows.
template <typename T, int TN> struct Wave {
  static constexpr int BK = Rows<T>::BK, CH = BK / 8, PL = Unit<T>::PLANES, BN = TN * 32, S = BK / 16;
  static constexpr int STAGE = PL * CH * BN * 16;             // bytes of a stage of W's image
  f16v acc[TN];
  Eight<T> a[S];                                              // this lane's part of its row: 8 elements of each 16

  // sums start at the bias: element e of a lane is column 8 (e / 4) + 4 half + e % 4 of the tile, row lane % 32
  static __device__ __forceinline__ f16v bias_of(const Gemm& g, int64_t col0, int half) {
    f16v t;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      float b[4] = {0.f, 0.f, 0.f, 0.f};
      const int64_t col = col0 + 2 * e + 4 * half;
      if (g.bias) load4((const T*)g.bias + col, g.N - col >= 4 ? 4 : (g.N > col ? (int)(g.N - col) : 0), b);
#pragma unroll
      for (int i = 0; i < 4; ++i) t[e + i] = b[i];
    }
    return t;
  }
  __device__ __forceinline__ void begin(const Gemm& g, int64_t col0, int half) {
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[j] = bias_of(g, col0 + j * 32, half);
  }

  // stage kt of the row whose lane part begins at p
  static __device__ __forceinline__ void fetch(const T* p, int64_t K, int kt, int half, bool over, Eight<T> (&to)[S]) {
    const T* q = p + (int64_t)kt * BK;
    const int64_t left = K - (int64_t)kt * BK;
    if (left >= BK) {
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < 8 / Unit<T>::W; ++i) to[s].q[i] = load16(q + 16 * s + i * Unit<T>::W);
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s) load8(q + 16 * s, left - 8 * half - 16 * s, over, to[s]);
    }
  }

  // Multiplies R blocks by the same stage of W. `from` points at this lane's chunks: stage + ((lane / 32) BN + lane % 32)
  // chunks. The next tile's chunks are read before a tile's products are issued.
  template <int R> static __device__ __forceinline__ void multiply(Wave (&v)[R], const char* from) {
    u4 y[2][PL];
    auto read = [&](int s, int j, u4 (&to)[PL]) __attribute__((always_inline)) {
#pragma unroll
      for (int p = 0; p < PL; ++p) to[p] = *reinterpret_cast<const u4*>(from + ((p * CH + 2 * s) * BN + j * 32) * 16);
    };
    read(0, 0, y[0]);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      u4 x[R][PL];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if constexpr (PL == 3) {
          float w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = __uint_as_float(v[r].a[s].q[i / 4][i % 4]);
          split8(w, x[r]);
        } else {
          x[r][0] = v[r].a[s].q[0];
        }
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int t = (s * TN + j) & 1;
        if (j + 1 < TN) read(s, j + 1, y[t ^ 1]);
        else if (s + 1 < S) read(s + 1, 0, y[t ^ 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if constexpr (PL == 3) {                             // small products first
            v[r].acc[j] = mfma(y[t][0], x[r][2], v[r].acc[j], T());
            v[r].acc[j] = mfma(y[t][2], x[r][0], v[r].acc[j], T());
            v[r].acc[j] = mfma(y[t][1], x[r][1], v[r].acc[j], T());
            v[r].acc[j] = mfma(y[t][0], x[r][1], v[r].acc[j], T());
            v[r].acc[j] = mfma(y[t][1], x[r][0], v[r].acc[j], T());
          }
          v[r].acc[j] = mfma(y[t][0], x[r][0], v[r].acc[j], T());
        }
      }
    }
  }

  __device__ __forceinline__ void finish(const Gemm& g, int64_t row, int64_t col0, int half) {
    const bool in = row < g.M;
    if constexpr (PL == 3) {
      float seen = 0.f;
      each<0, TN>([&](auto j) __attribute__((always_inline)) { seen += unsound(acc[j]); });
      if (__ballot(!(seen == 0.f))) {
        const int64_t mine = in ? row : g.M - 1;
        each<0, TN>([&](auto j) __attribute__((always_inline)) {
          const int64_t n = col0 + j * 32 + (threadIdx.x & 31), ni = n < g.N ? n : g.N - 1;
          again(acc[j], bias_of(g, col0 + j * 32, half), (const T*)g.b + (g.b_along ? ni * g.ldb : ni), g.b_along ? 1 : g.ldb, (const T*)g.a + mine * g.lda, 1, 0, g.K);
        });
      }
    }
    // all of the residual is on its way before the first store: the compiler may not move a load over one
    u4 res[TN][Out<T>::PIECES];
    if (g.residual) {
      const T* r = (const T*)g.residual + row * g.ld_residual + col0;
      each<0, TN>([&](auto j) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < Out<T>::PIECES; ++q) {
          const int64_t col = j * 32 + Out<T>::column(q, half), left = in ? g.N - col0 - col : 0;
          res[j][q] = load_piece(r + col, left >= Out<T>::WIDE ? Out<T>::WIDE : left > 0 ? (int)left : 0);
        }
      });
    }
    switch (g.act) {
      case ACT_RELU: rows_out<T, TN, ACT_RELU>(g, acc, res, row, col0, half, in); break;
      case ACT_GELU: rows_out<T, TN, ACT_GELU>(g, acc, res, row, col0, half, in); break;
      case ACT_SILU: rows_out<T, TN, ACT_SILU>(g, acc, res, row, col0, half, in); break;
      default: rows_out<T, TN, ACT_NONE>(g, acc, res, row, col0, half, in);
    }
  }
};

typedef __attribute__((address_space(3))) void* lds_ptr;

// fp32 232965 x 602 x 256 393 to 436 us, 165 to 183 TFLOP/s of fp32 products (990 to 1100 of bf16 ones), bound by the matrix cores,
// whose clock follows the data (357 us with x all zero, 393 half zero, 436 with none); bf16 65536 x 1024 x
// 512 87 us, 790 TFLOP/s, 8192 x 1024 x 4096 103, 665, bound by LDS reads and the barrier of each stage; 2449029 x 256 x 256 with
// a residual 1073 us, 3.5 TB/s: its rows are written in 32-byte pieces.
// With 128 columns fp32 takes all 168 registers of three waves a SIMD; its epilogue keeps up to 48 bytes a lane in scratch where the
// residual's pieces wait, the loop over stages none.
// W's stages go round two buffers in LDS, copied there by the memory unit itself while the stage before is multiplied; each
// buffer is an array of its own, so that the compiler sees that a copy into one does not touch the reads of the other.
template <typename T, int TN, int WAVES, int R>
__global__ __launch_bounds__(WAVES * 64, R == 2 ? 2 : TN == 4 ? 3 : 4) void rows_kernel(const Gemm g, const char* image, int ktiles) {
  using V = Wave<T, TN>;
  constexpr int STAGE = V::STAGE, PIECES = STAGE / 1024, PER = (PIECES + WAVES - 1) / WAVES;
  __shared__ __attribute__((aligned(16))) char even[STAGE];
  __shared__ __attribute__((aligned(16))) char odd[STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  // consecutive workgroups go round the 8 XCDs: the column tiles of a row block stay on one of them, one after the other
  const int64_t ntiles = (g.N + V::BN - 1) / V::BN, turn = blockIdx.x / 8;
  const int64_t nt = turn % ntiles, group = turn / ntiles * 8 + blockIdx.x % 8;
  const int64_t row = (group * WAVES + wave) * 32 * R + (lane & 31);
  if (group * WAVES * 32 * R >= g.M) return;
  const char* w = image + nt * ktiles * STAGE + lane * 16;
  const T* p[R];
  bool over[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t at = row + 32 * r;
    p[r] = (const T*)g.a + (at < g.M ? at : g.M - 1) * g.lda + 8 * half;
    over[r] = at + 1 < g.M && g.lda >= 8;
  }
  auto send = [&](int kt, char* to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int piece = i * WAVES + wave;
      piece = PIECES % WAVES == 0 || piece < PIECES ? piece : PIECES - 1;
      __builtin_amdgcn_global_load_lds((const void*)(w + (int64_t)kt * STAGE + piece * 1024), (lds_ptr)(to + piece * 1024), 16, 0, 0);
    }
  };
  // everything on its way has arrived, and every wave is done with what it read
  auto meet = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  V v[R];
  Eight<T> next[R][V::S];
  send(0, even);
#pragma unroll
  for (int r = 0; r < R; ++r) V::fetch(p[r], g.K, 0, half, over[r], v[r].a);
  each<0, R>([&](auto r) __attribute__((always_inline)) { v[r].begin(g, nt * V::BN, half); });
  meet();
  auto step = [&](int kt, const char* from, char* to) __attribute__((always_inline)) {
    if (kt + 1 < ktiles) {
      send(kt + 1, to);
#pragma unroll
      for (int r = 0; r < R; ++r) V::fetch(p[r], g.K, kt + 1, half, over[r], next[r]);
    }
    V::multiply(v, from + ((lane >> 5) * V::BN + (lane & 31)) * 16);
    meet();
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int s = 0; s < V::S; ++s) v[r].a[s] = next[r][s];
  };
  for (int kt = 0; kt < ktiles; kt += 2) {
    step(kt, even, odd);
    if (kt + 1 < ktiles) step(kt + 1, odd, even);
  }
  each<0, R>([&](auto r) __attribute__((always_inline)) { v[r].finish(g, row + 32 * r, nt * V::BN, half); });
}

// Columns a wave takes: all of a narrow output, else 128.
inline int rows_bn(int64_t N) { return N <= 32 ? 32 : N <= 64 ? 64 : 128; }

// Bytes of W's image.
template <typename T> int64_t rows_image(const Gemm& g) {
  const int64_t bn = rows_bn(g.N), bk = Rows<T>::BK;
  return ((g.N + bn - 1) / bn) * bn * ((g.K + bk - 1) / bk) * bk * Unit<T>::PLANES * 2;
}
// Whether a product runs on rows_kernel: with two workgroups of 128 rows for each compute unit, or where the contraction is so
// short that cutting it into slices would not pay for what that costs. rows_kernel against tiles: bf16 4096 x 1024 x 1024
// 25.6, 29.6 us; 8192 x 256 x 256 9.7, 19.9; 2048 x 1024 x 1024 23.7, 24.2; fp32 2048 x 256 x 256 16.1, 21.8; 65536 x 64 x 16
// 8.0, 9.4; but 16384 x 1433 x 16 46.9, 37.5, and bf16 1024 x 4096 x 4096 85.0, 58.2. A contraction of one or two stages leaves little
// to win and W's layout is a launch of its own: fp32 2708 x 16 x 1433 14.3, 11.0; 32768 x 64 x 128 12.4, 13.2; 60000 x 32 x 128
// 14.5, 19.4.
inline bool rows_fit(const Gemm& g) {
  const int64_t bn = rows_bn(g.N), groups = (g.M + 127) / 128 * ((g.N + bn - 1) / bn);
  return g.a_along && g.K > 0 && (groups >= 512 || (groups >= (g.K > 64 ? 32 : 384) && g.K <= 8 * groups)) && groups < (1 << 23)
      && g.K * g.N < (1LL << 34);                                      // launches stay below 2^32 lanes
}

// A wave of 16-bit values takes R = 2 row blocks against each chunk of W it reads: with one, a matrix instruction's 32 cycles
// take one 16-byte read a lane from LDS, which four such waves just saturate. That needs two workgroups for each compute unit
// (8192 x 4096 x 1024, one each: 106 us against 95 with R = 1) and a contraction long enough to hide the second block's
// epilogue. bf16, R = 1 against R = 2: 65536 x 1024 x 512 104, 87 us; 16384 x 1024 x 1024 59, 48; 8192 x 1024 x 4096 118, 103;
// 2449029 x 256 x 256 775, 715, but with a residual and saved bits 1128, 1171; 232965 x 41 x 256 38, 41. fp32 has 6 products
// to a chunk's three reads and stays at R = 1. (Keeping all of a narrow W in LDS and walking over the rows was slower:
// 131072 x 256 x 128 bf16 30 us, this 22.)
template <typename T, int TN>
int rows_launch(const Gemm& g, char* image) {
  constexpr int BN = TN * 32, BK = Rows<T>::BK, CH = BK / 8, STAGE = Unit<T>::PLANES * CH * BN * 16;
  const int64_t ktiles = (g.K + BK - 1) / BK, ntiles = (g.N + BN - 1) / BN;
  const Layout l{g.b, g.ldb, g.N, g.K, g.b_along, ktiles, ntiles, image};
  const int64_t chunks = ntiles * ktiles * CH * BN;
  hipLaunchKernelGGL((lay_out_kernel<T, BN>), dim3((uint32_t)((chunks + 255) / 256)), dim3(256), 0, g.stream, l);
  DGNN_LAUNCHED();
  const int64_t blocks = (g.M + 31) / 32;
  constexpr int WAVES = 4;
  const int64_t groups = (blocks + WAVES - 1) / WAVES, pairs = (groups + 1) / 2;
  if (sizeof(T) == 2 && TN == 4 && pairs * ntiles >= 512 && (g.K >= 512 || (g.K >= 128 && !g.residual && !g.save))) {
    if constexpr (sizeof(T) == 2 && TN == 4)
      hipLaunchKernelGGL((rows_kernel<T, TN, WAVES, 2>), dim3((uint32_t)((pairs + 7) / 8 * 8 * ntiles)), dim3(WAVES * 64), 0, g.stream, g, image, (int)ktiles);
  } else {
    hipLaunchKernelGGL((rows_kernel<T, TN, WAVES, 1>), dim3((uint32_t)((groups + 7) / 8 * 8 * ntiles)), dim3(WAVES * 64), 0, g.stream, g, image, (int)ktiles);
  }
  DGNN_LAUNCHED();
  return DGNN_OK;
}

// ---------------------------------------------------------------------------------------
// x^T p of fp32 matrices, the weight gradient over many rows: both operands keep the contraction across rows, and it is long
// (every node) while the output is small. A wave owns 32 columns of x and all the workgroup's columns of p; x goes from memory
// straight to the lanes (8 rows' values of a column each), p is turned and split once a workgroup on its way to LDS. The rows
// are cut into slices for 3 workgroups a compute unit, the tiles of a slice stay on one XCD, and a join adds the slices. Bound by
// x's and p's bytes: 232965 x 256 x 41 86 us with its join, 277 MB, 3.2 TB/s.
// (16-bit values would come 2 or 4 bytes a load here; the tiles of gemm_kernel load 16, which is worth more.)
// ---------------------------------------------------------------------------------------
template <int BN> struct Turn {                               // BN columns of 32 rows by 256 lanes: 8 rows of 2 columns a lane
  static constexpr int BK = 32, CH = BK / 8, GROUPS = BN / 2, UNITS = GROUPS * CH, STAGE = 3 * CH * BN * 16;
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  typedef uint32_t u2_at4 __attribute__((ext_vector_type(2), aligned(4)));
  u2 r[8];

  static __device__ __forceinline__ int place(int col) { return col ^ ((col >> 4) & 7); }

  uint32_t off;
  int col;
  bool pair;

  // `cols`: p's columns. A lane's distance from its row's start is 32 bits, the
  // rows' starts are the workgroup's: addresses cost scalar registers. A lane past the columns reads the first ones (its sums
  // are not kept); a pair that ends past them reads on into the next row, or is two loads where none follows
  __device__ __forceinline__ void begin(int64_t ld, int64_t cols, int tid) {
    col = tid % GROUPS * 2;
    col = col < cols ? col : 0;
    pair = col + 1 < cols;
    off = (uint32_t)((8 * (tid / GROUPS) * ld + col) * 4);
  }

  __device__ __forceinline__ void fetch(const float* p, int64_t ld, int64_t k0, int64_t kend, int64_t kall, int tid) {
    if (UNITS < 256 && tid >= UNITS) return;
    if (k0 + BK <= kend && k0 + BK < kall && ld >= 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = *reinterpret_cast<const u2_at4*>(reinterpret_cast<const char*>(p + (k0 + i) * ld) + off);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(p + (k0 + i) * ld) + off);
        r[i] = u2{0, 0};
        if (k0 + 8 * (tid / GROUPS) + i < kend) {
          r[i][0] = q[0];
          if (pair) r[i][1] = q[1];
        }
      }
    }
  }

  __device__ __forceinline__ void store(char* lds, int tid) const {
    if (UNITS < 256 && tid >= UNITS) return;
    char* const at = lds + (tid / GROUPS) * BN * 16;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      char* const to = at + place(tid % GROUPS * 2 + c) * 16;
      float v[8];
      u4 h[3];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i][c]);
      split8(v, h);
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<u4*>(to + p * CH * BN * 16) = h[p];
    }
  }
};

template <int TN>
__global__ __launch_bounds__(256, 3) void columns_kernel(const Gemm g) {
  constexpr int BN = TN * 32, BK = 32, S = BK / 16, CH = BK / 8, BM = 128;
  using B = Turn<BN>;
  __shared__ __attribute__((aligned(16))) char even[B::STAGE];
  __shared__ __attribute__((aligned(16))) char odd[B::STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
  const int64_t tiles = (g.M + BM - 1) / BM;
  int64_t tile = blockIdx.x % tiles, slice = blockIdx.x / tiles;
  if (g.slices >= 8) {                                         // consecutive workgroups go round the 8 XCDs
    tile = blockIdx.x / 8 % tiles;
    slice = blockIdx.x / 8 / tiles * 8 + blockIdx.x % 8;
    if (slice >= g.slices) return;
  }
  const int64_t row0 = tile * BM + wave * 32;                  // of the output, whose columns are one tile
  const int64_t kbeg = slice * g.slice_k, kend = kbeg + g.slice_k < g.K ? kbeg + g.slice_k : g.K;
  const float* const x = (const float*)g.a;
  const float* const p = (const float*)g.b;
  const int64_t mine = row0 + (lane & 31);                     // a lane's column of x; past the end the last one stands in
  const uint32_t off = (uint32_t)(((mine < g.M ? mine : g.M - 1) + 8 * half * g.lda) * 4);

  f16v acc[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) acc[j] = f16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  float cur[S][8], next[S][8];                                 // a lane's column of 8 rows of each 16
  auto fetch_x = [&](int64_t k0, float (&to)[S][8]) __attribute__((always_inline)) {
    const bool whole = k0 + BK <= kend;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float* q = reinterpret_cast<const float*>(reinterpret_cast<const char*>(x + (k0 + 16 * s + i) * g.lda) + off);
        if (whole) to[s][i] = *q;
        else to[s][i] = k0 + 16 * s + 8 * half + i < kend ? *q : 0.f;
      }
  };
  B b;
  b.begin(g.ldb, g.N, tid);
  if (kbeg < kend) {
    b.fetch(p, g.ldb, kbeg, kend, g.K, tid);
    fetch_x(kbeg, cur);
    b.store(even, tid);
  }
  __syncthreads();
  auto step = [&](int64_t k, const char* from, char* to) __attribute__((always_inline)) {
    const bool more = k + BK < kend;
    if (more) {
      b.fetch(p, g.ldb, k + BK, kend, g.K, tid);
      fetch_x(k + BK, next);
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      u4 f[3];
      split8(cur[s], f);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        u4 y[3];
#pragma unroll
        for (int q = 0; q < 3; ++q)
          y[q] = *reinterpret_cast<const u4*>(from + ((q * CH + 2 * s + half) * BN + B::place(j * 32 + (lane & 31))) * 16);
        acc[j] = mfma(f[2], y[0], acc[j], float());            // small products first
        acc[j] = mfma(f[0], y[2], acc[j], float());
        acc[j] = mfma(f[1], y[1], acc[j], float());
        acc[j] = mfma(f[1], y[0], acc[j], float());
        acc[j] = mfma(f[0], y[1], acc[j], float());
        acc[j] = mfma(f[0], y[0], acc[j], float());
      }
    }
    if (more) b.store(to, tid);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) cur[s][i] = next[s][i];
  };
  for (int64_t k = kbeg; k < kend; k += 2 * BK) {
    step(k, even, odd);
    if (k + BK < kend) step(k + BK, odd, even);
  }

  each<0, TN>([&](auto j) __attribute__((always_inline)) {
    const int64_t col = j * 32 + (lane & 31);
    if (__ballot(col < g.N && !(unsound(acc[j]) == 0.f)))
      again(acc[j], f16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0}, x + (mine < g.M ? mine : g.M - 1), g.lda, p + (col < g.N ? col : g.N - 1), g.ldb, kbeg, kend);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t row = row0 + 8 * (e / 4) + 4 * half + e % 4;
      if (row < g.M && col < g.N) {
        if (g.slices > 1) g.partial[(slice * g.M + row) * g.N + col] = acc[j][e];
        else ((float*)g.c)[row * g.ldc + col] = acc[j][e];
      }
    }
  });
}

// From 65536 rows up for outputs of one column tile, while a lane's distance from its row fits 32 bits. Against tiles: x^T p of
// 256 x 41 from 65536 rows 39.4, 47.4 us; 64 x 64 from 262144 57.8, 70.5. Wider outputs share the turned x among 256 columns
// there: 256 x 256 from 65536 79.2, 70.7; 602 x 256 from 232965 521, 511.
template <typename T> bool columns_fit(const Gemm& g) {
  return sizeof(T) == 4 && !g.a_along && g.K >= 65536 && g.N <= 128 && (8 * g.lda + g.M) * 4 <= 0xffffffffLL && 32 * g.ldb * 4 <= 0xffffffffLL;
}

inline int64_t columns_tiles(const Gemm& g) { return (g.M + 127) / 128; }

// Slices for 3 workgroups a compute unit, as many for each XCD, 256 rows at least, and no more partial sums than a quarter
// of what the operands weigh.
inline void columns_cut(Gemm& g) {
  const int64_t tiles = columns_tiles(g), most = (g.K + 255) / 256, heavy = g.K * (g.M + g.N) / (4 * g.M * g.N);
  int64_t want = 768 / (tiles < 768 ? tiles : 768);
  if (want > most) want = most;
  if (want > heavy) want = heavy;
  if (want >= 8) want = want / 8 * 8;
  if (want < 1) want = 1;
  g.slice_k = ((g.K + want - 1) / want + 31) / 32 * 32;
  g.slices = (int)((g.K + g.slice_k - 1) / g.slice_k);
}

inline int columns_launch(const Gemm& g) {
  const int64_t blocks = (g.slices >= 8 ? ((int64_t)g.slices + 7) / 8 * 8 : g.slices) * columns_tiles(g);
  const dim3 grid((uint32_t)blocks);
  switch (rows_bn(g.N)) {
    case 32: hipLaunchKernelGGL((columns_kernel<1>), grid, dim3(256), 0, g.stream, g); break;
    case 64: hipLaunchKernelGGL((columns_kernel<2>), grid, dim3(256), 0, g.stream, g); break;
    default: hipLaunchKernelGGL((columns_kernel<4>), grid, dim3(256), 0, g.stream, g);
  }
  DGNN_LAUNCHED();
  if (g.slices > 1) {
    join<float>(g);
    DGNN_LAUNCHED();
  }
  return DGNN_OK;
}

// ---------------------------------------------------------------------------------------
// A handful of rows: W's bytes are all there is, each is used once a row, so plain fused multiply-adds in fp32 keep up, in one
// launch while W is small. thin_across: W[k][n] with n contiguous; LANES lanes take 16 bytes each of a row of W, the others and
// the 16 waves further rows, all loads of a lane are on their way together, and the rows' sums meet by exchanges in the wave and
// through LDS. LANES is as small as it takes to have a workgroup for every compute unit; neighbouring column blocks, which share
// cache lines, run on one XCD. thin_along: W[n][k] with the contraction contiguous; a wave takes an output and all its lanes the
// contraction (four outputs a wave: 1 x 4096 x 4096 bf16 7.9 us against 6.2).
// One row: fp32 602 x 256 4.6 us, which is a launch and one trip to memory; bf16 4096 x 4096 9.4 us with its join, 3.6 TB/s.
// ---------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void thin_out(const Gemm& g, int64_t row, int64_t col, float t) {
  if (g.save && g.act > ACT_RELU) ((float*)g.save)[row * g.ld_save + col] = t;
  t = act_of<T>(g.act, t);
  if (g.residual) t += (float)((const T*)g.residual)[row * g.ld_residual + col];
  ((T*)g.c)[row * g.ldc + col] = (T)t;
}

template <typename T> __device__ __forceinline__ void widen16(u4 v, float (&out)[Unit<T>::W]) {
  union { u4 u; T e[Unit<T>::W]; } r;
  r.u = v;
#pragma unroll
  for (int i = 0; i < Unit<T>::W; ++i) out[i] = (float)r.e[i];
}

template <typename T, int ROWS, int WAVES, int U, int LEAST, int MOST>      // LEAST <= lanes <= MOST
__global__ __launch_bounds__(WAVES * 64) void thin_across_kernel(const Gemm g, int lanes) {
  constexpr int W = Unit<T>::W, WIDE = MOST * W, STAGED = 64 / LEAST * WAVES * U;
  __shared__ __attribute__((aligned(16))) float room[ROWS * (STAGED > WAVES * WIDE ? STAGED : WAVES * WIDE)];
  const int64_t kbeg = (int64_t)blockIdx.y * g.slice_k, kend = kbeg + g.slice_k < g.K ? kbeg + g.slice_k : g.K;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t each_xcd = (gridDim.x + 7) / 8, block = (int64_t)(blockIdx.x % 8) * each_xcd + blockIdx.x / 8;
  const int64_t col = (block * lanes + lane % lanes) * W, left = g.N - col;
  const int per = 64 / lanes * WAVES, mine = wave * (64 / lanes) + lane / lanes;      // rows of W a pass, this lane's among them
  const T* w = (const T*)g.b + col;
  const T* x = (const T*)g.a;
  float acc[ROWS][W];
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
#pragma unroll
    for (int i = 0; i < W; ++i) acc[m][i] = 0.f;
  for (int64_t base = kbeg; base < kend; base += (int64_t)per * U) {
    u4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = base + u * per + mine;
      v[u] = u4{0, 0, 0, 0};
      if (k < kend && left > 0) v[u] = left >= W ? load16(w + k * g.ldb) : load_some(w + k * g.ldb, left);
    }
    __syncthreads();
    for (int at = threadIdx.x; at < per * U * ROWS; at += WAVES * 64) {          // x's part, widened, the rows of a k side by side
      const int k = at % (per * U), m = at / (per * U);
      room[k * ROWS + m] = m < g.M && base + k < kend ? (float)x[m * g.lda + base + k] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (base + u * per + mine >= kend) continue;
      float f[W];
      widen16<T>(v[u], f);
      const float* s = room + (u * per + mine) * ROWS;
#pragma unroll
      for (int m = 0; m < ROWS; ++m) {
        const float sm = s[m];
#pragma unroll
        for (int i = 0; i < W; ++i) acc[m][i] = fmaf(sm, f[i], acc[m][i]);
      }
    }
  }
  __syncthreads();
  for (int d = lanes; d < 64; d <<= 1)
#pragma unroll
    for (int m = 0; m < ROWS; ++m)
#pragma unroll
      for (int i = 0; i < W; ++i) acc[m][i] += __shfl_xor(acc[m][i], d);
  if (lane < lanes)
#pragma unroll
    for (int m = 0; m < ROWS; ++m)
#pragma unroll
      for (int i = 0; i < W; ++i) room[(wave * ROWS + m) * WIDE + lane * W + i] = acc[m][i];
  __syncthreads();
  const int wide = lanes * W;
  for (int at = threadIdx.x; at < (ROWS * wide + 63) / 64 * 64; at += WAVES * 64) {      // whole waves: relu's bits are gathered below
    const int m = at / wide, c = at % wide;
    const int64_t n = block * wide + c;
    const bool in = m < ROWS && m < g.M && n < g.N;
    float t = 0.f;
    if (in) {
#pragma unroll
      for (int k = 0; k < WAVES; ++k) t += room[(k * ROWS + m) * WIDE + c];
      if (g.slices > 1) g.partial[((int64_t)blockIdx.y * g.M + m) * g.N + n] = t;
      else if (g.bias) t += (float)((const T*)g.bias)[n];
    }
    if (g.slices > 1) continue;
    if (g.save && g.act == ACT_RELU) {                         // a byte for 8 columns, up to the end of the row's last word
      const uint64_t bits = __ballot(in && !(t <= 0.f));
      if ((c & 7) == 0 && m < ROWS && m < g.M && n < (g.N + 31) / 32 * 32)
        ((uint8_t*)((uint32_t*)g.save + m * g.ld_save))[n / 8] = (uint8_t)(bits >> (lane & 56));
    }
    if (in) thin_out<T>(g, m, n, t);
  }
}

template <typename T, int ROWS>
__global__ __launch_bounds__(256) void thin_along_kernel(const Gemm g) {
  constexpr int W = Unit<T>::W;
  const int lane = threadIdx.x & 63;
  const int64_t col = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (col >= g.N) return;
  const T* const w = (const T*)g.b + col * g.ldb;
  float acc[ROWS];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) acc[m] = 0.f;
  for (int64_t k = lane * W; k < g.K; k += 64 * W) {
    const int64_t left = g.K - k;
    u4 s[ROWS];
    const u4 v = left >= W ? load16(w + k) : load_some(w + k, left);
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      const T* p = (const T*)g.a + (m < g.M ? m : g.M - 1) * g.lda + k;
      s[m] = left >= W ? load16(p) : load_some(p, left);
    }
    float f[W];
    widen16<T>(v, f);
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      float e[W];
      widen16<T>(s[m], e);
#pragma unroll
      for (int i = 0; i < W; ++i) acc[m] = fmaf(e[i], f[i], acc[m]);
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int m = 0; m < ROWS; ++m) acc[m] += __shfl_xor(acc[m], d);
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
    if (lane == m && m < g.M) thin_out<T>(g, m, col, g.bias ? acc[m] + (float)((const T*)g.bias)[col] : acc[m]);
}

// fp32: up to 4 rows, 8 where W keeps the contraction contiguous; 16 bits: up to 2, because a tile's matrix instructions take
// 32 rows as fast as one and 16-bit values as they come. These kernels against tiles: fp32 602 x 256 with 1, 4, 6 rows 4.6,
// 8.8, 11.6 against 10.9 us, W^T with 6 rows 5.9 against 9.9; bf16 4096 x 4096 with 1, 2, 3, 6 rows 9.5, 10.3, 11.7, 15.7
// against 11.4, 11.7, 11.9, 12.3, W^T with 1, 2 rows 6.2, 7.3 against 10.7.
template <typename T> bool thin_fit(const Gemm& g) { return g.a_along && g.M <= (sizeof(T) == 2 ? 2 : g.b_along ? 8 : 4); }

// Slices of W's rows: one while W times the rows is so small that the launch is what it costs (one row: fp32 1024 x 1024 5.0 us,
// cut 7.3; 2048 x 2048 6.6, cut 7.7); else as many as give 256 workgroups, which then read 1 KiB of a row at a time (16-byte
// columns of a long matrix all lie in a few of the memory's channels: one row, bf16 4096 x 4096 12.4 us, cut 9.5; four rows,
// fp32 1024 x 2048 10.0, cut 8.4).
template <typename T> void thin_cut(Gemm& g) {
  g.slices = 1;
  g.slice_k = g.K > 0 ? g.K : 1;
  if (g.b_along || g.M * g.K * g.N * (int64_t)sizeof(T) <= (16 << 20)) return;
  const int64_t blocks = (g.N + 64 * Unit<T>::W - 1) / (64 * Unit<T>::W);
  int64_t want = 256 / (blocks < 256 ? blocks : 256);
  const int64_t most = (g.K + 31) / 32;
  want = want < 2 ? 2 : want > most ? most : want;
  g.slice_k = ((g.K + want - 1) / want + 31) / 32 * 32;
  g.slices = (int)((g.K + g.slice_k - 1) / g.slice_k);
}

template <typename T, int ROWS>
int thin_along_launch(const Gemm& g) {
  hipLaunchKernelGGL((thin_along_kernel<T, ROWS>), dim3((uint32_t)((g.N + 3) / 4)), dim3(256), 0, g.stream, g);
  DGNN_LAUNCHED();
  return DGNN_OK;
}

template <typename T, int ROWS>
int thin_launch(const Gemm& g) {
  constexpr int W = Unit<T>::W;
  if (g.b_along) {
    return thin_along_launch<T, ROWS>(g);
  } else {
    const int64_t cols = (g.N + 31) / 32 * 32;
    if (g.slices == 1) {
      int lanes = 8;
      while (lanes > 2 && (g.N + lanes * W - 1) / (lanes * W) < 256) lanes /= 2;
      const int64_t blocks = (cols + lanes * W - 1) / (lanes * W);
      hipLaunchKernelGGL((thin_across_kernel<T, ROWS, 16, 4, 2, 8>), dim3((uint32_t)((blocks + 7) / 8 * 8)), dim3(1024), 0, g.stream, g, lanes);
    } else {
      const int64_t blocks = (cols + 64 * W - 1) / (64 * W);
      hipLaunchKernelGGL((thin_across_kernel<T, ROWS, 8, 16, 64, 64>), dim3((uint32_t)((blocks + 7) / 8 * 8), (uint32_t)g.slices), dim3(512), 0, g.stream, g, 64);
      DGNN_LAUNCHED();
      join<T>(g);
    }
  }
  DGNN_LAUNCHED();
  return DGNN_OK;
}

struct Shape { int bm, bn; };

// Tile by the sides of the output: the narrowest that covers it once (against the widest: 16 x 4096 x 4096 bf16 13.9, 18.0 us;
// 2708 x 1433 x 16 fp32 13.4, 15.4; 16384 x 602 x 64 fp32 26.7, 35.9). 128 x 64 also where the contraction is one or two stages,
// which need workgroups more than shared reads (2708 x 16 x 1433 fp32 11.0, 128 x 256 23). Else 128 x 256 on 8 waves of 64 x 64.
// 16-bit products whose operands both have to be turned in registers do better with two smaller workgroups a compute unit, one
// turning while the other multiplies (4096^3 bf16 202 us, 128 x 256 215; fp32, which multiplies six times as long, 1024^3 39.1,
// 128 x 256 34.6).
template <typename T> Shape shape_of(const Gemm& g) {
  const int64_t M = g.M, N = g.N;
  if (M <= 32) return {32, 128};
  if (N <= 32) return {128, 32};
  if (N <= 64 || (g.a_along && g.K <= 64)) return {128, 64};
  if (N <= 128 || (sizeof(T) == 2 && !g.a_along)) return {128, 128};
  return {128, 256};
}

// Workgroups a compute unit holds at once, by their LDS.
inline int resident_of(Shape s) { return s.bn == 256 ? 1 : s.bn == 128 && s.bm == 128 ? 2 : 3; }

inline int64_t tiles_of(Shape s, int64_t M, int64_t N) { return ((M + s.bm - 1) / s.bm) * ((N + s.bn - 1) / s.bn); }

template <typename T, bool AA, bool BA>
int gemm_launch(const Gemm& g) {
  const Shape s = shape_of<T>(g);
  const int64_t tiles = tiles_of(s, g.M, g.N);
  const dim3 grid((uint32_t)tiles, (uint32_t)g.slices);
  switch (s.bm * 1000 + s.bn) {
    case 32128: hipLaunchKernelGGL((gemm_kernel<T, AA, BA, 32, 128, 1, 4>), grid, dim3(256), 0, g.stream, g); break;
    case 128032: hipLaunchKernelGGL((gemm_kernel<T, AA, BA, 128, 32, 4, 1>), grid, dim3(256), 0, g.stream, g); break;
    case 128064: hipLaunchKernelGGL((gemm_kernel<T, AA, BA, 128, 64, 4, 1>), grid, dim3(256), 0, g.stream, g); break;
    case 128128: hipLaunchKernelGGL((gemm_kernel<T, AA, BA, 128, 128, 2, 2>), grid, dim3(256), 0, g.stream, g); break;
    default:
      if constexpr (AA || sizeof(T) == 4) hipLaunchKernelGGL((gemm_kernel<T, AA, BA, 128, 256, 2, 4>), grid, dim3(512), 0, g.stream, g);
      break;
  }
  DGNN_LAUNCHED();
  if (g.slices > 1 && !g.pieces) {
    join<T>(g);
    DGNN_LAUNCHED();
  }
  return DGNN_OK;
}

// What gemm_kernel multiplies where b comes in two pieces.
inline Gemm both_pieces(const Gemm& g) {
  Gemm wide = g;
  wide.N = 2 * g.N;
  return wide;
}

template <typename T>
int pieces_launch(const Gemm& g) {
  const int rc = gemm_launch<T, false, false>(both_pieces(g));
  if (rc != DGNN_OK) return rc;
  const int64_t fours = g.M * ((g.N + 3) / 4);
  hipLaunchKernelGGL((pieces_join_kernel<T>), dim3((uint32_t)((fours + 31) / 32)), dim3(256), 0, g.stream, g);
  DGNN_LAUNCHED();
  return DGNN_OK;
}


template <typename T>
int gemm_typed(const Gemm& g) {
  if constexpr (sizeof(T) == 2) {
    if (g.pieces) return pieces_launch<T>(g);
  }
  if (thin_fit<T>(g)) {
    if (g.M == 1) return thin_launch<T, 1>(g);
    if (g.M == 2) return thin_launch<T, 2>(g);
    if constexpr (sizeof(T) == 4) {
      if (g.M <= 4) return thin_launch<T, 4>(g);
      return thin_along_launch<T, 8>(g);
    }
  }
  if (g.image) {
    switch (rows_bn(g.N)) {
      case 32: return rows_launch<T, 1>(g, g.image);
      case 64: return rows_launch<T, 2>(g, g.image);
      default: return rows_launch<T, 4>(g, g.image);
    }
  }
  if constexpr (sizeof(T) == 4) {
    if (columns_fit<T>(g)) return columns_launch(g);
  }
  if (!g.a_along) return gemm_launch<T, false, false>(g);
  return g.b_along ? gemm_launch<T, true, true>(g) : gemm_launch<T, true, false>(g);
}

__attribute__((visibility("hidden"))) int gemm_f32(const Gemm& g);
__attribute__((visibility("hidden"))) int gemm_bf16(const Gemm& g);
__attribute__((visibility("hidden"))) int gemm_f16(const Gemm& g);

}  // namespace dgnn
