// dgnn_linear.hip -- C entries of the layer transform y = act(x W + b) + r and its gradients (include/dgnn_train.h): the
// argument checks, how a product is cut over the chip, and the slope / column-sum kernel. The matrix products themselves are
// in dgnn_gemm.h.

#include "dgnn_gemm.h"

#include <initializer_list>

namespace {

using namespace dgnn;

// ---------------------------------------------------------------------------------------
// p = dy act'(x W + b) and the sums of p's columns. Reads dy and what the forward pass saved once and writes p once, which is
// what bounds it: 232965 x 256 fp32 gelu 152 to 171 us, 716 MB, 4.2 to 4.7 TB/s; 8192 x 4096 bf16 gelu 65 us, 268 MB, 4.1
// TB/s. A row is taken by the fewest lanes (a power of two) that cover it with 4 columns each, 64 at most, so narrow rows fill a
// wave too; a lane keeps its columns' sums over the block's rows, in 64 bits (sums over every node cancel), the block adds its
// lanes in a fixed order and a second launch adds the blocks': no atomics, the same bits every run. Of 16-bit types p is rounded to
// the type, which is what the matrix cores take: dx and dw then carry p's rounding and their own, 1.4 times the error of their own
// alone (2^-9 a value for bf16). Where dw's would be more, it takes p in two pieces (takes_pieces below), the second of which is
// written behind the row's first ones.
// ---------------------------------------------------------------------------------------
struct Slope {
  const void* dy;
  const void* save;
  void* p;
  int64_t ld_dy, ld_save, ld_p, M, N, slab;      // rows a block takes
  int64_t second;                                // elements from a value of p to what its rounding left (0: not wanted)
  double* partial;                               // gridDim.y x N, or null
  int act, lanes;
};

template <typename T> __device__ __forceinline__ float slope_of(int act, float t) {
  if (act == ACT_GELU) {
    if constexpr (sizeof(T) == 2) {
      float e, tail;
      normal_tail(t, e, tail);
      return fmaf(t, e * 0.39894228040143268f, t < 0.f ? tail : 1.f - tail);
    } else {
      return 0.5f * (1.f + erff(t * 0.70710678118654752f)) + t * expf(-0.5f * t * t) * 0.39894228040143268f;
    }
  }
  const float s = sigmoid_of<T>(t);
  return s * (1.f + t * (1.f - s));
}

template <typename T>
__global__ __launch_bounds__(256) void slope_kernel(const Slope g) {
  typedef T quad __attribute__((ext_vector_type(4), aligned(sizeof(T) == 4 ? 4 : 2)));
  typedef float wide __attribute__((ext_vector_type(4), aligned(4)));
  __shared__ double sums[256][4];
  const int lane = threadIdx.x % g.lanes, group = threadIdx.x / g.lanes, groups = 256 / g.lanes;
  const int64_t col = ((int64_t)blockIdx.x * g.lanes + lane) * 4;
  const int64_t first = (int64_t)blockIdx.y * g.slab;
  const int64_t last = first + g.slab < g.M ? first + g.slab : g.M;
  const int have = g.N - col >= 4 ? 4 : (g.N > col ? (int)(g.N - col) : 0);
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  if (have > 0) {
    constexpr int AT_ONCE = 4;                               // rows whose loads are in flight together
    for (int64_t row0 = first + group; row0 < last; row0 += AT_ONCE * groups) {
      float v[AT_ONCE][4], pre[AT_ONCE][4];
      uint32_t word[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int64_t row = row0 + k * groups;
        const bool in = row < last;
        const T* dy = (const T*)g.dy + row * g.ld_dy + col;
        if (in && (have == 4 || (g.M - 1 - row) * g.ld_dy + g.N >= col + 4)) {             // what a load runs over is the next row
          const quad q = *reinterpret_cast<const quad*>(dy);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[k][i] = i < have ? (float)q[i] : 0.f;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[k][i] = in && i < have ? (float)dy[i] : 0.f;
        }
        if (g.act == ACT_RELU) word[k] = in ? ((const uint32_t*)g.save)[row * g.ld_save + col / 32] >> (col & 31) : 0;
        else if (g.act != ACT_NONE) {
          const float* at = (const float*)g.save + row * g.ld_save + col;
          if (in && (have == 4 || (g.M - 1 - row) * g.ld_save + g.N >= col + 4)) {
            const wide q = *reinterpret_cast<const wide*>(at);
#pragma unroll
            for (int i = 0; i < 4; ++i) pre[k][i] = q[i];
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) pre[k][i] = in && i < have ? at[i] : 0.f;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int64_t row = row0 + k * groups;
        if (row >= last) break;
        if (g.act == ACT_RELU) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[k][i] = (word[k] >> i) & 1 ? v[k][i] : 0.f;
        } else if (g.act != ACT_NONE) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[k][i] *= slope_of<T>(g.act, pre[k][i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += v[k][i];
        if (g.p) {
          T* p = (T*)g.p + row * g.ld_p + col;
          store4(p, have, v[k]);
          if (sizeof(T) == 2 && g.second) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float first = (float)(T)v[k][i];
              v[k][i] = fabsf(first) < __builtin_huge_valf() ? v[k][i] - first : 0.f;
            }
            store4(p + g.second, have, v[k]);
          }
        }
      }
    }
  }
  if (!g.partial) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) sums[threadIdx.x][i] = sum[i];
  __syncthreads();
  if (group == 0) {
    for (int k = 1; k < groups; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += sums[k * g.lanes + lane][i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < have) g.partial[(int64_t)blockIdx.y * g.N + col + i] = sum[i];
  }
}

// sums of the slabs' columns: 8 columns a block, 32 lanes each take every 32nd slab, added in their order
template <typename T>
__global__ __launch_bounds__(256) void slab_join_kernel(const double* __restrict__ partial, int64_t slabs, int64_t N, T* __restrict__ out) {
  __shared__ double sums[32][9];
  const int c = threadIdx.x & 7, k = threadIdx.x >> 3;
  const int64_t col = (int64_t)blockIdx.x * 8 + c;
  double t = 0.0;
  if (col < N) {
    for (int64_t s = k; s < slabs; s += 256) {               // 8 loads in flight, added in their order
      double v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = s + 32 * u < slabs ? partial[(s + 32 * u) * N + col] : 0.0;
#pragma unroll
      for (int u = 0; u < 8; ++u) t += v[u];
    }
  }
  sums[k][c] = t;
  __syncthreads();
  if (k == 0 && col < N) {
    for (int i = 1; i < 32; ++i) t += sums[i][c];
    out[col] = (T)(float)t;
  }
}

// ---------------------------------------------------------------------------------------
// The whole backward pass of a small layer (small_fit below) in one launch, where the launches are what it costs: a workgroup
// computes p = dy act'(x W + b) into LDS, in fp32 and for itself, and gives the gradients of `chunk` columns of x: their rows
// of dw = x^T p, their columns of dx = p W^T; the first workgroup adds p's columns up. Plain fused multiply-adds in fp32: few
// products average over few roundings, so p is not rounded to 16 bits here as it is on the way to the matrix cores.
// ---------------------------------------------------------------------------------------
constexpr int kSmall = 4096;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Small {
  const void *x, *w, *dy, *save;
  void *dx, *dw, *db;
  int64_t ldx, ldw, ldd, lds, lddx, lddw;
  int M, K, N, act, chunk;
};

// out(o, sum over l < L of f(o, l)) for o < count by 256 lanes: 1 to 64 lanes (a power of two) share a sum
template <typename S, typename F, typename G>
__device__ __forceinline__ void small_sums(int count, int L, F f, G out) {
  int share = 1;
  while (share < 64 && count * share * 2 <= 256) share *= 2;
  const int part = threadIdx.x % share;
  for (int base = 0; base < count; base += 256 / share) {
    const int o = base + threadIdx.x / share;
    S t = 0;
    if (o < count)
      for (int l = part; l < L; l += share) t = f(o, l, t);
    for (int d = 1; d < share; d <<= 1) t += __shfl_xor(t, d);
    if (o < count && part == 0) out(o, t);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void small_backward_kernel(const Small g) {
  __shared__ float p[kSmall], xs[kSmall], ws[kSmall + 16];
  const int M = g.M, N = g.N, k0 = blockIdx.x * g.chunk, KC = g.K - k0 < g.chunk ? g.K - k0 : g.chunk, pitch = N + 1 - (N & 1);
  for (int i = threadIdx.x; i < M * N; i += 256) {
    const int m = i / N, n = i % N;
    float v = (float)((const T*)g.dy)[m * g.ldd + n];
    if (g.act == ACT_RELU) v = ((const uint32_t*)g.save)[m * g.lds + n / 32] >> (n & 31) & 1 ? v : 0.f;
    else if (g.act != ACT_NONE) v *= slope_of<T>(g.act, ((const float*)g.save)[m * g.lds + n]);
    p[i] = v;
  }
  if (g.dw)
    for (int i = threadIdx.x; i < M * KC; i += 256) xs[i] = (float)((const T*)g.x)[i / KC * g.ldx + k0 + i % KC];
  if (g.dx)
    for (int i = threadIdx.x; i < KC * N; i += 256) ws[i / N * pitch + i % N] = (float)((const T*)g.w)[(k0 + i / N) * g.ldw + i % N];
  __syncthreads();
  if (g.dw)
    small_sums<float>(KC * N, M, [&](int o, int m, float t) { return fmaf(xs[m * KC + o / N], p[m * N + o % N], t); },
               [&](int o, float t) { ((T*)g.dw)[(int64_t)(k0 + o / N) * g.lddw + o % N] = (T)t; });
  if (g.dx)
    small_sums<float>(M * KC, N, [&](int o, int n, float t) { return fmaf(p[o / KC * N + n], ws[o % KC * pitch + n], t); },
               [&](int o, float t) { ((T*)g.dx)[(int64_t)(o / KC) * g.lddx + k0 + o % KC] = (T)t; });
  if (g.db && blockIdx.x == 0)
    small_sums<double>(N, M, [&](int n, int m, double t) { return t + p[m * N + n]; }, [&](int n, double t) { ((T*)g.db)[n] = (T)(float)t; });
}

// Columns of x a workgroup takes: p, x's and W's parts each have 4096 floats of LDS.
int64_t small_chunk(int64_t M, int64_t N) {
  const int64_t side = M > N ? M : N;
  return side <= kSmall / 16 ? 16 : kSmall / side;
}

// Each workgroup computes all of p for its own few columns, so what bounds the rule is that repeated work: p's values, and the
// workgroups, at most two a compute unit. With tall or wide p the columns are so few that x is read in pieces of 4 to 16 bytes
// a row. One launch against separate ones, gelu: fp32 8 x 1024 x 64 8.5, 19.2 us; 64 x 2048 x 32 19.6, 21.6; 1024 x 2048 x 4
// 33.6, 35.2; beyond the values 64 x 64 x 64 33.4, 23.6; 256 x 1024 x 16 37.2, 29.0; bf16 8 x 256 x 512 26.6, 23.8; beyond the
// workgroups fp32 1024 x 4096 x 1 46.0, 40.9; 4096 x 1024 x 1 74.6, 43.0; 4096 x 4096 x 1 289, 81; bf16 217, 58.
bool small_fit(int64_t M, int64_t K, int64_t N) {
  return M > 0 && N > 0 && K > 0 && M <= kSmall && N <= kSmall && M * N <= (N <= 4 ? kSmall : kSmall / 2) && ceil_div(K, small_chunk(M, N)) <= 512;
}

// dx of few values (takes_few below): a workgroup takes up to 8 of a row, p in fp32 from dy and what was saved, once for all of
// them. It is latency that it takes: bf16 gelu, with the slope's launch, 77 x 23 x 300 8.4 us, on tiles 13.5; 77 x 23 x 4000 11.9,
// 12.7; 2 x 1024 x 4096 11.2, 10.2; 2048 x 1 x 64 10.5, 8.2; past the rule 16 x 128 x 16384 22.3, 12.7.
constexpr int kFew = 8;

template <typename T>
__global__ __launch_bounds__(256) void few_inputs_kernel(const Small g) {
  __shared__ float sums[4][kFew];
  const int groups = (g.K + kFew - 1) / kFew, m = blockIdx.x / groups, k0 = blockIdx.x % groups * kFew, lane = threadIdx.x & 63;
  const T* const dy = (const T*)g.dy + m * g.ldd;
  const float* const pre = (const float*)g.save + m * g.lds;
  const T* w[kFew];
  float t[kFew];
#pragma unroll
  for (int i = 0; i < kFew; ++i) {
    w[i] = (const T*)g.w + (k0 + i < g.K ? k0 + i : g.K - 1) * g.ldw;             // past the end the last one stands in
    t[i] = 0.f;
  }
  for (int n0 = threadIdx.x; n0 < g.N; n0 += 512) {            // two columns of each operand in flight
    T c[2][kFew], d[2];
    float f[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int n = n0 + 256 * u < g.N ? n0 + 256 * u : n0;
      d[u] = dy[n];
      f[u] = pre[n];
#pragma unroll
      for (int i = 0; i < kFew; ++i) c[u][i] = w[i][n];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (n0 + 256 * u >= g.N) break;
      const float p = (float)d[u] * slope_of<T>(g.act, f[u]);
#pragma unroll
      for (int i = 0; i < kFew; ++i) t[i] = fmaf(p, (float)c[u][i], t[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kFew; ++i) {
    for (int d = 1; d < 64; d <<= 1) t[i] += __shfl_xor(t[i], d);
    if (lane == 0) sums[threadIdx.x >> 6][i] = t[i];
  }
  __syncthreads();
  const int k = threadIdx.x;
  if (k < kFew && k0 + k < g.K) ((T*)g.dx)[m * g.lddx + k0 + k] = (T)(sums[0][k] + sums[1][k] + sums[2][k] + sums[3][k]);
}

// ---------------------------------------------------------------------------------------
constexpr int64_t kCompute = 256;              // compute units

// A product whose output tiles do not fill the compute units is cut along its contraction, at 128 elements a slice or more:
// for one workgroup a unit in any case, for as many as fit while the partial sums weigh less than half the operands (x^T p of
// 2708 x 1433 x 16 fp32 15.4 us, with one a unit 18.8; 8192 x 1024 x 1024 bf16 46.5, 46.7).
void cut(Gemm& g, int32_t dtype) {
  const Shape shape = dtype == DGNN_F32 ? shape_of<float>(g) : shape_of<_Float16>(g);
  const int64_t tiles = tiles_of(shape, g.M, g.N), one = kCompute / (tiles > 0 ? tiles : 1);
  const int64_t most = ceil_div(g.K, 128), light = g.M > 0 && g.N > 0 ? g.K * (g.M + g.N) / (4 * g.M * g.N) : 1;
  int64_t want = one > light ? one : light < one * resident_of(shape) ? light : one * resident_of(shape);
  if (want > most) want = most;
  if (want < 1) want = 1;
  g.slice_k = ceil_div(ceil_div(g.K, want), 64) * 64;
  if (g.slice_k == 0) g.slice_k = 64;
  g.slices = (int)ceil_div(g.K, g.slice_k);
  if (g.slices < 1) g.slices = 1;
}

int64_t slope_lanes(int64_t N) {
  int64_t lanes = 1;
  while (lanes < 64 && lanes * 4 < N) lanes *= 2;
  return lanes;
}

int64_t slope_slab(int64_t M, int64_t N) {
  const int64_t groups = 256 / slope_lanes(N), across = ceil_div(N, 4 * slope_lanes(N));
  const int64_t blocks = 1024 / (across < 1024 ? across : 1024);
  return ceil_div(ceil_div(M, blocks < 1 ? 1 : blocks), groups) * groups;
}

bool known_type(int32_t dtype) { return dtype == DGNN_F32 || dtype == DGNN_BF16 || dtype == DGNN_F16; }
int64_t width(int32_t dtype) { return dtype == DGNN_F32 ? 4 : 2; }

bool sizes_ok(int64_t M, int64_t K, int64_t N) {
  return M >= 0 && K >= 0 && N >= 0 && M <= 0x7fffffffLL && K <= (1 << 24) && N <= (1 << 24);      // launches stay below 2^32 lanes
}

// a row-major rows x cols matrix: present, rows that do not overlap, elements aligned
bool matrix_ok(const void* p, int64_t ld, int64_t rows, int64_t cols, int64_t w) {
  if (rows == 0 || cols == 0) return true;
  return p && ld >= cols && (uintptr_t)p % (uintptr_t)w == 0;
}

// Where a matrix lies: rows of `row` bytes `pitch` apart (0: there is one), from `at` to before `end` (at == end: nowhere).
struct Place {
  uintptr_t at, end;
  int64_t pitch, row;
};

Place place(const void* p, int64_t ld, int64_t rows, int64_t cols, int64_t w) {
  if (!p || rows == 0 || cols == 0) return {0, 0, 0, 0};
  return {(uintptr_t)p, (uintptr_t)p + (uintptr_t)(((rows - 1) * ld + cols) * w), rows > 1 ? ld * w : 0, cols * w};
}

// no byte of one is a byte of the other; columns of one buffer, whose rows take turns, are apart
bool apart(const Place& a, const Place& b) {
  if (a.at == a.end || b.at == b.end || a.end <= b.at || b.end <= a.at) return true;
  const int64_t pitch = a.pitch ? a.pitch : b.pitch;
  if (pitch == 0 || (b.pitch && b.pitch != pitch)) return false;
  const int64_t d = a.at <= b.at ? (int64_t)(b.at - a.at) % pitch : (pitch - (int64_t)(a.at - b.at) % pitch) % pitch;
  return d >= a.row && d + b.row <= pitch;
}

// what a call writes is apart from what it reads and from what else it writes
bool apart(std::initializer_list<Place> written, std::initializer_list<Place> read) {
  for (const Place* a = written.begin(); a != written.end(); ++a) {
    for (const Place& b : read)
      if (!apart(*a, b)) return false;
    for (const Place* b = a + 1; b != written.end(); ++b)
      if (!apart(*a, *b)) return false;
  }
  return true;
}

// what the forward pass saved: relu's words, the others' floats
Place saved(const void* save, int64_t lds, int64_t M, int64_t N, int32_t act) {
  return place(act == ACT_NONE ? nullptr : save, lds, M, act == ACT_RELU ? (N + 31) / 32 : N, 4);
}
bool saved_ok(const void* save, int64_t lds, int64_t M, int64_t N, int32_t act) {
  return act == ACT_NONE || matrix_ok(save, lds, M, act == ACT_RELU ? (N + 31) / 32 : N, 4);
}

// How a product runs, by its sizes: a handful of rows on plain multiply-adds, over W's laid-out image where there are many rows,
// else by tiles, cut along the contraction where those are few. Returns the bytes of workspace that takes.
int64_t plan(Gemm& g, int32_t dtype) {
  if (g.pieces) {
    Gemm wide = both_pieces(g);
    cut(wide, dtype);
    g.slices = wide.slices;
    g.slice_k = wide.slice_k;
    return (int64_t)g.slices * g.M * wide.N * 4;
  }
  if (dtype == DGNN_F32 ? thin_fit<float>(g) : thin_fit<_Float16>(g)) {
    if (dtype == DGNN_F32) thin_cut<float>(g); else thin_cut<_Float16>(g);
    return g.slices > 1 ? (int64_t)g.slices * g.M * g.N * 4 : 0;
  }
  if (dtype == DGNN_F32 && columns_fit<float>(g)) {
    columns_cut(g);
    return g.slices > 1 ? (int64_t)g.slices * g.M * g.N * 4 : 0;
  }
  if (rows_fit(g)) {
    g.slices = 1;
    return dtype == DGNN_F32 ? rows_image<float>(g) : rows_image<_Float16>(g);
  }
  cut(g, dtype);
  return g.slices > 1 ? (int64_t)g.slices * g.M * g.N * 4 : 0;
}

// whether a grid holds the output's tiles, where the product runs by tiles
template <typename T> bool tiles_fit(const Gemm& g) {
  if (g.pieces) return tiles_of(shape_of<T>(both_pieces(g)), g.M, 2 * g.N) < (1 << 23);
  return thin_fit<T>(g) || columns_fit<T>(g) || rows_fit(g) || tiles_of(shape_of<T>(g), g.M, g.N) < (1 << 23);
}
bool launch_fits(const Gemm& g, int32_t dtype) { return dtype == DGNN_F32 ? tiles_fit<float>(g) : tiles_fit<_Float16>(g); }

int run(const Gemm& g, int32_t dtype, void* workspace, int64_t bytes, const char* who) {
  if (!launch_fits(g, dtype)) return dgnn_fail(DGNN_E_BADARG, "%s: too many tiles of output", who);
  Gemm h = g;
  const int64_t need = plan(h, dtype);
  if (need && (!workspace || bytes < need || (uintptr_t)workspace % 16))
    return dgnn_fail(DGNN_E_BADARG, "%s: workspace too small or misaligned (%lld bytes wanted)", who, (long long)need);
  if (h.slices > 1 || h.pieces) h.partial = (float*)workspace;
  else if (need) h.image = (char*)workspace;
  if (dtype == DGNN_F32) return gemm_f32(h);
  if (dtype == DGNN_BF16) return gemm_bf16(h);
  return gemm_f16(h);
}

}  // namespace

extern "C" {

int dgnn_linear_workspace(int32_t pass, int64_t M, int64_t K, int64_t N, int32_t dtype, int64_t* bytes) {
  if (!bytes || !known_type(dtype) || !sizes_ok(M, K, N)) return dgnn_fail(DGNN_E_BADARG, "linear_workspace: bad argument%s");
  *bytes = 0;
  Gemm g{};
  switch (pass) {
    case DGNN_LINEAR_FORWARD: g.M = M; g.N = N; g.K = K; g.a_along = true; break;
    case DGNN_LINEAR_GRAD_INPUT: g.M = M; g.N = K; g.K = N; g.a_along = true; break;
    case DGNN_LINEAR_GRAD_WEIGHT: g.M = K; g.N = N; g.K = M; break;
    case DGNN_LINEAR_SLOPE:
      if (M > 0 && N > 0) *bytes = ceil_div(M, slope_slab(M, N)) * N * 8;
      return DGNN_OK;
    default: return dgnn_fail(DGNN_E_BADARG, "linear_workspace: unknown pass%s (%lld)", "", pass);
  }
  if (g.M == 0 || g.N == 0) return DGNN_OK;
  *bytes = plan(g, dtype);
  return DGNN_OK;
}

int dgnn_linear_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                        const void* residual, int64_t ldr, void* y, int64_t ldy, void* save, int64_t lds,
                        int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t act,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  if (!known_type(dtype)) return dgnn_fail(DGNN_E_BADARG, "linear_forward: unknown type%s (%lld)", "", dtype);
  if (act < ACT_NONE || act > ACT_SILU) return dgnn_fail(DGNN_E_BADARG, "linear_forward: unknown activation%s (%lld)", "", act);
  if (!sizes_ok(M, K, N)) return dgnn_fail(DGNN_E_BADARG, "linear_forward: bad sizes%s");
  if (M == 0 || N == 0) return DGNN_OK;
  const int64_t b = width(dtype);
  if (!matrix_ok(x, ldx, M, K, b) || !matrix_ok(w, ldw, K, N, b) || !matrix_ok(y, ldy, M, N, b) || (uintptr_t)bias % b
      || (residual && !matrix_ok(residual, ldr, M, N, b)))
    return dgnn_fail(DGNN_E_BADARG, "linear_forward: null, misaligned or overlapping rows%s");
  if (save && !saved_ok(save, lds, M, N, act)) return dgnn_fail(DGNN_E_BADARG, "linear_forward: save is too narrow or misaligned%s");
  if (!apart({place(y, ldy, M, N, b), saved(save, lds, M, N, act)},
             {place(x, ldx, M, K, b), place(w, ldw, K, N, b), place(bias, N, 1, N, b), place(residual, ldr, M, N, b)}))
    return dgnn_fail(DGNN_E_BADARG, "linear_forward: y or save overlaps another operand%s");
  Gemm g{};
  g.a = x; g.lda = ldx; g.a_along = true;
  g.b = w; g.ldb = ldw; g.b_along = false;
  g.M = M; g.N = N; g.K = K;
  g.bias = bias; g.residual = residual; g.ld_residual = ldr;
  g.c = y; g.ldc = ldy;
  g.save = act == ACT_NONE ? nullptr : save; g.ld_save = lds;
  g.act = act;
  g.stream = (hipStream_t)stream;
  return run(g, dtype, workspace, workspace_bytes, "linear_forward");
}

static int slope(const void* dy, int64_t ldd, const void* save, int64_t lds, void* p, int64_t ldp, int64_t second, void* dbias,
                 int64_t M, int64_t N, int32_t dtype, int32_t act, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!known_type(dtype)) return dgnn_fail(DGNN_E_BADARG, "linear_slope: unknown type%s (%lld)", "", dtype);
  if (act < ACT_NONE || act > ACT_SILU) return dgnn_fail(DGNN_E_BADARG, "linear_slope: unknown activation%s (%lld)", "", act);
  if (!sizes_ok(M, 0, N)) return dgnn_fail(DGNN_E_BADARG, "linear_slope: bad sizes%s");
  if (N == 0) return DGNN_OK;
  const int64_t b = width(dtype);
  hipStream_t s = (hipStream_t)stream;
  if ((uintptr_t)dbias % b) return dgnn_fail(DGNN_E_BADARG, "linear_slope: misaligned dbias%s");
  if (M > 0) {
    if (!matrix_ok(dy, ldd, M, N, b) || (p && !matrix_ok(p, ldp, M, N, b)) || !saved_ok(save, lds, M, N, act))
      return dgnn_fail(DGNN_E_BADARG, "linear_slope: null, misaligned or overlapping rows%s");
    const Place from = place(p == dy && ldp == ldd ? nullptr : dy, ldd, M, N, b);          // p may be dy itself
    if (!apart({place(p, ldp, M, N, b), place(dbias, N, 1, N, b)}, {from, saved(save, lds, M, N, act)}))
      return dgnn_fail(DGNN_E_BADARG, "linear_slope: p or dbias overlaps another operand%s");
  }
  const int64_t lanes = slope_lanes(N), slab = M > 0 ? slope_slab(M, N) : 1, slabs = ceil_div(M, slab);
  if (dbias && slabs > 0 && (!workspace || workspace_bytes < slabs * N * 8 || (uintptr_t)workspace % 8))
    return dgnn_fail(DGNN_E_BADARG, "linear_slope: workspace too small%s (%lld bytes wanted)", "", slabs * N * 8);
  if (M > 0 && (p || dbias)) {
    const Slope g{dy, save, p, ldd, lds, ldp, M, N, slab, second, dbias ? (double*)workspace : nullptr, act, (int)lanes};
    const dim3 grid((uint32_t)ceil_div(N, 4 * lanes), (uint32_t)slabs);
    if (dtype == DGNN_F32) hipLaunchKernelGGL((slope_kernel<float>), grid, dim3(256), 0, s, g);
    else if (dtype == DGNN_BF16) hipLaunchKernelGGL((slope_kernel<__bf16>), grid, dim3(256), 0, s, g);
    else hipLaunchKernelGGL((slope_kernel<_Float16>), grid, dim3(256), 0, s, g);
    DGNN_LAUNCHED();
  }
  if (dbias) {
    const dim3 grid((uint32_t)ceil_div(N, 8));
    if (dtype == DGNN_F32) hipLaunchKernelGGL((slab_join_kernel<float>), grid, dim3(256), 0, s, (const double*)workspace, slabs, N, (float*)dbias);
    else if (dtype == DGNN_BF16) hipLaunchKernelGGL((slab_join_kernel<__bf16>), grid, dim3(256), 0, s, (const double*)workspace, slabs, N, (__bf16*)dbias);
    else hipLaunchKernelGGL((slab_join_kernel<_Float16>), grid, dim3(256), 0, s, (const double*)workspace, slabs, N, (_Float16*)dbias);
    DGNN_LAUNCHED();
  }
  return DGNN_OK;
}

int dgnn_linear_slope(const void* dy, int64_t ldd, const void* save, int64_t lds, void* p, int64_t ldp, void* dbias,
                      int64_t M, int64_t N, int32_t dtype, int32_t act, void* workspace, int64_t workspace_bytes, void* stream) {
  return slope(dy, ldd, save, lds, p, ldp, 0, dbias, M, N, dtype, act, workspace, workspace_bytes, stream);
}

int dgnn_linear_grad_input(const void* p, int64_t ldp, const void* w, int64_t ldw, const void* add, int64_t lda,
                           void* dx, int64_t ldx, int64_t M, int64_t K, int64_t N, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!known_type(dtype)) return dgnn_fail(DGNN_E_BADARG, "linear_grad_input: unknown type%s (%lld)", "", dtype);
  if (!sizes_ok(M, K, N)) return dgnn_fail(DGNN_E_BADARG, "linear_grad_input: bad sizes%s");
  if (M == 0 || K == 0) return DGNN_OK;
  const int64_t b = width(dtype);
  if (!matrix_ok(p, ldp, M, N, b) || !matrix_ok(w, ldw, K, N, b) || !matrix_ok(dx, ldx, M, K, b)
      || (add && !matrix_ok(add, lda, M, K, b)))
    return dgnn_fail(DGNN_E_BADARG, "linear_grad_input: null, misaligned or overlapping rows%s");
  if (!apart({place(dx, ldx, M, K, b)}, {place(p, ldp, M, N, b), place(w, ldw, K, N, b), place(add, lda, M, K, b)}))
    return dgnn_fail(DGNN_E_BADARG, "linear_grad_input: dx overlaps an input%s");
  Gemm g{};
  g.a = p; g.lda = ldp; g.a_along = true;
  g.b = w; g.ldb = ldw; g.b_along = true;
  g.M = M; g.N = K; g.K = N;
  g.residual = add; g.ld_residual = lda;
  g.c = dx; g.ldc = ldx;
  g.stream = (hipStream_t)stream;
  return run(g, dtype, workspace, workspace_bytes, "linear_grad_input");
}

static int grad_weight(const void* x, int64_t ldx, const void* p, int64_t ldp, bool pieces, void* dw, int64_t ldw,
                       int64_t M, int64_t K, int64_t N, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!known_type(dtype)) return dgnn_fail(DGNN_E_BADARG, "linear_grad_weight: unknown type%s (%lld)", "", dtype);
  if (!sizes_ok(M, K, N)) return dgnn_fail(DGNN_E_BADARG, "linear_grad_weight: bad sizes%s");
  if (K == 0 || N == 0) return DGNN_OK;
  const int64_t b = width(dtype);
  if (!matrix_ok(x, ldx, M, K, b) || !matrix_ok(p, ldp, M, N, b) || !matrix_ok(dw, ldw, K, N, b))
    return dgnn_fail(DGNN_E_BADARG, "linear_grad_weight: null, misaligned or overlapping rows%s");
  if (!apart({place(dw, ldw, K, N, b)}, {place(x, ldx, M, K, b), place(p, ldp, M, N, b)}))
    return dgnn_fail(DGNN_E_BADARG, "linear_grad_weight: dw overlaps an input%s");
  Gemm g{};
  g.a = x; g.lda = ldx; g.a_along = false;
  g.b = p; g.ldb = ldp; g.b_along = false;
  g.M = K; g.N = N; g.K = M;
  g.c = dw; g.ldc = ldw;
  g.pieces = pieces;
  g.stream = (hipStream_t)stream;
  return run(g, dtype, workspace, workspace_bytes, "linear_grad_weight");
}

int dgnn_linear_grad_weight(const void* x, int64_t ldx, const void* p, int64_t ldp, void* dw, int64_t ldw,
                            int64_t M, int64_t K, int64_t N, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  return grad_weight(x, ldx, p, ldp, false, dw, ldw, M, K, N, dtype, workspace, workspace_bytes, stream);
}

// Everything a gradient dy of y gives, in one call: what the three entries above compute, in the same order on the stream, so
// that one workspace serves them one after the other behind p's part of it.
// Where p of gelu or silu is rounded to 16 bits, a narrow layer's weight gradient takes it in two pieces, the rounded value and
// what that left: its few columns, or few values in all, average over few roundings (x behind an activation is positive, so all of
// a column's sums share the errors of its p), and a product that is bound by its bytes has room for the second pieces. All
// gradients of bf16 gelu with rounded p and with its pieces: 232965 x 256 x 41 135, 145 us; 232965 x 602 x 41 253, 242; 2449029 x
// 128 x 47 717, 834; 2000000 x 4 x 4 633, 438. Few weights in many columns pay more once p leaves the caches (1000000 x 1 x 88 376,
// 582), so they take the pieces up to 2^24 values of p only. Wider weight gradients and the input gradient, whose error is 1.4 times
// that of their own rounding, take the rounded values.
static bool takes_pieces(int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t act) {
  if (dtype == DGNN_F32 || act <= ACT_RELU || M == 0 || K == 0 || N == 0 || small_fit(M, K, N)) return false;
  return N <= 64 ? K * N <= (1 << 20) : K * N <= 4096 && M * N <= (1 << 24);
}

// Nor do the roundings of p average in an input gradient of a few values, whose product is no work.
static bool takes_few(int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t act) {
  return dtype != DGNN_F32 && act > ACT_RELU && M > 0 && K > 0 && N > 0 && M * K <= 2048 && M * K * N <= (1 << 24);
}

static Gemm weight_product(int64_t M, int64_t K, int64_t N, bool pieces) {
  Gemm g{};
  g.M = K; g.N = N; g.K = M;
  g.pieces = pieces;
  return g;
}

static int64_t backward_parts(int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t act, int64_t* p_bytes) {
  int64_t most = 0;
  const bool pieces = takes_pieces(M, K, N, dtype, act);
  for (int32_t pass = DGNN_LINEAR_SLOPE; pass <= DGNN_LINEAR_GRAD_WEIGHT; ++pass) {
    int64_t n = 0;
    (void)dgnn_linear_workspace(pass, M, K, N, dtype, &n);
    if (n > most) most = n;
  }
  *p_bytes = 0;
  if (small_fit(M, K, N)) return 0;
  if (pieces) {
    Gemm g = weight_product(M, K, N, true);
    const int64_t n = plan(g, dtype);
    if (n > most) most = n;
  }
  *p_bytes = act == ACT_NONE ? 0 : ceil_div(M * N * width(dtype) * (pieces ? 2 : 1), 256) * 256;
  return *p_bytes + most;
}

int dgnn_linear_backward_workspace(int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t act, int64_t* bytes) {
  if (!bytes || !known_type(dtype) || !sizes_ok(M, K, N) || act < ACT_NONE || act > ACT_SILU)
    return dgnn_fail(DGNN_E_BADARG, "linear_backward_workspace: bad argument%s");
  int64_t p;
  *bytes = backward_parts(M, K, N, dtype, act, &p);
  return DGNN_OK;
}

int dgnn_linear_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* dy, int64_t ldd,
                         const void* save, int64_t lds, void* dx, int64_t lddx, void* dw, int64_t lddw, void* dbias,
                         int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t act,
                         void* workspace, int64_t workspace_bytes, void* stream) {
  if (!known_type(dtype)) return dgnn_fail(DGNN_E_BADARG, "linear_backward: unknown type%s (%lld)", "", dtype);
  if (act < ACT_NONE || act > ACT_SILU) return dgnn_fail(DGNN_E_BADARG, "linear_backward: unknown activation%s (%lld)", "", act);
  if (!sizes_ok(M, K, N)) return dgnn_fail(DGNN_E_BADARG, "linear_backward: bad sizes%s");
  int64_t p_bytes;
  const int64_t need = backward_parts(M, K, N, dtype, act, &p_bytes);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return dgnn_fail(DGNN_E_BADARG, "linear_backward: workspace too small or misaligned%s (%lld bytes wanted)", "", need);
  const int64_t b = width(dtype);
  if (!matrix_ok(dy, ldd, M, N, b) || (dw && (!matrix_ok(x, ldx, M, K, b) || !matrix_ok(dw, lddw, K, N, b)))
      || (dx && (!matrix_ok(w, ldw, K, N, b) || !matrix_ok(dx, lddx, M, K, b))) || (uintptr_t)dbias % b || !saved_ok(save, lds, M, N, act))
    return dgnn_fail(DGNN_E_BADARG, "linear_backward: null, misaligned or overlapping rows%s");
  if (!apart({place(dx, lddx, M, K, b), place(dw, lddw, K, N, b), place(dbias, N, 1, N, b)},
             {place(dw ? x : nullptr, ldx, M, K, b), place(dx ? w : nullptr, ldw, K, N, b), place(dy, ldd, M, N, b), saved(save, lds, M, N, act)}))
    return dgnn_fail(DGNN_E_BADARG, "linear_backward: an output overlaps another operand%s");
  if (small_fit(M, K, N)) {
    if (!dx && !dw && !dbias) return DGNN_OK;
    const int64_t chunk = small_chunk(M, N);
    const Small g{x, w, dy, save, dx, dw, dbias, ldx, ldw, ldd, lds, lddx, lddw, (int)M, (int)K, (int)N, (int)act, (int)chunk};
    const dim3 grid(dx || dw ? (uint32_t)ceil_div(K, chunk) : 1);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DGNN_F32) hipLaunchKernelGGL((small_backward_kernel<float>), grid, dim3(256), 0, s, g);
    else if (dtype == DGNN_BF16) hipLaunchKernelGGL((small_backward_kernel<__bf16>), grid, dim3(256), 0, s, g);
    else hipLaunchKernelGGL((small_backward_kernel<_Float16>), grid, dim3(256), 0, s, g);
    DGNN_LAUNCHED();
    return DGNN_OK;
  }
  const bool pieces = dw && takes_pieces(M, K, N, dtype, act);
  const int64_t pitch = pieces ? 2 * N : N;
  Gemm to_x{}, to_w = weight_product(M, K, N, pieces);
  to_x.M = M; to_x.N = K; to_x.K = N; to_x.a_along = to_x.b_along = true;
  to_w.lda = ldx; to_w.ldb = act == ACT_NONE ? ldd : pitch;
  if ((dx && !launch_fits(to_x, dtype)) || (dw && !launch_fits(to_w, dtype))) return dgnn_fail(DGNN_E_BADARG, "linear_backward: too many tiles of output%s");
  char* rest = (char*)workspace + p_bytes;
  const void* p = dy;
  int64_t ldp = ldd;
  const bool few = takes_few(M, K, N, dtype, act), p_wanted = act != ACT_NONE && M > 0 && N > 0 && (dw || (dx && !few));
  if (p_wanted || dbias) {
    const int rc = slope(dy, ldd, save, lds, p_wanted ? workspace : nullptr, pitch, pieces ? N : 0, dbias, M, N, dtype, act, rest, need - p_bytes, stream);
    if (rc != DGNN_OK) return rc;
  }
  if (act != ACT_NONE) { p = workspace; ldp = pitch; }
  if (dx && few) {
    const Small g{x, w, dy, save, dx, dw, dbias, ldx, ldw, ldd, lds, lddx, lddw, (int)M, (int)K, (int)N, (int)act, 0};
    const dim3 grid((uint32_t)(M * ceil_div(K, kFew)));
    if (dtype == DGNN_BF16) hipLaunchKernelGGL((few_inputs_kernel<__bf16>), grid, dim3(256), 0, (hipStream_t)stream, g);
    else hipLaunchKernelGGL((few_inputs_kernel<_Float16>), grid, dim3(256), 0, (hipStream_t)stream, g);
    DGNN_LAUNCHED();
  } else if (dx) {
    const int rc = dgnn_linear_grad_input(p, ldp, w, ldw, nullptr, 0, dx, lddx, M, K, N, dtype, rest, need - p_bytes, stream);
    if (rc != DGNN_OK) return rc;
  }
  return dw ? grad_weight(x, ldx, p, ldp, pieces, dw, lddw, M, K, N, dtype, rest, need - p_bytes, stream) : DGNN_OK;
}

}  // extern "C"
