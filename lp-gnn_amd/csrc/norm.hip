// Layer norm over the rows of a node set, with an optional ReLU behind it:
//
//   mu = mean_j x_j,  s = 1 / sqrt(mean_j (x_j - mu)^2 + eps),  h_j = (x_j - mu) s,  y_j = act(h_j w_j + b_j)
//
// and its backward pass, with z_j = dy_j [h_j w_j + b_j > 0] (ReLU) or dy_j:
//
//   dx_j = s (z_j w_j - mean(z w) - h_j mean(z w h)),   dw_j = sum_rows z_j h_j,   db_j = sum_rows z_j
//
// x, y, dy, dx fp32, bf16 or fp16 (w, b, dw, db fp32 or that type); statistics and sums in fp32, one
// rounding on each store.  HBM-bound: a row is read once into registers, so the mean and the centred sum
// of squares are two exact passes over registers and not over memory (a one-pass sum of squares loses
// its digits where |mu| >> 1 / s).
//
// Rows of up to 2048 elements: G lanes (a power of two) of one wave hold a row, NV vectors of 16 bytes a
// lane, 64 / G rows a wave; the sums are butterflies over those lanes.  Rows are read with 16-byte loads
// whatever their alignment (the memory pipeline takes any element alignment), and the last vector of a
// row whose length is no multiple of the vector starts early enough to end with the row, its first `lo`
// elements (the neighbour's) masked out of every sum -- no scalar tail, no read past the row.
// Everything else (rows shorter than a vector or longer than 2048): one block a row, elements strided
// over its threads, three passes over a row that stays in L2.
//
// Weight gradients without atomics: a lane keeps its columns' sums of all its rows in registers (a
// persistent grid), the block adds its waves' sums in wave order in LDS and writes one partial row, and
// a second kernel adds the partial rows in block order: the same bits every run.
//
// Kernel times: forward 100 K x 1024 fp32 143 us (5.7 TB/s), 200 K x 2048 bf16 297 (5.5), 50001 x 1000 fp16 41
// (4.9, rows off cache lines), 200 x 128 2.8; backward of the first two 221 (5.6 TB/s) and 421 (5.8), with the ReLU 226
// and 432, their folds 5.  A block a row is far from that: 50 K x 4096 bf16 526 us forward (1.6 TB/s), 1.3 ms with
// the backward (1.3), 1.5 with the ReLU.
#include "common.h"

#include <type_traits>

namespace lpg {
namespace {

constexpr int kT = 256, kW = kT / 64;

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  return (float)v;
}

// 16 bytes at any element alignment
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T>
__device__ __forceinline__ void unpack(u32x4 v, float (&f)[16 / sizeof(T)]) {
  T t[16 / sizeof(T)];
  __builtin_memcpy(t, &v, 16);
#pragma unroll
  for (int j = 0; j < (int)(16 / sizeof(T)); ++j) f[j] = (float)t[j];
}
template <typename T>
__device__ __forceinline__ void stv(T *p, const float (&f)[16 / sizeof(T)]) {
  T t[16 / sizeof(T)];
#pragma unroll
  for (int j = 0; j < (int)(16 / sizeof(T)); ++j) t[j] = (T)f[j];
  u32x4 v;
  __builtin_memcpy(&v, t, 16);
  if constexpr (sizeof(T) == 2) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_at2 *>(p));
  else __builtin_nontemporal_store(v, reinterpret_cast<u32x4_at4 *>(p));
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
// One butterfly level: v + the v of the lane S away (xor), every lane of a group of 2 S ends with the
// same sum.  Levels 4 and 8 are mirrors: below them the lanes of a group of S already agree.
template <int S>
__device__ __forceinline__ float xor_add(float v) {
  if constexpr (S == 1) return dpp_add<0xB1>(v);        // quad_perm 1,0,3,2
  else if constexpr (S == 2) return dpp_add<0x4E>(v);   // quad_perm 2,3,0,1
  else if constexpr (S == 4) return dpp_add<0x141>(v);  // row_half_mirror
  else if constexpr (S == 8) return dpp_add<0x140>(v);  // row_mirror
  else if constexpr (S == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
}
template <int G>  // the sum over the G lanes of a row, in each of them
__device__ __forceinline__ float row_sum(float v) {
  if constexpr (G > 1) v = xor_add<1>(v);
  if constexpr (G > 2) v = xor_add<2>(v);
  if constexpr (G > 4) v = xor_add<4>(v);
  if constexpr (G > 8) v = xor_add<8>(v);
  if constexpr (G > 16) v = xor_add<16>(v);
  if constexpr (G > 32) v = xor_add<32>(v);
  return v;
}

struct FwdArgs {
  int64_t M, D, ldx, ldy;
  const void *x, *w, *b;
  void *y;
  float *mean, *rstd;
  float eps;
  int relu;
};
struct BwdArgs {
  int64_t M, D, ldx, lddy, lddx;
  const void *x, *dy, *w, *b;
  const float *mean, *rstd;
  void *dx;
  float *part;  // [gridDim.x][2][D], or NULL
  int relu;
};

// The columns of this lane's NV vectors: vector k starts at (k G + l) V; the last one of a row ends with
// the row (start D - V, elements below `lo` belong to the vector before), past the row lo = V.
template <int G, int NV, int V>
struct Cols {
  int c[NV];
  int lo;
  __device__ __forceinline__ Cols(int l, int D) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int at = (k * G + l) * V;
      c[k] = at + V <= D ? at : D - V;
      if (k == NV - 1) lo = at + V <= D ? 0 : (at < D ? at - (D - V) : V);
    }
  }
  __device__ __forceinline__ bool live(int k, int j) const { return k < NV - 1 || j >= lo; }
};

template <typename W, int G, int NV, int V>
__device__ __forceinline__ void load_cols(const void *p, const Cols<G, NV, V> &cs, float (&f)[NV][V], float none) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) f[k][j] = p ? to_f(static_cast<const W *>(p)[cs.c[k] + j]) : none;
}

template <typename T, typename W, int G, int NV>
__global__ __launch_bounds__(kT) void norm_fwd(FwdArgs a) {
  constexpr int V = 16 / sizeof(T), R = 64 / G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slot = lane / G;
  const Cols<G, NV, V> cs(lane % G, (int)a.D);
  float w[NV][V], b[NV][V];
  load_cols<W>(a.w, cs, w, 1.f);
  load_cols<W>(a.b, cs, b, 0.f);
  const float n = (float)a.D;
  const T *x = static_cast<const T *>(a.x);
  T *y = static_cast<T *>(a.y);
  for (int64_t r0 = ((int64_t)blockIdx.x * kW + wave) * R; r0 < a.M; r0 += (int64_t)gridDim.x * kW * R) {
    const int64_t row = r0 + slot;
    const T *xr = x + (row < a.M ? row : a.M - 1) * a.ldx;
    float f[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      u32x4 raw;
      __builtin_memcpy(&raw, xr + cs.c[k], 16);
      unpack<T>(raw, f[k]);
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) s += cs.live(k, j) ? f[k][j] : 0.f;
    const float mu = row_sum<G>(s) / n;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[k][j] -= mu;
        s = cs.live(k, j) ? __builtin_fmaf(f[k][j], f[k][j], s) : s;
      }
    const float rs = 1.f / sqrtf(row_sum<G>(s) / n + a.eps);
    if (row < a.M) {
      T *yr = y + row * a.ldy;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float z = __builtin_fmaf(f[k][j] * rs, w[k][j], b[k][j]);
          f[k][j] = a.relu && z < 0.f ? 0.f : z;  // (a NaN stays one)
        }
        if (k < NV - 1 || cs.lo < V) stv<T>(yr + cs.c[k], f[k]);
      }
      if (a.mean && lane % G == 0) {
        a.mean[row] = mu;
        a.rstd[row] = rs;
      }
    }
  }
}

// U rows a lane group at a time; the next rows' vectors are loaded while these are computed (up to NV = 4: with longer
// fp32 rows the registers hold more by occupancy than by a row ahead).
// Two waves a SIMD, where the row and its columns' sums leave registers for them (not the longest rows).
template <typename T, int NV>
constexpr int bwd_waves() {
  return NV < (sizeof(T) == 2 ? 4 : 8) ? 2 : 1;
}
template <typename T, typename W, int G, int NV, bool RELU, int U>
__global__ __launch_bounds__(kT, (bwd_waves<T, NV>())) void norm_bwd(BwdArgs a) {
  constexpr int V = 16 / sizeof(T), R = 64 / G;
  constexpr bool AHEAD = NV <= 4;
  // h and z of a row are needed twice, for the sums and for dx.  Of 16-bit rows from three vectors on they are
  // formed twice from the row as it was loaded: half the registers, which decide how many waves a SIMD holds
  constexpr bool TWICE = sizeof(T) == 2 && NV >= 3;
  __shared__ float red[2][G * NV * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slot = lane / G;
  const Cols<G, NV, V> cs(lane % G, (int)a.D);
  float w[NV][V], b[NV][V], dw[NV][V], db[NV][V];
  load_cols<W>(a.w, cs, w, 1.f);
  if constexpr (RELU) load_cols<W>(a.b, cs, b, 0.f);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[k][j] = db[k][j] = 0.f;
  const float n = (float)a.D;
  const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy);
  u32x4 xn[U][NV], gn[U][NV];
  float mun[U], rsn[U];
  const auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = r0 + u * R < a.M ? r0 + u * R : a.M - 1;
      const T *xr = x + at * a.ldx, *gr = dy + at * a.lddy;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        __builtin_memcpy(&xn[u][k], xr + cs.c[k], 16);
        __builtin_memcpy(&gn[u][k], gr + cs.c[k], 16);
      }
      mun[u] = a.mean[at];
      rsn[u] = a.rstd[at];
    }
  };
  const int64_t step = (int64_t)gridDim.x * kW * R * U, end = a.M + slot;  // (the waves' loops have no lanes out)
  int64_t r0 = ((int64_t)blockIdx.x * kW + wave) * R * U + slot;
  if (AHEAD && r0 < end) fetch(r0);
  for (; r0 < end; r0 += step) {
    if (!AHEAD) fetch(r0);
    u32x4 xc[U][NV], gc[U][NV];
    float muc[U], rsc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < NV; ++k) xc[u][k] = xn[u][k], gc[u][k] = gn[u][k];
      muc[u] = mun[u], rsc[u] = rsn[u];
    }
    if (AHEAD && r0 + step < end) fetch(r0 + step);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + u * R;
      const bool in = row < a.M;
      const float mu = muc[u], rs = rsc[u];
      const auto hz = [&](int k, float (&h)[V], float (&z)[V]) {
        unpack<T>(xc[u][k], h);
        unpack<T>(gc[u][k], z);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          h[j] = (h[j] - mu) * rs;
          if constexpr (RELU) z[j] = __builtin_fmaf(h[j], w[k][j], b[k][j]) > 0.f ? z[j] : 0.f;
        }
      };
      float c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float h[V], z[V];
        hz(k, h, z);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (k == NV - 1) z[j] = cs.live(k, j) ? z[j] : 0.f;
          const float zi = U * R > 1 ? (in ? z[j] : 0.f) : z[j];  // (a wave of one row has none past the end)
          dw[k][j] = __builtin_fmaf(zi, h[j], dw[k][j]);
          db[k][j] += zi;
          z[j] *= w[k][j];
          c1 += z[j];
          c2 = __builtin_fmaf(z[j], h[j], c2);
        }
      }
      c1 = row_sum<G>(c1) / n;
      c2 = row_sum<G>(c2) / n;
      if (in && a.dx) {
        T *dr = static_cast<T *>(a.dx) + row * a.lddx;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          float h[V], z[V];
          if constexpr (TWICE) asm volatile("" : "+v"(xc[u][k]), "+v"(gc[u][k]));  // (or the compiler keeps them)
          hz(k, h, z);
#pragma unroll
          for (int j = 0; j < V; ++j) h[j] = __builtin_fmaf(-h[j], c2, z[j] * w[k][j] - c1) * rs;
          if (k < NV - 1 || cs.lo < V) stv<T>(dr + cs.c[k], h);
        }
      }
    }
  }
  if (!a.part) return;  // (uniform: no barrier is skipped by some)
  // rows of one wave: lanes G apart hold the same columns
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      for (int o = G; o < 64; o <<= 1) {
        dw[k][j] += __shfl_xor(dw[k][j], o, 64);
        db[k][j] += __shfl_xor(db[k][j], o, 64);
      }
    }
  for (int q = 0; q < kW; ++q) {  // waves in order
    if (wave == q && slot == 0) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int i = (k * G + lane) * V + j;  // (by vector, not by column: the early last vector overlaps)
          red[0][i] = (q ? red[0][i] : 0.f) + dw[k][j];
          red[1][i] = (q ? red[1][i] : 0.f) + db[k][j];
        }
    }
    __syncthreads();
  }
  if (wave == 0 && slot == 0) {
    float *p = a.part + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (cs.live(k, j)) {
          const int i = (k * G + lane) * V + j;
          p[cs.c[k] + j] = red[0][i];
          p[a.D + cs.c[k] + j] = red[1][i];
        }
  }
}

__device__ __forceinline__ float block_sum(float v, float *red) {
  v = row_sum<64>(v);
  __syncthreads();  // (red may still be read from the sum before)
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int q = 1; q < kW; ++q) v += red[q];
  return v;
}

// any row length: one block a row
template <typename T, typename W>
__global__ __launch_bounds__(kT) void norm_fwd_any(FwdArgs a) {
  __shared__ float red[kW];
  const W *w = static_cast<const W *>(a.w), *b = static_cast<const W *>(a.b);
  const float n = (float)a.D;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    T *y = static_cast<T *>(a.y) + row * a.ldy;
    float s = 0.f;
    for (int64_t j = threadIdx.x; j < a.D; j += kT) s += to_f(x[j]);
    const float mu = block_sum(s, red) / n;
    s = 0.f;
    for (int64_t j = threadIdx.x; j < a.D; j += kT) s = __builtin_fmaf(to_f(x[j]) - mu, to_f(x[j]) - mu, s);
    const float rs = 1.f / sqrtf(block_sum(s, red) / n + a.eps);
    for (int64_t j = threadIdx.x; j < a.D; j += kT) {
      const float z = __builtin_fmaf((to_f(x[j]) - mu) * rs, w ? to_f(w[j]) : 1.f, b ? to_f(b[j]) : 0.f);
      y[j] = (T)(a.relu && z < 0.f ? 0.f : z);
    }
    if (a.mean && threadIdx.x == 0) {
      a.mean[row] = mu;
      a.rstd[row] = rs;
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(kT) void norm_bwd_any(BwdArgs a) {
  __shared__ float red[kW];
  const W *w = static_cast<const W *>(a.w), *b = static_cast<const W *>(a.b);
  const float n = (float)a.D;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + row * a.ldx, *dy = static_cast<const T *>(a.dy) + row * a.lddy;
    T *dx = static_cast<T *>(a.dx) + row * a.lddx;
    const float mu = a.mean[row], rs = a.rstd[row];
    const auto hz = [&](int64_t j, float &h, float &z) {
      const float wj = w ? to_f(w[j]) : 1.f;
      h = (to_f(x[j]) - mu) * rs;
      z = to_f(dy[j]);
      if (a.relu && !(__builtin_fmaf(h, wj, b ? to_f(b[j]) : 0.f) > 0.f)) z = 0.f;
      z *= wj;
    };
    float c1 = 0.f, c2 = 0.f, h, z;
    for (int64_t j = threadIdx.x; j < a.D; j += kT) {
      hz(j, h, z);
      c1 += z;
      c2 = __builtin_fmaf(z, h, c2);
    }
    c1 = block_sum(c1, red) / n;
    c2 = block_sum(c2, red) / n;
    for (int64_t j = threadIdx.x; j < a.D; j += kT) {
      hz(j, h, z);
      dx[j] = (T)(__builtin_fmaf(-h, c2, z - c1) * rs);
    }
  }
}

// the weight gradients' partial rows of norm_bwd_any: a thread a column, block (x, y) = (columns, rows)
template <typename T, typename W>
__global__ __launch_bounds__(kT) void norm_wgrad_any(BwdArgs a) {
  const int64_t j = (int64_t)blockIdx.x * kT + threadIdx.x;
  if (j >= a.D) return;
  const W *w = static_cast<const W *>(a.w), *b = static_cast<const W *>(a.b);
  const float wj = w ? to_f(w[j]) : 1.f, bj = b ? to_f(b[j]) : 0.f;
  float sw = 0.f, sb = 0.f;
  for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
    const float h = (to_f(static_cast<const T *>(a.x)[row * a.ldx + j]) - a.mean[row]) * a.rstd[row];
    float z = to_f(static_cast<const T *>(a.dy)[row * a.lddy + j]);
    if (a.relu && !(__builtin_fmaf(h, wj, bj) > 0.f)) z = 0.f;
    sw = __builtin_fmaf(z, h, sw);
    sb += z;
  }
  a.part[(int64_t)blockIdx.y * 2 * a.D + j] = sw;
  a.part[(int64_t)blockIdx.y * 2 * a.D + a.D + j] = sb;
}

// dw, db = the sums of the nblk partial rows [2 D]: a block takes 64 columns, a thread four of them and every
// 64th row (all its loads in flight), the 64 row classes are added by a fixed tree
constexpr int kFoldC = 64, kFoldT = 1024, kFoldR = kFoldT / (kFoldC / 4);
template <typename W>
__global__ __launch_bounds__(kFoldT) void norm_fold(int64_t nblk, int64_t D, const float *__restrict__ part, W *dw, W *db) {
  __shared__ float red[kFoldR][kFoldC];
  const int c = (int)threadIdx.x % (kFoldC / 4) * 4, r = (int)threadIdx.x / (kFoldC / 4);
  const int64_t j0 = (int64_t)blockIdx.x * kFoldC, j = j0 + c, n = 2 * D - j;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (n >= 4) {
#pragma unroll 8
    for (int64_t k = r; k < nblk; k += kFoldR) {
      float v[4];
      __builtin_memcpy(v, part + k * 2 * D + j, 16);
#pragma unroll
      for (int q = 0; q < 4; ++q) s[q] += v[q];
    }
  } else if (n > 0) {
    for (int64_t k = r; k < nblk; k += kFoldR)
      for (int q = 0; q < 4; ++q) s[q] += q < n ? part[k * 2 * D + j + q] : 0.f;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) red[r][c + q] = s[q];
  __syncthreads();
  const int col = (int)threadIdx.x % kFoldC, part_of = (int)threadIdx.x / kFoldC;  // 16 parts of 4 classes
  float t = (red[part_of * 4][col] + red[part_of * 4 + 1][col]) + (red[part_of * 4 + 2][col] + red[part_of * 4 + 3][col]);
  __syncthreads();
  red[part_of][col] = t;
  __syncthreads();
  if (threadIdx.x < kFoldC && j0 + col < 2 * D) {
    t = 0.f;
#pragma unroll
    for (int q = 0; q < kFoldT / kFoldC; ++q) t += red[q][col];
    const int64_t at = j0 + col;
    if (at < D) {
      if (dw) dw[at] = (W)t;
    } else if (db) {
      db[at - D] = (W)t;
    }
  }
}

template <typename T>
int vec_of() {
  return 16 / (int)sizeof(T);
}
template <typename T>
bool in_lanes(int64_t D) {
  return D >= vec_of<T>() && D <= 2048;
}

// f(G, NV as constants) for the row length D: the fewest lanes that hold the row in one vector each, else a
// whole wave and as many vectors as it takes.  (Eight lanes and up to four vectors a lane -- more rows a wave,
// fewer idle lanes -- was slower wherever rows do not start on cache lines: a store then covers 128 bytes of
// each of eight rows, partial lines at both ends.  400 K rows of 100 fp32 numbers: 77 us forward against 51.)
template <typename T, typename F>
void by_width(int64_t D, F f) {
  constexpr int V = 16 / sizeof(T);
  const int64_t nv = (D + V - 1) / V;
#define LPG_IC(k) std::integral_constant<int, k>()
  if (nv <= 1) f(LPG_IC(1), LPG_IC(1));
  else if (nv <= 2) f(LPG_IC(2), LPG_IC(1));
  else if (nv <= 4) f(LPG_IC(4), LPG_IC(1));
  else if (nv <= 8) f(LPG_IC(8), LPG_IC(1));
  else if (nv <= 16) f(LPG_IC(16), LPG_IC(1));
  else if (nv <= 32) f(LPG_IC(32), LPG_IC(1));
  else if (nv <= 64) f(LPG_IC(64), LPG_IC(1));
  else if (nv <= 128) f(LPG_IC(64), LPG_IC(2));
  else if (nv <= 192) f(LPG_IC(64), LPG_IC(3));
  else if (nv <= 256) f(LPG_IC(64), LPG_IC(4));
  else if constexpr (V == 4) {
    if (nv <= 320) f(LPG_IC(64), LPG_IC(5));
    else if (nv <= 384) f(LPG_IC(64), LPG_IC(6));
    else if (nv <= 448) f(LPG_IC(64), LPG_IC(7));
    else f(LPG_IC(64), LPG_IC(8));
  }
#undef LPG_IC
}

int64_t at_most(int64_t n, int64_t most) { return n < 1 ? 1 : (n > most ? most : n); }

template <typename T, typename W>
lpg_status fwd(const FwdArgs &a, hipStream_t s) {
  if (in_lanes<T>(a.D)) {
    by_width<T>(a.D, [&](auto g, auto nv) {
      constexpr int G = decltype(g)::value, NV = decltype(nv)::value, R = 64 / G * kW;
      auto k = norm_fwd<T, W, G, NV>;
      const int64_t nblk = at_most((a.M + R - 1) / R, resident_blocks(k, kT));
      hipLaunchKernelGGL(k, dim3((unsigned)nblk), dim3(kT), 0, s, a);
    });
  } else {
    hipLaunchKernelGGL((norm_fwd_any<T, W>), dim3((unsigned)at_most(a.M, 1 << 16)), dim3(kT), 0, s, a);
  }
  LPG_HIP(hipGetLastError());
  return LPG_OK;
}

// Partial rows of the weight gradients: the blocks of the backward grid.  Each block's rows amortise its
// partial (2 D floats out, read again by the fold) and the fold's walk over the partials.
constexpr int64_t kPartRows = 1024;

template <typename T, typename W>
lpg_status bwd(BwdArgs a, W *dw, W *db, float *part, hipStream_t s) {
  a.part = dw || db ? part : nullptr;
  int64_t nblk = 0;
  if (a.M > 0 && in_lanes<T>(a.D)) {
    by_width<T>(a.D, [&](auto g, auto nv) {
      // Two rows a lane group at a time where a row is one or two vectors a lane: one leaves too little in flight
      // (400 K x 129 bf16 82 us with one row, 75 with two; 100 K x 1023 131 and 121) -- unless that would leave
      // CUs without a block (small calls are latency)
      constexpr int G = decltype(g)::value, NV = decltype(nv)::value, U = NV <= 2 ? 2 : 1;
      constexpr int R = 64 / G * kW;
      const bool many = a.M >= (int64_t)R * U * device_cus();
      auto k = many ? (a.relu ? norm_bwd<T, W, G, NV, true, U> : norm_bwd<T, W, G, NV, false, U>)
                    : (a.relu ? norm_bwd<T, W, G, NV, true, 1> : norm_bwd<T, W, G, NV, false, 1>);
      const int64_t rows = many ? R * U : R, most = resident_blocks(k, kT);
      nblk = at_most((a.M + rows - 1) / rows, most < kPartRows ? most : kPartRows);
      hipLaunchKernelGGL(k, dim3((unsigned)nblk), dim3(kT), 0, s, a);
    });
    LPG_HIP(hipGetLastError());
  } else if (a.M > 0) {
    if (a.dx) {
      hipLaunchKernelGGL((norm_bwd_any<T, W>), dim3((unsigned)at_most(a.M, 1 << 16)), dim3(kT), 0, s, a);
      LPG_HIP(hipGetLastError());
    }
    if (a.part) {
      nblk = at_most(a.M, kPartRows);
      hipLaunchKernelGGL((norm_wgrad_any<T, W>), dim3((unsigned)((a.D + kT - 1) / kT), (unsigned)nblk), dim3(kT), 0, s,
                         a);
      LPG_HIP(hipGetLastError());
    }
  }
  if (a.part) {  // (no rows: the fold of no partials writes zeros)
    hipLaunchKernelGGL((norm_fold<W>), dim3((unsigned)((2 * a.D + kFoldC - 1) / kFoldC)), dim3(kFoldT), 0, s, nblk, a.D,
                       part, dw, db);
    LPG_HIP(hipGetLastError());
  }
  return LPG_OK;
}

}  // namespace
}  // namespace lpg

using namespace lpg;

// calls `f` with the element and weight types of the codes, or ends with LPG_ERR_INVALID
#define LPG_NORM_TYPES(what, f)                                                               \
  do {                                                                                        \
    if (dtype == LPG_F32 && wdtype == LPG_F32) return f(float, float);                        \
    if (dtype == LPG_BF16 && wdtype == LPG_F32) return f(__bf16, float);                      \
    if (dtype == LPG_BF16 && wdtype == LPG_BF16) return f(__bf16, __bf16);                    \
    if (dtype == LPG_F16 && wdtype == LPG_F32) return f(_Float16, float);                     \
    if (dtype == LPG_F16 && wdtype == LPG_F16) return f(_Float16, _Float16);                  \
    ::lpg::set_error(what ": dtype %d with weight dtype %d", (int)dtype, (int)wdtype);        \
    return LPG_ERR_INVALID;                                                                   \
  } while (0)

extern "C" lpg_status lpg_layer_norm_fwd(int32_t dtype, int32_t wdtype, int64_t M, int64_t D, const void *x, int64_t ldx,
                                         const void *w, const void *b, float eps, int32_t flags, void *y, int64_t ldy,
                                         float *mean, float *rstd, void *stream) {
  LPG_REQUIRE(M >= 0 && D >= 1 && D <= INT32_MAX, "lpg_layer_norm_fwd: need M >= 0, 1 <= D < 2^31");
  LPG_REQUIRE(ldx >= D && ldy >= D, "lpg_layer_norm_fwd: row strides below D");
  LPG_REQUIRE((flags & ~LPG_NORM_RELU) == 0, "lpg_layer_norm_fwd: unknown flags %d", (int)flags);
  LPG_REQUIRE(eps >= 0.f, "lpg_layer_norm_fwd: eps must not be negative");
  LPG_REQUIRE(!mean == !rstd, "lpg_layer_norm_fwd: mean and rstd come together");
  LPG_REQUIRE(M == 0 || (x && y), "lpg_layer_norm_fwd: NULL pointer");
  const FwdArgs a{M, D, ldx, ldy, x, w, b, y, mean, rstd, eps, (flags & LPG_NORM_RELU) ? 1 : 0};
#define F(T, W) M == 0 ? LPG_OK : fwd<T, W>(a, as_stream(stream))
  LPG_NORM_TYPES("lpg_layer_norm_fwd", F);
#undef F
}

extern "C" int64_t lpg_layer_norm_bwd_workspace_bytes(int64_t M, int64_t D) {
  if (M < 0 || D < 1) return -1;
  return (M < kPartRows ? (M < 1 ? 1 : M) : kPartRows) * 2 * D * (int64_t)sizeof(float);
}

extern "C" lpg_status lpg_layer_norm_bwd(int32_t dtype, int32_t wdtype, int64_t M, int64_t D, const void *x, int64_t ldx,
                                         const void *dy, int64_t lddy, const void *w, const void *b, const float *mean,
                                         const float *rstd, int32_t flags, void *dx, int64_t lddx, void *dw, void *db,
                                         void *workspace, void *stream) {
  LPG_REQUIRE(M >= 0 && D >= 1 && D <= INT32_MAX, "lpg_layer_norm_bwd: need M >= 0, 1 <= D < 2^31");
  LPG_REQUIRE(ldx >= D && lddy >= D && (!dx || lddx >= D), "lpg_layer_norm_bwd: row strides below D");
  LPG_REQUIRE((flags & ~LPG_NORM_RELU) == 0, "lpg_layer_norm_bwd: unknown flags %d", (int)flags);
  LPG_REQUIRE(M == 0 || (x && dy && mean && rstd), "lpg_layer_norm_bwd: NULL pointer");
  LPG_REQUIRE(!(dw || db) || workspace, "lpg_layer_norm_bwd: the weight gradients need the workspace");
  const BwdArgs a{M, D, ldx, lddy, lddx, x, dy, w, b, mean, rstd, dx, nullptr, (flags & LPG_NORM_RELU) ? 1 : 0};
#define F(T, W) \
  bwd<T, W>(a, static_cast<W *>(dw), static_cast<W *>(db), static_cast<float *>(workspace), as_stream(stream))
  LPG_NORM_TYPES("lpg_layer_norm_bwd", F);
#undef F
}
