// The fully connected layer in 8-bit integers, for evaluation:
//
//   top_m = max_k |x_mk|,  q_mk = round_half_even(127 x_mk / top_m),  x = [x1 | x2] (aggregate | own features)
//   y_mn = act((sum_k q_mk w_nk) (top_m / 127) ws_n + b_n)
//
// w int8 with a scale ws an output channel, quantised ahead.  The sum is exact (32-bit integers, K <=
// 131072), so every variant below gives the same bits.
//
// The quotient decides borders of whole numbers, so it is decided exactly: x (127 / top) in fp32 is off by
// less than 127 * 2^-23 < 2^-15.9; where it lies within 2^-15 of a border between two codes (one element
// in 16000), the border's side is found from the exact products instead (at_border).
//
// quant_rows_held, quant_rows: HBM-bound, x in, q out; 8 to 64 lanes hold a row in registers, rows longer than those
// hold take a wave and two passes (the second from cache).  32768 x 2048 fp16: 33 us, 6.1 TB/s (q stays in cache).
// fc_i8: MFMA- and LDS-bound (v_mfma_i32_16x16x64_i8), the k loop of the 16-bit kernel (fc_bf16.hip fc_bf16_p) on
// bytes: 128-byte k tiles staged by buffer_load ... lds into a swizzled image, two buffers (four in the small tile),
// one barrier a tile in its middle, fragment reads one half tile ahead, transposed fragments (W x A^T: a lane holds
// four consecutive columns of one row), stores straight from registers.  16384 x 2048, K = 4096: 109 us, 2.5 POPS;
// 100 K x 1024, K = 2048: 184 us, 2.3 (170 of it the 256 tile, 13 the 128 tile of the last rows), with its codes 276.  160
// k tiles of five output tiles in a row take a block 255 us, 1.6 us each with the stores, of which the MFMAs 0.86 at 2.4
// GHz; the first round's loads and the last one's stores are not hidden.
// fc_i8_row, fc_i8_some: few rows are bound by latency -- the second launch, the k loop's barriers -- and by
// w's bytes: every block quantises its rows into LDS itself, its first loads of w in flight meanwhile.  One row of
// 2048 to 1024 columns: 3.8 us.
#include "common.h"
#include "fc_common.h"

#include <type_traits>

namespace lpg {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int BK = 128;  // bytes of a k tile
constexpr float kTiny = 0x1p-100f;

__device__ __forceinline__ int swz(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }

// The row's factor 127 / top and scale top / 127, from the bits of its largest |x| (as unsigned numbers, so
// a NaN or an infinity is on top).
struct RowScale {
  float top, inv, scale;
  __device__ __forceinline__ explicit RowScale(uint32_t bits) {
    top = __uint_as_float(bits);
    const bool bad = bits >= 0x7f800000u, live = !bad && top >= kTiny;
    inv = live ? 127.f / top : 0.f;
    scale = bad ? __uint_as_float(0x7fc00000u) : (live ? top / 127.f : 0.f);
  }
};

// Which side of the border k + 1/2 the quotient 127 |x| / top lies on, exactly: the sign of 254 |x| - (2 k + 1)
// top, both products with their rounding errors (fma), their difference exact near the border.
__device__ __forceinline__ int at_border(float x, float top, float t) {
  const float big = top > 0x1p64f ? 0x1p-32f : 1.f;  // (no product past the range)
  const float ax = fabsf(x) * big, at = top * big, k = floorf(fabsf(t)), b = 2.f * k + 1.f;
  const float r = 254.f * ax, p = b * at;
  const float d = (r - p) + (__builtin_fmaf(254.f, ax, -r) - __builtin_fmaf(b, at, -p));
  const int n = (int)k;
  const int q = n + (d > 0.f ? 1 : (d < 0.f ? 0 : (n & 1)));
  return x < 0.f ? -q : q;
}

// The codes of f, packed four to a word.  x inv + 1.5 * 2^23 leaves the nearest whole number (halves to even) in
// the low byte of its bits, two's complement; what it lost tells how near a border was.  (inv = 0: zeros of
// finite f.)
template <int N>
__device__ __forceinline__ void quant(const float (&f)[N], const RowScale &s, uint32_t (&q)[(N + 3) / 4]) {
  constexpr float kMagic = 12582912.f;
  uint32_t c[N];
  float far = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float y = __builtin_fmaf(f[j], s.inv, kMagic);
    far = fmaxf(far, fabsf(__builtin_fmaf(f[j], s.inv, kMagic - y)));
    c[j] = __float_as_uint(y);
  }
  if (far > 0.5f - 0x1p-15f) {
#pragma unroll
    for (int j = 0; j < N; ++j) c[j] = (uint32_t)at_border(f[j], s.top, f[j] * s.inv);
  }
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j)
      q[j] = __builtin_amdgcn_perm(c[4 * j + 1], c[4 * j], 0x0c0c0400u) |
             __builtin_amdgcn_perm(c[4 * j + 3], c[4 * j + 2], 0x04000c0cu);
  } else {
    static_assert(N == 1, "vectors of four, or one");
    q[0] = c[0] & 0xffu;
  }
}

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// the largest over each G lanes, in all of them
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false));
}
template <int G>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  static_assert(G >= 8 && G <= 64, "8 to 64 lanes");
  v = dpp_max<0xB1>(v);   // quad_perm 1,0,3,2
  v = dpp_max<0x4E>(v);   // quad_perm 2,3,0,1
  v = dpp_max<0x141>(v);  // row_half_mirror
  if constexpr (G > 8) v = dpp_max<0x140>(v);  // row_mirror
  if constexpr (G > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
  }
  if constexpr (G > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(r[0], r[1]);
  }
  return v;
}

// The largest |x| of 16-byte vectors, kept as the types' own bits (their order is that of |x|, NaN on top): two
// 16-bit elements an operation.
template <typename T>
struct Top {
  typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
  u16x8 m = {0, 0, 0, 0, 0, 0, 0, 0};
  __device__ __forceinline__ void add(u32x4 v) {
    if constexpr (sizeof(T) == 2) {
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x8, v & 0x7fff7fffu));
    } else {
      m = __builtin_bit_cast(u16x8, __builtin_elementwise_max(__builtin_bit_cast(u32x4, m), v & 0x7fffffffu));
    }
  }
  __device__ __forceinline__ uint32_t bits() const {  // as fp32's
    uint32_t top = 0;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, abs_bits((float)__builtin_bit_cast(T, (unsigned short)m[j])));
    } else {
      const u32x4 w = __builtin_bit_cast(u32x4, m);
      top = max(max(w[0], w[1]), max(w[2], w[3]));
    }
    return top;
  }
};

template <typename T>
__device__ __forceinline__ void unpack(u32x4 v, float (&f)[16 / sizeof(T)]) {
  T t[16 / sizeof(T)];
  __builtin_memcpy(t, &v, 16);
#pragma unroll
  for (int j = 0; j < (int)(16 / sizeof(T)); ++j) f[j] = (float)t[j];
}

// 16 bytes at any element alignment, past the caches or through them
typedef unsigned int u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
template <bool PAST, typename T>
__device__ __forceinline__ u32x4 ld16(const T *p) {
  u32x4 v;
  if constexpr (PAST)
    v = __builtin_nontemporal_load(reinterpret_cast<const std::conditional_t<sizeof(T) == 2, u32x4_at2, u32x4_at4> *>(p));
  else __builtin_memcpy(&v, p, 16);
  return v;
}

// the largest |x| bits of the n elements at p, taken by threads t of nt
template <typename T>
__device__ __forceinline__ uint32_t part_max(const T *p, int n, int t, int nt) {
  constexpr int V = 16 / sizeof(T);
  Top<T> top;
  const int nv = n / V;
  for (int i = t; i < nv; i += nt) {
    u32x4 v;
    __builtin_memcpy(&v, p + i * V, 16);
    top.add(v);
  }
  const int at = nv * V + t;
  return max(top.bits(), at < n ? abs_bits((float)p[at]) : 0u);  // (fewer than V <= nt are left)
}

// ... and their codes, to q (any alignment)
template <typename T>
__device__ __forceinline__ void part_quant(const T *p, int n, int t, int nt, const RowScale &s, int8_t *q) {
  constexpr int V = 16 / sizeof(T);
  const int nv = n / V;
  for (int i = t; i < nv; i += nt) {
    u32x4 v;
    float f[V];
    uint32_t o[V / 4];
    __builtin_memcpy(&v, p + i * V, 16);
    unpack<T>(v, f);
    quant<V>(f, s, o);
    __builtin_memcpy(q + i * V, o, V);
  }
  const int at = nv * V + t;
  if (at < n) {
    const float f[1] = {(float)p[at]};
    uint32_t o[1];
    quant<1>(f, s, o);
    q[at] = (int8_t)o[0];
  }
}

// zeros from q[k] to q[end], q and end multiples of 16, by lanes l of G
__device__ __forceinline__ void zero_from(int8_t *q, int k, int end, int l, int G) {
  const int k16 = (k + 15) & ~15;
  for (int i = k + l; i < k16; i += G) q[i] = 0;
  for (int i = k16 + l * 16; i < end; i += G * 16) *reinterpret_cast<u32x4 *>(q + i) = u32x4{0u, 0u, 0u, 0u};
}

struct QuantArgs {
  int64_t M, ldx, ldx2, ldq;
  int K1, K2;
  const void *x, *x2;
  int8_t *q;
  float *scale;
  int past;  // x is read past the caches
};

template <typename T>
__global__ __launch_bounds__(256) void quant_rows(QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.M) return;
  const T *x = static_cast<const T *>(a.x) + row * a.ldx;
  const T *x2 = a.K2 ? static_cast<const T *>(a.x2) + row * a.ldx2 : nullptr;
  int8_t *q = a.q + row * a.ldq;
  uint32_t top = part_max(x, a.K1, lane, 64);
  if (a.K2) top = max(top, part_max(x2, a.K2, lane, 64));
  const RowScale s(lanes_max<64>(top));
  part_quant(x, a.K1, lane, 64, s, q);
  if (a.K2) part_quant(x2, a.K2, lane, 64, s, q + a.K1);
  zero_from(q, a.K1 + a.K2, (int)a.ldq, lane, 64);
  if (lane == 0) a.scale[row] = s.scale;
}

// A row of at most G NV vectors, held in the registers of G lanes: all its loads in flight together, read once.
// Vector i of the row is a vector of x or, from n1 on, of x2; where the columns are no multiple of V the last one
// starts early, to end with them (the elements it shares with the one before get the same codes twice).  REST: the
// columns that fill no vector (2 V - 2 at most) are single elements of the lanes instead, for K1 or K2 below V.
template <typename T, int G, int NV, bool REST>
struct HeldRow {
  static constexpr int V = 16 / sizeof(T), NR = REST ? (2 * V - 2 + G - 1) / G : 0;
  u32x4 v[NV];
  float rest[NR ? NR : 1];
  static __device__ __forceinline__ int count(int K) { return REST ? K / V : (K + V - 1) / V; }
  // where vector i of K columns starts
  static __device__ __forceinline__ int start(int i, int K) { return REST || i * V + V <= K ? i * V : K - V; }
  template <bool PAST = false>
  __device__ __forceinline__ void load(const T *x, int K1, const T *x2, int K2, int l) {
    const int n1 = count(K1), n2 = count(K2), r1 = K1 % V, r2 = K2 % V;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = k * G + l;
      v[k] = u32x4{0u, 0u, 0u, 0u};
      if (i < n1 + n2) v[k] = ld16<PAST>(i < n1 ? x + start(i, K1) : x2 + start(i - n1, K2));
    }
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const int i = k * G + l;
      rest[k] = i < r1 ? (float)x[n1 * V + i] : (i < r1 + r2 ? (float)x2[n2 * V + i - r1] : 0.f);
    }
  }
  __device__ __forceinline__ uint32_t top() const {  // of the row
    Top<T> t;
#pragma unroll
    for (int k = 0; k < NV; ++k) t.add(v[k]);
    uint32_t m = t.bits();
#pragma unroll
    for (int k = 0; k < NR; ++k) m = max(m, abs_bits(rest[k]));
    return lanes_max<G>(m);
  }
  __device__ __forceinline__ void store(const RowScale &s, int8_t *q, int K1, int K2, int l) const {
    const int n1 = count(K1), n2 = count(K2), r1 = K1 % V, r2 = K2 % V;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = k * G + l;
      if (i >= n1 + n2) continue;
      float f[V];
      uint32_t o[V / 4];
      unpack<T>(v[k], f);
      quant<V>(f, s, o);
      __builtin_memcpy(q + (i < n1 ? start(i, K1) : K1 + start(i - n1, K2)), o, V);
    }
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const int i = k * G + l;
      if (i < r1 + r2) {
        const float f[1] = {rest[k]};
        uint32_t o[1];
        quant<1>(f, s, o);
        q[i < r1 ? n1 * V + i : K1 + n2 * V + i - r1] = (int8_t)o[0];
      }
    }
  }
};

template <typename T, int G, int NV, bool REST = false>
__global__ __launch_bounds__(256) void quant_rows_held(QuantArgs a) {
  const int l = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G, at = row < a.M ? row : a.M - 1;
  HeldRow<T, G, NV, REST> h;
  const T *x = static_cast<const T *>(a.x) + at * a.ldx, *x2 = a.K2 ? static_cast<const T *>(a.x2) + at * a.ldx2 : nullptr;
  if (a.past) h.template load<true>(x, a.K1, x2, a.K2, l);
  else h.load(x, a.K1, x2, a.K2, l);
  const RowScale s(h.top());  // (of every lane: rows past the end are the last one again)
  if (row >= a.M) return;
  int8_t *q = a.q + row * a.ldq;
  h.store(s, q, a.K1, a.K2, l);
  zero_from(q, a.K1 + a.K2, (int)a.ldq, l, G);
  if (l == 0) a.scale[row] = s.scale;
}

struct FcArgs {
  int64_t M, N, ldq, ldw, ldy;
  int K;
  const int8_t *q, *w;
  const float *scale, *wscale, *bias;
  void *y;
  int64_t mt, nt;
  float lo;
  int past;  // y is stored past the caches
};

// 64 floats from p on (those past its n bytes: zeros) to LDS
__device__ __forceinline__ void dma4(uint64_t p, uint32_t n, float *lds, uint32_t voff) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((address_space(3))) void lds_v;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)p), hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void *>(((uint64_t)hi << 32) | lo), (short)0, (int)__builtin_amdgcn_readfirstlane(n), 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_v *)lds, 4, voff, 0, 0, 0);
#endif
}

// lo: 0 with the ReLU, -infinity without (a NaN stays one)
__device__ __forceinline__ float finish(int acc, float s, float ws, float b, float lo) {
  return __builtin_elementwise_maximum(((float)acc * s) * ws + b, lo);
}
template <typename T>
__device__ __forceinline__ uint32_t pair(float a, float b) {  // as two 16-bit numbers
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef T t16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), t16x2));
}

// WM x WN waves, each FM x FN fragments of 16 x 16, NB tiles of k in LDS.  ON: a block takes output tiles blockIdx.x,
// + gridDim.x, ... in one stream of k tiles, those of the next output tile in flight while this one is stored; else
// blockIdx.x is the only one.
template <typename T, int WM, int WN, int FM, int FN, int NB, bool ON>
__global__ __launch_bounds__(64 * WM * WN, 2) void fc_i8(FcArgs a) {
  constexpr int NW = WM * WN;
  constexpr int BM = WM * FM * 16, BN = WN * FN * 16;
  constexpr int A_BYTES = BM * BK, TILE_BYTES = A_BYTES + BN * BK;
  constexpr int PA = BM / 8, PT = PA + BN / 8, PPW = PT / NW;  // 1-KiB pieces: A, all, a wave
  static_assert(PA % NW == 0 && PT % NW == 0 && NW % 2 == 0 && PA % 2 == 0, "whole pieces a wave, of one row parity");
  // Behind the k tiles: the output tiles' row scales, channel scales and biases, staged with their first k tile.  Where a
  // tile has one k tile that is NB tiles ahead, before the barrier that all waves' stores of the tile before are behind:
  // NB + 2 tiles' are alive.  One array for all: beside a second one the compiler tells apart what the DMA writes, and
  // waits for it before every read.
  constexpr int SC = BM + 2 * BN, NS = ON ? NB + 2 : 1;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[NB * TILE_BYTES + NS * SC * 4];
  float *const sc = reinterpret_cast<float *>(smem + NB * TILE_BYTES);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int nk = (a.K + BK - 1) / BK, k16 = (a.K + 15) / 16 * 16;
  const uint32_t nwg = (uint32_t)(a.mt * a.nt), nt = (uint32_t)a.nt;

  // XCD-aware order: the blocks of one XCD take a contiguous range of (m, n) tiles
  const auto origin = [&](uint32_t tile, int64_t &m0, int64_t &n0) {
    const uint32_t xcd = tile % 8, q8 = nwg / 8, rr = nwg % 8;
    const uint32_t at = (xcd < rr ? xcd * (q8 + 1) : rr * (q8 + 1) + (xcd - rr) * q8) + tile / 8;
    m0 = (int64_t)(at / nt) * BM;
    n0 = (int64_t)(at % nt) * BN;
  };

  uint32_t vo[PPW];
#pragma unroll
  for (int p = 0; p < PPW; ++p) {
    const int q = wave + NW * p;
    const int row = (q < PA ? q : q - PA) * 8 + (lane >> 3);
    vo[p] = (uint32_t)(row * (q < PA ? a.ldq : a.ldw) + swz(row, lane & 7) * 16);
  }
  const int chunk_at = swz((wave & 1) * 8 + (lane >> 3), lane & 7) * 16;  // of all this wave's pieces

  // The next k tile to stage: of output tile s_tile, its number s_k.  Descriptors from row m0 of q / row n0 of w,
  // ending with the tile's last row: the lane offsets of rows past it are past the range and read zeros.  q's rows
  // hold zeros from K to the k tile's end; a row of w may end before it does (the lanes of those chunks get an
  // offset past the range).  Past the last one: the same instructions with empty ranges.
  uint32_t s_tile = blockIdx.x, s_scales = 0;
  int s_k = 0;
  uint64_t pa = 0, pw = 0;
  uint32_t na = 0, nw = 0;
  const auto open_tile = [&]() {  // of s_tile, for its first k tile
    const bool some = s_tile < nwg;
    int64_t m0, n0;
    origin(some ? s_tile : 0, m0, n0);
    const int64_t mrows = a.M - m0 < BM ? a.M - m0 : BM, ncols = a.N - n0 < BN ? a.N - n0 : BN;
    pa = (uint64_t)(a.q + m0 * a.ldq);
    pw = (uint64_t)(a.w + n0 * a.ldw);
    na = some ? (uint32_t)((mrows - 1) * a.ldq + nk * BK) : 0u;
    nw = some ? (uint32_t)((ncols - 1) * a.ldw + k16) : 0u;
    for (int i = wave; i < SC / 64; i += NW) {
      const bool row = i < BM / 64, col = !row && i < (BM + BN) / 64;
      const float *p = row ? a.scale + m0 : (col ? a.wscale + n0 : a.bias + (a.bias ? n0 : 0));
      const int at = (row ? i : (col ? i - BM / 64 : i - (BM + BN) / 64)) * 64;
      const uint32_t n = some && (row || col || a.bias) ? (uint32_t)(row ? mrows : ncols) * 4 : 0u;
      dma4((uint64_t)p, n, sc + s_scales * SC + i * 64, (uint32_t)(at + lane) * 4);
    }
    s_scales = s_scales + 1 < NS ? s_scales + 1 : 0;
    s_k = 0;
    s_tile = some ? s_tile + gridDim.x : nwg;
  };
  const auto stage = [&](int b) {
    unsigned char *base = smem + b * TILE_BYTES;
    const bool in = chunk_at < k16 - s_k * BK;
#pragma unroll
    for (int p = 0; p < PPW; ++p) {
      const int q = wave + NW * p;
      if (p < PA / NW) dma16(pa, ON || s_k < nk ? na : 0u, base + q * 1024, vo[p], s_k * BK);
      else dma16(pw, ON || s_k < nk ? nw : 0u, base + q * 1024, in ? vo[p] : 0x7fffff00u, s_k * BK);
    }
    ++s_k;
  };

  i32x4 acc[FM][FN];
  const int fr = lane & 15, fq = lane >> 4;
  auto rd = [&](int b, int s, i32x4(&av)[FM], i32x4(&bv)[FN]) {  // half s (64 k) of buffer b
    const unsigned char *As = smem + b * TILE_BYTES, *Bs = As + A_BYTES;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int row = wm * FM * 16 + i * 16 + fr;
      av[i] = *reinterpret_cast<const i32x4 *>(As + row * BK + swz(row, s * 4 + fq) * 16);
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int row = wn * FN * 16 + j * 16 + fr;
      bv[j] = *reinterpret_cast<const i32x4 *>(Bs + row * BK + swz(row, s * 4 + fq) * 16);
    }
  };
  auto mma = [&](const i32x4(&av)[FM], const i32x4(&bv)[FN]) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bv[j], av[i], acc[i][j], 0, 0, 0);
  };
  // this wave's DMA landed, but for the latest `later` operations, and its fragment reads returned; then all waves
  auto arrive = [&](auto later) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(later)::value) : "memory");
  };
  auto meet = [&]() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  T *y = static_cast<T *>(a.y);
  i32x4 a0[FM], b0[FN], a1[FM], b1[FN];
  static_assert((NB - 1) * PPW < 64, "vmcnt counts to 63");
#pragma unroll
  for (int t = 0; t < NB; ++t) {
    if (t == 0 || (ON && s_k == nk)) open_tile();
    stage(t);
  }
  __builtin_amdgcn_sched_barrier(0);
  arrive(std::integral_constant<int, (NB - 1) * PPW>());
  meet();
  rd(0, 0, a0, b0);
  constexpr int NR = FM + FN, NM = FM * FN;
  // stores of a whole tile, which the first wait after them leaves out (its k tile was staged before them)
  constexpr int STORES = FM * FN / (sizeof(T) == 2 ? 2 : 1), AFTER = (NB - 2) * PPW + STORES;
  static_assert(AFTER < 64, "vmcnt counts to 63");
  int b = 0, scales = 0;
  bool stored = false;  // a whole tile was, since the last wait
  const auto step = [&]() {  // one k tile
    __builtin_amdgcn_sched_barrier(0);
    rd(b, 1, a1, b1);
    mma(a0, b0);
    __builtin_amdgcn_sched_barrier(0);
    if (ON && stored) arrive(std::integral_constant<int, AFTER>());
    else arrive(std::integral_constant<int, (NB - 2) * PPW>());
    stored = false;
    meet();  // the next k tile landed; every wave is done reading buffer b
    stage(b);
    b = b + 1 < NB ? b + 1 : 0;
    rd(b, 0, a0, b0);
    mma(a1, b1);
    if constexpr (NM > PPW + NR) {  // DMA pieces, then the next tile's reads, one a MFMA
#pragma unroll
      for (int k = 0; k < PPW; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, NM - PPW - NR, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (uint32_t tile = blockIdx.x; tile < nwg; tile += gridDim.x) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    if constexpr (ON) {
#pragma unroll 1
      for (int t = 0; t < nk; ++t) {
        if (s_k == nk) open_tile();
        step();
      }
    } else {
      for (int t = 0; t + 1 < nk; ++t) step();
      rd(b, 1, a1, b1);
      mma(a0, b0);
      mma(a1, b1);
    }

    // a lane holds row 16 i + er, columns 16 j + 4 eq .. + 3 of its wave's part (its place found anew: nothing of the
    // epilogue is kept in registers through the k loop)
    int el = lane;
    asm volatile("" : "+v"(el));
    const int er = el & 15, eq = el >> 4;
    int64_t m0, n0;
    origin(tile, m0, n0);
    stored = m0 + BM <= a.M && n0 + BN <= a.N;
    const int64_t r0 = m0 + wm * FM * 16, c0 = n0 + wn * FN * 16;
    const float *rs = sc + scales * SC + wm * FM * 16 + er;
    const float *cs = sc + scales * SC + BM + wn * FN * 16 + eq * 4, *cb = cs + BN;
    scales = scales + 1 < NS ? scales + 1 : 0;
    float ws[FN][4], bb[FN][4];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) ws[j][r] = cs[j * 16 + r], bb[j][r] = cb[j * 16 + r];
    // all stores of the wave's part: of a whole tile past the caches or through them, or whatever exists of it
    const auto store = [&](auto how) {
      constexpr bool WHOLE = decltype(how)::value < 2, PAST = decltype(how)::value == 0;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int64_t row = r0 + i * 16 + er;
        const float s = rs[i * 16];
        const auto v = [&](int j, int r) { return finish(acc[i][j][r], s, ws[j][r], bb[j][r], a.lo); };
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            const int64_t c = c0 + j * 16 + eq * 4;
            const float out[4] = {v(j, 0), v(j, 1), v(j, 2), v(j, 3)};
            T *p = y + row * a.ldy + c;
            if constexpr (PAST) {
              u32x4 o;
              __builtin_memcpy(&o, out, 16);
              __builtin_nontemporal_store(o, reinterpret_cast<u32x4 *>(p));
            } else if (WHOLE || (row < a.M && c + 4 <= a.N)) {
              __builtin_memcpy(p, out, 16);
            } else if (row < a.M && c < a.N) {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (c + r < a.N) p[r] = out[r];
            }
          }
        } else {
          // Lanes eq = 0 .. 3 hold columns 4 eq .. + 3 of fragments j and j + 1; two exchanges between them leave
          // columns 8 eq .. + 7 of the 32 in each: rows leave as 16-byte stores, 64 bytes a row
          static_assert(FN % 2 == 0, "fragments in pairs");
#pragma unroll
          for (int j = 0; j < FN; j += 2) {
            u32x4 out;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              const auto x = __builtin_amdgcn_permlane32_swap(pair<T>(v(j, 2 * d), v(j, 2 * d + 1)),
                                                              pair<T>(v(j + 1, 2 * d), v(j + 1, 2 * d + 1)), false, false);
              const auto z = __builtin_amdgcn_permlane16_swap(x[0], x[1], false, false);
              out[d] = z[0];
              out[2 + d] = z[1];
            }
            const int64_t c = c0 + j * 16 + eq * 8;
            // (a store as soon as its numbers are: 16384 x 1024, K = 128 14.8 -> 12.9 us)
            __builtin_amdgcn_sched_barrier(0);
            T *p = y + row * a.ldy + c;
            if constexpr (PAST) {
              __builtin_nontemporal_store(out, reinterpret_cast<u32x4 *>(p));
            } else if (WHOLE || (row < a.M && c + 8 <= a.N)) {
              __builtin_memcpy(p, &out, 16);
            } else if (row < a.M && c < a.N) {
              T e[8];
              __builtin_memcpy(e, &out, 16);
#pragma unroll
              for (int r = 0; r < 8; ++r)
                if (c + r < a.N) p[r] = e[r];
            }
          }
        }
      }
    };
    if (stored && a.past) store(std::integral_constant<int, 0>());
    else if (stored) store(std::integral_constant<int, 1>());
    else store(std::integral_constant<int, 2>());
    if constexpr (!ON) break;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the empty DMAs have landed before the LDS is another block's)
}

struct RowsArgs {
  int64_t M, N, ldx, ldx2, ldw, ldy;
  int K1, K2;
  const void *x, *x2;
  const int8_t *w;
  const float *wscale, *bias;
  void *y;
  float lo;
};

// One row: every block quantises it into LDS, then a wave a column.
constexpr int kRowBytes = 32 * 1024;  // its longest row
template <typename T>
__global__ __launch_bounds__(256) void fc_i8_row(RowsArgs a) {
  extern __shared__ __attribute__((aligned(16))) int8_t qs[];  // kp bytes
  __shared__ uint32_t red[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int K = a.K1 + a.K2, k16 = (K + 15) / 16, kp = (K + 1023) / 1024 * 1024;
  const int64_t n = (int64_t)blockIdx.x * 4 + wave;
  const i32x4 *w = reinterpret_cast<const i32x4 *>(a.w + (n < a.N ? n : a.N - 1) * a.ldw);
  // the first chunks of this wave's column, in flight while the row is quantised
  constexpr int P = 4;
  i32x4 pre[P];
#pragma unroll
  for (int u = 0; u < P; ++u) pre[u] = u * 64 + lane < k16 ? w[u * 64 + lane] : i32x4{0, 0, 0, 0};
  const T *x = static_cast<const T *>(a.x), *x2 = static_cast<const T *>(a.x2);
  uint32_t top = part_max(x, a.K1, (int)threadIdx.x, 256);
  if (a.K2) top = max(top, part_max(x2, a.K2, (int)threadIdx.x, 256));
  top = lanes_max<64>(top);
  if (lane == 0) red[wave] = top;
  __syncthreads();
  const RowScale s(max(max(red[0], red[1]), max(red[2], red[3])));
  part_quant(x, a.K1, (int)threadIdx.x, 256, s, qs);
  if (a.K2) part_quant(x2, a.K2, (int)threadIdx.x, 256, s, qs + a.K1);
  for (int k = K + (int)threadIdx.x; k < kp; k += 256) qs[k] = 0;
  __syncthreads();
  int acc = 0;
  const auto dot = [&](i32x4 v, int c) {
    const i32x4 q = *reinterpret_cast<const i32x4 *>(qs + c * 16);
#pragma unroll
    for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_sdot4(v[r], q[r], acc, false);
  };
#pragma unroll
  for (int u = 0; u < P; ++u)
    if (u * 64 < k16) dot(pre[u], u * 64 + lane);  // (chunks past k16 are zeros; q is padded to whole kilobytes)
  for (int c = P * 64 + lane; c < k16; c += 64) dot(w[c], c);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
  if (lane == 0 && n < a.N)
    static_cast<T *>(a.y)[n] = (T)finish(acc, s.scale, a.wscale[n], a.bias ? a.bias[n] : 0.f, a.lo);
}

// Some rows: a block of eight waves takes 16 rows and 128 columns.  It quantises its rows into LDS, two a wave
// (every block of the row tile again), then each wave runs 16 columns with w's fragments straight from memory,
// eight k steps in flight: no barrier and no second launch, which is what a call of this size consists of.
constexpr int kSomeK = 1024;  // its longest row (16 of them and 16 bytes each in LDS)
constexpr int kSomeN = 128;
template <typename T, int NV>
__global__ __launch_bounds__(512) void fc_i8_some(RowsArgs a) {
  extern __shared__ __attribute__((aligned(16))) int8_t qs[];  // 16 rows of `pitch` bytes
  __shared__ float scales[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int P = 8;  // k steps of 64 bytes in flight
  const int K = a.K1 + a.K2, k16 = (K + 15) / 16 * 16, ks = (K + P * 64 - 1) / (P * 64) * P;
  const int pitch = ks * 64 + 16;  // (rows 16 bytes apart in the banks)
  const int64_t m0 = (int64_t)blockIdx.y * 16, n0 = (int64_t)blockIdx.x * kSomeN + wave * 16;
  const int fr = lane & 15, fq = lane >> 4;
  HeldRow<T, 64, NV, true> h[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = m0 + wave * 2 + i < a.M ? m0 + wave * 2 + i : a.M - 1;
    h[i].load(static_cast<const T *>(a.x) + row * a.ldx, a.K1,
              a.K2 ? static_cast<const T *>(a.x2) + row * a.ldx2 : nullptr, a.K2, lane);
  }
  const int8_t *w = a.w + (n0 + fr < a.N ? n0 + fr : a.N - 1) * a.ldw;
  // this lane's four columns: 4 fq .. + 3 of the wave's 16 (the last channel in place of those past N)
  float ws[4], bb[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t c = n0 + fq * 4 + r < a.N ? n0 + fq * 4 + r : a.N - 1;
    ws[r] = a.wscale[c];
    bb[r] = a.bias ? a.bias[c] : 0.f;
  }
  const auto load = [&](int t, i32x4(&v)[P]) {
#pragma unroll
    for (int u = 0; u < P; ++u) {
      const int k = (t + u) * 64 + fq * 16;
      v[u] = *reinterpret_cast<const i32x4 *>(w + (k < k16 ? k : 0));  // (past K: anything, q is zero there)
    }
  };
  i32x4 next[P];
  load(0, next);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const RowScale s(h[i].top());
    int8_t *q = qs + (wave * 2 + i) * pitch;
    h[i].store(s, q, a.K1, a.K2, lane);
    for (int k = K + lane; k < ks * 64; k += 64) q[k] = 0;
    if (lane == 0) scales[wave * 2 + i] = s.scale;
  }
  __syncthreads();
  i32x4 acc[2] = {i32x4{0, 0, 0, 0}, i32x4{0, 0, 0, 0}};
  for (int t = 0; t < ks; t += P) {
    i32x4 v[P], q[P];
#pragma unroll
    for (int u = 0; u < P; ++u) v[u] = next[u];
    if (t + P < ks) load(t + P, next);
#pragma unroll
    for (int u = 0; u < P; ++u) q[u] = *reinterpret_cast<const i32x4 *>(qs + fr * pitch + (t + u) * 64 + fq * 16);
#pragma unroll
    for (int u = 0; u < P; ++u) acc[u & 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[u], q[u], acc[u & 1], 0, 0, 0);
  }
  // a lane holds row fr of the tile and its four columns
  const int64_t row = m0 + fr, c = n0 + fq * 4;
  if (row >= a.M) return;
  T *y = static_cast<T *>(a.y) + row * a.ldy + c;
  T v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = (T)finish(acc[0][r] + acc[1][r], scales[fr], ws[r], bb[r], a.lo);
  if (c + 4 <= a.N) {
    __builtin_memcpy(y, v, sizeof(v));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (c + r < a.N) y[r] = v[r];
  }
}

template <typename T, int WM, int WN, int FM, int FN, int NB>
void launch_fc(FcArgs a, hipStream_t s) {
  a.mt = (a.M + WM * FM * 16 - 1) / (WM * FM * 16);
  a.nt = (a.N + WN * FN * 16 - 1) / (WN * FN * 16);
  const int64_t n = a.mt * a.nt;
  // The 256 tile leaves a CU room for one block: where there is more than a round of them, as many blocks as CUs that
  // go on (100 K x 1024, K = 2048 212 -> 193 us; one round 36.5 without, 37.9 with it).  Two blocks of the 128 tile
  // fill each other's time of the stores, but for short sums in many rounds (147 K x 1600, K = 38 174 -> 146; 60 K x
  // 384, K = 128, 2.7 rounds, 14.6 without, 15.4 with it).
  constexpr int BM = WM * FM * 16;
  if constexpr (BM >= 128) {
    const int64_t blocks = (BM == 256 ? 1 : 2) * device_cus();
    if (n > blocks * (BM == 256 ? 1 : 4)) {
      hipLaunchKernelGGL((fc_i8<T, WM, WN, FM, FN, NB, true>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((fc_i8<T, WM, WN, FM, FN, NB, false>), dim3((unsigned)n), dim3(64 * WM * WN), 0, s, a);
}

int64_t tiles(const FcArgs &a, int64_t b) { return ((a.M + b - 1) / b) * ((a.N + b - 1) / b); }

template <typename T>
lpg_status run_fc(const FcArgs &a, hipStream_t s) {
  // The largest tile that still gives most CUs a block; but 128 columns where half of the last 256 would be
  // empty, if that is all there are (100 K x 100, K = 100: 32.5 us against 43.8; x 128, K = 2048 164 and 176) or
  // the sums are short (60 K x 333, K = 512 58 and 65; K = 2048 145 and 139).
  const int64_t n128 = (a.N + 127) / 128;
  if (tiles(a, 256) >= 192 && (n128 % 2 == 0 || (n128 > 1 && a.K > 1024))) {
    // One block a CU: the last round of blocks takes as long as a full one.  Where it would be at most half
    // full, its rows go to the 128 tile (a quarter of the work, two blocks a CU): 34816 x 1024, K = 1024 (an eighth of
    // a round left) 54 -> 49 us, 24576 x 1024, K = 2048 (half) 56 -> 50; 26624 rows (five eighths) 57 -> 61.
    const int64_t cus = device_cus(), nt = (a.N + 255) / 256, n = tiles(a, 256), mt = n / cus * cus / nt;
    const int64_t m1 = mt * 256;
    if (n % cus != 0 && n % cus * 2 <= cus && mt > 0 && m1 < a.M) {
      FcArgs head = a, tail = a;
      head.M = m1;
      tail.M = a.M - m1;
      tail.q += m1 * a.ldq;
      tail.scale += m1;
      tail.y = static_cast<T *>(a.y) + m1 * a.ldy;
      launch_fc<T, 2, 4, 8, 4, 2>(head, s);
      LPG_HIP(hipGetLastError());
      launch_fc<T, 2, 2, 4, 4, 2>(tail, s);
    } else {
      launch_fc<T, 2, 4, 8, 4, 2>(a, s);
    }
  } else if (tiles(a, 128) >= 192) launch_fc<T, 2, 2, 4, 4, 2>(a, s);
  else launch_fc<T, 2, 2, 2, 2, 4>(a, s);
  LPG_HIP(hipGetLastError());
  return LPG_OK;
}

template <typename T>
lpg_status run_rows(const RowsArgs &a, hipStream_t s) {
  const int K = a.K1 + a.K2;
  if (a.M == 1) {
    hipLaunchKernelGGL(fc_i8_row<T>, dim3((unsigned)((a.N + 3) / 4)), dim3(256), (K + 1023) / 1024 * 1024, s, a);
  } else {
    constexpr int V = 16 / sizeof(T);
    const int nv = (a.K1 / V + a.K2 / V + 63) / 64;
    const auto go = [&](auto k) {
      hipLaunchKernelGGL(k, dim3((unsigned)((a.N + kSomeN - 1) / kSomeN), (unsigned)((a.M + 15) / 16)), dim3(512),
                         16 * ((K + 511) / 512 * 512 + 16), s, a);
    };
    if (nv <= 1) go(fc_i8_some<T, 1>);
    else if (nv <= 2 || sizeof(T) == 2) go(fc_i8_some<T, 2>);  // (16 bits: at most 128 vectors)
    else if constexpr (sizeof(T) == 4) go(fc_i8_some<T, 4>);   // (at most 256)
  }
  LPG_HIP(hipGetLastError());
  return LPG_OK;
}

// What lpg_fc_i8_rows takes: one row that fits its LDS; some rows up to 1024 columns long, as many blocks as CUs at
// most.  Then it is ahead of the two launches at every M (fp16, N = 1024: K = 512 5.0 us against 7.6 for 2 rows, 5.6 and
// 8.4 for 256; K = 1024 6.2 and 7.8 for 2, 7.2 and 8.8 for 64, 7.6 and 8.8 for 256).  Of longer rows the two are, at every
// M too (K = 1040 9.1 and 7.6 for 2, 10.1 and 8.9 for 128; K = 2048 10.6 and 9.2, 11.7 and 10.4).  With more blocks
// the rows that each quantises again cost more than the launch (2000 x 512, K = 256 13.6 and 7.3).
bool few_rows(int64_t M, int64_t N, int64_t K) {
  if (M <= 1) return (K + 1023) / 1024 * 1024 <= kRowBytes && (N + 3) / 4 <= most_blocks(256);
  return K <= kSomeK && (M + 15) / 16 <= 65535 && (M + 15) / 16 * ((N + kSomeN - 1) / kSomeN) <= device_cus();
}

constexpr int64_t kMaxK = 131072;  // 131072 * 127^2 < 2^31

}  // namespace
}  // namespace lpg

using namespace lpg;

#define LPG_I8_TYPES(what, f)                                                            \
  do {                                                                                   \
    if (dtype == LPG_F32) return f(float);                                               \
    if (dtype == LPG_BF16) return f(__bf16);                                             \
    if (dtype == LPG_F16) return f(_Float16);                                            \
    ::lpg::set_error(what ": dtype %d (LPG_BF16, LPG_F16 or LPG_F32)", (int)dtype);      \
    return LPG_ERR_INVALID;                                                              \
  } while (0)

// 160 MiB of codes: written by the one kernel and read by the other they stay in the 256 MiB of last-level cache (the
// streams of large x and y go past it).  Whole rounds of 256-row tiles, and up to a quarter more in place of a short
// last chunk.  200 K x 2048, K = 4096 bf16 with 64 / 96 / 160 / 192 MiB 1.83 / 1.72 / 1.66 / 1.64 ms, 150 K x 1500, K =
// 3000 fp16 0.95 / 0.81 / 0.80 / 0.85; half a chunk more instead of a quarter: 130 K x 1024, K = 1024 0.257 against 0.220.
extern "C" int64_t lpg_i8_chunk_rows(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 1 || K < 1) return -1;
  const int64_t ldq = (K + 127) / 128 * 128, nt = (N + 255) / 256, cus = device_cus();
  const int64_t rounds = ((int64_t)160 << 20) / ldq / 256 * nt / cus;
  int64_t rows = (rounds < 1 ? 1 : rounds) * cus / nt * 256;
  rows = rows < 256 ? 256 : rows;
  return M < rows + rows / 4 ? M : rows;
}

extern "C" lpg_status lpg_quant_i8(int32_t dtype, int64_t M, int64_t K1, const void *x, int64_t ldx, int64_t K2,
                                   const void *x2, int64_t ldx2, int8_t *q, int64_t ldq, float *scale, void *stream) {
  LPG_REQUIRE(M >= 0 && K1 >= 1 && K2 >= 0 && K1 <= kMaxK && K2 <= kMaxK && K1 + K2 <= kMaxK,
              "lpg_quant_i8: need M >= 0, K1 >= 1, K2 >= 0, K1 + K2 <= 131072");
  LPG_REQUIRE(ldx >= K1 && (K2 == 0 || ldx2 >= K2), "lpg_quant_i8: row strides below the columns");
  LPG_REQUIRE(ldq >= K1 + K2 && ldq % 128 == 0, "lpg_quant_i8: ldq must be a multiple of 128 that holds K1 + K2");
  LPG_REQUIRE(M == 0 || (x && q && scale && (K2 == 0 || x2)), "lpg_quant_i8: NULL pointer");
  LPG_REQUIRE(aligned16(q), "lpg_quant_i8: q must be 16-byte aligned");
  // x past the caches where it would push out the codes (100 K x 2048 fp32 with the product to 1024 469 -> 394 us, 376 by now,
  // 60 K x 2048 fp16 187 -> 177); a small x may still be in them (20000 x 1024 fp16 45 us through them, 47 past them)
  const int past = M * (K1 + K2) * (dtype == LPG_F32 ? 4 : 2) > (int64_t)128 << 20;
  const QuantArgs a{M, ldx, ldx2, ldq, (int)K1, (int)K2, x, x2, q, scale, past};
  const auto go = [&](auto kernel, int rows) -> lpg_status {
    const int64_t most = most_blocks(256) * rows, e = dtype == LPG_F32 ? 4 : 2;
    for (int64_t at = 0; at < M; at += most) {  // (one launch but for tens of millions of rows)
      QuantArgs b = a;
      b.M = M - at < most ? M - at : most;
      b.x = static_cast<const char *>(x) + at * ldx * e;
      b.x2 = K2 ? static_cast<const char *>(x2) + at * ldx2 * e : nullptr;
      b.q = q + at * ldq;
      b.scale = scale + at;
      hipLaunchKernelGGL(kernel, dim3((unsigned)((b.M + rows - 1) / rows)), dim3(256), 0, as_stream(stream), b);
      LPG_HIP(hipGetLastError());
    }
    return LPG_OK;
  };
  // The fewest lanes, from 8 on, that hold a row in up to four vectors each, else a wave and up to 16 vectors a lane:
  // what a row costs beside its elements (its largest, two divisions) is shared by as many rows of the wave as it holds
  // (700 K x 300 bf16: 340 us with a vector a lane and 64 lanes, 142 with three and 16; 1.6 M x 128 179 and 124).  Two
  // or four lanes cost more than they share (2.1 M x 100 155 us with eight, 211 with four); the shortest rows are faster
  // with a vector a lane (3.3 M x 64 163 us, two lanes of four 264); longer rows than 16 vectors a lane are read twice.
  const auto of = [&](auto t) -> lpg_status {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    if (K1 / V + K2 / V <= 8) return go(quant_rows_held<T, 8, 1, true>, 32);
    if (K1 < V || (K2 > 0 && K2 < V)) return go(quant_rows<T>, 4);  // (a part without a vector, beside a long one)
    const int64_t n = (K1 + V - 1) / V + (K2 + V - 1) / V;
    if (n <= 16) return go(quant_rows_held<T, 8, 2>, 32);
    if (n <= 24) return go(quant_rows_held<T, 8, 3>, 32);
    if (n <= 32) return go(quant_rows_held<T, 8, 4>, 32);
    if (n <= 48) return go(quant_rows_held<T, 16, 3>, 16);
    if (n <= 64) return go(quant_rows_held<T, 16, 4>, 16);
    if (n <= 96) return go(quant_rows_held<T, 32, 3>, 8);
    if (n <= 128) return go(quant_rows_held<T, 32, 4>, 8);
    if (n <= 192) return go(quant_rows_held<T, 64, 3>, 4);
    if (n <= 256) return go(quant_rows_held<T, 64, 4>, 4);
    if (n <= 384) return go(quant_rows_held<T, 64, 6>, 4);
    if (n <= 512) return go(quant_rows_held<T, 64, 8>, 4);
    if (n <= 1024) return go(quant_rows_held<T, 64, 16>, 4);
    return go(quant_rows<T>, 4);
  };
#define F(T) of(T{})
  LPG_I8_TYPES("lpg_quant_i8", F);
#undef F
}

extern "C" lpg_status lpg_fc_i8(int32_t dtype, int64_t M, int64_t N, int64_t K, const int8_t *q, int64_t ldq,
                                const float *scale, const int8_t *w, int64_t ldw, const float *wscale, const float *bias,
                                int32_t flags, void *y, int64_t ldy, void *stream) {
  LPG_REQUIRE(M >= 0 && N >= 1 && K >= 1 && K <= kMaxK, "lpg_fc_i8: need M >= 0, N >= 1, 1 <= K <= 131072");
  LPG_REQUIRE(ldq >= K && ldq % 128 == 0 && ldq <= kMaxK, "lpg_fc_i8: ldq must be a multiple of 128 that holds K");
  LPG_REQUIRE(ldw % 16 == 0 && ldw >= (K + 15) / 16 * 16 && ldw <= (int64_t)1 << 22,
              "lpg_fc_i8: ldw must be a multiple of 16 that holds K, at most 2^22");
  LPG_REQUIRE(ldy >= N && (flags & ~LPG_FC_RELU) == 0, "lpg_fc_i8: ldy below N or unknown flags");
  LPG_REQUIRE(w && wscale && (M == 0 || (q && scale && y)), "lpg_fc_i8: NULL pointer");
  LPG_REQUIRE(aligned16(q) && aligned16(w), "lpg_fc_i8: q and w must be 16-byte aligned");
  LPG_REQUIRE(((M + 63) / 64) <= INT32_MAX / ((N + 63) / 64), "lpg_fc_i8: too many tiles");
  // Past the caches go outputs that would push out the codes: not short sums' (100 K x 1024, K = 64 60 us through
  // them, 73 past them; fp32 100 K x 512, K = 512 95 and 117, x 1024, K = 1024 251 and 226), not small ones (20000 x
  // 1024, K = 1024 41 and 43; 200 K x 2048, K = 1024 629 and 537), only rows on whole lines (30000 x 1000, K = 2000 62 us
  // through them, 86 past them).
  const int64_t e = dtype == LPG_F32 ? 4 : 2;
  const int past = K > (e == 4 ? 512 : 128) && M * N * e > (int64_t)64 << 20 && ldy * e % 128 == 0 &&
                   reinterpret_cast<uintptr_t>(y) % 128 == 0;
  const FcArgs a{M, N, ldq, ldw, ldy, (int)K, q, w, scale, wscale, bias, y, 0, 0,
                 (flags & LPG_FC_RELU) ? 0.f : -INFINITY, past};
#define F(T) M == 0 ? LPG_OK : run_fc<T>(a, as_stream(stream))
  LPG_I8_TYPES("lpg_fc_i8", F);
#undef F
}

extern "C" lpg_status lpg_fc_i8_rows(int32_t dtype, int64_t M, int64_t N, int64_t K1, const void *x, int64_t ldx,
                                     int64_t K2, const void *x2, int64_t ldx2, const int8_t *w, int64_t ldw,
                                     const float *wscale, const float *bias, int32_t flags, void *y, int64_t ldy,
                                     void *stream) {
  LPG_REQUIRE(M >= 0 && N >= 1 && N <= INT32_MAX && K1 >= 1 && K2 >= 0 && K1 <= kMaxK && K2 <= kMaxK,
              "lpg_fc_i8_rows: need M >= 0, 1 <= N < 2^31, K1 >= 1, K2 >= 0, both at most 131072");
  const int64_t K = K1 + K2;
  LPG_REQUIRE(ldx >= K1 && (K2 == 0 || ldx2 >= K2) && ldy >= N, "lpg_fc_i8_rows: row strides below the columns");
  LPG_REQUIRE(ldw % 16 == 0 && ldw >= (K + 15) / 16 * 16, "lpg_fc_i8_rows: ldw must be a multiple of 16 that holds K");
  LPG_REQUIRE((flags & ~LPG_FC_RELU) == 0, "lpg_fc_i8_rows: unknown flags");
  LPG_REQUIRE(w && wscale && (M == 0 || (x && y && (K2 == 0 || x2))), "lpg_fc_i8_rows: NULL pointer");
  LPG_REQUIRE(aligned16(w), "lpg_fc_i8_rows: w must be 16-byte aligned");
  if (M > INT32_MAX || !few_rows(M, N, K)) {
    set_error("lpg_fc_i8_rows: too many or too long rows for one launch (use lpg_quant_i8 and lpg_fc_i8)");
    return LPG_ERR_UNSUPPORTED;
  }
  const RowsArgs a{M, N, ldx, ldx2, ldw, ldy, (int)K1, (int)K2, x, x2, w, wscale, bias, y,
                   (flags & LPG_FC_RELU) ? 0.f : -INFINITY};
#define F(T) M == 0 ? LPG_OK : run_rows<T>(a, as_stream(stream))
  LPG_I8_TYPES("lpg_fc_i8_rows", F);
#undef F
}
