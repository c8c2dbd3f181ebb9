// One AdamW step over many tensors at once, and the global gradient norm its clip needs.
//
//   g = c grad                                    (c = *grad_scale, or 1)
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32 whatever the parameters' type; moments in 32 bits, or in 8 (below).  HBM-bound: 28 bytes a
// number (16 in, 12 out) with fp32 moments, 16 with 8-bit ones, and ~20 operations; for a small model it
// is launch latency.  So: every tensor of the call in one launch (their pointers travel in the kernel
// arguments, no table on the device to fill or to keep), one block a chunk of one tensor,
// all of a thread's loads issued before the first use.
//
// 8-bit moments.  A block of 256 consecutive elements shares two fp32 scales: m and r = sqrt(v) are held
// as e4m3 numbers (torch.float8_e4m3fn) times largest / 448.  The root halves the exponent range v needs:
// 2^-17.8 of the block's largest r is 2^-35 of its largest v.  Rounding is random: 16 bits of a counter
// hash of (seed, step, tensor, element) are added below the kept mantissa before it is cut, so the stored
// number is right on average.  To nearest, a moment whose change in one step is below half a step of its
// format (3 %) would never move, and v changes by 0.1 % of itself in most steps (b2 = 0.999).  An r above
// zero never becomes zero (its parameter would be divided by eps alone).  A block that holds a NaN or an
// infinity gets the scale NaN: the state stays visibly bad, as it does in 32 bits.  The parameter update
// uses the moments before they are rounded.
//
// 67 M numbers: 279 us with fp32 moments (6.7 TB/s; bf16 parameters 254, 5.8), 180 with 8-bit ones (6.0), the norm 48
// (5.6) + 5; 4.2 M: 8-bit step 16, norm 5 + 3; 70 K in 22 tensors 3.8 us.
//
// The norm is summed in 64 bits, where products of fp32 numbers are exact, in a fixed order: the same list
// gives the same bits.  Split otherwise, the sums differ in their last 64-bit places, so the norm and the
// factor are the same 32-bit numbers or, where a border lies between them, neighbours.
#include "common.h"
#include "fc_common.h"  // lowbias32

namespace lpg {
namespace {

constexpr int kT = 256;
// Elements a block: the small chunk up to 16 M numbers in all (more waves in flight), the large one above it.  Of the
// step with 32-bit moments, 4.2 M numbers 21.7 -> 19.0 us with the small one, 67 M 319 -> 329; of the norm (a partial sum
// each) 4.2 M 8.3 -> 4.8, and of 67 M one block would have to add 16000 partial sums in place of 4000.  With 8-bit
// moments 1024: 67 M 182 us, with 2048 183, 4096 190; 4.2 M 15.5, 17.7 and 20.3.
constexpr int kChunk = 4096, kChunkS = 1024;
constexpr int kChunk8 = 1024;
constexpr int kNormChunk = 16384, kNormChunkS = 4096;
constexpr int64_t kSmall = (int64_t)1 << 24;
constexpr int kQ = 256;  // elements that share a scale

// Tensors a launch takes: the table is a kernel argument (at most 4 KB of them).
constexpr int kMany = 64, kMany8 = 56, kManyN = 128;

struct Table32 {
  lpg_adamw_hyper h;
  const float *scale;
  int count;
  uint32_t first[kMany];  // the first block of each tensor
  lpg_adamw_tensor t[kMany];
};
struct Table8 {
  lpg_adamw_hyper h;
  const float *scale;
  int count;
  uint32_t first[kMany8];
  lpg_adamw8_tensor t[kMany8];
};
struct TableN {
  double *part;
  int count;
  uint32_t first[kManyN];
  lpg_tensor t[kManyN];
};
static_assert(sizeof(Table32) <= 4096 && sizeof(Table8) <= 4096 && sizeof(TableN) <= 4096, "kernel arguments");

// the tensor of this block: the last one whose first block is not behind it
template <typename Tab>
__device__ __forceinline__ int tensor_of(const Tab &tab) {
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// four consecutive elements at any element alignment, non-temporal
template <typename T>
struct Four;
template <>
struct Four<float> {
  typedef unsigned int words __attribute__((ext_vector_type(4)));
  typedef unsigned int any __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct Four<__bf16> {
  typedef unsigned int words __attribute__((ext_vector_type(2)));
  typedef unsigned int any __attribute__((ext_vector_type(2), aligned(2)));
};
template <typename T>
__device__ __forceinline__ void ld4(const T *p, float (&f)[4]) {
  const typename Four<T>::words w = __builtin_nontemporal_load(reinterpret_cast<const typename Four<T>::any *>(p));
  T t[4];
  __builtin_memcpy(t, &w, sizeof(t));
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = (float)t[j];
}
template <typename T>
__device__ __forceinline__ void st4(T *p, const float (&f)[4]) {
  T t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = (T)f[j];
  typename Four<T>::words w;
  __builtin_memcpy(&w, t, sizeof(t));
  __builtin_nontemporal_store(w, reinterpret_cast<typename Four<T>::any *>(p));
}
// ... of which `n` (0 to 4) exist; the others read as zero and are not written
template <typename T>
__device__ __forceinline__ void ld_n(const T *p, int n, float (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = j < n ? (float)p[j] : 0.f;
}
template <typename T>
__device__ __forceinline__ void st_n(T *p, int n, const float (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) p[j] = (T)f[j];
}

__device__ __forceinline__ float new_p(const lpg_adamw_hyper &h, float p, float m, float r) {
  return p * h.keep - (m / (r * h.inv_root2 + h.eps)) * h.rate;
}

template <typename T, int CHUNK>
__global__ __launch_bounds__(kT) void adamw32(Table32 tab) {
  constexpr int U = CHUNK / (4 * kT);
  const int k = tensor_of(tab);
  const lpg_adamw_tensor &e = tab.t[k];
  const int64_t base = (int64_t)(blockIdx.x - tab.first[k]) * CHUNK;
  const float c = tab.scale ? *tab.scale : 1.f;
  const lpg_adamw_hyper h = tab.h;
  T *p = static_cast<T *>(e.p);
  const T *g = static_cast<const T *>(e.g);
  const auto update = [&](float (&pp)[4], float (&gg)[4], float (&mm)[4], float (&vv)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = gg[j] * c;
      mm[j] = mm[j] * h.beta1 + x * h.rest1;
      vv[j] = vv[j] * h.beta2 + (x * x) * h.rest2;
      pp[j] = new_p(h, pp[j], mm[j], sqrtf(vv[j]));
    }
  };
  if (base + CHUNK <= e.n) {
    float pp[U][4], gg[U][4], mm[U][4], vv[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = base + (u * kT + (int)threadIdx.x) * 4;
      ld4(g + i, gg[u]);
      ld4(e.m + i, mm[u]);
      ld4(e.v + i, vv[u]);
      ld4(p + i, pp[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = base + (u * kT + (int)threadIdx.x) * 4;
      update(pp[u], gg[u], mm[u], vv[u]);
      st4(e.m + i, mm[u]);
      st4(e.v + i, vv[u]);
      st4(p + i, pp[u]);
    }
  } else {
    for (int64_t i = base + (int)threadIdx.x * 4; i < e.n; i += kT * 4) {
      const int n = e.n - i < 4 ? (int)(e.n - i) : 4;
      float pp[4], gg[4], mm[4], vv[4];
      ld_n(g + i, n, gg);
      ld_n(e.m + i, n, mm);
      ld_n(e.v + i, n, vv);
      ld_n(p + i, n, pp);
      update(pp, gg, mm, vv);
      st_n(e.m + i, n, mm);
      st_n(e.v + i, n, vv);
      st_n(p + i, n, pp);
    }
  }
}

// the largest of the wave's 64 values (as unsigned numbers: the order of |x| of floats, NaN on top)
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  const auto dpp = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  v = max(v, dpp(v, std::integral_constant<int, 0xB1>()));   // quad_perm 1,0,3,2
  v = max(v, dpp(v, std::integral_constant<int, 0x4E>()));   // quad_perm 2,3,0,1
  v = max(v, dpp(v, std::integral_constant<int, 0x141>()));  // row_half_mirror
  v = max(v, dpp(v, std::integral_constant<int, 0x140>()));  // row_mirror
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(b[0], b[1]);
}

// The scales of a block's two moments, from the bits of their largest |x|, by one division of the wave: its
// lower half divides for m, its upper for r.  inv = 448 / largest takes the block to the format's range (below
// 1e-30 the block is zero: 448 / largest would overflow), scale = largest / 448 back.
struct Scales8 {
  float inv_m, inv_r, scale_m, scale_r;
  __device__ __forceinline__ Scales8(uint32_t mt, uint32_t rt, int lane) {
    const auto norm = [](uint32_t bits) { return bits < 0x7f800000u && __uint_as_float(bits) >= 1e-30f; };
    const bool lm = norm(mt), lr = norm(rt);
    // quarters of the wave: 448 / m, m / 448, 448 / r, r / 448
    const float top = __uint_as_float(lane < 32 ? mt : rt);
    const float v = lane & 16 ? top / 448.f : 448.f / top;
    const auto at = [&](int l) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), l)); };
    const auto scale = [&](uint32_t bits, bool live, int l) {
      return bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : (live ? at(l) : 0.f);
    };
    inv_m = lm ? at(0) : 0.f;
    inv_r = lr ? at(32) : 0.f;
    scale_m = scale(mt, lm, 16);
    scale_r = scale(rt, lr, 48);
  }
};

template <typename T>
__global__ __launch_bounds__(kT) void adamw8(Table8 tab) {
  constexpr int U = kChunk8 / (kQ * (kT / 64));  // scale blocks a wave
  const int k = tensor_of(tab);
  const lpg_adamw8_tensor &e = tab.t[k];
  const int64_t base = (int64_t)(blockIdx.x - tab.first[k]) * kChunk8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float c = tab.scale ? *tab.scale : 1.f;
  const lpg_adamw_hyper h = tab.h;
  const uint32_t key = (uint32_t)e.key;
  T *p = static_cast<T *>(e.p);
  const T *g = static_cast<const T *>(e.g);
  uint8_t *m8 = static_cast<uint8_t *>(e.m8), *r8 = static_cast<uint8_t *>(e.r8);
  float pp[U][4], gg[U][4], ms[U], rs[U];
  uint32_t mq[U], rq[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t q = base / kQ + u * (kT / 64) + wave, i = q * kQ + lane * 4;
    const int n = e.n - i >= 4 ? 4 : (e.n - i > 0 ? (int)(e.n - i) : 0);
    mq[u] = rq[u] = 0;
    if (n == 4) {
      ld4(g + i, gg[u]);
      ld4(p + i, pp[u]);
      __builtin_memcpy(&mq[u], m8 + i, 4);
      __builtin_memcpy(&rq[u], r8 + i, 4);
    } else {
      ld_n(g + i, n, gg[u]);
      ld_n(p + i, n, pp[u]);
      for (int j = 0; j < n; ++j) {
        mq[u] |= (uint32_t)m8[i + j] << (8 * j);
        rq[u] |= (uint32_t)r8[i + j] << (8 * j);
      }
    }
    const bool some = q * kQ < e.n;
    ms[u] = some ? e.ms[q] : 0.f;
    rs[u] = some ? e.rs[q] : 0.f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t q = base / kQ + u * (kT / 64) + wave, i = q * kQ + lane * 4;
    if (q * kQ >= e.n) continue;  // (the whole wave: what follows has every lane)
    const int n = e.n - i >= 4 ? 4 : (e.n - i > 0 ? (int)(e.n - i) : 0);
    const auto ma = __builtin_amdgcn_cvt_pk_f32_fp8(mq[u], false), mb = __builtin_amdgcn_cvt_pk_f32_fp8(mq[u], true);
    const auto ra = __builtin_amdgcn_cvt_pk_f32_fp8(rq[u], false), rb = __builtin_amdgcn_cvt_pk_f32_fp8(rq[u], true);
    float m[4] = {ma[0], ma[1], mb[0], mb[1]}, r[4] = {ra[0], ra[1], rb[0], rb[1]};
    uint32_t mt = 0, rt = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = gg[u][j] * c;
      m[j] = (m[j] * ms[u]) * h.beta1 + x * h.rest1;
      r[j] = r[j] * rs[u];
      r[j] = sqrtf((r[j] * r[j]) * h.beta2 + (x * x) * h.rest2);
      pp[u][j] = new_p(h, pp[u][j], m[j], r[j]);
      if (j < n) {  // (elements past the end have no say in the scale: theirs is 0 times a scale that may be NaN)
        mt = max(mt, __float_as_uint(fabsf(m[j])));
        rt = max(rt, __float_as_uint(fabsf(r[j])));
      }
    }
    const Scales8 sc(wave_max(mt), wave_max(rt), lane);
    // the random rounding is the conversion's own: its seed's upper 20 bits are added below the mantissa it
    // keeps (in the subnormal range, below the 2^-9 it counts in), here 16 random bits and four zeros
    uint32_t mo = 0, ro = 0;
    const float least = sc.inv_r > 0.f ? 0x1p-9f : 0.f;
    const auto put = [&](auto jc) {
      constexpr int j = decltype(jc)::value;
      const uint64_t at = (uint64_t)(i + j);
      const uint32_t bits = lowbias32((uint32_t)at ^ key ^ (uint32_t)(at >> 32) * 0x9e3779b9u);
      const float tm = __builtin_amdgcn_fmed3f(m[j] * sc.inv_m, -448.f, 448.f);
      const float tr = r[j] > 0.f ? fminf(fmaxf(r[j] * sc.inv_r, least), 448.f) : 0.f;
      mo = (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(tm, (int)(bits << 16), (int)mo, j);
      ro = (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(tr, (int)(bits & 0xffff0000u), (int)ro, j);
    };
    put(std::integral_constant<int, 0>());
    put(std::integral_constant<int, 1>());
    put(std::integral_constant<int, 2>());
    put(std::integral_constant<int, 3>());
    if (n == 4) {
      st4(p + i, pp[u]);
      __builtin_memcpy(m8 + i, &mo, 4);
      __builtin_memcpy(r8 + i, &ro, 4);
    } else {
      st_n(p + i, n, pp[u]);
      for (int j = 0; j < n; ++j) {
        m8[i + j] = (uint8_t)(mo >> (8 * j));
        r8[i + j] = (uint8_t)(ro >> (8 * j));
      }
    }
    if (lane == 0) {
      e.ms[q] = sc.scale_m;
      e.rs[q] = sc.scale_r;
    }
  }
}

// the block's sum, in thread 0 (one call a kernel)
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double red[kT / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T, int CHUNK>
__global__ __launch_bounds__(kT) void sumsq(TableN tab) {
  constexpr int U = CHUNK / (4 * kT);
  const int k = tensor_of(tab);
  const lpg_tensor &e = tab.t[k];
  const T *g = static_cast<const T *>(e.p);
  const int64_t base = (int64_t)(blockIdx.x - tab.first[k]) * CHUNK;
  double s = 0;
  const auto add = [&](const float (&f)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s = __builtin_fma((double)f[j], (double)f[j], s);
  };
  if (base + CHUNK <= e.n) {
    float f[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (ordinary loads, the step reads the gradients next: 67 M with the clip 362 -> 325 us)
      T t[4];
      __builtin_memcpy(t, g + base + (u * kT + (int)threadIdx.x) * 4, sizeof(t));
#pragma unroll
      for (int j = 0; j < 4; ++j) f[u][j] = (float)t[j];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) add(f[u]);
  } else {
    for (int64_t i = base + (int)threadIdx.x * 4; i < e.n; i += kT * 4) {
      float f[4];
      ld_n(g + i, e.n - i < 4 ? (int)(e.n - i) : 4, f);
      add(f);
    }
  }
  s = block_sum(s);
  if (threadIdx.x == 0) tab.part[blockIdx.x] = s;
}

__global__ __launch_bounds__(kT) void norm_scale(int64_t n, const double *__restrict__ part, double max_norm, float *norm,
                                                 float *scale) {
  double s = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += kT) s += part[i];
  s = block_sum(s);
  if (threadIdx.x == 0) {
    const double l = sqrt(s), f = max_norm / (l + 1e-6);
    *norm = (float)l;
    *scale = f > 1.0 ? 1.f : (float)f;  // (a NaN norm gives a NaN factor)
  }
}

int64_t blocks_of(int64_t n, int64_t chunk) { return (n + chunk - 1) / chunk; }

template <typename E>
bool small(int64_t count, const E *list) {
  int64_t n = 0;
  for (int64_t i = 0; i < count && n <= kSmall; ++i) n += list[i].n;
  return n <= kSmall;
}

bool hyper_ok(const lpg_adamw_hyper &h) {
  return h.beta1 >= 0.f && h.beta1 < 1.f && h.beta2 >= 0.f && h.beta2 < 1.f && h.eps >= 0.f;
}

// Fills tables of at most `many` tensors (those without elements left out) and launches each.
template <typename Tab, typename E, typename L>
lpg_status in_tables(Tab &tab, int many, int64_t chunk, int64_t count, const E *list, const char *what, L launch) {
  for (int64_t i = 0; i < count; ++i)  // (before the first launch: a refused call updates nothing)
    if (list[i].n > most_blocks(kT) * chunk) {
      set_error("%s: a tensor of %lld elements is too large", what, (long long)list[i].n);
      return LPG_ERR_UNSUPPORTED;
    }
  for (int64_t at = 0; at < count;) {
    int k = 0;
    int64_t blocks = 0;
    for (; at < count && k < many; ++at) {
      if (list[at].n == 0) continue;
      const int64_t b = blocks_of(list[at].n, chunk);
      if (blocks + b > most_blocks(kT)) break;
      tab.t[k] = list[at];
      tab.first[k++] = (uint32_t)blocks;
      blocks += b;
    }
    if (k == 0) continue;
    tab.count = k;
    launch(blocks);
    LPG_HIP(hipGetLastError());
  }
  return LPG_OK;
}

}  // namespace
}  // namespace lpg

using namespace lpg;

extern "C" lpg_status lpg_adamw(int32_t dtype, int64_t count, const lpg_adamw_tensor *tensors, const lpg_adamw_hyper *hyper,
                                const float *grad_scale, void *stream) {
  LPG_REQUIRE(dtype == LPG_F32 || dtype == LPG_BF16, "lpg_adamw: dtype %d (LPG_F32 or LPG_BF16)", (int)dtype);
  LPG_REQUIRE(count >= 0 && (count == 0 || tensors) && hyper, "lpg_adamw: NULL pointer or a negative count");
  LPG_REQUIRE(hyper_ok(*hyper), "lpg_adamw: need 0 <= beta < 1 and eps >= 0");
  for (int64_t i = 0; i < count; ++i)
    LPG_REQUIRE(tensors[i].n >= 0 && (tensors[i].n == 0 || (tensors[i].p && tensors[i].g && tensors[i].m && tensors[i].v)),
                "lpg_adamw: tensor %lld has a negative size or a NULL pointer", (long long)i);
  hipStream_t s = as_stream(stream);
  Table32 tab;
  tab.h = *hyper;
  tab.scale = grad_scale;
  const bool few = small(count, tensors);
  const auto kernel = dtype == LPG_F32 ? (few ? adamw32<float, kChunkS> : adamw32<float, kChunk>)
                                       : (few ? adamw32<__bf16, kChunkS> : adamw32<__bf16, kChunk>);
  return in_tables(tab, kMany, few ? kChunkS : kChunk, count, tensors, "lpg_adamw", [&](int64_t blocks) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kT), 0, s, tab);
  });
}

extern "C" lpg_status lpg_adamw8(int32_t dtype, int64_t count, const lpg_adamw8_tensor *tensors,
                                 const lpg_adamw_hyper *hyper, const float *grad_scale, void *stream) {
  LPG_REQUIRE(dtype == LPG_F32 || dtype == LPG_BF16, "lpg_adamw8: dtype %d (LPG_F32 or LPG_BF16)", (int)dtype);
  LPG_REQUIRE(count >= 0 && (count == 0 || tensors) && hyper, "lpg_adamw8: NULL pointer or a negative count");
  LPG_REQUIRE(hyper_ok(*hyper), "lpg_adamw8: need 0 <= beta < 1 and eps >= 0");
  for (int64_t i = 0; i < count; ++i) {
    const lpg_adamw8_tensor &t = tensors[i];
    LPG_REQUIRE(t.n >= 0 && (t.n == 0 || (t.p && t.g && t.m8 && t.ms && t.r8 && t.rs)),
                "lpg_adamw8: tensor %lld has a negative size or a NULL pointer", (long long)i);
  }
  hipStream_t s = as_stream(stream);
  Table8 tab;
  tab.h = *hyper;
  tab.scale = grad_scale;
  return in_tables(tab, kMany8, kChunk8, count, tensors, "lpg_adamw8", [&](int64_t blocks) {
    if (dtype == LPG_F32) hipLaunchKernelGGL((adamw8<float>), dim3((unsigned)blocks), dim3(kT), 0, s, tab);
    else hipLaunchKernelGGL((adamw8<__bf16>), dim3((unsigned)blocks), dim3(kT), 0, s, tab);
  });
}

extern "C" int64_t lpg_grad_norm_workspace_bytes(int64_t count, const lpg_tensor *tensors) {
  if (count < 0 || (count && !tensors)) return -1;
  for (int64_t i = 0; i < count; ++i)
    if (tensors[i].n < 0) return -1;
  const int64_t chunk = small(count, tensors) ? kNormChunkS : kNormChunk;
  int64_t blocks = 0;
  for (int64_t i = 0; i < count; ++i) blocks += blocks_of(tensors[i].n, chunk);
  return (blocks < 1 ? 1 : blocks) * (int64_t)sizeof(double);
}

extern "C" lpg_status lpg_grad_norm(int32_t dtype, int64_t count, const lpg_tensor *tensors, double max_norm, float *norm,
                                    float *scale, void *workspace, void *stream) {
  LPG_REQUIRE(dtype == LPG_F32 || dtype == LPG_BF16, "lpg_grad_norm: dtype %d (LPG_F32 or LPG_BF16)", (int)dtype);
  LPG_REQUIRE(count >= 0 && (count == 0 || tensors) && norm && scale && workspace,
              "lpg_grad_norm: NULL pointer or a negative count");
  LPG_REQUIRE(max_norm >= 0.0, "lpg_grad_norm: max_norm must not be negative");
  for (int64_t i = 0; i < count; ++i)
    LPG_REQUIRE(tensors[i].n >= 0 && (tensors[i].n == 0 || tensors[i].p),
                "lpg_grad_norm: tensor %lld has a negative size or a NULL pointer", (long long)i);
  hipStream_t s = as_stream(stream);
  TableN tab;
  double *part = static_cast<double *>(workspace);
  int64_t total = 0;
  const bool few = small(count, tensors);
  const auto kernel = dtype == LPG_F32 ? (few ? sumsq<float, kNormChunkS> : sumsq<float, kNormChunk>)
                                       : (few ? sumsq<__bf16, kNormChunkS> : sumsq<__bf16, kNormChunk>);
  const int64_t chunk = few ? kNormChunkS : kNormChunk;
  const lpg_status st = in_tables(tab, kManyN, chunk, count, tensors, "lpg_grad_norm", [&](int64_t blocks) {
    tab.part = part + total;
    total += blocks;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kT), 0, s, tab);
  });
  if (st != LPG_OK) return st;
  hipLaunchKernelGGL(norm_scale, dim3(1), dim3(kT), 0, s, total, part, max_norm, norm, scale);
  LPG_HIP(hipGetLastError());
  return LPG_OK;
}
