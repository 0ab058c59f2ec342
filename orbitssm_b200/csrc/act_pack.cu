// Activations kept in eight bits between the forward and the backward pass: a signed byte an element and one power of two
// for each 32 consecutive elements of a row (a row's last group may be shorter).
//
//   e = the least exponent in [-126, 122] with round(amax 2^-e) <= 127,   q = round_to_even(x 2^-e),   x^ = q 2^e
//
// The scale is a power of two, so x 2^-e is exact and the only rounding is the one to the whole number q: at most half a step,
// 2^(e-1).  A step smaller by half would round amax to 128 or more, so amax >= 63.75 steps and the error is at most amax / 127.5
// (reached: of a group whose largest is 127.5, the element 1 is restored as 0).  x^ has seven significant bits: exact in bfloat16
// as in float32.  e needs no division or logarithm: with amax = m 2^E, m in [1, 2), it is E - 6, or E - 5 where 64 m would round to 128.
// A step below 2^-126 is not taken (the restored values stay normal numbers; the error there is at most 2^-127, whatever amax).  Codes of the
// largest step (2^122) end at 63, so that x^ stays finite at the type's largest values (there off by one step at most).  Packing x^
// again restores the same values; the bytes are the same too, except at the largest step (codes of 63 come back as 126 of half of it).
// A non-finite element takes the code -128, which nothing else uses, and is restored as NaN; it does not enter amax, so its
// neighbours keep their precision.
//
// HBM-bound: es + 1 + 1/32 bytes an element in either direction; 16-byte accesses on both sides where rows allow.  Both directions
// of 67 million elements in rows of 1024: bfloat16 72 us (5.7 TB/s), float32 121 us (5.6 TB/s).
#include "common.cuh"
#include "../../include/orbit_b200.h"

namespace orbit {

constexpr int PACK_GROUP = 32, PACK_THREADS = 256;

// 16 consecutive elements held by one thread, as raw 32-bit words
template <typename T> struct Raw16;
template <> struct Raw16<__nv_bfloat16> {
  uint4 a, b;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    a = __ldcs(reinterpret_cast<const uint4*>(p));
    b = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
  }
  __device__ __forceinline__ void get(float (&f)[16]) const {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Raw16<float> {
  float4 v[4];
  __device__ __forceinline__ void load(const float* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __ldcs(reinterpret_cast<const float4*>(p) + i);
  }
  __device__ __forceinline__ void get(float (&f)[16]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[4 * i] = v[i].x; f[4 * i + 1] = v[i].y; f[4 * i + 2] = v[i].z; f[4 * i + 3] = v[i].w; }
  }
};

// bits of |x| where x is finite, else 0
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}
// biased exponent (e + 127, in [1, 249]) of a group from the bits of its largest finite |x|
__device__ __forceinline__ uint32_t group_exponent(uint32_t amax_bits) {
  const int E = (int)(amax_bits >> 23);                      // 0 for zero and subnormal maxima
  const int b = E - 6 + ((amax_bits & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
  return (uint32_t)max(b, 1);
}
constexpr uint32_t TOP_EXPONENT = 249;                       // the step 2^122
constexpr float TOP_VALUE = 0x1.f8p127f;                     // 63 steps of it

// x 2^-e plus 1.5 2^23: the low byte of the sum's bits is the rounded whole number (one rounding: the product is exact)
__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  const uint32_t q = __float_as_uint(fmaf(x, inv, 12582912.f));
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? 0x80u : q;
}
template <int N> __device__ __forceinline__ void keep_finite(float (&f)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (finite_abs_bits(f[j]) != 0u) f[j] = fminf(fmaxf(f[j], -TOP_VALUE), TOP_VALUE);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
__device__ __forceinline__ float inv_scale(uint32_t biased) { return __uint_as_float((254u - biased) << 23); }   // 2^-e

// byte k of `w` (codes with the sign bit flipped) times 2^e
__device__ __forceinline__ float value_of(uint32_t w_flipped, int k, float scale) {
  const float f = __uint_as_float(__byte_perm(w_flipped, 0x4b000000u, 0x7440 + k)) - 8388736.f;    // 2^23 + (q + 128) - (2^23 + 128)
  return f == -128.f ? __uint_as_float(0x7fffffffu) : f * scale;
}

// Rows that are whole numbers of groups and lie one after another: the array is a flat run of groups (67 million bfloat16 elements
// in rows of 1024: pack 37 us, unpack 35; by rows, as below, in rows of 1000: 49 and 41).  A thread owns 16 elements (half a
// group, one shuffle for the maximum), so that every access is 16 bytes wide; ITEMS of them in flight.
template <typename T, int ITEMS>
__global__ void __launch_bounds__(PACK_THREADS) pack_flat_kernel(const T* __restrict__ x, uint4* __restrict__ q,
                                                                 uint8_t* __restrict__ e, int64_t n16) {
  const int64_t base = ((int64_t)blockIdx.x * ITEMS) * PACK_THREADS + threadIdx.x;
  Raw16<T> raw[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (base + i * PACK_THREADS < n16) raw[i].load(x + (base + i * PACK_THREADS) * 16);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = base + i * PACK_THREADS;
    float f[16];
    raw[i].get(f);
    uint32_t m = 0;
    if (at < n16) {
#pragma unroll
      for (int j = 0; j < 16; ++j) m = max(m, finite_abs_bits(f[j]));
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));          // n16 is even: both halves of a group exist or neither
    if (at < n16) {
      const uint32_t b = group_exponent(m);
      const float inv = inv_scale(b);
      if (b == TOP_EXPONENT) keep_finite(f);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = pack4(code_of(f[4 * j], inv), code_of(f[4 * j + 1], inv), code_of(f[4 * j + 2], inv), code_of(f[4 * j + 3], inv));
      __stcs(q + at, make_uint4(w[0], w[1], w[2], w[3]));
      if ((at & 1) == 0) e[at >> 1] = (uint8_t)b;
    }
  }
}

template <typename T, int ITEMS>
__global__ void __launch_bounds__(PACK_THREADS) unpack_flat_kernel(const uint4* __restrict__ q, const uint8_t* __restrict__ e,
                                                                   T* __restrict__ x, int64_t n16) {
  const int64_t base = ((int64_t)blockIdx.x * ITEMS) * PACK_THREADS + threadIdx.x;
  uint4 raw[ITEMS];
  uint32_t ex[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = base + i * PACK_THREADS;
    if (at < n16) {
      raw[i] = __ldcs(q + at);
      ex[i] = e[at >> 1];
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t at = base + i * PACK_THREADS;
    if (at >= n16) break;
    const float s = __uint_as_float(ex[i] << 23);
    const uint32_t w[4] = {raw[i].x ^ 0x80808080u, raw[i].y ^ 0x80808080u, raw[i].z ^ 0x80808080u, raw[i].w ^ 0x80808080u};
    float f[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = value_of(w[j >> 2], j & 3, s);
    if constexpr (sizeof(T) == 2) {
      uint4* d = reinterpret_cast<uint4*>(x + at * 16);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        __stcs(d + h, make_uint4(pack_bf16(f[8 * h], f[8 * h + 1]), pack_bf16(f[8 * h + 2], f[8 * h + 3]),
                                 pack_bf16(f[8 * h + 4], f[8 * h + 5]), pack_bf16(f[8 * h + 6], f[8 * h + 7])));
    } else {
      float4* d = reinterpret_cast<float4*>(x + at * 16);
#pragma unroll
      for (int h = 0; h < 4; ++h) __stcs(d + h, make_float4(f[4 * h], f[4 * h + 1], f[4 * h + 2], f[4 * h + 3]));
    }
  }
}

// Any width, any row stride: four lanes own a group, eight elements each, in accesses of W elements (8, 4, 2 or 1: what the width,
// the row stride and the addresses allow) that the lanes take in turn, so that one access of the four lies side by side.
// ROW_ITEMS groups a lane in flight.  Both directions of 67 million bfloat16 elements in rows of 1000: 90 us (4.5 TB/s; eight lanes
// of four elements took 109), of 250: 113 us; odd widths move single bytes: 201 us in rows of 251.  Every lane of a warp takes part
// in the shuffles; the ones past the end hold nothing.
constexpr int ROW_ITEMS = 2, LANE_ELEMS = 8, GROUP_LANES = PACK_GROUP / LANE_ELEMS;
constexpr int ROW_GROUPS = PACK_THREADS / GROUP_LANES;                 // groups a block and item

// n / d for n < 2^31 without a division: (high word of n m, plus n) >> s, with 2^s the power of two at or above d and
// m = floor(2^32 (2^s - d) / d) + 1 (Granlund and Montgomery, Division by Invariant Integers using Multiplication, 1994)
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t d_) : d(d_), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

// W elements between memory and registers in the widest accesses (16 bytes at most)
template <int W> __device__ __forceinline__ void load_w(const __nv_bfloat16* p, float* f) {
  if constexpr (W == 8) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
    unpack_bf16(u.x, f[0], f[1]);
    unpack_bf16(u.y, f[2], f[3]);
    unpack_bf16(u.z, f[4], f[5]);
    unpack_bf16(u.w, f[6], f[7]);
  } else if constexpr (W == 4) {
    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
    unpack_bf16(u.x, f[0], f[1]);
    unpack_bf16(u.y, f[2], f[3]);
  } else if constexpr (W == 2) {
    unpack_bf16(__ldcs(reinterpret_cast<const uint32_t*>(p)), f[0], f[1]);
  } else {
    f[0] = ldf(p);
  }
}
template <int W> __device__ __forceinline__ void load_w(const float* p, float* f) {
  if constexpr (W >= 4) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const float4 u = __ldcs(reinterpret_cast<const float4*>(p + i));
      f[i] = u.x; f[i + 1] = u.y; f[i + 2] = u.z; f[i + 3] = u.w;
    }
  } else if constexpr (W == 2) {
    const float2 u = __ldcs(reinterpret_cast<const float2*>(p));
    f[0] = u.x; f[1] = u.y;
  } else {
    f[0] = __ldcs(p);
  }
}
template <int W> __device__ __forceinline__ void store_w(__nv_bfloat16* p, const float* f) {
  if constexpr (W == 8)
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])));
  else if constexpr (W == 4) __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3])));
  else if constexpr (W == 2) __stcs(reinterpret_cast<uint32_t*>(p), pack_bf16(f[0], f[1]));
  else stf(p, f[0]);
}
template <int W> __device__ __forceinline__ void store_w(float* p, const float* f) {
  if constexpr (W >= 4) {
#pragma unroll
    for (int i = 0; i < W; i += 4) __stcs(reinterpret_cast<float4*>(p + i), make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]));
  } else if constexpr (W == 2) __stcs(reinterpret_cast<float2*>(p), make_float2(f[0], f[1]));
  else __stcs(p, f[0]);
}
// bytes j .. j + W - 1 of the eight codes in w
template <int W> __device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t (&w)[2], int j) {
  if constexpr (W == 8) __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
  else if constexpr (W == 4) __stcs(reinterpret_cast<uint32_t*>(p), w[j >> 2]);
  else if constexpr (W == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)(w[j >> 2] >> (8 * (j & 3)));
  else *p = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
}
template <int W> __device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t (&w)[2], int j) {
  if constexpr (W == 8) {
    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
    w[0] = u.x; w[1] = u.y;
  } else if constexpr (W == 4) w[j >> 2] = __ldcs(reinterpret_cast<const uint32_t*>(p));
  else if constexpr (W == 2) w[j >> 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p) << (8 * (j & 3));
  else w[j >> 2] |= (uint32_t)*p << (8 * (j & 3));
}

template <typename T, int W>
__global__ void __launch_bounds__(PACK_THREADS) pack_rows_kernel(const T* __restrict__ x, int64_t xrs, uint8_t* __restrict__ q,
                                                                 uint8_t* __restrict__ e, uint32_t groups, int D, const FastDiv G) {
  const int sub = threadIdx.x % GROUP_LANES;
  const uint32_t first = blockIdx.x * (ROW_ITEMS * ROW_GROUPS) + threadIdx.x / GROUP_LANES;
  float f[ROW_ITEMS][LANE_ELEMS];
#pragma unroll
  for (int i = 0; i < ROW_ITEMS; ++i) {
    const uint32_t gid = first + i * ROW_GROUPS, row = G.quotient(gid);
    const int c = (int)(gid - row * G.d) * PACK_GROUP + sub * W;
#pragma unroll
    for (int j = 0; j < LANE_ELEMS; ++j) f[i][j] = 0.f;
#pragma unroll
    for (int j = 0; j < LANE_ELEMS; j += W)
      if (gid < groups && c + j * GROUP_LANES < D) load_w<W>(x + (int64_t)row * xrs + c + j * GROUP_LANES, f[i] + j);
  }
#pragma unroll
  for (int i = 0; i < ROW_ITEMS; ++i) {
    const uint32_t gid = first + i * ROW_GROUPS, row = G.quotient(gid);
    const int c = (int)(gid - row * G.d) * PACK_GROUP + sub * W;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < LANE_ELEMS; ++j) m = max(m, finite_abs_bits(f[i][j]));
#pragma unroll
    for (int o = 1; o < GROUP_LANES; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (gid < groups) {
      const uint32_t b = group_exponent(m);
      if (sub == 0) e[gid] = (uint8_t)b;
      const float inv = inv_scale(b);
      if (b == TOP_EXPONENT) keep_finite(f[i]);
      uint32_t w[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        w[j] = pack4(code_of(f[i][4 * j], inv), code_of(f[i][4 * j + 1], inv), code_of(f[i][4 * j + 2], inv), code_of(f[i][4 * j + 3], inv));
#pragma unroll
      for (int j = 0; j < LANE_ELEMS; j += W)
        if (c + j * GROUP_LANES < D) store_codes<W>(q + (int64_t)row * D + c + j * GROUP_LANES, w, j);
    }
  }
}

template <typename T, int W>
__global__ void __launch_bounds__(PACK_THREADS) unpack_rows_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e,
                                                                   T* __restrict__ x, uint32_t groups, int D, const FastDiv G) {
  const int sub = threadIdx.x % GROUP_LANES;
  const uint32_t first = blockIdx.x * (ROW_ITEMS * ROW_GROUPS) + threadIdx.x / GROUP_LANES;
  uint32_t w[ROW_ITEMS][2], ex[ROW_ITEMS];
#pragma unroll
  for (int i = 0; i < ROW_ITEMS; ++i) {
    const uint32_t gid = first + i * ROW_GROUPS, row = G.quotient(gid);
    const int c = (int)(gid - row * G.d) * PACK_GROUP + sub * W;
    w[i][0] = w[i][1] = ex[i] = 0u;
    if (gid < groups) {
#pragma unroll
      for (int j = 0; j < LANE_ELEMS; j += W)
        if (c + j * GROUP_LANES < D) load_codes<W>(q + (int64_t)row * D + c + j * GROUP_LANES, w[i], j);
      ex[i] = e[gid];
    }
  }
#pragma unroll
  for (int i = 0; i < ROW_ITEMS; ++i) {
    const uint32_t gid = first + i * ROW_GROUPS, row = G.quotient(gid);
    const int c = (int)(gid - row * G.d) * PACK_GROUP + sub * W;
    const float s = __uint_as_float(ex[i] << 23);
    float f[LANE_ELEMS];
#pragma unroll
    for (int j = 0; j < LANE_ELEMS; ++j) f[j] = value_of(w[i][j >> 2] ^ 0x80808080u, j & 3, s);
#pragma unroll
    for (int j = 0; j < LANE_ELEMS; j += W)
      if (gid < groups && c + j * GROUP_LANES < D) store_w<W>(x + (int64_t)row * D + c + j * GROUP_LANES, f + j);
  }
}

// elements an access may hold: rows begin at multiples of it on both sides (an access of values is 16 bytes at most)
template <typename T> static int row_width(const void* x, int64_t xrs, const void* q, int D) {
  for (int w = 8; w > 1; w >>= 1) {
    const uintptr_t bytes = w * sizeof(T) < 16 ? w * sizeof(T) : 16;
    if (D % w == 0 && xrs % w == 0 && reinterpret_cast<uintptr_t>(x) % bytes == 0 && reinterpret_cast<uintptr_t>(q) % w == 0) return w;
  }
  return 1;
}
// rows a launch takes: its groups are counted in 31 bits, the last block's overhang included
static int64_t rows_a_launch(int64_t G) { return ((1LL << 31) - ROW_ITEMS * ROW_GROUPS) / G; }

constexpr int64_t PACK_MAX_BLOCKS = 0x7fffffffLL;

template <typename T>
static int pack_t(const void* x, int64_t xrs, void* q, void* e, int64_t M, int D, cudaStream_t st) {
  const int G = (D + PACK_GROUP - 1) / PACK_GROUP;
  if (D % PACK_GROUP == 0 && xrs == D && aligned16(x) && aligned16(q)) {
    constexpr int ITEMS = sizeof(T) == 2 ? 2 : 1;
    const int64_t n16 = M * D / 16, blocks = (n16 + ITEMS * PACK_THREADS - 1) / (ITEMS * PACK_THREADS);
    ORBIT_REQUIRE(blocks <= PACK_MAX_BLOCKS, ERR_UNSUPPORTED, "orbit_act_pack: %lld elements are too many for one call", (long long)(M * D));
    pack_flat_kernel<T, ITEMS><<<(unsigned)blocks, PACK_THREADS, 0, st>>>((const T*)x, (uint4*)q, (uint8_t*)e, n16);
    ORBIT_CHECK_LAUNCH("pack_flat_kernel");
    return OK;
  }
  const int w = row_width<T>(x, xrs, q, D);
  const int64_t most = rows_a_launch(G);
  for (int64_t r = 0; r < M; r += most) {
    const uint32_t groups = (uint32_t)((M - r < most ? M - r : most) * G), blocks = (groups + ROW_ITEMS * ROW_GROUPS - 1) / (ROW_ITEMS * ROW_GROUPS);
    const T* xr = (const T*)x + r * xrs;
    uint8_t *qr = (uint8_t*)q + r * D, *er = (uint8_t*)e + r * G;
    if (w == 8) pack_rows_kernel<T, 8><<<blocks, PACK_THREADS, 0, st>>>(xr, xrs, qr, er, groups, D, FastDiv(G));
    else if (w == 4) pack_rows_kernel<T, 4><<<blocks, PACK_THREADS, 0, st>>>(xr, xrs, qr, er, groups, D, FastDiv(G));
    else if (w == 2) pack_rows_kernel<T, 2><<<blocks, PACK_THREADS, 0, st>>>(xr, xrs, qr, er, groups, D, FastDiv(G));
    else pack_rows_kernel<T, 1><<<blocks, PACK_THREADS, 0, st>>>(xr, xrs, qr, er, groups, D, FastDiv(G));
    ORBIT_CHECK_LAUNCH("pack_rows_kernel");
  }
  return OK;
}

template <typename T>
static int unpack_t(const void* q, const void* e, void* x, int64_t M, int D, cudaStream_t st) {
  const int G = (D + PACK_GROUP - 1) / PACK_GROUP;
  if (D % PACK_GROUP == 0 && aligned16(x) && aligned16(q)) {
    constexpr int ITEMS = 2;
    const int64_t n16 = M * D / 16, blocks = (n16 + ITEMS * PACK_THREADS - 1) / (ITEMS * PACK_THREADS);
    ORBIT_REQUIRE(blocks <= PACK_MAX_BLOCKS, ERR_UNSUPPORTED, "orbit_act_unpack: %lld elements are too many for one call", (long long)(M * D));
    unpack_flat_kernel<T, ITEMS><<<(unsigned)blocks, PACK_THREADS, 0, st>>>((const uint4*)q, (const uint8_t*)e, (T*)x, n16);
    ORBIT_CHECK_LAUNCH("unpack_flat_kernel");
    return OK;
  }
  const int w = row_width<T>(x, D, q, D);
  const int64_t most = rows_a_launch(G);
  for (int64_t r = 0; r < M; r += most) {
    const uint32_t groups = (uint32_t)((M - r < most ? M - r : most) * G), blocks = (groups + ROW_ITEMS * ROW_GROUPS - 1) / (ROW_ITEMS * ROW_GROUPS);
    const uint8_t *qr = (const uint8_t*)q + r * D, *er = (const uint8_t*)e + r * G;
    T* xr = (T*)x + r * D;
    if (w == 8) unpack_rows_kernel<T, 8><<<blocks, PACK_THREADS, 0, st>>>(qr, er, xr, groups, D, FastDiv(G));
    else if (w == 4) unpack_rows_kernel<T, 4><<<blocks, PACK_THREADS, 0, st>>>(qr, er, xr, groups, D, FastDiv(G));
    else if (w == 2) unpack_rows_kernel<T, 2><<<blocks, PACK_THREADS, 0, st>>>(qr, er, xr, groups, D, FastDiv(G));
    else unpack_rows_kernel<T, 1><<<blocks, PACK_THREADS, 0, st>>>(qr, er, xr, groups, D, FastDiv(G));
    ORBIT_CHECK_LAUNCH("unpack_rows_kernel");
  }
  return OK;
}

}  // namespace orbit

using namespace orbit;

extern "C" int orbit_act_pack(const void* x, int64_t x_row_stride, void* q, void* exponent, int64_t M, int D, int dtype, void* stream) {
  ORBIT_REQUIRE(M >= 0 && D > 0, ERR_BAD_ARG, "orbit_act_pack: bad sizes M=%lld D=%d", (long long)M, D);
  ORBIT_REQUIRE(dtype == BF16 || dtype == F32, ERR_BAD_ARG, "orbit_act_pack: unknown dtype code %d", dtype);
  if (M == 0) return OK;
  ORBIT_REQUIRE(x && q && exponent, ERR_BAD_ARG, "orbit_act_pack: null pointer");
  return dtype == BF16 ? pack_t<__nv_bfloat16>(x, x_row_stride, q, exponent, M, D, (cudaStream_t)stream)
                       : pack_t<float>(x, x_row_stride, q, exponent, M, D, (cudaStream_t)stream);
}

extern "C" int orbit_act_unpack(const void* q, const void* exponent, void* x, int64_t M, int D, int dtype, void* stream) {
  ORBIT_REQUIRE(M >= 0 && D > 0, ERR_BAD_ARG, "orbit_act_unpack: bad sizes M=%lld D=%d", (long long)M, D);
  ORBIT_REQUIRE(dtype == BF16 || dtype == F32, ERR_BAD_ARG, "orbit_act_unpack: unknown dtype code %d", dtype);
  if (M == 0) return OK;
  ORBIT_REQUIRE(x && q && exponent, ERR_BAD_ARG, "orbit_act_unpack: null pointer");
  return dtype == BF16 ? unpack_t<__nv_bfloat16>(q, exponent, x, M, D, (cudaStream_t)stream)
                       : unpack_t<float>(q, exponent, x, M, D, (cudaStream_t)stream);
}
