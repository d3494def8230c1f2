// Rows of heads for the cache kernels: loads and stores of 16- and 32-bit rows, the norm and
// the rotation of a row, and what the writes ask of their arguments.
#pragma once

#include <cmath>

#include "kernels.h"

namespace b200moe {
namespace {

constexpr int MAX_NEW_TOKENS = 16;

inline bool dtype_ok(int dt) { return dt == B200MOE_DT_F32 || dt == B200MOE_DT_F16 || dt == B200MOE_DT_BF16; }
inline size_t dt_bytes(int dt) { return dt == B200MOE_DT_F32 ? 4 : 2; }
// log2 of a power of two, -1 of another number
inline int log2_of(int n) {
  for (int i = 0; i < 31; ++i)
    if (n == 1 << i) return i;
  return -1;
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ------------------------------------------------------------- rows of 16 or 32 bits
// Eight consecutive elements as they lie in memory: one or two 16-byte words.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = e[i];
      else if constexpr (std::is_same<T, __half>::value) v[i] = __half2float(e[i]);
      else v[i] = __bfloat162float(e[i]);
    }
  }
};
__device__ __forceinline__ uint32_t pack2(const __half*, float a, float b) { return h2_as_u32(__floats2half2_rn(a, b)); }
__device__ __forceinline__ uint32_t pack2(const __nv_bfloat16*, float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(p, v[0], v[1]), pack2(p, v[2], v[3]), pack2(p, v[4], v[5]), pack2(p, v[6], v[7]));
  }
}
template <typename T>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(__float2half_rn(v));
  else return __bfloat162float(__float2bfloat16_rn(v));
}
// 2 or 4 consecutive elements; stored as a type known at run time
template <int N>
__device__ __forceinline__ void load_elems(const float* p, float (&v)[N]) {
  if constexpr (N == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
    const float2 a = *reinterpret_cast<const float2*>(p);
    v[0] = a.x; v[1] = a.y;
  }
}
template <int N>
__device__ __forceinline__ void store_as(void* p, int dtype, size_t i, const float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    if (dtype == B200MOE_DT_F32) *reinterpret_cast<float2*>(static_cast<float*>(p) + i + j) = make_float2(v[j], v[j + 1]);
    else if (dtype == B200MOE_DT_F16)
      *reinterpret_cast<__half2*>(static_cast<__half*>(p) + i + j) = __floats2half2_rn(v[j], v[j + 1]);
    else
      *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p) + i + j) = __floats2bfloat162_rn(v[j], v[j + 1]);
  }
}

// ------------------------------------------------------------------------- write
struct WriteArgs {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const float *q_norm, *k_norm;
  float eps;
  void *q_out, *k_out;
  void* slab;
  float* scales;                      // 8-bit cache
  int cache_dtype;                    // 16- or 32-bit cache
  const int32_t *start_positions, *new_lens, *page_ids;
  const float* freqs;
  int order, bs, sl, pages_per_seq, page_count, heads, kv_heads, stride, blocks, block_index, scale_block;
  int tiles;                          // of a sequence
  int stride_shift, block_shift;      // log2; -1 where the stride is no power of two
  unsigned kv_ctas;                   // CTAs of K and V
  int q_heads;                        // heads that a lane of the others takes
  int32_t* status;
};

// Cosine and sine of position * freq, the angle reduced to part of a turn first.
// 32-bit rows, and far angles: reduced in 64 bits; the half turns are rounded by 2^-25, which
// is pi 2^-25 of angle, and sincospif is good to an ulp or two: 2^-22 up to 2^25 turns (the
// products in 64 bits are off by 2^-52 of the turns, which shows above).
// 16-bit rows: the position (below 2^24, exact) times freq / (2 pi) as the sum of two floats
// u + u_lo.  Below 2^22 turns u_lo is at most an eighth, so that the integer part is dropped
// before and after the sum: the special-function unit's bounds hold within a turn only, 2^-21.4
// (sine) and 2^-21.2.  The sum is rounded by 2^-25 of a turn, the product with 2 pi by 2^-23
// and 2 pi itself by 2^-25 of it: 2^-20 in all, a 256th of half a step of fp16 just below one,
// and 1e-4 of a step of int8.  (With power series, good to 2^-22: 49.0 instead of 47.4 us for
// 4 x 2048 tokens of 48 + 16 heads, 8.0 instead of 7.2 for 777 of 32 + 8, and the same error of
// q, k and K's codes against 64 bits in three digits; sincospif 48.4 and 8.0.)
template <typename T>
__device__ __forceinline__ float2 cos_sin(long long pos, float freq) {
  constexpr double inv = 0.15915494309189533577;  // 1 / (2 pi)
  constexpr float inv_hi = static_cast<float>(inv), inv_lo = static_cast<float>(inv - inv_hi);
  const float p = static_cast<float>(static_cast<int>(pos)), g = freq * inv_hi, u = p * g;
  float sn, cs;
  if (sizeof(T) == 4 || pos >= 1 << 24 || !(fabsf(u) < 4194304.f)) {
    const double turns = static_cast<double>(pos) * (static_cast<double>(freq) * (2.0 * inv));  // halves
    sincospif(static_cast<float>(turns - 2.0 * rint(0.5 * turns)), &sn, &cs);
  } else {
    const float g_lo = fmaf(freq, inv_hi, -g) + freq * inv_lo, u_lo = fmaf(p, g_lo, fmaf(p, g, -u));
    const float r = (u - rintf(u)) + u_lo, angle = (r - rintf(r)) * 6.2831853071795864769f;
    sn = __sinf(angle);
    cs = __cosf(angle);
  }
  return make_float2(cs, sn);
}
// The eight elements of a row that lane c of HD / 8 has, so that it has whole pairs: in order
// 0 (pairs 2i, 2i + 1) elements 8c .. 8c + 7, in the HuggingFace order (pairs i, i + HD / 2)
// 4c .. 4c + 3 and as many behind HD / 2.  Its pairs' frequencies are 4c .. 4c + 3 either way.
template <int HD, int ORDER>
__device__ __forceinline__ int element(int c, int i) {
  return ORDER == 0 ? 8 * c + i : (i < 4 ? 4 * c + i : HD / 2 + 4 * c + i - 4);
}
template <typename T, int HD, int ORDER>
__device__ __forceinline__ void load_row(Raw8<T>& x, const T* row, int c) {
  if constexpr (ORDER == 0) {
    x.load(row + 8 * c);
  } else if constexpr (sizeof(T) == 4) {
    x.w[0] = *reinterpret_cast<const uint4*>(row + 4 * c);
    x.w[1] = *reinterpret_cast<const uint4*>(row + HD / 2 + 4 * c);
  } else {
    const uint2 lo = *reinterpret_cast<const uint2*>(row + 4 * c), hi = *reinterpret_cast<const uint2*>(row + HD / 2 + 4 * c);
    x.w[0] = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
}
template <typename T, int HD, int ORDER>
__device__ __forceinline__ void store_row(T* row, int c, const float (&v)[8]) {
  if constexpr (ORDER == 0) {
    store8(row + 8 * c, v);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(row + 4 * c) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(row + HD / 2 + 4 * c) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint2*>(row + 4 * c) = make_uint2(pack2(row, v[0], v[1]), pack2(row, v[2], v[3]));
    *reinterpret_cast<uint2*>(row + HD / 2 + 4 * c) = make_uint2(pack2(row, v[4], v[5]), pack2(row, v[6], v[7]));
  }
}

// Cosines and sines of a lane's four pairs.
struct Turn { float2 t[4]; };
template <typename T>
__device__ __forceinline__ Turn turn_of(long long pos, const float* freqs, int c) {
  Turn w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w.t[i] = cos_sin<T>(pos, freqs[4 * c + i]);
  return w;
}
// A lane's eight elements of a row, normed and rotated; LPR lanes have a row.
template <int LPR, int ORDER>
__device__ __forceinline__ void norm_rotate(float (&x)[8], const float (&w)[8], bool norm, float eps, const Turn& turn) {
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss * (1.f / (8 * LPR)) + eps);  // 2^-22; root and division cost a tenth of the kernel
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = w[i] * (x[i] * r);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    constexpr int STEP = ORDER == 0 ? 2 : 1, OTHER = ORDER == 0 ? 1 : 4;
    const float re = x[STEP * i], im = x[STEP * i + OTHER];
    x[STEP * i] = re * turn.t[i].x - im * turn.t[i].y;
    x[STEP * i + OTHER] = im * turn.t[i].x + re * turn.t[i].y;
  }
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What both writes ask of their arguments.
int check_write(const char* who, const WriteArgs& a, int io_dtype, int hd) {
  B200_REQUIRE(a.bs >= 0 && a.sl >= 1 && a.pages_per_seq >= 1 && a.heads >= 1, "%s: bad sizes", who);
  if (a.bs == 0) return B200MOE_OK;
  B200_REQUIRE(a.q && a.k && a.v && a.q_out && a.slab && a.start_positions && a.page_ids && a.freqs, "%s: NULL buffer",
               who);
  B200_REQUIRE(dtype_ok(io_dtype), "%s: unknown dtype", who);
  B200_REQUIRE(a.order == 0 || a.order == 1, "%s: rotation order %d (0 and 1 are known)", who, a.order);
  B200_REQUIRE(hd == 64 || hd == 128, "%s: head_dim %d (64 and 128 are built)", who, hd);
  B200_REQUIRE(a.kv_heads >= 1 && a.heads % a.kv_heads == 0, "%s: heads (%d) must be a multiple of the kv heads (%d)",
               who, a.heads, a.kv_heads);
  B200_REQUIRE(a.kv_heads <= 65535, "%s: kv_heads %d", who, a.kv_heads);
  B200_REQUIRE(a.stride >= 1 && a.blocks >= 1 && a.block_index >= 0 && a.block_index < a.blocks && a.page_count >= 1,
               "%s: bad cache geometry", who);
  const int64_t per16 = 16 / static_cast<int64_t>(dt_bytes(io_dtype));
  B200_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.q_out) && aligned16(a.k_out) &&
                   aligned16(a.slab) && a.q_stride % per16 == 0 && a.k_stride % per16 == 0 && a.v_stride % per16 == 0,
               "%s: buffers and row strides must be multiples of 16 bytes", who);
  B200_REQUIRE(a.q_stride >= static_cast<int64_t>(a.heads) * hd && a.k_stride >= static_cast<int64_t>(a.kv_heads) * hd &&
                   a.v_stride >= static_cast<int64_t>(a.kv_heads) * hd,
               "%s: a row stride is shorter than the row", who);
  B200_REQUIRE(a.k_out != a.k && a.k_out != a.v && a.q_out != a.k && a.q_out != a.v && a.k_out != a.q && a.q_out != a.q &&
                   a.q_out != a.k_out,
               "%s: q_out and k_out must not be inputs", who);
  // CTAs of K and V, and at most one for each 16 heads of a token
  const double grid = static_cast<double>(a.bs) * ((a.sl - 1) / 32 + 2) * a.kv_heads +
                      static_cast<double>(a.bs) * a.sl * (a.heads / 4 + 1) / 16 + 1;
  B200_REQUIRE(grid < 2147483647.0, "%s: %d sequences of %d tokens are too many for one call", who, a.bs, a.sl);
  return B200MOE_OK;
}

}  // namespace
}  // namespace b200moe
