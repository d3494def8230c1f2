// The 8-bit KV cache: its write (norms of queries and keys, rotation and quantisation in
// one pass), its read-back, and attention over it.
//
// Slab: [page][transformer block][kv head][K | V][position in page][head dim] codes of one
// byte, int8 or e4m3; scales: [page][transformer block][kv head][scale block][K | V] fp32.
// A code c stands for c * s.
#include <cuda_fp8.h>

#include <cmath>

#include "kernels.h"

namespace b200moe {
namespace {

constexpr int MAX_SCALE_BLOCK = 64;
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

// ------------------------------------------------------------------------- codes
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v & 0xffffu), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}
// Four codes as two fp16 pairs for the MMAs, exact: bytes (0, 2) and (1, 3).
// int8: 0x6400 | b is the fp16 number 1024 + b; the byte is biased to unsigned first.
// e4m3: its exponent and mantissa moved to fp16's places are the value times 2^-8 (the two
// biases differ by 8; subnormal codes become subnormal fp16 numbers), which goes into the
// scale: E4M3_UNIT.  Seven integer instructions, against three or four with the conversion
// instruction, which takes longer than they (42 us at 32 x 4000 positions, with it 51).
constexpr float E4M3_UNIT = 256.f;
template <int CODE>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& even, uint32_t& odd) {
  if constexpr (CODE == B200MOE_KV8_INT8) {
    const uint32_t x = w ^ 0x80808080u;
    const __half2 bias = u32_as_h2(0x64806480u);
    even = h2_as_u32(__hsub2(u32_as_h2(__byte_perm(x, 0x64646464u, 0x4240)), bias));
    odd = h2_as_u32(__hsub2(u32_as_h2(__byte_perm(x, 0x64646464u, 0x4341)), bias));
  } else {
    even = ((w << 7) & 0x3f803f80u) | ((w << 8) & 0x80008000u);
    odd = ((w >> 1) & 0x3f803f80u) | (w & 0x80008000u);
  }
}
template <int CODE, int N>
__device__ __forceinline__ void codes_to_floats(const uint32_t (&c)[N / 4], float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const uint32_t w = c[i];
    float2 f[2];
    if constexpr (CODE == B200MOE_KV8_INT8) {
      uint32_t even, odd;
      widen4<CODE>(w, even, odd);
      const float2 e = __half22float2(u32_as_h2(even)), o = __half22float2(u32_as_h2(odd));
      f[0] = make_float2(e.x, o.x);
      f[1] = make_float2(e.y, o.y);
    } else {
      f[0] = __half22float2(u32_as_h2(e4m3x2_to_h2(w)));
      f[1] = __half22float2(u32_as_h2(e4m3x2_to_h2(w >> 16)));
    }
    v[4 * i] = f[0].x; v[4 * i + 1] = f[0].y; v[4 * i + 2] = f[1].x; v[4 * i + 3] = f[1].y;
  }
}
// v[i] * (by + by_lo), values / scale at most 2^-10 above qmax, to the nearest codes: without
// clamping.  The factor is the sum of two floats because quotients halfway between two codes
// are common (half of the largest value of an int8 block is 63.5 steps): the product has to be
// that number again, to go to the even code, and with a factor off by 2^-24 it falls to either
// side.  (With one float the error of V against codes from 64-bit quotients is a tenth larger
// for bf16 rows and almost twice as large for fp16, all of it from these.)
template <int CODE>
__device__ __forceinline__ uint2 floats_to_codes(const float (&v)[8], float by, float by_lo) {
  uint32_t c[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = fmaf(v[4 * i + j], by, v[4 * i + j] * by_lo);
    if constexpr (CODE == B200MOE_KV8_INT8) {
      // in the last place of 1.5 * 2^23 + y stands y, rounded to even, in two's complement
      uint32_t n[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) n[j] = __float_as_uint(y[j] + 12582912.f);
      c[i] = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
    } else {
      c[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3) |
             static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3)) << 16;
    }
  }
  return make_uint2(c[0], c[1]);
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

enum { CACHE_INT8 = B200MOE_KV8_INT8, CACHE_E4M3 = B200MOE_KV8_E4M3, CACHE_PLAIN = 2 };

constexpr int WR_THREADS = 256;
constexpr int WR_WARPS = WR_THREADS / 32;
constexpr float QMAX[2] = {127.f, 448.f};

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
// max(m, |x|) for m >= 0, NaN where either is
__device__ __forceinline__ float max_nan(float m, float x) {
  float y;
  asm("{.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;}" : "=f"(y) : "f"(m), "f"(x));
  return y;
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
template <int HD, int ORDER>
__device__ __forceinline__ void store_codes(uint8_t* row, int c, uint2 v) {
  if constexpr (ORDER == 0) {
    *reinterpret_cast<uint2*>(row + 8 * c) = v;
  } else {
    *reinterpret_cast<uint32_t*>(row + 4 * c) = v.x;
    *reinterpret_cast<uint32_t*>(row + HD / 2 + 4 * c) = v.y;
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
// The scale of a block from the largest magnitude of its new rows (as bits) and, if it is
// continued, the scale it had (else 0); the factor to codes, qmax / amax of a fresh block and
// 1 / scale of a continued one, as an approximate reciprocal (scales are below 2^122) and what
// it lacks; and what the earlier codes are multiplied by: the scale grows by powers of two.
struct BlockScale { float s, inv, inv_lo, shrink; };
template <int KIND>
__device__ __forceinline__ BlockScale block_scale(unsigned bits, float before) {
  constexpr float qmax = QMAX[KIND], tiny = 7.888609052210118e-31f;  // 2^-100
  const float amax = __uint_as_float(bits);
  BlockScale r;
  r.inv = r.inv_lo = 0.f;
  r.shrink = 1.f;
  if (bits >= 0x7f800000u || before != before) {
    r.s = __uint_as_float(0x7fc00000u);
  } else if (before > 0.f) {
    r.s = before;
    // the smallest e with amax <= fits * 2^e, from the two exponents: their quotient can be beyond 2^128
    const float fits = before * qmax * (1.f + 0.0009765625f);
    if (amax > fits) {
      int ea, ef;
      const float ma = frexpf(amax, &ea), mf = frexpf(fits, &ef);
      const int e = ea - ef + (ma > mf);
      r.s = ldexpf(before, e);
      r.shrink = ldexpf(1.f, -e);
    }
    r.inv = rcp(r.s);
    r.inv_lo = fmaf(-r.inv, r.s, 1.f) * r.inv;
  } else if (amax < qmax * tiny) {
    r.s = 0.f;
  } else {
    r.s = amax / qmax;
    r.inv = rcp(r.s);
    r.inv_lo = fmaf(-r.inv, amax, qmax) * (r.inv * (1.f / qmax));
  }
  return r;
}

// Two kinds of CTAs.  kv_ctas of them have a (sequence, tile of TILE positions, kv head)
// each: its K and V.  Tiles are aligned in absolute positions, so that a tile holds whole
// scale blocks; K and V stay in registers from their load to their codes: one read of
// everything.  The others have the queries: a lane keeps its position's cosines and sines
// and takes four heads at once, q_heads in all.  HD / 8 lanes have a row (16-byte loads and
// stores of 16-bit rows), a warp two or four rows.  Bound by memory and by instructions alike
// (63 % of the issue slots, and waits for the loads of four CTAs an SM): 4 x 2048 tokens of
// 48 + 16 heads (268 MB) take 47 to 48 us, 5.6 TB/s.  On
// the way there: K, V and the queries of a kv head in one CTA 79 (the queries waited for the
// barriers of K and V); CTAs of two kinds, three an SM 66, four 60 (five, registers in memory,
// 54 instead of 47 later on; heads of 64 take five, 4 to 16 bytes of a thread's registers in
// memory: 4 x 2048 tokens of 16 + 8 heads 12.8 instead of 13.7, 8 x 2048 of fp16 to e4m3 25.7
// instead of 27.3, 4 x 1024 to a 16-bit cache and one of 777 as with four); K's and V's CTAs
// among the others instead of before them 52; rounding of the codes by an addition and the
// approximate reciprocal root 47.
template <typename T, int HD, int KIND, int TILE, int ORDER>
__global__ void __launch_bounds__(WR_THREADS, TILE == 32 ? (sizeof(T) == 4 ? 3 : HD == 64 ? 5 : 4) : 2) norm_rope_write_kernel(const WriteArgs a) {
  constexpr int LPR = HD / 8, RPW = 32 / LPR;                 // lanes per row, rows of a warp
  constexpr int RPP = WR_WARPS * RPW;                         // rows of a pass
  constexpr int PASSES = (TILE + RPP - 1) / RPP;
  constexpr int QB = 4;                                       // heads that a lane takes at once
  __shared__ long long s_row[TILE];     // K row of each position in the slab, in rows of HD elements; -1: not written
  __shared__ unsigned s_amax[2][TILE];  // of each scale block, as bits
  __shared__ uint32_t s_pair[TILE];     // scale pair of each position
  __shared__ float2 s_before;           // scales of a continued block
  grid_dep_wait();
  grid_dep_launch();
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int sub = warp * RPW + lane / LPR, c = lane % LPR;    // row of a pass, chunk of eight elements
  const T *q = static_cast<const T*>(a.q), *k = static_cast<const T*>(a.k), *v = static_cast<const T*>(a.v);
  // K and V's CTAs are spread evenly among the others
  unsigned kv_before, rest;
  if (gridDim.x < 65536) {
    const unsigned x = blockIdx.x * a.kv_ctas;
    kv_before = x / gridDim.x;
    rest = x - kv_before * gridDim.x;
  } else {
    const unsigned long long x = static_cast<unsigned long long>(blockIdx.x) * a.kv_ctas;
    kv_before = static_cast<unsigned>(x / gridDim.x);
    rest = static_cast<unsigned>(x - static_cast<unsigned long long>(kv_before) * gridDim.x);
  }
  if (rest + a.kv_ctas < gridDim.x) {
    const long long tokens = static_cast<long long>(a.bs) * a.sl, groups = (a.heads + a.q_heads - 1) / a.q_heads;
    const long long mine = static_cast<long long>(blockIdx.x - kv_before) * RPP + sub;
    const bool some = mine < tokens * groups;
    const long long item = some ? mine : tokens * groups - 1;  // all lanes take part in the shuffles
    const long long tok = item % tokens;
    const int h0 = static_cast<int>(item / tokens) * a.q_heads, h1 = min(h0 + a.q_heads, a.heads);
    const int b = static_cast<int>(tok / a.sl);
    const T* from = q + tok * a.q_stride;
    T* to = static_cast<T*>(a.q_out) + tok * a.heads * HD;
    const long long pos = max(a.start_positions[b], 0) + (tok - static_cast<long long>(b) * a.sl);
    const Turn turn = turn_of<T>(pos, a.freqs, c);
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = a.q_norm != nullptr ? a.q_norm[element<HD, ORDER>(c, i)] : 1.f;
    // every lane of a warp makes the same number of steps: heads behind the last are read again and not stored
    for (int d = 0; d < a.q_heads; d += QB) {
      Raw8<T> raw[QB];
#pragma unroll
      for (int g = 0; g < QB; ++g) load_row<T, HD, ORDER>(raw[g], from + min(h0 + d + g, h1 - 1) * HD, c);
#pragma unroll
      for (int g = 0; g < QB; ++g) {
        float x[8];
        raw[g].get(x);
        norm_rotate<LPR, ORDER>(x, w, a.q_norm != nullptr, a.eps, turn);
        if (some && h0 + d + g < h1) store_row<T, HD, ORDER>(to + (h0 + d + g) * HD, c, x);
      }
    }
    return;
  }
  const int kvh = kv_before % a.kv_heads, tile = kv_before / a.kv_heads % a.tiles, b = kv_before / a.kv_heads / a.tiles;
  const int start_in = a.start_positions[b];
  const long long start = start_in < 0 ? 0 : start_in;
  int count = start_in < 0 ? 0 : a.new_lens != nullptr ? a.new_lens[b] : a.sl;
  count = count < 0 ? 0 : count > a.sl ? a.sl : count;
  const long long p0 = (start / TILE + tile) * TILE;  // first position of the tile
  const int lo = static_cast<int>(start > p0 ? start - p0 : 0);
  const long long end = start + a.sl - p0, wend = start + count - p0;
  const int hi = static_cast<int>(end < TILE ? end : TILE);     // rows lo .. hi are rotated,
  const int whi = static_cast<int>(wend < TILE ? wend : TILE);  // rows lo .. whi written
  if (lo >= hi) return;

  // K and V are on their way while the angles are computed
  const long long tok0 = static_cast<long long>(b) * a.sl + (p0 - start);  // token of row 0
  Raw8<T> kr[PASSES], vr[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = lo + i * RPP + sub;
    kr[i].zero();
    vr[i].zero();
    if (r < hi) load_row<T, HD, ORDER>(kr[i], k + (tok0 + r) * a.k_stride + kvh * HD, c);
    if (r < whi) load_row<T, HD, ORDER>(vr[i], v + (tok0 + r) * a.v_stride + kvh * HD, c);
  }
  // earlier rows of a continued block included, if anything is written
  const int first = KIND == CACHE_PLAIN || whi <= lo ? lo : lo >> a.block_shift << a.block_shift;
  for (int r = first + t; r < whi; r += WR_THREADS) {
    const uint32_t pos = static_cast<uint32_t>(p0 + r), slot = a.stride_shift >= 0 ? pos >> a.stride_shift : pos / a.stride;
    const uint32_t off = pos - slot * a.stride;
    long long row = -1;
    const int page = slot < static_cast<uint32_t>(a.pages_per_seq) ? a.page_ids[static_cast<size_t>(b) * a.pages_per_seq + slot] : -1;
    if (page < 0 || page >= a.page_count) {
      atomicOr(a.status, DEV_ERR_BOUNDS);
    } else if constexpr (KIND == CACHE_PLAIN) {
      row = ((static_cast<long long>(page) * a.blocks + a.block_index) * 2 * a.stride + off) * a.kv_heads + kvh;
    } else {
      const uint32_t head = (static_cast<uint32_t>(page) * a.blocks + a.block_index) * a.kv_heads + kvh;
      row = head * 2u * a.stride + off;
      s_pair[r] = head * static_cast<uint32_t>(a.stride >> a.block_shift) + (off >> a.block_shift);
      if (r < lo && r == first) s_before = reinterpret_cast<const float2*>(a.scales)[s_pair[r]];
    }
    s_row[r] = row;
  }
  for (int i = t; i < 2 * TILE; i += WR_THREADS) (&s_amax[0][0])[i] = 0u;
  __syncthreads();
  // the warps that have rows go on
  const int kv_warps = min((hi - lo + RPW - 1) / RPW, WR_WARPS);
  auto kv_sync = [&] { asm volatile("bar.sync 1, %0;" ::"r"(kv_warps * 32) : "memory"); };
  if (warp < kv_warps) {
    float w[8], kx[PASSES][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = a.k_norm != nullptr ? a.k_norm[element<HD, ORDER>(c, i)] : 1.f;
    // all lanes take part in the shuffles of the norm and the rotation; rows outside lo .. hi are zeros, unused
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = lo + i * RPP + sub;
      if (lo + i * RPP >= hi) break;
      kr[i].get(kx[i]);
      norm_rotate<LPR, ORDER>(kx[i], w, a.k_norm != nullptr, a.eps, turn_of<T>(p0 + r, a.freqs, c));
      if (r < hi && a.k_out != nullptr)
        store_row<T, HD, ORDER>(static_cast<T*>(a.k_out) + ((tok0 + r) * a.kv_heads + kvh) * HD, c, kx[i]);
      if constexpr (KIND == CACHE_PLAIN) {
        if (r < whi && s_row[r] >= 0) {
          float y[8];
          vr[i].get(y);
#pragma unroll
          for (int j = 0; j < 8; ++j) kx[i][j] = round_to<T>(kx[i][j]);
          const size_t at = static_cast<size_t>(s_row[r]) * HD, v_at = at + static_cast<size_t>(a.stride) * a.kv_heads * HD;
          if (a.cache_dtype == B200MOE_DT_F32) {
            store_row<float, HD, ORDER>(static_cast<float*>(a.slab) + at, c, kx[i]);
            store_row<float, HD, ORDER>(static_cast<float*>(a.slab) + v_at, c, y);
          } else if (a.cache_dtype == B200MOE_DT_F16) {
            store_row<__half, HD, ORDER>(static_cast<__half*>(a.slab) + at, c, kx[i]);
            store_row<__half, HD, ORDER>(static_cast<__half*>(a.slab) + v_at, c, y);
          } else {
            store_row<__nv_bfloat16, HD, ORDER>(static_cast<__nv_bfloat16*>(a.slab) + at, c, kx[i]);
            store_row<__nv_bfloat16, HD, ORDER>(static_cast<__nv_bfloat16*>(a.slab) + v_at, c, y);
          }
        }
      } else {
        // the largest magnitude of the row, then of its scale block, NaN above all
        float y[8];
        vr[i].get(y);
        float mk = 0.f, mv = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          mk = max_nan(mk, kx[i][j]);
          mv = max_nan(mv, y[j]);
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) {
          mk = max_nan(mk, __shfl_xor_sync(0xffffffffu, mk, o));
          mv = max_nan(mv, __shfl_xor_sync(0xffffffffu, mv, o));
        }
        if (c == 0 && r < whi) {
          atomicMax(&s_amax[0][r >> a.block_shift], __float_as_uint(mk));
          atomicMax(&s_amax[1][r >> a.block_shift], __float_as_uint(mv));
        }
      }
    }
    if constexpr (KIND != CACHE_PLAIN) {
      kv_sync();
      uint8_t* slab = static_cast<uint8_t*>(a.slab);
      const size_t v_off = static_cast<size_t>(a.stride) * HD;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int r = lo + i * RPP + sub;
        if (r >= whi || s_row[r] < 0) continue;
        // every lane computes the scales of its row's block; the block's first new row stores them
        const int blk = r >> a.block_shift, at_blk = max(blk << a.block_shift, lo);
        const bool continued = lo > blk << a.block_shift;
        const float2 before = continued ? s_before : make_float2(0.f, 0.f);
        const BlockScale ks = block_scale<KIND>(s_amax[0][blk], before.x), vs = block_scale<KIND>(s_amax[1][blk], before.y);
        if (r == at_blk && c == 0) reinterpret_cast<float2*>(a.scales)[s_pair[r]] = make_float2(ks.s, vs.s);
        uint8_t* at = slab + static_cast<size_t>(s_row[r]) * HD;
        store_codes<HD, ORDER>(at, c, floats_to_codes<KIND>(kx[i], ks.inv, ks.inv_lo));
        float y[8];
        vr[i].get(y);
        store_codes<HD, ORDER>(at + v_off, c, floats_to_codes<KIND>(y, vs.inv, vs.inv_lo));
      }
      // the live rows of a continued block whose scale has grown
      if (first < lo && s_row[lo] >= 0) {
        const int blk = first >> a.block_shift;
        const float k_shrink = block_scale<KIND>(s_amax[0][blk], s_before.x).shrink;
        const float v_shrink = block_scale<KIND>(s_amax[1][blk], s_before.y).shrink;
        for (int i = sub; i < 2 * (lo - first); i += kv_warps * RPW) {
          const int kv = i & 1, r = first + (i >> 1);
          const float shrink = kv ? v_shrink : k_shrink;
          if (shrink == 1.f) continue;
          uint2* at = reinterpret_cast<uint2*>(slab + static_cast<size_t>(s_row[r]) * HD + (kv ? v_off : 0) + c * 8);
          const uint2 held = *at;
          const uint32_t c8[2] = {held.x, held.y};
          float y[8];
          codes_to_floats<KIND>(c8, y);
          *at = floats_to_codes<KIND>(y, shrink, 0.f);
        }
      }
    }
  }
}

template <typename T, int HD, int KIND, int TILE, int ORDER>
int launch_write(WriteArgs& a, cudaStream_t st) {
  a.tiles = a.sl == 1 ? 1 : (a.sl - 1) / TILE + 2;
  a.kv_ctas = static_cast<unsigned>(a.bs) * a.tiles * a.kv_heads;
  // as many heads a lane as leave work for eight CTAs per SM: a position's angles are computed once for each group
  constexpr int RPP = WR_THREADS / (HD / 8);
  const int64_t tokens = static_cast<int64_t>(a.bs) * a.sl, want = static_cast<int64_t>(sm_count()) * 8 * RPP;
  a.q_heads = 4;
  while (a.q_heads < a.heads && tokens * ((a.heads - 1) / (2 * a.q_heads) + 1) >= want) a.q_heads *= 2;
  const int64_t q_ctas = (tokens * ((a.heads - 1) / a.q_heads + 1) + RPP - 1) / RPP;
  B200_CHECK_CUDA(launch_dependent(norm_rope_write_kernel<T, HD, KIND, TILE, ORDER>,
                                   dim3(static_cast<unsigned>(a.kv_ctas + q_ctas)), dim3(WR_THREADS), 0, st, a));
  return B200MOE_OK;
}
template <typename T, int HD, int KIND>
int launch_write_tile(WriteArgs& a, cudaStream_t st) {
  if constexpr (KIND != CACHE_PLAIN)
    if (a.scale_block > 32) return a.order ? launch_write<T, HD, KIND, 64, 1>(a, st) : launch_write<T, HD, KIND, 64, 0>(a, st);
  return a.order ? launch_write<T, HD, KIND, 32, 1>(a, st) : launch_write<T, HD, KIND, 32, 0>(a, st);
}
template <typename T, int KIND>
int launch_write_hd(WriteArgs& a, int hd, cudaStream_t st) {
  return hd == 64 ? launch_write_tile<T, 64, KIND>(a, st) : launch_write_tile<T, 128, KIND>(a, st);
}
template <int KIND>
int launch_write_io(WriteArgs& a, int io_dtype, int hd, cudaStream_t st) {
  if (io_dtype == B200MOE_DT_F32) return launch_write_hd<float, KIND>(a, hd, st);
  if (io_dtype == B200MOE_DT_F16) return launch_write_hd<__half, KIND>(a, hd, st);
  return launch_write_hd<__nv_bfloat16, KIND>(a, hd, st);
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

int check_kv8(const char* who, const b200moe_kv8_cache_t* c, int32_t block_index) {
  B200_REQUIRE(c != nullptr, "%s: NULL cache geometry", who);
  B200_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim %d (64 and 128 are built)", who, c->head_dim);
  B200_REQUIRE(c->blocks >= 1 && c->stride >= 1 && c->kv_heads >= 1 && c->kv_heads <= 65535 && c->page_count >= 1 &&
                   block_index >= 0 && block_index < c->blocks,
               "%s: bad cache geometry", who);
  B200_REQUIRE(c->scale_block >= 1 && c->scale_block <= MAX_SCALE_BLOCK && (c->scale_block & (c->scale_block - 1)) == 0 &&
                   c->stride % c->scale_block == 0,
               "%s: scale_block %d must be a power of two up to %d that divides the stride (%d)", who, c->scale_block,
               MAX_SCALE_BLOCK, c->stride);
  B200_REQUIRE(static_cast<double>(c->page_count) * c->blocks * c->kv_heads * 2.0 * c->stride < 4294967295.0,
               "%s: the cache has more than 2^32 rows", who);
  B200_REQUIRE(c->code == B200MOE_KV8_INT8 || c->code == B200MOE_KV8_E4M3, "%s: unknown code %d", who, c->code);
  return B200MOE_OK;
}

// -------------------------------------------------------------------- read-back
struct ReadArgs {
  const uint8_t* slab;
  const float* scales;
  const int32_t *page_ids, *seq_lens;
  void *k_out, *v_out;
  int pages_per_seq, page_count, max_len, kv_heads, stride, blocks, block_index, stride_shift, block_shift;
  int32_t* status;
};

// One CTA per (sequence, kv head, 16 positions); a thread takes the codes of 16 bytes of
// output (eight, or four for fp32: whole sectors are loaded and stored), K and V of several
// rows at once.  Bound by HBM: 32 sequences of up to 4000 positions, 8 heads of 128, to bf16
// (723 MB) take 114 us, 6.3 TB/s; with rows in tiles of 64 and 128 positions 137 and 170, with
// the tile, head and sequence by division 119, with 16 codes per thread and 4-byte stores 310.
constexpr int RD_THREADS = 128, RD_TILE = 16;
template <typename T, int HD, int CODE>
__global__ void __launch_bounds__(RD_THREADS) kv8_read_kernel(const ReadArgs a) {
  constexpr int E = 16 / static_cast<int>(sizeof(T)), W = E / 4;
  constexpr int LPR = HD / E, RPP = RD_THREADS / LPR, PASSES = RD_TILE / RPP;
  grid_dep_wait();
  grid_dep_launch();
  const int tile = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int sub = threadIdx.x / LPR, c = threadIdx.x % LPR;
  const int len = a.seq_lens[b];
  const size_t v_off = static_cast<size_t>(a.stride) * HD;
  uint32_t kc[PASSES][W], vc[PASSES][W];
  float2 sc[PASSES];
  auto fetch = [](uint32_t (&to)[W], const uint8_t* from) {
    if constexpr (W == 2) {
      const uint2 w = *reinterpret_cast<const uint2*>(from);
      to[0] = w.x; to[W - 1] = w.y;
    } else {
      to[0] = *reinterpret_cast<const uint32_t*>(from);
    }
  };
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int pos = tile * RD_TILE + i * RPP + sub;
#pragma unroll
    for (int j = 0; j < W; ++j) kc[i][j] = vc[i][j] = 0u;
    sc[i] = make_float2(0.f, 0.f);
    if (pos < len && pos < a.max_len) {
      const int slot = a.stride_shift >= 0 ? pos >> a.stride_shift : pos / a.stride, off = pos - slot * a.stride;
      const int page = slot < a.pages_per_seq ? a.page_ids[static_cast<size_t>(b) * a.pages_per_seq + slot] : -1;
      if (page < 0 || page >= a.page_count) {
        atomicOr(a.status, DEV_ERR_BOUNDS);
      } else {
        const size_t head = (static_cast<size_t>(page) * a.blocks + a.block_index) * a.kv_heads + h;
        const uint8_t* at = a.slab + (head * 2 * a.stride + off) * HD + c * E;
        fetch(kc[i], at);
        fetch(vc[i], at + v_off);
        sc[i] = reinterpret_cast<const float2*>(a.scales)[head * (a.stride >> a.block_shift) + (off >> a.block_shift)];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int pos = tile * RD_TILE + i * RPP + sub;
    if (pos >= a.max_len) return;
    const size_t to = ((static_cast<size_t>(b) * a.max_len + pos) * a.kv_heads + h) * HD + c * E;
    const bool live = pos < len;  // a NaN scale shows in live rows only
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float y[E];
      codes_to_floats<CODE>(kv ? vc[i] : kc[i], y);
      const float s = kv ? sc[i].y : sc[i].x;
#pragma unroll
      for (int j = 0; j < E; ++j) y[j] = live ? y[j] * s : 0.f;
      T* p = static_cast<T*>(kv ? a.v_out : a.k_out) + to;
      if constexpr (E == 8) store8(p, y);
      else *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
    }
  }
}

template <typename T, int HD>
int launch_read(const ReadArgs& a, int code, dim3 grid, cudaStream_t st) {
  B200_CHECK_CUDA(launch_dependent(code == B200MOE_KV8_INT8 ? kv8_read_kernel<T, HD, B200MOE_KV8_INT8>
                                                           : kv8_read_kernel<T, HD, B200MOE_KV8_E4M3>,
                                   grid, dim3(RD_THREADS), 0, st, a));
  return B200MOE_OK;
}

// -------------------------------------------------------------------- attention
// o = sum_p softmax(S)_p c_v(p) s_v(p),  S = scale * s_k(p) * (q . c_k(p)).
//
// Both products run on tensor cores with the codes widened to fp16 in registers (int8 and
// e4m3 are exact there), positions and head elements as the rows of A, the query rows that
// share a kv head as the eight columns of B (mma.m16n8k16):
//   S^T[pos][row] = K[pos][:] . q[row][:]      O^T[d][row] = sum_pos V^T[d][pos] P^T[pos][row]
// so that eight rows cost one MMA per 16 positions and 16 elements, and nothing is padded
// beyond eight rows (G = heads / kv_heads rows for one new token, G * new_tokens for
// several; NT = 2 takes sixteen).
//   * K is the A operand as it lies: ldmatrix of 16-byte chunks gives a lane four
//     consecutive bytes of a row, and the order of the 16 elements of an MMA is free as
//     long as q's fragments have the same one (a lane holds q[16c + 4 tig .. + 3], the
//     elements 0, 2 and 1, 3 as pairs).
//   * V^T comes from ldmatrix.trans on pairs of bytes: a lane gets two elements of two
//     positions, and taking bytes 0, 2 and 1, 3 apart makes rows 2 gid and 2 gid + 1 of V^T.
//   * P^T is S^T's accumulator, packed and transposed within the warp (movmatrix).
// The scale of V joins the softmax: with t = S log2(e) + log2(s_v), P = 2^(t - max t) is at
// most 1 whatever the scales are, the sum of P c_v is the numerator and that of P / s_v
// the denominator.  q is fp16 with its largest value in [2^14, 2^15), P with 2^7 where the
// maximum is up to date (it is left behind by up to 2^8, so that the output is rescaled
// rarely): what rounding loses is 2^-11 of a value down to 2^-28 and 2^-21 of the largest,
// and 2^-32 of the largest P below.  A bf16 output's own rounding is eight times that; an fp16
// output would be off by a third more than its rounding, and P is the sum of two fp16 parts
// for it, 2^-22, at one and a half times the MMAs (32 x 4000 positions int8 41 us instead of
// 40, e4m3 46 instead of 42.5, four new tokens 53 instead of 48).  SPLIT (32-bit activations): q too.
//
// A warp owns units of 32 positions with its own softmax state and places for one unit's K
// and V, filled by 16-byte cp.async, each again as soon as it is read: no barrier between
// warps.  (Places for two units and fewer CTAs: the same time, 53 against 52 us when it was
// tried.)  Chunks are swizzled so that ldmatrix has no bank conflicts.  A step of the CTA is
// 128 positions.  The steps of all (sequence, kv head, row tile) segments form one list, cut
// into equal stretches, one for each resident CTA: ragged lengths leave no SM idle, and the
// cut does not depend on how wide the page table is.  A segment that lies within one stretch
// is finished there; of the others every CTA leaves a state (at most two: its first and its
// last segment), which the merge kernel joins.
// 32 sequences of 2000 to 4000 positions, 8 kv heads of 128, 32 heads (200 MB): int8 40 us,
// e4m3 42, 5.0 and 4.7 TB/s (a plain read of as much, by a reduction, 39 us); bound by HBM
// once under way, before by the chain of lengths, page ids and first rows (6 us), after by the
// merge (4 us).  With a CTA per position split of each sequence 68.  Several new tokens are
// bound by the instructions around the MMAs: 16 rows 48 us, 32 rows, in two tiles that each
// widen the codes, 88 us of the same cache (in one tile, q in shared memory, 86: not kept).
struct AttendArgs {
  const void* q;
  int64_t q_stride;
  int q_dtype;
  const uint8_t* slab;
  const float* scales;
  const int32_t *page_ids, *seq_lens;
  void* out;
  float* partial;  // [CTA][2: its first, its last segment][rows of a tile][HD + 4]: numerator, max, denominator
  int out_dtype, bs, sl, pages_per_seq, page_count, heads, kv_heads, stride, blocks, block_index;
  int stride_shift, block_shift;  // log2; -1 where the stride is no power of two
  int row_tiles, ctas;
  float scale, softcap;
  int32_t* status;
};

// In how many fp16 parts the operands are: one; P in two (fp16 outputs); q and P in two (32-bit
// activations, and softcaps above CAP_FAST: there what the fast form of the softcap is off by,
// CAP_FAST * 2^-22 = 2^-14 of a probability, would begin to show).
constexpr float CAP_FAST = 256.f;
enum { BITS_ONE = 0, BITS_P = 1, BITS_BOTH = 2 };
constexpr int AT_THREADS = 128, AT_WARPS = 4;
constexpr int AT_UNIT = 32;   // positions of a warp's step
constexpr int AT_STEP = AT_WARPS * AT_UNIT;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// mma_16816 that the compiler may move between the loads of other tiles
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Byte offset of 16-byte chunk c of row r in a tile of rows of HD bytes: the eight chunks
// that one ldmatrix phase reads (eight rows, one c) lie in eight different bank groups.
template <int HD>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  if constexpr (HD == 128) return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4));
  else return static_cast<uint32_t>((r >> 1) * 128 + ((((r & 1) * 4 + c) ^ ((r >> 1) & 3)) << 4));
}

// The sums of several states (max, denominator, numerator) of one row: weights 2^(m - M).
// Their roots are what is computed: where scales of V are far apart, 2^(m - M) can be below
// 2^-126 while the denominator of a state of small scales is as large, and is multiplied by
// one root after the other.
__device__ __forceinline__ float state_root(float m, float top) { return m == -INFINITY ? 0.f : ex2(0.5f * (m - top)); }

// Positions that a sequence's length names, and steps of its segments.
__device__ __forceinline__ int clamp_length(const AttendArgs& a, int len) {
  const int room = a.pages_per_seq * a.stride;
  return len < 0 ? 0 : len < room ? len : room;
}
__device__ __forceinline__ int live_positions(const AttendArgs& a, int b) { return clamp_length(a, a.seq_lens[b]); }
__device__ __forceinline__ int steps_of(int len) { return len > AT_STEP ? (len + AT_STEP - 1) / AT_STEP : 1; }

// Joining a segment in the middle of a stretch (the barrier and the output of the last one,
// q) takes a CTA as long as a step or two: in long stretches a segment counts START_STEPS
// more than it has, so that the CTAs that join one get fewer.  (0, 2, 3 at 32 x 4000
// positions: 16 rows 51, 48, 49 us; 8 rows 40, 41, 42.)
constexpr int START_STEPS = 2;
__device__ __forceinline__ int start_steps(int steps, int ctas) { return steps >= 4 * ctas ? START_STEPS : 0; }

// The list of steps, looked at by a whole warp: those of the sequences before `until` or,
// with until < 0, before the sequence that holds step `want`; each segment with `start` more.
struct ListSum { int before, seq; };
__device__ __forceinline__ ListSum walk_list(const AttendArgs& a, int lane, int until, int want, int start) {
  const int per_step = a.kv_heads * a.row_tiles, stop = until < 0 ? a.bs : until;
  int before = 0;
  for (int b0 = 0; b0 < stop; b0 += 32) {
    const int b = b0 + lane;
    const int own = b < stop ? (start + steps_of(live_positions(a, b))) * per_step : 0;
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (until < 0) {
      const unsigned past = __ballot_sync(0xffffffffu, before + sum > want && own > 0);
      if (past != 0) {
        const int at = __ffs(past) - 1;
        return {before + __shfl_sync(0xffffffffu, sum - own, at), b0 + at};
      }
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return {before, stop};
}
// First step of CTA i's stretch, and the CTA that holds step g: the first total % ctas
// stretches are one step longer than the others.
struct Stretches {
  int each, longer;
  __device__ Stretches(int total, int ctas) : each(total / ctas), longer(total - each * ctas) {}
  __device__ int begin(int i) const { return i * each + min(i, longer); }
  __device__ int cta_of(int g) const {
    const int cut = longer * (each + 1);
    return g < cut ? g / (each + 1) : longer + (g - cut) / each;
  }
};

// CTAs per SM, at 32 x 4000 positions against one less and one more.  HD 128: one row tile of
// bf16, int8 39 us (41, 46), e4m3 42 (45, 47); two of bf16 48 (83, 55); one of fp32 46.5 (70,
// 45.6) and 50.7 (69, 51.0).  HD 64, int8: bf16 17.3 (17.3, 17.7) and 21.8 with four tokens
// (22.3, 25.4); fp32 20.5 (19.6, 21.7) and 26.8 (25.8, 32.4).  Some of the variants with P or
// q in two parts keep 8 to 84 bytes of a thread's registers in memory.
template <int HD, int NT, int BITS>
constexpr int attend_resident() {
  if (HD == 128) return NT == 1 && BITS != BITS_BOTH ? 3 : 2;
  return NT == 1 ? 4 : 3;
}

template <int HD, int CODE, int NT, int BITS>
__global__ void __launch_bounds__(AT_THREADS, (attend_resident<HD, NT, BITS>())) kv8_attend_kernel(const AttendArgs a) {
  constexpr int CH = HD / 16;                       // chunks of a row: MMA steps of q.k, row tiles of V^T
  constexpr bool SPLIT = BITS == BITS_BOTH;
  constexpr int PARTS = SPLIT ? 2 : 1, P_PARTS = BITS == BITS_ONE ? 1 : 2;
  constexpr int ROWS = 8 * NT;
  constexpr int TILE = AT_UNIT * HD;                // bytes of a unit's K (or V)
  constexpr int OPITCH = HD + 8;                    // floats
  constexpr float P_TOP = 7.f, P_SLACK = 8.f;       // P is at most 2^7 when the maximum is taken, 2^15 before it is again
  extern __shared__ __align__(128) uint8_t smem[];  // [warp][K | V], then [warp][row][OPITCH] fp32
  float* s_o = reinterpret_cast<float*>(smem + AT_WARPS * 2 * TILE);
  __shared__ float4 s_pos[AT_WARPS][AT_UNIT];       // of each position: s_k, log2 s_v, 1 / s_v
  __shared__ float2 s_ml[AT_WARPS][ROWS];
  grid_dep_wait();
  grid_dep_launch();
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, gid = lane >> 2, tig = lane & 3;
  const int G = a.heads / a.kv_heads, rows = G * a.sl;
  const int real = walk_list(a, lane, a.bs, 0, 0).before, start = start_steps(real, a.ctas);
  const int total = real + start * a.bs * a.kv_heads * a.row_tiles, ctas = min(a.ctas, total);
  if (blockIdx.x >= ctas) return;
  const Stretches cut(total, ctas);
  const int g_begin = cut.begin(blockIdx.x), g_end = cut.begin(blockIdx.x + 1);
  const ListSum at = walk_list(a, lane, -1, g_begin, start);

  // Scores in halvings; with a softcap c, c tanh(x / c) = c - 2 c / (2^(2 log2(e) x / c) + 1):
  // two special functions, good to c 2^-22.  32-bit activations and caps above CAP_FAST take
  // tanhf, 2^-22 of the value.
  const float cap2 = a.softcap * LOG2E;
  const float to_score = a.softcap > 0.f ? a.scale / a.softcap * (SPLIT ? 1.f : 2.f * LOG2E) : a.scale * LOG2E;
  const uint32_t ring = smem_u32(smem) + warp * (2 * TILE);
  const size_t v_off = static_cast<size_t>(a.stride) * HD;
  // byte offsets in a tile that this lane addresses with ldmatrix: rows 16 h + (lane & 15), chunks 2 i + (lane >> 4)
  uint32_t ld_at[CH / 2];
#pragma unroll
  for (int i = 0; i < CH / 2; ++i) ld_at[i] = tile_at<HD>(lane & 15, 2 * i + (lane >> 4));

  // what of a segment lies in this stretch, and the warp's units of it
  struct Piece { int b, kvh, tile, len, x0, x1, steps, end, p_begin, p_end, units; };
  int seq_first = at.before, seq = at.seq;  // the current sequence and the first of its steps
  auto piece_at = [&](int g) {
    Piece p;
    p.len = live_positions(a, seq);
    p.steps = steps_of(p.len);
    while (g - seq_first >= (start + p.steps) * a.kv_heads * a.row_tiles) {  // at most once: g is a step of this or the next
      seq_first += (start + p.steps) * a.kv_heads * a.row_tiles;
      p.len = live_positions(a, ++seq);
      p.steps = steps_of(p.len);
    }
    const int seg = (g - seq_first) / (start + p.steps), x = g - seq_first - seg * (start + p.steps);
    p.b = seq;
    p.kvh = seg / a.row_tiles;
    p.tile = seg - p.kvh * a.row_tiles;
    p.end = min(g + start + p.steps - x, g_end);
    p.x0 = max(0, x - start);
    p.x1 = max(0, x + p.end - g - start);  // 0: no step of it
    p.p_begin = p.x0 * AT_STEP + warp * AT_UNIT;
    p.p_end = min(p.len, p.x1 * AT_STEP);
    p.units = p.p_end > p.p_begin ? (p.p_end - p.p_begin + AT_STEP - 1) / AT_STEP : 0;
    return p;
  };
  // the page of this lane's position of unit u, looked at one unit later; -1 behind the stretch
  auto page_of = [&](const Piece& p, int u) -> int {
    const int pos = p.p_begin + u * AT_STEP + lane;
    if (pos >= p.p_end) return -1;
    const int slot = a.stride_shift >= 0 ? pos >> a.stride_shift : pos / a.stride;
    return a.page_ids[static_cast<size_t>(p.b) * a.pages_per_seq + slot];
  };
  // of unit u: this lane's K row in the slab, in rows of HD bytes (~0: none), and its scales
  auto locate = [&](const Piece& p, int u, int page, float2& sc) -> uint32_t {
    sc = make_float2(0.f, -1.f);
    const int pos = p.p_begin + u * AT_STEP + lane;
    if (pos >= p.p_end) return 0xffffffffu;
    if (page < 0 || page >= a.page_count) {
      atomicOr(a.status, DEV_ERR_BOUNDS);
      return 0xffffffffu;
    }
    const int off = a.stride_shift >= 0 ? pos & (a.stride - 1) : pos % a.stride;
    const uint32_t head = (static_cast<uint32_t>(page) * a.blocks + a.block_index) * a.kv_heads + p.kvh;
    sc = reinterpret_cast<const float2*>(a.scales)[static_cast<size_t>(head) * (a.stride >> a.block_shift) +
                                                   (off >> a.block_shift)];
    return head * 2u * a.stride + off;
  };
  // starts the copies of a unit's K or V rows (zeros in the place of missing ones); one group per call, also without a unit
  auto issue = [&](bool unit, uint32_t row, int kv) {
    if (unit) {
      const uint32_t row0 = __shfl_sync(0xffffffffu, row, 0);
      const uint32_t to = ring + kv * TILE;
      constexpr int RPI = 32 / CH;  // rows of one pass of the warp
      const int r0 = lane / CH, c = lane % CH;
      const uint8_t* from = a.slab + (kv ? v_off : 0) + c * 16;
      if (__all_sync(0xffffffffu, row == row0 + lane && row != 0xffffffffu)) {  // within one page
        from += static_cast<size_t>(row0 + r0) * HD;
#pragma unroll
        for (int i = 0; i < AT_UNIT / RPI; ++i) copy16(to + tile_at<HD>(i * RPI + r0, c), from + i * RPI * HD, true);
      } else {
#pragma unroll
        for (int i = 0; i < AT_UNIT / RPI; ++i) {
          const int r = i * RPI + r0;
          const uint32_t at_row = __shfl_sync(0xffffffffu, row, r);
          const bool ok = at_row != 0xffffffffu;
          copy16(to + tile_at<HD>(r, c), from + static_cast<size_t>(ok ? at_row : 0u) * HD, ok);
        }
      }
    }
    copy_commit();
  };

  // q as it lies in memory: a lane's four elements of each chunk of its column's row
  uint32_t q_raw[NT][CH][SPLIT ? 4 : 2];
  auto load_q = [&](const Piece& p) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = p.tile * ROWS + 8 * n + gid;
      const int64_t from = (static_cast<int64_t>(p.b) * a.sl + r / G) * a.q_stride +
                           static_cast<int64_t>(p.kvh * G + r % G) * HD + 4 * tig;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int i = 0; i < (SPLIT ? 4 : 2); ++i) q_raw[n][c][i] = 0u;
        if (r < rows) {
          if (SPLIT && a.q_dtype == B200MOE_DT_F32) {
            const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const float*>(a.q) + from + 16 * c);
            q_raw[n][c][0] = w.x; q_raw[n][c][1] = w.y;
            if constexpr (SPLIT) { q_raw[n][c][2] = w.z; q_raw[n][c][3] = w.w; }
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const __half*>(a.q) + from + 16 * c);
            q_raw[n][c][0] = w.x; q_raw[n][c][1] = w.y;
          }
        }
      }
    }
  };
  auto q_values = [&](const uint32_t (&w)[SPLIT ? 4 : 2], float (&x)[4]) {
    if (SPLIT && a.q_dtype == B200MOE_DT_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(w[SPLIT ? e : 0]);
    } else if (a.q_dtype == B200MOE_DT_F16) {
      const float2 lo = __half22float2(u32_as_h2(w[0])), hi = __half22float2(u32_as_h2(w[1]));
      x[0] = lo.x; x[1] = lo.y; x[2] = hi.x; x[3] = hi.y;
    } else {
      x[0] = __uint_as_float(w[0] << 16); x[1] = __uint_as_float(w[0] & 0xffff0000u);
      x[2] = __uint_as_float(w[1] << 16); x[3] = __uint_as_float(w[1] & 0xffff0000u);
    }
  };

  // The copies of a unit are started as soon as the places of the one before are read, those
  // of the next segment's first unit during this segment's last.
  Piece next = piece_at(g_begin);
  float2 sc_now, sc_next;
  // before the first copies: behind all CTAs' of them it takes 4 us more (with two tiles of q or
  // more the registers would have to wait in memory)
  constexpr bool Q_FIRST = NT == 1;
  if constexpr (Q_FIRST) load_q(next);
  {
    const uint32_t row = locate(next, 0, page_of(next, 0), sc_next);
    issue(next.units > 0, row, 0);
    issue(next.units > 0, row, 1);
  }
  for (int g = g_begin; g < g_end;) {
    const Piece cur = next;
    if (cur.x1 == 0) break;  // the stretch ends before the segment's first step
    const int b = cur.b, kvh = cur.kvh, tile = cur.tile, units = cur.units;
    if (cur.x0 == 0 && t == 0 && a.seq_lens[b] > a.pages_per_seq * a.stride) atomicOr(a.status, DEV_ERR_BOUNDS);
    int page_next = page_of(cur, 1), page_after = -1;
    if (cur.end < g_end) {
      next = piece_at(cur.end);
      page_after = page_of(next, 0);
    } else {
      next.p_end = next.units = 0;
    }

    // q: column gid of B is row tile * ROWS + 8 n + gid; its values times a power of two
    if (!Q_FIRST || g != g_begin) load_q(cur);
    uint32_t qb[PARTS][NT][CH][2];
    float fold[NT][2];  // of this lane's accumulator columns 2 tig, 2 tig + 1: back to to_score units
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[CH][4], top = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        q_values(q_raw[n][c], x[c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[c][e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e <= top < 2^(e + 1), so that the largest value lies in [2^14, 2^15)
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      e = e < -100 || e > 127 ? -100 : e;
      if (__float_as_uint(top) == 0x7f800000u) e = 100;
      const float up = __uint_as_float(static_cast<uint32_t>(14 - e + 127) << 23);
      const float down = __uint_as_float(static_cast<uint32_t>(e - 14 + 127) << 23) * to_score;
      fold[n][0] = __shfl_sync(0xffffffffu, down, (2 * tig) * 4);
      fold[n][1] = __shfl_sync(0xffffffffu, down, (2 * tig + 1) * 4);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float u = x[c][i] * up, v = x[c][i + 2] * up;  // the codes' bytes (0, 2), (1, 3)
          const __half2 h = __floats2half2_rn(u, v);
          qb[0][n][c][i] = h2_as_u32(h);
          if constexpr (SPLIT) {
            const float2 f = __half22float2(h);
            qb[PARTS - 1][n][c][i] = h2_as_u32(__floats2half2_rn(u - f.x, v - f.y));
          }
        }
    }
    // the first position that a column does not see
    const int all_see = a.seq_lens[b] - a.sl + 1;
    auto seen = [&](int n, int j) { return all_see + (tile * ROWS + 8 * n + 2 * tig + j) / G; };

    float top_v = 0.f;  // largest scale of V that this lane has met
    float m[NT][2], l[NT][2], o[NT][CH][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) o[n][c][0] = o[n][c][1] = o[n][c][2] = o[n][c][3] = 0.f;
    }

    for (int u = 0; u < units; ++u) {
      sc_now = sc_next;
      {
        // dead positions (sc.y < 0: scales are never negative): weight 0 without touching the others
        const bool dead = sc_now.y < 0.f, bad = sc_now.y != sc_now.y;
        // A scale of 0 (codes all zero) may be any number: 2^-40 of the largest one that all columns
        // have seen so far, so that such positions keep their weight in 2^t / s_v and do not become
        // the maximum that the others' P are taken from.  At least 2^-100, as every other scale.
        if (cur.p_begin + u * AT_STEP + lane < all_see) top_v = fmaxf(top_v, sc_now.y);
        float vs = fmaxf(sc_now.y, 7.888609052210118e-31f);
        if (__any_sync(0xffffffffu, sc_now.y == 0.f)) {
          const int top = __reduce_max_sync(0xffffffffu, __float_as_int(top_v));
          if (sc_now.y == 0.f) vs = fmaxf(vs, __int_as_float(top) * 9.0949470177292824e-13f);
        }
        s_pos[warp][lane] = make_float4(sc_now.x * (CODE == B200MOE_KV8_E4M3 ? E4M3_UNIT : 1.f),
                                        dead ? -INFINITY : bad ? sc_now.y : __log2f(vs), dead ? 0.f : rcp(vs), 0.f);
      }
      copy_wait<1>();  // all but V of this unit
      __syncwarp();
      const uint32_t kt = ring, vt = kt + TILE;
      const int p0 = cur.p_begin + u * AT_STEP;

      // two accumulators for each 16 positions where there are no others to alternate with
      constexpr int ACC = NT == 1 ? 2 : 1;
      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float acc[ACC][NT][4];
#pragma unroll
        for (int k = 0; k < ACC; ++k)
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[k][n][0] = acc[k][n][1] = acc[k][n][2] = acc[k][n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
          uint32_t w[4];
          ldsm_x4(kt + ld_at[c / 2] + 16 * h * HD, w);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a0, a1, a2, a3;
            widen4<CODE>(w[2 * i], a0, a2);
            widen4<CODE>(w[2 * i + 1], a1, a3);
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma(acc[i % ACC][n], a0, a1, a2, a3, qb[p][n][c + i][0], qb[p][n][c + i][1]);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[h][n][k] = ACC == 2 ? acc[0][n][k] + acc[ACC - 1][n][k] : acc[0][n][k];
      }
      __syncwarp();  // K is read: its place takes that of the next unit
      const bool last = u + 1 == units;
      const uint32_t row_next = locate(last ? next : cur, last ? 0 : u + 1, last ? page_after : page_next, sc_next);
      page_next = page_of(cur, u + 2);
      const bool unit_next = !last || next.units > 0;
      issue(unit_next, row_next, 0);

      // scores of positions 16 h + 8 j + gid, columns 2 tig + e
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
      float ivs[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 f = s_pos[warp][16 * h + 8 * j + gid];
          ivs[h][j] = f.z;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float y = f.x * fold[n][e];
              float x;
              if (a.softcap > 0.f) {
                if constexpr (SPLIT) x = fmaf(cap2, tanhf(s[h][n][2 * j + e] * y), f.y);
                else x = fmaf(-2.f * cap2, rcp(ex2(s[h][n][2 * j + e] * y) + 1.f), cap2 + f.y);
              } else {
                x = fmaf(s[h][n][2 * j + e], y, f.y);
              }
              s[h][n][2 * j + e] = x;
            }
        }
      if (p0 + AT_UNIT > all_see) {  // the last positions: not all of them are seen by all columns
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (p0 + 16 * h + 8 * (k >> 1) + gid >= seen(n, k & 1)) s[h][n][k] = -INFINITY;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) top[n][k & 1] = fmaxf(top[n][k & 1], s[h][n][k]);
      // a column's maximum moves only when P could leave fp16's range
      bool moves = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v = top[n][e];
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          top[n][e] = v;
          moves |= v > m[n][e] + P_SLACK;
        }
      if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float m_new = fmaxf(m[n][e], top[n][e]);
            const float root = m_new == -INFINITY ? 1.f : state_root(m[n][e], m_new), alpha = root * root;
            m[n][e] = m_new;
            l[n][e] = l[n][e] * root * root;
#pragma unroll
            for (int c = 0; c < CH; ++c) { o[n][c][e] *= alpha; o[n][c][2 + e] *= alpha; }
          }
      }
      uint32_t pb[P_PARTS][NT][2][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float base0 = P_TOP - (m[n][0] == -INFINITY ? 0.f : m[n][0]);
        const float base1 = P_TOP - (m[n][1] == -INFINITY ? 0.f : m[n][1]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float u0 = ex2(s[h][n][2 * j] + base0), u1 = ex2(s[h][n][2 * j + 1] + base1);
            l[n][0] = fmaf(u0, ivs[h][j], l[n][0]);
            l[n][1] = fmaf(u1, ivs[h][j], l[n][1]);
            const __half2 hp = __floats2half2_rn(u0, u1);
            pb[0][n][h][j] = transpose8x8(h2_as_u32(hp));
            if constexpr (P_PARTS == 2) {
              const float2 f = __half22float2(hp);
              pb[P_PARTS - 1][n][h][j] = transpose8x8(h2_as_u32(__floats2half2_rn(u0 - f.x, u1 - f.y)));
            }
          }
      }
      copy_wait<1>();
      __syncwarp();
      if constexpr (SPLIT) {
        // the tensor cores cut off what a sum's last bit cannot hold: a unit's products are summed
        // apart and added with rounding, or a long stretch would lose 2^-25 at every step
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
          uint32_t w[2][4];
          ldsm_x4_trans(vt + ld_at[c / 2], w[0]);
          ldsm_x4_trans(vt + ld_at[c / 2] + 16 * HD, w[1]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float unit_o[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) unit_o[n][0] = unit_o[n][1] = unit_o[n][2] = unit_o[n][3] = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t a0, a1, a2, a3;
              widen4<CODE>(w[h][2 * i], a0, a1);
              widen4<CODE>(w[h][2 * i + 1], a2, a3);
#pragma unroll
              for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int n = 0; n < NT; ++n) mma(unit_o[n], a0, a1, a2, a3, pb[p][n][h][0], pb[p][n][h][1]);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int k = 0; k < 4; ++k) o[n][c + i][k] += unit_o[n][k];
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < CH; c += 2) {
            uint32_t w[4];
            ldsm_x4_trans(vt + ld_at[c / 2] + 16 * h * HD, w);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t a0, a1, a2, a3;
              widen4<CODE>(w[2 * i], a0, a1);
              widen4<CODE>(w[2 * i + 1], a2, a3);
#pragma unroll
              for (int p = 0; p < P_PARTS; ++p)
#pragma unroll
                for (int n = 0; n < NT; ++n) mma(o[n][c + i], a0, a1, a2, a3, pb[p][n][h][0], pb[p][n][h][1]);
            }
          }
      }
      __syncwarp();  // V and s_pos are read
      issue(unit_next, row_next, 1);
    }
    if (units == 0) {  // nothing of this segment for the warp: the next one's copies are started here
      const uint32_t row = locate(next, 0, page_after, sc_next);
      issue(next.units > 0, row, 0);
      issue(next.units > 0, row, 1);
    }
    // the four warps' states through shared memory
    __syncthreads();  // the last segment's are read
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * n + 2 * tig + e;
        float v = l[n][e];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        // the unit of the e4m3 codes: here and not in s_v, whose reciprocal it would push out of 32 bits
        if (gid == 0) s_ml[warp][r] = make_float2(m[n][e], CODE == B200MOE_KV8_E4M3 ? v * (1.f / E4M3_UNIT) : v);
#pragma unroll
        for (int c = 0; c < CH; ++c)
          *reinterpret_cast<float2*>(&s_o[(warp * ROWS + r) * OPITCH + 16 * c + 2 * gid]) =
              make_float2(o[n][c][e], o[n][c][2 + e]);
      }
    __syncthreads();
    const bool whole = cur.x0 == 0 && cur.x1 == cur.steps;
    float* part = a.partial + static_cast<size_t>(blockIdx.x * 2 + (g == g_begin ? 0 : 1)) * ROWS * (HD + 4);
    for (int i = t; i < ROWS * (HD / 4); i += AT_THREADS) {
      const int r = i / (HD / 4), d = i % (HD / 4) * 4, row = tile * ROWS + r;
      if (row >= rows) break;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < AT_WARPS; ++w) top = fmaxf(top, s_ml[w][r].x);
      float acc[4] = {0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
      for (int w = 0; w < AT_WARPS; ++w) {
        const float2 ml = s_ml[w][r];
        const float root = state_root(ml.x, top), f = root * root;
        den = fmaf(ml.y * root, root, den);
        const float4 v = *reinterpret_cast<const float4*>(&s_o[(w * ROWS + r) * OPITCH + d]);
        acc[0] = fmaf(v.x, f, acc[0]); acc[1] = fmaf(v.y, f, acc[1]);
        acc[2] = fmaf(v.z, f, acc[2]); acc[3] = fmaf(v.w, f, acc[3]);
      }
      if (whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = den == 0.f ? 0.f : acc[j] / den;
        store_as(a.out, a.out_dtype,
                 ((static_cast<size_t>(b) * a.sl + row / G) * a.heads + kvh * G + row % G) * HD + d, acc);
      } else {
        *reinterpret_cast<float4*>(part + r * (HD + 4) + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) *reinterpret_cast<float2*>(part + r * (HD + 4) + HD) = make_float2(top, den);
      }
    }
    g = cur.end;
  }
}

// Joins the states of the segments that lie in several CTAs' stretches: WPR warps per row,
// eight per CTA.  A segment of the ordinary batch has two or three states, one of a single
// long sequence some seventy: there one warp's loads would queue up (22 us instead of 3).
constexpr int MG_WARPS = 8;
template <int HD, int WPR>
__global__ void __launch_bounds__(32 * MG_WARPS) kv8_attend_merge_kernel(const AttendArgs a, int tile_rows) {
  constexpr int N = HD / 32;
  __shared__ float s_o[MG_WARPS][HD];
  __shared__ float2 s_ml[MG_WARPS];
  const int G = a.heads / a.kv_heads, rows = G * a.sl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WPR;
  const int at = blockIdx.x * (MG_WARPS / WPR) + warp / WPR;
  const int row = at % rows, kvh = at / rows % a.kv_heads, b = at / rows / a.kv_heads;
  if (b >= a.bs) return;  // whole warps; with WPR > 1 the grid has no such rows
  // The list once: its length, that of the sequences before this one, and this one's steps.
  // Before the wait it is a guess, with which the states' loads can start as soon as the wait
  // is over; the lengths are read again beside them (past L1, which may have kept the first
  // look).  Lengths are clamped to the page table, so that any guess names states in scratch.
  const int per_step = a.kv_heads * a.row_tiles;
  struct List { int real, before, steps; };
  auto look = [&] {
    List l{0, 0, 0};
    for (int i = lane; i < a.bs; i += 32) {
      const int n = steps_of(clamp_length(a, __ldcg(a.seq_lens + i)));
      l.real += n * per_step;
      l.before += i < b ? n * per_step : 0;
      l.steps += i == b ? n : 0;
    }
    l.real = __reduce_add_sync(0xffffffffu, l.real);
    l.before = __reduce_add_sync(0xffffffffu, l.before);
    l.steps = __reduce_add_sync(0xffffffffu, l.steps);
    return l;
  };
  // where the row's states are: the first CTA may have begun before this segment, and its state
  // is then its second; the others begin inside it
  const size_t pitch = static_cast<size_t>(tile_rows) * (HD + 4);
  struct States { int n; const float *first, *others; };
  auto find = [&](const List& l) {
    const int start = start_steps(l.real, a.ctas), total = l.real + start * a.bs * per_step;
    const int g0 = l.before + start * b * per_step + (kvh * a.row_tiles + row / tile_rows) * (start + l.steps);
    const Stretches cut(total, min(a.ctas, total));
    const int first = cut.cta_of(g0 + start), last = cut.cta_of(g0 + start + l.steps - 1);
    const float* at = a.partial + 2 * static_cast<size_t>(first) * pitch + row % tile_rows * (HD + 4);
    return States{last - first + 1, at + (cut.begin(first) < g0 ? pitch : 0), at};
  };
  constexpr int AT_ONCE = WPR == 1 ? 4 : 8;
  float v[AT_ONCE][N];
  float2 ml[AT_ONCE];
  auto load = [&](const States& in, int s0) {
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int s = s0 + k * WPR;
      ml[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int j = 0; j < N; ++j) v[k][j] = 0.f;
      if (s < in.n) {
        const float* from = s == 0 ? in.first : in.others + 2 * s * pitch;
        ml[k] = *reinterpret_cast<const float2*>(from + HD);
        load_elems(from + lane * N, v[k]);
      }
    }
  };
  const List guess = look();
  States in = find(guess);
  grid_dep_wait();
  grid_dep_launch();
  if (in.n > 1) load(in, part);
  const List list = look();
  if (list.real != guess.real || list.before != guess.before || list.steps != guess.steps) {
    in = find(list);
    if (in.n > 1) load(in, part);
  }
  if (in.n == 1) return;  // finished by that CTA
  float acc[N], top = -INFINITY, den = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  for (int s0 = part; s0 < in.n; s0 += AT_ONCE * WPR) {
    if (s0 != part) load(in, s0);
    float up = top;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) up = fmaxf(up, ml[k].x);
    const float root0 = state_root(top, up), f0 = root0 * root0;
    den = den * root0 * root0;
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] *= f0;
    top = up;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const float root = state_root(ml[k].x, top), f = root * root;
      den = fmaf(ml[k].y * root, root, den);
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = fmaf(v[k][j], f, acc[j]);
    }
  }
  const size_t to = ((static_cast<size_t>(b) * a.sl + row / G) * a.heads + kvh * G + row % G) * HD;
  if constexpr (WPR == 1) {
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = den == 0.f ? 0.f : acc[j] / den;
    store_as(a.out, a.out_dtype, to + lane * N, acc);
  } else {
    static_assert(WPR == 1 || WPR == MG_WARPS, "one row per CTA: all of its warps are here or none");
#pragma unroll
    for (int j = 0; j < N; ++j) s_o[warp][lane * N + j] = acc[j];
    if (lane == 0) s_ml[warp] = make_float2(top, den);
    __syncthreads();
    const int d = threadIdx.x * 2;
    if (d >= HD) return;
    top = -INFINITY;
#pragma unroll
    for (int w = 0; w < MG_WARPS; ++w) top = fmaxf(top, s_ml[w].x);
    float o[2] = {0.f, 0.f};
    den = 0.f;
#pragma unroll
    for (int w = 0; w < MG_WARPS; ++w) {
      const float root = state_root(s_ml[w].x, top), f = root * root;
      den = fmaf(s_ml[w].y * root, root, den);
      o[0] = fmaf(s_o[w][d], f, o[0]);
      o[1] = fmaf(s_o[w][d + 1], f, o[1]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) o[j] = den == 0.f ? 0.f : o[j] / den;
    store_as(a.out, a.out_dtype, to + d, o);
  }
}

template <int HD>
int launch_merge(const AttendArgs& a, int tile_rows, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(a.bs) * a.heads * a.sl;
  // states of a segment, about (8 x 8190 positions, 30 rows, 4.6 states: a warp per row 56 us in all, eight 64)
  const bool many = a.ctas > 6 * a.bs * a.kv_heads * a.row_tiles;
  if (many)
    B200_CHECK_CUDA(launch_dependent(kv8_attend_merge_kernel<HD, MG_WARPS>, dim3(static_cast<unsigned>(rows)),
                                     dim3(32 * MG_WARPS), 0, st, a, tile_rows));
  else
    B200_CHECK_CUDA(launch_dependent(kv8_attend_merge_kernel<HD, 1>, dim3(static_cast<unsigned>((rows + MG_WARPS - 1) / MG_WARPS)),
                                     dim3(32 * MG_WARPS), 0, st, a, tile_rows));
  return B200MOE_OK;
}

// Rows of a CTA's tile; CTAs of a call: as many as are resident at once, or one for each
// step of a full page table where those are fewer.
inline int attend_tile_rows(int rows) { return rows <= 8 ? 8 : 16; }
template <int HD>
int resident_ctas(int tile, int bits) {
  if (bits == BITS_BOTH) return tile == 16 ? attend_resident<HD, 2, BITS_BOTH>() : attend_resident<HD, 1, BITS_BOTH>();
  if (bits == BITS_P) return tile == 16 ? attend_resident<HD, 2, BITS_P>() : attend_resident<HD, 1, BITS_P>();
  return tile == 16 ? attend_resident<HD, 2, BITS_ONE>() : attend_resident<HD, 1, BITS_ONE>();
}
int attend_ctas(const b200moe_kv8_cache_t& c, int bs, int rows, int bits, int max_seq_len) {
  const int tile = attend_tile_rows(rows);
  const int64_t steps = (static_cast<int64_t>(max_seq_len) + AT_STEP - 1) / AT_STEP * bs * c.kv_heads * ((rows + tile - 1) / tile);
  const int64_t resident = static_cast<int64_t>(sm_count()) * 
                           (c.head_dim == 128 ? resident_ctas<128>(tile, bits) : resident_ctas<64>(tile, bits));
  return static_cast<int>(steps < resident ? steps : resident);
}

template <int HD, int CODE, int NT, int BITS>
int launch_attend(const AttendArgs& a, cudaStream_t st) {
  constexpr int SMEM = AT_WARPS * 2 * AT_UNIT * HD + AT_WARPS * 8 * NT * (HD + 8) * 4;
  auto kern = kv8_attend_kernel<HD, CODE, NT, BITS>;
  static bool configured[16] = {};
  int dev = 0;
  B200_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev >= 16 || !configured[dev]) {
    B200_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev < 16) configured[dev] = true;
  }
  B200_CHECK_CUDA(launch_dependent(kern, dim3(a.ctas), dim3(AT_THREADS), SMEM, st, a));
  return B200MOE_OK;
}
template <int HD, int CODE>
int launch_attend_rows(const AttendArgs& a, int bits, int tile_rows, cudaStream_t st) {
  const bool one = tile_rows == 8;
  if (bits == BITS_BOTH) return one ? launch_attend<HD, CODE, 1, BITS_BOTH>(a, st) : launch_attend<HD, CODE, 2, BITS_BOTH>(a, st);
  if (bits == BITS_P) return one ? launch_attend<HD, CODE, 1, BITS_P>(a, st) : launch_attend<HD, CODE, 2, BITS_P>(a, st);
  return one ? launch_attend<HD, CODE, 1, BITS_ONE>(a, st) : launch_attend<HD, CODE, 2, BITS_ONE>(a, st);
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" {

int b200moe_attn_norm_rope_kv8_write(const void* q, const void* k, const void* v, int io_dtype, int64_t q_stride,
                                     int64_t k_stride, int64_t v_stride, const float* q_norm, const float* k_norm,
                                     float eps, void* q_out, void* k_out, void* slab, float* scales,
                                     const b200moe_kv8_cache_t* cache, int32_t block_index,
                                     const int32_t* start_positions, const int32_t* new_lens,
                                     const int32_t* page_ids, const float* freqs, int order, int32_t bs,
                                     int32_t tokens_per_seq, int32_t pages_per_seq, int32_t heads, void* stream) {
  const char* who = "attn_norm_rope_kv8_write";
  if (const int rc = check_kv8(who, cache, block_index)) return rc;
  WriteArgs a{};
  a.q = q; a.k = k; a.v = v; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps; a.q_out = q_out; a.k_out = k_out;
  a.slab = slab; a.scales = scales; a.start_positions = start_positions; a.new_lens = new_lens;
  a.page_ids = page_ids; a.freqs = freqs; a.order = order; a.bs = bs; a.sl = tokens_per_seq;
  a.pages_per_seq = pages_per_seq; a.page_count = cache->page_count; a.heads = heads; a.kv_heads = cache->kv_heads;
  a.stride = cache->stride; a.blocks = cache->blocks; a.block_index = block_index; a.scale_block = cache->scale_block;
  a.stride_shift = log2_of(a.stride);
  a.block_shift = log2_of(a.scale_block);
  if (const int rc = check_write(who, a, io_dtype, cache->head_dim)) return rc;
  if (bs == 0) return B200MOE_OK;
  B200_REQUIRE(scales != nullptr && (reinterpret_cast<uintptr_t>(scales) & 7) == 0,
               "%s: scales must be given and 8-byte aligned", who);
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->code == B200MOE_KV8_INT8 ? launch_write_io<CACHE_INT8>(a, io_dtype, cache->head_dim, st)
                                         : launch_write_io<CACHE_E4M3>(a, io_dtype, cache->head_dim, st);
}

int b200moe_attn_norm_rope_kv_write(const void* q, const void* k, const void* v, int io_dtype, int64_t q_stride,
                                    int64_t k_stride, int64_t v_stride, const float* q_norm, const float* k_norm,
                                    float eps, void* q_out, void* k_out, void* slab, int cache_dtype,
                                    const b200moe_kv_cache_t* cache, int32_t block_index,
                                    const int32_t* start_positions, const int32_t* new_lens,
                                    const int32_t* page_ids, const float* freqs, int order, int32_t bs,
                                    int32_t tokens_per_seq, int32_t pages_per_seq, int32_t heads, void* stream) {
  const char* who = "attn_norm_rope_kv_write";
  B200_REQUIRE(cache != nullptr, "%s: NULL cache geometry", who);
  B200_REQUIRE(dtype_ok(cache_dtype), "%s: unknown dtype", who);
  WriteArgs a{};
  a.q = q; a.k = k; a.v = v; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps; a.q_out = q_out; a.k_out = k_out;
  a.slab = slab; a.cache_dtype = cache_dtype; a.start_positions = start_positions; a.new_lens = new_lens;
  a.page_ids = page_ids; a.freqs = freqs; a.order = order; a.bs = bs; a.sl = tokens_per_seq;
  a.pages_per_seq = pages_per_seq; a.page_count = cache->page_count; a.heads = heads; a.kv_heads = cache->kv_heads;
  a.stride = cache->stride; a.blocks = cache->blocks; a.block_index = block_index; a.scale_block = 1;
  a.stride_shift = log2_of(a.stride);
  if (const int rc = check_write(who, a, io_dtype, cache->head_dim)) return rc;
  if (bs == 0) return B200MOE_OK;
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  return launch_write_io<CACHE_PLAIN>(a, io_dtype, cache->head_dim, static_cast<cudaStream_t>(stream));
}

int b200moe_kv8_read(const void* slab, const float* scales, const b200moe_kv8_cache_t* cache, int32_t block_index,
                     const int32_t* page_ids, const int32_t* seq_lens, int32_t bs, int32_t pages_per_seq,
                     int32_t max_seq_len, void* k_out, void* v_out, int out_dtype, void* stream) {
  const char* who = "kv8_read";
  if (const int rc = check_kv8(who, cache, block_index)) return rc;
  B200_REQUIRE(bs >= 0 && bs <= 65535 && pages_per_seq >= 1 && max_seq_len >= 0, "%s: bad sizes", who);
  if (bs == 0 || max_seq_len == 0) return B200MOE_OK;
  B200_REQUIRE(slab && scales && page_ids && seq_lens && k_out && v_out, "%s: NULL buffer", who);
  B200_REQUIRE(dtype_ok(out_dtype), "%s: unknown dtype", who);
  B200_REQUIRE(aligned16(slab) && aligned16(k_out) && aligned16(v_out) && (reinterpret_cast<uintptr_t>(scales) & 7) == 0,
               "%s: slab and outputs must be 16-byte aligned, scales 8-byte", who);
  ReadArgs a;
  a.slab = static_cast<const uint8_t*>(slab); a.scales = scales; a.page_ids = page_ids; a.seq_lens = seq_lens;
  a.k_out = k_out; a.v_out = v_out; a.pages_per_seq = pages_per_seq;
  a.page_count = cache->page_count; a.max_len = max_seq_len; a.kv_heads = cache->kv_heads; a.stride = cache->stride;
  a.blocks = cache->blocks; a.block_index = block_index; a.stride_shift = log2_of(cache->stride); a.block_shift = log2_of(cache->scale_block);
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  const dim3 grid((max_seq_len - 1) / RD_TILE + 1, cache->kv_heads, bs);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool h64 = cache->head_dim == 64;
  if (out_dtype == B200MOE_DT_F32)
    return h64 ? launch_read<float, 64>(a, cache->code, grid, st) : launch_read<float, 128>(a, cache->code, grid, st);
  if (out_dtype == B200MOE_DT_F16)
    return h64 ? launch_read<__half, 64>(a, cache->code, grid, st) : launch_read<__half, 128>(a, cache->code, grid, st);
  return h64 ? launch_read<__nv_bfloat16, 64>(a, cache->code, grid, st)
             : launch_read<__nv_bfloat16, 128>(a, cache->code, grid, st);
}

size_t b200moe_kv8_attend_scratch_bytes(const b200moe_kv8_cache_t* cache, int32_t bs, int32_t new_tokens,
                                        int32_t heads, int32_t max_seq_len) {
  if (cache == nullptr || bs <= 0 || new_tokens <= 0 || new_tokens > MAX_NEW_TOKENS || heads <= 0 || max_seq_len <= 0 ||
      cache->kv_heads <= 0 || heads % cache->kv_heads != 0)
    return 0;
  const int rows = heads / cache->kv_heads * new_tokens;
  size_t most = 0;  // the activations' type is not known here: enough for any
  for (const int bits : {BITS_ONE, BITS_P, BITS_BOTH}) {
    const size_t n = static_cast<size_t>(attend_ctas(*cache, bs, rows, bits, max_seq_len)) * 2 *
                     attend_tile_rows(rows) * (cache->head_dim + 4) * sizeof(float);
    most = n > most ? n : most;
  }
  return most;
}

int b200moe_kv8_attend(const void* q, int q_dtype, int64_t q_stride, const void* slab, const float* scales,
                       const b200moe_kv8_cache_t* cache, int32_t block_index, const int32_t* page_ids,
                       const int32_t* seq_lens, int32_t bs, int32_t new_tokens, int32_t pages_per_seq,
                       int32_t heads, int32_t max_seq_len, float scale, float softcap, void* out, int out_dtype,
                       void* scratch, size_t scratch_bytes, void* stream) {
  const char* who = "kv8_attend";
  if (const int rc = check_kv8(who, cache, block_index)) return rc;
  B200_REQUIRE(bs >= 0 && bs <= 65535 && pages_per_seq >= 1 && heads >= 1 && max_seq_len >= 1, "%s: bad sizes", who);
  B200_REQUIRE(static_cast<int64_t>(pages_per_seq) * cache->stride <= 1 << 30, "%s: more than 2^30 positions", who);
  B200_REQUIRE(new_tokens >= 1 && new_tokens <= MAX_NEW_TOKENS, "%s: new_tokens %d (1 to %d)", who, new_tokens,
               MAX_NEW_TOKENS);
  B200_REQUIRE(std::isfinite(softcap), "%s: softcap must be finite", who);
  if (bs == 0) return B200MOE_OK;
  B200_REQUIRE(q && slab && scales && page_ids && seq_lens && out && scratch, "%s: NULL buffer", who);
  B200_REQUIRE(dtype_ok(q_dtype) && dtype_ok(out_dtype), "%s: unknown dtype", who);
  B200_REQUIRE(heads % cache->kv_heads == 0, "%s: heads (%d) must be a multiple of the kv heads (%d)", who, heads,
               cache->kv_heads);
  B200_REQUIRE(q_stride >= static_cast<int64_t>(heads) * cache->head_dim &&
                   q_stride % (16 / static_cast<int64_t>(dt_bytes(q_dtype))) == 0 && aligned16(q) && aligned16(out) &&
                   aligned16(slab) && aligned16(scratch) && (reinterpret_cast<uintptr_t>(scales) & 7) == 0,
               "%s: q, its row stride, out, slab and scratch must be multiples of 16 bytes, scales 8-byte aligned", who);
  const size_t need = b200moe_kv8_attend_scratch_bytes(cache, bs, new_tokens, heads, max_seq_len);
  if (scratch_bytes < need) {
    set_error("%s: scratch needs %zu bytes, got %zu", who, need, scratch_bytes);
    return B200MOE_ERR_WORKSPACE;
  }
  AttendArgs a;
  a.q = q; a.q_stride = q_stride; a.q_dtype = q_dtype; a.slab = static_cast<const uint8_t*>(slab); a.scales = scales;
  a.page_ids = page_ids; a.seq_lens = seq_lens; a.out = out; a.partial = static_cast<float*>(scratch);
  a.out_dtype = out_dtype; a.bs = bs; a.sl = new_tokens;
  a.pages_per_seq = pages_per_seq; a.page_count = cache->page_count; a.heads = heads; a.kv_heads = cache->kv_heads;
  a.stride = cache->stride; a.blocks = cache->blocks; a.block_index = block_index;
  const bool f32 = q_dtype == B200MOE_DT_F32 || out_dtype == B200MOE_DT_F32;
  const int bits = f32 || softcap > CAP_FAST ? BITS_BOTH : out_dtype == B200MOE_DT_F16 ? BITS_P : BITS_ONE;
  const int rows = heads / cache->kv_heads * new_tokens, tile = attend_tile_rows(rows), hd = cache->head_dim;
  a.row_tiles = (rows + tile - 1) / tile;
  a.ctas = attend_ctas(*cache, bs, rows, bits, max_seq_len);
  a.stride_shift = log2_of(a.stride);
  a.block_shift = log2_of(cache->scale_block);
  B200_REQUIRE(static_cast<double>(bs) * a.kv_heads * a.row_tiles *
                       (2.0 + START_STEPS + pages_per_seq * static_cast<double>(a.stride) / AT_STEP) < 2147483647.0,
               "%s: too many positions for one call", who);
  B200_REQUIRE(static_cast<int64_t>(bs) * heads * new_tokens <= 0x7fffffff, "%s: too many rows for one call", who);
  a.scale = scale; a.softcap = softcap;
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = cache->code == B200MOE_KV8_INT8;
  int rc;
  if (hd == 64)
    rc = i8 ? launch_attend_rows<64, B200MOE_KV8_INT8>(a, bits, tile, st)
            : launch_attend_rows<64, B200MOE_KV8_E4M3>(a, bits, tile, st);
  else
    rc = i8 ? launch_attend_rows<128, B200MOE_KV8_INT8>(a, bits, tile, st)
            : launch_attend_rows<128, B200MOE_KV8_E4M3>(a, bits, tile, st);
  if (rc) return rc;
  if (static_cast<int64_t>(pages_per_seq) * a.stride <= AT_STEP) return B200MOE_OK;  // no segment is longer than a step
  return hd == 64 ? launch_merge<64>(a, tile, st) : launch_merge<128>(a, tile, st);
}

}  // extern "C"
