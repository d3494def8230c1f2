// The 8-bit KV cache: its write (norms of queries and keys, rotation and quantisation in
// one pass), its read-back, and attention over it.
//
// Slab: [page][transformer block][kv head][K | V][position in page][head dim] codes of one
// byte, int8 or e4m3; scales: [page][transformer block][kv head][scale block][K | V] fp32.
// A code c stands for c * s.
#include <cuda_fp8.h>

#include "kernels.h"

namespace b200moe {
namespace {

constexpr int MAX_SCALE_BLOCK = 64;
constexpr int MAX_NEW_TOKENS = 16;

inline bool dtype_ok(int dt) { return dt == B200MOE_DT_F32 || dt == B200MOE_DT_F16 || dt == B200MOE_DT_BF16; }
inline size_t dt_bytes(int dt) { return dt == B200MOE_DT_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ------------------------------------------------------------- rows of 16 or 32 bits
// N consecutive elements as one load or store.
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
__device__ __forceinline__ void load_elems(const __half* p, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 f = __half22float2(reinterpret_cast<const __half2*>(p)[i / 2]);
    v[i] = f.x; v[i + 1] = f.y;
  }
}
template <int N>
__device__ __forceinline__ void load_elems(const __nv_bfloat16* p, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 f = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(p)[i / 2]);
    v[i] = f.x; v[i + 1] = f.y;
  }
}
__device__ __forceinline__ void store_pair(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void store_pair(__half* p, float a, float b) {
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b);
}
__device__ __forceinline__ void store_pair(__nv_bfloat16* p, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}
template <int N, typename T>
__device__ __forceinline__ void store_elems(T* p, const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) store_pair(p + i, v[i], v[i + 1]);
}
template <typename T>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(__float2half_rn(v));
  else return __bfloat162float(__float2bfloat16_rn(v));
}
template <int N>
__device__ __forceinline__ void store_as(void* p, int dtype, size_t i, const float (&v)[N]) {
  if (dtype == B200MOE_DT_F32) store_elems(static_cast<float*>(p) + i, v);
  else if (dtype == B200MOE_DT_F16) store_elems(static_cast<__half*>(p) + i, v);
  else store_elems(static_cast<__nv_bfloat16*>(p) + i, v);
}

// ------------------------------------------------------------------------- codes
template <int CODE>
__device__ __forceinline__ float code_to_float(uint8_t c) {
  if constexpr (CODE == B200MOE_KV8_INT8) return static_cast<float>(static_cast<int8_t>(c));
  else return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}
// y = value / scale, at most 2^-10 above qmax: rounds to a code without clamping
template <int CODE>
__device__ __forceinline__ uint8_t float_to_code(float y) {
  if constexpr (CODE == B200MOE_KV8_INT8) return static_cast<uint8_t>(__float2int_rn(y));
  else return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
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
  int tile, tiles;                    // positions per tile; tiles per sequence
  int32_t* status;
};

enum { CACHE_INT8 = B200MOE_KV8_INT8, CACHE_E4M3 = B200MOE_KV8_E4M3, CACHE_PLAIN = 2 };

constexpr int WR_THREADS = 256;
constexpr int WR_WARPS = WR_THREADS / 32;
constexpr int WR_TILE = 64;           // most positions of a tile
constexpr float QMAX[2] = {127.f, 448.f};

// A lane's N elements of a row, normed and rotated.  cs: the row's cosines and sines.
template <int HD>
__device__ __forceinline__ void norm_rotate(float (&x)[HD / 32], const float (&w)[HD / 32], bool norm, float eps,
                                            const float2* cs, int order, int lane) {
  constexpr int N = HD / 32;
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = 1.0f / sqrtf(ss / HD + eps);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = w[i] * (x[i] * r);
  }
  if (order == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 c = cs[(lane * N + i) / 2];
      const float re = x[i], im = x[i + 1];
      x[i] = re * c.x - im * c.y;
      x[i + 1] = im * c.x + re * c.y;
    }
  } else {  // the other half of the pair is 16 lanes away
    const float sign = lane < 16 ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float2 c = cs[(lane & 15) * N + i];
      const float other = __shfl_xor_sync(0xffffffffu, x[i], 16);
      x[i] = x[i] * c.x + sign * other * c.y;
    }
  }
}

// One CTA per (sequence, tile of positions, kv head): K and V of the tile and the queries
// of the heads that share the kv head.  Tiles are aligned in absolute positions, so that a
// tile holds whole scale blocks.  A warp takes one row at a time, a lane HD / 32
// consecutive elements of it.
template <typename T, int HD, int KIND>
__global__ void __launch_bounds__(WR_THREADS) norm_rope_write_kernel(const WriteArgs a) {
  constexpr int N = HD / 32;
  __shared__ float2 s_cs[WR_TILE][HD / 2];
  __shared__ long long s_row[WR_TILE];     // K row of each position in the slab, in rows of HD elements; -1: not written
  __shared__ unsigned s_amax[2][WR_TILE];  // of each scale block, as bits
  __shared__ float s_inv[2][WR_TILE], s_shrink[2];
  const int b = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles, kvh = blockIdx.y;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int G = a.heads / a.kv_heads, B = a.scale_block, TP = a.tile;
  const int start_in = a.start_positions[b];
  const long long start = start_in < 0 ? 0 : start_in;
  int count = start_in < 0 ? 0 : a.new_lens != nullptr ? a.new_lens[b] : a.sl;
  count = count < 0 ? 0 : count > a.sl ? a.sl : count;
  const long long p0 = (start / TP + tile) * TP;  // first position of the tile
  const int lo = static_cast<int>(start > p0 ? start - p0 : 0);
  const long long end = start + a.sl - p0, wend = start + count - p0;
  const int hi = static_cast<int>(end < TP ? end : TP);     // rows lo .. hi are rotated,
  const int whi = static_cast<int>(wend < TP ? wend : TP);  // rows lo .. whi written
  if (lo >= hi) return;

  for (int i = t; i < (hi - lo) * (HD / 2); i += WR_THREADS) {
    const int r = lo + i / (HD / 2), j = i % (HD / 2);
    // the angle in half turns, reduced in 64 bits: exact to 2^-24 at any position
    const double turns = static_cast<double>(p0 + r) * (static_cast<double>(a.freqs[j]) * 0.31830988618379067154);
    float sn, cs;
    sincospif(static_cast<float>(turns - 2.0 * rint(0.5 * turns)), &sn, &cs);
    s_cs[r][j] = make_float2(cs, sn);
  }
  const int first = lo - lo % (KIND == CACHE_PLAIN ? 1 : B);  // earlier rows of a continued block included
  for (int r = first + t; r < whi; r += WR_THREADS) {
    const long long pos = p0 + r, slot = pos / a.stride;
    long long row = -1;
    const int off = static_cast<int>(pos % a.stride);
    const long long page = slot < a.pages_per_seq ? a.page_ids[static_cast<size_t>(b) * a.pages_per_seq + slot] : -1;
    if (page < 0 || page >= a.page_count) {
      atomicOr(a.status, DEV_ERR_BOUNDS);
    } else if constexpr (KIND == CACHE_PLAIN) {
      row = (((page * a.blocks + a.block_index) * 2) * a.stride + off) * a.kv_heads + kvh;
    } else {
      row = ((page * a.blocks + a.block_index) * a.kv_heads + kvh) * 2 * a.stride + off;
    }
    s_row[r] = row;
  }
  for (int i = t; i < 2 * WR_TILE; i += WR_THREADS) (&s_amax[0][0])[i] = 0u;
  __syncthreads();

  float qw[N], kw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    qw[i] = a.q_norm != nullptr ? a.q_norm[lane * N + i] : 1.f;
    kw[i] = a.k_norm != nullptr ? a.k_norm[lane * N + i] : 1.f;
  }
  const T *q = static_cast<const T*>(a.q), *k = static_cast<const T*>(a.k), *v = static_cast<const T*>(a.v);
  const long long tok0 = static_cast<long long>(b) * a.sl + (p0 - start);  // token of row 0
  auto k_row = [&](int r, float (&x)[N]) {
    load_elems(k + (tok0 + r) * a.k_stride + kvh * HD + lane * N, x);
    norm_rotate<HD>(x, kw, a.k_norm != nullptr, a.eps, s_cs[r], a.order, lane);
  };
  auto v_row = [&](int r, float (&x)[N]) { load_elems(v + (tok0 + r) * a.v_stride + kvh * HD + lane * N, x); };

  // K: rotated rows; K and V: the largest magnitude of each scale block
  for (int r = lo + warp; r < hi; r += WR_WARPS) {
    float x[N];
    k_row(r, x);
    if (a.k_out != nullptr)
      store_elems(static_cast<T*>(a.k_out) + ((tok0 + r) * a.kv_heads + kvh) * HD + lane * N, x);
    if (r >= whi) continue;
    float y[N];
    v_row(r, y);
    if constexpr (KIND == CACHE_PLAIN) {
      if (s_row[r] < 0) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = round_to<T>(x[i]);
      const size_t at = static_cast<size_t>(s_row[r]) * HD + lane * N;
      store_as(a.slab, a.cache_dtype, at, x);
      store_as(a.slab, a.cache_dtype, at + static_cast<size_t>(a.stride) * a.kv_heads * HD, y);
    } else {
      unsigned mk = 0, mv = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        mk = max(mk, __float_as_uint(x[i]) & 0x7fffffffu);
        mv = max(mv, __float_as_uint(y[i]) & 0x7fffffffu);
      }
      mk = __reduce_max_sync(0xffffffffu, mk);
      mv = __reduce_max_sync(0xffffffffu, mv);
      if (lane == 0) {
        atomicMax(&s_amax[0][r / B], mk);
        atomicMax(&s_amax[1][r / B], mv);
      }
    }
  }
  // queries
  for (int i = warp; i < (hi - lo) * G; i += WR_WARPS) {
    const int r = lo + i / G, h = kvh * G + i % G;
    float x[N];
    load_elems(q + (tok0 + r) * a.q_stride + static_cast<long long>(h) * HD + lane * N, x);
    norm_rotate<HD>(x, qw, a.q_norm != nullptr, a.eps, s_cs[r], a.order, lane);
    store_elems(static_cast<T*>(a.q_out) + ((tok0 + r) * a.heads + h) * HD + lane * N, x);
  }
  if constexpr (KIND != CACHE_PLAIN) {
    __syncthreads();
    // the scale of each block: a thread for each block and K | V
    constexpr float qmax = QMAX[KIND];
    constexpr float tiny = 7.888609052210118e-31f;  // 2^-100
    for (int i = t; i < 2 * (TP / B); i += WR_THREADS) {
      const int blk = i >> 1, kv = i & 1;
      const int r0 = max(blk * B, lo), r1 = min(blk * B + B, whi);
      if (r0 >= r1 || s_row[r0] < 0) continue;
      const unsigned bits = s_amax[kv][blk];
      const float amax = __uint_as_float(bits);
      const long long row = s_row[r0];
      const long long pair = (row / (2 * a.stride)) * (a.stride / B) + (row % a.stride) / B;
      const bool continued = lo > blk * B;
      const float before = continued ? a.scales[2 * pair + kv] : 0.f;
      float s, shrink = 1.f;
      if (bits >= 0x7f800000u || before != before) {
        s = __uint_as_float(0x7fc00000u);
      } else if (before > 0.f) {
        s = before;
        const float ratio = amax / (before * qmax * (1.f + 0.0009765625f));
        if (ratio > 1.f) {
          int e;
          const float m = frexpf(ratio, &e);
          if (m == 0.5f) --e;
          s = ldexpf(before, e);
          shrink = ldexpf(1.f, -e);
        }
      } else {
        s = amax < qmax * tiny ? 0.f : amax / qmax;
      }
      if (!continued || s != before) a.scales[2 * pair + kv] = s;
      s_inv[kv][blk] = s > 0.f ? 1.f / s : 0.f;
      if (continued) s_shrink[kv] = s == s ? shrink : 1.f;
    }
    __syncthreads();
    uint8_t* slab = static_cast<uint8_t*>(a.slab);
    for (int r = lo + warp; r < whi; r += WR_WARPS) {
      if (s_row[r] < 0) continue;
      float x[N];
      uint8_t* at = slab + static_cast<size_t>(s_row[r]) * HD + lane * N;
      k_row(r, x);
#pragma unroll
      for (int i = 0; i < N; ++i) at[i] = float_to_code<KIND>(x[i] * s_inv[0][r / B]);
      v_row(r, x);
      at += static_cast<size_t>(a.stride) * HD;
#pragma unroll
      for (int i = 0; i < N; ++i) at[i] = float_to_code<KIND>(x[i] * s_inv[1][r / B]);
    }
    // the live rows of a continued block whose scale has grown
    if (first < lo && lo < whi && s_row[lo] >= 0) {
      for (int i = warp; i < 2 * (lo - first); i += WR_WARPS) {
        const int kv = i & 1, r = first + (i >> 1);
        if (s_shrink[kv] == 1.f) continue;
        uint8_t* at = slab + static_cast<size_t>(s_row[r] + (kv ? a.stride : 0)) * HD + lane * N;
#pragma unroll
        for (int j = 0; j < N; ++j) at[j] = float_to_code<KIND>(code_to_float<KIND>(at[j]) * s_shrink[kv]);
      }
    }
  }
}

template <typename T, int HD, int KIND>
int launch_write(const WriteArgs& a, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.bs) * a.tiles, a.kv_heads);
  norm_rope_write_kernel<T, HD, KIND><<<grid, WR_THREADS, 0, st>>>(a);
  B200_CHECK_CUDA(cudaGetLastError());
  return B200MOE_OK;
}
template <typename T, int KIND>
int launch_write_hd(const WriteArgs& a, int hd, cudaStream_t st) {
  return hd == 64 ? launch_write<T, 64, KIND>(a, st) : launch_write<T, 128, KIND>(a, st);
}
template <int KIND>
int launch_write_io(WriteArgs& a, int io_dtype, int hd, cudaStream_t st) {
  a.tile = KIND == CACHE_PLAIN ? 16 : a.scale_block > 16 ? a.scale_block : 16;
  a.tiles = a.sl == 1 ? 1 : (a.sl - 1) / a.tile + 2;
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
  const int64_t grid = static_cast<int64_t>(a.bs) * ((a.sl - 1) / 16 + 2);
  B200_REQUIRE(grid <= 0x7fffffff, "%s: %d sequences of %d tokens are too many for one call", who, a.bs, a.sl);
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
  B200_REQUIRE(c->code == B200MOE_KV8_INT8 || c->code == B200MOE_KV8_E4M3, "%s: unknown code %d", who, c->code);
  return B200MOE_OK;
}

// -------------------------------------------------------------------- read-back
struct ReadArgs {
  const uint8_t* slab;
  const float* scales;
  const int32_t *page_ids, *seq_lens;
  void *k_out, *v_out;
  int out_dtype, bs, pages_per_seq, page_count, max_len, kv_heads, stride, blocks, block_index, scale_block;
  int32_t* status;
};

// A thread per 16 codes: one 16-byte load, 16 values stored.
template <int HD, int CODE>
__global__ void __launch_bounds__(256) kv8_read_kernel(const ReadArgs a) {
  constexpr int VEC = HD / 16;
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  const size_t total = static_cast<size_t>(a.bs) * a.max_len * a.kv_heads * 2 * VEC;
  if (i >= total) return;
  // consecutive threads: chunk of the row, position, K | V, head, sequence
  const int c = static_cast<int>(i % VEC);
  const int pos = static_cast<int>(i / VEC % a.max_len);
  const int kv = static_cast<int>(i / VEC / a.max_len % 2);
  const int h = static_cast<int>(i / VEC / a.max_len / 2 % a.kv_heads);
  const int b = static_cast<int>(i / VEC / a.max_len / 2 / a.kv_heads);
  float y[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) y[j] = 0.f;
  if (pos < a.seq_lens[b]) {
    const int slot = pos / a.stride, off = pos % a.stride;
    const long long page = slot < a.pages_per_seq ? a.page_ids[static_cast<size_t>(b) * a.pages_per_seq + slot] : -1;
    if (page < 0 || page >= a.page_count) {
      atomicOr(a.status, DEV_ERR_BOUNDS);
    } else {
      const size_t head = (static_cast<size_t>(page) * a.blocks + a.block_index) * a.kv_heads + h;
      const uint4 raw = *reinterpret_cast<const uint4*>(a.slab + ((head * 2 + kv) * a.stride + off) * HD + 16 * c);
      const float s = a.scales[2 * (head * (a.stride / a.scale_block) + off / a.scale_block) + kv];
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = code_to_float<CODE>(static_cast<uint8_t>(w[j / 4] >> (8 * (j % 4)))) * s;
    }
  }
  const size_t at = ((static_cast<size_t>(b) * a.max_len + pos) * a.kv_heads + h) * HD + 16 * c;
  store_as(kv ? a.v_out : a.k_out, a.out_dtype, at, y);
}

// -------------------------------------------------------------------- attention
struct AttendArgs {
  const void* q;
  int64_t q_stride;
  const uint8_t* slab;
  const float* scales;
  const int32_t *page_ids, *seq_lens;
  void* out;
  int out_dtype, bs, sl, pages_per_seq, page_count, heads, kv_heads, stride, blocks, block_index, scale_block;
  float scale, softcap;
  int32_t* status;
};

// One CTA per (head, new token, sequence), a warp per position, HD / 32 elements per lane.
template <typename T, int HD, int CODE>
__global__ void __launch_bounds__(128) kv8_attend_kernel(const AttendArgs a) {
  constexpr int N = HD / 32;
  __shared__ float s_o[4][HD], s_m[4], s_l[4];
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = h / (a.heads / a.kv_heads);
  const int end = min(a.seq_lens[b] - a.sl + 1 + i, a.pages_per_seq * a.stride);
  float q[N], o[N], m = -INFINITY, l = 0.f;
  load_elems(static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * a.sl + i) * a.q_stride + h * HD + lane * N, q);
#pragma unroll
  for (int j = 0; j < N; ++j) o[j] = 0.f;
  for (int pos = warp; pos < end; pos += 4) {
    const int slot = pos / a.stride, off = pos % a.stride;
    const long long page = a.page_ids[static_cast<size_t>(b) * a.pages_per_seq + slot];
    if (page < 0 || page >= a.page_count) {
      if (lane == 0) atomicOr(a.status, DEV_ERR_BOUNDS);
      continue;
    }
    const size_t head = (static_cast<size_t>(page) * a.blocks + a.block_index) * a.kv_heads + kvh;
    const uint8_t* k = a.slab + (head * 2 * a.stride + off) * HD + lane * N;
    const uint8_t* v = k + static_cast<size_t>(a.stride) * HD;
    const float* sc = a.scales + 2 * (head * (a.stride / a.scale_block) + off / a.scale_block);
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) dot = fmaf(q[j], code_to_float<CODE>(k[j]), dot);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
    dot *= sc[0] * a.scale;
    if (a.softcap > 0.f) dot = a.softcap * tanhf(dot / a.softcap);
    const float m_new = fmaxf(m, dot), alpha = expf(m - m_new), p = expf(dot - m_new);
    m = m_new;
    l = l * alpha + p;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = o[j] * alpha + p * sc[1] * code_to_float<CODE>(v[j]);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) s_o[warp][lane * N + j] = o[j];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  __syncthreads();
  if (warp != 0) return;
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float den = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) o[j] = 0.f;
  for (int w = 0; w < 4; ++w) {
    if (s_l[w] == 0.f) continue;
    const float f = expf(s_m[w] - top);
    den += f * s_l[w];
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] += f * s_o[w][lane * N + j];
  }
#pragma unroll
  for (int j = 0; j < N; ++j) o[j] = den == 0.f ? 0.f : o[j] / den;
  store_as(a.out, a.out_dtype, ((static_cast<size_t>(b) * a.sl + i) * a.heads + h) * HD + lane * N, o);
}

template <typename T, int HD>
int launch_attend(const AttendArgs& a, int code, cudaStream_t st) {
  const dim3 grid(a.heads, a.sl, a.bs);
  if (code == B200MOE_KV8_INT8) kv8_attend_kernel<T, HD, B200MOE_KV8_INT8><<<grid, 128, 0, st>>>(a);
  else kv8_attend_kernel<T, HD, B200MOE_KV8_E4M3><<<grid, 128, 0, st>>>(a);
  B200_CHECK_CUDA(cudaGetLastError());
  return B200MOE_OK;
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
  B200_REQUIRE(bs >= 0 && pages_per_seq >= 1 && max_seq_len >= 0, "%s: bad sizes", who);
  if (bs == 0 || max_seq_len == 0) return B200MOE_OK;
  B200_REQUIRE(slab && scales && page_ids && seq_lens && k_out && v_out, "%s: NULL buffer", who);
  B200_REQUIRE(dtype_ok(out_dtype), "%s: unknown dtype", who);
  B200_REQUIRE(aligned16(slab) && aligned16(k_out) && aligned16(v_out) && (reinterpret_cast<uintptr_t>(scales) & 7) == 0,
               "%s: slab and outputs must be 16-byte aligned, scales 8-byte", who);
  ReadArgs a;
  a.slab = static_cast<const uint8_t*>(slab); a.scales = scales; a.page_ids = page_ids; a.seq_lens = seq_lens;
  a.k_out = k_out; a.v_out = v_out; a.out_dtype = out_dtype; a.bs = bs; a.pages_per_seq = pages_per_seq;
  a.page_count = cache->page_count; a.max_len = max_seq_len; a.kv_heads = cache->kv_heads; a.stride = cache->stride;
  a.blocks = cache->blocks; a.block_index = block_index; a.scale_block = cache->scale_block;
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  const size_t total = static_cast<size_t>(bs) * max_seq_len * cache->kv_heads * 2 * (cache->head_dim / 16);
  const size_t ctas = (total + 255) / 256;
  B200_REQUIRE(ctas <= 0x7fffffff, "%s: too many rows for one call", who);
  const unsigned grid = static_cast<unsigned>(ctas);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = cache->code == B200MOE_KV8_INT8;
  if (cache->head_dim == 64) {
    if (i8) kv8_read_kernel<64, B200MOE_KV8_INT8><<<grid, 256, 0, st>>>(a);
    else kv8_read_kernel<64, B200MOE_KV8_E4M3><<<grid, 256, 0, st>>>(a);
  } else {
    if (i8) kv8_read_kernel<128, B200MOE_KV8_INT8><<<grid, 256, 0, st>>>(a);
    else kv8_read_kernel<128, B200MOE_KV8_E4M3><<<grid, 256, 0, st>>>(a);
  }
  B200_CHECK_CUDA(cudaGetLastError());
  return B200MOE_OK;
}

size_t b200moe_kv8_attend_scratch_bytes(const b200moe_kv8_cache_t* cache, int32_t bs, int32_t new_tokens,
                                        int32_t heads, int32_t max_seq_len) {
  if (cache == nullptr || bs <= 0 || new_tokens <= 0 || heads <= 0 || max_seq_len <= 0) return 0;
  return 16;
}

int b200moe_kv8_attend(const void* q, int q_dtype, int64_t q_stride, const void* slab, const float* scales,
                       const b200moe_kv8_cache_t* cache, int32_t block_index, const int32_t* page_ids,
                       const int32_t* seq_lens, int32_t bs, int32_t new_tokens, int32_t pages_per_seq,
                       int32_t heads, int32_t max_seq_len, float scale, float softcap, void* out, int out_dtype,
                       void* scratch, size_t scratch_bytes, void* stream) {
  const char* who = "kv8_attend";
  if (const int rc = check_kv8(who, cache, block_index)) return rc;
  B200_REQUIRE(bs >= 0 && bs <= 65535 && pages_per_seq >= 1 && heads >= 1 && max_seq_len >= 1, "%s: bad sizes", who);
  B200_REQUIRE(new_tokens >= 1 && new_tokens <= MAX_NEW_TOKENS, "%s: new_tokens %d (1 to %d)", who, new_tokens,
               MAX_NEW_TOKENS);
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
  a.q = q; a.q_stride = q_stride; a.slab = static_cast<const uint8_t*>(slab); a.scales = scales;
  a.page_ids = page_ids; a.seq_lens = seq_lens; a.out = out; a.out_dtype = out_dtype; a.bs = bs; a.sl = new_tokens;
  a.pages_per_seq = pages_per_seq; a.page_count = cache->page_count; a.heads = heads; a.kv_heads = cache->kv_heads;
  a.stride = cache->stride; a.blocks = cache->blocks; a.block_index = block_index; a.scale_block = cache->scale_block;
  a.scale = scale; a.softcap = softcap;
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool h64 = cache->head_dim == 64;
  if (q_dtype == B200MOE_DT_F32)
    return h64 ? launch_attend<float, 64>(a, cache->code, st) : launch_attend<float, 128>(a, cache->code, st);
  if (q_dtype == B200MOE_DT_F16)
    return h64 ? launch_attend<__half, 64>(a, cache->code, st) : launch_attend<__half, 128>(a, cache->code, st);
  return h64 ? launch_attend<__nv_bfloat16, 64>(a, cache->code, st)
             : launch_attend<__nv_bfloat16, 128>(a, cache->code, st);
}

}  // extern "C"
