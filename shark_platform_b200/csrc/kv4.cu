// The 4-bit KV cache: its write (norms of queries and keys, rotation and quantisation in one
// pass), its read-back, and attention over it.
//
// Slab: [page][transformer block][kv head][K | V][position in page][head dim / 2] bytes, two
// codes each, the even element in the low half; scales: [page][transformer block][kv head]
// [K | V][position in page][head dim / 32] pairs of fp16, scale s and offset m of 32 values.
// A code c, 0 .. 15, stands for c * s + m.
#include "kv_attend.cuh"

namespace b200moe {
namespace {

constexpr int GROUP = 32;  // values of a scale

// ------------------------------------------------------------------------- write
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// N consecutive values of a lane, those of LANES neighbouring lanes being one group: their
// codes, N / 2 bytes, and the group's (scale, offset).  Infinities, NaN and scales or
// offsets beyond fp16's range make both NaN.  The quotient is taken with a reciprocal in two parts: quotients
// halfway between two codes are common (16-bit values and an 11-bit scale) and go to the even one.
template <int N, int LANES>
__device__ __forceinline__ uint32_t quantise(const float (&x)[8], int first, __half2& held) {
  float lo = x[first], hi = x[first];
#pragma unroll
  for (int i = 1; i < N; ++i) {
    lo = min_nan(lo, x[first + i]);
    hi = max_nan(hi, x[first + i]);
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  // (hi - lo) / 15, rounded: the quotient by the rounded reciprocal, then by what it leaves
  const float range = hi - lo, near = range * (1.f / 15.f), fifteenth = fmaf(fmaf(-15.f, near, range), 1.f / 15.f, near);
  held = __halves2half2(__float2half_rn(fifteenth), __float2half_rn(lo));
  const uint32_t bits = h2_as_u32(held);
  if ((bits & 0x7c00u) == 0x7c00u || (bits & 0x7c000000u) == 0x7c000000u) held = u32_as_h2(0x7fff7fffu);
  const float s = __low2float(held), m = __high2float(held);
  const float inv = s > 0.f ? rcp(s) : 0.f, inv_lo = fmaf(-inv, s, 1.f) * inv;
  // in the last place of 1.5 * 2^23 + y stands y, rounded to even (NaN gives 0); the upper bits
  // are the same for all and are taken off at once
  uint32_t codes = 0, all = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = x[first + i] - m;
    const float y = fminf(fmaxf(fmaf(d, inv, d * inv_lo), 0.f), 15.f);
    codes += __float_as_uint(y + 12582912.f) << (4 * i);
    all += 0x4b400000u << (4 * i);
  }
  return codes - all;
}
// The codes of a row's eight elements of lane c, and the scales of its groups.
template <int HD, int ORDER>
__device__ __forceinline__ void write_codes(const float (&x)[8], int c, bool some, uint8_t* codes, __half2* scales) {
  __half2 held;
  if constexpr (ORDER == 0) {
    const uint32_t w = quantise<8, 4>(x, 0, held);
    if (!some) return;
    *reinterpret_cast<uint32_t*>(codes + 4 * c) = w;
    if (c % 4 == 0) scales[c / 4] = held;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w = quantise<4, 8>(x, 4 * i, held);
      if (!some) continue;
      *reinterpret_cast<uint16_t*>(codes + i * (HD / 4) + 2 * c) = static_cast<uint16_t>(w);
      if (c % 8 == 0) scales[i * (HD / 64) + c / 8] = held;
    }
  }
}

// Rows are written alone: a CTA has tokens and either a few query heads or a few kv heads of
// each.  HD / 8 lanes have a row; a lane keeps its position's cosines and sines for all of its
// heads.  3 x 777 tokens of 32 + 16 heads (55 MB) 14.6 us, 4 x 2048 of 48 + 16 (272 MB) 51 us, 5.3 TB/s,
// 64 x 1 3.5 us.
template <typename T, int HD, int ORDER>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 3 : 4) norm_rope_write4_kernel(const WriteArgs a) {
  constexpr int LPR = HD / 8, RPW = 32 / LPR, RPP = 8 * RPW;  // lanes per row; rows of a warp, of the CTA
  constexpr int QB = 4, KB = 2;                               // heads that a lane takes at once
  grid_dep_wait();
  grid_dep_launch();
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, c = lane % LPR;
  const unsigned tok_ctas = a.kv_ctas;  // CTAs that one group of heads takes
  const int grp = static_cast<int>(blockIdx.x / tok_ctas), kv_groups = (a.kv_heads + a.tiles - 1) / a.tiles;
  const long long tokens = static_cast<long long>(a.bs) * a.sl;
  const long long mine = static_cast<long long>(blockIdx.x % tok_ctas) * RPP + warp * RPW + lane / LPR;
  const bool some = mine < tokens;
  const long long tok = some ? mine : tokens - 1;  // all lanes take part in the shuffles
  const int b = static_cast<int>(tok / a.sl), i = static_cast<int>(tok - static_cast<long long>(b) * a.sl);
  // the first rows are on their way while the angles are computed
  if (grp >= kv_groups) {
    const int h0 = (grp - kv_groups) * a.q_heads, h1 = min(h0 + a.q_heads, a.heads);
    const T* from = static_cast<const T*>(a.q) + tok * a.q_stride;
    T* to = static_cast<T*>(a.q_out) + tok * a.heads * HD;
    Raw8<T> raw[QB];
    auto fetch = [&](int h) {
#pragma unroll
      for (int g = 0; g < QB; ++g) load_row<T, HD, ORDER>(raw[g], from + min(h + g, h1 - 1) * HD, c);
    };
    fetch(h0);
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = a.q_norm != nullptr ? a.q_norm[element<HD, ORDER>(c, e)] : 1.f;
    // to 2^-22 for all types: a step of a code is far above the rows' own
    const Turn turn = turn_of<float>(static_cast<long long>(max(a.start_positions[b], 0)) + i, a.freqs, c);
    for (int h = h0; h < h1; h += QB) {
      if (h > h0) fetch(h);
#pragma unroll
      for (int g = 0; g < QB; ++g) {
        float x[8];
        raw[g].get(x);
        norm_rotate<LPR, ORDER>(x, w, a.q_norm != nullptr, a.eps, turn);
        if (some && h + g < h1) store_row<T, HD, ORDER>(to + (h + g) * HD, c, x);
      }
    }
    return;
  }
  const int h0 = grp * a.tiles, h1 = min(h0 + a.tiles, a.kv_heads);
  const T *k = static_cast<const T*>(a.k) + tok * a.k_stride, *v = static_cast<const T*>(a.v) + tok * a.v_stride;
  Raw8<T> kr[KB], vr[KB];
  auto fetch = [&](int first) {
#pragma unroll
    for (int g = 0; g < KB; ++g) {
      const int h = min(first + g, h1 - 1);
      load_row<T, HD, ORDER>(kr[g], k + h * HD, c);
      load_row<T, HD, 0>(vr[g], v + h * HD, c);
    }
  };
  fetch(h0);
  const int start = a.start_positions[b];
  const long long pos = static_cast<long long>(max(start, 0)) + i;
  // where the token's rows are in the cache; -1: not written
  const int count = start < 0 ? 0 : a.new_lens != nullptr ? min(a.new_lens[b], a.sl) : a.sl;
  long long page_row = -1;
  if (some && i < count) {
    const long long slot = a.stride_shift >= 0 ? pos >> a.stride_shift : pos / a.stride;
    const int page = slot < a.pages_per_seq ? a.page_ids[static_cast<size_t>(b) * a.pages_per_seq + slot] : -1;
    if (page < 0 || page >= a.page_count) atomicOr(a.status, DEV_ERR_BOUNDS);
    else
      page_row = (static_cast<long long>(page) * a.blocks + a.block_index) * a.kv_heads * 2 * a.stride + (pos - slot * a.stride);
  }
  T* k_out = a.k_out == nullptr ? nullptr : static_cast<T*>(a.k_out) + tok * a.kv_heads * HD;
  uint8_t* slab = static_cast<uint8_t*>(a.slab);
  __half2* scales = reinterpret_cast<__half2*>(a.scales);
  float w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = a.k_norm != nullptr ? a.k_norm[element<HD, ORDER>(c, e)] : 1.f;
  const Turn turn = turn_of<float>(pos, a.freqs, c);
  for (int first = h0; first < h1; first += KB) {
    if (first > h0) fetch(first);
#pragma unroll
    for (int g = 0; g < KB; ++g) {
      const int h = first + g;
      const bool live = some && h < h1, put = live && page_row >= 0;
      const size_t at = static_cast<size_t>(max(page_row, 0ll)) + static_cast<size_t>(min(h, h1 - 1)) * 2 * a.stride, v_at = at + a.stride;
      float x[8];
      kr[g].get(x);
      norm_rotate<LPR, ORDER>(x, w, a.k_norm != nullptr, a.eps, turn);
      if (live && k_out != nullptr) store_row<T, HD, ORDER>(k_out + h * HD, c, x);
      write_codes<HD, ORDER>(x, c, put, slab + at * (HD / 2), scales + at * (HD / GROUP));
      vr[g].get(x);
      write_codes<HD, 0>(x, c, put, slab + v_at * (HD / 2), scales + v_at * (HD / GROUP));
    }
  }
}

template <typename T, int HD>
int launch_write4(WriteArgs& a, cudaStream_t st) {
  // as many heads a lane as leave work for two CTAs per SM: a position's angles are computed once for
  // each group (eight CTAs: 4 x 2048 55 instead of 51 us, 3 x 777 15.7 instead of 14.6; one: 1 x 1500
  // 12.1 instead of 9.9)
  constexpr int RPP = 8 * (32 / (HD / 8));
  const int64_t tokens = static_cast<int64_t>(a.bs) * a.sl, tok_ctas = (tokens + RPP - 1) / RPP, want = sm_count() * 2ll;
  a.q_heads = 4;
  a.tiles = 2;  // kv heads of a lane
  while (a.q_heads < a.heads && tok_ctas * ((a.heads - 1) / (2 * a.q_heads) + 1) >= want) a.q_heads *= 2;
  while (a.tiles < a.kv_heads && tok_ctas * ((a.kv_heads - 1) / (2 * a.tiles) + 1) >= want) a.tiles *= 2;
  a.kv_ctas = static_cast<unsigned>(tok_ctas);
  const int64_t groups = (a.heads - 1) / a.q_heads + 1 + (a.kv_heads - 1) / a.tiles + 1;
  B200_REQUIRE(tok_ctas * groups < 2147483647, "attn_norm_rope_kv4_write: %d sequences of %d tokens are too many for one call",
               a.bs, a.sl);
  B200_CHECK_CUDA(launch_dependent(a.order ? norm_rope_write4_kernel<T, HD, 1> : norm_rope_write4_kernel<T, HD, 0>,
                                   dim3(static_cast<unsigned>(tok_ctas * groups)), dim3(256), 0, st, a));
  return B200MOE_OK;
}
template <typename T>
int launch_write4_hd(WriteArgs& a, int hd, cudaStream_t st) {
  return hd == 64 ? launch_write4<T, 64>(a, st) : launch_write4<T, 128>(a, st);
}

int check_kv4(const char* who, const b200moe_kv_cache_t* c, int32_t block_index) {
  B200_REQUIRE(c != nullptr, "%s: NULL cache geometry", who);
  B200_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim %d (64 and 128 are built)", who, c->head_dim);
  B200_REQUIRE(c->blocks >= 1 && c->stride >= 1 && c->kv_heads >= 1 && c->kv_heads <= 65535 && c->page_count >= 1 &&
                   block_index >= 0 && block_index < c->blocks,
               "%s: bad cache geometry", who);
  B200_REQUIRE(static_cast<double>(c->page_count) * c->blocks * c->kv_heads * 2.0 * c->stride < 4294967295.0,
               "%s: the cache has more than 2^32 rows", who);
  return B200MOE_OK;
}

// -------------------------------------------------------------------- read-back
struct Read4Args {
  const uint8_t* slab;
  const __half2* scales;
  const int32_t *page_ids, *seq_lens;
  void *k_out, *v_out;
  int pages_per_seq, page_count, max_len, kv_heads, stride, blocks, block_index, stride_shift;
  int32_t* status;
};

// The E values of a lane's codes: c as the last place of 2^23 + c.
template <int E>
__device__ __forceinline__ void values_of(uint32_t codes, __half2 held, float (&v)[E]) {
  const float s = __low2float(held), m = __high2float(held);
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = fmaf(__uint_as_float((codes >> (4 * i) & 15u) | 0x4b000000u) - 8388608.f, s, m);
}

// One CTA per (sequence, kv head, 16 positions); a thread takes the codes of 16 bytes of
// output, K and V of several rows at once.  Bound by HBM: 32 sequences of up to 4000 positions, 8
// heads of 128, to bf16 (648 MB) 115 us, 5.6 TB/s; to fp32 (1.17 GB) 205, 5.7.
constexpr int RD4_THREADS = 128, RD4_TILE = 16;
template <typename T, int HD>
__global__ void __launch_bounds__(RD4_THREADS) kv4_read_kernel(const Read4Args a) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  constexpr int LPR = HD / E, RPP = RD4_THREADS / LPR, PASSES = RD4_TILE / RPP;
  grid_dep_wait();
  grid_dep_launch();
  const int tile = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int sub = threadIdx.x / LPR, c = threadIdx.x % LPR;
  const int len = a.seq_lens[b];
  uint32_t codes[2][PASSES];
  __half2 held[2][PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int pos = tile * RD4_TILE + i * RPP + sub;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      codes[kv][i] = 0u;
      held[kv][i] = u32_as_h2(0u);
    }
    if (pos < len && pos < a.max_len) {
      const int slot = a.stride_shift >= 0 ? pos >> a.stride_shift : pos / a.stride, off = pos - slot * a.stride;
      const int page = slot < a.pages_per_seq ? a.page_ids[static_cast<size_t>(b) * a.pages_per_seq + slot] : -1;
      if (page < 0 || page >= a.page_count) {
        atomicOr(a.status, DEV_ERR_BOUNDS);
      } else {
        const size_t row = ((static_cast<size_t>(page) * a.blocks + a.block_index) * a.kv_heads + h) * 2 * a.stride + off;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const size_t at = row + (kv ? a.stride : 0);
          const uint8_t* from = a.slab + at * (HD / 2) + c * (E / 2);
          codes[kv][i] = E == 8 ? *reinterpret_cast<const uint32_t*>(from) : *reinterpret_cast<const uint16_t*>(from);
          held[kv][i] = a.scales[at * (HD / GROUP) + c * E / GROUP];
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int pos = tile * RD4_TILE + i * RPP + sub;
    if (pos >= a.max_len) return;
    const size_t to = ((static_cast<size_t>(b) * a.max_len + pos) * a.kv_heads + h) * HD + c * E;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float y[E];
      values_of<E>(codes[kv][i], held[kv][i], y);
      T* p = static_cast<T*>(kv ? a.v_out : a.k_out) + to;
      if constexpr (E == 8) store8(p, y);
      else *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
    }
  }
}
template <typename T>
int launch_read4(const Read4Args& a, int hd, dim3 grid, cudaStream_t st) {
  B200_CHECK_CUDA(launch_dependent(hd == 64 ? kv4_read_kernel<T, 64> : kv4_read_kernel<T, 128>, grid, dim3(RD4_THREADS), 0, st, a));
  return B200MOE_OK;
}

// -------------------------------------------------------------------- attention
// o = sum_p softmax(S)_p (c_v(p) s_v(p) + m_v(p)),  S = scale * q . (c_k(p) s_k(p) + m_k(p)),
// s and m by groups g of 32 elements.  Scales and offsets stay out of the products of codes:
//   S = scale * sum_g (s_kg (c_kg . q_g) + m_kg sum(q_g))
//   o_g = sum_p P s_vg c_vg + sum_p P m_vg
// Both products run on tensor cores, positions and head elements as the rows of A and the
// query rows that share a kv head as the eight columns of B (mma.m16n8k16), as over the 8-bit
// cache.  The codes need no conversion: a code c in the low bits of 16 is the fp16 number
// c 2^-24 (a subnormal one, which the MMAs take as it is), in bits 4 .. 7 it is c 2^-20.  Of a
// word of eight codes two masks give four of them as operands and a shift the others: five
// instructions.  What is 16 times too large is made up for in q (K: elements 1, 3, 5, 7 of
// eight have q / 16) or in the output (V: odd rows of V^T).
//   * K is the A operand as it lies: a lane gets eight consecutive elements of a row, and the
//     order of an MMA's 16 elements is free as long as q's fragments have the same one.
//   * V^T comes from ldmatrix.trans on pairs of bytes: four elements of two positions.
//   * P^T is S^T's accumulator, packed and transposed within the warp (movmatrix), and times
//     s_v of a group it is the B operand of that group's products.
//   * The offsets have products of their own: m_k[position][g] times the sums of q's groups
//     (as two fp16 parts, 22 bits), and m_v^T[g][position] times P^T.
// The magnitude of a position's V, a power of two 2^e above 15 |s_vg| and |m_vg|, joins the
// softmax as a scale of V does over the 8-bit cache: with t = S log2(e) + e, P = 2^(t - max t)
// times s_v 2^(4-e) and m_v 2^-e (at most 1) is the numerator's weight and P 2^-e the
// denominator's.  What fp16 rounds off is then 2^-11 of a value or 2^-25 of the largest one.
// P is in one fp16 part for bf16 outputs and in two, 2^-22, for others; q too in two for 32-bit
// activations (BITS_*), where the codes are taken less 8 and the offsets 8 s more, in two parts:
// the two sums no longer cancel each other, and what the MMAs round off is 2^-23 of the output
// instead of many times that (1e-5 of 300 positions' output, 1e-4 of 20000's).  Those offsets are
// brought to 2^14 by a power of two of each position: m + 8 s passes fp16's range where m and s do
// not, and below 2^-14 two parts of it would have few bits.
//
// A warp owns units of 32 positions with its own softmax state and two places for a unit's K
// and V, filled by cp.async while the other is worked on.  The list of steps, its stretches
// and the merge are those of the 8-bit cache.
//
// 32 sequences of 2000 to 4000 positions, 8 kv heads of 128, 32 heads (125 MB): bf16 36 us (int8
// codes, 200 MB: 40), fp16 42, fp32 60; one of 32768 20 us; 8 x 8190, 48 heads, five new tokens, in two
// tiles of 16 rows: bf16 54 us, fp16 64.  What bounds it: before the first rows 6 us, the merge 4 us, in
// between the chain of dependent instructions of a unit (700 of a warp, issued every second clock;
// 8 and 12 warps an SM take the same time within a tenth).
// CTAs per SM at 32 x 4000: two 38.8 us, three 36.1, four (128 registers, the warps' states joined
// in two halves) 43.9.  q loaded before the first copies, which helps over the 8-bit cache, costs
// registers that wait in memory: 37.5 us.
template <int HD, int NT, int BITS>
constexpr int attend4_resident() {
  return NT == 1 && BITS != BITS_BOTH ? 3 : 2;
}

// Byte offset of 16-byte chunk c of row r in a tile of rows of HD / 2 bytes: the eight chunks
// that one ldmatrix phase reads lie in eight different bank groups.
template <int HD>
__device__ __forceinline__ uint32_t tile4_at(int r, int c) {
  if constexpr (HD == 128) return static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  else return static_cast<uint32_t>(r * 32 + ((c ^ ((r >> 2) & 1)) << 4));
}
// the product alone: no sum to add to
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// the first of a sum (a constant once loops are unrolled), or one more
__device__ __forceinline__ void mma_next(bool first, float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (first) mma_first(c, a0, a1, a2, a3, b0, b1);
  else mma(c, a0, a1, a2, a3, b0, b1);
}
// mma_first with k = 8
__device__ __forceinline__ void mma_first_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
// Codes as A operands, bits 0 .. 3 (HIGH: 4 .. 7, 16 times as large) of each half of w: as they
// lie, subnormal numbers of 2^-24 (UNIT24), or CENTRED, less 8.  The MMAs align what they add by
// the operands' exponents, and a subnormal operand's leading zeros are bits lost below (8 to 11 of
// 24: 5e-6 of a score); centred codes are normal numbers.
constexpr float UNIT24 = 5.9604644775390625e-8f;
template <bool HIGH, bool CENTRED>
__device__ __forceinline__ uint32_t codes_of(uint32_t w) {
  const uint32_t x = w & (HIGH ? 0x00f000f0u : 0x000f000fu);
  if constexpr (!CENTRED) return x;
  return h2_as_u32(__hsub2(u32_as_h2(x | 0x64006400u), u32_as_h2(HIGH ? 0x64806480u : 0x64086408u)));
}
__device__ __forceinline__ void sts_words(uint32_t to, const uint32_t (&v)[4]) { sts128(to, v); }
__device__ __forceinline__ void sts_words(uint32_t to, const uint32_t (&v)[2]) {
  asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(to), "r"(v[0]), "r"(v[1]) : "memory");
}
template <int N>
__device__ __forceinline__ void copy_small(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? N : 0;
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// e, -10 .. 21, with 16 |s| and |m| of a position's groups below 2^e: from the exponents of the
// largest ones, 4 more for s (numbers below 2^-14 count as that).
template <int CH>
__device__ __forceinline__ int magnitude(const uint32_t (&w)[CH]) {
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < CH; ++c) top = __vmaxu2(top, w[c] & 0x7fff7fffu);
  return static_cast<int>(max((top & 0xffffu) + 0x1000u, top >> 16) >> 10) - 14;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

template <int HD, int NT, int BITS>
__global__ void __launch_bounds__(AT_THREADS, (attend4_resident<HD, NT, BITS>())) kv4_attend_kernel(const AttendArgs a) {
  constexpr int CH = HD / GROUP;                    // groups of a row: 16-byte chunks of its codes
  constexpr bool SPLIT = BITS == BITS_BOTH;
  constexpr int PARTS = SPLIT ? 2 : 1, P_PARTS = BITS == BITS_ONE ? 1 : 2;
  constexpr int ROWS = 8 * NT;
  constexpr int TILE = AT_UNIT * HD / 2, STILE = AT_UNIT * CH * 4;  // bytes of a unit's codes, scales of K (or V)
  constexpr int PLACE = 2 * (TILE + STILE);
  constexpr int OPITCH = HD + 8;                    // floats
  // P is at most 2^P_TOP when the maximum is taken, 2^15 before it is again; two parts of a P below
  // 2^-3 would end among fp16's subnormal numbers
  constexpr float P_TOP = P_PARTS == 2 ? 11.f : 7.f, P_SLACK = 15.f - P_TOP;
  extern __shared__ __align__(128) uint8_t smem[];  // [warp][2][K | V codes, K | V scales], then [warp][row][OPITCH] fp32
  float* s_o = reinterpret_cast<float*>(smem + AT_WARPS * 2 * PLACE);
  __shared__ float2 s_pos[AT_WARPS][AT_UNIT];       // of each position: e (-inf: dead), 2^-e
  __shared__ __align__(16) uint32_t s_sv[AT_WARPS][AT_UNIT / 2][CH], s_mv[PARTS][AT_WARPS][AT_UNIT / 2][CH];  // of two positions, times 2^(4 - e) and 2^-e
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

  // scores and softcap as over the 8-bit cache; q is brought to [2^9, 2^10)
  const float cap2 = a.softcap * LOG2E;
  const float to_score = a.softcap > 0.f ? a.scale / a.softcap * (SPLIT ? 1.f : 2.f * LOG2E) : a.scale * LOG2E;
  const uint32_t ring = smem_u32(smem) + warp * (2 * PLACE);
  // byte offsets in a tile that this lane addresses with ldmatrix: rows 16 h + (lane & 15), chunks 2 i + (lane >> 4)
  uint32_t ld_at[CH / 2];
#pragma unroll
  for (int i = 0; i < CH / 2; ++i) ld_at[i] = tile4_at<HD>(lane & 15, 2 * i + (lane >> 4));

  // what of a segment lies in this stretch, and the warp's units of it
  struct Piece { int b, kvh, tile, x0, x1, steps, end, p_begin, p_end, units; };
  struct Walk { int seq_first, seq; };  // the current sequence and the first of its steps
  auto piece_at = [&](Walk& w, int g) {
    Piece p;
    int len = live_positions(a, w.seq);
    p.steps = steps_of(len);
    while (g - w.seq_first >= (start + p.steps) * a.kv_heads * a.row_tiles) {  // at most once: g is a step of this or the next
      w.seq_first += (start + p.steps) * a.kv_heads * a.row_tiles;
      len = live_positions(a, ++w.seq);
      p.steps = steps_of(len);
    }
    const int seg = (g - w.seq_first) / (start + p.steps), x = g - w.seq_first - seg * (start + p.steps);
    p.b = w.seq;
    p.kvh = seg / a.row_tiles;
    p.tile = seg - p.kvh * a.row_tiles;
    p.end = min(g + start + p.steps - x, g_end);
    p.x0 = max(0, x - start);
    p.x1 = max(0, x + p.end - g - start);  // 0: no step of it
    p.p_begin = p.x0 * AT_STEP + warp * AT_UNIT;
    p.p_end = min(len, p.x1 * AT_STEP);
    p.units = p.p_end > p.p_begin ? (p.p_end - p.p_begin + AT_STEP - 1) / AT_STEP : 0;
    return p;
  };

  // The warp's units in order, as far as their copies have been started: `unit` of `ahead` is
  // the next one, and the page of this lane's position in it is on its way.
  Walk walk_ahead{at.before, at.seq};
  Piece ahead = piece_at(walk_ahead, g_begin);
  int unit = 0, page = -1;
  auto find_unit = [&] {  // skips segments that leave nothing for this warp
    while (unit >= ahead.units && ahead.end < g_end) {
      ahead = piece_at(walk_ahead, ahead.end);
      unit = 0;
    }
    const int pos = ahead.p_begin + unit * AT_STEP + lane;
    if (unit < ahead.units && pos < ahead.p_end)
      page = a.page_ids[static_cast<size_t>(ahead.b) * a.pages_per_seq + (a.stride_shift >= 0 ? pos >> a.stride_shift : pos / a.stride)];
  };
  // starts the copies of that unit (zeros in the place of missing rows) into place i: a mask of
  // the positions that are there; one group per call, also without a unit
  auto issue = [&](int i) -> uint32_t {
    uint32_t live = 0;
    if (unit < ahead.units) {
      const int pos = ahead.p_begin + unit * AT_STEP + lane;
      uint32_t row = 0;
      bool ok = pos < ahead.p_end;
      if (ok && (page < 0 || page >= a.page_count)) {
        atomicOr(a.status, DEV_ERR_BOUNDS);
        ok = false;
      }
      if (ok) {
        const int off = a.stride_shift >= 0 ? pos & (a.stride - 1) : pos % a.stride;
        row = ((static_cast<uint32_t>(page) * a.blocks + a.block_index) * a.kv_heads + ahead.kvh) * 2u * a.stride + off;
      }
      live = __ballot_sync(0xffffffffu, ok);
      const uint32_t to = ring + i * PLACE, row0 = __shfl_sync(0xffffffffu, row, 0);
      constexpr int RPI = 32 / CH;  // rows of one pass of the warp
      const int r0 = lane / CH, c = lane % CH;
      static_assert(RPI % 8 == 0, "passes are whole patterns of the swizzle apart");
      if (__all_sync(0xffffffffu, ok && row == row0 + lane)) {  // within one page
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const size_t first = static_cast<size_t>(row0) + (kv ? a.stride : 0);
          const uint8_t* from = a.slab + (first + r0) * (HD / 2) + c * 16;
          const uint32_t at = to + kv * TILE + tile4_at<HD>(r0, c);
#pragma unroll
          for (int j = 0; j < CH; ++j) copy16(at + j * RPI * (HD / 2), from + j * RPI * (HD / 2), true);
          copy_small<CH * 4>(to + 2 * TILE + kv * STILE + lane * (CH * 4),
                             reinterpret_cast<const uint8_t*>(a.scales) + (first + lane) * (CH * 4), true);
        }
      } else {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            const int r = j * RPI + r0;
            const size_t from = static_cast<size_t>(__shfl_sync(0xffffffffu, row, r)) + (kv ? a.stride : 0);
            copy16(to + kv * TILE + tile4_at<HD>(r, c), a.slab + from * (HD / 2) + c * 16, live >> r & 1);
          }
          copy_small<CH * 4>(to + 2 * TILE + kv * STILE + lane * (CH * 4),
                             reinterpret_cast<const uint8_t*>(a.scales) + (static_cast<size_t>(row) + (kv ? a.stride : 0)) * (CH * 4), ok);
        }
      }
      ++unit;
    }
    copy_commit();
    find_unit();
    return live;
  };
  find_unit();
  uint32_t live_now = issue(0), live_next = issue(1);
  int place = 0;

  Walk walk{at.before, at.seq};
  for (int g = g_begin; g < g_end;) {
    const Piece cur = piece_at(walk, g);
    if (cur.x1 == 0) break;  // the stretch ends before the segment's first step
    const int b = cur.b, kvh = cur.kvh, tile = cur.tile, units = cur.units;
    if (cur.x0 == 0 && t == 0 && a.seq_lens[b] > a.pages_per_seq * a.stride) atomicOr(a.status, DEV_ERR_BOUNDS);

    // q: column gid of B is row tile * ROWS + 8 n + gid, a lane's elements 8 tig .. + 7 of each
    // chunk; its values times a power of two, those of odd elements 1 / 16 of that
    uint32_t qb[PARTS][NT][CH][4], qs[NT];
    float fold[NT][2];  // of this lane's accumulator columns 2 tig, 2 tig + 1: back to to_score units
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = tile * ROWS + 8 * n + gid;
      const int64_t from = (static_cast<int64_t>(b) * a.sl + r / G) * a.q_stride + static_cast<int64_t>(kvh * G + r % G) * HD + 8 * tig;
      float x[CH][8], top = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[c][e] = 0.f;
        if (r < rows) {
          if (SPLIT && a.q_dtype == B200MOE_DT_F32) {
            Raw8<float> raw;
            raw.load(static_cast<const float*>(a.q) + from + 32 * c);
            raw.get(x[c]);
          } else if (a.q_dtype == B200MOE_DT_F16) {
            Raw8<__half> raw;
            raw.load(static_cast<const __half*>(a.q) + from + 32 * c);
            raw.get(x[c]);
          } else {
            Raw8<__nv_bfloat16> raw;
            raw.load(static_cast<const __nv_bfloat16*>(a.q) + from + 32 * c);
            raw.get(x[c]);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[c][e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^e <= top < 2^(e + 1), so that the largest value lies in [2^9, 2^10)
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      e = e < -100 || e > 127 ? -100 : e;
      if (__float_as_uint(top) == 0x7f800000u) e = 100;
      e = min(e, 100);  // q beyond becomes infinite
      const float up = __uint_as_float(static_cast<uint32_t>(9 - e + 127) << 23);
      const float down = __uint_as_float(static_cast<uint32_t>(e - 9 + 127 + (SPLIT ? 0 : 24)) << 23) * to_score;
      fold[n][0] = __shfl_sync(0xffffffffu, down, (2 * tig) * 4);
      fold[n][1] = __shfl_sync(0xffffffffu, down, (2 * tig + 1) * 4);
      float sum[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        sum[c] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[c][i] *= up;
          sum[c] += x[c][i];
        }
        sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], 1);
        sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // pairs (i, i + 4) of the word's eight codes
          const float f = i & 1 ? 0.0625f : 1.f, u = x[c][i] * f, v = x[c][i + 4] * f;
          const __half2 h = __floats2half2_rn(u, v);
          qb[0][n][c][i] = h2_as_u32(h);
          if constexpr (SPLIT) {
            const float2 y = __half22float2(h);
            qb[PARTS - 1][n][c][i] = h2_as_u32(__floats2half2_rn(u - y.x, v - y.y));
          }
        }
      }
      // the sums, B of mma_k8: k = 2 tig, 2 tig + 1 are groups 2 (tig % (CH / 2)), + 1, first the
      // upper parts, then the lower (for two groups nothing behind those)
      const int pair = tig % (CH / 2), part = tig / (CH / 2);
      float u = sum[0], v = sum[1];
      if constexpr (CH == 4) {
        u = pair ? sum[2] : u;
        v = pair ? sum[3] : v;
      }
      const __half2 h = __floats2half2_rn(u, v);
      const float2 y = __half22float2(h);
      qs[n] = part == 0 ? h2_as_u32(h) : part == 1 ? h2_as_u32(__floats2half2_rn(u - y.x, v - y.y)) : 0u;
    }
    // the first position that a column does not see
    const int all_see = a.seq_lens[b] - a.sl + 1;
    auto seen = [&](int n, int j) { return all_see + (tile * ROWS + 8 * n + 2 * tig + j) / G; };

    float m[NT][2], l[NT][2], o[NT][2 * CH][4], om[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
      om[n][0] = om[n][1] = om[n][2] = om[n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < 2 * CH; ++c) o[n][c][0] = o[n][c][1] = o[n][c][2] = o[n][c][3] = 0.f;
    }

    for (int u = 0; u < units; ++u) {
      copy_wait<1>();
      __syncwarp();
      const uint32_t kt = ring + place * PLACE, vt = kt + TILE, ks = kt + 2 * TILE, vs = ks + STILE;
      {
        // this lane's position: the magnitude of its V, and its scales and offsets in units of it
        uint32_t w[CH];
        if constexpr (CH == 4) lds128(vs + lane * 16, w);
        else lds64(vs + lane * 8, w);
        auto largest = [&] {  // |s| in the lower, |m| in the upper half
          uint32_t top = 0;
#pragma unroll
          for (int c = 0; c < CH; ++c) top = __vmaxu2(top, w[c] & 0x7fff7fffu);
          return top;
        };
        uint32_t top = largest();
        const bool dead = !(live_now >> lane & 1);
        if (__any_sync(0xffffffffu, (top & 0xffffu) >= 0x7c00u || top >= 0x7c000000u)) {
          // a group without finite scales is NaN in the sums of the columns that see it, zeros in the products
          const int behind = cur.p_begin + u * AT_STEP;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const bool bad = (w[c] & 0x7c00u) == 0x7c00u || (w[c] & 0x7c000000u) == 0x7c000000u;
            const uint32_t where = __ballot_sync(0xffffffffu, bad);
            if (bad) w[c] = 0u;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int count = seen(n, j) - behind;
                if (gid == c && count > 0 && (where << (32 - min(count, 32))) != 0u) om[n][j] = __int_as_float(0x7fffffff);
              }
          }
          top = largest();
        }
        const float2 f = __half22float2(u32_as_h2(top));
        const float most = fmaxf(fmaxf(f.x * 16.f, f.y), 2.f * UNIT24);
        const int e = static_cast<int>(__float_as_uint(most) >> 23) - 126;  // -22 .. 21
        const float shrink = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        s_pos[warp][lane] = make_float2(dead ? -INFINITY : static_cast<float>(e), dead ? 0.f : shrink);
        // Times 2^(4 - e) and 2^-e in two steps, each within fp16's range.
        // Even lanes put down the scales of two positions, odd ones their offsets.
        const int e1 = e >> 1, e2 = e - e1;
        const uint32_t by1 = static_cast<uint32_t>((4 - e1 + 15) << 10 | (15 - e1) << 26), by_2 = static_cast<uint32_t>((15 - e2) << 10 | (15 - e2) << 26);
        const uint32_t choose = lane & 1 ? 0x3276u : 0x5410u;
        uint32_t both[CH], lower[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          uint32_t own;
          if constexpr (SPLIT) {
            float2 y = __half22float2(u32_as_h2(w[c]));
            y = make_float2(y.x * shrink, fmaf(8.f, y.x, y.y) * shrink);
            const __half2 h = __floats2half2_rn(y.x * 16.f, y.y);
            own = h2_as_u32(h);
            const uint32_t low = h2_as_u32(__float2half2_rn(y.y - __high2float(h)));
            lower[c] = __byte_perm(low, __shfl_xor_sync(0xffffffffu, low, 1), choose);
          } else {
            own = h2_as_u32(__hmul2(__hmul2(u32_as_h2(w[c]), u32_as_h2(by1)), u32_as_h2(by_2)));
          }
          both[c] = __byte_perm(own, __shfl_xor_sync(0xffffffffu, own, 1), choose);
        }
        sts_words(smem_u32(lane & 1 ? &s_mv[0][warp][lane >> 1][0] : &s_sv[warp][lane >> 1][0]), both);
        if constexpr (SPLIT)
          if (lane & 1) sts_words(smem_u32(&s_mv[PARTS - 1][warp][lane >> 1][0]), lower);
      }
      __syncwarp();
      const int p0 = cur.p_begin + u * AT_STEP;

      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // scales and offsets of positions 16 h + gid and 8 behind it
        uint32_t w0[CH], w1[CH];
        if constexpr (CH == 4) {
          lds128(ks + (16 * h + gid) * 16, w0);
          lds128(ks + (16 * h + 8 + gid) * 16, w1);
        } else {
          lds64(ks + (16 * h + gid) * 8, w0);
          lds64(ks + (16 * h + 8 + gid) * 8, w1);
        }
        {
          const bool upper = CH == 4 && (tig & 1);
          const uint32_t u0 = upper ? w0[CH - 2] : w0[0], v0 = upper ? w0[CH - 1] : w0[1];
          const uint32_t u1 = upper ? w1[CH - 2] : w1[0], v1 = upper ? w1[CH - 1] : w1[1];
          uint32_t a0 = __byte_perm(u0, v0, 0x7632), a1 = __byte_perm(u1, v1, 0x7632), b0 = 0u, b1 = 0u;
          float unit[2] = {UNIT24, UNIT24};  // of the two positions' sums
          if constexpr (SPLIT) {  // 8 s more, in two parts of numbers below 2^15
            auto both = [](uint32_t u, uint32_t v, float by, uint32_t& hi, uint32_t& lo) {
              const float2 x = __half22float2(u32_as_h2(u)), y = __half22float2(u32_as_h2(v));
              const float f = fmaf(8.f, x.x, x.y) * by, g = fmaf(8.f, y.x, y.y) * by;
              const __half2 top = __floats2half2_rn(f, g);
              hi = h2_as_u32(top);
              lo = h2_as_u32(__floats2half2_rn(f - __low2float(top), g - __high2float(top)));
            };
            const int e0 = magnitude<CH>(w0), e1 = magnitude<CH>(w1);
            unit[0] = power_of_two(e0 - 14);
            unit[1] = power_of_two(e1 - 14);
            both(u0, v0, power_of_two(14 - e0), a0, b0);
            both(u1, v1, power_of_two(14 - e1), a1, b1);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (SPLIT) mma_first(s[h][n], a0, a1, b0, b1, qs[n], qs[n]);
            else mma_first_k8(s[h][n], a0, a1, qs[n]);
#pragma unroll
            for (int k = 0; k < 4; ++k) s[h][n][k] *= unit[k >> 1];
          }
        }
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
          uint32_t w[4];
          ldsm_x4(kt + ld_at[c / 2] + 16 * h * (HD / 2), w);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t x0 = w[2 * i], x1 = w[2 * i + 1], y0 = x0 >> 8, y1 = x1 >> 8;
            float acc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
              for (int p = 0; p < PARTS; ++p) {
                const uint32_t* q = qb[p][n][c + i];
                mma_next(p == 0, acc[n], codes_of<false, SPLIT>(x0), codes_of<false, SPLIT>(x1), codes_of<true, SPLIT>(x0), codes_of<true, SPLIT>(x1), q[0], q[1]);
                mma(acc[n], codes_of<false, SPLIT>(y0), codes_of<false, SPLIT>(y1), codes_of<true, SPLIT>(y0), codes_of<true, SPLIT>(y1), q[2], q[3]);
              }
              const float s0 = __low2float(u32_as_h2(w0[c + i])), s1 = __low2float(u32_as_h2(w1[c + i]));
              s[h][n][0] = fmaf(acc[n][0], s0, s[h][n][0]);
              s[h][n][1] = fmaf(acc[n][1], s0, s[h][n][1]);
              s[h][n][2] = fmaf(acc[n][2], s1, s[h][n][2]);
              s[h][n][3] = fmaf(acc[n][3], s1, s[h][n][3]);
            }
          }
        }
      }

      // scores of positions 16 h + 8 j + gid, columns 2 tig + e
      float top[NT][2], small[2][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 f = s_pos[warp][16 * h + 8 * j + gid];
          small[h][j] = f.y;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x;
              if (a.softcap > 0.f) {
                if constexpr (SPLIT) x = fmaf(cap2, tanhf(s[h][n][2 * j + e] * fold[n][e]), f.x);
                else x = fmaf(-2.f * cap2, rcp(ex2(s[h][n][2 * j + e] * fold[n][e]) + 1.f), cap2 + f.x);
              } else {
                x = fmaf(s[h][n][2 * j + e], fold[n][e], f.x);
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
        for (int e = 0; e < 2; ++e) moves |= top[n][e] > m[n][e] + P_SLACK;
      if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = top[n][e];
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
            const float m_new = fmaxf(m[n][e], v);
            const float root = m_new == -INFINITY ? 1.f : state_root(m[n][e], m_new), alpha = root * root;
            m[n][e] = m_new;
            l[n][e] = l[n][e] * root * root;
            om[n][e] *= alpha;
#pragma unroll
            for (int c = 0; c < 2 * CH; ++c) { o[n][c][e] *= alpha; o[n][c][2 + e] *= alpha; }
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
            l[n][0] = fmaf(u0, small[h][j], l[n][0]);
            l[n][1] = fmaf(u1, small[h][j], l[n][1]);
            const __half2 hp = __floats2half2_rn(u0, u1);
            pb[0][n][h][j] = transpose8x8(h2_as_u32(hp));
            if constexpr (P_PARTS == 2) {
              const float2 f = __half22float2(hp);
              pb[P_PARTS - 1][n][h][j] = transpose8x8(h2_as_u32(__floats2half2_rn(u0 - f.x, u1 - f.y)));
            }
          }
      }
      // The tensor cores cut off what a sum's last bit cannot hold, always towards zero, and the
      // codes' sums are many times the output (the offsets cancel them): a unit's products are
      // summed apart and added with rounding, or a long stretch would lose 2^-25 of them at every step.
      {
        float unit[NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < PARTS; ++i) {
            const uint32_t a0 = gid < CH ? s_mv[i][warp][8 * h + tig][gid % CH] : 0u, a2 = gid < CH ? s_mv[i][warp][8 * h + 4 + tig][gid % CH] : 0u;
#pragma unroll
            for (int p = 0; p < P_PARTS - i; ++p)
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma_next(h + i + p == 0, unit[n], a0, 0u, a2, 0u, pb[p][n][h][0], pb[p][n][h][1]);
          }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          om[n][0] += unit[n][0];
          om[n][1] += unit[n][1];
        }
      }
      // scales of the positions 2 tig, + 1 and eight behind them, of both halves
      uint32_t sv[2][2][CH];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t at = smem_u32(&s_sv[warp][8 * h + 4 * j + tig][0]);
          if constexpr (CH == 4) lds128(at, sv[h][j]);
          else lds64(at, sv[h][j]);
        }
#pragma unroll
      for (int c = 0; c < CH; c += 2) {
        uint32_t w[2][4];
        ldsm_x4_trans(vt + ld_at[c / 2], w[0]);
        ldsm_x4_trans(vt + ld_at[c / 2] + 16 * (HD / 2), w[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float unit[NT][2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x0 = w[h][2 * i], x1 = w[h][2 * i + 1], y0 = x0 >> 8, y1 = x1 >> 8;
            const __half2 s0 = u32_as_h2(sv[h][0][c + i]), s1 = u32_as_h2(sv[h][1][c + i]);
            auto products = [&](bool first, int n, uint32_t b0, uint32_t b1) {
              mma_next(first, unit[n][0], codes_of<false, SPLIT>(x0), codes_of<true, SPLIT>(x0), codes_of<false, SPLIT>(x1), codes_of<true, SPLIT>(x1), b0, b1);
              mma_next(first, unit[n][1], codes_of<false, SPLIT>(y0), codes_of<true, SPLIT>(y0), codes_of<false, SPLIT>(y1), codes_of<true, SPLIT>(y1), b0, b1);
            };
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const __half2 p0 = u32_as_h2(pb[0][n][h][0]), p1 = u32_as_h2(pb[0][n][h][1]);
              const __half2 b0 = __hmul2(p0, s0), b1 = __hmul2(p1, s1);
              products(h == 0, n, h2_as_u32(b0), h2_as_u32(b1));
              if constexpr (P_PARTS == 2)  // what the product lost, and the lower part's
                products(false, n, h2_as_u32(__hfma2(u32_as_h2(pb[P_PARTS - 1][n][h][0]), s0, __hfma2(p0, s0, __hneg2(b0)))),
                         h2_as_u32(__hfma2(u32_as_h2(pb[P_PARTS - 1][n][h][1]), s1, __hfma2(p1, s1, __hneg2(b1)))));
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int k = 0; k < 4; ++k) o[n][2 * (c + i) + y][k] += unit[n][y][k];
        }
      }
      __syncwarp();  // the place is read
      live_now = live_next;
      live_next = issue(place);
      place ^= 1;
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
        if (gid == 0) s_ml[warp][r] = make_float2(m[n][e], v);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const float off = __shfl_sync(0xffffffffu, om[n][e], c * 4 + tig);
          // scales are 16 times themselves, and odd elements' codes again
          constexpr float even = SPLIT ? 0.0625f : 0.0625f / UNIT24, odd = even * 0.0625f;
          const float(&d0)[4] = o[n][2 * c], (&d1)[4] = o[n][2 * c + 1];
          *reinterpret_cast<float4*>(&s_o[(warp * ROWS + r) * OPITCH + 32 * c + 4 * gid]) =
              make_float4(fmaf(d0[e], even, off), fmaf(d0[2 + e], odd, off), fmaf(d1[e], even, off), fmaf(d1[2 + e], odd, off));
        }
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

// CTAs of a call: as many as are resident at once, or one for each step of a full page table
// where those are fewer.
int attend4_ctas(const b200moe_kv_cache_t& c, int bs, int rows, int bits, int max_seq_len) {
  const int tile = attend_tile_rows(rows);
  const int64_t steps = (static_cast<int64_t>(max_seq_len) + AT_STEP - 1) / AT_STEP * bs * c.kv_heads * ((rows + tile - 1) / tile);
  const int64_t resident = static_cast<int64_t>(sm_count()) *
      (tile == 8 && bits != BITS_BOTH ? attend4_resident<128, 1, BITS_ONE>() : attend4_resident<128, 2, BITS_ONE>());
  return static_cast<int>(steps < resident ? steps : resident);
}

template <int HD, int NT, int BITS>
int launch_attend4(const AttendArgs& a, cudaStream_t st) {
  constexpr int SMEM = AT_WARPS * 2 * AT_UNIT * (HD + HD / GROUP * 8) + AT_WARPS * 8 * NT * (HD + 8) * 4;
  auto kern = kv4_attend_kernel<HD, NT, BITS>;
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
template <int HD>
int launch_attend4_rows(const AttendArgs& a, int bits, int tile_rows, cudaStream_t st) {
  const bool one = tile_rows == 8;
  if (bits == BITS_BOTH) return one ? launch_attend4<HD, 1, BITS_BOTH>(a, st) : launch_attend4<HD, 2, BITS_BOTH>(a, st);
  if (bits == BITS_P) return one ? launch_attend4<HD, 1, BITS_P>(a, st) : launch_attend4<HD, 2, BITS_P>(a, st);
  return one ? launch_attend4<HD, 1, BITS_ONE>(a, st) : launch_attend4<HD, 2, BITS_ONE>(a, st);
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" {

int b200moe_attn_norm_rope_kv4_write(const void* q, const void* k, const void* v, int io_dtype, int64_t q_stride,
                                     int64_t k_stride, int64_t v_stride, const float* q_norm, const float* k_norm,
                                     float eps, void* q_out, void* k_out, void* slab, void* scales,
                                     const b200moe_kv_cache_t* cache, int32_t block_index,
                                     const int32_t* start_positions, const int32_t* new_lens, const int32_t* page_ids,
                                     const float* freqs, int order, int32_t bs, int32_t tokens_per_seq,
                                     int32_t pages_per_seq, int32_t heads, void* stream) {
  const char* who = "attn_norm_rope_kv4_write";
  if (const int rc = check_kv4(who, cache, block_index)) return rc;
  WriteArgs a{};
  a.q = q; a.k = k; a.v = v; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps; a.q_out = q_out; a.k_out = k_out;
  a.slab = slab; a.scales = static_cast<float*>(scales); a.start_positions = start_positions; a.new_lens = new_lens;
  a.page_ids = page_ids; a.freqs = freqs; a.order = order; a.bs = bs; a.sl = tokens_per_seq;
  a.pages_per_seq = pages_per_seq; a.page_count = cache->page_count; a.heads = heads; a.kv_heads = cache->kv_heads;
  a.stride = cache->stride; a.blocks = cache->blocks; a.block_index = block_index; a.scale_block = 1;
  a.stride_shift = log2_of(a.stride);
  if (const int rc = check_write(who, a, io_dtype, cache->head_dim)) return rc;
  if (bs == 0) return B200MOE_OK;
  B200_REQUIRE(scales != nullptr && aligned16(scales), "%s: scales must be given and 16-byte aligned", who);
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (io_dtype == B200MOE_DT_F32) return launch_write4_hd<float>(a, cache->head_dim, st);
  if (io_dtype == B200MOE_DT_F16) return launch_write4_hd<__half>(a, cache->head_dim, st);
  return launch_write4_hd<__nv_bfloat16>(a, cache->head_dim, st);
}

int b200moe_kv4_read(const void* slab, const void* scales, const b200moe_kv_cache_t* cache, int32_t block_index,
                     const int32_t* page_ids, const int32_t* seq_lens, int32_t bs, int32_t pages_per_seq,
                     int32_t max_seq_len, void* k_out, void* v_out, int out_dtype, void* stream) {
  const char* who = "kv4_read";
  if (const int rc = check_kv4(who, cache, block_index)) return rc;
  B200_REQUIRE(bs >= 0 && bs <= 65535 && pages_per_seq >= 1 && max_seq_len >= 0, "%s: bad sizes", who);
  if (bs == 0 || max_seq_len == 0) return B200MOE_OK;
  B200_REQUIRE(slab && scales && page_ids && seq_lens && k_out && v_out, "%s: NULL buffer", who);
  B200_REQUIRE(dtype_ok(out_dtype), "%s: unknown dtype", who);
  B200_REQUIRE(aligned16(slab) && aligned16(k_out) && aligned16(v_out) && aligned16(scales),
               "%s: slab, scales and outputs must be 16-byte aligned", who);
  Read4Args a;
  a.slab = static_cast<const uint8_t*>(slab); a.scales = static_cast<const __half2*>(scales); a.page_ids = page_ids;
  a.seq_lens = seq_lens; a.k_out = k_out; a.v_out = v_out; a.pages_per_seq = pages_per_seq;
  a.page_count = cache->page_count; a.max_len = max_seq_len; a.kv_heads = cache->kv_heads; a.stride = cache->stride;
  a.blocks = cache->blocks; a.block_index = block_index; a.stride_shift = log2_of(cache->stride);
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  const dim3 grid((max_seq_len - 1) / RD4_TILE + 1, cache->kv_heads, bs);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == B200MOE_DT_F32) return launch_read4<float>(a, cache->head_dim, grid, st);
  if (out_dtype == B200MOE_DT_F16) return launch_read4<__half>(a, cache->head_dim, grid, st);
  return launch_read4<__nv_bfloat16>(a, cache->head_dim, grid, st);
}

size_t b200moe_kv4_attend_scratch_bytes(const b200moe_kv_cache_t* cache, int32_t bs, int32_t new_tokens, int32_t heads,
                                        int32_t max_seq_len) {
  if (cache == nullptr || bs <= 0 || new_tokens <= 0 || new_tokens > MAX_NEW_TOKENS || heads <= 0 || max_seq_len <= 0 ||
      cache->kv_heads <= 0 || heads % cache->kv_heads != 0)
    return 0;
  const int rows = heads / cache->kv_heads * new_tokens;
  // the activations' type is not known here: enough for the most CTAs
  return static_cast<size_t>(attend4_ctas(*cache, bs, rows, BITS_ONE, max_seq_len)) * 2 * attend_tile_rows(rows) *
         (cache->head_dim + 4) * sizeof(float);
}

int b200moe_kv4_attend(const void* q, int q_dtype, int64_t q_stride, const void* slab, const void* scales,
                       const b200moe_kv_cache_t* cache, int32_t block_index, const int32_t* page_ids,
                       const int32_t* seq_lens, int32_t bs, int32_t new_tokens, int32_t pages_per_seq, int32_t heads,
                       int32_t max_seq_len, float scale, float softcap, void* out, int out_dtype, void* scratch,
                       size_t scratch_bytes, void* stream) {
  const char* who = "kv4_attend";
  if (const int rc = check_kv4(who, cache, block_index)) return rc;
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
                   aligned16(slab) && aligned16(scratch) && aligned16(scales),
               "%s: q, its row stride, out, slab, scales and scratch must be multiples of 16 bytes", who);
  const size_t need = b200moe_kv4_attend_scratch_bytes(cache, bs, new_tokens, heads, max_seq_len);
  if (scratch_bytes < need) {
    set_error("%s: scratch needs %zu bytes, got %zu", who, need, scratch_bytes);
    return B200MOE_ERR_WORKSPACE;
  }
  AttendArgs a{};
  a.q = q; a.q_stride = q_stride; a.q_dtype = q_dtype; a.slab = static_cast<const uint8_t*>(slab);
  a.scales = static_cast<const float*>(scales);
  a.page_ids = page_ids; a.seq_lens = seq_lens; a.out = out; a.partial = static_cast<float*>(scratch);
  a.out_dtype = out_dtype; a.bs = bs; a.sl = new_tokens;
  a.pages_per_seq = pages_per_seq; a.page_count = cache->page_count; a.heads = heads; a.kv_heads = cache->kv_heads;
  a.stride = cache->stride; a.blocks = cache->blocks; a.block_index = block_index;
  const bool f32 = q_dtype == B200MOE_DT_F32 || out_dtype == B200MOE_DT_F32;
  const int bits = f32 || softcap > CAP_FAST ? BITS_BOTH : out_dtype == B200MOE_DT_F16 ? BITS_P : BITS_ONE;
  const int rows = heads / cache->kv_heads * new_tokens, tile = attend_tile_rows(rows), hd = cache->head_dim;
  a.row_tiles = (rows + tile - 1) / tile;
  a.ctas = attend4_ctas(*cache, bs, rows, bits, max_seq_len);
  a.stride_shift = log2_of(a.stride);
  B200_REQUIRE(static_cast<double>(bs) * a.kv_heads * a.row_tiles *
                       (2.0 + START_STEPS + pages_per_seq * static_cast<double>(a.stride) / AT_STEP) < 2147483647.0,
               "%s: too many positions for one call", who);
  B200_REQUIRE(static_cast<int64_t>(bs) * heads * new_tokens <= 0x7fffffff, "%s: too many rows for one call", who);
  a.scale = scale; a.softcap = usable_softcap(softcap);
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = hd == 64 ? launch_attend4_rows<64>(a, bits, tile, st) : launch_attend4_rows<128>(a, bits, tile, st);
  if (rc) return rc;
  if (static_cast<int64_t>(pages_per_seq) * a.stride <= AT_STEP) return B200MOE_OK;  // no segment is longer than a step
  return hd == 64 ? launch_merge<64>(a, tile, st) : launch_merge<128>(a, tile, st);
}

}  // extern "C"
