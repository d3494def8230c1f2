// Attention of whole prompts: packed sequences of different lengths, causal, grouped heads.
//
// Row i of a sequence of n rows of q and m rows of k and v attends k rows 0 .. m - n + i:
//   o_i = sum_j softmax_j(S_ij) v_j,   S_ij = scale * q_i . k_j  (softcap: c tanh(S_ij / c)).
// One pass over k and v with the running maximum m_i and sum l_i of each row:
//   m' = max(m, max_j S_ij),  l' = l 2^(m - m') + sum_j 2^(S_ij - m'),  o' likewise
// with scores in units of log 2.
//
// Work items: a tile of consecutive tokens of a sequence and the query heads of one kv head
// (of a group of more heads than a tile has rows, a part of them); row r of a tile is token
// r / heads, head r % heads, so that one read of k and v serves all of them.  A CTA takes items
// i, i + CTAs, ...; the list is ordered by the tile's place in its sequence, last tiles first:
// they have the most keys, and the short ones fill the end.  It is made on the device from the
// sequences' bounds, which the host does not know: by the loading warp for the others, or (32-bit
// rows) by every warp on its own.
#include "kv_attend.cuh"
#include "tcgen05.cuh"

namespace b200moe {
namespace {

struct PromptArgs {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // of tokens, in elements
  const int32_t *cu_q, *cu_k;            // [bs + 1]; cu_k NULL: as cu_q
  void* out;
  int64_t q_rows, k_rows;
  int out_dtype, bs, heads, kv_heads;
  int group, parts;       // heads of a tile; parts of a group of heads
  uint32_t inv_group;     // 2^16 / group, rounded up: exact quotients of rows of a tile
  int tokens;             // of a tile
  int splits;             // parts that the keys of a tile are cut into, at most
  unsigned units;         // parts of one kv head that should come out
  bool uneven;            // or two or three times as many, whichever ends first
  float cut;              // parts for each tile of keys, where the sequences are not looked at
  float* partial;         // [row of q][head][splits][HD + 4]: numerator, maximum, denominator; the first: cut
  float scale, softcap;
  int32_t* status;
};

// Where a sequence lies: within the rows there are, whatever the bounds say.
struct Span { int begin, len; };
__device__ __forceinline__ Span span_of(const int32_t* cu, int b, int64_t rows, int32_t* status) {
  const int64_t lo = cu[b], hi = cu[b + 1];
  const int64_t begin = lo < 0 ? 0 : lo > rows ? rows : lo, end = hi < begin ? begin : hi > rows ? rows : hi;
  if (status != nullptr && (begin != lo || end != hi)) atomicOr(status, DEV_ERR_BOUNDS);
  return {static_cast<int>(begin), static_cast<int>(end - begin)};
}

struct Item {
  int seq, tile, kvh, part, chunk;
  bool some;
};
// Keys that the last of `toks` tokens from tok0 on sees, of a sequence of n tokens and m keys.
__device__ __forceinline__ int keys_seen(int n, int m, int tok0, int toks) { return max(0, min(m, tok0 + toks + m - n)); }
// Parts of a tile's keys, `cut` of them for each tile of `step` keys; the first of the keys of part i.
__device__ __forceinline__ int chunks_of(int keys, int step, float cut, int splits) {
  return max(1, min(splits, __float2int_ru(fmaf(static_cast<float>((keys + step - 1) / step), cut, -1e-4f))));
}
__device__ __forceinline__ int chunk_begin(int keys, int step, int chunks, int i) {
  return static_cast<int>(static_cast<int64_t>((keys + step - 1) / step) * i / chunks) * step;
}
// The list of items, walked by a whole warp with rising indices.
struct ItemWalk {
  int t, b0;         // tiles with this place in their sequence are current, in 32 sequences from b0 on
  long long before;  // items before those
  int n, m;          // rows of q and k of sequence `lane`
  __device__ __forceinline__ static void lengths(const PromptArgs& a, int b, int& n, int& m) {
    n = b < a.bs ? span_of(a.cu_q, b, a.q_rows, nullptr).len : 0;
    m = b < a.bs ? span_of(a.cu_k != nullptr ? a.cu_k : a.cu_q, b, a.k_rows, nullptr).len : 0;
  }
  __device__ __forceinline__ ItemWalk(const PromptArgs& a, int lane) : t(0), b0(0), before(0) {
    lengths(a, lane, n, m);
    int most = (n + a.tokens - 1) / a.tokens;
    for (int b = lane + 32; b < a.bs; b += 32) most = max(most, (span_of(a.cu_q, b, a.q_rows, nullptr).len + a.tokens - 1) / a.tokens);
    t = __reduce_max_sync(0xffffffffu, most) - 1;
    if (blockIdx.x == 0)
      for (int b = lane; b < a.bs; b += 32) {
        span_of(a.cu_q, b, a.q_rows, a.status);
        if (a.cu_k != nullptr) span_of(a.cu_k, b, a.k_rows, a.status);
      }
  }
  // items of a sequence of n and m rows with tile t, apart from heads
  __device__ __forceinline__ static int chunks(const PromptArgs& a, int n, int m, int t, int step, float cut) {
    const int tok0 = t * a.tokens;
    if (tok0 >= n) return 0;
    return a.splits == 1 ? 1 : chunks_of(keys_seen(n, m, tok0, min(a.tokens, n - tok0)), step, cut, a.splits);
  }
  // Parts for each tile of keys, so that there are no more than a.units: the sum of ceil(x cut) over
  // tiles of x tiles of keys is at most the sum of x cut, and one for each.  (The largest cut, by a
  // search, ends the longest part 2 tiles of 28 earlier, and its code took 2 us to fetch and run.)
  __device__ __forceinline__ float cut(const PromptArgs& a, int step) const {
    if (a.splits == 1 || a.bs > 32) return a.cut;
    const unsigned count = (n + a.tokens - 1) / a.tokens, most = (m + step - 1) / step;
    const unsigned items = __reduce_add_sync(0xffffffffu, count), tiles = __reduce_add_sync(0xffffffffu, count * most);
    const unsigned longest = __reduce_max_sync(0xffffffffu, count > 0 ? most : 0);
    const float most_parts = __fdividef(static_cast<float>(a.splits), static_cast<float>(longest));
    auto within = [&](float units) {
      return fminf(most_parts, __fdividef(fmaxf(units - static_cast<float>(items), 0.f), static_cast<float>(tiles)));
    };
    if (tiles == 0) return 0.f;
    const float units = static_cast<float>(a.units);
    if (!a.uneven) return within(units);
    float best = 0.f, least = 3e38f;
#pragma unroll 1
    for (float r = 1.f; r <= 3.f; r += 1.f) {
      const float x = within(r * units);
      const int mine = chunks_of(m, step, x, a.splits);
      const float time = r * static_cast<float>(__reduce_max_sync(0xffffffffu, count > 0 ? (most + mine - 1) / mine : 0) + 2);
      if (time < least) least = time, best = x;
    }
    return best;
  }
  __device__ __forceinline__ Item find(const PromptArgs& a, int lane, int step, float cut, long long i) {
    const int each = a.kv_heads * a.parts;
    for (; t >= 0; --t, b0 = 0) {
      for (; b0 < a.bs; b0 += 32) {
        int nb = n, mb = m;
        if (a.bs > 32) lengths(a, b0 + lane, nb, mb);
        const int own = chunks(a, nb, mb, t, step, cut);
        int sum = own;
        if (a.splits == 1) {
          sum = __popc(__ballot_sync(0xffffffffu, own) & (0xffffffffu >> (31 - lane)));
        } else {
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
          }
        }
        const long long all = static_cast<long long>(__shfl_sync(0xffffffffu, sum, 31)) * each;
        if (i < before + all) {
          const int r = static_cast<int>(i - before), c = r / each, h = r - c * each;  // chunk c of those of 32 sequences
          const int which = __ffs(__ballot_sync(0xffffffffu, sum > c)) - 1;
          const int chunk = c - __shfl_sync(0xffffffffu, sum - own, which);
          return {b0 + which, t, h / a.parts, h % a.parts, chunk, true};
        }
        before += all;
      }
    }
    return {0, 0, 0, 0, 0, false};
  }
};
// The r-th item of a CTA: there and back through the CTAs, so that none gets the largest of every round.
__device__ __forceinline__ long long item_of(long long r) {
  return r * gridDim.x + (r & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// Rows of no sequence are zeros.
template <typename T>
__device__ __forceinline__ void zero_rest(const PromptArgs& a, int hd, int threads) {
  const int64_t first = a.bs > 0 ? max(static_cast<int64_t>(0), min(static_cast<int64_t>(a.cu_q[0]), a.q_rows)) : a.q_rows;
  const int64_t last = a.bs > 0 ? max(first, min(static_cast<int64_t>(a.cu_q[a.bs]), a.q_rows)) : a.q_rows;
  const int64_t row16 = static_cast<int64_t>(a.heads) * hd * sizeof(T) / 16, count = (first + a.q_rows - last) * row16;
  uint4* out = static_cast<uint4*>(a.out);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * threads + threadIdx.x; i < count; i += static_cast<int64_t>(gridDim.x) * threads)
    out[i < first * row16 ? i : i + (last - first) * row16] = make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void zero_rest(const PromptArgs& a, int hd, int threads) {
  if (a.out_dtype == B200MOE_DT_F32) zero_rest<float>(a, hd, threads);
  else zero_rest<__half>(a, hd, threads);
}

// ------------------------------------------------------------------ 32-bit rows
// Tiles of 64 (heads of 64) or 128 rows and 64 keys on the fp32 units: thread (ty, tx) of 8 or
// 16 by 16 has rows 8 ty .. + 7, keys tx + 16 j of the scores and elements 4 tx + 64 n .. + 3 of the output, so
// that 16 bytes from shared memory serve eight or four products.  K of the next tile is on its
// way while the softmax and V's products of this one run, V during the scores.  Everything is
// fp32.  6 x 777 tokens of 16 heads over 4 of 64 192 us, 25 TFLOP/s; 2048 of 32 over 8 of 128 963 us, 36 (torch's
// fused attention 2816):
// bound by shared memory (12 loads of 16 bytes for 128 products a thread) and by the few warps that
// fit.  (Four rows a thread 205, with K and V loaded in between 258 us; heads of 64 by 8 lanes a row and
// 64 threads, with a third fewer loads for a product, 276.)
constexpr int SP_KEYS = 64, SP_R = 8;
template <int HD>
struct SpCfg {
  // as many CTAs as shared memory and registers hold: 3 of 128 threads, 1 of 256
  static constexpr int ROWS = HD == 64 ? 64 : 128, THREADS = 2 * ROWS, RESIDENT = HD == 64 ? 3 : 1;
  static constexpr int PITCH = HD + 4, PP = SP_KEYS + 4;
  static constexpr int SMEM = ((ROWS + 2 * SP_KEYS) * PITCH + ROWS * PP) * 4;
};

template <int HD>
__global__ void __launch_bounds__(SpCfg<HD>::THREADS, SpCfg<HD>::RESIDENT) prompt_attend_kernel(const PromptArgs a) {
  constexpr int SP_ROWS = SpCfg<HD>::ROWS, SP_THREADS = SpCfg<HD>::THREADS, PITCH = SpCfg<HD>::PITCH, PP = SpCfg<HD>::PP, NO = HD / 64, C = HD / 4;
  extern __shared__ __align__(16) float sp_smem[];
  float *sq = sp_smem, *sk = sq + SP_ROWS * PITCH, *sv = sk + SP_KEYS * PITCH, *sp = sv + SP_KEYS * PITCH;
  grid_dep_wait();
  grid_dep_launch();
  const int t = threadIdx.x, lane = t & 31, ty = t >> 4, tx = t & 15;
  const float *q = static_cast<const float*>(a.q), *k = static_cast<const float*>(a.k), *v = static_cast<const float*>(a.v);
  const int G = a.heads / a.kv_heads;
  const float to_score = a.softcap > 0.f ? a.scale / a.softcap : a.scale * LOG2E, cap2 = a.softcap * LOG2E;
  ItemWalk walk(a, lane);
  for (long long r = 0;; ++r) {
    const Item it = walk.find(a, lane, SP_KEYS, 0.f, item_of(r));
    if (!it.some) break;
    const Span qs = span_of(a.cu_q, it.seq, a.q_rows, nullptr), ks = span_of(a.cu_k != nullptr ? a.cu_k : a.cu_q, it.seq, a.k_rows, nullptr);
    const int tok0 = it.tile * a.tokens, toks = min(a.tokens, qs.len - tok0);
    const int h0 = it.part * a.group, hs = min(a.group, G - h0), rows = toks * hs;
    const int shift = ks.len - qs.len;  // row i sees keys up to i + shift
    const int keys = keys_seen(qs.len, ks.len, tok0, toks);
    // 64 rows of K or V from key k0 on, zeros behind the last key; one group of copies
    auto fetch = [&](float* to, const float* from, int64_t stride, int k0) {
      from += (static_cast<int64_t>(ks.begin) + k0) * stride + it.kvh * HD;
#pragma unroll
      for (int i = 0; i < SP_KEYS * C / SP_THREADS; ++i) {
        const int e = i * SP_THREADS + t, j = e / C, c = e % C * 4;
        const bool some = k0 + j < keys;
        copy16(smem_u32(to + j * PITCH + c), some ? from + j * stride + c : from, some);
      }
      copy_commit();
    };
    __syncthreads();  // the last item's tiles are read
    if (keys > 0) fetch(sk, k, a.k_stride, 0);
    for (int e = t; e < SP_ROWS * C; e += SP_THREADS) {
      const int j = e / C, c = e % C * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j < rows)
        x = *reinterpret_cast<const float4*>(q + (static_cast<int64_t>(qs.begin) + tok0 + j / hs) * a.q_stride +
                                             static_cast<int64_t>(it.kvh * G + h0 + j % hs) * HD + c);
      *reinterpret_cast<float4*>(sq + j * PITCH + c) = x;
    }
    float m[SP_R], l[SP_R], o[SP_R][NO][4];
#pragma unroll
    for (int i = 0; i < SP_R; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int n = 0; n < NO; ++n) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
    }
    for (int k0 = 0; k0 < keys; k0 += SP_KEYS) {
      copy_wait<0>();
      __syncthreads();  // K is there, V of the last tile is read
      fetch(sv, v, a.v_stride, k0);
      float s[SP_R][4] = {};
#pragma unroll 2
      for (int d = 0; d < HD; d += 4) {
        float4 y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(sk + (tx + 16 * j) * PITCH + d);
#pragma unroll
        for (int i = 0; i < SP_R; ++i) {
          const float4 x = *reinterpret_cast<const float4*>(sq + (SP_R * ty + i) * PITCH + d);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[i][j] = fmaf(x.x, y[j].x, s[i][j]);
            s[i][j] = fmaf(x.y, y[j].y, s[i][j]);
            s[i][j] = fmaf(x.z, y[j].z, s[i][j]);
            s[i][j] = fmaf(x.w, y[j].w, s[i][j]);
          }
        }
      }
      __syncthreads();  // K is read: the next one takes its place
      if (k0 + SP_KEYS < keys) fetch(sk, k, a.k_stride, k0 + SP_KEYS);
      // where not all rows see all keys, a weight of -0 leaves infinities and NaN out (a seen key's
      // weight may be 0, and an infinity times that is NaN)
      const bool masked = k0 + SP_KEYS > tok0 + shift + 1;
#pragma unroll
      for (int i = 0; i < SP_R; ++i) {
        const int seen = masked ? min(ks.len, tok0 + (SP_R * ty + i) / hs + shift + 1) - k0 : SP_KEYS;
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = s[i][j] * to_score;
          if (a.softcap > 0.f) x = cap2 * tanhf(x);
          s[i][j] = tx + 16 * j < seen ? x : -INFINITY;
          top = fmaxf(top, s[i][j]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float m_new = fmaxf(m[i], top), from = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp2f(m[i] - from);
        m[i] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2f(s[i][j] - from);
          sum += p;
          sp[(SP_R * ty + i) * PP + tx + 16 * j] = s[i][j] == -INFINITY ? -0.f : p;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        l[i] = fmaf(l[i], alpha, sum);
#pragma unroll
        for (int n = 0; n < NO; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][n][e] *= alpha;
      }
      if (k0 + SP_KEYS < keys) copy_wait<1>();
      else copy_wait<0>();
      __syncthreads();  // V is there, and the weights
      auto products = [&](auto some, int from, int to) {
#pragma unroll 1
        for (int j = from; j < to; j += 4) {
          float4 p[SP_R];
#pragma unroll
          for (int i = 0; i < SP_R; ++i) p[i] = *reinterpret_cast<const float4*>(sp + (SP_R * ty + i) * PP + j);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
#pragma unroll
            for (int n = 0; n < NO; ++n) {
              const float4 y = *reinterpret_cast<const float4*>(sv + (j + jj) * PITCH + 4 * tx + 64 * n);
#pragma unroll
              for (int i = 0; i < SP_R; ++i) {
                const float w = jj == 0 ? p[i].x : jj == 1 ? p[i].y : jj == 2 ? p[i].z : p[i].w;
                if (decltype(some)::value && __float_as_uint(w) == 0x80000000u) continue;
                o[i][n][0] = fmaf(w, y.x, o[i][n][0]);
                o[i][n][1] = fmaf(w, y.y, o[i][n][1]);
                o[i][n][2] = fmaf(w, y.z, o[i][n][2]);
                o[i][n][3] = fmaf(w, y.w, o[i][n][3]);
              }
            }
        }
      };
      // keys that all rows see; those that some do
      const int all_see = masked ? max(0, tok0 + shift + 1 - k0) & ~3 : SP_KEYS;
      products(std::false_type(), 0, all_see);
      if (masked) products(std::true_type(), all_see, min(SP_KEYS, keys - k0));
    }
#pragma unroll
    for (int i = 0; i < SP_R; ++i) {
      const int row = SP_R * ty + i;
      if (row >= rows) continue;
      const float f = l[i] == 0.f ? 0.f : 1.f / l[i];
      const size_t to = ((static_cast<size_t>(qs.begin) + tok0 + row / hs) * a.heads + it.kvh * G + h0 + row % hs) * HD + 4 * tx;
#pragma unroll
      for (int n = 0; n < NO; ++n) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = l[i] == 0.f ? 0.f : o[i][n][e] * f;
        store_as(a.out, a.out_dtype, to + 64 * n, y);
      }
    }
  }
  zero_rest(a, HD, SP_THREADS);
}

template <int HD>
int launch_prompt(PromptArgs& a, cudaStream_t st) {
  const int G = a.heads / a.kv_heads;
  constexpr int ROWS = SpCfg<HD>::ROWS;
  a.group = G < ROWS ? G : ROWS;
  a.parts = (G + a.group - 1) / a.group;
  a.tokens = ROWS / a.group;
  a.splits = 1;
  auto kern = prompt_attend_kernel<HD>;
  B200_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SpCfg<HD>::SMEM));
  const int64_t items = (a.q_rows / a.tokens + a.bs) * a.kv_heads * a.parts + 1, resident = static_cast<int64_t>(sm_count()) * SpCfg<HD>::RESIDENT;
  B200_CHECK_CUDA(launch_dependent(kern, dim3(static_cast<unsigned>(items < resident ? items : resident)), dim3(SpCfg<HD>::THREADS),
                                   SpCfg<HD>::SMEM, st, a));
  return B200MOE_OK;
}

// ------------------------------------------------------------------ tensor cores
// 16-bit rows: an item is two tiles of 128 rows, S = Q K^T and O += P V by tcgen05.mma with the
// accumulators in tensor memory (S0, S1, O0, O1: all 512 columns at 128 elements a head).
//   warps 0-3, 4-7  the softmax of tile 0, 1: a thread has a row.  S out of tensor memory, its
//                   maximum, P = 2^(S - m) in the type of V back over it as the A operand of
//                   the second product.  O is rescaled when the maximum has grown by more
//                   than 2^P_SLACK, by the same threads.  The output at the end.
//   warps 8, 9      issue the MMAs of tile 0, 1: S(0), then PV(j), S(j + 1) ...; while one tile's
//                   products run the other's softmax does.
//   warp 10         makes the list of items and loads: Q of an item, K and V tiles of 128 keys
//                   (128-byte swizzle; K is K-major, V, whose keys are the reduction, MN-major)
//   warp 11         looks at V tiles whose keys not all rows see: rows behind the sequence are
//                   other data and become zeros, infinities and NaN too (a weight of zero does
//                   not hide them from the product); where those are is noted, and they are
//                   added at the end to the rows that see them.
// Sums and statistics are fp32.  P is rounded to the type of V, as the output is after it: the
// error against 64 bits is at most sqrt(2) of what rounding the output alone costs (2.1e-3 of 1.6e-3
// for bf16; P in two parts would cost half again as many MMAs), and for fp16 weights below 2^-24 of
// the largest what P_TOP says.
// An MMA reads P where a later one writes S: the tensor core executes a thread's MMAs in order.
//
// A step (128 keys of both tiles) needs 2048 clocks of the tensor core (4096 products a clock) and
// as many of the special-function unit (16 exponentials a clock), side by side; it takes about 3100:
// S out of tensor memory, the maximum and the way from the last P to the next S are in no other
// unit's shadow when both tiles wait.  One B200, 32 heads over 8 of 128, bf16, other inputs each time: 8192
// tokens 460 to 505 us by the clock that the power limit leaves (1.1 to 1.2 PFLOP/s; 420 at best on the
// same inputs again), 4096 123 us, 1.12; 16 x 1024 of 48 heads 272, with a softcap 475 (a polynomial of five
// products a pair of scores, and a minimum beside the maximum).  torch's fused attention: 394, 111 and 230.
// An item costs about two steps beside its own (start, last product, output).
// On the way there, 8192 tokens, the same inputs again: every role walking the list itself 545 us; descriptions of items
// with a run-time index, which puts them into local memory, 474; rows stored through shared memory
// 434.  Not kept: two threads a row, 16 warps (both tiles then wait and compute at the same time)
// 572 for 545; 3 to 8 of 16 pairs of exponentials as polynomials of degree 4 by the fp32 units 474 for
// 444; weights computed with the old maximum while the new one is found 499 for 446 (more live registers).
constexpr int TP_THREADS = 384, TP_ROWS = 128, TP_KEYS = 128, TP_SUB = 128 * 128;
constexpr int TP_WARP_MMA = 8, TP_WARP_LOAD = 10, TP_WARP_CLEAN = 11;
constexpr int TP_BAD = 4;   // items whose notes of bad values may be in use at once
constexpr int TP_WORK = 4;  // items whose descriptions may be in use at once

template <int HD>
struct TpCfg {
  static constexpr int SUBS = HD / 64, TILE = SUBS * TP_SUB;  // 128 rows of 64 elements each
  static constexpr int OFF_K = 2 * TILE, OFF_V = 4 * TILE, OFF_BAD = 6 * TILE;
  static constexpr int OFF_WORK = OFF_BAD + TP_BAD * 3 * HD * 4, OFF_BAR = OFF_WORK + TP_WORK * 64;
  static constexpr int SMEM = 1024 + OFF_BAR + 320;
  static_assert(SMEM <= 232448, "shared memory budget");
};
// P is 2^P_TOP for the maximum that was taken last, and at most 2^(P_TOP + P_SLACK).  fp16 ends at 2^16
// and has subnormal numbers below 2^-14: weights down to 2^-24 of the largest have all their bits, of
// smaller ones 2^-35 of it is lost at most.  (With P = 1 for the largest, 2^-25 of it: all of an output
// whose largest weights have values of zero.)  bf16 has the exponents of 32 bits.  Rescaling from 2^4 on
// instead, for one more bit: 16 x 1500 of 48 heads with a softcap 542 for 535 us.
template <typename T> constexpr float P_TOP_OF = std::is_same<T, __half>::value ? 10.f : 0.f;
template <typename T> constexpr float P_SLACK_OF = std::is_same<T, __half>::value ? 5.9f : 8.f;

// V as the B operand: 64 elements a row of 128 bytes, eight keys 1024 bytes apart, the next 64
// elements TP_SUB further.
__device__ __forceinline__ uint64_t smem_desc_v(uint32_t addr) {
  return smem_desc_sw128(addr) | static_cast<uint64_t>(TP_SUB >> 4) << 16;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* tmap, int32_t x, int32_t y, int32_t z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

// What the roles of a CTA know of an item.
struct Work {
  int q0, toks, tok0;     // first row of q, tokens (-1: no item, the list has ended), first token of the item
  int kvh, h0, hs;        // kv head; heads of its group: first, how many
  int k0, begin, end;     // first row of k; keys of this item
  int shift;              // token i sees keys up to i + shift
  int n0, n1;             // tiles of keys of each tile of rows
  int chunk, chunks;
  int unused[2];
  __device__ __forceinline__ int tiles() const { return max(n0, n1); }
  __device__ __forceinline__ int tiles_of(int g) const { return g == 0 ? n0 : n1; }
};
static_assert(sizeof(Work) == 64, "four 16-byte words");
__device__ __forceinline__ Work work_of(const PromptArgs& a, const Item& it, float cut) {
  Work w;
  const Span qs = span_of(a.cu_q, it.seq, a.q_rows, nullptr), ks = span_of(a.cu_k != nullptr ? a.cu_k : a.cu_q, it.seq, a.k_rows, nullptr);
  const int G = a.heads / a.kv_heads, per = a.tokens / 2;
  w.tok0 = it.tile * a.tokens;
  w.toks = min(a.tokens, qs.len - w.tok0);
  w.q0 = qs.begin + w.tok0;
  w.kvh = it.kvh;
  w.h0 = it.part * a.group;
  w.hs = min(a.group, G - w.h0);
  w.k0 = ks.begin;
  w.shift = ks.len - qs.len;
  const int keys = keys_seen(qs.len, ks.len, w.tok0, w.toks);
  w.chunk = it.chunk;
  w.chunks = a.splits == 1 ? 1 : chunks_of(keys, TP_KEYS, cut, a.splits);
  w.begin = w.chunks == 1 ? 0 : chunk_begin(keys, TP_KEYS, w.chunks, it.chunk);
  w.end = w.chunks == 1 ? keys : min(keys, chunk_begin(keys, TP_KEYS, w.chunks, it.chunk + 1));
  auto tiles = [&](int g) {
    const int mine = min(per, w.toks - g * per);
    const int last = mine > 0 ? min(w.end, keys_seen(qs.len, ks.len, w.tok0 + g * per, mine)) : 0;
    return last > w.begin ? (last - w.begin + TP_KEYS - 1) / TP_KEYS : 0;
  };
  w.n0 = tiles(0);
  w.n1 = tiles(1);
  return w;
}

// two fp32 numbers of one 64-bit register, and their arithmetic
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// NaN where one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void store_sector(void* to, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b) { return pack2(static_cast<const T*>(nullptr), a, b); }

// tanh(z) for |z| <= 1/2 is z times this polynomial in z^2 (minimax, off by 2^-20.8).
constexpr float TANH[4] = {0.999999463558197f, -0.33326318860054016f, 0.13190296292304993f, -0.044402219355106354f};

template <typename T, int HD, bool CAP>
__global__ void __launch_bounds__(TP_THREADS, 1)
prompt_attend_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const PromptArgs a) {
  using C = TpCfg<HD>;
  constexpr float P_TOP = P_TOP_OF<T>, P_SLACK = P_SLACK_OF<T>;
  extern __shared__ uint8_t tp_smem[];
  __shared__ int s_abort, s_any_bad[TP_BAD];
  __shared__ uint32_t s_tmem;
  const uint32_t base = (smem_u32(tp_smem) + 1023u) & ~1023u;
  uint8_t* generic = tp_smem + (base - smem_u32(tp_smem));
  int* s_bad = reinterpret_cast<int*>(generic + C::OFF_BAD);  // [item][NaN, +inf, -inf][element]: first key that has it
  Work* s_work = reinterpret_cast<Work*>(generic + C::OFF_WORK);
  int nb = 0;
  auto take = [&](int n) { const uint32_t b = base + C::OFF_BAR + 8u * nb; nb += n; return b; };
  const uint32_t q_full = take(1), q_empty = take(1), k_full = take(2), k_empty = take(2), v_full = take(2), v_clean = take(2),
                 v_empty = take(2), s_full = take(2), p_full = take(4), o_done = take(2), mma_done = take(2), w_full = take(TP_WORK),
                 w_empty = take(TP_WORK);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    s_abort = 0;
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int i = 0; i < 2; ++i) {
      for (const uint32_t b : {k_full, v_full, v_clean, s_full, o_done, mma_done}) mbar_init(b + 8u * i, 1);
      for (const uint32_t b : {k_empty, v_empty}) mbar_init(b + 8u * i, 2);                    // both issuers
      for (const uint32_t b : {p_full, p_full + 16u}) mbar_init(b + 8u * i, 4);                // one arrival per warp
    }
    for (int i = 0; i < TP_WORK; ++i) {
      mbar_init(w_full + 8u * i, 1);
      mbar_init(w_empty + 8u * i, 11);  // all warps but the list's own
    }
    fence_mbar_init();
  }
  if (warp == TP_WARP_MMA) {
    tmem_alloc(smem_u32(&s_tmem), 512);
    tmem_relinquish();
  }
  grid_dep_wait();
  grid_dep_launch();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  volatile int* abort_flag = &s_abort;
  auto wait = [&](uint32_t bar, uint32_t n) { return mbar_wait_warp(bar, n & 1u, abort_flag, a.status); };  // for its phase n
  // item i of this CTA; false: there is none
  auto next_work = [&](uint32_t i, Work& w) {
    if (!wait(w_full + 8u * (i % TP_WORK), i / TP_WORK)) return false;
    w = s_work[i % TP_WORK];
    return w.toks >= 0;
  };
  auto done_work = [&](uint32_t i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(w_empty + 8u * (i % TP_WORK));
  };
  const int per = a.tokens / 2, G = a.heads / a.kv_heads;

  // registers: 384 x 168 at launch = 128 x 88 + 256 x 208
  if (warp >= TP_WARP_MMA) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == TP_WARP_LOAD) {
      uint32_t loads = 0, tiles = 0;
      const uint32_t q_bytes = static_cast<uint32_t>(per * a.group) * HD * 2;
      ItemWalk walk(a, lane);
      const float cut = walk.cut(a, TP_KEYS);
      if (a.splits > 1 && blockIdx.x == 0 && lane == 0) a.partial[HD + 2] = cut;
      bool ok = true;
      auto publish = [&](uint32_t i, Work& w) {
        const Item it = walk.find(a, lane, TP_KEYS, cut, item_of(i));
        if (it.some) w = work_of(a, it, cut);
        else w.toks = -1;
        if (!wait(w_empty + 8u * (i % TP_WORK), i / TP_WORK + 1)) return false;
        if (lane == 0) {
          s_work[i % TP_WORK] = w;
          mbar_arrive(w_full + 8u * (i % TP_WORK));
        }
        __syncwarp();
        return true;
      };
      Work w, after;
      ok = publish(0, w);
      for (uint32_t i = 0; ok && w.toks >= 0; ++i, w = after) {
        const int n = w.tiles();
        if (n == 0) {
          ok = publish(i + 1, after);
          continue;
        }
        if (!(ok = wait(q_empty, loads + 1))) break;
        ++loads;
        if (elect_one()) {
          const int both = w.n1 > 0 ? 2 : 1;
          mbar_expect_tx(q_full, both * q_bytes);
          for (int g = 0; g < both; ++g)
            for (int s = 0; s < C::SUBS; ++s)
              tma_load_3d(base + g * C::TILE + s * TP_SUB, &tm_q, 64 * s, w.kvh * G + w.h0, w.q0 + g * per, q_full);
        }
        __syncwarp();
        for (int j = 0; j < n; ++j) {
          const uint32_t st = tiles & 1u, ph = tiles >> 1;
          const int row = w.k0 + w.begin + j * TP_KEYS;
          if (!(ok = wait(k_empty + 8u * st, ph + 1))) break;
          if (elect_one()) {
            mbar_expect_tx(k_full + 8u * st, C::TILE);
            for (int s = 0; s < C::SUBS; ++s)
              tma_load_3d(base + C::OFF_K + st * C::TILE + s * TP_SUB, &tm_k, 64 * s, w.kvh, row, k_full + 8u * st);
          }
          __syncwarp();
          if (!(ok = wait(v_empty + 8u * st, ph + 1))) {  // V of this tile is not loaded: nobody waits for it any more
            if (elect_one()) mbar_drain(k_full + 8u * st, ph & 1u, a.status);
            __syncwarp();
            break;
          }
          if (elect_one()) {
            mbar_expect_tx(v_full + 8u * st, C::TILE);
            for (int s = 0; s < C::SUBS; ++s)
              tma_load_3d(base + C::OFF_V + st * C::TILE + s * TP_SUB, &tm_v, 64 * s, w.kvh, row, v_full + 8u * st);
          }
          __syncwarp();
          ++tiles;
          if (j == min(n, 2) - 1 && !(ok = publish(i + 1, after))) break;  // while both places are full
        }
      }
      // do not leave while copies may still land in this CTA's shared memory
      if (elect_one()) {
        if (loads > 0) mbar_drain(q_full, (loads - 1) & 1u, a.status);
        for (uint32_t i = tiles > 2 ? tiles - 2 : 0; i < tiles; ++i) {
          mbar_drain(k_full + 8u * (i & 1u), (i >> 1) & 1u, a.status);
          mbar_drain(v_full + 8u * (i & 1u), (i >> 1) & 1u, a.status);
        }
      }
      __syncwarp();
    } else if (warp != TP_WARP_CLEAN) {
      const int g = warp - TP_WARP_MMA;
      constexpr uint32_t format = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
      const uint32_t idesc_s = (1u << 4) | format | (TP_KEYS / 8u) << 17 | (TP_ROWS / 16u) << 24 | (a.scale < 0.f ? 1u << 13 : 0u);  // bit 13: -Q
      constexpr uint32_t idesc_o = (1u << 4) | format | 1u << 16 | (HD / 8u) << 17 | (TP_ROWS / 16u) << 24;  // B is MN-major
      uint32_t loads = 0, tiles = 0, given = 0;  // items with keys; their tiles of keys; tiles of P taken
      bool ok = true;
      auto scores = [&](uint32_t st) {
        if (elect_one()) {
          const uint64_t q = smem_desc_sw128(base + g * C::TILE), k = smem_desc_sw128(base + C::OFF_K + st * C::TILE);
#pragma unroll
          for (int s = 0; s < HD / 16; ++s) {
            const uint64_t step = (s / 4) * (TP_SUB >> 4) + (s % 4) * 2;
            mma_ss(tmem + g * TP_KEYS, q + step, k + step, idesc_s, s > 0);
          }
          tc_commit(s_full + 8u * g);
        }
        __syncwarp();
      };
      // half of a tile's keys
      auto values = [&](uint32_t st, int part, bool first) {
        if (elect_one()) {
          const uint64_t v = smem_desc_v(base + C::OFF_V + st * C::TILE);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int s = part * 4 + i;
            mma_ts(tmem + 2 * TP_KEYS + g * HD, tmem + g * TP_KEYS + s * 8, v + s * (2048 >> 4), idesc_o, !first || part > 0 || i > 0);
          }
          if (part == 1) tc_commit(o_done + 8u * g);
        }
        __syncwarp();
      };
      Work w;
      for (uint32_t i = 0; ok && (ok = next_work(i, w)); ++i) {
        const int n = w.tiles(), own = w.tiles_of(g);
        done_work(i);
        if (n == 0) continue;
        if (!(ok = wait(q_full, loads) && wait(k_full + 8u * (tiles & 1u), tiles >> 1))) break;
        ++loads;
        tc_fence_after();
        if (own > 0) scores(tiles & 1u);
        if (elect_one()) {
          tc_commit(k_empty + 8u * (tiles & 1u));
          if (n == 1) tc_commit(q_empty);
        }
        __syncwarp();
        // both issuers wait for every tile, so that neither gives one back twice
        for (int j = 0; j < n; ++j, ++tiles) {
          const uint32_t st = tiles & 1u, next = (tiles + 1) & 1u;
          if (!(ok = wait(v_full + 8u * st, tiles >> 1) && wait(v_clean + 8u * st, tiles >> 1))) break;
          if (j < own) {
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              if (!(ok = wait(p_full + 16u * part + 8u * g, given))) break;
              tc_fence_after();
              values(st, part, j == 0);
            }
            if (!ok) break;
            ++given;
          }
          if (j + 1 < n) {
            if (!(ok = wait(k_full + 8u * next, (tiles + 1) >> 1))) break;
            tc_fence_after();
            if (j + 1 < own) scores(next);
          }
          if (elect_one()) {
            tc_commit(v_empty + 8u * st);
            if (j + 1 < n) tc_commit(k_empty + 8u * next);
            if (j + 2 == n) tc_commit(q_empty);
          }
          __syncwarp();
        }
      }
      // after a wait that ran out nobody else waits for the last MMAs
      if (elect_one()) tc_commit(mma_done + 8u * g);
      __syncwarp();
      mbar_drain(mma_done + 8u * g, 0, a.status);
    } else {
      constexpr uint32_t INF = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
      uint32_t loads = 0, tiles = 0;
      bool ok = true;
      Work w;
      for (uint32_t i = 0; ok && (ok = next_work(i, w)); ++i) {
        const int n = w.tiles();
        done_work(i);
        if (n == 0) continue;
        int* bad = s_bad + (loads % TP_BAD) * 3 * HD;
        bool fresh = true;
        for (int j = 0; j < n; ++j, ++tiles) {
          const uint32_t st = tiles & 1u;
          if (!(ok = wait(v_full + 8u * st, tiles >> 1))) break;
          const int first = w.begin + j * TP_KEYS;
          if (first + TP_KEYS > w.tok0 + w.shift + 1) {
            if (fresh) {
              for (int e = lane; e < 3 * HD; e += 32) bad[e] = 0x7fffffff;
              if (lane == 0) s_any_bad[loads % TP_BAD] = 0;
              fresh = false;
              __syncwarp();
            }
            const int have = min(TP_KEYS, w.end - first);
            const uint32_t tile = base + C::OFF_V + st * C::TILE;
            uint32_t top = 0;
            for (int s = 0; s < C::SUBS; ++s) {
              const int full = have * 8;  // 16-byte pieces of the rows there are
#pragma unroll 8
              for (int e = lane; e < full; e += 32) {
                uint32_t x[4];
                lds128(tile + s * TP_SUB + e * 16, x);
#pragma unroll
                for (int k = 0; k < 4; ++k) top = __vmaxu2(top, x[k] & 0x7fff7fffu);
              }
              const uint32_t zero[4] = {0u, 0u, 0u, 0u};
              for (int e = full + lane; e < TP_KEYS * 8; e += 32) sts128(tile + s * TP_SUB + e * 16, zero);
            }
            if (__any_sync(0xffffffffu, (top & 0xffffu) >= INF || (top >> 16) >= INF)) {
              uint16_t* v = reinterpret_cast<uint16_t*>(generic + C::OFF_V + st * C::TILE);
              for (int e = lane; e < have * HD; e += 32) {
                const int row = e / HD, d = e % HD;
                uint16_t* at = v + (d / 64) * (TP_SUB / 2) + row * 64 + ((d % 64 / 8) ^ (row & 7)) * 8 + d % 8;
                const uint32_t x = *at, mag = x & 0x7fffu;
                if (mag < INF) continue;
                atomicMin(bad + (mag > INF ? 0 : x & 0x8000u ? 2 : 1) * HD + d, first + row);
                *at = 0;
              }
              if (lane == 0) s_any_bad[loads % TP_BAD] = 1;
            }
            fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(v_clean + 8u * st);
        }
        ++loads;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int g = warp >> 2, row = (warp & 3) * 32 + lane;  // tile; row of it and lane of tensor memory
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16, s_at = tmem + lanes + g * TP_KEYS, o_at = tmem + lanes + 2 * TP_KEYS + g * HD;
    // (never zero: an unseen score is -infinity times it)
    const float by = fmaxf(CAP ? fabsf(a.scale) / a.softcap : fabsf(a.scale) * LOG2E, 1e-37f), cap2 = a.softcap * LOG2E;
    // c log2(e) tanh(S by) as a polynomial in S, where its coefficients are within 32 bits: with the
    // scale of a head of 64 or 128 for caps from 1e-3 to 7e4.  It is off by a part of the score, so that
    // the cap's size does not matter.
    const float by3 = by * by * by, poly[4] = {TANH[0] * cap2 * by, TANH[1] * cap2 * by3, TANH[2] * cap2 * by3 * (by * by), TANH[3] * cap2 * by3 * (by3 * by)};
    const bool usual = by > 1e-6f && by < 1e4f && cap2 > 1e-3f && poly[3] < -1e-38f;
    // Else c - 2 c / (exp(2 z) + 1), which is off by 2^-22 of the cap: for caps above CAP_FAST tanhf instead.
    const bool fast = a.softcap <= CAP_FAST;
    auto token_of = [&](int r) { return static_cast<int>((static_cast<uint32_t>(r) * a.inv_group) >> 16); };  // r / group
    const int mine = g * per + token_of(row);
    uint32_t loads = 0, tiles = 0;  // items with keys; S tiles taken
    bool ok = true;
    Work w;
    for (uint32_t i = 0; ok && (ok = next_work(i, w)); ++i) {
      const int seen = w.tok0 + mine + w.shift + 1;        // keys that this row sees
      const int all_see = w.tok0 + g * per + w.shift + 1;  // that all rows of the tile see
      const int begin = w.begin, own = w.tiles_of(g);
      const bool live = mine - g * per < per && mine < w.toks;  // rows behind the tokens hold anything: no vote is theirs
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < own; ++j, ++tiles) {
        if (!(ok = wait(s_full + 8u * g, tiles))) break;
        tc_fence_after();
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_at + 32 * c, v[c]);
        tmem_wait_ld();
        const int first = begin + j * TP_KEYS;
        const bool masked = first + TP_KEYS > all_see;

        const int some = masked ? seen - first : TP_KEYS;  // of the tile's keys, how many the row sees
        float top[4], up;
        bool small = true;  // softcap: the polynomial holds for all scores of the warp's rows
        if constexpr (CAP) {
          // the polynomial's range is looked at with zeros for unseen scores; then they become so
          // large that it falls (odd, its last coefficient negative) and their weights are zero
          auto unseen = [&](uint32_t value) {
            if (masked) {
#pragma unroll
              for (int c = 0; c < 4; ++c)
                if (__any_sync(0xffffffffu, 32 * c + 32 > some)) {
#pragma unroll
                  for (int e = 0; e < 32; ++e)
                    if (32 * c + e >= some) v[c][e] = value;
                }
            }
          };
          unseen(0u);
          float low[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            low[c] = top[c] = __uint_as_float(v[c][0]);
#pragma unroll
            for (int e = 1; e < 31; e += 2) {
              low[c] = min3(low[c], __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
              top[c] = max3(top[c], __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
            }
            low[c] = min3(low[c], __uint_as_float(v[c][31]), low[c]);
            top[c] = max3(top[c], __uint_as_float(v[c][31]), top[c]);
          }
          up = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * by;
          small = usual && __all_sync(0xffffffffu, !live || (up <= 0.5f && min3(min3(low[0], low[1], low[2]), low[3], low[3]) * by >= -0.5f));
          if (masked) {  // the zeros are no scores
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (__any_sync(0xffffffffu, 32 * c + 32 > some)) {
                top[c] = -INFINITY;
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (32 * c + e < some) top[c] = max3(top[c], __uint_as_float(v[c][e]), top[c]);
              }
            up = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * by;
            unseen(__float_as_uint(100.f / by));
          }
          up = up == -INFINITY ? up : cap2 * tanhf(up);
        } else {
          if (masked) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (__any_sync(0xffffffffu, 32 * c + 32 > some)) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (32 * c + e >= some) v[c][e] = 0xff800000u;
              }
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            top[c] = max3(__uint_as_float(v[c][0]), __uint_as_float(v[c][1]), __uint_as_float(v[c][0]));
#pragma unroll
            for (int e = 2; e < 32; e += 2) top[c] = max3(top[c], __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
          }
          up = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * by;
        }
        up = live ? up : 0.f;
        // The maximum is taken where it has grown by more than P_SLACK: what the weights are relative
        // to from here on.  An infinite score or none makes it NaN: for the whole row.
        if (j == 0) {
          m = up < INFINITY ? up : __int_as_float(0x7fffffff);
        } else if (__any_sync(0xffffffffu, !(up <= m + P_SLACK))) {
          const float m_new = up < INFINITY ? fmaxf(m, up) : __int_as_float(0x7fffffff);
          const float alpha = m_new == -INFINITY ? 1.f : ex2(m - m_new);
          m = m_new;
          l *= alpha;
          if (!(ok = wait(o_done + 8u * g, tiles - 1))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(o_at + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16(o_at + 16 * c, o);
          }
        }
        const float from = (m == -INFINITY ? 0.f : m) - P_TOP;
        const uint64_t by2 = pair(by, by), less = pair(-from, -from);
        uint64_t sum[2] = {0ull, 0ull};
        // P of 32 keys at a time; after 64 the first half of the product can start
        auto give = [&](int c, const uint32_t (&p)[16]) {
          tmem_st16(s_at + 16 * c, p);
          if (c % 2) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 16u * (c / 2) + 8u * g);
          }
        };
        if (!CAP || small) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const uint64_t s2 = pair(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1]));
              float x, y;
              if constexpr (CAP) {
                const uint64_t u = mul2(s2, s2);
                const uint64_t t = fma2(u, fma2(u, fma2(u, pair(poly[3], poly[3]), pair(poly[2], poly[2])), pair(poly[1], poly[1])), pair(poly[0], poly[0]));
                unpair(fma2(s2, t, less), x, y);
              } else {
                unpair(fma2(s2, by2, less), x, y);
              }
              x = ex2(x);
              y = ex2(y);
              sum[e % 2] = add2(sum[e % 2], pair(x, y));
              p[e] = pack16<T>(x, y);
            }
            give(c, p);
          }
        } else if constexpr (CAP) {  // S once more from tensor memory (P takes the part that is read)
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t z[32], p[16];
            tmem_ld32(s_at + 32 * c, z);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float x[2];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float t = __uint_as_float(z[2 * e + k]) * by;
                const float f = fast ? fmaf(-2.f * cap2, rcp(ex2(t * (2.f * LOG2E)) + 1.f), cap2 - from) : fmaf(cap2, tanhf(t), -from);
                x[k] = 32 * c + 2 * e + k < some ? ex2(f) : 0.f;
              }
              sum[e % 2] = add2(sum[e % 2], pair(x[0], x[1]));
              p[e] = pack16<T>(x[0], x[1]);
            }
            give(c, p);
          }
        }
        {
          float x, y;
          unpair(add2(sum[0], sum[1]), x, y);
          l += x + y;
        }
      }
      if (!ok) break;
      if (own > 0 && !(ok = wait(o_done + 8u * g, tiles - 1))) break;
      tc_fence_after();
      w = s_work[i % TP_WORK];
      // the last tile of keys is one that was looked at: before it the notes may be older ones
      const bool any_bad = own > 0 && w.begin + own * TP_KEYS > w.tok0 + w.shift + 1 && s_any_bad[loads % TP_BAD] != 0;
      const int* bad = s_bad + (loads % TP_BAD) * 3 * HD;
      const bool parts = w.chunks > 1;
      const float f = parts ? 1.f : l == 0.f ? 0.f : rcp(l);
      const int h = row - (mine - g * per) * a.group;
      const bool stored = live && h < w.hs;
      const int64_t at = (static_cast<int64_t>(w.q0) + mine) * a.heads + w.kvh * G + w.h0 + h;
      float* part = a.partial + (at * a.splits + w.chunk) * (HD + 4);
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        if (own > 0) {
          tmem_ld32(o_at + 32 * c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (any_bad) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int d = 32 * c + e;
            float x = __uint_as_float(o[e]);
            if (bad[d] < seen) x = __int_as_float(0x7fffffff);
            if (bad[HD + d] < seen) x += INFINITY;
            if (bad[2 * HD + d] < seen) x -= INFINITY;
            o[e] = __float_as_uint(x);
          }
        }
        if (stored) {  // whole sectors of 32 bytes
          if (parts) {  // (its rows are 16 bytes from those)
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(part + 32 * c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          } else if (a.out_dtype == B200MOE_DT_F32) {
            float* to = static_cast<float*>(a.out) + at * HD + 32 * c;
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              const uint32_t y[8] = {o[e], o[e + 1], o[e + 2], o[e + 3], o[e + 4], o[e + 5], o[e + 6], o[e + 7]};
              store_sector(to + e, y);
            }
          } else {
            uint16_t* to = static_cast<uint16_t*>(a.out) + at * HD + 32 * c;
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              uint32_t y[8];
              auto pack = [&](auto type) {
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = pack16<decltype(type)>(__uint_as_float(o[e + 2 * k]), __uint_as_float(o[e + 2 * k + 1]));
              };
              if (a.out_dtype == B200MOE_DT_F16) pack(__half());
              else pack(__nv_bfloat16());
              store_sector(to + e, y);
            }
          }
        }
        __syncwarp();  // the next load of tensor memory is the whole warp's
      }
      if (parts && stored) *reinterpret_cast<float2*>(part + HD) = make_float2(m, l);
      if (w.tiles() > 0) ++loads;
      done_work(i);
    }
  }
  zero_rest(a, HD, TP_THREADS);
  // everyone is done with tensor memory before it is freed
  tc_fence_before();
  __syncthreads();
  if (warp == TP_WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the rows whose keys were split: a warp per row and head.
template <int HD>
__global__ void __launch_bounds__(256) prompt_merge_kernel(const PromptArgs a) {
  constexpr int N = HD / 32;
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t row = at / a.heads;
  if (row >= a.q_rows) return;
  const float cut = a.partial[HD + 2];
  int chunks = 0;
  for (int b0 = 0; b0 < a.bs; b0 += 32) {
    const int b = b0 + lane;
    const Span qs = b < a.bs ? span_of(a.cu_q, b, a.q_rows, nullptr) : Span{0, 0};
    const bool here = row >= qs.begin && row < qs.begin + qs.len;
    const unsigned who = __ballot_sync(0xffffffffu, here);
    if (who == 0) continue;
    const int m = here ? span_of(a.cu_k != nullptr ? a.cu_k : a.cu_q, b, a.k_rows, nullptr).len : 0;
    const int own = here ? ItemWalk::chunks(a, qs.len, m, static_cast<int>(row - qs.begin) / a.tokens, TP_KEYS, cut) : 0;
    chunks = __shfl_sync(0xffffffffu, own, __ffs(who) - 1);
    break;
  }
  if (chunks <= 1) return;  // the output is there
  const float* part = a.partial + at * a.splits * (HD + 4);
  float top = -INFINITY, den = 0.f, acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  for (int c = 0; c < chunks; ++c) top = fmaxf(top, part[c * (HD + 4) + HD]);
  for (int c = 0; c < chunks; ++c) {
    float v[N];
    load_elems(part + c * (HD + 4) + lane * N, v);
    const float2 ml = *reinterpret_cast<const float2*>(part + c * (HD + 4) + HD);
    const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
    den = fmaf(ml.y, f, den);
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += ml.x == -INFINITY ? 0.f : v[j] * f;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = den == 0.f ? 0.f : acc[j] / den;
  store_as(a.out, a.out_dtype, static_cast<size_t>(at) * HD + lane * N, acc);
}

template <typename T, int HD, bool CAP>
int launch_prompt_tc(const PromptArgs& a, cudaStream_t st) {
  CUtensorMap q, k, v;
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  if (const int rc = make_tmap_heads(&q, a.q, bf16, a.q_rows, a.heads, HD, a.q_stride, a.tokens / 2, a.group)) return rc;
  if (const int rc = make_tmap_heads(&k, a.k, bf16, a.k_rows, a.kv_heads, HD, a.k_stride, TP_KEYS, 1)) return rc;
  if (const int rc = make_tmap_heads(&v, a.v, bf16, a.k_rows, a.kv_heads, HD, a.v_stride, TP_KEYS, 1)) return rc;
  auto kern = prompt_attend_tc_kernel<T, HD, CAP>;
  static bool configured[16] = {};
  int dev = 0;
  B200_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev >= 16 || !configured[dev]) {
    B200_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TpCfg<HD>::SMEM));
    if (dev < 16) configured[dev] = true;
  }
  const int64_t items = (a.q_rows / a.tokens + a.bs) * a.kv_heads * a.parts * a.splits + 1, sms = sm_count();
  B200_CHECK_CUDA(launch_dependent(kern, dim3(static_cast<unsigned>(items < sms ? items : sms)), dim3(TP_THREADS), TpCfg<HD>::SMEM, st,
                                   q, k, v, a));
  if (a.splits > 1)
    B200_CHECK_CUDA(launch_dependent(prompt_merge_kernel<HD>, dim3(static_cast<unsigned>((a.q_rows * a.heads + 7) / 8)), dim3(256), 0, st, a));
  return B200MOE_OK;
}
template <typename T>
int launch_prompt_tc_hd(const PromptArgs& a, int hd, cudaStream_t st) {
  if (a.softcap > 0.f) return hd == 64 ? launch_prompt_tc<T, 64, true>(a, st) : launch_prompt_tc<T, 128, true>(a, st);
  return hd == 64 ? launch_prompt_tc<T, 64, false>(a, st) : launch_prompt_tc<T, 128, false>(a, st);
}

// The shape of a call's items on the tensor cores.  Where there are fewer items than SMs (few
// rows, long keys) the keys of each are split: into as many parts as make the last SM finish
// first, in units of a tile of keys (1.5 us), with two for an item's start and end and two for
// the merge.  The lengths are on the device: here all sequences are taken to be as long as the mean.
// Of 2 to 32 sequences the kernel then cuts longer ones into more parts, up to three times as many,
// and no more in all than the rule's rounds of the SMs.  Where the mean asks for no parts, long keys
// (a quarter of the rows new at most, 8 tiles) get up to four, in the best of one to three rounds.
// 4 x 60 tokens behind 12000, 32 heads (32 items): 4 parts 63 us, 5 95, 6 90, 9 74, 13 87; 16 tokens
// behind 30000 (8 items): 16 parts 40 us, 13 44, 9 54, 4 99; unsplit 208 for 4 x 60 behind up to 16000.
// As many parts for each sequence, or by its length: 30 tokens behind 30000 and three times 1000
// 103 and 50 us; 8 x 16 behind 100 to 8000 60 and 34; 12 x 30 behind 500 to 11500 103 and 91; 4 x 60
// behind 10000 to 16000 73 and 68, all behind 12000 63 and 65.  One part, or up to four: 16 x 3 behind 1000 to 7000
// 89 and 75, one of them behind 16000, 4000 else, 192 and 88, all behind 4000 56 and 60.
struct PromptPlan { int group, parts, tokens, splits, units; bool uneven; float cut; };
constexpr int TP_MAX_SPLITS = 16;
PromptPlan plan_prompt(int64_t q_rows, int64_t k_rows, int bs, int heads, int kv_heads) {
  PromptPlan p{};
  const int G = heads / kv_heads;
  p.group = G < TP_ROWS ? G : TP_ROWS;
  p.parts = (G + p.group - 1) / p.group;
  p.tokens = 2 * (TP_ROWS / p.group);
  p.splits = p.units = 1;
  const int64_t n = bs > 0 ? (q_rows + bs - 1) / bs : 0, m = bs > 0 ? (k_rows + bs - 1) / bs : 0;
  const int64_t items = bs * ((n + p.tokens - 1) / p.tokens) * kv_heads * p.parts, tiles = (m + TP_KEYS - 1) / TP_KEYS;
  if (items >= sm_count()) return p;
  int64_t least = tiles + 2;
  for (int s = 2; s <= TP_MAX_SPLITS && s <= tiles; ++s) {
    const int64_t time = (items * s + sm_count() - 1) / sm_count() * ((tiles + s - 1) / s + 2) + 2;
    if (time < least) {
      least = time;
      p.splits = s;
    }
  }
  p.cut = static_cast<float>(p.splits) / static_cast<float>(std::max<int64_t>(tiles, 1));
  p.units = static_cast<int>((items * p.splits + sm_count() - 1) / sm_count() * sm_count() / (kv_heads * p.parts));
  if (bs > 1 && bs <= 32) {
    p.uneven = p.splits == 1 && tiles >= 8 && k_rows >= 4 * q_rows;
    p.splits = p.uneven ? 4 : p.splits > 1 ? std::min(TP_MAX_SPLITS, 3 * p.splits) : 1;
  }
  return p;
}

// ------------------------------------------------------------------ masks
// Whether masks are causal: one look at each number, a warp a row.  The number of tokens n is that of
// the rows that see their own position, found by 256 samples and a look between two of them: in a
// causal mask these are the first n.  Rows up to n then have to be zero up to their own position and
// masked behind it, others masked from that of row n on, so that no other mask passes, whatever n came out.
// Bound by memory: one mask of 8192 x 8192, 16 bits, 46 us; 4 of 2048 x 2048 20, with the call's work on the host.
constexpr int MASK_THREADS = 256;
struct MaskArgs {
  const void* mask;
  int64_t batch_stride, row_stride;
  int masks, rows, columns;
  const int32_t* new_lens;
  int bs, per;
  bool wide;  // rows are 16 bytes apart, and so aligned
  int32_t* status;
};
__device__ __forceinline__ float number(float x) { return x; }
__device__ __forceinline__ float number(__half x) { return __half2float(x); }
__device__ __forceinline__ float number(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__global__ void __launch_bounds__(MASK_THREADS) causal_mask_kernel(const MaskArgs a) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  grid_dep_wait();
  grid_dep_launch();
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, first = a.columns - a.rows;
  auto masked = [](float x) { return x <= -5000.f; };
  bool bad = false;
  for (int b = blockIdx.y; b < a.masks; b += gridDim.y) {
    const T* mask = static_cast<const T*>(a.mask) + b * a.batch_stride;
    auto sees_itself = [&](int64_t i) { return i < a.rows && !masked(number(mask[i * a.row_stride + first + i])); };
    const int step = (a.rows - 1) / MASK_THREADS + 1;
    const int samples = __syncthreads_count(sees_itself(static_cast<int64_t>(t) * step));
    int n = 0;
    if (samples > 0) {
      n = (samples - 1) * step + 1;
      for (int i = 1; i < step; i += MASK_THREADS)
        n += __syncthreads_count(i + t < step && sees_itself(static_cast<int64_t>(samples - 1) * step + i + t));
    }
    if (a.new_lens != nullptr) {
      if (a.per > 0) n = max(n, min(a.new_lens[b / a.per], a.rows));
      else
        for (int i = 0; i < a.bs; ++i) n = max(n, min(a.new_lens[i], a.rows));
    }
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * (MASK_THREADS / 32) + warp; i < a.rows; i += static_cast<int64_t>(gridDim.x) * (MASK_THREADS / 32)) {
      const T* row = mask + i * a.row_stride;
      const bool token = i < n;
      const int seen = first + (token ? static_cast<int>(i) + 1 : n);  // columns before it: zero, or (padding) anything
      auto look = [&](int j, float x) { bad |= j >= seen ? !masked(x) : token && x != 0.f; };
      const int from = token ? 0 : seen / E * E, wide = a.wide ? a.columns / E * E : from;
      for (int j = from + lane * E; j < wide; j += 32 * E) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + j);
        const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int e = 0; e < E; ++e) look(j + e, number(x[e]));
      }
      for (int j = max(from, wide) + lane; j < a.columns; j += 32) look(j, number(row[j]));
    }
  }
  if (bad) atomicOr(a.status, DEV_ERR_BOUNDS);
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" {

size_t b200moe_prompt_attend_scratch_bytes(int dtype, int32_t bs, int64_t q_rows, int64_t k_rows, int32_t heads,
                                           int32_t kv_heads, int32_t head_dim) {
  if (dtype == B200MOE_DT_F32 || bs <= 0 || q_rows <= 0 || k_rows <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 ||
      heads % kv_heads != 0)
    return 0;
  const int splits = plan_prompt(q_rows, k_rows, bs, heads, kv_heads).splits;
  return splits == 1 ? 0 : static_cast<size_t>(q_rows) * heads * splits * (head_dim + 4) * sizeof(float);
}

int b200moe_prompt_attend(const void* q, const void* k, const void* v, int dtype, int64_t q_stride, int64_t k_stride,
                          int64_t v_stride, const int32_t* cu_q, const int32_t* cu_k, int32_t bs, int64_t q_rows,
                          int64_t k_rows, int32_t heads, int32_t kv_heads, int32_t head_dim, float scale, float softcap,
                          void* out, int out_dtype, void* scratch, size_t scratch_bytes, void* stream) {
  const char* who = "prompt_attend";
  B200_REQUIRE(bs >= 0 && q_rows >= 0 && k_rows >= 0 && heads >= 1 && kv_heads >= 1, "%s: bad sizes", who);
  B200_REQUIRE(q_rows < 0x7fffffff && k_rows < 0x7fffffff, "%s: more than 2^31 rows", who);
  B200_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim %d (64 and 128 are built)", who, head_dim);
  B200_REQUIRE(heads % kv_heads == 0, "%s: heads (%d) must be a multiple of the kv heads (%d)", who, heads, kv_heads);
  B200_REQUIRE(heads <= 65536, "%s: heads %d", who, heads);
  B200_REQUIRE(dtype_ok(dtype) && dtype_ok(out_dtype), "%s: unknown dtype", who);
  B200_REQUIRE(std::isfinite(softcap), "%s: softcap must be finite", who);
  if (q_rows == 0) return B200MOE_OK;
  B200_REQUIRE(q && out && (bs == 0 || cu_q) && (k_rows == 0 || (k && v)), "%s: NULL buffer", who);
  const int64_t per16 = 16 / static_cast<int64_t>(dt_bytes(dtype));
  B200_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && q_stride % per16 == 0 &&
                   k_stride % per16 == 0 && v_stride % per16 == 0,
               "%s: buffers and row strides must be multiples of 16 bytes", who);
  B200_REQUIRE((reinterpret_cast<uintptr_t>(out) & 31) == 0, "%s: out must be 32-byte aligned", who);
  B200_REQUIRE(q_stride >= static_cast<int64_t>(heads) * head_dim && k_stride >= static_cast<int64_t>(kv_heads) * head_dim &&
                   v_stride >= static_cast<int64_t>(kv_heads) * head_dim,
               "%s: a row stride is shorter than the row", who);
  const size_t need = b200moe_prompt_attend_scratch_bytes(dtype, bs, q_rows, k_rows, heads, kv_heads, head_dim);
  if (scratch_bytes < need) {
    set_error("%s: scratch needs %zu bytes, got %zu", who, need, scratch_bytes);
    return B200MOE_ERR_WORKSPACE;
  }
  B200_REQUIRE(need == 0 || (scratch != nullptr && aligned16(scratch)), "%s: scratch must be given and 16-byte aligned", who);
  PromptArgs a{};
  a.partial = static_cast<float*>(scratch);
  a.q = q; a.k = k; a.v = v; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.cu_q = cu_q; a.cu_k = cu_k; a.out = out; a.q_rows = q_rows; a.k_rows = k_rows; a.out_dtype = out_dtype;
  a.bs = bs; a.heads = heads; a.kv_heads = kv_heads; a.scale = scale; a.softcap = usable_softcap(softcap);
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200MOE_DT_F32) return head_dim == 64 ? launch_prompt<64>(a, st) : launch_prompt<128>(a, st);
  if (k_rows == 0) {
    B200_CHECK_CUDA(cudaMemsetAsync(out, 0, static_cast<size_t>(q_rows) * heads * head_dim * dt_bytes(out_dtype), st));
    return B200MOE_OK;
  }
  const PromptPlan p = plan_prompt(q_rows, k_rows, bs, heads, kv_heads);
  a.group = p.group; a.inv_group = (65536 + p.group - 1) / p.group; a.parts = p.parts; a.tokens = p.tokens; a.splits = p.splits;
  a.cut = p.cut; a.units = p.units; a.uneven = p.uneven;
  return dtype == B200MOE_DT_F16 ? launch_prompt_tc_hd<__half>(a, head_dim, st) : launch_prompt_tc_hd<__nv_bfloat16>(a, head_dim, st);
}

int b200moe_causal_mask_check(const void* mask, int dtype, int64_t batch_stride, int64_t row_stride, int32_t masks,
                              int32_t rows, int32_t columns, const int32_t* new_lens, int32_t bs, int32_t per_seq,
                              void* stream) {
  const char* who = "causal_mask_check";
  B200_REQUIRE(masks >= 0 && rows >= 0 && columns >= rows && bs >= 0 && per_seq >= 0 && batch_stride >= 0 && row_stride >= 0,
               "%s: bad sizes", who);
  B200_REQUIRE(dtype_ok(dtype), "%s: unknown dtype", who);
  B200_REQUIRE(new_lens == nullptr || per_seq == 0 || static_cast<int64_t>(bs) * per_seq == masks,
               "%s: %d masks for %d sequences of %d each", who, masks, bs, per_seq);
  if (masks == 0 || rows == 0) return B200MOE_OK;
  B200_REQUIRE(mask != nullptr, "%s: NULL buffer", who);
  const int64_t bytes = static_cast<int64_t>(dt_bytes(dtype));
  B200_REQUIRE(reinterpret_cast<uintptr_t>(mask) % bytes == 0, "%s: mask is not aligned to its numbers", who);
  MaskArgs a{mask, batch_stride, row_stride, masks, rows, columns, new_lens, bs, per_seq,
             aligned16(mask) && batch_stride * bytes % 16 == 0 && row_stride * bytes % 16 == 0, device_status_ptr()};
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  const unsigned y = static_cast<unsigned>(std::min(masks, 65535));
  const int64_t row_ctas = (static_cast<int64_t>(rows) + MASK_THREADS / 32 - 1) / (MASK_THREADS / 32), most = sm_count() * 8 / static_cast<int64_t>(y) + 1;
  const dim3 grid(static_cast<unsigned>(std::min(row_ctas, most)), y);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kern = dtype == B200MOE_DT_F32 ? causal_mask_kernel<float> : dtype == B200MOE_DT_F16 ? causal_mask_kernel<__half> : causal_mask_kernel<__nv_bfloat16>;
  B200_CHECK_CUDA(launch_dependent(kern, grid, dim3(MASK_THREADS), 0, st, a));
  return B200MOE_OK;
}

}  // extern "C"
