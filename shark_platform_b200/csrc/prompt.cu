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
// they have the most keys, and the short ones fill the end.  It is made by every warp on its
// own from the sequences' bounds on the device: the host does not know them.
#include "kv_attend.cuh"

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
  int tokens;             // of a tile
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
  int seq, tile, kvh, part;
  bool some;
};
// The list of items, walked by a whole warp with rising indices.
struct ItemWalk {
  int t;         // tiles with this place in their sequence are current
  long long before;  // items before them
  __device__ __forceinline__ static int tiles_of(const PromptArgs& a, int b) {
    return b < a.bs ? (span_of(a.cu_q, b, a.q_rows, nullptr).len + a.tokens - 1) / a.tokens : 0;
  }
  __device__ __forceinline__ ItemWalk(const PromptArgs& a, int lane) : t(0), before(0) {
    int most = 0;
    int32_t* status = blockIdx.x == 0 && threadIdx.x < 32 ? a.status : nullptr;
    for (int b = lane; b < a.bs; b += 32) {
      most = max(most, tiles_of(a, b));
      if (status != nullptr) {
        span_of(a.cu_q, b, a.q_rows, status);
        if (a.cu_k != nullptr) span_of(a.cu_k, b, a.k_rows, status);
      }
    }
    t = __reduce_max_sync(0xffffffffu, most) - 1;
  }
  __device__ __forceinline__ Item find(const PromptArgs& a, int lane, long long i) {
    const int each = a.kv_heads * a.parts;
    for (; t >= 0; --t) {
      long long at = before;
      for (int b0 = 0; b0 < a.bs; b0 += 32) {
        const unsigned has = __ballot_sync(0xffffffffu, tiles_of(a, b0 + lane) > t);
        const int n = __popc(has);
        if (i < at + static_cast<long long>(n) * each) {
          const int r = static_cast<int>(i - at), which = r / each, h = r - which * each;
          const int b = b0 + static_cast<int>(__fns(has, 0, which + 1));
          return {b, t, h / a.parts, h % a.parts, true};
        }
        at += static_cast<long long>(n) * each;
      }
      before = at;
    }
    return {0, 0, 0, 0, false};
  }
};

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

// ------------------------------------------------------------------ 32-bit products
// Tiles of 64 rows and 64 keys on the fp32 units: thread (ty, tx) of 16 x 16 has rows
// 4 ty .. + 3, keys tx + 16 j of the scores and elements 4 tx + 64 j .. + 3 of the output.
// Everything is fp32.
constexpr int SP_ROWS = 64, SP_KEYS = 64, SP_THREADS = 256;

template <typename T, int HD>
__device__ __forceinline__ void load_tile(float* to, int pitch, const T* from, int64_t stride, int rows, int have) {
  constexpr int C = HD / 8;
  for (int i = threadIdx.x; i < rows * C; i += SP_THREADS) {
    const int r = i / C, c = i % C;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r < have) {
      Raw8<T> raw;
      raw.load(from + r * stride + c * 8);
      raw.get(x);
    }
    store8(to + r * pitch + c * 8, x);
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(SP_THREADS, 2) prompt_attend_kernel(const PromptArgs a) {
  constexpr int PITCH = HD + 4, PP = SP_KEYS + 4, NO = HD / 64;
  extern __shared__ __align__(16) float sp_smem[];
  float *sq = sp_smem, *skv = sq + SP_ROWS * PITCH, *sp = skv + SP_KEYS * PITCH;
  grid_dep_wait();
  grid_dep_launch();
  const int t = threadIdx.x, lane = t & 31, ty = t >> 4, tx = t & 15;
  const T *q = static_cast<const T*>(a.q), *k = static_cast<const T*>(a.k), *v = static_cast<const T*>(a.v);
  const int G = a.heads / a.kv_heads;
  const float to_score = a.softcap > 0.f ? a.scale / a.softcap : a.scale * LOG2E, cap2 = a.softcap * LOG2E;
  ItemWalk walk(a, lane);
  for (long long i = blockIdx.x;; i += gridDim.x) {
    const Item it = walk.find(a, lane, i);
    if (!it.some) break;
    const Span qs = span_of(a.cu_q, it.seq, a.q_rows, nullptr), ks = span_of(a.cu_k != nullptr ? a.cu_k : a.cu_q, it.seq, a.k_rows, nullptr);
    const int tok0 = it.tile * a.tokens, toks = min(a.tokens, qs.len - tok0);
    const int h0 = it.part * a.group, hs = min(a.group, G - h0), rows = toks * hs;
    const int shift = ks.len - qs.len;  // row i sees keys up to i + shift
    const int keys = max(0, min(ks.len, tok0 + toks + shift));
    __syncthreads();  // the last item's tiles are read
    for (int j = t; j < SP_ROWS * (HD / 8); j += SP_THREADS) {
      const int r = j / (HD / 8), c = j % (HD / 8);
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (r < rows) {
        Raw8<T> raw;
        raw.load(q + (static_cast<int64_t>(qs.begin) + tok0 + r / hs) * a.q_stride +
                 static_cast<int64_t>(it.kvh * G + h0 + r % hs) * HD + c * 8);
        raw.get(x);
      }
      store8(sq + r * PITCH + c * 8, x);
    }
    int seen[4];  // keys that this thread's rows see
#pragma unroll
    for (int r = 0; r < 4; ++r) seen[r] = min(ks.len, tok0 + (4 * ty + r) / hs + shift + 1);
    float m[4], l[4], o[4][NO][4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int n = 0; n < NO; ++n) o[r][n][0] = o[r][n][1] = o[r][n][2] = o[r][n][3] = 0.f;
    }
    for (int k0 = 0; k0 < keys; k0 += SP_KEYS) {
      const int have = min(SP_KEYS, keys - k0);
      __syncthreads();
      load_tile<T, HD>(skv, PITCH, k + (static_cast<int64_t>(ks.begin) + k0) * a.k_stride + it.kvh * HD, a.k_stride, SP_KEYS, have);
      __syncthreads();
      float s[4][4] = {};
#pragma unroll 4
      for (int d = 0; d < HD; d += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const float4*>(sq + (4 * ty + r) * PITCH + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(skv + (tx + 16 * j) * PITCH + d);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[r][j] = fmaf(x[r].x, y[j].x, s[r][j]);
            s[r][j] = fmaf(x[r].y, y[j].y, s[r][j]);
            s[r][j] = fmaf(x[r].z, y[j].z, s[r][j]);
            s[r][j] = fmaf(x[r].w, y[j].w, s[r][j]);
          }
      }
      __syncthreads();  // K is read: V takes its place
      load_tile<T, HD>(skv, PITCH, v + (static_cast<int64_t>(ks.begin) + k0) * a.v_stride + it.kvh * HD, a.v_stride, SP_KEYS, have);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = s[r][j] * to_score;
          if (a.softcap > 0.f) x = cap2 * tanhf(x);
          s[r][j] = k0 + tx + 16 * j < seen[r] ? x : -INFINITY;
          top = fmaxf(top, s[r][j]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float m_new = fmaxf(m[r], top), base = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp2f(m[r] - base);
        m[r] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2f(s[r][j] - base);
          sum += p;
          sp[(4 * ty + r) * PP + tx + 16 * j] = p;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        l[r] = fmaf(l[r], alpha, sum);
#pragma unroll
        for (int n = 0; n < NO; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[r][n][e] *= alpha;
      }
      __syncthreads();
      // where not all rows see all keys, a weight of zero leaves infinities and NaN out
      const bool masked = k0 + SP_KEYS > tok0 + shift + 1;
      auto products = [&](auto some) {
#pragma unroll 2
        for (int j = 0; j < SP_KEYS; j += 4) {
          float4 p[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) p[r] = *reinterpret_cast<const float4*>(sp + (4 * ty + r) * PP + j);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
#pragma unroll
            for (int n = 0; n < NO; ++n) {
              const float4 y = *reinterpret_cast<const float4*>(skv + (j + jj) * PITCH + 4 * tx + 64 * n);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float w = jj == 0 ? p[r].x : jj == 1 ? p[r].y : jj == 2 ? p[r].z : p[r].w;
                if (decltype(some)::value && w == 0.f) continue;
                o[r][n][0] = fmaf(w, y.x, o[r][n][0]);
                o[r][n][1] = fmaf(w, y.y, o[r][n][1]);
                o[r][n][2] = fmaf(w, y.z, o[r][n][2]);
                o[r][n][3] = fmaf(w, y.w, o[r][n][3]);
              }
            }
        }
      };
      if (masked) products(std::true_type());
      else products(std::false_type());
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * ty + r;
      if (row >= rows) continue;
      const float f = l[r] == 0.f ? 0.f : 1.f / l[r];
      const size_t to = ((static_cast<size_t>(qs.begin) + tok0 + row / hs) * a.heads + it.kvh * G + h0 + row % hs) * HD + 4 * tx;
#pragma unroll
      for (int n = 0; n < NO; ++n) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = l[r] == 0.f ? 0.f : o[r][n][e] * f;
        store_as(a.out, a.out_dtype, to + 64 * n, y);
      }
    }
  }
  zero_rest(a, HD, SP_THREADS);
}

template <typename T, int HD>
int launch_prompt(PromptArgs& a, cudaStream_t st) {
  constexpr int SMEM = (2 * SP_ROWS * (HD + 4) + SP_ROWS * (SP_KEYS + 4)) * 4;
  const int G = a.heads / a.kv_heads;
  a.group = G < SP_ROWS ? G : SP_ROWS;
  a.parts = (G + a.group - 1) / a.group;
  a.tokens = SP_ROWS / a.group;
  auto kern = prompt_attend_kernel<T, HD>;
  B200_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
  const int64_t items = (a.q_rows / a.tokens + a.bs) * a.kv_heads * a.parts + 1, resident = 2ll * sm_count();
  B200_CHECK_CUDA(launch_dependent(kern, dim3(static_cast<unsigned>(items < resident ? items : resident)), dim3(SP_THREADS), SMEM,
                                   st, a));
  return B200MOE_OK;
}
template <typename T>
int launch_prompt_hd(PromptArgs& a, int hd, cudaStream_t st) {
  return hd == 64 ? launch_prompt<T, 64>(a, st) : launch_prompt<T, 128>(a, st);
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" {

int b200moe_prompt_attend(const void* q, const void* k, const void* v, int dtype, int64_t q_stride, int64_t k_stride,
                          int64_t v_stride, const int32_t* cu_q, const int32_t* cu_k, int32_t bs, int64_t q_rows,
                          int64_t k_rows, int32_t heads, int32_t kv_heads, int32_t head_dim, float scale, float softcap,
                          void* out, int out_dtype, void* stream) {
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
  B200_REQUIRE(q_stride >= static_cast<int64_t>(heads) * head_dim && k_stride >= static_cast<int64_t>(kv_heads) * head_dim &&
                   v_stride >= static_cast<int64_t>(kv_heads) * head_dim,
               "%s: a row stride is shorter than the row", who);
  PromptArgs a{};
  a.q = q; a.k = k; a.v = v; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.cu_q = cu_q; a.cu_k = cu_k; a.out = out; a.q_rows = q_rows; a.k_rows = k_rows; a.out_dtype = out_dtype;
  a.bs = bs; a.heads = heads; a.kv_heads = kv_heads; a.scale = scale; a.softcap = softcap > 0.f ? softcap : 0.f;
  a.status = device_status_ptr();
  if (a.status == nullptr) return B200MOE_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200MOE_DT_F32) return launch_prompt_hd<float>(a, head_dim, st);
  if (dtype == B200MOE_DT_F16) return launch_prompt_hd<__half>(a, head_dim, st);
  return launch_prompt_hd<__nv_bfloat16>(a, head_dim, st);
}

}  // extern "C"
