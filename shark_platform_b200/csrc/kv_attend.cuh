// What the attention kernels over quantised caches have in common: the list of steps that is
// cut into stretches, the merge of the states that the stretches leave, and wrappers.
#pragma once

#include "kv_rows.cuh"

namespace b200moe {
namespace {

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
// Caps above 2^100 are taken as that, so that c log2(e) and scale / c stay numbers of 32 bits: up to
// scores of 2^88 either cap changes a score by less than 2^-24 of it.  0: no cap.
inline float usable_softcap(float c) { return c > 0.f ? fminf(c, 1.2676506e30f) : 0.f; }
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

// Joins the states of the segments that lie in several CTAs' stretches: WPR warps per row,
// eight per CTA.  A segment of the ordinary batch has two or three states, one of a single
// long sequence some seventy: there one warp's loads would queue up (22 us instead of 3).
constexpr int MG_WARPS = 8;
template <int HD, int WPR>
__global__ void __launch_bounds__(32 * MG_WARPS) kv_attend_merge_kernel(const AttendArgs a, int tile_rows) {
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
    B200_CHECK_CUDA(launch_dependent(kv_attend_merge_kernel<HD, MG_WARPS>, dim3(static_cast<unsigned>(rows)),
                                     dim3(32 * MG_WARPS), 0, st, a, tile_rows));
  else
    B200_CHECK_CUDA(launch_dependent(kv_attend_merge_kernel<HD, 1>, dim3(static_cast<unsigned>((rows + MG_WARPS - 1) / MG_WARPS)),
                                     dim3(32 * MG_WARPS), 0, st, a, tile_rows));
  return B200MOE_OK;
}

// Rows of a CTA's tile.
inline int attend_tile_rows(int rows) { return rows <= 8 ? 8 : 16; }

}  // namespace
}  // namespace b200moe
