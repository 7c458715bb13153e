// Paged attention: a call's parameters, the split of the work over the blocks, and the join of a (sequence, head) that
// several blocks worked on.
#pragma once
#include <math.h>

#include "common.cuh"
#include "kv.cuh"

namespace xcb {

struct AttnParams {
  KvLayer kv;
  const void* q;
  int64_t q_b, q_t, q_h;
  void* out;
  float* lse;
  const int32_t* seqs;
  int32_t batch, new_tokens, group, q_heads, rows, row_tiles, dim, window;
  float scale_log2;
  FastDiv group_div, head_div;  // head_div: by row_tiles
  int32_t* counters;            // [blocks], zero between calls
  float* part_ml;               // [2 * blocks][rows of a tile][2]
  float* part_o;                // [2 * blocks][rows of a tile][padded head_dim]
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// e^(a - b) in base 2 where b is a maximum that may be -inf (nothing seen yet)
__device__ __forceinline__ float ex2_diff(float a, float b) { return ex2(a - (b == -INFINITY ? 0.f : b)); }

// A run of chunks of one (sequence, kv head, row tile).
struct Seg {
  int b, j, row;        // sequence of the batch; head * row_tiles + tile; row of the page table
  int len, c0, c1, nch; // visible end; chunks [c0, c1) of nch
  int t0, t1, lo;       // positions of these chunks; the first that any row sees
  int left;             // chunks of the block's run after this segment
};

__device__ __forceinline__ int visible(const AttnParams& p, int b, int* row, int* lo) {
  const int s = p.seqs ? p.seqs[b] : b;
  int len = 0;
  if (s >= 0 && s < p.kv.max_seqs) {
    len = max(0, p.kv.lens[s]);
    len = (int)min((int64_t)len, (int64_t)p.kv.max_pages * p.kv.page_size);
  }
  *row = s;
  // the first new token stands at len - new_tokens and sees back to there + 1 - window
  *lo = p.window ? (int)max((int64_t)0, (int64_t)len - p.new_tokens + 1 - p.window) : 0;
  return len;
}
// Chunks of CH positions, counted from the multiple of `align` (a power of two) below the first visible position.
template <int CH>
__device__ __forceinline__ int chunks_of(int len, int lo, int align) {
  return max(1, (len - (lo & -align) + CH - 1) / CH);  // an empty sequence is one empty chunk: its rows are written too
}
template <int CH>
__device__ __forceinline__ void open_seg(const AttnParams& p, Seg& s, int c0, int units, int align) {
  s.len = visible(p, s.b, &s.row, &s.lo);
  s.nch = chunks_of<CH>(s.len, s.lo, align);
  s.c0 = c0;
  s.c1 = min(s.nch, c0 + units);
  s.left = units - (s.c1 - s.c0);
  s.t0 = (s.lo & -align) + c0 * CH;
  s.t1 = min(s.len, (s.lo & -align) + s.c1 * CH);
}
template <int CH>
__device__ __forceinline__ bool next_seg(const AttnParams& p, Seg& s, int align) {
  if (s.left <= 0) return false;
  if (++s.j == p.kv.kv_heads * p.row_tiles) {
    s.j = 0;
    if (++s.b >= p.batch) return false;
  }
  open_seg<CH>(p, s, 0, s.left, align);
  return true;
}

// The list of all chunks (sequence by sequence, head by head) in `blocks` runs whose lengths differ by one at most:
// block c's is [start(c), start(c + 1)).  Counts fit 31 bits (checked on the host).
struct Run {
  int blocks, each, longer;  // the first `longer` blocks have each + 1 chunks
  int u0, u1;                // this block's
  __device__ __forceinline__ int start(int c) const { return c * each + min(c, longer); }
  __device__ __forceinline__ int owner(int u) const {
    const int edge = longer * (each + 1);
    return u < edge ? u / (each + 1) : longer + (u - edge) / each;
  }
};
// All threads of the block (a multiple of 32, at most 1024).  s_sum: one value per warp; s_start: the place of u0.
// False: the block has no run.
template <int CH>
__device__ __forceinline__ bool plan_run(const AttnParams& p, int align, int* s_sum, int* s_start, Run& run) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
  const int heads = p.kv.kv_heads * p.row_tiles;
  const int per = (p.batch + blockDim.x - 1) / blockDim.x;
  const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    int row, lo;
    const int len = visible(p, b, &row, &lo);
    mine += chunks_of<CH>(len, lo, align) * heads;
    if (cta == 0 && (row < 0 || row >= p.kv.max_seqs)) atomicOr(p.kv.status, XCB_STATUS_BAD_SEQ);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) {
    const int v = s_sum[w];
    if (w < warp) before += v;
    all += v;
  }
  run.blocks = min((int)gridDim.x, all);
  if (cta >= run.blocks) return false;
  run.each = all / run.blocks;
  run.longer = all - run.each * run.blocks;
  run.u0 = run.start(cta);
  run.u1 = run.start(cta + 1);
  int at = before + incl - mine;
  if (run.u0 >= at && run.u0 < at + mine) {
    for (int b = b0; b < b1; ++b) {
      int row, lo;
      const int len = visible(p, b, &row, &lo);
      const int nch = chunks_of<CH>(len, lo, align);
      if (run.u0 < at + nch * heads) {
        s_start[0] = b;
        s_start[1] = (run.u0 - at) / nch;
        s_start[2] = (run.u0 - at) % nch;
        break;
      }
      at += nch * heads;
    }
  }
  __syncthreads();
  return true;
}

// Which blocks share a segment: those that own its first and its last chunk, and all between.
struct Split {
  int first, last, first_slot;
};
__device__ __forceinline__ Split split_of(const Run& r, const Seg& s, int unit) {
  const int a = unit - s.c0;  // its chunks in the list of all: a .. a + nch - 1
  Split x;
  x.first = r.owner(a);
  x.last = r.owner(a + s.nch - 1);
  // every block's part is that of its first chunk, but perhaps the first block's
  x.first_slot = 2 * x.first + (r.start(x.first) < a ? 1 : 0);
  return x;
}

// Warps `warp` of `warps` join the parts of a segment's rows in run order and write them out.
template <typename T, int RT, int DP>
__device__ __forceinline__ void join_parts(const AttnParams& p, const Split& x, int b, int h, int tile0, float vs,
                                           int warp, int warps) {
  constexpr int W = DP / 32;
  const int lane = threadIdx.x & 31;
  const int parts = x.last - x.first + 1;
  const int nrows = min(RT, p.rows - tile0);
  const auto slot_of = [&](int i) { return i == 0 ? x.first_slot : 2 * (x.first + i); };
  for (int rl = warp; rl < nrows; rl += warps) {
    float top = -INFINITY;
    for (int q = lane; q < parts; q += 32) top = fmaxf(top, __ldcg(p.part_ml + ((int64_t)slot_of(q) * RT + rl) * 2));
#pragma unroll
    for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    float sum = 0.f, acc[W];
#pragma unroll
    for (int w = 0; w < W; ++w) acc[w] = 0.f;
    for (int q0 = 0; q0 < parts; q0 += 32) {
      float wt = 0.f;
      if (q0 + lane < parts) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + ((int64_t)slot_of(q0 + lane) * RT + rl) * 2));
        wt = ex2_diff(ml.x, top);
        sum += wt * ml.y;
      }
      const int n = min(32, parts - q0);
#pragma unroll 8
      for (int q = 0; q < n; ++q) {
        const float wq = __shfl_sync(0xffffffffu, wt, q);
        const float* src = p.part_o + ((int64_t)slot_of(q0 + q) * RT + rl) * DP + lane * W;
        if constexpr (W == 2) {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          acc[0] += wq * v.x;
          acc[1] += wq * v.y;
        } else {
#pragma unroll
          for (int w = 0; w < W; w += 4) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(src + w));
            acc[w] += wq * v.x;
            acc[w + 1] += wq * v.y;
            acc[w + 2] += wq * v.z;
            acc[w + 3] += wq * v.w;
          }
        }
      }
    }
#pragma unroll
    for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const int r = tile0 + rl, tok = fdiv(r, p.group_div);
    const int64_t at = ((int64_t)b * p.new_tokens + tok) * p.q_heads + h * p.group + r - tok * p.group;
    const float inv = sum == 0.f ? 0.f : vs / sum;
    T* dst = (T*)p.out + at * p.dim + lane * W;
#pragma unroll
    for (int w = 0; w < W; w += 2)
      if (lane * W + w < p.dim) *reinterpret_cast<uint32_t*>(dst + w) = pack2<T>(acc[w] * inv, acc[w + 1] * inv);
    if (p.lse && lane == 0) p.lse[at] = sum == 0.f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
  }
}

}  // namespace xcb
