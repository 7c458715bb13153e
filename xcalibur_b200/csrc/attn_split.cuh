// Paged attention: a call's parameters, the split of the work over the blocks, and the record of a (sequence,
// head) that several blocks worked on.
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
  int32_t batch, new_tokens, group, q_heads, rows, row_tiles, dim, window, lead;
  float scale_log2;
  FastDiv group_div, head_div;  // head_div: by row_tiles
  int4* splits;                 // [blocks] the split segment whose first part a block holds (x < 0: none)
  int2* marked;                 // [blocks] first and last segment that a block left marks in (x > y: none)
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

// The work is a list of units: for every (sequence, kv head, row tile) `lead` units that stand for the cost of its start
// and end (queries, join, write), then its chunks of CH positions.  Blocks get equal runs of units; one that gets lead
// units alone has nothing to do there.

// A run of chunks of one (sequence, kv head, row tile).
struct Seg {
  int b, j, row;        // sequence of the batch; head * row_tiles + tile; row of the page table
  int len, c0, c1, nch; // visible end; chunks [c0, c1) of nch
  int t0, t1, lo;       // positions of these chunks; the first that any row sees
  int left;             // units of the block's run after this segment
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
// The segment of s.b, s.j from its unit u0 on, with `units` units left.  False: lead units alone were left.
template <int CH>
__device__ __forceinline__ bool open_seg(const AttnParams& p, Seg& s, int u0, int units, int align) {
  s.len = visible(p, s.b, &s.row, &s.lo);
  s.nch = chunks_of<CH>(s.len, s.lo, align);
  s.c0 = max(0, u0 - p.lead);
  s.c1 = min(s.nch, u0 + units - p.lead);
  s.left = u0 + units - (s.nch + p.lead);
  s.t0 = (s.lo & -align) + s.c0 * CH;
  s.t1 = min(s.len, (s.lo & -align) + s.c1 * CH);
  return s.c1 > s.c0;
}
template <int CH>
__device__ __forceinline__ bool next_seg(const AttnParams& p, Seg& s, int align) {
  if (s.left <= 0) return false;
  if (++s.j == p.kv.kv_heads * p.row_tiles) {
    s.j = 0;
    if (++s.b >= p.batch) return false;
  }
  return open_seg<CH>(p, s, 0, s.left, align);
}

// The units in `blocks` runs whose lengths differ by one at most: block c's is [start(c), start(c + 1)).  Counts fit 31
// bits (checked on the host).
struct Run {
  int blocks, each, longer;  // the first `longer` blocks have each + 1 units
  int u0, u1;                // this block's
  __device__ __forceinline__ int start(int c) const { return c * each + min(c, longer); }
  __device__ __forceinline__ int owner(int u) const {
    const int edge = longer * (each + 1);
    return u < edge ? u / (each + 1) : longer + (u - edge) / each;
  }
};
// All threads of the block of WARPS warps.  s_sum: one value per warp.  Puts the place of the run's start (sequence,
// head and row tile, unit of the segment) into s.b, s.j, *unit.  False: the block has no run.  The block meets at a
// barrier at least once.
template <int CH, int WARPS>
__device__ __forceinline__ bool plan_run(const AttnParams& p, int align, int* s_sum, int* s_start, Run& run, Seg& s,
                                         int* unit) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
  const int heads = p.kv.kv_heads * p.row_tiles;
  const bool small = p.batch <= 32;  // every warp plans for itself
  const int me = small ? lane : tid;
  const int per = small ? 1 : (p.batch + WARPS * 32 - 1) / (WARPS * 32);
  const int b0 = min(p.batch, me * per), b1 = min(p.batch, b0 + per);
  int mine = 0, units0 = 0;
  for (int b = b0; b < b1; ++b) {
    int row, lo;
    const int len = visible(p, b, &row, &lo);
    units0 = p.lead + chunks_of<CH>(len, lo, align);
    mine += units0 * heads;
    if (cta == 0 && warp == (small ? 0 : warp) && (row < 0 || row >= p.kv.max_seqs)) atomicOr(p.kv.status, XCB_STATUS_BAD_SEQ);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  int before = 0, all;
  if (small) {
    all = __shfl_sync(0xffffffffu, incl, 31);
  } else {
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int v = s_sum[w];
      if (w < warp) before += v;
      all += v;
    }
  }
  run.blocks = min((int)gridDim.x, all);
  if (cta >= run.blocks) return false;
  run.each = all / run.blocks;
  run.longer = all - run.each * run.blocks;
  run.u0 = run.start(cta);
  run.u1 = run.start(cta + 1);
  int at = before + incl - mine;
  const bool found = run.u0 >= at && run.u0 < at + mine;
  int place[3] = {0, 0, 0};
  if (found) {
    int b = b0;
    if (per > 1) {
      for (;; ++b) {
        int row, lo;
        const int len = visible(p, b, &row, &lo);
        units0 = p.lead + chunks_of<CH>(len, lo, align);
        if (b == b1 - 1 || run.u0 < at + units0 * heads) break;
        at += units0 * heads;
      }
    }
    place[0] = b;
    place[1] = (run.u0 - at) / units0;
    place[2] = (run.u0 - at) - place[1] * units0;
    if (!small) s_start[0] = place[0], s_start[1] = place[1], s_start[2] = place[2];
  }
  __syncthreads();
  if (small) {
    const int who = __ffs(__ballot_sync(0xffffffffu, found)) - 1;
    s.b = __shfl_sync(0xffffffffu, place[0], who);
    s.j = __shfl_sync(0xffffffffu, place[1], who);
    *unit = __shfl_sync(0xffffffffu, place[2], who);
  } else {
    s.b = s_start[0];
    s.j = s_start[1];
    *unit = s_start[2];
  }
  return true;
}

// A split segment's first block records it for the join: sequence, head and row tile, last block, slot of its part.  A
// block's part lies in the first of its two slots if the segment is the first that it works on, as it is for every
// block but perhaps the first.  `unit`: the list's index of the segment's chunk 0.
__device__ __forceinline__ int4 split_of(const Run& r, const Seg& s, int unit, int slot) {
  return make_int4(s.b, s.j, r.owner(unit + s.nch - 1), slot);
}

}  // namespace xcb
