// Attention of new tokens over the paged cache: one pass over the keys and values with a running maximum and sum.
//
// Mathematics: for a row (new token, query head) with scores s_j = scale * q . k_j over the visible j, a block of
// positions is summed up by (m, l, o) = (max s_j, sum e^(s_j - m), sum e^(s_j - m) v_j), and two such triples join as
// m = max, l = l1 e^(m1 - m) + l2 e^(m2 - m), o likewise; the result is o / l.  Exponentials are taken in base 2 with
// log2(e) folded into the scale.
//
// Bound: HBM.  All rows of one kv head (group * new tokens) share one read of its keys and values, so a 16-bit cache
// asks for `rows` flops per byte: 16 to 128, against ~255 where the tensor pipe would bound.
//
// Split: the work is cut into chunks of 16 * warps positions and the list of all chunks (sequence by sequence, head
// by head) into as many equal runs as there are SMs, found on the device from the lengths, so that ragged batches and
// single long sequences keep every SM busy alike and nothing waits for the host.  A (sequence, head) that lies in
// several runs is joined by the block that finishes it last, in run order whoever that is, so results do not depend on
// timing.
//
// Inside a block every group of WM warps streams its own 16 * WM positions through its own ring of shared-memory
// stages (cp.async, 16 bytes a lane, swizzled so that ldmatrix has no bank conflicts); with WM = 1 (up to 16 rows)
// warps never wait for one another but at the end of a (sequence, head).  WM = 2, 4, 8 spread up to 128 rows over
// the warps of a group, which share the stages.
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "kv.cuh"

namespace xcb {
namespace {

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
  float* part_ml;               // [2 * blocks][16 * WM][2]
  float* part_o;                // [2 * blocks][16 * WM][DP]
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// the rest of the 16 bytes is zeroed; with bytes = 0 nothing is read
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_16816(d, a[0], a[1], a[2], a[3], b0, b1);
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four e4m3 codes to two pairs of f16, exactly.
__device__ __forceinline__ void e4m3_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// e^(a - b) in base 2 where b is a maximum that may be -inf (nothing seen yet)
__device__ __forceinline__ float ex2_diff(float a, float b) { return ex2(a - (b == -INFINITY ? 0.f : b)); }

template <int DP, bool F8>
struct Shape {
  static constexpr int kWarps = DP == 256 ? 4 : 8;
  static constexpr int kPitch = DP * (F8 ? 1 : 2);   // bytes of one position's row in shared memory
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kTok = kPitch <= 128 ? 32 : 16;  // positions of a warp's step: 4 to 8 KB of keys and values
  static constexpr int kSub = kTok * kPitch;         // their keys (or values)
  static constexpr int kFit = 196608 / (kWarps * 2 * kSub);
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kRing = kWarps * kStages * 2 * kSub;
  static constexpr int kRedPitch = DP + 4;
  static constexpr int kRed = kWarps / 2 * 16 * kRedPitch * 4;
  static constexpr int kRedMl = kWarps / 2 * 16 * 2 * 4;
  static constexpr int kMasks = kWarps * kStages * 4;
  static constexpr int kScalars = kWarps * 8 + 16;
  static constexpr int kBytes = kRing + kRed + kRedMl + kMasks + kScalars;
};

// Byte offset of 16-byte chunk c of row r: rows that ldmatrix reads together fall into different banks.
template <int PITCH>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  return r * PITCH + ((PITCH >= 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4);
}

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
// Chunks are counted from the step that holds the first visible position.
template <int CH, int TOK>
__device__ __forceinline__ int chunks_of(int len, int lo) {
  return max(1, (len - lo / TOK * TOK + CH - 1) / CH);  // an empty sequence is one empty chunk: its rows are written too
}
template <int CH, int TOK>
__device__ __forceinline__ void open_seg(const AttnParams& p, Seg& s, int c0, int units) {
  s.len = visible(p, s.b, &s.row, &s.lo);
  s.nch = chunks_of<CH, TOK>(s.len, s.lo);
  s.c0 = c0;
  s.c1 = min(s.nch, c0 + units);
  s.left = units - (s.c1 - s.c0);
  s.t0 = s.lo / TOK * TOK + c0 * CH;
  s.t1 = min(s.len, s.lo / TOK * TOK + s.c1 * CH);
}
template <int CH, int TOK>
__device__ __forceinline__ bool next_seg(const AttnParams& p, Seg& s) {
  if (s.left <= 0) return false;
  if (++s.j == p.kv.kv_heads * p.row_tiles) {
    s.j = 0;
    if (++s.b >= p.batch) return false;
  }
  open_seg<CH, TOK>(p, s, 0, s.left);
  return true;
}

template <typename T, bool F8, int DP, int WM>
__global__ void __launch_bounds__(Shape<DP, F8>::kWarps * 32, 1) attn_kernel(const AttnParams p) {
  using S = Shape<DP, F8>;
  constexpr int NW = S::kWarps, WN = NW / WM, NS = S::kStages;
  constexpr int TOK = S::kTok, SN = TOK / 8;
  constexpr int TT = TOK * WM;      // positions of a group's tile
  constexpr int CH = TOK * NW;      // positions of a chunk
  constexpr int RT = 16 * WM;       // rows of a row tile
  constexpr int KS = DP / 16;       // 16-wide steps of the head dimension
  constexpr int NT = DP / 8;        // 8-wide column tiles of the output
  using M = typename std::conditional<F8, __half, T>::type;  // operand type of the tensor steps
  static_assert(WM <= NW, "a group has at most the block's warps");

  extern __shared__ __align__(1024) uint8_t smem[];  // all of the block's shared memory: steps start at multiples of 1 KB
  uint8_t* const ring = smem;
  float* const red = reinterpret_cast<float*>(smem + S::kRing);
  float* const red_ml = reinterpret_cast<float*>(smem + S::kRing + S::kRed);
  uint32_t* const masks = reinterpret_cast<uint32_t*>(smem + S::kRing + S::kRed + S::kRedMl);
  int64_t* const s_warp = reinterpret_cast<int64_t*>(smem + S::kRing + S::kRed + S::kRedMl + S::kMasks);
  int* const s_start = reinterpret_cast<int*>(s_warp + NW);  // [3]
  int& s_last = s_start[3];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grp = warp / WM, wm = warp % WM;
  const int g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x;

  // ---- this block's run of chunks -------------------------------------------------------------------------------
  int64_t total, u0, u1;
  {
    const int heads = p.kv.kv_heads * p.row_tiles;
    const int per = (p.batch + NW * 32 - 1) / (NW * 32);
    const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) {
      int row, lo;
      const int len = visible(p, b, &row, &lo);
      mine += (int64_t)chunks_of<CH, TOK>(len, lo) * heads;
      if (cta == 0 && (row < 0 || row >= p.kv.max_seqs)) atomicOr(p.kv.status, XCB_STATUS_BAD_SEQ);
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) before += s_warp[w];
      all += s_warp[w];
    }
    total = all;
    const int64_t n = min((int64_t)gridDim.x, total);
    if (cta >= n) return;
    u0 = cta * total / n;
    u1 = (cta + 1) * total / n;
    int64_t at = before + incl - mine;
    if (u0 >= at && u0 < at + mine) {
      for (int b = b0; b < b1; ++b) {
        int row, lo;
        const int len = visible(p, b, &row, &lo);
        const int nch = chunks_of<CH, TOK>(len, lo);
        if (u0 < at + (int64_t)nch * heads) {
          s_start[0] = b;
          s_start[1] = (int)((u0 - at) / nch);
          s_start[2] = (int)((u0 - at) % nch);
          break;
        }
        at += (int64_t)nch * heads;
      }
    }
    __syncthreads();
  }
  const int blocks = (int)min((int64_t)gridDim.x, total);

  // ---- the producing side of a warp: 16 positions per tile -------------------------------------------------------
  Seg ps;
  ps.b = s_start[0];
  ps.j = s_start[1];
  open_seg<CH, TOK>(p, ps, s_start[2], (int)(u1 - u0));
  Seg cs = ps;
  int ptile = grp;
  bool more = true;
  const int row_bytes = p.dim * (F8 ? 1 : 2);
  uint8_t* const my_ring = ring + warp * (NS * 2 * S::kSub);
  uint32_t* const my_masks = masks + warp * NS;

  // Of the step looked up last: which of its positions are there, and the byte offset of the first one's row (where
  // every step lies inside one page) or of lane's one.
  const bool in_page = p.kv.page_size % TOK == 0;
  int64_t f_off = 0;
  uint32_t f_mask = 0;
  const auto look_up = [&]() {
    f_mask = 0;
    while (more && ptile * TT >= ps.t1 - ps.t0) {
      more = next_seg<CH, TOK>(p, ps);
      ptile = grp;
    }
    if (!more) return;
    const int pos0 = ps.t0 + ptile * TT + wm * TOK;
    ptile += WN;
    const int32_t* const row = p.kv.table + (int64_t)ps.row * p.kv.max_pages;
    const int pos = in_page ? pos0 : pos0 + lane;
    const bool in = in_page ? pos0 < ps.t1 : lane < TOK && pos >= ps.lo && pos < ps.t1;
    bool ok = false;
    if (in) {
      const int pi = fdiv(pos, p.kv.page_div);
      const int page = row[pi];
      ok = (uint32_t)page < (uint32_t)p.kv.num_pages;
      if (!ok) atomicOr(p.kv.status, XCB_STATUS_BAD_PAGE);
      f_off = (((int64_t)page * p.kv.kv_heads + fdiv(ps.j, p.head_div)) * p.kv.page_size + (pos - pi * p.kv.page_size)) *
              row_bytes;
    }
    if (in_page) {
      const int from = max(0, ps.lo - pos0), to = min(TOK, ps.t1 - pos0);
      if (ok) f_mask = (uint32_t)(((1ull << to) - 1) & ~((1ull << from) - 1));
    } else {
      f_mask = __ballot_sync(0xffffffffu, ok);
    }
  };
  // This lane copies chunk lc of rows lr, lr + RPI, ...
  constexpr int RPI = 32 / S::kChunks, IT = TOK / RPI;
  const int lc = lane % S::kChunks, lr = lane / S::kChunks;
  const uint32_t l_dst = smem_u32(my_ring) + swz<S::kPitch>(lr, lc);
  const int64_t l_src = (int64_t)lr * row_bytes + lc * 16;
  const auto issue = [&](int stage, int64_t off, uint32_t mask) {
    if (lane == 0) my_masks[stage] = mask;
    if (!mask) return;
    const uint32_t dst = l_dst + stage * (2 * S::kSub);
    // row lr + i * RPI: the swizzle's exclusive or splits into the lane's part and the step's
    const auto at = [&](int i) {
      return (S::kPitch >= 128 ? dst ^ (((i * RPI) & 7) << 4) : dst) + i * RPI * S::kPitch;
    };
    const uint8_t* k = p.kv.k + off + l_src;
    if (in_page && mask == (uint32_t)((1ull << TOK) - 1)) {
      const uint8_t* v = k + p.kv.plane;
      if (row_bytes == S::kPitch) {
#pragma unroll
        for (int i = 0; i < IT; ++i) cp_async16(at(i), k + i * RPI * S::kPitch);
#pragma unroll
        for (int i = 0; i < IT; ++i) cp_async16(at(i) + S::kSub, v + i * RPI * S::kPitch);
      } else {
        const int n = lc * 16 < row_bytes ? 16 : 0;
        const int step = RPI * row_bytes;
        if (!n) k = v = p.kv.k;
#pragma unroll
        for (int i = 0; i < IT; ++i) cp_async16(at(i), n ? k + i * step : k, n);
#pragma unroll
        for (int i = 0; i < IT; ++i) cp_async16(at(i) + S::kSub, n ? v + i * step : v, n);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < IT; ++i) {
        const int r = lr + i * RPI;
        const int64_t o = in_page ? off + (int64_t)r * row_bytes : __shfl_sync(0xffffffffu, off, r);
        const bool in = lc * 16 < row_bytes && ((mask >> r) & 1u);
        const uint8_t* src = p.kv.k + (in ? o + lc * 16 : 0);
        const uint32_t d = smem_u32(my_ring) + stage * (2 * S::kSub) + swz<S::kPitch>(r, lc);
        cp_async16(d, src, in ? 16 : 0);
        cp_async16(d + S::kSub, src + p.kv.plane, in ? 16 : 0);
      }
    }
  };
  {
    int64_t off[NS - 1];
    uint32_t mask[NS - 1];
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
      look_up();
      off[s] = f_off;
      mask[s] = f_mask;
    }
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
      issue(s, off[s], mask[s]);
      cp_async_commit();
    }
    look_up();
  }

  // ldmatrix row addresses of this lane: keys as (position, dimension) pairs, values transposed
  const uint32_t k_lane = swz<S::kPitch>((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
  const uint32_t v_lane = swz<S::kPitch>(lane & 15, lane >> 4);

  // ---- the consuming side ----------------------------------------------------------------------------------------
  int stage = 0, fill = NS - 1;
  int64_t unit = u0;  // first chunk of the current segment
  do {
    const int h = fdiv(cs.j, p.head_div), tile0 = (cs.j - h * p.row_tiles) * RT;
    // this lane's two rows of the warp's 16
    const T* qrow[2];
    int hi[2], lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = tile0 + wm * 16 + g + 8 * i;
      qrow[i] = nullptr;
      hi[i] = cs.len;
      lo[i] = 0;
      if (r < p.rows) {
        const int l = fdiv(r, p.group_div);
        qrow[i] = (const T*)p.q + cs.b * p.q_b + l * p.q_t + (h * p.group + r - l * p.group) * p.q_h;
        hi[i] = cs.len - p.new_tokens + l + 1;
        lo[i] = p.window ? max(0, hi[i] - p.window) : 0;
      }
    }
    uint32_t qf[KS][4];
    float to_log2[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        if constexpr (F8) {
          // a step's contraction index runs over d = 4t, 4t+1 | 4t+2, 4t+3: the four codes a lane gets of a row
          uint2 v = make_uint2(0, 0);
          if (qrow[i] && kk * 16 < p.dim) v = *reinterpret_cast<const uint2*>(qrow[i] + kk * 16 + 4 * t);
          qf[kk][i] = v.x;
          qf[kk][2 + i] = v.y;
        } else {
          qf[kk][i] = qrow[i] && kk * 16 < p.dim ? *reinterpret_cast<const uint32_t*>(qrow[i] + kk * 16 + 2 * t) : 0u;
          qf[kk][2 + i] =
              qrow[i] && kk * 16 + 8 < p.dim ? *reinterpret_cast<const uint32_t*>(qrow[i] + kk * 16 + 8 + 2 * t) : 0u;
        }
      }
      to_log2[i] = p.scale_log2;
      if constexpr (F8) {
        if (p.kv.k_scale) to_log2[i] *= p.kv.k_scale[h];
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          // bf16 queries as f16: scaled by a power of two that brings the row's largest value to [2^14, 2^15), which
          // is exact down to 2^-38 of that value
          float top = 0.f;
#pragma unroll
          for (int kk = 0; kk < KS; ++kk) {
            const float2 a = unpack2<T>(qf[kk][i]), b = unpack2<T>(qf[kk][2 + i]);
            top = fmaxf(fmaxf(top, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(b.x), fabsf(b.y)));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int ex = (int)(__float_as_uint(top) >> 23);                // biased exponent, 255: not finite
          const int up = ex == 255 || ex == 0 ? 0 : max(-100, min(100, 127 + 14 - ex));
          const float mul = __uint_as_float((uint32_t)(127 + up) << 23), inv = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
          for (int kk = 0; kk < KS; ++kk) {
            const float2 a = unpack2<T>(qf[kk][i]), b = unpack2<T>(qf[kk][2 + i]);
            qf[kk][i] = pack2<__half>(a.x * mul, a.y * mul);
            qf[kk][2 + i] = pack2<__half>(b.x * mul, b.y * mul);
          }
          to_log2[i] *= inv;
        }
      }
    }
    // Scores are multiplied by to_log2 after the maximum is taken, so it is made positive (and never zero: -inf stays).
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (to_log2[i] < 0.f) {
        to_log2[i] = -to_log2[i];
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          qf[kk][i] ^= 0x80008000u;
          qf[kk][2 + i] ^= 0x80008000u;
        }
      }
      to_log2[i] = fmaxf(to_log2[i], 1e-37f);
    }
    float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

    for (int tile = grp; tile * TT < cs.t1 - cs.t0; tile += WN) {
      cp_async_wait<NS - 2>();
      if constexpr (WM == 1)
        __syncwarp();
      else
        named_bar(1 + grp, WM * 32);
      issue(fill, f_off, f_mask);  // into the stage that the tile before this one was read from
      cp_async_commit();
      look_up();

#pragma unroll 1
      for (int sub = 0; sub < WM; ++sub) {
        const uint32_t vm = masks[(grp * WM + sub) * NS + stage];
        if (!vm) continue;
        const uint8_t* const base = ring + (grp * WM + sub) * (NS * 2 * S::kSub) + stage * (2 * S::kSub);
        const uint32_t kb = smem_u32(base), vb = kb + S::kSub;
        const int pos0 = cs.t0 + tile * TT + sub * TOK;
        float s[SN][4];
#pragma unroll
        for (int n = 0; n < SN; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int b = 0; b < SN / 2; ++b) {
          // the swizzle again: chunk 2 kk + cc of the lane's row is the lane's address xor 32 kk
          const uint32_t ka = kb + k_lane + b * 16 * S::kPitch;
          if constexpr (F8) {
#pragma unroll
            for (int k2 = 0; k2 < KS / 2; ++k2) {
              uint32_t w[4];
              ldsm4(w, ka ^ (k2 << 5));
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                  uint32_t b0, b1;
                  e4m3_f16(w[2 * n + e], b0, b1);
                  mma16<M>(s[2 * b + n], qf[2 * k2 + e], b0, b1);
                }
            }
          } else {
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
              uint32_t w[4];
              ldsm4(w, ka ^ (kk << 5));
              mma16<M>(s[2 * b], qf[kk], w[0], w[1]);
              mma16<M>(s[2 * b + 1], qf[kk], w[2], w[3]);
            }
          }
        }
        // visible to some rows only: the last new_tokens - 1 positions and the window's edge
        const bool ragged = p.new_tokens > 1 && (pos0 + TOK > cs.len - p.new_tokens + 1 ||
                                                 (p.window && pos0 < cs.len - p.window));
        const auto seen = [&](int col, int i) {
          return ((vm >> col) & 1u) && (!ragged || (pos0 + col < hi[i] && pos0 + col >= lo[i]));
        };
        if (ragged || vm != (uint32_t)((1ull << TOK) - 1)) {
#pragma unroll
          for (int n = 0; n < SN; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (!seen(n * 8 + 2 * t + (c & 1), c >> 1)) s[n][c] = -INFINITY;
        }
        float mx[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mx[i] = fmaxf(s[0][2 * i], s[0][2 * i + 1]);
#pragma unroll
          for (int n = 1; n < SN; ++n) mx[i] = fmaxf(mx[i], fmaxf(s[n][2 * i], s[n][2 * i + 1]));
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2)) * to_log2[i];
        }
        if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
          float a[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float top = fmaxf(m[i], mx[i]);
            a[i] = ex2_diff(m[i], top);
            m[i] = top;
            l[i] *= a[i];
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[n][0] *= a[0];
            o[n][1] *= a[0];
            o[n][2] *= a[1];
            o[n][3] *= a[1];
          }
        }
        const float mm[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[n][c] = ex2(fmaf(s[n][c], to_log2[c >> 1], -mm[c >> 1]));
            l[c >> 1] += s[n][c];
          }
        // A value that is not finite at a position hidden from some rows would reach them as 0 * inf: such a tile is
        // summed by hand.
        bool odd = false;
        if (ragged) {
          bool bad = false;
#pragma unroll 1
          for (int i = lane; i < S::kSub / 16; i += 32) {
            const uint4 v4 = reinterpret_cast<const uint4*>(base + S::kSub)[i];
            const uint32_t v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if constexpr (F8) {
                // a byte with all seven low bits set carries into its eighth
                bad |= (((v[q] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
              } else {
                constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
                bad |= (v[q] & E) == E || ((v[q] >> 16) & E) == E;
              }
            }
          }
          odd = __any_sync(0xffffffffu, bad);
        }
        if (odd) {
#pragma unroll 1
          for (int col = 0; col < TOK; ++col) {
            float mine0 = 0.f, mine1 = 0.f;
#pragma unroll
            for (int n = 0; n < SN; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if ((col >> 3) == n && (col & 1) == e) {
                  mine0 = s[n][e];
                  mine1 = s[n][2 + e];
                }
            const int from = (lane & ~3) | ((col & 7) >> 1);
            const float p0 = __shfl_sync(0xffffffffu, mine0, from), p1 = __shfl_sync(0xffffffffu, mine1, from);
            const bool see0 = seen(col, 0), see1 = seen(col, 1);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int d = F8 ? (n >> 1) * 16 + 4 * t + 2 * e + (n & 1) : n * 8 + 2 * t + e;
                const int byte = d * (F8 ? 1 : 2);
                const uint8_t* at = base + S::kSub + swz<S::kPitch>(col, byte >> 4) + (byte & 15);
                float v;
                if constexpr (F8) {
                  uint32_t f, unused;
                  e4m3_f16(*at, f, unused);
                  v = unpack2<__half>(f).x;
                } else
                  v = unpack2<T>(*reinterpret_cast<const uint16_t*>(at)).x;
                if (see0) o[n][e] += p0 * v;
                if (see1) o[n][2 + e] += p1 * v;
              }
          }
          continue;
        }
        // The probabilities as operands.  Rounded once to 16 bits they would add an error as large as the output's own
        // rounding; for a 16-bit cache a second operand carries the rest.  An 8-bit cache's own rounding is coarser by
        // far, and one f16 operand serves.
#pragma unroll
        for (int b = 0; b < SN / 2; ++b) {
          uint32_t a_hi[4], a_lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = s[2 * b + (i >> 1)][2 * (i & 1)], y = s[2 * b + (i >> 1)][2 * (i & 1) + 1];
            a_hi[i] = pack2<M>(x, y);
            if constexpr (!F8) {
              const float2 f = unpack2<M>(a_hi[i]);
              a_lo[i] = pack2<M>(x - f.x, y - f.y);
            }
          }
          const uint32_t va = vb + v_lane + b * 16 * S::kPitch;
#pragma unroll
          for (int n2 = 0; n2 < S::kChunks / 2; ++n2) {
            uint32_t w[4];
            ldsm4_trans(w, va ^ (n2 << 5));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if constexpr (F8) {
                // bytes: position 2t (d, d+1), position 2t+1 (d, d+1): regroup by d
                uint32_t b0, b1, c0, c1;
                e4m3_f16(__byte_perm(w[2 * e], w[2 * e + 1], 0x6420), b0, b1);
                e4m3_f16(__byte_perm(w[2 * e], w[2 * e + 1], 0x7531), c0, c1);
                mma16<M>(o[4 * n2 + 2 * e], a_hi, b0, b1);
                mma16<M>(o[4 * n2 + 2 * e + 1], a_hi, c0, c1);
              } else {
                mma16<M>(o[2 * n2 + e], a_hi, w[2 * e], w[2 * e + 1]);
                mma16<M>(o[2 * n2 + e], a_lo, w[2 * e], w[2 * e + 1]);
              }
            }
          }
        }
      }
      stage = stage + 1 == NS ? 0 : stage + 1;
      fill = fill + 1 == NS ? 0 : fill + 1;
    }

    // ---- join the block's groups, a tree in fixed order ------------------------------------------------------------
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    // (row of the warp's 16, columns) of accumulator pair (n, i) are one float2 of the natural order, two strided
    // floats for an 8-bit cache
    const auto column = [&](int n, int e) { return F8 ? (n >> 1) * 16 + 4 * t + 2 * e + (n & 1) : n * 8 + 2 * t + e; };
#pragma unroll
    for (int half = WN / 2; half > 0; half >>= 1) {
      __syncthreads();
      if (grp >= half && grp < 2 * half) {
        float* dst = red + ((grp - half) * WM + wm) * 16 * S::kRedPitch;
        float* ml = red_ml + ((grp - half) * WM + wm) * 32;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (t == 0) *reinterpret_cast<float2*>(ml + 2 * (g + 8 * i)) = make_float2(m[i], l[i]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            dst[(g + 8 * i) * S::kRedPitch + column(n, 0)] = o[n][2 * i];
            dst[(g + 8 * i) * S::kRedPitch + column(n, 1)] = o[n][2 * i + 1];
          }
        }
      }
      __syncthreads();
      if (grp < half) {
        const float* src = red + (grp * WM + wm) * 16 * S::kRedPitch;
        const float* ml = red_ml + (grp * WM + wm) * 32;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 other = *reinterpret_cast<const float2*>(ml + 2 * (g + 8 * i));
          const float top = fmaxf(m[i], other.x);
          const float a = ex2_diff(m[i], top), b = ex2_diff(other.x, top);
          m[i] = top;
          l[i] = l[i] * a + other.y * b;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[n][2 * i] = o[n][2 * i] * a + src[(g + 8 * i) * S::kRedPitch + column(n, 0)] * b;
            o[n][2 * i + 1] = o[n][2 * i + 1] * a + src[(g + 8 * i) * S::kRedPitch + column(n, 1)] * b;
          }
        }
      }
    }

    const bool whole = cs.c0 == 0 && cs.c1 == cs.nch;
    const float vs = F8 && p.kv.v_scale ? p.kv.v_scale[h] : 1.f;
    const int slot = 2 * cta + (unit == u0 ? 0 : 1);
    if (grp == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rl = wm * 16 + g + 8 * i, r = tile0 + rl;
        if (r >= p.rows) continue;
        if (whole) {
          const int tok = fdiv(r, p.group_div);
          const int64_t at = ((int64_t)cs.b * p.new_tokens + tok) * p.q_heads + h * p.group + r - tok * p.group;
          const float inv = l[i] == 0.f ? 0.f : vs / l[i];
          T* dst = (T*)p.out + at * p.dim;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (F8) {
              if (n & 1) continue;
              const int d = column(n, 0);
              if (d < p.dim)
                *reinterpret_cast<uint2*>(dst + d) =
                    make_uint2(pack2<T>(o[n][2 * i] * inv, o[n + 1][2 * i] * inv),
                               pack2<T>(o[n][2 * i + 1] * inv, o[n + 1][2 * i + 1] * inv));
            } else {
              const int d = column(n, 0);
              if (d < p.dim)
                *reinterpret_cast<uint32_t*>(dst + d) = pack2<T>(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
            }
          }
          if (p.lse && t == 0) p.lse[at] = l[i] == 0.f ? -INFINITY : m[i] * 0.6931471805599453f + logf(l[i]);
        } else {
          float* po = p.part_o + ((int64_t)slot * RT + rl) * DP;
          if (t == 0) *reinterpret_cast<float2*>(p.part_ml + ((int64_t)slot * RT + rl) * 2) = make_float2(m[i], l[i]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (F8) {
              if (n & 1) continue;
              *reinterpret_cast<float4*>(po + column(n, 0)) =
                  make_float4(o[n][2 * i], o[n + 1][2 * i], o[n][2 * i + 1], o[n + 1][2 * i + 1]);
            } else {
              *reinterpret_cast<float2*>(po + column(n, 0)) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            }
          }
        }
      }
    }
    if (!whole) {
      // ---- the block that finishes a split (sequence, head) last joins its parts, in run order -----------------------
      const int64_t a = unit - cs.c0, z = a + cs.nch;  // its chunks in the list of all
      const int first = (int)(((a + 1) * blocks + total - 1) / total) - 1;
      const int last = (int)((z * blocks + total - 1) / total) - 1;
      __threadfence();
      __syncthreads();
      if (tid == 0) s_last = atomicAdd(&p.counters[first], 1) == last - first;
      __syncthreads();
      if (s_last) {
        __threadfence();
        if (tid == 0) p.counters[first] = 0;
        const int parts = last - first + 1;
        // every block's part is that of its first chunk, but perhaps the first block's
        const int first_slot = 2 * first + (first * total / blocks < a ? 1 : 0);
        const auto slot_of = [&](int c) { return c == first ? first_slot : 2 * c; };
        const int nrows = min(RT, p.rows - tile0);
        constexpr int W = DP / 32;
        for (int rl = warp; rl < nrows; rl += NW) {
          float top = -INFINITY;
          for (int q = lane; q < parts; q += 32)
            top = fmaxf(top, __ldcg(p.part_ml + ((int64_t)slot_of(first + q) * RT + rl) * 2));
#pragma unroll
          for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
          float sum = 0.f, acc[W];
#pragma unroll
          for (int w = 0; w < W; ++w) acc[w] = 0.f;
          for (int q0 = 0; q0 < parts; q0 += 32) {
            float wt = 0.f;
            if (q0 + lane < parts) {
              const float2 ml =
                  __ldcg(reinterpret_cast<const float2*>(p.part_ml + ((int64_t)slot_of(first + q0 + lane) * RT + rl) * 2));
              wt = ex2_diff(ml.x, top);
              sum += wt * ml.y;
            }
            const int n = min(32, parts - q0);
#pragma unroll 8
            for (int q = 0; q < n; ++q) {
              const float wq = __shfl_sync(0xffffffffu, wt, q);
              const float* src = p.part_o + ((int64_t)slot_of(first + q0 + q) * RT + rl) * DP + lane * W;
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
          const int64_t at = ((int64_t)cs.b * p.new_tokens + tok) * p.q_heads + h * p.group + r - tok * p.group;
          const float inv = sum == 0.f ? 0.f : vs / sum;
          T* dst = (T*)p.out + at * p.dim + lane * W;
#pragma unroll
          for (int w = 0; w < W; w += 2)
            if (lane * W + w < p.dim) *reinterpret_cast<uint32_t*>(dst + w) = pack2<T>(acc[w] * inv, acc[w + 1] * inv);
          if (p.lse && lane == 0) p.lse[at] = sum == 0.f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
        }
      }
    }
    unit += cs.c1 - cs.c0;
  } while (next_seg<CH, TOK>(p, cs));
  cp_async_wait<0>();
}

// ------------------------------------------------------------------------------------------------ host side
int dim_class(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Warps that share a tile: enough for all rows of a kv head, so that its keys and values are read once.
int row_warps(int rows, int dim) {
  const int most = dim_class(dim) == 256 ? 4 : 8;
  int wm = 1;
  while (wm < most && 16 * wm < rows) wm *= 2;
  return wm;
}

struct AttnWs {
  size_t counters, ml, o, total;
};
AttnWs attn_ws(int sms, int wm, int dp) {
  AttnWs w;
  w.counters = 0;
  w.ml = ((size_t)sms * 4 + 255) / 256 * 256;
  w.o = w.ml + ((size_t)2 * sms * 16 * wm * 8 + 255) / 256 * 256;
  w.total = w.o + (size_t)2 * sms * 16 * wm * dp * 4;
  return w;
}

template <typename T, bool F8, int DP, int WM>
int launch(const AttnParams& p, int sms, cudaStream_t stream) {
  constexpr int bytes = Shape<DP, F8>::kBytes;
  static_assert(bytes <= 227 * 1024, "the stages fit one SM");
  static bool ready[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return XCB_ERR_CUDA;
  if (dev >= kMaxDevices || !ready[dev]) {
    if (cudaFuncSetAttribute(attn_kernel<T, F8, DP, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess)
      return XCB_ERR_CUDA;
    if (dev < kMaxDevices) ready[dev] = true;
  }
  attn_kernel<T, F8, DP, WM><<<sms, Shape<DP, F8>::kWarps * 32, bytes, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? XCB_OK : XCB_ERR_CUDA;
}
template <typename T, bool F8, int DP>
int launch_wm(const AttnParams& p, int wm, int sms, cudaStream_t stream) {
  switch (wm) {
    case 1: return launch<T, F8, DP, 1>(p, sms, stream);
    case 2: return launch<T, F8, DP, 2>(p, sms, stream);
    case 4: return launch<T, F8, DP, 4>(p, sms, stream);
    default:
      if constexpr (DP <= 128) return launch<T, F8, DP, 8>(p, sms, stream);
      return XCB_ERR_UNSUPPORTED;
  }
}
template <typename T, bool F8>
int launch_dim(const AttnParams& p, int wm, int sms, cudaStream_t stream) {
  switch (dim_class(p.dim)) {
    case 64: return launch_wm<T, F8, 64>(p, wm, sms, stream);
    case 128: return launch_wm<T, F8, 128>(p, wm, sms, stream);
    default: return launch_wm<T, F8, 256>(p, wm, sms, stream);
  }
}

int heads_check(const XcbKvCache* c, int q_heads, int new_tokens) {
  if (q_heads <= 0 || new_tokens <= 0 || q_heads % c->kv_heads) return XCB_ERR_INVALID_ARG;
  if (q_heads > 65536 || new_tokens > 65536 || (int64_t)(q_heads / c->kv_heads) * new_tokens > 1 << 20)
    return XCB_ERR_UNSUPPORTED;
  return XCB_OK;
}

}  // namespace
}  // namespace xcb

using namespace xcb;

extern "C" {

size_t xcb_attn_workspace_bytes(const XcbKvCache* c, int32_t q_heads, int32_t new_tokens) {
  if (kv_check(c) != XCB_OK || heads_check(c, q_heads, new_tokens) != XCB_OK) return 0;
  const int sms = sm_count();
  return sms ? attn_ws(sms, row_warps(q_heads / c->kv_heads * new_tokens, c->head_dim), dim_class(c->head_dim)).total : 0;
}

int xcb_attn_workspace_init(void* ws, size_t bytes, cudaStream_t stream) {
  if (!ws) return XCB_ERR_INVALID_ARG;
  return cudaMemsetAsync(ws, 0, bytes, stream) == cudaSuccess ? XCB_OK : XCB_ERR_CUDA;
}

int xcb_paged_attention(const XcbKvCache* c, const XcbAttnArgs* a, void* ws, size_t ws_bytes, cudaStream_t stream) {
  int rc = kv_check(c);
  if (rc != XCB_OK) return rc;
  if (!a || a->batch < 0 || a->layer < 0 || a->layer >= c->layers || a->window < 0) return XCB_ERR_INVALID_ARG;
  if (a->dtype != XCB_DTYPE_BF16 && a->dtype != XCB_DTYPE_F16) return XCB_ERR_INVALID_ARG;
  if (c->dtype != XCB_DTYPE_E4M3 && c->dtype != a->dtype) return XCB_ERR_UNSUPPORTED;
  if ((rc = heads_check(c, a->q_heads, a->new_tokens)) != XCB_OK) return rc;
  if (a->batch > 1 << 20) return XCB_ERR_UNSUPPORTED;
  if (a->batch == 0) return XCB_OK;
  if (!a->seqs && a->batch > c->max_seqs) return XCB_ERR_INVALID_ARG;
  if (!a->q || !a->out || !ws || !kv_aligned(a->q, 16) || !kv_aligned(a->out, 16) || !kv_aligned(ws, 256) ||
      !kv_aligned(a->lse, 4) || !kv_aligned(a->seqs, 4) || a->q_stride[0] % 8 || a->q_stride[1] % 8 || a->q_stride[2] % 8)
    return XCB_ERR_INVALID_ARG;
  const int sms = sm_count();
  if (!sms) return XCB_ERR_CUDA;
  AttnParams p{};
  p.kv = kv_layer(c, a->layer);
  p.q = a->q;
  p.q_b = a->q_stride[0];
  p.q_t = a->q_stride[1];
  p.q_h = a->q_stride[2];
  p.out = a->out;
  p.lse = a->lse;
  p.seqs = a->seqs;
  p.batch = a->batch;
  p.new_tokens = a->new_tokens;
  p.q_heads = a->q_heads;
  p.group = a->q_heads / c->kv_heads;
  p.rows = p.group * a->new_tokens;
  p.dim = c->head_dim;
  p.window = a->window;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  const int wm = row_warps(p.rows, p.dim);
  p.row_tiles = (p.rows + 16 * wm - 1) / (16 * wm);
  p.group_div = fast_div((uint32_t)p.group);
  p.head_div = fast_div((uint32_t)p.row_tiles);
  const AttnWs w = attn_ws(sms, wm, dim_class(p.dim));
  if (ws_bytes < w.total) return XCB_ERR_WORKSPACE;
  p.counters = (int32_t*)((uint8_t*)ws + w.counters);
  p.part_ml = (float*)((uint8_t*)ws + w.ml);
  p.part_o = (float*)((uint8_t*)ws + w.o);
  if (c->dtype == XCB_DTYPE_E4M3)
    return a->dtype == XCB_DTYPE_BF16 ? launch_dim<__nv_bfloat16, true>(p, wm, sms, stream)
                                      : launch_dim<__half, true>(p, wm, sms, stream);
  return a->dtype == XCB_DTYPE_BF16 ? launch_dim<__nv_bfloat16, false>(p, wm, sms, stream)
                                    : launch_dim<__half, false>(p, wm, sms, stream);
}

}  // extern "C"
