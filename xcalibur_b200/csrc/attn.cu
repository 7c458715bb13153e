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
// Split: the work is cut into chunks of positions (16 or 32 for each consumer warp) and the list of all chunks (sequence
// by sequence, head by head) into as many equal runs as there are blocks (one or two an SM), found on the device from the
// lengths, so that ragged batches and single long sequences keep every SM busy alike and nothing waits for the host.  A (sequence, head) that lies in
// several runs is joined by a second, small kernel, in run order, so results do not depend on timing; it is launched
// along with the first and waits for it on the device.  (Joined by whichever block came last instead, 37 parts of
// 131072 positions took one SM 7 us behind all others, and every part a fence and an atomic, 1 to 2 us.)
//
// Inside a block four producer warps copy chunk after chunk into a ring of shared-memory stages (cp.async, 16 bytes a
// lane, swizzled so that ldmatrix has no bank conflicts, positions that are not there as zeros) and run ahead over the
// ends of segments; up to eight consumer warps compute.  Consumers are WN groups of WM warps: a group takes its share
// of a chunk's positions, the warps of a group 16 rows each (WM = 1, 2, 4, 8 for up to 128 rows; more rows are several
// tiles, each over the whole range of positions that any row of the sequence sees).  Stages pass between the two by
// mbarriers alone; groups meet at the end of a segment, where the rows' parts are joined.
//
// Measured, 8 query heads a kv head of 128: one sequence of 131072 tokens 51 us (80% of a copy's rate; 55 us on one GPU of
// four), 64 of up to 8192 tokens 49 us (81%), 777 tokens 8.5 us (latency: plan, first stage, join kernel); 8 bits, 128
// sequences 66 us (59%: each value is converted to 16 bits before its tensor step; f16 queries 72.5 us, whose probabilities
// go in two parts); 4 draft tokens of 48 sequences, 20 rows 58 us (45%: 12 of 32 rows of a tile are empty, and
// probabilities go in two parts).  A prompt of 4096 tokens, 4 kv heads, bf16: 3.1 ms, 3% of the dense products' rate for
// what it has to compute, and no less under a window: tiles compute hidden positions too.
//
// mma.sync m16n8k16 rather than tcgen05: with 16 rows a 16-bit chunk asks for an eighth of the former's rate, the rows
// are the M of its step as they are, and its accumulators stay in the registers that the softmax needs them in.  (A
// tcgen05 kernel took 57 / 124 / 223 us for the 131072 tokens, the 64 ragged sequences and the 8-bit ones: 128 rows a
// step, most of them empty, and 10 thousand cycles at each segment's end to bring the sums out of tensor memory.)
//
// Waits are bounded: one that runs out sets XCB_STATUS_DEVICE_TIMEOUT and a flag under which no wait waits and no copy
// is issued any more, and every warp runs to its end.
#include <type_traits>

#include "attn_split.cuh"

namespace xcb {
namespace {

constexpr uint64_t kWaitNs = 2000000000ull;
// Exponentials are taken in base 2 against a reference kLift below a maximum that moves only when a score exceeds it by
// more than kSlack (so the sums are rarely rescaled): up to 2^(kLift + kSlack).  As 32-bit sums and bf16 operands they
// have the same relative accuracy at any size.  An f16 operand has a fixed step below 2^-14, so there the two fill its
// upper range (2^15): a probability loses bits below 2^-25 of the largest one and is gone below 2^-36, e^-25.
template <typename M>
struct Reference {
  static constexpr float kLift = std::is_same<M, __half>::value ? 11.f : 0.f;
  static constexpr float kSlack = std::is_same<M, __half>::value ? 4.f : 8.f;
};

// the rest of the 16 bytes is zeroed; with bytes = 0 nothing is read
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
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
// An 8-bit cache of few rows: two blocks of half the warps, so that one computes while the other joins its warps' parts
// at a segment's end (128 sequences: 85.3 -> 66.3 us).  A 16-bit one is bound by its copies, which then have half the
// stages each: 48.8 -> 57.7 us (64 ragged sequences) with two.
constexpr int blocks_per_sm(bool f8, int dp, int wm) { return f8 && dp < 256 && wm <= 2 ? 2 : 1; }

template <int DP, bool F8, int WM>
struct Shape {
  static constexpr int kBlocks = blocks_per_sm(F8, DP, WM);  // of an SM
  static constexpr int kWarps = DP == 256 || kBlocks == 2 ? 4 : 8;  // consumers
  static constexpr int kProducers = 4;               // registers are given out by four warps: fewer would not free any
  static constexpr int kThreads = (kWarps + kProducers) * 32;
  // Two blocks of an SM start with 128 registers a thread; the consumers take over what the producers do not need.
  static constexpr int kProducerRegs = 56, kConsumerRegs = 200;
  static_assert(kBlocks == 1 || (kWarps == 4 && kProducerRegs + kConsumerRegs == 256), "what the block started with");
  static constexpr int kPitch = DP * (F8 ? 1 : 2);   // bytes of one position's row in shared memory
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kTok = kPitch <= 128 ? 32 : 16;  // positions of a warp's step: 4 to 8 KB of keys and values
  static constexpr int kCh = kTok * kWarps;          // positions of a chunk
  static constexpr int kHalf = kCh * kPitch;         // a stage: its keys, then its values
  static constexpr int kFit = 196608 / kBlocks / (2 * kHalf);
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kRing = kStages * 2 * kHalf;
  static constexpr int kRedPitch = DP + (kBlocks == 2 ? 4 : 8);  // floats
  static constexpr int kSlots = kWarps / 2;
  static constexpr int kRed = kSlots * 16 * kRedPitch * 4;
  static constexpr int kRedMl = kSlots * 16 * 2 * 4;
  static constexpr int kBars = 2 * kStages * 8;
  static constexpr int kMasks = kStages * (kCh / 32) * 4;
  static constexpr int kScalars = 20 * 4;            // sums of the warps, then: place of the run's start, two flags
  static constexpr int kBytes = kRing + kRed + kRedMl + kBars + kMasks + kScalars;
};

// Byte offset of 16-byte chunk c of row r: rows that ldmatrix reads together fall into different banks.
template <int PITCH>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  return r * PITCH + ((PITCH >= 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4);
}

__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {  // when this thread's copies so far have landed
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// A sum that came out as NaN although no score was one: an infinite value that a row sees makes its sum infinite, but the
// tensor steps add it times the second part of a probability too, which may be zero or of either sign.  Such an output is
// marked with a NaN of its own, and the join kernel looks through the values for what it should be.
constexpr uint16_t kMark = 0x7ffe;
template <typename T>
constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;

template <typename T, bool F8, int DP, int WM>
__global__ void __launch_bounds__(Shape<DP, F8, WM>::kThreads, Shape<DP, F8, WM>::kBlocks) attn_kernel(const __grid_constant__ AttnParams p) {
  pdl_launch_dependents();
  using S = Shape<DP, F8, WM>;
  constexpr int NW = S::kWarps, WN = NW / WM, NS = S::kStages;
  constexpr int TOK = S::kTok, SN = TOK / 8;
  constexpr int CH = S::kCh;
  constexpr int RT = 16 * WM;       // rows of a row tile
  constexpr int KS = DP / 16;       // 16-wide steps of the head dimension
  constexpr int NT = DP / 8;        // 8-wide column tiles of the output
  using M = typename std::conditional<F8, __half, T>::type;  // operand type of the tensor steps
  constexpr bool kTwo = !F8 || std::is_same<T, __half>::value;  // probabilities in two parts, see the second product
  static_assert(WM <= NW && CH % 32 == 0, "a group has at most the block's warps");

  extern __shared__ __align__(1024) uint8_t smem[];  // all of the block's shared memory: stages start at multiples of 1 KB
  uint8_t* const ring = smem;
  float* const red = reinterpret_cast<float*>(smem + S::kRing);
  float* const red_ml = reinterpret_cast<float*>(smem + S::kRing + S::kRed);
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + S::kRing + S::kRed + S::kRedMl);
  uint64_t* const empty = full + NS;
  uint32_t* const masks = reinterpret_cast<uint32_t*>(empty + NS);  // [NS][CH / 32]: positions that are there
  int* const s_sum = reinterpret_cast<int*>(masks + NS * (CH / 32));
  int* const s_start = s_sum + 12;  // [3]
  volatile int* const s_dead = s_sum + 16;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + i, S::kProducers * 33);  // every producer lane's copies, and the masks of its warp
      mbar_init(empty + i, NW);
    }
    fence_mbar_init();
    *s_dead = 0;
    p.marked[blockIdx.x] = make_int2(INT32_MAX, -1);
  }
  Run run;
  Seg cs;
  int u_seg;  // the unit of its first segment that the run starts with
  const bool work = plan_run<CH, S::kThreads / 32>(p, TOK, s_sum, s_start, run, cs, &u_seg) &&
                    open_seg<CH>(p, cs, u_seg, run.u1 - run.u0, TOK);
  if (!work) {  // no units, or lead units alone
    if (tid == 0) p.splits[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }

  const auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!*s_dead && !mbar_wait(bar, parity, kWaitNs, p.kv.status)) *s_dead = 1;
    __syncwarp();
  };
  const int row_bytes = p.dim * (F8 ? 1 : 2);

  if (warp >= NW) {
    // ---- producers: 32 positions at a time in turn -----------------------------------------------------------------------
    if constexpr (S::kBlocks == 2) {
      __syncwarp();
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kProducerRegs));
    }
    constexpr int NP = S::kProducers, UN = (CH / 32 + NP - 1) / NP, RPI = 32 / S::kChunks;
    const int me = warp - NW;
    const int lc = lane % S::kChunks, lr = lane / S::kChunks;  // this lane copies 16 bytes at lc of rows lr, lr + RPI, ..
    const int n_lane = lc * 16 < row_bytes ? 16 : 0;
    const uint8_t* const src0 = p.kv.k + (n_lane ? lc * 16 : 0);
    int ci = 0;
    bool more = true;
    // Of position `lane` of each 32 of the chunk to come: its page as read (-2: none wanted), and where in its page and
    // head it lies.  Nothing is made of the page before its chunk's turn: the read is under way meanwhile.
    int page[UN];
    uint32_t within[UN];
    const auto look_up = [&]() {
#pragma unroll
      for (int u = 0; u < UN; ++u) page[u] = -2;
      const int32_t* const row = p.kv.table + (int64_t)cs.row * p.kv.max_pages;
      const int h = fdiv(cs.j, p.head_div);
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int at = (u * NP + me) * 32, pos = cs.t0 + ci * CH + at + lane;
        if (at < CH && pos >= cs.lo && pos < cs.t1) {
          const int pi = fdiv(pos, p.kv.page_div);
          page[u] = row[pi];
          within[u] = (uint32_t)h * p.kv.page_size + (pos - pi * p.kv.page_size);
        }
      }
      if (++ci == cs.c1 - cs.c0) {
        more = next_seg<CH>(p, cs, TOK);
        ci = 0;
      }
    };
    const uint32_t page_rows = (uint32_t)p.kv.kv_heads * p.kv.page_size;
    look_up();
    int stage = 0;
    uint32_t parity = 1;  // the first round finds the stages empty
    for (;;) {
      uint32_t cur[UN];  // row in the layer's keys, or ~0
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const bool there = (uint32_t)page[u] < (uint32_t)p.kv.num_pages;
        if (!there && page[u] != -2) atomicOr(p.kv.status, XCB_STATUS_BAD_PAGE);
        cur[u] = there ? (uint32_t)page[u] * page_rows + within[u] : 0xffffffffu;
      }
      const bool again = more;
      if (again) look_up();
      wait(empty + stage, parity);
      if (!*s_dead) {
        const uint32_t dst0 = smem_u32(ring) + stage * (2 * S::kHalf);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          const int r0 = (u * NP + me) * 32;
          if (r0 >= CH) break;
          const uint32_t mask = __ballot_sync(0xffffffffu, cur[u] != 0xffffffffu);
          if (lane == 0) masks[stage * (CH / 32) + r0 / 32] = mask;
#pragma unroll 8
          for (int i = 0; i < 32 / RPI; ++i) {
            const int r = lr + i * RPI;
            const uint32_t at = __shfl_sync(0xffffffffu, cur[u], r);
            const bool in = at != 0xffffffffu;
            const uint8_t* const src = src0 + (in ? (uint64_t)at * (uint32_t)row_bytes : 0ull);
            const uint32_t dst = dst0 + swz<S::kPitch>(r0 + r, lc);
            cp_async16(dst, src, in ? n_lane : 0);
            cp_async16(dst + S::kHalf, src + p.kv.plane, in ? n_lane : 0);
          }
        }
      }
      cp_async_arrive(full + stage);
      __syncwarp();
      if (lane == 0) mbar_arrive(full + stage);
      if (!again) break;
      if (++stage == NS) {
        stage = 0;
        parity ^= 1;
      }
    }
    cp_async_wait_all();
    return;
  }

  // ---- consumers -----------------------------------------------------------------------------------------------------
  const int grp = warp / WM, wm = warp % WM;
  const int g = lane >> 2, t = lane & 3;
  if constexpr (S::kBlocks == 2) {
    __syncwarp();
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kConsumerRegs));
  }
  const int cta = blockIdx.x;
  // ldmatrix row addresses of this lane: keys as (position, dimension) pairs, values transposed
  const uint32_t k_lane = swz<S::kPitch>((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
  const uint32_t v_lane = swz<S::kPitch>(lane & 15, lane >> 4);
  const auto block_sync = [&]() {
    __syncwarp();
    named_bar(1, NW * 32);
  };

  // This lane's two rows of the warp's 16, as they lie in memory.
  uint32_t qf[KS][4];
  const auto load_q = [&](const Seg& sg) {
    const int h = fdiv(sg.j, p.head_div), tile0 = (sg.j - h * p.row_tiles) * RT;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = tile0 + wm * 16 + g + 8 * i;
      const bool in = r < p.rows;
      const int l = in ? fdiv(r, p.group_div) : 0;
      const T* const q = (const T*)p.q + (in ? sg.b * p.q_b + l * p.q_t + (h * p.group + r - l * p.group) * p.q_h : 0);
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        if constexpr (F8) {
          // a step's contraction index runs over d = 4t, 4t+1 | 4t+2, 4t+3: the four codes a lane gets of a row
          uint2 v = make_uint2(0, 0);
          if (in && kk * 16 < p.dim) v = *reinterpret_cast<const uint2*>(q + kk * 16 + 4 * t);
          qf[kk][i] = v.x;
          qf[kk][2 + i] = v.y;
        } else {
          qf[kk][i] = in && kk * 16 < p.dim ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + 2 * t) : 0u;
          qf[kk][2 + i] = in && kk * 16 + 8 < p.dim ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + 8 + 2 * t) : 0u;
        }
      }
    }
  };
  // Operands of the tensor steps from the rows, and the factors of their scores.
  const auto make_q = [&](int h, float (&to_log2)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      to_log2[i] = p.scale_log2;
      if constexpr (F8) {
        if (p.kv.k_scale) to_log2[i] *= p.kv.k_scale[h];
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          // bf16 queries as f16: scaled by a power of two that brings the row's largest value to [2^14, 2^15), exact
          // down to 2^-38 of that value.
          float top = 0.f;
#pragma unroll
          for (int kk = 0; kk < KS; ++kk) {
            const float2 a = unpack2<T>(qf[kk][i]), b = unpack2<T>(qf[kk][2 + i]);
            top = fmaxf(fmaxf(top, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(b.x), fabsf(b.y)));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int ex = (int)(__float_as_uint(top) >> 23);                // biased exponent, 255: not finite
          const int up = ex == 0 || ex == 255 ? 0 : max(-120, min(120, 127 + 14 - ex));
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
    // Scores are multiplied by to_log2 after the maximum is taken, so it is made positive (and never zero: -inf stays).  A
    // NaN stays one.
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
      if (to_log2[i] < 1e-37f) to_log2[i] = 1e-37f;
    }
  };
  // With an 8-bit cache the operands stay in shared memory, in the lanes' order, for all groups (in the join's buffer,
  // which is free between joins): the registers are needed for the keys' and values' conversions.
  uint4* const q_frag = reinterpret_cast<uint4*>(red);  // [WM][KS][32]
  static_assert(!F8 || WM * KS * 512 <= S::kRed, "the join's buffer holds the queries");
  if (!F8 || grp == 0) load_q(cs);

  int stage = 0;
  uint32_t parity = 0;
  int unit = run.u0 - u_seg + p.lead + cs.c0;  // the list's index of the segment's first chunk here
  int part_slot = 2 * cta;
  int4 split = make_int4(-1, 0, 0, 0);
  for (;;) {
    const int h = fdiv(cs.j, p.head_div), tile0 = (cs.j - h * p.row_tiles) * RT;
    // positions that this lane's two rows see
    int hi[2], lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = tile0 + wm * 16 + g + 8 * i;
      hi[i] = cs.len;
      lo[i] = 0;
      if (p.new_tokens > 1 && r < p.rows) {
        hi[i] = cs.len - p.new_tokens + fdiv(r, p.group_div) + 1;
        lo[i] = p.window && hi[i] > p.window ? hi[i] - p.window : 0;
      }
    }
    float to_log2[2];
    if constexpr (F8) {
      if constexpr (WN > 1) block_sync();  // the join has been read
      if (grp == 0) {
        make_q(h, to_log2);
        uint4* const dst = q_frag + wm * KS * 32 + lane;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) dst[kk * 32] = make_uint4(qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
        if (t == 0) {
          red_ml[wm * 16 + g] = to_log2[0];
          red_ml[wm * 16 + g + 8] = to_log2[1];
        }
      }
      if constexpr (WN > 1) {
        block_sync();
        to_log2[0] = red_ml[wm * 16 + g];
        to_log2[1] = red_ml[wm * 16 + g + 8];
      } else {
        __syncwarp();
      }
    } else {
      make_q(h, to_log2);
    }
    float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

    const int n_chunks = cs.c1 - cs.c0;
    for (int ci = 0; ci < n_chunks; ++ci) {
      wait(full + stage, parity);
      const uint8_t* const base0 = ring + stage * (2 * S::kHalf);
#pragma unroll 1
      for (int sub = 0; sub < WM; ++sub) {
        const int first = (grp * WM + sub) * TOK;  // of the chunk's positions
        const uint32_t word = masks[stage * (CH / 32) + first / 32];
        const uint32_t vm = TOK == 32 ? word : (word >> (first & 31)) & 0xffffu;
        if (!vm) continue;
        const uint8_t* const base = base0 + first * S::kPitch;  // values: kHalf further
        const uint32_t kb = smem_u32(base), vb = kb + S::kHalf;
        const int pos0 = cs.t0 + ci * CH + first;
        float s[SN][4];
#pragma unroll
        for (int n = 0; n < SN; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        // the swizzle again: chunk 2 kk + cc of the lane's row is the lane's address xor 32 kk
        if constexpr (F8) {
          const uint4* const q_lane = q_frag + wm * KS * 32 + lane;
#pragma unroll
          for (int k2 = 0; k2 < KS / 2; ++k2) {
            const uint4 qa = q_lane[2 * k2 * 32], qb = q_lane[(2 * k2 + 1) * 32];
#pragma unroll
            for (int b = 0; b < SN / 2; ++b) {
              uint32_t w[4];
              ldsm4(w, (kb + k_lane + b * 16 * S::kPitch) ^ (k2 << 5));
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                  uint32_t b0, b1;
                  e4m3_f16(w[2 * n], b0, b1);
                  mma16<M>(s[2 * b + n], {qa.x, qa.y, qa.z, qa.w}, b0, b1);
                  e4m3_f16(w[2 * n + 1], b0, b1);
                  mma16<M>(s[2 * b + n], {qb.x, qb.y, qb.z, qb.w}, b0, b1);
              }
            }
          }
        } else {
#pragma unroll
          for (int b = 0; b < SN / 2; ++b) {
            const uint32_t ka = kb + k_lane + b * 16 * S::kPitch;
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
        // m is the reference that sums and exponentials are taken against, not the maximum itself.
        constexpr float kLift = Reference<M>::kLift, kRise = kLift + Reference<M>::kSlack;
        if (__any_sync(0xffffffffu, mx[0] > m[0] + kRise || mx[1] > m[1] + kRise)) {
          float a[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float top = fmaxf(m[i], mx[i] - kLift);
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
          for (int i = lane; i < TOK * S::kPitch / 16; i += 32) {
            const uint4 v4 = reinterpret_cast<const uint4*>(base + S::kHalf)[i];
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
                const uint8_t* at = base + S::kHalf + swz<S::kPitch>(col, byte >> 4) + (byte & 15);
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
        // The probabilities as operands.  Rounded once to their type they would add an error as large as the output's own
        // rounding; a second operand carries the rest: 2^-16 of a probability is left in bf16, 2^-22 in f16 (2^-36 of the
        // largest one where that is more).  bf16 queries over an 8-bit cache alone take one part: its f16 has three bits
        // more than their output, whose error against 64 bits it raises from 0.001657 to 0.001664, and two parts take
        // 73.1 us instead of 66.4 (128 sequences).  With f16 queries it would be 0.00026 instead of 0.00021, for the same
        // tenth of the time.
#pragma unroll
        for (int b = 0; b < SN / 2; ++b) {
          uint32_t a_hi[4], a_lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = s[2 * b + (i >> 1)][2 * (i & 1)], y = s[2 * b + (i >> 1)][2 * (i & 1) + 1];
            a_hi[i] = pack2<M>(x, y);
            if constexpr (kTwo) {
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
                if constexpr (kTwo) {
                  mma16<M>(o[4 * n2 + 2 * e], a_lo, b0, b1);
                  mma16<M>(o[4 * n2 + 2 * e + 1], a_lo, c0, c1);
                }
              } else {
                mma16<M>(o[2 * n2 + e], a_hi, w[2 * e], w[2 * e + 1]);
                mma16<M>(o[2 * n2 + e], a_lo, w[2 * e], w[2 * e + 1]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + stage);
      if (++stage == NS) {
        stage = 0;
        parity ^= 1;
      }
    }
    Seg nx = cs;
    const bool more = next_seg<CH>(p, nx, TOK);

    // ---- join the block's groups and write -----------------------------------------------------------------------------
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    const bool whole = cs.c0 == 0 && cs.c1 == cs.nch;
    const float vs = F8 && p.kv.v_scale ? p.kv.v_scale[h] : 1.f;
    const int nrows = min(RT, p.rows - tile0);
    const auto place = [&](int r) {  // of row r of the kv head in the output
      const int tok = fdiv(r, p.group_div);
      return ((int64_t)cs.b * p.new_tokens + tok) * p.q_heads + h * p.group + r - tok * p.group;
    };
    const auto mark = [&](T* at, float x, float y) {
      uint16_t* const to = reinterpret_cast<uint16_t*>(at);
      if (isnan(x)) to[0] = kMark;
      if (isnan(y)) to[1] = kMark;
      const int seg = cs.b * p.kv.kv_heads * p.row_tiles + cs.j;
      atomicMin(&p.marked[cta].x, seg);
      atomicMax(&p.marked[cta].y, seg);
    };
    // A warp's part in a slot of the join buffer: rows of kRedPitch floats in the natural order of the dimensions, which
    // an 8-bit cache's accumulators hold four by four.
    const auto put = [&](int slot_) {
      float* const dst = red + slot_ * 16 * S::kRedPitch;
      float* const ml = red_ml + slot_ * 32;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float* const at = dst + (g + 8 * i) * S::kRedPitch;
        if (t == 0) *reinterpret_cast<float2*>(ml + 2 * (g + 8 * i)) = make_float2(m[i], l[i]);
        if constexpr (F8) {
#pragma unroll
          for (int n = 0; n < NT; n += 2)
            *reinterpret_cast<float4*>(at + n * 8 + 4 * t) =
                make_float4(o[n][2 * i], o[n + 1][2 * i], o[n][2 * i + 1], o[n + 1][2 * i + 1]);
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(at + n * 8 + 2 * t) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        }
      }
    };
    if constexpr (WN > 1) {
      // the upper half of the groups into the lower half's registers, these into the buffer, and all warps from there
      constexpr int HG = WN / 2;
      block_sync();
      if (grp >= HG) put((grp - HG) * WM + wm);
      block_sync();
      if (grp < HG) {
        const float* const src = red + (grp * WM + wm) * 16 * S::kRedPitch;
        const float* const ml = red_ml + (grp * WM + wm) * 32;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float* const at = src + (g + 8 * i) * S::kRedPitch;
          const float2 other = *reinterpret_cast<const float2*>(ml + 2 * (g + 8 * i));
          const float top = fmaxf(m[i], other.x);
          const float a = ex2_diff(m[i], top), b = ex2_diff(other.x, top);
          m[i] = top;
          l[i] = l[i] * a + other.y * b;
          if constexpr (F8) {
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
              const float4 v = *reinterpret_cast<const float4*>(at + n * 8 + 4 * t);
              o[n][2 * i] = o[n][2 * i] * a + v.x * b;
              o[n + 1][2 * i] = o[n + 1][2 * i] * a + v.y * b;
              o[n][2 * i + 1] = o[n][2 * i + 1] * a + v.z * b;
              o[n + 1][2 * i + 1] = o[n + 1][2 * i + 1] * a + v.w * b;
            }
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float2 v = *reinterpret_cast<const float2*>(at + n * 8 + 2 * t);
              o[n][2 * i] = o[n][2 * i] * a + v.x * b;
              o[n][2 * i + 1] = o[n][2 * i + 1] * a + v.y * b;
            }
          }
        }
        __syncwarp();
        put(grp * WM + wm);  // over what this warp alone has read
      }
      if (more && (!F8 || grp == 0)) load_q(nx);  // under way while the parts are joined
      block_sync();
      constexpr int V = DP / 4;  // threads of a row, four dimensions each
      for (int x = tid; x < nrows * V; x += NW * 32) {
        const int rl = x / V, d = (x - rl * V) * 4;
        const int w0 = rl >> 4, rr = rl & 15;  // the warp of a group that had the row
        float top = -INFINITY;
#pragma unroll
        for (int q = 0; q < HG; ++q) top = fmaxf(top, red_ml[(q * WM + w0) * 32 + 2 * rr]);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int q = 0; q < HG; ++q) {
          const float2 ml = *reinterpret_cast<const float2*>(red_ml + (q * WM + w0) * 32 + 2 * rr);
          const float4 v = *reinterpret_cast<const float4*>(red + ((q * WM + w0) * 16 + rr) * S::kRedPitch + d);
          const float a = ex2_diff(ml.x, top);
          sum += a * ml.y;
          acc.x += a * v.x;
          acc.y += a * v.y;
          acc.z += a * v.z;
          acc.w += a * v.w;
        }
        if (whole) {
          const int64_t at = place(tile0 + rl);
          const float inv = sum == 0.f ? 0.f : vs / sum;
          if (d < p.dim) {
            T* const dst = (T*)p.out + at * p.dim + d;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
            if (!F8 && isnan(acc.x + acc.y + acc.z + acc.w) && !isnan(sum)) {
              mark(dst, acc.x, acc.y);
              mark(dst + 2, acc.z, acc.w);
            }
          }
          if (p.lse && d == 0) p.lse[at] = sum == 0.f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
        } else {
          *reinterpret_cast<float4*>(p.part_o + ((int64_t)part_slot * RT + rl) * DP + d) = acc;
          if (d == 0) *reinterpret_cast<float2*>(p.part_ml + ((int64_t)part_slot * RT + rl) * 2) = make_float2(top, sum);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rl = wm * 16 + g + 8 * i;
        if (rl >= nrows) continue;
        const int64_t at = place(tile0 + rl);
        const float mul = !whole ? 1.f : l[i] == 0.f ? 0.f : vs / l[i];
        T* const dst = (T*)p.out + at * p.dim;
        float* const po = p.part_o + ((int64_t)part_slot * RT + rl) * DP;
        if (t == 0) {
          if (!whole)
            *reinterpret_cast<float2*>(p.part_ml + ((int64_t)part_slot * RT + rl) * 2) = make_float2(m[i], l[i]);
          else if (p.lse)
            p.lse[at] = l[i] == 0.f ? -INFINITY : m[i] * 0.6931471805599453f + logf(l[i]);
        }
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          // two column tiles: dimensions 16 (n / 2) .. + 15
          if constexpr (F8) {
            const int d = n * 8 + 4 * t;
            const float4 v = make_float4(o[n][2 * i] * mul, o[n + 1][2 * i] * mul, o[n][2 * i + 1] * mul, o[n + 1][2 * i + 1] * mul);
            if (!whole)
              *reinterpret_cast<float4*>(po + d) = v;
            else if (d < p.dim)
              *reinterpret_cast<uint2*>(dst + d) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = (n + e) * 8 + 2 * t;
              const float x = o[n + e][2 * i] * mul, y = o[n + e][2 * i + 1] * mul;
              if (!whole)
                *reinterpret_cast<float2*>(po + d) = make_float2(x, y);
              else if (d < p.dim) {
                *reinterpret_cast<uint32_t*>(dst + d) = pack2<T>(x, y);
                if (isnan(x + y) && !isnan(l[i])) mark(dst + d, x, y);
              }
            }
          }
        }
      }
    }
    if (WN == 1 && more) load_q(nx);
    if (!whole && cs.c0 == 0) split = split_of(run, cs, unit, part_slot);
    if (!more) break;
    unit += cs.nch - cs.c0 + p.lead;
    part_slot = 2 * cta + 1;
    cs = nx;
  }
  if (tid == 0) p.splits[cta] = split;
}

// Puts what they should be in the place of the marks in a segment's outputs (a warp a row, W dimensions a lane, as the
// join): weights are positive, so infinite values of one sign are the result, values of both signs or a NaN among them
// make it NaN.  The warp reads the columns of one lane's dimensions at a time, 128 positions a round: a path for values that
// are broken already (one infinite value under 131072 tokens: 3.8 ms instead of 0.05).
template <typename T, int W>
__device__ __noinline__ void mend(const AttnParams& p, int rt, int b, int j) {
  const int h = fdiv(j, p.head_div), tile0 = (j - h * p.row_tiles) * rt, lane = threadIdx.x & 31;
  int seq, first;
  const int len = visible(p, b, &seq, &first);
  for (int r = tile0 + blockIdx.y * 8 + (threadIdx.x >> 5); r < min(tile0 + rt, p.rows); r += gridDim.y * 8) {
    const int tok = fdiv(r, p.group_div);
    const int64_t place = ((int64_t)b * p.new_tokens + tok) * p.q_heads + h * p.group + r - tok * p.group;
    uint16_t* const out = (uint16_t*)p.out + place * p.dim;
    uint32_t mine = 0;  // a bit a dimension
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (lane * W < p.dim && out[lane * W + w] == kMark) mine |= 1u << w;
    const int end = len - p.new_tokens + tok + 1, from = p.window && end > p.window ? end - p.window : 0;
    for (uint32_t todo = __ballot_sync(0xffffffffu, mine != 0); todo; todo &= todo - 1) {
      const int who = __ffs(todo) - 1;
      const uint32_t want = __shfl_sync(0xffffffffu, mine, who);
      uint32_t seen = 0;  // +inf, -inf and NaN, 8 bits each
      for (int pos0 = from; pos0 < end; pos0 += 128) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int pos = pos0 + u * 32 + lane;
          if (pos >= end) continue;
          const int pi = fdiv(pos, p.kv.page_div);
          const int page = p.kv.table[(int64_t)seq * p.kv.max_pages + pi];
          if (page < 0 || page >= p.kv.num_pages) continue;
          const int64_t at = ((int64_t)page * p.kv.kv_heads + h) * p.kv.page_size + (pos - pi * p.kv.page_size);
          const uint16_t* const v = reinterpret_cast<const uint16_t*>(p.kv.k + p.kv.plane) + at * p.dim + who * W;
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const uint32_t x = v[w], size = x & 0x7fffu;
            if (size >= kInf<T>) seen |= 1u << (w + (size > kInf<T> ? 16 : x >> 15 ? 8 : 0));
          }
        }
        seen = __reduce_or_sync(0xffffffffu, seen);
        if (((seen >> 16 | (seen & seen >> 8)) & want) == want) break;
      }
      if (lane != who) continue;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t up = seen >> w & 1, down = seen >> (w + 8) & 1, nan = seen >> (w + 16) & 1;
        if (want >> w & 1) out[lane * W + w] = !nan && up != down ? (uint16_t)(kInf<T> | down << 15) : 0x7fff;
      }
    }
  }
}

// Joins the parts of the split segment that block blockIdx.x of attn_kernel began, if it did: a warp takes a row at a
// time, a lane DP / 32 dimensions, parts in run order.  And mends the outputs that the block marked.  Bound: latency, two
// or a few rounds of reads.  Two blocks an SM, of which a call has up to 2368: as many parts are read at once as that leaves
// registers for (verification 58.4 us; with 64 values a lane it spills, 59.9, or has one block an SM, 61.7).
template <typename T, bool F8, int DP>
__global__ void __launch_bounds__(256, 2) join_kernel(const __grid_constant__ AttnParams p, int rt) {
  constexpr int W = DP / 32, U = W == 8 ? 4 : 8;  // parts whose rows are read at once
  pdl_wait();
  const int4 sp = p.splits[blockIdx.x];
  if constexpr (!F8) {
    const int2 marked = p.marked[blockIdx.x];
    const int heads = p.kv.kv_heads * p.row_tiles;
    for (int seg = marked.x; seg <= marked.y; ++seg) mend<T, W>(p, rt, seg / heads, seg % heads);
  }
  if (sp.x < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bool odd = false;
  const int first = blockIdx.x, parts = sp.z - first + 1;
  const int h = fdiv(sp.y, p.head_div), tile0 = (sp.y - h * p.row_tiles) * rt;
  const int nrows = min(rt, p.rows - tile0);
  const float vs = p.kv.v_scale ? p.kv.v_scale[h] : 1.f;
  const auto slot_of = [&](int i) { return i == 0 ? sp.w : 2 * (first + i); };
  for (int rl = blockIdx.y * 8 + warp; rl < nrows; rl += gridDim.y * 8) {
    float top = -INFINITY, sum = 0.f, acc[W];
#pragma unroll
    for (int w = 0; w < W; ++w) acc[w] = 0.f;
    const float* const row_ml = p.part_ml + rl * 2;
    const float* const row_o = p.part_o + (int64_t)rl * DP + lane * W;
    for (int q0 = 0; q0 < parts; q0 += 32) {
      float2 ml = make_float2(-INFINITY, 0.f);
      if (q0 + lane < parts) ml = *reinterpret_cast<const float2*>(row_ml + (int64_t)slot_of(q0 + lane) * rt * 2);
      const int n = min(32, parts - q0);
      float wt = 0.f;
      for (int q = 0; q < n; q += U) {
        float v[U][W];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (q + u < n) {
            const float* const src = row_o + (int64_t)slot_of(q0 + q + u) * rt * DP;
            if constexpr (W == 2) {
              *reinterpret_cast<float2*>(v[u]) = *reinterpret_cast<const float2*>(src);
            } else {
#pragma unroll
              for (int w = 0; w < W; w += 4)
                *reinterpret_cast<float4*>(v[u] + w) = *reinterpret_cast<const float4*>(src + w);
            }
          }
        }
        if (q == 0) {  // the maxima of these 32 parts; what came before is scaled to the new one
          float now = ml.x;
#pragma unroll
          for (int s = 16; s; s >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, s));
          now = fmaxf(now, top);
          const float scale = ex2_diff(top, now);
          wt = ex2_diff(ml.x, now);
          top = now;
          sum = sum * scale + wt * ml.y;
#pragma unroll
          for (int w = 0; w < W; ++w) acc[w] *= scale;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float wq = __shfl_sync(0xffffffffu, wt, (q + u) & 31);
          if (q + u < n) {
#pragma unroll
            for (int w = 0; w < W; ++w) acc[w] += wq * v[u][w];
          }
        }
      }
    }
#pragma unroll
    for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const int r = tile0 + rl, tok = fdiv(r, p.group_div);
    const int64_t at = ((int64_t)sp.x * p.new_tokens + tok) * p.q_heads + h * p.group + r - tok * p.group;
    const float inv = sum == 0.f ? 0.f : vs / sum;
    T* const dst = (T*)p.out + at * p.dim + lane * W;
#pragma unroll
    for (int w = 0; w < W; w += 2)
      if (lane * W + w < p.dim) *reinterpret_cast<uint32_t*>(dst + w) = pack2<T>(acc[w] * inv, acc[w + 1] * inv);
    if constexpr (!F8) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (!isnan(acc[w]) || isnan(sum) || lane * W >= p.dim) continue;
        reinterpret_cast<uint16_t*>(dst)[w] = kMark;
        odd = true;
      }
    }
    if (p.lse && lane == 0) p.lse[at] = sum == 0.f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
  }
  if (__any_sync(0xffffffffu, odd)) mend<T, W>(p, rt, sp.x, sp.y);
}

// ------------------------------------------------------------------------------------------------ host side
int dim_class(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Warps that share a tile: enough for all rows of a kv head, so that its keys and values are read once.
int row_warps(int rows, int dim) {
  const int most = dim_class(dim) < 256 ? 8 : 4;
  int wm = 1;
  while (wm < most && 16 * wm < rows) wm *= 2;
  return wm;
}

struct AttnWs {
  size_t splits, marked, ml, o, total;
};
AttnWs attn_ws(int sms, int wm, int dp) {
  AttnWs w;
  w.splits = 0;
  w.marked = (size_t)sms * 16;
  w.ml = (w.marked + (size_t)sms * 8 + 255) / 256 * 256;
  w.o = w.ml + ((size_t)2 * sms * 16 * wm * 8 + 255) / 256 * 256;
  w.total = w.o + (size_t)2 * sms * 16 * wm * dp * 4;
  return w;
}

template <typename T, bool F8, int DP, int WM>
int launch(const AttnParams& p, int sms, cudaStream_t stream) {
  using S = Shape<DP, F8, WM>;
  constexpr int bytes = S::kBytes;
  static_assert(S::kBlocks * (bytes + 1024) <= 228 * 1024, "the stages fit one SM");
  sms *= S::kBlocks;  // from here on blocks
  static bool ready[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return XCB_ERR_CUDA;
  if (dev >= kMaxDevices || !ready[dev]) {
    if (cudaFuncSetAttribute(attn_kernel<T, F8, DP, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess)
      return XCB_ERR_CUDA;
    // A block that started with fewer registers (given out eight a thread at a time) than its warps come to hold would wait
    // for more without end.  The build checks what the compiler gave.
    if (S::kBlocks == 2) {
      cudaFuncAttributes at{};
      if (cudaFuncGetAttributes(&at, attn_kernel<T, F8, DP, WM>) != cudaSuccess) return XCB_ERR_CUDA;
      if ((at.numRegs + 7) / 8 * 8 * (S::kThreads / 32) < S::kWarps * S::kConsumerRegs + S::kProducers * S::kProducerRegs)
        return XCB_ERR_UNSUPPORTED;
    }
    if (dev < kMaxDevices) ready[dev] = true;
  }
  attn_kernel<T, F8, DP, WM><<<sms, S::kThreads, bytes, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return XCB_ERR_CUDA;
  // the join is launched along with it and waits on the device for its end
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  const int rt = 16 * WM;
  cfg.gridDim = dim3(sms, (unsigned)((p.rows < rt ? p.rows : rt) + 7) / 8);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<T, F8, DP>, p, rt) == cudaSuccess ? XCB_OK : XCB_ERR_CUDA;
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

AttnWs ws_of(const XcbKvCache* c, int sms, int rows) {
  const int wm = row_warps(rows, c->head_dim), dp = dim_class(c->head_dim);
  return attn_ws(sms * blocks_per_sm(c->dtype == XCB_DTYPE_E4M3, dp, wm), wm, dp);
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
  return sms ? ws_of(c, sms, q_heads / c->kv_heads * new_tokens).total : 0;
}

// A call writes every record and part of its workspace before the join reads it.
int xcb_attn_workspace_init(void* ws, size_t, cudaStream_t) { return ws ? XCB_OK : XCB_ERR_INVALID_ARG; }

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
  // What a segment's ends cost in chunks.  64 ragged sequences, 8 rows: 51.9 / 49.0 / 49.6 / 50.5 us with 1 / 2 / 3 / 4.
  // With more rows a chunk itself costs more: 4 draft tokens of 48 sequences, 20 rows: 59.1 / 59.8 / 62.1 with 1 / 2 / 3.
  // Where an SM has two blocks, a chunk is half as long: 128 sequences in 8 bits, 8 rows: 72.8 / 66.4 / 67.6 / 70.4 with 2 /
  // 3 / 4 / 5.
  p.lead = (p.rows <= 16 ? 2 : 1) + blocks_per_sm(c->dtype == XCB_DTYPE_E4M3, dim_class(p.dim), wm) - 1;
  p.group_div = fast_div((uint32_t)p.group);
  p.head_div = fast_div((uint32_t)p.row_tiles);
  // a row of a layer's keys has a 32-bit index, the list of chunks a 31-bit one
  if ((int64_t)c->num_pages * c->kv_heads * c->page_size >= (1ll << 32) - 1 ||
      (int64_t)a->batch * c->kv_heads * p.row_tiles * ((int64_t)c->max_pages * c->page_size / 64 + 1 + p.lead) >= 1ll << 31)
    return XCB_ERR_UNSUPPORTED;
  const AttnWs w = ws_of(c, sms, p.rows);
  if (ws_bytes < w.total) return XCB_ERR_WORKSPACE;
  p.splits = (int4*)((uint8_t*)ws + w.splits);
  p.marked = (int2*)((uint8_t*)ws + w.marked);
  p.part_ml = (float*)((uint8_t*)ws + w.ml);
  p.part_o = (float*)((uint8_t*)ws + w.o);
  if (c->dtype == XCB_DTYPE_E4M3)
    return a->dtype == XCB_DTYPE_BF16 ? launch_dim<__nv_bfloat16, true>(p, wm, sms, stream)
                                      : launch_dim<__half, true>(p, wm, sms, stream);
  return a->dtype == XCB_DTYPE_BF16 ? launch_dim<__nv_bfloat16, false>(p, wm, sms, stream)
                                    : launch_dim<__half, false>(p, wm, sms, stream);
}

}  // extern "C"
