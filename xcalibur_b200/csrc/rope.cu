// Norms of queries and keys per head, position rotation and the store of keys and values into the paged cache, in
// one pass over the new tokens.
//
// Mathematics: y = x * rsqrt(mean(x^2) + eps) * (w + offset); (a, b) -> (a cos - b sin, b cos + a sin) * mscale for
// each pair of the first rotary_dim values.  The angle is position * f_i.  In 32 bits that product is off by up to
// half a unit in its last place, 4e-3 radians at position 131072; here f_i / (2 pi) is a fraction of 2^64, so the
// product's low 64 bits are the exact fraction of a turn; its leading 32 bits, rounded to a float's 24, give the angle
// within 2^-26 turns (1e-7 radians) at any position.
//
// Bound: HBM for prompts (each value read once and written once; 8192 tokens of 40 heads of 128 move 168 MB in 33.5 us,
// 76% of a copy's rate; 48.3 us into 8 bits, 50%: two divisions a pair of values), latency for a decode step (one token
// 3.7 us, 64 tokens into 8 bits 4.8 us: a round of loads, the page lookup and the stores).  A head is held by D / 8
// lanes, 16 bytes each, so the norm is a few shuffles.  The sines of a token are computed once per block and shared
// through shared memory.
#include <cuda_fp8.h>

#include <type_traits>

#include "kv.cuh"

namespace xcb {
namespace {

constexpr int kThreads = 128;
constexpr float kSmall = 1.17549435e-38f;  // the smallest normal number

struct RopeParams {
  const void* src[3];          // q, k, v
  int64_t tok_stride[3], head_stride[3];
  void* q_out;
  void* k_out;
  int64_t q_out_tok, q_out_head, k_out_tok, k_out_head;
  const void* weight[2];
  const int32_t* positions;
  const int32_t* seqs;
  const uint64_t* turns;
  KvLayer kv;                  // kv.k == null: no cache
  int32_t tokens, heads[3], dim, rot, interleaved, weight_f32;
  int32_t block_tokens, few, groups[3];  // groups: rounds of heads of a kind, where a block takes one
  float eps, weight_offset, mscale;
};

// How a pair's two values lie: half the rotary dimension apart and that a multiple of 8 (partners are whole lanes), side
// by side (in one lane), or any other way (through shared memory).
enum Layout { kLanes, kPairs, kAny };

// Blocks of an SM: 64 registers each thread, or 80 where 64 do not hold the quantiser or the other layouts (kAny spills 12
// to 24 bytes of them even so).
template <bool F8, Layout L>
constexpr int kBlocks = F8 || L != kLanes ? 6 : 8;

// 1 / sqrt(x), x >= 0, within 2^-22; x may be below the normal range if `tiny`: three more instructions, which taken always
// would cost 1 % (a prompt of 8192 tokens 33.9 us instead of 33.5).
__device__ __forceinline__ float rsqrt_fast(float x, bool tiny) {
  float y;
  if (tiny)
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  else
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// LPH lanes hold one head (a power of two with 8 * LPH >= dim); F8: the cache holds e4m3.
//
// Norm and rotation in one form: with r = rsqrt(mean(x^2) + eps), out[d] = r (x[d] A[d] + x[d'] B[d]), d' the other one
// of d's pair, A[d] = w[d] cos, B[d] = +-w[d'] sin.  A lane makes its A and B once for all heads of its token, and
// partners pass between lanes as they were read, two to a word.  Many tokens: blocks stay and walk over batches of up
// to SLOTS tokens, with the weights in shared memory as 32-bit values.  The more tokens a batch has, the more heads use
// a lane's A and B, and the fewer blocks have work: a batch has as many as leave two blocks an SM (1531 tokens of 30
// heads of 80: 7.4 us with four, 9.1 with eight, 8.3 with two; 8192 of 40 of 128: 33.5 us with eight, 36.4 with four).
template <typename T, bool F8, int LPH, Layout L>
__global__ void __launch_bounds__(kThreads, kBlocks<F8, L>) rope_kernel(const __grid_constant__ RopeParams p) {
  constexpr int SLOTS = kThreads / LPH;
  constexpr int NB = 4;                        // heads that a lane reads at once
  __shared__ __align__(16) float s_cos[SLOTS][LPH * 4];
  __shared__ __align__(16) float s_sin[SLOTS][LPH * 4];
  __shared__ __align__(16) float s_w[2][LPH * 8];  // of queries and keys; 1 without a norm
  __shared__ int64_t s_row[SLOTS];             // element offset of the token's row under kv head 0, or -1
  __shared__ float s_x[SLOTS][LPH * 8];        // partners, where a pair is not a multiple of 8 values apart

  const int tid = threadIdx.x;
  const int half = p.rot >> 1;
  const int slot = tid / LPH, d0 = (tid % LPH) * 8;
  const int per_tok = SLOTS / p.block_tokens;  // block_tokens is a power of two <= SLOTS
  const int bt = slot / per_tok;
  // Few tokens: a block has one round of heads of one kind; many: all heads of all kinds.
  const int only = p.few ? (blockIdx.y < p.groups[0] ? 0 : blockIdx.y < p.groups[0] + p.groups[1] ? 1 : 2) : -1;
  const int round = only < 0 ? 0 : blockIdx.y - (only > 0 ? p.groups[0] : 0) - (only > 1 ? p.groups[1] : 0);

  if (only != 2) {
    for (int i = tid; i < 2 * p.dim; i += kThreads) {
      const int k = i >= p.dim, d = i - (k ? p.dim : 0);
      const void* const w = p.weight[k];
      s_w[k][d] = !w ? 1.f
                  : p.weight_f32 ? ((const float*)w)[d] + p.weight_offset
                                 : unpack2<T>(((const uint16_t*)w)[d]).x + p.weight_offset;
    }
  }
  const int lane = tid & 31;
  int partner = lane;
  if (L == kLanes && d0 < p.rot) partner = d0 < half ? lane + half / 8 : lane - half / 8;
  const uint32_t turned = d0 < p.rot ? ~0u : 0u;  // what does not turn adds 0, not 0 * infinity
  const float inv_dim = 1.f / p.dim;
  const auto other = [&](int d) { return d >= p.rot ? d : L == kPairs ? d ^ 1 : d < half ? d + half : d - half; };

  int tok0 = blockIdx.x * p.block_tokens, tok = 0;
  bool live = false;
  // The batch's sines, and where its tokens go.
  const auto prepare = [&]() {
    if (only != 2) {  // values do not turn
      for (int i = tid; i < p.block_tokens * half; i += kThreads) {
        const int b = i / half, j = i - b * half;
        if (tok0 + b < p.tokens) {
          const uint64_t phase = p.turns[j] * (uint64_t)(int64_t)p.positions[tok0 + b];
          float sn, cs;
          sincospif((float)(int32_t)(phase >> 32) * 4.656612873077393e-10f, &sn, &cs);  // 2^-31: turns * 2
          s_cos[b][j] = cs * p.mscale;
          s_sin[b][j] = sn * p.mscale;
        }
      }
    }
    if (p.kv.k && only != 0 && tid < p.block_tokens) {
      int64_t row = -1;
      if (tok0 + tid < p.tokens) {
        const int seq = p.seqs[tok0 + tid], pos = p.positions[tok0 + tid];
        if (seq >= p.kv.max_seqs) {
          atomicOr(p.kv.status, XCB_STATUS_BAD_SEQ);
        } else if (seq >= 0) {
          const int pi = pos >= 0 ? fdiv(pos, p.kv.page_div) : p.kv.max_pages;
          const int page = pi < p.kv.max_pages ? p.kv.table[(int64_t)seq * p.kv.max_pages + pi] : -1;
          if (page < 0 || page >= p.kv.num_pages)
            atomicOr(p.kv.status, XCB_STATUS_BAD_PAGE);
          else
            row = ((int64_t)page * p.kv.kv_heads * p.kv.page_size + (pos - pi * p.kv.page_size)) * p.dim;
        }
      }
      s_row[tid] = row;
    }
  };

  const auto heads_of = [&](auto kind_tag) {
    constexpr int KIND = decltype(kind_tag)::value;  // 0 queries, 1 keys, 2 values
    const int heads = p.heads[KIND];
    const int first = only < 0 ? slot % per_tok : round * SLOTS + slot;
    const int rounds = only < 0 ? (heads + per_tok - 1) / per_tok : 1;  // the same for every lane of a warp
    const T* const src = (const T*)p.src[KIND] + (live ? tok * p.tok_stride[KIND] + d0 : 0);
    const T* at_src = src + first * p.head_stride[KIND];
    const int64_t step = per_tok * p.head_stride[KIND];
    uint4 raw[NB];
    const auto load = [&](int i0) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        raw[b] = make_uint4(0, 0, 0, 0);
        if (live && first + (i0 + b) * per_tok < heads && i0 + b < rounds) raw[b] = *reinterpret_cast<const uint4*>(at_src);
        at_src += step;
      }
    };
    load(0);
    if (KIND == 0 || only > 0) {  // the reads are under way while the sines are computed
      prepare();
      __syncthreads();
    }
    float A[8], B[8];
    if constexpr (KIND < 2) {
      if (d0 < p.dim) {
        const float* const w = s_w[KIND];
        if (d0 >= p.rot) {
#pragma unroll
          for (int j = 0; j < 8; ++j) A[j] = w[d0 + j], B[j] = 0.f;
        } else if constexpr (L == kLanes) {  // eight of one half: their sines, and their partners' weights, lie in a row
          const int i = d0 < half ? d0 : d0 - half, o = d0 < half ? d0 + half : d0 - half;
          const float sign = d0 < half ? -1.f : 1.f;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float4 c = *reinterpret_cast<const float4*>(&s_cos[bt][i + 4 * q]), sn = *reinterpret_cast<const float4*>(&s_sin[bt][i + 4 * q]);
            const float4 a = *reinterpret_cast<const float4*>(w + d0 + 4 * q), e = *reinterpret_cast<const float4*>(w + o + 4 * q);
            A[4 * q] = a.x * c.x, A[4 * q + 1] = a.y * c.y, A[4 * q + 2] = a.z * c.z, A[4 * q + 3] = a.w * c.w;
            B[4 * q] = sign * e.x * sn.x, B[4 * q + 1] = sign * e.y * sn.y;
            B[4 * q + 2] = sign * e.z * sn.z, B[4 * q + 3] = sign * e.w * sn.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int d = d0 + j;
            A[j] = w[d];
            B[j] = 0.f;
            if (d < p.rot) {
              const int i = L == kPairs ? d >> 1 : (d < half ? d : d - half);
              A[j] *= s_cos[bt][i];
              B[j] = w[other(d)] * s_sin[bt][i];
              if (L == kPairs ? !(d & 1) : d < half) B[j] = -B[j];
            }
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) A[j] = B[j] = 0.f;
      }
    }
    T* at_q = (T*)p.q_out + (KIND == 0 ? tok * p.q_out_tok + first * p.q_out_head + d0 : 0);
    const int64_t q_step = per_tok * p.q_out_head;
    const int64_t row = KIND > 0 && p.kv.k && live ? s_row[bt] : -1;
    uint8_t* const plane = p.kv.k + (KIND == 2 ? p.kv.plane : 0);
    for (int i0 = 0; i0 < rounds; i0 += NB) {
      if (i0) load(i0);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (i0 + b >= rounds) break;
        const int h = first + (i0 + b) * per_tok;
        const bool on = live && h < heads;
        const uint32_t w[4] = {raw[b].x, raw[b].y, raw[b].z, raw[b].w};
        uint4 w16 = raw[b];
        float out[8];
        if constexpr (KIND < 2) {
          float x[8], y[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2<T>(w[j]);
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
          }
          if constexpr (L == kPairs) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = d0 + j < p.rot ? x[j ^ 1] : 0.f;
          } else if constexpr (L == kLanes) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = unpack2<T>(__shfl_sync(0xffffffffu, w[j], partner) & turned);
              y[2 * j] = f.x;
              y[2 * j + 1] = f.y;
            }
          } else {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) s_x[slot][d0 + j] = x[j];
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = d0 + j < p.rot ? s_x[slot][other(d0 + j)] : 0.f;
          }
          float r = 1.f;
          if (p.weight[KIND]) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
            for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            r = rsqrt_fast(ss * inv_dim + p.eps, !std::is_same<T, __half>::value && p.eps < kSmall);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) out[j] = r * (x[j] * A[j] + y[j] * B[j]);
          w16 = make_uint4(pack2<T>(out[0], out[1]), pack2<T>(out[2], out[3]), pack2<T>(out[4], out[5]),
                           pack2<T>(out[6], out[7]));
        } else if constexpr (F8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2<T>(w[j]);
            out[2 * j] = f.x;
            out[2 * j + 1] = f.y;
          }
        }
        if constexpr (KIND == 0) {
          if (on) *reinterpret_cast<uint4*>(at_q) = w16;
          at_q += q_step;
        } else {
          if (!on) continue;
          if (KIND == 1 && p.k_out) *reinterpret_cast<uint4*>((T*)p.k_out + tok * p.k_out_tok + h * p.k_out_head + d0) = w16;
          if (row < 0) continue;
          const int64_t at = row + (int64_t)h * p.kv.page_size * p.dim + d0;
          if constexpr (F8) {
            // Quantised from the 32-bit value, not from its 16-bit rounding.  Saturating conversion: infinities become
            // +-448, NaN stays NaN.
            const float* scales = KIND == 2 ? p.kv.v_scale : p.kv.k_scale;
            const float sc = scales ? scales[h] : 1.f;
            uint32_t c[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              c[j] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(out[2 * j], sc), __fdiv_rn(out[2 * j + 1], sc)),
                                              __NV_SATFINITE, __NV_E4M3);
            *reinterpret_cast<uint2*>(plane + at) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
          } else {
            *reinterpret_cast<uint4*>(plane + 2 * at) = w16;
          }
        }
      }
    }
  };
  for (;;) {
    tok = tok0 + bt;
    live = tok < p.tokens && d0 < p.dim;
    if (only <= 0) heads_of(std::integral_constant<int, 0>{});
    if (only < 0 || only == 1) heads_of(std::integral_constant<int, 1>{});
    if (only < 0 || only == 2) heads_of(std::integral_constant<int, 2>{});
    tok0 += gridDim.x * p.block_tokens;
    if (tok0 >= p.tokens) break;
    __syncthreads();  // the batch's sines have been read
  }
}

template <typename T, bool F8, Layout L>
int launch_layout(RopeParams& p, cudaStream_t stream) {
  const int lph = p.dim <= 64 ? 8 : p.dim <= 128 ? 16 : 32;
  const int slots = kThreads / lph;
  const int sms = sm_count();
  if (!sms) return XCB_ERR_CUDA;
  // Few tokens: one head per lane group, so that a call is a single round of loads.  Many: each lane group walks over
  // heads of one token with its A and B in registers, in batches as large as leave two blocks an SM.
  int groups = 0;
  for (int k = 0; k < 3; ++k) groups += p.groups[k] = (p.heads[k] + slots - 1) / slots;
  const bool few = (int64_t)p.tokens * groups <= 8ll * sms && groups <= 65535;
  p.block_tokens = 1;
  p.few = few;
  while (!few && p.block_tokens < slots && p.tokens / (2 * p.block_tokens) >= 2 * sms) p.block_tokens *= 2;
  const int batches = (p.tokens + p.block_tokens - 1) / p.block_tokens;
  const dim3 grid(few || batches < kBlocks<F8, L> * sms ? batches : kBlocks<F8, L> * sms, few ? groups : 1);
  switch (lph) {
    case 8: rope_kernel<T, F8, 8, L><<<grid, kThreads, 0, stream>>>(p); break;
    case 16: rope_kernel<T, F8, 16, L><<<grid, kThreads, 0, stream>>>(p); break;
    default: rope_kernel<T, F8, 32, L><<<grid, kThreads, 0, stream>>>(p); break;
  }
  return cudaGetLastError() == cudaSuccess ? XCB_OK : XCB_ERR_CUDA;
}

template <typename T, bool F8>
int launch(RopeParams& p, cudaStream_t stream) {
  if (p.interleaved) return launch_layout<T, F8, kPairs>(p, stream);
  return p.rot % 16 ? launch_layout<T, F8, kAny>(p, stream) : launch_layout<T, F8, kLanes>(p, stream);
}

bool strides_ok(const void* p, const int64_t* s) { return kv_aligned(p, 16) && s[0] % 8 == 0 && s[1] % 8 == 0; }

}  // namespace
}  // namespace xcb

using namespace xcb;

extern "C" int xcb_qk_norm_rope(const XcbKvCache* c, const XcbRopeArgs* a, cudaStream_t stream) {
  if (!a) return XCB_ERR_INVALID_ARG;
  if (c) {
    const int rc = kv_check(c);
    if (rc != XCB_OK) return rc;
    if (a->layer < 0 || a->layer >= c->layers || a->kv_heads != c->kv_heads || a->head_dim != c->head_dim)
      return XCB_ERR_INVALID_ARG;
    if (c->dtype != XCB_DTYPE_E4M3 && c->dtype != a->dtype) return XCB_ERR_UNSUPPORTED;
  }
  if (a->tokens > 1 << 30) return XCB_ERR_UNSUPPORTED;
  if (a->tokens < 0 || a->q_heads < 0 || a->kv_heads < 0 || a->head_dim <= 0 || a->rotary_dim < 0 ||
      a->rotary_dim > a->head_dim || a->rotary_dim % 2 || !(a->eps >= 0.f))
    return XCB_ERR_INVALID_ARG;
  if (a->dtype != XCB_DTYPE_BF16 && a->dtype != XCB_DTYPE_F16) return XCB_ERR_INVALID_ARG;
  if (a->weight_dtype != a->dtype && a->weight_dtype != XCB_DTYPE_F32) return XCB_ERR_INVALID_ARG;
  if (a->head_dim % 8 || a->head_dim > 256 || a->q_heads > 65536 || a->kv_heads > 65536) return XCB_ERR_UNSUPPORTED;
  if (a->tokens == 0) return XCB_OK;
  const int k_heads = a->k ? a->kv_heads : 0, v_heads = c ? a->kv_heads : 0;
  const int q_heads = a->q ? a->q_heads : 0;
  if (!a->positions || (a->rotary_dim && !a->turns) || (c && (!a->k || !a->v || !a->seqs))) return XCB_ERR_INVALID_ARG;
  if ((q_heads && !a->q_out) || (k_heads && !c && !a->k_out)) return XCB_ERR_INVALID_ARG;
  if (q_heads + k_heads + v_heads == 0) return XCB_OK;
  if ((q_heads && (!strides_ok(a->q, a->q_stride) || !strides_ok(a->q_out, a->q_out_stride))) ||
      (k_heads && !strides_ok(a->k, a->k_stride)) || (v_heads && !strides_ok(a->v, a->v_stride)) ||
      (a->k_out && !strides_ok(a->k_out, a->k_out_stride)) || !kv_aligned(a->q_weight, 16) ||
      !kv_aligned(a->k_weight, 16) || !kv_aligned(a->positions, 4) || !kv_aligned(a->seqs, 4) ||
      !kv_aligned(a->turns, 8))
    return XCB_ERR_INVALID_ARG;
  RopeParams p{};
  p.src[0] = a->q;
  p.src[1] = a->k;
  p.src[2] = a->v;
  p.tok_stride[0] = a->q_stride[0];
  p.tok_stride[1] = a->k_stride[0];
  p.tok_stride[2] = a->v_stride[0];
  p.head_stride[0] = a->q_stride[1];
  p.head_stride[1] = a->k_stride[1];
  p.head_stride[2] = a->v_stride[1];
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  p.q_out_tok = a->q_out_stride[0];
  p.q_out_head = a->q_out_stride[1];
  p.k_out_tok = a->k_out_stride[0];
  p.k_out_head = a->k_out_stride[1];
  p.weight[0] = a->q_weight;
  p.weight[1] = a->k_weight;
  p.positions = a->positions;
  p.seqs = a->seqs;
  p.turns = a->turns;
  if (c) p.kv = kv_layer(c, a->layer);
  p.tokens = a->tokens;
  p.heads[0] = q_heads;
  p.heads[1] = k_heads;
  p.heads[2] = v_heads;
  p.dim = a->head_dim;
  p.rot = a->rotary_dim;
  p.interleaved = a->interleaved != 0;
  p.weight_f32 = a->weight_dtype == XCB_DTYPE_F32;
  // A mean square of f16 values is zero or at least 2^-56, so there an epsilon below the normal range may as well be at its
  // edge: it keeps a head of zeros finite and changes nothing else.
  p.eps = a->dtype == XCB_DTYPE_F16 && a->eps > 0.f && a->eps < kSmall ? kSmall : a->eps;
  p.weight_offset = a->weight_offset;
  p.mscale = a->mscale;
  const bool f8 = c && c->dtype == XCB_DTYPE_E4M3;
  if (a->dtype == XCB_DTYPE_BF16) return f8 ? launch<__nv_bfloat16, true>(p, stream) : launch<__nv_bfloat16, false>(p, stream);
  return f8 ? launch<__half, true>(p, stream) : launch<__half, false>(p, stream);
}
