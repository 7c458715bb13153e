// Norms of queries and keys per head, position rotation and the store of keys and values into the paged cache, in
// one pass over the new tokens.
//
// Mathematics: y = x * rsqrt(mean(x^2) + eps) * (w + offset); (a, b) -> (a cos - b sin, b cos + a sin) * mscale for
// each pair of the first rotary_dim values.  The angle is position * f_i.  In 32 bits that product is off by up to
// half a unit in its last place, 4e-3 radians at position 131072; here f_i / (2 pi) is a fraction of 2^64, so the
// product's low 64 bits are the exact fraction of a turn, and its leading 32 bits give the angle to 2^-32 turns at
// any position.
//
// Bound: HBM (each value read once and written once).  A head is held by D / 8 lanes, 16 bytes each, so the norm is a
// few shuffles; a lane keeps its 8 cosines, sines and weights in registers for all heads of its token.  The sines of
// a token are computed once per block and shared through shared memory.
#include <cuda_fp8.h>

#include "kv.cuh"

namespace xcb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTok = 4;     // tokens per block
constexpr int kMaxHalf = 128;  // rotary_dim / 2

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
  int32_t block_tokens, block_heads;
  float eps, weight_offset, mscale;
};

// LPH lanes hold one head (a power of two with 8 * LPH >= dim); F8: the cache holds e4m3.
template <typename T, bool F8, int LPH>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeParams p) {
  constexpr int SLOTS = kThreads / LPH;
  __shared__ float s_cos[kMaxTok][kMaxHalf];
  __shared__ float s_sin[kMaxTok][kMaxHalf];
  __shared__ int64_t s_row[kMaxTok];           // element offset of the token's row under kv head 0, or -1
  __shared__ float s_x[SLOTS][LPH * 8];        // partners, where a pair is not 8 values apart

  const int tid = threadIdx.x;
  const int half = p.rot >> 1;
  const int tok0 = blockIdx.x * p.block_tokens;
  const int slot = tid / LPH, ln = tid % LPH, d0 = ln * 8;
  const int per_tok = SLOTS / p.block_tokens;  // block_tokens is a power of two <= kMaxTok <= SLOTS
  const int bt = slot / per_tok;
  const int tok = tok0 + bt;
  const int nheads = p.heads[0] + p.heads[1] + p.heads[2];
  const int h_begin = blockIdx.y * p.block_heads + slot % per_tok;
  const int h_end = min(nheads, (int)(blockIdx.y + 1) * p.block_heads);
  const bool live = tok < p.tokens && d0 < p.dim;

  const auto locate = [&](int h, int& kind, int& head) {
    kind = h < p.heads[0] ? 0 : (h < p.heads[0] + p.heads[1] ? 1 : 2);
    head = h - (kind > 0 ? p.heads[0] : 0) - (kind > 1 ? p.heads[1] : 0);
  };
  const auto load = [&](int h) -> uint4 {
    if (!live || h >= h_end) return make_uint4(0, 0, 0, 0);
    int kind, head;
    locate(h, kind, head);
    const T* x = (const T*)p.src[kind] + tok * p.tok_stride[kind] + head * p.head_stride[kind] + d0;
    return *reinterpret_cast<const uint4*>(x);
  };

  uint4 next = load(h_begin);  // under way while the sines are computed

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
  if (p.kv.k && tid < p.block_tokens) {
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
  __syncthreads();

  // this lane's part of the rotation: out[j] = y[j] * c[j] + partner[j] * s[j]
  float c[8], s[8], wq[8], wk[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int d = d0 + j;
    c[j] = 1.f;
    s[j] = 0.f;
    if (d < p.rot) {
      const int i = p.interleaved ? d >> 1 : (d < half ? d : d - half);
      c[j] = s_cos[bt][i];
      s[j] = s_sin[bt][i];
      if (p.interleaved ? !(d & 1) : d < half) s[j] = -s[j];
    }
    wq[j] = wk[j] = 1.f;
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if (p.weight[w] && d0 < p.dim) {
      float* dst = w ? wk : wq;
      if (p.weight_f32) {
        const float* g = (const float*)p.weight[w] + d0;
#pragma unroll
        for (int j = 0; j < 8; ++j) dst[j] = g[j] + p.weight_offset;
      } else {
        const uint4 g = *reinterpret_cast<const uint4*>((const T*)p.weight[w] + d0);
        const uint32_t* u = reinterpret_cast<const uint32_t*>(&g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack2<T>(u[j]);
          dst[2 * j] = f.x + p.weight_offset;
          dst[2 * j + 1] = f.y + p.weight_offset;
        }
      }
    }
  }
  const bool shuffled = !p.interleaved && (half & 7) == 0;
  const int lane = tid & 31;
  int partner = lane;
  if (shuffled && d0 < p.rot) partner = d0 < half ? lane + half / 8 : lane - half / 8;
  const float inv_dim = 1.f / p.dim;

  const int iters = (min(nheads, p.block_heads) + per_tok - 1) / per_tok;  // the same for every lane of a warp
  int h = h_begin;
  for (int it = 0; it < iters; ++it, h += per_tok) {
    const uint4 raw = next;
    next = load(h + per_tok);
    const bool on = live && h < h_end;
    int kind = 0, head = 0;
    if (on) locate(h, kind, head);
    float y[8];
    {
      const uint32_t* u = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2<T>(u[j]);
        y[2 * j] = f.x;
        y[2 * j + 1] = f.y;
      }
    }
    if (p.weight[0] || p.weight[1]) {  // uniform: every lane takes part in the shuffles
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += y[j] * y[j];
#pragma unroll
      for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (kind < 2 && p.weight[kind]) {
        const float r = rsqrtf(ss * inv_dim + p.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = y[j] * r * (kind ? wk[j] : wq[j]);
      }
    }
    float out[8];
    if (p.interleaved) {
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = y[j] * c[j] + y[j ^ 1] * s[j];
    } else if (shuffled) {
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = y[j] * c[j] + __shfl_sync(0xffffffffu, y[j], partner) * s[j];
    } else {
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) s_x[slot][d0 + j] = y[j];
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = d0 + j;
        const int q = d >= p.rot ? d : (d < half ? d + half : d - half);
        out[j] = y[j] * c[j] + s_x[slot][q] * s[j];
      }
    }
    if (!on) continue;
    uint4 w16;
    if (kind == 2) {
      w16 = raw;
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = y[j];
    } else {
      w16 = make_uint4(pack2<T>(out[0], out[1]), pack2<T>(out[2], out[3]), pack2<T>(out[4], out[5]),
                       pack2<T>(out[6], out[7]));
    }
    if (kind == 0) {
      if (p.q_out) *reinterpret_cast<uint4*>((T*)p.q_out + tok * p.q_out_tok + head * p.q_out_head + d0) = w16;
      continue;
    }
    if (kind == 1 && p.k_out)
      *reinterpret_cast<uint4*>((T*)p.k_out + tok * p.k_out_tok + head * p.k_out_head + d0) = w16;
    if (!p.kv.k || s_row[bt] < 0) continue;
    const int64_t at = s_row[bt] + (int64_t)head * p.kv.page_size * p.dim + d0;
    uint8_t* plane = p.kv.k + (kind == 2 ? p.kv.plane : 0);
    if constexpr (F8) {
      // Quantised from the 32-bit value, not from its 16-bit rounding.  Saturating conversion: infinities become
      // +-448, NaN stays NaN.
      const float* scales = kind == 2 ? p.kv.v_scale : p.kv.k_scale;
      const float sc = scales ? scales[head] : 1.f;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(out[2 * j], sc), __fdiv_rn(out[2 * j + 1], sc)),
                                        __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<uint2*>(plane + at) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    } else {
      *reinterpret_cast<uint4*>(plane + 2 * at) = w16;
    }
  }
}

template <typename T, bool F8>
int launch(RopeParams& p, cudaStream_t stream) {
  const int lph = p.dim <= 64 ? 8 : p.dim <= 128 ? 16 : 32;
  const int slots = kThreads / lph;
  const int nheads = p.heads[0] + p.heads[1] + p.heads[2];
  const int sms = sm_count();
  if (!sms) return XCB_ERR_CUDA;
  // Few tokens: one head per lane group, so that a call is a single round of loads.  Many: four tokens per block,
  // each lane group walking over its token's heads with the cosines in registers.
  const int groups = (nheads + slots - 1) / slots;
  if ((int64_t)p.tokens * groups <= 8ll * sms) {
    p.block_tokens = 1;
    p.block_heads = slots;
  } else {
    p.block_tokens = kMaxTok;
    p.block_heads = nheads;
  }
  const dim3 grid((p.tokens + p.block_tokens - 1) / p.block_tokens, (nheads + p.block_heads - 1) / p.block_heads);
  switch (lph) {
    case 8: rope_kernel<T, F8, 8><<<grid, kThreads, 0, stream>>>(p); break;
    case 16: rope_kernel<T, F8, 16><<<grid, kThreads, 0, stream>>>(p); break;
    default: rope_kernel<T, F8, 32><<<grid, kThreads, 0, stream>>>(p); break;
  }
  return cudaGetLastError() == cudaSuccess ? XCB_OK : XCB_ERR_CUDA;
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
  p.eps = a->eps;
  p.weight_offset = a->weight_offset;
  p.mscale = a->mscale;
  const bool f8 = c && c->dtype == XCB_DTYPE_E4M3;
  if (a->dtype == XCB_DTYPE_BF16) return f8 ? launch<__nv_bfloat16, true>(p, stream) : launch<__nv_bfloat16, false>(p, stream);
  return f8 ? launch<__half, true>(p, stream) : launch<__half, false>(p, stream);
}
