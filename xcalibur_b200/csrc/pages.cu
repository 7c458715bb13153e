// Page bookkeeping of the paged cache: growing, forking, rolling back and compacting sequences.
//
// The reference counts are the only record of what is free, so a caller may set tables, lengths and counts back from
// a copy of its own.  Free pages are handed out lowest id first; every result is independent of the order in which
// threads run (integer sums, minima, and prefix sums over lists).
//
// Bound: metadata calls are latency alone (one block, a few dependent rounds of memory: extend and truncate of 256
// sequences 13.4 us with the copy's launch, which finds nothing to do); page copies are HBM, two bytes of traffic per
// byte moved, in 16 KB pieces spread over the whole GPU (a pool of 1024 pages compacted in 126 us, 96% of a copy's
// rate; the part-full pages of 192 forked sequences in 69 us, 90%, as stretches of each head).  The copy is launched
// along with the planning kernel, which saves 0.6 us of the step.
#include "kv.cuh"

namespace xcb {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPerThread = 16;                 // pages per thread and scan step
constexpr int kScanTile = kPlanThreads * kPerThread;
constexpr int kCopyThreads = 256;
constexpr int kCopyPiece = 16384;              // bytes of one block's copy step

// Workspace, in ints.  Zero between calls, but for the lists.
struct KvWs {
  int* moves;    // [4]: number of copies in the lists, rest unused
  int* owner;    // [max_seqs]   INT_MAX - (first list index naming the sequence)
  int* first;    // [num_pages]  INT_MAX - (first list index that holds the shared page)
  int* holders;  // [num_pages]
  int* free;     // [num_pages]  free pages in ascending order, as many as are handed out
  int* src;      // [num_pages]
  int* dst;      // [num_pages]
  int* used;     // [num_pages]  tokens of the page to copy
  int* remap;    // [num_pages]
  int4* plan;    // [max_seqs] of xcb_kv_extend's list entries: pages held, pages wanted, last page, flags
  int* at;       // [max_seqs]   place of the entry's first new page in `free`
};
size_t ws_ints(const XcbKvCache* c) { return 4 + 6 * (size_t)c->max_seqs + 7 * (size_t)c->num_pages; }
KvWs ws_carve(const XcbKvCache* c, void* w) {
  int* p = (int*)w;
  const size_t n = c->num_pages;
  KvWs k;
  k.moves = p;
  k.plan = (int4*)(p + 4);
  k.at = p + 4 + 4 * (size_t)c->max_seqs;
  k.owner = k.at + c->max_seqs;
  k.first = k.owner + c->max_seqs;
  k.holders = k.first + n;
  k.free = k.holders + n;
  k.src = k.free + n;
  k.dst = k.src + n;
  k.used = k.dst + n;
  k.remap = k.used + n;
  return k;
}

struct PageParams {
  int32_t* table;
  int32_t* lens;
  int32_t* refs;
  int32_t* status;
  int32_t num_pages, page_size, max_seqs, max_pages;
  KvWs ws;
};

// Exclusive prefix sum of one value per thread over the block; *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int s_warp[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int w = s_warp[lane];
    int s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    s_warp[lane] = s;
  }
  __syncthreads();
  const int before = warp ? s_warp[warp - 1] : 0;
  *total = s_warp[kPlanThreads / 32 - 1];
  __syncthreads();
  return before + incl - v;
}

constexpr int kOk = 1, kShared = 2, kCopied = 4;

// One block: plans and books the growth of n <= max_seqs sequences; the copies of shared pages are left in the
// workspace's list for copy_kernel.  Every decision is taken from the state as the call found it and written to
// `plan`; the tables, lengths and counts change only after the last of them.
__global__ void __launch_bounds__(kPlanThreads) extend_kernel(const PageParams p, const int32_t* seqs,
                                                              const int32_t* add, int n) {
  __shared__ int s_moves;
  const int tid = threadIdx.x, lane = tid & 31;
  const int per = (n + kPlanThreads - 1) / kPlanThreads;
  const int b = min(n, tid * per), e = min(n, b + per);
  if (tid == 0) s_moves = 0;
  for (int i = b; i < e; ++i) {
    const int s = seqs[i];
    if (s >= 0 && s < p.max_seqs) atomicMax(&p.ws.owner[s], INT32_MAX - i);
  }
  __syncthreads();
  for (int i = b; i < e; ++i) {
    const int s = seqs[i], more = add[i];
    int4 g = make_int4(0, 0, -1, 0);
    if (s >= 0 && s < p.max_seqs && more >= 0 && __ldcg(&p.ws.owner[s]) == INT32_MAX - i) {
      const int len = p.lens[s];
      if (len >= 0 && (int64_t)len + more <= (int64_t)p.max_pages * p.page_size) {
        g.x = (int)(((int64_t)len + p.page_size - 1) / p.page_size);
        g.y = (int)(((int64_t)len + more + p.page_size - 1) / p.page_size);
        g.w = kOk;
        if (more && len % p.page_size) {
          g.z = p.table[(int64_t)s * p.max_pages + g.x - 1];
          if (g.z < 0 || g.z >= p.num_pages) {
            g = make_int4(0, 0, -1, 0);
          } else if (p.refs[g.z] > 1) {
            g.w |= kShared;
            atomicMax(&p.ws.first[g.z], INT32_MAX - i);
            atomicAdd(&p.ws.holders[g.z], 1);
          }
        }
      }
    }
    if (!(g.w & kOk)) atomicOr(p.status, XCB_STATUS_BAD_SEQ);
    p.ws.plan[i] = g;
  }
  __syncthreads();
  // Where every holder of a page grows, the first in the list keeps it and the others copy it.
  int mine = 0;
  for (int i = b; i < e; ++i) {
    int4 g = p.ws.plan[i];
    if ((g.w & kShared) &&
        !(__ldcg(&p.ws.holders[g.z]) == p.refs[g.z] && __ldcg(&p.ws.first[g.z]) == INT32_MAX - i)) {
      g.w |= kCopied;
      p.ws.plan[i] = g;
      ++mine;
    }
    mine += g.y - g.x;
  }
  int total;
  int at = block_scan(mine, &total);
  for (int i = b; i < e; ++i) {
    const int4 g = p.ws.plan[i];
    p.ws.at[i] = at;
    at += g.y - g.x + ((g.w & kCopied) ? 1 : 0);
  }
  // The first `total` free pages, in ascending order.
  int found = 0;
  for (int base = 0; base < p.num_pages && found < total; base += kScanTile) {
    const int q = base + tid * kPerThread;
    uint32_t empty = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j)
      if (q + j < p.num_pages && p.refs[q + j] == 0) empty |= 1u << j;
    int here;
    int r = found + block_scan(__popc(empty), &here);
    for (; empty && r < total; empty &= empty - 1, ++r) p.ws.free[r] = q + __ffs(empty) - 1;
    found += here;
  }
  __syncthreads();
  const bool enough = found >= total;
  if (!enough && tid == 0) atomicOr(p.status, XCB_STATUS_NO_PAGES);
  for (int k = 0; k < per; ++k) {  // the same count for every lane
    const int i = tid * per + k;
    const bool on = i < n;
    int4 g = on ? p.ws.plan[i] : make_int4(0, 0, -1, 0);
    const int s = on ? seqs[i] : -1;
    int from = on ? p.ws.at[i] : 0;
    int start = g.x;
    if (s >= 0 && s < p.max_seqs) p.ws.owner[s] = 0;
    if (g.w & kShared) {
      p.ws.first[g.z] = 0;
      p.ws.holders[g.z] = 0;
    }
    if (!(g.w & kOk) || !enough) g.y = start = 0;
    if (enough && (g.w & kOk)) {
      if (g.w & kCopied) {
        const int m = atomicAdd(&s_moves, 1);
        p.ws.src[m] = g.z;
        p.ws.dst[m] = p.ws.free[from];
        p.ws.used[m] = p.lens[s] % p.page_size;
        atomicSub(&p.refs[g.z], 1);
        --start;
      }
      p.lens[s] += add[i];
    }
    const int count = g.y - start;
    const int64_t row = (int64_t)s * p.max_pages + start;
    if (count > 0 && count <= 4) {
      for (int j = 0; j < count; ++j) {
        const int id = p.ws.free[from + j];
        p.refs[id] = 1;
        p.table[row + j] = id;
      }
    }
    // long growths, one warp each
    for (uint32_t big = __ballot_sync(0xffffffffu, count > 4); big; big &= big - 1) {
      const int who = __ffs(big) - 1;
      const int c = __shfl_sync(0xffffffffu, count, who), f = __shfl_sync(0xffffffffu, from, who);
      const int64_t r = __shfl_sync(0xffffffffu, row, who);
      for (int j = lane; j < c; j += 32) {
        const int id = p.ws.free[f + j];
        p.refs[id] = 1;
        p.table[r + j] = id;
      }
    }
  }
  __syncthreads();
  if (tid == 0) p.ws.moves[0] = s_moves;
}

// One block per entry: the new sequence holds the pages of the old one.
__global__ void __launch_bounds__(128) fork_kernel(const PageParams p, const int32_t* src, const int32_t* dst, int n) {
  const int i = blockIdx.x;
  const int s = src[i], d = dst[i];
  bool bad = s < 0 || s >= p.max_seqs || d < 0 || d >= p.max_seqs;
  for (int j = threadIdx.x; j < n; j += blockDim.x) bad |= src[j] == d || (j < i && dst[j] == d);
  int len = 0;
  if (!bad) {
    // dst[i] is written by this block alone: an earlier entry naming it would have made this one bad
    len = p.lens[s];
    bad = p.lens[d] != 0 || len < 0 || len > (int64_t)p.max_pages * p.page_size;
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) atomicOr(p.status, XCB_STATUS_BAD_SEQ);
    return;
  }
  const int have = (int)(((int64_t)len + p.page_size - 1) / p.page_size);
  for (int j = threadIdx.x; j < have; j += blockDim.x) {
    const int id = p.table[(int64_t)s * p.max_pages + j];
    p.table[(int64_t)d * p.max_pages + j] = id;
    if (id >= 0 && id < p.num_pages) atomicAdd(&p.refs[id], 1);
  }
  if (threadIdx.x == 0) p.lens[d] = len;
}

// One block per entry: pages past the new length are given back.
__global__ void __launch_bounds__(128) truncate_kernel(const PageParams p, const int32_t* seqs, const int32_t* lens,
                                                       int n) {
  const int i = blockIdx.x;
  const int s = seqs[i], to = lens ? lens[i] : 0;
  bool bad = s < 0 || s >= p.max_seqs;
  for (int j = threadIdx.x; j < i; j += blockDim.x) bad |= seqs[j] == s;
  int len = 0;
  if (!bad) {
    len = p.lens[s];
    bad = to < 0 || to > len || len > (int64_t)p.max_pages * p.page_size;
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) atomicOr(p.status, XCB_STATUS_BAD_SEQ);
    return;
  }
  const int keep = (int)(((int64_t)to + p.page_size - 1) / p.page_size);
  const int have = (int)(((int64_t)len + p.page_size - 1) / p.page_size);
  for (int j = keep + threadIdx.x; j < have; j += blockDim.x) {
    const int64_t at = (int64_t)s * p.max_pages + j;
    const int id = p.table[at];
    p.table[at] = -1;
    if (id >= 0 && id < p.num_pages) atomicSub(&p.refs[id], 1);
  }
  if (threadIdx.x == 0) p.lens[s] = to;
}

// One block: with L pages live, the k-th live page at or above L goes to the k-th free page below L.
__global__ void __launch_bounds__(kPlanThreads) compact_kernel(const PageParams p) {
  const int tid = threadIdx.x;
  const auto live_bits = [&](int q) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j)
      if (q + j < p.num_pages && p.refs[q + j] > 0) m |= 1u << j;
    return m;
  };
  int mine = 0;
  for (int q = tid * kPerThread; q < p.num_pages; q += kScanTile) mine += __popc(live_bits(q));
  int live;
  block_scan(mine, &live);
  int movers = 0, holes = 0;
  for (int base = 0; base < p.num_pages; base += kScanTile) {
    const int q = base + tid * kPerThread;
    const uint32_t m = live_bits(q);
    const int in = min(kPerThread, p.num_pages - q);      // of this thread's pages, those that exist
    const int low = max(0, min(in, live - q));            // and those below L
    const uint32_t all = in > 0 ? (1u << in) - 1 : 0, below = (1u << low) - 1;
    uint32_t up = m & ~below, down = ~m & below & all;
    int nu, nd;
    int u = movers + block_scan(__popc(up), &nu);
    int d = holes + block_scan(__popc(down), &nd);
    for (; up; up &= up - 1) p.ws.src[u++] = q + __ffs(up) - 1;
    for (; down; down &= down - 1) p.ws.dst[d++] = q + __ffs(down) - 1;
    for (int j = 0; j < in; ++j) p.ws.remap[q + j] = q + j;
    movers += nu;
    holes += nd;
  }
  __syncthreads();
  for (int k = tid; k < movers; k += kPlanThreads) {
    const int from = p.ws.src[k], to = p.ws.dst[k];
    p.ws.used[k] = p.page_size;
    p.ws.remap[from] = to;
    p.refs[to] = p.refs[from];
    p.refs[from] = 0;
  }
  if (tid == 0) p.ws.moves[0] = movers;
}

__global__ void __launch_bounds__(256) remap_kernel(const PageParams p) {
  const int64_t n = (int64_t)p.max_seqs * p.max_pages;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int id = p.table[i];
    if (id >= 0 && id < p.num_pages) {
      const int to = p.ws.remap[id];
      if (to != id) p.table[i] = to;
    }
  }
}

struct CopyParams {
  uint8_t* kv;
  int64_t plane;          // bytes of one layer's keys (or values)
  int64_t head_bytes;     // one page's bytes of one head
  int32_t token_bytes;    // one token's bytes of one head
  int32_t planes, heads, num_pages, page_size;
  int32_t pieces;         // copy steps of a whole page of one plane
  const int32_t* src;
  const int32_t* dst;
  const int32_t* used;    // tokens of each page to copy, or null: whole pages
  const int32_t* count;   // number of pairs, or null: n
  int32_t n;
  int32_t* status;
};

// A block copies a 16 KB piece of one page of one plane at a time.  Of a part-full page only the used tokens move: a
// stretch of each head.
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const CopyParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int pairs = p.count ? *p.count : p.n;
  const int64_t items = (int64_t)pairs * p.planes * p.pieces;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t pp = it / p.pieces;
    const int piece = (int)(it - pp * p.pieces);
    const int pair = (int)(pp / p.planes), plane = (int)(pp - (int64_t)pair * p.planes);
    const int src = p.src[pair], dst = p.dst[pair];
    if (src < 0 || src >= p.num_pages || dst < 0 || dst >= p.num_pages) {
      if (threadIdx.x == 0) atomicOr(p.status, XCB_STATUS_BAD_PAGE);
      continue;
    }
    const int used = p.used ? p.used[pair] : p.page_size;
    const bool whole = used == p.page_size;
    const int run = whole ? (int)(p.head_bytes * p.heads / 16) : used * p.token_bytes / 16;  // 16-byte words in a row
    const int words = whole ? run : run * p.heads;
    const int64_t page_bytes = p.head_bytes * p.heads;
    const uint8_t* from = p.kv + plane * p.plane + src * page_bytes;
    uint8_t* to = p.kv + plane * p.plane + dst * page_bytes;
    const int first = piece * (kCopyPiece / 16) + threadIdx.x;
    const int end = min(words, (piece + 1) * (kCopyPiece / 16));
    constexpr int U = kCopyPiece / 16 / kCopyThreads;
    uint4 v[U];
    int64_t off[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int w = first + u * kCopyThreads;
      if (w < end) {
        const int head = w / run;
        off[u] = head * p.head_bytes + (int64_t)(w - head * run) * 16;
        v[u] = __ldcs(reinterpret_cast<const uint4*>(from + off[u]));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + u * kCopyThreads < end) __stcs(reinterpret_cast<uint4*>(to + off[u]), v[u]);
  }
}

PageParams page_params(const XcbKvCache* c, void* ws) {
  PageParams p{};
  p.table = c->page_table;
  p.lens = c->seq_lens;
  p.refs = c->refcounts;
  p.status = c->status;
  p.num_pages = c->num_pages;
  p.page_size = c->page_size;
  p.max_seqs = c->max_seqs;
  p.max_pages = c->max_pages;
  if (ws) p.ws = ws_carve(c, ws);
  return p;
}

int page_check(const XcbKvCache* c) {
  const int rc = kv_check(c);
  if (rc != XCB_OK) return rc;
  if (!c->refcounts) return XCB_ERR_INVALID_ARG;
  // a copy step's word index is 32-bit
  if ((int64_t)c->kv_heads * c->page_size * c->head_dim * kv_elem_bytes(c->dtype) >= (1ll << 31)) return XCB_ERR_UNSUPPORTED;
  return XCB_OK;
}

int launch_copy(const XcbKvCache* c, const int* src, const int* dst, const int* used, const int* count, int n,
                cudaStream_t stream) {
  CopyParams p{};
  p.kv = (uint8_t*)c->kv;
  p.token_bytes = c->head_dim * kv_elem_bytes(c->dtype);
  p.head_bytes = (int64_t)c->page_size * p.token_bytes;
  p.heads = c->kv_heads;
  p.plane = (int64_t)c->num_pages * c->kv_heads * p.head_bytes;
  p.planes = 2 * c->layers;
  p.num_pages = c->num_pages;
  p.page_size = c->page_size;
  p.pieces = (int)((p.head_bytes * p.heads + kCopyPiece - 1) / kCopyPiece);
  p.src = src;
  p.dst = dst;
  p.used = used;
  p.count = count;
  p.n = n;
  p.status = c->status;
  const int sms = sm_count();
  if (!sms) return XCB_ERR_CUDA;
  const int64_t most = (int64_t)(n < c->num_pages ? n : c->num_pages) * p.planes * p.pieces;
  // Many short blocks rather than blocks that stay: the next one's list is read while others copy.  With 8 / 24 / 64 / 256
  // an SM: fork's growth 82.2 / 69.6 / 68.6 / 77.8 us, compaction 137 / 131 / 126 / 128, a step without copies 12.1 / 12.5.
  const int64_t grid = most < 64ll * sms ? most : 64ll * sms;
  // Launched along with the kernel before it, whose end it waits for on the device.
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kCopyThreads);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, copy_kernel, p) == cudaSuccess ? XCB_OK : XCB_ERR_CUDA;
}

int list_check(const XcbKvCache* c, const int32_t* a, const int32_t* b, int n) {
  if (n < 0 || n > c->max_seqs) return XCB_ERR_INVALID_ARG;
  if (n && (!a || !kv_aligned(a, 4) || !kv_aligned(b, 4))) return XCB_ERR_INVALID_ARG;
  return XCB_OK;
}

int ws_check(const XcbKvCache* c, const void* ws, size_t bytes) {
  if (!ws || !kv_aligned(ws, 16)) return XCB_ERR_INVALID_ARG;
  return bytes < xcb_kv_workspace_bytes(c) ? XCB_ERR_WORKSPACE : XCB_OK;
}

int launched() { return cudaGetLastError() == cudaSuccess ? XCB_OK : XCB_ERR_CUDA; }

}  // namespace
}  // namespace xcb

using namespace xcb;

extern "C" {

size_t xcb_kv_workspace_bytes(const XcbKvCache* c) { return kv_check(c) == XCB_OK ? ws_ints(c) * 4 : 0; }

int xcb_kv_workspace_init(const XcbKvCache* c, void* ws, size_t bytes, cudaStream_t stream) {
  int rc = kv_check(c);
  if (rc != XCB_OK) return rc;
  if ((rc = ws_check(c, ws, bytes)) != XCB_OK) return rc;
  return cudaMemsetAsync(ws, 0, ws_ints(c) * 4, stream) == cudaSuccess ? XCB_OK : XCB_ERR_CUDA;
}

int xcb_kv_extend(const XcbKvCache* c, const int32_t* seqs, const int32_t* new_tokens, int32_t n, void* ws,
                  size_t ws_bytes, cudaStream_t stream) {
  int rc = page_check(c);
  if (rc != XCB_OK) return rc;
  if ((rc = list_check(c, seqs, new_tokens, n)) != XCB_OK) return rc;
  if (n && !new_tokens) return XCB_ERR_INVALID_ARG;
  if ((rc = ws_check(c, ws, ws_bytes)) != XCB_OK) return rc;
  if (n == 0) return XCB_OK;
  const PageParams p = page_params(c, ws);
  extend_kernel<<<1, kPlanThreads, 0, stream>>>(p, seqs, new_tokens, n);
  if ((rc = launched()) != XCB_OK) return rc;
  return launch_copy(c, p.ws.src, p.ws.dst, p.ws.used, p.ws.moves, n, stream);
}

int xcb_kv_fork(const XcbKvCache* c, const int32_t* src, const int32_t* dst, int32_t n, cudaStream_t stream) {
  int rc = page_check(c);
  if (rc != XCB_OK) return rc;
  if ((rc = list_check(c, src, dst, n)) != XCB_OK) return rc;
  if (n == 0) return XCB_OK;
  if (!dst) return XCB_ERR_INVALID_ARG;
  fork_kernel<<<n, 128, 0, stream>>>(page_params(c, nullptr), src, dst, n);
  return launched();
}

int xcb_kv_truncate(const XcbKvCache* c, const int32_t* seqs, const int32_t* lens, int32_t n, cudaStream_t stream) {
  int rc = page_check(c);
  if (rc != XCB_OK) return rc;
  if ((rc = list_check(c, seqs, lens, n)) != XCB_OK) return rc;
  if (n == 0) return XCB_OK;
  truncate_kernel<<<n, 128, 0, stream>>>(page_params(c, nullptr), seqs, lens, n);
  return launched();
}

int xcb_kv_compact(const XcbKvCache* c, void* ws, size_t ws_bytes, cudaStream_t stream) {
  int rc = page_check(c);
  if (rc != XCB_OK) return rc;
  if ((rc = ws_check(c, ws, ws_bytes)) != XCB_OK) return rc;
  const int sms = sm_count();
  if (!sms) return XCB_ERR_CUDA;
  const PageParams p = page_params(c, ws);
  compact_kernel<<<1, kPlanThreads, 0, stream>>>(p);
  if ((rc = launched()) != XCB_OK) return rc;
  const int64_t blocks = ((int64_t)c->max_seqs * c->max_pages + 255) / 256;
  remap_kernel<<<(unsigned)(blocks < 4ll * sms ? blocks : 4ll * sms), 256, 0, stream>>>(p);
  if ((rc = launched()) != XCB_OK) return rc;
  // fewer than half of the pages can move
  return launch_copy(c, p.ws.src, p.ws.dst, p.ws.used, p.ws.moves, (c->num_pages + 1) / 2, stream);
}

int xcb_kv_copy_pages(const XcbKvCache* c, const int32_t* src, const int32_t* dst, int32_t n, cudaStream_t stream) {
  int rc = page_check(c);
  if (rc != XCB_OK) return rc;
  if (n < 0 || n > c->num_pages) return XCB_ERR_INVALID_ARG;
  if (n == 0) return XCB_OK;
  if (!src || !dst || !kv_aligned(src, 4) || !kv_aligned(dst, 4)) return XCB_ERR_INVALID_ARG;
  return launch_copy(c, src, dst, nullptr, nullptr, n, stream);
}

int xcb_kv_read_status(const XcbKvCache* c, int32_t* device_status, cudaStream_t stream) {
  if (!c || !c->status || !device_status) return XCB_ERR_INVALID_ARG;
  if (cudaMemcpyAsync(device_status, c->status, 4, cudaMemcpyDeviceToHost, stream) != cudaSuccess ||
      cudaMemsetAsync(c->status, 0, 4, stream) != cudaSuccess || cudaStreamSynchronize(stream) != cudaSuccess)
    return XCB_ERR_CUDA;
  return *device_status ? XCB_ERR_DEVICE : XCB_OK;
}

}  // extern "C"
