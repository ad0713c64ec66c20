// gr_paged_kv.cu — block tables, slot maps and the cache write of the paged KV
// cache, for B200 (sm_100a).
//
// extend_block_tables_kernel.  Two exclusive sums over the requests (new
// tokens, blocks taken) decide everything else, and they are short: every CTA
// computes them for itself, 256 or 2048 requests at a time in shared memory, and then
// writes its even share of the tile's requests, fresh blocks and tokens, each
// found by a binary search in the sums.  So the step is one launch without a
// grid-wide wait, and a batch of one long chunk spreads over the grid as well
// as one of many single tokens.  A token whose block is a fresh one reads its
// id from the free list, not from the table that another CTA may be writing.
// Bound: launch latency for decode steps, the binary searches' shared-memory
// chain for large ones.
//
// store_rows_kernel.  HBM-bound row copy: one warp per token copies K and V
// rows in 16-byte vectors, all loads of a pass (up to 8 per lane) before the
// first store; the row loads do not depend on the slot, so the slot's latency
// hides behind them.  Other layouts take an element-wise kernel.

#include <cstdint>
#include <cuda_runtime.h>
#include <mutex>

#include "../../include/gr_beam.h"
#include "gr_nvtx.h"

namespace grpk {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct TableParams {
  int32_t* table;
  const int32_t* cached;
  const int32_t* fresh;
  const int32_t* free_blocks;
  int32_t* cu;
  int32_t* seq_lens;
  int64_t* slots;
  int64_t* positions;
  int32_t* used;
  int32_t* err;
  int64_t table_stride;
  int num_seqs, num_tokens, num_free, block_size, max_blocks;
};

// Blocks of `tokens` (at most 2^31 - 1) tokens; 32-bit arithmetic, a 64-bit division is a
// subroutine several times as long.
__device__ __forceinline__ int blocks_of(int tokens, int bs) {
  return static_cast<int>((static_cast<uint32_t>(tokens) + static_cast<uint32_t>(bs) - 1u) / static_cast<uint32_t>(bs));
}

__device__ __forceinline__ int clamp32(int64_t v) { return v > 0x7FFFFFFF ? 0x7FFFFFFF : static_cast<int>(v); }

// Exclusive sums over the CTA's threads of two values; totals in t0 / t1.
__device__ __forceinline__ void scan2(int64_t& a, int64_t& b, int64_t& t0, int64_t& t1, int64_t (*part)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t a_in = a, b_in = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xFFFFFFFFu, a, o), y = __shfl_up_sync(0xFFFFFFFFu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  if (lane == 31) {
    part[warp][0] = a;
    part[warp][1] = b;
  }
  __syncthreads();
  a -= a_in;
  b -= b_in;
  t0 = t1 = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) {
      a += t0;
      b += t1;
    }
    t0 += part[w][0];
    t1 += part[w][1];
  }
}

// Last index in [0, n) whose value is <= x (values ascending, v[0] <= x).
__device__ __forceinline__ int last_le(const int64_t* v, int n, int64_t x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// kPerThread requests per thread and pass: 1 for the batch that fits a pass so
// (5.8 us with 8), 8 for larger ones (1500 requests: one pass of 2048 instead of
// six of 256).
template <int kPerThread>
__global__ void __launch_bounds__(kThreads) extend_block_tables_kernel(const TableParams P) {
  constexpr int kTile = kThreads * kPerThread;
  __shared__ int64_t s_cu[kTile + 1];      // first token of each request of the tile
  __shared__ int64_t s_base[kTile + 1];    // first fresh block of each
  __shared__ int32_t s_cached[kTile];
  __shared__ int64_t s_part[kWarps][2];
  const int64_t G = gridDim.x, me = blockIdx.x;
  const int bs = P.block_size;
  int64_t tok0 = 0, blk0 = 0;              // sums before the tile
  int bad = 0;
  for (int r0 = 0; r0 < P.num_seqs; r0 += kTile) {
    const int nr = min(kTile, P.num_seqs - r0);
    int c[kPerThread], f[kPerThread], take[kPerThread];
    int64_t a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int r = static_cast<int>(threadIdx.x) * kPerThread + i;
      c[i] = f[i] = 0;
      if (r < nr) {
        c[i] = P.cached[r0 + r];
        f[i] = P.fresh[r0 + r];
        if (c[i] < 0 || f[i] < 0 || static_cast<int64_t>(c[i]) + f[i] > 0x7FFFFFFF) {
          bad |= GR_DEVERR_BAD_RECORD;
          c[i] = max(c[i], 0);
          f[i] = 0;
        }
      }
      take[i] = blocks_of(c[i] + f[i], bs) - blocks_of(c[i], bs);
      a += f[i];
      b += take[i];
    }
    int64_t ta, tb;
    scan2(a, b, ta, tb, s_part);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int r = static_cast<int>(threadIdx.x) * kPerThread + i;
      s_cu[r] = tok0 + a;
      s_base[r] = blk0 + b;
      s_cached[r] = c[i];
      a += f[i];
      b += take[i];
    }
    if (threadIdx.x == 0) {
      s_cu[kTile] = tok0 + ta;
      s_base[kTile] = blk0 + tb;
    }
    __syncthreads();
    // requests: lengths and offsets
    for (int r = static_cast<int>(me * kThreads + threadIdx.x); r < nr; r += static_cast<int>(G * kThreads)) {
      P.cu[r0 + r] = clamp32(s_cu[r]);
      P.seq_lens[r0 + r] = s_cached[r] + static_cast<int>(s_cu[r + 1] - s_cu[r]);
    }
    // fresh blocks: entry e of the free list to its place in the table.  The loop ends with the
    // list, whatever the lengths ask for: lengths near 2^31 would make it 10^10 blocks.
    const int64_t tf = min(tb, max(static_cast<int64_t>(P.num_free) - blk0, static_cast<int64_t>(0)));
    if (tf < tb && me == 0 && threadIdx.x == 0) bad |= GR_DEVERR_NO_BLOCK;
    const int64_t eb = blk0 + tf * me / G, ee = blk0 + tf * (me + 1) / G;
    for (int64_t e = eb + threadIdx.x; e < ee; e += kThreads) {
      const int r = last_le(s_base, nr, e);
      const int64_t j = blocks_of(s_cached[r], bs) + (e - s_base[r]);
      if (j < P.max_blocks)
        P.table[(r0 + r) * P.table_stride + j] = P.free_blocks[e];
      else
        bad |= GR_DEVERR_NO_BLOCK;
    }
    // tokens
    const int64_t tb0 = tok0 + ta * me / G, te = tok0 + ta * (me + 1) / G;
    for (int64_t t = tb0 + threadIdx.x; t < te; t += kThreads) {
      if (t >= P.num_tokens) {
        bad |= GR_DEVERR_BAD_RECORD;
        break;
      }
      const int r = last_le(s_cu, nr, t);
      const int cach = s_cached[r];
      const int p = cach + static_cast<int>(t - s_cu[r]);
      const int j = p / bs, have = blocks_of(cach, bs);
      int id = -1;
      if (j < P.max_blocks) {
        if (j < have) {
          id = P.table[(r0 + r) * P.table_stride + j];
        } else {
          const int64_t e = s_base[r] + (j - have);
          if (e < P.num_free) id = P.free_blocks[e];
        }
      }
      if (id < 0) bad |= GR_DEVERR_NO_BLOCK;
      P.slots[t] = id < 0 ? -1 : static_cast<int64_t>(id) * bs + (p - j * bs);
      if (P.positions) P.positions[t] = p;
    }
    tok0 += ta;
    blk0 += tb;
    __syncthreads();
  }
  // entries behind the last request's tokens
  const int64_t pad = static_cast<int64_t>(P.num_tokens) - tok0;
  if (pad > 0) {
    for (int64_t t = tok0 + pad * me / G + threadIdx.x; t < tok0 + pad * (me + 1) / G; t += kThreads) {
      P.slots[t] = -1;
      if (P.positions) P.positions[t] = 0;
    }
  }
  if (me == 0 && threadIdx.x == 0) {
    P.cu[P.num_seqs] = clamp32(tok0);
    P.used[0] = clamp32(blk0);
  }
  if (bad && P.err) atomicOr(P.err, bad);
}

// ---- cache write -----------------------------------------------------------
struct StoreParams {
  const unsigned char* k;
  const unsigned char* v;
  unsigned char* kc;
  unsigned char* vc;
  const int64_t* slots;
  int32_t* err;
  int64_t num_tokens, num_slots;
  int block_size;
  int nvec;                                                     // 16-byte vectors per row (vector path)
  int64_t k_tok, v_tok, kc_block, kc_tok, vc_block, vc_tok;     // bytes (vector path), elements (generic)
  int heads, dim;
  int64_t k_head, k_dim, v_head, v_dim, kc_head, kc_dim, vc_head, vc_dim;   // elements (generic path)
};

constexpr int kVecs = 4;   // 16-byte vectors per lane and tensor in flight

__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

__global__ void __launch_bounds__(kThreads) store_rows_kernel(const StoreParams P) {
  const int lane = threadIdx.x & 31;
  const int64_t nwarps = static_cast<int64_t>(gridDim.x) * kWarps;
  for (int64_t t = static_cast<int64_t>(threadIdx.x >> 5) * gridDim.x + blockIdx.x; t < P.num_tokens; t += nwarps) {
    const int64_t slot = __ldg(P.slots + t);
    const uint4* k = reinterpret_cast<const uint4*>(P.k + t * P.k_tok);
    const uint4* v = reinterpret_cast<const uint4*>(P.v + t * P.v_tok);
    uint4 a[kVecs], b[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      if (u * 32 + lane < P.nvec) {
        a[u] = ld_stream(k + u * 32 + lane);
        b[u] = ld_stream(v + u * 32 + lane);
      }
    }
    if (slot < 0 || slot >= P.num_slots) {
      if (slot >= 0 && lane == 0 && P.err) atomicOr(P.err, GR_DEVERR_BAD_SLOT);
      continue;
    }
    const int64_t blk = slot / P.block_size, off = slot - blk * P.block_size;
    uint4* kc = reinterpret_cast<uint4*>(P.kc + blk * P.kc_block + off * P.kc_tok);
    uint4* vc = reinterpret_cast<uint4*>(P.vc + blk * P.vc_block + off * P.vc_tok);
    for (int vb = 0;;) {
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        if (vb + u * 32 + lane < P.nvec) {
          kc[vb + u * 32 + lane] = a[u];
          vc[vb + u * 32 + lane] = b[u];
        }
      }
      vb += 32 * kVecs;
      if (vb >= P.nvec) break;
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        if (vb + u * 32 + lane < P.nvec) {
          a[u] = ld_stream(k + vb + u * 32 + lane);
          b[u] = ld_stream(v + vb + u * 32 + lane);
        }
      }
    }
  }
}

// Element-wise copy with the caller's strides (any (head, dim) layout).
template <typename E>
__global__ void __launch_bounds__(kThreads) store_elems_kernel(const StoreParams P) {
  const int lane = threadIdx.x & 31;
  const int row = P.heads * P.dim;
  const E* K = reinterpret_cast<const E*>(P.k);
  const E* V = reinterpret_cast<const E*>(P.v);
  E* KC = reinterpret_cast<E*>(P.kc);
  E* VC = reinterpret_cast<E*>(P.vc);
  const int64_t nwarps = static_cast<int64_t>(gridDim.x) * kWarps;
  for (int64_t t = static_cast<int64_t>(threadIdx.x >> 5) * gridDim.x + blockIdx.x; t < P.num_tokens; t += nwarps) {
    const int64_t slot = __ldg(P.slots + t);
    if (slot < 0 || slot >= P.num_slots) {
      if (slot >= 0 && lane == 0 && P.err) atomicOr(P.err, GR_DEVERR_BAD_SLOT);
      continue;
    }
    const int64_t blk = slot / P.block_size, off = slot - blk * P.block_size;
    for (int e = lane; e < row; e += 32) {
      const int h = e / P.dim, d = e - h * P.dim;
      KC[blk * P.kc_block + off * P.kc_tok + h * P.kc_head + d * P.kc_dim] = K[t * P.k_tok + h * P.k_head + d * P.k_dim];
      VC[blk * P.vc_block + off * P.vc_tok + h * P.vc_head + d * P.vc_dim] = V[t * P.v_tok + h * P.v_head + d * P.v_dim];
    }
  }
}

static int g_sms[64];
static std::mutex g_mu;

// The current device's SM count (looked up once per device).
static int sm_count(int& out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return GR_ERR_NO_DEVICE;
  std::lock_guard<std::mutex> lock(g_mu);
  if (g_sms[dev] == 0 && cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    g_sms[dev] = 0;
    return GR_ERR_CUDA;
  }
  out = g_sms[dev];
  return GR_OK;
}

}  // namespace grpk

extern "C" int32_t gr_extend_block_tables(const gr_block_table_desc* d, int32_t* block_table, const int32_t* cached,
                                          const int32_t* fresh, const int32_t* free_blocks, int32_t* cu_seqlens,
                                          int32_t* seq_lens, int64_t* slot_mapping, int64_t* positions,
                                          int32_t* blocks_used, int32_t* err, void* stream) {
  gr::NvtxRange nvtx_range("gr_extend_block_tables");
  using namespace grpk;
  if (!d) return GR_ERR_NULL;
  if (d->num_seqs < 0 || d->num_tokens < 0 || d->num_free < 0 || d->block_size < 1 || d->max_blocks < 0 ||
      d->num_seqs > 0x7FFFFFFF - 4095 || (d->num_seqs > 1 && d->table_stride < d->max_blocks))
    return GR_ERR_BAD_DESC;
  if (!cu_seqlens || !blocks_used) return GR_ERR_NULL;
  if (d->num_seqs > 0 && (!cached || !fresh || !seq_lens || (d->max_blocks > 0 && !block_table))) return GR_ERR_NULL;
  if ((d->num_tokens > 0 && !slot_mapping) || (d->num_free > 0 && !free_blocks)) return GR_ERR_NULL;
  int sms = 0;
  const int rc = sm_count(sms);
  if (rc != GR_OK) return rc;
  TableParams P;
  P.table = block_table;
  P.cached = cached;
  P.fresh = fresh;
  P.free_blocks = free_blocks;
  P.cu = cu_seqlens;
  P.seq_lens = seq_lens;
  P.slots = slot_mapping;
  P.positions = positions;
  P.used = blocks_used;
  P.err = err;
  P.table_stride = d->table_stride;
  P.num_seqs = d->num_seqs;
  P.num_tokens = d->num_tokens;
  P.num_free = d->num_free;
  P.block_size = d->block_size;
  P.max_blocks = d->max_blocks;
  // about two tokens per thread, at most four CTAs per SM
  const int64_t work = static_cast<int64_t>(d->num_tokens) + d->num_seqs;
  const int64_t want = (work + 2 * kThreads - 1) / (2 * kThreads);
  const int64_t cap = static_cast<int64_t>(sms) * 4;
  const int grid = static_cast<int>(want < 1 ? 1 : (want < cap ? want : cap));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->num_seqs <= kThreads)
    extend_block_tables_kernel<1><<<grid, kThreads, 0, s>>>(P);
  else
    extend_block_tables_kernel<8><<<grid, kThreads, 0, s>>>(P);
  return cudaGetLastError() == cudaSuccess ? GR_OK : GR_ERR_CUDA;
}

extern "C" int32_t gr_store_kv(const gr_kv_store_desc* d, const void* k, const void* v, void* k_cache, void* v_cache,
                               const int64_t* slot_mapping, int32_t* err, void* stream) {
  gr::NvtxRange nvtx_range("gr_store_kv");
  using namespace grpk;
  if (!d) return GR_ERR_NULL;
  if (d->num_tokens < 0 || d->num_blocks < 0 || d->block_size < 1 || d->num_heads <= 0 || d->head_dim <= 0 ||
      static_cast<int64_t>(d->num_heads) * d->head_dim > 0x7FFFFFFF - 1023)
    return GR_ERR_BAD_DESC;
  if (d->elem_bytes != 1 && d->elem_bytes != 2 && d->elem_bytes != 4) return GR_ERR_DTYPE;
  if (d->num_tokens == 0) return GR_OK;
  if (!k || !v || !k_cache || !v_cache || !slot_mapping) return GR_ERR_NULL;
  int sms = 0;
  const int rc = sm_count(sms);
  if (rc != GR_OK) return rc;
  const int64_t es = d->elem_bytes, hd = d->head_dim;
  const int64_t row_bytes = static_cast<int64_t>(d->num_heads) * hd * es;
  StoreParams P;
  P.k = static_cast<const unsigned char*>(k);
  P.v = static_cast<const unsigned char*>(v);
  P.kc = static_cast<unsigned char*>(k_cache);
  P.vc = static_cast<unsigned char*>(v_cache);
  P.slots = slot_mapping;
  P.err = err;
  P.num_tokens = d->num_tokens;
  P.num_slots = d->num_blocks * d->block_size;
  P.block_size = d->block_size;
  P.nvec = static_cast<int>(row_bytes / 16);
  P.heads = d->num_heads;
  P.dim = d->head_dim;
  P.k_head = d->k_stride_head;
  P.k_dim = d->k_stride_dim;
  P.v_head = d->v_stride_head;
  P.v_dim = d->v_stride_dim;
  P.kc_head = d->kc_stride_head;
  P.kc_dim = d->kc_stride_dim;
  P.vc_head = d->vc_stride_head;
  P.vc_dim = d->vc_stride_dim;
  const auto packed = [&](int64_t head, int64_t dim) { return (dim == 1 || hd == 1) && (head == hd || d->num_heads == 1); };
  const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const int64_t strides = (d->k_stride_tok | d->v_stride_tok | d->kc_stride_block | d->kc_stride_tok |
                           d->vc_stride_block | d->vc_stride_tok) * es;
  const bool vec = packed(d->k_stride_head, d->k_stride_dim) && packed(d->v_stride_head, d->v_stride_dim) &&
                   packed(d->kc_stride_head, d->kc_stride_dim) && packed(d->vc_stride_head, d->vc_stride_dim) &&
                   row_bytes % 16 == 0 && strides % 16 == 0 && aligned(k) && aligned(v) && aligned(k_cache) &&
                   aligned(v_cache);
  const int64_t unit = vec ? es : 1;
  P.k_tok = d->k_stride_tok * unit;
  P.v_tok = d->v_stride_tok * unit;
  P.kc_block = d->kc_stride_block * unit;
  P.kc_tok = d->kc_stride_tok * unit;
  P.vc_block = d->vc_stride_block * unit;
  P.vc_tok = d->vc_stride_tok * unit;
  const int64_t want = (d->num_tokens + kWarps - 1) / kWarps;
  const int64_t cap = static_cast<int64_t>(sms) * 8;
  // few tokens: one CTA each until every SM has one, so that the rows spread
  const int64_t spread = d->num_tokens < sms ? d->num_tokens : sms;
  const int64_t g = want > spread ? want : spread;
  const int grid = static_cast<int>(g < cap ? g : cap);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (vec) {
    store_rows_kernel<<<grid, kThreads, 0, s>>>(P);
  } else if (es == 4) {
    store_elems_kernel<uint32_t><<<grid, kThreads, 0, s>>>(P);
  } else if (es == 2) {
    store_elems_kernel<uint16_t><<<grid, kThreads, 0, s>>>(P);
  } else {
    store_elems_kernel<uint8_t><<<grid, kThreads, 0, s>>>(P);
  }
  return cudaGetLastError() == cudaSuccess ? GR_OK : GR_ERR_CUDA;
}
