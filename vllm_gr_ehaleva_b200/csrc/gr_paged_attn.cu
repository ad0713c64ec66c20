// gr_paged_attn.cu — attention of a step's query tokens over the paged KV cache
// for B200 (sm_100a): whole prompts, chunks, single tokens and the beams of
// mega-requests in one batch.
//
// Mathematics.  For a query row with scaled scores s_k over the keys it sees,
// out = sum_k 2^(c s_k - m) v_k / l,  l = sum_k 2^(c s_k - m),  c = scale log2(e),
// lse = ln2 (m + log2 l): one pass over the keys with a running reference m.  m
// follows the running maximum only when that grows by more than 8 (a factor
// 256), so the accumulator is rescaled rarely and no term exceeds 2^8.
// Scores, m, l and the accumulator are fp32; the probabilities are rounded once
// to the cache's 16-bit type as the second product's operand (each term off by
// at most half a step, the sum l uses the unrounded ones).
//
// Rows.  The query heads of one KV head share its keys, so a tile of the first
// product holds (token, head of the group) rows: tp = floor(128 / group) tokens.
// Single tokens use group rows of the 128; their product time hides behind the
// cache reads, which bound them.
//
// Work.  A (query block, KV head) pair of n key tiles costs n + kCost units; the
// batch's units, in order, are cut into equal runs, one per CTA (one persistent
// CTA per SM), whatever the lengths (planned by a one-CTA kernel ahead, or, up to
// 96 query blocks, by every CTA for itself).  A border that
// falls into a short pair moves to the pair's nearer end; a longer pair is cut.
// The CTA with a cut pair's end owns it: the others leave partial outputs and
// log-sums in the workspace, which the owner joins in run order.  Where whole
// pairs already share out almost evenly, none is cut.  CTAs walk their
// runs from the end, so that an owner comes to the join last and the parts that
// it waits for came first in theirs, and it waits for lower-numbered CTAs only,
// which never wait for it.  For beams, key tiles between the tail and the block's
// first beam hold only other beams' tokens and are not visited.
//
// Kernel.  Warps 0 and 2 load keys and values (tensor-map copies of the blocks'
// rows, 128-byte swizzle, one ring of tiles), warp 1 issues the matrix products
// (S = Q K^T from shared memory, O += P V with P in tensor memory), warp 3 walks
// the run and hands out its pairs; the last warps are the softmax: one thread per
// row.  Two query tiles (kNQ = 2) have a softmax group each and alternate on the
// tensor pipe; one tile (kNQ = 1: no query of more than 128 rows, or heads above
// 128, whose accumulators leave no room) alternates two score buffers instead and
// has four more loading warps.  Heads above 128 move their tiles as two halves of
// 128 columns.  The kernel is picked for the whole batch by its longest query: one
// chunk beside 64 single tokens puts them into the kernel with two tiles (263 us
// instead of 183).  Every wait is bounded (GR_DEVERR_TIMEOUT).
//
// Bound and measured (32 query heads over 8 KV heads of 128, blocks of 16): 64
// single tokens over 2.5 GB of cache 6.4 TB/s, HBM, 98 % of a plain copy's rate
// (over 1.1 GB 6.0 TB/s for some milliseconds, 5.0 in runs of seconds, where the
// power limit holds); a prompt of 8192 1060 TFLOP/s for some milliseconds and 920 to
// 1000 in longer runs: the chain scores - softmax - product of a query tile
// (exponential unit and tensor pipe each near half of their rate), then the power
// limit (1.4 to 1.7 GHz).

#include <atomic>
#include <chrono>
#include <cstdint>
#include <cstdlib>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <mutex>

#include "../../include/gr_beam.h"
#include "gr_device.cuh"
#include "gr_nvtx.h"

namespace grpa {

using gr::mbar_arrive;
using gr::mbar_arrive_expect_tx;
using gr::mbar_init;
using gr::smem_u32;

constexpr int kRows = 128;            // rows of a query tile (the matrix product's M)
constexpr int kMaxCtas = 160;
constexpr int kSmallItems = 96;       // requests and query blocks that the CTAs plan for themselves
constexpr int kWorkRing = 4;          // (block, head) pairs handed out ahead
// The shares of the work, in units of a key tile (about 2 us with two query tiles).  Measured on
// 64 single tokens, a prompt of 8192, ragged chunks and beams: kCost 1 and 3, kMinRun 3 and 4,
// kJoin 3 and 8 are within 2 % of these on each, kMinRun 4 loses 10 % on two single tokens.
constexpr int kCost = 2;              // what a pair costs besides its key tiles
constexpr int kSnap = 8;              // longest pair that is never cut
constexpr int kMinRun = 2;            // what a CTA's run has at least, on average
constexpr int kJoin = 5;              // with whole pairs the longest run may be this much longer than with cut ones
constexpr int kSmemMax = 232448;      // shared memory a CTA may have
constexpr float kRescale = 8.0f;      // log2 of the growth of the maximum that is let stand

template <int DP_, int NQ_>
struct Shape {
  static constexpr int DP = DP_;                       // head dim, padded to 64 / 128 / 256
  static constexpr int NQ = NQ_;                       // query tiles per block
  static constexpr int BN = 128;                       // keys per tile
  static constexpr int CH = DP / 64;                   // 128-byte column chunks of a row
  static constexpr int SUB = DP == 256 ? 2 : 1;        // ring stages per tile: 128 columns each
  static constexpr int CHS = CH / SUB;                 // chunks of a stage
  static constexpr int kChunkQ = kRows * 128;          // bytes of one chunk of a query tile
  static constexpr int kChunkKV = BN * 128;
  static constexpr int kQTile = CH * kChunkQ;
  static constexpr int kStage = CHS * kChunkKV;
  static constexpr int kStages = DP == 64 ? 10 : (NQ == 2 || DP == 256 ? 5 : 6);
  // warps 0..3: loads, products, loads, schedule; kNQ = 1: four more that load; then the softmax
  static constexpr int kLoaders = NQ == 2 ? 1 : 3;     // warps that load keys (as many load values)
  static constexpr int kSoftmax = NQ == 2 ? 4 : 8;     // first softmax warp
  static constexpr int kThreads = 32 * kSoftmax + 128 * NQ;
  static constexpr int kColO = 2 * BN;                 // tensor memory: S0, S1, O0, (O1)
  static constexpr int kData = NQ * kQTile + kStages * kStage;
  static_assert(kColO + NQ * DP <= 512, "tensor memory columns");
};

// A (block, head) of a CTA's run, from the scheduling warp to the others.
struct Work {
  int req, q0;             // request, its first query token
  int len, ctx;            // its keys, the position of its query token 0
  int tail, steps;         // its beams
  int t0, nt;              // the block's query tokens, from t0 of the request
  int kvh;                 // KV head
  int ta, tb, n;           // its key tiles: [0, ta) and from tb on, n in all
  int j0, j1;              // those of the run
  int slots;               // query tiles with rows; 0: the run is over
  int part0;               // the first CTA with a part of the pair (this one's pair: j0 > 0, j1 = n)
};

struct Shared {
  uint64_t full[12], empty[12];
  uint64_t wk_full[kWorkRing], wk_empty[kWorkRing];
  Work work[kWorkRing];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_full[2];   // scores ready / probabilities ready
  uint64_t pv_done[2], o_free[2];  // product into O finished / O read out
  uint64_t drain;
  uint32_t tmem;
  int abort;
  // a small batch's plan: the runs' borders, the units before each query block, request and block
  int64_t part[13];
  int32_t border[kMaxCtas + 1], pre[kSmallItems + 1];
  uint8_t req[kSmallItems], blk[kSmallItems];
  int32_t items;
};

struct Run {                       // where a CTA's run starts
  int64_t u;                       // in units of the batch, KV heads outermost
  int32_t head, item;              // the pair that the run before it ends in
};

struct Params {
  const int32_t* table;
  const int32_t* cu;
  const int32_t* seq_lens;
  const int32_t* tail;
  const int32_t* steps;
  void* out;
  float* lse;
  int32_t* err;
  int64_t table_stride, num_blocks, out_tok, out_head;
  int num_seqs, num_tokens, heads, kv_heads, group, dim;
  int block_size, max_blocks, causal;
  int tp;                          // query tokens per tile
  int box;                         // rows of a block that one copy takes
  uint32_t div_mul, div_shift;     // x / block_size = (x * div_mul >> 32) >> div_shift for x < 2^31
  int out32;                       // output rows start on 32 bytes
  int flags;                       // 1: copies are not issued (test hook)
  float scale_log2;
  // plan and partials in the workspace
  int64_t* pre;                    // [items + 1] units of one KV head before each query block
  int2* item;                      // request, block
  int32_t* items;                  // how many
  Run* run;                        // [ctas + 1]
  uint64_t* flag;                  // [ctas][2][4] part written (query tile, warp of it): token, until its owner has read it
  uint64_t token;                  // of this call
  int small;                       // planned by the CTAs
  float4* part_o;                  // [ctas][2][NQ][DP / 4][128 rows]: a warp's stores of its 32 rows are whole lines
  float* part_lse;                 // [ctas][2][NQ][128 rows]
};

// ---------------------------------------------------------------- tensor core
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One lane of the warp, the same one every time.
__device__ __forceinline__ bool elect_lane() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(yes));
  return yes != 0;
}

// Everything the calling thread has issued to the tensor core so far arrives on bar when done.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// D (tensor memory, fp32) = A (shared memory) x B (shared memory), + D when acc.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// The same with A in tensor memory.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle: address, the two strides
// (all in 16-byte units), version 1, layout 2.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((lead >> 4) & 0x3FFFu) << 16) |
         (static_cast<uint64_t>((stride >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}

// 32 columns of this warp's 32 lanes.
__device__ __forceinline__ void tc_ld32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Tensor-map copies into this CTA's shared memory (no multicast).
__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (kBf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void st_global_32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// A wait by a whole warp.  One that gives up sets the CTA's abort flag, which
// ends every other wait; the warp's lanes leave together or not at all: they vote
// on the flag too, since lanes that read it apart may read it differently, and one
// that stayed would vote with lanes that have left.  The
// limit is a number of tries: reading the timer between them, or trying more
// often, takes issue slots from the warps that are waited for (32 x 128 beams
// behind 600 to 2600 keys: 614 k cycles with the timer, 575 k without, 770 k with
// a spin of test_wait).
constexpr int kTries = 500000;           // about 2 s: a try that fails sleeps some 4 us
constexpr int kPairTries = 16 * kTries;  // for waits that last as long as a pair does
__device__ __forceinline__ bool aborted(Shared* sh) {   // one answer for the warp
  return __any_sync(0xFFFFFFFFu, *reinterpret_cast<volatile int*>(&sh->abort));
}
__device__ __forceinline__ bool wait(Shared* sh, uint64_t* bar, uint32_t parity, int tries = kTries) {
  for (int i = 0; i < tries; ++i) {
    if (__all_sync(0xFFFFFFFFu, gr::mbar_try_wait(bar, parity))) return true;
    if (aborted(sh)) break;
  }
  *reinterpret_cast<volatile int*>(&sh->abort) = 1;
  return false;
}

// ---------------------------------------------------------------- geometry
struct Seq {          // a request
  int q0, n, len;     // first query token, query tokens, keys
  int ctx;            // position of query token 0 (negative when there are fewer keys than tokens)
  int tail, steps;    // beams (steps 0: none)
};

__device__ __forceinline__ Seq load_seq(const Params& P, int r, int* bad = nullptr) {
  Seq s;
  const int a = P.cu[r], b = P.cu[r + 1];
  const int len = P.seq_lens[r];
  const int a1 = min(max(a, 0), P.num_tokens), b1 = min(max(b, a1), P.num_tokens);
  s.q0 = a1;
  s.n = b1 - a1;
  const int64_t room = static_cast<int64_t>(P.max_blocks) * P.block_size;
  s.len = static_cast<int>(min(static_cast<int64_t>(max(len, 0)), room));
  if (bad && (a != a1 || b != b1 || s.len != len)) *bad = 1;
  s.ctx = s.len - s.n;
  s.tail = s.steps = 0;
  if (P.causal && P.steps != nullptr) {
    s.steps = max(P.steps[r], 0);
    s.tail = min(max(P.tail[r], 0), s.n);
  }
  return s;
}

// The key tiles of query tokens [t0, t1): [0, a) and [b, c) of BN keys each;
// at least one (a block without keys still writes its rows).
struct Tiles {
  int a, b, n;
};
template <int BN>
__device__ __forceinline__ Tiles key_tiles(const Seq& s, int causal, int t0, int t1) {
  const int hi = causal ? min(max(s.ctx + t1, 0), s.len) : s.len;
  const int c = (hi + BN - 1) / BN;
  Tiles t{c, c, 0};
  if (s.steps > 0 && t1 > s.tail) {
    const int first = max(s.ctx + s.tail, 0);
    const int fb = max(t0, s.tail);
    const int own = max(s.ctx + s.tail + (fb - s.tail) / s.steps * s.steps, 0);
    t.a = min((first + BN - 1) / BN, c);
    t.b = min(max(own / BN, t.a), c);
  }
  t.n = max(t.a + c - t.b, 1);
  return t;
}

__device__ __forceinline__ int blocks_of(const Seq& s, int per) { return (s.n + per - 1) / per; }

// Inclusive sum over a warp.
__device__ __forceinline__ int64_t warp_scan(int64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}

constexpr int kPlanThreads = 1024;

// Exclusive sum over a CTA of kT threads; total in `total`; part has kT / 32 + 1 places.
template <int kT>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t& total, int64_t* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t inc = warp_scan(v);
  __syncthreads();
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int64_t p = lane < kT / 32 ? part[lane] : 0;
    const int64_t q = warp_scan(p);
    if (lane < kT / 32) part[lane] = q - p;
    if (lane == 31) part[kT / 32] = q;
  }
  __syncthreads();
  total = part[kT / 32];
  return part[warp] + inc - v;
}

// Last index in [0, n) whose value is <= x (values ascending, v[0] <= x).
template <typename T>
__device__ __forceinline__ int last_le(const T* v, int n, int64_t x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Border c of `runs` runs over `all` units (`units` per KV head, `pre` before each of `items` query
// blocks): at the even share (a short pair's nearer end), and at the nearer end of the pair that the
// even share falls into.
struct Border {
  int64_t even, whole;
  int64_t pair;        // first unit of that pair
  int head, item;      // which it is
};
template <typename T>
__device__ __forceinline__ Border border(const T* pre, int items, int64_t units, int64_t all, int64_t runs, int c) {
  Border b{all, all, all, 0, items};
  if (c >= runs) return b;
  const int64_t u = all * c / runs;
  b.head = static_cast<int>(u / units);
  const int64_t in = u - b.head * units;
  b.item = last_le(pre, items, in);
  const int64_t span = pre[b.item + 1] - pre[b.item], off = in - pre[b.item];
  b.pair = u - off;
  b.whole = b.pair + (2 * off < span ? 0 : span);
  b.even = span <= kSnap ? b.whole : u;
  return b;
}
__device__ __forceinline__ int64_t runs_of(int64_t all, int ctas) {
  return min(static_cast<int64_t>(ctas), max(all / kMinRun, static_cast<int64_t>(all > 0)));
}

// The plan, by one CTA: the query blocks (request, block) in order, the exclusive
// sums of their units, and the borders of the CTAs' runs.
constexpr int kPlanItems = 1536;   // sums kept in shared memory for the search of the borders

template <int BN>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const Params P, int per, int max_items, int ctas) {
  __shared__ int64_t part[33];
  __shared__ int64_t s_pre[kPlanItems + 1];
  __shared__ int2 s_item[kPlanItems];
  __shared__ int64_t s_first[kPlanThreads];
  __shared__ int64_t s_border[kMaxCtas + 1];
  gr::pdl_trigger();
  int64_t items = 0, total;
  int bad = 0;
  for (int r0 = 0; r0 < P.num_seqs; r0 += kPlanThreads) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    const int nb = r < P.num_seqs ? blocks_of(load_seq(P, r, &bad), per) : 0;
    s_first[threadIdx.x] = block_scan<kPlanThreads>(nb, total, part);
    __syncthreads();
    // this pass's blocks, each by the last request that starts at or before it
    for (int64_t i = threadIdx.x; i < total && items + i < max_items; i += kPlanThreads) {
      const int lo = last_le(s_first, kPlanThreads, i);
      const int2 it = make_int2(r0 + lo, static_cast<int>(i - s_first[lo]));
      P.item[items + i] = it;
      if (items + i < kPlanItems) s_item[items + i] = it;
    }
    items += total;
  }
  if (bad && P.err) atomicOr(P.err, GR_DEVERR_BAD_RECORD);
  if (items > max_items) items = max_items;
  __syncthreads();
  int64_t units = 0;
  for (int64_t i0 = 0; i0 < items; i0 += kPlanThreads) {
    const int64_t i = i0 + threadIdx.x;
    int64_t u = 0;
    if (i < items) {
      const int2 it = i < kPlanItems ? s_item[i] : P.item[i];
      const Seq s = load_seq(P, it.x);
      u = key_tiles<BN>(s, P.causal, it.y * per, min(s.n, (it.y + 1) * per)).n + kCost;
    }
    const int64_t ex = block_scan<kPlanThreads>(u, total, part);
    if (i < items) {
      P.pre[i] = units + ex;
      if (i < kPlanItems) s_pre[i] = units + ex;
    }
    units += total;
  }
  if (threadIdx.x == 0) {
    P.pre[items] = units;
    P.items[0] = static_cast<int>(items);
    if (items <= kPlanItems) s_pre[items] = units;
  }
  __syncthreads();
  const int64_t* pre = items <= kPlanItems ? s_pre : P.pre;
  const int64_t all = units * P.kv_heads, runs = runs_of(all, ctas);
  const int c = threadIdx.x, n = static_cast<int>(items);
  const Border at = border(pre, n, units, all, runs, c);
  if (c <= ctas) s_border[c] = at.whole;
  __syncthreads();
  // the longest run of whole pairs
  const bool longer = c < ctas && s_border[c + 1] - s_border[c] > all / max(runs, static_cast<int64_t>(1)) + kJoin;
  const bool cut = __syncthreads_or(longer);
  if (c <= ctas) {
    // with the pair of the unit before the border
    Run r{cut ? at.even : at.whole, P.kv_heads - 1, n - 1};
    if (c < runs && r.u > at.pair) {
      r.head = at.head;
      r.item = at.item;
    } else if (c < runs) {
      r.head = at.item > 0 ? at.head : at.head - 1;
      r.item = at.item > 0 ? at.item - 1 : n - 1;
    }
    P.run[c] = r;
  }
}

// The same for a small batch, by every CTA for itself in its shared memory: one
// launch less, and the sums are a few hundred cycles.
template <class S>
__device__ __forceinline__ void plan_small(const Params& P, Shared* sh) {
  const int tid = threadIdx.x, ctas = gridDim.x;
  const int per = S::NQ * P.tp;
  int64_t total;
  int bad = 0;
  const int nb = tid < P.num_seqs ? blocks_of(load_seq(P, tid, &bad), per) : 0;
  const int64_t first = block_scan<S::kThreads>(nb, total, sh->part);
  if (bad && blockIdx.x == 0 && P.err) atomicOr(P.err, GR_DEVERR_BAD_RECORD);
  const int items = static_cast<int>(min(total, static_cast<int64_t>(kSmallItems)));
  if (tid <= P.num_seqs && tid <= kMaxCtas) sh->border[tid] = static_cast<int>(first);   // (for the search)
  __syncthreads();
  int64_t u = 0;
  if (tid < items) {
    const int r = last_le(sh->border, P.num_seqs, tid), b = tid - sh->border[r];
    const Seq s = load_seq(P, r);
    u = key_tiles<S::BN>(s, P.causal, b * per, min(s.n, (b + 1) * per)).n + kCost;
    sh->req[tid] = static_cast<uint8_t>(r);
    sh->blk[tid] = static_cast<uint8_t>(b);
  }
  int64_t units;
  const int64_t before = block_scan<S::kThreads>(u, units, sh->part);
  if (tid <= items) sh->pre[tid] = static_cast<int>(tid < items ? before : units);
  if (tid == 0) sh->items = items;
  __syncthreads();
  const int64_t all = units * P.kv_heads, runs = runs_of(all, ctas);
  const Border at = border(sh->pre, items, units, all, runs, tid);
  if (tid <= ctas) sh->border[tid] = static_cast<int>(at.whole);
  __syncthreads();
  const bool longer =
      tid < ctas && sh->border[tid + 1] - sh->border[tid] > all / max(runs, static_cast<int64_t>(1)) + kJoin;
  if (__syncthreads_or(longer) && tid <= ctas) sh->border[tid] = static_cast<int>(at.even);
}

__device__ __forceinline__ int tile_at(const Work& k, int j) { return j < k.ta ? j : j - k.ta + k.tb; }

// ---------------------------------------------------------------- roles
template <class S>
struct Ring {        // position in the ring of key and value tiles
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == S::kStages) {
      stage = 0;
      phase ^= 1u;
    }
  }
};

// The next (block, head) of the run; false at its end or when a wait gave up.
__device__ __forceinline__ bool next_work(Shared* sh, uint32_t& seq, Work& k) {
  const int at = seq % kWorkRing;
  if (!wait(sh, &sh->wk_full[at], (seq / kWorkRing) & 1u, kPairTries)) return false;
  k = sh->work[at];
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&sh->wk_empty[at]);
  ++seq;
  return k.slots > 0;
}

// Warp 3: walks the CTA's run from its end and hands out its pairs ahead of their
// use.  A pair of n key tiles spans kCost + n units: a border in the first kCost
// leaves it whole, a border behind cuts its key tiles.
template <class S>
__device__ __forceinline__ void schedule_role(const Params& P, Shared* sh) {
  const int lane = threadIdx.x & 31;
  const auto run_at = [&](int c) { return P.small ? static_cast<int64_t>(sh->border[c]) : P.run[c].u; };
  const int items = P.small ? sh->items : P.items[0];
  const int64_t begin = run_at(blockIdx.x);
  const int per = S::NQ * P.tp;
  int64_t u = run_at(blockIdx.x + 1);
  // the pair of the run's last unit, and where that begins
  int head, last;
  int64_t beg;
  if (P.small) {
    const int units = sh->pre[items];
    head = static_cast<int>((u - 1) / units);
    last = last_le(sh->pre, items, u - 1 - static_cast<int64_t>(head) * units);
    beg = static_cast<int64_t>(head) * units + sh->pre[last];
  } else {
    head = P.run[blockIdx.x + 1].head;
    last = P.run[blockIdx.x + 1].item;
    beg = head * P.pre[items] + P.pre[last];
  }
  uint32_t seq = 0;
  for (int i = last; u > begin; --i) {
    if (i < 0) {
      --head;
      i = items - 1;
    }
    const int2 it = P.small ? make_int2(sh->req[i], sh->blk[i]) : P.item[i];
    const Seq s = load_seq(P, it.x);
    Work k;
    k.req = it.x;
    k.q0 = s.q0;
    k.len = s.len;
    k.ctx = s.ctx;
    k.tail = s.tail;
    k.steps = s.steps;
    k.t0 = it.y * per;
    k.nt = min(s.n - k.t0, per);
    k.slots = k.nt > P.tp ? 2 : 1;
    k.kvh = head;
    const Tiles t = key_tiles<S::BN>(s, P.causal, k.t0, k.t0 + k.nt);
    k.ta = t.a;
    k.tb = t.b;
    k.n = t.n;
    const int span = t.n + kCost;
    if (u <= beg) beg = u - span;                    // behind the first pair
    const int hi = static_cast<int>(u - beg);        // end of the run in the pair
    const int lo = static_cast<int>(max(begin - beg, static_cast<int64_t>(0)));
    k.j0 = max(lo - kCost, 0);
    k.j1 = max(hi - kCost, 0);
    u = beg + lo;
    if (k.j1 <= k.j0) continue;
    k.part0 = blockIdx.x;
    if (k.j0 > 0 && k.j1 == k.n)                     // this CTA joins the parts
      do --k.part0; while (k.part0 > 0 && run_at(k.part0) > beg + kCost);
    const int at = seq % kWorkRing;
    if (!wait(sh, &sh->wk_empty[at], ((seq / kWorkRing) & 1u) ^ 1u, kPairTries)) return;
    if (lane == 0) {
      sh->work[at] = k;
      mbar_arrive(&sh->wk_full[at]);
    }
    ++seq;
  }
  const int at = seq % kWorkRing;
  if (!wait(sh, &sh->wk_empty[at], ((seq / kWorkRing) & 1u) ^ 1u, kPairTries)) return;
  if (lane == 0) {
    sh->work[at].slots = 0;
    mbar_arrive(&sh->wk_full[at]);
  }
}

// Warp 0: the block's queries once, then its key tiles; warp 2: its value tiles;
// `part` of the warps that share the tiles' copies (an issue takes some 100 cycles,
// and single tokens over blocks of 16 rows need 32 copies per 2 x 32 KB).
// Tiles take the ring's stages in the order in which the products first use them:
// K0 .. K(lead-1), V0, K(lead), V1, ...  A lane looks up one copy's block a tile
// ahead, one lane issues the copies.
template <class S, bool kKeys>
__device__ __forceinline__ void load_role(const Params& P, Shared* sh, uint32_t data, const CUtensorMap* mq,
                                          const CUtensorMap* map, int part) {
  const int lane = threadIdx.x & 31;
  Work k;
  Ring<S> ring;
  uint32_t qphase = 0, seq = 0, mine = 0;       // mine: bit per stage this warp has filled
  bool q_issued = false, ok = true;
  const uint32_t ringbase = data + S::NQ * S::kQTile;
  const int boxes = S::BN / P.box;
  const int oob = static_cast<int>(P.num_blocks);
  constexpr int kLead = S::NQ == 2 ? 1 : 2;
  int bad = 0;
  while (ok && next_work(sh, seq, k)) {
    if (kKeys && part == 0) {
      if (!wait(sh, &sh->q_empty, qphase ^ 1u, kPairTries)) break;
      if (lane == 0 && !(P.flags & 1)) {
        const int slots = S::NQ == 2 ? k.slots : 1;
        mbar_arrive_expect_tx(&sh->q_full, static_cast<uint32_t>(slots * S::CH * P.group * P.tp * 128));
        for (int q = 0; q < slots; ++q)
          for (int x = 0; x < S::CH; ++x)
            tma_load3(data + q * S::kQTile + x * S::kChunkQ, mq, x * 64, k.kvh * P.group, k.q0 + k.t0 + q * P.tp,
                      &sh->q_full);
        q_issued = true;
      }
      qphase ^= 1u;
    }
    const int n = k.j1 - k.j0;
    const int32_t* row = P.table + k.req * P.table_stride;
    // box `lane` of tile j: its block, and its first row in the block
    const auto look = [&](int j, int& id, int& off) {
      const int tok = tile_at(k, k.j0 + j) * S::BN + lane * P.box;
      const int blk = static_cast<int>(__umulhi(static_cast<uint32_t>(tok), P.div_mul) >> P.div_shift);
      id = oob;
      off = tok - blk * P.block_size;
      if (lane < boxes && tok < k.len) {
        const int v = __ldg(row + blk);
        if (v < 0 || v >= oob) bad = 1; else id = v;
      }
    };
    int id, off;
    look(0, id, off);
    for (int x = 0, ki = 0, vi = 0; x < 2 * S::SUB * n; ++x, ring.next()) {
      // (key and value stages, SUB to a tile)
      const bool is_k = ki < n * S::SUB && ki / S::SUB < vi / S::SUB + kLead && (vi % S::SUB == 0 || ki % S::SUB != 0);
      const int js = is_k ? ki++ : vi++;
      if (is_k != kKeys) continue;
      const int j = js / S::SUB, sub = js % S::SUB;
      const int id0 = id, off0 = off;
      if (sub == S::SUB - 1 && j + 1 < n) look(j + 1, id, off);
      if (!wait(sh, &sh->empty[ring.stage], ring.phase ^ 1u)) {
        ok = false;
        break;
      }
      if (!(P.flags & 1)) {
        if (part == 0 && lane == 0) mbar_arrive_expect_tx(&sh->full[ring.stage], S::kStage);
        mine |= 1u << ring.stage;
        const uint32_t dst = ringbase + ring.stage * S::kStage;
        for (int i = part; i < boxes; i += S::kLoaders) {
          const int b = __shfl_sync(0xFFFFFFFFu, id0, i), r = __shfl_sync(0xFFFFFFFFu, off0, i);
          if (lane == 0) {
#pragma unroll
            for (int c = 0; c < S::CHS; ++c)
              tma_load4(dst + c * S::kChunkKV + i * P.box * 128, map, (sub * S::CHS + c) * 64, k.kvh, r, b,
                        &sh->full[ring.stage]);
          }
        }
      }
    }
  }
  if (__any_sync(0xFFFFFFFFu, bad) && lane == 0 && P.err) atomicOr(P.err, GR_DEVERR_BAD_SLOT);
  // stays until the products have used the run's last tile, whichever warps loaded it: a role that
  // gives up after this warp's last issue finds it here, to wait for what is still in flight
  {
    const bool lap = ring.stage == 0;
    wait(sh, &sh->empty[lap ? S::kStages - 1 : ring.stage - 1], ring.phase ^ static_cast<uint32_t>(lap));
  }
  if (aborted(sh)) {
    // gave up: wait (bounded) for this warp's copies in flight before the shared memory goes
    for (int i = 0; i < S::kStages; ++i) {
      if (ring.stage == 0) {
        ring.stage = S::kStages;
        ring.phase ^= 1u;
      }
      --ring.stage;
      if (mine >> ring.stage & 1u) gr::mbar_wait_bounded(&sh->full[ring.stage], ring.phase);
    }
    if (__any_sync(0xFFFFFFFFu, q_issued)) gr::mbar_wait_bounded(&sh->q_full, qphase ^ 1u);
  }
}

// Warp 1: the matrix products, issued by one lane.  The issue of a product holds
// the warp about as long as the product takes, so whatever it does between two
// batches is time that the tensor pipe stands still.  All control flow is by the
// whole warp, so that operands are known to be uniform (2 to 6 % fewer cycles than
// a role of one lane: a prompt of 8192, 32 x 128 beams).
template <class S, bool kBf16>
__device__ __forceinline__ void mma_role(const Params& P, Shared* sh, uint32_t data) {
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, sh->tmem, 0);
  const bool leader = elect_lane();
  const auto commit = [&](uint64_t* bar) {
    if (leader) tc_commit(bar);
  };
  const uint32_t ringbase = data + S::NQ * S::kQTile;
  constexpr uint32_t kFmt = kBf16 ? 1u : 0u;
  // fp32 accumulators, A and B of one type, M = 128; B of the second product is stored along N
  constexpr uint32_t kIdescS = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((S::BN / 8) << 17) | ((kRows / 16) << 24);
  constexpr uint32_t kIdescO =
      (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((S::CHS * 64 / 8) << 17) | ((kRows / 16) << 24);

  const auto qk = [&](int q, int buf, int stage, int sub) {   // S[buf] (+)= Q[q] K^T over the stage's columns
    const uint64_t qa = smem_desc(data + q * S::kQTile + sub * S::CHS * S::kChunkQ, 16, 1024);
    const uint64_t ka = smem_desc(ringbase + stage * S::kStage, 16, 1024);
    if (leader) {
#pragma unroll
      for (int c = 0; c < S::CHS; ++c)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          tc_mma_ss(tmem + buf * S::BN, qa + ((c * S::kChunkQ + x * 32) >> 4), ka + ((c * S::kChunkKV + x * 32) >> 4),
                    kIdescS, (sub | c | x) != 0);
    }
    if (sub == S::SUB - 1) commit(&sh->s_full[buf]);
  };
  const auto pv = [&](int q, int buf, int stage, bool first, int sub) {   // the stage's columns of O[q] (+)= P[buf] V
    const uint64_t va = smem_desc(ringbase + stage * S::kStage, S::kChunkKV, 1024);
    if (leader) {
#pragma unroll
      for (int x = 0; x < S::BN / 16; ++x)
        tc_mma_ts(tmem + S::kColO + q * S::DP + sub * S::CHS * 64, tmem + buf * S::BN + x * 8, va + ((x * 2048) >> 4),
                  kIdescO, !(first && x == 0));
    }
    if (sub == S::SUB - 1) commit(&sh->pv_done[S::NQ == 2 ? q : buf]);
  };

  Ring<S> ring;
  uint32_t qphase = 0, pphase = 0, ofree = 3;   // one bit per buffer / tile
  uint32_t step = 0;    // score buffer of the next step (kNQ = 1)
  const auto take = [&](int& stage) {           // the next key or value tile
    if (!wait(sh, &sh->full[ring.stage], ring.phase)) return false;
    tc_fence_after();
    stage = ring.stage;
    ring.next();
    return true;
  };
  const auto probs = [&](int buf) {
    if (!wait(sh, &sh->p_full[buf], (pphase >> buf) & 1u)) return false;
    pphase ^= 1u << buf;
    return true;
  };
  const auto o_free = [&](int q) {              // the accumulator's last contents are read
    if (!wait(sh, &sh->o_free[q], (ofree >> q) & 1u)) return false;
    ofree ^= 1u << q;
    return true;
  };
  for (uint32_t seq = 0;; ++seq) {
    const int at = seq % kWorkRing;
    if (!wait(sh, &sh->wk_full[at], (seq / kWorkRing) & 1u, kPairTries)) return;
    const int slots = __shfl_sync(0xFFFFFFFFu, sh->work[at].slots, 0);
    const int n = __shfl_sync(0xFFFFFFFFu, sh->work[at].j1 - sh->work[at].j0, 0);
    if (leader) mbar_arrive(&sh->wk_empty[at]);
    if (slots == 0) return;
    if (!wait(sh, &sh->q_full, qphase)) return;
    qphase ^= 1u;
    int kstage = 0, vstage = 0;
    if (S::NQ == 2) {
      if (!take(kstage)) return;
      for (int q = 0; q < slots; ++q) qk(q, q, kstage, 0);
      commit(&sh->empty[kstage]);
      if (n == 1) commit(&sh->q_empty);
      for (int j = 0; j < n; ++j) {
        for (int q = 0; q < slots; ++q) {
          const bool last = q == slots - 1;
          if (q == 0 && !take(vstage)) return;
          if (j == 0 && !o_free(q)) return;
          if (!probs(q)) return;
          tc_fence_after();
          pv(q, q, vstage, j == 0, 0);
          if (last) commit(&sh->empty[vstage]);
          if (j + 1 < n) {
            if (q == 0 && !take(kstage)) return;
            qk(q, q, kstage, 0);
            if (last) {
              commit(&sh->empty[kstage]);
              if (j + 2 == n) commit(&sh->q_empty);
            }
          }
        }
      }
    } else {
      const auto keys = [&](int buf) {
#pragma unroll
        for (int sub = 0; sub < S::SUB; ++sub) {
          if (!take(kstage)) return false;
          qk(0, buf, kstage, sub);
          commit(&sh->empty[kstage]);
        }
        return true;
      };
      for (int j = 0; j < 2 && j < n; ++j) {
        if (!keys((step + j) & 1)) return;
        if (j + 1 == n) commit(&sh->q_empty);
      }
      for (int j = 0; j < n; ++j, ++step) {
        const int b = step & 1;
        if (!take(vstage)) return;
        if (j == 0 && !o_free(0)) return;
        if (!probs(b)) return;
        tc_fence_after();
        pv(0, b, vstage, j == 0, 0);
        commit(&sh->empty[vstage]);
#pragma unroll
        for (int sub = 1; sub < S::SUB; ++sub) {
          if (!take(vstage)) return;
          pv(0, b, vstage, j == 0, sub);
          commit(&sh->empty[vstage]);
        }
        if (j + 2 < n) {
          if (!keys(b)) return;
          if (j + 3 == n) commit(&sh->q_empty);
        }
      }
    }
  }
}

// Value rows behind the last key hold whatever the block held before, and
// 0 * NaN is NaN: the softmax warps of the first tile zero them before they
// hand over the probabilities that the product takes with these rows.
template <class S>
__device__ __forceinline__ void zero_tail(uint32_t tile, int from, int to) {
  const int n = (to - from) * 8;
  for (int e = threadIdx.x & 127; e < n * S::CHS; e += 128) {
    const int c = e / n, x = e - c * n;
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(tile + c * S::kChunkKV + from * 128 + x * 16), "r"(0)
                 : "memory");
  }
  gr::fence_proxy_async_smem();
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void st_release(uint64_t* p, uint64_t v) {
  asm volatile("st.release.gpu.global.b64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __forceinline__ uint64_t ld_acquire(const uint64_t* p) {
  uint64_t v;
  asm volatile("ld.acquire.gpu.global.b64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}

// 32 output columns from col on, as far as the head dim goes.
template <bool kBf16>
__device__ __forceinline__ void store32(const Params& P, unsigned char* row, int col, const float4* v) {
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    uint32_t w[8];
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      w[2 * z] = pack16<kBf16>(v[4 * y + z].x, v[4 * y + z].y);
      w[2 * z + 1] = pack16<kBf16>(v[4 * y + z].z, v[4 * y + z].w);
    }
    const int at = col + y * 16;
    unsigned char* to = row + at * 2;
    if (P.out32) {            // whole sectors; the head dim is a multiple of 16 then
      if (at < P.dim) st_global_32(to, w);
    } else {
      if (at < P.dim) *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
      if (at + 8 < P.dim) *reinterpret_cast<uint4*>(to + 16) = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
}

// Where CTA p has left its part of a pair that another one owns.
template <class S>
__device__ __forceinline__ int64_t part_at(int p, int slot) {
  return (static_cast<int64_t>(p) * 2 + 1) * S::NQ + slot;
}

// Waits (bounded; runs of many seconds may end some seconds apart) until the CTAs
// from part0 up to this one have left this warp's rows of their parts.
__device__ __forceinline__ bool wait_parts(const Params& P, Shared* sh, int part0, int slot, int warp) {
  bool ok = true;
  const uint64_t since = gr::global_timer_ns();
  for (int p = part0 + (threadIdx.x & 31); p < static_cast<int>(blockIdx.x); p += 32) {
    while (ok && ld_acquire(P.flag + (p * 2 + slot) * 4 + warp) != P.token)
      ok = *reinterpret_cast<volatile int*>(&sh->abort) == 0 && gr::global_timer_ns() - since < 10 * gr::kWaitLimitNs;
  }
  if (__all_sync(0xFFFFFFFFu, ok)) {
    __syncwarp();   // a vote orders no memory: all lanes read what each lane's flags stand for
    return true;
  }
  *reinterpret_cast<volatile int*>(&sh->abort) = 1;
  return false;
}

// The parts are read: their flags go back to 0, so that a replay of this call, which has the same
// token, waits again.
__device__ __forceinline__ void free_parts(const Params& P, int part0, int slot, int warp) {
  __syncwarp();
  for (int p = part0 + (threadIdx.x & 31); p < static_cast<int>(blockIdx.x); p += 32)
    P.flag[(p * 2 + slot) * 4 + warp] = 0;
}

// The join of a warp of at most 32 / kEach rows (single tokens, often cut over
// many CTAs): kEach lanes a row, this CTA's part read back from its place 0, and as
// many parts in flight as 32 vectors per lane allow.
template <class S, bool kBf16, int kEach>
__device__ __forceinline__ void join_few(const Params& P, const Work& k, int slot, int warp, int rows) {
  constexpr int kVecs = S::DP / 4 / kEach < 8 ? S::DP / 4 / kEach : 8;   // a lane's vectors of a part at a time
  constexpr int kAhead = 32 / kVecs;
  const int lane = threadIdx.x & 31;
  const int cta = blockIdx.x, parts = cta - k.part0 + 1;
  const int r = lane % (32 / kEach), q = lane / (32 / kEach);
  const int m_row = warp * 32 + min(r, rows - 1);
  const auto place = [&](int i) {
    const int p = k.part0 + i;
    return p == cta ? static_cast<int64_t>(p) * 2 * S::NQ + slot : part_at<S>(p, slot);
  };
  float top = -kInf;
#pragma unroll 4
  for (int i = q; i < parts; i += kEach) top = fmaxf(top, __ldcg(P.part_lse + place(i) * kRows + m_row));
#pragma unroll
  for (int o = 32 / kEach; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  const float ref = top == -kInf ? 0.0f : top;
  const int ti = m_row / P.group, g = m_row - ti * P.group;
  const int64_t t = static_cast<int64_t>(k.q0) + k.t0 + slot * P.tp + ti;
  const int h = k.kvh * P.group + g;
  unsigned char* orow = static_cast<unsigned char*>(P.out) + (t * P.out_tok + h * P.out_head) * 2;
#pragma unroll 1
  for (int x = q * kVecs * 4; x < S::DP; x += kEach * kVecs * 4) {
    float4 acc[kVecs];
#pragma unroll
    for (int y = 0; y < kVecs; ++y) acc[y] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
#pragma unroll 1
    for (int i = 0; i < parts; i += kAhead) {
      float4 v[kAhead][kVecs];
      float w[kAhead];
#pragma unroll
      for (int z = 0; z < kAhead; ++z) {
        const int64_t at = place(min(i + z, parts - 1));
        w[z] = i + z < parts ? __ldcg(P.part_lse + at * kRows + m_row) : -kInf;
#pragma unroll
        for (int y = 0; y < kVecs; ++y) v[z][y] = __ldcg(P.part_o + (at * (S::DP / 4) + x / 4 + y) * kRows + m_row);
      }
#pragma unroll
      for (int z = 0; z < kAhead; ++z) {
        if (i + z >= parts) break;
        const float wz = gr::fast_exp2(w[z] - ref);
        sum += wz;
#pragma unroll
        for (int y = 0; y < kVecs; ++y) {
          acc[y].x += wz * v[z][y].x;
          acc[y].y += wz * v[z][y].y;
          acc[y].z += wz * v[z][y].z;
          acc[y].w += wz * v[z][y].w;
        }
      }
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    if (r < rows) {
#pragma unroll
      for (int y = 0; y < kVecs; y += 2) {
        const int col = x + y * 4;
        if (col < P.dim)
          *reinterpret_cast<uint4*>(orow + col * 2) =
              make_uint4(pack16<kBf16>(acc[y].x * inv, acc[y].y * inv), pack16<kBf16>(acc[y].z * inv, acc[y].w * inv),
                         pack16<kBf16>(acc[y + 1].x * inv, acc[y + 1].y * inv),
                         pack16<kBf16>(acc[y + 1].z * inv, acc[y + 1].w * inv));
      }
      if (x == 0 && P.lse)
        P.lse[t * P.heads + h] = sum > 0.0f || sum != sum ? (ref + __log2f(sum)) * kLn2 : -kInf;
    }
  }
}

// The n lowest bits (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n >= 32 ? 0xFFFFFFFFu : (n <= 0 ? 0u : (1u << n) - 1u);
}

// The last warps: softmax of one query tile, one thread per row; also the rare
// rescaling of the accumulator, and the block's output.
template <class S, bool kBf16>
__device__ __forceinline__ void softmax_role(const Params& P, Shared* sh, uint32_t data, int slot) {
  constexpr int BN = S::BN, DP = S::DP;
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) & 3;
  const int m_row = warp * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
  const uint32_t tmem = sh->tmem + lanes;
  const uint32_t o_col = tmem + S::kColO + slot * DP;
  const float c = P.scale_log2;
  const int ti = m_row / P.group, g = m_row - ti * P.group;
  Work k;
  uint32_t seq = 0, sphase = 0, pvphase = 0;   // one bit per buffer
  uint32_t step = 0, tiles = 0;                // score buffer of the next step, tiles through the ring
  for (; next_work(sh, seq, k); tiles += 2 * S::SUB * (k.j1 - k.j0)) {
    if (S::NQ == 2 && slot >= k.slots) continue;
    const int n = k.j1 - k.j0;
    // this row: token, position, the keys it sees
    const int tok = k.t0 + slot * P.tp + ti;              // in the request
    const bool live = ti < P.tp && ti + slot * P.tp < k.nt;
    const int pos = k.ctx + tok;
    int lim = P.causal ? min(pos + 1, k.len) : k.len;
    int first = 0x7FFFFFFF, own = 0;
    if (k.steps > 0 && tok >= k.tail) {
      first = k.ctx + k.tail;
      own = first + (tok - k.tail) / k.steps * k.steps;
    }
    if (!live) lim = 0x7FFFFFFF, first = 0x7FFFFFFF;      // rows of no token: no mask, nothing stored
    const bool any_live = __any_sync(0xFFFFFFFFu, live);
    float m = -kInf, l = 0.0f;
    for (int j = 0; j < n; ++j) {
      const int b = S::NQ == 2 ? slot : static_cast<int>((step + j) & 1);
      const int key0 = tile_at(k, k.j0 + j) * BN;
      if (!wait(sh, &sh->s_full[b], (sphase >> b) & 1u)) return;
      sphase ^= 1u << b;
      tc_fence_after();
      // which product into O has finished when: kNQ = 2 orders it before these
      // scores, kNQ = 1 does not (the other buffer's is still to come)
      if (any_live) {
        const uint32_t s_col = tmem + b * BN;
        uint32_t sr[BN / 32][32], p[BN / 2];
        const auto load = [&] {   // the tile's scores, -inf where the row does not see the key
#pragma unroll
          for (int x = 0; x < BN / 32; ++x) tc_ld32(sr[x], s_col + x * 32);
          tc_wait_ld();
          const bool whole = key0 + BN <= lim && (key0 + BN <= first || key0 >= own);
          if (!__all_sync(0xFFFFFFFFu, whole)) {
            // one bit per key, then one select per score (comparisons per score
            // made this path 5 us per tile)
#pragma unroll
            for (int x = 0; x < BN / 32; ++x) {
              const uint32_t see = low_bits(lim - key0 - x * 32) &
                                   (low_bits(first - key0 - x * 32) | ~low_bits(own - key0 - x * 32));
#pragma unroll
              for (int y = 0; y < 32; ++y) sr[x][y] = see & (1u << y) ? sr[x][y] : 0xFF800000u;
            }
          }
        };
        const auto score = [&](int x) { return __uint_as_float(sr[x / 32][x % 32]); };
        const auto maximum = [&] {
          float t[4] = {-kInf, -kInf, -kInf, -kInf};
#pragma unroll
          for (int x = 0; x < BN; x += 2) t[x / 2 % 4] = max3(t[x / 2 % 4], score(x), score(x + 1));
          return max3(fmaxf(t[0], t[1]), t[2], t[3]);
        };
        // p = 2^(c s - c m), rounded; returns the unrounded sum
        const auto exponentials = [&] {
          const float mc = m == -kInf ? 0.0f : m * c;
          const uint64_t c2 = gr::pack2(c, c), n2 = gr::pack2(-mc, -mc);
          uint64_t a0 = 0, a1 = 0;   // (0.0f, 0.0f)
#pragma unroll
          for (int x = 0; x < BN; x += 2) {
            float e0, e1;
            gr::unpack2(gr::ffma2(gr::pack2(score(x), score(x + 1)), c2, n2), e0, e1);
            e0 = gr::fast_exp2(e0);
            e1 = gr::fast_exp2(e1);
            if (x & 2) a1 = gr::fadd2(a1, gr::pack2(e0, e1)); else a0 = gr::fadd2(a0, gr::pack2(e0, e1));
            p[x / 2] = pack16<kBf16>(e0, e1);
          }
          float x0, x1;
          gr::unpack2(gr::fadd2(a0, a1), x0, x1);
          return x0 + x1;
        };
        // a later tile's maximum becomes the reference: what is there of l and O is scaled
        const auto rescale = [&](bool grow, float top) {
          const float f = grow ? gr::fast_exp2((m - top) * c) : 1.0f;   // m = -inf: 0
          if (grow) m = top;
          l *= f;
          if (j == 0) return true;
          if (S::NQ == 1) {
            const int pb = b ^ 1;   // the previous key tile's product
            if (!wait(sh, &sh->pv_done[pb], ((pvphase >> pb) & 1u) ^ 1u)) return false;
            tc_fence_after();
          }
#pragma unroll 1
          for (int x = 0; x < DP; x += 32) {
            uint32_t o[32];
            tc_ld32(o, o_col + x);
            tc_wait_ld();
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
            tc_st32(o_col + x, o);
          }
          tc_wait_st();
          return true;
        };
        load();
        float sum;
        if constexpr (S::NQ == 2) {
          // the maximum first: a reference for the row's first keys, then only large growth counts
          const float top = maximum();
          const bool grow = live && ((top - m) * c > kRescale || (m == -kInf && top > -kInf));
          if (__any_sync(0xFFFFFFFFu, grow) && !rescale(grow, top)) return;
          sum = exponentials();
        } else {
          // One group of softmax warps is the chain's slowest link: later tiles are exponentiated
          // against the reference at hand and their maximum is taken meanwhile; where it has
          // grown too far, which is rare, the tile is done again.  (64 single tokens 304 -> 286 k
          // cycles; two query tiles, which fill each other's gaps, lose 1 to 3 % by it.)
          if (__any_sync(0xFFFFFFFFu, live && m == -kInf)) {
            const float top = maximum();
            if (m == -kInf) m = top;   // until now l = 0 and O = 0
          }
          while (true) {
            sum = exponentials();
            const float top = maximum();
            const bool grow = live && (top - m) * c > kRescale;
            if (!__any_sync(0xFFFFFFFFu, grow)) break;
            if (!rescale(grow, top)) return;
            load();
          }
        }
        l += sum;
#pragma unroll
        for (int h = 0; h < BN / 64; ++h) tc_st32(s_col + h * 32, *reinterpret_cast<uint32_t(*)[32]>(p + h * 32));
        tc_wait_st();
      }
      if (j == n - 1 && slot == 0) {
        // the pair's last value tile takes the last stages in the ring so far
        const int rows = k.len - key0;
        if (rows > 0 && rows < BN && rows % P.box != 0) {
#pragma unroll
          for (int sub = 0; sub < S::SUB; ++sub) {
            const uint32_t pos = tiles + 2 * S::SUB * n - S::SUB + sub, stage = pos % S::kStages;
            if (!wait(sh, &sh->full[stage], (pos / S::kStages) & 1u)) return;
            zero_tail<S>(data + S::NQ * S::kQTile + stage * S::kStage, rows, (rows / P.box + 1) * P.box);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->p_full[b]);
      pvphase ^= 1u << b;   // the parity of this tile's product, once flipped back
    }
    // the last product into O
    const int lb = S::NQ == 2 ? slot : static_cast<int>((step + n - 1) & 1);
    if (!wait(sh, &sh->pv_done[lb], ((pvphase >> lb) & 1u) ^ 1u)) return;
    tc_fence_after();
    if (S::NQ == 1) step += n;
    const bool owner = k.j0 > 0 && k.j1 == k.n;
    bool done = k.j0 == 0 && k.j1 == k.n;                  // this CTA stores the rows' outputs
    if (any_live) {
      const int rows = min(min(k.nt - slot * P.tp, P.tp) * P.group - warp * 32, 32);   // the warp's first lanes
      const int parts = owner ? static_cast<int>(blockIdx.x) - k.part0 : 0;            // other CTAs' parts
      float scale = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      float lse2 = l > 0.0f || l != l ? m * c + __log2f(l) : -kInf;
      float ref = 0.0f, norm = 0.0f;                       // of the join: weight of part p is 2^(lse_p - ref) norm
      if (owner && !wait_parts(P, sh, k.part0, slot, warp)) return;
      const bool direct = owner && rows > 16;              // rows stay with their lanes
      if (direct) {
        float top = lse2;
        for (int i = 0; i < parts; ++i) top = fmaxf(top, __ldcg(P.part_lse + part_at<S>(k.part0 + i, slot) * kRows + m_row));
        ref = top == -kInf ? 0.0f : top;
        const float own = gr::fast_exp2(lse2 - ref);
        float sum = own;
        for (int i = 0; i < parts; ++i)
          sum += gr::fast_exp2(__ldcg(P.part_lse + part_at<S>(k.part0 + i, slot) * kRows + m_row) - ref);
        norm = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
        scale *= own * norm;
        lse2 = sum > 0.0f || sum != sum ? ref + __log2f(sum) : -kInf;
        done = true;
      }
      const int64_t t = static_cast<int64_t>(k.q0) + tok;
      const int h = k.kvh * P.group + g;
      // a cut pair's part goes to place 1 of this CTA, where its owner looks for it; an owner's
      // own part to place 0
      const int64_t place = (static_cast<int64_t>(blockIdx.x) * 2 + (owner ? 0 : 1)) * S::NQ + slot;
      if (live) {
        if (done) {
          if (P.lse) P.lse[t * P.heads + h] = lse2 * kLn2;
        } else {
          P.part_lse[place * kRows + m_row] = lse2;
        }
      }
      unsigned char* orow = static_cast<unsigned char*>(P.out) + (t * P.out_tok + h * P.out_head) * 2;
      float4* prt = P.part_o + place * (DP / 4) * kRows + m_row;
      constexpr int kCols = 64;   // columns in registers at a time, beside those of two other parts
#pragma unroll 1
      for (int x0 = 0; x0 < DP; x0 += kCols) {
        uint32_t o[2][32];
        tc_ld32(o[0], o_col + x0);
        tc_ld32(o[1], o_col + x0 + 32);
        tc_wait_ld();
        float4 v[16];
#pragma unroll
        for (int y = 0; y < 16; ++y) {
          const uint32_t* from = &o[y / 8][y % 8 * 4];
          v[y] = make_float4(__uint_as_float(from[0]) * scale, __uint_as_float(from[1]) * scale,
                             __uint_as_float(from[2]) * scale, __uint_as_float(from[3]) * scale);
        }
        if (direct) {
#pragma unroll 1
          for (int i = 0; i < parts; i += 2) {
            float4 a[2][16];
            float wgt[2];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const int64_t at = part_at<S>(k.part0 + min(i + z, parts - 1), slot);
              wgt[z] = i + z < parts ? __ldcg(P.part_lse + at * kRows + m_row) : -kInf;
              const float4* from = P.part_o + (at * (DP / 4) + x0 / 4) * kRows + m_row;
#pragma unroll
              for (int y = 0; y < 16; ++y) a[z][y] = __ldcg(from + y * kRows);
            }
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              if (i + z >= parts) break;
              const float w = gr::fast_exp2(wgt[z] - ref) * norm;
#pragma unroll
              for (int y = 0; y < 16; ++y) {
                v[y].x = fmaf(w, a[z][y].x, v[y].x);
                v[y].y = fmaf(w, a[z][y].y, v[y].y);
                v[y].z = fmaf(w, a[z][y].z, v[y].z);
                v[y].w = fmaf(w, a[z][y].w, v[y].w);
              }
            }
          }
        }
        if (!live) continue;
        if (done) {
          store32<kBf16>(P, orow, x0, v);
          store32<kBf16>(P, orow, x0 + 32, v + 8);
        } else {
#pragma unroll
          for (int y = 0; y < 16; ++y) prt[(x0 / 4 + y) * kRows] = v[y];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->o_free[slot]);
      if (!done) {
        __syncwarp();   // orders the lanes' stores before lane 0's release, and before the reads of the join
        if (owner) {
          if (rows <= 4)
            join_few<S, kBf16, 8>(P, k, slot, warp, rows);
          else if (rows <= 8)
            join_few<S, kBf16, 4>(P, k, slot, warp, rows);
          else
            join_few<S, kBf16, 2>(P, k, slot, warp, rows);
        } else if (lane == 0) {
          st_release(P.flag + (blockIdx.x * 2 + slot) * 4 + warp, P.token);
        }
      }
      if (owner) free_parts(P, k.part0, slot, warp);
    } else {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->o_free[slot]);
    }
  }
}

template <class S, bool kBf16>
__global__ void __launch_bounds__(S::kThreads, 1)
    attention_kernel(const Params P, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv) {
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  Shared* sh = reinterpret_cast<Shared*>(raw + (base - smem_u32(raw)) + S::kData);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&sh->full[i], 1);
      mbar_init(&sh->empty[i], 1);
    }
    for (int i = 0; i < kWorkRing; ++i) {
      mbar_init(&sh->wk_full[i], 1);
      mbar_init(&sh->wk_empty[i], 2 * S::kLoaders + 1 + 4 * S::NQ);
    }
    mbar_init(&sh->q_full, 1);
    mbar_init(&sh->q_empty, 1);
    mbar_init(&sh->drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->p_full[i], 4);
      mbar_init(&sh->pv_done[i], 1);
      mbar_init(&sh->o_free[i], 4);
    }
    sh->abort = 0;
    gr::fence_mbar_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh->tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  bool busy;
  if (P.small) {
    plan_small<S>(P, sh);
    __syncthreads();
    busy = sh->border[blockIdx.x] < sh->border[blockIdx.x + 1];
  } else {
    gr::pdl_wait();      // the plan is complete
    busy = P.run[blockIdx.x].u < P.run[blockIdx.x + 1].u;
  }
  // registers: 12 warps of 168 at launch give 4 x 56 + 8 x 224 (kNQ = 2), and 8 x 80 + 4 x 240 leave some (kNQ = 1)
  static_assert(S::kThreads == 384, "register split");
  if (warp < S::kSoftmax) {
    if constexpr (S::NQ == 2) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    }
    if (!busy) {
    } else if (warp == 3) {
      schedule_role<S>(P, sh);
    } else if (warp == 1) {
      mma_role<S, kBf16>(P, sh, base);
      if (aborted(sh)) {   // products in flight finish before the tensor memory goes
        if (elect_lane()) tc_commit(&sh->drain);
        __syncwarp();
        gr::mbar_wait_bounded(&sh->drain, 0);
      }
    } else if (warp & 1) {
      load_role<S, false>(P, sh, base, &mq, &mv, warp / 2 - 1);   // 5, 7
    } else if (warp == 2) {
      load_role<S, false>(P, sh, base, &mq, &mv, 0);
    } else {
      load_role<S, true>(P, sh, base, &mq, &mk, warp / 2 - (warp > 0));   // 0, 4, 6
    }
  } else {
    if constexpr (S::NQ == 2) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 240;");
    }
    if (busy) softmax_role<S, kBf16>(P, sh, base, (warp - S::kSoftmax) >> 2);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && sh->abort && P.err) atomicOr(P.err, GR_DEVERR_TIMEOUT);
  if (warp == 2) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh->tmem));
  }
}

// ---------------------------------------------------------------- host
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static std::mutex g_mu;
static int g_sms[64];
static bool g_attr[64][6][2];

static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

struct Geometry {
  int dp, nq, bn, group, tp, box;
  int64_t max_items;
};

// What the descriptor allows, and the kernel that it picks.
static int geometry(const gr_paged_attn_desc* d, Geometry& g) {
  if (!d) return GR_ERR_NULL;
  if (d->num_seqs < 0 || d->num_tokens < 0 || d->num_heads <= 0 || d->num_kv_heads <= 0 || d->head_dim <= 0 ||
      d->block_size <= 0 || d->max_blocks < 0 || d->num_blocks < 0 || d->num_blocks >= 0x7FFFFFFF ||
      d->num_heads % d->num_kv_heads != 0 || (d->causal != 0 && d->causal != 1) || d->max_query_len < 0 ||
      !(d->scale > 0.0f) || d->scale > 2.0e38f || (d->num_seqs > 1 && d->table_stride < d->max_blocks) ||
      static_cast<int64_t>(d->max_blocks) * d->block_size > 0x7FFFFFFF - 1023 ||
      d->num_tokens > 0x7FFFFFFF - 1023 || d->num_seqs > 0x7FFFFFFF - 1023)
    return GR_ERR_BAD_DESC;
  if (d->dtype != GR_DTYPE_BF16 && d->dtype != GR_DTYPE_F16) return GR_ERR_DTYPE;
  g.group = d->num_heads / d->num_kv_heads;
  if (d->head_dim % 8 != 0 || d->head_dim > 256 || d->block_size % 8 != 0 || g.group > kRows) return GR_ERR_UNSUPPORTED;
  g.dp = d->head_dim <= 64 ? 64 : (d->head_dim <= 128 ? 128 : 256);
  g.tp = kRows / g.group;
  // one query tile where the longest query fits it, or the accumulators of two do not
  g.nq = (g.dp == 256 || static_cast<int64_t>(d->max_query_len) <= g.tp) ? 1 : 2;
  g.bn = 128;
  g.box = 8;
  while (g.box * 2 <= g.bn && d->block_size % (g.box * 2) == 0) g.box *= 2;
  const int64_t per = static_cast<int64_t>(g.nq) * g.tp;
  // one more for each request with tokens than whole blocks
  const int64_t some = d->num_seqs < d->num_tokens ? d->num_seqs : d->num_tokens;
  g.max_items = static_cast<int64_t>(d->num_tokens) / per + some;
  if (g.max_items > d->num_tokens) g.max_items = d->num_tokens;
  if (g.max_items > 0x7FFFFFFF) return GR_ERR_UNSUPPORTED;
  return GR_OK;
}

// Whether every CTA plans for itself: few query blocks, and units that fit 32 bits.
static bool small_plan(const gr_paged_attn_desc* d, const Geometry& g) {
  const int64_t tiles = static_cast<int64_t>(d->max_blocks) * d->block_size / 128 + 1 + kCost;
  return d->num_seqs <= kSmallItems && g.max_items <= kSmallItems &&
         tiles * kSmallItems * d->num_kv_heads < 0x7FFFFFFF;
}

// A number that no other call of this process has, and that stale memory holds by a chance of 2^-64.
static uint64_t next_token() {
  static std::atomic<uint64_t> next{static_cast<uint64_t>(std::chrono::steady_clock::now().time_since_epoch().count()) *
                                        0x9E3779B97F4A7C15ull ^ reinterpret_cast<uintptr_t>(&g_attr)};
  uint64_t t = next.fetch_add(0x9E3779B97F4A7C15ull, std::memory_order_relaxed);
  return t != 0 ? t : next.fetch_add(0x9E3779B97F4A7C15ull, std::memory_order_relaxed);
}

static size_t round256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

struct Layout {
  size_t run, flag, part_lse, part_o, pre, item, items, total;
};
static Layout layout(const gr_paged_attn_desc* d, const Geometry& g) {
  Layout l{};
  size_t at = 0;
  const auto take = [&](size_t n) {
    const size_t here = at;
    at += round256(n);
    return here;
  };
  l.run = take(sizeof(Run) * (kMaxCtas + 1));
  l.flag = take(sizeof(uint64_t) * kMaxCtas * 8);
  l.part_lse = take(sizeof(float) * kMaxCtas * 2 * g.nq * kRows);
  l.part_o = take(sizeof(float) * static_cast<size_t>(kMaxCtas) * 2 * g.nq * kRows * g.dp);
  l.pre = take(sizeof(int64_t) * (g.max_items + 1));
  l.item = take(sizeof(int2) * g.max_items);
  l.items = take(sizeof(int32_t));
  l.total = at;
  return l;
}

static bool encode(CUtensorMap* m, bool bf16, int rank, const void* base, const cuuint64_t* dims,
                   const cuuint64_t* strides, const cuuint32_t* box) {
  const EncodeFn fn = encode_fn();
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  return fn && fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                  const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K, typename... A>
static cudaError_t launch(K kern, dim3 grid, int threads, size_t smem, cudaStream_t s, bool after_own, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_own ? 1 : 0;   // only behind this call's own kernels
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <class S, bool kBf16>
static int run(const Params& P, const Geometry& g, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
               int dev, int sms, int kind, cudaStream_t s) {
  const size_t smem = 1024 + S::kData + sizeof(Shared);
  static_assert(1024 + S::kData + sizeof(Shared) <= kSmemMax, "shared memory");
  {
    std::lock_guard<std::mutex> lock(g_mu);
    if (!g_attr[dev][kind][kBf16]) {
      if (cudaFuncSetAttribute(attention_kernel<S, kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(smem)) != cudaSuccess)
        return GR_ERR_CUDA;
      g_attr[dev][kind][kBf16] = true;
    }
  }
  const int ctas = sms < kMaxCtas ? sms : kMaxCtas;
  if (!P.small &&
      launch(plan_kernel<S::BN>, dim3(1), kPlanThreads, 0, s, false, P, S::NQ * P.tp, static_cast<int>(g.max_items),
             ctas) != cudaSuccess)
    return GR_ERR_CUDA;
  if (launch(attention_kernel<S, kBf16>, dim3(ctas), S::kThreads, smem, s, !P.small, P, mq, mk, mv) != cudaSuccess)
    return GR_ERR_CUDA;
  return GR_OK;
}

}  // namespace grpa

extern "C" int32_t gr_paged_attention_workspace_size(const gr_paged_attn_desc* d, size_t* bytes) {
  using namespace grpa;
  if (!bytes) return GR_ERR_NULL;
  Geometry g;
  const int rc = geometry(d, g);
  if (rc != GR_OK) return rc;
  *bytes = layout(d, g).total;
  return GR_OK;
}

extern "C" int32_t gr_paged_attention(const gr_paged_attn_desc* d, const gr_paged_attn_io* io, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  gr::NvtxRange nvtx_range("gr_paged_attention");
  using namespace grpa;
  Geometry g;
  int rc = geometry(d, g);
  if (rc != GR_OK) return rc;
  if (!io) return GR_ERR_NULL;
  if ((io->beam_tail == nullptr) != (io->beam_steps == nullptr)) return GR_ERR_NULL;
  if (io->beam_steps != nullptr && !d->causal) return GR_ERR_BAD_DESC;
  if (d->num_seqs == 0 || d->num_tokens == 0) return GR_OK;
  if (!io->q || !io->cu_seqlens || !io->seq_lens || !io->out || !workspace) return GR_ERR_NULL;
  const bool keys = d->num_blocks > 0 && d->max_blocks > 0;
  if (keys && (!io->k_cache || !io->v_cache || !io->block_table)) return GR_ERR_NULL;
  const auto off16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  const auto off8 = [](int64_t a, int64_t n) { return n > 1 && (a % 8 != 0 || a <= 0 || a >= (1ll << 38)); };
  if (off16(io->q) || off16(io->out) || (keys && (off16(io->k_cache) || off16(io->v_cache))) ||
      off8(d->q_stride_tok, d->num_tokens) || off8(d->q_stride_head, d->num_heads) ||
      off8(d->out_stride_tok, d->num_tokens) || off8(d->out_stride_head, d->num_heads) ||
      off8(d->k_stride_block, d->num_blocks) || off8(d->k_stride_tok, d->block_size) ||
      off8(d->k_stride_head, d->num_kv_heads) || off8(d->v_stride_block, d->num_blocks) ||
      off8(d->v_stride_tok, d->block_size) || off8(d->v_stride_head, d->num_kv_heads))
    return GR_ERR_MISALIGNED;
  const Layout l = layout(d, g);
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return GR_ERR_MISALIGNED;
  if (workspace_bytes < l.total) return GR_ERR_WORKSPACE;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return GR_ERR_NO_DEVICE;
  {
    std::lock_guard<std::mutex> lock(g_mu);
    if (g_sms[dev] == 0 && cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      g_sms[dev] = 0;
      return GR_ERR_CUDA;
    }
    sms = g_sms[dev];
  }
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  Params P;
  P.table = io->block_table;
  P.cu = io->cu_seqlens;
  P.seq_lens = io->seq_lens;
  P.tail = io->beam_tail;
  P.steps = io->beam_steps;
  P.out = io->out;
  P.lse = io->lse;
  P.err = io->err;
  P.table_stride = d->table_stride;
  P.num_blocks = d->num_blocks;
  P.out_tok = d->out_stride_tok;
  P.out_head = d->out_stride_head;
  P.num_seqs = d->num_seqs;
  P.num_tokens = d->num_tokens;
  P.heads = d->num_heads;
  P.kv_heads = d->num_kv_heads;
  P.group = g.group;
  P.dim = d->head_dim;
  P.block_size = d->block_size;
  P.max_blocks = keys ? d->max_blocks : 0;
  P.causal = d->causal;
  P.tp = g.tp;
  P.box = g.box;
  // x / d = x * m >> (32 + s) for every x < 2^31, with s = ceil(log2 d) - 1 and m = ceil(2^(32 + s) / d) < 2^32:
  // x m = x 2^(32+s) / d + x e / d with e < d, and x e / d < 2^31 <= 2^(32+s) / d
  P.div_shift = 0;
  while ((2ll << P.div_shift) < d->block_size) ++P.div_shift;
  P.div_mul = static_cast<uint32_t>(((1ull << (32 + P.div_shift)) + d->block_size - 1) / d->block_size);
  P.out32 = (reinterpret_cast<uintptr_t>(io->out) & 31u) == 0 && d->head_dim % 16 == 0 &&
            (d->out_stride_tok % 16 == 0 || d->num_tokens == 1) && (d->out_stride_head % 16 == 0 || d->num_heads == 1);
  const char* stall = std::getenv("GR_TEST_STALL_COPIES");
  P.flags = stall && stall[0] == '1' ? 1 : 0;
  P.scale_log2 = d->scale * gr::kLog2e;
  P.run = reinterpret_cast<Run*>(ws + l.run);
  P.flag = reinterpret_cast<uint64_t*>(ws + l.flag);
  P.token = next_token();
  P.small = small_plan(d, g);
  P.part_lse = reinterpret_cast<float*>(ws + l.part_lse);
  P.part_o = reinterpret_cast<float4*>(ws + l.part_o);
  P.pre = reinterpret_cast<int64_t*>(ws + l.pre);
  P.item = reinterpret_cast<int2*>(ws + l.item);
  P.items = reinterpret_cast<int32_t*>(ws + l.items);
  const bool bf16 = d->dtype == GR_DTYPE_BF16;
  CUtensorMap mq, mk, mv;
  // a dimension of one entry takes any legal stride
  const auto bytes = [](int64_t stride, int64_t n) { return static_cast<cuuint64_t>(n > 1 ? stride * 2 : 16); };
  {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d->head_dim), static_cast<cuuint64_t>(d->num_heads),
                                static_cast<cuuint64_t>(d->num_tokens)};
    const cuuint64_t str[2] = {bytes(d->q_stride_head, d->num_heads), bytes(d->q_stride_tok, d->num_tokens)};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(g.group), static_cast<cuuint32_t>(g.tp)};
    if (!encode(&mq, bf16, 3, io->q, dims, str, box)) return GR_ERR_CUDA;
  }
  for (int i = 0; i < 2; ++i) {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d->head_dim), static_cast<cuuint64_t>(d->num_kv_heads),
                                static_cast<cuuint64_t>(d->block_size),
                                static_cast<cuuint64_t>(keys ? d->num_blocks : 1)};
    const cuuint64_t str[3] = {bytes(i ? d->v_stride_head : d->k_stride_head, d->num_kv_heads),
                               bytes(i ? d->v_stride_tok : d->k_stride_tok, d->block_size),
                               bytes(i ? d->v_stride_block : d->k_stride_block, keys ? d->num_blocks : 1)};
    const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(g.box), 1};
    // without keys no copy is in range: any readable address will do
    const void* base = keys ? (i ? io->v_cache : io->k_cache) : io->q;
    if (!encode(i ? &mv : &mk, bf16, 4, base, dims, str, box)) return GR_ERR_CUDA;
  }
  if (!keys) P.num_blocks = 1;   // the id behind the last block is 1: out of range
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto shape, int kind) {
    using S = decltype(shape);
    return bf16 ? run<S, true>(P, g, mq, mk, mv, dev, sms, kind, s) : run<S, false>(P, g, mq, mk, mv, dev, sms, kind, s);
  };
  if (g.dp == 64) return g.nq == 1 ? go(Shape<64, 1>{}, 0) : go(Shape<64, 2>{}, 1);
  if (g.dp == 128) return g.nq == 1 ? go(Shape<128, 1>{}, 2) : go(Shape<128, 2>{}, 3);
  return go(Shape<256, 1>{}, 4);
}
