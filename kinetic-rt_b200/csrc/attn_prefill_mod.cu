// Paged attention of prompt tokens with score modifications (bf16, GQA) on
// the tensor cores (tcgen05, accumulators in TMEM).
//
// Query row t of sequence s at position p, head h:
//   x_j = scale q . k_j;  x_j = c tanh(x_j / c);  x_j -= slope_h |p - j|
//   visible j: lo <= j < hi,  lo = max(0, kv_start[t], p - window + 1),
//                             hi = min(len_s, max(p + 1, prefix_s))
//   out = sum_j softmax(x)_j v_j,  lse = log sum_j exp(x_j);  nothing visible: 0 and -inf
//
// The unit of work (an item) is 256 rows of one KV head = two tiles of 128; a
// tile holds 128 / G query tokens x the G query heads of the KV head (rows
// token-major), so a K/V block that is fetched serves all of them.  A CTA per
// SM takes items from a queue, the heaviest of a sequence first.  Its warps:
//   * 0-3 and 4-7: softmax of tile 0 and tile 1, one thread per row (TMEM
//     lane), so maxima and sums need no exchange; 168 registers each, the
//     whole block of 64 scores stays in them;
//   * 8: TMA producer of K, which also finds the next item while the present
//     one is worked on; 11: producer of V.  Blocks of 64 tokens, 16 KB each, in
//     two rings of four stages; a block is four 16-token pages, two boxes each;
//   * 9 and 10: issue the UMMAs of tile 0 and tile 1: S = Q K^T (M = 128,
//     N = 64, both operands in shared memory) and O += P V (P from TMEM, V as
//     the MN-major operand).  Two warps, because the waits, descriptors and
//     commits of a step take longer than its 12 MMAs (one warp for both tiles:
//     2600 cycles a step, of which the tensor core worked half).
// Shared memory: Q 64 KB, rings 128 KB, output staging 32 KB.  TMEM, per tile:
// two S buffers of 64 columns and O of 128 (all 512 columns).  P (bf16, 32
// columns) overwrites its S.  Each tile has two blocks in flight: while the
// softmax works on block g, the tensor core has P V of block g - 1 and Q K^T of
// block g + 1 of the same tile to do, and those of the other tile.  With one
// buffer of 128 columns per tile the chain S -> weights -> P V -> next S
// bounded the kernel (4150 cycles for 128 keys and both tiles, where tensor
// core and special-function units need 2048 each).
//
// Few rows behind a long cache make fewer items than there are SMs; their keys
// are then split into pieces (of eight blocks at least), whose unnormalised
// sums a second kernel joins.  Measured, 8 tokens of 8 KV heads behind 65536:
// 726 us whole, 64 split; behind 8192: 100 and 25 to 28; behind 1024: 19 and 17.
// (Pieces of four blocks: 14 there, but a 512-token prompt takes 20 for 17.)
// The last items of a long causal prompt are split too where the others would
// end well before them.
//
// What bounds it: per 128 keys and pair of tiles the tensor core needs about
// 2560 cycles (2048 of arithmetic; at N = 64 Q K^T reads 6 KB of shared memory
// per 32 cycles of it), the special-function units 2048 for one ex2 a score.
// A step takes about 3500 without and 4500 with a cap: the softmax warps' issue
// slots (the cap's polynomial, maxima, packing) come on top of what the
// special-function units leave of them.  Measured at full clock: six chunks of
// 517 tokens behind 3700, 64 heads, 289 us = 982 TFLOP/s; 8 x 2048, 32 heads,
// causal, capped, 355 us = 775 TFLOP/s; 64 tokens alone, 9.9 us in a graph.
// Under the power cap of long runs 322 and 391 us.
// Steps that are spared:
//   * the reference that scores are taken against is the row's old maximum
//     unless it grew by more than 2^16 (weights then stay below that, and bf16
//     and the fp32 sum lose nothing by it); only then O and the sum are
//     rescaled, after the tile's last P V;
//   * under a distance bias blocks are taken from the last to the first: the
//     nearest keys then set the reference, where in ascending order it would
//     grow with every block (documents with a bias: 171 us, ascending 199);
//   * the cap is a polynomial of the score while scores are well below it, and
//     its value at the row's largest |score| serves as the reference.
//
// Statistics, sums and O are fp32; P is rounded to bf16 for P V (2^-8 of each
// weight at most, as V is).  Beside the split of its keys, a row's bits depend on
// its sequence alone: not on the next one's rows in its tile, unwritten cache
// slots or earlier contents of memory.
//
// Masked scores become -inf and weigh 0, but 0 * NaN or 0 * inf of a V row
// that only some of the CTA's rows may see would spoil the others.  So in
// blocks that are not visible to all live rows, V values that are not finite
// are set to 0 in shared memory before P V, and a CTA that found some adds
// them in its epilogue to the rows that do see them.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <cuda_runtime.h>

#include "../../include/krt.h"
#include "attn_mod.cuh"
#include "capi_internal.h"
#include "ptx.cuh"
#include "qkv_paged.cuh"

namespace krt {

constexpr int kApmRows = 128;    // rows of a tile (TMEM lanes)
constexpr int kApmBlock = 64;    // keys per block
constexpr int kApmPage = 16;     // tokens per TMA box
constexpr int kApmStages = 4;    // of K, and of V
constexpr int kApmSoftmaxWarps = 8;
constexpr int kApmMaxGroup = 16;  // query heads per KV head
constexpr int kApmThreads = 384;
constexpr uint32_t kApmTileBytes = 32768;  // Q tile: 128 rows x 128 dims bf16, two [128 x 128 B] halves
constexpr uint32_t kApmHalf = 16384;
constexpr uint32_t kApmKvBytes = 16384;    // K or V block: 64 tokens x 128 dims, two [64 x 128 B] halves
constexpr uint32_t kApmKvHalf = 8192;
constexpr uint32_t kApmOutBytes = 16384;   // 64 columns of a tile's output
constexpr float kApmLazy = 16.f;   // growth of a row's maximum (base 2) that is left unscaled
// A capped score of at most this (base 2) may serve as reference in the place of
// the row's maximum, which then lies at most twice as far below it: weights of
// 2^-100 and sums of them are normal floats.
constexpr float kApmBound = 50.f;
constexpr int kApmMaxPos = 1 << 30;
constexpr int kApmMinPiece = 8;   // key blocks of a piece at least, where an item is split
constexpr size_t kApmQueueAt = 256, kApmFlagsAt = 1024;  // in the workspace's header
constexpr int kApmMaxPieces = (kWsHeaderBytes - kApmFlagsAt) / 8;
constexpr size_t kApmPartBytes = (size_t)2 * kApmRows * kHeadDim * 4;  // a piece's O, both tiles
constexpr size_t kApmStatBytes = (size_t)2 * kApmRows * 8;             // its references and sums

struct ApmParams {
  __nv_bfloat16* out;
  float* lse;
  const __nv_bfloat16* pool;
  const int32_t* block_table;
  const int32_t* q_start;
  const int32_t* q_pos0;
  const int32_t* kv_start;
  const int32_t* prefix_lens;
  int* status;
  uint32_t* queue;           // [next piece, CTAs that are through], zero between launches
  int items, splits;         // items, and pieces of each, at most
  int piece;                 // key blocks of a piece at least
  float4* part_o;            // [piece][tile][column / 4][row]
  float2* part_ml;           // [piece][tile][row] reference and sum
  int32_t* part_flags;       // [piece][tile] V values that are not finite were taken out
  int num_tokens, num_seqs, bt_stride, bt_columns, num_blocks, tokens_per_block;
  int key_end;  // positions that a row of the block table holds: no key beyond them is visited
  int n_kv_heads, group, tile_tokens;  // tile_tokens = 128 / group
  uint32_t group_inv;                  // row / group = row * group_inv >> 16 for rows below 128
  int out_stride, lse_stride;
  ScoreMod mod;
};

// A piece of work: a pair of tiles of one sequence and KV head, and their keys
// or a part of those.  Filled in by the scheduling warp one ahead of the others.
struct ApmItem {
  int seq;                // -1: there is no more work
  int kvh;
  int t_first, q_len;     // the sequence's first row, and its rows
  int tok0, pos0;         // first token of the tiles; position of the sequence's first query
  int prefix;
  int first[2], end[2];   // key blocks of each tile, [first, end); both 0 without a live row
  int lo_all, hi_all;     // keys that some live row sees
  int lo_max, hi_min;     // keys that all live rows see
  int part;               // where the piece leaves its part of the result, -1: it is the whole item
};

struct ApmSmemTail {
  uint64_t full[2][kApmStages];   // K, V
  uint64_t empty[2][kApmStages];
  uint64_t item_full[2], item_empty[2];
  uint64_t q_full, q_empty;
  uint64_t s_full[2][2];  // per tile and buffer
  uint64_t p_full[2][2];
  uint64_t o_done[2];     // per tile: one phase per P V but an item's last
  uint64_t o_last[2];     // per tile: an item's last P V (two may be under way when the last P is reported)
  uint64_t drain[2];      // per tile: the MMAs issued before an abort
  ApmItem item[2];
  uint32_t tmem_base;
  int issued[3];          // blocks of K and of V, and pairs of Q tiles, requested
  int abort;
  int poison[2];          // per item: its number + 1 if a V value that is not finite was taken out of a
                          // partly visible block
  uint32_t bad[16];       // per block (ring): pages that could not be looked up
};

// (no room to round the base up: the kernel checks that it is 1024-byte aligned)
inline size_t apm_smem_bytes() {
  return (size_t)2 * kApmTileBytes + (size_t)2 * kApmStages * kApmKvBytes + 2 * kApmOutBytes + sizeof(ApmSmemTail);
}

__device__ __forceinline__ void apm_fail(const ApmParams& p, ApmSmemTail* tl, int code) {
  atomicOr(p.status, code);
  *reinterpret_cast<volatile int*>(&tl->abort) = 1;
}

// Exponent bits all ones in either bf16 half of w: a 1 in bit 15 or 31.
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }

// Pool slot of position j of the sequence, or -1.
__device__ __forceinline__ long long apm_slot(const ApmParams& p, const int32_t* table, int j) {
  const int col = j / p.tokens_per_block;
  if (col >= p.bt_columns) return -1;
  const int blk = table[col];
  if (blk < 0 || blk >= p.num_blocks) return -1;
  return (long long)blk * p.tokens_per_block + j % p.tokens_per_block;
}

// First position that the query at `pos` sees, apart from kv_start.
__device__ __forceinline__ int apm_lowest(const ApmParams& p, int pos) {
  return p.mod.window > 0 ? max(0, pos - p.mod.window + 1) : 0;
}

// End of the keys that the query at `pos` of a sequence of `len` tokens sees.
__device__ __forceinline__ int apm_highest(const ApmParams& p, int len, int prefix, int pos) {
  return min(min(len, p.key_end), max(pos + 1, prefix));
}

// Item number `index` (seq -1: there are fewer, or q_start decreases somewhere
// and they are more than num_tokens rows can give): sequences in order, the last
// (heaviest) tokens of each first, KV heads innermost.  By a whole warp, 128
// sequences at a time, so that their loads overlap.
__device__ __forceinline__ ApmItem apm_find(const ApmParams& p, int index, int lane) {
  const int tt = p.tile_tokens;
  const int kvh = index % p.n_kv_heads, target = index / p.n_kv_heads;
  int seq = -1, t_first = 0, q_len = 0, pos0 = 0, tok0 = 0, base = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < p.num_seqs && seq < 0 && index < p.items; s0 += 128) {
    int a[4], e[4], p0[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = s0 + 32 * k + lane;
      const bool in = s < p.num_seqs;
      a[k] = in ? p.q_start[s] : 0;
      e[k] = in ? p.q_start[s + 1] : 0;
      p0[k] = in ? p.q_pos0[s] : 0;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (s0 + 32 * k >= p.num_seqs) break;
      if (a[k] < 0 || e[k] > p.num_tokens || e[k] < a[k]) atomicOr(p.status, kStatusBadBlock);
      a[k] = max(a[k], 0);
      e[k] = min(e[k], p.num_tokens);
      const int n = e[k] > a[k] ? (e[k] - a[k] + 2 * tt - 1) / (2 * tt) : 0;
      int incl = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
      }
      const int excl = base + incl - n;
      const uint32_t hit = __ballot_sync(0xffffffffu, target >= excl && target < excl + n);
      if (hit != 0) {
        const int who = __ffs(hit) - 1;
        seq = s0 + 32 * k + who;
        t_first = __shfl_sync(0xffffffffu, a[k], who);
        q_len = __shfl_sync(0xffffffffu, e[k], who) - t_first;
        pos0 = __shfl_sync(0xffffffffu, p0[k], who);
        tok0 = (__shfl_sync(0xffffffffu, n, who) - 1 - (target - __shfl_sync(0xffffffffu, excl, who))) * 2 * tt;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  ApmItem it;
  it.seq = seq;
  it.kvh = kvh;
  it.t_first = t_first;
  it.q_len = q_len;
  it.tok0 = tok0;
  it.pos0 = pos0;
  it.prefix = p.prefix_lens && seq >= 0 ? p.prefix_lens[seq] : 0;
  it.lo_all = INT_MAX;
  it.hi_all = 0;
  it.lo_max = 0;
  it.hi_min = INT_MAX;
  const bool pos_ok = pos0 >= 0 && pos0 <= kApmMaxPos && q_len <= kApmMaxPos;
  if ((!pos_ok || pos0 + q_len > p.key_end) && lane == 0) atomicOr(p.status, kStatusBadBlock);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int lo_min = INT_MAX, hi_max = 0;  // over the tile's live rows
    const int from = tok0 + i * tt, to = min(from + tt, q_len) - 1;  // its tokens
    if (seq >= 0 && pos_ok && from <= to) {
      auto highest = [&](int pos) { return apm_highest(p, pos0 + q_len, it.prefix, pos); };
      if (p.kv_start == nullptr) {
        // bounds do not decrease from token to token; every row is live but for
        // those whose window lies beyond the block table
        const int lo = apm_lowest(p, pos0 + from), hi = highest(pos0 + to);
        if (lo < hi) {
          lo_min = lo;
          hi_max = hi;
          it.lo_max = max(it.lo_max, apm_lowest(p, pos0 + to));
          it.hi_min = min(it.hi_min, highest(pos0 + from));
        }
      } else {
        int lo_max = 0, hi_min = INT_MAX;
        for (int tok = from + lane; tok <= to; tok += 32) {
          const int lo = max(apm_lowest(p, pos0 + tok), p.kv_start[t_first + tok]), hi = highest(pos0 + tok);
          if (lo >= hi) continue;
          lo_min = min(lo_min, lo);
          lo_max = max(lo_max, lo);
          hi_min = min(hi_min, hi);
          hi_max = max(hi_max, hi);
        }
        lo_min = __reduce_min_sync(0xffffffffu, lo_min);
        hi_max = __reduce_max_sync(0xffffffffu, hi_max);
        it.lo_max = max(it.lo_max, (int)__reduce_max_sync(0xffffffffu, lo_max));
        it.hi_min = min(it.hi_min, (int)__reduce_min_sync(0xffffffffu, hi_min));
      }
    }
    it.first[i] = hi_max > 0 ? lo_min / kApmBlock : 0;
    it.end[i] = hi_max > 0 ? (hi_max + kApmBlock - 1) / kApmBlock : 0;
    it.lo_all = min(it.lo_all, lo_min);
    it.hi_all = max(it.hi_all, hi_max);
  }
  if (it.hi_all == 0) it.lo_all = 0;
  it.part = -1;
  return it;
}

// Key blocks per piece of the item, and how many pieces that makes.
__device__ __forceinline__ int apm_pieces(const ApmParams& p, const ApmItem& it, int* len) {
  const int blocks = (it.hi_all + kApmBlock - 1) / kApmBlock - it.lo_all / kApmBlock;
  *len = max(p.piece, (blocks + p.splits - 1) / p.splits);
  return max(1, (blocks + *len - 1) / *len);
}

// Cuts the item down to its piece z.
__device__ __forceinline__ void apm_cut(ApmItem& it, int z, int len, int part) {
  const int b0 = it.lo_all / kApmBlock + z * len, b1 = b0 + len;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    it.first[i] = max(it.first[i], b0);
    it.end[i] = min(it.end[i], b1);
    if (it.first[i] >= it.end[i]) it.first[i] = it.end[i] = 0;
  }
  it.lo_all = max(it.lo_all, b0 * kApmBlock);
  it.hi_all = (int)min((long long)it.hi_all, (long long)b1 * kApmBlock);
  it.part = part;
}

// Adds the V values that were taken out (dims d0 .. d1 - 1) to a row that sees them.
__device__ __forceinline__ void apm_add_back(const ApmParams& p, const ApmItem* at, int lo, int hi, __nv_bfloat16* out,
                                             int d0, int d1) {
#pragma unroll 1
  for (int j = lo; j < hi; ++j) {
    const int j0 = j / kApmBlock * kApmBlock;
    if (j0 >= at->lo_max && j0 + kApmBlock <= at->hi_min) {  // a block that was not cleaned
      j = j0 + kApmBlock - 1;
      continue;
    }
    const long long sl = apm_slot(p, p.block_table + (size_t)at->seq * p.bt_stride, j);
    if (sl < 0) continue;
    const __nv_bfloat16* v = p.pool + ((size_t)sl * 2 * p.n_kv_heads + p.n_kv_heads + at->kvh) * kHeadDim;
#pragma unroll 1
    for (int i = d0; i < d1; ++i) {
      const float f = __bfloat162float(v[i]);
      if (!isfinite(f)) out[i] = __float2bfloat16(__bfloat162float(out[i]) + f);
    }
  }
}

template <bool CAP, bool BIAS>
__global__ void __launch_bounds__(kApmThreads, 1)
    paged_attention_prefill_mod_kernel(const __grid_constant__ CUtensorMap tmap_q,
                                       const __grid_constant__ CUtensorMap tmap_kv,
                                       const __grid_constant__ ApmParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {  // swizzled tiles need it; the whole CTA
    if (threadIdx.x == 0) atomicOr(p.status, kStatusBadSplit);
    return;
  }
  uint8_t* q_smem = smem;
  uint8_t* k_smem = smem + 2 * kApmTileBytes;
  uint8_t* v_smem = k_smem + kApmStages * kApmKvBytes;
  uint8_t* out_smem = v_smem + kApmStages * kApmKvBytes;
  ApmSmemTail* tl = reinterpret_cast<ApmSmemTail*>(out_smem + 2 * kApmOutBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.group, tt = p.tile_tokens;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      for (int s = 0; s < kApmStages; ++s) {
        mbar_init(&tl->full[i][s], 1);
        mbar_init(&tl->empty[i][s], 2);  // both tiles' MMAs
      }
      for (int s = 0; s < 2; ++s) {
        mbar_init(&tl->s_full[i][s], 1);
        mbar_init(&tl->p_full[i][s], 4);
      }
      mbar_init(&tl->o_done[i], 1);
      mbar_init(&tl->o_last[i], 1);
      mbar_init(&tl->drain[i], 1);
      mbar_init(&tl->item_full[i], 1);
      mbar_init(&tl->item_empty[i], kApmSoftmaxWarps + 3);  // and V's producer, and both tiles' MMAs
      tl->poison[i] = 0;
    }
    mbar_init(&tl->q_full, 1);
    mbar_init(&tl->q_empty, 2);
    fence_mbar_init();
    tl->abort = 0;
    tl->issued[0] = tl->issued[1] = tl->issued[2] = 0;
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_kv);
  }
  if (warp == 9) {
    tmem_alloc(&tl->tmem_base, 512);
    tmem_relinquish();
  }
  pdl_wait();  // q, the pool and the lengths come from earlier kernels
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tl->tmem_base;
  volatile int* abort_flag = &tl->abort;
  // Item k lies in slot k & 1 while it is worked on.
  auto next_item = [&](int k) -> const ApmItem* {
    return mbar_wait_all(&tl->item_full[k & 1], (uint32_t)(k >> 1) & 1u, abort_flag) ? &tl->item[k & 1] : nullptr;
  };
  auto release_item = [&](int k) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&tl->item_empty[k & 1]);
  };

  if (warp == 8 || warp == 11) {
    // ------------------------------------------------ producers of K and of V
    // One lane issues all of a block's boxes, from values that the warp has in
    // common (boxes issued by several lanes take about 100 cycles each).  K's
    // producer also finds the work: when an item's last K is under way it takes
    // the next from the queue, so that nothing of this is waited for.
    const int kv = warp == 8 ? 0 : 1;
    const bool leader = elect_one();
    const uint64_t pol = make_l2_policy_evict_last();  // K and V are read again by other tiles
    const int outside = p.num_blocks * p.tokens_per_block;  // a box there reads zeros
    uint8_t* ring = kv ? v_smem : k_smem;
    int slot = 0, count = 0, q_count = 0;  // count: blocks requested so far
    uint32_t ph = 0;
    bool ok = true;
#pragma unroll 1
    for (int k = 0; ok; ++k) {
      ApmItem it;
      if (kv == 0) {
        uint32_t index = blockIdx.x;
        bool queued = k > 0;
#pragma unroll 1
        while (true) {
          if (queued) {
            if (lane == 0) index = gridDim.x + atomicAdd(p.queue, 1u);
            index = __shfl_sync(0xffffffffu, index, 0);
          }
          const int z = (int)(index % p.splits);
          it = apm_find(p, (int)(index / p.splits), lane);
          if (p.splits == 1 || it.seq < 0) break;
          int len;
          const int pieces = apm_pieces(p, it, &len);
          if (z < pieces) {
            if (pieces > 1) apm_cut(it, z, len, (int)index);
            break;
          }
          queued = true;  // the item has fewer pieces
        }
        if (k > 1 && !mbar_wait_all(&tl->item_empty[k & 1], (uint32_t)((k >> 1) - 1) & 1u, abort_flag)) {
          if (lane == 0) apm_fail(p, tl, kStatusTimeoutEmpty);
          break;
        }
        if (leader) {
          tl->item[k & 1] = it;
          mbar_arrive(&tl->item_full[k & 1]);
        }
        __syncwarp();
      } else {
        const ApmItem* at = next_item(k);
        if (at == nullptr) {
          if (lane == 0) apm_fail(p, tl, kStatusTimeoutFull);
          break;
        }
        it = *at;
        release_item(k);
      }
      if (it.seq < 0) {
        if (kv == 0 && leader) {
          // this CTA takes no more; the last one to say so leaves the queue empty for the next launch
          __threadfence();
          if (atomicAdd(p.queue + 1, 1u) + 1 == gridDim.x) {
            p.queue[0] = 0u;
            p.queue[1] = 0u;
          }
        }
        break;
      }
      const int g0 = it.lo_all / kApmBlock, g1 = (it.hi_all + kApmBlock - 1) / kApmBlock;
      const int32_t* table = p.block_table + (size_t)it.seq * p.bt_stride;
      // pool token of this lane's page of step o's block (lanes 0-3), -1 where the lookup failed
      auto look_up = [&](int o) {
        const int j = (BIAS ? g1 - 1 - o : g0 + o) * kApmBlock + (lane & 3) * kApmPage;
        int v = outside;
        if (o < g1 - g0 && j < it.hi_all && j + kApmPage > it.lo_all) v = (int)apm_slot(p, table, j);
        return v;
      };
      int pool_tok = look_up(0), next_tok = look_up(1);
      if (kv == 0 && g1 > g0) {
        if (q_count > 0 && !mbar_wait_all(&tl->q_empty, (uint32_t)(q_count - 1) & 1u, abort_flag)) {
          if (lane == 0) apm_fail(p, tl, kStatusTimeoutEmpty);
          break;
        }
        ++q_count;
        if (leader) {
          mbar_arrive_expect_tx(&tl->q_full, 4u * (uint32_t)(tt * G) * 128u);
#pragma unroll 1
          for (int i = 0; i < 4; ++i)
            tma_load_4d(q_smem + i * kApmHalf, &tmap_q, &tl->q_full, 0, it.kvh * G,
                        it.t_first + it.tok0 + (i >> 1) * tt, i & 1);
          tl->issued[2] = q_count;
        }
        __syncwarp();
      }
#pragma unroll 1
      for (int o = 0; o < g1 - g0; ++o) {
        const uint32_t bad = __ballot_sync(0xffffffffu, pool_tok < 0) & 15u;
        if (pool_tok < 0) pool_tok = outside;
        int page[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) page[c] = __shfl_sync(0xffffffffu, pool_tok, c);
        pool_tok = next_tok;
        next_tok = look_up(o + 2);  // two blocks ahead: the lookup is not waited for
        if (count >= kApmStages && !mbar_wait_all(&tl->empty[kv][slot], ph ^ 1u, abort_flag)) {
          if (lane == 0) apm_fail(p, tl, kStatusTimeoutEmpty);
          ok = false;
          break;
        }
        if (leader) {
          if (kv == 0) {
            *reinterpret_cast<volatile uint32_t*>(&tl->bad[count & 15]) = bad;
            if (bad != 0) atomicOr(p.status, kStatusBadBlock);
          }
          mbar_arrive_expect_tx(&tl->full[kv][slot], kApmKvBytes);
          uint8_t* dst = ring + (size_t)slot * kApmKvBytes;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tma_load_5d(dst + c * 2048, &tmap_kv, &tl->full[kv][slot], 0, page[c], 0, kv, it.kvh, pol);
            tma_load_5d(dst + c * 2048 + kApmKvHalf, &tmap_kv, &tl->full[kv][slot], 0, page[c], 1, kv, it.kvh, pol);
          }
          tl->issued[kv] = count + 1;
        }
        __syncwarp();
        ++count;
        if (++slot == kApmStages) {
          slot = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp > 8) {
    // ------------------------------------------------------------ UMMA issue
    // One warp per tile; the whole warp walks the loop, one lane issues.  Step
    // g: P V of block g, then Q K^T of block g + 2 into the buffer that this
    // frees.  MMAs of one thread run in the order of their issue.
    constexpr uint32_t kIdescQk = umma_idesc_bf16(128, 64);
    constexpr uint32_t kIdescPv = umma_idesc_bf16(128, 128) | kUmmaBMnMajor;
    const int i = warp - 9;
    const bool leader = elect_one();
    const uint32_t qd = umma_desc_lo(smem_u32(q_smem)) + i * (kApmTileBytes >> 4);
    const uint32_t kd = umma_desc_lo(smem_u32(k_smem));
    const uint32_t vd = umma_desc_lo_mn(smem_u32(v_smem), kApmKvHalf);
    const uint32_t s_col = tmem + i * 128, o_col = tmem + 256 + i * 128;
    int k_slot = 0, v_slot = 0, q_count = 0;
    uint32_t k_ph = 0, v_ph = 0;
    int done = 0;  // the tile's blocks of earlier items
    bool ok = true;
#pragma unroll 1
    for (int k = 0; ok; ++k) {
      const ApmItem* at = next_item(k);
      if (at == nullptr) {
        if (lane == 0) apm_fail(p, tl, kStatusTimeoutFull);
        ok = false;
        break;
      }
      const int seq = at->seq, g0 = at->lo_all / kApmBlock, g1 = (at->hi_all + kApmBlock - 1) / kApmBlock;
      const int steps = g1 - g0;
      // steps in which the tile takes part (one without a live row: in none)
      const bool any = at->end[i] > 0;
      const int t_begin = !any ? steps : BIAS ? g1 - at->end[i] : at->first[i] - g0;
      const int t_end = !any ? 0 : t_begin + at->end[i] - at->first[i];
      release_item(k);
      if (seq < 0) break;
      if (steps <= 0) continue;
      if (!mbar_wait_all(&tl->q_full, (uint32_t)q_count & 1u, abort_flag)) {
        if (lane == 0) apm_fail(p, tl, kStatusTimeoutFull);
        ok = false;
        break;
      }
      ++q_count;
#pragma unroll 1
      for (int g = -2; g < steps; ++g) {
        const int b = g - t_begin;             // the item's how-manieth block of the tile
        const uint32_t n = (uint32_t)(done + b);  // of all items; its buffer is n & 1
        const bool has_k = g + 2 < steps, has_v = g >= 0;
        if (has_k) ok = mbar_wait_all(&tl->full[0][k_slot], k_ph, abort_flag);
        if (has_v && ok) ok = mbar_wait_all(&tl->full[1][v_slot], v_ph, abort_flag);
        if (!ok) {
          if (lane == 0) apm_fail(p, tl, kStatusTimeoutFull);
          break;
        }
        if (g >= t_begin && g < t_end) {
          if (!mbar_wait_all(&tl->p_full[i][n & 1], (n >> 1) & 1u, abort_flag)) {
            if (lane == 0) apm_fail(p, tl, kStatusTimeoutAccum);
            ok = false;
            break;
          }
          tc_fence_after();
          // O += P V: 16 keys a step, 2048 bytes of V, 8 columns of P
          const uint32_t bd = vd + v_slot * (kApmKvBytes >> 4);
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_bf16_ts<kUmmaDescHiSw128>(o_col, s_col + (n & 1) * 64 + 8 * kk, bd + 128u * kk, kIdescPv,
                                             (b | kk) ? 1u : 0u);
            umma_commit(g + 1 < t_end ? &tl->o_done[i] : &tl->o_last[i]);
          }
          __syncwarp();
        }
        if (g + 2 >= t_begin && g + 2 < t_end) {
          tc_fence_after();
          // S = Q K^T: 16 dims a step, 32 bytes of each row
          const uint32_t bd = kd + k_slot * (kApmKvBytes >> 4);
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              umma_bf16_ss<kUmmaDescHiSw128>(s_col + (n & 1) * 64, qd + (kk >> 2) * (kApmHalf >> 4) + (kk & 3) * 2,
                                             bd + (kk >> 2) * (kApmKvHalf >> 4) + (kk & 3) * 2, kIdescQk, kk ? 1u : 0u);
            umma_commit(&tl->s_full[i][n & 1]);
          }
          __syncwarp();
        }
        if (leader) {
          if (has_v) umma_commit(&tl->empty[1][v_slot]);
          if (has_k) umma_commit(&tl->empty[0][k_slot]);
          if (g + 3 == steps) umma_commit(&tl->q_empty);  // the item's last Q K^T
        }
        __syncwarp();
        if (has_v && ++v_slot == kApmStages) {
          v_slot = 0;
          v_ph ^= 1u;
        }
        if (has_k && ++k_slot == kApmStages) {
          k_slot = 0;
          k_ph ^= 1u;
        }
      }
      done += t_end - (t_end == 0 ? 0 : t_begin);
    }
    if (!ok && leader) {  // what was issued reads shared memory and writes TMEM until it is done
      umma_commit(&tl->drain[i]);
      mbar_wait(&tl->drain[i], 0, nullptr);
    }
  } else {
    // --------------------------------------------------------------- softmax
    const int wg = warp >> 2;  // tile
    const int r = tid & 127;   // row of the tile
    const int row_tok = (int)(r * p.group_inv >> 16);  // its token
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + lanes + 256 + wg * 128;
    int done = 0, blocks = 0, last = 0, partial_pv = 0;  // of earlier items: the tile's blocks, the CTA's, o_last's and
                                                          // o_done's phases
    bool ok = true;
#pragma unroll 1
    for (int k = 0; ok; ++k) {
      const ApmItem* at = next_item(k);
      if (at == nullptr) {
        ok = false;
        break;
      }
      if (at->seq < 0) break;
      // ---- this row's bounds, and the warp's
      const int first = at->first[wg], n = at->end[wg] - first;  // the tile's key blocks
      int lo = 0, hi = INT_MAX;  // rows that are not live stay unmasked, their result is not used
      bool live = false;
      const int tok = at->tok0 + wg * tt + row_tok, pos = at->pos0 + tok;
      const bool valid = r < tt * G && tok < at->q_len;
      if (valid && n > 0) {
        const int l = max(apm_lowest(p, pos), p.kv_start ? p.kv_start[at->t_first + tok] : 0);
        const int h = apm_highest(p, at->pos0 + at->q_len, at->prefix, pos);
        live = l < h;
        if (live) {
          lo = l;
          hi = h;
        }
      }
      const int w_lo = __reduce_max_sync(0xffffffffu, live ? lo : 0);        // keys that all live rows of the
      const int w_hi = __reduce_min_sync(0xffffffffu, live ? hi : INT_MAX);  // warp see
      const int g0 = at->lo_all / kApmBlock, g1 = (at->hi_all + kApmBlock - 1) / kApmBlock;
      float m_ref = -INFINITY, l = 0.f;
      float slope2 = 0.f;
      if (BIAS && valid) slope2 = p.mod.slopes[at->kvh * G + r - row_tok * G] * 1.4426950408889634f;
#pragma unroll 1
      for (int b = 0; b < n; ++b) {
        const uint32_t nb = (uint32_t)(done + b);
        const uint32_t s_addr = tmem + lanes + wg * 128 + (nb & 1) * 64;
        if (!mbar_wait_all(&tl->s_full[wg][nb & 1], (nb >> 1) & 1u, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int g = BIAS ? first + n - 1 - b : first + b, j0 = g * kApmBlock;
        float x[64];
        tmem_ld32_nowait(s_addr, x);
        tmem_ld32_nowait(s_addr + 32, x + 32);
        const int m = blocks + (BIAS ? g1 - 1 - g : g - g0);  // of the CTA's blocks
        const uint32_t bad = *reinterpret_cast<volatile uint32_t*>(&tl->bad[m & 15]);
        const bool masked = j0 < w_lo || j0 + kApmBlock > w_hi || bad != 0;  // for some live row of the warp
        if (j0 < at->lo_max || j0 + kApmBlock > at->hi_min) {
          // not visible to all live rows of the CTA: V values that are not finite to zero
          if (!mbar_wait_warp(&tl->full[1][m % kApmStages], (uint32_t)(m / kApmStages) & 1u, abort_flag)) {
            ok = false;
            break;
          }
          uint4* v = reinterpret_cast<uint4*>(v_smem + (size_t)(m % kApmStages) * kApmKvBytes);
#pragma unroll 4
          for (int i = 0; i < 8; ++i) {
            uint4 q = v[i * 128 + r];
            if ((not_finite2(q.x) | not_finite2(q.y) | not_finite2(q.z) | not_finite2(q.w)) != 0) {
              // (slots that no row sees need not be added back: their scan would take 50
              // times the call itself where a fresh cache holds NaN)
              const int key = j0 + (((i * 128 + r) >> 3) & 63);
              if (key >= at->lo_all && key < at->hi_all) {
                *reinterpret_cast<volatile int*>(&tl->poison[k & 1]) = k + 1;
                __threadfence_block();
              }
              auto clean = [](uint32_t w) {
                const uint32_t f = not_finite2(w);
                return w & ((f & 0x8000u ? 0u : 0xFFFFu) | (f & 0x80000000u ? 0u : 0xFFFF0000u));
              };
              v[i * 128 + r] = make_uint4(clean(q.x), clean(q.y), clean(q.z), clean(q.w));
            }
          }
          // the tensor core sees the values written; P V starts when all four
          // warps have reported their P, so after all of the block is clean
          fence_proxy_async_smem();
        }
        tmem_wait_ld64(x);
        // ---- modifications (base 2).  `direct`: scores stay q . k, and the scale
        // or the cap's polynomial enters in the exponent
        bool direct = !CAP && !BIAS;
        float m_new = -INFINITY;
        f32x2 pc[5];  // the polynomial, kept in registers: as constants they slow the multiply-adds down
        if (CAP) {
#pragma unroll
          for (int c = 0; c < 5; ++c) {
            pc[c] = pair_of(p.mod.poly[c]);
            asm volatile("" : "+l"(pc[c]));
          }
          float a0 = 0.f, a1 = 0.f;
#pragma unroll
          for (int c = 0; c < 64; c += 4) {
            a0 = max3(a0, fabsf(x[c]), fabsf(x[c + 1]));
            a1 = max3(a1, fabsf(x[c + 2]), fabsf(x[c + 3]));
          }
          a0 = fmaxf(a0, a1);
          // The form is chosen for the warp, and none of its rows' bits may depend on
          // what lies beside the sequence: rows that are not live (the next
          // sequence's, or such as no load fills) have no vote, and in blocks with
          // invisible keys (unwritten cache slots) both forms give the same bits.
          const bool small = !__any_sync(0xffffffffu, live && !(a0 <= p.mod.poly_max));
          direct = !BIAS && small && !masked && p.mod.cap2 * 0.605f <= kApmBound;
          if (direct) {
            m_new = cap_at(a0, p.mod.poly);  // a reference no lower than the maximum
          } else if (small) {
#pragma unroll
            for (int c = 0; c < 64; c += 2) {
              const f32x2 v = pack2(x[c], x[c + 1]);
              unpack2(mul2(v, cap_poly(mul2(v, v), pc)), x[c], x[c + 1]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 64; ++c)
              x[c] = fabsf(x[c]) <= p.mod.poly_max ? cap_at(x[c], p.mod.poly)
                                                   : cap_score(x[c], p.mod.cap_in, p.mod.cap2);
          }
        }
        if (BIAS) {
          const float d0 = (float)(j0 - pos);
#pragma unroll
          for (int c = 0; c < 64; ++c) x[c] = fmaf(-slope2, fabsf(d0 + (float)c), CAP ? x[c] : x[c] * p.mod.mul);
        }
        if (masked) {
          // visible keys of the block as bits
          const int v0 = min(max(lo - j0, 0), 64), v1 = min(max(hi - j0, 0), 64);
          unsigned long long seen = v0 < v1 ? (~0ull >> (64 - (v1 - v0))) << v0 : 0ull;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if ((bad >> c) & 1u) seen &= ~(0xFFFFull << (16 * c));
          const uint32_t seen0 = (uint32_t)seen, seen1 = (uint32_t)(seen >> 32);
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            x[c] = (seen0 >> c) & 1u ? x[c] : -INFINITY;
            x[32 + c] = (seen1 >> c) & 1u ? x[32 + c] : -INFINITY;
          }
        }
        if (!(CAP && direct)) {
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 64; c += 4) {
            mx[0] = max3(mx[0], x[c], x[c + 1]);
            mx[1] = max3(mx[1], x[c + 2], x[c + 3]);
          }
          m_new = fmaxf(mx[0], mx[1]);
          if (direct) m_new *= p.mod.mul;
        }
        // ---- the row's reference
        const bool grow = m_new > m_ref + kApmLazy;  // also from -inf
        if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? ex2(m_ref - m_new) : 1.f;
          if (grow) m_ref = m_new;
          l *= f;
          if (b > 0) {
            // the previous block's P V may still run (the one before it is done: S
            // of this block was computed after it)
            if (!mbar_wait_warp(&tl->o_done[wg], (uint32_t)(partial_pv + b - 1) & 1u, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              float v[32];
              uint32_t w[32];
              tmem_ld32_nowait(o_addr + 32 * c, v);
              tmem_wait_ld32(v);
#pragma unroll
              for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i] * f);
              tmem_st32(o_addr + 32 * c, w);
            }
          }
        }
        // ---- weights: 2^(x - reference), packed to bf16 as they come
        const float neg = m_ref == -INFINITY ? 0.f : -m_ref;  // nothing seen yet: weights 0, NaN stays NaN
        const f32x2 neg2 = pack2(neg, neg);
        f32x2 sum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
        uint32_t pk[32];
        if (CAP && direct) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const f32x2 v = pack2(x[2 * c], x[2 * c + 1]);
            float e0, e1;
            unpack2(fma2(v, cap_poly(mul2(v, v), pc), neg2), e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            sum2[c & 1] = add2(sum2[c & 1], pack2(e0, e1));
            pk[c] = pack_bf16x2(e0, e1);
          }
        } else {
          const f32x2 mul_2 = pack2(p.mod.mul, p.mod.mul);
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            f32x2 y = pack2(x[2 * c], x[2 * c + 1]);
            y = (CAP || BIAS) ? add2(y, neg2) : fma2(y, mul_2, neg2);
            float e0, e1;
            unpack2(y, e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            sum2[c & 1] = add2(sum2[c & 1], pack2(e0, e1));
            pk[c] = pack_bf16x2(e0, e1);
          }
        }
        tmem_st32(s_addr, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tl->p_full[wg][nb & 1]);
        float s0, s1;
        unpack2(add2(sum2[0], sum2[1]), s0, s1);
        l += s0 + s1;
      }
      if (!ok) break;
      // ------------------------------------------------------------ the rows out
      if (n > 0) {
        if (!mbar_wait_all(&tl->o_last[wg], (uint32_t)last & 1u, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        ++last;
        partial_pv += n - 1;
      }
      if (at->part >= 0) {
        // a piece: the row's unnormalised sums for the kernel that joins them
        const size_t tile = (size_t)at->part * 2 + wg;
        if (valid) p.part_ml[tile * kApmRows + r] = live ? make_float2(m_ref, l) : make_float2(-INFINITY, 0.f);
        if (r == 0) p.part_flags[tile] = *reinterpret_cast<volatile int*>(&tl->poison[k & 1]) == k + 1;
        if (n > 0) {
          float4* dst = p.part_o + tile * (kHeadDim / 4) * kApmRows + r;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float o[32];
            tmem_ld32_nowait(o_addr + 32 * c, o);
            tmem_wait_ld32(o);
            if (valid) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                dst[(8 * c + i) * kApmRows] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
          }
        }
      } else {
        const int t = at->t_first + tok, head = at->kvh * G + r - row_tok * G;
        const float inv = !live || l == 0.f ? 0.f : 1.f / l;
        // Through shared memory, 64 columns at a time (16-byte pieces, 128-byte
        // swizzle), then whole rows: a row written by its thread alone would take
        // a memory transaction for every 16 bytes.
        uint8_t* stage = out_smem + wg * kApmOutBytes;
        const int rows = min(tt, at->q_len - at->tok0 - wg * tt) * G;  // rows of the tile that exist
        __nv_bfloat16* tile_out = p.out + (size_t)(at->t_first + at->tok0 + wg * tt) * p.out_stride +
                                  (size_t)at->kvh * G * kHeadDim + (lane & 7) * 8;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          float o[64];
          if (n > 0) {
            tmem_ld32_nowait(o_addr + 64 * c, o);
            tmem_ld32_nowait(o_addr + 64 * c + 32, o + 32);
          } else {
#pragma unroll
            for (int i = 0; i < 64; ++i) o[i] = 0.f;
          }
          tmem_wait_ld64(o);
          __syncwarp();  // the warp's rows of the first 64 columns are read
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = live ? pack_bf16x2(o[8 * i + 2 * e] * inv, o[8 * i + 2 * e + 1] * inv) : 0u;
            *reinterpret_cast<uint4*>(stage + r * 128 + ((i ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rr = (warp & 3) * 32 + 4 * i + (lane >> 3), tk = (int)(rr * p.group_inv >> 16);
            if (rr < rows)
              *reinterpret_cast<uint4*>(tile_out + (size_t)tk * p.out_stride + (rr - tk * G) * kHeadDim + 64 * c) =
                  *reinterpret_cast<const uint4*>(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
          }
        }
        // (O is read: the next item's first P, which its P V waits for, comes later)
        __syncwarp();  // (the row may have been written by other lanes)
        if (live && *reinterpret_cast<volatile int*>(&tl->poison[k & 1]) == k + 1) {
          apm_add_back(p, at, lo, hi, p.out + (size_t)t * p.out_stride + (size_t)head * kHeadDim, 0, kHeadDim);
        }
        if (valid && p.lse)
          p.lse[(size_t)t * p.lse_stride + head] =
              !live || l == 0.f ? -INFINITY : (m_ref == -INFINITY ? l : (m_ref + log2f(l)) * kLn2);
      }
      done += n;
      blocks += g1 - g0;
      release_item(k);
    }
    if (!ok && lane == 0) apm_fail(p, tl, kStatusTimeoutAccum);
  }
  tc_fence_before();
  __syncthreads();
  if (tl->abort && tid == 0) {
    // loads still in flight land (bounded waits) before the CTA's memory goes
    if (tl->issued[2] > 0) mbar_wait(&tl->q_full, (uint32_t)(tl->issued[2] - 1) & 1u, nullptr);
    for (int kv = 0; kv < 2; ++kv)
      for (int m = max(0, tl->issued[kv] - kApmStages); m < tl->issued[kv]; ++m)
        mbar_wait(&tl->full[kv][m % kApmStages], (uint32_t)(m / kApmStages) & 1u, nullptr);
  }
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of the items that were split.  A CTA takes 32 rows of a tile,
// a thread 16 dims of one row, so that a warp reads whole lines of the parts.
__global__ void __launch_bounds__(256) paged_attention_prefill_mod_join_kernel(const __grid_constant__ ApmParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = blockIdx.x >> 3, i = (blockIdx.x >> 2) & 1, r = (blockIdx.x & 3) * 32 + lane;
  pdl_wait();
  pdl_launch_dependents();
  const ApmItem it = apm_find(p, item, lane);
  if (it.seq < 0) return;
  int len;
  const int pieces = apm_pieces(p, it, &len);
  const int tok_in = (int)(r * p.group_inv >> 16), tok = it.tok0 + i * p.tile_tokens + tok_in;
  if (pieces == 1 || r >= p.tile_tokens * p.group || tok >= it.q_len) return;
  const size_t tile0 = (size_t)item * p.splits * 2 + i;  // of piece 0; the next piece's is 2 on
  const float2* ml = p.part_ml + tile0 * kApmRows + r;
  const float4* po = p.part_o + (tile0 * (kHeadDim / 4) + 4 * warp) * kApmRows + r;
  float M = -INFINITY, L = 0.f, acc[16];
  int poison = 0;
#pragma unroll 4
  for (int z = 0; z < pieces; ++z) {
    M = fmaxf(M, __ldcg(&ml[(size_t)z * 2 * kApmRows]).x);
    poison |= __ldcg(&p.part_flags[tile0 + 2 * z]);
  }
  const float mu = M == -INFINITY ? 0.f : M;  // nothing seen, or only NaN
#pragma unroll
  for (int d = 0; d < 16; ++d) acc[d] = 0.f;
#pragma unroll 4
  for (int z = 0; z < pieces; ++z) {
    const float2 w = __ldcg(&ml[(size_t)z * 2 * kApmRows]);
    float4 o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = __ldcg(&po[((size_t)z * 2 * (kHeadDim / 4) + c) * kApmRows]);
    if (w.x == -INFINITY && w.y == 0.f) continue;  // the row sees nothing of the piece; O may not be set
    const float f = ex2(w.x - mu);
    L += f * w.y;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      acc[4 * c] += f * o[c].x;
      acc[4 * c + 1] += f * o[c].y;
      acc[4 * c + 2] += f * o[c].z;
      acc[4 * c + 3] += f * o[c].w;
    }
  }
  const int t = it.t_first + tok, head = it.kvh * p.group + r - tok_in * p.group, pos = it.pos0 + tok;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint32_t w[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) w[d] = pack_bf16x2(acc[2 * d] * inv, acc[2 * d + 1] * inv);
  __nv_bfloat16* out = p.out + (size_t)t * p.out_stride + (size_t)head * kHeadDim;
  uint4* dst = reinterpret_cast<uint4*>(out + 16 * warp);
  dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
  dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  if (poison) {
    const int lo = max(apm_lowest(p, pos), p.kv_start ? p.kv_start[t] : 0);
    apm_add_back(p, &it, lo, apm_highest(p, it.pos0 + it.q_len, it.prefix, pos), out, 16 * warp, 16 * warp + 16);
  }
  if (p.lse && warp == 0)
    p.lse[(size_t)t * p.lse_stride + head] = L == 0.f ? -INFINITY : (M == -INFINITY ? L : (M + log2f(L)) * kLn2);
}

typedef void (*ApmKernel)(const CUtensorMap, const CUtensorMap, const ApmParams);
ApmKernel apm_kernel(bool cap, bool bias) {
  if (cap)
    return bias ? paged_attention_prefill_mod_kernel<true, true> : paged_attention_prefill_mod_kernel<true, false>;
  return bias ? paged_attention_prefill_mod_kernel<false, true> : paged_attention_prefill_mod_kernel<false, false>;
}

}  // namespace krt

using namespace krt;

namespace {

// Items (pairs of tiles of a KV head) of a call at most, however its tokens
// fall on the sequences.
long long apm_items(int num_tokens, int num_seqs, int n_heads, int n_kv_heads) {
  const int tile_tokens = kApmRows / (n_heads / n_kv_heads);
  return (num_tokens / (2 * tile_tokens) + (long long)num_seqs) * n_kv_heads;
}

int apm_max_pieces() { return std::min(3 * device_sm_count(), kApmMaxPieces); }

// Pieces that an item of so many key blocks is worth at most.
long long apm_worth(long long blocks) { return (blocks + kApmMinPiece - 1) / kApmMinPiece; }

long long apm_blocks(long long keys) { return (keys + kApmBlock - 1) / kApmBlock; }

}  // namespace

// ------------------------------------------------------------------ C ABI
extern "C" size_t krt_paged_attention_prefill_mod_workspace_size(int32_t num_tokens, int32_t num_seqs, int32_t n_heads,
                                                                 int32_t n_kv_heads, int32_t max_kv_len) {
  if (num_tokens <= 0 || num_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || max_kv_len <= 0 ||
      n_heads % n_kv_heads != 0 || n_heads / n_kv_heads > kApmMaxGroup)
    return 0;
  // status word, queue and flags; parts of items that are split
  const long long items = apm_items(num_tokens, num_seqs, n_heads, n_kv_heads);
  const long long worth = apm_worth(apm_blocks(max_kv_len));
  const long long most = apm_max_pieces();
  const size_t pieces = worth > 1 ? (size_t)std::min(most, std::min(items, most) * worth) : 0;
  return kModPartsAt + pieces * (kApmPartBytes + kApmStatBytes);
}

extern "C" int krt_paged_attention_prefill_mod(const krt_paged_prefill_attention_mod_args* a, void* stream) {
  const char* name = "krt_paged_attention_prefill_mod";
  if (!a) return set_error(KRT_ERR_INVALID, "%s: args is NULL", name);
  if (!a->q || !a->out || !a->kv_pool || !a->block_table || !a->q_start || !a->q_pos0 || !a->workspace)
    return set_error(KRT_ERR_INVALID, "%s: a required pointer is NULL", name);
  if (a->head_dim != kHeadDim) return set_error(KRT_ERR_UNSUPPORTED, "%s: head_dim must be 128", name);
  if (a->num_tokens <= 0 || a->num_seqs <= 0 || a->n_heads <= 0 || a->n_kv_heads <= 0 || a->max_kv_len <= 0)
    return set_error(KRT_ERR_INVALID, "%s: num_tokens, num_seqs, heads and max_kv_len must be positive", name);
  if (a->n_heads % a->n_kv_heads != 0 || a->n_heads / a->n_kv_heads > kApmMaxGroup || a->n_kv_heads > 65535)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: n_heads must be a multiple of n_kv_heads, at most 16 per KV head", name);
  if (a->tokens_per_block <= 0 || a->tokens_per_block % kApmPage != 0)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: tokens_per_block must be a multiple of 16", name);
  if (a->num_blocks <= 0 || a->block_table_stride <= 0)
    return set_error(KRT_ERR_INVALID, "%s: paged-cache geometry must be positive", name);
  const int columns = block_table_columns(a->block_table_columns, a->block_table_stride, a->num_seqs);
  if (columns < 0)
    return set_error(KRT_ERR_INVALID, "%s: block_table_columns must lie in 0 .. block_table_stride", name);
  if ((long long)a->num_blocks * a->tokens_per_block > INT_MAX - kApmPage)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: the pool may hold fewer than 2^31 - 16 tokens", name);
  if ((long long)columns * a->tokens_per_block < a->max_kv_len)
    return set_error(KRT_ERR_INVALID, "%s: the block table cannot hold max_kv_len tokens", name);
  if (a->q_stride < a->n_heads * kHeadDim || a->q_stride % 8 != 0 || a->out_stride < a->n_heads * kHeadDim ||
      a->out_stride % 8 != 0)
    return set_error(KRT_ERR_INVALID, "%s: q/out strides must cover the heads, multiples of 8", name);
  if (a->lse && a->lse_stride < a->n_heads)
    return set_error(KRT_ERR_INVALID, "%s: lse_stride must cover the heads", name);
  if (!(a->scale >= 0.f) || std::isinf(a->scale) || !(a->softcap >= 0.f) || std::isinf(a->softcap))
    return set_error(KRT_ERR_INVALID, "%s: scale and softcap must be finite and not negative", name);
  if (a->window < 0) return set_error(KRT_ERR_INVALID, "%s: window must not be negative", name);
  if ((reinterpret_cast<uintptr_t>(a->q) & 15) || (reinterpret_cast<uintptr_t>(a->out) & 15) ||
      (reinterpret_cast<uintptr_t>(a->kv_pool) & 15) || (reinterpret_cast<uintptr_t>(a->workspace) & 15))
    return set_error(KRT_ERR_INVALID, "%s: tensors must be 16-byte aligned", name);
  const size_t need = krt_paged_attention_prefill_mod_workspace_size(a->num_tokens, a->num_seqs, a->n_heads,
                                                                     a->n_kv_heads, a->max_kv_len);
  if (a->workspace_bytes < need)
    return set_error(KRT_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, a->workspace_bytes, need);
  ApmParams p;
  std::memset(&p, 0, sizeof(p));
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.lse = a->lse;
  p.pool = static_cast<const __nv_bfloat16*>(a->kv_pool);
  p.block_table = a->block_table;
  p.q_start = a->q_start;
  p.q_pos0 = a->q_pos0;
  p.kv_start = a->kv_start;
  p.prefix_lens = a->prefix_lens;
  p.status = static_cast<int*>(a->workspace);
  char* ws = static_cast<char*>(a->workspace);
  p.queue = reinterpret_cast<uint32_t*>(ws + kApmQueueAt);
  p.part_flags = reinterpret_cast<int32_t*>(ws + kApmFlagsAt);
  p.num_tokens = a->num_tokens;
  p.num_seqs = a->num_seqs;
  p.bt_stride = a->block_table_stride;
  p.bt_columns = columns;
  p.num_blocks = a->num_blocks;
  p.tokens_per_block = a->tokens_per_block;
  p.key_end = (int)std::min<long long>((long long)columns * a->tokens_per_block, INT_MAX - kApmBlock);
  p.n_kv_heads = a->n_kv_heads;
  p.group = a->n_heads / a->n_kv_heads;
  p.tile_tokens = kApmRows / p.group;
  p.group_inv = 65536u / p.group + 1;
  p.out_stride = a->out_stride;
  p.lse_stride = a->lse_stride;
  p.mod = make_score_mod(a->scale, a->softcap, a->alibi_slopes, a->window);
  const long long items = apm_items(a->num_tokens, a->num_seqs, a->n_heads, a->n_kv_heads), sms = device_sm_count();
  if (items > INT_MAX) return set_error(KRT_ERR_UNSUPPORTED, "%s: too many tokens or heads", name);
  // Few rows behind a long cache: items are split so that all SMs work.  Else
  // items that are longer than an SM's share of all by far are, so that none
  // ends late: the last rows of a long causal prompt (half a prompt's own keys
  // lie behind its average row; lengths are taken as equal).  4096 tokens of 8
  // heads on one KV head: 72 us whole, 57 split.
  long long longest = apm_blocks(a->max_kv_len), average = longest;
  if (a->window > 0)
    average = longest = std::min(longest, apm_blocks((long long)a->window + 2 * p.tile_tokens) + 1);
  else
    average = std::max(longest / 2, longest - apm_blocks(a->num_tokens / a->num_seqs) / 2);
  long long splits = std::min(sms / items, apm_worth(longest)), piece = kApmMinPiece;
  const long long share = (items * average + sms - 1) / sms;
  if (2 * items > sms && longest - share >= 20) {
    splits = std::min(apm_max_pieces() / items, (longest + share - 1) / share);
    piece = share;
  }
  p.items = (int)items;
  p.splits = (int)std::max(1ll, splits);
  p.piece = (int)piece;  // at least; `splits` of the item's real length otherwise
  p.part_ml = reinterpret_cast<float2*>(ws + kModPartsAt);
  p.part_o = reinterpret_cast<float4*>(ws + kModPartsAt + (size_t)items * p.splits * kApmStatBytes);
  CUtensorMap tmap_q, tmap_kv;
  int rc = make_tmap_bf16_5d_strided(&tmap_q, a->q, {64, (uint64_t)a->n_heads, (uint64_t)a->num_tokens, 2},
                                     {256, (uint64_t)a->q_stride * 2, 128},
                                     {64, (uint32_t)p.group, (uint32_t)p.tile_tokens, 1});
  if (rc) return rc;
  rc = make_tmap_pool_kv16(&tmap_kv, a->kv_pool, a->num_blocks, a->tokens_per_block, a->n_kv_heads, false);
  if (rc) return rc;
  ApmKernel kern = apm_kernel(a->softcap > 0.f, a->alibi_slopes != nullptr);
  const size_t smem = apm_smem_bytes();
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return cuda_error(e, name);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min(items * p.splits, sms), 1, 1);
  cfg.blockDim = dim3(kApmThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, tmap_q, tmap_kv, p);
  if (e == cudaSuccess && p.splits > 1) {
    cfg.gridDim = dim3((unsigned)items * 8, 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, paged_attention_prefill_mod_join_kernel, p);
  }
  if (e != cudaSuccess) return cuda_error(e, name);
  return clear_error();
}
