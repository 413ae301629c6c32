// Paged attention of prompt tokens with score modifications (bf16, GQA) on
// the tensor cores (tcgen05, accumulators in TMEM).
//
// Query row t of sequence s at position p, head h:
//   x_j = scale q . k_j;  x_j = c tanh(x_j / c);  x_j -= slope_h |p - j|
//   visible j: lo <= j < hi,  lo = max(0, kv_start[t], p - window + 1),
//                             hi = min(len_s, max(p + 1, prefix_s))
//   out = sum_j softmax(x)_j v_j,  lse = log sum_j exp(x_j);  nothing visible: 0 and -inf
//
// One CTA works on 256 rows = two tiles of 128 rows; a tile holds 128 / G
// query tokens x the G query heads of one KV head (rows token-major), so a
// K/V block that is fetched serves all of them.  Twenty warps:
//   * warps 0-7 and 8-15: softmax of tile 0 and tile 1.  Two threads share a
//     row (a TMEM lane): of a block's 128 keys the first takes 0-31 and 64-95,
//     the second the others;
//   * warp 16: TMA producer.  K and V blocks of 128 tokens alternate in a ring
//     of five 32 KB stages; a block is eight 16-token pages, two boxes each;
//   * warp 17: issues the UMMAs: S = Q K^T (M = N = 128, both operands in
//     shared memory) and O += P V (P from TMEM, V as the MN-major operand);
//   * warps 18 and 19 only complete the warpgroup that gives up registers.
// TMEM: S0, S1, O0, O1, 128 columns each (all 512).  P (bf16, 64 columns)
// overwrites its S.  Issue order QK0 QK1 | PV0 QK0' PV1 QK1' ...: while the
// softmax of one tile runs, the tensor core works for the other, and P V of
// the first 64 keys starts while the weights of the others are computed.
//
// What bounds it: per block and pair of tiles the tensor core needs 2048
// cycles, and so do the 2 x 128 x 128 ex2 of the special-function units (one a
// score, 16 a cycle); a tile's chain S -> weights -> P V -> next S must fit
// into the same time.  Hence no step that can be spared lies in the chain:
//   * the reference that scores are taken against is the row's old maximum
//     unless it grew by more than 2^8 (weights then stay below 256, and bf16
//     and the fp32 sum lose nothing by it).  The two threads of a row only
//     agree, by one barrier that ors their votes, that nothing grew; where it
//     did they exchange maxima and rescale O and the sum.  MMAs of the issuing
//     thread run in order, so a full S says that the tile's previous P V is
//     done and O may be rescaled;
//   * the cap is a polynomial of the score while scores are well below it, and
//     its value at the row's largest |score| serves as the reference;
//   * a quarter of the weights without a cap take 2^x by polynomial on the
//     multiply-add pipe.
//
// Statistics, sums and O are fp32; P is rounded to bf16 for P V (2^-9 of each
// weight, as V is).
//
// Masked scores become -inf and weigh 0, but 0 * NaN or 0 * inf of a V row
// that only some of the CTA's rows may see would spoil the others.  So in
// blocks that are not visible to all live rows, V values that are not finite
// are set to 0 in shared memory before P V, and a CTA that found some adds
// them in its epilogue to the rows that do see them.
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
constexpr int kApmBlock = 128;   // keys per block
constexpr int kApmPage = 16;     // tokens per TMA box
constexpr int kApmStages = 5;
constexpr int kApmSoftmaxWarps = 16;
constexpr int kApmThreads = 640;
constexpr uint32_t kApmTileBytes = 32768;  // 128 rows x 128 dims bf16, two [128 x 128 B] halves
constexpr uint32_t kApmHalf = 16384;
constexpr float kApmLazy = 8.f;   // growth of a row's maximum (base 2) that is left unscaled
constexpr float kApmBound = 50.f; // largest reference (base 2) that may lie above the row's maximum
constexpr int kApmMaxPos = 1 << 30;

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
  int num_tokens, num_seqs, bt_stride, num_blocks, tokens_per_block;
  int n_kv_heads, group, tile_tokens;  // tile_tokens = 128 / group
  int out_stride, lse_stride;
  ScoreMod mod;
};

struct ApmSmemTail {
  uint64_t full[kApmStages];
  uint64_t empty[kApmStages];
  uint64_t q_full;
  uint64_t s_full[2];
  uint64_t p_full[2][2];  // per tile: P of keys 0-63, of keys 64-127
  uint64_t o_full[2];
  uint64_t drain;      // the MMAs issued before an abort
  uint32_t tmem_base;
  int issued;          // K/V stages requested
  int abort;
  int poison;          // a V value that is not finite was taken out of a partly visible block
  // this CTA's work, read from here where it is needed: registers are short,
  // and a spilled one costs an L2 round trip (640 stacks do not fit in L1)
  int seq, tile;
  int t_first, q_len, tok0, pos0;  // first row and rows of the sequence, first token of the tiles, its position
  int lo_min, lo_max, hi_min, hi_max;  // over the CTA's live rows
  int scan[kApmThreads / 32];
  uint32_t bad[8];     // per block (ring): pages that could not be looked up
  float row_x[2][2][kApmRows];  // exchanged between the two threads of a row
};

// (no room to round the base up: the kernel checks that it is 1024-byte aligned)
inline size_t apm_smem_bytes() { return (size_t)(2 + kApmStages) * kApmTileBytes + sizeof(ApmSmemTail); }

__device__ __forceinline__ void apm_fail(const ApmParams& p, ApmSmemTail* tl, int code) {
  atomicOr(p.status, code);
  *reinterpret_cast<volatile int*>(&tl->abort) = 1;
}

// Register split after the prologue: 640 threads start with 96 registers each
// (61440); 512 x 104 + 128 x 64 = 61440.
constexpr int kApmRegsSoftmax = 104;
constexpr int kApmRegsOther = 64;
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Exponent bits all ones in either bf16 half of w: a 1 in bit 15 or 31.
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }

// 2^y of two values by polynomial: y = n + f, |f| <= 1/2 (n by adding 1.5 2^23,
// whose low mantissa bits then hold n), 2^f by the degree-4 polynomial with the
// smallest largest relative error (2.6e-6, fitted by reweighted least squares),
// n added to the exponent.  y is raised to -126: weights below 2^-126 of the
// reference come out as that, not 0, -inf included, so masked scores must not
// come here; NaN stays NaN.
__device__ __forceinline__ void ex2_poly2(f32x2 y, float& e0, float& e1) {
  float y0, y1, t0, t1;
  unpack2(y, y0, y1);
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y0) : "f"(y0), "f"(-126.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y1) : "f"(y1), "f"(-126.f));
  y = pack2(y0, y1);
  constexpr float kMagic = 12582912.f;
  const f32x2 t = add2(y, pack2(kMagic, kMagic));
  const f32x2 f = add2(y, mul2(add2(t, pack2(-kMagic, -kMagic)), pack2(-1.f, -1.f)));
  f32x2 q = fma2(pack2(0.009570102207362652f, 0.009570102207362652f), f, pack2(0.05591786280274391f, 0.05591786280274391f));
  q = fma2(q, f, pack2(0.240247443318367f, 0.240247443318367f));
  q = fma2(q, f, pack2(0.6931217908859253f, 0.6931217908859253f));
  q = fma2(q, f, pack2(0.9999992847442627f, 0.9999992847442627f));
  unpack2(q, e0, e1);
  unpack2(t, t0, t1);
  e0 = __uint_as_float(__float_as_uint(e0) + (__float_as_uint(t0) << 23));
  e1 = __uint_as_float(__float_as_uint(e1) + (__float_as_uint(t1) << 23));
}

// Pool slot of position j of the sequence, or -1.
__device__ __forceinline__ long long apm_slot(const ApmParams& p, const int32_t* table, int j) {
  const int col = j / p.tokens_per_block;
  if (col >= p.bt_stride) return -1;
  const int blk = table[col];
  if (blk < 0 || blk >= p.num_blocks) return -1;
  return (long long)blk * p.tokens_per_block + j % p.tokens_per_block;
}

template <bool CAP, bool BIAS>
__global__ void __launch_bounds__(kApmThreads, 1)
    paged_attention_prefill_mod_kernel(const __grid_constant__ CUtensorMap tmap_q,
                                       const __grid_constant__ CUtensorMap tmap_kv, const ApmParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {  // swizzled tiles need it; the whole CTA
    if (threadIdx.x == 0) atomicOr(p.status, kStatusBadSplit);
    return;
  }
  uint8_t* q_smem = smem;
  uint8_t* kv_smem = smem + 2 * kApmTileBytes;
  ApmSmemTail* tl = reinterpret_cast<ApmSmemTail*>(smem + (size_t)(2 + kApmStages) * kApmTileBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.group, tt = p.tile_tokens;

  if (tid == 0) {
    for (int s = 0; s < kApmStages; ++s) {
      mbar_init(&tl->full[s], 1);
      mbar_init(&tl->empty[s], 1);
    }
    mbar_init(&tl->q_full, 1);
    mbar_init(&tl->drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tl->s_full[i], 1);
      mbar_init(&tl->p_full[i][0], 8);
      mbar_init(&tl->p_full[i][1], 8);
      mbar_init(&tl->o_full[i], 1);
    }
    fence_mbar_init();
    tl->abort = 0;
    tl->issued = 0;
    tl->poison = 0;
    tl->seq = -1;
    tl->lo_min = INT_MAX;
    tl->lo_max = 0;
    tl->hi_min = INT_MAX;
    tl->hi_max = 0;
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_kv);
  }
  if (warp == 17) {
    tmem_alloc(&tl->tmem_base, 512);
    tmem_relinquish();
  }
  pdl_wait();  // q, the pool and the lengths come from earlier kernels
  pdl_launch_dependents();

  // ---- this CTA's (sequence, pair of tiles): sequences in order, the last
  // (heaviest) tokens of each first, KV heads innermost
  const int kvh = (int)(blockIdx.x % (unsigned)p.n_kv_heads);
  const int target = (int)(blockIdx.x / (unsigned)p.n_kv_heads);
  {
    int base = 0;
    for (int s0 = 0; s0 < p.num_seqs; s0 += kApmThreads) {
      const int s = s0 + tid;
      int n = 0;
      if (s < p.num_seqs) {
        int a = p.q_start[s], e = p.q_start[s + 1];
        if (a < 0 || e > p.num_tokens || e < a) {
          if (blockIdx.x == 0) atomicOr(p.status, kStatusBadBlock);
        }
        a = max(a, 0);
        e = min(e, p.num_tokens);
        if (e > a) n = (e - a + 2 * tt - 1) / (2 * tt);
      }
      int incl = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
      }
      __syncthreads();
      if (lane == 31) tl->scan[warp] = incl;
      __syncthreads();
      int before = base, total = base;
      for (int w = 0; w < kApmThreads / 32; ++w) {
        if (w < warp) before += tl->scan[w];
        total += tl->scan[w];
      }
      const int excl = before + incl - n;
      if (target >= excl && target < excl + n) {
        tl->seq = s;
        tl->tile = n - 1 - (target - excl);
      }
      base = total;
      if (target < base) break;  // uniform
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tl->tmem_base;
  const int seq = tl->seq;

  // ---- bounds of every row, and of the CTA
  int lo = 0, hi = INT_MAX;  // this row's; rows that are not live stay unmasked, their result is not used
  bool live = false, valid = false;
  int w_lo, w_hi;            // largest lo and smallest hi of the warp's live rows
  {
    int t_first = 0, q_len = 0, pos0 = 0, tok0 = 0;
    if (seq >= 0) {
      t_first = max(p.q_start[seq], 0);
      q_len = min(p.q_start[seq + 1], p.num_tokens) - t_first;
      pos0 = p.q_pos0[seq];
      tok0 = tl->tile * 2 * tt;
    }
    const bool pos_ok = pos0 >= 0 && pos0 <= kApmMaxPos && q_len <= kApmMaxPos;
    if (tid == 0) {
      tl->t_first = t_first;
      tl->q_len = q_len;
      tl->tok0 = tok0;
      tl->pos0 = pos0;
      if (!pos_ok) atomicOr(p.status, kStatusBadBlock);
    }
    const int r = tid & 127, tok = tok0 + (warp >> 3) * tt + r / G;
    valid = seq >= 0 && warp < kApmSoftmaxWarps && r < tt * G && tok < q_len;
    if (valid && pos_ok) {
      const int pos = pos0 + tok;
      int l = p.kv_start ? p.kv_start[t_first + tok] : 0;
      if (p.mod.window > 0) l = max(l, pos - p.mod.window + 1);
      l = max(l, 0);
      const int h = min(pos0 + q_len, max(pos + 1, p.prefix_lens ? p.prefix_lens[seq] : 0));
      live = l < h;
      if (live) {
        lo = l;
        hi = h;
      }
    }
    w_lo = __reduce_max_sync(0xffffffffu, live ? lo : 0);
    w_hi = __reduce_min_sync(0xffffffffu, live ? hi : INT_MAX);
    const int w_lo_min = __reduce_min_sync(0xffffffffu, live ? lo : INT_MAX);
    const int w_hi_max = __reduce_max_sync(0xffffffffu, live ? hi : 0);
    if (warp < kApmSoftmaxWarps && lane == 0) {
      atomicMax(&tl->lo_max, w_lo);
      atomicMin(&tl->hi_min, w_hi);
      atomicMin(&tl->lo_min, w_lo_min);
      atomicMax(&tl->hi_max, w_hi_max);
    }
  }
  __syncthreads();
  const int hi_max = tl->hi_max;
  const int blk0 = hi_max > 0 ? tl->lo_min / kApmBlock : 0;
  const int n = hi_max > 0 ? (hi_max + kApmBlock - 1) / kApmBlock - blk0 : 0;  // key blocks
  volatile int* abort_flag = &tl->abort;

  if (warp >= kApmSoftmaxWarps) {
    regs_dec<kApmRegsOther>();
    if (warp == 16 && n > 0) {
      // ------------------------------------------------------------ producer
      const uint64_t pol = make_l2_policy_evict_last();  // K and V are read again by other tiles
      if (lane == 0) {
        mbar_arrive_expect_tx(&tl->q_full, 4u * (uint32_t)(tt * G) * 128u);
#pragma unroll 1
        for (int i = 0; i < 2; ++i)
#pragma unroll 1
          for (int h = 0; h < 2; ++h)
            tma_load_4d(q_smem + i * kApmTileBytes + h * kApmHalf, &tmap_q, &tl->q_full, 0, kvh * G,
                        tl->t_first + tl->tok0 + i * tt, h);
      }
      const int outside = p.num_blocks * p.tokens_per_block;  // a box there reads zeros
      int s = 0;
      uint32_t ph = 0;
      bool alive = true;
      const int32_t* table = p.block_table + (size_t)seq * p.bt_stride;
      const int lo_min = tl->lo_min;
      int next_slot = -1;  // pool token of this lane's page in the next block
      auto look_up = [&](int b) {
        const int j = (blk0 + b) * kApmBlock + lane * kApmPage;
        int v = outside;
        bool bad = false;
        if (lane < 8 && j < hi_max && j + kApmPage > lo_min) {
          const long long sl = apm_slot(p, table, j);
          bad = sl < 0;
          if (!bad) v = (int)sl;
        }
        const uint32_t m = __ballot_sync(0xffffffffu, bad);
        if (m != 0 && lane == 0) atomicOr(p.status, kStatusBadBlock);
        next_slot = v;
        return m;
      };
#pragma unroll 1
      for (int b = 0; b < n && alive; ++b) {
        const uint32_t bad = look_up(b);
        if (lane == 0) *reinterpret_cast<volatile uint32_t*>(&tl->bad[b & 7]) = bad;
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          bool got = true;
          if (2 * b + kv >= kApmStages) got = mbar_wait_warp(&tl->empty[s], ph ^ 1u, abort_flag);
          if (!got) {
            if (lane == 0) apm_fail(p, tl, kStatusTimeoutEmpty);
            alive = false;
            break;
          }
          if (lane == 0) {
            mbar_arrive_expect_tx(&tl->full[s], kApmTileBytes);
            tl->issued = 2 * b + kv + 1;
          }
          __syncwarp();
          if (lane < 8) {
            uint8_t* dst = kv_smem + (size_t)s * kApmTileBytes + lane * 2048;
            tma_load_5d(dst, &tmap_kv, &tl->full[s], 0, next_slot, 0, kv, kvh, pol);
            tma_load_5d(dst + kApmHalf, &tmap_kv, &tl->full[s], 0, next_slot, 1, kv, kvh, pol);
          }
          if (++s == kApmStages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    } else if (warp == 17 && n > 0) {
      // ---------------------------------------------------------- UMMA issue
      // The whole warp walks the loop; one lane issues.
      constexpr uint32_t kIdescQk = umma_idesc_bf16(128, 128);
      constexpr uint32_t kIdescPv = umma_idesc_bf16(128, 128) | kUmmaBMnMajor;
      const bool leader = elect_one();
      const uint64_t qd = umma_desc_sw128(smem_u32(q_smem));
      const uint64_t kd = umma_desc_sw128(smem_u32(kv_smem));
      const uint64_t vd = umma_desc_sw128_mn(smem_u32(kv_smem), kApmHalf);
      auto qk = [&](int i, int slot) {  // S_i = Q_i K^T, 16 dims a step: 32 bytes of each row
        const uint64_t ad = qd + (uint64_t)(i * (kApmTileBytes >> 4));
        const uint64_t bd = kd + (uint64_t)(slot * (kApmTileBytes >> 4));
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint64_t d = (uint64_t)((kk >> 2) * (kApmHalf >> 4) + (kk & 3) * 2);
            umma_bf16_ss(tmem + i * 128, ad + d, bd + d, kIdescQk, kk ? 1u : 0u);
          }
          umma_commit(&tl->s_full[i]);
        }
      };
      auto pv = [&](int i, int slot, int h, uint32_t acc) {  // O_i += P_i V over keys 64 h .. 64 h + 63
        // 16 keys a step: 2048 bytes of V, 8 columns of P
        const uint64_t bd = vd + (uint64_t)(slot * (kApmTileBytes >> 4) + 512 * h);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_bf16_ts(tmem + 256 + i * 128, tmem + i * 128 + 32 * h + 8 * kk, bd + 128u * kk, kIdescPv,
                         kk ? 1u : acc);
        }
      };
      auto next = [](int& slot, uint32_t& ph) {
        if (++slot == kApmStages) {
          slot = 0;
          ph ^= 1u;
        }
      };
      int slot = 0;  // ring slot and phase of the load looked at
      uint32_t ph = 0;
      bool ok = mbar_wait_warp(&tl->q_full, 0, abort_flag) && mbar_wait_warp(&tl->full[0], 0, abort_flag);
      if (ok) {
        tc_fence_after();
        qk(0, 0);
        qk(1, 0);
        if (leader) umma_commit(&tl->empty[0]);
      } else if (lane == 0) {
        apm_fail(p, tl, kStatusTimeoutFull);
      }
#pragma unroll 1
      for (int b = 0; b < n && ok; ++b) {
        const bool more = b + 1 < n;
        next(slot, ph);
        const int v_slot = slot;
        ok = mbar_wait_warp(&tl->full[slot], ph, abort_flag);
        int k_slot = 0;
        if (more) {
          next(slot, ph);
          k_slot = slot;
          ok = ok && mbar_wait_warp(&tl->full[slot], ph, abort_flag);
        }
        if (!ok) {
          if (lane == 0) apm_fail(p, tl, kStatusTimeoutFull);
          break;
        }
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
#pragma unroll 1
          for (int h = 0; h < 2 && ok; ++h) {
            ok = mbar_wait_warp(&tl->p_full[i][h], (uint32_t)b & 1u, abort_flag);
            if (ok) {
              tc_fence_after();
              pv(i, v_slot, h, (uint32_t)(b | h) ? 1u : 0u);
            }
          }
          if (!ok) {
            if (lane == 0) apm_fail(p, tl, kStatusTimeoutAccum);
            break;
          }
          if (leader && i == 1) umma_commit(&tl->empty[v_slot]);
          if (more) {
            qk(i, k_slot);
            if (leader && i == 1) umma_commit(&tl->empty[k_slot]);
          } else if (leader) {
            umma_commit(&tl->o_full[i]);
          }
        }
      }
      if (!ok && leader) {  // what was issued reads shared memory and writes TMEM until it is done
        umma_commit(&tl->drain);
        mbar_wait(&tl->drain, 0, nullptr);
      }
    }
  } else {
    regs_inc<kApmRegsSoftmax>();
    // ------------------------------------------------------------- softmax
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int wg = warp >> 3;       // tile
    const int u = (warp >> 2) & 1;  // which of the row's two threads
    const int r = tid & 127;        // row of the tile
    const uint32_t s_addr = tmem + lanes + wg * 128;
    const uint32_t o_addr = tmem + lanes + 256 + wg * 128 + 64 * u;  // this thread's half of the row's output
    const int pair_bar = 1 + wg * 4 + (warp & 3);                    // barrier of the two warps of these rows
    float m_ref = -INFINITY, l = 0.f;
    float slope2 = 0.f;
    int pos = 0;
    if (BIAS) {
      pos = tl->pos0 + tl->tok0 + wg * tt + r / G;
      if (valid) slope2 = p.mod.slopes[kvh * G + r % G] * 1.4426950408889634f;
    }
    bool ok = true;
    for (int b = 0; b < n; ++b) {
      bool got = mbar_wait_warp(&tl->s_full[wg], (uint32_t)b & 1u, abort_flag);
      tc_fence_after();
      const int j0 = (blk0 + b) * kApmBlock;
      const uint32_t bad = *reinterpret_cast<volatile uint32_t*>(&tl->bad[b & 7]);
      const bool partial = j0 < tl->lo_max || j0 + kApmBlock > tl->hi_min;          // for some live row of the CTA
      const bool masked = j0 < w_lo || j0 + kApmBlock > w_hi || bad != 0;   // for some live row of the warp
      // this thread's keys: 32 u .. 32 u + 31 (chunk 0) and 64 + 32 u .. (chunk 1)
      float x[32], x1[32];
      tmem_ld32_nowait(s_addr + 64 + 32 * u, x1);
      tmem_ld32_nowait(s_addr + 32 * u, x);
      if (partial && got) {
        // partly visible block: V values that are not finite to zero
        const int m = 2 * b + 1;
        got = mbar_wait_warp(&tl->full[m % kApmStages], (uint32_t)(m / kApmStages) & 1u, abort_flag);
        uint4* v = reinterpret_cast<uint4*>(kv_smem + (size_t)(m % kApmStages) * kApmTileBytes);
#pragma unroll 4
        for (int i = 0; i < 8; ++i) {
          const int at = i * 256 + (tid & 255);
          uint4 q = v[at];
          if ((not_finite2(q.x) | not_finite2(q.y) | not_finite2(q.z) | not_finite2(q.w)) != 0) {
            *reinterpret_cast<volatile int*>(&tl->poison) = 1;
            __threadfence_block();
            auto clean = [](uint32_t w) {
              const uint32_t f = not_finite2(w);
              return w & ((f & 0x8000u ? 0u : 0xFFFFu) | (f & 0x80000000u ? 0u : 0xFFFF0000u));
            };
            v[at] = make_uint4(clean(q.x), clean(q.y), clean(q.z), clean(q.w));
          }
        }
        // the tensor core sees the values written; P V starts when all eight
        // warps have reported their P, so after all of the block is clean
        fence_proxy_async_smem();
      }
      tmem_wait_ld();
      // ---- modifications (base 2) of one chunk
      bool small = false;  // every |score| of the warp is within the cap's polynomial
      auto modify = [&](float* y, int h) {
        if (CAP) {
          if (small) {
            f32x2 pc[5];
#pragma unroll
            for (int k = 0; k < 5; ++k) pc[k] = pack2(p.mod.poly[k], p.mod.poly[k]);
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              const f32x2 v = pack2(y[c], y[c + 1]);
              unpack2(mul2(v, cap_poly(mul2(v, v), pc)), y[c], y[c + 1]);
            }
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) y[c] = cap_score(y[c], p.mod.cap_in, p.mod.cap2);
          }
        }
        const int k0 = j0 + 64 * h + 32 * u;  // position of the chunk's first key
        if (BIAS) {
          const float d0 = (float)(k0 - pos);
#pragma unroll
          for (int c = 0; c < 32; ++c) y[c] = fmaf(-slope2, fabsf(d0 + (float)c), CAP ? y[c] : y[c] * p.mod.mul);
        }
        if (masked) {
          const int v0 = lo - k0, v1 = hi - k0;
          const uint32_t pages = bad >> (4 * h + 2 * u);
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c < v0 || c >= v1 || ((pages >> (c / kApmPage)) & 1u)) y[c] = -INFINITY;
        }
      };
      auto max_of = [](const float* y) {
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          m0 = max3(m0, y[c], y[c + 1]);
          m1 = max3(m1, y[c + 2], y[c + 3]);
        }
        return fmaxf(m0, m1);
      };
      // `direct`: scores stay q . k, the cap's polynomial enters in the exponent
      bool direct = false;
      float m_new;
      if (CAP) {
        float a0 = 0.f, a1 = 0.f;
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          a0 = max3(a0, fabsf(x[c]), fabsf(x[c + 1]));
          a1 = max3(a1, fabsf(x1[c]), fabsf(x1[c + 1]));
        }
        a0 = fmaxf(a0, a1);
        small = !__any_sync(0xffffffffu, !(a0 <= p.mod.poly_max));
        direct = !BIAS && small && !masked && p.mod.cap2 * 0.605f <= kApmBound;
        const float w = a0 * a0;
        m_new = a0 * fmaf(fmaf(fmaf(fmaf(p.mod.poly[4], w, p.mod.poly[3]), w, p.mod.poly[2]), w, p.mod.poly[1]), w,
                          p.mod.poly[0]);
      }
      if (!direct) {
        modify(x1, 1);
        m_new = max_of(x1);
        modify(x, 0);
        m_new = fmaxf(m_new, max_of(x));
        if (!CAP && !BIAS) m_new *= p.mod.mul;
      }
      // ---- the row's reference.  The barrier also orders: both threads hold
      // their scores before either writes P over them
      if (named_bar_any(pair_bar, 64, !got || m_new > m_ref + kApmLazy)) {
        tl->row_x[wg][u][r] = m_new;
        if (named_bar_any(pair_bar, 64, !got)) {
          if (lane == 0) apm_fail(p, tl, kStatusTimeoutAccum);
          ok = false;
          break;
        }
        m_new = fmaxf(m_new, tl->row_x[wg][u ^ 1][r]);
        const bool grow = m_new > m_ref + kApmLazy;  // also from -inf
        const float f = grow ? ex2(m_ref - m_new) : 1.f;
        if (grow) m_ref = m_new;
        l *= f;
        if (b > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t v[16];
            tmem_ld16_nowait(o_addr + 16 * c, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
            tmem_st16(o_addr + 16 * c, v);
          }
        }
      }
      // ---- weights: 2^(x - reference), packed to bf16 as they come
      const float neg = m_ref == -INFINITY ? 0.f : -m_ref;  // nothing seen yet: weights 0, NaN stays NaN
      const f32x2 neg2 = pack2(neg, neg);
      f32x2 sum2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1) {  // P lies in the columns of keys 0-63: the second chunk's scores are still there
          tmem_ld32_nowait(s_addr + 64 + 32 * u, x);
          tmem_wait_ld();
          if (!direct && (CAP || BIAS || masked)) modify(x, 1);
        }
        uint32_t pk[16];
        if (CAP && direct) {
          f32x2 pc[5];
#pragma unroll
          for (int k = 0; k < 5; ++k) pc[k] = pack2(p.mod.poly[k], p.mod.poly[k]);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
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
          const bool poly = !CAP && !masked;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            f32x2 y = pack2(x[2 * c], x[2 * c + 1]);
            y = (CAP || BIAS) ? add2(y, neg2) : fma2(y, mul_2, neg2);
            float e0, e1;
            if (poly && (c & 3) == 3) {
              ex2_poly2(y, e0, e1);
            } else {
              unpack2(y, e0, e1);
              e0 = ex2(e0);
              e1 = ex2(e1);
            }
            sum2[c & 1] = add2(sum2[c & 1], pack2(e0, e1));
            pk[c] = pack_bf16x2(e0, e1);
          }
        }
        tmem_st16(s_addr + 32 * h + 16 * u, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tl->p_full[wg][h]);
      }
      float s0, s1;
      unpack2(add2(sum2[0], sum2[1]), s0, s1);
      l += s0 + s1;
    }
    // ------------------------------------------------------------ epilogue
    if (n > 0 && ok) ok = mbar_wait_warp(&tl->o_full[wg], 0, abort_flag);
    tc_fence_after();
    tl->row_x[wg][u][r] = l;
    if (named_bar_any(pair_bar, 64, !ok)) {
      if (lane == 0) apm_fail(p, tl, kStatusTimeoutAccum);
    } else {
      l += tl->row_x[wg][u ^ 1][r];
      const int seq = tl->seq, t_first = tl->t_first, q_len = tl->q_len, tok0 = tl->tok0 + wg * tt;
      const int kvh = (int)(blockIdx.x % (unsigned)p.n_kv_heads);
      const bool dead = !live || n == 0;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      // the row's output to shared memory (the Q tile is not read any more):
      // 16-byte pieces, 128-byte swizzle, then whole rows to global memory
      uint8_t* half_smem = q_smem + wg * kApmTileBytes + u * kApmHalf;
      const bool poison = n > 0 && *reinterpret_cast<volatile int*>(&tl->poison) != 0;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float v[32];
        if (n > 0) {
          tmem_ld32_nowait(o_addr + 32 * c, v);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = dead ? 0.f : v[i] * inv;
        if (poison && live) {
          for (int b = 0; b < n; ++b) {
            const int j0 = (blk0 + b) * kApmBlock;
            if (j0 >= tl->lo_max && j0 + kApmBlock <= tl->hi_min) continue;  // not cleaned
            for (int j = max(lo, j0); j < min(hi, j0 + kApmBlock); ++j) {
              const long long sl = apm_slot(p, p.block_table + (size_t)seq * p.bt_stride, j);
              if (sl < 0) continue;
              const __nv_bfloat16* vr =
                  p.pool + ((size_t)sl * 2 * p.n_kv_heads + p.n_kv_heads + kvh) * kHeadDim + 64 * u + 32 * c;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float f = __bfloat162float(vr[i]);
                if (!isfinite(f)) v[i] += f;
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 w = make_uint4(pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                                     pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
          *reinterpret_cast<uint4*>(half_smem + r * 128 + (((4 * c + i) ^ (r & 7)) << 4)) = w;
        }
      }
      if (valid && p.lse && u == 0)
        p.lse[(size_t)(t_first + tok0 + r / G) * p.lse_stride + kvh * G + r % G] =
            (dead || l == 0.f) ? -INFINITY : (m_ref == -INFINITY ? l : (m_ref + log2f(l)) * kLn2);
      __syncwarp();
      const int r0 = (warp & 3) * 32;
#pragma unroll 4
      for (int it = 0; it < 8; ++it) {
        const int rr = r0 + 4 * it + (lane >> 3), ch = lane & 7;
        const int tk = tok0 + rr / G;
        if (seq >= 0 && rr < tt * G && tk < q_len) {
          const uint4 w = *reinterpret_cast<const uint4*>(half_smem + rr * 128 + ((ch ^ (rr & 7)) << 4));
          *reinterpret_cast<uint4*>(p.out + (size_t)(t_first + tk) * p.out_stride +
                                    (size_t)(kvh * G + rr % G) * kHeadDim + 64 * u + ch * 8) = w;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tl->abort && tid == 0) {
    // loads still in flight land (bounded waits) before the CTA's memory goes
    mbar_wait(&tl->q_full, 0, nullptr);
    const int end = tl->issued;
    for (int m = end > kApmStages ? end - kApmStages : 0; m < end; ++m)
      mbar_wait(&tl->full[m % kApmStages], (uint32_t)(m / kApmStages) & 1u, nullptr);
  }
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

typedef void (*ApmKernel)(const CUtensorMap, const CUtensorMap, const ApmParams);
ApmKernel apm_kernel(bool cap, bool bias) {
  if (cap)
    return bias ? paged_attention_prefill_mod_kernel<true, true> : paged_attention_prefill_mod_kernel<true, false>;
  return bias ? paged_attention_prefill_mod_kernel<false, true> : paged_attention_prefill_mod_kernel<false, false>;
}

}  // namespace krt

using namespace krt;

// ------------------------------------------------------------------ C ABI
extern "C" size_t krt_paged_attention_prefill_mod_workspace_size(int32_t num_tokens, int32_t num_seqs, int32_t n_heads,
                                                                 int32_t n_kv_heads, int32_t max_kv_len) {
  if (num_tokens <= 0 || num_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 ||
      max_kv_len <= 0)
    return 0;
  return kWsHeaderBytes;
}

extern "C" int krt_paged_attention_prefill_mod(const krt_paged_prefill_attention_mod_args* a, void* stream) {
  const char* name = "krt_paged_attention_prefill_mod";
  if (!a) return set_error(KRT_ERR_INVALID, "%s: args is NULL", name);
  if (!a->q || !a->out || !a->kv_pool || !a->block_table || !a->q_start || !a->q_pos0 || !a->workspace)
    return set_error(KRT_ERR_INVALID, "%s: a required pointer is NULL", name);
  if (a->head_dim != kHeadDim) return set_error(KRT_ERR_UNSUPPORTED, "%s: head_dim must be 128", name);
  if (a->num_tokens <= 0 || a->num_seqs <= 0 || a->n_heads <= 0 || a->n_kv_heads <= 0 || a->max_kv_len <= 0)
    return set_error(KRT_ERR_INVALID, "%s: num_tokens, num_seqs, heads and max_kv_len must be positive", name);
  if (a->n_heads % a->n_kv_heads != 0 || a->n_heads / a->n_kv_heads > 16)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: n_heads must be a multiple of n_kv_heads, at most 16 per KV head", name);
  if (a->tokens_per_block <= 0 || a->tokens_per_block % kApmPage != 0)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: tokens_per_block must be a multiple of 16", name);
  if (a->num_blocks <= 0 || a->block_table_stride <= 0)
    return set_error(KRT_ERR_INVALID, "%s: paged-cache geometry must be positive", name);
  if ((long long)a->num_blocks * a->tokens_per_block > INT_MAX - kApmPage)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: the pool may hold fewer than 2^31 - 16 tokens", name);
  if ((long long)a->block_table_stride * a->tokens_per_block < a->max_kv_len)
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
  p.num_tokens = a->num_tokens;
  p.num_seqs = a->num_seqs;
  p.bt_stride = a->block_table_stride;
  p.num_blocks = a->num_blocks;
  p.tokens_per_block = a->tokens_per_block;
  p.n_kv_heads = a->n_kv_heads;
  p.group = a->n_heads / a->n_kv_heads;
  p.tile_tokens = kApmRows / p.group;
  p.out_stride = a->out_stride;
  p.lse_stride = a->lse_stride;
  p.mod = make_score_mod(a->scale, a->softcap, a->alibi_slopes, a->window);
  // at most this many pairs of tiles over all sequences, however the tokens fall on them
  const long long tiles = a->num_tokens / (2 * p.tile_tokens) + (long long)a->num_seqs;
  if (tiles * a->n_kv_heads > INT_MAX) return set_error(KRT_ERR_UNSUPPORTED, "%s: too many tokens or heads", name);
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
  cfg.gridDim = dim3((unsigned)(tiles * a->n_kv_heads), 1, 1);
  cfg.blockDim = dim3(kApmThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, tmap_q, tmap_kv, p);
  if (e != cudaSuccess) return cuda_error(e, name);
  return clear_error();
}
