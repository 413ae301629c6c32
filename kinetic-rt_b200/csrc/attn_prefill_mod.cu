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
// K/V block that is fetched serves all of them.  Twelve warps:
//   * warps 0-3 and 4-7: softmax of tile 0 and tile 1, one thread per row
//     (TMEM lane); the thread holds its 128 scores in registers, so maxima and
//     sums need no shuffles;
//   * warp 8: TMA producer.  K and V blocks of 128 tokens alternate in a ring
//     of five 32 KB stages; a block is eight 16-token pages, two boxes each;
//   * warp 9: issues the UMMAs: S = Q K^T (M = N = 128, both operands in
//     shared memory) and O += P V (P from TMEM, V as the MN-major operand);
//   * warps 10 and 11 only complete the third warpgroup, which gives its
//     registers to the other two.
// TMEM: S0, S1, O0, O1, 128 columns each (all 512).  P (bf16, 64 columns)
// overwrites its S.  Issue order QK0 QK1 | PV0 QK0' PV1 QK1' ...: while the
// softmax of one tile runs, the tensor core works for the other.  MMAs of the
// issuing thread run in order, so a full S also says that the tile's previous
// P V is done, and the row's O may then be rescaled by the softmax thread.
// That happens only where the row's maximum grew by more than 2^8: until then
// the old one stays the reference, weights stay below 256, and bf16 and the
// fp32 sum lose nothing by it.
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
constexpr int kApmThreads = 384;
constexpr uint32_t kApmTileBytes = 32768;  // 128 rows x 128 dims bf16, two [128 x 128 B] halves
constexpr uint32_t kApmHalf = 16384;
constexpr float kApmLazy = 8.f;  // growth of a row's maximum (base 2) that is left unscaled
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
  uint64_t p_full[2];
  uint64_t o_full[2];
  uint64_t drain;      // the MMAs issued before an abort
  uint32_t tmem_base;
  int issued;          // K/V stages requested
  int abort;
  int poison;          // a V value that is not finite was taken out of a partly visible block
  int seq, tile;       // this CTA's work
  int lo_min, lo_max, hi_min, hi_max;  // over the CTA's live rows
  int scan[kApmThreads / 32];
  uint32_t bad[8];     // per block (ring): pages that could not be looked up
};

inline size_t apm_smem_bytes() {
  return 1024 + (size_t)(2 + kApmStages) * kApmTileBytes + sizeof(ApmSmemTail);
}

__device__ __forceinline__ void apm_fail(const ApmParams& p, ApmSmemTail* tl, int code) {
  atomicOr(p.status, code);
  *reinterpret_cast<volatile int*>(&tl->abort) = 1;
}

// Register split after the prologue: 384 threads start with 168 registers
// each (64512); 2 x 128 x 208 + 128 x 80 = 63488.
constexpr int kApmRegsSoftmax = 208;
constexpr int kApmRegsOther = 80;
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
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
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
      mbar_init(&tl->p_full[i], 4);
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
  if (warp == 9) {
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
  int t_first = 0, q_len = 0, pos0 = 0, tok0 = 0;
  const int32_t* table = nullptr;
  if (seq >= 0) {
    t_first = max(p.q_start[seq], 0);
    q_len = min(p.q_start[seq + 1], p.num_tokens) - t_first;
    pos0 = p.q_pos0[seq];
    tok0 = tl->tile * 2 * tt;
    table = p.block_table + (size_t)seq * p.bt_stride;
  }
  const bool pos_ok = pos0 >= 0 && pos0 <= kApmMaxPos && q_len <= kApmMaxPos;
  if (!pos_ok && tid == 0) atomicOr(p.status, kStatusBadBlock);
  const int wg = warp >> 2;            // softmax: tile of this warp
  const int r = tid & 127;             // row of the tile
  const int tok = tok0 + wg * tt + r / G;
  const int head = kvh * G + r % G;
  const bool valid = seq >= 0 && warp < 8 && r < tt * G && tok < q_len;
  const int pos = pos0 + tok;
  int lo = 0, hi = INT_MAX;
  bool live = false;
  if (valid && pos_ok) {
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
  // rows that are not live stay unmasked: they compute something finite or
  // not, and their result is not used
  const int w_lo = __reduce_max_sync(0xffffffffu, live ? lo : 0);
  const int w_hi = __reduce_min_sync(0xffffffffu, live ? hi : INT_MAX);
  const int w_lo_min = __reduce_min_sync(0xffffffffu, live ? lo : INT_MAX);
  const int w_hi_max = __reduce_max_sync(0xffffffffu, live ? hi : 0);
  if (warp < 8 && lane == 0) {
    atomicMax(&tl->lo_max, w_lo);
    atomicMin(&tl->hi_min, w_hi);
    atomicMin(&tl->lo_min, w_lo_min);
    atomicMax(&tl->hi_max, w_hi_max);
  }
  __syncthreads();
  const int lo_min = tl->lo_min, lo_max = tl->lo_max, hi_min = tl->hi_min, hi_max = tl->hi_max;
  const int blk0 = hi_max > 0 ? lo_min / kApmBlock : 0;
  const int n = hi_max > 0 ? (hi_max + kApmBlock - 1) / kApmBlock - blk0 : 0;  // key blocks
  volatile int* abort_flag = &tl->abort;

  if (warp >= 8) {
    regs_dec<kApmRegsOther>();
    if (warp == 8 && n > 0) {
      // ------------------------------------------------------------ producer
      const uint64_t pol = make_l2_policy_evict_last();  // K and V are read again by other tiles
      if (lane == 0) {
        mbar_arrive_expect_tx(&tl->q_full, 4u * (uint32_t)(tt * G) * 128u);
        for (int i = 0; i < 2; ++i)
          for (int h = 0; h < 2; ++h)
            tma_load_4d(q_smem + i * kApmTileBytes + h * kApmHalf, &tmap_q, &tl->q_full, 0, kvh * G,
                        t_first + tok0 + i * tt, h);
      }
      const int outside = p.num_blocks * p.tokens_per_block;  // a box there reads zeros
      int s = 0;
      uint32_t ph = 0;
      bool alive = true;
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
      for (int b = 0; b < n && alive; ++b) {
        const uint32_t bad = look_up(b);
        if (lane == 0) *reinterpret_cast<volatile uint32_t*>(&tl->bad[b & 7]) = bad;
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
    } else if (warp == 9 && n > 0) {
      // ---------------------------------------------------------- UMMA issue
      if (lane == 0) {
        constexpr uint32_t kIdescQk = umma_idesc_bf16(128, 128);
        constexpr uint32_t kIdescPv = umma_idesc_bf16(128, 128) | kUmmaBMnMajor;
        auto slot_of = [](int m) { return m % kApmStages; };
        auto phase_of = [](int m) { return (uint32_t)(m / kApmStages) & 1u; };
        auto qk = [&](int i, int b) {  // S_i = Q_i K_b^T
          const uint32_t qa = smem_u32(q_smem + i * kApmTileBytes);
          const uint32_t ka = smem_u32(kv_smem + (size_t)slot_of(2 * b) * kApmTileBytes);
  #pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint64_t ad = umma_desc_sw128(qa + h * kApmHalf), bd = umma_desc_sw128(ka + h * kApmHalf);
  #pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_bf16(tmem + i * 128, ad + 2u * kk, bd + 2u * kk, kIdescQk, (h | kk) ? 1u : 0u);
          }
          umma_commit(&tl->s_full[i]);
        };
        auto pv = [&](int i, int b) {  // O_i += P_i V_b
          const uint32_t va = smem_u32(kv_smem + (size_t)slot_of(2 * b + 1) * kApmTileBytes);
          const uint64_t vd = umma_desc_sw128_mn(va, kApmHalf);
  #pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // 16 keys a step: 2048 bytes of V, 8 columns of P
            umma_bf16_ts(tmem + 256 + i * 128, tmem + i * 128 + 8 * kk, vd + 128u * kk, kIdescPv, (b | kk) ? 1u : 0u);
        };
        bool ok = mbar_wait(&tl->q_full, 0, abort_flag) && mbar_wait(&tl->full[0], 0, abort_flag);
        if (!ok) apm_fail(p, tl, kStatusTimeoutFull);
        if (ok) {
          tc_fence_after();
          qk(0, 0);
          qk(1, 0);
          umma_commit(&tl->empty[0]);
        }
        for (int b = 0; b < n && ok; ++b) {
          const bool more = b + 1 < n;
          ok = mbar_wait(&tl->full[slot_of(2 * b + 1)], phase_of(2 * b + 1), abort_flag) &&
               (!more || mbar_wait(&tl->full[slot_of(2 * b + 2)], phase_of(2 * b + 2), abort_flag));
          if (!ok) {
            apm_fail(p, tl, kStatusTimeoutFull);
            break;
          }
          for (int i = 0; i < 2; ++i) {
            if (!mbar_wait(&tl->p_full[i], (uint32_t)b & 1u, abort_flag)) {
              apm_fail(p, tl, kStatusTimeoutAccum);
              ok = false;
              break;
            }
            tc_fence_after();
            pv(i, b);
            if (i == 1) umma_commit(&tl->empty[slot_of(2 * b + 1)]);
            if (!more) umma_commit(&tl->o_full[i]);
            if (more) {
              qk(i, b + 1);
              if (i == 1) umma_commit(&tl->empty[slot_of(2 * b + 2)]);
            }
          }
        }
        if (!ok) {  // what was issued reads shared memory and writes TMEM until it is done
          umma_commit(&tl->drain);
          mbar_wait(&tl->drain, 0, nullptr);
        }
      }
    }
  } else {
    regs_inc<kApmRegsSoftmax>();
    // ------------------------------------------------------------- softmax
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + wg * 128;
    const uint32_t o_addr = tmem + lanes + 256 + wg * 128;
    float m_ref = -INFINITY, l = 0.f;
    float slope2 = 0.f;
    if (BIAS && valid) slope2 = p.mod.slopes[head] * 1.4426950408889634f;
    bool ok = true;
    for (int b = 0; b < n; ++b) {
      if (!mbar_wait_warp(&tl->s_full[wg], (uint32_t)b & 1u, abort_flag)) {
        if (lane == 0) apm_fail(p, tl, kStatusTimeoutAccum);
        ok = false;
        break;
      }
      tc_fence_after();
      const int j0 = (blk0 + b) * kApmBlock;
      const uint32_t bad = *reinterpret_cast<volatile uint32_t*>(&tl->bad[b & 7]);
      float x[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32_nowait(s_addr + 32 * c, x + 32 * c);
      tmem_wait_ld();
      // ---- modifications (base 2).  Without any, x stays q . k and the
      // scale enters the exponent's multiply-add.
      if (CAP) {
#pragma unroll
        for (int c = 0; c < 128; ++c) x[c] = cap_score(x[c], p.mod.cap_in, p.mod.cap2);
      }
      if (BIAS) {
        const float d0 = (float)(j0 - pos);  // exact: both below 2^24 in any cache that fits, else rounded once
#pragma unroll
        for (int c = 0; c < 128; ++c)
          x[c] = CAP ? fmaf(-slope2, fabsf(d0 + (float)c), x[c])
                     : fmaf(-slope2, fabsf(d0 + (float)c), x[c] * p.mod.mul);
      }
      if (j0 < w_lo || j0 + kApmBlock > w_hi || bad != 0) {
        const int v0 = lo - j0, v1 = hi - j0;
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (c < v0 || c >= v1 || ((bad >> (c / kApmPage)) & 1u)) x[c] = -INFINITY;
      }
      // ---- row maximum, reference, weights
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 128; ++c) mx[c & 3] = fmaxf(mx[c & 3], x[c]);
      float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      const float mul = (CAP || BIAS) ? 1.f : p.mod.mul;
      m_new *= mul;
      const bool grow = m_new > m_ref + kApmLazy;  // also from -inf
      if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? ex2(m_ref - m_new) : 1.f;
        if (grow) m_ref = m_new;
        l *= f;
        if (b > 0) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v[32];
            tmem_ld32_nowait(o_addr + 32 * c, v);
            tmem_wait_ld();
            uint32_t u[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(v[i] * f);
            tmem_st32(o_addr + 32 * c, u);
          }
        }
      }
      const float neg = m_ref == -INFINITY ? 0.f : -m_ref;  // nothing seen yet: weights 0, NaN stays NaN
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float e0 = ex2(fmaf(x[64 * h + 2 * c], mul, neg));
          const float e1 = ex2(fmaf(x[64 * h + 2 * c + 1], mul, neg));
          sum[2 * (c & 1)] += e0;
          sum[2 * (c & 1) + 1] += e1;
          pk[c] = pack_bf16x2(e0, e1);
        }
        tmem_st32(s_addr + 32 * h, pk);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      if (j0 < lo_max || j0 + kApmBlock > hi_min) {
        // partly visible block: V values that are not finite to zero
        const int m = 2 * b + 1;
        if (!mbar_wait_warp(&tl->full[m % kApmStages], (uint32_t)(m / kApmStages) & 1u, abort_flag)) {
          if (lane == 0) apm_fail(p, tl, kStatusTimeoutFull);
          ok = false;
          break;
        }
        uint4* v = reinterpret_cast<uint4*>(kv_smem + (size_t)(m % kApmStages) * kApmTileBytes);
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
          uint4 q = v[i * 128 + r];
          if ((not_finite2(q.x) | not_finite2(q.y) | not_finite2(q.z) | not_finite2(q.w)) != 0) {
            *reinterpret_cast<volatile int*>(&tl->poison) = 1;
            __threadfence_block();
            auto clean = [](uint32_t w) {
              const uint32_t f = not_finite2(w);
              return w & ((f & 0x8000u ? 0u : 0xFFFFu) | (f & 0x80000000u ? 0u : 0xFFFF0000u));
            };
            q = make_uint4(clean(q.x), clean(q.y), clean(q.z), clean(q.w));
            v[i * 128 + r] = q;
          }
        }
        // the tensor core sees the values written; P V starts when all four
        // warps have reported their P, so after all four quarters are clean
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tl->p_full[wg]);
    }
    // ------------------------------------------------------------ epilogue
    if (n > 0 && ok && !mbar_wait_warp(&tl->o_full[wg], 0, abort_flag)) {
      if (lane == 0) apm_fail(p, tl, kStatusTimeoutAccum);
      ok = false;
    }
    tc_fence_after();
    if (ok) {
      const bool dead = !live;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      // the row's output to shared memory (the Q tile is not read any more):
      // 16-byte pieces, 128-byte swizzle, then whole rows to global memory
      uint8_t* row_smem = q_smem + wg * kApmTileBytes + r * 128;
      const bool poison = n > 0 && *reinterpret_cast<volatile int*>(&tl->poison) != 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v[32];
        if (n > 0) {
          tmem_ld32_nowait(o_addr + 32 * c, v);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = (dead || n == 0) ? 0.f : v[i] * inv;
        if (poison && live) {
          for (int b = 0; b < n; ++b) {
            const int j0 = (blk0 + b) * kApmBlock;
            if (j0 >= lo_max && j0 + kApmBlock <= hi_min) continue;  // not cleaned
            for (int j = max(lo, j0); j < min(hi, j0 + kApmBlock); ++j) {
              const long long sl = apm_slot(p, table, j);
              if (sl < 0) continue;
              const __nv_bfloat16* vr =
                  p.pool + ((size_t)sl * 2 * p.n_kv_heads + p.n_kv_heads + kvh) * kHeadDim + 32 * c;
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
          const int ch = (c & 1) * 4 + i;
          *reinterpret_cast<uint4*>(row_smem + (c >> 1) * kApmHalf + ((ch ^ (r & 7)) << 4)) = w;
        }
      }
      if (valid && p.lse)
        p.lse[(size_t)(t_first + tok) * p.lse_stride + head] =
            (dead || n == 0 || l == 0.f) ? -INFINITY : (m_ref == -INFINITY ? l : (m_ref + log2f(l)) * kLn2);
      __syncwarp();
      const int r0 = (warp & 3) * 32;
#pragma unroll 4
      for (int it = 0; it < 16; ++it) {
        const int rr = r0 + 2 * it + (lane >> 4), ch = lane & 15;
        const int tk = tok0 + wg * tt + rr / G;
        if (seq >= 0 && rr < tt * G && tk < q_len) {
          const uint4 w = *reinterpret_cast<const uint4*>(q_smem + wg * kApmTileBytes + (ch >> 3) * kApmHalf + rr * 128 +
                                                          (((ch & 7) ^ (rr & 7)) << 4));
          *reinterpret_cast<uint4*>(p.out + (size_t)(t_first + tk) * p.out_stride +
                                    (size_t)(kvh * G + rr % G) * kHeadDim + ch * 8) = w;
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
  if (warp == 9) {
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
