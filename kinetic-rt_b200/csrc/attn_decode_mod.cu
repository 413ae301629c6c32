// Paged decode attention with score modifications (bf16, GQA): one query
// token per sequence, at position p = len - 1 of its sequence.
//
//   x_j = scale q . k_j;  x_j = c tanh(x_j / c);  x_j -= slope_h |p - j|
//   visible j: max(kv_start, p - window + 1, 0) <= j < len
//   out = sum_j softmax(x)_j v_j,  lse = log sum_j exp(x_j)
// over the pool that attn_decode.cu reads (token layout [K | V][kv_head][128]).
//
// Every visible K/V byte is read once, so the kernel is bound by HBM; the
// invisible ones (before the window or the document) are not read.  Grid
// (sequence, KV head, split of the visible 16-token chunks); two, four or eight
// warps take the CTA's chunks in turn, each with its own ring of three 8 KB
// stages (one 5-D TMA box = K and V of 16 tokens of one KV head, 128-byte
// swizzled; 192 KB under way per SM); Q K^T and P V on mma.sync m16n8k16 with
// the group's query heads in the rows (about 4 FLOP a byte: the tensor rate
// does not matter), statistics and sums in fp32; P is rounded to bf16 for P V
// (relative 2^-8 at most, as V is).  Warps merge in shared memory; splits
// through the shared memory of a cluster, or in the workspace by the last CTA to
// finish; always in split order, so results do not depend on which CTA that is.
// Measured: 128 sequences of 4224 tokens, 8 KV heads (2.2 GB) in 323 to 346 us
// (on different GPUs) = 6.4 to 6.9 TB/s; one sequence of 4224 tokens 9.5 us in a
// graph of such calls, of which about 5 are the launch, a CTA's start and its
// merges.  Pieces follow max_seq_len, not the lengths: that sequence under a
// bound of 32768 takes 17.7 us, of 131072 30.2.
//
// V rows of tokens that are not visible are set to zero in shared memory
// before P V: their weight is 0, and 0 * inf or 0 * NaN from a cache slot
// nothing was written to would spoil the row.  Only the first and last chunk
// of the visible range hold such tokens.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <cuda_runtime.h>

#include "../../include/krt.h"
#include "attn_mod.cuh"
#include "capi_internal.h"
#include "mma_frag.cuh"
#include "ptx.cuh"
#include "qkv_paged.cuh"

namespace krt {

constexpr int kAdmStages = 3;               // per warp
constexpr int kAdmChunk = 16;               // tokens per TMA box
constexpr uint32_t kAdmStageBytes = 8192;   // K and V of 16 tokens, one KV head
constexpr int kAdmMaxGroup = 16;            // query heads per KV head
constexpr int kAdmRowFloats = 4 + kHeadDim; // max, sum, (two unused), 128 outputs
constexpr int kAdmMaxCluster = 8;           // splits that merge through shared memory at most
constexpr int kAdmMaxCps = 1024;            // 16-token chunks per CTA at most

struct AdmParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  float* lse;                // [num_seqs, lse_stride] or NULL
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* kv_start;   // [num_seqs] or NULL
  float* part;               // [num_seqs][n_kv_heads][max_splits][group][kAdmRowFloats]
  uint32_t* counters;        // [num_seqs][n_kv_heads], zero between calls
  int* status;
  int bt_stride, num_blocks, tokens_per_block;
  int n_kv_heads, group;
  int q_stride, out_stride, lse_stride;
  int chunks_per_split, max_splits;
  int cluster;               // the splits of a (sequence, KV head) are one cluster
  int max_len;
  ScoreMod mod;
};

template <int WARPS>
struct AdmSmemTail {
  uint64_t full[WARPS][kAdmStages];
  int tok[kAdmMaxCps];  // first pool token of each of the CTA's chunks, -1 when the lookup failed
  int last;
};

template <int WARPS>
constexpr size_t adm_smem_bytes() {
  return 1024 + (size_t)WARPS * kAdmStages * kAdmStageBytes + sizeof(AdmSmemTail<WARPS>);
}

// One merged row: 8 output values (and, by the thread of the first 8, the lse).
__device__ __forceinline__ void adm_write_row(const AdmParams& p, int b, int head, int d0, const float* acc, float M,
                                              float L) {
  const float inv = L == 0.f ? 0.f : 1.f / L;  // nothing visible: zeros; NaN stays NaN
  const uint4 v = make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                             pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
  *reinterpret_cast<uint4*>(p.out + (size_t)b * p.out_stride + (size_t)head * kHeadDim + d0) = v;
  if (p.lse && d0 == 0)
    p.lse[(size_t)b * p.lse_stride + head] = L == 0.f ? -INFINITY : (M == -INFINITY ? L : (M + log2f(L)) * kLn2);
}

template <int WARPS, bool CAP, bool BIAS>
__global__ void __launch_bounds__(32 * WARPS, 8 / WARPS)
    paged_attention_decode_mod_kernel(const __grid_constant__ CUtensorMap tmap_kv, const AdmParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int kAdmWarps = WARPS, kAdmThreads = 32 * WARPS;
  auto* tl = reinterpret_cast<AdmSmemTail<WARPS>*>(smem + (size_t)kAdmWarps * kAdmStages * kAdmStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int b = blockIdx.x, kvh = blockIdx.y, z = blockIdx.z;
  const int G = p.group;

  if (lane == 0) {
    for (int s = 0; s < kAdmStages; ++s) mbar_init(&tl->full[warp][s], 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) tma_prefetch_desc(&tmap_kv);
  __syncwarp();
  pdl_wait();  // q and the pool come from the previous kernel
  pdl_launch_dependents();

  int len = p.seq_lens[b];
  if (len > p.max_len) {
    // beyond the grid (and the workspace): attend over the first max_len tokens and report it
    if (threadIdx.x == 0 && z == 0 && kvh == 0) atomicOr(p.status, kStatusBadBlock);
    len = p.max_len;
  }
  if (len < 0) len = 0;
  const int pos = len - 1;
  int lo = p.kv_start ? p.kv_start[b] : 0;
  if (p.mod.window > 0 && lo < len - p.mod.window) lo = len - p.mod.window;
  if (lo < 0) lo = 0;
  const int chunk0 = lo / kAdmChunk;
  const int n_chunks = lo < len ? (len + kAdmChunk - 1) / kAdmChunk - chunk0 : 0;
  const int splits = n_chunks > 0 ? (n_chunks + p.chunks_per_split - 1) / p.chunks_per_split : 1;
  if (z >= splits) return;  // the whole CTA: nothing of this sequence left for it
  const int c_begin = chunk0 + z * p.chunks_per_split;
  const int c_count = min(chunk0 + n_chunks, c_begin + p.chunks_per_split) - c_begin;

  // First pool token of every chunk of this CTA (-1 when the block id is out of
  // range: the chunk is masked).  The table holds the column: len <= max_len.
  for (int i = threadIdx.x; i < c_count; i += kAdmThreads) {
    const int tok = (c_begin + i) * kAdmChunk;
    const int blk = p.block_table[(size_t)b * p.bt_stride + tok / p.tokens_per_block];
    const int v = blk >= 0 && blk < p.num_blocks ? blk * p.tokens_per_block + tok % p.tokens_per_block : -1;
    if (v < 0) atomicOr(p.status, kStatusBadBlock);
    tl->tok[i] = v;
  }
  __syncthreads();
  uint8_t* wstage = smem + (size_t)warp * kAdmStages * kAdmStageBytes;
  const uint32_t wstage_u32 = smem_u32(wstage);
  // lane 0 issues this warp's loads: the k-th chunk of the warp is
  // warp + kAdmWarps * k of the CTA's and uses stage k % kAdmStages
  auto issue = [&](int k) {
    const int tok = tl->tok[warp + kAdmWarps * k];
    uint64_t* bar = &tl->full[warp][k % kAdmStages];
    mbar_arrive_expect_tx(bar, kAdmStageBytes);
    const uint64_t pol = make_l2_policy_evict_first();
    tma_load_5d(wstage + (size_t)(k % kAdmStages) * kAdmStageBytes, &tmap_kv, bar, 0, tok < 0 ? 0 : tok, 0, 0, kvh,
                pol);
  };
  const int my_chunks = c_count > warp ? (c_count - warp + kAdmWarps - 1) / kAdmWarps : 0;
  int issued = my_chunks < kAdmStages ? my_chunks : kAdmStages;
  if (lane == 0)
    for (int k = 0; k < issued; ++k) issue(k);

  // Query fragments (A operand, rows = query heads of the group, zero-padded
  // to 16): k-step ks covers dims 16 ks .. 16 ks + 15.
  uint32_t qa[8][4];
  {
    const __nv_bfloat16* qrow0 = p.q + (size_t)b * p.q_stride + (size_t)(kvh * G + g) * kHeadDim;
    const __nv_bfloat16* qrow1 = qrow0 + 8 * kHeadDim;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      const int d0 = 16 * ks + 2 * t4;
      qa[ks][0] = g < G ? *reinterpret_cast<const uint32_t*>(qrow0 + d0) : 0u;
      qa[ks][1] = g + 8 < G ? *reinterpret_cast<const uint32_t*>(qrow1 + d0) : 0u;
      qa[ks][2] = g < G ? *reinterpret_cast<const uint32_t*>(qrow0 + d0 + 8) : 0u;
      qa[ks][3] = g + 8 < G ? *reinterpret_cast<const uint32_t*>(qrow1 + d0 + 8) : 0u;
    }
  }
  float slope2[2] = {0.f, 0.f};  // distance bias of rows g and g + 8, base 2
  if (BIAS) {
    constexpr float kLog2e = 1.4426950408889634f;
    if (g < G) slope2[0] = p.mod.slopes[kvh * G + g] * kLog2e;
    if (g + 8 < G) slope2[1] = p.mod.slopes[kvh * G + g + 8] * kLog2e;
  }

  float o[16][4];
#pragma unroll
  for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m_r[2] = {-INFINITY, -INFINITY};  // running max of rows g and g + 8 (base-2 scores)
  float l_r[2] = {0.f, 0.f};              // this lane's share of the running sums
  bool ok = true;

  for (int k = 0; k < my_chunks; ++k) {
    const int s = k % kAdmStages;
    const uint32_t ph = (uint32_t)(k / kAdmStages) & 1u;
    if (!mbar_wait_warp(&tl->full[warp][s], ph, nullptr)) {
      ok = false;
      break;
    }
    const uint32_t st = wstage_u32 + (uint32_t)s * kAdmStageBytes;
    const int ci = warp + kAdmWarps * k;
    const int tok_base = (c_begin + ci) * kAdmChunk;
    // visible tokens of the chunk: [v0, v1)
    int v0 = lo - tok_base, v1 = len - tok_base;
    v0 = v0 < 0 ? 0 : v0;
    v1 = v1 > kAdmChunk ? kAdmChunk : v1;
    if (tl->tok[ci] < 0) v1 = 0;
    const bool partial = v0 > 0 || v1 < kAdmChunk;
    if (partial) {
      // V rows of invisible tokens to zero (two 2 KB halves, 8 16-byte pieces a row)
      uint4* vrows = reinterpret_cast<uint4*>(wstage + (size_t)s * kAdmStageBytes + 4096);
      for (int i = lane; i < 256; i += 32) {
        const int tok = (i >> 3) & 15;
        if (tok < v0 || tok >= v1) vrows[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();  // before a later TMA load rewrites the stage
      __syncwarp();
    }
    // ---- S = Q K^T for the 16 tokens (two n-tiles of 8)
    float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    {
      const int mat = lane >> 3, r = lane & 7;
      const int tok = r + 8 * (mat >> 1);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        const int half = ks >> 2, ch = 2 * (ks & 3) + (mat & 1);
        uint32_t bf[4];
        ldsm_x4(sw128_addr(st + (uint32_t)half * 2048u, tok, ch), bf);
        mma_bf16_16816(sc[0], qa[ks], bf[0], bf[1]);
        mma_bf16_16816(sc[1], qa[ks], bf[2], bf[3]);
      }
    }
    // ---- modifications, mask, online softmax (base 2)
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tk = 8 * j + 2 * t4 + (e & 1);
        float v = CAP ? cap_score(sc[j][e], p.mod.cap_in, p.mod.cap2) : sc[j][e] * p.mod.mul;
        if (CAP && p.mod.wide_cap && fabsf(sc[j][e]) <= p.mod.poly_max) v = cap_at(sc[j][e], p.mod.poly);
        if (BIAS) v = fmaf(-slope2[e >> 1], (float)(pos - tok_base - tk), v);  // j <= pos: the distance is >= 0
        if (tk < v0 || tk >= v1) v = -INFINITY;
        sc[j][e] = v;
        mx[e >> 1] = fmaxf(mx[e >> 1], v);
      }
    float corr[2], mu[2];
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
      mx[rr] = fmaxf(mx[rr], __shfl_xor_sync(0xffffffffu, mx[rr], 1));
      mx[rr] = fmaxf(mx[rr], __shfl_xor_sync(0xffffffffu, mx[rr], 2));
      const float m_new = fmaxf(m_r[rr], mx[rr]);
      mu[rr] = m_new == -INFINITY ? 0.f : m_new;  // nothing seen yet: weights 0, and a NaN score stays one
      corr[rr] = ex2(m_r[rr] - mu[rr]);
      m_r[rr] = m_new;
    }
    float pr[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) pr[j][e] = ex2(sc[j][e] - mu[e >> 1]);
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) l_r[rr] = l_r[rr] * corr[rr] + pr[0][2 * rr] + pr[0][2 * rr + 1] + pr[1][2 * rr] +
                                             pr[1][2 * rr + 1];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      o[j][0] *= corr[0];
      o[j][1] *= corr[0];
      o[j][2] *= corr[1];
      o[j][3] *= corr[1];
    }
    // ---- O += P V (P as the A operand: the S accumulators re-packed as bf16)
    uint32_t pa[4];
    pa[0] = pack_bf16x2(pr[0][0], pr[0][1]);
    pa[1] = pack_bf16x2(pr[0][2], pr[0][3]);
    pa[2] = pack_bf16x2(pr[1][0], pr[1][1]);
    pa[3] = pack_bf16x2(pr[1][2], pr[1][3]);
    {
      const int mat = lane >> 3, r = lane & 7;
      const int tok = r + 8 * (mat & 1);
#pragma unroll
      for (int jj = 0; jj < 8; ++jj) {
        const int half = jj >> 2, ch = 2 * (jj & 3) + (mat >> 1);
        uint32_t bf[4];
        ldsm_x4_trans(sw128_addr(st + 4096u + (uint32_t)half * 2048u, tok, ch), bf);
        mma_bf16_16816(o[2 * jj], pa, bf[0], bf[1]);
        mma_bf16_16816(o[2 * jj + 1], pa, bf[2], bf[3]);
      }
    }
    // ---- refill the stage with this warp's chunk k + kAdmStages
    __syncwarp();
    if (k + kAdmStages < my_chunks) {
      if (lane == 0) {
        fence_proxy_async_smem();  // the ldmatrix reads above come before the TMA rewrites the stage
        issue(k + kAdmStages);
      }
      issued = k + kAdmStages + 1;
    }
  }
  if (!ok && lane == 0) {
    // A load did not land in time: record it and wait (bounded) for every
    // load this warp still has in flight before the CTA may exit.
    atomicOr(p.status, kStatusTimeoutFull);
    for (int k = issued - kAdmStages > 0 ? issued - kAdmStages : 0; k < issued; ++k)
      mbar_wait(&tl->full[warp][k % kAdmStages], (uint32_t)(k / kAdmStages) & 1u, nullptr);
  }
#pragma unroll
  for (int rr = 0; rr < 2; ++rr) {
    l_r[rr] += __shfl_xor_sync(0xffffffffu, l_r[rr], 1);
    l_r[rr] += __shfl_xor_sync(0xffffffffu, l_r[rr], 2);
  }

  // ---- merge the warps: rows [warp][row][max, sum, 128 outputs] in the
  // (now idle) stage buffers
  __syncthreads();
  float* wrow = reinterpret_cast<float*>(smem);
  auto row_at = [&](int w, int row) { return wrow + ((size_t)w * kAdmMaxGroup + row) * kAdmRowFloats; };
#pragma unroll
  for (int rr = 0; rr < 2; ++rr) {
    const int row = g + 8 * rr;
    if (row >= G) continue;
    float* dst = row_at(warp, row);
    if (t4 == 0) {
      dst[0] = m_r[rr];
      dst[1] = l_r[rr];
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      *reinterpret_cast<float2*>(dst + 4 + 8 * j + 2 * t4) = make_float2(o[j][2 * rr], o[j][2 * rr + 1]);
    }
  }
  __syncthreads();
  // thread -> (row, 8 dims) pairs of the merged result
  const bool single = splits == 1;
  // this CTA's merged rows: behind the warps' rows, or in the workspace
  float* mine = wrow + WARPS * kAdmMaxGroup * kAdmRowFloats;
  float* part = p.cluster ? mine
                          : p.part + (((size_t)b * p.n_kv_heads + kvh) * p.max_splits + z) * (size_t)G * kAdmRowFloats;
  for (int idx = threadIdx.x; idx < G * 16; idx += kAdmThreads) {
    const int row = idx >> 4, d0 = (idx & 15) * 8;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kAdmWarps; ++w) M = fmaxf(M, row_at(w, row)[0]);
    float L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kAdmWarps; ++w) {
      const float* src = row_at(w, row);
      const float f = M == -INFINITY ? 1.f : ex2(src[0] - M);
      L += f * src[1];
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += f * src[4 + d0 + i];
    }
    if (single) {
      adm_write_row(p, b, kvh * G + row, d0, acc, M, L);
    } else {
      float* dst = part + (size_t)row * kAdmRowFloats;
      if (d0 == 0) {
        dst[0] = M;
        dst[1] = L;
      }
      *reinterpret_cast<float4*>(dst + 4 + d0) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(dst + 8 + d0) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
  }
  if (single) return;

  // ---- several splits, merged in their order.  at(k, i): four floats of split
  // k's rows from float i; in groups whose loads are all under way together
  auto join = [&](int idx, auto&& at) {
    const int row = idx >> 4, d0 = (idx & 15) * 8, first = row * kAdmRowFloats;
    float M = -INFINITY, L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int z0 = 0; z0 < splits; z0 += 8) {
      float m[8], ls[8];
      float4 lo4[8], hi4[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = z0 + k < splits;
        const int zz = in ? z0 + k : z0;
        const float4 ml = at(zz, first);
        m[k] = in ? ml.x : -INFINITY;
        ls[k] = in ? ml.y : 0.f;
        lo4[k] = at(zz, first + 4 + d0);
        hi4[k] = at(zz, first + 8 + d0);
      }
      float mx = M;
#pragma unroll
      for (int k = 0; k < 8; ++k) mx = fmaxf(mx, m[k]);
      const float mu = mx == -INFINITY ? 0.f : mx;  // nothing seen: factors 0 of zeros, NaN stays NaN
      const float keep = M == mx ? 1.f : ex2(M - mu);
      M = mx;
      L *= keep;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= keep;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (z0 + k >= splits) break;
        const float f = m[k] == mx ? 1.f : ex2(m[k] - mu);
        L += f * ls[k];
        acc[0] += f * lo4[k].x;
        acc[1] += f * lo4[k].y;
        acc[2] += f * lo4[k].z;
        acc[3] += f * lo4[k].w;
        acc[4] += f * hi4[k].x;
        acc[5] += f * hi4[k].y;
        acc[6] += f * hi4[k].z;
        acc[7] += f * hi4[k].w;
      }
    }
    adm_write_row(p, b, kvh * G + row, d0, acc, M, L);
  };
  if (p.cluster) {
    // the splits are the CTAs of a cluster (those beyond `splits` have left):
    // each reads its share of the rows from the others' shared memory
    cluster_sync();
    const uint32_t rows = smem_u32(mine);
    const int idx = z + splits * threadIdx.x;
    if (idx < G * 16)
      join(idx, [&](int k, int i) { return ld_cluster_f4(map_smem_to_rank(rows, (uint32_t)k) + 4u * (uint32_t)i); });
    cluster_sync();  // no CTA leaves while its rows are read
    return;
  }
  // through the workspace: the last CTA of this (sequence, KV head) merges
  __threadfence();  // this CTA's partial is visible GPU-wide before the count
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t* ctr = p.counters + (size_t)b * p.n_kv_heads + kvh;
    const uint32_t prev = atomicAdd(ctr, 1u);
    const bool last = prev + 1 == (uint32_t)splits;
    if (last) *ctr = 0u;  // ready for the next call
    tl->last = last ? 1 : 0;
  }
  __syncthreads();
  if (!tl->last) return;
  __threadfence();
  const float* base = p.part + ((size_t)b * p.n_kv_heads + kvh) * p.max_splits * (size_t)G * kAdmRowFloats;
  for (int idx = threadIdx.x; idx < G * 16; idx += kAdmThreads)
    join(idx, [&](int k, int i) {
      return __ldcg(reinterpret_cast<const float4*>(base + (size_t)k * G * kAdmRowFloats + i));
    });
}

typedef void (*AdmKernel)(const CUtensorMap, const AdmParams);
template <int WARPS>
AdmKernel adm_kernel(bool cap, bool bias) {
  if (cap)
    return bias ? paged_attention_decode_mod_kernel<WARPS, true, true>
                : paged_attention_decode_mod_kernel<WARPS, true, false>;
  return bias ? paged_attention_decode_mod_kernel<WARPS, false, true>
              : paged_attention_decode_mod_kernel<WARPS, false, false>;
}

}  // namespace krt

using namespace krt;

// ------------------------------------------------------------------ C ABI
namespace {

// 16-token chunks a sequence can have to read: all of max_seq_len, or what a
// window that starts inside a chunk touches.
int adm_max_chunks(int max_seq_len, int window) {
  const long long all = ((long long)max_seq_len + kAdmChunk - 1) / kAdmChunk;
  if (window <= 0) return (int)all;
  const long long win = ((long long)window + 2 * kAdmChunk - 2) / kAdmChunk;
  return (int)(win < all ? win : all);
}

// CTAs per (sequence, KV head): as many as fill the SMs once, but at most
// sqrt(chunks) / 2 (the merge grows with their number as the scan shrinks).
// More, smaller pieces lose: every CTA starts its pipeline, merges its warps
// and leaves an fp32 partial.  Measured (us, merged through the workspace),
// pairs x chunks, this rule against two CTAs per SM and more: 256 x 65 25.6 : 31.0, 160 x 63 17.5 : 25.6,
// 128 x 128 26.0 : 31.7, 8 x 512 14.7 : 17.1 (37 splits 26.8),
// 8 x 264 11.1 : 17.5.  Long scans that leave a tenth of the SMs idle are cut
// at 512 chunks, which evens out ragged lengths: 40 x 4096 177 : 190,
// 90 x 2048 187 : 205; where the SMs are full they are not: 24 x 4096
// 129 : 133.
int adm_splits(long long pairs, int max_chunks) {
  const long long sms = device_sm_count(), most = (long long)(std::sqrt((double)max_chunks) / 2);
  const long long s = std::max(1ll, std::min(sms / pairs, most));
  const int deepest = 10 * s * pairs >= 9 * sms && s * pairs <= sms ? kAdmMaxCps : kAdmMaxCps / 2;
  return (int)std::max<long long>(s, (max_chunks + deepest - 1) / deepest);
}

// Clusters of `size` CTAs of eight warps that can be resident at once on the
// current device (asked once per kernel, size and device).
int adm_clusters(bool cap, bool bias, int size) {
  static std::atomic<int> known[16][4][kAdmMaxCluster + 1];  // the count + 1, 0: not asked yet
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  std::atomic<int>* at = dev < 16 ? &known[dev][2 * cap + bias][size] : nullptr;
  if (at && (n = at->load(std::memory_order_relaxed)) != 0) return n - 1;
  AdmKernel kern = adm_kernel<8>(cap, bias);
  const size_t smem = adm_smem_bytes<8>();
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = (unsigned)size;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, 1, (unsigned)size);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (at) at->store(n + 1, std::memory_order_relaxed);
  return n;
}

// fp32 partial rows of the largest call of at most that many pairs and chunks
// (a row of every query head per split), so that a workspace made for the
// largest batch serves smaller ones, which have more splits each.
size_t adm_part_bytes(long long pairs, int group, int max_chunks) {
  const long long deepest = (max_chunks + kAdmMaxCps / 2 - 1) / (kAdmMaxCps / 2);
  const long long most = std::max(1, (int)(std::sqrt((double)max_chunks) / 2));
  const long long parts = std::max(pairs * deepest, std::min<long long>(device_sm_count(), pairs * most));
  return (size_t)parts * group * kAdmRowFloats * 4;
}

}  // namespace

extern "C" size_t krt_paged_attention_mod_workspace_size(int32_t num_seqs, int32_t n_heads, int32_t n_kv_heads,
                                                         int32_t max_seq_len, int32_t window) {
  if (num_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || max_seq_len <= 0 || window < 0 ||
      n_heads % n_kv_heads != 0 || n_heads / n_kv_heads > kAdmMaxGroup)
    return 0;
  const long long pairs = (long long)num_seqs * n_kv_heads;
  const size_t own = pairs > kModCounters ? (size_t)pairs * 4 : 0;
  return kModPartsAt + adm_part_bytes(pairs, n_heads / n_kv_heads, adm_max_chunks(max_seq_len, window)) + own;
}

extern "C" int krt_paged_attention_decode_mod(const krt_paged_attention_mod_args* a, void* stream) {
  const char* name = "krt_paged_attention_decode_mod";
  if (!a) return set_error(KRT_ERR_INVALID, "%s: args is NULL", name);
  if (!a->q || !a->kv_pool || !a->block_table || !a->seq_lens || !a->out || !a->workspace)
    return set_error(KRT_ERR_INVALID, "%s: a required pointer is NULL", name);
  if (a->num_seqs <= 0 || a->n_heads <= 0 || a->n_kv_heads <= 0 || a->max_seq_len <= 0)
    return set_error(KRT_ERR_INVALID, "%s: num_seqs, heads and max_seq_len must be positive", name);
  if (a->head_dim != kHeadDim) return set_error(KRT_ERR_UNSUPPORTED, "%s: head_dim must be 128", name);
  if (a->n_heads % a->n_kv_heads != 0 || a->n_heads / a->n_kv_heads > kAdmMaxGroup || a->n_kv_heads > 65535)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: n_heads must be a multiple of n_kv_heads, at most 16 per KV head", name);
  if (a->tokens_per_block <= 0 || a->tokens_per_block % kAdmChunk != 0)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: tokens_per_block must be a multiple of 16", name);
  if (a->num_blocks <= 0 || a->block_table_stride <= 0)
    return set_error(KRT_ERR_INVALID, "%s: paged-cache geometry must be positive", name);
  const int columns = block_table_columns(a->block_table_columns, a->block_table_stride, a->num_seqs);
  if (columns < 0)
    return set_error(KRT_ERR_INVALID, "%s: block_table_columns must lie in 0 .. block_table_stride", name);
  if ((long long)a->num_blocks * a->tokens_per_block > INT_MAX - kAdmChunk)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: the pool may hold fewer than 2^31 - 16 tokens", name);
  if ((long long)columns * a->tokens_per_block < a->max_seq_len)
    return set_error(KRT_ERR_INVALID, "%s: the block table cannot hold max_seq_len tokens", name);
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
  const size_t need = krt_paged_attention_mod_workspace_size(a->num_seqs, a->n_heads, a->n_kv_heads, a->max_seq_len,
                                                             a->window);
  if (a->workspace_bytes < need)
    return set_error(KRT_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, a->workspace_bytes, need);
  const int max_chunks = adm_max_chunks(a->max_seq_len, a->window);
  AdmParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.lse = a->lse;
  p.block_table = a->block_table;
  p.seq_lens = a->seq_lens;
  p.kv_start = a->kv_start;
  char* ws = static_cast<char*>(a->workspace);
  p.status = reinterpret_cast<int*>(ws);
  p.part = reinterpret_cast<float*>(ws + kModPartsAt);
  p.counters = reinterpret_cast<uint32_t*>(ws + kModCountersAt);
  p.bt_stride = a->block_table_stride;
  p.num_blocks = a->num_blocks;
  p.tokens_per_block = a->tokens_per_block;
  p.n_kv_heads = a->n_kv_heads;
  p.group = a->n_heads / a->n_kv_heads;
  p.q_stride = a->q_stride;
  p.out_stride = a->out_stride;
  p.lse_stride = a->lse_stride;
  p.max_len = a->max_seq_len;
  const long long pairs = (long long)a->num_seqs * a->n_kv_heads;
  const bool cap = a->softcap > 0.f, bias = a->alibi_slopes != nullptr;
  int splits = adm_splits(pairs, max_chunks);
  // Splits of one cluster merge through shared memory, 1.3 to 2 us sooner than
  // through the workspace (1 x 4224 tokens 10.9 : 9.0, 1 x 500 7.1 : 5.9,
  // 40 pairs x 188 chunks 17.9 : 15.9): as many of them as the clusters that
  // fit allow, unless the longer scan (90 ns a chunk) costs more than that.
  for (int c = std::min(splits, kAdmMaxCluster); c > 1; --c) {
    if ((long long)max_chunks * (splits - c) > 20ll * c * splits) break;
    if (adm_clusters(cap, bias, c) >= pairs) {
      splits = c;
      p.cluster = 1;
      break;
    }
  }
  p.chunks_per_split = (max_chunks + splits - 1) / splits;
  p.max_splits = (max_chunks + p.chunks_per_split - 1) / p.chunks_per_split;
  if (p.max_splits == 1 || (p.cluster && adm_clusters(cap, bias, p.max_splits) < pairs)) p.cluster = 0;
  if (p.max_splits > 65535) return set_error(KRT_ERR_UNSUPPORTED, "%s: max_seq_len is too long", name);
  p.mod = make_score_mod(a->scale, a->softcap, a->alibi_slopes, a->window);
  // The cap's exponent form is off by 2e-7 of the cap, up to 100 less than 1 % of
  // the weights' rounding to bf16; beyond, small scores take the polynomial too
  // (always: 341 us for 128 sequences of 4224, never: 329).
  p.mod.wide_cap = a->softcap > 100.f;
  CUtensorMap tmap;
  int rc = make_tmap_pool_kv16(&tmap, a->kv_pool, a->num_blocks, a->tokens_per_block, a->n_kv_heads, true);
  if (rc) return rc;
  // Eight warps and one CTA per SM, or four and two CTAs, so that all are
  // resident at once (clusters fit one per SM).  Of more CTAs than that, short
  // ones take two warps, four per SM: their start and end dominate.  Measured
  // (us), eight : four : two warps: 100 CTAs x 264 chunks 39.7 : 45.1,
  // 75 x 125 16.9 : 23.1; 160 x 63 23.2 : 17.5, 256 x 65 28.4 : 25.6;
  // 1600 x 1 33 : 18 : 10, 1600 x 32 78 : 70 : 67, 480 x 63 49 : 43 : 42;
  // ragged 512 x 264 127 : 133 : 139, 1024 x 264 245 : 251 : 265.
  const long long ctas = pairs * p.max_splits, sms = device_sm_count();
  const int warps = ctas <= sms ? 8 : ctas <= 2 * sms ? 4 : p.chunks_per_split <= 64 ? 2 : 8;
  AdmKernel kern = warps == 8   ? adm_kernel<8>(cap, bias)
                   : warps == 4 ? adm_kernel<4>(cap, bias)
                                : adm_kernel<2>(cap, bias);
  const size_t smem = warps == 8 ? adm_smem_bytes<8>() : warps == 4 ? adm_smem_bytes<4>() : adm_smem_bytes<2>();
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return cuda_error(e, name);
  if (pairs > kModCounters && p.max_splits > 1 && !p.cluster) {
    // more pairs than the workspace has counters for: behind the partials, where
    // other calls leave anything
    p.counters = reinterpret_cast<uint32_t*>(ws + kModPartsAt + adm_part_bytes(pairs, p.group, max_chunks));
    e = cudaMemsetAsync(p.counters, 0, (size_t)pairs * 4, (cudaStream_t)stream);
    if (e != cudaSuccess) return cuda_error(e, name);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a->num_seqs, (unsigned)a->n_kv_heads, (unsigned)p.max_splits);
  cfg.blockDim = dim3(32u * warps, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = (unsigned)p.max_splits;
  if (p.cluster) cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kern, tmap, p);
  if (e != cudaSuccess) return cuda_error(e, name);
  return clear_error();
}
