// Rotary positions of q and k, and k and v appended to the paged KV cache.
//
// For token t at position p and pair i of the first R dims of a q or k head,
//   angle = p * inv_freq[i]
//   (a, b) -> (a cos - b sin, b cos + a sin) * factor
// where (a, b) are dims (2i, 2i + 1) (interleaved) or (i, i + R / 2) (halves);
// dims R .. 127 pass through.  q goes to q_out, k and v to the slot of the
// token's cache index (token layout [K | V][kv_head][128] bf16).
//
// The kernel reads and writes every element once and is bound by HBM.  One to
// eight warps take a token: its threads ask for their first vectors, then
// compute the token's R / 2 cosines and sines into shared memory while those
// are under way; all heads share them.  The angle is taken in fp64 turns
// (p * inv_freq / 2 pi) and reduced to its fraction before the fp32 sine: at
// position 10^6 an fp32 angle would be off by 0.06.  This costs R / 2 fp64
// products a token, against R * heads products, and saves the table that limits
// the position.  Unit u of a head is two 8-element vectors that a thread loads,
// rotates and stores (16-byte accesses): the two partners of a half-split
// rotation, or two vectors of interleaved pairs.  Halves that end inside a
// vector go through shared memory.
//
// Measured: 16384 tokens of 32 + 8 heads (bf16, 403 MB) in 67 us = 6.0 TB/s;
// 32 k tokens of 8 + 1 heads (fp32 in, 250 MB) in 46 us = 5.4 TB/s: with ten
// heads the angles are a third of a warp's time on its token.  More warps
// matter more than vectors per thread: two fp32 units per thread (two CTAs per
// SM fewer) take 52 us, four bf16 units 72 us.  A CTA for four tokens with a
// barrier after the angles took 74 and 60.  64 tokens take 2.8 us in a graph.
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <cuda_runtime.h>

#include "../../include/krt.h"
#include "capi_internal.h"
#include "ptx.cuh"
#include "qkv_paged.cuh"

namespace krt {

constexpr int kRaThreads = 256;
constexpr int kRaUnits = 8;      // two-vector units per head

struct RaParams {
  const void *q, *k, *v;  // [num_tokens, *_stride] in, head h at h * 128
  const double* inv_freq;
  const int32_t* positions;
  const int32_t* cache_index;
  const int32_t* token_seq;
  const int32_t* block_table;
  __nv_bfloat16* pool;
  __nv_bfloat16* q_out;
  int* status;
  long long q_stride, k_stride, v_stride, q_out_stride;
  int num_tokens, n_heads, n_kv_heads, rotary_dim;
  int num_seqs, bt_stride, bt_columns, num_blocks, tokens_per_block;
  float factor;
};
// (a launch with more costs the host 0.3 us: 2.8 in all, where the kernel takes 2.6 for 64 tokens)
static_assert(sizeof(RaParams) <= 160);


// Eight elements as they lie in memory (read once: marked to leave the caches
// first), and as fp32.
template <typename T>
struct RaVec;
template <>
struct RaVec<float> {
  static constexpr int kBatch = 1;  // units a thread has under way
  float4 lo, hi;
  __device__ __forceinline__ void load(const float* src) {
    lo = __ldcs(reinterpret_cast<const float4*>(src));
    hi = __ldcs(reinterpret_cast<const float4*>(src) + 1);
  }
  __device__ __forceinline__ void get(float* x) const {
    x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
  }
};
template <>
struct RaVec<__nv_bfloat16> {
  static constexpr int kBatch = 2;
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* src) { v = __ldcs(reinterpret_cast<const uint4*>(src)); }
  __device__ __forceinline__ void get(float* x) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
__device__ __forceinline__ void ra_store8(__nv_bfloat16* dst, const float* x) {
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                              pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

// How pairs lie in a head: on dims (2i, 2i + 1); on (i, i + R / 2) with both
// halves whole vectors; or with halves that end inside a vector.
enum { kRaInterleaved = 0, kRaHalves = 1, kRaOddHalves = 2 };

// WARPS warps take a token; a CTA of eight holds 8 / WARPS tokens.
template <typename T, int MODE, int WARPS>
__global__ void __launch_bounds__(kRaThreads, 4) rope_append_kernel(const RaParams p) {
  constexpr int kLanes = 32 * WARPS, kRows = kLanes / kRaUnits;  // threads of a token, heads they have at a time
  constexpr int kBatch = RaVec<T>::kBatch;
  __shared__ float2 cs_all[kRaThreads / kLanes][64];  // of pair f at ra_at(f)
  __shared__ __align__(16) float rows[MODE == kRaOddHalves ? kRaThreads / kRaUnits : 1][kHeadDim + 4];
  const int part = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const int t = blockIdx.x * (kRaThreads / kLanes) + part;
  if (t >= p.num_tokens) return;  // all of the token's warps
  const int H = p.n_heads, K = p.n_kv_heads, heads = H + 2 * K, half = p.rotary_dim / 2;
  float2* cs = cs_all[part];
  // element j of the eight threads of a head in eight neighbouring words
  auto ra_at = [](int f) { return MODE == kRaInterleaved ? (f & 3) * 16 + (f >> 2) : (f & 7) * 8 + (f >> 3); };

  // A thread keeps its unit u of a head's eight; va, vb: the unit's two vectors
  // in a rotated head (in a V head u and u + 8).
  const int u = lane % kRaUnits, pairs_r = p.rotary_dim / 16;
  int va = u, vb = u + 8;
  if (MODE == kRaHalves) {
    va = u < pairs_r ? u : pairs_r + u;
    vb = u < pairs_r ? u + pairs_r : u + 8;
  }
  auto source = [&](int h) {
    return h < H       ? static_cast<const T*>(p.q) + t * p.q_stride + h * kHeadDim
           : h < H + K ? static_cast<const T*>(p.k) + t * p.k_stride + (h - H) * kHeadDim
                       : static_cast<const T*>(p.v) + t * p.v_stride + (h - H - K) * kHeadDim;
  };
  RaVec<T> a[kBatch], b[kBatch];
  auto fetch = [&](int head) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = head + i * kRows;
      if (h < heads) {
        const T* src = source(h);
        a[i].load(src + 8 * (h < H + K ? va : u));
        b[i].load(src + 8 * (h < H + K ? vb : u + 8));
      }
    }
  };

  pdl_wait();  // q, k, v come from the previous kernel
  pdl_launch_dependents();
  const int seq = p.token_seq[t], position = p.positions[t];
  int head = lane / kRaUnits;
  fetch(head);          // under way while the angles are computed
  if (seq < 0) return;  // padding (all threads of the token)
  long long slot = -1;  // in the pool; -1: k and v are not written
  const int at = p.cache_index ? p.cache_index[t] : position;
  const int col = at >= 0 ? at / p.tokens_per_block : -1;
  if (seq < p.num_seqs && col >= 0 && col < p.bt_columns) {
    const int blk = p.block_table[(size_t)seq * p.bt_stride + col];
    if (blk >= 0 && blk < p.num_blocks)
      slot = (long long)blk * p.tokens_per_block + (at - col * p.tokens_per_block);
  }
  if (slot < 0 && lane == 0) atomicOr(p.status, kStatusBadBlock);
  for (int f = lane; f < half; f += kLanes) {
    const double turns = (double)position * (p.inv_freq[f] * 0.15915494309189535);  // / 2 pi
    float sn, c;
    sincospif(2.f * (float)(turns - floor(turns)), &sn, &c);
    cs[ra_at(f)] = make_float2(c * p.factor, sn * p.factor);
  }
  if (WARPS == 1)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(1 + part), "r"(kLanes) : "memory");  // the token's warps

  for (const int last = slot >= 0 ? heads : H; head < last;) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = head + i * kRows;
      if (h >= last) break;
      const bool rot = h < H + K;
      __nv_bfloat16* dst = h < H ? p.q_out + t * p.q_out_stride + h * kHeadDim
                                 // pool slot: K heads, then V heads
                                 : p.pool + (slot * 2 * K + (h - H)) * kHeadDim;
      float x[8], y[8];
      a[i].get(x);
      b[i].get(y);
      if (rot && MODE == kRaInterleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (4 * u + j < half) {
            const float2 w = cs[16 * j + u];
            const float c = x[2 * j], d = x[2 * j + 1];
            x[2 * j] = c * w.x - d * w.y;
            x[2 * j + 1] = d * w.x + c * w.y;
          }
          if (4 * (u + 8) + j < half) {
            const float2 w = cs[16 * j + u + 8];
            const float c = y[2 * j], d = y[2 * j + 1];
            y[2 * j] = c * w.x - d * w.y;
            y[2 * j + 1] = d * w.x + c * w.y;
          }
        }
      } else if (rot && MODE == kRaHalves) {
        if (u < pairs_r) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 w = cs[8 * j + u];
            const float c = x[j], d = y[j];
            x[j] = c * w.x - d * w.y;
            y[j] = d * w.x + c * w.y;
          }
        }
      } else if (rot) {
        // partners do not fall on vectors: the head's eight threads exchange them
        // through shared memory
        float* row = rows[threadIdx.x / kRaUnits];
        const uint32_t peers = 0xFFu << (threadIdx.x & 24);
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          *reinterpret_cast<float4*>(row + 8 * u + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
          *reinterpret_cast<float4*>(row + 64 + 8 * u + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
        }
        __syncwarp(peers);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int dx = 8 * u + j, dy = dx + 64;
          if (dx < p.rotary_dim) {
            const int f = dx < half ? dx : dx - half;
            const float2 w = cs[ra_at(f)];
            const float o = row[dx < half ? dx + half : f];
            x[j] = dx < half ? x[j] * w.x - o * w.y : x[j] * w.x + o * w.y;
          }
          if (dy < p.rotary_dim) {
            const int f = dy < half ? dy : dy - half;
            const float2 w = cs[ra_at(f)];
            const float o = row[dy < half ? dy + half : f];
            y[j] = dy < half ? y[j] * w.x - o * w.y : y[j] * w.x + o * w.y;
          }
        }
        __syncwarp(peers);
      }
      ra_store8(dst + 8 * (rot ? va : u), x);
      ra_store8(dst + 8 * (rot ? vb : u + 8), y);
    }
    head += kBatch * kRows;
    fetch(head);
  }
}

typedef void (*RaKernel)(const RaParams);
template <typename T, int WARPS>
RaKernel ra_kernel_of(bool interleaved, int rotary_dim) {
  if (interleaved) return rope_append_kernel<T, kRaInterleaved, WARPS>;
  return rotary_dim % 16 == 0 ? rope_append_kernel<T, kRaHalves, WARPS> : rope_append_kernel<T, kRaOddHalves, WARPS>;
}
template <typename T>
RaKernel ra_kernel(bool interleaved, int rotary_dim, int warps) {
  return warps == 1   ? ra_kernel_of<T, 1>(interleaved, rotary_dim)
         : warps == 2 ? ra_kernel_of<T, 2>(interleaved, rotary_dim)
                      : ra_kernel_of<T, 8>(interleaved, rotary_dim);
}

}  // namespace krt

using namespace krt;

// ------------------------------------------------------------------ C ABI
extern "C" size_t krt_rope_append_workspace_size(void) { return kWsHeaderBytes; }

extern "C" int krt_rope_append(const krt_rope_append_args* a, void* stream) {
  const char* name = "krt_rope_append";
  if (!a) return set_error(KRT_ERR_INVALID, "%s: args is NULL", name);
  if (!a->q || !a->k || !a->v || !a->inv_freq || !a->positions || !a->token_seq || !a->block_table || !a->kv_pool ||
      !a->q_out || !a->workspace)
    return set_error(KRT_ERR_INVALID, "%s: a required pointer is NULL", name);
  if (a->num_tokens <= 0 || a->n_heads <= 0 || a->n_kv_heads <= 0)
    return set_error(KRT_ERR_INVALID, "%s: num_tokens and heads must be positive", name);
  if (a->head_dim != kHeadDim) return set_error(KRT_ERR_UNSUPPORTED, "%s: head_dim must be 128", name);
  if (a->n_heads > 4096 || a->n_kv_heads > 4096) return set_error(KRT_ERR_UNSUPPORTED, "%s: too many heads", name);
  if (a->rotary_dim < 2 || a->rotary_dim > kHeadDim || a->rotary_dim % 2 != 0)
    return set_error(KRT_ERR_INVALID, "%s: rotary_dim must be even, 2 to 128", name);
  const int dtype = a->dtype == 0 ? KRT_DTYPE_BFLOAT16 : a->dtype;
  if (dtype != KRT_DTYPE_BFLOAT16 && dtype != KRT_DTYPE_FLOAT32)
    return set_error(KRT_ERR_UNSUPPORTED, "%s: q, k and v are bfloat16 or float32", name);
  const int mult = dtype == KRT_DTYPE_FLOAT32 ? 4 : 8;  // 16 bytes
  if (a->q_stride < (int64_t)a->n_heads * kHeadDim || a->k_stride < (int64_t)a->n_kv_heads * kHeadDim ||
      a->v_stride < (int64_t)a->n_kv_heads * kHeadDim || a->q_out_stride < (int64_t)a->n_heads * kHeadDim ||
      a->q_stride % mult != 0 || a->k_stride % mult != 0 || a->v_stride % mult != 0 || a->q_out_stride % 8 != 0)
    return set_error(KRT_ERR_INVALID, "%s: strides must cover the heads and be multiples of 16 bytes", name);
  if ((reinterpret_cast<uintptr_t>(a->q) & 15) || (reinterpret_cast<uintptr_t>(a->k) & 15) ||
      (reinterpret_cast<uintptr_t>(a->v) & 15) || (reinterpret_cast<uintptr_t>(a->q_out) & 15) ||
      (reinterpret_cast<uintptr_t>(a->kv_pool) & 15) || (reinterpret_cast<uintptr_t>(a->inv_freq) & 7) ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 15))
    return set_error(KRT_ERR_INVALID, "%s: tensors must be 16-byte aligned (inv_freq 8)", name);
  if (a->num_seqs <= 0 || a->block_table_stride <= 0 || a->num_blocks <= 0 || a->tokens_per_block <= 0)
    return set_error(KRT_ERR_INVALID, "%s: paged-cache geometry must be positive", name);
  const int columns = block_table_columns(a->block_table_columns, a->block_table_stride, a->num_seqs);
  if (columns < 0)
    return set_error(KRT_ERR_INVALID, "%s: block_table_columns must lie in 0 .. block_table_stride", name);
  if (!std::isfinite(a->factor)) return set_error(KRT_ERR_INVALID, "%s: factor must be finite", name);
  if (a->workspace_bytes < kWsHeaderBytes)
    return set_error(KRT_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, a->workspace_bytes,
                     (size_t)kWsHeaderBytes);
  // q_out may not lie over q, k or v: a pair's two halves can belong to different
  // threads.  Rows of one pitch may alternate (columns of one wider tensor).
  const uint64_t in_size = dtype == KRT_DTYPE_FLOAT32 ? 4 : 2;
  const uint64_t o0 = reinterpret_cast<uintptr_t>(a->q_out), o_row = (uint64_t)a->n_heads * kHeadDim * 2;
  const uint64_t o_pitch = (uint64_t)a->q_out_stride * 2, o1 = o0 + (a->num_tokens - 1) * o_pitch + o_row;
  const struct { const void* p; int64_t stride; int heads; } ins[3] = {
      {a->q, a->q_stride, a->n_heads}, {a->k, a->k_stride, a->n_kv_heads}, {a->v, a->v_stride, a->n_kv_heads}};
  for (const auto& in : ins) {
    const uint64_t row = (uint64_t)in.heads * kHeadDim * in_size, pitch = (uint64_t)in.stride * in_size;
    const uint64_t i0 = reinterpret_cast<uintptr_t>(in.p), i1 = i0 + (a->num_tokens - 1) * pitch + row;
    if (o0 >= i1 || i0 >= o1) continue;
    // bytes from the start of an input row to that of the first q_out row behind it
    const uint64_t ahead = o0 >= i0 ? (o0 - i0) % pitch : (pitch - (i0 - o0) % pitch) % pitch;
    if (pitch == o_pitch && ahead >= row && ahead + o_row <= pitch) continue;
    return set_error(KRT_ERR_INVALID, "%s: q_out overlaps an input", name);
  }
  RaParams p;
  std::memset(&p, 0, sizeof(p));
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.inv_freq = a->inv_freq;
  p.positions = a->positions;
  p.cache_index = a->cache_index;
  p.token_seq = a->token_seq;
  p.block_table = a->block_table;
  p.pool = static_cast<__nv_bfloat16*>(a->kv_pool);
  p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
  p.status = static_cast<int*>(a->workspace);
  p.q_stride = a->q_stride;
  p.k_stride = a->k_stride;
  p.v_stride = a->v_stride;
  p.q_out_stride = a->q_out_stride;
  p.num_tokens = a->num_tokens;
  p.n_heads = a->n_heads;
  p.n_kv_heads = a->n_kv_heads;
  p.rotary_dim = a->rotary_dim;
  const bool interleaved = a->interleaved != 0;
  p.num_seqs = a->num_seqs;
  p.bt_stride = a->block_table_stride;
  p.bt_columns = columns;
  p.num_blocks = a->num_blocks;
  p.tokens_per_block = a->tokens_per_block;
  p.factor = a->factor == 0.f ? 1.f : a->factor;
  // Eight warps per token while the tokens are few, then two, or one where a
  // token has little work.  Measured (us), eight : two : one: 40 heads (bf16),
  // 300 tokens 3.5 : 4.8 : 7.4, 1500 8.8 : 8.4 : 9.8, 16000 87 : 66 : 68;
  // 9 heads (fp32), 300 2.7 : 3.1 : 3.7, 1500 5.9 : 4.5 : 4.6, 16000 55 : 29 : 25.
  const int sms = device_sm_count(), heads = a->n_heads + 2 * a->n_kv_heads;
  const int warps = a->num_tokens < 4 * sms ? 8 : heads >= 32 || a->num_tokens < 16 * sms ? 2 : 1;
  cudaLaunchConfig_t cfg = {};
  const int per_cta = 8 / warps;
  cfg.gridDim = dim3(((unsigned)a->num_tokens + per_cta - 1) / per_cta, 1, 1);
  cfg.blockDim = dim3(kRaThreads, 1, 1);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  RaKernel kern = dtype == KRT_DTYPE_FLOAT32 ? ra_kernel<float>(interleaved, p.rotary_dim, warps)
                                             : ra_kernel<__nv_bfloat16>(interleaved, p.rotary_dim, warps);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return cuda_error(e, name);
  return clear_error();
}
