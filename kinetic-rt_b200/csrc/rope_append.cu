// Rotary positions of q and k, and k and v appended to the paged KV cache.
//
// For token t at position p and pair i of the first R dims of a q or k head,
//   angle = p * inv_freq[i]
//   (a, b) -> (a cos - b sin, b cos + a sin) * factor
// where (a, b) are dims (2i, 2i + 1) (interleaved) or (i, i + R / 2) (halves);
// dims R .. 127 pass through.  q goes to q_out, k and v to the slot of the
// token's cache index (token layout [K | V][kv_head][128] bf16).
//
// The kernel reads and writes every element once and is bound by HBM.  A CTA
// takes a few tokens: its threads first compute each token's R / 2 cosines and
// sines into shared memory, shared by all heads.  The angle is taken in fp64
// turns (p * inv_freq / 2 pi) and reduced to its fraction before the fp32
// sine: at position 10^6 an fp32 angle would be off by 0.06.  This costs R / 2
// fp64 products a token, against R * heads products, and saves the table that
// limits the position.  Then unit u of a head is two 8-element vectors that a
// thread loads, rotates and stores (16-byte accesses): the two partners of a
// half-split rotation, or two vectors of interleaved pairs.
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
constexpr int kRaMaxTokens = 4;  // tokens per CTA at most
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
  int num_tokens, n_heads, n_kv_heads, rotary_dim, interleaved;
  int num_seqs, bt_stride, num_blocks, tokens_per_block;
  int tokens_per_cta;
  float factor;
};

__device__ __forceinline__ void ra_load8(const float* src, float* x) {
  const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void ra_load8(const __nv_bfloat16* src, float* x) {
  const uint4 v = *reinterpret_cast<const uint4*>(src);
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(p[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ float ra_load1(const float* src) { return *src; }
__device__ __forceinline__ float ra_load1(const __nv_bfloat16* src) { return __bfloat162float(*src); }

__device__ __forceinline__ void ra_store8(__nv_bfloat16* dst, const float* x) {
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                              pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

template <typename T>
__global__ void __launch_bounds__(kRaThreads) rope_append_kernel(const RaParams p) {
  __shared__ float2 cs[kRaMaxTokens][64];
  __shared__ long long slot[kRaMaxTokens];  // pool slot, -1: k and v are not written, -2: the token is skipped
  const int t0 = blockIdx.x * p.tokens_per_cta;
  const int nt = min(p.tokens_per_cta, p.num_tokens - t0);
  const int half = p.rotary_dim / 2;
  pdl_wait();  // q, k, v come from the previous kernel
  pdl_launch_dependents();
  if (threadIdx.x < nt) {
    const int t = t0 + threadIdx.x;
    const int seq = p.token_seq[t];
    long long s = -1;
    if (seq < 0) {
      s = -2;
    } else {
      const int at = p.cache_index ? p.cache_index[t] : p.positions[t];
      const int col = at >= 0 ? at / p.tokens_per_block : -1;
      if (seq < p.num_seqs && col >= 0 && col < p.bt_stride) {
        const int blk = p.block_table[(size_t)seq * p.bt_stride + col];
        if (blk >= 0 && blk < p.num_blocks) s = (long long)blk * p.tokens_per_block + at % p.tokens_per_block;
      }
      if (s < 0) atomicOr(p.status, kStatusBadBlock);
    }
    slot[threadIdx.x] = s;
  }
  for (int i = threadIdx.x; i < nt * half; i += kRaThreads) {
    const int t = i / half, f = i % half;
    const double turns = (double)p.positions[t0 + t] * (p.inv_freq[f] * 0.15915494309189535);  // / 2 pi
    float sn, c;
    sincospif(2.f * (float)(turns - floor(turns)), &sn, &c);
    cs[t][f] = make_float2(c * p.factor, sn * p.factor);
  }
  __syncthreads();

  const int H = p.n_heads, K = p.n_kv_heads;
  const int per_token = (H + 2 * K) * kRaUnits;
  const int vec_r = p.rotary_dim / 8, pairs_r = p.rotary_dim / 16;  // rotated vectors; half-split vector pairs
  const bool aligned = p.rotary_dim % 16 == 0;
  for (int i = threadIdx.x; i < nt * per_token; i += kRaThreads) {
    const int tl = i / per_token, r = i % per_token;
    const int head = r / kRaUnits, u = r % kRaUnits;
    const long long s = slot[tl];
    if (s == -2) continue;
    const size_t t = (size_t)(t0 + tl);
    const T* src;
    __nv_bfloat16* dst;
    if (head < H) {
      src = static_cast<const T*>(p.q) + t * p.q_stride + head * kHeadDim;
      dst = p.q_out + t * p.q_out_stride + head * kHeadDim;
    } else {
      if (s < 0) continue;
      const bool is_v = head >= H + K;
      const int kh = head - H - (is_v ? K : 0);
      src = is_v ? static_cast<const T*>(p.v) + t * p.v_stride + kh * kHeadDim
                 : static_cast<const T*>(p.k) + t * p.k_stride + kh * kHeadDim;
      dst = p.pool + ((size_t)s * 2 * K + (is_v ? K : 0) + kh) * kHeadDim;
    }
    const bool rot = head < H + K;
    // the unit's two vectors
    int va = u, vb = u + 8;
    if (rot && !p.interleaved && aligned) {
      va = u < pairs_r ? u : vec_r + (u - pairs_r);
      vb = u < pairs_r ? u + pairs_r : va + (8 - pairs_r);
    }
    float a[8], b[8];
    ra_load8(src + 8 * va, a);
    ra_load8(src + 8 * vb, b);
    if (rot) {
      const float2* cst = cs[tl];
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (8 * va + 2 * j < p.rotary_dim) {
            const float2 w = cst[4 * va + j];
            const float x = a[2 * j], y = a[2 * j + 1];
            a[2 * j] = x * w.x - y * w.y;
            a[2 * j + 1] = y * w.x + x * w.y;
          }
          if (8 * vb + 2 * j < p.rotary_dim) {
            const float2 w = cst[4 * vb + j];
            const float x = b[2 * j], y = b[2 * j + 1];
            b[2 * j] = x * w.x - y * w.y;
            b[2 * j + 1] = y * w.x + x * w.y;
          }
        }
      } else if (aligned) {
        if (u < pairs_r) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 w = cst[8 * va + j];
            const float x = a[j], y = b[j];
            a[j] = x * w.x - y * w.y;
            b[j] = y * w.x + x * w.y;
          }
        }
      } else {
        // partners do not fall on vectors: fetch each one by itself
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int da = 8 * va + j, db = 8 * vb + j;
          if (da < p.rotary_dim) {
            const int f = da < half ? da : da - half;
            const float2 w = cst[f];
            const float y = ra_load1(src + (da < half ? da + half : f));
            a[j] = da < half ? a[j] * w.x - y * w.y : a[j] * w.x + y * w.y;
          }
          if (db < p.rotary_dim) {
            const int f = db < half ? db : db - half;
            const float2 w = cst[f];
            const float y = ra_load1(src + (db < half ? db + half : f));
            b[j] = db < half ? b[j] * w.x - y * w.y : b[j] * w.x + y * w.y;
          }
        }
      }
    }
    ra_store8(dst + 8 * va, a);
    ra_store8(dst + 8 * vb, b);
  }
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
  if (!std::isfinite(a->factor)) return set_error(KRT_ERR_INVALID, "%s: factor must be finite", name);
  if (a->workspace_bytes < kWsHeaderBytes)
    return set_error(KRT_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, a->workspace_bytes,
                     (size_t)kWsHeaderBytes);
  // q_out may not lie over q, k or v: a pair's two halves can belong to different threads
  const size_t in_size = dtype == KRT_DTYPE_FLOAT32 ? 4 : 2;
  const uintptr_t o0 = reinterpret_cast<uintptr_t>(a->q_out);
  const uintptr_t o1 = o0 + ((size_t)(a->num_tokens - 1) * a->q_out_stride + (size_t)a->n_heads * kHeadDim) * 2;
  const struct { const void* p; int64_t stride; int heads; } ins[3] = {
      {a->q, a->q_stride, a->n_heads}, {a->k, a->k_stride, a->n_kv_heads}, {a->v, a->v_stride, a->n_kv_heads}};
  for (const auto& in : ins) {
    const uintptr_t i0 = reinterpret_cast<uintptr_t>(in.p);
    const uintptr_t i1 = i0 + ((size_t)(a->num_tokens - 1) * in.stride + (size_t)in.heads * kHeadDim) * in_size;
    if (o0 < i1 && i0 < o1) return set_error(KRT_ERR_INVALID, "%s: q_out overlaps an input", name);
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
  p.interleaved = a->interleaved != 0;
  p.num_seqs = a->num_seqs;
  p.bt_stride = a->block_table_stride;
  p.num_blocks = a->num_blocks;
  p.tokens_per_block = a->tokens_per_block;
  p.factor = a->factor == 0.f ? 1.f : a->factor;
  p.tokens_per_cta = a->num_tokens >= kRaMaxTokens * 2 * device_sm_count() ? kRaMaxTokens : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a->num_tokens + p.tokens_per_cta - 1) / p.tokens_per_cta), 1, 1);
  cfg.blockDim = dim3(kRaThreads, 1, 1);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = dtype == KRT_DTYPE_FLOAT32 ? cudaLaunchKernelEx(&cfg, rope_append_kernel<float>, p)
                                             : cudaLaunchKernelEx(&cfg, rope_append_kernel<__nv_bfloat16>, p);
  if (e != cudaSuccess) return cuda_error(e, name);
  return clear_error();
}
