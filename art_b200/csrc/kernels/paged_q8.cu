// Decode attention over a paged cache held in 8 bits (numbers and layout: kv_q8.cuh): one new token per sequence,
//     o_h = sum_j softmax_j(q_h . k_j / sqrt(hd)) v_j,   j < ctx_len,   k_j, v_j = code * scale of the block and kv head.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "host_utils.h"
#include "kv_q8.cuh"

namespace artb {

// A CTA per (sequence, query head); each warp takes every fourth key, a lane HD / 32 of its values.
template <int KIND, int HD>
__global__ void __launch_bounds__(128)
paged_decode_q8_kernel(const __nv_bfloat16* __restrict__ q, int ldq, const uint8_t* __restrict__ k_cache,
                       const uint8_t* __restrict__ v_cache, const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                       const int* __restrict__ block_table, int max_blocks, const int* __restrict__ ctx_len, int block_size,
                       int Hq, int Hkv, __nv_bfloat16* __restrict__ out, int ldo, float scale_log2, long num_blocks, int* status) {
  constexpr int PER = HD / 32;
  __shared__ float s_acc[4][HD], s_m[4], s_l[4];
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.x, head = blockIdx.y, kvh = head / (Hq / Hkv), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int len = ctx_len[seq];
  if (len > static_cast<long>(max_blocks) * block_size) {
    if (status) atomicMax(status, ST_BOUNDS);
    len = max_blocks * block_size;
  }
  float qv[PER], acc[PER], m = -INFINITY, l = 0.f;
  for (int i = 0; i < PER; ++i) {
    qv[i] = __bfloat162float(q[static_cast<size_t>(seq) * ldq + head * HD + lane * PER + i]) * scale_log2;
    acc[i] = 0.f;
  }
  auto value = [](const uint8_t* p, int i) {
    float f[4];
    q8_decode4<KIND>(p[i], f);
    return f[0];
  };
  for (int j = warp; j < len; j += 4) {
    const int blk = block_table[static_cast<size_t>(seq) * max_blocks + j / block_size];
    if (!q8_index_ok(blk, num_blocks, status)) continue;
    const size_t at = static_cast<size_t>(blk) * Hkv + kvh, row = (at * block_size + j % block_size) * HD + lane * PER;
    float s = 0.f;
    for (int i = 0; i < PER; ++i) s += qv[i] * value(k_cache + row, i);
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= k_scale[at];
    const float mn = fmaxf(m, s), c = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * c + p;
    for (int i = 0; i < PER; ++i) acc[i] = acc[i] * c + p * v_scale[at] * value(v_cache + row, i);
  }
  for (int i = 0; i < PER; ++i) s_acc[warp][lane * PER + i] = acc[i];
  s_m[warp] = m;
  s_l[warp] = l;
  __syncthreads();
  const float mm = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  for (int d = threadIdx.x; d < HD; d += 128) {
    float o = 0.f, sum = 0.f;
    for (int w = 0; w < 4 && len > 0; ++w) {
      const float c = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - mm);
      o += c * s_acc[w][d];
      sum += c * s_l[w];
    }
    out[static_cast<size_t>(seq) * ldo + head * HD + d] = __float2bfloat16(len > 0 ? o / sum : 0.f);
  }
}

}  // namespace artb

using namespace artb;

ARTB_EXPORT int artb_paged_decode_q8_bytes(int num_seqs, int Hq, int Hkv, int hd) {
  (void)hd;
  return num_seqs <= 0 || Hkv <= 0 || Hq % Hkv ? 0 : 16;
}

ARTB_EXPORT int artb_paged_decode_q8(const void* q, int ldq, const void* k_cache, const void* v_cache, const float* k_scale,
                                     const float* v_scale, const int* block_table, int max_blocks, const int* ctx_len,
                                     int block_size, int num_seqs, int Hq, int Hkv, int hd, void* out, int ldo, void* ws,
                                     long num_blocks, int kind, int* status, cudaStream_t st) {
  if (num_seqs <= 0) return 0;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 16 || block_size < 16 || (block_size & 15) || !ws) return ERR_BAD_SHAPE;
  const float scale_log2 = 1.4426950408889634f / sqrtf((float)hd);
#define ARTB_PQ(KIND_, HD_)                                                                                                   \
  if (kind == KIND_ && hd == HD_)                                                                                             \
    return static_cast<int>(launch_kernel(paged_decode_q8_kernel<KIND_, HD_>, dim3(num_seqs, Hq), dim3(128), 0, st,           \
                                          (const __nv_bfloat16*)q, ldq, (const uint8_t*)k_cache, (const uint8_t*)v_cache,     \
                                          k_scale, v_scale, block_table, max_blocks, ctx_len, block_size, Hq, Hkv,            \
                                          (__nv_bfloat16*)out, ldo, scale_log2, num_blocks, status));
  ARTB_PQ(Q8_E4M3, 128) ARTB_PQ(Q8_E4M3, 64) ARTB_PQ(Q8_E4M3, 32)
  ARTB_PQ(Q8_INT8, 128) ARTB_PQ(Q8_INT8, 64) ARTB_PQ(Q8_INT8, 32)
#undef ARTB_PQ
  return ERR_BAD_SHAPE;
}
