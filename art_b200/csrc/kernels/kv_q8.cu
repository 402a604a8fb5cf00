// Writing a paged cache that is held in 8 bits, and reading it back (numbers and layout: kv_q8.cuh).
//
// Write.  The rows of a call that fall in one block and kv head are quantised together: with a their largest |value| and
// 2^e the least power of two with a <= MAX 2^e,
//     s' = 2^e                if a row at the block's first place is among them (the block starts anew),
//     s' = max(s, 2^e)        otherwise, and where that raises the scale, c' = round(c s / s') for the block's other codes,
//     c  = round(x / s').
// For e4m3 a raised scale only lowers the exponents of the codes, exact until they become subnormal.  A value that is not
// finite has no code: it makes the scale NaN, which every read of that block and head shows until the block starts anew.
//
// Bound by bytes, 2 in and 1 out per value, and by latency where a decode step writes one token per sequence.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "host_utils.h"
#include "kv_q8.cuh"

namespace artb {

// A warp per (run of rows, kv head, keys or values).  A run is a stretch of neighbouring rows whose slots are neighbours in
// one block; the warps of a CTA look for runs that begin among its ROWS rows and follow them to their ends.
// A lane holds 8 values of a row: HD / 8 lanes to a row, 16 rows at a time in registers.
constexpr int KW_BATCH = 16;

template <int KIND, int HD, int ROWS>
__global__ void __launch_bounds__(128)
kv_write_q8_kernel(const __nv_bfloat16* __restrict__ qkv, int ld, int k_col, int v_col, const int* __restrict__ slot,
                   uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale, int M, int Hkv, int block_size,
                   long num_blocks, int* status) {
  constexpr int LPR = HD / 8, RPI = 32 / LPR, ITERS = KW_BATCH / RPI;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, part = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (part >= 2 * Hkv) return;
  const bool is_v = part >= Hkv;
  const int h = is_v ? part - Hkv : part;
  const __nv_bfloat16* x = qkv + (is_v ? v_col : k_col) + h * HD;
  uint8_t* cache = is_v ? v_cache : k_cache;
  float* scales = is_v ? v_scale : k_scale;
  const int row0 = blockIdx.x * ROWS, sub = lane / LPR, c = (lane % LPR) * 8;

  bool starts = false;
  if (lane < ROWS && row0 + lane < M) {
    const int r = row0 + lane, s = slot[r];
    starts = s >= 0 && (r == 0 || s % block_size == 0 || slot[r - 1] != s - 1);
  }
  for (uint32_t todo = __ballot_sync(0xffffffffu, starts); todo; todo &= todo - 1) {
    const int r0 = row0 + __ffs(todo) - 1, s0 = slot[r0];
    if (!q8_index_ok(s0, num_blocks * block_size, status)) continue;
    const long block = s0 / block_size;
    const int at = s0 - static_cast<int>(block) * block_size, most = min(block_size - at, M - r0);
    int n = 1;
    while (n < most) {                     // the run's length: 32 rows at a time
      const int r = r0 + n + lane;
      const uint32_t on = __ballot_sync(0xffffffffu, n + lane < most && slot[min(r, M - 1)] == s0 + n + lane);
      const int more = on == 0xffffffffu ? 32 : __ffs(~on) - 1;
      n += more;
      if (more < 32) break;
    }

    uint4 raw[ITERS];
    auto load = [&](int first) {
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        const int r = first + i * RPI + sub;
        raw[i] = r < n ? *reinterpret_cast<const uint4*>(x + static_cast<size_t>(r0 + r) * ld + c) : make_uint4(0, 0, 0, 0);
      }
    };
    // largest |value|: the bits of bf16 magnitudes order like integers, two at a time
    uint32_t top = 0;
    for (int first = 0; first < n; first += KW_BATCH) {
      load(first);
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        top = __vmaxu2(top, raw[i].x & 0x7fff7fffu);
        top = __vmaxu2(top, raw[i].y & 0x7fff7fffu);
        top = __vmaxu2(top, raw[i].z & 0x7fff7fffu);
        top = __vmaxu2(top, raw[i].w & 0x7fff7fffu);
      }
    }
    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));

    float* sp = scales + block * Hkv + h;
    const float held = *sp, mine = q8_pow2(q8_exponent<KIND>(top < 0x7f80u ? top << 16 : 0u));
    const bool anew = at == 0, bad = top >= 0x7f80u || (!anew && !(held <= 3.0e38f));       // not finite
    const float to = anew ? mine : fmaxf(held, mine), inv = 1.f / to;                       // exact: a power of two
    uint8_t* codes = cache + (block * Hkv + h) * block_size * HD;
    __syncwarp();
    if (lane == 0) *sp = bad ? __int_as_float(0x7fc00000) : to;
    if (!bad && !anew && to > held) {
      const float down = held * inv;
      for (int v = lane; v < block_size * (HD / 4); v += 32) {
        const int place = v / (HD / 4);
        if (place >= at && place < at + n) continue;
        uint32_t* p = reinterpret_cast<uint32_t*>(codes) + v;
        float f[4];
        q8_decode4<KIND>(*p, f);
        *p = q8_encode4<KIND>(f[0] * down, f[1] * down, f[2] * down, f[3] * down);
      }
    }
    for (int first = 0; first < n; first += KW_BATCH) {
      if (n > KW_BATCH) load(first);       // else the only batch is still in registers
#pragma unroll
      for (int i = 0; i < ITERS; ++i) {
        const int r = first + i * RPI + sub;
        if (r >= n) continue;
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[2 * j] = __uint_as_float(w[j] << 16) * inv;
          f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u) * inv;
        }
        uint2 out = make_uint2(q8_encode4<KIND>(f[0], f[1], f[2], f[3]), q8_encode4<KIND>(f[4], f[5], f[6], f[7]));
        if (bad) out = make_uint2(0, 0);
        *reinterpret_cast<uint2*>(codes + static_cast<size_t>(at + r) * HD + c) = out;
      }
    }
  }
}

// The cached keys and values at a list of slots -> k | v columns of dst [n, ld], as bf16 (exact: a code has at most 8 bits);
// rows with a negative slot become zeros.  A thread takes 16 codes.  Bound by bytes, 1 in and 2 out per value.
template <int KIND>
__global__ void __launch_bounds__(256)
kv_rows_q8_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const float* __restrict__ k_scale,
                  const float* __restrict__ v_scale, const int* __restrict__ slot, long n, __nv_bfloat16* __restrict__ dst, int ld,
                  int k_col, int v_col, int Hkv, int hd, int block_size, long num_blocks, int* status) {
  const int half = Hkv * hd / 16, vec = 2 * half;
  const long total = n * vec;
  for (long i = blockIdx.x * static_cast<long>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<long>(gridDim.x) * blockDim.x) {
    const long r = i / vec;
    int u = static_cast<int>(i - r * vec);
    const bool is_v = u >= half;
    u -= is_v ? half : 0;
    const int h = u * 16 / hd, d = u * 16 - h * hd, s = slot[r];
    uint4 raw = make_uint4(0, 0, 0, 0);
    float scale = 0.f;
    if (s >= 0 && q8_index_ok(s, num_blocks * block_size, status)) {
      const long head = s / block_size * static_cast<long>(Hkv) + h;
      raw = *reinterpret_cast<const uint4*>((is_v ? v_cache : k_cache) + (head * block_size + s % block_size) * hd + d);
      scale = (is_v ? v_scale : k_scale)[head];
    }
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[4];
      q8_decode4<KIND>(w[j], f);
      const __nv_bfloat162 lo = __floats2bfloat162_rn(f[0] * scale, f[1] * scale), hi = __floats2bfloat162_rn(f[2] * scale, f[3] * scale);
      o[2 * j] = *reinterpret_cast<const uint32_t*>(&lo);
      o[2 * j + 1] = *reinterpret_cast<const uint32_t*>(&hi);
    }
    uint4* to = reinterpret_cast<uint4*>(dst + r * ld + (is_v ? v_col : k_col) + h * hd + d);
    to[0] = make_uint4(o[0], o[1], o[2], o[3]);
    to[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

}  // namespace artb

using namespace artb;

// qkv [M, ld] bf16 with keys at k_col and values at v_col; slot [M]: block * block_size + place, < 0: the row is not written.
// A slot beyond the cache is not written either and reported through `status`.
ARTB_EXPORT int artb_kv_write_q8(const void* qkv, int ld, int k_col, int v_col, const int* slot, void* k_cache, void* v_cache,
                                 float* k_scale, float* v_scale, int M, int Hkv, int hd, int block_size, long num_blocks,
                                 int kind, int* status, cudaStream_t st) {
  if (M <= 0) return 0;
  if (Hkv <= 0 || block_size < 16 || (block_size & 15) || (ld & 7) || (k_col & 7) || (v_col & 7)) return ERR_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) return ERR_BAD_ALIGN;
#define ARTB_KW(KIND_, HD_)                                                                                                  \
  if (kind == KIND_ && hd == HD_) {                                                                                          \
    auto go = [&](auto kern, int rows) {                                                                                     \
      return static_cast<int>(launch_kernel(kern, dim3((M + rows - 1) / rows, (2 * Hkv + 3) / 4), dim3(128), 0, st,          \
                                            (const __nv_bfloat16*)qkv, ld, k_col, v_col, slot, (uint8_t*)k_cache,            \
                                            (uint8_t*)v_cache, k_scale, v_scale, M, Hkv, block_size, num_blocks, status));   \
    };                                                                                                                       \
    return go(kv_write_q8_kernel<KIND_, HD_, 1>, 1);                                                                         \
  }
  ARTB_KW(Q8_E4M3, 128) ARTB_KW(Q8_E4M3, 64) ARTB_KW(Q8_E4M3, 32)
  ARTB_KW(Q8_INT8, 128) ARTB_KW(Q8_INT8, 64) ARTB_KW(Q8_INT8, 32)
#undef ARTB_KW
  return ERR_BAD_SHAPE;
}

ARTB_EXPORT int artb_kv_rows_q8(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                                const int* slot, int n, void* dst, int ld, int k_col, int v_col, int Hkv, int hd, int block_size,
                                long num_blocks, int kind, int* status, cudaStream_t st) {
  if (n <= 0) return 0;
  if (Hkv <= 0 || hd < 16 || (hd & 15) || block_size < 1 || (ld & 7) || (k_col & 7) || (v_col & 7)) return ERR_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) return ERR_BAD_ALIGN;
  long blocks = (static_cast<long>(n) * (Hkv * hd / 8) + 255) / 256;
  if (blocks > 148L * 16) blocks = 148L * 16;
  auto go = [&](auto kern) {
    kern<<<(unsigned)blocks, 256, 0, st>>>((const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, slot, n,
                                           (__nv_bfloat16*)dst, ld, k_col, v_col, Hkv, hd, block_size, num_blocks, status);
    return (int)cudaGetLastError();
  };
  if (kind == Q8_E4M3) return go(kv_rows_q8_kernel<Q8_E4M3>);
  if (kind == Q8_INT8) return go(kv_rows_q8_kernel<Q8_INT8>);
  return ERR_BAD_SHAPE;
}
