// Numbers of a cache of keys and values held in 8 bits.
//
// Codes [blocks, Hkv, block_size, hd], e4m3 or int8, and one fp32 scale per block and kv head [blocks, Hkv]: value = code *
// scale.  The codes of a block and head are block_size * hd bytes in a row.  Scales are powers of two, so that x / scale is
// exact in fp32 and every code is one rounding of its value; the least such scale costs up to one bit of the 7 that int8 has
// and nothing of e4m3's 4, whose spacing goes with the value.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "ptx_sm100.cuh"

namespace artb {

enum Q8Kind : int { Q8_E4M3 = 0, Q8_INT8 = 1 };

// Arguments of the launches, as one block of memory each (ops/kv_q8.py packs them).
struct KvRowsArgs {               // rows [n, ld] bf16 with keys at k_col and values at v_col, their slots, and the cache
  int* status;
  void* rows;
  const int* slot;
  void *k_cache, *v_cache;
  float *k_scale, *v_scale;
  long num_blocks;
  int n, ld, k_col, v_col, Hkv, hd, block_size, kind;
};
struct PagedDecodeArgs {
  int* status;
  const void *q, *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int *block_table, *ctx_len;
  void *out, *ws;
  long num_blocks;
  int num_seqs, ldq, ldo, Hq, Hkv, hd, block_size, max_blocks, kind;
};

constexpr int Q8_LEAST_EXP = -126;       // the smallest scale is a normal fp32 number

// Index checks of these kernels are always on: slots and block tables come from memory, and a compare costs nothing beside
// the access it guards.
__device__ __forceinline__ bool q8_index_ok(long long i, long long n, int* status) {
  if (i < 0 || i >= n) {
    if (status) atomicMax(status, ST_BOUNDS);
    return false;
  }
  return true;
}

// Whether a slot, negative ones too, lies in the block of `size` tokens whose first slot is `first`, a multiple of size below 2^31.
__device__ __forceinline__ bool q8_in_block(int slot, int first, int size) {
  return static_cast<uint32_t>(slot) - static_cast<uint32_t>(first) < static_cast<uint32_t>(size);
}

__device__ __forceinline__ float q8_pow2(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127

// Exponent of the least power of two s with amax <= MAX * s (448 = 1.75 * 2^8, 127 = 1.984375 * 2^6), from the bits of a
// finite fp32 amax.  A subnormal amax is below every scale's range.
template <int KIND>
__device__ __forceinline__ int q8_exponent(uint32_t amax_bits) {
  constexpr int TOP = KIND == Q8_E4M3 ? 8 : 6;
  constexpr uint32_t FRACTION = KIND == Q8_E4M3 ? 0x600000u : 0x7e0000u;
  const int e = static_cast<int>(amax_bits >> 23) - 127 - TOP + ((amax_bits & 0x7fffffu) > FRACTION);
  return e < Q8_LEAST_EXP ? Q8_LEAST_EXP : e;
}

// Four values, already divided by their scale and so within the codes' range, to four codes: nearest, ties to even.
template <int KIND>
__device__ __forceinline__ uint32_t q8_encode4(float a, float b, float c, float d) {
  if (KIND == Q8_E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  // beside 1.5 * 2^23 the last bit of a float is 1: the sum is rounded to a whole number, whose low byte is the code
  constexpr float ONES = 12582912.f;
  const uint32_t x = __float_as_uint(a + ONES), y = __float_as_uint(b + ONES), z = __float_as_uint(c + ONES), w = __float_as_uint(d + ONES);
  return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

// Four codes to floats.
template <int KIND>
__device__ __forceinline__ void q8_decode4(uint32_t w, float (&f)[4]) {
  if (KIND == Q8_E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * i)), __NV_E4M3);
      const float2 v = __half22float2(__half2(h));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  }
}

// What becomes of the scale of a block and head when rows whose largest |value| has the bf16 bits `top` are written to it.
struct Q8Scale {
  float to;        // the scale, NaN where a value is not finite: that stays until the block starts anew
  float inv;       // 1 / to (exact: a power of two), NaN where the codes of the rows are to be zeros
  float down;      // what the codes of the block's other rows are multiplied by, 1: they stay
};

// `held`: the scale so far; `anew`: a row at the block's first place is among them.
template <int KIND>
__device__ __forceinline__ Q8Scale q8_new_scale(uint32_t top, float held, bool anew) {
  const float mine = q8_pow2(q8_exponent<KIND>(top < 0x7f80u ? top << 16 : 0u)), none = __int_as_float(0x7fc00000);
  if (top >= 0x7f80u || (!anew && !(held <= 3.0e38f))) return Q8Scale{none, none, 1.f};
  const float to = anew ? mine : fmaxf(held, mine), inv = 1.f / to;
  return Q8Scale{to, inv, !anew && to > held ? held * inv : 1.f};
}

// 16 codes times `down`, rounded once more; piece v of a block and head.
template <int KIND>
__device__ __forceinline__ uint4 q8_lower(uint4 old, float down) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&old);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float f[4];
    q8_decode4<KIND>(w[j], f);
    w[j] = q8_encode4<KIND>(f[0] * down, f[1] * down, f[2] * down, f[3] * down);
  }
  return old;
}

}  // namespace artb
