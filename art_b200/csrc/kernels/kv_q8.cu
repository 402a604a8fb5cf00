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

// A run is a stretch of neighbouring rows whose slots are neighbours in one block.  A warp takes a run's part for one kv head, of
// keys or of values: it looks for the runs that begin among its ROWS rows and follows them to their ends.  A lane holds 8 values
// of a row, HD / 8 lanes to a row: of up to 16 rows in registers, of longer runs in its own places of shared memory, where 32 rows
// are under way at a time; runs longer than that are read twice.  (14,000 rows in blocks of 32: 17.7 us, 19.1 with 16 rows of 32 in
// registers at a time.  Shared memory for runs of 16 too takes 0.8 us more than registers, of 11.8: 14,760 rows in blocks of 16.)
constexpr int KW_FIT = 32;
constexpr int KW_STEP = 256;             // rows of a call whose warps take a row each
template <int KIND, int HD>
struct KwRun {
  static constexpr int LPR = HD / 8, RPI = 32 / LPR, STEP = 16 / RPI;     // pieces of a lane per 16 rows
  static constexpr int PLACE = LPR * 16;                                  // bytes of a row

  const __nv_bfloat16* x;      // of the first row
  int ld, n, at, block_size;   // rows, the first one's place in the block
  uint8_t* codes;              // of the block
  float* sp;
  uint32_t top = 0;
  float inv;

  static __device__ __forceinline__ int sub() { return (threadIdx.x & 31) / LPR; }
  static __device__ __forceinline__ int col() { return (threadIdx.x & 31) % LPR * 8; }

  // largest |value|: the bits of bf16 magnitudes order like integers, two at a time
  __device__ __forceinline__ void look(const uint4& v) {
    top = __vmaxu2(top, v.x & 0x7fff7fffu);
    top = __vmaxu2(top, v.y & 0x7fff7fffu);
    top = __vmaxu2(top, v.z & 0x7fff7fffu);
    top = __vmaxu2(top, v.w & 0x7fff7fffu);
  }

  // The block's new scale from the one that all have read before; `tops`: a place for each of TEAM warps that share the run.
  template <int TEAM>
  __device__ __forceinline__ void rescale(float held, uint32_t* tops) {
    const int thread = TEAM > 1 ? threadIdx.x : threadIdx.x & 31;
    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
    if (TEAM > 1) {
      if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < TEAM; ++w) top = max(top, tops[w]);
    } else {
      __syncwarp();
    }
    const Q8Scale scale = q8_new_scale<KIND>(top, held, at == 0);
    inv = scale.inv;
    if (thread == 0) *sp = scale.to;
    if (scale.down != 1.f) {
      for (int v = thread; v < block_size * (HD / 16); v += TEAM * 32) {
        if (v / (HD / 16) >= at && v / (HD / 16) < at + n) continue;
        uint4* p = reinterpret_cast<uint4*>(codes) + v;
        *p = q8_lower<KIND>(*p, scale.down);
      }
    }
  }

  __device__ __forceinline__ void put(const uint4& v, int row) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = __uint_as_float(w[j] << 16) * inv;
      f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u) * inv;
    }
    uint2 out = make_uint2(q8_encode4<KIND>(f[0], f[1], f[2], f[3]), q8_encode4<KIND>(f[4], f[5], f[6], f[7]));
    if (isnan(inv)) out = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(codes + static_cast<size_t>(at + row) * HD + col()) = out;
  }

  // Up to ITERS * RPI rows from `lo` on, of each of TEAM warps; FULL: as many.
  template <int ITERS, bool FULL, int TEAM = 1>
  __device__ __forceinline__ void held(uint32_t* tops = nullptr, int lo = 0) {
    const float before = __ldcg(sp);
    uint4 raw[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      const int r = lo + i * RPI + sub();
      raw[i] = FULL || r < n ? *reinterpret_cast<const uint4*>(x + static_cast<size_t>(r) * ld + col()) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < ITERS; ++i) look(raw[i]);
    rescale<TEAM>(before, tops);
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
      if (FULL || lo + i * RPI + sub() < n) put(raw[i], lo + i * RPI + sub());
  }

  template <class F>
  __device__ __forceinline__ void pieces(int rows, F f) const {           // of this lane: the place in `room`, the row
#pragma unroll 1
    for (int b = 0; b < rows; b += 16) {
#pragma unroll
      for (int i = 0; i < STEP; ++i)
        if (b + i * RPI + sub() < rows) f(b * LPR + i * 32 + static_cast<int>(threadIdx.x & 31), b + i * RPI + sub());
    }
  }

  // TEAM warps share the rows, FIT of them each in `room` at a time
  template <int TEAM, int FIT>
  __device__ __forceinline__ void staged(uint4* room, uint32_t* tops) {
    const float before = __ldcg(sp);
    const int share = TEAM > 1 ? (n + 16 * TEAM - 1) / (16 * TEAM) * 16 : n;
    if (TEAM > 1 && share == 16) return held<STEP, false, TEAM>(tops, (threadIdx.x >> 5) * 16);
    const int lo = TEAM > 1 ? static_cast<int>(threadIdx.x >> 5) * share : 0, hi = min(n, lo + share);
    auto bring = [&](int first, int rows) {
      pieces(rows, [&](int place, int r) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(room + place)),
                     "l"(x + static_cast<size_t>(first + r) * ld + col())
                     : "memory");
      });
      asm volatile("cp.async.wait_all;" ::: "memory");                    // a lane reads what it brought itself
    };
    for (int first = lo; first < hi; first += FIT) {
      bring(first, min(FIT, hi - first));
      pieces(min(FIT, hi - first), [&](int place, int) { look(room[place]); });
    }
    rescale<TEAM>(before, tops);
    for (int first = lo; first < hi; first += FIT) {
      if (hi - lo > FIT) bring(first, min(FIT, hi - first));
      pieces(min(FIT, hi - first), [&](int place, int r) { put(room[place], first + r); });
    }
  }
};

// ROWS: a row per warp where a step's sequences bring one each (256 rows of 8 heads of 128: 4.1 us, 4.4 with four to a warp, 11.6 with
// sixteen; of 4 heads 2.7, 4.1 and 11.4), a block's worth where prompts bring many (14,000 rows, when that was 20 us: 26 with four to a
// warp, 64 with one).
// TEAM: of blocks of more than 32 rows a run is four warps', which find the same runs and share the rows of a long one (1000 rows in
// blocks of 64: 3.5 us, 7.1 with a warp to each; 8192 in blocks of 128: 17.1 and 23.3; but 512 rows in as many blocks 6.2 and 5.4, and
// 2000 rows in blocks of 32 6.9 and 5.0).
template <int KIND, int HD, int ROWS, int TEAM>
__global__ void __launch_bounds__(128, ROWS == 1 ? 8 : 7)
kv_write_q8_kernel(const __nv_bfloat16* __restrict__ qkv, int ld, int k_col, int v_col, const int* __restrict__ slot,
                   uint8_t* k_cache, uint8_t* v_cache, float* k_scale, float* v_scale, int M, int Hkv, int block_size,
                   int block_shift, long num_blocks, int* status) {
  static_assert(ROWS <= 16, "a warp sees 32 rows at once, and a run of 16 to its end");
  extern __shared__ uint4 kw_room[];           // where blocks have more than 16 rows
  __shared__ uint32_t s_top[4];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, part = TEAM > 1 ? blockIdx.y : blockIdx.y * 4 + (threadIdx.x >> 5), row0 = blockIdx.x * ROWS;
  if (part >= 2 * Hkv) return;
  const bool is_v = part >= Hkv;
  const int h = is_v ? part - Hkv : part;
  const __nv_bfloat16* x = qkv + (is_v ? v_col : k_col) + h * HD;
  uint8_t* cache = is_v ? v_cache : k_cache;
  float* scales = is_v ? v_scale : k_scale;

  if (ROWS == 16) {            // the rows are on their way to L2 while the slots are looked up: 10.6 us instead of 11.5 (14,760 rows);
                               // calls of fewer rows, which are in L2 already more often than not, lose 0.2 us by it
    constexpr int LINES = HD / 64 ? HD / 64 : 1;
    if ((TEAM == 1 || threadIdx.x < 32) && lane < ROWS * LINES && row0 + lane / LINES < M)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(x + static_cast<size_t>(row0 + lane / LINES) * ld + lane % LINES * 64));
  }
  const int s = row0 + lane < M ? slot[row0 + lane] : -1;
  int above = row0 > 0 ? slot[row0 - 1] : -1, seen[ROWS == 1 ? KW_STEP / 32 : 1];
  if (ROWS == 1) {             // all rows above, on their way together
#pragma unroll
    for (int i = 0; i < KW_STEP / 32; ++i) seen[i] = i * 32 + lane < row0 ? slot[i * 32 + lane] : -1;
  }
  int prev = __shfl_up_sync(0xffffffffu, s, 1);
  if (lane == 0) prev = above;
  const int blk = s < 0 ? 0 : block_shift >= 0 ? s >> block_shift : s / block_size;
  const bool goes_on = s > 0 && prev == s - 1 && s != blk * block_size;        // with the run of the row before
  const uint32_t on = __ballot_sync(0xffffffffu, goes_on), written = __ballot_sync(0xffffffffu, s >= 0);
  // A second run in a block would be a second warp's at the same scale: refused where it follows the first, rows that are not
  // written between them or not, and behind any other rows where the call is a step's (0.1 us of 2.7: 256 rows of 4 heads).
  bool astray;
  if (ROWS == 1) {
    const int first = __shfl_sync(0xffffffffu, blk, 0) * block_size;
    bool again = false;
#pragma unroll
    for (int i = 0; i < KW_STEP / 32; ++i) again |= q8_in_block(seen[i], first, block_size);
    astray = __any_sync(0xffffffffu, again) && s >= 0 && !goes_on;
  } else {
    if (above < 0 && (written & ((1u << ROWS) - 1)))
#pragma unroll 1
      for (int r = row0 - 2; r >= 0 && above < 0; r -= 256) {
        int v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = r - i * 32 >= lane ? slot[r - i * 32 - lane] : -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t found = __ballot_sync(0xffffffffu, v[i] >= 0);
          if (found && above < 0) above = __shfl_sync(0xffffffffu, v[i], __ffs(found) - 1);
        }
      }
    const uint32_t before = written & ((1u << lane) - 1u);
    const int near = __shfl_sync(0xffffffffu, s, before ? 31 - __clz(before) : 0);
    astray = s >= 0 && !goes_on && q8_in_block(before ? near : above, blk * block_size, block_size);
  }
  if (astray && lane < ROWS && status) atomicMax(status, ST_BAD_ARGS);
  // of a team, a run of 17 rows or more is all warps', one of fewer is one warp's
  const bool whose = TEAM == 1 || (lane & 3) == static_cast<int>(threadIdx.x >> 5) || (on >> lane >> 1 & 0xffffu) == 0xffffu;
  for (uint32_t todo = __ballot_sync(0xffffffffu, lane < ROWS && s >= 0 && !goes_on && !astray && whose); todo; todo &= todo - 1) {
    const int i = __ffs(todo) - 1, s0 = __shfl_sync(0xffffffffu, s, i), block = __shfl_sync(0xffffffffu, blk, i);
    if (!q8_index_ok(s0, num_blocks * block_size, status)) continue;
    const int r0 = row0 + i, at = s0 - block * block_size;
    const uint32_t ends = ~on & (0xfffffffeu << i);
    int n = (ends ? __ffs(ends) - 1 : 32) - i;
    while (!ends) {                          // longer than what is seen: 32 rows at a time
      const int most = min(block_size - at, M - r0);
      const uint32_t more = __ballot_sync(0xffffffffu, n + lane < most && slot[min(r0 + n + lane, M - 1)] == s0 + n + lane);
      n += more == 0xffffffffu ? 32 : __ffs(~more) - 1;
      if (more != 0xffffffffu) break;
    }
    const long head = static_cast<long>(block) * Hkv + h;
    KwRun<KIND, HD> run{x + static_cast<size_t>(r0) * ld, ld, n, at, block_size, cache + head * block_size * HD, scales + head};
    uint4* room = kw_room + (threadIdx.x >> 5) * KW_FIT * KwRun<KIND, HD>::LPR;
    if (n > 16) run.template staged<TEAM, KW_FIT>(room, s_top);           // one at most begins among 16 rows
    else if (n * (HD / 8) <= 32) run.template held<1, false>();
    else if (n == 16) run.template held<HD / 16, true>();                 // whole blocks, for the most part
    else run.template held<HD / 16, false>();
  }
}

// The cached keys and values at a list of slots -> k | v columns of dst [n, ld], as bf16 (exact: a code has at most 8 bits);
// rows with a negative slot become zeros.  A thread takes 16 codes of the same place in ROWS rows at a time, whose loads are in
// flight together, and stores them as 32 bytes where the destination allows.  Bound by bytes, 1 in and 2 out per value: 18.9 us
// for 32,000 rows of 4 heads of 128 (98 MB) with four rows, 20.1 with one; what fits the chip once takes one row: 300 of 2 heads
// of 64 take 2.1 us, 2.9 with four.
template <int KIND, int ROWS, bool WIDE>
__global__ void __launch_bounds__(256)
kv_rows_q8_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const float* __restrict__ k_scale,
                  const float* __restrict__ v_scale, const int* __restrict__ slot, int n, __nv_bfloat16* __restrict__ dst, int ld,
                  int k_col, int v_col, int Hkv, int hd, int block_size, int block_shift, long num_blocks, int* status) {
  pdl_wait();
  pdl_launch_dependents();
  const int half = Hkv * hd / 16;
  for (int at = threadIdx.x; at < 2 * half; at += blockDim.x) {
    const bool is_v = at >= half;
    const int u = (is_v ? at - half : at) * 16, h = u / hd, d = u - h * hd;
    const uint8_t* cache = (is_v ? v_cache : k_cache) + d;
    const float* scales = is_v ? v_scale : k_scale;
    __nv_bfloat16* to = dst + (is_v ? v_col : k_col) + u;
    for (int r0 = (blockIdx.x * blockDim.y + threadIdx.y) * ROWS; r0 < n; r0 += gridDim.x * blockDim.y * ROWS) {
      uint4 raw[ROWS];
      float scale[ROWS];
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        const int s = r0 + j < n ? slot[r0 + j] : -1;
        raw[j] = make_uint4(0, 0, 0, 0);
        scale[j] = 0.f;
        if (s >= 0 && q8_index_ok(s, num_blocks * block_size, status)) {
          const int block = block_shift >= 0 ? s >> block_shift : s / block_size;
          const long head = static_cast<long>(block) * Hkv + h;
          raw[j] = *reinterpret_cast<const uint4*>(cache + (head * block_size + (s - block * block_size)) * hd);
          scale[j] = scales[head];
        }
      }
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        if (r0 + j >= n) break;
        const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[4];
          q8_decode4<KIND>(w[i], f);
          o[2 * i] = pack_bf16x2(f[0] * scale[j], f[1] * scale[j]);
          o[2 * i + 1] = pack_bf16x2(f[2] * scale[j], f[3] * scale[j]);
        }
        if (WIDE) {
          asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + static_cast<size_t>(r0 + j) * ld), "r"(o[0]),
                       "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                       : "memory");
        } else {
          uint4* p = reinterpret_cast<uint4*>(to + static_cast<size_t>(r0 + j) * ld);
          p[0] = make_uint4(o[0], o[1], o[2], o[3]);
          p[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
    }
  }
}

}  // namespace artb

using namespace artb;

// slot: block * block_size + place, < 0: the row is not written.
// A slot beyond the cache is not written either and reported through `status`.  Runs of one block with rows of others between them are
// refused in calls of up to KW_STEP rows; in longer ones, where finding them would take a look at all rows for each run, they are
// written at the same time and what the block then holds is undefined.
ARTB_EXPORT int artb_kv_write_q8(const KvRowsArgs* a, cudaStream_t st) {
  const int M = a->n, ld = a->ld, Hkv = a->Hkv, hd = a->hd, block_size = a->block_size, kind = a->kind;
  if (M <= 0) return 0;
  if (Hkv <= 0 || block_size < 16 || (block_size & 15) || (ld & 7) || (a->k_col & 7) || (a->v_col & 7)) return ERR_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a->rows) | reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) return ERR_BAD_ALIGN;
  const int shift = (block_size & (block_size - 1)) ? -1 : __builtin_ctz(block_size);
#define ARTB_KW(KIND_, HD_)                                                                                                  \
  if (kind == KIND_ && hd == HD_) {                                                                                          \
    auto go = [&](auto kern, int rows, int parts) {                                                                          \
      const int room = block_size > 16 ? 4 * KW_FIT * KwRun<KIND_, HD_>::PLACE : 0;                                          \
      return static_cast<int>(launch_ahead(kern, dim3((M + rows - 1) / rows, (2 * Hkv + parts - 1) / parts), dim3(128), room, st, \
                                            (const __nv_bfloat16*)a->rows, ld, a->k_col, a->v_col, a->slot,                  \
                                            (uint8_t*)a->k_cache, (uint8_t*)a->v_cache, a->k_scale, a->v_scale, M, Hkv,      \
                                            block_size, shift, a->num_blocks, a->status));                                   \
    };                                                                                                                       \
    if (M <= KW_STEP) return go(kv_write_q8_kernel<KIND_, HD_, 1, 1>, 1, 4);                                                    \
    if (block_size > 32) return go(kv_write_q8_kernel<KIND_, HD_, 16, 4>, 16, 1);                                            \
    if (M <= 2048) return go(kv_write_q8_kernel<KIND_, HD_, 4, 1>, 4, 4);                                                    \
    return go(kv_write_q8_kernel<KIND_, HD_, 16, 1>, 16, 4);                                                                 \
  }
  ARTB_KW(Q8_E4M3, 128) ARTB_KW(Q8_E4M3, 64) ARTB_KW(Q8_E4M3, 32)
  ARTB_KW(Q8_INT8, 128) ARTB_KW(Q8_INT8, 64) ARTB_KW(Q8_INT8, 32)
#undef ARTB_KW
  return ERR_BAD_SHAPE;
}

ARTB_EXPORT int artb_kv_rows_q8(const KvRowsArgs* a, cudaStream_t st) {
  const int n = a->n, ld = a->ld, Hkv = a->Hkv, hd = a->hd, block_size = a->block_size, kind = a->kind;
  if (n <= 0) return 0;
  if (Hkv <= 0 || hd < 16 || (hd & 15) || block_size < 1 || (ld & 7) || (a->k_col & 7) || (a->v_col & 7)) return ERR_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a->rows) | reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) return ERR_BAD_ALIGN;
  const int vec = Hkv * hd / 8, bx = vec < 256 ? vec : 256, by = 256 / bx;
  const bool once = (static_cast<long>(n) + by - 1) / by <= 8L * sm_count();
  const long blocks = (static_cast<long>(n) + by * (once ? 1 : 4) - 1) / (by * (once ? 1 : 4));
  const int shift = (block_size & (block_size - 1)) ? -1 : __builtin_ctz(block_size);
  const bool wide = ((reinterpret_cast<uintptr_t>(a->rows) & 31) | (ld & 15) | (a->k_col & 15) | (a->v_col & 15)) == 0;
  auto go = [&](auto kern) {
    return static_cast<int>(launch_ahead(kern, dim3(static_cast<unsigned>(blocks < 1 << 20 ? blocks : 1 << 20)), dim3(bx, by), 0, st,
                                         (const uint8_t*)a->k_cache, (const uint8_t*)a->v_cache, a->k_scale, a->v_scale, a->slot, n,
                                         (__nv_bfloat16*)a->rows, ld, a->k_col, a->v_col, Hkv, hd, block_size, shift, a->num_blocks,
                                         a->status));
  };
#define ARTB_KR(KIND_)                                                                                                     \
  if (kind == KIND_) {                                                                                                     \
    if (once) return wide ? go(kv_rows_q8_kernel<KIND_, 1, true>) : go(kv_rows_q8_kernel<KIND_, 1, false>);                \
    return wide ? go(kv_rows_q8_kernel<KIND_, 4, true>) : go(kv_rows_q8_kernel<KIND_, 4, false>);                          \
  }
  ARTB_KR(Q8_E4M3)
  ARTB_KR(Q8_INT8)
#undef ARTB_KR
  return ERR_BAD_SHAPE;
}
