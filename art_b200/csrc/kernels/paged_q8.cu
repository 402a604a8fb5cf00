// Decode attention over a paged cache held in 8 bits (numbers and layout: kv_q8.cuh): one new token per sequence,
//     o_h = sum_j softmax_j(q_h . k_j / sqrt(hd)) v_j,   j < ctx_len,   k_j, v_j = code * scale of the block and kv head.
//
// The G = Hq / Hkv query heads of a kv head are the columns of one m16n8 tile (two for G > 8), so that keys and values are
// read once for all of them.  Both products have the cache's side as their rows,
//     S^T [16 keys x heads] = K Q^T,     O^T [hd x heads] = V^T P^T,
// and 16 keys are always of one block: a key scale is one factor of a tile of scores, a value scale one of a tile of weights, and
// no code is ever multiplied by either.  Codes become fp16 (exact: e4m3 and int8 have at most 8 significant bits) but for keys in
// int8, which are multiplied as they are.  A power of two per head brings the largest of its query to [2^14, 2^15); beside e4m3 keys
// queries are fp16 then (exact but for what is 2^-38 of the largest), beside int8 keys whole numbers of 16 bits (off by 1/2 at most:
// 2^-15 of the largest, where a key's code is off by 2^-8 of its block's largest), whose high and low bytes have a product each, in
// exact sums.  Widening int8 keys instead takes 70.5 us where this takes 66.8 (the 48 contexts below), under the power cap 77 and 73;
// four e4m3 codes are widened by two instructions where int8 takes five.  Weights are rounded to fp16.  The order in which a product
// sums is free, so a lane's fragments are neighbouring bytes: hd / 4 values of a key, and hd / 8 values of four keys, whose bytes are
// paired up in registers while they are widened.
//
// Bound by the cache's bytes, and beside them by what a launch begins and ends with.  256 contexts of 512 to 2032 keys, 28 / 4 heads
// of 128, e4m3 (338 MB, 52 us at the copy rate): 60 us, of which 3 pass before the first keys are asked for and 6 between the ends of
// the first and of the last warp's tiles.  48 contexts of 2000 to 6000, 32 / 8 heads, int8 (395 MB, 60 us): 66 us in bursts, 69 to
// 74, by the GPU, when the power cap has taken the clock to 1.85 or 1.75 GHz.  What else was tried on these two, when they took 61 and
// 70:
//   80, 90   each lane loads its fragments from global memory into registers, three CTAs of four warps per SM
//   72, 77   a fifth warp brings the tiles of the four, sixteen copies a turn from four lanes
//   65, 75   one CTA of eight warps per SM
//   71, 79   twice as many shares as fit the chip at a time
//   137, 154 four CTAs per SM with 128 registers a thread
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "host_utils.h"
#include "kv_q8.cuh"

namespace artb {

constexpr int PQ_KEYS = 32;              // keys of a tile: two stretches of 16, each within a block
constexpr int PQ_WARPS = 4;
constexpr int PQ_THREADS = PQ_WARPS * 32;
constexpr int PQ_MIN_TILES = 4;   // tiles of a CTA at least: one per warp
constexpr int PQ_ENTRIES = 1024;         // of a CTA's list of where sequences begin
constexpr int PQ_ROUND = 16;             // tiles that a warp looks up at a time
constexpr int PQ_NOTES = 2 * PQ_ROUND;   // and keeps noted: those in use and the next
constexpr float PQ_SLACK = 8.f;          // how far (in powers of two) a score may pass the reference before that moves

__host__ __device__ constexpr int pq_heads(int G) { return G > 8 ? 16 : 8; }
// tiles of a warp in shared memory
__host__ __device__ constexpr int pq_stages(int hd, int heads) { return hd == 128 ? 2 : hd == 64 ? (heads == 8 ? 3 : 2) : 4; }
__host__ __device__ constexpr int pq_ctas_per_sm(int hd) { return hd == 128 ? 2 : 3; }  // by shared memory
__host__ __device__ constexpr int pq_piece_floats(int heads, int hd) { return heads * hd + 2 * heads; }

template <int HD, int HEADS>
struct PqSmem {
  static constexpr int STRETCH = 16 * HD, STAGE = 4 * STRETCH, RING = pq_stages(HD, HEADS) * STAGE;      // keys, keys, values, values
  static constexpr int PIECE = pq_piece_floats(HEADS, HD) * 4;
  static constexpr int BYTES = 1024 + PQ_WARPS * (RING + PIECE);                                    // rings begin on 1024 bytes
  static_assert(PIECE <= RING, "a warp's last piece goes where its tiles were");
};

template <int BYTES>
__device__ __forceinline__ void pq_take(uint32_t* r, const uint8_t* p) {
  if (BYTES == 4) {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r[0] = v.x;
    r[1] = v.y;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r[0] = v.x;
    r[1] = v.y;
    r[2] = v.z;
    r[3] = v.w;
  }
}

// Where 16-byte piece `piece` of row `row` of a stretch lies: the copies spread a row's pieces by the row's number, so that the
// lanes of a fragment find theirs in different banks.
template <int HD>
__device__ __forceinline__ int pq_piece_at(int row, int piece) {
  return row * HD + ((piece ^ (HD == 128 ? row & 7 : HD == 64 ? row >> 1 & 3 : row >> 2 & 1)) << 4);
}

// Four codes to two pairs of fp16: bytes 0, 1 and bytes 2, 3.
template <int KIND>
__device__ __forceinline__ void pq_widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (KIND == Q8_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // 0x6400 | u is 1024 + u in fp16, and u = code + 128
    const uint32_t x = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 p = __hsub2(*reinterpret_cast<__half2*>(&a), off), q = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&p);
    hi = *reinterpret_cast<const uint32_t*>(&q);
  }
}

__device__ __forceinline__ void pq_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 32 int8 codes of 16 keys, as they lie in the cache, with the high bytes of the queries or, UNSIGNED, the low ones.  Each sum is
// below 128 * 255 * 128 and the two together below 2^30.
template <bool UNSIGNED>
__device__ __forceinline__ void pq_mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (UNSIGNED)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pq_transpose(uint32_t x) {       // an 8 x 8 tile of 16-bit numbers over the warp
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float pq_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pq_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int BYTES>
__device__ __forceinline__ void pq_put(__nv_bfloat16* dst, const uint32_t* r) {
  if (BYTES == 8) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(r[0], r[1]);
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(dst)[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
  }
}

// A tile: which of its sequence's it is; keys of each stretch (16, fewer at a context's end, 0 where its block is none), their rows
// in the codes and their scales.
struct __align__(16) PqNote {
  int seq, tile, len, keys;                 // keys: first stretch | second << 8
  float ks[2], vs[2];
  int row[2], none[2];
};

// What a warp leaves of a sequence that it has not read whole: tiles [lo, hi) of the sequence whose first tile is `first`.
struct PqPiece {
  int seq, len, first, lo, hi;
};

// not at all; to its end, and then others'; to its end, which is the warp's; beyond the warp's end
enum PqGoesOn : int { PQ_NOT = 0, PQ_THEN_OTHERS = 1, PQ_TO_ITS_END = 2, PQ_BEYOND = 3 };

// A piece as a warp's registers hold it, of the sums of some keys: heads n * 8 + 2t + x, values g * hd / 8 + 2j (acc[][][x]) and + 1
// (acc[][][2 + x]), references and sums of weights.  In memory: a float4 per lane, lanes side by side, then references and sums by
// head.
template <int NT, int JT>
struct PqSums {
  float m[NT][2], l[NT][2], acc[NT][JT][4];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m[n][x] = -INFINITY;
        l[n][x] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[n][j][x] = 0.f;
    }
  }

  template <bool GLOBAL>
  __device__ __forceinline__ void put(float* dst, int lane, int G) const {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (GLOBAL && n * 8 + 2 * t >= G) continue;              // no such heads
#pragma unroll
      for (int j = 0; j < JT; ++j) {
        float4* to = reinterpret_cast<float4*>(dst) + (n * JT + j) * 32 + lane;
        const float4 v = make_float4(acc[n][j][0], acc[n][j][1], acc[n][j][2], acc[n][j][3]);
        if (GLOBAL) __stcg(to, v);
        else *to = v;
      }
      if (g == 0) {
        float* tail = dst + NT * JT * 128 + n * 8 + 2 * t;
        *reinterpret_cast<float2*>(tail) = make_float2(m[n][0], m[n][1]);
        *reinterpret_cast<float2*>(tail + NT * 8) = make_float2(l[n][0], l[n][1]);
      }
    }
  }

  template <bool GLOBAL>
  __device__ __forceinline__ void get(const float* src, int lane, int G) {
    const int t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (GLOBAL && n * 8 + 2 * t >= G) continue;
#pragma unroll
      for (int j = 0; j < JT; ++j) {
        const float4* from = reinterpret_cast<const float4*>(src) + (n * JT + j) * 32 + lane;
        const float4 v = GLOBAL ? __ldcg(from) : *from;
        acc[n][j][0] = v.x;
        acc[n][j][1] = v.y;
        acc[n][j][2] = v.z;
        acc[n][j][3] = v.w;
      }
      const float2* tail = reinterpret_cast<const float2*>(src + NT * JT * 128 + n * 8 + 2 * t);
      const float2 a = GLOBAL ? __ldcg(tail) : tail[0], b = GLOBAL ? __ldcg(tail + NT * 4) : tail[NT * 4];
      m[n][0] = a.x;
      m[n][1] = a.y;
      l[n][0] = b.x;
      l[n][1] = b.y;
    }
  }

  // Both are taken to the larger reference; what has none counts nothing, and sums that are not numbers stay so.
  __device__ __forceinline__ void add(const PqSums& o) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float top = fmaxf(m[n][x], o.m[n][x]), r = top == -INFINITY ? 0.f : top;
        const float a = pq_exp2(m[n][x] - r), b = pq_exp2(o.m[n][x] - r);
        m[n][x] = top;
        l[n][x] = l[n][x] * a + o.l[n][x] * b;
#pragma unroll
        for (int j = 0; j < JT; ++j) {
          acc[n][j][x] = acc[n][j][x] * a + o.acc[n][j][x] * b;
          acc[n][j][2 + x] = acc[n][j][2 + x] * a + o.acc[n][j][2 + x] * b;
        }
      }
  }

  // The heads' result, `unit` times the sums over the sums of weights; `o`: the first head's row.
  __device__ __forceinline__ void write(__nv_bfloat16* o, float unit, int lane, int G) const {
    constexpr int HD = JT * 16;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int head = n * 8 + 2 * t + x;
        if (head >= G) continue;
        const float f = l[n][x] == 0.f ? 0.f : rcp_approx(l[n][x]);            // a small unit times that may be no normal number
        uint32_t r[JT];
#pragma unroll
        for (int j = 0; j < JT; ++j) r[j] = pack_bf16x2(acc[n][j][x] * f * unit, acc[n][j][2 + x] * f * unit);
        pq_put<JT * 4>(o + head * HD + g * (HD / 8), r);
      }
  }
};

// The sequences are laid end to end, in tiles of PQ_KEYS keys, and cut into equal shares, wherever sequences begin and end in
// them; a share belongs to Hkv neighbouring CTAs, one per kv head, and the shares together fill the chip once.  A CTA's share is
// cut again into four, one per warp, which goes through its tiles without a stop at the ends of sequences: its lanes look up
// sixteen tiles at a time (sequence, blocks, then scales) while those before are in use, and a tile's copies into shared memory
// start as soon as the warp has taken the last bytes of the one whose place it gets.  A sequence that one warp reads whole is
// written by it.  Of one that several warps of the CTA read, the first adds the others' pieces to its own; what still is a part then
// goes to the workspace, and the CTA that finishes last adds the parts up, in an order that is always the same.
template <int KIND, int HD, int HEADS>
__global__ void __launch_bounds__(PQ_THREADS, pq_ctas_per_sm(HD))
paged_decode_q8_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                       const __nv_bfloat16* __restrict__ q, int ldq, const float* __restrict__ k_scale,
                       const float* __restrict__ v_scale, const int* __restrict__ block_table, int max_blocks,
                       const int* __restrict__ ctx_len, int block_size, int sub_shift, int nseq, int G,
                       uint32_t per_share, __nv_bfloat16* __restrict__ out, int ldo, float* part, int* count, float scale_log2,
                       long num_blocks, int* status) {
  using S = PqSmem<HD, HEADS>;
  constexpr int NT = HEADS / 8, JT = HD / 16, KW = HD / 16, VW = HD / 32, STAGES = pq_stages(HD, HEADS);
  extern __shared__ uint8_t pq_smem_raw[];
  uint8_t* rings = pq_smem_raw + (1024 - (smem_u32(pq_smem_raw) & 1023));
  __shared__ int s_warp[PQ_WARPS], s_longest[PQ_WARPS], s_first[PQ_ENTRIES], s_len[PQ_ENTRIES];
  __shared__ volatile int s_abort;
  __shared__ int s_goes_on[PQ_WARPS];       // how a warp goes on with the sequence that the one before it ends in (PqGoesOn)
  __shared__ int4 s_part[2];                // sequences that the CTA is the last to finish a part of: number, first share, parts, 1
  __shared__ PqNote s_note[PQ_WARPS][PQ_NOTES];
  __shared__ __align__(8) uint64_t s_full[PQ_WARPS][STAGES];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid < PQ_WARPS * STAGES) {
    mbar_init(&s_full[0][0] + tid, 1);
    fence_mbar_init();
  }
  if (tid < PQ_WARPS) s_goes_on[tid] = PQ_NOT;
  if (tid < 2) s_part[tid] = make_int4(0, 0, 0, 0);
  if (tid == PQ_THREADS - 1) {
    s_abort = 0;
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  pdl_wait();
  const int Hkv = gridDim.x, kvh = blockIdx.x, shares = gridDim.y, share = blockIdx.y;
  const int table_keys = min(static_cast<long>(max_blocks) * block_size, 0x7fffffffL - PQ_KEYS);
  auto checked = [&](int n) {
    if (n > table_keys) {
      if (kvh == 0 && share == 0 && status) atomicMax(status, ST_BOUNDS);
      n = table_keys;
    }
    return max(n, 0);
  };
  auto tiles_in = [](int len) { return (len + PQ_KEYS - 1) / PQ_KEYS; };

  // Where sequences begin, in tiles: an entry for each (for `run` of them where there are very many), each thread's entries
  // first for themselves, then a scan over the threads.
  const int run = (nseq + PQ_ENTRIES - 1) / PQ_ENTRIES, entries = (nseq + run - 1) / run, mine = (entries + PQ_THREADS - 1) / PQ_THREADS;
  const int e0 = min(entries, tid * mine), e1 = min(entries, e0 + mine);
  auto empty = [&](int i) {                            // an empty context (the padding of a batch): zeros
    uint4* o = reinterpret_cast<uint4*>(out + static_cast<size_t>(i) * ldo + kvh * G * HD);
#pragma unroll 1
    for (int d = 0; d < G * HD / 8; ++d) o[d] = make_uint4(0, 0, 0, 0);
  };
  int own = 0, longest = 0;
  if (run == 1) {
    int len[PQ_ENTRIES / PQ_THREADS];                  // all lengths on their way at once
#pragma unroll
    for (int j = 0; j < PQ_ENTRIES / PQ_THREADS; ++j) len[j] = tid + j * PQ_THREADS < nseq ? ctx_len[tid + j * PQ_THREADS] : 0;
#pragma unroll
    for (int j = 0; j < PQ_ENTRIES / PQ_THREADS; ++j) {
      const int i = tid + j * PQ_THREADS;
      if (i >= nseq) break;
      const int n = checked(len[j]);
      s_len[i] = n;
      if (n == 0 && share == shares - 1) empty(i);
    }
    __syncthreads();
  }
#pragma unroll 1
  for (int e = e0; e < e1; ++e) {
    s_first[e] = own;
    if (run == 1) {
      own += tiles_in(s_len[e]);
      longest = max(longest, tiles_in(s_len[e]));
    } else {
#pragma unroll 1
      for (int i = e * run; i < min(nseq, (e + 1) * run); ++i) {
        const int n = checked(ctx_len[i]);
        own += tiles_in(n);
        if (n == 0 && share == shares - 1) empty(i);
      }
    }
  }
  int incl = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 31) {
    s_warp[warp] = incl;
    s_longest[warp] = longest;
  }
  __syncthreads();
  int total = 0, before = incl - own;
#pragma unroll
  for (int w = 0; w < PQ_WARPS; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
    longest = max(longest, s_longest[w]);
  }
#pragma unroll 1
  for (int e = e0; e < e1; ++e) s_first[e] += before;
  // The parts of a sequence are added up by one CTA.  With t microseconds for a warp's tile and p for a part of L tiles, shares of n
  // cost n / 4 t + L / n p, the least at n = 2 sqrt(L p / t); p goes with the part's size.  One context of 16,000 keys, 8 heads of 128
  // to a kv head: 12.6 us, 16.6 with shares as small as the chip has room for; 16 heads: 18.5 and 26.9.
  const int few = static_cast<int>(sqrtf(0.3f * HEADS * HD / 1024 * longest));
  const int per = max(max(PQ_MIN_TILES, few), static_cast<int>(__umulhi(total + shares - 1, per_share)) + (shares == 1));
  const int per_warp = (per + PQ_WARPS - 1) / PQ_WARPS;
  const int at = share * per;
  if (at >= total) return;                  // the whole CTA
  const int end = min(total, at + per);
  __syncthreads();

  const int lo = at + warp * per_warp, tiles = min(end, lo + per_warp) - lo;
  constexpr int SLOT = pq_piece_floats(HEADS, HD);
  // a CTA leaves at most two parts: of the sequence that it begins in the middle of, and of the one it ends in
  auto slot = [&](int sh, bool starts) { return part + static_cast<size_t>((sh * Hkv + kvh) * 2 + starts) * SLOT; };
  auto result = [&](int seq) { return out + static_cast<size_t>(seq) * ldo + kvh * G * HD; };
  auto piece_at = [&](int w) { return reinterpret_cast<float*>(rings + PQ_WARPS * S::RING + w * S::PIECE); };
  auto ring_at = [&](int w) { return reinterpret_cast<float*>(rings + w * S::RING); };
  auto locate = [&](int x, int& seq, int& len) {              // the sequence that tile x is of, and its first tile
    int a = 0, b = entries;
#pragma unroll 1
    while (b - a > 1) {
      const int mid = (a + b) >> 1;
      if (s_first[mid] <= x) a = mid;
      else b = mid;
    }
    int first = s_first[a];
    seq = a * run;
    len = run == 1 ? s_len[a] : checked(ctx_len[seq]);
#pragma unroll 1
    while (x >= first + tiles_in(len) && seq + 1 < nseq) {
      first += tiles_in(len);
      len = checked(ctx_len[++seq]);
    }
    return first;
  };
  // A part of a sequence is there (released with what the thread's warp wrote): number, first share, parts, whether it is the last.
  auto count_part = [&](int seq, int len, int first) {
    const int sh0 = first / per, parts = (first + tiles_in(len) - 1) / per - sh0 + 1;
    int seen;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(seen) : "l"(&count[seq * Hkv + kvh]) : "memory");
    return make_int4(seq, sh0, parts, seen == parts - 1);
  };
  PqSums<NT, JT> sums;
  auto& m = sums.m;
  auto& l = sums.l;
  auto& acc = sums.acc;
  PqPiece last, owed;            // the piece that the warp ends with, and the part that warp 0 leaves before
  bool open = false, owes = false;
  if (tiles > 0) {
    uint8_t* ring = rings + warp * S::RING;
    PqNote* notes = s_note[warp];
    const int subs = block_size >> 4;
    PqNote next;                            // this lane's tile of the round that is being looked up
    int blk[2];
    auto find = [&](int i) {                // which it is, and its blocks on their way
      if (lane >= PQ_ROUND || i >= tiles) return;
      const int x = lo + i, first = locate(x, next.seq, next.len);
      next.tile = x - first;
      const int left = next.len - next.tile * PQ_KEYS;
      next.keys = min(left, 16) | max(0, min(left - 16, 16)) << 8;
      const int* row = block_table + static_cast<size_t>(next.seq) * max_blocks;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int stretch = min(next.tile * 2 + u, (next.len - 1) >> 4), in = sub_shift >= 0 ? stretch >> sub_shift : stretch / subs;
        next.row[u] = (stretch - in * subs) * 16;
        blk[u] = __ldcg(row + in);
      }
    };
    auto place = [&](int i) {               // its rows, and its scales on their way
      if (lane >= PQ_ROUND || i >= tiles) return;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool good = q8_index_ok(blk[u], num_blocks, status);
        if (!good) next.keys &= u ? 0xff : 0xff00;
        const long head = good ? static_cast<long>(blk[u]) * Hkv + kvh : kvh;
        next.row[u] += static_cast<int>(head * block_size);
        next.ks[u] = __ldcg(k_scale + head);
        next.vs[u] = __ldcg(v_scale + head);
      }
    };
    auto note = [&](int i) {
      if (lane < PQ_ROUND && i < tiles) {
        int4* n = reinterpret_cast<int4*>(notes + i % PQ_NOTES);
        n[0] = make_int4(next.seq, next.tile, next.len, next.keys);
        *reinterpret_cast<float4*>(n + 1) = make_float4(next.ks[0], next.ks[1], next.vs[0], next.vs[1]);
        *reinterpret_cast<int2*>(n + 2) = make_int2(next.row[0], next.row[1]);
      }
      __syncwarp();
    };
    auto bring = [&](int i, int keys, int row0, int row1) {       // one lane; nothing of the stage is read any more
      uint64_t* full = &s_full[warp][i % STAGES];
      uint8_t* to = ring + i % STAGES * S::STAGE;
      const int bytes = ((keys & 0xff) ? 2 * S::STRETCH : 0) + ((keys >> 8) ? 2 * S::STRETCH : 0);
      mbar_expect_tx(full, bytes);
      if (keys & 0xff) {
        tma_load_2d(to, &k_map, 0, row0, full);
        tma_load_2d(to + 2 * S::STRETCH, &v_map, 0, row0, full);
      }
      if (keys >> 8) {
        tma_load_2d(to + S::STRETCH, &k_map, 0, row1, full);
        tma_load_2d(to + 3 * S::STRETCH, &v_map, 0, row1, full);
      }
    };
    // this lane's bytes of a stretch: of the keys g and g + 8, and of the values 2t, 2t + 1 (and 8 further)
    const int k_at[2] = {HD == 32 ? pq_piece_at<HD>(g, t >> 1) + (t & 1) * 8 : pq_piece_at<HD>(g, HD == 128 ? 2 * t : t),
                         HD == 128 ? pq_piece_at<HD>(g, 2 * t + 1) : 0};
    const int v_piece = HD == 128 ? g : HD == 64 ? g >> 1 : g >> 2, v_rest = HD == 128 ? 0 : HD == 64 ? (g & 1) * 8 : (g & 3) * 4;
    const int v_at[2] = {pq_piece_at<HD>(2 * t, v_piece) + v_rest, pq_piece_at<HD>(2 * t + 1, v_piece) + v_rest};

    uint32_t q_raw[NT][JT * 2], qf[NT][JT][2];
    float qs[NT][2], unit, per_unit;
    auto request_q = [&](int seq) {         // heads g (and g + 8), hd / 4 values: those that the lane holds of a key, in the same order
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int head = n * 8 + g;
        const uint4* row = reinterpret_cast<const uint4*>(q + static_cast<size_t>(seq) * ldq + (kvh * G + head) * HD + t * (HD / 4));
#pragma unroll
        for (int v = 0; v < JT / 2; ++v) {
          const uint4 x = head < G ? __ldcg(row + v) : make_uint4(0, 0, 0, 0);
          q_raw[n][4 * v] = x.x;
          q_raw[n][4 * v + 1] = x.y;
          q_raw[n][4 * v + 2] = x.z;
          q_raw[n][4 * v + 3] = x.w;
        }
      }
    };
    find(lane);
    request_q(__shfl_sync(0xffffffffu, next.seq, 0));
    place(lane);
    if (lane < min(STAGES, tiles)) bring(lane, next.keys, next.row[0], next.row[1]);
    note(lane);

    int piece_lo = notes[0].tile;
    bool fresh = true;
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
      if (fresh) {
        fresh = false;
        unit = per_unit = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t(&raw)[JT * 2] = q_raw[n], top = 0;
#pragma unroll
          for (int v = 0; v < JT * 2; ++v) top = __vmaxu2(top, raw[v] & 0x7fff7fffu);
          top = max(top & 0xffffu, top >> 16);
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int e = top >= 0x7f80u || top == 0 ? 0 : min(100, 14 + 127 - static_cast<int>(top >> 7));
          const float up = q8_pow2(e);
#pragma unroll
          for (int j = 0; j < JT; ++j) {
            float v[4];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              v[2 * x] = __uint_as_float(raw[2 * j + x] << 16) * up;
              v[2 * x + 1] = __uint_as_float(raw[2 * j + x] & 0xffff0000u) * up;
            }
            if constexpr (KIND == Q8_INT8) {         // whole numbers of 16 bits, by bytes: high ones and low ones of four
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) w[x] = __float_as_uint(v[x] + 12582912.f);
              const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
              qf[n][j][0] = __byte_perm(a, b, 0x7632);
              qf[n][j][1] = __byte_perm(a, b, 0x5410);
            } else {
              qf[n][j][0] = pq_half2(v[0], v[1]);
              qf[n][j][1] = pq_half2(v[2], v[3]);
            }
          }
          const float down = top >= 0x7f80u ? NAN : scale_log2 * q8_pow2(-e);       // whole numbers keep no NaN, nor an infinity
          qs[n][0] = __shfl_sync(0xffffffffu, down, 8 * t);          // of heads 2t and 2t + 1: the columns this lane gets
          qs[n][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
        }
        sums.clear();
      }
      const int stage = i % STAGES;
      const uint8_t* codes = ring + stage * S::STAGE;
      const bool came = mbar_wait_timed(&s_full[warp][stage], i / STAGES & 1);
      if (!__all_sync(0xffffffffu, came)) {
        if (status) atomicMax(status, ST_TIMEOUT_FULL);
        s_abort = 1;
        break;
      }
      const int4 n0 = *reinterpret_cast<const int4*>(notes + i % PQ_NOTES);
      const float4 n1 = *reinterpret_cast<const float4*>(notes[i % PQ_NOTES].ks);
      const int seq = n0.x, tile = n0.y, len = n0.z, keys[2] = {n0.w & 0xff, n0.w >> 8};
      const float ks[2] = {n1.x, n1.y};
      float vs[2] = {n1.z, n1.w};
      const bool ends = tile + 1 == tiles_in(len);
      if (ends && i + 1 < tiles) request_q(notes[(i + 1) % PQ_NOTES].seq);

      // scores: rows are the keys g and g + 8 of a stretch, columns the heads 2t and 2t + 1
      float s[2][NT][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t kr[2][KW];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint8_t* p = codes + u * S::STRETCH + r * 8 * HD;
          if (HD == 32) {
            pq_take<8>(kr[r], p + k_at[0]);
          } else {
            pq_take<16>(kr[r], p + k_at[0]);
            if (HD == 128) pq_take<16>(kr[r] + KW / 2, p + k_at[1]);
          }
        }
        if constexpr (KIND == Q8_INT8) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < JT; j += 2) {
              pq_mma_s8<false>(hi, kr[0][j], kr[1][j], kr[0][j + 1], kr[1][j + 1], qf[n][j][0], qf[n][j + 1][0]);
              pq_mma_s8<true>(lo, kr[0][j], kr[1][j], kr[0][j + 1], kr[1][j + 1], qf[n][j][1], qf[n][j + 1][1]);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) s[u][n][x] = static_cast<float>(hi[x] * 256 + lo[x]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) s[u][n][x] = 0.f;
#pragma unroll
          for (int j = 0; j < JT; ++j) {
            uint32_t a0, a1, a2, a3;
            pq_widen<KIND>(kr[0][j], a0, a2);
            pq_widen<KIND>(kr[1][j], a1, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) pq_mma(s[u][n], a0, a1, a2, a3, qf[n][j][0], qf[n][j][1]);
          }
        }
      }
      uint32_t vr[2][4][VW];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) pq_take<VW * 4>(vr[u][r], codes + (2 + u) * S::STRETCH + (r >> 1) * 8 * HD + v_at[r & 1]);
      const int ahead = i + STAGES;
      if (ahead % PQ_ROUND == PQ_ROUND / 2) find(ahead + PQ_ROUND / 2 + lane);
      if (ahead % PQ_ROUND == PQ_ROUND * 3 / 4) place(ahead + PQ_ROUND / 4 + lane);
      if (ahead % PQ_ROUND == 0) note(ahead + lane);
      __syncwarp();
      if (lane == 0 && ahead < tiles) {
        const PqNote* n = notes + ahead % PQ_NOTES;
        bring(ahead, n->keys, n->row[0], n->row[1]);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float f0 = qs[n][0] * ks[u], f1 = qs[n][1] * ks[u];
          s[u][n][0] *= f0;
          s[u][n][1] *= f1;
          s[u][n][2] *= f0;
          s[u][n][3] *= f1;
        }
      if (keys[0] + keys[1] < PQ_KEYS) {            // a context's last tile; what lies behind it may be any bits
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (g + (x >> 1) * 8 >= keys[u]) s[u][n][x] = -INFINITY;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int w = 0; w < VW; ++w)
              if (2 * t + (r & 1) + (r >> 1) * 8 >= keys[u]) vr[u][r][w] = 0;
          if (keys[u] == 0) vs[u] = 0.f;
        }
      }
      bool moves = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          top[n][x] = fmaxf(fmaxf(s[0][n][x], s[0][n][2 + x]), fmaxf(s[1][n][x], s[1][n][2 + x]));
          moves |= top[n][x] > m[n][x] + PQ_SLACK;
        }
      // weights are relative to a reference that need not be the maximum: while no score passes it by more than 2^8, which
      // fp16 and the sums bear, it stays, and with it everything summed so far
      if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float mx = top[n][x];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(m[n][x], mx), f = mn == -INFINITY ? 0.f : pq_exp2(m[n][x] - mn);
            m[n][x] = mn;
            l[n][x] *= f;
#pragma unroll
            for (int j = 0; j < JT; ++j) {
              acc[n][j][x] *= f;
              acc[n][j][2 + x] *= f;
            }
          }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float r0 = m[n][0] == -INFINITY ? 0.f : m[n][0], r1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[u][n][0] = pq_exp2(s[u][n][0] - r0);
          s[u][n][1] = pq_exp2(s[u][n][1] - r1);
          s[u][n][2] = pq_exp2(s[u][n][2] - r0);
          s[u][n][3] = pq_exp2(s[u][n][3] - r1);
          l[n][0] += s[u][n][0] + s[u][n][2];
          l[n][1] += s[u][n][1] + s[u][n][3];
        }
      }
      // Adds a stretch's values.  Sums are held in units of a scale: a weight is multiplied by the ratio of its own block's scale
      // to the unit before it is rounded.  Rows of the product are hd / 8 neighbouring values per g, two to a product.
      auto add = [&](int u) {
        const float ratio = vs[u] * per_unit;
        uint32_t pf[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          pf[n][0] = pq_transpose(pq_half2(s[u][n][0] * ratio, s[u][n][1] * ratio));
          pf[n][1] = pq_transpose(pq_half2(s[u][n][2] * ratio, s[u][n][3] * ratio));
        }
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362 : 0x5140;
            uint32_t a0, a1, a2, a3;
            pq_widen<KIND>(__byte_perm(vr[u][0][w], vr[u][1][w], sel), a0, a1);
            pq_widen<KIND>(__byte_perm(vr[u][2][w], vr[u][3][w], sel), a2, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) pq_mma(acc[n][2 * w + half], a0, a1, a2, a3, pf[n][0], pf[n][1]);
          }
      };
      // The unit follows the scales when a ratio leaves [1/2, 64], so that weights keep their fp16 precision and range whatever the
      // scales of a sequence's blocks are.  It falls no further than the sums bear: a block of zeros has the least scale there is,
      // and one after the other they would take any sum out of fp32's range.  Beside sums of 2^118 units or more the weights of
      // smaller blocks are rounded to 2^-25 units.
      if (unit == 0.f) {
        unit = vs[0] != 0.f ? vs[0] : vs[1];
        per_unit = unit != 0.f ? rcp_approx(unit) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (!(vs[u] >= 0.5f * unit && vs[u] <= 64.f * unit) && vs[u] != 0.f) {
          float largest = 0.f;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) largest = fmaxf(largest, fabsf(acc[n][j][x]));       // not what is no number
          const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(largest));
          const int room = min(max(245 - static_cast<int>(top >> 23), 0), 126);                // sums stay below 2^119
          const float most = q8_pow2(room), f = fminf(unit * rcp_approx(vs[u]), most);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) acc[n][j][x] *= f;
          unit = f < most || top == 0 ? vs[u] : unit * q8_pow2(-room);
          per_unit = rcp_approx(unit);
        }
        add(u);
      }

      if (i + 1 == tiles || ends) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], o);
        if (piece_lo == 0 && ends) {
          sums.write(result(seq), unit, lane, G);
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < JT; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) acc[n][j][x] *= unit;
          const PqPiece piece{seq, len, lo + i - tile, piece_lo, tile + 1};
          if (i + 1 == tiles) {               // stays in registers
            open = true;
            last = piece;
          } else if (warp == 0) {             // the end of a sequence that an earlier CTA begins
            sums.template put<true>(slot(share, false), lane, G);
            owes = true;
            owed = piece;
          } else {                            // the end of one that an earlier warp begins
            sums.template put<false>(piece_at(warp), lane, G);
            if (lane == 0) s_goes_on[warp] = PQ_THEN_OTHERS;
          }
        }
        piece_lo = 0;                         // the next sequence begins with the next tile
        fresh = true;
      }
    }
  }
  pdl_launch_dependents();
  const bool follows = open && warp > 0 && last.lo > 0;        // a warp before this one begins it
  if (follows) {
    __syncwarp();
    sums.template put<false>(ring_at(warp), lane, G);          // where its tiles were
    if (lane == 0) s_goes_on[warp] = last.hi == tiles_in(last.len) ? PQ_TO_ITS_END : PQ_BEYOND;
  }
  __syncthreads();
  if (s_abort) {                              // no copy may outlive the CTA
    if (lane < STAGES) mbar_wait_timed(&s_full[warp][lane], 0, 100), mbar_wait_timed(&s_full[warp][lane], 1, 100);
    if (tid == 0) {                           // what was computed is lost, but the parts are counted as ever: the next launch finds zeros
      auto count_lost = [&](int seq, int len, int first) {
        if (count_part(seq, len, first).w) count[seq * Hkv + kvh] = 0;
      };
      int seq, len, first = locate(at, seq, len);
      if (first < at) count_lost(seq, len, first);
      first = locate(end - 1, seq, len);
      if (first >= at && first + tiles_in(len) > end) count_lost(seq, len, first);
    }
    return;
  }
  bool gives = false;
  if (open && !follows) {
    bool ended = last.hi == tiles_in(last.len);
#pragma unroll 1
    for (int w = warp + 1; w < PQ_WARPS && !ended; ++w) {
      const int how = s_goes_on[w];
      if (how == PQ_NOT) break;               // the CTA ends in it
      PqSums<NT, JT> o;
      o.template get<false>(how == PQ_THEN_OTHERS ? piece_at(w) : ring_at(w), lane, G);
      sums.add(o);
      ended = how != PQ_BEYOND;
    }
    if (ended && last.lo == 0) {
      sums.write(result(last.seq), 1.f, lane, G);
    } else {
      sums.template put<true>(slot(share, last.lo == 0), lane, G);
      gives = true;
    }
  }
  // lane 0: the part of a sequence that the CTA begins in the middle of, lane 1: of the one it ends in
  const bool middle = owes || (gives && last.lo > 0);
  __syncwarp();
  if (lane == 0 ? middle : lane == 1 && gives && last.lo == 0) {
    const PqPiece piece = lane == 0 && owes ? owed : last;
    const int4 counted = count_part(piece.seq, piece.len, piece.first);
    if (counted.w) s_part[lane] = counted;
  }
  __syncthreads();
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    if (!s_part[k].w) continue;
    const int seq = s_part[k].x, parts = s_part[k].z, stride = Hkv * 2 * SLOT;
    const float* part0 = slot(s_part[k].y, false);             // the first part lies behind it, the others there
    constexpr int BATCH = NT == 2 && HD > 32 ? 2 : NT * JT > 4 ? 3 : 4;      // parts whose loads are in flight, by registers
    // few parts are one warp's, the two sequences' then two warps'
    const int team = min(PQ_WARPS, (parts + BATCH - 1) / BATCH), me = (warp + PQ_WARPS - k) % PQ_WARPS;
    sums.clear();
    if (me < team) {
#pragma unroll 1
      for (int p = me; p < parts; p += team * BATCH) {
        PqSums<NT, JT> o[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
          const int which = p + b * team;
          o[b].clear();
          if (which < parts) o[b].template get<true>(part0 + static_cast<size_t>(which) * stride + (which == 0 ? SLOT : 0), lane, G);
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) sums.add(o[b]);
      }
    }
    if (team > 1) {
      if (me > 0 && me < team) sums.template put<false>(piece_at(me), lane, G);
      __syncthreads();
      if (me == 0) {
#pragma unroll 1
        for (int w = 1; w < team; ++w) {
          PqSums<NT, JT> o;
          o.template get<false>(piece_at(w), lane, G);
          sums.add(o);
        }
      }
    }
    if (me == 0) {
      sums.write(result(seq), 1.f, lane, G);
      if (lane == 0) count[seq * Hkv + kvh] = 0;               // as the next launch expects it
    }
    if (team > 1) __syncthreads();
  }
}

// whole shares: one CTA per kv head in each
static int pq_shares(int hd, int Hkv) {
  const int shares = sm_count() * pq_ctas_per_sm(hd) / Hkv;
  return shares < 1 ? 1 : shares;
}

static long pq_part_bytes(int Hq, int Hkv, int hd) {
  return static_cast<long>(pq_shares(hd, Hkv)) * Hkv * 2 * pq_piece_floats(pq_heads(Hq / Hkv), hd) * 4;
}

// The codes as rows of hd bytes, brought 16 at a time.
static int pq_map(CUtensorMap* map, const void* codes, long rows, int hd) {
  auto enc = get_tmap_encoder();
  if (!enc) return ERR_NO_DRIVER;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(hd)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(hd), 16}, steps[2] = {1, 1};
  const CUtensorMapSwizzle spread = hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : hd == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, steps,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, spread, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : ERR_TMAP;
}

}  // namespace artb

using namespace artb;

// Bytes of workspace: two parts per CTA, then counters [num_seqs * Hkv] (zero before the first call, zero again after each, one whose
// waits ran out too).  The counters lie behind what does not depend on the batch, so that a call with fewer sequences leaves those of a
// larger one alone.
ARTB_EXPORT int artb_paged_decode_q8_bytes(int num_seqs, int Hq, int Hkv, int hd) {
  if (num_seqs <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > 16) return 0;
  return static_cast<int>(pq_part_bytes(Hq, Hkv, hd) + (static_cast<long>(num_seqs) * Hkv + 3) / 4 * 16);
}

// q [num_seqs, ldq], out [num_seqs, ldo] bf16; block_table [num_seqs, max_blocks]; a context that its table row cannot hold is cut
// off, keys whose table entry is no block are left out, and both are reported through `status`.
ARTB_EXPORT int artb_paged_decode_q8(const PagedDecodeArgs* args, cudaStream_t st) {
  const auto [status, q, k_cache, v_cache, k_scale, v_scale, block_table, ctx_len, out, ws, num_blocks, num_seqs, ldq, ldo, Hq, Hkv, hd,
              block_size, max_blocks, kind] = *args;
  if (num_seqs <= 0) return 0;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 16 || block_size < 16 || (block_size & 15) || max_blocks < 1 || num_blocks < 1 || (ldq & 7) ||
      (ldo & 7) || !ws)
    return ERR_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(ws) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
       reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15)
    return ERR_BAD_ALIGN;
  if (num_blocks * Hkv * block_size > 0x7fffffffL) return ERR_TOO_LARGE;        // rows are numbered with 31 bits
  const long most = static_cast<long>(max_blocks) * block_size;                 // keys of a context, and so are all tiles
  if ((((most < 0x7fffffffL ? most : 0x7fffffffL) + PQ_KEYS - 1) / PQ_KEYS) * num_seqs > 0x7f000000L) return ERR_TOO_LARGE;
  int dev_ = 0;
  if (cudaGetDevice(&dev_) != cudaSuccess || dev_ < 0 || dev_ >= 64) return ERR_BAD_SHAPE;
  const float scale_log2 = 1.4426950408889634f / sqrtf((float)hd);
  float* part = static_cast<float*>(ws);
  int* count = reinterpret_cast<int*>(static_cast<char*>(ws) + pq_part_bytes(Hq, Hkv, hd));
  const int heads = pq_heads(Hq / Hkv);
  if (hd != 128 && hd != 64 && hd != 32) return ERR_BAD_SHAPE;
  const int shares = pq_shares(hd, Hkv), subs = block_size / 16, sub_shift = (subs & (subs - 1)) ? -1 : __builtin_ctz(subs);
  // 2^32 / shares, rounded up: a share is a product instead of a division, and never too small
  const uint32_t per_share = shares == 1 ? 0xffffffffu : static_cast<uint32_t>(((1ull << 32) + shares - 1) / shares);
  CUtensorMap k_map, v_map;
  int rc = pq_map(&k_map, k_cache, num_blocks * Hkv * block_size, hd);
  if (!rc) rc = pq_map(&v_map, v_cache, num_blocks * Hkv * block_size, hd);
  if (rc) return rc;
#define ARTB_PQ(KIND_, HD_, HEADS_)                                                                                           \
  if (kind == KIND_ && hd == HD_ && heads == HEADS_) {                                                                        \
    static bool cfgd[64] = {false};   /* the attribute is per device */                                                       \
    if (!cfgd[dev_]) {                                                                                                        \
      cudaError_t e = cudaFuncSetAttribute(paged_decode_q8_kernel<KIND_, HD_, HEADS_>, cudaFuncAttributeMaxDynamicSharedMemorySize, \
                                           PqSmem<HD_, HEADS_>::BYTES);                                                       \
      if (e != cudaSuccess) return static_cast<int>(e);                                                                       \
      cfgd[dev_] = true;                                                                                                      \
    }                                                                                                                         \
    return static_cast<int>(launch_ahead(paged_decode_q8_kernel<KIND_, HD_, HEADS_>, dim3(Hkv, shares), dim3(PQ_THREADS),       \
                                          PqSmem<HD_, HEADS_>::BYTES, st, k_map, v_map, (const __nv_bfloat16*)q, ldq,         \
                                          k_scale, v_scale, block_table, max_blocks, ctx_len, block_size, sub_shift, num_seqs, \
                                          Hq / Hkv, per_share, (__nv_bfloat16*)out, ldo, part, count, scale_log2, num_blocks, \
                                          status));                                                                           \
  }
#define ARTB_PQ_KIND(KIND_)                                                                                                   \
  ARTB_PQ(KIND_, 128, 8) ARTB_PQ(KIND_, 128, 16) ARTB_PQ(KIND_, 64, 8) ARTB_PQ(KIND_, 64, 16) ARTB_PQ(KIND_, 32, 8)           \
  ARTB_PQ(KIND_, 32, 16)
  ARTB_PQ_KIND(Q8_E4M3)
  ARTB_PQ_KIND(Q8_INT8)
#undef ARTB_PQ_KIND
#undef ARTB_PQ
  return ERR_BAD_SHAPE;
}
