// Decode attention over a paged cache held in 8 bits (numbers and layout: kv_q8.cuh): one new token per sequence,
//     o_h = sum_j softmax_j(q_h . k_j / sqrt(hd)) v_j,   j < ctx_len,   k_j, v_j = code * scale of the block and kv head.
//
// The G = Hq / Hkv query heads of a kv head are the columns of one m16n8 tile (two for G > 8), so that keys and values are
// read once for all of them.  Both products have the cache's side as their rows,
//     S^T [16 keys x heads] = K Q^T,     O^T [hd x heads] = V^T P^T,
// and 16 keys are always of one block: a scale is one factor of a score tile and of a value tile's product, and no code is
// ever multiplied by it.  Codes become fp16 (exact: e4m3 and int8 have at most 8 significant bits), queries too, after a power
// of two per head that brings their largest to 2^14 (exact but for what is 2^-38 of it); weights are rounded to fp16.
//
// No shared memory on the way in.  The order in which a product sums is free, so each lane loads the bytes that its own
// fragments need, in 16-byte pieces: hd / 4 neighbouring values of its keys, and hd / 8 neighbouring values of four keys, whose
// bytes are paired up in registers while they are widened.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "host_utils.h"
#include "kv_q8.cuh"

namespace artb {

constexpr int PQ_KEYS = 32;              // keys of a tile: two stretches of 16, each within a block
constexpr int PQ_MIN_TILES = 4;          // tiles of a CTA at least: one per warp
constexpr int PQ_LENS = 256;             // context lengths that a CTA keeps at hand
constexpr float PQ_SLACK = 8.f;          // how far (in powers of two) a score may pass the reference before that moves

__host__ __device__ constexpr int pq_heads(int G) { return G > 8 ? 16 : 8; }
// by registers: a warp holds 8 * PQ_KEYS / 32 * hd bytes of keys and values and hd * heads sums
__host__ __device__ constexpr int pq_ctas_per_sm(int hd, int heads) { return hd == 128 ? (heads == 8 ? 3 : 2) : hd == 64 && heads == 16 ? 3 : 4; }
__host__ __device__ constexpr int pq_piece_floats(int heads, int hd) { return heads * hd + ((2 * heads + 3) & ~3); }

template <int BYTES>
__device__ __forceinline__ void pq_load(uint32_t* r, const uint8_t* p) {
  if (BYTES == 4) {
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(r[0]) : "l"(p));
  } else if (BYTES == 8) {
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r[4 * i]), "=r"(r[4 * i + 1]), "=r"(r[4 * i + 2]), "=r"(r[4 * i + 3])
                   : "l"(p + 16 * i));
  }
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

__device__ __forceinline__ void pq_store4(__nv_bfloat16* dst, const float4& o, float sum) {
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const __nv_bfloat162 a = __floats2bfloat162_rn(o.x * inv, o.y * inv), b = __floats2bfloat162_rn(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// Where a warp stands in the tiles of all sequences.
struct PqAt {
  int seq, tile, len;
};

// What a warp leaves of a sequence that it has not read whole: tiles [lo, hi) of the sequence whose first tile is `first`.
struct PqPiece {
  int seq, len, first, lo, hi;
};

// The sequences are laid end to end, in tiles of PQ_KEYS keys, and cut into equal shares, wherever sequences begin and end in
// them; a share belongs to Hkv neighbouring CTAs, one per kv head, and the shares together fill the chip once.  A CTA's share is
// cut again into four, one per warp.  A warp goes through its tiles without a stop at the ends of sequences: keys of the next
// tile are requested as soon as the scores have been taken from those of this one, values once they have been added up, and
// table entries a tile before that.  A sequence that one warp reads whole is written by it.  The pieces of others meet in shared
// memory, and what still is a part then goes to the workspace; the CTA that finishes last adds the parts up in their order.
template <int KIND, int HD, int HEADS>
__global__ void __launch_bounds__(128, pq_ctas_per_sm(HD, HEADS))
paged_decode_q8_kernel(const __nv_bfloat16* __restrict__ q, int ldq, const uint8_t* __restrict__ k_cache,
                       const uint8_t* __restrict__ v_cache, const float* __restrict__ k_scale, const float* __restrict__ v_scale,
                       const int* __restrict__ block_table, int max_blocks, const int* __restrict__ ctx_len, int block_size,
                       int nseq, int Hq, int Hkv, __nv_bfloat16* __restrict__ out, int ldo, float* part, int* count,
                       float scale_log2, long num_blocks, int* status) {
  constexpr int NT = HEADS / 8, JT = HD / 16, KW = HD / 16, VW = HD / 32;
  constexpr int PF = pq_piece_floats(HEADS, HD);
  extern __shared__ __align__(16) float pq_smem[];          // [8 pieces][PF]: sums [HEADS][HD], reference [HEADS], sum [HEADS]
  __shared__ int s_warp[4], s_len[PQ_LENS], s_done;
  __shared__ PqAt s_start[4];
  __shared__ int s_first[4];
  __shared__ PqPiece s_piece[8];
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = Hq / Hkv, shares = gridDim.x / Hkv, share = blockIdx.x / Hkv, kvh = blockIdx.x - share * Hkv;
  const int table_keys = min(static_cast<long>(max_blocks) * block_size, 0x7fffffffL - PQ_KEYS);
  auto length = [&](int i) {
    int n = ctx_len[i];
    if (n > table_keys) {
      if (blockIdx.x == 0 && status) atomicMax(status, ST_BOUNDS);
      n = table_keys;
    }
    return max(n, 0);
  };
  auto tiles_in = [](int len) { return (len + PQ_KEYS - 1) / PQ_KEYS; };

  // where the share begins: each thread sums the tiles of a run of sequences, then a scan over the threads
  const int run = (nseq + 127) / 128, i0 = min(nseq, tid * run), i1 = min(nseq, i0 + run);
  int own = 0;
  for (int i = i0; i < i1; ++i) {
    const int len = length(i);
    own += tiles_in(len);
    if (len == 0 && share == shares - 1) {           // an empty context (the padding of a batch): zeros
      uint4* o = reinterpret_cast<uint4*>(out + static_cast<size_t>(i) * ldo + kvh * G * HD);
      for (int d = 0; d < G * HD / 8; ++d) o[d] = make_uint4(0, 0, 0, 0);
    }
  }
  int incl = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_warp[warp] = incl;
  if (tid < 8) s_piece[tid].seq = -1;
  __syncthreads();
  int total = 0, before = incl - own;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  const int per = max(PQ_MIN_TILES, (total + shares - 1) / shares), per_warp = (per + 3) / 4;
  const int at = share * per;
  if (at >= total) return;                  // the whole CTA
  const int end = min(total, at + per);
  for (int w = 0; w < 4; ++w) {
    const int x = at + w * per_warp;
    if (x < end && before <= x && x < before + own) {
      int i = i0, b = before, len;
      for (;; ++i) {
        len = length(i);
        const int n = tiles_in(len);
        if (x < b + n) break;
        b += n;
      }
      s_start[w] = PqAt{i, x - b, len};
      s_first[w] = b;
    }
  }
  __syncthreads();
  const int seq0 = s_start[0].seq;
  for (int i = tid; i < PQ_LENS; i += 128) s_len[i] = seq0 + i < nseq ? length(seq0 + i) : 0x7fffffff - PQ_KEYS;
  __syncthreads();

  const int lo = at + warp * per_warp, count_tiles = min(end, lo + per_warp) - lo;
  if (count_tiles > 0) {
    const int subs = block_size / 16, sub_shift = (subs & (subs - 1)) == 0 ? 31 - __clz(subs) : -1;
    auto next = [&](PqAt x) {
      if (++x.tile * PQ_KEYS >= x.len) {
        x.tile = 0;
        do {
          ++x.seq;
          x.len = x.seq - seq0 < PQ_LENS ? s_len[x.seq - seq0] : x.seq < nseq ? length(x.seq) : 0x7fffffff - PQ_KEYS;
        } while (x.len <= 0);
      }
      return x;
    };
    // the blocks of a tile's two stretches; the second may have no keys, and is then read where the first lies
    auto blocks_of = [&](const PqAt& x, bool any, int (&blk)[2]) {
      const int* row = block_table + static_cast<size_t>(x.seq) * max_blocks;
      const int last = (x.len - 1) >> 4;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int sb = min(x.tile * 2 + s, last);
        blk[s] = any ? __ldcg(row + (sub_shift >= 0 ? sb >> sub_shift : sb / subs)) : 0;
      }
    };
    uint32_t kr[2][2][KW], vr[2][4][VW];
    float ks[2], vs[2], ks_next[2], vs_next[2];
    int keys[2], keys_next[2];                      // of each stretch: 16, fewer at a context's end, 0 where its block is none
    size_t off[2];                                  // of the stretch that is being requested, in the codes of keys and of values
    uint32_t head[2];                               // and its scale
    const uint8_t* k_lane = k_cache + g * HD + t * (HD / 4);
    const uint8_t* v_lane = v_cache + 2 * t * HD + g * (HD / 8);
    auto load_k = [&](const PqAt& x, const int (&blk)[2], int (&n)[2], float (&scale)[2]) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int sb = min(x.tile * 2 + s, (x.len - 1) >> 4);
        const bool good = static_cast<unsigned>(blk[s]) < static_cast<unsigned long>(num_blocks);
        if (!good && status) atomicMax(status, ST_BOUNDS);
        n[s] = good ? max(0, min(16, x.len - (x.tile * 2 + s) * 16)) : 0;
        head[s] = static_cast<uint32_t>(good ? blk[s] : 0) * Hkv + kvh;
        off[s] = static_cast<size_t>(head[s]) * (block_size * HD) + (sb - (sub_shift >= 0 ? sb >> sub_shift << sub_shift : sb / subs * subs)) * (16 * HD);
        pq_load<HD / 4>(kr[s][0], k_lane + off[s]);
        pq_load<HD / 4>(kr[s][1], k_lane + off[s] + 8 * HD);
        scale[s] = __ldcg(k_scale + head[s]);
      }
    };
    auto load_v = [&](float (&scale)[2]) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        pq_load<HD / 8>(vr[s][0], v_lane + off[s]);
        pq_load<HD / 8>(vr[s][1], v_lane + off[s] + HD);
        pq_load<HD / 8>(vr[s][2], v_lane + off[s] + 8 * HD);
        pq_load<HD / 8>(vr[s][3], v_lane + off[s] + 9 * HD);
        scale[s] = __ldcg(v_scale + head[s]);
      }
    };

    PqAt a = s_start[warp];
    int blk_next[2], first = s_first[warp], piece_lo = a.tile;
    {
      int blk[2];
      blocks_of(a, true, blk);
      load_k(a, blk, keys, ks);
      load_v(vs);
    }
    PqAt b = next(a);
    blocks_of(b, count_tiles > 1, blk_next);

    uint32_t qf[NT][JT][2];
    float qs[NT][2], m[NT][2], l[NT][2], acc[NT][JT][4], unit, per_unit;
    bool fresh = true;
    for (int i = 0; i < count_tiles; ++i) {
      if (fresh) {
        fresh = false;
        unit = per_unit = 0.f;
        // heads g (and g + 8), hd / 4 values from t * hd / 4 on: the order in which the lanes hold the keys
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t raw[JT * 2], top = 0;
          const int head = n * 8 + g;
          const __nv_bfloat16* row = q + static_cast<size_t>(a.seq) * ldq + (kvh * G + head) * HD + t * (HD / 4);
#pragma unroll
          for (int v = 0; v < JT * 2 / 4; ++v) {
            const uint4 x = head < G ? __ldcg(reinterpret_cast<const uint4*>(row) + v) : make_uint4(0, 0, 0, 0);
            raw[4 * v] = x.x;
            raw[4 * v + 1] = x.y;
            raw[4 * v + 2] = x.z;
            raw[4 * v + 3] = x.w;
          }
#pragma unroll
          for (int v = 0; v < JT * 2; ++v) top = __vmaxu2(top, raw[v] & 0x7fff7fffu);
          top = max(top & 0xffffu, top >> 16);
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int e = top >= 0x7f80u || top == 0 ? 0 : min(100, 14 + 127 - static_cast<int>(top >> 7));
          const float up = q8_pow2(e);
#pragma unroll
          for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              qf[n][j][x] = pq_half2(__uint_as_float(raw[2 * j + x] << 16) * up, __uint_as_float(raw[2 * j + x] & 0xffff0000u) * up);
          const float down = scale_log2 * q8_pow2(-e);
          qs[n][0] = __shfl_sync(0xffffffffu, down, 8 * t);          // of heads 2t and 2t + 1: the columns this lane gets
          qs[n][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
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
      const PqAt c = next(b);
      int blk_after[2];
      blocks_of(c, i + 2 < count_tiles, blk_after);

      // scores: rows are the keys g and g + 8 of a stretch, columns the heads 2t and 2t + 1
      float s[2][NT][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[u][n][x] = 0.f;
#pragma unroll
        for (int j = 0; j < JT; ++j) {
          uint32_t a0, a1, a2, a3;
          pq_widen<KIND>(kr[u][0][j], a0, a2);
          pq_widen<KIND>(kr[u][1][j], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) pq_mma(s[u][n], a0, a1, a2, a3, qf[n][j][0], qf[n][j][1]);
        }
      }
      if (i + 1 < count_tiles) load_k(b, blk_next, keys_next, ks_next);
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
      // The unit follows the scales when a ratio leaves [1/2, 64], so that weights keep their fp16 precision and range whatever
      // the scales of a sequence's blocks are.
      auto fits = [&](float x) { return (x >= 0.5f * unit && x <= 64.f * unit) || x == 0.f; };
      if (fits(vs[0]) && fits(vs[1])) {
        add(0);
        add(1);
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (!fits(vs[u])) {
            const float f = fminf(unit / vs[u], 1.2e27f);    // 2^90: beside sums that large a weight is nothing
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < JT; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[n][j][x] *= f;
            unit = unit == 0.f ? vs[u] : unit / f;
            per_unit = 1.f / unit;
          }
          add(u);
        }
      }
      if (i + 1 < count_tiles) load_v(vs_next);

      const int tiles = tiles_in(a.len);
      if (i + 1 == count_tiles || a.tile + 1 == tiles) {
        const bool whole = piece_lo == 0 && a.tile + 1 == tiles;
        const int where = warp * 2 + (piece_lo == 0);
        float* piece = pq_smem + where * PF;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float sum = l[n][x];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const int head = n * 8 + 2 * t + x;
#pragma unroll
            for (int j = 0; j < JT; ++j) {
              acc[n][j][x] *= unit;
              acc[n][j][2 + x] *= unit;
            }
            if (whole) {
              if (head < G) {
                __nv_bfloat16* o_row = out + static_cast<size_t>(a.seq) * ldo + (kvh * G + head) * HD + g * (HD / 8);
#pragma unroll
                for (int j = 0; j < JT; j += 2)
                  pq_store4(o_row + 2 * j, make_float4(acc[n][j][x], acc[n][j][2 + x], acc[n][j + 1][x], acc[n][j + 1][2 + x]), sum);
              }
            } else {
              float* dst = piece + head * HD + g * (HD / 8);
#pragma unroll
              for (int j = 0; j < JT; j += 2)
                *reinterpret_cast<float4*>(dst + 2 * j) = make_float4(acc[n][j][x], acc[n][j][2 + x], acc[n][j + 1][x], acc[n][j + 1][2 + x]);
              if (g == 0) {
                piece[HEADS * HD + head] = m[n][x];
                piece[HEADS * HD + HEADS + head] = sum;
              }
            }
          }
        if (!whole && lane == 0) s_piece[where] = PqPiece{a.seq, a.len, first, piece_lo, a.tile + 1};
        first = lo + i + 1;                   // the next sequence begins with the next tile
        piece_lo = 0;
        fresh = true;
      }
      a = b;
      b = c;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        keys[u] = keys_next[u];
        blk_next[u] = blk_after[u];
        ks[u] = ks_next[u];
        vs[u] = vs_next[u];
      }
    }
  }
  pdl_launch_dependents();
  __syncthreads();

  // the pieces in their order: neighbours of one sequence are added up
  for (int p0 = 0; p0 < 8;) {
    const PqPiece head_piece = s_piece[p0];
    if (head_piece.seq < 0) {
      ++p0;
      continue;
    }
    int p1 = p0 + 1, hi = head_piece.hi;
    for (int p = p0 + 1; p < 8; ++p) {
      if (s_piece[p].seq < 0) continue;
      if (s_piece[p].seq != head_piece.seq) break;
      hi = s_piece[p].hi;
      p1 = p + 1;
    }
    const int seq = head_piece.seq, first = head_piece.first, tiles = tiles_in(head_piece.len);
    const bool whole = head_piece.lo == 0 && hi == tiles;
    __nv_bfloat16* o_row = out + static_cast<size_t>(seq) * ldo + kvh * G * HD;
    // a CTA leaves at most two parts: of the sequence that it begins in the middle of, and of the one it ends in
    const int slot_floats = pq_piece_floats(G, HD);
    auto slot = [&](int sh, bool starts) { return part + static_cast<size_t>((sh * Hkv + kvh) * 2 + starts) * slot_floats; };
    float* w = slot(share, head_piece.lo == 0);
    for (int idx = tid; idx < G * (HD / 4); idx += 128) {
      const int r = idx / (HD / 4);
      float mm = -INFINITY, sum = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int p = p0; p < p1; ++p)
        if (s_piece[p].seq >= 0) mm = fmaxf(mm, pq_smem[p * PF + HEADS * HD + r]);
      for (int p = p0; p < p1; ++p) {
        if (s_piece[p].seq < 0) continue;
        const float* x = pq_smem + p * PF;
        const float mp = x[HEADS * HD + r], f = mp == -INFINITY ? (x[HEADS * HD + HEADS + r] == 0.f ? 0.f : 1.f) : pq_exp2(mp - mm);
        const float4 v = *reinterpret_cast<const float4*>(x + idx * 4);
        sum = fmaf(x[HEADS * HD + HEADS + r], f, sum);
        o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
      }
      if (whole) {
        pq_store4(o_row + idx * 4, o, sum);
      } else {
        *reinterpret_cast<float4*>(w + idx * 4) = o;
        if (idx * 4 == r * HD) {
          w[G * HD + r] = mm;
          w[G * HD + G + r] = sum;
        }
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      const int sh0 = first / per, parts = (first + tiles - 1) / per - sh0 + 1;
      if (tid == 0) s_done = atomicAdd(&count[seq * Hkv + kvh], 1) == parts - 1;
      __syncthreads();
      if (s_done) {
        __threadfence();
        for (int idx = tid; idx < G * HD / 4; idx += 128) {
          const int r = idx / (HD / 4);
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
          float mx = -INFINITY, sum = 0.f;
          for (int q0 = 0; q0 < parts; q0 += 8) {          // eight parts' loads in flight
            float m[8], l[8];
            float4 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float* sl = slot(sh0 + min(q0 + j, parts - 1), q0 + j == 0);
              m[j] = __ldcg(sl + G * HD + r);
              l[j] = __ldcg(sl + G * HD + G + r);
              v[j] = __ldcg(reinterpret_cast<const float4*>(sl) + idx);
            }
            float mn = mx;
#pragma unroll
            for (int j = 0; j < 8; ++j) mn = fmaxf(mn, q0 + j < parts ? m[j] : -INFINITY);
            const float c = mx == -INFINITY ? 1.f : pq_exp2(mx - mn);        // nothing yet, or what has no reference
            mx = mn;
            o = make_float4(o.x * c, o.y * c, o.z * c, o.w * c);
            sum *= c;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float f = q0 + j >= parts ? 0.f : m[j] == -INFINITY ? (l[j] == 0.f ? 0.f : 1.f) : pq_exp2(m[j] - mn);
              if (f != 0.f) {
                sum = fmaf(l[j], f, sum);
                o = make_float4(fmaf(v[j].x, f, o.x), fmaf(v[j].y, f, o.y), fmaf(v[j].z, f, o.z), fmaf(v[j].w, f, o.w));
              }
            }
          }
          pq_store4(o_row + idx * 4, o, sum);
        }
        if (tid == 0) count[seq * Hkv + kvh] = 0;            // as the next launch expects it
      }
      __syncthreads();                                       // s_done is read before the next part sets it
    }
    p0 = p1;
  }
}

template <int HD, int HEADS>
constexpr int pq_smem_bytes() {
  return 8 * pq_piece_floats(HEADS, HD) * 4;
}

// whole shares: one CTA per kv head in each
static int pq_grid(int hd, int Hq, int Hkv) {
  const int shares = sm_count() * pq_ctas_per_sm(hd, pq_heads(Hq / Hkv)) / Hkv;
  return (shares < 1 ? 1 : shares) * Hkv;
}

static long pq_part_bytes(int Hq, int Hkv, int hd) {
  return (static_cast<long>(pq_grid(hd, Hq, Hkv)) * 2 * pq_piece_floats(Hq / Hkv, hd) * 4 + 15) / 16 * 16;
}

}  // namespace artb

using namespace artb;

// Bytes of workspace: two parts per CTA, then counters [num_seqs * Hkv] (zero before the first call, zero again after each).  The
// counters lie behind what does not depend on the batch, so that a call with fewer sequences leaves those of a larger one alone.
ARTB_EXPORT int artb_paged_decode_q8_bytes(int num_seqs, int Hq, int Hkv, int hd) {
  if (num_seqs <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || Hq / Hkv > 16) return 0;
  return static_cast<int>(pq_part_bytes(Hq, Hkv, hd) + (static_cast<long>(num_seqs) * Hkv + 3) / 4 * 16);
}

// q [num_seqs, ldq], out [num_seqs, ldo] bf16; block_table [num_seqs, max_blocks]; a context that its table row cannot hold is cut
// off, keys whose table entry is no block are left out, and both are reported through `status`.
ARTB_EXPORT int artb_paged_decode_q8(const void* q, int ldq, const void* k_cache, const void* v_cache, const float* k_scale,
                                     const float* v_scale, const int* block_table, int max_blocks, const int* ctx_len,
                                     int block_size, int num_seqs, int Hq, int Hkv, int hd, void* out, int ldo, void* ws,
                                     long num_blocks, int kind, int* status, cudaStream_t st) {
  if (num_seqs <= 0) return 0;
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 16 || block_size < 16 || (block_size & 15) || max_blocks < 1 || num_blocks < 1 || (ldq & 7) ||
      (ldo & 7) || !ws)
    return ERR_BAD_SHAPE;
  if ((reinterpret_cast<uintptr_t>(ws) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
       reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15)
    return ERR_BAD_ALIGN;
  int dev_ = 0;
  if (cudaGetDevice(&dev_) != cudaSuccess || dev_ < 0 || dev_ >= 64) return ERR_BAD_SHAPE;
  const float scale_log2 = 1.4426950408889634f / sqrtf((float)hd);
  float* part = static_cast<float*>(ws);
  int* count = reinterpret_cast<int*>(static_cast<char*>(ws) + pq_part_bytes(Hq, Hkv, hd));
  const int heads = pq_heads(Hq / Hkv);
#define ARTB_PQ(KIND_, HD_, HEADS_)                                                                                           \
  if (kind == KIND_ && hd == HD_ && heads == HEADS_) {                                                                        \
    static bool cfgd[64] = {false};   /* the attribute is per device */                                                       \
    if (!cfgd[dev_]) {                                                                                                        \
      cudaError_t e = cudaFuncSetAttribute(paged_decode_q8_kernel<KIND_, HD_, HEADS_>, cudaFuncAttributeMaxDynamicSharedMemorySize, \
                                           pq_smem_bytes<HD_, HEADS_>());                                                     \
      if (e != cudaSuccess) return static_cast<int>(e);                                                                       \
      cfgd[dev_] = true;                                                                                                      \
    }                                                                                                                         \
    return static_cast<int>(launch_kernel(paged_decode_q8_kernel<KIND_, HD_, HEADS_>, dim3(pq_grid(HD_, Hq, Hkv)), dim3(128), \
                                          pq_smem_bytes<HD_, HEADS_>(), st, (const __nv_bfloat16*)q, ldq,                     \
                                          (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale, block_table,    \
                                          max_blocks, ctx_len, block_size, num_seqs, Hq, Hkv, (__nv_bfloat16*)out, ldo, part, \
                                          count, scale_log2, num_blocks, status));                                            \
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
