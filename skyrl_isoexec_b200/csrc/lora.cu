// Low-rank adapters of many requests beside a shared projection, with their gradients.
//
//   forward     h[t] = s_a (x[t] A_a^T),   out[t] = y[t] + h[t] B_a^T        a = adapter of token t
//   backward    g[t] = s_a (dy[t] B_a),    dx[t] = g[t] A_a (+ base),        dA_a = sum_t g[t]^T x[t],   dB_a = sum_t dy[t]^T h[t]
//
// x [T, K], y / dy [T, N], A [E, r, K], B [E, N, r] bf16, s [E] fp32; r is a multiple of 8 up to 128. Tokens without an
// adapter keep y (dx: base or zero).
//
// The rank is small, so every one of these products is bound by reading and writing the token rows. The forward is one
// kernel: a cluster of CTAs owns a tile of 16 or 64 tokens of ONE adapter, its warps split K, the partial h are summed in
// a fixed order through shared and distributed shared memory, and the same warps split N to add h B^T to y. x is read
// once, y read and out written once, h never goes through memory on the way. The backward's g and dx are the same kernel
// with the factors read across their rows. h and g are kept in 32 bits until they become operands of the second product:
// there each is the sum of two bf16 numbers (its rounding and the rest, 16 bits together), so the only rounding to 8 bits
// that shows is that of the output (parts that carry all 24 bits move as many results over a rounding border: the 32-bit sums'
// order does). Products run on mma.sync (532 TFLOP/s here; rank 16 needs 105 of them at the copy rate,
// rank 64 420): with N or K of 8 to 128 a tcgen05 tile is mostly empty, and rows may lie anywhere. Small tiles take operands
// straight from global memory in fragments of 16 bytes a lane: a contraction may take its elements in any order as long as
// both operands agree, so a lane's 8 neighbours feed two products of depth 16.
//
// Measured (6.54 TB/s is a copy): 48 tokens of 32 adapters, 4096 -> 6144, rank 16: 7.8 us, of which 5 are the latency of one
// token's; 8192 tokens, 4096 -> 24576, rank 16: 163 us, 5.3 TB/s; dx the other way 105 us, 4.5 TB/s; dB 81 us, 5.0 TB/s;
// 4093 tokens, 4096 -> 4096, rank 64: 34 us, 3.2 TB/s, bound by shared memory and the two products of each h; 8192 tokens of 4
// adapters, 4096 -> 4096, rank 128: 114 us.
#include "bw_common.cuh"
#include "host_util.h"

#include <cooperative_groups.h>

namespace {
using namespace bw;
namespace cg = cooperative_groups;

constexpr int kMaxAdapters = 1024;
constexpr int kMaxRank = 128;
constexpr int kSmall = 16, kLarge = 64;      // tokens a tile

// ------------------------------------------------------------------------------------------------ plan
// Stable counting sort of the tokens by adapter (out of range: behind all others) and the tiles of both sizes.
// One CTA; warp w owns tokens [w per, (w+1) per), so a token's place depends on the ids alone.
__global__ void __launch_bounds__(1024)
lora_plan_kernel(const int* __restrict__ ids, int T, int E, int* __restrict__ perm, int* __restrict__ offsets, int4* __restrict__ tiles_s,
                 int4* __restrict__ tiles_l, int* __restrict__ n_tiles) {
  extern __shared__ int sm[];                // [warps][E + 1] counts, then first places
  const int G = E + 1, W = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* total = sm + W * G;                   // [G]
  for (int i = threadIdx.x; i < W * G; i += blockDim.x) sm[i] = 0;
  __syncthreads();
  const int per = ((T + W - 1) / W + 31) & ~31;
  const int lo = min(T, warp * per), hi = min(T, lo + per);
  int* mine = sm + warp * G;
  for (int i = lo; i < hi; i += 32) {
    const bool in = i + lane < hi;
    int a = in ? ids[i + lane] : -2;
    if (in && (a < 0 || a >= E)) a = E;
    const unsigned same = __match_any_sync(0xffffffffu, a);
    if (in && (same & ((1u << lane) - 1)) == 0) mine[a] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int a = threadIdx.x; a < G; a += blockDim.x) {
    int run = 0;
    for (int w = 0; w < W; ++w) {
      const int c = sm[w * G + a];
      sm[w * G + a] = run;
      run += c;
    }
    total[a] = run;
  }
  __syncthreads();
  __shared__ int s_off[kMaxAdapters + 2], s_ts[kMaxAdapters + 2], s_tl[kMaxAdapters + 2];
  if (warp == 0) {                           // first token and first tiles of every group
    int c0 = 0, c1 = 0, c2 = 0;
    for (int a0 = 0; a0 < G; a0 += 32) {
      const int a = a0 + lane;
      const int n = a < G ? total[a] : 0;
      int v0 = n, v1 = (n + kSmall - 1) / kSmall, v2 = (n + kLarge - 1) / kLarge;
      const int u0 = v0, u1 = v1, u2 = v2;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int w0 = __shfl_up_sync(0xffffffffu, v0, d), w1 = __shfl_up_sync(0xffffffffu, v1, d), w2 = __shfl_up_sync(0xffffffffu, v2, d);
        if (lane >= d) v0 += w0, v1 += w1, v2 += w2;
      }
      if (a < G) s_off[a] = c0 + v0 - u0, s_ts[a] = c1 + v1 - u1, s_tl[a] = c2 + v2 - u2;
      c0 += __shfl_sync(0xffffffffu, v0, 31), c1 += __shfl_sync(0xffffffffu, v1, 31), c2 += __shfl_sync(0xffffffffu, v2, 31);
    }
    if (lane == 0) s_off[G] = c0, n_tiles[0] = c1, n_tiles[1] = c2;
  }
  __syncthreads();
  for (int a = threadIdx.x; a <= G; a += blockDim.x) offsets[a] = s_off[a];
  for (int i = lo; i < hi; i += 32) {
    const bool in = i + lane < hi;
    int a = in ? ids[i + lane] : -2;
    if (in && (a < 0 || a >= E)) a = E;
    const unsigned same = __match_any_sync(0xffffffffu, a);
    const int before = __popc(same & ((1u << lane) - 1));
    int at = 0;
    if (in) at = mine[a];
    __syncwarp();
    if (in && before == 0) mine[a] = at + __popc(same);
    __syncwarp();
    if (in) perm[s_off[a] + at + before] = i + lane;
  }
  // tiles: (adapter or -1, first place in perm, tokens)
  for (int a = warp; a < G; a += W) {
    const int n = total[a], o = s_off[a], id = a < E ? a : -1;
    for (int i = lane; i * kSmall < n; i += 32) tiles_s[s_ts[a] + i] = make_int4(id, o + i * kSmall, min(kSmall, n - i * kSmall), 0);
    for (int i = lane; i * kLarge < n; i += 32) tiles_l[s_tl[a] + i] = make_int4(id, o + i * kLarge, min(kLarge, n - i * kLarge), 0);
  }
}

// ------------------------------------------------------------------------------------------------ fragments
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint4 ld16(const __nv_bfloat16* p, bool ok) {
  return ok ? *reinterpret_cast<const uint4*>(p) : make_uint4(0u, 0u, 0u, 0u);
}
// x = hi + lo, two bf16 numbers; packed pairs. An infinite number leaves no rest (infinity less infinity is none)
__device__ __forceinline__ float rest_of(float x, float hi) { return fabsf(hi) < INFINITY ? x - hi : 0.f; }
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const __nv_bfloat162 l = __floats2bfloat162_rn(rest_of(x, __low2float(h)), rest_of(y, __high2float(h)));
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

struct ApplyArgs {
  const __nv_bfloat16* in;        // [T, K] rows that are contracted (x, or dy)
  const __nv_bfloat16* base;      // [T, N] added to (y, or the other part of dx); null: nothing
  __nv_bfloat16* out;             // [T, N]; null: only h is wanted
  const __nv_bfloat16* down;      // factor of the first product: [E, r, K], or across: [E, K, r]
  const __nv_bfloat16* up;        // factor of the second: [E, N, r], or across: [E, r, N]
  const float* scale;             // [E]
  const int* perm;
  const int4* tiles;
  const int* n_tiles;
  __nv_bfloat16* h;               // [2, T, r] in the plan's order: s h as a bf16 and the rest; may be null
  long long ld_in, ld_base, ld_out;
  int T, K, N, r;
};

constexpr int kWarps = 8;
// shared memory: partial sums [kWarps][16][8 RT + 4] fp32, their sum [16][8 RT + 4], a warp's 2 KB for factors that are
// read across
template <int RT>
constexpr int apply_smem(bool across) {
  return (kWarps + 1) * 16 * (8 * RT + 4) * 4 + (across ? kWarps * 2048 : 0);
}

// Small tiles: 16 tokens of one adapter. RT: rank in groups of 8 (r <= 8 RT); ACROSS: factors stored with the contracted
// index outermost for the first product and innermost for the second (the backward).
template <int RT, bool ACROSS>
__global__ void __launch_bounds__(kWarps * 32) lora_apply_kernel(const __grid_constant__ ApplyArgs p) {
  constexpr int LD = 8 * RT + 4;                       // floats a row of h
  constexpr int KS = RT < 2 ? 1 : RT / 2;              // depth-16 steps over the rank
  extern __shared__ __align__(16) float smem[];
  if (blockIdx.y >= p.n_tiles[0]) return;              // the same for the whole cluster
  const int4 tile = p.tiles[blockIdx.y];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int c = gridDim.x, rank_cta = blockIdx.x;
  const int parts = kWarps * c, part = rank_cta * kWarps + warp;
  const int r0 = g, r1 = r0 + 8;             // rows of the tile held by this lane
  const bool ok0 = r0 < tile.z, ok1 = r1 < tile.z;
  const long long row0 = p.perm[tile.y + (ok0 ? r0 : 0)], row1 = p.perm[tile.y + (ok1 ? r1 : 0)];
  const int chunks = (p.N + 31) >> 5;
  const int n_lo = static_cast<int>(static_cast<long long>(chunks) * part / parts), n_hi = static_cast<int>(static_cast<long long>(chunks) * (part + 1) / parts);

  if (tile.x < 0) {                                    // no adapter: the base alone
    if (p.out == nullptr || p.out == p.base) return;
    for (int n = n_lo; n < n_hi; ++n) {
      const int col = n * 32 + 8 * t;
      if (col >= p.N) break;
      if (ok0) *reinterpret_cast<uint4*>(p.out + row0 * p.ld_out + col) = ld16(p.base + row0 * p.ld_base + col, p.base != nullptr);
      if (ok1) *reinterpret_cast<uint4*>(p.out + row1 * p.ld_out + col) = ld16(p.base + row1 * p.ld_base + col, p.base != nullptr);
    }
    return;
  }

  // ---- first product: this warp's part of K
  float acc[RT][4];
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
  const int steps = (p.K + 31) >> 5;
  const int k_lo = static_cast<int>(static_cast<long long>(steps) * part / parts), k_hi = static_cast<int>(static_cast<long long>(steps) * (part + 1) / parts);
  const __nv_bfloat16* x0 = p.in + row0 * p.ld_in;
  const __nv_bfloat16* x1 = p.in + row1 * p.ld_in;
  const __nv_bfloat16* down = p.down + static_cast<size_t>(tile.x) * p.r * p.K;
  const uint32_t scratch = smem_u32(smem + (kWarps + 1) * 16 * LD) + warp * 2048;
#pragma unroll 2
  for (int s = k_lo; s < k_hi; ++s) {
    const int k = s * 32 + 8 * t;
    const bool in = k < p.K;
    const uint4 a = ld16(x0 + k, in), b = ld16(x1 + k, in);
    if constexpr (!ACROSS) {
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        const uint4 f = ld16(down + static_cast<size_t>(8 * j + g) * p.K + k, in && (RT <= 2 || 8 * j < p.r));
        mma16816(acc[j], a.x, b.x, a.y, b.y, f.x, f.y);
        mma16816(acc[j], a.z, b.z, a.w, b.w, f.z, f.w);
      }
    } else {
      // rows of the factor are k: lane l brings row l. Matrix i of a transposed read holds the rows with the same place
      // among a lane's pairs, so that the products get the same k as above
      const int kr = s * 32 + lane;
      const uint32_t put = scratch + ((((lane >> 1) & 3) * 8 + 2 * (lane >> 3) + (lane & 1)) << 4);
#pragma unroll
      for (int j0 = 0; j0 < RT; j0 += 4) {
        __syncwarp();
#pragma unroll
        for (int j = j0; j < (RT < j0 + 4 ? RT : j0 + 4); ++j) {
          const uint4 f = ld16(down + static_cast<size_t>(kr) * p.r + 8 * j, kr < p.K && (RT <= 2 || 8 * j < p.r));
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(put + (j - j0) * 512), "r"(f.x), "r"(f.y), "r"(f.z), "r"(f.w) : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int j = j0; j < (RT < j0 + 4 ? RT : j0 + 4); ++j) {
          uint32_t f[4];
          ldsm4t(scratch + (j - j0) * 512 + lane * 16, f);
          mma16816(acc[j], a.x, b.x, a.y, b.y, f[0], f[1]);
          mma16816(acc[j], a.z, b.z, a.w, b.w, f[2], f[3]);
        }
      }
    }
  }

  // ---- h: sum over the warps, then over the cluster, both in order
  float* sum = smem + kWarps * 16 * LD;
  {
    float* mine = smem + warp * 16 * LD;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      const bool real = RT <= 2 || 8 * j < p.r;        // ranks that only fill up are zero, not 0 times an infinite x
      *reinterpret_cast<float2*>(mine + r0 * LD + 8 * j + 2 * t) = real ? make_float2(acc[j][0], acc[j][1]) : make_float2(0.f, 0.f);
      *reinterpret_cast<float2*>(mine + r1 * LD + 8 * j + 2 * t) = real ? make_float2(acc[j][2], acc[j][3]) : make_float2(0.f, 0.f);
    }
  }
  __syncthreads();
  const float sc = p.scale[tile.x];
  constexpr int kVals = 16 * 8 * RT;
  for (int i = threadIdx.x * 4; i < kVals; i += kWarps * 32 * 4) {
    const int at = (i / (8 * RT)) * LD + i % (8 * RT);
    float4 v = *reinterpret_cast<const float4*>(smem + at);
#pragma unroll
    for (int q = 1; q < kWarps; ++q) {
      const float4 w = *reinterpret_cast<const float4*>(smem + q * 16 * LD + at);
      v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
    }
    *reinterpret_cast<float4*>(sum + at) = v;
  }
  float* fin = smem;                                   // the cluster's sum, scaled, replaces the first partial
  if (c > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    for (int i = threadIdx.x * 4; i < kVals; i += kWarps * 32 * 4) {
      const int at = (i / (8 * RT)) * LD + i % (8 * RT);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float4 w[8];                                     // all of them asked for before the first is used
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < c) w[q] = *reinterpret_cast<const float4*>(cl.map_shared_rank(sum, q) + at);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < c) v.x += w[q].x, v.y += w[q].y, v.z += w[q].z, v.w += w[q].w;
      *reinterpret_cast<float4*>(fin + at) = make_float4(v.x * sc, v.y * sc, v.z * sc, v.w * sc);
    }
    cl.sync();                                         // nobody reads a peer's sum after this
  } else {
    __syncthreads();
    for (int i = threadIdx.x * 4; i < kVals; i += kWarps * 32 * 4) {
      const int at = (i / (8 * RT)) * LD + i % (8 * RT);
      const float4 v = *reinterpret_cast<const float4*>(sum + at);
      *reinterpret_cast<float4*>(fin + at) = make_float4(v.x * sc, v.y * sc, v.z * sc, v.w * sc);
    }
    __syncthreads();
  }
  if (p.h != nullptr && rank_cta == 0) {
    for (int i = threadIdx.x * 2; i < tile.z * p.r; i += kWarps * 32 * 2) {
      const int row = i / p.r, q = i % p.r;
      uint32_t hi, lo;
      split2(fin[row * LD + q], fin[row * LD + q + 1], hi, lo);
      const size_t at = static_cast<size_t>(tile.y + row) * p.r + q;
      *reinterpret_cast<uint32_t*>(p.h + at) = hi;
      *reinterpret_cast<uint32_t*>(p.h + static_cast<size_t>(p.T) * p.r + at) = lo;
    }
  }
  if (p.out == nullptr) return;

  // ---- second product: this warp's columns. Tile j of a chunk holds the columns with the same place among a lane's
  // pairs, so a lane ends with 8 neighbouring columns of its two rows
  uint32_t hi[KS][4], lo[KS][4];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    // ranks of the two pairs of a step: as a lane's wide load of B brings them, or in order where the factor is read across
    const int qa = ACROSS ? 16 * s + 2 * t : RT == 1 ? 2 * t : RT == 2 ? 4 * t : (s >> 1) * 32 + 8 * t + 4 * (s & 1);
    const int qb = ACROSS ? qa + 8 : qa + 2;
    const float2 z = make_float2(0.f, 0.f);
    const float2 f0 = *reinterpret_cast<const float2*>(fin + r0 * LD + qa), f1 = *reinterpret_cast<const float2*>(fin + r1 * LD + qa);
    const float2 f2 = RT == 1 ? z : *reinterpret_cast<const float2*>(fin + r0 * LD + qb), f3 = RT == 1 ? z : *reinterpret_cast<const float2*>(fin + r1 * LD + qb);
    split2(f0.x, f0.y, hi[s][0], lo[s][0]);
    split2(f1.x, f1.y, hi[s][1], lo[s][1]);
    split2(f2.x, f2.y, hi[s][2], lo[s][2]);
    split2(f3.x, f3.y, hi[s][3], lo[s][3]);
  }
  const __nv_bfloat16* up = p.up + static_cast<size_t>(tile.x) * p.r * p.N;
  for (int n = n_lo; n < n_hi; ++n) {
    const int col = n * 32 + 8 * t;
    const bool in = col < p.N;
    const uint4 y0 = ld16(p.base + row0 * p.ld_base + col, in && p.base != nullptr), y1 = ld16(p.base + row1 * p.ld_base + col, in && p.base != nullptr);
    float o[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    if constexpr (!ACROSS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int bc = n * 32 + (g >> 1) * 8 + 2 * j + (g & 1);
        const __nv_bfloat16* f = up + static_cast<size_t>(bc) * p.r;
        const bool inb = bc < p.N;
        if constexpr (RT == 1) {
          const uint32_t b = inb ? *reinterpret_cast<const uint32_t*>(f + 2 * t) : 0u;
          mma16816(o[j], hi[0][0], hi[0][1], hi[0][2], hi[0][3], b, 0u);
          mma16816(o[j], lo[0][0], lo[0][1], lo[0][2], lo[0][3], b, 0u);
        } else if constexpr (RT == 2) {
          const uint2 b = inb ? *reinterpret_cast<const uint2*>(f + 4 * t) : make_uint2(0u, 0u);
          mma16816(o[j], hi[0][0], hi[0][1], hi[0][2], hi[0][3], b.x, b.y);
          mma16816(o[j], lo[0][0], lo[0][1], lo[0][2], lo[0][3], b.x, b.y);
        } else {
#pragma unroll
          for (int q = 0; q < RT / 4; ++q) {
            const uint4 b = ld16(f + 32 * q + 8 * t, inb && 32 * q + 8 * t < p.r);
            mma16816(o[j], hi[2 * q][0], hi[2 * q][1], hi[2 * q][2], hi[2 * q][3], b.x, b.y);
            mma16816(o[j], lo[2 * q][0], lo[2 * q][1], lo[2 * q][2], lo[2 * q][3], b.x, b.y);
            mma16816(o[j], hi[2 * q + 1][0], hi[2 * q + 1][1], hi[2 * q + 1][2], hi[2 * q + 1][3], b.z, b.w);
            mma16816(o[j], lo[2 * q + 1][0], lo[2 * q + 1][1], lo[2 * q + 1][2], lo[2 * q + 1][3], b.z, b.w);
          }
        }
      }
    } else {
      // rows of the factor are ranks: 8 of them x 32 columns at a time, each lane's 4 pairs of columns into the 4 tiles
#pragma unroll
      for (int i0 = 0; i0 < RT; i0 += 4) {
        __syncwarp();
#pragma unroll
        for (int i = i0; i < (RT < i0 + 4 ? RT : i0 + 4); ++i) {
          const uint4 f = ld16(up + static_cast<size_t>(8 * i + g) * p.N + col, in && (RT <= 2 || 8 * i < p.r));
          const uint32_t put = scratch + (i - i0) * 128 + lane * 4;
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(put), "r"(f.x) : "memory");
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(put + 512), "r"(f.y) : "memory");
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(put + 1024), "r"(f.z) : "memory");
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(put + 1536), "r"(f.w) : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t b[4];
          ldsm4t(scratch + j * 512 + lane * 16, b);      // ranks 8 i0 .. 8 i0 + 31 of tile j; what RT does not fill is not used
          mma16816(o[j], hi[i0 / 2][0], hi[i0 / 2][1], hi[i0 / 2][2], hi[i0 / 2][3], b[0], RT == 1 ? 0u : b[1]);
          mma16816(o[j], lo[i0 / 2][0], lo[i0 / 2][1], lo[i0 / 2][2], lo[i0 / 2][3], b[0], RT == 1 ? 0u : b[1]);
          if constexpr (RT >= 4) {
            mma16816(o[j], hi[i0 / 2 + 1][0], hi[i0 / 2 + 1][1], hi[i0 / 2 + 1][2], hi[i0 / 2 + 1][3], b[2], b[3]);
            mma16816(o[j], lo[i0 / 2 + 1][0], lo[i0 / 2 + 1][1], lo[i0 / 2 + 1][2], lo[i0 / 2 + 1][3], b[2], b[3]);
          }
        }
      }
    }
    uint4 w0, w1;
    const __nv_bfloat162* b0 = reinterpret_cast<const __nv_bfloat162*>(&y0);
    const __nv_bfloat162* b1 = reinterpret_cast<const __nv_bfloat162*>(&y1);
    __nv_bfloat162* v0 = reinterpret_cast<__nv_bfloat162*>(&w0);
    __nv_bfloat162* v1 = reinterpret_cast<__nv_bfloat162*>(&w1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v0[j] = __floats2bfloat162_rn(__low2float(b0[j]) + o[j][0], __high2float(b0[j]) + o[j][1]);
      v1[j] = __floats2bfloat162_rn(__low2float(b1[j]) + o[j][2], __high2float(b1[j]) + o[j][3]);
    }
    if (in && ok0) *reinterpret_cast<uint4*>(p.out + row0 * p.ld_out + col) = w0;
    if (in && ok1) *reinterpret_cast<uint4*>(p.out + row1 * p.ld_out + col) = w1;
  }
}

// ------------------------------------------------------------------------------------------------ large tiles
// 64 tokens of one adapter a cluster, for batches whose adapters have many tokens. What the small kernel asks for and waits
// for, this one keeps in flight: a ring of kRing stages that asynchronous copies fill, 64 of K (or of N) by the tile's 64
// rows and the factor's part, goes on through both products, so the columns' first stages are under way while the cluster
// adds up h. Warp (m, f) owns 16 rows and one half of a stage. A stage is stored in 16-byte pieces whose place within the
// row is xored with bits of the row's number: reads of 8 rows at once, and of 2 rows' half lines, meet 8 different bank
// groups. The loop was bound by its instructions at first (69 % of issue slots, 4.8 TB/s), so what a thread copies next is
// held as running pointers.
constexpr int kRing = 4;

template <int RT>
constexpr int tile_stage() {
  return 64 * 128 + 64 * 16 * RT;
}
template <int RT>
constexpr int tile_smem() {
  return kRing * tile_stage<RT>() + 2 * 64 * (8 * RT + 4) * 4;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// byte of a 16-byte piece: rows of 8 pieces (64 numbers), or of RT pieces (the rank)
__device__ __forceinline__ uint32_t wide_at(int row, int piece) { return row * 128 + ((piece ^ (((row & 1) << 2) | ((row >> 1) & 3))) << 4); }
template <int RT>
__device__ __forceinline__ uint32_t narrow_at(int row, int piece) {
  const int x = RT >= 8 ? row & 7 : RT == 4 ? (row >> 1) & 3 : RT == 2 ? (row >> 2) & 1 : 0;
  return row * 16 * RT + ((piece ^ x) << 4);
}

// What one thread copies of a factor's part of a stage: piece v of rows row, row + kRows, ... The rows are ranks (8 RT of
// them, 64 numbers wide) or places along K / N (64 of them, the rank wide); SPREAD stores those places so that the 8 rows
// of a matrix are columns a lane then holds side by side (see the second product).
template <int RT, bool RANKS, bool SPREAD>
struct Feed {
  static constexpr int kTimes = (64 * RT + 255) / 256, kRows = RANKS ? 32 : 256 / RT;
  const __nv_bfloat16* src;
  int at, width, r;                     // first number (RANKS), or place, of this thread's next piece
  bool ok;
  __device__ __forceinline__ Feed(const __nv_bfloat16* f, int start, int width_, int r_) : width(width_), r(r_) {
    const int row = RANKS ? threadIdx.x >> 3 : threadIdx.x / RT, v = RANKS ? threadIdx.x & 7 : threadIdx.x % RT;
    ok = RANKS || v * 8 < r;
    at = start + (RANKS ? v * 8 : row);
    src = f + (RANKS ? static_cast<size_t>(row) * width + at : static_cast<size_t>(at) * r + v * 8);
  }
  __device__ __forceinline__ void copy(uint32_t dst, const __nv_bfloat16* anywhere) {
    const int row0 = RANKS ? threadIdx.x >> 3 : threadIdx.x / RT, v = RANKS ? threadIdx.x & 7 : threadIdx.x % RT;
    if (RT >= 4 || threadIdx.x < 64 * RT) {
#pragma unroll
      for (int i = 0; i < kTimes; ++i) {
        int row = row0 + i * kRows;
        const bool in = RANKS ? at < width && (RT <= 2 || row < r) : ok && at + i * kRows < width;
        const __nv_bfloat16* from = src + (RANKS ? static_cast<size_t>(i * kRows) * width : static_cast<size_t>(i * kRows) * r);
        if (SPREAD) row = (row & 32) | (((row >> 1) & 3) << 3) | (((row >> 3) & 3) << 1) | (row & 1);
        cp16(dst + (RANKS ? wide_at(row, v) : narrow_at<RT>(row, v)), in ? from : anywhere, in);
      }
    }
    at += 64;
    src += RANKS ? 64 : 64 * r;
  }
};

// CTAs a multiprocessor are what keeps its memory busy: the compiler is held to the registers that allow 4 (rank 16: 212 us
// at 8192 x 4096 -> 24576 with 3, 187 with 4) or 3 and 2 for the larger ranks (64: 87 us with 1 at 4096 -> 4096, 66 with 2)
template <int RT, bool ACROSS>
__global__ void __launch_bounds__(256, RT <= 2 ? 4 : RT <= 4 ? 3 : RT <= 8 ? 2 : 1) lora_tile_kernel(const __grid_constant__ ApplyArgs p) {
  constexpr int LD = 8 * RT + 4;
  constexpr int KS = RT < 2 ? 1 : RT / 2;
  extern __shared__ __align__(128) uint8_t raw[];
  if (blockIdx.y >= p.n_tiles[0]) return;              // the same for the whole cluster
  const int4 tile = p.tiles[blockIdx.y];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int c = gridDim.x, rank_cta = blockIdx.x;
  const int mt = warp & 3, hf = warp >> 2;
  const int n_all = (p.N + 63) >> 6, k_all = (p.K + 63) >> 6;
  const int n_lo = static_cast<int>(static_cast<long long>(n_all) * rank_cta / c), n_hi = static_cast<int>(static_cast<long long>(n_all) * (rank_cta + 1) / c);
  const int k_lo = static_cast<int>(static_cast<long long>(k_all) * rank_cta / c), k_hi = static_cast<int>(static_cast<long long>(k_all) * (rank_cta + 1) / c);
  // rows that this thread copies (piece ch of each), and rows that it stores
  const int ra = tid >> 3, rb = ra + 32, ch = tid & 7;
  const bool oka = ra < tile.z, okb = rb < tile.z;
  const long long rowa = p.perm[tile.y + (oka ? ra : 0)], rowb = p.perm[tile.y + (okb ? rb : 0)];
  if (tile.x < 0) {                                    // no adapter: the base alone
    if (p.out == nullptr || p.out == p.base) return;
    for (int n = n_lo; n < n_hi; ++n) {
      const int col = n * 64 + ch * 8;
      if (col >= p.N) break;
      if (oka) *reinterpret_cast<uint4*>(p.out + rowa * p.ld_out + col) = ld16(p.base + rowa * p.ld_base + col, p.base != nullptr);
      if (okb) *reinterpret_cast<uint4*>(p.out + rowb * p.ld_out + col) = ld16(p.base + rowb * p.ld_base + col, p.base != nullptr);
    }
    return;
  }
  const uint32_t ring = smem_u32(raw);
  float* hsum = reinterpret_cast<float*>(raw + kRing * tile_stage<RT>());
  float* hfin = hsum + 64 * LD;
  const int nk = k_hi - k_lo, total = nk + (p.out != nullptr ? n_hi - n_lo : 0);
  const __nv_bfloat16* down = p.down + static_cast<size_t>(tile.x) * p.r * p.K;
  const __nv_bfloat16* up = p.up + static_cast<size_t>(tile.x) * p.r * p.N;
  Feed<RT, !ACROSS, false> feed_down(down, k_lo * 64, p.K, p.r);
  Feed<RT, ACROSS, !ACROSS> feed_up(up, n_lo * 64, p.N, p.r);
  const uint32_t da = wide_at(ra, ch), db = wide_at(rb, ch);
  const __nv_bfloat16 *pa = p.in + rowa * p.ld_in + k_lo * 64 + ch * 8, *pb = p.in + rowb * p.ld_in + k_lo * 64 + ch * 8;
  int col = k_lo * 64 + ch * 8, fed = 0;
  uint32_t slot = ring;                                // where the next stage goes
  auto load = [&]() {
    if (fed < total) {
      if (fed == nk) {
        pa = p.base + rowa * p.ld_base + n_lo * 64 + ch * 8, pb = p.base + rowb * p.ld_base + n_lo * 64 + ch * 8;
        col = n_lo * 64 + ch * 8;
      }
      const bool first = fed < nk, in = col < (first ? p.K : p.N);
      if (first || p.base != nullptr) {
        cp16(slot + da, in ? pa : p.in, in && oka);
        cp16(slot + db, in ? pb : p.in, in && okb);
      }
      if (first) feed_down.copy(slot + 8192, p.in);
      else feed_up.copy(slot + 8192, p.in);
      pa += 64, pb += 64, col += 64;
      ++fed;
      slot = slot == ring + (kRing - 1) * tile_stage<RT>() ? ring : slot + tile_stage<RT>();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) load();

  // ---- first product
  float acc[RT][4];
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
  const int l8 = lane & 7, lm = lane >> 3;             // row and matrix that this lane's address is for
  uint32_t st = ring;                                  // the stage that is read
  for (int i = 0; i < nk; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
    __syncthreads();                                   // the stage has landed, and everybody is done with the one before
    load();
    const uint32_t fs = st + 8192;
    uint32_t a[2][4];
#pragma unroll
    for (int s = 0; s < 2; ++s) ldsm4(st + wide_at(mt * 16 + l8 + 8 * (lm & 1), hf * 4 + 2 * s + (lm >> 1)), a[s]);
    // products that add to the same sums stand apart: one waits 23 cycles for the other
    constexpr int kGroup = RT < 8 ? RT : 8;
#pragma unroll
    for (int j0 = 0; j0 < RT; j0 += kGroup) {
      uint32_t b[kGroup][4];
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
        if constexpr (ACROSS) ldsm4t(fs + narrow_at<RT>(hf * 32 + lm * 8 + l8, j0 + j), b[j]);
        else ldsm4(fs + wide_at((j0 + j) * 8 + l8, hf * 4 + lm), b[j]);
      }
#pragma unroll
      for (int j = 0; j < kGroup; ++j) mma16816(acc[j0 + j], a[0][0], a[0][1], a[0][2], a[0][3], b[j][0], b[j][1]);
#pragma unroll
      for (int j = 0; j < kGroup; ++j) mma16816(acc[j0 + j], a[1][0], a[1][1], a[1][2], a[1][3], b[j][2], b[j][3]);
    }
    st = st == ring + (kRing - 1) * tile_stage<RT>() ? ring : st + tile_stage<RT>();
  }

  // ---- h: the two halves, then the cluster in order: each CTA adds up its share of the rows and hands it to all
  const int r0 = mt * 16 + g, r1 = r0 + 8;
  if (hf == 1) {
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      *reinterpret_cast<float2*>(hfin + r0 * LD + 8 * j + 2 * t) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(hfin + r1 * LD + 8 * j + 2 * t) = make_float2(acc[j][2], acc[j][3]);
    }
  }
  __syncthreads();
  if (hf == 0) {
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      const float2 u = *reinterpret_cast<const float2*>(hfin + r0 * LD + 8 * j + 2 * t), v = *reinterpret_cast<const float2*>(hfin + r1 * LD + 8 * j + 2 * t);
      const bool real = RT <= 2 || 8 * j < p.r;        // ranks that only fill up are zero, not 0 times an infinite x
      *reinterpret_cast<float2*>(hsum + r0 * LD + 8 * j + 2 * t) = real ? make_float2(acc[j][0] + u.x, acc[j][1] + u.y) : make_float2(0.f, 0.f);
      *reinterpret_cast<float2*>(hsum + r1 * LD + 8 * j + 2 * t) = real ? make_float2(acc[j][2] + v.x, acc[j][3] + v.y) : make_float2(0.f, 0.f);
    }
  }
  const float sc = p.scale[tile.x];
  float* fin = hsum;
  if (c > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    const int rows = 64 / c;
    for (int i = tid * 4; i < rows * 8 * RT; i += 1024) {
      const int at = (rank_cta * rows + i / (8 * RT)) * LD + i % (8 * RT);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float4 w[8];                                     // all of them asked for before the first is used
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < c) w[q] = *reinterpret_cast<const float4*>(cl.map_shared_rank(hsum, q) + at);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < c) v.x += w[q].x, v.y += w[q].y, v.z += w[q].z, v.w += w[q].w;
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < c) *reinterpret_cast<float4*>(cl.map_shared_rank(hfin, q) + at) = v;
    }
    cl.sync();                                         // nobody reaches into a peer after this
    fin = hfin;
  } else {
    __syncthreads();
  }
  if (p.h != nullptr && rank_cta == 0) {
    for (int i = tid * 2; i < tile.z * p.r; i += 512) {
      const int row = i / p.r, q = i % p.r;
      uint32_t hi, lo;
      split2(fin[row * LD + q] * sc, fin[row * LD + q + 1] * sc, hi, lo);
      const size_t at = static_cast<size_t>(tile.y + row) * p.r + q;
      *reinterpret_cast<uint32_t*>(p.h + at) = hi;
      *reinterpret_cast<uint32_t*>(p.h + static_cast<size_t>(p.T) * p.r + at) = lo;
    }
  }
  if (p.out == nullptr) return;

  // ---- second product
  uint32_t hi[KS][4], lo[KS][4];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int q = 16 * s + 2 * t;
    const float2 z = make_float2(0.f, 0.f);
    const float2 f0 = *reinterpret_cast<const float2*>(fin + r0 * LD + q), f1 = *reinterpret_cast<const float2*>(fin + r1 * LD + q);
    const float2 f2 = RT == 1 ? z : *reinterpret_cast<const float2*>(fin + r0 * LD + q + 8), f3 = RT == 1 ? z : *reinterpret_cast<const float2*>(fin + r1 * LD + q + 8);
    split2(f0.x * sc, f0.y * sc, hi[s][0], lo[s][0]);
    split2(f1.x * sc, f1.y * sc, hi[s][1], lo[s][1]);
    split2(f2.x * sc, f2.y * sc, hi[s][2], lo[s][2]);
    split2(f3.x * sc, f3.y * sc, hi[s][3], lo[s][3]);
  }
  const int sa = mt * 16 + g, sb = sa + 8;             // rows that this lane stores, piece hf * 4 + t
  __nv_bfloat16* outa = p.out + static_cast<long long>(p.perm[tile.y + (sa < tile.z ? sa : 0)]) * p.ld_out;
  __nv_bfloat16* outb = p.out + static_cast<long long>(p.perm[tile.y + (sb < tile.z ? sb : 0)]) * p.ld_out;
  int oc = n_lo * 64 + (hf * 4 + t) * 8;               // first of the 8 columns that this lane stores
  for (int i = nk; i < total; ++i, oc += 64) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
    __syncthreads();
    load();
    const uint32_t fs = st + 8192;
    auto factor = [&](int oct, int j) {                // address of this lane's row of the matrix (8 ranks oct) x (8 columns j)
      if constexpr (ACROSS) return fs + wide_at(oct * 8 + l8, hf * 4 + j);
      else return fs + narrow_at<RT>(hf * 32 + j * 8 + l8, oct);
    };
    auto fetch = [&](uint32_t at, uint32_t(&b)[4]) {
      if constexpr (ACROSS) ldsm4t(at, b);
      else ldsm4(at, b);
    };
    float o[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) o[j][q] = 0.f;
    if constexpr (RT == 1) {
      uint32_t b[4];
      fetch(factor(0, lm), b);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mma16816(o[j], hi[0][0], hi[0][1], hi[0][2], hi[0][3], b[j], 0u);
        mma16816(o[j], lo[0][0], lo[0][1], lo[0][2], lo[0][3], b[j], 0u);
      }
    } else if constexpr (RT == 2) {
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        uint32_t b[4];
        fetch(factor(lm & 1, j + (lm >> 1)), b);
        mma16816(o[j], hi[0][0], hi[0][1], hi[0][2], hi[0][3], b[0], b[1]);
        mma16816(o[j + 1], hi[0][0], hi[0][1], hi[0][2], hi[0][3], b[2], b[3]);
        mma16816(o[j], lo[0][0], lo[0][1], lo[0][2], lo[0][3], b[0], b[1]);
        mma16816(o[j + 1], lo[0][0], lo[0][1], lo[0][2], lo[0][3], b[2], b[3]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < RT / 4; ++q) {
        uint32_t b[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) fetch(factor(4 * q + lm, j), b[j]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int j = 0; j < 4; ++j) mma16816(o[j], hi[2 * q + k][0], hi[2 * q + k][1], hi[2 * q + k][2], hi[2 * q + k][3], b[j][2 * k], b[j][2 * k + 1]);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma16816(o[j], lo[2 * q + k][0], lo[2 * q + k][1], lo[2 * q + k][2], lo[2 * q + k][3], b[j][2 * k], b[j][2 * k + 1]);
        }
      }
    }
    uint4 w0, w1;
    if constexpr (!ACROSS) {
      // tile j holds the columns 8 t + 2 j of this half: the lane has 8 neighbours of each of its rows
      uint4 y0 = make_uint4(0u, 0u, 0u, 0u), y1 = y0;
      if (p.base != nullptr) {
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(y0.x), "=r"(y0.y), "=r"(y0.z), "=r"(y0.w) : "r"(st + wide_at(sa, hf * 4 + t)) : "memory");
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(y1.x), "=r"(y1.y), "=r"(y1.z), "=r"(y1.w) : "r"(st + wide_at(sb, hf * 4 + t)) : "memory");
      }
      const __nv_bfloat162* b0 = reinterpret_cast<const __nv_bfloat162*>(&y0);
      const __nv_bfloat162* b1 = reinterpret_cast<const __nv_bfloat162*>(&y1);
      __nv_bfloat162* v0 = reinterpret_cast<__nv_bfloat162*>(&w0);
      __nv_bfloat162* v1 = reinterpret_cast<__nv_bfloat162*>(&w1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v0[j] = __floats2bfloat162_rn(__low2float(b0[j]) + o[j][0], __high2float(b0[j]) + o[j][1]);
        v1[j] = __floats2bfloat162_rn(__low2float(b1[j]) + o[j][2], __high2float(b1[j]) + o[j][3]);
      }
    } else {
      // tile j holds columns 8 j of this half: the sum replaces the base in the stage (rows and pieces of this warp alone),
      // so that rows leave 64 bytes at a time
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t at = st + wide_at(mt * 16 + g, hf * 4 + j) + u * 1024 + t * 4;
          float2 y = make_float2(0.f, 0.f);
          if (p.base != nullptr) {
            uint32_t w;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
            const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&w);
            y = make_float2(__low2float(v), __high2float(v));
          }
          const __nv_bfloat162 v = __floats2bfloat162_rn(y.x + o[j][2 * u], y.y + o[j][2 * u + 1]);
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(*reinterpret_cast<const uint32_t*>(&v)) : "memory");
        }
      }
      __syncwarp();
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w0.x), "=r"(w0.y), "=r"(w0.z), "=r"(w0.w) : "r"(st + wide_at(sa, hf * 4 + t)) : "memory");
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w1.x), "=r"(w1.y), "=r"(w1.z), "=r"(w1.w) : "r"(st + wide_at(sb, hf * 4 + t)) : "memory");
    }
    if (oc < p.N) {
      if (sa < tile.z) *reinterpret_cast<uint4*>(outa + oc) = w0;
      if (sb < tile.z) *reinterpret_cast<uint4*>(outb + oc) = w1;
    }
    st = st == ring + (kRing - 1) * tile_stage<RT>() ? ring : st + tile_stage<RT>();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ------------------------------------------------------------------------------------------------ gradients of the factors
// G[rank, col] = sum over an adapter's tokens of h[t, rank] z[t, col]. A CTA owns 128 columns of one adapter, its cluster
// splits the adapter's tokens. Tokens are the contracted index, so both operands are read across (transposed reads of
// shared memory) from tiles of 64 tokens that asynchronous copies bring in kStages deep; a thread looks up the rows it
// copies one tile ahead. Warp (w, f) owns 32 columns, all ranks and one half of a tile's tokens. h is the two bf16 numbers
// that the kernels above stored; sums are fp32, those of the halves and of the cluster are added in order.
// An infinite z times h's two parts, whose signs may differ, is no number where z h is infinite. So a cluster that finds one
// among its results sums the first parts alone once more and takes those sums there.
struct GradArgs {
  const __nv_bfloat16* h;     // [2, T, r], plan's order
  const __nv_bfloat16* z;     // [T, C] rows by token
  __nv_bfloat16* out;         // [E, r, C], or by columns [E, C, r]
  long long ld_z;
  int C, by_cols;
  const int* perm;
  const int* offsets;
  int T, r;
};
constexpr int kTok = 64, kCols = 128, kStages = 3;
constexpr int kZRow = kCols * 2 + 16;                  // bytes a row in shared memory: 16 more spread the transposed reads

template <int RT>
constexpr int grad_stage() {
  return kTok * kZRow + 2 * kTok * 16 * RT;
}
template <int RT>
constexpr int grad_smem() {
  const int ring = kStages * grad_stage<RT>(), sums = kCols * (8 * RT + 4) * 4;
  return (ring > sums ? ring : sums) + 16;             // and the word of grad_sums
}

// BOTH: both parts of h, or the first alone for the results that were no numbers. A word behind the ring, set in every CTA of
// the cluster, says that there are such.
template <int RT, bool BOTH>
__device__ __forceinline__ void grad_sums(const GradArgs& p) {
  extern __shared__ __align__(128) uint8_t raw[];
  int* again = reinterpret_cast<int*>(raw + grad_smem<RT>() - 16);
  const int c = gridDim.x, rank_cta = blockIdx.x, a = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, l8 = lane & 7, lm = lane >> 3;
  const int cg4 = warp & 3, hf = warp >> 2;
  const int col0 = blockIdx.y * kCols;
  const int t0 = p.offsets[a], t1 = p.offsets[a + 1];
  const int tiles = (t1 - t0 + kTok - 1) / kTok;
  const int lo = static_cast<int>(static_cast<long long>(tiles) * rank_cta / c), hi = static_cast<int>(static_cast<long long>(tiles) * (rank_cta + 1) / c);
  const uint32_t base = smem_u32(raw);
  // this thread copies piece ch of rows rr + 16 i
  const int rr = tid >> 4, ch = tid & 15;
  const bool in = col0 + ch * 8 < p.C;
  const __nv_bfloat16* zc = p.z + (in ? col0 + ch * 8 : 0);
  int next[4];
  auto look = [&](int tile) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = t0 + tile * kTok + rr + 16 * i;
      next[i] = tile < hi && at < t1 ? p.perm[at] : -1;
    }
  };
  auto load = [&](int tile) {                          // after look(tile)
    if (tile < hi) {
      const uint32_t st = base + (tile % kStages) * grad_stage<RT>();
      const int first = t0 + tile * kTok;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool ok = in && next[i] >= 0;
        cp16(st + (rr + 16 * i) * kZRow + ch * 16, ok ? zc + static_cast<long long>(next[i]) * p.ld_z : p.z, ok);
      }
#pragma unroll
      for (int i = tid; i < 2 * kTok * RT; i += 256) {
        const int part = i / (kTok * RT), row = i / RT % kTok, v = i % RT;
        const bool ok = first + row < t1 && v * 8 < p.r;
        cp16(st + kTok * kZRow + part * kTok * 16 * RT + narrow_at<RT>(row, v),
             ok ? p.h + (static_cast<size_t>(part) * p.T + first + row) * p.r + v * 8 : p.h, ok);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float acc[2][RT][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < RT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    look(lo + s);
    load(lo + s);
  }
  look(lo + kStages - 1);
  for (int tile = lo; tile < hi; ++tile) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();                                   // the tile has landed, and everybody is done with the one before
    load(tile + kStages - 1);
    look(tile + kStages);
    const uint32_t st = base + (tile % kStages) * grad_stage<RT>();
    const uint32_t hs = st + kTok * kZRow;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = hf * 32 + s * 16;
      // columns are the rows of the product: matrices (tokens k..k+7 | k+8..k+15) x (columns 0..7 | 8..15)
      uint32_t za[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) ldsm4t(st + (k + l8 + 8 * (lm >> 1)) * kZRow + (cg4 * 32 + m * 16 + 8 * (lm & 1)) * 2, za[m]);
      constexpr int kGroup = RT < 4 ? RT : 4;
#pragma unroll
      for (int j0 = 0; j0 < RT; j0 += kGroup) {
        uint32_t b[kGroup][4];                         // (hi, lo) x (tokens k..k+7 | k+8..k+15)
#pragma unroll
        for (int j = 0; j < kGroup; ++j) ldsm4t(hs + (lm >> 1) * kTok * 16 * RT + narrow_at<RT>(k + l8 + 8 * (lm & 1), j0 + j), b[j]);
#pragma unroll
        for (int u = 0; u < (BOTH ? 4 : 2); u += 2)
#pragma unroll
          for (int j = 0; j < kGroup; ++j)
#pragma unroll
            for (int m = 0; m < 2; ++m) mma16816(acc[m][j0 + j], za[m][0], za[m][1], za[m][2], za[m][3], b[j][u], b[j][u + 1]);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // sums of this CTA: [column][rank], the halves in order
  constexpr int LD = 8 * RT + 4;
  float* mine = reinterpret_cast<float*>(raw);
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int turn = 1; turn >= 0; --turn) {
    if (hf == turn) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float2* w = reinterpret_cast<float2*>(mine + (cg4 * 32 + m * 16 + g + 8 * u) * LD + 8 * j + 2 * t);
            float2 v = make_float2(acc[m][j][2 * u], acc[m][j][2 * u + 1]);
            if (turn == 0) v.x += w->x, v.y += w->y;
            *w = v;
          }
    }
    if (turn == 1) __syncthreads();
  }
  // the cluster's CTAs share the columns
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  __nv_bfloat16* out = p.out + static_cast<size_t>(a) * p.r * p.C;
  const int share = kCols / c;
  for (int i = tid; i < share * 2 * RT; i += 256) {
    const int col = rank_cta * share + (p.by_cols ? i / (2 * RT) : i % share), q = 4 * (p.by_cols ? i % (2 * RT) : i / share);
    float4 w[8], v = make_float4(0.f, 0.f, 0.f, 0.f);  // all of them asked for before the first is used
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < c) w[k] = *reinterpret_cast<const float4*>(cl.map_shared_rank(mine, k) + col * LD + q);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < c) v.x += w[k].x, v.y += w[k].y, v.z += w[k].z, v.w += w[k].w;
    if (col0 + col < p.C && q < p.r) {
      if constexpr (!BOTH) {                           // only what was no number is taken
        const __nv_bfloat16* had = p.by_cols ? out + static_cast<size_t>(col0 + col) * p.r + q : out + static_cast<size_t>(q) * p.C + col0 + col;
        const size_t step = p.by_cols ? 1 : p.C;
        const float x = __bfloat162float(had[0]), y = __bfloat162float(had[step]), z = __bfloat162float(had[2 * step]), u = __bfloat162float(had[3 * step]);
        v = make_float4(x == x ? x : v.x, y == y ? y : v.y, z == z ? z : v.z, u == u ? u : v.w);
      } else if (v.x != v.x || v.y != v.y || v.z != v.z || v.w != v.w) {
        for (int k = 0; k < c; ++k) *cl.map_shared_rank(again, k) = 1;
      }
      const __nv_bfloat162 lo2 = __floats2bfloat162_rn(v.x, v.y), hi2 = __floats2bfloat162_rn(v.z, v.w);
      if (p.by_cols) {
        uint2 both;
        both.x = *reinterpret_cast<const uint32_t*>(&lo2), both.y = *reinterpret_cast<const uint32_t*>(&hi2);
        *reinterpret_cast<uint2*>(out + static_cast<size_t>(col0 + col) * p.r + q) = both;
      } else {
        __nv_bfloat16* to = out + static_cast<size_t>(q) * p.C + col0 + col;
        to[0] = lo2.x, to[p.C] = lo2.y, to[2 * static_cast<size_t>(p.C)] = hi2.x, to[3 * static_cast<size_t>(p.C)] = hi2.y;
      }
    }
  }
  cl.sync();                                           // nobody reads a peer's sums after this, and all know of the results
}
template <int RT>
__device__ __noinline__ void grad_sums_of_first_parts(const GradArgs& p) {
  grad_sums<RT, false>(p);
}

template <int RT>
__global__ void __launch_bounds__(256, RT <= 2 ? 3 : RT <= 8 ? 2 : 1) lora_grad_kernel(const __grid_constant__ GradArgs p) {
  extern __shared__ __align__(128) uint8_t raw[];
  int* again = reinterpret_cast<int*>(raw + grad_smem<RT>() - 16);
  if (threadIdx.x == 0) *again = 0;                   // (the cluster's barrier in front of the sums stands between this and the first to set it)
  grad_sums<RT, true>(p);
  if (*again) grad_sums_of_first_parts<RT>(p);      // (out of line: the registers are the first sweep's)
}

// ------------------------------------------------------------------------------------------------ launches
template <auto Kern, typename Args>
int launch(const Args& args, dim3 grid, int smem, cudaStream_t s) {
  return ixh::launch_cluster<Kern>(args, grid, 256, grid.x, smem, smem, false, s);
}

template <int RT>
int apply_tile(const ApplyArgs& a, int large, int across, dim3 grid, cudaStream_t s) {
  if (large && across) return launch<lora_tile_kernel<RT, true>>(a, grid, tile_smem<RT>(), s);
  if (large) return launch<lora_tile_kernel<RT, false>>(a, grid, tile_smem<RT>(), s);
  if (across) return launch<lora_apply_kernel<RT, true>>(a, grid, apply_smem<RT>(true), s);
  return launch<lora_apply_kernel<RT, false>>(a, grid, apply_smem<RT>(false), s);
}

inline int bound_tiles(int T, int E, int size) {
  const int groups = E + 1 < T ? E + 1 : T;
  const long long b = static_cast<long long>(T) / size + groups;
  return static_cast<int>(b < T ? b : T);
}

}  // namespace

IX_API int ix_lora_max_adapters() { return kMaxAdapters; }
// Upper bound of the number of tiles of the small (large = 0) or large size: the tile lists hold that many int4.
IX_API int ix_lora_max_tiles(int T, int E, int large) { return bound_tiles(T, E, large ? kLarge : kSmall); }

// ids int32 [T]; perm int32 [T]; offsets int32 [E + 2]; tiles int4; n_tiles int32 [2] (small, large).
IX_API int ix_lora_plan(const void* ids, int T, int E, void* perm, void* offsets, void* tiles_small, void* tiles_large, void* n_tiles, void* stream) {
  if (T <= 0) return 0;
  if (E < 1 || E > kMaxAdapters) return ixh::fail(ixh::IX_EARG, "lora: 1 to %d adapters, not %d", kMaxAdapters, E);
  // warps: as many as the counters leave room for (48 KB without an opt-in)
  int warps = 32;
  while (warps > 1 && (warps + 1) * (E + 1) * 4 > 34 * 1024) warps >>= 1;
  lora_plan_kernel<<<1, warps * 32, (warps + 1) * (E + 1) * 4, reinterpret_cast<cudaStream_t>(stream)>>>(
      static_cast<const int*>(ids), T, E, static_cast<int*>(perm), static_cast<int*>(offsets), static_cast<int4*>(tiles_small),
      static_cast<int4*>(tiles_large), static_cast<int*>(n_tiles));
  IX_CUDA(cudaGetLastError());
  return 0;
}

// across = 0: out = base + s (in down^T) up^T, down [E, r, K], up [E, N, r]. across = 1: the same with down [E, K, r] and
// up [E, r, N]. base null: zero; out null: only h. h (may be null): bf16 [2, T, r]. All leading dimensions multiples of 8.
IX_API int ix_lora_apply(const void* in, long long ld_in, const void* base, long long ld_base, void* out, long long ld_out, const void* down,
                         const void* up, const void* scale, const void* perm, const void* tiles_small, const void* tiles_large, const void* n_tiles,
                         void* h, int T, int K, int N, int r, int E, int across, void* stream) {
  if (T <= 0) return 0;
  if (r < 8 || r > kMaxRank || r % 8) return ixh::fail(ixh::IX_EARG, "lora: rank %d is not a multiple of 8 up to %d", r, kMaxRank);
  if (K < 8 || N < 8 || K % 8 || N % 8) return ixh::fail(ixh::IX_EARG, "lora: widths %d and %d must be multiples of 8", K, N);
  if (ld_in % 8 || ld_base % 8 || ld_out % 8) return ixh::fail(ixh::IX_EARG, "lora: row strides must be multiples of 8");
  ApplyArgs a;
  a.in = static_cast<const __nv_bfloat16*>(in);
  a.base = static_cast<const __nv_bfloat16*>(base);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.down = static_cast<const __nv_bfloat16*>(down);
  a.up = static_cast<const __nv_bfloat16*>(up);
  a.scale = static_cast<const float*>(scale);
  a.perm = static_cast<const int*>(perm);
  a.h = static_cast<__nv_bfloat16*>(h);
  a.ld_in = ld_in, a.ld_base = ld_base, a.ld_out = ld_out;
  a.T = T, a.K = K, a.N = N, a.r = r;
  // large tiles where adapters have many tokens: they read the factors a quarter as often
  const int large = T / E >= 48;
  a.tiles = static_cast<const int4*>(large ? tiles_large : tiles_small);
  a.n_tiles = static_cast<const int*>(n_tiles) + large;
  const int tiles = bound_tiles(T, E, large ? kLarge : kSmall);
  if (tiles > 65535) return ixh::fail(ixh::IX_ESIZE, "lora: %d tokens of %d adapters make more than 65535 tiles", T, E);
  // CTAs a tile: as many as run together, but not beyond eight steps (small: one a warp) each. 8192 tokens 4096 -> 4096: 44 us
  // with 4 at rank 16 (2: 48, 8: 45), 52 with 2 at rank 32 (4: 66), 61 with 2 at rank 64 (4: 66, 1: 75). Where a tile of rank
  // up to 16 has a long row to write, once more (ranks 32 and 64 do not gain). Rank 16, K 4096, N 4096 / 8192 / 16384 / 24576,
  // without and with it: 8192 tokens (4 CTAs) 46, 46 / 68, 69 / 127, 114 / 191, 164; 12288 (2 CTAs) 63, 66 / 101, 102 / 183, 187 /
  // 262, 272; 32768 (1 CTA) 167, 153 / 285, 252 / 550, 455 / 791, 664. Next to the rule's border at 8192 tokens, N 12288: 100, 92
  int c = 1;
  const int widest = (K > N ? K : N) / 32;
  const int together = 148 * (!large || r <= 16 ? 4 : r <= 32 ? 3 : r <= 64 ? 2 : 1);
  while (c < 8 && tiles * c * 2 <= together && widest > c * 8) c *= 2;
  if (large && r <= 16 && !across && c < 8 && N / 64 >= 64 * c) c *= 2;
  const dim3 grid(c, tiles);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (r <= 8) return apply_tile<1>(a, large, across, grid, s);
  if (r <= 16) return apply_tile<2>(a, large, across, grid, s);
  if (r <= 32) return apply_tile<4>(a, large, across, grid, s);
  if (r <= 64) return apply_tile<8>(a, large, across, grid, s);
  return apply_tile<16>(a, large, across, grid, s);
}

namespace {

// One factor's gradient.
int factor_grad(const GradArgs& a, int E, cudaStream_t s) {
  const int T = a.T, r = a.r, tiles = (a.C + kCols - 1) / kCols;
  if (T <= 0) {
    IX_CUDA(cudaMemsetAsync(a.out, 0, static_cast<size_t>(E) * r * a.C * 2, s));
    return 0;
  }
  // CTAs an adapter's columns, with at least four tiles of an average adapter's tokens each: what gives the shortest run of
  // CTAs one after another on a multiprocessor's places, the fewest where that is equal (8192 tokens x 24576: 79 us with 2,
  // 117 with 1, 84 with 4; 463 tokens an adapter: 8 us with 2, 11 with 4)
  const long long places = 148 * (r <= 16 ? 3 : r <= 64 ? 2 : 1), all = static_cast<long long>(tiles) * E;
  int c = 1;
  long long best = (all + places - 1) / places * 8;
  for (int k = 2; k <= 8 && T / E >= k * 4 * kTok; k *= 2) {
    const long long turns = (all * k + places - 1) / places * (8 / k);
    if (turns < best) best = turns, c = k;
  }
  const dim3 grid(c, tiles, E);
  if (r <= 8) return launch<lora_grad_kernel<1>>(a, grid, grad_smem<1>(), s);
  if (r <= 16) return launch<lora_grad_kernel<2>>(a, grid, grad_smem<2>(), s);
  if (r <= 32) return launch<lora_grad_kernel<4>>(a, grid, grad_smem<4>(), s);
  if (r <= 64) return launch<lora_grad_kernel<8>>(a, grid, grad_smem<8>(), s);
  return launch<lora_grad_kernel<16>>(a, grid, grad_smem<16>(), s);
}

}  // namespace

// Backward of out = y + s (x A^T) B^T: g = s dy B, dx = base + g A (dx null: not wanted; base null: zero), dA = g^T x and
// dB = dy^T h by adapter (null: not wanted; zero for an adapter without tokens). h: what ix_lora_apply stored; g: bf16 [2, T, r]
// scratch, needed for dA. dx may be base.
IX_API int ix_lora_backward(const void* dy, long long ld_dy, const void* x, long long ld_x, const void* base, long long ld_base, void* dx,
                            long long ld_dx, const void* A, const void* B, const void* scale, const void* perm, const void* tiles_small,
                            const void* tiles_large, const void* n_tiles, const void* offsets, const void* h, void* g, void* dA, void* dB, int T,
                            int K, int N, int r, int E, void* stream) {
  if (T > 0 && dA != nullptr && g == nullptr) return ixh::fail(ixh::IX_EARG, "lora: the gradient of A needs scratch for g");
  if (T > 0 && dB != nullptr && h == nullptr) return ixh::fail(ixh::IX_EARG, "lora: the gradient of B needs the forward's h");
  if (r < 8 || r > kMaxRank || r % 8) return ixh::fail(ixh::IX_EARG, "lora: rank %d is not a multiple of 8 up to %d", r, kMaxRank);
  if (K < 8 || N < 8 || K % 8 || N % 8) return ixh::fail(ixh::IX_EARG, "lora: widths %d and %d must be multiples of 8", K, N);
  if (T > 0 && (ld_dy % 8 || ld_x % 8)) return ixh::fail(ixh::IX_EARG, "lora: row strides must be multiples of 8");
  if (dx != nullptr || dA != nullptr) {
    const int rc = ix_lora_apply(dy, ld_dy, base, ld_base, dx, ld_dx, B, A, scale, perm, tiles_small, tiles_large, n_tiles, dA != nullptr ? g : nullptr,
                                 T, N, K, r, E, 1, stream);
    if (rc) return rc;
  }
  // (both in one launch were 126 us at 8192 tokens x 4096 and 24576 instead of 107: the one cut into parts suits only one)
  GradArgs a = {};
  a.perm = static_cast<const int*>(perm), a.offsets = static_cast<const int*>(offsets);
  a.T = T, a.r = r;
  int rc = 0;
  if (dB != nullptr) {
    a.h = static_cast<const __nv_bfloat16*>(h), a.z = static_cast<const __nv_bfloat16*>(dy), a.out = static_cast<__nv_bfloat16*>(dB);
    a.ld_z = ld_dy, a.C = N, a.by_cols = 1;
    rc = factor_grad(a, E, reinterpret_cast<cudaStream_t>(stream));
  }
  if (rc == 0 && dA != nullptr) {
    a.h = static_cast<const __nv_bfloat16*>(g), a.z = static_cast<const __nv_bfloat16*>(x), a.out = static_cast<__nv_bfloat16*>(dA);
    a.ld_z = ld_x, a.C = K, a.by_cols = 0;
    rc = factor_grad(a, E, reinterpret_cast<cudaStream_t>(stream));
  }
  return rc;
}
