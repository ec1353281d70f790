// One AdamW step over many tensors in one launch, the two moments held in 32 bits or in 8.
//
//   g = grad * grad_scale;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// 8-bit states: 256 consecutive elements of a tensor share one fp32 scale (largest magnitude / 448) and each holds an e4m3
// code of value / scale. The second moment is held by its square root, which halves the range the code has to span, and
// a code of a positive root is never zero: a mean that still moves would otherwise be divided by eps alone. The update
// itself uses the moments before they are rounded; that rounding (half a step of e4m3, 2^-4 of the value) is what the
// next step starts from.
//
// The tensors' addresses stand in a table in device memory that is laid out once, with one entry of a chunk map for every
// kChunk elements, so the launch does not grow with the number of tensors. A warp owns the 256 elements of a scale.
#include "bw_common.cuh"
#include "host_util.h"

#include <cuda_fp8.h>

namespace {
using namespace bw;

constexpr int kBlock = 256;           // elements that share a scale
constexpr int kThreads = 256;
constexpr int kVec = 8;               // elements a thread
constexpr int kChunk = kThreads * kVec;

struct Entry {                        // 64 bytes; filled by ops/optim.py
  void* p;                            // parameters (fp32, or bf16 with fp32 masters)
  const void* g;
  long long n;                        // elements
  long long offset;                   // first element of the tensor's section in the state buffers, a multiple of 256
  float weight_decay;
  int vec;                            // p and g start on 16-byte boundaries
  long long pad[3];
};
static_assert(sizeof(Entry) == 64, "table layout");

struct Args {
  const Entry* table;
  const int2* chunks;                 // (tensor, chunk of it)
  float* master;                      // null when the parameters are fp32
  void* m;                            // fp32, or e4m3 codes
  void* v;
  float* m_scale;
  float* v_scale;
  const float* grad_scale;            // may be null
  float b1, nb1, b2, nb2, eps, lr, step_size, rsqrt_bc2;
};

template <typename T>
__device__ __forceinline__ void load8(const T* src, long long i, long long n, bool vec, float (&x)[kVec]) {
  if (vec && i + kVec <= n) {
    if constexpr (sizeof(T) == 2) {
      const uint4 a = *reinterpret_cast<const uint4*>(src + i);
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[2 * j] = __low2float(h[j]), x[2 * j + 1] = __high2float(h[j]);
    } else {
      const float4 a = *reinterpret_cast<const float4*>(src + i), b = *reinterpret_cast<const float4*>(src + i + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    x[j] = 0.f;
    if (i + j < n) {
      if constexpr (sizeof(T) == 2) x[j] = __bfloat162float(src[i + j]);
      else x[j] = src[i + j];
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* dst, long long i, long long n, bool vec, const float (&x)[kVec]) {
  if (vec && i + kVec <= n) {
    if constexpr (sizeof(T) == 2) {
      uint4 a;
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&a);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
      *reinterpret_cast<uint4*>(dst + i) = a;
    } else {
      *reinterpret_cast<float4*>(dst + i) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(dst + i + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    if (i + j < n) {
      if constexpr (sizeof(T) == 2) dst[i + j] = __float2bfloat16_rn(x[j]);
      else dst[i + j] = x[j];
    }
  }
}

__device__ __forceinline__ void decode8(const void* codes, long long at, float scale, float (&x)[kVec]) {
  const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(codes) + at);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = j < 2 ? c.x : c.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * (j & 1))), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    x[2 * j] = __fmul_rn(f.x, scale), x[2 * j + 1] = __fmul_rn(f.y, scale);
  }
}

// Square root: the approximation and one step of Newton's method, s + (v - s^2) / (2 s), to the last place. Where v is next to
// the smallest numbers the approximation stands (v - s^2 would be rounded away).
__device__ __forceinline__ float root_of(float v) {
  float s, r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(s) : "f"(v));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return v > 1e-30f && v < 1e38f ? fmaf(fmaf(-s, s, v), 0.5f * r, s) : s;
}

// Codes and scale of the warp's 256 values. `root`: a positive value's code is at least the smallest one.
template <bool ROOT>
__device__ __forceinline__ void encode8(void* codes, float* scales, long long at, float (&x)[kVec]) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < kVec; ++j) top = fmaxf(top, fabsf(x[j]));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  float s = __fmul_rn(top, 1.f / 448.f);
  if (s < 1.17549435e-38f) s = 0.f;              // below the normal numbers the quotient would be noise: the block is zero
  // 256 quotients by one divisor: one reciprocal a block, then x * r corrected by its own remainder, which rounds as the
  // division does (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990)
  const float r = s > 0.f ? __frcp_rn(s) : 0.f;
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a = __fmul_rn(x[2 * j], r), b = __fmul_rn(x[2 * j + 1], r);
    a = fmaf(fmaf(-a, s, x[2 * j]), r, a), b = fmaf(fmaf(-b, s, x[2 * j + 1]), r, b);
    if (ROOT) {
      a = a > 0.f ? fmaxf(a, 0.001953125f) : a;
      b = b > 0.f ? fmaxf(b, 0.001953125f) : b;
    }
    w[j >> 1] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)) << (16 * (j & 1));
  }
  *reinterpret_cast<uint2*>(static_cast<uint8_t*>(codes) + at) = make_uint2(w[0], w[1]);
  if ((threadIdx.x & 31) == 0) scales[at / kBlock] = s;
}

template <typename P, typename G, bool BITS8>
__global__ void __launch_bounds__(kThreads, BITS8 ? 5 : 4) tensor_adamw_kernel(Args a) {
  const int2 where = a.chunks[blockIdx.x];
  const Entry e = a.table[where.x];
  const long long first = static_cast<long long>(where.y) * kChunk + static_cast<long long>(threadIdx.x >> 5) * kBlock;
  if (first >= e.n) return;                       // a whole warp: no section of the state buffers is there
  const long long i = first + (threadIdx.x & 31) * kVec;
  const long long at = e.offset + i;
  const float gs = a.grad_scale ? a.grad_scale[0] : 1.f;
  float p[kVec], g[kVec], m[kVec], v[kVec];
  load8(static_cast<const G*>(e.g), i, e.n, e.vec, g);
  if constexpr (sizeof(P) == 2) load8(a.master + e.offset, i, e.n, true, p);
  else load8(static_cast<const P*>(e.p), i, e.n, e.vec, p);
  if constexpr (BITS8) {
    decode8(a.m, at, a.m_scale[at / kBlock], m);
    decode8(a.v, at, a.v_scale[at / kBlock], v);
  } else {
    load8(static_cast<const float*>(a.m) + e.offset, i, e.n, true, m);
    load8(static_cast<const float*>(a.v) + e.offset, i, e.n, true, v);
  }
  const float keep = 1.f - a.lr * e.weight_decay;
  float root[kVec];
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    // products and sums rounded one by one: the codes of the 8-bit states then do not depend on what the compiler fuses
    const float x = __fmul_rn(g[j], gs);
    const float vo = BITS8 ? __fmul_rn(v[j], v[j]) : v[j];
    m[j] = __fadd_rn(__fmul_rn(a.b1, m[j]), __fmul_rn(a.nb1, x));
    v[j] = __fadd_rn(__fmul_rn(a.b2, vo), __fmul_rn(__fmul_rn(a.nb2, x), x));
    root[j] = root_of(v[j]);
    p[j] = p[j] * keep - __fdividef(a.step_size * m[j], root[j] * a.rsqrt_bc2 + a.eps);
  }
  if constexpr (sizeof(P) == 2) store8(a.master + e.offset, i, e.n, true, p);
  store8(static_cast<P*>(e.p), i, e.n, e.vec, p);
  if constexpr (BITS8) {
    encode8<false>(a.m, a.m_scale, at, m);
    encode8<true>(a.v, a.v_scale, at, root);
  } else {
    store8(static_cast<float*>(a.m) + e.offset, i, e.n, true, m);
    store8(static_cast<float*>(a.v) + e.offset, i, e.n, true, v);
  }
}

template <typename P, typename G>
int launch(const Args& a, int chunks, int bits8, cudaStream_t s) {
  if (bits8) tensor_adamw_kernel<P, G, true><<<chunks, kThreads, 0, s>>>(a);
  else tensor_adamw_kernel<P, G, false><<<chunks, kThreads, 0, s>>>(a);
  IX_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace

// Elements covered by one entry of the chunk map.
IX_API int ix_tensor_adamw_chunk() { return kChunk; }

// table: one Entry a tensor; chunks: `n_chunks` pairs (tensor, chunk). master: null exactly when param_dtype is fp32.
// Types: 0 = bf16, 1 = fp32. step >= 1.
IX_API int ix_tensor_adamw(const void* table, const void* chunks, int n_chunks, int param_dtype, int grad_dtype, int bits8,
                           void* master, void* m, void* v, void* m_scale, void* v_scale, const void* grad_scale, double lr,
                           double beta1, double beta2, double eps, long long step, void* stream) {
  if (n_chunks <= 0) return 0;
  if (step < 1) return ixh::fail(ixh::IX_EARG, "tensor_adamw: step must be at least 1");
  if ((param_dtype == 0) != (master != nullptr)) return ixh::fail(ixh::IX_EARG, "tensor_adamw: bf16 parameters need fp32 masters, fp32 ones have none");
  if (bits8 && (!m_scale || !v_scale)) return ixh::fail(ixh::IX_EARG, "tensor_adamw: 8-bit states need their scales");
  Args a;
  a.table = static_cast<const Entry*>(table);
  a.chunks = static_cast<const int2*>(chunks);
  a.master = static_cast<float*>(master);
  a.m = m, a.v = v;
  a.m_scale = static_cast<float*>(m_scale), a.v_scale = static_cast<float*>(v_scale);
  a.grad_scale = static_cast<const float*>(grad_scale);
  const double bc1 = 1.0 - pow(beta1, static_cast<double>(step)), bc2 = 1.0 - pow(beta2, static_cast<double>(step));
  a.b1 = static_cast<float>(beta1), a.nb1 = static_cast<float>(1.0 - beta1);
  a.b2 = static_cast<float>(beta2), a.nb2 = static_cast<float>(1.0 - beta2);
  a.eps = static_cast<float>(eps), a.lr = static_cast<float>(lr);
  a.step_size = static_cast<float>(lr / bc1), a.rsqrt_bc2 = static_cast<float>(1.0 / sqrt(bc2));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (param_dtype == 0) return grad_dtype == 0 ? launch<__nv_bfloat16, __nv_bfloat16>(a, n_chunks, bits8, s) : launch<__nv_bfloat16, float>(a, n_chunks, bits8, s);
  return grad_dtype == 0 ? launch<float, __nv_bfloat16>(a, n_chunks, bits8, s) : launch<float, float>(a, n_chunks, bits8, s);
}
