// Shared device/host helpers of the B200 quantize-then-attend library.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace sage {

constexpr int HD = 128;        // head dim
constexpr int TILE = 128;      // query tile == key tile == prologue token tile
constexpr float I8_MAX = 127.0f;
constexpr float F8_MAX = 448.0f;
constexpr float SCALE_FLOOR = 1e-12f;
constexpr float LOG2E_F = 1.4426950408889634f;

// Control block of the prologue (device memory, zeroed by a small kernel at the start of every call).
struct CtrlHeader {
  // per head: [0] arrivals of the K mean kernel, [1] V tiles quantised so far, [2] max V scale bits, [3] arrivals
  // of the V mean kernel (smooth_v), laid out as four arrays of BH words; then one status word
  // (non-zero when a wait inside the quantiser ran out), one pad word and the quantiser's 64-bit
  // work counter; the fp64 partial sums (shared by the two mean launches, which run one after the
  // other) follow at `partial_off`.
  // (four more words follow the work counter: the attention kernel's count of skipped
  // (warp, key tile) pairs, then three spare words; all of them are cleared by the same kernel)
  static __host__ __device__ inline size_t words(int64_t bh) { return (size_t)4 * (size_t)bh + 8; }
  static __host__ __device__ inline size_t status_word(int64_t bh) { return (size_t)4 * (size_t)bh; }
  static __host__ __device__ inline size_t partial_off(int64_t bh) {
    return (words(bh) * 4 + 255) / 256 * 256;
  }
};

// Programmatic dependent launch.  A kernel launched with launch_after_predecessor() may be placed
// on the GPU while the kernel before it on the stream is still draining; it must call
// wait_for_predecessor() before it touches anything that kernel (or anything earlier on the
// stream) wrote.  allow_successor() in the earlier kernel says "my CTAs are all resident, the
// next kernel's may be scheduled as mine retire".  Without the launch attribute both calls are
// no-ops, so the kernels behave the same under a plain launch.
#ifdef __CUDACC__
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_successor() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... KArgs, typename... Args>
inline cudaError_t launch_after_predecessor(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem,
                                            cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}
#endif

// How many CTAs share one head's sequence in the mean kernel on a device with `sms` SMs: one full
// wave of four resident CTAs per SM, at least 256 tokens per CTA, at most 64 splits.
inline int kmean_splits(int64_t bh, int64_t n, int sms) {
  int64_t want = (4 * (int64_t)sms) / bh;
  int64_t cap = (n + 255) / 256;
  if (want > cap) want = cap;
  if (want > 64) want = 64;
  if (want < 1) want = 1;
  return (int)want;
}
// The scratch for the partial sums is sized without a device at hand, for the largest SM count
// an sm_100 part has; a launch never uses more splits than that.
constexpr int KMEAN_SIZING_SMS = 160;
inline int kmean_splits_max(int64_t bh, int64_t n) { return kmean_splits(bh, n, KMEAN_SIZING_SMS); }

template <typename T> struct Elem;
template <> struct Elem<__half> {
  static __device__ __forceinline__ float2 cvt2(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
};
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float2 cvt2(uint32_t w) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  }
};

// 16 bytes = 8 elements -> 8 floats (exact widening).
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float* x) {
  float2 a = Elem<T>::cvt2(u.x), b = Elem<T>::cvt2(u.y), c = Elem<T>::cvt2(u.z), d = Elem<T>::cvt2(u.w);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}

// Two floats -> two 16-bit values (a in the low half), round to nearest even.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Two floats -> two e4m3 bytes (a in the low byte), round to nearest even, saturating.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}

// ---- quantising a row (one scale per token and head) -------------------------------------------------
#ifdef __CUDACC__
__device__ __forceinline__ float quarter_warp_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return x;
}
// rn(a / d) for a compile-time divisor: rc = rn(1/d) is a constant, the rest is Markstein's sequence
// (checked against true division over every mantissa of several binades for d = 127 and 448).
template <int DIV>
__device__ __forceinline__ float div_const(float a) {
  constexpr float d = (float)DIV, rc = 1.0f / (float)DIV;
  const float q0 = __fmul_rn(a, rc);
  const float r = __fmaf_rn(-q0, d, a);
  return __fmaf_rn(r, rc, q0);
}
__device__ __forceinline__ uint32_t i8x4_magic2(float2 ab, float2 cd) {
  const float2 m = make_float2(12582912.0f, 12582912.0f);
  const float2 u = __fadd2_rn(ab, m), v = __fadd2_rn(cd, m);
  return __byte_perm(__byte_perm(__float_as_uint(u.x), __float_as_uint(u.y), 0x0040),
                     __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x0040), 0x5410);
}

// Largest magnitude of eight packed 16-bit values: exact on the packed form, half the instructions.
template <typename T> struct Packed16;
template <> struct Packed16<__half> { typedef __half2 Pair; };
template <> struct Packed16<__nv_bfloat16> { typedef __nv_bfloat162 Pair; };
template <typename T>
__device__ __forceinline__ float absmax16(const uint4& u, const uint4& v) {
  typedef typename Packed16<T>::Pair Pair;
  const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
  Pair m = __habs2(*reinterpret_cast<const Pair*>(&w[0]));
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const Pair*>(&w[i])));
  const float2 f = Elem<T>::cvt2(*reinterpret_cast<const uint32_t*>(&m));
  return fmaxf(f.x, f.y);
}
__device__ __forceinline__ float absmax3(float m, float2 x) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(x.x)), "f"(fabsf(x.y)));
  return r;
}
// e4m3 codes of rn(x / s) for four values, given rc = rn(1/s).  The remainder is taken as q0*s - x and
// subtracted, which keeps the sign of a zero x; the packed operations have no negation, so the
// steps divide -x (all signs turn around, those of zeros too) and the codes' sign bits are flipped back.
__device__ __forceinline__ uint32_t e4m3x4_quot(float2 a, float2 b, float s, float rc) {
  const float2 nrc = make_float2(-rc, -rc), s2 = make_float2(s, s);
  const float2 qa = __fmul2_rn(a, nrc), qb = __fmul2_rn(b, nrc);
  const float2 ya = __ffma2_rn(__ffma2_rn(qa, s2, a), nrc, qa), yb = __ffma2_rn(__ffma2_rn(qb, s2, b), nrc, qb);
  return e4m3x4(ya.x, ya.y, yb.x, yb.y) ^ 0x80808080u;
}
#endif

}  // namespace sage
