// Operators around a quantised, paged K/V cache that move data: rotary positions, quantising new keys
// and values as they are written, and reading sequences back in 16 bits.  (Attention over the cache:
// sage_cache_attn.cu.)  All of them are bound by HBM for long calls and by one launch for short ones.
//
// A cache holds pages of page_size tokens.  For every (page, head, token of the page): a row of
// `width` one-byte K codes (int8 or e4m3), one of V codes (e4m3), and an fp32 scale for each.  The
// rows are 64 bytes wide for heads of up to 64 columns and 128 bytes otherwise, zero-filled; the code
// of column d is byte d.  Value = code * scale, plus the shift of K if the cache has one.
#include <algorithm>
#include <atomic>

#include "sage_common.cuh"
#include "sage_internal.h"

namespace sage {

namespace {

// Small CTAs: the loads of one fill the pauses of others.  With 256 threads: 27 280 x 48 heads written 193 us (128: 178),
// rotary of 8771 x 96 heads 71.5 (68.2), read back alike.
constexpr int CACHE_THREADS = 128;

// 16-byte accesses of data that is not used again soon
__device__ __forceinline__ uint4 ld_stream(const void* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ void st_stream(void* p, const uint4& v) { __stcs(reinterpret_cast<uint4*>(p), v); }

// 32 bytes in one access where WIDE says that the address is a multiple of 32, in two of 16 otherwise (every sector of
// 32 bytes is then written twice in halves: 27 280 x 48 heads read back 213 us, 197 in one).
template <bool WIDE> __device__ __forceinline__ void st_stream32(void* p, const uint4& a, const uint4& b, bool lo, bool hi) {
  if (WIDE) {
    if (lo)
      asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                   ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
  } else {
    if (lo) st_stream(p, a);
    if (hi) st_stream(reinterpret_cast<uint8_t*>(p) + 16, b);
  }
}

// The larger of two magnitudes, NaN if either is (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---- rotary positions --------------------------------------------------------------------------------
// Pair (a, b) of a row at position p becomes (a c - b s, b c + a s), c = m cos(p f), s = m sin(p f).
// One CTA per token: its cosines and sines are worked out once, in shared memory, and serve all heads of
// Q and K.  The angle is a product and a reduction by whole turns in 64 bits (in 32 a position of 10^5
// would leave 8 bits of it), then sincosf of at most pi.
// Bound by HBM: 8771 tokens x 96 heads, half of each turned, 67 us = 6.4 TB/s, what a plain copy reaches; 4 x 4096 tokens
// x 40 heads, 59 us = 5.7.  A step of 16 tokens is a launch, 3.4 us.
struct RotaryKArgs {
  const void *q, *k, *pos;
  void *q_out, *k_out;
  const double* freq;
  long long q_s[3], k_s[3], qo_s[3], ko_s[3];   // (batch, head, row) strides in elements
  long long pos_s[2];                           // (batch, row) strides
  float magnitude;                              // factor on the cosines and sines, its sign apart
  int Hq, Hk, N, D, rot, pos64, backward, copy_q, copy_k;
};

// VEC: elements of a row that a thread takes at a time from either half of the pairs (8, or 4 where half
// of the turned columns is no multiple of 8); interleaved pairs sit in the same 8 elements.
template <typename T, bool INTERLEAVED, int VEC>
__global__ void __launch_bounds__(CACHE_THREADS) rotary_kernel(const RotaryKArgs a) {
  __shared__ float2 cs[HD / 2];
  const long long b = (long long)blockIdx.x / a.N, n = (long long)blockIdx.x % a.N;
  const int half = a.rot / 2;
  {
    const long long at = b * a.pos_s[0] + n * a.pos_s[1];
    const double p = a.pos64 ? (double)reinterpret_cast<const long long*>(a.pos)[at] : (double)reinterpret_cast<const int*>(a.pos)[at];
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
      const double angle = p * a.freq[i];
      const double turns = rint(angle * 0.15915494309189535);
      const double rest = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, angle));   // 2 pi in two parts
      float s, c;
      sincosf((float)rest, &s, &c);
      s = a.backward ? -s : s;
      cs[i] = make_float2(c * a.magnitude, s * a.magnitude);
    }
  }
  __syncthreads();
  // items of a row: those that turn, then the columns that are copied, 8 at a time
  const int turning = INTERLEAVED ? a.rot / 8 : half / VEC;
  const int tail = (a.D - a.rot) / 8, items = turning + tail;
  const int per = (int)blockDim.x / items;                  // rows at a time
  const int item = (int)threadIdx.x % items, r0 = (int)threadIdx.x / items;
  if (r0 >= per) return;
  const int rows = a.Hq + a.Hk;
  const long long q_in = b * a.q_s[0] + n * a.q_s[2], q_to = b * a.qo_s[0] + n * a.qo_s[2];
  const long long k_in = b * a.k_s[0] + n * a.k_s[2], k_to = b * a.ko_s[0] + n * a.ko_s[2];
  // four 16-byte loads at a time before the first store
  constexpr int BATCH = INTERLEAVED ? 4 : 2;
  const int at = item >= turning ? a.rot + 8 * (item - turning) : VEC * item;
  for (int r1 = r0; r1 < rows; r1 += BATCH * per) {
    uint4 u[BATCH], w[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int r = r1 + i * per;
      const bool is_q = r < a.Hq;
      if (r >= rows || (item >= turning && !(is_q ? a.copy_q : a.copy_k))) continue;
      const T* src = is_q ? reinterpret_cast<const T*>(a.q) + q_in + r * a.q_s[1] : reinterpret_cast<const T*>(a.k) + k_in + (r - a.Hq) * a.k_s[1];
      if (INTERLEAVED || VEC == 8 || item >= turning) {
        u[i] = ld_stream(src + at);
        if (!INTERLEAVED && item < turning) w[i] = ld_stream(src + half + at);
      } else {
        const uint2 lo = __ldcs(reinterpret_cast<const uint2*>(src + at)), hi = __ldcs(reinterpret_cast<const uint2*>(src + half + at));
        u[i] = make_uint4(lo.x, lo.y, 0u, 0u);
        w[i] = make_uint4(hi.x, hi.y, 0u, 0u);
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int r = r1 + i * per;
      const bool is_q = r < a.Hq;
      if (r >= rows || (item >= turning && !(is_q ? a.copy_q : a.copy_k))) continue;
      T* dst = is_q ? reinterpret_cast<T*>(a.q_out) + q_to + r * a.qo_s[1] : reinterpret_cast<T*>(a.k_out) + k_to + (r - a.Hq) * a.ko_s[1];
      if (item >= turning) {
        st_stream(dst + at, u[i]);
      } else if (INTERLEAVED) {
        float x[8];
        unpack8<T>(u[i], x);
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 t = cs[4 * item + e];
          o[e] = pack2<T>(x[2 * e] * t.x - x[2 * e + 1] * t.y, x[2 * e + 1] * t.x + x[2 * e] * t.y);
        }
        st_stream(dst + at, make_uint4(o[0], o[1], o[2], o[3]));
      } else {
        float x[8], y[8];
        uint32_t o[4], p[4];
        unpack8<T>(u[i], x);
        unpack8<T>(w[i], y);
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          const float2 t0 = cs[VEC * item + 2 * e], t1 = cs[VEC * item + 2 * e + 1];
          o[e] = pack2<T>(x[2 * e] * t0.x - y[2 * e] * t0.y, x[2 * e + 1] * t1.x - y[2 * e + 1] * t1.y);
          p[e] = pack2<T>(y[2 * e] * t0.x + x[2 * e] * t0.y, y[2 * e + 1] * t1.x + x[2 * e + 1] * t1.y);
        }
        if (VEC == 8) {
          st_stream(dst + at, make_uint4(o[0], o[1], o[2], o[3]));
          st_stream(dst + half + at, make_uint4(p[0], p[1], p[2], p[3]));
        } else {
          __stcs(reinterpret_cast<uint2*>(dst + at), make_uint2(o[0], o[1]));
          __stcs(reinterpret_cast<uint2*>(dst + half + at), make_uint2(p[0], p[1]));
        }
      }
    }
  }
}

// ---- quantising new rows into their pages ------------------------------------------------------------
// A group of LANES neighbouring lanes takes one (token, head): its K row and its V row, 16 columns per
// lane, all loads up front; the largest magnitude of a row is a few shuffles.  The arithmetic is the
// quantiser's (codes and scales are the bits that sage_prologue gives for the same rows): scale =
// max(amax / 127 or 448, 1e-12), code = rne(x / scale).  A row that holds a NaN or an infinity gets the scale
// NaN and codes of 0, so that no code is ever a NaN: a key that a mask hides cannot reach a product.
// Bound by HBM: 27 280 tokens x 48 heads 178 us = 5.7 TB/s (0.87 of a copy); 8771 x 8 heads 13 us = 4.2 TB/s, of which a
// launch and the first loads are 4.  32-byte loads, as when reading back, took 198 us for the former.

// Largest magnitude of sixteen packed values, NaN if one is.
template <typename T>
__device__ __forceinline__ float absmax16_nan(const uint4& u, const uint4& v) {
  typedef typename Packed16<T>::Pair Pair;
  const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
  Pair m = __habs2(*reinterpret_cast<const Pair*>(&w[0]));
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const Pair*>(&w[i])));
  const float2 f = Elem<T>::cvt2(*reinterpret_cast<const uint32_t*>(&m));
  return max_nan(f.x, f.y);
}

struct WriteKArgs {
  const void *k, *v, *slots;
  uint8_t *kc, *vc;
  float *ks, *vs;
  const float* shift;
  long long k_st, k_sh, v_st, v_sh;
  long long tokens, total_slots;
  int H, D, page_shift, slots64;
};

template <typename T, bool INT8, bool IS_K>
__device__ __forceinline__ float quant_row16(const uint4& u0, const uint4& u1, const float* shift, int col, int lanes, uint4* codes) {
  constexpr int QDIV = IS_K && INT8 ? 127 : 448;
  float x[16];
  unpack8<T>(u0, x);
  unpack8<T>(u1, x + 8);
  if (IS_K && shift != nullptr) {
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float4 m = __ldg(reinterpret_cast<const float4*>(shift + col + e));
      x[e] = __fsub_rn(x[e], m.x); x[e + 1] = __fsub_rn(x[e + 1], m.y); x[e + 2] = __fsub_rn(x[e + 2], m.z); x[e + 3] = __fsub_rn(x[e + 3], m.w);
    }
  }
  float amax = 0.f;
  if (IS_K && shift != nullptr) {
#pragma unroll
    for (int e = 0; e < 16; ++e) amax = max_nan(amax, fabsf(x[e]));
  } else {
    amax = absmax16_nan<T>(u0, u1);
  }
  for (int o = lanes / 2; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (!(amax <= 3.402823466e38f)) {                  // a NaN or an infinity somewhere in the row
    *codes = make_uint4(0u, 0u, 0u, 0u);
    return __int_as_float(0x7fffffff);
  }
  const float s = fmaxf(div_const<QDIV>(amax), SCALE_FLOOR);
  const float rc = __frcp_rn(s);
  const float2* x2 = reinterpret_cast<const float2*>(x);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (IS_K && INT8) {
      const float2 rc2 = make_float2(rc, rc), ns2 = make_float2(-s, -s);
      const float2 qa = __fmul2_rn(x2[2 * i], rc2), qb = __fmul2_rn(x2[2 * i + 1], rc2);
      w[i] = i8x4_magic2(__ffma2_rn(__ffma2_rn(qa, ns2, x2[2 * i]), rc2, qa), __ffma2_rn(__ffma2_rn(qb, ns2, x2[2 * i + 1]), rc2, qb));
    } else {
      w[i] = e4m3x4_quot(x2[2 * i], x2[2 * i + 1], s, rc);
    }
  }
  *codes = make_uint4(w[0], w[1], w[2], w[3]);
  return s;
}

template <typename T, bool INT8, int WIDTH>
__global__ void __launch_bounds__(CACHE_THREADS) cache_write_kernel(const WriteKArgs a) {
  constexpr int LANES = WIDTH / 16, ROWS = CACHE_THREADS / LANES;
  const int c = (int)threadIdx.x % LANES, col = 16 * c;
  // ROWS neighbouring tokens of one head: their codes and scales lie next to each other in a page (token by token and
  // head by head every scale would be a write of 4 bytes to a sector of its own)
  const unsigned block = blockIdx.x / (unsigned)a.H;
  const int h = (int)(blockIdx.x - block * a.H);
  long long token = (long long)block * ROWS + threadIdx.x / LANES;
  const bool live = token < a.tokens;
  token = live ? token : 0;
  const long long slot = !live ? -1 : a.slots64 ? reinterpret_cast<const long long*>(a.slots)[token] : (long long)reinterpret_cast<const int*>(a.slots)[token];
  const bool store = live && slot >= 0 && slot < a.total_slots;
  const T* k = reinterpret_cast<const T*>(a.k) + token * a.k_st + h * a.k_sh + col;
  const T* v = reinterpret_cast<const T*>(a.v) + token * a.v_st + h * a.v_sh + col;
  const bool lo = live && col < a.D, hi = live && col + 8 < a.D;
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
  const uint4 k0 = lo ? ld_stream(k) : none, k1 = hi ? ld_stream(k + 8) : none, v0 = lo ? ld_stream(v) : none, v1 = hi ? ld_stream(v + 8) : none;
  uint4 kw, vw;
  // (the shift is padded to the row's width with zeros)
  const float ks = quant_row16<T, INT8, true>(k0, k1, a.shift ? a.shift + (long long)h * WIDTH : nullptr, col, LANES, &kw);
  const float vs = quant_row16<T, INT8, false>(v0, v1, nullptr, col, LANES, &vw);
  if (!store) return;
  const long long page = slot >> a.page_shift, off = slot & ((1LL << a.page_shift) - 1);
  const long long at = ((page * a.H + h) << a.page_shift) + off;
  *reinterpret_cast<uint4*>(a.kc + at * WIDTH + col) = kw;
  *reinterpret_cast<uint4*>(a.vc + at * WIDTH + col) = vw;
  if (c == 0) { a.ks[at] = ks; a.vs[at] = vs; }
}

// ---- reading back --------------------------------------------------------------------------------------
// A CTA takes ROWS consecutive rows of the packed output and a share of the heads, a token per group of
// LANES lanes.  Consecutive tokens of a page and head lie next to each other in the cache, so a
// warp reads whole lines of codes and of scales.  value = code * scale (+ shift), in fp32, rounded once.
// Bound by HBM, two thirds of it writes: 27 280 tokens x 48 heads 197 us = 5.2 TB/s (0.79 of a copy).  More in flight
// does not help: with 2 heads at a time and 5 CTAs of 256 threads an SM 241 us, with 8 and 2 CTAs 232.
struct ReadKArgs {
  const uint8_t *kc, *vc;
  const float *ks, *vs, *shift;
  const int *table, *cu;
  void *k_out, *v_out;
  long long table_st, k_st, k_sh, v_st, v_sh, total;
  int n_seq, table_width, pages, H, D, page_shift;
};

// 16 codes -> 16 values, in pairs
template <bool INT8>
__device__ __forceinline__ void decode16(const uint4& u, float2* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (INT8) {
      const uint32_t t = w[i] ^ 0x80808080u;         // code + 128, then 2^23 + it as a float
      const float2 bias = make_float2(-8388736.0f, -8388736.0f);
      x[2 * i] = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(t, 0x4B000000u, 0x7440)), __uint_as_float(__byte_perm(t, 0x4B000000u, 0x7441))), bias);
      x[2 * i + 1] = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(t, 0x4B000000u, 0x7442)), __uint_as_float(__byte_perm(t, 0x4B000000u, 0x7443))), bias);
    } else {
      const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] & 0xFFFFu), __NV_E4M3);
      const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] >> 16), __NV_E4M3);
      x[2 * i] = __half22float2(*reinterpret_cast<const __half2*>(&lo));
      x[2 * i + 1] = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    }
  }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store16(T* dst, const float2* x, bool lo, bool hi) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack2<T>(x[i].x, x[i].y);
  st_stream32<WIDE>(dst, make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7]), lo, hi);
}

template <typename T, bool INT8, int WIDTH, bool WIDE>
__global__ void __launch_bounds__(CACHE_THREADS, 6) cache_read_kernel(const ReadKArgs a) {
  constexpr int LANES = WIDTH / 16, ROWS = CACHE_THREADS / LANES;
  constexpr int BATCH = 4;                           // heads whose codes are in flight together
  __shared__ long long where[ROWS];                  // first row of the token's page in head 0, plus its offset; -1: none
  const long long row0 = (long long)blockIdx.x * ROWS;
  if (threadIdx.x < ROWS) {
    const long long row = row0 + threadIdx.x;
    long long at = -2;                               // behind the last sequence: left as it is
    if (row < a.total && row >= a.cu[0] && row < a.cu[a.n_seq]) {
      int lo = 0, hi = a.n_seq;                      // cu[lo] <= row < cu[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.cu[mid] <= row) lo = mid; else hi = mid;
      }
      const long long t = row - a.cu[lo], p = t >> a.page_shift;
      at = -1;                                       // no such page: zeros
      if (t >= 0 && p < a.table_width) {
        const long long page = a.table[lo * a.table_st + p];
        if (page >= 0 && page < a.pages) at = ((page * a.H) << a.page_shift) + (t & ((1LL << a.page_shift) - 1));
      }
    }
    where[threadIdx.x] = at;
  }
  __syncthreads();
  const int r = (int)threadIdx.x / LANES, col = 16 * ((int)threadIdx.x % LANES);
  const long long row = row0 + r, at0 = where[r];
  if (at0 == -2) return;
  const bool lo = col < a.D, hi = col + 8 < a.D;
  T* k_out = reinterpret_cast<T*>(a.k_out) + row * a.k_st + col;
  T* v_out = reinterpret_cast<T*>(a.v_out) + row * a.v_st + col;
  const int step = (int)gridDim.y;
  for (int h0 = blockIdx.y; h0 < a.H; h0 += BATCH * step) {
    uint4 kw[BATCH], vw[BATCH];
    float ks[BATCH], vs[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = h0 + i * step;
      kw[i] = vw[i] = make_uint4(0u, 0u, 0u, 0u);
      ks[i] = vs[i] = 0.f;
      if (h < a.H && at0 >= 0) {
        const long long at = at0 + ((long long)h << a.page_shift);
        kw[i] = ld_stream(a.kc + at * WIDTH + col);
        vw[i] = ld_stream(a.vc + at * WIDTH + col);
        ks[i] = __ldg(a.ks + at);
        vs[i] = __ldg(a.vs + at);
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = h0 + i * step;
      if (h < a.H) {
        float2 x[8];
        const float2 k2 = make_float2(ks[i], ks[i]), v2 = make_float2(vs[i], vs[i]);
        decode16<INT8>(kw[i], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul2_rn(x[e], k2);
        if (a.shift != nullptr && at0 >= 0) {
          const float4* m4 = reinterpret_cast<const float4*>(a.shift + h * WIDTH + col);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 m = __ldg(m4 + e);
            x[2 * e] = __fadd2_rn(x[2 * e], make_float2(m.x, m.y));
            x[2 * e + 1] = __fadd2_rn(x[2 * e + 1], make_float2(m.z, m.w));
          }
        }
        store16<T, WIDE>(k_out + h * a.k_sh, x, lo, hi);
        decode16<false>(vw[i], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul2_rn(x[e], v2);
        store16<T, WIDE>(v_out + h * a.v_sh, x, lo, hi);
      }
    }
  }
}

// Whether every run of 16 columns of the rows lies on a multiple of 32 bytes, and none is cut off.
bool in_32s(const void* p, long long s0, long long s1, int d) {
  return (reinterpret_cast<uintptr_t>(p) & 31u) == 0 && s0 % 16 == 0 && s1 % 16 == 0 && d % 16 == 0;
}

template <typename T>
cudaError_t launch_rotary_t(const RotaryKArgs& a, bool interleaved, long long blocks, cudaStream_t st) {
  const int half = a.rot / 2;
  const bool vec8 = interleaved || half % 8 == 0;
  const int items = (interleaved ? a.rot / 8 : half / (vec8 ? 8 : 4)) + (a.D - a.rot) / 8;
  // four rows per thread, so that a CTA's loads are in flight together, and a thread per pair at least
  int threads = (items * ((a.Hq + a.Hk + 3) / 4) + 31) / 32 * 32;
  threads = std::min(CACHE_THREADS, std::max(64, threads));
  const dim3 grid((unsigned)blocks);
  if (interleaved) rotary_kernel<T, true, 8><<<grid, threads, 0, st>>>(a);
  else if (vec8) rotary_kernel<T, false, 8><<<grid, threads, 0, st>>>(a);
  else rotary_kernel<T, false, 4><<<grid, threads, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T, bool INT8>
cudaError_t launch_write_t(const WriteKArgs& a, int width, cudaStream_t st) {
  const long long per = CACHE_THREADS / (width / 16), blocks = (a.tokens + per - 1) / per * a.H;
  const dim3 grid((unsigned)blocks);
  if (width == 64) cache_write_kernel<T, INT8, 64><<<grid, CACHE_THREADS, 0, st>>>(a);
  else cache_write_kernel<T, INT8, 128><<<grid, CACHE_THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T, bool INT8>
cudaError_t launch_read_t(const ReadKArgs& a, int width, cudaStream_t st) {
  const long long per = CACHE_THREADS / (width / 16), blocks = (a.total + per - 1) / per;
  // heads shared out until there are a few CTAs per SM
  const long long want = 8LL * sm_count();
  const dim3 grid((unsigned)blocks, (unsigned)std::max(1LL, std::min((long long)a.H, want / blocks)));
  const bool wide = in_32s(a.k_out, a.k_st, a.k_sh, a.D) && in_32s(a.v_out, a.v_st, a.v_sh, a.D);
  if (width == 64) (wide ? cache_read_kernel<T, INT8, 64, true> : cache_read_kernel<T, INT8, 64, false>)<<<grid, CACHE_THREADS, 0, st>>>(a);
  else (wide ? cache_read_kernel<T, INT8, 128, true> : cache_read_kernel<T, INT8, 128, false>)<<<grid, CACHE_THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 64 && (sms = known[dev].load(std::memory_order_relaxed)) > 0) return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 64) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

cudaError_t launch_rotary(const RotaryParams& p, cudaStream_t st) {
  RotaryKArgs a;
  a.q = p.q; a.k = p.k; a.pos = p.pos; a.q_out = p.q_out; a.k_out = p.k_out; a.freq = p.freq;
  bool same_q = p.q == p.q_out, same_k = p.k == p.k_out;
  for (int i = 0; i < 3; ++i) {
    a.q_s[i] = p.q_strides[i]; a.qo_s[i] = p.qo_strides[i]; a.k_s[i] = p.k_strides[i]; a.ko_s[i] = p.ko_strides[i];
    same_q = same_q && a.q_s[i] == a.qo_s[i]; same_k = same_k && a.k_s[i] == a.ko_s[i];
  }
  a.pos_s[0] = p.pos_strides[0]; a.pos_s[1] = p.pos_strides[1];
  a.magnitude = p.magnitude; a.Hq = (int)p.Hq; a.Hk = (int)p.Hk; a.N = (int)p.N; a.D = (int)p.D; a.rot = (int)p.rot;
  a.pos64 = p.pos64; a.backward = p.backward; a.copy_q = !same_q; a.copy_k = !same_k;
  return p.dtype == 0 ? launch_rotary_t<__half>(a, p.interleaved != 0, p.B * p.N, st)
                      : launch_rotary_t<__nv_bfloat16>(a, p.interleaved != 0, p.B * p.N, st);
}

cudaError_t launch_cache_write(const CacheView& c, const CacheWriteParams& p, cudaStream_t st) {
  WriteKArgs a;
  a.k = p.k; a.v = p.v; a.slots = p.slots; a.kc = c.k_codes; a.vc = c.v_codes; a.ks = c.k_scale; a.vs = c.v_scale; a.shift = c.k_shift;
  a.k_st = p.k_strides[0]; a.k_sh = p.k_strides[1]; a.v_st = p.v_strides[0]; a.v_sh = p.v_strides[1];
  a.tokens = p.tokens; a.total_slots = c.pages << c.page_shift;
  a.H = (int)c.H; a.D = (int)c.D; a.page_shift = c.page_shift; a.slots64 = p.slots64;
  if (p.dtype == 0) return c.int8 ? launch_write_t<__half, true>(a, c.width, st) : launch_write_t<__half, false>(a, c.width, st);
  return c.int8 ? launch_write_t<__nv_bfloat16, true>(a, c.width, st) : launch_write_t<__nv_bfloat16, false>(a, c.width, st);
}

cudaError_t launch_cache_read(const CacheView& c, const CacheReadParams& p, cudaStream_t st) {
  ReadKArgs a;
  a.kc = c.k_codes; a.vc = c.v_codes; a.ks = c.k_scale; a.vs = c.v_scale; a.shift = c.k_shift;
  a.table = p.table; a.cu = p.cu; a.k_out = p.k_out; a.v_out = p.v_out; a.table_st = p.table_stride;
  a.k_st = p.k_strides[0]; a.k_sh = p.k_strides[1]; a.v_st = p.v_strides[0]; a.v_sh = p.v_strides[1];
  a.total = p.total; a.n_seq = (int)p.n_seq; a.table_width = (int)p.table_width; a.pages = (int)c.pages;
  a.H = (int)c.H; a.D = (int)c.D; a.page_shift = c.page_shift;
  if (p.dtype == 0) return c.int8 ? launch_read_t<__half, true>(a, c.width, st) : launch_read_t<__half, false>(a, c.width, st);
  return c.int8 ? launch_read_t<__nv_bfloat16, true>(a, c.width, st) : launch_read_t<__nv_bfloat16, false>(a, c.width, st);
}

}  // namespace sage
