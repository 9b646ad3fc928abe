// What the kernels of sageattn_cached share: arguments, the line of work, and its division (see sage_cache_attn.cu).
#pragma once

#include <algorithm>
#include <atomic>

#include "sage_common.cuh"
#include "sage_internal.h"
#include "sage_ptx.cuh"

namespace sage {

constexpr float LN2_F = 0.6931471805599453f;
constexpr float NO_MAX = -3.0e38f;
// Weights of V enter their product in fp16.  A row's largest one is put at 2^TOP_LOG2, and the row is scaled anew once one
// passes 2^LIMIT_LOG2 (fp16 ends below 2^16): a weight keeps its 11 bits down to 2^-18 of the largest and is lost below 2^-29 of
// it.  At 2^0 that was 2^-25: 262 144 keys at 2^-25.2 of a first one, 6.8e-3 of the output.  The room above keeps rows from being
// scaled anew with every new maximum: 8 x 16 384 keys, some of them four times as large as the others, 256 rows: 204.8 us at
// 2^0, 211.2 at 2^4, 214.5 at 2^6, 217 at 2^8; 32 rows 105, 107, 110.5, 109.6.  Beyond 2^4 nothing is to be had: the fp32
// accumulators lose up to 2^-23 of the sum per 16 keys, more than this.
constexpr int TOP_LOG2 = 4, LIMIT_LOG2 = 15;

struct CacheAttnKArgs {
  const void* q;
  void* out;
  float* lse;
  const uint8_t *kc, *vc;
  const float *ks, *vs, *shift;
  const int *table, *seqlens, *cu_q;
  const uint8_t* tree;
  float* part_o;             // (2 x stretches, part_rows, WIDTH)
  float2* part_ml;           // (2 x stretches, part_rows): running maximum (log2 domain), sum
  long long q_st, q_sh, o_st, o_sh, table_st, tree_st;
  long long total_q;
  int n_seq, table_width, pages, page_shift, Hq, Hkv, group, max_q, D;
  int max_stretches;         // the line of steps is cut into so many stretches
  int part_rows;             // rows of a partial result: those of a row tile that can exist
  float sm_scale, scale_log2;
};

// A sequence as the kernels see it: lengths clamped, so that no access leaves the tensors whatever the arrays hold.
struct Seq {
  int q0, q_len, len;
};
__device__ __forceinline__ Seq seq_of(const CacheAttnKArgs& a, int b) {
  Seq s;
  if (a.cu_q == nullptr) {                           // max_q new tokens for every sequence
    s.q0 = b * a.max_q;
    s.q_len = a.max_q;
  } else {
    const long long q0 = min(max((long long)__ldg(a.cu_q + b), 0LL), a.total_q);
    s.q0 = (int)q0;
    s.q_len = (int)min(max(min((long long)__ldg(a.cu_q + b + 1), a.total_q) - q0, 0LL), (long long)a.max_q);
  }
  s.len = (int)min(max((long long)__ldg(a.seqlens + b), 0LL), (long long)a.table_width << a.page_shift);
  return s;
}
__device__ __forceinline__ int row_tiles(const CacheAttnKArgs& a, const Seq& s, int rows) { return (s.q_len * a.group + rows - 1) / rows; }
// (an empty sequence's rows are written too)
__device__ __forceinline__ int key_steps(const Seq& s, int keys) { return max(1, (s.len + keys - 1) / keys); }

// The line of steps (of so many keys each): sequence by sequence, K/V head by K/V head, row tile by row tile (of so many
// rows each), step by step, and behind every unit UNIT_STEPS more places that stand for what a unit costs beyond its keys
// (fetching Q, writing the rows): without them a stretch through many short sequences takes several times as long as one
// through a long one (32 ragged sequences of up to 8192 keys, a token each: 56 us without them, 45 with them at the time).
// There are fewer than 2^31 places, the host sees to that.  The line's stretches differ by one place at most; a line of
// fewer places than stretches wanted leaves the last ones out.
constexpr int UNIT_STEPS = 4;
struct Line {
  unsigned total, n, per, longer;                    // places, stretches, places of a stretch, stretches that have one more
  __device__ __forceinline__ Line(unsigned places, int most) : total(places) {
    n = min((unsigned)most, places);
    per = n ? places / n : 0u;
    longer = places - n * per;
  }
  __device__ __forceinline__ unsigned begin(unsigned x) const { return x * per + min(x, longer); }
  // the stretch that has place u
  __device__ __forceinline__ unsigned of(unsigned u) const {
    const unsigned in_longer = longer * (per + 1);
    return u < in_longer ? u / (per + 1) : longer + (u - in_longer) / per;
  }
};
__device__ __forceinline__ unsigned places_of_seq(const CacheAttnKArgs& a, int b, int rows, int keys) {
  if (b >= a.n_seq) return 0;
  const Seq s = seq_of(a, b);
  return (unsigned)a.Hkv * row_tiles(a, s, rows) * (key_steps(s, keys) + UNIT_STEPS);
}

// All threads of a CTA call this: the line, the sequence in which the CTA's stretch `which` (of OWN) begins (n_seq: it
// has none), and the number of places before that sequence.
template <int THREADS, int OWN> struct PlaceScratch {
  unsigned sum[THREADS / 32], found[OWN], before[OWN];
};
template <int THREADS, int OWN>
__device__ __forceinline__ Line find_place(const CacheAttnKArgs& a, int rows, int keys, PlaceScratch<THREADS, OWN>& sh, int which, int& seq,
                                           unsigned& places_before) {
  constexpr int WARPS = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned total = 0;
  if (a.n_seq > THREADS) {                           // the length of the line first
    unsigned mine = 0;
    for (int b = tid; b < a.n_seq; b += THREADS) mine += places_of_seq(a, b, rows, keys);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sh.sum[warp] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += sh.sum[w];
    __syncthreads();
  }
  if (tid < OWN) sh.found[tid] = a.n_seq;
  Line line(total, a.max_stretches);
  unsigned base = 0;
  for (int b0 = 0; b0 < a.n_seq; b0 += THREADS) {
    const unsigned n = places_of_seq(a, b0 + tid, rows, keys);
    unsigned upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) sh.sum[warp] = upto;
    __syncthreads();
    unsigned before = base + upto - n;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += sh.sum[w];
      base += sh.sum[w];
    }
    if (a.n_seq <= THREADS) line = Line(base, a.max_stretches);
#pragma unroll
    for (int w = 0; w < OWN; ++w) {
      const unsigned x = blockIdx.x * OWN + w, want = line.begin(x);
      if (x < line.n && want >= before && want - before < n) { sh.found[w] = b0 + tid; sh.before[w] = before; }
    }
    __syncthreads();
  }
  seq = (int)sh.found[which];
  places_before = sh.before[which];
  return line;
}

// A position on the line, within a stretch.
struct Cursor {
  Seq s;
  int b, h, rt, kt;          // sequence, K/V head, row tile, step
  int n_rt, n_kt;
  int left;                  // places of the stretch from this one on; the walk is over when none is
  int into;                  // places of the stretch before the unit's first (below 0: the unit began before the stretch)
};
__device__ __forceinline__ void enter_seq(const CacheAttnKArgs& a, Cursor& c, int rows, int keys) {
  c.s = seq_of(a, c.b);
  c.n_rt = row_tiles(a, c.s, rows);
  c.n_kt = key_steps(c.s, keys);
}
// From any place of a unit (`at` of them into it) to the first of the next one.
__device__ __forceinline__ void next_unit(const CacheAttnKArgs& a, Cursor& c, int at, int rows, int keys) {
  const int rest = c.n_kt + UNIT_STEPS - at;
  c.left -= rest;
  c.into += c.n_kt + UNIT_STEPS;
  c.kt = 0;
  if (c.left <= 0 || ++c.rt < c.n_rt) return;
  c.rt = 0;
  if (++c.h < a.Hkv) return;
  c.h = 0;
  do {
    if (++c.b >= a.n_seq) { c.left = 0; return; }
    enter_seq(a, c, rows, keys);
  } while (c.n_rt == 0);
}
__device__ __forceinline__ void next_step(const CacheAttnKArgs& a, Cursor& c, int rows, int keys) {
  if (c.kt + 1 < c.n_kt) {
    ++c.kt;
    --c.left;
  } else {
    next_unit(a, c, c.kt, rows, keys);
  }
}
// The first step of the stretch from place `first` on, in the sequence that find_place gave.
__device__ __forceinline__ void enter_line(const CacheAttnKArgs& a, Cursor& c, unsigned first, unsigned end, unsigned before, int rows, int keys) {
  enter_seq(a, c, rows, keys);
  const unsigned rest = first - before, per = (unsigned)(c.n_kt + UNIT_STEPS), unit = rest / per;
  const int at = (int)(rest - unit * per);
  c.h = (int)(unit / (unsigned)c.n_rt);
  c.rt = (int)unit - c.h * c.n_rt;
  c.kt = at;
  c.left = (int)(end - first);
  c.into = -at;
  if (at >= c.n_kt) next_unit(a, c, at, rows, keys);
}

// sum += x with the rounding error carried along: a row may see 2^30 keys, and weights that are each below the last bit of
// the sum so far still count.
__device__ __forceinline__ void add_carrying(float& sum, float& carry, float x) {
  const float y = x - carry, t = sum + y;
  carry = (t - sum) - y;
  sum = t;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  const int bytes = there ? 16 : 0;                  // 0: filled with zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float lds_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
// sm_scale * (row of Q) . (shift of the K/V head), by one warp
template <typename T>
__device__ __forceinline__ float shift_dot(const CacheAttnKArgs& a, const T* q, int h, int width, int lane) {
  float d = 0.f;
  for (int i = lane; i < a.D; i += 32) d = fmaf((float)q[i], __ldg(a.shift + (long long)h * width + i), d);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  return d * a.sm_scale;
}
// Two fp16 values of Q, an infinity as a NaN.  A row that holds one has no softmax; its scores may all be -infinity, which is what
// a key that is not seen gets.
__device__ __forceinline__ uint32_t inf_to_nan(uint32_t w) {
  const __half2 h = *reinterpret_cast<const __half2*>(&w), x = __hfma2(h, __half2half2(__ushort_as_half(0)), h);
  return *reinterpret_cast<const uint32_t*>(&x);
}
// Four e4m3 codes -> two registers of two fp16 each.
__device__ __forceinline__ void e4m3_quad(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, x;\n\tcvt.rn.f16x2.e4m3x2 %1, y;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
// Four K codes -> two registers of two fp16 each.
template <bool INT8>
__device__ __forceinline__ void k_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (INT8) {
    const uint32_t t = w ^ 0x80808080u;                              // code + 128 in a byte; 0x6400 + it is 1024 + it
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));     // 1024 + 128
    uint32_t u = __byte_perm(t, 0x64646464u, 0x4140), v = __byte_perm(t, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&u), bias), y = __hsub2(*reinterpret_cast<__half2*>(&v), bias);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    e4m3_quad(w, lo, hi);
  }
}
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Runs something once per device (a kernel's attributes; doing it twice at the same time does no harm).
struct DeviceOnce {
  std::atomic<unsigned long long> done{0};           // a bit per device; further ones ask every time
  template <typename F> cudaError_t run(F&& f) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = f();
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
  }
};
// Joins partial results (see sage_cache_attn.cu); rows and keys are those of a row tile and of a step.
cudaError_t launch_cache_combine(const CacheAttnKArgs& a, int dtype, int rows, int keys, int width, int max_rt, cudaStream_t st);
// The kernel for many rows (see sage_cache_tree.cu); status_host: optional pinned word for its bounded waits.
cudaError_t launch_cache_tree(CacheAttnKArgs& a, const CacheView& c, int dtype, int sms, int32_t* status_host, cudaStream_t st);
// How a call is served, as host arithmetic: rows of a row tile, keys of a step, stretches at most on any device.
struct CacheForm {
  bool tree;
  int rows, keys, max_stretches;
};
CacheForm cache_form(int64_t rows);

}  // namespace sage
