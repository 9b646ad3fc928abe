// sageattn_cached for many rows: trees and chains of drafted tokens whose rows (new token x query head of the
// group) fill the tensor core's 128-row operand.  Same formulas, line of work and partial results as
// sage_cache_attn.cu; the products are tcgen05.mma with accumulators in TMEM.
//
// A CTA takes a row tile of NQ x 128 rows and walks its stretch of the keys, 64 at a time:
//   warps 0 .. 4 NQ - 1   softmax: a thread owns a row (32x32b TMEM loads: a lane is a row), so that maxima and sums
//                         need no other lane; its weights go back to TMEM as fp16, over the scores they came from, and
//                         are the A operand of P V from there
//   the next four warps   fetch the one-byte codes (cp.async, some tiles ahead; every thread reads back only what it
//                         fetched), turn them into fp16 -- exact -- and write them to shared memory as the operands
//                         want them (128-byte swizzle)
//   NQ more warps         a thread each that issues the products of 128 rows (idle warps complete the warpgroup, whose
//                         registers the softmax takes over)
// Scores have two buffers in TMEM: those of the next tile are under way while the softmax works on a tile, and P V
// follows behind.  K is a K-major operand; V, whose rows are keys too, is the MN-major B operand of P V: both are
// written alike, a row of 64 columns in 128 bytes.  Heads of more than 64 columns take two such halves; columns 16 p ..
// 16 p + 7 of a row go to piece p of the first half and the next 8 to piece p of the second, for K, Q and V alike, so
// that the eight lanes that write the pieces of a row reach all banks (the order of an inner product's columns is
// free, and that of V's is undone where the output is written).
//
// The scale of V goes into the exponent: e = score + log2(scale), the weight is 2^(e - m) and the row's sum takes the weight
// over the scale, so that one maximum serves both the softmax and fp16's range: m is 2^TOP_LOG2 below the largest e.
//
// NQ = 2 (rows beyond 128): one CTA per SM with all 512 TMEM columns.  NQ = 1: two CTAs per SM.  (Rows are added to a
// CTA before CTAs are: a tile's codes are fetched and converted once per CTA.  Figures of both: cache_form.)
//
// What bounds it.  8 x 16 384 keys x 8 heads, 256 rows: 212 us in a graph = 646 TFLOP/s, 0.39 of the rate of a large 16-bit
// product; a chain of 512 new tokens, 2048 rows: 1512 us = 716.  A tile of 64 keys takes about 3000 cycles of an SM, and no part
// of it alone decides: the tensor pipe is busy a third of them, MUFU a third, half of the issue slots are used, and shared
// memory serves threads in 43 % and the tensor pipe in 39 %.  When it took 213 us, it would have been 173 without the softmax's
// arithmetic, 195 without fetching and converting the codes, 108 without either's work and one product per tile; twice the
// softmax warps (half the keys of a row each), separate warps for K and V, separate threads for the two products, or
// a row's scores spread over four lanes (fewer reads of scales) took 211 to 231.  The issuing warps spill: 372 bytes of stores
// and 224 of loads per thread at width 128 (472 and 284 at 64), the 128-row form 428 to 440 and 312 to 372.
// 4 x 8771 keys, 84 rows: 37 us for 3.9 us of bytes; the same cycles for tiles that are two thirds full.
//
// Every wait is bounded (about a second): it then leaves a code in the caller's pinned host word, the CTA drains
// its products, frees its TMEM and returns.
#include "sage_cache_attn.cuh"

namespace sage {

namespace {

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
constexpr uint32_t WAIT_CYCLES = 2000000000u;        // about a second of SM clock
struct Watch {
  volatile uint32_t* abort;                          // in shared memory: someone of this CTA gave up
  int32_t* host;                                     // optional pinned word
};
__device__ __forceinline__ uint32_t clock32() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%clock;" : "=r"(t));
  return t;
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {             // (sleeps up to 20 us for it)
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
  return ok != 0u;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const Watch& w, int code) {
  if (__builtin_expect(mbar_try(bar, parity), 1)) return true;
  const uint32_t t0 = clock32();
#pragma unroll 1
  while (!mbar_try(bar, parity)) {
    if (*w.abort) return false;
    if (clock32() - t0 > WAIT_CYCLES) {
      *w.abort = 1u;
      if (w.host != nullptr) *reinterpret_cast<volatile int32_t*>(w.host) = code;
      return false;
    }
  }
  return true;
}
// Until this CTA's own products are complete, whoever has given up on anything: what they read and write stays theirs.
__device__ __forceinline__ void drain_wait(uint32_t bar, const Watch& w, int code) {
  const uint32_t t0 = clock32();
#pragma unroll 1
  while (!mbar_try(bar, 0)) {
    if (clock32() - t0 > WAIT_CYCLES) {
      if (w.host != nullptr) *reinterpret_cast<volatile int32_t*>(w.host) = code;
      return;
    }
  }
}
enum { CODE_LOAD = 1, CODE_MMA = 2, CODE_SOFTMAX = 4 };   // the bits of the framework's status words

// Descriptors of operands in shared memory have the same upper word throughout (rows of 128 bytes, swizzled, eight of
// them 1024 bytes apart); of the lower one the address moves, by constants within a tile.
constexpr uint32_t DESC_HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_desc, uint32_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
               ::"r"(d), "r"(a_desc), "r"(b_desc), "r"(idesc), "r"(accumulate), "n"(DESC_HIGH) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
               ::"r"(d), "r"(a_tmem), "r"(b_desc), "r"(idesc), "r"(accumulate), "n"(DESC_HIGH) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr) : "memory");
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts_f32(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }

// Descriptors of 128-byte rows in the 128-byte swizzle, 8-row groups 1024 bytes apart: as a K-major operand, and as
// an MN-major one whose next 64 columns lie `lead` bytes further.
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr, uint32_t lead) { return ((addr & 0x3FFFFu) >> 4) | ((lead >> 4) << 16); }

// 16 codes -> 16 fp16 in eight registers, exact.
template <bool INT8>
__device__ __forceinline__ void codes_to_half(const uint4& u, uint32_t (&h)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) k_halves<INT8>(w[i], h[2 * i], h[2 * i + 1]);
}

constexpr int KT = 64;                               // keys of a tile
template <int WIDTH, int NQ> struct TreeShape {
  static constexpr int SOFTMAX = 128 * NQ, LOADERS = 128, THREADS = SOFTMAX + LOADERS + 128;
  static constexpr int CTAS_PER_SM = NQ == 1 ? 2 : 1;
  // Registers per thread: at launch (what __launch_bounds__ leaves: 65536 / threads of the SM, in eights), and after the
  // warpgroups have shared them out.  setmaxnreg.inc waits until the pool holds what it asks for, so that the shares
  // must not add up to more than the launch has.
  static constexpr int REGS_LAUNCH = NQ == 1 ? 80 : 128, REGS_SOFTMAX = NQ == 1 ? 120 : 168, REGS_LOADER = NQ == 1 ? 72 : 112,
                       REGS_ISSUER = NQ == 1 ? 48 : 64;
  static_assert(NQ * REGS_SOFTMAX + REGS_LOADER + REGS_ISSUER <= (NQ + 2) * REGS_LAUNCH, "setmaxnreg would wait forever");
  // Stages of K and V as operands, and of codes as they come: a ring of four for NQ = 2 (213 us at the time; codes held in registers a
  // tile ahead 243), none for NQ = 1, whose two CTAs share the memory: codes come through registers and leave room for two
  // stages of operands (8 x 16 384 keys, 128 rows: 150 us; with a ring and one stage 181).  Slots of scales: one is written
  // once the scores STAGES tiles back are complete, which means that the softmax is done with the tile two before that.
  static constexpr int STAGES = 2, SLOTS = 4, RAW_STAGES = NQ == 1 ? 0 : 4;
  static_assert(SLOTS >= STAGES + 2, "");
  static constexpr uint32_t HALVES = WIDTH / 64;
  static constexpr uint32_t Q_HALF = 128 * 128, Q_TILE = HALVES * Q_HALF;             // 128 rows of 128 bytes
  static constexpr uint32_t KV_HALF = KT * 128, KV_TILE = HALVES * KV_HALF;
  static constexpr uint32_t RAW_TILE = 2 * KT * WIDTH + 2 * KT * 4;                   // codes and scales of K and V as they come
  static constexpr uint32_t OFF_Q = 0, OFF_K = NQ * Q_TILE, OFF_V = OFF_K + STAGES * KV_TILE, OFF_RAW = OFF_V + STAGES * KV_TILE;
  static constexpr uint32_t OFF_SC = OFF_RAW + RAW_STAGES * RAW_TILE;
  // of a tile: scales of K, log2 and reciprocal of the scales of V, and for every 32 keys {two words with a bit for each: the
  // first alone for a key that does not exist, the second alone for a NaN in K, both for one in V alone; the largest and
  // the smallest log2 of a scale of V}
  static constexpr uint32_t SLOT_LV = KT * 4, SLOT_RV = KT * 8, SLOT_SUM = KT * 12, SLOT = SLOT_SUM + KT / 2;
  static constexpr uint32_t OFF_ROW = OFF_SC + SLOTS * SLOT;                          // two floats per row
  static constexpr uint32_t OFF_BAR = OFF_ROW + SOFTMAX * 8;
  // Barriers: per half of the rows (QF) and score buffer (SF, PF, PV), per stage (KF, KE, VF, VE), per slot (SC).  A wait by
  // parity must find its barrier in the phase it waits for, or just past it.  Those of a half count its own tiles: the
  // scores of a tile are issued after P V of the tile two before, which waited for that tile's weights.  Those of the
  // stages are waited for by loaders and issuers, which go through every tile, whether or not a half has rows.  The slots'
  // are the exception: the softmax of a half without rows passes over a unit's tiles, and its next tile may be many phases
  // ahead of the slot's barrier, where a wait by parity means nothing.  It therefore waits for its scores first.  Their products
  // were issued after KF of the tile, which every loader warp arrives on after SC, so that the slot's phase is complete
  // by then; and it is the last one that is, for a slot is written again only after the scores two tiles on, which follow
  // this tile's weights.
  static constexpr int B_QF = 0, B_PV = 2, B_SF = 6, B_PF = 10, B_DRAIN = 14, B_KF = 15, B_KE = B_KF + STAGES, B_VF = B_KE + STAGES,
                       B_VE = B_VF + STAGES, B_SC = B_VE + STAGES, B_COUNT = B_SC + SLOTS;
  static constexpr uint32_t OFF_MISC = OFF_BAR + (B_COUNT * 8 + 15) / 16 * 16, USED = OFF_MISC + 16;
  static constexpr uint32_t BYTES = USED + 1024;                                      // slack for the 1024-byte alignment
  static constexpr uint32_t TMEM_COLS = NQ * (2 * KT + WIDTH) <= 256 ? 256 : 512;
  static constexpr int ROWS = 128 * NQ;
};

template <typename T, bool INT8, int WIDTH, int NQ>
__global__ void __launch_bounds__(TreeShape<WIDTH, NQ>::THREADS, TreeShape<WIDTH, NQ>::CTAS_PER_SM)
cache_tree_kernel(const CacheAttnKArgs a, int32_t* status_host) {
  using L = TreeShape<WIDTH, NQ>;
  constexpr int ROWS = L::ROWS;
  constexpr uint32_t IDESC_QK = (1u << 4) | ((uint32_t)(KT >> 3) << 17) | (8u << 24);
  constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(WIDTH >> 3) << 17) | (8u << 24);   // B is MN-major
  extern __shared__ uint8_t smem_raw[];
  __shared__ PlaceScratch<L::THREADS, 1> place_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  allow_successor();
  Cursor cur;
  unsigned before;
  const Line line = find_place<L::THREADS, 1>(a, ROWS, KT, place_s, 0, cur.b, before);
  if (cur.b >= a.n_seq) return;                      // (the whole CTA)
  enter_line(a, cur, line.begin(blockIdx.x), line.begin(blockIdx.x + 1), before, ROWS, KT);
  if (cur.left <= 0) return;

  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, bar0 = base + L::OFF_BAR;
  uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(gbase + L::OFF_MISC);   // [0] TMEM address, [1] abort
  const Watch watch = {misc + 1, status_host};
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(bar(L::B_QF + i), 4);
    for (int i = 0; i < 4; ++i) { mbar_init(bar(L::B_SF + i), 1); mbar_init(bar(L::B_PF + i), 4); mbar_init(bar(L::B_PV + i), 1); }
    for (int i = 0; i < L::STAGES; ++i) {
      mbar_init(bar(L::B_KF + i), 4); mbar_init(bar(L::B_KE + i), NQ);
      mbar_init(bar(L::B_VF + i), 4); mbar_init(bar(L::B_VE + i), NQ);
    }
    for (int i = 0; i < L::SLOTS; ++i) mbar_init(bar(L::B_SC + i), KT / 32);
    mbar_init(bar(L::B_DRAIN), NQ);
    misc[1] = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  constexpr int ISSUER = (L::SOFTMAX + L::LOADERS) / 32;
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + L::OFF_MISC), "r"(L::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = misc[0];
  auto tmem_s = [&](int g, int buf) { return tmem + (uint32_t)((2 * g + buf) * KT); };
  auto tmem_o = [&](int g) { return tmem + (uint32_t)(2 * NQ * KT + g * WIDTH); };
  // halves of a row tile that hold rows
  auto halves_of = [&](const Cursor& c) { return NQ == 2 && c.s.q_len * a.group - c.rt * ROWS > 128 ? 2 : 1; };

  if (tid < L::SOFTMAX) {
    // ------------------------------------------------- softmax -------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::REGS_SOFTMAX));
    const int g = warp >> 2, r = tid & 127;
    const uint32_t lane_sel = (uint32_t)(warp & 3) << 21;                             // 32 lanes of TMEM per warp
    const uint32_t o_addr = tmem_o(g) + lane_sel;
    // Of row r: [r] what undoes its power of two (read once; a NaN from then on: the row sees one in V alone), [128 + r] its
    // product with the shift.
    float* row_at = reinterpret_cast<float*>(gbase + L::OFF_ROW) + 256 * g;
    // Rows of 2 * WIDTH bytes in this half's Q tile: piece c of row r, where Q goes and outputs pass through.
    uint8_t* q_tile = gbase + L::OFF_Q + g * L::Q_TILE;
    auto staged = [&](int row, int c) { return reinterpret_cast<uint4*>(q_tile + (c >> 3) * L::Q_HALF + row * 128 + 16 * ((c & 7) ^ (row & 7))); };
    // A warp moves whole rows of its 32: PIECES lanes a row, RPI rows at a time.
    constexpr int PIECES = WIDTH / 8, RPI = 32 / PIECES;
    const int c_l = lane % PIECES, row_l = 32 * (warp & 3) + lane / PIECES;
    bool ok = true;
    int n = 0, done = 0;                             // tiles of the CTA, and of this half, that are behind
    while (ok && cur.left > 0) {
      const int count = min(cur.left, cur.n_kt - cur.kt), kt0 = cur.kt;
      const int first_row = cur.rt * ROWS + 128 * g, live = cur.s.q_len * a.group - first_row;   // rows of this half that exist
      const int rr = first_row + r, tok = rr / a.group;
      const bool exists = r < live;
      // (offset of a row of q or out in elements)
      auto row_of = [&](int row, long long st, long long sh) -> long long {
        const int x = first_row + row, token = x / a.group;
        return (long long)(cur.s.q0 + token) * st + (long long)(cur.h * a.group + x - token * a.group) * sh;
      };
      if (g < halves_of(cur)) {
        const bool whole = kt0 == 0 && count == cur.n_kt, dots = whole && a.lse != nullptr && a.shift != nullptr;
        float shift[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};                    // of this lane's columns
        if (dots) {
#pragma unroll
          for (int e = 0; e < 8; ++e) shift[e] = __ldg(a.shift + (long long)cur.h * WIDTH + 8 * c_l + e);
        }
#pragma unroll 8
        for (int i = 0; i < 32 / RPI; ++i) {
          const int row = row_l + i * RPI;
          uint4 u = make_uint4(0u, 0u, 0u, 0u);
          if (row < live && 8 * c_l < a.D) u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + row_of(row, a.q_st, a.q_sh) + 8 * c_l));
          if (dots) {
            float x[8], d = 0.f;
            unpack8<T>(u, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) d = fmaf(x[e], shift[e], d);
#pragma unroll
            for (int o = PIECES / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
            if (c_l == 0) row_at[128 + row] = d * a.sm_scale;
          }
          float back = 1.f;                          // what undoes the row's power of two
          if (!__is_same(T, __half)) {               // bf16: the row's largest element to [2^14, 2^15)
            float x[8], amax = 0.f;
            unpack8<T>(u, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
#pragma unroll
            for (int o = PIECES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const int field = (int)(__float_as_uint(amax) >> 23);
            float up = 1.f;
            if (field > 14 && field < 255) {
              const int f = min(254, 268 - field);
              up = __uint_as_float((uint32_t)f << 23);
              back = f <= 253 ? __uint_as_float((uint32_t)(254 - f) << 23) : 5.877471754111438e-39f;
            }
            u = make_uint4(pack2<__half>(x[0] * up, x[1] * up), pack2<__half>(x[2] * up, x[3] * up), pack2<__half>(x[4] * up, x[5] * up),
                           pack2<__half>(x[6] * up, x[7] * up));
          }
          u = make_uint4(inf_to_nan(u.x), inf_to_nan(u.y), inf_to_nan(u.z), inf_to_nan(u.w));
          *staged(row, WIDTH == 128 ? (c_l & 1) * 8 + (c_l >> 1) : c_l) = u;
          if (c_l == 0) row_at[row] = fmaxf(a.scale_log2 * back, 1.17549435e-38f);    // (a masked score stays -infinity)
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::B_QF + g));
        const float row_c = row_at[r];
        const int ctx = cur.s.len - cur.s.q_len;
        const int plain_end = a.tree ? max(ctx, 0) : max(0, min(cur.s.len, ctx + first_row / a.group + 1));   // keys below need no mask
        const int lim = exists ? (a.tree ? cur.s.len : min(cur.s.len, ctx + tok + 1)) : 0;
        const uint8_t* tree_row = a.tree ? a.tree + (long long)(cur.s.q0 + tok) * a.tree_st : nullptr;
        // m: running maximum of e; l: sum of the weights of V over their scales, and what its rounding carries
        float m = NO_MAX, l = 0.f, l_carry = 0.f;
        const float2 c2 = make_float2(row_c, row_c);

        for (int t = 0; t < count; ++t) {
          const int k = done + t, buf = k & 1;       // tiles of this half so far
          ok = mbar_wait(bar(L::B_SF + 2 * g + buf), (uint32_t)(k >> 1) & 1u, watch, CODE_SOFTMAX) &&
               mbar_wait(bar(L::B_SC + (n + t) % L::SLOTS), (uint32_t)((n + t) / L::SLOTS) & 1u, watch, CODE_SOFTMAX);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint32_t s_addr = tmem_s(g, buf) + lane_sel;
          uint32_t x[64];
          tmem_ld32(s_addr, x);
          tmem_ld32(s_addr + 32, x + 32);
          const uint8_t* slot_at = gbase + L::OFF_SC + ((n + t) % L::SLOTS) * L::SLOT;
          const float4* sk4 = reinterpret_cast<const float4*>(slot_at);
          const float4* lv4 = reinterpret_cast<const float4*>(slot_at + L::SLOT_LV);
          const float4* rv4 = reinterpret_cast<const float4*>(slot_at + L::SLOT_RV);
          const uint4* sums = reinterpret_cast<const uint4*>(slot_at + L::SLOT_SUM);
          const uint4 sum0 = sums[0], sum1 = sums[1];
          const int key0 = (kt0 + t) * KT;
          const bool masked = key0 + KT > plain_end || (sum0.x | sum0.y | sum1.x | sum1.y) != 0u;
          const float lv_top = fmaxf(__uint_as_float(sum0.z), __uint_as_float(sum1.z)), lv_low = fminf(__uint_as_float(sum0.w), __uint_as_float(sum1.w));
          uint32_t bits[2] = {0xffffffffu, 0xffffffffu};
          if (masked) {                              // a bit per key that this row sees
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
              const int k0 = key0 + 32 * ch, upto = lim - k0;
              uint32_t b = upto >= 32 ? 0xffffffffu : upto <= 0 ? 0u : (1u << upto) - 1u;
              b &= ~(ch ? sum1.x & ~sum1.y : sum0.x & ~sum0.y);
              if (tree_row != nullptr && b != 0u && k0 + 32 > ctx) {
                uint32_t hidden = 0u;                // (sixteen bytes in flight at a time)
#pragma unroll 1
                for (int i0 = 0; i0 < 32; i0 += 16)
#pragma unroll
                  for (int i = 0; i < 16; ++i) {
                    const int at = k0 + i0 + i - ctx;
                    const uint32_t seen = at >= 0 && (b >> (i0 + i) & 1u) ? __ldg(tree_row + at) : 1u;
                    hidden |= (seen == 0u ? 1u : 0u) << (i0 + i);
                  }
                b &= ~hidden;
              }
              bits[ch] = b;
              if (b & (ch ? sum1.x & sum1.y : sum0.x & sum0.y)) row_at[r] = __int_as_float(0x7fffffff);
            }
            __syncwarp();
          }
          tmem_ld_wait();
          if (masked) {
            // What this row does not see becomes -infinity before anything is made of it, what it sees of a key that holds
            // a NaN in K becomes one (such keys' scales stand at 1, so that they reach no other row).
            const uint32_t nan0 = sum0.y & ~sum0.x, nan1 = sum1.y & ~sum1.x;
#pragma unroll
            for (int i = 0; i < 64; ++i) {
              const uint32_t nan = i < 32 ? nan0 : nan1;
              x[i] = !(bits[i / 32] >> (i & 31) & 1u) ? 0xff800000u : (nan >> (i & 31) & 1u) ? 0x7fffffffu : x[i];
            }
          }
          // A bound of the row's largest e: the largest score, and the largest log2 of a scale of V; where those scales
          // differ by more than 2^8 within the tile, or some are not this row's to see, the largest e itself.
          float2* x2 = reinterpret_cast<float2*>(x);
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float4 sk = sk4[i];
            x2[2 * i] = __fmul2_rn(x2[2 * i], make_float2(sk.x, sk.y));
            x2[2 * i + 1] = __fmul2_rn(x2[2 * i + 1], make_float2(sk.z, sk.w));
            top = max3(max3(top, x2[2 * i].x, x2[2 * i].y), x2[2 * i + 1].x, x2[2 * i + 1].y);
          }
          top = fmaf(top, row_c, lv_top);
          if (masked || lv_top - lv_low > 8.f) {
            const float* lv = reinterpret_cast<const float*>(lv4);
            top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 64; ++i) top = fmaxf(top, fmaf(__uint_as_float(x[i]), row_c, lv[i]));
          }
          if (__any_sync(0xffffffffu, top > m + LIMIT_LOG2)) {
            // the maximum moves; the sum and the accumulator follow
            top = top > m + LIMIT_LOG2 ? top - TOP_LOG2 : m;           // (each row by itself)
            const float fade = ex2(m - top);
            m = top;
            l *= fade;
            l_carry *= fade;
            if (t > 0) {                             // (the unit's first product overwrites the accumulator)
              ok = __all_sync(0xffffffffu, mbar_wait(bar(L::B_PV + 2 * g + (buf ^ 1)), (uint32_t)((k - 1) >> 1) & 1u, watch, CODE_SOFTMAX));
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int ch = 0; ch < WIDTH / 16; ++ch) {
                uint32_t o[16];
                tmem_ld16(o_addr + 16 * ch, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fade);
                tmem_st16(o_addr + 16 * ch, o);
              }
            }
          }
          float2 l2 = make_float2(0.f, 0.f);
          const float2 nm2 = make_float2(-m, -m);
#pragma unroll
          for (int ch = 0; ch < 2; ++ch) {
            uint32_t pw[16];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int j = 8 * ch + i;
              const float4 lv = lv4[j], rv = rv4[j];
              const float2 u = __ffma2_rn(x2[2 * j], c2, __fadd2_rn(make_float2(lv.x, lv.y), nm2));
              const float2 v = __ffma2_rn(x2[2 * j + 1], c2, __fadd2_rn(make_float2(lv.z, lv.w), nm2));
              const float2 w = make_float2(ex2(u.x), ex2(u.y)), z = make_float2(ex2(v.x), ex2(v.y));
              l2 = __ffma2_rn(w, make_float2(rv.x, rv.y), l2);
              l2 = __ffma2_rn(z, make_float2(rv.z, rv.w), l2);
              pw[2 * i] = pack2<__half>(w.x, w.y);
              pw[2 * i + 1] = pack2<__half>(z.x, z.y);
            }
            tmem_st16(s_addr + 16 * ch, pw);         // over the scores, which are in registers
          }
          add_carrying(l, l_carry, l2.x + l2.y);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(L::B_PF + 2 * g + buf));
        }
        if (!ok) break;
        done += count;
        // ---- the rows of this stretch of the unit, through shared memory to whole rows
        ok = __all_sync(0xffffffffu, mbar_wait(bar(L::B_PV + 2 * g + ((done - 1) & 1)), (uint32_t)((done - 1) >> 1) & 1u, watch, CODE_SOFTMAX));
        if (!ok) break;
        tc_fence_after();
        const bool poisoned = isnan(row_at[r]);      // the row sees a NaN in V alone: its output is one, its sum is not
        // a unit that began before this stretch, or with it: its part is the stretch's first, else its last
        const long long part_row = (2LL * blockIdx.x + (cur.into > 0 ? 1 : 0)) * a.part_rows + 128 * g;
        if (whole) {
          const float inv = poisoned ? __int_as_float(0x7fffffff) : l == 0.f ? 0.f : __fdividef(1.f, l);
#pragma unroll 1
          for (int ch = 0; ch < WIDTH / 16; ++ch) {
            uint32_t o[16];
            tmem_ld16(o_addr + 16 * ch, o);
            tmem_ld_wait();
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = pack2<T>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
            *staged(r, 2 * ch) = make_uint4(h[0], h[1], h[2], h[3]);
            *staged(r, 2 * ch + 1) = make_uint4(h[4], h[5], h[6], h[7]);
          }
          __syncwarp();
          const int col = WIDTH == 128 ? 16 * (c_l & 7) + 8 * (c_l >> 3) : 8 * c_l;
#pragma unroll 4
          for (int i = 0; i < 32 / RPI; ++i) {
            const int row = row_l + i * RPI;
            if (row < live && col < a.D)
              *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + row_of(row, a.o_st, a.o_sh) + col) = *staged(row, c_l);
          }
        } else {
          // (the columns stay in the order of the accumulator: cache_combine_kernel puts them right)
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
#pragma unroll 1
            for (int ch = 0; ch < WIDTH / 32; ++ch) {
              uint32_t o[16];
              tmem_ld16(o_addr + half * (WIDTH / 2) + 16 * ch, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = poisoned ? 0x7fffffffu : o[i];
#pragma unroll
              for (int i = 0; i < 4; ++i) *staged(r, 4 * ch + i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
            __syncwarp();
#pragma unroll 4
            for (int i = 0; i < 32 / RPI; ++i) {
              const int row = row_l + i * RPI;
              if (row < live) *reinterpret_cast<uint4*>(a.part_o + (part_row + row) * WIDTH + half * (WIDTH / 2) + 4 * c_l) = *staged(row, c_l);
            }
            __syncwarp();
          }
          if (exists) a.part_ml[part_row + r] = make_float2(m, l);
        }
        tc_fence_before();
        if (exists && whole && a.lse != nullptr) {
          float v = l == 0.f ? -INFINITY : (m + __log2f(l)) * LN2_F;
          if (dots && l != 0.f) v += row_at[128 + r];                  // the keys as they were before the shift was taken off
          a.lse[(long long)(cur.s.q0 + tok) * a.Hq + cur.h * a.group + rr - tok * a.group] = v;
        }
        __syncwarp();                                // (the rows that passed through are read before the next Q is written)
      }
      n += count;
      next_unit(a, cur, cur.kt, ROWS, KT);
    }
  } else if (tid < L::SOFTMAX + L::LOADERS) {
    // ------------------------------------------------- loaders -------------------------------------------------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_LOADER));
    const int ct = tid - L::SOFTMAX;
    constexpr int PIECES = WIDTH / 16, RPI = 128 / PIECES, N_CHUNK = KT / RPI;        // rows of 128 threads; chunks per thread
    const int piece = ct % PIECES, row_l = ct / PIECES;
    Cursor ahead = cur;                              // the tile that is fetched next
    auto row_of = [&](int page, int key) -> long long {
      return (((long long)page * a.Hkv + ahead.h) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
    };
    // The scales of this thread's key of tile n: a scale of K below zero says that there is no such key.
    auto store_scales = [&](int n, float sk, float sv) {
      if (ct < KT) {
        const uint32_t sc = base + L::OFF_SC + (n % L::SLOTS) * L::SLOT;
        const bool none = sk < 0.f, nan_k = isnan(sk), nan_v = !nan_k && isnan(sv);
        // (0: a row that nothing wrote, all codes 0, a part of the sum; written ones are 1e-12 at least.  The sum takes weights of
        // up to 2^LIMIT_LOG2 over this: 2^30 keys of them stay below fp32's largest.)
        const float v = none || nan_k || nan_v ? 1.f : fmaxf(sv, 1e-20f);
        sts_f32(sc + 4 * ct, none || nan_k ? 1.f : fmaxf(sk, 1e-30f));
        sts_f32(sc + L::SLOT_LV + 4 * ct, __log2f(v));
        sts_f32(sc + L::SLOT_RV + 4 * ct, __fdividef(1.f, v));
        const uint32_t first32 = __ballot_sync(0xffffffffu, none || nan_v), second32 = __ballot_sync(0xffffffffu, nan_k || nan_v);
        // (positive floats are ordered as their bits are)
        const float big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))), small = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(v)));
        if (lane == 0) sts16(sc + L::SLOT_SUM + 16 * (ct >> 5), first32, second32, __float_as_uint(__log2f(big)), __float_as_uint(__log2f(small)));
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::B_SC + n % L::SLOTS));
      }
    };
    // This thread's pieces of a tile, turned into fp16, to the operand at `stage`.
    auto store_codes = [&](const uint4 (&codes)[N_CHUNK], uint32_t stage, bool as_int8) {
#pragma unroll
      for (int i = 0; i < N_CHUNK; ++i) {
        const int row = i * RPI + row_l;
        uint32_t h[8];
        if (as_int8) codes_to_half<true>(codes[i], h); else codes_to_half<false>(codes[i], h);
        const uint32_t to = stage + row * 128;
        if (WIDTH == 128) {
          const uint32_t at = to + 16 * (piece ^ (row & 7));
          sts16(at, h[0], h[1], h[2], h[3]);
          sts16(at + L::KV_HALF, h[4], h[5], h[6], h[7]);
        } else {
          sts16(to + 16 * ((2 * piece) ^ (row & 7)), h[0], h[1], h[2], h[3]);
          sts16(to + 16 * ((2 * piece + 1) ^ (row & 7)), h[4], h[5], h[6], h[7]);
        }
      }
      fence_async_smem();
      __syncwarp();
    };
    auto stage_free = [&](int b, int n) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar(b + n % L::STAGES), ((uint32_t)(n / L::STAGES) & 1u) ^ 1u, watch, CODE_LOAD));
    };
    if constexpr (L::RAW_STAGES > 0) {
      // Page ids: every warp keeps 32 of the sequence's, one per lane, and the 32 behind them, asked for long before
      // they are needed.
      int window = -1, window_next = -1, window_first = 0, window_b = -1;
      auto ids_from = [&](int first) -> int {
        return first + lane < a.table_width ? __ldg(a.table + ahead.b * a.table_st + first + lane) : -1;
      };
      auto find_window = [&]() {
        const int first = (ahead.kt * KT) >> a.page_shift;                              // (a tile's pages never lie in two windows)
        if (ahead.b == window_b && first >= window_first && first < window_first + 32) return;
        if (ahead.b == window_b && first == window_first + 32) {
          window = window_next;
          window_first += 32;
        } else {
          window_b = ahead.b;
          window_first = first & ~31;
          window = ids_from(window_first);
        }
        window_next = ids_from(window_first + 32);
      };
      // The next tile's codes and scales into the ring: this thread's 16-byte pieces of K, of V, and the scales of key ct.
      const uint32_t raw = base + L::OFF_RAW + 16 * ct, raw_scales = base + L::OFF_RAW + 2 * KT * WIDTH + 4 * ct;
      int issued = 0;
      auto issue_next = [&]() {
        if (ahead.left > 0) {
          find_window();
          const uint32_t slot = (uint32_t)(issued % L::RAW_STAGES) * L::RAW_TILE;
          auto place_of = [&](int row, bool& there) -> long long {
            const int key = ahead.kt * KT + row, block = key & ~15;
            const int page = __shfl_sync(0xffffffffu, window, ((block >> a.page_shift) - window_first) & 31);
            there = block < ahead.s.len && (unsigned)page < (unsigned)a.pages;
            return there ? row_of(page, key) : 0;
          };
          bool there;
#pragma unroll
          for (int i = 0; i < N_CHUNK; ++i) {
            const long long at = place_of(i * RPI + row_l, there) * WIDTH + 16 * piece;
            copy16(raw + slot + i * 2048, a.kc + at, there);
            copy16(raw + slot + (N_CHUNK + i) * 2048, a.vc + at, there);
          }
          const long long at = place_of(ct & (KT - 1), there);
          if (ct < KT) {
            if (there) {
              copy4(raw_scales + slot, a.ks + at);
              copy4(raw_scales + slot + KT * 4, a.vs + at);
            } else {                                   // no such key: a scale below zero says so
              sts_f32(raw_scales + slot, -1.f);
              sts_f32(raw_scales + slot + KT * 4, 0.f);
            }
          }
          ++issued;
          next_step(a, ahead, ROWS, KT);
        }
        copy_commit();
      };
      auto convert = [&](uint32_t from, uint32_t stage, bool as_int8) {
        uint4 codes[N_CHUNK];
#pragma unroll
        for (int i = 0; i < N_CHUNK; ++i) codes[i] = lds16(from + i * 2048);
        store_codes(codes, stage, as_int8);
      };
#pragma unroll 1
      for (int i = 0; i < L::RAW_STAGES; ++i) issue_next();
      for (int n = 0; n < issued; ++n) {
        const int st = n % L::STAGES;
        const uint32_t slot = (uint32_t)(n % L::RAW_STAGES) * L::RAW_TILE;
        copy_wait<L::RAW_STAGES - 1>();
        if (!stage_free(L::B_KE, n)) break;
        if (ct < KT) store_scales(n, lds_f32(raw_scales + slot), lds_f32(raw_scales + slot + KT * 4));
        convert(raw + slot, base + L::OFF_K + st * L::KV_TILE, INT8);
        if (lane == 0) mbar_arrive(bar(L::B_KF + st));
        if (!stage_free(L::B_VE, n)) break;
        convert(raw + slot + N_CHUNK * 2048, base + L::OFF_V + st * L::KV_TILE, false);
        if (lane == 0) mbar_arrive(bar(L::B_VF + st));
        issue_next();
      }
      copy_wait<0>();                                // (a wait that gave up leaves none of its own copies in flight)
    } else {
      // of tile `ahead`: the page of each chunk's row, and of the key whose scales this thread fetches
      int pages[N_CHUNK], s_page = -1;
      auto page_of = [&](int key) -> int { return key < ahead.s.len ? __ldg(a.table + ahead.b * a.table_st + (key >> a.page_shift)) : -1; };
      auto fetch_pages = [&]() {
#pragma unroll
        for (int i = 0; i < N_CHUNK; ++i) pages[i] = page_of(ahead.kt * KT + ((i * RPI + row_l) & ~15));
        if (ct < KT) s_page = page_of(ahead.kt * KT + (ct & ~15));
      };
      uint4 kr[N_CHUNK], vr[N_CHUNK];
      float sk = 0.f, sv = 0.f;
      auto fetch = [&](const uint8_t* codes, uint4 (&to)[N_CHUNK]) {
#pragma unroll
        for (int i = 0; i < N_CHUNK; ++i) {
          to[i] = make_uint4(0u, 0u, 0u, 0u);
          if ((unsigned)pages[i] < (unsigned)a.pages)
            to[i] = __ldcs(reinterpret_cast<const uint4*>(codes + row_of(pages[i], ahead.kt * KT + i * RPI + row_l) * WIDTH + 16 * piece));
        }
      };
      auto fetch_scales = [&]() {
        if (ct < KT) {
          const bool there = (unsigned)s_page < (unsigned)a.pages;
          const long long at = there ? row_of(s_page, ahead.kt * KT + ct) : 0;
          sk = there ? __ldg(a.ks + at) : -1.f;
          sv = there ? __ldg(a.vs + at) : 0.f;
        }
      };
      auto advance = [&]() {                         // on to the next tile, whose pages are asked for at once
        next_step(a, ahead, ROWS, KT);
        if (ahead.left > 0) fetch_pages();
      };
      fetch_pages();
      fetch(a.kc, kr);
      fetch_scales();
      fetch(a.vc, vr);
      advance();
      bool more = true;
      for (int n = 0; more; ++n) {
        const int st = n % L::STAGES;
        more = ahead.left > 0;                       // `ahead` is tile n + 1
        if (!stage_free(L::B_KE, n)) break;
        store_scales(n, sk, sv);
        store_codes(kr, base + L::OFF_K + st * L::KV_TILE, INT8);
        if (lane == 0) mbar_arrive(bar(L::B_KF + st));
        if (more) {
          fetch(a.kc, kr);
          fetch_scales();
        }
        if (!stage_free(L::B_VE, n)) break;
        store_codes(vr, base + L::OFF_V + st * L::KV_TILE, false);
        if (lane == 0) mbar_arrive(bar(L::B_VF + st));
        if (more) {
          fetch(a.vc, vr);
          advance();
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_ISSUER));
    const int g = warp - ISSUER;
    if (g < NQ && lane == 0) {
      // ------------------------------------------------- products ------------------------------------------------------
      bool ok = true;
      int n = 0, k = 0, segments = 0;                                 // k: tiles of this half so far
      // scores of tile n into buffer `to`
      auto issue_qk = [&](int to) -> bool {
        const int st = n % L::STAGES;
        if (!mbar_wait(bar(L::B_KF + st), (uint32_t)(n / L::STAGES) & 1u, watch, CODE_MMA)) return false;
        tc_fence_after();
        const uint32_t q_at = desc_k(base + L::OFF_Q + g * L::Q_TILE), k_at = desc_k(base + L::OFF_K + st * L::KV_TILE);
#pragma unroll
        for (int i = 0; i < WIDTH / 16; ++i)
          mma_ss(tmem_s(g, to), q_at + (((i >> 2) * L::Q_HALF + 32 * (i & 3)) >> 4), k_at + (((i >> 2) * L::KV_HALF + 32 * (i & 3)) >> 4), IDESC_QK, i > 0);
        tc_commit(bar(L::B_SF + 2 * g + to));
        tc_commit(bar(L::B_KE + st));
        ++n;
        return true;
      };
      while (ok && cur.left > 0) {
        const int count = min(cur.left, cur.n_kt - cur.kt), n0 = n;
        if (g < halves_of(cur)) {
          ok = mbar_wait(bar(L::B_QF + g), (uint32_t)segments & 1u, watch, CODE_MMA);
          ++segments;
          ok = ok && issue_qk(k & 1);
          for (int t = 0; ok && t < count; ++t, ++k) {
            // (the buffer of the tile before: its P V is ahead of these products in this thread's order)
            if (t + 1 < count && !issue_qk((k + 1) & 1)) { ok = false; break; }
            const int st = (n0 + t) % L::STAGES;
            ok = mbar_wait(bar(L::B_VF + st), (uint32_t)((n0 + t) / L::STAGES) & 1u, watch, CODE_MMA) &&
                 mbar_wait(bar(L::B_PF + 2 * g + (k & 1)), (uint32_t)(k >> 1) & 1u, watch, CODE_MMA);
            if (!ok) break;
            tc_fence_after();
            const uint32_t v_at = desc_mn(base + L::OFF_V + st * L::KV_TILE, L::KV_HALF);
#pragma unroll
            for (int i = 0; i < KT / 16; ++i)
              mma_ts(tmem_o(g), tmem_s(g, k & 1) + 8 * i, v_at + (2048 * i >> 4), IDESC_PV, t > 0 || i > 0);
            tc_commit(bar(L::B_PV + 2 * g + (k & 1)));
            tc_commit(bar(L::B_VE + st));
          }
        } else {                                     // no rows here: the stages are free as far as this half goes
          for (int t = 0; ok && t < count; ++t, ++n) {
            const int st = n % L::STAGES;
            ok = mbar_wait(bar(L::B_KF + st), (uint32_t)(n / L::STAGES) & 1u, watch, CODE_MMA);
            if (ok) mbar_arrive(bar(L::B_KE + st));
            ok = ok && mbar_wait(bar(L::B_VF + st), (uint32_t)(n / L::STAGES) & 1u, watch, CODE_MMA);
            if (ok) mbar_arrive(bar(L::B_VE + st));
          }
        }
        next_unit(a, cur, cur.kt, ROWS, KT);
      }
      tc_commit(bar(L::B_DRAIN));                    // every product issued is complete before the TMEM is freed
      drain_wait(bar(L::B_DRAIN), watch, CODE_MMA);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == ISSUER) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM_COLS) : "memory");
  }
}

template <typename T, bool INT8, int WIDTH, int NQ>
cudaError_t launch_tree(CacheAttnKArgs& a, int sms, int32_t* status_host, cudaStream_t st) {
  using L = TreeShape<WIDTH, NQ>;
  auto kern = cache_tree_kernel<T, INT8, WIDTH, NQ>;
  static DeviceOnce once;
  cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::BYTES); });
  if (e != cudaSuccess) return e;
  const long long rows = (long long)a.max_q * a.group, rts = (rows + L::ROWS - 1) / L::ROWS;
  const long long steps = (long long)a.n_seq * a.Hkv * rts * (UNIT_STEPS + std::max<long long>(1, (((long long)a.table_width << a.page_shift) + KT - 1) / KT));
  a.max_stretches = std::min(std::min(sms, 160) * L::CTAS_PER_SM, cache_form(rows).max_stretches);
  kern<<<(unsigned)std::min<long long>(a.max_stretches, steps), L::THREADS, L::BYTES, st>>>(a, status_host);
  return cudaGetLastError();
}

template <typename T, bool INT8, int WIDTH>
cudaError_t launch_tree_rows(CacheAttnKArgs& a, int sms, int32_t* status_host, cudaStream_t st) {
  return cache_form((int64_t)a.max_q * a.group).rows == 128 ? launch_tree<T, INT8, WIDTH, 1>(a, sms, status_host, st)
                                                            : launch_tree<T, INT8, WIDTH, 2>(a, sms, status_host, st);
}
template <typename T>
cudaError_t launch_tree_type(CacheAttnKArgs& a, const CacheView& c, int sms, int32_t* status_host, cudaStream_t st) {
  if (c.width == 64) return c.int8 ? launch_tree_rows<T, true, 64>(a, sms, status_host, st) : launch_tree_rows<T, false, 64>(a, sms, status_host, st);
  return c.int8 ? launch_tree_rows<T, true, 128>(a, sms, status_host, st) : launch_tree_rows<T, false, 128>(a, sms, status_host, st);
}

}  // namespace

cudaError_t launch_cache_tree(CacheAttnKArgs& a, const CacheView& c, int dtype, int sms, int32_t* status_host, cudaStream_t st) {
  return dtype == 0 ? launch_tree_type<__half>(a, c, sms, status_host, st) : launch_tree_type<__nv_bfloat16>(a, c, sms, status_host, st);
}

}  // namespace sage
