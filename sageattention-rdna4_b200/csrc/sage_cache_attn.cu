// Attention of new tokens over a quantised, paged K/V cache (layout: sage_cache.cu): one token per
// sequence, a chain of them (each sees the keys up to its own), or a tree of drafted tokens (a mask says
// which of them each sees).
//
// Rows.  The Hq / Hkv query heads of a K/V head share its keys, so the rows of a unit are the pairs
// (new token, query head of the group), token by token; up to 8 * NB rows make a row tile.
//
// Products.  The cache is read in its one-byte codes and the 16-bit products take them exactly: int8 and
// e4m3 codes are both fp16 numbers.  Scores are transposed, S^T = K Q^T, and so is the output, O^T = V^T P^T:
// the 16-row operand of mma.m16n8k16 is then 16 keys (or 16 columns of V), and the 8-column one is 8 query
// rows, so that a single query row wastes 7 of 8 columns and not 15 of 16 rows.  The inner dimension of a
// product may be walked in any order, if both operands walk it alike:
//   S^T   lane (g = lane / 4, c = lane % 4) reads the 32 bytes c of key rows g and g + 8; its k-step s is
//         bytes 4s .. 4s+3 of them, and Q is laid out to match
//   O^T   lane (g, c) reads the 16 bytes g of the keys 2c, 2c+1, 2c+8, 2c+9 and pairs the bytes of two keys;
//         its rows of step j are the columns 16g + 2j and 16g + 2j + 1 of V
// so that every shared-memory read is 16 bytes wide and no code is moved between lanes.  16-byte pieces of a
// row are stored at piece ^ (row & 7), which spreads both reads over all banks.
//
// Numerics.  Q in fp16: bf16 rows are scaled by a power of two each, which is undone in the score's factor, so
// that no bit is lost but in elements 2^-28 below their row's largest.  Scores, maxima, sums and outputs in
// fp32.  A weight enters the second product as fp16(p * v_scale * N), where N is a factor per row that puts the
// largest one seen between 2^4 and 2^15 (fp16 has 11 bits there; its relative error, 2^-11, is that of the output format).
// The running maximum moves only when a score passes it by 2^15, and N when a weight does: the accumulator is
// rarely touched.  Weights keep 11 bits down to 2^-18 of the row's largest, 2^-29 of it is what each may lose, and the fp32
// accumulator loses up to 2^-23 of its sum with every 16 keys: what bounds a row of very many keys (2^20: 2^-7 at worst, where
// all errors have one sign).
//
// Work.  The steps of 32 keys of all (sequence, K/V head, row tile) units are numbered in one line, and every
// warp of the GPU takes an equal stretch of it, by itself: its own ring of cp.async stages, no barrier, no spinning
// wait.  So ragged batches and single long sequences alike fill the GPU; lengths are read on the device.  A unit
// that lies in several stretches leaves partial rows in the workspace, which cache_combine_kernel joins in the
// order of the keys.
//
// What bounds it.  The cache's bytes: 4 x 47 520 keys x 48 heads, 357 to 371 us in a graph = 6.5 to 6.7 TB/s, the rate of a
// plain copy (called one by one with other inputs each time, 372 to 410 from GPU to GPU).  32 ragged sequences of up to 8192
// keys x 8 heads: 43 us = 4.5 TB/s; joining the parts, the launches and the two to three units that a warp begins take the
// difference.  One sequence of 16 384 keys: 15.5 us, of which 6 are the cache's bytes and the rest the chain launch, lengths,
// pages, codes, parts, join.  16 rows instead of 8 cost instructions (codes are unpacked once for all rows of a tile): 8 x
// 16 384 keys x 8 heads 54 us with 8 rows, 63 with 16.
#include "sage_cache_attn.cuh"

namespace sage {

namespace {

constexpr int CA_WARPS = 4, CA_THREADS = 32 * CA_WARPS;
constexpr int CA_KEYS = 32;                    // keys of a step: two blocks of 16
constexpr float LIMIT = (float)(1 << LIMIT_LOG2);

__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Shared memory of a CTA: a ring per warp.
template <int WIDTH, int STAGES> struct CaSmem {
  static constexpr uint32_t CODES = CA_KEYS * WIDTH;
  static constexpr uint32_t STAGE = 2 * CODES + 2 * CA_KEYS * 4;     // K, V, and the scales of each
  static constexpr uint32_t BYTES = CA_WARPS * STAGES * STAGE;
};

// NB: blocks of 8 query rows in a row tile.
template <typename T, bool INT8, int WIDTH, int NB, int STAGES, int CTAS_PER_SM>
__global__ void __launch_bounds__(CA_THREADS, CTAS_PER_SM) cache_attn_kernel(const CacheAttnKArgs a) {
  using L = CaSmem<WIDTH, STAGES>;
  constexpr int ROWS = 8 * NB, KSTEPS = WIDTH / 16, PIECES = WIDTH / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ PlaceScratch<CA_THREADS, CA_WARPS> place_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const unsigned stretch = blockIdx.x * CA_WARPS + warp;
  allow_successor();
  Cursor cur;
  unsigned before;
  const Line line = find_place(a, ROWS, CA_KEYS, place_s, warp, cur.b, before);
  if (cur.b >= a.n_seq) return;
  enter_line(a, cur, line.begin(stretch), line.begin(stretch + 1), before, ROWS, CA_KEYS);
  if (cur.left <= 0) return;
  Cursor ahead = cur;                                // the step whose loads are issued next
  const uint32_t ring = smem_u32(smem) + warp * STAGES * L::STAGE;

  // The 32 keys of the step at `ahead` into stage s.  Lane l copies piece l % PIECES of rows l / PIECES + i * RPI;
  // (row & 7) of the swizzle is that of the lane's first row, but for a change of one bit in every other copy.
  constexpr int RPI = 32 / PIECES;                   // rows of one copy instruction
  const int row_l = lane / PIECES, piece_l = lane % PIECES;
  const uint32_t dst_even = row_l * WIDTH + 16 * (WIDTH == 128 ? piece_l ^ row_l : piece_l ^ (row_l >> 1));
  const uint8_t *k_lane = a.kc + 16 * lane, *v_lane = a.vc + 16 * lane;
  const float* s_lane = ((lane & 7) < 4 ? a.ks : a.vs) + 4 * (lane & 3);
  int pages[2];                                      // of the step at `ahead`, fetched a step early
  auto fetch_pages = [&]() {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const int key0 = ahead.kt * CA_KEYS + 16 * blk;
      pages[blk] = key0 < ahead.s.len ? __ldg(a.table + ahead.b * a.table_st + (key0 >> a.page_shift)) : -1;
    }
  };
  auto issue = [&](int s) {
    const uint32_t st = ring + s * L::STAGE;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {              // 16 keys of one page
      const int key0 = ahead.kt * CA_KEYS + 16 * blk, page = pages[blk];
      const bool there = (unsigned)page < (unsigned)a.pages;
      const long long row = there ? ((((long long)page * a.Hkv + ahead.h) << a.page_shift) + (key0 & ((1 << a.page_shift) - 1))) : 0;
      const uint8_t *k = k_lane + row * WIDTH, *v = v_lane + row * WIDTH;
      const uint32_t dst = st + blk * 16 * WIDTH;
#pragma unroll
      for (int i = 0; i < 16 / RPI; ++i) {
        const uint32_t to = dst + i * RPI * WIDTH + (WIDTH == 128 ? dst_even ^ (64u * (i & 1)) : dst_even);
        copy16(to, k + i * RPI * WIDTH, there);
        copy16(to + L::CODES, v + i * RPI * WIDTH, there);
      }
      // scales: 32 of K, then 32 of V
      if (there) {
        if (lane < 8) copy16(st + 2 * L::CODES + (lane < 4 ? 0 : 128) + 64 * blk + 16 * (lane & 3), s_lane + row, true);
      } else if (lane < 16) {                        // no such keys: a scale below zero says so
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(st + 2 * L::CODES + 64 * blk + 4 * lane), "f"(-1.0f) : "memory");
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(st + 2 * L::CODES + 128 + 64 * blk + 4 * lane), "f"(0.0f) : "memory");
      }
    }
  };
  // Rows of Q of the unit at `cur`: lane (g, c) fetches columns c * WIDTH / 4 .. of rows 8 nb + g.
  uint4 q_raw[NB][WIDTH / 32];
  auto fetch_q = [&]() {
    const int live = cur.s.q_len * a.group - cur.rt * ROWS;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = 8 * nb + g, rr = cur.rt * ROWS + r, tok = rr / a.group, head = cur.h * a.group + rr - tok * a.group;
      const T* src = reinterpret_cast<const T*>(a.q) + (long long)(cur.s.q0 + tok) * a.q_st + (long long)head * a.q_sh;
#pragma unroll
      for (int i = 0; i < WIDTH / 32; ++i) {
        const int col = c * (WIDTH / 4) + 8 * i;
        q_raw[nb][i] = r < live && col < a.D ? __ldg(reinterpret_cast<const uint4*>(src + col)) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  fetch_pages();
  fetch_q();
  // the step at `ahead` into stage s, and on to the next one
  auto issue_next = [&](int s) {
    if (ahead.left > 0) {
      issue(s);
      next_step(a, ahead, ROWS, CA_KEYS);
      if (ahead.left > 0) fetch_pages();
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue_next(s);

  uint32_t qf[NB][KSTEPS][2];                        // Q^T: k-step s of query row 8 nb + g
  float row_c[NB][2];                                // score factor of rows 8 nb + 2c + {0, 1}
  int row_lim[NB][2], row_tok[NB][2];                // keys that a row may see; its token within the sequence
  float m[NB][2], l[NB][2], lc[NB][2], nf[NB][2];    // running maximum, this lane's sum and what its rounding carries, factor N
  float o[NB][KSTEPS][4];                            // O^T: columns 16g + 2j + {0, 1} of rows 8 nb + 2c + {0, 1}
  int plain_end = 0;                                 // keys below this need no mask

  int stage = 0;
  bool fresh = true;
  for (;;) {
    // the stage that was read last is free: fetch into it
    __syncwarp();
    issue_next(stage == 0 ? STAGES - 1 : stage - 1);
    if (fresh) {
      fresh = false;
      const int live = min(ROWS, cur.s.q_len * a.group - cur.rt * ROWS);      // rows of this tile that exist
      const int ctx = cur.s.len - cur.s.q_len;
      const int t_first = cur.rt * ROWS / a.group;
      plain_end = a.tree ? max(ctx, 0) : max(0, min(cur.s.len, ctx + t_first + 1));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float x[WIDTH / 4], amax = 0.f;
#pragma unroll
        for (int i = 0; i < WIDTH / 32; ++i) unpack8<T>(q_raw[nb][i], x + 8 * i);
        float back = 1.f;                            // what undoes the row's power of two
        if (sizeof(T) == 2 && !__is_same(T, __half)) {
#pragma unroll
          for (int i = 0; i < WIDTH / 4; ++i) amax = fmaxf(amax, fabsf(x[i]));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          // amax -> [2^14, 2^15): the exponent field of 2^(14 - e) is 127 + 14 - e = 268 - field(amax)
          const int field = (int)(__float_as_uint(amax) >> 23);
          if (field > 14 && field < 255) {
            const int f = min(254, 268 - field);
            const float up = __uint_as_float((uint32_t)f << 23);
#pragma unroll
            for (int i = 0; i < WIDTH / 4; ++i) x[i] *= up;
            back = f <= 253 ? __uint_as_float((uint32_t)(254 - f) << 23) : 5.877471754111438e-39f;
          }
        }
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
          qf[nb][s][0] = inf_to_nan(pack2<__half>(x[4 * s], x[4 * s + 1]));
          qf[nb][s][1] = inf_to_nan(pack2<__half>(x[4 * s + 2], x[4 * s + 3]));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // rows 2c + e sit with lane g' = 2c + e of the Q fragments
          row_c[nb][e] = fmaxf(a.scale_log2 * __shfl_sync(0xffffffffu, back, 4 * (2 * c + e)), 1.17549435e-38f);   // (a masked score stays -infinity)
          const int r2 = 8 * nb + 2 * c + e, tok2 = (cur.rt * ROWS + r2) / a.group;
          row_tok[nb][e] = tok2;
          row_lim[nb][e] = r2 < live ? (a.tree ? cur.s.len : min(cur.s.len, ctx + tok2 + 1)) : 0;
          m[nb][e] = NO_MAX; l[nb][e] = 0.f; lc[nb][e] = 0.f; nf[nb][e] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nb][j][e] = 0.f;
      }
    }

    copy_wait<STAGES - 1>();
    __syncwarp();

    const uint32_t st = ring + stage * L::STAGE, scales = st + 2 * L::CODES + 4 * g;
    const int key0 = cur.kt * CA_KEYS;
    // ---- S^T = K Q^T, two blocks of 16 keys
    float s[2][NB][4];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[blk][nb][e] = 0.f;
#pragma unroll
      for (int half = 0; half < WIDTH / 64; ++half) {
        // 16 bytes of rows g and g + 8: four k-steps
        const int p = WIDTH == 128 ? (2 * c + half) ^ (g & 7) : c ^ ((g >> 1) & 3);
        const uint4 u = lds16(st + (16 * blk + g) * WIDTH + 16 * p), v = lds16(st + (16 * blk + g + 8) * WIDTH + 16 * p);
        const uint32_t r0[4] = {u.x, u.y, u.z, u.w}, r1[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t f[4];
          k_halves<INT8>(r0[i], f[0], f[2]);
          k_halves<INT8>(r1[i], f[1], f[3]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma16816(s[blk][nb], f, qf[nb][4 * half + i][0], qf[nb][4 * half + i][1]);
        }
      }
    }
    // ---- weights: key blk * 16 + g + 8 * (e / 2), row 2c + e % 2
    float sk[2][2], sv[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) { sk[i >> 1][i & 1] = lds_f32(scales + 32 * i); sv[i >> 1][i & 1] = lds_f32(scales + 128 + 32 * i); }
    const bool absent = fminf(fminf(sk[0][0], sk[0][1]), fminf(sk[1][0], sk[1][1])) < 0.f;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[blk][nb][e] *= sk[blk][e >> 1];
    const bool masked = key0 + 32 > plain_end || __any_sync(0xffffffffu, absent);
    if (masked) {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 16 * blk + g + 8 * (e >> 1), x = e & 1;
            bool seen = key < row_lim[nb][x] && !(sk[blk][e >> 1] < 0.f);
            if (a.tree != nullptr && seen) {
              const int j = key - (cur.s.len - cur.s.q_len);
              if (j >= 0) seen = a.tree[(long long)(cur.s.q0 + row_tok[nb][x]) * a.tree_st + j] != 0;
            }
            if (!seen) s[blk][nb][e] = -INFINITY;
          }
    }
    uint32_t pf[2][NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float p[2][4], w[2][4];
      float p_top = 0.f, w_top = 0.f;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[blk][e] = ex2(fmaf(s[blk][nb][e], row_c[nb][e & 1], -m[nb][e & 1]));
          w[blk][e] = p[blk][e] * (sv[blk][e >> 1] * nf[nb][e & 1]);
          p_top = fmaxf(p_top, p[blk][e]);
          w_top = fmaxf(w_top, w[blk][e]);
        }
      if (__any_sync(0xffffffffu, fmaxf(p_top, w_top) > LIMIT)) {
        // new maxima and factors; the sums and the accumulator follow
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float top = m[nb][x];
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, s[i >> 1][nb][2 * (i & 1) + x] * row_c[nb][x]);
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, sh));
          // (each row by itself: what another row sees moves nothing here)
          float big = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (s[i >> 1][nb][2 * (i & 1) + x] != -INFINITY) big = fmaxf(big, w[i >> 1][2 * (i & 1) + x]);
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, sh));
          if (!(top > m[nb][x] + LIMIT_LOG2 || big > LIMIT)) top = m[nb][x];
          const bool move = top != m[nb][x] || big > LIMIT;
          const float fade = ex2(m[nb][x] - top);
          big = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = ex2(fmaf(s[i >> 1][nb][2 * (i & 1) + x], row_c[nb][x], -top));
            p[i >> 1][2 * (i & 1) + x] = v;
            if (s[i >> 1][nb][2 * (i & 1) + x] != -INFINITY) big = fmaxf(big, v * sv[i >> 1][i & 1]);
          }
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, sh));
          // N for the largest weight of this step, or what leaves the accumulator as it is where that holds larger ones
          // (nothing but values of 0 here, or fade 0: infinite, the other one counts; both: there is nothing to scale)
          float n_new = nf[nb][x], scale = fade;
          const float n_least = fminf(__fdividef((float)(1 << TOP_LOG2), big), n_new > 0.f ? __fdividef(n_new, fade) : INFINITY);
          if (move && n_least < INFINITY) {
            if (n_new > 0.f) scale = fade * __fdividef(n_least, n_new);
            n_new = n_least;
          }
          m[nb][x] = top;
          nf[nb][x] = n_new;
          l[nb][x] *= fade;
          lc[nb][x] *= fade;
#pragma unroll
          for (int j = 0; j < KSTEPS; ++j) { o[nb][j][x] *= scale; o[nb][j][2 + x] *= scale; }
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i >> 1][2 * (i & 1) + x] = p[i >> 1][2 * (i & 1) + x] * (sv[i >> 1][i & 1] * n_new);
        }
      }
      if (masked) {                                  // a masked weight is an exact zero whatever its key's scale holds
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (s[i >> 2][nb][i & 3] == -INFINITY) w[i >> 2][i & 3] = 0.f;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) add_carrying(l[nb][x], lc[nb][x], (p[0][x] + p[0][2 + x]) + (p[1][x] + p[1][2 + x]));
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const __half2 u = __floats2half2_rn(w[blk][0], w[blk][1]), v = __floats2half2_rn(w[blk][2], w[blk][3]);
        pf[blk][nb][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&u));
        pf[blk][nb][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&v));
      }
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const uint32_t vt = st + L::CODES + 16 * blk * WIDTH;
      uint32_t x[4][WIDTH / 32];                     // keys 2c, 2c+1, 2c+8, 2c+9: this lane's WIDTH / 8 columns
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 2 * c + (i & 1) + 8 * (i >> 1);
        if (WIDTH == 128) {
          const uint4 u = lds16(vt + r * WIDTH + 16 * (g ^ (r & 7)));
          x[i][0] = u.x; x[i][1] = u.y; x[i][WIDTH / 32 - 2] = u.z; x[i][WIDTH / 32 - 1] = u.w;
        } else {
          const uint2 u = lds8(vt + r * WIDTH + 16 * ((g >> 1) ^ ((r >> 1) & 3)) + 8 * (g & 1));
          x[i][0] = u.x; x[i][1] = u.y;
        }
      }
#pragma unroll
      for (int i = 0; i < WIDTH / 32; ++i) {
        // bytes 4i .. 4i+3: columns paired over two keys
        const uint32_t a01 = __byte_perm(x[0][i], x[1][i], 0x5140), a23 = __byte_perm(x[0][i], x[1][i], 0x7362);
        const uint32_t b01 = __byte_perm(x[2][i], x[3][i], 0x5140), b23 = __byte_perm(x[2][i], x[3][i], 0x7362);
        uint32_t f[4], h[4];
        e4m3_quad(a01, f[0], f[1]);
        e4m3_quad(b01, f[2], f[3]);
        e4m3_quad(a23, h[0], h[1]);
        e4m3_quad(b23, h[2], h[3]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          mma16816(o[nb][2 * i], f, pf[blk][nb][0], pf[blk][nb][1]);
          mma16816(o[nb][2 * i + 1], h, pf[blk][nb][0], pf[blk][nb][1]);
        }
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;

    // ---- end of the unit, or of the stretch
    const bool last_of_unit = cur.kt + 1 == cur.n_kt;
    if (last_of_unit || cur.left == 1) {
      const bool whole = last_of_unit && cur.into >= 0;                // all of the unit's steps were here
      // a unit that began before this stretch, or with it: its part is the stretch's first, else its last
      const long long slot = 2LL * stretch + (cur.into > 0 ? 1 : 0);
      const int live = min(ROWS, cur.s.q_len * a.group - cur.rt * ROWS);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float sum = l[nb][x];
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, sh);
          const int r = 8 * nb + 2 * c + x;
          const float inv_n = nf[nb][x] > 0.f ? __fdividef(1.f, nf[nb][x]) : 0.f;
          if (r < live) {
            if (whole) {
              const int tok = row_tok[nb][x], head = cur.h * a.group + cur.rt * ROWS + r - tok * a.group;
              const float inv = sum == 0.f ? 0.f : __fdividef(inv_n, sum);
              T* dst = reinterpret_cast<T*>(a.out) + (long long)(cur.s.q0 + tok) * a.o_st + (long long)head * a.o_sh + (WIDTH / 8) * g;
#pragma unroll
              for (int j = 0; j < KSTEPS; ++j)
                if ((WIDTH / 8) * g + 2 * j < a.D) *reinterpret_cast<uint32_t*>(dst + 2 * j) = pack2<T>(o[nb][j][x] * inv, o[nb][j][2 + x] * inv);
              if (a.lse != nullptr && g == 0) a.lse[(long long)(cur.s.q0 + tok) * a.Hq + head] = sum == 0.f ? -INFINITY : (m[nb][x] + __log2f(sum)) * LN2_F;
            } else {
              float* dst = a.part_o + (slot * a.part_rows + r) * WIDTH + (WIDTH / 8) * g;
#pragma unroll
              for (int j = 0; j < KSTEPS; j += 2)
                *reinterpret_cast<float4*>(dst + 2 * j) = make_float4(o[nb][j][x] * inv_n, o[nb][j][2 + x] * inv_n, o[nb][j + 1][x] * inv_n, o[nb][j + 1][2 + x] * inv_n);
              if (g == 0) a.part_ml[slot * a.part_rows + r] = make_float2(m[nb][x], sum);
            }
          }
        }
      if (whole && a.lse != nullptr && a.shift != nullptr) {           // the keys as they were before the shift was taken off
        __syncwarp();
        for (int r = 0; r < live; ++r) {
          const int rr = cur.rt * ROWS + r, tok = rr / a.group, head = cur.h * a.group + rr - tok * a.group;
          const float d = shift_dot(a, reinterpret_cast<const T*>(a.q) + (long long)(cur.s.q0 + tok) * a.q_st + (long long)head * a.q_sh, cur.h, WIDTH, lane);
          float* at = a.lse + (long long)(cur.s.q0 + tok) * a.Hq + head;
          if (lane == 0 && *at != -INFINITY) *at += d;                  // (a row that sees no key stays, whatever its Q holds)
        }
        __syncwarp();
      }
      next_step(a, cur, ROWS, CA_KEYS);
      if (cur.left <= 0) return;
      fresh = true;
      fetch_q();
      continue;
    }
    ++cur.kt;
    --cur.left;
  }
}

// Joins the parts of the units that lie in several stretches, in a fixed order.  With all eight warps of a CTA on a row
// the parts are spread over them (few rows, many parts: a step of one token); with one each (many rows, two or three
// parts) a warp adds a row's by itself, and takes rows_per_warp of them.  A warp has AT_ONCE parts in flight.
// (launch_combine_t chooses)
constexpr int CC_WARPS = 8, CC_THREADS = 32 * CC_WARPS;
template <typename T, int WARPS_PER_ROW, int AT_ONCE>
__global__ void __launch_bounds__(CC_THREADS) cache_combine_kernel(const CacheAttnKArgs a, int rows, int keys, int width, int max_rt, int rows_per_warp, bool permuted) {
  __shared__ unsigned total_s[CC_WARPS], before_s[CC_WARPS];
  __shared__ float acc_s[CC_WARPS][HD];
  __shared__ float2 ml_s[CC_WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, share = warp % WARPS_PER_ROW;
  // blockIdx.x = ((sequence * Hkv) + head) * max_rt + row tile
  const unsigned bh = blockIdx.x / (unsigned)max_rt;
  const int rt = (int)(blockIdx.x - bh * max_rt), b = (int)(bh / (unsigned)a.Hkv), h = (int)(bh - (unsigned)b * a.Hkv);
  const Seq s = seq_of(a, b);                        // (the lengths are older than the attention kernel)
  // places before this sequence, and in all
  unsigned before = 0, total = 0;
  for (int i = tid; i < a.n_seq; i += CC_THREADS) {
    const unsigned n = places_of_seq(a, i, rows, keys);
    total += n;
    if (i < b) before += n;
  }
  total = __reduce_add_sync(0xffffffffu, total);
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) { total_s[warp] = total; before_s[warp] = before; }
  __syncthreads();
  total = 0; before = 0;
#pragma unroll
  for (int w = 0; w < CC_WARPS; ++w) { total += total_s[w]; before += before_s[w]; }
  const Line line(total, a.max_stretches);
  const int n_kt = key_steps(s, keys);
  const unsigned u0 = before + ((unsigned)h * row_tiles(a, s, rows) + rt) * (n_kt + UNIT_STEPS);
  const int c0 = total > 0 ? (int)line.of(u0) : 0, c1 = total > 0 ? (int)line.of(u0 + n_kt - 1) : 0;
  wait_for_predecessor();
  // no such row, or written by the one that had all of its unit  (the whole CTA leaves, or whole warps of rows)
  if (rt >= row_tiles(a, s, rows) || c0 == c1) return;
  constexpr int STRIDE = CC_WARPS / WARPS_PER_ROW;
#pragma unroll 1
  for (int k = 0; k < rows_per_warp; ++k) {
    const int r = (blockIdx.y * rows_per_warp + k) * STRIDE + warp / WARPS_PER_ROW;
    const int rr = rt * rows + r;
    if (r >= rows || rr >= s.q_len * a.group) return;                  // (nor any behind it)
    auto at_of = [&](int x) { return (2LL * x + (u0 > line.begin(x) ? 1 : 0)) * a.part_rows + r; };
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f, top = NO_MAX;
    const bool mine = 4 * lane < width;
    for (int i0 = c0 + share; i0 <= c1; i0 += WARPS_PER_ROW * AT_ONCE) {
      float2 ml[AT_ONCE];
      float4 v[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const int i = i0 + j * WARPS_PER_ROW;
        ml[j] = make_float2(NO_MAX, 0.f);
        v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i <= c1) {
          const long long at = at_of(i);
          ml[j] = a.part_ml[at];
          if (mine) v[j] = *reinterpret_cast<const float4*>(a.part_o + at * width + 4 * lane);
        }
      }
      float up = top;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) up = fmaxf(up, ml[j].x);
      const float fade = ex2(top - up);
      acc.x *= fade; acc.y *= fade; acc.z *= fade; acc.w *= fade; sum *= fade;
      top = up;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const float weight = ex2(ml[j].x - top);
        sum = fmaf(ml[j].y, weight, sum);
        acc.x = fmaf(v[j].x, weight, acc.x); acc.y = fmaf(v[j].y, weight, acc.y); acc.z = fmaf(v[j].z, weight, acc.z); acc.w = fmaf(v[j].w, weight, acc.w);
      }
    }
    const int tok = rr / a.group, head = h * a.group + rr - tok * a.group;
    T* dst = reinterpret_cast<T*>(a.out) + (long long)(s.q0 + tok) * a.o_st + (long long)head * a.o_sh;
    if (WARPS_PER_ROW == 1) {
      const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
      // (the many-row kernel leaves the columns of wide heads in the order of its accumulator)
      const int n = 4 * lane, col = permuted && width == 128 ? 16 * ((n >> 3) & 7) + 8 * (n >> 6) + (n & 7) : n;
      if (mine && col < a.D) *reinterpret_cast<uint2*>(dst + col) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
    } else {
      if (mine) *reinterpret_cast<float4*>(&acc_s[warp][4 * lane]) = acc;
      if (lane == 0) ml_s[warp] = make_float2(top, sum);
      __syncthreads();
      top = NO_MAX; sum = 0.f;
      float weight[CC_WARPS];
#pragma unroll
      for (int w = 0; w < CC_WARPS; ++w) top = fmaxf(top, ml_s[w].x);
#pragma unroll
      for (int w = 0; w < CC_WARPS; ++w) { weight[w] = ex2(ml_s[w].x - top); sum = fmaf(ml_s[w].y, weight[w], sum); }
      const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
      if (tid < a.D) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < CC_WARPS; ++w) v = fmaf(acc_s[w][tid], weight[w], v);
        dst[tid] = from_float<T>(v * inv);
      }
    }
    if (a.lse != nullptr && share == WARPS_PER_ROW - 1) {
      float v = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * LN2_F;
      if (a.shift != nullptr && sum != 0.f)
        v += shift_dot(a, reinterpret_cast<const T*>(a.q) + (long long)(s.q0 + tok) * a.q_st + (long long)head * a.q_sh, h, width, lane);
      if (lane == 0) a.lse[(long long)(s.q0 + tok) * a.Hq + head] = v;
    }
  }
}

constexpr int CTAS_PER_SM = 2;
constexpr int SIZING_SMS = 160;                      // largest SM count of an sm_100 part: the workspace is sized without a device at hand

template <typename T, bool INT8, int WIDTH, int NB>
cudaError_t launch_attn(CacheAttnKArgs& a, int sms, cudaStream_t st) {
  constexpr int STAGES = 3;
  auto kern = cache_attn_kernel<T, INT8, WIDTH, NB, STAGES, CTAS_PER_SM>;
  constexpr uint32_t smem = CaSmem<WIDTH, STAGES>::BYTES;
  static DeviceOnce once;
  cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); });
  if (e != cudaSuccess) return e;
  a.max_stretches = std::min(sms, SIZING_SMS) * CTAS_PER_SM * CA_WARPS;
  const long long rts = ((long long)a.max_q * a.group + 8 * NB - 1) / (8 * NB);
  const long long steps = (long long)a.n_seq * a.Hkv * rts * (UNIT_STEPS + std::max<long long>(1, (((long long)a.table_width << a.page_shift) + CA_KEYS - 1) / CA_KEYS));
  kern<<<(unsigned)std::min<long long>(a.max_stretches / CA_WARPS, (steps + CA_WARPS - 1) / CA_WARPS), CA_THREADS, smem, st>>>(a);
  return cudaGetLastError();
}

template <typename T, bool INT8, int WIDTH>
cudaError_t launch_rows(CacheAttnKArgs& a, int rows, int sms, cudaStream_t st) {
  return rows == 8 ? launch_attn<T, INT8, WIDTH, 1>(a, sms, st) : launch_attn<T, INT8, WIDTH, 2>(a, sms, st);
}

template <typename T>
cudaError_t launch_type(CacheAttnKArgs& a, const CacheView& c, int rows, int sms, cudaStream_t st) {
  if (c.width == 64) return c.int8 ? launch_rows<T, true, 64>(a, rows, sms, st) : launch_rows<T, false, 64>(a, rows, sms, st);
  return c.int8 ? launch_rows<T, true, 128>(a, rows, sms, st) : launch_rows<T, false, 128>(a, rows, sms, st);
}

template <typename T>
cudaError_t launch_combine_t(const CacheAttnKArgs& a, int rows, int keys, int width, int max_rt, cudaStream_t st) {
  const unsigned units = (unsigned)((long long)a.n_seq * a.Hkv * max_rt);
  const bool permuted = cache_form((int64_t)a.max_q * a.group).tree;
  // All of a CTA on a row while the rows make eight CTAs an SM at most (few rows mean many parts each); a row per warp
  // beyond that, and four where even those are more: what a CTA does before its first row (it finds the unit's place in the
  // line, for which it reads every sequence's length) would be most of its time.  With the attention before it: 2048 units
  // of 4 rows over 300 keys 74.0 us with a CTA per row, 48.5 with a row per warp, 46.7 with four; one unit of 4 rows over 16 384
  // keys 15.5, 28.4 and 35.6; 32 units of 84 rows 37.0 us with a row per warp, 52.8 with four; 296 units of 256 rows 99.4 and
  // 72.1.  Parts in flight: registers decide how many CTAs are on an SM (80 with eight, 56 with four): 32 ragged sequences 45.1 us
  // with eight, 43.0 with four; 64 units of 256 rows 217.4 and 212.4; but 32 units of 84 rows, ten parts each, 37.0 and 38.9.
  constexpr unsigned long long ROOM = 8 * SIZING_SMS;
  if (!permuted && (unsigned long long)units * a.part_rows <= ROOM)
    return launch_after_predecessor(cache_combine_kernel<T, CC_WARPS, 4>, dim3(units, (unsigned)a.part_rows), dim3(CC_THREADS), 0, st, a, rows, keys, width,
                                    max_rt, 1, false);
  const unsigned ctas = (unsigned)((a.part_rows + CC_WARPS - 1) / CC_WARPS);
  if ((unsigned long long)units * ctas <= ROOM)
    return launch_after_predecessor(cache_combine_kernel<T, 1, 8>, dim3(units, ctas), dim3(CC_THREADS), 0, st, a, rows, keys, width, max_rt, 1, permuted);
  return launch_after_predecessor(cache_combine_kernel<T, 1, 4>, dim3(units, (ctas + 3) / 4), dim3(CC_THREADS), 0, st, a, rows, keys, width, max_rt, 4, permuted);
}

}  // namespace

cudaError_t launch_cache_combine(const CacheAttnKArgs& a, int dtype, int rows, int keys, int width, int max_rt, cudaStream_t st) {
  return dtype == 0 ? launch_combine_t<__half>(a, rows, keys, width, max_rt, st) : launch_combine_t<__nv_bfloat16>(a, rows, keys, width, max_rt, st);
}

// Which kernel, and rows of its row tiles.  All figures for 8 K/V heads, in a graph; the first is with the form that is taken.
//   8-row tiles up to 8 rows: a token of 4 query heads, 32 ragged sequences of up to 8192 keys, 42.5 us; with 16-row tiles
//   47.5 (8 x 16384 keys, 8 rows: 53.5 and 57.4).
//   16-row tiles of mma.sync up to 32 rows, whose keys are then read twice, but mostly from L2: 8 x 16384 keys, 32 rows,
//   107 us, with tcgen05 143; 16 rows 63 and 139.  48 rows: 144 with tcgen05, 151 with three such tiles (4 x 8771 keys: 41
//   and 31; long contexts, where more is at stake, decide).
//   tcgen05, 128 rows and two CTAs an SM up to 128 rows: 8 x 16384 keys, 128 rows, 153 us, with the 256-row form 179; 84
//   rows of 4 x 8771 keys 37 and 43.  256 rows and one CTA beyond: 160 rows 210 us, with 128-row tiles 278; 256 rows 212 and 284.
CacheForm cache_form(int64_t rows) {
  if (rows <= 32) return {false, rows <= 8 ? 8 : 16, CA_KEYS, SIZING_SMS * CTAS_PER_SM * CA_WARPS};
  return rows <= 128 ? CacheForm{true, 128, 64, 2 * SIZING_SMS} : CacheForm{true, 256, 64, SIZING_SMS};
}

size_t cache_attention_scratch(int64_t Hq, int64_t Hkv, int64_t max_q) {
  const int64_t rows = max_q * (Hq / Hkv);
  const CacheForm f = cache_form(rows);
  return (size_t)2 * f.max_stretches * std::min<int64_t>(rows, f.rows) * (HD * sizeof(float) + sizeof(float2));
}

cudaError_t launch_cache_attention(const CacheView& c, const CacheAttnParams& p, cudaStream_t st) {
  CacheAttnKArgs a;
  a.q = p.q; a.out = p.out; a.lse = p.lse; a.kc = c.k_codes; a.vc = c.v_codes; a.ks = c.k_scale; a.vs = c.v_scale; a.shift = c.k_shift;
  a.table = p.table; a.seqlens = p.seqlens; a.cu_q = p.cu_q; a.tree = p.tree;
  a.q_st = p.q_strides[0]; a.q_sh = p.q_strides[1]; a.o_st = p.o_strides[0]; a.o_sh = p.o_strides[1];
  a.table_st = p.table_stride; a.tree_st = p.tree_stride; a.total_q = p.total_q;
  a.n_seq = (int)p.n_seq; a.table_width = (int)p.table_width; a.pages = (int)c.pages; a.page_shift = c.page_shift;
  a.Hq = (int)p.Hq; a.Hkv = (int)c.H; a.group = (int)(p.Hq / c.H); a.max_q = (int)p.max_q; a.D = (int)c.D;
  a.sm_scale = p.sm_scale; a.scale_log2 = std::min(p.sm_scale * LOG2E_F, 3.0e38f);
  const int64_t rows = p.max_q * a.group;
  const CacheForm f = cache_form(rows);
  a.part_rows = (int)std::min<int64_t>(rows, f.rows);
  a.part_o = reinterpret_cast<float*>(p.scratch);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)2 * f.max_stretches * a.part_rows * HD);
  const int sms = sm_count();
  const cudaError_t e = f.tree ? launch_cache_tree(a, c, p.dtype, sms, p.status_host, st)
                               : p.dtype == 0 ? launch_type<__half>(a, c, f.rows, sms, st) : launch_type<__nv_bfloat16>(a, c, f.rows, sms, st);
  if (e != cudaSuccess) return e;
  return launch_cache_combine(a, p.dtype, f.rows, f.keys, c.width, (int)((rows + f.rows - 1) / f.rows), st);
}

}  // namespace sage
