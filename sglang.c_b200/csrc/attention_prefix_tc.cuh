// The prefixes' parts of attention over shared prefixes on the tensor cores: bfloat16, head sizes up to 128 (multiples of 8; in
// tiles of 64 or 128 columns, zeros behind a head's own: its last columns lie outside of the tensor that the copies read).
//
// One block per multiprocessor, a share of the tiles of 128 keys each (see the plan).  Scores S = Q K^T of 128 rows by 128 keys
// go into tensor memory; a thread has a row of them, takes its maximum, turns them into bfloat16 weights
// P = 2^(S c - m c) and puts these where the scores were, from where the second product O += P V takes them as its
// first operand.  O stays in tensor memory and is scaled only where a row's maximum has grown by more than 2^8 (any
// reference gives the same quotient; weights up to 2^8 lose no digits).  Two groups of four warps work in turn, so that one's
// products run under the other's exponentials:
//   rows of a group's key head <= 128: both groups have the same rows, and every other tile of keys each: what bounds it is
//     the keys' way from memory, and a tile is met by 128 rows at most whatever is done;
//   more: an item has 256 rows, 128 a group of warps, and each tile is met by both: half of the traffic for the same work.
// What bounds it: a row warp's way through a step of 64 keys, one thing after the other (wait, scores out of tensor memory, maximum,
// exponentials, rounding, store, arrival) with one other row warp beside it on its scheduler.  Of the 1.06 us between two steps of
// 256 rows of 64 it works 0.93, of 1.12 with rows of 128 0.96 to 0.99, of 0.8 with 64 rows 0.64, and waits 0.13 to 0.16 for products.  No
// unit is what it waits for: 256 requests of 32 heads of 128 over 8 on 32,768 keys take 163 us alone, 0.85 PFLOP/s, with the tensor
// pipe 42 % busy, the special-function units 44 % and the issue slots 43 %; without any exponentials the whole call fell from 187
// to 180 us.  Ahead of that a block's first scores: the plan 1.0 to 1.4 us, queries to shared memory 1.4 (8 rows) to 6.9 (256 of 128), the first
// keys and product 1 to 2.
// Keys and values come page by page through the block table by TMA, in boxes of the largest power of two of rows that
// divides the page, into a ring of tiles.  (No multicast.)
#pragma once
#include <string.h>

#include "attention_prefix.cuh"
#include "tc_common.cuh"

namespace prefix {
using namespace tc;

constexpr int TC_KEYS = 128;             // keys a tile
constexpr int TC_HALF = 64;              // keys a step: a group of warps has two buffers of scores
constexpr int TC_SLOT = 256;             // rows of a workspace slot
constexpr int TC_WG = 128;               // threads (rows) of a group of warps
constexpr int TC_MMA_WARP = 8, TC_LOAD_WARP = 10;     // (warps 0-7 rows; 8 and 9 products; 10 loads keys, 11 values)
constexpr int TC_THREADS = 384;
constexpr int TC_TILE = TC_KEYS * 128;   // bytes of 128 rows by 64 columns
constexpr int TC_MAX_RING = 4;

struct TcCtl {
  uint64_t full[2][TC_MAX_RING], empty[2][TC_MAX_RING];       // of keys, of values
  uint64_t q_full, s_full[2][2], p_ready[2][2], o_done[2], o_full[2];
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ void mma_bf16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<unsigned long long&>(x)), "l"(reinterpret_cast<unsigned long long&>(y)));
  return reinterpret_cast<float2&>(r);
}
// byte offset of 16-byte piece c (0..7) of row r in a tile of rows of 128 bytes with the 128-byte swizzle
__device__ __forceinline__ uint32_t sw128(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// Tiles of a segment that group w of the warps works on, and its i-th.
__device__ __forceinline__ int tiles_of(bool pair, int tiles, int w) { return pair ? tiles : (tiles + 1 - w) / 2; }
__device__ __forceinline__ int tile_of(bool pair, int w, int i) { return pair ? i : 2 * i + w; }

// RING: tiles of keys in shared memory, and as many of values.
template <int D, int RING>
__global__ void __launch_bounds__(TC_THREADS, 1)
prefix_tc_kernel(const __grid_constant__ CUtensorMap map_kv, const Args a, int box) {
  constexpr int DB = D / 64, UNIT = DB * TC_TILE;
  constexpr uint32_t TMEM_COLS = 512;               // scores and weights: 64 columns a buffer, 0..255; sums 256..256 + 2 D
  // All shared memory is dynamic, so the tiles begin where the 128-byte swizzle needs them, on a multiple of 1024.
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;                               // two tiles of rows
  uint8_t* ring = sQ + 2 * UNIT;                    // RING tiles of keys, RING of values
  TcCtl& ctl = *reinterpret_cast<TcCtl*>(ring + 2 * RING * UNIT);
  Plan& plan = *reinterpret_cast<Plan*>(ring + 2 * RING * UNIT + sizeof(TcCtl));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023u) {                     // never seen; the tiles would be mis-swizzled
    if (threadIdx.x == 0 && a.err) atomicOr(a.err, SGLC_FLAG_WAIT);
    pdl_wait();
    return;
  }
  if (threadIdx.x == 0) {
    for (int h = 0; h < 2; h++)
      for (int i = 0; i < RING; i++) {
        mbar_init(&ctl.full[h][i], 1);
        mbar_init(&ctl.empty[h][i], 2);
      }
    mbar_init(&ctl.q_full, 2 * TC_WG);
    for (int w = 0; w < 2; w++) {
      for (int b = 0; b < 2; b++) {
        mbar_init(&ctl.s_full[w][b], 1);
        mbar_init(&ctl.p_ready[w][b], TC_WG);
      }
      mbar_init(&ctl.o_done[w], 1);                 // (every product's end; o_full: the last one of an item's piece)
      mbar_init(&ctl.o_full[w], 1);
    }
    ctl.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == TC_MMA_WARP) {
    tmem_alloc(&ctl.tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch_dependents();                          // (not before: the second launch reads what came before this one)
  make_plan(a, plan);
  record_groups(a, plan);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = ctl.tmem_base;
  volatile int* abort_flag = &ctl.abort_flag;
  const int gq = a.gq;

  if (warp >= TC_LOAD_WARP) {
    // ---- loads, a warp for keys and one for values: a lane a box ----
    // (a copy takes a warp's turn for 200 cycles, whoever issues it: 16 pages of 16 rows a tile were 3,250 cycles in one warp)
    const int half = warp - TC_LOAD_WARP;
    uint8_t* mine = ring + half * RING * UNIT;
    // A lane holds the page of one of 32 boxes, and of one of the 32 behind them: a look into the table takes longer than a
    // tile's copies, and with one a tile ahead the loads were what the others waited for.
    Segment s = first_segment(a, plan);
    int j = 0, req = keeper(a, s);
    auto page_id = [&](int b) {                     // box b from the piece's first key on
      const long long key = (long long)s.tile * TC_KEYS + (long long)b * box;
      if (key >= s.keys || key >= (long long)(s.tile + s.tiles) * TC_KEYS) return -1;
      const int page = page_of(a, req, (int)key);
      return page < 0 ? a.n_pages : page;           // (a page outside reads as zeros)
    };
    const int of_tile = TC_KEYS / box;
    int id = page_id(lane), id_next = page_id(32 + lane), held = 0;
    uint32_t u = 0;
    bool ok = true;
    for (; s.tiles > 0; u++) {
      const int slot = u % RING, key0 = (s.tile + j) * TC_KEYS, boxes = (min(TC_KEYS, s.keys - key0) + box - 1) / box;
      if (u >= RING) {
        int w = 1;
        if (lane == 0) w = mbar_wait(&ctl.empty[half][slot], (u / RING - 1) & 1, abort_flag) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, w, 0) != 0;
        if (!ok) break;
      }
      if (lane == 0) mbar_expect_tx(&ctl.full[half][slot], (uint32_t)boxes * DB * box * 128u);
      __syncwarp();
      for (int b0 = 0; b0 < boxes; b0 += 32) {
        const int first = j * of_tile + b0;         // (a multiple of the tile's boxes, or of 32)
        if (first >= held + 32) {
          held += 32;
          id = id_next;
          id_next = page_id(held + 32 + lane);
        }
        const int page = __shfl_sync(0xffffffffu, id, (first - held + lane) & 31), b = b0 + lane;
        if (b < boxes && lane < of_tile) {
          const int in_page = (key0 + b * box) % a.page_size;
#pragma unroll
          for (int blk = 0; blk < DB; blk++)
            tma_load_5d(mine + slot * UNIT + blk * TC_TILE + b * box * 128, &map_kv, &ctl.full[half][slot], blk * 64, in_page, s.hk, half,
                        page);
        }
      }
      if (++j == s.tiles) {
        s = next_segment(a, plan, s);
        req = keeper(a, s);
        j = held = 0;
        if (s.tiles > 0) {
          id = page_id(lane);
          id_next = page_id(32 + lane);
        }
      }
    }
    if (!ok)                                        // given up: what is still on its way here lands first (a limit again)
      for (uint32_t z = u - RING; z < u; z++)
        for (uint32_t i = 0; i < c_wait_limit && !mbar_try_wait(&ctl.full[half][z % RING], (z / RING) & 1); i++) {
        }
  } else if (warp >= TC_MMA_WARP) {
    // ---- products: a warp a group of rows' warps, whose elected thread issues them (an elected one, so that descriptors stay
    // in uniform registers: issued by lane 0 of the whole warp a product took 150 cycles; one thread for both groups was
    // what the others waited for: a wait that has nothing to wait for takes it 200 cycles) ----
    // Step i of a group is half i % 2 of its tile i / 2, in buffer i % 2.  The weights of step i go over its scores;
    // behind the product that takes them come the scores of step i + 2, and those of i + 1 are there meanwhile.
    if (elect_one()) {
      constexpr uint32_t idesc_s = idesc_bf16_f32(128, TC_HALF, 0, 0);    // rows and keys both by columns of the head
      constexpr uint32_t idesc_o = idesc_bf16_f32(128, D, 0, 1);          // values as they lie: keys by rows
      const int w = warp - TC_MMA_WARP;
      const uint32_t k_at = smem_u32(ring), v_at = k_at + RING * UNIT, tS = tmem + w * 128, tO = tmem + 256 + w * D;
      uint32_t u0 = 0, q_turn = 0, turn = 0;
      bool ok = true;
      for (Segment s = first_segment(a, plan); s.tiles > 0 && ok; s = next_segment(a, plan, s)) {
        const bool pair = s.shift == 8;
        const uint32_t q_at = smem_u32(sQ) + w * UNIT;
        ok = mbar_wait(&ctl.q_full, q_turn & 1, abort_flag);
        if (!ok) break;
        q_turn++;
        // a tile is given back when both groups have taken it: where it is this one's alone, by two arrivals
        auto give_back = [&](uint64_t* bar) {
          mma_commit(bar);
          if (!pair) mbar_arrive(bar);
        };
        auto scores = [&](int i) {
          const uint32_t u = u0 + tile_of(pair, w, i >> 1), slot = u % RING;
          if ((i & 1) == 0) {
            ok = mbar_wait(&ctl.full[0][slot], (u / RING) & 1, abort_flag);
            if (!ok) return;
            tc_fence_after_sync();
          }
          const uint32_t k0 = k_at + slot * UNIT + (i & 1) * (TC_HALF * 128);
#pragma unroll
          for (int k = 0; k < D / 16; k++) {
            const uint32_t off = (k / 4) * TC_TILE + (k % 4) * 32;
            mma_bf16(tS + (i & 1) * TC_HALF, smem_desc_k_sw128(q_at + off), smem_desc_k_sw128(k0 + off), idesc_s, k > 0 ? 1u : 0u);
          }
          mma_commit(&ctl.s_full[w][i & 1]);
          if (i & 1) give_back(&ctl.empty[0][slot]);
        };
        const int n = 2 * tiles_of(pair, s.tiles, w);
        for (int i = 0; i < 2 && n > 0 && ok; i++) scores(i);
        for (int i = 0; i < n && ok; i++) {
          const uint32_t u = u0 + tile_of(pair, w, i >> 1), slot = u % RING;
          if ((i & 1) == 0) ok = mbar_wait(&ctl.full[1][slot], (u / RING) & 1, abort_flag);
          if (ok) ok = mbar_wait(&ctl.p_ready[w][i & 1], (turn >> 1) & 1, abort_flag);
          if (!ok) break;
          turn++;
          tc_fence_after_sync();
          const uint32_t v0 = v_at + slot * UNIT + (i & 1) * (TC_HALF * 128);
#pragma unroll
          for (int k = 0; k < TC_HALF / 16; k++)
            mma_bf16_ta(tO, tS + (i & 1) * TC_HALF + k * 8, smem_desc_mn_sw128(v0 + k * 2048, TC_TILE, 1024), idesc_o,
                        (i > 0 || k > 0) ? 1u : 0u);
          mma_commit(&ctl.o_done[w]);
          if (i & 1) give_back(&ctl.empty[1][slot]);
          if (i + 1 == n) mma_commit(&ctl.o_full[w]);
          if (i + 2 < n) scores(i + 2);
        }
        u0 += s.tiles;
      }
    }
  } else {
    // ---- rows: a thread a row; group w of four warps ----
    const int w = warp >> 2, row = threadIdx.x & (TC_WG - 1);
    const uint32_t lanes = (uint32_t)(warp & 3) << 21, tS = tmem + w * 128 + lanes, tO = tmem + 256 + w * D + lanes;
    const float c2 = a.scale * LOG2E;
    uint32_t turn = 0, u0 = 0, o_turn = 0;          // steps, tiles and pieces so far
    bool ok = true;
    for (Segment s = first_segment(a, plan); s.tiles > 0; s = next_segment(a, plan, s)) {
      const bool pair = s.shift == 8;
      const int rows = min(1 << s.shift, s.n_rows - s.row0);         // of this item
      // (where both groups have the same rows, the second has them 64 lanes on: up to 64 rows then keep all four schedulers
      // busy, not two of them twice)
      const int mine = pair ? w * TC_WG + row : (row + w * 64) & (TC_WG - 1);
      const int n = s.row0 + mine, t = s.t0 + (unsigned)n / (unsigned)gq;
      const bool valid = mine < rows;
      const int lim = valid ? visible(a, t, s.keys) : 0;
      // both groups are done with the item before (its products have been waited for): queries of this one
      asm volatile("bar.sync 1, 256;" ::: "memory");
      // (all 256 threads, pieces of 16 bytes side by side: a thread a row took 12,000 cycles for 256 rows of 128; four asked for
      // at a time, and rows off 16 bytes in a loop of their own: the less code there is to fetch, the sooner a block begins)
      auto query = [&](int at) {                     // where piece `at` lies, or null: zeros
        const int r = at / (D / 8), c = at % (D / 8), nr = s.row0 + r, tr = (unsigned)nr / (unsigned)gq;
        const __nv_bfloat16* from = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)(s.t0 + tr) * a.q_stride + (size_t)(s.hk * gq + nr - tr * gq) * a.D + c * 8;
        return r < rows && c * 8 < a.D ? from : nullptr;
      };
      auto put = [&](int at, uint4 x) {
        const int r = at / (D / 8), c = at % (D / 8);
        uint8_t* to = sQ + (c / 8) * TC_TILE;
        *reinterpret_cast<uint4*>(to + (r / TC_WG) * UNIT + sw128(r % TC_WG, c % 8)) = x;
        if (!pair) *reinterpret_cast<uint4*>(to + UNIT + sw128((r + 64) & (TC_WG - 1), c % 8)) = x;
      };
      const int pieces = (D / 8) << s.shift;         // (a multiple of 4 for each thread)
      if (a.q_vec) {
        for (int x0 = threadIdx.x; x0 < pieces; x0 += 4 * 2 * TC_WG) {
          uint4 x[4];
#pragma unroll
          for (int u = 0; u < 4; u++) {
            const __nv_bfloat16* from = query(x0 + u * 2 * TC_WG);
            x[u] = from ? *reinterpret_cast<const uint4*>(from) : make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (int u = 0; u < 4; u++) put(x0 + u * 2 * TC_WG, x[u]);
        }
      } else {
#pragma unroll 1
        for (int at = threadIdx.x; at < pieces; at += 2 * TC_WG) {
          const unsigned short* h = reinterpret_cast<const unsigned short*>(query(at));
          put(at, h ? make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16)
                    : make_uint4(0u, 0u, 0u, 0u));
        }
      }
      fence_async_proxy();
      mbar_arrive(&ctl.q_full);
      const bool busy = (mine & ~31) < rows;         // this warp has rows at all
      const int steps = 2 * tiles_of(pair, s.tiles, w);
      float m = -INFINITY, l = 0.0f;
      for (int i = 0; i < steps && ok; i++, turn++) {
        ok = mbar_wait(&ctl.s_full[w][i & 1], (turn >> 1) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after_sync();
        if (busy) {
          const uint32_t at = tS + (i & 1) * TC_HALF;
          uint32_t v[2][32];
          tmem_ld_32x32(at, v[0]);
          tmem_ld_32x32(at + 32, v[1]);
          tmem_ld_wait();
          const int in_step = lim - (s.tile + tile_of(pair, w, i >> 1)) * TC_KEYS - (i & 1) * TC_HALF;    // keys of it the row sees
          if (!__all_sync(0xffffffffu, in_step >= TC_HALF)) {
#pragma unroll
            for (int x = 0; x < TC_HALF; x++)
              if (x >= in_step) v[x >> 5][x & 31] = 0xff800000u;              // -inf
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int x = 0; x < TC_HALF; x++) mx[x & 3] = fmaxf(mx[x & 3], __uint_as_float(v[x >> 5][x & 31]));
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          float alpha = 1.0f;
          if (m == -INFINITY) {
            m = top;                                 // (a row's first keys: its sums are zero)
          } else if ((top - m) * c2 > 8.0f) {
            alpha = ex2((m - top) * c2);
            l *= alpha;
            m = top;
          }
          if (__any_sync(0xffffffffu, alpha != 1.0f)) {
            // The sums are scaled once the product before this step is done.  (The one before that is: this step's scores
            // came behind it.)
            ok = mbar_wait(&ctl.o_done[w], (turn - 1) & 1, abort_flag);
            tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; ok && c < D; c += 32) {
              uint32_t o[32];
              tmem_ld_32x32(tO + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 32; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
              tmem_st_32x32(tO + c, o);
            }
          }
          const float neg = m == -INFINITY ? 0.0f : -m * c2;
          float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
          uint32_t p[32];
#pragma unroll
          for (int x = 0; x < 32; x++) {
            const uint32_t* y = &v[x / 16][2 * (x % 16)];
            const float2 e = fma2(make_float2(__uint_as_float(y[0]), __uint_as_float(y[1])), make_float2(c2, c2), make_float2(neg, neg));
            const __nv_bfloat162 hh = __floats2bfloat162_rn(ex2(e.x), ex2(e.y));
            p[x] = *reinterpret_cast<const uint32_t*>(&hh);
            // (the sum is of the rounded weights, which the values get: a row of one large weight has no error of it)
            sum[x & 1] = add2(sum[x & 1], make_float2(__uint_as_float(p[x] << 16), __uint_as_float(p[x] & 0xffff0000u)));
          }
          tmem_st_32x32(at, p);
          sum[0] = add2(sum[0], sum[1]);
          l += sum[0].x + sum[0].y;
          tmem_st_wait();
        }
        const int tile = tile_of(pair, w, i >> 1), in_tile = s.keys - (s.tile + tile) * TC_KEYS;
        if (in_tile < TC_KEYS && (i & 1) == 0) {
          // The end of the prefix: behind its last key a tile of values holds what the page or the ring held, which may be no
          // number.  It becomes zeros, as the weights there are, before the weights are handed on.  (The parity tells this
          // tile's landing, as the one that had its place in the ring before has landed: in the same piece it was this
          // group's too, the ring being even, and behind a product that these scores came behind; a tile of an earlier piece may
          // have been the other group's, but both groups waited for their last products of it ahead of the barrier above.  Where
          // both groups take the tile both write the zeros.)
          const uint32_t u = u0 + tile, slot = u % RING;
          ok = mbar_wait(&ctl.full[1][slot], (u / RING) & 1, abort_flag);
          if (!ok) break;
          for (int x = row; x < (TC_KEYS - in_tile) * 8 * DB; x += TC_WG) {
            const int r = in_tile + x / (8 * DB), c = x % (8 * DB);
            *reinterpret_cast<uint4*>(ring + (RING + slot) * UNIT + (c / 8) * TC_TILE + r * 128 + (c % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_proxy();
        }
        tc_fence_before_sync();
        mbar_arrive(&ctl.p_ready[w][i & 1]);
      }
      if (steps > 0 && ok) {
        ok = mbar_wait(&ctl.o_full[w], o_turn++ & 1, abort_flag);
        tc_fence_after_sync();
      }
      if (threadIdx.x == 0) record_item(a, s);
      if (__all_sync(0xffffffffu, ok) && busy) {
        const long long at = (long long)(blockIdx.x + s.item) * TC_SLOT + (pair ? 0 : w * TC_WG) + mine;
        const bool there = valid && slot_ok(a, s);
        if (there) a.part_ml[at] = make_float2(m == -INFINITY ? -INFINITY : m * c2, l);
        if (steps > 0) {
          // More than 64 rows (32 of two blocks of columns) go out by way of where the queries were, so that eight lanes store 128 bytes side by side: a thread a row, 16
          // bytes of 32 rows a store, took 2.6 us for 256 rows of 64 and 5.5 for rows of 128 (96 rows of 96, a whole call: 26.1 us,
          // 23.8 this way; 64 rows of 128: 23.5 and 22.9).  Of fewer rows a store reaches few lines, and the way round is the longer one (a
          // whole call with 8 rows of 64: 56.3 us, 57.6 this way; with 64: 39.4 and 39.9).
          if (rows * DB <= 64) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld_32x32(tO + c, o);
              tmem_ld_wait();
              if (there)
#pragma unroll
                for (int x = 0; x < 32; x += 4)
                  if (c + x < a.D) *reinterpret_cast<uint4*>(a.part_o + at * a.D + c + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
            }
          } else {
            uint8_t* turn_at = sQ + w * UNIT + (warp & 3) * 32 * 128;
            const unsigned rows_there = __ballot_sync(0xffffffffu, there);
            const long long at0 = at - lane;           // (a warp's rows lie side by side in the slot)
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld_32x32(tO + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 32; x += 4)
                *reinterpret_cast<uint4*>(turn_at + sw128(lane, x / 4)) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
              __syncwarp();
#pragma unroll 2
              for (int x = 0; x < 8; x++) {
                const int r = 4 * x + (lane >> 3), k = lane & 7;
                if ((rows_there >> r & 1) && c + 4 * k < a.D)
                  *reinterpret_cast<uint4*>(a.part_o + (at0 + r) * a.D + c + 4 * k) = *reinterpret_cast<const uint4*>(turn_at + sw128(r, k));
              }
              __syncwarp();
            }
          }
        }
      }
      tc_fence_before_sync();
      u0 += s.tiles;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && ctl.abort_flag && a.err) atomicOr(a.err, SGLC_FLAG_WAIT);
  if (warp == TC_MMA_WARP) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// One layer's pages [n_pages][2][Hkv][page_size][D] as a 5-D tensor, in boxes of `box` rows of one page and head, 64 columns wide.
static inline bool make_kv_map(CUtensorMap* out, const Args& a, int box) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t D = a.D, ps = a.page_size, Hkv = a.Hkv;
  cuuint64_t dims[5] = {D, ps, Hkv, 2, (cuuint64_t)a.n_pages};
  cuuint64_t strides[4] = {D * 2, ps * D * 2, Hkv * ps * D * 2, 2 * Hkv * ps * D * 2};
  cuuint32_t boxes[5] = {64, (cuuint32_t)box, 1, 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(a.cache), dims, strides, boxes, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// (internal linkage: what it keeps must not be one with that of another library built from this file)
template <int D, int RING>
static int launch_tc(const Args& a, cudaStream_t stream) {
  static_assert(RING % 2 == 0 && RING <= TC_MAX_RING, "the ring's barriers");
  constexpr size_t smem = (size_t)(2 + 2 * RING) * (D / 64) * TC_TILE + sizeof(TcCtl) + sizeof(Plan);
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  int box = 1;
  while (box < TC_KEYS && a.page_size % (box * 2) == 0) box *= 2;
  CUtensorMap map;
  memset(&map, 0, sizeof(map));
  if (!make_kv_map(&map, a, box)) return SGLC_ERR_UNSUPPORTED;
  static std::atomic<unsigned long long> done{0};
  const int code = allow_shared(prefix_tc_kernel<D, RING>, (int)smem, done);
  if (code) return code;
  return sglc_launch(prefix_tc_kernel<D, RING>, dim3(a.n_blocks), dim3(TC_THREADS), smem, stream, 1, true, map, a, box);
}
}  // namespace prefix
