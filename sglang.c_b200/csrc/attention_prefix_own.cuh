// The second launch of attention over shared prefixes for bfloat16 heads of 64 and 128: the tokens' own keys, and all parts
// joined.
//
// An item is up to 16 rows of one key head: the query heads of a token, or those of several tokens that stand side by side
// (where requests bring several, most of them share their keys).  A warp takes 16 keys at a time on the warp-level
// tensor-core instruction: 16 x 16 scores, their weights as bfloat16, 16 x D sums.  (tcgen05 would want 128 rows; here a
// few rows meet keys that nobody else reads, and what bounds it is instructions and the keys' way from memory: on
// multiply-adds, 1,961 tokens of 16 heads with 30 keys each took 50 us, this way 16.)
// Operands come from global memory straight into the instruction's registers, 16 bytes a lane: with lane = 4 g + q, a lane
// holds of key g the columns 8 q .. 8 q + 7 of each block of 32.  Which column is called which along the sum over
// columns does not matter as long as queries and keys agree; and of the values, whose 8 x 8 pieces are transposed in
// registers, a lane ends with eight neighbouring columns of a row of sums, as the parts and the results lie in memory.
#pragma once
#include <type_traits>

#include "attention_prefix.cuh"

namespace prefix {
constexpr int MT = 128;                  // threads
constexpr int MR = 16;                   // rows of an item
constexpr int JOIN_ONE = 8, JOIN_TWO = 4;      // items a multiprocessor from which an item has one warp, two

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit elements, two neighbours of row lane / 4 in a lane, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// WARPS: of an item; a block has four.  tokens: of an item; heads: rows of a token.
template <int D, int WARPS>
__global__ void __launch_bounds__(MT)
prefix_join_kernel(const Args a, int tokens, int heads) {
  extern __shared__ __align__(16) float sm[];          // [4 warps][16 rows][D + 2], then factors: for items of several warps
  constexpr int ITEMS = 4 / WARPS, B = D / 32;
  typedef __nv_bfloat16 T;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int share = blockIdx.z, shares = gridDim.z;
  if (shares > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_launch_dependents();
  const int head_chunks = (a.gq + MR - 1) / MR, hk = blockIdx.y / head_chunks, head0 = (blockIdx.y - hk * head_chunks) * MR;
  const int t_first = (blockIdx.x * ITEMS + warp / WARPS) * tokens;
  const int walker = share * WARPS + warp % WARPS, walkers = WARPS * shares;

  // lane i knows token i of the item: its group (the last one that begins at or before it), request and range of own keys
  const int tl = t_first + lane;
  int group = -1, t0 = 0, t1 = 0, req = -1, lo = 0, hi = 0;
  for (int x = 0; x < a.G; x += 32) {
    const int start = x + lane < a.G ? a.group_start[x + lane] : 0x7fffffff;
    for (int i = 0; i < tokens; i++) {
      const int n = __popc(__ballot_sync(0xffffffffu, start <= t_first + i));
      if (lane == i) group += n;
    }
  }
  bool inside = lane < tokens && tl < a.T && group >= 0;
  if (inside) {
    group_tokens(a, group, t0, t1);
    const int pos = a.positions[tl], r = a.token_req ? a.token_req[tl] : tl, end = a.group_start[a.G];
    lo = prefix_length(a, group);
    inside = tl >= t0 && tl < t1;
    if (inside) {
      if (pos > a.last_position || r < 0 || r >= a.R) flag_index(a);
      hi = min(pos, a.last_position) + 1;
      req = r >= 0 && r < a.R ? r : -1;
      if (!sees_all(pos, lo)) {                        // inside the prefix, whose pages the group's first request names
        lo = 0;
        req = request_of(a, t0);
      }
    } else if (tl < end) {
      flag_index(a);                                   // starts that do not ascend
    }
  }
  // this lane's rows of sums: g and g + 8
  int row_token[2], row_lo[2], row_hi[2];
  bool row_in[2];
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const int r = g + 8 * x, i = (unsigned)r / (unsigned)heads, h = r - i * heads;
    row_token[x] = i;
    row_in[x] = __shfl_sync(0xffffffffu, (int)inside, i & 31) && i < tokens && head0 + h < a.gq;
    row_lo[x] = __shfl_sync(0xffffffffu, lo, i & 31);
    row_hi[x] = __shfl_sync(0xffffffffu, req >= 0 ? hi : 0, i & 31);
  }
  const float c2 = a.scale * LOG2E;
  uint32_t qf[B][2][4];                                // queries: [block of 32 columns][step of 16][instruction's registers]
#pragma unroll
  for (int x = 0; x < 2; x++) {
    const int r = g + 8 * x, h = r - row_token[x] * heads;
    const T* src = reinterpret_cast<const T*>(a.q) + (size_t)(t_first + row_token[x]) * a.q_stride + (size_t)(hk * a.gq + head0 + h) * D + 8 * q;
#pragma unroll
    for (int b = 0; b < B; b++) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row_in[x]) {
        if (a.q_vec) {
          v = *reinterpret_cast<const uint4*>(src + 32 * b);
        } else {
          const unsigned short* s = reinterpret_cast<const unsigned short*>(src + 32 * b);
          v = make_uint4(s[0] | (uint32_t)s[1] << 16, s[2] | (uint32_t)s[3] << 16, s[4] | (uint32_t)s[5] << 16, s[6] | (uint32_t)s[7] << 16);
        }
      }
      qf[b][0][x] = v.x;
      qf[b][0][2 + x] = v.y;
      qf[b][1][x] = v.z;
      qf[b][1][2 + x] = v.w;
    }
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};      // (l: this lane's share of a row's sum)
  float o[B][4][4];                                    // [block][pair of columns 8 q + 2 j][row g: 0, 1; row g + 8: 2, 3]
#pragma unroll
  for (int b = 0; b < B; b++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) o[b][j][i] = 0.0f;
  const size_t v_at = value_offset(a);
  // A tile's rows do not see the same keys, and a weight of 0 times an infinite value, or one that is no number, is no number:
  // where the sums end with such, the walk is done again, with the values row by row as that row sees them.
  auto walk = [&](auto row_by_row) {
    // one request after the other (their tokens need not stand together)
    unsigned todo = __ballot_sync(0xffffffffu, inside && req >= 0 && hi > lo);
    while (todo) {
      const int who = __shfl_sync(0xffffffffu, req, __ffs(todo) - 1);
      const unsigned same = __ballot_sync(0xffffffffu, inside && req == who) & todo;
      todo &= ~same;
      const bool mine = same >> lane & 1;
      const int first = __reduce_min_sync(0xffffffffu, mine ? lo : 0x7fffffff), last = __reduce_max_sync(0xffffffffu, mine ? hi : 0);
      int from[2], to[2];
#pragma unroll
      for (int x = 0; x < 2; x++) {
        const bool here = row_in[x] && (same >> (row_token[x] & 31) & 1);
        from[x] = here ? row_lo[x] : 0x7fffffff;
        to[x] = here ? row_hi[x] : 0;
      }
      int block0 = -64, id = -1;                         // 32 pages at a time, a lane an id
      for (long long key_at = first + 16LL * walker; key_at < last; key_at += 16LL * walkers) {
        const int key0 = (int)key_at;
        uint4 kv[2][2][B];                               // [keys g, g + 8][keys, values][block]
        const int page_block = block_in(a, key0), top_block = block_in(a, min(key0 + 15, last - 1));
        if (top_block >= block0 + 32 || page_block < block0) {
          block0 = page_block;
          id = (long long)(block0 + lane) * a.page_size < last ? page_of(a, who, (block0 + lane) * a.page_size) : -1;
        }
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const int key = key0 + 8 * x + g, block = block_in(a, key);
          const int page = __shfl_sync(0xffffffffu, id, (block - block0) & 31);
          const bool there = key < last && page >= 0;
          const T* src = reinterpret_cast<const T*>(a.cache) +
                         (((size_t)(there ? page : 0) * 2 * a.Hkv + hk) * a.page_size + (there ? key - block * a.page_size : 0)) * D + 8 * q;
#pragma unroll
          for (int b = 0; b < B; b++) {
            kv[x][0][b] = kv[x][1][b] = make_uint4(0u, 0u, 0u, 0u);
            if (there) {
              kv[x][0][b] = *reinterpret_cast<const uint4*>(src + 32 * b);
              kv[x][1][b] = *reinterpret_cast<const uint4*>(src + v_at + 32 * b);
            }
          }
        }
        float s[2][4];                                   // scores: [keys 0..7, 8..15][row g: keys 2 q, 2 q + 1; row g + 8]
#pragma unroll
        for (int x = 0; x < 2; x++) {
#pragma unroll
          for (int i = 0; i < 4; i++) s[x][i] = 0.0f;
#pragma unroll
          for (int b = 0; b < B; b++) {
            mma_16816(s[x], qf[b][0], kv[x][0][b].x, kv[x][0][b].y);
            mma_16816(s[x], qf[b][1], kv[x][0][b].z, kv[x][0][b].w);
          }
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int key = key0 + 8 * x + 2 * q + (i & 1);
            s[x][i] = key >= from[i >> 1] && key < to[i >> 1] ? s[x][i] * c2 : -INFINITY;
            top[i >> 1] = fmaxf(top[i >> 1], s[x][i]);
          }
        bool moved = false;
        float f[2], ref[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
          top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
          top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
          top[x] = fmaxf(top[x], m[x]);
          ref[x] = top[x] == -INFINITY ? 0.0f : top[x];
          f[x] = ex2(m[x] - ref[x]);
          moved |= top[x] > m[x];
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int x = 0; x < 2; x++) {
            l[x] *= f[x];
            m[x] = top[x];
          }
#pragma unroll
          for (int b = 0; b < B; b++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
              for (int i = 0; i < 4; i++) o[b][j][i] *= f[i >> 1];
        }
        uint32_t p[4];
#pragma unroll
        for (int x = 0; x < 2; x++) {
          // (sums of the rounded weights, which the values get)
#pragma unroll
          for (int y = 0; y < 2; y++) {
            const uint32_t w = pack_bf16(ex2(s[x][2 * y] - ref[y]), ex2(s[x][2 * y + 1] - ref[y]));
            l[y] += __uint_as_float(w << 16) + __uint_as_float(w & 0xffff0000u);
            p[2 * x + y] = w;
          }
        }
#pragma unroll
        for (int b = 0; b < B; b++) {
          const uint32_t v0[4] = {kv[0][1][b].x, kv[0][1][b].y, kv[0][1][b].z, kv[0][1][b].w};
          const uint32_t v1[4] = {kv[1][1][b].x, kv[1][1][b].y, kv[1][1][b].z, kv[1][1][b].w};
          if constexpr (!decltype(row_by_row)::value) {
#pragma unroll
            for (int j = 0; j < 4; j++) mma_16816(o[b][j], p, transposed(v0[j]), transposed(v1[j]));
          } else {
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll 1
              for (int i = 0; i < 8; i++) {              // row i + 8 x, which lanes 4 i .. 4 i + 3 have
                const int begin = __shfl_sync(0xffffffffu, from[x], 4 * i), end = __shfl_sync(0xffffffffu, to[x], 4 * i);
                const bool see0 = key0 + g >= begin && key0 + g < end, see1 = key0 + 8 + g >= begin && key0 + 8 + g < end;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  float one[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                  mma_16816(one, p, transposed(see0 ? v0[j] : 0u), transposed(see1 ? v1[j] : 0u));
                  if (g == i) {
                    o[b][j][2 * x] += one[2 * x];
                    o[b][j][2 * x + 1] += one[2 * x + 1];
                  }
                }
              }
          }
        }
      }
    }
  };
  walk(std::false_type());
  if (tokens > 1) {
    float number = 0.0f;
#pragma unroll
    for (int b = 0; b < B; b++)
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) number = fmaf(o[b][j][i], 0.0f, number);
    if (__any_sync(0xffffffffu, number != number)) {
#pragma unroll
      for (int x = 0; x < 2; x++) m[x] = -INFINITY, l[x] = 0.0f;
#pragma unroll
      for (int b = 0; b < B; b++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int i = 0; i < 4; i++) o[b][j][i] = 0.0f;
      walk(std::true_type());
    }
  }
#pragma unroll
  for (int x = 0; x < 2; x++) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
  }
  const int g0 = __shfl_sync(0xffffffffu, group, row_token[0] & 31), g1 = __shfl_sync(0xffffffffu, group, row_token[1] & 31);
  const int s0 = __shfl_sync(0xffffffffu, t0, row_token[0] & 31), s1 = __shfl_sync(0xffffffffu, t0, row_token[1] & 31);
  const int e0 = __shfl_sync(0xffffffffu, t1, row_token[0] & 31), e1 = __shfl_sync(0xffffffffu, t1, row_token[1] & 31);
  pdl_wait();                                          // the prefixes' parts are there
  // (both rows' parts together: a part is a chain of three reads)
  Parts ps[2];
#pragma unroll
  for (int x = 0; x < 2; x++) {
    ps[x].n = 0;
    if (!row_in[x] || row_lo[x] == 0) continue;
    const int from = x ? s1 : s0, h = g + 8 * x - row_token[x] * heads;
    ps[x] = parts_of(a, x ? g1 : g0, from, x ? e1 : e0, hk, (t_first + row_token[x] - from) * a.gq + head0 + h);
  }
  for (int j = walker; j < max(ps[0].n, ps[1].n); j += walkers) {
    float2 ml[2];
    float4 v[2][B][2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const long long at = j < ps[x].n ? part_row(a, ps[x], j) : -1;
      ml[x] = make_float2(-INFINITY, 0.0f);
      if (at >= 0) {
        ml[x] = a.part_ml[at];
#pragma unroll
        for (int b = 0; b < B; b++) {
          v[x][b][0] = *reinterpret_cast<const float4*>(a.part_o + at * D + 32 * b + 8 * q);
          v[x][b][1] = *reinterpret_cast<const float4*>(a.part_o + at * D + 32 * b + 8 * q + 4);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
      if (ml[x].y == 0.0f) continue;                   // nothing was seen and no sums were written (NaN is not 0)
      const float top = fmaxf(m[x], ml[x].x), ref = top == -INFINITY ? 0.0f : top, f = ex2(m[x] - ref), f2 = ex2(ml[x].x - ref);
      m[x] = top;
      l[x] = l[x] * f + ml[x].y * f2;
#pragma unroll
      for (int b = 0; b < B; b++) {
        const float w[8] = {v[x][b][0].x, v[x][b][0].y, v[x][b][0].z, v[x][b][0].w, v[x][b][1].x, v[x][b][1].y, v[x][b][1].z, v[x][b][1].w};
#pragma unroll
        for (int i = 0; i < 8; i++) o[b][i >> 1][2 * x + (i & 1)] = o[b][i >> 1][2 * x + (i & 1)] * f + w[i] * f2;
      }
    }
  }
  if constexpr (WARPS == 1) {
#pragma unroll
    for (int x = 0; x < 2; x++) {
      if (!row_in[x]) continue;
      const int h = g + 8 * x - row_token[x] * heads;
      const float f = l[x] == 0.0f ? 0.0f : 1.0f / l[x];
      T* to = reinterpret_cast<T*>(a.out) + (size_t)(t_first + row_token[x]) * a.o_stride + (size_t)(hk * a.gq + head0 + h) * D + 8 * q;
#pragma unroll
      for (int b = 0; b < B; b++) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = l[x] == 0.0f ? 0.0f : o[b][i >> 1][2 * x + (i & 1)] * f;
        store8(to + 32 * b, a.o_vec, v);
      }
    }
  } else {
    // the item's warps, and the cluster's blocks
    constexpr int one = MR * (D + 2);
    const int parts = WARPS * shares, warp0 = warp / WARPS * WARPS, me = threadIdx.x % (WARPS * 32);
#pragma unroll
    for (int x = 0; x < 2; x++) {
      float* to = sm + warp * one + (g + 8 * x) * (D + 2);
      if (row_in[x]) {
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
          for (int i = 0; i < 8; i++) to[32 * b + 8 * q + i] = o[b][i >> 1][2 * x + (i & 1)];
        if (q == 0) {
          to[D] = m[x];
          to[D + 1] = l[x];
        }
      }
    }
    if (shares > 1) {
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");     // (of the start)
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
      __syncthreads();
    }
    auto other = [&](int z, int i) {                   // word i of warp z of the item
      const float* at = sm + (warp0 + z % WARPS) * one + i;
      if (z < WARPS) return *at;
      uint32_t there;
      float v;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(z / WARPS));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
      return v;
    };
    const int rows = min(tokens * heads, MR);
    float* factor = sm + 4 * one + warp0 * MR * shares;
    const int r_tok = me < rows ? (unsigned)me / (unsigned)heads : 0;
    const bool me_in = __shfl_sync(0xffffffffu, (int)inside, r_tok & 31) && me < rows && head0 + me - r_tok * heads < a.gq;
    if (share == 0 && me < MR) {
      const int at = me * (D + 2) + D;
      float M = -INFINITY, total = 0.0f;
      if (me_in)
        for (int z = 0; z < parts; z++) M = fmaxf(M, other(z, at));
      const float ref = M == -INFINITY ? 0.0f : M;
      if (me_in)
        for (int z = 0; z < parts; z++) {
          const float f = ex2(other(z, at) - ref);
          factor[me * parts + z] = f;
          total = fmaf(f, other(z, at + 1), total);
        }
      const float f = total == 0.0f ? 0.0f : 1.0f / total;
      for (int z = 0; z < parts; z++) factor[me * parts + z] = me_in ? factor[me * parts + z] * f : -1.0f;       // (-1: no such row)
    }
    __syncthreads();
    if (share == 0)
      for (int x = me; x < rows * D; x += WARPS * 32) {
        const int r = x / D, c = x - r * D;
        if (factor[r * parts] < 0.0f) continue;
        float sum = 0.0f;
        for (int z = 0; z < parts; z++) sum = fmaf(factor[r * parts + z], other(z, r * (D + 2) + c), sum);
        const int i = (unsigned)r / (unsigned)heads;
        reinterpret_cast<T*>(a.out)[(size_t)(t_first + i) * a.o_stride + (size_t)(hk * a.gq + head0 + r - i * heads) * D + c] =
            __float2bfloat16_rn(sum);
      }
    if (shares > 1) {                                  // (block 0 has read the others' shared memory)
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
  }
}

template <int D, int WARPS>
int launch_join(const Args& a, int tokens, int heads, int shares, cudaStream_t stream) {
  const size_t smem = WARPS == 1 ? 0 : (size_t)(4 * MR * (D + 2) + 4 * MR * shares) * 4;
  static_assert((4 * MR * (D + 2) + 4 * MR * 8) * 4 <= 48 * 1024, "shared memory without an attribute");
  const long long chunks = ((long long)a.T + tokens - 1) / tokens;
  return sglc_launch(prefix_join_kernel<D, WARPS>, dim3((unsigned)((chunks * WARPS + 3) / 4), a.Hkv * ((a.gq + MR - 1) / MR), shares),
                     dim3(MT), smem, stream, shares, true, a, tokens, heads);
}
// Tokens an item: as many as fill 16 rows, where a request brings so many.  As far as sizes tell, that is: the host knows tokens and
// rows of the table, not which rows have tokens, nor how many each.  Rows that no token has make items smaller (69 requests of 28 tokens
// of 16 heads of 64: 43 us with a table of 69 rows; with 1,024 an item is a token, the multiply-add kernel's, and the call takes
// 77), and a long portion beside single tokens makes an item of those a walk over sixteen requests (900 tokens of a request 60 us, 60
// requests of a token 27, both in a call 174).
static inline int join_tokens(const Args& a) {
  const int heads = a.gq < MR ? a.gq : MR;
  int tokens = 1;
  while (tokens * 2 * heads <= MR && (long long)tokens * 2 * a.R <= a.T) tokens *= 2;
  return tokens;
}
// Four rows an item and more: below, the 16 rows of the instruction are mostly empty and the multiply-add kernel wins (64
// requests of 25 heads of one: 55 against 44 us for the whole call, 100 of 16 heads over 8: 36 against 27; 256 of
// 32 heads over 8: 187 against 205).
static inline bool join_pays(const Args& a) { return a.tc && (a.D == 64 || a.D == 128) && join_tokens(a) * a.gq >= 4; }
// Warps an item: one where the items fill the multiprocessors' warps, else two, else four, and blocks of a
// cluster while there are fewer than four a multiprocessor and 64 keys or more are left for each.
template <int D>
int run_join(const Args& a, int max_own, cudaStream_t stream) {
  const int heads = a.gq < MR ? a.gq : MR, tokens = join_tokens(a);
  const long long items = ((long long)a.T + tokens - 1) / tokens * a.Hkv * ((a.gq + MR - 1) / MR);
  if (items >= JOIN_ONE * a.sms) return launch_join<D, 1>(a, tokens, heads, 1, stream);
  if (items >= JOIN_TWO * a.sms) return launch_join<D, 2>(a, tokens, heads, 1, stream);
  int shares = 1;
  while (shares < 8 && items * shares * 2 <= 4LL * a.sms && max_own >= 64 * shares * 2) shares *= 2;
  return launch_join<D, 4>(a, tokens, heads, shares, stream);
}
}  // namespace prefix
