// What the launches of attention over shared prefixes agree on: the plan of items and shares that each block makes from
// the groups' lengths, where parts lie in the workspace, and access to the paged cache with every index checked.
#pragma once
#include <atomic>

#include "common.cuh"

namespace prefix {
constexpr int MAX_GROUPS = 256;
constexpr int GENERAL_KEYS = 64;          // a tile's keys in 32-bit arithmetic
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
  const void* q;
  long long q_stride;
  int q_vec;                              // rows of queries can be read 16 bytes at a time
  const void* cache;                      // [n_pages][2][Hkv][page_size][D]
  const int* table;
  long long bt_stride;
  const int *token_req, *positions, *group_start, *shared_len;
  void* out;
  long long o_stride;
  int o_vec;                              // (so can rows of results)
  int T, R, G, H, Hkv, gq, D, page_size, n_pages;        // gq: query heads of a key head
  int page_shift;                         // log2 of the page size, or -1
  int last_position;                      // the last one that a row of the table has room for
  float scale;
  int* err;
  // the launch
  int sms, n_blocks, slot_rows, key_shift, row_shift, lanes;       // log2 of a tile's keys, of an item's rows (not tc)
  int tc;                                 // the tensor-core kernel
  long long slots;
  float* part_o;                          // [slots][slot_rows][D]: sums, against a maximum
  float2* part_ml;                        // [slots][slot_rows]: that maximum (times log2 e), sum of weights
  int* first_item;                        // [G]: items of the groups before, or -1: no prefix, or one that no request names
  int2* item_blocks;                      // [slots]: the first and the last block that has a piece of the item
};

// Per group: first token, keys of the prefix, rows a key head, and what lies before it: items and tiles.
struct Plan {
  int t0[MAX_GROUPS], keys[MAX_GROUPS], rows[MAX_GROUPS];
  int items[MAX_GROUPS + 1];
  long long tiles[MAX_GROUPS + 1];
  long long at, end;                      // this block's share of the tiles
};

__device__ __forceinline__ void flag_index(const Args& a) {
  if (a.err) atomicOr(a.err, SGLC_FLAG_INDEX);
}
__device__ __forceinline__ int request_of(const Args& a, int t) {
  const int r = a.token_req ? a.token_req[t] : t;
  if (r >= 0 && r < a.R) return r;
  flag_index(a);
  return -1;
}
__device__ __forceinline__ int block_in(const Args& a, int key) {
  return a.page_shift >= 0 ? key >> a.page_shift : (int)((unsigned)key / (unsigned)a.page_size);
}
__device__ __forceinline__ int page_of(const Args& a, int req, int key) {
  if (req < 0) return -1;
  const int page = a.table[(size_t)req * a.bt_stride + block_in(a, key)];
  if (page >= 0 && page < a.n_pages) return page;
  flag_index(a);
  return -1;
}
__device__ __forceinline__ size_t row_at(const Args& a, int page, int hk, int key) {
  return (((size_t)page * 2 * a.Hkv + hk) * a.page_size + (key - block_in(a, key) * a.page_size)) * a.D;
}
__device__ __forceinline__ size_t value_offset(const Args& a) { return (size_t)a.Hkv * a.page_size * a.D; }
// A token inside a prefix of `keys` sees only its first ones, and is the second launch's with all of them: in a tile that
// rows beside it see further into, the first would give it weights of 0 times values that it must not see, which are no
// zeros where those are infinite or no numbers.
__device__ __forceinline__ bool sees_all(int position, int keys) { return position >= keys - 1; }
// keys of a prefix of `keys` that token t gets from the first launch
__device__ __forceinline__ int visible(const Args& a, int t, int keys) { return sees_all(a.positions[t], keys) ? keys : 0; }

// A group's tokens and how many keys of its prefix there are.
__device__ __forceinline__ void group_tokens(const Args& a, int g, int& t0, int& t1) {
  t0 = min(max(a.group_start[g], 0), a.T);
  t1 = min(max(a.group_start[g + 1], t0), a.T);
}
__device__ __forceinline__ int prefix_length(const Args& a, int g) { return min(max(a.shared_len[g], 0), a.last_position + 1); }

// Rows of an item of a group of so many rows a key head, as a power of two.
__device__ __forceinline__ int item_shift(const Args& a, int rows) { return !a.tc ? a.row_shift : rows <= 128 ? 7 : 8; }
__device__ __forceinline__ int items_of(const Args& a, int rows) { return (int)(((long long)rows + (1 << item_shift(a, rows)) - 1) >> item_shift(a, rows)); }
__device__ __forceinline__ int tiles_of_keys(const Args& a, int keys) { return (keys + (1 << a.key_shift) - 1) >> a.key_shift; }
// (a division of 64 bits takes a hundred instructions)
__device__ __forceinline__ long long divide(long long x, int y) {
  return (unsigned long long)x >> 32 ? x / y : (long long)((unsigned)x / (unsigned)y);
}

// All tiles, items one after the other, go to the blocks in equal shares: block b has the tiles from b * tiles / blocks on, and
// no share is empty.  Such shares end inside items, and a piece of an item costs a block its start (queries, first keys) and its end
// (sums out to the workspace) beside its tiles, about as much as PIECE tiles.  So where that is less, blocks take whole items, from b *
// items / blocks on.  (144 items of 12 tiles for 148 blocks: in shares of 11.7 a call takes 49.6 us, whole 45.4; 25 of 64 tiles
// stay with shares.)
constexpr int PIECE = 3;
__device__ __forceinline__ void take_share(const Args& a, Plan& p, int items, long long tiles, int longest) {
  // (a warp; the rule in floats, the same ones in every block: every block waits for this)
  const int blocks = (int)min((long long)a.n_blocks, tiles), x = blockIdx.x + (threadIdx.x & 1);      // its share's start and end
  long long at = 0;
  if (tiles > 0 && (int)blockIdx.x < blocks) {
    const float each = __fdividef(1.0f, (float)blocks), share = ceilf((float)tiles * each), n = (float)longest;
    const float pieces = share < 2.0f ? 1.0f : 2.0f + floorf(__fdividef(share - 2.0f, n));             // (at most)
    // (a part of a round is 1 / 296 or more: what the reciprocal's rounding adds is none)
    if (ceilf((float)items * each - 1e-3f) * (n + PIECE) >= share + PIECE * pieces) {
      at = divide(tiles * x, blocks);
    } else {
      const int takers = min(blocks, items), item = (int)divide((long long)items * min(x, takers), takers);
      int g = 0;
      for (; p.items[g + 1] < item; g++) {
      }
      at = p.tiles[g] + (long long)(item - p.items[g]) * tiles_of_keys(a, p.keys[g]);
    }
  }
  if (threadIdx.x < 2) (threadIdx.x ? p.end : p.at) = at;
}

// Every thread of the block calls it.
__device__ __forceinline__ void make_plan(const Args& a, Plan& p) {
  for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
    const int length = prefix_length(a, g);
    int t0, t1;
    group_tokens(a, g, t0, t1);
    const int keys = t1 > t0 ? length : 0;
    p.t0[g] = t0;
    p.keys[g] = keys;
    p.rows[g] = (t1 - t0) * a.gq;
    p.items[g + 1] = keys > 0 ? a.Hkv * items_of(a, p.rows[g]) : 0;
  }
  __syncthreads();
  if (threadIdx.x < 32) {                 // sums over the groups before
    int items = 0, longest = 0;
    long long tiles = 0;
    for (int g0 = 0; g0 < a.G; g0 += 32) {
      const int g = g0 + threadIdx.x;
      int x = g < a.G ? p.items[g + 1] : 0;
      const int kt = x > 0 ? tiles_of_keys(a, p.keys[g]) : 0;
      long long y = (long long)x * kt;
      longest = max(longest, __reduce_max_sync(0xffffffffu, kt));
      for (int o = 1; o < 32 && o < a.G; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, x, o);
        const long long v = __shfl_up_sync(0xffffffffu, y, o);
        if ((int)threadIdx.x >= o) {
          x += u;
          y += v;
        }
      }
      if (g < a.G) {
        p.items[g + 1] = items + x;
        p.tiles[g + 1] = tiles + y;
      }
      const int last = min(31, a.G - 1 - g0);
      items += __shfl_sync(0xffffffffu, x, last);
      tiles += __shfl_sync(0xffffffffu, y, last);
    }
    if (threadIdx.x == 0) p.items[0] = 0, p.tiles[0] = 0;
    __syncwarp();
    take_share(a, p, items, tiles, longest);
  }
  __syncthreads();
}

// A block's piece of an item.
struct Segment {
  int item, hk, row0;                     // item counted over all groups; its key head and first row of that
  int t0, n_rows, keys;                   // the group's first token, rows a key head, prefix
  int shift;                              // log2 of an item's rows
  int tile, tiles;                        // tiles of keys: the first, how many
  long long at, end;                      // the piece's first tile and the end of the block's share, counted over all items
};
__device__ __forceinline__ Segment segment_at(const Args& a, const Plan& p, long long at, long long end) {
  Segment s;
  s.at = at;
  s.end = end;
  s.tiles = 0;
  if (at >= end) return s;
  int lo = 0, hi = a.G;                   // the last group whose tiles begin at or before `at` (it has some)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.tiles[mid] <= at) lo = mid; else hi = mid;
  }
  s.t0 = p.t0[lo];
  s.n_rows = p.rows[lo];
  s.keys = p.keys[lo];
  s.shift = item_shift(a, s.n_rows);
  const int kt = tiles_of_keys(a, s.keys), rt = items_of(a, s.n_rows);
  const int n = (int)divide(at - p.tiles[lo], kt);
  s.tile = (int)(at - p.tiles[lo] - (long long)n * kt);
  s.tiles = (int)min((long long)(kt - s.tile), end - at);
  s.item = p.items[lo] + n;
  s.hk = (unsigned)n / (unsigned)rt;
  s.row0 = (n - s.hk * rt) << s.shift;
  return s;
}
__device__ __forceinline__ Segment first_segment(const Args& a, const Plan& p) { return segment_at(a, p, p.at, p.end); }
__device__ __forceinline__ Segment next_segment(const Args& a, const Plan& p, const Segment& s) {
  return segment_at(a, p, s.at + s.tiles, s.end);
}

// Whose pages hold a segment's keys: the request of the group's first token (-1: there is no such one).
__device__ __forceinline__ int keeper(const Args& a, const Segment& s) { return s.tiles > 0 ? request_of(a, s.t0) : -1; }

// The piece that block b finds of item i lies in slot b + i of the workspace: along the shares either the block or the item
// goes up by one, so no two pieces meet in one slot.  Every piece has a slot, unless the groups' starts do not ascend and
// their tokens overlap.
__device__ __forceinline__ bool slot_ok(const Args& a, const Segment& s) {
  if (blockIdx.x + (long long)s.item < a.slots) return true;
  flag_index(a);
  return false;
}
// For the second launch: where a group's items begin (block 0 says it), and an item's first and last block (each says it
// of itself).
__device__ __forceinline__ void record_groups(const Args& a, const Plan& p) {
  if (blockIdx.x == 0)
    for (int g = threadIdx.x; g < a.G; g += blockDim.x) a.first_item[g] = p.keys[g] > 0 ? p.items[g] : -1;
}
__device__ __forceinline__ void record_item(const Args& a, const Segment& s) {
  if (s.item >= a.slots) return;
  if (s.tile == 0) a.item_blocks[s.item].x = blockIdx.x;
  if ((s.tile + s.tiles) << a.key_shift >= s.keys) a.item_blocks[s.item].y = blockIdx.x;
}
// The parts of row n of a group and key head.
struct Parts {
  int n;                                  // how many
  int halves;                             // of a slot's: two groups of warps of the tensor-core kernel share rows of few
  long long slot;                         // the first one's slot
  int row;                                // the row in a slot
};
__device__ __forceinline__ Parts parts_of(const Args& a, int g, int t0, int t1, int hk, int n) {
  const int rows = (t1 - t0) * a.gq, shift = item_shift(a, rows);
  const int first = a.first_item[g], item = first + hk * items_of(a, rows) + (n >> shift);
  Parts x = {0, a.tc && shift == 7 ? 2 : 1, 0, n & ((1 << shift) - 1)};
  if (first < 0 || item < 0 || item >= a.slots) return x;
  const int2 b = a.item_blocks[item];
  if (b.x < 0 || b.y < b.x || b.y >= a.n_blocks) return x;       // (a first launch that gave up)
  x.n = x.halves * (b.y - b.x + 1);
  x.slot = (long long)b.x + item;
  return x;
}
// The workspace's row of part j, or -1: there is no such slot.
__device__ __forceinline__ long long part_row(const Args& a, const Parts& x, int j) {
  const long long slot = x.slot + (x.halves == 2 ? j >> 1 : j);
  return slot < 0 || slot >= a.slots ? -1 : slot * a.slot_rows + (x.halves == 2 ? (j & 1) * 128 : 0) + x.row;
}

// 2^x by the special-function unit, 2 units in the last place (-inf gives 0)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two products and sums at a time, each rounded as one alone.
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(reinterpret_cast<unsigned long long&>(x)), "l"(reinterpret_cast<unsigned long long&>(y)),
      "l"(reinterpret_cast<unsigned long long&>(z)));
  return reinterpret_cast<float2&>(r);
}

// eight entries of a row; vec: it begins on 16 bytes
__device__ __forceinline__ void load8(const float* p, int vec, float (&v)[8]) {
  if (vec) {
    const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = p[i];
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int vec, float (&v)[8]) {
  if (vec) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __bfloat162float(p[i]);
  }
}
__device__ __forceinline__ void store8(float* p, int vec, const float (&v)[8]) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = v[i];
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, int vec, const float (&v)[8]) {
  if (vec) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = __float2bfloat16_rn(v[i]);
  }
}

// Lets a kernel take so much shared memory, once a device (a bit each; beyond 64 of them at every call).
template <typename... KArgs>
static int allow_shared(void (*kernel)(KArgs...), int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return 0;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return (int)e;
  done.fetch_or(bit, std::memory_order_release);
  return 0;
}
}  // namespace prefix
