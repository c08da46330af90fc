// Attention of a step's tokens over the paged cache where the requests of a group share a long prefix: its keys and values
// are read once for all tokens of the group, a token's own keys behind it for that token.
//   token t of group g, at position p:  out = sum_j softmax_j(scale q.k_j) v_j  over the keys j <= p; of these,
//   j < shared_g lie in the pages that the group's first request names, the others in those of the token's own request.
// A softmax over parts of the keys joins exactly: with (m, l, O) = (max, sum exp(s - m), sum exp(s - m) v) of each part and
// M the largest m, out = sum exp(m - M) O / sum exp(m - M) l.
//
// Two launches.  The first makes the prefixes' parts: an item is (group, key head, some rows), a row a (token, query head of
// that key head), so keys serve rows from shared memory; the tiles of keys of all items, one after the other, are dealt to
// the blocks in equal shares, so a block's share may end inside an item and every block has the same work, whatever the
// lengths.  What a block finds for (a piece of) an item goes to the workspace.  The second launch makes the tokens' own parts,
// waits for the first, and joins all parts of a (token, head).  Its blocks may begin once all of the first's have, but find
// room only where those leave it: on the tensor cores a block takes 61,440 of a multiprocessor's 65,536 registers.  So with
// items for some multiprocessors only the two run side by side (8 requests of 12 heads on 512 keys: all own keys are done before the
// first launch's last sums are out), and with items for all of them the second's blocks begin as the first's end (64 of 25 heads on
// 8,192 keys: from 16 us on, the first's last sums are out at 20, and 18 of 800 blocks are done with their own keys by then).
#include "attention_prefix.cuh"
#include "attention_prefix_own.cuh"
#include "attention_prefix_tc.cuh"

SGLC_DEFINE_ERROR_STRING()

namespace {
using namespace prefix;

// ---- prefixes, 32-bit arithmetic: float32, and bfloat16 heads of more than 128 ------------------------------------------------
// A tile of 16 R rows by 64 keys: a thread has R x 4 scores, fed by 16-byte reads of queries and keys from shared memory (for R
// = 4 eight for 64 multiply-adds), and R rows by D / 16 columns of the sums.  R = 4 where groups have many rows; R = 1 where
// they have up to 32: most of 64 rows would be empty, and what bounds such a call is the time of a few tiles (22 requests of
// 12 heads on two prefixes of 1,000: 28 us a call with 64 rows a tile, 19 with 16).
constexpr int GT = 256;                   // threads
constexpr int GK = GENERAL_KEYS;

template <typename T, int NC, int R>      // NC: blocks of 64 columns
__global__ void __launch_bounds__(GT)
prefix_general_kernel(const Args a) {
  constexpr int GR = 16 * R;
  extern __shared__ __align__(16) float sm[];
  const int D = a.D, DS = D + 4;          // (rows of queries and keys four words apart from the banks' period)
  float* sQ = sm;                         // [GR][DS]
  float* sK = sQ + GR * DS;               // [GK][DS]
  float* sV = sK + GK * DS;               // [GK][NC * 64]
  float* sP = sV + GK * NC * 64;          // [GR][GK + 4]
  __shared__ Plan plan;
  __shared__ int lim[GR], sPage[GK];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  pdl_wait();
  pdl_launch_dependents();                // (here and not before: the second launch reads what came before this one)
  make_plan(a, plan);
  record_groups(a, plan);
  const float c2 = a.scale * LOG2E;
  const int gq = a.gq;
  for (Segment s = first_segment(a, plan); s.tiles > 0; s = next_segment(a, plan, s)) {
    const int row0 = s.row0, rows = min(GR, s.n_rows - row0), req = keeper(a, s);
    __syncthreads();
    for (int x = tid; x < GR * (D / 8); x += GT) {
      const int row = x / (D / 8), d = x % (D / 8) * 8;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = 0.0f;
      if (row < rows) {
        const int n = row0 + row, t = s.t0 + n / gq, h = s.hk * gq + n % gq;
        load8(reinterpret_cast<const T*>(a.q) + (size_t)t * a.q_stride + (size_t)h * D + d, a.q_vec, v);
      }
#pragma unroll
      for (int i = 0; i < 8; i++) sQ[row * DS + d + i] = v[i];
    }
    if (tid < GR) lim[tid] = tid < rows ? visible(a, s.t0 + (row0 + tid) / gq, s.keys) : 0;
    float m[R], l[R], o[R][NC][4];
#pragma unroll
    for (int i = 0; i < R; i++) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int u = 0; u < 4; u++) o[i][c][u] = 0.0f;
    }
    // (a tile's pages are looked up a tile ahead)
    auto page_id = [&](int j) {
      const int key = (s.tile + j) * GK + tid;
      return tid < GK && j < s.tiles && key < s.keys ? page_of(a, req, key) : -1;
    };
    int page_next = page_id(0);
    for (int j = 0; j < s.tiles; j++) {
      const int key0 = (s.tile + j) * GK;
      __syncthreads();
      if (tid < GK) sPage[tid] = page_next;
      __syncthreads();
      page_next = page_id(j + 1);
#pragma unroll
      for (int x0 = 0; x0 < GK * NC * 8; x0 += 2 * GT) {       // (two pieces of keys and of values on their way a thread)
        float k[2][8], v[2][8];
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int x = x0 + u * GT + tid, row = x / (NC * 8), d = x % (NC * 8) * 8, page = sPage[row];
#pragma unroll
          for (int i = 0; i < 8; i++) k[u][i] = v[u][i] = 0.0f;
          if (d < D && page >= 0) {
            const size_t at = row_at(a, page, s.hk, key0 + row) + d;
            load8(reinterpret_cast<const T*>(a.cache) + at, 1, k[u]);
            load8(reinterpret_cast<const T*>(a.cache) + at + value_offset(a), 1, v[u]);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int x = x0 + u * GT + tid, row = x / (NC * 8), d = x % (NC * 8) * 8;
          if (d < D)
#pragma unroll
            for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4*>(&sK[row * DS + d + i]) = make_float4(k[u][i], k[u][i + 1], k[u][i + 2], k[u][i + 3]);
#pragma unroll
          for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4*>(&sV[row * NC * 64 + d + i]) = make_float4(v[u][i], v[u][i + 1], v[u][i + 2], v[u][i + 3]);
        }
      }
      __syncthreads();
      float x[R][4];
#pragma unroll
      for (int i = 0; i < R; i++)
#pragma unroll
        for (int u = 0; u < 4; u++) x[i][u] = 0.0f;
      for (int d = 0; d < D; d += 4) {
        float4 q4[R], k4[4];
#pragma unroll
        for (int i = 0; i < R; i++) q4[i] = *reinterpret_cast<const float4*>(&sQ[(ty * R + i) * DS + d]);
#pragma unroll
        for (int u = 0; u < 4; u++) k4[u] = *reinterpret_cast<const float4*>(&sK[(tx + 16 * u) * DS + d]);
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
          for (int u = 0; u < 4; u++) {
            x[i][u] = fmaf(q4[i].x, k4[u].x, x[i][u]);
            x[i][u] = fmaf(q4[i].y, k4[u].y, x[i][u]);
            x[i][u] = fmaf(q4[i].z, k4[u].z, x[i][u]);
            x[i][u] = fmaf(q4[i].w, k4[u].w, x[i][u]);
          }
      }
#pragma unroll
      for (int i = 0; i < R; i++) {
        const int row = ty * R + i, n = lim[row] - key0;      // keys of this tile that the row sees
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; u++) {
          if (tx + 16 * u >= n) x[i][u] = -INFINITY;
          mx = fmaxf(mx, x[i][u]);
        }
#pragma unroll
        for (int w = 1; w < 16; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        mx *= c2;
        if (mx > m[i]) {
          const float f = exp2f(m[i] - mx);                   // (0 where nothing was seen before)
          m[i] = mx;
          l[i] *= f;
#pragma unroll
          for (int c = 0; c < NC; c++)
#pragma unroll
            for (int u = 0; u < 4; u++) o[i][c][u] *= f;
        }
        const float ref = m[i] == -INFINITY ? 0.0f : m[i];
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const float p = exp2f(fmaf(x[i][u], c2, -ref));
          l[i] += p;
          sP[row * (GK + 4) + tx + 16 * u] = p;
        }
      }
      __syncwarp();                       // (a row's weights are made and used by the same half of a warp)
#pragma unroll 2
      for (int key = 0; key < GK; key += 4) {
        float4 p4[R];
#pragma unroll
        for (int i = 0; i < R; i++) p4[i] = *reinterpret_cast<const float4*>(&sP[(ty * R + i) * (GK + 4) + key]);
#pragma unroll
        for (int c = 0; c < NC; c++) {
          float4 v4[4];
#pragma unroll
          for (int u = 0; u < 4; u++) v4[u] = *reinterpret_cast<const float4*>(&sV[(key + u) * NC * 64 + c * 64 + tx * 4]);
#pragma unroll
          for (int i = 0; i < R; i++) {
            const float w[4] = {p4[i].x, p4[i].y, p4[i].z, p4[i].w};
#pragma unroll
            for (int u = 0; u < 4; u++) {
              o[i][c][0] = fmaf(w[u], v4[u].x, o[i][c][0]);
              o[i][c][1] = fmaf(w[u], v4[u].y, o[i][c][1]);
              o[i][c][2] = fmaf(w[u], v4[u].z, o[i][c][2]);
              o[i][c][3] = fmaf(w[u], v4[u].w, o[i][c][3]);
            }
          }
        }
      }
    }
    if (tid == 0) record_item(a, s);
    const size_t slot = (size_t)(blockIdx.x + s.item) * a.slot_rows;
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int row = ty * R + i;
#pragma unroll
      for (int w = 1; w < 16; w <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
      if (row < rows && slot_ok(a, s)) {
        if (tx == 0) a.part_ml[slot + row] = make_float2(m[i], l[i]);
#pragma unroll
        for (int c = 0; c < NC; c++)
          if (c * 64 + tx * 4 < D)
            *reinterpret_cast<float4*>(a.part_o + (slot + row) * D + c * 64 + tx * 4) =
                make_float4(o[i][c][0], o[i][c][1], o[i][c][2], o[i][c][3]);
      }
    }
  }
}

// ---- a token's own keys, and the parts joined ------------------------------------------------------------------------------
// An item is HC query heads of one key head of one token.  A warp, or four, or a cluster of blocks of four take an item: a
// row of keys lies over LW lanes of a warp, eight entries a lane, and each such part of a warp (a walker) walks keys of its
// own with a running maximum of its own, then, once the first launch is done, parts of the prefix in the same way.  Walkers
// meet by shuffles, warps in shared memory, blocks through the cluster's.  What bounds it: the keys' and the parts' way from
// memory, and for few items the chain token -> request -> page -> key; so a lane of the warp holds a page's id each, and the
// keys of a round are asked for together.  (64 requests of 25 heads of 64 with up to 300 keys: 26 us alone, 62 MB.)
constexpr int OT = 128;

constexpr int OWN_ONE = 16, OWN_TWO = 4;    // items a multiprocessor from which an item has one warp, two

// Eight entries as they lie in memory.
template <typename T> struct Raw;
template <> struct Raw<__nv_bfloat16> {
  uint4 x;
  __device__ __forceinline__ void take(const __nv_bfloat16* p) { x = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { x = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float2 (&v)[4]) const {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};
template <> struct Raw<float> {
  float4 x, y;
  __device__ __forceinline__ void take(const float* p) {
    x = *reinterpret_cast<const float4*>(p);
    y = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void zero() { x = y = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  __device__ __forceinline__ void get(float2 (&v)[4]) const {
    v[0] = make_float2(x.x, x.y);
    v[1] = make_float2(x.z, x.w);
    v[2] = make_float2(y.x, y.y);
    v[3] = make_float2(y.z, y.w);
  }
};

// A part of a softmax: maximum (times log2 e), sum of weights, and eight columns of the weighted sum.
struct State {
  float m, l;
  float2 o[4];
  __device__ __forceinline__ void join(float m2, float l2, const float2 (&o2)[4]) {
    const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.0f : top, f = ex2(m - ref), f2 = ex2(m2 - ref);
    m = top;
    l = l * f + l2 * f2;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = make_float2(o[i].x * f + o2[i].x * f2, o[i].y * f + o2[i].y * f2);
  }
};

// Keys of a walker a round: as many scores (keys x heads) as the walker has lanes, within what the registers hold.
__host__ __device__ constexpr int round_keys(int size, int HC, int LW) {
  const int most = 4 / (size == 4 ? 2 : 1), fit = LW / HC;
  return fit < most ? fit : most;
}

// LW: lanes of a row.  WARPS: of an item; a block has four.
template <typename T, int HC, int LW, int WARPS>
__global__ void __launch_bounds__(OT, HC == 1 ? 6 : HC == 2 ? 4 : 3)
prefix_own_kernel(const Args a) {
  extern __shared__ __align__(16) float sm[];          // [4 warps][HC][D + 2], then [HC][warps of an item]: for items of several
  constexpr int per_warp = 32 / LW, ITEMS = 4 / WARPS;
  const int D = a.D, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = a.gq;
  const int of_warp = lane / LW, sub = lane % LW;
  const int share = blockIdx.z, shares = gridDim.z;
  if (shares > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_launch_dependents();
  const int t = blockIdx.x * ITEMS + warp / WARPS, h0 = blockIdx.y * HC, hk = h0 / gq;
  // the token's group: the last one that begins at or before it
  int g = -1;
  for (int x = 0; x < a.G; x += 32) g += __popc(__ballot_sync(0xffffffffu, x + lane < a.G && a.group_start[x + lane] <= t));
  int t0 = 0, t1 = 0;
  if (g >= 0) group_tokens(a, g, t0, t1);
  const bool inside = g >= 0 && t >= t0 && t < t1;
  // (starts that do not ascend, with the token behind this group's end and before the last one's)
  if (g >= 0 && !inside && t < min(a.group_start[a.G], a.T)) flag_index(a);
  int keys = inside ? prefix_length(a, g) : 0;           // of the prefix, by parts; own keys lie behind them
  const int walker = (share * WARPS + warp % WARPS) * per_warp + of_warp;
  const int walkers = WARPS * shares * per_warp, d = sub * 8;
  const bool cols = d < D;
  State st[HC];
#pragma unroll
  for (int h = 0; h < HC; h++) {
    st[h].m = -INFINITY;
    st[h].l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) st[h].o[i] = make_float2(0.0f, 0.0f);
  }
  if (inside) {
    const float c2 = a.scale * LOG2E;
    const int pos = a.positions[t];
    int req = request_of(a, t);
    if (pos > a.last_position) flag_index(a);
    if (!sees_all(pos, keys)) {                        // inside the prefix, whose pages the group's first request names
      keys = 0;
      req = request_of(a, t0);
    }
    const int end = req < 0 ? keys : min(pos, a.last_position) + 1;          // own keys: keys .. end - 1
    float2 q[HC][4];
#pragma unroll
    for (int h = 0; h < HC; h++) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = 0.0f;
      if (cols) load8(reinterpret_cast<const T*>(a.q) + (size_t)t * a.q_stride + (size_t)(h0 + h) * D + d, a.q_vec, x);
#pragma unroll
      for (int i = 0; i < 4; i++) q[h][i] = make_float2(x[2 * i], x[2 * i + 1]);
    }
    // A round: U keys' scores with HC heads are NV sums over the walker's lanes.  They are summed by halves: at each of the
    // first levels a lane keeps one half of the sums and gives its part of the others away, so that NV sums take
    // NV - 1 shuffles and a lane has one at the end, number sub / COPIES; it makes that one's weight, and the weights go round.
    constexpr int U = round_keys(sizeof(T), HC, LW), NV = U * HC, COPIES = LW / NV;
    const int my_u = sub / COPIES / HC, base = lane & ~(LW - 1);
    float m = -INFINITY, l = 0.0f;                     // of this lane's head; weights of its place among the sums only
    const size_t v_at = value_offset(a);
    // 32 pages at a time, a lane an id
    for (int block0 = block_in(a, keys); (long long)block0 * a.page_size < end; block0 += 32) {
      const long long stop = min((long long)end, (long long)(block0 + 32) * a.page_size);
      const int first = max(keys, block0 * a.page_size), last = (int)stop;
      const int id = (long long)(block0 + lane) * a.page_size < last ? page_of(a, req, (block0 + lane) * a.page_size) : -1;
      for (int key0 = first + (walker - of_warp) * U; key0 < last; key0 += walkers * U) {
        // (the bounds are the warp's: its lanes take the shuffles together)
        Raw<T> k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int key = key0 + u * per_warp + of_warp, block = block_in(a, key);
          const int page = __shfl_sync(0xffffffffu, id, (block - block0) & 31);
          k[u].zero();
          v[u].zero();
          if (key < last && page >= 0 && cols) {
            const T* x = reinterpret_cast<const T*>(a.cache) + (((size_t)page * 2 * a.Hkv + hk) * a.page_size + (key - block * a.page_size)) * D + d;
            k[u].take(x);
            v[u].take(x + v_at);
          }
        }
        float s[NV];
#pragma unroll
        for (int u = 0; u < U; u++) {
          float2 x[4];
          k[u].get(x);
#pragma unroll
          for (int h = 0; h < HC; h++) {
            float2 e = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 4; i++) e = fma2(q[h][i], x[i], e);
            s[u * HC + h] = e.x + e.y;
          }
        }
#pragma unroll
        for (int w = LW / 2, n = NV; w > 0; w >>= 1) {
          const bool up = sub & w;
          if (n > 1) {
            n >>= 1;
#pragma unroll
            for (int i = 0; i < NV / 2; i++)
              if (i < n) {
                const float give = up ? s[i] : s[n + i], keep = up ? s[n + i] : s[i];
                s[i] = keep + __shfl_xor_sync(0xffffffffu, give, w);
              }
          } else {
            s[0] += __shfl_xor_sync(0xffffffffu, s[0], w);
          }
        }
        float score = key0 + my_u * per_warp + of_warp < last ? s[0] * c2 : -INFINITY, top = score;
#pragma unroll
        for (int w = LW / 2; w >= HC * COPIES; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        top = fmaxf(top, m);
        const float ref = top == -INFINITY ? 0.0f : top;
        if (__any_sync(0xffffffffu, top > m)) {
          const float f = ex2(m - ref);                // (0 where nothing was seen before)
          l *= f;
          m = top;
#pragma unroll
          for (int h = 0; h < HC; h++) {
            const float fh = __shfl_sync(0xffffffffu, f, base + h * COPIES);
#pragma unroll
            for (int i = 0; i < 4; i++) st[h].o[i] = make_float2(st[h].o[i].x * fh, st[h].o[i].y * fh);
          }
        }
        const float p = ex2(score - ref);
        l += p;
#pragma unroll
        for (int u = 0; u < U; u++) {
          float2 x[4];
          v[u].get(x);
#pragma unroll
          for (int h = 0; h < HC; h++) {
            const float ph = __shfl_sync(0xffffffffu, p, base + (u * HC + h) * COPIES);
#pragma unroll
            for (int i = 0; i < 4; i++) st[h].o[i] = fma2(make_float2(ph, ph), x[i], st[h].o[i]);
          }
        }
      }
    }
#pragma unroll
    for (int w = LW / 2; w >= HC * COPIES; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
#pragma unroll
    for (int h = 0; h < HC; h++) {
      st[h].m = __shfl_sync(0xffffffffu, m, base + h * COPIES);
      st[h].l = __shfl_sync(0xffffffffu, l, base + h * COPIES);
    }
  }
  pdl_wait();                                          // the prefixes' parts are there
  if (keys > 0) {
    const Parts ps = parts_of(a, g, t0, t1, hk, (t - t0) * gq + h0 - hk * gq);
    for (int j = walker; j < ps.n; j += walkers) {
      const long long at = part_row(a, ps, j);
      if (at < 0) continue;
      float2 ml[HC], o[HC][4];
#pragma unroll
      for (int h = 0; h < HC; h++) {
        Raw<float> x;
        x.zero();
        ml[h] = a.part_ml[at + h];
        if (cols) x.take(a.part_o + (at + h) * D + d);
        x.get(o[h]);
      }
#pragma unroll
      for (int h = 0; h < HC; h++)
        if (ml[h].y != 0.0f) st[h].join(ml[h].x, ml[h].y, o[h]);       // (0: nothing was seen and no sums were written; NaN is not 0)
    }
  }
  // the warp's walkers
#pragma unroll
  for (int h = 0; h < HC; h++)
#pragma unroll
    for (int w = 16; w >= LW; w >>= 1) {
      float2 o[4];
      const float m = __shfl_xor_sync(0xffffffffu, st[h].m, w), l = __shfl_xor_sync(0xffffffffu, st[h].l, w);
#pragma unroll
      for (int i = 0; i < 4; i++)
        o[i] = make_float2(__shfl_xor_sync(0xffffffffu, st[h].o[i].x, w), __shfl_xor_sync(0xffffffffu, st[h].o[i].y, w));
      st[h].join(m, l, o);
    }
  if constexpr (WARPS == 1) {
    if (inside && of_warp == 0 && cols) {
#pragma unroll
      for (int h = 0; h < HC; h++) {
        const float f = st[h].l == 0.0f ? 0.0f : 1.0f / st[h].l;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = st[h].l == 0.0f ? 0.0f : (i & 1 ? st[h].o[i / 2].y : st[h].o[i / 2].x) * f;
        store8(reinterpret_cast<T*>(a.out) + (size_t)t * a.o_stride + (size_t)(h0 + h) * D + d, a.o_vec, o);
      }
    }
  } else {
    // the item's warps, and the cluster's blocks
    const int one = HC * (D + 2), parts = WARPS * shares, warp0 = warp / WARPS * WARPS, mine = threadIdx.x % (WARPS * 32);
    if (of_warp == 0) {
#pragma unroll
      for (int h = 0; h < HC; h++) {
        float* to = sm + warp * one + h * (D + 2);
        if (cols)
#pragma unroll
          for (int i = 0; i < 8; i++) to[d + i] = i & 1 ? st[h].o[i / 2].y : st[h].o[i / 2].x;
        if (sub == 0) {
          to[D] = st[h].m;
          to[D + 1] = st[h].l;
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
    float* factor = sm + 4 * one + warp0 * HC * shares;
    if (share == 0 && mine < HC) {
      const int at = mine * (D + 2) + D;
      float M = -INFINITY, total = 0.0f;
      for (int z = 0; z < parts; z++) M = fmaxf(M, other(z, at));
      const float ref = M == -INFINITY ? 0.0f : M;
      for (int z = 0; z < parts; z++) {
        const float f = ex2(other(z, at) - ref);
        factor[mine * parts + z] = f;
        total = fmaf(f, other(z, at + 1), total);
      }
      const float f = total == 0.0f ? 0.0f : 1.0f / total;
      for (int z = 0; z < parts; z++) factor[mine * parts + z] *= f;
    }
    __syncthreads();
    if (share == 0 && inside)
      for (int x = mine; x < HC * D; x += WARPS * 32) {
        const int h = x / D, c = x - h * D;
        float sum = 0.0f;
        for (int z = 0; z < parts; z++) sum = fmaf(factor[h * parts + z], other(z, h * (D + 2) + c), sum);
        reinterpret_cast<T*>(a.out)[(size_t)t * a.o_stride + (size_t)(h0 + h) * D + c] = from_f32<T>(sum);
      }
    if (shares > 1) {                                  // (block 0 has read the others' shared memory)
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
  }
}

template <typename T, int NC, int R>
int launch_general(const Args& a, cudaStream_t stream) {
  constexpr int GR = 16 * R;
  const size_t smem = (size_t)((GR + GK) * (a.D + 4) + GK * NC * 64 + GR * (GK + 4)) * 4;
  static std::atomic<unsigned long long> done{0};
  const int code = allow_shared(prefix_general_kernel<T, NC, R>, ((GR + GK) * (NC * 64 + 4) + GK * NC * 64 + GR * (GK + 4)) * 4, done);
  if (code) return code;
  return sglc_launch(prefix_general_kernel<T, NC, R>, dim3(a.n_blocks), dim3(GT), smem, stream, 1, true, a);
}
template <typename T, int NC>
int rows_general(const Args& a, cudaStream_t stream) {
  return a.row_shift == 4 ? launch_general<T, NC, 1>(a, stream) : launch_general<T, NC, 4>(a, stream);
}
template <typename T>
int run_general(const Args& a, cudaStream_t stream) {
  if constexpr (sizeof(T) == 4) {                      // (bfloat16 heads of up to 128: the tensor cores')
    if (a.D <= 64) return rows_general<T, 1>(a, stream);
    if (a.D <= 128) return rows_general<T, 2>(a, stream);
  }
  return a.D <= 192 ? rows_general<T, 3>(a, stream) : rows_general<T, 4>(a, stream);
}

template <typename T, int HC, int LW, int WARPS>
int launch_own(const Args& a, int shares, cudaStream_t stream) {
  const size_t smem = WARPS == 1 ? 0 : (size_t)(4 * HC * (a.D + 2) + 4 * HC * shares) * 4;
  return sglc_launch(prefix_own_kernel<T, HC, LW, WARPS>, dim3((a.T * WARPS + 3) / 4, a.H / HC, shares), dim3(OT), smem, stream, shares,
                     true, a);
}
template <typename T, int HC, int LW>
int warps_own(const Args& a, int max_own, cudaStream_t stream) {
  // A warp an item where the items fill the multiprocessors' warps, else two, else four, and blocks of a cluster while
  // there are fewer than four a multiprocessor and 64 keys or more are left for each.  (By the items' number: the host knows no
  // lengths.  Where one request has many more keys of its own than the others, its items' warps walk them alone: 256 requests of 25
  // heads of 64 on 1,024 keys with 150 of their own take 73 us, with one of them at 3,000 259 us, at 30,000 2,120.)
  const long long items = (long long)a.T * (a.H / HC);
  if (items >= OWN_ONE * a.sms) return launch_own<T, HC, LW, 1>(a, 1, stream);
  if (items >= OWN_TWO * a.sms) return launch_own<T, HC, LW, 2>(a, 1, stream);
  int shares = 1;
  while (shares < 8 && items * shares * 2 <= 4LL * a.sms && max_own >= 64 * shares * 2) shares *= 2;
  return launch_own<T, HC, LW, 4>(a, shares, stream);
}
template <typename T, int LW>
int choose_own(const Args& a, int max_own, cudaStream_t stream) {
  const int gq = a.H / a.Hkv;
  if constexpr (LW >= 4)
    if (gq % 4 == 0) return warps_own<T, 4, LW>(a, max_own, stream);
  if constexpr (LW >= 2)
    if (gq % 2 == 0) return warps_own<T, 2, LW>(a, max_own, stream);
  return warps_own<T, 1, LW>(a, max_own, stream);
}
template <typename T>
int run_own(const Args& a, int max_own, cudaStream_t stream) {
  switch (a.lanes) {
    case 1: return choose_own<T, 1>(a, max_own, stream);
    case 2: return choose_own<T, 2>(a, max_own, stream);
    case 4: return choose_own<T, 4>(a, max_own, stream);
    case 8: return choose_own<T, 8>(a, max_own, stream);
    case 16: return choose_own<T, 16>(a, max_own, stream);
    default: return choose_own<T, 32>(a, max_own, stream);
  }
}

int multiprocessors() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n;
}

// The launch's blocks, rows an item and slots of the workspace, from sizes alone.
bool lay_out(Args* a, int dtype) {
  a->sms = multiprocessors();
  if (a->sms <= 0) return false;
  a->gq = a->H / a->Hkv;
  a->tc = dtype == SGLC_BF16 && a->D <= 128;
  a->n_blocks = a->tc ? a->sms : 2 * a->sms;
  a->row_shift = (long long)a->T * a->gq <= 32LL * a->G ? 4 : 6;             // (rows of a group's key head, on average)
  a->slot_rows = a->tc ? TC_SLOT : 1 << a->row_shift;
  a->key_shift = a->tc ? 7 : 6;
  static_assert(TC_KEYS == 128 && GENERAL_KEYS == 64, "as the shift says");
  const long long rows = (long long)a->T * a->gq;
  a->slots = a->n_blocks + a->Hkv * (rows / a->slot_rows + a->G);      // (items of 128 rows are the only ones of their group)
  a->lanes = 1;
  while (a->lanes * 8 < a->D) a->lanes *= 2;
  return true;
}
// floats of workspace: the parts' sums, their (maximum, sum of weights), the groups' first items, the items' blocks
long long words(const Args& a) { return a.slots * a.slot_rows * (a.D + 2) + (a.G + 1) / 2 * 2 + 2 * a.slots; }
bool sizes_ok(int T, int R, int G, int H, int Hkv, int D) {
  return T >= 0 && R >= 0 && G >= 0 && H > 0 && H <= 65535 && Hkv > 0 && H % Hkv == 0 && D > 0;
}
}  // namespace

// Floats of workspace that sglc_attention_prefix needs, or -1: the sizes are not taken.
SGLC_API long long sglc_attention_prefix_workspace(int T, int G, int H, int Hkv, int D, int dtype) {
  if (!sizes_ok(T, 0, G, H, Hkv, D) || D % 8 || D > 256 || G > MAX_GROUPS) return -1;
  Args a = {};
  a.T = T; a.G = G; a.H = H; a.Hkv = Hkv; a.D = D;
  if (!lay_out(&a, dtype)) return -1;
  return words(a);
}

// q, out [T][stride] and cache, one layer's pages [n_pages][2][Hkv][page_size][D], of one dtype; table [R][bt_stride],
// bt_width entries a row; token_req, positions [T]; group_start [G + 1]: the first token of each group, ascending;
// shared_len [G].  Tokens before group_start[0] and from group_start[G] on are left out.  max_own: about how many keys of
// its own a token has (it only sizes the launch).  workspace: floats, 16-byte aligned.  err: gets 4 where an index is out of
// range (a request, a page, a position beyond the table): what it names is not read.
SGLC_API int sglc_attention_prefix(const void* q, long long q_stride, const void* cache, const int* table, long long bt_stride,
                                   int bt_width, int R, const int* token_req, const int* positions, const int* group_start,
                                   const int* shared_len, int G, void* out, long long o_stride, int T, int H, int Hkv, int D,
                                   int page_size, int n_pages, float scale, int max_own, float* workspace, long long ws_floats,
                                   int dtype, int* err, cudaStream_t stream) {
  if (!sizes_ok(T, R, G, H, Hkv, D) || page_size <= 0 || n_pages < 0 || bt_width < 0 || !(scale > 0.0f) ||
      (dtype != SGLC_F32 && dtype != SGLC_BF16))
    return SGLC_ERR_ARGUMENT;
  // (items of all groups are counted in 32 bits, also where starts do not ascend and groups overlap)
  if (D % 8 || D > 256 || G > MAX_GROUPS || (long long)T * H > 0x20000000LL || n_pages == 0 || ((uintptr_t)cache & 15))
    return SGLC_ERR_UNSUPPORTED;
  if (T == 0 || G == 0) return SGLC_OK;
  Args a = {};
  a.q = q; a.q_stride = q_stride; a.cache = cache;
  a.q_vec = ((uintptr_t)q & 15) == 0 && q_stride * (dtype == SGLC_F32 ? 4 : 2) % 16 == 0;
  a.table = table; a.bt_stride = bt_stride; a.R = R;
  a.token_req = token_req; a.positions = positions; a.group_start = group_start; a.shared_len = shared_len;
  a.out = out; a.o_stride = o_stride;
  a.T = T; a.G = G; a.H = H; a.Hkv = Hkv; a.D = D; a.page_size = page_size; a.n_pages = n_pages; a.scale = scale;
  const long long room = (long long)bt_width * page_size;
  a.page_shift = page_size & (page_size - 1) ? -1 : __builtin_ctz(page_size);
  a.last_position = (int)(room > 0x7fff0000LL ? 0x7fff0000LL : room) - 1;        // (so that a step of keys further is a number still)
  a.err = err;
  if (!lay_out(&a, dtype)) return SGLC_ERR_ARGUMENT;
  if (words(a) > ws_floats || ((uintptr_t)workspace & 15)) return SGLC_ERR_ARGUMENT;
  a.part_o = workspace;
  a.part_ml = reinterpret_cast<float2*>(workspace + a.slots * a.slot_rows * D);
  a.first_item = reinterpret_cast<int*>(a.part_ml + a.slots * a.slot_rows);
  a.item_blocks = reinterpret_cast<int2*>(a.first_item + (G + 1) / 2 * 2);
  a.o_vec = ((uintptr_t)out & 15) == 0 && o_stride * (dtype == SGLC_F32 ? 4 : 2) % 16 == 0;
  const int code = a.tc ? (D <= 64 ? launch_tc<64, 4>(a, stream) : launch_tc<128, 2>(a, stream))
                        : dtype == SGLC_F32 ? run_general<float>(a, stream) : run_general<__nv_bfloat16>(a, stream);
  if (code) return code;
  if (join_pays(a)) return D == 64 ? run_join<64>(a, max_own, stream) : run_join<128>(a, max_own, stream);
  return dtype == SGLC_F32 ? run_own<float>(a, max_own, stream) : run_own<__nv_bfloat16>(a, max_own, stream);
}
