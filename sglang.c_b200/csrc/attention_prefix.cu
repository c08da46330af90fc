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
// which it does while the first still runs, waits for that, and joins all parts of a (token, head).
#include "attention_prefix.cuh"
#include "attention_prefix_tc.cuh"

SGLC_DEFINE_ERROR_STRING()

namespace {
using namespace prefix;

// ---- prefixes, 32-bit arithmetic (any head size that is a multiple of 8, up to 256) -----------------------------------------
// A tile of 64 rows by 64 keys: a thread has 4 x 4 scores, fed by 16-byte reads of queries and keys from shared memory (8 for
// 64 multiply-adds), and 4 rows by D / 16 columns of the sums.
constexpr int GT = 256;                   // threads
constexpr int GR = GENERAL_ROWS, GK = GENERAL_KEYS;

template <typename T, int NC>             // NC: blocks of 64 columns
__global__ void __launch_bounds__(GT)
prefix_general_kernel(const Args a) {
  extern __shared__ __align__(16) float sm[];
  const int D = a.D, DS = D + 4;          // (rows of queries and keys four words apart from the banks' period)
  float* sQ = sm;                         // [GR][DS]
  float* sK = sQ + GR * DS;               // [GK][DS]
  float* sV = sK + GK * DS;               // [GK][NC * 64]
  float* sP = sV + GK * NC * 64;          // [GR][GK + 4]
  __shared__ Plan plan;
  __shared__ int lim[GR];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  pdl_wait();
  pdl_launch_dependents();                // (here and not before: the second launch reads what came before this one)
  make_plan(a, plan);
  record_groups(a, plan);
  const float c2 = a.scale * LOG2E;
  const int gq = a.H / a.Hkv;
  for (Segment s = first_segment(a, plan); s.tiles > 0; s = next_segment(a, plan, s)) {
    const int row0 = s.row_tile * GR, rows = min(GR, s.n_rows - row0);
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
    float m[4], l[4], o[4][NC][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
#pragma unroll
      for (int c = 0; c < NC; c++)
#pragma unroll
        for (int u = 0; u < 4; u++) o[i][c][u] = 0.0f;
    }
    for (int j = 0; j < s.tiles; j++) {
      const int key0 = (s.tile + j) * GK;
      __syncthreads();
      for (int x = tid; x < GK * NC * 8; x += GT) {
        const int row = x / (NC * 8), d = x % (NC * 8) * 8, key = key0 + row;
        float k[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) k[i] = v[i] = 0.0f;
        if (d < D && key < s.keys) {
          const int page = page_of(a, s.req, key);
          if (page >= 0) {
            const size_t at = row_at(a, page, s.hk, key) + d;
            load8(reinterpret_cast<const T*>(a.cache) + at, 1, k);
            load8(reinterpret_cast<const T*>(a.cache) + at + value_offset(a), 1, v);
          }
        }
        if (d < D)
#pragma unroll
          for (int i = 0; i < 8; i++) sK[row * DS + d + i] = k[i];
#pragma unroll
        for (int i = 0; i < 8; i++) sV[row * NC * 64 + d + i] = v[i];
      }
      __syncthreads();
      float x[4][4];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int u = 0; u < 4; u++) x[i][u] = 0.0f;
      for (int d = 0; d < D; d += 4) {
        float4 q4[4], k4[4];
#pragma unroll
        for (int i = 0; i < 4; i++) q4[i] = *reinterpret_cast<const float4*>(&sQ[(ty * 4 + i) * DS + d]);
#pragma unroll
        for (int u = 0; u < 4; u++) k4[u] = *reinterpret_cast<const float4*>(&sK[(tx + 16 * u) * DS + d]);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int u = 0; u < 4; u++) {
            x[i][u] = fmaf(q4[i].x, k4[u].x, x[i][u]);
            x[i][u] = fmaf(q4[i].y, k4[u].y, x[i][u]);
            x[i][u] = fmaf(q4[i].z, k4[u].z, x[i][u]);
            x[i][u] = fmaf(q4[i].w, k4[u].w, x[i][u]);
          }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int row = ty * 4 + i, n = lim[row] - key0;      // keys of this tile that the row sees
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
        float4 p4[4];
#pragma unroll
        for (int i = 0; i < 4; i++) p4[i] = *reinterpret_cast<const float4*>(&sP[(ty * 4 + i) * (GK + 4) + key]);
#pragma unroll
        for (int c = 0; c < NC; c++) {
          float4 v4[4];
#pragma unroll
          for (int u = 0; u < 4; u++) v4[u] = *reinterpret_cast<const float4*>(&sV[(key + u) * NC * 64 + c * 64 + tx * 4]);
#pragma unroll
          for (int i = 0; i < 4; i++) {
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
    for (int i = 0; i < 4; i++) {
      const int row = ty * 4 + i;
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
// keys of a round are asked for together.
constexpr int OT = 128;

// Eight entries as they lie in memory.
template <typename T> struct Raw;
template <> struct Raw<__nv_bfloat16> {
  uint4 x;
  __device__ __forceinline__ void take(const __nv_bfloat16* p) { x = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { x = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Raw<float> {
  float4 x, y;
  __device__ __forceinline__ void take(const float* p) {
    x = *reinterpret_cast<const float4*>(p);
    y = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void zero() { x = y = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  }
};

// A part of a softmax: maximum (times log2 e), sum of weights, and eight columns of the weighted sum.
struct State {
  float m, l, o[8];
  __device__ __forceinline__ void join(float m2, float l2, const float (&o2)[8]) {
    const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.0f : top, f = exp2f(m - ref), f2 = exp2f(m2 - ref);
    m = top;
    l = l * f + l2 * f2;
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = o[i] * f + o2[i] * f2;
  }
};

// LW: lanes of a row, or 0: a.lanes.  warps: 1 or 4 of an item.
template <typename T, int HC, int LW>
__global__ void __launch_bounds__(OT)
prefix_own_kernel(const Args a, int warps) {
  extern __shared__ __align__(16) float sm[];          // [4 warps][HC][D + 2], for items of four warps
  const int D = a.D, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gq = a.H / a.Hkv;
  const int width = LW ? LW : a.lanes, of_warp = lane / width, sub = lane % width, per_warp = 32 / width;
  const int share = blockIdx.z, shares = gridDim.z;
  if (shares > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_launch_dependents();
  const int chunks = a.H / HC;
  const long long item = warps == 1 ? (long long)blockIdx.x * 4 + warp : blockIdx.x;
  const bool real = item < (long long)a.T * chunks;
  const int t = real ? (int)(item / chunks) : 0, h0 = (int)(item - (long long)t * chunks) * HC, hk = real ? h0 / gq : 0;
  // the token's group: the last one that begins at or before it
  int g = -1;
  for (int x = 0; real && x < a.G; x += 32) g += __popc(__ballot_sync(0xffffffffu, x + lane < a.G && a.group_start[x + lane] <= t));
  int t0 = 0, t1 = 0;
  if (g >= 0) group_tokens(a, g, t0, t1);
  const bool inside = g >= 0 && t >= t0 && t < t1;
  // (starts that do not ascend, with the token behind this group's end and before the last one's)
  if (g >= 0 && !inside && t < a.group_start[a.G]) flag_index(a);
  const int keys = inside ? prefix_keys(a, g, t0, t1) : 0, walker = warps == 1 ? of_warp : (share * 4 + warp) * per_warp + of_warp;
  const int walkers = (warps == 1 ? 1 : 4 * shares) * per_warp, d = sub * 8;
  const bool cols = d < D;
  State st[HC];
#pragma unroll
  for (int h = 0; h < HC; h++) {
    st[h].m = -INFINITY;
    st[h].l = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) st[h].o[i] = 0.0f;
  }
  if (inside) {
    const float c2 = a.scale * LOG2E;
    const int pos = a.positions[t], req = request_of(a, t);
    if (pos > a.last_position) flag_index(a);
    const int end = req < 0 ? keys : min(pos, a.last_position) + 1;          // own keys: keys .. end - 1
    float q[HC][8];
#pragma unroll
    for (int h = 0; h < HC; h++) {
#pragma unroll
      for (int i = 0; i < 8; i++) q[h][i] = 0.0f;
      if (cols) load8(reinterpret_cast<const T*>(a.q) + (size_t)t * a.q_stride + (size_t)(h0 + h) * D + d, a.q_vec, q[h]);
    }
    constexpr int U = sizeof(T) == 2 && HC < 4 ? 4 : 2;          // keys of a walker a round
    const size_t v_at = value_offset(a);
    // 32 pages at a time, a lane an id
    for (int block0 = (unsigned)keys / (unsigned)a.page_size; (long long)block0 * a.page_size < end; block0 += 32) {
      const long long stop = min((long long)end, (long long)(block0 + 32) * a.page_size);
      const int first = max(keys, block0 * a.page_size), last = (int)stop;
      const int id = (long long)(block0 + lane) * a.page_size < last ? page_of(a, req, (block0 + lane) * a.page_size) : -1;
      for (int key0 = first + (walker - of_warp) * U; key0 < last; key0 += walkers * U) {
        // (the bounds are the warp's: its lanes take the shuffles together)
        Raw<T> k[U], v[U];
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int key = key0 + u * per_warp + of_warp;
          const int page = __shfl_sync(0xffffffffu, id, ((unsigned)key / (unsigned)a.page_size - block0) & 31);
          in[u] = key < last;
          k[u].zero();
          v[u].zero();
          if (in[u] && page >= 0 && cols) {
            const T* x = reinterpret_cast<const T*>(a.cache) + row_at(a, page, hk, key) + d;
            k[u].take(x);
            v[u].take(x + v_at);
          }
        }
#pragma unroll
        for (int h = 0; h < HC; h++) {
          float s[U], mx = -INFINITY;
#pragma unroll
          for (int u = 0; u < U; u++) {
            float x[8];
            k[u].get(x);
            s[u] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) s[u] = fmaf(q[h][i], x[i], s[u]);
          }
#pragma unroll
          for (int w = 1; w < (LW ? LW : 32); w <<= 1) {
            if (!LW && w >= width) break;
#pragma unroll
            for (int u = 0; u < U; u++) s[u] += __shfl_xor_sync(0xffffffffu, s[u], w);
          }
#pragma unroll
          for (int u = 0; u < U; u++) {
            s[u] = in[u] ? s[u] : -INFINITY;
            mx = fmaxf(mx, s[u]);
          }
          mx *= c2;
          if (mx > st[h].m) {
            const float f = exp2f(st[h].m - mx);
            st[h].m = mx;
            st[h].l *= f;
#pragma unroll
            for (int i = 0; i < 8; i++) st[h].o[i] *= f;
          }
          const float ref = st[h].m == -INFINITY ? 0.0f : st[h].m;
#pragma unroll
          for (int u = 0; u < U; u++) {
            const float p = exp2f(fmaf(s[u], c2, -ref));
            float x[8];
            v[u].get(x);
            st[h].l += p;
#pragma unroll
            for (int i = 0; i < 8; i++) st[h].o[i] = fmaf(p, x[i], st[h].o[i]);
          }
        }
      }
    }
  }
  pdl_wait();                                          // the prefixes' parts are there
  if (keys > 0) {
    const Parts ps = parts_of(a, g, t0, t1, hk, (t - t0) * gq + h0 - hk * gq);
    for (int j = walker; j < ps.n; j += walkers) {
      const long long at = part_row(a, ps, j);
      if (at < 0) continue;
#pragma unroll
      for (int h = 0; h < HC; h++) {
        const float2 ml = a.part_ml[at + h];
        if (ml.y == 0.0f) continue;                    // nothing was seen and no sums were written (NaN is not 0)
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = 0.0f;
        if (cols) load8(a.part_o + (at + h) * D + d, 1, o);
        st[h].join(ml.x, ml.y, o);
      }
    }
  }
  // the warp's walkers
#pragma unroll
  for (int h = 0; h < HC; h++)
#pragma unroll
    for (int w = 16; w >= (LW ? LW : 1); w >>= 1) {
      if (!LW && w < width) break;
      float o[8];
      const float m = __shfl_xor_sync(0xffffffffu, st[h].m, w), l = __shfl_xor_sync(0xffffffffu, st[h].l, w);
#pragma unroll
      for (int i = 0; i < 8; i++) o[i] = __shfl_xor_sync(0xffffffffu, st[h].o[i], w);
      st[h].join(m, l, o);
    }
  if (warps == 1) {
    if (inside && of_warp == 0 && cols) {
#pragma unroll
      for (int h = 0; h < HC; h++) {
        const float f = st[h].l == 0.0f ? 0.0f : 1.0f / st[h].l;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = st[h].l == 0.0f ? 0.0f : st[h].o[i] * f;
        store8(reinterpret_cast<T*>(a.out) + (size_t)t * a.o_stride + (size_t)(h0 + h) * D + d, a.o_vec, o);
      }
    }
    return;
  }
  // the block's warps, and the cluster's blocks
  const int one = HC * (D + 2);
  if (of_warp == 0) {
#pragma unroll
    for (int h = 0; h < HC; h++) {
      float* to = sm + warp * one + h * (D + 2);
      if (cols)
#pragma unroll
        for (int i = 0; i < 8; i++) to[d + i] = st[h].o[i];
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
  if (share == 0 && inside) {
    auto other = [&](int z, int i) {                   // word i of warp z of the cluster
      if (z < 4) return sm[z * one + i];
      uint32_t there;
      float v;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(sm + (z & 3) * one + i)), "r"(z >> 2));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
      return v;
    };
    for (int x = threadIdx.x; x < HC * D; x += OT) {
      const int h = x / D, c = x - h * D, at = h * (D + 2);
      float M = -INFINITY, sum = 0.0f, total = 0.0f;
      for (int z = 0; z < 4 * shares; z++) M = fmaxf(M, other(z, at + D));
      const float ref = M == -INFINITY ? 0.0f : M;
      for (int z = 0; z < 4 * shares; z++) {
        const float f = exp2f(other(z, at + D) - ref);
        sum = fmaf(f, other(z, at + c), sum);
        total = fmaf(f, other(z, at + D + 1), total);
      }
      reinterpret_cast<T*>(a.out)[(size_t)t * a.o_stride + (size_t)(h0 + h) * D + c] = from_f32<T>(total == 0.0f ? 0.0f : sum / total);
    }
  }
  if (shares > 1) {                                    // (block 0 has read the others' shared memory)
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

template <typename T, int NC>
int launch_general(const Args& a, cudaStream_t stream) {
  const size_t smem = (size_t)((GR + GK) * (a.D + 4) + GK * NC * 64 + GR * (GK + 4)) * 4;
  const cudaError_t e = cudaFuncSetAttribute(prefix_general_kernel<T, NC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             ((GR + GK) * (NC * 64 + 4) + GK * NC * 64 + GR * (GK + 4)) * 4);
  if (e != cudaSuccess) return (int)e;
  return sglc_launch(prefix_general_kernel<T, NC>, dim3(a.n_blocks), dim3(GT), smem, stream, 1, true, a);
}
template <typename T>
int run_general(const Args& a, cudaStream_t stream) {
  switch ((a.D + 63) / 64) {
    case 1: return launch_general<T, 1>(a, stream);
    case 2: return launch_general<T, 2>(a, stream);
    case 3: return launch_general<T, 3>(a, stream);
    default: return launch_general<T, 4>(a, stream);
  }
}

template <typename T, int HC, int LW>
int launch_own(const Args& a, int warps, int shares, cudaStream_t stream) {
  const size_t smem = warps == 1 ? 0 : (size_t)4 * HC * (a.D + 2) * 4;
  const long long items = (long long)a.T * (a.H / HC);
  return sglc_launch(prefix_own_kernel<T, HC, LW>, dim3((unsigned)(warps == 1 ? (items + 3) / 4 : items), 1, shares), dim3(OT), smem,
                     stream, shares, true, a, warps);
}
template <typename T, int HC>
int choose_own(const Args& a, int warps, int shares, cudaStream_t stream) {
  if (a.lanes == 8) return launch_own<T, HC, 8>(a, warps, shares, stream);
  if (a.lanes == 16) return launch_own<T, HC, 16>(a, warps, shares, stream);
  return launch_own<T, HC, 0>(a, warps, shares, stream);
}
template <typename T>
int run_own(const Args& a, int max_own, cudaStream_t stream) {
  const int gq = a.H / a.Hkv, hc = gq % 4 == 0 ? 4 : gq % 2 == 0 ? 2 : 1;
  const long long items = (long long)a.T * (a.H / hc);
  // A warp an item where the items fill the multiprocessors and their own keys are few; else four, and blocks of a
  // cluster while there are fewer than four a multiprocessor and 64 keys or more are left for each.
  const int warps = items >= 16LL * a.sms && max_own <= 128 ? 1 : 4;
  int shares = 1;
  while (warps == 4 && shares < 8 && items * shares * 2 <= 4LL * a.sms && max_own >= 64 * shares * 2) shares *= 2;
  if (hc == 4) return choose_own<T, 4>(a, warps, shares, stream);
  if (hc == 2) return choose_own<T, 2>(a, warps, shares, stream);
  return choose_own<T, 1>(a, warps, shares, stream);
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
  a->tc = dtype == SGLC_BF16 && (a->D == 64 || a->D == 128);
  a->n_blocks = a->tc ? a->sms : 2 * a->sms;
  a->slot_rows = a->tc ? TC_SLOT : GENERAL_ROWS;
  a->key_tile = a->tc ? TC_KEYS : GENERAL_KEYS;
  const long long rows = (long long)a->T * (a->H / a->Hkv);
  a->slots = a->n_blocks + a->Hkv * (rows / a->slot_rows + a->G);      // (items of 128 rows are the only ones of their group)
  a->lanes = 1;
  while (a->lanes * 8 < a->D) a->lanes *= 2;
  return true;
}
// floats of workspace: the parts' sums, their (maximum, sum of weights), the groups' first items, the items' blocks
long long words(const Args& a) { return a.slots * a.slot_rows * (a.D + 2) + (a.G + 1) / 2 * 2 + 2 * a.slots; }
bool sizes_ok(int T, int R, int G, int H, int Hkv, int D) {
  return T >= 0 && R >= 0 && G >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && D > 0;
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
  if (D % 8 || D > 256 || G > MAX_GROUPS || (long long)T * H > 0x7fffffffLL || ((uintptr_t)cache & 15)) return SGLC_ERR_UNSUPPORTED;
  if (T == 0 || G == 0) return SGLC_OK;
  Args a = {};
  a.q = q; a.q_stride = q_stride; a.cache = cache;
  a.q_vec = ((uintptr_t)q & 15) == 0 && q_stride * (dtype == SGLC_F32 ? 4 : 2) % 16 == 0;
  a.table = table; a.bt_stride = bt_stride; a.R = R;
  a.token_req = token_req; a.positions = positions; a.group_start = group_start; a.shared_len = shared_len;
  a.out = out; a.o_stride = o_stride;
  a.T = T; a.G = G; a.H = H; a.Hkv = Hkv; a.D = D; a.page_size = page_size; a.n_pages = n_pages; a.scale = scale;
  const long long room = (long long)bt_width * page_size;
  a.last_position = (int)(room > 0x7ffffff0LL ? 0x7ffffff0LL : room) - 1;
  a.err = err;
  if (!lay_out(&a, dtype)) return SGLC_ERR_ARGUMENT;
  if (words(a) > ws_floats || ((uintptr_t)workspace & 15)) return SGLC_ERR_ARGUMENT;
  a.part_o = workspace;
  a.part_ml = reinterpret_cast<float2*>(workspace + a.slots * a.slot_rows * D);
  a.first_item = reinterpret_cast<int*>(a.part_ml + a.slots * a.slot_rows);
  a.item_blocks = reinterpret_cast<int2*>(a.first_item + (G + 1) / 2 * 2);
  a.o_vec = ((uintptr_t)out & 15) == 0 && o_stride * (dtype == SGLC_F32 ? 4 : 2) % 16 == 0;
  const int code = a.tc ? (D == 64 ? launch_tc<64, 4>(a, stream) : launch_tc<128, 2>(a, stream)) : dtype == SGLC_F32 ? run_general<float>(a, stream) : run_general<__nv_bfloat16>(a, stream);
  if (code) return code;
  return dtype == SGLC_F32 ? run_own<float>(a, max_own, stream) : run_own<__nv_bfloat16>(a, max_own, stream);
}
