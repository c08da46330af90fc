// Of every row of logits: the log-probability of a given token and its place in the order of choice, the entropy of the
// row's distribution, and its best tokens with their log-probabilities.
//   m = max l,  s = sum exp(l - m),  w = sum (l - m) exp(l - m):
//   logprob(t) = (l_t - m) - log s,   entropy = log s - w / s,
//   place(t) = how many tokens come before t: those of a larger logit, and of the same one with a smaller id.
// The row is read once: a thread keeps (m, s, w) of the entries it meets, sixteen at a time, scaled to its running maximum,
// and the place is a count of those few sixteens that reach the token's logit.  The best k come from the threads'
// maxima: k groups of threads have a maximum of T or more for T the k-th largest of the groups', so the best k are T or more,
// and they lie in the few stretches of a thread's turns whose own maximum is: only those (an eighth of a thread's
// entries each, for about 31 threads at k = 20: a sixtieth of the row, still in L2) are looked at again.
// Sums are 32-bit, a thread's over V / 256 entries and then pairwise.  The exponential is the special-function unit's
// (2 ulp) of a difference taken exactly as it is rounded, so no logit is too large for it.
// What bounds it on a B200: float32, the logits' way from memory and the last rows' blocks (2,048 rows of 50,257: 82 us, 4.9 TB/s);
// bfloat16, no one thing (777 rows of 128,000: 63 us, 3.2 TB/s): twice the entries a byte keep the issue slots 64 % busy and the
// special-function units 42 %, DRAM 39 %, a thread has two pieces of 16 bytes in flight where float32 has four, and 777 rows
// are 1.3 rounds of 592 resident blocks; few rows, what follows the pass (64 rows with 20 best 13 us, one row 7).  A turn with a
// forbidden entry (-inf) makes its exponentials twice, see there; the entropy's sums are made whether it is asked for or not.  Blocks of
// 256 threads, four a multiprocessor: with 512 or 1,024 a row's end, where threads wait for one another, was the longer.
#include "common.cuh"

SGLC_DEFINE_ERROR_STRING()

namespace {
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int RESIDENT = 4;              // blocks a multiprocessor holds
constexpr int MAX_TOP = 64;
constexpr int ROOM = 1024;               // entries above the threshold that are sorted in shared memory
constexpr int SEGMENTS = 8;              // stretches of a thread's turns whose maxima are kept
constexpr int MAX_SHARES = 8;            // blocks of a row (one cluster)
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Args {
  const void* logits;
  long long ld;                          // elements between rows
  int V, k;
  const int* tokens;
  float *logprob, *entropy;
  int* place;
  int* top_ids;
  float* top_logprobs;
  long long top_ld;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two at a time, each rounded as one alone.
#define SGLC_TWO(name, op)                                                                                                       \
  __device__ __forceinline__ float2 name(float2 x, float2 y) {                                                                   \
    unsigned long long r;                                                                                                        \
    asm(op ".rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<unsigned long long&>(x)), "l"(reinterpret_cast<unsigned long long&>(y))); \
    return reinterpret_cast<float2&>(r);                                                                                         \
  }
SGLC_TWO(add2, "add")
SGLC_TWO(mul2, "mul")
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(reinterpret_cast<unsigned long long&>(x)), "l"(reinterpret_cast<unsigned long long&>(y)),
      "l"(reinterpret_cast<unsigned long long&>(z)));
  return reinterpret_cast<float2&>(r);
}

// the largest of the warp (numbers; NaN is passed over)
__device__ __forceinline__ float warp_maximum(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  typedef float4 Raw;
  __device__ static Raw none() { return make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }
  __device__ static void open(const Raw& x, float (&v)[4]) { v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  typedef uint4 Raw;
  __device__ static Raw none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }       // (-inf)
  __device__ static void open(const Raw& x, float (&v)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

// the order of choice: larger logits first, then smaller ids; NaN as the lowest, -0 as 0
__device__ __forceinline__ float ranked(float v) { return v == v ? v + 0.0f : -INFINITY; }
__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ unsigned long long key_of(float v, int id) {
  return ((unsigned long long)ordered(v) << 32) | (unsigned)~id;      // (never 0: that is "no entry")
}

// Maximum; how many entries are it; sum over the others; sum of (l - m) exp(l - m), in units of log 2.  The ones are kept apart
// so that log(n + s) of a row with one likely token, log1p(s), has the digits of s and not what 1 + s leaves of them.
struct Sums {
  float m, n, s, w;
  __device__ __forceinline__ void rescale(float top) {        // to a larger maximum
    if (m > -INFINITY) {
      const float d = (m - top) * LOG2E, f = ex2(d);
      // (a factor of 0 drops the share whole: 0 * -inf would make NaN of it)
      w = f > 0.0f ? f * fmaf(d, n + s, w) : s * 0.0f;
      s = (n + s) * f;
      n = 0.0f;
    }
    m = top;
  }
};
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  if (a.m > b.m) b.rescale(a.m);
  if (b.m > a.m) a.rescale(b.m);
  return {a.m, a.n + b.n, a.s + b.s, a.w + b.w};
}

struct Shared {
  Sums warp_sums[WARPS];
  int warp_count[WARPS];
  float group[64];                        // maxima of groups of threads
  float seg[SEGMENTS][THREADS];           // a thread's maxima of stretches of its turns
  int chosen[SEGMENTS * THREADS];         // (stretch, thread)
  int n_chosen, n_above;
  float threshold;
  unsigned long long above[ROOM];
  unsigned long long list[MAX_TOP];       // the block's best, in order
  int scan[WARPS + 1];
  // block 0 of a row's cluster: what each block found
  Sums row_sums[MAX_SHARES];
  int row_count[MAX_SHARES];
  unsigned long long row_list[MAX_SHARES * MAX_TOP];
};

// A block's part of a row: whole 16-byte pieces first..last-1 counted from the row's first aligned one, and, in block 0, the
// entries before and behind all pieces.
template <typename T>
struct Part {
  const T* row;
  int head, first, last, tail, V;         // tail: id of the first entry behind the pieces
  bool ends;                              // this block has head and tail
  static constexpr int N = Vec<T>::N;
  __device__ int rounds() const { return (last - first + THREADS - 1) / THREADS; }
  __device__ int id_of(int piece) const { return head + piece * N; }
  __device__ bool is_in(int piece) const { return piece < last; }
  __device__ typename Vec<T>::Raw raw(int piece) const {       // (-inf where the part ends)
    return piece < last ? __ldg(reinterpret_cast<const typename Vec<T>::Raw*>(row + id_of(piece))) : Vec<T>::none();
  }
  __device__ bool take(int piece, float (&v)[N]) const {
    Vec<T>::open(raw(piece), v);
    return piece < last;
  }
  // the loose entry of thread `t`, or -1
  __device__ int loose(int t) const {
    if (!ends) return -1;
    if (t < head) return t;
    const int id = tail + t - head;
    return id < V ? id : -1;
  }
};

template <typename T>
__global__ void __launch_bounds__(THREADS, RESIDENT)
token_logprobs_kernel(const Args a) {
  constexpr int N = Vec<T>::N;
  constexpr int DEEP = 16 / N;            // pieces in flight a thread
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int share = blockIdx.z, shares = gridDim.z;
  // (that this block has begun, for the others of the row's cluster, which store into block 0's shared memory below)
  if (shares > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  pdl_launch_dependents();
  auto part_of = [&](long long row) {
    Part<T> x;
    x.row = reinterpret_cast<const T*>(a.logits) + row * a.ld;
    x.V = a.V;
    x.head = min(a.V, (int)((16 - ((uintptr_t)x.row & 15)) & 15) / (int)sizeof(T));
    const int pieces = (a.V - x.head) / N;
    x.tail = x.head + pieces * N;
    x.first = (int)((long long)pieces * share / shares);
    x.last = (int)((long long)pieces * (share + 1) / shares);
    x.ends = share == 0;
    return x;
  };
  // (the first pieces are asked for ahead of the chain row -> token -> its logit)
  typename Vec<T>::Raw next[DEEP];
  const long long r = blockIdx.x;
  const Part<T> p = part_of(r);
#pragma unroll
  for (int u = 0; u < DEEP; u++) next[u] = p.raw(p.first + tid + u * THREADS);
  const int tok = a.tokens ? a.tokens[r] : -1;
  const float tv_raw = tok >= 0 && tok < a.V ? to_f32(p.row[tok]) : 0.0f;
  const bool asked = tok >= 0 && tok < a.V;
  const float tv = asked ? ranked(tv_raw) : INFINITY;
  const bool counts = asked && a.place;

  // ---- one pass: maximum, sums, count; sixteen entries of a thread at a time ----
  // The reference is the warp's: a thread's own would be moved by some thread of the warp at nearly every turn.
  Sums x = {-INFINITY, 0.0f, 0.0f, 0.0f};
  float best = -INFINITY;                 // this thread's maximum
  int count = 0;
  // entries of the token's logit count before it by their ids; of a piece of 16 bytes all ids are smaller or none is
  // (the token's own piece is looked at once more below)
  const float above = __uint_as_float(tv >= 0.0f ? __float_as_uint(tv) + 1u : __float_as_uint(tv) - 1u);       // the next larger
  // (rounds are the warp's: a thread past the part's end reads -inf)
  const int turns = (p.last - p.first + THREADS * DEEP - 1) / (THREADS * DEEP), stretch = (turns + SEGMENTS - 1) / SEGMENTS;
  float seg_best = -INFINITY;
  int seg = 0, seg_turn = 0;
  for (int q = p.first + tid; q - tid < p.last; q += THREADS * DEEP) {
    float v[DEEP][N];
#pragma unroll
    for (int u = 0; u < DEEP; u++) Vec<T>::open(next[u], v[u]);
#pragma unroll
    for (int u = 0; u < DEEP; u++) next[u] = p.raw(q + (DEEP + u) * THREADS);
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 16; i++) top[i & 3] = fmaxf(top[i & 3], v[i / N][i % N]);
    top[0] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    seg_best = fmaxf(seg_best, top[0]);
    if (++seg_turn == stretch) {
      sh.seg[seg++][tid] = seg_best;
      best = fmaxf(best, seg_best);
      seg_best = -INFINITY;
      seg_turn = 0;
    }
    const float warp_top = warp_maximum(top[0]);
    const bool reaches = warp_top >= x.m;              // (then some of these may be the maximum, and are counted)
    if (warp_top > x.m) x.rescale(warp_top);
    const float m = x.m == -INFINITY ? 0.0f : x.m;
    float2 s = make_float2(0.0f, 0.0f), w = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float2 d = mul2(add2(make_float2(v[i / N][i % N], v[i / N][i % N + 1]), make_float2(-m, -m)), make_float2(LOG2E, LOG2E));
      const float2 e = make_float2(ex2(d.x), ex2(d.y));
      s = add2(s, e);
      w = fma2(d, e, w);
    }
    if (reaches) {                                     // (few turns: the sum again, without what is counted)
      s = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float e = ex2((v[i / N][i % N] - m) * LOG2E);
        if (e == 1.0f) x.n += 1.0f;
        else s.x += e;
      }
    }
    if (!(w.x + w.y == w.x + w.y)) {
      // an entry at -inf, where the exponential is 0 and the product with it should be: once more, with a bound (or an entry
      // that is no number, and remains it)
      w = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float d = (v[i / N][i % N] - m) * LOG2E;
        w.x = fmaf(fmaxf(d, -200.0f), ex2(d), w.x);
      }
    }
    x.s += s.x + s.y;
    x.w += w.x + w.y;
    if (counts && top[0] >= tv) {
      if (tv > -INFINITY) {
#pragma unroll
        for (int u = 0; u < DEEP; u++) {
          const float from = p.id_of(q + u * THREADS) + N <= tok ? tv : above;
#pragma unroll
          for (int i = 0; i < N; i++) count += v[u][i] >= from;
        }
      }
    }
    if (counts && tv == -INFINITY) {                   // (a token that is not allowed: NaN counts as it, too)
#pragma unroll
      for (int i = 0; i < 16; i++) count += p.is_in(q + i / N * THREADS) && (ranked(v[i / N][i % N]) > tv || p.id_of(q + i / N * THREADS) + i % N < tok);
    }
  }
  if (seg_turn > 0) {
    sh.seg[seg++][tid] = seg_best;
    best = fmaxf(best, seg_best);
  }
  auto place_of = [&](float y, int id) { count += ranked(y) > tv || (ranked(y) == tv && id < tok); };
  // single entries that are looked at below: before and behind the pieces; of the token's own piece
  const int my_loose = p.loose(tid);
  const float loose = my_loose >= 0 ? to_f32(p.row[my_loose]) : -INFINITY;
  const int own_piece = asked && tok >= p.head ? (tok - p.head) / N : -1, own_id = p.id_of(own_piece) + tid;
  const bool owns = counts && tid < N && own_piece >= p.first && own_piece < p.last && own_id < tok;
  const float own = owns ? ranked(to_f32(p.row[own_id])) : 0.0f;

  if (owns && tv > -INFINITY) count += own == tv;       // the token's own piece: equal logits of smaller ids
  if (p.ends) {
    const float warp_top = warp_maximum(loose);
    if (warp_top > x.m) x.rescale(warp_top);
    if (my_loose >= 0) {
      const float d = (loose - (x.m == -INFINITY ? 0.0f : x.m)) * LOG2E, e = ex2(d);
      if (e == 1.0f) x.n += 1.0f;
      else x.s += e;
      x.w = fmaf(fmaxf(d, -200.0f), e, x.w);
      best = fmaxf(best, loose);
      if (counts) place_of(loose, my_loose);
    }
  }
  best = ranked(best);

  // ---- the block's sums and count (warp 0), and a threshold for its best k ----
  // At least k entries reach the threshold: it is the k-th largest of the maxima of G = 32 (64) groups of threads.  In random
  // order G (H_G - H_(G-k)) entries do on average, H_n = 1 + 1/2 + .. + 1/n: entries from the largest down until k groups have
  // one (31 at k = 20, 130 at 32, 304 at 64), and so many threads at most have them.
  const int k = a.k, groups = k <= 32 ? 32 : 64, of_group = THREADS / groups;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {                 // (the warp's lanes have one reference)
    x.n += __shfl_xor_sync(0xffffffffu, x.n, o);
    x.s += __shfl_xor_sync(0xffffffffu, x.s, o);
    x.w += __shfl_xor_sync(0xffffffffu, x.w, o);
  }
  count = __reduce_add_sync(0xffffffffu, count);
  if (lane == 0) {
    sh.warp_sums[warp] = x;
    sh.warp_count[warp] = count;
  }
  if (k > 0) {
    float top = best;
    for (int o = of_group / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane % of_group == 0) sh.group[tid / of_group] = top;
  }
  if (tid == 0) {
    sh.n_chosen = 0;
    sh.n_above = 0;
  }
  __syncthreads();
  if (warp == 0) {
    x = lane < WARPS ? sh.warp_sums[lane] : Sums{-INFINITY, 0.0f, 0.0f, 0.0f};
    count = __reduce_add_sync(0xffffffffu, lane < WARPS ? sh.warp_count[lane] : 0);
    const float top = warp_maximum(x.m);
    if (top > x.m) x.rescale(top);
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) {
      x.n += __shfl_xor_sync(0xffffffffu, x.n, o);
      x.s += __shfl_xor_sync(0xffffffffu, x.s, o);
      x.w += __shfl_xor_sync(0xffffffffu, x.w, o);
    }
    for (int me = lane; k > 0 && me < groups; me += 32) {
      const float mine = sh.group[me];
      int rank = 0;
      for (int u = 0; u < groups; u++) rank += sh.group[u] > mine || (sh.group[u] == mine && u < me);
      if (rank == k - 1) sh.threshold = mine;
    }
    if (lane == 0 && shares == 1) sh.row_sums[0] = x;
  }
  // what is known of the row, and of token `id` with logit v at place i of the order
  auto give_row = [&](const Sums& x, int count) {
    const float total = x.n + x.s;
    const bool none = total == 0.0f;                        // every entry at -inf (NaN is not 0)
    const float log_s = x.n == 1.0f ? log1pf(x.s) : logf(total);
    a.logprob[r] = !asked ? 0.0f : none ? -INFINITY : (tv_raw - x.m) - log_s;
    if (a.entropy) a.entropy[r] = none ? 0.0f : log_s - LN2 * (x.w / total);
    if (a.place) a.place[r] = asked ? count : -1;
  };
  auto give_top = [&](const Sums& x, unsigned long long key, int i) {
    const float total = x.n + x.s, log_s = x.n == 1.0f ? log1pf(x.s) : logf(total), v = unordered((unsigned)(key >> 32));
    a.top_ids[r * a.top_ld + i] = (int)~(unsigned)key;
    a.top_logprobs[r * a.top_ld + i] = total == 0.0f ? -INFINITY : (v - x.m) - log_s;
  };

  // ---- the block's best k ----
  if (k > 0) {
    __syncthreads();
    float T0 = sh.threshold;
    // the stretches with entries at the threshold or above, and those entries; where these are too many (equal logits), or the
    // threshold is -inf (few tokens allowed), only what is above it, and then equal ones from the smallest id on
    bool ties = T0 > -INFINITY;
    if (best >= T0)
      for (int i = 0; i < seg; i++)
        if (ties ? ranked(sh.seg[i][tid]) >= T0 : ranked(sh.seg[i][tid]) > T0) sh.chosen[atomicAdd(&sh.n_chosen, 1)] = i * THREADS + tid;
    __syncthreads();
    const int rounds = p.rounds(), of_seg = stretch * DEEP, items = sh.n_chosen * of_seg;
    // f(value, id) of every entry of the chosen stretches, and of those before and behind the pieces
    auto again = [&](auto&& f) {
      for (int c0 = tid; c0 < items; c0 += 2 * THREADS) {
        typename Vec<T>::Raw x[2];
        int q[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {                 // (two on their way at a time)
          const int c = c0 + u * THREADS, which = (unsigned)c / (unsigned)of_seg;
          q[u] = p.last;
          if (c < items) {
            const int st = sh.chosen[which];
            q[u] = p.first + st % THREADS + (st / THREADS * of_seg + c - which * of_seg) * THREADS;
          }
          x[u] = p.raw(q[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
          float v[N];
          Vec<T>::open(x[u], v);
          if (p.is_in(q[u]))
#pragma unroll
            for (int i = 0; i < N; i++) f(ranked(v[i]), p.id_of(q[u]) + i);
        }
      }
      if (my_loose >= 0) f(ranked(loose), my_loose);
    };
    auto collect = [&]() {
      again([&](float v, int id) {
        if (ties ? v >= T0 : v > T0) {
          const int at = atomicAdd(&sh.n_above, 1);
          if (at < ROOM) sh.above[at] = key_of(v, id);
        }
      });
      __syncthreads();
    };
    collect();
    if (ties && sh.n_above > ROOM) {
      ties = false;
      __syncthreads();
      if (tid == 0) sh.n_above = 0;
      __syncthreads();
      collect();
    }
    if (sh.n_above > ROOM) {
      // More entries above the threshold than there is room for (large logits at one stride): the k-th largest value
      // itself, bit by bit, by counting.  It becomes the threshold, so fewer than k entries are above it.
      unsigned low = ordered(T0);
      for (int bit = 31; bit >= 0; bit--) {
        // the largest u >= ordered(T0) such that k entries or more are at least u
        const unsigned u = (low & (0xffffffffu << bit)) | (1u << bit);
        if (u <= low) continue;
        int n = 0;
        again([&](float v, int) { n += ordered(v) >= u; });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        __syncthreads();
        if (lane == 0) sh.scan[warp] = n;
        __syncthreads();
        n = 0;
        for (int w = 0; w < WARPS; w++) n += sh.scan[w];
        if (n >= k) low = u;
      }
      T0 = unordered(low);
      __syncthreads();
      if (tid == 0) sh.n_above = 0;
      __syncthreads();
      collect();
    }
    const int n_above = sh.n_above;
    if (shares == 1 && ties) {                              // the usual end: whoever ranks an entry gives it out
      x = sh.row_sums[0];
      if (tid == 0) give_row(x, count);
      for (int c = tid; c < n_above; c += THREADS) {
        const unsigned long long key = sh.above[c];
        int before = 0;
        for (int u = 0; u < n_above; u++) before += sh.above[u] > key;
        if (before < k) give_top(x, key, before);
      }
      return;
    }
    for (int c = tid; c < n_above; c += THREADS) {
      const unsigned long long key = sh.above[c];
      int before = 0;
      for (int u = 0; u < n_above; u++) before += sh.above[u] > key;
      if (before < k) sh.list[before] = key;
    }
    // entries equal to the threshold, the smallest ids first, until there are k: rounds of pieces ascend in id, between the
    // loose entries before and behind them
    int have = min(n_above, k);
    auto fill = [&](const float* v, int n, int id0) {
      int mine = 0;
      for (int i = 0; i < n; i++) mine += ranked(v[i]) == T0;
      int run = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
      }
      __syncthreads();
      if (lane == 31) sh.scan[warp] = run;
      __syncthreads();
      int before = have + run - mine, total = 0;
      for (int w = 0; w < WARPS; w++) {
        if (w < warp) before += sh.scan[w];
        total += sh.scan[w];
      }
      for (int i = 0; i < n; i++)
        if (ranked(v[i]) == T0) {
          if (before < k) sh.list[before] = key_of(T0, id0 + i);
          before++;
        }
      have += total;
    };
    auto fill_loose = [&](int from, int to) {             // (ids from..to-1: fewer than a piece's entries)
      if (p.ends && have < k && from < to) {
        float v[1] = {0.0f};
        const bool in = from + tid < to;
        if (in) v[0] = to_f32(p.row[from + tid]);
        fill(v, in ? 1 : 0, from + tid);
      }
    };
    if (!ties) fill_loose(0, p.head);
    for (int i = 0; !ties && i < rounds && have < k; i++) {
      float v[N];
      const int q = p.first + tid + i * THREADS;
      const bool in = p.take(q, v);
      fill(v, in ? N : 0, p.id_of(q));
    }
    if (!ties) fill_loose(p.tail, p.V);
    have = min(have, k);
    if (tid >= have && tid < k) sh.list[tid] = 0;           // a part of fewer than k entries
    __syncthreads();
  }

  // ---- the row's parts come together in block 0 of the cluster ----
  if (shares > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    auto there = [](const void* local) {
      uint32_t at;
      asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(local)));
      return at;
    };
    if (tid == 0) {
      const float f[4] = {x.m, x.n, x.s, x.w};
#pragma unroll
      for (int i = 0; i < 4; i++)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there(&sh.row_sums[share]) + 4 * i), "f"(f[i]) : "memory");
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(there(&sh.row_count[share])), "r"(count) : "memory");
    }
    if (tid < k)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(there(&sh.row_list[share * k + tid])), "l"(sh.list[tid]) : "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (share != 0) return;
    x = sh.row_sums[0];
    count = sh.row_count[0];
    for (int i = 1; i < shares; i++) {
      x = join(x, sh.row_sums[i]);
      count += sh.row_count[i];
    }
    for (int c = tid; c < shares * k; c += THREADS) {
      const unsigned long long key = sh.row_list[c];
      int before = 0;
      for (int u = 0; u < shares * k; u++) before += sh.row_list[u] > key;
      if (before < k && key) sh.list[before] = key;
    }
    __syncthreads();
  }

  if (shares == 1 && k > 0) x = sh.row_sums[0];
  if (tid == 0) give_row(x, count);
  if (tid < k) give_top(x, sh.list[tid], tid);
}

// Blocks of a row.  Few rows are dealt to several blocks each, down to 512 pieces of 16 bytes a block.
int shares_of(int n_rows, int V, int size) {
  int s = 1;
  while (s < MAX_SHARES && n_rows * s * 2 <= 296 && (long long)V * size / 16 / (s * 2) >= 512) s *= 2;
  return s;
}
}  // namespace

// logits: n_rows rows of V entries, ld elements apart, dtype float or bfloat16.  tokens: int32 or null (no token is asked
// for); one outside 0..V-1 asks for nothing: logprob 0, place -1.  entropy, place: may be null.  k <= 64 best
// tokens a row into top_ids and top_logprobs, rows top_ld apart.
SGLC_API int sglc_token_logprobs(const void* logits, long long ld, int dtype, int n_rows, int V, const int* tokens,
                                 float* logprob, float* entropy, int* place, int k, int* top_ids, float* top_logprobs,
                                 long long top_ld, cudaStream_t stream) {
  if (n_rows <= 0) return n_rows < 0 ? SGLC_ERR_ARGUMENT : SGLC_OK;
  if (V <= 0 || k < 0 || k > V || (dtype != SGLC_F32 && dtype != SGLC_BF16)) return SGLC_ERR_ARGUMENT;
  if (k > MAX_TOP) return SGLC_ERR_UNSUPPORTED;
  const Args a = {logits, ld, V, k, tokens, logprob, entropy, place, top_ids, top_logprobs, top_ld};
  const int shares = shares_of(n_rows, V, dtype == SGLC_F32 ? 4 : 2);
  const dim3 grid(n_rows, 1, shares);
  if (dtype == SGLC_F32) return sglc_launch(token_logprobs_kernel<float>, grid, dim3(THREADS), 0, stream, shares, true, a);
  return sglc_launch(token_logprobs_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, stream, shares, true, a);
}
