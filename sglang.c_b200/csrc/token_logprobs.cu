// Of every row of logits: the log-probability of a given token and its place in the order of choice, the entropy of the
// row's distribution, and its best tokens with their log-probabilities.
//   m = max l,  s = sum exp(l - m),  w = sum (l - m) exp(l - m):
//   logprob(t) = (l_t - m) - log s,   entropy = log s - w / s,
//   place(t) = how many tokens come before t: those of a larger logit, and of the same one with a smaller id.
// The row is read once: a thread keeps (m, s, w) of the entries it meets, sixteen at a time, scaled to its running maximum,
// and the place is a count of those few sixteens that reach the token's logit.  The best k come from the threads'
// maxima: k groups of threads have a maximum of T or more for T the k-th largest of the groups', so the best k are T or more,
// and they lie with the few threads whose own maximum is: only those threads' pieces (a tenth of the row, still in
// L2) are looked at again.
// Sums are 32-bit, a thread's over V / 256 entries and then pairwise.  The exponential is the special-function unit's
// (2 ulp) of a difference taken exactly as it is rounded, so no logit is too large for it.
#include "common.cuh"

SGLC_DEFINE_ERROR_STRING()

namespace {
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_TOP = 64;
constexpr int ROOM = 1024;               // entries above the threshold that are sorted in shared memory
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
  __device__ static void take(const float* p, float (&v)[4]) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void take(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
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
  int chosen[THREADS];
  int n_chosen, n_above, n_out;
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
  __device__ bool take(int piece, float (&v)[N]) const {
    if (piece < last) {
      Vec<T>::take(row + id_of(piece), v);
      return true;
    }
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = -INFINITY;
    return false;
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
__global__ void __launch_bounds__(THREADS)
token_logprobs_kernel(const Args a) {
  constexpr int N = Vec<T>::N;
  constexpr int DEEP = 16 / N;            // pieces in flight a thread
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int share = blockIdx.z, shares = gridDim.z;
  const long long r = blockIdx.x;
  // (that this block has begun, for the others of the row's cluster, which store into block 0's shared memory below)
  if (shares > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  pdl_launch_dependents();
  Part<T> p;
  p.row = reinterpret_cast<const T*>(a.logits) + r * a.ld;
  p.V = a.V;
  p.head = min(a.V, (int)((16 - ((uintptr_t)p.row & 15)) & 15) / (int)sizeof(T));
  const int pieces = (a.V - p.head) / N;
  p.tail = p.head + pieces * N;
  p.first = (int)((long long)pieces * share / shares);
  p.last = (int)((long long)pieces * (share + 1) / shares);
  p.ends = share == 0;
  const int tok = a.tokens ? a.tokens[r] : -1;
  const bool asked = tok >= 0 && tok < a.V;
  const float tv_raw = asked ? to_f32(p.row[tok]) : 0.0f;
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
  for (int q = p.first + tid; q - lane < p.last; q += THREADS * DEEP) {
    float v[DEEP][N];
#pragma unroll
    for (int u = 0; u < DEEP; u++) p.take(q + u * THREADS, v[u]);
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 16; i++) top[i & 3] = fmaxf(top[i & 3], v[i / N][i % N]);
    top[0] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    best = fmaxf(best, top[0]);
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
  auto place_of = [&](float y, int id) { count += ranked(y) > tv || (ranked(y) == tv && id < tok); };
  if (counts && tv > -INFINITY && tid < N) {           // the token's own piece: equal logits of smaller ids
    const int piece = (tok - p.head) / N, id = p.id_of(piece) + tid;
    if (tok >= p.head && piece >= p.first && piece < p.last && id < tok) count += ranked(to_f32(p.row[id])) == tv;
  }
  const int my_loose = p.loose(tid);
  const float loose = my_loose >= 0 ? to_f32(p.row[my_loose]) : -INFINITY;
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

#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums y = {__shfl_xor_sync(0xffffffffu, x.m, o), __shfl_xor_sync(0xffffffffu, x.n, o),
                    __shfl_xor_sync(0xffffffffu, x.s, o), __shfl_xor_sync(0xffffffffu, x.w, o)};
    x = join(x, y);
    count += __shfl_xor_sync(0xffffffffu, count, o);
  }
  if (lane == 0) {
    sh.warp_sums[warp] = x;
    sh.warp_count[warp] = count;
  }
  if (tid == 0) {
    sh.n_chosen = 0;
    sh.n_above = 0;
  }
  __syncthreads();
  x = sh.warp_sums[0];
  count = sh.warp_count[0];
#pragma unroll
  for (int w = 1; w < WARPS; w++) {
    x = join(x, sh.warp_sums[w]);
    count += sh.warp_count[w];
  }

  // ---- the block's best k ----
  const int k = a.k;
  if (k > 0) {
    // A threshold that at least k entries reach: the k-th largest of the maxima of 32 (64) groups of threads.  About
    // -32 ln(1 - k / 32) entries reach it (31 at k = 20), in as many threads at most, if large ones are anywhere.
    const int of_group = k <= 32 ? 8 : 4;
    float top = best;
    for (int o = of_group / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane % of_group == 0) sh.group[tid / of_group] = top;
    __syncthreads();
    if (warp == 0) {
      for (int half = 0; half < (k <= 32 ? 1 : 2); half++) {
        const int me = lane + 32 * half;
        const float mine = sh.group[me];
        int rank = 0;
        for (int u = 0; u < (k <= 32 ? 32 : 64); u++) rank += sh.group[u] > mine || (sh.group[u] == mine && u < me);
        if (rank == k - 1) sh.threshold = mine;
      }
    }
    __syncthreads();
    float T0 = sh.threshold;
    // the threads with entries at the threshold or above, and those entries; where these are too many (equal logits), or the
    // threshold is -inf (few tokens allowed), only what is above it, and then equal ones from the smallest id on
    bool ties = T0 > -INFINITY;
    if (ties ? best >= T0 : best > T0) sh.chosen[atomicAdd(&sh.n_chosen, 1)] = tid;
    __syncthreads();
    const int n_chosen = sh.n_chosen, rounds = p.rounds();
    // f(value, id) of every entry of the chosen threads
    auto again = [&](auto&& f) {
      for (int c = tid; c < n_chosen * rounds; c += THREADS) {
        const int t = sh.chosen[c / rounds], q = p.first + t + c % rounds * THREADS;
        float v[N];
        if (p.take(q, v)) {
#pragma unroll
          for (int i = 0; i < N; i++) f(ranked(v[i]), p.id_of(q) + i);
        }
      }
      if (tid < n_chosen) {
        const int id = p.loose(sh.chosen[tid]);
        if (id >= 0) f(ranked(to_f32(p.row[id])), id);
      }
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

  const float total = x.n + x.s;
  const bool none = total == 0.0f;                          // every entry at -inf (NaN is not 0)
  const float log_s = x.n == 1.0f ? log1pf(x.s) : logf(total);
  if (tid == 0) {
    a.logprob[r] = !asked ? 0.0f : none ? -INFINITY : (tv_raw - x.m) - log_s;
    if (a.entropy) a.entropy[r] = none ? 0.0f : log_s - LN2 * (x.w / total);
    if (a.place) a.place[r] = asked ? count : -1;
  }
  if (tid < k) {
    const unsigned long long key = sh.list[tid];
    const int id = (int)~(unsigned)key;
    a.top_ids[r * a.top_ld + tid] = id;
    const float v = unordered((unsigned)(key >> 32));
    a.top_logprobs[r * a.top_ld + tid] = none ? -INFINITY : (v - x.m) - log_s;
  }
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
