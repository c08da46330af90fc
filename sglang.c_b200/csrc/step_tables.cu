// A step's arrays made on the device from the requests' lengths: where each request's tokens start, the pages they need
// (taken from the pool's free stack, the top first, in the order of the requests, as the host's pool hands them out),
// the block tables' new entries, and of every token its request, position and cache slot.
//   start_r = sum of q over the requests before r;  held_r = ceil(kv_r / P);  need_r = ceil((kv_r + q_r) / P) - held_r;
//   page j of request r's new ones: free[n_free - 1 - (sum of need before r) - j];
//   token i of request r: position p = kv_r + i, slot table[r][p / P] * P + p % P.
// All or nothing: lengths that do not fit set the status word and nothing else is written.
//
// What bounds it: a launch and a chain of dependent reads (lengths -> scan -> search -> page -> slot); the words written
// are 12 bytes a token.  5 to 6 us a call in a row on a B200, for 64 requests of a token as for 260,000 tokens of 515.  One launch,
// no block waits for another: every block scans all requests' lengths (they are a few kilobytes) into its own shared memory,
// and takes its share of the tokens and of the new pages, whose page it finds in the free stack itself, without the table
// entry that another block writes.
#include "common.cuh"

SGLC_DEFINE_ERROR_STRING()

namespace {
constexpr int THREADS = 512;
constexpr int MAX_REQUESTS = 16384;       // three words each in shared memory
constexpr int OVERLAP = -4;               // (a launcher's code: what is written lies in what is read)
enum { PAGES_SHORT = 1, ROW_SHORT = 2, TOKENS_MANY = 4, BAD_LENGTH = 8 };

struct Args {
  const int *q_len, *kv_len, *free_pages, *n_free;
  int* table;
  long long bt_stride;
  int bt_width, free_cap, R, page_size, t_cap;
  int *q_start, *new_len, *token_req, *positions, *slots, *left, *status;
  int vec;                                // the tokens' arrays begin on 16 bytes
};

// What the warps find of their runs of requests.
struct Warps {
  long long q[THREADS / 32], p[THREADS / 32];
  int bad[THREADS / 32];
};

// the last r of 0..n-1 with first[r] <= x (first ascends; requests without any share their successor's start)
__device__ __forceinline__ int find(const int* first, int n, int x) {
  int lo = 0, hi = n;                     // first[lo] <= x < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS)
step_tables_kernel(const Args a) {
  extern __shared__ int sm[];
  const int R = a.R, P = a.page_size, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* start = sm;                        // [R + 1]: lengths first, then first tokens
  int* taken = sm + R + 1;                // [R + 1]: pages that the requests before take
  int* kv = sm + 2 * (R + 1);             // [R]
  __shared__ Warps warps;
  // (The arrays written here are what later kernels of a step read ahead of their own wait, so this kernel lets none
  // of them begin before it ends: there is no early release of dependents.)
  pdl_wait();
  for (int r = tid; r < R; r += THREADS) {
    start[r] = a.q_len[r];
    kv[r] = a.kv_len[r];
  }
  const int n_free = *a.n_free;
  __syncthreads();
  // a run of requests a thread: its sums, then the sums before it
  const int per = (R + THREADS - 1) / THREADS, r0 = min(R, tid * per), r1 = min(R, r0 + per);
  long long q_sum = 0, p_sum = 0;
  int bad = 0;
  for (int r = r0; r < r1; r++) {
    const int q = start[r], k = kv[r];
    if (q < 0 || k < 0 || (long long)q + k > 0x7fffffffLL - P) {
      bad |= BAD_LENGTH;
      continue;
    }
    const int all = (int)(((unsigned)(k + q) + P - 1) / P);
    if (q > 0 && all > a.bt_width) bad |= ROW_SHORT;
    q_sum += q;
    p_sum += all - (int)(((unsigned)k + P - 1) / P);
  }
  long long q_run = q_sum, p_run = p_sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, q_run, o), y = __shfl_up_sync(0xffffffffu, p_run, o);
    if (lane >= o) {
      q_run += x;
      p_run += y;
    }
  }
  bad = __reduce_or_sync(0xffffffffu, (unsigned)bad);
  if (lane == 31) {
    warps.q[warp] = q_run;
    warps.p[warp] = p_run;
    warps.bad[warp] = bad;
  }
  __syncthreads();
  long long q_all = 0, p_all = 0, q_before = 0, p_before = 0;
  bad = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; w++) {
    if (w == warp) {
      q_before = q_all;
      p_before = p_all;
    }
    q_all += warps.q[w];
    p_all += warps.p[w];
    bad |= warps.bad[w];
  }
  if (n_free < 0 || n_free > a.free_cap) bad |= BAD_LENGTH;
  if (p_all > n_free) bad |= PAGES_SHORT;
  if (q_all > a.t_cap) bad |= TOKENS_MANY;
  const bool first_block = blockIdx.x == 0;
  if (bad) {                              // (the same in every block)
    if (first_block && tid == 0) *a.status = bad;
    return;
  }
  {
    int q = (int)(q_before + q_run - q_sum), p = (int)(p_before + p_run - p_sum);
    for (int r = r0; r < r1; r++) {
      const int len = start[r], k = kv[r];
      start[r] = q;
      taken[r] = p;
      q += len;
      p += (int)(((unsigned)(k + len) + P - 1) / P) - (int)(((unsigned)k + P - 1) / P);
    }
  }
  const int T = (int)q_all, n_new = (int)p_all;
  if (tid == 0) {
    start[R] = T;
    taken[R] = n_new;
    if (first_block) {
      *a.status = 0;
      *a.left = n_free - n_new;
    }
  }
  __syncthreads();
  const int id = blockIdx.x * THREADS + tid, all = gridDim.x * THREADS;
  for (int r = id; r <= R; r += all) {
    a.q_start[r] = start[r];
    if (r < R) a.new_len[r] = kv[r] + start[r + 1] - start[r];
  }
  const int* top = a.free_pages + n_free - 1;
  for (int j = id; j < n_new; j += all) {
    const int r = find(taken, R, j);
    a.table[(size_t)r * a.bt_stride + ((unsigned)kv[r] + P - 1) / P + (j - taken[r])] = top[-j];
  }
  // four tokens a thread: one search, then on from request to request
  for (long long t0 = 4LL * id; t0 < T; t0 += 4LL * all) {
    int r = find(start, R, (int)t0);
    const int n = min(4, T - (int)t0);
    int req[4], pos[4], slot[4];
    int block = -1, page = 0, of = -1;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (i < n) {
        const int t = (int)t0 + i;
        while (t >= start[r + 1]) r++;    // (r < R: t < start[R])
        const int p = kv[r] + t - start[r];
        const int b = (unsigned)p / (unsigned)P;
        if (b != block || r != of) {
          const int held = ((unsigned)kv[r] + P - 1) / P;
          page = b < held ? a.table[(size_t)r * a.bt_stride + b] : top[-(taken[r] + b - held)];
          block = b;
          of = r;
        }
        req[i] = r;
        pos[i] = p;
        slot[i] = page * P + (p - b * P);
      }
    }
    if (a.vec && n == 4) {
      *reinterpret_cast<int4*>(a.token_req + t0) = make_int4(req[0], req[1], req[2], req[3]);
      *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (i < n) {
          a.token_req[t0 + i] = req[i];
          a.positions[t0 + i] = pos[i];
          a.slots[t0 + i] = slot[i];
        }
    }
  }
  __threadfence();                        // (see above: readers that do not wait begin once every block has ended)
}

// `words` words from `at` on.
struct Span {
  const int* at;
  long long words;
  bool meets(const Span& x) const {
    const uintptr_t p = (uintptr_t)at, q = (uintptr_t)x.at;
    return words > 0 && x.words > 0 && p < q + 4 * (uintptr_t)x.words && q < p + 4 * (uintptr_t)words;
  }
};
// Whether what a call may write shares words with anything else of it.  (Every block reads all lengths, and none waits for
// another: block 0 would change them under those that begin later.  Of the table only its rows count, not what lies between.)
bool overlaps(const Args& a) {
  const Span read[] = {{a.q_len, a.R}, {a.kv_len, a.R}, {a.free_pages, a.free_cap}, {a.n_free, 1}};
  const Span written[] = {{a.q_start, a.R + 1LL}, {a.new_len, a.R}, {a.token_req, a.t_cap}, {a.positions, a.t_cap}, {a.slots, a.t_cap},
                          {a.left, 1}, {a.status, 1}};
  auto in_table = [&](const Span& x) {
    const uintptr_t base = (uintptr_t)a.table, end = (uintptr_t)x.at + 4 * (uintptr_t)x.words;
    if (x.words <= 0 || a.R <= 0 || a.bt_width <= 0 || end <= base) return false;
    // the last row that begins before its end
    const uintptr_t pitch = 4 * (uintptr_t)(a.bt_stride > 0 ? a.bt_stride : 1), last = (end - 1 - base) / pitch, rows = (uintptr_t)a.R - 1;
    const Span row = {a.table + (long long)(last < rows ? last : rows) * a.bt_stride, a.bt_width};
    return row.meets(x);
  };
  for (const Span& x : read)
    if (in_table(x)) return true;
  for (const Span& x : written) {
    if (in_table(x)) return true;
    for (const Span& y : read)
      if (x.meets(y)) return true;
    for (const Span& y : written)
      if (&x < &y && x.meets(y)) return true;
  }
  return false;
}
}  // namespace

// Whether arrays of a call overlap as sglc_step_tables does not take them (1 or 0); no memory is touched.
SGLC_API int sglc_step_tables_overlap(const int* q_len, const int* kv_len, const int* free_pages, int free_cap, const int* n_free,
                                      int* table, long long bt_stride, int bt_width, int R, int* q_start, int* new_len,
                                      int* token_req, int* positions, int* slots, int t_cap, int* left, int* status) {
  const Args a = {q_len, kv_len, free_pages, n_free, table, bt_stride, bt_width, free_cap, R, 1, t_cap, q_start, new_len,
                  token_req, positions, slots, left, status, 0};
  return overlaps(a);
}

// All arrays int32.  table [R][bt_stride], bt_width entries a row; free_pages: a stack of free_cap words of which the
// first *n_free are free pages, the top last; t_cap: room for tokens in token_req, positions, slots.  What
// is written lies apart from all else (-4 where it does not).  *status: 0, or why nothing was written: 1 too few pages, 2 a table row too
// short, 4 more tokens than t_cap, 8 a length below zero or beyond 2^31, or n_free outside the stack.
SGLC_API int sglc_step_tables(const int* q_len, const int* kv_len, const int* free_pages, int free_cap, const int* n_free,
                              int* table, long long bt_stride, int bt_width, int R, int page_size, int* q_start, int* new_len,
                              int* token_req, int* positions, int* slots, int t_cap, int* left, int* status,
                              cudaStream_t stream) {
  if (R < 0 || page_size <= 0 || page_size > (1 << 20) || t_cap < 0 || bt_width < 0 || free_cap < 0) return SGLC_ERR_ARGUMENT;
  if (R > MAX_REQUESTS) return SGLC_ERR_UNSUPPORTED;
  const Args a = {q_len, kv_len, free_pages, n_free, table, bt_stride, bt_width, free_cap, R, page_size, t_cap, q_start, new_len,
                  token_req, positions, slots, left, status,
                  (((uintptr_t)token_req | (uintptr_t)positions | (uintptr_t)slots) & 15) == 0};
  if (overlaps(a)) return OVERLAP;
  const size_t smem = (size_t)(3 * R + 2) * 4;
  // The 48 KB that a block has without an attribute are for both kinds of shared memory, the kernel's own words too (from 4,069
  // requests on).  One value for all sizes: two threads may be here at once.
  if (smem + sizeof(Warps) > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (3 * MAX_REQUESTS + 2) * 4);
    if (e != cudaSuccess) return (int)e;
  }
  const long long pieces = ((long long)t_cap + 4 * THREADS - 1) / (4 * THREADS);
  const int blocks = (int)(pieces < 1 ? 1 : pieces > 296 ? 296 : pieces);
  return sglc_launch(step_tables_kernel, dim3(blocks), dim3(THREADS), smem, stream, 1, true, a);
}
