// The page table of a paged K/V cache on the GPU, and the writes into its pages.
//
// A cache of `pages` pages of `page` tokens (a power of two) serves requests of different lengths: request b's
// token t lies in page table[b][t / page], at t % page.  Pages no request holds lie in a stack `free` with `count`
// entries, top last.  A step adds new_lens[b] tokens to every request; its rows lie one request after another (packed,
// or `padded` rows each with the tokens at the end).  All of it is decided here from the lengths on the GPU, so that a
// step can be captured and needs no length on the host.
#include "paged_tiles.h"

namespace qkv {
namespace {

// a request's four words of step state lie in LDS (64 KB); sums over kPlanThreads of pages, or rows, fit an int
constexpr int kMaxRequests = kMaxPlanned;
constexpr int kPlanThreads = 1024;
constexpr int64_t kMaxCount = kMaxPlannedRows;

__device__ __forceinline__ int ceil_pages(int64_t tokens, int shift) {
  return static_cast<int>((tokens + ((1 << shift) - 1)) >> shift);
}

// Inclusive prefix sums of two values over the workgroup's threads; tot_* receive the sums.  Two barriers.
__device__ __forceinline__ void block_scan2(int& x, int& y, int& tot_x, int& tot_y, int* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  x = wave_incl_scan(x);
  y = wave_incl_scan(y);
  __syncthreads();   // the previous scan's readers are done
  if (lane == 63) {
    part[2 * wave] = x;
    part[2 * wave + 1] = y;
  }
  __syncthreads();
  int bx = 0, by = 0;
  tot_x = tot_y = 0;
  for (int w = 0; w < waves; ++w) {
    const int px = part[2 * w], py = part[2 * w + 1];
    if (w < wave) {
      bx += px;
      by += py;
    }
    tot_x += px;
    tot_y += py;
  }
  x += bx;
  y += by;
}

// The last index i of the ascending v[0..n] with v[i] <= x (v[0] <= x).
__device__ __forceinline__ int last_at_most(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

struct PlanArgs {
  const int32_t* new_lens;
  int32_t *table, *lens, *free, *count;
  int64_t table_ld;
  int requests, width, pages, shift, rows, padded;
  int32_t *cu, *kv_lens, *positions, *failed;
  int64_t* slots;
};

// Slot and position of row `row`, which belongs to request b with `end` its first row behind, kv tokens after the step
// (0: not served) and `fresh` of them new; page_of(k) is the request's k-th page.
template <typename F>
__device__ __forceinline__ void put_row(const PlanArgs& a, int row, bool inside, int end, int kv, int fresh, F&& page_of) {
  int pos = -1;
  int64_t slot = -1;
  if (inside && kv > 0) {
    const int p = kv - (end - row);
    if (p >= kv - fresh) {
      pos = p;
      slot = (static_cast<int64_t>(page_of(p >> a.shift)) << a.shift) + (p & ((1 << a.shift) - 1));
    }
  }
  a.positions[row] = pos;
  a.slots[row] = slot;
}

// One workgroup decides the whole step: prefix sums over the requests of the pages they need and of their rows, then
// the page table's new entries, and (WITH_ROWS) every row's slot.
template <bool WITH_ROWS>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
  __shared__ int s_cu[kMaxRequests + 1], s_off[kMaxRequests], s_len[kMaxRequests], s_new[kMaxRequests];
  __shared__ int part[2 * kPlanThreads / 64];
  __shared__ int s_failed;
  const int tid = threadIdx.x;
  if (tid == 0) s_failed = 0;
  const int count = min(max(*a.count, 0), a.pages);
  int row_carry = 0, page_carry = 0, taken = 0;
  for (int b0 = 0; b0 < a.requests; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const bool is = b < a.requests;
    const int len = is ? max(a.lens[b], 0) : 0;
    const int fresh = is ? max(a.new_lens[b], 0) : 0;
    const int have = ceil_pages(len, a.shift), want = ceil_pages(static_cast<int64_t>(len) + fresh, a.shift);
    const bool fits = want <= a.width && (a.padded == 0 || fresh <= a.padded);
    const int need = fits ? min(want - have, a.pages + 1) : 0;
    // a request's rows past the buffer count as one more than the buffer, so that the sums stay in range
    int rows = is ? (a.padded ? a.padded : min(fresh, a.rows + 1)) : 0;
    int up_rows = rows, up_pages = need, tot_rows, tot_pages;
    block_scan2(up_rows, up_pages, tot_rows, tot_pages, part);
    up_rows += row_carry;
    up_pages += page_carry;
    const bool served = fits && (need == 0 || up_pages <= count) && up_rows <= a.rows;
    if (is) {
      s_cu[b] = min(up_rows - rows, a.rows);
      s_off[b] = up_pages - need;
      s_len[b] = len;
      s_new[b] = served ? fresh : -1;
      const int kv = served ? len + fresh : 0;
      a.kv_lens[b] = kv;
      a.cu[b] = s_cu[b];
      if (served) a.lens[b] = kv;
      else if (fresh > 0) atomicAdd(&s_failed, 1);
    }
    row_carry = min(row_carry + tot_rows, a.rows + 1);
    page_carry = min(page_carry + tot_pages, a.pages + 1);
    // pages are taken by the requests up to the last served one that needs some
    int t = served && need > 0 ? up_pages : 0;
    for (int m = 32; m >= 1; m >>= 1) t = max(t, shfl_xor_i(t, m));
    __syncthreads();
    if ((tid & 63) == 0) part[tid >> 6] = t;
    __syncthreads();
    for (int w = 0; w < kPlanThreads / 64; ++w) taken = max(taken, part[w]);
  }
  const int end = min(row_carry, a.rows);
  if (tid == 0) {
    s_cu[a.requests] = end;
    a.cu[a.requests] = end;
    *a.failed = s_failed;
    *a.count = count - taken;
  }
  __syncthreads();
  const int n = a.requests;
  for (int g = tid; g < taken; g += kPlanThreads) {
    const int b = last_at_most(s_off, n - 1, g);
    const int k = ceil_pages(s_len[b], a.shift) + (g - s_off[b]);
    if (s_new[b] >= 0 && k < a.width) a.table[b * a.table_ld + k] = a.free[count - 1 - g];
  }
  if constexpr (WITH_ROWS) {
    for (int row = tid; row < a.rows; row += kPlanThreads) {
      const int b = last_at_most(s_cu, n - 1, row);
      const int fresh = s_new[b], len = s_len[b], have = ceil_pages(len, a.shift);
      put_row(a, row, row < end, s_cu[b + 1], fresh < 0 ? 0 : len + fresh, fresh, [&](int k) -> int {
        // a page of this step comes from the stack, which the launch leaves as it is
        return k < have ? a.table[b * a.table_ld + k] : a.free[count - 1 - (s_off[b] + k - have)];
      });
    }
  }
}

// The rows of a step with many rows, in a launch of its own behind plan_kernel<false>.
__global__ __launch_bounds__(256) void plan_rows_kernel(PlanArgs a) {
  __shared__ int s_cu[kMaxRequests + 1];
  for (int i = threadIdx.x; i <= a.requests; i += 256) s_cu[i] = a.cu[i];
  __syncthreads();
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows) return;
  const int b = last_at_most(s_cu, a.requests - 1, row);
  put_row(a, row, row < s_cu[a.requests], s_cu[b + 1], a.kv_lens[b], max(a.new_lens[b], 0),
          [&](int k) -> int { return a.table[b * a.table_ld + k]; });
}

struct ReleaseArgs {
  const int32_t* keep;
  int32_t *table, *lens, *free, *count;
  int64_t table_ld;
  int requests, width, pages, shift;
};

// Pages behind the first keep[b] tokens go back to the stack, the first of them on top: what the last step took comes
// to lie as it was.
__global__ __launch_bounds__(kPlanThreads) void release_kernel(ReleaseArgs a) {
  __shared__ int s_off[kMaxRequests], s_stay[kMaxRequests];
  __shared__ int part[2 * kPlanThreads / 64];
  const int tid = threadIdx.x;
  const int count = min(max(*a.count, 0), a.pages);
  int carry = 0;
  for (int b0 = 0; b0 < a.requests; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const bool is = b < a.requests;
    const int now = is ? max(a.lens[b], 0) : 0;
    const int keep = is ? min(max(a.keep[b], 0), now) : 0;
    const int have = min(ceil_pages(now, a.shift), a.width), stay = min(ceil_pages(keep, a.shift), have);
    const int gone = min(have - stay, a.pages + 1);
    int up = gone, none = 0, tot, tot_none;
    block_scan2(up, none, tot, tot_none, part);
    if (is) {
      s_off[b] = carry + up - gone;
      s_stay[b] = stay;
      a.lens[b] = keep;
    }
    carry = min(carry + tot, a.pages + 1);
  }
  __syncthreads();
  const int total = min(carry, a.pages - count);   // more cannot have been taken
  if (tid == 0) *a.count = count + total;
  for (int g = tid; g < total; g += kPlanThreads) {
    const int b = last_at_most(s_off, a.requests - 1, g);
    const int k = s_stay[b] + (g - s_off[b]);
    if (k < a.width) {
      int32_t* e = a.table + b * a.table_ld + k;
      a.free[count + total - 1 - g] = *e;
      *e = -1;
    }
  }
}

struct ShareArgs {
  const int32_t *parents, *cu, *kv_lens, *lens;
  int requests, rows;
  SharedPlan p;
};
constexpr uint32_t kNobody = 0xFFFFFFFFu;

// Request b's parent, or -1; its rows, and how many of them, the last ones, have a token.
struct Heir {
  int parent, end, rows, tokens;
};
__device__ __forceinline__ Heir heir_of(const ShareArgs& a, int b) {
  const int row0 = min(max(a.cu[b], 0), a.rows);
  Heir h;
  h.end = min(max(a.cu[b + 1], row0), a.rows);
  h.rows = h.end - row0;
  h.tokens = min(h.rows, max(a.kv_lens[b], 0));
  h.parent = a.parents[b];
  // a parent without tokens is none, nor is a request's own
  if (static_cast<unsigned>(h.parent) >= static_cast<unsigned>(a.requests) || h.parent == b || a.lens[h.parent] <= 0 ||
      a.kv_lens[b] <= 0)
    h.parent = -1;
  return h;
}

// What is known of a row: its position, its place among its parent's heirs, the heir at that place.
__device__ __forceinline__ void put_shared_row(const ShareArgs& a, const int* cu, int row) {
  int pos = -1, rank = -2;
  const int b = last_at_most(cu, a.requests - 1, row);
  if (row >= cu[0] && row < cu[a.requests]) {
    const Heir h = heir_of(a, b);
    rank = -1;
    const int nth = row - (h.end - h.tokens);
    if (nth >= 0 && row < h.end) {
      pos = a.p.before[b] + max(a.kv_lens[b], 0) - (h.end - row);
      if (h.parent >= 0 && a.p.starts[b] + nth < a.rows) {   // always so where cu_rows ascends
        rank = a.p.starts[b] + nth;
        a.p.order[rank] = row;
      }
    }
  }
  a.p.positions[row] = pos;
  a.p.rank[row] = rank;
}

// One workgroup sorts the requests by parent, then by themselves (keys differ, so the order is one whatever runs first),
// and prefix sums of their tokens give every heir its place.
template <bool WITH_ROWS>
__global__ __launch_bounds__(kPlanThreads) void share_kernel(ShareArgs a) {
  __shared__ uint32_t s_key[kMaxRequests];
  __shared__ int s_start[kMaxRequests], s_cu[kMaxRequests + 1];
  __shared__ int part[2 * kPlanThreads / 64];
  const int tid = threadIdx.x;
  int n = 1;
  while (n < a.requests) n <<= 1;
  for (int b = tid; b < n; b += kPlanThreads) {
    uint32_t key = kNobody;
    if (b < a.requests) {
      const Heir h = heir_of(a, b);
      if (h.parent >= 0 && h.tokens > 0) key = static_cast<uint32_t>(h.parent) << 12 | static_cast<uint32_t>(b);
      s_cu[b] = h.end - h.rows;
      if (b == a.requests - 1) s_cu[a.requests] = h.end;
      a.p.before[b] = h.parent >= 0 ? a.lens[h.parent] : 0;
      a.p.parent_lens[b] = max(a.lens[b], 0);
      a.p.starts[b] = 0;
    }
    s_key[b] = key;
  }
  __syncthreads();
  for (int k = 2; k <= n; k <<= 1)   // bitonic: ascending runs of k keys
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = tid; i < n; i += kPlanThreads) {
        const int other = i ^ j;
        if (other > i) {
          const uint32_t x = s_key[i], y = s_key[other];
          if ((x > y) == ((i & k) == 0)) {
            s_key[i] = y;
            s_key[other] = x;
          }
        }
      }
      __syncthreads();
    }
  int carry = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const uint32_t key = i < n ? s_key[i] : kNobody;
    const int b = static_cast<int>(key & 4095u);
    const int m = key == kNobody ? 0 : heir_of(a, b).tokens;
    int up = m, none = 0, tot, tot_none;
    block_scan2(up, none, tot, tot_none, part);
    if (i < n) s_start[i] = carry + up - m;
    if (key != kNobody) a.p.starts[b] = carry + up - m;
    carry += tot;
  }
  __syncthreads();
  for (int p = tid; p <= a.requests; p += kPlanThreads) {
    int lo = 0, hi = n;   // the first key of parent p or a later one
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_key[mid] != kNobody && s_key[mid] >> 12 < static_cast<uint32_t>(p)) lo = mid + 1;
      else hi = mid;
    }
    a.p.heirs_cu[p] = lo < n && s_key[lo] != kNobody ? s_start[lo] : carry;
  }
  if constexpr (WITH_ROWS) {
    __threadfence_block();
    __syncthreads();   // before and starts, which this workgroup wrote
    for (int row = tid; row < a.rows; row += kPlanThreads) put_shared_row(a, s_cu, row);
  }
}

// The same for at most kCounted requests: an heir's place is the sum of the tokens of all requests before its own in that
// order, added up one by one; no sort, and two barriers (5 requests: 2.3 us, 65: 3.7; 512 take 18, as 513 do sorted).
constexpr int kCounted = 512;
template <bool WITH_ROWS>
__global__ __launch_bounds__(kPlanThreads) void share_few_kernel(ShareArgs a) {
  __shared__ __attribute__((aligned(16))) uint2 s_heir[kCounted];   // key, tokens
  __shared__ int s_cu[kCounted + 1], s_start[kCounted], s_before[kCounted], s_kv[kCounted], s_end[kCounted];
  const int tid = threadIdx.x;
  const int even = (a.requests + 1) & -2;
  for (int b = tid; b < even; b += blockDim.x) {
    uint2 heir = make_uint2(kNobody, 0u);
    if (b < a.requests) {
      const Heir h = heir_of(a, b);
      const int own = max(a.lens[b], 0);
      if (h.parent >= 0 && h.tokens > 0) heir = make_uint2(static_cast<uint32_t>(h.parent) << 12 | static_cast<uint32_t>(b), h.tokens);
      s_cu[b] = h.end - h.rows;
      if (b == a.requests - 1) s_cu[a.requests] = h.end;
      s_before[b] = h.parent >= 0 ? a.lens[h.parent] : 0;
      s_kv[b] = max(a.kv_lens[b], 0);
      s_end[b] = h.end;
      a.p.before[b] = s_before[b];
      a.p.parent_lens[b] = own;
    }
    s_heir[b] = heir;
  }
  __syncthreads();
  for (int b = tid; b <= a.requests; b += blockDim.x) {
    const uint32_t mine = b < a.requests ? s_heir[b].x : 0u, first = static_cast<uint32_t>(b) << 12;
    uint32_t start = 0, heirs = 0;
#pragma unroll 4
    for (int i = 0; i < even; i += 2) {
      const uint4 two = *reinterpret_cast<const uint4*>(s_heir + i);
      start += (two.x < mine ? two.y : 0u) + (two.z < mine ? two.w : 0u);
      heirs += (two.x < first ? two.y : 0u) + (two.z < first ? two.w : 0u);
    }
    a.p.heirs_cu[b] = static_cast<int>(heirs);
    if (b < a.requests) {
      s_start[b] = static_cast<int>(start);
      a.p.starts[b] = mine == kNobody ? 0 : static_cast<int>(start);
    }
  }
  if constexpr (WITH_ROWS) {
    __syncthreads();
    for (int row = tid; row < a.rows; row += blockDim.x) {
      int pos = -1, rank = -2;
      if (row >= s_cu[0] && row < s_cu[a.requests]) {
        const int b = last_at_most(s_cu, a.requests - 1, row);
        rank = -1;
        const int back = s_end[b] - row;   // 1: the last one
        if (back > 0 && back <= s_kv[b]) {
          pos = s_before[b] + s_kv[b] - back;
          const int place = s_start[b] + static_cast<int>(s_heir[b].y) - back;
          if (s_heir[b].x != kNobody && place < a.rows) {   // always so where cu_rows ascends
            rank = place;
            a.p.order[place] = row;
          }
        }
      }
      a.p.positions[row] = pos;
      a.p.rank[row] = rank;
    }
  }
}

__global__ __launch_bounds__(256) void share_rows_kernel(ShareArgs a) {
  __shared__ int s_cu[kMaxRequests + 1];
  for (int i = threadIdx.x; i <= a.requests; i += 256) s_cu[i] = min(max(a.cu[i], 0), a.rows);
  __syncthreads();
  const int row = blockIdx.x * 256 + threadIdx.x;
  if (row < a.rows) put_shared_row(a, s_cu, row);
}

struct AppendArgs {
  const uint16_t *k, *v;
  uint16_t *kp, *vp;
  int64_t k_row, k_head, v_row, v_head;
  int64_t kp_page, kp_head, kp_tok, vp_page, vp_head, vp_tok;
  const int64_t* slots;
  int64_t units, n_slots;   // 16-byte units of K (as many of V); slots of the cache
  int units_head, units_row, shift;
};

// 16 bytes of K and of V a thread: a row's units lie in a row of the source and, head by head, in a page.
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (u >= a.units) return;
  const int64_t row = u / a.units_row;
  const int in_row = static_cast<int>(u - row * a.units_row);
  const int head = in_row / a.units_head, c = 8 * (in_row - head * a.units_head);
  const int64_t slot = a.slots[row];
  if (slot < 0 || slot >= a.n_slots) return;
  const int64_t page = slot >> a.shift, at = slot & ((1 << a.shift) - 1);
  const uint4 x = load16u(a.k + row * a.k_row + head * a.k_head + c);
  const uint4 y = load16u(a.v + row * a.v_row + head * a.v_head + c);
  *reinterpret_cast<uint4*>(a.kp + page * a.kp_page + head * a.kp_head + at * a.kp_tok + c) = x;
  *reinterpret_cast<uint4*>(a.vp + page * a.vp_page + head * a.vp_head + at * a.vp_tok + c) = y;
}

// Rows up to which the one workgroup of plan_kernel also writes the slots.
constexpr int64_t kPlanRowsInOne = 4096;

int check_table(const char* what, const void* table, int64_t table_ld, const void* lens, const void* free,
                const void* count, int64_t requests, int64_t width, int64_t pages, int64_t page) {
  if (!table || !lens || !free || !count) return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  if (requests < 1 || width < 1 || table_ld < width || pages < 1)
    return fail(QKV_ERR_INVALID, "%s: bad sizes", what);
  if (pages > kMaxCount)
    return fail(QKV_ERR_UNSUPPORTED, "%s: at most %lld pages", what, static_cast<long long>(kMaxCount));
  if (page < 16 || page > 4096 || (page & (page - 1)))
    return fail(QKV_ERR_UNSUPPORTED, "%s: page must be a power of two in [16, 4096], got %lld", what,
                static_cast<long long>(page));
  if (requests > kMaxRequests)
    return fail(QKV_ERR_UNSUPPORTED, "%s: at most %d requests, got %lld", what, kMaxRequests,
                static_cast<long long>(requests));
  if (width > (1ll << 30) / page) return fail(QKV_ERR_UNSUPPORTED, "%s: a table row covers at most 2^30 tokens", what);
  return QKV_OK;
}

}  // namespace
}  // namespace qkv

using namespace qkv;

QKV_EXPORT int qkv_paged_plan(const int32_t* new_lens, int32_t* table, int64_t table_ld, int32_t* lens, int32_t* free,
                              int32_t* count, int64_t requests, int64_t width, int64_t pages, int64_t page,
                              int64_t rows, int64_t padded, int32_t* cu_rows, int32_t* kv_lens, int64_t* slots,
                              int32_t* positions, int32_t* failed, void* stream) {
  const char* what = "qkv_paged_plan";
  if (const int rc = check_table(what, table, table_ld, lens, free, count, requests, width, pages, page)) return rc;
  if (!new_lens || !cu_rows || !kv_lens || !slots || !positions || !failed)
    return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  if (rows > kMaxCount) return fail(QKV_ERR_UNSUPPORTED, "%s: at most %lld rows", what, static_cast<long long>(kMaxCount));
  if (rows < 1 || padded < 0 || (padded > 0 && requests * padded != rows))
    return fail(QKV_ERR_INVALID, "%s: bad sizes (rows must be requests * padded where padded is given)", what);
  PlanArgs a{new_lens, table, lens, free, count, table_ld, static_cast<int>(requests), static_cast<int>(width),
             static_cast<int>(pages), __builtin_ctz(static_cast<unsigned>(page)), static_cast<int>(rows),
             static_cast<int>(padded), cu_rows, kv_lens, positions, failed, slots};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows <= kPlanRowsInOne) {
    plan_kernel<true><<<1, kPlanThreads, 0, st>>>(a);
  } else {
    plan_kernel<false><<<1, kPlanThreads, 0, st>>>(a);
    plan_rows_kernel<<<static_cast<unsigned>(cdiv(rows, 256)), 256, 0, st>>>(a);
  }
  return check_launch(what);
}

QKV_EXPORT int qkv_paged_release(const int32_t* keep, int32_t* table, int64_t table_ld, int32_t* lens, int32_t* free,
                                 int32_t* count, int64_t requests, int64_t width, int64_t pages, int64_t page,
                                 void* stream) {
  const char* what = "qkv_paged_release";
  if (const int rc = check_table(what, table, table_ld, lens, free, count, requests, width, pages, page)) return rc;
  if (!keep) return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  ReleaseArgs a{keep, table, lens, free, count, table_ld, static_cast<int>(requests), static_cast<int>(width),
                static_cast<int>(pages), __builtin_ctz(static_cast<unsigned>(page))};
  release_kernel<<<1, kPlanThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  return check_launch(what);
}

QKV_EXPORT int qkv_paged_append(const void* key, const int64_t* key_strides, const void* value,
                                const int64_t* value_strides, void* k_pages, const int64_t* k_strides, void* v_pages,
                                const int64_t* v_strides, int64_t pages, int64_t page, int64_t kv_heads,
                                int64_t head_dim, const int64_t* slots, int64_t rows, void* stream) {
  const char* what = "qkv_paged_append";
  if (!key_strides || !value_strides || !k_pages || !k_strides || !v_pages || !v_strides ||
      (rows > 0 && (!key || !value || !slots)))
    return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  if (rows < 0 || rows > (1 << 30) || pages < 1 || pages > (1ll << 30) || kv_heads < 1 || kv_heads > 65536 ||
      head_dim < 8 || head_dim > 65536 || head_dim % 8)
    return fail(QKV_ERR_INVALID, "%s: bad sizes (head_dim must be a multiple of 8)", what);
  if (page < 16 || page > 4096 || (page & (page - 1)))
    return fail(QKV_ERR_UNSUPPORTED, "%s: page must be a power of two in [16, 4096], got %lld", what,
                static_cast<long long>(page));
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 || v_strides[i] % 8 || !aligned(k_pages, 16) || !aligned(v_pages, 16))
      return fail(QKV_ERR_INVALID, "%s: page rows must be 16-byte aligned", what);
  if (rows == 0) return QKV_OK;
  const int64_t units_head = head_dim / 8, units_row = units_head * kv_heads;
  AppendArgs a{static_cast<const uint16_t*>(key), static_cast<const uint16_t*>(value),
               static_cast<uint16_t*>(k_pages), static_cast<uint16_t*>(v_pages),
               key_strides[0], key_strides[1], value_strides[0], value_strides[1],
               k_strides[0], k_strides[1], k_strides[2], v_strides[0], v_strides[1], v_strides[2],
               slots, rows * units_row, pages * page, static_cast<int>(units_head), static_cast<int>(units_row),
               __builtin_ctz(static_cast<unsigned>(page))};
  const int64_t grid = cdiv(a.units, 256);
  // a grid has less than 2^32 threads
  if (grid >= (1 << 24)) return fail(QKV_ERR_UNSUPPORTED, "%s: too many rows", what);
  append_kernel<<<static_cast<unsigned>(grid), 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return check_launch(what);
}

QKV_EXPORT int64_t qkv_paged_share_words(int64_t rows, int64_t requests) {
  if (rows < 1 || rows > kMaxCount || requests < 1 || requests > kMaxRequests) return -1;
  return SharedPlan::words(rows, requests);
}

QKV_EXPORT int qkv_paged_share(const int32_t* parents, const int32_t* cu_rows, const int32_t* kv_lens,
                               const int32_t* lens, int64_t requests, int64_t rows, int32_t* shared, void* stream) {
  const char* what = "qkv_paged_share";
  if (!parents || !cu_rows || !kv_lens || !lens || !shared) return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  if (qkv_paged_share_words(rows, requests) < 0)
    return fail(QKV_ERR_UNSUPPORTED, "%s: 1 to %d requests and 1 to %lld rows, got %lld and %lld", what, kMaxRequests,
                static_cast<long long>(kMaxCount), static_cast<long long>(requests), static_cast<long long>(rows));
  ShareArgs a{parents, cu_rows, kv_lens, lens, static_cast<int>(requests), static_cast<int>(rows),
              SharedPlan(shared, rows, requests)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool few = requests <= kCounted, one = rows <= kPlanRowsInOne;
  // (a row's search takes longer than a request's count)
  const unsigned threads = few && requests <= 256 && (rows <= 256 || !one) ? 256 : kPlanThreads;
  if (few && one) share_few_kernel<true><<<1, threads, 0, st>>>(a);
  else if (few) share_few_kernel<false><<<1, threads, 0, st>>>(a);
  else if (one) share_kernel<true><<<1, threads, 0, st>>>(a);
  else share_kernel<false><<<1, threads, 0, st>>>(a);
  if (!one) {
    share_rows_kernel<<<static_cast<unsigned>(cdiv(rows, 256)), 256, 0, st>>>(a);
  }
  return check_launch(what);
}
