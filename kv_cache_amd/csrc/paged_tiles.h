// What the attention kernels over a paged K/V cache share: a workgroup's search of its work, the rows of a tile and what
// they see, the score forms, the bodies of the two kernels, the joining of parts, and the shapes of their launches.
// Described in paged_attention.hip.
#pragma once

#include "attend.h"

namespace qkv {

constexpr int kMaxPlanned = 4096;             // requests of a planned step
constexpr int64_t kMaxPlannedRows = 1 << 20;   // and its rows (or pages)

// The rows of requests that continue another request's tokens, their parent's, gathered by parent (paged.hip writes it,
// int32 words from one address).  Row order[i] of heirs_cu[a] <= i < heirs_cu[a + 1] is a's heir and sees its
// parent_lens[a] tokens; rank is order's inverse (-1: a row without a parent or token, -2: no request's row).  before[b]
// tokens come before request b's own, so that its row is at positions[row] (-1 without a token).  starts[b]: the place
// of b's first heir.
struct SharedPlan {
  int32_t *positions, *rank, *order, *heirs_cu, *starts, *parent_lens, *before;
  SharedPlan(int32_t* at, int64_t rows, int64_t requests)
      : positions(at), rank(at + rows), order(at + 2 * rows), heirs_cu(at + 3 * rows), starts(heirs_cu + requests + 1),
        parent_lens(starts + requests), before(parent_lens + requests) {}
  static int64_t words(int64_t rows, int64_t requests) { return 3 * rows + 4 * requests + 1; }
};

// A call of the attention over pages as the C interface takes it.
struct PagedCall {
  const void* query;
  const int64_t* q_strides;
  const void *k_pages, *v_pages;
  const int64_t* page_strides;
  const void *k_scales, *v_scales;
  const int64_t* scale_strides;
  int64_t pages, page;
  const int32_t* table;
  int64_t table_ld, width, requests;
  const int32_t *cu_rows, *kv_lens;
  int64_t rows, max_rows, q_heads, kv_heads, head_dim;
  float scaling, softcap;
  const float* slopes;
  const int32_t *prefix_lens, *first_keys;
  void* workspace;
  int64_t workspace_bytes;
  void* out;
  const int64_t* out_strides;
  int dtype;
  void* stream;
};
// Over codes: the kernels of each format are compiled in a file of their own.
int paged_call_fp8(const PagedCall& c, const char* what);
int paged_call_fp4(const PagedCall& c, const char* what);
int shared_call_fp8(const PagedCall& c, const int32_t* plan, const char* what);
int shared_call_fp4(const PagedCall& c, const int32_t* plan, const char* what);

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;      // keys per step of the rows kernel; splits are multiples of it
constexpr int kRowsM = 128;    // rows of a tile of the rows kernel
constexpr int kTokenM = 16;    // rows of a column set of the token kernel, which has one or two
constexpr int kRound = 512;    // workgroups that run at once: two a CU
// Three a CU of the token kernel with one column set over rows of at most 64 bytes (29 requests of up to 32001 keys in fp4:
// 152 us, 170 with two; over the 128 bytes of fp8 two are as fast or faster, 8 requests of up to 16384 keys 46.8 and 49.9).
constexpr int kShortRound = 768, kShortRow = 64;
constexpr int kRowsJoins = 8, kTokenJoins = 4;   // workgroups that join a tile's parts; of a column set's
constexpr int kStep = 32;      // keys a wave of the token kernel takes at a time
// The weights exp(s - m) are rounded to the dtype for the product with V, half a step each (2^-8 in bf16, 2^-11 in
// fp16): the matrix instruction takes both operands in one 16-bit type, and a second product for what the rounding took
// would double that half of the matrix work.  The sums are of the rounded weights, so that V is weighted by a partition
// of one.  Scores, maxima, sums and outputs stay in 32 bits (one token over 500 keys, bf16, against 64 bits: off by 2.8e-4
// on average, 2.0e-4 with weights in 32 bits; by 6.1e-3 at most either way, the output's own rounding).
// fp16 weights are scaled by 2^6: they stay below 2^14 (lazy rescaling lets them reach 2^8) and normal down to 2^-20
// of the row's largest, so that the small weights of long rows keep their bits.
template <bool F16>
constexpr float kShift = F16 ? 6.0f : 0.0f;

template <bool F16>
constexpr uint32_t kOnes = F16 ? 0x3C003C00u : 0x3F803F80u;   // a pair of 1.0

// What pages hold: 16-bit values, or codes of 8 or 4 bits (e4m3, e2m1 with the even channel in the low half) whose
// blocks of 32 channels have a scale byte s each: a code stands for its value times 2^(s - 127), s = 255 for NaN.
constexpr int kHalfPages = 0, kFp8Pages = 1, kFp4Pages = 2;
constexpr int kScaleBlock = 32;

struct PagedArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  int64_t q_row, q_head, page, head, o_row, o_head;   // strides; pages of K and V share theirs (codes: in bytes)
  uint32_t tok;                                       // (page * tok fits 31 bits)
  const int32_t *table, *cu, *kv_lens, *prefix, *first;
  const float* slopes;
  int64_t table_ld;
  int width, pages, shift, requests, rows, kv_heads, group;
  int per_group;            // 65536 / group + 1: i * per_group >> 16 is i / group for rows of a tile (i < 128)
  float scale_log2, tanh_scale, cap_log2;   // scaling * log2(e); 2 * scaling / cap * log2(e); cap * log2(e)
  // Scores are kept as products q.k, or in log2 units where there is a cap: what takes them to log2 units, and a slope
  // to theirs.
  float unit_log2, slope_unit;
  int wide;                                 // the cap is larger than kNearCap
  const uint8_t *k_scales, *v_scales;       // of codes: [pages][head][token][block], the last two without gaps
  int64_t s_page, s_head;                   // their strides
  // Requests that continue another's tokens (SharedPlan).  at: for every (row, KV head), then for every (place in order,
  // KV head), where its parts lie.
  const int32_t *order, *rank, *heirs_cu, *parent_lens, *before, *positions;
  int2* at;
};

// What one class of requests is worked by: tiles of `tokens` tokens, for requests of more than `above` and at most
// `most` rows, split along the keys into chunks of at least `min_keys`.
struct PagedClass {
  int tokens, above, most, min_keys;
  int round;           // workgroups that run at once
  float per_round;     // 1.0001 / round
  int finer;           // more than one round of chunks where one does not come out even
  int max_parts;       // parts the workspace holds
  int max_joins;       // items of the kernel that joins them
  float *acc, *ml;     // them: weighted values, then (maximum, sum)
};

// A workgroup's work.
struct Where {
  int b, tile, head, split, n_split, part, row0, n_rows, kv, chunk;
  int heirs, alone;   // where requests share: rows are those of b's heirs; b has no parent
};

__device__ __forceinline__ int rows_of(const PagedArgs& a, int b, int& row0) {
  row0 = min(max(a.cu[b], 0), a.rows);
  return min(max(a.cu[b + 1], row0), a.rows) - row0;
}

// Sum (wave total in lane 63) and maximum over the wave by DPP moves within rows of 16 lanes and across them: a
// shuffle through LDS takes several times as long, and locate and the kernels' heads are chains of these.
__device__ __forceinline__ int wave_scan(int v) {   // inclusive prefix sum
  auto add = [&](auto ctrl, auto rows) {
    v += __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});   // row_shr 1, 2, 4, 8
  add(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});   // row_bcast 15 and 31
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});
  return v;
}
__device__ __forceinline__ float lane63(float v) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_total(float v) {
  auto add = [&](auto ctrl, auto rows) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, decltype(rows)::value,
                                                    0xF, false));
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});
  return lane63(v);
}
__device__ __forceinline__ int wave_max_i(int x) {
  auto fold = [&](auto ctrl, auto rows) {
    x = max(x, static_cast<int>(dpp_mov<decltype(ctrl)::value, decltype(rows)::value>(static_cast<uint32_t>(x),
                                                                                      static_cast<uint32_t>(x))));
  };
  using std::integral_constant;
  fold(integral_constant<int, 0xB1>{}, integral_constant<int, 0xF>{});   // quad_perm, then row mirrors
  fold(integral_constant<int, 0x4E>{}, integral_constant<int, 0xF>{});
  fold(integral_constant<int, 0x141>{}, integral_constant<int, 0xF>{});
  fold(integral_constant<int, 0x140>{}, integral_constant<int, 0xF>{});
  fold(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});
  fold(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});
  return __builtin_amdgcn_readlane(x, 63);
}

// Which (request, tile, KV head, chunk of keys) workgroup `item` of a class has; false if there are fewer.  Every
// workgroup derives it from the lengths: the total work W = sum_b tiles_b * keys_b * heads over the workgroups that run
// at once gives the keys of a chunk, C (chunk_of); request b is split into S_b = ceil(keys_b / C), and an
// exclusive prefix sum of tiles_b * heads * S_b over the requests gives its first item.  PER_TILE: items are the
// (tile, head) of requests with S_b > 1 only, for the kernel that joins the parts.
// The head runs fastest (consecutive workgroups go to different XCDs, so that with 8 KV heads an XCD's L2 serves one
// head), then the tile from the last one on (under a causal mask the longest).
// W is taken in fp32, every workgroup in the same order, and C a ten-thousandth larger, so that W / C stays below its
// bound whatever was rounded.  Up to 64 requests every wave does it for itself (four requests a lane, so that 256 do,
// took 100 requests of up to 2000 keys from 114 to 120 us).
template <bool PER_TILE>
__device__ __forceinline__ bool locate(const PagedArgs& a, const PagedClass& c, int item, Where& w) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  struct Share {
    int nt, keys, row0, n_rows;
  };
  auto share_of = [&](int b) {
    Share s{0, 0, 0, 0};
    if (b < a.requests) {
      s.n_rows = rows_of(a, b, s.row0);
      if (s.n_rows > c.above && s.n_rows <= c.most) {
        s.nt = (s.n_rows + c.tokens - 1) / c.tokens;
        s.keys = static_cast<int>(min(static_cast<int64_t>(max(a.kv_lens[b], 0)), static_cast<int64_t>(a.width) << a.shift));
      }
    }
    return s;
  };
  auto round_up = [&](float keys) {
    const int least = max(c.min_keys, static_cast<int>(fminf(keys, 1073741824.0f)) + 1);   // no request has more than 2^30 keys
    return __builtin_amdgcn_readfirstlane((least + kTile - 1) & -kTile);
  };
  // `per` keys for each of the workgroups that run at once.  One round of them is best where it comes out even (one
  // request of 131011 keys: 92 us, 97 in two rounds).  The last chunks of several requests differ, and a second round
  // of a few workgroups costs as much as a full one: then two rounds, or three where chunks stay above 2048 keys (32
  // requests of up to 32768: 574, 543, 527 us with one, two, three; 8 of up to 16384: two 82, three 85).
  auto chunk_of = [&](float per) { return round_up(fmaxf(per * (1.0f / 3.0f), fminf(per * 0.5f, 2048.0f))); };
  auto splits_of = [&](const Share& s, int chunk) { return s.keys > chunk ? (s.keys + chunk - 1) / chunk : 1; };
  int at, part, nt;
  if (a.requests <= 64) {
    const Share s = share_of(lane);
    const float per = wave_total(static_cast<float>(s.nt) * static_cast<float>(s.keys)) * a.kv_heads * c.per_round;
    w.chunk = round_up(per);
    if (c.finer) {
      // the shortest chunks, up to a fifth longer, that make one round (4 requests of up to 30000 keys: 70 us, 74 in
      // two; 8 of up to 16384: 77, 80 with chunks that make a little more than one)
      const int tiles = s.nt * a.kv_heads;
      int i = 0;
      for (; i < 4; ++i) {
        w.chunk = round_up(per * (1.0f + 0.0667f * i));
        // without a division: one more or less is near enough to choose by
        const int ns = static_cast<int>(static_cast<float>(s.keys - 1) * __builtin_amdgcn_rcpf(static_cast<float>(w.chunk))) + 1;
        if (__builtin_amdgcn_readlane(wave_scan(tiles * ns), 63) <= c.round) break;
      }
      if (i == 4) w.chunk = chunk_of(per);
    }
    const int ns = splits_of(s, w.chunk), tiles = s.nt * a.kv_heads;
    const int parts = ns > 1 ? tiles * ns : 0, items = PER_TILE ? (ns > 1 ? tiles : 0) : tiles * ns;
    const int begin = wave_scan(items) - items, part_begin = wave_scan(parts) - parts;
    const uint64_t hit = __ballot(item >= begin && item - begin < items);
    if (!hit) return false;
    w.b = __builtin_ctzll(hit);
    at = item - __builtin_amdgcn_readlane(begin, w.b);
    part = __builtin_amdgcn_readlane(part_begin, w.b);
    nt = __builtin_amdgcn_readlane(s.nt, w.b);
    w.kv = __builtin_amdgcn_readlane(s.keys, w.b);
    w.n_split = __builtin_amdgcn_readlane(ns, w.b);
    w.row0 = __builtin_amdgcn_readlane(s.row0, w.b);
    w.n_rows = __builtin_amdgcn_readlane(s.n_rows, w.b);
  } else {
    __shared__ float s_tot[4];
    __shared__ int s_part[8], s_hit[8];
    float total = 0.0f;
    for (int b0 = 0; b0 < a.requests; b0 += 256) {
      const Share s = share_of(b0 + tid);
      total += static_cast<float>(s.nt) * static_cast<float>(s.keys);
    }
    total = wave_total(total);
    if (lane == 0) s_tot[wave] = total;
    if (tid == 0) s_hit[0] = -1;
    __syncthreads();
    const float per = ((s_tot[0] + s_tot[1]) + (s_tot[2] + s_tot[3])) * a.kv_heads * c.per_round;
    w.chunk = c.finer ? chunk_of(per) : round_up(per);
    int carry = 0, part_carry = 0;
    for (int b0 = 0; b0 < a.requests; b0 += 256) {
      const Share s = share_of(b0 + tid);
      const int ns = splits_of(s, w.chunk), tiles = s.nt * a.kv_heads;
      const int parts = ns > 1 ? tiles * ns : 0, items = PER_TILE ? (ns > 1 ? tiles : 0) : tiles * ns;
      const int up = wave_scan(items), up_part = wave_scan(parts);
      if (lane == 63) {
        s_part[2 * wave] = up;
        s_part[2 * wave + 1] = up_part;
      }
      __syncthreads();
      int begin = carry + up - items, part_begin = part_carry + up_part - parts;
      for (int i = 0; i < 4; ++i) {
        if (i < wave) {
          begin += s_part[2 * i];
          part_begin += s_part[2 * i + 1];
        }
        carry += s_part[2 * i];
        part_carry += s_part[2 * i + 1];
      }
      if (item >= begin && item - begin < items) {   // one thread at most
        s_hit[0] = b0 + tid;
        s_hit[1] = item - begin;
        s_hit[2] = part_begin;
        s_hit[3] = s.nt;
        s_hit[4] = s.keys;
        s_hit[5] = ns;
        s_hit[6] = s.row0;
        s_hit[7] = s.n_rows;
      }
      __syncthreads();
      if (s_hit[0] >= 0 || item < carry) break;   // the same for every thread
    }
    w.b = __builtin_amdgcn_readfirstlane(s_hit[0]);
    if (w.b < 0) return false;
    at = __builtin_amdgcn_readfirstlane(s_hit[1]);
    part = __builtin_amdgcn_readfirstlane(s_hit[2]);
    nt = __builtin_amdgcn_readfirstlane(s_hit[3]);
    w.kv = __builtin_amdgcn_readfirstlane(s_hit[4]);
    w.n_split = __builtin_amdgcn_readfirstlane(s_hit[5]);
    w.row0 = __builtin_amdgcn_readfirstlane(s_hit[6]);
    w.n_rows = __builtin_amdgcn_readfirstlane(s_hit[7]);
  }
  // divisions are done by the vector unit; what they give is the same in every lane
  const int rest = __builtin_amdgcn_readfirstlane(at / a.kv_heads);
  w.head = at - rest * a.kv_heads;
  w.split = __builtin_amdgcn_readfirstlane(rest / nt);
  w.tile = nt - 1 - (rest - w.split * nt);
  w.part = part + (w.head * nt + w.tile) * w.n_split;
  // always so where cu_rows ascends; otherwise nothing is written out of bounds
  if (w.n_split > 1 && (w.part < 0 || w.part > c.max_parts - w.n_split)) return false;
  if (!PER_TILE) w.part += w.split;
  return true;
}

// What a lane needs of its row: the keys [lo, hi) it sees, its position, its score bias.
struct Row {
  int64_t q_at, o_at;   // its offsets in q and out
  int lo, hi, pos;
  float slope;          // slope in the units that the scores are kept in
  bool on;
};

// Tokens before the own ones of w's request.
template <bool SH>
__device__ __forceinline__ int before_of(const PagedArgs& a, const Where& w) {
  return SH && !w.heirs ? max(a.before[w.b], 0) : 0;
}
// Keys, among those that w counts, that every row sees; the first one that row `row` sees.
template <bool SH>
__device__ __forceinline__ int prefix_of(const PagedArgs& a, const Where& w) {
  return a.prefix ? max(a.prefix[w.b], 0) - before_of<SH>(a, w) : 0;
}
template <bool SH>
__device__ __forceinline__ int first_of(const PagedArgs& a, const Where& w, int64_t row) {
  return max(0, max(0, a.first[row]) - before_of<SH>(a, w));
}

// Row `i` of the tile, G heads a token.  A row the tile does not have sees everything, so that it asks for no mask.
template <bool FORM, bool SH = false>
__device__ __forceinline__ Row row_of(const PagedArgs& a, const PagedClass& c, const Where& w, int i) {
  const int t = i * a.per_group >> 16, g = i - t * a.group;
  const int token = w.tile * c.tokens + t;
  Row r;
  r.on = t < c.tokens && token < w.n_rows;
  int64_t row = w.row0 + (r.on ? token : 0);
  if (SH && w.heirs) row = min(max(a.order[row], 0), a.rows - 1);
  const int head = w.head * a.group + (r.on ? g : 0);
  r.q_at = row * a.q_row + head * a.q_head;
  r.o_at = row * a.o_row + head * a.o_head;
  r.lo = 0;
  r.hi = 0x7FFFFFFF;
  r.slope = 0.0f;
  if (SH && w.heirs) {
    r.pos = FORM && a.slopes ? a.positions[row] : 0;
    if (r.on) r.hi = w.kv;
  } else {
    r.pos = a.kv_lens[w.b] - w.n_rows + token;
  }
  if (r.on) {
    if (!(SH && w.heirs)) {
      r.hi = 0;
      if (r.pos >= 0) r.hi = min(w.kv, max(r.pos + 1, prefix_of<SH>(a, w)));
    }
    if (a.first) r.lo = first_of<SH>(a, w, row);
    if (FORM && a.slopes) r.slope = a.slope_unit * a.slopes[head];
  }
  return r;
}

// cap * tanh(x / cap) in log2 units, of a product q.k.  Near: 1 - 2 / (exp(2x) + 1), in error by 2^-22 of the cap or
// so, which for caps up to kNearCap is below 2^-14.  For larger ones that error would show, and small x take the odd
// polynomial (next term x^11 / 113: below 2^-26 of x at 0.25).
constexpr float kNearCap = 256.0f;
__device__ __forceinline__ float near_cap(const PagedArgs& a, float qk) {
  const float t = __builtin_amdgcn_exp2f(qk * a.tanh_scale);
  return __builtin_fmaf(-2.0f * a.cap_log2, __builtin_amdgcn_rcpf(t + 1.0f), a.cap_log2);
}
__device__ __forceinline__ float wide_cap(const PagedArgs& a, float qk) {
  const float x = qk * a.tanh_scale * (0.5f / kLog2e), y = x * x;
  float p = __builtin_fmaf(y, 62.0f / 2835.0f, -17.0f / 315.0f);
  p = __builtin_fmaf(y, p, 2.0f / 15.0f);
  p = __builtin_fmaf(y, p, -1.0f / 3.0f);
  return fabsf(x) < 0.25f ? a.cap_log2 * __builtin_fmaf(x * y, p, x) : near_cap(a, qk);
}

// Scores of N products q.k, the i-th with key first_key + off(i); the branches are the same for every lane.
template <int N, typename V, typename F>
__device__ __forceinline__ void form_scores(const PagedArgs& a, const Row& r, int first_key, V& s, F off) {
  if (a.cap_log2 == 0.0f) {
    // as they are
  } else if (!a.wide) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = near_cap(a, s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = wide_cap(a, s[i]);
  }
  if (a.slopes) {
    const float away = static_cast<float>(r.pos - first_key);
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __builtin_fmaf(-r.slope, fabsf(away - static_cast<float>(off(i))), s[i]);
  }
}

// The id of the page with key `key`, or -1 where the request has none there (wave-uniform).
__device__ __forceinline__ int page_id(const PagedArgs& a, const Where& w, int key) {
  if (key >= w.kv) return -1;
  // through the constant address space: a scalar load, whatever the kernel stores meanwhile (a vector load would be
  // waited for together with every load into LDS before it)
  const auto* row = (const __attribute__((address_space(4))) int32_t*)(a.table + w.b * a.table_ld);
  const int id = row[key >> a.shift];
  return static_cast<unsigned>(id) < static_cast<unsigned>(a.pages) ? id : -1;
}

template <bool F16>
__device__ __forceinline__ bool not_finite(uint32_t half) {
  constexpr uint32_t e = F16 ? 0x7C00u : 0x7F80u;
  return (half & e) == e;
}

// Takes the infinities and NaN out of eight 16-bit values; true if there were any.
template <bool F16>
__device__ __forceinline__ bool clean(u32x4_t& x) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = not_finite<F16>(x[i]), hi = not_finite<F16>(x[i] >> 16);
    x[i] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
    any |= lo | hi;
  }
  return any;
}

// 16-byte unit `u` of row `r` of a [rows][D] tile in LDS lies at unit u ^ swizzle(r) of its row: the 16-byte reads of
// 8 rows at one unit, and the transposing reads of 8 rows, then fall on different banks.
template <int D>
__device__ __forceinline__ int swizzle(int r) {
  return D == 128 ? (r & 7) << 1 : ((r >> 1) & 3) << 1;
}

typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

// Four rows r0 .. r0+3 (by the address) of one column each: transposing read of 8 bytes a lane.
__device__ __forceinline__ u32x2_t read_tr(const uint16_t* p) {
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)p));
}

// 16 bytes a lane from memory to LDS, at `to` (wave-uniform) + 16 bytes * lane, without registers; ONCE: with the
// non-temporal hint, for what no other workgroup reads.
template <bool ONCE = false>
__device__ __forceinline__ void load_lds16(const char* from, uint16_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)to, 16, 0, ONCE ? 2 : 0);
}
// The wave's loads have landed, and its reads of the step before have left LDS.
__device__ __forceinline__ void wave_landed() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

// Eight values of codes, two words of fp8 or one of fp4, under the scale byte `scale`.  The conversion scales exactly, but
// for fp16 values below its least normal one, and gives NaN under 255.
template <bool F16, int FMT>
__device__ __forceinline__ u32x4_t values8(uint32_t w0, uint32_t w1, uint32_t scale) {
  const float s = __uint_as_float(scale << 23);
  const auto u = [](auto x) { return __builtin_bit_cast(uint32_t, x); };
  if constexpr (FMT == kFp8Pages && F16)
    return u32x4_t{u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, false)), u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, true)),
                   u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, false)), u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, true))};
  else if constexpr (FMT == kFp8Pages)
    return u32x4_t{u(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false)), u(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true)),
                   u(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false)), u(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true))};
  else if constexpr (F16)
    return u32x4_t{u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w0, s, 0)), u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w0, s, 1)),
                   u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w0, s, 2)), u(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w0, s, 3))};
  else
    return u32x4_t{u(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, s, 0)), u(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, s, 1)),
                   u(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, s, 2)), u(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, s, 3))};
}
// Unit j (of 8 values) of the 16 or 32 that 16 bytes of codes hold.
template <bool F16, int FMT>
__device__ __forceinline__ u32x4_t unit_of(u32x4_t codes, int j, uint32_t scale) {
  return FMT == kFp8Pages ? values8<F16, FMT>(codes[2 * j], codes[2 * j + 1], scale) : values8<F16, FMT>(codes[j], 0, scale);
}
// Rows kernel: a thread that converts 16 bytes of a row has several units of 8 channels.  It writes the j-th of them to
// LDS behind the j-th ones of the row's other threads, so that these lie side by side: unit u of a row holds the channels
// of unit unit_at(u), in Q's order for the products with K and in the outputs' for those with V.  (A thread's own units
// side by side, half of the LDS cycles were conflicts, where it is two fifths; the times are as far apart as two cards'.)
template <int D, int FMT>
__device__ __forceinline__ constexpr int unit_at(int u) {
  if (FMT == kHalfPages) return u;
  const int threads = (FMT == kFp8Pages ? D : D / 2) / 16, each = D / 8 / threads;
  return each * (u % threads) + u / threads;
}
template <int D, int FMT>
constexpr int kRowBytes = FMT == kHalfPages ? 2 * D : FMT == kFp8Pages ? D : D / 2;

// V of channel d of the token at `in_page` of page `id`, as 16 bits.
template <int D, bool F16, int FMT>
__device__ __forceinline__ uint16_t value_at(const PagedArgs& a, int head, int id, int in_page, int d) {
  if constexpr (FMT == kHalfPages) {
    return a.v[id * a.page + head * a.head + in_page * a.tok + d];
  } else {
    const auto* codes = reinterpret_cast<const uint8_t*>(a.v) + id * a.page + head * a.head + in_page * a.tok;
    const uint32_t scale = a.v_scales[id * a.s_page + head * a.s_head + in_page * (D / kScaleBlock) + d / kScaleBlock];
    const uint32_t code = FMT == kFp8Pages ? codes[d] : codes[d / 2] >> 4 * (d & 1);
    return static_cast<uint16_t>(values8<F16, FMT>(code, 0, scale)[0]);
  }
}

template <bool F16>
__device__ __forceinline__ f32x16_t mfma_32x32x16(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
}

// Where requests share, parts count from w.part units of kPartUnit rows, and the tile's first workgroup notes where
// the parts of its (row, KV head)s are, in tiles of M rows: (first row, parts << 4 | M / kPartUnit), 0 parts where it
// writes the output itself.
constexpr int kPartUnit = 16;
template <int M>
__device__ __forceinline__ void note_parts(const PagedArgs& a, const PagedClass& c, const Where& w) {
  const int t = threadIdx.x, token = w.tile * c.tokens + t;
  if (w.split != 0 || t >= c.tokens || token >= w.n_rows) return;
  const int64_t i = w.row0 + token + (w.heirs ? a.rows : 0);
  const int n = w.n_split == 1 && w.alone ? 0 : w.n_split;
  a.at[i * a.kv_heads + w.head] = make_int2(w.part * kPartUnit + t * a.group, n << 4 | M / kPartUnit);
}

// ---------------------------------------------------------------------------
// Tiles of 128 rows.  Wave w holds rows 32w .. 32w+31 as columns of S^T and O^T; a lane holds one row's scores of 16
// of the 32 keys of a score tile (its other half-wave the others), and one row's outputs.  K and V of 64 keys lie in
// LDS, double-buffered: the next tile's loads, straight into LDS, are issued before this one is computed and waited
// for behind it, one barrier a tile.  Two workgroups a CU, so that one's softmax runs beside the other's products:
// products of the next tile beside this one's softmax within a wave took more registers than there are for two
// workgroups, and more time (2370 us at 2048 x 65536, 2600 in halves of a tile; 2180 as it was then).
// ---------------------------------------------------------------------------
template <int D, bool F16, bool FORM, int FMT = kHalfPages, bool SH = false>
__device__ __forceinline__ void rows_body(const PagedArgs& a, const PagedClass& c, const Where& w, uint16_t* stage0,
                                          uint16_t* stage1) {
  constexpr int KS = D / 16;               // steps of 16 channels of Q.K
  constexpr int DB = D / 32;               // blocks of 32 channels of P.V
  constexpr int UR = D / 8;                // 16-byte units of a row
  constexpr int NU = kTile * UR / 256;     // units a thread stages of K, and of V
  uint16_t *kbuf0 = stage0, *vbuf0 = stage0 + kTile * D, *kbuf1 = stage1, *vbuf1 = stage1 + kTile * D;
  __shared__ int s_odd[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, l32 = lane & 31;
  const float ninf = -__builtin_huge_valf();
  const Row r = row_of<FORM, SH>(a, c, w, 32 * wave + l32);

  // Keys that all rows see, and that any row sees, of the workgroup and of the wave (the wave's first key apart).  They
  // follow from the first and the last token; only first_keys have to be read, two tokens a lane.
  const int n_tok = min(c.tokens, w.n_rows - w.tile * c.tokens);
  const bool heirs = SH && w.heirs;   // they see all of the parent's
  const int pos0 = heirs ? 0 : a.kv_lens[w.b] - w.n_rows + w.tile * c.tokens;
  const int prefix = heirs ? w.kv : prefix_of<SH>(a, w);
  auto hi_of = [&](int token) { return pos0 + token < 0 ? 0 : min(w.kv, max(pos0 + token + 1, prefix)); };
  int wg_all_lo = 0, wg_lo = 0;
  if (a.first) {
    const int64_t at = w.row0 + w.tile * c.tokens;
    const auto first = [&](int64_t row) {
      return first_of<SH>(a, w, heirs ? min(max(a.order[row], 0), a.rows - 1) : row);
    };
    const int f0 = first(at + min(lane, n_tok - 1)), f1 = first(at + min(lane + 64, n_tok - 1));
    wg_all_lo = wave_max_i(max(f0, f1));
    wg_lo = -wave_max_i(max(-f0, -f1));
  }
  const int wg_all_hi = hi_of(0), wg_hi = hi_of(n_tok - 1);
  const int tok_a = 32 * wave * a.per_group >> 16, tok_b = (32 * wave + 31) * a.per_group >> 16;
  const int any_hi = tok_a < n_tok ? hi_of(min(tok_b, n_tok - 1)) : 0;
  const int begin = max(w.split * w.chunk, wg_lo / kTile * kTile);
  const int end = static_cast<int>(min(static_cast<int64_t>(w.split + 1) * w.chunk, static_cast<int64_t>(wg_hi)));

  u32x4_t qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const uint4 x = load16u(a.q + r.q_at + 8 * (unit_at<D, FMT>(2 * s) + half * unit_at<D, FMT>(1)));
    qf[s] = r.on ? u32x4_t{x.x, x.y, x.z, x.w} : u32x4_t{0u, 0u, 0u, 0u};
  }

  f32x16_t o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  float m = ninf, l = 0.0f;

  // A thread stages unit u_col of row u_row (+ 256 / UR per pass) of the tile: rows of one pass and wave lie in one
  // 16-key group, so in one page, and their address is a wave-uniform base and a constant offset.  LDS holds unit
  // tid of a pass at place tid, the swizzle is in which column is read.
  const int u_row = tid / UR, u_col = (tid % UR) ^ swizzle<D>(tid / UR);
  const uint32_t off = 2 * ((u_row & 15) * a.tok + 8 * u_col);
  constexpr int EB = FMT == kHalfPages ? 2 : 1;   // bytes a stride counts
  const char* kh = reinterpret_cast<const char*>(a.k) + EB * w.head * a.head;
  const char* vh = reinterpret_cast<const char*>(a.v) + EB * w.head * a.head;
  const int page_mask = (1 << a.shift) - 1;
  auto group_of = [&](int u) { return NU == 4 ? u : 2 * u + (wave >> 1); };   // of pass u and this wave
  const int64_t page_bytes = EB * a.page;
  const uint32_t tok_bytes = EB * a.tok;
  const auto* table_row = (const __attribute__((address_space(4))) int32_t*)(a.table + w.b * a.table_ld);
  // The pages of a tile's four 16-key groups, -1 where there is none: the table's entries are read all at once (past
  // the request's end its last one), and before they are needed.
  struct Pages {
    int id[4];
  };
  auto pages_of = [&](int t0) __attribute__((always_inline)) {
    Pages p;
#pragma unroll
    for (int g = 0; g < 4; ++g) p.id[g] = table_row[min(t0 + 16 * g, w.kv - 1) >> a.shift];
    return p;
  };
  bool hole = false;   // the loaded tile has keys without a page
  // Codes go by way of registers: a thread stages 16 bytes of a row, so QC channels under one scale, QP times.
  constexpr int QU = FMT ? kRowBytes<D, FMT> / 16 : 1, QC = FMT == kFp4Pages ? 32 : 16;
  constexpr int QR = 256 / QU, QP = FMT ? (kTile * QU + 255) / 256 : 1;   // rows of a pass; passes
  struct Staged {
    u32x4_t k[QP], v[QP];
    uint32_t ks[QP], vs[QP];
  };
  const int q_row = tid / QU, q_unit = tid % QU;
  const uint32_t q_off = (q_row & 15) * tok_bytes + 16 * q_unit;
  const uint32_t qs_off = (q_row & 15) * (D / kScaleBlock) + q_unit * QC / kScaleBlock;
  auto load = [&](int t0, Pages p, uint16_t* kb, uint16_t* vb, Staged& staged) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (static_cast<unsigned>(p.id[g]) >= static_cast<unsigned>(a.pages)) p.id[g] = -1;
    hole = (p.id[0] | p.id[1] | p.id[2] | p.id[3]) < 0;
    if constexpr (FMT != kHalfPages) {
#pragma unroll
      for (int u = 0; u < QP; ++u) {
        // the 16-key group of a thread's row: the same for a wave where it has at most 16 rows
        const int g = QU >= 4 ? (u * QR + wave * (64 / QU)) >> 4 : (q_row >> 4) & 3;
        const int id = max(g < 2 ? (g == 0 ? p.id[0] : p.id[1]) : (g == 2 ? p.id[2] : p.id[3]), 0);
        const int in_page = (t0 + 16 * g) & page_mask;
        const int64_t at = id * page_bytes + in_page * tok_bytes;
        const int64_t s_at = id * a.s_page + w.head * a.s_head + in_page * (D / kScaleBlock);
        if (kTile * QU >= 256 || q_row < kTile) {
          staged.k[u] = *reinterpret_cast<const u32x4_t*>(kh + at + q_off);
          staged.v[u] = *reinterpret_cast<const u32x4_t*>(vh + at + q_off);
          staged.ks[u] = a.k_scales[s_at + qs_off];
          staged.vs[u] = a.v_scales[s_at + qs_off];
        }
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int id = max(NU == 4 ? p.id[u % 4] : wave >> 1 ? p.id[(2 * u + 1) % 4] : p.id[2 * u % 4], 0);
      const int64_t at = id * page_bytes + ((t0 + 16 * group_of(u)) & page_mask) * tok_bytes;
      load_lds16(kh + at + off, kb + 8 * (256 * u + 64 * wave));
      load_lds16(vh + at + off, vb + 8 * (256 * u + 64 * wave));
    }
  };
  // Where some row does not see all of a tile, what of V no row may read (a page's rest) becomes zero before it is
  // used, and so do infinities and NaN, which a zero weight would not hide; add_odd adds those to the rows that do
  // see them.  A wave cleans what it loaded itself, so that the barrier behind the loads serves for both.
  auto put_codes = [&](int t0, bool masked, bool holes, uint16_t* kb, uint16_t* vb, int buf, const Staged& staged)
                       __attribute__((always_inline)) {
    bool odd = false;
    if (kTile * QU >= 256 || q_row < kTile) {
#pragma unroll
      for (int u = 0; u < QP; ++u) {
        const int row = u * QR + q_row;
        const bool rest = masked && (t0 + row >= w.kv || (holes && page_id(a, w, t0 + (row & -16)) < 0));
#pragma unroll
        for (int j = 0; j < QC / 8; ++j) {
          const int to = row * D + 8 * ((q_unit + QU * j) ^ swizzle<D>(row));
          *reinterpret_cast<u32x4_t*>(kb + to) = unit_of<F16, FMT>(staged.k[u], j, staged.ks[u]);
          u32x4_t x = unit_of<F16, FMT>(staged.v[u], j, staged.vs[u]);
          if (masked) {
            x = u32x4_t{rest ? 0u : x[0], rest ? 0u : x[1], rest ? 0u : x[2], rest ? 0u : x[3]};
            odd |= clean<F16>(x);
          }
          *reinterpret_cast<u32x4_t*>(vb + to) = x;
        }
      }
    }
    if (masked) s_odd[buf][wave] = __ballot(odd) != 0;
  };
  auto clean_tile = [&](int t0, bool holes, uint16_t* vb, int buf) {
    u32x4_t x[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) x[u] = *reinterpret_cast<u32x4_t*>(vb + 8 * (256 * u + tid));
    bool odd = false;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const bool rest = t0 + u_row + u * (256 / UR) >= w.kv || (holes && page_id(a, w, t0 + 16 * group_of(u)) < 0);
      if (rest) x[u] = u32x4_t{0u, 0u, 0u, 0u};
      const bool any = !rest && clean<F16>(x[u]);
      odd |= any;
      if (rest || any) *reinterpret_cast<u32x4_t*>(vb + 8 * (256 * u + tid)) = x[u];
    }
    s_odd[buf][wave] = __ballot(odd) != 0;
  };
  auto add_odd = [&](int t0) {
#pragma unroll 1
    for (int j = 0; j < kTile; ++j) {
      const int key = t0 + j, id = page_id(a, w, key);
      if (id < 0) continue;
      if (!(r.on && key >= r.lo && key < r.hi)) continue;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint16_t x = value_at<D, F16, FMT>(a, w.head, id, key & page_mask, 4 * half + 8 * unit_at<D, FMT>(4 * d + (i >> 2)) + (i & 3));
          if (not_finite<F16>(x)) o[d][i] += half_to_f32<F16>(x);
          if ((i & 3) == 3) __builtin_amdgcn_sched_barrier(0);
        }
    }
  };

  const int k_at = l32 * D, k_sw = swizzle<D>(l32);
  const int v_row = 4 * half + ((lane & 15) >> 2), v_unit = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), v_el = 4 * (lane & 1);
  auto compute = [&](int t0, bool masked, bool holes, const uint16_t* kb_, const uint16_t* vb_, int buf, auto&& between)
                     __attribute__((always_inline)) {
    if (t0 >= any_hi) {   // no row of the wave sees any of it
      between();
      return;
    }
    f32x16_t s[2];
    {
      u32x4_t kf[2][KS];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          kf[kb][ks] = *reinterpret_cast<const u32x4_t*>(kb_ + kb * 32 * D + k_at + 8 * ((2 * ks + half) ^ k_sw));
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[kb] = mfma_32x32x16<F16>(kf[kb][ks], qf[ks], s[kb]);
      }
      // four fragments ahead of the matrix instruction that takes them (2170 -> 2088 us at 2048 x 65536, 32/8 heads;
      // all of them first: 2245)
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);   // LDS reads
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // matrix instruction
        if (i < 2 * KS - 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    }
    if constexpr (FMT != kHalfPages && !FORM) {
      __builtin_amdgcn_sched_barrier(0);
      between();
    }
    const int key0 = t0 + 4 * half;   // element i of tile kb: key0 + 32 kb + 8 (i / 4) + i % 4
    if constexpr (FORM) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        form_scores<16>(a, r, key0 + 32 * kb, s[kb], [](int i) { return 8 * (i >> 2) + (i & 3); });
    }
    if (masked) {
      const int from = r.lo - key0;
      const unsigned span = static_cast<unsigned>(max(r.hi - r.lo, 0));
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (static_cast<unsigned>(32 * kb + 8 * (i >> 2) + (i & 3) - from) >= span) s[kb][i] = ninf;
          if ((i & 3) == 3) __builtin_amdgcn_sched_barrier(0);   // few lane masks live at a time
        }
      if (holes) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (page_id(a, w, t0 + 16 * g) < 0) {   // a page the request does not have
#pragma unroll
            for (int i = 0; i < 8; ++i) s[g >> 1][8 * (g & 1) + i] = ninf;
          }
      }
    }
    float cm = s[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) cm = fmaxf(cm, s[kb][i]);
    cm = max_x32(cm);
    const float sl = a.unit_log2;
    cm = cm * sl - kShift<F16>;
    const float mn = fmaxf(m, cm);
    if (__ballot(mn > m + kLazyLog2)) {   // wave-uniform
      const float al = mn == ninf ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      l *= al;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= al;
      m = mn;
    }
    const float ms = m == ninf ? 0.0f : m;
    float sum0 = 0.0f, sum1 = 0.0f;
    u32x4_t p[4];   // B operands of P.V: 16 keys each
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][4 * q + i], sl, -ms));
        const u32x2_t x = pack4_half<F16>(e);
        sum0 = dot2_half<F16>(x[0], kOnes<F16>, sum0);   // of the rounded weights, which V is weighted by
        sum1 = dot2_half<F16>(x[1], kOnes<F16>, sum1);
        p[2 * kb + (q >> 1)][2 * (q & 1)] = x[0];
        p[2 * kb + (q >> 1)][2 * (q & 1) + 1] = x[1];
      }
    l += sum0 + sum1;
    if constexpr (FMT != kHalfPages && FORM) {   // (behind the first product, the score forms would spill registers)
      __builtin_amdgcn_sched_barrier(0);
      between();
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const int r0 = 16 * ks + v_row, r1 = r0 + 8;
        const u32x2_t x = read_tr(vb_ + r0 * D + 8 * ((4 * d + v_unit) ^ swizzle<D>(r0)) + v_el);
        const u32x2_t y = read_tr(vb_ + r1 * D + 8 * ((4 * d + v_unit) ^ swizzle<D>(r1)) + v_el);
        o[d] = mfma_32x32x16<F16>(u32x4_t{x[0], x[1], y[0], y[1]}, p[ks], o[d]);
      }
    if (masked && (s_odd[buf][0] | s_odd[buf][1] | s_odd[buf][2] | s_odd[buf][3])) add_odd(t0);
  };

  // One barrier a tile: the next tile's loads are issued before this one is computed, and have landed behind it.
  bool holes, masked;   // of the tile that has landed
  auto landed = [&](int t0, uint16_t* kb, uint16_t* vb, int buf, const Staged& staged) __attribute__((always_inline)) {
    if constexpr (FMT == kHalfPages) wave_landed();
    holes = hole, masked = t0 < wg_all_lo || t0 + kTile > wg_all_hi || holes;
    if constexpr (FMT != kHalfPages) {
      if (t0 < end) put_codes(t0, masked, holes, kb, vb, buf, staged);
    } else {
      if (masked && t0 < end) clean_tile(t0, holes, vb, buf);
    }
    __syncthreads();
  };
  auto turn = [&](int t0, const uint16_t* kb_, const uint16_t* vb_, int buf, uint16_t* kn, uint16_t* vn)
                  __attribute__((always_inline)) {
    const Pages next = pages_of(t0 + kTile);
    Staged staged;
    const auto ahead = [&]() __attribute__((always_inline)) {
      if (t0 + kTile < end) load(t0 + kTile, next, kn, vn, staged);
    };
    // codes go to registers, which the first product has most need of: they are loaded behind it
    if constexpr (FMT == kHalfPages) ahead();
    compute(t0, masked, holes, kb_, vb_, buf, [&]() __attribute__((always_inline)) {
      if constexpr (FMT != kHalfPages) ahead();
    });
    landed(t0 + kTile, kn, vn, buf ^ 1, staged);
  };
  if (begin < end) {
    Staged staged;
    load(begin, pages_of(begin), kbuf0, vbuf0, staged);
    landed(begin, kbuf0, vbuf0, 0, staged);
    for (int t0 = begin; t0 < end; t0 += 2 * kTile) {
      turn(t0, kbuf0, vbuf0, 0, kbuf1, vbuf1);
      if (t0 + kTile < end) turn(t0 + kTile, kbuf1, vbuf1, 1, kbuf0, vbuf0);
    }
  }

  l = sum_x32(l);
  if (SH) note_parts<kRowsM>(a, c, w);
  if (w.n_split == 1 && (!SH || w.alone)) {
    // by way of LDS (the wave's own part: the loop's last barrier has passed), so that whole rows are stored: 2.5 us a
    // workgroup for 8-byte stores to 32 rows at a time
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* mine = stage0 + wave * 32 * D;
    int own = l32;
    asm("" : "+v"(own));   // own * D is not l32 * D of the loop, which would be kept, and spilled, for it
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float x[4] = {o[d][4 * q] * inv, o[d][4 * q + 1] * inv, o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv};
        *reinterpret_cast<u32x2_t*>(mine + own * D + 8 * (unit_at<D, FMT>(4 * d + q) ^ (own & (UR - 1))) + 4 * half) = pack4_half<F16>(x);
      }
#pragma unroll
    for (int i = 0; i < 32 * UR / 64; ++i) {
      const int row = i * (64 / UR) + lane / UR, unit = lane % UR;
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(mine + row * D + 8 * (unit ^ (row & (UR - 1))));
      const Row ro = row_of<false, SH>(a, c, w, 32 * wave + row);
      if (ro.on) *reinterpret_cast<u32x4_t*>(a.out + ro.o_at + 8 * unit) = x;
    }
    return;
  }
  const int64_t at = static_cast<int64_t>(w.part) * (SH ? kPartUnit : kRowsM) + 32 * wave + l32;
  if (half == 0) {
    c.ml[2 * at] = m;
    c.ml[2 * at + 1] = l;
  }
  if (l == 0.0f) return;   // the joining kernel leaves it out
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<float4*>(c.acc + at * D + 4 * half + 8 * unit_at<D, FMT>(4 * d + q)) =
          make_float4(o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]);
}

// ---------------------------------------------------------------------------
// Tiles of at most 16 NQ rows: NQ sets of 16 columns of 16-wide score tiles.  Wave w takes steps w, w + 4, ... of 32
// keys of the workgroup's chunk; K goes from memory to the matrix instruction's registers, V through the wave's own
// part of LDS (as it lies, read transposed), no barrier until the waves are joined at the end.  V is loaded with the
// non-temporal hint, whole rows at a time; K without, since two loads share each of its 128-byte lines (32 requests of up
// to 32768 keys: 530 us, 6.14 TB/s; both with the hint 548, neither 582, K alone 556).
// ---------------------------------------------------------------------------
template <int D, bool F16, bool FORM, int NQ, int FMT = kHalfPages, bool SH = false>
__device__ __forceinline__ void token_body(const PagedArgs& a, const PagedClass& c, const Where& w, uint16_t* stage0,
                                           uint16_t* stage1) {
  constexpr int KS = D / 32;               // steps of 32 channels of Q.K
  constexpr int DB = D / 16;               // blocks of 16 channels of P.V
  constexpr int UR = D / 8;                // 16-byte units of a row
  constexpr int NV = kStep * UR / 64;      // units of V a lane stages
  constexpr int PASS = 64 / UR;            // rows of V a load covers
  __shared__ float s_m[4][kTokenM], s_l[4][kTokenM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4, c16 = lane & 15;
  const float ninf = -__builtin_huge_valf();
  Row r[NQ];
  u32x4_t qf[NQ][KS];
  int lo = 0, hi = 0x7FFFFFFF, first = 0x7FFFFFFF, last = 0;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    r[n] = row_of<FORM, SH>(a, c, w, 16 * n + c16);
    lo = max(lo, r[n].lo);
    hi = min(hi, r[n].hi);
    if (r[n].on) first = min(first, r[n].lo), last = max(last, r[n].hi);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      // the channels of a step are those that a lane's bytes of K hold
      const int ch = FMT == kHalfPages ? 32 * s + 8 * g4 : FMT == kFp8Pages ? 64 * (s >> 1) + 16 * g4 + 8 * (s & 1) : D / 4 * g4 + 8 * s;
      const uint4 x = load16u(a.q + r[n].q_at + ch);
      qf[n][s] = r[n].on ? u32x4_t{x.x, x.y, x.z, x.w} : u32x4_t{0u, 0u, 0u, 0u};
    }
  }
  const int all_lo = wave_max_i(lo), all_hi = -wave_max_i(-hi), any_lo = -wave_max_i(-first), any_hi = wave_max_i(last);
  const int begin = max(w.split * w.chunk, any_lo / kTile * kTile);
  const int end = static_cast<int>(min(static_cast<int64_t>(w.split + 1) * w.chunk, static_cast<int64_t>(any_hi)));

  f32x4_t o[NQ][DB];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = ninf;
    l[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[n][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  constexpr int EB = FMT == kHalfPages ? 2 : 1;   // bytes a stride counts
  const int page_mask = (1 << a.shift) - 1;
  const int64_t page_bytes = EB * a.page;
  const uint32_t tok_bytes = EB * a.tok;
  const char* kh = reinterpret_cast<const char*>(a.k) + EB * w.head * a.head;
  const char* vh = reinterpret_cast<const char*>(a.v) + EB * w.head * a.head;
  const uint32_t k_off = c16 * tok_bytes + 16 * g4;
  // row u * PASS + lane / UR of V; its swizzle goes by the row's low bits, so by the parity of u where PASS is 4
  const uint32_t v_off0 = lane / UR * tok_bytes + 16 * ((lane % UR) ^ swizzle<D>(lane / UR));
  const uint32_t v_off1 = lane / UR * tok_bytes + 16 * ((lane % UR) ^ swizzle<D>(PASS + lane / UR));
  const auto* table_row = (const __attribute__((address_space(4))) int32_t*)(a.table + w.b * a.table_ld);
  // Codes of V go by way of registers into one buffer: a lane has QC channels of one row, QP rows of a step.
  constexpr int QU = FMT ? kRowBytes<D, FMT> / 16 : 1, QC = FMT == kFp4Pages ? 32 : 16;
  constexpr int QR = 64 / QU, QP = FMT ? kStep / QR : 1;              // rows of a load; loads
  constexpr int KW = FMT ? kRowBytes<D, FMT> / 16 : 4;                // words of K a lane has of a key
  constexpr int SB = D / kScaleBlock;
  struct Step {
    u32x4_t k[2][FMT ? (KW + 3) / 4 : KS];
    uint32_t ks[2];
    u32x4_t v[QP];
    uint32_t vs[QP];
    int id[2];
  };
  const int q_row = lane / QU, q_unit = lane % QU;
  struct Entries {
    int v[2];
  };
  auto entries_of = [&](int t0) __attribute__((always_inline)) {   // of the step's two 16-key groups
    Entries e;
#pragma unroll
    for (int t = 0; t < 2; ++t) e.v[t] = table_row[min(t0 + 16 * t, w.kv - 1) >> a.shift];
    return e;
  };
  auto load_codes = [&](int t0, const Entries& e, Step& x) __attribute__((always_inline)) {
    int64_t at[2], s_at[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = t0 + 16 * t;
      x.id[t] = key < w.kv && static_cast<unsigned>(e.v[t]) < static_cast<unsigned>(a.pages) ? e.v[t] : -1;
      const int id = max(x.id[t], 0), in_page = key & page_mask;
      at[t] = id * page_bytes + in_page * tok_bytes;
      s_at[t] = id * a.s_page + w.head * a.s_head + in_page * SB;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* kp = kh + at[t] + c16 * tok_bytes;
      if constexpr (KW >= 4) {
#pragma unroll
        for (int s = 0; s < KW / 4; ++s) {
          // once where one load takes a whole row (fp8, D 128: two loads share its line)
          const auto* from = reinterpret_cast<const u32x4_t*>(kp + 16 * g4 + 64 * s);
          x.k[t][s] = KW == 4 ? __builtin_nontemporal_load(from) : *from;
        }
      } else {
        const u32x2_t y = *reinterpret_cast<const u32x2_t*>(kp + 8 * g4);
        x.k[t][0] = u32x4_t{y[0], y[1], 0u, 0u};
      }
      const uint8_t* sp = a.k_scales + s_at[t] + c16 * SB;
      x.ks[t] = SB == 4 ? *reinterpret_cast<const uint32_t*>(sp) : *reinterpret_cast<const uint16_t*>(sp);
    }
#pragma unroll
    for (int u = 0; u < QP; ++u) {
      // the 16-key group of a lane's row: the same for the wave where a load has at most 16 rows
      const bool second = QR <= 16 ? u * QR >= 16 : q_row >= 16;
      const int row = (u * QR + q_row) & 15;
      const char* vp = vh + (second ? at[1] : at[0]) + row * tok_bytes + 16 * q_unit;
      x.v[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(vp));
      x.vs[u] = a.v_scales[(second ? s_at[1] : s_at[0]) + row * SB + q_unit * QC / kScaleBlock];
    }
  };
  auto load = [&](int t0, const Entries& e, Step& x, uint16_t* vt) __attribute__((always_inline)) {
    if constexpr (FMT != kHalfPages) {
      load_codes(t0, e, x);
      return;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = t0 + 16 * t;
      x.id[t] = key < w.kv && static_cast<unsigned>(e.v[t]) < static_cast<unsigned>(a.pages) ? e.v[t] : -1;
      const int64_t at = max(x.id[t], 0) * page_bytes + (key & page_mask) * tok_bytes;
      const char* vp = vh + at;
#pragma unroll
      for (int u = t * NV / 2; u < (t + 1) * NV / 2; ++u)
        load_lds16<true>(vp + u * PASS % 16 * tok_bytes + (u % 2 ? v_off1 : v_off0), vt + 8 * 64 * u);
      const char* kp = kh + at;
#pragma unroll
      for (int s = 0; s < KS; ++s) x.k[t][s] = *reinterpret_cast<const u32x4_t*>(kp + k_off + 64 * s);
    }
  };
  // `ahead` is called when the codes in x are used up.
  auto compute = [&](int t0, Step& x, uint16_t* vt, auto&& ahead) __attribute__((always_inline)) {
    const int id[2] = {x.id[0], x.id[1]};
    const bool masked = t0 < all_lo || t0 + kStep > all_hi || (id[0] | id[1]) < 0;
    bool odd = false;
    u32x4_t kf[2][KS];
    if constexpr (FMT != kHalfPages) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t sw = x.ks[t] >> 8 * (FMT == kFp4Pages && SB == 4 ? g4 : g4 >> 1);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if constexpr (FMT == kFp8Pages)
            kf[t][ks] = values8<F16, FMT>(x.k[t][ks >> 1][2 * (ks & 1)], x.k[t][ks >> 1][2 * (ks & 1) + 1],
                                          sw >> 16 * (ks >> 1) & 0xFFu);
          else
            kf[t][ks] = values8<F16, FMT>(x.k[t][0][ks], 0, sw & 0xFFu);
        }
      }
#pragma unroll
      for (int u = 0; u < QP; ++u) {
        const int row = u * QR + q_row;
        const bool rest = masked && (t0 + row >= w.kv || (row >= 16 ? id[1] : id[0]) < 0);
#pragma unroll
        for (int j = 0; j < QC / 8; ++j) {
          u32x4_t y = unit_of<F16, FMT>(x.v[u], j, x.vs[u]);
          if (masked) {
            y = u32x4_t{rest ? 0u : y[0], rest ? 0u : y[1], rest ? 0u : y[2], rest ? 0u : y[3]};
            odd |= clean<F16>(y);
          }
          *reinterpret_cast<u32x4_t*>(vt + row * D + 8 * ((q_unit * (QC / 8) + j) ^ swizzle<D>(row))) = y;
        }
      }
      ahead();
    } else if (masked) {   // as in rows_body; a wave's LDS operations keep their order
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        u32x4_t* p = reinterpret_cast<u32x4_t*>(vt + 8 * (64 * u + lane));
        u32x4_t y = *p;
        if (id[u * PASS / 16] < 0 || t0 + u * PASS + lane / UR >= w.kv) y = u32x4_t{0u, 0u, 0u, 0u};
        else odd |= clean<F16>(y);
        *p = y;
      }
    }
    f32x4_t s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[n][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          if constexpr (FMT != kHalfPages) s[n][t] = mfma_16x16x32<F16>(kf[t][ks], qf[n][ks], s[n][t]);
          else s[n][t] = mfma_16x16x32<F16>(x.k[t][ks], qf[n][ks], s[n][t]);
        }
    u32x4_t p[NQ];
    float mn[NQ];
    bool raise = false;
    const float sl = a.unit_log2;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float cm = ninf;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key0 = t0 + 16 * t + 4 * g4;
        if constexpr (FORM) form_scores<4>(a, r[n], key0, s[n][t], [](int i) { return i; });
        if (masked) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (id[t] < 0 || key0 + i < r[n].lo || key0 + i >= r[n].hi) s[n][t][i] = ninf;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) cm = fmaxf(cm, s[n][t][i]);
      }
      mn[n] = fmaxf(m[n], max_x32(max_x16(cm)) * sl - kShift<F16>);
      raise |= mn[n] > m[n] + kLazyLog2;
    }
    if (__ballot(raise)) {   // wave-uniform
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float al = mn[n] == ninf ? 1.0f : __builtin_amdgcn_exp2f(m[n] - mn[n]);
        l[n] *= al;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][d][i] *= al;
        m[n] = mn[n];
      }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const float ms = m[n] == ninf ? 0.0f : m[n];
      float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][t][i], sl, -ms));
        const u32x2_t y = pack4_half<F16>(e);
        sum0 = dot2_half<F16>(y[0], kOnes<F16>, sum0);
        sum1 = dot2_half<F16>(y[1], kOnes<F16>, sum1);
        p[n][2 * t] = y[0];
        p[n][2 * t + 1] = y[1];
      }
      l[n] += sum0 + sum1;
    }
    // element j of a lane's step: key 16 (j / 4) + 4 g4 + j % 4, of P and of V alike
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const int r0 = 4 * g4 + (c16 >> 2), r1 = r0 + 16, unit = 2 * d + ((lane & 3) >> 1), el = 4 * (lane & 1);
      const u32x2_t y = read_tr(vt + r0 * D + 8 * (unit ^ swizzle<D>(r0)) + el);
      const u32x2_t z = read_tr(vt + r1 * D + 8 * (unit ^ swizzle<D>(r1)) + el);
#pragma unroll
      for (int n = 0; n < NQ; ++n) o[n][d] = mfma_16x16x32<F16>(u32x4_t{y[0], y[1], z[0], z[1]}, p[n], o[n][d]);
    }
    if (masked && __ballot(odd)) {
#pragma unroll 1
      for (int j = 0; j < kStep; ++j) {
        const int key = t0 + j, page = page_id(a, w, key);
        if (page < 0) continue;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          if (!(r[n].on && key >= r[n].lo && key < r[n].hi)) continue;
#pragma unroll
          for (int d = 0; d < DB; ++d) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint16_t y = value_at<D, F16, FMT>(a, w.head, page, key & page_mask, 4 * g4 + 16 * d + i);
              if (not_finite<F16>(y)) o[n][d][i] += half_to_f32<F16>(y);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
  };

  // A step's loads are issued when those of the step before have landed, and land while that one is computed.  (Issued
  // before that wait, two steps deep, 32 requests of up to 32768 keys take 547 us instead of 529: eight waves a CU with
  // 16 KB each on its way are enough.)
  Step x0, x1;
  Entries e;
  uint16_t *vt0 = stage0 + wave * kStep * D, *vt1 = stage1 + wave * kStep * D;
  int t0 = begin + kStep * wave;
  if (t0 < end) {
    load(t0, entries_of(t0), x0, vt0);
    e = entries_of(t0 + 4 * kStep);
  }
  if constexpr (FMT != kHalfPages) {
    // A step's codes leave their registers for the next step's as soon as they are converted.
    while (t0 < end) {
      compute(t0, x0, vt0, [&]() __attribute__((always_inline)) {
        if (t0 + 4 * kStep < end) {
          load(t0 + 4 * kStep, e, x0, vt0);
          e = entries_of(t0 + 8 * kStep);
        }
      });
      t0 += 4 * kStep;
    }
  }
  auto turn = [&](Step& x, uint16_t* vt, Step& xn, uint16_t* vn) __attribute__((always_inline)) {
    wave_landed();
    if (t0 + 4 * kStep < end) {
      load(t0 + 4 * kStep, e, xn, vn);
      e = entries_of(t0 + 8 * kStep);
    }
    compute(t0, x, vt, [] {});
    t0 += 4 * kStep;
  };
  while (FMT == kHalfPages && t0 < end) {
    turn(x0, vt0, x1, vt1);
    if (t0 >= end) break;
    turn(x1, vt1, x0, vt0);
  }

  if (SH) note_parts<NQ * kTokenM>(a, c, w);
  // the four waves' parts, joined
  float* acc = reinterpret_cast<float*>(stage0);   // [4][16][D]
  constexpr int E = D / 16;                        // values a thread joins
  const int jr = tid >> 4, d0 = (tid & 15) * E;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const float ln = sum_x32(sum_x16(l[n]));
    __syncthreads();   // stage0 is done with
    if (lane < kTokenM) {
      s_m[wave][lane] = m[n];
      s_l[wave][lane] = ln;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
      *reinterpret_cast<f32x4_t*>(acc + (wave * kTokenM + c16) * D + 16 * d + 4 * g4) = o[n][d];
    __syncthreads();
    float mj = s_m[0][jr];
#pragma unroll
    for (int i = 1; i < 4; ++i) mj = fmaxf(mj, s_m[i][jr]);
    float lj = 0.0f, y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s_l[i][jr] == 0.0f) continue;
      const float f = __builtin_amdgcn_exp2f(s_m[i][jr] - mj);
      lj = __builtin_fmaf(s_l[i][jr], f, lj);
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = __builtin_fmaf(acc[(i * kTokenM + jr) * D + d0 + e], f, y[e]);
    }
    if (w.n_split == 1 && (!SH || w.alone)) {
      const Row ro = row_of<false, SH>(a, c, w, 16 * n + jr);
      if (!ro.on) continue;
      const float inv = lj == 0.0f ? 0.0f : 1.0f / lj;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const float z[4] = {y[e] * inv, y[e + 1] * inv, y[e + 2] * inv, y[e + 3] * inv};
        *reinterpret_cast<u32x2_t*>(a.out + ro.o_at + d0 + e) = pack4_half<F16>(z);
      }
      continue;
    }
    const int64_t at = static_cast<int64_t>(w.part) * (SH ? kPartUnit : NQ * kTokenM) + 16 * n + jr;
    if ((tid & 15) == 0) {
      c.ml[2 * at] = mj;
      c.ml[2 * at + 1] = lj;
    }
#pragma unroll
    for (int e = 0; e < E; e += 4)
      *reinterpret_cast<float4*>(c.acc + at * D + d0 + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
  }
}

// Joins the parts of the tiles whose keys were split.  G workgroups share a tile's rows, R at a time; each walks a
// row's parts in P groups, part s in group s % P, which are joined in order, so that the result does not depend
// on which workgroup was done first.  Tiles of the token kernel have few rows and up to a thousand parts (one row at a
// time), those of the rows kernel many rows and few parts.
template <int D, bool F16, int M, int R, int G>
__device__ __forceinline__ bool join_body(const PagedArgs& a, const PagedClass& c, int item) {
  constexpr int L = D / 4;             // lanes of a row, 4 values each
  constexpr int P = 256 / (R * L);
  __shared__ float s_acc[P][R][D], s_m[P][R], s_l[P][R];
  Where w;
  if (!locate<true>(a, c, item / G, w)) return false;
  const int in_tile = threadIdx.x / L % R, group = threadIdx.x / (L * R), d0 = 4 * (threadIdx.x % L);
  const int n_rows = min(c.tokens, w.n_rows - w.tile * c.tokens) * a.group;
  const float ninf = -__builtin_huge_valf();
  for (int rows_at = item % G * R; rows_at < n_rows; rows_at += G * R) {
    const int row = rows_at + in_tile;
    float m = ninf, l = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float mp, float lp, float4 x) {
      if (lp == 0.0f) mp = ninf, x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // a part without keys holds no values
      const float mn = fmaxf(m, mp), base = mn == ninf ? 0.0f : mn;
      const float fo = __builtin_amdgcn_exp2f(m - base), fn = __builtin_amdgcn_exp2f(mp - base);
      l = __builtin_fmaf(lp, fn, l * fo);
      y.x = __builtin_fmaf(x.x, fn, y.x * fo);
      y.y = __builtin_fmaf(x.y, fn, y.y * fo);
      y.z = __builtin_fmaf(x.z, fn, y.z * fo);
      y.w = __builtin_fmaf(x.w, fn, y.w * fo);
      m = mn;
    };
    const int64_t at = static_cast<int64_t>(w.part) * M + row;   // of part 0
    constexpr int U = 4;   // parts whose loads are issued together
    for (int s0 = group; s0 < w.n_split; s0 += U * P) {
      float mp[U], lp[U];
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t p = at + static_cast<int64_t>(min(s0 + u * P, w.n_split - 1)) * M;
        mp[u] = c.ml[2 * p];
        lp[u] = c.ml[2 * p + 1];
        x[u] = *reinterpret_cast<const float4*>(c.acc + p * D + d0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (s0 + u * P < w.n_split) add(mp[u], lp[u], x[u]);
    }
    if constexpr (P > 1) {
      __syncthreads();   // the row before is done with
      *reinterpret_cast<float4*>(&s_acc[group][in_tile][d0]) = y;
      if (d0 == 0) {
        s_m[group][in_tile] = m;
        s_l[group][in_tile] = l;
      }
      __syncthreads();
      if (group > 0) continue;
#pragma unroll
      for (int p = 1; p < P; ++p)
        add(s_m[p][in_tile], s_l[p][in_tile], *reinterpret_cast<const float4*>(&s_acc[p][in_tile][d0]));
    }
    const Row r = row_of<false>(a, c, w, row);
    if (!r.on) continue;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float z[4] = {y.x * inv, y.y * inv, y.z * inv, y.w * inv};
    *reinterpret_cast<u32x2_t*>(a.out + r.o_at + d0) = pack4_half<F16>(z);
  }
  return true;
}

// The launches of a call, from what the host knows: rows, requests, and the tokens a table row covers.
struct Shape {
  PagedClass cls;
  int64_t items, parts;   // workgroups; parts in the workspace
};

// Tiles of m rows for requests of more than `above` and at most `most` rows.
Shape shape_of(bool token, int64_t m, int64_t above, int64_t most, int64_t rows, int64_t requests, int64_t max_keys,
               int64_t kv_heads, int64_t group, int round) {
  Shape s{};
  s.cls.tokens = static_cast<int>(m / group);
  s.cls.above = static_cast<int>(above);
  s.cls.most = static_cast<int>(most);
  // up to 512 keys the launch that joins parts costs more than a split gives (one request of 500 keys: 12.8 us, 17.1 split)
  s.cls.min_keys = token && max_keys <= 512 ? 512 : 256;
  const int64_t target = token && requests > 1 ? 3 * round : round;   // the most that chunk_of asks for
  s.cls.round = round;
  s.cls.per_round = 1.0001f / static_cast<float>(round);
  s.cls.finer = token && requests > 1;
  if (rows == 0 || s.cls.tokens == 0) return s;
  const int64_t some = std::min(requests, rows);
  const int64_t tiles = (most <= s.cls.tokens ? some : (rows + some * (s.cls.tokens - 1)) / s.cls.tokens) * kv_heads;
  s.items = tiles;
  if (max_keys > s.cls.min_keys) {
    // sum over the requests of tiles * ceil(keys / C) <= W / C + tiles, W / C <= target; where a request is split its
    // ceil(keys / C) is at most 2 keys / C
    s.items = std::min(tiles + target, tiles * cdiv(max_keys, s.cls.min_keys));
    s.parts = std::min<int64_t>(2 * target, s.items);
    s.cls.max_joins = static_cast<int>(std::min<int64_t>(target, tiles) * (token ? m / kTokenM * kTokenJoins : kRowsJoins));
  }
  s.cls.max_parts = static_cast<int>(s.parts);
  return s;
}

// One column set where every request's rows fit it, two where they fit those; otherwise the rows kernel, and two
// column sets for the requests that fit them.
struct Plan {
  Shape rows, token;
  int sets;
};
Plan plan_of(int64_t rows, int64_t max_rows, int64_t requests, int64_t max_keys, int64_t kv_heads, int64_t group,
             int64_t row_bytes) {
  constexpr int64_t kAny = 0x7FFFFFFF;
  Plan p{};
  max_rows = std::max<int64_t>(max_rows, 1);
  p.sets = max_rows * group <= kTokenM ? 1 : 2;
  const int64_t m = p.sets * kTokenM;
  if (max_rows * group <= m) {   // a longer request, if there is one after all, takes several tiles
    p.token = shape_of(true, m, 0, kAny, rows, requests, max_keys, kv_heads, group, p.sets == 1 && row_bytes <= kShortRow ? kShortRound : kRound);
    return p;
  }
  p.token = shape_of(true, m, 0, m / group, rows, requests, max_keys, kv_heads, group, kRound);
  p.rows = shape_of(false, kRowsM, m / group, kAny, rows, requests, max_keys, kv_heads, group, kRound);
  return p;
}

int64_t part_floats(int64_t m, int64_t head_dim) { return m * (head_dim + 2); }

bool good_sizes(int64_t rows, int64_t requests, int64_t width, int64_t page, int64_t q_heads, int64_t kv_heads,
                int64_t head_dim) {
  return rows >= 0 && rows <= (1 << 30) && requests >= 1 && requests <= (1 << 20) && width >= 1 && page >= 16 &&
         page <= 4096 && !(page & (page - 1)) && width <= (1ll << 30) / page && kv_heads >= 1 &&
         q_heads >= kv_heads && q_heads % kv_heads == 0 && q_heads <= 65536 && q_heads / kv_heads <= kRowsM &&
         (head_dim == 64 || head_dim == 128);
}

int64_t workspace_bytes(const Plan& p, int64_t head_dim) {
  return 4 * (p.rows.parts * part_floats(kRowsM, head_dim) + p.token.parts * part_floats(p.sets * kTokenM, head_dim));
}

// Both kernels stage K and V in two halves of LDS, of which the compiler sees that reads of one need not wait for
// the loads into the other.
template <int D, bool F16, bool FORM, int FMT, int NQ>
__global__ __launch_bounds__(256, FMT != kHalfPages && NQ == 1 ? 3 : 2) void paged_token_kernel(PagedArgs a, PagedClass c) {
  __shared__ __attribute__((aligned(16))) uint16_t stage0[2 * kTile * D], stage1[2 * kTile * D];
  Where w;
  if (locate<false>(a, c, blockIdx.x, w)) token_body<D, F16, FORM, NQ, FMT>(a, c, w, stage0, stage1);
}
// Requests of both classes in one launch, the long ones first.
template <int D, bool F16, bool FORM, int FMT>
__global__ __launch_bounds__(256, D == 64 && !(FORM && FMT != kHalfPages) ? 3 : 2) void paged_rows_kernel(PagedArgs a, PagedClass rows, PagedClass token,
                                                                          int n_rows) {
  __shared__ __attribute__((aligned(16))) uint16_t stage0[2 * kTile * D], stage1[2 * kTile * D];
  Where w;
  if (static_cast<int>(blockIdx.x) < n_rows) {
    if (locate<false>(a, rows, blockIdx.x, w)) rows_body<D, F16, FORM, FMT>(a, rows, w, stage0, stage1);
  } else {
    if (locate<false>(a, token, blockIdx.x - n_rows, w)) token_body<D, F16, FORM, 2, FMT>(a, token, w, stage0, stage1);
  }
}

template <int D, bool F16, int NQ>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, PagedClass rows, PagedClass token, int n_rows) {
  // few workgroups for the many items there may be: a workgroup without work costs a microsecond, in rounds
  if (static_cast<int>(blockIdx.x) < n_rows) {
    for (int i = blockIdx.x; i < rows.max_joins && join_body<D, F16, kRowsM, 8, kRowsJoins>(a, rows, i); i += n_rows)
      __syncthreads();
  } else {
    constexpr int G = NQ * kTokenJoins;
    for (int i = blockIdx.x - n_rows; i < token.max_joins && join_body<D, F16, NQ * kTokenM, 1, G>(a, token, i);
         i += gridDim.x - n_rows)
      __syncthreads();
  }
}

template <int D, bool F16, bool FORM, int FMT>
int launch(const PagedArgs& a, const Plan& p, hipStream_t st, const char* what) {
  const auto n = [](int64_t x) { return static_cast<unsigned>(x); };
  if (p.rows.items) {
    paged_rows_kernel<D, F16, FORM, FMT><<<n(p.rows.items + p.token.items), 256, 0, st>>>(
        a, p.rows.cls, p.token.cls, static_cast<int>(p.rows.items));
  } else if (p.sets == 1) {
    paged_token_kernel<D, F16, FORM, FMT, 1><<<n(p.token.items), 256, 0, st>>>(a, p.token.cls);
  } else {
    paged_token_kernel<D, F16, FORM, FMT, 2><<<n(p.token.items), 256, 0, st>>>(a, p.token.cls);
  }
  const int64_t joins = std::min(p.rows.cls.max_joins, 2 * kRound);
  const int64_t all = joins + std::min(p.token.cls.max_joins, 2 * kRound);
  if (all) {
    if (p.sets == 1)
      paged_join_kernel<D, F16, 1><<<n(all), 256, 0, st>>>(a, p.rows.cls, p.token.cls, static_cast<int>(joins));
    else
      paged_join_kernel<D, F16, 2><<<n(all), 256, 0, st>>>(a, p.rows.cls, p.token.cls, static_cast<int>(joins));
  }
  return check_launch(what);
}

// Checks a call and fills in the kernels' arguments, but for the workspace.
int make_args(const PagedCall& c, const char* what, int fmt, bool* f16, PagedArgs* to) {
  if (!c.q_strides || !c.k_pages || !c.v_pages || !c.page_strides || !c.table || !c.cu_rows || !c.kv_lens ||
      !c.out_strides || (c.rows > 0 && (!c.query || !c.out)) || (fmt && (!c.k_scales || !c.v_scales || !c.scale_strides)))
    return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  if (const int rc = half_dtype(c.dtype, what, f16)) return rc;
  if (!good_sizes(c.rows, c.requests, c.width, c.page, c.q_heads, c.kv_heads, c.head_dim) || c.table_ld < c.width ||
      c.pages < 1 || c.pages > (1ll << 30) || c.max_rows < 0)
    return fail(QKV_ERR_UNSUPPORTED, "%s: unsupported sizes (head_dim 64 or 128, page a power of two in [16, 4096], "
                "q_heads a multiple of kv_heads and at most %d times as many)", what, kRowsM);
  // so that scaling / softcap, and slopes / scaling, stay finite
  const auto usable = [](float x) { return x >= 0x1p-60f && x <= 0x1p60f; };
  if (!usable(c.scaling) || !(c.softcap == 0.0f || usable(c.softcap)))
    return fail(QKV_ERR_INVALID, "%s: scaling must be in [2^-60, 2^60] and softcap 0 or there", what);
  const int unit = fmt ? 16 : 8;   // strides in 16 bytes
  bool good = aligned(c.k_pages, 16) && aligned(c.v_pages, 16) && aligned(c.out, 16) && c.out_strides[0] % 8 == 0 &&
              c.out_strides[1] % 8 == 0;
  for (int i = 0; i < 3; ++i) good = good && c.page_strides[i] % unit == 0;
  if (!good) return fail(QKV_ERR_INVALID, "%s: pages and output must be 16-byte aligned", what);
  if (c.page_strides[2] < 0 || c.page_strides[2] >= (1 << 30) / c.page)
    return fail(QKV_ERR_UNSUPPORTED, "%s: a page's tokens must lie within 2^30 elements", what);
  if (fmt && (!aligned(c.k_scales, 4) || !aligned(c.v_scales, 4) || c.scale_strides[0] % 4 || c.scale_strides[1] % 4))
    return fail(QKV_ERR_INVALID, "%s: scales must be 4-byte aligned", what);
  PagedArgs a{};
  a.q = static_cast<const uint16_t*>(c.query);
  a.k = static_cast<const uint16_t*>(c.k_pages);
  a.v = static_cast<const uint16_t*>(c.v_pages);
  a.out = static_cast<uint16_t*>(c.out);
  a.q_row = c.q_strides[0], a.q_head = c.q_strides[1];
  a.page = c.page_strides[0], a.head = c.page_strides[1], a.tok = static_cast<uint32_t>(c.page_strides[2]);
  a.o_row = c.out_strides[0], a.o_head = c.out_strides[1];
  a.table = c.table, a.cu = c.cu_rows, a.kv_lens = c.kv_lens, a.prefix = c.prefix_lens, a.first = c.first_keys;
  a.slopes = c.slopes;
  a.table_ld = c.table_ld;
  a.width = static_cast<int>(c.width), a.pages = static_cast<int>(c.pages);
  a.shift = __builtin_ctz(static_cast<unsigned>(c.page));
  a.requests = static_cast<int>(c.requests), a.rows = static_cast<int>(c.rows);
  a.kv_heads = static_cast<int>(c.kv_heads), a.group = static_cast<int>(c.q_heads / c.kv_heads);
  a.per_group = 65536 / a.group + 1;
  a.scale_log2 = c.scaling * kLog2e;
  a.tanh_scale = c.softcap > 0.0f ? 2.0f * kLog2e * c.scaling / c.softcap : 0.0f;
  a.cap_log2 = c.softcap * kLog2e;
  a.wide = c.softcap > kNearCap;
  a.unit_log2 = c.softcap > 0.0f ? 1.0f : a.scale_log2;
  a.slope_unit = c.softcap > 0.0f ? kLog2e : 1.0f / c.scaling;
  if (fmt) {
    a.k_scales = static_cast<const uint8_t*>(c.k_scales), a.v_scales = static_cast<const uint8_t*>(c.v_scales);
    a.s_page = c.scale_strides[0], a.s_head = c.scale_strides[1];
  }
  *to = a;
  return QKV_OK;
}

template <int FMT>
int paged_call(const PagedCall& c, const char* what) {
  bool f16;
  PagedArgs a;
  if (const int rc = make_args(c, what, FMT, &f16, &a)) return rc;
  Plan p = plan_of(c.rows, c.max_rows, c.requests, c.width * c.page, c.kv_heads, a.group,
                   FMT == kHalfPages ? 2 * c.head_dim : FMT == kFp8Pages ? c.head_dim : c.head_dim / 2);
  // a grid has less than 2^32 threads
  if (p.rows.items + p.token.items >= (1 << 24)) return fail(QKV_ERR_UNSUPPORTED, "%s: too many rows", what);
  const int64_t need = workspace_bytes(p, c.head_dim);
  if (need > 0 && (!c.workspace || c.workspace_bytes < need || !aligned(c.workspace, 16)))
    return fail(QKV_ERR_INVALID, "%s: workspace must be 16-byte aligned and hold %lld bytes", what,
                static_cast<long long>(need));
  if (c.rows == 0) return QKV_OK;
  p.rows.cls.acc = static_cast<float*>(c.workspace);
  p.token.cls.acc = p.rows.cls.acc + c.head_dim * p.rows.parts * kRowsM;
  p.rows.cls.ml = p.token.cls.acc + c.head_dim * p.token.parts * p.sets * kTokenM;
  p.token.cls.ml = p.rows.cls.ml + 2 * p.rows.parts * kRowsM;
  hipStream_t st = static_cast<hipStream_t>(c.stream);
  const bool form = c.softcap > 0.0f || c.slopes;
  return with_half(f16, [&](auto h) {
    constexpr bool F = decltype(h)::value;
    if (c.head_dim == 128) return form ? launch<128, F, true, FMT>(a, p, st, what) : launch<128, F, false, FMT>(a, p, st, what);
    return form ? launch<64, F, true, FMT>(a, p, st, what) : launch<64, F, false, FMT>(a, p, st, what);
  });
}

}  // namespace
}  // namespace qkv
