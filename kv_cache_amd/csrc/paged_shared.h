// Attention of requests that continue another request's tokens, their parent's: each parent's keys are read for all rows
// behind it together, once for every tile of 128 (row, query head)s.
//
// A row sees its parent's tokens and then its own request's up to itself.  A tile holds either rows of one request over
// its own keys, or heirs of one parent, of whatever requests, over the parent's; tiles are those of the two bodies of
// paged_tiles.h, and one launch does both kinds.  The tiles' keys are split into chunks of about the same length, so that
// the launch's workgroups are as even as they can be; a (row, head)'s parts, its own and its parent's, are joined by a
// second launch in their order.  Only tiles in one chunk of rows without a parent write the output themselves.
// 64 requests behind 32768 tokens, up to 600 of their own, 32/8 heads: 67 us and 7 for the join (843 us where every
// request reads the prefix itself); twice the prefix takes 36 us more, the rate of a large library product.
#pragma once

#include "paged_tiles.h"

namespace qkv {
namespace {

constexpr int kRounds = 2;         // most workgroups that chunks are cut for, in rounds of those that run at once
constexpr int kLaneRequests = 2;   // requests of a lane in the search of a workgroup's work without barriers

struct SharedArgs {
  PagedClass rows, token;   // acc and ml of rows serve both
  int token_units;          // of kPartUnit rows in a part of the token class
  int max_units;
};

// What request b has to be done: [0] its heirs over its tokens, [1] its rows over their own.
struct Shares {
  int nt[2], keys[2], n_rows[2], row0[2];
};

// Which work workgroup `item` has: 0 none, 1 rows' tile, 2 a token tile.
__device__ __forceinline__ int locate_shared(const PagedArgs& a, const SharedArgs& c, int item, Where& w) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float per_rows = 1.0f / static_cast<float>(c.rows.tokens), per_token = 1.0f / static_cast<float>(max(c.token.tokens, 1));
  auto shares_of = [&](int b) {
    Shares s{};
    if (b >= a.requests) return s;
    const auto tokens_of = [&](int n) { return min(max(n, 0), a.width << a.shift); };   // (at most 2^30)
    s.n_rows[1] = rows_of(a, b, s.row0[1]);
    s.keys[1] = tokens_of(a.kv_lens[b]);
    s.row0[0] = min(max(a.heirs_cu[b], 0), a.rows);
    s.n_rows[0] = min(max(a.heirs_cu[b + 1], s.row0[0]), a.rows) - s.row0[0];
    s.keys[0] = tokens_of(a.parent_lens[b]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // ceil(rows / tokens of a tile): half a row from the next whole number, which 2^20 rows are not rounded over
      const float per = s.n_rows[i] > c.token.tokens ? per_rows : per_token;
      s.nt[i] = s.n_rows[i] ? static_cast<int>((static_cast<float>(s.n_rows[i]) - 0.5f) * per) + 1 : 0;
    }
    return s;
  };
  // one more or less is as good: what a chunk holds follows from their number (below)
  auto splits_of = [&](int keys) {
    return keys > w.chunk ? static_cast<int>(static_cast<float>(keys - 1) * __builtin_amdgcn_rcpf(static_cast<float>(w.chunk))) + 1 : 1;
  };
  auto units_of = [&](int n_rows) { return n_rows > c.token.tokens ? kRowsM / kPartUnit : c.token_units; };
  auto work_of = [&](const Shares& s) {
    return static_cast<float>(s.nt[0]) * static_cast<float>(s.keys[0]) +
           static_cast<float>(s.nt[1]) * static_cast<float>(s.keys[1]);
  };
  auto round_up = [&](float keys) {
    const int least = max(c.rows.min_keys, static_cast<int>(fminf(keys, 1073741824.0f)) + 1);
    return __builtin_amdgcn_readfirstlane((least + kTile - 1) & -kTile);
  };
  // How much of the workgroups that run at once a request's tiles take under w.chunk: a chunk counts as one, keys that fill
  // none as their share and what a workgroup costs by itself.
  auto slots_of = [&](const Shares& s) {
    const float per = __builtin_amdgcn_rcpf(static_cast<float>(w.chunk));
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float share = static_cast<float>(s.keys[i]) * per;
      sum += static_cast<float>(s.nt[i]) * (share > 1.0f ? ceilf(share) : fminf(1.0f, share + 0.1f));
    }
    return sum * a.kv_heads;
  };
  // One round of chunks where one comes out, up to a fifth longer than the work's share (64 requests behind 32768 keys: 82
  // us in all, 92 in two rounds), else two.
  auto set_chunk = [&](float per, auto&& slots) {
    for (int i = 0; i < 4; ++i) {
      w.chunk = round_up(per * (1.0f + 0.0667f * i));
      if (slots() <= static_cast<float>(kRound)) return;
    }
    w.chunk = round_up(per * 0.5f);
  };
  int kind, at, nt;
  const int parts = (a.requests + 63) >> 6;   // of 64 requests
  if (parts <= kLaneRequests) {
    // every wave for itself, kLaneRequests a lane
    Shares s[kLaneRequests];
    float work = 0.0f;
#pragma unroll
    for (int k = 0; k < kLaneRequests; ++k) {
      s[k] = Shares{};
      if (k < parts) s[k] = shares_of(64 * k + lane);
      work += work_of(s[k]);
    }
    set_chunk(wave_total(work) * a.kv_heads * c.rows.per_round, [&] {
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < kLaneRequests; ++k)
        if (k < parts) sum += slots_of(s[k]);
      return wave_total(sum);
    });
    int item0 = 0, unit0 = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < kLaneRequests; ++k) {
        if (found || k >= parts) continue;   // the same for every lane
        const int ns = splits_of(s[k].keys[i]), items = s[k].nt[i] * a.kv_heads * ns;
        const int mine = items * units_of(s[k].n_rows[i]), up = wave_scan(items), up_units = wave_scan(mine);
        const int begin = item0 + up - items, unit = unit0 + up_units - mine;
        const uint64_t hit = __ballot(item >= begin && item - begin < items);
        if (hit) {
          const int from = __builtin_ctzll(hit);
          found = true;
          kind = i;
          w.b = 64 * k + from;
          at = item - __builtin_amdgcn_readlane(begin, from);
          w.part = __builtin_amdgcn_readlane(unit, from);
          nt = __builtin_amdgcn_readlane(s[k].nt[i], from);
          w.kv = __builtin_amdgcn_readlane(s[k].keys[i], from);
          w.n_split = __builtin_amdgcn_readlane(ns, from);
          w.row0 = __builtin_amdgcn_readlane(s[k].row0[i], from);
          w.n_rows = __builtin_amdgcn_readlane(s[k].n_rows[i], from);
        }
        item0 += __builtin_amdgcn_readlane(up, 63);
        unit0 += __builtin_amdgcn_readlane(up_units, 63);
      }
    if (!found) return 0;
  } else {
    __shared__ float s_tot[4];
    __shared__ int s_part[8], s_hit[9];
    auto total = [&](auto&& f) {   // over all requests; the same in every thread
      float sum = 0.0f;
      for (int b0 = 0; b0 < a.requests; b0 += 256) sum += f(shares_of(b0 + tid));
      sum = wave_total(sum);
      __syncthreads();
      if (lane == 0) s_tot[wave] = sum;
      __syncthreads();
      return (s_tot[0] + s_tot[1]) + (s_tot[2] + s_tot[3]);
    };
    if (tid == 0) s_hit[0] = -1;
    set_chunk(total(work_of) * a.kv_heads * c.rows.per_round, [&] { return total(slots_of); });
    int carry = 0, unit_carry = 0;
    for (int i = 0; i < 2; ++i) {
      for (int b0 = 0; b0 < a.requests; b0 += 256) {
        const Shares s = shares_of(b0 + tid);
        const int ns = splits_of(i ? s.keys[1] : s.keys[0]), tiles = i ? s.nt[1] : s.nt[0], n = i ? s.n_rows[1] : s.n_rows[0];
        const int items = tiles * a.kv_heads * ns, mine = items * units_of(n);
        const int up = wave_scan(items), up_units = wave_scan(mine);
        __syncthreads();
        if (lane == 63) {
          s_part[2 * wave] = up;
          s_part[2 * wave + 1] = up_units;
        }
        __syncthreads();
        int begin = carry + up - items, unit = unit_carry + up_units - mine;
        for (int v = 0; v < 4; ++v) {
          if (v < wave) {
            begin += s_part[2 * v];
            unit += s_part[2 * v + 1];
          }
          carry += s_part[2 * v];
          unit_carry += s_part[2 * v + 1];
        }
        if (item >= begin && item - begin < items) {   // one thread at most
          s_hit[0] = b0 + tid;
          s_hit[1] = item - begin;
          s_hit[2] = unit;
          s_hit[3] = tiles;
          s_hit[4] = i ? s.keys[1] : s.keys[0];
          s_hit[5] = ns;
          s_hit[6] = i ? s.row0[1] : s.row0[0];
          s_hit[7] = n;
          s_hit[8] = i;
        }
        __syncthreads();
        if (s_hit[0] >= 0 || item < carry) break;   // the same for every thread
      }
      if (s_hit[0] >= 0 || item < carry) break;
    }
    w.b = __builtin_amdgcn_readfirstlane(s_hit[0]);
    if (w.b < 0) return 0;
    at = __builtin_amdgcn_readfirstlane(s_hit[1]);
    w.part = __builtin_amdgcn_readfirstlane(s_hit[2]);
    nt = __builtin_amdgcn_readfirstlane(s_hit[3]);
    w.kv = __builtin_amdgcn_readfirstlane(s_hit[4]);
    w.n_split = __builtin_amdgcn_readfirstlane(s_hit[5]);
    w.row0 = __builtin_amdgcn_readfirstlane(s_hit[6]);
    w.n_rows = __builtin_amdgcn_readfirstlane(s_hit[7]);
    kind = __builtin_amdgcn_readfirstlane(s_hit[8]);
  }
  w.heirs = kind == 0;
  w.alone = !w.heirs && a.before[w.b] <= 0;
  const int units = units_of(w.n_rows);
  // as many keys for each of the tile's chunks, all of them in one
  w.chunk = w.kv;
  if (w.n_split > 1) w.chunk = __builtin_amdgcn_readfirstlane(((w.kv + w.n_split - 1) / w.n_split + kTile - 1) & -kTile);
  const int rest = __builtin_amdgcn_readfirstlane(at / a.kv_heads);
  w.head = at - rest * a.kv_heads;
  w.split = __builtin_amdgcn_readfirstlane(rest / nt);
  w.tile = nt - 1 - (rest - w.split * nt);
  w.part += (w.head * nt + w.tile) * w.n_split * units;
  // always so where the rows ascend; otherwise nothing is written out of bounds
  if (w.part < 0 || w.part > c.max_units - w.n_split * units) return 0;
  w.part += w.split * units;
  return w.n_rows > c.token.tokens ? 1 : 2;
}

template <int D, bool F16, bool FORM, int FMT, int NQ>
__global__ __launch_bounds__(256, D == 64 && !FORM ? 3 : 2) void paged_shared_kernel(PagedArgs a, SharedArgs c) {
  __shared__ __attribute__((aligned(16))) uint16_t stage0[2 * kTile * D], stage1[2 * kTile * D];
  Where w;
  const int kind = locate_shared(a, c, blockIdx.x, w);
  if (kind == 1) rows_body<D, F16, FORM, FMT, true>(a, c.rows, w, stage0, stage1);
  else if (kind == 2) token_body<D, F16, FORM, NQ, FMT, true>(a, c.token, w, stage0, stage1);
}

// Joins the parts of R (row, query head)s a workgroup, each in 256 / (R * D / 4) groups that take every so many'th part
// and are then joined in order.
template <int D, bool F16, int R>
__global__ __launch_bounds__(256) void paged_shared_join_kernel(PagedArgs a, SharedArgs c) {
  constexpr int L = D / 4, P = 256 / (R * L);   // lanes of a (row, head), 4 values each; groups
  __shared__ float s_acc[P][R][D], s_m[P][R], s_l[P][R];
  const int in = threadIdx.x / L % R, group = threadIdx.x / (L * R), d0 = 4 * (threadIdx.x % L);
  const int heads = a.kv_heads * a.group;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * R + in;
  const int64_t row = pair / heads;
  const int head = static_cast<int>(pair - row * heads), kv = head / a.group;
  const float ninf = -__builtin_huge_valf();
  int n[2] = {0, 0}, step[2] = {0, 0};
  int64_t from[2] = {0, 0};
  bool on = false;
  if (row < a.rows) {
    const int rank = a.rank[row];
    if (rank >= -1 && rank < a.rows) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {   // its own, its parent's
        if (i == 1 && rank < 0) break;
        const int2 e = a.at[(i ? static_cast<int64_t>(a.rows) + rank : row) * a.kv_heads + kv];
        n[i] = e.y >> 4;
        step[i] = (e.y & 15) * kPartUnit;
        from[i] = e.x + head - kv * a.group;
        // always so where the rows ascend
        if (n[i] < 0 || e.x < 0 || step[i] == 0 || from[i] + static_cast<int64_t>(max(n[i] - 1, 0)) * step[i] >= static_cast<int64_t>(c.max_units) * kPartUnit)
          n[i] = 0;
        if (i == 0) on = n[0] > 0;   // else the output is written already
      }
    }
  }
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
  const int all = on ? n[0] + n[1] : 0;
  constexpr int U = 4;   // parts whose loads are issued together
  for (int s0 = group; s0 < all; s0 += U * P) {
    float mp[U], lp[U];
    float4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = min(s0 + u * P, all - 1);
      const int64_t p = s < n[0] ? from[0] + static_cast<int64_t>(s) * step[0] : from[1] + static_cast<int64_t>(s - n[0]) * step[1];
      mp[u] = c.rows.ml[2 * p];
      lp[u] = c.rows.ml[2 * p + 1];
      x[u] = *reinterpret_cast<const float4*>(c.rows.acc + p * D + d0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * P < all) add(mp[u], lp[u], x[u]);
  }
  if constexpr (P > 1) {
    *reinterpret_cast<float4*>(&s_acc[group][in][d0]) = y;
    if (d0 == 0) {
      s_m[group][in] = m;
      s_l[group][in] = l;
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int p = 1; p < P; ++p) add(s_m[p][in], s_l[p][in], *reinterpret_cast<const float4*>(&s_acc[p][in][d0]));
  }
  if (!on) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const float z[4] = {y.x * inv, y.y * inv, y.z * inv, y.w * inv};
  *reinterpret_cast<u32x2_t*>(a.out + row * a.o_row + head * a.o_head + d0) = pack4_half<F16>(z);
}

// The launches of a call.  Tiles: one for each request with rows and one for each of its heirs' parents, and those that
// full tiles of rows make; where keys are split, sum over the tiles of ceil(keys / chunk) <= rounds + tiles.
struct SharedShape {
  SharedArgs c;
  int sets;
  int64_t items, units;
};
SharedShape shared_shape_of(int64_t rows, int64_t max_rows, int64_t requests, int64_t max_keys, int64_t kv_heads,
                            int64_t group) {
  SharedShape s{};
  s.sets = std::max<int64_t>(max_rows, 1) * group <= kTokenM ? 1 : 2;
  s.c.token_units = s.sets * kTokenM / kPartUnit;
  s.c.token.tokens = static_cast<int>(s.sets * kTokenM / group);
  s.c.rows.tokens = static_cast<int>(kRowsM / group);
  s.c.rows.min_keys = 256;
  s.c.rows.per_round = 1.0001f / static_cast<float>(kRound);
  const int64_t some = std::min(requests, rows), more = max_keys > 256 ? kRounds * kRound : 0;
  const int64_t large = rows > s.c.token.tokens ? 2 * kv_heads * (rows / s.c.rows.tokens + std::min(requests, rows / (s.c.token.tokens + 1))) + more : 0;
  const int64_t small = s.c.token.tokens ? 2 * kv_heads * some + more : 0;
  s.items = 2 * kv_heads * (some + rows / s.c.rows.tokens) + more;
  s.units = large * (kRowsM / kPartUnit) + small * s.c.token_units;
  return s;
}
int64_t shared_bytes(const SharedShape& s, int64_t rows, int64_t kv_heads, int64_t head_dim) {
  return s.units * kPartUnit * 4 * (head_dim + 2) + 16 * rows * kv_heads;
}

// What a call may have: a grid has less than 2^32 threads, and the parts' rows are counted in 31 bits.
constexpr int64_t kMaxPairs = 1 << 26;   // (row, query head)s
bool good_shared(const SharedShape& s, int64_t rows, int64_t requests, int64_t q_heads) {
  return requests <= kMaxPlanned && rows <= kMaxPlannedRows && s.items < (1 << 24) && s.units < (1 << 27) &&
         rows * q_heads < kMaxPairs;
}

template <int D, bool F16, bool FORM, int FMT>
int launch_shared(const PagedArgs& a, const SharedShape& s, hipStream_t st, const char* what) {
  const unsigned n = static_cast<unsigned>(s.items);
  if (s.sets == 1) paged_shared_kernel<D, F16, FORM, FMT, 1><<<n, 256, 0, st>>>(a, s.c);
  else paged_shared_kernel<D, F16, FORM, FMT, 2><<<n, 256, 0, st>>>(a, s.c);
  const int64_t pairs = static_cast<int64_t>(a.rows) * a.kv_heads * a.group;
  // The fewer (row, head)s, the more parts each has: few have a workgroup each, more four a workgroup (51 requests' 7
  // drafts: 99 us in all, 106 with one), many, of prompts, eight.
  if (pairs <= 1024) paged_shared_join_kernel<D, F16, 1><<<static_cast<unsigned>(pairs), 256, 0, st>>>(a, s.c);
  else if (pairs <= 16384) paged_shared_join_kernel<D, F16, 4><<<static_cast<unsigned>(cdiv(pairs, 4)), 256, 0, st>>>(a, s.c);
  else paged_shared_join_kernel<D, F16, 8><<<static_cast<unsigned>(cdiv(pairs, 8)), 256, 0, st>>>(a, s.c);
  return check_launch(what);
}

template <int FMT>
int shared_call(const PagedCall& c, const int32_t* plan, const char* what) {
  bool f16;
  PagedArgs a;
  if (const int rc = make_args(c, what, FMT, &f16, &a)) return rc;
  if (!plan) return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  SharedShape s = shared_shape_of(c.rows, c.max_rows, c.requests, c.width * c.page, c.kv_heads, a.group);
  if (!good_shared(s, c.rows, c.requests, c.q_heads))
    return fail(QKV_ERR_UNSUPPORTED, "%s: too many rows or requests (at most %d requests and %lld rows, and fewer than %lld "
                "rows times query heads), got %lld requests, %lld rows, %lld heads", what, kMaxPlanned,
                static_cast<long long>(kMaxPlannedRows), static_cast<long long>(kMaxPairs), static_cast<long long>(c.requests),
                static_cast<long long>(c.rows), static_cast<long long>(c.q_heads));
  const int64_t need = shared_bytes(s, c.rows, c.kv_heads, c.head_dim);
  if (c.rows > 0 && (!c.workspace || c.workspace_bytes < need || !aligned(c.workspace, 16)))
    return fail(QKV_ERR_INVALID, "%s: workspace must be 16-byte aligned and hold %lld bytes", what,
                static_cast<long long>(need));
  if (c.rows == 0) return QKV_OK;
  const SharedPlan p(const_cast<int32_t*>(plan), c.rows, c.requests);
  a.positions = p.positions, a.rank = p.rank, a.order = p.order, a.heirs_cu = p.heirs_cu, a.parent_lens = p.parent_lens,
  a.before = p.before;
  s.c.max_units = static_cast<int>(s.units);
  s.c.rows.acc = s.c.token.acc = static_cast<float*>(c.workspace);
  s.c.rows.ml = s.c.token.ml = s.c.rows.acc + c.head_dim * s.units * kPartUnit;
  a.at = reinterpret_cast<int2*>(s.c.rows.ml + 2 * s.units * kPartUnit);
  hipStream_t st = static_cast<hipStream_t>(c.stream);
  const bool form = c.softcap > 0.0f || c.slopes;
  return with_half(f16, [&](auto h) {
    constexpr bool F = decltype(h)::value;
    if (c.head_dim == 128)
      return form ? launch_shared<128, F, true, FMT>(a, s, st, what) : launch_shared<128, F, false, FMT>(a, s, st, what);
    return form ? launch_shared<64, F, true, FMT>(a, s, st, what) : launch_shared<64, F, false, FMT>(a, s, st, what);
  });
}

}  // namespace
}  // namespace qkv
