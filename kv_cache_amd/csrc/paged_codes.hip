// Quantised pages of a paged K/V cache: rows written as codes of 8 or 4 bits with a scale for each 32 channels, and
// tokens read back as rows.
//
// A block's scale is 2^e, e the least integer from -100 on with amax <= T 2^e: T = 464 (e4m3) or 7 (e2m1), up to which a
// magnitude still rounds to the largest code, 448 or 6, so that no value is off by more than half a step.  Powers of two
// make every step of it exact but the one rounding, x 2^-e to the nearest code, halves to the even one; a 16-bit value of
// the cache's dtype holds each code times its scale, so reading back rounds nothing (below 2^-14 fp16 has fewer bits).
// Magnitudes whose code would stand for more than the dtype holds (over 1.875 * 2^15 or 1.5 * 2^15 in fp16, 2^127 in bf16)
// take that largest value.  A block with an infinity or NaN has the scale byte 255 and reads as NaN.
//
// Both kernels move 16 bytes of 16-bit rows a thread and array, so four threads a block: the maximum of a block takes
// two moves within a quad.  Bound by memory: 2 + 1/32 + 1 (or 1/2) bytes a value (8188 rows of 8 x 128 into fp8: 11.8 us,
// 4.3 TB/s; 31385 tokens read back: 33 us, 5.8 TB/s; few rows: 2.8 and 3.8 us, dependent loads).
#include "paged_tiles.h"

namespace qkv {
namespace {

// The rows, or tokens, of a call.
struct RowsOf {
  const int64_t* slots;                                   // of append
  const int32_t *table, *cu, *kv_lens;                    // of read
  int64_t table_ld;
  int requests, width;
  int rows, shift, units_head, units_row, pages, per_wg;
};
struct Rows16 {
  uint16_t *k, *v;
  int64_t k_row, k_head, v_row, v_head;
};
struct CodePages {
  uint8_t *k, *v, *k_scales, *v_scales;
  int64_t page, head, tok, s_page, s_head;   // strides in bytes, K's and V's
};

template <int FMT>
struct Coding {   // largest code, what of the largest 16-bit exponent it may take, its edge in a scale's bits
  static constexpr float most = FMT == kFp8Pages ? 448.0f : 6.0f;
  static constexpr uint32_t fraction = FMT == kFp8Pages ? 0x700000u : 0x400000u;   // of 1.875; of 1.5
  // e + 127 = exponent of amax - below, one more where its fraction is over that of T (0.8125, 0.75)
  static constexpr uint32_t carry = 0x7FFFFFu - (FMT == kFp8Pages ? 0x680000u : 0x600000u);
  static constexpr int below = FMT == kFp8Pages ? 8 : 2;
};

// Eight channels: their codes and the block's scale byte.
template <bool F16, int FMT>
__device__ __forceinline__ u32x2_t encode8(uint4 x, uint32_t& scale) {
  using C = Coding<FMT>;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  float f[8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = half_lo<F16>(w[i]), f[2 * i + 1] = half_hi<F16>(w[i]);
    top = max(top, max(__float_as_uint(f[2 * i]) & 0x7FFFFFFFu, __float_as_uint(f[2 * i + 1]) & 0x7FFFFFFFu));
  }
  top = max(top, dpp_mov<0xB1>(top, top));   // over the quad
  top = max(top, dpp_mov<0x4E>(top, top));
  const bool odd = top >= 0x7F800000u;
  constexpr uint32_t limit = (F16 ? (127u + 15u) << 23 : (127u + 127u) << 23) | C::fraction;
  const int byte = max(static_cast<int>((min(top, limit) + C::carry) >> 23) - C::below, 27);
  scale = odd ? 255u : static_cast<uint32_t>(byte);
  const float inv = odd ? 0.0f : __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float l = __uint_as_float(limit), z = __builtin_amdgcn_fmed3f(f[i], -l, l);
    const float y = __builtin_amdgcn_fmed3f(z * inv, -C::most, C::most);
    f[i] = odd ? 0.0f : y;   // (0 times an infinity is NaN)
  }
  u32x2_t c{0u, 0u};
  if constexpr (FMT == kFp8Pages) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int y = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
      y = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], y, true);
      c[i] = static_cast<uint32_t>(y);
    }
  } else {
    uint32_t y = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0], f[1], 1.0f, 0);
    y = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(y, f[2], f[3], 1.0f, 1);
    y = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(y, f[4], f[5], 1.0f, 2);
    c[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(y, f[6], f[7], 1.0f, 3);
  }
  return c;
}

template <int FMT>
__device__ __forceinline__ void store_codes(uint8_t* row, int c, u32x2_t x) {
  if constexpr (FMT == kFp8Pages) *reinterpret_cast<u32x2_t*>(row + c) = x;
  else *reinterpret_cast<uint32_t*>(row + c / 2) = x[0];
}

template <bool F16, int FMT>
__global__ __launch_bounds__(256) void append_codes_kernel(RowsOf r, Rows16 x, CodePages p) {
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = u / r.units_row;
  if (row >= r.rows) return;   // (a quad belongs to one row)
  const int64_t slot = r.slots[row];
  if (slot < 0 || slot >= static_cast<int64_t>(r.pages) << r.shift) return;
  const int in_row = static_cast<int>(u - row * r.units_row);
  const int head = in_row / r.units_head, c = 8 * (in_row - head * r.units_head);
  const int64_t id = slot >> r.shift, at = slot & ((1 << r.shift) - 1);
  const uint4 k = load16u(x.k + row * x.k_row + head * x.k_head + c);
  const uint4 v = load16u(x.v + row * x.v_row + head * x.v_head + c);
  uint32_t ks, vs;
  const u32x2_t kc = encode8<F16, FMT>(k, ks), vc = encode8<F16, FMT>(v, vs);
  const int64_t to = id * p.page + head * p.head + at * p.tok;
  store_codes<FMT>(p.k + to, c, kc);
  store_codes<FMT>(p.v + to, c, vc);
  if ((threadIdx.x & 3) == 0) {
    const int64_t s = id * p.s_page + head * p.s_head + at * (r.units_head / 4) + c / kScaleBlock;
    p.k_scales[s] = static_cast<uint8_t>(ks);
    p.v_scales[s] = static_cast<uint8_t>(vs);
  }
}

// Eight channels of a token as 16-bit values.
template <bool F16, int FMT>
__device__ __forceinline__ u32x4_t decode8(const uint8_t* row, const uint8_t* scales, int c) {
  if constexpr (FMT == kHalfPages) return *reinterpret_cast<const u32x4_t*>(row + 2 * c);
  if constexpr (FMT == kFp8Pages) {
    const u32x2_t w = *reinterpret_cast<const u32x2_t*>(row + c);
    return values8<F16, FMT>(w[0], w[1], scales[c / kScaleBlock]);
  }
  return values8<F16, FMT>(*reinterpret_cast<const uint32_t*>(row + c / 2), 0, scales[c / kScaleBlock]);
}

// A workgroup's first threads find its rows' requests and slots, then all of them move the rows.
template <bool F16, int FMT>
__global__ __launch_bounds__(256) void read_kernel(RowsOf r, Rows16 x, CodePages p) {
  __shared__ int64_t s_slot[256];   // -1: zeros, -2: no request's row
  const int tid = threadIdx.x;
  const int row0 = blockIdx.x * r.per_wg, n = min(r.per_wg, r.rows - row0);
  if (tid < n) {
    const int row = row0 + tid;
    int lo = 0, hi = r.requests;   // the last b with cu[b] <= row, as binary search has it (cu ascends)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (r.cu[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    int64_t slot = -2;
    if (lo < r.requests && r.cu[lo] <= row) {
      const int64_t pos = static_cast<int64_t>(r.kv_lens[lo]) - (r.cu[lo + 1] - row);
      slot = -1;
      if (pos >= 0 && pos >> r.shift < r.width) {
        const int id = r.table[lo * r.table_ld + (pos >> r.shift)];
        if (static_cast<unsigned>(id) < static_cast<unsigned>(r.pages))
          slot = (static_cast<int64_t>(id) << r.shift) + (pos & ((1 << r.shift) - 1));
      }
    }
    s_slot[tid] = slot;
  }
  __syncthreads();
  for (int u = tid; u < n * r.units_row; u += 256) {
    const int i = u / r.units_row, in_row = u - i * r.units_row;
    const int head = in_row / r.units_head, c = 8 * (in_row - head * r.units_head);
    const int64_t slot = s_slot[i], row = row0 + i;
    if (slot == -2) continue;
    u32x4_t k{0u, 0u, 0u, 0u}, v = k;
    if (slot >= 0) {
      const int64_t id = slot >> r.shift, at = slot & ((1 << r.shift) - 1);
      const int64_t from = id * p.page + head * p.head + at * p.tok;
      const int64_t s = FMT == kHalfPages ? 0 : id * p.s_page + head * p.s_head + at * (r.units_head / 4);
      k = decode8<F16, FMT>(p.k + from, p.k_scales + s, c);
      v = decode8<F16, FMT>(p.v + from, p.v_scales + s, c);
    }
    *reinterpret_cast<u32x4_t*>(x.k + row * x.k_row + head * x.k_head + c) = k;
    *reinterpret_cast<u32x4_t*>(x.v + row * x.v_row + head * x.v_head + c) = v;
  }
}

// Checks what both calls share and fills it in.
int make_pages(const char* what, int code, const void* k_pages, const void* v_pages, const int64_t* page_strides,
               const void* k_scales, const void* v_scales, const int64_t* scale_strides, int64_t pages, int64_t page,
               int64_t kv_heads, int64_t head_dim, int64_t rows, RowsOf* r, CodePages* p) {
  if (!k_pages || !v_pages || !page_strides || (code && (!k_scales || !v_scales || !scale_strides)))
    return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  if (rows < 0 || rows > (1 << 30) || pages < 1 || pages > (1ll << 30) || kv_heads < 1 || kv_heads > 65536 ||
      head_dim < kScaleBlock || head_dim > 65536 || head_dim % kScaleBlock)
    return fail(QKV_ERR_INVALID, "%s: bad sizes (head_dim must be a multiple of %d)", what, kScaleBlock);
  if (page < 16 || page > 4096 || (page & (page - 1)))
    return fail(QKV_ERR_UNSUPPORTED, "%s: page must be a power of two in [16, 4096], got %lld", what,
                static_cast<long long>(page));
  const int unit = code ? 16 : 8;
  for (int i = 0; i < 3; ++i)
    if (page_strides[i] % unit || !aligned(k_pages, 16) || !aligned(v_pages, 16))
      return fail(QKV_ERR_INVALID, "%s: page rows must be 16-byte aligned", what);
  const int64_t bytes = code ? 1 : 2;
  *p = CodePages{static_cast<uint8_t*>(const_cast<void*>(k_pages)), static_cast<uint8_t*>(const_cast<void*>(v_pages)),
                 static_cast<uint8_t*>(const_cast<void*>(k_scales)), static_cast<uint8_t*>(const_cast<void*>(v_scales)),
                 bytes * page_strides[0], bytes * page_strides[1], bytes * page_strides[2],
                 code ? scale_strides[0] : 0, code ? scale_strides[1] : 0};
  r->units_head = static_cast<int>(head_dim / 8);
  if (r->units_head * kv_heads > (1 << 20)) return fail(QKV_ERR_UNSUPPORTED, "%s: too many channels", what);
  r->units_row = static_cast<int>(r->units_head * kv_heads);
  r->rows = static_cast<int>(rows), r->pages = static_cast<int>(pages);
  r->shift = __builtin_ctz(static_cast<unsigned>(page));
  return QKV_OK;
}

}  // namespace
}  // namespace qkv

using namespace qkv;

QKV_EXPORT int qkv_paged_append_codes(const void* key, const int64_t* key_strides, const void* value,
                                      const int64_t* value_strides, void* k_pages, void* v_pages,
                                      const int64_t* page_strides, void* k_scales, void* v_scales,
                                      const int64_t* scale_strides, int code, int64_t pages, int64_t page,
                                      int64_t kv_heads, int64_t head_dim, const int64_t* slots, int64_t rows, int dtype,
                                      void* stream) {
  const char* what = "qkv_paged_append_codes";
  if (code != QKV_CODE_FP8 && code != QKV_CODE_FP4)
    return fail(QKV_ERR_INVALID, "%s: code %d is not fp8 (%d) or fp4 (%d)", what, code, QKV_CODE_FP8, QKV_CODE_FP4);
  if (!key_strides || !value_strides || (rows > 0 && (!key || !value || !slots)))
    return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  bool f16;
  if (const int rc = half_dtype(dtype, what, &f16)) return rc;
  RowsOf r{};
  CodePages p;
  if (const int rc = make_pages(what, code, k_pages, v_pages, page_strides, k_scales, v_scales, scale_strides, pages, page,
                                kv_heads, head_dim, rows, &r, &p))
    return rc;
  const int64_t grid = cdiv(rows * r.units_row, 256);
  // a grid has less than 2^32 threads
  if (grid >= (1 << 24)) return fail(QKV_ERR_UNSUPPORTED, "%s: too many rows", what);
  if (rows == 0) return QKV_OK;
  r.slots = slots;
  Rows16 x{static_cast<uint16_t*>(const_cast<void*>(key)), static_cast<uint16_t*>(const_cast<void*>(value)), key_strides[0],
           key_strides[1], value_strides[0], value_strides[1]};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_half(f16, [&](auto h) {
    constexpr bool F = decltype(h)::value;
    if (code == QKV_CODE_FP8) append_codes_kernel<F, kFp8Pages><<<static_cast<unsigned>(grid), 256, 0, st>>>(r, x, p);
    else append_codes_kernel<F, kFp4Pages><<<static_cast<unsigned>(grid), 256, 0, st>>>(r, x, p);
    return check_launch(what);
  });
}

QKV_EXPORT int qkv_paged_read(const void* k_pages, const void* v_pages, const int64_t* page_strides, const void* k_scales,
                              const void* v_scales, const int64_t* scale_strides, int code, int64_t pages, int64_t page,
                              int64_t kv_heads, int64_t head_dim, const int32_t* table, int64_t table_ld, int64_t width,
                              int64_t requests, const int32_t* cu_rows, const int32_t* kv_lens, int64_t rows, void* key,
                              const int64_t* key_strides, void* value, const int64_t* value_strides, int dtype,
                              void* stream) {
  const char* what = "qkv_paged_read";
  if (code < 0 || code > QKV_CODE_FP4)
    return fail(QKV_ERR_INVALID, "%s: code %d is not 0, fp8 (%d) or fp4 (%d)", what, code, QKV_CODE_FP8, QKV_CODE_FP4);
  if (!table || !cu_rows || !kv_lens || !key_strides || !value_strides || (rows > 0 && (!key || !value)))
    return fail(QKV_ERR_INVALID, "%s: null pointer", what);
  bool f16;
  if (const int rc = half_dtype(dtype, what, &f16)) return rc;
  RowsOf r{};
  CodePages p;
  if (const int rc = make_pages(what, code, k_pages, v_pages, page_strides, k_scales, v_scales, scale_strides, pages, page,
                                kv_heads, head_dim, rows, &r, &p))
    return rc;
  if (requests < 1 || requests > (1 << 20) || width < 1 || width > (1ll << 30) / page || table_ld < width)
    return fail(QKV_ERR_INVALID, "%s: bad sizes of the table", what);
  if (!aligned(key, 16) || !aligned(value, 16) || key_strides[0] % 8 || key_strides[1] % 8 || value_strides[0] % 8 ||
      value_strides[1] % 8)
    return fail(QKV_ERR_INVALID, "%s: rows must be 16-byte aligned", what);
  if (rows == 0) return QKV_OK;
  r.table = table, r.cu = cu_rows, r.kv_lens = kv_lens, r.table_ld = table_ld;
  r.requests = static_cast<int>(requests), r.width = static_cast<int>(width);
  // enough workgroups to fill the GPU first, then up to 2048 units a workgroup, eight a thread
  r.per_wg = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({rows / 1024, 2048 / r.units_row, 256})));
  const int64_t grid = cdiv(rows, r.per_wg);
  if (grid >= (1 << 24)) return fail(QKV_ERR_UNSUPPORTED, "%s: too many rows", what);
  Rows16 x{static_cast<uint16_t*>(key), static_cast<uint16_t*>(value), key_strides[0], key_strides[1], value_strides[0],
           value_strides[1]};
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_half(f16, [&](auto h) {
    constexpr bool F = decltype(h)::value;
    const unsigned g = static_cast<unsigned>(grid);
    if (code == QKV_CODE_FP8) read_kernel<F, kFp8Pages><<<g, 256, 0, st>>>(r, x, p);
    else if (code == QKV_CODE_FP4) read_kernel<F, kFp4Pages><<<g, 256, 0, st>>>(r, x, p);
    else read_kernel<F, kHalfPages><<<g, 256, 0, st>>>(r, x, p);
    return check_launch(what);
  });
}
