// origami_append.hip -- new tokens into the paged KV cache: queries and keys normalised per
// head and rotated to their positions on the way, keys and values written to their slots.
//
// For a row x of D channels (one token, one head):
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w          (where a norm weight is given)
//   for each pair (a, b) of the rotated channels, with the position's cos and sin:
//   a' = a cos - b sin,  b' = b cos + a sin          (where a table is given)
// in binary32, rounded once, to the type that is stored.
//
// Every row is read and written once.  L lanes take a row, 8 channels each (16 bytes of a 16-bit
// row), so that the mean and a pair's partner are exchanged between lanes of one wave and nothing
// goes through LDS; the query, key and value rows of all tokens are one launch, since a decode
// step has far too few rows to fill one with each.
//
// Instructions bound it before memory does: of the 16 bytes that a lane moves, a hundred or two.
// So a workgroup is one wave with rows of one kind of one token, whose pointers, strides, slot,
// position and angles are then scalar, the sum over a row's lanes is made of lane moves within the
// adds, and the root is the instruction's.  8192 tokens of 32 + 8 + 8 heads of 128 with norms take
// 38 us (5.4 TB/s; all times are of passes in a graph) and, with nothing in a cache, 53; with
// kinds mixed in a wave, exchanges through the LDS crossbar and the exact root and quotient it was
// 50 and 68.  128 threads take 42 and 52 and leave half of a workgroup idle where a layer has few
// heads; 256 take 45; a token's workgroups in a row 43; loads of weights and angles ahead of the
// row's sum 42.  One token takes 2.9 us, which is a launch.
#include <cmath>

#include "origami_element.h"
#include "origami_internal.h"

namespace {

using namespace origami_element;
using origami_internal::aligned16;
using origami_internal::cache_geometry;
using origami_internal::cache_scale;
using origami_internal::check_launch;
using origami_internal::fail;

constexpr int kThreads = 64;

// Rows of one of the inputs, or of the rotated queries: element (token, head, channel) is at
// token * token_stride + head * head_stride + channel.
struct Rows {
  void* data;
  int64_t token, head;  // strides, in elements
  bool vec;             // every row starts on 16 bytes
};

struct AppendParams {
  Rows query, key, value, out;
  const void* norm[2];  // weights of the queries' and the keys' norm, or null
  bool norm_wide, norm_vec;  // weights are float32; they start on 16 bytes
  float eps;
  const float* cos_sin;  // [table_rows, rot]: the cosines of a position's pairs, then the sines
  int64_t table_rows;
  int32_t rot;
  bool interleaved;  // pairs are (2i, 2i + 1); else (i, i + rot / 2)
  bool table_vec;    // a lane's pairs are whole vectors of the table and of its neighbours
  const int64_t *positions, *slots;
  uint8_t* cache;
  int64_t blk_stride, half_stride, num_slots;  // rows of H * D, as cache_geometry
  Divisor block_size;
  float scale[2];  // an fp8 cache holds key / scale[0] and value / scale[1]
  int32_t Hq, H, D;
  float inverse_D;
  int32_t query_groups, groups;  // workgroups of a token's queries, and of its keys or values
};

// The sum of v over L neighbouring lanes, the same bits in each of them.
template <int L>
__device__ __forceinline__ float sum_lanes(float v) {
  v = fold_lanes<L == 8 ? 8 : 16>(v, [](float a, float b) { return a + b; });
  if constexpr (L == 32) v += __shfl_xor(v, 16);
  return v;
}

// 1 / sqrt(v) of v >= 0, to 1 ulp; small v is scaled, since the instruction takes no subnormals.
__device__ __forceinline__ float inverse_root(float v) {
  const bool small = v < 0x1p-96f;
  return __builtin_amdgcn_rsqf(small ? v * 0x1p64f : v) * (small ? 0x1p32f : 1.0f);
}

template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p, bool vec) {
  if (vec) return *reinterpret_cast<const Vec8<T>*>(p);
  Vec8<T> v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = p[j];
  return v;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, Vec8<T> v, bool vec) {
  if (vec) {
    *reinterpret_cast<Vec8<T>*>(p) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) p[j] = v[j];
}

__device__ __forceinline__ float weight_at(const AppendParams& p, const void* w, int e, bf16) {
  return p.norm_wide ? static_cast<const float*>(w)[e]
                     : static_cast<float>(static_cast<const bf16*>(w)[e]);
}
__device__ __forceinline__ float weight_at(const AppendParams& p, const void* w, int e, f16) {
  return p.norm_wide ? static_cast<const float*>(w)[e]
                     : static_cast<float>(static_cast<const f16*>(w)[e]);
}

// The normalised and rotated channels 8 c .. 8 c + 7 of a row of query or key; `x` holds
// them as loaded, zero past D.  All L lanes of the row call it.
template <typename T, int L>
__device__ __forceinline__ void norm_rotate(const AppendParams& p, const T* row, const void* w,
                                            const float* table, int c, float (&x)[8]) {
  float r = 1.0f;
  if (w) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
    r = inverse_root(sum_lanes<L>(sum) * p.inverse_D + p.eps);
    if (8 * c < p.D) {
      if (p.norm_vec && !p.norm_wide) {
        const Vec8<T> wv = *reinterpret_cast<const Vec8<T>*>(static_cast<const T*>(w) + 8 * c);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x[j] * r * static_cast<float>(wv[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x[j] * r * weight_at(p, w, 8 * c + j, T());
      }
    }
  }
  if (!table) return;
  const int half = p.rot / 2;
  if (p.table_vec) {
    if (p.interleaved) {
      if (8 * c < p.rot) {
        const Float4 cs = *reinterpret_cast<const Float4*>(table + 4 * c);
        const Float4 sn = *reinterpret_cast<const Float4*>(table + half + 4 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = x[2 * j], b = x[2 * j + 1];
          x[2 * j] = a * cs[j] - b * sn[j];
          x[2 * j + 1] = b * cs[j] + a * sn[j];
        }
      }
    } else {
      const int hc = half / 8;
      const bool first = c < hc, turned = c < 2 * hc;
      const int lane = static_cast<int>(threadIdx.x & 63);
      const int from = turned ? (first ? lane + hc : lane - hc) : lane;
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = __shfl(x[j], from);
      if (turned) {
        const float* t = table + 8 * (first ? c : c - hc);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const Float4 cs = *reinterpret_cast<const Float4*>(t + 4 * q);
          const Float4 sn = *reinterpret_cast<const Float4*>(t + half + 4 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float o = y[4 * q + j] * sn[j];
            x[4 * q + j] = x[4 * q + j] * cs[j] + (first ? -o : o);
          }
        }
      }
    }
    return;
  }
  // pairs that no vector holds: a channel's partner is read again from the row
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = 8 * c + j;
    y[j] = x[j];
    if (e < p.rot) {
      const int pair = p.interleaved ? e / 2 : e % half;
      const bool first = p.interleaved ? e % 2 == 0 : e < half;
      const int other = p.interleaved ? (e ^ 1) : (first ? e + half : e - half);
      float o = static_cast<float>(row[other]);
      if (w) o = o * r * weight_at(p, w, other, T());
      o *= table[half + pair];
      y[j] = x[j] * table[pair] + (first ? -o : o);
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = y[j];
}

// One workgroup: kThreads / L rows of one kind (blockIdx.y) of one token (blockIdx.x), whose
// strides, slot, position and angles are the same for all of them.
template <typename T, bool FP8, int L>
__global__ __launch_bounds__(kThreads) void append_kv_kernel(AppendParams p) {
  constexpr int kRows = kThreads / L;
  const int64_t token = blockIdx.x;
  const int c = static_cast<int>(threadIdx.x % L), row = static_cast<int>(threadIdx.x / L);
  int group = blockIdx.y;
  int kind = 0;  // of the queries, keys or values
  if (group >= p.query_groups) {
    group -= p.query_groups;
    kind = group < p.groups ? 1 : 2;
    group -= kind == 1 ? 0 : p.groups;
  }
  const int h0 = group * kRows;
  if (h0 + row >= (kind == 0 ? p.Hq : p.H)) return;
  const bool live = 8 * c < p.D;

  const Rows& in = kind == 0 ? p.query : (kind == 1 ? p.key : p.value);
  const T* const src =
      static_cast<const T*>(in.data) + token * in.token + h0 * in.head + row * in.head;
  Vec8<T> raw = {};
  if (live) raw = load8(src + 8 * c, in.vec);

  const float* table = nullptr;
  bool placed = true;
  if (p.cos_sin) {
    const int64_t pos = p.positions[token];
    placed = pos >= 0 && pos < p.table_rows;
    table = p.cos_sin + (placed ? pos : 0) * p.rot;
  }
  const void* const w = kind == 2 ? nullptr : p.norm[kind];
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = static_cast<float>(raw[j]);
  if (kind != 2) {
    if (w || table) {
      norm_rotate<T, L>(p, src, w, table, c, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[j] = static_cast<T>(placed ? x[j] : 0.0f);
    }
  }
  if (!live) return;
  if (kind == 0) {
    store8(static_cast<T*>(p.out.data) + token * p.out.token + h0 * p.out.head +
               row * p.out.head + 8 * c,
           raw, p.out.vec);
    return;
  }
  const int64_t slot = p.slots[token];
  if (!placed || slot < 0 || slot >= p.num_slots) return;
  const int at_slot = static_cast<int>(slot);  // num_slots fits 31 bits
  const int block = divide(at_slot, p.block_size);
  const int64_t at = block * p.blk_stride + (at_slot - block * p.block_size.d) +
                     (kind == 1 ? 0 : p.half_stride);
  const int64_t e = (at * p.H + h0) * p.D + (row * p.D + 8 * c);
  if constexpr (FP8) {
    const float scale = p.scale[kind - 1];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fp8_clamp(x[j] / scale);
    U32x2 o;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * q], x[4 * q + 1], 0, false);
      v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * q + 2], x[4 * q + 3], v, true);
      o[q] = static_cast<uint32_t>(v);
    }
    *reinterpret_cast<U32x2*>(p.cache + e) = o;
  } else {
    *reinterpret_cast<Vec8<T>*>(p.cache + 2 * e) = raw;
  }
}

template <typename T, bool FP8, int L>
int launch_rows(AppendParams p, uint32_t tokens, hipStream_t stream) {
  constexpr int kRows = kThreads / L;
  p.query_groups = (p.Hq + kRows - 1) / kRows;
  p.groups = (p.H + kRows - 1) / kRows;
  const dim3 grid(tokens, p.query_groups + 2 * p.groups), block(kThreads);
  hipLaunchKernelGGL((append_kv_kernel<T, FP8, L>), grid, block, 0, stream, p);
  return check_launch("append_kv_kernel");
}

template <typename T, bool FP8>
int launch_append(const AppendParams& p, uint32_t tokens, hipStream_t stream) {
  return p.D <= 64    ? launch_rows<T, FP8, 8>(p, tokens, stream)
         : p.D <= 128 ? launch_rows<T, FP8, 16>(p, tokens, stream)
                      : launch_rows<T, FP8, 32>(p, tokens, stream);
}

Rows rows_of(const void* data, const int64_t* strides) {
  return Rows{const_cast<void*>(data), strides[0], strides[1],
              aligned16(data) && strides[0] % 8 == 0 && strides[1] % 8 == 0};
}

}  // namespace

extern "C" int origami_append_kv_cache(
    const void* key, const void* value, const void* query, void* query_out, int64_t dtype,
    const int64_t* strides, int64_t tokens, int64_t query_heads, void* kv_cache,
    int64_t cache_dtype, int64_t cache_layout, int64_t num_blocks, int64_t block_size,
    int64_t heads, int64_t head_dim, const int64_t* slots, const int64_t* positions,
    const float* cos_sin, int64_t table_rows, int64_t rotary_dim, int64_t interleaved,
    const void* query_norm, const void* key_norm, int64_t norm_dtype, double eps, double k_scale,
    double v_scale, origami_stream_t stream_) {
  AppendParams p{};
  ORIGAMI_REQUIRE(dtype == ORIGAMI_DTYPE_FLOAT16 || dtype == ORIGAMI_DTYPE_BFLOAT16,
                  "keys and values must be float16 or bfloat16");
  ORIGAMI_REQUIRE(cache_dtype == dtype || cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN,
                  "kv_cache must have the keys' dtype or be float8_e4m3fn");
  ORIGAMI_REQUIRE(tokens >= 0 && query_heads >= 0 && heads > 0,
                  "tokens and heads must not be negative");
  ORIGAMI_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 256,
                  "head_dim must be a multiple of 8, at most 256");
  ORIGAMI_REQUIRE(num_blocks >= 0 && block_size > 0, "cache block size must be positive");
  if (int rc = cache_geometry(cache_layout, num_blocks, block_size, &p.blk_stride,
                              &p.half_stride))
    return rc;
  ORIGAMI_REQUIRE(block_size <= INT32_MAX / (num_blocks > 0 ? num_blocks : 1),
                  "the cache has too many token slots");
  ORIGAMI_REQUIRE(query_heads == 0 || tokens == 0 || (query != nullptr && query_out != nullptr),
                  "rotated queries need an output");
  ORIGAMI_REQUIRE(cos_sin == nullptr || (rotary_dim > 0 && rotary_dim % 2 == 0 &&
                                         rotary_dim <= head_dim && table_rows > 0 &&
                                         (positions != nullptr || tokens == 0)),
                  "rotation needs positions and an even rotary size of at most head_dim");
  ORIGAMI_REQUIRE((query_norm == nullptr && key_norm == nullptr) || norm_dtype == dtype ||
                      norm_dtype == ORIGAMI_DTYPE_FLOAT32,
                  "norm weights must have the keys' dtype or be float32");
  ORIGAMI_REQUIRE(eps >= 0.0 && std::isfinite(static_cast<float>(eps)),
                  "eps must not be negative or infinite");
  ORIGAMI_REQUIRE(cache_scale(k_scale) && cache_scale(v_scale),
                  "cache scales must be positive and finite in binary32");
  ORIGAMI_REQUIRE(cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN || (k_scale == 1.0 && v_scale == 1.0),
                  "cache scales are for float8_e4m3fn caches");
  ORIGAMI_REQUIRE(aligned16(kv_cache), "kv_cache must be 16-byte aligned");
  // a launch has at most 2^32 threads in x, and 65535 workgroups in y
  ORIGAMI_REQUIRE(heads <= 65535 && query_heads <= 65535 - 2 * heads &&
                      tokens < (int64_t(1) << 25),
                  "too many rows for one call");
  for (int i = 0; i < (query_heads > 0 ? 8 : 4); ++i)
    ORIGAMI_REQUIRE(strides[i] >= 0, "row strides must not be negative");
  if (tokens == 0) return ORIGAMI_OK;
  ORIGAMI_REQUIRE(key != nullptr && value != nullptr && slots != nullptr &&
                      (kv_cache != nullptr || num_blocks == 0),
                  "keys, values, slots and the cache must not be null");

  p.key = rows_of(key, strides);
  p.value = rows_of(value, strides + 2);
  p.query = rows_of(query, strides + 4);
  p.out = rows_of(query_out, strides + 6);
  p.norm[0] = query_norm;
  p.norm[1] = key_norm;
  p.norm_wide = norm_dtype == ORIGAMI_DTYPE_FLOAT32;
  p.norm_vec = aligned16(query_norm) && aligned16(key_norm);
  p.eps = static_cast<float>(eps);
  p.cos_sin = cos_sin;
  p.table_rows = table_rows;
  p.rot = static_cast<int32_t>(rotary_dim);
  p.interleaved = interleaved != 0;
  p.table_vec = aligned16(cos_sin) && rotary_dim % (interleaved ? 8 : 16) == 0;
  p.positions = positions;
  p.slots = slots;
  p.cache = static_cast<uint8_t*>(kv_cache);
  p.num_slots = num_blocks * block_size;
  p.block_size = divisor(block_size);
  p.scale[0] = static_cast<float>(k_scale);
  p.scale[1] = static_cast<float>(v_scale);
  p.Hq = static_cast<int32_t>(query_heads);
  p.H = static_cast<int32_t>(heads);
  p.D = static_cast<int32_t>(head_dim);
  p.inverse_D = 1.0f / static_cast<float>(head_dim);
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const uint32_t n = static_cast<uint32_t>(tokens);
  const bool fp8 = cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN;
  if (dtype == ORIGAMI_DTYPE_BFLOAT16)
    return fp8 ? launch_append<bf16, true>(p, n, stream) : launch_append<bf16, false>(p, n, stream);
  return fp8 ? launch_append<f16, true>(p, n, stream) : launch_append<f16, false>(p, n, stream);
}
