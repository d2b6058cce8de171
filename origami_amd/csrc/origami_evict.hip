// origami_evict.hip -- eviction from the paged KV cache by accumulated attention weight.
//
// weigh_kernel (weigh_few_kernel where the rows are few) adds up, for each cached token t and cache
// head, the weights that the queries give it:
//   out_t = weights_t + sum_q exp(scale (q . k_t) - lse_q)
// with lse_q the logarithm of the sum of exponentials that the attention returned for the row, so
// that no maximum is needed.  select_kernel finds the tokens that a head keeps, the newest and
// those of the largest sums, and move_kernel copies their rows, in order, to blocks of their own.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "origami_element.h"
#include "origami_internal.h"

namespace {

using namespace origami_element;
using origami_internal::aligned16;
using origami_internal::cache_geometry;
using origami_internal::cache_scale;
using origami_internal::check_launch;
using origami_internal::fail;

constexpr float kLog2e = 1.4426950408889634f;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kWeighUnits = 2048, kMostWeighParts = 32, kWeighWaves = 2048;

// ---------------------------------------------------------------------------
// Adding up the weights
// ---------------------------------------------------------------------------

struct WeighParams {
  const void* query;
  int64_t q_token, q_head;  // strides, in elements
  bool q_vec;               // its rows start on 16 bytes
  const float* lse;         // [tokens, query heads]
  const uint8_t* cache;     // the keys
  int64_t blk_stride;       // rows of H * D, as cache_geometry
  int64_t num_blocks;
  const int64_t *tables, *lengths, *starts;
  int64_t table_stride;
  Divisor block_size, requests, H, G;
  Divisor tiles;  // ranges of a request's tokens, where the rows are few
  int32_t rest;   // places past max_tokens that a range copies
  Divisor parts;  // of the rows that see a tile, each of which a workgroup adds up
  int32_t tokens, Hq, D, max_tokens, places;
  float scale;  // includes the keys' scale
  const float* weights;  // null: zeros
  float* out;
  int64_t w_request, w_head, o_request, o_head;  // strides, in elements
  float* part_sums;  // [parts][requests][H][max_tokens], where there are several
};


template <int MR>
using Tile = float __attribute__((ext_vector_type(MR * MR / 64)));

// c + a b, where a lane has 8 values of row (a) and column (b) lane % MR, from 8 (lane / MR) on;
// value x of the result is in column lane % MR and row 4 (lane / MR) + x % 4 + (256 / MR) (x / 4).
template <typename T, int MR>
__device__ __forceinline__ Tile<MR> mfma(Vec8<T> a, Vec8<T> b, Tile<MR> c) {
  if constexpr (MR == 16) {
    if constexpr (std::is_same<T, bf16>::value)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  } else {
    if constexpr (std::is_same<T, bf16>::value)
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
}

// Where piece `piece` (16 bytes) of row `row` is in LDS: 16 lanes read the same piece of 16 rows.
template <int DP>
__device__ __forceinline__ int query_piece(int row, int piece) {
  return row * (DP / 8) + (piece ^ (DP == 64 ? (row >> 1) & 7 : row & 15));
}

// Dwords of a cache row, which starts on four bytes where it holds 4-bit values.
template <int DWORDS>
struct __attribute__((aligned(4))) Dwords {
  uint32_t w[DWORDS];
};

// One workgroup: 32 tokens of one KV head of one request for each of eight waves, against the query
// rows that see any of them or a part of those rows, in stages of 64.  The keys stay in registers,
// as the second operand, so that a token's scores are in the lanes of one column and are added up
// where they are; the queries go through LDS, a stage ahead.
//
// The exponentials and masks beside the products bound it: two prompts of up to 4096 tokens, 28
// query heads of 128 channels over 4 heads in 4 bits, take 139 to 154 us on different boxes (723 to
// 653 TFLOP/s, matrix units busy in 37% of the CUs' busy cycles); without parts of the rows and
// stages of 64 they took 926.
//
// The order of the channels in the products is free as long as keys and queries have the same: a
// lane's 16 bytes of a key are 8, 16 or 32 channels in a row, whole loads of the cache's row.
template <typename T, Cell CELL, int DP>
__global__ __launch_bounds__(512, DP <= 128 ? 2 : 1) void weigh_kernel(WeighParams p) {
  constexpr int MR = 32, NT = 1, NW = 8, kThreads = 64 * NW, SUB = 2, ROWS = SUB * MR;
  constexpr int NG = 64 / MR, KS = DP / (8 * NG), NCH = DP / 8, ACC = MR * MR / 64;
  constexpr int kWhole = CELL == kFp4 ? 4 : (CELL == kFp8 ? 2 : 1);
  constexpr int NPE = kWhole < KS ? kWhole : KS;  // pieces of 8 channels in a load
  constexpr int kPiece = CELL == kFp4 ? 4 : (CELL == kFp8 ? 8 : 16);
  constexpr int kTokens = NW * NT * MR;
  constexpr int QL = (ROWS * NCH + kThreads - 1) / kThreads;
  __shared__ U32x4 queries[2][ROWS * NCH];
  __shared__ alignas(16) float lses[2][ROWS];
  __shared__ alignas(16) int limits[2][ROWS];
  __shared__ int least[2][SUB];  // the smallest limit of a tile's rows
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane % MR, q4 = lane / MR;

  // the first tokens, which most rows see, first; the same part of the rows on the same chiplet
  int u = divide(static_cast<int>(blockIdx.x), p.parts);
  const int part = static_cast<int>(blockIdx.x) - u * p.parts.d;
  const int v = divide(u, p.H), h = u - v * p.H.d;
  const int tile = divide(v, p.requests), r = v - tile * p.requests.d;
  const int t0 = tile * kTokens;
  if (t0 >= p.places) return;

  // The blocks and the sums so far are asked for before the length is known: up to the bounds that
  // the host has they can be read.
  const int first_t = t0 + wave * NT * MR;  // of this wave
  const int64_t* const table = p.tables + r * p.table_stride;
  int64_t ids[NT] = {};
#pragma unroll
  for (int n = 0; n < NT; ++n)
    if (p.max_tokens > 0)
      ids[n] = table[divide(min(first_t + n * MR + c, p.max_tokens - 1), p.block_size)];
  const int length =
      static_cast<int>(min(max(p.lengths[r], int64_t(0)), int64_t(3) << 29));
  const int end = min(length, p.max_tokens);
  const float* const weights =
      p.weights ? p.weights + r * p.w_request + h * p.w_head : nullptr;
  float* const out = p.out + r * p.o_request + h * p.o_head;
  float* const sums =
      p.part_sums + ((static_cast<int64_t>(part) * p.requests.d + r) * p.H.d + h) * p.max_tokens;
  if (t0 >= end) {
    // of several parts the join takes care of these
    if (p.parts.d > 1) return;
    for (int i = threadIdx.x; i < kTokens; i += kThreads)
      if (t0 + i < p.places && out != weights)
        out[t0 + i] = weights ? weights[t0 + i] : 0.0f;
    return;
  }

  int q_first = r, q_count = 1;
  if (p.starts) {
    const int64_t n = p.tokens;
    const int64_t a = min(max(p.starts[r], int64_t(0)), n);
    q_first = static_cast<int>(a);
    q_count = static_cast<int>(min(max(p.starts[r + 1], a), n) - a);
  }
  const int before = length - q_count;  // tokens before the queries' (may be negative)

  // the keys
  const int bytes = row_bytes_of(CELL, p.D);
  Vec8<T> kf[NT][KS];
  bool there[NT];
  float old[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int t = first_t + n * MR + c;
    const int block = divide(t, p.block_size);
    const int64_t id = ids[n];
    there[n] = t < end && id >= 0 && id < p.num_blocks;
    old[n] = weights && p.parts.d == 1 && t < p.places ? weights[t] : 0.0f;
    const int64_t at = there[n] ? id * p.blk_stride + (t - block * p.block_size.d) : 0;
    const uint8_t* const row = p.cache + (at * p.H.d + h) * bytes;
#pragma unroll
    for (int j = 0; j < KS / NPE; ++j) {
      const int ch = (j * NG + q4) * NPE * 8;  // of the load's first piece
      Dwords<NPE * kPiece / 4> raw = {};
      const uint8_t* const src = row + ch / 8 * kPiece;
      float scale = 0.0f;
      if (there[n] && ch < p.D) {
        if (ch + NPE * 8 <= p.D) {
          raw = *reinterpret_cast<const Dwords<NPE * kPiece / 4>*>(src);
        } else {
#pragma unroll
          for (int i = 0; i < NPE; ++i)
            if (ch + 8 * i < p.D)
#pragma unroll
              for (int x = 0; x < kPiece / 4; ++x)
                raw.w[i * kPiece / 4 + x] =
                    *reinterpret_cast<const uint32_t*>(src + i * kPiece + 4 * x);
        }
        if constexpr (CELL == kFp4) scale = fp4_scale(row[p.D / 2 + ch / 32]);
      }
#pragma unroll
      for (int i = 0; i < NPE; ++i) {
        U32x4 wide;
        if constexpr (CELL == kFp4)
          wide = fp4_expand<T>(raw.w[i], scale);
        else if constexpr (CELL == kFp8)
          wide = fp8_expand<T>(U32x2{raw.w[2 * i], raw.w[2 * i + 1]});
        else
          wide = U32x4{raw.w[0], raw.w[1], raw.w[2], raw.w[3]};
        kf[n][j * NPE + i] = __builtin_bit_cast(Vec8<T>, wide);
      }
    }
  }

  // Query i / G sees the tokens up to before + i / G: rows from the first that sees one of these.
  const int all_rows = q_count * p.G.d;
  int row0 = min(max(t0 - before, 0), q_count) * p.G.d / MR * MR, rows = all_rows;
  if (p.parts.d > 1) {
    const int stages = (rows - row0 + ROWS - 1) / ROWS;
    const int each = divide(stages + p.parts.d - 1, p.parts) * ROWS;
    row0 = min(row0 + part * each, rows);
    rows = min(row0 + each, rows);
  }
  U32x4 qr[QL];
  float lse = 0.0f;
  int limit = 0;
  const auto load_rows = [&](int from) {
#pragma unroll
    for (int l = 0; l < QL; ++l) {
      const int i = l * kThreads + threadIdx.x, row = from + i / NCH, d = i % NCH * 8;
      qr[l] = U32x4{0, 0, 0, 0};
      if (i < ROWS * NCH && row < rows && d < p.D) {
        const int qi = divide(row, p.G), head = h * p.G.d + row - qi * p.G.d;
        const T* const src =
            static_cast<const T*>(p.query) + (q_first + qi) * p.q_token + head * p.q_head + d;
        if (p.q_vec) {
          qr[l] = *reinterpret_cast<const U32x4*>(src);
        } else {
          Vec8<T> v;
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = src[j];
          qr[l] = __builtin_bit_cast(U32x4, v);
        }
      }
    }
    if (threadIdx.x < ROWS) {
      const int row = from + threadIdx.x;
      limit = 0;
      lse = 0.0f;
      if (row < rows) {
        const int qi = divide(row, p.G), head = h * p.G.d + row - qi * p.G.d;
        lse = p.lse[static_cast<int64_t>(q_first + qi) * p.Hq + head];
        // a row that saw nothing gives no weight
        limit = lse == -INFINITY ? 0 : max(before + qi + 1, 0);
      }
    }
  };
  const auto store_rows = [&](int buf) {
#pragma unroll
    for (int l = 0; l < QL; ++l) {
      const int i = l * kThreads + threadIdx.x;
      if (i < ROWS * NCH) queries[buf][query_piece<DP>(i / NCH, i % NCH)] = qr[l];
    }
    if (wave == 0) {  // ROWS <= 64
      int low = lane < ROWS ? limit : INT32_MAX;
#pragma unroll
      for (int x = 1; x < MR; x <<= 1) low = min(low, __shfl_xor(low, x));
      if (lane < ROWS) {
        lses[buf][lane] = lse;
        limits[buf][lane] = limit;
        if (c == 0) least[buf][lane / MR] = low;
      }
    }
  };

  // sums of binary32 with what they lose
  float sum[NT], lost[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) sum[n] = lost[n] = 0.0f;
  int buf = 0;
  if (row0 < rows) {
    load_rows(row0);
    store_rows(0);
  }
  for (int from = row0; from < rows; from += ROWS) {
    __syncthreads();
    const bool more = from + ROWS < rows;
    if (more) load_rows(from + ROWS);
#pragma unroll
    for (int m = 0; m < SUB; ++m) {
      // rows of the result that this lane has, four at a time
      const auto mine = [&](int x) { return MR * m + 4 * q4 + 256 / MR * (x / 4); };
      Tile<MR> s[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < ACC; ++x) s[n][x] = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int piece = (k / NPE * NG + q4) * NPE + k % NPE;
        const Vec8<T> qf =
            __builtin_bit_cast(Vec8<T>, queries[buf][query_piece<DP>(MR * m + c, piece)]);
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n] = mfma<T, MR>(qf, kf[n][k], s[n]);
      }
      const bool whole =
          __builtin_amdgcn_readfirstlane(least[buf][m]) >= first_t + NT * MR;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int t = first_t + n * MR + c;
        float e[ACC];
#pragma unroll
        for (int x = 0; x < ACC; x += 4) {
          const Float4 below = *reinterpret_cast<const Float4*>(&lses[buf][mine(x)]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            e[x + j] = __builtin_amdgcn_exp2f(kLog2e * fmaf(s[n][x + j], p.scale, -below[j]));
        }
        if (!whole) {
#pragma unroll
          for (int x = 0; x < ACC; ++x)
            e[x] = t < limits[buf][mine(x) + x % 4] ? e[x] : 0.0f;
        }
#pragma unroll
        for (int step = 1; step < ACC; step *= 2)
#pragma unroll
          for (int x = 0; x < ACC; x += 2 * step) e[x] += e[x + step];
        const float add = e[0] - lost[n], next = sum[n] + add;
        lost[n] = next < INFINITY ? (next - sum[n]) - add : 0.0f;
        sum[n] = next;
      }
    }
    buf ^= 1;
    if (more) store_rows(buf);
  }

#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float v = sum[n];
#pragma unroll
    for (int x = MR; x < 64; x <<= 1) v += __shfl_xor(v, x);
    const int t = first_t + n * MR + c;
    if (q4 != 0 || t >= p.places) continue;
    if (p.parts.d > 1) {
      if (t < p.max_tokens) sums[t] = there[n] ? v : 0.0f;
      continue;
    }
    if (there[n])
      out[t] = old[n] + v;
    else if (out != weights)
      out[t] = old[n];
  }
}

// Adds the parts of each place, in their order, with what the sums lose.
__global__ __launch_bounds__(256) void weigh_join_kernel(WeighParams p) {
  const int row = static_cast<int>(blockIdx.y), r = divide(row, p.H), h = row - r * p.H.d;
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= p.places) return;
  const float* const weights = p.weights ? p.weights + r * p.w_request + h * p.w_head : nullptr;
  float* const out = p.out + r * p.o_request + h * p.o_head;
  const int end = static_cast<int>(
      min(max(p.lengths[r], int64_t(0)), static_cast<int64_t>(p.max_tokens)));
  if (t >= end) {  // where there may be no parts
    if (out != weights) out[t] = weights ? weights[t] : 0.0f;
    return;
  }
  const int64_t all = static_cast<int64_t>(p.requests.d) * p.H.d * p.max_tokens;
  const float* const src = p.part_sums + static_cast<int64_t>(row) * p.max_tokens + t;
  float sum = 0.0f, lost = 0.0f;
#pragma unroll 4
  for (int i = 0; i < p.parts.d; ++i) {
    const float add = src[i * all] - lost, next = sum + add;
    lost = next < INFINITY ? (next - sum) - add : 0.0f;
    sum = next;
  }
  out[t] = (weights ? weights[t] : 0.0f) + sum;
}

// Parts of the rows: as many as give every CU a few workgroups, of four stages at least.
int64_t most_weigh_parts(int64_t tokens, int64_t query_heads, int64_t heads, int64_t requests) {
  const int64_t rows = tokens * (query_heads / heads);
  if (requests == 0 || rows <= 16 * requests) return 1;
  return std::max<int64_t>(std::min(rows / requests / 256, kMostWeighParts), 1);
}
int64_t weigh_parts(int64_t tokens, int64_t query_heads, int64_t heads, int64_t requests,
                    int64_t max_tokens) {
  const int64_t most = most_weigh_parts(tokens, query_heads, heads, requests);
  if (most == 1 || max_tokens == 0) return 1;
  return std::min(ceil_div(kWeighUnits, requests * heads * ceil_div(max_tokens, 256)), most);
}

// Zeros, for what a lane reads of rows that are not in the cache and of channels past the last.
__device__ const U32x4 kZeroRow[33] = {};

// One wave: a range of the tokens of one KV head of one request against its query rows, few as in a
// decode step.  Memory bounds it.  The queries stay in registers;
// the keys come 64 tokens at a step (32 past 128 channels) and a step ahead, and their blocks two
// steps, so that a wave waits for memory as seldom as can be: 16 requests of 2048 to 8192 tokens
// and 8 heads of 128 take 47 us among other work (39 alone, 4.3 TB/s), in e4m3 24 and in 4 bits 20;
// with workgroups that ended after 256 tokens 52 and in 4 bits 33.  Waves next to each other are
// heads of the same tokens, and ranges of a request follow each other over the chiplets, as in the
// attention.
//
// Drafts of 17 to 32 rows beside shorter ones have two products a key (16 requests of 3 and 5
// queries with 4 query heads a cache head: 48 us, in 4 bits 25).  Past that the queries are loaded
// anew for each step of keys, 16 rows at a time, which is slow (1 us each), but their request alone
// is: one of 900 queries among 300 of one takes 3.4 ms.  To go over the keys anew for each 16 rows
// took 81, 37 us and 10.1 ms, and a rounding each.
template <typename T, Cell CELL, int DP, bool WHOLE>
__global__ __launch_bounds__(256, 2) void weigh_few_kernel(WeighParams p, Divisor beside,
                                                           int chunk) {
  constexpr int MR = 16, NG = 4, NT = DP == 256 ? 2 : 4, KS = DP / (8 * NG), STEP = NT * MR;
  constexpr int kWhole = CELL == kFp4 ? 4 : (CELL == kFp8 ? 2 : 1);
  constexpr int NPE = kWhole < KS ? kWhole : KS;  // pieces of 8 channels in a load
  constexpr int kPiece = CELL == kFp4 ? 4 : (CELL == kFp8 ? 8 : 16);
  constexpr int LJ = KS / NPE, DW = NPE * kPiece / 4;  // loads of a key, and their dwords
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane % MR, q4 = lane / MR;
  const int eight = static_cast<int>(blockIdx.x >> 3), some = divide(eight, beside);
  const int unit = ((some * 8 + static_cast<int>(blockIdx.x & 7)) * beside.d + eight -
                    some * beside.d) * 4 + wave;
  const int u = divide(unit, p.H), h = unit - u * p.H.d;
  const int r = divide(u, p.tiles);
  if (r >= p.requests.d) return;
  const int turned = u - r * p.tiles.d + r;
  const int t0 = (turned - divide(turned, p.tiles) * p.tiles.d) * chunk;

  const int64_t* const table = p.tables + r * p.table_stride;
  const int tl = lane % STEP;
  const auto block_of = [&](int t) -> int64_t {  // up to max_tokens the tables can be read
    return t < p.max_tokens ? table[divide(t, p.block_size)] : -1;
  };
  const int64_t id = block_of(t0 + tl);
  int64_t ahead = block_of(t0 + STEP + tl);
  const int length =
      static_cast<int>(min(max(p.lengths[r], int64_t(0)), int64_t(3) << 29));
  const int end = min(length, p.max_tokens);
  const float* const weights =
      p.weights ? p.weights + r * p.w_request + h * p.w_head : nullptr;
  float* const out = p.out + r * p.o_request + h * p.o_head;
  // places past the tokens are copied, if they are elsewhere: those up to the bound with the
  // range's, those past it with all ranges alike
  if (out != weights && p.rest > 0) {
    constexpr int kEach = 8;
    const int64_t rest0 = p.max_tokens + static_cast<int64_t>(t0 / chunk) * p.rest;
    const int rest1 = static_cast<int>(min(rest0 + p.rest, static_cast<int64_t>(p.places)));
    for (int64_t t = rest0 + lane; t < rest1; t += 64 * kEach) {
      float w[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        w[i] = weights && t + 64 * i < rest1 ? weights[t + 64 * i] : 0.0f;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (t + 64 * i < rest1) out[t + 64 * i] = w[i];
    }
  }
  const int t1 = min(t0 + chunk, out == weights ? end : p.max_tokens);
  if (t0 >= t1) return;
  int q_first = r, q_count = 1;
  if (p.starts) {
    const int64_t n = p.tokens;
    const int64_t a = min(max(p.starts[r], int64_t(0)), n);
    q_first = static_cast<int>(a);
    q_count = static_cast<int>(min(max(p.starts[r + 1], a), n) - a);
  }
  const int before = length - q_count, rows = q_count * p.G.d;

  const int bytes = row_bytes_of(CELL, p.D);
  const uint32_t pitch = static_cast<uint32_t>(p.H.d) * bytes;
  const uint8_t* const head_rows = p.cache + static_cast<int64_t>(h) * bytes;
  const uint8_t* const zeros = reinterpret_cast<const uint8_t*>(kZeroRow);
  const auto row_of = [&](int t, int64_t id) -> int {  // of the cache, -1 where t has none
    if (t >= end || id < 0 || id >= p.num_blocks) return -1;
    return static_cast<int>(id * p.blk_stride + t - divide(t, p.block_size) * p.block_size.d);
  };
  struct Step {
    Dwords<DW> raw[NT][LJ];
    uint32_t scale[NT][LJ];
    float old;   // the sum so far of token number `lane` of the step
    bool there;  // whether it is in the cache
  };
  const auto load_step = [&](Step& s, int mine, int t, const float* sums) {
    s.there = mine >= 0;
    s.old = sums && t + tl < t1 ? sums[t + tl] : 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int at = __shfl(mine, MR * n + c);
      const uint8_t* const row =
          head_rows + static_cast<uint64_t>(static_cast<uint32_t>(at)) * pitch;
#pragma unroll
      for (int j = 0; j < LJ; ++j) {
        const int ch = (j * NG + q4) * NPE * 8;
        const bool in = at >= 0 && ch < p.D;
        if constexpr (WHOLE) {
          s.raw[n][j] =
              *reinterpret_cast<const Dwords<DW>*>(in ? row + ch / 8 * kPiece : zeros);
        } else {
#pragma unroll
          for (int i = 0; i < NPE; ++i) {
            const auto piece = *reinterpret_cast<const Dwords<kPiece / 4>*>(
                in && ch + 8 * i < p.D ? row + (ch / 8 + i) * kPiece : zeros);
#pragma unroll
            for (int x = 0; x < kPiece / 4; ++x) s.raw[n][j].w[i * kPiece / 4 + x] = piece.w[x];
          }
        }
        if constexpr (CELL == kFp4) s.scale[n][j] = *(in ? row + p.D / 2 + ch / 32 : zeros);
      }
    }
  };

  // 16 query rows: of the product, and of what this lane has of its result (rows 4 q4 .. 4 q4 + 3).
  struct Rows16 {
    Vec8<T> q[KS];
    float below[4];
    int limit[4];
  };
  const auto load_rows = [&](Rows16& o, int from) {
    {
      const int row = from + c, qi = divide(row, p.G), head = h * p.G.d + row - qi * p.G.d;
      const T* const src =
          static_cast<const T*>(p.query) + (q_first + qi) * p.q_token + head * p.q_head;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d = ((k / NPE * NG + q4) * NPE + k % NPE) * 8;
        o.q[k] = Vec8<T>{};
        if (row < rows && d < p.D) {
          if (p.q_vec) {
            o.q[k] = *reinterpret_cast<const Vec8<T>*>(src + d);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) o.q[k][j] = src[d + j];
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int row = from + 4 * q4 + x, qi = divide(row, p.G);
      o.below[x] = 0.0f;
      o.limit[x] = 0;
      if (row < rows) {
        const float lse =
            p.lse[static_cast<int64_t>(q_first + qi) * p.Hq + h * p.G.d + row - qi * p.G.d];
        o.below[x] = lse;
        // a row that saw nothing gives no weight
        o.limit[x] = lse == -INFINITY ? 0 : before + qi + 1;
      }
    }
  };
  // What this lane's rows give the token of its column in tile n.
  const auto weights_of = [&](const Rows16& q, const Step& s, int n, int t) -> float {
    Tile<MR> score = {};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int j = k / NPE, i = k % NPE;
      U32x4 wide;
      if constexpr (CELL == kFp4)
        wide = fp4_expand<T>(s.raw[n][j].w[i], fp4_scale(s.scale[n][j]));
      else if constexpr (CELL == kFp8)
        wide = fp8_expand<T>(U32x2{s.raw[n][j].w[2 * i], s.raw[n][j].w[2 * i + 1]});
      else
        wide = U32x4{s.raw[n][j].w[0], s.raw[n][j].w[1], s.raw[n][j].w[2], s.raw[n][j].w[3]};
      score = mfma<T, MR>(q.q[k], __builtin_bit_cast(Vec8<T>, wide), score);
    }
    const int at = t + MR * n + c;
    float e[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      e[x] = __builtin_amdgcn_exp2f(kLog2e * fmaf(score[x], p.scale, -q.below[x]));
      e[x] = at < q.limit[x] ? e[x] : 0.0f;
    }
    return (e[0] + e[1]) + (e[2] + e[3]);
  };
  const auto finish = [&](const Step& s, float (&v)[NT], int t) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      v[n] += __shfl_xor(v[n], 16);
      v[n] += __shfl_xor(v[n], 32);
    }
    float mine = v[0];  // of token number `lane`, which is in tile lane / 16
#pragma unroll
    for (int n = 1; n < NT; ++n) mine = q4 % NT == n ? v[n] : mine;
    if (lane < STEP && t + tl < t1) {
      if (s.there)
        out[t + tl] = s.old + mine;
      else if (out != weights)
        out[t + tl] = s.old;
    }
  };

  // Over the steps, with the keys of the next on their way.
  const auto each_step = [&](auto compute) __attribute__((always_inline)) {
    Step even, other;
    load_step(even, row_of(t0 + tl, id), t0, weights);
    __builtin_amdgcn_sched_barrier(0);
    for (int t = t0; t < t1; t += 2 * STEP) {
      int mine = row_of(t + STEP + tl, ahead);
      ahead = block_of(t + 2 * STEP + tl);
      load_step(other, mine, t + STEP, weights);
      compute(even, t);
      if (t + STEP >= t1) break;
      mine = row_of(t + 2 * STEP + tl, ahead);
      ahead = block_of(t + 3 * STEP + tl);
      load_step(even, mine, t + 2 * STEP, weights);
      compute(other, t + STEP);
    }
  };

  constexpr int kHeld = DP <= 128 ? 2 : 1;  // of 16 rows each that there are registers for
  if (rows > kHeld * MR) {
    // One of the batch's longer requests: each step's keys against all rows that see any of them,
    // 16 at a time and the next ones ahead, in sums of binary32 with what they lose.
    const auto first_row = [&](int t) {
      return min(max(t - before, 0), q_count) * p.G.d / MR * MR;
    };
    Rows16 next;
    load_rows(next, first_row(t0));
    const auto compute = [&](const Step& s, int t) __attribute__((always_inline)) {
      float sum[NT] = {}, lost[NT] = {};
      for (int from = first_row(t); from < rows; from += MR) {
        const Rows16 q = next;
        load_rows(next, from + MR < rows ? from + MR : first_row(t + STEP));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float add = weights_of(q, s, n, t) - lost[n], total = sum[n] + add;
          lost[n] = total < INFINITY ? (total - sum[n]) - add : 0.0f;
          sum[n] = total;
        }
      }
      finish(s, sum, t);
    };
    if constexpr (CELL == kWide) {  // there are registers for the keys of one step
      int64_t block = id;
      for (int t = t0; t < t1; t += STEP) {
        Step s;
        load_step(s, row_of(t + tl, block), t, weights);
        block = block_of(t + STEP + tl);
        compute(s, t);
      }
    } else {
      each_step(compute);
    }
    return;
  }

  const auto held_rows = [&](auto count) __attribute__((always_inline)) {
    constexpr int N = decltype(count)::value;
    Rows16 q[N];
#pragma unroll
    for (int i = 0; i < N; ++i) load_rows(q[i], MR * i);
    const auto compute = [&](const Step& s, int t) __attribute__((always_inline)) {
      float v[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        v[n] = weights_of(q[0], s, n, t);
#pragma unroll
        for (int i = 1; i < N; ++i) v[n] += weights_of(q[i], s, n, t);
      }
      finish(s, v, t);
    };
    each_step(compute);
  };
  if (kHeld > 1 && rows > MR)
    held_rows(std::integral_constant<int, kHeld>{});
  else  // with no query row the sums stay what they are
    held_rows(std::integral_constant<int, 1>{});
}

// Whether there are places past max_tokens that are copied: not if they are where they go.
bool copies_rest(const WeighParams& p) {
  return p.places > p.max_tokens && (p.out != p.weights || p.w_request != p.o_request ||
                                     p.w_head != p.o_head);
}

template <typename T, Cell CELL, int DP>
int launch_weigh_few(WeighParams p, int64_t requests, hipStream_t stream) {
  // ranges of 64 tokens and more, for about 2048 waves; ranges without tokens where places past the
  // bound are copied, 512 and more of them each
  const int64_t most = std::max<int64_t>(ceil_div(p.max_tokens, 64), 1);
  const int64_t waves = std::max<int64_t>(kWeighWaves / (requests * p.H.d), 1);
  const int64_t wanted = std::min(waves, most);
  const int64_t chunk = std::max<int64_t>(ceil_div(ceil_div(p.max_tokens, wanted), 64), 1) * 64;
  const int64_t rest = copies_rest(p) ? p.places - p.max_tokens : 0;
  const int64_t tiles = std::max({ceil_div(p.max_tokens, chunk),
                                  std::min(waves, ceil_div(rest, 512)), int64_t(1)});
  p.tiles = divisor(tiles);
  p.rest = static_cast<int32_t>(ceil_div(rest, tiles));
  const int64_t units = requests * p.H.d * p.tiles.d;
  const Divisor beside = divisor(std::max(p.H.d / 4, 1));
  const int64_t workgroups = ceil_div(ceil_div(units, 4), 8 * beside.d) * 8 * beside.d;
  ORIGAMI_REQUIRE(workgroups < (int64_t(1) << 32) / 256, "too many tokens for one call");
  const dim3 grid(static_cast<unsigned>(workgroups)), block(256);
  constexpr int kLoad = CELL == kFp4 ? 32 : (CELL == kFp8 ? 16 : 8);
  constexpr int kChannels = kLoad < DP / 4 ? kLoad : DP / 4;  // of a load
  if (p.D % kChannels == 0)
    hipLaunchKernelGGL((weigh_few_kernel<T, CELL, DP, true>), grid, block, 0, stream, p, beside,
                       static_cast<int>(chunk));
  else if constexpr (kChannels > 8)
    hipLaunchKernelGGL((weigh_few_kernel<T, CELL, DP, false>), grid, block, 0, stream, p, beside,
                       static_cast<int>(chunk));
  return check_launch("weigh_few_kernel");
}

template <typename T, Cell CELL, int DP>
int launch_weigh(const WeighParams& p, int64_t requests, hipStream_t stream) {
  // rows of 16 where the requests have no more on average
  if (static_cast<int64_t>(p.tokens) * p.G.d <= 16 * requests)
    return launch_weigh_few<T, CELL, DP>(p, requests, stream);
  constexpr int64_t kMost = (int64_t(1) << 32) / 512;  // workgroups of a launch
  ORIGAMI_REQUIRE(requests * p.H.d * ceil_div(p.places, 256) < kMost,
                  "too many tokens for one call");
  const int64_t tiles = ceil_div(copies_rest(p) ? p.places : p.max_tokens, 256);
  if (tiles == 0) return ORIGAMI_OK;  // no tokens, and no places elsewhere
  // of several parts the join copies what is past the bound
  const int64_t units =
      requests * p.H.d * (p.parts.d > 1 ? ceil_div(p.max_tokens, 256) * p.parts.d : tiles);
  ORIGAMI_REQUIRE(units < kMost, "too many tokens for one call");
  const dim3 grid(static_cast<unsigned>(units)), block(512);
  hipLaunchKernelGGL((weigh_kernel<T, CELL, DP>), grid, block, 0, stream, p);
  if (int rc = check_launch("weigh_kernel")) return rc;
  if (p.parts.d == 1) return ORIGAMI_OK;
  const dim3 joins(static_cast<unsigned>(tiles), static_cast<unsigned>(requests * p.H.d));
  hipLaunchKernelGGL(weigh_join_kernel, joins, dim3(256), 0, stream, p);
  return check_launch("weigh_join_kernel");
}

template <typename T, Cell CELL>
int launch_weigh(const WeighParams& p, int64_t requests, hipStream_t stream) {
  return p.D <= 64    ? launch_weigh<T, CELL, 64>(p, requests, stream)
         : p.D <= 128 ? launch_weigh<T, CELL, 128>(p, requests, stream)
                      : launch_weigh<T, CELL, 256>(p, requests, stream);
}

template <typename T>
int launch_weigh(const WeighParams& p, Cell cell, int64_t requests, hipStream_t stream) {
  if (cell == kFp8) return launch_weigh<T, kFp8>(p, requests, stream);
  if (cell == kFp4) return launch_weigh<T, kFp4>(p, requests, stream);
  return launch_weigh<T, kWide>(p, requests, stream);
}

// ---------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------

struct EvictParams {
  uint8_t* cache;
  int64_t blk_stride, half_stride, num_blocks;  // rows of H * D, as cache_geometry
  const int64_t *tables, *out_tables, *lengths;
  int64_t table_stride, out_table_stride;
  Divisor block_size, H;
  int32_t max_tokens, keep, recent, out_places;
  const float* weights;
  float* out_weights;
  int64_t w_request, w_head, o_request, o_head;  // strides, in elements
  int64_t* kept;  // [requests, H, keep]
  int32_t row_bytes;
  Divisor pieces;     // of a row, in loads
  Divisor row_tiles;  // of a request's kept tokens
};

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64, kBins = 2048;

// What is kept of one request's head: all of the newest `recent`, and of the others those with the
// largest weights, of equal ones the first.
struct Share {
  int tokens, kept, older, need;  // `need` of the first `older` tokens
};

__device__ __forceinline__ Share share_of(const EvictParams& p, int r) {
  Share s;
  s.tokens =
      static_cast<int>(min(max(p.lengths[r], int64_t(0)), static_cast<int64_t>(p.max_tokens)));
  s.kept = min(s.tokens, p.keep);
  const int last = min(p.recent, s.kept);
  s.older = s.tokens - last;
  s.need = s.kept - last;
  return s;
}

// Weights as whole numbers in the same order; both zeros are one, NaN is the largest.
__device__ __forceinline__ uint32_t rank_of(float w) {
  const uint32_t b = __builtin_bit_cast(uint32_t, w);
  if (w != w) return 0xffffffffu;
  if (w == 0.0f) return 0x80000000u;
  return b >> 31 ? ~b : b | 0x80000000u;
}

// The sum of x over a wave's first 16 lanes, of which the others have the same.
__device__ __forceinline__ uint32_t sum16(uint32_t x) {
  x += lane_moved<0xb1>(x);
  x += lane_moved<0x4e>(x);
  x += lane_moved<0x141>(x);
  x += lane_moved<0x140>(x);
  return __builtin_amdgcn_readfirstlane(x);
}

// x summed over this lane and those before it.
__device__ __forceinline__ uint32_t sum_upto(uint32_t x, int lane) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const uint32_t other = __shfl_up(x, i);
    x += lane >= i ? other : 0;
  }
  return x;
}

// How many of the bits are of lanes before this one.
__device__ __forceinline__ uint32_t before_lane(uint64_t bits) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(bits >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(bits), 0));
}

__device__ __forceinline__ float weight_of(uint32_t rank) {
  return __builtin_bit_cast(float, rank >> 31 ? rank ^ 0x80000000u : ~rank);
}

// One workgroup: the tokens that one head of one request keeps.  The rank of the last of them is
// found by its digits, from the highest, from counts of the ranks that have the digits before it
// (four counts of each digit, for lanes in turn, since weights have few exponents); then the tokens
// are listed in their order, KEYS times 1024 of them at a time.
//
// The workgroup has a CU to itself, and instructions bound it: a lane keeps the ranks of KEYS
// places, which are read and made once, steps without tokens are left out, and the lists are
// counted with scalar instructions.  4 requests of 8 heads and 20000 to 32768 tokens take 27 us,
// 8000 to 8192 tokens 13, with the 32 places that long lists need 17; with every step taken 31 and
// 22.  With weights kept in place of ranks 20000 to 32768 took 39, with weights read anew in each
// pass 50.  More than KEYS times 1024 tokens are read five times.
template <int KEYS>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(EvictParams p) {
  constexpr int kCopies = 4, kStep = kSelectThreads, kRound = KEYS * kStep;
  __shared__ alignas(16) uint32_t bins[kCopies * kBins];
  __shared__ uint32_t wave_sum[kSelectWaves];
  __shared__ uint32_t found[2];
  __shared__ uint32_t sure_count[KEYS * kSelectWaves], same_count[KEYS * kSelectWaves];
  const int r = divide(static_cast<int>(blockIdx.x), p.H);
  const int h = static_cast<int>(blockIdx.x) - r * p.H.d;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Share s = share_of(p, r);
  const float* const w = p.weights + r * p.w_request + h * p.w_head;
  float* const out_w = p.out_weights + r * p.o_request + h * p.o_head;
  int64_t* const kept = p.kept + static_cast<int64_t>(blockIdx.x) * p.keep;

  // This wave's steps of the places from..end, counted anew for each loop: else the compiler keeps
  // all their conditions.
  const auto steps_of = [&](int from, int end) __attribute__((always_inline)) -> int {
    int n = __builtin_amdgcn_readfirstlane((end - from - wave * 64 + kStep - 1) / kStep);
    asm volatile("" : "+s"(n));
    return n;
  };

  // This lane's ranks from place `from` on: of places from + j kStep + tid, and 0, which no weight
  // has, where there is no older token.
  uint32_t rank[KEYS] = {};
  const auto load_ranks = [&](int from) __attribute__((always_inline)) {
    float x[KEYS] = {};
    const int steps = steps_of(from, s.older);
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      if (j < steps) x[j] = w[min(from + j * kStep + tid, s.older - 1)];
    }
#pragma unroll
    for (int j = 0; j < KEYS; ++j)
      rank[j] = from + j * kStep + tid < s.older ? rank_of(x[j]) : 0;
  };
  if (s.older > 0) load_ranks(0);

  // ranks above `cut` are kept, and the first `ties` of those equal to it
  uint32_t cut = 0, ties = 0;
  if (s.need == 0) {
    cut = 0xffffffffu;
  } else if (s.need < s.older) {
    uint32_t left = s.need;
    // the digit of BITS bits from SHIFT on; 0 in place of a rank is below all and changes nothing
    const auto find = [&](auto shift_, auto bits_) __attribute__((always_inline)) {
      constexpr int SHIFT = decltype(shift_)::value, BITS = decltype(bits_)::value;
      constexpr int DONE = SHIFT + BITS;  // the digits from this bit on are known
      for (int i = tid; i < kCopies * kBins / 4; i += kSelectThreads)
        reinterpret_cast<U32x4*>(bins)[i] = U32x4{0, 0, 0, 0};
      __syncthreads();
      for (int from = 0; from < s.older; from += kRound) {
        if (s.older > kRound) load_ranks(from);
        const int steps = steps_of(from, s.older);
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
          if (j < steps && (DONE == 32 || (rank[j] >> (DONE % 32)) == (cut >> (DONE % 32))))
            atomicAdd(&bins[kCopies * ((rank[j] >> SHIFT) & ((1u << BITS) - 1)) + lane % kCopies],
                      1u);
        }
      }
      __syncthreads();
      // thread i has digits 2 i and 2 i + 1 from the highest down
      const auto count = [&](int d) {
        const U32x4 c = *reinterpret_cast<const U32x4*>(&bins[kCopies * d]);
        return c[0] + c[1] + c[2] + c[3];
      };
      const uint32_t high = count(kBins - 1 - 2 * tid), low = count(kBins - 2 - 2 * tid);
      uint32_t upto = sum_upto(high + low, lane);
      if (lane == 63) wave_sum[wave] = upto;
      __syncthreads();
      const int one = lane % kSelectWaves;
      upto += sum16(one < wave ? wave_sum[one] : 0);
      const uint32_t above = upto - high - low;
      if (above < left && upto >= left) {
        const bool second = above + high < left;
        found[0] = kBins - 1 - 2 * tid - second;
        found[1] = above + (second ? high : 0);
      }
      __syncthreads();
      cut |= found[0] << SHIFT;
      left -= found[1];
    };
    find(std::integral_constant<int, 21>{}, std::integral_constant<int, 11>{});
    find(std::integral_constant<int, 10>{}, std::integral_constant<int, 11>{});
    find(std::integral_constant<int, 0>{}, std::integral_constant<int, 10>{});
    ties = left;
  }  // else all

  // The sure ones and those equal to the cut among 64 places each, as bits of the lanes.
  const auto sures_of = [&](int j, int from) -> uint64_t {
    const int at = from + j * kStep + wave * 64;  // the first of the places
    const uint64_t above = __ballot(rank[j] > cut);
    if (at + 64 <= s.older) return above;
    return above | __ballot(at + lane >= s.older && at + lane < s.tokens);
  };
  const auto sames_of = [&](int j) { return ties ? __ballot(rank[j] == cut) : 0ull; };
  uint32_t sure_base = 0, same_base = 0;
  for (int from = 0; from < s.tokens; from += kRound) {
    if (s.tokens > kRound && s.older > 0) load_ranks(from);
    uint32_t sures_here = 0, sames_here = 0;  // lane j: of step j
    const int steps = steps_of(from, s.tokens);
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      if (j >= steps) continue;
      const uint32_t a = __popcll(sures_of(j, from)), b = __popcll(sames_of(j));
      sures_here = lane == j ? a : sures_here;
      sames_here = lane == j ? b : sames_here;
    }
    __syncthreads();
    if (lane < KEYS) {
      sure_count[lane * kSelectWaves + wave] = sures_here;
      same_count[lane * kSelectWaves + wave] = sames_here;
    }
    __syncthreads();
    if (wave < 2) {  // a wave for each kind: the sums before each count
      uint32_t* const counts = wave == 0 ? sure_count : same_count;
      constexpr int kEach = KEYS * kSelectWaves / 64;
      uint32_t c[kEach], total = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        c[i] = counts[lane * kEach + i];
        total += c[i];
      }
      const uint32_t upto = sum_upto(total, lane);
      uint32_t before = upto - total;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        counts[lane * kEach + i] = before;
        before += c[i];
      }
      if (lane == 63) found[wave] = upto;
    }
    __syncthreads();
    if (lane < KEYS) {
      sures_here = sure_count[lane * kSelectWaves + wave];
      sames_here = same_count[lane * kSelectWaves + wave];
    }
    const int again = steps_of(from, s.tokens);
#pragma unroll
    for (int j = 0; j < KEYS; ++j) {
      if (j >= again) continue;
      asm volatile("" : "+v"(rank[j]));  // bits are made anew: there are no registers for all
      const uint64_t sures = sures_of(j, from), sames = sames_of(j);
      if ((sures | sames) == 0) continue;
      const uint32_t same = same_base + __builtin_amdgcn_readlane(sames_here, j);
      uint32_t at = sure_base + __builtin_amdgcn_readlane(sures_here, j) + before_lane(sures);
      bool keep = __builtin_amdgcn_inverse_ballot_w64(sures);
      if (sames == 0) {
        at += min(same, ties);
      } else {
        const uint32_t same_rank = same + before_lane(sames);
        keep |= __builtin_amdgcn_inverse_ballot_w64(sames) && same_rank < ties;
        at += min(same_rank, ties);
      }
      if (keep) {
        const int t = from + j * kStep + tid;
        kept[at] = t;
        out_w[at] = t < s.older ? weight_of(rank[j]) : w[t];
      }
    }
    sure_base += found[0];
    same_base += found[1];
  }
  for (int i = s.kept + tid; i < p.keep; i += kSelectThreads) kept[i] = -1;
  for (int i = s.kept + tid; i < p.out_places; i += kSelectThreads) out_w[i] = 0.0f;
}

constexpr int kMoveThreads = 256, kMoveTokens = 8;

// One workgroup: kMoveTokens new tokens of a request, all heads, keys and values.  V: what a load
// has.  Memory bounds it where rows are whole 16 bytes: 33 MB of keys and as much of values go in
// 22 to 24 us (5.7 TB/s, both ways counted), as 1024 rows of 1024 channels in e4m3 or 4096 of 1024
// in bfloat16 of each request.  Rows in 4 bits go by dwords, with a quotient, a place and two block
// ids for each, and are parts of lines (49 and 47 MB are read): the same rows, 36 and 18 MB each
// way, take 21 and 13.5 us (3.4 and 2.6 TB/s).
template <typename V>
__global__ __launch_bounds__(kMoveThreads) void move_kernel(EvictParams p) {
  const int r = divide(static_cast<int>(blockIdx.x), p.row_tiles);
  const int j0 = (static_cast<int>(blockIdx.x) - r * p.row_tiles.d) * kMoveTokens;
  const int kept = share_of(p, r).kept;
  if (j0 >= kept) return;
  const int count = min(kMoveTokens, kept - j0);
  const int64_t* const table = p.tables + r * p.table_stride;
  const int64_t* const out_table = p.out_tables + r * p.out_table_stride;
  const int rows = count * p.H.d, all = rows * p.pieces.d;
  for (int i = threadIdx.x; i < all; i += kMoveThreads) {
    const int row = divide(i, p.pieces), piece = i - row * p.pieces.d;
    const int j = j0 + divide(row, p.H), h = row - (j - j0) * p.H.d;
    const int t = static_cast<int>(p.kept[(static_cast<int64_t>(r) * p.H.d + h) * p.keep + j]);
    const int from_block = divide(t, p.block_size), to_block = divide(j, p.block_size);
    const int64_t from = table[from_block], to = out_table[to_block];
    if (to < 0 || to >= p.num_blocks) continue;
    const bool in = from >= 0 && from < p.num_blocks;
    const int64_t src =
        (in ? from : 0) * p.blk_stride + (t - from_block * p.block_size.d);
    const int64_t dst = to * p.blk_stride + (j - to_block * p.block_size.d);
    V v[2] = {};
#pragma unroll
    for (int half = 0; half < 2; ++half)
      if (in)
        v[half] = *reinterpret_cast<const V*>(
            p.cache + ((src + half * p.half_stride) * p.H.d + h) * p.row_bytes +
            piece * static_cast<int>(sizeof(V)));
#pragma unroll
    for (int half = 0; half < 2; ++half)
      *reinterpret_cast<V*>(p.cache + ((dst + half * p.half_stride) * p.H.d + h) * p.row_bytes +
                            piece * static_cast<int>(sizeof(V))) = v[half];
  }
}

int check_cache(int64_t cache_layout, int64_t num_blocks, int64_t block_size, int64_t heads,
                int64_t head_dim, const void* kv_cache, int64_t* blk_stride,
                int64_t* half_stride) {
  ORIGAMI_REQUIRE(heads > 0, "heads must be positive");
  // a token's bytes, 512 a head at most, are counted in 31 bits
  ORIGAMI_REQUIRE(heads <= INT32_MAX / 512, "too many heads for one call");
  ORIGAMI_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 256,
                  "head_dim must be a multiple of 8, at most 256");
  ORIGAMI_REQUIRE(num_blocks >= 0 && block_size > 0, "cache block size must be positive");
  if (int rc = cache_geometry(cache_layout, num_blocks, block_size, blk_stride, half_stride))
    return rc;
  ORIGAMI_REQUIRE(block_size <= INT32_MAX / 2 / std::max<int64_t>(num_blocks, 1),
                  "the cache has too many token slots");
  ORIGAMI_REQUIRE(aligned16(kv_cache), "kv_cache must be 16-byte aligned");
  return ORIGAMI_OK;
}

bool paged_dtype(int64_t dtype) {
  return dtype == ORIGAMI_DTYPE_FLOAT16 || dtype == ORIGAMI_DTYPE_BFLOAT16 ||
         dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN || dtype == ORIGAMI_DTYPE_FLOAT4_E2M1;
}

constexpr int64_t kMostTokens = int64_t(1) << 30;

int check_weigh_sizes(int64_t tokens, int64_t query_heads, int64_t heads, int64_t requests,
                      int64_t places) {
  ORIGAMI_REQUIRE(heads > 0 && query_heads > 0 && query_heads % heads == 0,
                  "query heads must be a multiple of the cache's heads");
  ORIGAMI_REQUIRE(tokens >= 0 && requests >= 0 && places >= 0,
                  "token counts must not be negative");
  ORIGAMI_REQUIRE(places <= kMostTokens, "too many tokens for one call");
  ORIGAMI_REQUIRE(tokens < (int64_t(1) << 24) / query_heads, "too many query rows for one call");
  ORIGAMI_REQUIRE(requests < (int64_t(1) << 24) / heads, "too many requests for one call");
  return ORIGAMI_OK;
}

int64_t weigh_workspace(int64_t parts, int64_t requests, int64_t heads, int64_t max_tokens) {
  return parts > 1 ? parts * requests * heads * max_tokens * 4 : 0;
}

}  // namespace

extern "C" {

int64_t origami_accumulate_attention_weights_workspace(int64_t tokens, int64_t query_heads,
                                                       int64_t heads, int64_t requests,
                                                       int64_t places) {
  if (check_weigh_sizes(tokens, query_heads, heads, requests, places)) return -1;
  // the largest for any bound up to `places`: of those with some number of parts the last one
  int64_t bytes = 0;
  for (int64_t n = most_weigh_parts(tokens, query_heads, heads, requests); n > 1; --n) {
    const int64_t tiles = (kWeighUnits - 1) / (requests * heads * (n - 1));
    bytes = std::max(bytes, weigh_workspace(n, requests, heads, std::min(tiles * 256, places)));
  }
  return bytes;
}

int origami_accumulate_attention_weights(
    const void* query, int64_t dtype, const int64_t* strides, int64_t tokens, int64_t query_heads,
    const float* lse, const void* kv_cache, int64_t cache_dtype, int64_t cache_layout,
    int64_t num_blocks, int64_t block_size, int64_t heads, int64_t head_dim,
    const int64_t* block_tables, int64_t table_stride, int64_t table_blocks,
    const int64_t* lengths, int64_t requests, const int64_t* query_starts, int64_t max_tokens,
    double scale, double k_scale, const float* weights, float* out, int64_t places,
    const int64_t* weight_strides, void* workspace, int64_t workspace_bytes,
    origami_stream_t stream_) {
  WeighParams p{};
  int64_t half_stride;
  ORIGAMI_REQUIRE(dtype == ORIGAMI_DTYPE_FLOAT16 || dtype == ORIGAMI_DTYPE_BFLOAT16,
                  "queries must be float16 or bfloat16");
  ORIGAMI_REQUIRE(cache_dtype == dtype || cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN ||
                      cache_dtype == ORIGAMI_DTYPE_FLOAT4_E2M1,
                  "kv_cache must have the queries' dtype or be float8_e4m3fn or in 4 bits");
  if (int rc = check_cache(cache_layout, num_blocks, block_size, heads, head_dim, kv_cache,
                           &p.blk_stride, &half_stride))
    return rc;
  ORIGAMI_REQUIRE(max_tokens >= 0 && table_blocks >= 0, "token counts must not be negative");
  if (int rc = check_weigh_sizes(tokens, query_heads, heads, requests, places)) return rc;
  ORIGAMI_REQUIRE(max_tokens <= places, "max_tokens exceeds the weights' places");
  ORIGAMI_REQUIRE(ceil_div(max_tokens, block_size) <= table_blocks,
                  "max_tokens exceeds the block tables");
  ORIGAMI_REQUIRE(query_starts != nullptr || tokens == requests,
                  "without query_starts every request has one query token");
  ORIGAMI_REQUIRE(cache_scale(k_scale), "cache scales must be positive and finite in binary32");
  ORIGAMI_REQUIRE(cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN || k_scale == 1.0,
                  "cache scales are for float8_e4m3fn caches");
  p.scale = static_cast<float>(scale * k_scale);
  ORIGAMI_REQUIRE(std::isfinite(p.scale), "scale must be finite in binary32");
  ORIGAMI_REQUIRE(strides[0] >= 0 && strides[1] >= 0, "row strides must not be negative");
  for (int i = 0; i < 4; ++i)
    ORIGAMI_REQUIRE(weight_strides[i] >= 0, "weight strides must not be negative");
  ORIGAMI_REQUIRE(table_stride >= 0, "the table stride must not be negative");
  if (requests == 0 || places == 0) return ORIGAMI_OK;
  ORIGAMI_REQUIRE((tokens == 0 || (query != nullptr && lse != nullptr)) && out != nullptr &&
                      lengths != nullptr && (block_tables != nullptr || max_tokens == 0) &&
                      (kv_cache != nullptr || num_blocks == 0),
                  "queries, weights, lengths, tables and the cache must not be null");
  const int64_t parts = weigh_parts(tokens, query_heads, heads, requests, max_tokens);
  // the join has a workgroup row for every request and head
  ORIGAMI_REQUIRE(parts == 1 || requests * heads <= 65535, "too many requests for one call");
  ORIGAMI_REQUIRE(workspace_bytes >= weigh_workspace(parts, requests, heads, max_tokens) &&
                      (parts == 1 || workspace != nullptr) && aligned16(workspace),
                  "the workspace of the weights is too small");
  p.parts = divisor(parts);
  p.requests = divisor(requests);
  p.part_sums = static_cast<float*>(workspace);
  p.query = query;
  p.q_token = strides[0];
  p.q_head = strides[1];
  p.q_vec = aligned16(query) && strides[0] % 8 == 0 && strides[1] % 8 == 0;
  p.lse = lse;
  p.cache = static_cast<const uint8_t*>(kv_cache);
  p.num_blocks = num_blocks;
  p.tables = block_tables;
  p.lengths = lengths;
  p.starts = query_starts;
  p.table_stride = table_stride;
  p.block_size = divisor(block_size);
  p.H = divisor(heads);
  p.G = divisor(query_heads / heads);
  p.tokens = static_cast<int32_t>(tokens);
  p.Hq = static_cast<int32_t>(query_heads);
  p.D = static_cast<int32_t>(head_dim);
  p.max_tokens = static_cast<int32_t>(max_tokens);
  p.places = static_cast<int32_t>(places);
  p.weights = weights;
  p.out = out;
  p.w_request = weight_strides[0];
  p.w_head = weight_strides[1];
  p.o_request = weight_strides[2];
  p.o_head = weight_strides[3];
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  return dtype == ORIGAMI_DTYPE_BFLOAT16
             ? launch_weigh<bf16>(p, cell_of(cache_dtype), requests, stream)
             : launch_weigh<f16>(p, cell_of(cache_dtype), requests, stream);
}

int origami_evict_kv_cache(
    void* kv_cache, int64_t cache_dtype, int64_t cache_layout, int64_t num_blocks,
    int64_t block_size, int64_t heads, int64_t head_dim, const int64_t* block_tables,
    int64_t table_stride, int64_t table_blocks, const int64_t* lengths, int64_t requests,
    int64_t max_tokens, const float* weights, int64_t places, const int64_t* out_tables,
    int64_t out_table_stride, int64_t out_table_blocks, int64_t keep, int64_t recent,
    int64_t* kept, float* out_weights, int64_t out_places, const int64_t* weight_strides,
    origami_stream_t stream_) {
  EvictParams p{};
  ORIGAMI_REQUIRE(paged_dtype(cache_dtype),
                  "kv_cache must be float16, bfloat16 or float8_e4m3fn or in 4 bits");
  if (int rc = check_cache(cache_layout, num_blocks, block_size, heads, head_dim, kv_cache,
                           &p.blk_stride, &p.half_stride))
    return rc;
  ORIGAMI_REQUIRE(requests >= 0 && max_tokens >= 0 && places >= 0 && keep >= 0 && recent >= 0 &&
                      out_places >= 0 && table_blocks >= 0 && out_table_blocks >= 0,
                  "token counts must not be negative");
  ORIGAMI_REQUIRE(max_tokens <= kMostTokens && keep <= kMostTokens && out_places <= kMostTokens,
                  "too many tokens for one call");
  ORIGAMI_REQUIRE(requests < (int64_t(1) << 22) / heads, "too many requests for one call");
  ORIGAMI_REQUIRE(max_tokens <= places, "max_tokens exceeds the weights' places");
  const int64_t most = std::min(keep, max_tokens);
  ORIGAMI_REQUIRE(most <= out_places, "what is kept exceeds the places of out_weights");
  ORIGAMI_REQUIRE(ceil_div(max_tokens, block_size) <= table_blocks,
                  "max_tokens exceeds the block tables");
  ORIGAMI_REQUIRE(ceil_div(most, block_size) <= out_table_blocks,
                  "what is kept exceeds the new block tables");
  for (int i = 0; i < 4; ++i)
    ORIGAMI_REQUIRE(weight_strides[i] >= 0, "weight strides must not be negative");
  ORIGAMI_REQUIRE(table_stride >= 0 && out_table_stride >= 0,
                  "the table strides must not be negative");
  const int row_bytes = row_bytes_of(cell_of(cache_dtype), static_cast<int>(head_dim));
  // rows that are whole 16 bytes move so, others by 4
  const int load = row_bytes % 16 == 0 ? 16 : 4;
  ORIGAMI_REQUIRE(heads <= INT32_MAX / kMoveTokens / 128, "too many heads for one call");
  const int64_t tiles = std::max<int64_t>(ceil_div(most, kMoveTokens), 1);
  ORIGAMI_REQUIRE(tiles < (int64_t(1) << 24) / std::max<int64_t>(requests, 1),
                  "too many tokens for one call");
  if (requests == 0) return ORIGAMI_OK;
  ORIGAMI_REQUIRE(lengths != nullptr && (weights != nullptr || max_tokens == 0) &&
                      (kept != nullptr || keep == 0) &&
                      (out_weights != nullptr || out_places == 0) &&
                      (block_tables != nullptr || max_tokens == 0) &&
                      (out_tables != nullptr || most == 0) &&
                      (kv_cache != nullptr || num_blocks == 0),
                  "weights, lengths, tables, results and the cache must not be null");
  p.cache = static_cast<uint8_t*>(kv_cache);
  p.num_blocks = num_blocks;
  p.tables = block_tables;
  p.out_tables = out_tables;
  p.lengths = lengths;
  p.table_stride = table_stride;
  p.out_table_stride = out_table_stride;
  p.block_size = divisor(block_size);
  p.H = divisor(heads);
  p.max_tokens = static_cast<int32_t>(max_tokens);
  p.keep = static_cast<int32_t>(keep);
  p.recent = static_cast<int32_t>(std::min(recent, kMostTokens));
  p.out_places = static_cast<int32_t>(out_places);
  p.weights = weights;
  p.out_weights = out_weights;
  p.w_request = weight_strides[0];
  p.w_head = weight_strides[1];
  p.o_request = weight_strides[2];
  p.o_head = weight_strides[3];
  p.kept = kept;
  p.row_bytes = row_bytes;
  p.pieces = divisor(row_bytes / load);
  p.row_tiles = divisor(tiles);
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const dim3 lists(static_cast<unsigned>(requests * heads)), threads(kSelectThreads);
  if (max_tokens <= 4 * kSelectThreads)
    hipLaunchKernelGGL(select_kernel<4>, lists, threads, 0, stream, p);
  else if (max_tokens <= 16 * kSelectThreads)
    hipLaunchKernelGGL(select_kernel<16>, lists, threads, 0, stream, p);
  else
    hipLaunchKernelGGL(select_kernel<32>, lists, threads, 0, stream, p);
  if (int rc = check_launch("select_kernel")) return rc;
  if (most == 0) return ORIGAMI_OK;
  const dim3 grid(static_cast<unsigned>(requests * tiles)), block(kMoveThreads);
  if (load == 16)
    hipLaunchKernelGGL(move_kernel<U32x4>, grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL(move_kernel<uint32_t>, grid, block, 0, stream, p);
  return check_launch("move_kernel");
}

}  // extern "C"
