// origami_attention.hip -- attention over the paged KV cache for a batch that shares a prefix.
//
// For a query row q (one token, one query head) over the keys k_t and values v_t it sees:
//   s_t = scale * (q . k_t),  out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  m = max_t s_t
// The tokens come in parts (the prefix, the request's own tokens, ranges of either).  A part
// gives m, the sum l and the unnormalised row O in binary32; parts are joined with the weights
// exp(m_part - m), so that no part waits for another.  Scores, maxima, sums and O are binary32;
// the exponentials are rounded to the queries' type for the matrix instruction, which adds half a
// step of the weighted mean of |v|, about what rounding the result does.
//
// Where requests have too few rows to fill workgroups by themselves, the rows of all of them are
// one matrix against each tile of the prefix, so its keys and values are read once (64 requests
// over 32768 tokens and 33 thousand of their own: 282 MB from memory of 281 that there are).  Else
// each request reads the prefix with its own tokens; the bound of a request's queries decides for
// the whole batch (plan_of).  With few rows a call is bound by memory and, below some tens of
// microseconds, by the chain of loads at a workgroup's start (lengths, block ids, rows); with rows
// by the hundred by the vector instructions of the softmax, which are as many cycles as the
// products' matrix instructions and run beside them only in part: 710 to 815 TFLOP/s (600 to 525
// us, on different boxes) for prompts of up to 1024 tokens after 8192, with the matrix units busy
// in 46% of the CUs' busy cycles, where a large library product reaches 1150.
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

// Rows of a workgroup, and its waves.  Waves take 16 or 32 rows; in the larger shapes more of them
// have rows of their own, in the smaller ones more have tokens of their own.  Four waves are half
// of a CU's LDS and registers with up to 128 channels, so that one workgroup's start and end are
// beside another's products (against eight waves: 93 us for 103 for 64 requests over 32768
// tokens, 34 for 40 for 16 over 16384 in e4m3).  The last shape, for requests of many rows and 65
// to 128 channels, shares tiles among eight waves: 536 us for 616 for prompts of up to 1024 tokens
// after 8192.  With 64 channels it is the slower one: 427 us for 406 to 413 for the same prompts,
// 242 for 199 to 209 with 12 heads in half precision.  With more channels there are the first two
// shapes, and a workgroup to a CU.
constexpr int kShapeRows[4] = {16, 64, 128, 256};
constexpr int kShapeWaves[4] = {4, 4, 4, 8};

constexpr int kJoinThreads = 256, kJoinWaves = kJoinThreads / 64;
// Exponentials are taken 2^kLift times as large for half precision, so that those of tokens far
// below the maximum keep their precision (down to 2^-24 of the largest) and sums of 2^30 of
// the largest stay far from binary32's limit.
template <typename T>
constexpr float kLift = std::is_same<T, f16>::value ? 10.0f : 0.0f;
// How far (in powers of two) the maximum may rise before what is summed so far is scaled down;
// 2^(kLift + kSlack) is within half precision.
template <typename T>
constexpr float kSlack = std::is_same<T, f16>::value ? 4.0f : 8.0f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

constexpr int64_t kCus = 256;
constexpr int kFewParts = 8;
constexpr int kMaxParts = 1024;  // of a row: twice kCus at most of either kind
constexpr int64_t kMostUnits = (int64_t(1) << 32) / 512;  // workgroups of 512 threads in a launch

// The work of one kind: row tiles of every KV head, over ranges of tokens.
struct Group {
  int32_t units;   // workgroups
  int32_t shape;   // kShapeRows[shape] rows each, at most
  Divisor tiles;   // row tiles of a request, or of the batch
  int32_t splits;  // ranges of `chunk` tokens
  int32_t chunk;
  int32_t slot;    // the partial results' first slot
  int32_t first;   // the first token of range 0
};

struct AttendParams {
  const void* query;
  int64_t q_token, q_head;  // strides, in elements
  void* out;
  int64_t o_token, o_head;
  bool out_vec;  // its rows start on 8 bytes
  float* lse;  // [tokens, query heads], or null
  const uint8_t* cache;
  int64_t blk_stride, half_stride;  // rows of H * D, as cache_geometry
  int64_t num_blocks;
  const int64_t *prefix_ids, *tables, *own_tokens, *starts;
  int64_t table_stride;
  Divisor block_size, requests, H, G;
  int32_t prefix, max_own, max_query;
  int32_t tokens, Hq, D;
  float scale, v_scale;  // scale includes log2 e and the keys' scale
  Group group[2];        // the prefix with the whole batch's rows; each request's rows
  int32_t slots;
  float *part_o, *part_ml;  // [slots][rows][D], [slots][rows][2]
};

// A load that is known to be from memory and not from LDS (whose waits it would share).
template <typename V>
__device__ __forceinline__ V load_global(const uint8_t* p) {
  return *(const __attribute__((address_space(1))) V*)(reinterpret_cast<uintptr_t>(p));
}

// What a lane reads of a row that is not in the cache, and of channels past the last.
__device__ const U32x4 kZeros = {0, 0, 0, 0};

// MR x MR scores or results: value x of a lane is in column lane % MR and in row
// 4 (lane / MR) + x % 4 + (256 / MR) (x / 4).
template <int MR>
using Tile = float __attribute__((ext_vector_type(MR * MR / 64)));

// c + a b, where a lane has 8 values of row (a) and column (b) lane % MR, from 8 (lane / MR) on.
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

typedef short Short4 __attribute__((ext_vector_type(4)));

// Four tokens' values of one channel: 16 lanes read four rows of 16 channels, 8 bytes a lane
// (lane 4 k + q: channels 4 q .. 4 q + 3 of row k), and each gets its channel's column.
__device__ __forceinline__ U32x2 read_column(const uint8_t* p) {
  return __builtin_bit_cast(U32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) Short4*)p));
}

// Four channels of a cache row.
template <typename T, bool FP8>
__device__ __forceinline__ Float4 four_values(const uint8_t* row, int ch) {
  Float4 out;
  if constexpr (FP8) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + ch);
    const Vec2<T> a = fp8_pair<false>(w, T()), b = fp8_pair<true>(w, T());
    out = Float4{static_cast<float>(a[0]), static_cast<float>(a[1]), static_cast<float>(b[0]),
                 static_cast<float>(b[1])};
  } else {
    const Vec4<T> v = *reinterpret_cast<const Vec4<T>*>(row + 2 * ch);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = static_cast<float>(v[j]);
  }
  return out;
}

// Infinities and NaN among eight values become 0; whether there were any.
template <typename T>
__device__ __forceinline__ bool drop_odd(U32x4& w) {
  constexpr uint32_t low = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u, high = low << 16;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool l = (w[i] & low) == low, h = (w[i] & high) == high;
    odd |= l || h;
    w[i] = (l ? 0u : w[i] & 0xffffu) | (h ? 0u : w[i] & 0xffff0000u);
  }
  return odd;
}
// The same for e4m3, whose NaN is all ones but the sign.
template <typename T>
__device__ __forceinline__ bool drop_odd(U32x2& w) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 32; j += 8)
      if (((w[i] >> j) & 0x7fu) == 0x7fu) {
        odd = true;
        w[i] &= ~(0xffu << j);
      }
  return odd;
}

// Four values rounded to T; `vec`: rows start on 8 bytes.
template <typename T>
__device__ __forceinline__ void store4(T* dst, Float4 v, bool vec) {
  Vec4<T> w;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = static_cast<T>(v[j]);
  if (vec) {
    *reinterpret_cast<Vec4<T>*>(dst) = w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) dst[j] = w[j];
}

// A request's place in the batch.
struct Request {
  int32_t first, count;  // its query tokens
  int32_t own;           // its own tokens, up to the bound
  int32_t before;        // of all its own tokens, those before its queries (may be negative)
};

__device__ __forceinline__ Request request_of(const AttendParams& p, int r) {
  Request q{r, 1, 0, 0};
  if (p.starts) {
    const int64_t n = p.tokens;
    const int64_t a = min(max(p.starts[r], int64_t(0)), n);
    const int64_t b = min(max(p.starts[r + 1], a), n);
    q.first = static_cast<int32_t>(a);
    q.count = static_cast<int32_t>(min(b - a, static_cast<int64_t>(p.max_query)));
  }
  // The queries' places follow from the whole length; the bound only hides tokens.  Lengths past
  // any bound (2^30) and any number of queries (2^24) besides are the same.
  const int32_t length =
      static_cast<int32_t>(min(max(p.own_tokens[r], int64_t(0)), int64_t(3) << 29));
  q.own = min(length, p.max_own);
  q.before = length - q.count;
  return q;
}

__device__ __forceinline__ uint32_t as_u32(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ float as_float(uint32_t x) { return __builtin_bit_cast(float, x); }

// The largest of the values of lanes c, c + MR, ..., without a trip through LDS.
template <int MR>
__device__ __forceinline__ float max_over_groups(float x) {
  if constexpr (MR == 16) {
    const auto pair = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
    const uint32_t one = pair[0], other = pair[1];
    x = fmaxf(as_float(one), as_float(other));
  }
  const auto pair = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
  const uint32_t one = pair[0], other = pair[1];
  return fmaxf(as_float(one), as_float(other));
}

// x folded over the wave, without a trip through LDS.
template <typename Fold>
__device__ __forceinline__ float fold_wave(float x, Fold fold) {
  x = fold_lanes<16>(x, fold);
  const auto rows = __builtin_amdgcn_permlane16_swap(as_u32(x), as_u32(x), false, false);
  uint32_t one = rows[0], other = rows[1];
  x = fold(as_float(one), as_float(other));
  const auto halves = __builtin_amdgcn_permlane32_swap(as_u32(x), as_u32(x), false, false);
  one = halves[0];
  other = halves[1];
  return fold(as_float(one), as_float(other));
}

// Where the 16-byte piece `piece` of token `tok`'s row is in LDS, in pieces of its row.  Keys are
// read by 16 lanes from the same piece of 16 tokens, values by 32 lanes from pieces next to each
// other (2 of 8 tokens, or 4 of 4): with the token's low bits in the piece's number these
// are in different banks (of 256 bytes: two 128-byte rows of 64 channels, one of 128).
template <int DP>
__device__ __forceinline__ int key_piece(int tok, int piece) {
  return piece ^ (DP == 64 ? (tok >> 1) & 7 : tok & 15);
}
template <int DP, int MR>
__device__ __forceinline__ int value_piece(int tok, int piece) {
  const int t = DP == 64 ? tok >> 1 : tok;
  if (MR == 16) return piece ^ ((t & (DP == 64 ? 3 : 7)) << 1);
  return piece ^ ((t & (DP == 64 ? 1 : 3)) << 2);
}

// The values of MR channels (tile d) of a tile's k-th part, as V P takes them: value j is that
// of token 4 (lane / MR) + j % 4 + (256 / MR) (2 k + j / 4).
template <typename T, int DP, int MR>
__device__ __forceinline__ Vec8<T> read_values(const uint8_t* values, int lane, int k, int d) {
  constexpr int NCH = DP / 8;
  const int c16 = lane & 15;
  U32x4 out;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int tok = 256 / MR * (2 * k + j) + 4 * (lane / MR) + (c16 >> 2);
    const int piece = MR / 8 * d + (MR == 32 ? ((lane >> 4) & 1) * 2 : 0) + ((c16 & 3) >> 1);
    const U32x2 w =
        read_column(values + (tok * NCH + value_piece<DP, MR>(tok, piece)) * 16 + (c16 & 1) * 8);
    out[2 * j] = w[0];
    out[2 * j + 1] = w[1];
  }
  return __builtin_bit_cast(Vec8<T>, out);
}

template <int N>
using Int = std::integral_constant<int, N>;

// Tokens that a team of waves (the WR waves with the same tokens) has in LDS at a time.
template <int DP, int WR>
constexpr int kTeamTokens = WR == 8 || (WR == 4 && DP == 64) ? 64 : 32;

// One workgroup: WR MR rows of one KV head over a range of tokens.  Its NW waves are WR row waves
// by WT token waves: a wave takes MR rows, and of every WT kTeamTokens tokens its share.  Rows
// (queries, results, sums) stay in registers; keys and values go through LDS, where the WR waves
// of a team share them, and the next ones are on their way to registers meanwhile.  They go
// through registers for e4m3, which is widened on the way, and for the tiles that some rows see in
// part, whose odd values are dropped; other tiles do not need it, but loads of theirs straight to
// LDS have not been measured.  With WR = 1 no wave needs another until the end; else buffers take
// turns, so that one barrier a tile is enough.
template <typename T, bool FP8, int DP, int MR, int WR, int NW>
__device__ __forceinline__ void attend(const AttendParams& p, const Group& g, int unit, bool batch,
                                       uint8_t* lds, float* ml) {
  constexpr int WT = NW / WR, TT = kTeamTokens<DP, WR>;
  constexpr int NG = 64 / MR;             // lane groups: the depth of a product is 8 NG
  constexpr int KS = DP / (8 * NG);       // depth steps of K Q
  constexpr int DT = DP / MR;             // channel tiles of V P
  constexpr int X = TT / NG;              // scores of a lane in a tile
  constexpr int ACC = MR * MR / 64;       // values of a lane in a tile
  constexpr int STRIDE = 4 * NG;          // tokens between a lane's groups of four
  constexpr int NCH = DP / 8;             // 16-byte pieces of a row in LDS
  constexpr int RPI = 64 / NCH;           // rows of one load
  constexpr int IT = TT / (RPI * WR);     // loads of a tile
  constexpr bool kAhead = WR == 8;        // scores are a step ahead: see below
  constexpr int kBuffers = WR == 1 ? 1 : (kAhead ? 3 : 2);
  constexpr int kTile = TT * DP * 2;      // bytes of a team's keys
  // one value for the wave, so that what follows from it is scalar and its conditions are branches
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wr = wave % WR, wt = wave / WR;
  const int c = lane % MR, q4 = lane / MR;

  // The unit: row tiles of the same keys are 8 units apart, so that they run on the same chiplet
  // at about the same time and its L2 gives the keys to all but the first.
  const int eight = unit >> 3, eighth = unit & 7;
  int u = divide(eight, g.tiles);
  const int tile = eight - u * g.tiles.d;
  u = u * 8 + eighth;
  const int uh = divide(u, p.H), h = u - uh * p.H.d;
  int r = 0, split = uh;
  if (!batch) {
    split = divide(uh, p.requests);
    r = uh - split * p.requests.d;
  }
  if (split >= g.splits) return;
  const int t0 = g.first + split * g.chunk;
  const int64_t* const table = p.tables + static_cast<int64_t>(r) * p.table_stride;
  // The block of token t.  Blocks of the first tokens are asked for before the request's length is
  // known: up to the bounds that the host has, the tables can be read.
  const int bound = batch ? p.prefix : p.prefix + p.max_own;
  const auto block_of = [&](int t, int before) -> int64_t {
    if (t >= before) return -1;
    const bool pre = t < p.prefix;
    return (pre ? p.prefix_ids : table)[divide(pre ? t : t - p.prefix, p.block_size)];
  };
  constexpr int kRound = WT * TT;  // tokens of a step of the workgroup
  const int tl = lane % TT;
  int t = t0 + wt * TT;  // the first of this wave's tokens
  const int64_t first = block_of(t + tl, bound);
  int64_t ahead = block_of(t + kRound + tl, bound);

  const Request rq = batch ? Request{0, p.tokens, 0, 0} : request_of(p, r);
  const int rows = rq.count * p.G.d, row0 = tile * WR * MR;
  if (row0 >= rows) return;
  const int end = batch ? p.prefix : p.prefix + rq.own;  // of the tokens, prefix first

  // this lane's row
  const int row = row0 + wr * MR + c;
  const auto seen_by = [&](int i) -> int {  // tokens that row i sees
    return p.prefix +
           (batch ? 0 : min(max(rq.before + divide(i, p.G) + 1, 0), rq.own));
  };
  const int limit = seen_by(row);
  // the scale's sign goes with the queries, and so does a scale of zero, so that hidden scores of
  // -infinity stay what they are
  const float scale = p.scale == 0.0f ? 1.0f : fabsf(p.scale);
  Vec8<T> qf[KS];
  {
    const int qi = divide(row, p.G), head = h * p.G.d + row - qi * p.G.d;
    const T* const src =
        static_cast<const T*>(p.query) + (rq.first + qi) * p.q_token + head * p.q_head;
    const bool vec =
        ((reinterpret_cast<uintptr_t>(p.query) | 2 * p.q_token | 2 * p.q_head) & 15) == 0;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int d = 8 * (NG * k + q4);
      qf[k] = Vec8<T>{};
      if (row < rows && d < p.D) {
        if (vec) {
          qf[k] = *reinterpret_cast<const Vec8<T>*>(src + d);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) qf[k][j] = src[d + j];
        }
        if (p.scale <= 0.0f) qf[k] = p.scale == 0.0f ? Vec8<T>{} : -qf[k];
      }
    }
  }
  // The tokens that some row of the workgroup sees, and those that all rows of the wave see;
  // limits grow along the rows.
  const int most = seen_by(min(row0 + WR * MR, rows) - 1);
  const int least = seen_by(min(row0 + wr * MR, rows - 1));
  const int nearest = seen_by(row0);  // the tokens that all rows of the workgroup see
  const int t1 = min(min(end, most), t0 + g.chunk);

  Tile<MR> o[DT];
  float base = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int x = 0; x < ACC; ++x) o[d][x] = 0.0f;

  uint8_t* const team = lds + wt * kBuffers * 2 * kTile;
  const int piece = lane % NCH, sub = lane / NCH;
  const bool has = 8 * piece < p.D;
  constexpr int cell = FP8 ? 1 : 2;
  const int64_t pitch = static_cast<int64_t>(p.H.d) * p.D * cell;
  const uint8_t* const keys =
      p.cache + (static_cast<int64_t>(h) * p.D + (has ? 8 * piece : 0)) * cell;
  const int64_t to_values = p.half_stride * pitch;

  // the cache row of token t, -1 where it has none
  const auto row_of = [&](int t, int64_t id) -> int {
    if (t >= t1 || id < 0 || id >= p.num_blocks) return -1;
    const int i = t < p.prefix ? t : t - p.prefix;
    return static_cast<int>(id * p.blk_stride + i - divide(i, p.block_size) * p.block_size.d);
  };
  using Raw = typename std::conditional<FP8, U32x2, U32x4>::type;
  Raw kr[IT], vr[IT];
  const auto load_tile = [&](int mine) {
    const uint8_t* const zeros = reinterpret_cast<const uint8_t*>(&kZeros);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = __shfl(mine, (i * WR + wr) * RPI + sub);
      const bool in = r >= 0 && has;
      const uint8_t* const src = keys + r * pitch;
      kr[i] = load_global<Raw>(in ? src : zeros);
      vr[i] = load_global<Raw>(in ? src + to_values : zeros);
    }
  };
  // Where some rows may not see some of a tile's tokens: a hidden token's weight is 0, but 0 times
  // an infinity or NaN is NaN.  Such values go in as 0, and reach the rows that see them at the
  // end.
  bool odd = false;
  const auto drop_odd_values = [&](int t) {
    if (min(t + TT, t1) > nearest)
#pragma unroll
      for (int i = 0; i < IT; ++i) odd |= drop_odd<T>(vr[i]);
  };
  const auto store_tile = [&](uint8_t* buf) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int tok = (i * WR + wr) * RPI + sub;
      U32x4 kv, vv;
      if constexpr (FP8) {
        kv = fp8_expand<T>(kr[i]);
        vv = fp8_expand<T>(vr[i]);
      } else {
        kv = kr[i];
        vv = vr[i];
      }
      *reinterpret_cast<U32x4*>(buf + (tok * NCH + key_piece<DP>(tok, piece)) * 16) = kv;
      *reinterpret_cast<U32x4*>(buf + kTile + (tok * NCH + value_piece<DP, MR>(tok, piece)) * 16) =
          vv;
    }
  };

  // With one buffer a wave's tile goes to LDS before its products, and the next one is on its way
  // to registers.  With two, the next tile goes to LDS in the middle of a tile's products, and
  // the one after it is on its way.
  int mine = row_of(t + tl, first), turn = 0;
  uint64_t there = __ballot(mine >= 0), next_there = 0;  // twice 32 tokens where TT is 32
  if (t0 < t1) {
    load_tile(mine);
    mine = row_of(t + kRound + tl, ahead);
    ahead = block_of(t + 2 * kRound + tl, t1);
    if constexpr (kBuffers > 1) {
      drop_odd_values(t);
      store_tile(team);
      load_tile(mine);
      next_there = __ballot(mine >= 0);
      mine = row_of(t + 2 * kRound + tl, ahead);
      ahead = block_of(t + 3 * kRound + tl, t1);
      __syncthreads();
    }
  }
  // A step: the maxima and sums with `count` scores a lane of the tokens from `ts` on, with the
  // instructions of `between` among those of the exponentials; then O += V P.
  const auto soften = [&](auto& sc, auto count, int ts, uint64_t seen, bool whole, auto between,
                          const uint8_t* vb) {
    constexpr int N = decltype(count)::value;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int tok = STRIDE * (i / 4) + 4 * q4 + i % 4;
        if (ts + tok >= limit || !((seen >> tok) & 1)) sc[i / ACC][i % ACC] = -INFINITY;
      }
    }
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) best = fmaxf(best, sc[i / ACC][i % ACC]);
    best = max_over_groups<MR>(best) * scale;
    const bool rises = best > base + kSlack<T>;
    if (__any(rises)) {  // each row by itself: no row's rounding depends on another
      const float next = rises ? best : base;
      const float keep = __builtin_amdgcn_exp2f(base - (next == -INFINITY ? 0.0f : next));
      base = next;
      sum *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= keep;
    }
    between();
    const float below = kLift<T> - (base == -INFINITY ? 0.0f : base);
    Vec8<T> pf[N / 8];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = __builtin_amdgcn_exp2f(fmaf(sc[i / ACC][i % ACC], scale, below));
      sum += e;
      pf[i / 8][i % 8] = static_cast<T>(e);
    }
    // O += V P
#pragma unroll
    for (int k = 0; k < N / 8; ++k)
#pragma unroll
      for (int d = 0; d < DT; ++d)
        o[d] = mfma<T, MR>(read_values<T, DP, MR>(vb, lane, k, d), pf[k], o[d]);
  };
  // S = K Q: row c against token STRIDE (i / 4) + 4 q4 + i % 4, all tiles of 16 or 32 tokens
  // together, so that no product waits for the one before it
  const auto score = [&](auto& sc, auto tiles, const uint8_t* kb) {
    constexpr int N = decltype(tiles)::value;
#pragma unroll
    for (int m = 0; m < N; ++m)
#pragma unroll
      for (int x = 0; x < ACC; ++x) sc[m][x] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int m = 0; m < N; ++m) {
        const int tok = MR * m + c;
        const Vec8<T> kf = *reinterpret_cast<const Vec8<T>*>(
            kb + (tok * NCH + key_piece<DP>(tok, NG * k + q4)) * 16);
        sc[m] = mfma<T, MR>(kf, qf[k], sc[m]);
      }
  };
  // with a barrier in it, the loop is the same for all waves
  if constexpr (kAhead) {
    // A tile is two steps, and the products K Q of a step run under the exponentials of the one
    // before: the vector unit has as much to do for a step as the matrix unit.  The first step of
    // the next tile comes before the last one's values are done with, hence three buffers.
    static_assert(TT == 64 && MR == 32 && WT == 1, "two steps of 32 tokens");
    constexpr int kHalf = TT / 2 * DP * 2;  // bytes of a step's keys
    Tile<MR> sa[1], sb[1];
    int next = 1;
    if (t0 < t1) score(sa, Int<1>{}, team);
    for (; t < t1; t += kRound) {
      uint8_t* const buf = team + turn * 2 * kTile;
      uint8_t* const other = team + next * 2 * kTile;
      const bool whole = there == ~0ull && t + TT <= least;
      drop_odd_values(t + kRound);
      soften(sa, Int<X / 2>{}, t, there, whole, [&] { score(sb, Int<1>{}, buf + kHalf); },
             buf + kTile);
      store_tile(other);
      load_tile(mine);
      __syncthreads();
      soften(sb, Int<X / 2>{}, t + TT / 2, there >> 32, whole,
             [&] { score(sa, Int<1>{}, other); }, buf + kTile + kHalf);
      there = next_there;
      next_there = __ballot(mine >= 0);
      mine = row_of(t + 3 * kRound + tl, ahead);
      ahead = block_of(min(t + 4 * kRound + tl, t1 - 1), t1);
      turn = next;
      next = next == 2 ? 0 : next + 1;
    }
  } else {
    for (int tb = t0; (WR == 1 ? t : tb) < t1; tb += kRound, t += kRound) {
      uint8_t* const buf = team + turn * 2 * kTile;
      if constexpr (kBuffers == 1) {
        drop_odd_values(t);
        store_tile(buf);
        __builtin_amdgcn_wave_barrier();
        load_tile(mine);
        next_there = __ballot(mine >= 0);
        mine = row_of(t + 2 * kRound + tl, ahead);
        ahead = block_of(min(t + 3 * kRound + tl, t1 - 1), t1);
      } else {
        drop_odd_values(t + kRound);
      }
      const bool whole = there == ~0ull && t + TT <= least;
      Tile<MR> sc[X / ACC];
      score(sc, Int<X / ACC>{}, buf);
      if constexpr (kBuffers == 2) {
        store_tile(team + (turn ^ 1) * 2 * kTile);
        load_tile(mine);
      }
      soften(sc, Int<X>{}, t, there, whole, [] {}, buf + kTile);
      there = next_there;
      if constexpr (kBuffers == 1) {
        __builtin_amdgcn_wave_barrier();
      } else {
        next_there = __ballot(mine >= 0);
        mine = row_of(t + 3 * kRound + tl, ahead);
        ahead = block_of(min(t + 4 * kRound + tl, t1 - 1), t1);
        __syncthreads();
        turn ^= 1;
      }
    }
  }

#pragma unroll
  for (int x = MR; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
  if (t1 > nearest) odd = __syncthreads_or(odd);

  // Calls add(row of the cache's values) for the tokens among which drop_odd_values left out
  // infinities and NaN, as far as a row sees them.  The first ones may be tokens before those,
  // whose values have been added already, and an infinity or NaN twice is the same.
  const auto each_odd_token = [&](int row, auto add) {
    for (int i = max(t0, nearest - TT); i < min(t1, seen_by(row)); ++i) {
      const int at_row = row_of(i, block_of(i, t1));
      if (at_row >= 0)
        add(p.cache + (at_row + p.half_stride) * pitch + static_cast<int64_t>(h) * p.D * cell);
    }
  };
  const auto odd_part = [](Float4 v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = fabsf(v[j]) < INFINITY ? 0.0f : v[j];
    return v;
  };
  // Four channels of a row's result, and with the first ones its maximum and sum.
  const auto put = [&](int row, int ch, Float4 v, float base, float sum) {
    if (row >= rows || ch >= p.D) return;
    const int qi = divide(row, p.G), head = h * p.G.d + row - qi * p.G.d;
    const int64_t n = rq.first + qi, at = n * p.Hq + head;
    if (p.slots > 1) {
      const int64_t slot =
          (g.slot + split) * (static_cast<int64_t>(p.tokens) * p.Hq) + at;
      if (ch == 0) {
        p.part_ml[2 * slot] = base - kLift<T>;
        p.part_ml[2 * slot + 1] = sum;
      }
      // without a token the join does not read the rest
      if (sum != 0.0f) *reinterpret_cast<Float4*>(p.part_o + slot * p.D + ch) = v;
    } else {
      // a row without a weight is zero also where a value is infinite or NaN
      if (sum == 0.0f) v = Float4{0.0f, 0.0f, 0.0f, 0.0f};
      const float inv = sum == 0.0f ? 0.0f : p.v_scale / sum;
      store4(static_cast<T*>(p.out) + n * p.o_token + head * p.o_head + ch, v * inv, p.out_vec);
      if (p.lse && ch == 0)
        p.lse[at] = sum == 0.0f ? -INFINITY : kLn2 * (base - kLift<T> + log2f(sum));
    }
  };

  if constexpr (WT > 1) {
    // Join the token waves through LDS.  With one row wave each leaves its part in its own tiles,
    // which no other wave reads, and all waves add up a share of the rows; else all but the
    // first token wave leave theirs, which that one adds to its own.
    constexpr int M = WR * MR, kPitch = DP + 4, kPart = WR == 1 ? 2 * kTile : M * kPitch * 4;
    static_assert((WR > 1 || MR * kPitch * 4 <= 2 * kTile) &&
                      (WT - 1) * kPart <= 512 * DP, "LDS");
    if constexpr (WR > 1) __syncthreads();
    const int mr = wr * MR + c;
    const auto part_row = [&](int w, int r) {
      return reinterpret_cast<float*>(lds + (WR == 1 ? w : w - 1) * kPart) + r * kPitch;
    };
    if (WR == 1 || wt != 0) {
      if (q4 == 0) {
        ml[(wt * M + mr) * 2] = base;
        ml[(wt * M + mr) * 2 + 1] = sum;
      }
      float* const dst = part_row(wt, mr) + 4 * q4;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < ACC; x += 4)
          *reinterpret_cast<Float4*>(dst + MR * d + 256 / MR * (x / 4)) =
              Float4{o[d][x], o[d][x + 1], o[d][x + 2], o[d][x + 3]};
    }
    __syncthreads();
    if constexpr (WR == 1) {
      for (int i = threadIdx.x; i < M * (DP / 4); i += 64 * NW) {
        const int r = i / (DP / 4), ch = 4 * (i % (DP / 4));
        float most = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < WT; ++w) most = fmaxf(most, ml[(w * M + r) * 2]);
        const float zero = most == -INFINITY ? 0.0f : most;
        Float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WT; ++w) {
          const float weight = __builtin_amdgcn_exp2f(ml[(w * M + r) * 2] - zero);
          total += ml[(w * M + r) * 2 + 1] * weight;
          v += *reinterpret_cast<const Float4*>(part_row(w, r) + ch) * weight;
        }
        if (odd)
          each_odd_token(row0 + r, [&](const uint8_t* values) {
            v += odd_part(four_values<T, FP8>(values, min(ch, p.D - 4)));
          });
        put(row0 + r, ch, v, most, total);
      }
      return;
    }
    if (wt != 0) return;
    const float mine_base = base;
#pragma unroll
    for (int w = 1; w < WT; ++w) base = fmaxf(base, ml[(w * M + mr) * 2]);
    const float zero = base == -INFINITY ? 0.0f : base;
    const float own_weight = __builtin_amdgcn_exp2f(mine_base - zero);
    sum *= own_weight;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] *= own_weight;
#pragma unroll 1
    for (int w = 1; w < WT; ++w) {
      const float weight = __builtin_amdgcn_exp2f(ml[(w * M + mr) * 2] - zero);
      sum += ml[(w * M + mr) * 2 + 1] * weight;
      const float* const src = part_row(w, mr) + 4 * q4;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < ACC; x += 4) {
          const Float4 v = *reinterpret_cast<const Float4*>(src + MR * d + 256 / MR * (x / 4));
          o[d][x] += v[0] * weight;
          o[d][x + 1] += v[1] * weight;
          o[d][x + 2] += v[2] * weight;
          o[d][x + 3] += v[3] * weight;
        }
    }
  }
  int again = row;  // where the row is, anew: there are no registers to keep it through the loop
  asm volatile("" : "+v"(again));
  if (odd)
    each_odd_token(again, [&](const uint8_t* values) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < ACC; x += 4) {
          const int ch = MR * d + 4 * q4 + 256 / MR * (x / 4);
          const Float4 v = odd_part(four_values<T, FP8>(values, min(ch, p.D - 4)));
#pragma unroll
          for (int j = 0; j < 4; ++j) o[d][x + j] += v[j];
        }
    });
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int x = 0; x < ACC; x += 4)
      put(again, MR * d + 4 * q4 + 256 / MR * (x / 4),
          Float4{o[d][x], o[d][x + 1], o[d][x + 2], o[d][x + 3]}, base, sum);
}

template <typename T, bool FP8, int DP, int SHAPE>
__device__ __forceinline__ void attend_shape(const AttendParams& p, int kind, int unit,
                                             uint8_t* lds, float* ml) {
  constexpr int MR = SHAPE == 0 || DP == 256 ? 16 : 32;
  attend<T, FP8, DP, MR, kShapeRows[SHAPE] / MR, kShapeWaves[SHAPE]>(p, p.group[kind], unit,
                                                                    kind == 0, lds, ml);
}

// The prefix in workgroups of shape S0 and the requests in those of S1, in one launch.
template <typename T, bool FP8, int DP, int S0, int S1>
__global__ __launch_bounds__(64 * kShapeWaves[S0], DP == 256 ? 1 : 2)
    void attend_kernel(AttendParams p) {
  __shared__ alignas(16) uint8_t lds[(S0 == 3 ? 768 : 512) * DP];
  __shared__ float ml[512];  // maxima and sums of the token waves' rows
  int unit = static_cast<int>(blockIdx.x);
  const int kind = unit >= p.group[0].units;
  unit -= kind ? p.group[0].units : 0;
  if (S0 == S1 || kind == 1)
    attend_shape<T, FP8, DP, S1>(p, S0 == S1 ? kind : 1, unit, lds, ml);
  else
    attend_shape<T, FP8, DP, S0>(p, 0, unit, lds, ml);
}

// Joins the parts of each row: out = v_scale sum_s w_s O_s / sum_s w_s l_s with
// w_s = 2^(m_s - max m).  For few parts: 4 channels a lane, `lanes` lanes a row.  Sums are loaded
// once it is known which there are: loading them beside the maxima cost 0.3 us of 12.2 for one
// request, and 30 of 530 for four prompts, whose parts are not all there.
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void join_few_kernel(AttendParams p, int lanes) {
  const int64_t all = static_cast<int64_t>(p.tokens) * p.Hq;
  const int64_t row =
      static_cast<int64_t>(blockIdx.x) * (kJoinThreads / lanes) + threadIdx.x / lanes;
  const int ch = 4 * (threadIdx.x % lanes);
  if (row >= all || ch >= p.D) return;
  const int64_t n = row / p.Hq, head = row - n * p.Hq;
  if (p.starts && (n < p.starts[0] || n >= p.starts[p.requests.d])) return;
  float m[kFewParts], l[kFewParts], best = -INFINITY, total = 0.0f;
#pragma unroll
  for (int s = 0; s < kFewParts; ++s) {
    const int64_t slot = min(s, p.slots - 1) * all + row;
    m[s] = p.part_ml[2 * slot];
    l[s] = s < p.slots ? p.part_ml[2 * slot + 1] : 0.0f;
    best = fmaxf(best, m[s]);
  }
  const float zero = best == -INFINITY ? 0.0f : best;
  Float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int s = 0; s < kFewParts; ++s)
    if (l[s] != 0.0f) {  // else no token: nothing was written
      const float w = __builtin_amdgcn_exp2f(m[s] - zero);
      total += l[s] * w;
      o += *reinterpret_cast<const Float4*>(p.part_o + (s * all + row) * p.D + ch) * w;
    }
  const float inv = total == 0.0f ? 0.0f : p.v_scale / total;
  store4(static_cast<T*>(p.out) + n * p.o_token + head * p.o_head + ch, o * inv, p.out_vec);
  if (p.lse && ch == 0) p.lse[row] = total == 0.0f ? -INFINITY : kLn2 * (best + log2f(total));
}

// For many parts: a workgroup takes `4 lanes` channels of one row.  It first lists the parts that
// have tokens with their weights, then its lane groups add them up in turn, several loads each on
// their way: 8 us for 128 rows of 412 parts, where one wave a row after the other took 55.  Waves
// meet three times; a tree of steps through LDS and maxima by its crossbar cost 0.5 us more.
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(AttendParams p, int lanes, int blocks) {
  __shared__ float weight[kMaxParts];
  __shared__ int which[kMaxParts];
  __shared__ float wave_best[kJoinWaves], wave_sum[kJoinWaves];
  __shared__ int counts[kMaxParts / kJoinThreads][kJoinWaves];
  __shared__ Float4 part[kJoinThreads];
  const int64_t all = static_cast<int64_t>(p.tokens) * p.Hq;
  const int64_t row = blockIdx.x / blocks;
  const int ch = 4 * (static_cast<int>(blockIdx.x % blocks) * lanes + threadIdx.x % lanes);
  const int team = threadIdx.x / lanes, teams = kJoinThreads / lanes;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t n = row / p.Hq, head = row - n * p.Hq;
  if (p.starts && (n < p.starts[0] || n >= p.starts[p.requests.d])) return;

  constexpr int kEach = kMaxParts / kJoinThreads;
  float m[kEach], l[kEach], best = -INFINITY;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int s = i * kJoinThreads + threadIdx.x;
    m[i] = -INFINITY;
    l[i] = 0.0f;
    if (s < p.slots) {
      m[i] = p.part_ml[2 * (s * all + row)];
      l[i] = p.part_ml[2 * (s * all + row) + 1];
    }
    best = fmaxf(best, m[i]);
  }
  best = fold_wave(best, [](float a, float b) { return fmaxf(a, b); });
  uint64_t has[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) has[i] = __ballot(l[i] != 0.0f);
  if (lane == 0) {
    wave_best[wave] = best;
#pragma unroll
    for (int i = 0; i < kEach; ++i) counts[i][wave] = __popcll(has[i]);
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) best = fmaxf(best, wave_best[w]);
  const float zero = best == -INFINITY ? 0.0f : best;
  float sum = 0.0f;
  int parts = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    int at = parts + __popcll(has[i] & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
      at += w < wave ? counts[i][w] : 0;
      parts += counts[i][w];
    }
    if (l[i] != 0.0f) {
      const float w = __builtin_amdgcn_exp2f(m[i] - zero);
      sum += l[i] * w;
      weight[at] = w;
      which[at] = i * kJoinThreads + threadIdx.x;
    }
  }
  sum = fold_wave(sum, [](float a, float b) { return a + b; });
  if (lane == 0) wave_sum[wave] = sum;
  __syncthreads();

  const float* const src = p.part_o + row * p.D + min(ch, p.D - 4);
  Float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = team; s < parts; s += teams)
    o += *reinterpret_cast<const Float4*>(src + which[s] * all * p.D) * weight[s];
  for (int x = lanes; x < 64; x <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], x);
  if (lane < lanes) part[wave * lanes + lane] = o;
  __syncthreads();
  if (team != 0 || ch >= p.D) return;
  float total = wave_sum[0];
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) {
    total += wave_sum[w];
    o += part[w * lanes + lane];
  }
  const float inv = total == 0.0f ? 0.0f : p.v_scale / total;
  store4(static_cast<T*>(p.out) + n * p.o_token + head * p.o_head + ch, o * inv, p.out_vec);
  if (p.lse && ch == 0) p.lse[row] = total == 0.0f ? -INFINITY : kLn2 * (best + log2f(total));
}

template <typename T, bool FP8, int DP, int S0, int S1>
int launch_shapes(const AttendParams& p, hipStream_t stream) {
  const dim3 grid(p.group[0].units + p.group[1].units), block(64 * kShapeWaves[S0]);
  hipLaunchKernelGGL((attend_kernel<T, FP8, DP, S0, S1>), grid, block, 0, stream, p);
  return check_launch("attend_kernel");
}

template <typename T, bool FP8, int DP>
int launch_units(const AttendParams& p, hipStream_t stream) {
  // the batch has at least a request's rows: s0 >= s1
  const int s1 = p.group[1].shape, s0 = p.group[0].units ? p.group[0].shape : s1;
  if constexpr (DP == 128)
    if (s0 == 3) return launch_shapes<T, FP8, DP, 3, 3>(p, stream);
  if constexpr (DP <= 128)
    if (s0 == 2)
      return s1 == 0   ? launch_shapes<T, FP8, DP, 2, 0>(p, stream)
             : s1 == 1 ? launch_shapes<T, FP8, DP, 2, 1>(p, stream)
                       : launch_shapes<T, FP8, DP, 2, 2>(p, stream);
  if constexpr (DP <= 128)
    if (s0 == 1 && s1 == 0) return launch_shapes<T, FP8, DP, 1, 0>(p, stream);
  if (s0 == 1) return launch_shapes<T, FP8, DP, 1, 1>(p, stream);
  return launch_shapes<T, FP8, DP, 0, 0>(p, stream);
}

template <typename T, bool FP8>
int launch_attend(const AttendParams& p, hipStream_t stream) {
  const int rc = p.D <= 64    ? launch_units<T, FP8, 64>(p, stream)
                 : p.D <= 128 ? launch_units<T, FP8, 128>(p, stream)
                              : launch_units<T, FP8, 256>(p, stream);
  if (rc) return rc;
  const dim3 block(kJoinThreads);
  if (p.slots == 1) return ORIGAMI_OK;
  const int lanes = p.D <= 64 ? 16 : (p.D <= 128 ? 32 : 64);  // of a whole row
  const int64_t rows = static_cast<int64_t>(p.tokens) * p.Hq, per = kJoinThreads / lanes;
  if (p.slots <= kFewParts) {
    const dim3 joins(static_cast<unsigned>((rows + per - 1) / per));
    hipLaunchKernelGGL(join_few_kernel<T>, joins, block, 0, stream, p, lanes);
  } else {
    // with few rows, workgroups of 32 channels, so that the GPU has enough of them
    const int some = rows < 2 * kCus ? 8 : lanes;
    const int blocks = (p.D + 4 * some - 1) / (4 * some);
    const dim3 joins(static_cast<unsigned>(rows * blocks));
    hipLaunchKernelGGL(join_kernel<T>, joins, block, 0, stream, p, some, blocks);
  }
  return check_launch("join_kernel");
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The split of a call into units, from sizes that the host has.
struct Plan {
  Group group[2];
  int64_t slots, units;
};

// Units of one kind, before they are split: `count` of them, `live` with rows if the requests are
// of one size, over `span` tokens; microseconds of a unit's start and end, and of a token.
struct Kind {
  int shape = 0;
  int64_t tiles = 0, count = 0, live = 0, span = 0, fill = kCus;
  double token = 0.0;

  int64_t chunk(int64_t splits) const { return ceil_div(ceil_div(span, splits), 64) * 64; }
  int64_t splits(int64_t wanted) const {
    const int64_t most = std::min<int64_t>(std::max<int64_t>(span / 128, 1), 2 * kCus);
    const int64_t s = std::min(std::max<int64_t>(wanted, 1), most);
    return span > 0 ? ceil_div(span, chunk(s)) : 1;
  }
};

// Measured on MI355X: microseconds that a workgroup takes besides its tokens, and bytes and
// operations of one CU in a microsecond while all of them work.  Times change by 2% at most where
// any of the three is half or twice as large: the split needs to be near only.
constexpr double kUnitTime = 6.0, kCuBytes = 20e3, kCuFlops = 3.2e6;

// Microseconds of a call whose kinds are split in s0 and s1 ranges: workgroups of the first kind go
// to the CUs in order, then those of the second; and joining the parts of `rows` rows.
double call_time(const Kind& k0, int64_t s0, const Kind& k1, int64_t s1, int64_t rows,
                 int64_t head_dim) {
  const int64_t n0 = k0.live * s0, n1 = k1.live * s1;
  const double t0 = n0 ? kUnitTime + k0.token * k0.chunk(s0) : 0.0;
  const double t1 = kUnitTime + k1.token * k1.chunk(s1);
  const int64_t full = n0 / k1.fill, rest = n0 % k1.fill, early = k1.fill - rest;
  double end = (rest ? full + 1 : full) * t0;
  const int64_t beside = rest ? early * static_cast<int64_t>(t0 / t1) : 0;
  if (rest && n1 <= early)
    end = std::max(end, full * t0 + t1);
  else if (n1 > beside)
    end += ceil_div(n1 - beside, k1.fill) * t1;
  const int64_t slots = s1 + (n0 ? s0 : 0);
  return end + (slots > 1 ? 4.0 + slots * rows * head_dim * 8 / (kCus * kCuBytes) : 0.0);
}

Plan plan_of(int64_t tokens, int64_t query_heads, int64_t heads, int64_t head_dim,
             int64_t prefix, int64_t requests, int64_t max_query, int64_t max_own, int64_t cell) {
  const int64_t G = query_heads / heads, last = head_dim <= 128 ? 2 : 1;
  // Where the bound of a request's rows fills workgroups by itself, every request reads the prefix
  // with its own tokens; that is slow for requests of few rows beside one of many.
  const bool apart = requests > 1 && prefix > 0 && max_query * G < kShapeRows[last];
  const auto kind_of = [&](int shape, int64_t n, int64_t rows, int64_t all_rows, int64_t span) {
    Kind k;
    k.shape = shape;
    while (k.shape < last && rows > kShapeRows[k.shape]) ++k.shape;
    if (!apart && k.shape == 2 && rows > kShapeRows[2] && head_dim > 64) k.shape = 3;
    const int64_t unit_rows = kShapeRows[k.shape];
    k.tiles = std::max<int64_t>(ceil_div(rows, unit_rows), 1);
    k.count = n * heads * k.tiles;
    k.live = std::max<int64_t>(
        std::min(k.count, heads * (ceil_div(all_rows, unit_rows) + n / 2)), 1);
    k.span = span;
    k.fill = head_dim <= 128 && k.shape < 3 ? 2 * kCus : kCus;  // workgroups that the CUs hold
    k.token = k.fill / kCus * std::max(2.0 * head_dim * cell / kCuBytes,
                                     4.0 * head_dim * unit_rows / kCuFlops);
    return k;
  };
  Kind k0;
  if (apart) k0 = kind_of(0, 1, tokens * G, tokens * G, prefix);
  // past 128 channels the kinds have one shape: two there do not fit the scalar registers
  const Kind k1 = kind_of(head_dim > 128 ? k0.shape : 0, requests, max_query * G, tokens * G,
                          (apart ? 0 : prefix) + max_own);
  // The requests' ranges are tried in a few sizes, the prefix's so that all workgroups are one to
  // four rounds on the CUs.
  int64_t best0 = 1, best1 = 1;
  double least = 0.0;
  for (const int64_t want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 64, 128, 256}) {
    const int64_t s1 = k1.splits(want);
    for (int round = 1; round <= 4; ++round) {
      const int64_t s0 = apart ? k0.splits((k1.fill * round - k1.live * s1) / k0.live) : 1;
      const double time = call_time(k0, s0, k1, s1, tokens * query_heads, head_dim);
      if (least == 0.0 || time < least) {
        least = time;
        best0 = s0;
        best1 = s1;
      }
      if (!apart) break;
    }
    if (s1 < want) break;
  }
  Plan plan{};
  const auto put = [&](Group& g, const Kind& k, int64_t splits, int64_t first) {
    const int64_t units = ceil_div(k.count / k.tiles * splits, 8) * 8 * k.tiles;
    plan.units += units;
    g.units = static_cast<int32_t>(std::min<int64_t>(units, INT32_MAX));
    g.shape = k.shape;
    g.tiles = divisor(k.tiles);
    g.splits = static_cast<int32_t>(splits);
    g.chunk = static_cast<int32_t>(k.chunk(splits));
    g.slot = static_cast<int32_t>(plan.slots);  // of the partial results
    g.first = static_cast<int32_t>(first);
    plan.slots += splits;
  };
  if (apart) put(plan.group[0], k0, best0, 0);
  put(plan.group[1], k1, best1, apart ? prefix : 0);
  return plan;
}

int64_t workspace_bytes_of(const Plan& plan, int64_t tokens, int64_t query_heads,
                           int64_t head_dim) {
  return plan.slots > 1 ? plan.slots * tokens * query_heads * (head_dim + 2) * 4 : 0;
}

// A request's query tokens at most: no more than there are, and one, which each has where no
// query_starts say otherwise.
int64_t bound_of_queries(int64_t max_query, int64_t tokens) {
  return std::max<int64_t>(std::min(max_query, tokens), 1);
}

int check_sizes(int64_t tokens, int64_t query_heads, int64_t heads, int64_t head_dim,
                int64_t prefix_tokens, int64_t requests, int64_t max_query, int64_t max_own) {
  ORIGAMI_REQUIRE(heads > 0 && query_heads > 0 && query_heads % heads == 0,
                  "query heads must be a multiple of the cache's heads");
  ORIGAMI_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 256,
                  "head_dim must be a multiple of 8, at most 256");
  ORIGAMI_REQUIRE(tokens >= 0 && requests >= 0 && prefix_tokens >= 0 && max_query >= 0 &&
                      max_own >= 0,
                  "token counts must not be negative");
  constexpr int64_t kMostTokens = int64_t(1) << 30;
  ORIGAMI_REQUIRE(prefix_tokens <= kMostTokens && max_own <= kMostTokens - prefix_tokens,
                  "too many tokens for one call");
  // a launch has at most 2^32 threads in x; every request has a workgroup a head at least
  ORIGAMI_REQUIRE(tokens < (int64_t(1) << 24) / query_heads, "too many query rows for one call");
  ORIGAMI_REQUIRE(requests < kMostUnits / heads, "too many requests for one call");
  return ORIGAMI_OK;
}

}  // namespace

extern "C" {

int64_t origami_shared_prefix_attention_workspace(int64_t tokens, int64_t query_heads,
                                                  int64_t heads, int64_t head_dim,
                                                  int64_t prefix_tokens, int64_t requests,
                                                  int64_t max_query_tokens,
                                                  int64_t max_own_tokens, int64_t cache_dtype) {
  const int64_t cell_bytes = cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN ? 1 : 2;
  if (check_sizes(tokens, query_heads, heads, head_dim, prefix_tokens, requests, max_query_tokens,
                  max_own_tokens))
    return -1;
  max_query_tokens = bound_of_queries(max_query_tokens, tokens);
  return workspace_bytes_of(plan_of(tokens, query_heads, heads, head_dim, prefix_tokens,
                                    requests, max_query_tokens, max_own_tokens, cell_bytes),
                            tokens, query_heads, head_dim);
}

int origami_shared_prefix_attention(
    const void* query, int64_t dtype, const int64_t* strides, int64_t tokens, int64_t query_heads,
    const void* kv_cache, int64_t cache_dtype, int64_t cache_layout, int64_t num_blocks,
    int64_t block_size, int64_t heads, int64_t head_dim, const int64_t* prefix_block_ids,
    int64_t prefix_block_count, int64_t prefix_tokens, const int64_t* block_tables,
    int64_t table_stride, int64_t table_blocks, const int64_t* own_tokens, int64_t requests,
    const int64_t* query_starts, int64_t max_query_tokens, int64_t max_own_tokens, double scale,
    double k_scale, double v_scale, void* out, float* lse, void* workspace,
    int64_t workspace_bytes, origami_stream_t stream_) {
  AttendParams p{};
  ORIGAMI_REQUIRE(dtype == ORIGAMI_DTYPE_FLOAT16 || dtype == ORIGAMI_DTYPE_BFLOAT16,
                  "queries must be float16 or bfloat16");
  ORIGAMI_REQUIRE(cache_dtype == dtype || cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN,
                  "kv_cache must have the queries' dtype or be float8_e4m3fn");
  if (int rc = check_sizes(tokens, query_heads, heads, head_dim, prefix_tokens, requests,
                           max_query_tokens, max_own_tokens))
    return rc;
  ORIGAMI_REQUIRE(num_blocks >= 0 && block_size > 0, "cache block size must be positive");
  if (int rc = cache_geometry(cache_layout, num_blocks, block_size, &p.blk_stride,
                              &p.half_stride))
    return rc;
  ORIGAMI_REQUIRE(block_size <= INT32_MAX / 2 / std::max<int64_t>(num_blocks, 1),
                  "the cache has too many token slots");
  ORIGAMI_REQUIRE(prefix_block_count >= 0 && table_blocks >= 0 &&
                      ceil_div(prefix_tokens, block_size) <= prefix_block_count,
                  "prefix tokens exceed the prefix blocks");
  ORIGAMI_REQUIRE(ceil_div(max_own_tokens, block_size) <= table_blocks,
                  "max_own_tokens exceeds the block tables");
  ORIGAMI_REQUIRE(query_starts != nullptr || tokens == requests,
                  "without query_starts every request has one query token");
  max_query_tokens = bound_of_queries(max_query_tokens, tokens);
  ORIGAMI_REQUIRE(cache_scale(k_scale) && cache_scale(v_scale),
                  "cache scales must be positive and finite in binary32");
  const float log2_scale = static_cast<float>(scale * k_scale) * kLog2e;
  ORIGAMI_REQUIRE(std::isfinite(log2_scale), "scale must be finite in binary32");
  ORIGAMI_REQUIRE(cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN || (k_scale == 1.0 && v_scale == 1.0),
                  "cache scales are for float8_e4m3fn caches");
  ORIGAMI_REQUIRE(aligned16(kv_cache), "kv_cache must be 16-byte aligned");
  for (int i = 0; i < 4; ++i)
    ORIGAMI_REQUIRE(strides[i] >= 0, "row strides must not be negative");
  ORIGAMI_REQUIRE(table_stride >= 0, "the table stride must not be negative");
  if (tokens == 0 || requests == 0) return ORIGAMI_OK;
  ORIGAMI_REQUIRE(query != nullptr && out != nullptr && own_tokens != nullptr &&
                      (kv_cache != nullptr || num_blocks == 0) &&
                      (prefix_block_ids != nullptr || prefix_tokens == 0) &&
                      (block_tables != nullptr || max_own_tokens == 0),
                  "queries, output, lengths, tables and the cache must not be null");

  const bool fp8 = cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN;
  const Plan plan = plan_of(tokens, query_heads, heads, head_dim, prefix_tokens, requests,
                            max_query_tokens, max_own_tokens, fp8 ? 1 : 2);
  ORIGAMI_REQUIRE(plan.units < kMostUnits, "too many row tiles for one call");
  ORIGAMI_REQUIRE(workspace_bytes >= workspace_bytes_of(plan, tokens, query_heads, head_dim) &&
                      (plan.slots == 1 || workspace != nullptr) && aligned16(workspace),
                  "attention workspace is too small");
  p.query = query;
  p.q_token = strides[0];
  p.q_head = strides[1];
  p.out = out;
  p.o_token = strides[2];
  p.o_head = strides[3];
  p.out_vec = ((reinterpret_cast<uintptr_t>(out) | 2 * strides[2] | 2 * strides[3]) & 7) == 0;
  p.lse = lse;
  p.cache = static_cast<const uint8_t*>(kv_cache);
  p.num_blocks = num_blocks;
  p.prefix_ids = prefix_block_ids;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.own_tokens = own_tokens;
  p.starts = query_starts;
  p.block_size = divisor(block_size);
  p.prefix = static_cast<int32_t>(prefix_tokens);
  p.max_own = static_cast<int32_t>(max_own_tokens);
  p.max_query = static_cast<int32_t>(max_query_tokens);
  p.tokens = static_cast<int32_t>(tokens);
  p.requests = divisor(requests);
  p.Hq = static_cast<int32_t>(query_heads);
  p.H = divisor(heads);
  p.G = divisor(query_heads / heads);
  p.D = static_cast<int32_t>(head_dim);
  p.scale = log2_scale;
  p.v_scale = static_cast<float>(v_scale);
  p.group[0] = plan.group[0];
  p.group[1] = plan.group[1];
  p.slots = static_cast<int32_t>(plan.slots);
  const int64_t parts = plan.slots * tokens * query_heads;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + parts * head_dim;
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (dtype == ORIGAMI_DTYPE_BFLOAT16)
    return fp8 ? launch_attend<bf16, true>(p, stream) : launch_attend<bf16, false>(p, stream);
  return fp8 ? launch_attend<f16, true>(p, stream) : launch_attend<f16, false>(p, stream);
}

}  // extern "C"
