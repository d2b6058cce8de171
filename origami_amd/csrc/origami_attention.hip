// origami_attention.hip -- attention over the paged KV cache for a batch that shares a prefix.
//
// For a query row q (one token, one query head) over the keys k_t and values v_t it sees:
//   s_t = scale * (q . k_t),  out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  m = max_t s_t
// The tokens come in parts (the prefix, the request's own tokens, ranges of either).  A part
// gives m, the sum l and the unnormalised row O in binary32; parts are joined with the weights
// exp(m_part - m), so that no part waits for another.
#include <type_traits>

#include "origami_element.h"
#include "origami_internal.h"

namespace {

using namespace origami_element;
using origami_internal::aligned16;
using origami_internal::cache_geometry;
using origami_internal::check_launch;
using origami_internal::fail;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kStep = 32;  // tokens of one product P V (the depth of its matrix instruction)
// Exponentials are taken 2^kLift times as large for half precision, so that those of tokens far
// below the maximum keep their precision (down to 2^-24 of the largest) and sums of 2^30 of
// the largest stay far from binary32's limit.
template <typename T>
constexpr float kLift = std::is_same<T, f16>::value ? 10.0f : 0.0f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The work of one kind: row tiles of every KV head, over ranges of tokens.
struct Group {
  int32_t units;   // workgroups
  int32_t tiles;   // row tiles of a request, or of the batch
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
  float* lse;  // [tokens, query heads], or null
  const uint8_t* cache;
  int64_t blk_stride, half_stride;  // rows of H * D, as cache_geometry
  int64_t num_blocks;
  const int64_t *prefix_ids, *tables, *own_tokens, *starts;
  int64_t table_stride;
  int32_t block_size, prefix, max_own, max_query;
  int32_t tokens, requests, Hq, H, G, D;
  float scale, v_scale;  // scale includes log2 e and the keys' scale
  Group shared, each;    // the prefix with the whole batch's rows; each request's rows
  int32_t slots;
  float *part_o, *part_ml;  // [slots][rows][D], [slots][rows][2]
};

template <typename T>
__device__ __forceinline__ Float4 mfma16(Vec8<T> a, Vec8<T> b, Float4 c);
template <>
__device__ __forceinline__ Float4 mfma16<bf16>(Vec8<bf16> a, Vec8<bf16> b, Float4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ Float4 mfma16<f16>(Vec8<f16> a, Vec8<f16> b, Float4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

typedef short Short4 __attribute__((ext_vector_type(4)));

// Four tokens' values of one channel: 16 lanes read four rows of 16 channels, 8 bytes a lane
// (lane 4 k + q: channels 4 q .. 4 q + 3 of row k), and each gets its channel's column.
__device__ __forceinline__ U32x2 read_column(const uint8_t* p) {
  return __builtin_bit_cast(U32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) Short4*)p));
}

// Whether one of the two 16-bit values in `w` is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, bf16>::value ? 0x7f80u : 0x7c00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

// A request's place in the batch.
struct Request {
  int32_t first, count;  // its query tokens
  int32_t own;           // its own tokens
};

__device__ __forceinline__ Request request_of(const AttendParams& p, int r) {
  Request q{r, 1, 0};
  if (p.starts) {
    const int64_t n = p.tokens;
    const int64_t a = min(max(p.starts[r], int64_t(0)), n);
    const int64_t b = min(max(p.starts[r + 1], a), n);
    q.first = static_cast<int32_t>(a);
    q.count = static_cast<int32_t>(min(b - a, static_cast<int64_t>(p.max_query)));
  }
  q.own = static_cast<int32_t>(
      min(max(p.own_tokens[r], int64_t(0)), static_cast<int64_t>(p.max_own)));
  return q;
}

// One workgroup: 16 MT rows of one KV head over a range of tokens, which its four waves take
// in turn, 32 at a time.  A wave holds its rows' queries and results in registers and its
// tokens' keys and values in LDS, and needs no other wave until the end.
template <typename T, bool FP8, int DP, int MT>
__device__ void attend(const AttendParams& p, const Group& g, int unit, bool batch, uint8_t* lds) {
  constexpr int KS = DP / 32, DT = DP / 16;    // depth steps of Q K, channel tiles of P V
  constexpr int NCH = DP / 8;                  // 16-byte pieces of a row in LDS
  constexpr int RPI = 64 / NCH, IT = kStep / RPI;  // rows of one load, loads of a step
  constexpr int M = 16 * MT;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;

  // the unit: KV head fastest
  int u = unit;
  const int h = u % p.H;
  u /= p.H;
  int r = 0;
  Request rq{0, p.tokens, 0};
  if (!batch) {
    r = u % p.requests;
    u /= p.requests;
    rq = request_of(p, r);
  }
  const int tile = u % g.tiles, split = u / g.tiles;
  const int rows = rq.count * p.G, row0 = tile * M;
  if (row0 >= rows) return;
  const int end = batch ? p.prefix : p.prefix + rq.own;  // of the tokens, prefix first
  const int64_t* const table = p.tables + static_cast<int64_t>(r) * p.table_stride;

  // this lane's rows
  int limit[MT];  // tokens the row sees
  int64_t at[MT];  // its row of the partial results, -1 past the last
  Vec8<T> qf[MT][KS];
  int most = 0, least = INT32_MAX;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = row0 + 16 * m + c;
    const bool live = row < rows;
    const int i = live ? row / p.G : 0, head = h * p.G + (live ? row - i * p.G : 0);
    limit[m] = batch ? p.prefix : p.prefix + min(max(rq.own - rq.count + i + 1, 0), rq.own);
    const int64_t n = rq.first + i;
    at[m] = live ? n * p.Hq + head : -1;
    const T* const src = static_cast<const T*>(p.query) + n * p.q_token + head * p.q_head;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int d = 32 * k + 8 * q4;
      qf[m][k] = Vec8<T>{};
      if (live && d < p.D) {
        if (((reinterpret_cast<uintptr_t>(p.query) | 2 * p.q_token | 2 * p.q_head) & 15) == 0) {
          qf[m][k] = *reinterpret_cast<const Vec8<T>*>(src + d);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) qf[m][k][j] = src[d + j];
        }
      }
    }
    if (live) {
      most = max(most, limit[m]);
      least = min(least, limit[m]);
    }
  }
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) {
    most = max(most, __shfl_xor(most, x));
    least = min(least, __shfl_xor(least, x));
  }
  const int t0 = g.first + split * g.chunk;
  const int t1 = min(min(end, most), t0 + g.chunk);

  Float4 o[MT][DT];
  float top[MT], sum[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    top[m] = -INFINITY;
    sum[m] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[m][d] = Float4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  constexpr int kTile = kStep * DP * 2;  // bytes of a wave's keys
  uint8_t* const ks = lds + wave * 2 * kTile;
  uint8_t* const vs = ks + kTile;
  const int piece = lane % NCH, sub = lane / NCH;
  const bool has = 8 * piece < p.D;
  const int64_t cell = FP8 ? 1 : 2;
  const int64_t pitch = static_cast<int64_t>(p.H) * p.D * cell;
  const int64_t col = (static_cast<int64_t>(h) * p.D + 8 * piece) * cell;
  const int64_t vhalf = p.half_stride * pitch;

  // the cache row of token t, -1 where it has none
  const auto cache_row = [&](int t) -> int {
    if (t >= t1) return -1;
    const bool pre = t < p.prefix;
    const int i = pre ? t : t - p.prefix, b = i / p.block_size;
    const int64_t id = pre ? p.prefix_ids[b] : table[b];
    if (id < 0 || id >= p.num_blocks) return -1;
    return static_cast<int>(id * p.blk_stride + (i - b * p.block_size));
  };

  for (int t = t0 + wave * kStep; t < t1; t += kWaves * kStep) {
    const int mine = cache_row(t + (lane & 31));
    const uint32_t there = static_cast<uint32_t>(__ballot(mine >= 0));
    // keys and values of 32 tokens into LDS, zero where there are none
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int tok = i * RPI + sub;
      const int at_row = __shfl(mine, tok);
      U32x4 kv = {}, vv = {};
      if (at_row >= 0 && has) {
        const uint8_t* const src = p.cache + at_row * pitch + col;
        if constexpr (FP8) {
          kv = fp8_expand<T>(*reinterpret_cast<const U32x2*>(src));
          vv = fp8_expand<T>(*reinterpret_cast<const U32x2*>(src + vhalf));
        } else {
          kv = *reinterpret_cast<const U32x4*>(src);
          vv = *reinterpret_cast<const U32x4*>(src + vhalf);
        }
      }
      *reinterpret_cast<U32x4*>(ks + (tok * NCH + piece) * 16) = kv;
      *reinterpret_cast<U32x4*>(vs + (tok * NCH + piece) * 16) = vv;
    }
    __builtin_amdgcn_wave_barrier();

    // S = K Q: token 16 s + 4 q4 + i against row c
    Float4 sc[MT][2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int m = 0; m < MT; ++m) sc[m][s] = Float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const Vec8<T> kf =
            *reinterpret_cast<const Vec8<T>*>(ks + ((16 * s + c) * NCH + 4 * k + q4) * 16);
#pragma unroll
        for (int m = 0; m < MT; ++m) sc[m][s] = mfma16<T>(kf, qf[m][k], sc[m][s]);
      }
    }
    const bool whole = there == 0xffffffffu && t + kStep <= least;
    Vec8<T> pf[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float best = top[m];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = 16 * s + 4 * q4 + i;
          float v = sc[m][s][i] * p.scale;
          if (!whole && (t + tok >= limit[m] || !((there >> tok) & 1))) v = -INFINITY;
          sc[m][s][i] = v;
          best = fmaxf(best, v);
        }
      best = fmaxf(best, __shfl_xor(best, 16));
      best = fmaxf(best, __shfl_xor(best, 32));
      const float keep = __builtin_amdgcn_exp2f(top[m] - (best == -INFINITY ? 0.0f : best));
      const float base = best == -INFINITY ? 0.0f : best - kLift<T>;
      top[m] = best;
      sum[m] *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[m][d] *= keep;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(sc[m][s][i] - base);
          sum[m] += e;
          pf[m][4 * s + i] = static_cast<T>(e);
        }
    }
    // O += V P: channel 16 d + 4 q4 + i of row c
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      U32x4 vf;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int tok = 16 * s + 4 * q4 + (c >> 2);
        const U32x2 w = read_column(vs + (tok * NCH + 2 * d + ((c & 3) >> 1)) * 16 + (c & 1) * 8);
        vf[2 * s] = w[0];
        vf[2 * s + 1] = w[1];
      }
      if (!whole && __any(not_finite<T>(vf[0]) || not_finite<T>(vf[1]) || not_finite<T>(vf[2]) ||
                          not_finite<T>(vf[3]))) {
        // an infinity or NaN reaches only the rows that see its token: row by row, with the
        // tokens that the row does not see taken as zero
        for (int m = 0; m < MT; ++m)
          for (int x = 0; x < 16; ++x) {
            const int lim = __shfl(limit[m], x);
            Vec8<T> v = __builtin_bit_cast(Vec8<T>, vf);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (t + 16 * (j >> 2) + 4 * q4 + (j & 3) >= lim) v[j] = static_cast<T>(0.0f);
            const Float4 add = mfma16<T>(v, pf[m], Float4{0.0f, 0.0f, 0.0f, 0.0f});
            if (x == c) o[m][d] += add;
          }
        continue;
      }
      const Vec8<T> v = __builtin_bit_cast(Vec8<T>, vf);
#pragma unroll
      for (int m = 0; m < MT; ++m) o[m][d] = mfma16<T>(v, pf[m], o[m][d]);
    }
    __builtin_amdgcn_wave_barrier();
  }

  // join the waves: the largest maximum, then the weighted sums
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    sum[m] += __shfl_xor(sum[m], 16);
    sum[m] += __shfl_xor(sum[m], 32);
  }
  __syncthreads();
  float* const ml = reinterpret_cast<float*>(lds);  // [wave][M][2]
  float* const ol = ml + kWaves * M * 2;            // [M][DP + 4], one wave after the other
  constexpr int kPitch = DP + 4;
  if (q4 == 0)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      ml[(wave * M + 16 * m + c) * 2] = top[m];
      ml[(wave * M + 16 * m + c) * 2 + 1] = sum[m];
    }
  __syncthreads();
  float best[MT], total[MT], weight[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    best[m] = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) best[m] = fmaxf(best[m], ml[(w * M + 16 * m + c) * 2]);
    const float base = best[m] == -INFINITY ? 0.0f : best[m];
    total[m] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      total[m] += ml[(w * M + 16 * m + c) * 2 + 1] *
                  __builtin_amdgcn_exp2f(ml[(w * M + 16 * m + c) * 2] - base);
    weight[m] = __builtin_amdgcn_exp2f(top[m] - base);
  }
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          Float4* const dst =
              reinterpret_cast<Float4*>(ol + (16 * m + c) * kPitch + 16 * d + 4 * q4);
          o[m][d] *= weight[m];
          if (w > 0) o[m][d] += *dst;
          *dst = o[m][d];
        }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (at[m] < 0) continue;
    if (p.slots > 1) {
      const int64_t all = static_cast<int64_t>(p.tokens) * p.Hq;
      const int64_t slot = (g.slot + split) * all + at[m];
      if (q4 == 0) {
        p.part_ml[2 * slot] = best[m] - kLift<T>;
        p.part_ml[2 * slot + 1] = total[m];
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int ch = 16 * d + 4 * q4;
        if (ch < p.D)
          *reinterpret_cast<Float4*>(p.part_o + slot * p.D + ch) =
              *reinterpret_cast<const Float4*>(ol + (16 * m + c) * kPitch + ch);
      }
    } else {
      const float inv = total[m] == 0.0f ? 0.0f : p.v_scale / total[m];
      const int64_t n = at[m] / p.Hq, head = at[m] - n * p.Hq;
      T* const dst = static_cast<T*>(p.out) + n * p.o_token + head * p.o_head;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int ch = 16 * d + 4 * q4;
        if (ch < p.D) {
          const Float4 v = *reinterpret_cast<const Float4*>(ol + (16 * m + c) * kPitch + ch);
#pragma unroll
          for (int j = 0; j < 4; ++j) dst[ch + j] = static_cast<T>(v[j] * inv);
        }
      }
      if (p.lse && q4 == 0)
        p.lse[at[m]] = total[m] == 0.0f ? -INFINITY : kLn2 * (best[m] - kLift<T> + log2f(total[m]));
    }
  }
}

template <typename T, bool FP8, int DP>
__global__ __launch_bounds__(kThreads) void attend_kernel(AttendParams p) {
  __shared__ alignas(16) uint8_t lds[kWaves * 2 * kStep * DP * 2];
  const int unit = static_cast<int>(blockIdx.x);
  if (unit < p.shared.units)
    attend<T, FP8, DP, 1>(p, p.shared, unit, true, lds);
  else
    attend<T, FP8, DP, 1>(p, p.each, unit - p.shared.units, false, lds);
}

// Joins the parts of each row: 4 channels a lane.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(AttendParams p, int lanes) {
  const int64_t all = static_cast<int64_t>(p.tokens) * p.Hq;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / lanes) + threadIdx.x / lanes;
  const int ch = 4 * (threadIdx.x % lanes);
  if (row >= all) return;
  const int64_t n = row / p.Hq, head = row - n * p.Hq;
  if (p.starts && (n < p.starts[0] || n >= p.starts[p.requests])) return;
  float best = -INFINITY;
  for (int s = 0; s < p.slots; ++s) best = fmaxf(best, p.part_ml[2 * (s * all + row)]);
  const float base = best == -INFINITY ? 0.0f : best;
  float total = 0.0f;
  Float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < p.slots; ++s) {
    const int64_t slot = s * all + row;
    const float l = p.part_ml[2 * slot + 1];
    if (l == 0.0f) continue;  // no token: nothing was written
    const float w = __builtin_amdgcn_exp2f(p.part_ml[2 * slot] - base);
    total += l * w;
    if (ch < p.D) o += *reinterpret_cast<const Float4*>(p.part_o + slot * p.D + ch) * w;
  }
  const float inv = total == 0.0f ? 0.0f : p.v_scale / total;
  T* const dst = static_cast<T*>(p.out) + n * p.o_token + head * p.o_head;
  if (ch < p.D)
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[ch + j] = static_cast<T>(o[j] * inv);
  if (p.lse && ch == 0) p.lse[row] = total == 0.0f ? -INFINITY : kLn2 * (best + log2f(total));
}

template <typename T, bool FP8>
int launch_attend(const AttendParams& p, hipStream_t stream) {
  const dim3 grid(p.shared.units + p.each.units), block(kThreads);
  if (p.D <= 64)
    hipLaunchKernelGGL((attend_kernel<T, FP8, 64>), grid, block, 0, stream, p);
  else if (p.D <= 128)
    hipLaunchKernelGGL((attend_kernel<T, FP8, 128>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((attend_kernel<T, FP8, 256>), grid, block, 0, stream, p);
  if (int rc = check_launch("attend_kernel")) return rc;
  if (p.slots == 1) return ORIGAMI_OK;
  const int lanes = p.D <= 64 ? 16 : (p.D <= 128 ? 32 : 64);
  const int64_t rows = static_cast<int64_t>(p.tokens) * p.Hq, per = kThreads / lanes;
  hipLaunchKernelGGL(join_kernel<T>, dim3(static_cast<unsigned>((rows + per - 1) / per)), block, 0,
                     stream, p, lanes);
  return check_launch("join_kernel");
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The split of a call into units, from sizes that the host has.
struct Plan {
  Group shared, each;
  int64_t slots, units;
};

Plan plan_of(int64_t tokens, int64_t query_heads, int64_t heads, int64_t prefix,
             int64_t requests, int64_t max_query, int64_t max_own) {
  Plan plan{};
  const int64_t G = query_heads / heads, M = 16;
  const bool apart = requests > 1 && prefix > 0;
  const int64_t chunk = 512;
  int64_t units = 0, slot = 0;
  const auto fill = [&](Group& g, int64_t n, int64_t rows, int64_t first, int64_t span) {
    const int64_t splits = span > 0 ? ceil_div(span, chunk) : 1, tiles = ceil_div(rows, M);
    units += n * heads * tiles * splits;
    g.units = static_cast<int32_t>(n * heads * tiles * splits);
    g.tiles = static_cast<int32_t>(tiles);
    g.splits = static_cast<int32_t>(splits);
    g.chunk = static_cast<int32_t>(chunk);
    g.slot = static_cast<int32_t>(slot);
    g.first = static_cast<int32_t>(first);
    slot += splits;
  };
  if (apart) fill(plan.shared, 1, tokens * G, 0, prefix);
  fill(plan.each, requests, max_query * G, apart ? prefix : 0, (apart ? 0 : prefix) + max_own);
  plan.slots = slot;
  plan.units = units;
  return plan;
}

int64_t workspace_bytes_of(const Plan& plan, int64_t tokens, int64_t query_heads,
                           int64_t head_dim) {
  return plan.slots > 1 ? plan.slots * tokens * query_heads * (head_dim + 2) * 4 : 0;
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
  ORIGAMI_REQUIRE(max_query <= tokens, "max_query_tokens exceeds the query tokens");
  ORIGAMI_REQUIRE(prefix_tokens + max_own <= (int64_t(1) << 30), "too many tokens for one call");
  ORIGAMI_REQUIRE(tokens <= INT32_MAX / query_heads, "too many query rows for one call");
  return ORIGAMI_OK;
}

}  // namespace

extern "C" {

int64_t origami_shared_prefix_attention_workspace(int64_t tokens, int64_t query_heads,
                                                  int64_t heads, int64_t head_dim,
                                                  int64_t prefix_tokens, int64_t requests,
                                                  int64_t max_query_tokens,
                                                  int64_t max_own_tokens) {
  if (check_sizes(tokens, query_heads, heads, head_dim, prefix_tokens, requests, max_query_tokens,
                  max_own_tokens))
    return -1;
  return workspace_bytes_of(plan_of(tokens, query_heads, heads, prefix_tokens, requests,
                                    max_query_tokens, max_own_tokens),
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
  ORIGAMI_REQUIRE(num_blocks == 0 || block_size <= INT32_MAX / 2 / num_blocks,
                  "the cache has too many token slots");
  ORIGAMI_REQUIRE(prefix_block_count >= 0 && table_blocks >= 0 &&
                      ceil_div(prefix_tokens, block_size) <= prefix_block_count,
                  "prefix tokens exceed the prefix blocks");
  ORIGAMI_REQUIRE(ceil_div(max_own_tokens, block_size) <= table_blocks,
                  "max_own_tokens exceeds the block tables");
  ORIGAMI_REQUIRE(query_starts != nullptr || (tokens == requests && max_query_tokens <= 1),
                  "without query_starts every request has one query token");
  ORIGAMI_REQUIRE(k_scale > 0.0 && v_scale > 0.0, "cache scales must be positive");
  ORIGAMI_REQUIRE(cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN || (k_scale == 1.0 && v_scale == 1.0),
                  "cache scales are for float8_e4m3fn caches");
  ORIGAMI_REQUIRE(aligned16(kv_cache), "kv_cache must be 16-byte aligned");
  if (tokens == 0 || requests == 0) return ORIGAMI_OK;

  const Plan plan = plan_of(tokens, query_heads, heads, prefix_tokens, requests, max_query_tokens,
                            max_own_tokens);
  ORIGAMI_REQUIRE(plan.units <= INT32_MAX, "too many row tiles for one call");
  ORIGAMI_REQUIRE(workspace_bytes >= workspace_bytes_of(plan, tokens, query_heads, head_dim) &&
                      (plan.slots == 1 || workspace != nullptr) && aligned16(workspace),
                  "attention workspace is too small");
  p.query = query;
  p.q_token = strides[0];
  p.q_head = strides[1];
  p.out = out;
  p.o_token = strides[2];
  p.o_head = strides[3];
  p.lse = lse;
  p.cache = static_cast<const uint8_t*>(kv_cache);
  p.num_blocks = num_blocks;
  p.prefix_ids = prefix_block_ids;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.own_tokens = own_tokens;
  p.starts = query_starts;
  p.block_size = static_cast<int32_t>(block_size);
  p.prefix = static_cast<int32_t>(prefix_tokens);
  p.max_own = static_cast<int32_t>(max_own_tokens);
  p.max_query = static_cast<int32_t>(max_query_tokens);
  p.tokens = static_cast<int32_t>(tokens);
  p.requests = static_cast<int32_t>(requests);
  p.Hq = static_cast<int32_t>(query_heads);
  p.H = static_cast<int32_t>(heads);
  p.G = static_cast<int32_t>(query_heads / heads);
  p.D = static_cast<int32_t>(head_dim);
  p.scale = static_cast<float>(scale * k_scale) * kLog2e;
  p.v_scale = static_cast<float>(v_scale);
  p.shared = plan.shared;
  p.each = plan.each;
  p.slots = static_cast<int32_t>(plan.slots);
  const int64_t parts = plan.slots * tokens * query_heads;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + parts * head_dim;
  const hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const bool fp8 = cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN;
  if (dtype == ORIGAMI_DTYPE_BFLOAT16)
    return fp8 ? launch_attend<bf16, true>(p, stream) : launch_attend<bf16, false>(p, stream);
  return fp8 ? launch_attend<f16, true>(p, stream) : launch_attend<f16, false>(p, stream);
}

}  // extern "C"
